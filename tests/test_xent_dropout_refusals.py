"""Refusals of the cross entropy from hidden rows and of dropout at the C-ABI,
before anything is launched, on pointers that are never followed; the
generator's published answers; the copies' hazards.  No GPU needed."""

import math
import os
import shutil
import subprocess

import numpy as np
import pytest

from mi355x_pjrt import _lib
from test_asm_hazards import _COPY, HIPCC, KDIR, ROOT, hazards
from xent_dropout_ref import philox

BF16, F16, F32, F64, S16, S32, S64 = 13, 10, 11, 12, 3, 4, 5
P, Q, R = 1 << 20, 1 << 21, 1 << 22  # stand for aligned device memory


@pytest.fixture(scope="module")
def lib():
    return _lib.load_kernels()


def _refused(lib, code, word, rc):
    assert rc == code
    assert word in lib.mk_last_error().decode()


def test_loss(lib):
    def loss(t=BF16, rows=4, width=64, vocab=100, x=P, ldx=64, w=Q, ldw=64, lt=S32, labels=R, out=R, lse=R, ws=R):
        return lib.mk_linear_xent(None, t, rows, width, vocab, x, ldx, w, ldw, lt, labels, 1, -100, out, lse, ws)

    _refused(lib, 2, "io_type", loss(t=F64))
    _refused(lib, 2, "label_type", loss(lt=S16))
    for kw in (dict(rows=-1), dict(width=0), dict(vocab=0), dict(vocab=-5)):
        _refused(lib, 1, "shape", loss(**kw))
    _refused(lib, 1, "pitch", loss(ldx=-64))
    _refused(lib, 1, "pitch", loss(ldw=-1))
    for kw in (dict(rows=1 << 31), dict(vocab=1 << 31), dict(width=(1 << 20) + 1)):
        _refused(lib, 2, "at most", loss(**kw))
    for name in ("x", "w", "labels", "ws"):
        _refused(lib, 1, "null", loss(**{name: None}))
    for name, off in (("x", 1), ("w", 1), ("labels", 2), ("out", 2), ("lse", 1), ("ws", 8)):
        _refused(lib, 1, "aligned", loss(**{name: P + off}))
    _refused(lib, 2, "tiles", loss(rows=(1 << 31) - 1, vocab=(1 << 31) - 1))
    _refused(lib, 2, "tiles", loss(rows=1 << 30, vocab=2))
    assert loss(rows=0, x=None) == 0


def test_gradient(lib):
    def grad(t=BF16, dt=BF16, rows=4, width=64, vocab=100, x=P, ldx=64, w=Q, ldw=64, lt=S64, labels=R, lse=R, rg=None,
             dx=R, lddx=64, dw=2 * R, lddw=64, ws=R):
        return lib.mk_linear_xent_bwd(None, t, dt, rows, width, vocab, x, ldx, w, ldw, lt, labels, 0, 0, lse, rg, 1.0, dx,
                                      lddx, dw, lddw, ws)

    _refused(lib, 2, "io_type", grad(t=F64))
    _refused(lib, 2, "dw_type", grad(dt=F16))
    _refused(lib, 2, "dw_type", grad(t=F32, dt=BF16))
    _refused(lib, 1, "overlap", grad(lddx=63))
    _refused(lib, 1, "overlap", grad(lddw=63))
    _refused(lib, 1, "shape", grad(vocab=0))
    for name in ("x", "w", "labels", "lse", "ws"):
        _refused(lib, 1, "null", grad(**{name: None}))
    for name, off in (("x", 1), ("w", 1), ("labels", 4), ("lse", 2), ("rg", 2), ("dx", 1), ("dw", 1), ("ws", 4)):
        _refused(lib, 1, "aligned", grad(**{name: P + off}))
    _refused(lib, 1, "over x", grad(dx=P))
    _refused(lib, 1, "over w", grad(dw=Q))
    for kw in (dict(dx=Q), dict(dw=P), dict(dx=R, dw=R)):
        _refused(lib, 1, "over", grad(**kw))
    _refused(lib, 2, "tiles", grad(rows=(1 << 31) - 1, width=4096, vocab=2, ldx=4096, ldw=4096, lddx=4096, lddw=4096))
    assert grad(dx=None, dw=None) == 0
    assert grad(rows=0, dw=None) == 0


def test_workspaces(lib):
    """Sized by shapes and alignment alone; a copy of operands off the 16-byte boundaries is counted."""
    def loss(x, ldx, w, ldw, width=64):
        return lib.mk_linear_xent_workspace_bytes(BF16, 1000, width, 5000, x, ldx, w, ldw)

    plain = loss(P, 64, Q, 64)
    assert 0 < plain < 1000 * 5000 // 8  # far less than the logits
    assert loss(P + 2, 64, Q, 64) == plain + 1000 * 64 * 2
    assert loss(P, 65, Q, 64) == plain + 1000 * 64 * 2
    assert loss(P, 64, Q, 72) == plain
    assert loss(P, 64, Q + 8, 64) >= plain + 5000 * 64 * 2
    assert loss(P, 60, Q, 60, width=60) >= plain + 6000 * 64 * 2
    assert lib.mk_linear_xent_workspace_bytes(BF16, 0, 64, 5000, P, 64, Q, 64) == 0

    def grad(rows, vocab, ignore=0):
        return lib.mk_linear_xent_bwd_workspace_bytes(BF16, rows, 768, vocab, P, 768, Q, 768, ignore)

    # g of one piece, and sums of dx: not g of the whole vocabulary
    assert grad(65536, 131072) < 65536 * 131072 * 2 // 10
    assert grad(1000, 5000, 1) == grad(1000, 5000) + 1000 * 768 * 2
    assert lib.mk_dropout_add_bwd_workspace_bytes(0, 768) == 0
    # a partial row for each run of rows, never more than there are rows; and at most 1024 blocks
    # of 256 threads write them, 8 columns a thread, so no more than 1024 * 2048 numbers
    for rows in (1, 3, 1000, 1 << 20):
        for cols in (1, 100, 768, 1001, 16384):
            size = lib.mk_dropout_add_bwd_workspace_bytes(rows, cols)
            assert cols * 4 <= size <= min(rows * cols, 1024 * 2048) * 4


def test_dropout(lib):
    def fwd(t=BF16, rows=4, cols=64, x=P, ldx=64, b=None, r=None, ldr=64, p=0.1, step=None, out=Q, ldo=64):
        return lib.mk_dropout_add(None, t, rows, cols, x, ldx, b, r, ldr, p, 1, 2, step, out, ldo)

    def bwd(t=BF16, rows=4, cols=64, dy=P, ld=64, p=0.1, step=None, dx=Q, lddx=64, cs=R, ws=R):
        return lib.mk_dropout_add_bwd(None, t, rows, cols, dy, ld, p, 1, 2, step, dx, lddx, cs, ws)

    for f in (fwd, bwd):
        _refused(lib, 2, "io_type", f(t=S32))
        _refused(lib, 1, "shape", f(rows=-1))
        _refused(lib, 2, "2^32", f(rows=1 << 32))
        _refused(lib, 2, "2^31", f(cols=(1 << 31) + 1))
        for p in (-1e-9, 1.0000001, math.inf, math.nan):
            _refused(lib, 1, "p must", f(p=p))
        _refused(lib, 1, "aligned", f(step=P + 4))
        assert f(cols=0) == 0
    for name in ("x", "out"):
        _refused(lib, 1, "null", fwd(**{name: None}))
    for name in ("x", "out", "b", "r"):
        _refused(lib, 1, "aligned", fwd(**{name: P + 1}))
    _refused(lib, 1, "overlap", fwd(ldo=63))
    _refused(lib, 1, "pitch", fwd(ldx=-64))
    _refused(lib, 1, "another pitch", fwd(out=P, ldx=72))
    _refused(lib, 1, "another pitch", fwd(out=P, x=R, r=P, ldr=0))
    assert fwd(rows=0, x=None) == 0
    for name in ("dy", "dx", "ws"):
        _refused(lib, 1, "null", bwd(**{name: None}))
    for name, off in (("dy", 1), ("dx", 1), ("cs", 2), ("ws", 2)):
        _refused(lib, 1, "aligned", bwd(**{name: P + off}))
    _refused(lib, 1, "overlap", bwd(lddx=63))
    _refused(lib, 1, "another pitch", bwd(dx=P, lddx=72))
    assert bwd(rows=0, cs=None) == 0


def test_philox_known_answers():
    """The generator's published answers for all zeros, all ones and the digits of pi."""
    f = 0xFFFFFFFF
    for ctr, key, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                           ((f, f, f, f), (f, f), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                           ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                            (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v) for v in philox(np.array(ctr, np.uint64), key)) == want


def test_wrappers_take_device_tensors():
    import torch

    from mi355x_pjrt import kernels as K

    x, w, labels, z = torch.zeros(4, 64), torch.zeros(9, 64), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    for f in (lambda: K.linear_xent(x, w, labels), lambda: K.linear_xent_bwd(x, w, labels, z),
              lambda: K.dropout_add(x, 0.1, 1), lambda: K.dropout_add_bwd(x, 0.1, 1)):
        with pytest.raises(ValueError, match="device"):
            f()


@pytest.mark.skipif(not shutil.which(HIPCC) and not os.path.exists(HIPCC), reason="hipcc not available")
def test_lds_copies_have_no_sgpr_hazard(tmp_path):
    out = tmp_path / "linear_xent.s"
    cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "-I" + KDIR, "--cuda-device-only", "-S",
           os.path.join(KDIR, "linear_xent.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)
    asm = out.read_text()
    assert sum(1 for line in asm.splitlines() if _COPY.match(line.strip())) > 0
    assert hazards(asm) == []
