"""Which kernels the losses without logits and dropout run, by the host code as it
stands (tests/xent_routes_check.cc): the sizes that test_gpu_xent_tiles.py compares
with the definitions reach every one of them.  Nothing here runs on a GPU."""

import os
import shutil
import subprocess

import pytest

from xent_cases import DROP_GRADS, DROPS, FEW, PIECES, TILES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM", "/opt/rocm")
HIPCC = os.path.join(ROCM, "bin", "hipcc")
TYPES = {"bf16": 13, "f16": 10, "f32": 11}

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) or not shutil.which("g++"), reason="hipcc or g++ not available")


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("xent")
    inc, kdir = os.path.join(ROOT, "include"), os.path.join(ROOT, "mccl-jax_amd", "src", "kernels")
    objs, exe = [], str(tmp / "check")
    for src in (os.path.join(ROOT, "tests", "xent_routes_check.cc"), os.path.join(kdir, "dropout.hip")):
        objs.append(str(tmp / (os.path.basename(src) + ".o")))
        subprocess.run([HIPCC, "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-fPIC", "-I" + inc, "-I" + kdir,
                        "-x", "hip", "-c", src, "-o", objs[-1]], check=True, timeout=300)
    # the device code's sections are left out: their registration is recorded, not read
    subprocess.run(["g++", *objs, "-o", exe, "-Wl,--unresolved-symbols=ignore-all"], check=True, timeout=300)

    def ask(calls):
        r = subprocess.run([exe], input="\n".join(" ".join(map(str, c)) for c in calls), capture_output=True, text=True,
                           timeout=60)
        assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
        out = r.stdout.splitlines()
        return [line.split() for line in out[:len(calls)]], {line[len("compiled "):] for line in out[len(calls):]}

    return ask


def _calls(cases):
    out = []
    for rows, width, vocab, t, dw, ignore in cases:
        for kind in ("loss", "grad"):
            out.append((kind, TYPES[t], TYPES[dw], rows, width, vocab, width, width, 0, int(ignore)))
    return out


def test_every_kernel_is_compared(ask):
    drops = [("drop", TYPES[t], r, c, 0) for r, c, t in DROPS]
    drops += [("dropgrad", TYPES[t], r, c, s) for r, c, t in DROP_GRADS for s in (0, 1)]
    launches, compiled = ask(_calls(TILES + PIECES + FEW) + drops)
    reached = {k.split(":")[0] for line in launches for k in line}
    # no rows: a gradient of zeros (test_gpu_linear_xent.py has it of every type)
    assert compiled - reached == {"zero<unsignedshort>", "zero<unsignedint>"}


@pytest.mark.parametrize("t", ["Bf16", "F16"])
def test_large_tiles_follow_each_other(ask, t):
    """Tiles, workgroups and k tiles of the kernels that go from tile to tile."""
    launches, _ = ask(_calls(TILES))
    for kernel in ("loss", "grad"):
        name = f"{kernel}<{t},Shape<256,256>>"
        seen = [tuple(map(int, k.split(":")[1].split("/"))) for line in launches for k in line if k.startswith(name)]
        assert any(tiles >= 3 * groups and deep > 4 for tiles, groups, deep in seen), (name, seen)
        assert any(tiles % groups for tiles, groups, _ in seen), (name, seen)


def test_pieces(ask):
    """Weights off the 16-byte boundaries are copied in more than one piece, forward and backward."""
    calls = _calls(PIECES)
    for call, line in zip(calls, ask(calls)[0]):
        copies = sum(k.startswith("pack") for k in line)
        assert copies >= (2 if call[4] == 1025 else 0), (call, line)
        assert any(k.startswith(("loss<", "grad<")) for k in line), (call, line)


def test_grids_hold_at_the_largest_sizes(ask):
    big = [("loss", 13, 13, 1 << 20, 768, 131072, 768, 768, 0, 0), ("grad", 13, 11, 1 << 20, 768, 131072, 768, 768, 0, 1),
           ("grad", 10, 10, 1, 1 << 20, 1000, 1 << 20, 1 << 20, 0, 0), ("loss", 11, 11, 32, 64, 1 << 28, 64, 64, 0, 0),
           ("grad", 11, 11, 1 << 22, 64, 2, 64, 64, 1, 1), ("drop", 13, 1 << 22, 4096, 0),
           ("dropgrad", 11, 1 << 22, 4096, 1), ("drop", 11, (1 << 32) - 1, 1, 0)]
    for call, line in zip(big, ask(big)[0]):
        assert line and not any("too-large" in k for k in line), (call, line)
