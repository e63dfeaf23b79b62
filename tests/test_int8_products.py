"""The kernel that each of the eight-bit products in int8_products.py runs on, that
every kernel built is among them, and which results go past the caches: the host code
of gemm_int8.hip linked against a HIP runtime that only records its launches
(tests/int8_routes_check.cc).  Nothing here runs on a GPU."""

import os
import shutil
import subprocess

import pytest

from int8_products import BF16, DEEP, F16, F32, FEW, STREAMED, TILED, lines, pitch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM", "/opt/rocm")
HIPCC = os.path.join(ROCM, "bin", "hipcc")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) or not shutil.which("g++"),
                                reason="hipcc or g++ not available")


@pytest.fixture(scope="module")
def routes(tmp_path_factory):
    """f(products): what each (c_type, M, K, N, lda, ldb, ldc) is launched as, and all kernels there are."""
    tmp = tmp_path_factory.mktemp("routes")
    obj, exe = str(tmp / "check.o"), str(tmp / "check")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-fPIC",
                    "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "mccl-jax_amd", "src", "kernels"),
                    "-x", "hip", "-c", os.path.join(ROOT, "tests", "int8_routes_check.cc"), "-o", obj],
                   check=True, timeout=300)
    # the device code's sections are left out: their registration is recorded, not read
    subprocess.run(["g++", obj, "-o", exe, "-Wl,--unresolved-symbols=ignore-all"], check=True, timeout=300)

    def ask(products):
        r = subprocess.run([exe], input="\n".join(" ".join(map(str, p)) for p in products), capture_output=True,
                           text=True, timeout=60)
        assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
        out = r.stdout.splitlines()
        return out[:len(products)], {line[len("compiled "):] for line in out[len(products):]}

    return ask


def _grid(k):
    return (k + 15) // 16 * 16


def test_each_product_runs_on_its_kernel_and_each_kernel_has_one(routes):
    asked, want = [], []
    for name, m, n, ks, on_grid in TILED:
        for k in ks:
            for t in (BF16, F16, F32):
                ld = pitch(k, on_grid)
                asked.append((t, m, k, n, ld, ld, n + 5))
                want.append(f"{name}, {t}> cached")
    for name, m, n, ks, on_grid in FEW:
        for k in ks:
            ld = pitch(k, on_grid)
            asked.append((BF16, m, k, n, ld, ld, n + 5))
            want.append(name)
    for name, m, n in DEEP:
        asked.append((F32, m, 131071, n, 131072, 131072, n))
        want.append(f"{name}, {F32}> cached")
    for name, t, m, n, k in STREAMED:
        ld = _grid(k) if "true" in name else k
        asked.append((t, m, k, n, ld, ld, lines(n)))
        want.append(f"{name}, {t}> streamed")
    got, compiled = routes(asked)
    for p, g, w in zip(asked, got, want):
        assert g == w, p
    assert {g.split(">")[0] for g in got} == {c.split(">")[0] for c in compiled}


def test_what_goes_past_the_caches(routes):
    """C of 192 MiB and more with whole rows on the 128-byte lines; not a few columns of a wide buffer."""
    mib = 1 << 20
    got, _ = routes([(BF16, 8192, 4096, 16384, 4096, 4096, 16384), (BF16, 8192, 4096, 16384, 4096, 4096, 16385),
                     (BF16, 8192, 4096, 64, 4096, 4096, 16384), (F32, 65536, 256, 512, 256, 256, 65536),
                     (F32, 65536, 256, 768, 256, 256, 65536), (BF16, 6144, 512, 16384, 512, 512, 16384),
                     (BF16, 6143, 512, 16384, 512, 512, 32768)])
    assert 6144 * 16384 * 2 == 192 * mib and 65536 * 768 * 4 == 192 * mib
    assert [g.split("> ")[1] for g in got] == ["streamed", "cached", "cached", "cached", "streamed", "streamed", "cached"]
