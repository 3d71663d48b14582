"""Host side of the training operators over the stand-in driver of tests/fake_driver: which kernels a call
launches and with which shape, and what it refuses before any GPU work."""
import os
import subprocess

import pytest

from conftest import ROOT
from test_host_logic import CUDA_INC, FAKE_SRC, fake, run  # noqa: F401  (fixture and helper)


def test_layernorm_forms_and_shapes(fake, tmp_path):  # noqa: F811
    res, L, _ = run(fake, tmp_path, """
d = sm.Device(0); p = 1 << 20
for rows, cols, dt, wdt, ld, x in ((1, 1024, sm.BF16, sm.BF16, 1024, p), (16384, 4096, sm.BF16, sm.F32, 4096, p), (4099, 1031, sm.F32, sm.F32, 1031, p),
                                   (1000, 64, sm.F16, sm.F16, 64, p), (1000, 64, sm.F16, sm.F16, 64, p + 2), (5, 16384, sm.F32, sm.F32, 16388, p),
                                   (5, 16384, sm.F32, sm.F32, 16385, p), (3, 1, sm.F32, sm.F32, 1, p), (0, 64, sm.F32, sm.F32, 64, p)):
    d.layernorm(2 * p, x, p, p, rows, cols, dtype=dt, wdtype=wdt, ldx=ld)
d.sync(); d.close()
""")
    assert res.returncode == 0, res.stderr
    assert [(l["kernel"], l["grid"][0], l["block"][0]) for l in L] == [
        ("layernorm_bf16_v8", 1, 128), ("layernorm_bf16_f32_v32", 592, 128), ("layernorm_f32_s16", 888, 96),
        ("layernorm_f16_v32", 16, 128), ("layernorm_f16_s8", 63, 128), ("layernorm_f32_vx", 5, 512), ("layernorm_f32_sx", 5, 512),
        ("layernorm_f32_s8", 1, 128)]
    assert all(l["overlap"] == 1 for l in L)


def test_layernorm_backward_launches(fake, tmp_path):  # noqa: F811
    res, L, _ = run(fake, tmp_path, """
d = sm.Device(0); p = 1 << 20
def bwd(rows, cols, dt, wdt, dx=2 * p, dw=3 * p, db=4 * p):
    n = d.layernorm_backward_workspace(rows, cols, dt, wdt)
    d.layernorm_backward(dx, dw, db, 5 * p, 6 * p, 7 * p, 8 * p, 9 * p, rows, cols, 10 * p, n, dtype=dt, wdtype=wdt)
bwd(16384, 4096, sm.BF16, sm.F32)
bwd(64, 1024, sm.F16, sm.F16, dw=0, db=0)
bwd(100, 20000, sm.F32, sm.F32)
bwd(100, 20000, sm.F32, sm.F32, dx=0)
bwd(0, 20000, sm.F32, sm.F32)
bwd(50, 100, sm.F32, sm.F32, dx=0, dw=0, db=0)
d.sync(); d.close()
""")
    assert res.returncode == 0, res.stderr
    assert [(l["kernel"], l["grid"][:2]) for l in L] == [
        ("layernorm_bwd_bf16_f32_v16", (296, 1)), ("layernorm_param_grad_f32", (128, 2)), ("layernorm_bwd_f16_v8", (64, 1)),
        ("layernorm_bwd_f32_loop", (100, 1)), ("layernorm_bwd_columns_f32", (79, 64)), ("layernorm_param_grad_f32", (625, 2)),
        ("layernorm_bwd_columns_f32", (79, 64)), ("layernorm_param_grad_f32", (625, 2)), ("layernorm_param_grad_f32", (625, 2))]


@pytest.mark.parametrize("call", [
    "d.layernorm(p, 0, p, p, 4, 8)", "d.layernorm(0, p, p, p, 4, 8)", "d.layernorm(p, p + 2, p, p, 4, 8)", "d.layernorm(p, 2 * p, p + 1, p, 4, 8)",
    "d.layernorm(p, 2 * p, p, p, -1, 8)", "d.layernorm(p, 2 * p, p, p, 4, 0)", "d.layernorm(p, 2 * p, p, p, 4, 8, ldx=7)",
    "d.layernorm(p, 2 * p, p, p, 4, 8, ldy=7)", "d.layernorm(p, p, p, p, 4, 8, ldy=9)", "d.layernorm(p, 2 * p, p, p, 4, 8, eps=-1.0)",
    "d.layernorm(p, 2 * p, p, p, 4, 8, eps=float('nan'))", "d.layernorm(p, 2 * p, p, p, 4, 8, dtype=sm.F32, wdtype=sm.BF16)",
    "d.layernorm(p, 2 * p, p, p, 4, 8, dtype=sm.BF16, wdtype=sm.F16)", "d.layernorm(p, 2 * p, p, p, 4, 8, dtype=sm.F64, wdtype=sm.F64)",
    "d.layernorm(p, 2 * p, p, p, 1 << 40, 8, ldx=1 << 40)", "d.layernorm(p, 2 * p, p, p, 4, 8, mean=p + 2)",
    "d.layernorm_backward(p, p, p, 0, p, p, p, p, 4, 8, p, 1 << 20)", "d.layernorm_backward(p, p, p, 2 * p, 3 * p, p, 0, p, 4, 8, p, 1 << 20)",
    "d.layernorm_backward(2 * p, p, p, 2 * p, 3 * p, p, p, p, 4, 8, p, 1 << 20)", "d.layernorm_backward(3 * p, p, p, 2 * p, 3 * p, p, p, p, 4, 8, p, 1 << 20)",
    "d.layernorm_backward(p, p, p, 2 * p, 3 * p, p, p, p, 4, 8, p, 16)", "d.layernorm_backward(p, p, p, 2 * p, 3 * p, p, p, p, 4, 8, 0, 0)",
    "d.layernorm_backward(p, p, p, 2 * p, 3 * p, p, p, p, 4, 8, p + 8, 1 << 20)", "d.layernorm_backward(p, p + 1, p, 2 * p, 3 * p, p, p, p, 4, 8, p, 1 << 20)",
    "d.layernorm_backward(p, p, p, 2 * p, 3 * p, p, p, p, 4, 8, p, 1 << 20, lddy=3)", "d.layernorm_backward(p, p, p, 2 * p, 3 * p, p, p, p, 4, 0, p, 1 << 20)",
    "d.layernorm(p, 2 * p, p, p, 4, (1 << 30) + 1)", "d.layernorm(p, 2 * p, p, p, 4, 8, mean=p, rstd=p)",
    "d.layernorm_backward(4 * p, p, 5 * p, 2 * p, 3 * p, p, p, p, 1, (1 << 30) + 1, p, 1 << 50)", "d.layernorm_backward_workspace(1, (1 << 30) + 1)",
    "d.layernorm_backward(4 * p, 5 * p, 5 * p, 2 * p, 3 * p, p, p, p, 4, 8, p, 1 << 20)",
    "d.layernorm_backward_workspace(4, 0)", "d.layernorm_backward_workspace(-1, 8)", "d.layernorm_backward_workspace(1, 8, sm.I32)",
])
def test_layernorm_refusals(fake, tmp_path, call):  # noqa: F811
    res, L, _ = run(fake, tmp_path, """
d = sm.Device(0); p = 1 << 20
try:
    %s
except sm.Sm100Error as e:
    assert e.code == sm.ERR_ARG, e
else:
    raise SystemExit("not refused")
d.close()
""" % call)
    assert res.returncode == 0, res.stderr
    assert not L


KERNELS = os.path.join(ROOT, "booth_b200", "csrc", "kernels")


@pytest.fixture(scope="module")
def fake3(tmp_path_factory, sm):
    if not os.path.exists(os.path.join(CUDA_INC, "cuda.h")):
        pytest.skip("cuda.h not found")
    out = tmp_path_factory.mktemp("fake_driver_train") / "libcuda_fake_train.so"
    subprocess.run(["gcc", "-std=c99", "-O1", "-shared", "-fPIC", "-I", CUDA_INC, "-I", os.path.dirname(FAKE_SRC), "-I", KERNELS,
                    os.path.join(os.path.dirname(FAKE_SRC), "fake_cuda_train.c"), "-o", str(out)], check=True)
    return str(out)


def products(lines):
    return [dict(zip(ln.split()[1::2], map(float, ln.split()[2::2]))) for ln in lines if ln.startswith("product")]


def test_orthogonalise_launches(fake3, tmp_path):
    res, L, lines = run(fake3, tmp_path, """
d = sm.Device(0); p = 1 << 20
def go(b, r, c, dt, steps):
    n = d.orthogonalise_workspace(b, r, c, dt)
    d.orthogonalise(p, 2 * p, b, r, c, 4 * p, n, dtype=dt, steps=steps)
go(1, 4096, 4096, sm.BF16, 2)
go(3, 1000, 500, sm.F32, 1)
d.sync(); d.close()
""")
    assert res.returncode == 0, res.stderr
    assert [l["kernel"] for l in L] == ["orth_norm", "orth_split"] + ["orth_product_1_256"] * 6 + ["orth_norm", "orth_split", "orth_product_2_128", "orth_product_2_64", "orth_product_2_128"]
    assert all(l["overlap"] == 1 for l in L)
    assert all(l["shmem"] == 230400 and l["block"] == (384, 1, 1) for l in L if l["kernel"].startswith("orth_product"))
    P = products(lines)
    assert [(p["mode"], p["rows"], p["cols"], p["K"], p["batch"], p["tall"]) for p in P] == [
        (0, 4096, 4096, 4096, 1, 0), (1, 4096, 4096, 4096, 1, 0), (2, 4096, 4096, 4096, 1, 0),
        (0, 4096, 4096, 4096, 1, 0), (1, 4096, 4096, 4096, 1, 0), (3, 4096, 4096, 4096, 1, 0),
        (0, 500, 500, 1000, 3, 1), (1, 500, 500, 500, 3, 1), (3, 500, 1000, 500, 3, 1)]
    # X is kept times 2^14, S = A + b / 2c times 2^12, Q = c S S + (a - b^2 / 4c) times 2^11 with the default coefficients
    a, b, c = 3.4445, -4.7750, 2.0315
    want = [(2.0 ** -16, b / (2 * c) * 2 ** 12), (c * 2.0 ** -13, (a - b * b / (4 * c)) * 2 ** 11), (2.0 ** -11, 0), (2.0 ** -25, 0)]
    for p, k in zip(P, (0, 1, 2, 0, 1, 3, 0, 1, 3)):
        assert (p["alpha"], p["diag"]) == pytest.approx(want[k], rel=1e-6)
    maps = [ln for ln in lines if ln.startswith("tensormap3")]
    # one plane: hi and lo of both copies of X, S and Q; rows a multiple of 64 apart
    assert maps[:6] == ["tensormap3 dims 4096 4096 1 strides 8192 33554432 box 64 64 1"] * 6
    assert maps[6:] == ["tensormap3 dims 1000 500 3 strides 2048 1024000 box 64 64 1"] * 4 + ["tensormap3 dims 500 500 3 strides 1024 512000 box 64 64 1"] * 4


def test_cubic_has_no_polynomial_product(fake3, tmp_path):
    res, L, lines = run(fake3, tmp_path, """
d = sm.Device(0); p = 1 << 20
n = d.orthogonalise_workspace(1, 64, 64)
d.orthogonalise(p, 2 * p, 1, 64, 64, 4 * p, n, steps=2, abc=(1.5, -0.5, 0.0))
d.sync(); d.close()
""")
    assert res.returncode == 0, res.stderr
    P = products(lines)
    assert [p["mode"] for p in P] == [0, 2, 0, 3]
    assert [P[0]["alpha"], P[0]["diag"], P[1]["alpha"]] == pytest.approx([-0.5 * 2.0 ** -14, 1.5 * 2 ** 14, 2.0 ** -14])


def test_muon_parameters(fake3, tmp_path):
    res, L, lines = run(fake3, tmp_path, """
d = sm.Device(0); p = 1 << 20
n = d.orthogonalise_workspace(1, 300, 200, sm.F32)
d.muon_step(p, 2 * p, 3 * p, 1, 300, 200, 4 * p, n, lr=0.1, scale=4.0, weight_decay=0.5, gdtype=sm.BF16, steps=1)
d.sync(); d.close()
""")
    assert res.returncode == 0, res.stderr
    last = products(lines)[-1]
    assert last["mode"] == 3 and last["keep"] == pytest.approx(0.95) and last["alpha"] == pytest.approx(-0.4 * 2.0 ** -25)


def test_a_wait_that_ran_out_is_reported_once(fake3, tmp_path):
    res, _, _ = run(fake3, tmp_path, """
import os
d = sm.Device(0); p = 1 << 20
n = d.orthogonalise_workspace(1, 64, 64)
os.environ["FAKE_CUDA_ORTH_STATUS"] = "2"
import ctypes; ctypes.CDLL(None).setenv(b"FAKE_CUDA_ORTH_STATUS", b"2", 1)
d.orthogonalise(p, 2 * p, 1, 64, 64, 4 * p, n)
try:
    d.sync()
except sm.Sm100Error as e:
    assert e.code == sm.ERR_CUDA and "orth_product gave up" in str(e) and "code 2" in str(e), e
else:
    raise SystemExit("not reported")
d.sync()
ctypes.CDLL(None).unsetenv(b"FAKE_CUDA_ORTH_STATUS")
d.orthogonalise(p, 2 * p, 1, 64, 64, 4 * p, n)
d.sync(); d.close()
""")
    assert res.returncode == 0, res.stderr


@pytest.mark.parametrize("call", [
    "d.orthogonalise(0, p, 1, 8, 8, p, big)", "d.orthogonalise(p, 0, 1, 8, 8, p, big)", "d.orthogonalise(p, 2 * p, 0, 8, 8, p, big)",
    "d.orthogonalise(p, 2 * p, 1, 0, 8, p, big)", "d.orthogonalise(p, 2 * p, 1, 8, 0, p, big)", "d.orthogonalise(p, 2 * p, 1, (1 << 20) + 1, 8, p, big)",
    "d.orthogonalise(p, 2 * p, 65536, 8, 8, p, big)", "d.orthogonalise(p, 2 * p, 1, 8, 8, 0, big)", "d.orthogonalise(p, 2 * p, 1, 8, 8, p + 64, big)",
    "d.orthogonalise(p, 2 * p, 1, 8, 8, p, d.orthogonalise_workspace(1, 8, 8) - 1)", "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, steps=0)",
    "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, steps=65)", "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, eps=0.0)",
    "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, abc=(1.0, float('nan'), 0.0))", "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, abc=(1.0, 1.0, 0.1))", "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, abc=(float('inf'), 1.0, 0.0))",
    "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, ld_in=7)", "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, ld_out=7)",
    "d.orthogonalise(p, 2 * p, 2, 8, 8, p, big, stride_in=7)", "d.orthogonalise(p, 2 * p, 2, 8, 8, p, big, stride_out=-64)",
    "d.orthogonalise(p, p, 1, 8, 8, p, big, ld_out=9)", "d.orthogonalise(p, p, 2, 8, 8, p, big, stride_out=65)", "d.orthogonalise(p + 2, 2 * p, 1, 8, 8, p, big)",
    "d.orthogonalise(p, 2 * p, 1, 8, 8, p, big, dtype=sm.F64)", "d.orthogonalise(p, 2 * p, 2, 8, 8, p, big, stride_in=1 << 60)",
    "d.orthogonalise_workspace(0, 8, 8)", "d.orthogonalise_workspace(1, 8, 8, sm.I32)",
    "d.muon_step(0, p, 2 * p, 1, 8, 8, p, big, lr=0.1)", "d.muon_step(p, p, 2 * p, 1, 8, 8, p, big, lr=0.1)", "d.muon_step(p, 2 * p, p, 1, 8, 8, p, big, lr=0.1)",
    "d.muon_step(3 * p, 2 * p, 2 * p, 1, 8, 8, p, big, lr=0.1)", "d.muon_step(p, 2 * p, 3 * p, 1, 8, 8, p, big, lr=float('nan'))",
    "d.muon_step(p, 2 * p, 3 * p, 1, 8, 8, p, big, lr=0.1, momentum=1.5)", "d.muon_step(p, 2 * p, 3 * p, 1, 8, 8, p, big, lr=0.1, weight_decay=float('inf'))",
    "d.muon_step(p, 2 * p, 3 * p, 1, 8, 8, p, 100, lr=0.1)", "d.muon_step(p, 2 * p, 3 * p, 1, 8, 8, p, big, lr=0.1, mdtype=sm.F64)",
    "d.muon_step(p, 2 * p, 3 * p, 1, 8, 8, p, big, lr=0.1, ld_m=4)", "d.muon_step(p, 2 * p, 3 * p, 1, 8, 8, p, big, lr=0.1, steps=0)",
])
def test_orthogonalise_and_muon_refusals(fake3, tmp_path, call):
    res, L, _ = run(fake3, tmp_path, """
d = sm.Device(0); p = 1 << 20; big = 1 << 30
try:
    %s
except sm.Sm100Error as e:
    assert e.code == sm.ERR_ARG, e
else:
    raise SystemExit("not refused")
d.close()
""" % call)
    assert res.returncode == 0, res.stderr
    assert not L


def test_muon_launches_nothing_when_a_map_fails(fake, tmp_path):  # noqa: F811
    """The plain stand-in driver refuses maps of three dimensions: the momentum must not have changed by then."""
    res, L, _ = run(fake, tmp_path, """
d = sm.Device(0); p = 1 << 20
n = d.orthogonalise_workspace(1, 64, 64, sm.F32)
try:
    d.muon_step(p, 2 * p, 3 * p, 1, 64, 64, 4 * p, n, lr=0.1)
except sm.Sm100Error as e:
    assert e.code != sm.ERR_ARG, e
else:
    raise SystemExit("not refused")
d.close()
""")
    assert res.returncode == 0, res.stderr
    assert not [l for l in L if l["kernel"].startswith("orth")]


def test_the_silent_producer_is_the_first_product_only(fake3, tmp_path):
    res, _, lines = run(fake3, tmp_path, """
d = sm.Device(0); p = 1 << 20
n = d.orthogonalise_workspace(1, 64, 64)
d.orthogonalise(p, 2 * p, 1, 64, 64, 4 * p, n, steps=2 | sm.NS_TEST_SILENT_PRODUCER)
d.orthogonalise(p, 2 * p, 1, 64, 64, 4 * p, n, steps=1)
for steps in (sm.NS_TEST_SILENT_PRODUCER, 65 | sm.NS_TEST_SILENT_PRODUCER):
    try:
        d.orthogonalise(p, 2 * p, 1, 64, 64, 4 * p, n, steps=steps)
    except sm.Sm100Error as e:
        assert e.code == sm.ERR_ARG, e
    else:
        raise SystemExit("not refused")
d.sync(); d.close()
""")
    assert res.returncode == 0, res.stderr
    assert [p["silent"] for p in products(lines)] == [1, 0, 0, 0, 0, 0, 0, 0, 0]


# (batch, rows, cols, ld, stride) of matrices that share elements, and of such that do not
SHARED = [(2, 8, 8, 8, 8), (2, 8, 8, 16, 16), (3, 4, 8, 8, 24), (2, 8, 8, 20, 14), (4, 5, 6, 18, 10), (65535, 8, 8, 1 << 19, 9), (2, 8, 8, 9, 65)]
APART = [(2, 8, 8, 8, 64), (2, 8, 8, 16, 8), (3, 8, 8, 24, 8), (4, 2, 4, 12, 8 * 3 + 4), (3, 2, 4, 12, 8), (2, 1, 8, 8, 8), (2, 8, 1, 2, 1), (2, 8, 8, 9, 71), (2, 8, 8, 20, 10)]


def elements_apart(batch, rows, cols, ld, stride):
    starts = sorted(k * stride + r * ld for k in range(batch) for r in range(rows))
    return all(b - a >= cols for a, b in zip(starts, starts[1:]))


def test_layouts_are_what_they_are_listed_as():
    assert not any(elements_apart(*s) for s in SHARED) and all(elements_apart(*s) for s in APART)


@pytest.mark.parametrize("shape", SHARED + APART)
def test_matrices_that_are_written_lie_apart(fake3, tmp_path, shape):
    """What two matrices share would be written by two blocks in no order: refused for out, w and m, allowed for what is only read."""
    res, L, _ = run(fake3, tmp_path, """
d = sm.Device(0); p = 1 << 20; big = 1 << 34
n, r, c, ld, stride = %s
wide = dict(ld_in=c, stride_in=r * c)
calls = [lambda: d.orthogonalise(p, 2 * p, n, r, c, 4 * p, big, ld_out=ld, stride_out=stride, steps=1, **wide),
         lambda: d.orthogonalise(p, p, n, r, c, 4 * p, big, ld_out=ld, stride_out=stride, ld_in=ld, stride_in=stride, steps=1),
         lambda: d.muon_step(p, 2 * p, 3 * p, n, r, c, 4 * p, big, lr=0.1, ld_w=ld, stride_w=stride, steps=1),
         lambda: d.muon_step(p, 2 * p, 3 * p, n, r, c, 4 * p, big, lr=0.1, ld_m=ld, stride_m=stride, steps=1)]
for call in calls:
    try:
        call()
        assert %s, "not refused"
    except sm.Sm100Error as e:
        assert not %s and e.code == sm.ERR_ARG, e
d.orthogonalise(p, 2 * p, n, r, c, 4 * p, big, ld_in=ld, stride_in=stride, steps=1)
d.muon_step(p, 2 * p, 3 * p, n, r, c, 4 * p, big, lr=0.1, ld_g=ld, stride_g=stride, steps=1)
d.sync(); d.close()
""" % (shape, shape in APART, shape in APART))
    assert res.returncode == 0, res.stderr


def test_a_replay_whose_wait_ran_out_is_reported_and_others_cost_no_copy(fake3, tmp_path):
    """A captured call runs behind the library's back. Its word in the host's memory says when the status is worth
    reading; as long as it does not, waits read nothing from the GPU."""
    res, _, lines = run(fake3, tmp_path, """
import ctypes
libc = ctypes.CDLL(None)
d = sm.Device(0); p = 1 << 20
n = d.orthogonalise_workspace(1, 64, 64)
d.orthogonalise(p, 2 * p, 1, 64, 64, 4 * p, n)
d.sync()                        # reads the status once: a call was enqueued
for _ in range(5):
    d.sync()
libc.setenv(b"FAKE_CUDA_ORTH_REPLAY", b"3", 1)
try:
    d.sync()
except sm.Sm100Error as e:
    assert e.code == sm.ERR_CUDA and "code 3" in str(e), e
else:
    raise SystemExit("not reported")
for _ in range(5):
    d.sync()
d.close()
""")
    assert res.returncode == 0, res.stderr
    assert lines.count("d2h_now") == 2, lines
