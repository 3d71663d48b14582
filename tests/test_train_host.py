"""Host side of the training operators over the stand-in driver of tests/fake_driver: which kernels a call
launches and with which shape, and what it refuses before any GPU work."""
import pytest

from test_host_logic import fake, run  # noqa: F401  (fixture and helper)


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
        ("layernorm_bf16_v8", 1, 128), ("layernorm_bf16_f32_v16", 592, 256), ("layernorm_f32_s16", 1480, 96),
        ("layernorm_f16_v8", 63, 128), ("layernorm_f16_s8", 63, 128), ("layernorm_f32_v32", 5, 512), ("layernorm_f32_loop", 5, 512),
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
