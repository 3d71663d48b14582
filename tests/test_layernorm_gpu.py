"""Layer normalisation and its gradient against a plain statement in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32) and h = finfo(type).eps / 2 (half a step of the stored type):
a stored value is off by h |value| for its own rounding (f16 also by 2^-25, half its smallest step), and by what
fp32 arithmetic leaves. A group adds at most 32 values a thread in sequence and then 10 levels of a tree, and the
loop form cols / 512 a thread; each result is a handful of further roundings. SUMS(n) bounds the roundings of one
such sum, and every formula below multiplies it with the sum of the magnitudes of the terms it is made of."""
import pytest
import torch

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]

# one value, widths below a vector, a warp's share, the borders of the forms (256, 1024, 4096, 8192, 16384) and beyond, odd ones
SHAPES = [(1, 1), (3, 2), (130, 5), (7, 8), (1, 16), (9, 31), (1000, 64), (65, 250), (33, 256), (33, 257), (4, 264), (700, 1000), (301, 1024),
          (5, 1025), (900, 1032), (2, 4096), (640, 4096), (3, 4097), (400, 5000), (3, 8191), (3, 8192), (2, 8193), (4, 10000), (3, 16384), (2, 16385), (1, 40000)]


def SUMS(cols):
    return 48 + cols / 512


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -126


def code(sm, t):
    return {torch.float32: sm.F32, torch.bfloat16: sm.BF16, torch.float16: sm.F16}[t]


def strided(t, pad, offset=0):
    """t in a wider matrix whose other columns hold a marker, `offset` elements into its storage."""
    r, c = t.shape
    flat = torch.full((r * (c + pad) + offset,), 7.25, dtype=t.dtype, device=t.device)
    v = flat[offset:].view(r, c + pad)
    v[:, :c] = t
    return flat, v[:, :c]


def make(rows, cols, t, wt, seed=0, mean=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g, device="cuda") + mean * torch.randn(rows, 1, generator=g, device="cuda")).to(t)
    w = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(wt)
    b = (0.3 * torch.randn(cols, generator=g, device="cuda")).to(wt)
    dy = torch.randn(rows, cols, generator=g, device="cuda").to(t)
    return x, w, b, dy


def forward64(x, w, b, eps):
    x = x.double()
    mean = x.mean(1)
    var = (x - mean[:, None]).square().mean(1)
    rstd = 1 / (var + eps).sqrt()
    y = (x - mean[:, None]) * rstd[:, None]
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd


def check_forward(x, w, b, eps, y, mean, rstd):
    ry, rm, rr = forward64(x, w, b, eps)
    k = SUMS(x.shape[1]) * U
    xd = x.double()
    mag = (xd.abs() + rm.abs()[:, None]) * rr[:, None] * (1 if w is None else w.double().abs()) + (0 if b is None else b.double().abs())
    tol = half_step(x.dtype) * ry.abs() + k * mag + tiny(x.dtype)
    assert bool(((y.double() - ry).abs() <= tol).all()), ((y.double() - ry).abs() - tol).max()
    if mean is not None:
        assert bool(((mean.double() - rm).abs() <= k * xd.abs().mean(1) + 2.0 ** -126).all())
        # d rstd / rstd = -d var rstd^2 / 2: the variance carries k of itself and the square of the mean's error
        assert bool(((rstd.double() - rr).abs() <= rr * (k + 2 * U + (U * rm.abs() * rr) ** 2)).all())


def run_forward(dev, sm, x, w, b, eps=1e-5, y=None, stats=True):
    y = torch.empty(x.shape, dtype=x.dtype, device="cuda") if y is None else y
    mean = torch.empty(x.shape[0], device="cuda") if stats else None
    rstd = torch.empty(x.shape[0], device="cuda") if stats else None
    torch.cuda.synchronize()
    dev.layernorm(y.data_ptr(), x.data_ptr(), 0 if w is None else w.data_ptr(), 0 if b is None else b.data_ptr(), x.shape[0], x.shape[1], eps=eps,
                  dtype=code(sm, x.dtype), wdtype=code(sm, x.dtype if w is None else w.dtype), mean=mean.data_ptr() if stats else 0,
                  rstd=rstd.data_ptr() if stats else 0, ldx=x.stride(0), ldy=y.stride(0))
    dev.sync()
    return y, mean, rstd


def run_backward(dev, sm, dy, x, w, mean, rstd, dx=None, want="dx dw db"):
    r, c = x.shape
    wt = x.dtype if w is None else w.dtype
    dx = torch.empty(r, c, dtype=x.dtype, device="cuda") if dx is None else dx
    dw, db = (torch.full((c,), 3.0, dtype=wt, device="cuda") for _ in range(2))
    n = dev.layernorm_backward_workspace(r, c, code(sm, x.dtype), code(sm, wt))
    ws = torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    dev.layernorm_backward(dx.data_ptr() if "dx" in want else 0, dw.data_ptr() if "dw" in want else 0, db.data_ptr() if "db" in want else 0,
                           dy.data_ptr(), x.data_ptr(), 0 if w is None else w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), r, c, ws.data_ptr(), n,
                           dtype=code(sm, x.dtype), wdtype=code(sm, wt), lddx=dx.stride(0), lddy=dy.stride(0), ldx=x.stride(0))
    dev.sync()
    return dx, dw, db


def backward64(dy, x, w, mean, rstd):
    dy, x, m, r = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    xh = (x - m) * r
    wd = dy if w is None else dy * w.double()
    p, q = wd.mean(1, keepdim=True), (wd * xh).mean(1, keepdim=True)
    return r * (wd - p - xh * q), (dy * xh).sum(0), dy.sum(0)


def check_backward(dy, x, w, mean, rstd, dx, dw, db):
    rdx, rdw, rdb = backward64(dy, x, w, mean, rstd)
    k = SUMS(x.shape[1]) * U
    d, xa, r = dy.double().abs(), (x.double().abs() + mean.double().abs()[:, None]) * rstd.double()[:, None], rstd.double()[:, None]
    wd = d if w is None else d * w.double().abs()
    if dx is not None:
        tol = half_step(x.dtype) * rdx.abs() + k * r * (wd + wd.mean(1, keepdim=True) + xa * (wd * xa).mean(1, keepdim=True)) + tiny(x.dtype)
        assert bool(((dx.double() - rdx).abs() <= tol).all()), ((dx.double() - rdx).abs() - tol).max()
    # a column is added over at most all the rows in sequence, then over the blocks in double, then rounded once to fp32 on the way
    kr = (min(x.shape[0], 600) + 8) * U
    for got, want, mag in ((dw, rdw, (d * xa).sum(0)), (db, rdb, d.sum(0))):
        if got is not None:
            tol = half_step(got.dtype) * want.abs() + kr * mag + tiny(got.dtype)
            assert bool(((got.double() - want).abs() <= tol).all()), ((got.double() - want).abs() - tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("t,wt", PAIRS)
def test_forward_and_backward(dev, sm, rows, cols, t, wt):
    x, w, b, dy = make(rows, cols, TYPES[t], TYPES[wt], seed=rows + cols)
    y, mean, rstd = run_forward(dev, sm, x, w, b)
    check_forward(x, w, b, 1e-5, y, mean, rstd)
    check_backward(dy, x, w, mean, rstd, *run_backward(dev, sm, dy, x, w, mean, rstd))


@pytest.mark.gpu
@pytest.mark.parametrize("t,wt", PAIRS)
@pytest.mark.parametrize("rows,cols,pad,offset", [(37, 96, 8, 0), (37, 96, 8, 8), (37, 96, 3, 0), (9, 1024, 8, 1), (50, 1031, 5, 3), (5, 4104, 24, 16), (3, 16384, 1, 0)])
def test_pitches_offsets_and_what_lies_between_rows(dev, sm, rows, cols, pad, offset, t, wt):
    x, w, b, dy = make(rows, cols, TYPES[t], TYPES[wt], seed=5)
    _, xs = strided(x, pad, offset)
    flat, ys = strided(torch.zeros_like(x), pad, offset)
    y, mean, rstd = run_forward(dev, sm, xs, w, b, y=ys)
    check_forward(x, w, b, 1e-5, y, mean, rstd)
    assert bool((flat[:offset] == 7.25).all()) and bool((flat[offset:].view(rows, -1)[:, cols:] == 7.25).all())
    _, ds = strided(dy, pad, offset)
    flat, out = strided(torch.zeros_like(x), pad, offset)
    check_backward(dy, x, w, mean, rstd, *run_backward(dev, sm, ds, xs, w, mean, rstd, dx=out))
    assert bool((flat[:offset] == 7.25).all()) and bool((flat[offset:].view(rows, -1)[:, cols:] == 7.25).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [40, 1024, 5000, 5001, 17000])
def test_rows_far_from_zero_and_rows_of_one_value(dev, sm, cols):
    x, w, b, _ = make(11, cols, torch.float32, torch.float32, seed=2)
    x += 1000.0
    x[3] = -2.5
    y, mean, rstd = run_forward(dev, sm, x, w, b)
    check_forward(x, w, b, 1e-5, y, mean, rstd)
    assert bool((y[3] == b).all()) and mean[3].item() == -2.5


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [24, 1000, 1024, 6001, 20000])
def test_absent_parameters_in_place_and_non_finite_rows(dev, sm, cols):
    x, w, b, dy = make(6, cols, torch.bfloat16, torch.bfloat16, seed=3)
    x[2, cols // 2] = float("inf")
    x[4, 0] = float("nan")
    keep = [0, 1, 3, 5]
    for pw, pb in ((None, None), (w, None), (None, b)):
        y, mean, rstd = run_forward(dev, sm, x, pw, pb)
        check_forward(x[keep], pw, pb, 1e-5, y[keep], mean[keep], rstd[keep])
        assert bool(y[2].isnan().all()) and bool(y[4].isnan().all()) and bool(mean[4].isnan()) and bool(rstd[2].isnan())
    z = x.clone()
    y, mean, rstd = run_forward(dev, sm, x, w, b)
    run_forward(dev, sm, z, w, b, y=z, stats=False)
    assert torch.equal(z.view(torch.int16)[keep], y.view(torch.int16)[keep])
    sub = (dy[keep].contiguous(), x[keep].contiguous(), mean[keep], rstd[keep])
    check_backward(sub[0], sub[1], None, sub[2], sub[3], *run_backward(dev, sm, sub[0], sub[1], None, sub[2], sub[3]))
    for want in ("dx", "dw", "db", "dw db", "dx db"):
        dx, dw, db = run_backward(dev, sm, sub[0], sub[1], w, sub[2], sub[3], want=want)
        check_backward(sub[0], sub[1], w, sub[2], sub[3], dx if "dx" in want else None, dw if "dw" in want else None, db if "db" in want else None)
        assert "dw" in want or bool((dw == 3).all())
        assert "db" in want or bool((db == 3).all())


@pytest.mark.gpu
def test_no_rows(dev, sm):
    dw, db = torch.ones(70, device="cuda"), torch.ones(70, device="cuda")
    ws = torch.empty(dev.layernorm_backward_workspace(0, 70), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    dev.layernorm(0, 0, 0, 0, 0, 70)
    dev.layernorm_backward(0, dw.data_ptr(), db.data_ptr(), 0, 0, 0, 0, 0, 0, 70, ws.data_ptr(), ws.numel())
    dev.sync()
    assert not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_offsets_past_32_bits(dev, sm, t):
    x, w, b, dy = make(3, 4096, TYPES[t], torch.float32, seed=4)
    ld = (1 << 31) // 2 + 8
    wide = [torch.empty(2 * ld + 4096, dtype=TYPES[t], device="cuda") for _ in range(3)]
    xs, ys, ds = (v.as_strided((3, 4096), (ld, 1)) for v in wide)
    xs.copy_(x)
    y, mean, rstd = run_forward(dev, sm, xs, w, b, y=ys)
    check_forward(x, w, b, 1e-5, y, mean, rstd)
    ds.copy_(dy)
    check_backward(dy, x, w, mean, rstd, *run_backward(dev, sm, ds, xs, w, mean, rstd, dx=ys))


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits_and_can_be_captured(dev, sm):
    x, w, b, dy = make(2000, 1000, torch.bfloat16, torch.float32, seed=6)
    y, mean, rstd = run_forward(dev, sm, x, w, b)
    first = run_backward(dev, sm, dy, x, w, mean, rstd)
    again = run_backward(dev, sm, dy, x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    stream = torch.cuda.ExternalStream(dev.stream)
    outs = [torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w), torch.zeros_like(mean), torch.zeros_like(rstd)]
    n = dev.layernorm_backward_workspace(2000, 1000, sm.BF16, sm.F32)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        dev.layernorm(outs[0].data_ptr(), x.data_ptr(), w.data_ptr(), b.data_ptr(), 2000, 1000, dtype=sm.BF16, wdtype=sm.F32,
                      mean=outs[4].data_ptr(), rstd=outs[5].data_ptr())
        dev.layernorm_backward(outs[1].data_ptr(), outs[2].data_ptr(), outs[3].data_ptr(), dy.data_ptr(), x.data_ptr(), w.data_ptr(),
                               outs[4].data_ptr(), outs[5].data_ptr(), 2000, 1000, ws.data_ptr(), n, dtype=sm.BF16, wdtype=sm.F32)
    for _ in range(2):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], y) and all(torch.equal(p, q) for p, q in zip(outs[1:4], first))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [6, 65])
def test_gradient_agrees_with_differences(dev, sm, cols):
    """Central differences of the 64-bit forward in x, w and b: their own error is O(step^2) ~ 1e-6 here."""
    x, w, b, dy = make(4, cols, torch.float32, torch.float32, seed=8)
    _, mean, rstd = run_forward(dev, sm, x, w, b)
    dx, dw, db = run_backward(dev, sm, dy, x, w, mean, rstd)
    x, w, b, dy = x.double(), w.double(), b.double(), dy.double()
    step = 1e-4

    def loss(x, w, b):
        return (forward64(x, w, b, 1e-5)[0] * dy).sum()

    for p, grad in ((x, dx), (w, dw), (b, db)):
        flat = p.view(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 17)):
            old = flat[i].item()
            flat[i] = old + step
            hi = loss(x, w, b)
            flat[i] = old - step
            lo = loss(x, w, b)
            flat[i] = old
            assert abs(((hi - lo) / (2 * step)).item() - grad.view(-1)[i].item()) < 1e-4 * (1 + grad.abs().max().item())


# every group of threads takes more rows than its ring holds, rows start at every offset from 16 bytes
WALKS = [(60000, 7, 2, 1), (60000, 33, 4, 3), (15000, 257, 2, 5), (7000, 1001, 4, 1), (1500, 4099, 2, 7), (800, 9001, 6, 3), (20000, 40, 8, 8), (3000, 5000, 8, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,pad,offset", WALKS)
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_long_walks_take_nothing_from_neighbours(dev, sm, rows, cols, pad, offset, t):
    """What lies between the rows is NaN, and in the second half so is every seventh row of x: neither may reach another row."""
    x, w, b, dy = make(rows, cols, TYPES[t], torch.float32, seed=rows)

    def within_nan(v):
        flat, view = strided(v, pad, offset)
        hold = v.clone()
        flat.fill_(float("nan"))
        view.copy_(hold)
        return view

    xs, ds = within_nan(x), within_nan(dy)
    y, mean, rstd = run_forward(dev, sm, xs, w, b)
    check_forward(x, w, b, 1e-5, y, mean, rstd)
    check_backward(dy, x, w, mean, rstd, *run_backward(dev, sm, ds, xs, w, mean, rstd))
    bad = torch.arange(3, rows, 7, device="cuda")
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[bad] = False
    xs[bad] = float("nan")
    y, mean, rstd = run_forward(dev, sm, xs, w, b)
    check_forward(x[keep], w, b, 1e-5, y[keep], mean[keep], rstd[keep])
    assert bool(y[bad].isnan().all())
    dx, _, _ = run_backward(dev, sm, ds, xs, w, mean, rstd)
    rdx = run_backward(dev, sm, dy[keep].contiguous(), x[keep].contiguous(), w, mean[keep], rstd[keep], want="dx")[0]
    check_backward(dy[keep], x[keep], w, mean[keep], rstd[keep], dx[keep], None, None)
    check_backward(dy[keep], x[keep], w, mean[keep], rstd[keep], rdx, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1, 2, 3, 5, 7, 9, 15, 17])
@pytest.mark.parametrize("t", ["f32", "f16"])
def test_short_rows_at_every_offset(dev, sm, cols, t):
    for offset in range(9):
        x, w, b, dy = make(200, cols, TYPES[t], torch.float32, seed=offset)
        _, xs = strided(x, 1 + offset % 3, offset)
        _, ds = strided(dy, 2, 8 - offset)
        flat, ys = strided(torch.zeros_like(x), 3, 2)
        y, mean, rstd = run_forward(dev, sm, xs, w, b, y=ys)
        check_forward(x, w, b, 1e-5, y, mean, rstd)
        assert bool((flat[2:].view(200, -1)[:, cols:] == 7.25).all())
        check_backward(dy, x, w, mean, rstd, *run_backward(dev, sm, ds, xs, w, mean, rstd))


def exact_sums(rows, cols, t, seed=0):
    """Values n / 64 with whole n, |n| <= 200, and row sums of their own choice: any order of adding up to 2^24 / 200
    of them is exact in fp32. Means between 1e-4 and 1e-2 where the width allows, both signs."""
    g = torch.Generator().manual_seed(seed)
    n = (64 * torch.randn(rows, cols, generator=g)).round().clamp(-190, 190).long()
    want = (64 * cols * 10 ** (-4 + 2 * torch.rand(rows, generator=g))).round().long().clamp_min(1) * (1 - 2 * (torch.arange(rows) % 2))
    off = want - n.sum(1)
    n += off.div(cols, rounding_mode="floor")[:, None] + (torch.arange(cols)[None] < (off % cols)[:, None])
    assert bool((n.sum(1) == want).all()) and int(n.abs().max()) <= 200
    return (n / 64).to(TYPES[t]).cuda(), want.double().cuda() / 64 / cols


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 1024), (5, 1031), (400, 1024), (400, 600), (300, 1031), (300, 5000), (3, 5001), (2, 10000), (3, 12001), (3, 20000), (2, 40000)])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_small_means_keep_their_digits(dev, sm, rows, cols, t):
    """The sum is exact; 1 / cols and the product with it are rounded once each (2 steps of 2^-24, and their product)."""
    x, want = exact_sums(rows, cols, t, seed=cols)
    assert torch.equal(x.double().mean(1), want)
    _, mean, rstd = run_forward(dev, sm, x, None, None)
    off = (mean.double() - want).abs() / want.abs()
    assert bool((off <= 2.01 * U).all()), off.max()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [64, 1024, 1031, 5000, 10000, 20000])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_means_of_rows_far_from_zero(dev, sm, cols, t):
    """m + dm: the correction dm is a mean of differences x - m, each rounded by U of itself and added up with SUMS roundings;
    1 / cols, the product with it and the last sum are rounded once each."""
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn(50, cols, generator=g) + 1000 * (1 - 2 * (torch.arange(50) % 2))[:, None]).to(TYPES[t]).cuda()
    _, mean, _ = run_forward(dev, sm, x, None, None)
    want = x.double().mean(1)
    spread = (x.double() - want[:, None]).abs().mean(1) + 2 * SUMS(cols) * U * want.abs()      # about m, which itself is off by a sum's roundings
    assert bool(((mean.double() - want).abs() <= U * want.abs() + (SUMS(cols) + 4) * U * spread).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [24, 1000, 1024, 6001, 20000])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_the_mean_of_a_row_with_infinities(dev, sm, cols, t):
    """One infinity, or several of one sign, are the row's mean; both signs, or a NaN beside them, leave none."""
    inf, nan = float("inf"), float("nan")
    x = make(6, cols, TYPES[t], TYPES[t], seed=cols)[0]
    x[0, cols // 2] = inf
    x[1, 0] = -inf
    x[2, 0] = x[2, cols - 1] = inf
    x[3, 1], x[3, cols - 2] = inf, -inf
    x[4, 3], x[4, cols - 4] = inf, nan
    y, mean, rstd = run_forward(dev, sm, x, None, None)
    assert mean[:3].tolist() == [inf, -inf, inf] and bool(mean[3:5].isnan().all()) and bool(mean[5].isfinite())
    assert bool(y[:5].isnan().all()) and bool(rstd[:5].isnan().all()) and bool(y[5].isfinite().all())


def residual_rows(rows, cols, seed):
    """Rows of a residual stream: a few channels larger than the rest, a small mean of its own in every row."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * (1 + 4 * (torch.rand(cols, generator=g) < 0.02))
    return x - x.mean(1, keepdim=True) + 2e-3 * torch.randn(rows, 1, generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("each", [1, 300])
def test_means_of_centred_rows_carry_a_sums_rounding_and_no_bias(dev, sm, t, each):
    """Row by row (the form of few rows) and all at once. The partial sums of such a row reach 2^5 to 2^6 at the last two levels of
    the tree, where a rounding is 2^-18 / sqrt(12) in the root mean square, and halve with every second level below: some 2.5e-6 in
    all, 2.4e-9 of the mean. Four times that is allowed; what differences from a mean of their own lose together is 2e-8."""
    x = residual_rows(300, 1024, 11).to(TYPES[t]).cuda()
    mean = torch.cat([run_forward(dev, sm, x[i:i + each], None, None)[1] for i in range(0, 300, each)])
    assert (mean.double() - x.double().mean(1)).square().mean().sqrt().item() <= 1e-8


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1024, 1031, 6001, 20000])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_a_row_whose_sum_overflows_has_no_rstd(dev, sm, cols, t):
    """1024 values of 3e36 are beyond fp32: no form may make a finite rstd out of that."""
    x = make(3, cols, TYPES[t], TYPES[t], seed=cols)[0]
    x[1] = 3e36
    y, mean, rstd = run_forward(dev, sm, x, None, None)
    assert not bool(mean[1].isfinite()) and bool(rstd[1].isnan()) and bool(y[1].isnan().all())
    keep = [0, 2]
    check_forward(x[keep], None, None, 1e-5, y[keep], mean[keep], rstd[keep])
