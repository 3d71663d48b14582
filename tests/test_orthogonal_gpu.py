"""Newton-Schulz orthogonalisation and the Muon update against the iteration in 64 bits.

Tolerance. A step is computed as S = X Xt + beta I, Q = c S S + gamma I, X' = Q X (beta = b / 2c, gamma = a - b^2 / 4c; with
c = 0, Q = b A + a I). With r the relative rounding of an operand (2^-11 for one fp16 plane, 2^-21 for two: hi + lo, and lo.lo
left out of the products) and t the error of a product's sum relative to the product of the operands' magnitudes (the tensor
core drops what lies below the last bit of its sum, 2^-23 an add; one plane: an add per 16 of K; two planes: 24 adds
a chunk of 128, and one fp32 add, 2^-24, per chunk), it makes, to first order in Frobenius norms (|.|_F, |.|_2 and |.| the
element-wise magnitude),
    dS  = 2 r |X|_2 |X|_F + t | |X||Xt| |_F + r |S|_F
    dQ  = |c| (2 |S|_2 dS + r |S|_2 |S|_F + t | |S||S| |_F) + r |Q|_F
    dX' = |X|_2 dQ + 2 r |Q|_2 |X|_F + t | |Q||X| |_F + 2^-21 |X'|_F
(X is stored in two planes in both cases; one plane leaves out Q X_lo outside the diagonal blocks, whose norm is at most 2 |Q|_2)
and later steps carry it on with the Lipschitz constant of x -> a x + b x^3 + c x^5, taken on singular value pairs from
[0, s]: max over [0, s] of |f'(x)| and |f(x) / x|. The sum of these, with a tenth for second order, and half a step of the
result's type on every element is the bound. The norms come from the 64-bit iteration itself."""
import pytest
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ABC = (3.4445, -4.7750, 2.0315)


def code(sm, t):
    return {torch.float32: sm.F32, torch.bfloat16: sm.BF16, torch.float16: sm.F16}[t]


def iterate64(g, t, steps=5, abc=ABC, eps=1e-7):
    """The result for [batch, rows, cols] in 64 bits and the bound on each matrix's Frobenius error before the last rounding."""
    a, b, c = (torch.tensor(v, dtype=torch.float32).double().item() for v in abc)      # the coefficients as the call receives them
    eps = torch.tensor(eps, dtype=torch.float32).double().item()
    x = g.double()
    tall = x.shape[1] > x.shape[2]
    x = x.mT if tall else x
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + eps)
    one = t == torch.bfloat16
    r = 2.0 ** -11 if one else 2.0 ** -21

    def adds(k):
        return (k / 16 + 1) * 2.0 ** -23 if one else 24 * 2.0 ** -23 + (k / 128 + 1) * 2.0 ** -24

    def fro(m):
        return m.square().sum((1, 2)).sqrt()

    # the singular values follow the scalar iteration: one decomposition gives the norms of every step
    sv = torch.linalg.eigvalsh(x @ x.mT).clamp_min(0).sqrt()
    err = 2.0 ** -21 * fro(x)
    for _ in range(steps):
        A = x @ x.mT
        P = b * A + c * A @ A
        y = a * x + P @ x
        s0, X2 = sv, sv.amax(1)
        sv = (a * sv + b * sv ** 3 + c * sv ** 5).abs()
        k, l = x.shape[1], x.shape[2]
        eye = torch.eye(k, dtype=x.dtype, device=x.device)
        S = A + (b / (2 * c) if c else 0.0) * eye
        Q = P + a * eye
        S2 = (s0 ** 2 + (b / (2 * c) if c else 0.0)).abs().amax(1)
        Q2 = (a + b * s0 ** 2 + c * s0 ** 4).abs().amax(1)
        dS = 2 * r * X2 * fro(x) + adds(l) * fro(x.abs() @ x.abs().mT) + r * fro(S)
        if c:
            dQ = abs(c) * (2 * S2 * dS + r * S2 * fro(S) + adds(k) * fro(S.abs() @ S.abs())) + r * fro(Q)
        else:
            dQ = abs(b) * dS + r * fro(Q)
        local = X2 * dQ + 2 * r * Q2 * fro(x) + adds(k) * fro(Q.abs() @ x.abs()) + 2.0 ** -21 * fro(y)
        grid = torch.linspace(1e-4, 1, 200, dtype=torch.float64, device=x.device)[None] * X2[:, None]
        lip = torch.maximum((a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs(), (a + b * grid ** 2 + c * grid ** 4).abs()).amax(1)
        err = lip * err + local
        x = y
    return (x.mT if tall else x), 1.1 * err


def check(got, want, err):
    h = torch.finfo(got.dtype).eps / 2
    tol = err + h * want.square().sum((1, 2)).sqrt() + (2.0 ** -25 * want[0].numel() ** 0.5 if got.dtype == torch.float16 else 0)
    off = (got.double() - want).square().sum((1, 2)).sqrt()
    assert bool((off <= tol).all()), (off, tol)


def matrices(batch, rows, cols, t, seed=0, kind="noise"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(batch, rows, cols, generator=g, device="cuda")
    if kind == "rank":          # a few directions far above the rest
        k = min(4, rows, cols)
        x = 1e-2 * x + torch.randn(batch, rows, k, generator=g, device="cuda") @ torch.randn(batch, k, cols, generator=g, device="cuda")
    return (1e-3 * x).to(t)


def run(dev, sm, g, out=None, **kw):
    n, r, c = g.shape
    out = torch.full_like(g, 5.0) if out is None else out
    size = dev.orthogonalise_workspace(n, r, c, code(sm, g.dtype))
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")       # NaN in every type: nothing may rely on it
    torch.cuda.synchronize()
    dev.orthogonalise(out.data_ptr(), g.data_ptr(), n, r, c, ws.data_ptr(), size, dtype=code(sm, g.dtype), ld_in=g.stride(1), stride_in=g.stride(0),
                      ld_out=out.stride(1), stride_out=out.stride(0), **kw)
    dev.sync()
    return out


SHAPES = [(1, 1, 1), (1, 1, 9), (1, 7, 1), (2, 3, 5), (1, 16, 16), (3, 8, 200), (1, 63, 65), (1, 64, 64), (5, 33, 31), (1, 65, 130), (2, 128, 128), (1, 127, 129),
          (1, 129, 257), (1, 300, 77), (1, 256, 256), (2, 257, 255), (1, 40, 3000), (1, 2000, 24), (1, 520, 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols", SHAPES)
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["noise", "rank"])
def test_orthogonalise(dev, sm, batch, rows, cols, t, kind):
    g = matrices(batch, rows, cols, TYPES[t], seed=rows + cols, kind=kind)
    check(run(dev, sm, g), *iterate64(g, g.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols", [(1, 2304, 2304), (40, 256, 300), (1, 1100, 4200), (9, 700, 513)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_many_tiles(dev, sm, batch, rows, cols, t):
    """Sizes at which the CTA-pair form runs, with ragged edges, several waves and several matrices."""
    g = matrices(batch, rows, cols, TYPES[t], seed=1)
    check(run(dev, sm, g), *iterate64(g, g.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("steps,abc", [(1, ABC), (2, ABC), (9, ABC), (12, (1.875, -1.25, 0.375)), (8, (1.5, -0.5, 0.0))])
def test_steps_and_coefficients(dev, sm, t, steps, abc):
    g = matrices(2, 90, 150, TYPES[t], seed=3)
    want, err = iterate64(g, g.dtype, steps, abc)
    check(run(dev, sm, g, steps=steps, abc=abc), want, err)
    if steps == 12:             # the classical quintic converges: singular values at one
        s = torch.linalg.svdvals(run(dev, sm, g, steps=steps, abc=abc).double())
        assert bool(((s - 1).abs() < (1e-5 if t == "f32" else 2e-2)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(96, 160), (161, 95), (300, 300)])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_pitches_strides_and_what_lies_between(dev, sm, rows, cols, t):
    g = matrices(3, rows, cols, TYPES[t], seed=4)
    want, err = iterate64(g, g.dtype)
    for pad, gap, shift in ((8, 0, 0), (3, 5, 1), (4, 64, 4)):
        big_in = torch.full((shift + 3 * (rows * (cols + pad) + gap),), 9.0, dtype=g.dtype, device="cuda")
        big_out = big_in.clone()
        view = [b[shift:].as_strided((3, rows, cols), (rows * (cols + pad) + gap, cols + pad, 1), b.storage_offset() + shift) for b in (big_in, big_out)]
        view[0].copy_(g)
        before = big_in.clone()
        check(run(dev, sm, view[0], out=view[1]), want, err)
        assert torch.equal(big_in, before)
        view[1].fill_(9.0)
        assert bool((big_out == 9.0).all())
        check(run(dev, sm, view[0], out=view[0]), want, err)


@pytest.mark.gpu
def test_zero_matrix_scale_and_non_finite_neighbours(dev, sm):
    g = matrices(4, 140, 200, torch.float32, seed=5)
    clean = run(dev, sm, g)
    bad = g.clone()
    bad[1] = 0
    bad[2, 5, 7] = float("nan")
    got = run(dev, sm, bad)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[3], clean[3])
    assert not got[1].any() and bool(got[2].isnan().any())
    bad[2, 5, 7] = float("inf")
    got = run(dev, sm, bad)
    assert torch.equal(got[0], clean[0]) and not bool(got[2].isfinite().all())
    for f in (1e-30, 1e24):     # squares beyond fp32's range on both sides; eps matters below, not above
        s = g * f
        check(run(dev, sm, s, eps=1e-37), *iterate64(s, g.dtype, eps=1e-37))


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_identity_follows_the_scalar_iteration(dev, sm, t):
    for n in (16, 200, 512):
        x = 1 / n ** 0.5
        for _ in range(5):
            x = ABC[0] * x + ABC[1] * x ** 3 + ABC[2] * x ** 5
        g = (7.0 * torch.eye(n, device="cuda"))[None].to(TYPES[t])
        got = run(dev, sm, g)
        assert bool((got[0] - torch.diag(got[0].diagonal()) == 0).all())
        want, err = iterate64(g, g.dtype)
        assert bool(((want[0].diagonal() - x).abs() < 1e-5).all())          # 64 bits, but the coefficients as fp32 and eps
        check(got, want, err)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_same_bits_capture_and_two_handles_at_once(dev, sm, t):
    g = matrices(1, 600, 1000, TYPES[t], seed=6)
    first = run(dev, sm, g)
    assert torch.equal(run(dev, sm, g), first)
    n = dev.orthogonalise_workspace(1, 600, 1000, code(sm, g.dtype))
    stream = torch.cuda.ExternalStream(dev.stream)
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [torch.zeros_like(g) for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    torch.cuda.synchronize()
    for k in range(2):
        with torch.cuda.graph(graphs[k], stream=stream):
            dev.orthogonalise(outs[k].data_ptr(), g.data_ptr(), 1, 600, 1000, ws[k].data_ptr(), n, dtype=code(sm, g.dtype))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):          # each graph has its own workspace: replays may overlap
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    dev.sync()                  # reads the status word of the replays
    other = sm.Device(0)
    try:
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            dev.orthogonalise(outs[0].data_ptr(), g.data_ptr(), 1, 600, 1000, ws[0].data_ptr(), n, dtype=code(sm, g.dtype))
            other.orthogonalise(outs[1].data_ptr(), g.data_ptr(), 1, 600, 1000, ws[1].data_ptr(), n, dtype=code(sm, g.dtype))
        dev.sync()
        other.sync()
        assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    finally:
        other.close()


def muon64(w, m, g, lr, scale, mu, decay, nesterov, wt, **kw):
    f = lambda v: torch.tensor(v, dtype=torch.float32).double().item()  # noqa: E731  (as the call receives it)
    mu, lr, scale, decay = f(mu), f(lr), f(scale), f(decay)
    m64 = mu * m.double() + (1 - mu) * g.double()
    stored = m64.to(m.dtype).double()
    u = mu * stored + (1 - mu) * g.double() if nesterov else stored
    o, err = iterate64(u, wt, **kw)
    # u itself is formed in fp32: three roundings of its two terms
    err = err + 485 * 4 * 2.0 ** -24 * (u.square().sum((1, 2)).sqrt() + g.double().square().sum((1, 2)).sqrt()) / u.square().sum((1, 2)).sqrt().clamp_min(1e-30)
    return (1 - lr * decay) * w.double() - lr * scale * o, m64, lr * abs(scale) * err


def run_muon(dev, sm, w, m, g, **kw):
    n, r, c = w.shape
    size = dev.orthogonalise_workspace(n, r, c, code(sm, w.dtype))
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    dev.muon_step(w.data_ptr(), m.data_ptr(), g.data_ptr(), n, r, c, ws.data_ptr(), size, wdtype=code(sm, w.dtype), mdtype=code(sm, m.dtype),
                  gdtype=code(sm, g.dtype), ld_w=w.stride(1), stride_w=w.stride(0), ld_m=m.stride(1), stride_m=m.stride(0), ld_g=g.stride(1), stride_g=g.stride(0), **kw)
    dev.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("wt,mt,gt", [("f32", "f32", "f32"), ("f32", "f32", "bf16"), ("bf16", "bf16", "bf16"), ("bf16", "f32", "bf16"), ("f32", "bf16", "f16"), ("f16", "f32", "f16")])
@pytest.mark.parametrize("batch,rows,cols", [(1, 1, 6), (2, 64, 96), (1, 130, 61), (3, 200, 259), (1, 513, 300)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(dev, sm, wt, mt, gt, batch, rows, cols, nesterov):
    w = (matrices(batch, rows, cols, torch.float32, seed=7) * 30).to(TYPES[wt])
    m, g = matrices(batch, rows, cols, TYPES[mt], seed=8), matrices(batch, rows, cols, TYPES[gt], seed=9)
    args = dict(lr=0.02, scale=0.2 * max(rows, cols) ** 0.5)
    want_w, want_m, err = muon64(w, m, g, args["lr"], args["scale"], 0.9, 0.05, nesterov, w.dtype)
    before, m0 = g.clone(), m.double()
    w0 = w.double()
    run_muon(dev, sm, w, m, g, momentum=0.9, weight_decay=0.05, nesterov=nesterov, **args)
    assert torch.equal(g, before)
    # the momentum: two products and a sum in fp32, one rounding to its type (f16's smallest step is 2^-24)
    tol = torch.finfo(m.dtype).eps / 2 * want_m.abs() + 4 * 2.0 ** -24 * (m0.abs() + g.double().abs()) + (2.0 ** -25 if mt == "f16" else 0)
    assert bool(((m.double() - want_m).abs() <= tol).all())
    # the weight: the bound of the orthogonalised update, three fp32 roundings, one to the stored type. A momentum that rounds to the
    # other neighbour than the 64-bit one moves u by a step of its type in that place.
    flips = 0.0
    if mt != "f32":
        flip = (m.double() - want_m.to(m.dtype).double()).square().sum((1, 2)).sqrt()
        flips = 0.02 * args["scale"] * 485 * flip / (g.double().square().sum((1, 2)).sqrt() * 0.05)
    h = torch.finfo(w.dtype).eps / 2
    tol = err + flips + (h + 3 * 2.0 ** -24) * (w0.square().sum((1, 2)).sqrt() + want_w.square().sum((1, 2)).sqrt()) + (2.0 ** -25 * (rows * cols) ** 0.5 if wt == "f16" else 0)
    off = (w.double() - want_w).square().sum((1, 2)).sqrt()
    assert bool((off <= tol).all()), (off, tol)


@pytest.mark.gpu
def test_muon_step_strided_and_without_gradient(dev, sm):
    w, m, g = (matrices(2, 90, 130, torch.float32, seed=s) for s in (1, 2, 3))
    ref = [w.clone(), m.clone()]
    run_muon(dev, sm, ref[0], ref[1], g, lr=0.01, scale=2.0, weight_decay=0.1)
    wide = [torch.full((2, 90, 130 + p), 4.0, device="cuda") for p in (1, 4, 7)]
    views = [x[:, :, :130] for x in wide]
    for v, x in zip(views, (w, m, g)):
        v.copy_(x)
    run_muon(dev, sm, *views, lr=0.01, scale=2.0, weight_decay=0.1)
    assert torch.equal(views[1], ref[1])
    # the norms differ by the order of double sums, far below the float they are rounded to
    assert torch.equal(views[0], ref[0])
    assert all(bool((x[:, :, 130:] == 4.0).all()) for x in wide)
    z = torch.zeros_like(g)
    run_muon(dev, sm, w, z, torch.zeros_like(g), lr=0.5, weight_decay=0.5)
    assert not z.any() and torch.equal(w, matrices(2, 90, 130, torch.float32, seed=1) * 0.75)


@pytest.mark.gpu
def test_a_training_step_of_a_normalised_linear_layer(dev, sm):
    """The operators as they are used together: y = LN(x) W and its gradients (the products by the library's GEMM),
    then one Muon step on W; each piece against the same in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens, width, out = 384, 256, 512
    x = torch.randn(tokens, width, generator=g, device="cuda") * 3 + 1
    ln_w, ln_b = 1 + 0.1 * torch.randn(width, generator=g, device="cuda"), 0.1 * torch.randn(width, generator=g, device="cuda")
    w = torch.randn(width, out, generator=g, device="cuda") / width ** 0.5
    target = torch.randn(tokens, out, generator=g, device="cuda")
    m = torch.zeros_like(w)
    leaves = [t.double().requires_grad_() for t in (x, ln_w, ln_b, w)]
    h64 = torch.nn.functional.layer_norm(leaves[0], (width,), leaves[1], leaves[2], 1e-5)
    loss = (h64 @ leaves[3] - target.double()).square().sum() / tokens
    loss.backward()
    h, xt = torch.empty_like(x), torch.empty(width, tokens, device="cuda")
    mean, rstd = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda")
    y, dw, dh, dx = torch.empty_like(target), torch.empty_like(w), torch.empty_like(x), torch.empty_like(x)
    dln = [torch.empty(width, device="cuda") for _ in range(2)]
    n1, n2 = dev.layernorm_backward_workspace(tokens, width), dev.orthogonalise_workspace(1, width, out)
    ws = torch.empty(max(n1, n2), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.ExternalStream(dev.stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        dev.layernorm(h.data_ptr(), x.data_ptr(), ln_w.data_ptr(), ln_b.data_ptr(), tokens, width, mean=mean.data_ptr(), rstd=rstd.data_ptr())
        dev.gemm(y.data_ptr(), h.data_ptr(), w.data_ptr(), tokens, out, width)
        dy = 2 / tokens * (y - target)
        xt.copy_(h.t())
        wt = w.t().contiguous()
        dev.gemm(dw.data_ptr(), xt.data_ptr(), dy.data_ptr(), width, out, tokens)
        dev.gemm(dh.data_ptr(), dy.data_ptr(), wt.data_ptr(), tokens, width, out)
        dev.layernorm_backward(dx.data_ptr(), dln[0].data_ptr(), dln[1].data_ptr(), dh.data_ptr(), x.data_ptr(), ln_w.data_ptr(), mean.data_ptr(),
                               rstd.data_ptr(), tokens, width, ws.data_ptr(), n1)
        dev.muon_step(w.data_ptr(), m.data_ptr(), dw.data_ptr(), 1, width, out, ws.data_ptr(), n2, lr=0.02, scale=1.0)
    dev.sync()
    # the GEMM is good to 1e-6 relative to its operands' magnitudes; three of them follow one another
    for got, leaf in ((dx, leaves[0]), (dln[0], leaves[1]), (dln[1], leaves[2]), (dw, leaves[3])):
        assert (got.double() - leaf.grad).norm() <= 1e-5 * leaf.grad.norm()
    want, want_m, err = muon64(leaves[3].detach()[None], torch.zeros_like(m)[None], dw[None], 0.02, 1.0, 0.95, 0.0, True, torch.float32)
    assert bool(((w.double() - want[0]).norm() <= err + 4 * 2.0 ** -24 * want.norm()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("wt", ["f32", "bf16"])
@pytest.mark.parametrize("batch,rows,cols", [(1, 64, 64), (3, 130, 61), (1, 700, 500), (1, 600, 1000), (2, 2304, 2200)])
def test_a_wait_that_runs_out_leaves_the_weights(sm, wt, batch, rows, cols):
    """Failure detection without a fault: the first product's producers stay silent, so its bounded waits (50 ms here) run out and
    everything behind it works on planes nobody wrote. The weights, and an orthogonalisation's result, stay as they were;
    the next call that waits reports it, and the handle works as before."""
    d = sm.Device(0)
    try:
        d.gemm_wait_limit(50)
        w, m, g = (matrices(batch, rows, cols, TYPES[wt], seed=s) for s in (11, 12, 13))
        w0, m0, args = w.clone(), m.clone(), dict(lr=0.02, scale=1.0, weight_decay=0.1)
        with pytest.raises(sm.Sm100Error, match="gave up waiting on a barrier"):
            run_muon(d, sm, w, m, g, steps=5 | sm.NS_TEST_SILENT_PRODUCER, **args)
        assert torch.equal(w, w0) and not torch.equal(m, m0)
        out = torch.full_like(g, 5.0)
        size = d.orthogonalise_workspace(batch, rows, cols, code(sm, g.dtype))
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for steps in (1 | sm.NS_TEST_SILENT_PRODUCER, 5):       # the call behind it, before anybody has asked, leaves its result too
            d.orthogonalise(out.data_ptr(), g.data_ptr(), batch, rows, cols, ws.data_ptr(), size, dtype=code(sm, g.dtype), steps=steps)
        with pytest.raises(sm.Sm100Error, match="gave up waiting on a barrier"):
            d.sync()
        assert bool((out == 5).all())
        d.sync()
        check(run(d, sm, g), *iterate64(g, g.dtype))
        m.copy_(m0)
        run_muon(d, sm, w, m, g, **args)
        want, _, _ = muon64(w0, m0, g, 0.02, 1.0, 0.95, 0.1, True, w.dtype)
        assert not torch.equal(w, w0) and bool(((w.double() - want).norm() < 0.1 * (w0.double() - want).norm()))
    finally:
        d.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(70, 90), (200, 64)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_matrices_side_by_side_and_shared_sources(dev, sm, rows, cols, t):
    """Three matrices as column ranges of one wide matrix, out of one wide source; and three windows of one source, a row further on each."""
    g = matrices(1, rows, 3 * cols, TYPES[t], seed=21)[0]
    out = torch.full((rows, 3 * cols + 5), 5.0, dtype=g.dtype, device="cuda")
    side = [x.as_strided((3, rows, cols), (cols, x.stride(0), 1)) for x in (g, out)]
    check(run(dev, sm, side[0], out=side[1]), *iterate64(side[0], g.dtype))
    assert bool((out[:, 3 * cols:] == 5.0).all())
    overlap = g.as_strided((3, rows, cols), (cols, cols, 1))
    got = run(dev, sm, overlap, out=torch.zeros(3, rows, cols, dtype=g.dtype, device="cuda"))
    check(got, *iterate64(overlap, g.dtype))


@pytest.mark.gpu
def test_a_replayed_wait_that_runs_out_is_reported(sm):
    """The same out of a graph: the library does not see the replay, and hears of it by the word in the host's memory."""
    d = sm.Device(0)
    try:
        d.gemm_wait_limit(50)
        g = matrices(1, 200, 300, torch.float32, seed=14)
        out = torch.full_like(g, 5.0)
        size = d.orthogonalise_workspace(1, 200, 300)
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        torch.cuda.synchronize()
        for graph, steps in zip(graphs, (5 | sm.NS_TEST_SILENT_PRODUCER, 5)):
            with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(d.stream)):
                d.orthogonalise(out.data_ptr(), g.data_ptr(), 1, 200, 300, ws.data_ptr(), size, steps=steps)
        d.sync()
        side = torch.cuda.Stream()
        for _ in range(2):
            with torch.cuda.stream(side):
                graphs[0].replay()
            torch.cuda.synchronize()
            assert bool((out == 5).all())
            with pytest.raises(sm.Sm100Error, match="gave up waiting on a barrier"):
                d.sync()
            d.sync()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        d.sync()
        check(out, *iterate64(g, g.dtype))
    finally:
        d.close()
