"""The training operators' measured cases: layer normalisation forward and backward, the orthogonalisation of
a matrix by Newton-Schulz products, and the Muon update built on it.

``own = False`` computes them in elementary torch operations in fp32; ``own = True`` makes the calls that a
program makes of booth_b200. Both take what ``prepare`` returns.
"""
import math

import torch

own = False

LN_EPS = 1e-5
NS_STEPS = 5
NS_ABC = (3.4445, -4.7750, 2.0315)      # the quintic a x + b x^3 + c x^5 of the Muon optimiser
NS_EPS = 1e-7
MU, LR, DECAY = 0.95, 0.02, 0.01        # momentum, learning rate, decoupled weight decay

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one token's activations in a decoder of width 1024: latency is all there is
        {"name": "ln fwd 1x1024 bf16", "op": "layernorm", "rows": 1, "cols": 1024, "type": "bf16", "wtype": "bf16", "pad": 0},
        # a training micro-batch, mixed precision: bf16 activations, fp32 parameters
        {"name": "ln fwd 16384x4096 bf16", "op": "layernorm", "rows": 16384, "cols": 4096, "type": "bf16", "wtype": "f32", "pad": 0},
        # a width that no vector divides, rows that begin anywhere, in fp32
        {"name": "ln fwd 4099x1031 f32", "op": "layernorm", "rows": 4099, "cols": 1031, "type": "f32", "wtype": "f32", "pad": 0},
        # the backward pass of a few rows (one short sequence)
        {"name": "ln bwd 64x1024 f16", "op": "layernorm_backward", "rows": 64, "cols": 1024, "type": "f16", "wtype": "f16", "pad": 0},
        # the backward pass of the training micro-batch
        {"name": "ln bwd 16384x4096 bf16", "op": "layernorm_backward", "rows": 16384, "cols": 4096, "type": "bf16", "wtype": "f32", "pad": 0},
        # fp32 rows that are a column range of a wider matrix, wide
        {"name": "ln bwd 2050x10000 f32 slice", "op": "layernorm_backward", "rows": 2050, "cols": 10000, "type": "f32", "wtype": "f32", "pad": 48},
        # one small square weight's gradient
        {"name": "orth 256x256 f32", "op": "orthogonalise", "batch": 1, "rows": 256, "cols": 256, "type": "f32", "pad": 0},
        # a tall odd matrix (a projection to a vocabulary of odd size) in fp32
        {"name": "orth 2049x1000 f32", "op": "orthogonalise", "batch": 1, "rows": 2049, "cols": 1000, "type": "f32", "pad": 0},
        # the largest square weight in bf16
        {"name": "orth 8192x8192 bf16", "op": "orthogonalise", "batch": 1, "rows": 8192, "cols": 8192, "type": "bf16", "pad": 0},
        # the layers of a small model stacked, weights in bf16
        {"name": "muon 12x 768x2048 bf16", "op": "muon_step", "batch": 12, "rows": 768, "cols": 2048, "gtype": "bf16", "type": "bf16", "mtype": "bf16"},
        # a feed-forward weight: fp32 master weights and momentum, bf16 gradient
        {"name": "muon 4096x1024 f32", "op": "muon_step", "batch": 1, "rows": 4096, "cols": 1024, "gtype": "bf16", "type": "f32", "mtype": "f32"},
        # a large square weight in mixed precision
        {"name": "muon 4096x4096 f32", "op": "muon_step", "batch": 1, "rows": 4096, "cols": 4096, "gtype": "bf16", "type": "f32", "mtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layernorm", "layernorm_backward", "orthogonalise", "muon_step"])
    if op in ("layernorm", "layernorm_backward"):
        while True:
            rows, cols = _log(rng, 1, 32768), _log(rng, 16, 16384)
            if rng.random() < 0.6:
                cols = max(16, cols // 8 * 8)
            if rows * cols <= 1 << 26:
                break
        t = rng.choice(["f32", "bf16", "f16"])
        return {"op": op, "rows": rows, "cols": cols, "type": t, "wtype": rng.choice([t, "f32"]), "pad": rng.choice([0, 0, 8, rng.randrange(1, 100)])}
    while True:
        rows, cols = _log(rng, 16, 8192), _log(rng, 16, 8192)
        batch = rng.choice([1, 1, 1, _log(rng, 2, 32)])
        if rng.random() < 0.6:
            rows, cols = max(16, rows // 64 * 64), max(16, cols // 64 * 64)
        s, l = min(rows, cols), max(rows, cols)
        if batch * s * s * l <= 1 << 38 and batch * rows * cols <= 1 << 26:
            break
    if op == "orthogonalise":
        return {"op": op, "batch": batch, "rows": rows, "cols": cols, "type": rng.choice(["f32", "bf16", "f16"]), "pad": rng.choice([0, 0, 8, 5])}
    t = rng.choice(["f32", "bf16"])
    return {"op": op, "batch": batch, "rows": rows, "cols": cols, "gtype": rng.choice([t, "bf16"]), "type": t, "mtype": rng.choice([t, "f32"])}


def work(case):
    if case["op"] in ("layernorm", "layernorm_backward"):
        r, c, e, we = case["rows"], case["cols"], SIZE[case["type"]], SIZE[case["wtype"]]
        if case["op"] == "layernorm":
            return {"bytes": 2 * r * c * e + 2 * c * we + 8 * r, "flops": 8 * r * c}
        return {"bytes": 3 * r * c * e + 3 * c * we + 8 * r, "flops": 16 * r * c}
    n = case["batch"] * case["rows"] * case["cols"]
    s, l = min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # X Xt and A A are symmetric: half of their products are enough
    flops = case["batch"] * NS_STEPS * (s * s * l + s * s * s + 2 * s * s * l)
    if case["op"] == "orthogonalise":
        return {"bytes": 2 * n * SIZE[case["type"]], "flops": flops}
    return {"bytes": n * (SIZE[case["gtype"]] + 2 * SIZE[case["mtype"]] + 2 * SIZE[case["type"]]), "flops": flops}


# ---- inputs ----

def _padded(t, pad):
    """t as the leading columns of a matrix whose rows are `pad` elements longer."""
    if not pad:
        return t
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + pad, dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


def _gradient(g, batch, rows, cols):
    """A gradient's shape of spectrum: noise of many tokens under eight dominant directions, small in size."""
    k = min(8, rows, cols)
    u = torch.randn(batch, rows, k, generator=g, device="cuda")
    v = torch.randn(batch, k, cols, generator=g, device="cuda")
    return 1e-3 * (torch.randn(batch, rows, cols, generator=g, device="cuda") + u @ v)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op in ("layernorm", "layernorm_backward"):
        r, c, t, wt = case["rows"], case["cols"], TYPES[case["type"]], TYPES[case["wtype"]]
        # a residual stream: a few channels far larger than the rest, a mean of its own in every row
        x = torch.randn(r, c, generator=g, device="cuda") * (1 + 4 * (torch.rand(c, generator=g, device="cuda") < 0.02))
        x += torch.randn(r, 1, generator=g, device="cuda")
        s["x"] = _padded(x.to(t), case["pad"])
        s["w"] = (1 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(wt)
        if op == "layernorm":
            s["b"] = (0.2 * torch.randn(c, generator=g, device="cuda")).to(wt)
        else:
            s["dy"] = _padded((0.1 * torch.randn(r, c, generator=g, device="cuda")).to(t), case["pad"])
            xd = s["x"].double()
            mean = xd.mean(-1)
            s["mean"] = mean.float()
            s["rstd"] = torch.rsqrt((xd - mean[:, None]).square().mean(-1) + LN_EPS).float()
        return s
    b, r, c = case["batch"], case["rows"], case["cols"]
    if op == "orthogonalise":
        s["g"] = _padded(_gradient(g, b, r, c).to(TYPES[case["type"]]), case["pad"])
        return s
    s["g"] = _gradient(g, b, r, c).to(TYPES[case["gtype"]])
    s["m"] = (0.5 * _gradient(g, b, r, c)).to(TYPES[case["mtype"]])
    s["w"] = (torch.randn(b, r, c, generator=g, device="cuda") / math.sqrt(c)).to(TYPES[case["type"]])
    s["scale"] = 0.2 * math.sqrt(max(r, c))        # the update's rms near Adam's
    return s


# ---- plain forms ----

def _newton_schulz(u, steps=NS_STEPS):
    """u in fp32 or fp64, [batch, rows, cols]; the quintic iteration from its Frobenius-normalised value."""
    a, b, c = NS_ABC
    tall = u.shape[-2] > u.shape[-1]
    x = u.mT if tall else u
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "layernorm":
        x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
        mean = x.mean(-1, keepdim=True)
        d = x - mean
        rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + LN_EPS)
        return {"y": (d * rstd * w + b).to(s["x"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if op == "layernorm_backward":
        x, dy, w = s["x"].float(), s["dy"].float(), s["w"].float()
        rstd = s["rstd"][:, None]
        xhat = (x - s["mean"][:, None]) * rstd
        wdy = w * dy
        c1 = wdy.mean(-1, keepdim=True)
        c2 = (wdy * xhat).mean(-1, keepdim=True)
        dx = rstd * (wdy - c1 - xhat * c2)
        return {"dx": dx.to(s["x"].dtype), "dw": (dy * xhat).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["w"].dtype)}
    if op == "orthogonalise":
        return {"out": _newton_schulz(s["g"].float()).to(s["g"].dtype)}
    g = s["g"].float()
    s["m"].copy_(MU * s["m"].float() + (1 - MU) * g)
    u = MU * s["m"].float() + (1 - MU) * g
    s["w"].copy_((1 - LR * DECAY) * s["w"].float() - LR * s["scale"] * _newton_schulz(u))
    return {"w": s["w"], "m": s["m"]}


# ---- the framework's calls ----

_program = {}


def _device(gpu):
    """This program's handle of a GPU, and its stream with its raw address."""
    if gpu not in _program:
        import booth_b200
        dev = booth_b200.Device(gpu)
        types = {torch.float32: booth_b200.F32, torch.bfloat16: booth_b200.BF16, torch.float16: booth_b200.F16}
        _program[gpu] = dev, types, torch.cuda.ExternalStream(dev.stream, device=gpu), dev.stream
    return _program[gpu]


def _framework(s):
    """The operators run on their handle's stream. The program's torch work joins it from the first call on, so that one stream
    orders everything; a caller on another stream (inside a `with torch.cuda.stream(...)`, in another thread) is ordered by
    events on both sides, and the allocator is told of the tensors that both streams use."""
    gpu = (s["x"] if "x" in s else s["g"]).get_device()
    first = gpu not in _program
    dev, types, stream, raw = _device(gpu)
    if torch._C._cuda_getCurrentRawStream(gpu) == raw:      # 0.1 us; torch.cuda.current_stream makes an object, 1.2 us
        return _calls(s, dev, types)
    caller = torch.cuda.current_stream(gpu)
    stream.wait_stream(caller)
    with torch.cuda.stream(stream):
        out = _calls(s, dev, types)
    caller.wait_stream(stream)
    for t in s.values():
        if isinstance(t, torch.Tensor):
            t.record_stream(stream)
    for t in out.values():
        t.record_stream(caller)
    if first and gpu == torch.cuda.current_device():
        torch.cuda.set_stream(stream)
    return out


def _calls(s, dev, types):
    case = s["case"]
    op = case["op"]
    if op == "layernorm":
        x, w, b = s["x"], s["w"], s["b"]
        r, c = x.shape
        y = torch.empty(r, c, dtype=x.dtype, device=x.device)
        mean = torch.empty(r, dtype=torch.float32, device=x.device)
        rstd = torch.empty(r, dtype=torch.float32, device=x.device)
        dev.layernorm(y.data_ptr(), x.data_ptr(), w.data_ptr(), b.data_ptr(), r, c, eps=LN_EPS, dtype=types[x.dtype], wdtype=types[w.dtype],
                      mean=mean.data_ptr(), rstd=rstd.data_ptr(), ldx=x.stride(0), ldy=c)
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "layernorm_backward":
        x, dy, w = s["x"], s["dy"], s["w"]
        r, c = x.shape
        dx = torch.empty(r, c, dtype=x.dtype, device=x.device)
        dw, db = torch.empty_like(w), torch.empty_like(w)
        dtype, wdtype = types[x.dtype], types[w.dtype]
        ws = torch.empty(dev.layernorm_backward_workspace(r, c, dtype, wdtype), dtype=torch.uint8, device=x.device)
        dev.layernorm_backward(dx.data_ptr(), dw.data_ptr(), db.data_ptr(), dy.data_ptr(), x.data_ptr(), w.data_ptr(), s["mean"].data_ptr(),
                               s["rstd"].data_ptr(), r, c, ws.data_ptr(), ws.numel(), dtype=dtype, wdtype=wdtype, lddx=c, lddy=dy.stride(0), ldx=x.stride(0))
        return {"dx": dx, "dw": dw, "db": db}
    if op == "orthogonalise":
        g = s["g"]
        n, r, c = g.shape
        out = torch.empty(n, r, c, dtype=g.dtype, device=g.device)
        ws = torch.empty(dev.orthogonalise_workspace(n, r, c, types[g.dtype]), dtype=torch.uint8, device=g.device)
        dev.orthogonalise(out.data_ptr(), g.data_ptr(), n, r, c, ws.data_ptr(), ws.numel(), dtype=types[g.dtype], steps=NS_STEPS, abc=NS_ABC, eps=NS_EPS,
                          ld_in=g.stride(1), stride_in=g.stride(0))
        return {"out": out}
    g, m, w = s["g"], s["m"], s["w"]
    n, r, c = g.shape
    ws = torch.empty(dev.orthogonalise_workspace(n, r, c, types[w.dtype]), dtype=torch.uint8, device=g.device)
    dev.muon_step(w.data_ptr(), m.data_ptr(), g.data_ptr(), n, r, c, ws.data_ptr(), ws.numel(), lr=LR, scale=s["scale"], momentum=MU, weight_decay=DECAY,
                  nesterov=True, wdtype=types[w.dtype], mdtype=types[m.dtype], gdtype=types[g.dtype], steps=NS_STEPS, abc=NS_ABC, eps=NS_EPS)
    return {"w": w, "m": m}


def run(state):
    return _framework(state) if own else _plain(state)


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layernorm":
        x = s["x"].double()
        mu = x.sum(1) / x.shape[1]
        var = torch.einsum("ij,ij->i", x - mu[:, None], x - mu[:, None]) / x.shape[1]
        r = 1.0 / (var + LN_EPS).sqrt()
        return {"y": torch.addcmul(s["b"].double(), (x - mu[:, None]) * r[:, None], s["w"].double()), "mean": mu, "rstd": r}
    if case["op"] == "layernorm_backward":
        x, dy, w = s["x"].double(), s["dy"].double(), s["w"].double()
        n, r = x.shape[1], s["rstd"].double()
        xh = (x - s["mean"].double()[:, None]) * r[:, None]
        p = torch.einsum("ij,j->i", dy, w) / n
        q = torch.einsum("ij,j,ij->i", dy, w, xh) / n
        dx = torch.einsum("ij,j,i->ij", dy, w, r) - (p * r)[:, None] - xh * (q * r)[:, None]
        return {"dx": dx, "dw": torch.einsum("ij,ij->j", dy, xh), "db": torch.einsum("ij->j", dy)}
    a, b, c = NS_ABC
    if case["op"] == "orthogonalise":
        u = s["g"].double()
    else:
        g = s["g"].double()
        m = (MU * s["m"].double() + (1 - MU) * g).to(s["m"].dtype)
        u = MU * m.double() + (1 - MU) * g
    # the same quintic from products with x alone: y = x xt x, then a x + b y + c x xt y
    x = u if u.shape[1] <= u.shape[2] else u.transpose(1, 2)
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + NS_EPS)
    for _ in range(NS_STEPS):
        xxt = torch.einsum("bik,bjk->bij", x, x)
        y = torch.bmm(xxt, x)
        x = torch.baddbmm(a * x + b * y, xxt, y, alpha=c)
    o = x if u.shape[1] <= u.shape[2] else x.transpose(1, 2)
    if case["op"] == "orthogonalise":
        return {"out": o}
    return {"w": s["w"].double() * (1 - LR * DECAY) - o * (LR * s["scale"]), "m": m.double() if m.dtype != torch.float32 else MU * s["m"].double() + (1 - MU) * g}
