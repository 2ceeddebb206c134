"""The operators of a normalised, Muon-trained denoiser, as cases that can be timed and compared.

Three operators: layer norm over the channels of channels-last rows (forward, and forward with all gradients),
orthogonalisation of a matrix by Newton-Schulz products, and the Muon optimizer step over a flat parameter buffer that
uses it.  With ``own`` false ``run`` computes them from elementary torch operations in 32 bits; with ``own`` true it makes
the calls a user of madiff_amd makes.

Newton-Schulz, for G [m, n] with m <= n (otherwise on the transpose):  X = G / max(|G|_F, eps), then `steps` times
    A = X X^T,   X <- a X + (b A + c A A) X          (a, b, c) = (3.4445, -4.7750, 2.0315)
Muon (Nesterov form), for every matrix of the buffer:
    M <- mu M + (1 - mu) G,   O = newton_schulz((1 - mu) G + mu M),   W <- (1 - lr wd) W - lr s O
with s = 0.2 sqrt(max(m, n)), so that an update's root mean square is that of an Adam step of the same rate.
"""
import math

import torch

own = False

DEV = "cuda"
EPS_NORM = 1e-5
EPS_NS = 1e-7
NS = (3.4445, -4.7750, 2.0315)
STEPS = 5
LR, MU, WD, EMA_BETA = 2e-4, 0.95, 0.01, 0.995
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one environment, three agents, at the U-Net's bottleneck while planning: a call that is all latency
        dict(name="norm fwd 18x1024 bf16", op="norm", grad=False, rows=18, cols=1024, dtype="bf16"),
        # the first skip's attention input in a training step of 256 windows, three agents, twelve time steps
        dict(name="norm train 9216x512 bf16", op="norm", grad=True, rows=9216, cols=512, dtype="bf16"),
        # the fp32 build with a width that is no multiple of anything: rows begin at odd addresses
        dict(name="norm train 6151x777 fp32", op="norm", grad=True, rows=6151, cols=777, dtype="fp32"),
        # guided sampling of many episodes: wide rows, forward only
        dict(name="norm fwd 4093x16384 bf16", op="norm", grad=False, rows=4093, cols=16384, dtype="bf16"),
        # the largest batches: bandwidth alone counts
        dict(name="norm train 262144x1024 bf16", op="norm", grad=True, rows=262144, cols=1024, dtype="bf16"),
        # one small layer (the output projection of a narrow net): latency
        dict(name="ortho 16x128 fp32", op="ortho", batch=1, rows=16, cols=128, dtype="fp32"),
        # a stack of bf16 gradients of odd sizes
        dict(name="ortho 12x333x1001 bf16", op="ortho", batch=12, rows=333, cols=1001, dtype="bf16"),
        # tall matrices: the time projections, stacked
        dict(name="ortho 5x2048x256 fp32", op="ortho", batch=5, rows=2048, cols=256, dtype="fp32"),
        # the widest convolutions of the full network (1024 channels in and out, five taps)
        dict(name="ortho 7x1024x5120 fp32", op="ortho", batch=7, rows=1024, cols=5120, dtype="fp32"),
        # optimizer step of a test-sized network: many small matrices in one call
        dict(name="muon dim 16", op="muon", dim=16, mults="1-4-8", features=10, ema=False),
        # a middle-sized network whose observation width is odd, with its moving average
        dict(name="muon dim 64", op="muon", dim=64, mults="1-2-4-8", features=31, ema=True),
        # the full network
        dict(name="muon dim 128", op="muon", dim=128, mults="1-4-8", features=16, ema=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "norm", "ortho", "ortho", "muon"))
    if op == "norm":
        cols = _log(rng, 16, 16384)
        rows = _log(rng, 1, min(262144, (1 << 28) // cols))
        return dict(op=op, grad=rng.random() < 0.6, rows=rows, cols=cols, dtype=rng.choice(("bf16", "fp32")))
    if op == "ortho":
        rows, cols = _log(rng, 8, 4096), _log(rng, 8, 6000)
        s, l = min(rows, cols), max(rows, cols)
        s = min(s, 1500)
        rows, cols = (s, l) if rows <= cols else (l, s)
        most = 3 * 7 * 1024 * 1024 * 5120 // (3 * s * s * l + s ** 3)
        return dict(op=op, batch=_log(rng, 1, max(1, min(24, most))), rows=rows, cols=cols, dtype=rng.choice(("bf16", "fp32")))
    return dict(op=op, dim=8 * rng.randint(1, 13), mults=rng.choice(("1-4-8", "1-2-4-8", "1-2-4", "1-3-5")), features=rng.randint(5, 90),
                ema=rng.random() < 0.5)


def _matrices(case):
    """(rows, cols) of the weight matrices of a temporal U-Net with cross-agent attention on its skips: two residual
    blocks a level (two five-tap convolutions, a time projection, a 1x1 where the width changes), the resampling
    convolutions, the attention projections and the inverse-dynamics head."""
    dim, f = case["dim"], case["features"]
    widths = [f] + [dim * int(k) for k in case["mults"].split("-")]
    pairs = list(zip(widths[:-1], widths[1:]))
    emb = 2 * dim
    got = [(4 * dim, dim), (dim, 4 * dim)] * 2 + [(dim, 1)]

    def block(i, o):
        return [(o, 5 * i), (o, 5 * o), (o, emb)] + ([(o, i)] if i != o else [])

    def attention(c):
        return [(c // 4, c), (c // 4, c), (c, c), (c // 4, emb), (c // 4, emb), (c, emb)]

    for k, (i, o) in enumerate(pairs):
        got += block(i, o) + block(o, o) + ([(o, 3 * o)] if k < len(pairs) - 1 else [])
    top = widths[-1]
    got += block(top, top) * 2 + attention(top)
    for i, o in reversed(pairs[1:]):
        got += attention(o) + block(2 * o, i) + block(i, i) + [(i, 4 * i)]
    got += [(dim, 5 * dim), (f, dim), (256, 2 * f), (256, 256), (5, 256)]
    return got


def _layout(case):
    """[(offset, rows, cols)] in a flat buffer, each matrix on a 16-byte boundary, and the buffer's length."""
    at, got = 0, []
    for r, c in _matrices(case):
        got.append((at, r, c))
        at += (r * c + 3) // 4 * 4
    return got, at


# ---------------------------------------------------------------------------------------------------- inputs
def _gradient(g, batch, rows, cols):
    """A batch of matrices with the spectrum a layer's gradient has: a few strong directions over a floor of noise."""
    rank = max(1, min(rows, cols) // 8)
    fall = torch.arange(1, rank + 1, device=DEV, dtype=torch.float32).pow(-0.7)
    u = torch.randn(batch, rows, rank, device=DEV, generator=g) * fall
    v = torch.randn(batch, rank, cols, device=DEV, generator=g)
    return (u @ v + 0.1 * torch.randn(batch, rows, cols, device=DEV, generator=g)) * 1e-3


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "norm":
        rows, cols, t = case["rows"], case["cols"], TYPES[case["dtype"]]
        wide = 1.0 + 4.0 * (torch.rand(cols, device=DEV, generator=g) < 0.02)
        x = torch.randn(rows, cols, device=DEV, generator=g).mul_(wide).add_(0.5 * torch.randn(rows, 1, device=DEV, generator=g))
        s = dict(x=x.to(t), weight=1.0 + 0.2 * torch.randn(cols, device=DEV, generator=g), bias=0.1 * torch.randn(cols, device=DEV, generator=g))
        if case["grad"]:
            s["dy"] = (1e-2 * torch.randn(rows, cols, device=DEV, generator=g)).to(t)
        return s
    if case["op"] == "ortho":
        return dict(x=_gradient(g, case["batch"], case["rows"], case["cols"]).to(TYPES[case["dtype"]]))
    mats, n = _layout(case)
    s = {k: torch.zeros(n, device=DEV) for k in ("p", "g", "m")}
    for at, r, c in mats:
        for k, v in (("p", torch.randn(r * c, device=DEV, generator=g) / math.sqrt(c)), ("g", _gradient(g, 1, r, c)), ("m", _gradient(g, 1, r, c))):
            s[k][at:at + r * c] = v.view(-1)
    if case["ema"]:
        s["e"] = s["p"] + 1e-3 * torch.randn(n, device=DEV, generator=g) * (s["p"] != 0)
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["op"] == "norm" and case["grad"]:
        for k in ("x", "weight", "bias"):
            s[k].requires_grad_(True)
    if case["op"] == "muon":
        s["mats"], n = _layout(case)
        s["shadow"] = torch.zeros(n, device=DEV, dtype=torch.bfloat16)       # the weights' bf16 copies that the products read
        if own:
            from madiff_amd.muon import MuonPlan
            s["plan"] = MuonPlan(s["mats"], device=DEV, scales=[0.2 * math.sqrt(max(r, c)) for _, r, c in s["mats"]])
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"norm": _norm, "ortho": _ortho, "muon": _muon}[state["case"]["op"]](state)


def _norm(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    if own:
        from madiff_amd import ops
        y = ops.layer_norm(x, w, b, eps=EPS_NORM)
        if "dy" not in s:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    with torch.no_grad():
        xf = x.float()
        d = xf - xf.mean(-1, keepdim=True)
        rstd = (d.square().mean(-1, keepdim=True) + EPS_NORM).rsqrt()
        xh = d * rstd
        y = (xh * w + b).to(x.dtype)
        if "dy" not in s:
            return {"y": y}
        dy = s["dy"].float()
        dh = dy * w
        dx = rstd * (dh - dh.mean(-1, keepdim=True) - xh * (dh * xh).mean(-1, keepdim=True))
        return {"y": y, "dx": dx.to(x.dtype), "dweight": (dy * xh).sum(0), "dbias": dy.sum(0)}


def _newton_schulz(x):
    a, b, c = NS
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(EPS_NS)
    for _ in range(STEPS):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def _ortho(s):
    if own:
        from madiff_amd import ops
        return ops.orthogonalize(s["x"], steps=STEPS, coefficients=NS, eps=EPS_NS)
    return _newton_schulz(s["x"].float()).to(s["x"].dtype).contiguous()


def _muon(s):
    if own:
        s["plan"].step(s["p"], s["g"], s["m"], lr=LR, momentum=MU, nesterov=True, weight_decay=WD, shadow=s["shadow"],
                       ema=s.get("e"), ema_beta=EMA_BETA)
    else:
        s["m"].mul_(MU).add_(s["g"], alpha=1 - MU)
        u = (1 - MU) * s["g"] + MU * s["m"]
        for at, r, c in s["mats"]:
            w = s["p"][at:at + r * c].view(r, c)
            w.mul_(1 - LR * WD).sub_(_newton_schulz(u[at:at + r * c].view(r, c)), alpha=LR * 0.2 * math.sqrt(max(r, c)))
        s["shadow"].copy_(s["p"])
        if "e" in s:
            s["e"].mul_(EMA_BETA).add_(s["p"], alpha=1 - EMA_BETA)
    return {k: s[k] for k in ("p", "m", "shadow", "e") if k in s}


# ---------------------------------------------------------------------------------------------------- cost
def _ns_flops(r, c):
    """The two symmetric products of a step at half their entries, and the third whole."""
    s, l = min(r, c), max(r, c)
    return STEPS * (s * s * l + s ** 3 + 2 * s * s * l)


def work(case):
    if case["op"] == "norm":
        n, e = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
        if case["grad"]:        # x and dy read, y and dx written, gain, shift and their gradients
            return {"bytes": 4 * n * e + 16 * case["cols"], "flops": 18 * n}
        return {"bytes": 2 * n * e + 8 * case["cols"], "flops": 8 * n}
    if case["op"] == "ortho":
        e = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * e * case["batch"] * case["rows"] * case["cols"], "flops": case["batch"] * _ns_flops(case["rows"], case["cols"])}
    mats = _matrices(case)
    n = sum(r * c for r, c in mats)   # weights and momentum read and written, the gradient read, the bf16 copy written, the average read and written
    return {"bytes": n * (4 * 5 + 2 + (8 if case["ema"] else 0)), "flops": sum(_ns_flops(r, c) for r, c in mats)}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _polar_polynomial(g):
    """The composed Newton-Schulz polynomial of g in float64, through the Gram matrix of the shorter side:
    O = P(K) g / |g|, with P(K) the running product of q(K_k) = a + b K_k + c K_k^2 and K_{k+1} = q(K_k) K_k q(K_k)."""
    a, b, c = NS
    x = g.double()
    flip = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if flip else x
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp_min(EPS_NS)
    eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    k, p = torch.matmul(x, x.transpose(-1, -2).contiguous()), eye
    for _ in range(STEPS):
        q = a * eye + torch.matmul(k, b * eye + c * k)
        p, k = torch.matmul(q, p), torch.matmul(torch.matmul(q, k), q)
    x = torch.matmul(p, x)
    return x.transpose(-1, -2).contiguous() if flip else x


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        x, w, b = (s[k].double() for k in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS_NORM)
        xh = x.sub_(mean).div_(sd)
        out = {"y": torch.addcmul(b, xh, w)}
        if case["grad"]:
            dy = s["dy"].double()
            out["dbias"], out["dweight"] = dy.sum(0), torch.mul(dy, xh).sum(0)
            dy.mul_(w)
            along = torch.mul(dy, xh).mean(-1, keepdim=True)
            out["dx"] = dy.sub_(dy.mean(-1, keepdim=True)).sub_(xh.mul_(along)).div_(sd)
        return out
    if case["op"] == "ortho":
        return _polar_polynomial(s["x"])
    mats, n = _layout(case)
    p, g, m = (s[k].double() for k in ("p", "g", "m"))
    m = m * MU + g * (1 - MU)
    for at, r, c in mats:
        u = (g[at:at + r * c] * (1 - MU) + m[at:at + r * c] * MU).view(r, c)
        p[at:at + r * c] = p[at:at + r * c] * (1 - LR * WD) - LR * 0.2 * math.sqrt(max(r, c)) * _polar_polynomial(u).reshape(-1)
    out = {"p": p, "m": m, "shadow": p.clone()}
    if case["ema"]:
        out["e"] = s["e"].double() * EMA_BETA + p * (1 - EMA_BETA)
    return out
