"""Cases of the dense operators (layer norm, dropout, gated feed-forward) and their plain forms.

`own` false: elementary torch operations, in 32 bits, rounded once at the end.  `own` true: the
calls a user makes of quickrank_amd.dense.  Both take what `prepare` gives."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")
EPS = 1e-5

# the counter-based generator: SplitMix64's finalizer over a Weyl sequence of words, four elements a word
WEYL, MUL1, MUL2, ALL = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB, (1 << 64) - 1


def listed():
    return [
        # the standardised features of one query's 100 candidates, at serving time: a call's latency
        dict(name="norm one query", op="norm", rows=100, cols=136, type="f32", params="f32"),
        # the features of a whole training set (1M documents x 136), normalised once per epoch
        dict(name="norm training set", op="norm", rows=1_000_000, cols=136, type="f32", params="f32"),
        # the hidden activations of a training batch, backward, all three gradients
        dict(name="norm gradient hidden", op="norm_grad", rows=65_536, cols=2048, type="bf16", params="bf16"),
        # rows of odd length and a ragged number of documents, parameters kept in 32 bits
        dict(name="norm gradient odd", op="norm_grad", rows=71_291, cols=1001, type="f16", params="f32"),
        # hidden activations of one query's candidates: a call's latency
        dict(name="dropout one query", op="drop", rows=100, cols=512, type="f32", residual=False, p=0.2),
        # the end of a residual branch on a training batch: drop, scale, add
        dict(name="dropout residual", op="drop", rows=65_536, cols=2048, type="bf16", residual=True, p=0.1),
        # the backward pass of a ragged batch: rows that do not fill their last words
        dict(name="dropout gradient odd", op="drop_grad", rows=99_991, cols=1145, type="f16", residual=False, p=0.5),
        # one document scored by itself: bound by reading the weights
        dict(name="ffn one document", op="ffn", m=1, k=1024, n=4096, type="bf16", act="silu", save=False),
        # the 100 candidates of one query on their 136 features, in the features' own 32 bits
        dict(name="ffn one query", op="ffn", m=100, k=136, n=512, type="f32", act="gelu", save=False),
        # the forward pass of a training batch, projections saved for the backward pass
        dict(name="ffn batch", op="ffn", m=32_768, k=1024, n=4096, type="bf16", act="silu", save=True),
        # the backward pass of a training batch
        dict(name="ffn gradient batch", op="ffn_grad", m=16_384, k=1024, n=4096, type="bf16", act="silu"),
        # the first layer's backward pass over 1000 queries' features: few weights, a long sum over documents
        dict(name="ffn gradient features", op="ffn_grad", m=100_000, k=136, n=512, type="f32", act="silu"),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm; every other one odd."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v | 1 if rng.random() < 0.5 else v))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "drop", "drop_grad", "ffn", "ffn_grad"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op.startswith("ffn"):
        k, n = _spread(rng, 8, 2048), _spread(rng, 8, 8192)
        most = (64_000 if kind != "f32" else 16_000) * 1_000_000
        m = _spread(rng, 1, max(1, min(131_072, most // (k * n))))
        case = dict(op=op, m=m, k=k, n=n, type=kind, act=rng.choice(ACTS))
        return dict(case, save=rng.random() < 0.5) if op == "ffn" else case
    # (a norm over a few columns leaves next to nothing of its gradient but rounding)
    cols = _spread(rng, 8 if op.startswith("norm") else 1, 16_384)
    rows = _spread(rng, 1, max(1, min(1_000_000, 130_000_000 // cols)))
    if op.startswith("norm"):
        return dict(op=op, rows=rows, cols=cols, type=kind, params=rng.choice([kind, "f32"]))
    return dict(op=op, rows=rows, cols=cols, type=kind, residual=op == "drop" and rng.random() < 0.5,
                p=round(rng.uniform(0.0, 0.6), 3))


def _normal(g, shape, kind, scale=1.0, shift=0.0):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return x.mul_(scale).add_(shift).to(TYPES[kind])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s, kind, op = dict(case), case["type"], case["op"]
    if op.startswith("ffn"):
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = _normal(g, (m, k), kind)
        s["wg"], s["wu"] = (_normal(g, (n, k), kind, k ** -0.5) for _ in range(2))
        if op == "ffn_grad":  # what the forward pass of the same step has left
            s["g"], s["u"] = ((s["x"].float() @ s[w].float().T).to(TYPES[kind]) for w in ("wg", "wu"))
            s["dh"] = _normal(g, (m, n), kind)
        return s
    shape = (case["rows"], case["cols"])
    if op.startswith("norm"):
        s["x"] = _normal(g, shape, kind, 1.5, 0.5)
        s["w"] = _normal(g, shape[1:], case["params"], 0.2, 1.0)
        s["b"] = _normal(g, shape[1:], case["params"], 0.2)
        if op == "norm_grad":
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = ((x - s["mean"][:, None]).square().mean(1) + EPS).rsqrt()
            s["dy"] = _normal(g, shape, kind)
        return s
    s["x"] = _normal(g, shape, kind)
    s["res"] = _normal(g, shape, kind) if case["residual"] else None
    s["seed"], s["offset"] = seed * 7 + 1, 1000 + seed % 97
    return s


# -- plain forms -----------------------------------------------------------------------------------

def _signed(v):
    v &= ALL
    return v - (1 << 64) if v >> 63 else v


def _mix(z):
    """SplitMix64's finalizer of int64 tensors (products wrap; shifts made logical by a mask)."""
    z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * _signed(MUL1)
    z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * _signed(MUL2)
    return z ^ ((z >> 31) & ((1 << 33) - 1))


def _drop(x, res, p, seed, offset):
    limit = round(p * 65536)
    key = int(_mix(torch.tensor(_signed(seed))))
    n = x.numel()
    word = torch.arange(-(-n // 4), device=x.device, dtype=torch.int64)
    word = _mix((word + (offset + 1)) * _signed(WEYL) + key)
    part = torch.stack([(word >> s) & 0xFFFF for s in (0, 16, 32, 48)], 1).reshape(-1)[:n].reshape(x.shape)
    y = torch.where(part >= limit, x.float() * (65536.0 / (65536 - limit)), 0.0)
    return (y if res is None else y + res.float()).to(x.dtype)


def _act(name, g):
    """(the activation, its derivative) of g."""
    if name == "relu":
        return torch.clamp(g, min=0), (g > 0).to(g.dtype)
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    sig = 1 / (1 + torch.exp(-g))
    if name == "sigmoid":
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


def _norm(s):
    x = s["x"].float()
    mean = x.mean(1)
    rstd = ((x - mean[:, None]).square().mean(1) + EPS).rsqrt()
    y = (x - mean[:, None]) * rstd[:, None] * s["w"].float() + s["b"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _norm_grad(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    hat = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["w"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    t = s["w"].dtype
    return {"dx": dx.to(s["x"].dtype), "dw": (dy * hat).sum(0).to(t), "db": dy.sum(0).to(t)}


def _ffn(s):
    x, t = s["x"].float(), s["x"].dtype
    g, u = x @ s["wg"].float().T, x @ s["wu"].float().T
    h = (_act(s["act"], g)[0] * u).to(t)
    return {"h": h, "g": g.to(t), "u": u.to(t)} if s["save"] else {"h": h}


def _ffn_grad(s):
    x, t, dh = s["x"].float(), s["x"].dtype, s["dh"].float()
    a, d = _act(s["act"], s["g"].float())
    dg, du = dh * s["u"].float() * d, dh * a
    dx = dg @ s["wg"].float() + du @ s["wu"].float()
    return {"dx": dx.to(t), "dwg": (dg.T @ x).to(t), "dwu": (du.T @ x).to(t)}


def run(state):
    s, op = state, state["op"]
    if own:
        from quickrank_amd import dense
        if op == "norm":
            y, mean, rstd = dense.layer_norm(s["x"], s["w"], s["b"], EPS)
            return {"y": y, "mean": mean, "rstd": rstd}
        if op == "norm_grad":
            dx, dw, db = dense.layer_norm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"])
            return {"dx": dx, "dw": dw, "db": db}
        if op == "drop":
            return {"y": dense.dropout(s["x"], s["p"], s["seed"], s["offset"], residual=s["res"])}
        if op == "drop_grad":
            return {"dx": dense.dropout_backward(s["x"], s["p"], s["seed"], s["offset"])}
        if op == "ffn":
            out = dense.gated_ffn(s["x"], s["wg"], s["wu"], s["act"], save=s["save"])
            return dict(zip(("h", "g", "u"), out)) if s["save"] else {"h": out}
        dx, dwg, dwu = dense.gated_ffn_backward(s["dh"], s["x"], s["wg"], s["wu"], s["g"], s["u"], s["act"])
        return {"dx": dx, "dwg": dwg, "dwu": dwu}
    if op == "norm":
        return _norm(s)
    if op == "norm_grad":
        return _norm_grad(s)
    if op == "ffn":
        return _ffn(s)
    if op == "ffn_grad":
        return _ffn_grad(s)
    y = _drop(s["x"], s["res"], s["p"], s["seed"], s["offset"])
    return {"y" if op == "drop" else "dx": y}


def work(case):
    e, op = BYTES[case["type"]], case["op"]
    if op.startswith("ffn"):
        m, k, n = case["m"], case["k"], case["n"]
        if op == "ffn":
            return {"bytes": e * (m * k + 2 * n * k + m * n * (3 if case["save"] else 1)), "flops": 4 * m * n * k}
        return {"bytes": e * (3 * m * n + 2 * m * k + 4 * n * k), "flops": 8 * m * n * k}
    size, cols = case["rows"] * case["cols"], case["cols"]
    if op == "norm":
        return {"bytes": 2 * e * size + 8 * case["rows"] + 2 * BYTES[case["params"]] * cols, "flops": 8 * size}
    if op == "norm_grad":
        return {"bytes": 3 * e * size + 8 * case["rows"] + 3 * BYTES[case["params"]] * cols, "flops": 15 * size}
    return {"bytes": e * size * (3 if case["residual"] else 2), "flops": 2 * size}


# -- the definitions in 64 bits ----------------------------------------------------------------------

def _exact_bits(n, seed, offset):
    """The 16-bit numbers of n elements, with 64-bit products put together from 16-bit ones (none wraps)."""
    def limbs(v):
        return [(v >> s) & 0xFFFF for s in (0, 16, 32, 48)]

    def times(a, c):
        c, out, carry = limbs(c), [], 0
        for i in range(4):
            t = carry + sum(a[j] * c[i - j] for j in range(i + 1))
            out.append(t & 0xFFFF)
            carry = t >> 16
        return out

    def plus(a, b):
        out, carry = [], 0
        for p, q in zip(a, b):
            t = p + q + carry
            out.append(t & 0xFFFF)
            carry = t >> 16
        return out

    def fold(a, s):  # a ^ (a >> s)
        q, r = divmod(s, 16)
        up = list(a) + [0] * 5
        return [a[i] ^ ((up[i + q] >> r) | ((up[i + q + 1] << (16 - r)) & 0xFFFF)) for i in range(4)]

    def finish(a):
        return fold(times(fold(times(fold(a, 30), MUL1), 27), MUL2), 31)

    key = finish(limbs(seed & ALL))
    count = torch.arange(offset + 1, offset + 1 + (n + 3) // 4, dtype=torch.int64, device="cuda")
    return torch.stack(finish(plus(times(limbs(count), WEYL), key)), -1).flatten()[:n]


def _exact_act(name, g):
    """(the activation, its derivative) from the definition, the derivative by autograd."""
    g = g.detach().requires_grad_(True)
    f = {"relu": torch.relu, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[name](g)
    d, = torch.autograd.grad(f.sum(), g)
    return f.detach(), d


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    op = case["op"]
    if op in ("drop", "drop_grad"):
        limit = int(math.floor(case["p"] * 65536 + 0.5))
        kept = _exact_bits(s["x"].numel(), s["seed"], s["offset"]).view(s["x"].shape) >= limit
        y = torch.zeros_like(d["x"])
        y[kept] = d["x"][kept] / (1 - limit / 65536)
        if d["res"] is not None:
            y += d["res"]
        return {"y" if op == "drop" else "dx": y}
    if op == "norm":
        var, mean = torch.var_mean(d["x"], 1, correction=0)
        y = torch.addcmul(d["b"], (d["x"] - mean.unsqueeze(1)) / (var + EPS).sqrt().unsqueeze(1), d["w"])
        return {"y": y, "mean": mean, "rstd": 1 / (var + EPS).sqrt()}
    if op == "norm_grad":
        c = case["cols"]
        hat = (d["x"] - d["mean"].unsqueeze(1)).mul_(d["rstd"].unsqueeze(1))
        a, b = d["dy"] @ d["w"], (d["dy"] * hat) @ d["w"]  # a row's sums of g and of g times hat
        dx = torch.addcmul(d["dy"] * d["w"] - (a / c).unsqueeze(1), hat, (b / c).unsqueeze(1), value=-1)
        return {"dx": dx.mul_(d["rstd"].unsqueeze(1)), "dw": torch.linalg.vecdot(d["dy"], hat, dim=0),
                "db": torch.ones(case["rows"], dtype=torch.float64, device="cuda") @ d["dy"]}
    if op == "ffn":
        g, u = torch.nn.functional.linear(d["x"], torch.cat([d["wg"], d["wu"]])).split(case["n"], 1)
        h = _exact_act(case["act"], g)[0] * u
        return {"h": h, "g": g, "u": u} if case["save"] else {"h": h}
    a, slope = _exact_act(case["act"], d["g"])
    both = torch.cat([d["dh"] * d["u"] * slope, d["dh"] * a], 1)
    dw = both.T.contiguous() @ d["x"]
    return {"dx": both @ torch.cat([d["wg"], d["wu"]]), "dwg": dw[:case["n"]], "dwu": dw[case["n"]:]}
