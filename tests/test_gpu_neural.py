"""The neural scorer (quickrank_amd/neural.py): the dense operators run together, under the lambda pass."""
import numpy as np
import pytest
import torch

from datagen import make_dataset

pytestmark = pytest.mark.gpu


def scorer(**kw):
    from quickrank_amd.neural import NeuralScorer
    return NeuralScorer(**{**dict(blocks=2, units=48, drop=0.2, steps=3, seed=5), **kw})


def reference(s, x, offsets):
    """Scores of the same parameters in 64 bits (leaves that autograd follows), masks from the operator itself."""
    from quickrank_amd import dense
    p = {k: v.double().requires_grad_(True) for k, v in s.params.items()}

    def norm(z, name):
        mean, var = z.mean(1, keepdim=True), z.var(1, keepdim=True, unbiased=False)
        return (z - mean) / (var + 1e-5).sqrt() * p[f"norm_{name}.weight"] + p[f"norm_{name}.bias"]
    z = norm(x.double(), "in")
    for b in range(s.blocks):
        y = norm(z, b)
        g = y @ p[f"gate_{b}"].T
        h = (g * torch.sigmoid(g) * (y @ p[f"up_{b}"].T)) @ p[f"down_{b}"].T
        if offsets is not None:
            # (in f32: the scale is that of the mask's 16 bits)
            h = h * dense.dropout(torch.ones(h.shape, device=h.device), s.drop, s.seed, offsets[b]).double()
        z = z + h
    return norm(z, "out") @ p["score"], p


def test_scores_and_gradients_against_64_bits():
    """136 features, 48 units, 300 documents.  Every product and sum is f32 over at most 300 terms: 2^-24 a step, some
    300 steps a layer, seven layers forward and seven back, relative to the largest value of a result."""
    s = scorer()
    x = torch.randn(300, 136, generator=torch.Generator().manual_seed(1)).cuda()
    s.init(136)
    tol = 2.0 ** -24 * 300 * 14
    for train in (False, True):
        s.drawn = 100
        scores, kept = s.forward(x, train=train)
        offsets = [k[7] for k in kept[1:-1]] if train else None
        want, p = reference(s, x, offsets)
        assert (scores.double() - want).abs().max() <= tol * want.abs().max()
    ds = torch.randn(300, generator=torch.Generator().manual_seed(2)).cuda()
    grads = s.backward(kept, ds)
    (want * ds.double()).sum().backward()
    assert set(grads) == set(s.params)
    for name, leaf in p.items():
        assert grads[name].shape == leaf.shape
        assert (grads[name].double() - leaf.grad).abs().max() <= tol * leaf.grad.abs().max(), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_learns_from_the_lambda_pass(dtype):
    """learn() runs on ragged queries; each step's gradient is that of the context's pseudo-responses for its scores."""
    from quickrank_amd import Context
    x, labels, qoff = make_dataset(nq=12, docs_per_query=25, F=40, seed=3)
    s = scorer(dtype=dtype, units=24)
    s.init(40)
    before = {k: v.clone() for k, v in s.params.items()}
    seen = []
    inner = s.backward

    def backward(kept, ds):
        seen.append((s.ctx.get_scores(), ds.cpu().numpy()))
        return inner(kept, ds)
    s.backward = backward
    s.learn(x, labels, qoff)
    assert len(s.train_metric) == 3 and all(np.isfinite(s.train_metric)) and len(seen) == 3
    assert all(torch.isfinite(v).all() and not torch.equal(v, before[k]) for k, v in s.params.items())
    other = Context(0)
    other.upload(x, labels, qoff)
    for scores, ds in seen:
        other.set_scores(scores)
        other.compute_lambdas("NDCG", 10)
        assert np.array_equal(ds, (-other.get_pseudo()[0]).astype(np.float32))
    a, b = s.score_dataset(x), s.score_dataset(x)
    assert a.shape == (len(x),) and np.array_equal(a, b) and np.isfinite(a).all()
    # one document by itself: the same function of its row, by the few-rows kernels.  Sums of another order may round the
    # other way, a step (two units) of each of the some 12 results on the way; a row of 40 such errors reaches the score
    # through a vector of length 1, so grows by at most 40^1/2: 12 x 2 x 6.4 = 154, and the branches add to the row
    one = s.score_dataset(x[7:8])
    unit = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    assert abs(one[0] - a[7]) <= unit * 200 * max(1.0, np.abs(a).max())
    other.close()


@pytest.mark.parametrize("dtype,shift,scale", [(torch.bfloat16, 1e4, 1.0), (torch.bfloat16, -300.0, 0.5), (torch.float16, 2e5, 3e4),
                                               (torch.float16, 1000.0, 0.25), (torch.float32, 1e4, 1.0)])
def test_raw_features_keep_their_digits(dtype, shift, scale):
    """Features are standardised from the 32 bits they come in, whatever type the scorer computes in.  No blocks: the score is
    norm(norm(x)) w with two roundings of half a step on the way.  A rounding of the first result moves the second by at most
    as much (a projection, times a scale of 1), so the score is off by |w| 136^1/2 (1.05 + 1) half steps, and f32's own."""
    s = scorer(blocks=0, drop=0.0, dtype=dtype)
    s.init(136)
    x = (torch.randn(300, 136, generator=torch.Generator().manual_seed(4)) * scale + shift).cuda()
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    # (f32: the mean and the difference from it are off by some steps of the shift)
    own = 2.0 ** -24 * (8 * abs(shift) / scale + 300)
    want, p = reference(s, x, None)
    scores, kept = s.forward(x, train=True)
    assert (scores.double() - want).abs().max() <= (2.1 * half + own) * 136 ** 0.5 * float(p["score"].detach().norm())
    # the first norm's gradients: the sums of |terms|, each off by the roundings of eight factors
    ds = torch.randn(300, generator=torch.Generator().manual_seed(2)).cuda()
    grads = s.backward(kept, ds)
    (want * ds.double()).sum().backward()
    hat = (x.double() - x.double().mean(1, keepdim=True)) / (x.double().var(1, keepdim=True, unbiased=False) + 1e-5).sqrt()
    g = (ds.double()[:, None] * p["score"]).abs()
    dz = g + g.mean(1, keepdim=True) + hat.abs() * (g * hat.abs()).mean(1, keepdim=True)
    for name, terms in (("norm_in.weight", dz * hat.abs()), ("norm_in.bias", dz)):
        assert ((grads[name].double() - p[name].grad).abs() <= (8 * half + 4 * own) * 1.1 * terms.sum(0)).all(), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_optimizer_holds_32_bits(dtype):
    """Parameters in 16 bits are rounded from ones in 32 that the optimizer steps, whose moments have 32 bits too: steps below a
    rounding of a parameter add up, squares of small gradients do not vanish."""
    x, labels, qoff = make_dataset(nq=12, docs_per_query=25, F=40, seed=3)
    s = scorer(dtype=dtype, units=24, drop=0.0, steps=60, rate=1e-5)
    s.init(40)
    before = {k: v.clone() for k, v in s.params.items()}
    seen = []
    plain = torch.optim.Adam

    def adam(*a, **kw):
        seen.append(plain(*a, **kw))
        return seen[-1]
    torch.optim.Adam = adam
    try:
        s.learn(x, labels, qoff)
    finally:
        torch.optim.Adam = plain
    state = [v for st in seen[0].state.values() for v in st.values() if v.dim()]
    assert len(state) == 2 * len(s.params) and all(v.dtype == torch.float32 and torch.isfinite(v).all() for v in state)
    for name, v in s.params.items():
        assert v.dtype == before[name].dtype and torch.isfinite(v).all(), name
    for name in ("gate_0", "up_1", "down_0"):
        # at least 2^-6: one step of 1e-5 is below half a step of bf16 there (2^-14) and 1.4 half steps of f16 (2^-17)
        old = before[name].float().abs() >= 2.0 ** -6
        moved = (s.params[name] != before[name])[old].double().mean()
        # sixty steps of one direction are 6e-4, ten half steps of bf16's smallest of these and one of its largest (0.3)
        assert moved > 0.1, (name, float(moved))
