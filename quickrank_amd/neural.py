"""A neural document scorer on the operators of dense.py, trained by the lambda pass.

A document's score is a function of its feature row alone, as an ensemble's is: normalised features, residual
blocks  z + dropout(gated_ffn(layer_norm(z)) w_down^T),  a last layer norm and one weight vector.  The gradient
that reaches the scores is the one the trees are fitted to (LambdaMart::compute_pseudoresponses,
lambdamart.cc:62-152): the context ranks the scorer's scores and its pseudo-responses are walked up.  As of
trainer.Mart there are learn() on rows, labels and query offsets and score_dataset() on rows (a scorer is
`params`, plain tensors: there is no file format of its own); the scores can also be what boosting starts
from (Context.set_scores)."""
import numpy as np
import torch

from . import dense
from ._capi import Context


class NeuralScorer:
    def __init__(self, blocks=2, units=512, act="silu", drop=0.1, rate=1e-3, steps=100, metric="NDCG", cutoff=10,
                 dtype=torch.float32, seed=0, device=0, ctx=None):
        self.blocks, self.units, self.act, self.drop = blocks, units, act, drop
        self.rate, self.steps, self.metric, self.cutoff = rate, steps, metric, cutoff
        self.dtype, self.seed, self.device = dtype, seed, torch.device("cuda", device)
        self.ctx = ctx if ctx is not None else Context(device)
        self.params, self.leaves, self.drawn, self.train_metric = {}, {}, 0, []

    def init(self, features):
        """Parameters for rows of `features` values: norms and the last vector in f32, products in self.dtype."""
        g = torch.Generator(device=self.device)
        g.manual_seed(self.seed)

        def normal(rows, cols):
            return (torch.randn((rows, cols), generator=g, device=self.device) * cols ** -0.5).to(self.dtype)
        p = {}
        for b in ["in", *range(self.blocks), "out"]:
            p[f"norm_{b}.weight"] = torch.ones(features, device=self.device)
            p[f"norm_{b}.bias"] = torch.zeros(features, device=self.device)
        for b in range(self.blocks):
            p[f"gate_{b}"], p[f"up_{b}"] = normal(self.units, features), normal(self.units, features)
            p[f"down_{b}"] = normal(features, self.units)
        p["score"] = torch.randn(features, generator=g, device=self.device) * features ** -0.5
        self.params, self.leaves = p, {}

    def optimizer(self):
        """Adam over the parameters, in 32 bits: where the operators read 16-bit ones, those are rounded after each step from
        leaves in f32 (in bf16 a step below 2^-9 of a parameter would be lost, in f16 the square of a gradient)."""
        self.leaves = {name: v if v.dtype == torch.float32 else v.float() for name, v in self.params.items()}
        return torch.optim.Adam(list(self.leaves.values()), lr=self.rate)

    def _norm(self, z, name):
        return dense.layer_norm(z, self.params[f"norm_{name}.weight"], self.params[f"norm_{name}.bias"])

    @torch.no_grad()
    def forward(self, x, train=False):
        """(scores f32, what backward needs) of rows on the device; without train nothing is dropped and
        the blocks keep nothing."""
        # (features are standardised from f32: in 16 bits large ones would be infinite, small differences gone)
        x = x.to(torch.float32)
        z, mean, rstd = self._norm(x, "in")
        z = z.to(self.dtype)
        kept = [(x, mean, rstd)]
        for b in range(self.blocks):
            y, mean, rstd = self._norm(z, b)
            gate, up, down = (self.params[f"{n}_{b}"] for n in ("gate", "up", "down"))
            if not train:
                z = z + dense.gated_ffn(y, gate, up, self.act) @ down.T
                continue
            h, g, u = dense.gated_ffn(y, gate, up, self.act, save=True)
            offset = self.drawn
            self.drawn += dense.dropout_words(z)
            kept.append((z, mean, rstd, y, h, g, u, offset))
            z = dense.dropout(h @ down.T, self.drop, self.seed, offset, residual=z)
        y, mean, rstd = self._norm(z, "out")
        kept.append((z, mean, rstd, y))
        return y.float() @ self.params["score"], kept

    @torch.no_grad()
    def backward(self, kept, dscores):
        """The parameters' gradients for the scores' (f32 [rows])."""
        p, out = self.params, {}

        def norm(dy, name, x, mean, rstd):
            dx, out[f"norm_{name}.weight"], out[f"norm_{name}.bias"] = dense.layer_norm_backward(
                dy, x, p[f"norm_{name}.weight"], mean, rstd)
            return dx
        z, mean, rstd, y = kept[-1]
        out["score"] = y.float().T @ dscores
        dz = norm((dscores[:, None] * p["score"]).to(self.dtype), "out", z, mean, rstd)
        for b in reversed(range(self.blocks)):
            z, mean, rstd, y, h, g, u, offset = kept[1 + b]
            branch = dense.dropout_backward(dz, self.drop, self.seed, offset)
            out[f"down_{b}"] = branch.T @ h
            dy, out[f"gate_{b}"], out[f"up_{b}"] = dense.gated_ffn_backward(
                branch @ p[f"down_{b}"], y, p[f"gate_{b}"], p[f"up_{b}"], g, u, self.act)
            dz = dz + norm(dy, b, z, mean, rstd)
        norm(dz.to(torch.float32), "in", *kept[0])
        return out

    def step(self, x, optimizer):
        """One pass over the uploaded training set's rows: scores, their lambdas, the update of the parameters by what
        optimizer() has given (or, without a call of it, by an optimizer of the parameters themselves)."""
        scores, kept = self.forward(x, train=True)
        self.ctx.set_scores(scores.double().cpu().numpy())
        self.ctx.compute_lambdas(self.metric, self.cutoff)
        lam, _ = self.ctx.get_pseudo()
        # (the pseudo-responses point where the scores should go; an optimizer steps against a gradient)
        grads = self.backward(kept, torch.from_numpy(-lam).to(self.device, torch.float32))
        leaves = self.leaves or self.params
        for name, leaf in leaves.items():
            leaf.grad = grads[name].to(leaf.dtype)
        optimizer.step()
        for name, param in self.params.items():
            if param is not leaves[name]:
                param.copy_(leaves[name])
        self.train_metric.append(self.ctx.metric_last())

    def learn(self, x, labels, qoff):
        x = np.ascontiguousarray(x, np.float32)
        self.ctx.upload(x, labels, qoff)
        if not self.params:
            self.init(x.shape[1])
        rows = torch.from_numpy(x).to(self.device)
        optimizer = self.optimizer()
        for _ in range(self.steps):
            self.step(rows, optimizer)
        return self

    def score_dataset(self, x):
        """f64 [rows], as Mart.score_dataset."""
        rows = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(self.device)
        return self.forward(rows)[0].double().cpu().numpy()
