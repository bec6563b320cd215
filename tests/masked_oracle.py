"""Masked attention in 64 bits, written from its definition, with bounds on the errors of an implementation that rounds as the kernels do.

The bounds count roundings, each at most u = eps / 2 of the 16-bit type relative to the value: of the weights that enter the second product
(and the gradient of values), of dS, and of every result.  `SLACK` covers what is done in 32 bits: scores and their exponents (sums of up to
128 products, exponents of up to about 60: below 2^-16 relative of a weight) and the sums.
"""
import math

import torch

SLACK = 2.0 ** -13


def _u(dtype):
    return torch.finfo(dtype).eps / 2


class Oracle:
    """One call: query [B, M, H, d], key, value [B, L, Hk, d] and the rules of masked_attention."""

    def __init__(self, query, key, value, scale=1.0, causal=False, prefix=None, documents=None, slopes=None, cap=None):
        B, M, H, d = query.shape
        L, Hk = key.shape[1], key.shape[2]
        self.dtype, self.scale, self.shape, self.group = query.dtype, scale, (B, M, H, L, Hk), H // Hk
        self.q = query.double().transpose(1, 2)                                    # [B, H, M, d]
        self.k, self.v = (t.double().transpose(1, 2).repeat_interleave(H // Hk, 1) for t in (key, value))
        pos, j = torch.arange(M, device=query.device) + L - M, torch.arange(L, device=query.device)
        seen = torch.ones(B, M, L, dtype=torch.bool, device=query.device)
        if causal:
            seen = (j <= pos[:, None]).expand(B, M, L)
            if prefix is not None:
                seen = seen | (j < prefix[:, None, None])
        if documents is not None:
            mine = documents[:, L - M:, None]
            seen = seen & (mine == documents[:, None, :]) & (mine >= 0)
        self.seen = seen[:, None]
        x = scale * (self.q @ self.k.transpose(-1, -2))
        self.gain = 1.0
        if cap:
            t = torch.tanh(x / cap)
            x, self.gain = cap * t, 1 - t * t
        if slopes is not None:
            x = x - slopes.double().view(1, H, 1, 1) * (pos[:, None] - j).abs()
        x = torch.where(self.seen, x, -math.inf)
        lse = torch.logsumexp(x, -1)
        self.p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[..., None])
        self.lse = lse.transpose(1, 2)
        self.o = self.p @ self.v
        self.out = self.o.transpose(1, 2)
        self.spread = self.p @ self.v.abs()                                        # sum of p |v|
        u = _u(self.dtype)
        # fp16 weights are at least one for a row's largest, and below 2^-14 absolute: half a step is 2^-25
        floor = L * 2.0 ** -25 if self.dtype == torch.float16 else 0.0
        self.o_tol = (u + SLACK) * self.spread + u * self.o.abs() + floor * (self.v.abs().amax() if L else 0.0) + 1e-30

    def check(self, out, lse=None):
        err = (out.double().transpose(1, 2) - self.o).abs()
        assert torch.isfinite(out).all()
        worst = (err / self.o_tol).max().item() if err.numel() else 0.0
        assert worst <= 1.0, f"out: {worst:.3f} of the bound"
        if lse is not None:
            empty = self.lse == -math.inf
            assert torch.equal(lse == -math.inf, empty)
            if (~empty).any():
                assert ((lse.double() - self.lse).abs()[~empty] <= 2.0 ** -15 * (1 + self.lse[~empty].abs())).all()
        return worst

    def gradients(self, grad_out):
        """dq, dk, dv and the bounds on their errors, in the operands' layouts."""
        B, M, H, L, Hk = self.shape
        u = _u(self.dtype)
        g = grad_out.double().transpose(1, 2)
        dp = g @ self.v.transpose(-1, -2)
        delta = (g * self.o).sum(-1, keepdim=True)
        ds = self.p * (dp - delta) * self.gain
        # delta comes from the rounded result; what is done in 32 bits counts relative to the terms of the difference
        d_delta = (g.abs() * self.o_tol).sum(-1, keepdim=True)
        ds_tol = u * ds.abs() + self.p * (d_delta + SLACK * (g.abs() @ self.v.abs().transpose(-1, -2) + (g.abs() * self.spread).sum(-1, keepdim=True)))
        heads = lambda x: x.view(B, Hk, self.group, L, -1).sum(2).transpose(1, 2)  # noqa: E731
        dq = self.scale * (ds @ self.k)
        dk = self.scale * (ds.transpose(-1, -2) @ self.q)
        dv = self.p.transpose(-1, -2) @ g
        dq_tol = self.scale * (ds_tol @ self.k.abs()) + u * dq.abs()
        dk_tol = self.scale * (ds_tol.transpose(-1, -2) @ self.q.abs())
        dv_tol = ((u + SLACK) * self.p).transpose(-1, -2) @ g.abs()
        dk, dv = heads(dk), heads(dv)
        tiny = 2.0 ** -24 if self.dtype == torch.float16 else 1e-30                 # half a step of fp16's subnormal results
        return ((dq.transpose(1, 2), dq_tol.transpose(1, 2) + tiny), (dk, heads(dk_tol) + u * dk.abs() + tiny),
                (dv, heads(dv_tol) + u * dv.abs() + tiny))

    def check_gradients(self, grad_out, grads):
        for name, got, (want, tol) in zip(("dq", "dk", "dv"), grads, self.gradients(grad_out)):
            assert torch.isfinite(got).all(), name
            worst = ((got.double() - want).abs() / tol).max().item() if want.numel() else 0.0
            assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"
