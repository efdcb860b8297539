"""The losses at the vocabulary projection in 64 bits, with bounds on what a kernel may be off.

Bounds, element by element, from the roundings that the kernels make:

* a logit is a sum of D products in 32 bits, 16 at a time: each of the D / 16 additions (and the 16
  products' alignment) loses at most 2^-23 of the sum of the magnitudes S,
      dz = (D / 16 + 16) * 2^-23 * S;
* lse and a logit at a target are then off by dz / tau each, and by a few steps of 32 bits of
  themselves (exp2, log, sums of up to 256 terms per tile: 2^-18 relative of the sum of exponentials);
* G = g (p - q) is rounded to the operands' type (half a step h), p and q are off by a relative 2 dz /
  tau + 2^-18; in half precision, steps below 2^-14 are 2^-24 wide, whatever the value;
* numbers below 2^-126, the smallest normal number of 32 bits and of bf16, may be zeros: the
  exponentials (scaled by at most the largest g), and a result;
* the products with G accumulate n terms in 32 bits, at most (n / 16 + 16 + 16) * 2^-23 of the
  magnitudes' sum (splits and pieces included), and round to the operands' type once.
"""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def targets_of(index, ignore_index):
    """Cross entropy as a sparse distribution: (kept, index K=1, q K=1)."""
    kept = index != ignore_index
    return kept, torch.where(kept, index, 0)[:, None].long(), torch.ones(len(index), 1, dtype=torch.float64,
                                                                         device=index.device)


def teacher_of(logits, index, tau):
    """A teacher's entries as a sparse distribution; entries of one token stand together in its first."""
    there = (index >= 0) & (logits.double() != -math.inf)
    kept = there.any(1)
    q = torch.zeros(logits.shape, dtype=torch.float64, device=logits.device)
    l = torch.where(there, logits.double() / tau, -math.inf)
    q[kept] = torch.softmax(l[kept], dim=1)
    return kept, torch.where(there, index, 0).long(), torch.where(there, q, 0.0)


def reference(hidden, weight, kept, index, q, tau, reduction, up):
    """(loss, its bound, d_hidden, its bound, d_weight, its bound); rows not kept are left out of everything."""
    dtype, (T, D), V = hidden.dtype, hidden.shape, weight.shape[0]
    dev, f64 = hidden.device, torch.float64
    h, w = hidden[kept].double(), weight.double()
    index, q = index[kept], q[kept]
    n = len(h)
    z = h @ w.T
    dz = (D / 16 + 16) * 2.0 ** -23 * (h.abs() @ w.abs().T)
    dense = torch.zeros(n, V, dtype=f64, device=dev).scatter_add_(1, index, q)
    lse = torch.logsumexp(z / tau, 1) if n else torch.zeros(0, dtype=f64, device=dev)
    logp = z / tau - lse[:, None]
    log_dense = torch.where(dense > 0, dense, 1.0).log()
    rows = tau ** 2 * (dense * (log_dense - logp)).sum(1)
    zmax = dz.max(1).values if n else lse
    off = tau ** 2 * (2 * zmax / tau + 2.0 ** -18 +
                      2.0 ** -21 * (lse.abs() + (dense * (logp.abs() + (z / tau).abs() + log_dense.abs())).sum(1)))
    loss, bound = torch.zeros(T, dtype=f64, device=dev), torch.zeros(T, dtype=f64, device=dev)
    loss[kept], bound[kept] = rows, off
    if reduction == "none":
        g = up.double()[kept]
    else:
        loss, bound = loss.sum(), bound.sum()
        g = up.double().expand(n)
        if reduction == "mean":
            loss, bound, g = loss / max(n, 1), bound / max(n, 1), g / max(n, 1)
        bound = bound + 2.0 ** -23 * loss.abs()
    p = logp.exp()
    G = tau * g[:, None] * (p - dense)
    hs = half_step(dtype)
    rel = 2 * zmax[:, None] / tau + 2.0 ** -18
    E = hs * G.abs() + (tau * g.abs())[:, None] * (p * rel + dense * 2.0 ** -18)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    if n:  # G is scaled to at most 1 before it is rounded
        E = E + tau * g.abs().max() * tiny

    def product(a, e, b):
        d = a @ b
        steps = (a.shape[1] / 16 + 32) * 2.0 ** -23
        return d, (e + steps * (a.abs() + e)) @ b.abs() * (1 + hs) + hs * d.abs() + 2.0 ** -22 * d.abs() + tiny
    dh, dh_off = torch.zeros(T, D, dtype=f64, device=dev), torch.zeros(T, D, dtype=f64, device=dev)
    if n:
        dh[kept], dh_off[kept] = product(G, E, w)
        dw, dw_off = product(G.T, E.T, h)
    else:
        dw, dw_off = torch.zeros(V, D, dtype=f64, device=dev), torch.zeros(V, D, dtype=f64, device=dev)
    return loss, bound, dh, dh_off, dw, dw_off


def check(name, got, want, bound):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    if bool(bad.any()):
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {i}: got "
                             f"{float(got[i])}, want {float(want[i])} +- {float(bound[i])}")
