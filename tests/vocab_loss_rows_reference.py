"""The gradients of the losses at the vocabulary projection in 64 bits, with bounds that go by each row's own weight.

vocab_loss_reference grants every element of G what the largest row's weight costs. Here a row's gradient
is held to its own size, element by element, from the roundings that the kernels make:

* a logit is off by dz, p and q by a relative 2 dz / tau + 2^-18 (see vocab_loss_reference);
* G = p - q, times the row's weight or the part of it in [1, 2), is rounded to half a step h of the
  operands' type. bf16 reaches 2^-126 of the largest row's weight: 2^-100 for weights up to 2^26 apart. In half precision G is held times 2^14, where steps below 2^-14
  are 2^-24 wide: off by 2^-25 of that, 2^-39 |g_t| of its own;
* weights of rows that differ in half precision: the row's power of two goes to d_hidden in 32 bits, and to
  d_weight on a copy of hidden that is scaled until its largest element is 2^14 or more. What that copy loses
  below 2^-14 is 2^-25 of that: 2^-39 A for A = max_t |g_t| max_d |h_td|, times the part of G in [1, 2);
* the products add n terms in 32 bits, at most (n / 16 + 32) 2^-23 of the magnitudes' sum, and round to the
  operands' type once, in half precision by no less than 2^-25.
"""
import torch

import vocab_loss_reference as ref


def gradients(hidden, weight, kept, index, q, tau, up):
    """(d_hidden, its bound, d_weight, its bound) for a weight `up` of each row's loss."""
    dtype, (T, D), V = hidden.dtype, hidden.shape, weight.shape[0]
    dev, f64 = hidden.device, torch.float64
    half = dtype == torch.float16
    hs = ref.half_step(dtype)
    h, w, g = hidden[kept].double(), weight.double(), up.double()[kept]
    n = len(h)
    z = h @ w.T
    dz = ((D / 16 + 16) * 2.0 ** -23 * (h.abs() @ w.abs().T)).max(1, keepdim=True).values
    dense = torch.zeros(n, V, dtype=f64, device=dev).scatter_add_(1, index[kept], q[kept])
    p = torch.softmax(z / tau, 1)
    P = tau * (p - dense)  # G without the row's weight
    tiny = 2.0 ** -39 if half else 2.0 ** -100
    E = hs * P.abs() + tau * (p * (2 * dz / tau + 2.0 ** -18) + dense * 2.0 ** -18 + tiny)
    least = 2.0 ** -25 if half else 2.0 ** -126

    def bound(magnitude, off, want, terms):
        return (off + (terms / 16 + 32) * 2.0 ** -23 * (magnitude + off)) * (1 + hs) + (hs + 2.0 ** -22) * want.abs() + least

    gh, dh, dh_off = g[:, None].abs(), torch.zeros(T, D, dtype=f64, device=dev), torch.zeros(T, D, dtype=f64, device=dev)
    want = P @ w
    dh[kept] = g[:, None] * want
    dh_off[kept] = bound(gh * (P.abs() @ w.abs()), gh * (E @ w.abs()), dh[kept], V)
    dw = (g[:, None] * P).T @ h
    off = (gh * E).T @ h.abs()
    if half and n:
        off = off + 2.0 ** -39 * float((gh * h.abs()).max()) * 2 * (P.abs() + E).sum(0)[:, None]
    dw_off = bound((gh * P.abs()).T @ h.abs(), off, dw, n)
    return dh, dh_off, dw, dw_off
