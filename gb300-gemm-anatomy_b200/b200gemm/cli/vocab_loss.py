"""Losses at the vocabulary projection: check, then time, on the LLM projection's operands.

Default: M=8192 activations ~ N(0,1), the 128256 x 4096 projection ~ N(0,0.02),
seed 2 (the LLM projection config), one random token (--loss ce) or --top random
teacher logits (--loss kd) per row. Each way is checked first on sampled rows
against IEEE fp32 logits (losses within 1e-3, gradients within a relative 1e-2),
then timed with CUDA events over back-to-back calls:
  forward   the loss of every row
  train     the mean loss and the gradients of the activations and the weight
Prints one CSV row per way: milliseconds, TFLOP/s of the products that the way
cannot do without (2 M V D forward, 6 M V D train) and the peak memory that the
call allocated.
"""
from __future__ import annotations

import argparse
import sys

WAYS = ("forward", "train")


def build_arg_parser():
    p = argparse.ArgumentParser(prog="vocab_loss", description=__doc__.split("\n\n")[0])
    p.add_argument("--loss", choices=("ce", "kd"), default="ce")
    p.add_argument("--way", choices=WAYS + ("both",), default="both")
    p.add_argument("--rows", type=int, default=8192)
    p.add_argument("--vocab", type=int, default=128256)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--top", type=int, default=64)
    p.add_argument("--temperature", type=float, default=1.0)
    p.add_argument("--ignored", type=float, default=0.0, help="share of the rows without a loss")
    p.add_argument("--dtype", choices=("bf16", "fp16"), default="bf16")
    p.add_argument("--iterations", type=int, default=10)
    p.add_argument("--warmup", type=int, default=3)
    return p


def _check(h, w, index, q, kept, tau, loss, dh, dw):
    """Sampled rows (and, with gradients, sampled tokens) against IEEE fp32 logits; NaN is out of every limit."""
    import torch
    rows, vocab = h.shape[0], w.shape[0]
    if not bool(kept.any()):
        return
    sample = kept.nonzero()[:, 0]
    sample = sample[:: max(1, len(sample) // 48)]
    z = (h[sample].float() @ w.float().t()) / tau
    logp = torch.log_softmax(z, 1)
    qs, at = q[sample], index[sample].clamp(min=0)
    dense = torch.zeros_like(z).scatter_add_(1, at, qs)
    want = tau ** 2 * (torch.xlogy(dense, dense) - dense * logp).sum(1)
    if loss is not None:
        err = float((loss[sample] - want).abs().max())
        if not err <= 1e-3 * tau ** 2:
            raise RuntimeError(f"losses are off by {err}")
    if dh is None:
        return
    n = int(kept.sum())
    grad = tau / n * (logp.exp() - dense)
    want_h = grad @ w.float()
    errs = {"the activations": float((dh[sample].float() - want_h).norm() / want_h.norm())}
    cols = torch.unique(at.flatten())[:64]
    col_of = torch.full((vocab,), -1, dtype=torch.long, device=h.device)
    col_of[cols] = torch.arange(len(cols), device=h.device)
    want_w = torch.zeros(len(cols), h.shape[1], device=h.device)
    for r in kept.nonzero()[:, 0].split(1024):
        z = (h[r].float() @ w.float().t()) / tau
        g = (z[:, cols] - torch.logsumexp(z, 1, keepdim=True)).exp()
        c = col_of[index[r].clamp(min=0)]
        g.scatter_add_(1, c.clamp(min=0), torch.where(c >= 0, -q[r], 0.0))
        want_w += tau / n * g.t() @ h[r].float()
    errs["the weight"] = float((dw[cols].float() - want_w).norm() / want_w.norm())
    for name, err in errs.items():
        if not err <= 1e-2:
            raise RuntimeError(f"gradients of {name} are off by a relative {err}")


def run(args):
    import torch

    from .. import operands, vocab_loss

    dev = torch.device("cuda", torch.cuda.current_device())
    torch.backends.cuda.matmul.allow_tf32 = False
    h, w = operands.llm_operands_device(args.vocab, args.hidden, dev, m=args.rows)
    if args.dtype == "fp16":
        h, w = h.half(), w.half()
    g = torch.Generator(device=dev).manual_seed(3)
    kept = torch.ones(args.rows, dtype=torch.bool, device=dev)
    kept[torch.randperm(args.rows, generator=g, device=dev)[:int(args.rows * args.ignored)]] = False
    if args.loss == "ce":
        target = torch.randint(0, args.vocab, (args.rows,), generator=g, device=dev)
        target[~kept] = vocab_loss.IGNORE_INDEX
        index, q = target[:, None], kept[:, None].float()
        call = lambda a, b, r: vocab_loss.linear_cross_entropy(a, b, target, reduction=r)  # noqa: E731
    else:
        logits = torch.randn(args.rows, args.top, generator=g, device=dev) * 3
        index = torch.randint(0, args.vocab, (args.rows, args.top), generator=g, device=dev)
        index[~kept] = -1
        q = torch.softmax(logits / args.temperature, 1) * kept[:, None]
        call = lambda a, b, r: vocab_loss.linear_distillation(  # noqa: E731
            a, b, logits, index, temperature=args.temperature, reduction=r)
    hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()

    def forward():
        return call(h, w, "none"), None, None

    def train():
        loss = call(hg, wg, "mean")
        return (None, *torch.autograd.grad(loss, (hg, wg)))

    rows = []
    for way, fn in (("forward", forward), ("train", train)):
        if args.way not in (way, "both"):
            continue
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = fn()
        peak = torch.cuda.max_memory_allocated() - before
        _check(h, w, index, q, kept, args.temperature, *out)
        del out
        for _ in range(args.warmup):
            fn()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        e0.record()
        for _ in range(args.iterations):
            fn()
        e1.record()
        torch.cuda.synchronize()
        ms = e0.elapsed_time(e1) / args.iterations
        flop = (2.0 if way == "forward" else 6.0) * int(kept.sum()) * args.vocab * args.hidden
        rows.append((args.loss, way, args.dtype, args.rows, args.vocab, args.hidden,
                     args.top if args.loss == "kd" else 1, int(kept.sum()), f"{ms:.4f}", f"{flop / ms / 1e9:.1f}",
                     f"{peak / 2 ** 20:.1f}"))
    return rows


def main(argv=None) -> int:
    parser = build_arg_parser()
    try:
        args = parser.parse_args(argv)
    except SystemExit as exc:
        return 2 if exc.code else 0
    if args.iterations < 1 or args.warmup < 0 or args.rows < 1 or not 0.0 <= args.ignored < 1.0:
        print("vocab_loss: ERROR: --iterations and --rows must be >= 1, --ignored in [0, 1)", file=sys.stderr)
        return 2
    if args.loss == "ce" and args.temperature != 1.0:
        print("vocab_loss: ERROR: --temperature belongs to --loss kd", file=sys.stderr)
        return 2
    try:
        import torch
        if not torch.cuda.is_available():
            raise RuntimeError("no CUDA device is visible")
        rows = run(args)
    except Exception as exc:
        print(f"vocab_loss: ERROR: {type(exc).__name__}: {exc}", file=sys.stderr)
        return 1
    print("loss,way,dtype,rows,vocab,hidden,top,rows_with_loss,ms,tflops,peak_mib")
    for r in rows:
        print(",".join(str(x) for x in r))
    return 0


if __name__ == "__main__":
    sys.exit(main())
