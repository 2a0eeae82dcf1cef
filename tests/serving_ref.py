"""Plain 64-bit implementations of the serving operators, and the error bounds
their kernels are held to."""

import math

import numpy as np
import torch

LOG2E_ULP = 2.0 ** -21          # exp2 and its argument, relative, per weight


def attention_rows(q, k, v, seen, scale):
    """q [n, nh, hd], k, v [m, nkv, hd], seen bool [n, m] -> (out, lse, out_err, lse_err) in 64 bits.

    ``out_err`` bounds a kernel that multiplies 16-bit operands exactly, sums
    in 32 bits and rounds each softmax weight once to the operands' type:
    a score is off by at most (hd + 2) 2^-24 sum |q k| scale, a weight by twice
    that (its own exponential and the sum it is divided by) plus half a step
    of its type, and the result is rounded once more (``assert_attention``).

    fp16 has a least normal number, 2^-14, below which its half step is 2^-25
    and no longer relative.  The kernels scale the weights so that a row's
    largest is at least 2^7 (its exponent's reference is never less than 7
    under the running maximum), so the sum that divides them is at least 2^7
    too, and a small weight adds at most 2^-25 / 2^7 |v| = 2^-32 |v|."""
    n, nh, hd = q.shape
    nkv = k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    least = 2.0 ** -32 if q.dtype == torch.float16 else 0.0
    q, k, v = (t.double().cpu() for t in (q, k, v))
    seen = seen.cpu()
    out = torch.zeros(n, nh, hd, dtype=torch.float64)
    err = torch.zeros_like(out)
    lse = torch.full((n, nh), -math.inf, dtype=torch.float64)
    lse_err = torch.zeros_like(lse)
    live = seen.any(1)
    if not live.any():
        return out, lse, err, lse_err
    for h in range(nh):
        kh = torch.where(seen.any(0)[:, None], k[:, h // (nh // nkv)], 0.0)   # keys nobody sees do not count
        vh = torch.where(seen.any(0)[:, None], v[:, h // (nh // nkv)], 0.0)
        z = (q[:, h] @ kh.t() * scale).masked_fill(~seen, -math.inf)
        lse[:, h] = torch.logsumexp(z, 1)
        p = torch.where(seen & live[:, None], torch.exp(z - lse[:, h, None]), 0.0)
        out[:, h] = p @ vh
        off = ((q[:, h].abs() @ kh.abs().t() * scale).masked_fill(~seen, 0.0).amax(1) * (hd + 2) * 2.0 ** -24
               + LOG2E_ULP)
        terms = seen.sum(1).clamp(min=1).double().log2() + 130       # additions a partial sum goes through
        err[:, h] = (u + 2 * off + terms * 2.0 ** -24)[:, None] * (p @ vh.abs()) + least * (seen.double() @ vh.abs())
        lse_err[:, h] = off + terms * 2.0 ** -24 + torch.where(live, lse[:, h].abs(), 0.0) * 2.0 ** -22
    return out, lse, err, lse_err


def assert_attention(out, lse, want):
    ref, ref_lse, err, lse_err = want
    u, tiny = torch.finfo(out.dtype).eps / 2, torch.finfo(out.dtype).tiny     # below tiny a half step is u * tiny
    got = out.double().cpu()
    assert torch.isfinite(got).all()
    tol = err + u * (ref.abs() + err).clamp(min=tiny) + 2.0 ** -30
    worst = ((got - ref).abs() / tol).max()
    assert worst <= 1, f"output off by {float(worst):.3g} of its bound"
    if lse is not None:
        got = lse.double().cpu()
        empty = torch.isneginf(ref_lse)
        assert torch.equal(torch.isneginf(got), empty)
        worst = torch.where(empty, 0.0, (got - ref_lse).abs() / (lse_err + 2.0 ** -30)).max()
        assert worst <= 1, f"lse off by {float(worst):.3g} of its bound"


def commit_walk(tokens, parents, predicted, ctx, live, max_ctx):
    """The accepted path of one row."""
    path = []
    if live <= 0 or not 0 <= ctx < max_ctx:
        return path
    path = [0]
    while ctx + len(path) < max_ctx:
        c = path[-1]
        fits = [n for n in range(c + 1, live) if parents[n] == c and tokens[n] == predicted[c]]
        if not fits:
            break
        path.append(fits[0])
    return path


def logprob_rows(x, tokens, num_top):
    """x [M, V] any float type -> dict of 64-bit values; ``tops`` ordered by (value, lowest index)."""
    y = x.double().cpu().numpy()
    tok = tokens.cpu().numpy()
    M, V = y.shape
    got = {"lse": np.zeros(M), "logprob": np.zeros(M), "entropy": np.zeros(M),
           "top_index": np.zeros((M, num_top), np.int64), "top_logprob": np.zeros((M, num_top))}
    for r in range(M):
        m = y[r].max()
        if np.isneginf(m):
            lse, logp, ent = -np.inf, np.full(V, -np.inf), 0.0
        else:
            e = np.exp(y[r] - m)
            lse = m + np.log(e.sum())
            logp = (y[r] - m) - np.log(e.sum())          # (m + log may not be representable beside m)
            p = np.exp(logp)
            ent = -np.sum(np.where(p > 0, p * np.where(p > 0, logp, 0), 0))
        got["lse"][r], got["entropy"][r] = lse, ent
        got["logprob"][r] = logp[tok[r]] if 0 <= tok[r] < V else np.nan
        order = np.lexsort((np.arange(V), -y[r]))[:num_top]
        got["top_index"][r], got["top_logprob"][r] = order, logp[order]
    return got
