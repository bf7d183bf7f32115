"""64-bit references of the library's operators on device tensors, with the error each output value
may have: the bounds count the roundings a result passes through (half a step of its type each)."""
import math

import torch


def attention(q, k, v, q_ranges, kv_ranges, scale, window=0, prefix_k=None, prefix_v=None):
    """(want, bound, touched): the attention rows of the definition in float64, how far a computed row may
    be off, and which rows belong to a sequence."""
    dtype, dim = q.dtype, q.shape[2]
    group = q.shape[1] // k.shape[1]
    u = torch.finfo(dtype).eps / 2
    # The smallest step of a probability: fp16 has 2^-24 below its normal range (bf16's is negligible).
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    q64, k64, v64 = (t.double() for t in (q, k, v))
    if prefix_k is None:
        pk, pv = k64[:0], v64[:0]
    else:
        pk, pv = prefix_k.double(), prefix_v.double()
    want = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(want)
    touched = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    for (q0, n), (k0, m) in zip(q_ranges, kv_ranges):
        first = m - n  # own place of query 0
        n_cut, m_cut = max(0, min(n, q.shape[0] - q0)), max(0, min(m, k.shape[0] - k0))
        if n_cut == 0:
            continue
        touched[q0:q0 + n_cut] = True
        keys = torch.cat([pk, k64[k0:k0 + m_cut]]).repeat_interleave(group, 1)
        vals = torch.cat([pv, v64[k0:k0 + m_cut]]).repeat_interleave(group, 1)
        place = torch.arange(n_cut, device=q.device)[:, None] + first
        key = torch.arange(-pk.shape[0], m_cut, device=q.device)[None, :]
        seen = (key <= place) | (key < 0)
        if window:
            seen &= (key > place - window) | (key < 0)
        if keys.shape[0] == 0:
            continue
        rows = q64[q0:q0 + n_cut]
        s = torch.einsum("thd,khd->htk", rows, keys) * scale
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
        p = torch.exp(s - top)
        l = p.sum(-1, keepdim=True)
        some = seen.any(1)
        p = torch.where(l > 0, p / l, p)
        # Masked places weigh nothing whatever their value holds.
        vis = vals.permute(1, 0, 2)
        vis = torch.where(torch.isfinite(vis), vis, torch.zeros_like(vis))
        o = torch.matmul(p, vis)
        a = torch.matmul(p, vis.abs())
        # Scores: fp32 sums of dim products, each within (dim + 8) half steps (2^-24) of the sum of the
        # products' magnitudes, doubled for the tensor core's truncated additions; they move every
        # probability and the sum alike, by 2 ds at most.
        mag = torch.einsum("thd,khd->htk", rows.abs(), keys.abs()).amax(-1, keepdim=True) * scale
        ds = (dim + 8) * 2.0 ** -23 * mag
        vmax = vis.abs().amax((0, 1)) if vis.numel() else 0.0
        # A probability's rounding (u), the scores' error, exponentials and fp32 sums (2^-20), the
        # subnormal probabilities, and the result's own rounding.
        b = (u + 2 * ds + 2.0 ** -20) * a + tiny * seen.sum(1)[None, :, None] * vmax / l.clamp_min(1.0) + u * o.abs() + tiny
        want[q0:q0 + n_cut] = torch.where(some[:, None, None], o.permute(1, 0, 2), torch.zeros_like(o.permute(1, 0, 2)))
        bound[q0:q0 + n_cut] = b.permute(1, 0, 2)
    return want, bound, touched


def check(got, want, bound):
    """got within bound of want everywhere; the message names the worst place."""
    err = (got.double() - want).abs()
    over = err - bound
    assert not torch.isnan(got).any(), "NaN in the output"
    worst = int(over.argmax()) if over.numel() else 0
    assert over.numel() == 0 or float(over.flatten()[worst]) <= 0, (
        f"off by {float(err.flatten()[worst]):.3e} where {float(bound.flatten()[worst]):.3e} is allowed, at {worst}")


def linear_q4(x, values, scales, mins):
    """(want, bound) of linear_q4 in float64."""
    n, half = values.shape
    group = 2 * half // scales.shape[1]
    q = torch.empty((n, 2 * half), dtype=torch.float64, device=x.device)
    q[:, 0::2] = (values % 16).double()
    q[:, 1::2] = (values // 16).double()
    s = scales.double().repeat_interleave(group, 1)
    lo = -8.0 * s if mins is None else mins.double().repeat_interleave(group, 1)
    x64 = x.double()
    want = x64 @ (q * s + lo).T
    # Products and sums in fp32 over the parts q s and min (or 8 s) of each weight: at most k + 16
    # roundings of half a step (2^-24), doubled for the tensor core's truncated additions; then the
    # result's own rounding (with fp16's smallest half step).
    mag = x64.abs() @ (q * s.abs() + lo.abs()).T
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    return want, (2 * half + 16) * 2.0 ** -23 * mag + torch.finfo(x.dtype).eps / 2 * want.abs() + tiny


def linear_q4_by_steps(x, values, scales, mins):
    """(want, bound) of linear_q4 in float64, the bound by the steps a sum passes through.

    A group's products with the 4-bit integers are summed by 16-wide tensor products, `group / 16` in a row: each
    aligns its 16 products and the sum so far to the largest and truncates, 18 terms of 2^-23 of what the group
    holds.  The groups' sums are then scaled into a running sum, one or two roundings (2^-24) a group of whatever
    that sum holds by then; the 16 parts of k it may be split into are joined in order.  Partial sums of any run of
    groups are at most twice the largest prefix, plus one group's part before its minimum joins it."""
    n, half = values.shape
    groups = scales.shape[1]
    group = 2 * half // groups
    q = torch.stack([values & 15, values >> 4], -1).double().view(n, groups, group)
    if mins is None:
        q = q - 8
    xg = x.double().view(x.shape[0], groups, group)
    want = torch.empty((x.shape[0], n), dtype=torch.float64, device=x.device)
    bound = torch.empty_like(want)
    sums, mags = xg.sum(2), xg.abs().sum(2)
    step = max(1, (1 << 26) // max(1, x.shape[0] * groups))
    for a in range(0, n, step):
        s = scales[a:a + step].double()[None]
        part = torch.einsum("rgk,ngk->rng", xg, q[a:a + step]) * s
        mag = torch.einsum("rgk,ngk->rng", xg.abs(), q[a:a + step].abs()) * s.abs()
        whole, low = part, 0.0
        if mins is not None:
            m = mins[a:a + step].double()[None]
            whole = part + sums[:, None] * m
            low = (mags[:, None] * m.abs()).sum(2)
        run = whole.cumsum(2)
        most = 2 * run.abs().amax(2) + mag.amax(2)
        want[:, a:a + step] = run[..., -1]
        # A sum of x over a group: at most 16 roundings of half a step, and its product's own.
        bound[:, a:a + step] = (18 * group / 16 * 2.0 ** -23 * mag.sum(2) + 18 * 2.0 ** -24 * low
                                + (2 * groups + 16) * 2.0 ** -24 * most)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    return want, bound + torch.finfo(x.dtype).eps / 2 * (want.abs() + bound) + tiny
