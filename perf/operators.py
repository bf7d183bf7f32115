"""Workloads of the library's operators for causal embedding towers and few-row products.

    attention_causal  prompts of different lengths packed back to back, grouped heads, causal
    attention_prefix  texts behind one shared instruction, whose keys and values exist once
    linear_q4         products of a few rows with 4-bit weights and group scales

Each case is given as plain values; `prepare` makes what a program holds before the call, `run`
makes one pass -- through the library's entry points when `own` is true, in elementary torch
operations when it is false -- and `exact` computes the same outputs in 64 bits from the
operators' definitions.
"""
import importlib
import math
import random

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _library():
    return importlib.import_module("gemma-embed-swift_b200")


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # Eight short search queries at the text encoder's own head layout (3 heads, 1 KV head of
        # 256): the smallest call, where the launches' latency is most of the time.
        dict(name="causal queries", op="causal", dtype="f16", heads=3, kv_heads=1, dim=256, nseq=8, shortest=5, longest=40,
             window=0, fused=True, ragged=11),
        # A document batch: the size and lengths of the benchmark's text batch (64 texts, about
        # 300 tokens each) at a common grouped layout.
        dict(name="causal documents", op="causal", dtype="bf16", heads=32, kv_heads=8, dim=128, nseq=64, shortest=33,
             longest=577, window=0, fused=True, ragged=12),
        # The same kind of batch under the text encoder's layout and its 512-token sliding window,
        # texts up to the encoder's 2048 tokens.
        dict(name="causal sliding window", op="causal", dtype="f16", heads=3, kv_heads=1, dim=256, nseq=48, shortest=300,
             longest=2048, window=512, fused=True, ragged=13),
        # Long documents at 64 wide heads without grouping (the vision tower's head width).
        dict(name="causal long, 64 wide", op="causal", dtype="f16", heads=12, kv_heads=12, dim=64, nseq=3, shortest=5000,
             longest=8191, window=0, fused=False, ragged=14),
        # Four very long documents: bound by the matrix products.
        dict(name="causal long, grouped", op="causal", dtype="bf16", heads=32, kv_heads=8, dim=128, nseq=4, shortest=6001,
             longest=9000, window=0, fused=False, ragged=15),
        # The last token of each text behind a long shared instruction with examples: single-token
        # rows, a long prefix, own keys of a search query's length.
        dict(name="prefix last tokens", op="prefix", dtype="bf16", heads=32, kv_heads=8, dim=128, prefix=4096, nseq=64,
             queries=1, shortest=9, longest=200, ragged=21),
        # Two texts only, at the text encoder's head layout, behind a very long prefix: few rows,
        # so the prefix has to be split over the GPU.
        dict(name="prefix two texts", op="prefix", dtype="f16", heads=3, kv_heads=1, dim=256, prefix=16384, nseq=2, queries=1,
             shortest=70, longest=300, ragged=22),
        # Search queries behind their task's instruction: every token of each query, prefix of an
        # instruction with a few examples.
        dict(name="prefix queries", op="prefix", dtype="f16", heads=16, kv_heads=4, dim=128, prefix=1000, nseq=96, queries=0,
             shortest=4, longest=48, ragged=23),
        # Whole documents behind a shared instruction.
        dict(name="prefix documents", op="prefix", dtype="bf16", heads=32, kv_heads=8, dim=128, prefix=1536, nseq=24, queries=0,
             shortest=100, longest=1100, ragged=24),
        # One row through a projection of the text encoder's width (768 -> gate and up of 1152).
        dict(name="q4 one row, small", op="q4", dtype="f16", rows=1, n=2304, k=768, group=32, mins=False, ragged=31),
        # One row through a large layer: bound by the weights' bytes.
        dict(name="q4 one row, large", op="q4", dtype="f16", rows=1, n=16384, k=8192, group=32, mins=False, ragged=32),
        # A few queries at once through a larger one, scales and minima for groups of 128.
        dict(name="q4 twelve rows", op="q4", dtype="bf16", rows=12, n=28671, k=8192, group=128, mins=True, ragged=33),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["causal", "prefix", "q4"])
    dtype = rng.choice(["f16", "bf16"])
    ragged = rng.randrange(1 << 30)
    if op == "q4":
        group = rng.choice([32, 64, 128])
        return dict(op=op, dtype=dtype, rows=_spread(rng, 1, 64), n=_spread(rng, 1, 28000), k=group * _spread(rng, 1, 8192 // group),
                    group=group, mins=rng.random() < 0.5, ragged=ragged)
    dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8] if dim < 256 else [1, 2, 4])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8] if kv_heads < 8 else [1, 2, 4])
    if op == "causal":
        longest = _spread(rng, 1, 8000)
        shortest = _spread(rng, 1, longest)
        nseq = _spread(rng, 1, max(1, min(200, (24000 if dim < 256 else 12000) // longest)))
        window = rng.choice([0, 0, _spread(rng, 1, 4096)])
        return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, nseq=nseq, shortest=shortest, longest=longest,
                    window=window, fused=rng.random() < 0.5, ragged=ragged)
    longest = _spread(rng, 1, 2000)
    shortest = _spread(rng, 1, longest)
    queries = rng.choice([0, 1, 1, _spread(rng, 1, 16)])
    nseq = _spread(rng, 1, max(1, min(128, 12000 // longest)))
    return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, prefix=_spread(rng, 1, 16384 if queries else 2048),
                nseq=nseq, queries=queries, shortest=shortest, longest=longest, ragged=ragged)


def _lengths(case):
    """The sequences' lengths: the longest once, the others spread between the bounds."""
    rng = random.Random(case["ragged"])
    lens = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["nseq"] - 1)] + [case["longest"]]
    rng.shuffle(lens)
    return lens


def _query_lengths(case, lens):
    """Queries of each sequence: all of its tokens, or its last ones."""
    return [min(n, case["queries"]) if case["queries"] else n for n in lens]


def _ranges(lens):
    out, at = [], 0
    for n in lens:
        out.append((at, n))
        at += n
    return out


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    if case["op"] == "q4":
        n, k, g = case["n"], case["k"], case["group"]
        values = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        # Weights of a trained layer: about 1 / sqrt(k), so a group's step is near 2 / 8 of that.
        step = 0.25 / math.sqrt(k)
        scales = (step * (0.5 + torch.rand((n, k // g), generator=gen, device="cuda"))).to(torch.float16)
        mins = None
        if case["mins"]:
            mins = (-8.0 * scales.float() * (0.9 + 0.2 * torch.rand((n, k // g), generator=gen, device="cuda"))).to(torch.float16)
        state = dict(case=case, x=normal(case["rows"], k), values=values, scales=scales, mins=mins)
        if own:
            state["weight"] = _library().Q4Weight(values, scales, mins)
        return state
    lens = _lengths(case)
    heads, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    total = sum(lens)
    state = dict(case=case, kv_ranges=_ranges(lens), scale=1.0 / math.sqrt(d))
    qlens = lens
    if case["op"] == "causal" and case["fused"]:
        # q, k and v as the column ranges of one projection's rows.
        rows = normal(total, (heads + 2 * kvh) * d)
        state["q"] = rows[:, : heads * d].unflatten(1, (heads, d))
        state["k"] = rows[:, heads * d : (heads + kvh) * d].unflatten(1, (kvh, d))
        state["v"] = rows[:, (heads + kvh) * d :].unflatten(1, (kvh, d))
    else:
        if case["op"] == "prefix":
            qlens = _query_lengths(case, lens)
            state["prefix_k"] = normal(case["prefix"], kvh, d)
            state["prefix_v"] = normal(case["prefix"], kvh, d)
        state["q"] = normal(sum(qlens), heads, d)
        state["k"] = normal(total, kvh, d)
        state["v"] = normal(total, kvh, d)
    state["q_ranges"] = _ranges(qlens)
    # The ranges as the program holds them on the device, (start, length) rows.
    state["kv_seqs"] = torch.tensor(state["kv_ranges"], dtype=torch.int32, device="cuda")
    state["q_seqs"] = torch.tensor(state["q_ranges"], dtype=torch.int32, device="cuda")
    return state


# ------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        lib = _library()
        if case["op"] == "causal":
            return lib.attention_causal(state["q"], state["k"], state["v"], state["q_seqs"], scale=state["scale"],
                                        window=case["window"])
        if case["op"] == "prefix":
            return lib.attention_prefix(state["q"], state["k"], state["v"], state["q_seqs"], state["kv_seqs"], state["prefix_k"],
                                        state["prefix_v"], scale=state["scale"])
        return lib.linear_q4(state["x"], state["weight"])
    if case["op"] == "q4":
        return _plain_q4(state)
    return _plain_attention(state)


def _plain_attention(state):
    case = state["case"]
    window = case.get("window", 0)
    heads, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    group = heads // kvh
    q, k, v = state["q"], state["k"], state["v"]
    prefix = case.get("prefix", 0)
    if prefix:
        pk = state["prefix_k"].float().permute(1, 2, 0)  # [KV][D][P]
        pv = state["prefix_v"].float().permute(1, 0, 2)  # [KV][P][D]
    out = torch.empty((q.shape[0], heads, d), device=q.device, dtype=q.dtype)
    block = 1024  # query rows at a time, so that the scores stay within a few GB
    for (q0, nq), (k0, nk) in zip(state["q_ranges"], state["kv_ranges"]):
        kt = k[k0 : k0 + nk].float().permute(1, 2, 0)
        vt = v[k0 : k0 + nk].float().permute(1, 0, 2)
        if prefix:
            kt = torch.cat([pk, kt], 2)
            vt = torch.cat([pv, vt], 1)
        for b0 in range(0, nq, block):
            n = min(block, nq - b0)
            # Query i of the sequence stands at its key nk - nq + i, behind the prefix.
            at = torch.arange(b0, b0 + n, device=q.device) + (nk - nq)
            qt = q[q0 + b0 : q0 + b0 + n].float().unflatten(1, (kvh, group)).permute(1, 2, 0, 3)  # [KV][G][n][D]
            scores = torch.matmul(qt.reshape(kvh, group * n, d), kt).mul_(state["scale"]).view(kvh, group, n, -1)
            key = torch.arange(-prefix, nk, device=q.device)
            hidden = key[None, :] > at[:, None]
            if window:
                hidden |= key[None, :] <= at[:, None] - window
            scores.masked_fill_(hidden, float("-inf"))
            scores -= scores.amax(-1, keepdim=True)
            scores.exp_()
            total = scores.sum(-1)
            rows = torch.matmul(scores.view(kvh, group * n, -1), vt).view(kvh, group, n, d) / total[..., None]
            out[q0 + b0 : q0 + b0 + n] = rows.permute(2, 0, 1, 3).reshape(n, heads, d).to(out.dtype)
    return out


def _plain_q4(state):
    values, scales, mins = state["values"], state["scales"], state["mins"]
    n, half = values.shape
    q = torch.stack([values & 15, values >> 4], -1).view(n, scales.shape[1], -1).float()
    if mins is None:
        w = (q - 8.0) * scales.float()[..., None]
    else:
        w = q * scales.float()[..., None] + mins.float()[..., None]
    x = state["x"]
    return torch.matmul(x.float(), w.view(n, 2 * half).t()).to(x.dtype)


# ------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "q4":
        x, g = state["x"].double(), case["group"]
        out = torch.empty((case["rows"], case["n"]), device=x.device, dtype=torch.float64)
        step = 4096
        for r in range(0, case["n"], step):
            byte = state["values"][r : r + step].to(torch.int64)
            w = torch.empty((byte.shape[0], case["k"]), device=x.device, dtype=torch.float64)
            w[:, 0::2] = (byte % 16).double()
            w[:, 1::2] = (byte // 16).double()
            s = state["scales"][r : r + step].double().repeat_interleave(g, 1)
            if state["mins"] is None:
                w = (w - 8) * s
            else:
                w = w * s + state["mins"][r : r + step].double().repeat_interleave(g, 1)
            out[:, r : r + step] = x @ w.T
        return out
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    if case["op"] == "prefix":
        pk, pv = state["prefix_k"].double(), state["prefix_v"].double()
    else:
        pk, pv = k[:0], v[:0]
    p, window = pk.shape[0], case.get("window", 0)
    out = torch.zeros(q.shape, device=q.device, dtype=torch.float64)
    for (q0, nq), (k0, nk) in zip(state["q_ranges"], state["kv_ranges"]):
        first = p + nk - nq  # the place of the sequence's first query among prefix and own keys
        for h in range(heads):
            keys = torch.cat([pk[:, h // group], k[k0 : k0 + nk, h // group]])
            vals = torch.cat([pv[:, h // group], v[k0 : k0 + nk, h // group]])
            for b in range(0, nq, 2048):
                e = min(nq, b + 2048)
                lo = max(0, first + b - window + 1) if window else 0
                hi = first + e  # no query of this block sees a key past its own place
                s = q[q0 + b : q0 + e, h] @ keys[lo:hi].T * state["scale"]
                place = torch.arange(first + b, first + e, device=q.device)[:, None]
                key = torch.arange(lo, hi, device=q.device)[None, :]
                seen = key <= place
                if window:
                    seen = seen & (key > place - window)
                out[q0 + b : q0 + e, h] = torch.softmax(s.where(seen, -math.inf), -1) @ vals[lo:hi]
    return out


# ------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "q4":
        n, k, r = case["n"], case["k"], case["rows"]
        groups = n * (k // case["group"])
        return {"bytes": n * k // 2 + 2 * groups * (2 if case["mins"] else 1) + 2 * r * (k + n), "flops": 2 * r * n * k}
    lens = _lengths(case)
    heads, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    qlens = _query_lengths(case, lens) if case["op"] == "prefix" else lens
    prefix, window = case.get("prefix", 0), case.get("window", 0)
    pairs = 0
    for nq, nk in zip(qlens, lens):
        if window and window < nk:
            pairs += window * (window + 1) // 2 + (nk - window) * window
        else:
            pairs += nq * prefix + nq * nk - nq * (nq - 1) // 2
    return {"bytes": 2 * d * (2 * heads * sum(qlens) + 2 * kvh * (sum(lens) + prefix)), "flops": 4 * d * heads * pairs}
