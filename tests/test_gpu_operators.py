"""The operators on device tensors (attention_causal, attention_prefix, linear_q4) on a B200, against
64-bit references (operator_reference.py): lengths from none to long, ragged and odd sizes, strides,
masks that leave rows empty, what masked places hold, streams and CUDA graphs."""
import math

import numpy as np
import pytest

import operator_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = ["f16", "bf16"]


@pytest.fixture(scope="module")
def torch(cuda_device):
    import torch
    return torch


def dt(torch, name):
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def normal(torch, seed, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt(torch, dtype))


def ranges(lens, gap=0):
    out, at = [], 0
    for n in lens:
        out.append((at, n))
        at += n + gap
    return out


def dev(torch, r):
    return torch.tensor(r if len(r) else np.zeros((0, 2)), dtype=torch.int32, device="cuda").reshape(-1, 2)


def check_causal(ge, torch, lens, heads, kvh, dim, dtype, window=0, scale=None, seed=1, gap=0, fused=True):
    r = ranges(lens, gap)
    total = sum(lens) + gap * len(lens)
    if fused:
        rows = normal(torch, seed, (total, (heads + 2 * kvh) * dim), dtype)
        q = rows[:, :heads * dim].unflatten(1, (heads, dim))
        k = rows[:, heads * dim:(heads + kvh) * dim].unflatten(1, (kvh, dim))
        v = rows[:, (heads + kvh) * dim:].unflatten(1, (kvh, dim))
    else:
        q, k, v = (normal(torch, seed + i, (total, h, dim), dtype) for i, h in enumerate((heads, kvh, kvh)))
    out = torch.full((total, heads, dim), 7.0, dtype=q.dtype, device="cuda")
    got = ge.attention_causal(q, k, v, dev(torch, r), scale=scale, window=window, out=out)
    assert got is out
    want, bound, touched = ref.attention(q, k, v, r, r, 1 / math.sqrt(dim) if scale is None else scale, window)
    ref.check(out[touched], want[touched], bound[touched])
    assert (out[~touched] == 7.0).all()  # rows of no sequence stay as they were


HEADS = [(1, 1, 64), (12, 12, 64), (4, 1, 64), (3, 1, 256), (8, 2, 128), (6, 2, 128), (2, 2, 256), (14, 2, 128), (8, 1, 256),
         (5, 5, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,dim", HEADS)
@pytest.mark.parametrize("lens", [[1], [2, 1, 3], [127, 128, 129, 1, 64, 65], [0, 5, 0, 300, 17, 0], [700]])
def test_causal_lengths(ge, torch, heads, kvh, dim, dtype, lens):
    check_causal(ge, torch, lens, heads, kvh, dim, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,dim", [(3, 1, 256), (8, 2, 128), (2, 2, 64)])
@pytest.mark.parametrize("window", [1, 2, 63, 128, 200, 5000, 2**31 - 1])
def test_causal_window(ge, torch, heads, kvh, dim, dtype, window):
    check_causal(ge, torch, [1, 130, 300, 77, 513], heads, kvh, dim, dtype, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_causal_gaps_and_dense_rows(ge, torch, dtype):
    check_causal(ge, torch, [40, 1, 200], 8, 2, 128, dtype, gap=9, fused=False)
    check_causal(ge, torch, [40, 0, 200], 3, 1, 256, dtype, gap=3)


@pytest.mark.parametrize("heads,kvh,dim", [(128, 1, 64), (100, 1, 64), (33, 1, 128), (64, 4, 64)])
def test_causal_many_heads_to_a_kv_head(ge, torch, heads, kvh, dim):
    check_causal(ge, torch, [3, 70, 150], heads, kvh, dim, "f16")


@pytest.mark.parametrize("heads,kvh,dim", [(8, 2, 128), (3, 1, 256), (4, 4, 64)])
def test_causal_many_sequences(ge, torch, heads, kvh, dim):
    lens = [int(n) for n in np.random.default_rng(5).integers(0, 90, 400)]
    check_causal(ge, torch, lens, heads, kvh, dim, "bf16")


@pytest.mark.parametrize("heads,kvh,dim,n", [(8, 2, 128, 3001), (3, 1, 256, 2049), (4, 4, 64, 4097), (1, 1, 128, 6000)])
def test_causal_long(ge, torch, heads, kvh, dim, n):
    check_causal(ge, torch, [n, 33], heads, kvh, dim, "f16", fused=False)


@pytest.mark.parametrize("scale", [1e-4, 0.125, 3.0])
def test_causal_scales(ge, torch, scale):
    """From nearly uniform weights to weights on one key."""
    check_causal(ge, torch, [200, 31], 8, 2, 128, "bf16", scale=scale)
    check_causal(ge, torch, [200, 31], 3, 1, 256, "f16", scale=scale)


@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256)])
def test_causal_growing_scores(ge, torch, heads, kvh, dim):
    """Every key scores higher than all before it, so a running maximum moves at every step."""
    n = 600
    q = torch.full((n, heads, dim), 0.5, dtype=torch.float16, device="cuda")
    k = (torch.arange(n, device="cuda", dtype=torch.float32)[:, None, None] * 0.02).expand(n, kvh, dim).half().contiguous()
    v = normal(torch, 3, (n, kvh, dim), "f16")
    r = [(0, n)]
    got = ge.attention_causal(q, k, v, dev(torch, r), scale=0.2)
    want, bound, _ = ref.attention(q, k, v, r, r, 0.2)
    ref.check(got, want, bound)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256)])
def test_causal_ignores_what_masked_places_hold(ge, torch, heads, kvh, dim, bad):
    """Rows of no sequence, other sequences and later tokens may hold anything."""
    q, k, v = (normal(torch, 4 + i, (260, h, dim), "f16") for i, h in enumerate((heads, kvh, kvh)))
    r = [(3, 90), (100, 97), (197, 50)]
    want, bound, touched = ref.attention(q, k, v, r, r, 1 / math.sqrt(dim))
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[:3] = bad          # before the first
        t[93:100] = bad      # between two
        t[247:] = bad        # behind the last
        t[196] = bad         # the last token of the second sequence: its own row alone sees it
        t[92, 0, 5] = bad    # one value of the first sequence's last token
    got = ge.attention_causal(q, k2, v2, dev(torch, r))
    clean = touched.clone()
    clean[196] = clean[92] = False
    ref.check(got[clean], want[clean], bound[clean])


def test_causal_nan_reaches_the_rows_that_see_it(ge, torch):
    q, k, v = (normal(torch, 14 + i, (200, h, 128), "bf16") for i, h in enumerate((4, 1, 1)))
    v[70, 0, 9] = float("nan")
    r = [(0, 200)]
    got = ge.attention_causal(q, k, v, dev(torch, r))
    assert not torch.isnan(got[:70]).any()
    assert torch.isnan(got[70:, :, 9]).all()
    rest = torch.ones(128, dtype=torch.bool, device="cuda")
    rest[9] = False
    assert not torch.isnan(got[:, :, rest]).any()


def test_causal_lowest_and_highest_values(ge, torch):
    """Scores at the types' limits: one key far above all others, products that overflow 16 bits."""
    q, k, v = (normal(torch, 24 + i, (150, h, 64), "f16") for i, h in enumerate((2, 1, 1)))
    k[40] = 60000.0
    k[41] = -65504.0
    v[40] = 65504.0
    v[41] = -65504.0
    r = [(0, 150)]
    got = ge.attention_causal(q, k, v, dev(torch, r), scale=1e-6)
    want, bound, _ = ref.attention(q, k, v, r, r, 1e-6)
    ref.check(got, want, bound)


def prefix_case(torch, plen, qlens, klens, heads, kvh, dim, dtype, seed=1, order=None, gap=0):
    qr = ranges(qlens)
    kr = ranges(klens, gap)
    if order is not None:
        by = [kr[i] for i in order]
        kr = by
    nkv = max([s + n for s, n in kr] + [0]) + gap
    q = normal(torch, seed, (sum(qlens), heads, dim), dtype)
    k, v = normal(torch, seed + 1, (nkv, kvh, dim), dtype), normal(torch, seed + 2, (nkv, kvh, dim), dtype)
    pk, pv = normal(torch, seed + 3, (plen, kvh, dim), dtype), normal(torch, seed + 4, (plen, kvh, dim), dtype)
    return q, k, v, qr, kr, pk, pv


def check_prefix(ge, torch, *args, **kw):
    q, k, v, qr, kr, pk, pv = prefix_case(torch, *args, **kw)
    scale = 1 / math.sqrt(q.shape[2])
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv, out=out)
    want, bound, touched = ref.attention(q, k, v, qr, kr, scale, prefix_k=pk, prefix_v=pv)
    ref.check(out[touched], want[touched], bound[touched])
    assert (out[~touched] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,dim", HEADS)
@pytest.mark.parametrize("plen", [0, 1, 129, 1000])
def test_prefix_single_tokens(ge, torch, heads, kvh, dim, dtype, plen):
    check_prefix(ge, torch, plen, [1] * 9, [1, 5, 128, 129, 31, 0, 300, 64, 2], heads, kvh, dim, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,dim", [(8, 2, 128), (3, 1, 256), (4, 4, 64), (7, 1, 64)])
@pytest.mark.parametrize("qlens,klens", [([5, 130, 64], [5, 130, 64]), ([3, 0, 40, 1], [10, 7, 45, 0]), ([200], [257]),
                                         ([6, 4], [3, 0])])  # the last: more queries than keys
def test_prefix_texts(ge, torch, heads, kvh, dim, dtype, qlens, klens):
    for plen in (0, 200):
        check_prefix(ge, torch, plen, qlens, klens, heads, kvh, dim, dtype)


@pytest.mark.parametrize("heads,kvh,dim", [(3, 1, 256), (8, 2, 128), (2, 1, 64)])
@pytest.mark.parametrize("plen,n", [(8000, 1), (4097, 3), (130, 2), (0, 2)])
def test_prefix_few_rows_long(ge, torch, heads, kvh, dim, plen, n):
    """Few query rows before many keys: the work is split over the keys."""
    check_prefix(ge, torch, plen, [1] * n, [2500 + 700 * i for i in range(n)], heads, kvh, dim, "bf16")


@pytest.mark.parametrize("gap", [0, 50])
@pytest.mark.parametrize("heads,kvh,dim", [(8, 2, 128), (3, 1, 256)])
def test_prefix_key_ranges_in_any_order(ge, torch, heads, kvh, dim, gap):
    n = 40
    klens = [int(x) for x in np.random.default_rng(3).integers(0, 120, n)]
    order = [int(i) for i in np.random.default_rng(4).permutation(n)]
    check_prefix(ge, torch, 300, [1] * n, klens, heads, kvh, dim, "f16", order=order, gap=gap)
    check_prefix(ge, torch, 300, [1] * n, klens, heads, kvh, dim, "f16", gap=gap)


def test_prefix_shared_key_range(ge, torch):
    """The same key range named by several sequences, one of them empty."""
    q, k, v, qr, kr, pk, pv = prefix_case(torch, 70, [2, 3, 1, 4], [90, 20, 5, 60], 8, 2, 128, "bf16")
    kr = [kr[0], kr[0], (0, 0), kr[0]]
    got = ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv)
    want, bound, _ = ref.attention(q, k, v, qr, kr, 1 / math.sqrt(128), prefix_k=pk, prefix_v=pv)
    ref.check(got, want, bound)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prefix_cache_slots_hold_anything_past_their_ranges(ge, torch, dim, bad):
    """Fixed slots of a cache, each filled in part: what lies behind a slot's keys does not matter."""
    lens = [1, 40, 100, 0, 64, 13]
    slot = 100
    kr = [(slot * i, n) for i, n in enumerate(lens)]
    q = normal(torch, 1, (len(lens), 4, dim), "f16")
    k, v = normal(torch, 2, (slot * len(lens), 2, dim), "f16"), normal(torch, 3, (slot * len(lens), 2, dim), "f16")
    pk, pv = normal(torch, 4, (130, 2, dim), "f16"), normal(torch, 5, (130, 2, dim), "f16")
    qr = [(i, 1) for i in range(len(lens))]
    want, bound, _ = ref.attention(q, k, v, qr, kr, 1 / math.sqrt(dim), prefix_k=pk, prefix_v=pv)
    for s, n in kr:
        k[s + n:s + slot] = bad
        v[s + n:s + slot] = bad
    got = ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv)
    ref.check(got, want, bound)


def test_ranges_outside_the_tensors_are_cut(ge, torch):
    q, k, v = (normal(torch, 5 + i, (50, h, 64), "f16") for i, h in enumerate((2, 1, 1)))
    out = torch.full_like(q, 7.0)
    ge.attention_causal(q, k, v, dev(torch, [(0, 20), (30, 1000), (50, 4), (-3, 2), (1 << 30, 5)]), out=out)
    r = [(0, 20), (30, 20)]
    want, bound, touched = ref.attention(q, k, v, r, r, 0.125)
    ref.check(out[:20], want[:20], bound[:20])
    assert (out[20:30] == 7.0).all()
    assert not torch.isnan(out[30:]).any()


def test_prefix_equals_causal_of_the_whole_text(ge, torch):
    """The prompt attention makes the prefix' rows and the texts' together; behind the shared prefix the
    texts' rows are the same within both bounds."""
    heads, kvh, dim, plen = 8, 2, 128, 333
    lens = [17, 128, 1, 60]
    q, k, v, qr, kr, pk, pv = prefix_case(torch, plen, lens, lens, heads, kvh, dim, "bf16")
    got = ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv)
    want, bound, _ = ref.attention(q, k, v, qr, kr, 1 / math.sqrt(dim), prefix_k=pk, prefix_v=pv)
    ref.check(got, want, bound)
    pq = normal(torch, 77, (plen, heads, dim), "bf16")
    for (s, n) in qr:
        whole = ge.attention_causal(torch.cat([pq, q[s:s + n]]), torch.cat([pk, k[s:s + n]]), torch.cat([pv, v[s:s + n]]),
                                    dev(torch, [(0, plen + n)]))
        err = (whole[plen:].double() - got[s:s + n].double()).abs()
        assert (err <= 2 * bound[s:s + n]).all()


def test_attention_across_32_bit_offsets(ge, torch):
    """Key rows whose element offsets pass 2^31: a wide cache row of which the call reads some columns."""
    width, rows = 1 << 16, 33000  # 4.3 GB of fp16
    cache = torch.empty((rows, width), dtype=torch.float16, device="cuda")
    k = cache[:, :128].unflatten(1, (1, 128))
    v = cache[:, width - 128:].unflatten(1, (1, 128))
    k[rows - 400:] = normal(torch, 1, (400, 1, 128), "f16")
    v[rows - 400:] = normal(torch, 2, (400, 1, 128), "f16")
    q = normal(torch, 3, (3, 4, 128), "f16")
    empty = torch.empty((0, 1, 128), dtype=torch.float16, device="cuda")
    qr, kr = [(0, 3)], [(rows - 400, 400)]
    got = ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), empty, empty)
    want, bound, _ = ref.attention(q, k[rows - 400:].contiguous(), v[rows - 400:].contiguous(), qr, [(0, 400)], 1 / math.sqrt(128))
    ref.check(got, want, bound)


# ---------------------------------------------------------------------------- 4-bit products
def q4(torch, ge, n, k, group, mins, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    values = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((n, k // group), generator=g, device="cuda") * 0.02 + 1e-3).half()
    lows = (torch.randn((n, k // group), generator=g, device="cuda") * 0.05).half() if mins else None
    return ge.Q4Weight(values, scales, lows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,units", [(1, 1, 1), (1, 777, 6), (2, 64, 3), (5, 300, 7), (8, 129, 16), (9, 1000, 5), (16, 17, 33),
                                          (17, 255, 9), (33, 130, 4), (64, 515, 11)])
def test_linear_q4(ge, torch, dtype, mins, group, rows, n, units):
    k = group * units
    w = q4(torch, ge, n, k, group, mins, seed=rows + n)
    x = normal(torch, rows, (rows, k), dtype)
    out = torch.full((rows, n + 5), 7.0, dtype=x.dtype, device="cuda")
    got = ge.linear_q4(x, w, out=out[:, :n])
    want, bound = ref.linear_q4(x, w.values, w.scales, w.mins)
    ref.check(got, want, bound)
    assert (out[:, n:] == 7.0).all()


@pytest.mark.parametrize("rows", [1, 12, 40])
def test_linear_q4_large(ge, torch, rows):
    w = q4(torch, ge, 5003, 8192, 32, False)
    x = normal(torch, 3, (rows, 8192), "bf16")
    want, bound = ref.linear_q4(x, w.values, w.scales, w.mins)
    ref.check(ge.linear_q4(x, w), want, bound)
    w = q4(torch, ge, 300, 65536, 64, True)
    x = normal(torch, 4, (rows, 65536), "f16", 0.1)
    want, bound = ref.linear_q4(x, w.values, w.scales, w.mins)
    ref.check(ge.linear_q4(x, w), want, bound)


def test_linear_q4_strided_rows(ge, torch):
    w = q4(torch, ge, 96, 256, 32, True)
    x = normal(torch, 5, (6, 1024), "f16")[:, 512:768]
    want, bound = ref.linear_q4(x, w.values, w.scales, w.mins)
    ref.check(ge.linear_q4(x, w), want, bound)


@pytest.mark.parametrize("kind", ["Q4_0", "Q4_1"])
def test_linear_q4_from_gguf_blocks(ge, torch, kind):
    n, k = 70, 160
    rng = np.random.default_rng(8)
    per = 20 if kind == "Q4_1" else 18
    blocks = rng.integers(0, 256, (n, k // 32, per), dtype=np.uint8)
    half = lambda a: np.ascontiguousarray(a.astype(np.float16)).view(np.uint8).reshape(n, k // 32, 2)
    d, m = rng.uniform(0.01, 0.02, (n, k // 32)), rng.uniform(-0.1, 0.1, (n, k // 32))
    blocks[..., :2] = half(d)
    if kind == "Q4_1":
        blocks[..., 2:4] = half(m)
    w = ge.Q4Weight.from_blocks(blocks.tobytes(), kind, n, k)
    q = blocks[..., per - 16:]
    q = np.concatenate([q & 15, q >> 4], -1).astype(np.float64)  # element j: low half of byte j, then the high halves
    d, m = d.astype(np.float16).astype(np.float64)[..., None], m.astype(np.float16).astype(np.float64)[..., None]
    dense = ((q - 8) * d if kind == "Q4_0" else q * d + m).reshape(n, k)
    x = normal(torch, 9, (3, k), "f16")
    want = x.double() @ torch.from_numpy(dense).cuda().T
    _, bound = ref.linear_q4(x, w.values, w.scales, w.mins)
    ref.check(ge.linear_q4(x, w), want, bound)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_linear_q4_rows_stay_apart(ge, torch, bad):
    """A row that holds NaN or infinities leaves the other rows as they are, bit for bit."""
    w = q4(torch, ge, 200, 512, 64, True)
    x = normal(torch, 6, (5, 512), "bf16")
    clean = ge.linear_q4(x, w)
    x[2, 100] = bad
    got = ge.linear_q4(x, w)
    keep = [0, 1, 3, 4]
    assert torch.equal(got[keep], clean[keep])
    assert not torch.isfinite(got[2]).any()


# ---------------------------------------------------------------------------- together, streams, graphs
def layer(ge, torch, x, wq, wk, wv, wo, seqs, kv_seqs, pk, pv, heads, kvh, dim):
    q = ge.linear_q4(x, wq).unflatten(1, (heads, dim))
    k = ge.linear_q4(x, wk).unflatten(1, (kvh, dim))
    v = ge.linear_q4(x, wv).unflatten(1, (kvh, dim))
    o = ge.attention_prefix(q, k, v, seqs, kv_seqs, pk, pv)
    return ge.linear_q4(o.flatten(1), wo)


def layer_inputs(ge, torch, dtype="f16"):
    heads, kvh, dim, hidden = 8, 2, 64, 256
    r = ranges([9, 1, 14])
    x = normal(torch, 1, (24, hidden), dtype)
    ws = [q4(torch, ge, n, k, 32, False, seed=i) for i, (n, k) in
          enumerate([(heads * dim, hidden), (kvh * dim, hidden), (kvh * dim, hidden), (hidden, heads * dim)])]
    pq, pk, pv = (normal(torch, 5 + i, (90, h, dim), dtype) for i, h in enumerate((heads, kvh, kvh)))
    return x, ws, dev(torch, r), r, pq, pk, pv, (heads, kvh, dim)


def test_a_causal_layer_of_queries(ge, torch):
    """An instruction's prompt attention once, then short queries behind it through 4-bit projections: every
    step against its own 64-bit reference on the same inputs."""
    x, ws, seqs, r, pq, pk, pv, (heads, kvh, dim) = layer_inputs(ge, torch)
    whole = [(0, 90)]
    po = ge.attention_causal(pq, pk, pv, dev(torch, whole))
    want, bound, _ = ref.attention(pq, pk, pv, whole, whole, 1 / math.sqrt(dim))
    ref.check(po, want, bound)
    qkv = []
    for w in ws[:3]:
        y = ge.linear_q4(x, w)
        want, bound = ref.linear_q4(x, w.values, w.scales, w.mins)
        ref.check(y, want, bound)
        qkv.append(y.unflatten(1, (-1, dim)))
    o = ge.attention_prefix(*qkv, seqs, seqs, pk, pv)
    want, bound, _ = ref.attention(*qkv, r, r, 1 / math.sqrt(dim), prefix_k=pk, prefix_v=pv)
    ref.check(o, want, bound)
    y = ge.linear_q4(o.flatten(1), ws[3])
    want, bound = ref.linear_q4(o.flatten(1), ws[3].values, ws[3].scales, None)
    ref.check(y, want, bound)
    assert torch.equal(y, layer(ge, torch, x, *ws, seqs, seqs, pk, pv, heads, kvh, dim))


def test_streams_and_graphs(ge, torch):
    """The same bits on another stream, by a raw handle, and from two captured graphs replayed at once;
    a replay reads what its inputs hold then, new lengths among it."""
    x, ws, seqs, r, pq, pk, pv, hkd = layer_inputs(ge, torch)
    first = layer(ge, torch, x, *ws, seqs, seqs, pk, pv, *hkd)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = ge.linear_q4(x, ws[0], stream=side)
    raw = ge.linear_q4(x, ws[0], stream=side.cuda_stream)
    q = out.unflatten(1, (hkd[0], hkd[2]))
    side.synchronize()
    assert torch.equal(out, ge.linear_q4(x, ws[0])) and torch.equal(raw, out)
    k = normal(torch, 8, (24, hkd[1], hkd[2]), "f16")
    a = ge.attention_causal(q, k, k, seqs)
    torch.cuda.synchronize()
    b = ge.attention_causal(q, k, k, seqs, stream=side)
    side.synchronize()
    assert torch.equal(a, b)
    graphs, outs = [], []
    ranges_dev = seqs.clone()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(ge, torch, x, *ws, ranges_dev, ranges_dev, pk, pv, *hkd))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    ranges_dev.copy_(dev(torch, [(0, 2), (2, 20), (22, 2)]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], layer(ge, torch, x, *ws, ranges_dev, ranges_dev, pk, pv, *hkd))


def test_runs_repeat_bit_for_bit(ge, torch):
    q, k, v, qr, kr, pk, pv = prefix_case(torch, 5000, [1] * 20, [100 + 9 * i for i in range(20)], 8, 2, 128, "bf16")
    a = ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv)
    for _ in range(5):
        assert torch.equal(a, ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv))


def test_wrappers_refuse_what_does_not_fit(ge, torch):
    z = lambda *s, d=torch.float16: torch.zeros(s, dtype=d, device="cuda")
    q, k, s = z(8, 4, 64), z(8, 2, 64), z(1, 2, d=torch.int32)
    w = ge.Q4Weight(z(8, 32, d=torch.uint8), z(8, 2))
    bad = [
        lambda: ge.attention_causal(q, k, z(8, 1, 64), s),
        lambda: ge.attention_causal(q, z(7, 2, 64), z(7, 2, 64), s),
        lambda: ge.attention_causal(q, k, z(8, 2, 64, d=torch.bfloat16), s),
        lambda: ge.attention_causal(q.float(), k.float(), k.float(), s),
        lambda: ge.attention_causal(q, k, k, s.long()),
        lambda: ge.attention_causal(q, k, k, z(2, d=torch.int32)),
        lambda: ge.attention_causal(q, k, k, s.cpu()),
        lambda: ge.attention_causal(q.transpose(0, 1).contiguous().transpose(0, 1), k, k, s),
        lambda: ge.attention_causal(z(8, 4, 96), z(8, 2, 96), z(8, 2, 96), s),
        lambda: ge.attention_causal(q, k, k, s, out=z(8, 4, 128)),
        lambda: ge.attention_causal(q, k, k, s, scale=-1.0),
        lambda: ge.attention_causal(q, k, k, s, window=-1),
        lambda: ge.attention_causal(z(1, 4, 64).expand(8, 4, 64), k, k, s),
        lambda: ge.attention_prefix(q, k, k, s, z(2, 2, d=torch.int32), k, k),
        lambda: ge.attention_prefix(q, k, k, s, s, k, z(7, 2, 64)),
        lambda: ge.attention_prefix(q, k, k, s, s, z(8, 4, 64), z(8, 4, 64)),
        lambda: ge.linear_q4(z(2, 32), w),
        lambda: ge.linear_q4(z(65, 64), w),
        lambda: ge.linear_q4(z(64, 2).t(), w),
        lambda: ge.linear_q4(z(2, 64), w, out=z(2, 9)),
        lambda: ge.linear_q4(z(2 * 64 + 1)[1:].view(2, 64), w),
        lambda: ge.Q4Weight(z(8, 32, d=torch.uint8), z(8, 3)),
        lambda: ge.Q4Weight(z(8, 32, d=torch.uint8), z(8, 2), z(8, 1)),
        lambda: ge.Q4Weight(z(8, 32), z(8, 2)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ge.GemmaEmbedError) as e:
            call()
        assert e.value.case == "invalidOptions", i
    assert ge.attention_causal(z(0, 4, 64), z(0, 2, 64), z(0, 2, 64), s).shape == (0, 4, 64)
    assert ge.linear_q4(z(0, 64), w).shape == (0, 8)


def test_another_device_than_the_current_one(ge, torch):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    q = torch.randn(9, 4, 64, device="cuda:1").half()
    k = torch.randn(9, 2, 64, device="cuda:1").half()
    s = torch.tensor([[0, 9]], dtype=torch.int32, device="cuda:1")
    with torch.cuda.device(0):
        got = ge.attention_causal(q, k, k, s)
        assert torch.cuda.current_device() == 0
    want, bound, _ = ref.attention(q, k, k, [(0, 9)], [(0, 9)], 0.125)
    ref.check(got, want, bound)


@pytest.mark.parametrize("seqs", [[(40, 8)], [(0, 0)], [(100, 28), (100, 28)], [(0, 128), (5, 3), (60, 10)], [(64, 900)]])
def test_rows_of_no_sequence_and_shared_rows(ge, torch, seqs):
    """Most rows in no sequence, and ranges that share rows: no row outside every range is touched, rows of one
    range alone are right (shared ones are unspecified)."""
    q, k, v = (normal(torch, 31 + i, (1000, h, 64), "f16") for i, h in enumerate((2, 1, 1)))
    out = torch.full_like(q, 7.0)
    ge.attention_causal(q, k, v, dev(torch, seqs), out=out)
    cover = torch.zeros(1000, dtype=torch.int32, device="cuda")
    for s, n in seqs:
        cover[s:s + n] += 1
    assert (out[cover == 0] == 7.0).all()
    if (cover < 2).all():
        want, bound, touched = ref.attention(q, k, v, seqs, seqs, 0.125)
        ref.check(out[touched], want[touched], bound[touched])


def test_causal_more_sequences_than_the_plan_holds_in_one_cta(ge, torch):
    """Thousands of short sequences (their plan is a cluster's), some of them empty, among long ones."""
    lens = [int(n) for n in np.random.default_rng(6).integers(0, 12, 6000)]
    lens[100] = 900
    lens[4000] = 300
    check_causal(ge, torch, lens, 4, 2, 64, "f16")
    check_causal(ge, torch, lens, 2, 1, 256, "bf16", window=5)


@pytest.mark.parametrize("heads,kvh,dim", [(8, 2, 128), (3, 1, 256), (2, 2, 64)])
def test_prefix_scattered_slots(ge, torch, heads, kvh, dim):
    """A few sequences in a cache of many slots, in no order: the keys between them are no row's."""
    rng = np.random.default_rng(12)
    slot, slots, used = 640, 64, 23
    klens = [int(x) for x in rng.integers(0, 200, used)]
    qlens = [int(x) for x in rng.integers(0, 4, used)]
    kr = [(int(s) * slot, n) for s, n in zip(rng.permutation(slots)[:used], klens)]
    qr = ranges(qlens)
    q = normal(torch, 1, (sum(qlens), heads, dim), "bf16")
    k, v = (torch.full((slots * slot, kvh, dim), float("nan"), dtype=q.dtype, device="cuda") for _ in range(2))
    for i, (s, n) in enumerate(kr):
        k[s:s + n], v[s:s + n] = normal(torch, 100 + i, (n, kvh, dim), "bf16"), normal(torch, 200 + i, (n, kvh, dim), "bf16")
    pk, pv = normal(torch, 4, (77, kvh, dim), "bf16"), normal(torch, 5, (77, kvh, dim), "bf16")
    got = ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv)
    want, bound, _ = ref.attention(q, k, v, qr, kr, 1 / math.sqrt(dim), prefix_k=pk, prefix_v=pv)
    ref.check(got, want, bound)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_small_probabilities_keep_their_sum(ge, torch, dim):
    """One key far above all the others, whose value is 0: fp16 outputs are the sum of hundreds of
    probabilities of 2^-24.6, held to 2^-24 in steps of 2^-31."""
    n = 512
    q, k, v = (torch.zeros((n, 1, dim), dtype=torch.float16, device="cuda") for _ in range(3))
    q[:, :, 0] = 1.0
    k[1:, :, 0] = -17.05
    v[1:] = 16.0
    got = ge.attention_causal(q, k, v, dev(torch, [(0, n)]), scale=1.0).double()
    want, _, _ = ref.attention(q, k, v, [(0, n)], [(0, n)], 1.0)
    # Half a step of a probability below fp16's normal range, 2^-25 / 2^7, relative to 2^-24.6; exponentials and
    # sums (2^-18); the result's own half step, relative and below the normal range.
    bound = want * (2.0 ** -(25 + 7 - 24.6) + 2.0 ** -18 + 2.0 ** -11) + 2.0 ** -25
    ref.check(got, want, bound)


@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256)])
def test_an_infinite_value_every_row_sees(ge, torch, heads, kvh, dim):
    """Every row is recomputed; its other columns are as without it."""
    n = 3000
    q, k, v = (normal(torch, 40 + i, (n, h, dim), "f16") for i, h in enumerate((heads, kvh, kvh)))
    v[0, :, 3] = float("inf")
    got = ge.attention_causal(q, k, v, dev(torch, [(0, n)]))
    want, bound, _ = ref.attention(q, k, v, [(0, n)], [(0, n)], 1 / math.sqrt(dim))
    assert not torch.isfinite(got[:, :, 3]).any()
    keep = [i for i in range(dim) if i != 3]
    ref.check(got[..., keep], want[..., keep], bound[..., keep])


def test_inputs_dropped_while_another_stream_reads_them(ge, torch):
    """Memory of inputs that were dropped after the call is not given out again before its work is done."""
    q, k, v = (normal(torch, 50 + i, (700, h, 128), "bf16") for i, h in enumerate((8, 2, 2)))
    s = dev(torch, [(0, 700)])
    w = q4(torch, ge, 600, 512, 32, False)
    x = normal(torch, 9, (4, 512), "f16")
    want, y = ge.attention_causal(q, k, v, s), ge.linear_q4(x, w)
    side = torch.cuda.Stream()
    a, b, c, d, e = q.clone(), k.clone(), v.clone(), s.clone(), x.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    got = ge.attention_causal(a, b, c, d, stream=side)
    z = ge.linear_q4(e, w, stream=side)
    del a, b, c, d, e
    junk = [torch.full_like(t, 7) for t in (q, k, v, s, x) for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(z, y)
    del junk


def test_inputs_that_require_a_gradient_are_refused(ge, torch):
    q, k, s = normal(torch, 1, (8, 4, 64), "f16"), normal(torch, 2, (8, 2, 64), "f16"), dev(torch, [(0, 8)])
    w = q4(torch, ge, 8, 64, 32, False)
    want = ge.attention_causal(q, k, k, s)
    x = q.flatten(1)[:, :64].contiguous()
    y = ge.linear_q4(x, w)
    q.requires_grad_()
    x.requires_grad_()
    for call in (lambda: ge.attention_causal(q, k, k, s), lambda: ge.attention_prefix(q, k, k, s, s, k, k), lambda: ge.linear_q4(x, w)):
        with pytest.raises(ge.GemmaEmbedError) as e:
            call()
        assert e.value.case == "invalidOptions"
    with torch.no_grad():
        assert torch.equal(ge.attention_causal(q, k, k, s), want) and torch.equal(ge.linear_q4(x, w), y)


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("rows", [3, 20])
def test_linear_q4_wide(ge, torch, rows, mins):
    """More output columns than the SMs hold at once."""
    w = q4(torch, ge, 41003, 320, 32, mins)
    x = normal(torch, 11, (rows, 320), "bf16")
    want, bound = ref.linear_q4(x, w.values, w.scales, w.mins)
    ref.check(ge.linear_q4(x, w), want, bound)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_linear_q4_scales_off_16_bytes(ge, torch, group):
    n, k = 301, 1024
    w = q4(torch, ge, n, k, group, True)
    off = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
    x = normal(torch, 12, (6, k), "f16")
    want = ge.linear_q4(x, w)
    assert torch.equal(ge.linear_q4(x, ge.Q4Weight(w.values, off(w.scales), w.mins)), want)
    assert torch.equal(ge.linear_q4(x, ge.Q4Weight(w.values, w.scales, off(w.mins))), want)


@pytest.mark.parametrize("offset,extra", [(8, 0), (0, 8), (16, 16)])
def test_outputs_in_wider_rows(ge, torch, offset, extra):
    """Rows of `out` on 16- and on 32-byte boundaries, beside columns that stay as they are."""
    heads, kvh, dim, n = 4, 2, 64, 150
    q, k, v = (normal(torch, 60 + i, (n, h, dim), "f16") for i, h in enumerate((heads, kvh, kvh)))
    wide = torch.full((n, heads * dim + 32 + extra), 7.0, dtype=q.dtype, device="cuda")
    out = wide[:, offset:offset + heads * dim].unflatten(1, (heads, dim))
    ge.attention_causal(q, k, v, dev(torch, [(0, n)]), out=out)
    want, bound, _ = ref.attention(q, k, v, [(0, n)], [(0, n)], 0.125)
    ref.check(out, want, bound)
    assert (wide[:, :offset] == 7.0).all() and (wide[:, offset + heads * dim:] == 7.0).all()


@pytest.mark.parametrize("heads,kvh", [(1, 1), (16, 1), (32, 1), (64, 1), (128, 1), (64, 2), (12, 2)])
@pytest.mark.parametrize("gap", [0, 3])
def test_causal_128_wide_outputs(ge, torch, heads, kvh, gap):
    """Every way a warp's rows may lie in `out`: tokens with all their heads, parts of a token's heads, rows of
    no sequence among them, a last tile that ends inside."""
    check_causal(ge, torch, [40, 1, 130, 7], heads, kvh, 128, "bf16", gap=gap)


def test_outputs_and_scales_that_require_a_gradient_are_refused(ge, torch):
    w = q4(torch, ge, 8, 64, 32, True)
    x = normal(torch, 1, (2, 64), "f16")
    q, k, s = normal(torch, 1, (8, 4, 64), "f16"), normal(torch, 2, (8, 2, 64), "f16"), dev(torch, [(0, 8)])
    grad = lambda t: t.detach().clone().requires_grad_()
    for call in (lambda: ge.linear_q4(x, w, out=grad(normal(torch, 2, (2, 8), "f16"))),
                 lambda: ge.Q4Weight(w.values, grad(w.scales), w.mins), lambda: ge.Q4Weight(w.values, w.scales, grad(w.mins)),
                 lambda: ge.attention_causal(q, k, k, s, out=grad(q))):
        with pytest.raises(ge.GemmaEmbedError) as e:
            call()
        assert e.value.case == "invalidOptions"
