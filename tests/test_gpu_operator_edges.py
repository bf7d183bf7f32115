"""The operators on device tensors at the edges of what their calls allow, on a B200: infinities and sums past
the types, and what a caller relies on around a call."""
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import operator_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(cuda_device):
    import torch
    return torch


def dt(torch, name):
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def normal(torch, seed, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt(torch, dtype))


def dev(torch, r):
    return torch.tensor(r, dtype=torch.int32, device="cuda").reshape(-1, 2)


# ---------------------------------------------------------------------------- 4-bit products
def q4(torch, ge, n, k, group, mins, seed=1, step=0.02):
    g = torch.Generator(device="cuda").manual_seed(seed)
    values = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((n, k // group), generator=g, device="cuda") * step + step / 20).half()
    lows = (torch.randn((n, k // group), generator=g, device="cuda") * 2.5 * step).half() if mins else None
    return ge.Q4Weight(values, scales, lows)


def dense(torch, w):
    """The weights in float64, which holds them exactly."""
    q = torch.stack([w.values & 15, w.values >> 4], -1).flatten(1).double()
    s = w.scales.double().repeat_interleave(w.group, 1)
    return (q - 8) * s if w.mins is None else q * s + w.mins.double().repeat_interleave(w.group, 1)


def by_terms(torch, x, w):
    """x w^T from the definition, each sum over its terms as they are: infinities and NaN as IEEE has them."""
    return torch.stack([(row.double()[None] * dense(torch, w)).sum(1) for row in x])


def check_same(torch, got, want, bound):
    """Finite where `want` is and within bound, else the same infinity or NaN."""
    want_t = want.to(got.dtype).double()  # what passes the type's largest number is its infinity
    finite = torch.isfinite(want_t)
    assert torch.equal(torch.isnan(got), torch.isnan(want_t))
    inf = torch.isinf(want_t)
    assert torch.equal(got[inf].double(), want_t[inf])
    assert torch.isfinite(got[finite]).all()
    assert ((got.double() - want).abs()[finite] <= bound[finite]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group,k,n,rows", [(32, 96, 5, 1), (64, 512, 300, 5), (128, 1152, 37, 12), (32, 4096, 2500, 20), (64, 320, 130, 40)])
def test_linear_q4_infinite_inputs(ge, torch, dtype, mins, group, k, n, rows):
    """Rows with an infinity give what the definition gives -- an infinity of the weight's sign, NaN where the
    weight is 0 -- and leave the other rows alone bit for bit."""
    w = q4(torch, ge, n, k, group, mins)
    x = normal(torch, 3, (rows, k), dtype)
    clean = ge.linear_q4(x, w)
    hit = sorted({0, rows // 2, rows - 1})
    for i, r in enumerate(hit):
        x[r, (k - 1, 7, k // 2)[i]] = (math.inf, -math.inf, math.inf)[i]
    got = ge.linear_q4(x, w)
    check_same(torch, got[hit], by_terms(torch, x[hit], w), torch.zeros((len(hit), n), device="cuda"))
    rest = [r for r in range(rows) if r not in hit]
    assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("mins", [False, True])
def test_linear_q4_two_infinities_and_nan(ge, torch, mins):
    w = q4(torch, ge, 77, 256, 32, mins)
    x = normal(torch, 4, (3, 256), "f16")
    x[0, 3], x[0, 200] = math.inf, -math.inf
    x[1, 9] = math.nan
    check_same(torch, ge.linear_q4(x, w), by_terms(torch, x, w), ref.linear_q4(x.nan_to_num(0, 0, 0), w.values, w.scales, w.mins)[1])


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", [(1, 33, 128), (12, 300, 640), (40, 50, 2048)])
def test_linear_q4_sums_past_32_bits(ge, torch, mins, group, rows, n, k):
    """bf16 values near the type's largest: sums of x times the 4-bit integers pass fp32, the scaled ones do not."""
    w = q4(torch, ge, n, k, group, mins, step=1e-4)
    x = (torch.sign(normal(torch, 5, (rows, k), "bf16").float()) * 2e38).bfloat16()
    x[0] = 2e38
    want = by_terms(torch, x, w)
    bound = ref.linear_q4(x, w.values, w.scales, w.mins)[1]
    check_same(torch, ge.linear_q4(x, w), want, bound)


def test_linear_q4_infinite_scales(ge, torch):
    """A scale or minimum of infinity meets every weight of its group."""
    w = q4(torch, ge, 20, 256, 32, True)
    w.scales[3, 2] = math.inf
    w.mins[5, 0] = -math.inf
    w.scales[7, 7] = math.nan
    x = normal(torch, 6, (2, 256), "f16")
    keep = [i for i in range(20) if i not in (3, 5, 7)]
    got = ge.linear_q4(x, w)
    want = by_terms(torch, x, w)
    bound = ref.linear_q4(x, w.values, w.scales.nan_to_num(0, 0, 0), w.mins.nan_to_num(0, 0, 0))[1]
    check_same(torch, got, want, bound)
    assert torch.isfinite(got[:, keep]).all()


# ---------------------------------------------------------------------------- attention
@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256), (6, 2, 128)])
def test_scores_of_minus_infinity_alone(ge, torch, heads, kvh, dim):
    """A row all of whose keys score -infinity is 0 / 0; with one finite score it is that key's value, and a row
    that sees no key stays 0."""
    n, dead = 300, 170
    q, k, v = (normal(torch, 70 + i, (n, h, dim), "f16") for i, h in enumerate((heads, kvh, kvh)))
    q[..., 0] = 1.0
    k[:dead, :, 0] = -math.inf
    k[dead + 1:, :, 0] = -math.inf
    got = ge.attention_causal(q, k, v, dev(torch, [(0, n)]))
    assert torch.isnan(got[:dead]).all()
    assert torch.equal(got[dead:], v[dead].repeat_interleave(heads // kvh, 0)[None].expand(n - dead, -1, -1))
    # Short sequences, whose rows share a tile.
    r = [(0, 40), (dead - 20, 21), (200, 9)]
    out = ge.attention_causal(q, k, v, dev(torch, r), out=torch.full_like(q, 7.0))
    assert torch.isnan(out[:40]).all() and torch.isnan(out[dead - 20:dead]).all() and torch.isnan(out[200:209]).all()
    assert torch.equal(out[dead], v[dead].repeat_interleave(heads // kvh, 0))
    assert (out[40:dead - 20] == 7.0).all() and (out[dead + 1:200] == 7.0).all() and (out[209:] == 7.0).all()


@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256)])
@pytest.mark.parametrize("plen,own", [(2000, 700), (2000, 0), (0, 900), (5, 3)])
def test_scores_of_minus_infinity_alone_across_pieces(ge, torch, heads, kvh, dim, plen, own):
    """The same where the keys are split: single tokens behind a prefix, one of them without keys of its own."""
    q, k, v = (normal(torch, 80 + i, (r, h, dim), "f16") for i, (r, h) in enumerate(((3, heads), (own, kvh), (own, kvh))))
    pk, pv = normal(torch, 84, (plen, kvh, dim), "f16"), normal(torch, 85, (plen, kvh, dim), "f16")
    q[..., 0] = 1.0
    k[..., 0] = pk[..., 0] = -math.inf
    qr, kr = [(0, 1), (1, 1), (2, 1)], [(0, own), (0, own // 2), (0, 0)]
    call = lambda: ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv)
    got = call()
    sees = [plen + m > 0 for _, m in kr]
    for i, s in enumerate(sees):
        assert torch.isnan(got[i]).all() if s else (got[i] == 0).all()
    if plen:
        pk[plen // 3, :, 0] = 0.0
        assert torch.equal(call(), pv[plen // 3].repeat_interleave(heads // kvh, 0)[None].expand(3, -1, -1))


@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("heads,kvh,dim", [(1, 1, 128), (3, 1, 256), (1, 1, 64)])
def test_scores_of_minus_infinity_alone_in_a_cut_prompt(ge, torch, heads, kvh, dim, window):
    """One long prompt, whose few items are cut along the keys."""
    n = 2500
    q, k, v = (normal(torch, 90 + i, (n, h, dim), "bf16") for i, h in enumerate((heads, kvh, kvh)))
    q[..., 0] = 1.0
    k[..., 0] = -math.inf
    k[1000, :, 0] = 0.0
    got = ge.attention_causal(q, k, v, dev(torch, [(0, n)]), window=window)
    end = 1000 + window if window else n
    assert torch.isnan(got[:1000]).all() and torch.isnan(got[end:]).all()
    assert torch.equal(got[1000:end], v[1000].repeat_interleave(heads // kvh, 0)[None].expand(end - 1000, -1, -1))


# ---------------------------------------------------------------------------- what a caller relies on around a call
def test_outputs_dropped_while_the_current_stream_reads_them(ge, torch):
    """An output made on another stream and dropped while the current one still reads it: the next call on that
    stream does not get its memory."""
    w = q4(torch, ge, 5000, 512, 32, False)
    x = normal(torch, 9, (4, 512), "f16")
    q, k, v = (normal(torch, 50 + i, (700, h, 128), "bf16") for i, h in enumerate((8, 2, 2)))
    s = dev(torch, [(0, 700)])
    xs, vs = [x * i for i in range(1, 5)], [v * i for i in range(1, 5)]
    calls = [lambda i, stream=None: ge.linear_q4(xs[i], w, stream=stream),
             lambda i, stream=None: ge.attention_causal(q, k, vs[i], s, stream=stream),
             lambda i, stream=None: ge.attention_prefix(q, k, vs[i], s, s, k, v, stream=stream)]
    for call in calls:
        want = call(0)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        call(0, side)  # kernels loaded, memory of the stream's own
        torch.cuda.synchronize()
        made = call(0, side)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(100_000_000)
        read = made.clone()
        del made
        with torch.cuda.stream(side):  # not behind the sleeping stream
            others = [call(i) for i in range(1, 4)]
        torch.cuda.synchronize()
        assert torch.equal(read, want)
        del others


def test_outputs_beside_inputs_in_the_same_rows(ge, torch):
    """`out` as columns of the rows that q, k and v are columns of: allowed, and nothing else changes; over any of
    them it is refused."""
    heads, kvh, dim, n = 4, 2, 64, 150
    wide = normal(torch, 60, (n, (2 * heads + 2 * kvh) * dim), "f16")
    q, k, v, out = (t.unflatten(1, (-1, dim)) for t in wide.split([heads * dim, kvh * dim, kvh * dim, heads * dim], 1))
    s = dev(torch, [(0, n)])
    want, before = ge.attention_causal(q, k, v, s), wide[:, :(heads + 2 * kvh) * dim].clone()
    ge.attention_causal(q, k, v, s, out=out)
    assert torch.equal(out, want) and torch.equal(wide[:, :(heads + 2 * kvh) * dim], before)
    w = q4(torch, ge, 64, 64, 32, False)
    x = normal(torch, 61, (5, 128), "f16")
    y = ge.linear_q4(x[:, :64], w)
    assert torch.equal(ge.linear_q4(x[:, :64], w, out=x[:, 64:]), y)
    for call in (lambda: ge.attention_causal(q, k, v, s, out=q), lambda: ge.attention_prefix(q, k, v, s, s, k, v, out=q),
                 lambda: ge.linear_q4(x[:, :64], w, out=x[:, 32:96]), lambda: ge.linear_q4(x[:, :64], w, out=x[:, :64])):
        with pytest.raises(ge.GemmaEmbedError) as e:
            call()
        assert e.value.case == "invalidOptions" and "overlap" in str(e.value)


WAITS_RUN_OUT = """
import ctypes, importlib, sys
import torch
ge = importlib.import_module("gemma-embed-swift_b200")
lib = importlib.import_module("gemma-embed-swift_b200._lib")
expect_lost = sys.argv[1] == "lost"
for heads, kvh, dim in ((8, 2, 128), (3, 1, 256), (2, 2, 64), (6, 2, 128)):
    for lens, gap in (([5, 40, 9], 3), ([700, 20, 300], 7), ([90] * 60, 1), ([3000], 2)):
        total = sum(lens) + gap * len(lens)
        seqs, inside, at = [], torch.zeros(total, dtype=torch.bool, device="cuda"), 0
        for n in lens:
            seqs.append((at, n))
            inside[at:at + n] = True
            at += n + gap
        s = torch.tensor(seqs, dtype=torch.int32, device="cuda")
        q, k = (torch.randn(total, h, dim, device="cuda").to(torch.bfloat16) for h in (heads, kvh))
        pk = torch.randn(600, kvh, dim, device="cuda").to(torch.bfloat16)
        for call in (lambda o: ge.attention_causal(q, k, k, s, out=o), lambda o: ge.attention_prefix(q, k, k, s, s, pk, pk, out=o)):
            out = call(torch.full_like(q, 7.0))
            assert (out[~inside] == 7.0).all(), "rows of no sequence"
            if expect_lost:
                assert torch.isnan(out[inside]).all(), (heads, dim, lens)
            else:
                assert torch.isfinite(out[inside]).all()
# The status a C caller finds in the workspace's first word.
q = torch.randn(900, 4, 64, device="cuda").half()
s = torch.tensor([[0, 900]], dtype=torch.int32, device="cuda")
shape = lib.GeAttentionShape(0, 4, 4, 64, 0.125, 0, 256, 256, 256, 0, 0, 256)
n = ctypes.c_int64(0)
assert lib.lib().ge_attention_workspace(0, ctypes.byref(shape), 900, 0, ctypes.byref(n)) == 0
ws, out = torch.full((n.value,), 255, dtype=torch.uint8, device="cuda"), torch.empty_like(q)
torch.cuda.synchronize()
assert lib.lib().ge_attention_causal(0, shape, q.data_ptr(), q.data_ptr(), q.data_ptr(), 900, s.data_ptr(), 1, out.data_ptr(),
                                     ws.data_ptr(), n.value, None) == 0
torch.cuda.synchronize()
assert ws[:4].view(torch.int32).item() == (12 if expect_lost else 0)
print("as expected")
"""


@pytest.mark.parametrize("limit,outcome", [("0", "lost"), (None, "kept"), ("1000000000", "kept")])
def test_rows_of_a_wait_that_ran_out_are_nan(cuda_device, limit, outcome):
    """With no time to wait every wait of the attention kernels runs out: its rows are NaN, no other row is
    touched, the status says so, and the process goes on."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = {k: v for k, v in os.environ.items() if k != "GE_ATTENTION_WAIT_NS"}
    if limit is not None:
        env["GE_ATTENTION_WAIT_NS"] = limit
    r = subprocess.run([sys.executable, "-c", WAITS_RUN_OUT, outcome], cwd=root, env={**env, "PYTHONPATH": root}, capture_output=True,
                       text=True, timeout=200)
    assert r.returncode == 0 and "as expected" in r.stdout, r.stderr[-2000:]


# ---------------------------------------------------------------------------- nothing lost, nothing twice
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k,dtype", [(1, 300, 65536, "f16"), (12, 300, 65536, "bf16"), (40, 130, 65536, "f16"), (1, 2500, 8192, "bf16"),
                                            (9, 5003, 8192, "f16"), (17, 41003, 8192, "bf16"), (32, 41003, 8192, "f16"),
                                            (12, 38001, 8192 + 384, "f16"), (5, 768, 1152, "bf16"), (64, 2400, 4096, "f16")])
def test_linear_q4_by_steps(ge, torch, rows, n, k, dtype, group, mins):
    """Against the bound that sees a lost stage, unit or minimum: long sums of many chunks of x, several passes over
    the column tiles, every number of rows to a launch."""
    w = q4(torch, ge, n, k, group, mins, seed=rows + k)
    x = normal(torch, rows, (rows, k), dtype)
    want, bound = ref.linear_q4_by_steps(x, w.values, w.scales, w.mins)
    ref.check(ge.linear_q4(x, w), want, bound)


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("n,k", [(50, 256), (300, 1152), (41003, 2048), (70, 8192 + 128), (300, 65536)])
def test_linear_q4_single_weights(ge, torch, n, k, group, mins):
    """Rows of x with one 1 give the weights themselves: at the borders of units, stages, chunks of x and parts of k,
    for every number of rows to a launch."""
    w = q4(torch, ge, n, k, group, mins, seed=7)
    table = dense(torch, w)
    places = sorted({p for at in (0, 32, 128, 256, 512, 1024, 4096, 8192, 16384, 32768, k // 3 // 256 * 256, k // 2 // 256 * 256, k)
                     for p in (at - 1, at, at + 7, at + 8) if 0 <= p < k})
    for rows in (1, 8, 13, 32, 64):
        for first in range(0, len(places), rows):
            at = torch.tensor(places[first:first + rows], device="cuda")
            x = torch.zeros((len(at), k), dtype=torch.float16, device="cuda")
            x[torch.arange(len(at), device="cuda"), at] = 1.0
            want = table[:, at].T
            # scale q (or q - 8) is exact in 32 bits; the minimum's product and the result round once each.
            ref.check(ge.linear_q4(x, w), want, (2.0 ** -11 + 2.0 ** -23) * want.abs() + 2.0 ** -25)


def marked(torch, rows, kvh, dim, dtype, keys, value):
    """Values of 0 but for keys[c] in column c, of every head."""
    v = torch.zeros((rows, kvh, dim), dtype=dt(torch, dtype), device="cuda")
    c = torch.arange(len(keys), device="cuda")
    v[torch.as_tensor(keys, device="cuda"), :, c] = value
    return v


def each_key(ge, torch, heads, kvh, dim, dtype, qr, kr, nkv, plen=None, window=0, keys=None):
    """Uniform weights (q = 0): a row that sees n keys gives value / n in the column of every key it sees, once,
    and 0 in the others'.  `keys`: which of the prefix' and own rows to mark (all)."""
    ntok, pre, value = max(s + n for s, n in qr), plen or 0, 1024.0
    q = torch.zeros((ntok, heads, dim), dtype=dt(torch, dtype), device="cuda")
    k = normal(torch, 1, (nkv, kvh, dim), dtype)
    pk = normal(torch, 2, (pre, kvh, dim), dtype)
    place = torch.full((ntok,), -1, device="cuda")  # of a row among its sequence's keys
    start, lost = torch.zeros(ntok, dtype=torch.long, device="cuda"), torch.ones(ntok, dtype=torch.bool, device="cuda")
    for (s, n), (ks, m) in zip(qr, kr):
        place[s:s + n] = torch.arange(n, device="cuda") + m - n
        start[s:s + n] = ks
        lost[s:s + n] = False
    lo = (place - window + 1).clamp_min(0) if window else torch.zeros_like(place)
    count = pre + (place + 1 - lo).clamp_min(0)
    keys = list(range(pre + nkv)) if keys is None else keys
    u = torch.finfo(q.dtype).eps / 2
    qs, ks = dev(torch, qr), dev(torch, kr)
    for first in range(0, len(keys), dim):
        part = keys[first:first + dim]
        both = marked(torch, pre + nkv, kvh, dim, dtype, part, value)
        pv, v = both[:pre], both[pre:]
        if plen is None:
            got = ge.attention_causal(q, k, v, qs, window=window)
        else:
            got = ge.attention_prefix(q, k, v, qs, ks, pk, pv)
        key = torch.as_tensor(part, device="cuda")[None] - pre
        own = key - start[:, None]
        seen = (key < 0) | ((own >= lo[:, None]) & (own <= place[:, None]) & (place >= 0)[:, None])
        want = torch.zeros((ntok, dim), dtype=torch.float64, device="cuda")
        want[:, :len(part)] = seen * value / count.clamp_min(1)[:, None].double()
        # Exponentials of 0 and the sums of their equals (2^-20 together), the result's rounding.
        bound = (u + 2.0 ** -20) * want + (2.0 ** -25 if dtype == "f16" else 0.0) * (want > 0)
        err = (got.double() - want[:, None]).abs()
        bad = (err > bound[:, None]) & ~lost[:, None, None]
        assert not bad.any(), (first, bad.nonzero()[:3].tolist())


SHAPES = [(8, 2, 128, "bf16"), (3, 1, 256, "f16"), (4, 4, 64, "f16"), (2, 1, 64, "bf16")]


@pytest.mark.parametrize("heads,kvh,dim,dtype", SHAPES)
@pytest.mark.parametrize("plen,n", [(8000, 1), (4097, 3), (127, 2), (128, 2), (129, 2), (1, 5), (0, 2)])
def test_prefix_every_key_once(ge, torch, heads, kvh, dim, dtype, plen, n):
    """Single tokens whose keys are cut into pieces: every prefix and own key counts once."""
    kr = []
    for i in range(n):
        kr.append((sum(m for _, m in kr), 1500 + 389 * i))
    each_key(ge, torch, heads, kvh, dim, dtype, [(i, 1) for i in range(n)], kr, sum(m for _, m in kr), plen)


@pytest.mark.parametrize("heads,kvh,dim,dtype", SHAPES)
def test_prefix_every_key_once_in_scattered_slots(ge, torch, heads, kvh, dim, dtype):
    """Slots in no order with keys of no row between them, some ranges shared, some empty; last tokens and texts."""
    slot, rng = 400, np.random.default_rng(3)
    order = [int(i) for i in rng.permutation(24)[:14]]
    kr = [(slot * i, int(m)) for i, m in zip(order, rng.integers(0, 300, 14))]
    kr[5], kr[9] = kr[2], (17, 0)
    qr, at = [], 0
    for n in rng.integers(0, 9, 14):
        qr.append((at, int(n)))
        at += int(n)
    qr[3] = (qr[3][0], 0)
    for plen in (0, 257):
        each_key(ge, torch, heads, kvh, dim, dtype, qr, kr, slot * 24, plen)


@pytest.mark.parametrize("heads,kvh,dim,dtype", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 127, 128, 129, 700])
def test_causal_every_key_once(ge, torch, heads, kvh, dim, dtype, window):
    """A cut prompt beside short ones, and a batch whose sequences share tiles."""
    for lens in ([2500, 33], [1, 130, 300, 77, 513, 0, 128]):
        r = []
        for n in lens:
            r.append((sum(m for _, m in r), n))
        keys = None if len(lens) == 2 else list(range(0, sum(lens), 3)) + [sum(lens) - 1]
        each_key(ge, torch, heads, kvh, dim, dtype, r, r, sum(lens), window=window, keys=keys)


@pytest.mark.parametrize("heads,kvh,dim,dtype", SHAPES)
@pytest.mark.parametrize("plen,own", [(8000, 2500), (4097, 1), (0, 3000), (300, 64)])
def test_one_key_holds_all_the_weight(ge, torch, heads, kvh, dim, dtype, plen, own):
    """Each row asks for one key, which scores far above all others: its value comes back, from either side of
    every border of blocks and pieces."""
    rows = dim
    total = plen + own
    step = max(1, total // 700)
    keys = sorted({p for p in list(range(0, total, step)) + [plen - 1, plen, plen + 1, plen - 2, total - 1, total - 2]
                   + [b + d for b in range(0, total, 128) for d in (-1, 0)] if 0 <= p < total})
    both_v = normal(torch, 5, (total, kvh, dim), dtype)
    s = dev(torch, [(i, 1) for i in range(rows)])
    ks = dev(torch, [(0, own)] * rows)
    q = torch.zeros((rows, heads, dim), dtype=dt(torch, dtype), device="cuda")
    for h in range(heads):
        q[torch.arange(rows, device="cuda"), h, (torch.arange(rows, device="cuda") + h) % dim] = 8.0
    group = heads // kvh
    u = torch.finfo(q.dtype).eps / 2
    for first in range(0, len(keys), dim):
        part = (keys[first:first + dim] * dim)[:dim]
        both_k = torch.zeros((total, kvh, dim), dtype=q.dtype, device="cuda")
        both_k[torch.as_tensor(part, device="cuda"), :, torch.arange(dim, device="cuda")] = 8.0
        got = ge.attention_prefix(q, both_k[plen:], both_v[plen:], s, ks, both_k[:plen], both_v[:plen], scale=1.0).double()
        for h in range(heads):
            column = (torch.arange(rows, device="cuda") + h) % dim
            # A key may be marked in several columns where there are fewer keys than columns: still one key a row.
            key = torch.as_tensor(part, device="cuda")[column]
            want = both_v[key, h // group].double()
            # The other keys' weights: e^-64 each, below 2^-25 of fp16 and 2^-60 of bf16 in all.
            err = (got[:, h] - want).abs()
            assert (err <= (u + 2.0 ** -20) * want.abs() + 2.0 ** -24 * both_v.abs().max()).all(), (first, h)


# ---------------------------------------------------------------------------- how calls are made
FIRST_CALL_IN_A_CAPTURE = """
import importlib
import torch
ge = importlib.import_module("gemma-embed-swift_b200")
dev = "cuda"
q, k = (torch.randn(300, h, 128, device=dev).half() for h in (8, 2))
s = torch.tensor([[0, 200], [200, 100]], dtype=torch.int32, device=dev)
one = torch.tensor([[0, 1], [1, 1]], dtype=torch.int32, device=dev)
w = ge.Q4Weight(torch.randint(0, 256, (500, 256), dtype=torch.uint8, device=dev), torch.rand(500, 16, device=dev).half())
x = torch.randn(3, 512, device=dev).half()
big = torch.randn(3000, 2, 128, device=dev).half()
torch.cuda.synchronize()
calls = [lambda: ge.attention_causal(q, k, k, s), lambda: ge.attention_prefix(q[:2], k, k, one, s, big, big), lambda: ge.linear_q4(x, w)]
held = []
for call in calls:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    held.append((g, out))
for (g, out), call in zip(held, calls):
    out.fill_(7.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call())
print("as expected")
"""


def test_the_first_call_of_a_process_may_be_captured(cuda_device):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE], cwd=root, env={**os.environ, "PYTHONPATH": root}, capture_output=True,
                       text=True, timeout=200)
    assert r.returncode == 0 and "as expected" in r.stdout, r.stderr[-2000:]


def test_a_side_stream_within_a_capture(ge, torch):
    """Calls on a forked stream inside a capture, joined before its end: replays give the eager results."""
    w = q4(torch, ge, 900, 256, 64, True)
    x = normal(torch, 1, (7, 256), "bf16")
    q, k, v = (normal(torch, 2 + i, (400, h, 64), "bf16") for i, h in enumerate((4, 2, 2)))
    s = dev(torch, [(0, 150), (150, 250)])
    want = [ge.linear_q4(x, w), ge.attention_causal(q, k, v, s), ge.attention_prefix(q, k, v, s, s, k, v)]
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        got = [ge.linear_q4(x, w, stream=side), ge.attention_causal(q, k, v, s, stream=side)]
        got.append(ge.attention_prefix(q, k, v, s, s, k, v))  # beside them
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        for t in got:
            t.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_of_several_threads(ge, torch):
    """Threads with streams of their own, a launch policy and an error message each."""
    w = q4(torch, ge, 900, 256, 64, True)
    xs = [normal(torch, i, (7, 256), "f16") for i in range(4)]
    q, k = (normal(torch, 20 + i, (700, h, 128), "f16") for i, h in enumerate((8, 2)))
    s = dev(torch, [(0, 500), (500, 200)])
    wants = [(ge.linear_q4(x, w), ge.attention_causal(q * (i + 1), k, k, s)) for i, x in enumerate(xs)]
    qs = [q * (i + 1) for i in range(4)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    y, o = ge.linear_q4(xs[i], w), ge.attention_causal(qs[i], k, k, s)
                    with pytest.raises(ge.GemmaEmbedError) as e:
                        ge.attention_causal(q, k, k, s, scale=-1.0) if i % 2 else ge.linear_q4(xs[i][:, :32], w)
                    assert ("scale" if i % 2 else "x must be") in str(e.value)
                torch.cuda.current_stream().synchronize()
                assert torch.equal(y, wants[i][0]) and torch.equal(o, wants[i][1])
        except BaseException as e:
            failed.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (3, 1, 256), (2, 2, 64), (3, 1, 64)])
def test_causal_across_32_bit_offsets(ge, torch, heads, kvh, dim):
    """q, k, v and out as columns of rows whose element offsets pass 2^31, whole items, pieces and recomputed rows."""
    width, rows = 1 << 16, 34000  # 4.5 GB of fp16
    cache = torch.empty((rows, width), dtype=torch.float16, device="cuda")
    part = lambda at, h: cache[:, at:at + h * dim].unflatten(1, (h, dim))
    q, k, v, out = part(0, heads), part(8192, kvh), part(20000, kvh), part(width - heads * dim, heads)
    for lens in ([900], [60] * 15):
        r = ranges_from(rows - sum(lens) - 3, lens)
        a, b = rows - sum(lens) - 10, rows
        for i, t in enumerate((q, k, v)):
            t[a:] = normal(torch, i, tuple(t[a:].shape), "f16")
        for bad in (None, math.inf):
            out[a:] = 7.0
            if bad is not None:
                v[r[0][0], :, 3] = bad
            ge.attention_causal(q, k, v, dev(torch, r), out=out)
            own = [(s - a, n) for s, n in r]
            want, bound, touched = ref.attention(q[a:b].contiguous(), k[a:b].contiguous(), v[a:b].contiguous(), own, own, 1 / math.sqrt(dim))
            keep = [c for c in range(dim) if bad is None or c != 3]
            got = out[a:b][..., keep]
            ref.check(got[touched], want[touched][..., keep], bound[touched][..., keep])
            assert (got[~touched] == 7.0).all()


def ranges_from(at, lens):
    out = []
    for n in lens:
        out.append((at, n))
        at += n
    return out


def test_linear_q4_across_32_bit_offsets(ge, torch):
    """Weights of more than 2^32 bytes, x and out as columns of rows further apart than 2^31 elements."""
    n, k = 140_003, 65536
    values = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda")
    scales = (torch.rand((n, k // 32), device="cuda") * 0.02 + 1e-3).half()
    w = ge.Q4Weight(values, scales)
    x = normal(torch, 1, (2, k), "f16", 0.1)
    got = ge.linear_q4(x, w)
    for at in (0, 65530, 131064, n - 20):
        want, bound = ref.linear_q4_by_steps(x, values[at:at + 20].contiguous(), scales[at:at + 20].contiguous(), None)
        ref.check(got[:, at:at + 20], want, bound)
    del w, values, scales
    stride = (1 << 31) + 64
    far = torch.empty(stride + 2048, dtype=torch.float16, device="cuda")
    w = q4(torch, ge, 500, 512, 32, True)
    x = far.as_strided((2, 512), (stride, 1))
    x.copy_(normal(torch, 2, (2, 512), "f16"))
    out = far.as_strided((2, 500), (stride, 1), 1024)
    want, bound = ref.linear_q4_by_steps(x.contiguous(), w.values, w.scales, w.mins)
    ref.check(ge.linear_q4(x, w, out=out), want, bound)


# ---------------------------------------------------------------------------- values up to the type's largest
@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_causal_values_at_the_types_limits(ge, torch, heads, kvh, dim, sign):
    """A row's result is a mean of values: bf16's largest, in columns beside ordinary and tiny ones, do not overflow
    on the way, in whole items and in pieces."""
    top = sign * torch.finfo(torch.bfloat16).max
    for lens in ([40, 300, 7], [2600]):
        n = sum(lens)
        q, k, v = (normal(torch, 30 + i, (n, h, dim), "bf16") for i, h in enumerate((heads, kvh, kvh)))
        v[..., 0] = top                                             # in every key
        v[..., 1] = torch.where(torch.arange(n, device="cuda") % 2 == 0, top, -top)[:, None]
        v[::3, :, 2] = top
        v[..., 3] = 1e-36 * v[..., 4].float()
        r = ranges_from(0, lens)
        got = ge.attention_causal(q, k, v, dev(torch, r))
        want, bound, _ = ref.attention(q, k, v, r, r, 1 / math.sqrt(dim))
        assert torch.isfinite(got).all()
        ref.check(got, want, bound)


@pytest.mark.parametrize("heads,kvh,dim", [(8, 2, 128), (3, 1, 256), (2, 2, 64)])
@pytest.mark.parametrize("plen,own", [(6000, 900), (0, 5000), (300, 50)])
def test_prefix_values_at_the_types_limits(ge, torch, heads, kvh, dim, plen, own):
    """The same where pieces are joined: the largest values in all pieces, or in one."""
    top = torch.finfo(torch.bfloat16).max
    rows = 5
    q = normal(torch, 1, (rows, heads, dim), "bf16")
    k, v = normal(torch, 2, (own, kvh, dim), "bf16"), normal(torch, 3, (own, kvh, dim), "bf16")
    pk, pv = normal(torch, 4, (plen, kvh, dim), "bf16"), normal(torch, 5, (plen, kvh, dim), "bf16")
    v[..., 0] = pv[..., 0] = top
    v[..., 1] = -top
    v[own // 2:, :, 2] = top
    pv[plen // 3:plen // 2, :, 3] = -top
    qr, kr = [(i, 1) for i in range(rows)], [(0, own - i) for i in range(rows)]
    got = ge.attention_prefix(q, k, v, dev(torch, qr), dev(torch, kr), pk, pv)
    want, bound, _ = ref.attention(q, k, v, qr, kr, 1 / math.sqrt(dim), prefix_k=pk, prefix_v=pv)
    assert torch.isfinite(got).all()
    ref.check(got, want, bound)


# ---------------------------------------------------------------------------- thousands of sequences
def shuffled(rng, lens, gap=0):
    """Ranges of these lengths in memory order, named in another."""
    r = []
    at = 0
    for n in lens:
        r.append((at, int(n)))
        at += int(n) + gap
    return [r[i] for i in rng.permutation(len(r))], max(a + n for a, n in r)


@pytest.mark.parametrize("heads,kvh,dim,dtype", SHAPES)
@pytest.mark.parametrize("window,gap", [(0, 0), (3, 2)])
def test_thousands_of_sequences_every_key_once(ge, torch, heads, kvh, dim, dtype, window, gap):
    """Short texts, empty ones among them, beside a few long ones, in no order."""
    rng = np.random.default_rng(7)
    lens = rng.integers(0, 4, 1500)
    lens[[100, 900]] = 700, 300
    r, total = shuffled(rng, lens, gap)
    each_key(ge, torch, heads, kvh, dim, dtype, r, r, total, window=window, keys=list(range(0, total, 5)))


@pytest.mark.parametrize("heads,kvh,dim,dtype", SHAPES)
def test_thousands_of_last_tokens_every_key_once(ge, torch, heads, kvh, dim, dtype):
    rng = np.random.default_rng(8)
    kr, nkv = shuffled(rng, rng.integers(0, 6, 1300), 1)
    kr[7], kr[8] = kr[1200], (3, 500)
    qr, ntok = shuffled(rng, rng.integers(0, 3, 1300))
    each_key(ge, torch, heads, kvh, dim, dtype, qr, kr, nkv + 600, 130, keys=list(range(0, 130 + nkv, 7)))


def test_thousands_of_ranges_that_share_rows_or_leave_the_tensors(ge, torch):
    """Rows of one range alone are right, rows of none untouched, whatever the others name: the same range many
    times, ranges within ranges, starts and ends past the last row."""
    n, rng = 4000, np.random.default_rng(9)
    q, k, v = (normal(torch, 31 + i, (n, h, 64), "f16") for i, h in enumerate((2, 1, 1)))
    r = [(int(i) * 2, 2) for i in rng.permutation(900)]              # [0, 1800): two rows each
    r += [(2000, 40)] * 300 + [(2100, 200), (2150, 10), (2200, 300)] + [(2900 + i, 3) for i in range(50)]
    r += [(3000, 500), (3900, 1 << 30), (4000, 5), (1 << 30, 7), (-3, 2), (3700, 0), (3701, 0)]
    r = [r[i] for i in rng.permutation(len(r))]
    out = torch.full_like(q, 7.0)
    ge.attention_causal(q, k, v, dev(torch, r), out=out)
    cover = torch.zeros(n, dtype=torch.int32, device="cuda")
    cut = [(s, min(m, n - s)) for s, m in r if 0 <= s < n and m > 0]
    for s, m in cut:
        cover[s:s + m] += 1
    assert (out[cover == 0] == 7.0).all() and (cover > 1).sum() > 100
    want, bound, _ = ref.attention(q, k, v, cut, cut, 0.125)  # shared rows hold the last range's: not looked at
    alone = cover == 1
    ref.check(out[alone], want[alone], bound[alone])


def test_time_of_many_sequences_grows_with_their_number(ge, torch):
    """300,000 single tokens: a few ms, where a look through all sequences for every tile would take 100 times that."""
    n = 300_000
    q, k = normal(torch, 1, (n, 4, 64), "f16"), normal(torch, 2, (n, 1, 64), "f16")
    s = torch.stack([torch.arange(n, device="cuda"), torch.ones(n, device="cuda")], 1).int()
    for _ in range(2):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        got = ge.attention_causal(q, k, k, s)
        b.record()
        torch.cuda.synchronize()
    assert torch.equal(got, k.expand(-1, 4, -1))
    assert a.elapsed_time(b) < 50


@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256)])
@pytest.mark.parametrize("plen,own", [(3000, 500), (0, 2500), (40, 60)])
@pytest.mark.parametrize("weight", ["underflows", "none"])
def test_no_weight_times_an_infinite_value(ge, torch, heads, kvh, dim, plen, own, weight):
    """A key with an infinite value whose weight is 0 -- far below another's, or a score of -infinity -- gives NaN in
    that column, wherever the keys are cut, and the others' mean in the other columns."""
    total, dtype = plen + own, torch.float16
    q = torch.zeros((3, heads, dim), dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    ks, vs = normal(torch, 1, (total, kvh, dim), "f16"), normal(torch, 2, (total, kvh, dim), "f16")
    ks[..., 0] = -2000.0  # e^-4000 beside a key of 2000
    ks[total - 5, :, 0] = 2000.0
    for at in (0, total // 3, total - 1):
        k, v = ks.clone(), vs.clone()
        if weight == "none":
            k[at, :, 0] = -math.inf
        v[at, :, 7] = math.inf
        qr, kr = [(i, 1) for i in range(3)], [(0, own)] * 3
        got = ge.attention_prefix(q, k[plen:], v[plen:], dev(torch, qr), dev(torch, kr), k[:plen], v[:plen], scale=1.0)
        want = vs[total - 5].repeat_interleave(heads // kvh, 0)[None].expand(3, -1, -1)
        assert torch.isnan(got[..., 7]).all()
        rest = [c for c in range(dim) if c != 7]
        assert torch.equal(got[..., rest], want[..., rest])


@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256)])
@pytest.mark.parametrize("dtype,size", [("f16", 60000.0), ("bf16", 3e9), ("bf16", 1e18), ("f16", 3000.0)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_whose_steps_an_exponent_feels(ge, torch, heads, kvh, dim, dtype, size, sign):
    """Scores of 10^7 to 10^36, all positive or all negative: the largest of a row holds all the weight, in whole
    items and where the keys are cut."""
    for lens in ([40, 200, 7], [2300]):
        n = sum(lens)
        g = torch.Generator(device="cuda").manual_seed(n)
        q, v = torch.zeros((n, heads, dim), device="cuda"), normal(torch, 3, (n, kvh, dim), dtype)
        q[..., 1] = size
        k = torch.zeros((n, kvh, dim), device="cuda")
        # From size / 2 on in steps of size / 128: equal, or far apart.
        k[..., 1] = sign * size * (64 + torch.randint(0, 30, (n, kvh), generator=g, device="cuda")) / 128
        q, k = q.to(v.dtype), k.to(v.dtype)
        r = ranges_from(0, lens)
        got = ge.attention_causal(q, k, v, dev(torch, r), scale=1.0).double()
        group, u = heads // kvh, torch.finfo(v.dtype).eps / 2
        for s, m in r:
            for h in range(heads):
                score = k[s:s + m, h // group, 1].double()
                top = torch.cummax(score, 0).values
                at = (score[None] == top[:, None]) & (torch.arange(m, device="cuda")[None] <= torch.arange(m, device="cuda")[:, None])
                w = at.double() / at.sum(1, keepdim=True)
                vals = v[s:s + m, h // group].double()
                err = (got[s:s + m, h] - w @ vals).abs()
                # Weights of 1 / ties in 32 bits, then the result's rounding.
                assert (err <= (u + 2.0 ** -18) * (w @ vals.abs()) + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256), (6, 2, 128)])
@pytest.mark.parametrize("lens", [[1, 2, 3, 40, 90], [700, 33], [2600]])
def test_means_of_the_largest_value_are_finite(ge, torch, dtype, heads, kvh, dim, lens):
    """Every key has the type's largest (or lowest) value in some columns: so has every row, whatever its weights
    were rounded to."""
    n = sum(lens)
    top = torch.finfo(dt(torch, dtype)).max
    q, k, v = (normal(torch, 30 + i, (n, h, dim), dtype) for i, h in enumerate((heads, kvh, kvh)))
    v[..., 5], v[..., 6] = top, -top
    r = ranges_from(0, lens)
    got = ge.attention_causal(q, k, v, dev(torch, r)).double()
    u = torch.finfo(dt(torch, dtype)).eps / 2
    assert torch.isfinite(got).all()
    # A probability's rounding, exponentials and sums.
    assert ((got[..., 5] - top).abs() <= (2 * u + 2.0 ** -18) * top).all() and ((got[..., 6] + top).abs() <= (2 * u + 2.0 ** -18) * top).all()
    want, bound, _ = ref.attention(q, k, v, r, r, 1 / math.sqrt(dim))
    ref.check(got, want, bound)
    v[0, :, 5] = math.inf  # an infinity stays one
    got = ge.attention_causal(q, k, v, dev(torch, r))
    assert torch.isinf(got[:lens[0], :, 5]).all() and torch.isfinite(got[lens[0]:]).all()


@pytest.mark.parametrize("ntok", [1, 5, 1023, 1024, 1025, 3000])
def test_thousands_of_sequences_over_few_rows(ge, torch, ntok):
    """More sequences than rows: nearly all are empty, or lie past the last row."""
    q, k, v = (normal(torch, 31 + i, (ntok, h, 64), "f16") for i, h in enumerate((2, 1, 1)))
    out = torch.full_like(q, 7.0)
    ge.attention_causal(q, k, v, torch.zeros((5000, 2), dtype=torch.int32, device="cuda"), out=out)
    assert (out == 7.0).all()
    s = torch.zeros((5000, 2), dtype=torch.int32, device="cuda")
    s[1200:2400, 0], s[1200:2400, 1] = ntok, 9
    s[4999] = torch.tensor([ntok // 2, ntok - ntok // 2])
    ge.attention_causal(q, k, v, s, out=out)
    r = [(ntok // 2, ntok - ntok // 2)]
    want, bound, touched = ref.attention(q, k, v, r, r, 0.125)
    ref.check(out[touched], want[touched], bound[touched])
    assert (out[~touched] == 7.0).all()


@pytest.mark.parametrize("heads,kvh,dim", [(65535, 65535, 64), (65408, 511, 64), (6000, 6000, 256), (12800, 100, 128)])
def test_many_heads_few_rows(ge, torch, heads, kvh, dim):
    """The most heads there may be, with one of their own and with 128 to a KV head."""
    n = 3
    q, k, v = (normal(torch, 31 + i, (n, h, dim), "bf16") for i, h in enumerate((heads, kvh, kvh)))
    r = [(0, 1), (1, 2)]
    got = ge.attention_causal(q, k, v, dev(torch, r))
    want, bound, _ = ref.attention(q, k, v, r, r, 1 / math.sqrt(dim))
    ref.check(got, want, bound)
    pk = normal(torch, 5, (150, kvh, dim), "bf16")
    got = ge.attention_prefix(q, k, v, dev(torch, r), dev(torch, r), pk, pk)
    want, bound, _ = ref.attention(q, k, v, r, r, 1 / math.sqrt(dim), prefix_k=pk, prefix_v=pk)
    ref.check(got, want, bound)


def test_thousands_of_sequences_in_a_graph(ge, torch):
    """Captured, and replayed with other ranges in the same tensor, bit for bit as outside."""
    rng = np.random.default_rng(4)
    lens = rng.integers(0, 5, 2500)
    lens[3] = 900
    r, n = shuffled(rng, lens)
    other, m = shuffled(rng, lens[::-1].copy())
    assert n == m
    q, k, v = (normal(torch, 31 + i, (n, h, 128), "bf16") for i, h in enumerate((8, 2, 2)))
    s = dev(torch, r)
    wants = [ge.attention_causal(q, k, v, dev(torch, t)) for t in (r, other)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ge.attention_causal(q, k, v, s)
    for t, want in ((r, wants[0]), (other, wants[1]), (r, wants[0])):
        s.copy_(dev(torch, t))
        got.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
