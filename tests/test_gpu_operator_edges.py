"""The operators on device tensors at the edges of what their calls allow, on a B200: infinities and sums past
the types, and what a caller relies on around a call."""
import math
import os
import subprocess
import sys

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
