"""Operators on device tensors, what needs no GPU: refusals of the C entry points (every argument is
checked before a device is touched) and the repacking of GGUF's 4-bit blocks."""
import ctypes
import importlib

import numpy as np
import pytest

FAKE = 1 << 20  # a pointer that is never followed: the calls below are refused, or have no rows


@pytest.fixture(scope="module")
def lib(ge):
    return importlib.import_module("gemma-embed-swift_b200._lib")


def shape(lib, **over):
    s = lib.GeAttentionShape()
    base = dict(dtype=0, heads=4, kv_heads=2, head_dim=64, scale=0.125, window=0, q_stride=256, k_stride=128, v_stride=128,
                prefix_k_stride=128, prefix_v_stride=128, out_stride=256)
    for n, v in {**base, **over}.items():
        setattr(s, n, v)
    return s


def causal(lib, s, **over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, ntok=8, seqs=FAKE, nseq=1, out=FAKE, ws=FAKE, nbytes=1 << 30)
    a.update(over)
    L = lib.lib()
    rc = L.ge_attention_causal(0, ctypes.byref(s), a["q"], a["k"], a["v"], a["ntok"], a["seqs"], a["nseq"], a["out"],
                               a["ws"], a["nbytes"], None)
    return rc, (L.ge_last_error(None) or b"").decode()


def prefix(lib, s, **over):
    a = dict(q=FAKE, ntok=8, k=FAKE, v=FAKE, nkv=8, pk=FAKE, pv=FAKE, plen=4, qs=FAKE, ks=FAKE, nseq=1, out=FAKE, ws=FAKE,
             nbytes=1 << 30)
    a.update(over)
    L = lib.lib()
    rc = L.ge_attention_prefix(0, ctypes.byref(s), a["q"], a["ntok"], a["k"], a["v"], a["nkv"], a["pk"], a["pv"], a["plen"],
                               a["qs"], a["ks"], a["nseq"], a["out"], a["ws"], a["nbytes"], None)
    return rc, (L.ge_last_error(None) or b"").decode()


@pytest.mark.parametrize("over", [
    dict(dtype=2), dict(dtype=-1), dict(head_dim=96), dict(head_dim=0), dict(heads=5), dict(heads=0), dict(kv_heads=0),
    dict(heads=-4, kv_heads=-2), dict(heads=258, kv_heads=2), dict(heads=65536 * 2, kv_heads=2), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(q_stride=248),
    dict(q_stride=260), dict(k_stride=64), dict(v_stride=0), dict(out_stride=257), dict(q_stride=1 << 40)])
def test_attention_refuses_bad_shapes(lib, over):
    rc, msg = causal(lib, shape(lib, **over))
    assert rc == 9 and msg.startswith("invalid options: ")


@pytest.mark.parametrize("over", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(seqs=None), dict(seqs=FAKE + 2),
                                  dict(q=FAKE + 2), dict(k=FAKE + 8), dict(v=FAKE + 4), dict(out=FAKE + 2), dict(ntok=-1),
                                  dict(nseq=-1), dict(ntok=(1 << 30) + 1)])
def test_causal_refuses_bad_arguments(lib, over):
    rc, msg = causal(lib, shape(lib), **over)
    assert rc == 9 and msg.startswith("invalid options: ")


@pytest.mark.parametrize("over", [dict(q=None), dict(pk=None), dict(pv=None), dict(pk=FAKE + 2), dict(pv=FAKE + 8), dict(k=None),
                                  dict(qs=None), dict(ks=None), dict(ks=FAKE + 1), dict(plen=-1), dict(nkv=-1), dict(ntok=-2),
                                  dict(plen=(1 << 30) + 1)])
def test_prefix_refuses_bad_arguments(lib, over):
    rc, msg = prefix(lib, shape(lib), **over)
    assert rc == 9 and msg.startswith("invalid options: ")


def test_prefix_refuses_a_window(lib):
    rc, msg = prefix(lib, shape(lib, window=16))
    assert rc == 9 and "window" in msg


def test_null_shape_is_refused(lib):
    L = lib.lib()
    assert L.ge_attention_causal(0, None, FAKE, FAKE, FAKE, 8, FAKE, 1, FAKE, FAKE, 1 << 30, None) == 9
    n = ctypes.c_int64(0)
    assert L.ge_attention_workspace(0, None, 8, 0, ctypes.byref(n)) == 9
    assert L.ge_attention_workspace(0, ctypes.byref(shape(lib)), 8, 0, None) == 9
    assert L.ge_attention_workspace(0, ctypes.byref(shape(lib)), -1, 0, ctypes.byref(n)) == 9


def test_calls_without_rows_do_nothing(lib):
    """No rows or no sequences: accepted with whatever pointers, and no device is touched."""
    assert causal(lib, shape(lib), ntok=0, q=None, k=None, v=None, out=None)[0] == 0
    assert causal(lib, shape(lib), nseq=0, seqs=None)[0] == 0
    assert prefix(lib, shape(lib), ntok=0, q=None, out=None)[0] == 0
    assert lib.lib().ge_linear_q4(0, 0, None, 32, 0, 32, None, None, None, 32, 8, None, 8, None) == 0
    assert lib.lib().ge_linear_q4(0, 0, None, 32, 1, 32, None, None, None, 32, 0, None, 8, None) == 0


@pytest.mark.parametrize("over", [
    dict(dtype=2), dict(rows=-1), dict(rows=65), dict(group=16), dict(group=0), dict(k=48), dict(k=0), dict(k=65536 + 32),
    dict(n=-1), dict(x=None), dict(values=None), dict(scales=None), dict(out=None), dict(x=FAKE + 8), dict(values=FAKE + 4),
    dict(scales=FAKE + 1), dict(mins=FAKE + 1), dict(out=FAKE + 1), dict(x_stride=56), dict(x_stride=68), dict(out_stride=7)])
def test_linear_q4_refuses_bad_arguments(lib, over):
    a = dict(dtype=0, x=FAKE, x_stride=64, rows=2, k=64, values=FAKE, scales=FAKE, mins=None, group=32, n=8, out=FAKE, out_stride=8)
    a.update(over)
    L = lib.lib()
    rc = L.ge_linear_q4(0, a["dtype"], a["x"], a["x_stride"], a["rows"], a["k"], a["values"], a["scales"], a["mins"], a["group"],
                        a["n"], a["out"], a["out_stride"], None)
    assert rc == 9 and (L.ge_last_error(None) or b"").startswith(b"invalid options: ")


def repack(lib, blocks, kind, n, k):
    values, scales, mins = np.zeros((n, k // 2), np.uint8), np.zeros((n, k // 32), np.uint16), np.zeros((n, k // 32), np.uint16)
    u8, u16 = ctypes.POINTER(ctypes.c_uint8), ctypes.POINTER(ctypes.c_uint16)
    rc = lib.lib().ge_q4_repack(blocks.ctypes.data_as(u8), kind, n, k, values.ctypes.data_as(u8), scales.ctypes.data_as(u16),
                                mins.ctypes.data_as(u16))
    assert rc == 0
    return values, scales, mins


@pytest.mark.parametrize("kind,per", [(2, 18), (3, 20)])
@pytest.mark.parametrize("n,k", [(1, 32), (3, 96), (5, 256)])
def test_q4_repack_matches_the_block_layout(lib, kind, per, n, k):
    """GGUF's Q4_0 (fp16 scale, 16 bytes) and Q4_1 (scale, min, 16 bytes) blocks: byte j holds elements j and
    j + 16 of the block."""
    rng = np.random.default_rng(n * k + kind)
    blocks = rng.integers(0, 256, (n, k // 32, per), dtype=np.uint8)
    values, scales, mins = repack(lib, np.ascontiguousarray(blocks), kind, n, k)
    assert np.array_equal(scales, blocks[..., :2].copy().view(np.uint16)[..., 0])
    if kind == 3:
        assert np.array_equal(mins, blocks[..., 2:4].copy().view(np.uint16)[..., 0])
    q = blocks[..., per - 16:]
    want = np.concatenate([q & 15, q >> 4], -1).reshape(n, k)
    got = np.stack([values & 15, values >> 4], -1).reshape(n, k)
    assert np.array_equal(got, want)


def test_q4_repack_refusals(lib):
    u8, u16 = ctypes.POINTER(ctypes.c_uint8), ctypes.POINTER(ctypes.c_uint16)
    b = np.zeros(64, np.uint8)
    p8, p16 = b.ctypes.data_as(u8), b.ctypes.data_as(u16)
    call = lib.lib().ge_q4_repack
    assert call(p8, 8, 1, 32, p8, p16, None) == 3  # Q8_0
    assert call(p8, 2, 1, 31, p8, p16, None) == 9
    assert call(p8, 2, -1, 32, p8, p16, None) == 9
    assert call(p8, 3, 1, 32, p8, p16, None) == 9  # Q4_1 without room for the mins
    assert call(None, 2, 1, 32, p8, p16, None) == 9
    assert call(None, 2, 0, 32, None, None, None) == 0


def test_python_wrappers_refuse_host_tensors(ge):
    import torch
    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    seqs = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: ge.attention_causal(q, q, q, seqs), lambda: ge.attention_prefix(q, q, q, seqs, seqs, q, q),
                 lambda: ge.Q4Weight(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.float16)),
                 lambda: ge.attention_prefix(q, q, q, seqs, seqs, None, None)):
        with pytest.raises(ge.GemmaEmbedError) as e:
            call()
        assert e.value.case == "invalidOptions"
    with pytest.raises(ge.GemmaEmbedError) as e:
        ge.Q4Weight.from_blocks(b"", "Q8_0", 1, 32)
    assert e.value.case == "unsupportedTensorType"
    with pytest.raises(ge.GemmaEmbedError) as e:
        ge.Q4Weight.from_blocks(b"\0" * 17, "Q4_0", 1, 32)
    assert e.value.case == "invalidOptions"


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_attention_refuses_scales_past_the_kernels_units(lib, scale):
    """A finite scale whose product with log2 e is not: a zero query's scores would be 0 x infinity."""
    for call in (causal, prefix):
        rc, msg = call(lib, shape(lib, scale=scale))
        assert rc == 9 and "scale" in msg


class Recorder:
    """In place of the library: notes the calls, and answers that all is well."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*a):
            self.calls.append((name, a))
            return 0
        return call


@pytest.fixture()
def hostside(ge, monkeypatch):
    """The wrappers up to the library's call, with tensors of any device taken for CUDA tensors."""
    ops = importlib.import_module("gemma-embed-swift_b200.operators")
    rec = Recorder()
    monkeypatch.setattr(ops, "_on_device", lambda name, t, device=None: t.get_device())
    monkeypatch.setattr(ops, "_stream", lambda stream, device: (0, None))
    monkeypatch.setattr(ops, "_workspace_bytes", lambda *a: 256)
    monkeypatch.setattr(ops._lib, "lib", lambda: rec)
    return ops, rec


def meta(*shape, dtype="float16"):
    """A tensor of any size without memory."""
    import torch
    return torch.empty(shape, dtype=getattr(torch, dtype), device="meta")


@pytest.mark.parametrize("window,handed", [(0, 0), (5, 5), (2**31 - 1, 2**31 - 1), (2**31, 2**31 - 1), (2**32, 2**31 - 1),
                                           (2**32 + 1, 2**31 - 1), (2**70, 2**31 - 1), (-1, None), (-2**32, None), (-2**32 + 7, None)])
def test_windows_past_32_bits(hostside, ge, window, handed):
    """A window longer than any range is no window; nothing wraps to a small one."""
    import torch
    ops, rec = hostside
    q, s = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int32)
    if handed is None:
        with pytest.raises(ge.GemmaEmbedError) as e:
            ops.attention_causal(q, q, q, s, window=window)
        assert e.value.case == "invalidOptions" and not rec.calls
    else:
        ops.attention_causal(q, q, q, s, window=window)
        (name, a), = rec.calls
        assert name == "ge_attention_causal" and a[1].window == handed


def test_counts_past_32_bits_are_refused(hostside, ge):
    """Row, head and sequence counts and weight sizes whose lowest 32 bits would pass for others."""
    ops, rec = hostside
    big = 1 << 32
    q, k, s = meta(8, 4, 64), meta(8, 2, 64), meta(1, 2, dtype="int32")
    w = lambda n, k: ops.Q4Weight(meta(n, k // 2, dtype="uint8"), meta(n, k // 32))
    bad = [lambda: ops.attention_causal(meta(big + 8, 4, 64), meta(big + 8, 2, 64), meta(big + 8, 2, 64), s),
           lambda: ops.attention_causal(meta(0, big + 4, 64), meta(0, 2, 64), meta(0, 2, 64), s),
           lambda: ops.attention_causal(q, k, k, meta(big, 2, dtype="int32")),
           lambda: ops.attention_causal(q, k, k, meta(big + 1, 2, dtype="int32")),
           lambda: ops.attention_prefix(q, meta(big, 2, 64), meta(big, 2, 64), s, s, k, k),
           lambda: ops.attention_prefix(q, k, k, s, s, meta(big, 2, 64), meta(big, 2, 64)),
           lambda: ops.linear_q4(meta(big, 64), w(8, 64)),
           lambda: ops.linear_q4(meta(1, 64).expand(big + 2, 64), w(8, 64)),
           lambda: ops.linear_q4(meta(65, 64), w(8, 64)),
           lambda: ops.linear_q4(meta(2, 64), w(big + 8, 64)),
           lambda: ops.linear_q4(meta(2, big + 64), w(8, big + 64))]
    for i, call in enumerate(bad):
        with pytest.raises(ge.GemmaEmbedError) as e:
            call()
        assert e.value.case == "invalidOptions" and not rec.calls, i


def test_dual_tensors_are_refused(hostside, ge):
    """Forward-mode differentiation: a tangent would be dropped without a word."""
    import torch
    import torch.autograd.forward_ad as forward
    ops, rec = hostside
    q, k, s = torch.zeros(4, 2, 64).half(), torch.zeros(4, 1, 64).half(), torch.zeros(1, 2, dtype=torch.int32)
    x, o = torch.zeros(2, 64).half(), torch.zeros(2, 8).half()
    w = ops.Q4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2).half())
    with forward.dual_level():
        d = lambda t: forward.make_dual(t, torch.ones_like(t))
        bad = [lambda: ops.attention_causal(d(q), k, k, s), lambda: ops.attention_causal(q, d(k), k, s),
               lambda: ops.attention_causal(q, k, d(k), s), lambda: ops.attention_causal(q, k, k, s, out=d(q)),
               lambda: ops.attention_prefix(q, k, k, s, s, d(k), k), lambda: ops.attention_prefix(q, k, k, s, s, k, d(k)),
               lambda: ops.linear_q4(d(x), w), lambda: ops.linear_q4(x, w, out=d(o)),
               lambda: ops.Q4Weight(w.values, d(w.scales)), lambda: ops.Q4Weight(w.values, w.scales, d(w.scales))]
        for i, call in enumerate(bad):
            for context in (torch.enable_grad, torch.no_grad):
                with context(), pytest.raises(ge.GemmaEmbedError) as e:
                    call()
                assert e.value.case == "invalidOptions" and "tangent" in str(e.value), i
        assert not rec.calls
        ops.attention_causal(q, k, k, s)  # others pass inside a level too
        ops.linear_q4(x, w)
    assert [name for name, _ in rec.calls] == ["ge_attention_causal", "ge_linear_q4"]


def test_scales_that_require_a_gradient_by_the_call_are_refused(hostside, ge):
    """A weight made while no gradients are recorded, or whose scales came to require one afterwards."""
    import torch
    ops, rec = hostside
    x = torch.zeros(2, 64).half()
    values, scales = torch.zeros(8, 32, dtype=torch.uint8), lambda: torch.zeros(8, 2).half()
    with torch.no_grad():
        first = ops.Q4Weight(values, scales().requires_grad_())
    later = ops.Q4Weight(values, scales(), scales())
    later.mins.requires_grad_()
    for w in (first, later):
        with pytest.raises(ge.GemmaEmbedError) as e:
            ops.linear_q4(x, w)
        assert e.value.case == "invalidOptions" and "gradient" in str(e.value) and not rec.calls
    with torch.no_grad():
        ops.linear_q4(x, first)
        ops.linear_q4(x, later)
    assert len(rec.calls) == 2


def test_a_given_out_counts_as_changed(hostside):
    """Autograd's saved values: an `out` that another operation kept for its backward pass is known to have changed,
    views and their base alike; inference tensors, which count nothing, pass."""
    import torch
    ops, _ = hostside
    q, k, s = torch.zeros(4, 2, 64).half(), torch.zeros(4, 1, 64).half(), torch.zeros(1, 2, dtype=torch.int32)
    x = torch.zeros(2, 64).half()
    w = ops.Q4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2).half())
    wide, o = torch.zeros(2, 16).half(), torch.zeros(4, 2, 64).half()
    for call, out, base in ((lambda t: ops.linear_q4(x, w, out=t), wide[:, 8:], wide),
                            (lambda t: ops.attention_causal(q, k, k, s, out=t), o, o),
                            (lambda t: ops.attention_prefix(q, k, k, s, s, k, k, out=t), o, o)):
        p = torch.ones(out.shape, requires_grad=True)
        y = (p.half() * out).sum()
        before = base._version
        assert call(out) is out
        assert base._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with torch.inference_mode():
            call(out.clone())
    with torch.inference_mode():
        held = torch.zeros(2, 8).half()
    ops.linear_q4(x, w, out=held)


def q4_call(lib, device=-1, **over):
    a = dict(dtype=0, x=FAKE, x_stride=64, rows=2, k=64, values=FAKE << 1, scales=FAKE << 2, mins=None, group=32, n=8, out=FAKE << 3,
             out_stride=8)
    a.update(over)
    L = lib.lib()
    rc = L.ge_linear_q4(device, a["dtype"], a["x"], a["x_stride"], a["rows"], a["k"], a["values"], a["scales"], a["mins"], a["group"],
                        a["n"], a["out"], a["out_stride"], None)
    return rc, (L.ge_last_error(None) or b"").decode()


# Addresses of arrays far apart; of the calls below those that are not refused for their arguments name no device.
Q, K, V, PK, PV, OUT = (FAKE << i for i in range(1, 7))
ROW = 2 * 256  # bytes of a row of 4 heads of 64
WIDE = {n + "_stride": 1 << 38 for n in ("q", "k", "v", "prefix_k", "prefix_v", "out")}


def apart(call, lib, s, **over):
    L = lib.lib()
    a = dict(q=Q, k=K, v=V, out=OUT, ntok=8, nkv=8, pk=PK, pv=PV, plen=4)
    a.update(over)
    if call == "causal":
        rc = L.ge_attention_causal(-1, ctypes.byref(s), a["q"], a["k"], a["v"], a["ntok"], FAKE, 1, a["out"], FAKE, 1 << 30, None)
    else:
        rc = L.ge_attention_prefix(-1, ctypes.byref(s), a["q"], a["ntok"], a["k"], a["v"], a["nkv"], a["pk"], a["pv"], a["plen"], FAKE,
                                   FAKE, 1, a["out"], FAKE, 1 << 30, None)
    return rc, (L.ge_last_error(None) or b"").decode()


@pytest.mark.parametrize("over,strides,refused", [
    (dict(), {}, False),
    (dict(out=Q), {}, True),                                  # in place
    (dict(out=Q + 8 * ROW), {}, False),                       # right behind q
    (dict(out=Q + 8 * ROW - 16), {}, True),                   # its last 16 bytes
    (dict(q=OUT + 8 * ROW), {}, False),
    (dict(q=OUT + 8 * ROW - 16), {}, True),
    (dict(out=K), {}, True), (dict(out=V), {}, True),
    (dict(out=K - 8 * ROW), {}, False), (dict(out=V - 8 * ROW + 16), {}, True),
    (dict(out=Q + ROW), dict(q_stride=512, out_stride=512), False),       # columns of the same wide rows
    (dict(out=Q + ROW - 16), dict(q_stride=512, out_stride=512), True),   # one column in common
    (dict(out=Q + ROW + 16), dict(q_stride=512, out_stride=512), True),   # into q's next row
    (dict(q=OUT + ROW), dict(q_stride=512, out_stride=512), False),
    (dict(out=Q + ROW), dict(q_stride=512, out_stride=768), True),        # spans that meet, strides that do not
    (dict(ntok=1, out=Q + ROW), {}, False), (dict(ntok=1, out=Q + ROW - 16), {}, True),
    (dict(ntok=1, out=Q), dict(q_stride=4096), True),
    (dict(ntok=1 << 30, out=Q - ROW), WIDE, False),
    (dict(ntok=1 << 30, out=Q - 16), WIDE, True)])
def test_outputs_over_inputs_are_refused(lib, over, strides, refused):
    for call in ("causal", "prefix"):
        rc, msg = apart(call, lib, shape(lib, **strides), **over)
        assert (rc == 9 and "overlap" in msg) if refused else rc == 8, msg


@pytest.mark.parametrize("over,refused", [(dict(out=PK), True), (dict(out=PV + 16), True), (dict(plen=0, pk=OUT, pv=OUT), False),
                                          (dict(nkv=0, k=OUT, v=OUT), False), (dict(nkv=2, out=K + 512), False),
                                          (dict(nkv=2, out=K + 512 - 16), True)])
def test_outputs_over_the_prefix_or_keys_are_refused(lib, over, refused):
    rc, msg = apart("prefix", lib, shape(lib), **over)
    assert (rc == 9 and "overlap" in msg) if refused else rc == 8, msg


@pytest.mark.parametrize("over,refused", [
    (dict(), False), (dict(out=FAKE, n=64, out_stride=64), True), (dict(out=FAKE + 2 * 128), False), (dict(out=FAKE + 2 * 128 - 2), True),
    (dict(x_stride=128, out=FAKE + 128, out_stride=128), False), (dict(x_stride=128, out=FAKE + 126, out_stride=128), True),
    (dict(out=FAKE << 1), True), (dict(out=(FAKE << 1) + 8 * 32), False), (dict(out=(FAKE << 2) + 30), True), (dict(out=(FAKE << 2) + 32), False),
    (dict(mins=FAKE << 3), True), (dict(mins=(FAKE << 3) + 32), False), (dict(mins=(FAKE << 3) + 30), True)])
def test_linear_q4_outputs_over_inputs_are_refused(lib, over, refused):
    rc, msg = q4_call(lib, **over)
    assert (rc == 9 and "overlap" in msg) if refused else rc == 8, msg


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("k", [1152, 8192, 65536])
def test_the_4bit_bound_sees_what_is_lost(k, group, mins):
    """The bound that the GPU results are held to leaves no room for a stage of 256 weights, a group's minimum, one
    32-weight unit or another row's x."""
    import torch

    import operator_reference as ref
    g = torch.Generator().manual_seed(k + group)
    n, rows = 24, 3
    values = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand((n, k // group), generator=g) * 0.02 + 1e-3).half()
    lows = (torch.randn((n, k // group), generator=g) * 0.05).half() if mins else None
    x = torch.randn((rows, k), generator=g).half()
    want, bound = ref.linear_q4_by_steps(x, values, scales, lows)
    same, loose = ref.linear_q4(x, values, scales, lows)
    assert torch.allclose(want, same, rtol=0, atol=1e-9 * float(same.abs().max())) and (bound <= loose).all()

    def off(x=x, scales=scales, lows=lows):  # the share of outputs past the bound
        wrong, _ = ref.linear_q4(x, values, scales, lows)
        return float(((wrong - want).abs() > bound).double().mean())
    for at in (0, k // 2 // 256 * 256, (k - 1) // 256 * 256):
        lost = x.clone()
        lost[:, at:at + 256] = 0
        assert off(x=lost) > 0.8
        lost = x.clone()
        lost[:, at:at + 32] = 0
        assert off(x=lost) > 0.5
        if mins:
            less = lows.clone()
            less[:, at // group] = 0
            assert off(lows=less) > 0.25  # some minima are near 0, some sums of x too
    assert off(x=x[[1, 2, 0]]) > 0.9


def test_more_sequences_than_32_bit_offsets_reach_are_refused(lib):
    """(start, length) words are indexed in 32 bits: 2^30 sequences at most."""
    L = lib.lib()
    s = shape(lib)
    for nseq, code in ((1 << 30, 8), ((1 << 30) + 1, 9), ((1 << 31) - 1, 9)):  # 8: the device, which comes later
        assert L.ge_attention_causal(-1, ctypes.byref(s), Q, K, V, 8, FAKE, nseq, OUT, FAKE, 1 << 30, None) == code
        assert L.ge_attention_prefix(-1, ctypes.byref(s), Q, 8, K, V, 8, PK, PV, 4, FAKE, FAKE, nseq, OUT, FAKE, 1 << 30, None) == code
