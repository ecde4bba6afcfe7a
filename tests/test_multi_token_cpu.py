"""Refusals and host logic of the ops that take several new tokens at once: all of it before any device work."""

from __future__ import annotations

import math

import pytest
import torch

from deltaforge_b200 import _lib, ops

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def rotary_args(**over):
    a = dict(query=z(2, 3, 4, 32), key=z(2, 3, 2, 32), positions=z(2, 3, dtype=torch.int32), inv_freq=z(8, dtype=torch.float64), factor=1.0, interleaved=False)
    return {**a, **over}


def append_args(**over):
    a = dict(value=z(2, 3, 2, 32), key_cache=z(2, 2, 16, 32), value_cache=z(2, 2, 16, 32), cache_len=z(2, dtype=torch.int32))
    return {**rotary_args(), **a, **over}


@pytest.mark.parametrize(
    "over,match",
    [
        (dict(query=z(2, 3, 32)), "expected query and key"),
        (dict(key=z(2, 4, 2, 32)), "does not match query"),
        (dict(key=z(2, 3, 0, 32)), "at least one head"),
        (dict(key=z(2, 3, 2, 32, dtype=F16)), "must both be"),
        (dict(query=z(2, 3, 4, 32, dtype=torch.float64), key=z(2, 3, 2, 32, dtype=torch.float64)), "must both be"),
        (dict(positions=z(2, 3, dtype=F32)), "positions must be int32 or int64"),
        (dict(positions=z(2, 4, dtype=torch.int32)), "positions must be int32 or int64"),
        (dict(positions=z(3, 2, dtype=torch.int32).t()), "must be contiguous"),
        (dict(inv_freq=z(8, dtype=BF16)), "inv_freq must be"),
        (dict(inv_freq=z(17, dtype=F32)), "rotary_dim 34"),
        (dict(inv_freq=z(0, dtype=F32)), "rotary_dim 0"),
        (dict(query=z(2, 3, 32, 4).transpose(2, 3)), "last dimension contiguous"),
    ],
)
def test_rotary_refusals(over, match):
    with pytest.raises(ValueError, match=match):
        ops.rotary_qk(**rotary_args(**over))


@pytest.mark.parametrize(
    "over,match",
    [
        (dict(value=z(2, 3, 1, 32)), "must match key"),
        (dict(key_cache=z(2, 2, 16)), "caches must both be"),
        (dict(value_cache=z(2, 2, 15, 32)), "caches must both be"),
        (dict(key_cache=z(2, 3, 16, 32), value_cache=z(2, 3, 16, 32)), "do not match batch"),
        (dict(key_cache=z(2, 2, 16, 32, dtype=F16)), "caches must be"),
        (dict(cache_len=z(2, dtype=torch.int64)), "cache_len must be"),
        (dict(cache_len=z(3, dtype=torch.int32)), "cache_len must be"),
        (dict(key_cache=z(1, 2, 16, 32).expand(2, 2, 16, 32)), "expanded"),
    ],
)
def test_rotary_append_refusals(over, match):
    with pytest.raises(ValueError, match=match):
        ops.rotary_append(**append_args(**over))


def tree_args(**over):
    a = dict(query=z(2, 5, 4, 64), key_cache=z(2, 2, 16, 64), value_cache=z(2, 2, 16, 64), cache_len=z(2, dtype=torch.int32), parents=z(2, 5, dtype=torch.int32), scale=0.125)
    return {**a, **over}


@pytest.mark.parametrize(
    "over,match",
    [
        (dict(query=z(2, 5, 64)), "expected query"),
        (dict(query=z(2, 5, 4, 64, dtype=F32)), "bfloat16 or float16"),
        (dict(query=z(2, 5, 3, 64)), "do not divide"),
        (dict(query=z(2, 5, 4, 96), key_cache=z(2, 2, 16, 96), value_cache=z(2, 2, 16, 96)), "head dim 96"),
        (dict(query=z(2, 5, 4, 64, dtype=F16)), "caches must be"),
        (dict(key_cache=z(3, 2, 16, 64), value_cache=z(3, 2, 16, 64)), "do not match batch"),
        (dict(key_cache=z(2, 2, 0, 64), value_cache=z(2, 2, 0, 64)), "one cache row"),
        (dict(parents=z(2, 4, dtype=torch.int32)), "parents must be"),
        (dict(parents=z(2, 5, dtype=torch.int64)), "parents must be"),
        (dict(query=z(2, 65, 4, 64), parents=z(65, dtype=torch.int32)), "at most 64 nodes"),
        (dict(key_cache=z(2, 2, 16, 68)[..., :64]), "16-byte boundaries"),
        (dict(cache_len=z(2, 1, dtype=torch.int32)), "cache_len must be"),
    ],
)
def test_tree_attention_refusals(over, match):
    with pytest.raises(ValueError, match=match):
        ops.tree_attention(**tree_args(**over))


def delta_args(**over):
    a = dict(
        state=z(2, 4, 16, 24, dtype=F32), query=z(2, 5, 2, 16), key=z(2, 5, 2, 16), value=z(2, 5, 4, 24), g=z(2, 5, 4, dtype=F32), beta=z(2, 5, 4, dtype=F32),
        lengths=None, qk_l2norm=True,
    )  # fmt: skip
    return {**a, **over}


@pytest.mark.parametrize(
    "over,match",
    [
        (dict(state=z(2, 4, 16, 24)), "state must be fp32"),
        (dict(state=z(4, 16, 24, dtype=F32)), "state must be fp32"),
        (dict(key=z(2, 4, 2, 16)), "query and key must be"),
        (dict(query=z(2, 5, 3, 16), key=z(2, 5, 3, 16)), "do not divide"),
        (dict(query=z(2, 5, 0, 16), key=z(2, 5, 0, 16)), "do not divide"),
        (dict(value=z(2, 5, 4, 16)), "value has shape"),
        (dict(value=z(2, 5, 4, 24, dtype=F16)), "must be bfloat16"),
        (dict(g=z(2, 5, 2, dtype=F32)), "g must be"),
        (dict(beta=z(2, 5, 4, dtype=torch.int32)), "beta must be"),
        (dict(lengths=z(3, dtype=torch.int32)), "lengths must be"),
        (dict(lengths=z(2, dtype=torch.int64)), "lengths must be"),
        (dict(state=z(2, 4, 12, 24, dtype=F32), query=z(2, 5, 2, 12), key=z(2, 5, 2, 12)), "key dim 12"),
        (dict(state=z(2, 4, 136, 24, dtype=F32), query=z(2, 5, 2, 136), key=z(2, 5, 2, 136)), "key dim 136"),
        (dict(state=z(2, 4, 16, 20, dtype=F32), value=z(2, 5, 4, 20)), "value dim 20"),
    ],
)
def test_delta_rule_refusals(over, match):
    with pytest.raises(ValueError, match=match):
        ops.delta_rule_chunk(**delta_args(**over))


def test_delta_tree_refusals():
    a = delta_args()
    del a["lengths"]
    with pytest.raises(ValueError, match="parents must be"):
        ops.delta_rule_tree(**a, parents=z(2, 4, dtype=torch.int32))
    a.update(query=z(2, 65, 2, 16), key=z(2, 65, 2, 16), value=z(2, 65, 4, 24), g=z(2, 65, 4, dtype=F32), beta=z(2, 65, 4, dtype=F32))
    with pytest.raises(ValueError, match="at most 64 nodes"):
        ops.delta_rule_tree(**a, parents=z(2, 65, dtype=torch.int32))


def test_cpu_tensors_are_refused():
    d = delta_args()
    del d["lengths"]
    for call in (
        lambda: ops.rotary_qk(**rotary_args()),
        lambda: ops.rotary_append(**append_args()),
        lambda: ops.tree_attention(**tree_args()),
        lambda: ops.delta_rule_chunk(**delta_args()),
        lambda: ops.delta_rule_tree(**d, parents=z(2, 5, dtype=torch.int32)),
    ):
        with pytest.raises(RuntimeError, match="no PyTorch fallback"):
            call()


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    assert lib.dfb_rotary(None, None) == 2 and lib.dfb_tree_attention(None, None) == 2 and lib.dfb_delta_chunk(None, None) == 2
    r = _lib.RotaryDesc()
    r.batch = r.tokens = r.hq = r.hkv = 1
    r.d, r.rotary_dim = 8, 3
    assert lib.dfb_rotary(r, None) == 2 and b"even" in lib.dfb_last_error()
    r.rotary_dim = 4
    assert lib.dfb_rotary(r, None) == 2 and b"null" in lib.dfb_last_error()
    t = _lib.TreeAttnDesc()
    t.batch = t.nodes = t.hq = t.hkv = 1
    t.d, t.max_seq = 48, 8
    assert lib.dfb_tree_attention(t, None) == 2 and b"head dim" in lib.dfb_last_error()
    t.d, t.nodes = 64, 65
    assert lib.dfb_tree_attention(t, None) == 2 and b"at most 64" in lib.dfb_last_error()
    t.nodes, t.max_seq = 1, 4096
    t.q = t.kcache = t.vcache = t.cache_len = t.parents = t.out = 16  # never dereferenced: the scratch check comes first
    need = lib.dfb_tree_attn_scratch_bytes(1, 1, 1, 1, 64, 4096)
    assert need > 0
    assert lib.dfb_tree_attention(t, None) == 2 and b"scratch" in lib.dfb_last_error()
    d = _lib.DeltaChunkDesc()
    d.batch = d.tokens = d.hk = d.hv = 1
    d.dk, d.dv = 12, 16
    assert lib.dfb_delta_chunk(d, None) == 2 and b"unsupported" in lib.dfb_last_error()
    d.dk, d.tokens = 16, 64
    d.state = d.state_out = d.q = d.k = d.v = d.g = d.beta = d.out = 16
    assert lib.dfb_delta_chunk(d, None) == 2 and b"scratch" in lib.dfb_last_error()
    d.parents, d.lengths = 16, 16
    assert lib.dfb_delta_chunk(d, None) == 2 and b"no lengths" in lib.dfb_last_error()


def test_scratch_sizes():
    lib = _lib.load()
    assert lib.dfb_delta_chunk_scratch_bytes(1, 64, 16, 32, 128, 128, 0) == 16 * 32768 + 32 * (8 * 8192 + 768)
    # a long prompt is walked in segments: the scratch stays bounded
    assert lib.dfb_delta_chunk_scratch_bytes(1, 1 << 20, 16, 32, 128, 128, 0) <= 256 << 20
    assert lib.dfb_delta_chunk_scratch_bytes(16, 1, 16, 32, 128, 128, 0) == 0  # token by token
    assert lib.dfb_delta_chunk_scratch_bytes(16, 1, 16, 32, 128, 128, 1) > 0
    assert lib.dfb_delta_chunk_scratch_bytes(0, 5, 1, 1, 8, 8, 0) == 0
    assert lib.dfb_tree_attn_scratch_bytes(64, 1, 16, 4, 256, 32) == 0  # one split


def test_rope_frequencies():
    f, factor = ops.rope_frequencies(64, 1e7, device="cpu")
    want = [1e7 ** (-2 * i / 64) for i in range(32)]
    assert factor == 1.0 and f.dtype == torch.float64 and torch.allclose(f, torch.tensor(want, dtype=torch.float64), rtol=1e-15)
    lin, _ = ops.rope_frequencies(64, 1e7, stretch=4.0, method="linear", device="cpu")
    assert torch.equal(lin, f / 4)
    base, _ = ops.rope_frequencies(64, 1e7, stretch=4.0, method="base", device="cpu")
    assert base[0] == 1.0 and math.isclose(base[-1], f[-1] / 4, rel_tol=1e-12)
    parts, factor = ops.rope_frequencies(64, 1e7, stretch=4.0, trained_len=32768, device="cpu")
    turns = 32768 * f / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], f[turns >= 32]) and torch.allclose(parts[turns <= 1], f[turns <= 1] / 4, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and bool(((parts < f) & (parts > f / 4))[between].all()) and math.isclose(factor, 0.1 * math.log(4) + 1)
    for bad in (dict(rotary_dim=3), dict(stretch=0.5), dict(method="other"), dict(fast_turns=1.0)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**{"rotary_dim": 64, "theta": 1e4, "device": "cpu", **bad})


def test_fake_kernels_give_shapes():
    with torch._subclasses.fake_tensor.FakeTensorMode():
        r = rotary_args()
        q, k = torch.ops.dfb200.rotary_qk(**{n: torch.empty(t.shape, dtype=t.dtype) if isinstance(t, torch.Tensor) else t for n, t in r.items()})
        assert q.shape == (2, 3, 4, 32) and k.shape == (2, 3, 2, 32)
        t = {n: torch.empty(x.shape, dtype=x.dtype) if isinstance(x, torch.Tensor) else x for n, x in tree_args().items()}
        assert torch.ops.dfb200.tree_attention(**t).shape == (2, 5, 4, 64)
        d = {n: torch.empty(x.shape, dtype=x.dtype) if isinstance(x, torch.Tensor) else x for n, x in delta_args().items()}
        out, state = torch.ops.dfb200.delta_rule_chunk(**d)
        assert out.shape == (2, 5, 4, 24) and out.dtype == BF16 and state.shape == (2, 4, 16, 24) and state.dtype == F32


@pytest.mark.parametrize("source,kernel", [("tree_attention.cu", "tree_merge_kernel"), ("tree_attention_tc.cu", "tree_tc_merge_kernel")])
def test_merge_kernels_wait_before_any_return(source, kernel):
    """They are launched while the attention grid still runs, and what follows in the stream is ordered behind them alone: a
    thread that returned before the wait could let it read an output that is still being written."""
    text = (_lib._build.CSRC / source).read_text()
    body = text[text.index(f" {kernel}(const") :]
    body = body[: body.index("\n}\n")]
    assert body.count("pdl_wait();") == 1
    assert "return" not in body[: body.index("pdl_wait();")]


def test_tree_attention_orders_its_stores_before_the_next_units_copies():
    """A unit's end writes the ring by ordinary stores, and the next unit's copies go to the same bytes through the async proxy:
    the writers' fence stands before the barrier that lets the loading warp go on."""
    text = (_lib._build.CSRC / "tree_attention_tc.cu").read_text()
    end = text.index("queries, O and the flags may be written again")
    written = text.rindex("*(float4*)(stage", 0, end)
    barrier = text.rindex("__syncthreads();", 0, end)
    assert "fence_async();" in text[written:barrier]


@pytest.mark.parametrize("source,kernel", [("tree_attention_tc.cu", "tree_attention_tc_kernel"), ("delta_scan.cu", "delta_scan_kernel")])
def test_a_wait_that_ran_out_leaves_nothing_under_way(source, kernel):
    """Copies into shared memory and products in tensor memory that a kernel has started end before it gives that memory back."""
    text = (_lib._build.CSRC / source).read_text()
    body = text[text.index(f" {kernel}(const") :]
    body = body[: body.index("\n}\n")]
    assert "wait_out(&full[" in body
    end = body[body.rindex("if (*failed)") : body.index("tcgen05.dealloc")]
    assert "commit(&drained);" in end and "wait_out(&drained, 0);" in end
    assert "__syncthreads();" in end[end.index("wait_out(&drained") :]


# ---------------------------------------------------------------- the wrapper that passes the dispatcher by


def _read(x):
    import ctypes

    return list((ctypes.c_float * x.numel()).from_address(x.data_ptr()))


@ops._eager
@torch.library.custom_op("dfb200_test::weighted", mutates_args=())
def weighted(query: torch.Tensor, key: torch.Tensor, factor: float, lengths: torch.Tensor | None) -> torch.Tensor:
    """An op under the wrapper that runs here, and that like those of the package reads memory."""
    return torch.tensor([factor * a + b for a, b in zip(_read(query), _read(key))]).view(query.shape)


@weighted.op.register_fake
def _(query, key, factor, lengths):
    return query.new_empty(query.shape)


@ops._eager
@torch.library.custom_op("dfb200_test::append_one", mutates_args=("key_cache", "value_cache"))
def append_one(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor) -> torch.Tensor:
    key_cache.data.add_(1.0)  # (past the version counter, as a kernel writes)
    value_cache.data.add_(1.0)
    return query.clone()


@append_one.op.register_fake
def _(query, key_cache, value_cache):
    return query.new_empty(query.shape)


def call_weighted(a, b):
    return weighted(a, b, 2.0, None)


def pair(seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(3, 4, generator=g), torch.randn(3, 4, generator=g)


def test_wrapper_calls_the_function_itself_for_plain_tensors(monkeypatch):
    a, b = pair()
    with monkeypatch.context() as m:  # the op is not called
        m.setattr(type(weighted.op), "__call__", lambda *x: pytest.fail("went through the dispatcher"))
        assert torch.equal(call_weighted(a, b), 2 * a + b)
        assert torch.equal(weighted(torch.nn.Parameter(a, requires_grad=False), b, 2.0, None), 2 * a + b)
        with torch.no_grad():
            assert torch.equal(weighted(a.clone().requires_grad_(), b, 2.0, None), 2 * a + b)
    assert torch.equal(weighted(a, key=b, factor=2.0, lengths=None), 2 * a + b)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_wrapper_under_a_jit_trace():
    a, b = pair()
    traced = torch.jit.trace(call_weighted, (a, b))
    a, b = pair(1)
    assert torch.equal(traced(a, b), 2 * a + b)
    assert "dfb200_test::weighted" in str(traced.graph)


def test_wrapper_under_compilation():
    a, b = pair()
    compiled = torch.compile(call_weighted, fullgraph=True, backend="eager")
    assert torch.equal(compiled(a, b), 2 * a + b)


def test_wrapper_sees_negative_views():
    a, b = pair()
    for x, y in ((torch._neg_view(a), b), (a, torch._neg_view(b)), (torch.complex(b, a).conj().imag.view(-1)[:1], b[0, :1])):
        assert x.is_neg() or y.is_neg()
        assert torch.equal(call_weighted(x, y), 2 * x + y)


def test_wrapper_under_a_function_mode():
    class Seen(torch.overrides.TorchFunctionMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    a, b = pair()
    with Seen() as seen:
        out = call_weighted(a, b)
    assert torch.equal(out, 2 * a + b) and any("weighted" in x for x in seen.names)


@pytest.mark.filterwarnings("ignore")
def test_wrapper_under_vmap_and_with_gradients_meta_and_fake_tensors():
    a, b = pair()
    assert torch.equal(torch.func.vmap(call_weighted)(a, b), 2 * a + b)
    x = a.clone().requires_grad_()
    y = call_weighted(x, b)
    assert y.requires_grad and y.grad_fn is not None  # the op: it says at the backward pass that it has none
    with pytest.raises(Exception, match="autograd|backward|Autograd"):
        y.sum().backward()
    assert call_weighted(a.to("meta"), b.to("meta")).is_meta
    with torch._subclasses.fake_tensor.FakeTensorMode() as mode:
        assert call_weighted(mode.from_tensor(a), mode.from_tensor(b)).shape == a.shape


def test_wrapper_moves_the_version_counters_of_what_an_op_writes():
    q, kc, vc = torch.zeros(2), torch.zeros(3), torch.zeros(3)
    for n in range(1, 4):
        append_one(q, kc, vc)
        assert kc._version == vc._version == n and q._version == 0 and kc[0] == n
    with torch.inference_mode():
        inner = torch.zeros(3)
        append_one(q, kc, inner)  # (an inference tensor has no version)
    assert kc._version == 4 and inner[0] == 1


def test_remembered_scratch_sizes_are_bounded():
    assert ops._scratch_bytes.cache_info().maxsize is not None
    for tokens in range(65, 65 + 2 * ops._scratch_bytes.cache_info().maxsize):
        ops._scratch_bytes("dfb_delta_chunk_scratch_bytes", 1, tokens, 2, 4, 128, 128, 0)
    assert ops._scratch_bytes.cache_info().currsize <= ops._scratch_bytes.cache_info().maxsize
    assert ops._scratch_bytes("dfb_delta_chunk_scratch_bytes", 1, 64, 16, 32, 128, 128, 0) == _lib.load().dfb_delta_chunk_scratch_bytes(1, 64, 16, 32, 128, 128, 0)


def test_strides_of_dimensions_of_one_may_be_anything():
    """A cache of one sequence, of one head or of one row, cut out of a buffer whose other strides are odd."""
    for shape, stride in (((1, 2, 16, 64), (4097, 1024, 64, 1)), ((2, 1, 16, 64), (1024, 33, 64, 1)), ((2, 2, 1, 64), (128, 64, 65, 1))):
        cache = torch.empty_strided(shape, stride, dtype=BF16).zero_()
        n, hkv, _, _ = shape
        a = tree_args(query=z(n, 5, 4, 64), key_cache=cache, value_cache=cache, cache_len=z(n, dtype=torch.int32), parents=z(n, 5, dtype=torch.int32))
        with pytest.raises(RuntimeError, match="no PyTorch fallback"):  # past all that is checked before the device
            ops.tree_attention(**a)
    one = torch.empty_strided((1, 1, 4, 64), (3, 5, 64, 1), dtype=BF16)
    assert ops._aligned_rows(one) is one and ops._aligned_rows(one, expanded=False) is one
    assert ops._aligned_rows(z(1, 1, 4, 72)[..., 4:68]) is not one
    wide = z(2, 1, 1, 64).expand(2, 3, 4, 64)
    assert ops._aligned_rows(wide) is wide and ops._aligned_rows(wide, expanded=False).is_contiguous()
    odd = torch.zeros(2, 3, 4, 68, dtype=BF16)[..., :64]
    assert ops._aligned_rows(odd) is not odd


def rotary_desc(hq, hkv, d, rotary_dim, dtype=2):
    r = _lib.RotaryDesc()
    r.batch = r.tokens = 1
    r.hq, r.hkv, r.d, r.rotary_dim, r.dtype = hq, hkv, d, rotary_dim, dtype
    r.q = r.k = r.pos = r.inv_freq = r.q_out = r.k_out = 16  # never dereferenced: there is no device, or the check comes first
    for s in (r.q_stride, r.k_stride):
        s[0], s[1], s[2] = hq * d, hq * d, d
    return r


def wrong_quotients(n, heads):
    """Whether some x below heads * n has x * ceil(2^32 / n) >> 32 != x / n: the kernel's division, tried at the ends of all heads"""
    m = -(-(1 << 32) // n)
    return any(x * m >> 32 != x // n for h in range(heads) for x in (h * n, h * n + n - 1))


@pytest.mark.parametrize("hq,hkv,d,rotary_dim", [(16, 4, 256, 64), (60, 4, 12011, 8), (40, 40, 8192 + 512, 512), (1, 1, 70001, 2), (32, 32, 4096, 4096 // 8), (200, 8, 6000, 6)])
def test_rotary_refuses_heads_whose_division_is_not_exact(hq, hkv, d, rotary_dim):
    if torch.cuda.is_available():
        pytest.skip("descriptors without memory behind them are for machines without a device")
    lib = _lib.load()
    vec = 4 if d % 4 == 0 and rotary_dim % 8 == 0 else 1  # fp32 vectors of 16 bytes
    n = (d - rotary_dim) // vec
    if not wrong_quotients(n, hq + hkv):
        assert lib.dfb_rotary(rotary_desc(hq, hkv, d, rotary_dim), None) != 2
        return
    assert lib.dfb_rotary(rotary_desc(hq, hkv, d, rotary_dim), None) == 2 and b"too many" in lib.dfb_last_error()
