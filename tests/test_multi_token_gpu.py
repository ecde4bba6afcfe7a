"""The ops that take several new tokens of a sequence at once, against plain 64-bit implementations of their definitions.

Tolerances are counted in roundings. A rounding to type t moves a value by at most h(t) = finfo(t).eps / 2 relative to it.

* rotary: one rounding of the result, h(t)|x'|, plus fp32 arithmetic on cos, sin (argument, function, product, sum: at most
  8 roundings of terms no larger than |x| + |y|): 8 h(fp32) (|x| + |y|) factor.
* tree attention: the result's rounding h(t)|o|; probabilities rounded to t: h(t) sum p|v|; scores in fp32: an error ds <= 2 D h(fp32)
  scale |q|.|k| (largest over the test) and the exponential's 2^-21 change each p by ds + 2^-21 relative, twice (numerator, sum), and
  accumulation over n keys by n h(fp32): (2 ds + 2^-20 + n 2^-24) sum p|v|.
* delta rule, output: its rounding h(bf16)|o|; q S with S in 11 bits: h(fp16) |q|.|S|; P V' with both in 11 bits: 2 h(fp16) |P|.|V'|. The
  absolute sums are bounded through the recurrence run on absolute values of the terms that a step adds (see _scale).
* delta rule, state: operands in 22 bits, three products in a row, fp32 sums of 128 + 64 terms: (3 * 2 * 2^-22 + 192 * 2^-24)
  per chunk, at most as many chunks as there are, relative to the largest |state| of the head.
"""

from __future__ import annotations

import pytest
import torch

from deltaforge_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32, F64, I32 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32
DEV = "cuda"


def half(t):
    return torch.finfo(t).eps / 2


def rnd(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def at_odd_offset(x):
    """The same tensor, contiguous, three elements into its storage."""
    return torch.cat((x.new_zeros(3), x.flatten()))[3:].view(x.shape)


def within(got, want, bound):
    assert got.shape == want.shape
    bad = int((~torch.isfinite(got.double())).sum())
    assert bad == 0, f"{bad} values are not finite"
    err = (got.double() - want).abs()
    excess, worst = (err - bound).max().item(), err.max().item()
    assert excess <= 0, f"worst excess {excess:.3g}, worst error {worst:.3g}"


# ---------------------------------------------------------------- rotary positions


def rotary_ref(x, pos, inv, factor, interleaved):
    """(rotated in 64 bits, |x| + |y| of each element's pair)"""
    r = 2 * inv.numel()
    a = pos.double()[:, :, None, None] * inv.double()
    c, s = a.cos() * factor, a.sin() * factor
    y, size = x.double().clone(), torch.zeros_like(x, dtype=F64)
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, w = x.double()[..., lo], x.double()[..., hi]
    y[..., lo], y[..., hi] = u * c - w * s, w * c + u * s
    size[..., lo] = size[..., hi] = (u.abs() + w.abs()) * factor
    return y, size


def rotary_bound(want, size, dtype):
    return half(dtype) * want.abs() + 8 * half(F32) * (1 + half(dtype)) * size


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize(
    "b,t,hq,hkv,d,r,start",
    [(1, 1, 16, 4, 256, 64, 4096), (2, 5, 3, 1, 32, 32, 0), (1, 130, 2, 2, 64, 16, 250000), (3, 7, 5, 2, 40, 12, 77), (1, 2, 1, 1, 10, 6, 2**31 - 9), (1, 3, 2, 1, 512, 512, 100000)],
)
def test_rotary_qk(b, t, hq, hkv, d, r, start, dtype, interleaved):
    q, k = rnd(1, b, t, hq, d, dtype=dtype), rnd(2, b, t, hkv, d, dtype=dtype)
    pos = (start + torch.arange(t)[None] + torch.arange(b)[:, None]).to(torch.int64 if start > 2**30 else I32).to(DEV)
    inv, factor = ops.rope_frequencies(r, 1e4, stretch=2.0)
    q0, k0 = q.clone(), k.clone()
    for got, x in zip(ops.rotary_qk(q, k, pos, inv, factor, interleaved), (q, k)):
        want, size = rotary_ref(x, pos, inv, factor, interleaved)
        within(got, want, rotary_bound(want, size, dtype))
        assert torch.equal(got[..., r:], x[..., r:]) and got.dtype == dtype
    assert torch.equal(q, q0) and torch.equal(k, k0)


def test_rotary_reads_views_of_a_fused_row_and_transposed_heads():
    b, t, hq, hkv, d = 2, 9, 4, 2, 64
    row = rnd(3, b, t, (hq + 2 * hkv) * d + 3, dtype=BF16)  # an odd row width: rows start anywhere
    q, k = row[..., 1 : 1 + hq * d].unflatten(-1, (hq, d)), row[..., 1 + hq * d : 1 + (hq + hkv) * d].unflatten(-1, (hkv, d))
    pos = torch.arange(t, dtype=I32, device=DEV).expand(b, t)
    inv, factor = ops.rope_frequencies(32, 1e7)
    for got, x in zip(ops.rotary_qk(q, k, pos, inv, factor, False), (q, k)):
        want, size = rotary_ref(x, pos, inv, factor, False)
        within(got, want, rotary_bound(want, size, BF16))
    heads_first = rnd(4, b, hq, t, d, dtype=BF16)
    got, _ = ops.rotary_qk(heads_first.transpose(1, 2), k, pos, inv.float(), factor, True)
    want, size = rotary_ref(heads_first.transpose(1, 2), pos, inv.float(), factor, True)
    within(got, want, rotary_bound(want, size, BF16))


@pytest.mark.parametrize("dtype,d,r", [(BF16, 256, 64), (F32, 24, 24)])
def test_rotary_append_writes_its_rows_and_no_others(dtype, d, r):
    b, t, hq, hkv, rows = 3, 6, 4, 2, 16
    q, k, v = rnd(5, b, t, hq, d, dtype=dtype), rnd(6, b, t, hkv, d, dtype=dtype), rnd(7, b, t, hkv, d, dtype=dtype)
    kc, vc = rnd(8, b, hkv, rows, d, dtype=dtype), rnd(9, b, hkv, rows, d, dtype=dtype)
    k0, v0 = kc.clone(), vc.clone()
    lens = torch.tensor([0, rows - 4, -2], dtype=I32, device=DEV)  # whole, past the end after four rows, before the start
    pos = torch.arange(b * t, dtype=torch.int64, device=DEV).view(b, t)
    inv, factor = ops.rope_frequencies(r, 1e6)
    got = ops.rotary_append(q, k, v, pos, inv, factor, False, kc, vc, lens)
    want, size = rotary_ref(q, pos, inv, factor, False)
    within(got, want, rotary_bound(want, size, dtype))
    _, k_rot = ops.rotary_qk(q, k, pos, inv, factor, False)
    for i, n in enumerate(lens.tolist()):
        for j in range(t):
            if 0 <= n + j < rows:
                k0[i, :, n + j], v0[i, :, n + j] = k_rot[i, j], v[i, j]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_rotary_of_nothing():
    inv, factor = ops.rope_frequencies(16, 1e4)
    q, k = ops.rotary_qk(rnd(1, 2, 0, 4, 32, dtype=BF16), rnd(1, 2, 0, 2, 32, dtype=BF16), torch.zeros((2, 0), dtype=I32, device=DEV), inv, factor, False)
    assert q.shape == (2, 0, 4, 32) and k.shape == (2, 0, 2, 32)


# ---------------------------------------------------------------- trees


def paths(parents):
    """Per row its ancestors and itself, oldest first; None where the row holds no node."""
    found = []
    for i, p in enumerate(parents):
        found.append(None if p < -1 or p >= i else ([] if p == -1 or found[p] is None else found[p]) + [i])
    return found


def random_tree(seed, n):
    g = torch.Generator().manual_seed(seed)
    return [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(n)]


def tree_ref(q, kc, vc, lens, parents, scale):
    """(output, sum p|v|) in 64 bits, keys gathered row by row"""
    b, n, hq, d = q.shape
    hkv, rows = kc.shape[1], kc.shape[2]
    out, size = torch.zeros(b, n, hq, d, dtype=F64, device=DEV), torch.zeros(b, n, hq, d, dtype=F64, device=DEV)
    for i in range(b):
        for j, path in enumerate(paths(parents[i])):
            if path is None:
                continue
            at = [r for r in list(range(lens[i])) + [lens[i] + x for x in path] if r < rows]
            if not at:
                continue
            kk, vv = kc[i, :, at].double(), vc[i, :, at].double()
            s = torch.einsum("hgd,hkd->hgk", q[i, j].double().view(hkv, hq // hkv, d), kk) * scale
            p = torch.softmax(s, -1)
            out[i, j] = (p @ vv).reshape(hq, d)
            size[i, j] = (p @ vv.abs()).reshape(hq, d)
    return out, size


def tree_bound(want, size, q, kc, scale, n_keys):
    dt, d = q.dtype, q.shape[-1]
    longest = q.double().norm(dim=-1).max() * kc.double().nan_to_num(0, 0, 0).norm(dim=-1).max()  # |q|.|k| is at most this
    ds = 2 * d * half(F32) * scale * longest.item()
    return half(dt) * want.abs() + (half(dt) + 2 * ds + 2**-20 + n_keys * 2**-24) * size * (1 + 2**-6)


TREES = {
    "one": lambda n: [-1] * n,
    "chain": lambda n: list(range(-1, n - 1)),
    "random": lambda n: random_tree(n, n),
    "star": lambda n: [-1] + [0] * (n - 1),
}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(
    "b,n,hq,hkv,d,rows,lens,tree",
    [
        (1, 1, 16, 4, 256, 70, [64], "one"),
        (2, 16, 16, 4, 256, 400, [383, 1], "random"),
        (1, 64, 16, 4, 256, 300, [200], "random"),
        (3, 7, 8, 8, 128, 90, [0, 31, 83], "chain"),
        (2, 33, 4, 1, 64, 1200, [1000, 64], "random"),
        (2, 64, 2, 1, 32, 4096, [4032, 17], "star"),
        (1, 5, 24, 2, 64, 8, [3], "random"),
        (2, 3, 3, 3, 32, 2, [0, 0], "chain"),  # more nodes than rows: keys past the cache are lost
        (3, 33, 2, 2, 64, 7, [0, 0, 7], "random"),  # and so do nodes whose whole path lies there: zeros
        (2, 13, 2, 2, 32, 1, [0, 1], "one"),
        (2, 40, 4, 1, 256, 5, [0, 2], "one"),
        # heads enough for the form that reads the cache once for 128 rows
        (8, 12, 16, 4, 256, 300, [288, 0, 1, 127, 128, 129, 250, 90], "random"),
        (9, 64, 12, 4, 128, 200, [136, 0, 63, 64, 65, 100, 1, 128, 31], "random"),
        (16, 9, 8, 4, 64, 700, [691, 0, 5, 130, 600, 64, 63, 384] * 2, "chain"),
        (11, 17, 3, 3, 256, 20, [3] * 11, "star"),
        (9, 33, 8, 4, 64, 1, [1, 1, 1, 0, 0, 0, 0, 0, 0], "one"),
        (4, 48, 16, 16, 128, 130, [0, 100, 130, 127], "one"),
        (1, 16, 16, 4, 128, 20000, [19984], "random"),
    ],
)
def test_tree_attention(b, n, hq, hkv, d, rows, lens, tree, dtype):
    q = rnd(11, b, n, hq, d, dtype=dtype)
    kc, vc = rnd(12, b, hkv, rows, d, dtype=dtype), rnd(13, b, hkv, rows, d, dtype=dtype)
    parents = [TREES[tree](n) for _ in range(b)]
    scale = d**-0.5
    want, size = tree_ref(q, kc, vc, lens, parents, scale)
    for i, m in enumerate(lens):  # what lies behind the tree is never read
        kc[i, :, m + n :], vc[i, :, m + n :] = torch.nan, torch.inf
    got = ops.tree_attention(q, kc, vc, torch.tensor(lens, dtype=I32, device=DEV), torch.tensor(parents, dtype=I32, device=DEV), scale)
    within(got, want, tree_bound(want, size, q, kc, scale, rows))


@pytest.mark.parametrize("hq,hkv,d", [(16, 4, 256), (4, 2, 64), (44, 11, 256), (32, 16, 64)])
def test_tree_attention_rows_without_a_node_and_values_no_one_sees(hq, hkv, d):
    b, n, rows = 3, 12, 80
    q, kc, vc = rnd(21, b, n, hq, d, dtype=BF16), rnd(22, b, hkv, rows, d, dtype=BF16), rnd(23, b, hkv, rows, d, dtype=BF16)
    lens = [50, 0, 13]
    # sequence 0: rows 9.. hold no node; 1: none does; 2: a node whose parent is an empty row hangs on the prefix
    parents = [[-1, 0, 0, 1, 1, 2, -1, 6, 6] + [-2] * 3, [-2] * n, [-1, 0, 7, 2, -5, 4, 5, 3, 99, 8, 9, 1]]
    want, size = tree_ref(q, kc, vc, lens, parents, 0.1)
    bound = tree_bound(want, size, q, kc, 0.1, rows)
    lt, pt = torch.tensor(lens, dtype=I32, device=DEV), torch.tensor(parents, dtype=I32, device=DEV)
    empty = torch.tensor([[p is None for p in paths(x)] for x in parents], device=DEV)
    got = ops.tree_attention(q, kc, vc, lt, pt, 0.1)
    within(got, want, bound)
    assert bool((got[empty] == 0).all())
    # a leaf's key and value turn to NaN and infinity: only the leaf itself changes
    for leaf, bad_k, bad_v in ((4, torch.nan, 1.0), (4, 1.0, torch.inf), (8, torch.nan, torch.nan), (5, 1.0, -torch.inf)):
        k2, v2 = kc.clone(), vc.clone()
        k2[0, :, lens[0] + leaf] *= bad_k
        v2[0, :, lens[0] + leaf] *= bad_v
        g2 = ops.tree_attention(q, k2, v2, lt, pt, 0.1)
        others = torch.ones(b, n, dtype=torch.bool, device=DEV)
        others[0, leaf] = False
        within(g2[others], want[others], bound[others])
        assert not bool(torch.isfinite(g2[0, leaf].float()).any())
    # an empty row's key and value may be anything
    k2, v2 = kc.clone(), vc.clone()
    k2[0, :, lens[0] + 9 : lens[0] + 12], v2[0, :, lens[0] + 9 : lens[0] + 12] = torch.inf, torch.nan
    assert torch.equal(ops.tree_attention(q, k2, v2, lt, pt, 0.1), got)


@pytest.mark.parametrize("hq,hkv", [(8, 2), (64, 16)])
def test_tree_attention_layouts_streams_and_graphs(hq, hkv):
    b, n, d, rows = 2, 9, 128, 700
    lens, parents = [600, 320], random_tree(5, n)
    q, kc, vc = rnd(31, b, n, hq, d, dtype=BF16), rnd(32, b, hkv, rows, d, dtype=BF16), rnd(33, b, hkv, rows, d, dtype=BF16)
    lt, pt = torch.tensor(lens, dtype=I32, device=DEV), torch.tensor(parents, dtype=I32, device=DEV)
    base = ops.tree_attention(q, kc, vc, lt, pt, 0.09)
    want, size = tree_ref(q, kc, vc, lens, [parents] * b, 0.09)
    within(base, want, tree_bound(want, size, q, kc, 0.09, rows))
    # heads first, rows of a wider buffer, one sequence's cache for both
    assert torch.equal(ops.tree_attention(q.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, lt, pt, 0.09), base)
    wide = torch.zeros(b, hkv, rows, 2 * d, dtype=BF16, device=DEV)
    wide[..., :d], wide[..., d:] = kc, vc
    assert torch.equal(ops.tree_attention(q, wide[..., :d], wide[..., d:], lt, pt.expand(b, n).contiguous(), 0.09), base)
    shared = ops.tree_attention(q, kc[:1].expand(b, -1, -1, -1), vc[:1].expand(b, -1, -1, -1), lt, pt, 0.09)
    within(shared[:1], want[:1], tree_bound(want, size, q, kc, 0.09, rows)[:1])  # (an expanded cache takes the other kernel)
    odd = rnd(31, b, n, hq, d + 1, dtype=BF16)[..., :d]  # rows on odd elements: copied
    assert torch.equal(ops.tree_attention(odd, kc, vc, lt, pt, 0.09), ops.tree_attention(odd.contiguous(), kc, vc, lt, pt, 0.09))
    assert torch.equal(ops.tree_attention(at_odd_offset(q), kc, vc, lt, pt, 0.09), base)
    # two streams at once, and a captured graph whose lengths change between replays
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got.append(ops.tree_attention(q, kc, vc, lt, pt, 0.09))
    torch.cuda.synchronize()
    assert all(torch.equal(x, base) for x in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.tree_attention(q, kc, vc, lt, pt, 0.09)
    for new in ([600, 320], [0, 691], [1, 5]):
        lt.copy_(torch.tensor(new, dtype=I32))
        graph.replay()
        assert torch.equal(out, ops.tree_attention(q, kc, vc, lt, pt, 0.09))


@pytest.mark.parametrize("hq,hkv,n", [(4, 2, 5), (40, 20, 30)])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_tree_attention_scales(hq, hkv, n, scale):
    b, d, rows = 2, 64, 200
    q, kc, vc = rnd(35, b, n, hq, d, dtype=F16, scale=0.5), rnd(36, b, hkv, rows, d, dtype=F16, scale=0.5), rnd(37, b, hkv, rows, d, dtype=F16)
    lens, parents = [150, 20], random_tree(9, n)
    want, size = tree_ref(q, kc, vc, lens, [parents] * b, scale)
    got = ops.tree_attention(q, kc, vc, torch.tensor(lens, dtype=I32, device=DEV), torch.tensor(parents, dtype=I32, device=DEV), scale)
    within(got, want, tree_bound(want, size, q, kc, abs(scale), rows))


@pytest.mark.parametrize("n,hq", [(3, 4), (20, 2)])
def test_offsets_past_32_bits_in_a_long_cache(n, hq):
    """One sequence of 9 million rows of 256: element offsets up to 2.3e9. All keys but a few are zero, so the scores are known."""
    d, rows = 256, 9_000_000
    kc, vc = torch.zeros(1, 1, rows, d, dtype=BF16, device=DEV), torch.zeros(1, 1, rows, d, dtype=BF16, device=DEV)
    q, k, v = rnd(38, 1, n, hq, d, dtype=BF16), rnd(39, 1, n, 1, d, dtype=BF16), rnd(40, 1, n, 1, d, dtype=BF16)
    at = [5, 8_388_609, 8_900_000]  # the second and the third lie past 2^31 elements
    kc[0, 0, at], vc[0, 0, at] = rnd(41, 3, d, dtype=BF16), rnd(42, 3, d, dtype=BF16)
    length = rows - n
    lens = torch.tensor([length], dtype=I32, device=DEV)
    inv, factor = ops.rope_frequencies(64, 1e6)
    pos = (length + torch.arange(n, dtype=I32, device=DEV))[None]
    tq = ops.rotary_append(q, k, v, pos, inv, factor, False, kc, vc, lens)
    assert torch.equal(kc[0, 0, length:], ops.rotary_qk(q, k, pos, inv, factor, False)[1][0, :, 0]) and torch.equal(vc[0, 0, length:], v[0, :, 0])
    scale = 0.25  # scores of about 4: the few rows and the millions of zeros both count
    got = ops.tree_attention(tq, kc, vc, lens, torch.arange(-1, n - 1, dtype=I32, device=DEV), scale)
    for i in range(n):
        seen = at + [length + j for j in range(i + 1)]
        s = torch.einsum("hd,kd->hk", tq[0, i].double(), kc[0, 0, seen].double()) * scale
        w = s.exp() / (s.exp().sum(-1, keepdim=True) + rows - n - len(at))
        want, size = w @ vc[0, 0, seen].double(), w @ vc[0, 0, seen].double().abs()
        # as in tree_bound; the sum of 9 million ones is exact below 2^24 and grows in steps of a tile's sum
        ds = 2 * d * half(F32) * scale * (tq.double().norm(dim=-1).max() * kc[0, 0, seen].double().norm(dim=-1).max()).item()
        within(got[0, i], want, half(BF16) * want.abs() + (half(BF16) + 2 * ds + 2**-20 + rows / 128 * 2**-24) * size * (1 + 2**-6))


# ---------------------------------------------------------------- the delta rule


def delta_inputs(seed, b, t, hk, hv, dk, dv, l2norm, rate=0.3):
    q, k, v = rnd(seed, b, t, hk, dk), rnd(seed + 1, b, t, hk, dk), rnd(seed + 2, b, t, hv, dv, dtype=BF16)
    k = k + 0.7 * rnd(seed + 6, 1, 1, hk, dk)  # keys with a direction in common, as activations have
    if not l2norm:
        q, k = q / q.norm(dim=-1, keepdim=True) * dk**-0.5, k / k.norm(dim=-1, keepdim=True)
    g = -rate * rnd(seed + 3, b, t, hv).abs()
    beta = torch.sigmoid(rnd(seed + 4, b, t, hv))
    return rnd(seed + 5, b, hv, dk, dv, scale=0.5), q.to(BF16), k.to(BF16), v, g, beta


def _normalised(q, k, hv, l2norm):
    q, k = q.double(), k.double()
    if l2norm:
        q = q / (q.square().sum(-1, keepdim=True) + 1e-6).sqrt() * q.shape[-1] ** -0.5
        k = k / (k.square().sum(-1, keepdim=True) + 1e-6).sqrt()
    return q.repeat_interleave(hv // q.shape[2], 2), k.repeat_interleave(hv // k.shape[2], 2)


def _step(s, size, q, k, v, g, beta):
    """One token; `size` follows the same recurrence with every term's absolute value (what roundings are relative to)."""
    s, size = s * g.exp()[..., None, None], size * g.exp()[..., None, None]
    d = (v - torch.einsum("...kv,...k->...v", s, k)) * beta[..., None]
    s = s + k[..., :, None] * d[..., None, :]
    size = size + k.abs()[..., :, None] * d.abs()[..., None, :]
    return s, size, torch.einsum("...kv,...k->...v", s, q), torch.einsum("...kv,...k->...v", size, q.abs())


def delta_ref(state, q, k, v, g, beta, lengths, l2norm):
    q, k = _normalised(q, k, v.shape[2], l2norm)
    s, size = state.double(), state.double().abs()
    out, osize = torch.zeros(v.shape, dtype=F64, device=DEV), torch.zeros(v.shape, dtype=F64, device=DEV)
    for b in range(v.shape[0]):
        sb, zb = s[b].clone(), size[b].clone()
        for t in range(v.shape[1] if lengths is None else max(0, min(lengths[b], v.shape[1]))):
            sb, zb, out[b, t], osize[b, t] = _step(sb, zb, q[b, t], k[b, t], v[b, t].double(), g[b, t].double(), beta[b, t].double())
        s[b], size[b] = sb, zb
    return out, osize, s


def delta_out_bound(want, size):
    return half(BF16) * want.abs() + 3 * half(F16) * (1 + 2**-6) * size + 2**-20 * size


def delta_state_bound(want, tokens):
    chunks = max(1, -(-tokens // 64))
    return chunks * (3 * 2 * 2**-22 + 192 * 2**-24) * want.abs().amax((-1, -2), keepdim=True) + 1e-30


@pytest.mark.parametrize("l2norm", [False, True])
@pytest.mark.parametrize(
    "b,t,hk,hv,dk,dv",
    [(1, 1, 2, 4, 128, 128), (2, 3, 1, 1, 16, 16), (1, 64, 2, 4, 128, 128), (2, 65, 2, 2, 64, 128), (1, 200, 3, 9, 96, 80), (3, 129, 2, 4, 8, 8), (1, 17, 1, 2, 128, 264), (2, 24, 2, 6, 72, 104), (5, 12, 2, 32, 128, 128), (1, 25, 16, 32, 128, 128), (20, 70, 2, 8, 128, 64), (1, 1337, 16, 32, 64, 32)],
)
def test_delta_rule_chunk(b, t, hk, hv, dk, dv, l2norm):
    a = delta_inputs(41, b, t, hk, hv, dk, dv, l2norm)
    s0 = a[0].clone()
    out, state = ops.delta_rule_chunk(*a, None, l2norm)
    want, size, s = delta_ref(*a, None, l2norm)
    within(out, want, delta_out_bound(want, size))
    within(state, s, delta_state_bound(s, t))
    assert torch.equal(a[0], s0)


@pytest.mark.parametrize("t,hv", [(5, 4), (150, 4), (150, 40)])  # (the last: more heads than run at once)
def test_delta_rule_lengths_and_what_lies_behind_them(t, hv):
    b, hk, dk, dv = 6, 2, 128, 128
    a = list(delta_inputs(51, b, t, hk, hv, dk, dv, True))
    lens = [t, 0, 1, t // 2, t + 7, -3]
    want, size, s = delta_ref(*a, lens, True)
    for i, n in enumerate(lens):  # padding may hold anything
        n = max(0, n)
        for x in a[1:]:
            x[i, n:] = torch.nan
    lt = torch.tensor(lens, dtype=I32, device=DEV)
    out, state = ops.delta_rule_chunk(*a, lt, True)
    within(out, want, delta_out_bound(want, size))
    within(state, s, delta_state_bound(s, t))
    assert torch.equal(state[1], a[0][1]) and torch.equal(state[5], a[0][5])
    for i, n in enumerate(lens):
        assert bool((out[i, max(0, n) :] == 0).all())


def test_delta_rule_in_pieces_equals_the_whole():
    """A prompt in two calls that hand the state on, at a border that no chunk has."""
    a = delta_inputs(61, 1, 333, 2, 4, 128, 128, True)
    out, state = ops.delta_rule_chunk(*a, None, True)
    want, size, s = delta_ref(*a, None, True)
    o1, s1 = ops.delta_rule_chunk(a[0], *(x[:, :100] for x in a[1:]), None, True)
    o2, s2 = ops.delta_rule_chunk(s1, *(x[:, 100:] for x in a[1:]), None, True)
    within(torch.cat((o1, o2), 1), want, delta_out_bound(want, size))
    within(s2, s, delta_state_bound(s, 333))
    within(state, s, delta_state_bound(s, 333))


def test_delta_rule_agrees_with_its_single_step():
    a = delta_inputs(71, 3, 4, 4, 4, 64, 64, False)
    out, state = ops.delta_rule_chunk(*a, None, False)
    s = a[0]
    for t in range(4):
        o, s = ops.delta_rule_step(s, *(x[:, t] for x in a[1:]))
        assert bool(((out[:, t].float() - o).abs() <= 2 * half(BF16) * o.abs() + 2**-9 * o.abs().max()).all())
    within(state, s.double(), 2 * delta_state_bound(s.double(), 4))


@pytest.mark.parametrize("kind", ["strong decay", "no decay", "reset", "same keys", "beta 0 and 1", "large", "zero keys"])
def test_delta_rule_at_its_edges(kind):
    b, t, hk, hv, dk, dv = 1, 100, 1, 2, 64, 32
    st, q, k, v, g, beta = delta_inputs(81, b, t, hk, hv, dk, dv, True)
    if kind == "strong decay":
        g = g * 200
    elif kind == "no decay":
        g = g * 0
    elif kind == "reset":
        g[:, ::7] = -torch.inf
    elif kind == "same keys":
        k = k[:, :1].expand(b, t, hk, dk)
    elif kind == "beta 0 and 1":
        beta = (torch.arange(t, device=DEV) % 3 != 0).float()[None, :, None].expand(b, t, hv)
    elif kind == "large":
        q, k, v, st = q * 2**60, k * 2**50, v * 2**40, st * 2**40
    else:
        k = k * 0
    want, size, s = delta_ref(st, q, k, v, g, beta, None, True)
    out, state = ops.delta_rule_chunk(st, q, k, v, g, beta, None, True)
    within(out, want, delta_out_bound(want, size) + 1e-30)
    within(state, s, delta_state_bound(s, t) + 2**-20 * size.amax())


def tree_delta_ref(state, q, k, v, g, beta, parents, l2norm):
    q, k = _normalised(q, k, v.shape[2], l2norm)
    out, osize = torch.zeros(v.shape, dtype=F64, device=DEV), torch.zeros(v.shape, dtype=F64, device=DEV)
    for b, tree in enumerate(parents):
        states = []
        for t, p in enumerate(tree):
            if p < -1 or p >= t:
                states.append(None)
                continue
            s, z = (state[b].double(), state[b].double().abs()) if p == -1 or states[p] is None else states[p]
            s, z, out[b, t], osize[b, t] = _step(s, z, q[b, t], k[b, t], v[b, t].double(), g[b, t].double(), beta[b, t].double())
            states.append((s, z))
    return out, osize


@pytest.mark.parametrize("l2norm", [False, True])
@pytest.mark.parametrize("b,n,hk,hv,dk,dv,tree", [(1, 1, 2, 4, 128, 128, "one"), (2, 16, 2, 4, 128, 128, "random"), (1, 64, 1, 3, 96, 80, "chain"), (3, 37, 2, 2, 64, 16, "random"), (1, 64, 1, 1, 128, 128, "star"), (20, 9, 4, 16, 64, 40, "random"), (12, 33, 8, 32, 128, 136, "random")])
def test_delta_rule_tree(b, n, hk, hv, dk, dv, tree, l2norm):
    a = delta_inputs(91, b, n, hk, hv, dk, dv, l2norm)
    s0 = a[0].clone()
    parents = [TREES[tree](n) for _ in range(b)]
    got = ops.delta_rule_tree(*a, torch.tensor(parents, dtype=I32, device=DEV), l2norm)
    want, size = tree_delta_ref(*a, parents, l2norm)
    within(got, want, delta_out_bound(want, size))
    assert torch.equal(a[0], s0)
    if tree == "chain":  # a chain is a prompt
        within(got, ops.delta_rule_chunk(*a, None, l2norm)[0].double(), 2 * delta_out_bound(want, size))


@pytest.mark.parametrize("hk,hv", [(2, 4), (40, 160)])
def test_delta_rule_tree_rows_without_a_node(hk, hv):
    b, n, dk, dv = 2, 12, 128, 128
    a = list(delta_inputs(95, b, n, hk, hv, dk, dv, True))
    parents = [[-1, 0, 7, 2, -5, 4, 5, 3, 99, 8, 9, 1], [-2] * n]
    want, size = tree_delta_ref(*a, parents, True)
    empty = torch.tensor([[p is None for p in paths(x)] for x in parents], device=DEV)
    for x in a[1:]:
        x[empty] = torch.nan
    got = ops.delta_rule_tree(*a, torch.tensor(parents, dtype=I32, device=DEV), True)
    within(got, want, delta_out_bound(want, size))
    assert bool((got[empty] == 0).all())


def test_delta_rule_layouts_streams_and_graphs():
    b, t, hk, hv, dk, dv = 2, 90, 2, 4, 128, 128
    st, q, k, v, g, beta = delta_inputs(97, b, t, hk, hv, dk, dv, True)
    base = ops.delta_rule_chunk(st, q, k, v, g, beta, None, True)
    row = torch.cat([x.flatten(2) for x in (q, k, v)], -1)
    cut = [x.unflatten(-1, (h, 128)) for x, h in zip(row.split([hk * dk, hk * dk, hv * dv], -1), (hk, hk, hv))]
    odd = torch.cat([rnd(1, b, t, 1, dtype=BF16), row], -1)[..., 1:]  # rows on odd elements: copied
    cut2 = [x.unflatten(-1, (h, 128)) for x, h in zip(odd.split([hk * dk, hk * dk, hv * dv], -1), (hk, hk, hv))]
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    for x in (cut, cut2, heads_first, [at_odd_offset(x) for x in (q, k, v)], [q, k, at_odd_offset(v)]):
        got = ops.delta_rule_chunk(st.transpose(2, 3).contiguous().transpose(2, 3), *x, g.transpose(1, 2).contiguous().transpose(1, 2), beta, None, True)
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got.append(ops.delta_rule_chunk(st, q, k, v, g, beta, None, True))
    torch.cuda.synchronize()
    assert all(torch.equal(x, base[0]) and torch.equal(y, base[1]) for x, y in got)
    lens = torch.full((b,), t, dtype=I32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, state = ops.delta_rule_chunk(st, q, k, v, g, beta, lens, True)
    for new in ([t, t], [0, 33], [64, 65]):
        lens.copy_(torch.tensor(new, dtype=I32))
        graph.replay()
        want = ops.delta_rule_chunk(st, q, k, v, g, beta, lens, True)
        assert torch.equal(out, want[0]) and torch.equal(state, want[1])


def test_delta_rule_long_prompt_in_segments():
    """Three segments, each prepared beside the scan of the one before: alone, on two streams at once, and replayed from a
    graph with lengths that end in each of them."""
    b, t, hk, hv, dk, dv = 1, 7000, 16, 32, 128, 8
    a = delta_inputs(121, b, t, hk, hv, dk, dv, True)
    out, state = ops.delta_rule_chunk(*a, None, True)
    want, size, s = delta_ref(*a, None, True)
    within(out, want, delta_out_bound(want, size))
    within(state, s, delta_state_bound(s, t))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for x in (s1, s2):
            with torch.cuda.stream(x):
                got.append(ops.delta_rule_chunk(*a, None, True))
    torch.cuda.synchronize()
    assert all(torch.equal(x, out) and torch.equal(y, state) for x, y in got)
    lens = torch.full((b,), t, dtype=I32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, st = ops.delta_rule_chunk(*a, lens, True)
    for n in (t, 0, 1152, 1153, 4000, 1, t):
        lens.fill_(n)
        graph.replay()
        assert torch.equal(o[:, :n], out[:, :n]) and bool((o[:, n:] == 0).all())
        if n == t:
            assert torch.equal(st, state)
        elif n == 0:
            assert torch.equal(st, a[0])
        else:
            assert torch.equal(st, ops.delta_rule_chunk(*a, lens, True)[1])


@pytest.mark.parametrize("t", [7, 100])
def test_delta_rule_expanded_inputs(t):
    b, hk, hv, dk, dv = 2, 4, 8, 64, 64
    st, q, k, v, g, beta = delta_inputs(131, b, t, hk, hv, dk, dv, True)
    q, k, v = q[:1].expand(b, t, hk, dk), k[:, :, :1].expand(b, t, hk, dk), v[:, :, :1].expand(b, t, hv, dv)
    g, beta = g[:, :1].expand(b, t, hv), beta[:1].expand(b, t, hv)
    got = ops.delta_rule_chunk(st[:1].expand(b, hv, dk, dv), q, k, v, g, beta, None, True)
    want = ops.delta_rule_chunk(st[:1].repeat(b, 1, 1, 1), *(x.contiguous() for x in (q, k, v, g, beta)), None, True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_nothing_to_do():
    st, q, k, v, g, beta = delta_inputs(99, 2, 4, 1, 2, 16, 16, True)
    none = [x[:, :0] for x in (q, k, v, g, beta)]
    out, state = ops.delta_rule_chunk(st, *none, None, True)
    assert out.shape == (2, 0, 2, 16) and torch.equal(state, st) and state.data_ptr() != st.data_ptr()
    assert ops.delta_rule_tree(st, *none, torch.zeros((2, 0), dtype=I32, device=DEV), True).shape == (2, 0, 2, 16)
    q, c = rnd(1, 2, 0, 4, 64, dtype=BF16), rnd(2, 2, 2, 8, 64, dtype=BF16)
    assert ops.tree_attention(q, c, c, torch.zeros(2, dtype=I32, device=DEV), torch.zeros((2, 0), dtype=I32, device=DEV), 1.0).shape == q.shape


# ---------------------------------------------------------------- a run of them together


def test_a_tree_is_verified_and_a_path_accepted():
    """One attention and one DeltaNet layer: a prompt, then a drafted tree in one pass, then the accepted path through the
    recurrence; every node's output is what decoding its path token by token gives."""
    b, prompt, n, hq, hkv, d, r, rows = 2, 70, 11, 8, 2, 128, 32, 128
    hk, hv, dk, dv = 2, 4, 128, 128
    tree = random_tree(3, n)
    depth = torch.tensor([len(p) - 1 for p in paths(tree)], device=DEV)
    parents = torch.tensor(tree, dtype=I32, device=DEV)
    inv, factor = ops.rope_frequencies(r, 1e7)
    q, k, v = (rnd(i, b, prompt + n, h, d, dtype=BF16) for i, h in ((101, hq), (102, hkv), (103, hkv)))
    st, dq, dkey, dval, g, beta = delta_inputs(111, b, prompt + n, hk, hv, dk, dv, True)
    kc, vc = torch.full((b, hkv, rows, d), torch.nan, dtype=BF16, device=DEV), torch.full((b, hkv, rows, d), torch.nan, dtype=BF16, device=DEV)
    at = torch.arange(prompt, dtype=I32, device=DEV).expand(b, prompt).contiguous()
    zero = torch.zeros(b, dtype=I32, device=DEV)
    cached = zero + prompt
    # the prompt
    ops.rotary_append(q[:, :prompt], k[:, :prompt], v[:, :prompt], at, inv, factor, False, kc, vc, zero)
    _, state = ops.delta_rule_chunk(st, *(x[:, :prompt] for x in (dq, dkey, dval, g, beta)), None, True)
    # the tree: every node one step past its parent
    pos = (prompt + depth).to(I32).expand(b, n).contiguous()
    tq = ops.rotary_append(q[:, prompt:], k[:, prompt:], v[:, prompt:], pos, inv, factor, False, kc, vc, cached)
    attn = ops.tree_attention(tq, kc, vc, cached, parents, d**-0.5)
    lin = ops.delta_rule_tree(state, *(x[:, prompt:] for x in (dq, dkey, dval, g, beta)), parents, True)
    want, size = tree_ref(tq, kc, vc, [prompt] * b, [tree] * b, d**-0.5)
    within(attn, want, tree_bound(want, size, tq, kc, d**-0.5, rows))
    want, size = tree_delta_ref(state, *(x[:, prompt:] for x in (dq, dkey, dval, g, beta)), [tree] * b, True)
    within(lin, want, delta_out_bound(want, size))
    # Against the single-token ops: each side rounds to bf16 once and its operands to 8 or 11 bits, together below
    # 2^-7 |o| + 2^-7 sum |terms|, where the sums of this data's terms stay near 1
    for node, path in enumerate(paths(tree)):
        row = [prompt + j for j in path]
        keys = torch.cat((kc[:, :, :prompt], kc[:, :, row]), 2)
        vals = torch.cat((vc[:, :, :prompt], vc[:, :, row]), 2)
        one = ops.gqa_decode_attention(tq[:, node].contiguous(), keys.contiguous(), vals.contiguous(), d**-0.5)
        assert bool(((attn[:, node].float() - one.float()).abs() <= 2e-2 * one.float().abs() + 1e-2).all())
        o, _ = ops.delta_rule_chunk(state, *(x[:, row] for x in (dq, dkey, dval, g, beta)), None, True)
        assert bool(((lin[:, node].float() - o[:, -1].float()).abs() <= 2e-2 * o[:, -1].float().abs() + 1e-2).all())
    # sequence 0 accepts the longest path, sequence 1 nothing
    best = max(paths(tree), key=len)
    row = [prompt + j for j in best]
    after = ops.delta_rule_chunk(state, *(x[:, row] for x in (dq, dkey, dval, g, beta)), torch.tensor([len(best), 0], dtype=I32, device=DEV), True)[1]
    whole = ops.delta_rule_chunk(st, *(torch.cat((x[:, :prompt], x[:, row]), 1) for x in (dq, dkey, dval, g, beta)), None, True)[1]
    assert torch.equal(after[1], state[1])
    within(after[0], whole[0].double(), 4 * delta_state_bound(whole[0].double(), prompt + n))


# ---------------------------------------------------------------- what follows a call in its stream


@pytest.mark.parametrize("b,hq,hkv,d,n,rows,lens", [(16, 16, 8, 128, 17, 1500, 1400), (16, 16, 8, 64, 9, 128, 100), (9, 16, 4, 256, 5, 128, 123)])
def test_tree_attention_has_ended_before_the_next_kernel_reads(b, hq, hkv, d, n, rows, lens):
    """Every unit is one part here, so the merge has nothing to do. The queries change from call to call: an output read too early
    would be that of another call. Eager and in a captured graph."""
    kc, vc = rnd(141, b, hkv, rows, d, dtype=BF16), rnd(142, b, hkv, rows, d, dtype=BF16)
    lt, pt = torch.full((b,), lens, dtype=I32, device=DEV), torch.tensor(random_tree(7, n), dtype=I32, device=DEV)
    qs = [rnd(143 + i, b, n, hq, d, dtype=BF16) for i in range(3)]
    base = []
    for q in qs:
        o = ops.tree_attention(q, kc, vc, lt, pt, d**-0.5)
        torch.cuda.synchronize()
        base.append(o.clone())
    want, size = tree_ref(qs[0][:1], kc[:1], vc[:1], [lens], [pt.tolist()], d**-0.5)
    within(base[0][:1], want, tree_bound(want, size, qs[0], kc, d**-0.5, rows))
    got = []
    for i in range(30):
        got.append(ops.tree_attention(qs[i % 3], kc, vc, lt, pt, d**-0.5).clone())
    torch.cuda.synchronize()
    assert all(torch.equal(x, base[i % 3]) for i, x in enumerate(got))
    q = qs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy = ops.tree_attention(q, kc, vc, lt, pt, d**-0.5).clone()
    for i in range(9):
        q.copy_(qs[i % 3])
        graph.replay()
        assert torch.equal(copy, base[i % 3])


@pytest.mark.parametrize("b,hq,hkv,d,n", [(40, 16, 4, 256, 6), (60, 20, 4, 128, 7), (37, 12, 6, 64, 31)])
def test_tree_attention_of_many_ragged_units_repeats_itself(b, hq, hkv, d, n):
    """Each CTA walks through several units of different lengths, whose copies follow the stores of the unit before."""
    rows = 1500
    g = torch.Generator().manual_seed(b)
    lens = [0, 1, rows - n, 128 - n, 127] + torch.randint(0, rows - n, (b - 5,), generator=g).tolist()
    q = rnd(151, b, n, hq, d, dtype=BF16)
    kc, vc = rnd(152, b, hkv, rows, d, dtype=BF16), rnd(153, b, hkv, rows, d, dtype=BF16)
    parents = [random_tree(i, n) for i in range(b)]
    lt, pt = torch.tensor(lens, dtype=I32, device=DEV), torch.tensor(parents, dtype=I32, device=DEV)
    base = ops.tree_attention(q, kc, vc, lt, pt, d**-0.5)
    want, size = tree_ref(q, kc, vc, lens, parents, d**-0.5)
    within(base, want, tree_bound(want, size, q, kc, d**-0.5, rows))
    for _ in range(20):
        assert torch.equal(ops.tree_attention(q, kc, vc, lt, pt, d**-0.5), base)


# ---------------------------------------------------------------- scores of any size


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,hq,hkv,n,d", [(2, 4, 2, 5, 64), (2, 40, 20, 30, 64), (3, 4, 2, 40, 256), (8, 16, 4, 17, 256)])
@pytest.mark.parametrize("size_of_scores", [2850, 5710, 10_000, 23_000, 100_000, -2870, -5700, -23_000, -100_000])
def test_tree_attention_with_large_scores(size_of_scores, b, hq, hkv, n, d, dtype):
    """All scores lie near one large number, whose place against a coarse grid must not matter; differences between them are
    ordinary. Queries and keys are whole numbers, so that every score is exact in fp32; what remains of the error ds of
    `tree_bound` is scale log2(e) (two roundings), its product with the score and the difference to the maximum: 4 h(fp32) |score|."""
    rows, scale = 700, 0.25
    g = torch.Generator().manual_seed(n)
    q = torch.randint(-2, 3, (b, n, hq, d), generator=g).to(dtype).to(DEV)
    kc = torch.randint(-1, 2, (b, hkv, rows, d), generator=g).to(dtype).to(DEV)
    vc = rnd(161, b, hkv, rows, d, dtype=dtype)
    q[..., 0], kc[..., 0] = 256, round(size_of_scores / (256 * scale))
    q[..., 1], kc[..., 1] = 8, (torch.arange(rows, device=DEV) // 128 - 3).to(dtype)  # the maximum moves from tile to tile
    lens = [rows - n] + [int(torch.randint(0, rows - n, (1,), generator=g)) for _ in range(b - 1)]
    parents = [random_tree(i, n) for i in range(b)]
    want, size = tree_ref(q, kc, vc, lens, parents, scale)
    got = ops.tree_attention(q, kc, vc, torch.tensor(lens, dtype=I32, device=DEV), torch.tensor(parents, dtype=I32, device=DEV), scale)
    ds = 4 * half(F32) * (abs(size_of_scores) * 1.01 + 1000)
    within(got, want, half(dtype) * want.abs() + (half(dtype) + 2 * ds + 2**-20 + rows * 2**-24) * size * (1 + 2**-6))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,hq,hkv,n,d", [(2, 4, 2, 5, 64), (2, 40, 20, 30, 64), (1, 8, 2, 12, 256), (8, 16, 4, 17, 256)])
@pytest.mark.parametrize("gap", [9.0, 14.0, 17.0])
def test_tree_attention_behind_one_dominant_key(gap, b, hq, hkv, n, d, dtype):
    """One key takes nearly all of the weight and has a value of zero (an attention sink): the output is the sum over the others,
    whose probabilities lie e^-gap below the largest one, in fp16's subnormal range if they were held relative to it."""
    rows = 3000
    q, kc = torch.zeros(b, n, hq, d, dtype=dtype, device=DEV), torch.zeros(b, hkv, rows, d, dtype=dtype, device=DEV)
    q[..., 3], kc[:, :, 1, 3] = 1.0, gap
    kc[..., 5], q[..., 5] = rnd(171, b, hkv, rows, dtype=dtype), 0.25
    kc[:, :, 1, 5] = 0.0
    vc = rnd(172, b, hkv, rows, d, dtype=dtype, scale=64.0) + 64.0
    vc[:, :, 1] = 0.0
    lens, parents = [rows - n] * b, [random_tree(i, n) for i in range(b)]
    want, size = tree_ref(q, kc, vc, lens, parents, 1.0)
    got = ops.tree_attention(q, kc, vc, torch.tensor(lens, dtype=I32, device=DEV), torch.tensor(parents, dtype=I32, device=DEV), 1.0)
    within(got, want, tree_bound(want, size, q, kc, 1.0, rows))


# ---------------------------------------------------------------- chunks whose update is nothing, or small beside a bound on it


@pytest.mark.parametrize("l2norm", [False, True])
@pytest.mark.parametrize("dk,dv,hv", [(128, 128, 4), (64, 40, 2)])
@pytest.mark.parametrize("kind", ["beta 0", "keys and values 0", "beta 0 and no decay", "forgotten", "forgotten by all", "small"])
def test_delta_rule_state_after_a_chunk_that_adds_little(kind, dk, dv, hv, l2norm):
    """The state's scale in the next chunk follows from a bound on this chunk's update. Tokens 64 .. 127 add nothing at all, or the
    largest values of theirs are forgotten within the chunk, or are far below the state."""
    t = 260
    st, q, k, v, g, beta = delta_inputs(181, 1, t, 2, hv, dk, dv, l2norm)
    mid = slice(64, 128)
    if kind.startswith("beta 0"):
        beta[:, mid] = 0.0
        if kind != "beta 0":
            g[:, mid] = 0.0
    elif kind == "keys and values 0":
        k[:, mid], v[:, mid] = 0.0, 0.0
    elif kind == "small":
        v[:, mid] *= 2.0**-40
        st, beta[:, 64:65] = st * 0.0, 1.0
        v[:, :64] *= 2.0**-40
    else:
        v[:, 64:68] *= 2.0**18
        g[:, 70] = -40.0  # e^-40 of 2^18 is 1e-12
        if kind == "forgotten by all":
            g[:, 127] = -60.0
    want, size, s = delta_ref(st, q, k, v, g, beta, None, l2norm)
    out, state = ops.delta_rule_chunk(st, q, k, v, g, beta, None, l2norm)
    within(out, want, delta_out_bound(want, size))
    within(state, s, delta_state_bound(s, t))
    # the outputs of the chunk behind it hold to the bound of the state, up to their own rounding to 11 and 8 bits; with a query that
    # reads the state alone (beta 0 from there on) no product of new terms covers an error of it
    beta[:, 128:], g[:, 128:] = 0.0, 0.0
    want, size, s = delta_ref(st, q, k, v, g, beta, None, l2norm)
    out, state = ops.delta_rule_chunk(st, q, k, v, g, beta, None, l2norm)
    within(out, want, delta_out_bound(want, size))
    within(state, s, delta_state_bound(s, t))


# ---------------------------------------------------------------- the ops as a compiled, traced or plain call


def small_calls():
    """(name, function of its tensors alone, tensors) of each of the five ops"""
    b, t, hq, hkv, d = 2, 5, 4, 2, 64
    q, k, v = rnd(191, b, t, hq, d, dtype=BF16), rnd(192, b, t, hkv, d, dtype=BF16), rnd(193, b, t, hkv, d, dtype=BF16)
    kc, vc = rnd(194, b, hkv, 40, d, dtype=BF16), rnd(195, b, hkv, 40, d, dtype=BF16)
    pos = torch.arange(b * t, dtype=I32, device=DEV).view(b, t)
    inv, factor = ops.rope_frequencies(32, 1e4)
    lens, parents = torch.tensor([30, 7], dtype=I32, device=DEV), torch.tensor(random_tree(2, t), dtype=I32, device=DEV)
    st, dq, dk, dv, g, beta = delta_inputs(196, b, t, 2, 4, 64, 32, True)
    return [
        ("rotary_qk", lambda q, k, pos, inv: ops.rotary_qk(q, k, pos, inv, factor, True), (q, k, pos, inv)),
        ("rotary_append", lambda q, k, v, pos, inv, kc, vc, n: (ops.rotary_append(q, k, v, pos, inv, factor, False, kc, vc, n), kc, vc), (q, k, v, pos, inv, kc, vc, lens)),
        ("tree_attention", lambda q, kc, vc, n, p: ops.tree_attention(q, kc, vc, n, p, 0.125), (q, kc, vc, lens, parents)),
        ("delta_rule_chunk", lambda s, q, k, v, g, b: ops.delta_rule_chunk(s, q, k, v, g, b, None, True), (st, dq, dk, dv, g, beta)),
        ("delta_rule_tree", lambda s, q, k, v, g, b, p: ops.delta_rule_tree(s, q, k, v, g, b, p, True), (st, dq, dk, dv, g, beta, parents)),
    ]


def same(x, y):
    x, y = (z if isinstance(z, tuple) else (z,) for z in (x, y))
    return len(x) == len(y) and all(torch.equal(u, w) for u, w in zip(x, y))


@pytest.mark.parametrize("which", range(5))
def test_compiled_and_dispatched_calls_equal_plain_ones(which):
    name, call, tensors = small_calls()[which]
    want = call(*(x.clone() for x in tensors))
    torch._dynamo.reset()
    assert same(torch.compile(call, fullgraph=True, backend="aot_eager")(*(x.clone() for x in tensors)), want)
    traced = torch.jit.trace(call, tuple(x.clone() for x in tensors), check_trace=False)
    assert same(traced(*(x.clone() for x in tensors)), want)


def test_negative_views_are_read_as_what_they_stand_for():
    _, call, (st, q, k, v, g, beta) = small_calls()[3]
    want = call(-st, -q, k, v, g, -beta)
    assert same(call(torch._neg_view(st), torch._neg_view(q), k, v, g, torch._neg_view(beta)), want)
    q, pos = rnd(197, 1, 3, 2, 16), torch.arange(3, dtype=I32, device=DEV)[None]
    inv, factor = ops.rope_frequencies(16, 1e4)
    assert same(ops.rotary_qk(torch._neg_view(q), q, pos, inv, factor, False), ops.rotary_qk(-q, q, pos, inv, factor, False))


def test_the_caches_versions_move_with_an_append():
    _, call, tensors = small_calls()[1]
    before = [x._version for x in tensors]
    call(*tensors)
    moved = [x._version - y for x, y in zip(tensors, before)]
    assert moved == [0, 0, 0, 0, 0, 1, 1, 0]


# ---------------------------------------------------------------- strides that no address depends on


@pytest.mark.parametrize("b,hkv,rows,n,group", [(1, 2, 300, 7, 2), (3, 1, 300, 33, 4), (33, 1, 200, 20, 2), (2, 2, 1, 3, 2), (1, 40, 150, 30, 1)])
def test_tree_attention_with_odd_strides_of_dimensions_of_one(b, hkv, rows, n, group):
    d = 64
    q = rnd(201, b, n, hkv * group, d, dtype=BF16)
    kc, vc = rnd(202, b, hkv, rows, d, dtype=BF16), rnd(203, b, hkv, rows, d, dtype=BF16)
    lt, pt = torch.full((b,), max(0, rows - n), dtype=I32, device=DEV), torch.tensor(random_tree(3, n), dtype=I32, device=DEV)

    def odd(x):
        y = x.as_strided(x.shape, tuple(s if m > 1 else 2 * s + 5 for s, m in zip(x.stride()[:3], x.shape)) + (1,))
        assert torch.equal(x, y) and any(s % 8 for s in y.stride()[:3])
        return y

    want = ops.tree_attention(q, kc, vc, lt, pt, 0.125)
    assert torch.equal(ops.tree_attention(q, odd(kc), odd(vc), lt, pt, 0.125), want)


def test_delta_rule_with_odd_strides_of_dimensions_of_one():
    st, q, k, v, g, beta = delta_inputs(205, 1, 70, 1, 1, 64, 64, True)
    want = ops.delta_rule_chunk(st, q, k, v, g, beta, None, True)
    cut = [x.as_strided(x.shape, (3, x.stride(1), 7, 1)) for x in (q, k, v)]
    got = ops.delta_rule_chunk(st, *cut, g, beta, None, True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
