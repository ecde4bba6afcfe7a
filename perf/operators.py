"""What is measured of the operators that take several new tokens of a sequence at once.

Four operators of one set: rotary positions (with the cache write), attention of a tree of drafted tokens over the KV
cache, the gated delta rule over a prompt, and the gated delta rule over a tree of drafted tokens. ``run`` computes a case
in elementary torch operations, or, with ``own`` set, through the ops of ``deltaforge_b200.ops``.
"""

import math

import torch

own = False

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "fp16": F16, "fp32": F32}
CHUNK = 64  # tokens per chunk of the plain form of the delta rule


def listed():
    return [
        # the smallest call: one new token of one sequence, its key and value appended to the cache
        dict(name="rotary 1 token append", op="rotary", batch=1, tokens=1, hq=16, hkv=4, dim=256, rotary=64, interleaved=False, append=True, start=4096, stretch=1.0, dtype="bf16"),
        # a prompt of 8192 tokens of the benchmark model's attention layers, written to the cache
        dict(name="rotary 8192 prompt append", op="rotary", batch=1, tokens=8192, hq=16, hkv=4, dim=256, rotary=64, interleaved=False, append=True, start=0, stretch=1.0, dtype="bf16"),
        # interleaved pairs over the whole head, ragged batch, far positions of a context stretched four times
        dict(name="rotary interleaved stretched", op="rotary", batch=5, tokens=777, hq=12, hkv=2, dim=128, rotary=128, interleaved=True, append=False, start=200000, stretch=4.0, dtype="fp16"),
        # one token over 4096 cached rows: the single-token form of the tree attention
        dict(name="tree attention 1 node", op="tree_attention", batch=1, nodes=1, hq=16, hkv=4, dim=256, context=4096, empty=0, dtype="bf16"),
        # a draft of 16 nodes on the benchmark's context
        dict(name="tree attention 16 nodes", op="tree_attention", batch=1, nodes=16, hq=16, hkv=4, dim=256, context=4096, empty=0, dtype="bf16"),
        # many sequences of ragged length, a small odd tree, one query head per KV head, a shorter head
        dict(name="tree attention 24 ragged", op="tree_attention", batch=24, nodes=7, hq=8, hkv=8, dim=128, context=5000, empty=1, dtype="fp16"),
        # the largest trees over long caches
        dict(name="tree attention 8 x 64 long", op="tree_attention", batch=8, nodes=64, hq=16, hkv=4, dim=256, context=32768, empty=0, dtype="bf16"),
        # one token of 16 sequences: the single-token form of the delta rule
        dict(name="delta rule 16 x 1", op="delta_chunk", batch=16, tokens=1, hk=16, hv=32, dk=128, dv=128, ragged=False, norm=True),
        # one long prompt of the benchmark model's DeltaNet layers
        dict(name="delta rule 8192 prompt", op="delta_chunk", batch=1, tokens=8192, hk=16, hv=32, dk=128, dv=128, ragged=False, norm=True),
        # a padded batch of prompts of odd lengths
        dict(name="delta rule 6 x 1001 ragged", op="delta_chunk", batch=6, tokens=1001, hk=16, hv=32, dk=128, dv=128, ragged=True, norm=True),
        # a draft of 16 nodes of one sequence
        dict(name="delta tree 16 nodes", op="delta_tree", batch=1, tokens=16, hk=16, hv=32, dk=128, dv=128, empty=0, norm=True),
        # the largest trees, of 16 sequences
        dict(name="delta tree 16 x 64", op="delta_tree", batch=16, tokens=64, hk=16, hv=32, dk=128, dv=128, empty=3, norm=True),
    ]


def _log(rng, low, high):
    return min(high, int(low * (high / low + 1) ** rng.random()))


def draw(rng):
    op = rng.choice(["rotary", "tree_attention", "delta_chunk", "delta_tree"])
    if op == "rotary":
        hq, hkv, dim = rng.choice([(16, 4, 256), (2, 1, 32), (8, 8, 64), (12, 2, 128), (16, 2, 256)])
        batch = _log(rng, 1, 16)
        return dict(
            op=op, batch=batch, tokens=_log(rng, 1, 8192 // batch), hq=hq, hkv=hkv, dim=dim, rotary=rng.choice([dim, dim // 2, dim // 4]),
            interleaved=rng.random() < 0.4, append=rng.random() < 0.6, start=_log(rng, 1, 250000), stretch=rng.choice([1.0, 2.0, 4.0, 7.5]),
            dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
        )  # fmt: skip
    if op == "tree_attention":
        hq, hkv, dim = rng.choice([(16, 4, 256), (16, 4, 256), (2, 1, 32), (8, 8, 64), (12, 2, 128), (16, 2, 256)])
        batch, nodes = _log(rng, 1, 32), _log(rng, 1, 64)
        return dict(
            op=op, batch=batch, nodes=nodes, hq=hq, hkv=hkv, dim=dim, context=_log(rng, 1, 8 * 32768 // max(8, batch)), empty=rng.choice([0, 0, 1]),
            dtype=rng.choice(["bf16", "bf16", "fp16"]),
        )  # fmt: skip
    hk, hv, dk, dv = rng.choice([(16, 32, 128, 128), (16, 32, 128, 128), (2, 4, 16, 16), (4, 4, 64, 128), (3, 9, 96, 80), (8, 16, 128, 64)])
    if op == "delta_chunk":
        batch = _log(rng, 1, 16)
        return dict(op=op, batch=batch, tokens=_log(rng, 1, 8192 // batch), hk=hk, hv=hv, dk=dk, dv=dv, ragged=rng.random() < 0.5, norm=rng.random() < 0.7)
    return dict(op=op, batch=_log(rng, 1, 16), tokens=_log(rng, 1, 64), hk=hk, hv=hv, dk=dk, dv=dv, empty=rng.choice([0, 0, 2]), norm=rng.random() < 0.7)


# ---- inputs ---------------------------------------------------------------------------------------------------------


class _Maker:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator("cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype=F32, scale=1.0):
        return (torch.randn(*shape, generator=self.g, device="cuda") * scale).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")

    def whole(self, low, high, *shape):  # low..high, both included
        return torch.randint(low, high + 1, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def parents(self, batch, nodes, empty):
        """Random trees; the last `empty` rows of the first sequence hold no node."""
        p = (self.uniform(batch, nodes) * (torch.arange(nodes, device="cuda") + 1)).floor().to(torch.int32) - 1
        if empty:
            p[0, max(0, nodes - empty) :] = -2
        return p


def _frequencies(case):
    """Inverse frequencies in 64 bits and the factor on cos and sin. A context stretched beyond the trained length divides
    the frequencies that turn less than once over that length by the stretch, keeps those that turn 32 times and more, and
    goes linearly in between; the factor is 0.1 ln(stretch) + 1."""
    r, theta, trained, stretch = case["rotary"], 1e7, 32768, case["stretch"]
    f = theta ** (-torch.arange(0, r, 2, dtype=F64) / r)
    if stretch == 1.0:
        return f, 1.0
    keep = ((trained * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
    return f * keep + f / stretch * (1 - keep), 0.1 * math.log(stretch) + 1.0


def prepare(case, seed):
    m, b, op = _Maker(seed), case["batch"], case["op"]
    s = {"case": case}
    if op == "rotary":
        t, hq, hkv, d, dt = case["tokens"], case["hq"], case["hkv"], case["dim"], TYPES[case["dtype"]]
        # one fused projection row per token, as the attention layers compute it: queries, keys and values are views of it
        row = m.normal(b, t, (hq + 2 * hkv) * d, dtype=dt)
        s["q"] = row[..., : hq * d].view(b, t, hq, d)
        s["k"] = row[..., hq * d : (hq + hkv) * d].view(b, t, hkv, d)
        s["v"] = row[..., (hq + hkv) * d :].view(b, t, hkv, d)
        f, s["factor"] = _frequencies(case)
        s["inv_freq"] = f.cuda()
        if case["append"]:
            s["len"] = m.whole(0, 5, b)  # rows that each sequence's cache holds already
            rows = t + 8
            s["kc"], s["vc"] = m.normal(b, hkv, rows, d, dtype=dt), m.normal(b, hkv, rows, d, dtype=dt)
            first = s["len"] + case["start"]
        else:
            first = m.whole(case["start"], case["start"] + 5, b)
        s["pos"] = (first[:, None] + torch.arange(t, device="cuda", dtype=torch.int32)).contiguous()
        return s
    if op == "tree_attention":
        n, hq, hkv, d, ctx, dt = case["nodes"], case["hq"], case["hkv"], case["dim"], case["context"], TYPES[case["dtype"]]
        s["q"] = m.normal(b, n, hq, d, dtype=dt)
        s["kc"], s["vc"] = m.normal(b, hkv, ctx + n, d, dtype=dt), m.normal(b, hkv, ctx + n, d, dtype=dt)
        s["len"] = m.whole(ctx // 2, ctx, b)
        s["len"][0] = ctx
        s["parents"] = m.parents(b, n, case["empty"])
        s["scale"] = d**-0.5
        return s
    t, hk, hv, dk, dv = case["tokens"], case["hk"], case["hv"], case["dk"], case["dv"]
    # what the causal convolution and its SiLU leave: a row of q | k | v per token
    row = torch.nn.functional.silu(m.normal(b, t, 2 * hk * dk + hv * dv)).to(BF16)
    q, k = row[..., : hk * dk].view(b, t, hk, dk), row[..., hk * dk : 2 * hk * dk].view(b, t, hk, dk)
    if not case["norm"]:  # the caller has normalised them
        q = (q.to(F32) / (q.to(F32).square().sum(-1, keepdim=True) + 1e-6).sqrt() * dk**-0.5).to(BF16)
        k = (k.to(F32) / (k.to(F32).square().sum(-1, keepdim=True) + 1e-6).sqrt()).to(BF16)
    s["q"], s["k"], s["v"] = q, k, row[..., 2 * hk * dk :].view(b, t, hv, dv)
    rate = 16 * m.uniform(hv)  # exp(A_log), and a time step spread over its logarithm, as such layers are initialised
    step = torch.exp(m.uniform(b, t, hv) * 4.6 - 6.9 + m.normal(hv, scale=0.5))
    s["g"] = -(rate * step)
    s["beta"] = torch.sigmoid(m.normal(b, t, hv))
    s["state"] = m.normal(b, hv, dk, dv, scale=0.3)
    if op == "delta_tree":
        s["parents"] = m.parents(b, t, case["empty"])
    else:
        s["lengths"] = m.whole(max(0, t // 3), t, b) if case["ragged"] else None
        if case["ragged"]:
            s["lengths"][0] = t
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    if op == "rotary":
        return _plain_rotary(s)
    if op == "tree_attention":
        return _plain_tree_attention(s)
    if op == "delta_tree":
        return _plain_delta_tree(s)
    return _plain_delta(s)


def _own(s, op):
    from deltaforge_b200 import ops

    c = s["case"]
    if op == "rotary":
        if c["append"]:
            q = ops.rotary_append(s["q"], s["k"], s["v"], s["pos"], s["inv_freq"], s["factor"], c["interleaved"], s["kc"], s["vc"], s["len"])
            return q, s["kc"], s["vc"]
        return ops.rotary_qk(s["q"], s["k"], s["pos"], s["inv_freq"], s["factor"], c["interleaved"])
    if op == "tree_attention":
        return ops.tree_attention(s["q"], s["kc"], s["vc"], s["len"], s["parents"], s["scale"])
    if op == "delta_tree":
        return ops.delta_rule_tree(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"], s["parents"], c["norm"])
    return ops.delta_rule_chunk(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"], s["lengths"], c["norm"])


def _plain_rotary(s):
    c = s["case"]
    r = c["rotary"]
    angle = s["pos"].to(F64)[..., None] * s["inv_freq"]  # 64 bits: far positions
    cos, sin = (angle.cos() * s["factor"]).to(F32)[:, :, None], (angle.sin() * s["factor"]).to(F32)[:, :, None]

    def turn(x):
        y = x.to(F32)
        if c["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., : r // 2], y[..., r // 2 : r]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned, y[..., r:]), -1).to(x.dtype)

    q, k = turn(s["q"]), turn(s["k"])
    if not c["append"]:
        return q, k
    b, t = s["pos"].shape
    which = torch.arange(b, device="cuda")[:, None].expand(b, t)
    rows = s["len"][:, None].long() + torch.arange(t, device="cuda")
    s["kc"][which, :, rows] = k
    s["vc"][which, :, rows] = s["v"]
    return q, s["kc"], s["vc"]


def _ancestors(parents):
    """[batch, i, j]: j is i or an ancestor of i, both being nodes; and which rows are nodes."""
    b, n = parents.shape
    at = torch.arange(n, device=parents.device)
    node = (parents >= -1) & (parents < at)
    up = (parents[..., None] == at) & node[..., None]
    up = up & node[:, None]
    reach = (up | torch.eye(n, dtype=torch.bool, device=parents.device)).to(F32)
    for _ in range(6):  # paths of up to 64 steps by squaring
        reach = ((reach @ reach) > 0).to(F32)
    return (reach > 0) & node[..., None] & node[:, None], node


def _plain_tree_attention(s):
    q, kc, vc, n_cached = s["q"], s["kc"], s["vc"], s["len"].long()
    b, n, hq, d = q.shape
    hkv, rows = kc.shape[1], kc.shape[2]
    reach, node = _ancestors(s["parents"])
    at = torch.arange(rows, device=q.device)
    which = (at - n_cached[:, None])[:, None].expand(b, n, rows)  # row -> node number
    seen = torch.gather(reach, 2, which.clamp(0, n - 1)) & (which >= 0) & (which < n)
    seen = (seen | (which < 0)) & node[..., None]
    x = q.to(F32).view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d) * s["scale"]
    score = (x @ kc.to(F32).transpose(-1, -2)).view(b, hkv, hq // hkv, n, rows)
    score = score.masked_fill(~seen[:, None, None], -torch.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    o = p.view(b, hkv, -1, rows) @ vc.to(F32)
    o = o.view(b, hkv, hq // hkv, n, d) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).to(q.dtype)


def _delta_inputs(s):
    """q, k, v, g, beta per value head as [batch, heads, tokens, ...] in 32 bits."""
    hv = s["v"].shape[2]
    q, k = s["q"].to(F32), s["k"].to(F32)
    if s["case"]["norm"]:
        q = q / (q.square().sum(-1, keepdim=True) + 1e-6).sqrt() * q.shape[-1] ** -0.5
        k = k / (k.square().sum(-1, keepdim=True) + 1e-6).sqrt()
    q, k = (x.repeat_interleave(hv // x.shape[2], 2).transpose(1, 2) for x in (q, k))
    return q, k, s["v"].to(F32).transpose(1, 2), s["g"].transpose(1, 2), s["beta"].transpose(1, 2)


def _unit_lower_inverse(a):
    """(I + a)^-1 for strictly lower a of width 64: diagonal blocks of twice the width from two of half, six times."""
    inv = torch.eye(a.shape[-1], device=a.device, dtype=a.dtype).expand_as(a).clone()
    at = torch.arange(a.shape[-1], device=a.device)
    for w in (1, 2, 4, 8, 16, 32):  # the lower left block of each pair of diagonal blocks is -T22 A21 T11
        pair = (at[:, None] // (2 * w) == at // (2 * w)) & (at[:, None] // w != at // w)
        inv = inv - inv @ (a * pair) @ inv
    return inv


def _chunk_matrices(q, k, g_sum, beta, seen):
    """T diag(beta) and the masked, decayed q k^T of each chunk; seen[i, j]: j is i or before it."""
    decay = (g_sum[..., :, None] - g_sum[..., None, :]).masked_fill(~seen, -torch.inf).exp()
    strict = seen & ~torch.eye(seen.shape[-1], dtype=torch.bool, device=seen.device)
    a = beta[..., None] * (k @ k.transpose(-1, -2)) * decay * strict
    return _unit_lower_inverse(a) * beta[..., None, :], (q @ k.transpose(-1, -2)) * decay


def _pad(x, n, dim):
    shape = list(x.shape)
    shape[dim] = n - shape[dim]
    return torch.cat((x, x.new_zeros(shape)), dim)


def _plain_delta(s):
    q, k, v, g, beta = _delta_inputs(s)
    b, h, t, dk = q.shape
    if s["lengths"] is not None:  # tokens past a sequence's length change nothing
        live = (torch.arange(t, device=q.device) < s["lengths"][:, None])[:, None]
        g, beta = g * live, beta * live
    n = -(-t // CHUNK) * CHUNK
    q, k, v = (_pad(x, n, 2).view(b, h, n // CHUNK, CHUNK, -1) for x in (q, k, v))
    g, beta = (_pad(x, n, 2).view(b, h, n // CHUNK, CHUNK) for x in (g, beta))
    total = g.to(F64).cumsum(-1)
    seen = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    tri, qk = _chunk_matrices(q, k, total, beta, seen)
    tri, qk = tri.to(F32), qk.to(F32)
    into = total.exp().to(F32)[..., None]
    out_of = (total[..., -1:] - total).exp().to(F32)[..., None]
    qi, ki, ko = q * into, k * into, (k * out_of).transpose(-1, -2)
    tv, tk = tri @ v, tri @ ki
    end = into[..., -1:, :]
    state, o = s["state"], torch.empty_like(v)
    for c in range(n // CHUNK):  # the recurrence over chunks
        new = tv[:, :, c] - tk[:, :, c] @ state
        o[:, :, c] = qi[:, :, c] @ state + qk[:, :, c] @ new
        state = state * end[:, :, c] + ko[:, :, c] @ new
    o = o.view(b, h, n, -1)[:, :, :t].transpose(1, 2)
    if s["lengths"] is not None:
        o = o * live.transpose(1, 2)[..., None]
    return o.to(BF16).contiguous(), state


def _plain_delta_tree(s):
    q, k, v, g, beta = _delta_inputs(s)
    t = q.shape[2]
    reach, node = _ancestors(_pad(s["parents"], 64, 1) if t < 64 else s["parents"])
    if t < 64:
        inside = torch.arange(64, device=q.device) < t
        reach, node = reach & inside[:, None] & inside, node & inside
        q, k, v, g, beta = (_pad(x, 64, 2) for x in (q, k, v, g, beta))
    seen = reach[:, None]
    total = (seen * g.to(F64)[:, :, None]).sum(-1)  # along the path of each node
    tri, qk = _chunk_matrices(q, k, total, beta, seen)
    into = total.exp().to(F32)[..., None]
    new = tri.to(F32) @ (v - (k * into) @ s["state"])
    o = (q * into) @ s["state"] + qk.to(F32) @ new
    return (o * node[:, None, :, None])[:, :, :t].transpose(1, 2).to(BF16).contiguous()


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "tree_attention": _exact_tree_attention, "delta_chunk": _exact_delta, "delta_tree": _exact_delta_tree}[case["op"]](s)


def _exact_rotary(s):
    c = s["case"]
    r = c["rotary"]
    angle = s["pos"].to(F64)[:, :, None, None] * s["inv_freq"]
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)

    def rotate(x):
        y = x.to(F64).clone()
        pairs = y[..., :r].unflatten(-1, (r // 2, 2)) if c["interleaved"] else y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y[..., :r] = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return y

    q, k = rotate(s["q"]), rotate(s["k"])
    if not c["append"]:
        return q, k
    kc, vc = s["kc"].to(F64), s["vc"].to(F64)
    for i, n in enumerate(s["len"].tolist()):
        kc[i, :, n : n + c["tokens"]] = k[i].transpose(0, 1)
        vc[i, :, n : n + c["tokens"]] = s["v"][i].to(F64).transpose(0, 1)
    return q, kc, vc


def _paths(parents):
    """For each row the list of its ancestors and itself, oldest first; None where the row holds no node."""
    found = []
    for i, p in enumerate(parents):
        found.append(None if p < -1 or p >= i else ([] if p == -1 or found[p] is None else found[p]) + [i])
    return found


def _exact_tree_attention(s):
    q = s["q"].to(F64)
    b, n, hq, d = q.shape
    hkv = s["kc"].shape[1]
    o = torch.zeros_like(q)
    for i, (cached, parents) in enumerate(zip(s["len"].tolist(), s["parents"].tolist())):
        mask = torch.zeros(n, cached + n, dtype=torch.bool)
        for j, path in enumerate(_paths(parents)):
            if path is not None:
                mask[j, :cached] = True
                mask[j, [cached + x for x in path]] = True
        mask = mask.cuda()
        some = mask.any(-1)
        for h in range(hkv):
            k, v = s["kc"][i, h, : cached + n].to(F64), s["vc"][i, h, : cached + n].to(F64)
            x = torch.einsum("ngd,kd->ngk", q[i].view(n, hkv, -1, d)[:, h], k) * s["scale"]
            x = x.masked_fill(~mask[:, None], -torch.inf)
            w = torch.softmax(x[some], -1)
            o[i].view(n, hkv, -1, d)[some, h] = w @ v
    return o


def _exact_step(state, q, k, v, g, beta):
    """One token of [batch, heads] recurrences."""
    state = state * g.exp()[..., None, None]
    delta = (v - (state * k[..., None]).sum(-2)) * beta[..., None]
    state = state + k[..., None] * delta[..., None, :]
    return state, (state * q[..., None]).sum(-2)


def _exact_inputs(s):
    hk, hv = s["q"].shape[2], s["v"].shape[2]
    at = torch.arange(hv, device="cuda") // (hv // hk)
    q, k = s["q"].to(F64), s["k"].to(F64)
    if s["case"]["norm"]:
        q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) / q.shape[-1] ** 0.5
        k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    return q[:, :, at], k[:, :, at], s["v"].to(F64), s["g"].to(F64), s["beta"].to(F64)


def _exact_delta(s):
    q, k, v, g, beta = _exact_inputs(s)
    state, o = s["state"].to(F64), torch.zeros_like(v)
    for t in range(q.shape[1]):
        after, row = _exact_step(state, q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t])
        if s["lengths"] is None:
            state, o[:, t] = after, row
        else:
            live = (s["lengths"] > t)[:, None, None]
            state, o[:, t] = torch.where(live[..., None], after, state), torch.where(live, row, 0.0)
    return o, state


def _exact_delta_tree(s):
    q, k, v, g, beta = _exact_inputs(s)
    o = torch.zeros_like(v)
    for i, parents in enumerate(s["parents"].tolist()):
        states = []
        for t, p in enumerate(parents):
            if p < -1 or p >= t:
                states.append(None)
                continue
            before = s["state"][i].to(F64) if p == -1 or states[p] is None else states[p]
            after, o[i, t] = _exact_step(before, q[i, t], k[i, t], v[i, t], g[i, t], beta[i, t])
            states.append(after)
    return o


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    b, op = case["batch"], case["op"]
    if op == "rotary":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        heads = hq + (2 if case["append"] else 1) * hkv
        return {"bytes": 2 * b * t * heads * d * TYPES[case["dtype"]].itemsize + 4 * b * t + 8 * (case["rotary"] // 2), "flops": 6 * b * t * (hq + hkv) * (case["rotary"] // 2)}
    if op == "tree_attention":
        n, hq, hkv, d = case["nodes"], case["hq"], case["hkv"], case["dim"]
        keys = case["context"] + (b - 1) * 0.75 * case["context"] + b * n  # the first sequence is full, the others three quarters on average
        return {"bytes": 4 * keys * hkv * d + 4 * b * n * hq * d + 4 * b * (n + 1), "flops": 4 * keys * n * hq * d}
    t, hk, hv, dk, dv = case["tokens"], case["hk"], case["hv"], case["dk"], case["dv"]
    live = t * (1 + (b - 1) * 2 / 3) if case.get("ragged") else b * t
    states = 1 if op == "delta_tree" else 2
    return {"bytes": live * (4 * hk * dk + 2 * hv * dv + 8 * hv) + b * t * 2 * hv * dv + states * 4 * b * hv * dk * dv, "flops": 7 * live * hv * dk * dv}
