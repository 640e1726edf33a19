"""The serving step of a batch whose requests share a long prefix, as measured work.

Three operators, each with its plain form in 32-bit torch operations and the framework's call:
  slots   block tables and slot maps from request lengths (loopspec_b200.slots)
  qk      per-head norm of q and k, rotation, K/V written to their slots (loopspec_b200.qk_norm)
  attn    attention over one shared prefix and each request's own suffix (loopspec_b200.prefix_attention)
"""

import types

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# (query heads, KV heads, head size): the repository's configurations and two generic grouped ones
HEADS = [(4, 4, 64), (4, 1, 64), (2, 2, 128), (32, 8, 64), (16, 16, 128), (32, 8, 128), (28, 4, 128)]


# ------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step: every request gets one token, a few cross into a new block
        {"name": "slots decode 61", "op": "slots", "requests": 61, "page": 16, "longest": 4096, "grow": 1, "shrink": 0},
        # speculative step with page size 1: up to 8 drafts appended, rejected ones rolled back
        {"name": "slots drafts 517", "op": "slots", "requests": 517, "page": 1, "longest": 1024, "grow": 8, "shrink": 8},
        # prompts admitted together: ragged, thousands of tokens each
        {"name": "slots prompts 96", "op": "slots", "requests": 96, "page": 64, "longest": 128, "grow": 2048, "shrink": 0},
        # one token of one request, the smallest call
        {"name": "qk token f32", "op": "qk", "tokens": 1, "heads": 16, "kv_heads": 16, "dim": 128, "rot": 128,
         "type": "f32", "cache": "bf16", "interleaved": False},
        # a decode batch
        {"name": "qk batch bf16", "op": "qk", "tokens": 67, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "type": "bf16", "cache": "bf16", "interleaved": False},
        # a prompt chunk; half of each head is rotated, in neighbouring pairs
        {"name": "qk prompt f16", "op": "qk", "tokens": 8191, "heads": 16, "kv_heads": 16, "dim": 128, "rot": 64,
         "type": "f16", "cache": "f16", "interleaved": True},
        # the tiny model: four requests behind a short prefix
        {"name": "attn tiny", "op": "attn", "requests": 4, "new": 1, "prefix": 333, "suffix": 65, "page": 1,
         "heads": 4, "kv_heads": 4, "dim": 64, "type": "f32", "cache": "bf16"},
        # a decode batch of the 16-head model in the engine's own types, page size 1
        {"name": "attn decode f32", "op": "attn", "requests": 16, "new": 1, "prefix": 2048, "suffix": 700, "page": 1,
         "heads": 16, "kv_heads": 16, "dim": 128, "type": "f32", "cache": "bf16"},
        # a large decode batch behind a long document, grouped heads
        {"name": "attn decode long", "op": "attn", "requests": 64, "new": 1, "prefix": 32768, "suffix": 513, "page": 16,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "cache": "bf16"},
        # speculative lanes: up to five tokens for each request, some with none
        {"name": "attn drafts f16", "op": "attn", "requests": 33, "new": 5, "prefix": 5001, "suffix": 1400, "page": 64,
         "heads": 28, "kv_heads": 4, "dim": 128, "type": "f16", "cache": "f16"},
        # question prompts behind a shared document: thousands of query rows
        {"name": "attn prompts", "op": "attn", "requests": 8, "new": 509, "prefix": 16384, "suffix": 600, "page": 16,
         "heads": 32, "kv_heads": 8, "dim": 64, "type": "bf16", "cache": "bf16"},
        {"name": "attn prompts wide", "op": "attn", "requests": 4, "new": 700, "prefix": 8192, "suffix": 700, "page": 32,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "cache": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        cost = w["bytes"] + w["flops"] / 200
        most[c["op"]] = max(most.get(c["op"], 0), cost)
    while True:
        op = rng.choice(["slots", "qk", "attn", "attn"])
        if op == "slots":
            c = {"op": op, "requests": _log(rng, 1, 2048), "page": rng.choice([1, 16, 32, 64, 128]),
                 "longest": _log(rng, 16, 4096), "grow": _log(rng, 1, 2048), "shrink": rng.choice([0, 0, 8, 100])}
        else:
            heads, kv_heads, dim = rng.choice(HEADS)
            cache = rng.choice(["bf16", "bf16", "f16"])
            kind = rng.choice([cache, cache, "f32"])
            c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "type": kind, "cache": cache}
            if op == "qk":
                c.update(tokens=_log(rng, 1, 8192), rot=rng.choice([dim, dim, dim // 2]),
                         interleaved=rng.random() < 0.3)
            else:
                new = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 700)])
                c.update(requests=_log(rng, 1, 128), new=new, prefix=_log(rng, 64, 40000),
                         suffix=max(new, _log(rng, 8, 2000)), page=rng.choice([1, 16, 32, 64, 128]))
        w = work(c)
        rows = c.get("requests", 1) * c.get("new", 1) * c.get("heads", 1)
        scores = rows * (c.get("prefix", 0) + c.get("suffix", 0))     # the plain form holds them all
        if w["bytes"] + w["flops"] / 200 <= most[op] and scores <= 2.2e9:
            return c


def work(case):
    if case["op"] == "slots":
        r, g = case["requests"], case["grow"]
        tokens = r if g == 1 else r * g / 2
        blocks = tokens / case["page"]
        return {"bytes": 4 * (4 * r + 3 * tokens + 2 * blocks), "flops": 0}
    size, cache = DTYPES[case["type"]].itemsize, DTYPES[case["cache"]].itemsize
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "qk":
        t = case["tokens"]
        moved = t * d * ((h + 2 * kv) * size + h * size + 2 * kv * cache) + t * (4 * case["rot"] + 8)
        return {"bytes": moved, "flops": t * (h + kv) * d * 8}
    r, new, p, s = (case[k] for k in ("requests", "new", "prefix", "suffix"))
    tokens = max(1, _mean_new(new) * r)
    own_keys = r * (s + new) / 2 if s > new else r * s         # suffix lengths are spread over [new, s]
    seen = tokens * p + own_keys * _mean_new(new) - (r * _mean_new(new) ** 2 / 2 if new > 1 else 0)
    return {"bytes": (p + own_keys) * kv * d * 2 * cache + 2 * tokens * h * d * size, "flops": 4 * h * d * seen}


def _mean_new(new):
    return 1 if new == 1 else new / 2 if new <= 8 else 0.75 * new


# ------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = types.SimpleNamespace(case=case, op=case["op"])
    {"slots": _prepare_slots, "qk": _prepare_qk, "attn": _prepare_attn}[case["op"]](s, case, g)
    return s


def _ints(g, low, high, n):
    """n whole numbers of [low, high], on the GPU."""
    return torch.randint(low, high + 1, (n,), generator=g, device="cuda", dtype=torch.int64)


def _spread(g, low, high, n):
    """n whole numbers spread evenly over [low, high], high among them, in an order of the seed's: their sum is the case's."""
    even = high - (torch.arange(n, dtype=torch.int64, device="cuda") * (high - low + 1)).div(n, rounding_mode="floor")
    return even[torch.randperm(n, generator=g, device="cuda")]


def _prepare_slots(s, case, g):
    r, page = case["requests"], case["page"]
    s.page, s.base = page, 1000
    lens = _spread(g, 0, case["longest"], r)
    if case["grow"] == 1 and not case["shrink"]:
        delta = torch.ones_like(lens)
    else:
        delta = _spread(g, -case["shrink"], case["grow"], r).maximum(-lens)
    have = (lens + page - 1) // page
    width = (case["longest"] + case["grow"]) // page + 1
    s.n_blocks = int(have.sum()) + r * (case["grow"] // page + 2)
    order = torch.randperm(s.n_blocks, generator=g, device="cuda").to(torch.int32)
    start = have.cumsum(0) - have
    col = torch.arange(width, device="cuda")
    at = (start[:, None] + col).clamp(max=s.n_blocks - 1)
    s.table = torch.where(col < have[:, None], order[at], -1).contiguous()
    used = int(have.sum())
    s.free = torch.full((s.n_blocks,), -1, dtype=torch.int32, device="cuda")
    s.free[: s.n_blocks - used] = order[used:]
    s.count = torch.tensor([s.n_blocks - used], dtype=torch.int32, device="cuda")
    s.lens, s.delta = lens.to(torch.int32), delta.to(torch.int32)
    s.max_tokens = -(-int(delta.clamp(min=0).sum()) // 64) * 64 + 64     # a buffer with room to spare
    _with_own_slots(s)


def _prepare_qk(s, case, g):
    t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    kind, cache = DTYPES[case["type"]], DTYPES[case["cache"]]
    s.heads, s.kv_heads, s.dim, s.rot, s.eps = h, kv, d, case["rot"], 1e-6
    s.interleaved = case["interleaved"]
    scale = torch.rand(h + 2 * kv, 1, generator=g, device="cuda") * 3 + 0.2
    x = torch.randn(t, h + 2 * kv, d, generator=g, device="cuda") * scale
    s.qkv = x.to(kind).view(t, -1)
    s.q_weight = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
    s.k_weight = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
    limit = 32768
    inv = 10000.0 ** (-torch.arange(0, s.rot, 2, dtype=torch.float64, device="cuda") / s.rot)
    angle = torch.arange(limit, dtype=torch.float64, device="cuda")[:, None] * inv
    s.rope = torch.stack([angle.cos(), angle.sin()], 1).to(torch.float32)       # [limit, 2, rot / 2]
    s.positions = _ints(g, 0, limit - 1, t).to(torch.int32)
    n_slots = t + t // 4 + 16
    s.slots = torch.randperm(n_slots, generator=g, device="cuda")[:t].to(torch.int32)
    s.k_pool = torch.zeros(n_slots, kv, d, dtype=cache, device="cuda")
    s.v_pool = torch.zeros(n_slots, kv, d, dtype=cache, device="cuda")
    s.out = torch.empty(t, h, d, dtype=kind, device="cuda")
    _with_status(s)


def _prepare_attn(s, case, g):
    r, new, p, page = case["requests"], case["new"], case["prefix"], case["page"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    kind, cache = DTYPES[case["type"]], DTYPES[case["cache"]]
    if new == 1:
        count = torch.ones(r, dtype=torch.int64, device="cuda")
    else:
        count = _spread(g, 0 if new <= 8 else new // 2, new, r)
    lens = _ints(g, min(new, case["suffix"]), case["suffix"], r).maximum(count)
    s.max_new, s.max_len = new, int(max(new, case["suffix"]))
    s.prefix, s.page, s.scale = p, page, d ** -0.5
    width = -(-s.max_len // page)
    prefix_blocks = -(-p // page)
    n_blocks = prefix_blocks + r * width + 3
    order = torch.randperm(n_blocks, generator=g, device="cuda").to(torch.int32)
    s.prefix_table = order[:prefix_blocks].contiguous()
    s.table = order[prefix_blocks:prefix_blocks + r * width].view(r, width).contiguous()
    s.lens = lens.to(torch.int32)
    start = torch.zeros(r + 1, dtype=torch.int64, device="cuda")
    start[1:] = count.cumsum(0)
    s.start = start.to(torch.int32)
    t = int(start[-1])
    s.requests = torch.repeat_interleave(torch.arange(r, device="cuda"), count)
    s.k_pool = torch.randn(n_blocks * page, kv, d, generator=g, device="cuda").to(cache)
    s.v_pool = torch.randn(n_blocks * page, kv, d, generator=g, device="cuda").to(cache)
    s.q = (2.5 * torch.randn(t, h, d, generator=g, device="cuda")).to(kind)
    s.out = torch.empty_like(s.q)
    _with_own_attn(s)


def _with_status(s):
    s.status = None
    if own:
        from loopspec_b200.status import DeviceStatus
        s.status = DeviceStatus("cuda")


def _with_own_slots(s):
    """The buffers that a program keeps for the slot maps."""
    _with_status(s)
    if own:
        from loopspec_b200.slots import SlotMap
        s.map = SlotMap(s.lens.numel(), s.max_tokens, "cuda")


def _with_own_attn(s):
    """The workspace that a program keeps for the attention."""
    _with_status(s)
    if own:
        from loopspec_b200.prefix_attention import workspace_bytes
        need = workspace_bytes(s.q.shape[0], s.q.shape[1], s.k_pool.shape[1], s.q.shape[2],
                               n_requests=s.lens.numel(), prefix_len=s.prefix, max_new=s.max_new, max_len=s.max_len)
        s.workspace = torch.zeros(need, dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------------ passes
def run(state):
    if own:
        return {"slots": _own_slots, "qk": _own_qk, "attn": _own_attn}[state.op](state)
    return {"slots": _plain_slots, "qk": _plain_qk, "attn": _plain_attn}[state.op](state)


def _own_slots(s):
    from loopspec_b200.slots import build_slots
    m = build_slots(s.lens, s.delta, s.table, s.free, s.count, page_size=s.page, n_blocks=s.n_blocks, base=s.base,
                    out=s.map, status=s.status)
    return [m.slots, m.positions, m.requests, m.token_start, m.lens, m.free_count, s.table, s.free]


def _own_qk(s):
    from loopspec_b200.qk_norm import qk_norm_rope
    q = qk_norm_rope(s.qkv, s.q_weight, s.k_weight, s.rope, s.positions, s.k_pool, s.v_pool, s.slots, eps=s.eps,
                     interleaved=s.interleaved, out=s.out, status=s.status)
    return [q, s.k_pool, s.v_pool]


def _own_attn(s):
    from loopspec_b200.prefix_attention import prefix_attention
    return prefix_attention(s.q, s.k_pool, s.v_pool, s.prefix_table, s.prefix, s.table, s.lens, s.start,
                            page_size=s.page, max_new=s.max_new, max_len=s.max_len, scale=s.scale, out=s.out,
                            workspace=s.workspace, status=s.status)


def _plain_slots(s):
    page, limit = s.page, s.max_tokens
    lens, delta = s.lens.long(), s.delta.long()
    new = lens + delta
    have, need = (lens + page - 1) // page, (new + page - 1) // page
    grow, back = (need - have).clamp(min=0), (have - need).clamp(min=0)
    grow_end, back_end, tok = grow.cumsum(0), back.cumsum(0), delta.clamp(min=0)
    count, tok_end = s.count.long(), tok.cumsum(0)
    r, width = s.table.shape
    col = torch.arange(width, device="cuda")
    # blocks given back go on the stack in request order, then in block order; one spare place takes what is not given
    gives = (col >= need[:, None]) & (col < have[:, None])
    place = count + (back_end - back)[:, None] + col - need[:, None]
    cap = s.free.numel()
    stack = torch.cat([s.free, s.free.new_zeros(r * width + 1)])
    spare = stack.numel() - 1
    stack[torch.where(gives, place, spare)] = s.table
    # the k-th new block is the k-th from the top
    takes = (col >= have[:, None]) & (col < need[:, None])
    top = count + back_end[-1] - 1 - ((grow_end - grow)[:, None] + col - have[:, None])
    s.table = torch.where(takes, stack[top.clamp(min=0, max=spare)], s.table)
    count = count + back_end[-1] - grow_end[-1]
    at = torch.arange(cap, device="cuda")
    s.free = torch.where((at >= s.count) & (at < count), stack[:cap], s.free)
    # the new tokens
    k = torch.arange(limit, device="cuda")
    i = torch.searchsorted(tok_end, k, right=True)
    live = k < tok_end[-1]
    i = i.clamp(max=r - 1)
    pos = lens[i] + k - (tok_end - tok)[i]
    slot = s.table[i, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    int32 = torch.int32
    start = torch.cat([tok_end.new_zeros(1), tok_end]).to(int32)
    return [torch.where(live, slot, -1).to(int32), torch.where(live, pos + s.base, 0).to(int32),
            torch.where(live, i, -1).to(int32), start, new.to(int32), count.to(int32), s.table, s.free]


def _plain_qk(s):
    t, h, kv, d, rot = s.qkv.shape[0], s.heads, s.kv_heads, s.dim, s.rot
    x = s.qkv.view(t, h + 2 * kv, d).float()
    qk = x[:, :h + kv]
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + s.eps)
    weight = torch.cat([s.q_weight.float().expand(h, d), s.k_weight.float().expand(kv, d)])
    qk = qk * weight
    table = s.rope[s.positions.long()][:, None]
    c, sn = table[:, :, 0], table[:, :, 1]
    if s.interleaved:
        a, b = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    else:
        a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    qk = torch.cat([turned, qk[..., rot:]], -1)
    slots = s.slots.long()
    s.k_pool[slots] = qk[:, h:].to(s.k_pool.dtype)
    s.v_pool[slots] = x[:, h + kv:].to(s.v_pool.dtype)
    return [qk[:, :h].to(s.qkv.dtype), s.k_pool, s.v_pool]


def _plain_attn(s):
    t, h, d = s.q.shape
    kv, r = s.k_pool.shape[1], s.lens.numel()
    group, page = h // kv, s.page
    q = s.q.float().view(t, kv, group, d) * s.scale
    # the prefix, once for all
    j = torch.arange(s.prefix, device="cuda")
    slots = s.prefix_table[j // page].long() * page + j % page
    k, v = s.k_pool[slots].float(), s.v_pool[slots].float()
    by_head = q.permute(1, 0, 2, 3).reshape(kv, t * group, d)
    far = torch.matmul(by_head, k.permute(1, 2, 0))                                   # [kv, t * group, prefix]
    # each request's own keys, with the queries padded to max_new a request
    l = torch.arange(s.max_len, device="cuda")
    lens, start = s.lens.long(), s.start.long()
    inside = l < lens[:, None]
    at = torch.where(inside, s.table[:, l // page].long() * page + l % page, 0)
    own_k = s.k_pool[at].float()
    own_v = torch.where(inside[:, :, None, None], s.v_pool[at].float(), 0)
    n = start[1:] - start[:-1]
    step = torch.arange(s.max_new, device="cuda")
    token = (start[:-1, None] + step).clamp(max=t - 1)
    padded = q[token].permute(0, 2, 1, 3, 4).reshape(r, kv, s.max_new * group, d)
    near = torch.matmul(padded, own_k.permute(0, 2, 3, 1))                            # [r, kv, max_new * group, max_len]
    seen = inside[:, None] & (l <= (lens - n)[:, None, None] + step[:, None])         # [r, max_new, max_len]
    near = near.view(r, kv, s.max_new, group, -1).masked_fill(~seen[:, None, :, None], float("-inf"))
    i = s.requests
    nth = torch.arange(t, device="cuda") - start[i]
    near_t = near[i, :, nth].permute(1, 0, 2, 3).reshape(kv, t * group, -1)           # [kv, t * group, max_len]
    top = torch.maximum(far.amax(-1), near_t.amax(-1))[..., None]
    far = torch.exp(far - top)
    near_t = torch.exp(near_t - top)
    total = far.sum(-1) + near_t.sum(-1)
    out = torch.matmul(far, v.permute(1, 0, 2)).view(kv, t, group, d)
    weights = torch.zeros_like(near)
    weights[i, :, nth] = near_t.view(kv, t, group, -1).transpose(0, 1)
    mine = torch.matmul(weights.view(r, kv, s.max_new * group, -1), own_v.permute(0, 2, 1, 3))
    mine = mine.view(r, kv, s.max_new, group, d)[i, :, nth]
    out = (out.transpose(0, 1) + mine) / total.view(kv, t, group, 1).transpose(0, 1)
    return out.reshape(t, h, d).to(s.q.dtype)


# ------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["op"] == "slots":
        return None                      # whole numbers
    s = prepare(case, seed)
    if case["op"] == "qk":
        return _exact_qk(s)
    if work(case)["flops"] > 6e11:
        return None
    return _exact_attn(s)


def _exact_qk(s):
    t, h, kv, d, rot = s.qkv.shape[0], s.heads, s.kv_heads, s.dim, s.rot
    x = s.qkv.double().view(t, h + 2 * kv, d)

    def normed(part, weight):
        return part / (part.pow(2).sum(-1, keepdim=True) / d + s.eps).sqrt() * weight.double()

    # a rotation is a product of complex numbers
    turn = torch.view_as_complex(s.rope.double()[s.positions.long()].transpose(1, 2).contiguous())[:, None]

    def turned(part):
        head = part[..., :rot]
        if s.interleaved:
            z = torch.view_as_complex(head.reshape(t, -1, rot // 2, 2).contiguous()) * turn
            head = torch.view_as_real(z).reshape(t, -1, rot)
        else:
            z = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * turn
            head = torch.cat([z.real, z.imag], -1)
        return torch.cat([head, part[..., rot:]], -1)

    k_pool, v_pool = s.k_pool.double(), s.v_pool.double()
    k_pool[s.slots.long()] = turned(normed(x[:, h:h + kv], s.k_weight))
    v_pool[s.slots.long()] = x[:, h + kv:]
    return [turned(normed(x[:, :h], s.q_weight)), k_pool, v_pool]


def _exact_attn(s):
    """Request by request: the prefix's and the request's own rows in one list, one softmax over it."""
    t, h, d = s.q.shape
    kv = s.k_pool.shape[1]
    out = torch.zeros(t, h, d, dtype=torch.float64, device="cuda")
    page = s.page

    def rows(table, n):
        offset = torch.arange(page, device="cuda")
        return (table.long()[:, None] * page + offset).flatten()[:n]

    start, lens = s.start.tolist(), s.lens.tolist()
    shared = rows(s.prefix_table, s.prefix)
    for i, length in enumerate(lens):
        a, b = start[i], start[i + 1]
        if a == b:
            continue
        at = torch.cat([shared, rows(s.table[i], length)])
        hidden = torch.ones(b - a, length, dtype=torch.bool, device="cuda").triu(length - (b - a) + 1)
        hidden = torch.cat([hidden.new_zeros(b - a, s.prefix), hidden], 1)
        for head in range(h):
            of = head // (h // kv)
            score = s.q[a:b, head].double() @ s.k_pool[at, of].double().T * s.scale
            weight = torch.softmax(score.masked_fill(hidden, -torch.inf), -1)
            out[a:b, head] = weight @ s.v_pool[at, of].double()
    return out
