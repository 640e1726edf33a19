"""Plain 64-bit restatements of the shared-prefix operators, on the CPU, written from their formulas."""

import torch


def slots_reference(lens, delta, table, stack, count, page):
    """Lists in, lists out: (tokens [(slot, position, request)], start, lens, table, stack, count)."""
    lens, table, stack = list(lens), [list(r) for r in table], list(stack)
    blocks = [-(-n // page) for n in lens]
    free = stack[:count]
    for i, d in enumerate(delta):
        need = -(-(lens[i] + d) // page)
        free += table[i][need:blocks[i]] if need < blocks[i] else []
    tokens, start = [], [0]
    for i, d in enumerate(delta):
        for b in range(blocks[i], -(-(lens[i] + d) // page)):
            table[i][b] = free.pop()
        for pos in range(lens[i], lens[i] + d):
            tokens.append((table[i][pos // page] * page + pos % page, pos, i))
        start.append(len(tokens))
        lens[i] += d
    # entries of the stack that no push reached keep their old values
    height = len(free)
    stack[count:height] = free[count:height]
    return tokens, start, lens, table, stack, height


def qk_norm_reference(qkv, q_weight, k_weight, rope, positions, n_heads, n_kv, hd, eps, interleaved):
    """(q, k, v) in float64 from any input types."""
    x = qkv.double().view(qkv.shape[0], n_heads + 2 * n_kv, hd)
    rot = 2 * rope.shape[2]
    table = rope.double()[positions.long()]
    c, s = table[:, None, 0], table[:, None, 1]

    def one(part, weight):
        y = part / torch.sqrt((part * part).mean(-1, keepdim=True) + eps) * weight.double()
        out = y.clone()
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        return out
    return one(x[:, :n_heads], q_weight), one(x[:, n_heads:n_heads + n_kv], k_weight), x[:, n_heads + n_kv:]


def table_slots(table, n, page):
    pos = torch.arange(n)
    return table.long()[pos // page] * page + pos % page


def prefix_attention_reference(q, k_pool, v_pool, prefix_table, prefix_len, block_table, lens, start, page, scale):
    """(out float64 [T, nh, hd], largest sum |q_i k_i| * scale over the visible pairs, largest visible |v|),
    one token at a time over the positions that it sees."""
    T, nh, hd = q.shape
    G = nh // k_pool.shape[1]
    out = torch.zeros(T, nh, hd, dtype=torch.float64)
    most_score = most_v = 0.0
    shared = table_slots(prefix_table, prefix_len, page) if prefix_len else torch.zeros(0, dtype=torch.long)
    for i in range(len(lens)):
        n = int(start[i + 1] - start[i])
        own = table_slots(block_table[i], int(lens[i]), page) if int(lens[i]) else shared[:0]
        for j in range(n):
            t = int(start[i]) + j
            at = torch.cat([shared, own[:max(0, int(lens[i]) - n + j + 1)]])
            if not len(at):
                continue
            k = k_pool[at].double().repeat_interleave(G, 1)
            v = v_pool[at].double().repeat_interleave(G, 1)
            s = torch.einsum("hd,nhd->hn", q[t].double(), k) * scale
            out[t] = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), v)
            most_score = max(most_score, float(torch.einsum("hd,nhd->hn", q[t].double().abs(), k.abs()).max()) * scale)
            most_v = max(most_v, float(v.abs().max()))
    return out, most_score, most_v
