"""Infinities and NaN in keys and values that a token sees: what the formula gives in 64 bits, element by element.

A score of +inf makes its row NaN, a score of -inf has weight 0, a row whose
every score is -inf is 0 / 0; an infinite value is infinite in its own
dimension, however small its weight. Finite elements are held to the bound of
test_gpu_prefix_attention.py, with the largest score and value taken from the
same inputs before the infinities went in: neither an excluded position nor
another dimension adds to the error of what is finite.
"""

import pytest
import torch

from test_gpu_prefix_attention import ALL, UNIT, call, make

pytestmark = pytest.mark.gpu

INF = float("inf")

# ways through the kernels: one pass for prompts, prompts in several key ranges,
# the shared prefix for many rows, everything in the stream kernel
PROMPT = dict(counts=[130], lens=[200], prefix=0, nh=64, nkv=32)
RANGES = dict(counts=[150, 140], lens=[150, 190], prefix=2500, nh=4, nkv=2)
SHARED = dict(counts=[1] * 30, lens=[4] * 30, prefix=700, nh=2, nkv=2)
STREAM = dict(counts=[1, 2], lens=[40, 60], prefix=90, nh=4, nkv=2)


def built(way, page, hd, kind, cache, **kw):
    w = dict(way)
    return list(make(w["counts"], w["lens"], w["prefix"], page, w["nh"], w["nkv"], hd, kind, cache, **kw))


def slots_of(c, page, request):
    """Slots of the positions that the request's last token sees, the prefix's first."""
    table, prefix, block_table, lens = c[3], c[4], c[5], c[6]
    own = torch.arange(int(lens[request]))
    shared = torch.arange(prefix)
    return torch.cat([table.long()[shared // page] * page + shared % page,
                      block_table[request].long()[own // page] * page + own % page])


def reference(c, page):
    """(out, largest sum |q_i k_i| * scale, largest |v|) in float64, a request at a time."""
    q, k, v, _, prefix, _, lens, start = c
    T, nh, hd = q.shape
    G = nh // k.shape[1]
    out = torch.zeros(T, nh, hd, dtype=torch.float64, device="cuda")
    A = V = 0.0
    for i in range(len(lens)):
        a, b, n = int(start[i]), int(start[i + 1]), int(lens[i])
        at = slots_of(c, page, i)
        if a == b or not len(at):
            continue
        x, ki = q[a:b].cuda().double(), k[at].cuda().double().repeat_interleave(G, 1)
        vi = v[at].cuda().double().repeat_interleave(G, 1)
        seen = torch.arange(len(at), device="cuda") <= prefix + n - (b - a) + torch.arange(b - a, device="cuda")[:, None]
        s = torch.einsum("thd,nhd->htn", x, ki) * hd ** -0.5
        p = torch.softmax(torch.where(seen, s, -INF), -1)
        rows = torch.einsum("htn,nhd->thd", p, vi)
        out[a:b] = torch.where(seen.any(1)[:, None, None], rows, 0)
        A = max(A, float(torch.einsum("thd,nhd->htn", x.abs(), ki.abs()).max()) * hd ** -0.5)
        V = max(V, float(vi.abs().max()))
    return out, A, V


def check(out, bad, clean, page, kind, cache):
    ref = reference(bad, page)[0]
    _, A, V = reference(clean, page)
    got = out.double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got == INF, ref == INF) and torch.equal(got == -INF, ref == -INF)
    hd, L = ref.shape[2], bad[4] + int(bad[6].max())
    d = A * (hd / 8 + 4) * 2.0 ** -23
    p = 0.0 if kind == "f32" else UNIT[cache]
    bound = V * (2 * (2 * d + 2.0 ** -20 + p) + (L / 8 + 64) * 2.0 ** -23) + UNIT[kind] * ref.abs() + 2.0 ** -24
    fine = torch.isfinite(ref)
    assert bool(((got - ref).abs() <= bound)[fine].all())
    return ref


def signs(c):
    """q of the first dimension: +1 and -1 in turn."""
    q = c[0]
    q[:, :, 0] = (1 - 2 * (torch.arange(q.shape[0]) % 2)).to(q.dtype)[:, None]


HALVES = [("bf16", "bf16"), ("f16", "f16")]
SINGLE = [("f32", "bf16"), ("f32", "f16")]
INFINITE_KEY = [(PROMPT, 160), (RANGES, 2630), (RANGES, 1000), (SHARED, 640), (STREAM, 80)]
KEY_IDS = ["prompt", "ranges", "ranges-prefix", "shared", "stream"]


def infinite_key(way, first, hd, kind, cache):
    """Scores of +inf and of -inf, by the sign of q, at each of 16 neighbouring positions."""
    page = 16
    clean = built(way, page, hd, kind, cache, seed=hd)
    signs(clean)
    slots = slots_of(clean, page, 0)
    k = clean[1]
    for pos in range(first, first + 16):
        if pos >= len(slots):
            continue
        bad = [clean[0], k.clone(), *clean[2:]]
        bad[1][slots[pos], :, 0] = INF
        ref = check(call(tuple(bad), page), bad, clean, page, kind, cache)
        assert bool(torch.isnan(ref).any()) and bool(torch.isfinite(ref).any())


@pytest.mark.parametrize("kind,cache", HALVES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("way,first", INFINITE_KEY, ids=KEY_IDS)
def test_an_infinite_key(way, first, hd, kind, cache):
    infinite_key(way, first, hd, kind, cache)


@pytest.mark.parametrize("kind,cache", SINGLE)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("way,first", INFINITE_KEY, ids=KEY_IDS)
def test_an_infinite_key_with_fp32_queries(way, first, hd, kind, cache):
    infinite_key(way, first, hd, kind, cache)


def only_minus_infinity(way, hd, kind, cache):
    """0 / 0, as the formula says: not the zeros of a row that sees nothing."""
    page = 16
    clean = built(way, page, hd, kind, cache, seed=hd)
    clean[0][:, :, 0] = -1
    bad = [clean[0], clean[1].clone(), *clean[2:]]
    bad[1][slots_of(clean, page, 0), :, 0] = INF
    ref = check(call(tuple(bad), page), bad, clean, page, kind, cache)
    assert bool(torch.isnan(ref[0]).all())


ONLY = [dict(PROMPT, lens=[130]), dict(STREAM, prefix=0, lens=[1, 2]), dict(STREAM, prefix=3)]
ONLY_IDS = ["prompt", "own", "prefix"]


@pytest.mark.parametrize("kind,cache", HALVES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("way", ONLY, ids=ONLY_IDS)
def test_rows_whose_every_score_is_minus_infinity(way, hd, kind, cache):
    only_minus_infinity(way, hd, kind, cache)


@pytest.mark.parametrize("kind,cache", SINGLE)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("way", ONLY, ids=ONLY_IDS)
def test_rows_whose_every_score_is_minus_infinity_with_fp32_queries(way, hd, kind, cache):
    only_minus_infinity(way, hd, kind, cache)


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("way,positions", [(PROMPT, (0, 37, 70)), (RANGES, (1, 700, 2499, 2500)), (SHARED, (0, 333, 699)),
                                           (STREAM, (0, 89, 90))], ids=["prompt", "ranges", "shared", "stream"])
def test_an_infinite_value(way, positions, hd, kind, cache):
    """Infinite in its own dimension, with its sign; two of opposite sign are NaN there."""
    page = 16
    clean = built(way, page, hd, kind, cache, seed=hd, spread=1.0)
    slots = slots_of(clean, page, 0)
    bad = [clean[0], clean[1], clean[2].clone(), *clean[3:]]
    for pos in positions:
        bad[2][slots[pos], 0, 5] = INF
        bad[2][slots[pos], -1, hd - 1] = -INF
    bad[2][slots[positions[0]], 0, 9] = INF
    bad[2][slots[positions[1]], 0, 9] = -INF
    ref = check(call(tuple(bad), page), bad, clean, page, kind, cache)
    assert bool(torch.isposinf(ref[0, 0, 5])) and bool(torch.isneginf(ref[0, -1, -1])) and bool(torch.isnan(ref[0, 0, 9]))


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("way", [PROMPT, RANGES, SHARED, STREAM], ids=["prompt", "ranges", "shared", "stream"])
def test_an_infinite_value_of_small_weight(way, hd, kind, cache):
    """A weight of e^-25, below what 16-bit floats with 5 exponent bits hold, still counts."""
    page = 16
    clean = built(way, page, hd, kind, cache, seed=hd)
    clean[0][:] = 1
    clean[1][:] = 25 * hd ** -0.5
    slots = slots_of(clean, page, 0)
    clean[1][slots[20]] = 0
    bad = [clean[0], clean[1], clean[2].clone(), *clean[3:]]
    bad[2][slots[20], :, 3] = INF
    ref = check(call(tuple(bad), page), bad, clean, page, kind, cache)
    assert bool(torch.isposinf(ref[0, :, 3]).all())
