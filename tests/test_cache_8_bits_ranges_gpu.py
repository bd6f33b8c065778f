"""The paged cache in 8 bits where its numbers lie far apart or next to a border, against the definitions in 64 bits.

Tolerances are those of the other tests of this cache: outputs of attention within 2^-7 of the magnitudes that enter the sum
(half a step of bfloat16 is 2^-8, weights in half precision 2^-11 each), codes and scales equal.
"""

import pytest
import torch

from test_cache_8_bits_gpu import DEV, Cache, _attention, _check, _context, _exponent, _nearest, _turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fastgen_b200.csrc.ops import Ops
    return Ops(torch.bfloat16, DEV)


def _copies(ops, k, v, kv, page, copies):
    """A cache whose requests, ``copies`` of them, all read the same pages, which hold ``k`` and ``v``."""
    n, size = k.shape[0], k.shape[1] // kv
    cache = Cache(ops, copies, -(-n // page), kv, page, size, spare=1)
    cache.table[:] = cache.table[:1].clone()
    cache.write(k.to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV), 0, 0)
    return cache


def _check_copies(ops, cache, q, n, heads, copies, scale, sinks=None):
    """Single tokens of requests that all are alike: the first against the formula, the others against the first's."""
    rows = q.to(torch.bfloat16).to(DEV).expand(copies, -1).contiguous()
    out = torch.empty_like(rows)
    ops.attention(rows, out, cache.memory, _context([n - 1] * copies, [1] * copies), heads, cache.kv, cache.size, None, scale, sinks=sinks)
    ops.check_status()
    want, room = _attention(cache, rows[:1], _context([n - 1], [1]), heads, scale, sinks=sinks)
    assert float(room.amin()) > 0
    _check(out, want.expand(copies, -1), room.expand(copies, -1))


@pytest.mark.parametrize("copies", [1, 64])
@pytest.mark.parametrize("sink", [False, True])
def test_sums_over_many_values_of_zero(ops, copies, sink):
    """Ten thousand keys whose values are zero (their pages' scale is 2^-100) before two thousand ordinary ones, all of the same
    weight.  One request is spread over blocks, of 64 a block walks whole stretches of zeros."""
    size, page, kv, n = 64, 64, 8, 12000
    g = torch.Generator().manual_seed(1)
    k = torch.zeros(n, kv * size)
    v = torch.randn(n, kv * size, generator=g) + 2.0
    v[:10000] = 0
    cache = _copies(ops, k, v, kv, page, copies)
    sinks = torch.full((kv,), 9.0, device=DEV) if sink else None  # (e^9 is two thirds of the keys)
    _check_copies(ops, cache, torch.randn(1, kv * size, generator=g), n, kv, copies, 0.125, sinks)


# (scores in natural units and magnitudes of stretches of 32 tokens, four of them to 128 keys)
@pytest.mark.parametrize("scores,magnitudes", [
    ([0, 0], [0.0, 2.0 ** 49]),                      # zeros, then values whose scale is 2^140 of theirs
    ([0, 0], [2.0 ** 49, 0.0]),
    ([0, -4], [2.0 ** -42, 2.0 ** 108]),             # nearly all weight on small values, the sum carried by large ones
    ([-4, 0], [2.0 ** 108, 2.0 ** -42]),
    ([0, 0, 0, 0, -3, -2], [2.0 ** -92, 2.0 ** -30, 1.0, 2.0 ** 40, 2.0 ** 70, 2.0 ** 100]),
    ([0, -30, -60], [0.0, 2.0 ** 20, 2.0 ** 108]),   # the largest weights have no value at all
    ([5, 5, 5, 5], [0.0, 2.0 ** -100, 2.0 ** -91, 2.0 ** -90]),  # the lowest scales
    ([0] * 12, [0.0, 1.0] * 6),
])
@pytest.mark.parametrize("copies", [1, 700])
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_values_far_apart(ops, scores, magnitudes, copies, sink, page):
    size, each = 128, 32
    n = each * len(scores)
    g = torch.Generator().manual_seed(n)
    k = torch.zeros(n, size)
    k[:, 0] = torch.tensor(scores).float().repeat_interleave(each)
    v = (1.0 + torch.rand(n, size, generator=g)) * torch.tensor(magnitudes).repeat_interleave(each)[:, None]
    cache = _copies(ops, k, v, 1, page, copies)
    q = torch.zeros(1, size)
    q[0, 0] = 1.0
    _check_copies(ops, cache, q, n, 1, copies, 1.0, torch.tensor([2.0], device=DEV) if sink else None)


@pytest.mark.parametrize("up", [-60, 0, 60, 108])
def test_capped_scores_of_small_queries_and_large_keys(ops, up):
    """Keys of 2^up against queries of 2^(-up - 4): the scores are ordinary ones, and capped as such."""
    size, n = 128, 200
    g = torch.Generator().manual_seed(3)
    k = torch.rand(n, 1, generator=g).expand(n, size) * 1.7 * 2.0 ** up
    v = torch.randn(n, size, generator=g)
    cache = _copies(ops, k, v, 1, 64, 1)
    q = torch.full((1, size), 1.99 * 2.0 ** (-up - 5), dtype=torch.bfloat16, device=DEV)
    out = torch.empty_like(q)
    ctx = _context([n - 1], [1])
    ops.attention(q, out, cache.memory, ctx, 1, 1, size, None, 0.5, softcap=3.0)
    ops.check_status()
    _check(out, *_attention(cache, q, ctx, 1, 0.5, softcap=3.0))


def _near_borders(size, page, place, magnitude, pairs, seed, factors=None):
    """Rotations (pair, position at slot ``place`` of a page, the two numbers) whose larger result lies within 2^-22 of
    448 * 2^e, and that result in 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    freqs = (10000.0 ** (-torch.arange(size // 2, device=DEV).double() * 2 / size)).float()
    found = []
    for _ in range(24):
        n = 20_000_000
        pair = torch.randint(1, size // 2, (n,), generator=g, device=DEV)
        pos = (torch.randint(1, 4000 // page, (n,), generator=g, device=DEV) * page + place).to(torch.int32)
        a, b = (torch.randn(n, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        angle = (pos.float() * freqs[pair]).double()
        c, s = torch.cos(angle), torch.sin(angle)
        if magnitude != 1.0:
            f = torch.where(pair < pairs, magnitude, 1.0).double()
            c, s = c * f, s * f
        x, y = a.double(), b.double()
        rstd = torch.ones(n, device=DEV)
        if factors is not None:
            rstd = 0.5 + torch.rand(n, generator=g, device=DEV)
            x, y = x * rstd.double() * factors.double()[2 * pair], y * rstd.double() * factors.double()[2 * pair + 1]
        big = torch.maximum((x * c - y * s).abs(), (y * c + x * s).abs())
        m, _e = torch.frexp(big)
        hit = torch.nonzero((m - 0.875).abs() < 0.875 * 2.0 ** -22).flatten()
        found.append((pair[hit], pos[hit], a[hit], b[hit], rstd[hit], big[hit]))
    return freqs, [torch.cat(x) for x in zip(*found)]


@pytest.mark.parametrize("size,page", [(64, 16), (128, 64), (256, 256)])
@pytest.mark.parametrize("way", ["single", "behind", "run", "run behind"])
@pytest.mark.parametrize("option", ["keys", "values", "norm", "norm a head", "magnitude"])
def test_scales_next_to_a_border(ops, size, page, way, option):
    """A page whose largest turned number lies within 2^-22 of 448 * 2^e, on either side of it: the smallest 2^e at which 448
    reaches that number's 64-bit value.  (Float32 sees one in ten of them on the wrong side.)"""
    from dataclasses import replace
    place = 0 if way == "single" else 3
    first = 2 if "behind" in way else 0  # tokens of the page that are cached before
    magnitude, pairs = (1.25, size // 4) if option == "magnitude" else (1.0, 0)
    g = torch.Generator().manual_seed(size)
    weights = (0.5 + torch.rand(size, generator=g)).to(DEV) if option.startswith("norm") else None
    freqs, (pair, pos, a, b, rstd, big) = _near_borders(size, page, place, magnitude, pairs, size + len(way), weights)
    n = pair.numel()
    assert n > 100
    cache = Cache(ops, n, 1, 1, page, size)
    table = cache.table.expand(-1, 4000 // page + 1).contiguous()
    memory = replace(cache.memory, block_table=table)
    tokens = 1 if way in ("single", "behind") else page // 2 + 7
    begin = place if tokens == 1 else first
    rows = torch.zeros(n, tokens, size, dtype=torch.bfloat16, device=DEV)
    each = torch.arange(n, device=DEV)
    rows[each, place - begin, 2 * pair] = a
    rows[each, place - begin, 2 * pair + 1] = b
    rows = rows.view(n * tokens, size)
    nothing = torch.zeros_like(rows)
    start = (pos // page * page)[:, None]
    if first or tokens == 1 and place:
        t = torch.arange(begin, device=DEV, dtype=torch.int32)
        zeros = torch.zeros(n * begin, size, dtype=torch.bfloat16, device=DEV)
        ops.rope_kv8_write(zeros, zeros, zeros, (start + t).flatten().to(torch.int32), each.repeat_interleave(begin).to(torch.int32),
                           None, memory, 1, 1, size)
    at = (start + begin + torch.arange(tokens, device=DEV)).flatten().to(torch.int32)
    req = each.repeat_interleave(tokens).to(torch.int32)
    heads, norm = 1, None
    if option.startswith("norm"):
        heads = 3 if option == "norm a head" else 1
        factors = torch.full((n * tokens, heads + 1), 7.0, device=DEV)  # (the last column is the keys')
        factors[:, -1] = rstd.repeat_interleave(tokens)
        norm = factors, weights.repeat(heads), weights
    k, v = (nothing, rows) if option == "values" else (rows, nothing)
    ops.rope_kv8_write(nothing.repeat(1, heads), k, v, at, req, freqs, memory, heads, 1, size, v_freqs=freqs if option == "values" else None, qk_norm=norm,
                       magnitude=magnitude, rot_pairs=pairs)
    ops.check_status()
    scales = (memory.v_scales if option == "values" else memory.k_scales)[table[:, 0].long(), 0].double()
    assert torch.equal(scales, torch.exp2(_exponent(big).double()))


@pytest.mark.parametrize("size,page,heads,kv", [(64, 16, 6, 2), (128, 64, 8, 4), (256, 128, 4, 2)])
@pytest.mark.parametrize("option", ["plain", "values turned", "norm a token", "norm a head", "magnitude"])
@pytest.mark.parametrize("wide", [0, 3])
def test_all_codes_and_scales_of_mixed_steps(ops, size, page, heads, kv, option, wide):
    """Portions and single tokens, from the start of a page, inside one and behind cached tokens, with rows on and off 16 bytes: every
    code and every scale is the 64-bit numbers'.  (A million numbers: float32 leaves some 25 codes in doubt.)"""
    g = torch.Generator().manual_seed(size + len(option) + wide)
    tokens = 600_000 // (kv * size)
    cached = [0, 5, page - 2, 2 * page + 1, page, 0, 3] + [page + i for i in range(20)]
    new = [tokens // 2, tokens // 4, tokens // 4, 3 * page, 2, 1, 1] + [1] * 20
    cache = Cache(ops, len(new), -(-(max(new) + 4 * page) // page), kv, page, size)
    for s, c in enumerate(cached):
        if c:
            cache.fill(s, c, s, spread=2.0 ** (s % 3 - 1))
    pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)]).to(torch.int32).to(DEV)
    req = torch.cat([torch.full((n,), s) for s, n in enumerate(new)]).to(torch.int32).to(DEV)
    t = pos.numel()
    q, k, v = (torch.randn(t, n * size + wide, generator=g).to(torch.bfloat16).to(DEV)[:, wide:] for n in (heads, kv, kv))
    freqs = (10000.0 ** (-torch.arange(size // 2).double() * 2 / size)).float().to(DEV)
    v_freqs = freqs.flip(0).contiguous() if option == "values turned" else None
    magnitude, pairs = (1.25, size // 4) if option == "magnitude" else (1.0, 0)
    k64, v64 = (x.double().reshape(t, kv, size) for x in (k, v))
    norm = None
    if option.startswith("norm"):
        columns = 2 if option == "norm a token" else heads + kv
        norm = ((0.5 + torch.rand(t, columns, generator=g)).to(DEV), torch.ones(heads * size, device=DEV), (0.5 + torch.rand(kv * size, generator=g)).to(DEV))
        k64 = k64 * (norm[0][:, 1:2] if columns == 2 else norm[0][:, heads:]).double()[:, :, None] * norm[2].double().view(kv, size)
    k64 = _turned(k64, pos, freqs, magnitude, pairs)
    if v_freqs is not None:
        v64 = _turned(v64, pos, v_freqs)
    held = [cache.entries(s, max(c, 1)) for s, c in enumerate(cached)]
    before = [cache.memory.k_scales.clone(), cache.memory.v_scales.clone()]
    ops.rope_kv8_write(q, k, v, pos, req, freqs, cache.memory, heads, kv, size, v_freqs=v_freqs, qk_norm=norm, magnitude=magnitude, rot_pairs=pairs)
    ops.check_status()
    start = 0
    for s, (c, n) in enumerate(zip(cached, new)):
        got = cache.entries(s, c + n)
        for which, mine in enumerate((k64, v64)):
            scales = (cache.memory.k_scales, cache.memory.v_scales)[which]
            for lp in range(c // page, (c + n - 1) // page + 1):
                pid = int(cache.table[s, lp])
                a, b = max(c, lp * page), min(c + n, (lp + 1) * page)
                rows = mine[start + a - c : start + b - c].transpose(0, 1)
                e = _exponent(rows.abs().amax((1, 2)))
                if a > lp * page:
                    e = torch.maximum(e, _exponent(before[which][pid].double() * 448))
                unit = torch.exp2(e.double())
                assert torch.equal(scales[pid].double(), unit), (s, lp, which)
                unit = unit[:, None, None]
                want = torch.cat([_nearest(held[s][which][:, lp * page : a] / unit), _nearest(rows / unit)], 1) * unit
                assert torch.equal(got[which][:, lp * page : b], want), (s, lp, which)
        start += n
