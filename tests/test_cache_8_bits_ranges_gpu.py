"""The paged cache in 8 bits where its numbers lie far apart or next to a border, against the definitions in 64 bits.

Tolerances are those of the other tests of this cache: outputs of attention within 2^-7 of the magnitudes that enter the sum
(half a step of bfloat16 is 2^-8, weights in half precision 2^-11 each), codes and scales equal.
"""

import pytest
import torch

from test_cache_8_bits_gpu import DEV, Cache, _attention, _check, _context

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
