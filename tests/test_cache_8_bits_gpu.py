"""The paged cache in 8 bits: its write, its values, and attention over it, against the definitions in 64 bits.

Tolerances.  A code is the nearest e4m3 number of an entry over its scale.  The kernel rotates in float32, where the entry
may be a few 2^-24 off, so a code next to a border may be the neighbouring one: an entry is then one step off, at most
2^-3 of itself (twice the half step, 2^-4) or 2^-9 scales, and such entries are fewer than one in a thousand.  Without a
rotation codes are equal.  Outputs of attention are rounded to bfloat16 (2^-8 of the value at most, half a step) on top of
weights in half precision (2^-11 of each) and sums in float32: 2^-7 of the largest magnitude that enters the sum holds them.
"""

from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from fastgen_b200.csrc.ops import Ops
    return Ops(torch.bfloat16, DEV)


def _code_values():
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        out.append(float("nan") if c & 127 == 127 else -v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _nearest(x):
    """x rounded to the nearest e4m3 number, ties to even; NaN where it is not finite."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp_min(-6) - 3)
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, torch.full_like(x, float("nan")))


def _exponent(amax):
    """The smallest whole e in [-100, 100] with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax)
    e = e - 9 + (m > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(-100, 100)


def _log2(scale):
    """The exponent of a power of two (torch.log2 may be off by a last place)."""
    return torch.frexp(scale)[1] - 1


class Cache:
    """A cache in 8 bits of one run, with what it stands for beside it in 64 bits."""

    def __init__(self, ops, slots, width, kv, page, size, layers=1, layer=0, spare=3):
        from fastgen_b200.cache import LayerMemory
        self.kv, self.page, self.size, self.width = kv, page, size, width
        n = slots * width + spare
        g = torch.Generator().manual_seed(slots * 31 + width)
        # what a former owner left: any codes, NaN codes among them
        pools = [torch.randint(0, 256, (layers, n, kv, page * size), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2)]
        for p in pools:
            p[..., ::7] = 0x7F
        self.k_pool = pools[0].view(layers, n, kv, page, size).view(torch.float8_e4m3fn)
        self.v_pool = pools[1].view(layers, n, kv, page // 4, size, 4).view(torch.float8_e4m3fn)
        self.scales = [torch.exp2(torch.randint(-20, 20, (layers, n, kv), generator=g).float()).to(DEV) for _ in range(2)]
        self.table = torch.randperm(n, generator=g)[: slots * width].view(slots, width).to(torch.int32).to(DEV)
        self.memory = LayerMemory(k_pages=self.k_pool[layer], v_pages=self.v_pool[layer], block_table=self.table, page_size=page,
                                  k_scales=self.scales[0][layer], v_scales=self.scales[1][layer],
                                  tensor_maps=ops.make_kv8_tensor_maps(self.k_pool, self.v_pool), layer_index=layer)
        self.ops = ops
        self.values = _code_values()

    def entries(self, slot, n):
        """What the first ``n`` tokens of a request stand for: keys and values [kv, n, size] in 64 bits."""
        mem, pages = self.memory, self.table[slot, : -(-n // self.page)].long()
        k = self.values[mem.k_pages.view(torch.uint8)[pages].long()] * mem.k_scales[pages].double()[..., None, None]
        v = self.values[mem.v_pages.view(torch.uint8)[pages].long()] * mem.v_scales[pages].double()[..., None, None, None]
        k = k.permute(1, 0, 2, 3).reshape(self.kv, -1, self.size)[:, :n]
        v = v.permute(1, 0, 2, 4, 3).reshape(self.kv, -1, self.size)[:, :n]
        return k, v

    def fill(self, slot, n, seed, spread=1.0):
        """Tokens 0 .. n - 1 of a request written in two portions without a rotation."""
        g = torch.Generator().manual_seed(seed)
        x = [(torch.randn(n, self.kv * self.size, generator=g) * spread).to(torch.bfloat16).to(DEV) for _ in range(2)]
        cut = n // 3
        for a, b in ((0, cut), (cut, n)):
            if a < b:
                self.write(x[0][a:b], x[1][a:b], slot, a)

    def write(self, k, v, slot, start, **options):
        t = k.shape[0]
        pos = torch.arange(start, start + t, dtype=torch.int32, device=DEV)
        req = torch.full((t,), slot, dtype=torch.int32, device=DEV)
        q = torch.zeros(t, self.kv * self.size, dtype=torch.bfloat16, device=DEV)
        return self.ops.rope_kv8_write(q, k, v, pos, req, None, self.memory, self.kv, self.kv, self.size, **options)


def _context(cached, new, slots=None):
    """A step's context: sequences that hold ``cached`` tokens and bring ``new``."""
    from fastgen_b200.engine.step import StepContext
    ctx = StepContext(torch.device(DEV))
    slots = list(range(len(cached))) if slots is None else slots
    ctx.pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)]).to(torch.int32).to(DEV)
    ctx.req = torch.cat([torch.full((n,), s) for s, n in zip(slots, new)]).to(torch.int32).to(DEV)
    ctx.host_seq_slot, ctx.host_seq_cached = slots, list(cached)
    for n in new:
        ctx.host_seq_start.append(ctx.host_seq_start[-1] + n)
    ctx.n_tokens, ctx.n_seqs, ctx.longest = sum(new), len(new), max(new)
    ctx.seq_slot, ctx.seq_start, ctx.seq_cached = (
        torch.tensor(x, dtype=torch.int32, device=DEV) for x in (slots, ctx.host_seq_start, list(cached)))
    return ctx


# -- the write -------------------------------------------------------------------------------------


def _turned(x, pos, freqs, magnitude=1.0, pairs=None):
    a = (pos.float()[:, None] * freqs[None, :]).double()
    c, s = torch.cos(a), torch.sin(a)
    if magnitude != 1.0:
        c[:, :pairs] *= magnitude
        s[:, :pairs] *= magnitude
    re, im = x[..., 0::2], x[..., 1::2]
    c, s = c[:, None], s[:, None]
    return torch.stack([re * c - im * s, im * c + re * s], 3).flatten(2)


@pytest.mark.parametrize("size,page,heads,kv", [(64, 16, 3, 1), (64, 64, 8, 2), (128, 32, 14, 2), (128, 64, 32, 8), (128, 256, 4, 4), (256, 128, 10, 5)])
@pytest.mark.parametrize("option", ["plain", "values turned", "norm a token", "norm a head", "off 16 bytes", "magnitude"])
def test_write_of_mixed_steps(ops, size, page, heads, kv, option):
    """Several portions and single tokens, behind cached entries, over page edges, with padding between: queries, scales and
    codes by the definition; pages of others, and slots behind the last token, stay as they were."""
    g = torch.Generator().manual_seed(size + page + len(option))
    lengths = [(0, 2 * page + 3), (page - 1, 1), (page - 2, 5), (page, 1), (0, 1), (5, page + 7), (3 * page - 1, 1), (2, 3)]
    cache = Cache(ops, len(lengths), 5, kv, page, size)
    for s, (cached, _) in enumerate(lengths):
        if cached:
            cache.fill(s, cached, s)
    # tokens of request -1 between the sequences: nothing of theirs is written
    pos, req = [], []
    for s, (cached, n) in enumerate(lengths):
        pos += list(range(cached, cached + n)) + [0, 1]
        req += [s] * n + [-1, -1]
    pos, req = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (pos, req))
    t = pos.numel()
    wide = 3 if option == "off 16 bytes" else 0
    rows = [torch.randn(t, n * size + wide, generator=g).to(torch.bfloat16).to(DEV)[:, wide:] for n in (heads, kv, kv)]
    q, k, v = rows
    v[3] *= 300.0  # one token far larger than its page
    k[-3] *= 2.0 ** -40
    freqs = (10000.0 ** (-torch.arange(size // 2).double() * 2 / size)).float().to(DEV)
    v_freqs = freqs.flip(0).contiguous() if option == "values turned" else None
    norm, factors = None, None
    if option == "norm a token":
        rstd = (0.5 + torch.rand(t, 2, generator=g)).to(DEV)
        norm = (rstd, torch.rand(heads * size, generator=g).to(DEV), torch.rand(kv * size, generator=g).to(DEV))
        factors = [rstd[:, :1].double(), rstd[:, 1:].double()]
    elif option == "norm a head":
        rstd = (0.5 + torch.rand(t, heads + kv, generator=g)).to(DEV)
        norm = (rstd, torch.rand(heads * size, generator=g).to(DEV), None)
        factors = [rstd[:, :heads].double(), rstd[:, heads:].double()]
    magnitude, pairs = (1.25, size // 4) if option == "magnitude" else (1.0, 0)
    before = [x.clone() for x in (cache.memory.k_pages.view(torch.uint8), cache.memory.v_pages.view(torch.uint8), *[s for s in (cache.memory.k_scales, cache.memory.v_scales)])]
    held = [cache.entries(s, max(c, 1)) for s, (c, _) in enumerate(lengths)]
    out = ops.rope_kv8_write(q, k, v, pos, req, freqs, cache.memory, heads, kv, size, v_freqs=v_freqs, qk_norm=norm,
                             magnitude=magnitude, rot_pairs=pairs)
    ops.check_status()
    q64, k64, v64 = (x.double().view(t, -1, size) for x in (q, k, v))
    if norm is not None:
        q64 = q64 * factors[0][..., None] * (norm[1].double().view(heads, size) if norm[1] is not None else 1.0)
        k64 = k64 * factors[1][..., None] * (norm[2].double().view(kv, size) if norm[2] is not None else 1.0)
    q64, k64 = _turned(q64, pos, freqs, magnitude, pairs), _turned(k64, pos, freqs, magnitude, pairs)
    if v_freqs is not None:
        v64 = _turned(v64, pos, v_freqs)
    live = req >= 0
    want_q = q64.flatten(1)[live]
    assert bool(((out[live].double() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -20 * (1 + want_q.abs().amax(1, keepdim=True))).all())
    touched, off, total = set(), 0, 0
    start = 0
    for s, (cached, n) in enumerate(lengths):
        for which, new in (("k", k64), ("v", v64)):
            got = cache.entries(s, cached + n)[which == "v"]
            old = held[s][which == "v"][:, :cached]
            scales = cache.memory.k_scales if which == "k" else cache.memory.v_scales
            old_scales = before[2 + (which == "v")]
            for lp in range(cached // page, (cached + n - 1) // page + 1):
                pid = int(cache.table[s, lp])
                touched.add(pid)
                a, b = max(cached, lp * page), min(cached + n, (lp + 1) * page)
                mine = new[start + a - cached : start + b - cached]  # [tokens, kv, size]
                e = _exponent(mine.abs().amax((0, 2)))
                if a > lp * page:
                    e = torch.maximum(e, _log2(old_scales[pid]).to(e.dtype))
                # (a largest entry next to a border may take either exponent)
                got_e = _log2(scales[pid]).to(e.dtype)
                assert bool(((got_e - e).abs() <= (0 if which == "v" and v_freqs is None else 1)).all()), (s, lp, which)
                unit = scales[pid].double()[:, None, None]
                want = torch.cat([_nearest(old[:, lp * page : a] / unit), _nearest(mine.transpose(0, 1) / unit)], 1) * unit
                diff = (got[:, lp * page : b] - want).abs()
                exact = which == "v" and v_freqs is None
                assert bool((diff <= (0.0 if exact else 1.0) * torch.maximum(2.0 ** -3 * want.abs(), 2.0 ** -9 * unit)).all()), (s, lp, which)
                off, total = off + int((diff > 0).sum()), total + diff.numel()
        start += n + 2
    assert off <= total // 1000
    # nothing else has changed: other pages, and the slots behind the last token
    others = torch.tensor([p for p in range(before[0].shape[0]) if p not in touched], device=DEV)
    for x, y in zip(before, (cache.memory.k_pages.view(torch.uint8), cache.memory.v_pages.view(torch.uint8), cache.memory.k_scales, cache.memory.v_scales)):
        assert torch.equal(x[others], y[others])
    for s, (cached, n) in enumerate(lengths):
        pid, used = int(cache.table[s, (cached + n - 1) // page]), (cached + n - 1) % page + 1
        assert torch.equal(before[0][pid][:, used:], cache.memory.k_pages.view(torch.uint8)[pid][:, used:])
        old_v, new_v = (x[pid].transpose(2, 3).reshape(kv, page, size) for x in (before[1], cache.memory.v_pages.view(torch.uint8)))
        assert torch.equal(old_v[:, used:], new_v[:, used:])


@pytest.mark.parametrize("size,option", [(64, "plain"), (128, "plain"), (256, "plain"), (128, "values turned"), (128, "norm a token"), (64, "norm a head"),
                                         (128, "every pair in doubt"), (64, "half turned")])
def test_codes_are_the_nearest_in_64_bits(ops, size, option):
    """Four million turned numbers, of a prompt and of single tokens: each has the code of its 64-bit value.  (Float32 alone puts
    one in a million next to a border on the wrong side.)"""
    page, kv, t = 64, 8, 4096 * 128 // size
    g = torch.Generator().manual_seed(size)
    cache = Cache(ops, 64, -(-t // page), kv, page, size)
    k, v = ((torch.randn(t, kv * size, generator=g)).to(torch.bfloat16).to(DEV) for _ in range(2))
    freqs = (10000.0 ** (-torch.arange(size // 2) / (size // 2))).float().to(DEV)
    rstd = weights = None
    if option == "every pair in doubt":
        # numbers that lie between two codes before they are turned by next to nothing
        freqs.fill_(2.0 ** -40)
        k = ((torch.randint(8, 16, k.shape, generator=g) + 0.5) * 2.0).to(torch.bfloat16).to(DEV)
    elif option == "half turned":
        freqs[size // 4 :] = 0
    if option == "norm a token":
        rstd, weights = torch.rand(t, 2, generator=g).to(DEV) + 0.5, torch.rand(kv * size, generator=g).to(DEV) + 0.5
    elif option == "norm a head":
        rstd, weights = torch.rand(t, 2 * kv, generator=g).to(DEV) + 0.5, torch.rand(kv * size, generator=g).to(DEV) + 0.5
    options = dict(v_freqs=freqs if option == "values turned" else None, qk_norm=None if rstd is None else (rstd, weights, weights))
    q = torch.zeros(t, kv * size, dtype=torch.bfloat16, device=DEV)
    singles = torch.arange(60, dtype=torch.int32, device=DEV)
    for pos, req in ((torch.arange(t, dtype=torch.int32, device=DEV), torch.full((t,), 63, dtype=torch.int32, device=DEV)), (singles % 30 * page, singles)):
        n = pos.numel()
        wide = dict(options, qk_norm=None if rstd is None else (rstd[:n].contiguous(), weights, weights))
        ops.rope_kv8_write(q[:n], k[:n], v[:n], pos, req, freqs, cache.memory, kv, kv, size, **wide)
        x = k[:n].double().view(n, kv, size)
        if rstd is not None:
            x = x * (rstd[:n, 1:2] if rstd.shape[1] == 2 else rstd[:n, kv:]).double()[:, :, None] * weights.double().view(kv, size)
        x, y = _turned(x, pos, freqs), v[:n].double().view(n, kv, size)
        if option == "values turned":
            y = _turned(y, pos, freqs)
        at = cache.table[req.long(), (pos // page).long()].long()
        mem = cache.memory
        kc = cache.values[mem.k_pages.view(torch.uint8)[at, :, (pos % page).long()].long()]
        vc = cache.values[mem.v_pages.view(torch.uint8)[at, :, (pos % page // 4).long(), :, (pos % 4).long()].long()]
        assert torch.equal(kc, _nearest(x / mem.k_scales[at].double()[..., None]))
        assert torch.equal(vc, _nearest(y / mem.v_scales[at].double()[..., None]))
    ops.check_status()


@pytest.mark.parametrize("size", [64, 128])
def test_write_of_unusual_numbers(ops, size):
    """Zeros, the ends of bfloat16's range, infinities and NaN: the others of the page keep their scale and their codes."""
    page, kv = 16, 2
    cache = Cache(ops, 6, 1, kv, page, size)
    x = torch.randn(16, kv * size, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    zero = torch.zeros_like(x)
    cache.write(zero, zero, 0, 0)
    assert bool((cache.entries(0, 16)[0] == 0).all()) and bool((cache.memory.k_scales[int(cache.table[0, 0])] == 2.0 ** -100).all())
    cache.write(zero[:3], zero[:3], 1, 0)
    cache.write(x[:2], x[:2], 1, 3)  # a page of zeros grows
    k, v = cache.entries(1, 5)
    assert bool((k[:, :3] == 0).all()) and bool((v[:, :3] == 0).all())
    unit = cache.memory.v_scales[int(cache.table[1, 0])].double()[:, None, None]
    want = x[:2].double().view(2, kv, size).transpose(0, 1)
    assert torch.equal(v[:, 3:], _nearest(want / unit) * unit)
    poison = x.clone()
    poison[4, 3], poison[5, size + 1], poison[6, 0] = float("inf"), float("nan"), -float("inf")
    cache.write(poison, poison, 2, 0)
    got = cache.entries(2, 16)[1]
    bad = ~torch.isfinite(poison.view(16, kv, size).transpose(0, 1))
    assert torch.equal(torch.isnan(got), bad)
    unit = torch.exp2(_exponent(poison.double().nan_to_num(0.0, 0.0, 0.0).abs().view(16, kv, size).amax((0, 2))).double())[:, None, None]
    want = _nearest(poison.double().view(16, kv, size).transpose(0, 1) / unit) * unit
    assert torch.equal(got[~bad], want[~bad])
    big = x * 2.0 ** 120
    cache.write(big, big, 3, 0)
    got = cache.entries(3, 16)[1]
    want = big.double().view(16, kv, size).transpose(0, 1)
    assert bool((got.abs() <= 448 * 2.0 ** 100).all()) and bool((got.sign()[want.abs() > 2.0 ** 100] == want.sign()[want.abs() > 2.0 ** 100]).all())
    ops.check_status()


def test_write_twice_and_values(ops):
    """The same step once more changes nothing; the values read back are the entries, in pages asked for twice, too."""
    page, kv, size = 32, 3, 128
    cache = Cache(ops, 2, 4, kv, page, size)
    cache.fill(0, 90, 5, spread=3.0)
    g = torch.Generator().manual_seed(9)
    k, v = ((torch.randn(9, kv * size, generator=g) * 40).to(torch.bfloat16).to(DEV) for _ in range(2))
    cache.write(k, v, 0, 90)
    state = [x.clone() for x in (cache.memory.k_pages.view(torch.uint8), cache.memory.v_pages.view(torch.uint8), cache.memory.k_scales, cache.memory.v_scales)]
    cache.write(k, v, 0, 90)
    for x, y in zip(state, (cache.memory.k_pages.view(torch.uint8), cache.memory.v_pages.view(torch.uint8), cache.memory.k_scales, cache.memory.v_scales)):
        assert torch.equal(x, y)
    pages = cache.table[0, [2, 0, 2]].contiguous()
    keys, values = ops.kv8_values(cache.memory, pages)
    k64, v64 = cache.entries(0, 96)
    for i, lp in enumerate((2, 0, 2)):
        for got, want in ((keys, k64), (values, v64)):
            assert torch.equal(got[i].double(), want[:, lp * page : (lp + 1) * page])
    ops.kv8_values(cache.memory, torch.tensor([-1, 10 ** 6], dtype=torch.int32, device=DEV))
    from fastgen_b200.csrc.ops import KernelError
    with pytest.raises(KernelError, match="block-table entry"):
        ops.check_status()


# -- attention -------------------------------------------------------------------------------------


def _attention(cache, q, ctx, heads, scale, window=0, chunk=0, softcap=0.0, sinks=None):
    """The formula in 64 bits, and what a row's outputs may be off by."""
    kv, size = cache.kv, cache.size
    want = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    room = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for s, slot in enumerate(ctx.host_seq_slot):
        a, b, cached = ctx.host_seq_start[s], ctx.host_seq_start[s + 1], ctx.host_seq_cached[s]
        k, v = cache.entries(slot, cached + b - a)
        i = torch.arange(cached, cached + b - a, device=DEV)[:, None]
        j = torch.arange(cached + b - a, device=DEV)[None, :]
        hidden = j > i
        if window:
            hidden = hidden | (j <= i - window)
        if chunk:
            hidden = hidden | (j // chunk != i // chunk)
        for h in range(heads):
            g = h // (heads // kv)
            z = q[a:b, h * size : (h + 1) * size].double() @ k[g].T * scale
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            z = z.masked_fill(hidden, -float("inf"))
            if sinks is not None:
                z = torch.cat([z, sinks[h].double().expand(b - a, 1)], 1)
            p = torch.softmax(z, 1)[:, : cached + b - a]
            # (an entry of a key that is not seen may be a NaN)
            seen = torch.where(p.amax(0)[:, None] > 0, v[g], torch.zeros_like(v[g]))
            want[a:b, h * size : (h + 1) * size] = p @ seen
            room[a:b, h * size : (h + 1) * size] = p @ seen.abs()
    return want, room


def _check(got, want, room):
    assert bool(torch.isfinite(got).all())
    worst = float(((got.double() - want).abs() / (room + 1e-30)).max())
    assert bool(((got.double() - want).abs() <= 2.0 ** -7 * room + 1e-30).all()), worst


@pytest.mark.parametrize("size,page,heads,kv", [
    (64, 16, 4, 4), (64, 64, 8, 1), (64, 32, 28, 4), (128, 64, 32, 8), (128, 16, 3, 1), (128, 128, 16, 1), (128, 256, 20, 2), (256, 64, 7, 1),
    (256, 32, 16, 2)])
@pytest.mark.parametrize("option", ["plain", "window", "chunk", "cap", "sinks"])
def test_single_tokens(ops, size, page, heads, kv, option):
    """Requests of all lengths from one token on, over tile and page edges, more heads a group than an instruction's columns."""
    lengths = [1, 2, 15, 16, 17, 127, 128, 129, 300, 255, 257, 700, 1]
    cache = Cache(ops, len(lengths), -(-700 // page), kv, page, size, layers=2, layer=1)
    for s, n in enumerate(lengths):
        cache.fill(s, n, 3 * s + size, spread=2.0 ** (s % 5 - 2))
    g = torch.Generator().manual_seed(heads)
    q = (torch.randn(len(lengths), heads * size, generator=g) * 2).to(torch.bfloat16).to(DEV)
    ctx = _context([n - 1 for n in lengths], [1] * len(lengths))
    args = dict(window=dict(window=100), chunk=dict(chunk=48), cap=dict(softcap=5.0), sinks=dict(sinks=torch.randn(heads, generator=g).to(DEV)),
                plain={})[option]
    out = torch.empty_like(q)
    call = dict(args)
    window = call.pop("window", None)
    turned = ops.attention(q, out, cache.memory, ctx, heads, kv, size, window, size ** -0.5, **call)
    ops.check_status()
    assert turned is False
    _check(out, *_attention(cache, q, ctx, heads, size ** -0.5, **args))
    again = torch.empty_like(q)
    for _ in range(3):
        ops.attention(q, again, cache.memory, ctx, heads, kv, size, window, size ** -0.5, **call)
        assert torch.equal(out, again)


@pytest.mark.parametrize("requests,length", [(1, 9000), (3, 5000), (70, 150), (600, 20), (150, 1000)])
def test_single_tokens_of_many_and_long_requests(ops, requests, length):
    """Runs that many blocks share, blocks that hold many runs, more requests than blocks."""
    size, page, heads, kv = 64, 64, 8, 2
    g = torch.Generator().manual_seed(requests)
    lengths = [max(1, int(length * float(x))) for x in torch.rand(requests, generator=g)]
    lengths[0] = length
    cache = Cache(ops, requests, -(-length // page), kv, page, size)
    x = torch.randn(length, kv * size, generator=g).to(torch.bfloat16).to(DEV)
    for s, n in enumerate(lengths):
        cache.write(x[:n] * (1 + s % 3), x[-n:], s, 0)
    q = torch.randn(requests, heads * size, generator=g).to(torch.bfloat16).to(DEV)
    ctx = _context([n - 1 for n in lengths], [1] * requests)
    out = torch.empty_like(q)
    ops.attention(q, out, cache.memory, ctx, heads, kv, size, None, size ** -0.5)
    ops.check_status()
    _check(out, *_attention(cache, q, ctx, heads, size ** -0.5))


def test_single_tokens_with_scales_far_apart(ops):
    """Pages whose scales lie 2^200 apart, weights that are tiny beside the first key's, queries at the ends of their range."""
    size, page, kv, n = 128, 16, 1, 200
    cache = Cache(ops, 4, 13, kv, page, size)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(n, size, generator=g) for _ in range(2))
    up = torch.exp2(torch.randint(-95, 95, (13,), generator=g).float()).repeat_interleave(page)[:n, None]
    cache.write(k.to(torch.bfloat16).to(DEV), (v * up).to(torch.bfloat16).to(DEV), 0, 0)
    cache.write((k * 2.0 ** -60).to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV), 1, 0)
    # a first key that takes nearly all weight and whose value is zero
    v[0] = 0
    k[0] = 60.0
    cache.write(k.to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV), 2, 0)
    cache.write(k.to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV), 3, 0)
    q = torch.randn(4, size, generator=g)
    q[1] *= 2.0 ** 62
    q[2] = 0.03
    q[3] *= 2.0 ** -60
    q[3, 5] = 0.25
    q = q.to(torch.bfloat16).to(DEV)
    ctx = _context([n - 1] * 4, [1] * 4)
    out = torch.empty_like(q)
    ops.attention(q, out, cache.memory, ctx, 1, kv, size, None, size ** -0.5)
    ops.check_status()
    _check(out, *_attention(cache, q, ctx, 1, size ** -0.5))


def test_single_tokens_beside_padding_and_poison(ops):
    """Padding lanes write nothing; a NaN among a request's entries or queries stays with that request; entries of a page's
    former owner, NaN codes too, are nobody's."""
    size, page, heads, kv = 128, 64, 8, 2
    cache = Cache(ops, 5, 4, kv, page, size)
    for s in range(5):
        cache.fill(s, 130 + s, s)
    x = torch.zeros(1, kv * size, dtype=torch.bfloat16, device=DEV)
    x[0, 5] = float("nan")
    cache.write(x, x * 0 + 1, 1, 131)
    q = torch.randn(7, heads * size, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    q[3, 2] = float("inf")
    ctx = _context([129, 131, 131, 132, 133], [1] * 5)
    from fastgen_b200.engine.step import SingleTokens
    lanes = SingleTokens(torch.tensor([0, -1, 1, 2, 3, -1, 4], dtype=torch.int32, device=DEV),
                         torch.tensor([0, 6, 1, 2, 3, 6, 4], dtype=torch.int32, device=DEV), 7, 256, None, 5 * 256)
    ctx.single_tokens = lambda: lanes
    out = torch.full_like(q, 7.0)
    ops.attention(q, out, cache.memory, ctx, heads, kv, size, None, size ** -0.5)
    ops.check_status()
    assert bool((out[5:] == 7.0).all())
    want, room = _attention(cache, q, ctx, heads, size ** -0.5)
    for row in (0, 2, 4):
        _check(out[row], want[row], room[row])
    assert bool(torch.isnan(out[1][: heads // kv * size]).all())  # the poisoned key's head
    _check(out[1][heads // kv * size :], want[1][heads // kv * size :], room[1][heads // kv * size :])
    assert bool(torch.isnan(out[3][:size]).all()) and bool(torch.isfinite(out[3][size:]).all())


def test_outputs_turned_back(ops):
    """Single tokens alone: the kernel turns outputs by position * frequency; beside prompts the caller does."""
    size, page, heads, kv = 64, 64, 4, 2
    cache = Cache(ops, 3, 12, kv, page, size)
    lengths = [3, 200, 640]
    for s, n in enumerate(lengths):
        cache.fill(s, n, s)
    q = torch.randn(3, heads * size, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(DEV)
    freqs = -(10000.0 ** (-torch.arange(size // 2).double() * 2 / size)).float().to(DEV)
    ctx = _context([n - 1 for n in lengths], [1] * 3)
    out = torch.empty_like(q)
    assert ops.attention(q, out, cache.memory, ctx, heads, kv, size, None, size ** -0.5, out_freqs=freqs) is True
    want, room = _attention(cache, q, ctx, heads, size ** -0.5)
    want = _turned(want.view(3, heads, size), ctx.pos, freqs).flatten(1)
    pair = room.view(3, -1, 2).sum(2, keepdim=True).expand(-1, -1, 2).reshape(3, -1)
    _check(out, want, pair)


@pytest.mark.parametrize("size,page,heads,kv", [(64, 16, 4, 2), (64, 64, 7, 1), (128, 64, 32, 8), (128, 128, 6, 2), (256, 32, 4, 1)])
@pytest.mark.parametrize("option", ["plain", "window", "chunk", "cap", "sinks"])
def test_prompt_portions(ops, size, page, heads, kv, option):
    """Portions of prompts behind cached tokens beside single tokens, in one step."""
    cached, new = [0, 130, 7, 299, 40, 0], [200, 1, 65, 2, 1, 1]
    cache = Cache(ops, len(new), -(-301 // page) + 1, kv, page, size)
    for s, (c, n) in enumerate(zip(cached, new)):
        cache.fill(s, c + n, s + size)
    g = torch.Generator().manual_seed(page)
    q = torch.randn(sum(new), heads * size, generator=g).to(torch.bfloat16).to(DEV)
    ctx = _context(cached, new)
    args = dict(window=dict(window=50), chunk=dict(chunk=64), cap=dict(softcap=4.0), sinks=dict(sinks=torch.randn(heads, generator=g).to(DEV)),
                plain={})[option]
    call = dict(args)
    window = call.pop("window", None)
    out = torch.full_like(q, float("nan"))
    ops.attention(q, out, cache.memory, ctx, heads, kv, size, window, size ** -0.5, **call)
    ops.check_status()
    want, room = _attention(cache, q, ctx, heads, size ** -0.5, **args)
    # (prompts run on the 16-bit kernels, whose weights are rounded to bfloat16: 2^-8 of each and of the result)
    _check(out, want, 2 * room)


@pytest.mark.parametrize("size,page", [(64, 16), (64, 64), (128, 32), (128, 128), (128, 256), (256, 16)])
@pytest.mark.parametrize("option", ["plain", "window", "chunk"])
def test_pages_that_were_given_back(ops, size, page, option):
    """Pages that no later query sees are gone from the table and hold other sequences' NaNs, as does the pool that portions read."""
    kv, heads = 2, 4
    cached, new = [0, 700, 300, 513, 640], [150, 40, 1, 2, 1]
    cache = Cache(ops, len(new), -(-760 // page) + 1, kv, page, size)
    for s, (c, n) in enumerate(zip(cached, new)):
        cache.fill(s, c + n, s + size)
    args = dict(window=dict(window=100), chunk=dict(chunk=192), plain={})[option]
    ctx = _context(cached, new)
    g = torch.Generator().manual_seed(page)
    q = torch.randn(sum(new), heads * size, generator=g).to(torch.bfloat16).to(DEV)
    want, room = _attention(cache, q, ctx, heads, size ** -0.5, **args)
    for s, c in enumerate(cached):
        first = max(0, c + 1 - 100) if option == "window" else c // 192 * 192 if option == "chunk" else 0
        for logical in range(first // page):
            at = int(cache.table[s, logical])
            for pool in (cache.memory.k_pages, cache.memory.v_pages):
                pool.view(torch.uint8)[at] = 0x7F
            cache.table[s, logical] = -1
    for pool in ops.kv8_expanded(cache.memory)[:2]:
        pool.fill_(float("nan"))
    out = torch.empty_like(q)
    call = dict(args)
    window = call.pop("window", None)
    ops.attention(q, out, cache.memory, ctx, heads, kv, size, window, size ** -0.5, **call)
    ops.check_status()
    _check(out, want, 2 * room)


def test_the_first_call_is_not_captured(ops):
    """Work buffers are made outside a capture; what needs them inside one is refused, and served after a first call."""
    from fastgen_b200.csrc.ops import Ops
    size, page, heads, kv = 64, 32, 4, 2
    cache = Cache(ops, 2, 8, kv, page, size)
    for s in range(2):
        cache.fill(s, 200, s)
    fresh = Ops(torch.bfloat16, DEV)
    for ctx in (_context([199], [1]), _context([150], [50])):
        q = torch.randn(ctx.n_tokens, heads * size, device=DEV).to(torch.bfloat16)
        out, want = torch.zeros_like(q), torch.zeros_like(q)
        ops.attention(q, want, cache.memory, ctx, heads, kv, size, None, 0.1)
        with pytest.raises(RuntimeError, match="graph capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                fresh.attention(q, out, cache.memory, ctx, heads, kv, size, None, 0.1)
        fresh.attention(q, out, cache.memory, ctx, heads, kv, size, None, 0.1)
        assert torch.equal(out, want)


def test_attention_on_two_streams_and_in_graphs(ops):
    """A call on another stream is ordered behind the first; a captured call gives the eager one's bits, for other lengths than
    it was captured with, too."""
    from fastgen_b200.engine.step import SingleTokens
    size, page, heads, kv = 128, 64, 8, 2
    cache = Cache(ops, 4, 20, kv, page, size)
    for s in range(4):
        cache.fill(s, 1200, s)
    q = torch.randn(4, heads * size, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)

    def context(lengths):
        ctx = _context([n - 1 for n in lengths], [1] * 4)
        lanes = SingleTokens(ctx.req, torch.arange(4, dtype=torch.int32, device=DEV), 4, 1280, None, 4 * 1280)
        ctx.single_tokens = lambda: lanes
        return ctx

    first, second = context([1200, 3, 700, 129]), context([5, 1100, 128, 1000])
    want = []
    for ctx in (first, second):
        out = torch.empty_like(q)
        ops.attention(q, out, cache.memory, ctx, heads, kv, size, None, 0.1)
        want.append(out)
    side = torch.cuda.Stream()
    outs = [torch.empty_like(q) for _ in range(8)]
    side.wait_stream(torch.cuda.current_stream())
    for i, out in enumerate(outs):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            ops.attention(q, out, cache.memory, (first, second)[i % 2], heads, kv, size, None, 0.1)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, want[i % 2])
    out = torch.empty_like(q)
    pos = first.pos.clone()
    first.pos = pos
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention(q, out, cache.memory, first, heads, kv, size, None, 0.1)
    for ctx, expect in ((second, want[1]), (context([1200, 3, 700, 129]), want[0])):
        pos.copy_(ctx.pos)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expect)
    ops.check_status()


def test_attention_right_behind_the_write_of_a_prompt(ops):
    """A single token that reads what the launch before it wrote, all of it: the same with and without a pause between."""
    size, page, heads, kv, n = 128, 64, 8, 8, 8000
    cache = Cache(ops, 1, -(-n // page), kv, page, size)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(1, heads * size, generator=g).to(torch.bfloat16).to(DEV)
    ctx, out, want = _context([n - 1], [1]), torch.empty_like(q), torch.empty_like(q)
    for _ in range(6):
        k, v = ((torch.randn(n, kv * size, generator=g)).to(torch.bfloat16).to(DEV) for _ in range(2))
        torch.cuda.synchronize()
        cache.write(k, v, 0, 0)
        ops.attention(q, out, cache.memory, ctx, heads, kv, size, None, 0.1)
        torch.cuda.synchronize()
        ops.attention(q, want, cache.memory, ctx, heads, kv, size, None, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    ops.check_status()


def test_bad_pages_are_reported(ops):
    from fastgen_b200.csrc.ops import KernelError
    size, page, heads, kv = 64, 64, 2, 1
    cache = Cache(ops, 2, 4, kv, page, size)
    for s in range(2):
        cache.fill(s, 200, s)
    cache.table[0, 1] = -1
    q = torch.randn(2, heads * size).to(torch.bfloat16).to(DEV)
    ctx = _context([199, 199], [1, 1])
    out = torch.empty_like(q)
    ops.attention(q, out, cache.memory, ctx, heads, kv, size, None, 0.1)
    with pytest.raises(KernelError, match="block-table entry"):
        ops.check_status()
    want, room = _attention(cache, q[1:], _context([199], [1], [1]), heads, 0.1)
    _check(out[1:], want, room)
    x = torch.zeros(3, kv * size, dtype=torch.bfloat16, device=DEV)
    before = cache.memory.k_pages.view(torch.uint8).clone()
    for start in (70, -5, -500):  # a page that is not there, positions that are none
        cache.write(x, x, 0, start)
        with pytest.raises(KernelError, match="block-table entry"):
            ops.check_status()
    assert torch.equal(before, cache.memory.k_pages.view(torch.uint8))


def test_refusals(ops):
    """What the calls do not take, they refuse before anything is launched."""
    from dataclasses import replace
    from fastgen_b200.csrc.ops import KernelError, Ops
    cache = Cache(ops, 1, 2, 2, 64, 64)
    mem = cache.memory
    q = torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(1, 2 * 64, dtype=torch.bfloat16, device=DEV)
    at = torch.zeros(1, dtype=torch.int32, device=DEV)
    ctx = _context([0], [1])
    with pytest.raises(ValueError, match="bfloat16 rows"):
        ops.rope_kv8_write(q.float(), k, k, at, at, None, mem, 4, 2, 64)
    with pytest.raises(ValueError, match="bfloat16 rows"):
        ops.rope_kv8_write(q, k, k[:, :64], at, at, None, mem, 4, 2, 64)
    with pytest.raises(ValueError, match="wanted, got"):
        ops.rope_kv8_write(q, k, k, at, at, None, replace(mem, k_scales=mem.k_scales[:1]), 4, 2, 64)
    with pytest.raises(ValueError, match="wanted, got"):
        ops.attention(q, q.clone(), replace(mem, v_pages=mem.k_pages), ctx, 4, 2, 64, None, 1.0)
    for field in ("k_pages", "v_pages", "k_scales", "v_scales", "block_table"):
        with pytest.raises(ValueError, match="on one GPU"):
            ops.attention(q, q.clone(), replace(mem, **{field: getattr(mem, field).cpu()}), ctx, 4, 2, 64, None, 1.0)
    with pytest.raises(ValueError, match="bfloat16 rows"):
        ops.rope_kv8_write(q.cpu(), k, k, at, at, None, mem, 4, 2, 64)
    with pytest.raises(AssertionError):
        ops.attention(q[:, :128], q.clone(), mem, ctx, 4, 2, 64, None, 1.0)
    with pytest.raises(ValueError, match="keeps first positions"):
        ops.attention(q, q.clone(), mem, ctx, 4, 2, 64, 10, 1.0, keep_first=4)
    with pytest.raises(ValueError, match="serves bfloat16"):
        Ops(torch.float32, DEV).attention(q, q.clone(), mem, ctx, 4, 2, 64, None, 1.0)
    with pytest.raises(ValueError, match="pages of 24 tokens"):
        ops.make_kv8_tensor_maps(torch.zeros(1, 2, 2, 24, 64, device=DEV).to(torch.float8_e4m3fn), None)
    with pytest.raises(KernelError, match="row strides"):
        wide = torch.zeros(1, 4 * 64 + 4, dtype=torch.bfloat16, device=DEV)
        ops.attention(wide[:, : 4 * 64].expand(1, -1), q.clone(), mem, SimpleNamespace(
            single_tokens=ctx.single_tokens, longest=1, pos=ctx.pos, attention_tiles=ctx.attention_tiles), 4, 2, 64, None, 1.0)
