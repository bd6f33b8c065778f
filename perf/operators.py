"""Operators for serving in fewer bits: a paged cache held in 8 bits, and products with 4-bit weights.

Four operators, one pass through one of them a case:

* ``write``: queries and keys of a step's tokens are rotated, keys and values are written to their pages in 8 bits
  (e4m3 codes with one power of two for each page and key/value head); what the pages that the step touched then stand
  for is read back.
* ``single``: attention of a batch of decoded tokens over such a cache.
* ``prompt``: attention of prompt portions over such a cache.
* ``product``: ``x @ w.T`` with weights of 4 bits and a scale for each group of columns of a row.

Definitions that the plain form, ``exact`` and the kernels share:

* a page of one head holds codes ``c`` and a scale ``2^e`` with the smallest whole ``e >= -100`` at which every entry's
  magnitude is at most ``448 * 2^e`` (448 is e4m3's largest number); its entries are ``c * 2^e``, ``c`` being the entry
  over the scale rounded to the nearest e4m3 number, ties to even.  A write that starts at a page's first slot chooses
  ``e`` from the step's own tokens; one that goes on behind cached entries never lowers ``e``, and where it raises it
  the cached codes are rounded again at the new scale.
* keys are ``[page, head, slot, size]``; values ``[page, head, slot / 4, size, 4]``: the codes of four tokens side by side.
* the rotation's angle is the float32 product of position and frequency, as everywhere in this package.
* a 4-bit code ``n`` (0..15) stands for ``(n - 8) * scale``; two codes a byte, the even column in the low half.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
ROPE_BASE = 500000.0
LARGEST = 448.0
LOWEST_EXPONENT = -100


# -- the cases -----------------------------------------------------------------------------------


def _cache(op, name=None, **sizes):
    case = dict(op=op, head_dim=128, heads=32, kv_heads=8, page=64, singles=0, prompts=0, tokens=0, context=0,
                ragged=False, window=0, softcap=0.0, sinks=False)
    case.update(sizes)
    return dict(name=name, **case) if name is not None else case


def _product(name=None, **sizes):
    case = dict(op="product", m=1, n=4096, k=4096, group=128, bias=False)
    case.update(sizes)
    return dict(name=name, **case) if name is not None else case


def listed():
    return [
        # one request being decoded, the smallest call there is
        _cache("write", "write b1", head_dim=64, singles=1, context=300),
        # a batch of decoded tokens, requests of all lengths
        _cache("write", "write b64 ragged", singles=64, context=1400, ragged=True),
        # a step of continuous batching: a prompt beside running requests
        _cache("write", "write 2048+20", singles=20, prompts=1, tokens=2048, context=900, ragged=True),
        # one chat request: a short context, where latency counts
        _cache("single", "single b1 ctx300", head_dim=64, singles=1, context=300),
        # the benchmark's decode: batch 8 at a context of 4,096
        _cache("single", "single b8 ctx4096", singles=8, context=4096),
        # a full batch of requests of all lengths
        _cache("single", "single b64 ragged", singles=64, context=2800, ragged=True),
        # two readers of long documents on a model with small heads
        _cache("single", "single b2 ctx30000", head_dim=64, singles=2, context=30000),
        # the benchmark's prompt
        _cache("prompt", "prompt 2048", prompts=1, tokens=2048),
        # the last portion of a long document
        _cache("prompt", "portion 512 on 16384", prompts=1, tokens=512, context=16384),
        # the fused query, key and value projection for one token
        _product("product m1 6144x4096", n=6144),
        # gate and up projection for a small batch
        _product("product m8 28672x4096", m=8, n=28672),
        # the down projection for a full batch
        _product("product m64 4096x14336", m=64, k=14336),
    ]


def _log(rng, lo, hi):
    """A whole number from ``lo`` to ``hi``, spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case of any operator, at sizes up to those of the list."""
    op = rng.choice(["write", "single", "single", "prompt", "product", "product"])
    if op == "product":
        group = rng.choice([32, 64, 128])
        k = group * _log(rng, 2, 14336 // group)
        n = _log(rng, 16, min(28672, 58_000_000 // k))
        return _product(m=_log(rng, 1, 64), n=n, k=k, group=group, bias=rng.random() < 0.3)
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([16, 32, 64, 64, 128])
    sizes = dict(head_dim=head_dim, kv_heads=kv_heads, heads=heads, page=page)
    wide = heads * head_dim
    if op == "write":
        return _cache(op, singles=_log(rng, 1, 64), prompts=rng.randint(0, 2), tokens=_log(rng, 2, min(1000, 4_000_000 // wide)),
                      context=_log(rng, 16, 1400), ragged=rng.random() < 0.7, **sizes)
    options = dict(window=rng.choice([0, 0, 0, 100, 1024]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                   sinks=rng.random() < 0.25)
    if op == "single":
        batch = _log(rng, 1, 64)
        keys = 90_000_000 // (kv_heads * head_dim)
        return _cache(op, singles=batch, context=_log(rng, 1, min(30000, keys // batch)), ragged=rng.random() < 0.6,
                      **options, **sizes)
    prompts = rng.randint(1, 3)
    tokens = _log(rng, 2, 1024 // prompts)
    context = min(16384, 30_000_000_000 // wide // (tokens * prompts) - tokens)
    return _cache(op, prompts=prompts, tokens=tokens, context=_log(rng, 1, context) - 1, ragged=rng.random() < 0.6,
                  **options, **sizes)


def _lengths(case):
    """(tokens cached before the step, tokens the step brings) of every sequence, prompts first."""
    out = []
    for i in range(case["prompts"]):
        share = 1.0 - 0.55 * i / case["prompts"] if case["ragged"] else 1.0
        out.append((int(case["context"] * share) if case["op"] == "prompt" else 0, max(2, int(case["tokens"] * share))))
    for i in range(case["singles"]):
        # a ragged batch: every length between a token or two and the longest
        share = (0.618 * (i + 1)) % 1.0 if case["ragged"] and i else 1.0
        out.append((int(case["context"] * share), 1))
    return out


def _first_visible(p, window):
    return max(0, p - window + 1) if window else 0


def work(case):
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + 2 * n * (k // case["group"]) + 2 * m * (n + k) + 2 * n * case["bias"],
                "flops": 2 * m * n * k}
    size, heads, kv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    lengths = _lengths(case)
    tokens = sum(new for _, new in lengths)
    if case["op"] == "write":
        touched = sum((c + new - 1) // page - c // page + 1 for c, new in lengths)
        # queries in and out, keys and values in, their codes out; the touched pages' entries, read back in 16 bits
        return {"bytes": 4 * tokens * heads * size + 6 * tokens * kv * size + 6 * touched * kv * page * size,
                "flops": tokens * (heads + kv) * size * 3}
    # every key and value that some query of its sequence sees once, a byte each, and queries and outputs
    keys = sum(c + new - _first_visible(c, case["window"]) for c, new in lengths)
    pairs = sum(p + 1 - _first_visible(p, case["window"]) for c, new in lengths for p in range(c, c + new))
    return {"bytes": 2 * keys * kv * size + 4 * tokens * heads * size, "flops": 4 * pairs * heads * size}


# -- inputs --------------------------------------------------------------------------------------


def _exponent(amax):
    """The smallest whole e >= LOWEST_EXPONENT with amax <= 448 * 2^e, as float32."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    e = exponent.to(torch.float32) - 9.0 + (mantissa > 0.875).to(torch.float32)
    return torch.where(amax > 0, e, torch.full_like(e, LOWEST_EXPONENT)).clamp_min(LOWEST_EXPONENT)


def _round_codes(x):
    """x rounded to the nearest e4m3 number, as codes."""
    return x.to(torch.float32).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["op"] == "product":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        # activations behind a norm, a few channels larger than the rest; trained weights, a scale a group
        x = randn(m, k) * (1.0 + 4.0 * (torch.rand(k, generator=gen, device=DEV) < 0.01))
        codes = torch.empty(n, k // 2, dtype=torch.uint8, device=DEV)
        scales = torch.empty(n, k // group, dtype=torch.bfloat16, device=DEV)
        rows = max(1, 50_000_000 // k)
        for r in range(0, n, rows):
            w = randn(min(rows, n - r), k // group, group) * 0.02
            s = (w.abs().amax(-1) / 7.0).to(torch.bfloat16)
            c = (torch.round(w / s.float().unsqueeze(-1)).clamp(-8, 7) + 8).to(torch.uint8).view(w.shape[0], k)
            codes[r : r + rows] = c[:, 0::2] | (c[:, 1::2] << 4)
            scales[r : r + rows] = s
        state = dict(case=case, x=x.to(torch.bfloat16), codes=codes, scales=scales,
                     bias=randn(n).to(torch.bfloat16) if case["bias"] else None)
        if own:
            # the handles that a model keeps: the kernels' face and the layer's weight
            from fastgen_b200.csrc.ops import Ops
            from fastgen_b200.weights import Weight4

            state["ops"] = Ops(torch.bfloat16, DEV)
            state["weight"] = Weight4(codes, scales)
        return state

    size, heads, kv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    lengths = _lengths(case)
    n_seqs = len(lengths)
    width = max((c + new - 1) // page + 1 for c, new in lengths)
    counts = [(c + new - 1) // page + 1 for c, new in lengths]
    n_pages = sum(counts) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((n_seqs, width), -1, dtype=torch.int32, device=DEV)
    held = torch.zeros(n_pages, dtype=torch.int64, device=DEV)
    # a "write" finds what was cached before the step; attention what is cached behind the write
    at = 0
    for s, (cached, new) in enumerate(lengths):
        n = counts[s]
        table[s, :n] = order[at : at + n]
        tokens = cached if case["op"] == "write" else cached + new
        held[order[at : at + n].long()] = (tokens - torch.arange(n, device=DEV) * page).clamp(0, page)
        at += n
    pools = []
    for _ in range(2):
        # some channels of keys and values are several times larger than the rest, and heads differ
        spread = (1.0 + 5.0 * (torch.rand(kv, 1, size, generator=gen, device=DEV) < 0.03)) * (
            0.5 + torch.rand(kv, 1, 1, generator=gen, device=DEV))
        codes = torch.empty(n_pages, kv, page, size, dtype=torch.float8_e4m3fn, device=DEV)
        scales = torch.empty(n_pages, kv, device=DEV)
        some = max(1, 60_000_000 // (kv * page * size))
        for p in range(0, n_pages, some):
            x = randn(min(some, n_pages - p), kv, page, size) * spread
            x *= (torch.arange(page, device=DEV)[None, :] < held[p : p + some, None])[:, None, :, None]
            e = _exponent(x.abs().amax((2, 3)))
            codes[p : p + some] = _round_codes(x * torch.exp2(-e)[:, :, None, None])
            scales[p : p + some] = torch.exp2(e)
        pools.append((codes, scales, spread))
    (k_codes, k_scales, k_spread), (v_codes, v_scales, v_spread) = pools
    v_codes = v_codes.view(torch.uint8).view(n_pages, kv, page // 4, 4, size).transpose(3, 4).contiguous()
    tokens = sum(new for _, new in lengths)
    pos = torch.cat([torch.arange(c, c + new, device=DEV) for c, new in lengths]).to(torch.int32)
    req = torch.cat([torch.full((new,), s, device=DEV) for s, (_, new) in enumerate(lengths)]).to(torch.int32)
    state = dict(case=case, pos=pos, req=req, table=table, k_pages=k_codes, k_scales=k_scales,
                 v_pages=v_codes.view(torch.float8_e4m3fn), v_scales=v_scales, scale=size ** -0.5,
                 sinks=randn(heads) if case["sinks"] else None)
    state["q"] = randn(tokens, heads * size).to(torch.bfloat16)
    if case["op"] == "write":
        # now and then a token is larger than what its page has seen
        grow = 1.0 + 2.0 * (torch.rand(tokens, 1, 1, generator=gen, device=DEV) < 0.1)
        state["k"] = (randn(tokens, kv, size) * k_spread[:, 0] * grow).view(tokens, kv * size).to(torch.bfloat16)
        state["v"] = (randn(tokens, kv, size) * v_spread[:, 0] * grow).view(tokens, kv * size).to(torch.bfloat16)
        state["freqs"] = (ROPE_BASE ** (-torch.arange(size // 2, device=DEV, dtype=torch.float64) * 2 / size)).float()
        # the pages that the step touches, the slot of the first new token in each, and every token's page among them
        touched, first, of_token = [], [], []
        for s, (cached, new) in enumerate(lengths):
            base = len(touched)
            for lp in range(cached // page, (cached + new - 1) // page + 1):
                touched.append((s, lp))
                first.append(max(cached - lp * page, 0))
            of_token += [base + p // page - cached // page for p in range(cached, cached + new)]
        at = torch.tensor(touched, device=DEV)
        state["touched"] = table[at[:, 0], at[:, 1]].contiguous()
        state["first"] = torch.tensor(first, device=DEV)
        state["of_token"] = torch.tensor(of_token, device=DEV)
    else:
        # queries in rows of equal length for the plain form: token of (sequence, place), -1 where there is none
        longest = max(new for _, new in lengths)
        starts = torch.tensor([0] + [new for _, new in lengths], device=DEV).cumsum(0)[:-1]
        news = torch.tensor([new for _, new in lengths], device=DEV)
        place = torch.arange(longest, device=DEV)[None, :]
        state["token_at"] = torch.where(place < news[:, None], starts[:, None] + place, -1)
        state["out"] = torch.zeros(tokens, heads * size, dtype=torch.bfloat16, device=DEV)
    if own:
        # the handles that an engine keeps: the kernels' face, a layer's memory and the step's lists
        from fastgen_b200.cache import LayerMemory
        from fastgen_b200.csrc.ops import Ops
        from fastgen_b200.engine.step import StepContext

        ops = Ops(torch.bfloat16, DEV)
        state["ops"] = ops
        state["memory"] = LayerMemory(
            k_pages=state["k_pages"], v_pages=state["v_pages"], block_table=table, page_size=page,
            k_scales=k_scales, v_scales=v_scales,
            tensor_maps=ops.make_kv8_tensor_maps(state["k_pages"][None], state["v_pages"][None]), layer_index=0)
        ctx = StepContext(torch.device(DEV))
        ctx.pos, ctx.req, ctx.n_tokens, ctx.n_seqs = pos, req, tokens, n_seqs
        ctx.host_seq_slot = list(range(n_seqs))
        ctx.host_seq_cached = [c for c, _ in lengths]
        for _, new in lengths:
            ctx.host_seq_start.append(ctx.host_seq_start[-1] + new)
        ctx.longest = max(new for _, new in lengths)
        sequences = ctx.host_seq_slot, ctx.host_seq_start, ctx.host_seq_cached
        ctx.seq_slot, ctx.seq_start, ctx.seq_cached = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in sequences)
        state["ctx"] = ctx
    return state


# -- the operators -------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        ops = state["ops"]
        if case["op"] == "product":
            return ops.linear(state["x"], state["weight"], bias=state["bias"])
        size, heads, kv = case["head_dim"], case["heads"], case["kv_heads"]
        if case["op"] == "write":
            q = ops.rope_kv8_write(state["q"], state["k"], state["v"], state["pos"], state["req"], state["freqs"],
                                   state["memory"], heads, kv, size)
            keys, values = ops.kv8_values(state["memory"], state["touched"])
            return {"q": q, "keys": keys, "values": values}
        ops.attention(state["q"], state["out"], state["memory"], state["ctx"], heads, kv, size, case["window"] or None,
                      state["scale"], softcap=case["softcap"] or None, sinks=state["sinks"])
        return state["out"]
    if case["op"] == "product":
        return _plain_product(state)
    if case["op"] == "write":
        return _plain_write(state)
    return _plain_attention(state)


def _plain_product(state):
    codes, scales = state["codes"], state["scales"]
    n, half = codes.shape
    w = torch.stack([codes & 15, codes >> 4], dim=2).to(torch.float32) - 8.0
    w = (w.view(n, scales.shape[1], -1) * scales.float().unsqueeze(2)).view(n, 2 * half)
    y = state["x"].float() @ w.T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(torch.bfloat16)


def _turn(x, pos, freqs):
    """Adjacent pairs of x [T, heads, size] (64 bits) turned by the float32 angle position * frequency."""
    angle = (pos.to(torch.float32)[:, None] * freqs[None, :]).to(torch.float64)
    cos, sin = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], dim=3).flatten(2)


def _plain_write(state):
    case = state["case"]
    size, kv, page = case["head_dim"], case["kv_heads"], case["page"]
    pos, touched, first, of_token = state["pos"], state["touched"].long(), state["first"], state["of_token"]
    tokens = pos.numel()
    # a key's entries lie next to borders of the 8-bit numbers: 64 bits until they are rounded
    q = _turn(state["q"].double().view(tokens, -1, size), pos, state["freqs"]).flatten(1).to(torch.bfloat16)
    keys = _turn(state["k"].double().view(tokens, kv, size), pos, state["freqs"])
    out = {"q": q}
    for name, new in (("keys", keys), ("values", state["v"].double().view(tokens, kv, size))):
        if name == "keys":
            codes = state["k_pages"].view(torch.uint8)[touched].view(torch.float8_e4m3fn).to(torch.float32)
            scales = state["k_scales"][touched]
        else:
            codes = state["v_pages"].view(torch.uint8)[touched].view(torch.float8_e4m3fn).to(torch.float32)
            codes, scales = codes.transpose(3, 4).reshape(-1, kv, page, size), state["v_scales"][touched]
        amax = torch.zeros(touched.numel(), kv, dtype=torch.float64, device=DEV)
        amax.index_reduce_(0, of_token, new.abs().amax(2), "amax")
        e = _exponent(amax)
        old = torch.log2(scales)
        e = torch.where(first[:, None] > 0, torch.maximum(e, old), e)
        again = _round_codes(codes * torch.exp2(old - e)[:, :, None, None]).to(torch.float32)
        cached = torch.arange(page, device=DEV)[None, :] < first[:, None]
        codes = torch.where(cached[:, None, :, None], again, codes)
        fresh = _round_codes(new * torch.exp2(-e.double())[of_token][:, :, None]).to(torch.float32)
        codes[of_token, :, (pos % page).long()] = fresh
        out[name] = (codes * torch.exp2(e)[:, :, None, None]).to(torch.bfloat16)
    return out


def _plain_attention(state):
    case = state["case"]
    size, heads, kv, page, window = case["head_dim"], case["heads"], case["kv_heads"], case["page"], case["window"]
    token_at, table = state["token_at"], state["table"].clamp_min(0).long()
    n_seqs, longest = token_at.shape
    length = table.shape[1] * page
    k = state["k_pages"].view(torch.uint8)[table].view(torch.float8_e4m3fn).to(torch.float32)
    k = (k * state["k_scales"][table][..., None, None]).transpose(1, 2).reshape(n_seqs, kv, length, size)
    v = state["v_pages"].view(torch.uint8)[table].view(torch.float8_e4m3fn).to(torch.float32)
    v = v.transpose(4, 5).reshape(n_seqs, -1, kv, page, size) * state["v_scales"][table][..., None, None]
    v = v.transpose(1, 2).reshape(n_seqs, kv, length, size)
    q = state["q"].float().view(-1, kv, heads // kv, size)[token_at.clamp_min(0)]  # [sequence, place, kv, group, size]
    q = q.permute(0, 2, 3, 1, 4).reshape(n_seqs, kv, -1, size)
    s = (q @ k.transpose(2, 3)).view(n_seqs, kv, -1, longest, length) * state["scale"]
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    p = torch.where(token_at >= 0, state["pos"].long()[token_at.clamp_min(0)], 0)  # [sequence, place]
    j = torch.arange(length, device=DEV)
    seen = j[None, None, :] <= p[..., None]
    if window:
        seen = seen & (j[None, None, :] > p[..., None] - window)
    s = torch.where(seen[:, None, None], s, -math.inf)
    top = s.amax(4, keepdim=True)
    if state["sinks"] is not None:
        sinks = state["sinks"].view(1, kv, -1, 1, 1)
        top = torch.maximum(top, sinks)
    w = torch.exp(s - top)
    total = w.sum(4, keepdim=True)
    if state["sinks"] is not None:
        total = total + torch.exp(sinks - top)
    o = (w.view(n_seqs, kv, -1, length) @ v).view(n_seqs, kv, -1, longest, size) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n_seqs * longest, heads * size)
    return o[(token_at >= 0).view(-1)].to(torch.bfloat16)


# -- the same from the definitions, in 64 bits ----------------------------------------------------


def _code_values():
    """What the 256 codes of e4m3 stand for: sign, four bits of exponent with bias 7, three of mantissa."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.ldexp(8 + m, e - 10) if e else math.ldexp(m, -9)
        out.append(math.nan if c & 127 == 127 else -v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _nearest_code_value(x):
    """x (64 bits) rounded to three bits behind the leading one, steps of 2^-9 at the least, ties to even."""
    _, e = torch.frexp(x)  # |x| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp_min(-6) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "product":
        out = []
        for r in range(0, case["n"], 4096):
            codes, scales = st["codes"][r : r + 4096].long(), st["scales"][r : r + 4096].double()
            w = torch.empty(codes.shape[0], case["k"], dtype=torch.float64, device=DEV)
            w[:, 0::2] = codes % 16 - 8
            w[:, 1::2] = codes // 16 - 8
            w *= scales.repeat_interleave(case["group"], dim=1)
            out.append(torch.einsum("mk,nk->mn", st["x"].double(), w))
        y = torch.cat(out, 1)
        return y if st["bias"] is None else y + st["bias"].double()
    size, heads, kv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    values = _code_values()
    lengths = _lengths(case)
    if case["op"] == "write":
        tokens = st["pos"].numel()
        angle = (st["pos"].float().unsqueeze(1) * st["freqs"]).double()
        phase = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)

        def turned(x, n):
            z = torch.view_as_complex(x.double().view(tokens, n, size // 2, 2)) * phase
            return torch.view_as_real(z).reshape(tokens, n, size)

        out = {"q": turned(st["q"], heads).reshape(tokens, heads * size)}
        for name, new in (("keys", turned(st["k"], kv)), ("values", st["v"].double().view(tokens, kv, size))):
            pools = (st["k_pages"], st["k_scales"]) if name == "keys" else (st["v_pages"], st["v_scales"])
            pages, t = [], 0
            for s, (cached, n) in enumerate(lengths):
                at = cached
                while at < cached + n:
                    slot = at % page
                    some = min(page - slot, cached + n - at)
                    lp = int(st["table"][s, at // page])
                    old = values[pools[0].view(torch.uint8)[lp].long()]
                    if name == "values":
                        old = old.permute(0, 1, 3, 2).reshape(kv, page, size)
                    before = pools[1][lp].double()
                    mine = new[t : t + some]
                    need = torch.ceil(torch.log2(mine.abs().amax((0, 2)) / LARGEST).clamp_min(LOWEST_EXPONENT))
                    scale = torch.exp2(need)
                    scale = torch.maximum(scale, before) if slot else scale
                    if slot:
                        old[:, :slot] = _nearest_code_value(old[:, :slot] * (before / scale)[:, None, None])
                    old[:, slot : slot + some] = _nearest_code_value(mine.transpose(0, 1) / scale[:, None, None])
                    pages.append(old * scale[:, None, None])
                    at, t = at + some, t + some
            out[name] = torch.stack(pages)
        return out
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    start = 0
    for s, (cached, new) in enumerate(lengths):
        total = cached + new
        lps = st["table"][s, : -(-total // page)].long()
        k = values[st["k_pages"].view(torch.uint8)[lps].long()] * st["k_scales"][lps].double()[:, :, None, None]
        v = values[st["v_pages"].view(torch.uint8)[lps].long()] * st["v_scales"][lps].double()[:, :, None, None, None]
        k = k.permute(1, 0, 2, 3).reshape(kv, -1, size)[:, :total]
        v = v.permute(1, 0, 2, 4, 3).reshape(kv, -1, size)[:, :total]
        i = torch.arange(cached, total, device=DEV)[:, None]
        j = torch.arange(total, device=DEV)[None, :]
        hidden = (j > i) | (j <= i - case["window"]) if case["window"] else j > i
        for h in range(heads):
            g = h // (heads // kv)
            q = st["q"][start : start + new, h * size : (h + 1) * size].double()
            z = (q @ k[g].T) * st["scale"]
            if case["softcap"]:
                z = torch.tanh(z / case["softcap"]) * case["softcap"]
            z = z.masked_fill(hidden, -math.inf)
            if st["sinks"] is not None:
                z = torch.cat([z, st["sinks"][h].double().expand(new, 1)], 1)
            out[start : start + new, h * size : (h + 1) * size] = torch.softmax(z, 1)[:, :total] @ v[g]
        start += new
    return out
