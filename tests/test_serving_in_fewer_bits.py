"""Serving with a cache in 8 bits and with 4-bit weights: what is refused (on the CPU), and whole models through the engine."""

import queue

import numpy as np
import pytest
import torch

import helpers as H

DEV = "cuda:0"


# -- refusals and layouts: no GPU -------------------------------------------------------------------


def test_weights_of_4_bits_stand_for_what_they_say():
    from fastgen_b200.weights import Weight4
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 256, (7, 192), generator=g, dtype=torch.uint8)
    for group in (32, 64, 128):
        scales = torch.rand(7, 384 // group, generator=g).to(torch.bfloat16)
        w = Weight4(codes, scales)
        want = torch.stack([codes & 15, codes >> 4], 2).view(7, 384).double() - 8
        want = (want.view(7, -1, group) * scales.double()[..., None]).view(7, 384)
        assert torch.equal(w.dequantize(torch.float64), want) and w.shape == (7, 384) and w.numel() == 7 * 384
        assert torch.equal(w[2:5].dequantize(torch.float64), want[2:5])
        assert w.nbytes() == 7 * 192 + 2 * scales.numel()


def test_codes_may_be_a_view():
    from fastgen_b200.weights import Weight4
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(0, 256, (64, 6), dtype=torch.uint8, generator=g).t()  # [6, 64], columns neighbours in memory
    scales = torch.rand(2, 6, generator=g).bfloat16().t()
    assert torch.equal(Weight4(codes, scales).dequantize(), Weight4(codes.contiguous(), scales.contiguous()).dequantize())


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantized_weights_are_the_nearest(group):
    """Half a step of the scale, and what rounding the scale to bfloat16 (2^-8 of it) leaves at the ends, 7 steps away."""
    from fastgen_b200.weights import Weight4
    g = torch.Generator().manual_seed(group)
    w = torch.randn(33, 3 * 128, generator=g)
    w[4, :group] = 0
    w[5] *= 1e-30
    q = Weight4.quantize(w.t().contiguous().t(), group)
    steps = (w.view(33, -1, group).abs().amax(2, keepdim=True) / 7).expand(-1, -1, group).reshape(w.shape)
    # (a scale that bfloat16 holds as a subnormal number has fewer bits; these are all normal ones)
    assert bool(((q.dequantize() - w).abs() <= (0.5 * (1 + 2.0 ** -8) + 7 * 2.0 ** -8) * steps).all())
    assert bool((q.dequantize()[4, :group] == 0).all())


def test_refused_weights():
    from fastgen_b200.csrc.ops import check_weight_bits
    from fastgen_b200.weights import Weight4
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.bfloat16)
    Weight4(codes, scales)
    for bad in ((codes.int(), scales), (codes, scales.float()), (codes, scales[:3]), (codes, torch.zeros(4, 8, dtype=torch.bfloat16)),
                (codes, torch.zeros(4, 3, dtype=torch.bfloat16)), (codes[:0], scales[:0]), (codes, torch.zeros(4, 0, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            Weight4(*bad)
    with pytest.raises(ValueError, match="no multiple"):
        Weight4.quantize(torch.zeros(4, 100))
    with pytest.raises(ValueError, match="groups of 16"):
        Weight4.quantize(torch.zeros(4, 128), 16)
    with pytest.raises(ValueError):
        Weight4.quantize(torch.zeros(4, 128, dtype=torch.int32))
    with pytest.raises(TypeError):
        Weight4(codes, scales)[1]
    check_weight_bits(torch.float32, 16, 128)
    check_weight_bits(torch.bfloat16, 4, 32)
    for bad in ((torch.bfloat16, 8, 128), (torch.float32, 4, 128), (torch.bfloat16, 4, 100)):
        with pytest.raises(ValueError):
            check_weight_bits(*bad)


def test_refused_caches():
    from fastgen_b200.cache import CacheManager
    from fastgen_b200.csrc.ops import Ops
    from fastgen_b200.parts.base import CacheSpec
    with pytest.raises(ValueError, match="16 bits an entry"):
        CacheManager([CacheSpec(1, 64)], [None], [None], 16, 4, 1, 64, cache_bits=4)
    with pytest.raises(ValueError, match="keys and values"):
        CacheManager([CacheSpec(1, 64, n_pools=1)], [None], [None], 16, 4, 1, 64, device="cpu", cache_bits=8)
    for size, page, why in ((64, 16, None), (256, 256, None), (48, 64, "head size"), (128, 24, "pages"), (128, 8, "pages"), (128, 512, "pages")):
        got = Ops.kv8_supported(size, page)
        assert (got is None) if why is None else why in got


def test_pools_of_a_cache_in_8_bits():
    """The manager's bookkeeping is the same; its pools are codes and scales."""
    from fastgen_b200.cache import CacheManager
    from fastgen_b200.parts.base import CacheSpec
    m = CacheManager([CacheSpec(2, 64)] * 3, [None] * 3, [None] * 3, 16, 5, 2, 80, device="cpu", cache_bits=8)
    mem = m.memory(2)
    assert mem.k_pages.shape == (5, 2, 16, 64) and mem.v_pages.shape == (5, 2, 4, 64, 4)
    assert mem.k_pages.dtype == mem.v_pages.dtype == torch.float8_e4m3fn
    assert mem.k_scales.shape == mem.v_scales.shape == (5, 2) and mem.k_scales.dtype == torch.float32 and mem.layer_index == 2
    assert mem.k_scales.data_ptr() == m.groups[0].k_scales[2].data_ptr()
    r = m.admit("a")
    m.reserve(r, 70)
    m.flush_tables()
    m.check()
    plain = CacheManager([CacheSpec(2, 64)], [None], [None], 16, 5, 2, 80, device="cpu").memory(0)
    assert plain.k_scales is None and plain.v_scales is None


def test_signatures_belong_to_their_library():
    import re
    from pathlib import Path
    from fastgen_b200.csrc import build, kv8_ops
    csrc = Path(build.__file__).parent
    names = set(re.findall(r'extern "C" \w[\w\s\*]*?\b(fg_\w+)\(', (csrc / "kv8.cu").read_text()))
    assert set(kv8_ops.SIGNATURES) <= names
    called = set(re.findall(r"\blib\.(fg_kv8_\w+)\(", Path(kv8_ops.__file__).read_text()))
    assert called <= set(kv8_ops.SIGNATURES)


# -- models ------------------------------------------------------------------------------------------


def _run(model_dir, steps, page, max_tokens, cache_bits=16, weight_bits=16, weight_group=64, graphs=True, max_requests=4,
         max_step_tokens=None):
    from fastgen_b200.engine import Engine, Model, StepEntry
    model = Model.load(model_dir, torch.bfloat16, DEV, weight_bits=weight_bits, weight_group=weight_group)
    n_pages = -(-max_tokens // page)
    engine = Engine(model, page_size=page, n_pages=n_pages, max_requests=max_requests, max_length=min(model.args.max_positions, n_pages * page),
                    use_graphs=graphs, max_step_tokens=max_step_tokens, cache_bits=cache_bits)
    outputs, live = {}, set()
    for st in steps:
        entries = []
        for e in st["entries"]:
            if e["id"] not in live:
                engine.admit(e["id"])
                live.add(e["id"])
            entries.append(StepEntry(e["id"], e["tokens"], e["want"]))
        logits = engine.step(entries)
        if logits is not None:
            outputs[st["step"]] = logits.float().cpu().numpy()
        engine.ops.check_status()
        for rid in st["end"]:
            engine.release(rid)
            live.discard(rid)
    return outputs, engine


def _requests(vocab, lengths, seed):
    return {f"r{i}": H.random_tokens(vocab, n, seed + i) for i, n in enumerate(lengths)}


@pytest.mark.gpu
@pytest.mark.parametrize("name,page", [("tiny_d", 16), ("tiny_d", 64), ("tiny_e", 32), ("tiny_e", 128)])
def test_models_with_a_cache_in_8_bits(tmp_path, name, page):
    """Whole prompts, portions and single tokens, requests that follow one another on the same pages, with and without graphs.
    An entry is off by 2^-4 of itself at most, a random rounding: rows of logits stay within 2^-4 of the plain model's norm (a
    wrong page or scale puts them as far away as the row is long)."""
    model_dir = H.make_model_dir(tmp_path, name)
    requests = _requests(H.CONFIGS[name][0]["vocab_size"], [150, 3, 77, 200, 65], 5)
    worst = 0.0
    by_plan = {}
    for plan, steps in (("whole", H.plan_whole(requests)), ("tail", H.plan_decode_tail(requests, 40)), ("portions", H.plan_portions(requests)),
                        ("mixed", H.plan_mixed(requests, 3))):
        for graphs in (True, False):
            out, engine = _run(model_dir, steps, page, H.max_live_tokens(steps, max(64, page)) + 4 * page, cache_bits=8, graphs=graphs,
                               max_step_tokens=256 if graphs else None)
            assert engine.cache.groups[0].k_pages.dtype == torch.float8_e4m3fn
            got = H.collect(steps, out)
            by_plan[plan, graphs] = got
            for rid, tokens in requests.items():
                want = H.plain_logits(model_dir, tokens)
                for p, row in got[rid].items():
                    off = float(np.linalg.norm(row - want[p]) / np.linalg.norm(want[p]))
                    worst = max(worst, off)
                    assert off <= 2.0 ** -4, (plan, rid, p, off)
    print(f"worst row {worst:.4f}")


def _pegurax():
    import test_pegurax_gpu as m
    return m, "pc", (m.T_L2, 0.0, 1.0)  # pairs whose attention has chunks, head sizes 64 and 128 in one model


def _palulorn():
    import test_palulorn_gpu as m
    layers = [m._layer("attention", m._attn(6, 3, 64, 32, 0.1, conv=2, rot=(8, 5000.0, 8.0), window=20), m._moe(6, 3, 40, (3, 2), 2.0, 24)),
              m._layer("parallel", m._pair(m._sink(4, 2, 64, 0.15, (0.5, 7)), m._memory(3, 24, 40, 10.0)), m._moe(5, 2, 24)),
              m._layer("attention", m._attn(2, 1, 128, 48, 0.12, conv=4, rot=(24, 300.0, None), window=70), None)]
    m.CONFIGS["fewer bits"] = (dict(architecture="Palulorn", vocab=211, width=96, norm=dict(eps=1e-5), embedding=dict(scale=3.0),
                                    loop=dict(start=1, stop=3, times=2), layers=layers), 21)
    return m, "fewer bits", (m.T_L2, m.T_SHARE, m.T_FAR)  # sinks, values that are keys, windows, convolutions, layers passed twice


@pytest.mark.gpu
@pytest.mark.parametrize("design", [_pegurax, _palulorn])
def test_other_designs_with_a_cache_in_8_bits(tmp_path, design):
    """Mixers that join attention with others, through the engine, held to that design's own bfloat16 rule widened by the
    entries' rounding: an entry is off by 2^-4 of itself at most, so attention's outputs are off by 2^-4 of the largest value
    where bfloat16 has them off by its 2^-8, and what the design's rule allows a row (``T_L2`` of its norm) grows by 2^-4.
    Where the rule lets a share of the rows be ``T_FAR`` times as far, because a read-out that nearly cancels carries what
    comes in at full size, that factor is on both.  On average, where roundings are random, rows are within half."""
    m, name, (room, share, far_times) = design()
    room += 2.0 ** -4
    folder = m.model_dir(tmp_path, name, torch.bfloat16)
    vocab = m.CONFIGS[name][0]["vocab"]
    requests = _requests(vocab, [150, 3, 77, 200], 5)
    steps = H.plan_mixed(requests, 3)
    for graphs in (True, False):
        out, engine = _run(folder, steps, 32, H.max_live_tokens(steps, 64) + 512, cache_bits=8, graphs=graphs,
                           max_step_tokens=256 if graphs else None)
        assert all(g.k_pages.dtype == torch.float8_e4m3fn for g in engine.cache.groups)
        got = H.collect(steps, out)
        far = []
        for rid, tokens in requests.items():
            want = m.plain_logits(folder, tokens)
            far += [float(np.linalg.norm(row - want[p]) / np.linalg.norm(want[p])) for p, row in got[rid].items()]
        print(f"worst row {max(far):.4f}, average {np.mean(far):.4f}")
        assert max(far) <= far_times * room and np.mean(far) <= room / 2
        assert sum(x > room for x in far) <= share * len(far)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64])
def test_models_with_4_bit_weights(tmp_path, group):
    """The plain model with the matrices that the codes stand for, under the rule of bfloat16 models."""
    import plain_llama as pl
    from fastgen_b200.weights import Weight4
    from safetensors.torch import load_file, save_file
    model_dir = H.make_model_dir(tmp_path, "tiny_b")
    tensors = load_file(str(model_dir / "model.safetensors"))
    for n, t in tensors.items():
        if "_proj" in n:
            # (the rows of queries and keys are reordered as they are bound; groups lie within rows)
            tensors[n] = Weight4.quantize(t, group).dequantize(torch.float32)
    copy = tmp_path / "dense"
    copy.mkdir()
    save_file(tensors, str(copy / "model.safetensors"))
    (copy / "config.json").write_text((model_dir / "config.json").read_text())
    requests = _requests(320, [90, 5, 200], 11)
    for steps in (H.plan_whole(requests), H.plan_decode_tail(requests, 30), H.plan_mixed(requests, 2)):
        out, engine = _run(model_dir, steps, 16, H.max_live_tokens(steps) + 64, weight_bits=4, weight_group=group, max_step_tokens=256)
        assert isinstance(engine.model.blocks[0].ffn.w13, Weight4) and isinstance(engine.model.blocks[0].mixer.wqkv, Weight4)
        H.compare(copy, requests, H.collect(steps, out), torch.bfloat16)
    whole = _run(model_dir, [], 16, 64)[1].model.weight_bytes()
    assert engine.model.weight_bytes() < 0.5 * whole


@pytest.mark.gpu
def test_generation_in_fewer_bits(tmp_path):
    """``GenArgs(cache_bits=8, weight_bits=4)`` through the generator: continuous batching gives a request the tokens it gets
    alone, or one whose logit is as near as the batches' roundings (16-bit activations, 2^-8 of the row's largest)."""
    import json
    from fastgen_b200.engine import Fastgen, GenArgs, HfLoader, Packet
    from fastgen_b200.weights import write_random_model
    cfg = dict(H.TINY_D, intermediate_size=384)
    model_dir = write_random_model(tmp_path / "m", cfg, 3, dtype=torch.bfloat16, norm_jitter=0.1)
    assert json.loads((model_dir / "config.json").read_text())["intermediate_size"] == 384
    prompts = [H.random_tokens(300, n, n) for n in (5, 1, 130, 40, 66, 200)]

    def generate(batch, which):
        fg = Fastgen.build(HfLoader(model_dir), GenArgs(use_sampling=False, max_gen=12, cache_block=32, max_seq=1024, max_batch=batch,
                                                       max_prefill=96, cache_bits=8, weight_bits=4, weight_group=128), device=DEV)
        q = queue.Queue()
        for i in which:
            q.put(Packet(thread_id=i, tokens=prompts[i]))
        q.put(None)
        got = {p.thread_id: p for p in fg.generate(q)}
        assert all(p.error is None for p in got.values())
        fg.destroy()
        return {i: p.tokens for i, p in got.items()}

    together = generate(6, range(6))
    assert all(len(together[i]) == 12 for i in range(6))
    same = 0
    for i in range(6):
        alone = generate(1, [i])[i]
        same += alone == together[i]
    assert same >= 3  # (greedy tokens part ways for good where two logits are within a rounding)


@pytest.mark.gpu
def test_models_that_cannot_be_served_in_fewer_bits(tmp_path):
    from fastgen_b200.engine import Engine, Model
    d = H.make_model_dir(tmp_path, "tiny_d")
    with pytest.raises(ValueError, match="no multiple of the group"):
        Model.load(d, torch.bfloat16, DEV, weight_bits=4)  # a feed-forward of 344
    with pytest.raises(ValueError, match="serve bfloat16"):
        Model.load(d, torch.float32, DEV, weight_bits=4)
    model = Model.load(d, torch.bfloat16, DEV)
    with pytest.raises(ValueError, match="pages of 24 tokens"):
        Engine(model, page_size=24, n_pages=4, max_requests=1, cache_bits=8)
    with pytest.raises(ValueError, match="16 bits an entry"):
        Engine(model, page_size=32, n_pages=4, max_requests=1, cache_bits=4)
    with pytest.raises(ValueError, match="serves bfloat16"):
        Engine(Model.load(d, torch.float32, DEV), page_size=32, n_pages=4, max_requests=1, cache_bits=8)
    small = Model.load(H.make_model_dir(tmp_path, "tiny_b"), torch.bfloat16, DEV)
    with pytest.raises(ValueError, match="head size 32"):
        Engine(small, page_size=32, n_pages=4, max_requests=1, cache_bits=8)
