"""What serving in fewer bits counts of its memory and its traffic."""

import pytest
import torch

import helpers as H

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _folder(tmp_path):
    from fastgen_b200.weights import write_random_model
    return write_random_model(tmp_path / "m", dict(H.TINY_D, intermediate_size=384), 3, dtype=torch.bfloat16, norm_jitter=0.1)


def test_the_budget_holds_a_16_bit_copy_of_4_bit_weights(tmp_path):
    """Steps of many tokens expand a matrix at a time: the cache gets what is left beside the largest."""
    from fastgen_b200.engine import Fastgen, GenArgs, HfLoader
    args = GenArgs(use_sampling=False, max_gen=4, cache_block=32, max_batch=2, gpu_gb=0.103, prefill_gb=0.1, weight_bits=4)
    fg = Fastgen.build(HfLoader(_folder(tmp_path)), args, device=DEV)
    cfg = H.TINY_D
    rows = max(2 * 384, (cfg["num_attention_heads"] + 2 * cfg["num_key_value_heads"]) * cfg.get("head_dim", cfg["hidden_size"] // cfg["num_attention_heads"]))
    largest = 2 * rows * cfg["hidden_size"]
    assert fg.model.expanded_weight_bytes() == largest > 0
    per_token = fg.model.cache_bytes_per_token(2)
    expect = (int(0.103e9) - fg.model.weight_bytes() - largest - int(0.1e9)) // per_token
    assert fg.max_seq == -(-expect // 32) * 32 and expect > 32
    fg.destroy()


@pytest.mark.parametrize("page", [16, 64])
def test_the_budget_holds_the_scales_of_an_8_bit_cache(tmp_path, page):
    """What the pools of an engine hold for each token: codes, scales and the one layer that portions read."""
    from fastgen_b200.engine import Fastgen, GenArgs, HfLoader
    args = GenArgs(use_sampling=False, max_gen=4, cache_block=page, max_batch=2, gpu_gb=0.103, prefill_gb=0.1, cache_bits=8, num_cuda_graphs=1)
    fg = Fastgen.build(HfLoader(_folder(tmp_path)), args, device=DEV)
    grp = fg.engine.cache.groups[0]
    held = {t.data_ptr(): t.numel() * t.element_size() for t in (grp.k_pages, grp.v_pages, grp.k_scales, grp.v_scales, *fg.engine.memories[0].expanded[:2])}
    per_token = fg.model.cache_bytes_per_token(1, page)
    assert sum(held.values()) / fg.max_seq <= per_token < sum(held.values()) / fg.max_seq + 1
    expect = (int(0.103e9) - fg.model.weight_bytes() - int(0.1e9)) // per_token
    assert fg.max_seq == -(-expect // page) * page and expect > page
    fg.destroy()


def test_what_a_step_of_single_tokens_reads(tmp_path, monkeypatch, capsys):
    """The serving benchmark's share of the memory rate counts codes and scales of a cached token, not the pool of portions."""
    import json
    import sys
    from fastgen_b200.engine import Model
    from fastgen_b200.tools import serve_bench
    model = Model.load(_folder(tmp_path), torch.bfloat16, DEV)
    codes = 2 * 2 * 2 * 64  # layers, keys and values, heads of 64
    assert model.cache_bytes_per_token(1, 64, expanded=False) == codes + 1  # 8 scales of 4 bytes a page of 64, rounded up
    assert model.cache_bytes_per_token(1, 64) == codes + 1 + 2 * 2 * 2 * 64
    assert model.cache_bytes_per_token(2, 64, expanded=False) == 2 * codes == model.cache_bytes_per_token(2)
    got = []
    plain = serve_bench.roofline_of
    monkeypatch.setattr(serve_bench, "roofline_of", lambda log, cfg, weights, per_token, *rest: got.append(per_token) or plain(log, cfg, weights, per_token, *rest))
    monkeypatch.setattr(sys, "argv", ["serve_bench", "--shape", "1b", "--layers", "2", "--requests", "2", "--cache-bits", "8", "--arrive-over", "0"])
    assert serve_bench.main() == 0
    shape = serve_bench.SHAPES["1b"]
    heads, size = shape["num_key_value_heads"], shape["head_dim"]
    assert got == [2 * 2 * heads * size + -(-2 * 2 * heads * 4 // 64)]
    assert json.loads(capsys.readouterr().out.strip().splitlines()[-1])["errors"] == 0
