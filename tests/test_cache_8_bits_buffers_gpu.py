"""The work buffers of the cache in 8 bits: engines that come and go."""

import gc

import pytest
import torch

import helpers as H
from test_cache_8_bits_gpu import DEV, Cache, _context

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ops():
    from fastgen_b200.csrc.ops import Ops
    return Ops(torch.bfloat16, DEV)


def test_an_engine_takes_its_pages_with_it(tmp_path):
    """The pages that prompt portions read are the engine's: nothing of them is left when it goes, whatever the size of the next."""
    from fastgen_b200.engine import Engine, Model, StepEntry
    model = Model.load(H.make_model_dir(tmp_path, "tiny_d"), torch.bfloat16, DEV)
    prompt = H.random_tokens(200, 100, 3)
    held = []
    for n_pages in (64, 512, 128, 256, 64):
        engine = Engine(model, page_size=32, n_pages=n_pages, max_requests=2, max_length=512, use_graphs=False, cache_bits=8)
        engine.admit("a")
        engine.step([StepEntry("a", prompt, [99])])
        engine.ops.check_status()
        del engine
        gc.collect()
        held.append(torch.cuda.memory_allocated(DEV))
    assert len(set(held[1:])) == 1, held


def test_pages_of_another_shape_are_refused(ops):
    from dataclasses import replace
    cache, other = Cache(ops, 1, 2, 2, 32, 64), Cache(ops, 1, 3, 2, 32, 64)
    memory = replace(cache.memory, expanded=ops.make_kv8_expanded(tuple(other.memory.k_pages.shape)))
    q = torch.zeros(5, 4 * 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="comes with the expanded pages"):
        ops.attention(q, q.clone(), memory, _context([0], [5]), 4, 2, 64, None, 1.0)
