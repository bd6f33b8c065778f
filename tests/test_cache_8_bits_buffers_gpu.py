"""The work buffers of the cache in 8 bits: streams, threads, engines that come and go."""

import ctypes
import gc
import threading

import pytest
import torch

import helpers as H
from test_cache_8_bits_gpu import DEV, Cache, _context

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ops():
    from fastgen_b200.csrc.ops import Ops
    return Ops(torch.bfloat16, DEV)


def _case(ops, seed, lengths=(700, 90), portion=40):
    """A cache with its call: single tokens beside a portion of a prompt."""
    size, page, heads, kv = 64, 32, 4, 2
    cache = Cache(ops, len(lengths) + 1, 30, kv, page, size)
    for s, n in enumerate((*lengths, 300 + portion)):
        cache.fill(s, n, 10 * seed + s)
    ctx = _context([n - 1 for n in lengths] + [300], [1] * len(lengths) + [portion])
    q = torch.randn(ctx.n_tokens, heads * size, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)

    def call():
        out = torch.empty_like(q)
        ops.attention(q, out, cache.memory, ctx, heads, kv, size, None, 0.1)
        return out

    return call


def test_a_stream_that_is_gone(ops):
    """A stream of another library is used and destroyed; later calls have nothing to do with it."""
    call = _case(ops, 1)
    want = call()
    torch.cuda.synchronize()
    runtime = ctypes.CDLL("libcudart.so.12")
    for _ in range(3):
        handle = ctypes.c_void_p()
        assert runtime.cudaStreamCreate(ctypes.byref(handle)) == 0
        with torch.cuda.stream(torch.cuda.ExternalStream(handle.value, device=DEV)):
            got = call()
        torch.cuda.synchronize()
        assert runtime.cudaStreamDestroy(handle) == 0
        assert torch.equal(got, want) and torch.equal(call(), want)
    torch.cuda.synchronize()


def test_threads_on_streams_of_their_own(ops):
    """Threads that call at the same time, each on its stream and its cache of one and the same shape."""
    calls = [_case(ops, seed) for seed in range(4)]
    wants = [call() for call in calls]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                if not torch.equal(calls[i](), wants[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    ops.check_status()
    assert not wrong


def test_threads_on_one_stream(ops):
    calls = [_case(ops, seed) for seed in range(4)]
    wants = [call() for call in calls]
    got = [[] for _ in calls]

    def work(i):
        for _ in range(40):
            got[i].append(calls[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ops.check_status()
    assert all(torch.equal(x, want) for mine, want in zip(got, wants) for x in mine)


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
