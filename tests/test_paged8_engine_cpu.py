"""The 8-bit paged cache in the serving engine (CPU)."""
import pytest
import torch

from complexity_framework_b200 import ComplexityModel, ModelConfig
from complexity_framework_b200.inference import (BatchConfig, ContinuousBatcher, GenerationConfig,
                                                 InferenceConfig, InferenceEngine, OutOfPages,
                                                 Paged8Pool, PagePool, Request, SeqChunk)

CFG = dict(hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
           vocab_size=256, intermediate_size=64, shared_intermediate_size=64, num_experts=2, top_k=1,
           max_position_embeddings=512)


def model():
    torch.manual_seed(0)
    return ComplexityModel(ModelConfig(**CFG)).eval()


def prompts(*lens):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 256, (n,), generator=g).tolist() for n in lens]


def fill(pool, seq, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    pool.allocate_sequence(seq)
    b = pool.batch([SeqChunk(seq, 0, n)])
    kv = torch.randn(2, pool.num_layers, n, pool.num_kv_heads, pool.head_dim, generator=g)
    for layer in range(pool.num_layers):
        b.write(layer, kv[0, layer], kv[1, layer])
    b.commit()
    return kv


@pytest.mark.parametrize("kv_dtype,step", [("int8", 0.5 / 127), ("fp8", 2.0 ** -4)])
def test_pool_holds_what_was_written(kv_dtype, step):
    pool = Paged8Pool(3, 2, 8, 12, device="cpu", dtype=torch.float32, kv_dtype=kv_dtype)
    kv = fill(pool, 7, 37)
    for got, want in zip(pool.read(7), kv):
        assert got.shape == (3, 2, 37, 8)
        # one rounding of values within the largest magnitude
        assert (got.transpose(1, 2) - want).abs().max() <= step * want.abs().max() * (1 + 1e-5)
    pool.fork_sequence(7, 8)
    assert all(torch.equal(a, b) for a, b in zip(pool.read(7), pool.read(8)))
    pool.truncate_sequence(8, 20)
    assert pool.lengths[8] == 20 and len(pool.pages[8]) == 2
    assert torch.equal(pool.read(8)[0], pool.read(7)[0][:, :, :20])
    pool.reset()
    assert len(pool.free) == 12 and not pool.dropped


def test_attend_is_near_the_exact_cache():
    """A ragged step (a decode token, a long and a short chunk) over both caches."""
    torch.manual_seed(3)
    exact = PagePool(1, 2, 16, 40, 16, dtype=torch.float32)
    small = Paged8Pool(1, 2, 16, 40, dtype=torch.float32)
    for pool in (exact, small):
        fill(pool, 0, 30, 1)
        fill(pool, 1, 100, 2)
        fill(pool, 2, 5, 3)
    chunks = [SeqChunk(0, 30, 1), SeqChunk(1, 100, 90), SeqChunk(2, 5, 3)]
    k, v, q = torch.randn(94, 2, 16), torch.randn(94, 2, 16), torch.randn(94, 8, 16)
    outs = []
    for pool in (exact, small):
        b = pool.batch(chunks)
        b.write(0, k, v)
        outs.append(b.attend(0, q, 0.25))
        b.commit()
        assert [pool.lengths[i] for i in range(3)] == [31, 190, 8]
    # int8 keys move a score by at most scale * |q|_1 * half a step, values by half a step, and
    # a step is largest|x| / 127 with |x| < 4.5 here
    half = 4.5 / 127 / 2
    score = 0.25 * q.abs().sum(-1).max().item() * half
    bound = half + 4.5 * 2 * (torch.tensor(2 * score).exp().item() - 1)
    assert (outs[0] - outs[1]).abs().max() <= bound


def test_evict_keeps_heavy_and_recent_tokens():
    pool = Paged8Pool(2, 2, 8, 16, dtype=torch.float32, track_mass=True)
    fill(pool, 0, 50)
    fill(pool, 1, 10)
    before = pool.read(0)
    heavy = [3, 17, 30, 31]
    for j in heavy:
        pool.mass[:, pool.pages[0][j // 16], :, j % 16] = 5.0 + j
    free = len(pool.free)
    pool.evict([0, 1], budget=12, recent=8)
    assert pool.lengths == {0: 12, 1: 10} and pool.dropped == {0: 38, 1: 0}
    assert len(pool.free) == free + 3                      # four pages became one
    keep = heavy + list(range(42, 50))
    for got, want in zip(pool.read(0), before):
        step = want.abs().max() / 127                      # rounded once more
        assert (got - want[:, :, keep]).abs().max() <= 0.5 * step * (1 + 1e-5)
    # the next token takes slot 12 at position 50, with no mass yet
    pool.mass[:, pool.pages[0][0]] = 3.0
    b = pool.batch([SeqChunk(0, 50, 1)])
    b.write(0, torch.ones(1, 2, 8), torch.ones(1, 2, 8))
    assert b.positions.tolist() == [50] and b.kv_lens.tolist() == [13]
    assert (pool.mass[0, pool.pages[0][0], :, 12] == 0).all()
    b.commit()
    assert pool.lengths[0] == 13
    with pytest.raises(OutOfPages):
        pool.free.clear()
        pool.evict([0], budget=4, recent=2)


@pytest.mark.parametrize("kv_dtype", ["int8", "fp8"])
def test_engine_generates(kv_dtype):
    m = model()
    eng = InferenceEngine(m, InferenceConfig(max_cache_length=256, max_batch_size=4,
                                             kv_cache_dtype=kv_dtype, prefill_chunk_size=32))
    out = eng.generate_tokens(prompts(5, 70, 33), GenerationConfig(max_new_tokens=9))
    assert [len(o) for o in out] == [9, 9, 9]
    assert len(eng.pool.free) == eng.pool.num_pages
    # the tokens do not depend on how requests are batched
    for p, o in zip(prompts(5, 70, 33), out):
        alone = InferenceEngine(m, InferenceConfig(max_cache_length=256, max_batch_size=4,
                                                   kv_cache_dtype=kv_dtype, prefill_chunk_size=32))
        assert alone.generate_tokens([p], GenerationConfig(max_new_tokens=9)) == [o]


def test_engine_evicts_to_the_budget():
    eng = InferenceEngine(model(), InferenceConfig(
        max_cache_length=256, max_batch_size=2, kv_cache_dtype="int8", kv_evict_budget=40,
        kv_evict_recent=16, kv_evict_slack=24, prefill_chunk_size=30))
    rids = [eng.add_request(p, GenerationConfig(max_new_tokens=60)) for p in prompts(100, 20)]
    seen = 0
    while eng.has_pending():
        eng.step()
        seen = max([seen] + list(eng.pool.lengths.values()))
    assert seen <= 40 + 24 + 29                              # a chunk may land on a full budget
    assert eng.stats["evictions"] >= 4
    assert [len(eng.requests[r].output) for r in rids] == [60, 60]
    assert len(eng.pool.free) == eng.pool.num_pages


def test_budget_that_is_never_reached_changes_nothing():
    m = model()
    outs = [InferenceEngine(m, InferenceConfig(max_cache_length=128, max_batch_size=2,
                                               kv_cache_dtype="int8", kv_evict_budget=b))
            .generate_tokens(prompts(30, 12), GenerationConfig(max_new_tokens=8)) for b in (0, 100)]
    assert outs[0] == outs[1]


def test_batcher_and_refusals():
    m = model()
    b = ContinuousBatcher(m, BatchConfig(max_batch_size=2, kv_cache_dtype="fp8"))
    b.add_request(Request(prompts(9)[0], max_tokens=3, temperature=0.0))
    assert [len(r.output_ids) for r in b.run_until_complete()] == [3]
    for bad in (dict(kv_cache_dtype="int4"), dict(kv_evict_budget=10),
                dict(kv_cache_dtype="int8", page_size=32),
                dict(kv_cache_dtype="int8", kv_evict_budget=10, kv_evict_recent=11),
                dict(kv_cache_dtype="int8", kv_evict_budget=10, kv_evict_recent=1, kv_evict_slack=0)):
        with pytest.raises(ValueError):
            InferenceEngine(m, InferenceConfig(max_cache_length=64, max_batch_size=1, **bad))
    pool = Paged8Pool(1, 1, 8, 2, dtype=torch.float32)
    fill(pool, 0, 20)
    with pytest.raises(RuntimeError):
        pool.evict([0], 8, 2)
