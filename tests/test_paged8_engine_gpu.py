"""The 8-bit paged cache in the serving engine, on the kernels."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
           vocab_size=2048, intermediate_size=256, shared_intermediate_size=512, num_experts=4,
           top_k=2, max_position_embeddings=1024)


def engine(model, **kw):
    from complexity_framework_b200.inference import InferenceConfig, InferenceEngine

    return InferenceEngine(model, InferenceConfig(**{"max_cache_length": 512, "max_batch_size": 8,
                                                     **kw}))


def model():
    from complexity_framework_b200 import ComplexityModel, ModelConfig

    torch.manual_seed(0)
    return ComplexityModel(ModelConfig(**CFG)).cuda().to(torch.bfloat16).eval()


def prompts():
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 2048, (n,), generator=g).tolist() for n in (5, 17, 140, 33, 64, 300)]


@pytest.mark.parametrize("kv_dtype", ["int8", "fp8"])
@pytest.mark.parametrize("budget", [0, 96])
def test_graph_decode_matches_eager(kv_dtype, budget):
    """Decode steps replayed from CUDA graphs (padded rows, page tables that an eviction
    replaces) give the eager engine's tokens."""
    from complexity_framework_b200.inference import GenerationConfig
    from complexity_framework_b200.ops import check_errors

    m, outs = model(), {}
    for graph in (False, True):
        eng = engine(m, cuda_graph_decode=graph, kv_cache_dtype=kv_dtype, kv_evict_budget=budget,
                     kv_evict_recent=32, kv_evict_slack=16, prefill_chunk_size=128)
        rids = [eng.add_request(p, GenerationConfig(max_new_tokens=12 + 7 * i))
                for i, p in enumerate(prompts())]
        while eng.has_pending():
            eng.step()
        outs[graph] = [eng.requests[r].output for r in rids]
        assert (eng.stats.get("graph_steps", 0) > 0) == graph
        assert (eng.stats.get("evictions", 0) > 0) == (budget > 0)
        assert len(eng.pool.free) == eng.pool.num_pages
    check_errors(0)
    assert outs[True] == outs[False]


@pytest.mark.parametrize("kv_dtype", ["int8", "fp8"])
def test_kernels_match_the_reference_operators(kv_dtype):
    """The same ragged steps through a pool on the GPU and one on the CPU."""
    from complexity_framework_b200.inference import Paged8Pool, SeqChunk

    torch.manual_seed(4)
    pools = [Paged8Pool(1, 2, 64, 60, dtype=torch.bfloat16, device=d, kv_dtype=kv_dtype,
                        track_mass=True) for d in ("cuda", "cpu")]
    at = {0: 0, 1: 0, 2: 0}
    for p in pools:
        for s in at:
            p.allocate_sequence(s)
    for new in ((40, 200, 3), (1, 1, 1), (5, 130, 1), (1, 1, 40)):
        chunks = [SeqChunk(s, at[s], n) for s, n in enumerate(new)]
        N = sum(new)
        k, v = torch.randn(2, N, 2, 64).bfloat16()
        q = torch.randn(N, 8, 64).bfloat16()
        outs = []
        for p in pools:
            b = p.batch(chunks)
            b.write(0, k.to(p.device), v.to(p.device))
            outs.append(b.attend(0, q.to(p.device), 0.125).float().cpu())
            b.commit()
        for s, n in enumerate(new):
            at[s] += n
        # both round to bf16 (2^-8 of values below 4), the kernels also P to f16
        assert (outs[0] - outs[1]).abs().max() <= 4 * (2.0 ** -8 + 2.0 ** -10)
    assert torch.allclose(pools[0].scales.cpu(), pools[1].scales, rtol=2.0 ** -22)
    m = [p.mass.cpu() for p in pools]
    assert torch.allclose(m[0], m[1], rtol=1e-4, atol=1e-5)


def test_cache_memory_is_half():
    from complexity_framework_b200.inference import Paged8Pool, PagePool

    a = PagePool(2, 8, 128, 100, device="cuda").memory_usage()["gb_total"]
    b = Paged8Pool(2, 8, 128, 100, device="cuda").memory_usage()["gb_total"]
    assert b < 0.51 * a


def test_refusals():
    from complexity_framework_b200.inference import Paged8Pool

    with pytest.raises(ValueError):
        Paged8Pool(1, 2, 96, 4, device="cuda")
    with pytest.raises(ValueError):
        Paged8Pool(1, 2, 64, 4, device="cuda", dtype=torch.float32)
