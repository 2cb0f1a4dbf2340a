"""The 8-bit paged KV cache on the CPU where values are not finite and sequences change hands."""
import pytest
import torch

from paged8_oracle import PAGE, Layer, attention, f64

from complexity_framework_b200.ops import paged8

INT8, FP8 = torch.int8, torch.float8_e4m3fn


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [INT8, FP8])
def test_a_later_block_that_is_not_finite_is_masked(dtype):
    """Rows before the block see and weigh the tokens before it as if it were not there."""
    L = Layer([64], 1, 16, dtype, "cpu", seed=2)
    q = torch.randn(20, 2, 16)
    m = torch.zeros(2, L.num_pages, 1, PAGE)
    outs = []
    for i in range(2):
        outs.append(paged8.paged8_attention(q, L.codes, L.scales, L.table, ints([0, 20]), L.kv_lens,
                                            scale=0.25, max_q_len=20, mass=m[i]))
        L.scales[int(L.table[0, 3])] = float("nan")
        L.codes[int(L.table[0, 3])] = 0
    assert torch.equal(outs[0][:4], outs[1][:4])         # positions 44 .. 47 see blocks 0 .. 2
    assert torch.isnan(outs[1][4:]).all()
    # the first rows alone: their weights are numbers
    m[0] = 0
    paged8.paged8_attention(q[:4], L.codes, L.scales, L.table, ints([0, 4]), ints([48]), scale=0.25,
                            max_q_len=4, mass=m[0])
    assert torch.isfinite(m[0]).all() and abs(m[0].sum().item() - 8) < 1e-4


def test_weights_of_hidden_tokens_are_not_touched_by_nan_rows():
    """A row that is not a number weighs the tokens it sees only."""
    L = Layer([40], 1, 16, INT8, "cpu", seed=2)
    q = torch.randn(20, 2, 16)
    q[3] = float("nan")                                     # at position 23
    m = torch.zeros(L.num_pages, 1, PAGE)
    paged8.paged8_attention(q, L.codes, L.scales, L.table, ints([0, 20]), L.kv_lens, scale=0.25,
                            max_q_len=20, mass=m)
    q[3] = 0
    weights = attention(L, q, [0, 20], 0.25)[2][0]
    got = m[L.table[0].long(), 0].reshape(-1)[:40]
    assert torch.isnan(got[:24]).all()
    assert (f64(got[24:]) - weights[0, 24:]).abs().max() < 1e-5


@pytest.mark.parametrize("top", [float("inf"), float("nan")])
def test_recent_tokens_stay_beside_masses_that_are_not_finite(top):
    """The last tokens are kept whatever the older ones' masses are."""
    L = Layer([40], 1, 8, INT8, "cpu", extra_pages=3)
    mass = torch.rand(L.num_pages, 1, PAGE)
    for j in range(2, 30):
        mass[int(L.table[0, j // PAGE]), 0, j % PAGE] = top
    keep = paged8.paged8_evict(L.codes, L.scales, mass, L.table, L.kv_lens, ints([L.spare[:1]]),
                               budget=12, recent=5)
    assert keep[0, 0].tolist() == list(range(2, 9)) + list(range(35, 40))


def test_static_batch_follows_a_sequence_whose_pages_change(monkeypatch):
    """A row's page table after its sequence was freed and allocated anew under the same id,
    forked into, or cut and grown again, with its old pages in other hands."""
    from complexity_framework_b200.inference import Paged8Pool

    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    pool = Paged8Pool(1, 1, 8, 20, dtype=torch.float32)
    batch = pool.static_batch(2, 8, 127)

    def step(seq, position):
        batch.fill([(seq, 1, position)])
        batch.commit()
        n = len(pool.pages[seq])
        assert batch.page_table[0, :n].tolist() == pool.pages[seq]

    def grow(seq, tokens):
        if seq not in pool.pages:
            pool.allocate_sequence(seq)
        pool.reserve(seq, tokens - pool.lengths[seq])
        pool.lengths[seq] = tokens

    grow(0, 40)
    step(0, 40)
    pool.free_sequence(0)
    grow(1, 20)
    grow(0, 30)
    step(0, 30)
    pool.truncate_sequence(0, 10)
    grow(1, 40)
    grow(0, 33)
    step(0, 33)
    pool.fork_sequence(1, 0)
    grow(2, 20)
    step(0, 40)


def small_model():
    from complexity_framework_b200 import ComplexityModel, ModelConfig

    torch.manual_seed(0)
    return ComplexityModel(ModelConfig(
        hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
        vocab_size=256, intermediate_size=64, shared_intermediate_size=64, num_experts=2, top_k=1,
        max_position_embeddings=512)).eval()


def test_paged_logits_over_an_8_bit_pool():
    """A prompt, then four drafted tokens at once: the logits of the same tokens one by one."""
    from complexity_framework_b200.inference import Paged8Pool, SeqChunk, paged_logits

    m = small_model()
    toks = torch.randint(0, 256, (24,), generator=torch.Generator().manual_seed(1)).tolist()
    logits = []
    for steps in ((20, 4), (20, 1, 1, 1, 1)):
        pool = Paged8Pool(2, 2, 16, 4, dtype=torch.float32)
        pool.allocate_sequence(0)
        at, rows = 0, []
        for n in steps:
            rows += paged_logits(m, pool, [SeqChunk(0, at, n)], toks[at:at + n],
                                 all_positions=True)[0]
            at += n
        logits.append(torch.stack(rows))
    assert logits[0].shape == (24, 256)
    # the prompt's chunk is the same call; a block's older codes may be rounded once more when
    # tokens arrive one by one, half a step of 1/127 of the largest value
    assert torch.equal(logits[0][:20], logits[1][:20])
    assert (logits[0] - logits[1]).abs().max() <= logits[0].abs().max() / 16


@pytest.mark.parametrize("lens,num_pages", [((100,), 8), ((70, 60, 50), 14)])
def test_engine_evicts_with_no_page_free(lens, num_pages):
    """Requests that fill the pool are cut to the budget, not refused the next token's page."""
    from complexity_framework_b200.inference import (GenerationConfig, InferenceConfig,
                                                     InferenceEngine)

    eng = InferenceEngine(small_model(), InferenceConfig(
        max_cache_length=512, max_batch_size=4, num_pages=num_pages, kv_cache_dtype="int8",
        kv_evict_budget=40, kv_evict_recent=16, kv_evict_slack=16, prefill_chunk_size=128))
    g = torch.Generator().manual_seed(1)
    rids = [eng.add_request(torch.randint(0, 256, (n,), generator=g).tolist(),
                            GenerationConfig(max_new_tokens=90)) for n in lens]
    while eng.has_pending():
        eng.step()
    assert [len(eng.requests[r].output) for r in rids] == [90] * len(lens)
    assert eng.stats["evictions"] >= 2 * len(lens)
    assert len(eng.pool.free) == eng.pool.num_pages


def test_pages_held_for_evictions():
    """No sequence takes them; an eviction does, and gives back as many."""
    from complexity_framework_b200.inference import OutOfPages, Paged8Pool

    pool = Paged8Pool(1, 1, 8, 4, dtype=torch.float32, track_mass=True, evict_pages=2)
    assert len(pool.free) == pool.num_pages == 6
    pool.allocate_sequence(0)
    pool.allocate_sequence(1)
    assert pool.can_reserve(0, 64) and not pool.can_reserve(0, 65)
    pool.reserve(0, 64)
    pool.lengths[0] = 64
    pool.reserve(0, 0)
    with pytest.raises(OutOfPages):
        pool.reserve(1, 1)
    pool.evict([0], budget=32, recent=8)
    assert len(pool.free) == 4 and pool.lengths[0] == 32
    pool.reserve(1, 32)
    with pytest.raises(OutOfPages):
        pool.fork_sequence(0, 2)


def test_small_budgets_and_the_recent_tokens_option():
    """A budget below 64 needs no further option; batcher and command line can set the rest."""
    from complexity_framework_b200.cli.app import _engine_config, build_parser
    from complexity_framework_b200.inference import (BatchConfig, ContinuousBatcher,
                                                     InferenceConfig, InferenceEngine)

    m = small_model()
    for budget, want in ((1, 0), (48, 24), (64, 64), (1024, 64)):
        eng = InferenceEngine(m, InferenceConfig(max_cache_length=64, max_batch_size=1,
                                                 kv_cache_dtype="int8", kv_evict_budget=budget))
        assert eng.kv_evict_recent == want
    b = ContinuousBatcher(m, BatchConfig(max_batch_size=1, max_sequence_length=64,
                                         kv_cache_dtype="fp8", kv_evict_budget=48,
                                         kv_evict_recent=8, kv_evict_slack=5))
    got = b.engine.config
    assert (got.kv_evict_budget, got.kv_evict_recent, got.kv_evict_slack) == (48, 8, 5)
    base = ["bench-infer", "--model", "x", "--kv-cache-dtype", "int8", "--kv-evict-budget", "48"]
    for more, recent, slack in (([], None, 256),
                                (["--kv-evict-recent", "7", "--kv-evict-slack", "9"], 7, 9)):
        c = _engine_config(build_parser().parse_args(base + more))
        assert (c.kv_evict_budget, c.kv_evict_recent, c.kv_evict_slack) == (48, recent, slack)
        InferenceEngine(m, c)
    with pytest.raises(ValueError):
        InferenceEngine(m, InferenceConfig(max_cache_length=64, max_batch_size=1,
                                           kv_cache_dtype="int8", kv_evict_budget=48,
                                           kv_evict_recent=49))
