"""8-bit paged KV cache kernels on calls that own part of a batch, on rows and lengths at their
limits, and on inputs far apart in size, against the 64-bit oracle (tests/paged8_oracle.py).

Tolerances.  Probabilities are rounded to f16 (2^-11 of each; 2^-25 of the largest below f16's
normal range), values and the long chunks' queries are exact, the result is rounded to the
output's type (2^-9 bf16, 2^-12 f16), all doubled for the 32-bit sums; the error of a score
enters the exponential.
"""
import math

import pytest
import torch

from paged8_oracle import PAGE, Layer, attention, f64, score_error

pytestmark = pytest.mark.gpu
INT8, FP8 = torch.int8, torch.float8_e4m3fn


def ops():
    from complexity_framework_b200.ops import paged8
    return paged8


def clean():
    from complexity_framework_b200.ops import check_errors
    check_errors(0)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def soil():
    """Leave NaN in the memory that the next workspaces are made from."""
    torch.cuda.empty_cache()
    held = [torch.full((n,), float("nan"), device="cuda") for n in [1 << 18] * 8 + [1 << 24] * 4]
    torch.cuda.synchronize()
    del held


def check(L, new, hq, io, part=None, mass=False, q=None, seed=1, q_err=0.0, **kw):
    """One call for the sequences of ``part`` (start, end; default: all); the other rows of
    ``out`` and the other tokens' masses have to stay.  ``q_err``: error of the scores beside
    those of the sums."""
    a, e = part or (0, len(new))
    cu = offsets(new)
    g = torch.Generator().manual_seed(seed)
    if q is None:
        q = (torch.randn(cu[-1], hq, L.d, generator=g) * 1.5).to(io).cuda()
    out = torch.full((cu[-1], hq, L.d), 7.0, dtype=io, device="cuda")
    m_in = m_out = None
    if mass:
        m_in = torch.rand(L.num_pages, L.hkv, PAGE, generator=g).cuda()
        m_out = torch.full_like(m_in, -7.0)
    soil()
    ops().paged8_attention(q, L.codes, L.scales, L.table[a:e], ints(cu)[a:e + 1], L.kv_lens[a:e],
                           scale=L.d ** -0.5, mass=m_in, mass_out=m_out, out=out,
                           **{"max_q_len": max(new[a:e]), **kw})
    clean()
    want, spread, weights, mag = attention(L, q, cu, L.d ** -0.5)
    top = max([float(L.values(i)[1].abs().max()) for i in range(a, e) if L.lens[i]] or [0.0])
    s_err = math.log(2) * score_error(mag) + 2.0 ** -19 + q_err
    o_err = 2.0 ** -8 if io == torch.bfloat16 else 2.0 ** -11
    tol = want.abs() * o_err + spread * (2.0 ** -10 + 2 * s_err) + top * max(L.lens) * 2.0 ** -24 \
        + 1e-30
    mine = slice(cu[a], cu[e])
    off = (f64(out) - want).abs()[mine]
    assert (off <= tol[mine]).all(), ((off / tol[mine]).max().item(), off.max().item())
    rest = torch.ones(cu[-1], dtype=torch.bool)
    rest[mine] = False
    assert (out.cpu()[rest] == 7).all()
    if mass:
        got, before = f64(m_out), f64(m_in)
        seen = torch.zeros_like(got, dtype=torch.bool)
        for i in range(a, e):
            for j in range(L.lens[i]):
                p, s = int(L.table[i, j // PAGE]), j % PAGE
                seen[p, :, s] = True
                w = weights[i][:, j]
                err = (got[p, :, s] - before[p, :, s] - w).abs()
                assert (err <= w * s_err + got[p, :, s] * 2.0 ** -23).all(), (i, j, err, w)
        assert (got[~seen] == -7).all()
    return out


# ------------------------------------------------------------- long chunks cut along the cache
@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("part", [(1, 2), (2, 3), (1, 3)])
def test_a_long_chunk_writes_its_own_rows(part, mass):
    """A prompt chunk beside a decode token and another chunk, one call for each run of
    sequences into one output; the table is wide enough for the chunk's keys to be split."""
    L = Layer([1101, 300, 90], 2, 64, INT8, "cuda", seed=3)
    check(L, [1, 300, 90], 8, torch.bfloat16, part=part, mass=mass)


@pytest.mark.parametrize("dtype,io,hq,hkv,d", [(INT8, torch.bfloat16, 8, 2, 128),
                                               (FP8, torch.float16, 14, 2, 64)])
def test_long_chunk_over_live_splits(dtype, io, hq, hkv, d):
    """Several splits with keys in each; in the shorter sequence some are empty."""
    L = Layer([2300, 600], hkv, d, dtype, "cuda", seed=5)
    check(L, [130, 77], hq, io, mass=True)


def test_prompt_beside_a_running_request():
    """A step with a decode token of 1100 cached tokens and a prompt of 300, through the pools:
    the kernels against the operators on the CPU."""
    from complexity_framework_b200.inference import Paged8Pool, SeqChunk

    torch.manual_seed(4)
    pools = [Paged8Pool(1, 2, 64, 100, dtype=torch.bfloat16, device=d, track_mass=True)
             for d in ("cuda", "cpu")]
    at = {0: 0, 1: 0}
    for step in (((0, 1100),), ((0, 1), (1, 300))):
        chunks = [SeqChunk(s, at[s], n) for s, n in step]
        N = sum(n for _, n in step)
        k, v = torch.randn(2, N, 2, 64).bfloat16()
        q = torch.randn(N, 8, 64).bfloat16()
        outs = []
        for p in pools:
            for s, _ in step:
                if s not in p.pages:
                    p.allocate_sequence(s)
            b = p.batch(chunks)
            b.write(0, k.to(p.device), v.to(p.device))
            soil()
            outs.append(b.attend(0, q.to(p.device), 0.125).float().cpu())
            b.commit()
        for s, n in step:
            at[s] += n
        # both round to bf16 (2^-8 of values below 4), the kernels also P to f16
        assert (outs[0] - outs[1]).abs().max() <= 4 * (2.0 ** -8 + 2.0 ** -10)
    clean()
    assert torch.allclose(pools[0].mass.cpu(), pools[1].mass, rtol=1e-4, atol=1e-5)


def test_engine_prompt_joins_a_running_request():
    """A request's logits do not change when a prompt joins its batch."""
    from complexity_framework_b200 import ComplexityModel, ModelConfig
    from complexity_framework_b200.inference import (GenerationConfig, InferenceConfig,
                                                     InferenceEngine)

    torch.manual_seed(0)
    m = ComplexityModel(ModelConfig(
        hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
        vocab_size=2048, intermediate_size=256, shared_intermediate_size=512, num_experts=4,
        top_k=2, max_position_embeddings=2048)).cuda().to(torch.bfloat16).eval()
    for layer in m.layers:
        layer.self_attn.o_proj.weight.data *= 16          # the attention's part of the logits
    g = torch.Generator().manual_seed(1)
    first, second = (torch.randint(0, 2048, (n,), generator=g).tolist() for n in (1100, 300))
    seen, logits = [], m.logits
    m.logits = lambda h: (seen[-1].append(logits(h)[0, 0].float()), logits(h))[1]
    for joins in (False, True):
        seen.append([])
        eng = InferenceEngine(m, InferenceConfig(max_cache_length=1536, max_batch_size=2,
                                                 kv_cache_dtype="int8", prefill_chunk_size=2048,
                                                 cuda_graph_decode=False))
        eng.add_request(first, GenerationConfig(max_new_tokens=3))
        eng.step()
        if joins:
            eng.add_request(second, GenerationConfig(max_new_tokens=1))
        soil()
        eng.step()                                         # its next token, with the prompt beside
    clean()
    # the same sums in 32 bits; the matrix products of 1 and 301 rows round to bf16 apart
    for a, b in zip(*seen):
        assert (a - b).abs().max() <= 2.0 ** -5 * a.abs().max()


# ----------------------------------------------------------- rows before a sequence's first token
@pytest.mark.parametrize("lens,new,hq,hkv", [([1], [2], 2, 2), ([3], [4], 2, 2), ([3], [4], 14, 2),
                                             ([3, 40], [4, 5], 14, 2), ([1030, 2], [1, 5], 3, 3)])
def test_weights_with_rows_before_the_first_token(lens, new, hq, hkv):
    """An odd group and an odd number of such rows: of two neighbouring rows one sees keys."""
    L = Layer(lens, hkv, 64, INT8, "cuda", seed=3)
    check(L, new, hq, torch.bfloat16, mass=True)


# -------------------------------------------------------------------- append of part of a batch
@pytest.mark.parametrize("dtype", [INT8, FP8])
@pytest.mark.parametrize("part", [(1, 4), (2, 5), (3, 4), (4, 5)])
def test_append_of_part_of_a_batch(dtype, part):
    """Uneven chunks of a call that begins past row 16: the same cache as on the CPU."""
    from complexity_framework_b200.ops import paged8

    new = [70, 1, 90, 300, 2]
    a, e = part
    cu = offsets(new)
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn(2, cu[-1], 2, 64, generator=g).bfloat16()
    caches = []
    for device in ("cuda", "cpu"):
        L = Layer([100, 40, 90, 307, 50], 2, 64, dtype, device, seed=3)
        # a first block that is not finite: codes of 0 where tokens are added, else as it was
        L.scales[int(L.table[a, 0])] = float("nan")
        mass = torch.ones(L.num_pages, 2, PAGE, device=device)
        paged8.paged8_append(k.to(device), v.to(device), L.codes, L.scales, L.table[a:e],
                             torch.tensor(cu[a:e + 1], dtype=torch.int32, device=device),
                             L.kv_lens[a:e], max_q_len=max(new[a:e]), mass=mass)
        caches.append((f64(L.codes), f64(L.scales), mass.cpu()))
    clean()
    for x, y in zip(*caches):
        assert torch.allclose(x, y, rtol=2.0 ** -22, atol=0, equal_nan=True)


# ---------------------------------------------------------------- chunks longer than max_q_len
@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("new,max_q_len,hq", [([2, 0], 1, 8), ([0, 2], 1, 8), ([7, 1], 6, 10)])
def test_short_chunk_longer_than_max_q_len_is_reported(new, max_q_len, hq, mass):
    """Also where the kernels' rows, a multiple of eight, would hold it; the tables are full."""
    from complexity_framework_b200.ops import check_errors

    L = Layer([48, 48], 2, 64, INT8, "cuda", seed=3)
    q = torch.randn(sum(new), hq, 64, device="cuda").bfloat16()
    m = torch.zeros(L.num_pages, 2, PAGE, device="cuda") if mass else None
    ops().paged8_attention(q, L.codes, L.scales, L.table, ints(offsets(new)), L.kv_lens,
                           scale=0.1, max_q_len=max_q_len, mass=m)
    with pytest.raises(RuntimeError, match="code=4 site=71"):
        check_errors(0)
    clean()


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("new,max_q_len", [([20, 1], 19), ([1, 70], 69), ([70, 70], 33)])
def test_long_chunk_longer_than_max_q_len_is_reported(new, max_q_len, mass):
    """Also within the last tile of rows."""
    from complexity_framework_b200.ops import check_errors

    L = Layer([100, 80], 2, 64, INT8, "cuda", seed=3)
    q = torch.randn(sum(new), 16, 64, device="cuda").bfloat16()
    m = torch.zeros(L.num_pages, 2, PAGE, device="cuda") if mass else None
    ops().paged8_attention(q, L.codes, L.scales, L.table, ints(offsets(new)), L.kv_lens,
                           scale=0.1, max_q_len=max_q_len, mass=m)
    with pytest.raises(RuntimeError, match="code=4 site=84"):
        check_errors(0)
    clean()


@pytest.mark.parametrize("new,max_q_len", [([2, 1], 1), ([1, 33], 32), ([100, 1, 1, 1], 99)])
def test_append_longer_than_max_q_len_is_reported(new, max_q_len):
    """Whether or not its blocks fit what the launch covers, in both enumerations."""
    from complexity_framework_b200.ops import check_errors

    L = Layer([100] * len(new), 2, 64, INT8, "cuda", seed=3)
    k = torch.randn(sum(new), 2, 64, device="cuda").bfloat16()
    ops().paged8_append(k, k, L.codes, L.scales, L.table, ints(offsets(new)), L.kv_lens,
                        max_q_len=max_q_len)
    with pytest.raises(RuntimeError, match="code=4 site=59"):
        check_errors(0)
    clean()


# ------------------------------------------------------------------------------- no new tokens
@pytest.mark.parametrize("hq", [1, 100])
@pytest.mark.parametrize("width", [4, 80])
def test_weights_pass_through_a_call_without_new_tokens(hq, width):
    L = Layer([40, 0, 17], 1, 64, INT8, "cuda", seed=3, width=width)
    q = torch.empty(0, hq, 64, dtype=torch.bfloat16, device="cuda")
    m_in = torch.rand(L.num_pages, 1, PAGE, device="cuda")
    m_out = torch.full_like(m_in, -7.0)
    out = ops().paged8_attention(q, L.codes, L.scales, L.table, ints([0] * 4), L.kv_lens,
                                 scale=1.0, max_q_len=9, mass=m_in, mass_out=m_out)
    clean()
    assert out.shape == q.shape
    want = torch.full_like(m_in, -7.0)
    for i, n in enumerate(L.lens):
        for j in range(n):
            at = int(L.table[i, j // PAGE]), 0, j % PAGE
            want[at] = m_in[at]
    assert torch.equal(m_out, want)


# ------------------------------------------------------------------------------------ workspaces
@pytest.mark.parametrize("new,limit", [(1, 8 << 20), (8, 24 << 20)])
def test_kept_scores_stay_within_the_workspace(new, limit):
    """Weights of short chunks over a table far wider than the sequences."""
    seqs = 12
    lens = [20 + 30 * i for i in range(seqs)]
    L = Layer(lens, 2, 64, INT8, "cuda", seed=3, width=4096)
    q = torch.randn(seqs * new, 8, 64, device="cuda").bfloat16()
    cu = ints(offsets([new] * seqs))
    m = torch.zeros(2, L.num_pages, 2, PAGE, device="cuda")
    outs, peak = [], []
    for i, ws in enumerate((4 << 30, limit)):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        outs.append(ops().paged8_attention(q, L.codes, L.scales, L.table, cu, L.kv_lens,
                                           scale=0.125, max_q_len=new, mass=m[i],
                                           workspace_bytes=ws))
        peak.append(torch.cuda.max_memory_allocated() - held)
    clean()
    assert peak[0] > 2 * limit and peak[1] <= limit + (1 << 20), peak   # beside the output
    # other chunks of the cache, the same sums
    assert (outs[0].float() - outs[1].float()).abs().max() < 2.0 ** -6
    assert torch.allclose(m[0], m[1], rtol=1e-4, atol=1e-6)


# ------------------------------------------------------------------------- layouts and ranges of q
@pytest.mark.parametrize("new", [[1, 3], [60, 20]])
def test_q_of_a_fused_projection(new):
    hq, hkv, d = 14, 2, 64
    L = Layer([200, 70], hkv, d, INT8, "cuda", seed=3)
    n = sum(new)
    kqv = torch.randn(n, (2 * hkv + hq) * d, device="cuda").bfloat16()
    check(L, new, hq, torch.bfloat16, q=kqv[:, hkv * d:(hkv + hq) * d].view(n, hq, d))


@pytest.mark.parametrize("new", [1, 40])
def test_zero_and_uneven_value_scales(new):
    """V blocks of zeros, and blocks whose scales lie far apart, in both attention kernels."""
    L = Layer([200, 100], 2, 64, INT8, "cuda", seed=9)
    L.scales[::3, :, 1] = 0
    L.scales[1::3, :, 1] *= 1e-4
    L.codes[::3, :, 1] = 0
    check(L, [new, new], 8, torch.bfloat16, mass=True)


@pytest.mark.parametrize("new", [1, 40])
def test_q_elements_far_apart(new):
    """Short chunks hold q in f16 scaled by the row's largest element: elements more than 2^17
    below it lose bits, at most 2^-25 of the largest each; small codes beside the offset of
    128 that int8 codes carry through the score's sum."""
    L = Layer([150, 70], 2, 64, INT8, "cuda", seed=9)
    L.codes[..., 0, :, :] //= 32
    q = torch.randn(2 * new, 8, 64) * 2.0 ** -21
    q[..., 5] = 1.0
    k = torch.cat([L.values(i)[0].reshape(-1, 64) for i in range(2)])
    lost = 2.0 ** -25 * k.abs().sum(-1).max().item() / 8
    offset = 128 * L.scales.max().item() * q.abs().sum(-1).max().item() / 8
    check(L, [new, new], 8, torch.bfloat16, q=q.bfloat16().cuda(), mass=True,
          q_err=lost + math.log(2) * score_error(offset))


@pytest.mark.parametrize("new", [[1, 3], [60, 20]])
def test_expanded_q(new):
    """One row for all tokens: strides that no TMA map may have."""
    L = Layer([200, 70], 2, 64, INT8, "cuda", seed=3)
    q = torch.randn(1, 14, 64, device="cuda").bfloat16().expand(sum(new), 14, 64)
    check(L, new, 14, torch.bfloat16, q=q)


@pytest.mark.parametrize("heads", [1, 8])
def test_nan_rows_weigh_the_tokens_they_see_only(heads):
    """In both attention kernels."""
    L = Layer([40], 1, 64, INT8, "cuda", seed=2)
    q = torch.randn(20, heads, 64, device="cuda").bfloat16()
    m = torch.zeros(2, L.num_pages, 1, PAGE, device="cuda")
    outs = []
    for i in range(2):
        outs.append(ops().paged8_attention(q, L.codes, L.scales, L.table, ints([0, 20]), L.kv_lens,
                                           scale=0.125, max_q_len=20, mass=m[i]))
        q[3] = float("nan")                                 # at position 23
    clean()
    rows = torch.tensor([t != 3 for t in range(20)], device="cuda")
    assert torch.equal(outs[0][rows], outs[1][rows]) and torch.isnan(outs[1][3]).all()
    clear, nan = (x[L.table[0].long(), 0].reshape(-1)[:40] for x in m)
    assert torch.isnan(nan[:24]).all() and torch.equal(clear[24:], nan[24:])
