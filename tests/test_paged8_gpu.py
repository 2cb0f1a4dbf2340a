"""8-bit paged KV cache kernels against 64-bit oracles (tests/paged8_oracle.py).

Tolerances.  Scales: one fp32 division.  Codes: half a code step, plus what an fp32
reciprocal and product move a value by.  Attention: the probabilities are rounded to f16 in
decode and short chunks (2^-11 of each, and 2^-25 of the largest below f16's normal range),
and probabilities and values to bf16 in long chunks (2^-9 each); the result is rounded to the
output type (2^-9 bf16, 2^-12 f16).  Weights: the error of a score enters the exponential.
"""
import math

import pytest
import torch

from paged8_oracle import LEVELS, PAGE, Layer, attention, f64, half_ulp, keep_order, score_error

pytestmark = pytest.mark.gpu
INT8, FP8 = torch.int8, torch.float8_e4m3fn


def ops():
    from complexity_framework_b200.ops import paged8
    return paged8


def clean():
    from complexity_framework_b200.ops import check_errors
    check_errors(0)


def check_codes(codes, want, dtype, what=""):
    """codes: 64-bit values of the stored codes; want: real numbers they should be nearest to."""
    slack = LEVELS[dtype] * 2.0 ** -21
    off = (codes - want).abs() - half_ulp(torch.maximum(codes.abs(), want.abs()), dtype)
    assert off.max().item() <= slack, (what, off.max().item())


# ------------------------------------------------------------------------------ append
APPEND = [
    # (lens after the append, new tokens of each)
    ([1], [1]),
    ([16, 17, 1, 0, 33], [1, 1, 1, 1, 1]),                 # block starts, a first token, padding
    ([40, 7, 100], [19, 7, 3]),                            # chunks that begin and end inside a block
    ([300, 5, 16, 64], [257, 1, 16, 48]),                  # uneven: one long chunk among short ones
    ([2000], [1999]),
]


@pytest.mark.parametrize("lens,new", APPEND)
@pytest.mark.parametrize("dtype", [INT8, FP8])
@pytest.mark.parametrize("hkv,d,io", [(2, 64, torch.bfloat16), (8, 128, torch.float16),
                                      (1, 128, torch.bfloat16)])
def test_append(lens, new, dtype, hkv, d, io):
    L = Layer(lens, hkv, d, dtype, "cuda", seed=3)
    before, s_before = f64(L.codes), f64(L.scales)
    g = torch.Generator().manual_seed(5)
    N = sum(new)
    k = (torch.randn(N, hkv, d, generator=g) * torch.logspace(-2, 2, N)[:, None, None]).to(io)
    v = torch.randn(N, hkv, d, generator=g).to(io)
    v[N // 2] = 0
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    ops().paged8_append(k.cuda(), v.cuda(), L.codes, L.scales, L.table,
                        torch.tensor(cu, dtype=torch.int32, device="cuda"), L.kv_lens,
                        max_q_len=max(new))
    clean()
    after, s_after = f64(L.codes), f64(L.scales)
    touched = set()
    for i, n in enumerate(lens):
        start = n - new[i]
        for b in range(max(start, 0) // PAGE, -(-n // PAGE)):
            page = int(L.table[i, b])
            touched.add(page)
            lo, hi = max(start, b * PAGE), min(n, (b + 1) * PAGE)
            rows = slice(cu[i] + lo - start, cu[i] + hi - start)
            x = torch.stack((f64(k[rows]), f64(v[rows]))).permute(2, 0, 1, 3)
            older = lo - b * PAGE
            s = x.abs().amax((-1, -2)) / LEVELS[dtype]
            if older:
                s = torch.maximum(s, s_before[page])
            assert torch.allclose(s_after[page], s, rtol=2.0 ** -23, atol=0)
            div = torch.where(s > 0, s, 1.0)[..., None, None]
            check_codes(after[page][:, :, older:older + hi - lo], x / div, dtype, (i, b))
            if older:
                want = before[page][:, :, :older] * (s_before[page][..., None, None] / div)
                check_codes(after[page][:, :, :older], want, dtype, (i, b, "older"))
            assert torch.equal(after[page][:, :, older + hi - lo:],
                               before[page][:, :, older + hi - lo:])
    rest = [p for p in range(L.num_pages) if p not in touched]
    assert torch.equal(after[rest], before[rest]) and torch.equal(s_after[rest], s_before[rest])


@pytest.mark.parametrize("dtype", [INT8, FP8])
def test_append_strided_rows_and_steps(dtype):
    """k and v as slices of one fused projection, appended token by token: the same cache as
    from dense copies."""
    hkv, d, hq, n = 2, 64, 4, 37
    kqv = torch.randn(n, (2 * hkv + hq) * d, device="cuda").bfloat16()
    k = kqv[:, :hkv * d].view(n, hkv, d)
    v = kqv[:, (hkv + hq) * d:].view(n, hkv, d)
    got = []
    for dense in (False, True):
        L = Layer([n], hkv, d, dtype, "cuda", fill=False)
        for t in range(n):
            a, b = k[t:t + 1], v[t:t + 1]
            if dense:
                a, b = a.contiguous().clone(), b.contiguous().clone()
            ops().paged8_append(a, b, L.codes, L.scales, L.table,
                                torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                                torch.tensor([t + 1], dtype=torch.int32, device="cuda"),
                                max_q_len=1)
        got.append((f64(L.codes), f64(L.scales), L))
    clean()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    x = got[0][2].values(0)
    want = torch.stack((f64(k), f64(v))).transpose(1, 2)
    # a token is rounded once, and again at most once for each growth of its block's scale
    top = f64(got[0][2].scales).max() * LEVELS[dtype]
    step = top / 127 / 2 if dtype == INT8 else top * 2.0 ** -4
    assert (x - want).abs().max() <= 16 * step


def test_append_resets_the_new_tokens_mass():
    L = Layer([20, 0, 33], 2, 64, INT8, "cuda", seed=3)
    mass = torch.ones(L.num_pages, 2, PAGE, device="cuda")
    k = torch.randn(10, 2, 64, device="cuda").bfloat16()
    ops().paged8_append(k, k, L.codes, L.scales, L.table,
                        torch.tensor([0, 6, 7, 10], dtype=torch.int32, device="cuda"), L.kv_lens,
                        max_q_len=6, mass=mass)
    clean()
    want = torch.ones(L.num_pages, 2, PAGE)
    for i, (lo, hi) in {0: (14, 20), 2: (30, 33)}.items():
        for j in range(lo, hi):
            want[int(L.table[i, j // PAGE]), :, j % PAGE] = 0
    assert torch.equal(mass.cpu(), want)


def test_append_extremes():
    """Zero blocks, subnormal magnitudes, infinities and NaN: other blocks are untouched."""
    hkv, d = 2, 64
    for dtype in (INT8, FP8):
        L = Layer([64], hkv, d, dtype, "cuda", fill=False)
        k = torch.randn(64, hkv, d, device="cuda").bfloat16()
        v = torch.zeros_like(k)
        k[0:16] = 0
        k[16:32, 0] = 1e-39
        k[33, 0, 5] = float("inf")
        k[34, 1, 7] = float("nan")
        ops().paged8_append(k, v, L.codes, L.scales, L.table,
                            torch.tensor([0, 64], dtype=torch.int32, device="cuda"), L.kv_lens,
                            max_q_len=64)
        clean()
        x = L.values(0)
        assert (x[0, :, :16] == 0).all() and (x[1] == 0).all()
        want = f64(k[16:32, 0])
        # the codes resolve 1/448 (1/127) of the block's magnitude; the scale is subnormal
        assert (x[0, 0, 16:32] - want).abs().max() <= want.abs().max() * 2.0 ** -4
        assert not torch.isfinite(x[0, 0, 32:48]).all() and not torch.isfinite(x[0, 1, 32:48]).any()
        assert torch.isfinite(x[0, :, 48:]).all() and torch.isfinite(x[0, 1, 16:32]).all()


# -------------------------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", [INT8, FP8])
@pytest.mark.parametrize("hkv,d,io,layers", [(2, 64, torch.bfloat16, None),
                                             (3, 128, torch.float16, 3)])
def test_read(dtype, hkv, d, io, layers):
    lens = [1, 0, 16, 53]
    L = Layer(lens, hkv, d, dtype, "cuda", layers=layers, width=5)
    k, v = ops().paged8_read(L.codes, L.scales, L.table, L.kv_lens, dtype=io)
    clean()
    for lay in range(layers or 1):
        for i, n in enumerate(lens):
            want = L.values(i, layer=lay if layers else None)
            for x, got in zip(want, (k, v)):
                got = got[lay, i] if layers else got[i]
                assert torch.equal(got[:, :n].cpu(), x.float().to(io))  # the product fits 32 bits
                assert (got[:, n:] == 0).all()


# --------------------------------------------------------------------------- attention
def run_attention(lens, new, hq, hkv, d, dtype, io, seed=0, mass=False, width=None, qscale=1.5,
                  layer=None):
    L = layer or Layer(lens, hkv, d, dtype, "cuda", seed=seed, width=width)
    g = torch.Generator().manual_seed(seed + 1)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = (torch.randn(cu[-1], hq, d, generator=g) * qscale).to(io)
    m_in = m_out = None
    if mass:
        m_in = torch.rand(L.num_pages, hkv, PAGE, generator=g).cuda()
        m_out = torch.full_like(m_in, -7.0)
    out = ops().paged8_attention(q.cuda(), L.codes, L.scales, L.table,
                                 torch.tensor(cu, dtype=torch.int32, device="cuda"), L.kv_lens,
                                 scale=d ** -0.5, max_q_len=max(new), mass=m_in, mass_out=m_out)
    clean()
    want, spread, weights, mag = attention(L, q, cu, d ** -0.5)
    rows = max(new) * (hq // hkv)
    p_err = 2.0 ** -10 if rows <= 16 else 2.0 ** -8
    top = max([float(L.values(i)[1].abs().max()) for i, n in enumerate(lens) if n] or [0.0])
    s_err = math.log(2) * score_error(mag) + 2.0 ** -19
    o_err = 2.0 ** -8 if io == torch.bfloat16 else 2.0 ** -11
    tol = want.abs() * o_err + spread * (p_err + 2 * s_err) + top * max(lens) * 2.0 ** -24 + 1e-30
    off = (f64(out) - want).abs()
    assert (off <= tol).all(), ((off / tol).max().item(), off.max().item())
    if mass:
        m_out, m_in = f64(m_out), f64(m_in)
        seen = torch.zeros_like(m_out, dtype=torch.bool)
        for i, n in enumerate(lens):
            for j in range(n):
                p, s = int(L.table[i, j // PAGE]), j % PAGE
                seen[p, :, s] = True
                w = weights[i][:, j]
                err = (m_out[p, :, s] - m_in[p, :, s] - w).abs()
                assert (err <= w * s_err + m_out[p, :, s] * 2.0 ** -23).all(), (i, j, err, w)
        assert (m_out[~seen] == -7).all()
    return out


DECODE = [
    ([1], 4, 2, 64), ([15, 16, 17, 0, 31], 8, 8, 128), ([700, 1, 333, 129], 32, 8, 128),
    ([257, 64], 14, 2, 64), ([90, 260], 8, 1, 128), ([130], 10, 1, 64), ([200, 5], 16, 1, 128),
    ([45], 24, 1, 64), ([70, 33], 80, 2, 64), ([1000, 1, 40], 33, 1, 128),
]


@pytest.mark.parametrize("lens,hq,hkv,d", DECODE)
@pytest.mark.parametrize("dtype,io", [(INT8, torch.bfloat16), (FP8, torch.bfloat16),
                                      (INT8, torch.float16), (FP8, torch.float16)])
def test_decode(lens, hq, hkv, d, dtype, io):
    run_attention(lens, [1] * len(lens), hq, hkv, d, dtype, io, mass=io == torch.bfloat16)


def test_sequences_without_new_tokens():
    """They have no rows; their weights pass through.  Table widths of both work splits."""
    for width in (8, 200):
        for new in ([1, 0, 2], [0, 100, 0]):
            run_attention([100, 37, 120], new, 4, 2, 64, INT8, torch.bfloat16, mass=True,
                          width=width)


def test_many_sequences():
    """More sequences than one pass of the work split's sums takes, uneven ones among them."""
    lens = [(7 * i) % 50 for i in range(300)]
    run_attention(lens, [1] * 300, 2, 1, 64, INT8, torch.bfloat16, mass=True, width=60)
    run_attention(lens, [3] * 300, 2, 1, 64, FP8, torch.bfloat16, width=4)


def test_decode_long_split():
    """Many splits, page-table rows wider than the sequences, more than 32 pages a warp."""
    run_attention([9000, 70, 3100], [1, 1, 1], 4, 1, 128, INT8, torch.bfloat16, mass=True,
                  width=1000)
    run_attention([9001] * 40, [1] * 40, 4, 4, 64, FP8, torch.bfloat16, width=563)
    run_attention([5000, 0, 900, 2111], [5, 1, 7, 3], 8, 2, 128, INT8, torch.bfloat16, mass=True,
                  width=400)


CHUNKS = [
    ([40, 7], [5, 2], 8, 2, 64), ([16, 33, 1], [16, 17, 1], 4, 4, 128),
    ([300, 129, 20], [65, 129, 1], 8, 2, 128), ([150], [37], 14, 2, 64),
    ([500], [200], 16, 1, 64), ([3, 200], [5, 100], 4, 2, 128),   # two rows before the first token
    ([400, 0], [130, 4], 4, 1, 128),
]


@pytest.mark.parametrize("lens,new,hq,hkv,d", CHUNKS)
@pytest.mark.parametrize("dtype,io", [(INT8, torch.bfloat16), (FP8, torch.float16)])
@pytest.mark.parametrize("mass", [False, True])
def test_chunks(lens, new, hq, hkv, d, dtype, io, mass):
    run_attention(lens, new, hq, hkv, d, dtype, io, mass=mass, seed=4)


def test_chunk_in_parts():
    """A workspace too small for all sequences: they are expanded one after another."""
    L = Layer([300, 129, 200], 2, 64, INT8, "cuda", seed=1)
    cu = torch.tensor([0, 100, 150, 350], dtype=torch.int32, device="cuda")
    q = torch.randn(350, 8, 64, device="cuda").bfloat16()
    m = torch.zeros(2, L.num_pages, 2, PAGE, device="cuda")
    outs = [ops().paged8_attention(q, L.codes, L.scales, L.table, cu, L.kv_lens, scale=0.125,
                                   max_q_len=200, mass=m[i], workspace_bytes=ws)
            for i, ws in enumerate((4 << 30, 1))]
    clean()
    assert (outs[0].float() - outs[1].float()).abs().max() < 2.0 ** -6  # other splits, same sums
    assert torch.allclose(m[0], m[1], rtol=1e-4, atol=1e-6)


def test_peaked_and_large_scores():
    """Scores far apart (one key takes all the weight), large and tiny q: no overflow."""
    for qs in (100.0, 1e-6, 2e4):
        run_attention([333, 20], [1, 1], 4, 2, 64, INT8, torch.bfloat16, qscale=qs, mass=True)
    run_attention([333, 200], [60, 100], 4, 2, 64, FP8, torch.bfloat16, qscale=30.0, mass=True)


def test_zero_and_uneven_value_scales():
    """V blocks of zeros, and blocks whose scales lie far apart, keep their softmax weight."""
    L = Layer([200, 100], 2, 64, INT8, "cuda", seed=9)
    s = L.scales.clone()
    s[::3, :, 1] = 0
    s[1::3, :, 1] *= 1e-4
    L.codes[::3, :, 1] = 0
    L.scales.copy_(s)
    run_attention([200, 100], [1, 1], 8, 2, 64, INT8, torch.bfloat16, layer=L, mass=True)


def test_unwritten_tail_is_not_read():
    """Codes past a sequence's last token are NaN: no output sees them."""
    for new in (1, 40):
        L = Layer([50, 83], 2, 128, FP8, "cuda", seed=2)
        for i, n in enumerate(L.lens):
            page = int(L.table[i, n // PAGE])
            L.codes.view(torch.uint8)[page, :, :, n % PAGE:] = 0x7F
        run_attention([50, 83], [new, new], 8, 2, 128, FP8, torch.bfloat16, layer=L, mass=True)


def test_zero_key_blocks():
    """Blocks of zero keys (scale 0), one of them the last and partly empty."""
    for new in (1, 70):
        L = Layer([100], 2, 64, INT8, "cuda", seed=9)
        for b in (1, 6):
            L.scales[int(L.table[0, b]), :, 0] = 0
            L.codes[int(L.table[0, b]), :, 0] = 0
        run_attention([100], [new], 4, 2, 64, INT8, torch.bfloat16, layer=L, mass=True)


@pytest.mark.parametrize("heads", [1, 8])
def test_later_nan_block_is_masked(heads):
    """A block that is not finite is seen by the rows at or after it only."""
    for dtype in (INT8, FP8):
        L = Layer([64], 1, 64, dtype, "cuda", seed=2)
        q = torch.randn(20, heads, 64, device="cuda").bfloat16()
        args = (torch.tensor([0, 20], dtype=torch.int32, device="cuda"), L.kv_lens)
        good = ops().paged8_attention(q, L.codes, L.scales, L.table, *args, scale=0.125,
                                      max_q_len=20)
        L.scales[int(L.table[0, 3])] = float("nan")
        L.codes[int(L.table[0, 3])] = 0
        bad = ops().paged8_attention(q, L.codes, L.scales, L.table, *args, scale=0.125,
                                     max_q_len=20)
        clean()
        assert torch.equal(good[:4], bad[:4])        # positions 44 .. 47 see blocks 0 .. 2
        assert torch.isnan(bad[4:].float()).all()


def test_in_place_mass_strided_q_and_repeatability():
    L = Layer([70, 130], 2, 64, INT8, "cuda", seed=1)
    kqv = torch.randn(2, (4 + 8) * 64, device="cuda").bfloat16()
    q = kqv[:, 128:128 + 512].view(2, 8, 64)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    m0 = torch.rand(L.num_pages, 2, PAGE, device="cuda")
    a, b = m0.clone(), m0.clone()
    o1 = ops().paged8_attention(q, L.codes, L.scales, L.table, cu, L.kv_lens, scale=0.125,
                                max_q_len=1, mass=a)
    o2 = ops().paged8_attention(q.contiguous(), L.codes, L.scales, L.table, cu, L.kv_lens,
                                scale=0.125, max_q_len=1, mass=m0, mass_out=b)
    o3 = ops().paged8_attention(q, L.codes, L.scales, L.table, cu, L.kv_lens, scale=0.125,
                                max_q_len=1)
    clean()
    assert torch.equal(o1, o2) and torch.equal(a, b)
    assert torch.equal(o1, o3)


def test_other_stream():
    L = Layer([300, 40], 2, 64, INT8, "cuda", seed=1)
    q = torch.randn(2, 8, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    call = lambda: ops().paged8_attention(q, L.codes, L.scales, L.table, cu, L.kv_lens,  # noqa: E731
                                          scale=0.125, max_q_len=1)
    want = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_offsets_past_32_bits():
    """Pages whose codes lie beyond 2^31 and 2^32 bytes of the pool."""
    hkv, d = 8, 128
    pages = (9 << 29) // (hkv * 2 * PAGE * d)                  # 4.8e9 bytes
    codes = torch.zeros(pages, hkv, 2, PAGE, d, dtype=torch.int8, device="cuda")
    scales = torch.zeros(pages, hkv, 2, device="cuda")
    small = Layer([40], hkv, d, INT8, "cuda", seed=3)
    big_table = torch.tensor([[pages - 1, pages // 2 + 3, pages - 7]], dtype=torch.int32,
                             device="cuda")
    t = small.table[0].long()
    codes[big_table[0].long()] = small.codes[t]
    scales[big_table[0].long()] = small.scales[t]
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 32, d, device="cuda").bfloat16()
    k, v = torch.randn(2, 1, hkv, d, device="cuda").bfloat16()
    for c, s, tb in ((small.codes, small.scales, small.table), (codes, scales, big_table)):
        ops().paged8_append(k, v, c, s, tb, cu, small.kv_lens, max_q_len=1)
    a = ops().paged8_attention(q, small.codes, small.scales, small.table, cu, small.kv_lens,
                               scale=0.1, max_q_len=1)
    b = ops().paged8_attention(q, codes, scales, big_table, cu, small.kv_lens, scale=0.1,
                               max_q_len=1)
    ra = ops().paged8_read(small.codes, small.scales, small.table, small.kv_lens)
    rb = ops().paged8_read(codes, scales, big_table, small.kv_lens)
    clean()
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(ra, rb))


# ------------------------------------------------------------------------------- evict
EVICT = [
    ([100], 50, 10), ([33, 16, 1, 0, 200], 32, 8), ([70, 90], 45, 0), ([70, 90], 45, 45),
    ([300], 1, 0), ([300, 20], 17, 3), ([1500, 4096], 777, 100),
]


@pytest.mark.parametrize("lens,budget,recent", EVICT)
@pytest.mark.parametrize("dtype,hkv,d,layers", [(INT8, 2, 64, None), (FP8, 3, 128, 2)])
def test_evict(lens, budget, recent, dtype, hkv, d, layers):
    kept = [min(n, budget) for n in lens]
    extra = sum(-(-n // PAGE) for n in kept) + 2
    L = Layer(lens, hkv, d, dtype, "cuda", extra_pages=extra, layers=layers, seed=6)
    lead = (layers,) if layers else ()
    g = torch.Generator().manual_seed(8)
    mass = torch.rand(*lead, L.num_pages, hkv, PAGE, generator=g).pow(4)
    mass = torch.where(mass < 0.05, torch.zeros_like(mass), (mass * 64).round() / 64)  # many ties
    width = max(1, max(-(-n // PAGE) for n in kept))
    dst, at = torch.zeros(len(lens), width, dtype=torch.int32), 0
    for i, n in enumerate(kept):
        b = -(-n // PAGE)
        dst[i, :b] = torch.tensor(L.spare[at:at + b], dtype=torch.int32)
        at += b
    mass_d = mass.cuda()
    old_codes, old_scales = f64(L.codes), f64(L.scales)
    keep = ops().paged8_evict(L.codes, L.scales, mass_d, L.table, L.kv_lens, dst.cuda(),
                              budget=budget, recent=recent).cpu()
    clean()
    new_codes, new_scales, new_mass = f64(L.codes), f64(L.scales), mass_d.cpu()
    if not layers:
        old_codes, old_scales, new_codes, new_scales, new_mass, mass, keep = (
            x[None] for x in (old_codes, old_scales, new_codes, new_scales, new_mass, mass, keep))
    for lay in range(layers or 1):
        for i, n in enumerate(lens):
            pages = L.table[i, :-(-n // PAGE)].long().cpu()
            for h in range(hkv):
                m = mass[lay][pages][:, h].reshape(-1)[:n].tolist()
                idx = keep_order(m, budget, recent)
                assert keep[lay, i, h, :len(idx)].tolist() == idx
                assert (keep[lay, i, h, len(idx):] == -1).all()
                for b in range(-(-len(idx) // PAGE)):
                    js = torch.tensor(idx[b * PAGE:(b + 1) * PAGE])
                    to = int(dst[i, b])
                    s_old = old_scales[lay, pages[js // PAGE], h]              # [n, 2]
                    s = s_old.amax(0)
                    assert torch.equal(new_scales[lay, to, h], s)
                    c_old = old_codes[lay, pages[js // PAGE], h, :, js % PAGE]  # [n, 2, D]
                    want = (c_old * (s_old / s)[..., None]).transpose(0, 1)
                    got = new_codes[lay, to, h]
                    check_codes(got[:, :len(js)], want, dtype, (i, h, b))
                    same = s_old == s
                    for x in range(2):
                        assert torch.equal(got[x, :len(js)][same[:, x]], c_old[:, x][same[:, x]])
                    assert (got[:, len(js):] == 0).all()
                    assert torch.equal(new_mass[lay, to, h, :len(js)],
                                       torch.tensor([m[j] for j in js.tolist()]))
                    assert (new_mass[lay, to, h, len(js):] == 0).all()
    # the old pages stay as they were
    old_pages = torch.unique(torch.cat([L.table[i, :-(-n // PAGE)] for i, n in enumerate(lens)])).long().cpu()
    assert torch.equal(new_codes[:, old_pages], old_codes[:, old_pages])


def test_evict_row_longer_than_shared_memory():
    """More tokens than the selection keeps in shared memory."""
    n, budget, recent = 50001, 1000, 77
    L = Layer([n], 1, 64, INT8, "cuda", extra_pages=80, seed=1)
    mass = torch.rand(L.num_pages, 1, PAGE)
    dst = torch.tensor([L.spare[:63]], dtype=torch.int32, device="cuda")
    keep = ops().paged8_evict(L.codes, L.scales, mass.cuda(), L.table, L.kv_lens, dst,
                              budget=budget, recent=recent)
    clean()
    m = mass[L.table[0].long().cpu()].reshape(-1)[:n].tolist()
    assert keep[0, 0].tolist() == keep_order(m, budget, recent)


def test_decode_after_evict_matches_kept_tokens():
    """Attention over the evicted cache is attention over the kept tokens."""
    lens, budget, recent, hkv, d = [100, 40], 48, 16, 2, 64
    L = Layer(lens, hkv, d, INT8, "cuda", extra_pages=10, seed=6)
    mass = torch.rand(L.num_pages, hkv, PAGE, device="cuda")
    dst = torch.tensor([L.spare[0:3], L.spare[3:6]], dtype=torch.int32, device="cuda")
    ops().paged8_evict(L.codes, L.scales, mass, L.table, L.kv_lens, dst, budget=budget,
                       recent=recent)
    L.lens, L.table = [48, 40], dst
    L.kv_lens = torch.tensor(L.lens, dtype=torch.int32, device="cuda")
    run_attention(L.lens, [1, 1], 8, hkv, d, INT8, torch.bfloat16, layer=L, mass=True)


# --------------------------------------------------------------------- refusals, reports
def test_refusals():
    p8 = ops()
    L = Layer([40, 20], 2, 64, INT8, "cuda")
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 8, 64, device="cuda").bfloat16()
    k = torch.randn(2, 2, 64, device="cuda").bfloat16()
    at = lambda q=q, codes=L.codes, scales=L.scales, table=L.table, cu=cu, lens=L.kv_lens, **kw: (  # noqa: E731
        p8.paged8_attention(q, codes, scales, table, cu, lens,
                            **{"scale": 1.0, "max_q_len": 1, **kw}))
    at()
    bad = [lambda: at(q=q.float()), lambda: at(q=q[:, :7]), lambda: at(q=q[..., :32]),
           lambda: at(q=q.cpu()), lambda: at(codes=L.codes.float()),
           lambda: at(codes=L.codes[:, :, :, :8]), lambda: at(scales=L.scales.half()),
           lambda: at(scales=L.scales[:-1]), lambda: at(table=L.table.long()),
           lambda: at(table=L.table[:1]), lambda: at(cu=cu[:2]), lambda: at(lens=L.kv_lens.cpu()),
           lambda: at(max_q_len=0), lambda: at(scale=0.0), lambda: at(scale=float("nan")), lambda: at(mass=torch.zeros(1, 2, 16, device="cuda")),
           lambda: at(out=torch.empty_like(q, dtype=torch.float16)),
           lambda: p8.paged8_append(k, k[:1], L.codes, L.scales, L.table, cu, L.kv_lens,
                                    max_q_len=1),
           lambda: p8.paged8_append(k[:, :1], k[:, :1], L.codes, L.scales, L.table, cu, L.kv_lens,
                                    max_q_len=1),
           lambda: p8.paged8_read(L.codes, L.scales, L.table, L.kv_lens, dtype=torch.float32),
           lambda: p8.paged8_evict(L.codes, L.scales,
                                   torch.zeros(L.num_pages, 2, 16, device="cuda"), L.table,
                                   L.kv_lens, L.table[:1], budget=8, recent=2)]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(ValueError):
        at(mass_out=torch.zeros(L.num_pages, 2, 16, device="cuda"))
    with pytest.raises(ValueError):
        p8.paged8_evict(L.codes, L.scales, torch.zeros(L.num_pages, 2, 16, device="cuda"), L.table,
                        L.kv_lens, L.table, budget=8, recent=9)
    with pytest.raises(RuntimeError):
        at(q=q.clone().requires_grad_())
    odd = Layer([40], 2, 96, INT8, "cuda")
    with pytest.raises(RuntimeError):
        p8.paged8_read(odd.codes, odd.scales, odd.table, odd.kv_lens)
    clean()


def test_device_side_reports():
    """A page outside the pool, a length past the table and a chunk past max_q_len are
    reported, not followed: the kernels check them before any access."""
    from complexity_framework_b200.ops import check_errors

    p8 = ops()
    q = torch.randn(2, 8, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for what in ("page", "length", "chunk"):
        L = Layer([40, 20], 2, 64, INT8, "cuda")
        c = cu
        if what == "page":
            L.table[0, 1] = L.num_pages + 5
        elif what == "length":
            L.kv_lens[1] = 49
        else:
            L.kv_lens[0], c = 40, torch.tensor([0, 2, 2], dtype=torch.int32, device="cuda")
        heads = 8 if what != "chunk" else 16
        qq = q if heads == 8 else torch.randn(2, 16, 64, device="cuda").bfloat16()
        p8.paged8_attention(qq, L.codes, L.scales, L.table, c, L.kv_lens, scale=1.0, max_q_len=1)
        with pytest.raises(RuntimeError, match="code=4"):
            check_errors(0)
    check_errors(0)
