"""The 8-bit paged KV cache operators on the CPU against 64-bit oracles."""
import pytest
import torch

from paged8_oracle import LEVELS, PAGE, Layer, attention, f64, half_ulp, keep_order

from complexity_framework_b200.ops import paged8

INT8, FP8 = torch.int8, torch.float8_e4m3fn


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [INT8, FP8])
def test_append_read_round_trip(dtype):
    hkv, d, n = 2, 24, 37
    L = Layer([n, 0], hkv, d, dtype, "cpu", fill=False, width=3)
    k, v = torch.randn(2, n, hkv, d)
    k[16:32] = 0
    for a, b in ((0, 5), (5, 6), (6, 37)):       # a chunk, a token, a chunk over two blocks
        paged8.paged8_append(k[a:b], v[a:b], L.codes, L.scales, L.table, ints([0, b - a, b - a]),
                             ints([b, 0]), max_q_len=b - a)
    got = paged8.paged8_read(L.codes, L.scales, L.table, L.kv_lens, dtype=torch.float32)
    for x, y in zip((k, v), got):
        assert (y[0, :, n:] == 0).all() and (y[1] == 0).all()
        top = x.abs().max().item()
        # at most two growths of a block's scale: three roundings
        step = top / 127 / 2 if dtype == INT8 else top * 2.0 ** -4
        assert (y[0, :, :n] - x.transpose(0, 1)).abs().max() <= 3 * step
    assert (got[0][0, :, 16:32] == 0).all()


@pytest.mark.parametrize("lens,new", [([1, 0, 33], [1, 1, 1]), ([40, 5], [7, 5]), ([3], [5])])
def test_attention_and_mass(lens, new):
    L = Layer(lens, 2, 16, INT8, "cpu")
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], 6, 16)
    mass = torch.rand(L.num_pages, 2, PAGE)
    before = mass.clone()
    out = paged8.paged8_attention(q, L.codes, L.scales, L.table, ints(cu), L.kv_lens, scale=0.25,
                                  max_q_len=max(new), mass=mass)
    want, _, weights, _ = attention(L, q, cu, 0.25)
    assert (f64(out) - want).abs().max() < 1e-4       # 32-bit sums of values below 4
    for i, n in enumerate(lens):
        for j in range(n):
            p = int(L.table[i, j // PAGE])
            got = (mass - before)[p, :, j % PAGE].double()
            assert (got - weights[i][:, j]).abs().max() < 1e-5


@pytest.mark.parametrize("dtype,layers", [(INT8, None), (FP8, 2)])
def test_evict(dtype, layers):
    lens, budget, recent = [50, 16, 3], 20, 4
    L = Layer(lens, 2, 8, dtype, "cpu", extra_pages=6, layers=layers)
    lead = (layers,) if layers else ()
    mass = (torch.rand(*lead, L.num_pages, 2, PAGE) * 8).round()
    old = [x.clone() for x in (L.codes, L.scales, mass)]
    dst = ints([[L.spare[0], L.spare[1]], [L.spare[2], 0], [L.spare[3], 0]])
    keep = paged8.paged8_evict(L.codes, L.scales, mass, L.table, L.kv_lens, dst, budget=budget,
                               recent=recent)
    for lay in range(layers or 1):
        pick = (lambda t: t[lay]) if layers else (lambda t: t)
        for i, n in enumerate(lens):
            pages = L.table[i, :-(-n // PAGE)].long()
            for h in range(2):
                idx = keep_order(pick(old[2])[pages][:, h].reshape(-1)[:n].tolist(), budget, recent)
                assert pick(keep)[i, h].tolist() == idx + [-1] * (budget - len(idx))
                for at, j in enumerate(idx):
                    page, to = pages[j // PAGE], dst[i, at // PAGE]
                    was = f64(pick(old[0])[page, h, :, j % PAGE])
                    ratio = (pick(old[1])[page, h] / pick(L.scales)[to, h]).double()[:, None]
                    now = f64(pick(L.codes)[to, h, :, at % PAGE])
                    slack = half_ulp(torch.maximum(now.abs(), (was * ratio).abs()), dtype)
                    assert ((now - was * ratio).abs() <= slack + LEVELS[dtype] * 2.0 ** -21).all()
                    assert pick(mass)[to, h, at % PAGE] == pick(old[2])[page, h, j % PAGE]


def test_refusals():
    L = Layer([20], 2, 16, INT8, "cpu")
    q = torch.randn(1, 4, 16)
    with pytest.raises(ValueError):
        paged8.paged8_attention(q[:, :3], L.codes, L.scales, L.table, ints([0, 1]), L.kv_lens,
                                scale=1.0, max_q_len=1)
    with pytest.raises(ValueError):
        paged8.paged8_attention(q, L.codes.float(), L.scales, L.table, ints([0, 1]), L.kv_lens,
                                scale=1.0, max_q_len=1)
    with pytest.raises(ValueError):
        paged8.paged8_attention(q, L.codes, L.scales, L.table, ints([0, 1]), L.kv_lens, scale=1.0,
                                max_q_len=1, mass_out=torch.zeros(1))
    with pytest.raises(ValueError):
        paged8.paged8_append(q, q[:, :2], L.codes, L.scales, L.table, ints([0, 1]), L.kv_lens,
                             max_q_len=1)
    with pytest.raises(ValueError):
        paged8.paged8_evict(L.codes, L.scales, torch.zeros(L.num_pages, 2, PAGE), L.table, L.kv_lens,
                            L.table, budget=0, recent=0)
    with pytest.raises(RuntimeError):
        paged8.paged8_attention(q.clone().requires_grad_(), L.codes, L.scales, L.table,
                                ints([0, 1]), L.kv_lens, scale=1.0, max_q_len=1)
