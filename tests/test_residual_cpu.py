"""The residual join and counter-based dropout on the CPU: formulas, generator, refusals."""
import pytest
import torch

from complexity_framework_b200.ops import residual as R


def test_generator_known_answers():
    # published known answers of Philox4x32-10: counter 0 under keys 0 and all ones
    def words(seed, stream, n=8):
        u = R._random16(n, torch.tensor([seed]), stream)
        return [int(u[2 * i] | (u[2 * i + 1] << 16)) for i in range(n // 2)]

    assert words(0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]

    def plain(counter, key):  # in Python's integers
        c, k = list(counter), list(key)
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return c

    assert plain([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6,
                                                         0x6D5451FD]
    for seed, stream in ((-1, 0), (0x123456789ABCDEF, 7), (-2 ** 63, 2 ** 32 - 1)):
        key = seed & (2 ** 64 - 1)
        key = [key & 0xFFFFFFFF, key >> 32]
        got = words(seed, stream, 24)
        assert got == sum((plain([i, 0, stream, 0], key) for i in range(3)), [])


def test_dropout_share_and_values():
    x = torch.randn(1000, 333)
    for p in (0.0, 0.1, 0.5, 1.0):
        y = R.dropout(x, p, 5)
        f = R.dropout_factors(x.shape, p, 5)
        assert torch.equal(y, torch.where(f == 0, 0.0, x * f))
        share = float((y == 0).float().mean())
        # five standard deviations of a binomial share of n elements
        assert abs(share - p) <= 5 * (p * (1 - p) / x.numel()) ** 0.5 + 2 ** -17
    assert torch.equal(R.dropout(x, 0.0, 5), x)
    assert not torch.equal(R.dropout(x, 0.5, 5), R.dropout(x, 0.5, 6))
    assert not torch.equal(R.dropout(x, 0.5, 5), R.dropout(x, 0.5, 5, stream=1))
    assert torch.equal(R.dropout(x, 0.5, 5), R.dropout(x, 0.5, torch.tensor([5])))
    assert torch.equal(R.dropout(x, 0.5, 2 ** 64 - 3), R.dropout(x, 0.5, -3))


def test_dropped_elements_are_zero():
    x = torch.full((64, 8), float("nan"))
    y = R.dropout(x, 0.5, 1)
    f = R.dropout_factors(x.shape, 0.5, 1)
    assert bool((y[f == 0] == 0).all()) and bool(y[f != 0].isnan().all())


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("norm", [True, False])
def test_join_gradients_against_differences(post, gate, p, norm):
    g = torch.Generator().manual_seed(3)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)

    x, b = r(3, 5), r(3, 5)
    ws = [r(5) if on else None for on in (post, gate, norm)]

    def f(*ts):
        it = iter(ts[2:])
        w1, gt, w2 = [next(it) if w is not None else None for w in ws]
        new, y = R.residual_norm(ts[0], ts[1], branch_weight=w1, gate=gt, norm_weight=w2,
                                 scale=0.7, p=p, seed=9 if p else None)
        return (new,) if y is None else (new, y)

    assert torch.autograd.gradcheck(f, (x, b, *[w for w in ws if w is not None]))


def test_join_parts():
    x, b, w = torch.randn(4, 6), torch.randn(4, 6), torch.rand(6) + 0.5
    new, y = R.residual_norm(x, b)
    assert y is None and torch.equal(new, x + b)
    new, y = R.residual_norm(x, b, gate=w, scale=0.5)
    torch.testing.assert_close(new, x + 0.5 * w * b)
    new, y = R.residual_norm(x, b, branch_weight=w, norm_weight=w)
    n = w * b / (b.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    torch.testing.assert_close(new, x + n)
    torch.testing.assert_close(y, w * new / (new.square().mean(-1, keepdim=True) + 1e-6).sqrt())
    new, y = R.residual_norm(x[:0], b[:0], norm_weight=w)
    assert new.shape == y.shape == (0, 6)


def test_refusals():
    x = torch.randn(4, 6)
    with pytest.raises(ValueError, match="p must"):
        R.dropout(x, 1.5, 0)
    with pytest.raises(ValueError, match="p must"):
        R.residual_norm(x, x, p=-0.1)
    with pytest.raises(ValueError, match="seed"):
        R.residual_norm(x, x, p=0.1)
    with pytest.raises(ValueError, match="one element"):
        R.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="int64"):
        R.dropout(x, 0.1, torch.zeros(1))
    with pytest.raises(ValueError, match="64 bits"):
        R.dropout(x, 0.1, 2 ** 64)
    with pytest.raises(ValueError, match="32 bits"):
        R.dropout(x, 0.1, 0, stream=2 ** 32)
    with pytest.raises(TypeError, match="floating"):
        R.dropout(torch.ones(3, dtype=torch.int64), 0.1, 0)
    with pytest.raises(ValueError, match="branch must"):
        R.residual_norm(x, x[:2])
    with pytest.raises(ValueError, match="gate must"):
        R.residual_norm(x, x, gate=torch.ones(4))
    with pytest.raises(TypeError, match="norm_weight must"):
        R.residual_norm(x, x, norm_weight=torch.ones(6, dtype=torch.bfloat16))


def test_new_seed():
    torch.manual_seed(0)
    a, b = R.new_seed("cpu"), R.new_seed("cpu")
    assert a.dtype == torch.int64 and a.shape == (1,) and not torch.equal(a, b)
