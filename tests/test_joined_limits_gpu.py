"""Loss options and joined residuals at the borders of their calls, on the kernels."""
import pytest
import torch

from complexity_framework_b200.core.losses import causal_lm_loss_from_hidden
from complexity_framework_b200.ops import check_errors
from complexity_framework_b200.ops.vocab_loss import vocab_cross_entropy

pytestmark = pytest.mark.gpu


def rows(T=70, V=333, H=64, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    h = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, H, generator=g, device="cuda") * 0.2).bfloat16()
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    y[::5] = -100
    return h, w, y


# ------------------------------------------- calls of the loss that have no kernel
@pytest.mark.parametrize("scale", [0.0, -0.5])
def test_any_logit_scale(scale):
    """A scale that is not positive is PyTorch's: the loop rounds the logits to bf16 (2^-9 of
    some 3 at most) before it scales them, and the mean loss is off by no more."""
    h, w, y = rows()
    h.requires_grad_()
    w.requires_grad_()
    got = causal_lm_loss_from_hidden(h, w, y, logit_scale=scale)
    want = torch.nn.functional.cross_entropy(scale * h.double() @ w.double().t(), y)
    z = (h.double() @ w.double().t()).abs().max()
    assert abs(float(got.detach()) - float(want.detach())) <= 2 * abs(scale) * 2.0 ** -8 * float(z) + 1e-5
    for a, b in zip(torch.autograd.grad(got, (h, w)), torch.autograd.grad(want, (h, w))):
        assert float((a.double() - b).norm()) <= 2.0 ** -6 * float(b.norm())


def test_transforms_and_forward_derivatives():
    """torch.func and forward-mode differentiation, which the kernels take no part in."""
    import torch.autograd.forward_ad as fa

    h, w, y = rows()

    def loss(h):
        return causal_lm_loss_from_hidden(h, w, y, checkpoint_chunks=False)

    a = h.clone().requires_grad_()
    want = torch.autograd.grad(loss(a), a)[0].double()
    got = torch.func.grad(loss)(h).double()
    # two ways of rounding a gradient: each off by two roundings to 8 bits at most
    assert float((got - want).norm()) <= 4 * 2.0 ** -8 * float(want.norm())
    three = torch.func.vmap(loss)(torch.stack((h, h * 2, h)))
    one = torch.stack([loss(v) for v in (h, h * 2, h)])
    # logits of up to some 6 rounded to 8 bits by one of the two
    assert float((three - one).abs().max()) <= 6 * 2.0 ** -8
    t = torch.randn(h.shape, device="cuda").bfloat16()
    with fa.dual_level():
        out = fa.unpack_dual(loss(fa.make_dual(h, t)))
    slope = float((want * t.double()).sum())
    mag = float((want * t.double()).abs().sum())
    assert abs(float(out.tangent) - slope) <= 4 * 2.0 ** -8 * mag


# ----------------------------------------------------------------- very many rows
def test_losses_of_very_many_rows():
    """More rows than the blocks of the gathering kernel take at a time, ignored ones among them:
    with a hidden size of 8 and one-hot states the logits are entries of the weight."""
    T, V = 700001, 40
    g = torch.Generator("cuda").manual_seed(2)
    w = torch.randn(V, 8, generator=g, device="cuda").bfloat16().requires_grad_()
    k = torch.randint(0, 8, (T,), generator=g, device="cuda")
    h = torch.nn.functional.one_hot(k, 8).bfloat16().requires_grad_()
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    y[torch.rand(T, generator=g, device="cuda") < 0.3] = -100
    got = vocab_cross_entropy(h, w, y, reduction="none")
    table = -torch.log_softmax(w.detach().double().t(), -1)  # [8, V]
    want = torch.where(y == -100, 0.0, table[k, y.clamp_min(0)])
    # losses of up to some 10: a few roundings to 24 bits and the exponentials' 2^-20
    assert float((got.detach().double() - want).abs().max()) <= 2.0 ** -18
    up = torch.randint(1, 3, (T,), generator=g, device="cuda").float()
    dh, dw = torch.autograd.grad(got, (h, w), up)
    on = (y != -100).double()[:, None]
    dz = up.double()[:, None] * on * ((-table[k]).exp()
                                      - torch.nn.functional.one_hot(y.clamp_min(0), V))
    rh, rw = dz @ w.detach().double(), dz.t() @ h.detach().double()
    # dz rounded to 8 bits, then the result
    assert bool(((dh.double() - rh).abs() <= 2.0 ** -7 * (dz.abs() @ w.detach().double().abs())
                 + 2.0 ** -20).all())
    assert bool(((dw.double() - rw).abs() <= 2.0 ** -7 * (dz.abs().t() @ h.detach().double())
                 + 2.0 ** -20).all())
    check_errors()


def test_time_grows_with_the_rows():
    """Four times the rows take four times as long (less, as far as launches count), not sixteen
    times."""
    w = torch.randn(32, 8, device="cuda").bfloat16()

    def best(T):
        h = torch.randn(T, 8, device="cuda").bfloat16()
        y = torch.randint(0, 32, (T,), device="cuda")
        out = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            vocab_cross_entropy(h, w, y)
            b.record()
            b.synchronize()
            out.append(a.elapsed_time(b))
        return min(out)

    few, many = best(1 << 20), best(1 << 22)
    assert many <= 7 * few, (few, many)
