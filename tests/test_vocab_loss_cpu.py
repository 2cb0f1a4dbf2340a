"""Cross-entropy over the vocabulary on the CPU: formulas and refusals."""
import pytest
import torch
import torch.nn.functional as F

from complexity_framework_b200.ops.vocab_loss import token_logprobs, vocab_cross_entropy


def make(T=7, V=11, H=6, dtype=torch.float64):
    g = torch.Generator().manual_seed(1)
    h = torch.randn(T, H, generator=g, dtype=dtype, requires_grad=True)
    w = torch.randn(V, H, generator=g, dtype=dtype, requires_grad=True)
    y = torch.randint(0, V, (T,), generator=g)
    y[2] = -100
    return h, w, y


@pytest.mark.parametrize("smooth", [0.0, 0.2, 1.0])
@pytest.mark.parametrize("z", [0.0, 0.01])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_against_logits(smooth, z, scale):
    h, w, y = make()
    logits = (h @ w.t()) * scale
    lse = torch.logsumexp(logits, -1)
    want = F.cross_entropy(logits, y, label_smoothing=smooth, reduction="none")
    want = want + z * torch.where(y != -100, lse.square(), 0.0)
    kw = dict(label_smoothing=smooth, z_loss=z, logit_scale=scale)
    for red, ref in (("none", want), ("sum", want.sum()), ("mean", want.sum() / 6)):
        got = vocab_cross_entropy(h, w, y, reduction=red, **kw)
        torch.testing.assert_close(got, ref)
        u = torch.randn_like(ref)
        for a, b in zip(torch.autograd.grad(got, (h, w), u, retain_graph=True),
                        torch.autograd.grad(ref, (h, w), u, retain_graph=True)):
            torch.testing.assert_close(a, b)
    assert torch.autograd.gradcheck(lambda a, b: vocab_cross_entropy(a, b, y, reduction="none", **kw),
                                    (h, w))


def test_logprobs_and_shapes():
    h, w, y = make(T=8)
    y3 = y.view(2, 4)
    got = token_logprobs(h.view(2, 4, 6), w, y3, logit_scale=0.8)
    ref = torch.log_softmax((h @ w.t()) * 0.8, -1).gather(1, y.clamp_min(0)[:, None])[:, 0]
    torch.testing.assert_close(got.view(-1), torch.where(y == -100, 0.0, ref))
    assert got.shape == (2, 4)


def test_nothing_counted():
    h, w, y = make()
    y = torch.full_like(y, -1)
    loss = vocab_cross_entropy(h, w, y, ignore_index=-1)
    assert float(loss) == 0
    assert all(bool((g == 0).all()) for g in torch.autograd.grad(loss, (h, w)))
    assert float(vocab_cross_entropy(h[:0], w, y[:0])) == 0


def test_ignored_rows_reach_nothing():
    h, w, y = make()
    clean = vocab_cross_entropy(h, w, y)
    g0 = torch.autograd.grad(clean, (h, w))
    bad = h.detach().clone()
    bad[2] = float("nan")
    bad.requires_grad_()
    loss = vocab_cross_entropy(bad, w, y)
    g1 = torch.autograd.grad(loss, (bad, w))
    assert torch.equal(loss, clean) and torch.equal(g0[0], g1[0]) and torch.equal(g0[1], g1[1])


def test_refusals():
    h, w, y = make()
    with pytest.raises(ValueError, match="reduction"):
        vocab_cross_entropy(h, w, y, reduction="batch")
    with pytest.raises(ValueError, match="label_smoothing"):
        vocab_cross_entropy(h, w, y, label_smoothing=1.5)
    with pytest.raises(ValueError, match="z_loss"):
        vocab_cross_entropy(h, w, y, z_loss=-1.0)
    with pytest.raises(ValueError, match="targets must"):
        vocab_cross_entropy(h, w, y[:3])
    with pytest.raises(TypeError, match="int64"):
        vocab_cross_entropy(h, w, y.int())
    with pytest.raises(ValueError, match=r"\[V, H\]"):
        vocab_cross_entropy(h, w.t(), y)
    with pytest.raises(ValueError, match="neither a word"):
        vocab_cross_entropy(h, w, torch.full_like(y, 11))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="logit_scale"):
            vocab_cross_entropy(h, w, y, logit_scale=scale)
    with pytest.raises(ValueError, match="workspace"):
        vocab_cross_entropy(h, w, y, workspace_bytes=-1)
