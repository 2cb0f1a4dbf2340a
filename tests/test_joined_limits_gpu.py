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


def test_second_derivatives():
    """Gradients of gradients, against the formula in 64 bits."""
    h, w, y = rows()
    gen = torch.Generator("cuda").manual_seed(5)
    u, v = (torch.randn(t.shape, generator=gen, device="cuda") for t in (h, w))
    up = torch.randn(70, generator=gen, device="cuda")

    def second(f, h, w, factor):
        h, w, factor = (t.detach().clone().requires_grad_() for t in (h, w, factor))
        hh = h * 1.0  # not a leaf
        loss = f(hh, w)
        if loss.dim():
            first = torch.autograd.grad(loss, (hh, w), factor.to(loss.dtype), create_graph=True)
        else:
            first = torch.autograd.grad(loss, (hh, w), factor[0].to(loss.dtype), create_graph=True)
        dot = (first[0] * u.to(first[0].dtype)).sum() + (first[1] * v.to(first[1].dtype)).sum()
        return [t.detach().double() for t in first], \
            [t.double() for t in torch.autograd.grad(dot, (h, w, factor))]

    def kernel(**kw):
        return lambda h, w: vocab_cross_entropy(h, w, y, **kw)

    def formula(smooth=0.0, z=0.0, scale=1.0, reduction="mean"):
        def f(h, w):
            zl = scale * h @ w.t()
            keep = y != -100
            lse = torch.logsumexp(zl, -1)
            loss = lse - (1 - smooth) * zl.gather(1, y.clamp_min(0)[:, None])[:, 0] \
                - smooth * zl.mean(-1) + z * lse ** 2
            loss = torch.where(keep, loss, 0.0)
            return {"none": loss, "sum": loss.sum(), "mean": loss.sum() / keep.sum()}[reduction]
        return f

    for red in ("none", "sum", "mean"):
        for smooth, z, scale in ((0.0, 0.0, 1.0), (0.1, 1e-2, 0.5)):
            got = second(kernel(label_smoothing=smooth, z_loss=z, logit_scale=scale,
                                reduction=red), h, w, up)
            want = second(formula(smooth, z, scale, red), h.double(), w.double(), up.double())
            # the first gradient is the kernels': dz and the result rounded to 8 bits
            for a, b in zip(got[0], want[0]):
                assert float((a - b).norm()) <= 2 * 2.0 ** -8 * float(b.norm())
            # u and v are rounded to 8 bits, then the result: 2^-9 each in the mean
            for a, b in zip(got[1], want[1]):
                assert float((a - b).norm()) <= 4 * 2.0 ** -8 * float(b.norm())
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    plain = torch.autograd.grad(vocab_cross_entropy(a, b, y), (a, b))
    graph = torch.autograd.grad(vocab_cross_entropy(a, b, y), (a, b), create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(plain, graph))
    # the frozen one has no part
    only = torch.autograd.grad(vocab_cross_entropy(a, w, y), a, create_graph=True)[0]
    assert torch.autograd.grad(only.float().square().sum(), a)[0].isfinite().all()
    check_errors()


def test_second_derivatives_in_other_layouts():
    """A weight that is copied for the call, three dimensions, a node that is called by itself."""
    h, w, y = rows()
    wt = w.t().contiguous().requires_grad_()
    a = h.clone().requires_grad_()
    b, c = w.clone().requires_grad_(), h.view(2, 35, 64).clone().requires_grad_()
    out = []
    for x, m, leaf, t in ((a, wt.t(), wt, y), (c, b, b, y.view(2, 35))):
        loss = vocab_cross_entropy(x, m, t, z_loss=1e-3)
        gx, gm = torch.autograd.grad(loss, (x, m), create_graph=True)
        out.append(torch.autograd.grad(gx.float().square().sum() + gm.float().square().sum(),
                                       (x, leaf)))
    assert torch.equal(out[0][0], out[1][0].view(70, 64)) and torch.equal(out[0][1].t(), out[1][1])
    loss = vocab_cross_entropy(a, b, y)
    want = torch.autograd.grad(loss, (a, b), retain_graph=True)
    got = loss.grad_fn(torch.ones((), device="cuda"))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_errors()


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


# ------------------------------------------------------- joins of many rows, in parts
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
LEFT_OUT = ["none", "w1", "gate", "w2", "dy", "dx", "w1 w2", "w1 gate w2"]


@pytest.mark.parametrize("left_out", LEFT_OUT)
@pytest.mark.parametrize("H", [264, 896, 903, 2048, 8192])
@pytest.mark.parametrize("dtype,p", [("bf16", 0.0), ("bf16", 0.2), ("fp32", 0.2)])
def test_join_parts_with_many_rows(left_out, H, dtype, p):
    """Rows enough that one or two warps take a row each, without a norm, gate or gradient."""
    from test_residual_gpu import call, check, make, oracle

    off = left_out.split()
    t = make(2501, H, DT[dtype], "w1" not in off, "gate" not in off, "w2" not in off, seed=H)
    if "dy" in off or "dx" in off:
        from complexity_framework_b200.ops import residual as R

        one = {**t, **{k: torch.zeros_like(t[k]) for k in ("dx", "dy") if k in off}}
        want, tol = oracle(one, 0.7, p, 3, 0)
        leaf = {k: t[k].detach().clone().requires_grad_() for k in ("x", "b", "w1", "gate", "w2")}
        new, y = R.residual_norm(leaf["x"], leaf["b"], branch_weight=leaf["w1"],
                                 gate=leaf["gate"], norm_weight=leaf["w2"], scale=0.7, p=p,
                                 seed=3)
        (new if "dy" in off else y).backward(t["dx" if "dy" in off else "dy"])
        got = {"d" + k: v.grad for k, v in leaf.items() if v.grad is not None}
        assert ("dw2" in got) == ("dx" in off)
    else:
        want, tol = oracle(t, 0.7, p, 3, 0)
        got = call(t, 0.7, p, 3 if p else None, 0)
    check(got, want, tol, DT[dtype])
    check_errors()


@pytest.mark.parametrize("graph", [False, True])
def test_resumed_run_goes_on_with_the_masks(tmp_path, graph):
    """A learning rate of nearly nothing: the losses of a step differ by their masks alone.  The
    model's other kernels add some gradients by atomics, which reach a loss by less than 1e-3."""
    from complexity_framework_b200 import ComplexityModel
    from complexity_framework_b200.config import ModelConfig
    from complexity_framework_b200.training import Trainer, TrainingConfig

    def trainer():
        torch.manual_seed(0)
        m = ComplexityModel(ModelConfig(
            hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
            intermediate_size=256, shared_intermediate_size=256, vocab_size=1000, num_experts=2,
            top_k=2, max_position_embeddings=256, residual_dropout=0.3, embedding_dropout=0.2,
            norm_placement="sandwich"))
        return Trainer(m, TrainingConfig(learning_rate=1e-8, precision="bf16", warmup_steps=0,
                                         lr_scheduler="constant", weight_decay=0.0,
                                         cuda_graph=graph, cuda_graph_warmup=2,
                                         skip_param_update_check=True,
                                         checkpoint_dir=str(tmp_path)))

    ids = torch.randint(0, 1000, (2, 64)).pin_memory()
    a = trainer()
    for _ in range(4):
        a.train_step(ids)
    a.save_checkpoint()
    want = [a.train_step(ids) for _ in range(4)]
    b = trainer()
    torch.cuda.manual_seed(77)
    assert b.resume("auto")
    got = [b.train_step(ids) for _ in range(4)]
    spread = max(abs(p - q) for p in want for q in want)
    assert spread > 5e-3
    assert max(abs(p - q) for p, q in zip(got, want)) <= 1e-3, (got, want)
    check_errors()
