"""Cross-entropy over the vocabulary on the GPU, against 64-bit formulas."""
import pytest
import torch

from complexity_framework_b200.ops import check_errors
from complexity_framework_b200.ops.vocab_loss import token_logprobs, vocab_cross_entropy

pytestmark = pytest.mark.gpu


def make(T, V, H, ignored=0.0, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    h = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, H, generator=g, device="cuda") * (2.0 / H ** 0.5)).bfloat16()
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    y[torch.rand(T, generator=g, device="cuda") < ignored] = -100
    return h, w, y


def oracle(h, w, y, up, smooth=0.0, z=0.0, scale=1.0):
    """Row losses and the gradients of sum(up * losses) in 64 bits, with bounds.

    A logit's 32-bit sum over H products has at most H / 16 + 2 additions in sequence, each off
    by at most 2^-23 of the magnitudes' sum; the exponentials are off by 2^-20 at most (2^-22
    of ex2.approx, and the argument's rounding).  The gradient of a logit is rounded to bf16
    (2^-8), summed in 32 bits over V (or T) products, and the sum is rounded to bf16."""
    h, w, up = h.double(), w.double(), up.double()
    T, H = h.shape
    V = w.shape[0]
    ok = y != -100
    h = torch.where(ok[:, None], h, 0.0)
    zl = scale * h @ w.t()
    lse = torch.logsumexp(zl, -1)
    zy = zl.gather(1, y.clamp_min(0)[:, None])[:, 0]
    loss = torch.where(ok, lse - (1 - smooth) * zy - smooth * zl.mean(-1) + z * lse ** 2, 0.0)
    ez = (H / 16 + 2) * 2.0 ** -23 * abs(scale) * (h.abs() @ w.abs().t()).amax(-1) \
        + 2.0 ** -20 + 2.0 ** -22 * zl.abs().amax(-1)
    loss_tol = 2 * ez * (1 + 2 * z * lse.abs()) + 2.0 ** -22 * loss.abs()
    q = torch.full_like(zl, smooth / V)
    q.scatter_add_(1, y.clamp_min(0)[:, None], torch.full_like(zl[:, :1], 1 - smooth))
    g = torch.where(ok, up, 0.0)[:, None] * scale
    p = (zl - lse[:, None]).exp()
    a = 1 + 2 * z * lse[:, None]
    dz = g * (p * a - q)
    dz_tol = g.abs() * (p * a.abs() * 2 * ez[:, None] + p * 2 * z * ez[:, None]) \
        + (2.0 ** -8 + 2.0 ** -22) * dz.abs() + 2.0 ** -22 * g.abs() * (p * a.abs() + q) \
        + 2.0 ** -126 * (1 + g.abs() * a.abs())  # what is below the smallest normal becomes 0
    dh, dw = dz @ w, dz.t() @ h
    dh_tol = dz_tol @ w.abs() + (V / 16 + 2) * 2.0 ** -23 * (dz.abs() @ w.abs()) + 2.0 ** -8 * dh.abs()
    dw_tol = dz_tol.t() @ h.abs() + (T / 16 + 2) * 2.0 ** -23 * (dz.abs().t() @ h.abs()) \
        + 2.0 ** -8 * dw.abs()
    return loss, loss_tol, dh, dh_tol, dw, dw_tol


def oracle_loss(h, w, y):
    """Losses and their bounds alone (see ``oracle``), a few rows at a time."""
    out = []
    for a in range(0, h.shape[0], 32):
        hh, yy = h[a:a + 32].double(), y[a:a + 32]
        zl = hh @ w.double().t()
        lse = torch.logsumexp(zl, -1)
        loss = torch.where(yy != -100, lse - zl.gather(1, yy.clamp_min(0)[:, None])[:, 0], 0.0)
        ez = (h.shape[1] / 16 + 2) * 2.0 ** -23 * (hh.abs() @ w.double().abs().t()).amax(-1) \
            + 2.0 ** -20 + 2.0 ** -22 * zl.abs().amax(-1)
        # sums of exponentials over the words: 32 in a row, then 4, 4 chunks, 7000 / 32 halves
        out.append((loss, 2 * ez + 2.0 ** -22 * loss.abs() + 260 * 2.0 ** -24))
    return [torch.cat(t) for t in zip(*out)]


def close(got, want, tol, name):
    err = (got.double() - want).abs()
    assert bool((err <= tol + 1e-38).all()), (name, float((err / (tol + 1e-38)).max()))


def check(T, V, H, ignored=0.0, seed=0, ws=None, **kw):
    h, w, y = make(T, V, H, ignored, seed)
    h.requires_grad_()
    w.requires_grad_()
    opt = {} if ws is None else {"workspace_bytes": ws}
    args = dict(label_smoothing=kw.get("smooth", 0.0), z_loss=kw.get("z", 0.0),
                logit_scale=kw.get("scale", 1.0), **opt)
    up = torch.randn(T, device="cuda")
    rows = vocab_cross_entropy(h, w, y, reduction="none", **args)
    got = torch.autograd.grad(rows, (h, w), up)
    loss, lt, dh, dht, dw, dwt = oracle(h.detach(), w.detach(), y, up, **kw)
    close(rows.detach(), loss, lt, "rows")
    close(got[0], dh, dht, "dh")
    close(got[1], dw, dwt, "dw")
    n = max(1, int((y != -100).sum()))
    for red, f in (("mean", 1.0 / n), ("sum", 1.0)):
        total = vocab_cross_entropy(h, w, y, reduction=red, **args)
        got = torch.autograd.grad(total, (h, w), torch.tensor(0.75, device="cuda"))
        ones = torch.full((T,), 0.75 * f, device="cuda", dtype=torch.float64)
        loss, lt, dh, dht, dw, dwt = oracle(h.detach(), w.detach(), y, ones, **kw)
        mag = loss.abs().sum() * f
        # the sum of T losses in 32 bits: fewer than T / 1024 + 12 additions in sequence
        close(total.detach(), loss.sum() * f, lt.sum() * f + (T / 1024 + 12) * 2.0 ** -24 * mag, red)
        close(got[0], dh, dht, red + " dh")
        close(got[1], dw, dwt, red + " dw")
    check_errors()


@pytest.mark.parametrize("T,V,H", [
    (1, 32, 8), (1, 1, 64), (2, 31, 72), (19, 33, 64), (64, 256, 128), (65, 257, 136),
    (127, 1000, 264), (128, 511, 72), (129, 1000, 64), (300, 2049, 520), (700, 5003, 1032)])
def test_sizes(T, V, H):
    check(T, V, H)


@pytest.mark.parametrize("smooth,z,scale", [(0.1, 0.0, 1.0), (0.0, 1e-3, 1.0), (0.2, 1e-4, 0.25),
                                            (1.0, 0.0, 1.5), (0.0, 0.0, 1e-3)])
def test_options(smooth, z, scale):
    check(150, 777, 200, ignored=0.3, smooth=smooth, z=z, scale=scale)


@pytest.mark.parametrize("ignored", [0.5, 0.97, 1.1])
@pytest.mark.parametrize("T", [1, 70, 513])
def test_ignored(T, ignored):
    check(T, 600, 72, ignored=ignored)


@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("ws", [0, 1 << 18])
def test_pieces_of_the_vocabulary(T, ws):
    check(T, 5003, 96, ignored=0.2, ws=ws, smooth=0.1, z=1e-3)


def test_wide():
    check(40, 50021, 256)
    check(900, 3001, 4096, ignored=0.2)


def test_rows_in_parts():
    """More statistics than are held at a time (256 MB): 7000 half tiles of 128 words."""
    T, V, H = 4300, 896000, 8
    h, w, y = make(T, V, H, ignored=0.2)
    rows = vocab_cross_entropy(h, w, y, reduction="none")
    pick = torch.cat((torch.arange(0, T, 37), torch.arange(T - 70, T))).cuda()
    loss, tol, *_ = oracle_loss(h[pick], w, y[pick])
    close(rows[pick], loss, tol, "rows")
    y[500:] = -100  # all counted rows in the first part
    few = vocab_cross_entropy(h, w, y, reduction="none")
    assert torch.equal(few[:500], rows[:500]) and bool((few[500:] == 0).all())
    check_errors()


def test_large_logits():
    """Logits of some hundreds: every other word's probability is 0."""
    h, w, y = make(100, 1000, 128)
    w *= 40
    h.requires_grad_()
    w.requires_grad_()
    rows = vocab_cross_entropy(h, w, y, reduction="none")
    up = torch.ones(100, device="cuda")
    loss, lt, dh, dht, dw, dwt = oracle(h.detach(), w.detach(), y, up)
    got = torch.autograd.grad(rows, (h, w), up)
    close(rows.detach(), loss, lt, "rows")
    close(got[0], dh, dht, "dh")
    close(got[1], dw, dwt, "dw")


def test_confident_rows():
    """Losses far below the logits' size: with one-hot hidden states the logits are entries of the
    weight, exact in 32 bits, and the loss is off by a few roundings of its own size and of the
    differences that enter it (2^-20 covers the exponentials), not of the logits' 60."""
    V, H = 1000, 64
    w = torch.randn(V, H, device="cuda").bfloat16()
    y = torch.randint(0, V, (H,), device="cuda")
    top = torch.rand(H, device="cuda") * 8 + 56
    w[y, torch.arange(H, device="cuda")] = top.bfloat16()
    w[(y + 1) % V, torch.arange(H, device="cuda")] = (top - 6).bfloat16()
    h = torch.eye(H, device="cuda").bfloat16()
    got = vocab_cross_entropy(h, w, y, reduction="none")
    z = w.t().double()
    want = torch.logsumexp(z - z.gather(1, y[:, None]), -1)
    assert bool(((got.double() - want).abs() <= 2.0 ** -20 * want + 2.0 ** -23).all())


def test_logprobs():
    h, w, y = make(70, 999, 96, 0.3)
    got = token_logprobs(h.view(2, 35, 96), w, y.view(2, 35), logit_scale=1.25)
    loss, lt, *_ = oracle(h, w, y, torch.ones(70, device="cuda"), scale=1.25)
    close(got.view(-1), -loss, lt, "logprobs")
    assert bool((got.view(-1)[y == -100] == 0).all())


def test_deterministic_and_other_stream():
    h, w, y = make(3000, 4001, 256, 0.1)
    h.requires_grad_()
    w.requires_grad_()

    def go():
        loss = vocab_cross_entropy(h, w, y, label_smoothing=0.1)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    a, b = go(), go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = go()
    torch.cuda.current_stream().wait_stream(side)
    for x, y1, z in zip(a, b, c):
        assert torch.equal(x, y1) and torch.equal(x, z)


def test_one_gradient_and_twice():
    h, w, y = make(100, 500, 64, 0.1)
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = vocab_cross_entropy(hg, wg, y)
    both = torch.autograd.grad(loss, (hg, wg), retain_graph=True)
    again = torch.autograd.grad(loss, (hg, wg))
    only_h = torch.autograd.grad(vocab_cross_entropy(hg, w, y), hg)[0]
    only_w = torch.autograd.grad(vocab_cross_entropy(h, wg, y), wg)[0]
    assert torch.equal(both[0], again[0]) and torch.equal(both[1], again[1])
    assert torch.equal(only_h, both[0]) and torch.equal(only_w, both[1])


def test_layouts():
    h, w, y = make(50, 300, 64)
    want = vocab_cross_entropy(h, w, y, reduction="none")
    wide = torch.zeros(50, 130, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:65] = h
    flat = torch.zeros(300 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = w.reshape(-1)
    y2 = torch.stack((y, y), -1)[:, 0]
    for a, b, c in ((wide[:, 1:65], w, y), (h.t().contiguous().t(), flat[1:].view(300, 64), y2),
                    (h, w.t().contiguous().t(), y)):
        assert torch.equal(vocab_cross_entropy(a, b, c, reduction="none"), want)
    lw = w.t().contiguous().t().requires_grad_()
    la = wide.requires_grad_()
    loss = vocab_cross_entropy(la[:, 1:65], lw, y)
    g = torch.autograd.grad(loss, (la, lw))
    hr, wr = h.clone().requires_grad_(), w.clone().requires_grad_()
    r = torch.autograd.grad(vocab_cross_entropy(hr, wr, y), (hr, wr))
    assert torch.equal(g[0][:, 1:65], r[0]) and torch.equal(g[1], r[1])


def test_ignored_rows_reach_nothing():
    h, w, y = make(200, 500, 64, 0.5)
    bad = torch.where((y == -100)[:, None], float("nan"), h.float()).bfloat16()
    out = []
    for x in (h, bad):
        x = x.clone().requires_grad_()
        ww = w.clone().requires_grad_()
        loss = vocab_cross_entropy(x, ww, y)
        out.append((loss.detach(), *torch.autograd.grad(loss, (x, ww))))
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_rows_that_are_not_finite():
    h, w, y = make(70, 500, 64)
    want = vocab_cross_entropy(h, w, y, reduction="none")
    h2 = h.clone()
    h2[3, 5] = float("inf")
    h2[66, 0] = float("nan")
    got = vocab_cross_entropy(h2, w, y, reduction="none")
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[[3, 66]] = False
    assert torch.equal(got[keep], want[keep]) and not bool(got[~keep].isfinite().any())
    w2 = w.clone()
    w2[:256] = float("-inf")  # logits of -inf and inf (or NaN): the row is not finite
    got = vocab_cross_entropy(h.abs() + 0.1, w2.float().clamp(min=-1e30).bfloat16(), y,
                              reduction="none")
    assert bool(got[y >= 256].isfinite().all())  # words of probability 0 over a whole tile


def test_empty():
    h, w, y = make(4, 50, 64)
    h, w = h[:0].requires_grad_(), w.requires_grad_()
    loss = vocab_cross_entropy(h, w, y[:0])
    g = torch.autograd.grad(loss, (h, w))
    assert float(loss) == 0 and g[0].shape == (0, 64) and bool((g[1] == 0).all())
    assert vocab_cross_entropy(h, w, y[:0], reduction="none").shape == (0,)


def test_graph_capture():
    h, w, y = make(300, 2000, 128, 0.2)
    h.requires_grad_()
    w.requires_grad_()

    def go():
        loss = vocab_cross_entropy(h, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = go()
    for seed in (3, 4):  # other rows, another number of ignored targets
        h2, _, y2 = make(300, 2000, 128, 0.3 * seed - 0.8, seed)
        with torch.no_grad():
            h.copy_(h2)
        y.copy_(y2)
        graph.replay()
        for a, b in zip(outs, go()):
            assert torch.equal(a, b)


def test_targets_out_of_range():
    h, w, y = make(10, 50, 64)
    y[4], y[5] = 50, -3
    rows = vocab_cross_entropy(h, w, y, reduction="none")
    assert bool(rows[[4, 5]].isnan().all()) and bool(rows[[0, 1, 2, 3, 6, 7, 8, 9]].isfinite().all())
    with pytest.raises(RuntimeError, match="device error"):
        check_errors()
    check_errors()


def test_refusals():
    h, w, y = make(10, 50, 64)
    with pytest.raises(TypeError, match="bfloat16"):
        vocab_cross_entropy(h.float(), w, y)
    with pytest.raises(TypeError, match="bfloat16"):
        vocab_cross_entropy(h, w.float(), y)
    with pytest.raises(ValueError, match="multiple of 8"):
        vocab_cross_entropy(h[:, :60], w[:, :60], y)
    with pytest.raises(RuntimeError, match="CUDA"):
        vocab_cross_entropy(h, w, y.cpu())
    wg = w.clone().requires_grad_()
    loss = vocab_cross_entropy(h, wg, y)
    with torch.no_grad():
        wg.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
