"""The residual join and counter-based dropout on the GPU, against 64-bit formulas."""
import pytest
import torch

from complexity_framework_b200.ops import residual as R

pytestmark = pytest.mark.gpu

EPS = 1e-6
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(T, H, dt, post, gate, norm, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    t = {"x": (3 * r(T, H)).to(dt), "b": r(T, H).to(dt),
         "w1": (1 + 0.3 * r(H)).to(dt) if post else None,
         "gate": (1 + 0.3 * r(H)).to(dt) if gate else None,
         "w2": (1 + 0.3 * r(H)).to(dt) if norm else None,
         "dx": r(T, H).to(dt), "dy": r(T, H).to(dt) if norm else None}
    return t


def oracle(t, scale, p, seed, stream):
    """Outputs, gradients and their bounds in 64 bits.  A bound counts the rounding of each
    result, `half` (half a step of the type); what the saved x', rounded once, costs the
    gradients through the second norm; and the 32-bit sums, `tiny` of the summed magnitudes."""
    dt = t["x"].dtype
    half, tiny = torch.finfo(dt).eps / 2, 64 * 2.0 ** -24
    d = {k: None if v is None else v.double() for k, v in t.items()}
    H = d["x"].shape[-1]
    one = torch.ones((), dtype=torch.float64, device="cuda")
    w1, gate, w2 = [one if d[k] is None else d[k] for k in ("w1", "gate", "w2")]
    m = one
    if p > 0:
        m = R.dropout_factors(d["x"].shape, p, seed, stream=stream, device="cuda").double()
    r1 = (d["b"].square().mean(-1, keepdim=True) + EPS).rsqrt() if t["w1"] is not None else one
    bh = d["b"] * r1
    u = m * gate * w1 * bh
    new = d["x"] + scale * u
    out, tol = {"new": new}, {"new": half * new.abs() + tiny * (d["x"].abs() + (scale * u).abs())}
    g, g_tol = d["dx"], torch.zeros_like(new)
    if t["w2"] is not None:
        r2 = (new.square().mean(-1, keepdim=True) + EPS).rsqrt()
        xh = new * r2
        out["y"] = w2 * xh
        tol["y"] = half * out["y"].abs() + tiny * (w2.abs() * r2 * (d["x"].abs() + (scale * u).abs()))
        dn = w2 * d["dy"]
        mean = (dn * xh).mean(-1, keepdim=True)
        mean_abs = (dn * xh).abs().mean(-1, keepdim=True)
        g = g + r2 * (dn - xh * mean)
        # x + scale u may cancel: the error of x' counts its terms, not x' itself, and
        # xh = x' r2 and the mean of dn xh inherit it
        xh_tol = r2 * tol["new"] + tiny * xh.abs()
        mean_tol = (dn.abs() * xh_tol).mean(-1, keepdim=True) + tiny * mean_abs
        g_tol = r2 * (xh_tol * mean.abs() + (xh.abs() + xh_tol) * mean_tol) \
            + tiny * (d["dx"].abs() + r2 * (dn.abs() + xh.abs() * mean_abs))
        out["dw2"] = (d["dy"] * xh).sum(0)
        tol["dw2"] = (d["dy"].abs() * (xh_tol + tiny * xh.abs())).sum(0) + half * out["dw2"].abs()
    out["dx"], tol["dx"] = g, half * g.abs() + g_tol
    s = scale * m * g
    s_tol = abs(scale) * m * g_tol
    if t["gate"] is not None:
        out["dgate"] = (s * w1 * bh).sum(0)
        tol["dgate"] = ((s_tol + tiny * s.abs()) * (w1 * bh).abs()).sum(0) + half * out["dgate"].abs()
    db, db_tol = s * gate * w1, s_tol * (gate * w1).abs()
    if t["w1"] is not None:
        out["dw1"] = (s * gate * bh).sum(0)
        tol["dw1"] = ((s_tol + tiny * s.abs()) * (gate * bh).abs()).sum(0) + half * out["dw1"].abs()
        mean, mean_abs = [(v * bh).mean(-1, keepdim=True) for v in (db, db.abs())]
        mean_abs = (db * bh).abs().mean(-1, keepdim=True)
        mean_tol = (db_tol * bh.abs()).mean(-1, keepdim=True)
        db_tol = r1 * (db_tol + bh.abs() * mean_tol + tiny * (db.abs() + bh.abs() * mean_abs))
        db = r1 * (db - bh * mean)
    out["db"], tol["db"] = db, half * db.abs() + db_tol + tiny * db.abs()
    return out, tol


def call(t, scale, p, seed, stream, grad=True):
    leaf = {k: None if t[k] is None else t[k].detach().requires_grad_(grad)
            for k in ("x", "b", "w1", "gate", "w2")}
    new, y = R.residual_norm(leaf["x"], leaf["b"], branch_weight=leaf["w1"], gate=leaf["gate"],
                             norm_weight=leaf["w2"], scale=scale, p=p, seed=seed, stream=stream,
                             eps=EPS)
    out = {"new": new.detach()}
    if y is not None:
        out["y"] = y.detach()
    if not grad:
        return out
    outs, ups = [new], [t["dx"]]
    if y is not None:
        outs.append(y)
        ups.append(t["dy"])
    torch.autograd.backward(outs, ups)
    for k in leaf:
        if leaf[k] is not None:
            out["d" + k] = leaf[k].grad
    return out


def check(got, want, tol, dt):
    small = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps  # a subnormal step
    for k, v in got.items():
        assert v.dtype == dt
        err = (v.double() - want[k]).abs()
        bad = err > tol[k] + small
        assert not bool(bad.any()), (k, float((err / (tol[k] + small)).max()))


SHAPES = [(1, 8), (3, 24), (65, 72), (7, 256), (130, 896), (300, 1024), (5, 1111), (33, 2056),
          (9, 4096), (2, 8192), (1, 1), (4, 3), (3, 8191), (29, 903), (17, 4095), (2, 6001)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H", SHAPES)
def test_join_everything(T, H, dtype):
    t = make(T, H, DT[dtype], True, True, True)
    want, tol = oracle(t, 0.5, 0.2, 77, 3)
    check(call(t, 0.5, 0.2, 77, 3), want, tol, DT[dtype])


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("H", [896, 77])
def test_join_parts(post, gate, p, norm, H):
    t = make(301, H, torch.bfloat16, post, gate, norm, seed=4)
    want, tol = oracle(t, 1.0, p, 5, 0)
    check(call(t, 1.0, p, 5 if p else None, 0), want, tol, torch.bfloat16)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("H", [16384, 16370, 12345])
def test_join_widest(H, dtype):
    t = make(11, H, DT[dtype], True, True, True)
    want, tol = oracle(t, 1.0, 0.1, 8, 0)
    check(call(t, 1.0, 0.1, 8, 0), want, tol, DT[dtype])


def test_join_too_wide():
    for H in (16392, 16371):
        z = torch.zeros(1, H, device="cuda", dtype=torch.bfloat16)
        with pytest.raises(ValueError, match="too wide"):
            R.residual_norm(z, z)


def test_forward_alone_is_the_same():
    t = make(65, 896, torch.bfloat16, True, True, True)
    a = call(t, 0.5, 0.1, 1, 0)
    with torch.no_grad():
        b = call(t, 0.5, 0.1, 1, 0, grad=False)
    assert torch.equal(a["new"], b["new"]) and torch.equal(a["y"], b["y"])


def test_many_rows_are_deterministic():
    t = make(20011, 896, torch.bfloat16, True, True, True)
    want, tol = oracle(t, 0.5, 0.1, 1, 0)
    a = call(t, 0.5, 0.1, 1, 0)
    check(a, want, tol, torch.bfloat16)
    b = call(t, 0.5, 0.1, 1, 0)
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H", [264, 903, 1000, 1017, 1024])
def test_rows_for_every_warp(H, dtype):
    """Enough rows that one or two warps take a row each."""
    t = make(2501, H, DT[dtype], True, True, True, seed=H)
    want, tol = oracle(t, 0.7, 0.1, 3, 0)
    check(call(t, 0.7, 0.1, 3, 0), want, tol, DT[dtype])


@pytest.mark.parametrize("which", ["x", "b", "w1", "gate", "w2"])
def test_one_gradient_at_a_time(which):
    t = make(65, 136, torch.bfloat16, True, True, True)
    full = call(t, 0.5, 0.1, 1, 0)
    leaf = {k: t[k].detach().clone() for k in ("x", "b", "w1", "gate", "w2")}
    leaf[which].requires_grad_()
    new, y = R.residual_norm(leaf["x"], leaf["b"], branch_weight=leaf["w1"], gate=leaf["gate"],
                             norm_weight=leaf["w2"], scale=0.5, p=0.1, seed=1, eps=EPS)
    if which == "w2":
        assert new.requires_grad  # one autograd node gives both
    torch.autograd.backward([new, y], [t["dx"], t["dy"]])
    assert torch.equal(leaf[which].grad, full["d" + which])


@pytest.mark.parametrize("used", ["new", "y"])
def test_one_output_used(used):
    t = make(65, 136, torch.float32, True, True, True)
    z = {**t, ("dy" if used == "new" else "dx"): torch.zeros_like(t["dx"])}
    want, tol = oracle(z, 0.5, 0.1, 1, 0)
    leaf = {k: t[k].detach().clone().requires_grad_() for k in ("x", "b", "w1", "gate", "w2")}
    new, y = R.residual_norm(leaf["x"], leaf["b"], branch_weight=leaf["w1"], gate=leaf["gate"],
                             norm_weight=leaf["w2"], scale=0.5, p=0.1, seed=1, eps=EPS)
    if used == "new":
        new.backward(t["dx"])
        assert leaf["w2"].grad is None
    else:
        y.backward(t["dy"])
    check({"d" + k: v.grad for k, v in leaf.items() if v.grad is not None}, want, tol,
          torch.float32)


def test_layouts():
    """Strided, offset and 3-D inputs, an expanded gate and strided gradients."""
    t = make(24, 64, torch.bfloat16, True, True, True)
    want = call(t, 0.5, 0.1, 1, 0)
    wide = torch.zeros(24, 130, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:65], wide[:, 65:129] = t["x"], t["b"]
    flat = torch.zeros(24 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = t["dx"].reshape(-1)
    for x, b, dx in ((wide[:, 1:65], wide[:, 65:129], t["dx"].t().contiguous().t()),
                     (t["x"], t["b"].t().contiguous().t(), flat[1:].view(24, 64))):
        got = call({**t, "x": x, "b": b, "dx": dx}, 0.5, 0.1, 1, 0)
        for k in want:
            assert torch.equal(got[k], want[k]), k
    t3 = {k: v.view(2, 12, 64) if v.dim() == 2 else v for k, v in t.items()}
    got = call(t3, 0.5, 0.1, 1, 0)
    assert torch.equal(got["db"].view(24, 64), want["db"])
    g = torch.full((1,), 0.5, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    new, _ = R.residual_norm(t["x"], t["b"], gate=g.expand(64))
    new.backward(t["dx"])
    ref = (t["dx"].double() * t["b"].double()).sum()
    mag = (t["dx"].double() * t["b"].double()).abs().sum()
    # 64 channel sums rounded to bf16, their sum rounded again
    assert abs(float(g.grad) - float(ref)) <= float(mag) * 2.0 ** -8 * 2


def test_empty_and_not_finite():
    t = make(0, 64, torch.bfloat16, True, True, True)
    got = call(t, 1.0, 0.1, 1, 0)
    assert got["new"].shape == (0, 64) and bool((got["dw2"] == 0).all())
    t = make(6, 64, torch.bfloat16, False, True, False)
    clean = call(t, 1.0, 0.5, 1, 0)
    f = R.dropout_factors((6, 64), 0.5, 1, device="cuda")
    t["b"] = torch.where(f == 0, float("nan"), t["b"].float()).bfloat16()
    got = call(t, 1.0, 0.5, 1, 0)  # what is dropped does not count
    for k in clean:
        assert torch.equal(got[k], clean[k]), k
    t = make(6, 64, torch.bfloat16, True, True, True)
    t["b"][2, 5] = float("inf")
    got = call(t, 1.0, 0.0, None, 0)
    assert bool(got["new"][2].isnan().any()) and bool(got["new"][[0, 1, 3, 4, 5]].isfinite().all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 65537])
def test_dropout(n, dtype):
    dt = DT[dtype]
    x = torch.randn(n, device="cuda").to(dt).requires_grad_()
    dy = torch.randn(n, device="cuda").to(dt)
    for p, seed, stream in ((0.1, 3, 0), (0.5, -7, 2 ** 32 - 1), (0.0, 1, 1), (1.0, 1, 1)):
        f = R.dropout_factors((n,), p, seed, stream=stream, device="cuda")
        y = R.dropout(x, p, seed, stream=stream)
        assert torch.equal(y, (x.detach().float() * f).to(dt))
        (dx,) = torch.autograd.grad(y, x, dy)
        assert torch.equal(dx, (dy.float() * f).to(dt))
        assert torch.equal(R.dropout(x, p, torch.tensor([seed], device="cuda"), stream=stream), y)


def philox(block, stream, seed):
    """Random bits of one block in Python's integers: 8 x 16 bits."""
    c, k = [block & 0xFFFFFFFF, block >> 32, stream, 0], [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [v >> s & 0xFFFF for v in c for s in (0, 16)]


@pytest.mark.parametrize("H", [520, 515])
def test_more_elements_than_31_bits(H):
    T = 2 ** 31 // H + 3
    x = torch.ones(T, H, device="cuda", dtype=torch.bfloat16)
    y = R.dropout(x, 0.5, 12345, stream=6)
    new, n = R.residual_norm(x, x, norm_weight=x[0], p=0.5, seed=12345, stream=6)
    for row in (0, T // 2, T - 1):
        e = [row * H + c for c in range(H)]
        bits = {b: philox(b, 6, 12345) for b in range(e[0] // 8, e[-1] // 8 + 1)}
        want = torch.tensor([2.0 if bits[i // 8][i % 8] >= 32768 else 0.0 for i in e])
        assert torch.equal(y[row].cpu().float(), want)
        assert torch.equal(new[row].cpu().float(), 1 + want)
        ref = (1 + want.double()) / ((1 + want.double()).square().mean() + 1e-6).sqrt()
        assert bool(((n[row].cpu().double() - ref).abs() <= 2.0 ** -8 * ref).all())


def test_dropout_layouts():
    base = torch.randn(9, 34, device="cuda", dtype=torch.float16)
    for x in (base[:, 1:], base.t(), base.reshape(-1)[1:], base[:0]):
        f = R.dropout_factors(x.shape, 0.25, 11, device="cuda")
        assert torch.equal(R.dropout(x, 0.25, 11), (x.float() * f).half())
    nan = torch.full((64,), float("nan"), device="cuda")
    f = R.dropout_factors((64,), 0.5, 1, device="cuda")
    y = R.dropout(nan, 0.5, 1)
    assert bool((y[f == 0] == 0).all()) and bool(y[f != 0].isnan().all())


def test_graph_replays_draw_new_masks():
    t = make(64, 896, torch.bfloat16, True, True, True)
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    leaf = {k: t[k].detach().clone().requires_grad_() for k in ("x", "b", "w1", "gate", "w2")}

    def step():
        seed.random_()
        new, y = R.residual_norm(leaf["x"], leaf["b"], branch_weight=leaf["w1"],
                                 gate=leaf["gate"], norm_weight=leaf["w2"], p=0.5, seed=seed,
                                 eps=EPS)
        return (new.detach(), y.detach(), *torch.autograd.grad((new, y), tuple(leaf.values()),
                                                               (t["dx"], t["dy"])))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        s = int(seed)
        seen.append(s)
        want = call(t, 1.0, 0.5, s, 0)
        for got, k in zip(outs, ("new", "y", "dx", "db", "dw1", "dgate", "dw2")):
            assert torch.equal(got, want[k]), k
    assert len(set(seen)) == 3


def test_seed_changed_before_backward_is_refused():
    x = torch.randn(8, 8, device="cuda", requires_grad=True)
    seed = R.new_seed("cuda")
    y = R.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_two_threads():
    """Calls of one kernel with small and large rows from two threads at once."""
    import threading

    small = make(40, 1032, torch.bfloat16, True, True, True)
    large = make(40, 2048, torch.bfloat16, True, True, True)
    want = [call(t, 0.5, 0.1, 1, 0) for t in (small, large)]
    bad = []

    def go(t, w):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                got = call(t, 0.5, 0.1, 1, 0)
                torch.cuda.current_stream().synchronize()
                bad.extend(k for k in w if not torch.equal(got[k], w[k]))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=go, args=a) for a in zip((small, large), want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_another_stream():
    t = make(2048, 896, torch.bfloat16, True, True, True)
    want = call(t, 0.5, 0.1, 1, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(t, 0.5, 0.1, 1, 0)
    torch.cuda.current_stream().wait_stream(side)
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_refusals():
    x = torch.randn(4, 8, device="cuda")
    with pytest.raises(TypeError, match="bfloat16"):
        R.dropout(x.double(), 0.1, 0)
    with pytest.raises(TypeError, match="bfloat16"):
        R.residual_norm(x.double(), x.double())
    with pytest.raises(ValueError, match="device"):
        R.residual_norm(x, x.cpu())
    with pytest.raises(ValueError, match="branch must"):
        R.residual_norm(x, x[:2])
    with pytest.raises(ValueError, match="gate must"):
        R.residual_norm(x, x, gate=x[0, :4])
    with pytest.raises(TypeError, match="norm_weight must"):
        R.residual_norm(x, x, norm_weight=x[0].bfloat16())
    with pytest.raises(TypeError, match="bfloat16"):
        R.residual_norm(x.long(), x.long())
    with pytest.raises(ValueError, match="scale must"):
        R.residual_norm(x, x, scale=float("nan"))
    with pytest.raises(ValueError, match="eps must"):
        R.residual_norm(x, x, norm_weight=x[0], eps=-1.0)
    with pytest.raises(ValueError, match="seed"):
        R.residual_norm(x, x, p=0.1)
    with pytest.raises(ValueError, match="device"):
        R.dropout(x, 0.1, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="once_differentiable|twice"):
        z = x.clone().requires_grad_()
        y = R.dropout(z, 0.5, 1)
        (g,) = torch.autograd.grad(y.square().sum(), z, create_graph=True)
        g.sum().backward()
