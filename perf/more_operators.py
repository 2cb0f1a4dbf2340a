"""Cases of the operators around a decoder's blocks: the joins of the residual stream
(norms before and after a block, gate, residual scale, dropout), dropout by itself, and the
cross-entropy over the vocabulary without its logits.

``run`` computes a case in elementary torch operations in 32 bits, or, with ``own`` set,
through ``complexity_framework_b200.ops.residual`` and ``.ops.vocab_loss``.
"""
import math

import torch

own = False

EPS = 1e-6
IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------- the cases
def _loss(name, tokens, vocab, hidden, mode, ignored=0.0, smoothing=0.0, z_loss=0.0, scale=1.0):
    """mode: "mean" (training loss and its gradients), "rows" (log-probability of every token
    and the gradients of a weighted sum of them), "score" (the log-probabilities alone)."""
    return {"name": name, "op": "loss", "tokens": tokens, "vocab": vocab, "hidden": hidden,
            "mode": mode, "ignored": ignored, "smoothing": smoothing, "z_loss": z_loss,
            "scale": scale}


def _join(name, tokens, hidden, dtype, grad, post=True, gate=True, p=0.0, scale=1.0, norm=True):
    """grad: the forward and its gradients, or the forward alone; post: the branch is
    normalised; gate: a learned gate of each channel; norm: the next block's norm follows."""
    return {"name": name, "op": "join", "tokens": tokens, "hidden": hidden, "dtype": dtype,
            "grad": grad, "post": post, "gate": gate, "p": p, "scale": scale, "norm": norm}


def _drop(name, tokens, hidden, dtype, p):
    return {"name": name, "op": "dropout", "tokens": tokens, "hidden": hidden, "dtype": dtype,
            "p": p}


def listed():
    return [
        # the training loss of the 200M model's step: 16 sequences of 2048 tokens
        _loss("loss_200m", 32768, 32000, 896, "mean"),
        # the 7B preset's loss over one sequence: wide rows, 100000 words
        _loss("loss_7b", 4096, 100000, 4096, "mean"),
        # a packed batch with prompt tokens ignored, smoothing, z-loss, a muP logit scale and a
        # vocabulary that is no multiple of anything
        _loss("loss_regularised", 3001, 50021, 1024, "mean", ignored=0.4, smoothing=0.1,
              z_loss=1e-4, scale=0.25),
        # policy-gradient fine-tuning: log-probabilities of sampled tokens and their gradients
        _loss("logprobs_policy", 4095, 32000, 2048, "rows", ignored=0.25, scale=1.25),
        # scoring the choices of one question: few tokens, no gradient; latency
        _loss("logprobs_score", 19, 32000, 896, "score"),
        # a unit-test-sized model's training step: latency
        _loss("loss_small", 65, 1000, 72, "mean", ignored=0.1),
        # one join of the 200M model's training step, with everything on
        _join("join_200m", 32768, 896, "bf16", True, p=0.1, scale=0.5),
        # one join of a wide model's training step, no dropout
        _join("join_wide", 8191, 4096, "bf16", True),
        # serving: a decode batch of 64 requests; latency
        _join("join_decode", 64, 4096, "bf16", False),
        # an fp32 experiment of odd width, without the branch's norm
        _join("join_odd", 1003, 1111, "fp32", True, post=False, p=0.2),
        # embedding dropout of the 200M model's step
        _drop("dropout_200m", 32768, 896, "bf16", 0.1),
        # dropout inside a small encoder, odd width
        _drop("dropout_small", 77, 515, "fp16", 0.05),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "loss", "loss", "join", "join", "dropout"])
    if op == "loss":
        mode = rng.choice(["mean", "mean", "rows", "score"])
        hidden = 8 * _log(rng, 8, 512)
        vocab = _log(rng, 300, 60000)
        most = min(16384, (4096 * 60000 * 2048) // (hidden * vocab))
        tokens = _log(rng, 1, most if mode != "score" else min(most, 4096))
        c = _loss("", tokens, vocab, hidden, mode, ignored=rng.choice([0.0, 0.0, 0.3, 0.9]),
                  scale=rng.choice([1.0, 1.0, 0.5, 1.4]))
        if mode == "mean":
            c["smoothing"] = rng.choice([0.0, 0.0, 0.05, 0.2])
            c["z_loss"] = rng.choice([0.0, 0.0, 1e-4, 1e-3])
    else:
        hidden = rng.choice([_log(rng, 24, 8192), 8 * _log(rng, 8, 1024), 128 * rng.randint(1, 32)])
        tokens = _log(rng, 1, max(1, min(40000, (1 << 25) // hidden)))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        p = rng.choice([0.0, 0.05, 0.1, 0.5])
        if op == "dropout":
            c = _drop("", tokens, hidden, dtype, p if p > 0 else 0.3)
        else:
            c = _join("", tokens, hidden, dtype, rng.random() < 0.75, post=rng.random() < 0.7,
                      gate=rng.random() < 0.7, p=p, scale=rng.choice([1.0, 0.5, 0.2236]),
                      norm=rng.random() < 0.8)
    del c["name"]
    return c


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    T, H = case["tokens"], case["hidden"]
    st = {"case": case}
    if case["op"] == "loss":
        V = case["vocab"]
        # word frequencies fall off as 1 / rank^1.1 (the inverse of the distribution at u)
        u = torch.rand(T, generator=gen, device="cuda", dtype=torch.float64)
        y = (1 - u * (1 - (V + 1.0) ** -0.1)).pow(-10).long().sub_(1).clamp_(0, V - 1)
        w = normal(V, H).mul_(2.0 / math.sqrt(H)).bfloat16()
        # normalised hidden states that lean towards their next word, some more than others
        h = normal(T, H)
        h += (torch.rand(T, 1, generator=gen, device="cuda") * 2.0) * w[y].float()
        h *= torch.rsqrt(h.pow(2).mean(-1, keepdim=True))
        if case["ignored"] > 0:
            y[torch.rand(T, generator=gen, device="cuda") < case["ignored"]] = IGNORE
        st.update(h=h.bfloat16(), w=w, y=y)
        if case["mode"] == "rows":  # advantages
            st["g"] = normal(T)
        if case["mode"] != "score":
            st["h"].requires_grad_()
            st["w"].requires_grad_()
        return st
    dt = DTYPES[case["dtype"]]
    st["seed"] = torch.randint(-2 ** 62, 2 ** 62, (1,), generator=gen, device="cuda")
    if case["op"] == "dropout":
        st["x"] = normal(T, H).to(dt).requires_grad_()
        st["dy"] = normal(T, H).to(dt)
        return st
    # a residual stream has a few channels of larger magnitude
    chan = torch.ones(H, device="cuda")
    chan[torch.randperm(H, generator=gen, device="cuda")[:max(1, H // 64)]] = 8.0
    st["x"] = (normal(T, H) * chan).to(dt)
    st["b"] = (normal(T, H) * 0.7).to(dt)
    for key, on in (("w1", case["post"]), ("gate", case["gate"]), ("w2", case["norm"])):
        st[key] = (1.0 + 0.2 * normal(H)).to(dt) if on else None
    if case["grad"]:
        st["dx"] = normal(T, H).to(dt)
        st["dy"] = normal(T, H).to(dt) if case["norm"] else None
        for key in ("x", "b", "w1", "gate", "w2"):
            if st[key] is not None:
                st[key].requires_grad_()
    return st


# ------------------------------------------------------------ plain forms, 32 bits
def _wide(a, b):
    """High and low 32 bits of a 32-bit constant times 32-bit values held in int64."""
    lo = (b & 0xFFFF) * a
    hi = (b >> 16) * a
    mid = (lo >> 16) + (hi & 0xFFFF)
    return (hi >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)


def _random16(seed, blocks):
    """Philox4x32-10: 16 random bits for each of 8 elements of ``blocks`` blocks, [blocks, 8].
    The key is the seed, the counter (block, 0)."""
    s = seed.reshape(())
    k0, k1 = s & 0xFFFFFFFF, (s >> 32) & 0xFFFFFFFF
    n = torch.arange(blocks, device=seed.device, dtype=torch.int64)
    c0, c1 = n & 0xFFFFFFFF, n >> 32
    c2, c3 = torch.zeros_like(n), torch.zeros_like(n)
    for _ in range(10):
        h0, l0 = _wide(0xD2511F53, c0)
        h1, l1 = _wide(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([v for c in (c0, c1, c2, c3) for v in (c & 0xFFFF, c >> 16)], -1)


def _factor(seed, p, rows, cols):
    """0 for what is dropped, 1 / (kept share) for what is kept, [rows, cols] in 32 bits."""
    t = int(p * 65536 + 0.5)
    u = _random16(seed, -(-rows * cols // 8)).reshape(-1)[:rows * cols].view(rows, cols)
    return (u >= t).float() * (65536.0 / (65536 - t))


def _plain_loss(st):
    c = st["case"]
    h, w, y = st["h"].detach().float(), st["w"].detach().float(), st["y"]
    V, s, e, lam = c["vocab"], c["scale"], c["smoothing"], c["z_loss"]
    z = torch.matmul(h, w.t())
    if s != 1.0:
        z *= s
    top = z.amax(-1, keepdim=True)
    lse = (z - top).exp_().sum(-1, keepdim=True).log() + top
    valid = y != IGNORE
    at = torch.where(valid, y, torch.zeros_like(y))[:, None]
    zy = z.gather(1, at)
    loss = lse - (1 - e) * zy + lam * lse * lse
    if e > 0:
        loss = loss - e * z.mean(-1, keepdim=True)
    loss = torch.where(valid[:, None], loss, torch.zeros_like(loss))[:, 0]
    if c["mode"] == "score":
        return -loss
    n = valid.sum().clamp_min(1)
    g = valid / n if c["mode"] == "mean" else torch.where(valid, -st["g"], torch.zeros_like(st["g"]))
    g = g[:, None]
    z.sub_(lse).exp_().mul_(g * (1 + 2 * lam * lse))
    if e > 0:
        z.sub_(g * (e / V))
    z.scatter_add_(1, at, -(1 - e) * g)
    if s != 1.0:
        z *= s
    dh, dw = torch.matmul(z, w), torch.matmul(z.t(), h)
    out = loss.sum() / n if c["mode"] == "mean" else -loss
    return out, dh.bfloat16(), dw.bfloat16()


def _plain_join(st):
    c = st["case"]
    dt = DTYPES[c["dtype"]]
    f = {k: None if st[k] is None else st[k].detach().float() for k in ("x", "b", "w1", "gate", "w2")}
    x, b, w1, gate, w2 = f["x"], f["b"], f["w1"], f["gate"], f["w2"]
    H, s = c["hidden"], c["scale"]
    m = _factor(st["seed"], c["p"], *x.shape) if c["p"] > 0 else None
    if w1 is not None:
        r1 = torch.rsqrt(b.pow(2).sum(-1, keepdim=True) / H + EPS)
        bh = b * r1
        n = bh * w1
    else:
        n = b
    u = n if gate is None else n * gate
    if m is not None:
        u = u * m
    new = x + s * u
    out = [new.to(dt)]
    if w2 is not None:
        r2 = torch.rsqrt(new.pow(2).sum(-1, keepdim=True) / H + EPS)
        xh = new * r2
        out.append((xh * w2).to(dt))
    if not c["grad"]:
        return out
    g = st["dx"].float()
    dw2 = None
    if w2 is not None:
        dy = st["dy"].float()
        dw2 = (dy * xh).sum(0)
        dn = dy * w2
        g = g + r2 * (dn - xh * ((dn * xh).sum(-1, keepdim=True) / H))
    t = g * s
    if m is not None:
        t = t * m
    out += [g.to(dt)]
    dgate = (t * n).sum(0) if gate is not None else None
    if gate is not None:
        t = t * gate
    dw1 = None
    if w1 is not None:
        dw1 = (t * bh).sum(0)
        dn = t * w1
        t = r1 * (dn - bh * ((dn * bh).sum(-1, keepdim=True) / H))
    out.append(t.to(dt))
    out += [v.to(dt) for v in (dw1, dgate, dw2) if v is not None]
    return out


def _plain_dropout(st):
    c = st["case"]
    x, dy = st["x"].detach(), st["dy"]
    m = _factor(st["seed"], c["p"], *x.shape)
    return (x.float() * m).to(x.dtype), (dy.float() * m).to(dy.dtype)


# ------------------------------------------------------------------ one pass
def _own_loss(st):
    from complexity_framework_b200.ops.vocab_loss import token_logprobs, vocab_cross_entropy

    c = st["case"]
    if c["mode"] == "mean":
        out = vocab_cross_entropy(st["h"], st["w"], st["y"], ignore_index=IGNORE,
                                  label_smoothing=c["smoothing"], z_loss=c["z_loss"],
                                  logit_scale=c["scale"])
        return (out.detach(), *torch.autograd.grad(out, (st["h"], st["w"])))
    out = token_logprobs(st["h"], st["w"], st["y"], ignore_index=IGNORE, logit_scale=c["scale"])
    if c["mode"] == "score":
        return out
    return (out.detach(), *torch.autograd.grad(out, (st["h"], st["w"]), st["g"]))


def _own_join(st):
    from complexity_framework_b200.ops.residual import residual_norm

    c = st["case"]
    new, y = residual_norm(st["x"], st["b"], branch_weight=st["w1"], gate=st["gate"],
                           norm_weight=st["w2"], scale=c["scale"], p=c["p"],
                           seed=st["seed"] if c["p"] > 0 else None, eps=EPS)
    outs = [new] if y is None else [new, y]
    if not c["grad"]:
        return outs
    leaves = [st[k] for k in ("x", "b", "w1", "gate", "w2") if st[k] is not None]
    grads = [st["dx"]] if y is None else [st["dx"], st["dy"]]
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, grads))


def _own_dropout(st):
    from complexity_framework_b200.ops.residual import dropout

    y = dropout(st["x"], st["case"]["p"], st["seed"])
    return y.detach(), torch.autograd.grad(y, st["x"], st["dy"])[0]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"loss": _own_loss, "join": _own_join, "dropout": _own_dropout}[op](state)
    return {"loss": _plain_loss, "join": _plain_join, "dropout": _plain_dropout}[op](state)


# ------------------------------------------------------- definition, 64 bits
def _exact_loss(st):
    """Log-probabilities and gradients a few rows at a time, through log_softmax in 64 bits."""
    c = st["case"]
    h, w, y = st["h"].detach().double(), st["w"].detach().double(), st["y"]
    T, V, s, e = c["tokens"], c["vocab"], c["scale"], c["smoothing"]
    valid = y != IGNORE
    n = max(1, int(valid.sum()))
    rows = torch.zeros(T, device="cuda", dtype=torch.float64)
    dh = torch.zeros_like(h)
    dw = torch.zeros_like(w) if c["mode"] != "score" else None
    step = max(1, (1 << 27) // V)
    for a in range(0, T, step):
        ok = valid[a:a + step]
        at = y[a:a + step].clamp_min(0)[:, None]
        z = (h[a:a + step] @ w.t()) * s
        logp = torch.log_softmax(z, -1)
        lse = z[:, :1] - logp[:, :1]
        q = torch.full_like(z, e / V)                      # the smoothed target distribution
        q.scatter_add_(1, at, torch.full_like(at, 1 - e, dtype=torch.float64))
        value = -(q * logp).sum(-1) + c["z_loss"] * lse[:, 0] ** 2
        rows[a:a + step] = torch.where(ok, value, 0.0)
        if dw is None:
            continue
        p = logp.exp()
        dz = p - q + (2 * c["z_loss"]) * lse * p
        up = ok / n if c["mode"] == "mean" else torch.where(ok, -st["g"][a:a + step].double(), 0.0)
        dz *= s * up[:, None]
        dh[a:a + step] = dz @ w
        dw += dz.t() @ h[a:a + step]
    if c["mode"] == "score":
        return -rows
    return rows.sum() / n if c["mode"] == "mean" else -rows, dh, dw


def _keep64(seed, p, rows, cols):
    """The generator on the CPU, in numpy's unsigned 64-bit arithmetic."""
    import numpy as np

    key = int(seed.item()) & 0xFFFFFFFFFFFFFFFF
    n = np.arange(-(-rows * cols // 8), dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    c = [n & low, n >> np.uint64(32), np.zeros_like(n), np.zeros_like(n)]
    for i in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        k0 = np.uint64(((key & 0xFFFFFFFF) + i * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = np.uint64(((key >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k0, b & low, (a >> np.uint64(32)) ^ c[3] ^ k1, a & low]
    u = np.stack([v.astype(np.uint32) for v in c], -1).view(np.uint16)
    t = int(p * 65536 + 0.5)
    kept = torch.from_numpy(u.reshape(-1)[:rows * cols] >= t).cuda().view(rows, cols)
    return kept.double() * (65536 / (65536 - t))


def _exact_join(st):
    c = st["case"]
    leaf = {k: None if st[k] is None else st[k].detach().double().requires_grad_(c["grad"])
            for k in ("x", "b", "w1", "gate", "w2")}
    u = leaf["b"]
    if leaf["w1"] is not None:
        u = leaf["w1"] * (u / (u.square().mean(-1, keepdim=True) + EPS).sqrt())
    if leaf["gate"] is not None:
        u = u * leaf["gate"]
    if c["p"] > 0:
        u = u * _keep64(st["seed"], c["p"], *u.shape)
    new = leaf["x"] + c["scale"] * u
    outs, ups = [new], [st.get("dx")]
    if leaf["w2"] is not None:
        outs.append(leaf["w2"] * (new / (new.square().mean(-1, keepdim=True) + EPS).sqrt()))
        ups.append(st.get("dy"))
    if not c["grad"]:
        return outs
    leaves = [v for v in leaf.values() if v is not None]
    grads = torch.autograd.grad(outs, leaves, [g.double() for g in ups])
    return [o.detach() for o in outs] + list(grads)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "loss":
        return _exact_loss(st)
    if case["op"] == "join":
        return _exact_join(st)
    m = _keep64(st["seed"], case["p"], *st["x"].shape)
    return st["x"].detach().double() * m, st["dy"].double() * m


# ------------------------------------------------------------ bytes and operations
def work(case):
    T, H = case["tokens"], case["hidden"]
    if case["op"] == "loss":
        V, grad = case["vocab"], case["mode"] != "score"
        # three products with a gradient, one without (computing the logits a second time,
        # which not keeping them costs, is not counted)
        b = 2 * (T * H + V * H) * (2 if grad else 1) + 8 * T + (4 if case["mode"] == "mean" else 4 * T)
        if case["mode"] == "rows":
            b += 4 * T
        return {"bytes": b, "flops": (6 if grad else 2) * T * V * H}
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "dropout":
        return {"bytes": 4 * T * H * size, "flops": 2 * T * H}
    weights = case["post"] + case["gate"] + case["norm"]
    rows = 3 + case["norm"]                   # x, branch, the new stream, its norm
    if case["grad"]:
        rows += 3 + case["norm"]              # their gradients: dx', dy read; dx, dbranch written
        weights *= 2
    return {"bytes": (rows * T + weights) * H * size, "flops": (30 if case["grad"] else 10) * T * H}
