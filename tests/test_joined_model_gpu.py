"""Models whose branches join the residual stream through norms, gates and dropout, with the
loss over the vocabulary without logits, on the kernels."""
import copy

import pytest
import torch

from complexity_framework_b200 import ComplexityModel
from complexity_framework_b200.config import ModelConfig
from complexity_framework_b200.core.losses import causal_lm_loss_from_hidden, model_token_logprobs
from complexity_framework_b200.ops import check_errors
from complexity_framework_b200.ops.residual import dropout, new_seed, residual_norm
from complexity_framework_b200.ops.vocab_loss import vocab_cross_entropy
from complexity_framework_b200.rl.grpo import sequence_log_probs
from complexity_framework_b200.training import Trainer, TrainingConfig

pytestmark = pytest.mark.gpu

FULL = dict(norm_placement="sandwich", residual_gate_init=0.5, residual_scale=0.7)


def model(**kw):
    base = dict(hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                intermediate_size=256, shared_intermediate_size=256, vocab_size=1000,
                num_experts=2, top_k=2, max_position_embeddings=256)
    base.update(kw)
    torch.manual_seed(0)
    return ComplexityModel(ModelConfig(**base)).to("cuda", torch.bfloat16)


def cosine(a, b):
    a, b = a.double().flatten(), b.double().flatten()
    return float(a @ b / (a.norm() * b.norm()))


def test_model_against_fp32():
    """The bf16 model on the kernels and its copy in fp32: every activation, weight gradient and
    product is rounded to 8 bits some 20 times on the way, each rounding off by 2^-8 at most and
    independent of the others, so gradients agree in direction to well within 1 - (20 * 2^-8)^2."""
    m = model(**FULL)
    ref = copy.deepcopy(m).float()
    ids = torch.randint(0, 1000, (2, 64), device="cuda")
    kw = dict(label_smoothing=0.1, z_loss_coef=1e-3)
    a, b = m.loss(ids, **kw), ref.loss(ids, **kw)
    a.backward()
    b.backward()
    assert abs(float(a.detach()) - float(b.detach())) <= 20 * 2.0 ** -8
    for (n, p), (_, q) in zip(m.named_parameters(), ref.named_parameters()):
        assert cosine(p.grad, q.grad) >= 1 - (20 * 2.0 ** -8) ** 2, n
    check_errors()


def test_operators_together():
    """Embedding dropout, two joins and the loss in a row, against the same in 64 bits with the
    masks that the seeds stand for (the bf16 run rounds five results on the way)."""
    torch.manual_seed(1)
    T, H, V = 130, 264, 777
    mk = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    leaves = {"x": mk(T, H), "b1": mk(T, H), "b2": mk(T, H), "w1": 1 + 0.1 * mk(H),
              "gate": 1 + 0.1 * mk(H), "w2": 1 + 0.1 * mk(H), "head": mk(V, H) * 0.1}
    y = torch.randint(0, V, (T,), device="cuda")
    y[::7] = -100
    seed = new_seed("cuda")

    def run(t, fp):
        g = {k: v.bfloat16().to(fp).requires_grad_() for k, v in t.items()}
        if fp == torch.bfloat16:
            h = dropout(g["x"], 0.1, seed)
            h, _ = residual_norm(h, g["b1"], branch_weight=g["w1"], gate=g["gate"], scale=0.5,
                                 p=0.2, seed=seed, stream=1)
            _, n = residual_norm(h, g["b2"], branch_weight=g["w1"], norm_weight=g["w2"], p=0.2,
                                 seed=seed, stream=2)
            loss = vocab_cross_entropy(n, g["head"], y, label_smoothing=0.1)
        else:
            c = {k: v.cpu() for k, v in g.items()}
            s = seed.cpu()
            h = dropout(c["x"], 0.1, s)
            h, _ = residual_norm(h, c["b1"], branch_weight=c["w1"], gate=c["gate"], scale=0.5,
                                 p=0.2, seed=s, stream=1)
            _, n = residual_norm(h, c["b2"], branch_weight=c["w1"], norm_weight=c["w2"], p=0.2,
                                 seed=s, stream=2)
            loss = vocab_cross_entropy(n, c["head"], y.cpu(), label_smoothing=0.1)
        return loss.detach(), torch.autograd.grad(loss, tuple(g.values()))

    a, ga = run(leaves, torch.bfloat16)
    b, gb = run(leaves, torch.float64)
    # the logits are sums of 264 products of about 1 x 0.1 with n off by 3 * 2^-8 at most
    assert abs(float(a) - float(b)) <= 3 * 2.0 ** -8 * 264 ** 0.5 * 0.1 * 4
    for k, p, q in zip(leaves, ga, gb):
        assert cosine(p, q) >= 1 - (8 * 2.0 ** -8) ** 2, k


@pytest.mark.parametrize("kw", [dict(vocab_size=1000), dict(vocab_size=1024, scale=0.5)])
def test_loss_where_the_fused_mean_does_not_apply(kw):
    V, s = kw["vocab_size"], kw.get("scale", 1.0)
    h = torch.randn(3, 50, 128, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(V, 128, device="cuda") * 0.1).bfloat16().requires_grad_()
    y = torch.randint(0, V, (3, 50), device="cuda")
    got = causal_lm_loss_from_hidden(h, w, y, logit_scale=s)
    want = torch.nn.functional.cross_entropy(
        (s * h.double() @ w.double().t()).view(-1, V), y.view(-1))
    # logits of some 4, 128-product sums in 32 bits
    assert abs(float(got.detach()) - float(want.detach())) <= 1e-4
    ga, gb = torch.autograd.grad(got, (h, w)), torch.autograd.grad(want, (h, w))
    for a, b in zip(ga, gb):
        assert cosine(a, b) >= 1 - (3 * 2.0 ** -8) ** 2


def test_logprobs_without_logits():
    m = model(use_mup_output_mult=True, mup_base_width=128).eval()
    with torch.no_grad():
        lp, mask = sequence_log_probs(m, [[5, 6, 7], [8]], [[9, 10], [11, 12, 13]])
        ids = torch.tensor([[5, 6, 7, 9, 10], [8, 11, 12, 13, 0]], device="cuda")
        hidden = m(ids, return_logits=False)["last_hidden_state"].double()
        full = torch.log_softmax(hidden @ m.output_weight().double().t() * 0.5, -1)
    assert abs(float(lp[0, 1]) - float(full[0, 3, 10])) <= 1e-4
    assert abs(float(lp[1, 2]) - float(full[1, 2, 13])) <= 1e-4
    assert mask.tolist() == [[1, 1, 0], [1, 1, 1]]
    tgt = torch.randint(0, 1000, (2, 5), device="cuda")
    model_token_logprobs(m, ids, tgt).sum().backward()
    assert m.embed_tokens.weight.grad is not None
    check_errors()


def test_decoding_follows_the_forward():
    m = model(**FULL).eval()
    prompt = [3, 14, 159, 265, 358]
    out = m.generate(torch.tensor([prompt]), max_new_tokens=6)[0]
    with torch.no_grad():
        lg = m(torch.tensor([out[:-1]], device="cuda"))["logits"][0].float()
    for i in range(len(prompt), len(out)):
        row = lg[i - 1]  # the chosen word's logit is the largest, up to rounding of 8-bit logits
        assert float(row.max() - row[out[i]]) <= 2.0 ** -6 * max(1.0, float(row.abs().max()))


def test_recomputed_blocks_draw_the_same_masks():
    m = model(residual_dropout=0.3, embedding_dropout=0.1, **FULL).train()
    ids = torch.randint(0, 1000, (2, 64), device="cuda")
    grads = []
    for ckpt in (False, True, True):
        (m.gradient_checkpointing_enable if ckpt else m.gradient_checkpointing_disable)()
        m.zero_grad()
        torch.manual_seed(7)
        m.loss(ids, label_smoothing=0.1).backward()
        grads.append([p.grad.clone() for p in m.parameters()])
    # the model's other kernels add some gradients by atomics: equal up to roundings to 8 bits
    for a, b, c in zip(*grads):
        assert cosine(a, b) >= 1 - (4 * 2.0 ** -8) ** 2 and cosine(b, c) >= 1 - (4 * 2.0 ** -8) ** 2


@pytest.mark.parametrize("graph", [False, True])
def test_training_steps(graph):
    m = model(residual_dropout=0.2, embedding_dropout=0.1, **FULL)
    tr = Trainer(m, TrainingConfig(learning_rate=0.0 + 1e-8, precision="bf16", grad_clip=1.0,
                                   warmup_steps=0, lr_scheduler="constant", weight_decay=0.0,
                                   cuda_graph=graph, label_smoothing=0.1, z_loss_coef=1e-4,
                                   skip_param_update_check=True))
    ids = torch.randint(0, 1000, (2, 64)).pin_memory()
    losses = [tr.train_step(ids) for _ in range(8)]
    assert all(v == v and v < 20 for v in losses)
    assert len(set(losses)) >= 7  # every step draws other masks, replayed ones too
    check_errors()
