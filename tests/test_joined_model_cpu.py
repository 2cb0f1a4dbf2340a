"""Models whose branches join the residual stream through norms, gates and dropout, smoothed
losses and log-probabilities without logits: CPU paths."""
import pytest
import torch
import torch.nn.functional as F

from complexity_framework_b200 import ComplexityModel
from complexity_framework_b200.config import ModelConfig
from complexity_framework_b200.core.layers import ResidualJoin, RMSNorm
from complexity_framework_b200.core.losses import (causal_lm_loss, causal_lm_loss_from_hidden,
                                                   model_token_logprobs)
from complexity_framework_b200.rl.grpo import sequence_log_probs
from complexity_framework_b200.training import TrainingConfig


def tiny(**kw):
    base = dict(hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                intermediate_size=64, shared_intermediate_size=64, vocab_size=97, num_experts=2,
                top_k=2, max_position_embeddings=64)
    base.update(kw)
    torch.manual_seed(0)
    return ComplexityModel(ModelConfig(**base))


FULL = dict(norm_placement="sandwich", residual_gate_init=0.5, residual_scale=0.7)


def test_defaults_are_plain_blocks():
    m = tiny()
    assert not m.config.joined_residual and not any("join" in k for k in m.state_dict())


def test_block_is_its_formula():
    m = tiny(**FULL).eval()
    for p in m.parameters():
        if p.dim() == 1:
            p.data.add_(0.1 * torch.randn_like(p))
    block, x = m.layers[0], torch.randn(2, 5, 64)
    ids = torch.randint(0, 97, (2, 5))

    def rms(v, w):
        return w * v * torch.rsqrt(v.square().mean(-1, keepdim=True) + m.config.norm_eps)

    a = block.self_attn(block.input_layernorm(x))[0]
    j = block.attn_join
    y = x + 0.7 * j.gate * rms(a, j.weight)
    b = block.mlp(rms(y, block.post_attention_layernorm.weight), token_ids=ids)
    j = block.mlp_join
    want = y + 0.7 * j.gate * rms(b, j.weight)
    torch.testing.assert_close(block(x, token_ids=ids)[0], want, rtol=1e-5, atol=1e-5)


def test_every_parameter_learns():
    m = tiny(residual_dropout=0.1, embedding_dropout=0.1, **FULL).train()
    ids = torch.randint(0, 97, (2, 9))
    m.loss(ids, label_smoothing=0.1, z_loss_coef=1e-3).backward()
    for n, p in m.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()), n
        if "join" in n:
            assert float(p.grad.abs().max()) > 0, n


def test_dropout_is_for_training_and_repeats_under_a_seed():
    m = tiny(residual_dropout=0.3, embedding_dropout=0.2)
    ids = torch.randint(0, 97, (2, 9))
    m.eval()
    assert torch.equal(m(ids)["logits"], m(ids)["logits"])
    m.train()
    torch.manual_seed(5)
    a = m(ids)["logits"]
    b = m(ids)["logits"]
    torch.manual_seed(5)
    assert torch.equal(a, m(ids)["logits"]) and not torch.equal(a, b)


def test_recomputed_blocks_draw_the_same_masks():
    m = tiny(residual_dropout=0.3, **FULL).train()
    ids = torch.randint(0, 97, (2, 9))
    grads = []
    for ckpt in (False, True):
        (m.gradient_checkpointing_enable if ckpt else m.gradient_checkpointing_disable)()
        m.zero_grad()
        torch.manual_seed(7)
        m.loss(ids).backward()
        grads.append([p.grad.clone() for p in m.parameters()])
    for a, b in zip(*grads):
        torch.testing.assert_close(a, b)


def test_paged_decoding_follows_the_forward():
    m = tiny(**FULL).eval()
    prompt = [3, 14, 15, 92]
    out = m.generate(torch.tensor([prompt]), max_new_tokens=4)[0]
    ids = list(prompt)
    for _ in range(4):
        ids.append(int(m(torch.tensor([ids]))["logits"][0, -1].argmax()))
    assert out == ids


def test_decoding_drops_nothing_in_training_mode():
    from complexity_framework_b200.inference import beam_search

    m = tiny(residual_dropout=0.5, embedding_dropout=0.5, **FULL)
    want = beam_search(m.eval(), [3, 14, 15], num_beams=2, max_new_tokens=4)["tokens"]
    assert beam_search(m.train(), [3, 14, 15], num_beams=2, max_new_tokens=4)["tokens"] == want


def test_config_round_trip_and_refusals(tmp_path):
    m = tiny(residual_dropout=0.1, **FULL)
    m.save_pretrained(tmp_path)
    back = ComplexityModel.from_pretrained(tmp_path)
    assert back.config.joined_residual and back.config.residual_dropout == 0.1
    for (n, a), (_, b) in zip(m.state_dict().items(), back.state_dict().items()):
        assert torch.equal(a, b), n
    for bad in (dict(norm_placement="post"), dict(residual_dropout=1.0),
                dict(embedding_dropout=-0.1), dict(residual_scale=float("nan"))):
        with pytest.raises(ValueError):
            ModelConfig(**bad)
    with pytest.raises(ValueError, match="label_smoothing"):
        TrainingConfig(label_smoothing=2.0)
    with pytest.raises(NotImplementedError):
        m.layers[0].forward_sp(None, None, 1, 1, None)
    from complexity_framework_b200.quantization.gguf import export_gguf
    from complexity_framework_b200.utils.conversion import save_to_huggingface

    for export in (export_gguf, save_to_huggingface):
        with pytest.raises(ValueError, match="branches"):
            export(m, str(tmp_path / "x"))
    m.train()
    m.layers[0].self_attn.tp_group = object()
    with pytest.raises(NotImplementedError, match="tensor parallelism"):
        m.layers[0](torch.zeros(1, 2, 64), token_ids=torch.zeros(1, 2, dtype=torch.long))


def test_join_with_another_norm():
    j = ResidualJoin(8, gate_init=1.0).eval()
    x, b = torch.randn(3, 8), torch.randn(3, 8)
    ln = torch.nn.LayerNorm(8)
    new, y = j(x, b, ln)
    torch.testing.assert_close(y, ln(new))
    n = RMSNorm(8, eps=1e-3)  # an eps of its own is kept
    torch.testing.assert_close(j(x, b, n)[1], n(j(x, b)[0]))


@pytest.mark.parametrize("smooth,z,scale", [(0.1, 0.0, 1.0), (0.0, 1e-2, 0.5), (0.2, 1e-3, 1.0)])
def test_loss_options(smooth, z, scale):
    h = torch.randn(2, 7, 16, requires_grad=True)
    w = torch.randn(37, 16, requires_grad=True)
    y = torch.randint(0, 37, (2, 7))
    y[0, 3] = -100
    want, _ = causal_lm_loss((h @ w.t()) * scale, y, label_smoothing=smooth, z_loss_coef=z)
    for chunk in (3, 8192):
        got = causal_lm_loss_from_hidden(h, w, y, label_smoothing=smooth, z_loss_coef=z,
                                         logit_scale=scale, chunk_tokens=chunk)
        torch.testing.assert_close(got, want)
        for a, b in zip(torch.autograd.grad(got, (h, w)),
                        torch.autograd.grad(want, (h, w), retain_graph=True)):
            torch.testing.assert_close(a, b)


def test_logprobs():
    m = tiny(use_mup_output_mult=True, mup_base_width=32).eval()
    ids = torch.randint(0, 97, (2, 6))
    tgt = torch.roll(ids, -1, 1)
    tgt[:, -1] = -100
    lp = model_token_logprobs(m, ids, tgt)
    want = torch.log_softmax(m(ids)["logits"], -1).gather(-1, tgt.clamp_min(0)[..., None])[..., 0]
    torch.testing.assert_close(lp, torch.where(tgt == -100, 0.0, want))
    out, mask = sequence_log_probs(m, [[1, 2], [3], []], [[4, 5, 6], [7], [8, 9]])
    assert mask.tolist() == [[1, 1, 1], [1, 0, 0], [0, 1, 0]]
    full = torch.log_softmax(m(torch.tensor([[1, 2, 4, 5, 6]]))["logits"][0], -1)
    torch.testing.assert_close(out[0], full[[1, 2, 3], [4, 5, 6]])
    alone = torch.log_softmax(m(torch.tensor([[8, 9]]))["logits"][0], -1)
    torch.testing.assert_close(out[2, 1], alone[0, 9])
