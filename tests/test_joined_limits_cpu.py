"""Loss options and joined residuals on the paths beside the plain model: sequence-parallel and
pipeline losses, data-parallel ranks, resumed runs, exports."""
import types

import pytest
import torch
import torch.nn.functional as F

from complexity_framework_b200 import ComplexityModel
from complexity_framework_b200.config import ModelConfig


def tiny(**kw):
    base = dict(hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                intermediate_size=64, shared_intermediate_size=64, vocab_size=97, num_experts=2,
                top_k=2, max_position_embeddings=64)
    base.update(kw)
    torch.manual_seed(0)
    return ComplexityModel(ModelConfig(**base))


FULL = dict(norm_placement="sandwich", residual_gate_init=0.5, residual_scale=0.7)
MUP = dict(use_mup_output_mult=True, mup_base_width=16)  # logits times 1 / 4


# ------------------------------------------------------------- the logit scale
def test_sequence_parallel_loss_scales_the_logits():
    """The sequence-parallel loss of one rank that holds every token is the model's loss."""
    m = tiny(**MUP).train()
    with torch.no_grad():
        m.embed_tokens.weight.mul_(50)  # logits large enough that their scale matters
    ids = torch.randint(0, 97, (2, 9))
    m.sp_ws = types.SimpleNamespace(world=1, rank=0, begin_step=lambda: None)
    for layer in m.layers:
        layer.forward_sp = lambda x, ids, B, S, ws, f=layer: f(
            x.view(B, S, -1), token_ids=ids)[0].view(B * S, -1)
    for kw in ({}, dict(label_smoothing=0.1, z_loss_coef=1e-2)):
        torch.testing.assert_close(m._loss_sp(ids, None, -100, **kw), m.loss(ids, **kw))


def test_pipeline_stage_loss_scales_the_logits():
    from complexity_framework_b200.parallel.pipeline_parallel import PipelineStage

    m = tiny(**MUP)
    with torch.no_grad():
        m.embed_tokens.weight.mul_(50)
    ids = torch.randint(0, 97, (2, 9))
    stage = PipelineStage(m, 0, 2, True, True)
    torch.testing.assert_close(stage.loss(stage(None, ids), ids), m.loss(ids))


def test_weighted_fine_tuning_loss_scales_the_logits():
    from complexity_framework_b200.training.sft import weighted_sft_loss

    m = tiny(**MUP)
    with torch.no_grad():
        m.embed_tokens.weight.mul_(50)
    ids = torch.randint(0, 97, (2, 9))
    labels = torch.randint(0, 97, (2, 9))
    labels[0, :3] = -100
    ones = torch.ones(2, 9, dtype=torch.long)
    got = weighted_sft_loss(m, ids, torch.stack((labels, ones), -1))
    torch.testing.assert_close(got, m.loss(ids, labels))


# -------------------------------------------------------- dropout across ranks
def test_embedding_dropout_is_refused_under_tensor_parallelism():
    """The ranks of a group hold one replicated stream, which different masks would part."""
    m = tiny(embedding_dropout=0.1).train()
    m.tp_group = object()
    with pytest.raises(NotImplementedError, match="embedding_dropout under tensor parallelism"):
        m(torch.randint(0, 97, (1, 4)))
    m.eval()
    m(torch.randint(0, 97, (1, 4)))


def _rank_masks(rank, port, out):
    import torch.distributed as dist

    from complexity_framework_b200.core.layers import ResidualJoin

    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    try:
        out[rank] = _masks(ResidualJoin)
    finally:
        dist.destroy_process_group()


def _masks(ResidualJoin):
    """What a join and a model's embedding dropout keep, under one seed."""
    torch.manual_seed(3)
    x = torch.zeros(16, 64)
    join = ResidualJoin(64, norm=False, p=0.5).train()(x, torch.ones(16, 64))[0]
    m = tiny(embedding_dropout=0.5).train()
    kept = []
    m.layers[0].register_forward_pre_hook(lambda _, args: kept.append(args[0] != 0))
    m(torch.arange(8).view(1, 8))
    return (join != 0).tolist(), kept[0].tolist()


def test_data_parallel_ranks_draw_masks_of_their_own():
    """Ranks that are seeded alike, as the training scripts seed them."""
    import socket

    import torch.multiprocessing as mp

    from complexity_framework_b200.core.layers import ResidualJoin

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    with ctx.Manager() as manager:
        out = manager.dict()
        procs = [ctx.Process(target=_rank_masks, args=(r, port, out)) for r in range(2)]
        for p in procs:
            p.start()
        for p in procs:
            p.join(180)
        assert [p.exitcode for p in procs] == [0, 0]
        a, b = out[0], out[1]
    for i in range(2):
        assert a[i] != b[i]
    assert a == _masks(ResidualJoin)  # the first rank's are those of a process by itself


# ------------------------------------------------------------------ resumed runs
def test_resumed_run_goes_on_with_the_masks(tmp_path):
    """Two steps, a checkpoint and two more steps of another process are four steps of one."""
    from complexity_framework_b200.training import Trainer, TrainingConfig

    ids = torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(1))

    def trainer():
        m = tiny(residual_dropout=0.3, embedding_dropout=0.2, **FULL)
        return Trainer(m, TrainingConfig(max_steps=8, learning_rate=1e-3, precision="fp32",
                                         warmup_steps=0, checkpoint_dir=str(tmp_path)),
                       device=torch.device("cpu"))

    a = trainer()
    for _ in range(2):
        a.train_step(ids)
    a.save_checkpoint()
    want = [a.train_step(ids) for _ in range(2)]
    b = trainer()
    torch.manual_seed(77)
    assert b.resume("auto") and b.global_step == 2
    assert [b.train_step(ids) for _ in range(2)] == want
    # a checkpoint without the generators' state, as older ones are, still resumes
    for f in tmp_path.glob("*/rng_rank*.pt"):
        f.unlink()
    assert trainer().resume("auto")


# ------------------------------------------------------------- scoring of choices
class _Words:
    pad_token_id = 0

    @staticmethod
    def encode(text):
        return [int(t) for t in text.split()]


def test_choices_without_a_context():
    """The first token of a sequence follows nothing and is not scored."""
    from complexity_framework_b200.evaluation.benchmarks import choice_logprobs

    m = tiny().eval()
    with torch.no_grad():
        lp = torch.log_softmax(m(torch.tensor([[5, 6, 7]]))["logits"][0], -1)
        one = float(lp[0, 6])
        two = one + float(lp[1, 7])
    for normalize, want in ((False, [one, two]), (True, [one, two / 2])):
        got = choice_logprobs(m, _Words, "", ["5 6", "5 6 7"], normalize)
        assert got == pytest.approx(want, abs=1e-5)
    with pytest.raises(ValueError, match="nothing to score"):
        choice_logprobs(m, _Words, "", ["5", "5 6"])
    want = choice_logprobs(m, _Words, "5", ["6", "6 7"])
    assert want == pytest.approx([one, two / 2], abs=1e-5)


# ---------------------------------------------------------------- joins in a model
@pytest.mark.parametrize("stream,weights", [(torch.bfloat16, torch.float32),
                                            (torch.float32, torch.bfloat16)])
def test_join_with_weights_of_another_type(stream, weights):
    """The wider type of the two, as the plain norms compute."""
    from complexity_framework_b200.core.layers import ResidualJoin, RMSNorm

    torch.manual_seed(0)
    j = ResidualJoin(8, gate_init=0.7).to(weights).eval()
    j.weight.data.add_(0.1 * torch.randn(8))
    n = RMSNorm(8).to(weights)
    x, b = torch.randn(3, 8).to(stream), torch.randn(3, 8).to(stream)
    new, y = j(x, b, n)
    want = ResidualJoin(8, gate_init=0.7).eval()
    want.load_state_dict({k: v.float() for k, v in j.state_dict().items()})
    a, c = want(x.float(), b.float(), RMSNorm(8))
    assert new.dtype == y.dtype == torch.float32
    torch.testing.assert_close(new, a)
    torch.testing.assert_close(y, c)


# ------------------------------------------------------------------------- exports
def test_exports_ask_the_model_about_its_joins(tmp_path):
    """A configuration that is handed over may be any object with the layout's fields; what the
    layout cannot hold is the model's."""
    from complexity_framework_b200.quantization.gguf import export_gguf
    from complexity_framework_b200.utils.conversion import save_to_huggingface

    m = tiny(tie_word_embeddings=False)
    fields = {k: v for k, v in m.config.to_dict().items()
              if not k.startswith("residual") and k not in ("norm_placement", "embedding_dropout")}
    plain = types.SimpleNamespace(**fields)
    save_to_huggingface(m, str(tmp_path / "a"), config=plain)
    m.config = plain
    export_gguf(m, tmp_path / "m.gguf")
    with pytest.raises(ValueError, match="branches"):
        save_to_huggingface(tiny(**FULL), str(tmp_path / "b"), config=plain)


def test_pipeline_stage_of_a_model_with_a_plain_configuration():
    from complexity_framework_b200.parallel.pipeline_parallel import PipelineStage

    m = tiny()
    m.config = types.SimpleNamespace(hidden_size=64, num_hidden_layers=2)
    PipelineStage(m, 0, 1, True, False)


# ------------------------------------------------------------------ training options
def test_loss_options_beside_a_loss_of_ones_own_are_told(caplog):
    from complexity_framework_b200.training import Trainer, TrainingConfig

    def own(model, ids, labels):
        return model.loss(ids, labels)

    kw = dict(device=torch.device("cpu"), compute_loss=own)
    for opt in (dict(label_smoothing=0.1), dict(z_loss_coef=1e-4)):
        caplog.clear()
        Trainer(tiny(), TrainingConfig(precision="fp32", **opt), **kw)
        assert "compute_loss" in caplog.text and next(iter(opt)) in caplog.text
    caplog.clear()
    Trainer(tiny(), TrainingConfig(precision="fp32"), **kw)
    assert "compute_loss" not in caplog.text
