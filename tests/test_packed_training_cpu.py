"""A model on packed documents -- lookup with positions that start again, attention inside the documents, loss without
logits -- gives the loss and the gradients of the documents one by one through the separate steps."""
import pytest
import torch

from mist_b200.config import ModelConfig
from mist_b200.models.provider import base_model_provider
from mist_b200.modules.layers import ParallelMHA
from mist_b200.ops import functional as F

LENS = [9, 1, 20, 0, 14]
CU = [0, 9, 10, 30, 30, 44]
BASE = dict(hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, max_position_embeddings=32,
            vocab_size=250, params_dtype="float32", add_encoder=True, add_decoder=False, use_flash_attn=True)
FAMILIES = {
    "gpt": dict(name="gpt2-t", encoder_attn_mask_type="causal"),
    "gpt_tied": dict(name="gpt2-t", encoder_attn_mask_type="causal", tie_word_embeddings=True),
    "llama": dict(name="llama-t", encoder_attn_mask_type="causal", mlp_type="gated_mlp", normalization="rmsnorm",
                  position_embedding_type="rotary", rotary_emb_fraction=1.0, num_heads_kv=2),
    "falcon": dict(name="falcon-t", encoder_attn_mask_type="causal", parallel_block=True, position_embedding_type="rotary",
                   rotary_emb_fraction=0.5),
    "bert": dict(name="bert-t", encoder_attn_mask_type="padding", num_tokentypes=2),
}


def build(family, device="cpu", dtype=torch.float32, **more):
    torch.manual_seed(0)
    return base_model_provider(ModelConfig(**{**BASE, **FAMILIES[family], **more}), device=device, dtype=dtype)


def batch(rows, device="cpu", vocab=250, total=48, ends=CU):
    """Ids and labels of ``rows`` rows of tokens in all; the last token of a document and the padding carry no label."""
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, vocab, (rows, total // rows), generator=g)
    labels = torch.randint(0, vocab, (total,), generator=g)
    labels[[e - 1 for e in ends if e]] = -100
    labels[ends[-1]:] = -100
    return ids.to(device), labels.view(ids.shape).to(device)


def labelled(family):
    return "lm_labels" if family == "bert" else "labels"


def one_by_one(model, family, ids, labels, ends=CU):
    ids, labels, loss = ids.reshape(1, -1), labels.reshape(1, -1), 0.0
    for a, b in zip(ends, ends[1:]):
        if b > a:
            loss = loss + model(ids[:, a:b], **{labelled(family): labels[:, a:b]}) * (b - a)
    return loss / ids.numel()


def gradients(model, loss):
    model.zero_grad()
    loss.backward()
    return {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("family", sorted(FAMILIES))
@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("recompute", [0, 1])
def test_packed_step_is_the_documents_one_by_one(family, rows, recompute):
    ids, labels = batch(rows)
    plain, fused = build(family), build(family, fused_lm_loss=True)
    fused.load_state_dict(plain.state_dict())
    fused.language_model.encoder.gradient_checkpointing = recompute
    want = one_by_one(plain, family, ids, labels)
    got = fused(ids, attention_mask=F.PackedSequences(CU, 48), **{labelled(family): labels})
    assert abs(got.item() - want.item()) < 1e-5
    a, b = gradients(fused, got), gradients(plain, want)
    assert set(a) == set(b)
    for n in a:
        assert torch.allclose(a[n], b[n], atol=1e-5, rtol=1e-4), n


@pytest.mark.parametrize("family", ["gpt", "t5"])
def test_fused_loss_alone(family):
    """Without packing the switch changes nothing but how the loss is computed."""
    from mist_b200.models.provider import get_inputs_provider
    FAMILIES.setdefault("t5", dict(name="t5-t", encoder_attn_mask_type="padding", decoder_attn_mask_type="causal",
                                   add_decoder=True))
    data = get_inputs_provider(FAMILIES[family]["name"])(2, 32, 250, "cpu", seed=3)
    plain, fused = build(family), build(family, fused_lm_loss=True)
    fused.load_state_dict(plain.state_dict())
    x, y = plain(**data), fused(**data)
    assert abs(x.item() - y.item()) < 1e-5
    a, b = gradients(plain, x), gradients(fused, y)
    assert all(torch.allclose(a[n], b[n], atol=1e-5, rtol=1e-4) for n in a) and set(a) == set(b)


def test_logits_are_the_same_without_labels():
    ids, _ = batch(1)
    plain, fused = build("gpt"), build("gpt", fused_lm_loss=True)
    fused.load_state_dict(plain.state_dict())
    assert torch.equal(plain(ids[:, :9]), fused(ids[:, :9]))
    packed = fused(ids, attention_mask=F.PackedSequences(CU, 48))
    assert torch.allclose(packed[:, 10:30], plain(ids[:, 10:30]), atol=1e-5)


def test_refusals():
    seqs = F.PackedSequences([0, 8])
    x = torch.randn(1, 8, 32)
    with pytest.raises(NotImplementedError):
        ParallelMHA(32, 4, causal=True, use_flash_attn=False)(x, attention_mask=seqs)
    with pytest.raises(NotImplementedError):
        ParallelMHA(32, 4, cross_attn=True)(x, x_kv=x, kv_mask=seqs)
    with pytest.raises(NotImplementedError):
        ParallelMHA(32, 4, causal=True, rotary_emb_dim=8, rotary_emb_interleaved=True)(x, attention_mask=seqs)
    with pytest.raises(ValueError):
        ParallelMHA(32, 4, causal=True)(x, attention_mask=F.PackedSequences([0, 7]))


@pytest.mark.parametrize("micro", [1, 2])
def test_a_session_takes_one_packing_per_micro_batch(micro):
    from mist_b200.api import TrainingSession
    from mist_b200.config import load_config
    vec = "[1,1,1,0,0,0,0,0,0,0]"
    cfg, _ = load_config("config", [
        "experiment=gpt2-1.3b", "model=gpt2/1.3b", "model.params_dtype=float32", "training.params_dtype=float32",
        "hardware.num_gpus_per_node=1", "model.hidden_size=32", "model.intermediate_size=64", "model.num_attention_heads=4",
        "model.num_heads_kv=4", "model.num_hidden_layers=1", "model.vocab_size=256", "training.vocab_size=256",
        "training.max_sequence_length=24", f"training.global_batch_size={micro}", "strategy.layer_partitions=[1]",
        "strategy.device_assignment=[[1,1]]", "strategy.gradient_checkpointing=[0]",
        f"strategy.gradient_accumulation_steps={micro}", f"strategy.stage_strategies=[{vec}]",
        f"strategy.pre_post_strategy_array={vec}"], check_world_size=False)
    sess = TrainingSession(cfg, seed=3, device=torch.device("cpu"), hp=dict(lr=1e-3))
    ids = torch.randint(0, 256, (micro, 24), generator=torch.Generator().manual_seed(2))
    packings = [F.PackedSequences(cu, 24) for cu in ([0, 5, 24], [0, 24])]
    with torch.no_grad():
        want = sum(sess.model(ids[i:i + 1], attention_mask=packings[i], labels=ids[i:i + 1]) for i in range(micro)) / micro
    with pytest.raises(ValueError, match="micro batches"):
        sess.step_on_device_batch(dict(input_ids=ids, labels=ids, attention_mask=packings * 2))
    got = sess.step_on_device_batch(dict(input_ids=ids, labels=ids, attention_mask=packings[:micro]))
    sess.finish()
    assert abs(float(got) - float(want)) < 1e-5
