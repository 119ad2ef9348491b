"""Packed documents through whole models on the GPU: the same as the documents one by one through the separate steps.

Both sides round to bf16 at some 20 places of a block (activations, their gradients), each off by at most 2^-8 and with
no common sign: over two blocks and both sides 80 roundings of 2^-9 rms and less, so the gradients may differ by
2^-9 * 80 ** 0.5 = 1.7 % of their norm; 4 % leaves room for the smallest of them.  The loss differs by the rounding of the
logits on one side (2^-8 of logits below 1)."""
import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import native
from tests.test_packed_training_cpu import FAMILIES, batch, build, gradients, labelled, one_by_one

pytestmark = pytest.mark.gpu
DEV = "cuda"
LENS = [200, 1, 129, 0, 77, 300]
CU = [0] + torch.tensor(LENS).cumsum(0).tolist()
WIDE = dict(hidden_size=256, intermediate_size=512, num_attention_heads=4, max_position_embeddings=512, vocab_size=1000,
            params_dtype="bfloat16", fused_lm_loss=True)


@pytest.mark.parametrize("family", [f for f in sorted(FAMILIES) if f != "t5"])
@pytest.mark.parametrize("rows,recompute", [(1, 0), (2, 1)])
def test_packed_step_is_the_documents_one_by_one(family, rows, recompute):
    total = 720
    ids, labels = batch(rows, DEV, 1000, total, CU)
    fused = build(family, DEV, torch.bfloat16, **WIDE)
    plain = build(family, DEV, torch.bfloat16, **{**WIDE, "fused_lm_loss": False})
    plain.load_state_dict(fused.state_dict())
    fused.language_model.encoder.gradient_checkpointing = recompute
    seqs = F.PackedSequences(torch.tensor(CU, device=DEV), total)
    got = fused(ids, attention_mask=seqs, **{labelled(family): labels})
    want = one_by_one(plain, family, ids, labels, CU)
    assert abs(got.item() - want.item()) < 2 ** -8
    a, b = gradients(fused, got), gradients(plain, want)
    native.check_status()
    assert set(a) == set(b)
    for n in a:
        assert (a[n].float() - b[n].float()).norm() <= 0.04 * b[n].float().norm() + 1e-6, n


def _session(fused, zero):
    from mist_b200.api import build_training
    vec = [1, 1, 1, *zero, 0, 0, 0, 0]
    return build_training("config", [
        "experiment=template-b200", "model=gpt2/1.3b", "hardware.num_gpus_per_node=1", "model.hidden_size=256",
        "model.intermediate_size=512", "model.num_attention_heads=4", "model.num_heads_kv=4", "model.num_hidden_layers=2",
        "model.vocab_size=1000", "training.vocab_size=1000", "training.max_sequence_length=720",
        "training.global_batch_size=2", "strategy.layer_partitions=[2]", "strategy.device_assignment=[[1,1]]",
        "strategy.gradient_checkpointing=[1]", "strategy.gradient_accumulation_steps=2",
        f"strategy.stage_strategies=[{vec}]".replace(" ", ""), f"strategy.pre_post_strategy_array={vec}".replace(" ", ""),
        f"+model.fused_lm_loss={'true' if fused else 'false'}"], seed=3, hp=dict(lr=1e-3))


@pytest.mark.parametrize("zero", [(0, 0, 0), (1, 1, 0)])
def test_training_session_with_two_micro_batches(zero):
    """Gradients of both operators in their buckets, over two micro batches with packings of their own."""
    ids, labels = batch(1, DEV, 1000, 1440, CU)
    ids, labels = ids.view(2, 720), labels.view(2, 720)
    other = [0, 300, 720]
    losses = []
    for fused in (True, False):
        sess = _session(fused, zero)
        data = {"input_ids": ids, "labels": labels,
                "attention_mask": [F.PackedSequences(torch.tensor(c, device=DEV), 720) for c in (CU, other)]}
        losses.append([float(sess.step_on_device_batch(data)) for _ in range(4)])
        sess.finish()
    a, b = losses
    assert all(abs(x - y) < 2 ** -6 for x, y in zip(a, b)), losses      # four updates of weights that differ by roundings
    assert a[3] != a[0]


def test_generation_takes_explicit_positions():
    """Cached decoding passes positions: the lookup with explicit positions gives the logits of the whole sequence."""
    from mist_b200.inference import kv_cache
    model = build("gpt", DEV, torch.bfloat16, **WIDE).eval()
    ids = torch.randint(0, 1000, (2, 12), device=DEV)
    with torch.no_grad():
        whole = model(ids).view(2, 12, -1).float()
        with kv_cache(model, 2, 12) as ip:
            for t in range(12):
                pos = torch.full((2, 1), t, device=DEV)
                step = model(ids[:, t:t + 1], position_ids=pos).view(2, -1).float()
                ip.seqlen_offset += 1
                # bf16 activations on both sides, through other kernels: 2^-8 at some ten places in a row
                assert (step - whole[:, t]).norm() <= 10 * 2 ** -8 * whole[:, t].norm(), t
