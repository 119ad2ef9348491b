"""The symbolic trace prices the operators that run: the embedding's backward pass, the loss with its projection."""
import pickle

import pytest
import sympy as sp
import torch

from mist_b200.analyzer.layer_analyzer import analysis_cache_name, trace_and_analyze
from mist_b200.config import ModelConfig
from mist_b200.ops import functional as F
from mist_b200.ops import linear_xent

H, V, S = 2048, 32000, 1024
FAMILIES = {
    "gpt2-t": dict(encoder_attn_mask_type="causal"),
    "gpt2-tied": dict(encoder_attn_mask_type="causal", tie_word_embeddings=True),
    "llama-t": dict(encoder_attn_mask_type="causal", mlp_type="gated_mlp", normalization="rmsnorm",
                    position_embedding_type="rotary", rotary_emb_fraction=1.0),
    "bert-t": dict(encoder_attn_mask_type="padding", add_pooler=True, num_tokentypes=2),
    "t5-t": dict(encoder_attn_mask_type="padding", decoder_attn_mask_type="causal", add_decoder=True),
}


def _cfg(name, **more):
    base = dict(name=name, hidden_size=H, intermediate_size=4 * H, num_hidden_layers=2, num_attention_heads=16,
                max_position_embeddings=S, vocab_size=V, params_dtype="bfloat16", add_encoder=True, add_decoder=False,
                use_flash_attn=True)
    return ModelConfig(**{**base, **FAMILIES[name], **more})


def _node(info, op):
    return [n for n in info.nodes if n.op == op]


def _at(expr, b):
    return float(sp.sympify(expr).subs({s: b for s in sp.sympify(expr).free_symbols}))


@pytest.mark.parametrize("name", ["gpt2-t", "llama-t"])
def test_embedding_holds_a_sort_and_no_table(name):
    (node,) = _node(trace_and_analyze(_cfg(name), S).pre, "embedding")
    for b in (1, 8):
        tokens, wpe = b * S, S * H * 2 if name == "gpt2-t" else 0
        area = 16 * tokens + 8 * (tokens // 32) * (H + H // 256)
        assert area + wpe <= _at(node.bwd_workspace, b) <= area + wpe + 16 * H
    assert _at(node.bwd_workspace, 1) < V * H


@pytest.mark.parametrize("name", sorted(FAMILIES))
def test_the_fused_loss_is_traced(name):
    plain, fused = trace_and_analyze(_cfg(name), S).post, trace_and_analyze(_cfg(name, fused_lm_loss=True), S).post
    assert _node(plain, "cross_entropy") and not _node(plain, "linear_cross_entropy")
    assert not _node(fused, "cross_entropy")
    (node,) = _node(fused, "linear_cross_entropy")
    assert plain.num_params == fused.num_params and _at(plain.fwd.flops, 2) == pytest.approx(_at(fused.fwd.flops, 2), rel=1e-3)
    assert node.spec["vocab"] == V and node.spec["k"] == H
    pickle.loads(pickle.dumps(fused))
    for b in (1, 4, 64):             # 64: 65536 rows of 32000 logits are more than 2 GiB, so the logits are computed twice
        rows = b * S
        kept = linear_xent.kept_bytes(rows, V)
        keeps = kept <= F.Settings.xent_keep_bytes
        assert keeps == (b < 64)
        assert _at(node.saved_extra, b) == (kept - 4 * rows if keeps else 4 * rows)      # the loss itself is an output
        assert _at(node.flops_bwd, b) == (4 if keeps else 6) * rows * H * V
        assert _at(node.bwd_workspace, b) >= min(2 * rows * V, F.Settings.xent_piece_bytes)
        assert _at(fused.bwd.peak, b) > 0 and _at(fused.fwd.saved, b) > 0


def test_without_kept_logits_memory_falls(monkeypatch):
    plain = trace_and_analyze(_cfg("gpt2-t"), S).post
    monkeypatch.setattr(F.Settings, "xent_keep_bytes", 0)
    fused = trace_and_analyze(_cfg("gpt2-t", fused_lm_loss=True), S).post
    assert _at(fused.fwd.saved, 16) + 16 * S * V * 2 * 0.9 < _at(plain.fwd.saved, 16)
    assert _at(fused.bwd.peak, 16) < _at(plain.bwd.peak, 16)


def test_caches_of_the_two_are_apart():
    names = {analysis_cache_name(_cfg("gpt2-t", fused_lm_loss=f), S, 1, False) for f in (False, True)}
    assert len(names) == 2


def test_caches_go_by_the_limits_of_the_loss(monkeypatch):
    cfg = _cfg("gpt2-t", fused_lm_loss=True)
    first = analysis_cache_name(cfg, S, 1, False)
    monkeypatch.setattr(F.Settings, "xent_keep_bytes", 0)
    assert analysis_cache_name(cfg, S, 1, False) != first
