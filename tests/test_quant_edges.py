"""Quantised models and stores on the host: what counting, moving, loading and calling them may not change (no GPU
needed)."""
import torch

from latest_exact_match_attention_b200.model import ModelConfig, Transformer


def small(**kw):
    torch.manual_seed(0)
    return Transformer(ModelConfig(vocab_size=128, depth=2, dim=64, num_heads=4, d_qk=32, d_v=16, dim_ff=128, **kw))


def test_a_shared_embedding_is_counted_once():
    m = small()
    m.lm_head.weight = m.tok_emb.weight
    table = 128 * 64
    body = sum(p.numel() for n, p in m.named_parameters()) - table      # a shared parameter has one name
    assert m.n_params() == body + table and m.n_params(embedding=False) == body
    m.quantize_weights_(group=64)                                       # the head has weights of its own from here on
    assert m.n_params() == body + 2 * table and m.n_params(embedding=False) == body
