"""Quantised models and stores on the host: what counting, moving, loading and calling them may not change (no GPU
needed)."""
import pytest
import torch

from latest_exact_match_attention_b200._lib import LemaError
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


def store_without_a_gpu(quant):
    """The fields the checks read: no call below gets as far as a launch."""
    from latest_exact_match_attention_b200.cache import HashStore
    st = HashStore.__new__(HashStore)
    st.dtype, st.d_v, st.groups, st.quant, st._index, st.vbytes = torch.bfloat16, 16, 4, quant, 0, 32
    st.table = torch.empty(0)
    return st


@pytest.mark.parametrize("quant", [None, "int8"])
def test_half_a_step_refuses_rows_that_do_not_match_its_codes(quant):
    """Fewer or narrower rows than codes would be read or written past their end."""
    from latest_exact_match_attention_b200.cache import Buffers, LayerStore
    st = store_without_a_gpu(quant)
    k, v = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 16, dtype=torch.bfloat16)
    for rows in (v[:2], v[:, :8], torch.zeros(16, 4, dtype=torch.bfloat16)):
        for phase in (1, 2):
            with pytest.raises(ValueError, match="rows must be"):
                st.exchange_phase(k, k, rows, rows.clone(), 0, phase)
    view = LayerStore(st, Buffers(torch.bfloat16, None), 0, 4)
    with pytest.raises(ValueError, match="rows must be"):
        view.lookup(k.view(1, 4, 1), k.view(1, 4, 1), v[:2].view(1, 2, 1, 16))


def test_half_a_step_on_raw_rows_checks_their_bytes_and_layout():
    st = store_without_a_gpu(None)
    k, v = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 16, dtype=torch.float32)
    for phase in (1, 2):
        with pytest.raises(ValueError, match="64 bytes"):
            st.exchange_phase(k, k, v, v.clone(), 0, phase)
    with pytest.raises(ValueError, match="contiguous"):
        st.exchange_phase(k, k, v.bfloat16(), torch.zeros(16, 4, dtype=torch.bfloat16).t(), 0, 1)


def test_a_step_with_key_codes_of_the_other_width_gets_as_far_as_the_device():
    from latest_exact_match_attention_b200.cache import Buffers, LayerStore
    view = LayerStore(store_without_a_gpu("int8"), Buffers(torch.bfloat16, None), 0, 4)
    k, v = torch.zeros(1, 4, 1, dtype=torch.int32), torch.zeros(1, 4, 1, 16, dtype=torch.bfloat16)
    for q, k2 in ((k, k.long()), (k.long(), k), (k, k)):
        with pytest.raises(LemaError, match="the store is on"):
            view.exchange(q, k2, v, check=False)
