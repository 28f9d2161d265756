"""Quantised models and stores on the host: what counting, moving, loading and calling them may not change (no GPU
needed)."""
import pytest
import torch

from latest_exact_match_attention_b200._lib import LemaError
from latest_exact_match_attention_b200.model import ModelConfig, Transformer
from latest_exact_match_attention_b200.quant import Int4Module


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


def test_buffers_that_a_module_gave_up_are_freed():
    import gc
    import weakref
    moves = [lambda m: m._apply(torch.clone), lambda m: m.to("meta"), lambda m: m.half(),
             lambda m: m.load_state_dict({k: v.clone() for k, v in m.state_dict().items()}, assign=True),
             lambda m: [setattr(x, "packed", x.packed.clone()) or setattr(x, "scales", x.scales.clone())
                        for x in m.modules() if isinstance(x, Int4Module)]]
    for move in moves:
        m = small().quantize_weights_(group=64)
        held = [x for x in m.modules() if isinstance(x, Int4Module)]
        assert len(held) == 2 * 4 + 1
        for x in held:
            x.weight4                                    # as a forward would have
        before = [(name, weakref.ref(b), b.data_ptr()) for x in held for name, b in (("packed", x.packed), ("scales", x.scales))]
        move(m)
        gc.collect()
        kept = {b.data_ptr() for x in held for b in x.buffers()}
        assert all(ref() is None or at in kept for _, ref, at in before)
        assert all(x.weight4.packed is x.packed and x.weight4.scales is x.scales for x in held)


def test_a_state_dict_of_another_group_leaves_the_scales():
    m = small().quantize_weights_(group=64)
    other = small().to(torch.float16).quantize_weights_(group=32).state_dict()      # fp16 scales, twice as many
    before = {k: v.clone() for k, v in m.state_dict().items() if k.endswith("scales")}
    with pytest.raises(RuntimeError, match="scales"):
        m.load_state_dict(other)
    after = m.state_dict()
    for k, v in before.items():
        if v.shape != other[k].shape:
            assert after[k].dtype == torch.bfloat16 and torch.equal(after[k], v)
    assert any(v.shape != other[k].shape for k, v in before.items())
