"""Quantised serving on the host: the layout of 4-bit weights, the formats of held rows, and what the
entry points refuse before they touch a device (no GPU needed)."""
import ctypes

import pytest
import torch

from latest_exact_match_attention_b200 import _lib, quant
from latest_exact_match_attention_b200._lib import LemaError
from latest_exact_match_attention_b200.quant import Int4Weight, dequantize_rows, quantize_rows, row_bytes


def random_weight(n, k, group, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    scales = (0.5 + torch.rand(n, -(-k // group), generator=g)).to(dtype)
    return codes, scales


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (16, 64, 64), (17, 65, 32), (40, 200, 128), (8, 640, 128)])
def test_pack_round_trip(n, k, group):
    c, s = random_weight(n, k, group)
    w = Int4Weight.pack(c, s, group)
    c2, s2 = w.codes()
    assert torch.equal(c, c2) and torch.equal(s, s2)
    assert torch.equal(w.dequantize(), c.float() * s.float().repeat_interleave(group, 1)[:, :k])
    cu, su = random_weight(n, k, group, seed=1)
    p = Int4Weight.pack_gate_up(c, s, cu, su, group)
    (g2, gs2), (u2, us2) = p.codes()
    assert torch.equal(g2, c) and torch.equal(gs2, s) and torch.equal(u2, cu) and torch.equal(us2, su)
    assert w.nbytes() == w.packed.numel() * 4 + w.scales.numel() * 2


def test_layout_is_the_documented_one():
    """Field of feature 16 b + 8 i + a at input 64 c + 32 h + 8 t + 4 j + 2 p + e, by the header's formula."""
    n, k = 40, 130
    c, s = random_weight(n, k, 32)
    w = Int4Weight.pack(c, s, 32).packed
    for f, x in [(0, 0), (39, 129), (17, 64), (8, 37), (31, 127), (5, 90)]:
        b, i, a = f // 16, f % 16 // 8, f % 8
        cc, h, t, j, p, e = x // 64, x % 64 // 32, x % 32 // 8, x % 8 // 4, x % 4 // 2, x % 2
        word = int(w[b, cc, 8 * 0 + 4 * a + t, 2 * h + j]) & 0xFFFFFFFF
        assert (word >> (16 * e + 8 * p + 4 * i)) & 15 == int(c[f, x]) + 8
    assert int(w[2, 2, 31, 3]) & 0xFFFFFFFF == 0x88888888        # padding is a zero weight


def test_quantize_weight_is_round_to_nearest():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(24, 150, generator=g) * 0.1
    w[3] = 0
    q, s = quant.quantize_weight(w, 64)
    assert q.dtype == torch.int8 and s.dtype == torch.bfloat16 and s.shape == (24, 3)
    d = q.double() * s.double().repeat_interleave(64, 1)[:, :150]
    # half a step; the largest value can sit beyond 7.5 steps by the scale's own rounding, which
    # the code -8 ... 7 then clips: amax / s is at most 7 (1 + 2^-8), within half a step of 7
    step = s.double().repeat_interleave(64, 1)[:, :150]
    assert bool(((w.double() - d).abs() <= 0.5 * step * (1 + 2.0 ** -20)).all())
    assert bool((q[3] == 0).all()) and bool((s[3] == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "fp8", "int4"])
@pytest.mark.parametrize("d", [1, 7, 8, 24, 33, 64, 256])
def test_row_formats_round_trip(fmt, d):
    """A held value is within half a step of its own: int formats s / 2 (s = amax / 127 or / 7, plus the
    2^-24 roundings of s and of the product), e4m3 half an ulp (2^-4 relative, 2^-10 s below 2^-6 s)."""
    g = torch.Generator().manual_seed(d)
    v = (torch.randn(50, d, generator=g) * torch.exp(2 * torch.randn(50, 1, generator=g))).to(torch.bfloat16)
    v[0] = 0
    rows = quantize_rows(v, fmt)
    assert rows.dtype == torch.uint8 and rows.shape == (50, row_bytes(fmt, d)) and row_bytes(fmt, d) % 16 == 0
    assert row_bytes(fmt, d) == _lib.lib().lema_quant_row_bytes(quant.ROW_FORMATS[fmt], d)
    back = dequantize_rows(rows, fmt, d, torch.float32).double()
    x = v.double()
    if fmt == "fp8":
        amax = x.abs().amax(1, keepdim=True)
        bound = torch.maximum(x.abs() * 2.0 ** -4, amax / 448 * 2 * 2.0 ** -10)
    else:
        wide, top = (d, 127) if fmt == "int8" else (32, 7)
        pad = torch.nn.functional.pad(x, (0, -d % wide)).unflatten(1, (-1, wide))
        amax = pad.abs().amax(2, keepdim=True).expand_as(pad).flatten(1)[:, :d]
        bound = amax / top * (0.5 + top * 2.0 ** -23)
    assert bool(((back - x).abs() <= bound).all())
    assert bool((back[0] == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "fp8", "int4"])
def test_rows_with_what_no_code_can_hold(fmt):
    v = torch.randn(6, 40)
    v[1, 3] = float("inf")
    v[2, 39] = float("nan")
    v[3] = 2.0 ** -149                    # the smallest magnitudes there are
    v[4] = torch.finfo(torch.float32).max
    back = dequantize_rows(quantize_rows(v, fmt), fmt, 40, torch.float32)
    lone = 32 if fmt == "int4" else 40    # the scale group around the infinity
    assert bool(back[1, :lone].isnan().all()) and bool(back[1, lone:].isfinite().all())
    assert bool(back[2, 32 if fmt == "int4" else 0:].isnan().all())
    assert bool(back[0].isfinite().all()) and bool(back[3].isfinite().all())
    assert bool(((back[4] / v[4] - 1).abs() < 2.0 ** -3).all())


def test_sizes_of_rows():
    assert [row_bytes(f, 24) for f in ("int8", "fp8", "int4")] == [32, 32, 16]
    assert [row_bytes(f, 64) for f in ("int8", "fp8", "int4")] == [80, 80, 48]
    L = _lib.lib()
    assert L.lema_quant_row_bytes(0, 24) == 0 and L.lema_quant_row_bytes(4, 24) == 0
    assert L.lema_quant_row_bytes(1, 0) == 0 and L.lema_quant_row_bytes(1, 257) == 0
    with pytest.raises(ValueError, match="row format"):
        row_bytes("int5", 24)
    with pytest.raises(ValueError, match="1 to 256"):
        row_bytes("int8", 257)


def test_weights_that_are_refused():
    c, s = random_weight(16, 64, 64)
    with pytest.raises(ValueError, match="group"):
        Int4Weight.pack(c, s, 48)
    with pytest.raises(ValueError, match="scales"):
        Int4Weight.pack(c, s, 32)
    with pytest.raises(ValueError, match="scales"):
        Int4Weight.pack(c, s.float(), 64)
    with pytest.raises(ValueError, match="int8"):
        Int4Weight.pack(c.int(), s, 64)
    with pytest.raises(ValueError, match="-8"):
        Int4Weight.pack(c + 1, s, 64)
    with pytest.raises(ValueError, match="differ"):
        Int4Weight.pack_gate_up(c, s, c[:8], s[:8], 64)
    w = Int4Weight.pack(c, s, 64)
    with pytest.raises(ValueError, match="not a packed"):
        Int4Weight(w.packed, w.scales, 17, 64, 64)
    with pytest.raises(LemaError, match="CUDA tensors only"):
        quant.int4_linear(torch.zeros(1, 64), w)
    with pytest.raises(LemaError, match="gate/up"):
        quant.int4_swiglu(torch.zeros(1, 64), w)
    with pytest.raises(LemaError, match="int4_swiglu"):
        quant.int4_linear(torch.zeros(1, 64), Int4Weight.pack_gate_up(c, s, c, s, 64))


def rc(name, *args):
    return getattr(_lib.lib(), name)(*args)


def test_c_arguments_are_checked_on_the_host():
    P = ctypes.c_void_p(1 << 20)   # never dereferenced: every call below fails validation first
    O = ctypes.c_void_p((1 << 20) + 1)

    def linear(x=P, dtype=1, M=4, K=64, ldx=64, w=P, s=P, sdt=1, group=64, N=16, gated=0, r=None, ldr=16, y=P, ldy=16):
        return rc("lema_int4_linear", x, dtype, M, K, ldx, w, s, sdt, group, N, gated, r, ldr, y, ldy, None, None)
    assert linear(dtype=3) == 1 and linear(sdt=0) == 1 and linear(group=16) == 1
    assert linear(M=-1) == 1 and linear(K=0) == 1 and linear(N=0) == 1 and linear(K=1 << 24) == 1
    assert linear(ldx=63) == 1 and linear(ldy=15) == 1 and linear(r=P, ldr=15) == 1
    assert linear(gated=1, r=P) == 1
    assert linear(x=None) == 1 and linear(w=None) == 1 and linear(s=None) == 1 and linear(y=None) == 1
    assert linear(w=ctypes.c_void_p((1 << 20) + 8)) == 1 and linear(x=O) == 1 and linear(y=O) == 1
    assert linear(M=0, x=None, y=None) == 0      # no rows: nothing to do

    def ex(table=P, cap=100, fmt=1, dtype=1, d=24, q=P, k=P, cb=4, v=P, o=P, n=8, T=1, g0=0, c=P, ws=None, wsb=0,
           sg=0, ss=0, heads=0, st=(0, 0, 0, 0, 0, 0), phase=3):
        return rc("lema_store_exchange_quant", table, cap, fmt, dtype, d, q, k, cb, v, o, n, T, g0, c, None, ws, wsb,
                  sg, ss, heads, *st, phase, None)
    assert ex(fmt=0) == 1 and ex(fmt=4) == 1 and ex(d=0) == 1 and ex(d=257) == 1 and ex(dtype=7) == 1
    assert ex(cb=2) == 1 and ex(cap=0) == 1 and ex(n=7, T=2) == 1 and ex(g0=-1) == 1 and ex(phase=0) == 1
    assert ex(n=8, T=2, phase=1) == 1 and ex(sg=4) == 1 and ex(sg=8, ss=101) == 1
    assert ex(n=6, heads=4) == 1 and ex(heads=4, st=(48, 48, 47, 48, 48, 48)) == 1
    assert ex(table=None) == 1 and ex(table=ctypes.c_void_p((1 << 20) + 8)) == 1 and ex(c=None) == 1
    assert ex(q=None) == 1 and ex(v=None) == 1 and ex(q=O) == 1 and ex(o=O) == 1
    assert ex(n=8, T=2) == 3                     # T > 1 needs a workspace
    assert ex(n=0, table=None) == 0


def test_modules_keep_their_scales_and_load(tmp_path):
    from latest_exact_match_attention_b200.model import ModelConfig, Transformer
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=128, depth=2, dim=64, num_heads=4, d_qk=32, d_v=16, dim_ff=128)
    m = Transformer(cfg).quantize_weights_(group=32)
    assert m.blocks[0].attn.q_proj.weight.shape == (128, 64)        # codes keep their weights
    before = m.lm_head.scales.clone()
    m.to(torch.float16)
    assert m.lm_head.scales.dtype == torch.bfloat16 and torch.equal(m.lm_head.scales, before)
    torch.save(m.state_dict(), tmp_path / "m.pt")
    m2 = Transformer(cfg).quantize_weights_(group=32).to(torch.float16)
    m2.load_state_dict(torch.load(tmp_path / "m.pt"))
    assert torch.equal(m2.blocks[1].mlp.gate_up.packed, m.blocks[1].mlp.gate_up.packed)
    with pytest.raises(ValueError, match="bias"):
        quant.Int4Linear.from_linear(torch.nn.Linear(64, 16))


def test_a_quantised_model_counts_copies_and_is_quantised_once():
    import copy

    from latest_exact_match_attention_b200.model import ModelConfig, Transformer
    cfg = ModelConfig(vocab_size=128, depth=2, dim=64, num_heads=4, d_qk=32, d_v=16, dim_ff=128)
    m = Transformer(cfg)
    whole, body = m.n_params(), m.n_params(embedding=False)
    m.quantize_weights_(group=64)
    assert (m.n_params(), m.n_params(embedding=False)) == (whole, body)
    with pytest.raises(ValueError, match="already"):
        m.quantize_weights_()
    w = m.lm_head.weight4
    assert m.lm_head.weight4 is w
    c = copy.deepcopy(m)
    assert c.lm_head.weight4.packed is c.lm_head.packed and c.lm_head.packed is not m.lm_head.packed
    m.lm_head.packed = m.lm_head.packed.clone()          # a replaced buffer is the weight from then on
    assert m.lm_head.weight4.packed is m.lm_head.packed
    with pytest.raises(ValueError, match="group"):
        Transformer(cfg).quantize_weights_(group=48)


def test_a_quantised_store_refuses_tensors_of_another_device():
    # the fields the checks read, without a GPU: nothing below gets as far as a launch
    from latest_exact_match_attention_b200.cache import Buffers, HashStore, LayerStore
    st = HashStore.__new__(HashStore)
    st.dtype, st.d_v, st.groups, st.quant, st._index = torch.bfloat16, 16, 4, "int8", 0
    st.table = torch.empty(0)
    k, v = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 16, dtype=torch.bfloat16)
    with pytest.raises(LemaError, match="the store is on"):
        st.exchange(k, k, v, torch.empty_like(v), 1, 0)
    for phase in (1, 2):
        with pytest.raises(LemaError, match="the store is on"):
            st.exchange_phase(k, k, v, torch.empty_like(v), 0, phase)
    view = LayerStore(st, Buffers(torch.bfloat16, None), 0, 4)
    with pytest.raises(LemaError, match="the store is on"):       # a decode step
        view.exchange(k.view(1, 4, 1), k.view(1, 4, 1), v.view(1, 4, 1, 16), check=False)


def test_a_state_dict_brings_its_scales_unrounded():
    # a model quantised from fp16 weights has fp16 scales, one from fp32 or bf16 weights bf16 scales
    from latest_exact_match_attention_b200.model import ModelConfig, Transformer
    torch.manual_seed(2)
    cfg = ModelConfig(vocab_size=128, depth=1, dim=64, num_heads=4, d_qk=32, d_v=16, dim_ff=128)
    half = Transformer(cfg).to(torch.float16).quantize_weights_(group=64)
    wide = Transformer(cfg).quantize_weights_(group=64)
    for a, b in ((half, wide), (wide, half)):
        state = {k: v.clone() for k, v in a.state_dict().items()}
        c = Transformer(cfg).to(b.tok_emb.weight.dtype).quantize_weights_(group=64)
        assert c.lm_head.scales.dtype == b.lm_head.scales.dtype != state["lm_head.scales"].dtype
        c.load_state_dict(state)
        for name in ("lm_head", "blocks.0.attn.o_proj", "blocks.0.mlp.gate_up", "blocks.0.mlp.down"):
            got, want = c.get_submodule(name), a.get_submodule(name)
            assert got.scales.dtype == want.scales.dtype and torch.equal(got.scales, want.scales)
            assert got.weight4.scales is got.scales
