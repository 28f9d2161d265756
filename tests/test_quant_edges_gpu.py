"""Quantised serving where its kernels meet: the rule that picks one, the ends of 16-bit ranges, and the bytes a
quantised store holds."""
import gc
import weakref

import pytest
import torch

from latest_exact_match_attention_b200 import quant
from latest_exact_match_attention_b200._lib import call, check_status, device_status, ptr, stream_handle
from latest_exact_match_attention_b200.cache import HashStore, LemaCache
from latest_exact_match_attention_b200.model import ModelConfig
from latest_exact_match_attention_b200.quant import Int4Weight, dequantize_rows, quantize_rows

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def weight(n, k, group, scale_dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    scales = ((0.5 + torch.rand(n, -(-k // group), generator=g)) / (4.6 * k ** 0.5)).to(scale_dtype)
    return codes.to(dev), scales.to(dev)


def dense64(codes, scales, group):
    return codes.double() * scales.double().repeat_interleave(group, 1)[:, : codes.shape[1]]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("block_rows_of_each_sm", [7.99, 8, 9])
@pytest.mark.parametrize("M", [16, 17, 32])
def test_up_to_32_rows_multiply_codes_exactly(cuda, M, block_rows_of_each_sm, dtype):
    """Whatever the weight's width. One non-zero input a row makes an output one product s q x: x has 8 significant
    bits, s 8 or 11, q 4, so fp32 holds it (23 at most) and the output is that number rounded once. A weight rounded
    to 16 bits before the product gives another number for many of them."""
    sms = torch.cuda.get_device_properties(cuda).multi_processor_count
    N, K, group = int(sms * block_rows_of_each_sm) * 16, 128, 64
    c, s = weight(N, K, group, dtype, M, cuda)
    x = torch.zeros(M, K)
    m = torch.arange(M)
    x[m, (37 * m + 5) % K] = 1 + (2 * m + 1) / 128
    x = x.to(dtype).to(cuda)
    want = (x.double() @ dense64(c, s, group).t()).to(F32).to(dtype)
    assert torch.equal(quant.int4_linear(x, Int4Weight.pack(c, s, group)), want)
    # and rows give the same bits in whatever company up to 32, gate/up pairs too (half the width for as many block rows)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype).to(cuda)
    w = Int4Weight.pack(c, s, group)
    gu = Int4Weight.pack_gate_up(c[: N // 2], s[: N // 2], c[N // 2:], s[N // 2:], group)
    for call, packed in ((quant.int4_linear, w), (quant.int4_swiglu, gu)):
        parts = torch.cat([call(x[i:i + 8].contiguous(), packed) for i in range(0, M, 8)])
        assert torch.equal(call(x, packed), parts)
    check_status(cuda)


def check_products(x, s_dtype, spread, M, N, K, group, seed, dev, residual):
    """fp16 rows against 64-bit sums, gate/up pairs too. spread [N, groups]: powers of two of the scales."""
    c, s = weight(N, K, group, s_dtype, seed, dev)
    s = (s.float() / s.float().abs().amax() * 2.0 ** spread.to(dev)).to(s_dtype)
    w = dense64(c, s, group)
    # fp32 sums (2^-23 of the magnitudes an addition), half a step of 2^-11 a weight, or, for scales far below the
    # feature's largest, three times half a step of fp16's subnormals under its power of two, 2^-25 2^(e - 12)
    low = 3 * 2.0 ** (torch.floor(torch.log2(s.double().abs().amax(1))) - 12 - 25)
    mag = x.double().abs() @ w.abs().t()
    off = mag * ((K + 8) * 2.0 ** -23 + 2.0 ** -11) + x.double().abs().sum(1, keepdim=True) * low
    ref = x.double() @ w.t()
    r = torch.randn(M, N, generator=torch.Generator().manual_seed(seed)).half().to(dev) if residual else None
    got = quant.int4_linear(x, Int4Weight.pack(c, s, group), residual=r)
    check_status(dev)
    full = ref if r is None else ref + r.double()
    bound = off + 2.0 ** -11 * (full.abs() + off) + 2.0 ** -25        # the output's rounding, subnormals too
    err = (got.double() - full).abs()
    ok = full.abs() + off < 65504                                     # what fp16 holds; past it infinities
    assert bool((err <= bound)[ok].all()), f"{float((err / bound)[ok].nan_to_num(nan=1e9).max()):.3g} of the bound"
    assert float(ok.double().mean()) > 0.99
    past = full.abs() - off > 65520
    assert torch.equal(got[past], torch.sign(full[past]).half() * float("inf"))
    gu = quant.int4_swiglu(x, Int4Weight.pack_gate_up(c, s, c, s, group))
    want = ref * torch.sigmoid(ref) * ref
    ok = want.abs() + 1.1 * off * (2 * ref.abs() + off) < 60000
    bound = 1.1 * off * (ref.abs() + off) + ref.abs() * off
    bound = bound + (2.0 ** -11 + 2.0 ** -17) * (want.abs() + bound) + 2.0 ** -25
    assert bool(((gu.double() - want).abs() <= bound)[ok].all()) and int(ok.sum()) > 0


@pytest.mark.parametrize("M,N,K,group", [(33, 100, 320, 64), (64, 256, 4096, 128), (300, 272, 1096, 32), (2100, 1000, 200, 32)])
@pytest.mark.parametrize("s_dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["large", "small", "both"])
def test_fp16_rows_through_weights_beyond_fp16(cuda, kind, s_dtype, M, N, K, group):
    """Weights s q above 65504 and, with bf16 scales, far below fp16's smallest, in tiles alone and with K split: sums that
    fp16 holds come out, within the rounding of the weights' significant bits. Features differ, and in "both" the
    groups of a feature."""
    g = torch.Generator().manual_seed(M)
    groups = -(-K // group)
    top = 15 if s_dtype == F16 else 20
    if kind == "large":
        spread, size = torch.randint(8, top + 1, (N, 1), generator=g).expand(N, groups).double(), 2.0 ** -13
    elif kind == "small":
        spread, size = torch.randint(-12 if s_dtype == F16 else -26, -6, (N, 1), generator=g).expand(N, groups).double(), 2.0 ** 6
    else:
        spread, size = torch.randint(-8, top + 1, (N, groups), generator=g).double(), 2.0 ** -13
    x = (torch.randn(M, K, generator=g).clamp(-4, 4) * size).half().to(cuda)
    check_products(x, s_dtype, spread, M, N, K, group, M + K, cuda, residual=M % 2 == 1)


@pytest.mark.parametrize("M", [3, 40, 400])
@pytest.mark.parametrize("s_dtype", [BF16, F16])
def test_features_without_a_usable_scale_touch_only_themselves(cuda, s_dtype, M):
    """All-zero, infinite and NaN scales in fp16 rows' weights, few rows and tiles alike."""
    N, K, group = 72, 256, 64
    c, s = weight(N, K, group, s_dtype, 1, cuda)
    c = torch.where(c == 0, torch.ones_like(c), c)
    x = torch.rand(M, K, generator=torch.Generator().manual_seed(M)).add(0.5).half().to(cuda)
    clean = quant.int4_linear(x, Int4Weight.pack(c, s, group))
    s[5], s[17, 2], s[40, 0] = 0, float("inf"), float("nan")
    got = quant.int4_linear(x, Int4Weight.pack(c, s, group))
    others = [n for n in range(N) if n not in (5, 17, 40)]
    assert torch.equal(got[:, others], clean[:, others])
    assert bool((got[:, 5] == 0).all()) and not bool(got[:, [17, 40]].isfinite().any())


@pytest.mark.parametrize("fmt", ["int8", "fp8", "int4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [40, 7])
def test_held_bytes_are_those_of_quantize_rows(cuda, fmt, dtype, d):
    """Byte for byte, and the values given back bit for bit (NaNs aside: any NaN): random rows, zeros of both signs, the ends
    of the type, and amplitudes so small that a scale is a subnormal or zero."""
    fi = torch.finfo(dtype)
    tiny = fi.smallest_normal * fi.eps
    g = torch.Generator().manual_seed(d)
    rows = torch.randn(300, d, generator=g) * torch.exp(3 * torch.randn(300, 1, generator=g))
    sign = torch.where(torch.rand(64, d, generator=g) < 0.5, -1.0, 1.0)
    steps = torch.arange(1, 65)[:, None] * torch.rand(64, d, generator=g).add(0.01)      # amax of 1 to 64 subnormal steps
    more = [rows, sign * steps.round() * tiny, torch.zeros(1, d), -torch.zeros(1, d), torch.full((1, d), -tiny),
            torch.full((1, d), 63 * tiny), torch.full((1, d), -64 * tiny), torch.full((1, d), -fi.max), rows[:8] * fi.smallest_normal,
            torch.linspace(-190, 190, d)[None] * tiny]
    rows = torch.cat(more).to(dtype)
    bad = rows[:3].clone()
    bad[0, 1], bad[1, d - 1], bad[2, 0] = float("inf"), float("nan"), float("-inf")
    rows = torch.cat([rows, bad])
    P = rows.shape[0]
    code = torch.arange(P, dtype=torch.int32, device=cuda)
    st = HashStore(d, groups=P, dtype=dtype, capacity=4 * P, device=cuda, quant=fmt)
    out = torch.empty(P, d, dtype=dtype, device=cuda)
    for _ in range(2):
        st.exchange(code, code, rows.to(cuda), out, 1, 0)
    want = quantize_rows(rows, fmt)
    state = st.table.view(-1)[: 16 * st.cap].view(torch.int64).view(st.cap, 2)[:, 1].cpu()
    live = (state >= 2).nonzero().squeeze(1)
    held = torch.empty_like(want)
    held[state[live] - 2] = st.table.view(-1)[16 * st.cap:].view(st.cap, -1)[live.to(cuda)].cpu()
    assert live.numel() == P
    wrong = (held != want).any(1).nonzero().squeeze(1).tolist()
    assert not wrong, f"row {wrong[0]}: {rows[wrong[0]].tolist()}"
    back = dequantize_rows(want, fmt, d, dtype)
    ints = torch.int32 if dtype == F32 else torch.int16
    assert bool(((out.cpu().view(ints) == back.view(ints)) | (out.cpu().isnan() & back.isnan())).all())


@pytest.mark.parametrize("quant", [None, "int8"])
def test_a_step_takes_key_codes_of_the_other_width(cuda, quant):
    """As a prompt's chunk and a store of raw rows do: key codes become the query codes' type."""
    cfg = ModelConfig(vocab_size=128, depth=1, dim=64, num_heads=4, d_qk=32, d_v=16)
    c = [LemaCache(cfg, dtype=BF16, batch=1, max_cache_len=40, device=cuda, quant=quant) for _ in range(2)]
    g = torch.Generator().manual_seed(0)
    for _ in range(20):
        q, k = (torch.randint(0, 5, (1, 4, 1), generator=g).to(torch.int32).to(cuda) for _ in range(2))
        v = torch.randn(1, 4, 1, 16, generator=g).to(BF16).to(cuda)
        assert torch.equal(c[0].layer(0).exchange(q, k, v), c[1].layer(0).exchange(q, k.long(), v))
    assert torch.equal(c[0].counts(), c[1].counts())


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_a_captured_chunk_has_a_workspace_of_its_own(cuda, fmt):
    """It needs no reservation, replays after a larger eager call and beside another graph, and goes with the graph."""
    P, T, d = 4, 64, 24
    g = torch.Generator().manual_seed(1)

    def items(t, at):
        q, k = (torch.randint(at, at + 300, (P * t,), generator=g).to(torch.int32).to(cuda) for _ in range(2))
        return q, k, torch.randn(P * t, d, generator=g).to(BF16).to(cuda)

    def store():
        return HashStore(d, groups=P, dtype=BF16, capacity=40000, device=cuda, quant=fmt)

    sets = [items(T, 0), items(T, 1000), items(40 * T, 5000)]
    st, ref = store(), store()
    warm = [torch.empty_like(s[2]) for s in sets]
    st.exchange(*sets[0], warm[0], T, 0)                             # the kernels' first launches are not captured
    old = weakref.ref(st._ws)
    outs, graphs = [torch.empty_like(s[2]) for s in sets], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            st.exchange(*sets[i], outs[i], T, 0, check=False)
    st.exchange(*sets[2], outs[2], 40 * T, 0)
    gc.collect()
    assert old() is None                                             # replaced by the larger call's, held by no graph
    for _ in range(2):
        for gr in graphs:
            gr.replay()
    for i in (0, 2, 0, 1, 0, 1):
        ref.exchange(*sets[i], warm[i], T if i < 2 else 40 * T, 0)
    st.check()
    assert all(torch.equal(a, b) for a, b in zip(outs, warm))
    assert torch.equal(st.counts, ref.counts)
    fresh = store()                                                  # captured before any eager call of its own
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fresh.exchange(*sets[0], outs[0], T, 0, check=False)
    other = store()
    for _ in range(2):
        graph.replay()
        other.exchange(*sets[0], warm[0], T, 0)
    fresh.check()
    assert torch.equal(outs[0], warm[0]) and torch.equal(fresh.counts, other.counts)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,K", [(8192, 333), (2048, 1501), (50304, 100)])
@pytest.mark.parametrize("M", [33, 64, 96, 128])
def test_unaligned_rows_through_wide_weights_give_the_bits_of_aligned_ones(cuda, M, N, K, dtype):
    """The same kernel as aligned rows take, plain and gate/up, whatever makes them unaligned."""
    c, s = weight(N, K, 64, dtype, M, cuda)
    w = Int4Weight.pack(c, s, 64)
    gu = Int4Weight.pack_gate_up(c[: N // 2], s[: N // 2], c[N // 2:], s[N // 2:], 64)
    ka = -(-K // 8) * 8
    room = torch.randn(M, ka, generator=torch.Generator().manual_seed(K)).to(dtype).to(cuda)
    x = room[:, :K]                                                  # 16-byte aligned rows
    flat = torch.empty(M * ka + 1, dtype=dtype, device=cuda)[1:].view(M, ka)
    flat.copy_(room)
    for call, packed in ((quant.int4_linear, w), (quant.int4_swiglu, gu)):
        want = call(x, packed)
        assert torch.equal(call(x.contiguous(), packed), want) and torch.equal(call(flat[:, :K], packed), want)
    check_status(cuda)


@pytest.mark.parametrize("M", [17, 32, 33, 37, 100])
def test_unaligned_rows_through_narrow_weights(cuda, M):
    """Too little work for a copy: exact products still."""
    N, K = 200, 333
    c, s = weight(N, K, 64, F16, M, cuda)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).half().to(cuda)
    got = quant.int4_linear(x, Int4Weight.pack(c, s, 64))
    w = dense64(c, s, 64)
    ref = x.double() @ w.t()
    off = (x.double().abs() @ w.abs().t()) * (K + 8) * 2.0 ** -23
    assert bool(((got.double() - ref).abs() <= off + 2.0 ** -11 * (ref.abs() + off) + 2.0 ** -25).all())


def test_packing_needs_a_few_bytes_a_weight(cuda):
    """The codes themselves are one byte each, the packed weight half a byte."""
    N, K = 4096, 4096
    c, s = weight(N, K, 128, BF16, 0, "cpu")
    c, s = c.to(cuda), s.to(cuda)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    w = Int4Weight.pack(c, s, 128)
    assert torch.cuda.max_memory_allocated() - base <= 5 * N * K
    back, _ = w.codes()
    assert torch.equal(back, c)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,N,K,group", [(3, 17, 64, 32), (32, 40, 72, 64), (70, 33, 128, 32), (130, 130, 192, 128), (300, 257, 1096, 64),
                                         (2500, 1001, 136, 32)])
def test_values_written_at_odd_offsets_and_strides(cuda, M, N, K, group, dtype, gated):
    """y inside a larger buffer, off by one element and rows an odd number apart, the residual likewise: the bits of the plain
    call (the same kernel and tiles), the 64-bit sums within their rounding, and nothing outside y."""
    (c, s), (c2, s2) = weight(N, K, group, dtype, M, cuda), weight(N, K, group, dtype, M + 1, cuda)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(N)).to(dtype).to(cuda)
    w = Int4Weight.pack_gate_up(c, s, c2, s2, group) if gated else Int4Weight.pack(c, s, group)
    wide = N + 2 + (N + 1) % 2                                       # odd
    room = torch.randn(M + 2, wide, generator=torch.Generator().manual_seed(K)).to(dtype).to(cuda)
    r = None if gated else room[1: M + 1, 1: N + 1]
    buf = torch.full((M + 2, wide), 7.0, dtype=dtype, device=cuda)
    y = buf[1: M + 1, 1: N + 1]
    tag = {BF16: 1, F16: 2}[dtype]
    call("lema_int4_linear", ptr(x), tag, M, K, K, ptr(w.packed), ptr(w.scales), tag, group, N, int(gated), ptr(r), wide,
         y.data_ptr(), wide, ptr(device_status(cuda)), stream_handle(cuda))
    check_status(cuda)
    plain = quant.int4_swiglu(x, w) if gated else quant.int4_linear(x, w, r.contiguous())
    assert torch.equal(y, plain)
    h = half_step(dtype)
    a, b = dense64(c, s, group), dense64(c2, s2, group)
    # a product: fp32 sums of at most K terms (2^-23 each) and half a step a weight
    off = [(x.double().abs() @ m.abs().t()) * ((K + 8) * 2.0 ** -23 + h) for m in (a, b)]
    gate, up = x.double() @ a.t(), x.double() @ b.t()
    if gated:
        silu = gate * torch.sigmoid(gate)
        ref = silu * up
        off = 1.1 * off[0] * (up.abs() + off[1]) + silu.abs() * off[1] + 2.0 ** -17 * ref.abs()
    else:
        ref, off = gate + r.double(), off[0] + 2.0 ** -24 * (gate.abs() + r.double().abs())
    assert bool(((y.double() - ref).abs() <= off + h * (ref.abs() + off) + torch.finfo(dtype).tiny).all())
    outside = buf.clone()
    outside[1: M + 1, 1: N + 1] = 7.0
    assert bool((outside == 7.0).all())


@pytest.mark.parametrize("fmt", [None, "int8", "fp8", "int4"])
@pytest.mark.parametrize("P", [30, 5000, 9000])
def test_half_steps_at_high_load(cuda, fmt, P):
    """Lookups then inserts give the rows and entries of the combined step while a table fills to 0.95."""
    d, steps = 24, 19
    pair = [HashStore(d, groups=P, dtype=BF16, capacity=20 * P, device=cuda, quant=fmt, segments=3) for _ in range(2)]
    g = torch.Generator(device=cuda).manual_seed(P)
    out = [torch.empty(P, d, dtype=BF16, device=cuda) for _ in range(2)]
    found = 0
    for t in range(steps):
        k = torch.full((P,), 977 * t + 5, dtype=torch.int32, device=cuda)              # a new key a step
        q = (torch.randint(0, max(1, t), (P,), device=cuda, generator=g) * 977 + 5).to(torch.int32)
        q = torch.where(torch.rand(P, device=cuda, generator=g) < 0.3, q + 1, q)       # absent ones, to the end of their chain
        v = torch.randn(P, d, device=cuda, generator=g).to(BF16)
        pair[0].exchange(q, k, v, out[0], 1, 0)
        out[1].fill_(3.0)
        pair[1].exchange_phase(q, None, None, out[1], 0, 1)
        pair[1].exchange_phase(None, k, v, None, 0, 2)
        assert torch.equal(out[0], out[1])
        found += int((out[0] != 0).any(1).sum())
    pair[1].check()
    assert torch.equal(pair[0].counts, pair[1].counts) and int(pair[0].counts.min()) == steps
    assert 0.5 * P * (steps - 1) < found < 0.9 * P * steps


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_a_replaced_workspace_is_not_handed_out_while_another_stream_uses_it(cuda, fmt):
    P, T, d = 8, 2048, 16
    st = HashStore(d, groups=P, dtype=BF16, capacity=400000, device=cuda, quant=fmt)

    def items(t):
        k = torch.arange(P * t, dtype=torch.int32, device=cuda)
        return k, k, torch.zeros(P * t, d, dtype=BF16, device=cuda), torch.empty(P * t, d, dtype=BF16, device=cuda), t, 0
    small, large = items(T), items(4 * T)
    st.exchange(*small)
    old, size = st._ws.data_ptr(), st._ws.numel()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                    # some 50 ms: the exchanges below are still to come
        st.exchange(*small, check=False)
        st.exchange(*large, check=False)
    assert st._ws.data_ptr() != old
    again = torch.empty(size, dtype=torch.uint8, device=cuda)
    assert again.data_ptr() != old
    torch.cuda.synchronize()
    st.check()
    # partition p: codes p T ... of the small calls, 4 p T ... of the large one; shared in partition 0 alone
    assert len(st) == P * 4 * T + (P - 1) * T


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_a_store_stays_on_the_device_it_was_made_on(cuda, fmt):
    """Its workspace and streams too: the device it was given without an index is the one current then."""
    st = HashStore(16, groups=4, dtype=BF16, device="cuda", quant=fmt)
    assert st.device == st.table.device and st.device.index == torch.cuda.current_device()
    cache = LemaCache(ModelConfig(vocab_size=128, depth=1, dim=64, num_heads=4, d_qk=32, d_v=16), device="cuda", quant=fmt)
    assert cache.store.device.index is not None


@pytest.mark.parametrize("quant", [None, "int8"])
def test_half_steps_take_key_codes_of_the_other_width(cuda, quant):
    cfg = ModelConfig(vocab_size=128, depth=1, dim=64, num_heads=4, d_qk=32, d_v=16)
    c = [LemaCache(cfg, dtype=BF16, batch=1, max_cache_len=40, device=cuda, quant=quant) for _ in range(2)]
    g = torch.Generator().manual_seed(3)
    for _ in range(20):
        q, k = ((torch.randint(0, 5, (1, 4, 1), generator=g) - 3).to(torch.int32).to(cuda) for _ in range(2))
        v = torch.randn(1, 4, 1, 16, generator=g).to(BF16).to(cuda)
        s, got = c[1].layer(0).lookup(q, k.long(), v)
        c[1].layer(0).insert(s)
        assert torch.equal(c[0].layer(0).exchange(q, k, v), got)
    assert torch.equal(c[0].counts(), c[1].counts())
