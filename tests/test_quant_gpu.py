"""Quantised serving on the GPU: products with 4-bit weights against 64-bit sums, and the store with
rows held in 8 or 4 bits against a dictionary of rows quantised in plain torch."""
import numpy as np
import pytest
import torch

from latest_exact_match_attention_b200 import quant
from latest_exact_match_attention_b200._lib import LemaError, check_status
from latest_exact_match_attention_b200.cache import HashStore, LemaCache
from latest_exact_match_attention_b200.decode import decoder
from latest_exact_match_attention_b200.model import ModelConfig, Transformer
from latest_exact_match_attention_b200.quant import Int4Weight, dequantize_rows, quantize_rows

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def weight(n, k, group, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    scales = ((0.5 + torch.rand(n, -(-k // group), generator=g)) / (4.6 * k ** 0.5)).to(F16 if dtype == F16 else BF16)
    return codes.to(dev), scales.to(dev)


def dense64(codes, scales, group):
    return codes.double() * scales.double().repeat_interleave(group, 1)[:, : codes.shape[1]]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def sum_bound(x, w, dtype):
    """How far a sum over K products may be from the exact one, [M, N]. The products of integer codes with
    16-bit inputs are exact; each of at most K fp32 additions may be off by 2^-23 of the magnitudes summed so far
    (tensor cores may truncate), and the scaling by 2^-23. Many rows multiply weights rounded to the rows' 16-bit
    type: half a step of each product more. fp32 rows are cut into exact parts."""
    mag = x.double().abs() @ w.abs().t()
    per = (x.shape[1] + 8) * 2.0 ** -23 + (half_step(dtype) if dtype != F32 else 0)
    return mag * per


SHAPES = [(1, 16, 64), (1, 1, 1), (2, 17, 65), (8, 48, 128), (9, 100, 200), (16, 1536, 1536), (17, 40, 72), (33, 1000, 1100),
          (64, 256, 512), (65, 130, 192), (100, 128, 64), (127, 272, 320), (128, 128, 128), (129, 1024, 1024), (200, 24, 2048),
          (256, 1536, 1536), (300, 333, 777), (1000, 512, 448), (1, 50304, 128), (2048, 640, 512), (5000, 128, 96)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_int4_linear_against_64_bit_sums(cuda, M, N, K, dtype):
    group = (32, 64, 128)[(M + N + K) % 3]
    c, s = weight(N, K, group, dtype, M + N, cuda)
    g = torch.Generator().manual_seed(M * 7 + K)
    x = torch.randn(M, K, generator=g).to(dtype).to(cuda)
    r = torch.randn(M, N, generator=g).to(dtype).to(cuda) if M % 2 else None
    w = dense64(c, s, group)
    got = quant.int4_linear(x, Int4Weight.pack(c, s, group), residual=r)
    check_status(cuda, "int4_linear")
    assert got.dtype == dtype and got.shape == (M, N)
    ref = x.double() @ w.t() + (r.double() if r is not None else 0)
    bound = sum_bound(x, w, dtype) * (1 + half_step(dtype)) + half_step(dtype) * ref.abs() + 2.0 ** -24 * (ref.abs() + 1)
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} of the bound"
    # two independent roundings (weights in many rows, the output): each at most half a step, so at most
    # half a step / sqrt(3) in the mean square
    if dtype != F32 and N * M > 500:
        assert float((got.double() - ref).norm() / ref.norm()) <= half_step(dtype) * (2 / 3) ** 0.5


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,F,K", [(1, 8, 64), (1, 5, 33), (3, 64, 128), (8, 2816, 1024), (16, 100, 200), (40, 96, 160), (64, 128, 256),
                                   (96, 72, 512), (130, 200, 192), (256, 1024, 512), (700, 333, 328), (3000, 64, 128)])
def test_int4_swiglu_against_64_bit_sums(cuda, M, F, K, dtype):
    group = (32, 64, 128)[(M + F) % 3]
    (cg, sg), (cu, su) = weight(F, K, group, dtype, M, cuda), weight(F, K, group, dtype, M + 1, cuda)
    x = (torch.randn(M, K, generator=torch.Generator().manual_seed(F)) * 2).to(dtype).to(cuda)
    got = quant.int4_swiglu(x, Int4Weight.pack_gate_up(cg, sg, cu, su, group))
    check_status(cuda, "int4_swiglu")
    wg, wu = dense64(cg, sg, group), dense64(cu, su, group)
    gate, up = x.double() @ wg.t(), x.double() @ wu.t()
    silu = gate * torch.sigmoid(gate)
    ref = silu * up
    # |silu'| <= 1.1; the exponential, the quotient and the product are within 2^-20 together
    bg, bu = sum_bound(x, wg, dtype), sum_bound(x, wu, dtype)
    bound = 1.1 * bg * (up.abs() + bu) + (silu.abs()) * bu
    bound = bound + (half_step(dtype) + 2.0 ** -20) * (ref.abs() + bound) + torch.finfo(dtype).tiny
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("M", [3, 150])
def test_int4_linear_takes_views(cuda, M):
    K, N = 192, 80
    c, s = weight(N, K, 64, BF16, 1, cuda)
    w = Int4Weight.pack(c, s, 64)
    big = torch.randn(M, 3 * K + 8, device=cuda).to(BF16)
    want = quant.int4_linear(big[:, K:2 * K].contiguous(), w)
    assert torch.equal(quant.int4_linear(big[:, K:2 * K], w), want)            # rows apart, 16-byte aligned
    odd = torch.empty(M, K + 5, device=cuda, dtype=BF16)
    odd[:, 1:K + 1] = big[:, K:2 * K]
    assert torch.equal(quant.int4_linear(odd[:, 1:K + 1], w), want) or M > 32  # unaligned rows: the few-rows kernel
    off = quant.int4_linear(odd[:, 1:K + 1], w).float() - want.float()
    assert float(off.norm() / want.float().norm()) <= 2 * half_step(BF16)
    assert torch.equal(quant.int4_linear(big[:, K:2 * K].t().contiguous().t(), w), want)   # columns apart: copied
    assert torch.equal(quant.int4_linear(big[:, K:2 * K].reshape(1, M, 1, K), w), want.view(1, M, 1, N))
    assert torch.equal(quant.int4_linear(big[0, K:2 * K], w), quant.int4_linear(big[:1, K:2 * K], w)[0])
    one = big[:1, K:2 * K].expand(M, K)                                        # one row for all
    assert torch.equal(quant.int4_linear(one, w), quant.int4_linear(one.contiguous(), w))
    rbig = torch.randn(M, 2 * N, device=cuda).to(BF16)
    assert torch.equal(quant.int4_linear(big[:, K:2 * K], w, rbig[:, N:]),
                       quant.int4_linear(big[:, K:2 * K], w, rbig[:, N:].contiguous()))
    assert quant.int4_linear(big[:0, :K], w).shape == (0, N)


def test_int4_linear_refuses(cuda):
    c, s = weight(32, 64, 64, BF16, 0, cuda)
    w = Int4Weight.pack(c, s, 64)
    x = torch.randn(4, 64, device=cuda).to(BF16)
    with pytest.raises(LemaError, match="rows of 64"):
        quant.int4_linear(x[:, :32], w)
    with pytest.raises(LemaError, match="fp32, bf16 or fp16"):
        quant.int4_linear(x.double(), w)
    with pytest.raises(LemaError, match="residual"):
        quant.int4_linear(x, w, x)
    with pytest.raises(LemaError, match="residual"):
        quant.int4_linear(x, w, torch.zeros(4, 32, device=cuda))
    with pytest.raises(LemaError, match="CUDA tensors only"):
        quant.int4_linear(x, w.to("cpu"))


@pytest.mark.parametrize("M", [2, 100])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_with_infinities_touch_only_themselves(cuda, M, dtype):
    K, N = 160, 48
    c, s = weight(N, K, 32, dtype, 5, cuda)
    c = torch.where(c == 0, torch.ones_like(c), c)
    x = torch.randn(M, K, device=cuda).to(dtype)
    w = Int4Weight.pack(c, s, 32)
    clean = quant.int4_linear(x, w)
    x[1, 7] = float("inf")
    got = quant.int4_linear(x, w)
    assert torch.equal(got[0], clean[0])
    if M > 2:
        assert torch.equal(got[2:], clean[2:])
    assert torch.equal(got[1], torch.where(c[:, 7] > 0, float("inf"), float("-inf")).to(dtype))
    x[1, 7] = float("nan")
    got = quant.int4_linear(x, w)
    assert bool(got[1].isnan().all()) and torch.equal(got[0], clean[0])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_int4_products_repeat_capture_and_share(cuda, M):
    """The same bits every time, on any stream, from a graph, and from two streams at once."""
    K, N = 512, 768
    c, s = weight(N, K, 128, BF16, 2, cuda)
    w = Int4Weight.pack(c, s, 128)
    xs = [torch.randn(M, K, device=cuda).to(BF16) for _ in range(2)]
    want = [quant.int4_linear(x, w) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        a = quant.int4_linear(xs[0], w)
        with torch.cuda.stream(side):
            b = quant.int4_linear(xs[1], w)
        torch.cuda.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = quant.int4_linear(quant.int4_linear(static, w)[:, :K], w)
    for x in xs:
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, quant.int4_linear(quant.int4_linear(x, w)[:, :K], w))


def test_rows_behind_the_last_are_left(cuda):
    """The outputs' neighbours keep their bytes: y is written in place of a slice of a larger buffer."""
    from latest_exact_match_attention_b200._lib import call, ptr, stream_handle
    for M, N, K in [(3, 17, 64), (70, 33, 128), (130, 130, 192)]:
        c, s = weight(N, K, 32, BF16, M, cuda)
        w = Int4Weight.pack(c, s, 32)
        x = torch.randn(M, K, device=cuda).to(BF16)
        buf = torch.full((M + 2, N + 3), 7.0, dtype=BF16, device=cuda)
        y = buf[1: M + 1, 1: N + 1]
        call("lema_int4_linear", ptr(x), 1, M, K, K, ptr(w.packed), ptr(w.scales), 1, 32, N, 0, None, N, y.data_ptr(), N + 3,
             None, stream_handle(cuda))
        assert torch.equal(y, quant.int4_linear(x, w)) or M > 32
        frame = buf.clone()
        frame[1: M + 1, 1: N + 1] = 7.0
        assert bool((frame == 7.0).all())


# ------------------------------------------------------------------ the store


class Dict:
    """The store's semantics, partition by partition, on rows quantised in plain torch (on the host)."""

    def __init__(self, P, d, fmt, dtype):
        self.m, self.d, self.fmt, self.dtype = [dict() for _ in range(P)], d, fmt, dtype

    def exchange(self, q, k, v):
        """q, k [P, T] codes, v [P, T, d] (host): the retrieved rows [P, T, d]."""
        held = dequantize_rows(quantize_rows(v, self.fmt), self.fmt, self.d, self.dtype)
        out = torch.zeros_like(v)
        q, k = q.tolist(), k.tolist()
        for p, m in enumerate(self.m):
            for t in range(v.shape[1]):
                if q[p][t] in m:
                    out[p, t] = m[q[p][t]]
                m[k[p][t]] = held[p, t]
        return out


def same(a, b):
    """Equal bits, NaNs at the same places."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def stream(rng, P, T, d, dtype, span=30, wide=False):
    q, k = (rng.integers(0, span, size=(P, T)).astype(np.int64 if wide else np.int32) for _ in range(2))
    if wide:
        q, k = q * 0x1234567890123, k * 0x1234567890123
    v = rng.standard_normal((P, T, d)) * np.exp(2 * rng.standard_normal((P, T, 1)))
    return torch.from_numpy(q), torch.from_numpy(k), torch.from_numpy(v).to(dtype)


@pytest.mark.parametrize("fmt", ["int8", "fp8", "int4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("P,d,T", [(5, 24, 1), (70, 24, 40), (3, 64, 200), (9, 1, 17), (4, 7, 9), (6, 33, 1), (2, 130, 30), (3, 256, 12)])
def test_store_holds_what_the_formats_say(cuda, P, d, T, dtype, fmt):
    rng = np.random.default_rng(P * d + T)
    st = HashStore(d, groups=P + 3, dtype=dtype, capacity=40 * (P + 3), device=cuda, quant=fmt)
    ref = Dict(P, d, fmt, dtype)
    for _ in range(4 if T > 1 else 12):
        q, k, v = stream(rng, P, T, d, dtype, wide=d % 2 == 0)
        out = torch.full((P * T, d), float("nan"), dtype=dtype, device=cuda)
        st.exchange(q.to(cuda).view(-1), k.to(cuda).view(-1), v.to(cuda).view(-1, d), out, T, 3)
        assert torch.equal(out.cpu().view(P, T, d), ref.exchange(q, k, v))
    assert [int(c) for c in st.counts.cpu()] == [0, 0, 0] + [len(m) for m in ref.m]
    g, c, rows = st.dump()
    got = {(int(a) - 3, int(b)): r for a, b, r in zip(g, c, rows.cpu())}
    want = {(p, key & (0xFFFFFFFFFFFFFFFF if d % 2 == 0 else 0xFFFFFFFF)): r for p, m in enumerate(ref.m) for key, r in m.items()}
    assert got.keys() == want.keys() and all(torch.equal(got[key], want[key]) for key in want)


@pytest.mark.parametrize("fmt", ["int8", "fp8", "int4"])
@pytest.mark.parametrize("lanes", ["8", "16", "32"])
def test_every_group_of_lanes_gives_the_same_bytes(cuda, fmt, lanes, monkeypatch):
    monkeypatch.setenv("LEMA_K3_GROUP", lanes)
    rng = np.random.default_rng(4)
    P, d = 40, 24
    st = HashStore(d, groups=P, dtype=BF16, capacity=1100, device=cuda, quant=fmt, segments=4)   # load up to 0.95
    ref = Dict(P, d, fmt, BF16)
    for T in (30, 1, 1, 1, 17):
        q, k, v = stream(rng, P, T, d, BF16, span=26)
        out = torch.empty(P * T, d, dtype=BF16, device=cuda)
        st.exchange(q.to(cuda).view(-1), k.to(cuda).view(-1), v.to(cuda).view(-1, d), out, T, 0)
        assert torch.equal(out.cpu().view(P, T, d), ref.exchange(q, k, v))
    live = st.table.view(-1)[: 16 * st.cap].view(torch.int64).view(st.cap, 2)[:, 1] >= 2
    rows = st.table.view(-1)[16 * st.cap:].view(st.cap, -1)[live]
    g, c, vals = st.dump()
    key = {(p, k): r for p, m in enumerate(ref.m) for k, r in m.items()}
    for a, b, held, v in zip(g.tolist(), c.tolist(), rows.cpu(), vals.cpu()):
        assert torch.equal(v, key[(a, b)])
        used = quant.row_bytes(fmt, d)
        assert held.numel() == used and not held[28 if fmt != "int4" else 16:].any()      # the padding is zero


@pytest.mark.parametrize("fmt", ["int8", "fp8", "int4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_at_the_ends_of_their_type(cuda, fmt, dtype):
    """Subnormal, largest, infinite and NaN values, ties and zeros: the same bits as in plain torch."""
    d = 40
    fi = torch.finfo(dtype)
    rows = [torch.zeros(d), torch.full((d,), fi.max), torch.full((d,), -fi.max), torch.full((d,), fi.smallest_normal),
            torch.full((d,), fi.smallest_normal * fi.eps), torch.linspace(-127, 127, d), torch.arange(d) * 0.5 - 7,
            torch.linspace(-7, 7, d) * fi.smallest_normal, torch.linspace(-1, 1, d) * 190 * fi.smallest_normal * fi.eps,
            torch.linspace(-448, 448, d), torch.linspace(-449, 449, d), 2.0 ** torch.linspace(-20, 8, d), torch.ones(d) * float("inf")]
    rows = torch.stack(rows).to(dtype)
    rows = torch.cat([rows, rows[5:7].clone()])
    rows[-1, 3] = float("nan")
    rows[-2, 35] = float("-inf")
    rng = np.random.default_rng(1)
    rows = torch.cat([rows, (torch.from_numpy(rng.integers(-254, 255, (200, d))) / 2).to(dtype)])      # ties of int8, and near them
    P = rows.shape[0]
    code = torch.arange(P, dtype=torch.int32, device=cuda)
    st = HashStore(d, groups=P, dtype=dtype, capacity=4 * P, device=cuda, quant=fmt)
    out = torch.empty(P, d, dtype=dtype, device=cuda)
    st.exchange(code, code, rows.to(cuda), out, 1, 0)
    assert bool((out == 0).all())
    st.exchange(code, code, rows.to(cuda), out, 1, 0)
    want = dequantize_rows(quantize_rows(rows, fmt), fmt, d, dtype)
    assert same(out.cpu(), want)
    assert bool(want[1].isfinite().all())
    # the same rows inside one call (T = 2: the second position finds the first's key)
    st2 = HashStore(d, groups=P, dtype=dtype, capacity=4 * P, device=cuda, quant=fmt)
    two = code.repeat_interleave(2)
    out2 = torch.empty(2 * P, d, dtype=dtype, device=cuda)
    st2.exchange(two, two, rows.to(cuda).repeat_interleave(2, 0), out2, 2, 0)
    assert same(out2.cpu().view(P, 2, d)[:, 1], want) and bool((out2.view(P, 2, d)[:, 0] == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "fp8", "int4"])
def test_any_chunking_gives_the_same_rows(cuda, fmt):
    B, H, T, d = 2, 3, 60, 24
    cfg = ModelConfig(vocab_size=128, depth=1, dim=H * d, num_heads=H, d_qk=32, d_v=d)
    rng = np.random.default_rng(8)
    q, k, v = stream(rng, B * H, T, d, BF16)
    q, k, v = q.view(B, H, T).to(cuda), k.view(B, H, T).to(cuda), v.view(B, H, T, d).to(cuda)
    v = v.transpose(1, 2).contiguous().transpose(1, 2)           # as a projection leaves it
    got = []
    for step in (60, 16, 7, 1):
        c = LemaCache(cfg, dtype=BF16, batch=B, max_cache_len=T, device=cuda, quant=fmt)
        parts = [c.layer(0).exchange(q[..., s:s + step], k[..., s:s + step], v[:, :, s:s + step]).clone() for s in range(0, T, step)]
        got.append(torch.cat(parts, 2))
        c.check()
    assert all(torch.equal(got[0], g) for g in got[1:])
    c = LemaCache(cfg, dtype=BF16, batch=B, max_cache_len=T, device=cuda, quant=fmt)
    split = []
    for t in range(T):
        s, rows = c.layer(0).lookup(q[..., t:t + 1], k[..., t:t + 1], v[:, :, t:t + 1])
        split.append(rows.clone())
        c.layer(0).insert(s)
    assert torch.equal(torch.cat(split, 2), got[0])


def test_a_full_quantised_store_raises(cuda):
    st = HashStore(16, groups=64, dtype=BF16, capacity=32, device=cuda, quant="int4")
    k = torch.arange(64, dtype=torch.int32, device=cuda)
    v = torch.zeros(64, 16, dtype=BF16, device=cuda)
    with pytest.raises(RuntimeError, match="full"):
        st.exchange(k, k, v, torch.empty_like(v), 1, 0)
    assert len(st) == 32


def test_quantised_store_refuses(cuda):
    with pytest.raises(ValueError, match="row format"):
        HashStore(16, groups=4, device=cuda, quant="int2")
    with pytest.raises(ValueError, match="1 to 256"):
        HashStore(300, groups=4, device=cuda, quant="int8")
    st = HashStore(16, groups=4, dtype=BF16, device=cuda, quant="int8")
    k = torch.zeros(4, dtype=torch.int32, device=cuda)
    v = torch.zeros(4, 16, device=cuda)
    with pytest.raises(ValueError, match="quantises"):
        st.exchange(k, k, v, torch.empty_like(v), 1, 0)
    with pytest.raises(ValueError, match="rows"):
        st.exchange(k, k, v[:, :8].to(BF16), torch.empty(4, 8, dtype=BF16, device=cuda), 1, 0)
    with pytest.raises(ValueError, match="outside"):
        st.exchange(k, k, v.to(BF16), torch.empty(4, 16, dtype=BF16, device=cuda), 1, 1)


@pytest.mark.parametrize("T", [1, 3])
def test_quantised_store_refuses_host_tensors(cuda, T):
    st = HashStore(16, groups=4, dtype=BF16, device="cuda", quant="int8")     # no index: the current device
    k = torch.zeros(4 * T, dtype=torch.int32, device=cuda)
    v = torch.ones(4 * T, 16, dtype=BF16, device=cuda)
    o = torch.empty_like(v)
    for args in ((k.cpu(), k, v, o), (k, k.cpu(), v, o), (k, k, v.cpu(), o), (k, k, v, o.cpu())):
        with pytest.raises(LemaError, match="the store is on"):
            st.exchange(*args, T, 0)
    assert len(st) == 0
    st.exchange(k, k, v, o, T, 0)
    assert len(st) == 4


# ------------------------------------------------------------------ together, in the model


def model(dev, dtype=BF16, group=64):
    torch.manual_seed(1)
    m = Transformer(ModelConfig(vocab_size=512, depth=2, dim=256, num_heads=8, d_qk=32, d_v=32)).to(dev).to(dtype).eval()
    return m


def test_quantised_model_is_the_model_of_its_dequantised_weights(cuda):
    """fp32: a model whose weights are replaced by what the codes stand for gives the same logits up to fp32
    sums in another order. fp32 logits of two fp32 models differ by sums of at most 768 terms in each of 2 layers
    of 4 products: 2^-24 * sqrt(768) * 8 < 2e-5 of their size in the mean square, held to 1e-4."""
    m, ref = model(cuda, F32), model(cuda, F32)
    m.quantize_weights_(group=64)
    for b, r in zip(m.blocks, ref.blocks):
        gate, up = b.mlp.gate_up.weight4.dequantize()
        for lin, w in ((r.attn.v_proj, b.attn.v_proj.weight4.dequantize()), (r.attn.o_proj, b.attn.o_proj.weight4.dequantize()),
                       (r.mlp.gate, gate), (r.mlp.up, up), (r.mlp.down, b.mlp.down.weight4.dequantize())):
            lin.weight.data.copy_(w)
    ref.lm_head.weight.data.copy_(m.lm_head.weight4.dequantize())
    idx = torch.randint(0, 60, (3, 50), device=cuda)
    a, b = m(idx).double(), ref(idx).double()
    assert float((a - b).norm() / b.norm()) < 1e-4
    c = m.new_cache("hbm", max_cache_len=64, batch=3)
    chunks = torch.cat([m(idx[:, s:s + 10], cache=c) for s in range(0, 50, 10)], 1).double()
    assert float((chunks - a).norm() / a.norm()) < 1e-4


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("fmt", [None, "int8", "fp8", "int4"])
def test_graph_decoding_with_both_quantised(cuda, fmt, split, monkeypatch):
    """Prefill through the quantised store, then decode: one graph per step gives the eager tokens and entries."""
    monkeypatch.setenv("LEMA_DECODE_SPLIT", split)
    m = model(cuda).quantize_weights_(group=64)
    prompt = torch.randint(0, 60, (4, 16), device=cuda)
    caches = [m.new_cache("hbm", max_cache_len=64, batch=4, quant=fmt) for _ in range(2)]
    for c in caches:
        m(prompt[:, :-1], cache=c, return_logits=False)
    t, eager = prompt[:, -1:], []
    for _ in range(30):
        t = m(t, cache=caches[0]).argmax(-1)
        eager.append(t.clone())
    d = decoder(m, caches[1], tok=prompt[:, -1:])
    graph = [d.step().clone() for _ in range(30)]
    caches[1].check()
    assert torch.equal(torch.cat(eager, 1), torch.cat(graph, 1))
    assert torch.equal(caches[0].counts(), caches[1].counts())
    a, b = (sorted(zip(*(x.tolist() for x in c.dump()[:4]), c.dump()[4].float().tolist())) for c in caches)
    assert a == b
    if fmt is not None:
        assert caches[0].nbytes() < m.new_cache("hbm", max_cache_len=64, batch=4).nbytes()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_unaligned_rows_take_the_many_rows_kernel(cuda, dtype):
    """Odd widths and offsets are copied into aligned rows: the same numbers as from aligned rows of the same values."""
    M, K, N = 180, 150, 64
    c, s = weight(N, K, 64, dtype, 9, cuda)
    w = Int4Weight.pack(c, s, 64)
    room = torch.randn(M + 1, 160, device=cuda).to(dtype)
    want = quant.int4_linear(room[:M, :K], w)                       # 16-byte aligned rows
    assert torch.equal(quant.int4_linear(room[:M, :K].contiguous(), w), want)            # rows of 300 bytes
    flat = torch.empty(M * 160 + 1, dtype=dtype, device=cuda)[1:]
    flat.view(M, 160).copy_(room[:M])
    assert torch.equal(quant.int4_linear(flat.view(M, 160)[:, :K], w), want)             # off by one element
    assert torch.equal(quant.int4_linear(room[:M, :K].reshape(2, M // 2, K), w), want.view(2, M // 2, N))
    assert torch.equal(quant.int4_linear(room[:M, :K].reshape(M // 2, 2, K).transpose(0, 1), w), want.view(M // 2, 2, N).transpose(0, 1))


@pytest.mark.parametrize("dtype,scale", [(BF16, F16), (F16, BF16), (F32, F16)])
@pytest.mark.parametrize("M", [1, 12, 30, 100, 300])
def test_scales_of_another_type_than_the_rows(cuda, M, dtype, scale):
    N, K = 72, 320
    c, s = weight(N, K, 64, scale, M, cuda)
    assert s.dtype == scale
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype).to(cuda)
    got = quant.int4_linear(x, Int4Weight.pack(c, s, 64))
    w = dense64(c, s, 64)
    ref = x.double() @ w.t()
    bound = sum_bound(x, w, dtype) * (1 + half_step(dtype)) + half_step(dtype) * ref.abs() + 2.0 ** -24 * (ref.abs() + 1)
    assert bool(((got.double() - ref).abs() <= bound).all())
    gu = quant.int4_swiglu(x, Int4Weight.pack_gate_up(c, s, c, s, 64))
    assert bool(gu.isfinite().all()) and gu.shape == (M, N)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K", [40, 64, 72, 96, 104, 136, 160, 200, 296])
@pytest.mark.parametrize("M", [7, 33, 140])
def test_every_tail_of_k(cuda, M, K, group):
    """K ends inside a block, inside a half block and inside a scale group, in both kernels."""
    N = 40
    c, s = weight(N, K, group, BF16, K, cuda)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).to(BF16).to(cuda)
    got = quant.int4_linear(x, Int4Weight.pack(c, s, group))
    w = dense64(c, s, group)
    ref = x.double() @ w.t()
    bound = sum_bound(x, w, BF16) * (1 + half_step(BF16)) + half_step(BF16) * ref.abs() + 2.0 ** -24 * (ref.abs() + 1)
    assert bool(((got.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("M,N,K", [(4096, 1024, 8192), (64, 128, 65536)])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_exact(cuda, monkeypatch, M, N, K):
    """Waits bounded to 1 ns run out (tiles alone, and tiles whose K a cluster splits): the status word says so, nothing
    hangs, and the next call with the usual bound gives the bits of the first. A wait is given up after eight tries,
    which the hardware may each suspend for about a microsecond: an accumulator here takes 128 stages, over 40 us."""
    c, s = weight(N, K, 128, BF16, 0, cuda)
    w = Int4Weight.pack(c, s, 128)
    x = torch.randn(M, K, device=cuda).to(BF16)
    want = quant.int4_linear(x, w)
    check_status(cuda)
    monkeypatch.setenv("LEMA_WAIT_NS", "1")
    quant.int4_linear(x, w)
    torch.cuda.synchronize()
    with pytest.raises(LemaError, match="ran out"):
        check_status(cuda, "int4_linear")
    monkeypatch.delenv("LEMA_WAIT_NS")
    assert torch.equal(quant.int4_linear(x, w), want)
    check_status(cuda)


def test_a_captured_chunk_keeps_its_workspace(cuda):
    """A graph of a prefill chunk still replays after a larger eager call replaced the store's workspace."""
    P, T, d = 4, 64, 24
    rng = np.random.default_rng(3)
    st = HashStore(d, groups=P, dtype=BF16, capacity=40000, device=cuda, quant="int8")
    q, k, v = (t.to(cuda) for t in stream(rng, P, T, d, BF16, span=500))
    out = torch.empty(P * T, d, dtype=BF16, device=cuda)
    st.exchange(q, k, v, out, T, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st.exchange(q, k, v, out, T, 0, check=False)
    want = torch.empty_like(out)
    st.exchange(q, k, v, want, T, 0)
    big = [t.to(cuda) for t in stream(rng, P, 40 * T, d, BF16, span=500)]
    codes = [b + 1000 for b in big[:2]]                       # other codes: the graph's own entries stay
    st.exchange(*codes, big[2], torch.empty(P * 40 * T, d, dtype=BF16, device=cuda), 40 * T, 0)
    fill = [torch.randint(0, 255, (1 << 20,), dtype=torch.uint8, device=cuda) for _ in range(8)]
    graph.replay()
    st.check()
    assert torch.equal(out, want) and len(fill) == 8


def test_other_shapes_of_codes_and_rows_are_the_same_items(cuda):
    B, H, d = 3, 4, 16
    st = [HashStore(d, groups=B * H, dtype=BF16, capacity=1000, device=cuda, quant="int8") for _ in range(2)]
    k = torch.arange(B * H, dtype=torch.int32, device=cuda) % 5
    v = torch.randn(B * H, d, device=cuda).to(BF16)
    out = [torch.empty(B * H, d, dtype=BF16, device=cuda), torch.empty(B, H, 1, d, dtype=BF16, device=cuda)]
    for _ in range(2):
        st[0].exchange(k, k, v, out[0], 1, 0)
        st[1].exchange(k.view(B, H, 1), k.view(B, H, 1), v.view(B, H, 1, d), out[1], 1, 0)
        assert torch.equal(out[0], out[1].view(B * H, d))
    with pytest.raises(ValueError, match="key codes"):
        st[0].exchange(k, k[:5], v, out[0], 1, 0)


@pytest.mark.parametrize("M,N,K,group,gated", [(4096, 512, 1536, 128, True), (6000, 1536, 1024, 64, False), (3000, 1000, 1096, 32, False),
                                               (512, 2048, 1536, 128, True), (200, 1536, 4096, 128, False), (40, 1536, 1536, 32, True)])
def test_many_rows_give_the_same_bits_every_time(cuda, M, N, K, group, gated):
    """Back to back, and behind passes that empty the caches: a missing wait anywhere in the ring shows as other bits."""
    c, s = weight(N, K, group, BF16, M, cuda)
    w = Int4Weight.pack_gate_up(c, s, c, s, group) if gated else Int4Weight.pack(c, s, group)
    call = quant.int4_swiglu if gated else quant.int4_linear
    x = torch.randn(M, K, device=cuda).to(BF16)
    want = call(x, w).clone()
    room = torch.empty(256 << 20, dtype=torch.uint8, device=cuda)
    other = torch.zeros((), dtype=torch.long, device=cuda)
    for i in range(60):
        if i % 3 == 0:
            room.fill_(i)
        other += (call(x, w) != want).sum()
    assert int(other) == 0
    check_status(cuda)


@pytest.mark.parametrize("M", [3, 64])
def test_weights_past_four_gigabytes(cuda, M):
    """The last block rows of a packed weight of 4.3 GB give what they give alone."""
    N, K = 131072 + 40, 65536
    rb = -(-N // 16)
    packed = torch.randint(-(1 << 31), 1 << 31, (rb, K // 64, 32, 4), dtype=torch.int32, device=cuda)
    scales = torch.rand(rb, K // 128, 8, 2, device=cuda).mul_(0.01).to(BF16)
    x = torch.randn(M, K, device=cuda).to(BF16)
    whole = quant.int4_linear(x, Int4Weight(packed, scales, N, K, 128))
    first = (rb // 8 - 2) * 8                            # two whole tiles of 8 block rows, and the ragged one
    n = N - 16 * first
    tail = quant.int4_linear(x, Int4Weight(packed[first:].contiguous(), scales[first:].contiguous(), n, K, 128))
    check_status(cuda)
    assert whole.shape == (M, N)
    # the same sums; a tile's split of K, and so their order, goes by the number of tiles
    assert float((whole[:, 16 * first:].double() - tail.double()).norm() / tail.double().norm()) <= 2 * half_step(BF16)
    assert bool(whole.isfinite().all())


def test_rows_of_a_table_past_four_gigabytes(cuda):
    P, d, cap = 3000, 24, 130_000_000                    # rows from 2.1 to 6.2 GB of a 6.2 GB table
    st = HashStore(d, groups=P, dtype=BF16, capacity=cap, device=cuda, quant="int8")
    assert st.nbytes() > 6_000_000_000
    ref = Dict(P, d, "int8", BF16)
    rng = np.random.default_rng(12)
    for T in (1, 5, 1, 1):
        q, k, v = stream(rng, P, T, d, BF16, span=6)
        out = torch.empty(P * T, d, dtype=BF16, device=cuda)
        st.exchange(q.to(cuda), k.to(cuda), v.to(cuda), out, T, 0)
        assert torch.equal(out.cpu().view(P, T, d), ref.exchange(q, k, v))
    assert len(st) == sum(len(m) for m in ref.m)
