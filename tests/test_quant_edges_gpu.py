"""Quantised serving where its kernels meet: the rule that picks one, the ends of 16-bit ranges, and the bytes a
quantised store holds."""
import pytest
import torch

from latest_exact_match_attention_b200 import quant
from latest_exact_match_attention_b200._lib import check_status
from latest_exact_match_attention_b200.quant import Int4Weight

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
