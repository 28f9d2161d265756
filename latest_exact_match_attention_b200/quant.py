"""Quantised serving: products with 4-bit weights, and the formats of value rows held in 8 or 4 bits.

    Int4Weight                 a projection's weight in 4 bits with group scales, laid out for the kernel
    quantize_weight(w, group)  round-to-nearest codes and scales of a weight
    int4_linear(x, w, r)       x @ dequantised(w).T (+ r)
    int4_swiglu(x, w)          silu(x @ gate.T) * (x @ up.T), both weights in 4 bits, one kernel
    Int4Linear, Int4SwiGLU     the modules `Transformer.quantize_weights_` puts in the model
    ROW_FORMATS, row_bytes, quantize_rows, dequantize_rows
                               the store's quantised rows (LemaCache(quant=...)) in plain torch

A weight is w[n][k] = s[n][k // group] * q[n][k] with q in -8 ... 7 and 16-bit scales: 4.125 bits a weight
with group 128. The kernels take rows in fp32, bf16 or fp16, any shape, one row to whole prompts; see
lema_int4_linear in include/lema_b200.h for the layout and the arithmetic. The reference has no quantised
form; the layers are those of code/lema/model.py:85-93 (SwiGLU), 160-163 (v_proj, o_proj) and 264 (lm_head).

Inference only: outputs carry no autograd graph. CUDA tensors only (packing itself also runs on the CPU,
so a checkpoint can be prepared without a GPU).
"""
from __future__ import annotations

import torch
from torch import nn

from ._lib import DTYPE_TAG, F32, LemaError, _status_words, device_status, lib, require_cuda

__all__ = ["Int4Weight", "Int4Linear", "Int4SwiGLU", "quantize_weight", "int4_linear", "int4_swiglu",
           "ROW_FORMATS", "row_bytes", "quantize_rows", "dequantize_rows"]

GROUPS = (32, 64, 128)
FEW_ROWS = 32       # up to this many rows have a kernel of their own, which reads rows of any alignment
# Unaligned 16-bit rows: above FEW_ROWS that kernel takes them too, 32 at a time with checked loads; a call on an aligned
# copy takes about 20 us of host time and 9 to 25 on the device. Rows are copied where there are many of them and where
# blocks of 16 x 64 weights times 32-row tiles exceed COPY_WORK (fp16, as they are / copied, us a call): 37 rows
# 1000 x 1100 (2268) 10.5 / 19.9, 64 rows 1000 x 2501 (5040) 15.9 / 20.1, 33 rows 8192 x 333 (6144) 17.3 / 19.7, 128 rows
# 4096 x 333 (6144) 22.1 / 19.7, 96 rows 1000 x 2501 (7560) 30.1 / 20.3, 33 rows 50304 x 1100 (113184) 173 / 29, 128 rows 515 / 31.
COPY_ROWS = 128
COPY_WORK = 6000

# ------------------------------------------------------------------ 4-bit weights


def quantize_weight(w: torch.Tensor, group: int = 128, scale_dtype: torch.dtype | None = None):
    """Round-to-nearest codes int8 [N, K] and scales [N, ceil(K / group)] of a weight [N, K]:
    s = amax / 7 of each `group` inputs, rounded to `scale_dtype` (fp16 for an fp16 weight, else
    bf16), q = rint(w / s) in -8 ... 7. An all-zero group has scale 0."""
    if w.dim() != 2:
        raise ValueError(f"a weight is [N, K], got {tuple(w.shape)}")
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}, got {group}")
    N, K = w.shape
    dt = scale_dtype or (torch.float16 if w.dtype == torch.float16 else torch.bfloat16)
    f = torch.nn.functional.pad(w.detach().float(), (0, -K % group)).view(N, -1, group)
    s = (f.abs().amax(-1) / 7).to(dt)
    sf = s.float()[..., None]
    q = torch.where(sf > 0, f / sf, torch.zeros_like(f)).round().clamp(-8, 7)
    return q.view(N, -1)[:, :K].to(torch.int8), s


def _block_rows(codes: torch.Tensor, scales: torch.Tensor, per: int):
    """Codes + 8 and scales padded to whole blocks, [n_rb, per, K padded to 64], [n_rb, per, G]."""
    N, K = codes.shape
    u = torch.nn.functional.pad((codes + 8).to(torch.uint8), (0, -K % 64, 0, -N % per), value=8)
    s = torch.nn.functional.pad(scales, (0, 0, 0, -N % per))
    return u.view(-1, per, u.shape[1]), s.view(-1, per, s.shape[1])


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, group: int):
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}, got {group}")
    if codes.dim() != 2 or codes.dtype != torch.int8 or not codes.numel():
        raise ValueError(f"codes must be a non-empty int8 [N, K], got {codes.dtype} {tuple(codes.shape)}")
    want = (codes.shape[0], -(-codes.shape[1] // group))
    if tuple(scales.shape) != want or scales.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"scales must be bf16 or fp16 [N, ceil(K / group)] = {list(want)}, got "
                         f"{scales.dtype} {tuple(scales.shape)}")
    if scales.device != codes.device:
        raise ValueError(f"codes on {codes.device}, scales on {scales.device}")
    lo, hi = (int(v) for v in codes.aminmax())
    if lo < -8 or hi > 7:
        raise ValueError(f"codes must lie in -8 ... 7, got {lo} ... {hi}")


class Int4Weight:
    """A [n, k] weight (gated: a gate and an up weight of n features each) in the kernel's layout:
    `packed` int32 [block rows, block columns, 32, 4] and `scales` [block rows, groups, 8, 2]."""

    __slots__ = ("packed", "scales", "n", "k", "group", "gated")

    def __init__(self, packed, scales, n: int, k: int, group: int, gated: bool = False):
        self.packed, self.scales, self.n, self.k, self.group, self.gated = packed, scales, n, k, group, gated
        per = 8 if gated else 16
        rb = -(-n // per)
        if group not in GROUPS or packed.dtype != torch.int32 or scales.dtype not in (torch.bfloat16, torch.float16) \
                or tuple(packed.shape) != (rb, -(-k // 64), 32, 4) or tuple(scales.shape) != (rb, -(-k // group), 8, 2) \
                or not packed.is_contiguous() or not scales.is_contiguous() or packed.device != scales.device:
            raise ValueError(f"not a packed 4-bit weight of {n} x {k}, group {group}: packed {packed.dtype} "
                             f"{tuple(packed.shape)}, scales {scales.dtype} {tuple(scales.shape)}")

    @staticmethod
    def pack(codes: torch.Tensor, scales: torch.Tensor, group: int = 128) -> "Int4Weight":
        """From codes int8 [N, K] in -8 ... 7 and scales [N, ceil(K / group)] (bf16 or fp16)."""
        _check_codes(codes, scales, group)
        u, s = _block_rows(codes, scales, 16)
        return Int4Weight._lay_out(u, s, codes.shape[0], codes.shape[1], group, False)

    @staticmethod
    def pack_gate_up(gate: torch.Tensor, gate_scales: torch.Tensor, up: torch.Tensor, up_scales: torch.Tensor,
                     group: int = 128) -> "Int4Weight":
        """The gate and up weights of one MLP, [F, K] each: block rows of 8 gate features and the 8
        up features of the same indices, so that one lane's sums hold both."""
        _check_codes(gate, gate_scales, group)
        _check_codes(up, up_scales, group)
        if gate.shape != up.shape or gate_scales.dtype != up_scales.dtype or gate.device != up.device:
            raise ValueError(f"gate and up differ: {tuple(gate.shape)} {gate_scales.dtype} on {gate.device}, "
                             f"{tuple(up.shape)} {up_scales.dtype} on {up.device}")
        (ug, sg), (uu, su) = _block_rows(gate, gate_scales, 8), _block_rows(up, up_scales, 8)
        return Int4Weight._lay_out(torch.cat([ug, uu], 1), torch.cat([sg, su], 1), gate.shape[0], gate.shape[1], group, True)

    @staticmethod
    def _lay_out(u, s, n, k, group, gated):
        rb, _, kp = u.shape
        # rows i a (feature 8 i + a); inputs c h t j p e (64 c + 32 h + 8 t + 4 j + 2 p + e)
        # each a field of bits 16 e + 8 p + 4 i, one at a time: no 32-bit copy of every code
        u = u.view(rb, 2, 8, kp // 64, 2, 4, 2, 2, 2).permute(8, 7, 1, 0, 3, 2, 5, 4, 6).reshape(8, -1)
        words = u[0].to(torch.int32)
        for field in range(1, 8):
            words |= u[field].to(torch.int32) << 4 * field
        return Int4Weight(words.view(rb, kp // 64, 32, 4).contiguous(), s.unflatten(1, (2, 8)).permute(0, 3, 2, 1).contiguous(), n, k, group, gated)

    def codes(self):
        """The codes int8 and scales as packed: [n, k], [n, groups] (gated: a pair of them)."""
        rb, kb = self.packed.shape[:2]
        shift = torch.arange(8, device=self.packed.device, dtype=torch.int32) * 4
        u = ((self.packed.view(rb, kb, 8, 4, 2, 2, 1) >> shift) & 15).view(rb, kb, 8, 4, 2, 2, 2, 2, 2)
        u = u.permute(0, 8, 2, 1, 4, 3, 5, 7, 6).reshape(rb, 16, kb * 64)[..., : self.k]
        q, s = (u - 8).to(torch.int8), self.scales.permute(0, 3, 2, 1).flatten(1, 2)
        if not self.gated:
            return q.reshape(-1, self.k)[: self.n], s.reshape(rb * 16, -1)[: self.n]
        return tuple((q[:, i:i + 8].reshape(-1, self.k)[: self.n], s[:, i:i + 8].reshape(rb * 8, -1)[: self.n])
                     for i in (0, 8))

    def dequantize(self):
        """The weight in fp32: [n, k] (gated: the pair (gate, up))."""
        def dense(q, s):
            return q.float() * s.float().repeat_interleave(self.group, 1)[:, : self.k]
        c = self.codes()
        return (dense(*c[0]), dense(*c[1])) if self.gated else dense(*c)

    def to(self, device) -> "Int4Weight":
        return Int4Weight(self.packed.to(device), self.scales.to(device), self.n, self.k, self.group, self.gated)

    def nbytes(self) -> int:
        return self.packed.numel() * 4 + self.scales.numel() * self.scales.element_size()


def _product(name: str, x: torch.Tensor, w: Int4Weight, residual: torch.Tensor | None) -> torch.Tensor:
    # a decode step makes several of these calls a layer and its kernels take a few microseconds: the
    # common case (rows side by side) stays short
    packed, k, n = w.packed, w.k, w.n
    dev = packed.device
    if x.device != dev or not x.is_cuda or (residual is not None and residual.device != dev):
        require_cuda(x, packed, residual)
    tag = DTYPE_TAG.get(x.dtype)
    if tag is None:
        raise LemaError(f"{name} takes fp32, bf16 or fp16 rows, got {x.dtype}")
    shape = x.shape
    if not shape or shape[-1] != k:
        raise LemaError(f"{name}: rows of {k} values wanted, got {tuple(shape)}")
    ldx = k
    if not x.is_contiguous():
        x = x if len(shape) == 2 else x.reshape(-1, k)
        ldx = x.stride(0)
        if x.stride(1) != 1 or (x.shape[0] > 1 and ldx < k):
            x, ldx = x.contiguous(), k
    M = x.numel() // k
    if (M > FEW_ROWS and ((ldx | x.data_ptr() >> 1) & 7) and tag != F32 and k >= 64
            and (M > COPY_ROWS or (packed.numel() >> 7) * ((M + 31) >> 5) > COPY_WORK)):
        # rows that the many-rows kernel cannot load in 16-byte pieces: an aligned copy of them
        ldx = -(-k // 8) * 8
        rows = x.new_empty((M, ldx))
        rows[:, :k].copy_(x if x.dim() == 2 else x.view(M, k))
        x = rows
    y = x.new_empty((M, n)) if len(shape) == 2 else x.new_empty(shape[:-1] + (n,))
    rp, ldr = None, n
    if residual is not None:
        if residual.shape != y.shape or residual.dtype != x.dtype:
            raise LemaError(f"{name}: the residual must be {x.dtype} {tuple(y.shape)}, got {residual.dtype} "
                            f"{tuple(residual.shape)}")
        if not residual.is_contiguous():
            residual = residual if len(shape) == 2 else residual.reshape(-1, n)
            ldr = residual.stride(0)
            if residual.stride(1) != 1 or (M > 1 and ldr < n):
                residual, ldr = residual.contiguous(), n
        rp = residual.data_ptr()
    if M == 0:
        return y
    idx, scales = dev.index, w.scales
    status = _status_words.get(idx)
    if status is None:
        status = device_status(dev)
    args = (x.data_ptr(), tag, M, k, ldx, packed.data_ptr(), scales.data_ptr(), DTYPE_TAG[scales.dtype], w.group, n,
            w.gated, rp, ldr, y.data_ptr(), n, status.data_ptr(), torch._C._cuda_getCurrentRawStream(idx))
    L = lib()
    if idx == torch._C._cuda_getDevice():
        rc = L.lema_int4_linear(*args)
    else:
        with torch.cuda.device(dev):
            rc = L.lema_int4_linear(*args)
    if rc:
        raise LemaError(f"{name} failed (code {rc}): {L.lema_last_error().decode(errors='replace')}")
    return y


def int4_linear(x: torch.Tensor, w: Int4Weight, residual: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] times the dequantised weight's transpose, plus `residual` [..., N] if given, in x's
    dtype: fp32 sums, one rounding."""
    if w.gated:
        raise LemaError("int4_linear takes a plain weight; a gate/up pair goes to int4_swiglu")
    return _product("int4_linear", x, w, residual)


def int4_swiglu(x: torch.Tensor, w: Int4Weight) -> torch.Tensor:
    """silu(x @ gate.T) * (x @ up.T) for a gate/up pair (`Int4Weight.pack_gate_up`): [..., F] in x's
    dtype, rounded once from the fp32 sums."""
    if not w.gated:
        raise LemaError("int4_swiglu takes a gate/up pair (Int4Weight.pack_gate_up)")
    return _product("int4_swiglu", x, w, None)


class Int4Module(nn.Module):
    """Holds an Int4Weight as buffers, so that it moves, saves and loads with the model."""

    def __init__(self, w: Int4Weight):
        super().__init__()
        self.n, self.k, self.group, self.gated = w.n, w.k, w.group, w.gated
        self.register_buffer("packed", w.packed)
        self.register_buffer("scales", w.scales)
        self._weight = w

    def _apply(self, fn, recurse=True):
        # .to(dtype) casts floating buffers: the scales keep their own 16-bit type, uncast
        before = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != before.dtype:
            self.scales = before.to(self.scales.device)
        self._weight = None     # it holds the buffers that a move has just replaced
        return self

    def __setattr__(self, name, value):
        super().__setattr__(name, value)
        if name in ("packed", "scales"):
            super().__setattr__("_weight", None)

    def _load_from_state_dict(self, state_dict, prefix, *args):
        # a state dict's scales come in with their own 16-bit type: cast to this module's, weights would change
        s = state_dict.get(prefix + "scales")
        if (s is not None and s.shape == self.scales.shape and s.dtype != self.scales.dtype
                and s.dtype in (torch.bfloat16, torch.float16)):
            self.scales = self.scales.to(s.dtype)
        super()._load_from_state_dict(state_dict, prefix, *args)

    @property
    def weight4(self) -> Int4Weight:
        """The buffers as an Int4Weight (made anew when the module's buffers have been replaced)."""
        w, packed, scales = self._weight, self.packed, self.scales
        if w is None or w.packed is not packed or w.scales is not scales:
            w = self._weight = Int4Weight(packed, scales, self.n, self.k, self.group, self.gated)
        return w

    def n_weights(self) -> int:
        return self.n * self.k * (2 if self.gated else 1)

    def extra_repr(self) -> str:
        return f"{self.k} -> {self.n}, 4 bits, group {self.group}"


class Int4Linear(Int4Module):
    """nn.Linear without bias, its weight in 4 bits."""

    @classmethod
    def from_linear(cls, lin: nn.Linear, group: int = 128) -> "Int4Linear":
        if lin.bias is not None:
            raise ValueError("the model's projections have no bias")
        return cls(Int4Weight.pack(*quantize_weight(lin.weight, group), group))

    def forward(self, x, residual=None):
        return int4_linear(x, self.weight4, residual)


class Int4SwiGLU(nn.Module):
    """The MLP of code/lema/model.py:85-93 with 4-bit weights: one kernel for the gate and up products
    and the activation, one for the down product with the residual added."""

    def __init__(self, gate_up: Int4Weight, down: Int4Weight):
        super().__init__()
        self.gate_up = Int4Module(gate_up)
        self.down = Int4Linear(down)

    @classmethod
    def from_mlp(cls, mlp, group: int = 128) -> "Int4SwiGLU":
        gu = Int4Weight.pack_gate_up(*quantize_weight(mlp.gate.weight, group), *quantize_weight(mlp.up.weight, group), group)
        return cls(gu, Int4Weight.pack(*quantize_weight(mlp.down.weight, group), group))

    def forward(self, x, residual=None):
        return self.down(int4_swiglu(x, self.gate_up.weight4), residual)


# ------------------------------------------------------------------ quantised rows of the store

ROW_FORMATS = {"int8": 1, "fp8": 2, "int4": 3}     # LEMA_ROWS_* of include/lema_b200.h
_ROW_GROUP = 32                                     # values a scale covers in an int4 row
MAX_ROW_VALUES = 256


def row_bytes(fmt: str, d_v: int) -> int:
    """Bytes of a held row of d_v values (a multiple of 16)."""
    if fmt not in ROW_FORMATS:
        raise ValueError(f"row format must be one of {tuple(ROW_FORMATS)}, got {fmt!r}")
    if not 1 <= d_v <= MAX_ROW_VALUES:
        raise ValueError(f"a quantised row holds 1 to {MAX_ROW_VALUES} values, got d_v = {d_v}")
    chunks = -(-d_v // 8)
    n = chunks * 8 + 4 if fmt != "int4" else chunks * 4 + 4 * -(-chunks // 4)
    return -(-n // 16) * 16


def quantize_rows(v: torch.Tensor, fmt: str) -> torch.Tensor:
    """The held rows, uint8 [..., row_bytes], of value rows [..., d_v]: what the store's exchange
    writes (include/lema_b200.h, lema_store_exchange_quant), in plain torch."""
    d = v.shape[-1]
    nb = row_bytes(fmt, d)
    f = torch.nn.functional.pad(v.float(), (0, -d % 8))
    wide = _ROW_GROUP if fmt == "int4" else f.shape[-1]
    g = torch.nn.functional.pad(f, (0, -f.shape[-1] % wide)).unflatten(-1, (-1, wide))
    amax = g.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(amax)
    amax = torch.where(bad, torch.zeros_like(amax), amax).double()
    g = torch.where(bad, torch.zeros_like(g), g).double()
    if fmt == "fp8":
        m, e = torch.frexp(amax / 448)
        s = ((torch.where(m == 0.5, e - 1, e).clamp(min=-126) + 127) << 23).view(torch.float32)
        s = torch.where(amax > 0, s, torch.full_like(s, 2.0 ** -126))
        codes = (g / s.double()).float().to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        top = 127.0 if fmt == "int8" else 7.0
        s = (amax / top).float()
        codes = torch.where(s > 0, g / s.double(), 0.0).round().clamp(-top, top).to(torch.int8).view(torch.uint8)
    codes = codes.flatten(-2)[..., : f.shape[-1]]
    if fmt == "int4":
        codes = (codes[..., 0::2] & 15) | (codes[..., 1::2] << 4)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    s = s.squeeze(-1).contiguous().view(torch.int32)
    s = torch.where(bad.squeeze(-1), torch.full_like(s, 0x7FC00000), s)
    row = torch.cat([codes.contiguous(), s.contiguous().view(torch.uint8)], -1)
    return torch.nn.functional.pad(row, (0, nb - row.shape[-1]))


def dequantize_rows(rows: torch.Tensor, fmt: str, d_v: int, dtype: torch.dtype) -> torch.Tensor:
    """The values [..., d_v] that held rows stand for, rounded to `dtype` as the exchange does."""
    if rows.dtype != torch.uint8 or rows.shape[-1] != row_bytes(fmt, d_v):
        raise ValueError(f"held rows are uint8 [..., {row_bytes(fmt, d_v)}], got {rows.dtype} {tuple(rows.shape)}")
    chunks = -(-d_v // 8)
    if fmt == "int4":
        b = rows[..., : chunks * 4]
        c = torch.stack([b & 15, b >> 4], -1).flatten(-2).to(torch.int8)
        c = torch.where(c > 7, c - 16, c).float()
    else:
        b = rows[..., : chunks * 8].contiguous()
        c = (b.view(torch.int8) if fmt == "int8" else b.view(torch.float8_e4m3fn)).float()
    groups = -(-chunks // 4) if fmt == "int4" else 1
    at = chunks * (4 if fmt == "int4" else 8)
    s = rows[..., at: at + 4 * groups].contiguous().view(torch.float32)
    s = s.repeat_interleave(_ROW_GROUP if fmt == "int4" else chunks * 8, -1)[..., : chunks * 8]
    top = torch.finfo(dtype).max          # a code rounded up must not turn a finite value infinite
    return (c * s)[..., :d_v].clamp(-top, top).to(dtype)
