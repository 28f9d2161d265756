// Products with 4-bit weights and group scales: y[m][n] = sum_k x[m][k] * s[n][k / g] * q[n][k], q in
// -8 ... 7, and silu(gate) * up of two such products (the projections, MLP and head of
// code/lema/model.py:85-93, 160-175, 264 with weights held in 4 bits).
//
// Few rows (decode): bound by the weights' bytes, N K / 2. The weights are laid out as the fragments
// of mma.m16n8k16 with features as the M side: a lane's 16-byte load is its share of a block of 16
// features x 64 inputs, four K16 steps, and a warp's load is 512 contiguous bytes. The inputs' order
// inside a block is free as long as x follows it; here a lane's 8 values of a half block are 8
// consecutive inputs, so x is read in 16-byte loads as well.
// A nibble u = q + 8 becomes the 16-bit float 128 + u (bf16) or 1024 + u (fp16) by one AND-OR, and one
// packed subtraction gives q, exact in both types. The products of one scale group are summed by the
// tensor cores in fp32 from exact integers; only then the group's sum is scaled, in fp32: no weight is
// rounded. fp32 inputs are cut into three bf16 parts of 8 significant bits each (exactly their 24),
// multiplied in turn into the same sums.
// A warp holds kR block rows and every KS-th block of K; the KS warps of the same block rows lie in one CTA and
// their sums meet in shared memory, added in the warps' order: results do not depend on timing. KS is chosen
// so that the card is full of warps: a token through a 1536 x 1536 projection has 96 block rows and takes 16
// warps for each, the vocabulary's 3144 block rows one each. What bounds the small calls is the latency of a
// few dependent loads, so every warp keeps kDeep blocks (words, scales and inputs) in flight in registers; the large
// ones are bound by the instructions issued, about 106 a block of 1024 weights where rows are whole (kWhole: K a
// multiple of 64, 16-byte aligned rows, so that no load is checked; rows past the last read the last again, and
// what they give is dropped). A ring in shared memory (cp.async) instead of registers was no faster.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "int4.cuh"

namespace lema {
namespace w4 {

constexpr int kWarps = 8, kMaxSplit = 16;  // warps of a CTA (or as many as share a block row), and of a block row
constexpr int64_t kMaxRows = 32;  // more rows go to the tcgen05 kernel where it can read x

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<float>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma<__nv_bfloat16>(c, a, b0, b1);
}

// The first product of a sum: c = a b.
template <typename T>
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_first<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
template <>
__device__ __forceinline__ void mma_first<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
template <>
__device__ __forceinline__ void mma_first<float>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_first<__nv_bfloat16>(c, a, b0, b1);
}

// 8 consecutive inputs of one row as they lie in memory, zeros past the row's end.
template <typename T>
struct Raw {
  uint32_t v[2 * sizeof(T)];
  __device__ __forceinline__ void load_whole(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
  }
  __device__ __forceinline__ void load(const T* p, int k, int K, int vec) {  // p: input k
    if (vec && k + 8 <= K) {
      load_whole(p);
    } else if constexpr (sizeof(T) == 2) {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = k + 2 * i < K ? h[2 * i] : 0, hi = k + 2 * i + 1 < K ? h[2 * i + 1] : 0;
        v[i] = lo | (hi << 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = k + i < K ? __float_as_uint(p[i]) : 0u;
    }
  }
};

// The B fragments they make: four pairs of 16-bit values; one part for 16-bit rows, three bf16 parts for fp32 rows.
template <typename T> struct Parts { static constexpr int kN = 1; };
template <> struct Parts<float> { static constexpr int kN = 3; };
template <typename T>
__device__ __forceinline__ void cut(const Raw<T>& r, uint32_t (&b)[1][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) b[0][i] = r.v[i];
}
__device__ __forceinline__ void cut(const Raw<float>& r, uint32_t (&b)[3][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t p[3][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      // the upper 16 bits are a bf16 with 8 of the 24 significant bits; what is left is exact.
      // An infinity or a NaN goes into the first part alone (a NaN as a quiet one).
      float v = __uint_as_float(r.v[2 * i + e]);
      const bool finite = (r.v[2 * i + e] & 0x7F800000u) != 0x7F800000u;
      if (v != v) v = __uint_as_float(0x7FC00000u);
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        p[q][e] = __float_as_uint(v) & 0xFFFF0000u;
        v = finite ? v - __uint_as_float(p[q][e]) : 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) b[q][i] = (p[q][0] >> 16) | p[q][1];
  }
}

// How blocks are read: kWhole, kWholeHalf (a scale covers 32 inputs, half a block): rows whole (see above) and scales
// of the rows' own 16-bit type (bf16 for fp32 rows). kAny: everything else, checked.
enum Mode { kWhole, kWholeHalf, kAny };

// kNT token tiles of 8 rows and one block row of 16 features a warp.
template <typename T, int kNT, bool kGated, Mode kMode>
struct Rows {
  static constexpr bool kChecked = kMode == kAny;
  static constexpr int kGroups = kMode == kWhole ? 1 : 2;  // scales of a block
  static constexpr int kDeep = kNT == 4 || (sizeof(T) == 4 && kNT == 2) ? 1 : (sizeof(T) == 4 ? 2 : 4);

  struct Block {
    uint4 w;
    uint32_t s[kGroups];  // rows g (low half) and g + 8
    Raw<T> x[kNT][2];
  };
  // Where a lane reads next: words and scales of block row rb, 2 x 8 inputs of rows m + 8 n + g.
  struct Source {
    const uint4* w;
    const uint32_t* s;
    const T* x[kNT];
    int kb;
  };
  __device__ static __forceinline__ Source source(const Args& a, int rb, int64_t m, int kb, int lane) {
    const int g = lane >> 2, t = lane & 3;
    Source src;
    src.w = a.w + (static_cast<int64_t>(rb) * a.n_kb + kb) * 32 + lane;
    src.s = reinterpret_cast<const uint32_t*>(a.scales) + static_cast<int64_t>(rb) * a.n_groups * 8 + g;
#pragma unroll
    for (int n = 0; n < kNT; ++n)  // a row past the last is the last again
      src.x[n] = static_cast<const T*>(a.x) + min(m + 8 * n + g, a.M - 1) * a.ldx + kb * 64 + 8 * t;
    src.kb = kb;
    return src;
  }
  // The next block, `split` blocks of K apart.
  __device__ static __forceinline__ void load(Block& b, const Args& a, Source& src, int split, int lane) {
    b.w = __ldg(src.w);
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      int grp = (src.kb * 64 + 32 * h) >> a.log_group;
      if (kChecked) grp = min(grp, a.n_groups - 1);
      b.s[h] = __ldg(src.s + grp * 8);
    }
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (kChecked)
          b.x[n][h].load(src.x[n] + 32 * h, src.kb * 64 + 32 * h + 8 * (lane & 3), a.K, a.vec);
        else
          b.x[n][h].load_whole(src.x[n] + 32 * h);
      }
      src.x[n] += 64 * split;
    }
    src.w += 32 * split;
    src.kb += split;
  }

  __device__ static __forceinline__ float scale(uint32_t two, int hi, const Args& a) {
    const uint16_t bits = static_cast<uint16_t>(hi ? two >> 16 : two);
    return scale_of(bits, kChecked ? a.scale_bf16 : !std::is_same<T, __half>::value);
  }
  __device__ static __forceinline__ void add(const Block& b, const Args& a, float (&acc)[kNT][4]) {
    float part[kNT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t x[kNT][Parts<T>::kN][4];
#pragma unroll
      for (int n = 0; n < kNT; ++n) cut(b.x[n][h], x[n]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t f[4];
        Unpack<T>::run(h == 0 ? (j == 0 ? b.w.x : b.w.y) : (j == 0 ? b.w.z : b.w.w), f);
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int q = 0; q < Parts<T>::kN; ++q) {
            if (j == 0 && q == 0 && (kGroups == 2 || h == 0))
              mma_first<T>(part[n], f, x[n][q][2 * j], x[n][q][2 * j + 1]);
            else
              mma<T>(part[n], f, x[n][q][2 * j], x[n][q][2 * j + 1]);
          }
      }
      if (kGroups == 2 || h == 1) {
        const uint32_t two = b.s[kGroups == 2 ? h : 0];
        const float s0 = scale(two, 0, a), s1 = scale(two, 1, a);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          acc[n][0] = fmaf(s0, part[n][0], acc[n][0]);
          acc[n][1] = fmaf(s0, part[n][1], acc[n][1]);
          acc[n][2] = fmaf(s1, part[n][2], acc[n][2]);
          acc[n][3] = fmaf(s1, part[n][3], acc[n][3]);
        }
      }
    }
  }

  // The four outputs of lane l's sums s: features of rows l / 4 and l / 4 + 8 of block row rb, rows m + 2 (l % 4), + 1.
  __device__ static __forceinline__ void finish(const Args& a, int rb, int64_t m, int l, const float4& s) {
    if (rb >= a.n_rb) return;
    m += 2 * (l & 3);
    T* y = static_cast<T*>(a.y);
    if constexpr (kGated) {
      const int f = rb * 8 + (l >> 2);
      if (f >= a.N) return;
      if (m < a.M) y[m * a.ldy + f] = from_f<T>(gate_up(s.x, s.z));
      if (m + 1 < a.M) y[(m + 1) * a.ldy + f] = from_f<T>(gate_up(s.y, s.w));
    } else {
      const T* res = static_cast<const T*>(a.r);
      const float v[2][2] = {{s.x, s.y}, {s.z, s.w}};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int f = rb * 16 + (l >> 2) + 8 * i;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (f < a.N && m + e < a.M)
            y[(m + e) * a.ldy + f] = from_f<T>(v[i][e] + (res != nullptr ? to_f(res[(m + e) * a.ldr + f]) : 0.f));
      }
    }
  }
};

template <typename T, int kNT, bool kGated, Mode kMode>
__global__ void __launch_bounds__(32 * kMaxSplit) rows_kernel(const Args a, int split) {
  using R = Rows<T, kNT, kGated, kMode>;
  __shared__ float4 sums[kMaxSplit][kNT][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rb = blockIdx.x * ((blockDim.x >> 5) / split) + warp / split, first = warp % split;
  griddep_launch();
  if (rb < a.n_rb && first < a.n_kb)  // while the previous kernel ends (a hint: it reads nothing)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(a.w + (static_cast<int64_t>(rb) * a.n_kb + first) * 32 + lane));
  griddep_wait();  // launched as a dependent: x and the residual first
  const int64_t m_tiles = (a.M + 8 * kNT - 1) / (8 * kNT);
#pragma unroll 1
  for (int64_t mt = blockIdx.y; mt < m_tiles; mt += gridDim.y) {
    const int64_t m0 = mt * (8 * kNT);
    float acc[kNT][4];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[n][c] = 0.f;
    if (rb < a.n_rb) {
      typename R::Block blk[R::kDeep];
      typename R::Source src = R::source(a, rb, m0, first, lane);
#pragma unroll
      for (int u = 0; u < R::kDeep; ++u)
        if (src.kb < a.n_kb) R::load(blk[u], a, src, split, lane);
#pragma unroll 1
      for (int kb = first; kb < a.n_kb;) {
#pragma unroll
        for (int u = 0; u < R::kDeep; ++u, kb += split) {
          if (kb >= a.n_kb) break;
          R::add(blk[u], a, acc);
          if (src.kb < a.n_kb) R::load(blk[u], a, src, split, lane);
        }
      }
    }
    if (split == 1) {
#pragma unroll
      for (int n = 0; n < kNT; ++n) R::finish(a, rb, m0 + 8 * n, lane, make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]));
      continue;
    }
    __syncthreads();  // the previous tile's sums have been read
#pragma unroll
    for (int n = 0; n < kNT; ++n) sums[warp][n][lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
    __syncthreads();
    // the split warps of a block row share its token tiles
    for (int n = first; n < kNT; n += split) {
      const int w0 = warp - first;
      float4 s = sums[w0][n][lane];
      for (int q = 1; q < split; ++q) {
        const float4 o = sums[w0 + q][n][lane];
        s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
      }
      R::finish(a, rb, m0 + 8 * n, lane, s);
    }
  }
}

template <typename T, int kNT>
int launch_rows(const Args& a, bool gated, int sms, cudaStream_t stream) {
  // warps a block row: up to about 24 on every SM, and a block of K for each
  int split = 1;
  while (split < kMaxSplit && static_cast<int64_t>(a.n_rb) * split * 2 <= 24 * static_cast<int64_t>(sms) && 2 * split <= a.n_kb) split *= 2;
  const int warps = std::max(kWarps, split), per_cta = warps / split;
  const int64_t tiles = (a.M + 8 * kNT - 1) / (8 * kNT);
  const dim3 grid(static_cast<unsigned>((a.n_rb + per_cta - 1) / per_cta), static_cast<unsigned>(std::min<int64_t>(tiles, 65535)));
  const dim3 block(static_cast<unsigned>(32 * warps));
  const bool whole = a.vec && a.K % 64 == 0 && a.scale_bf16 == !std::is_same<T, __half>::value;
  const auto go = [&](auto kernel) {
    LEMA_CUDA_TRY(launch_dependent(kernel, grid, block, 0, stream, a, split));
    return static_cast<int>(LEMA_OK);
  };
  if (!whole) return gated ? go(rows_kernel<T, kNT, true, kAny>) : go(rows_kernel<T, kNT, false, kAny>);
  if (a.log_group == 5) return gated ? go(rows_kernel<T, kNT, true, kWholeHalf>) : go(rows_kernel<T, kNT, false, kWholeHalf>);
  return gated ? go(rows_kernel<T, kNT, true, kWhole>) : go(rows_kernel<T, kNT, false, kWhole>);
}

template <typename T>
int run_rows(const Args& a, bool gated, int sms, cudaStream_t stream) {
  if (a.M <= 8) return launch_rows<T, 1>(a, gated, sms, stream);
  if constexpr (sizeof(T) == 2)
    if (a.M > 16) return launch_rows<T, 4>(a, gated, sms, stream);
  return launch_rows<T, 2>(a, gated, sms, stream);
}

}  // namespace w4
}  // namespace lema

extern "C" int lema_int4_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* packed,
                                const void* scales, int scale_dtype, int group, int64_t N, int gated,
                                const void* residual, int64_t ldr, void* y, int64_t ldy, uint32_t* status,
                                void* stream) {
  using namespace lema;
  clear_error();
  if (dtype != LEMA_F32 && dtype != LEMA_BF16 && dtype != LEMA_F16) return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: dtype tag %d", dtype);
  if (scale_dtype != LEMA_BF16 && scale_dtype != LEMA_F16) return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: scales are bf16 or fp16 (dtype tag %d)", scale_dtype);
  if (group != 32 && group != 64 && group != 128) return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: a scale covers 32, 64 or 128 inputs, got %d", group);
  if (M < 0 || K <= 0 || N <= 0) return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: bad shape M=%lld K=%lld N=%lld", (long long)M, (long long)K, (long long)N);
  if (M >= (int64_t(1) << 31) || K >= (int64_t(1) << 24) || N >= (int64_t(1) << 24))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: shape too large (M=%lld K=%lld N=%lld)", (long long)M, (long long)K, (long long)N);
  if (gated && residual != nullptr) return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: no residual with a gated product");
  if (M > 1 && (ldx < K || ldy < N || (residual != nullptr && ldr < N)))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: rows overlap (ldx=%lld ldr=%lld ldy=%lld)", (long long)ldx, (long long)ldr, (long long)ldy);
  if (M == 0) return LEMA_OK;
  if (x == nullptr || packed == nullptr || scales == nullptr || y == nullptr) return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: null pointer");
  const int64_t es = dtype == LEMA_F32 ? 4 : 2;
  if (!aligned(packed, 16) || !aligned(scales, 4) || !aligned(x, es) || !aligned(y, es) || !aligned(residual, es))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: packed weights must be 16-byte aligned, scales 4, the others to their elements");
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return LEMA_ERR_CUDA;
  if (dev->cc_major != 10) return fail(LEMA_ERR_UNSUPPORTED, "built for sm_100a; device is sm_%d%d", dev->cc_major, dev->cc_minor);
  w4::Args a{};
  a.w = static_cast<const uint4*>(packed);
  a.scales = static_cast<const uint16_t*>(scales);
  a.x = x;
  a.r = residual;
  a.y = y;
  a.ldx = ldx;
  a.ldr = ldr;
  a.ldy = ldy;
  a.M = M;
  a.K = static_cast<int>(K);
  a.N = static_cast<int>(N);
  a.n_rb = static_cast<int>(gated ? (N + 7) / 8 : (N + 15) / 16);
  a.n_kb = static_cast<int>((K + 63) / 64);
  a.n_groups = static_cast<int>((K + group - 1) / group);
  a.log_group = group == 32 ? 5 : (group == 64 ? 6 : 7);
  a.scale_bf16 = scale_dtype == LEMA_BF16;
  a.vec = aligned(x, 16) && (M == 1 || (ldx * es) % 16 == 0);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Up to 32 rows multiply the codes exactly, whatever the weight's width and the card (17 to 32 rows through 50304 x 1536
  // would take 32 instead of 43 us in the many-rows kernel, with rounded weights; through 1536 x 4096 8.3 instead of 5.7)
  if (M > w4::kMaxRows && w4::tile_ok(a, dtype)) return w4::run_tile(a, dtype, gated != 0, status, s);
  if (dtype == LEMA_F32) return w4::run_rows<float>(a, gated != 0, dev->sms, s);
  if (dtype == LEMA_BF16) return w4::run_rows<__nv_bfloat16>(a, gated != 0, dev->sms, s);
  return w4::run_rows<__half>(a, gated != 0, dev->sms, s);
}
