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
// A CTA of 8 warps holds a few block rows; the warps take the K blocks in turn and their sums meet in
// shared memory, in the warps' order: results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "int4.cuh"

namespace lema {
namespace w4 {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
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

// 8 consecutive inputs as packed pairs: one part for 16-bit rows, three bf16 parts for fp32 rows.
template <typename T> struct Parts { static constexpr int kN = 1; };
template <> struct Parts<float> { static constexpr int kN = 3; };

template <typename T>
__device__ __forceinline__ void load_x(const T* row, int k, int K, int vec, uint32_t (&b)[1][4]) {
  if (vec && k + 8 <= K) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + k));
    b[0][0] = v.x; b[0][1] = v.y; b[0][2] = v.z; b[0][3] = v.w;
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(row) + k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = k + 2 * i < K ? h[2 * i] : 0, hi = k + 2 * i + 1 < K ? h[2 * i + 1] : 0;
      b[0][i] = lo | (hi << 16);
    }
  }
}
__device__ __forceinline__ void load_x(const float* row, int k, int K, int vec, uint32_t (&b)[3][4]) {
  float f[8];
  if (vec && k + 8 <= K) {
    const float4 u = __ldg(reinterpret_cast<const float4*>(row + k)), v = __ldg(reinterpret_cast<const float4*>(row + k) + 1);
    f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w; f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = k + i < K ? row[k + i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t p[3][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      // the upper 16 bits are a bf16 with 8 of the 24 significant bits; what is left is exact.
      // An infinity or a NaN goes into the first part alone (a NaN as a quiet one).
      float v = f[2 * i + e];
      const bool finite = (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u;
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

// kNT token tiles of 8 rows and kR block rows of 16 features a CTA.
template <typename T, int kNT, int kR, bool kGated>
__global__ void __launch_bounds__(kThreads) rows_kernel(const Args a) {
  __shared__ float4 sums[kWarps][kR][kNT][32];
  griddep_launch();
  griddep_wait();  // launched as a dependent: x and the residual first
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rb0 = blockIdx.x * kR;
  const T* x = static_cast<const T*>(a.x);
  const int64_t m_tiles = (a.M + 8 * kNT - 1) / (8 * kNT);
  for (int64_t mt = blockIdx.y; mt < m_tiles; mt += gridDim.y) {
    const int64_t m0 = mt * (8 * kNT);
    float acc[kR][kNT][4];
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][n][c] = 0.f;
    for (int kb = warp; kb < a.n_kb; kb += kWarps) {
      uint4 w[kR];
#pragma unroll
      for (int r = 0; r < kR; ++r)
        w[r] = rb0 + r < a.n_rb ? __ldg(a.w + (static_cast<int64_t>(rb0 + r) * a.n_kb + kb) * 32 + lane)
                                : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kb * 64 + h * 32 + t * 8;
        uint32_t b[kNT][Parts<T>::kN][4];
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          const int64_t m = m0 + n * 8 + g;
          if (m < a.M) {
            load_x(x + m * a.ldx, k, a.K, a.vec, b[n]);
          } else {
#pragma unroll
            for (int q = 0; q < Parts<T>::kN; ++q)
#pragma unroll
              for (int i = 0; i < 4; ++i) b[n][q][i] = 0;
          }
        }
        const int grp = min((kb * 64 + h * 32) >> a.log_group, a.n_groups - 1);
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const uint32_t* words = reinterpret_cast<const uint32_t*>(&w[r]);
          float part[kNT][4];
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) part[n][c] = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t f[4];
            Unpack<T>::run(words[2 * h + j], f);
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
              for (int q = 0; q < Parts<T>::kN; ++q) mma<T>(part[n], f, b[n][q][2 * j], b[n][q][2 * j + 1]);
          }
          const int rb = min(rb0 + r, a.n_rb - 1);
          const uint32_t two = __ldg(reinterpret_cast<const uint32_t*>(a.scales) + (static_cast<int64_t>(rb) * a.n_groups + grp) * 8 + g);
          const float s0 = scale_of(static_cast<uint16_t>(two), a.scale_bf16), s1 = scale_of(static_cast<uint16_t>(two >> 16), a.scale_bf16);
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            acc[r][n][0] = fmaf(s0, part[n][0], acc[r][n][0]);
            acc[r][n][1] = fmaf(s0, part[n][1], acc[r][n][1]);
            acc[r][n][2] = fmaf(s1, part[n][2], acc[r][n][2]);
            acc[r][n][3] = fmaf(s1, part[n][3], acc[r][n][3]);
          }
        }
      }
    }
    __syncthreads();  // the previous tile's sums have been read
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int n = 0; n < kNT; ++n)
        sums[warp][r][n][lane] = make_float4(acc[r][n][0], acc[r][n][1], acc[r][n][2], acc[r][n][3]);
    __syncthreads();
    // each thread finishes the four outputs (features i, i + 8; rows 2 t, 2 t + 1) of a lane
    for (int i = threadIdx.x; i < kR * kNT * 32; i += kThreads) {
      const int l = i & 31, n = (i >> 5) % kNT, r = (i >> 5) / kNT;
      float4 s = sums[0][r][n][l];
#pragma unroll
      for (int q = 1; q < kWarps; ++q) {
        const float4 o = sums[q][r][n][l];
        s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
      }
      const int rb = rb0 + r;
      if (rb >= a.n_rb) continue;
      const int64_t m = m0 + n * 8 + 2 * (l & 3);
      T* y = static_cast<T*>(a.y);
      if constexpr (kGated) {
        const int f = rb * 8 + (l >> 2);
        if (f < a.N) {
          if (m < a.M) y[m * a.ldy + f] = from_f<T>(gate_up(s.x, s.z));
          if (m + 1 < a.M) y[(m + 1) * a.ldy + f] = from_f<T>(gate_up(s.y, s.w));
        }
      } else {
        const T* res = static_cast<const T*>(a.r);
        const float v[2][2] = {{s.x, s.y}, {s.z, s.w}};
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const int f = rb * 16 + (l >> 2) + 8 * i2;
          if (f >= a.N) continue;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (m + e < a.M)
              y[(m + e) * a.ldy + f] = from_f<T>(v[i2][e] + (res != nullptr ? to_f(res[(m + e) * a.ldr + f]) : 0.f));
        }
      }
    }
  }
}

template <typename T, int kNT, int kR>
int launch_rows(const Args& a, bool gated, cudaStream_t stream) {
  const int64_t tiles = (a.M + 8 * kNT - 1) / (8 * kNT);
  const dim3 grid(static_cast<unsigned>((a.n_rb + kR - 1) / kR), static_cast<unsigned>(std::min<int64_t>(tiles, 65535)));
  if (gated)
    LEMA_CUDA_TRY(launch_dependent(rows_kernel<T, kNT, kR, true>, grid, dim3(kThreads), 0, stream, a));
  else
    LEMA_CUDA_TRY(launch_dependent(rows_kernel<T, kNT, kR, false>, grid, dim3(kThreads), 0, stream, a));
  return LEMA_OK;
}

template <typename T>
int run_rows(const Args& a, bool gated, cudaStream_t stream) {
  if (a.M <= 8) return launch_rows<T, 1, 1>(a, gated, stream);
  if (a.M <= 16) return launch_rows<T, 2, 1>(a, gated, stream);
  return launch_rows<T, 4, 1>(a, gated, stream);
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
  if (M > w4::kMaxRows && w4::tile_ok(a, dtype)) return w4::run_tile(a, dtype, gated != 0, status, s);
  if (dtype == LEMA_F32) return w4::run_rows<float>(a, gated != 0, s);
  if (dtype == LEMA_BF16) return w4::run_rows<__nv_bfloat16>(a, gated != 0, s);
  return w4::run_rows<__half>(a, gated != 0, s);
}
