// What the two kernels of products with 4-bit weights share (int4_linear.cu: few rows; int4_tile.cu:
// many): the arguments, the unpacking of a fragment word, and the activation.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace lema {
namespace w4 {

struct Args {
  const uint4* w;           // [n_rb][n_kb][32]
  const uint16_t* scales;   // [n_rb][n_groups][8][2]
  const void* x;
  const void* r;
  void* y;
  int64_t ldx, ldr, ldy;    // elements
  int64_t M;
  int K, N;                 // inputs, output features
  int n_rb, n_kb, n_groups;
  int log_group;            // 5, 6 or 7
  int scale_bf16;
  int vec;                  // x rows readable in whole aligned chunks of 8 values
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float scale_of(uint16_t bits, int bf16) {
  return bf16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16) : __half2float(__ushort_as_half(bits));
}

// Four pairs of weights of one word as 16-bit floats of type T (the A fragment of one K16 step).
template <typename T> struct Unpack;
template <> struct Unpack<__nv_bfloat16> {
  __device__ static __forceinline__ void run(uint32_t w, uint32_t (&a)[4]) {
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.f, 136.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = ((w >> (4 * j)) & 0x000F000Fu) | 0x43004300u;  // 128 + u
      const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), off);
      a[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
};
template <> struct Unpack<__half> {
  __device__ static __forceinline__ void run(uint32_t w, uint32_t (&a)[4]) {
    const __half2 off = __floats2half2_rn(1032.f, 1032.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = ((w >> (4 * j)) & 0x000F000Fu) | 0x64006400u;  // 1024 + u
      const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), off);
      a[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
};
template <> struct Unpack<float> : Unpack<__nv_bfloat16> {};

// silu(g) * u in fp32.
__device__ __forceinline__ float gate_up(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// Many rows (int4_tile.cu): x in 16 bits, rows readable by TMA (tile_ok).
bool tile_ok(const Args& a, int dtype);
int run_tile(const Args& a, int dtype, bool gated, uint32_t* status, cudaStream_t stream);

}  // namespace w4
}  // namespace lema
