// Products of many rows with 4-bit weights (int4_linear.cu's definition; prompts and large decode batches):
// bound by the tensor cores, 2 M N K operations. One persistent CTA per SM walks tiles of 128 weight rows
// (features) x BN tokens, features on the M side of tcgen05.mma so that the weights' fragment layout is
// also this kernel's and a small batch needs no padding to 128 rows. Warp roles:
//   warp 0      TMA producer: BN x 64 tiles of x (128-byte swizzle) into a ring of stages;
//   warp 1      MMA issuer: per stage 4 x tcgen05.mma M128 N(BN) K16 into one of two fp32 TMEM
//               accumulators; tcgen05.commit frees the stage;
//   warps 2-5   epilogue: a lane holds one feature, a TMEM column one token; adds the residual or applies
//               the activation (a gate and its up feature are 8 lanes apart) and rounds once;
//   warps 6-21  dequantisation, four sets of 4 warps that take the stages in turn: each warp turns two blocks
//               of 16 features x 64 inputs a stage into 16-bit floats and writes them where the MMA's A
//               operand expects them (the same swizzle).
// Here a weight is rounded: s * q (8 + 4 significant bits, or 11 + 4) is rounded once to the rows' 16-bit
// type, since the tensor core multiplies one type and a tile cannot scale its sums by groups without
// reading the accumulator back every 32 to 128 inputs. That is half a step a weight, the rounding that a
// 16-bit checkpoint of the same weights has (fp16's subnormals included).
//
// Every wait is bounded (tcgen05.cuh); a wait that runs out sets the abort flag and
// LEMA_STATUS_PROBE_LIMIT, and the CTA drains its copies and MMAs and frees its TMEM.
#include <algorithm>

#include "int4.cuh"
#include "tcgen05.cuh"

namespace lema {
namespace w4 {

using namespace tc;

constexpr int kTileRows = 128;                    // weight rows a tile
constexpr int kABytes = kTileRows * kBK * 2;      // 16 KiB
constexpr int kTileBlocks = kTileRows / 16;       // block rows a tile
constexpr int kSets = 4;                          // sets of dequantising warps; set i fills stages i, i + kSets, ...
constexpr int kSetWarps = 4;
constexpr int kMine = kTileBlocks / kSetWarps;    // block rows a warp
constexpr int kTileThreads = 32 * (6 + kSets * kSetWarps);

template <int BN>
struct Tile {
  static constexpr int kBBytes = BN * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = BN == 64 ? 8 : 4;
  static constexpr uint32_t kTmemCols = 2 * BN;
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + 1024 /* alignment */ + 512 /* barriers */;
};

struct TileArgs {
  Args a;
  uint32_t* status;
  uint64_t wait_ns;
  int64_t n_tiles;
  int f_tiles;       // tiles along the weight rows
  int pairs;         // rows of y and of the residual hold whole aligned pairs of features
};

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using P = __nv_bfloat162;
  static constexpr int kBf16 = 1;
  __device__ static __forceinline__ uint32_t from_f(float a, float b) {
    const P p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  __device__ static __forceinline__ float2 to_f2(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const P*>(&v)); }
};
template <> struct Pair<__half> {
  using P = __half2;
  static constexpr int kBf16 = 0;
  __device__ static __forceinline__ uint32_t from_f(float a, float b) {
    const P p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  __device__ static __forceinline__ float2 to_f2(uint32_t v) { return __half22float2(*reinterpret_cast<const P*>(&v)); }
};

// The scale of one row of a fragment: kSame (the scales have the rows' type) as a pair for a 16-bit multiply,
// whose exact operands' product rounds once, else as fp32.
template <typename T, bool kSame> struct RowScale;
template <typename T> struct RowScale<T, true> {
  uint32_t s;
  __device__ __forceinline__ RowScale(uint32_t two, int hi, int) : s(hi ? (two >> 16) | (two & 0xFFFF0000u) : (two & 0xFFFFu) | (two << 16)) {}
  __device__ __forceinline__ uint32_t times(uint32_t q) const {
    const typename Pair<T>::P r = __hmul2(*reinterpret_cast<const typename Pair<T>::P*>(&q), *reinterpret_cast<const typename Pair<T>::P*>(&s));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <typename T> struct RowScale<T, false> {
  float s;
  __device__ __forceinline__ RowScale(uint32_t two, int hi, int scale_bf16)
      : s(scale_of(static_cast<uint16_t>(hi ? two >> 16 : two), scale_bf16)) {}
  __device__ __forceinline__ uint32_t times(uint32_t q) const {
    const float2 v = Pair<T>::to_f2(q);
    return Pair<T>::from_f(v.x * s, v.y * s);
  }
};

// wait_phase by a whole warp: every lane gets the same answer, so that all of them go on or none does.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status, uint64_t wait_ns) {
  return __all_sync(0xFFFFFFFFu, wait_phase(bar, parity, abort_flag, status, wait_ns));
}

__device__ __forceinline__ void mma_16bit(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  mma_bf16(d_tmem, a_desc, b_desc, idesc, acc);  // kind::f16; the types are the descriptor's
}

template <typename T, int BN, bool kGated, bool kSame>
__global__ void __launch_bounds__(kTileThreads, 1) tile_kernel(const __grid_constant__ CUtensorMap map_x, const TileArgs p) {
  using TL = Tile<BN>;
  constexpr int kStages = TL::kStages, kStageBytes = TL::kStageBytes;
  // instruction descriptor (tcgen05.mma kind::f16): fp32 accumulator, A and B of type T (0 fp16, 1 bf16), both
  // K-major, N >> 3 at bits 17-22, M >> 4 at bits 24-28
  constexpr uint32_t kType = Pair<T>::kBf16;
  constexpr uint32_t kInstrDesc = (1u << 4) | (kType << 7) | (kType << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(kTileRows >> 4) << 24);
  static_assert(kStages % kSets == 0 && kTileBlocks % kSetWarps == 0, "whole shares");
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  unsigned char* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t sbase = smem_addr(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  // barriers: x full, weights full, empty [kStages each], acc_full[2], acc_empty[2], drain
  const uint32_t bar0 = smem_addr(bars);
  auto xfull_bar = [&](int s) { return bar0 + 8u * s; };
  auto wfull_bar = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto empty_bar = [&](int s) { return bar0 + 8u * (2 * kStages + s); };
  auto accf_bar = [&](int a) { return bar0 + 8u * (3 * kStages + a); };
  auto acce_bar = [&](int a) { return bar0 + 8u * (3 * kStages + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (3 * kStages + 4);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 3 * kStages + 5);
  volatile uint32_t* s_abort = s_tmem + 1;

  const Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(xfull_bar(s), 1);
      mbar_init(wfull_bar(s), kSetWarps);
      mbar_init(empty_bar(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(accf_bar(i), 1);
      mbar_init(acce_bar(i), 4);  // one arrival per epilogue warp
    }
    mbar_init(drain_bar, 1);
    *s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(s_tmem)), "r"(TL::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *s_tmem;
  griddep_wait();  // launched as a dependent: x and the residual are read only from here on

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (x)
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, issued = 0, last_ph = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; ok && tile < p.n_tiles; tile += gridDim.x) {
        const int m0 = static_cast<int>(tile / p.f_tiles) * BN;
        for (int kb = 0; kb < a.n_kb; ++kb) {
          if (!wait_phase(empty_bar(s), ph ^ 1u, s_abort, p.status, p.wait_ns)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(xfull_bar(s), TL::kBBytes);
          tma_load_2d(sbase + s * kStageBytes + kABytes, &map_x, xfull_bar(s), kb * kBK, m0);
          issued |= 1u << s;
          last_ph = (last_ph & ~(1u << s)) | (ph << s);
          if (++s == kStages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // copies still in flight must land before the CTA's shared memory goes away
      for (int i = 0; i < kStages; ++i)
        if (issued & (1u << i)) drain_phase(xfull_bar(i), (last_ph >> i) & 1u, p.status);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int s = 0, acc = 0;
      uint32_t ph = 0, aph = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; ok && tile < p.n_tiles; tile += gridDim.x) {
        if (!wait_phase(acce_bar(acc), aph ^ 1u, s_abort, p.status, p.wait_ns)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = 0; kb < a.n_kb; ++kb) {
          if (!wait_phase(xfull_bar(s), ph, s_abort, p.status, p.wait_ns) ||
              !wait_phase(wfull_bar(s), ph, s_abort, p.status, p.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = sbase + s * kStageBytes;
          const uint64_t a_desc = sw128_desc(a_addr), b_desc = sw128_desc(a_addr + kABytes);
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk)
            mma_16bit(d_tmem, a_desc + 2u * kk, b_desc + 2u * kk, kInstrDesc, (kb | kk) != 0 ? 1u : 0u);
          mma_commit(empty_bar(s));
          if (++s == kStages) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (!ok) break;
        mma_commit(accf_bar(acc));
        if (++acc == 2) {
          acc = 0;
          aph ^= 1u;
        }
      }
      mma_commit(drain_bar);  // nothing this thread issued may still run at exit
      drain_phase(drain_bar, 0, p.status);
    }
    __syncwarp();
  } else if (warp < 6) {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;  // a warp reads TMEM lanes 32 * (warp % 4) ... + 31
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const T* res = static_cast<const T*>(a.r);
    T* y = static_cast<T*>(a.y);
    int acc = 0;
    uint32_t aph = 0;
    for (int64_t tile = blockIdx.x; tile < p.n_tiles; tile += gridDim.x) {
      if (!warp_wait(accf_bar(acc), aph, s_abort, p.status, p.wait_ns)) break;
      tc_fence_after();
      const int64_t m0 = (tile / p.f_tiles) * BN;
      const int row = static_cast<int>(tile % p.f_tiles) * kTileRows + quarter * 32 + lane;  // weight row
      for (int j = 0; j < BN / 32; ++j) {
        const int64_t m = m0 + j * 32;
        if (m >= a.M) break;  // warp-uniform
        uint32_t r[32];
        tmem_load32(tmem_base + lane_base + static_cast<uint32_t>(acc * BN + j * 32), r);
        if constexpr (kGated) {
          // block rows hold 8 gate rows, then the 8 up rows of the same features: lanes l and l ^ 8 swap one
          // value of each pair of tokens, and each finishes one token
          const bool gate = (row & 8) == 0;
          const int f = (row >> 4) * 8 + (row & 7);
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float even = __uint_as_float(r[c]), odd = __uint_as_float(r[c + 1]);
            const float other = __shfl_xor_sync(0xFFFFFFFFu, gate ? odd : even, 8);
            const float v = gate ? gate_up(even, other) : gate_up(other, odd);
            const int64_t t = m + c + (gate ? 0 : 1);
            if (f < a.N && t < a.M) y[t * a.ldy + f] = from_f<T>(v);
          }
        } else {
          // lanes l and l ^ 1 swap one value of each pair of tokens: each finishes two features of one token,
          // so that residual and output move in 32-bit words where rows allow it
          const int odd = lane & 1, f = row & ~1;
          float v[16][2];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float lo = __uint_as_float(r[2 * c]), hi = __uint_as_float(r[2 * c + 1]);
            const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? lo : hi, 1);
            v[c][0] = odd ? other : lo;
            v[c][1] = odd ? hi : other;
          }
          if (p.pairs) {
            if (res != nullptr) {
              uint32_t rs[16];  // all of them in flight before the first store
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const int64_t t = m + 2 * c + odd;
                rs[c] = f < a.N && t < a.M ? *reinterpret_cast<const uint32_t*>(res + t * a.ldr + f) : 0u;
              }
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const float2 add = Pair<T>::to_f2(rs[c]);
                v[c][0] += add.x;
                v[c][1] += add.y;
              }
            }
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const int64_t t = m + 2 * c + odd;
              if (f < a.N && t < a.M) *reinterpret_cast<uint32_t*>(y + t * a.ldy + f) = Pair<T>::from_f(v[c][0], v[c][1]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const int64_t t = m + 2 * c + odd;
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (f + e < a.N && t < a.M)
                  y[t * a.ldy + f + e] = from_f<T>(v[c][e] + (res != nullptr ? to_f(res[t * a.ldr + f + e]) : 0.f));
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acce_bar(acc));
      if (++acc == 2) {
        acc = 0;
        aph ^= 1u;
      }
    }
  } else {
    // ------------------------------------------------------------ dequantisation
    const int set = (warp - 6) / kSetWarps, blk0 = (warp - 6) % kSetWarps * kMine, g = lane >> 2, t = lane & 3;
    // Odd rows take their upper half first: the eight lanes of one write phase then cover all banks.
    const bool odd = g & 1;
    // row r's 16-byte chunk c lies at r * 128 + ((c ^ (r & 7)) << 4) of the stage
    const uint32_t row0 = (blk0 * 16 + g) * 128;
    const uint32_t c0 = row0 + (((odd ? 4 : 0) + t) ^ g) * 16, c1 = row0 + (((odd ? 0 : 4) + t) ^ g) * 16;
    const int sc_second = a.log_group == 5 ? 8 : 0;  // to the upper half's scales
    int s = set, skip = set;  // skip: stages until this set's next one
    uint32_t ph = 1;
    for (int64_t tile = blockIdx.x; tile < p.n_tiles; tile += gridDim.x) {
      const int rb0 = static_cast<int>(tile % p.f_tiles) * kTileBlocks + blk0;
      const uint4* wp[kMine];
      const uint32_t* sp[kMine];
#pragma unroll
      for (int b = 0; b < kMine; ++b) {
        const int rb = min(rb0 + b, a.n_rb - 1);  // block rows past the last are computed and dropped
        wp[b] = a.w + static_cast<int64_t>(rb) * a.n_kb * 32 + lane;
        sp[b] = reinterpret_cast<const uint32_t*>(a.scales) + static_cast<int64_t>(rb) * a.n_groups * 8 + g;
      }
      uint4 next[kMine];
      uint32_t next_sc[kMine][2];
      auto fetch = [&](int kb) {
        const int grp = (kb * kBK) >> a.log_group;
        const int up = grp + 1 < a.n_groups ? sc_second : 0;
#pragma unroll
        for (int b = 0; b < kMine; ++b) {
          next[b] = __ldg(wp[b] + kb * 32);
          next_sc[b][0] = __ldg(sp[b] + grp * 8);
          next_sc[b][1] = __ldg(sp[b] + grp * 8 + up);
        }
      };
      int kb = skip;
      if (kb < a.n_kb) fetch(kb);
      for (; kb < a.n_kb; kb += kSets) {
        uint4 w[kMine];
        uint32_t sc[kMine][2];
#pragma unroll
        for (int b = 0; b < kMine; ++b) {
          w[b] = next[b];
          sc[b][0] = next_sc[b][0];
          sc[b][1] = next_sc[b][1];
        }
        if (kb + kSets < a.n_kb) fetch(kb + kSets);
        unsigned char* dst = smem + s * kStageBytes;
#pragma unroll
        for (int b = 0; b < kMine; ++b) {
          uint4 v[2][2];  // [row g / g + 8][first or second half written]: 8 consecutive inputs each
          const uint32_t words[4] = {odd ? w[b].z : w[b].x, odd ? w[b].w : w[b].y, odd ? w[b].x : w[b].z, odd ? w[b].y : w[b].w};
          const uint32_t two[2] = {odd ? sc[b][1] : sc[b][0], odd ? sc[b][0] : sc[b][1]};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t f0[4], f1[4];
            Unpack<T>::run(words[2 * h], f0);
            Unpack<T>::run(words[2 * h + 1], f1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const RowScale<T, kSame> rs(two[h], i, a.scale_bf16);
              v[i][h].x = rs.times(f0[i]);
              v[i][h].y = rs.times(f0[i + 2]);
              v[i][h].z = rs.times(f1[i]);
              v[i][h].w = rs.times(f1[i + 2]);
            }
          }
          if (b == 0 && !warp_wait(empty_bar(s), ph, s_abort, p.status, p.wait_ns)) goto done;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            *reinterpret_cast<uint4*>(dst + c0 + b * 2048 + i * 1024) = v[i][0];
            *reinterpret_cast<uint4*>(dst + c1 + b * 2048 + i * 1024) = v[i][1];
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads through the async proxy
        __syncwarp();
        if (lane == 0) mbar_arrive(wfull_bar(s));
        s += kSets;
        if (s >= kStages) {
          s -= kStages;
          ph ^= 1u;
        }
      }
      skip = kb - a.n_kb;
    }
  done:;
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TL::kTmemCols) : "memory");
  }
}

bool tile_ok(const Args& a, int dtype) {
  return dtype != LEMA_F32 && a.K >= kBK && (a.ldx * 2) % 16 == 0 && aligned(a.x, 16);
}

template <typename T, int BN, bool kGated, bool kSame>
int launch_tile(const CUtensorMap& map, const TileArgs& p, int64_t grid, cudaStream_t stream) {
  const auto kernel = tile_kernel<T, BN, kGated, kSame>;
  LEMA_TRY(kernel_facts(reinterpret_cast<const void*>(kernel), Tile<BN>::kSmemBytes, 0, 0, nullptr));
  LEMA_CUDA_TRY(launch_dependent(kernel, dim3(static_cast<unsigned>(grid)), dim3(kTileThreads), Tile<BN>::kSmemBytes, stream, map, p));
  return LEMA_OK;
}

template <typename T, int BN>
int launch_width(const CUtensorMap& map, const TileArgs& p, int64_t grid, bool gated, cudaStream_t stream) {
  const bool same = p.a.scale_bf16 == Pair<T>::kBf16;
  if (gated) return same ? launch_tile<T, BN, true, true>(map, p, grid, stream) : launch_tile<T, BN, true, false>(map, p, grid, stream);
  return same ? launch_tile<T, BN, false, true>(map, p, grid, stream) : launch_tile<T, BN, false, false>(map, p, grid, stream);
}

template <typename T>
int launch_type(int bn, const CUtensorMap& map, const TileArgs& p, int64_t grid, bool gated, cudaStream_t stream) {
  if (bn == 64) return launch_width<T, 64>(map, p, grid, gated, stream);
  if (bn == 128) return launch_width<T, 128>(map, p, grid, gated, stream);
  return launch_width<T, 256>(map, p, grid, gated, stream);
}

int run_tile(const Args& a, int dtype, bool gated, uint32_t* status, cudaStream_t stream) {
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return LEMA_ERR_CUDA;
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return fail(LEMA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  TileArgs p{};
  p.a = a;
  p.status = status;
  p.wait_ns = wait_limit_ns();
  p.f_tiles = (a.n_rb + kTileBlocks - 1) / kTileBlocks;
  p.pairs = a.N % 2 == 0 && a.ldy % 2 == 0 && aligned(a.y, 4) && (a.r == nullptr || (a.ldr % 2 == 0 && aligned(a.r, 4)));
  // the widest tile that still gives every SM a tile
  int bn = 256;
  while (bn > 64 && (a.M <= bn / 2 || ((a.M + bn - 1) / bn) * p.f_tiles < dev->sms)) bn /= 2;
  p.n_tiles = ((a.M + bn - 1) / bn) * p.f_tiles;
  CUtensorMap map;
  if (!encode_kmajor(enc, &map, a.x, a.M, a.K, a.ldx, bn,
                     dtype == LEMA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: tensor map encoding failed (M=%lld K=%d ldx=%lld)", (long long)a.M, a.K, (long long)a.ldx);
  const int64_t grid = std::min<int64_t>(p.n_tiles, dev->sms);
  if (dtype == LEMA_BF16) return launch_type<__nv_bfloat16>(bn, map, p, grid, gated, stream);
  return launch_type<__half>(bn, map, p, grid, gated, stream);
}

}  // namespace w4
}  // namespace lema
