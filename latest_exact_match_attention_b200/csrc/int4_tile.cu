// Products of many rows with 4-bit weights (int4_linear.cu's definition; prompts and large decode batches).
// The floor is the tensor cores' 2 M N K operations; bound by the dequantisation (below). One persistent CTA per SM walks tiles of 128 weight rows
// (features) x BN tokens, features on the M side of tcgen05.mma so that the weights' fragment layout is
// also this kernel's and a small batch needs no padding to 128 rows. Warp roles:
//   warp 0      TMA producer: BN x 64 tiles of x (128-byte swizzle) into a ring of stages;
//   warp 1      MMA issuer: per stage 4 x tcgen05.mma M128 N(BN) K16 into one of two fp32 TMEM
//               accumulators; tcgen05.commit frees the stage;
//   warps 2-5   epilogue: a lane holds one feature, a TMEM column one token; adds the residual or applies
//               the activation (a gate and its up feature are 8 lanes apart) and rounds once;
//   the others  dequantisation, four sets of 2 or 4 warps that take the stages in turn: each warp turns four or
//               two blocks of 16 features x 64 inputs a stage into 16-bit floats and writes them where the MMA's
//               A operand expects them (the same swizzle). Its words and scales are loaded a stage of its own
//               ahead. (Brought by TMA into a ring in shared memory instead they were 1 to 3% faster, and wrong
//               unless a slot was given back only behind the proxy fence that follows the last use of its words.)
// What bounds it, measured with parts left out: 8192 rows through 4096 x 4096 take 207 us, 6% less without the
// subtraction and the product of every weight, 166 where the tensor cores wait for no weights at all; a stage takes
// 0.36 us in narrow tiles (0.21 without dequantisation: four MMAs of 64 tokens, their issue and the ring's waits)
// and 0.42 in tiles of 256 tokens.
// Here a weight is rounded: s * q (8 + 4 significant bits, or 11 + 4) is rounded once to the rows' 16-bit
// type, since the tensor core multiplies one type and a tile cannot scale its sums by groups without
// reading the accumulator back every 32 to 128 inputs. That is half a step a weight, the rounding that a
// 16-bit checkpoint of the same weights has. fp16 has too short a range for every s q (|s| above 8188, bf16 scales
// below 2^-14): a feature's weights are held times a power of two that its largest scale sets, so that none is
// infinite and, of bf16 scales, none of at least 2^-25 of the feature's largest a subnormal; the sums are brought back
// in fp32. (fp16's own subnormal products are exact, so fp16 scales are only ever brought down.) Both the
// dequantising and the epilogue's warps read a tile's scales for it first: 0.5 us of 64 rows 1536 x 4096 in groups of 128
// (9.7 -> 10.2), 2 in groups of 32 (10.1 -> 12.2); 8192 rows gate/up 170 -> 178, 16384 rows 182 -> 185.
//
// Every wait is bounded (tcgen05.cuh); a wait that runs out sets the abort flag and
// LEMA_STATUS_PROBE_LIMIT, and the CTA drains its copies and MMAs and frees its TMEM.
#include <algorithm>
#include <type_traits>

#include "int4.cuh"
#include "tcgen05.cuh"

namespace lema {
namespace w4 {

using namespace tc;

constexpr int kTileRows = 128;                    // weight rows a tile
constexpr int kABytes = kTileRows * kBK * 2;      // 16 KiB
constexpr int kTileBlocks = kTileRows / 16;       // block rows a tile
// Sets of dequantising warps; set i fills stages i, i + kSets, ... Stages are a multiple of kSets, so that the phase
// before the one that a set waits for is one that this set has seen: a parity cannot tell a phase from the one two
// before it.
constexpr int kSets = 4;

constexpr int kSplits[] = {1, 2, 3, 4, 6, 8};  // CTAs of a cluster that may share a tile's K

// Room for tiles of up to BN tokens.
template <int BN>
struct Tile {
  static constexpr int kStageBytes = kABytes + BN * kBK * 2;
  static constexpr int kStages = BN == 64 ? 8 : 4;
  // narrow tiles are bound by how long a block takes, wide ones by the instructions for all of them: half the warps
  // with twice the blocks each spend fewer on waiting and addresses (8192 rows gate/up 2 x 4096 x 1536: 166 -> 160 us;
  // 64 rows 1536 x 4096 in narrow tiles: 9.0 -> 9.9)
  static constexpr int kSetWarps = BN == 64 ? 4 : 2;
  static constexpr int kMine = kTileBlocks / kSetWarps;  // block rows a warp
  static constexpr int kThreads = 32 * (6 + kSets * kSetWarps);
  static constexpr uint32_t kTmemCols = 2 * BN;
  static constexpr int kUnitBytes = 8 * kTileRows * 4;  // 8 tokens of a tile's sums
  // What a CTA of a split tile receives: the others' sums of its units (256 tokens: 16 units at 2 CTAs, 30 at 6, 28 at 8).
  static constexpr int exchange_bytes() {
    int most = 0;
    for (const int split : kSplits) most = std::max(most, (split - 1) * ((BN / 8 + split - 1) / split) * kUnitBytes);
    return most;
  }
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + 1024 /* alignment */ + 512 /* barriers */;
};

struct TileArgs {
  Args a;
  uint32_t* status;
  uint64_t wait_ns;
  int64_t n_tiles;
  int f_tiles;       // tiles along the weight rows
  int bn;            // tokens a tile, a multiple of 32
  int split;         // CTAs of a cluster that share a tile's K (1: none)
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

// fp16 rows: a feature's weights times 2^shift (the head of this file), |s q| 2^shift < 65520. largest: the bits of
// the feature's largest |s|, fp16 (kSame) or bf16.
template <bool kSame>
__device__ __forceinline__ int shift_of(uint32_t largest) {
  if constexpr (kSame) return min(0, 27 - static_cast<int>(largest >> 10));   // 12 - (exponent - 15)
  // within fp32's powers of two, and 2^-shift too: what the upper end costs is far below fp16's smallest value
  return max(-116, min(126, 139 - static_cast<int>(largest >> 7)));           // 12 - (exponent - 127)
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }  // -126 ... 127

// The scale of one row of a fragment: kSame (the scales have the rows' type) as a pair for a 16-bit multiply,
// whose exact operands' product rounds once, else as fp32. up: 2^shift of an fp16 row.
template <typename T, bool kSame> struct RowScale;
template <typename T> struct RowScale<T, true> {
  uint32_t s;
  __device__ __forceinline__ RowScale(uint32_t two, int hi, int, uint32_t up) : s(hi ? (two >> 16) | (two & 0xFFFF0000u) : (two & 0xFFFFu) | (two << 16)) {
    if constexpr (std::is_same<T, __half>::value) s = times(up);
  }
  __device__ __forceinline__ uint32_t times(uint32_t q) const {
    const typename Pair<T>::P r = __hmul2(*reinterpret_cast<const typename Pair<T>::P*>(&q), *reinterpret_cast<const typename Pair<T>::P*>(&s));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <typename T> struct RowScale<T, false> {
  float s;
  __device__ __forceinline__ RowScale(uint32_t two, int hi, int scale_bf16, uint32_t up)
      : s(scale_of(static_cast<uint16_t>(hi ? two >> 16 : two), scale_bf16)) {
    if constexpr (std::is_same<T, __half>::value) s *= __uint_as_float(up);
  }
  __device__ __forceinline__ uint32_t times(uint32_t q) const {
    const float2 v = Pair<T>::to_f2(q);
    return Pair<T>::from_f(v.x * s, v.y * s);
  }
};

// wait_phase by a whole warp: every lane gets the same answer, so that all of them go on or none does.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status, uint64_t wait_ns) {
  return __all_sync(0xFFFFFFFFu, wait_phase(bar, parity, abort_flag, status, wait_ns));
}

__device__ __forceinline__ bool warp_ready(uint32_t bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity)); }

__device__ __forceinline__ void mma_16bit(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  mma_bf16(d_tmem, a_desc, b_desc, idesc, acc);  // kind::f16; the types are the descriptor's
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 16 bytes into the shared memory of CTA `rank` of the cluster, at this CTA's address `addr`.
__device__ __forceinline__ void store_remote(uint32_t addr, uint32_t rank, float a, float b, float c, float d) {
  uint32_t to;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(addr), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

// silu(g) * u with approximate exponential and reciprocal: within 2^-17 of the value for |g| < 87 (the exponent's
// product is off by half a unit in its last place, |g| 2^-24 of it), far inside the 16-bit rounding that follows;
// below -87 zero, where silu is under 2^-119. The exact quotient's slow path kept the epilogue behind the tiles:
// 8192 rows, 2 x 4096 x 1536: 287 -> 214 us.
__device__ __forceinline__ float gate_up_fast(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r * u;
}

// A fragment's row g lies at row slot(g) of its 8 rows of the A operand: with consecutive g four rows apart, the eight
// lanes of one write phase (two g, four chunks each) cover all banks of the swizzled rows. row_of(slot(g)) == g.
__device__ __forceinline__ int slot_of(int g) { return ((g & 1) << 2) | (g >> 1); }
__device__ __forceinline__ int row_of(int slot) { return ((slot & 3) << 1) | (slot >> 2); }

// The outputs of kCols tokens of this lane's weight row, from their fp32 sums: residual or activation, one
// rounding, stores. m: the first token.
template <typename T, bool kGated, int kCols>
__device__ __forceinline__ void finish(const TileArgs& p, int row, int64_t m, const float (&r)[kCols]) {
  const Args& a = p.a;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kCols), a.M - m));  // tokens there are
  // lanes l and l ^ 4 hold two adjacent features; the first finishes both for one token of a pair, the second for
  // the other, so that outputs and residual move in 32-bit words where rows allow it
  const int odd = (row >> 2) & 1;
  float v[kGated ? kCols / 4 : kCols / 2][2];
  int f, step, first;  // v[i]: features f, f + 1 of token first + i * step
  if constexpr (kGated) {
    // block rows hold 8 gate rows, then the 8 up rows of the same features: lanes l and l ^ 8 swap one
    // value of each pair of tokens, and each applies the activation to one token
    const bool gate = (row & 8) == 0;
    float act[kCols / 2];
#pragma unroll
    for (int c = 0; c < kCols / 2; ++c) {
      const float other = __shfl_xor_sync(0xFFFFFFFFu, gate ? r[2 * c + 1] : r[2 * c], 8);
      act[c] = gate_up_fast(gate ? r[2 * c] : other, gate ? other : r[2 * c + 1]);
    }
#pragma unroll
    for (int c = 0; c < kCols / 4; ++c) {
      const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? act[2 * c] : act[2 * c + 1], 4);
      v[c][0] = odd ? other : act[2 * c];
      v[c][1] = odd ? act[2 * c + 1] : other;
    }
    f = (row >> 4) * 8 + 2 * (row & 3);
    step = 4;
    first = 2 * odd + (gate ? 0 : 1);
  } else {
#pragma unroll
    for (int c = 0; c < kCols / 2; ++c) {
      const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? r[2 * c] : r[2 * c + 1], 4);
      v[c][0] = odd ? other : r[2 * c];
      v[c][1] = odd ? r[2 * c + 1] : other;
    }
    f = (row & ~7) + 2 * (row & 3);
    step = 2;
    first = odd;
  }
  constexpr int kN = kGated ? kCols / 4 : kCols / 2;
  if (f >= a.N) return;
  T* y = static_cast<T*>(a.y) + (m + first) * a.ldy + f;
  const T* res = kGated || a.r == nullptr ? nullptr : static_cast<const T*>(a.r) + (m + first) * a.ldr + f;
  const int64_t dy = step * a.ldy, dr = step * a.ldr;
  if (p.pairs) {
    if (res != nullptr) {
      uint32_t rs[kN];  // all of them in flight before the first store
#pragma unroll
      for (int i = 0; i < kN; ++i) rs[i] = first + i * step < rows ? *reinterpret_cast<const uint32_t*>(res + i * dr) : 0u;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float2 add = Pair<T>::to_f2(rs[i]);
        v[i][0] += add.x;
        v[i][1] += add.y;
      }
    }
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (first + i * step < rows) *reinterpret_cast<uint32_t*>(y + i * dy) = Pair<T>::from_f(v[i][0], v[i][1]);
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if (first + i * step >= rows) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (f + e < a.N) y[i * dy + e] = from_f<T>(v[i][e] + (res != nullptr ? to_f(res[i * dr + e]) : 0.f));
    }
  }
}

template <typename T, int BN, bool kGated, bool kSame, bool kSplit>
__global__ void __launch_bounds__(Tile<BN>::kThreads, 1) tile_kernel(const __grid_constant__ CUtensorMap map_x, const TileArgs p) {
  using TL = Tile<BN>;
  constexpr int kStages = TL::kStages, kStageBytes = TL::kStageBytes, kSetWarps = TL::kSetWarps, kMine = TL::kMine;
  // instruction descriptor (tcgen05.mma kind::f16): fp32 accumulator, A and B of type T (0 fp16, 1 bf16), both
  // K-major, N >> 3 at bits 17-22, M >> 4 at bits 24-28
  constexpr uint32_t kType = Pair<T>::kBf16;
  const uint32_t instr_desc = (1u << 4) | (kType << 7) | (kType << 10) | (uint32_t(p.bn >> 3) << 17) | (uint32_t(kTileRows >> 4) << 24);
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

  constexpr bool kShift = std::is_same<T, __half>::value;
  const Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // what brings the sums of row `row_in` of tile f_tile back (kShift): one over its feature's power of two
  auto back = [&](int f_tile, int row_in) {
    const int rb = min(f_tile * kTileBlocks + (row_in >> 4), a.n_rb - 1);
    const uint16_t* s = a.scales + static_cast<int64_t>(rb) * a.n_groups * 16 + row_of(row_in & 7) * 2 + ((row_in >> 3) & 1);
    uint32_t largest = 0;
#pragma unroll 8
    for (int grp = 0; grp < a.n_groups; ++grp) largest = max(largest, __ldg(s + grp * 16) & 0x7FFFu);
    return power_of_two(-shift_of<kSame>(largest));
  };
  // this CTA's tiles, and its share of their K blocks
  // (grid: x the CTAs of a cluster, y the tiles; read as blockIdx and gridDim everywhere, which keeps the loops'
  // counters and the MMA's descriptors in uniform registers: copies of them cost 8% at 16384 rows)
  const int split = kSplit ? p.split : 1, rank = kSplit ? static_cast<int>(blockIdx.x) : 0;
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * a.n_kb / split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * a.n_kb / split);
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
  griddep_launch();
  griddep_wait();  // launched as a dependent: x and the residual are read only from here on

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (x)
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, issued = 0, last_ph = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.y; ok && tile < p.n_tiles; tile += gridDim.y) {
        const int m0 = static_cast<int>(tile / p.f_tiles) * p.bn;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_phase(empty_bar(s), ph ^ 1u, s_abort, p.status, p.wait_ns)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(xfull_bar(s), static_cast<uint32_t>(p.bn * kBK * 2));
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
      for (int64_t tile = blockIdx.y; ok && tile < p.n_tiles; tile += gridDim.y) {
        if (!wait_phase(acce_bar(acc), aph ^ 1u, s_abort, p.status, p.wait_ns)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = kb0; kb < kb1; ++kb) {
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
            mma_16bit(d_tmem, a_desc + 2u * kk, b_desc + 2u * kk, instr_desc, (kb - kb0) | kk ? 1u : 0u);
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
    int acc = 0;
    uint32_t aph = 0;
    for (int64_t tile = blockIdx.y; !kSplit && tile < p.n_tiles; tile += gridDim.y) {
      float times = 1.f;
      if constexpr (kShift) times = back(static_cast<int>(tile % p.f_tiles), quarter * 32 + lane);
      if (!warp_wait(accf_bar(acc), aph, s_abort, p.status, p.wait_ns)) break;
      tc_fence_after();
      const int64_t m0 = (tile / p.f_tiles) * p.bn;
      const int row = static_cast<int>(tile % p.f_tiles) * kTileRows + quarter * 32 + lane;  // weight row
      for (int j = 0; j < p.bn; j += 32) {
        const int64_t m = m0 + j;
        if (m >= a.M) break;  // warp-uniform
        uint32_t r[32];
        tmem_load32(tmem_base + lane_base + static_cast<uint32_t>(acc * BN + j), r);
        float v[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = kShift ? __uint_as_float(r[c]) * times : __uint_as_float(r[c]);
        finish<T, kGated, 32>(p, row, m, v);
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
    // row r's 16-byte chunk c lies at r * 128 + ((c ^ (r & 7)) << 4) of the stage
    const uint32_t row0 = (blk0 * 16 + slot_of(g)) * 128;
    const uint32_t c0 = row0 + (t ^ slot_of(g)) * 16, c1 = row0 + ((4 + t) ^ slot_of(g)) * 16;
    const int sc_second = a.log_group == 5 ? 8 : 0;  // to the upper half's scales
    int s = set, skip = kb0 + set;  // skip: the place along K of this set's next stage
    uint32_t ph = 1;
    for (int64_t tile = blockIdx.y; tile < p.n_tiles; tile += gridDim.y) {
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
          next_sc[b][0] = next_sc[b][1] = __ldg(sp[b] + grp * 8);
          if (up != 0) next_sc[b][1] = __ldg(sp[b] + grp * 8 + up);
        }
      };
      int kb = skip;
      if (kb < kb1) fetch(kb);
      uint32_t shift[kMine][2];  // 2^shift of rows g and g + 8 (kShift): a pair of fp16, or fp32
      if constexpr (kShift) {
        uint32_t top[kMine];  // of rows g and g + 8, the lanes of a row each a quarter of its groups
#pragma unroll
        for (int b = 0; b < kMine; ++b) top[b] = 0;
#pragma unroll (16 / kMine)
        for (int grp = t; grp < a.n_groups; grp += 4)
#pragma unroll
          for (int b = 0; b < kMine; ++b) top[b] = __vmaxu2(top[b], __ldg(sp[b] + grp * 8) & 0x7FFF7FFFu);
#pragma unroll
        for (int b = 0; b < kMine; ++b) {
          top[b] = __vmaxu2(top[b], __shfl_xor_sync(0xFFFFFFFFu, top[b], 1));
          top[b] = __vmaxu2(top[b], __shfl_xor_sync(0xFFFFFFFFu, top[b], 2));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int e = shift_of<kSame>(i ? top[b] >> 16 : top[b] & 0xFFFFu);
            if constexpr (kSame)
              shift[b][i] = Pair<T>::from_f(power_of_two(e), power_of_two(e));
            else
              shift[b][i] = __float_as_uint(power_of_two(e));
          }
        }
      }
      for (; kb < kb1; kb += kSets) {
        uint4 w[kMine];
        uint32_t sc[kMine][2];
#pragma unroll
        for (int b = 0; b < kMine; ++b) {
          w[b] = next[b];
          sc[b][0] = next_sc[b][0];
          sc[b][1] = next_sc[b][1];
        }
        fetch(min(kb + kSets, kb1 - 1));
        unsigned char* dst = smem + s * kStageBytes;
#pragma unroll
        for (int b = 0; b < kMine; ++b) {
          uint4 v[2][2];  // [row g / g + 8][half]: 8 consecutive inputs each
          const uint32_t words[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t f0[4], f1[4];
            Unpack<T>::run(words[2 * h], f0);
            Unpack<T>::run(words[2 * h + 1], f1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const RowScale<T, kSame> rs(sc[b][h], i, a.scale_bf16, kShift ? shift[b][i] : 0u);
              v[i][h].x = rs.times(f0[i]);
              v[i][h].y = rs.times(f0[i + 2]);
              v[i][h].z = rs.times(f1[i]);
              v[i][h].w = rs.times(f1[i + 2]);
            }
          }
          if (b == 0 && !warp_ready(empty_bar(s), ph) && !warp_wait(empty_bar(s), ph, s_abort, p.status, p.wait_ns)) goto done;
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
      skip = kb - kb1 + kb0;
    }
  done:;
  }

  if constexpr (kSplit) {
    // One tile a cluster: CTA q of it finishes units u = q, q + split, ... of 8 tokens. When all CTAs' products are done,
    // and with them the last read of any stage, every CTA sends its sums of the others' units over their stages; all
    // meet again, and the sums are added in the order of the ranks.
    const int64_t m0 = static_cast<int64_t>(blockIdx.y / p.f_tiles) * p.bn;
    const int quarter = warp & 3, row_in = quarter * 32 + lane;
    const int row = static_cast<int>(blockIdx.y % p.f_tiles) * kTileRows + row_in;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const bool live = warp >= 2 && warp < 6;
    const int mine = (p.bn / 8 + split - 1) / split;  // units of one CTA
    // where source q's sums of my unit k lie: [q or q - 1][k][two halves of 4 tokens][128 rows], over the stages
    // (launch_tile checks that they hold it)
    auto place = [&](int src, int dst, int k) {
      return sbase + static_cast<uint32_t>(((src < dst ? src : src - 1) * mine + k) * TL::kUnitBytes + row_in * 16);
    };
    bool ok = false;
    float times = 1.f;
    if (live) {
      if constexpr (kShift) times = back(static_cast<int>(blockIdx.y % p.f_tiles), row_in);
      ok = warp_wait(accf_bar(0), 0, s_abort, p.status, p.wait_ns);
      tc_fence_after();
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (live && ok) {
      for (int u = 0; u < p.bn / 8; ++u) {
        const int to = u % split;
        if (to == rank || m0 + u * 8 >= a.M) continue;  // warp-uniform
        uint32_t r[8];
        tmem_load8(tmem_base + lane_base + static_cast<uint32_t>(u * 8), r);
        const uint32_t at = place(rank, to, u / split);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          store_remote(at + h * (TL::kUnitBytes / 2), to, __uint_as_float(r[4 * h]), __uint_as_float(r[4 * h + 1]),
                       __uint_as_float(r[4 * h + 2]), __uint_as_float(r[4 * h + 3]));
      }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (live && ok) {
      for (int k = 0; k < mine; ++k) {
        const int u = k * split + rank;
        if (u * 8 >= p.bn || m0 + u * 8 >= a.M) break;  // warp-uniform
        uint32_t r[8];
        tmem_load8(tmem_base + lane_base + static_cast<uint32_t>(u * 8), r);
        float v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = 0.f;
        for (int q = 0; q < split; ++q) {
          if (q == rank) {
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] += __uint_as_float(r[c]);
            continue;
          }
          const uint32_t at = place(q, rank, k);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float f[4];
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3])
                         : "r"(at + h * (TL::kUnitBytes / 2))
                         : "memory");
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * h + c] += f[c];
          }
        }
        if constexpr (kShift) {
#pragma unroll
          for (int c = 0; c < 8; ++c) v[c] *= times;
        }
        finish<T, kGated, 8>(p, row, m0 + u * 8, v);
      }
    }
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

template <typename T, int BN, bool kGated, bool kSame, bool kSplit>
int launch_tile(const CUtensorMap& map, const TileArgs& p, int grid, cudaStream_t stream) {
  static_assert(!kSplit || Tile<BN>::exchange_bytes() <= Tile<BN>::kStages * Tile<BN>::kStageBytes, "the exchange stays inside the stages");
  const auto kernel = tile_kernel<T, BN, kGated, kSame, kSplit>;
  LEMA_TRY(kernel_facts(reinterpret_cast<const void*>(kernel), Tile<BN>::kSmemBytes, 0, 0, nullptr));
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>(p.split), static_cast<unsigned>(grid));
  cfg.blockDim = dim3(Tile<BN>::kThreads);
  cfg.dynamicSmemBytes = Tile<BN>::kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  if (pdl_enabled()) {  // a dependent launch, see common.cuh
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.split > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(p.split);
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  LEMA_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map, p));
  return LEMA_OK;
}

template <typename T, int BN, bool kGated, bool kSame>
int launch_split(const CUtensorMap& map, const TileArgs& p, int grid, cudaStream_t stream) {
  if (p.split > 1) return launch_tile<T, BN, kGated, kSame, true>(map, p, grid, stream);
  return launch_tile<T, BN, kGated, kSame, false>(map, p, grid, stream);
}

template <typename T, int BN>
int launch_width(const CUtensorMap& map, const TileArgs& p, int grid, bool gated, cudaStream_t stream) {
  const bool same = p.a.scale_bf16 == Pair<T>::kBf16;
  if (gated) return same ? launch_split<T, BN, true, true>(map, p, grid, stream) : launch_split<T, BN, true, false>(map, p, grid, stream);
  return same ? launch_split<T, BN, false, true>(map, p, grid, stream) : launch_split<T, BN, false, false>(map, p, grid, stream);
}

template <typename T>
int launch_type(const CUtensorMap& map, const TileArgs& p, int grid, bool gated, cudaStream_t stream) {
  if (p.bn <= 64) return launch_width<T, 64>(map, p, grid, gated, stream);
  if (p.bn <= 128) return launch_width<T, 128>(map, p, grid, gated, stream);
  return launch_width<T, 256>(map, p, grid, gated, stream);
}

// The tile width and the split of K with the least estimated time (us): rounds of tiles over the SMs, or of
// clusters over what can be resident at once, each of n_kb / split stages of 0.36 (the dequantising warps', up to 128
// tokens) to 0.42 (256 tokens), and a fixed part: filling the ring, the last epilogue, a split's exchange. A stage
// costs the same at 64 and 128 tokens, so wide tiles split over more CTAs beat narrow ones. Measured, 1536 x 4096:
// 64 rows 9.0 split 8 ways, 28 not split; 256 rows 14.1 (tiles of 128, split 4), 14.8 (256, 8), 18.5 (64, 2), 27.9 (64,
// not split); 512 rows 18.3 (256, 4), 27.9 (128, not split). Gate/up 2 x 4096 x 1536, 256 rows: 14.3 (128, not
// split), 17.9 (256, 2), 21.0 (64, not split). Of nine such shapes the estimate picks the fastest or one within 7%.
template <int BN>
int clusters_at_once(int split, int* out) {
  const auto kernel = tile_kernel<__nv_bfloat16, BN, false, true, true>;  // the others' resources are the same
  return kernel_facts(reinterpret_cast<const void*>(kernel), Tile<BN>::kSmemBytes, Tile<BN>::kThreads, split, out);
}

int choose_shape(TileArgs& p, int sms) {
  double best = 0;
  for (const int bn : {32, 64, 128, 256}) {
    if (bn > 32 && bn / 2 >= p.a.M) break;  // wider than the rows there are
    const int64_t tiles = ((p.a.M + bn - 1) / bn) * p.f_tiles;
    for (const int split : kSplits) {
      int at_once = sms;
      if (split > 1) {
        if (tiles * split > sms || p.a.n_kb < 3 * split) continue;
        LEMA_TRY(bn <= 64 ? clusters_at_once<64>(split, &at_once)
                          : (bn == 128 ? clusters_at_once<128>(split, &at_once) : clusters_at_once<256>(split, &at_once)));
        if (at_once < 1) continue;
      }
      const double rounds = static_cast<double>((tiles + at_once - 1) / at_once);
      const double stage = 0.36 + 0.0005 * std::max(0, bn - 128);
      const double us = rounds * ((p.a.n_kb + split - 1) / split) * stage + 0.01 * bn + (split > 1 ? 1.5 + 0.01 * bn : 0);
      if (best == 0 || us < best) {
        best = us;
        p.bn = bn;
        p.split = split;
        p.n_tiles = tiles;
      }
    }
  }
  return LEMA_OK;
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
  LEMA_TRY(choose_shape(p, dev->sms));
  CUtensorMap map;
  if (!encode_kmajor(enc, &map, a.x, a.M, a.K, a.ldx, p.bn,
                     dtype == LEMA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "int4_linear: tensor map encoding failed (M=%lld K=%d ldx=%lld)", (long long)a.M, a.K, (long long)a.ldx);
  const int grid = static_cast<int>(std::min<int64_t>(p.n_tiles, dev->sms));
  if (dtype == LEMA_BF16) return launch_type<__nv_bfloat16>(map, p, grid, gated, stream);
  return launch_type<__half>(map, p, grid, gated, stream);
}

}  // namespace w4
}  // namespace lema
