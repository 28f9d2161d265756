// What the exchanges of the HBM store share (store.cu: opaque value rows; store_quant.cu: rows
// held in 8 or 4 bits): the arguments, the table's layout, the probing groups of lanes, and the
// matching of a prefill chunk. The protocol is described at the head of store.cu.
#pragma once

#include <cuda_runtime.h>

#include "common.cuh"
#include "match.cuh"

namespace lema {
namespace k3 {

constexpr uint64_t kEmpty = 0, kLocked = 1;
constexpr int kThreads = 256;

struct Args {
  unsigned char* table;  // the header array
  unsigned char* rows;   // the row array, table + 16 * cap
  uint64_t cap;
  int64_t stride;        // bytes per row in the row array
  int64_t vbytes;
  const void* qc;
  const void* kc;
  const unsigned char* v;
  unsigned char* out;
  int64_t n, T;
  uint64_t g0;
  int64_t* counts;
  uint32_t* status;
  const int32_t* src;
  const void* lt_code;
  const int32_t* lt_pos;
  const int32_t* lt_count;
  uint64_t seg_groups;  // > 0: groups [k * seg_groups, (k + 1) * seg_groups) have their home
  uint64_t seg_slots;   //   slots in [k * seg_slots, (k + 1) * seg_slots); probing still wraps cap
  // strided value and output rows (heads > 0): item (partition p = b * heads + h, position t)
  // reads its value row at v + b * v_sb + h * v_sh + t * v_st and writes its output row at
  // out + b * o_sb + h * o_sh + t * o_st (bytes); heads = 0: rows of item i at i * vbytes
  int64_t heads, v_sb, v_sh, v_st, o_sb, o_sh, o_st;
  int phase;  // T == 1: 3 = look up then insert, 1 = look up only, 2 = insert only
};

__device__ __forceinline__ int64_t row_off(const Args& a, int64_t p, int64_t t, bool out) {
  if (a.heads == 0) return (p * a.T + t) * a.vbytes;
  const int64_t b = p / a.heads, h = p - b * a.heads;
  return out ? b * a.o_sb + h * a.o_sh + t * a.o_st : b * a.v_sb + h * a.v_sh + t * a.v_st;
}
template <typename Vec>
__device__ __forceinline__ const Vec* v_row(const Args& a, int64_t p, int64_t t) {
  return reinterpret_cast<const Vec*>(a.v + row_off(a, p, t, false));
}
template <typename Vec>
__device__ __forceinline__ Vec* out_row(const Args& a, int64_t p, int64_t t) {
  return reinterpret_cast<Vec*>(a.out + row_off(a, p, t, true));
}

// Home slot of (group, code): a 64-bit mix mapped by multiply-high onto the whole table, or,
// when the table is segmented, onto the group's segment. Probing continues across segment
// ends and wraps at cap either way, so capacity and fullness are those of one shared table;
// segmenting only keeps one layer's exchange (its groups) inside a slice of the table.
__device__ __forceinline__ uint64_t home_hash(uint64_t code, uint64_t group) {
  return fmix64(code ^ fmix64(group ^ 0x5851F42D4C957F2Dull));
}
__device__ __forceinline__ uint64_t home(uint64_t code, uint64_t group, const Args& a) {
  const uint64_t h = home_hash(code, group);
  if (a.seg_groups == 0) return __umul64hi(h, a.cap);
  return (group / a.seg_groups) * a.seg_slots + __umul64hi(h, a.seg_slots);
}

__device__ __forceinline__ uint64_t ld_acquire(const uint64_t* p) {
  uint64_t v;
  asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ void st_release(uint64_t* p, uint64_t v) {
  asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

// Probing is done by a GROUP of kG = 8 lanes per item: each round trip the group reads the
// next kG consecutive headers (one per lane, 16 bytes each: 128 contiguous bytes) and decides
// with one ballot which slot, in probe order, ends the probe (its entry, or an empty slot).
// A chain of c slots then costs about c / 8 dependent round trips instead of c: at load 0.95
// an unsuccessful linear probe averages ~200 slots. Calls with few items (a batch-1 decode
// step has 64 per layer) use whole warps instead (kWideG = 32 slots per round trip): the
// lanes are there for free; mid-sized calls (a batch-256 decode step: 16384 items per layer)
// use 16 lanes, measured 3.5% faster per step than 32 (fewer waves of warps) and 8% faster
// than 8 (fewer round trips at load 0.65).
constexpr int kG = 8;
constexpr int kWideG = 32;
constexpr int kMidG = 16;
constexpr int64_t kWideMaxItems = 4096;   // up to this many items per call: 32-lane groups
constexpr int64_t kMidMaxItems = 16384;   // up to this many: 16-lane groups

template <int G>
struct Lane {
  int j;           // index in the group
  int gbase;       // the group's first lane in the warp
  unsigned gmask;  // the group's lanes
  __device__ __forceinline__ unsigned bits(unsigned ballot) const {
    return G == 32 ? ballot : (ballot >> gbase) & ((1u << G) - 1u);
  }
};
template <int G>
__device__ __forceinline__ Lane<G> group_lane() {
  const int lane = threadIdx.x & 31;
  const int base = lane & ~(G - 1);
  return Lane<G>{lane & (G - 1), base, G == 32 ? 0xFFFFFFFFu : (((1u << G) - 1u) << base)};
}

__device__ __forceinline__ uint64_t wrap_add(uint64_t s, uint64_t d, uint64_t cap) {
  s += d;
  while (s >= cap) s -= cap;
  return s;
}

__device__ __forceinline__ uint64_t* header(const Args& a, uint64_t s) {
  return reinterpret_cast<uint64_t*>(a.table) + 2 * s;
}
template <typename Vec>
__device__ __forceinline__ Vec* row_of(const Args& a, uint64_t s) {
  return reinterpret_cast<Vec*>(a.rows + s * a.stride);
}
// (code, state) of slot s, through L2: other items of the same launch may claim slots of it
__device__ __forceinline__ void read_header(const Args& a, uint64_t s, uint64_t& code, uint64_t& state) {
  const ulonglong2 h = __ldcg(reinterpret_cast<const ulonglong2*>(header(a, s)));
  code = h.x;
  state = h.y;
}

// T > 1: fills src, lt_code, lt_pos and lt_count of `a` for its n items in partitions of T: each
// query's latest earlier key inside the chunk, and each partition's distinct key codes with
// their last positions (in the workspace, store_workspace_bytes(n, T, code_bytes) bytes).
int chunk_match(Args& a, void* ws, size_t ws_bytes, int code_bytes, cudaStream_t stream);

// Lanes per item for a call of n items (LEMA_K3_WIDE_MAX, LEMA_K3_GROUP override).
int group_lanes(int64_t n);

}  // namespace k3

size_t store_workspace_bytes(int64_t n, int64_t T, int code_bytes);

}  // namespace lema
