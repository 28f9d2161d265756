// K3 with value rows held in 8 or 4 bits: the exchange of store.cu (same table, probing and claim
// protocol; code/lema/csrc/store.cpp:122-162 for the semantics) where a key's row is quantised in
// registers as it is written and a found row is given back as the values its codes stand for.
// Every row costs the store 32 instead of 48 bytes (24 bf16 values in 8 bits) or 16 (in 4 bits).
//
// A held row: codes of chunks of 8 values (8 bytes a chunk, 4 in int4; the last chunk padded with
// code 0), then the fp32 scales, then zeros up to a multiple of 16 bytes. Codes are computed in
// fp32 and rounded once, ties to even:
//   int8   s = amax / 127 of the row,           code = clamp(rne(v / s), -127, 127)
//   int4   s = amax / 7 of each 32 values,      code = clamp(rne(v / s), -7, 7)
//   fp8    s = the smallest power of two with amax / s <= 448 (a float format's relative step does
//          not depend on the scale, and the quotient is then exact), code = e4m3(v / s)
// and the value given back is s * code, rounded once to the values' type and saturated to its largest
// finite number (a code rounded up must not turn a finite value infinite). The integer quotients
// are the exactly rounded ones: a product with 1 / s gives a candidate that is off by at most one,
// and the remainder v - code * s, exact in one fma, decides. A group with an infinity or a NaN
// comes back as NaN (its scale is NaN): neither can be told by 8 bits of a shared scale.
//
// A group of G lanes serves one item (store.cu), lane j the values 8 j ... 8 j + 7, so d_v <= 8 G
// and a row is one code word and one scale a lane. A decode step takes store.cu's groups (a round trip of
// a long probe chain reads G headers); a prefill chunk's many items are bound by instructions and header
// sectors instead and take the fewest lanes that hold a row, at least 4, and divide by multiplication.
// 1024 partitions x 1024 positions of 24 values, load 0.5, overwriting:
// resolve 138 -> 71 us, insert 125 -> 71; claiming new slots 312 -> 98 (one 16-byte compare-and-swap a claim
// instead of lock, code, fence and state, and claims counted once a warp). An in-chunk match (T > 1) reads the 16-bit row
// of its source and gives back the same numbers the store would: any chunking of a sequence gives
// the same results.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "store.cuh"

namespace lema {
namespace k3 {

constexpr int kMaxQuantDim = 256;  // 8 values a lane, at most 32 lanes an item

// Division of n < 2^31 by a divisor known on the host: (mulhi(n, m) + n) >> s.
struct Divisor {
  uint32_t d, m, s;
  Divisor() = default;
  explicit Divisor(uint32_t by) : d(by), s(0) {
    while ((uint64_t(1) << s) < by) ++s;
    m = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << s) - by)) / by + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

struct QArgs {
  Args a;          // a.vbytes: bytes of a held row; strides of v and out always set (a.heads >= 1)
  int d;           // values per row
  int chunks;      // of 8 values
  int cb;          // bytes per code word of codes, 4 or 8
  int v_vec, o_vec;  // whole chunks readable / writable as 16-byte words
  Divisor by_t, by_heads;
  uint64_t home_base, home_span;  // where the call's groups have their home slots, if in one segment (span > 0)
};

template <int F> struct Format;  // F: LEMA_ROWS_*
template <> struct Format<LEMA_ROWS_INT8> { using Word = uint2; static constexpr int kGroupChunks = 0; };
template <> struct Format<LEMA_ROWS_FP8> { using Word = uint2; static constexpr int kGroupChunks = 0; };
template <> struct Format<LEMA_ROWS_INT4> { using Word = uint32_t; static constexpr int kGroupChunks = 4; };

// One lane's share of a held row.
template <int F> struct Frag {
  typename Format<F>::Word w;
  float s;
};
template <int F>
__device__ __forceinline__ Frag<F> zero_frag() {
  Frag<F> f;
  f.w = zero_vec<typename Format<F>::Word>();
  f.s = 0.f;
  return f;
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Values 8 j ... of a row of d; zeros past its end.
template <typename T>
__device__ __forceinline__ void load8(const unsigned char* row, int j, int d, int vec, float (&f)[8]) {
  const T* p = reinterpret_cast<const T*>(row) + 8 * j;
  const int n = d - 8 * j;
  if (vec && n >= 8) {
    union { uint4 u[sizeof(T) / 2]; T t[8]; } r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f(r.t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? to_f(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(unsigned char* row, int j, int d, int vec, const float (&f)[8]) {
  T* p = reinterpret_cast<T*>(row) + 8 * j;
  const int n = d - 8 * j;
  if (vec && n >= 8) {
    union { uint4 u[sizeof(T) / 2]; T t[8]; } r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.t[i] = from_f<T>(f[i]);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.u[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_f<T>(f[i]);
  }
}

// The lane's 8 values as codes and the scale of their group; all G lanes call it (lanes past the
// row's chunks with zeros).
template <int F, int G>
__device__ __forceinline__ Frag<F> quantise(const float (&f)[8], const Lane<G>& L) {
  // the largest magnitude, by its bits: a NaN is above infinity, and both above every number
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  constexpr int kSpan = Format<F>::kGroupChunks ? Format<F>::kGroupChunks : G;
#pragma unroll
  for (int o = kSpan / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(L.gmask, m, o));
  Frag<F> q = zero_frag<F>();
  if (m >= 0x7F800000u) {
    q.s = __uint_as_float(0x7FC00000u);
    return q;
  }
  if constexpr (F == LEMA_ROWS_FP8) {
    // 448 = 1.75 * 2^8: one step more where the significand is above 1.75
    const int p = max(-126, static_cast<int>(m >> 23) - 127 - ((m & 0x7FFFFFu) <= 0x600000u ? 8 : 7));
    q.s = __uint_as_float(static_cast<uint32_t>(p + 127) << 23);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - p) << 23);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * inv, f[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    q.w = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
  } else {
    constexpr float kTop = F == LEMA_ROWS_INT8 ? 127.f : 7.f;
    q.s = __fdiv_rn(__uint_as_float(m), kTop);
    // rows near the bottom of fp32's range are lifted, so that 1 / s exists; where the scale itself rounds to 0 (fp32 rows
    // below 64 of the smallest steps there are, int4: 4) the codes are 0
    const float lift = q.s < 0x1p-100f ? (q.s > 0.f ? 0x1p100f : 0.f) : 1.f;
    const float s = q.s * lift;
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = f[i] * lift;
      float c = fminf(fmaxf(rintf(v * inv), -kTop), kTop);
      const float r = fmaf(-c, s, v);
      const float r2 = 2.f * fabsf(r);
      if (r2 > s || (r2 == s && (static_cast<int>(c) & 1))) c = fminf(fmaxf(c + copysignf(1.f, r), -kTop), kTop);
      const int code = static_cast<int>(c);
      if constexpr (F == LEMA_ROWS_INT8)
        w[i >> 2] |= static_cast<uint32_t>(code & 0xFF) << (8 * (i & 3));
      else
        w[0] |= static_cast<uint32_t>(code & 0xF) << (4 * i);
    }
    if constexpr (F == LEMA_ROWS_INT8)
      q.w = make_uint2(w[0], w[1]);
    else
      q.w = w[0];
  }
  return q;
}

template <typename T> struct Largest;
template <> struct Largest<float> { static constexpr float kV = 3.402823466e38f; };
template <> struct Largest<__nv_bfloat16> { static constexpr float kV = 3.3895313892515355e38f; };
template <> struct Largest<__half> { static constexpr float kV = 65504.f; };
// v within +-top; a NaN stays one.
__device__ __forceinline__ float saturate(float v, float top) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(top));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(-top));
  return r;
}

template <int F>
__device__ __forceinline__ void values_of(const Frag<F>& q, float (&f)[8]) {
  if constexpr (F == LEMA_ROWS_FP8) {
    const uint32_t w[2] = {q.w.x, q.w.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
      const float2 p = __half22float2(__half2(h));
      f[2 * i] = p.x * q.s;
      f[2 * i + 1] = p.y * q.s;
    }
  } else if constexpr (F == LEMA_ROWS_INT8) {
    const uint32_t w[2] = {q.w.x, q.w.y};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = static_cast<float>(static_cast<int>(w[i >> 2] << (24 - 8 * (i & 3))) >> 24) * q.s;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(static_cast<int>(q.w << (28 - 4 * i)) >> 28) * q.s;
  }
}

// The lane's share of slot s's held row; lanes past the row's chunks get zeros.
template <int F, int G>
__device__ __forceinline__ Frag<F> load_frag(const QArgs& q, uint64_t s, const Lane<G>& L) {
  using Word = typename Format<F>::Word;
  Frag<F> r = zero_frag<F>();
  if (L.j < q.chunks) {
    const unsigned char* row = q.a.rows + s * q.a.stride;
    r.w = reinterpret_cast<const Word*>(row)[L.j];
    constexpr int gc = Format<F>::kGroupChunks;
    r.s = reinterpret_cast<const float*>(row + q.chunks * static_cast<int>(sizeof(Word)))[gc ? L.j / gc : 0];
  }
  return r;
}
// Writes it; the padding behind the scales too, so that equal rows are equal bytes.
template <int F, int G>
__device__ __forceinline__ void store_frag(const QArgs& q, uint64_t s, const Frag<F>& r, const Lane<G>& L) {
  using Word = typename Format<F>::Word;
  unsigned char* row = q.a.rows + s * q.a.stride;
  constexpr int gc = Format<F>::kGroupChunks;
  const int codes = q.chunks * static_cast<int>(sizeof(Word));
  const int groups = gc ? (q.chunks + gc - 1) / gc : 1;
  float* scales = reinterpret_cast<float*>(row + codes);
  if (L.j < q.chunks) {
    reinterpret_cast<Word*>(row)[L.j] = r.w;
    if (gc ? L.j % (gc ? gc : 1) == 0 : L.j == 0) scales[gc ? L.j / gc : 0] = r.s;
  }
  const int pad = (static_cast<int>(q.a.vbytes) - codes) / 4 - groups;  // at most 3 words
  if (L.j < pad) scales[groups + L.j] = 0.f;
}
__device__ __forceinline__ const unsigned char* v_at(const QArgs& q, uint32_t p, uint32_t t) {
  const uint32_t b = q.by_heads.quotient(p), h = p - b * q.by_heads.d;
  return q.a.v + b * q.a.v_sb + h * q.a.v_sh + t * q.a.v_st;
}
__device__ __forceinline__ unsigned char* out_at(const QArgs& q, uint32_t p, uint32_t t) {
  const uint32_t b = q.by_heads.quotient(p), h = p - b * q.by_heads.d;
  return q.a.out + b * q.a.o_sb + h * q.a.o_sh + t * q.a.o_st;
}
template <typename T, int F, int G>
__device__ __forceinline__ Frag<F> quantise_row(const QArgs& q, uint32_t p, uint32_t t, const Lane<G>& L) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.f;
  if (L.j < q.chunks) load8<T>(v_at(q, p, t), L.j, q.d, q.v_vec, f);
  return quantise<F, G>(f, L);
}
template <typename T, int F, int G>
__device__ __forceinline__ void emit_row(const QArgs& q, uint32_t p, uint32_t t, const Frag<F>& r, const Lane<G>& L) {
  if (L.j >= q.chunks) return;
  float f[8];
  values_of<F>(r, f);
  // (an integer code's s * code is within a rounding of fp32 of the row's largest value: 16-bit types round it back)
  if constexpr (F == LEMA_ROWS_FP8 || sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = saturate(f[i], Largest<T>::kV);
  }
  store8<T>(out_at(q, p, t), L.j, q.d, q.o_vec, f);
}

__device__ __forceinline__ uint64_t code_at(const void* p, uint32_t i, int cb) {
  return cb == 4 ? static_cast<uint64_t>(static_cast<const uint32_t*>(p)[i]) : static_cast<const uint64_t*>(p)[i];
}

// home() without its division where all groups of the call share a segment (a layer's call does).
__device__ __forceinline__ uint64_t home_of(const QArgs& q, uint64_t code, uint64_t group) {
  if (q.home_span == 0) return home(code, group, q.a);
  return q.home_base + __umul64hi(home_hash(code, group), q.home_span);
}
// (code, state) of slot s in one 16-byte access, as claim() writes them.
__device__ __forceinline__ void read_slot(const Args& a, uint64_t s, uint64_t& code, uint64_t& state) {
  asm volatile(
      "{\n\t.reg .b128 h;\n\t"
      "ld.relaxed.gpu.global.b128 h, [%2];\n\t"
      "mov.b128 {%0, %1}, h;\n\t}"
      : "=l"(code), "=l"(state)
      : "l"(header(a, s))
      : "memory");
}
// Empty -> (code, state) in one 16-byte compare-and-swap: a prober sees the slot empty or with its code, so the
// slot needs no locked state and no release store behind the row. The row is read by later launches only: within
// one launch nobody else looks for this (group, code).
__device__ __forceinline__ int claim(uint64_t* hdr, uint64_t code, uint64_t state) {
  uint64_t was_code, was_state;
  asm volatile(
      "{\n\t.reg .b128 e, n, o;\n\t"
      "mov.b128 e, {%3, %3};\n\t"
      "mov.b128 n, {%4, %5};\n\t"
      "atom.relaxed.gpu.global.cas.b128 o, [%2], e, n;\n\t"
      "mov.b128 {%0, %1}, o;\n\t}"
      : "=l"(was_code), "=l"(was_state)
      : "l"(hdr), "l"(kEmpty), "l"(code), "l"(state)
      : "memory");
  return (was_code | was_state) == 0;
}

// One item's lookup (want_q) and insert (want_k), their probes interleaved round trip by round
// trip as in store.cu's exchange_both: each round reads the next window of headers of both. The
// retrieved share goes to `got` (zeros on a miss). `mine` is the row to insert. Returns 1 for a
// newly claimed slot, 0 for an overwrite or no insert, -1 when every slot was probed (full).
// Where both probes end at one slot (query code == key code) the group barrier before the write
// orders every lane's reads of the old row, its scale included, before any lane's writes.
template <int F, int G>
__device__ int probe(const QArgs& q, uint64_t g, uint64_t qcode, uint64_t kcode, bool want_q, bool want_k,
                     const Frag<F>& mine, Frag<F>& got, const Lane<G>& L) {
  const Args& a = q.a;
  const uint64_t tag = g + 2;
  uint64_t sq = want_q ? home_of(q, qcode, g) : 0, sk = want_k ? home_of(q, kcode, g) : 0;
  uint64_t tq = 0, tk = 0;
  bool qdone = !want_q;
  int kres = want_k ? 2 : 0;  // 2: probing
  got = zero_frag<F>();
  Frag<F> spec = zero_frag<F>();
  if (want_q) spec = load_frag<F, G>(q, sq, L);  // a hit at home costs one round trip
  while (!qdone || kres == 2) {
    uint64_t qcd = 0, qst = 0, kcd = 0, kst = 0;
    if (!qdone) read_slot(a, wrap_add(sq, L.j, a.cap), qcd, qst);
    if (kres == 2) read_slot(a, wrap_add(sk, L.j, a.cap), kcd, kst);
    if (!qdone) {
      const bool valid = tq + L.j < a.cap;  // no slot twice within one cycle of the table
      const unsigned hit = L.bits(__ballot_sync(L.gmask, valid && qst == tag && qcd == qcode));
      const unsigned emp = L.bits(__ballot_sync(L.gmask, valid && qst == kEmpty));
      const unsigned stop = hit | emp;
      if (stop) {
        const int k = __ffs(stop) - 1;
        qdone = true;
        if ((hit >> k) & 1u) got = (tq == 0 && k == 0) ? spec : load_frag<F, G>(q, wrap_add(sq, k, a.cap), L);
      } else {
        sq = wrap_add(sq, G, a.cap);
        tq += G;
        qdone = tq >= a.cap;
      }
    }
    if (kres == 2) {
      const bool valid = tk + L.j < a.cap;
      const unsigned own = L.bits(__ballot_sync(L.gmask, valid && kst == tag && kcd == kcode));
      const unsigned emp = L.bits(__ballot_sync(L.gmask, valid && kst == kEmpty));
      const unsigned stop = own | emp;
      if (stop) {
        const int k = __ffs(stop) - 1;
        const uint64_t slot = wrap_add(sk, k, a.cap);
        __syncwarp(L.gmask);
        if ((own >> k) & 1u) {
          store_frag<F, G>(q, slot, mine, L);
          kres = 0;
        } else {
          int won = 0;
          if (L.j == k) won = claim(header(a, slot), kcode, tag);
          won = __shfl_sync(L.gmask, won, L.gbase + k);
          if (won) {
            store_frag<F, G>(q, slot, mine, L);
            kres = 1;
          } else {
            sk = wrap_add(slot, 1, a.cap);
            tk += static_cast<uint64_t>(k) + 1;
            if (tk >= a.cap) kres = -1;
          }
        }
      } else {
        sk = wrap_add(sk, G, a.cap);
        tk += G;
        if (tk >= a.cap) kres = -1;
      }
    }
  }
  return kres;
}

// r: probe's answer for partition p, in the first lane of each group (0 in the others). Whole warps call it: claims
// of one partition are added once a warp.
__device__ __forceinline__ void count_claims(const Args& a, uint32_t p, int r) {
  if (r < 0) raise_status(a.status, LEMA_STATUS_TABLE_FULL);
  const unsigned claims = __ballot_sync(kFullMask, r > 0);
  if (claims == 0) return;
  const int first = __ffs(claims) - 1;
  const uint32_t of_first = __shfl_sync(kFullMask, p, first);  // by every lane, before the test that some would skip
  const bool one = __all_sync(kFullMask, r <= 0 || p == of_first);
  if (one ? (threadIdx.x & 31) == first : r > 0)
    atomicAdd(reinterpret_cast<unsigned long long*>(a.counts + p), one ? static_cast<unsigned long long>(__popc(claims)) : 1ull);
}

// T == 1: item i is partition i; phase 3 looks up and inserts, 1 and 2 do one of the two.
template <typename T, int F, int G>
__global__ void __launch_bounds__(kThreads) quant_step(const QArgs q) {
  griddep_wait();  // launched as a dependent: the codes and values first
  const uint32_t i = blockIdx.x * (kThreads / G) + threadIdx.x / G;
  const Lane<G> L = group_lane<G>();
  const bool want_q = q.a.phase & 1, want_k = q.a.phase & 2;
  int r = 0;
  if (i < q.a.n) {  // whole groups
    const uint64_t qcode = want_q ? code_at(q.a.qc, i, q.cb) : 0, kcode = want_k ? code_at(q.a.kc, i, q.cb) : 0;
    Frag<F> mine = zero_frag<F>(), got;
    if (want_k) mine = quantise_row<T, F, G>(q, i, 0, L);
    r = probe<F, G>(q, q.a.g0 + i, qcode, kcode, want_q, want_k, mine, got, L);
    if (want_q) emit_row<T, F, G>(q, i, 0, got, L);
  }
  if (want_k) count_claims(q.a, i, L.j == 0 ? r : 0);
}

// T > 1, after the matcher: a query with an in-chunk match gets the numbers its source row would
// be held as; any other looks the store up.
template <typename T, int F, int G>
__global__ void __launch_bounds__(kThreads) quant_resolve(const QArgs q) {
  griddep_wait();
  const uint32_t i = blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (i >= q.a.n) return;
  const Lane<G> L = group_lane<G>();
  const uint32_t p = q.by_t.quotient(i);
  const int32_t s = q.a.src[i];
  Frag<F> got;
  if (s >= 0) {
    got = quantise_row<T, F, G>(q, p, s, L);
  } else {
    probe<F, G>(q, q.a.g0 + static_cast<uint64_t>(p), code_at(q.a.qc, i, q.cb), 0, true, false, zero_frag<F>(), got, L);
  }
  emit_row<T, F, G>(q, p, i - p * q.by_t.d, got, L);
}

// T > 1: each partition's distinct key codes once, with the row of their last position.
template <typename T, int F, int G>
__global__ void __launch_bounds__(kThreads) quant_insert(const QArgs q) {
  griddep_wait();
  const uint32_t i = blockIdx.x * (kThreads / G) + threadIdx.x / G;
  const Lane<G> L = group_lane<G>();
  const uint32_t p = q.by_t.quotient(i);
  int r = 0;
  if (i < q.a.n && static_cast<int32_t>(i - p * q.by_t.d) < q.a.lt_count[p]) {  // whole groups
    const Frag<F> mine = quantise_row<T, F, G>(q, p, q.a.lt_pos[i], L);
    Frag<F> got;
    r = probe<F, G>(q, q.a.g0 + p, 0, code_at(q.a.lt_code, i, q.cb), false, true, mine, got, L);
  }
  count_claims(q.a, p, L.j == 0 ? r : 0);
}

template <typename T, int F, int G>
int run_quant(QArgs& q, void* ws, size_t ws_bytes, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((q.a.n * G + kThreads - 1) / kThreads)), block(kThreads);
  if constexpr (G >= 8) {
    if (q.a.T == 1) {
      LEMA_CUDA_TRY(launch_dependent(quant_step<T, F, G>, grid, block, 0, stream, q));
      return LEMA_OK;
    }
  }
  LEMA_TRY(chunk_match(q.a, ws, ws_bytes, q.cb, stream));
  LEMA_CUDA_TRY(launch_dependent(quant_resolve<T, F, G>, grid, block, 0, stream, q));
  LEMA_CUDA_TRY(launch_dependent(quant_insert<T, F, G>, grid, block, 0, stream, q));
  return LEMA_OK;
}

template <typename T, int F>
int run_lanes(QArgs& q, void* ws, size_t ws_bytes, cudaStream_t stream) {
  // a decode step: store.cu's lanes. Above 8192 items 8 lanes instead of 16 are faster at low loads and lose far more at high
  // ones, whose chains they walk in twice the round trips (int8, half of the lookups missing, us a layer with 8 / 16 lanes at
  // loads 0.35, 0.65, 0.9: 8320 items 5.1 / 6.2, 8.0 / 7.2, 59 / 38; 16384 items 7.7 / 11.3, 12.4 / 13.0, 87 / 51).
  int G = q.a.T == 1 ? group_lanes(q.a.n) : 4;
  while (G < q.chunks) G *= 2;
  if (G == 32) return run_quant<T, F, 32>(q, ws, ws_bytes, stream);
  if (G == 16) return run_quant<T, F, 16>(q, ws, ws_bytes, stream);
  if (G == 8) return run_quant<T, F, 8>(q, ws, ws_bytes, stream);
  return run_quant<T, F, 4>(q, ws, ws_bytes, stream);
}

template <typename T>
int run_format(int format, QArgs& q, void* ws, size_t ws_bytes, cudaStream_t stream) {
  if (format == LEMA_ROWS_INT8) return run_lanes<T, LEMA_ROWS_INT8>(q, ws, ws_bytes, stream);
  if (format == LEMA_ROWS_FP8) return run_lanes<T, LEMA_ROWS_FP8>(q, ws, ws_bytes, stream);
  return run_lanes<T, LEMA_ROWS_INT4>(q, ws, ws_bytes, stream);
}

}  // namespace k3

// Bytes of a held row of d values, or 0 for an unknown format or width.
int64_t quant_row_bytes(int format, int64_t d) {
  if (d < 1 || d > k3::kMaxQuantDim) return 0;
  const int64_t chunks = (d + 7) / 8;
  if (format == LEMA_ROWS_INT8 || format == LEMA_ROWS_FP8) return static_cast<int64_t>(round_up(chunks * 8 + 4, 16));
  if (format == LEMA_ROWS_INT4) return static_cast<int64_t>(round_up(chunks * 4 + (chunks + 3) / 4 * 4, 16));
  return 0;
}

}  // namespace lema

extern "C" int64_t lema_quant_row_bytes(int format, int64_t d_v) { return lema::quant_row_bytes(format, d_v); }

extern "C" int lema_store_exchange_quant(void* table, int64_t cap, int format, int dtype, int64_t d_v,
                                         const void* qcodes, const void* kcodes, int code_bytes,
                                         const void* values, void* out, int64_t n, int64_t T, int64_t g0,
                                         int64_t* counts, uint32_t* status, void* workspace,
                                         size_t workspace_bytes, int64_t seg_groups, int64_t seg_slots,
                                         int64_t heads, int64_t v_sb, int64_t v_sh, int64_t v_st, int64_t o_sb,
                                         int64_t o_sh, int64_t o_st, int phase, void* stream) {
  using namespace lema;
  clear_error();
  const int64_t vbytes = quant_row_bytes(format, d_v);
  if (format != LEMA_ROWS_INT8 && format != LEMA_ROWS_FP8 && format != LEMA_ROWS_INT4)
    return fail(LEMA_ERR_INVALID_ARGUMENT, "row format %d: int8 (%d), fp8 (%d) or int4 (%d)", format, LEMA_ROWS_INT8, LEMA_ROWS_FP8, LEMA_ROWS_INT4);
  if (vbytes == 0) return fail(LEMA_ERR_INVALID_ARGUMENT, "d_v = %lld: quantised rows hold 1 to %d values", (long long)d_v, k3::kMaxQuantDim);
  if (dtype != LEMA_F32 && dtype != LEMA_BF16 && dtype != LEMA_F16) return fail(LEMA_ERR_INVALID_ARGUMENT, "dtype tag %d", dtype);
  if (code_bytes != 4 && code_bytes != 8) return fail(LEMA_ERR_INVALID_ARGUMENT, "code_bytes must be 4 or 8, got %d", code_bytes);
  if (cap < 1) return fail(LEMA_ERR_INVALID_ARGUMENT, "capacity must be >= 1 slot, got %lld", (long long)cap);
  if (n < 0 || T <= 0 || n % T != 0) return fail(LEMA_ERR_INVALID_ARGUMENT, "items must be partitions x T (n = %lld, T = %lld)", (long long)n, (long long)T);
  if (n >= (int64_t(1) << 31) || heads >= (int64_t(1) << 31)) return fail(LEMA_ERR_INVALID_ARGUMENT, "2^31 - 1 items in one call at most, got %lld", (long long)n);
  if (g0 < 0) return fail(LEMA_ERR_INVALID_ARGUMENT, "negative group offset");
  if (seg_groups < 0 || seg_slots < 0 || (seg_groups > 0) != (seg_slots > 0))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "segments: groups and slots per segment both positive or both 0");
  if (seg_groups > 0 && n > 0 && ((g0 + n / T - 1) / seg_groups + 1) * seg_slots > cap)
    return fail(LEMA_ERR_INVALID_ARGUMENT, "group %lld's segment lies past the table's %lld slots", (long long)(g0 + n / T - 1), (long long)cap);
  if (phase < 1 || phase > 3 || (phase != 3 && T != 1))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "phase %d: 3 (both), or 1 / 2 (lookups / inserts only, T = 1)", phase);
  if (heads < 0 || (heads > 0 && (n / T) % heads != 0))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "strided rows: %lld partitions are not whole groups of heads = %lld", (long long)(n / T), (long long)heads);
  if (n == 0) return LEMA_OK;
  if (table == nullptr || !aligned(table, 16)) return fail(LEMA_ERR_INVALID_ARGUMENT, "table must be a 16-byte aligned device pointer");
  if (counts == nullptr || ((phase & 1) && (qcodes == nullptr || out == nullptr)) || ((phase & 2) && (kcodes == nullptr || values == nullptr)))
    return fail(LEMA_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (!aligned(qcodes, code_bytes) || !aligned(kcodes, code_bytes)) return fail(LEMA_ERR_INVALID_ARGUMENT, "codes not aligned to their width");
  const int64_t es = dtype == LEMA_F32 ? 4 : 2;
  if (!aligned(values, es) || !aligned(out, es) || !aligned(counts, 8)) return fail(LEMA_ERR_INVALID_ARGUMENT, "values, out and counts must be aligned to their elements");
  const size_t need = store_workspace_bytes(n, T, code_bytes);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return fail(LEMA_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (need > 0 && !aligned(workspace, 256)) return fail(LEMA_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  k3::QArgs q{};
  k3::Args& a = q.a;
  if (heads > 0) {
    a.heads = heads;
    a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
    a.o_sb = o_sb; a.o_sh = o_sh; a.o_st = o_st;
    if ((v_sb | v_sh | v_st | o_sb | o_sh | o_st) % es != 0)
      return fail(LEMA_ERR_INVALID_ARGUMENT, "strided rows: strides must be whole elements");
  } else {  // item i's rows at i * d_v elements
    a.heads = 1;
    a.v_sb = a.o_sb = T * d_v * es;
    a.v_st = a.o_st = d_v * es;
  }
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return LEMA_ERR_CUDA;
  if (dev->cc_major != 10) return fail(LEMA_ERR_UNSUPPORTED, "built for sm_100a; device is sm_%d%d", dev->cc_major, dev->cc_minor);
  a.phase = phase;
  a.table = static_cast<unsigned char*>(table);
  a.cap = static_cast<uint64_t>(cap);
  a.rows = a.table + 16 * a.cap;
  a.stride = vbytes;
  a.vbytes = vbytes;
  a.qc = qcodes;
  a.kc = kcodes;
  a.v = static_cast<const unsigned char*>(values);
  a.out = static_cast<unsigned char*>(out);
  a.n = n;
  a.T = T;
  a.g0 = static_cast<uint64_t>(g0);
  a.counts = counts;
  a.status = status;
  a.seg_groups = static_cast<uint64_t>(seg_groups);
  a.seg_slots = static_cast<uint64_t>(seg_slots);
  q.d = static_cast<int>(d_v);
  q.chunks = static_cast<int>((d_v + 7) / 8);
  q.cb = code_bytes;
  q.v_vec = aligned(values, 16) && (a.v_sb | a.v_sh | a.v_st) % 16 == 0;
  q.o_vec = aligned(out, 16) && (a.o_sb | a.o_sh | a.o_st) % 16 == 0;
  q.by_t = k3::Divisor(static_cast<uint32_t>(T));
  q.by_heads = k3::Divisor(static_cast<uint32_t>(a.heads));
  if (seg_groups == 0) {
    q.home_span = a.cap;
  } else if (g0 / seg_groups == (g0 + n / T - 1) / seg_groups) {
    q.home_base = static_cast<uint64_t>(g0 / seg_groups * seg_slots);
    q.home_span = a.seg_slots;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == LEMA_F32) return k3::run_format<float>(format, q, workspace, workspace_bytes, s);
  if (dtype == LEMA_BF16) return k3::run_format<__nv_bfloat16>(format, q, workspace, workspace_bytes, s);
  return k3::run_format<__half>(format, q, workspace, workspace_bytes, s);
}
