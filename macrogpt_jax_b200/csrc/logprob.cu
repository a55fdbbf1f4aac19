// Operators on rows of lm_head logits next to the cross-entropy of xent.cu: log probabilities of
// given tokens with the row's entropy and top alternatives (ufp8_logprob_*), and distillation from
// a teacher's top logits (ufp8_distill_*).
//
// Mathematics.  With temperature T, c = log2(e) / T, m = max_v x_v of a row and z_v = (x_v - m) c:
//   s = sum_v 2^z_v,   t = sum_v 2^z_v z_v,   l2 = log2 s,
//   log p_v = ln 2 (z_v - l2),   H = ln 2 (l2 - t / s)   (both terms of H are >= 0: no cancellation).
// Working with the difference x - m, never with x c, keeps a row of the type's lowest value finite.
// Partials (m, s, t) of two parts merge as M = max(m, m'), d = (m - M) c <= 0:
//   s -> 2^d s,  t -> 2^d (t + d s),  and the same for the primed part, then add.
// All of it is f32, merged in a fixed order; 2^x is the MUFU ex2.approx (2 ulp).
//
//   rowstat_kernel   one CTA per row (or a cluster of them) streams the row once, a running (m, s, t) per
//                    thread, and notes where its largest elements may be; those are read again at the end.
//                    Bound: HBM; next the ex2 of every logit (XU pipe 74 % busy).  4096 x 128256 bf16
//                    (1.05 GB): 154-158 us for log probabilities, 162-164 with the entropy, 157-160 against 64
//                    teacher entries (6.4-6.8 TB/s), 214-217 with 64 alternatives, 313 with 256; 1 x 128256:
//                    3.7 us, 7.2 with 8.
//   rowgrad_kernel   the gradient of both operators: p_v (A + B log2 p_v) with row factors A, B, plus
//                    weights at a few columns (the token, the alternatives, the teacher's entries).
//                    Bound: HBM, read and write.  Same size: 336-347 us (6.1-6.3 TB/s) with up to 64 entries;
//                    360 with 65, 387 with 128, 538 with 256, since each 2 KB of a row looks through all entries
//                    past 64 again.  As fp8 (16384 x 128256, soft cap): 2.1 ms, 3.0 TB/s, bound by instructions;
//                    the pass for the exact amax before it 1.2 ms.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <cmath>
#include <type_traits>

#include "fp8cast.cuh"
#include "internal.h"

namespace ufp8 {
namespace {

constexpr int kThreads = 256;  // of a gradient CTA; a statistics CTA has 256, 128 or 64
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 256;
constexpr int kMaxEntries = 1024;   // teacher entries of a row
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -INFINITY;

__device__ __forceinline__ float ex2a(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max that returns NaN when an operand is NaN
__device__ __forceinline__ float maxn(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint4 ld16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// ---- element types ---------------------------------------------------------------------------
struct Bf16 {
  using raw = uint16_t;
  static constexpr int kElems = 8;    // elements of a unit (16 bytes)
  static constexpr int kKeyBits = 16;
  static __device__ __forceinline__ float to_f(raw r) { return __uint_as_float(static_cast<uint32_t>(r) << 16); }
  static __device__ __forceinline__ raw from_f(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
};
struct F32 {
  using raw = float;
  static constexpr int kElems = 4;
  static constexpr int kKeyBits = 32;
  static __device__ __forceinline__ float to_f(raw r) { return r; }
  static __device__ __forceinline__ raw from_f(float f) { return f; }
};

constexpr int kUnits = 4;  // units per thread and tile, per lane and chunk: 64 bytes of loads in flight

template <class T>
struct Unit {
  uint4 w;
};

template <class T>
__device__ __forceinline__ void unpack(const Unit<T>& u, float (&v)[T::kElems]) {
  const uint32_t w[4] = {u.w.x, u.w.y, u.w.z, u.w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T::kElems == 8) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      v[i] = __uint_as_float(w[i]);
    }
  }
}

// Element j of a unit, j not known at compile time.
template <class T>
__device__ __forceinline__ float pick(const Unit<T>& u, int j) {
  constexpr int kPer = T::kElems / 4;  // elements of a 32-bit word
  const uint32_t lo = (j / kPer & 1) ? u.w.y : u.w.x, hi = (j / kPer & 1) ? u.w.w : u.w.z;
  const uint32_t w = (j / kPer & 2) ? hi : lo;
  return __uint_as_float(kPer == 1 ? w : (j & 1) ? w & 0xFFFF0000u : w << 16);
}

// A row as units of kElems elements that start on 16-byte boundaries: unit i covers the columns from
// kElems i - off on, where off elements lie between the boundary at or below the row's first
// element and that element.  Only the first and the last unit can reach outside the row; those read
// their columns one by one and hold -inf elsewhere.
template <class T>
struct Row {
  const typename T::raw* p;
  int off;
  int V;
  int units;
  __device__ __forceinline__ Row(const void* base, int64_t elem, int v) {
    p = static_cast<const typename T::raw*>(base) + elem;
    off = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(typename T::raw));
    V = v;
    units = (v + off + T::kElems - 1) / T::kElems;
  }
  // V < 2^31 - 2^20: a column a tile past the row's end still fits
  __device__ __forceinline__ int col(int i) const { return i * T::kElems - off; }
  __device__ __forceinline__ Unit<T> load(int i) const {
    const int c = col(i);
    Unit<T> u;
    if (c >= 0 && c + T::kElems <= V) {
      u.w = ld16(p + c);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < T::kElems; ++j) {
        const uint32_t b = __float_as_uint((c + j >= 0 && c + j < V) ? T::to_f(p[c + j]) : kNegInf);
        if constexpr (T::kElems == 8)
          w[j / 2] = j % 2 ? (w[j / 2] | (b & 0xFFFF0000u)) : b >> 16;
        else
          w[j] = b;
      }
      u.w = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return u;
  }
};

struct RowsArgs {
  const void* x;
  int64_t rows, inner, stride_outer, stride_inner;
  int V;
  const uint8_t* mask;
  float c2;     // log2(e) / temperature
  float inv_t;  // 1 / temperature
};

// Row r as (outer, inner) indices: 32-bit arithmetic, since rows < 2^31, and none for one level.
struct RowIndex {
  int o, i;
  __device__ __forceinline__ RowIndex(const RowsArgs& a, int r) : o(0), i(r) {
    if (a.rows > a.inner) {
      o = static_cast<unsigned>(r) / static_cast<unsigned>(a.inner);
      i = r - o * static_cast<int>(a.inner);
    }
  }
  __device__ __forceinline__ int64_t elem(int64_t stride_outer, int64_t stride_inner) const {
    return o * stride_outer + i * stride_inner;
  }
};

__device__ __forceinline__ int64_t load_id(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// Column of a token: negative tokens count from the end; outside [-V, V): none (-1).
__device__ __forceinline__ int token_col(int64_t t, int V) {
  if (t < 0) t += V;
  return (t >= 0 && t < V) ? static_cast<int>(t) : -1;
}

// Two f32 at once (one issue slot of the FMA pipe for both).
__device__ __forceinline__ uint64_t pk(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpk(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ uint64_t neg2(uint64_t a) { return a ^ 0x8000000080000000ull; }

// ---- running softmax statistics -----------------------------------------------------------------
struct Stat {
  float m, s, t;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
__device__ __forceinline__ float warp_maxn(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = maxn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

// (s, t) moved to the maximum M >= a.m.  -1000: the power is 0, and 0 times the clamped d stays 0
// (an empty part, m = -inf, has s = t = 0).
__device__ __forceinline__ void rescale(Stat& a, float M, float c2) {
  const float d = a.m == kNegInf ? -1000.0f : maxn(__fmul_rn(__fsub_rn(a.m, M), c2), -1000.0f);
  const float f = ex2a(d);
  a.t = __fmul_rn(f, __fmaf_rn(d, a.s, a.t));
  a.s = __fmul_rn(f, a.s);
  a.m = M;
}

// The merge of the lanes' parts, the same in every lane.  A NaN makes s NaN.
__device__ __forceinline__ Stat warp_merge(Stat a, float c2) {
  rescale(a, warp_maxn(a.m), c2);
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  return a;
}

// The maximum of a unit, NaN if one of its elements is.
template <class T>
__device__ __forceinline__ float unit_max(const Unit<T>& u) {
  if constexpr (T::kElems == 8) {
    uint32_t a, b;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(u.w.x), "r"(u.w.y));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(u.w.z), "r"(u.w.w));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
    return maxn(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u));
  } else {
    float v[4];
    unpack<T>(u, v);
    return maxn(maxn(v[0], v[1]), maxn(v[2], v[3]));
  }
}

// A thread's units of one tile into its running statistics; cm is their maximum.
template <class T, bool kEnt>
__device__ __forceinline__ void fold_tile(const Unit<T> (&w)[kUnits], float cm, Stat& a, float c2) {
  if (!(cm <= a.m)) rescale(a, cm, c2);
  const float mz = a.m == kNegInf ? 0.0f : a.m;
  const uint64_t nm = pk(-mz, -mz), c22 = pk(c2, c2);
  uint64_t s = 0, t = 0;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    float v[T::kElems];
    unpack<T>(w[u], v);
#pragma unroll
    for (int j = 0; j < T::kElems; j += 2) {
      float z0, z1;
      uint64_t z = mul2(add2(pk(v[j], v[j + 1]), nm), c22);
      unpk(z, z0, z1);
      if (kEnt) {  // below the smallest f32 the power is 0, and 0 * z has to stay 0 for z = -inf
        z0 = maxn(z0, -160.0f);
        z1 = maxn(z1, -160.0f);
        z = pk(z0, z1);
      }
      const uint64_t e = pk(ex2a(z0), ex2a(z1));
      s = add2(s, e);
      if (kEnt) t = fma2(e, z, t);
    }
  }
  float lo, hi;
  unpk(s, lo, hi);
  a.s = __fadd_rn(a.s, __fadd_rn(lo, hi));
  if (kEnt) {
    unpk(t, lo, hi);
    a.t = __fadd_rn(a.t, __fadd_rn(lo, hi));
  }
}

// ---- the largest k of a row ---------------------------------------------------------------------
// A key orders an element by value (NaN above all, -0 equal to 0) and then by column, lower first:
// the value's bits mapped to an unsigned order, above ib bits of (2^ib - 1 - column).  Keys of a row
// are distinct, so the k largest are one set whatever the order in which they were found.
__device__ __forceinline__ uint32_t value_order(float x) {
  uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));  // one zero
  b ^= static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u;
  return x != x ? 0xFFFFFFFFu : b;
}
template <class T>
__device__ __forceinline__ uint64_t make_key(float x, uint32_t col, int ib) {
  return (static_cast<uint64_t>(value_order(x) >> (32 - T::kKeyBits)) << ib) | (((1ull << ib) - 1ull) - col);
}
template <class T>
__device__ __forceinline__ float key_value(uint64_t key, int ib) {
  uint32_t b = static_cast<uint32_t>(key >> ib) << (32 - T::kKeyBits);
  if (!(b & 0x80000000u) && T::kKeyBits == 16) b |= 0xFFFFu;  // the dropped low half of ~bits
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
}
__device__ __forceinline__ uint32_t key_col(uint64_t key, int ib) {
  return static_cast<uint32_t>(((1ull << ib) - 1ull) - (key & ((1ull << ib) - 1ull)));
}

// The float of a 32-bit order (the value bits of an F32 key).
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
// The upper 16 bits of x's order.
__device__ __forceinline__ uint32_t order16(float x) { return value_order(x) >> 16; }

constexpr int kRegion = 512;  // candidate keys of a warp; at least kMaxTop + the 256 columns of a warp's units
constexpr int kSlots = 32;    // entries per thread of the table of maxima
constexpr int kFinal = 256;   // keys that are put in order by comparing all with all; >= kMaxTop
constexpr int kMaxParts = 8;  // CTAs of a cluster that share a row

// Shared memory for the search, by CTA size: the table (kSlots x kThr orders), the items and the gathered keys, or,
// once those are of no use, a region per warp.
template <int kThr>
struct TopLayout {
  static constexpr int kItems = 4 * kThr;
  static constexpr int kGather = kThr >= 128 ? 1024 : 512;
  static constexpr size_t kTableBytes = sizeof(uint16_t) * kSlots * kThr;
  static constexpr size_t kItemBytes = sizeof(uint32_t) * kItems;
  static constexpr size_t kFast = kTableBytes + kItemBytes + sizeof(uint64_t) * kGather;
  static constexpr size_t kSlow = sizeof(uint64_t) * kRegion * (kThr / 32);
  static constexpr size_t kBytes = kFast > kSlow ? kFast : kSlow;
};

template <int kThr>
struct TopShared {
  uint32_t hist[256];
  uint32_t maxima[kThr];  // order16 of a thread's maximum over the even / odd slots of the table
  uint32_t reached;       // order16 that at least k elements of the CTA's columns reach (0: not known)
  int items, n;        // entries of the item list, gathered keys
  int n_last, pushed;  // keys in `last`, keys brought to the first CTA
  int bin, above, in_bin;
  float m, ls;
  alignas(16) uint64_t last[kFinal];
};

// What the CTAs of a cluster bring to the first one of it.
struct PartsShared {
  Stat stat[kMaxParts];
  int count[kMaxParts];
  uint32_t reached[kMaxParts];
};

// The largest 16-bit order that at least k of the maxima reach, found bit by bit by one warp; 0 where there
// are fewer than k.  Each maximum stands for an element of its own, so k elements reach the result.
template <int kThr>
__device__ __forceinline__ uint32_t reached_by(const uint32_t* maxima, int k) {
  constexpr int kPer = kThr / 32;
  const bool halves = k > kThr / 2;  // two values per thread: closer for a large k
  uint32_t lo[kPer], hi[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t w = maxima[i * 32 + (threadIdx.x & 31)];
    lo[i] = w & 0xFFFFu;
    hi[i] = w >> 16;
    if (!halves) lo[i] = max(lo[i], hi[i]);
  }
  if (k > kThr * (halves ? 2 : 1)) return 0;
  // the bits that all have in common need no counting
  uint32_t mn = lo[0], mx = lo[0];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    mn = min(mn, halves ? min(lo[i], hi[i]) : lo[i]);
    mx = max(mx, halves ? max(lo[i], hi[i]) : lo[i]);
  }
  mn = __reduce_min_sync(0xFFFFFFFFu, mn);
  mx = __reduce_max_sync(0xFFFFFFFFu, mx);
  if (mn == mx) return mx;
  uint32_t bit = 0x80000000u >> __clz(mn ^ mx);
  uint32_t b = mx & ~(2 * bit - 1);
#pragma unroll 1
  for (; bit; bit >>= 1) {
    const uint32_t c = b | bit;
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) cnt += lo[i] >= c;
    if (halves) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) cnt += hi[i] >= c;
    }
    if (__reduce_add_sync(0xFFFFFFFFu, cnt) >= k) b = c;
  }
  return b;
}
// The float just below all of an order16's: two steps, since one step below 0 is the order of -0, which
// compares as 0.  NaN, which nothing is <= to, for 0 and for the order of -inf.
__device__ __forceinline__ float below_order(uint32_t reached) {
  return reached ? order_value((reached << 16) - 2u) : __int_as_float(0x7FC00000);
}

// One warp: leaves the k largest of keys[0, n), n > k, in keys[0, k); returns a bound b with exactly k
// keys >= b.
__device__ __noinline__ uint64_t warp_keep_largest(uint64_t* keys, int n, int k, int bits) {
  const int lane = threadIdx.x & 31;
  uint64_t b = 0;
  for (int bit = bits - 1; bit >= 0; --bit) {
    const uint64_t c = b | (1ull << bit);
    int cnt = 0;
    for (int i = lane; i < n; i += 32) cnt += keys[i] >= c;
    cnt = __reduce_add_sync(0xFFFFFFFFu, cnt);
    if (cnt >= k) b = c;
    if (cnt == k) break;
  }
  int left = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const uint64_t key = i0 + lane < n ? keys[i0 + lane] : 0;
    const bool keep = i0 + lane < n && key >= b;
    const unsigned who = __ballot_sync(0xFFFFFFFFu, keep);  // all of these are read before one is written
    if (keep) keys[left + __popc(who & ((1u << lane) - 1u))] = key;
    left += __popc(who);
    __syncwarp();
  }
  return b;
}

// A bound b with exactly k keys >= b among the warps' lists, which hold more than k: radix selection from
// the key's top bits in digits of eight.  Whole CTA; begins and ends with a barrier.
template <int kThr>
__device__ uint64_t select_bound(const uint64_t* mine, int n_mine, int k, int bits, TopShared<kThr>& sh) {
  const int lane = threadIdx.x & 31;
  uint64_t bound = 0;
  int need = k, shift = bits;
  __syncthreads();
  while (shift > 0) {
    const int w = shift < 8 ? shift : 8;
    const int top = shift;
    shift -= w;
    for (int i = threadIdx.x; i < 256; i += kThr) sh.hist[i] = 0;
    __syncthreads();
    for (int i = lane; i < n_mine; i += 32) {
      const uint64_t key = mine[i];
      if ((key >> top) == (bound >> top)) atomicAdd(&sh.hist[(key >> shift) & ((1u << w) - 1u)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // lane l holds bins 255 - 8 l ... 248 - 8 l, largest first
      const int hi = 255 - 8 * lane;
      int sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += static_cast<int>(sh.hist[hi - j]);
      int pre = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, pre, o);
        if (lane >= o) pre += up;
      }
      int before = pre - sum;
      if (before < need && pre >= need) {  // exactly one lane
        for (int j = 0; j < 8; ++j) {
          const int c = static_cast<int>(sh.hist[hi - j]);
          if (before + c >= need) {
            sh.bin = hi - j;
            sh.above = before;
            sh.in_bin = c;
            break;
          }
          before += c;
        }
      }
    }
    __syncthreads();
    bound |= static_cast<uint64_t>(sh.bin) << shift;
    need -= sh.above;
    const bool whole = sh.in_bin == need;  // the whole bin belongs to the k largest
    __syncthreads();                       // everyone has read the choice before the next digit
    if (whole) break;
  }
  return bound;
}

// Bit j: element j of the unit at columns from c on lies in the row and is not <= thr.
template <class T>
__device__ __forceinline__ unsigned above(const Unit<T>& w, float thr, int c, int V) {
  constexpr int kE = T::kElems;
  float v[kE];
  unpack<T>(w, v);
  unsigned hit = 0;
#pragma unroll
  for (int j = 0; j < kE; ++j) hit |= !(v[j] <= thr) ? 1u << j : 0u;
  if (c < 0) hit &= 0xFFu << min(-c, kE);
  if (c + kE > V) hit &= ((1u << kE) - 1u) >> min(c + kE - V, kE);
  return hit;
}

// A warp's search of a whole row for candidates, for rows with more elements at the bound than fit.  An
// element is a candidate if it is above `thr`, below which k elements of the row lie: either those that
// `reached` vouches for (equal elements included, since those k may stand further right), or k of the
// warp's own earlier columns (equal elements excluded).  A NaN threshold lets everything through.
template <class T>
struct Search {
  uint64_t* keys;  // kRegion
  int n = 0;
  int k, ib;
  float thr;
  __device__ __forceinline__ Search(uint64_t* region, int k_, int ib_, uint32_t reached)
      : keys(region), k(k_), ib(ib_), thr(below_order(reached)) {}
  // unit: the columns from c on for every lane, right of all columns before
  __device__ __forceinline__ void take(const Unit<T>& unit, float mx, int c, int V) {
    unsigned hit = !(mx <= thr) ? above<T>(unit, thr, c, V) : 0;
    unsigned who = __ballot_sync(0xFFFFFFFFu, hit != 0);
    if (who == 0) return;
    if (n > kRegion - 256) {
      const float own = key_value<T>(warp_keep_largest(keys, n, k, T::kKeyBits + ib), ib);
      n = k;
      thr = fmaxf(thr, own);  // the one that is not NaN
    }
    const int lane = threadIdx.x & 31;
    do {
      if (hit) {
        const int j = __ffs(hit) - 1;
        hit &= hit - 1;
        const float x = pick<T>(unit, j);
        keys[n + __popc(who & ((1u << lane) - 1u))] = make_key<T>(x, static_cast<uint32_t>(c + j), ib);
      }
      n += __popc(who);
      who = __ballot_sync(0xFFFFFFFFu, hit != 0);
    } while (who);
    __syncwarp();
  }
};

// ---- forward ------------------------------------------------------------------------------------
struct StatArgs {
  RowsArgs r;
  int part_bits;  // log2 of the CTAs that share a row
  // token_logprobs
  const void* tokens;  // may be null
  int token_bytes;
  int k;
  int ib;   // column bits of a key
  int cap;  // keys that a CTA brings to the first one of its cluster
  float* logprob;
  float* entropy;
  float* top_lp;
  int64_t* top_id;
  // distillation
  const void* ids;
  int id_bytes;
  const void* teacher;
  int teacher_f32;
  int K;
  float* loss;
  // [rows][4]: m, log2 s, then the entropy, or the teacher's m and log2 s
  float4* stats;
};

__device__ __forceinline__ float teacher_val(const StatArgs& a, int64_t i) {
  return a.teacher_f32 ? static_cast<const float*>(a.teacher)[i]
                       : Bf16::to_f(static_cast<const uint16_t*>(a.teacher)[i]);
}
// A teacher entry: its column's logit (NaN: an id past the last column) and the teacher's value there.
struct Entry {
  bool has;
  float t, x;
};
template <class T>
__device__ __forceinline__ Entry teacher_entry(const StatArgs& a, int64_t e, const Row<T>& x) {
  const int64_t id = load_id(a.ids, a.id_bytes, e);
  Entry r{id >= 0, kNegInf, __int_as_float(0x7FC00000)};
  if (r.has) r.t = teacher_val(a, e);
  if (r.has && id < a.r.V) r.x = T::to_f(x.p[id]);
  return r;
}

// One warp: the row's loss sum_j q_j (log q_j - log p_{id_j}) over the entries with id >= 0, and the
// teacher's (max, log2 sum).  Entries whose teacher value is -inf have q = 0 and contribute 0; a row
// without any weight has loss 0 (and max -inf, which the gradient reads as "no entry").  The first 64
// entries come loaded.
template <class T>
__device__ __forceinline__ float distill_row(const StatArgs& a, int64_t base, const Row<T>& x, const Entry (&first)[2],
                                             float m, float ls, float* tm_out, float* tl_out) {
  const int lane = threadIdx.x & 31;
  const float c2 = a.r.c2;
  float tm = maxn(first[0].t, first[1].t);
  for (int j = 64 + lane; j < a.K; j += 32)
    if (load_id(a.ids, a.id_bytes, base + j) >= 0) tm = maxn(tm, teacher_val(a, base + j));
  tm = warp_maxn(tm);
  *tm_out = tm;
  *tl_out = 0.0f;
  if (tm == kNegInf) return 0.0f;
  float ts = 0.0f;
  for (int k = 0; k < 2; ++k)
    if (first[k].has) ts = __fadd_rn(ts, ex2a(__fmul_rn(__fsub_rn(first[k].t, tm), c2)));
  for (int j = 64 + lane; j < a.K; j += 32)
    if (load_id(a.ids, a.id_bytes, base + j) >= 0)
      ts = __fadd_rn(ts, ex2a(__fmul_rn(__fsub_rn(teacher_val(a, base + j), tm), c2)));
  ts = warp_sum(ts);
  const float tl = log2f(ts), tls = logf(ts);
  *tl_out = tl;
  float sum = 0.0f;
  auto add = [&](const Entry& e) {
    const float td = __fsub_rn(e.t, tm);
    const float q = ex2a(__fmaf_rn(td, c2, -tl));
    if (!e.has || q == 0.0f) return;
    const float lp = __fmaf_rn(__fsub_rn(e.x, m), a.r.inv_t, -ls);
    sum = __fmaf_rn(q, __fsub_rn(__fmaf_rn(td, a.r.inv_t, -tls), lp), sum);
  };
  add(first[0]);
  add(first[1]);
  for (int j = 64 + lane; j < a.K; j += 32) add(teacher_entry(a, base + j, x));
  return warp_sum(sum);
}

// What a statistics kernel computes besides (m, s).
enum Mode { kPlain = 0, kEntropy = 1, kTopK = 2, kTeacher = 3 };  // kTopK: with the entropy

template <class T, int kThr>
__device__ __forceinline__ void load_tile(const Row<T>& x, int u0, int u_end, Unit<T> (&w)[kUnits]) {
  const int tid = threadIdx.x;
  constexpr int kTile = kThr * kUnits;
  if (u0 + kTile <= u_end && x.col(u0) >= 0 && x.col(u0 + kTile) <= x.V) {
    const uint4* p = reinterpret_cast<const uint4*>(x.p + x.col(u0)) + tid;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) w[u].w = ld16(p + u * kThr);
  } else {
    constexpr uint32_t kFill = T::kElems == 8 ? 0xFF80FF80u : 0xFF800000u;  // -inf
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int i = u0 + u * kThr + tid;
      if (i < u_end)
        w[u] = x.load(i);
      else
        w[u].w = make_uint4(kFill, kFill, kFill, kFill);
    }
  }
}

// The warp's candidates among the CTA's units [u_begin, u_end), into its region; returns their number.
template <class T, int kThr>
__device__ __noinline__ int search_row(const Row<T>& x, int u_begin, int u_end, int k, int ib, uint32_t reached,
                                       uint64_t* region) {
  Search<T> top(region, k, ib, reached);
  for (int u0 = u_begin; u0 < u_end; u0 += kThr * kUnits) {
    Unit<T> w[kUnits];
    load_tile<T, kThr>(x, u0, u_end, w);
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      top.take(w[u], unit_max<T>(w[u]), x.col(u0 + u * kThr + threadIdx.x), x.V);
  }
  return top.n;
}

// (Keeping candidates while the row streams took 549 us at 4096 x 128256 with 64 alternatives: early bounds are loose,
// and most warps met a candidate in most tiles.  The table costs the stream one 16-bit store per thread and tile.)
// The k largest of the CTA's units [u_begin, u_end), and a few more, as keys: this warp's list (*mine, *n_mine);
// returns the number of all warps.  *all: the lists one after another (null: they are apart).  `reached` is a
// bound that k of the elements reach, `best` the thread's maximum.  The table says which thread and which
// tiles saw a maximum that reaches it; those (little more than k) are read once more, each unit by one
// thread.  Where too many elements equal the bound (a constant row, say), the row is searched as a whole.
template <class T, int kThr>
__device__ __forceinline__ int find_top(const Row<T>& x, int u_begin, int u_end, int per_slot, int slots, uint32_t best,
                                        int k, int ib, char* mem, TopShared<kThr>& sh, const uint64_t** mine,
                                        int* n_mine, const uint64_t** all) {
  using L = TopLayout<kThr>;
  constexpr int kTile = kThr * kUnits;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint16_t* table = reinterpret_cast<const uint16_t*>(mem);
  uint32_t* items = reinterpret_cast<uint32_t*>(mem + L::kTableBytes);
  uint64_t* gather = reinterpret_cast<uint64_t*>(mem + L::kTableBytes + L::kItemBytes);
  const uint32_t reached = sh.reached;
  const float thr = below_order(reached);
  if (__any_sync(0xFFFFFFFFu, best >= reached)) {
    unsigned hits = 0;  // the lane's slots; kSlots <= 32
#pragma unroll 4
    for (int slot = 0; slot < slots; ++slot)
      hits |= table[slot * kThr + tid] >= reached ? 1u << slot : 0u;
    const int mine_n = __popc(hits);
    int before = mine_n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, before, o);
      if (lane >= o) before += up;
    }
    int at = 0;
    if (lane == 31) at = atomicAdd(&sh.items, before);
    at = __shfl_sync(0xFFFFFFFFu, at, 31) + before - mine_n;
    for (; hits; hits &= hits - 1, ++at)
      if (at < L::kItems) items[at] = static_cast<uint32_t>((__ffs(hits) - 1) << 16 | tid);
  }
  __syncthreads();
  const int m = sh.items;
  if (m <= L::kItems) {
    constexpr int kFlight = 2;  // units per thread whose loads are in flight together
#pragma unroll 1
    for (int q0 = tid; q0 < m * kUnits; q0 += kFlight * kThr) {
#pragma unroll 1
      for (int tile = 0; tile < per_slot; ++tile) {
        Unit<T> w[kFlight];
        int i[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
          const int q = q0 + f * kThr;
          i[f] = u_end;
          if (q < m * kUnits) {
            const uint32_t item = items[q / kUnits];
            i[f] = u_begin + (static_cast<int>(item >> 16) * per_slot + tile) * kTile + q % kUnits * kThr +
                   (item & 0xFFFFu);
            if (i[f] < u_end) w[f] = x.load(i[f]);
          }
        }
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
          if (i[f] >= u_end) continue;
          for (unsigned hit = above<T>(w[f], thr, x.col(i[f]), x.V); hit; hit &= hit - 1) {
            const int j = __ffs(hit) - 1;
            const int at = atomicAdd(&sh.n, 1);
            if (at < L::kGather) gather[at] = make_key<T>(pick<T>(w[f], j), static_cast<uint32_t>(x.col(i[f]) + j), ib);
          }
        }
      }
    }
  }
  __syncthreads();
  const int n = sh.n;
  if (m <= L::kItems && n <= L::kGather) {
    const int per = (n + kThr / 32 - 1) / (kThr / 32);
    *mine = gather + warp * per;
    *n_mine = max(0, min(per, n - warp * per));
    *all = gather;
    return n;
  }
  *all = nullptr;
  __syncthreads();  // the table, the items and the gathered keys give way to the regions
  uint64_t* region = reinterpret_cast<uint64_t*>(mem) + warp * kRegion;
  *mine = region;
  *n_mine = search_row<T, kThr>(x, u_begin, u_end, k, ib, reached, region);
  if (tid == 0) sh.n = 0;
  __syncthreads();
  if ((tid & 31) == 0) atomicAdd(&sh.n, *n_mine);
  __syncthreads();
  return sh.n;
}

// Those >= bound of the n keys in the warps' lists (k of them at least), cut to exactly k if there are more than
// `most` (>= k), into sh.last in any order; returns their number.  sh.n_last is 0 before.  Whole CTA; ends with a
// barrier.
template <int kThr>
__device__ __forceinline__ int collect(const uint64_t* mine, int n_mine, int n, int k, int most, uint64_t bound,
                                       int bits, TopShared<kThr>& sh) {
  const int lane = threadIdx.x & 31;
  if (n > most && bound) {
    int c = 0;
    for (int i = lane; i < n_mine; i += 32) c += mine[i] >= bound;
    c = __reduce_add_sync(0xFFFFFFFFu, c);
    if (lane == 0) atomicAdd(&sh.n_last, c);
    __syncthreads();
    n = sh.n_last;
    __syncthreads();
    if (threadIdx.x == 0) sh.n_last = 0;
    __syncthreads();
  }
  if (n > most) bound = select_bound<kThr>(mine, n_mine, k, bits, sh);
  for (int i = lane; i < n_mine; i += 32)
    if (mine[i] >= bound) sh.last[atomicAdd(&sh.n_last, 1)] = mine[i];
  __syncthreads();
  return sh.n_last;
}

// One CTA per row, or a cluster of 2 to 8 that share a row's units and bring their parts to the first of them.
// kAhead: tiles whose loads are in flight together, 2 where few CTAs run.  Resident CTAs, measured at 4096 x 128256
// (2048 x 50257 in f32): without alternatives 6 per SM; with 64 of them 5 (bf16; 4: 227 us, 5: 216 us) or 4 (f32).
constexpr int min_ctas(bool top, bool f32, int threads, int ahead) {
  return (ahead > 1 ? 2 : !top ? 6 : f32 || threads < 256 ? 4 : 5) * 256 / threads;
}
template <class T, int kThr, int kMode, int kAhead>
__global__ void __launch_bounds__(kThr, min_ctas(kMode == kTopK, T::kKeyBits > 16, kThr, kAhead))
    rowstat_kernel(const StatArgs a) {
  constexpr bool kEnt = kMode == kEntropy || kMode == kTopK;
  constexpr bool kTop = kMode == kTopK;
  constexpr int kNWarps = kThr / 32;
  constexpr int kTile = kThr * kUnits;  // units of a tile
  extern __shared__ __align__(16) char mem[];  // kTop: TopLayout, then the keys of the cluster's CTAs
  __shared__ Stat sh_stat[kNWarps];
  __shared__ PartsShared parts;
  __shared__ TopShared<kTop ? kThr : 32> sh;
  const int row = blockIdx.x >> a.part_bits, n_parts = 1 << a.part_bits;
  const int part = blockIdx.x & (n_parts - 1);
  const int tid = threadIdx.x, warp = tid >> 5;
  const float c2 = a.r.c2;

  if (a.r.mask && a.r.mask[row] == 0) {  // nothing of the row is read
    if (part > 0) return;
    if (tid == 0) {
      if (a.logprob) a.logprob[row] = 0.0f;
      if (a.entropy) a.entropy[row] = 0.0f;
      if (kMode == kTeacher) a.loss[row] = 0.0f;
      if (a.stats) a.stats[row] = make_float4(kNegInf, 0.0f, kMode == kTeacher ? kNegInf : 0.0f, 0.0f);
    }
    if constexpr (kTop)
      for (int j = tid; j < a.k; j += kThr) {
        a.top_lp[static_cast<int64_t>(row) * a.k + j] = kNegInf;
        a.top_id[static_cast<int64_t>(row) * a.k + j] = -1;
      }
    return;
  }
  namespace cg = cooperative_groups;
  if (n_parts > 1) cg::this_cluster().barrier_arrive();  // "started", awaited before the others' memory is used

  const Row<T> x(a.r.x, RowIndex(a.r, row).elem(a.r.stride_outer, a.r.stride_inner), a.r.V);
  // This CTA's units; parts begin at a multiple of 8 units (128 bytes).
  const int per_part = n_parts == 1 ? x.units : (((x.units + n_parts - 1) >> a.part_bits) + 7) & ~7;
  const int u_begin = min(part * per_part, x.units), u_end = min(u_begin + per_part, x.units);

  // The few logits that the row's results need by column, before the stream.
  float x_tok = __int_as_float(0x7FC00000);
  Entry entry[2];
  if constexpr (kMode == kTeacher) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      entry[k].has = false;
      entry[k].t = kNegInf;
      if (part == 0 && tid < 32 && k * 32 + tid < a.K)
        entry[k] = teacher_entry(a, static_cast<int64_t>(row) * a.K + k * 32 + tid, x);
    }
  } else if (part == 0 && tid == 0 && a.logprob) {
    const int col = token_col(load_id(a.tokens, a.token_bytes, row), a.r.V);
    if (col >= 0) x_tok = T::to_f(x.p[col]);
  }

  Stat st{kNegInf, 0.0f, 0.0f};
  // kTop: the table of maxima, a slot for every per_slot tiles
  uint16_t* table = reinterpret_cast<uint16_t*>(mem);
  const int tiles = (u_end - u_begin + kTile - 1) / kTile;
  const int per_slot = (tiles + kSlots - 1) / kSlots;
  int slot = 0, in_slot = 0;
  uint32_t best[2] = {0, 0}, order = 0;

  if (kTop && tid == 0) sh.items = sh.n = sh.n_last = sh.pushed = 0;

  for (int first = u_begin; first < u_end; first += kAhead * kTile) {
    Unit<T> w[kAhead][kUnits];
#pragma unroll
    for (int h = 0; h < kAhead; ++h)
      if (h == 0 || first + h * kTile < u_end) load_tile<T, kThr>(x, first + h * kTile, u_end, w[h]);
#pragma unroll
    for (int h = 0; h < kAhead; ++h) {
      const int u0 = first + h * kTile;
      if (h > 0 && u0 >= u_end) break;
      float cm = unit_max<T>(w[h][0]);
#pragma unroll
      for (int u = 1; u < kUnits; ++u) cm = maxn(cm, unit_max<T>(w[h][u]));
      fold_tile<T, kEnt>(w[h], cm, st, c2);
      if constexpr (kTop) {
        order = max(order, order16(cm));
        if (++in_slot == per_slot || u0 + kTile >= u_end) {
          table[slot * kThr + tid] = static_cast<uint16_t>(order);
          if (slot & 1)
            best[1] = max(best[1], order);
          else
            best[0] = max(best[0], order);
          ++slot;
          in_slot = 0;
          order = 0;
        }
      }
    }
  }

  st = warp_merge(st, c2);
  if ((tid & 31) == 0) sh_stat[warp] = st;
  if constexpr (kTop) sh.maxima[tid] = best[0] | best[1] << 16;
  __syncthreads();
  if (warp == 0) {
    st = tid < kNWarps ? sh_stat[tid] : Stat{kNegInf, 0.0f, 0.0f};
    st = warp_merge(st, c2);
  }
  const uint64_t *mine = nullptr, *all = nullptr;
  int n_mine = 0, n = 0;
  const int bits = T::kKeyBits + a.ib;
  uint64_t bound = 0;
  if constexpr (kTop) {
    if (warp == 1) {
      const uint32_t r = reached_by<kThr>(sh.maxima, a.k);
      if ((tid & 31) == 0) sh.reached = r;
    }
    __syncthreads();
    n = find_top<T, kThr>(x, u_begin, u_end, per_slot, slot, max(best[0], best[1]), a.k, a.ib, mem, sh, &mine, &n_mine,
                          &all);
  }

  if (n_parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    uint64_t* part_keys = reinterpret_cast<uint64_t*>(mem + TopLayout<kThr>::kBytes);  // [n_parts][cap]
    if constexpr (kTop) {
      if (n > a.cap) {
        n = collect<kThr>(mine, n_mine, n, a.k, a.k, 0, bits, sh);
        const int per = (n + kNWarps - 1) / kNWarps;
        mine = sh.last + warp * per;
        n_mine = max(0, min(per, n - warp * per));
        __syncthreads();
        if (tid == 0) sh.n_last = 0;
      }
    }
    cluster.barrier_wait();
    if constexpr (kTop) {
      uint64_t* to = cluster.map_shared_rank(part_keys + part * a.cap, 0);
      for (int i = tid & 31; i < n_mine; i += 32) to[atomicAdd(&sh.pushed, 1)] = mine[i];
    }
    if (tid == 0) {
      PartsShared* to = cluster.map_shared_rank(&parts, 0);
      to->stat[part] = st;
      to->count[part] = n;
      if constexpr (kTop) to->reached[part] = sh.reached;
    }
    cluster.sync();
    if (part > 0) return;
    if (warp == 0) {
      st = tid < n_parts ? parts.stat[tid] : Stat{kNegInf, 0.0f, 0.0f};
      st = warp_merge(st, c2);
    }
    if constexpr (kTop) {
      static_assert(kNWarps >= kMaxParts || kThr < 256, "a warp takes a part's keys");
      mine = part_keys + warp * a.cap;
      n_mine = warp < n_parts ? parts.count[warp] : 0;
      n = 0;
      uint32_t reached = 0;  // k elements of one part reach its bound, so the row's k largest do
      for (int i = 0; i < n_parts; ++i) {
        n += parts.count[i];
        reached = max(reached, parts.reached[i]);
      }
      bound = static_cast<uint64_t>(reached) << (bits - 16);
    }
  }

  if (warp == 0) {
    const float l2 = log2f(st.s), ls = logf(st.s);
    if constexpr (kMode == kTeacher) {
      float tm, tl;
      const float loss = distill_row<T>(a, static_cast<int64_t>(row) * a.K, x, entry, st.m, ls, &tm, &tl);
      if (tid == 0) {
        a.loss[row] = loss;
        if (a.stats) a.stats[row] = make_float4(st.m, l2, tm, tl);
      }
    } else if (tid == 0) {
      const float H = kEnt ? __fmul_rn(kLn2, __fsub_rn(l2, __fdiv_rn(st.t, st.s))) : 0.0f;
      if (a.logprob) a.logprob[row] = __fmaf_rn(__fsub_rn(x_tok, st.m), a.r.inv_t, -ls);
      if (a.entropy) a.entropy[row] = H;
      if (a.stats) a.stats[row] = make_float4(st.m, l2, H, 0.0f);
      sh.m = st.m;
      sh.ls = ls;
    }
  }
  if constexpr (kTop) {
    // V >= k: there are k keys at least.  One CTA's keys, if they are not many, are compared where they are.
    const uint64_t* last = all;
    if (n_parts > 1 || n > kFinal || all == nullptr) {
      n = collect<kThr>(mine, n_mine, n, a.k, kFinal, bound, bits, sh);
      last = sh.last;
    } else {
      __syncthreads();  // sh.m, sh.ls
    }
    const float m = sh.m, ls = sh.ls;
    int group = 1;  // threads that share the comparisons of a key
    while (group < 8 && 2 * group * n <= kThr) group *= 2;
    for (int i0 = 0; i0 < n; i0 += kThr / group) {
      const int i = i0 + tid / group;
      const uint64_t key = i < n ? last[i] : ~0ull;
      int rank = 0;
#pragma unroll 4
      for (int j = 2 * (tid % group); j < n; j += 2 * group) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(last + j);
        rank += (two.x > key) + (j + 1 < n && two.y > key);
      }
      for (int o = 1; o < group; o <<= 1) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, o);
      if (i < n && tid % group == 0 && rank < a.k) {
        const uint32_t col = key_col(key, a.ib);
        const float xv = T::kKeyBits == 16 ? key_value<T>(key, a.ib) : T::to_f(x.p[col]);
        a.top_lp[static_cast<int64_t>(row) * a.k + rank] = __fmaf_rn(__fsub_rn(xv, m), a.r.inv_t, -ls);
        a.top_id[static_cast<int64_t>(row) * a.k + rank] = col;
      }
    }
  }
}

// ---- backward -----------------------------------------------------------------------------------
struct GradArgs {
  RowsArgs r;
  const float4* stats;
  // token_logprobs: upstream gradients (null: none) with a stride per row (0: one value for all)
  const void* tokens;
  int token_bytes;
  const float* dlogprob;
  int64_t dlogprob_stride;
  const float* dentropy;
  int64_t dentropy_stride;
  const float* dtop;  // [rows][k] contiguous
  const int64_t* top_id;
  int k;
  // distillation
  const void* ids;
  int id_bytes;
  const void* teacher;
  int teacher_f32;
  int K;
  const float* dloss;
  int64_t dloss_stride;
  // fp8 output (an output head's logits): its format, whether *amax is the largest |output| (else a bound of
  // it), 1 / cap of logits that are cap * tanh(.) (0: not capped), and 1 / scale
  int fmt;
  int exact;
  float inv_cap;
  float* amax;
  float* inv_scale;
  void* out;
  int64_t out_outer, out_inner;  // row strides of the output
  int tasks;     // tasks of a row
  int per_task;  // chunks of a task
};

// Entry j < n of a row: its column (-1: none) and the value that its weight comes from.
template <bool kDistill>
__device__ __forceinline__ void load_entry(const GradArgs& a, int64_t row, int j, int* id, float* val) {
  if constexpr (kDistill) {
    const int64_t e = row * a.K + j;
    const int64_t i = load_id(a.ids, a.id_bytes, e);
    *id = (i >= 0 && i < a.r.V) ? static_cast<int>(i) : -1;
    *val = a.teacher_f32 ? static_cast<const float*>(a.teacher)[e]
                         : Bf16::to_f(static_cast<const uint16_t*>(a.teacher)[e]);
  } else if (a.dlogprob && j == 0) {
    *id = token_col(load_id(a.tokens, a.token_bytes, row), a.r.V);
    *val = a.dlogprob[row * a.dlogprob_stride];
  } else {
    const int64_t e = row * a.k + j - (a.dlogprob ? 1 : 0);
    *id = static_cast<int>(a.top_id[e]);
    *val = a.dtop[e];
  }
}

// The largest |dlogits| that the rows' results allow, and the fp8 scale from it: |p - [label]|, |p - q| and the
// derivative of the soft cap are at most 1, and p |log p + H| <= 1 / e + H.  The gradient itself can be thousands
// of times smaller (an entropy bonus on flat rows, a student close to its teacher).  e5m2 covers that: an element
// keeps its precision down to 2^-29.8 of the bound (2^-14 / 57344) and is lost below 2^-32.8, in sum at most 2^-15.8
// of it in a row of 131072 columns.  e4m3 does not (2^-14.8 and 2^-18.8 of the bound; V 128256, normal logits,
// entropy alone: 97 % of the elements flushed to 0); it goes with the measured amax (a.exact).  A NaN is above all.
// One CTA, a thread per row: below 10 us at 16384 rows, but 2.3 ms with gradients of 256 alternatives each, whose
// sums a thread reads alone.
template <bool kDistill>
__global__ void __launch_bounds__(1024) rowamax_kernel(const GradArgs a) {
  uint32_t top = 0;
  for (int64_t r = threadIdx.x; r < a.r.rows; r += 1024) {
    const float4 st = a.stats[r];
    if ((a.r.mask && a.r.mask[r] == 0) || (kDistill && st.z == kNegInf)) continue;
    float v;
    if constexpr (kDistill) {
      v = fabsf(a.dloss[r * a.dloss_stride]);
    } else {
      v = a.dlogprob ? fabsf(a.dlogprob[r * a.dlogprob_stride]) : 0.0f;
      if (a.dentropy) v = __fmaf_rn(fabsf(a.dentropy[r * a.dentropy_stride]), __fadd_rn(0.368f, fabsf(st.z)), v);
      if (a.dtop)
        for (int j = 0; j < a.k; ++j) v = __fadd_rn(v, fabsf(a.dtop[r * a.k + j]));
    }
    top = max(top, __float_as_uint(__fmul_rn(v, a.r.inv_t)) & 0x7FFFFFFFu);
  }
  __shared__ uint32_t part[32];
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x < 32) {
    top = __reduce_max_sync(0xFFFFFFFFu, part[threadIdx.x]);
    if (threadIdx.x == 0) {
      const float amax = __uint_as_float(top);
      *a.amax = amax;
      *a.inv_scale = __fdiv_rn(1.0f, scale_from_amax(amax, a.fmt));
    }
  }
}

// Eight values of at most the format's largest (up to rounding) as fp8.  One finiteness test of their sum decides
// whether the codes of NaN and infinities are needed.
__device__ __forceinline__ uint2 to_fp8(const float (&v)[8], int fmt) {
  const float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  const __nv_fp8_interpretation_t kind = fmt == UFP8_E4M3 ? __NV_E4M3 : __NV_E5M2;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = isfinite(sum) ? static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]),
                                                                          __NV_SATFINITE, kind))
                         : cvt2(v[2 * i], v[2 * i + 1], fmt);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// The warps of a resident grid walk (row, task) units on their own, without a barrier (with one step per CTA all
// waited for the warp that sorted the entries in: 458 us at 4096 x 128256 with 64 of them, 336-347 so); a task is
// `per_task` chunks of a row, a chunk 2 KB of it, kUnits 16-byte loads a lane.  Per task the warp works out the row
// factors; per chunk it adds the weights of the row's entries that fall into it into `wt`, one f32 per
// column and zero elsewhere, in entry order, so that the result does not depend on timing.  Then
// v = p * factor + weight, and a lane with a weight in its columns sets those back to zero.
// kFp8: the logits are an output head's (bf16): the soft cap's derivative, and fp8 output by the scale of
// rowamax_kernel, or, with a.exact, of the kAmax pass before this one: the same arithmetic on the same logits, which
// keeps the largest |v| instead of storing.  The scale then multiplies the finished value, so that none of them
// exceeds the format's largest; with the bound it goes into the factors.
enum GradOut { kLike = 0, kFp8 = 1, kAmax = 2 };
template <class T, bool kDistill, int kOut>
__global__ void __launch_bounds__(kThreads, 4) rowgrad_kernel(const GradArgs a) {
  constexpr int kChunk = 32 * kUnits;  // units of a chunk
  constexpr int kE = T::kElems;
  constexpr bool kHead = kOut != kLike;
  extern __shared__ float4 wt_all[];    // kWarps * kChunk * kE floats
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float4* wt4 = wt_all + warp * kChunk * (kE / 4);
  float* wt = reinterpret_cast<float*>(wt4);
  // unit wi = (row, task) = (wi / tasks, wi % tasks), advanced by the grid's warps without divisions
  const int rows = static_cast<int>(a.r.rows);
  const unsigned first = blockIdx.x * kWarps + warp, step = gridDim.x * kWarps;
  const int step_r = static_cast<int>(step / a.tasks), step_t = static_cast<int>(step % a.tasks);
  int row = static_cast<int>(first / a.tasks), task = static_cast<int>(first % a.tasks);
  const uint64_t c22 = pk(a.r.c2, a.r.c2), cap2 = pk(a.inv_cap, a.inv_cap);
  const float scale = kOut == kFp8 ? scale_from_amax(*a.amax, a.fmt) : 1.0f;
  const bool late = kOut == kFp8 && a.exact;
  const float sc = late ? 1.0f : scale;
  if (late && blockIdx.x == 0 && threadIdx.x == 0) *a.inv_scale = __fdiv_rn(1.0f, scale);
  const uint64_t late2 = pk(scale, scale);
  float largest = 0.0f;  // kAmax: |v| so far, NaN once one is
  const int n = kDistill ? a.K : (a.dlogprob ? 1 : 0) + (a.dtop ? a.k : 0);
  if (n > 0)
    for (int i = lane; i < kChunk * (kE / 4); i += 32) wt4[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __syncwarp();
  for (; row < rows; row += step_r, task += step_t) {
    if (task >= a.tasks) {
      task -= a.tasks;
      if (++row >= rows) break;
    }
    const RowIndex ri(a.r, row);
    const Row<T> x(a.r.x, ri.elem(a.r.stride_outer, a.r.stride_inner), a.r.V);
    using Out = std::conditional_t<kHead, uint8_t, typename T::raw>;
    Out* o = static_cast<Out*>(a.out) + ri.elem(a.out_outer, a.out_inner);
    // the units' first elements lie on multiples of a unit in the output, too
    const bool vec = kOut == kAmax || ((reinterpret_cast<uintptr_t>(o) - x.off * sizeof(Out)) & (kE * sizeof(Out) - 1)) == 0;
    const float4 st = a.stats[row];
    const bool dead = (a.r.mask && a.r.mask[row] == 0) || (kDistill && st.z == kNegInf);
    int u0 = task * a.per_task * kChunk;
    const int u_end = min(u0 + a.per_task * kChunk, x.units);
    float A = 0.0f, B = 0.0f;
    int id0[2] = {-1, -1};  // the first 64 entries stay with their lanes
    float val0[2] = {0.0f, 0.0f};
    if (!dead) {
      if (lane < n) load_entry<kDistill>(a, row, lane, &id0[0], &val0[0]);
      if (32 + lane < n) load_entry<kDistill>(a, row, 32 + lane, &id0[1], &val0[1]);
      if constexpr (kDistill) {
        A = __fmul_rn(a.dloss[row * a.dloss_stride], a.r.inv_t);
      } else {
        const float g = a.dlogprob ? __fmul_rn(a.dlogprob[row * a.dlogprob_stride], a.r.inv_t) : 0.0f;
        const float h = a.dentropy ? __fmul_rn(a.dentropy[row * a.dentropy_stride], a.r.inv_t) : 0.0f;
        float top = 0.0f;
        if (a.dtop) {
          for (int j = lane; j < a.k; j += 32)
            top = __fmaf_rn(a.dtop[static_cast<int64_t>(row) * a.k + j], a.r.inv_t, top);
          top = warp_sum(top);
        }
        A = -__fmaf_rn(h, st.z, __fadd_rn(g, top));
        B = __fmul_rn(-h, kLn2);
      }
      if (kHead) {
        A = __fmul_rn(A, sc);
        B = __fmul_rn(B, sc);
      }
    }
    const uint64_t nm = pk(-st.x, -st.x), nl = pk(-st.y, -st.y);
    const uint64_t A2 = pk(A, A), B2 = pk(B, B);
    for (; u0 < u_end; u0 += kChunk) {
      const int lo = x.col(u0), hi = x.col(u0 + kChunk);
      const bool whole = lo >= 0 && hi <= x.V && vec;  // every unit is 16-byte loads and stores
      Unit<T> w[kUnits];
      unsigned flag = 0;  // bit u: unit u of this lane holds a weight
      if (!dead) {
        if (whole) {
          const uint4* p = reinterpret_cast<const uint4*>(x.p + lo) + lane;
#pragma unroll
          for (int u = 0; u < kUnits; ++u) w[u].w = ld16(p + u * 32);
        } else {
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
            const int i = u0 + u * 32 + lane;
            if (i < x.units) w[u] = x.load(i);
          }
        }
        for (int j0 = 0; j0 < n; j0 += 32) {
          int id = j0 == 0 ? id0[0] : id0[1];
          float val = j0 == 0 ? val0[0] : val0[1];
          if (j0 > 32) {
            id = -1;
            if (j0 + lane < n) load_entry<kDistill>(a, row, j0 + lane, &id, &val);
          }
          const bool in = id >= 0 && id >= lo && id < hi;
          const unsigned active = __ballot_sync(0xFFFFFFFFu, in);
          if (active == 0) continue;
          const float ew = kDistill ? __fmul_rn(-A, ex2a(__fmaf_rn(__fsub_rn(val, st.z), a.r.c2, -st.w)))
                                    : __fmul_rn(__fmul_rn(val, a.r.inv_t), sc);
          const int at = id - lo;
          for (unsigned left = active; left; left &= left - 1) {  // in entry order
            const int src = __ffs(left) - 1;
            const int sat = __shfl_sync(0xFFFFFFFFu, at, src);
            const float sw = __shfl_sync(0xFFFFFFFFu, ew, src);
            if (lane == (sat / kE & 31)) {  // the lane that owns the column
              wt[sat] = __fadd_rn(wt[sat], sw);
              flag |= 1u << (sat / (32 * kE));
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int i = u0 + u * 32 + lane;
        if (!whole && i >= x.units) continue;
        float g[kE];
        if (dead) {
#pragma unroll
          for (int j = 0; j < kE; ++j) g[j] = 0.0f;
        } else {
          float v[kE];
          unpack<T>(w[u], v);
#pragma unroll
          for (int j = 0; j < kE; j += 2) {
            // log2 p; below -160 the power is 0 and 0 * log2 p has to stay 0
            float z0, z1;
            unpk(fma2(add2(pk(v[j], v[j + 1]), nm), c22, nl), z0, z1);
            if (!kDistill) {
              z0 = maxn(z0, -160.0f);
              z1 = maxn(z1, -160.0f);
            }
            const uint64_t f = kDistill ? A2 : fma2(B2, pk(z0, z1), A2);
            unpk(mul2(pk(ex2a(z0), ex2a(z1)), f), g[j], g[j + 1]);
          }
          if ((flag >> u) & 1u) {
            float4* q = wt4 + (u * 32 + lane) * (kE / 4);
#pragma unroll
            for (int j = 0; j < kE; j += 4) {
              const float4 f = q[j / 4];
              g[j] = __fadd_rn(g[j], f.x);
              g[j + 1] = __fadd_rn(g[j + 1], f.y);
              g[j + 2] = __fadd_rn(g[j + 2], f.z);
              g[j + 3] = __fadd_rn(g[j + 3], f.w);
              q[j / 4] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
          }
          if (kHead && a.inv_cap > 0.0f) {
#pragma unroll
            for (int j = 0; j < kE; j += 2) {
              const uint64_t t = mul2(pk(v[j], v[j + 1]), cap2);  // times tanh' = 1 - (x / cap)^2
              unpk(mul2(pk(g[j], g[j + 1]), fma2(t, neg2(t), pk(1.0f, 1.0f))), g[j], g[j + 1]);
            }
          }
        }
        const int c = x.col(i);
        if constexpr (kOut == kAmax) {
          if (whole) {
#pragma unroll
            for (int j = 0; j < kE; ++j) largest = maxn(largest, fabsf(g[j]));
          } else {
#pragma unroll
            for (int j = 0; j < kE; ++j)
              if (c + j >= 0 && c + j < x.V) largest = maxn(largest, fabsf(g[j]));
          }
          continue;
        }
        if (late) {
#pragma unroll
          for (int j = 0; j < kE; j += 2) unpk(mul2(pk(g[j], g[j + 1]), late2), g[j], g[j + 1]);
        }
        // streaming stores: 4 % faster at 212 MB of gradient, 1 % at 1 GB
        if (whole || (vec && c >= 0 && c + kE <= x.V)) {
          if constexpr (kHead) {
            __stcs(reinterpret_cast<uint2*>(o + c), to_fp8(g, a.fmt));
          } else {
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if constexpr (kE == 8) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(g[2 * j], g[2 * j + 1]);
                q[j] = *reinterpret_cast<const uint32_t*>(&b);
              } else {
                q[j] = __float_as_uint(g[j]);
              }
            }
            __stcs(reinterpret_cast<uint4*>(o + c), make_uint4(q[0], q[1], q[2], q[3]));
          }
        } else {
#pragma unroll
          for (int j = 0; j < kE; ++j)
            if (c + j >= 0 && c + j < x.V) {
              if constexpr (kHead)
                o[c + j] = static_cast<uint8_t>(cvt2(g[j], 0.0f, a.fmt));
              else
                o[c + j] = T::from_f(g[j]);
            }
        }
      }
    }
  }
  if constexpr (kOut == kAmax) {
    const uint32_t bits = __float_as_uint(largest) & 0x7FFFFFFFu;  // in the values' order, a NaN above all
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, bits);
    if (lane == 0) atomicMax(reinterpret_cast<unsigned int*>(a.amax), top);
  }
}

// ---- host ---------------------------------------------------------------------------------------
bool al(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Checks the rows and fills a; *empty: there is nothing to launch.
int rows_args(const ufp8_logit_rows* x, RowsArgs* a, const char* who) {
  if (!x) return set_error(UFP8_ERR_INVALID, "%s: null rows", who);
  if (x->dtype != UFP8_OUT_BF16 && x->dtype != UFP8_OUT_F32)
    return set_error(UFP8_ERR_INVALID, "%s: dtype %d is not UFP8_OUT_BF16/UFP8_OUT_F32", who, x->dtype);
  if (x->rows < 0 || x->V < 1) return set_error(UFP8_ERR_INVALID, "%s: rows must be >= 0 and V >= 1", who);
  const int64_t most = (int64_t(1) << 31) - (int64_t(1) << 20);  // an index past the end still fits 32 bits
  if (x->rows >= most) return set_error(UFP8_ERR_INVALID, "%s: rows exceed 2^31", who);
  if (x->V >= most) return set_error(UFP8_ERR_INVALID, "%s: V exceeds 2^31", who);
  if (x->rows > 0 && x->inner < 1) return set_error(UFP8_ERR_INVALID, "%s: inner must be >= 1", who);
  if (!(x->temperature > 0.0f) || std::isinf(x->temperature))
    return set_error(UFP8_ERR_INVALID, "%s: temperature must be finite and > 0", who);
  const double c2 = 1.4426950408889634 / static_cast<double>(x->temperature);
  if (c2 > 1e30 || c2 < 1e-30) return set_error(UFP8_ERR_INVALID, "%s: temperature %g is out of range", who,
                                                static_cast<double>(x->temperature));
  if (x->rows > 0 && !x->ptr) return set_error(UFP8_ERR_INVALID, "%s: null logits", who);
  if (!al(x->ptr, x->dtype == UFP8_OUT_F32 ? 4 : 2))
    return set_error(UFP8_ERR_ALIGN, "%s: logits not aligned to their type", who);
  a->x = x->ptr;
  a->rows = x->rows;
  a->inner = x->inner;
  a->stride_outer = x->stride_outer;
  a->stride_inner = x->stride_inner;
  a->V = static_cast<int>(x->V);
  a->mask = x->mask;
  a->c2 = static_cast<float>(c2);
  a->inv_t = static_cast<float>(1.0 / static_cast<double>(x->temperature));
  return UFP8_OK;
}

int check_ids(const void* p, int bytes, const char* what, const char* who) {
  if (bytes != 4 && bytes != 8) return set_error(UFP8_ERR_INVALID, "%s: %s of %d bytes (4 or 8)", who, what, bytes);
  if (!al(p, bytes)) return set_error(UFP8_ERR_ALIGN, "%s: %s not aligned to their type", who, what);
  return UFP8_OK;
}

// Output rows may not overlap: each lies behind the one before it.
int check_out(const ufp8_logit_rows* x, int64_t outer, int64_t inner, const char* who) {
  if (x->rows == 0) return UFP8_OK;
  if (inner < x->V || (x->rows > x->inner && outer < (x->inner - 1) * inner + x->V))
    return set_error(UFP8_ERR_INVALID, "%s: output rows overlap", who);
  return UFP8_OK;
}

template <class T, int kThr, int kMode, int kAhead>
int launch_stat(StatArgs& a, int part_bits, const DeviceInfo& dev, cudaStream_t s) {
  a.part_bits = part_bits;
  a.cap = 2 * a.k;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.r.rows << part_bits));
  cfg.blockDim = dim3(kThr);
  cfg.dynamicSmemBytes = kMode == kTopK ? TopLayout<kThr>::kBytes : 0;
  if (kMode == kTopK && part_bits) cfg.dynamicSmemBytes += (sizeof(uint64_t) * a.cap) << part_bits;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1u << part_bits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = part_bits ? 1 : 0;
  static thread_local int smem_dev = -1;  // more than 48 KB of dynamic shared memory is asked for once per device
  cudaError_t e = cudaSuccess;
  if (kMode == kTopK && smem_dev != dev.device) {
    e = cudaFuncSetAttribute(rowstat_kernel<T, kThr, kMode, kAhead>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(TopLayout<kThr>::kBytes + sizeof(uint64_t) * 2 * kMaxTop * kMaxParts));
    if (e == cudaSuccess) smem_dev = dev.device;
  }
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, rowstat_kernel<T, kThr, kMode, kAhead>, a);
  return e == cudaSuccess ? UFP8_OK : cuda_error(e, "row statistics launch");
}

// CTAs of a row and threads of a CTA, by rows per SM and the row's length (us with 256 threads / as chosen, entropy
// or 20 alternatives, on 148 SMs).
template <class T, int kMode>
int launch_stat(StatArgs& a, const DeviceInfo& dev, cudaStream_t s) {
  constexpr bool kTop = kMode == kTopK, kF32 = T::kKeyBits > 16;
  constexpr int kTile = 256 * kUnits * T::kElems;  // columns
  const int64_t rows = a.r.rows, V = a.r.V, sm = dev.sm_count, tiles = V / kTile;
  // A sweep without alternatives (620-1900 rows x 2-20 tiles of columns, both types; 256 threads, two parts, 128
  // threads) has the choice below within 5 % of the best of the three at 193 of 243 sizes, 1 % off on average.  The
  // borders at 8 and 14 tiles lie between the sizes of the first sweep (3, 12, 15) and are not the best for f32 rows of
  // 14 tiles and more, where one part of 256 (620 x 58709: 31.5 as chosen, 25.9) or 128 threads (1100 x 58709: 49.6,
  // 43.8) would be faster, nor for 2 tiles of bf16 (1100 x 19114: 14.8, 12.8 with 128 threads).
  // Few rows: a row is split as long as its parts are whole tiles and all CTAs run at once (those that search for
  // alternatives take more of an SM).  1 x 128256: 11.7 / 3.7; 48: 12.2 / 5.7; 148: 12.4 / 10.9; 300: 21 / 19.
  int bits = 0;
  while (bits < 3 && (rows << (bits + 1)) <= (kTop ? 27 * sm / 10 : 11 * sm / 2) && (V >> bits) > kTile) ++bits;
  // Long rows whose halves still balance better.  600 x 128256: 35.6 / 32.4; 1055: 52.8 / 50.9; 1300 would lose.
  if (!kTop && bits == 0 && rows <= 15 * sm / 2 && tiles >= 14) bits = 1;
  if (rows >= 4 * sm) {
    // Many short rows: smaller CTAs, more of which are resident, hide each other's ends.  8000 x 1500: 29 / 12.8,
    // with alternatives 88 / 31.
    if (V <= 8192 && a.k <= 64) return launch_stat<T, 64, kMode, 1>(a, 0, dev, s);
    // The same for longer ones (6000 x 32000 with alternatives: 107 / 95), and where the rows are more than one wave of
    // 256 threads each but not of 128 (1055 x 50257 f32: 41.8 / 36.1; 900 x 128256 with alternatives: 59 / 56).
    const bool shorter = V <= (kTop ? (kF32 ? 65536 : 32768) : 16384);
    const bool one_wave = kTop ? rows > (kF32 ? 4 : 5) * sm && rows <= 8 * sm
                               : rows > 6 * sm && rows <= 12 * sm && tiles >= 8 && tiles < 14;
    if (a.k <= 128 && (shorter || one_wave)) return launch_stat<T, 128, kMode, 1>(a, 0, dev, s);
  }
  // Two tiles of loads in flight take twice the registers: where two CTAs per SM are all there are.
  return (rows << bits) <= 2 * sm ? launch_stat<T, 256, kMode, 2>(a, bits, dev, s)
                                  : launch_stat<T, 256, kMode, 1>(a, bits, dev, s);
}

template <int kMode>
int launch_stat(StatArgs& a, int dtype, const DeviceInfo& dev, cudaStream_t s) {
  return dtype == UFP8_OUT_F32 ? launch_stat<F32, kMode>(a, dev, s) : launch_stat<Bf16, kMode>(a, dev, s);
}

template <class T, bool kDistill, int kOut>
int launch_grad(GradArgs& a, const DeviceInfo& dev, cudaStream_t s) {
  constexpr int kChunk = 32 * kUnits;
  // a row that starts off a 16-byte boundary can need one unit more
  const int64_t chunks = ((static_cast<int64_t>(a.r.V) + T::kElems - 1) / T::kElems + 1 + kChunk - 1) / kChunk;
  const bool entries = kDistill ? a.K > 0 : (a.dlogprob || a.dtop);
  const size_t smem = entries ? sizeof(float) * T::kElems * kChunk * kWarps : 0;
  // one wave: CTAs beyond the resident ones would start when the first are done
  static thread_local int dev_of[2] = {-1, -1}, per_sm[2] = {0, 0};
  if (dev_of[entries] != dev.device) {
    int n = 0;
    const cudaError_t e =
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, rowgrad_kernel<T, kDistill, kOut>, kThreads, smem);
    if (e != cudaSuccess) return cuda_error(e, "cudaOccupancyMaxActiveBlocksPerMultiprocessor(row gradient)");
    per_sm[entries] = n < 1 ? 1 : n;
    dev_of[entries] = dev.device;
  }
  const int64_t cap = static_cast<int64_t>(dev.sm_count) * per_sm[entries];
  // Longer tasks spread the row's set-up over more columns, as long as every warp still gets several.
  a.per_task = 1;
  while (a.per_task < 4 && a.per_task < chunks && a.r.rows * chunks >= cap * kWarps * 8 * a.per_task) a.per_task *= 2;
  a.tasks = static_cast<int>((chunks + a.per_task - 1) / a.per_task);
  const int64_t work = (a.r.rows * a.tasks + kWarps - 1) / kWarps;
  rowgrad_kernel<T, kDistill, kOut><<<static_cast<unsigned>(work < cap ? work : cap), kThreads, smem, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? UFP8_OK : cuda_error(e, "row gradient launch");
}

template <bool kDistill>
int launch_grad(GradArgs& a, int dtype, const DeviceInfo& dev, cudaStream_t s) {
  if (a.exact && a.r.rows > 0) {  // checked: fp8 output, bf16
    const cudaError_t e = cudaMemsetAsync(a.amax, 0, sizeof(float), s);
    if (e != cudaSuccess) return cuda_error(e, "cudaMemsetAsync(amax)");
    if (int rc = launch_grad<Bf16, kDistill, kAmax>(a, dev, s)) return rc;
    return launch_grad<Bf16, kDistill, kFp8>(a, dev, s);
  }
  if (a.fmt != UFP8_LIKE_LOGITS) {  // checked: bf16
    rowamax_kernel<kDistill><<<1, 1024, 0, s>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_error(e, "row amax launch");
    return a.r.rows == 0 ? UFP8_OK : launch_grad<Bf16, kDistill, kFp8>(a, dev, s);
  }
  return dtype == UFP8_OUT_F32 ? launch_grad<F32, kDistill, kLike>(a, dev, s)
                               : launch_grad<Bf16, kDistill, kLike>(a, dev, s);
}

// The output head's part of a backward: soft cap and fp8 output, for bf16 logits.
int head_args(const ufp8_logit_rows* x, float cap, int fmt, float* amax, float* inv_scale, GradArgs* a,
              const char* who) {
  const bool exact = fmt >= 0 && (fmt & UFP8_AMAX_EXACT);
  if (exact) fmt &= ~UFP8_AMAX_EXACT;
  const bool fp8 = fmt == UFP8_E4M3 || fmt == UFP8_E5M2;
  if (!fp8 && fmt != UFP8_LIKE_LOGITS)
    return set_error(UFP8_ERR_INVALID, "%s: fmt %d is not UFP8_E4M3/UFP8_E5M2/UFP8_LIKE_LOGITS", who, fmt);
  if (!(cap >= 0.0f) || std::isinf(cap))
    return set_error(UFP8_ERR_INVALID, "%s: cap must be 0 or a finite positive value", who);
  if (cap > 0.0f && !fp8) return set_error(UFP8_ERR_UNSUPPORTED, "%s: cap needs fp8 output", who);
  if (fp8 && x->dtype != UFP8_OUT_BF16) return set_error(UFP8_ERR_UNSUPPORTED, "%s: fp8 output needs bf16 logits", who);
  if (fp8 && (!amax || !inv_scale)) return set_error(UFP8_ERR_INVALID, "%s: null amax or inv_scale", who);
  if (!al(amax, 4) || !al(inv_scale, 4))
    return set_error(UFP8_ERR_ALIGN, "%s: amax or inv_scale not 4-byte aligned", who);
  a->fmt = fmt;
  a->exact = exact;
  a->inv_cap = cap > 0.0f ? 1.0f / cap : 0.0f;
  a->amax = amax;
  a->inv_scale = inv_scale;
  return UFP8_OK;
}

}  // namespace
}  // namespace ufp8

using namespace ufp8;

extern "C" int ufp8_logprob_forward(const ufp8_logit_rows* x, const void* tokens, int token_bytes, int64_t top_k,
                                    float* logprob, float* entropy, float* top_logprobs, int64_t* top_ids,
                                    float* stats, ufp8_stream_t stream) {
  const char* who = "ufp8_logprob_forward";
  StatArgs a{};
  if (int rc = rows_args(x, &a.r, who)) return rc;
  if (top_k < 0 || top_k > kMaxTop) return set_error(UFP8_ERR_INVALID, "%s: top_k must be 0..%d", who, kMaxTop);
  if (top_k > x->V) return set_error(UFP8_ERR_INVALID, "%s: top_k exceeds V", who);
  if (logprob || tokens)
    if (int rc = check_ids(tokens, token_bytes, "tokens", who)) return rc;
  if (!al(stats, 16)) return set_error(UFP8_ERR_ALIGN, "%s: stats not 16-byte aligned", who);
  if (x->rows == 0) return UFP8_OK;
  if (!logprob && !entropy && !top_k && !stats) return set_error(UFP8_ERR_INVALID, "%s: no output requested", who);
  if ((logprob != nullptr) != (tokens != nullptr))
    return set_error(UFP8_ERR_INVALID, "%s: tokens and logprob go together", who);
  if (top_k > 0 && (!top_logprobs || !top_ids)) return set_error(UFP8_ERR_INVALID, "%s: null top output", who);
  DeviceInfo* dev;
  if (int rc = device_info(&dev)) return rc;
  a.tokens = tokens;
  a.token_bytes = token_bytes;
  a.k = static_cast<int>(top_k);
  a.ib = 1;
  while ((int64_t(1) << a.ib) < x->V) ++a.ib;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_lp = top_logprobs;
  a.top_id = top_ids;
  a.stats = reinterpret_cast<float4*>(stats);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (top_k > 0) return launch_stat<kTopK>(a, x->dtype, *dev, s);
  return entropy ? launch_stat<kEntropy>(a, x->dtype, *dev, s) : launch_stat<kPlain>(a, x->dtype, *dev, s);
}

extern "C" int ufp8_logprob_backward(const ufp8_logit_rows* x, const float* stats, const void* tokens,
                                     int token_bytes, const float* dlogprob, int64_t dlogprob_stride,
                                     const float* dentropy, int64_t dentropy_stride, const float* dtop,
                                     const int64_t* top_ids, int64_t top_k, float cap, int fmt,
                                     void* dlogits, int64_t out_stride_outer, int64_t out_stride_inner, float* amax,
                                     float* inv_scale, ufp8_stream_t stream) {
  const char* who = "ufp8_logprob_backward";
  GradArgs a{};
  if (int rc = rows_args(x, &a.r, who)) return rc;
  if (top_k < 0 || top_k > kMaxTop) return set_error(UFP8_ERR_INVALID, "%s: top_k must be 0..%d", who, kMaxTop);
  if (int rc = check_out(x, out_stride_outer, out_stride_inner, who)) return rc;
  if (int rc = head_args(x, cap, fmt, amax, inv_scale, &a, who)) return rc;
  if (dlogprob)
    if (int rc = check_ids(tokens, token_bytes, "tokens", who)) return rc;
  if (!al(stats, 16)) return set_error(UFP8_ERR_ALIGN, "%s: stats not 16-byte aligned", who);
  if (fmt == UFP8_LIKE_LOGITS && !al(dlogits, x->dtype == UFP8_OUT_F32 ? 4 : 2))
    return set_error(UFP8_ERR_ALIGN, "%s: dlogits not aligned to their type", who);
  if (x->rows == 0 && fmt == UFP8_LIKE_LOGITS) return UFP8_OK;
  if (x->rows > 0 && (!stats || !dlogits)) return set_error(UFP8_ERR_INVALID, "%s: null stats or dlogits", who);
  if (x->rows > 0 && dlogprob && !tokens) return set_error(UFP8_ERR_INVALID, "%s: null tokens", who);
  if (dtop && (!top_ids || top_k == 0)) return set_error(UFP8_ERR_INVALID, "%s: null top_ids", who);
  DeviceInfo* dev;
  if (int rc = device_info(&dev)) return rc;
  a.stats = reinterpret_cast<const float4*>(stats);
  a.tokens = tokens;
  a.token_bytes = token_bytes;
  a.dlogprob = dlogprob;
  a.dlogprob_stride = dlogprob_stride;
  a.dentropy = dentropy;
  a.dentropy_stride = dentropy_stride;
  a.dtop = dtop;
  a.top_id = top_ids;
  a.k = static_cast<int>(top_k);
  a.out = dlogits;
  a.out_outer = out_stride_outer;
  a.out_inner = out_stride_inner;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return launch_grad<false>(a, x->dtype, *dev, s);
}

namespace {
int distill_check(const ufp8_logit_rows* x, const void* ids, int id_bytes, const void* teacher, int teacher_dtype,
                  int64_t entries, const char* who) {
  if (entries < 0 || entries > kMaxEntries)
    return set_error(UFP8_ERR_INVALID, "%s: entries must be 0..%d", who, kMaxEntries);
  if (teacher_dtype != UFP8_OUT_BF16 && teacher_dtype != UFP8_OUT_F32)
    return set_error(UFP8_ERR_INVALID, "%s: teacher_dtype %d is not UFP8_OUT_BF16/UFP8_OUT_F32", who, teacher_dtype);
  if (int rc = check_ids(ids, id_bytes, "teacher ids", who)) return rc;
  if (!al(teacher, teacher_dtype == UFP8_OUT_F32 ? 4 : 2))
    return set_error(UFP8_ERR_ALIGN, "%s: teacher not aligned to its type", who);
  if (x->rows > 0 && entries > 0 && (!ids || !teacher))
    return set_error(UFP8_ERR_INVALID, "%s: null teacher ids or logits", who);
  return UFP8_OK;
}
}  // namespace

extern "C" int ufp8_distill_forward(const ufp8_logit_rows* x, const void* teacher_ids, int id_bytes,
                                    const void* teacher, int teacher_dtype, int64_t entries, float* loss, float* stats,
                                    ufp8_stream_t stream) {
  const char* who = "ufp8_distill_forward";
  StatArgs a{};
  if (int rc = rows_args(x, &a.r, who)) return rc;
  if (int rc = distill_check(x, teacher_ids, id_bytes, teacher, teacher_dtype, entries, who)) return rc;
  if (!al(stats, 16)) return set_error(UFP8_ERR_ALIGN, "%s: stats not 16-byte aligned", who);
  if (x->rows == 0) return UFP8_OK;
  if (!loss) return set_error(UFP8_ERR_INVALID, "%s: null loss", who);
  DeviceInfo* dev;
  if (int rc = device_info(&dev)) return rc;
  a.ids = teacher_ids;
  a.id_bytes = id_bytes;
  a.teacher = teacher;
  a.teacher_f32 = teacher_dtype == UFP8_OUT_F32;
  a.K = static_cast<int>(entries);
  a.loss = loss;
  a.stats = reinterpret_cast<float4*>(stats);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return launch_stat<kTeacher>(a, x->dtype, *dev, s);
}

extern "C" int ufp8_distill_backward(const ufp8_logit_rows* x, const float* stats, const void* teacher_ids,
                                     int id_bytes, const void* teacher, int teacher_dtype, int64_t entries,
                                     const float* dloss, int64_t dloss_stride, float cap, int fmt,
                                     void* dlogits, int64_t out_stride_outer, int64_t out_stride_inner, float* amax,
                                     float* inv_scale, ufp8_stream_t stream) {
  const char* who = "ufp8_distill_backward";
  GradArgs a{};
  if (int rc = rows_args(x, &a.r, who)) return rc;
  if (int rc = distill_check(x, teacher_ids, id_bytes, teacher, teacher_dtype, entries, who)) return rc;
  if (int rc = check_out(x, out_stride_outer, out_stride_inner, who)) return rc;
  if (int rc = head_args(x, cap, fmt, amax, inv_scale, &a, who)) return rc;
  if (!al(stats, 16)) return set_error(UFP8_ERR_ALIGN, "%s: stats not 16-byte aligned", who);
  if (fmt == UFP8_LIKE_LOGITS && !al(dlogits, x->dtype == UFP8_OUT_F32 ? 4 : 2))
    return set_error(UFP8_ERR_ALIGN, "%s: dlogits not aligned to their type", who);
  if (x->rows == 0 && fmt == UFP8_LIKE_LOGITS) return UFP8_OK;
  if (x->rows > 0 && (!stats || !dlogits || !dloss))
    return set_error(UFP8_ERR_INVALID, "%s: null stats, dloss or dlogits", who);
  DeviceInfo* dev;
  if (int rc = device_info(&dev)) return rc;
  a.stats = reinterpret_cast<const float4*>(stats);
  a.ids = teacher_ids;
  a.id_bytes = id_bytes;
  a.teacher = teacher;
  a.teacher_f32 = teacher_dtype == UFP8_OUT_F32;
  a.K = static_cast<int>(entries);
  a.dloss = dloss;
  a.dloss_stride = dloss_stride;
  a.out = dlogits;
  a.out_outer = out_stride_outer;
  a.out_inner = out_stride_inner;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return launch_grad<true>(a, x->dtype, *dev, s);
}
