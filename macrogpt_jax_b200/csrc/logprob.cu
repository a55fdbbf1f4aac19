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
//   rowstat_kernel   one CTA per row streams the row once, a running (m, s, t) per thread,
//                    and in the same pass keeps the candidates for the top alternatives.
//   rowgrad_kernel   the gradient of both operators: p_v (A + B log2 p_v) with row factors A, B, plus
//                    weights at a few columns (the token, the alternatives, the teacher's entries).
#include <cuda_bf16.h>

#include <cmath>

#include "internal.h"

namespace ufp8 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSub = kThreads * 8;  // columns that one unit (8 elements) of every thread covers
constexpr int kCand = 4096;         // candidate keys of a CTA; >= kMaxTop + kSub
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
  static constexpr int kWords = 1;    // 16-byte words of a unit
  static constexpr int kUnits = 4;    // units per thread and tile
  static constexpr int kKeyBits = 16;
  static __device__ __forceinline__ float to_f(raw r) { return __uint_as_float(static_cast<uint32_t>(r) << 16); }
  static __device__ __forceinline__ raw from_f(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
};
struct F32 {
  using raw = float;
  static constexpr int kWords = 2;
  static constexpr int kUnits = 2;
  static constexpr int kKeyBits = 32;
  static __device__ __forceinline__ float to_f(raw r) { return r; }
  static __device__ __forceinline__ raw from_f(float f) { return f; }
};

template <class T>
struct Unit {
  uint4 w[T::kWords];
};

template <class T>
__device__ __forceinline__ void unpack(const Unit<T>& u, float (&v)[8]) {
  if constexpr (T::kWords == 1) {
    const uint32_t w[4] = {u.w[0].x, u.w[0].y, u.w[0].z, u.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __uint_as_float(u.w[i].x);
      v[4 * i + 1] = __uint_as_float(u.w[i].y);
      v[4 * i + 2] = __uint_as_float(u.w[i].z);
      v[4 * i + 3] = __uint_as_float(u.w[i].w);
    }
  }
}

// A row as units of 8 elements that start on 16-byte boundaries: unit i covers the columns
// [8 i - off, 8 i - off + 8) where off elements lie between the boundary at or below the row's first
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
    units = (v + off + 7) >> 3;
  }
  // V < 2^31 - 2^20: a column a tile past the row's end still fits
  __device__ __forceinline__ int col(int i) const { return i * 8 - off; }
  __device__ __forceinline__ Unit<T> load(int i) const {
    const int c = col(i);
    Unit<T> u;
    if (c >= 0 && c + 8 <= V) {
#pragma unroll
      for (int k = 0; k < T::kWords; ++k) u.w[k] = ld16(reinterpret_cast<const uint4*>(p + c) + k);
    } else {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (c + j >= 0 && c + j < V) ? T::to_f(p[c + j]) : kNegInf;
      uint32_t* w = &u.w[0].x;
      if constexpr (T::kWords == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = (__float_as_uint(v[2 * j]) >> 16) | (__float_as_uint(v[2 * j + 1]) & 0xFFFF0000u);
      } else {
        u.w[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        u.w[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
      }
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

// ---- running softmax statistics -----------------------------------------------------------------
struct Stat {
  float m, s, t;
};

// (m, s, t) <- (m, s, t) + (m2, s2, t2).  A NaN in either part makes s NaN.
__device__ __forceinline__ void merge(Stat& a, const Stat& b, float c2) {
  const float M = maxn(a.m, b.m);
  if (M == kNegInf) return;  // both empty
  // 2^-1000 is 0, and the clamp keeps 0 * d finite
  const float da = a.m == kNegInf ? -1000.0f : maxn(__fmul_rn(a.m - M, c2), -1000.0f);
  const float db = b.m == kNegInf ? -1000.0f : maxn(__fmul_rn(b.m - M, c2), -1000.0f);
  const float fa = ex2a(da), fb = ex2a(db);
  a.t = __fadd_rn(__fmul_rn(fa, __fmaf_rn(da, a.s, a.t)), __fmul_rn(fb, __fmaf_rn(db, b.s, b.t)));
  a.s = __fadd_rn(__fmul_rn(fa, a.s), __fmul_rn(fb, b.s));
  a.m = M;
}

// Eight values into the running statistics; cm is their maximum (NaN if one is NaN).
template <bool kEnt>
__device__ __forceinline__ void fold8(const float (&v)[8], float cm, Stat& a, float c2) {
  if (!(cm <= a.m)) {
    const float d = a.m == kNegInf ? -1000.0f : maxn(__fmul_rn(a.m - cm, c2), -1000.0f);
    const float f = ex2a(d);
    if (kEnt) a.t = __fmul_rn(f, __fmaf_rn(d, a.s, a.t));
    a.s = __fmul_rn(f, a.s);
    a.m = cm;
  }
  const float mz = a.m == kNegInf ? 0.0f : a.m;
  float s = 0.0f, t = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // -160: below the smallest f32, so the power is 0, and 0 * z stays 0 for z = -inf
    const float z = maxn(__fmul_rn(__fsub_rn(v[j], mz), c2), -160.0f);
    const float e = ex2a(z);
    s = __fadd_rn(s, e);
    if (kEnt) t = __fmaf_rn(e, z, t);
  }
  a.s = __fadd_rn(a.s, s);
  if (kEnt) a.t = __fadd_rn(a.t, t);
}

// The CTA's statistics, merged lane by lane (a butterfly that is commutative bit for bit) and then
// warp by warp; valid in thread 0 .. 31 after the barrier inside.
__device__ __forceinline__ Stat block_merge(Stat a, Stat* sh, float c2) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor_sync(0xFFFFFFFFu, a.m, o);
    b.s = __shfl_xor_sync(0xFFFFFFFFu, a.s, o);
    b.t = __shfl_xor_sync(0xFFFFFFFFu, a.t, o);
    merge(a, b, c2);
  }
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  Stat r = sh[0];
  for (int w = 1; w < kWarps; ++w) merge(r, sh[w], c2);
  return r;
}

// ---- the largest k of a row ---------------------------------------------------------------------
// A key orders an element by value (NaN above all, -0 equal to 0) and then by column, lower first:
// the value's bits mapped to an unsigned order, above ib bits of (2^ib - 1 - column).  Keys of a row
// are distinct, so the k largest are one set whatever the order in which they were found.
template <class T>
__device__ __forceinline__ uint64_t make_key(float x, uint32_t col, int ib) {
  uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));  // one zero
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (x != x) b = 0xFFFFFFFFu;
  b >>= 32 - T::kKeyBits;
  return (static_cast<uint64_t>(b) << ib) | (((1ull << ib) - 1ull) - col);
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

struct TopShared {
  uint32_t hist[256];
  int cnt;
  int bin, above, in_bin;
  float tau[kWarps];
};

// keys[0, n) -> those >= bound (and, with below_col >= 0, of a column < below_col), in any order at
// keys[0, sh.cnt).  Whole CTA; ends with a barrier.
__device__ __forceinline__ int filter_keys(uint64_t* keys, int n, uint64_t bound, int64_t below_col, int ib,
                                           TopShared& sh) {
  __syncthreads();
  if (threadIdx.x == 0) sh.cnt = 0;
  for (int b = 0; b < n; b += kThreads) {
    const int i = b + static_cast<int>(threadIdx.x);
    const uint64_t key = i < n ? keys[i] : 0;
    const bool keep = i < n && key >= bound && (below_col < 0 || key_col(key, ib) < below_col);
    __syncthreads();  // this block is read before anything is written to it
    if (keep) keys[atomicAdd(&sh.cnt, 1)] = key;
  }
  __syncthreads();
  const int left = sh.cnt;
  __syncthreads();
  return left;
}

// Keeps the k largest of keys[0, n), n > k, by radix selection from the key's top bits in digits of
// eight; returns a bound b with exactly k keys >= b.  Whole CTA.
__device__ uint64_t keep_largest(uint64_t* keys, int n, int k, int bits, int ib, TopShared& sh) {
  uint64_t bound = 0;
  int need = k, shift = bits;
  while (shift > 0) {
    const int w = shift < 8 ? shift : 8;
    const int top = shift;
    shift -= w;
    sh.hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t key = keys[i];
      if ((key >> top) == (bound >> top)) atomicAdd(&sh.hist[(key >> shift) & ((1u << w) - 1u)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // lane l holds bins 255 - 8 l ... 248 - 8 l, largest first
      const int hi = 255 - 8 * static_cast<int>(threadIdx.x);
      int sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += static_cast<int>(sh.hist[hi - j]);
      int pre = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, pre, o);
        if (static_cast<int>(threadIdx.x) >= o) pre += up;
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
    if (sh.in_bin == need) break;  // the whole bin belongs to the k largest
    __syncthreads();               // everyone has read the choice before the next digit
  }
  filter_keys(keys, n, bound, -1, ib, sh);
  return bound;
}

// ---- forward ------------------------------------------------------------------------------------
struct StatArgs {
  RowsArgs r;
  // token_logprobs
  const void* tokens;  // may be null
  int token_bytes;
  int k;
  int ib;  // column bits of a key
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
  return a.teacher_f32 ? static_cast<const float*>(a.teacher)[i] : Bf16::to_f(static_cast<const uint16_t*>(a.teacher)[i]);
}
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

// One warp: the row's loss sum_j q_j (log q_j - log p_{id_j}) over the entries with id >= 0, and the
// teacher's (max, log2 sum).  Entries whose teacher value is -inf have q = 0 and contribute 0; a row
// without any weight has loss 0 (and max -inf, which the gradient reads as "no entry").
template <class T>
__device__ __forceinline__ float distill_row(const StatArgs& a, int64_t row, const Row<T>& x, float m, float ls,
                                             float* tm_out, float* tl_out) {
  const int lane = threadIdx.x & 31;
  const float c2 = a.r.c2;
  const int64_t base = row * a.K;
  float tm = kNegInf;
  for (int j = lane; j < a.K; j += 32)
    if (load_id(a.ids, a.id_bytes, base + j) >= 0) tm = maxn(tm, teacher_val(a, base + j));
  tm = warp_maxn(tm);
  *tm_out = tm;
  *tl_out = 0.0f;
  if (tm == kNegInf) return 0.0f;
  float ts = 0.0f;
  for (int j = lane; j < a.K; j += 32)
    if (load_id(a.ids, a.id_bytes, base + j) >= 0)
      ts = __fadd_rn(ts, ex2a(__fmul_rn(__fsub_rn(teacher_val(a, base + j), tm), c2)));
  ts = warp_sum(ts);
  const float tl = log2f(ts), tls = logf(ts);
  *tl_out = tl;
  float sum = 0.0f;
  for (int j = lane; j < a.K; j += 32) {
    const int64_t id = load_id(a.ids, a.id_bytes, base + j);
    if (id < 0) continue;
    const float td = __fsub_rn(teacher_val(a, base + j), tm);
    const float q = ex2a(__fmaf_rn(td, c2, -tl));
    if (q == 0.0f) continue;
    const float xv = id < a.r.V ? T::to_f(x.p[id]) : __int_as_float(0x7FC00000);
    const float lp = __fmaf_rn(__fsub_rn(xv, m), a.r.inv_t, -ls);
    sum = __fmaf_rn(q, __fsub_rn(__fmaf_rn(td, a.r.inv_t, -tls), lp), sum);
  }
  return warp_sum(sum);
}

template <class T, bool kEnt, bool kTop, bool kDistill>
__global__ void __launch_bounds__(kThreads) rowstat_kernel(const StatArgs a) {
  extern __shared__ uint64_t keys[];  // kTop: kCand
  __shared__ Stat sh_stat[kWarps];
  __shared__ TopShared sh;
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const float c2 = a.r.c2;

  if (a.r.mask && a.r.mask[row] == 0) {  // nothing of the row is read
    if (tid == 0) {
      if (a.logprob) a.logprob[row] = 0.0f;
      if (a.entropy) a.entropy[row] = 0.0f;
      if (kDistill) a.loss[row] = 0.0f;
      if (a.stats) a.stats[row] = make_float4(kNegInf, 0.0f, kDistill ? kNegInf : 0.0f, 0.0f);
    }
    if (kTop && tid < a.k) {
      a.top_lp[static_cast<int64_t>(row) * a.k + tid] = kNegInf;
      a.top_id[static_cast<int64_t>(row) * a.k + tid] = -1;
    }
    return;
  }

  const Row<T> x(a.r.x, RowIndex(a.r, row).elem(a.r.stride_outer, a.r.stride_inner), a.r.V);
  Stat st{kNegInf, 0.0f, 0.0f};
  float tau = kNegInf;     // every one of the k largest so far is >= tau ...
  bool inclusive = true;   // ... and a later element equal to it may still belong to them
  if (kTop && tid == 0) sh.cnt = 0;

  constexpr int kTile = kThreads * T::kUnits;  // units of a tile
  for (int u0 = 0; u0 < x.units; u0 += kTile) {
    Unit<T> w[T::kUnits];
    float mx[T::kUnits];
#pragma unroll
    for (int u = 0; u < T::kUnits; ++u) {
      const int i = u0 + u * kThreads + tid;
      if (i < x.units)
        w[u] = x.load(i);
      else
        w[u].w[0] = w[u].w[T::kWords - 1] = T::kWords == 1
                                                ? make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u)
                                                : make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
    }
#pragma unroll
    for (int u = 0; u < T::kUnits; ++u) {
      float v[8];
      unpack<T>(w[u], v);
      mx[u] = maxn(maxn(maxn(v[0], v[1]), maxn(v[2], v[3])), maxn(maxn(v[4], v[5]), maxn(v[6], v[7])));
      fold8<kEnt>(v, mx[u], st, c2);
    }
    if constexpr (kTop) {
      // Columns grow from tile to tile and, inside a tile, from unit to unit.
      if (u0 == 0) {
        // tau = min over groups of threads of the group's largest unit maximum, with at least k groups:
        // k elements of this tile are >= tau.  (fmaxf skips NaN maxima: the bound only gets lower.)
        float g = kNegInf;
#pragma unroll
        for (int u = 0; u < T::kUnits; ++u) g = fmaxf(g, mx[u]);
        int tpg = 32;
        while (tpg > 1 && kThreads / tpg < a.k) tpg >>= 1;
        for (int o = 1; o < tpg; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
        for (int o = tpg; o < 32; o <<= 1) g = fminf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
        if ((tid & 31) == 0) sh.tau[tid >> 5] = g;
        __syncthreads();
        tau = sh.tau[0];
        for (int i = 1; i < kWarps; ++i) tau = fminf(tau, sh.tau[i]);
      }
      auto append = [&](int u) {
        bool high = false;
        if (inclusive ? !(mx[u] < tau) : !(mx[u] <= tau)) {
          float v[8];
          unpack<T>(w[u], v);
          const int c = x.col(u0 + u * kThreads + tid);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if ((inclusive ? !(v[j] < tau) : !(v[j] <= tau)) && c + j >= 0 && c + j < x.V) {
              const int pos = atomicAdd(&sh.cnt, 1);
              if (pos < kCand) keys[pos] = make_key<T>(v[j], static_cast<uint32_t>(c + j), a.ib);
              high |= pos >= kCand / 2;
            }
          }
        }
        return high;
      };
      bool high = false;
#pragma unroll
      for (int u = 0; u < T::kUnits; ++u) high |= append(u);
      if (__syncthreads_or(high)) {
        int n = sh.cnt;
        __syncthreads();
        auto shrink = [&]() {
          const uint64_t bound = keep_largest(keys, n, a.k, T::kKeyBits + a.ib, a.ib, sh);
          n = a.k;
          tau = key_value<T>(bound, a.ib);
          inclusive = false;
        };
        if (n > kCand) {
          // Too many for the buffer: drop this tile's keys and take its units one at a time, each
          // of which (kSub columns) fits behind at most kCand - kSub keys.
          n = filter_keys(keys, kCand, 0, x.col(u0) < 0 ? 0 : x.col(u0), a.ib, sh);
#pragma unroll
          for (int u = 0; u < T::kUnits; ++u) {
            if (n > kCand - kSub) shrink();
            append(u);
            __syncthreads();
            n = sh.cnt;
            __syncthreads();
          }
        }
        if (n > kCand / 2) shrink();
      }
      inclusive = false;  // later columns lose a tie
    }
  }

  const Stat r = block_merge(st, sh_stat, c2);
  const float l2 = log2f(r.s), ls = logf(r.s);
  if constexpr (kDistill) {
    if (tid < 32) {
      float tm, tl;
      const float loss = distill_row<T>(a, row, x, r.m, ls, &tm, &tl);
      if (tid == 0) {
        a.loss[row] = loss;
        if (a.stats) a.stats[row] = make_float4(r.m, l2, tm, tl);
      }
    }
    return;
  } else {
    if (tid == 0) {
      const float H = kEnt ? __fmul_rn(kLn2, __fsub_rn(l2, __fdiv_rn(r.t, r.s))) : 0.0f;
      if (a.logprob) {
        const int col = token_col(load_id(a.tokens, a.token_bytes, row), a.r.V);
        const float xv = col >= 0 ? T::to_f(x.p[col]) : __int_as_float(0x7FC00000);
        a.logprob[row] = __fmaf_rn(__fsub_rn(xv, r.m), a.r.inv_t, -ls);
      }
      if (a.entropy) a.entropy[row] = H;
      if (a.stats) a.stats[row] = make_float4(r.m, l2, H, 0.0f);
    }
    if constexpr (kTop) {
      int n = sh.cnt;
      __syncthreads();
      if (n > a.k) keep_largest(keys, n, a.k, T::kKeyBits + a.ib, a.ib, sh);
      n = a.k;  // V >= k: there are k
      if (tid < n) {
        const uint64_t key = keys[tid];
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += keys[i] > key;
        const uint32_t col = key_col(key, a.ib);
        const float xv = T::to_f(x.p[col]);
        a.top_lp[static_cast<int64_t>(row) * a.k + rank] = __fmaf_rn(__fsub_rn(xv, r.m), a.r.inv_t, -ls);
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
  void* out;
  int64_t out_outer, out_inner;  // row strides of the output
  int tasks;     // tasks of a row
  int per_task;  // chunks of a task
};

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

// The warps of a resident grid walk (row, task) units on their own, without a barrier; a task is `per_task`
// chunks of a row, a chunk 2 KB of it, kUnits 16-byte loads a lane.  Per task the warp works out the row
// factors; per chunk it adds the weights of the row's entries that fall into it into `wt`, one f32 per
// column and zero elsewhere, in entry order, so that the result does not depend on timing.  Then
// v = p * factor + weight, and a lane with a weight in its columns sets those back to zero.
template <class T, bool kDistill>
__global__ void __launch_bounds__(kThreads, 4) rowgrad_kernel(const GradArgs a) {
  constexpr int kChunk = 32 * T::kUnits;  // units of a chunk
  extern __shared__ float4 wt_all[];      // kWarps * kChunk * 8 floats
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float4* wt4 = wt_all + warp * kChunk * 2;
  float* wt = reinterpret_cast<float*>(wt4);
  // unit wi = (row, task) = (wi / tasks, wi % tasks), advanced by the grid's warps without divisions
  const int rows = static_cast<int>(a.r.rows);
  const unsigned first = blockIdx.x * kWarps + warp, step = gridDim.x * kWarps;
  const int step_r = static_cast<int>(step / a.tasks), step_t = static_cast<int>(step % a.tasks);
  int row = static_cast<int>(first / a.tasks), task = static_cast<int>(first % a.tasks);
  const uint64_t c22 = pk(a.r.c2, a.r.c2);
  const int n = kDistill ? a.K : (a.dlogprob ? 1 : 0) + (a.dtop ? a.k : 0);
  if (n > 0)
    for (int i = lane; i < kChunk * 2; i += 32) wt4[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __syncwarp();
  for (; row < rows; row += step_r, task += step_t) {
    if (task >= a.tasks) {
      task -= a.tasks;
      if (++row >= rows) break;
    }
    const RowIndex ri(a.r, row);
    const Row<T> x(a.r.x, ri.elem(a.r.stride_outer, a.r.stride_inner), a.r.V);
    typename T::raw* o = static_cast<typename T::raw*>(a.out) + ri.elem(a.out_outer, a.out_inner);
    const bool vec = ((reinterpret_cast<uintptr_t>(o) ^ reinterpret_cast<uintptr_t>(x.p)) & 15u) == 0;
    const float4 st = a.stats[row];
    const bool dead = (a.r.mask && a.r.mask[row] == 0) || (kDistill && st.z == kNegInf);
    int u0 = task * a.per_task * kChunk;
    const int u_end = min(u0 + a.per_task * kChunk, x.units);
    float A = 0.0f, B = 0.0f;
    int id0 = -1;  // the first 32 entries stay with their lanes
    float val0 = 0.0f;
    if (!dead) {
      if (lane < n) load_entry<kDistill>(a, row, lane, &id0, &val0);
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
    }
    const uint64_t nm = pk(-st.x, -st.x), nl = pk(-st.y, -st.y);
    const uint64_t A2 = pk(A, A), B2 = pk(B, B);
    for (; u0 < u_end; u0 += kChunk) {
      const int lo = x.col(u0), hi = x.col(u0 + kChunk);
      const bool whole = lo >= 0 && hi <= x.V && vec;  // every unit is 16-byte loads and stores
      Unit<T> w[T::kUnits];
      unsigned flag = 0;  // bit u: unit u of this lane holds a weight
      if (!dead) {
        if (whole) {
          const uint4* p = reinterpret_cast<const uint4*>(x.p + lo) + lane * T::kWords;
#pragma unroll
          for (int u = 0; u < T::kUnits; ++u)
#pragma unroll
            for (int k = 0; k < T::kWords; ++k) w[u].w[k] = ld16(p + u * 32 * T::kWords + k);
        } else {
#pragma unroll
          for (int u = 0; u < T::kUnits; ++u) {
            const int i = u0 + u * 32 + lane;
            if (i < x.units) w[u] = x.load(i);
          }
        }
        for (int j0 = 0; j0 < n; j0 += 32) {
          int id = id0;
          float val = val0;
          if (j0 > 0) {
            id = -1;
            if (j0 + lane < n) load_entry<kDistill>(a, row, j0 + lane, &id, &val);
          }
          const bool in = id >= 0 && id >= lo && id < hi;
          const unsigned active = __ballot_sync(0xFFFFFFFFu, in);
          if (active == 0) continue;
          const float ew = kDistill ? __fmul_rn(-A, ex2a(__fmaf_rn(__fsub_rn(val, st.z), a.r.c2, -st.w)))
                                    : __fmul_rn(val, a.r.inv_t);
          const int at = id - lo;
          for (unsigned left = active; left; left &= left - 1) {  // in entry order
            const int src = __ffs(left) - 1;
            const int sat = __shfl_sync(0xFFFFFFFFu, at, src);
            const float sw = __shfl_sync(0xFFFFFFFFu, ew, src);
            if (lane == ((sat >> 3) & 31)) {  // the lane that owns the column
              wt[sat] = __fadd_rn(wt[sat], sw);
              flag |= 1u << (sat >> 8);
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < T::kUnits; ++u) {
        const int i = u0 + u * 32 + lane;
        if (!whole && i >= x.units) continue;
        float v[8];
        if (dead) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        } else {
          unpack<T>(w[u], v);
          float e[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
          if ((flag >> u) & 1u) {
            float4* q = wt4 + (u * 32 + lane) * 2;
            const float4 q0 = q[0], q1 = q[1];
            e[0] = q0.x, e[1] = q0.y, e[2] = q0.z, e[3] = q0.w, e[4] = q1.x, e[5] = q1.y, e[6] = q1.z, e[7] = q1.w;
            q[0] = q[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          }
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            // log2 p; below -160 the power is 0 and 0 * log2 p has to stay 0
            float z0, z1;
            unpk(fma2(add2(pk(v[j], v[j + 1]), nm), c22, nl), z0, z1);
            if (!kDistill) {
              z0 = maxn(z0, -160.0f);
              z1 = maxn(z1, -160.0f);
            }
            const uint64_t f = kDistill ? A2 : fma2(B2, pk(z0, z1), A2);
            unpk(fma2(pk(ex2a(z0), ex2a(z1)), f, pk(e[j], e[j + 1])), v[j], v[j + 1]);
          }
        }
        const int c = x.col(i);
        if (whole || (vec && c >= 0 && c + 8 <= x.V)) {
          if constexpr (T::kWords == 1) {
            uint4 q;
            uint32_t* qw = &q.x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
              qw[j] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(o + c) = q;
          } else {
            reinterpret_cast<float4*>(o + c)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(o + c)[1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (c + j >= 0 && c + j < x.V) o[c + j] = T::from_f(v[j]);
        }
      }
    }
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
  if (x->rows >= (int64_t(1) << 31)) return set_error(UFP8_ERR_INVALID, "%s: rows exceed 2^31", who);
  if (x->V >= (int64_t(1) << 31) - (int64_t(1) << 20)) return set_error(UFP8_ERR_INVALID, "%s: V exceeds 2^31", who);
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

template <class T, bool kEnt, bool kTop, bool kDistill>
int launch_stat(const StatArgs& a, cudaStream_t s) {
  const size_t smem = kTop ? sizeof(uint64_t) * kCand : 0;
  rowstat_kernel<T, kEnt, kTop, kDistill><<<static_cast<unsigned>(a.r.rows), kThreads, smem, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? UFP8_OK : cuda_error(e, "row statistics launch");
}

template <class T>
int launch_logprob(const StatArgs& a, bool ent, cudaStream_t s) {
  if (a.k > 0) return ent ? launch_stat<T, true, true, false>(a, s) : launch_stat<T, false, true, false>(a, s);
  return ent ? launch_stat<T, true, false, false>(a, s) : launch_stat<T, false, false, false>(a, s);
}

template <class T, bool kDistill>
int launch_grad(GradArgs& a, const DeviceInfo& dev, cudaStream_t s) {
  constexpr int kChunk = 32 * T::kUnits;
  // a row that starts off a 16-byte boundary can need one unit more
  const int64_t chunks = ((static_cast<int64_t>(a.r.V) + 7) / 8 + 1 + kChunk - 1) / kChunk;
  const bool entries = kDistill ? a.K > 0 : (a.dlogprob || a.dtop);
  const size_t smem = entries ? sizeof(float) * 8 * kChunk * kWarps : 0;
  // one wave: CTAs beyond the resident ones would start when the first are done
  static thread_local int dev_of[2] = {-1, -1}, per_sm[2] = {0, 0};
  if (dev_of[entries] != dev.device) {
    int n = 0;
    const cudaError_t e =
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, rowgrad_kernel<T, kDistill>, kThreads, smem);
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
  rowgrad_kernel<T, kDistill><<<static_cast<unsigned>(work < cap ? work : cap), kThreads, smem, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? UFP8_OK : cuda_error(e, "row gradient launch");
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
  const bool ent = entropy != nullptr;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return x->dtype == UFP8_OUT_F32 ? launch_logprob<F32>(a, ent, s) : launch_logprob<Bf16>(a, ent, s);
}

extern "C" int ufp8_logprob_backward(const ufp8_logit_rows* x, const float* stats, const void* tokens,
                                     int token_bytes, const float* dlogprob, int64_t dlogprob_stride,
                                     const float* dentropy, int64_t dentropy_stride, const float* dtop,
                                     const int64_t* top_ids, int64_t top_k, void* dlogits,
                                     int64_t out_stride_outer, int64_t out_stride_inner, ufp8_stream_t stream) {
  const char* who = "ufp8_logprob_backward";
  GradArgs a{};
  if (int rc = rows_args(x, &a.r, who)) return rc;
  if (top_k < 0 || top_k > kMaxTop) return set_error(UFP8_ERR_INVALID, "%s: top_k must be 0..%d", who, kMaxTop);
  if (int rc = check_out(x, out_stride_outer, out_stride_inner, who)) return rc;
  if (dlogprob)
    if (int rc = check_ids(tokens, token_bytes, "tokens", who)) return rc;
  if (!al(stats, 16)) return set_error(UFP8_ERR_ALIGN, "%s: stats not 16-byte aligned", who);
  if (!al(dlogits, x->dtype == UFP8_OUT_F32 ? 4 : 2))
    return set_error(UFP8_ERR_ALIGN, "%s: dlogits not aligned to their type", who);
  if (x->rows == 0) return UFP8_OK;
  if (!stats || !dlogits) return set_error(UFP8_ERR_INVALID, "%s: null stats or dlogits", who);
  if (dlogprob && !tokens) return set_error(UFP8_ERR_INVALID, "%s: null tokens", who);
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
  return x->dtype == UFP8_OUT_F32 ? launch_grad<F32, false>(a, *dev, s) : launch_grad<Bf16, false>(a, *dev, s);
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
  return x->dtype == UFP8_OUT_F32 ? launch_stat<F32, false, false, true>(a, s)
                                  : launch_stat<Bf16, false, false, true>(a, s);
}

extern "C" int ufp8_distill_backward(const ufp8_logit_rows* x, const float* stats, const void* teacher_ids,
                                     int id_bytes, const void* teacher, int teacher_dtype, int64_t entries,
                                     const float* dloss, int64_t dloss_stride, void* dlogits,
                                     int64_t out_stride_outer, int64_t out_stride_inner, ufp8_stream_t stream) {
  const char* who = "ufp8_distill_backward";
  GradArgs a{};
  if (int rc = rows_args(x, &a.r, who)) return rc;
  if (int rc = distill_check(x, teacher_ids, id_bytes, teacher, teacher_dtype, entries, who)) return rc;
  if (int rc = check_out(x, out_stride_outer, out_stride_inner, who)) return rc;
  if (!al(stats, 16)) return set_error(UFP8_ERR_ALIGN, "%s: stats not 16-byte aligned", who);
  if (!al(dlogits, x->dtype == UFP8_OUT_F32 ? 4 : 2))
    return set_error(UFP8_ERR_ALIGN, "%s: dlogits not aligned to their type", who);
  if (x->rows == 0) return UFP8_OK;
  if (!stats || !dlogits || !dloss) return set_error(UFP8_ERR_INVALID, "%s: null stats, dloss or dlogits", who);
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
  return x->dtype == UFP8_OUT_F32 ? launch_grad<F32, true>(a, *dev, s) : launch_grad<Bf16, true>(a, *dev, s);
}
