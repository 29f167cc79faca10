// Log probabilities of given tokens with entropy and the most likely alternatives, and the gradient of both sums.
//
//   l = sum e^(z - m),  logprob = (z_y - m) - log l,  entropy = log l - sum (z - m) e^(z - m) / l      (m: the row's maximum)
//   dz_v = g_lp (1[v = y] - p_v) - g_H p_v (log p_v + H)
//
// Forward is one pass over the logits: a warp takes segments of 1024 consecutive logits (512 in fp32), the next one in flight while
// it works; every lane carries its own (m, l, sum) and rescales them when a segment brings a larger maximum. With 16-bit logits
// instructions are as near a bound as HBM (an exponential a logit is 11.6 of the 16 a clock that a multiprocessor has, at the
// card's copy rate), so maximum and clamp work on packed pairs, sums and products on fp32 pairs, and the row's ragged ends have a
// path of their own. For the alternatives the maximum of every granule (8, 64 or 512 consecutive logits, by the vocabulary) is
// kept: the k largest logits lie in the k granules that come first by (maximum, lowest index), so only those are read again (from
// L2). One warp finds the k-th largest maximum bit by bit (a count over its lanes each; 16-bit logits have 16 or 19 bits to
// find). With few rows a cluster of up to 8 blocks shares a row and joins its parts through distributed shared memory. (Blocks that
// stay, with a warp of their own for the alternatives of the row before, were slower: 359 against 242 us for 4096 x 128256 and
// k = 20, as that warp shares its multiprocessor's issue slots.)
// The backward pass reads the logits once more and writes their gradient: HBM-bound.
// Measured (device time, bf16): 4096 x 128256 without alternatives 157 us = 6.7 TB/s, with 5 178, with 20 186 (after seconds of load,
// under the power limit, 177, 179 to 204 and 191 to 196); 8 x 128256 with 5 7.0 us; 3001 x 32000 fp32 forward and backward 195 us =
// 5.9 TB/s of 1.15 GB.
// The reference computes losses only (fla/modules/fused_linear_cross_entropy.py:516-679); it has no per-token scores.
#include <cooperative_groups.h>
#include <type_traits>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include "sm100.cuh"
#include "host_utils.h"
#include "token_logprobs_launch.h"

namespace cg = cooperative_groups;

namespace hippo {
constexpr int kLpThreads = kLpWarps * 32;            // at most
constexpr int kMaxGranules = 1024, kCand = 1024, kMaxTop = 32;
constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float lp_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float lp_lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// two fp32 in one register pair
__device__ __forceinline__ uint64_t pack(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpack(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

// Order of the values as signed integers; -0 counts as 0, every NaN as the largest.
__device__ __forceinline__ int order_key(float x) {
  const int b = __float_as_int(x + 0.f);
  if ((b & 0x7fffffff) > 0x7f800000) return 0x7fffffff;               // (-inf is far above the smallest integer)
  return b < 0 ? b ^ 0x7fffffff : b;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

__device__ __forceinline__ float key_value(int k) { return __int_as_float(k < 0 ? k ^ 0x7fffffff : k); }

// 8 consecutive logits as they are loaded. max(): the largest, NaN if there is one. clamp(lo): what is below lo (far below the
// maximum: its exponential is 0) or NaN becomes lo. kLow: maxima above it leave room for such a lo.
template <typename T> struct Vec8;
template <> struct Vec8<float> {
  float f[8];
  static constexpr float kLow = -1e38f;
  __device__ void load(const float* p) {
    const float4 a = __ldg((const float4*)p), b = __ldg((const float4*)p + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  __device__ void set(int i, float x) { f[i] = x; }
  __device__ void fill(float x) { for (int i = 0; i < 8; ++i) f[i] = x; }
  __device__ float max() const {
    float m = f[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(f[i]));
    return m;
  }
  __device__ void clamp(float lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fmaxf(f[i], lo);
  }
  __device__ void get(float* o) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = f[i];
  }
};
template <> struct Vec8<__nv_bfloat16> {
  __nv_bfloat162 h[4];
  static constexpr float kLow = -1e38f;
  __device__ void load(const __nv_bfloat16* p) { *(uint4*)h = __ldg((const uint4*)p); }
  __device__ void set(int i, __nv_bfloat16 x) { if (i & 1) h[i >> 1].y = x; else h[i >> 1].x = x; }
  __device__ void fill(float x) { for (int i = 0; i < 4; ++i) h[i] = __float2bfloat162_rn(x); }
  __device__ float max() const {
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __bfloat162float(__hmax_nan(m.x, m.y));
  }
  __device__ void clamp(float lo) {
    const __nv_bfloat162 l = __bfloat162bfloat162(__float2bfloat16_rd(lo));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2(h[i], l);
  }
  __device__ void get(float* o) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = *(const uint32_t*)&h[i];
      o[2 * i] = __uint_as_float(w << 16);
      o[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
    }
  }
};
template <> struct Vec8<__half> {
  __half2 h[4];
  static constexpr float kLow = -6e4f;
  __device__ void load(const __half* p) { *(uint4*)h = __ldg((const uint4*)p); }
  __device__ void set(int i, __half x) { if (i & 1) h[i >> 1].y = x; else h[i >> 1].x = x; }
  __device__ void fill(float x) { for (int i = 0; i < 4; ++i) h[i] = __float2half2_rn(x); }
  __device__ float max() const {
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __half2float(__hmax_nan(m.x, m.y));
  }
  __device__ void clamp(float lo) {
    const __half2 l = __half2half2(__float2half_rd(lo));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2(h[i], l);
  }
  __device__ void get(float* o) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 v = __half22float2(h[i]); o[2 * i] = v.x; o[2 * i + 1] = v.y; }
  }
};

struct LpArgs {
  const void* z; long long ld; long long rows; int V;
  const long long* ids; int top;
  float *logprob, *entropy; float2* stat; float* top_lp; long long* top_id;   // stat: (m, log l), not their sum: m may swallow log l
};

__device__ __forceinline__ float log_prob(float z, float2 ml) { return ml.x == -INFINITY ? -INFINITY : (z - ml.x) - ml.y; }

struct LpStat { float m, l, s; };                    // maximum, sum of e^(z - m), sum of (z - m) log2(e) e^(z - m)
// A row is cut in vectors of 8 from the aligned address at or before its start: index v of that grid is logit v - skew. What lies
// outside [0, V) is not read and counts as -inf.
template <typename T> __device__ __forceinline__ void load_vec(const T* base, int skew, int V, int v, Vec8<T>& x) {
  if (v >= skew && v + 8 <= skew + V) { x.load(base + v); return; }
  x.fill(-INFINITY);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (v + i >= skew && v + i < skew + V) x.set(i, base[v + i]);
}

// Joins NV vectors with maximum mx (NaN if one is NaN) to a lane's statistics.
template <typename T, int NV> __device__ __forceinline__ void lp_add(LpStat& st, Vec8<T> (&x)[NV], float mx) {
  if (mx > st.m || mx != mx) {
    const float d = (st.m - mx) * kL2e, p = lp_ex2(d);
    st.m = mx;
    st.s = p == 0.f ? 0.f : p * (st.s + d * st.l);
    st.l *= p;
  }
  if (!(st.m > Vec8<T>::kLow)) {                     // masked by the type's lowest values, or nothing yet, or NaN: one at a time
    if (st.m == -INFINITY) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8];
      x[i].get(f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = fmaxf((f[j] - st.m) * kL2e, -200.f), p = lp_ex2(d);
        st.l += p;
        st.s += p * d;
      }
    }
    return;
  }
  // below the clamp (z - m) log2(e) stays finite and its exponential is 0 all the same
  const float lo = st.m - fmaxf(104.f, fabsf(st.m) * 0.015625f);
  const uint64_t off = pack(-st.m, -st.m), l2e = pack(kL2e, kL2e);
  uint64_t l2[2] = {0, 0}, s2[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    x[i].clamp(lo);
    float f[8];
    x[i].get(f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t d = mul2(add2(pack(f[2 * j], f[2 * j + 1]), off), l2e);
      float d0, d1;
      unpack(d, d0, d1);
      const uint64_t p = pack(lp_ex2(d0), lp_ex2(d1));
      l2[j & 1] = add2(l2[j & 1], p);
      s2[j & 1] = fma2(p, d, s2[j & 1]);
    }
  }
  float u, v;
  unpack(add2(l2[0], l2[1]), u, v);
  st.l += u + v;
  unpack(add2(s2[0], s2[1]), u, v);
  st.s += u + v;
}

// candidates are ordered by (value, lowest index) as one whole number
__device__ __forceinline__ unsigned long long cand_of(int key, int index) {
  return ((unsigned long long)((unsigned)key ^ 0x80000000u) << 32) | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ unsigned cand_index(unsigned long long c) { return 0xffffffffu - (unsigned)c; }

// A row of logits as its readers see it.
template <typename T> struct LpRow {
  const T *z, *base;
  int skew, span, segs, inner0, inner1;              // segments; those from inner0 up to inner1 lie inside the row
  static constexpr int NV = sizeof(T) == 2 ? 4 : 2, kSeg = NV * 256;       // vectors a lane, logits a segment
  __device__ LpRow(const LpArgs& a, long long row) {
    z = (const T*)a.z + row * a.ld;
    skew = (int)(((uintptr_t)z & 15) / sizeof(T));
    base = z - skew;
    span = skew + a.V;
    segs = (span + kSeg - 1) / kSeg;
    inner0 = skew ? 1 : 0;
    inner1 = span / kSeg;
  }
  __device__ void load(int g, Vec8<T> (&x)[NV]) const {
    const int v = g * kSeg + (threadIdx.x & 31) * 8;
    if (g >= inner0 && g < inner1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) x[i].load(base + v + i * 256);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) load_vec(base, skew, span - skew, v + i * 256, x[i]);
    }
  }
};

// One segment: statistics of the lane, the granules' maxima. GR: logits a granule (0: no alternatives are asked for).
template <typename T, int GR> __device__ __forceinline__ void lp_segment(const LpRow<T>& r, int g, Vec8<T> (&x)[LpRow<T>::NV], LpStat& st, float* gran) {
  constexpr int NV = LpRow<T>::NV, kSeg = LpRow<T>::kSeg;
  const int lane = threadIdx.x & 31;
  float m[NV], mx;
#pragma unroll
  for (int i = 0; i < NV; ++i) m[i] = x[i].max();
  mx = m[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(mx) : "f"(m[i]));
  if constexpr (GR == 512) {
#pragma unroll
    for (int i = 0; i < NV; i += 2) {
      float k;
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(k) : "f"(m[i]), "f"(m[i + 1]));
      asm("redux.sync.max.NaN.f32 %0, %0, 0xffffffff;" : "+f"(k));
      if (lane == 0) gran[g * (kSeg / 512) + i / 2] = k;               // (behind the row's last granule: -inf)
    }
  } else if constexpr (GR > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float k = m[i];
      if (GR == 64)
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) asm("max.NaN.f32 %0, %0, %1;" : "+f"(k) : "f"(__shfl_xor_sync(0xffffffffu, k, d)));
      const int at = g * (kSeg / GR) + (i * 256 + lane * 8) / GR;
      if (lane % (GR / 8) == 0 && at * GR < r.span) gran[at] = k;
    }
  }
  lp_add<T, NV>(st, x, mx);
}

__device__ __forceinline__ LpStat lp_warp_join(LpStat st) {
  const float m = key_value(__reduce_max_sync(0xffffffffu, order_key(st.m)));
  const float d = (st.m - m) * kL2e, p = m == -INFINITY ? 0.f : lp_ex2(d);
  // a part of weight 0 leaves nothing (its distance may be infinite)
  float l = st.l * p, s = p == 0.f ? 0.f : p * (st.s + d * st.l);
#pragma unroll
  for (int k = 16; k; k >>= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, k);
    s += __shfl_xor_sync(0xffffffffu, s, k);
  }
  return {m, l, s};
}

// What a row gets from its statistics and the logit of its token; returns (m, log l).
__device__ __forceinline__ float2 lp_finish(const LpArgs& a, long long row, bool scored, float zy, LpStat st) {
  const float2 ml = make_float2(st.m, lp_lg2(st.l) * kLn2);
  a.logprob[row] = scored ? log_prob(zy, ml) : 0.f;
  a.entropy[row] = st.m == -INFINITY ? 0.f : ml.y - st.s / st.l * kLn2;
  if (a.stat) a.stat[row] = ml;
  return ml;
}

struct LpSelect {
  int pick[kMaxTop];
  unsigned long long cand[kCand];
  int n;
  unsigned floor;
};

// The alternatives of a row from the maxima of its granules, by the whole block.
template <typename T, int GR>
__device__ __forceinline__ void lp_select(const LpArgs& a, long long row, const LpRow<T>& r, const float* gran, LpSelect& s, const float2& s_ml) {
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, w = tid >> 5, warps = threads >> 5;
  const int grans = (r.span + GR - 1) / GR, want = min(a.top, grans);
  // keys as unsigned integers without the low bits that this type's values never differ in
  constexpr int kShift = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;
  if (w == 0) {
    auto pick = [&](auto count) {
      constexpr int K = decltype(count)::value;
      unsigned key[K], t = 0;                        // of granules lane, lane + 32, ...; 0 is below every key
#pragma unroll
      for (int i = 0; i < K; ++i) key[i] = i * 32 + lane < grans ? ((unsigned)order_key(gran[i * 32 + lane]) ^ 0x80000000u) >> kShift : 0u;
      // t: the largest number that `want` keys reach, or a smaller one that exactly `want` keys reach; it begins like all keys do
      unsigned most = key[0], least = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < K; ++i) {
        most = max(most, key[i]);
        least = min(least, i * 32 + lane < grans ? key[i] : 0xffffffffu);
      }
      most = __reduce_max_sync(0xffffffffu, most);
      least = __reduce_min_sync(0xffffffffu, least);
      int reach = grans, bit = 31 - __clz(most ^ least);               // -1 where all are equal
      t = bit < 0 ? most : most & ~((2u << bit) - 1);
      while (bit >= 0 && reach != want) {            // two bits a round: three numbers to try, their counts side by side
        const int low = bit ? bit - 1 : 0;
        const unsigned c1 = t | 1u << low, c2 = bit ? t | 1u << bit : 0xffffffffu, c3 = c2 | 1u << low;
        unsigned n1 = 0, n23 = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) {
          n1 += key[i] >= c1;
          n23 += (key[i] >= c2 ? 1u : 0u) + (key[i] >= c3 ? 0x10000u : 0u);
        }
        n1 = __reduce_add_sync(0xffffffffu, n1);
        n23 = __reduce_add_sync(0xffffffffu, n23);
        const int r3 = bit ? (int)(n23 >> 16) : 0, r2 = bit ? (int)(n23 & 0xffffu) : 0, r1 = (int)n1;
        if (r3 >= want) { t = c3; reach = r3; }
        else if (r2 >= want) { t = c2; reach = r2; }
        else if (r1 >= want) { t = c1; reach = r1; }
        bit -= 2;
      }
      // keys above t (where exactly `want` reach it: from t on), lane by lane
      const bool exact = reach == want;
      int mine = 0;
#pragma unroll
      for (int i = 0; i < K; ++i) mine += key[i] > t || (exact && key[i] == t && i * 32 + lane < grans);
      int at = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, at, d);
        if (lane >= d) at += y;
      }
      const int above = __shfl_sync(0xffffffffu, at, 31);
      at -= mine;
#pragma unroll
      for (int i = 0; i < K; ++i)
        if (key[i] > t || (exact && key[i] == t && i * 32 + lane < grans)) s.pick[at++] = i * 32 + lane;
      // then those equal to t by lowest index as long as there is room
      if (!exact) {
        int have = above;
#pragma unroll
        for (int i = 0; i < K; ++i) {
          const bool tie = key[i] == t && i * 32 + lane < grans;
          const unsigned e = __ballot_sync(0xffffffffu, tie);
          const int p = have + __popc(e & ((1u << lane) - 1));
          if (tie && p < want) s.pick[p] = i * 32 + lane;
          have += __popc(e);
          if (have >= want) break;
        }
      }
      if (lane == 0) { s.n = 0; s.floor = t; }
    };
    if (grans <= 256) pick(std::integral_constant<int, 8>()); else pick(std::integral_constant<int, 32>());
  }
  __syncthreads();
  // candidates: logits of those granules that reach the smallest of their maxima (fewer granules than `top`: all logits)
  float floor = -INFINITY;
  if (want == a.top) {
    const int k = (int)((s.floor << kShift) ^ 0x80000000u);          // (a bit pattern between two values is as good a bound)
    floor = key_value(k);
    if (floor != floor) floor = k > 0 ? INFINITY : -INFINITY;        // beyond the infinities
  }
  constexpr int VPG = GR / 8, U = 5;                 // vectors a granule, vectors a thread has in flight
  for (int q0 = 0; q0 < want * VPG; q0 += U * threads) {
    Vec8<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = q0 + u * threads + tid;
      if (q < want * VPG) load_vec(r.base, r.skew, a.V, s.pick[q / VPG] * GR + q % VPG * 8, x[u]);
    }
    unsigned long long hits = 0;                     // bit 8u + j: logit j of vector u
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (q0 + u * threads + tid >= want * VPG || x[u].max() < floor) continue;      // (NaN is not below)
      float f[8];
      x[u].get(f);
      unsigned hit = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) hit |= (f[j] < floor ? 0u : 1u) << j;
      hits |= (unsigned long long)hit << (8 * u);
    }
    for (; hits; hits &= hits - 1) {
      const int b = __ffsll(hits) - 1, q = q0 + (b >> 3) * threads + tid, i = s.pick[q / VPG] * GR + q % VPG * 8 + (b & 7) - r.skew;
      if (i < 0 || i >= a.V) continue;
      const int at = atomicAdd(&s.n, 1);             // the order of arrival does not matter: candidates are ranked below
      if (at < kCand) s.cand[at] = cand_of(order_key(to_f(r.z[i])), i);
    }
  }
  __syncthreads();
  const float2 ml = s_ml;
  auto put = [&](int rank, unsigned long long c) {
    const unsigned v = cand_index(c);
    a.top_id[row * a.top + rank] = v;
    a.top_lp[row * a.top + rank] = log_prob(key_value((int)((unsigned)(c >> 32) ^ 0x80000000u)), ml);
  };
  const int n = s.n;
  if (n <= kCand) {
    // rank: number of candidates before this one (all are different), counted by 8 threads a candidate
    for (int i0 = 0; i0 < n; i0 += threads / 8) {
      const int i = i0 + tid / 8;
      const unsigned long long c = i < n ? s.cand[i] : 0ull;
      int rank = 0;
      for (int j = tid & 7; j < n; j += 8) rank += s.cand[j] > c;
#pragma unroll
      for (int k = 1; k < 8; k <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, k);
      if (i < n && rank < a.top && (tid & 7) == 0) put(rank, c);
    }
    return;
  }
  // Many equal logits (a row of constants): a round for each alternative, the next one below the last. No list, exact.
  unsigned long long below = ~0ull;
  for (int q = 0; q < a.top; ++q) {
    unsigned long long best = 0;
    for (int i = tid; i < want * VPG; i += threads) {
      const int v = s.pick[i / VPG] * GR + i % VPG * 8;
      Vec8<T> x;
      load_vec(r.base, r.skew, a.V, v, x);
      float f[8];
      x.get(f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned long long c = cand_of(order_key(f[j]), v + j - r.skew);
        if (v + j >= r.skew && v + j < r.span && c < below && c > best) best = c;
      }
    }
    for (int d = 16; d; d >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, d);
      if (o > best) best = o;
    }
    __syncthreads();
    if (lane == 0) s.cand[w] = best;
    __syncthreads();
    for (int i = 0; i < warps; ++i)
      if (s.cand[i] > best) best = s.cand[i];
    below = best;
    if (tid == 0) put(q, best);
  }
}

// gridDim.x = rows * blocks of a cluster.
template <typename T, int GR>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(LpArgs a) {
  cg::cluster_group cl = cg::this_cluster();
  const int part = (int)cl.block_rank(), parts = (int)cl.num_blocks();
  const long long row = blockIdx.x / parts;
  __shared__ float s_gran[GR ? kMaxGranules : 1];    // the granules' maxima (of all parts, in part 0)
  __shared__ LpStat s_stat[kLpWarps], s_part[8];
  __shared__ LpSelect s_sel[1];
  __shared__ float2 s_ml;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, warps = blockDim.x >> 5;
  const LpRow<T> r(a, row);
  float* gran0 = GR ? cl.map_shared_rank(s_gran, 0) : nullptr;
  if (parts > 1) cl.sync();                          // part 0 runs: its shared memory may be written
  bool scored = false;
  float zy = 0.f;
  if (part == 0 && w == warps - 1 && lane == 0) {    // the last warp finishes the row; its token's logit is under way from here on
    const long long y = a.ids[row];
    scored = y >= 0 && y < a.V;
    if (scored) zy = to_f(r.z[y]);
  }

  LpStat st{-INFINITY, 0.f, 0.f};
  const int step = parts * warps;
  int g = part * warps + w;
  Vec8<T> next[LpRow<T>::NV];
  if (g < r.segs) r.load(g, next);
  for (; g < r.segs; g += step) {
    Vec8<T> x[LpRow<T>::NV];
#pragma unroll
    for (int i = 0; i < LpRow<T>::NV; ++i) x[i] = next[i];
    if (g + step < r.segs) r.load(g + step, next);
    lp_segment<T, GR>(r, g, x, st, gran0);
  }
  st = lp_warp_join(st);
  if (lane == 0) s_stat[w] = st;
  __syncthreads();
  if (w == warps - 1) {
    st = lane < warps ? s_stat[lane] : LpStat{-INFINITY, 0.f, 0.f};
    st = lp_warp_join(st);
    if (parts > 1 && lane == 0) *cl.map_shared_rank(&s_part[part], 0) = st;
  }
  if (parts > 1) {
    cl.sync();
    if (part) return;                                // part 0 has everything and reads no other block's memory from here on
    if (w == warps - 1) {
      st = lane < parts ? s_part[lane] : LpStat{-INFINITY, 0.f, 0.f};
      st = lp_warp_join(st);
    }
  }
  if (w == warps - 1 && lane == 0) s_ml = lp_finish(a, row, scored, zy, st);
  if constexpr (GR > 0) lp_select<T, GR>(a, row, r, s_gran, s_sel[0], s_ml);
}

struct LpGradArgs {
  const void* z; long long ld; long long rows; int V;
  const long long* ids;
  const float2* stat; const float *entropy, *g_lp, *g_h;           // g_lp or g_h may be null
  void* dz;                                          // [rows][V]
};

__device__ __forceinline__ void store8(float* p, const float* f) {
  ((float4*)p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  ((float4*)p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* f) {
  uint4 o;
  __nv_bfloat162* h = (__nv_bfloat162*)&o;
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  *(uint4*)p = o;
}
__device__ __forceinline__ void store8(__half* p, const float* f) {
  uint4 o;
  __half2* h = (__half2*)&o;
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  *(uint4*)p = o;
}
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }

// grid: (chunks of a row, rows); 256 threads x 2 vectors of 8
constexpr int kGradThreads = 256, kGradVecs = 2, kGradChunk = kGradThreads * kGradVecs * 8;
template <typename T> __global__ void __launch_bounds__(kGradThreads) token_logprobs_grad_kernel(LpGradArgs a) {
  const long long row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.ld;
  T* dz = (T*)a.dz + row * a.V;
  const int skew = (int)(((uintptr_t)z & 15) / sizeof(T));
  const bool aligned = (((uintptr_t)z ^ (uintptr_t)dz) & 15) == 0;
  const T* base = z - skew;
  const float2 ml = a.stat[row];
  const float H = a.entropy[row];
  const bool empty = ml.x == -INFINITY;
  const long long y = a.ids[row];
  const bool scored = y >= 0 && y < a.V;
  const float gl = scored && a.g_lp ? a.g_lp[row] : 0.f, gh = a.g_h ? a.g_h[row] : 0.f;
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int v = blockIdx.y * kGradChunk + u * kGradThreads * 8 + threadIdx.x * 8;
    if (v >= skew + a.V) continue;
    Vec8<T> x;
    load_vec(base, skew, a.V, v, x);
    float f[8];
    x.get(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = (f[i] - ml.x) - ml.y, p = empty ? 0.f : lp_ex2(d * kL2e);
      float r = p == 0.f ? 0.f : -p * (gl + gh * (d + H));           // an impossible token has no share in the entropy
      if (v + i - skew == y && !empty) r += gl;
      f[i] = r;
    }
    if (aligned && v >= skew && v + 8 <= skew + a.V) { store8(dz + (v - skew), f); continue; }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v + i >= skew && v + i < skew + a.V) put(dz + (v + i - skew), f[i]);
  }
}

template <typename T, int GR> int launch_granule(const LpArgs& a, cudaStream_t st) {
  // Parts of a row (a cluster): while a multiprocessor gets three of them at most and every warp 1024 logits. 8 x 128256: 4.2 us
  // with 8 parts, 10.0 with 1; 74 rows 8.6 with 4, 10.0 with 8 (clusters leave gaps); 256 rows 16.0 with 1, 16.7 with 2; 8 x 16000
  // 3.5 with 1, 3.9 with 2.
  const int sms = sm_count();
  int parts = 1;
  while (parts < 8 && a.rows * parts * 2 <= 3ll * sms && a.V >= parts * 2 * kLpWarps * 1024) parts *= 2;
  const int segs = max(1, a.V / parts / LpRow<T>::kSeg);
  const int threads = 32 * logprob_warps(a.rows, parts, segs, sms, a.top > 0);
  if (parts == 1) {
    token_logprobs_kernel<T, GR><<<(unsigned)a.rows, threads, 0, st>>>(a);
    return (int)cudaGetLastError();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * parts));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, GR>, a);
}
template <typename T> int launch_logprobs(const LpArgs& a, cudaStream_t st) {
  // Granules: as large as leaves 7 of them to 4 alternatives. 4096 rows of 32000, 32 alternatives: granules of 512 take 93 us, of 64
  // 109; of 16000, 20 alternatives: 63 against 56; of 2000, 20 alternatives: granules of 64 25 us, of 8 21.
  if (a.top == 0) return launch_granule<T, 0>(a, st);
  if (a.V >= 896 * a.top) return launch_granule<T, 512>(a, st);
  if (a.V >= 112 * a.top) return launch_granule<T, 64>(a, st);
  return launch_granule<T, 8>(a, st);
}
template <typename T> int launch_grad(const LpGradArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)a.rows, (unsigned)((a.V + 7 + kGradChunk - 1) / kGradChunk));
  token_logprobs_grad_kernel<T><<<grid, kGradThreads, 0, st>>>(a);
  return (int)cudaGetLastError();
}
}  // namespace hippo

using namespace hippo;

// logits [rows][V] (row pitch ld elements), dtype 0 bf16, 1 fp16, 2 fp32; out fp32 [rows] logprob, entropy, [rows][2] stat (or null);
// with top > 0 top_lp [rows][top], top_id [rows][top]. One block of arguments, as in kv8.cu.
struct LpCall {
  const void* z; const long long* ids; float *logprob, *entropy, *stat, *top_lp; long long* top_id; void* stream;
  long long ld, rows;
  int V, top, dtype;
};
extern "C" int hippo_token_logprobs(const LpCall* c) {
  if (c->rows <= 0) return 0;
  if (c->V < 1 || c->V > (kMaxGranules - 1) * 512 || c->top < 0 || c->top > kMaxTop || c->top > c->V || c->rows > 0x0fffffffll) return -1;
  LpArgs a{c->z, c->ld, c->rows, c->V, c->ids, c->top, c->logprob, c->entropy, (float2*)c->stat, c->top_lp, c->top_id};
  cudaStream_t st = (cudaStream_t)c->stream;
  if (c->dtype == 0) return launch_logprobs<__nv_bfloat16>(a, st);
  if (c->dtype == 1) return launch_logprobs<__half>(a, st);
  if (c->dtype == 2) return launch_logprobs<float>(a, st);
  return -1;
}

// dz [rows][V] from the gradients of logprob and entropy (either may be null)
struct LpGradCall {
  const void* z; const long long* ids; const float *stat, *entropy, *g_lp, *g_h; void *dz, *stream;
  long long ld, rows;
  int V, dtype;
};
extern "C" int hippo_token_logprobs_grad(const LpGradCall* c) {
  if (c->rows <= 0) return 0;
  if (c->V < 1 || c->rows > 0x7fffffffll) return -1;
  LpGradArgs a{c->z, c->ld, c->rows, c->V, c->ids, (const float2*)c->stat, c->entropy, c->g_lp, c->g_h, c->dz};
  cudaStream_t st = (cudaStream_t)c->stream;
  if (c->dtype == 0) return launch_grad<__nv_bfloat16>(a, st);
  if (c->dtype == 1) return launch_grad<__half>(a, st);
  if (c->dtype == 2) return launch_grad<float>(a, st);
  return -1;
}
