// Log probabilities of given tokens with entropy and the most likely alternatives, and the gradient of both sums.
//
//   l = sum e^(z - m),  logprob = (z_y - m) - log l,  entropy = log l - sum (z - m) e^(z - m) / l      (m: the row's maximum)
//   dz_v = g_lp (1[v = y] - p_v) - g_H p_v (log p_v + H)
//
// Forward is one pass over the logits: a warp takes segments of 512 consecutive logits, every lane carries its own (m, l, sum) and
// rescales them when a segment brings a larger maximum; the maximum of each segment is kept. The k largest logits lie in the k
// segments that come first by (maximum, lowest index), so only those are read again (from L2). Bound by HBM for many rows; for few
// rows a cluster of up to 8 CTAs shares a row and joins its parts through distributed shared memory.
// The backward pass reads the logits once more and writes their gradient: HBM-bound.
// The reference computes losses only (fla/modules/fused_linear_cross_entropy.py:516-679); it has no per-token scores.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include "sm100.cuh"
#include "host_utils.h"

namespace cg = cooperative_groups;

namespace hippo {
constexpr int kLpThreads = 512, kLpWarps = kLpThreads / 32, kSeg = 512, kPerLane = kSeg / 32;
constexpr int kMaxSegs = 1024, kCand = 1024, kMaxTop = 32;
constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float lp_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float lp_lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// Order of the values as signed integers; -0 counts as 0, every NaN as the largest.
__device__ __forceinline__ int order_key(float x) {
  const int b = __float_as_int(x + 0.f);
  if ((b & 0x7fffffff) > 0x7f800000) return 0x7fffffff;
  return b < 0 ? b ^ 0x7fffffff : b;
}

// 8 consecutive logits
__device__ __forceinline__ void load8(const float* p, float* f) {
  const float4 a = __ldg((const float4*)p), b = __ldg((const float4*)p + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* f) {
  const uint4 a = __ldg((const uint4*)p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void load8(const __half* p, float* f) {
  const uint4 a = __ldg((const uint4*)p);
  const __half2* h = (const __half2*)&a;
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 v = __half22float2(h[i]); f[2 * i] = v.x; f[2 * i + 1] = v.y; }
}
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

struct LpArgs {
  const void* z; long long ld; long long rows; int V;
  const long long* ids; int top;
  float *logprob, *entropy; float2* stat; float* top_lp; long long* top_id;   // stat: (m, log l), not their sum: m may swallow log l
};

__device__ __forceinline__ float log_prob(float z, float2 ml) { return ml.x == -INFINITY ? -INFINITY : (z - ml.x) - ml.y; }

struct LpStat { float m, l, s; };                    // maximum, sum of e^(z - m), sum of (z - m) log2(e) e^(z - m)
__device__ __forceinline__ LpStat lp_join(LpStat a, LpStat b) {
  LpStat r;
  r.m = (a.m != a.m || b.m != b.m) ? __int_as_float(0x7fffffff) : fmaxf(a.m, b.m);
  if (r.m == -INFINITY) { r.l = r.s = 0.f; return r; }
  const float da = (a.m - r.m) * kL2e, db = (b.m - r.m) * kL2e;
  const float pa = lp_ex2(da), pb = lp_ex2(db);
  r.l = a.l * pa + b.l * pb;
  // a part of weight 0 leaves nothing (its distance may be infinite)
  r.s = (pa == 0.f ? 0.f : pa * (a.s + da * a.l)) + (pb == 0.f ? 0.f : pb * (b.s + db * b.l));
  return r;
}

// A row is cut in vectors of 8 from the aligned address at or before its start: index v of that grid is logit v - skew. What lies
// outside [0, V) is not read and counts as -inf.
template <typename T> __device__ __forceinline__ void load_row8(const T* base, int skew, int V, int v, float* f) {
  if (v >= skew && v + 8 <= skew + V) { load8(base + v, f); return; }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (v + i >= skew && v + i < skew + V) ? to_f(base[v + i]) : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(LpArgs a) {
  cg::cluster_group cl = cg::this_cluster();
  const int part = (int)cl.block_rank(), parts = (int)cl.num_blocks();
  const long long row = blockIdx.x / parts;
  __shared__ int s_seg[kMaxSegs];                    // order keys of the segments' maxima (of all parts, in part 0)
  __shared__ LpStat s_stat[kLpWarps], s_part[8];
  __shared__ int s_pick[kMaxTop];
  __shared__ unsigned long long s_cand[kCand];
  __shared__ int s_n, s_floor;
  __shared__ float2 s_ml;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const T* z = (const T*)a.z + row * a.ld;
  const int skew = (int)(((uintptr_t)z & 15) / sizeof(T)) & 7;
  const T* base = z - skew;
  const int segs = (skew + a.V + kSeg - 1) / kSeg;
  int* seg0 = cl.map_shared_rank(s_seg, 0);
  if (parts > 1) cl.sync();                          // part 0 runs: its shared memory may be written

  LpStat st{-INFINITY, 0.f, 0.f};
  for (int g = part * kLpWarps + w; g < segs; g += parts * kLpWarps) {
    float f[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane / 8; ++i) load_row8(base, skew, a.V, g * kSeg + i * 256 + lane * 8, f + 8 * i);
    float mx = f[0];
    bool nan = f[0] != f[0];
#pragma unroll
    for (int i = 1; i < kPerLane; ++i) { mx = fmaxf(mx, f[i]); nan |= f[i] != f[i]; }
    if (nan) mx = __int_as_float(0x7fffffff);
    if (a.top > 0) {
      const int k = __reduce_max_sync(0xffffffffu, order_key(mx));
      if (lane == 0) seg0[g] = k;
    }
    if (mx > st.m || mx != mx) {
      const LpStat old = st;
      st.m = mx;
      const float d = (old.m - mx) * kL2e, p = lp_ex2(d);
      st.l = old.l * p;
      st.s = p == 0.f ? 0.f : p * (old.s + d * old.l);
    }
    if (st.m == -INFINITY) continue;
    const float off = st.m;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const float d = (f[i] - off) * kL2e, p = lp_ex2(d);
      st.l += p;
      st.s += p == 0.f ? 0.f : p * d;
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    LpStat o;
    o.m = __shfl_xor_sync(0xffffffffu, st.m, d);
    o.l = __shfl_xor_sync(0xffffffffu, st.l, d);
    o.s = __shfl_xor_sync(0xffffffffu, st.s, d);
    st = lp_join(st, o);
  }
  if (lane == 0) s_stat[w] = st;
  if (tid == 0) s_n = 0;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kLpWarps; ++i) st = lp_join(st, s_stat[i]);
    *cl.map_shared_rank(&s_part[part], 0) = st;
  }
  cl.sync();
  if (part) return;                                  // part 0 has everything and reads no other block's memory from here on
  if (tid == 0) {
    st = s_part[0];
    for (int i = 1; i < parts; ++i) st = lp_join(st, s_part[i]);
    const float2 ml = make_float2(st.m, lp_lg2(st.l) * kLn2);
    const long long y = a.ids[row];
    a.logprob[row] = y >= 0 && y < a.V ? log_prob(to_f(z[y]), ml) : 0.f;
    a.entropy[row] = st.m == -INFINITY ? 0.f : ml.y - st.s / st.l * kLn2;
    a.stat[row] = ml;
    s_ml = ml;
  }
  if (a.top == 0) return;
  // the first `top` segments by (maximum, lowest index): one warp, keys in registers, a round each
  const int want = min(a.top, segs);
  if (w == 0) {
    int key[kMaxSegs / 32];
    unsigned taken = 0;
#pragma unroll
    for (int i = 0; i < kMaxSegs / 32; ++i) key[i] = i * 32 + lane < segs ? s_seg[i * 32 + lane] : (int)0x80000000;
    for (int r = 0; r < want; ++r) {
      int best = (int)0x80000000, at = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < kMaxSegs / 32; ++i)
        if (!(taken >> i & 1) && i * 32 + lane < segs && (key[i] > best || at == 0x7fffffff)) { best = key[i]; at = i * 32 + lane; }
      const int top = __reduce_max_sync(0xffffffffu, best);
      const int win = __reduce_min_sync(0xffffffffu, best == top ? at : 0x7fffffff);
      if (at == win) taken |= 1u << (win >> 5);
      if (lane == 0) { s_pick[r] = win; s_floor = top; }
    }
  }
  __syncthreads();
  // candidates: logits of those segments that reach the smallest of their maxima (fewer segments than `top`: all logits)
  const int floor_key = want < a.top ? (int)0x80000000 : s_floor;
  for (int r = w; r < want; r += kLpWarps) {
    const int g = s_pick[r];
#pragma unroll
    for (int i = 0; i < kPerLane / 8; ++i) {
      float f[8];
      const int v = g * kSeg + i * 256 + lane * 8;
      load_row8(base, skew, a.V, v, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = order_key(f[j]);
        if (v + j >= skew && v + j < skew + a.V && k >= floor_key) {
          const int at = atomicAdd(&s_n, 1);         // the order of arrival does not matter: candidates are ranked below
          if (at < kCand) s_cand[at] = ((unsigned long long)((unsigned)k ^ 0x80000000u) << 32) | (0xffffffffu - (unsigned)(v + j - skew));
        }
      }
    }
  }
  __syncthreads();
  const float2 ml = s_ml;
  const int n = s_n;
  if (n <= kCand) {
    // rank = number of candidates before this one in (value, lowest index) order; all are different
    for (int i = tid; i < n; i += kLpThreads) {
      const unsigned long long c = s_cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += s_cand[j] > c;
      if (rank < a.top) {
        const unsigned v = 0xffffffffu - (unsigned)c;
        a.top_id[row * a.top + rank] = v;
        a.top_lp[row * a.top + rank] = log_prob(to_f(z[v]), ml);
      }
    }
    return;
  }
  // Many equal logits (a row of constants): a round for each alternative, the next key below the last one. No list, exact.
  unsigned long long below = ~0ull;
  for (int r = 0; r < a.top; ++r) {
    unsigned long long best = 0;
    for (int q = w; q < want; q += kLpWarps)
      for (int i = 0; i < kPerLane / 8; ++i) {
        float f[8];
        const int v = s_pick[q] * kSeg + i * 256 + lane * 8;
        load_row8(base, skew, a.V, v, f);
        for (int j = 0; j < 8; ++j) {
          if (v + j < skew || v + j >= skew + a.V) continue;
          const unsigned long long c = ((unsigned long long)((unsigned)order_key(f[j]) ^ 0x80000000u) << 32) | (0xffffffffu - (unsigned)(v + j - skew));
          if (c < below && c > best) best = c;
        }
      }
    for (int d = 16; d; d >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, d);
      if (o > best) best = o;
    }
    if (lane == 0) s_cand[w] = best;
    __syncthreads();
    for (int i = 0; i < kLpWarps; ++i) if (s_cand[i] > best) best = s_cand[i];
    __syncthreads();
    below = best;
    if (tid == 0) {
      const unsigned v = 0xffffffffu - (unsigned)best;
      a.top_id[row * a.top + r] = v;
      a.top_lp[row * a.top + r] = log_prob(to_f(z[v]), ml);
    }
  }
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
  const int skew = (int)(((uintptr_t)z & 15) / sizeof(T)) & 7;
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
    float f[8];
    load_row8(base, skew, a.V, v, f);
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

template <typename T> int launch_logprobs(const LpArgs& a, int parts, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * parts));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a);
}
template <typename T> int launch_grad(const LpGradArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)a.rows, (unsigned)((a.V + 7 + kGradChunk - 1) / kGradChunk));
  token_logprobs_grad_kernel<T><<<grid, kGradThreads, 0, st>>>(a);
  return (int)cudaGetLastError();
}
}  // namespace hippo

using namespace hippo;

// logits [rows][V] (row pitch ld elements), dtype 0 bf16, 1 fp16, 2 fp32; out fp32 [rows] logprob, entropy, [rows][2] stat; with top > 0
// top_lp [rows][top], top_id [rows][top].
extern "C" int hippo_token_logprobs(const void* z, int dtype, long long ld, long long rows, int V, const long long* ids, int top,
                                    float* logprob, float* entropy, float* stat, float* top_lp, long long* top_id, void* stream) {
  if (rows <= 0) return 0;
  if (V < 1 || V > (kMaxSegs - 1) * kSeg || top < 0 || top > kMaxTop || top > V || rows > 0x0fffffffll) return -1;
  LpArgs a{z, ld, rows, V, ids, top, logprob, entropy, (float2*)stat, top_lp, top_id};
  // parts of a row: as many CTAs as fill the card once, but no part below one segment a warp
  int parts = 1;
  while (parts < 8 && rows * parts * 2 <= 2 * sm_count() && V >= parts * 2 * kLpWarps * kSeg) parts *= 2;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == 0) return launch_logprobs<__nv_bfloat16>(a, parts, st);
  if (dtype == 1) return launch_logprobs<__half>(a, parts, st);
  if (dtype == 2) return launch_logprobs<float>(a, parts, st);
  return -1;
}

extern "C" int hippo_token_logprobs_grad(const void* z, int dtype, long long ld, long long rows, int V, const long long* ids,
                                         const float* stat, const float* entropy, const float* g_lp, const float* g_h, void* dz,
                                         void* stream) {
  if (rows <= 0) return 0;
  if (V < 1 || rows > 0x7fffffffll) return -1;
  LpGradArgs a{z, ld, rows, V, ids, (const float2*)stat, entropy, g_lp, g_h, dz};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == 0) return launch_grad<__nv_bfloat16>(a, st);
  if (dtype == 1) return launch_grad<__half>(a, st);
  if (dtype == 2) return launch_grad<float>(a, st);
  return -1;
}
