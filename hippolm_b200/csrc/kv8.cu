// 8-bit paged key / value cache: planning (block tables and slot maps) and the quantising write.
//
// Cache: codes [2][blocks][heads][bs][D] (int8 or e4m3; keys, then values), scales [2][blocks][heads] fp32 = 2^e. A value is
// code * scale. With a power of two the scaled value is rounded exactly once (x * 2^-e is exact), and a block whose scale has to
// grow by 2^k only shifts its older codes: exact in e4m3 above the subnormals, one more rounding in int8.
// The reference has no cache (src/models/model.py:180-219 re-runs the forward for every token).
#include <type_traits>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "sm100.cuh"
#include "kv8_common.cuh"

namespace hippo {

// ------------------------------------------------------------------------------------------------ planning
// One CTA of 1024 threads walks the requests 1024 at a time: a thread owns a request, prefix sums over the CTA give the
// positions in the stack of free blocks, in the packed tokens, and decide who still fits. Blocks pushed, blocks popped and slots are
// then dealt out one by one to all threads, which find their request by bisection of the sums in shared memory (a request may
// own one block or hundreds). Released requests push first. The work is a few dependent loads and barriers (latency-bound: 4.2 us for
// 16 requests of a token); more CTAs would need a grid-wide order between pushes and pops.
constexpr int kPlanThreads = 1024, kBatch = 4;        // entries a thread has in flight

__device__ __forceinline__ long long block_inclusive_scan(long long v, long long* warp_sum, long long& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) warp_sum[w] = x;
  __syncthreads();
  if (w == 0) {
    long long s = warp_sum[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += y;
    }
    warp_sum[lane] = s;
  }
  __syncthreads();
  total = warp_sum[31];
  const long long before = w ? warp_sum[w - 1] : 0;
  __syncthreads();                                   // warp_sum is free for the next scan
  return x + before;
}

// slot of the token at position `pos` of a request whose table row is `row`; -1 where the row holds no block there
__device__ __forceinline__ long long slot_of(const int* row, int pos, int sh) {
  const int b = row[pos >> sh];
  return b < 0 ? -1ll : ((long long)b << sh) + (pos & ((1 << sh) - 1));
}

// first index whose sum is above p (the sums ascend, the last one is above p)
__device__ __forceinline__ int owner_of(const int* sum, int p) {
  int lo = 0;
#pragma unroll
  for (int step = kPlanThreads / 2; step; step >>= 1)
    if (sum[lo + step - 1] <= p) lo += step;
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) kv8_plan_kernel(
    int* table, long long table_ld, int M, const int* __restrict__ lens, const int* __restrict__ new_lens, int N,
    int* free_list, int cap, const int* __restrict__ free_count, const unsigned char* __restrict__ release, int sh,
    long long num_tokens, long long* __restrict__ slots, int* __restrict__ lens_out, int* __restrict__ count_out,
    unsigned char* __restrict__ served, int* __restrict__ cu, int write_slots) {
  __shared__ long long warp_sum[32];
  __shared__ int s_sum[kPlanThreads];                // blocks pushed or popped up to and with this request of the chunk
  __shared__ int s_have[kPlanThreads];               // blocks it had
  __shared__ int s_end[kPlanThreads], s_pos[kPlanThreads];      // packed end of its tokens, position of its first one (-1: not served)
  const int tid = threadIdx.x;
  const int bs1 = (1 << sh) - 1;
  const long long room = (long long)M << sh;
  long long count = min(max(*free_count, 0), cap), total;

  if (release) {
    for (int base = 0; base < N; base += kPlanThreads) {
      const int n = base + tid;
      int back = 0;
      if (n < N && release[n]) back = (int)((min((long long)max(lens[n], 0), room) + bs1) >> sh);
      const long long sum = block_inclusive_scan(back, warp_sum, total);
      s_sum[tid] = (int)min(sum, (long long)0x7fffffff);
      __syncthreads();
      // what does not fit the list any more (more blocks than it holds: a table that is not ours) is dropped
      const int push = (int)min(total, cap - count);
      for (int p0 = tid; p0 < push; p0 += kBatch * kPlanThreads) {
        int got[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int p = p0 + i * kPlanThreads;
          if (p >= push) break;
          const int r = owner_of(s_sum, p);
          got[i] = table[(long long)(base + r) * table_ld + p - (r ? s_sum[r - 1] : 0)];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (p0 + i * kPlanThreads < push) free_list[count + p0 + i * kPlanThreads] = got[i];
      }
      count += push;
      __syncthreads();                               // pushes are visible to the pops of every thread; s_sum is free
    }
  }

  long long tokens = 0, asked = 0, used = 0;         // packed tokens, blocks asked for, blocks handed out so far
  for (int base = 0; base < N; base += kPlanThreads) {
    const int n = base + tid;
    const bool in = n < N, gone = in && release && release[n];
    long long len = in && !gone ? min((long long)max(lens[n], 0), room) : 0;
    const int want = in ? max(new_lens[n], 0) : 0;
    const long long end = tokens + block_inclusive_scan(want, warp_sum, total);
    const long long chunk_begin = tokens;
    tokens += total;
    const bool fits = in && !gone && len + want <= room && end <= num_tokens;
    const int have = (int)((len + bs1) >> sh);
    int need = fits ? (int)((len + want + bs1) >> sh) - have : 0;
    const long long top = asked + block_inclusive_scan(need, warp_sum, total);
    asked += total;
    const bool ok = want == 0 || (fits && (need == 0 || top <= count));
    // the requests that get blocks are a prefix of those that ask: their sums without the refused ones are the same
    const long long mine = block_inclusive_scan(ok ? need : 0, warp_sum, total);
    s_sum[tid] = (int)mine;
    s_have[tid] = have;
    s_end[tid] = (int)min(end, num_tokens);
    s_pos[tid] = ok && in ? (int)len : -1;
    if (in) {
      lens_out[n] = (int)(ok ? len + want : len);
      served[n] = ok;
      if (cu) cu[n + 1] = (int)min(end, (long long)0x7fffffff);
    }
    __syncthreads();
    const int pops = (int)total;
    for (int p0 = tid; p0 < pops; p0 += kBatch * kPlanThreads) {
      int got[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (p0 + i * kPlanThreads < pops) got[i] = free_list[count - 1 - used - p0 - i * kPlanThreads];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int p = p0 + i * kPlanThreads;
        if (p >= pops) break;
        const int r = owner_of(s_sum, p);
        table[(long long)(base + r) * table_ld + s_have[r] + p - (r ? s_sum[r - 1] : 0)] = got[i];
      }
    }
    used += pops;
    if (write_slots) {
      __syncthreads();                               // the popped blocks are in the table
      const int last = (int)min(tokens, num_tokens);
      for (int t0 = (int)min(chunk_begin, num_tokens) + tid; t0 < last; t0 += kBatch * kPlanThreads) {
        long long got[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int t = t0 + i * kPlanThreads;
          if (t >= last) break;
          const int r = owner_of(s_end, t), first = r ? s_end[r - 1] : (int)chunk_begin;
          got[i] = s_pos[r] < 0 ? -1ll : slot_of(table + (long long)(base + r) * table_ld, s_pos[r] + t - first, sh);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (t0 + i * kPlanThreads < last) slots[t0 + i * kPlanThreads] = got[i];
      }
    }
    __syncthreads();
  }
  if (write_slots)
    for (long long t = min(tokens, num_tokens) + tid; t < num_tokens; t += kPlanThreads) slots[t] = -1;
  if (tid == 0) {
    if (cu) cu[0] = 0;
    *count_out = (int)(count - used);
  }
}

// Slot map of many tokens (prompts): 4 tokens a thread, the request of the first found in the packed ends, the table rows stay in
// L1. Runs behind the planning kernel, whose single CTA would write 8 bytes a token at one SM's rate: 32 000 tokens 7.6 us with this
// kernel, 19.2 without, 8 192 7.3 and 8.3, 2 048 7.3 and 5.5. The second launch costs the host some 5 us, so that it is taken from
// 16 thousand tokens on, where the device is the longer of the two.
__global__ void __launch_bounds__(256) kv8_slots_kernel(
    const int* __restrict__ table, long long table_ld, const int* __restrict__ lens_out, const unsigned char* __restrict__ served,
    const int* __restrict__ cu, int N, int sh, long long num_tokens, long long* __restrict__ slots) {
  const long long t0 = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (t0 >= num_tokens) return;
  int lo = 0, hi = N;                                // first n with cu[n + 1] > t0, N behind the last token
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t0) hi = mid; else lo = mid + 1;
  }
  int n = lo;
  for (int i = 0; i < 4 && t0 + i < num_tokens; ++i) {
    const long long t = t0 + i;
    while (n < N && cu[n + 1] <= t) ++n;
    long long slot = -1;
    if (n < N && served[n])                          // lens_out counts the new tokens: the last one is at lens_out - 1
      slot = slot_of(table + (long long)n * table_ld, lens_out[n] - (int)(cu[n + 1] - t), sh);
    slots[t] = slot;
  }
}

// ------------------------------------------------------------------------------------------------ write
// 8 consecutive values as they are loaded, and as fp32. amax() joins their sizes to a running maximum of absolute values (as bits,
// infinities and NaN on top; a pair for the 16-bit types); bits() makes fp32 bits of it.
template <typename T> struct Row8;
template <> struct Row8<float> {
  float4 a, b;
  __device__ void load(const float* p) { a = __ldg((const float4*)p); b = __ldg((const float4*)p + 1); }
  __device__ void zero() { a = b = make_float4(0, 0, 0, 0); }
  __device__ void get(float* f) const { f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w; }
  __device__ uint32_t amax(uint32_t m) const {
    float f[8];
    get(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    return m;
  }
  static __device__ uint32_t bits(uint32_t m) { return m; }
};
template <> struct Row8<__nv_bfloat16> {
  uint4 a;
  __device__ void load(const __nv_bfloat16* p) { a = __ldg((const uint4*)p); }
  __device__ void zero() { a = make_uint4(0, 0, 0, 0); }
  __device__ void get(float* f) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  __device__ uint32_t amax(uint32_t m) const {
    const __nv_bfloat162* h = (const __nv_bfloat162*)&a;
    __nv_bfloat162 r = *(const __nv_bfloat162*)&m;
#pragma unroll
    for (int i = 0; i < 4; ++i) r = __hmax2_nan(r, __habs2(h[i]));
    return *(const uint32_t*)&r;
  }
  static __device__ uint32_t bits(uint32_t m) { return max(m & 0xffffu, m >> 16) << 16; }
};
template <> struct Row8<__half> {
  uint4 a;
  __device__ void load(const __half* p) { a = __ldg((const uint4*)p); }
  __device__ void zero() { a = make_uint4(0, 0, 0, 0); }
  __device__ void get(float* f) const {
    const __half2* h = (const __half2*)&a;
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 v = __half22float2(h[i]); f[2 * i] = v.x; f[2 * i + 1] = v.y; }
  }
  __device__ uint32_t amax(uint32_t m) const {
    const __half2* h = (const __half2*)&a;
    __half2 r = *(const __half2*)&m;
#pragma unroll
    for (int i = 0; i < 4; ++i) r = __hmax2_nan(r, __habs2(h[i]));
    return *(const uint32_t*)&r;
  }
  static __device__ uint32_t bits(uint32_t m) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))));
  }
};

// What a run of new tokens does to its (block, head): the exponent of the scale, how far older codes shift, poison.
struct RunScale { int e, down; bool bad; };
template <int E4M3> __device__ __forceinline__ RunScale run_scale(uint32_t amax, float old_scale, bool holds) {
  RunScale r;
  r.bad = amax >= 0x7f800000u || (holds && isnan_bits(old_scale));
  r.e = scale_exponent<E4M3>(r.bad ? 0u : amax);
  r.down = 0;
  if (holds && !r.bad) {
    const int old = max((int)((__float_as_uint(old_scale) >> 23) & 255) - 127, kMinExp);
    r.e = max(r.e, old);
    r.down = old - r.e;
  }
  return r;
}

// older codes of the block shift by 2^down (threads `i` of `step` take 16 bytes each)
template <int E4M3> __device__ __forceinline__ void shift_codes(uint8_t* codes, int bytes, int down, int i, int step) {
  const float f = pow2f(max(down, -126));
  for (int o = i * 16; o < bytes; o += step * 16) {
    uint4 w = *(uint4*)(codes + o);
    uint8_t* c = (uint8_t*)&w;
#pragma unroll
    for (int j = 0; j < 16; ++j) c[j] = encode1<E4M3>(decode1<E4M3>(c[j]) * f);
    *(uint4*)(codes + o) = w;
  }
}

template <int E4M3, typename R> __device__ __forceinline__ uint2 encode_row(const R& r, float inv, bool bad) {
  if (bad) return make_uint2(0, 0);
  float f[8];
  r.get(f);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= inv;
  return encode8<E4M3>(f);
}

struct WriteArgs {
  const void *k, *v;
  long long k_t, k_h, v_t, v_h;                      // strides in elements
  const long long* slots;
  long long T, limit;                                // tokens, blocks * bs
  uint8_t* codes;
  float* scales;
  int H, sh;
  long long half_codes, half_scales;                 // elements of the key half
};

__device__ __forceinline__ bool slot_ok(const WriteArgs& a, long long s) { return s >= 0 && s < a.limit; }
// token t continues the run of token t - 1: the next slot of the same block
__device__ __forceinline__ bool continues(const WriteArgs& a, long long prev, long long s) {
  return slot_ok(a, prev) && s == prev + 1 && (s & ((1 << a.sh) - 1)) != 0;
}

// scale = 2^e with the smallest e under which a run's largest value (and the older ones of its block) fit the codes; code =
// round(x 2^-e). One CTA for the runs that start in a window of W tokens, and for a few (head, half) pairs. It finds the runs
// (consecutive tokens in consecutive slots of one block) by ballots. Runs of up to kShort tokens (decoding: one) go to groups of lanes
// that hold a row, 128 / (D / 8) of them at work, kHeld rows in registers at a time (of a longer one the first are read again, from
// L1); longer runs (prompts) are read once into registers by the whole CTA, the next pair's rows in flight while this one's are
// reduced and stored. With kShort 12 instead of 4, 2000 x 8 tokens of 16 heads of 128 take 42 us, not 78 (196 MB: 4.7 TB/s); with 16,
// the ends of 24 x 1040 cost 2 us more. A single token has a form of its own (2000 x 1, 32 heads: 24.0 us against 26.7 with the one for four).
// HBM and issue slots both bound prompts (24 x 1040 tokens, 16 heads of 128, bf16 -> e4m3: 307 MB in 57.4 us = 5.3 TB/s; issue 65 %),
// latency a token a request (32 x 1, 32 heads: 2.8 us).
constexpr int kShort = 12, kHeld = 4;

template <typename T, int D, int E4M3, int BS> struct WriteShape {
  static constexpr int kBytes = BS * D * (int)sizeof(T);                 // a run at most
  static constexpr int kBlocks = kBytes <= 4096 ? 8 : kBytes <= 8192 ? 7 : kBytes <= 16384 ? 5 : 3;    // what the registers allow
};

template <typename T, int D, int E4M3, int BS>
__global__ void __launch_bounds__(128, WriteShape<T, D, E4M3, BS>::kBlocks) kv8_write_kernel(WriteArgs a, int W, int pairs) {
  constexpr int LPR = D / 8, RPP = 128 / LPR, P = (BS + RPP - 1) / RPP;   // lanes a row, rows a pass, passes
  __shared__ unsigned s_cont[4];                     // bit i: token w0 + i continues the run of the token before it
  __shared__ int s_run[BS], s_n[2];                  // first token | length << 8: short runs from the front, long ones from the back
  __shared__ uint32_t s_max[2][4];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int first = blockIdx.y * pairs, last = min(first + pairs, 2 * a.H);
  const long long w0 = (long long)blockIdx.x * W;
  bool ok = false, cont = false;
  if (tid < W + BS && w0 + tid < a.T) {
    const long long s = a.slots[w0 + tid], prev = w0 + tid > 0 ? a.slots[w0 + tid - 1] : -1;
    ok = slot_ok(a, s);
    cont = ok && continues(a, prev, s);
  }
  const unsigned bc = __ballot_sync(0xffffffffu, cont);
  if (lane == 0) s_cont[w] = bc;
  if (tid < 2) s_n[tid] = 0;
  __syncthreads();
  if (tid < W && ok && !cont) {                      // the first token of a run: consecutive bits behind it
    const unsigned long long c0 = s_cont[0] | ((unsigned long long)s_cont[1] << 32), c1 = s_cont[2] | ((unsigned long long)s_cont[3] << 32);
    const unsigned long long rest = tid == 63 ? c1 : (c0 >> (tid + 1)) | (c1 << (63 - tid));
    const int L = min(~rest ? __ffsll(~rest) : 64, BS);
    if (L <= kShort) s_run[atomicAdd(&s_n[0], 1)] = tid | L << 8;        // (runs are independent: their order does not matter)
    else s_run[BS - 1 - atomicAdd(&s_n[1], 1)] = tid | L << 8;
  }
  __syncthreads();
  const int shorts = s_n[0], longs = s_n[1];
  const int r0 = tid / LPR, col = (tid % LPR) * 8;

  auto source = [&](int pair, long long t) {
    const int h = pair >> 1;
    return pair & 1 ? (const T*)a.v + t * a.v_t + h * a.v_h + col : (const T*)a.k + t * a.k_t + h * a.k_h + col;
  };
  for (int u = r0; u < shorts * (last - first); u += RPP) {
    const int run = s_run[u / (last - first)], pair = first + u % (last - first), L = run >> 8;
    const long long t = w0 + (run & 255), s = a.slots[t];
    const int off = (int)(s & (BS - 1));
    const long long bh = (s >> a.sh) * a.H + (pair >> 1), ld = pair & 1 ? a.v_t : a.k_t;
    float* scale = a.scales + (pair & 1 ? a.half_scales : 0) + bh;
    uint8_t* codes = a.codes + (pair & 1 ? a.half_codes : 0) + bh * BS * D;
    const T* x = source(pair, t);
    const float old = off ? *scale : 0.f;
    const unsigned group = (LPR == 16 ? 0xffffu : 0xffu) << (lane & ~(LPR - 1) & 31);
    auto store = [&](auto held, auto reload) {       // `held` rows in registers at a time; a run of more is read again to be encoded
      constexpr int K = decltype(held)::value;
      constexpr bool kReload = decltype(reload)::value;
      Row8<T> row[K];
      auto load = [&](int i0) {
#pragma unroll
        for (int i = 0; i < K; ++i)
          if (i0 + i < L) row[i].load(x + (i0 + i) * ld); else row[i].zero();
      };
      uint32_t m = 0;
      int i0 = kReload ? (L - 1) / K * K : 0;         // from the last rows, so that the first ones stay in registers
#pragma unroll 1
      for (;; i0 -= K) {
        load(i0);
#pragma unroll
        for (int i = 0; i < K; ++i) m = row[i].amax(m);
        if (!kReload || i0 == 0) break;
      }
      m = Row8<T>::bits(m);
#pragma unroll
      for (int d = 1; d < LPR; d <<= 1) m = max(m, __shfl_xor_sync(group, m, d));
      const RunScale rs = run_scale<E4M3>(m, old, off > 0);
      if (rs.down < 0) shift_codes<E4M3>(codes, off * D, rs.down, tid % LPR, LPR);
      const float inv = pow2f(-rs.e);
#pragma unroll 1
      for (;;) {
#pragma unroll
        for (int i = 0; i < K; ++i)
          if (i0 + i < L) *(uint2*)(codes + (off + i0 + i) * D + col) = encode_row<E4M3>(row[i], inv, rs.bad);
        if (!kReload || (i0 += K) >= L) break;
        load(i0);
      }
      __syncwarp(group);                             // every lane has read the old scale
      if (tid % LPR == 0) *scale = rs.bad ? __uint_as_float(0x7fffffffu) : pow2f(rs.e);
    };
    if (L == 1) store(std::integral_constant<int, 1>(), std::false_type());
    else if (L <= kHeld) store(std::integral_constant<int, kHeld>(), std::false_type());
    else store(std::integral_constant<int, kHeld>(), std::true_type());
  }

  for (int q = 0; q < longs; ++q) {
    const int run = s_run[BS - 1 - q], L = run >> 8;
    const long long t = w0 + (run & 255), s = a.slots[t];
    const int off = (int)(s & (BS - 1));
    const long long block = (s >> a.sh) * a.H;
    Row8<T> next[P];
    float next_old = 0.f;
    const T* xk = source(0, t) + r0 * a.k_t;         // this thread's first row, of head 0
    const T* xv = source(1, t) + r0 * a.v_t;
    auto load = [&](int pair) {
      const T* x = pair & 1 ? xv + (pair >> 1) * a.v_h : xk + (pair >> 1) * a.k_h;
      const long long step = RPP * (pair & 1 ? a.v_t : a.k_t);
#pragma unroll
      for (int p = 0; p < P; ++p, x += step)
        if (r0 + p * RPP < L) next[p].load(x); else next[p].zero();
      if (off) next_old = a.scales[(pair & 1 ? a.half_scales : 0) + block + (pair >> 1)];
    };
    load(first);
    for (int pair = first; pair < last; ++pair) {
      Row8<T> row[P];
#pragma unroll
      for (int p = 0; p < P; ++p) row[p] = next[p];
      const float old = next_old;
      if (pair + 1 < last) load(pair + 1);
      const long long bh = block + (pair >> 1);
      uint8_t* codes = a.codes + (pair & 1 ? a.half_codes : 0) + bh * BS * D;
      uint32_t m = 0;
#pragma unroll
      for (int p = 0; p < P; ++p) m = row[p].amax(m);
      m = __reduce_max_sync(0xffffffffu, Row8<T>::bits(m));
      uint32_t* sm = s_max[pair & 1];                // a warp is at most one pair ahead of the others
      if (lane == 0) sm[w] = m;
      __syncthreads();                               // also: every thread has read the old scale
      m = max(max(sm[0], sm[1]), max(sm[2], sm[3]));
      const RunScale rs = run_scale<E4M3>(m, old, off > 0);
      if (rs.down < 0) shift_codes<E4M3>(codes, off * D, rs.down, tid, 128);
      const float inv = pow2f(-rs.e);
      uint8_t* dst = codes + (off + r0) * D + col;
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (r0 + p * RPP < L) *(uint2*)(dst + p * RPP * D) = encode_row<E4M3>(row[p], inv, rs.bad);
      if (tid == 0) a.scales[(pair & 1 ? a.half_scales : 0) + bh] = rs.bad ? __uint_as_float(0x7fffffffu) : pow2f(rs.e);
    }
    __syncthreads();                                 // s_max is free for the next run
  }
}

template <typename T, int D, int E4M3> int launch_write(const WriteArgs& a, int window, cudaStream_t st) {
  // 2 pairs a block spread few tokens over more of them (32 single tokens 2.9 us against 3.6, 1000 in prompts 8.8 against 11.5),
  // 4 share the search for the runs (25k tokens 57 against 63)
  const int bs = 1 << a.sh, pairs = a.T * a.H <= 32768 ? 2 : 4, groups = (2 * a.H + pairs - 1) / pairs;
  int W = window;
  if (W == 0) {                                      // some two thousand blocks, or a window of a whole block's tokens
    W = 4;                                           // (24 x 1040 tokens 77 us with windows of 4, 58 of 32; 32 x 1 2.8 and 7.6)
    while (W < bs && (a.T + W - 1) / W * groups > 2048) W *= 2;
  }
  if (W < 1 || W > bs) return -1;
  const dim3 grid((unsigned)((a.T + W - 1) / W), (unsigned)groups);
  if (a.sh == 4) kv8_write_kernel<T, D, E4M3, 16><<<grid, 128, 0, st>>>(a, W, pairs);
  else if (a.sh == 5) kv8_write_kernel<T, D, E4M3, 32><<<grid, 128, 0, st>>>(a, W, pairs);
  else kv8_write_kernel<T, D, E4M3, 64><<<grid, 128, 0, st>>>(a, W, pairs);
  return (int)cudaGetLastError();
}
template <typename T> int dispatch_write(const WriteArgs& a, int D, int e4m3, int window, cudaStream_t st) {
  if (D == 128) return e4m3 ? launch_write<T, 128, 1>(a, window, st) : launch_write<T, 128, 0>(a, window, st);
  if (D == 64) return e4m3 ? launch_write<T, 64, 1>(a, window, st) : launch_write<T, 64, 0>(a, window, st);
  return -1;
}
}  // namespace hippo

using namespace hippo;

// Arguments come as one block (a packed struct costs the caller a fifth of converting twenty arguments one by one).

// table [N][M] int32 (row pitch table_ld), lens / new_lens [N], free_list [cap], free_count [1], release [N] or null; out: slots
// [num_tokens], lens_out [N], count_out [1], served [N], cu [N + 1]
// (ends of the packed tokens; null: the planning block writes the slots itself).
struct KvPlanCall {
  int* table; const int *lens, *new_lens; int* free_list; const int* free_count; const unsigned char* release;
  long long* slots; int *lens_out, *count_out; unsigned char* served; int* cu; void* stream;
  long long table_ld, num_tokens;
  int M, N, cap, block_size;
};
extern "C" int hippo_kv8_plan(const KvPlanCall* c) {
  const int sh = c->block_size == 16 ? 4 : c->block_size == 32 ? 5 : c->block_size == 64 ? 6 : -1;
  if (sh < 0 || c->N < 1 || c->M < 1 || c->cap < 1 || c->num_tokens < 0 || c->num_tokens > 0x7fffffffll) return -1;
  const bool many = c->cu != nullptr;
  cudaStream_t st = (cudaStream_t)c->stream;
  kv8_plan_kernel<<<1, kPlanThreads, 0, st>>>(c->table, c->table_ld, c->M, c->lens, c->new_lens, c->N, c->free_list, c->cap,
                                              c->free_count, c->release, sh, c->num_tokens, c->slots, c->lens_out, c->count_out,
                                              c->served, c->cu, many ? 0 : 1);
  const cudaError_t first = cudaGetLastError();
  if (first != cudaSuccess) return (int)first;       // the ends of the tokens and the table are the first kernel's
  if (many)
    kv8_slots_kernel<<<(unsigned)((c->num_tokens + 1023) / 1024), 256, 0, st>>>(c->table, c->table_ld, c->lens_out, c->served,
                                                                                c->cu, c->N, sh, c->num_tokens, c->slots);
  return (int)cudaGetLastError();
}

// k / v: [T][H][D] with strides (elements); dtype 0 bf16, 1 fp16, 2 fp32; codes / scales of `blocks` blocks; window: tokens a
// CTA looks through (1 .. block_size), 0 = by size.
struct KvWriteCall {
  const void *k, *v; const long long* slots; void* codes; float* scales; void* stream;
  long long k_t, k_h, v_t, v_h, T, blocks;
  int H, D, block_size, dtype, e4m3, window;
};
extern "C" int hippo_kv8_write(const KvWriteCall* c) {
  if (c->T <= 0) return 0;
  const int sh = c->block_size == 16 ? 4 : c->block_size == 32 ? 5 : c->block_size == 64 ? 6 : -1;
  if (sh < 0 || c->H < 1 || 2 * c->H > 65535 || c->blocks < 1 || c->T > 0x7fffffffll) return -1;
  WriteArgs a{c->k, c->v, c->k_t, c->k_h, c->v_t, c->v_h, c->slots, c->T, c->blocks << sh, (uint8_t*)c->codes, c->scales, c->H, sh,
              ((c->blocks * c->H) << sh) * c->D, c->blocks * c->H};
  cudaStream_t st = (cudaStream_t)c->stream;
  if (c->dtype == 0) return dispatch_write<__nv_bfloat16>(a, c->D, c->e4m3, c->window, st);
  if (c->dtype == 1) return dispatch_write<__half>(a, c->D, c->e4m3, c->window, st);
  if (c->dtype == 2) return dispatch_write<float>(a, c->D, c->e4m3, c->window, st);
  return -1;
}
