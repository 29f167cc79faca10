// One query token per sequence against the 8-bit paged cache: o = sum_j softmax_j(scale q.k_j) v_j with k_j = s_K code, v_j = s_V code
// and one (s_K, s_V) per (block, kv head).
//
// Bound by HBM: a token and kv head costs 2 D bytes of codes, read once for all query heads that share the kv head. Work is cut in
// tiles of 32 tokens; the tiles of all (sequence, kv head, group of 8 query heads) form one list that is divided evenly over all
// warps of one resident wave, whatever the lengths. A warp streams its tiles through its own TMA ring (no block-wide barrier in the
// loop) and carries the running maximum and sum; a unit that spans several warps leaves partial (m, l, o) rows that a second, small
// kernel joins in the order of the tokens, so results do not depend on timing.
//
// Arithmetic: codes are exact in fp16, so mma.m16n8k16 (fp16 operands, fp32 accumulators) is exact for them; the query and the
// probabilities are split in two fp16 terms that sit in rows 0-7 and 8-15 of the A operand (one thread holds both sums), which keeps
// 21 bits or more of each. Legacy mma is deliberate: with 1 to 8 live rows a 128-row tcgen05 tile would multiply zeros, and the
// kernel waits for memory, not for the tensor pipe.
// In the reference a decoding step re-runs the whole forward (src/models/model.py:180-219).
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include "sm100.cuh"
#include "host_utils.h"
#include "kv8_common.cuh"

namespace hippo {
constexpr int kTile = 32, kWarps = 4, kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;

struct KvAttnArgs {
  const void* q; void* out;
  long long q_n, q_h;                                // query strides in elements; out is [N][Hq][D]
  const float* scales; long long half_scales;
  const int* table; long long table_ld; int M;
  const int* lens;
  int N, H, G, QG, sh, blocks, dtype;                // kv heads, query heads a kv head, groups of 8 of them
  long long half_rows;                               // cache rows (of D bytes) of the key half
  float scale;
  float* part; float* part_ml; int4* desc; int NW, rows;   // parts of `rows` query rows each, two a worker
};

template <int D> struct KvShape {
  static constexpr int kStageBytes = 2 * kTile * D;
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kSmem = kWarps * kWarpBytes + 1024;
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// two codes (bytes 0,1 or 2,3 of w) -> two fp16, exactly. int8 goes through 1024 + (code + 128), whose low byte is the biased code.
template <int E4M3> __device__ __forceinline__ uint32_t codes2(uint32_t w, bool upper) {
  uint32_t r;
  if (E4M3) {
    const uint16_t p = upper ? (uint16_t)(w >> 16) : (uint16_t)w;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(p));
    return r;
  }
  r = __byte_perm(w ^ 0x80808080u, 0x64646464u, upper ? 0x4342 : 0x4140);
  const __half2 h = __hsub2(*(__half2*)&r, __half2half2(__ushort_as_half(0x6480)));          // 1152
  return *(const uint32_t*)&h;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *(const uint32_t*)&h;
  lo = pack2(a - f.x, b - f.y);
}

__device__ __forceinline__ float load_q(const KvAttnArgs& a, long long i) {
  if (a.dtype == 0) return __bfloat162float(((const __nv_bfloat16*)a.q)[i]);
  if (a.dtype == 1) return __half2float(((const __half*)a.q)[i]);
  return ((const float*)a.q)[i];
}
__device__ __forceinline__ void store_out(const KvAttnArgs& a, long long i, float x, float y) {      // elements i, i + 1
  if (a.dtype == 0) ((__nv_bfloat162*)a.out)[i >> 1] = __floats2bfloat162_rn(x, y);
  else if (a.dtype == 1) ((__half2*)a.out)[i >> 1] = __floats2half2_rn(x, y);
  else ((float2*)a.out)[i >> 1] = make_float2(x, y);
}

__device__ __forceinline__ int cached_len(const KvAttnArgs& a, int n) {
  return (int)min((long long)max(a.lens[n], 0), (long long)a.M << a.sh);
}

// Where a warp stands in the list of tiles: sequence, unit = (kv head, group of 8 query heads), tile of the unit.
struct Cursor {
  int n, unit, tile, len, tiles;
  long long left;                                    // tiles of the warp's range that are still ahead, this one included
  __device__ void next_sequence(const KvAttnArgs& a) {
    do { ++n; len = n < a.N ? cached_len(a, n) : 0; } while (n < a.N && len == 0);
    tiles = (len + kTile - 1) / kTile;
  }
  __device__ void advance(const KvAttnArgs& a) {
    --left;
    if (left <= 0) return;
    if (++tile < tiles) return;
    tile = 0;
    if (++unit < a.H * a.QG) return;
    unit = 0;
    next_sequence(a);
  }
};

template <int D, int E4M3>
__global__ void __launch_bounds__(kThreads, 3) kv8_attention_kernel(const __grid_constant__ CUtensorMap codes_map, KvAttnArgs a) {
  using S = KvShape<D>;
  constexpr int KS = D / 16, NT = D / 8;             // k steps of q.k, n tiles of p.v
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kWarps][S::kStages];
  __shared__ float s_scale[kWarps][S::kStages][4];   // K, V scale of the tile's first 16 tokens, K, V of the others
  __shared__ int s_there[kWarps][S::kStages];        // which 16-token groups of the tile lie in a block of the pool
  __shared__ long long s_pre[kThreads + 1];
  __shared__ long long s_warp[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int units = a.H * a.QG;

  // rows of empty sequences
  for (long long i = (long long)blockIdx.x * kThreads + tid; i < (long long)a.N * a.H * a.G * (D / 2); i += (long long)gridDim.x * kThreads) {
    const int n = (int)(i / (a.H * a.G * (D / 2)));
    if (a.lens[n] <= 0) store_out(a, i * 2, 0.f, 0.f);
  }

  // tiles before every thread's share of the sequences
  const int share = (a.N + kThreads - 1) / kThreads;
  long long mine = 0;
  for (int n = tid * share; n < min(a.N, (tid + 1) * share); ++n) mine += (long long)((cached_len(a, n) + kTile - 1) / kTile) * units;
  long long inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) s_warp[w] = inc;
  if (tid == 0) {
    for (int i = 0; i < kWarps; ++i)
      for (int j = 0; j < S::kStages; ++j) mbar_init(&full[i][j], 5);      // TMA bytes + four lanes' scale copies
    fence_barrier_init();
  }
  __syncthreads();
  for (int i = 0; i < w; ++i) inc += s_warp[i];
  s_pre[tid + 1] = inc;
  if (tid == 0) s_pre[0] = 0;
  __syncthreads();
  const long long total = s_pre[kThreads];

  // no more workers than tiles: every part between a unit's first and last worker is then written
  const int worker = blockIdx.x * kWarps + w, nw = (int)min((long long)a.NW, total);
  const long long begin = worker < nw ? total * worker / nw : 0, end = worker < nw ? total * (worker + 1) / nw : 0;
  int4 found = make_int4(-1, 0, 0, 0);               // unit that begins here and ends in a later worker
  uint8_t* ring = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023) + w * S::kWarpBytes;

  if (begin < end) {
    Cursor put;                                      // next tile to fetch
    {
      int lo = 0, hi = kThreads - 1;
      while (lo < hi) { const int mid = (lo + hi) >> 1; if (s_pre[mid + 1] > begin) hi = mid; else lo = mid + 1; }
      long long at = s_pre[lo];
      int n = lo * share;
      for (;;) {                                     // the sequence of the share that holds `begin`
        put.len = cached_len(a, n);
        put.tiles = (put.len + kTile - 1) / kTile;
        const long long c = (long long)put.tiles * units;
        if (at + c > begin) break;
        at += c; ++n;
      }
      put.n = n;
      put.unit = (int)((begin - at) / put.tiles);
      put.tile = (int)((begin - at) - (long long)put.unit * put.tiles);
      put.left = end - begin;
    }
    Cursor get = put;
    // fetching: lanes hold 32 entries of the table row
    int held_n = -1, held_base = 0, held = -1;
    const int box = min(kTile, 1 << a.sh);           // rows of one TMA box
    auto fetch = [&](int stage) {
      const int tok = put.tile * kTile, blk = tok >> a.sh;
      const int base = blk & ~31;                    // a tile never spans two batches of 32 entries (at most 2 blocks, even start)
      if (held_n != put.n || held_base != base) {
        held_n = put.n; held_base = base;
        const int j = base + lane;
        held = j < a.M && ((long long)j << a.sh) < put.len ? a.table[(long long)put.n * a.table_ld + j] : -1;
        if (held >= a.blocks) held = -1;
      }
      const int h = put.unit / a.QG;
      const int b0 = __shfl_sync(0xffffffffu, held, blk - base);
      const int b1 = a.sh == 4 ? __shfl_sync(0xffffffffu, held, (blk + 1 - base) & 31) : b0;
      const bool second = a.sh == 4 && tok + 16 < put.len;          // the tile's second block holds tokens
      const int there = a.sh == 4 ? (b0 >= 0 ? 1 : 0) | (second && b1 >= 0 ? 2 : 0) : (b0 >= 0 ? 3 : 0);
      uint64_t* bar = &full[w][stage];
      uint8_t* dst = ring + stage * S::kStageBytes;
      if (lane == 0) {
        s_there[w][stage] = there;
        const int boxes = a.sh == 4 ? __popc(there) : (there ? 1 : 0);
        mbar_expect_tx(bar, (uint32_t)(boxes * 2 * box * D));
        const int in = tok & ((1 << a.sh) - 1);
        if (there & 1) {
          const int y = (int)((((long long)b0 * a.H + h) << a.sh) + in);
          tma_load_2d(dst, &codes_map, bar, 0, y);
          tma_load_2d(dst + kTile * D, &codes_map, bar, 0, (int)(y + a.half_rows));
        }
        if (a.sh == 4 && (there & 2)) {
          const int y = (int)(((long long)b1 * a.H + h) << a.sh);
          tma_load_2d(dst + 16 * D, &codes_map, bar, 0, y);
          tma_load_2d(dst + kTile * D + 16 * D, &codes_map, bar, 0, (int)(y + a.half_rows));
        }
      }
      if (lane < 4) {
        const int b = lane < 2 ? b0 : b1;
        if (there & (lane < 2 ? 1 : 2)) {
          const float* src = a.scales + (lane & 1) * a.half_scales + (long long)b * a.H + h;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&s_scale[w][stage][lane])), "l"(src) : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
      }
      put.advance(a);
    };
    const int g = lane >> 2, c = lane & 3;           // row of the fragments (query head), column pair
#pragma unroll 1
    for (int i = 0; i < S::kStages; ++i)
      if (put.left > 0) fetch(i);
    __syncwarp();

    uint32_t qf[KS][4];
    float o[NT][4];
    float m = -INFINITY, mv = -INFINITY, l = 0.f, f = 0.f;
    bool alive = true, fresh = true, whole = true, first = true;
    int stage = 0, phase = 0, tile0 = 0;
    long long unit_tile0 = 0;
    while (get.left > 0 && alive) {
      const int n = get.n, unit = get.unit, h = unit / a.QG, g0 = (unit - h * a.QG) * 8;
      if (fresh) {                                   // a new unit: its query rows, normalised to [1, 2) and split in two fp16
        fresh = false;
        tile0 = get.tile;
        unit_tile0 = end - get.left - get.tile;
        whole = get.tile == 0;
        float x[D / 4];
        float top = 0.f;
        const bool row = g0 + g < a.G;
        const long long qi = (long long)n * a.q_n + (long long)(h * a.G + g0 + g) * a.q_h + c * (D / 4);
#pragma unroll
        for (int i = 0; i < D / 4; ++i) x[i] = row ? load_q(a, qi + i) : 0.f;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 126);
        const float down = pow2f(-e);
        f = pow2f(e) * a.scale * kLog2e;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          split2(x[4 * i] * down, x[4 * i + 1] * down, qf[i][0], qf[i][1]);
          split2(x[4 * i + 2] * down, x[4 * i + 3] * down, qf[i][2], qf[i][3]);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m = mv = -INFINITY; l = 0.f;
      }
      if (!mbar_wait(&full[w][stage], phase, kWaitTmaFull, worker)) { alive = false; break; }
      const uint8_t* kt = ring + stage * S::kStageBytes;
      const uint8_t* vt = kt + kTile * D;
      const int there = s_there[w][stage];
      const int valid = min(kTile, get.len - get.tile * kTile);
      const bool ragged = valid < kTile || there != 3;
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
        const int r = j * 8 + g;
#pragma unroll
        for (int q4 = 0; q4 < D / 64; ++q4) {
          const int chunk = D == 128 ? (2 * c + q4) ^ (r & 7) : c ^ ((r >> 1) & 3);
          const uint4 x = *(const uint4*)(kt + r * D + chunk * 16);
          const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mma16816(s[j], qf[q4 * 4 + i], codes2<E4M3>(word[i], false), codes2<E4M3>(word[i], true));
        }
      }
      const float ks0 = s_scale[w][stage][0], vs0 = s_scale[w][stage][1], ks1 = s_scale[w][stage][2], vs1 = s_scale[w][stage][3];
      // log2 of the value scale: whole part and a factor in [1, 2) (1 for the powers of two that the write kernel stores)
      const float ev0 = (float)((int)((__float_as_uint(vs0) >> 23) & 255) - 127), ev1 = (float)((int)((__float_as_uint(vs1) >> 23) & 255) - 127);
      const float fv0 = isnan_bits(vs0) ? vs0 : __uint_as_float((__float_as_uint(vs0) & 0x807fffffu) | 0x3f800000u);
      const float fv1 = isnan_bits(vs1) ? vs1 : __uint_as_float((__float_as_uint(vs1) & 0x807fffffu) | 0x3f800000u);
      float x[8], mx = -INFINITY, mxv = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float y = (s[j][i] + s[j][i + 2]) * (f * (j < 2 ? ks0 : ks1));
          if (ragged && (j * 8 + 2 * c + i >= valid || !(there >> (j >> 1) & 1))) y = -INFINITY;
          x[2 * j + i] = y;
          mx = fmaxf(mx, y);
          mxv = fmaxf(mxv, y + (j < 2 ? ev0 : ev1));
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, 2));
      const float m1 = fmaxf(m, mx), mv1 = fmaxf(mv, mxv);
      const float mu = m1 == -INFINITY ? 0.f : m1, mvu = mv1 == -INFINITY ? 0.f : mv1;
      l *= ex2(m - mu);
      const float alpha = ex2(mv - mvu);
      if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
        for (int i = 0; i < NT; ++i) { o[i][0] *= alpha; o[i][1] *= alpha; o[i][2] *= alpha; o[i][3] *= alpha; }
      }
      m = m1; mv = mv1;
      float p[8];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float y = x[2 * j + i];
          l += ex2(y - mu);
          float pv = ex2(y + (j < 2 ? ev0 : ev1) - mvu) * (j < 2 ? fv0 : fv1);
          if (y == -INFINITY) pv = 0.f;              // a group outside the pool leaves its scales unset
          p[2 * j + i] = pv;
        }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        uint32_t pa[4];
        split2(p[4 * kk], p[4 * kk + 1], pa[0], pa[1]);
        split2(p[4 * kk + 2], p[4 * kk + 3], pa[2], pa[3]);
        constexpr int W = D / 32;                    // 32-bit words a lane reads of a row: D / 8 bytes at column g
        uint32_t v[4][W];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = kk * 16 + 2 * c + (i & 1) + (i >> 1) * 8;
          if (D == 128) {
            const uint4 y = *(const uint4*)(vt + r * D + ((g ^ (r & 7)) * 16));
            v[i][0] = y.x; v[i][1] = y.y; v[i][W - 2] = y.z; v[i][W - 1] = y.w;
          } else {
            const uint2 y = *(const uint2*)(vt + r * D + (((g >> 1) ^ ((r >> 1) & 3)) * 16) + (g & 1) * 8);
            v[i][0] = y.x; v[i][1] = y.y;
          }
          if (ragged && (r >= valid || !(there >> kk & 1))) {       // bytes behind the last token may be NaN codes
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] = 0;
          }
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const uint32_t a01 = __byte_perm(v[0][j], v[1][j], 0x5140), a23 = __byte_perm(v[0][j], v[1][j], 0x7362);
          const uint32_t b01 = __byte_perm(v[2][j], v[3][j], 0x5140), b23 = __byte_perm(v[2][j], v[3][j], 0x7362);
          mma16816(o[4 * j], pa, codes2<E4M3>(a01, false), codes2<E4M3>(b01, false));
          mma16816(o[4 * j + 1], pa, codes2<E4M3>(a01, true), codes2<E4M3>(b01, true));
          mma16816(o[4 * j + 2], pa, codes2<E4M3>(a23, false), codes2<E4M3>(b23, false));
          mma16816(o[4 * j + 3], pa, codes2<E4M3>(a23, true), codes2<E4M3>(b23, true));
        }
      }
      __syncwarp();                                  // every lane has read the stage
      if (put.left > 0) fetch(stage);
      if (++stage == S::kStages) { stage = 0; phase ^= 1; }

      const bool last_of_unit = get.tile + 1 == get.tiles;
      const int tiles = get.tiles;
      get.advance(a);
      if (last_of_unit || get.left <= 0) {           // the unit, or this warp's part of it, is done
        float lt = l + __shfl_xor_sync(0xffffffffu, l, 1);
        lt += __shfl_xor_sync(0xffffffffu, lt, 2);
        const bool row = g0 + g < a.G;
        const float back = lt == 0.f ? 0.f : ex2(mv - m);           // o is held relative to the maximum of p s_V, l to that of p
        if (whole && last_of_unit) {
          const float r = lt == 0.f ? 0.f : back / lt;
          const long long oi = ((long long)n * a.H * a.G + h * a.G + g0 + g) * D + c * (D / 4);
          if (row) {
#pragma unroll
            for (int i = 0; i < NT; i += 2) store_out(a, oi + i, (o[i][0] + o[i][2]) * r, (o[i + 1][0] + o[i + 1][2]) * r);
#pragma unroll
            for (int i = 0; i < NT; i += 2) store_out(a, oi + NT + i, (o[i][1] + o[i][3]) * r, (o[i + 1][1] + o[i + 1][3]) * r);
          }
        } else {
          // a worker has at most two parts: of the unit at its start (slot 0), and of one that begins inside it (slot 1)
          const int sl = worker * 2 + (first ? 0 : 1);
          if (row) {
            float* dst = a.part + ((long long)sl * a.rows + g) * D + c * (D / 4);
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
              *(float2*)(dst + i) = make_float2((o[i][0] + o[i][2]) * back, (o[i + 1][0] + o[i + 1][2]) * back);
              *(float2*)(dst + NT + i) = make_float2((o[i][1] + o[i][3]) * back, (o[i + 1][1] + o[i + 1][3]) * back);
            }
            if (c == 0) *(float2*)(a.part_ml + ((long long)sl * a.rows + g) * 2) = make_float2(m, lt);
          }
          if (whole) {                               // begins here, goes on: this worker's unit to join
            const long long last = unit_tile0 + tiles - 1;
            found = make_int4(n, unit, sl, (int)(last * nw / total));   // the last worker, but for the rounding down of the ranges
            while (total * (found.w + 1) / nw <= last) ++found.w;
            while (total * found.w / nw > last) --found.w;
          }
        }
        fresh = true;
        first = false;
      }
    }
    if (!alive) {                                    // a wait ran out: let the copies in flight land before the block ends
      for (int i = 0; i < S::kStages; ++i) mbar_wait(&full[w][i], phase, kWaitTmaFull, -1);
      found.x = -1;
    }
  }
  if (lane == 0) a.desc[worker] = found;
}

// Joins the parts of the unit that begins in worker blockIdx.x: parts in order, weights 2^(m_i - m).
template <int D> __global__ void __launch_bounds__(128) kv8_join_kernel(KvAttnArgs a) {
  const int4 d = a.desc[blockIdx.x];
  if (d.x < 0) return;
  const int w0 = blockIdx.x, w1 = min(d.w, a.NW - 1), h = d.y / a.QG, g0 = (d.y - h * a.QG) * 8;
  constexpr int TPR = D / 2, ROWS = 128 / TPR;       // two columns a thread
  const int col = (threadIdx.x % TPR) * 2;
  for (int g = threadIdx.x / TPR; g < 8 && g0 + g < a.G; g += ROWS) {
    float m = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
    for (int i = w0; i <= w1; ++i) {
      const long long sl = (long long)(i == w0 ? d.z : 2 * i) * a.rows + g;
      const float2 ml = *(const float2*)(a.part_ml + sl * 2);
      const float2 v = *(const float2*)(a.part + sl * D + col);
      const float m1 = fmaxf(m, ml.x), mu = m1 == -INFINITY ? 0.f : m1;
      const float p = ex2(m - mu), r = ex2(ml.x - mu);
      l = l * p + ml.y * r;
      x = x * p + v.x * r;
      y = y * p + v.y * r;
      m = m1;
    }
    const float r = l == 0.f ? 0.f : 1.f / l;
    store_out(a, ((long long)d.x * a.H * a.G + h * a.G + g0 + g) * D + col, x * r, y * r);
  }
}

template <int D, int E4M3> int launch_kv8_attention(const KvAttnArgs& a, const CUtensorMap& map, int grid, cudaStream_t st) {
  using S = KvShape<D>;
  static bool set[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16 || !set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kv8_attention_kernel<D, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 16) set[dev] = true;
  }
  kv8_attention_kernel<D, E4M3><<<grid, kThreads, S::kSmem, st>>>(map, a);
  kv8_join_kernel<D><<<a.NW, 128, 0, st>>>(a);
  return (int)cudaGetLastError();
}
}  // namespace hippo

using namespace hippo;

// q [N][Hq][D] (strides in elements), out [N][Hq][D], codes [2][blocks][H][bs][D], scales [2][blocks][H], table [N][M] (pitch
// table_ld); dtype 0 bf16, 1 fp16, 2 fp32. workers: warps of the launch, a multiple of 4; ws: workers * 2 * min(Hq / H, 8) * (D + 2)
// floats, then workers * 4 ints, 16-byte aligned. One block of arguments, as in kv8.cu.
struct KvAttendCall {
  const void* q; void* out; const void* codes; const float* scales; const int *table, *lens; float* ws; void* stream;
  long long q_n, q_h, table_ld, blocks;
  int N, H, Hq, D, block_size, M, dtype, e4m3, workers;
  float scale;
};
extern "C" int hippo_kv8_attention(const KvAttendCall* c) {
  const int sh = c->block_size == 16 ? 4 : c->block_size == 32 ? 5 : c->block_size == 64 ? 6 : -1;
  if (sh < 0 || c->N < 1 || c->M < 1 || c->H < 1 || c->Hq % c->H || c->blocks < 1 || c->workers < kWarps || c->workers % kWarps ||
      c->dtype < 0 || c->dtype > 2 || (c->D != 64 && c->D != 128))
    return -1;
  const int D = c->D;
  const long long half_rows = (c->blocks * c->H) << sh;
  if (2 * half_rows > 0x7fffffffll) return -2;       // TMA coordinates are 32-bit
  auto fn = get_encode_fn();
  if (!fn) return -100;
  CUtensorMap map;
  const int box = c->block_size < kTile ? c->block_size : kTile;
  const cuuint64_t dim[2] = {(cuuint64_t)D, (cuuint64_t)(2 * half_rows)}, pitch[1] = {(cuuint64_t)D};
  const cuuint32_t bx[2] = {(cuuint32_t)D, (cuuint32_t)box}, one[2] = {1, 1};
  const CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(c->codes), dim, pitch, bx, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return -102 - (int)r;
  const int G = c->Hq / c->H, rows = G < 8 ? G : 8;
  const long long parts = 2ll * c->workers * rows;
  KvAttnArgs a{c->q, c->out, c->q_n, c->q_h, c->scales, c->blocks * c->H, c->table, c->table_ld, c->M, c->lens, c->N, c->H, G,
               (G + 7) / 8, sh, (int)c->blocks, c->dtype, half_rows, c->scale, c->ws, c->ws + parts * D,
               (int4*)(c->ws + parts * (D + 2)), c->workers, rows};
  cudaStream_t st = (cudaStream_t)c->stream;
  const int grid = c->workers / kWarps;
  if (D == 128) return c->e4m3 ? launch_kv8_attention<128, 1>(a, map, grid, st) : launch_kv8_attention<128, 0>(a, map, grid, st);
  return c->e4m3 ? launch_kv8_attention<64, 1>(a, map, grid, st) : launch_kv8_attention<64, 0>(a, map, grid, st);
}
