// One query token per sequence against the 8-bit paged cache: o = sum_j softmax_j(scale q.k_j) v_j with k_j = s_K code, v_j = s_V code
// and one (s_K, s_V) per (block, kv head).
//
// Bound by HBM: a token and kv head costs 2 D bytes of codes, read once for the query heads that share the kv head (up to 8 of them
// together). Work is cut in tiles of 32 tokens (64 for head_dim 64: 8 KB); the tiles of all (sequence, kv head, group of query heads)
// form one list that is divided evenly over one resident wave of one-warp blocks, whatever the lengths (the start of a unit counts as
// one more tile: its query rows and its result cost about as much). A warp streams its tiles through a TMA ring and carries the
// running maximum and sum; a unit that spans several warps leaves partial (m, l, o) rows that a second, small kernel joins in a fixed
// order, so results do not depend on timing.
//
// Arithmetic: codes are exact in fp16, so mma.m16n8k16 (fp16 operands, fp32 accumulators) is exact for them. They are the 16-row
// operand of both products (S^T = K q^T, O^T = V^T P^T); the 8 columns are 4 query heads, each as two fp16 terms of the query and of
// the probabilities, whose two sums meet in one thread. Both are brought to fp16's range first: two terms hold 22 bits of a value
// down to 2^-16 of the row's largest, and steps of 2^-38 of it below. P^T comes from the scores' fragments by movmatrix. The
// converted codes, not the tensor pipe, set the instruction count, so the narrow side of the product is the query's. Legacy mma is
// deliberate: with 1 to 8 live columns a 128-row tcgen05 tile would multiply zeros, and the kernel waits for memory.
//
// Measured, both kernels (device time in a row of calls, inputs above L2): 32 sequences of 6001 to 8192 tokens, 32 heads of 128, e4m3:
// 300 us = 6.2 TB/s; 16 x 4096 tokens, 32 heads of 128: 94 us = 5.7 TB/s (int8 90); 2 x 131072, 4 heads of 128: 50.3 to 51.9 us = 5.2 TB/s;
// 16 x 4096, 64 heads on 8 of 128: 38.6 us; 1 x 500, 16 heads: 9.0 us. Short calls wait for lens -> table -> first tiles (5 us) and for
// the join (3.4 us, of long sequences 6.7).
// In the reference a decoding step re-runs the whole forward (src/models/model.py:180-219).
#include <type_traits>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include "sm100.cuh"
#include "host_utils.h"
#include "ring.h"
#include "kv8_common.cuh"

namespace hippo {
constexpr int kUnits = 4;                            // workers whose units a block of the joining kernel looks after
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities (times their value scale, relative to the largest: 0 .. 1) are multiplied by 2^15 before they are split: fp16's smallest
// step, 2^-24, then is 2^-39 of the largest, so that thousands of weak tokens beside a strong one keep their share.
constexpr float kLift = 32768.f;

struct KvAttnArgs {
  const void* q; void* out;
  long long q_n, q_h;                                // query strides in elements; out is [N][Hq][D]
  const float* scales; long long half_scales;
  const int* table; long long table_ld; int M;
  const int* lens;
  int N, H, G, QG, sh, blocks, dtype;                // kv heads, query heads a kv head, groups of 4 or 8 of them
  long long half_rows;                               // cache rows (of D bytes) of the key half
  float scale;
  float* part; float* part_ml; int4* desc; int NW, rows;   // parts of `rows` query rows each, two a worker
};

template <int D, int SETS> struct KvShape {
  static constexpr int kTile = 4096 / D, kGroups = kTile / 16;       // tokens, groups of 16 of them (a block holds one or more)
  static constexpr int kStageBytes = 2 * kTile * D;
  // More registers than twelve blocks leave keep the compiler from spilling (two groups of heads of 128) and let it run further
  // ahead (one): eight blocks with a deeper ring. 16 x 4096 x 32 heads of 128: 93 us against 96.
  static constexpr int kBlocks = D * SETS > 64 ? 8 : 12, kStages = kBlocks == 8 ? 3 : 2;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {       // 8 x 8 fp16, a pair a lane
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// four codes -> four fp16, exactly: bytes 0, 1 in `lo`, bytes 2, 3 in `hi`. int8 goes through 1024 + (code + 128), whose low byte is
// the biased code.
template <int E4M3> __device__ __forceinline__ void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    return;
  }
  w ^= 0x80808080u;
  const uint32_t l = __byte_perm(w, 0x64646464u, 0x4140), h = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));       // 1152
  const __half2 x = __hsub2(*(const __half2*)&l, bias), y = __hsub2(*(const __half2*)&h, bias);
  lo = *(const uint32_t*)&x;
  hi = *(const uint32_t*)&y;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}

// N consecutive query values (16-byte aligned) as fp32
template <int N> __device__ __forceinline__ void load_q(const KvAttnArgs& a, long long i, float (&x)[N]) {
  if (a.dtype == 2) {
    const float4* p = (const float4*)((const float*)a.q + i);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const float4 v = __ldg(p + j);
      x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
    }
    return;
  }
  uint4 v[N / 8];
#pragma unroll
  for (int j = 0; j < N / 8; ++j) v[j] = __ldg((const uint4*)((const __half*)a.q + i) + j);
#pragma unroll
  for (int j = 0; j < N / 8; ++j) {
    const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = a.dtype == 0 ? make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u))
                                    : __half22float2(*(const __half2*)&w[k]);
      x[8 * j + 2 * k] = f.x; x[8 * j + 2 * k + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void store_out(const KvAttnArgs& a, long long i, float x, float y) {      // elements i, i + 1
  if (a.dtype == 0) ((__nv_bfloat162*)a.out)[i >> 1] = __floats2bfloat162_rn(x, y);
  else if (a.dtype == 1) ((__half2*)a.out)[i >> 1] = __floats2half2_rn(x, y);
  else ((float2*)a.out)[i >> 1] = make_float2(x, y);
}

__device__ __forceinline__ int cached_len(const KvAttnArgs& a, int n) {
  return (int)min((long long)max(a.lens[n], 0), (long long)a.M << a.sh);
}

// Where a warp stands in the list of tiles: sequence, kv head, group of query heads, tile.
template <int kTile> struct Cursor {
  int n, h, grp, tile, len, tiles, left;             // left: places of the warp's range that are still ahead, this tile's included
  __device__ void advance(const KvAttnArgs& a) {
    if (--left <= 0 || ++tile < tiles) return;
    tile = 0;
    if (--left <= 0 || ++grp < a.QG) return;         // the next unit's first place has no tile
    grp = 0;
    if (++h < a.H) return;
    h = 0;
    do { ++n; len = n < a.N ? cached_len(a, n) : 0; } while (n < a.N && len == 0);
    tiles = (len + kTile - 1) / kTile;
  }
};

// SETS: groups of 4 query heads that one pass over the codes serves
template <int D, int E4M3, int SETS>
__global__ void __launch_bounds__(32, KvShape<D, SETS>::kBlocks) kv8_attention_kernel(const __grid_constant__ CUtensorMap codes_map, KvAttnArgs a) {
  using S = KvShape<D, SETS>;
  constexpr int kTile = S::kTile, NG = S::kGroups;
  constexpr int KS = D / 16, MT = D / 16, DL = D / 8;        // k steps of K q, row tiles of V^T P, output columns a lane
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[S::kStages];
  __shared__ float2 s_scale[S::kStages][NG];         // K and V scale of every 16 tokens of the tile
  __shared__ unsigned s_there[S::kStages];           // bit 2g: tokens and a block of the pool in group g of the tile
  const int lane = threadIdx.x;
  const int units = a.H * a.QG;
  asm volatile("griddepcontrol.launch_dependents;");

  // rows of empty sequences
  for (int n = blockIdx.x; n < a.N; n += gridDim.x)
    if (a.lens[n] <= 0)
      for (int i = lane; i < a.H * a.G * (D / 2); i += 32) store_out(a, (long long)n * a.H * a.G * D + i * 2, 0.f, 0.f);

  // places before every lane's share of the sequences: a unit has one more than tiles
  const int share = (a.N + 31) / 32;
  int mine = 0;                                      // (the host has seen to it that all places are below 2^31)
  for (int n = lane * share; n < min(a.N, (lane + 1) * share); ++n) {
    const int len = cached_len(a, n);
    if (len > 0) mine += ((len + kTile - 1) / kTile + 1) * units;
  }
  int inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 0) {
    for (int j = 0; j < S::kStages; ++j) mbar_init(&full[j], 1 + 2 * NG);      // TMA bytes, the lanes' scale copies
    fence_barrier_init();
  }
  __syncwarp();
  const int total = __shfl_sync(0xffffffffu, inc, 31);

  // no more workers than half the places: each has two at least, so one tile or more of every unit between its ends
  const int worker = blockIdx.x, nw = min(a.NW, total >> 1);
  const int each = nw ? total / nw : 0, odd = total - each * nw;         // the first `odd` workers have one place more
  const int begin = worker < nw ? each * worker + min(worker, odd) : 0;
  const int end = worker < nw ? begin + each + (worker < odd) : 0;
  // unit that begins here and ends in a later worker: sequence, first query head * 16 + query rows, slot, last worker
  int4 found = make_int4(-1, 0, 0, 0);
  uint8_t* ring = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);

  if (begin < end) {
    Cursor<kTile> put;                               // next tile to fetch
    {
      const int lo = __ffs(__ballot_sync(0xffffffffu, inc > begin)) - 1;
      int at = __shfl_sync(0xffffffffu, inc - mine, lo);
      int n = lo * share;
      for (;;) {                                     // the sequence of the share that holds `begin`
        put.len = cached_len(a, n);
        put.tiles = (put.len + kTile - 1) / kTile;
        const int c = put.len > 0 ? (put.tiles + 1) * units : 0;
        if (at + c > begin) break;
        at += c; ++n;
      }
      put.n = n;
      const int unit = (begin - at) / (put.tiles + 1);
      put.tile = begin - at - unit * (put.tiles + 1) - 1;
      put.left = end - begin;
      if (put.tile < 0) { put.tile = 0; --put.left; }
      put.h = unit / a.QG;
      put.grp = unit - put.h * a.QG;
    }
    Cursor<kTile> get = put;
    // fetching: lanes hold 32 entries of the table row
    int held_n = -1, held_base = 0, held = -1;
    const int box = min(kTile, 1 << a.sh);           // rows of one TMA box
    const int half_rows = (int)a.half_rows;
    auto fetch = [&](int stage) {
      const int tok = put.tile * kTile, blk = tok >> a.sh;
      const int base = blk & ~31;                    // a tile never spans two batches of 32 entries (its blocks start at a multiple)
      if (held_n != put.n || held_base != base) {
        held_n = put.n; held_base = base;
        const int j = base + lane;
        held = j < a.M && ((long long)j << a.sh) < put.len ? a.table[(long long)put.n * a.table_ld + j] : -1;
        if (held >= a.blocks) held = -1;
      }
      // lanes 2g and 2g + 1: 16 tokens from 16g on, their key and their value side
      const int grp = lane >> 1, first = tok + grp * 16;
      const int b = __shfl_sync(0xffffffffu, held, (first >> a.sh) & 31);
      const bool there = lane < 2 * NG && first < put.len && b >= 0, box_here = there && (grp * 16 & (box - 1)) == 0;
      const unsigned m = __ballot_sync(0xffffffffu, there), boxes = __ballot_sync(0xffffffffu, box_here);
      uint64_t* bar = &full[stage];
      if (lane < 2 * NG) {
        if (lane == 0) {
          s_there[stage] = m;
          mbar_expect_tx(bar, (uint32_t)(__popc(boxes) * box * D));
        }
        const int bh = b * a.H + put.h;              // below 2^31 with the rows of all blocks
        if (there) {
          const float* src = a.scales + (lane & 1 ? a.half_scales : 0) + bh;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32((float*)&s_scale[stage][0] + lane)), "l"(src) : "memory");
        }
        if (box_here)
          tma_load_2d(ring + stage * S::kStageBytes + (lane & 1) * kTile * D + grp * 16 * D, &codes_map, bar, 0,
                      (bh << a.sh) + (first & ((1 << a.sh) - 1)) + (lane & 1 ? half_rows : 0));
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
      }
      put.advance(a);
    };
    const int g = lane >> 2, c = lane & 3;           // fragments: row (token, output column group) / column of the query side; query head
#pragma unroll 1
    for (int i = 0; i < S::kStages; ++i)
      if (put.left > 0) fetch(i);
    __syncwarp();

    uint32_t qf[SETS][KS][2];
    float o[SETS][MT][4];
    float m[SETS], mv[SETS], l[SETS], f[SETS];       // maximum of the scores, of scores + log2 of the value scale; sum; factor of the scores
    bool alive = true, fresh = true, whole = true, first = true;
    int stage = 0, phase = 0;
    // smem offsets of this lane: K rows g (+ 8), 16 bytes at chunk 2c (D 128) or c (D 64); V rows 2c (+ 1, 8, 9), D / 8 bytes at column g
    const uint32_t k_at = g * D + (D == 128 ? ((2 * c) ^ g) * 16 : (c ^ ((g >> 1) & 3)) * 16);
    while (get.left > 0) {
      const int n = get.n, h = get.h, g0 = get.grp * 4 * SETS;
      if (fresh) {                                   // a new unit: its query rows, brought to fp16's range and split in two fp16
        fresh = false;
        whole = get.tile == 0;
#pragma unroll
        for (int t = 0; t < SETS; ++t) {
          const int qh = g0 + t * 4 + (g >> 1);      // column g of the query side: head g / 2, its high (even) or low term
          const bool row = qh < a.G;
          const long long qi = (long long)n * a.q_n + (long long)(h * a.G + qh) * a.q_h + c * (D / 4);
          float x[D / 4] = {}, top = 0.f;
          if (row) load_q(a, qi, x);
#pragma unroll
          for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // the largest element lies in [2^14, 2^15) then, so fp16's smallest step is 2^-38 of it
          const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100) - 14;     // -114 .. 114
          const float down = pow2f(-e);
          f[t] = __shfl_sync(0xffffffffu, pow2f(e), c * 8) * a.scale * kLog2e;       // of head c: its column 2c is lane 8c's
#pragma unroll
          for (int i = 0; i < D / 4; ++i) {
            x[i] *= down;
            if (g & 1) x[i] -= __half2float(__float2half_rn(x[i]));
          }
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            qf[t][i][0] = pack2(x[4 * i], x[4 * i + 1]);
            qf[t][i][1] = pack2(x[4 * i + 2], x[4 * i + 3]);
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
          m[t] = mv[t] = -INFINITY; l[t] = 0.f;
        }
      }
      const bool landed = mbar_wait(&full[stage], phase, kWaitTmaFull, worker);
      if (!__all_sync(0xffffffffu, landed)) { alive = false; break; }     // each lane has its own limit: the warp gives up together
      const uint8_t* kt = ring + stage * S::kStageBytes;
      const uint8_t* vt = kt + kTile * D;
      const int valid = min(kTile, get.len - get.tile * kTile);
      const unsigned there = s_there[stage];
      const bool ragged = valid < kTile || there != (1u << 2 * NG) - 1;
      float2 sc[NG];
#pragma unroll
      for (int j = 0; j < NG; ++j) sc[j] = s_scale[stage][j];
      uint32_t pb[SETS][2 * NG];                     // P^T as the second operand: a k step for each 16 tokens
      {
        float s[SETS][NG][4];
#pragma unroll
        for (int t = 0; t < SETS; ++t)
#pragma unroll
          for (int j = 0; j < NG; ++j) s[t][j][0] = s[t][j][1] = s[t][j][2] = s[t][j][3] = 0.f;
#pragma unroll
        for (int q4 = 0; q4 < D / 64; ++q4)
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            const uint4 x = *(const uint4*)(kt + j * 16 * D + (k_at ^ (q4 * 16)));           // row 16j + g
            const uint4 y = *(const uint4*)(kt + j * 16 * D + 8 * D + (k_at ^ (q4 * 16)));   // row 16j + g + 8
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a0, a1, a2, a3;
              codes4<E4M3>(xw[i], a0, a2);
              codes4<E4M3>(yw[i], a1, a3);
#pragma unroll
              for (int t = 0; t < SETS; ++t) mma16816(s[t][j], a0, a1, a2, a3, qf[t][q4 * 4 + i][0], qf[t][q4 * 4 + i][1]);
            }
          }
#pragma unroll
        for (int t = 0; t < SETS; ++t) {
          // tokens 16j + g and 16j + g + 8 of query head c, and with the value scale's logarithm
          float y[2 * NG], z[2 * NG];
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            const float fk = f[t] * sc[j].x, lv = log2f(sc[j].y);
            y[2 * j] = (s[t][j][0] + s[t][j][1]) * fk; y[2 * j + 1] = (s[t][j][2] + s[t][j][3]) * fk;
            z[2 * j] = y[2 * j] + lv; z[2 * j + 1] = y[2 * j + 1] + lv;
          }
          if (ragged) {
#pragma unroll
            for (int i = 0; i < 2 * NG; ++i)
              if (i * 8 + g >= valid || !(there >> (i & ~1) & 1)) y[i] = z[i] = -INFINITY;
          }
          float mx = y[0], mz = z[0];
#pragma unroll
          for (int i = 1; i < 2 * NG; ++i) { mx = fmaxf(mx, y[i]); mz = fmaxf(mz, z[i]); }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            mz = fmaxf(mz, __shfl_xor_sync(0xffffffffu, mz, d));
          }
          mx = fmaxf(mx, m[t]); mz = fmaxf(mz, mv[t]);
          const float mu = mx == -INFINITY ? 0.f : mx, mzu = mz == -INFINITY ? 0.f : mz;
          const float alpha = ex2(mv[t] - mzu);
          l[t] *= ex2(m[t] - mu);
          m[t] = mx; mv[t] = mz;
          if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
            for (int i = 0; i < MT; ++i) { o[t][i][0] *= alpha; o[t][i][1] *= alpha; o[t][i][2] *= alpha; o[t][i][3] *= alpha; }
          }
#pragma unroll
          for (int i = 0; i < 2 * NG; ++i) {
            l[t] += ex2(y[i] - mu);
            const float p = ex2(z[i] - mzu) * kLift;
            pb[t][i] = transpose8x8(pack2(p, p - __half2float(__float2half_rn(p))));
          }
        }
      }
#pragma unroll
      for (int kk = 0; kk < NG; ++kk) {
        constexpr int W = D / 32;                    // 32-bit words a lane reads of a row
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
        }
        if (ragged) {                                // bytes behind the last token may be NaN codes
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t keep = kk * 16 + 2 * c + (i & 1) + (i >> 1) * 8 < valid && (there >> 2 * kk & 1) ? 0xffffffffu : 0u;
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] &= keep;
          }
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
          // bytes 4j .. 4j + 3 of the four rows: pairs of tokens for each output column
          uint32_t x0, x1, x2, x3, y0, y1, y2, y3;
          codes4<E4M3>(__byte_perm(v[0][j], v[1][j], 0x5140), x0, x1);
          codes4<E4M3>(__byte_perm(v[2][j], v[3][j], 0x5140), y0, y1);
          codes4<E4M3>(__byte_perm(v[0][j], v[1][j], 0x7362), x2, x3);
          codes4<E4M3>(__byte_perm(v[2][j], v[3][j], 0x7362), y2, y3);
#pragma unroll
          for (int t = 0; t < SETS; ++t) {
            mma16816(o[t][2 * j], x0, x1, y0, y1, pb[t][2 * kk], pb[t][2 * kk + 1]);
            mma16816(o[t][2 * j + 1], x2, x3, y2, y3, pb[t][2 * kk], pb[t][2 * kk + 1]);
          }
        }
      }
      __syncwarp();                                  // every lane has read the stage
      if (put.left > 0) fetch(stage);
      if (++stage == S::kStages) { stage = 0; phase ^= 1; }

      const int tile = get.tile, tiles = get.tiles, left = get.left;
      get.advance(a);
      if (tile + 1 == tiles || get.left <= 0) {      // the unit, or this warp's part of it, is done
        // a worker has at most two parts: of the unit at its start (slot 0), and of one that begins inside it (slot 1)
        const bool done = whole && tile + 1 == tiles;
        const int sl = worker * 2 + (first ? 0 : 1);
#pragma unroll
        for (int t = 0; t < SETS; ++t) {
          float lt = l[t];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) lt += __shfl_xor_sync(0xffffffffu, lt, d);
          // o is held relative to the maximum of p s_V and kLift times as large, l relative to the maximum of p
          const float back = lt == 0.f ? 0.f : ex2(mv[t] - m[t]) * (1.f / kLift), r = done ? (lt == 0.f ? 0.f : back / lt) : back;
          const int row = t * 4 + c;                 // this lane: query head c of the set, output columns DL g ...
          if (g0 + row >= a.G) continue;
          if (done) {
            const long long oi = ((long long)n * a.H * a.G + h * a.G + g0 + row) * D + g * DL;
#pragma unroll
            for (int i = 0; i < MT; ++i) store_out(a, oi + 2 * i, (o[t][i][0] + o[t][i][1]) * r, (o[t][i][2] + o[t][i][3]) * r);
          } else {
            float* dst = a.part + ((long long)sl * a.rows + row) * D + g * DL;
#pragma unroll
            for (int i = 0; i < MT; ++i) *(float2*)(dst + 2 * i) = make_float2((o[t][i][0] + o[t][i][1]) * r, (o[t][i][2] + o[t][i][3]) * r);
            if (g == 0) *(float2*)(a.part_ml + ((long long)sl * a.rows + row) * 2) = make_float2(m[t], lt);
          }
        }
        if (whole && !done) {                        // begins here, goes on: this worker's unit to join
          const int last = end - left - tile + tiles - 1, wide = (each + 1) * odd;     // place of its last tile
          found = make_int4(n, (h * a.G + g0) << 4 | min(4 * SETS, a.G - g0), sl, last < wide ? last / (each + 1) : odd + (last - wide) / each);
        }
        fresh = true;
        first = false;
      }
    }
    if (!alive) {                                    // a wait ran out: the copies of the tiles from `get` to `put` land before the block ends
      for (int i = 0; i < S::kStages && get.left != put.left; ++i) {
        const RingPlace r = ring_place(stage, phase, i, S::kStages);
        mbar_wait(&full[r.stage], r.parity, kWaitTmaFull, -1);
        get.advance(a);
      }
      found.x = -1;
    }
  }
  if (lane == 0) a.desc[worker] = found;
}

// Joins the parts of the units that begin in four workers of the first kernel: (m, l, o) of the parts in order, rescaled whenever a
// batch of them brings a larger m. The kernel is a chain of dependent reads (3 to 4 us after the first one's end), so a batch's
// maxima and rows are under way together. A warp takes a row of few parts by itself; the rows of a unit of many (a long sequence) are
// shared by the warps, one of which joins their sums in order. Blocks of eight warps for four workers: with four warps for two
// 2 x 131072 tokens take 52.7 us, not 50.5, with two for one 57.0.
constexpr int kJoinWarps = 8, kFewParts = 4;
struct JoinUnit {
  int n, head0, w0, slot0, parts, rows;              // sequence, first query head, first worker and its slot, query rows
};
template <int D> __global__ void __launch_bounds__(kJoinWarps * 32, 3) kv8_join_kernel(KvAttnArgs a, int per_unit) {
  constexpr int C = D / 32;                          // columns a lane
  __shared__ float s_o[kJoinWarps][D], s_m[kJoinWarps], s_l[kJoinWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  auto unit = [&](int k) {
    const int w0 = blockIdx.x * kUnits + k;
    const int4 d = a.desc[w0];
    return d.x < 0 ? JoinUnit{} : JoinUnit{d.x, d.y >> 4, w0, d.z, min(d.w, a.NW - 1) - w0 + 1, d.y & 15};
  };
  struct Sum { float m, l, o[C]; };
  // parts first, first + step, ... of a row
  auto gather = [&](const JoinUnit& u, int row, int first, int step, auto batch) {
    constexpr int B = decltype(batch)::value;
    Sum t{-INFINITY, 0.f, {}};
#pragma unroll 1
    for (int i0 = first; i0 < u.parts; i0 += B * step) {
      float2 ml[B];
      float x[B][C];
#pragma unroll
      for (int j = 0; j < B; ++j) {
        const int i = i0 + j * step;
        ml[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < C; ++k) x[j][k] = 0.f;
        if (i < u.parts) {
          const long long sl = (long long)(i == 0 ? u.slot0 : 2 * (u.w0 + i)) * a.rows + row;
          ml[j] = *(const float2*)(a.part_ml + sl * 2);
          if (C == 4) *(float4*)x[j] = *(const float4*)(a.part + sl * D + lane * 4);
          else *(float2*)x[j] = *(const float2*)(a.part + sl * D + lane * 2);
        }
      }
      float m = t.m;
#pragma unroll
      for (int j = 0; j < B; ++j) m = fmaxf(m, ml[j].x);
      const float mu = m == -INFINITY ? 0.f : m, back = ex2(t.m - mu);
      t.m = m;
      t.l *= back;
#pragma unroll
      for (int k = 0; k < C; ++k) t.o[k] *= back;
#pragma unroll
      for (int j = 0; j < B; ++j) {
        const float r = ex2(ml[j].x - mu);
        t.l += ml[j].y * r;
#pragma unroll
        for (int k = 0; k < C; ++k) t.o[k] += x[j][k] * r;
      }
    }
    return t;
  };
  auto put = [&](const JoinUnit& u, int row, const Sum& t) {
    const float r = t.l == 0.f ? 0.f : 1.f / t.l;
    const long long oi = ((long long)u.n * a.H * a.G + u.head0 + row) * D + lane * C;
#pragma unroll
    for (int j = 0; j < C; j += 2) store_out(a, oi + j, t.o[j] * r, t.o[j + 1] * r);
  };
  for (int t = w; t < kUnits * per_unit; t += kJoinWarps) {
    const JoinUnit u = unit(t % kUnits);
    const int row = t / kUnits;
    if (row >= u.rows || u.parts > kFewParts) continue;
    put(u, row, gather(u, row, 0, 1, std::integral_constant<int, kFewParts>()));
  }
#pragma unroll 1
  for (int k = 0; k < kUnits; ++k) {
    const JoinUnit u = unit(k);
    if (u.parts <= kFewParts) continue;
    // the rows side by side, `team` warps each
    const int team = u.rows > 4 ? 1 : u.rows > 2 ? 2 : u.rows > 1 ? 4 : 8, row = w / team, first = w % team;
    const bool on = row < u.rows;
    Sum t{-INFINITY, 0.f, {}};
    if (on) t = gather(u, row, first, team, std::integral_constant<int, 8>());
    if (team == 1) {
      if (on) put(u, row, t);
      continue;
    }
#pragma unroll
    for (int j = 0; j < C; ++j) s_o[w][lane * C + j] = t.o[j];
    if (lane == 0) { s_m[w] = t.m; s_l[w] = t.l; }
    __syncthreads();
    if (on && first == 0) {
      float m = t.m;
      for (int i = 1; i < team; ++i) m = fmaxf(m, s_m[w + i]);
      const float mu = m == -INFINITY ? 0.f : m;
      Sum all{m, 0.f, {}};
      for (int i = 0; i < team; ++i) {
        const float r = ex2(s_m[w + i] - mu);
        all.l += s_l[w + i] * r;
#pragma unroll
        for (int j = 0; j < C; ++j) all.o[j] += s_o[w + i][lane * C + j] * r;
      }
      put(u, row, all);
    }
    __syncthreads();
  }
}

template <int D, int E4M3, int SETS> int launch_sets(const KvAttnArgs& a, const CUtensorMap& map, cudaStream_t st) {
  using S = KvShape<D, SETS>;
  static bool set[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16 || !set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kv8_attention_kernel<D, E4M3, SETS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 16) set[dev] = true;
  }
  kv8_attention_kernel<D, E4M3, SETS><<<a.NW, 32, S::kSmem, st>>>(map, a);
  const cudaError_t first = cudaGetLastError();
  if (first != cudaSuccess) return (int)first;       // the joining kernel would follow descriptors that nobody wrote
  // the joining kernel is launched while the first one runs and waits for its end on the device
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.NW / kUnits));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, kv8_join_kernel<D>, a, 4 * SETS);
}
template <int D, int E4M3> int launch_kv8_attention(const KvAttnArgs& a, const CUtensorMap& map, cudaStream_t st) {
  // five to eight heads on one kv head read the codes once together (16 x 4096 tokens, 64 heads on 8: 38 us, in passes of four 48)
  return a.G <= 4 ? launch_sets<D, E4M3, 1>(a, map, st) : launch_sets<D, E4M3, 2>(a, map, st);
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
  if (sh < 0 || c->N < 1 || c->M < 1 || c->H < 1 || c->Hq % c->H || c->blocks < 1 || c->workers < kUnits || c->workers % kUnits ||
      c->dtype < 0 || c->dtype > 2 || (c->D != 64 && c->D != 128))
    return -1;
  const int D = c->D;
  const long long half_rows = (c->blocks * c->H) << sh;
  if (2 * half_rows > 0x7fffffffll) return -2;       // TMA coordinates are 32-bit
  const long long groups = (long long)c->N * c->H * ((c->Hq / c->H + 7) / 8);
  if (groups * ((((long long)c->M << sh) + 4096 / D - 1) / (4096 / D) + 1) > 0x7fffffffll) return -3;
  if (((uintptr_t)c->q & 15) || c->q_n * (c->dtype == 2 ? 4 : 2) % 16 || c->q_h * (c->dtype == 2 ? 4 : 2) % 16) return -4;
  auto fn = get_encode_fn();
  if (!fn) return -100;
  CUtensorMap map;
  const int tile = 4096 / D, box = c->block_size < tile ? c->block_size : tile;
  const cuuint64_t dim[2] = {(cuuint64_t)D, (cuuint64_t)(2 * half_rows)}, pitch[1] = {(cuuint64_t)D};
  const cuuint32_t bx[2] = {(cuuint32_t)D, (cuuint32_t)box}, one[2] = {1, 1};
  const CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(c->codes), dim, pitch, bx, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return -102 - (int)r;
  const int G = c->Hq / c->H, rows = G < 8 ? G : 8;
  const long long parts = 2ll * c->workers * rows;
  KvAttnArgs a{c->q, c->out, c->q_n, c->q_h, c->scales, c->blocks * c->H, c->table, c->table_ld, c->M, c->lens, c->N, c->H, G,
               G <= 4 ? 1 : (G + 7) / 8, sh, (int)c->blocks, c->dtype, half_rows, c->scale, c->ws, c->ws + parts * D,
               (int4*)(c->ws + parts * (D + 2)), c->workers, rows};
  cudaStream_t st = (cudaStream_t)c->stream;
  if (D == 128) return c->e4m3 ? launch_kv8_attention<128, 1>(a, map, st) : launch_kv8_attention<128, 0>(a, map, st);
  return c->e4m3 ? launch_kv8_attention<64, 1>(a, map, st) : launch_kv8_attention<64, 0>(a, map, st);
}
