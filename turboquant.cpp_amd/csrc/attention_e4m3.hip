// Attention over the 8-bit cache (cache_e4m3.h) on the matrix cores.
//
//   s_ij = f(scale q_i . k_j)      f: the cap and the bias by distance of score_mod.h
//   p_ij = exp(s_ij) / (sum over the j that i sees, and the sink)
//   o_i  = sum_j p_ij v_j          and, if asked for, w_j += sum over i and the heads of a kv head of p_ij
//
// Codes become bfloat16 with their scale in one instruction for two, without rounding, and both products run on
// v_mfma_f32_16x16x32_bf16 with sums in 32 bits: S^T = K Q^T with 16 keys as rows and 16 columns (tokens of a head in prompts, heads
// of a kv head in decoding), O^T += V^T P^T with 16 dimensions as rows.  Block jt of a tile's keys is positions 16 jt .. 16 jt + 15,
// so lane (r, c) holds the scores of positions 16 jt + 4 c + v of column r, and the pages hold values in that order: the
// probabilities are the second product's operand as they stand.
// Queries of the 32-bit library are cut into three bfloat16 pieces (24 bits: nothing is lost), and so are its probabilities: codes
// have one piece, so three products give what 32-bit arithmetic would.  In the bfloat16 library probabilities are rounded to
// bfloat16 for the product with the values (half a step, 2^-8 of each), as its other attention kernels do; their sum is of the numbers before.
// The running maximum is only moved where a tile's is more than 2^8 above it, so that the sums are rescaled a few times a row and not
// at every tile; probabilities are then at most 256, which neither type minds.
#include "cache_e4m3.h"
#include "score_mod.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

#define LOG2E 1.4426950408889634f
#if defined(TQ_ACT_F32)
#define PIECES 3
#else
#define PIECES 1
#endif

struct E4m3Attn {
  const act_t* q;               // [T][nh][hd]
  act_t* out;                   // [T][nh][hd]
  const int* cu;                // [B + 1]
  const int* slots;
  const int* start;
  int B, nh, nkv, window;
  float scale;
  ScoreMod mod;
  float* partial;               // decoding: [B][nh][max_runs][hd + 2]
  int max_runs;
  float* scores;                // decoding with weights: [B][nh][ld_scores], a column's scores in units of log2
  int64_t ld_scores;
  float* lse;                   // with weights: [T][nh] log2 of a row's sum of 2^score, the sink's included
  E4m3Pages pages;
};

// Eight codes, times a power of two, as the operand of a product.
__device__ __forceinline__ bf16x8 numbers(uint32_t a, uint32_t b, float scale) {
  const u32x4 w = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true))};
  return __builtin_bit_cast(bf16x8, w);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
// Eight numbers as PIECES operands whose sum they are.
__device__ __forceinline__ void pieces_of(const float (&x)[8], bf16x8 (&out)[PIECES]) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const u32x4 w = {pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7])};
    out[p] = __builtin_bit_cast(bf16x8, w);
    if (p + 1 < PIECES)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fabsf((float)out[p][i]) == INFINITY ? 0.f : y[i] - (float)out[p][i];      // (an infinite query has one piece)
  }
}
__device__ __forceinline__ bf16x8 nothing() {
  const u32x4 w = {0u, 0u, 0u, 0u};
  return __builtin_bit_cast(bf16x8, w);
}
// Eight numbers of a query from dimension d on; zeros behind the head's end and for a column without a query.
__device__ __forceinline__ void load_query(bf16x8 (&out)[PIECES], const act_t* row, int d, int hd, bool valid) {
  if (!valid || d >= hd) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) out[p] = nothing();
    return;
  }
#if defined(TQ_ACT_BF16)
  out[0] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(row + d));
#else
  const float4 a = *reinterpret_cast<const float4*>(row + d), b = *reinterpret_cast<const float4*>(row + d + 4);
  const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  pieces_of(x, out);
#endif
}
__device__ __forceinline__ float group_max(float v) { return with_lane_xor<32>(with_lane_xor<16>(v, LanesMax()), LanesMax()); }
__device__ __forceinline__ float group_sum(float v) { return with_lane_xor<32>(with_lane_xor<16>(v, LanesSum()), LanesSum()); }
__device__ __forceinline__ float changed_score(float s, const ScoreMod& m, float r1, float r2, int dist) {
#if defined(TQ_ACT_BF16)
  return mod_score_fast(s, m.cap, m.r1 != nullptr, r1, r2, dist);
#else
  return mod_score(s, m.cap, m.r1 != nullptr, r1, r2, dist);
#endif
}

// Scores of a tile to units of log2 and -inf where the column does not see the position, for one group of 16 columns.
template <bool MOD>
__device__ __forceinline__ void final_scores(f32x4 (&s)[4], const E4m3Attn& a, float r1, float r2, int pos0, int p, int lo, bool masked) {
  const int c = (threadIdx.x % 64) / 16;
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int key = pos0 + 16 * jt + 4 * c + v;
      float x = s[jt][v] * (MOD ? a.scale : a.scale * LOG2E);
      if constexpr (MOD) x = changed_score(x, a.mod, r1, r2, p - key) * LOG2E;
      if (masked) x = key <= p && key >= lo ? x : -INFINITY;
      s[jt][v] = x;
    }
}
// The part of a tile between its products for one group of 16 columns: scores in, probabilities as operands out.
template <int DT>
__device__ __forceinline__ void softmax_tile(f32x4 (&s)[4], f32x4 (&o)[DT], float& m, float& l, bf16x8 (&pf)[2][PIECES]) {
  float top = -INFINITY;
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
#pragma unroll
    for (int v = 0; v < 4; ++v) top = fmaxf(top, s[jt][v]);
  top = group_max(top);
  // (a column's own decision: whatever the wave's other columns hold, its sums are the same)
  const bool moves = top > m + 8.f || (m == -INFINITY && top > m);
  if (__any(moves)) {
    const float to = moves ? top : m, alpha = moves ? __builtin_amdgcn_exp2f(m - to) : 1.f;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int v = 0; v < 4; ++v) o[dt][v] *= alpha;
    m = to;
  }
  const float use = m == -INFINITY ? 0.f : m;      // nothing seen yet: 2^(-inf - 0) = 0
  float sum = 0.f;
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      s[jt][v] = __builtin_amdgcn_exp2f(s[jt][v] - use);
      sum += s[jt][v];
    }
  l += group_sum(sum);
#pragma unroll
  for (int pr = 0; pr < 2; ++pr) {
    const float x[8] = {s[2 * pr][0], s[2 * pr][1], s[2 * pr][2], s[2 * pr][3], s[2 * pr + 1][0], s[2 * pr + 1][1], s[2 * pr + 1][2], s[2 * pr + 1][3]};
    pieces_of(x, pf[pr]);
  }
}
// 1 / l; a row that sees nothing but scores of -inf has no weight to share out: 0.  (NaN stays.)
__device__ __forceinline__ float over(float l) { return l == 0.f ? 0.f : 1.0f / l; }
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l); }

// ------------------------------------------------------------------------------------------ single tokens
// One new token per sequence.  grid (runs, nkv * ceil(g / 16), B), block 64: a wave takes a run of tiles for up to 16 of the g heads
// of a kv head and leaves unnormalised sums, maximum and denominator; a second kernel joins the runs in order.  How the tiles
// are cut into runs depends on the token's own position only, so a token's result does not depend on what else the step holds.
// A whole tile (16 KiB with heads of 128) is in registers while the one before it is worked on: codes take half the registers that
// the numbers would.
__host__ __device__ __forceinline__ int e4m3_tiles_per_run(int p) { return p >= 4096 ? 3 : 1; }
__host__ __device__ __forceinline__ int e4m3_runs_at(int p) { return p / E4M3_TILE / e4m3_tiles_per_run(p) + 1; }
static int e4m3_most_runs(int max_end) {
  const int tiles = (max_end + E4M3_TILE - 1) / E4M3_TILE;
  return max(min(tiles, 64), (tiles + 2) / 3) + 1;
}

template <int DT>
struct TileCodes {
  u32x4 k[4][DT / 4], v[DT];
  f32x4 ks, vs;
};
template <int DT>
__device__ __forceinline__ void fetch(TileCodes<DT>& t, const E4m3Pages& p, const int* row, int tile, int kvh) {
  const int lane = threadIdx.x % 64, r = lane % 16, c = lane / 16;
  int in_page;
  int64_t head = e4m3_head_of(p, row, tile, kvh, in_page);
  if (head < 0) head = 0;      // (no page: the host has checked that there is one)
  const int64_t at = e4m3_tile_at(p, head, in_page), scales = e4m3_scale_at(p, head, in_page);
  t.ks = *reinterpret_cast<const f32x4*>(p.k_scale + scales);
  t.vs = *reinterpret_cast<const f32x4*>(p.v_scale + scales);
  // (chunks behind the head's end: the last one again, against zeros of the query; dimensions behind it are not stored)
#pragma unroll
  for (int ks = 0; ks < DT / 4; ++ks) {
    const int ch = min(4 * ks + c, p.hd / 16 - 1);
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
      t.k[jt][ks] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.k + at + ch * 1024 + (16 * jt + r) * 16));
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int d = min(16 * dt, p.hd - 16) + r;
    t.v[dt] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.v + at + d * 64 + 16 * c));
  }
}

template <int DT, bool MOD>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(DT > 8 ? 1 : 2))) void e4m3_decode_kernel(E4m3Attn a) {
  const int b = blockIdx.z, g = a.nh / a.nkv, ngc = (g + 15) / 16, kvh = blockIdx.y / ngc, cg = blockIdx.y % ngc;
  const int lane = threadIdx.x, r = lane % 16, c = lane / 16, hd = a.pages.hd;
  const int p = a.start[b], lo = reach_lo(p, a.window, a.mod.chunk);
  const int S = e4m3_tiles_per_run(p), n_runs = e4m3_runs_at(p);
  if ((int)blockIdx.x >= n_runs) return;
  const bool valid = cg * 16 + r < g;
  const int h = kvh * g + (valid ? cg * 16 + r : 0);
  const int* row = a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride;
  const float r1 = MOD && a.mod.r1 ? a.mod.r1[h] : 0.f, r2 = MOD && a.mod.r1 ? a.mod.r2[h] : 0.f;
  bf16x8 qf[2 * (DT / 4)][PIECES];
  const act_t* qrow = a.q + ((int64_t)a.cu[b] * a.nh + h) * hd;
#pragma unroll
  for (int ks = 0; ks < DT / 4; ++ks)
#pragma unroll
    for (int half = 0; half < 2; ++half) load_query(qf[2 * ks + half], qrow, 64 * ks + 16 * c + 8 * half, hd, valid);
  for (int run = blockIdx.x; run < n_runs; run += gridDim.x) {
    const int beg = max(run * S, lo / E4M3_TILE), end = min((run + 1) * S, p / E4M3_TILE + 1);
    if (beg >= end) continue;
    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    auto step = [&](const TileCodes<DT>& t, int tile) {
      const int pos0 = tile * E4M3_TILE;
      f32x4 s[4];
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        s[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < DT / 4; ++ks)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const bf16x8 kf = numbers(t.k[jt][ks][2 * half], t.k[jt][ks][2 * half + 1], t.ks[jt]);
#pragma unroll
            for (int pc = PIECES - 1; pc >= 0; --pc)
              s[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[2 * ks + half][pc], s[jt], 0, 0, 0);
          }
      }
      final_scores<MOD>(s, a, r1, r2, pos0, p, lo, pos0 + E4M3_TILE - 1 > p || pos0 < lo);
      if (a.scores && valid) {
        float* at = a.scores + ((int64_t)b * a.nh + h) * a.ld_scores + pos0 + 4 * c;
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) *reinterpret_cast<f32x4*>(at + 16 * jt) = s[jt];
      }
      bf16x8 pf[2][PIECES];
      softmax_tile<DT>(s, o, m, l, pf);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
          const bf16x8 lo8 = numbers(t.v[dt][2 * pr], t.v[dt][2 * pr], t.vs[2 * pr]);
          const bf16x8 hi8 = numbers(t.v[dt][2 * pr + 1], t.v[dt][2 * pr + 1], t.vs[2 * pr + 1]);
          const bf16x8 vf = __builtin_shufflevector(lo8, hi8, 0, 1, 2, 3, 8, 9, 10, 11);
#pragma unroll
          for (int pc = PIECES - 1; pc >= 0; --pc) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[pr][pc], o[dt], 0, 0, 0);
        }
    };
    TileCodes<DT> t0, t1;
    fetch<DT>(t0, a.pages, row, beg, kvh);
    for (int tile = beg; tile < end; tile += 2) {
      if (tile + 1 < end) fetch<DT>(t1, a.pages, row, tile + 1, kvh);
      step(t0, tile);
      if (tile + 1 < end) {
        if (tile + 2 < end) fetch<DT>(t0, a.pages, row, tile + 2, kvh);
        step(t1, tile + 1);
      }
    }
    if (!valid) continue;
    float* out = a.partial + (((int64_t)b * a.nh + h) * a.max_runs + run) * (hd + 2);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      if (16 * dt < hd)
#pragma unroll
        for (int v = 0; v < 4; ++v) out[16 * dt + 4 * c + v] = o[dt][v];
    if (c == 0) {
      out[hd] = m;
      out[hd + 1] = l;
    }
  }
}

// Joins the runs of one (sequence, head) in order: grid (nh, B), a wave to every 64 dimensions, each working out the runs' weights
// for itself, 64 runs at a time.
__global__ __launch_bounds__(256) void e4m3_join_kernel(E4m3Attn a) {
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x % 64, hd = a.pages.hd;
  const int p = a.start[b], lo = reach_lo(p, a.window, a.mod.chunk), S = e4m3_tiles_per_run(p);
  const int beg = lo / E4M3_TILE / S, end = p / E4M3_TILE / S + 1, stride = hd + 2;
  const float* part = a.partial + ((int64_t)b * a.nh + h) * a.max_runs * stride;
  float m = a.mod.sink ? a.mod.sink[h] * LOG2E : -INFINITY;
  for (int i = beg + lane; i < end; i += 64) m = fmaxf(m, part[(int64_t)i * stride + hd]);
  m = wave_max(m);
  const float use = m == -INFINITY ? 0.f : m;
  float l = a.mod.sink ? __builtin_amdgcn_exp2f(a.mod.sink[h] * LOG2E - use) : 0.f;
  const int d = threadIdx.x;
  float acc = 0.f;
  for (int i0 = beg; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    float w = 0.f, wl = 0.f;
    if (i < end) {
      w = __builtin_amdgcn_exp2f(part[(int64_t)i * stride + hd] - use);
      wl = w * part[(int64_t)i * stride + hd + 1];
    }
    l += wave_sum(wl);
    const int n = min(64, end - i0);
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const float wj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), j));
      if (d < hd) acc = fmaf(wj, part[(int64_t)(i0 + j) * stride + d], acc);
    }
  }
  const int64_t t = a.cu[b];
  if (d < hd) a.out[(t * a.nh + h) * hd + d] = from_f32<act_t>(acc * over(l));
  if (a.lse && d == 0) a.lse[t * a.nh + h] = lse_of(m, l);
}

// The weights that a step of single tokens gives its positions: grid (tiles of 256 positions, nkv, B), a thread to a position.
__global__ __launch_bounds__(256) void e4m3_decode_weights_kernel(E4m3Attn a) {
  const int j = blockIdx.x * 256 + threadIdx.x, kvh = blockIdx.y, b = blockIdx.z, g = a.nh / a.nkv;
  const int p = a.start[b], lo = reach_lo(p, a.window, a.mod.chunk);
  if (j > p || j < lo) return;
  int in_page;
  const int64_t head = e4m3_head_of(a.pages, a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride, j / E4M3_TILE, kvh, in_page);
  if (head < 0) return;
  float w = 0.f;
  for (int i = 0; i < g; ++i) {
    const int h = kvh * g + i;
    w += __builtin_amdgcn_exp2f(a.scores[((int64_t)b * a.nh + h) * a.ld_scores + j] - a.lse[(int64_t)a.cu[b] * a.nh + h]);
  }
  a.pages.weight[head * a.pages.page_size + in_page * E4M3_TILE + j % E4M3_TILE] += w;
}

// ------------------------------------------------------------------------------------------ prompts
// grid (blocks of 64 QG new tokens x heads x sequences, the last blocks first), block 256: wave w takes QG groups of 16 tokens.  The
// cache already holds the step's keys and values.  A tile of codes is in registers on its way (32 bytes a thread and operand with
// heads of 128) while the one before becomes bfloat16 in LDS, once for all waves: the matrix cores then work on numbers as in a
// cache of 16 bits, and only memory sees that there are half the bytes.
template <int DT>
__device__ __forceinline__ int k_at(int row, int ch) { return row * (16 * DT) + ((ch ^ (row & (DT % 8 == 0 ? 15 : 7))) << 3); }
__device__ __forceinline__ int v_at(int d, int ch) { return d * E4M3_TILE + ((ch ^ (d & 7)) << 3); }

template <int DT, int QG, bool MOD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DT > 8 ? 1 : 2))) void e4m3_prompt_kernel(E4m3Attn a, int n_blocks) {
  extern __shared__ __attribute__((aligned(16))) __bf16 tiles[];
  constexpr int KS = DT / 2, CH = (E4M3_TILE * DT + 255) / 256, BUF = 2 * E4M3_TILE * 16 * DT;
  const int per_block = a.nh * a.B, hd = a.pages.hd;
  const int blk = n_blocks - 1 - (int)blockIdx.x / per_block, h = (int)blockIdx.x % per_block % a.nh, b = (int)blockIdx.x % per_block / a.nh;
  const int tid = threadIdx.x, lane = tid % 64, r = lane % 16, c = lane / 16, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int t0 = a.cu[b], n = a.cu[b + 1] - t0, qb = blk * 64 * QG;
  if (qb >= n) return;
  const int start = a.start[b], kvh = h / (a.nh / a.nkv);
  const int* row = a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride;
  const float r1 = MOD && a.mod.r1 ? a.mod.r1[h] : 0.f, r2 = MOD && a.mod.r1 ? a.mod.r2[h] : 0.f;
  bf16x8 qf[QG][KS][PIECES];
  f32x4 o[QG][DT];
  float m[QG], l[QG];
  int p[QG], lo[QG];
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const int qi = qb + (wave * QG + g) * 16 + r;
    const bool valid = qi < n;
    p[g] = valid ? start + qi : -1;
    lo[g] = reach_lo(p[g], a.window, a.mod.chunk);
    const act_t* qrow = a.q + ((int64_t)(t0 + (valid ? qi : 0)) * a.nh + h) * hd;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) load_query(qf[g][ks], qrow, 32 * ks + 8 * c, hd, valid);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[g][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[g] = a.mod.sink ? a.mod.sink[h] * LOG2E : -INFINITY;
    l[g] = a.mod.sink && m[g] != -INFINITY ? 1.f : 0.f;
  }
  const int wg_last = start + min(qb + 64 * QG, n) - 1;
  const int tile_beg = reach_lo(start + qb, a.window, a.mod.chunk) / E4M3_TILE, tile_end = wg_last / E4M3_TILE + 1;
  const int wq0 = qb + wave * 16 * QG;
  const bool has = wq0 < n;
  const int first = start + wq0, last = start + min(wq0 + 16 * QG, n) - 1;
  const int lo_last = reach_lo(last, a.window, a.mod.chunk);
  const int wave_beg = reach_lo(first, a.window, a.mod.chunk) / E4M3_TILE, wave_end = has ? last / E4M3_TILE + 1 : 0;

  u32x4 pk[CH], pv[CH];
  f32x4 ks4, vs4;
  const int chunks = E4M3_TILE * (hd / 16);
  auto fetch_tile = [&](int tile) {
    int in_page;
    int64_t head = e4m3_head_of(a.pages, row, tile, kvh, in_page);
    if (head < 0) head = 0;
    const int64_t at = e4m3_tile_at(a.pages, head, in_page), scales = e4m3_scale_at(a.pages, head, in_page);
    ks4 = *reinterpret_cast<const f32x4*>(a.pages.k_scale + scales);
    vs4 = *reinterpret_cast<const f32x4*>(a.pages.v_scale + scales);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at16 = min(tid + 256 * i, chunks - 1) * 16;
      pk[i] = *reinterpret_cast<const u32x4*>(a.pages.k + at + at16);
      pv[i] = *reinterpret_cast<const u32x4*>(a.pages.v + at + at16);
    }
  };
  auto stage = [&](__bf16* Ks) {
    __bf16* Vs = Ks + E4M3_TILE * 16 * DT;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = min(tid + 256 * i, chunks - 1), kr = at % 64, ch = at / 64, d = at / 4, vc = at % 4;
      const int blk16 = kr / 16;
      const float f = blk16 == 0 ? ks4[0] : blk16 == 1 ? ks4[1] : blk16 == 2 ? ks4[2] : ks4[3];
      *reinterpret_cast<bf16x8*>(Ks + k_at<DT>(kr, 2 * ch)) = numbers(pk[i][0], pk[i][1], f);
      *reinterpret_cast<bf16x8*>(Ks + k_at<DT>(kr, 2 * ch + 1)) = numbers(pk[i][2], pk[i][3], f);
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        const bf16x8 x = numbers(pv[i][2 * pr], pv[i][2 * pr], vs4[2 * pr]), y = numbers(pv[i][2 * pr + 1], pv[i][2 * pr + 1], vs4[2 * pr + 1]);
        *reinterpret_cast<bf16x8*>(Vs + v_at(d, 2 * vc + pr)) = __builtin_shufflevector(x, y, 0, 1, 2, 3, 8, 9, 10, 11);
      }
    }
  };
  // what lies behind a head's end in LDS is read against zeros of the queries (keys) or not stored (values): it has to be finite
  if (hd < 16 * DT) {
    for (int i = tid; i < 2 * BUF / 8; i += 256) *reinterpret_cast<bf16x8*>(tiles + 8 * i) = nothing();
    __syncthreads();
  }
  fetch_tile(tile_beg);
  stage(tiles);
  if (tile_beg + 1 < tile_end) fetch_tile(tile_beg + 1);
  __syncthreads();
  int cur = 0;
  for (int tile = tile_beg; tile < tile_end; ++tile, cur ^= BUF) {
    if (tile + 1 < tile_end) {
      stage(tiles + (cur ^ BUF));
      if (tile + 2 < tile_end) fetch_tile(tile + 2);
    }
    if (tile >= wave_beg && tile < wave_end) {
      const __bf16 *Ks = tiles + cur, *Vs = Ks + E4M3_TILE * 16 * DT;
      const int pos0 = tile * E4M3_TILE;
      const bool masked = pos0 + E4M3_TILE - 1 > first || pos0 < lo_last;
      f32x4 s[QG][4];
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
#pragma unroll
        for (int g = 0; g < QG; ++g) s[g][jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const bf16x8 kf = *reinterpret_cast<const bf16x8*>(Ks + k_at<DT>(16 * jt + r, 4 * ks + c));
#pragma unroll
          for (int g = 0; g < QG; ++g)
#pragma unroll
            for (int pc = PIECES - 1; pc >= 0; --pc) s[g][jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[g][ks][pc], s[g][jt], 0, 0, 0);
        }
      }
      bf16x8 pf[QG][2][PIECES];
#pragma unroll
      for (int g = 0; g < QG; ++g) {
        final_scores<MOD>(s[g], a, r1, r2, pos0, p[g], lo[g], masked);
        softmax_tile<DT>(s[g], o[g], m[g], l[g], pf[g]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
          const bf16x8 vf = *reinterpret_cast<const bf16x8*>(Vs + v_at(16 * dt + r, 2 * c + pr));
#pragma unroll
          for (int g = 0; g < QG; ++g)
#pragma unroll
            for (int pc = PIECES - 1; pc >= 0; --pc) o[g][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[g][pr][pc], o[g][dt], 0, 0, 0);
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    if (p[g] < 0) continue;
    const float inv = over(l[g]);
    const int64_t at = (int64_t)(t0 + p[g] - start) * a.nh + h;
    if (a.lse && c == 0) a.lse[at] = lse_of(m[g], l[g]);
    act_t* orow = a.out + at * hd;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      if (16 * dt < hd) {
        const f32x4 x = o[g][dt] * inv;
#if defined(TQ_ACT_BF16)
        *reinterpret_cast<uint2*>(orow + 16 * dt + 4 * c) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
#else
        *reinterpret_cast<f32x4*>(orow + 16 * dt + 4 * c) = x;
#endif
      }
  }
}

// The weights that a prompt gives its positions, from the scores once more and the rows' sums: grid (tiles, nkv, B), block 256.  A
// workgroup keeps a tile's keys in registers and goes through the tokens that may see it and the heads of its kv head, 16 tokens of one
// head to a wave at a time; one sum over lanes and waves at the end, in a fixed order.
template <int DT, bool MOD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DT > 8 ? 1 : 2))) void e4m3_prompt_weights_kernel(E4m3Attn a) {
  __shared__ float sums[4][E4M3_TILE];
  const int kvh = blockIdx.y, b = blockIdx.z, g = a.nh / a.nkv, hd = a.pages.hd;
  const int tid = threadIdx.x, lane = tid % 64, r = lane % 16, c = lane / 16, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int t0 = a.cu[b], n = a.cu[b + 1] - t0, start = a.start[b];
  const int tile = reach_lo(start, a.window, a.mod.chunk) / E4M3_TILE + (int)blockIdx.x, pos0 = tile * E4M3_TILE;
  if (n <= 0 || pos0 >= start + n) return;
  TileCodes<DT> t;
  const int* row = a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride;
  fetch<DT>(t, a.pages, row, tile, kvh);
  // the tokens that may see a position of the tile: from the tile's first to the last whose reach has its last
  const int from = max(pos0 - start, 0) / 16;
  int to = n;
  if (a.window > 0) to = (int)min((int64_t)to, (int64_t)pos0 + E4M3_TILE - 1 + a.window - start);
  if (a.mod.chunk > 0) to = (int)min((int64_t)to, (int64_t)((pos0 + E4M3_TILE - 1) / a.mod.chunk + 1) * a.mod.chunk - start);
  const int items = ((to + 15) / 16 - from) * g;
  f32x4 acc[4];
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) acc[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i = wave; i < items; i += 4) {
    const int h = kvh * g + i % g, qi = (from + i / g) * 16 + r;
    const bool valid = qi < n;
    const int p = valid ? start + qi : -1, lo = reach_lo(p, a.window, a.mod.chunk);
    const int64_t at = (int64_t)(t0 + (valid ? qi : 0)) * a.nh + h;
    const float lse = a.lse[at];
    const float r1 = MOD && a.mod.r1 ? a.mod.r1[h] : 0.f, r2 = MOD && a.mod.r1 ? a.mod.r2[h] : 0.f;
    f32x4 s[4];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) s[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < DT / 4; ++ks)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        bf16x8 qf[PIECES];
        load_query(qf, a.q + at * hd, 64 * ks + 16 * c + 8 * half, hd, valid);
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
          const bf16x8 kf = numbers(t.k[jt][ks][2 * half], t.k[jt][ks][2 * half + 1], t.ks[jt]);
#pragma unroll
          for (int pc = PIECES - 1; pc >= 0; --pc) s[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[pc], s[jt], 0, 0, 0);
        }
      }
    final_scores<MOD>(s, a, r1, r2, pos0, p, lo, true);
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[jt][v] += __builtin_amdgcn_exp2f(s[jt][v] - lse);
  }
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float x = lanes_fold<16>(acc[jt][v], LanesSum());
      if (r == 0) sums[wave][16 * jt + 4 * c + v] = x;
    }
  __syncthreads();
  if (tid < E4M3_TILE && pos0 + tid < start + n) {
    int in_page;
    const int64_t head = e4m3_head_of(a.pages, row, tile, kvh, in_page);
    if (head >= 0)
      a.pages.weight[head * a.pages.page_size + in_page * E4M3_TILE + tid] += (sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid]);
  }
}

// ------------------------------------------------------------------------------------------ launch
template <int DT, bool MOD>
static int launch_decode(const E4m3Attn& a, int max_end, hipStream_t st) {
  const int g = a.nh / a.nkv;
  hipLaunchKernelGGL((e4m3_decode_kernel<DT, MOD>), dim3(e4m3_runs_at(max_end > 0 ? max_end - 1 : 0), a.nkv * ((g + 15) / 16), a.B), dim3(64), 0, st, a);
  hipLaunchKernelGGL(e4m3_join_kernel, dim3(a.nh, a.B), dim3((a.pages.hd + 63) / 64 * 64), 0, st, a);
  if (a.scores) hipLaunchKernelGGL(e4m3_decode_weights_kernel, dim3((max_end + 255) / 256, a.nkv, a.B), dim3(256), 0, st, a);
  return 0;
}
template <int DT, int QG, bool MOD>
static int launch_prompt(const E4m3Attn& a, int max_new, hipStream_t st) {
  const size_t shmem = 2 * (size_t)2 * E4M3_TILE * 16 * DT * sizeof(__bf16);
  const hipError_t e = hipFuncSetAttribute((const void*)e4m3_prompt_kernel<DT, QG, MOD>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem);
  if (e != hipSuccess) return (int)e;
  const int n_blocks = (max_new + 64 * QG - 1) / (64 * QG);
  if ((int64_t)n_blocks * a.nh * a.B > 0xFFFFFF) return TQ_ERR_UNSUPPORTED;      // (a launch's threads are counted in 32 bits)
  hipLaunchKernelGGL((e4m3_prompt_kernel<DT, QG, MOD>), dim3(n_blocks * a.nh * a.B), dim3(256), shmem, st, a, n_blocks);
  return 0;
}
template <int DT, bool MOD>
static int launch_as(const E4m3Attn& a, int decode, int max_new, int max_end, hipStream_t st) {
  if (decode) return launch_decode<DT, MOD>(a, max_end, st);
  // two groups of 16 tokens to a wave halve the reads from LDS, where that leaves the chip two workgroups to a compute unit
  const bool two = PIECES == 1 && DT <= 8 && (int64_t)((max_new + 127) / 128) * a.nh * a.B >= 512;
  const int rc = two ? launch_prompt<DT, (PIECES == 1 && DT <= 8) ? 2 : 1, MOD>(a, max_new, st) : launch_prompt<DT, 1, MOD>(a, max_new, st);
  if (rc) return rc;
  if (a.lse)
    hipLaunchKernelGGL((e4m3_prompt_weights_kernel<DT, MOD>), dim3((max_end + E4M3_TILE - 1) / E4M3_TILE, a.nkv, a.B), dim3(256), 0, st, a);
  return 0;
}
template <int DT>
static int launch(const E4m3Attn& a, int decode, int max_new, int max_end, hipStream_t st) {
  return a.mod.cap > 0.f || a.mod.r1 ? launch_as<DT, true>(a, decode, max_new, max_end, st) : launch_as<DT, false>(a, decode, max_new, max_end, st);
}

// Floats of scratch: for decoding the runs' sums, with weights the scores and the rows' sums too; for prompts with weights the rows' sums.
TQ_API int64_t tq_e4m3_attention_scratch(int T, int B, int nh, int hd, int max_end, int decode, int weights) {
  const int64_t rows = weights ? (int64_t)T * nh : 0;
  if (!decode) return rows;
  const int64_t ld = (max_end + E4M3_TILE - 1) / E4M3_TILE * E4M3_TILE;
  return (int64_t)B * nh * e4m3_most_runs(max_end) * (hd + 2) + (weights ? (int64_t)B * nh * ld : 0) + rows + 4;
}

// q, out [T][nh][hd]; tokens as runs (cu, slots, start) whose keys and values the cache holds already.  decode != 0: one token per
// sequence.  weight (null: none): every position's is raised by what it receives.  max_end: the largest position + 1.
TQ_API int tq_e4m3_attention(const void* q, void* out, const int* cu, const int* slots, const int* start, int T, int B, int nh, int nkv,
                             int hd, int window, float scale, float softcap, const float* r1, const float* r2, int chunk,
                             const float* sink, const void* k, const void* v, const float* k_scale, const float* v_scale, float* weight,
                             const int* table, int bt_stride, int page_size, int heads, int head0, float* scratch, int decode, int max_new,
                             int max_end, hipStream_t st) {
  if (B <= 0 || T <= 0) return 0;
  if ((r1 == nullptr) != (r2 == nullptr) || chunk < 0 || softcap < 0.f || window < 0 || nh <= 0 || max_new <= 0 || max_end <= 0) return TQ_ERR_BAD_ARG;
  if (!e4m3_pages_fit(page_size, heads, head0, nkv, hd) || nh % nkv != 0 || nh > 65535 || B > 65535) return TQ_ERR_UNSUPPORTED;
  if ((decode || weight) && !scratch) return TQ_ERR_BAD_ARG;
  E4m3Attn a{(const act_t*)q, (act_t*)out, cu, slots, start, B, nh, nkv, window, scale, ScoreMod{softcap, r1, r2, chunk, sink, nullptr, 0},
             nullptr, e4m3_most_runs(max_end), nullptr, 0, nullptr,
             E4m3Pages{(uint8_t*)k, (uint8_t*)v, (float*)k_scale, (float*)v_scale, weight, table, bt_stride, page_size, heads, head0, hd}};
  if (decode) {
    // (the scores first: their rows are read and written 16 bytes at a time)
    if (weight) {
      a.ld_scores = (max_end + E4M3_TILE - 1) / E4M3_TILE * E4M3_TILE;
      a.scores = scratch;
      scratch += (int64_t)B * nh * a.ld_scores;
    }
    a.partial = scratch;
    scratch += (int64_t)B * nh * a.max_runs * (hd + 2);
  }
  if (weight) a.lse = scratch;
  const int dt = hd / 16;
  const int rc = dt <= 4 ? launch<4>(a, decode, max_new, max_end, st) : dt <= 8 ? launch<8>(a, decode, max_new, max_end, st)
               : dt <= 12 ? launch<12>(a, decode, max_new, max_end, st) : launch<16>(a, decode, max_new, max_end, st);
  if (rc) return rc;
  TQ_LAUNCH_CHECK();
  return 0;
}
