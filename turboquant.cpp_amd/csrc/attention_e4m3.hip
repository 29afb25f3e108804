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

// What becomes of a product (final_scores), worked out once on the host.
struct Change {
  float scale2, cap2;           // scale, cap in units of log2
  float ky, k2;                 // scale / cap; 2 log2(e) scale / cap
  float near[5];                // tanh(y) / y in powers of y^2, times scale2
};
static Change change_of(float scale, float cap) {
  Change c{scale * LOG2E, cap * LOG2E, cap > 0.f ? scale / cap : 0.f, cap > 0.f ? 2.f * LOG2E * scale / cap : 0.f, {}};
  const double p[5] = {0.99999998675739, -0.33333067944422656, 0.13324750504782334, -0.05298423882762508, 0.017131344428621548};
  for (int i = 0; i < 5; ++i) c.near[i] = (float)(p[i] * (double)scale * 1.4426950408889634);
  return c;
}

struct E4m3Attn {
  const act_t* q;               // [T][nh][hd]
  act_t* out;                   // [T][nh][hd]
  const int* cu;                // [B + 1]
  const int* slots;
  const int* start;
  int B, nh, nkv, window;
  float scale;
  ScoreMod mod;
  Change ch;
  float* partial;               // decoding: [B][nh][max_runs][hd + 2]
  int max_runs;
  float* scores;                // with weights: decoding [B][nh][ld_scores], a column's scores in units of log2; prompts [B][cuts][nh][ld_scores], a
                                // cut's sums of probabilities
  int64_t ld_scores;
  float* lse;                   // prompts with weights: [T][nh] log2 of a row's sum of 2^score, the sink's included
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
// Eight numbers of a query from dimension d on.
__device__ __forceinline__ void load_query(bf16x8 (&out)[PIECES], const act_t* row, int d) {
#if defined(TQ_ACT_BF16)
  out[0] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(row + d));
#else
  const float4 a = *reinterpret_cast<const float4*>(row + d), b = *reinterpret_cast<const float4*>(row + d + 4);
  const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  pieces_of(x, out);
#endif
}
// The same, and zeros behind the head's end and for a column without a query (whose row is some other's: a read without a condition does not
// keep the next from being on its way).
__device__ __forceinline__ void load_query(bf16x8 (&out)[PIECES], const act_t* row, int d, int hd, bool valid) {
  load_query(out, row, min(d, hd - 8));
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const u32x4 w = __builtin_bit_cast(u32x4, out[p]), none = {0u, 0u, 0u, 0u};
    out[p] = __builtin_bit_cast(bf16x8, valid && d < hd ? w : none);
  }
}
__device__ __forceinline__ float group_max(float v) { return with_lane_xor<32>(with_lane_xor<16>(v, LanesMax()), LanesMax()); }
__device__ __forceinline__ float group_sum(float v) { return with_lane_xor<32>(with_lane_xor<16>(v, LanesSum()), LanesSum()); }
// Scores of a tile as the softmax takes them, and -inf where the column does not see the position, for one group of 16 columns.  MOD:
// scaled, capped, biased, in units of log2; else (a positive scale alone) as the product left them, and the scale joins the exponent.
// The cap in the bfloat16 library, cap tanh(y) with y = x / cap, as good as 32 bits allow, for the weights that positions receive: up to |y| = 1/2
// y P(y^2), P of degree 4 through tanh(y) / y at the five Chebyshev nodes (off by 1.3e-8 of itself); beyond, 1 - 2 / (e^(2 |y|) + 1), whose second term
// is small enough there, and which needs no bounds: e^.. may be infinite.  (That one alone is off by 2^-23 of the cap, whatever the score:
// 2e-6 of a weight at a cap of 50.)  A tile without large scores, as most are, passes the second form over.  In one that has some a score's own size
// decides where weights come of it (`exact`: single tokens with weights, prompts' second pass); else the second form serves for all of the tile.
// 2,048 tokens of 28 heads behind as many, a cap of 30, scores of a standard deviation of 0.9, 3.6 and 7.2: 167, 169 and 184 us, with weights 293, 297 and
// 364 (175, 176 and 178, with weights 300, 298 and 300 with the second form alone).
__device__ __forceinline__ float capped(float s, const Change& ch) {
  const float y = s * ch.ky, z = y * y;
  return s * fmaf(z, fmaf(z, fmaf(z, fmaf(z, ch.near[4], ch.near[3]), ch.near[2]), ch.near[1]), ch.near[0]);
}
__device__ __forceinline__ float capped_far(float s, const Change& ch) {
  const float e = __builtin_amdgcn_exp2f(fabsf(s) * fabsf(ch.k2));
  return copysignf(fmaf(-2.f * ch.cap2, __builtin_amdgcn_rcpf(e + 1.f), ch.cap2), s * ch.k2);
}
template <bool MOD>
__device__ __forceinline__ void final_scores(f32x4 (&s)[4], const E4m3Attn& a, bool exact, float r1, float r2, int pos0, int p, int lo, bool masked) {
  const int c = (threadIdx.x % 64) / 16;
  if constexpr (MOD) {
#if defined(TQ_ACT_BF16)
    if (a.mod.cap > 0.f) {
      float top = 0.f;
#pragma unroll
      for (int jt = 0; jt < 4; ++jt)
#pragma unroll
        for (int v = 0; v < 4; ++v) top = fmaxf(top, fabsf(s[jt][v]));
      const bool far = __any(top * fabsf(a.ch.ky) > 0.5f);
      if (far && exact) {
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
#pragma unroll
          for (int v = 0; v < 4; ++v) s[jt][v] = fabsf(s[jt][v] * a.ch.ky) > 0.5f ? capped_far(s[jt][v], a.ch) : capped(s[jt][v], a.ch);
      } else if (far) {
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
#pragma unroll
          for (int v = 0; v < 4; ++v) s[jt][v] = capped_far(s[jt][v], a.ch);
      } else {
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
#pragma unroll
          for (int v = 0; v < 4; ++v) s[jt][v] = capped(s[jt][v], a.ch);
      }
    } else {
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) s[jt] *= a.ch.scale2;
    }
    if (a.mod.r1)
#pragma unroll
      for (int jt = 0; jt < 4; ++jt)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          s[jt][v] -= r1 * __builtin_amdgcn_logf(fmaf(r2, (float)max(p - (pos0 + 16 * jt + 4 * c + v), 0), 1.f));
#else
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        s[jt][v] = mod_score(s[jt][v] * a.scale, a.mod.cap, a.mod.r1 != nullptr, r1, r2, p - (pos0 + 16 * jt + 4 * c + v)) * LOG2E;
#endif
  }
  if (masked) {
    asm volatile("");      // (a branch: as conditions the comparisons would be a third of the instructions of tiles that need none)
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int key = pos0 + 16 * jt + 4 * c + v;
        s[jt][v] = key <= p && key >= lo ? s[jt][v] : -INFINITY;
      }
  }
}
// The part of a tile between its products for one group of 16 columns: scores in, probabilities as operands out.  `scale2`: what is left
// to multiply the scores by (final_scores), positive.  l is the lane's share of a column's sum: the four lanes' shares are added at the end.
template <int DT>
__device__ __forceinline__ void softmax_tile(f32x4 (&s)[4], f32x4 (&o)[DT], float& m, float& l, float scale2, bf16x8 (&pf)[2][PIECES]) {
  float top = -INFINITY;
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
#pragma unroll
    for (int v = 0; v < 4; ++v) top = fmaxf(top, s[jt][v]);
  top = group_max(top) * scale2;
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
      s[jt][v] = __builtin_amdgcn_exp2f(fmaf(s[jt][v], scale2, -use));
      sum += s[jt][v];
    }
  l += sum;
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
// One new token per sequence, or none.  A wave takes tiles for up to 16 of the g heads of a kv head, run by run, and leaves a run's unnormalised
// sums, maximum and denominator; the runs are then joined in order.  How the tiles are cut into runs depends on the token's own
// position and on g only, so a token's result does not depend on what else the step holds.  Up to SHORT_END positions a workgroup does
// it all, its waves' runs meeting in LDS: one launch.  Beyond, a wave streams through as many runs as make some thousands of
// waves, and a second launch joins.
// Bound by the bytes of the cache: 16 KiB of codes a tile with heads of 128.  A tile's keys are asked for as soon as the one before
// has been multiplied, its values when that one's have: 64 registers hold what is on its way and what is worked on.
// Runs leave g (hd + 2) numbers of 32 bits each, written and read again, for 128 hd bytes a tile: with more heads to a kv head they
// are longer.
#define SHORT_END 1024
#define SHORT_WAVES 8
__host__ __device__ __forceinline__ int e4m3_tiles_per_run(int p, int g) { return p < SHORT_END ? 1 : max(p < 4096 ? 1 : 3, min(4, (g + 1) / 2)); }
__host__ __device__ __forceinline__ int e4m3_runs_at(int p, int g) { return p / E4M3_TILE / e4m3_tiles_per_run(p, g) + 1; }
// Most runs of a token at a position below max_end.
static int e4m3_most_runs(int max_end, int g) {
  int most = 1;
  const int ends[4] = {SHORT_END, 4096, max_end, 0};
  for (int e : ends)
    if (e > 0) most = max(most, e4m3_runs_at(min(e, max_end) - 1, g));
  return most;
}

template <int DT, bool MOD>
struct DecodeWave {
  const E4m3Attn& a;
  const int* row;
  int kvh, p, lo, h, r, c;
  bool valid;
  float r1, r2;
  bf16x8 qf[2 * (DT / 4)][PIECES];
  u32x4 k[4][DT / 4], v[DT];
  f32x4 ks, vs;
  f32x4 o[DT];
  float m, l;

  __device__ __forceinline__ DecodeWave(const E4m3Attn& args, int b, int kv, int cg) : a(args), kvh(kv) {
    const int lane = threadIdx.x % 64, g = a.nh / a.nkv;
    r = lane % 16;
    c = lane / 16;
    p = a.start[b];
    lo = reach_lo(p, a.window, a.mod.chunk);
    valid = cg * 16 + r < g;
    h = kvh * g + (valid ? cg * 16 + r : 0);
    row = a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride;
    r1 = MOD && a.mod.r1 ? a.mod.r1[h] : 0.f;
    r2 = MOD && a.mod.r1 ? a.mod.r2[h] : 0.f;
    clear();
  }
  // (behind the first tile's codes, which are then on their way)
  __device__ __forceinline__ void take_query(int b) {
    const int hd = a.pages.hd;
    const act_t* qrow = a.q + ((int64_t)a.cu[b] * a.nh + h) * hd;
#pragma unroll
    for (int s = 0; s < DT / 4; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half) load_query(qf[2 * s + half], qrow, 64 * s + 16 * c + 8 * half, hd, valid);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }
  __device__ __forceinline__ int64_t place(int tile, int64_t& scales) const {
    int in_page;
    int64_t head = e4m3_head_of(a.pages, row, tile, kvh, in_page);
    if (head < 0) head = 0;      // (no page: the host has checked that there is one)
    scales = e4m3_scale_at(a.pages, head, in_page);
    return e4m3_tile_at(a.pages, head, in_page);
  }
  // (chunks behind the head's end: the last one again, against zeros of the query; dimensions behind it are not stored)
  __device__ __forceinline__ void fetch_k(int tile) {
    int64_t scales;
    const uint8_t* at = a.pages.k + place(tile, scales);
    ks = *reinterpret_cast<const f32x4*>(a.pages.k_scale + scales);
#pragma unroll
    for (int s = 0; s < DT / 4; ++s) {
      const int ch = min(4 * s + c, a.pages.hd / 16 - 1);
#pragma unroll
      for (int jt = 0; jt < 4; ++jt)
        k[jt][s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at + (uint32_t)(ch * 1024 + (16 * jt + r) * 16)));
    }
  }
  __device__ __forceinline__ void fetch_v(int tile) {
    int64_t scales;
    const uint8_t* at = a.pages.v + place(tile, scales);
    vs = *reinterpret_cast<const f32x4*>(a.pages.v_scale + scales);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      v[dt] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at + (uint32_t)((min(16 * dt, a.pages.hd - 16) + r) * 64 + 16 * c)));
  }
  // One tile; `next`, if there is one, is asked for meanwhile.
  __device__ __forceinline__ void step(int b, int tile, int next) {
    const int pos0 = tile * E4M3_TILE;
    f32x4 s[4];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      s[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DT / 4; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const bf16x8 kf = numbers(k[jt][i][2 * half], k[jt][i][2 * half + 1], ks[jt]);
#pragma unroll
          for (int pc = PIECES - 1; pc >= 0; --pc)
            s[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[2 * i + half][pc], s[jt], 0, 0, 0);
        }
    }
    if (next >= 0) fetch_k(next);
    final_scores<MOD>(s, a, a.scores != nullptr, r1, r2, pos0, p, lo, pos0 + E4M3_TILE - 1 > p || pos0 < lo);
    if (a.scores && valid) {
      float* at = a.scores + ((int64_t)b * a.nh + h) * a.ld_scores + pos0 + 4 * c;
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) *reinterpret_cast<f32x4*>(at + 16 * jt) = MOD ? s[jt] : s[jt] * a.ch.scale2;
    }
    bf16x8 pf[2][PIECES];
    softmax_tile<DT>(s, o, m, l, MOD ? 1.f : a.ch.scale2, pf);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        const bf16x8 x = numbers(v[dt][2 * pr], v[dt][2 * pr], vs[2 * pr]), y = numbers(v[dt][2 * pr + 1], v[dt][2 * pr + 1], vs[2 * pr + 1]);
        const bf16x8 vf = __builtin_shufflevector(x, y, 0, 1, 2, 3, 8, 9, 10, 11);
#pragma unroll
        for (int pc = PIECES - 1; pc >= 0; --pc) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[pr][pc], o[dt], 0, 0, 0);
      }
    if (next >= 0) fetch_v(next);
  }
  // A run's sums to its place, and a new run.
  __device__ __forceinline__ void leave(float* out) {
    l = group_sum(l);
    if (valid) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        if (16 * dt < a.pages.hd)
#pragma unroll
          for (int e = 0; e < 4; ++e) out[16 * dt + 4 * c + e] = o[dt][e];
      if (c == 0) {
        out[a.pages.hd] = m;
        out[a.pages.hd + 1] = l;
      }
    }
    clear();
  }
};

// The maximum of a head's runs [beg, end), `stride` numbers apart, and the sink; and the sum of their denominators brought to it, 64
// runs at a time.  `w`: of the first 64 runs, the lane's run's factor.
__device__ __forceinline__ void join_sums(const E4m3Attn& a, const float* part, int stride, int beg, int end, int h, float& m, float& l, float& w) {
  const int lane = threadIdx.x % 64, hd = a.pages.hd;
  // (the first 64 runs' two numbers at once: most sequences have no more)
  const float* mine = part + (int64_t)min(beg + lane, end - 1) * stride + hd;
  const float m0 = mine[0], l0 = mine[1];
  m = fmaxf(a.mod.sink ? a.mod.sink[h] * LOG2E : -INFINITY, beg + lane < end ? m0 : -INFINITY);
  for (int i = beg + 64 + lane; i < end; i += 64) m = fmaxf(m, part[(int64_t)i * stride + hd]);
  m = wave_max(m);
  const float use = m == -INFINITY ? 0.f : m;
  l = a.mod.sink ? __builtin_amdgcn_exp2f(a.mod.sink[h] * LOG2E - use) : 0.f;
  w = beg + lane < end ? __builtin_amdgcn_exp2f(m0 - use) : 0.f;
  l += wave_sum(beg + lane < end ? w * l0 : 0.f);
  for (int i0 = beg + 64; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    l += wave_sum(i < end ? __builtin_amdgcn_exp2f(part[(int64_t)i * stride + hd] - use) * part[(int64_t)i * stride + hd + 1] : 0.f);
  }
}
// Joins the runs of one head and writes the output row; gives log2 of the row's sum.  Values are added in four strands by run, and the
// strands at the end.  MINE: the wave shares the head with three others and takes strand `mine` (the strands meet in `strands`,
// [4][256]); else it takes all four.  E: 64 dimensions that a head has at most.
template <bool MINE, int E>
__device__ __forceinline__ float join_runs(const E4m3Attn& a, const float* part, int stride, int beg, int end, int h, int64_t t, int mine, float* strands) {
  constexpr int NS = MINE ? 1 : 4, NJ = MINE ? 16 : 1;
  const int lane = threadIdx.x % 64, hd = a.pages.hd;
  float v[NJ][E] = {};
  // a strand's values of 64 runs are asked for before the factors are known
  auto ask = [&](int i0) {
#pragma unroll
    for (int k = 0; k < NJ; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (64 * e < hd && i0 + 4 * k + mine < end) v[k][e] = part[(int64_t)(i0 + 4 * k + mine) * stride + min(64 * e + lane, hd - 1)];
  };
  if constexpr (MINE) ask(beg);
  float m, l, w;
  join_sums(a, part, stride, beg, end, h, m, l, w);
  const float use = m == -INFINITY ? 0.f : m;
  float acc[NS][E] = {};
  for (int i0 = beg; i0 < end; i0 += 64) {
    if (i0 > beg) {
      w = i0 + lane < end ? __builtin_amdgcn_exp2f(part[(int64_t)(i0 + lane) * stride + hd] - use) : 0.f;
      if constexpr (MINE) ask(i0);
    }
    const int n = min(64, end - i0);
    if constexpr (MINE) {
#pragma unroll
      for (int k = 0; k < NJ; ++k) {
        if (4 * k + mine >= n) break;
        const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), 4 * k + mine));
#pragma unroll
        for (int e = 0; e < E; ++e) acc[0][e] = fmaf(ws, v[k][e], acc[0][e]);
      }
    } else {
#pragma unroll 2
      for (int j = 0; j < n; j += 4) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (j + s >= n) break;
          const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), j + s));
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (64 * e < hd) acc[s][e] = fmaf(ws, part[(int64_t)(i0 + j + s) * stride + min(64 * e + lane, hd - 1)], acc[s][e]);
        }
      }
    }
  }
  const float inv = over(l);
  act_t* out = a.out + (t * a.nh + h) * hd;
  if constexpr (MINE) {
#pragma unroll
    for (int e = 0; e < E; ++e) strands[256 * mine + 64 * e + lane] = acc[0][e];
    __syncthreads();
    const int d = threadIdx.x;
    if (d < hd) out[d] = from_f32<act_t>(((strands[d] + strands[256 + d]) + (strands[512 + d] + strands[768 + d])) * inv);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (64 * e + lane < hd) out[64 * e + lane] = from_f32<act_t>(((acc[0][e] + acc[1][e]) + (acc[2][e] + acc[3][e])) * inv);
  }
  return lse_of(m, l);
}
// The weights of one token that four neighbouring positions from j on (of one tile, a multiple of four) receive: sums over the g heads
// of a kv head, whose sums `lse` has.  `ask` first, for eight heads' scores.
struct WeightOf {
  f32x4 s[8];
  __device__ __forceinline__ void ask(const E4m3Attn& a, int b, int kvh, int i0, int j) {
    const int g = a.nh / a.nkv;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < g) s[i] = *reinterpret_cast<const f32x4*>(a.scores + ((int64_t)b * a.nh + kvh * g + i0 + i) * a.ld_scores + j);
  }
  __device__ __forceinline__ void add(const E4m3Attn& a, const int* row, int b, int kvh, int j, int lo, int p, const float* lse) {
    const int g = a.nh / a.nkv;
    int in_page;
    const int64_t head = e4m3_head_of(a.pages, row, j / E4M3_TILE, kvh, in_page);
    if (head < 0) return;
    f32x4* to = reinterpret_cast<f32x4*>(a.pages.weight + head * a.pages.page_size + in_page * E4M3_TILE + j % E4M3_TILE);
    const f32x4 was = *to;
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < g; i0 += 8) {
      if (i0) ask(a, b, kvh, i0, j);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < g)
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] += __builtin_amdgcn_exp2f(s[i][e] - lse[i0 + i]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = j + e >= lo && j + e <= p ? was[e] + w[e] : was[e];
    *to = w;
  }
};

// Runs of all but the shortest sequences: grid (waves, nkv * ceil(g / 16), B), block 64; a wave streams through neighbouring runs.
template <int DT, bool MOD>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(DT > 12 || DT * PIECES > 24 ? 1 : DT * PIECES >= 8 ? 2 : 3))) void e4m3_decode_kernel(E4m3Attn a) {
  const int b = blockIdx.z, g = a.nh / a.nkv, ngc = (g + 15) / 16;
  const int p = a.start[b], S = e4m3_tiles_per_run(p, g), lo = reach_lo(p, a.window, a.mod.chunk);
  const int first_run = lo / E4M3_TILE / S, n_runs = e4m3_runs_at(p, g) - first_run, each = (n_runs + (int)gridDim.x - 1) / (int)gridDim.x;
  const int run0 = first_run + (int)blockIdx.x * each, run1 = min(run0 + each, first_run + n_runs);
  if (run0 >= run1 || a.cu[b + 1] == a.cu[b]) return;
  DecodeWave<DT, MOD> w(a, b, blockIdx.y / ngc, blockIdx.y % ngc);
  const int beg = max(run0 * S, lo / E4M3_TILE), end = min(run1 * S, p / E4M3_TILE + 1);
  float* out = a.partial + ((int64_t)b * a.nh + w.h) * a.max_runs * (a.pages.hd + 2);
  w.fetch_k(beg);
  w.fetch_v(beg);
  w.take_query(b);
  for (int tile = beg; tile < end; ++tile) {
    w.step(b, tile, tile + 1 < end ? tile + 1 : -1);
    if ((tile + 1) % S == 0 || tile + 1 == end) w.leave(out + (int64_t)(tile / S) * (a.pages.hd + 2));
  }
}

// Joins them: blocks 0 .. nh B - 1 a head each, four waves with a strand of its runs each; behind them, with weights, blocks of 1,024 positions
// of one (sequence, kv head), which work the heads' sums out for themselves.
template <int E>
__global__ __launch_bounds__(256) void e4m3_join_kernel(E4m3Attn a, int blocks_of_weights) {
  __shared__ float lds[4 * 256];
  const int stride = a.pages.hd + 2, g = a.nh / a.nkv, wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const bool joins = (int)blockIdx.x < a.nh * a.B;
  const int x = joins ? (int)blockIdx.x : (int)blockIdx.x - a.nh * a.B;
  const int b = joins ? x / a.nh : x / blocks_of_weights / a.nkv;
  const int p = a.start[b], lo = reach_lo(p, a.window, a.mod.chunk), S = e4m3_tiles_per_run(p, g);
  const int beg = lo / E4M3_TILE / S, end = p / E4M3_TILE / S + 1;
  if (a.cu[b + 1] == a.cu[b]) return;
  if (joins) {
    const int h = x % a.nh;
    join_runs<true, E>(a, a.partial + ((int64_t)b * a.nh + h) * a.max_runs * stride, stride, beg, end, h, a.cu[b], wave, lds);
    return;
  }
  const int kvh = x / blocks_of_weights % a.nkv, j0 = x % blocks_of_weights * 1024, j = j0 + 4 * (int)threadIdx.x;
  if (j0 > p || j0 + 1023 < lo) return;
  const int* row = a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride;
  const bool has = j + 3 >= lo && j <= p;
  WeightOf of;
  if (has) of.ask(a, b, kvh, 0, j);
#pragma unroll 2
  for (int i = wave; i < g; i += 4) {      // (at most 1,024 heads to a kv head: the launcher has checked)
    const int h = kvh * g + i;
    float m, l, w;
    join_sums(a, a.partial + ((int64_t)b * a.nh + h) * a.max_runs * stride, stride, beg, end, h, m, l, w);
    if (lane == 0) lds[i] = lse_of(m, l);
  }
  __syncthreads();
  if (has) of.add(a, row, b, kvh, j, lo, p, lds);
}

// A step whose sequences all hold at most SHORT_END positions: grid (nkv * ceil(g / 16), B), one launch.
template <int DT, bool MOD>
__global__ __launch_bounds__(64 * SHORT_WAVES) __attribute__((amdgpu_waves_per_eu(DT * PIECES > 8 ? 1 : 2))) void e4m3_short_kernel(E4m3Attn a) {
  extern __shared__ float sums[];      // [runs][heads of the workgroup][hd + 2]
  __shared__ float lse[16];
  const int b = blockIdx.y, g = a.nh / a.nkv, ngc = (g + 15) / 16, kvh = blockIdx.x / ngc, cg = blockIdx.x % ngc;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, stride = a.pages.hd + 2, heads = min(16, g - 16 * cg);
  DecodeWave<DT, MOD> w(a, b, kvh, cg);
  const int beg = w.lo / E4M3_TILE, end = w.p / E4M3_TILE + 1;
  if (a.cu[b + 1] == a.cu[b]) return;
  if (beg + wave < end) {
    w.fetch_k(beg + wave);
    w.fetch_v(beg + wave);
  }
  w.take_query(b);
  for (int tile = beg + wave; tile < end; tile += SHORT_WAVES) {
    w.step(b, tile, tile + SHORT_WAVES < end ? tile + SHORT_WAVES : -1);
    w.leave(sums + ((tile - beg) * heads + min(w.r, heads - 1)) * stride);
  }
  __syncthreads();
  for (int i = wave; i < heads; i += SHORT_WAVES) {
    const float x = join_runs<false, DT <= 8 ? 2 : 4>(a, sums + i * stride, heads * stride, 0, end - beg, kvh * g + 16 * cg + i, a.cu[b], -1, nullptr);
    if (lane == 0) lse[i] = x;
  }
  if (!a.scores) return;
  __threadfence_block();      // (the scores that the workgroup's waves have written)
  __syncthreads();
  for (int j = w.lo / 4 * 4 + 4 * (int)threadIdx.x; j <= w.p; j += 256 * SHORT_WAVES) {
    WeightOf of;
    of.ask(a, b, kvh, 0, j);
    of.add(a, w.row, b, kvh, j, w.lo, w.p, lse);
  }
}

// ------------------------------------------------------------------------------------------ prompts
// grid (blocks of 64 QG new tokens x heads x sequences, the last blocks first), block 256: wave w takes QG groups of 16 tokens.  The
// cache already holds the step's keys and values.  A tile of codes is in registers on its way (32 bytes a thread and operand with
// heads of 128) while the one before becomes bfloat16 in LDS, once for all waves: the matrix cores then work on numbers as in a
// cache of 16 bits, and only memory sees that there are half the bytes.
template <int DT>
__device__ __forceinline__ int k_at(int row, int ch) { return row * (16 * DT) + ((ch ^ (row & (DT % 8 == 0 ? 15 : 7))) << 3); }
__device__ __forceinline__ int v_at(int d, int ch) { return d * E4M3_TILE + ((ch ^ (d & 7)) << 3); }

// HALVES 2: twice the waves, and tiles by turns: four waves take the first, third, .. tile, the other four the others, for the same tokens;
// their sums meet in LDS at the end.  For prompts with few workgroups, whose last blocks' tiles would else follow one another on a chip that is mostly idle.
template <int DT, int QG, bool MOD, int HALVES>
__global__ __launch_bounds__(256 * HALVES) __attribute__((amdgpu_waves_per_eu(DT > 8 ? 1 : 2))) void e4m3_prompt_kernel(E4m3Attn a, int n_blocks) {
  extern __shared__ __attribute__((aligned(16))) __bf16 tiles[];
  constexpr int KS = DT / 2, CH = (E4M3_TILE * DT + 255) / 256, BUF = 2 * E4M3_TILE * 16 * DT;
  constexpr bool AHEAD = DT <= 8 && PIECES == 1;
  const int per_block = a.nh * a.B, hd = a.pages.hd;
  const int blk = n_blocks - 1 - (int)blockIdx.x / per_block, h = (int)blockIdx.x % per_block % a.nh, b = (int)blockIdx.x % per_block / a.nh;
  const int half = HALVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
  const int tid = threadIdx.x % 256, lane = tid % 64, r = lane % 16, c = lane / 16, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int t0 = a.cu[b], n = a.cu[b + 1] - t0, qb = blk * 64 * QG;
  if (qb >= n) return;
  const int start = a.start[b], kvh = h / (a.nh / a.nkv);
  const int* row = a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride;
  const float r1 = MOD && a.mod.r1 ? a.mod.r1[h] : 0.f, r2 = MOD && a.mod.r1 ? a.mod.r2[h] : 0.f;
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
  const int tile0 = tile_beg + half;
  if (tile0 < tile_end) fetch_tile(tile0);      // (on its way while the queries are)
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
    m[g] = a.mod.sink && half == 0 ? a.mod.sink[h] * LOG2E : -INFINITY;
    l[g] = m[g] != -INFINITY && c == 0 ? 1.f : 0.f;      // (the sink counts once)
  }
  __bf16* mine = tiles + half * 2 * BUF;
  // what lies behind a head's end in LDS is read against zeros of the queries (keys) or not stored (values): it has to be finite
  if (hd < 16 * DT) {
    for (int i = tid; i < 2 * BUF / 8; i += 256) *reinterpret_cast<bf16x8*>(mine + 8 * i) = nothing();
    __syncthreads();
  }
  if (tile0 < tile_end) {
    stage(mine);
    if (tile0 + HALVES < tile_end) fetch_tile(tile0 + HALVES);
  }
  __syncthreads();
  int cur = 0;
  for (int at = tile_beg; at < tile_end; at += HALVES, cur ^= BUF) {      // (as often for either half)
    const int tile = at + half;
    if (tile + HALVES < tile_end) {
      stage(mine + (cur ^ BUF));
      if (tile + 2 * HALVES < tile_end) fetch_tile(tile + 2 * HALVES);
    }
    if (tile >= wave_beg && tile < wave_end) {
      const __bf16 *Ks = mine + cur, *Vs = Ks + E4M3_TILE * 16 * DT;
      const int pos0 = tile * E4M3_TILE;
      const bool masked = pos0 + E4M3_TILE - 1 > first || pos0 < lo_last;
      // Operands are asked for ahead of their products, as many as there are registers for: half of the keys before the first product, the
      // other half during it, the first values before the softmax.
      bf16x8 kf[4][KS], vf[2][DT];
      f32x4 s[QG][4];
      auto ask_k = [&](int jt) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[jt][ks] = *reinterpret_cast<const bf16x8*>(Ks + k_at<DT>(16 * jt + r, 4 * ks + c));
      };
      auto scores = [&](int jt) {
#pragma unroll
        for (int g = 0; g < QG; ++g) s[g][jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int g = 0; g < QG; ++g)
#pragma unroll
            for (int pc = PIECES - 1; pc >= 0; --pc) s[g][jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[jt][ks], qf[g][ks][pc], s[g][jt], 0, 0, 0);
      };
      auto ask_v = [&](int pr) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vf[pr][dt] = *reinterpret_cast<const bf16x8*>(Vs + v_at(16 * dt + r, 2 * c + pr));
      };
      ask_k(0);
      ask_k(1);
      if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
      ask_k(2);
      scores(0);
      ask_k(3);
      scores(1);
      if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
      scores(2);
      scores(3);
      ask_v(0);
      if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
      bf16x8 pf[QG][2][PIECES];
#pragma unroll
      for (int g = 0; g < QG; ++g) {
        final_scores<MOD>(s[g], a, false, r1, r2, pos0, p[g], lo[g], masked);
        softmax_tile<DT>(s[g], o[g], m[g], l[g], MOD ? 1.f : a.ch.scale2, pf[g]);
      }
      ask_v(1);
      if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int pr = 0; pr < 2; ++pr)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int g = 0; g < QG; ++g)
#pragma unroll
            for (int pc = PIECES - 1; pc >= 0; --pc) o[g][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[pr][dt], pf[g][pr][pc], o[g][dt], 0, 0, 0);
    }
    __syncthreads();
  }
#pragma unroll
  for (int g = 0; g < QG; ++g) l[g] = group_sum(l[g]);
  if constexpr (HALVES == 2) {
    static_assert(QG * DT * 4 * 64 * 16 + QG * 4 * 64 * 8 <= 2 * HALVES * BUF * 2, "the second half's sums fit into the tiles' place");
    f32x4* sums = reinterpret_cast<f32x4*>(tiles);
    float2* ml = reinterpret_cast<float2*>(sums + 4 * QG * DT * 64);
    if (half == 1) {
#pragma unroll
      for (int g = 0; g < QG; ++g) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) sums[((wave * QG + g) * DT + dt) * 64 + lane] = o[g][dt];
        ml[(wave * QG + g) * 64 + lane] = make_float2(m[g], l[g]);
      }
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      const float2 other = ml[(wave * QG + g) * 64 + lane];
      const float to = fmaxf(m[g], other.x), use = to == -INFINITY ? 0.f : to;
      const float mine_by = __builtin_amdgcn_exp2f(m[g] - use), other_by = __builtin_amdgcn_exp2f(other.x - use);
      l[g] = fmaf(other.y, other_by, l[g] * mine_by);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f32x4 x = sums[((wave * QG + g) * DT + dt) * 64 + lane];
#pragma unroll
        for (int v = 0; v < 4; ++v) o[g][dt][v] = fmaf(x[v], other_by, o[g][dt][v] * mine_by);
      }
      m[g] = to;
    }
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

// The weights that a prompt gives its positions, from the scores once more and the rows' sums: grid (tiles / 4, nh, B * cuts), block 256.  A
// wave keeps a tile's keys in registers, as numbers; the workgroup goes through the tokens of its cut that may see one of its four
// tiles, 32 at a time, which come through LDS once for the four waves (each wave for itself asked the caches for 4 KiB of queries
// for every 16 products, and waited: 166 us for 4,096 tokens of 28 heads).  A wave sums its own columns, in order, and at the end
// over lanes; a second kernel adds the columns' sums over cuts and a kv head's heads.
#define WEIGHT_TOKENS 32
template <int DT, bool MOD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DT * PIECES > 8 ? (DT * PIECES > 16 ? 1 : 2) : 3))) void e4m3_prompt_weights_kernel(E4m3Attn a, int cuts, int cut) {
  constexpr int KS = 2 * (DT / 4), PITCH = 16 * DT + 16 / (int)sizeof(act_t), PER = 16 / (int)sizeof(act_t);      // (numbers to 16 bytes)
  constexpr int CH = (WEIGHT_TOKENS * 16 * DT / PER + 255) / 256;
  extern __shared__ __attribute__((aligned(16))) act_t qs[];      // [2][32][PITCH]
  __shared__ float lses[2][WEIGHT_TOKENS];
  const int h = blockIdx.y, kvh = h / (a.nh / a.nkv), b = blockIdx.z / cuts, hd = a.pages.hd;
  const int tid = threadIdx.x, lane = tid % 64, r = lane % 16, c = lane / 16, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int t0 = a.cu[b], n = a.cu[b + 1] - t0, start = a.start[b];
  const int q_beg = (int)(blockIdx.z % cuts) * cut, q_end = min(q_beg + cut, n);      // (cut: a multiple of 32)
  const int tile0 = reach_lo(start, a.window, a.mod.chunk) / E4M3_TILE + 4 * (int)blockIdx.x, tile = tile0 + wave;
  if (n <= 0 || tile0 * E4M3_TILE >= start + n) return;
  const int pos0 = tile * E4M3_TILE;
  const bool has = pos0 < start + n;
  const int* row = a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride;
  const float r1 = MOD && a.mod.r1 ? a.mod.r1[h] : 0.f, r2 = MOD && a.mod.r1 ? a.mod.r2[h] : 0.f;
  bf16x8 kf[4][KS];
  {
    int in_page;
    int64_t head = e4m3_head_of(a.pages, row, has ? tile : tile0, kvh, in_page);
    if (head < 0) head = 0;
    const uint8_t* at = a.pages.k + e4m3_tile_at(a.pages, head, in_page);
    const f32x4 scale = *reinterpret_cast<const f32x4*>(a.pages.k_scale + e4m3_scale_at(a.pages, head, in_page));
#pragma unroll
    for (int i = 0; i < KS / 2; ++i)
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(at + min(4 * i + c, hd / 16 - 1) * 1024 + (16 * jt + r) * 16);
        kf[jt][2 * i] = numbers(w[0], w[1], scale[jt]);
        kf[jt][2 * i + 1] = numbers(w[2], w[3], scale[jt]);
      }
  }
  // the tokens that may see a position of the four tiles: from the first tile's first to the last whose reach has the last one's last
  const int from = max(tile0 * E4M3_TILE - start, q_beg) / WEIGHT_TOKENS * WEIGHT_TOKENS, end_pos = (tile0 + 4) * E4M3_TILE - 1;
  int to = q_end;
  if (a.window > 0) to = (int)min((int64_t)to, (int64_t)end_pos + a.window - start);
  if (a.mod.chunk > 0) to = (int)min((int64_t)to, (int64_t)(end_pos / a.mod.chunk + 1) * a.mod.chunk - start);
  const int chunks = hd / PER;      // of 16 bytes in a row
  u32x4 pq[CH];
  float plse = 0.f;
  auto ask = [&](int q0) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int i = min(tid + 256 * j, WEIGHT_TOKENS * chunks - 1);
      pq[j] = *reinterpret_cast<const u32x4*>(a.q + ((int64_t)(t0 + min(q0 + i / chunks, n - 1)) * a.nh + h) * hd + i % chunks * PER);
    }
    if (tid < WEIGHT_TOKENS) plse = a.lse[(int64_t)(t0 + min(q0 + tid, n - 1)) * a.nh + h];
  };
  f32x4 acc[4];
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) acc[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (from < to) ask(from);
  // (a condition at every read would keep the next from being on its way: rows are filled up with zeros once)
  for (int i = tid; i < 2 * WEIGHT_TOKENS * (DT - hd / 16); i += 256) {
    act_t* at = qs + i / (DT - hd / 16) * PITCH + hd + i % (DT - hd / 16) * 16;
#pragma unroll
    for (int e = 0; e < 16; e += PER) *reinterpret_cast<u32x4*>(at + e) = u32x4{0u, 0u, 0u, 0u};
  }
  int buf = 0;
  for (int q0 = from; q0 < to; q0 += WEIGHT_TOKENS, buf ^= 1) {
    // (one barrier a round: the buffer that is written was last read before the one before)
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int i = min(tid + 256 * j, WEIGHT_TOKENS * chunks - 1);
      *reinterpret_cast<u32x4*>(qs + (buf * WEIGHT_TOKENS + i / chunks) * PITCH + i % chunks * PER) = pq[j];
    }
    if (tid < WEIGHT_TOKENS) lses[buf][tid] = plse;
    __syncthreads();
    if (q0 + WEIGHT_TOKENS < to) ask(q0 + WEIGHT_TOKENS);
    if (!has) continue;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int q1 = q0 + 16 * half, qi = q1 + r;
      // some of the 16 tokens sees some of the tile
      if (q1 >= n || start + min(q1 + 15, n - 1) < pos0 || reach_lo(start + q1, a.window, a.mod.chunk) >= pos0 + E4M3_TILE) continue;
      const int p = qi < n ? start + qi : -1, lo = reach_lo(p, a.window, a.mod.chunk);
      const act_t* qrow = qs + (buf * WEIGHT_TOKENS + 16 * half + r) * PITCH;
      f32x4 s[4];
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) s[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        bf16x8 qf[PIECES];
        load_query(qf, qrow, 64 * (ks / 2) + 16 * c + 8 * (ks % 2));
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
#pragma unroll
          for (int pc = PIECES - 1; pc >= 0; --pc) s[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[jt][ks], qf[pc], s[jt], 0, 0, 0);
      }
      const float sum = lses[buf][16 * half + r];
      // every token of the 16 sees the whole tile: nothing to compare
      const bool masked = q1 + 15 >= n || start + q1 < pos0 + E4M3_TILE - 1 || reach_lo(start + q1 + 15, a.window, a.mod.chunk) > pos0;
      final_scores<MOD>(s, a, true, r1, r2, pos0, p, lo, false);
#pragma unroll
      for (int jt = 0; jt < 4; ++jt)
#pragma unroll
        for (int v = 0; v < 4; ++v) s[jt][v] = __builtin_amdgcn_exp2f(fmaf(s[jt][v], MOD ? 1.f : a.ch.scale2, -sum));
      // (by its place, not by a score of -inf: the sum of a row that is not a number is none either, and would reach positions it does not see)
      if (masked) {
        asm volatile("");      // (a branch, as in final_scores)
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int key = pos0 + 16 * jt + 4 * c + v;
            s[jt][v] = key <= p && key >= lo ? s[jt][v] : 0.f;
          }
      }
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) acc[jt] += s[jt];
    }
  }
  if (!has) return;
  float* out = a.scores + ((int64_t)blockIdx.z * a.nh + h) * a.ld_scores + pos0;
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    f32x4 x;
#pragma unroll
    for (int v = 0; v < 4; ++v) x[v] = lanes_fold<16>(acc[jt][v], LanesSum());
    if (r == 0) *reinterpret_cast<f32x4*>(out + 16 * jt + 4 * c) = x;
  }
}
// grid (blocks of 1,024 positions, nkv, B): a thread adds what four neighbouring positions have received.
__global__ __launch_bounds__(256) void e4m3_add_weights_kernel(E4m3Attn a, int cuts) {
  const int kvh = blockIdx.y, b = blockIdx.z, g = a.nh / a.nkv, j = (int)blockIdx.x * 1024 + 4 * (int)threadIdx.x;
  const int n = a.cu[b + 1] - a.cu[b], start = a.start[b], lo = reach_lo(start, a.window, a.mod.chunk);
  if (n <= 0 || j >= start + n || j + 3 < lo) return;
  int in_page;
  const int64_t head = e4m3_head_of(a.pages, a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride, j / E4M3_TILE, kvh, in_page);
  if (head < 0) return;
  f32x4* to = reinterpret_cast<f32x4*>(a.pages.weight + head * a.pages.page_size + in_page * E4M3_TILE + j % E4M3_TILE);
  f32x4 w = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < cuts; ++i) {
    const float* from = a.scores + (((int64_t)b * cuts + i) * a.nh + kvh * g) * a.ld_scores + j;
#pragma unroll 4
    for (int h = 0; h < g; ++h) w += *reinterpret_cast<const f32x4*>(from + h * a.ld_scores);
  }
  f32x4 was = *to;
#pragma unroll
  for (int e = 0; e < 4; ++e) was[e] = j + e >= lo && j + e < start + n ? was[e] + w[e] : was[e];
  *to = was;
}

// ------------------------------------------------------------------------------------------ launch
// Waves of a step beyond which a wave takes more runs instead: three rounds of two waves to a SIMD.  us of the runs of 8 sequences of 8,192 tokens (16
// heads) and of 64 of 300 to 4,100 (28 heads on 4): with 2,048 waves 47 and 50, 3,072 52 and 46, 4,096 53 and 50, 6,144 47 and 41, 8,192 52 and
// 41.  (Three waves to a SIMD, with some of their registers in scratch memory: 58 and 43 at best.)
#define DECODE_WAVES 6144
// Cuts of a prompt's tokens for the columns' sums: as many as make some thousands of workgroups, of 256 tokens at least.
static int e4m3_cuts(int B, int nh, int max_new, int max_end) {
  const int64_t groups = (int64_t)((max_end + 4 * E4M3_TILE - 1) / (4 * E4M3_TILE)) * nh * B;
  return (int)max((int64_t)1, min((int64_t)(max_new + 255) / 256, 4096 / groups));
}
// Whether heads of 16 DT numbers can go through one launch (wider ones: two waves to a SIMD have too few registers), and with how many bytes
// of shared memory a step up to position max_end does; 0 where it takes two launches and scratch.
#define SHORT_HEADS(DT) ((DT) <= 12 && (DT) * PIECES <= 24)
static size_t e4m3_short_bytes(int max_end, int g, int hd) {
  const size_t shmem = (size_t)((max_end + E4M3_TILE - 1) / E4M3_TILE) * g * (hd + 2) * sizeof(float);
  return max_end <= SHORT_END && g <= 16 && shmem + 16 * sizeof(float) <= 64 * 1024 ? shmem : 0;      // (and the heads' sums of 16)
}
template <int DT, bool MOD>
static int launch_decode(const E4m3Attn& a, int max_end, hipStream_t st) {
  const int g = a.nh / a.nkv, columns = a.nkv * ((g + 15) / 16);
  if constexpr (SHORT_HEADS(DT)) {
    if (const size_t shmem = e4m3_short_bytes(max_end, g, a.pages.hd)) {
      hipLaunchKernelGGL((e4m3_short_kernel<DT, MOD>), dim3(columns, a.B), dim3(64 * SHORT_WAVES), shmem, st, a);
      return 0;
    }
  }
  const int waves = min(a.max_runs, max(1, DECODE_WAVES / (columns * a.B)));
  hipLaunchKernelGGL((e4m3_decode_kernel<DT, MOD>), dim3(waves, columns, a.B), dim3(64), 0, st, a);
  const int blocks = a.scores ? (max_end + 1023) / 1024 : 0;
  if ((int64_t)a.nh * a.B + (int64_t)blocks * a.nkv * a.B > 0xFFFFFF) return TQ_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(e4m3_join_kernel<DT <= 8 ? 2 : 4>, dim3(a.nh * a.B + blocks * a.nkv * a.B), dim3(256), 0, st, a, blocks);
  return 0;
}
template <int DT, int QG, bool MOD, int HALVES>
static int launch_prompt(const E4m3Attn& a, int max_new, hipStream_t st) {
  const size_t shmem = HALVES * 2 * (size_t)2 * E4M3_TILE * 16 * DT * sizeof(__bf16);
  if (shmem > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)e4m3_prompt_kernel<DT, QG, MOD, HALVES>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem);
    if (e != hipSuccess) return (int)e;
  }
  const int n_blocks = (max_new + 64 * QG - 1) / (64 * QG);
  if ((int64_t)n_blocks * a.nh * a.B > 0x7FFFFF) return TQ_ERR_UNSUPPORTED;      // (a launch's threads are counted in 32 bits)
  hipLaunchKernelGGL((e4m3_prompt_kernel<DT, QG, MOD, HALVES>), dim3(n_blocks * a.nh * a.B), dim3(256 * HALVES), shmem, st, a, n_blocks);
  return 0;
}
template <int DT, bool MOD>
static int launch_as(const E4m3Attn& a, int decode, int max_new, int max_end, hipStream_t st) {
  if (decode) return launch_decode<DT, MOD>(a, max_end, st);
  // Two groups of 16 tokens to a wave halve the reads from LDS, and the chip does 733 TFLOP/s instead of 505 (8,192 tokens of 16 heads of
  // 128), but it takes enough workgroups that the last blocks, which see most, do not stand alone: 2,048 tokens, 256 of
  // them, take 47 us so and 42 with one group; 4,096 tokens, 512 of them, 101 and 136.  (These and the next were timed in turn before the
  // first tile was asked for ahead of the queries, which takes some 2 us off each: the 42 are 40 now.)
  constexpr int TWO = PIECES == 1 && DT <= 8 ? 2 : 1, HALVES = DT <= 8 ? 2 : 1;
  const int64_t of_two = (int64_t)((max_new + 127) / 128) * a.nh * a.B, of_one = (int64_t)((max_new + 63) / 64) * a.nh * a.B;
  const bool two = TWO == 2 && of_two > 256;
  // Tiles by turns in two halves of a workgroup: with few workgroups (4,096 tokens of 16 heads 134 -> 101 us, 2,048 of them 50 -> 42,
  // 1,024 25 -> 19); with 1,536 of them 193 -> 232.
  // Blocks behind a short window have no tiles to share (tokens of a 32-bit prompt behind 256 positions: 18 -> 20 us).
  const int seen = a.window > 0 ? min(max_end, a.window + 64) : max_end;
  const bool halves = HALVES == 2 && (two ? of_two : of_one) <= 512 && seen >= 8 * E4M3_TILE;
  const int rc = two ? (halves ? launch_prompt<DT, TWO, MOD, HALVES>(a, max_new, st) : launch_prompt<DT, TWO, MOD, 1>(a, max_new, st))
                     : (halves ? launch_prompt<DT, 1, MOD, HALVES>(a, max_new, st) : launch_prompt<DT, 1, MOD, 1>(a, max_new, st));
  if (rc || !a.lse) return rc;
  const int tiles = (max_end + E4M3_TILE - 1) / E4M3_TILE, cuts = e4m3_cuts(a.B, a.nh, max_new, max_end), cut = ((max_new + cuts - 1) / cuts + WEIGHT_TOKENS - 1) / WEIGHT_TOKENS * WEIGHT_TOKENS;
  if ((int64_t)a.B * cuts > 65535) return TQ_ERR_UNSUPPORTED;
  const size_t shmem = 2 * (size_t)WEIGHT_TOKENS * (16 * DT * sizeof(act_t) + 16);      // at most 65.5 KiB
  if (shmem > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)e4m3_prompt_weights_kernel<DT, MOD>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL((e4m3_prompt_weights_kernel<DT, MOD>), dim3((tiles + 3) / 4, a.nh, a.B * cuts), dim3(256), shmem, st, a, cuts, cut);
  hipLaunchKernelGGL(e4m3_add_weights_kernel, dim3((max_end + 1023) / 1024, a.nkv, a.B), dim3(256), 0, st, a, cuts);
  return 0;
}
template <int DT>
static int launch(const E4m3Attn& a, int decode, int max_new, int max_end, hipStream_t st) {
  return a.mod.cap > 0.f || a.mod.r1 || !(a.scale > 0.f) ? launch_as<DT, true>(a, decode, max_new, max_end, st) : launch_as<DT, false>(a, decode, max_new, max_end, st);
}

// Floats of scratch: for decoding the runs' sums, with weights the scores too; for prompts with weights the columns' and the rows' sums.
// max_new: the longest run.
TQ_API int64_t tq_e4m3_attention_scratch(int T, int B, int nh, int nkv, int hd, int max_new, int max_end, int decode, int weights) {
  const int64_t ld = (max_end + E4M3_TILE - 1) / E4M3_TILE * E4M3_TILE;
  if (!decode) return weights ? (int64_t)B * e4m3_cuts(B, nh, max_new, max_end) * nh * ld + (int64_t)T * nh : 0;
  // (the kernels are made for heads of 4, 8, 12 and 16 times 16 numbers)
  if (SHORT_HEADS((hd + 63) / 64 * 4) && e4m3_short_bytes(max_end, nh / nkv, hd)) return weights ? (int64_t)B * nh * ld : 0;
  return (int64_t)B * nh * e4m3_most_runs(max_end, nh / nkv) * (hd + 2) + (weights ? (int64_t)B * nh * ld : 0);
}

// q, out [T][nh][hd]; tokens as runs (cu, slots, start) whose keys and values the cache holds already.  decode != 0: one token per
// sequence, or none.  weight (null: none): every position's is raised by what it receives.  max_end: the largest position + 1.
TQ_API int tq_e4m3_attention(const void* q, void* out, const int* cu, const int* slots, const int* start, int T, int B, int nh, int nkv,
                             int hd, int window, float scale, float softcap, const float* r1, const float* r2, int chunk,
                             const float* sink, const void* k, const void* v, const float* k_scale, const float* v_scale, float* weight,
                             const int* table, int bt_stride, int page_size, int heads, int head0, float* scratch, int decode, int max_new,
                             int max_end, hipStream_t st) {
  if (B <= 0 || T <= 0) return 0;
  if ((r1 == nullptr) != (r2 == nullptr) || chunk < 0 || softcap < 0.f || window < 0 || nh <= 0 || max_new <= 0 || max_end <= 0) return TQ_ERR_BAD_ARG;
  if (!e4m3_pages_fit(page_size, heads, head0, nkv, hd) || nh % nkv != 0 || nh > 65535 || nh / nkv > 1024 || B > 65535) return TQ_ERR_UNSUPPORTED;
  if (!scratch && tq_e4m3_attention_scratch(T, B, nh, nkv, hd, max_new, max_end, decode, weight != nullptr)) return TQ_ERR_BAD_ARG;
  E4m3Attn a{(const act_t*)q, (act_t*)out, cu, slots, start, B, nh, nkv, window, scale, ScoreMod{softcap, r1, r2, chunk, sink, nullptr, 0},
             change_of(scale, softcap), nullptr, e4m3_most_runs(max_end, nh / nkv), nullptr, 0, nullptr,
             E4m3Pages{(uint8_t*)k, (uint8_t*)v, (float*)k_scale, (float*)v_scale, weight, table, bt_stride, page_size, heads, head0, hd}};
  if (weight) {      // (first: its rows are read and written 16 bytes at a time)
    a.ld_scores = (max_end + E4M3_TILE - 1) / E4M3_TILE * E4M3_TILE;
    a.scores = scratch;
    scratch += (decode ? (int64_t)B : (int64_t)B * e4m3_cuts(B, nh, max_new, max_end)) * nh * a.ld_scores;
    if (!decode) a.lse = scratch;
  }
  if (decode) a.partial = scratch;
  const int dt = hd / 16;
  const int rc = dt <= 4 ? launch<4>(a, decode, max_new, max_end, st) : dt <= 8 ? launch<8>(a, decode, max_new, max_end, st)
               : dt <= 12 ? launch<12>(a, decode, max_new, max_end, st) : launch<16>(a, decode, max_new, max_end, st);
  if (rc) return rc;
  TQ_LAUNCH_CHECK();
  return 0;
}
