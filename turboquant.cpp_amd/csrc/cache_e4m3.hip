// The 8-bit cache (cache_e4m3.h): the write that fills its pages, and eviction, which copies chosen positions into other pages.
#include "cache_e4m3.h"

// ------------------------------------------------------------------------------------------ rotation, rounding, write
struct E4m3Write {
  const float* x;               // [T][ld]: queries, keys, values of a token side by side
  int64_t ld;
  const void* bias;             // null, or one row added to every token's, of bias_type
  int bias_type;
  const int* positions;         // [T] what the rotation turns by
  const float* inv_freq;        // [rot / 2]
  int pairing, rot;
  float amp;
  const int* cu;                // [B + 1]
  const int* slots;             // [B]
  const int* start;             // [B] place of each sequence's first new token in the cache
  act_t* q;                     // [T][nh * hd]
  int T, B, nh, nkv, hd;
  int tiles;                    // most tiles that a sequence's new tokens touch
  int q_tokens, q_heads;        // tokens and heads of a workgroup of queries
  E4m3Pages pages;
  int write;
};

__device__ __forceinline__ float bias_at(const E4m3Write& a, int i) {
  return a.bias_type == TQ_BF16 ? to_f32(((const bf16_t*)a.bias)[i]) : ((const float*)a.bias)[i];
}
// Sine and cosine of the exact product p * f: the rounded product's, turned on by the small angle that the rounding left out (positions
// of a long cache: at 100,000 the rounded product of a fast pair is off by up to 0.004).
__device__ __forceinline__ void turn_of(int p, float f, float amp, float& cs, float& sn) {
  const float pf = (float)p, hi = pf * f, lo = fmaf(pf, f, -hi);
  float s, c;
  sincosf(hi, &s, &c);
  const float l2 = lo * lo, ls = lo * fmaf(l2, -1.f / 6.f, 1.f), lc = l2 * fmaf(l2, 1.f / 24.f, -0.5f);      // sin lo, cos lo - 1
  sn = amp * (s + fmaf(c, ls, s * lc));
  cs = amp * (c + fmaf(-s, ls, c * lc));
}

// A workgroup takes either one tile of 64 positions of one sequence and kv head (keys and values: a row that is not finite in one
// is marked in both), or the queries of q_tokens tokens and q_heads heads.  Keys and values pass through LDS in 32 bits, where the
// keys are rotated, since a block's scale has to be known before its first code.
// Bound by the bytes (a prompt) or by the launch (single tokens).
__global__ __launch_bounds__(256) void e4m3_write_kernel(E4m3Write a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int hd = a.hd, n = a.rot / 2, tid = threadIdx.x;
  const int kv_groups = a.write ? a.tiles * a.nkv * a.B : 0;
  if ((int)blockIdx.x >= kv_groups) {
    // queries: the angles of the workgroup's tokens once, then four neighbouring numbers of a head at a time
    const int w = (int)blockIdx.x - kv_groups, per = (a.nh + a.q_heads - 1) / a.q_heads;
    const int t0 = w / per * a.q_tokens, h0 = w % per * a.q_heads;
    const int nt = min(a.q_tokens, a.T - t0), heads = min(a.q_heads, a.nh - h0);
    float2* turn = reinterpret_cast<float2*>(lds);
    for (int i = tid; i < nt * n; i += 256) {
      float c, s;
      turn_of(a.positions[t0 + i / n], a.inv_freq[i % n], a.amp, c, s);
      turn[i] = make_float2(c, s);
    }
    __syncthreads();
    const int fours = hd / 4, items = nt * heads * fours;
    for (int i = tid; i < items; i += 256) {
      const int d = i % fours * 4, h = h0 + i / fours % heads, t = i / (fours * heads);
      const float* row = a.x + (int64_t)(t0 + t) * a.ld + (int64_t)h * hd;
      float4 v = *reinterpret_cast<const float4*>(row + d);
      float x[4] = {v.x, v.y, v.z, v.w}, o[4];
      if (a.bias)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += bias_at(a, h * hd + d + j);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = d + j;
        o[j] = x[j];
        if (e < 2 * n) {
          const int pair = a.pairing == 0 ? (e < n ? e : e - n) : e / 2;
          const bool low = a.pairing == 0 ? e < n : e % 2 == 0;
          const int other = a.pairing == 0 ? (low ? e + n : e - n) : e ^ 1;
          float y = a.pairing == 0 ? row[other] + (a.bias ? bias_at(a, h * hd + other) : 0.f) : x[j ^ 1];
          const float2 cs = turn[t * n + pair];
          o[j] = low ? x[j] * cs.x - y * cs.y : y * cs.y + x[j] * cs.x;
        }
      }
      act_t* out = a.q + ((int64_t)(t0 + t) * a.nh + h) * hd + d;
#if defined(TQ_ACT_BF16)
      *reinterpret_cast<uint2*>(out) = make_uint2(f32_to_bf16_pair(o[0], o[1]), f32_to_bf16_pair(o[2], o[3]));
#else
      *reinterpret_cast<float4*>(out) = make_float4(o[0], o[1], o[2], o[3]);
#endif
    }
    return;
  }
  const int kvh = (int)blockIdx.x % a.nkv, b = (int)blockIdx.x / a.nkv % a.B, nth = (int)blockIdx.x / a.nkv / a.B;
  const int t0 = a.cu[b], count = a.cu[b + 1] - t0, start = a.start[b];
  const int tile = start / E4M3_TILE + nth, pos0 = tile * E4M3_TILE;
  if (count <= 0 || pos0 >= start + count) return;
  const int r0 = max(start - pos0, 0), r1 = min(start + count - pos0, E4M3_TILE);      // the tile's rows that are new
  const int old0 = r0 / E4M3_BLOCK * E4M3_BLOCK;      // rows old0 .. r0 - 1 share the first new row's block
  int in_page;
  const int64_t head = e4m3_head_of(a.pages, a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride, tile, kvh, in_page);
  if (head < 0) return;
  const int stride = hd + 4;
  float* K = lds;                                  // [64][hd + 4]
  float* V = K + E4M3_TILE * stride;
  __shared__ uint32_t top[2][4];
  __shared__ int bad[E4M3_TILE];
  __shared__ float inverse[2][4], ratio[2];
  if (tid < 8) top[tid / 4][tid % 4] = 0u;
  if (tid < E4M3_TILE) bad[tid] = 0;
  const int rows = r1 - r0, fours = hd / 4;
  const int64_t first = (int64_t)(t0 + pos0 + r0 - start);      // packed row of the tile's first new row
  for (int i = tid; i < 2 * rows * fours; i += 256) {
    const int d = i % fours * 4, m = i / fours % 2, r = i / (2 * fours);
    const int col = (a.nh + m * a.nkv + kvh) * hd + d;
    float4 v = *reinterpret_cast<const float4*>(a.x + (first + r) * a.ld + col);
    if (a.bias) v = make_float4(v.x + bias_at(a, col), v.y + bias_at(a, col + 1), v.z + bias_at(a, col + 2), v.w + bias_at(a, col + 3));
    *reinterpret_cast<float4*>((m ? V : K) + (r0 + r) * stride + d) = v;
  }
  __syncthreads();
  for (int i = tid; i < rows * n; i += 256) {
    const int pair = i % n, r = i / n;
    const int lo = a.pairing == 0 ? pair : 2 * pair, hi = a.pairing == 0 ? pair + n : 2 * pair + 1;
    float cs, sn;
    turn_of(a.positions[first + r], a.inv_freq[pair], a.amp, cs, sn);
    float* row = K + (r0 + r) * stride;
    const float x = row[lo], y = row[hi];
    row[lo] = x * cs - y * sn;
    row[hi] = x * sn + y * cs;
  }
  __syncthreads();
  // rows that are not finite, then the blocks' largest magnitudes without them
  for (int i = tid; i < 2 * rows * fours; i += 256) {
    const int d = i % fours * 4, m = i / fours % 2, r = r0 + i / (2 * fours);
    const float4 v = *reinterpret_cast<const float4*>((m ? V : K) + r * stride + d);
    if (!(fabsf(v.x) < E4M3_TOO_LARGE && fabsf(v.y) < E4M3_TOO_LARGE && fabsf(v.z) < E4M3_TOO_LARGE && fabsf(v.w) < E4M3_TOO_LARGE))
      bad[r] = 1;
  }
  __syncthreads();
  for (int i = tid; i < 2 * rows * fours; i += 256) {
    const int d = i % fours * 4, m = i / fours % 2, r = r0 + i / (2 * fours);
    if (bad[r]) continue;
    const float4 v = *reinterpret_cast<const float4*>((m ? V : K) + r * stride + d);
    atomicMax(&top[m][r / E4M3_BLOCK], __float_as_uint(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)))));
  }
  __syncthreads();
  if (tid < 8) {
    const int m = tid / 4, j = tid % 4;
    if (j * E4M3_BLOCK < r1 && (j + 1) * E4M3_BLOCK > r0) {
      float* at = (m ? a.pages.v_scale : a.pages.k_scale) + e4m3_scale_at(a.pages, head, in_page) + j;
      float scale = e4m3_scale(__uint_as_float(top[m][j]));
      if (j == r0 / E4M3_BLOCK) {
        const float was = old0 < r0 ? *at : 0.f;
        scale = fmaxf(scale, was);
        ratio[m] = was * e4m3_inverse(scale);      // what the rows before the new ones are multiplied by (1: they stay)
      }
      *at = scale;
      inverse[m][j] = e4m3_inverse(scale);
    }
  }
  __syncthreads();
  uint8_t* kt = a.pages.k + e4m3_tile_at(a.pages, head, in_page);
  uint8_t* vt = a.pages.v + e4m3_tile_at(a.pages, head, in_page);
  const int from_k = ratio[0] != 1.f ? old0 : r0, from_v = ratio[1] != 1.f ? old0 : r0;
  for (int i = tid; i < (r1 - from_k) * (hd / 16); i += 256) {
    const int r = from_k + i % (r1 - from_k), ch = i / (r1 - from_k);
    uint4* at = reinterpret_cast<uint4*>(kt + ch * 16 * E4M3_TILE + r * 16);
    uint4 w;
    if (r < r0) {
      w = *at;
      const float f = ratio[0];
      w = make_uint4(e4m3_rescale(w.x, f, f, f, f), e4m3_rescale(w.y, f, f, f, f), e4m3_rescale(w.z, f, f, f, f), e4m3_rescale(w.w, f, f, f, f));
    } else if (bad[r]) {
      w = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
    } else {
      const float f = inverse[0][r / E4M3_BLOCK];
      const float4* row = reinterpret_cast<const float4*>(K + r * stride + ch * 16);
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = e4m3_codes(row[j].x * f, row[j].y * f, row[j].z * f, row[j].w * f);
      w = make_uint4(c[0], c[1], c[2], c[3]);
    }
    *at = w;
  }
  for (int i = tid; i < 16 * hd; i += 256) {
    // four positions of one dimension: 16 j + 4 c ..
    const int d = i % hd, j = i / hd / 4, c = i / hd % 4, p = 16 * j + 4 * c;
    if (p >= r1 || p + 4 <= from_v) continue;
    uint32_t* at = reinterpret_cast<uint32_t*>(vt + d * E4M3_TILE + 16 * c + 4 * j);
    const bool whole = p >= r0 && p + 4 <= r1;
    const uint32_t was = whole ? 0u : *at;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = p + e >= r0 && p + e < r1 && !bad[p + e] ? V[(p + e) * stride + d] * inverse[1][j] : 0.f;
    uint32_t w = e4m3_codes(x[0], x[1], x[2], x[3]);
    if (!whole) {
      const uint32_t turned = p < r0 && from_v < r0 ? e4m3_rescale(was, ratio[1], ratio[1], ratio[1], ratio[1]) : was;
      uint32_t mine = 0u, before = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mine |= p + e >= r0 && p + e < r1 ? 0xffu << 8 * e : 0u;
        before |= p + e < r0 ? 0xffu << 8 * e : 0u;
      }
      w = (w & mine) | (turned & before) | (was & ~(mine | before));
    }
    *at = w;
  }
  if (a.pages.weight) {
    float* at = a.pages.weight + head * a.pages.page_size + in_page * E4M3_TILE;
    if (tid >= r0 && tid < r1) at[tid] = 0.f;
  }
}

// x float [T][ld] with (nh + 2 nkv) * hd numbers a row; positions [T] turn the rotation, places in the cache come from the runs:
// sequence b's tokens cu[b] .. cu[b + 1] - 1 go to places start[b], start[b] + 1, .. of slot slots[b].  k == null: nothing is
// written, the queries alone are rotated.  weight (null: none) is zeroed at the new places.  max_new: the longest run.
TQ_API int tq_e4m3_write(const float* x, int64_t ld, const void* bias, int bias_type, const int* positions, const float* inv_freq,
                         int pairing, int rot, float amp, const int* cu, const int* slots, const int* start, void* q, int T, int B,
                         int max_new, int nh, int nkv, int hd, void* k, void* v, float* k_scale, float* v_scale, float* weight,
                         const int* table, int bt_stride, int page_size, int heads, int head0, hipStream_t st) {
  if (T <= 0 || B <= 0) return 0;
  if (rot < 0 || rot > hd || (rot & 1) || (pairing != 0 && pairing != 1) || (bias && bias_type != TQ_F32 && bias_type != TQ_BF16)) return TQ_ERR_BAD_ARG;
  if (ld < (int64_t)(nh + 2 * nkv) * hd || ld % 4 != 0 || (uintptr_t)x % 16 != 0 || nh <= 0 || max_new <= 0) return TQ_ERR_BAD_ARG;
  if (!e4m3_pages_fit(page_size, heads, head0, k ? nkv : 1, hd)) return TQ_ERR_UNSUPPORTED;
  E4m3Write a{x, ld, bias, bias_type, positions, inv_freq, pairing, rot, amp, cu, slots, start, (act_t*)q, T, B, nh, nkv, hd,
              (max_new + E4M3_TILE - 2) / E4M3_TILE + 1, 1, nh,
              E4m3Pages{(uint8_t*)k, (uint8_t*)v, k_scale, v_scale, weight, table, bt_stride, page_size, heads, head0, hd}, k != nullptr};
  // queries: as many tokens and heads to a workgroup as leave the chip a thousand of them
  a.q_heads = nh;
  while (a.q_heads > 1 && (int64_t)T * ((nh + a.q_heads - 1) / a.q_heads) < 1024) a.q_heads = (a.q_heads + 1) / 2;
  while (a.q_tokens < 8 && (int64_t)T / a.q_tokens >= 4096) a.q_tokens *= 2;
  const int64_t kv_groups = a.write ? (int64_t)a.tiles * nkv * B : 0;
  const int64_t groups = kv_groups + (int64_t)((T + a.q_tokens - 1) / a.q_tokens) * ((nh + a.q_heads - 1) / a.q_heads);
  if (groups > 0xFFFFFF) return TQ_ERR_UNSUPPORTED;      // (a launch's threads are counted in 32 bits)
  size_t shmem = (size_t)a.q_tokens * (rot / 2) * sizeof(float2);
  if (a.write) shmem = max(shmem, 2 * (size_t)E4M3_TILE * (hd + 4) * sizeof(float));
  if (shmem > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)e4m3_write_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(e4m3_write_kernel, dim3((unsigned)groups), dim3(256), shmem, st, a);
  TQ_LAUNCH_CHECK();
  return 0;
}

// ------------------------------------------------------------------------------------------ eviction: the choice
// One workgroup per sequence, layer and kv head.  The sequence's first `first` and last `recent` positions stay; of the others the
// `m` with the largest weights, a tie going to the lowest position.  The m-th largest weight is found byte by byte from the top: a
// histogram of the next byte of the weights that share the bytes found so far, and the bin in which the m-th lies.  Weights are
// compared as integers that are ordered as the floats are (NaN above all).  Then the positions are listed in order.
// Weights are read once: up to CHOICE_HELD of them stay in LDS, the others are read again from L2.
#define CHOICE_HELD 16384
struct E4m3Choice {
  const int* slots;
  const int* lengths;
  int* kept;                    // [B][heads][keep]
  int keep, first, recent, slots_of_table, max_length;
  E4m3Pages pages;
};
__device__ __forceinline__ uint32_t ordered(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);      // (-0 equals 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__global__ __launch_bounds__(1024) void e4m3_choice_kernel(E4m3Choice a) {
  extern __shared__ uint32_t held[];
  __shared__ uint32_t hist[16][256];
  __shared__ int waves[16];
  __shared__ uint32_t found[2];      // bytes found so far; how many of the bin are wanted
  const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int slot = a.slots[b];
  int* out = a.kept + ((int64_t)b * a.pages.heads + head) * a.keep;
  int n = slot >= 0 && slot < a.slots_of_table ? a.lengths[b] : 0;
  n = min(max(n, 0), a.max_length);
  if (n <= a.keep) {      // everything stays
    for (int i = tid; i < a.keep; i += 1024) out[i] = i < n ? i : -1;
    return;
  }
  const int* row = a.pages.table + (int64_t)slot * a.pages.bt_stride;
  const int lo = a.first, hi = n - a.recent;      // (first + recent <= keep < n)
  const uint32_t m = (uint32_t)(a.keep - a.first - a.recent);
  auto read = [&](int j) -> uint32_t {
    const int page = row[j / a.pages.page_size];
    return page < 0 ? 0u : ordered(a.pages.weight[((int64_t)page * a.pages.heads + head) * a.pages.page_size + j % a.pages.page_size]);
  };
  const int in_lds = min(hi, lo + CHOICE_HELD);
  for (int j = lo + tid; j < in_lds; j += 1024) held[j - lo] = read(j);
  auto key = [&](int j) -> uint32_t { return j < in_lds ? held[j - lo] : read(j); };
  uint32_t prefix = 0u, want = m;
  if (m > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 16 * 256; i += 1024) hist[i / 256][i % 256] = 0u;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += 1024) {
        const uint32_t k = key(j);
        if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[wave][k >> shift & 255u], 1u);
      }
      __syncthreads();
      if (tid < 256) {
        uint32_t s = 0u;
#pragma unroll
        for (int w = 0; w < 16; ++w) s += hist[w][tid];
        hist[0][tid] = s;
      }
      __syncthreads();
      if (wave == 0) {
        // four bins to a lane, from the highest: lane l holds bins 255 - 4 l .. 252 - 4 l
        uint32_t c[4], mine = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += c[i] = hist[0][255 - 4 * lane - i];
        uint32_t above = (uint32_t)wave_scan_add((int)mine) - mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (above < want && above + c[i] >= want) {      // one bin alone
            found[0] = prefix << 8 | (uint32_t)(255 - 4 * lane - i);
            found[1] = want - above;
          }
          above += c[i];
        }
      }
      __syncthreads();
      prefix = found[0];
      want = found[1];
    }
  }
  // prefix is the m-th largest weight, and the `want` first positions with that weight stay
  int at = 0;      // kept so far
  uint32_t same = 0u;      // of them and those left out, positions with that weight
  for (int j0 = 0; j0 < n; j0 += 1024) {
    const int j = j0 + tid;
    const bool between = j >= lo && j < hi;
    const uint32_t k = between && m > 0 ? key(j) : 0u;
    const bool equal = between && m > 0 && k == prefix;
    const uint64_t eq = __ballot(equal);
    if (lane == 0) waves[wave] = __popcll(eq);
    __syncthreads();
    uint32_t before = same, all = 0u;
    for (int w = 0; w < 16; ++w) {
      before += w < wave ? waves[w] : 0;
      all += waves[w];
    }
    before += __popcll(eq & ((1ull << lane) - 1ull));
    same += all;
    const bool stays = j < n && (!between || (m > 0 && (k > prefix || (equal && before < want))));
    const uint64_t st = __ballot(stays);
    __syncthreads();
    if (lane == 0) waves[wave] = __popcll(st);
    __syncthreads();
    int to = at, total = 0;
    for (int w = 0; w < 16; ++w) {
      to += w < wave ? waves[w] : 0;
      total += waves[w];
    }
    to += __popcll(st & ((1ull << lane) - 1ull));
    if (stays && to < a.keep) out[to] = j;
    at += total;
    __syncthreads();
  }
}

// kept [B][heads][keep]: the chosen positions in ascending order, for every layer and kv head; a sequence of keep positions or
// fewer keeps all of them, with -1 behind.
TQ_API int tq_e4m3_choose(const int* slots, const int* lengths, int B, int max_length, int keep, int first, int recent, int* kept,
                          const float* weight, const int* table, int slots_of_table, int bt_stride, int page_size, int heads,
                          hipStream_t st) {
  if (B <= 0) return 0;
  if (keep < 1 || first < 0 || recent < 0 || first > keep - recent || !weight || page_size < 1 || heads < 1) return TQ_ERR_BAD_ARG;
  if (B > 65535 || max_length < 0 || max_length > (int64_t)bt_stride * page_size) return TQ_ERR_UNSUPPORTED;
  E4m3Choice a{slots, lengths, kept, keep, first, recent, slots_of_table, max_length,
               E4m3Pages{nullptr, nullptr, nullptr, nullptr, (float*)weight, table, bt_stride, page_size, heads, 0, 16}};
  const size_t shmem = (size_t)(max_length < CHOICE_HELD ? max_length : CHOICE_HELD) * 4;
  const hipError_t e = hipFuncSetAttribute((const void*)e4m3_choice_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(e4m3_choice_kernel, dim3(heads, B), dim3(1024), shmem, st, a);
  TQ_LAUNCH_CHECK();
  return 0;
}

// ------------------------------------------------------------------------------------------ eviction: the move
// A workgroup fills one tile of 64 positions of one sequence, layer and kv head from the positions that were chosen, each wherever it
// lies: keys 16 bytes at a time, values, whose positions lie side by side, by bytes out of the source's tiles, which pass through LDS
// one after the other (positions are in ascending order).  A block's scale is the largest of its positions' blocks; the codes
// of the others are brought to it.  Rows behind the last position are zeros up to the end of their page.
struct E4m3Move {
  const int* src;
  const int* dst;
  const int* kept;
  int keep, slots_of_table;
  E4m3Pages pages;
};
__global__ __launch_bounds__(256) void e4m3_move_kernel(E4m3Move a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];      // two of [hd][68]: the source's values, the destination's
  __shared__ int from[E4M3_TILE];
  __shared__ int64_t head_of[E4M3_TILE];
  __shared__ float scale[2][E4M3_TILE], ratio[2][E4M3_TILE];
  const int hd = a.pages.hd, tid = threadIdx.x, b = blockIdx.z, head = blockIdx.y, tile = blockIdx.x, per = a.pages.page_size / E4M3_TILE;
  const int s = a.src[b], t = a.dst[b];
  if (s < 0 || s >= a.slots_of_table || t < 0 || t >= a.slots_of_table) return;
  const int to_page = a.pages.table[(int64_t)t * a.pages.bt_stride + tile / per];
  if (to_page < 0) return;
  const int* row = a.pages.table + (int64_t)s * a.pages.bt_stride;
  const int64_t to = (int64_t)to_page * a.pages.heads + head;
  const int in_page = tile % per;
  if (tid < E4M3_TILE) {
    const int i = tile * E4M3_TILE + tid;
    int j = i < a.keep ? a.kept[((int64_t)b * a.pages.heads + head) * a.keep + i] : -1;
    if (j >= 0 && (j >= a.pages.bt_stride * a.pages.page_size || row[j / a.pages.page_size] < 0)) j = -1;
    from[tid] = j;
    const int64_t h = j < 0 ? 0 : (int64_t)row[j / a.pages.page_size] * a.pages.heads + head;
    head_of[tid] = h;
    const int64_t at = h * a.pages.page_size + (j < 0 ? 0 : j % a.pages.page_size);
    scale[0][tid] = j < 0 ? 0.f : a.pages.k_scale[at / E4M3_BLOCK];
    scale[1][tid] = j < 0 ? 0.f : a.pages.v_scale[at / E4M3_BLOCK];
    if (a.pages.weight) a.pages.weight[to * a.pages.page_size + in_page * E4M3_TILE + tid] = j < 0 ? 0.f : a.pages.weight[at];
  }
  uint8_t* mine = tiles + hd * 68;
  for (int i = tid; i < hd * 17; i += 256) reinterpret_cast<uint32_t*>(mine)[i] = 0u;
  __syncthreads();
  if (tid < 2 * E4M3_TILE) {
    const int m = tid / E4M3_TILE, i = tid % E4M3_TILE;
    float top = 0.f;
    for (int e = 0; e < E4M3_BLOCK; ++e) top = fmaxf(top, scale[m][i / E4M3_BLOCK * E4M3_BLOCK + e]);
    ratio[m][i] = scale[m][i] * e4m3_inverse(top);
    if (i % E4M3_BLOCK == 0) (m ? a.pages.v_scale : a.pages.k_scale)[e4m3_scale_at(a.pages, to, in_page) + i / E4M3_BLOCK] = top;
  }
  __syncthreads();
  uint8_t* kt = a.pages.k + e4m3_tile_at(a.pages, to, in_page);
  for (int i = tid; i < E4M3_TILE * (hd / 16); i += 256) {
    const int r = i % E4M3_TILE, ch = i / E4M3_TILE, j = from[r];
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (j >= 0) {
      w = *reinterpret_cast<const uint4*>(a.pages.k + e4m3_tile_at(a.pages, head_of[r], j % a.pages.page_size / E4M3_TILE) +
                                          ch * 16 * E4M3_TILE + j % E4M3_TILE * 16);
      const float f = ratio[0][r];
      if (f != 1.f)
        w = make_uint4(e4m3_rescale(w.x, f, f, f, f), e4m3_rescale(w.y, f, f, f, f), e4m3_rescale(w.z, f, f, f, f), e4m3_rescale(w.w, f, f, f, f));
    }
    *reinterpret_cast<uint4*>(kt + ch * 16 * E4M3_TILE + r * 16) = w;
  }
  // values: runs of destination rows that come from one tile of the source (the same for all threads)
  for (int r = 0; r < E4M3_TILE;) {
    const int j = from[r];
    if (j < 0) {
      ++r;
      continue;
    }
    int end = r + 1;
    while (end < E4M3_TILE && from[end] >= 0 && from[end] / E4M3_TILE == j / E4M3_TILE) ++end;
    const uint32_t* vt = reinterpret_cast<const uint32_t*>(a.pages.v + e4m3_tile_at(a.pages, head_of[r], j % a.pages.page_size / E4M3_TILE));
    for (int i = tid; i < hd * 16; i += 256) reinterpret_cast<uint32_t*>(tiles)[i / 16 * 17 + i % 16] = vt[i];
    __syncthreads();
    for (int i = tid; i < hd * (end - r); i += 256) {
      const int d = i % hd, q = r + i / hd, p = from[q] % E4M3_TILE;
      mine[d * 68 + q % 16 / 4 * 16 + q / 16 * 4 + q % 4] = tiles[d * 68 + p % 16 / 4 * 16 + p / 16 * 4 + p % 4];
    }
    __syncthreads();
    r = end;
  }
  uint32_t* vt = reinterpret_cast<uint32_t*>(a.pages.v + e4m3_tile_at(a.pages, to, in_page));
  for (int i = tid; i < hd * 16; i += 256) {
    const int d = i / 16, c = i % 16 / 4, j = i % 4, p = 16 * j + 4 * c;
    vt[i] = e4m3_rescale(reinterpret_cast<const uint32_t*>(mine)[d * 17 + i % 16], ratio[1][p], ratio[1][p + 1], ratio[1][p + 2], ratio[1][p + 3]);
  }
}

// Fills the pages of the table's rows dst[b] with the positions kept[b][layer, kv head] of its rows src[b], whose pages are others.
// Whole pages are written: ceil(keep / page_size) of them.
TQ_API int tq_e4m3_move(const int* src, const int* dst, int B, const int* kept, int keep, int hd, void* k, void* v, float* k_scale,
                        float* v_scale, float* weight, const int* table, int slots_of_table, int bt_stride, int page_size, int heads,
                        hipStream_t st) {
  if (B <= 0) return 0;
  if (keep < 1) return TQ_ERR_BAD_ARG;
  if (!e4m3_pages_fit(page_size, heads, 0, 1, hd) || heads > 65535 || B > 65535 || keep > (int64_t)bt_stride * page_size) return TQ_ERR_UNSUPPORTED;
  E4m3Move a{src, dst, kept, keep, slots_of_table,
             E4m3Pages{(uint8_t*)k, (uint8_t*)v, k_scale, v_scale, weight, table, bt_stride, page_size, heads, 0, hd}};
  const int tiles = (keep + page_size - 1) / page_size * (page_size / E4M3_TILE);
  hipLaunchKernelGGL(e4m3_move_kernel, dim3(tiles, heads, B), dim3(256), 2 * (size_t)hd * 68, st, a);
  TQ_LAUNCH_CHECK();
  return 0;
}
