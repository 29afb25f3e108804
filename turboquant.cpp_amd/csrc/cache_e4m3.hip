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
  int kv_heads;                 // kv heads that a workgroup of keys and values goes through, one after the other
  int q_tokens, q_heads;        // tokens and heads of a workgroup of queries
  E4m3Pages pages;
  int write;
};
#define WRITE_THREADS 512
#define WRITE_HEADS 8             // most kv heads of a workgroup

__device__ __forceinline__ float bias_at(const E4m3Write& a, int i) {
  return a.bias_type == TQ_BF16 ? to_f32(((const bf16_t*)a.bias)[i]) : ((const float*)a.bias)[i];
}
__device__ __forceinline__ float4 bias_four(const E4m3Write& a, int i) {
  if (a.bias_type == TQ_F32) return *reinterpret_cast<const float4*>((const float*)a.bias + i);
  const uint2 w = *reinterpret_cast<const uint2*>((const bf16_t*)a.bias + i);
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ float4 plus(float4 x, float4 y) { return make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w); }
// Numbers col .. col + 3 of a token whose row begins `at` numbers behind `base`: 32 bits of offset from an address that all lanes share.
__device__ __forceinline__ float4 four_at(const float* base, uint32_t at, int col) { return *reinterpret_cast<const float4*>(base + (at + (uint32_t)col)); }
// Sine and cosine of the exact product p * f (48 bits, which 64-bit numbers hold), in 64 bits: reduced to an eighth of a turn about the
// nearest quarter, then the series of sine and cosine, whose first omitted terms are r^13 / 13! and r^12 / 12! (1e-10 and less).  In 32
// bits the product alone would be off by 0.004 at position 100,000, and the keys' codes would differ from exact ones more often than
// rounding makes them (with 1 ulp of error in the sine, 1.5 times as far from 64 bits as correctly rounded sines).
struct Turn {
  double c, s;
};
__device__ __forceinline__ Turn turn_at(double x) {
  const double k = rint(x * 0.63661977236758134308);      // 2 / pi
  const double r = fma(k, -6.123233995736766036e-17, fma(k, -1.5707963267948965580, x)), z = r * r;      // pi / 2 in two parts
  const double s = r * (1. + z * (-1. / 6 + z * (1. / 120 + z * (-1. / 5040 + z * (1. / 362880 + z * (-1. / 39916800))))));
  const double c = 1. + z * (-0.5 + z * (1. / 24 + z * (-1. / 720 + z * (1. / 40320 + z * (-1. / 3628800)))));
  const int q = (int)((int64_t)k & 3);
  return Turn{q == 0 ? c : q == 1 ? -s : q == 2 ? -c : s, q == 0 ? s : q == 1 ? c : q == 2 ? -s : -c};
}
__device__ __forceinline__ float2 turn_of(int p, float f, float amp) {
  const Turn t = turn_at((double)p * (double)f);
  return make_float2(amp * (float)t.c, amp * (float)t.s);
}
// The cosines and sines of a tile's `rows` new tokens, [rows][n], by all threads.  A thread's rows whose positions follow one another take them from
// the first's by the sum of two angles, four operations instead of some forty, in 64 bits: at most TURN_ROWS - 1 times, each of which adds the
// step's error to what there is, so that they are off by 8 times what the series are at most, 2^-30.  A thread with fewer than four rows works each
// out, and asks for no other positions.  Against each worked out: 4,096 tokens of 16 heads on 16 45.4 -> 41.1 us, of 28 on 4 33.7 -> 32.6, ragged turns
// of 3 to 900 51.4 -> 50.6; but 8 turns of 40 to 300 15.2 -> 16.0 and 32-bit ones of 1 to 333 10.3 -> 10.5, whose tiles are mostly new in part.  (Tiles
// that are new in part by a loop of their own: those 15.2 and 10.4, but the long prompt 42.9.)
#define TURN_ROWS 8
__device__ __forceinline__ void turns_of(const E4m3Write& a, const int* positions, int rows, int n, float2* turns) {
  const int share = min(TURN_ROWS, rows * n / WRITE_THREADS), each = share < 4 ? 1 : share, parts = (rows + each - 1) / each;
  for (int i = threadIdx.x; i < parts * n; i += WRITE_THREADS) {
    const int f = i % n, r0 = i / n * each, count = min(each, rows - r0), p0 = positions[r0];
    const double freq = (double)a.inv_freq[f];
    bool follow = true;
    if (count > 1)
#pragma unroll
      for (int u = 1; u < TURN_ROWS; ++u) follow = follow && positions[r0 + min(u, count - 1)] == p0 + min(u, count - 1);
    Turn t = turn_at((double)p0 * freq), step = t;
    if (count > 1) step = turn_at(freq);
#pragma unroll 1
    for (int u = 0; u < count; ++u) {
      turns[(r0 + u) * n + f] = make_float2(a.amp * (float)t.c, a.amp * (float)t.s);
      t = follow ? Turn{t.c * step.c - t.s * step.s, t.s * step.c + t.c * step.s} : turn_at((double)positions[r0 + min(u + 1, count - 1)] * freq);
    }
  }
}
// Four neighbouring numbers of a head from dimension d on, rotated, in two steps: what is read, and what becomes of it (`turn`: the token's
// cosines and sines).  FOURS: four numbers rotate alike (pairs by halves, a multiple of four of them, or neighbouring pairs, an even
// number of them).
struct Raw {
  float4 x, y;      // the numbers, and with pairs by halves their partners
};
// (Nothing waits in here: all that a thread needs is asked for before the first of it is used.)
template <bool FOURS>
__device__ __forceinline__ int partner_of(const E4m3Write& a, int d) {
  const int n = a.rot / 2;
  return FOURS && a.pairing == 0 && d < 2 * n ? (d < n ? d + n : d - n) : d;
}
template <bool FOURS>
__device__ __forceinline__ Raw read_four(const E4m3Write& a, const float* base, uint32_t at, int col, int d) {
  return Raw{four_at(base, at, col + d), four_at(base, at, col + partner_of<FOURS>(a, d))};
}
template <bool FOURS>
__device__ __forceinline__ void add_bias(const E4m3Write& a, Raw& w, int col, int d) {
  w.x = plus(w.x, bias_four(a, col + d));
  w.y = plus(w.y, bias_four(a, col + partner_of<FOURS>(a, d)));
}
template <bool FOURS>
__device__ __forceinline__ float4 rotated(const E4m3Write& a, const Raw& w, const float* base, uint32_t at, int col, int d, const float2* turn) {
  const int n = a.rot / 2;
  const float4 x = w.x, y = w.y;
  if (d >= 2 * n) return x;
  if constexpr (FOURS) {
    if (a.pairing == 1) {
      const float2 t0 = turn[d / 2], t1 = turn[d / 2 + 1];
      return make_float4(x.x * t0.x - x.y * t0.y, x.x * t0.y + x.y * t0.x, x.z * t1.x - x.w * t1.y, x.z * t1.y + x.w * t1.x);
    }
    const bool low = d < n;
    const float2* t = turn + (low ? d : d - n);
    const float2 t0 = t[0], t1 = t[1], t2 = t[2], t3 = t[3];
    const float f = low ? -1.f : 1.f;
    return make_float4(x.x * t0.x + f * y.x * t0.y, x.y * t1.x + f * y.y * t1.y, x.z * t2.x + f * y.z * t2.y, x.w * t3.x + f * y.w * t3.y);
  }
  float o[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = d + j;
    if (e < 2 * n) {
      const bool low = a.pairing == 0 ? e < n : e % 2 == 0;
      const int other = col + (a.pairing == 0 ? (low ? e + n : e - n) : e ^ 1);
      const float z = base[at + (uint32_t)other] + (a.bias ? bias_at(a, other) : 0.f);
      const float2 t = turn[a.pairing == 0 ? (low ? e : e - n) : e / 2];
      o[j] = o[j] * t.x + (low ? -z : z) * t.y;
    }
  }
  return make_float4(o[0], o[1], o[2], o[3]);
}
__device__ __forceinline__ float largest(float4 v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }
__device__ __forceinline__ bool all_usable(float4 v) {
  return fabsf(v.x) < E4M3_TOO_LARGE && fabsf(v.y) < E4M3_TOO_LARGE && fabsf(v.z) < E4M3_TOO_LARGE && fabsf(v.w) < E4M3_TOO_LARGE;
}

// A workgroup takes either one tile of 64 positions of one sequence and up to kv_heads kv heads in turn (keys and values: a row that is
// not finite in one is marked in both), or the queries of q_tokens tokens and q_heads heads.  The tokens' cosines and sines are worked
// out once and kept in LDS.  Every number is read once (keys and queries that rotate by halves: twice) and stays in registers until its block's
// scale is known: a thread holds four neighbouring numbers of KI rows of keys, in an order that gives a wave rows of one block only,
// and 16 positions of KI / 4 dimensions of values, the 16 codes that lie side by side in the page.
// Bound by the bytes: 4,096 tokens of 16 heads of 128 on 16, 134 MB, take 37 us (3.6 TB/s; a large copy does 5.1).
template <int KI, bool FOURS>
__global__ __launch_bounds__(WRITE_THREADS) __attribute__((amdgpu_waves_per_eu(KI > 4 ? 2 : 4))) void e4m3_write_kernel(E4m3Write a) {
  extern __shared__ __attribute__((aligned(16))) float2 turns[];
  const int hd = a.hd, n = a.rot / 2, fours = hd / 4;
  int tid = threadIdx.x;
  const uint32_t ld = (uint32_t)a.ld;
  const int kv_per = (a.nkv + a.kv_heads - 1) / max(a.kv_heads, 1), kv_groups = a.write ? a.tiles * kv_per * a.B : 0;
  if ((int)blockIdx.x >= kv_groups) {
    const int w = (int)blockIdx.x - kv_groups, per = (a.nh + a.q_heads - 1) / a.q_heads;
    const int t0 = w / per * a.q_tokens, h0 = w % per * a.q_heads;
    const int nt = min(a.q_tokens, a.T - t0), heads = min(a.q_heads, a.nh - h0);
    // four items of a thread are on their way at a time, the first of them while the angles are worked out (4,096 tokens of 28 heads: 32.6 -> 29.2 us);
    // a workgroup's few rows give a thread an angle or two, so that no sum of angles would be shared
    const int items = nt * heads * fours;
    const float* base = a.x + (int64_t)t0 * a.ld;
    Raw raw[4];
    auto ask = [&](int i0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(i0 + u * WRITE_THREADS, items - 1), d = i % fours * 4, th = i / fours;
        raw[u] = read_four<FOURS>(a, base, (uint32_t)(th / heads) * ld, (h0 + th % heads) * hd, d);
      }
    };
    ask(tid);
    for (int i = tid; i < nt * n; i += WRITE_THREADS) turns[i] = turn_of(a.positions[t0 + i / n], a.inv_freq[i % n], a.amp);
    __syncthreads();
    for (int i0 = tid; i0 < items; i0 += 4 * WRITE_THREADS) {
      if (i0 != tid) ask(i0);
      if (a.bias)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = min(i0 + u * WRITE_THREADS, items - 1);
          add_bias<FOURS>(a, raw[u], (h0 + i / fours % heads) * hd, i % fours * 4);
        }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * WRITE_THREADS, d = i % fours * 4, th = i / fours, h = h0 + th % heads, t = th / heads;
        if (i >= items) break;
        const float4 o = rotated<FOURS>(a, raw[u], base, (uint32_t)t * ld, h * hd, d, turns + t * n);
        act_t* out = a.q + ((int64_t)(t0 + t) * a.nh + h) * hd + d;
#if defined(TQ_ACT_BF16)
        *reinterpret_cast<uint2*>(out) = make_uint2(f32_to_bf16_pair(o.x, o.y), f32_to_bf16_pair(o.z, o.w));
#else
        *reinterpret_cast<float4*>(out) = o;
#endif
      }
    }
    return;
  }
  constexpr int VI = KI / 4;
  const int kvh0 = (int)blockIdx.x % kv_per * a.kv_heads, b = (int)blockIdx.x / kv_per % a.B, nth = (int)blockIdx.x / kv_per / a.B;
  const int t0 = a.cu[b], count = a.cu[b + 1] - t0, start = a.start[b];
  const int tile = start / E4M3_TILE + nth, pos0 = tile * E4M3_TILE;
  if (count <= 0 || pos0 >= start + count) return;
  const int r0 = max(start - pos0, 0), r1 = min(start + count - pos0, E4M3_TILE);      // the tile's rows that are new
  const int old0 = r0 / E4M3_BLOCK * E4M3_BLOCK;      // rows old0 .. r0 - 1 share the first new row's block
  __shared__ uint32_t top[WRITE_HEADS][2][4];         // the blocks' largest magnitudes, as bits
  __shared__ uint32_t bad[WRITE_HEADS][2];            // rows that are not finite, a bit each
  __shared__ float inverse[2][2][4], ratio[2][2];     // by turns, so that a wave may still read the last head's
  for (int i = tid; i < WRITE_HEADS * 8; i += WRITE_THREADS) top[i / 8][i / 4 % 2][i % 4] = 0u;
  if (tid < WRITE_HEADS * 2) bad[tid / 2][tid % 2] = 0u;
  const int64_t first = (int64_t)t0 + pos0 - start;      // packed row of the tile's row 0 (rows before r0 are not read)
  const int lane = tid % 64;
  const float* base = a.x + first * a.ld;
  float v[VI][16];
  // (rows that are not new, and places behind the last item, read what lies next: one address instead of a condition around every load)
  auto ask_values = [&](int kvh) {
    const int vcol = (a.nh + a.nkv + kvh) * hd;
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int at = tid + i * WRITE_THREADS, d = at % hd, c = min(at / hd, 3);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int r = min(max(16 * (j / 4) + 4 * c + j % 4, r0), r1 - 1);
        v[i][j] = base[(uint32_t)r * ld + (uint32_t)(vcol + d)];
      }
    }
  };
  int in_page;
  const int64_t head0 = e4m3_head_of(a.pages, a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride, tile, kvh0, in_page);
  if (head0 < 0) return;
  ask_values(kvh0);      // (on their way while the angles are worked out)
  turns_of(a, a.positions + first + r0, r1 - r0, n, turns);
  __syncthreads();
#pragma unroll 1
  for (int hi = 0; hi < a.kv_heads && kvh0 + hi < a.nkv; ++hi) {
    // (places are worked out anew for every head: kept, they would be more registers than a wave has)
    asm volatile("" : "+v"(tid));
    const int kvh = kvh0 + hi, kcol = (a.nh + kvh) * hd;
    const int64_t head = head0 + hi;
    float4 k[KI];
    {
      Raw raw[KI];
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int at = tid + i * WRITE_THREADS, r = min(max(at / fours, r0), r1 - 1);
        raw[i] = read_four<FOURS>(a, base, (uint32_t)r * ld, kcol, at % fours * 4);
      }
      if (a.bias) {
#pragma unroll
        for (int i = 0; i < KI; ++i) add_bias<FOURS>(a, raw[i], kcol, (tid + i * WRITE_THREADS) % fours * 4);
#pragma unroll
        for (int i = 0; i < VI; ++i) {
          const float add = bias_at(a, kcol + a.nkv * hd + (tid + i * WRITE_THREADS) % hd);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[i][j] += add;
        }
      }
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int at = tid + i * WRITE_THREADS, r = min(max(at / fours, r0), r1 - 1), d = at % fours * 4;
        k[i] = rotated<FOURS>(a, raw[i], base, (uint32_t)r * ld, kcol, d, turns + (r - r0) * n);
        if (at / fours != r) k[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int c = (tid + i * WRITE_THREADS) / hd;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int r = 16 * (j / 4) + 4 * c + j % 4;
          if (c >= 4 || r < r0 || r >= r1) v[i][j] = 0.f;
        }
      }
    }
    // largest magnitudes by block, and rows that are not finite
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int r = (tid + i * WRITE_THREADS) / fours;
      const float m = wave_max(largest(k[i]));
      if (lane == 0 && r < E4M3_TILE) atomicMax(&top[hi][0][r / E4M3_BLOCK], __float_as_uint(m));
      if (!all_usable(k[i])) atomicOr(&bad[hi][r / 32], 1u << r % 32);
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int c = (tid + i * WRITE_THREADS) / hd;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 x = make_float4(v[i][4 * j], v[i][4 * j + 1], v[i][4 * j + 2], v[i][4 * j + 3]);
        const float m = wave_max(largest(x));
        if (lane == 0) atomicMax(&top[hi][1][j], __float_as_uint(m));
        if (!all_usable(x))
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 16 * j + 4 * c + e;
            if (!(fabsf(v[i][4 * j + e]) < E4M3_TOO_LARGE)) atomicOr(&bad[hi][r / 32], 1u << r % 32);
          }
      }
    }
    __syncthreads();
    const uint32_t bad0 = bad[hi][0], bad1 = bad[hi][1];
    auto is_bad = [&](int r) { return ((r < 32 ? bad0 : bad1) >> (r % 32) & 1u) != 0u; };
    if (bad0 | bad1) {      // once more without those rows (the same way for all threads)
      __syncthreads();
      if (tid < 8) top[hi][tid / 4][tid % 4] = 0u;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int r = (tid + i * WRITE_THREADS) / fours;
        if (r < E4M3_TILE && !is_bad(r)) atomicMax(&top[hi][0][r / E4M3_BLOCK], __float_as_uint(largest(k[i])));
      }
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int c = (tid + i * WRITE_THREADS) / hd;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c < 4 && !is_bad(16 * (j / 4) + 4 * c + j % 4)) atomicMax(&top[hi][1][j / 4], __float_as_uint(fabsf(v[i][j])));
      }
      __syncthreads();
    }
    if (tid < 8) {
      const int m = tid / 4, j = tid % 4;
      if (j * E4M3_BLOCK < r1 && (j + 1) * E4M3_BLOCK > r0) {
        float* at = (m ? a.pages.v_scale : a.pages.k_scale) + e4m3_scale_at(a.pages, head, in_page) + j;
        float scale = e4m3_scale(__uint_as_float(top[hi][m][j]));
        if (j == r0 / E4M3_BLOCK) {
          const float was = old0 < r0 ? *at : 0.f;
          scale = fmaxf(scale, was);
          ratio[hi % 2][m] = was * e4m3_inverse(scale);      // what the rows before the new ones are multiplied by (1: they stay)
        }
        *at = scale;
        inverse[hi % 2][m][j] = e4m3_inverse(scale);
      }
    }
    __syncthreads();
    uint8_t* kt = a.pages.k + e4m3_tile_at(a.pages, head, in_page);
    uint8_t* vt = a.pages.v + e4m3_tile_at(a.pages, head, in_page);
    const float rk = ratio[hi % 2][0], rv = ratio[hi % 2][1];
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int at = tid + i * WRITE_THREADS, r = at / fours, d = at % fours * 4;
      uint32_t* to = reinterpret_cast<uint32_t*>(kt + d / 16 * (16 * E4M3_TILE) + r * 16 + d % 16);
      if (r >= r0 && r < r1) {
        const float f = inverse[hi % 2][0][r / E4M3_BLOCK];
        *to = is_bad(r) ? 0x7f7f7f7fu : e4m3_codes(k[i].x * f, k[i].y * f, k[i].z * f, k[i].w * f);
      } else if (r >= old0 && r < r0 && rk != 1.f) {
        *to = e4m3_rescale(*to, rk, rk, rk, rk);
      }
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int at = tid + i * WRITE_THREADS, d = at % hd, c = at / hd;
      if (c >= 4) break;
      uint32_t* to = reinterpret_cast<uint32_t*>(vt + d * E4M3_TILE + 16 * c);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = inverse[hi % 2][1][j];      // (of a block that is not written: whatever it is, its codes are not used)
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = is_bad(16 * j + 4 * c + e) ? 0.f : v[i][4 * j + e] * f;
        w[j] = e4m3_codes(x[0], x[1], x[2], x[3]);
      }
      if (r0 == 0 && r1 == E4M3_TILE) {
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        continue;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int p = 16 * j + 4 * c;
        uint32_t mine = 0u, before = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mine |= p + e >= r0 && p + e < r1 ? 0xffu << 8 * e : 0u;
          before |= p + e >= old0 && p + e < r0 ? 0xffu << 8 * e : 0u;
        }
        if (rv == 1.f) before = 0u;
        if (mine == 0xffffffffu) to[j] = w[j];
        else if (mine | before) {
          const uint32_t was = to[j], turned = before ? e4m3_rescale(was, rv, rv, rv, rv) : 0u;
          to[j] = (w[j] & mine) | (turned & before) | (was & ~(mine | before));
        }
      }
    }
    if (a.pages.weight && tid >= r0 && tid < r1) a.pages.weight[head * a.pages.page_size + in_page * E4M3_TILE + tid] = 0.f;
    if (hi + 1 < a.kv_heads && kvh + 1 < a.nkv) ask_values(kvh + 1);
  }
}

// One new token to a sequence, or none: a wave takes a head of a row's queries, or the key and value of a kv head of a sequence's token, four
// neighbouring numbers a lane, and the waves of a workgroup, which do the one or the other, share the token's cosines and sines.  (Rows of queries
// are as many as sequences, and taken by themselves: where a sequence brings no token there are rows that belong to none.)  The same roundings
// as above.  Bound by the reads that follow one another
// and by fetching the code: 8 tokens of 16 heads of 128 on 16 take 5.0 us, and 10.2 in the kernel above, whose code is many times as long.
template <bool FOURS>
__global__ __launch_bounds__(256) void e4m3_write_one_kernel(E4m3Write a) {
  extern __shared__ __attribute__((aligned(16))) float2 turns[];
  const int hd = a.hd, n = a.rot / 2, b = blockIdx.y, lane = threadIdx.x % 64, of_queries = (a.nh + 3) / 4;
  const bool keys = (int)blockIdx.x >= of_queries;
  const int t = keys ? a.cu[b] : b;
  if (keys && a.cu[b + 1] == t) return;
  const int kvh = ((int)blockIdx.x - of_queries) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64), h = keys ? a.nh + kvh : kvh + of_queries * 4;
  const bool mine = h < (keys ? a.nh + a.nkv : a.nh), has = 4 * lane < hd;
  const int d = has ? 4 * lane : 0, col = mine ? h * hd : 0, vcol = mine && keys ? col + a.nkv * hd : col;
  const float* base = a.x + (int64_t)t * a.ld;
  Raw raw = read_four<FOURS>(a, base, 0, col, d);
  float4 v = four_at(base, 0, vcol + d);
  const int pos = a.start[b], row = pos % E4M3_TILE, j = row / E4M3_BLOCK, in_block = row % E4M3_BLOCK;
  int in_page = 0;
  const int64_t head = mine && keys ? e4m3_head_of(a.pages, a.pages.table + (int64_t)a.slots[b] * a.pages.bt_stride, pos / E4M3_TILE, kvh, in_page) : -1;
  const int64_t scale_at = head < 0 ? 0 : e4m3_scale_at(a.pages, head, in_page) + j;
  const float held_k = head >= 0 && in_block > 0 ? a.pages.k_scale[scale_at] : 0.f, held_v = head >= 0 && in_block > 0 ? a.pages.v_scale[scale_at] : 0.f;
  if (a.bias) {
    add_bias<FOURS>(a, raw, col, d);
    v = plus(v, bias_four(a, vcol + d));
  }
  for (int i = threadIdx.x; i < n; i += 256) turns[i] = turn_of(a.positions[t], a.inv_freq[i], a.amp);
  __syncthreads();
  if (!mine || (keys && head < 0)) return;
  const float4 k = rotated<FOURS>(a, raw, base, 0, col, d, turns);
  if (!keys) {
    if (!has) return;
    act_t* out = a.q + ((int64_t)t * a.nh + h) * hd + d;
#if defined(TQ_ACT_BF16)
    *reinterpret_cast<uint2*>(out) = make_uint2(f32_to_bf16_pair(k.x, k.y), f32_to_bf16_pair(k.z, k.w));
#else
    *reinterpret_cast<float4*>(out) = k;
#endif
    return;
  }
  const bool bad = __any(!all_usable(k) || !all_usable(v));      // (lanes without numbers of their own hold the head's first)
  const float scale_k = fmaxf(e4m3_scale(bad ? 0.f : wave_max(largest(k))), held_k), scale_v = fmaxf(e4m3_scale(bad ? 0.f : wave_max(largest(v))), held_v);
  const float fk = e4m3_inverse(scale_k), fv = e4m3_inverse(scale_v);
  if (lane == 0) {
    a.pages.k_scale[scale_at] = scale_k;
    a.pages.v_scale[scale_at] = scale_v;
    if (a.pages.weight) a.pages.weight[head * a.pages.page_size + in_page * E4M3_TILE + row] = 0.f;
  }
  if (!has) return;
  uint8_t* kt = a.pages.k + e4m3_tile_at(a.pages, head, in_page) + d / 16 * (16 * E4M3_TILE) + d % 16;
  uint8_t* vt = a.pages.v + e4m3_tile_at(a.pages, head, in_page) + d * E4M3_TILE + 4 * j;
  *reinterpret_cast<uint32_t*>(kt + row * 16) = bad ? 0x7f7f7f7fu : e4m3_codes(k.x * fk, k.y * fk, k.z * fk, k.w * fk);
  const uint32_t vc = bad ? 0u : e4m3_codes(v.x * fv, v.y * fv, v.z * fv, v.w * fv);
#pragma unroll
  for (int e = 0; e < 4; ++e) vt[e * E4M3_TILE + in_block / 4 * 16 + in_block % 4] = (uint8_t)(vc >> 8 * e);
  // what the block holds already, where its scale has grown
  if (in_block > 0 && scale_k != held_k) {
    const float f = held_k * fk;
    for (int r = row - in_block; r < row; ++r) {
      uint32_t* to = reinterpret_cast<uint32_t*>(kt + r * 16);
      *to = e4m3_rescale(*to, f, f, f, f);
    }
  }
  if (in_block > 0 && scale_v != held_v) {
    const float f = held_v * fv;
    for (int i = 0; i < 4 * ((in_block + 3) / 4); ++i) {      // (dimension i % 4, positions 4 (i / 4) .. of the block)
      uint32_t* to = reinterpret_cast<uint32_t*>(vt + i % 4 * E4M3_TILE + i / 4 * 16);
      const uint32_t before = in_block - i / 4 * 4 >= 4 ? 0xffffffffu : (1u << 8 * (in_block - i / 4 * 4)) - 1u, old = *to;
      *to = (e4m3_rescale(old, f, f, f, f) & before) | (old & ~before);
    }
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
  if (ld < (int64_t)(nh + 2 * nkv) * hd || ld % 4 != 0 || ld > (1 << 25) || (uintptr_t)x % 16 != 0 || nh <= 0 || max_new <= 0) return TQ_ERR_BAD_ARG;
  if (!e4m3_pages_fit(page_size, heads, head0, k ? nkv : 1, hd)) return TQ_ERR_UNSUPPORTED;
  E4m3Write a{x, ld, bias, bias_type, positions, inv_freq, pairing, rot, amp, cu, slots, start, (act_t*)q, T, B, nh, nkv, hd,
              (max_new + E4M3_TILE - 2) / E4M3_TILE + 1, 1, 1, nh,
              E4m3Pages{(uint8_t*)k, (uint8_t*)v, k_scale, v_scale, weight, table, bt_stride, page_size, heads, head0, hd}, k != nullptr};
  // as many heads, and tokens of queries, to a workgroup (which share the angles) as leave the chip a few workgroups to a compute unit
  while (a.write && a.kv_heads < WRITE_HEADS && a.kv_heads < nkv && (int64_t)a.tiles * B * nkv / a.kv_heads >= 1024) a.kv_heads *= 2;
  while (a.q_heads > 1 && (int64_t)T * ((nh + a.q_heads - 1) / a.q_heads) < 512) a.q_heads = (a.q_heads + 1) / 2;
  while (a.q_tokens < 8 && T / a.q_tokens >= 1024) a.q_tokens *= 2;
  const int64_t kv_groups = a.write ? (int64_t)a.tiles * ((nkv + a.kv_heads - 1) / a.kv_heads) * B : 0;
  const int64_t groups = kv_groups + (int64_t)((T + a.q_tokens - 1) / a.q_tokens) * ((nh + a.q_heads - 1) / a.q_heads);
  if (groups > 0x7FFFFF) return TQ_ERR_UNSUPPORTED;      // (a launch's threads are counted in 32 bits)
  // at most 64 KiB for the angles of 64 rows of 256 numbers, and the kernel has less than 1 KiB beside them
  const size_t shmem = (size_t)(a.write ? min(E4M3_TILE, max(max_new, a.q_tokens)) : a.q_tokens) * (rot / 2) * sizeof(float2);
  const dim3 grid((unsigned)groups), block(WRITE_THREADS);
  const bool fours = rot % (pairing == 0 ? 8 : 4) == 0;
  if (max_new == 1 && T == B && T <= 65535) {
    const dim3 one((nh + 3) / 4 + (k ? (nkv + 3) / 4 : 0), T);
    if (fours) hipLaunchKernelGGL(e4m3_write_one_kernel<true>, one, dim3(256), rot / 2 * sizeof(float2), st, a);
    else hipLaunchKernelGGL(e4m3_write_one_kernel<false>, one, dim3(256), rot / 2 * sizeof(float2), st, a);
    TQ_LAUNCH_CHECK();
    return 0;
  }
  const auto kernel = hd <= 128 ? (fours ? e4m3_write_kernel<4, true> : e4m3_write_kernel<4, false>) : fours ? e4m3_write_kernel<8, true> : e4m3_write_kernel<8, false>;
  if (shmem > 63 * 1024) {      // (with what the kernel has beside it more than goes unasked)
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(kernel, grid, block, shmem, st, a);
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
// Sums of all threads' numbers: of those in front of a thread, and of all.  `waves`: 16 words of LDS.
__device__ __forceinline__ int sum_before(int v, int* waves, int& all) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int upto = wave_scan_add(v);
  __syncthreads();
  if (lane == 63) waves[wave] = upto;
  __syncthreads();
  int before = upto - v;
  all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    before += w < wave ? waves[w] : 0;
    all += waves[w];
  }
  return before;
}
__global__ __launch_bounds__(1024) void e4m3_choice_kernel(E4m3Choice a) {
  extern __shared__ uint32_t held[];
  __shared__ uint32_t hist[4][256];
  __shared__ int waves[16];
  __shared__ uint32_t found[3];      // bytes found so far; how many of the bin are wanted; whether that is all of it
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
  int shift = 24;
  if (m > 0) {
    for (;; shift -= 8) {
      hist[tid / 256][tid % 256] = 0u;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += 1024) {
        const uint32_t k = key(j);
        if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[wave % 4][k >> shift & 255u], 1u);
      }
      __syncthreads();
      if (wave == 0) {
        // four bins to a lane, from the highest: lane l holds bins 255 - 4 l .. 252 - 4 l
        uint32_t c[4], mine = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int bin = 255 - 4 * lane - i;
          mine += c[i] = hist[0][bin] + hist[1][bin] + hist[2][bin] + hist[3][bin];
        }
        uint32_t above = (uint32_t)wave_scan_add((int)mine) - mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (above < want && above + c[i] >= want) {      // one bin alone
            found[0] = prefix << 8 | (uint32_t)(255 - 4 * lane - i);
            found[1] = want - above;
            found[2] = above + c[i] == want;
          }
          above += c[i];
        }
      }
      __syncthreads();
      prefix = found[0];
      want = found[1];
      if (shift == 0 || found[2]) break;      // (a bin that stays whole needs no more bytes)
    }
  }
  // prefix is what the m-th largest weight's bytes from `shift` on are: larger ones stay, and of those with these bytes the `want` first.
  // A thread takes neighbouring positions, so that two sums over threads place them all.
  const int each = (n + 1023) / 1024, j0 = tid * each, j1 = min(j0 + each, n);
  int equal = 0, stay = 0, all;
  for (int j = j0; j < j1; ++j) {
    if (j < lo || j >= hi) ++stay;
    else if (m > 0) {
      const uint32_t k = key(j) >> shift;
      equal += k == prefix;
      stay += k > prefix;
    }
  }
  const int equal_before = sum_before(equal, waves, all);
  int left = max((int)want - equal_before, 0);
  if (m == 0) left = 0;
  int to = sum_before(stay + min(left, equal), waves, all);
  for (int j = j0; j < j1; ++j) {
    bool s = j < lo || j >= hi;
    if (!s && m > 0) {
      const uint32_t k = key(j) >> shift;
      s = k > prefix || (k == prefix && left-- > 0);
    }
    if (s && to < a.keep) out[to++] = j;
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
  if (shmem > 56 * 1024) {      // (with what the kernel has beside it more than goes unasked; always the most: another thread's launch may come between)
    const hipError_t e = hipFuncSetAttribute((const void*)e4m3_choice_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, CHOICE_HELD * 4);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(e4m3_choice_kernel, dim3(heads, B), dim3(1024), shmem, st, a);
  TQ_LAUNCH_CHECK();
  return 0;
}

// ------------------------------------------------------------------------------------------ eviction: the move
// A workgroup fills one tile of 64 positions of one sequence, layer and kv head from the positions that were chosen, each wherever it
// lies: keys 16 bytes at a time; values, whose positions lie side by side, by bytes out of the source's tiles, which come through LDS whole
// (positions are in ascending order: a tile of which half the positions stay comes from two or three).  A thread
// puts 16 positions of a dimension together.  A block's scale is the largest of its positions' blocks; the codes of the others are
// brought to it.  Rows behind the last position are zeros up to the end of their page.
// Bound by the bytes: lines of the source are read whole, twice what stays where every other position does.  Half of 8 sequences of
// 8,192 positions, 6 layers and 16 kv heads of 128, 1.6 GB read and 0.8 written, take 532 us (a large copy of as many bytes 470).
#define MOVE_PITCH 80      // bytes between the dimensions of a tile in LDS: 16 of them, four positions each, touch banks of their own
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
struct E4m3Move {
  const int* src;
  const int* dst;
  const int* kept;
  int keep, slots_of_table, tiles;
  int at_once;                  // tiles of values that come through LDS at a time
  E4m3Pages pages;
};
template <int VI>
__global__ __launch_bounds__(256) void e4m3_move_kernel(E4m3Move a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];      // [at_once][hd][80]
  __shared__ int from[E4M3_TILE], at_slot[E4M3_TILE], n_slots;      // places in the source; which of its tiles (numbered as they come)
  __shared__ int64_t head_of[E4M3_TILE];
  __shared__ int64_t tile_of[E4M3_TILE];      // where the numbered tiles lie
  __shared__ float scale[2][E4M3_TILE], ratio[2][E4M3_TILE];
  // neighbouring tiles, which share lines of the source, on one die: workgroups are dealt to the eight dies by turns
  const int64_t all = gridDim.x, at_once = all % 8 == 0 ? (int64_t)(blockIdx.x % 8) * (all / 8) + blockIdx.x / 8 : blockIdx.x;
  const int tile = (int)(at_once % a.tiles), head = (int)(at_once / a.tiles % a.pages.heads), b = (int)(at_once / a.tiles / a.pages.heads);
  const int hd = a.pages.hd, tid = threadIdx.x, per = a.pages.page_size / E4M3_TILE;
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
    int page = j >= 0 && j / a.pages.page_size < a.pages.bt_stride ? row[j / a.pages.page_size] : -1;
    if (page < 0) j = -1;
    const int64_t h = j < 0 ? 0 : (int64_t)page * a.pages.heads + head;
    const int64_t at = h * a.pages.page_size + (j < 0 ? 0 : j % a.pages.page_size);
    scale[0][tid] = j < 0 ? 0.f : a.pages.k_scale[at / E4M3_BLOCK];
    scale[1][tid] = j < 0 ? 0.f : a.pages.v_scale[at / E4M3_BLOCK];
    if (a.pages.weight) a.pages.weight[to * a.pages.page_size + in_page * E4M3_TILE + tid] = j < 0 ? 0.f : a.pages.weight[at];
    from[tid] = j;
    head_of[tid] = h;
    const int mine = j < 0 ? -1 : j / E4M3_TILE, before = __shfl_up(mine, 1);
    const uint64_t begins = __ballot(mine >= 0 && (tid == 0 || mine != before));
    const int slot = __popcll(begins & (~0ull >> (63 - tid))) - 1;
    at_slot[tid] = j < 0 ? -1 : slot;
    if (begins >> tid & 1ull) tile_of[slot] = e4m3_tile_at(a.pages, h, j % a.pages.page_size / E4M3_TILE);
    if (tid == 0) n_slots = __popcll(begins);
  }
  __syncthreads();
  if (tid < 2 * E4M3_TILE) {
    const int m = tid / E4M3_TILE, i = tid % E4M3_TILE;
    float top = 0.f;
    for (int e = 0; e < E4M3_BLOCK; ++e) top = fmaxf(top, scale[m][i / E4M3_BLOCK * E4M3_BLOCK + e]);
    ratio[m][i] = scale[m][i] * e4m3_inverse(top);
    if (i % E4M3_BLOCK == 0) (m ? a.pages.v_scale : a.pages.k_scale)[e4m3_scale_at(a.pages, to, in_page) + i / E4M3_BLOCK] = top;
  }
  // keys on their way
  u32x4_t keys[2 * VI];
#pragma unroll
  for (int i = 0; i < 2 * VI; ++i) {
    const int at = tid + 256 * i, r = at % E4M3_TILE, ch = at / E4M3_TILE, j = from[r];
    keys[i] = u32x4_t{0u, 0u, 0u, 0u};
    if (ch < hd / 16 && j >= 0)
      keys[i] = *reinterpret_cast<const u32x4_t*>(a.pages.k + e4m3_tile_at(a.pages, head_of[r], j % a.pages.page_size / E4M3_TILE) +
                                                  ch * 16 * E4M3_TILE + j % E4M3_TILE * 16);
  }
  // this thread's 16 positions (of quarter c) in the source
  const int c = tid % 4;
  int off[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int p = 16 * (i / 4) + 4 * c + i % 4, q = from[p] % E4M3_TILE;
    off[i] = from[p] < 0 ? -1 : at_slot[p] * (hd * MOVE_PITCH) + q % 16 / 4 * 16 + q / 16 * 4 + q % 4;
  }
  uint32_t w[2 * VI][4] = {};
  const int slots = n_slots;
  for (int s0 = 0; s0 < slots; s0 += a.at_once) {
    const int n = min(a.at_once, slots - s0);
    if (s0) __syncthreads();
    for (int i = tid; i < n * hd * 4; i += 256)
      *reinterpret_cast<u32x4_t*>(tiles + i / 4 * MOVE_PITCH + i % 4 * 16) =
          *reinterpret_cast<const u32x4_t*>(a.pages.v + tile_of[s0 + i / (hd * 4)] + i % (hd * 4) * 16);
    __syncthreads();
    const int lo = s0 * (hd * MOVE_PITCH), hi = lo + n * (hd * MOVE_PITCH);
#pragma unroll
    for (int k = 0; k < 2 * VI; ++k) {
      const int d = tid / 4 + 64 * k;
      if (d < hd)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (off[i] >= lo && off[i] < hi) w[k][i / 4] |= (uint32_t)tiles[off[i] - lo + d * MOVE_PITCH] << 8 * (i % 4);
    }
  }
  __syncthreads();
  uint8_t* kt = a.pages.k + e4m3_tile_at(a.pages, to, in_page);
#pragma unroll
  for (int i = 0; i < 2 * VI; ++i) {
    const int at = tid + 256 * i, r = at % E4M3_TILE, ch = at / E4M3_TILE;
    if (ch >= hd / 16) break;
    const float f = ratio[0][r];
    if (f != 1.f)
#pragma unroll
      for (int e = 0; e < 4; ++e) keys[i][e] = e4m3_rescale(keys[i][e], f, f, f, f);
    *reinterpret_cast<u32x4_t*>(kt + ch * 16 * E4M3_TILE + r * 16) = keys[i];
  }
  uint8_t* vt = a.pages.v + e4m3_tile_at(a.pages, to, in_page);
#pragma unroll
  for (int k = 0; k < 2 * VI; ++k) {
    const int d = tid / 4 + 64 * k;
    if (d >= hd) break;
    u32x4_t o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* f = ratio[1] + 16 * j + 4 * c;
      o[j] = e4m3_rescale(w[k][j], f[0], f[1], f[2], f[3]);
    }
    *reinterpret_cast<u32x4_t*>(vt + d * E4M3_TILE + 16 * c) = o;
  }
}

// Fills the pages of the table's rows dst[b] with the positions kept[b][layer, kv head] of its rows src[b], whose pages are others.
// Whole pages are written: ceil(keep / page_size) of them.
TQ_API int tq_e4m3_move(const int* src, const int* dst, int B, const int* kept, int keep, int hd, void* k, void* v, float* k_scale,
                        float* v_scale, float* weight, const int* table, int slots_of_table, int bt_stride, int page_size, int heads,
                        hipStream_t st) {
  if (B <= 0) return 0;
  if (keep < 1) return TQ_ERR_BAD_ARG;
  if (!e4m3_pages_fit(page_size, heads, 0, 1, hd) || keep > (int64_t)bt_stride * page_size) return TQ_ERR_UNSUPPORTED;
  E4m3Move a{src, dst, kept, keep, slots_of_table, (keep + page_size - 1) / page_size * (page_size / E4M3_TILE), 1,
             E4m3Pages{(uint8_t*)k, (uint8_t*)v, k_scale, v_scale, weight, table, bt_stride, page_size, heads, 0, hd}};
  const int64_t groups = (int64_t)a.tiles * heads * B;
  if (groups > 0xFFFFFF) return TQ_ERR_UNSUPPORTED;      // (a launch's threads are counted in 32 bits)
  // Many workgroups hide one another's waiting, the more the less memory each takes (us of the move above with one, two and three tiles:
  // 532, 567, 654); few of them wait less often with more tiles (96 of them, one sequence: 9.6, 8.3, 7.9).
  if (groups <= 2048) a.at_once = 3;
  const size_t shmem = (size_t)a.at_once * hd * MOVE_PITCH;      // at most 60 KiB
  if (hd <= 128) hipLaunchKernelGGL(e4m3_move_kernel<1>, dim3((unsigned)groups), dim3(256), shmem, st, a);
  else hipLaunchKernelGGL(e4m3_move_kernel<2>, dim3((unsigned)groups), dim3(256), shmem, st, a);
  TQ_LAUNCH_CHECK();
  return 0;
}
