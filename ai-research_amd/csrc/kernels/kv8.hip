// kv8.hip -- the paged 8-bit K/V cache: append (per-head RMSNorm, rotary
// positions, quantization, cache write), read-back, and attention, for gfx950.
//
// A page holds page_tokens tokens of every kv head; 16 tokens of a head are a
// block with one scale for its keys and one for its values, a power of two
// 2^e with the least e for which the block's largest magnitude is <= 127 2^e.
// Powers of two because a block's scale grows as tokens are appended to it: the
// codes already there are then shifted (one more rounding, of at most half a
// step), a value code * 2^e is exact in every float type, and the scales enter
// products without a rounding.  They cost up to one of the 8 bits.
//
// Codes lie as the matrix instructions take them:
//   K block [D / 16][16 tokens][16 dims]: a lane's 16 bytes are the A operand of
//     v_mfma_i32_16x16x64_i8 (row = token, 16 dims of the sum) as loaded;
//   V block [4 groups][D][4 tokens]: a lane's 16 bytes are 4 tokens of 4 dims;
//     the sum of the second product runs over tokens, in a lane.
// Either way a wave's load is 1 KB in a row.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../common/kv8_args.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

namespace {

// (uniform to the compiler too)
__device__ __forceinline__ uint32_t wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// First row and number of rows of sequence s, whatever seq_start holds.
__device__ __forceinline__ uint32_t seq_rows(const Kv8Rows& b, uint32_t s, uint32_t* first) {
  const uint32_t r0 = min(b.seq_start[s], b.num_rows), r1 = min(b.seq_start[s + 1], b.num_rows);
  *first = r0;
  return r1 > r0 ? min(r1 - r0, b.max_rows) : 0u;
}

// The page of block `blk` of sequence s, or num_pages where there is none (past
// the table's end, or an entry that names no page).
__device__ __forceinline__ uint32_t page_of(const Kv8View& c, const Kv8Rows& b, uint32_t s, uint64_t blk) {
  const uint64_t i = blk >> (c.page_shift - 4);
  if (i >= b.max_pages) return c.num_pages;
  return min(b.pages[(uint64_t)s * b.max_pages + i], c.num_pages);
}

// Index of (page, head, block) among the cache's blocks (the host refuses 2^32).
__device__ __forceinline__ uint32_t block_at(const Kv8View& c, uint32_t page, uint32_t head, uint64_t blk) {
  const uint32_t sh = c.page_shift - 4;
  return ((page * c.nkv + head) << sh) + ((uint32_t)blk & ((1u << sh) - 1u));
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const double u = __shfl_xor(v, off, 64);
    v = u > v ? u : v;
  }
  return v;
}

// The wave's sums of N values (a power of two) at once: lane l gets that of value l
// mod N.  While there are several, lanes exchange halves of them.
template <int N, typename T>
__device__ __forceinline__ T wave_sums(T (&v)[N]) {
  const uint32_t lane = threadIdx.x & 63;
  int bit = 1;
#pragma unroll
  for (int n = N; n > 1; n >>= 1, bit <<= 1) {
#pragma unroll
    for (int i = 0; i < n / 2; i++) {
      const bool odd = lane & bit;
      const T keep = odd ? v[2 * i + 1] : v[2 * i], give = odd ? v[2 * i] : v[2 * i + 1];
      v[i] = keep + __shfl_xor(give, bit, 64);
    }
  }
#pragma unroll
  for (int off = N; off < 64; off <<= 1) v[0] += __shfl_xor(v[0], off, 64);
  return v[0];
}

// Lane l's value, in every lane.
__device__ __forceinline__ float lane_value(float v, int l) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), l));
}
__device__ __forceinline__ double lane_value(double v, int l) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), l);
  return __longlong_as_double((long long)(lo | hi << 32));
}

// v^-1/2 to an ulp or two: the instruction's estimate and two steps of Newton's.
__device__ __forceinline__ double inverse_root(double v) {
  double y = __builtin_amdgcn_rsq(v);
#pragma unroll
  for (int i = 0; i < 2; i++) y = fma(y * 0.5, fma(-(v * y), y, 1.0), y);
  return y;
}

// Dims of pair i < D / 2 of a head: (i, i + rot / 2) for the rotated ones, the
// others' halves after them.
__device__ __forceinline__ void pair_dims(uint32_t i, uint32_t D, uint32_t rot, uint32_t* d0, uint32_t* d1) {
  const uint32_t half = rot / 2;
  *d0 = i < half ? i : rot + (i - half);
  *d1 = *d0 + (i < half ? half : (D - rot) / 2);
}

// ---------------------------------------------------------------------------
// Append.  A workgroup takes 16 token places of a sequence (one block) and one
// key head, one value head or KV8_Q_HEADS query heads, one a wave.  A code is
// decided next to a rounding border, so keys and values are computed in 64 bits, and
// the codes do not depend on the order of any 32-bit sum.  Angles in 64 bits too, for positions
// far out: two sines and cosines per pair and a run of rows, the rows between by
// rotating on.  What a workgroup waits for is on its way before it computes the
// angles: the whole of its rows, and the codes already there.  (2000 rows of 16 query
// and 8 key heads of 256: 34 us, 3.1 TB/s; the vector units are busy for 58% of it, and
// the waves, four a SIMD, wait for 54%.  Every head's workgroup works out the angles of its
// block anew.  One row: 5 us.)
// ---------------------------------------------------------------------------
struct Angle {
  double c, s;
};

// Half turns a token of pair i: theta^(-2 i / rot) / pi to an ulp or two, 2^x with x =
// i * (-2 log2(theta) / rot) as the sum of two.
__device__ __forceinline__ double half_turns(uint32_t i, const Kv8AppendArgs& a) {
  const double x = (double)i * a.log_hi, x_lo = fma((double)i, a.log_hi, -x) + (double)i * a.log_lo;
  const double f = exp2(x) * 0.3183098861837907;
  return fma(f, x_lo * 0.6931471805599453, f);
}

// The angle of g half turns a token at position pos (the whole turns go first, without
// a rounding).
__device__ __forceinline__ Angle angle(double pos, double g) {
  const double t = pos * g, lo = fma(pos, g, -t);
  Angle r;
  sincospi((t - 2.0 * rint(t * 0.5)) + lo, &r.s, &r.c);
  return r;
}

// ang[row][pair] for rows [0, nr) at positions pos0 + row.
__device__ __forceinline__ void block_angles(Angle* ang, uint64_t pos0, uint32_t nr, const Kv8AppendArgs& a) {
  const uint32_t half = a.rot / 2;
  if (half == 0) return;
  const uint32_t teams = nr > 1 && 256u / half > 1 ? min(256u / half, nr) : 1u;
  const uint32_t per = (nr + teams - 1) / teams;
  for (uint32_t t = threadIdx.x; t < half * teams; t += 256) {
    const uint32_t i = t % half, r0 = (t / half) * per, r1 = min(r0 + per, nr);
    if (r0 >= r1) continue;
    const double f = half_turns(i, a);
    Angle g = angle((double)(pos0 + r0), f), st{1.0, 0.0};
    if (r1 - r0 > 1) st = angle(1.0, f);
    for (uint32_t r = r0; r < r1; r++) {
      ang[r * half + i] = g;
      g = Angle{g.c * st.c - g.s * st.s, g.c * st.s + g.s * st.c};
    }
  }
}

// A row's elements of a lane's pairs: loads, and their dims.
template <int NP>
__device__ __forceinline__ void load_pairs(const float* in, uint32_t D, uint32_t rot, float (&x0)[NP], float (&x1)[NP]) {
#pragma unroll
  for (int m = 0; m < NP; m++) {
    const uint32_t i = (threadIdx.x & 63) + 64 * m;
    x0[m] = x1[m] = 0.f;
    if (i < D / 2) {
      uint32_t d0, d1;
      pair_dims(i, D, rot, &d0, &d1);
      x0[m] = in[d0];
      x1[m] = in[d1];
    }
  }
}

// Query heads: a wave a head, a few of its rows of the block at a time.
template <int NP>
__device__ __forceinline__ void append_q(const Kv8AppendArgs& a, Angle* ang, uint64_t pos0, uint32_t row0, uint32_t nr,
                                         uint32_t group) {
  constexpr int R = NP == 4 ? 4 : 8;
  const uint32_t lane = threadIdx.x & 63, h = group * KV8_Q_HEADS + wave_id();
  const uint32_t D = a.c.D, half = a.rot / 2;
  const bool mine = h < a.nq;
  const float* in = a.q + (uint64_t)row0 * a.qs + (uint64_t)h * D;
  float* out = a.qo + (uint64_t)row0 * a.nq * D + (uint64_t)h * D;
  float x0[R][NP], x1[R][NP];
  const auto load = [&](uint32_t first) {
#pragma unroll
    for (int j = 0; j < R; j++)
      if (mine && first + j < nr) load_pairs<NP>(in + (uint64_t)(first + j) * a.qs, D, a.rot, x0[j], x1[j]);
  };
  load(0);
  block_angles(ang, pos0, nr, a);
  __syncthreads();
  for (uint32_t first = 0; first < nr; first += R) {
    float ss[R];
#pragma unroll
    for (int j = 0; j < R; j++) {
      ss[j] = 0.f;
      if (!mine || first + j >= nr) continue;
#pragma unroll
      for (int m = 0; m < NP; m++) ss[j] += x0[j][m] * x0[j][m] + x1[j][m] * x1[j][m];
    }
    // of row first + lane mod R (once a row: in 64 bits, with one rounding)
    const float root = (float)inverse_root((double)wave_sums<R>(ss) / (double)D + (double)a.eps);
#pragma unroll
    for (int j = 0; j < R; j++) {
      const uint32_t r = first + j;
      if (!mine || r >= nr) continue;
      __builtin_amdgcn_sched_barrier(0);  // (a row's angles and norms at a time in registers)
      const float inv = lane_value(root, j);
#pragma unroll
      for (int m = 0; m < NP; m++) {
        const uint32_t i = lane + 64 * m;
        if (i >= D / 2) continue;
        uint32_t d0, d1;
        pair_dims(i, D, a.rot, &d0, &d1);
        const float u = x0[j][m] * inv * a.qn[d0], w = x1[j][m] * inv * a.qn[d1];
        float c = 1.f, s = 0.f;
        if (i < half) {
          c = (float)ang[r * half + i].c;
          s = (float)ang[r * half + i].s;
        }
        out[(uint64_t)r * a.nq * D + d0] = u * c - w * s;
        out[(uint64_t)r * a.nq * D + d1] = u * s + w * c;
      }
    }
    load(first + R);
  }
}

// Places of a block's element (token, dim) and 16-byte pieces.
__device__ __forceinline__ uint32_t k_place(uint32_t t, uint32_t d) { return (d >> 4) * 256 + t * 16 + (d & 15); }
__device__ __forceinline__ uint32_t v_place(uint32_t t, uint32_t d, uint32_t D) { return (t >> 2) * 4 * D + d * 4 + (t & 3); }

template <int NP, bool IS_K>
__device__ __forceinline__ void append_kv(const Kv8AppendArgs& a, Angle* ang, int8_t* tile, double* red, uint64_t pos0,
                                          uint32_t row0, uint32_t o0, uint32_t nr, uint32_t head, uint32_t at) {
  const uint32_t lane = threadIdx.x & 63, wave = wave_id();
  const uint32_t D = a.c.D, half = a.rot / 2, o1 = o0 + nr;
  int8_t* codes = (IS_K ? a.c.k : a.c.v) + (uint64_t)at * (KV8_BLOCK * D);
  float* scale = (IS_K ? a.c.ks : a.c.vs) + at;
  const float* src = (IS_K || a.k_eq_v ? a.k : a.v) + (uint64_t)head * D;
  // wave w: token places 4 w .. 4 w + 3 of the block
  float f0[4][NP], f1[4][NP];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t t = wave * 4 + j;
    if (t >= o0 && t < o1) load_pairs<NP>(src + (uint64_t)(row0 + t - o0) * a.kvs, D, a.rot, f0[j], f1[j]);
  }
  const float old = o0 > 0 ? *scale : 0.f;
  // the codes already there (a fresh block's places without a token become 0)
  int4* t4 = reinterpret_cast<int4*>(tile);
  for (uint32_t i = threadIdx.x; i < D; i += 256) t4[i] = o0 > 0 ? reinterpret_cast<const int4*>(codes)[i] : int4{0, 0, 0, 0};
  if (IS_K) {
    block_angles(ang, pos0, nr, a);
    __syncthreads();
  }

  double x0[4][NP], x1[4][NP], ss[4], amax = 0.0, odd = 0.0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t t = wave * 4 + j;
    ss[j] = 0.0;
    if (t < o0 || t >= o1) continue;
#pragma unroll
    for (int m = 0; m < NP; m++) {
      x0[j][m] = (double)f0[j][m];
      x1[j][m] = (double)f1[j][m];
      ss[j] += x0[j][m] * x0[j][m] + x1[j][m] * x1[j][m];
    }
  }
  const double root = inverse_root(wave_sums<4>(ss) / (double)D + (double)a.eps);  // of place 4 wave + lane mod 4
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t t = wave * 4 + j;
    if (t < o0 || t >= o1) continue;
    __builtin_amdgcn_sched_barrier(0);  // (as above)
    const double inv = lane_value(root, j);
#pragma unroll
    for (int m = 0; m < NP; m++) {
      const uint32_t i = lane + 64 * m;
      if (i >= D / 2) continue;
      double u = x0[j][m] * inv, w = x1[j][m] * inv;
      if (IS_K) {
        uint32_t d0, d1;
        pair_dims(i, D, a.rot, &d0, &d1);
        u *= (double)a.kn[d0];
        w *= (double)a.kn[d1];
        if (i < half) {
          const Angle g = ang[(t - o0) * half + i];
          const double y = u * g.c - w * g.s;
          w = u * g.s + w * g.c;
          u = y;
        }
      }
      x0[j][m] = u;
      x1[j][m] = w;
      amax = fmax(amax, fmax(fabs(u), fabs(w)));
      odd = fma(u, 0.0, fma(w, 0.0, odd));  // NaN once there is a NaN or an infinity
    }
  }
  amax = wave_max(amax);
  if (__any(odd != odd)) amax = HUGE_VAL;
  if (lane == 0) red[wave] = amax;
  __syncthreads();
  amax = fmax(fmax(red[0], red[1]), fmax(red[2], red[3]));

  // least e with amax <= 127 2^e (127 = 0.9921875 * 2^7), not below f32's normal range
  float fresh = 0.f;
  if (amax > 0.0) {
    int e;
    const double m = frexp(amax, &e);
    fresh = amax < HUGE_VAL ? (float)ldexp(1.0, max(m <= 0.9921875 ? e - 7 : e - 6, -126)) : __builtin_nanf("");
  }
  const float now = old != old || fresh != fresh ? __builtin_nanf("") : fmaxf(old, fresh);
  const bool grown = o0 > 0 && now > old;
  if (grown) {  // shift the codes already there
    const float by = old / now;
    for (uint32_t i = threadIdx.x; i < o0 * D; i += 256) {
      const uint32_t t = i / D, d = i - t * D, p = IS_K ? k_place(t, d) : v_place(t, d, D);
      tile[p] = (int8_t)(int)rintf((float)tile[p] * by);
    }
  }
  const double inv = now > 0.f ? 1.0 / (double)now : 0.0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t t = wave * 4 + j;
    if (t < o0 || t >= o1) continue;
#pragma unroll
    for (int m = 0; m < NP; m++) {
      const uint32_t i = lane + 64 * m;
      if (i >= D / 2) continue;
      uint32_t d0, d1;
      pair_dims(i, D, a.rot, &d0, &d1);
      // (at most 127 in magnitude; a NaN becomes 0)
      tile[IS_K ? k_place(t, d0) : v_place(t, d0, D)] = (int8_t)(int)rint(x0[j][m] * inv);
      tile[IS_K ? k_place(t, d1) : v_place(t, d1, D)] = (int8_t)(int)rint(x1[j][m] * inv);
    }
  }
  __syncthreads();
  // pieces of 16 bytes: of one token (K), of the four tokens of a group (V)
  const uint32_t lo = grown ? 0u : o0;
  for (uint32_t i = threadIdx.x; i < D; i += 256) {
    const uint32_t t = IS_K ? i & 15 : (i / (D / 4)) * 4;
    const bool out = IS_K ? t >= lo && t < o1 : t + 3 >= lo && t < o1;
    if (out) reinterpret_cast<int4*>(codes)[i] = t4[i];
  }
  if (threadIdx.x == 0 && !(now == old && o0 > 0)) *scale = now;
}

// grid (2 nkv + query groups, blocks a sequence's rows can touch, sequences)
template <int NP>
__device__ __forceinline__ void append(const Kv8AppendArgs& a) {
  extern __shared__ char lds[];
  const uint32_t seq = blockIdx.z, unit = blockIdx.x;
  uint32_t first;
  const uint32_t rows = seq_rows(a.b, seq, &first);
  const uint64_t past = a.b.past[seq], blk = past / KV8_BLOCK + blockIdx.y;
  const uint64_t p0 = max(past, blk * KV8_BLOCK), p1 = min(past + rows, (blk + 1) * KV8_BLOCK);
  if (p0 >= p1) return;
  const uint32_t nr = (uint32_t)(p1 - p0), row0 = first + (uint32_t)(p0 - past), nkv = a.c.nkv;
  double* red = reinterpret_cast<double*>(lds);
  int8_t* tile = reinterpret_cast<int8_t*>(lds + 32);
  Angle* ang = reinterpret_cast<Angle*>(lds + 32 + KV8_BLOCK * a.c.D);
  if (unit < 2 * nkv) {
    const uint32_t head = unit >> 1, page = page_of(a.c, a.b, seq, blk);
    if (page >= a.c.num_pages) return;  // no page: nothing is kept
    const uint32_t at = block_at(a.c, page, head, blk);
    const uint32_t o0 = (uint32_t)(p0 - blk * KV8_BLOCK);
    if (unit & 1) {
      append_kv<NP, false>(a, ang, tile, red, p0, row0, o0, nr, head, at);
    } else {
      append_kv<NP, true>(a, ang, tile, red, p0, row0, o0, nr, head, at);
    }
  } else {
    append_q<NP>(a, ang, p0, row0, nr, unit - 2 * nkv);
  }
}

// ---------------------------------------------------------------------------
// Attention.  A workgroup takes 16 query columns (consecutive rows times the
// query heads of one kv head) and a share of their tokens; its four waves take
// the share's steps of 32 tokens in turn, each with its own running maximum
// and sum, and are joined through LDS.
//
//   S^T (tokens x columns) = K . Q^T    v_mfma_i32_16x16x64_i8: the codes as they
//       lie, Q as four signed base-256 digits of a 31-bit fixed-point number per
//       row (the digit sums are exact; 31 bits keep what the f32 row has)
//   O^T (dims x columns) += V^T . P^T   v_mfma_f32_16x16x32_f16: the codes as f16
//       (exact), P times the block's scale as two f16 halves (22 bits)
//
// S^T leaves a lane the scores of tokens 4 g .. 4 g + 3 (g = lane / 16) of both
// 16-token blocks of a step for its column, which is the B operand of the
// second product: P needs no exchange between lanes.
// P's halves hold the column's weights p 2^e (e its block's scale exponent) in units
// that follow the largest of them so far, which is over 2^14 units (2^10 in the kernel of
// many columns) and at most 2^15: half a step of the lower half, 2^-25 units, may be lost of
// each.  Blocks that a column does not see, or sees with little weight, do not move its
// unit, whatever their scales are.
// ---------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -3.402823466e38f;  // maximum and unit of a column that has seen nothing
constexpr float kNoUnit = -100000.f;
constexpr int kTop = 15;  // the largest weight is at most 2^kTop units
constexpr int kLazy = 4;  // of the kernel of many columns

__device__ __forceinline__ f16x8 codes_f16(uint32_t a, uint32_t b) {
  // byte ^ 0x80 under the exponent of 1024 is 1152 + code
  a ^= 0x80808080u;
  b ^= 0x80808080u;
  union {
    uint32_t w[4];
    f16x2 h[4];
    f16x8 v;
  } u;
  u.w[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
  u.w[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
  u.w[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
  u.w[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
  const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
  for (int i = 0; i < 4; i++) u.h[i] = u.h[i] - off;
  return u.v;
}

// a tile of columns of one kv head of a sequence, and its token range
struct Tile {
  uint32_t seq, head, first, rows, col0, ncol;
  uint64_t past, lo, hi;  // tokens [lo, hi) are visible to one of its columns
  uint32_t step0, steps;  // steps of 32 tokens that hold them
  uint32_t all0, all1;    // steps [all0, all1): every token visible to every column, where there is a page
};

// false: the tile has no row
__device__ __forceinline__ bool tile_of(const Kv8AttnArgs& a, uint32_t seq, uint32_t head, uint32_t tile, uint32_t width,
                                        Tile* t) {
  const uint32_t G = a.nq / a.c.nkv;
  t->rows = seq_rows(a.b, seq, &t->first);
  t->seq = seq;
  t->head = head;
  t->col0 = tile * width;
  const uint64_t cols = (uint64_t)t->rows * G;
  if (t->col0 >= cols) return false;
  t->ncol = (uint32_t)min((uint64_t)width, cols - t->col0);
  t->past = a.b.past[seq];
  const uint64_t p0 = t->past + t->col0 / G, p1 = t->past + (t->col0 + t->ncol - 1) / G;
  const uint64_t lo = a.window && p0 + 1 > a.window ? p0 + 1 - a.window : 0;
  const uint64_t held = (uint64_t)a.b.max_pages << a.c.page_shift;  // tokens the table can name
  const uint64_t hi = min(p1 + 1, held);
  t->lo = lo;
  t->hi = hi;
  t->all0 = a.window && p1 + 1 > a.window ? (uint32_t)((p1 + KV8_STEP - a.window) / KV8_STEP) : 0;
  t->all1 = (uint32_t)((p0 + 1) / KV8_STEP);
  t->step0 = (uint32_t)(lo / KV8_STEP);
  t->steps = hi > lo ? (uint32_t)((hi + KV8_STEP - 1) / KV8_STEP) - t->step0 : 0u;
  return true;
}

// A step's codes of keys or values in registers, with its scales.
template <int NL>
struct Codes {
  i32x4 c[2][NL];
  float s[2];
  bool has[2];
};

// The pages of 32 steps (s, s + stride, ...), two blocks each, in a wave's lanes.
__device__ __forceinline__ uint32_t step_pages(const Kv8AttnArgs& a, const Tile& t, uint32_t s, uint32_t stride) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t blk = 2 * ((uint64_t)s + stride * (lane >> 1)) + (lane & 1);
  // a block that no column sees may hold anything, scales too
  const bool some = blk * KV8_BLOCK < t.hi && (blk + 1) * KV8_BLOCK > t.lo;
  return some ? page_of(a.c, a.b, t.seq, blk) : a.c.num_pages;
}

// A lane's 16-byte piece of a block: 16 dims of a token (K), 4 tokens of 4 dims (V),
// dims 64 l ...  FULL: the head has 64 dims for every l; else pieces of dims it does
// not have are read from the block's first ones, and meet zeros of Q or are not
// written.
template <bool FULL, bool IS_K>
__device__ __forceinline__ uint32_t piece_at(uint32_t l, uint32_t D) {
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  if (IS_K) return FULL || 64 * l + 16 * g < D ? l * 1024 + lane * 16 : n * 16;
  return FULL || 64 * l + 4 * n < D ? g * 4 * D + l * 256 + n * 16 : 0;
}

// STREAM: nothing is read again, and the codes pass by the caches.
template <int NL, bool FULL, bool STREAM, bool IS_K>
__device__ __forceinline__ void load_codes(const Kv8AttnArgs& a, const Tile& t, uint32_t step, uint32_t pages, uint32_t i,
                                           Codes<NL>* s) {
  const uint32_t D = FULL ? 64 * NL : a.c.D;
#pragma unroll
  for (int b = 0; b < 2; b++) {
    const uint64_t blk = (uint64_t)step * 2 + b;
    const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)pages, (int)(2 * i + b));
    s->has[b] = page < a.c.num_pages;
    const uint32_t at = block_at(a.c, s->has[b] ? page : 0, t.head, blk);
    s->s[b] = (IS_K ? a.c.ks : a.c.vs)[at];
    const int8_t* c = (IS_K ? a.c.k : a.c.v) + (uint64_t)at * (KV8_BLOCK * D);
#pragma unroll
    for (int l = 0; l < NL; l++) {
      const i32x4* p = reinterpret_cast<const i32x4*>(c + piece_at<FULL, IS_K>(l, D));
      s->c[b][l] = STREAM ? __builtin_nontemporal_load(p) : *p;
    }
  }
}

// A column's running softmax: m is what is subtracted from its scores, l their sum, and o
// the sums of weights 2^(s - m + e) times codes, in units of 2^(E - kTop + LAZY); unit is
// one over that (0: no weight yet; infinite where f32 does not hold it).  m and E are whole
// numbers, so that their changes turn the sums by powers of two.
template <int NL>
struct Run {
  f32x4 o[NL][4];
  float m, l, E, unit;
};

template <int NL>
__device__ __forceinline__ void clear(Run<NL>* r) {
#pragma unroll
  for (int l = 0; l < NL; l++)
#pragma unroll
    for (int j = 0; j < 4; j++) r->o[l][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  r->m = kNoMax;
  r->l = 0.f;
  r->E = kNoUnit;
  r->unit = 0.f;
}

// The four digit sums of a score.  Two at a time are exact as integers (at most
// 257 * 128 * 127 * 512 < 2^31).
__device__ __forceinline__ float digit_sum(int d3, int d2, int d1, int d0) {
  return fmaf((float)((d3 << 8) + d2), 65536.f, (float)((d1 << 8) + d0));
}

// Over the four lanes of a column (lane, lane ^ 16, ^ 32, ^ 48).
__device__ __forceinline__ float column_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Two numbers as f16, to nearest.
__device__ __forceinline__ f16x2 half2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_convertvector((f32x2{a, b}), f16x2);
}

// Whether a block's scale is a number (uniform).
__device__ __forceinline__ bool scale_number(float v) {
  return (uint32_t)__builtin_amdgcn_readfirstlane(__float_as_uint(v)) < 0x7f800000u;
}

// The softmax of a step's scores sc, in units of log2 (-inf: not seen): the halves
// of P for the second product, and the running values.  vs: the blocks' scales of V.
// What is subtracted from the scores follows their maximum, and the unit the largest
// weight, when those are over them by more than LAZY, so P is at most 2^LAZY (and its
// halves are in units that much larger): with 16 columns one or another has a new maximum
// in most steps of a prompt, and each costs a product for every sum.  (Prompts of 2000
// tokens: LAZY 4 108 us, 2 109, 1 and 0 112; what is lost is 2^-35 of the largest weight
// then, far below f32's 2^-24.)
template <int NL, int LAZY>
__device__ __forceinline__ void soft_step(const float (&sc)[2][4], const float (&vs)[2], const bool (&has)[2], Run<NL>* r,
                                          f16x8* phi, f16x8* plo) {
  float e[2], v[2], mx[2];  // the blocks' scales that count (0: none) and their exponents
#pragma unroll
  for (int b = 0; b < 2; b++) {
    const uint32_t bits = __builtin_amdgcn_readfirstlane(__float_as_uint(vs[b]));
    const bool some = has[b] && bits - 1u < 0x7f800000u - 1u;
    e[b] = some ? (float)((int)(bits >> 23) - 127) : -INFINITY;
    v[b] = some ? __uint_as_float(bits) : 0.f;
    mx[b] = fmaxf(fmaxf(sc[b][0], sc[b][1]), fmaxf(sc[b][2], sc[b][3]));
  }
  const float top = fmaxf(mx[0], mx[1]), most = fmaxf((mx[0] - r->m) + e[0], (mx[1] - r->m) + e[1]);
  if (__any(top > r->m + LAZY || most > r->E + LAZY)) {
    const float t = column_max(top), m = t > r->m + LAZY ? ceilf(t) : r->m;
    const float w = column_max(fmaxf((mx[0] - m) + e[0], (mx[1] - m) + e[1]));
    const float by = r->m - m, moved = fmaxf(r->E + by, kNoUnit), E = w > moved + LAZY ? ceilf(w) : moved;
    const float turn = __builtin_amdgcn_exp2f(by + (r->E - E));
    r->l *= __builtin_amdgcn_exp2f(by);
    r->m = m;
    r->E = E;
    r->unit = E == kNoUnit ? 0.f : ldexpf(1.f, kTop - LAZY - (int)E);
    if (__any(turn != 1.f)) {
#pragma unroll
      for (int l = 0; l < NL; l++)
#pragma unroll
        for (int j = 0; j < 4; j++) r->o[l][j] *= turn;
    }
  }
  float w[2][4], sum = 0.f;
  bool far = false;
#pragma unroll
  for (int b = 0; b < 2; b++) {
    const float mul = v[b] * r->unit;
    far |= !(mul <= 0x1p90f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float p = __builtin_amdgcn_exp2f(sc[b][i] - r->m);
      sum += p;
      w[b][i] = p * mul;
    }
  }
  // (a scale so far over the unit that only a p below f32's range makes a weight of it)
  if (__any(far)) {
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        w[b][i] = __builtin_amdgcn_exp2f((sc[b][i] - r->m) + (e[b] - r->E + (float)(kTop - LAZY)));
  }
  union {
    f16x2 h[4];
    f16x8 v;
  } hi, lo;
#pragma unroll
  for (int b = 0; b < 2; b++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float x = w[b][2 * i], y = w[b][2 * i + 1];
      const f16x2 h = half2(x, y);
      hi.h[2 * b + i] = h;
      lo.h[2 * b + i] = half2(x - (float)h[0], y - (float)h[1]);
    }
  r->l += sum;
  *phi = hi.v;
  *plo = lo.v;
}

// Whether the column at token pos sees token t.
__device__ __forceinline__ bool visible(int64_t t, int64_t pos, uint32_t window) {
  return t <= pos && (window == 0 || t > pos - (int64_t)window);
}

// The digit sums are used behind a branch: the compiler (ROCm 7.2) counts the eight
// wait states from a matrix instruction to a read of its result within a block,
// and put the read right behind the branch of one that ended with the products.
__device__ __forceinline__ void settle(i32x4 (&acc)[2][4]) {
  asm volatile("s_nop 7"
               : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[0][2]), "+v"(acc[0][3]), "+v"(acc[1][0]), "+v"(acc[1][1]),
                 "+v"(acc[1][2]), "+v"(acc[1][3]));
}

// What digit sums are multiplied with, but for their block's scale: a lane's column's unit and
// the constants, times 2^lift, which the scales are divided by.
struct Factor {
  float mul;
  int lift;
};

// Of digits in units of 2^e (odd: of a row with a NaN or an infinity).  Queries so small that their
// factor is below f32's range (x < -125) have scores that count only under scales far above 1, and
// lend that range to them, as far as the wave's largest queries can do without scales below
// 2^(lift - 126).  (The test for it costs prompts up to 1%.)
__device__ __forceinline__ Factor factor_of(int e, bool odd, float scale) {
  const float c = scale * kLog2e;
  const int x = e + (int)((__float_as_uint(c) >> 23) & 255u) - 127;
  Factor f{0.f, 0};
  if (__any(!odd && x < -125)) {
    int most = odd ? -1000 : x;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) most = max(most, __shfl_xor(most, off, 64));
    f.lift = __builtin_amdgcn_readfirstlane(min(80, max(0, 49 - most)));
  }
  f.mul = odd ? __builtin_nanf("") : ldexpf(c, e + f.lift);
  return f;
}

// Scores, in units of log2, from their digit sums; -inf: not seen.
__device__ __forceinline__ void finish_scores(const Kv8AttnArgs& a, i32x4 (&acc)[2][4], const float (&ks)[2],
                                              const float (&vs)[2], const bool (&has)[2], Factor f, const Tile& t,
                                              int64_t pos, uint32_t step, float (&sc)[2][4]) {
  const uint32_t g = (threadIdx.x & 63) >> 4;
  settle(acc);
  float by[2] = {ks[0], ks[1]};
  if (f.lift != 0) {
#pragma unroll
    for (int b = 0; b < 2; b++) by[b] = ldexpf(by[b], -f.lift);
  }
#pragma unroll
  for (int b = 0; b < 2; b++) {
    // (powers of two and the constant: one rounding, of the constant.  NaN where a scale of the
    // block is no number, so that what sees one of its tokens is NaN)
    const float mul = f.mul * (scale_number(vs[b]) ? by[b] : __builtin_nanf(""));
#pragma unroll
    for (int i = 0; i < 4; i++) sc[b][i] = digit_sum(acc[b][3][i], acc[b][2][i], acc[b][1][i], acc[b][0][i]) * mul;
  }
  // unless every token of the step is seen by every column
  if (!has[0] || !has[1] || step < t.all0 || step >= t.all1) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const int64_t t0 = (int64_t)step * KV8_STEP + b * KV8_BLOCK + 4 * g;
#pragma unroll
      for (int i = 0; i < 4; i++) sc[b][i] = has[b] && visible(t0 + i, pos, a.window) ? sc[b][i] : -INFINITY;
    }
  }
}

// Scores of a step's tokens 4 g .. of both blocks for a lane's column.
template <int NL>
__device__ __forceinline__ void score_step(const Kv8AttnArgs& a, const Codes<NL>& k, const float (&vs)[2], const i32x4* qd,
                                           Factor f, const Tile& t, int64_t pos, uint32_t step, float (&sc)[2][4]) {
  const uint32_t lane = threadIdx.x & 63;
  i32x4 acc[2][4];
  asm volatile("" ::: "memory");  // the digits are read in every step, not held
#pragma unroll
  for (int d = 0; d < 4; d++) acc[0][d] = acc[1][d] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int l = 0; l < NL; l++) {
#pragma unroll
    for (int d = 0; d < 4; d++) {
      const i32x4 q = qd[(d * NL + l) * 64 + lane];
      acc[0][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k.c[0][l], q, acc[0][d], 0, 0, 0);
      acc[1][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k.c[1][l], q, acc[1][d], 0, 0, 0);
    }
  }
  finish_scores(a, acc, k.s, vs, k.has, f, t, pos, step, sc);
}

template <int NL>
__device__ __forceinline__ void value_step(const Codes<NL>& v, f16x8 hi, f16x8 lo, Run<NL>* r) {
#pragma unroll
  for (int l = 0; l < NL; l++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const f16x8 x = codes_f16((uint32_t)v.c[0][l][j], (uint32_t)v.c[1][l][j]);
      r->o[l][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, hi, r->o[l][j], 0, 0, 0);
      r->o[l][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, lo, r->o[l][j], 0, 0, 0);
    }
}

// The address of a column's row of one head.
__device__ __forceinline__ uint64_t row_at(const Kv8AttnArgs& a, const Tile& t, uint32_t col) {
  const uint32_t G = a.nq / a.c.nkv;
  return ((uint64_t)(t.first + col / G) * a.nq + (uint64_t)t.head * G + col % G) * a.c.D;
}

// Signed base-256 digits of four 31-bit numbers, digit by digit: digit d of v is
// byte d of (v + 0x80808080) ^ 0x80808080.
__device__ __forceinline__ void digits4(const int (&v)[4], int (&w)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; i++) u[i] = ((uint32_t)v[i] + 0x80808080u) ^ 0x80808080u;
  // bytes of u[0], u[1] in turn, then of all four
  const uint32_t a0 = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), a1 = __builtin_amdgcn_perm(u[1], u[0], 0x07030602u);
  const uint32_t b0 = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u), b1 = __builtin_amdgcn_perm(u[3], u[2], 0x07030602u);
  w[0] = (int)__builtin_amdgcn_perm(b0, a0, 0x05040100u);
  w[1] = (int)__builtin_amdgcn_perm(b0, a0, 0x07060302u);
  w[2] = (int)__builtin_amdgcn_perm(b1, a1, 0x05040100u);
  w[3] = (int)__builtin_amdgcn_perm(b1, a1, 0x07060302u);
}

// A lane's part of its column's query row (dims 64 l + 16 g ..) as digits; the row's
// largest magnitude decides their unit.
template <int NL>
__device__ __forceinline__ Factor load_q(const Kv8AttnArgs& a, const float* q, i32x4 (&qd)[4][NL]) {
  const uint32_t g = (threadIdx.x & 63) >> 4, D = a.c.D;
  f32x4 x[NL][4];
  float amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int l = 0; l < NL; l++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[l][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (64 * l + 16 * g < D) x[l][j] = *reinterpret_cast<const f32x4*>(q + 64 * l + 16 * g + 4 * j);
    }
#pragma unroll
  for (int l = 0; l < NL; l++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        amax = fmaxf(amax, fabsf(x[l][j][i]));
        bad |= !(fabsf(x[l][j][i]) < INFINITY);
      }
  if (bad) amax = INFINITY;
  amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
  amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
  bad = amax == INFINITY;
  int e = 0;
  if (!bad) frexpf(amax, &e);
#pragma unroll
  for (int l = 0; l < NL; l++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      int v[4], w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = bad ? 0 : (int)rintf(ldexpf(x[l][j][i], 30 - e));
      digits4(v, w);
#pragma unroll
      for (int d = 0; d < 4; d++) qd[d][l][j] = w[d];
    }
  return factor_of(e - 30, bad, a.scale);
}

// A wave's part of the query row q (dims 64 l + 16 g .. for every fourth l).
template <int NL>
__device__ __forceinline__ void load_row(const float* q, uint32_t D, f32x4 (&x)[(NL + 3) / 4][4]) {
  const uint32_t g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < (NL + 3) / 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t d = 64 * (wave_id() + 4 * i) + 16 * g + 4 * j;
      x[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (d < D) x[i][j] = *reinterpret_cast<const f32x4*>(q + d);
    }
}

// The tile's query columns as digits in LDS, qd[digit][l][lane] (dims 64 l + 16 g
// .. of column n); a wave makes every fourth l.  A row's largest magnitude (joined
// through qm) decides its unit.
template <int NL>
__device__ __forceinline__ Factor stage_q(const Kv8AttnArgs& a, const f32x4 (&x)[(NL + 3) / 4][4], float* qm, i32x4* qd) {
  constexpr int NS = (NL + 3) / 4;
  const uint32_t lane = threadIdx.x & 63, wave = wave_id(), n = lane & 15;
  float amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < NS; i++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
        amax = fmaxf(amax, fabsf(x[i][j][c]));
        bad |= !(fabsf(x[i][j][c]) < INFINITY);
      }
  if (bad) amax = INFINITY;
  amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
  amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
  if (lane < 16) qm[wave * 16 + n] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; w++) amax = fmaxf(amax, qm[w * 16 + n]);
  bad = amax == INFINITY;
  int e = 0;
  if (!bad) frexpf(amax, &e);
#pragma unroll
  for (int i = 0; i < NS; i++) {
    const uint32_t l = wave + 4 * i;
    if (l >= NL) continue;
    i32x4 w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      int v[4], u[4];
#pragma unroll
      for (int c = 0; c < 4; c++) v[c] = bad ? 0 : (int)rintf(ldexpf(x[i][j][c], 30 - e));
      digits4(v, u);
#pragma unroll
      for (int d = 0; d < 4; d++) w[d][j] = u[d];
    }
#pragma unroll
    for (int d = 0; d < 4; d++) qd[(d * NL + l) * 64 + lane] = w[d];
  }
  __syncthreads();
  return factor_of(e - 30, bad, a.scale);
}

// A lane's sums of its column (dims d0 + 16 g + 4 i .. for each i), times by 2^n (in that
// order: a result below f32's normal range is rounded once).
__device__ __forceinline__ void write_dims(const f32x4 (&o)[4], float* to, uint32_t d0, uint32_t D, float by, int n) {
  const uint32_t g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t d = d0 + 16 * g + 4 * i;
    f32x4 x;
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = ldexpf(o[j][i] * by, n);
    if (d < D) *reinterpret_cast<f32x4*>(to + d) = x;
  }
}

// Few query columns (one tile): the workgroup's waves take its steps in turn.  The
// tokens' bytes bound it, so a wave has the next step's keys on the way while it
// weighs this step's values, and the next values while it scores; the query
// digits are in LDS to leave the registers to them.  (Heads of 256 over 8 key heads: 32
// rows over 20 - 4000 tokens 55 us, 4.8 TB/s of codes; one row over 120000 80 us, 6.2.)
// grid (tiles * splits, kv heads, sequences)
template <int NL, bool FULL, bool STREAM>
__device__ __forceinline__ void attend(const Kv8AttnArgs& a) {
  extern __shared__ __align__(16) char lds[];
  const uint32_t lane = threadIdx.x & 63, wave = wave_id(), n = lane & 15, g = lane >> 4;
  const uint32_t D = a.c.D, G = a.nq / a.c.nkv;
  const uint32_t split = blockIdx.x % a.nsplit, tile = blockIdx.x / a.nsplit;
  Tile t;
  if (!tile_of(a, blockIdx.z, blockIdx.y, tile, KV8_COLS, &t)) return;
  const uint32_t per = kv8_split_steps(t.steps, a.nsplit, a.chunk);
  const uint32_t s0 = t.step0 + split * per, end = t.step0 + t.steps;
  if (split > 0 && s0 >= end) return;
  const uint32_t s1 = min(s0 + per, end);

  float* lm = reinterpret_cast<float*>(lds);                   // [4][16]
  float *ll = lm + 64, *le = ll + 64;                          // [4][16]
  i32x4* qd = reinterpret_cast<i32x4*>(lds + KV8_ATTN_HEAD);   // [4][NL][64]
  f32x4* lo = reinterpret_cast<f32x4*>(lds + KV8_ATTN_HEAD);   // [4 waves][NL][4][64 lanes], after the steps
  uint32_t pages = step_pages(a, t, s0 + wave, 4);
  const uint32_t col = t.col0 + min(n, t.ncol - 1);  // columns past the last repeat it
  f32x4 row[(NL + 3) / 4][4];
  load_row<NL>(a.q + row_at(a, t, col), D, row);
  __builtin_amdgcn_sched_barrier(0);
  const int64_t pos = (int64_t)(t.past + col / G);
  Codes<NL> k, v;
  uint32_t i = 0, s = s0 + wave;
  if (s < s1) {
    load_codes<NL, FULL, STREAM, true>(a, t, s, pages, 0, &k);
    load_codes<NL, FULL, STREAM, false>(a, t, s, pages, 0, &v);
  }
  const Factor qf = stage_q<NL>(a, row, lm, qd);
  Run<NL> r;
  clear<NL>(&r);
  for (; s < s1; s += 4) {
    float sc[2][4];
    score_step<NL>(a, k, v.s, qd, qf, t, pos, s, sc);
    const bool more = s + 4 < s1;
    if (++i == 32 && more) {
      i = 0;
      pages = step_pages(a, t, s + 4, 4);
    }
    if (more) load_codes<NL, FULL, STREAM, true>(a, t, s + 4, pages, i, &k);
    __builtin_amdgcn_sched_barrier(0);
    f16x8 hi, lo;
    soft_step<NL, 0>(sc, v.s, v.has, &r, &hi, &lo);
    value_step<NL>(v, hi, lo, &r);
    if (more) load_codes<NL, FULL, STREAM, false>(a, t, s + 4, pages, i, &v);
    __builtin_amdgcn_sched_barrier(0);
  }
  r.l += __shfl_xor(r.l, 16, 64);
  r.l += __shfl_xor(r.l, 32, 64);

  // Join the waves: m, l and E of all, then each wave the sums of a quarter of the dims.
  if (lane < 16) {
    lm[wave * 16 + n] = r.m;
    ll[wave * 16 + n] = r.l;
    le[wave * 16 + n] = r.E;
  }
  __syncthreads();
  float M = kNoMax, L = 0.f, E = kNoUnit;
#pragma unroll
  for (int w = 0; w < 4; w++) M = fmaxf(M, lm[w * 16 + n]);
#pragma unroll
  for (int w = 0; w < 4; w++) {
    L += ll[w * 16 + n] * __builtin_amdgcn_exp2f(lm[w * 16 + n] - M);
    E = fmaxf(E, le[w * 16 + n] + (lm[w * 16 + n] - M));
  }
  const float f = __builtin_amdgcn_exp2f((r.m - M) + (r.E - E));
#pragma unroll
  for (int l = 0; l < NL; l++)
#pragma unroll
    for (int j = 0; j < 4; j++) lo[((wave * NL + l) * 4 + j) * 64 + lane] = r.o[l][j] * f;
  __syncthreads();
  if (n >= t.ncol) return;
  const bool only = per >= t.steps;  // the only split that runs
  float* to;
  float by = 1.f;
  int unit = 0;
  if (only) {
    to = a.out + row_at(a, t, col);
    by = L == 0.f ? 0.f : 1.f / L;  // nothing visible: 0
    unit = (int)E - kTop;
  } else {
    const uint64_t place = ((uint64_t)blockIdx.z * a.c.nkv + t.head) * (gridDim.x / a.nsplit) + tile;
    to = a.part + ((place * a.nsplit + split) * KV8_COLS + n) * (D + KV8_PART);
    if (wave == 0 && g == 0) {
      to[D] = M;
      to[D + 1] = L;
      to[D + 2] = E;
    }
  }
#pragma unroll
  for (int i = 0; i < (NL + 3) / 4; i++) {
    const uint32_t l = wave + 4 * i;
    if (l >= NL) break;
    f32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[j] = lo[(l * 4 + j) * 64 + lane];
#pragma unroll
      for (int w = 1; w < 4; w++) x[j] += lo[((w * NL + l) * 4 + j) * 64 + lane];
    }
    write_dims(x, to, 64 * l, D, by, unit);
  }
}

// Many query columns (a prompt's).  A step of 16 columns of 256 dims is 64 matrix
// instructions (1024 cycles of a SIMD) and about 310 vector ones (1240 cycles), which run
// beside each other only from different waves: two workgroups a CU, which no barrier
// couples, give every SIMD two waves for that.  A workgroup takes 32 columns: waves 0 and 1 sixteen each
// for the even steps, waves 2 and 3 the same for the odd ones, joined at the end,
// so that the workgroups of a causal prompt are short and many enough to even out
// over the CUs.  The codes of a step come through LDS once for its two waves, the values'
// already as f16, whose conversion is as much vector work as the softmax; the next
// step's are on their way to registers meanwhile.  (A prompt of 2000 tokens, 16 heads of
// 256 over 8 key heads: 97 us, 66 GFLOP made, the matrix cores busy for 32% of it, the
// vector units for 50%.  64 columns a workgroup took 3% less, but 13 - 20% more for prompts of
// 350 - 650 tokens.)
// grid (tiles * kv heads, 1, sequences), the tiles that see most first; the heads in
// turn, so that with eight of them a head's workgroups share an XCD's L2.
template <int NL, bool FULL>
__device__ __forceinline__ void attend_rows(const Kv8AttnArgs& a) {
  extern __shared__ __align__(16) char lds[];
  constexpr int NS = (NL + 1) / 2;
  constexpr uint32_t kPieces = 2 * NL * 64, vPieces = 4 * NL * 64;  // 16 bytes each, of a step
  const uint32_t lane = threadIdx.x & 63, wave = wave_id(), n = lane & 15, g = lane >> 4;
  const uint32_t part = wave & 1, par = wave >> 1;
  const uint32_t D = FULL ? 64 * NL : a.c.D, G = a.nq / a.c.nkv;
  const uint32_t head = blockIdx.x % a.c.nkv, tile = gridDim.x / a.c.nkv - 1 - blockIdx.x / a.c.nkv;
  Tile t;
  if (!tile_of(a, blockIdx.z, head, tile, KV8_ROW_COLS, &t)) return;
  const uint32_t s0 = t.step0, s1 = t.step0 + t.steps;
  i32x4* kb = reinterpret_cast<i32x4*>(lds) + par * (kPieces + vPieces);
  f16x8* vb = reinterpret_cast<f16x8*>(kb + kPieces);

  // this wave's columns (past the last they repeat it), and what they see
  const uint32_t c0 = t.col0 + part * KV8_COLS, last = t.col0 + t.ncol - 1, col = min(c0 + n, last);
  const int64_t pos = (int64_t)(t.past + col / G);
  Tile mine = t;
  {
    const uint64_t p0 = t.past + min(c0, last) / G, p1 = t.past + min(c0 + KV8_COLS - 1, last) / G;
    mine.step0 = a.window && p0 + 1 > a.window ? (uint32_t)((p0 + 1 - a.window) / KV8_STEP) : 0;
    mine.steps = (uint32_t)(p1 / KV8_STEP) + 1 - mine.step0;
    mine.all0 = a.window && p1 + 1 > a.window ? (uint32_t)((p1 + KV8_STEP - a.window) / KV8_STEP) : 0;
    mine.all1 = (uint32_t)((p0 + 1) / KV8_STEP);
  }

  uint32_t pages = step_pages(a, t, s0 + par, 2), at = 0;
  i32x4 kc[2][NS], vc[2][NS];
  float ks[2], vs[2], ks_next[2], vs_next[2];
  bool has[2], has_next[2];
  const auto load = [&](uint32_t step) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const uint64_t blk = (uint64_t)step * 2 + b;
      const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)pages, (int)(2 * at + b));
      has_next[b] = page < a.c.num_pages;
      const uint32_t place = block_at(a.c, has_next[b] ? page : 0, t.head, blk);
      ks_next[b] = a.c.ks[place];
      vs_next[b] = a.c.vs[place];
      const int8_t* k = a.c.k + (uint64_t)place * (KV8_BLOCK * D);
      const int8_t* v = a.c.v + (uint64_t)place * (KV8_BLOCK * D);
#pragma unroll
      for (int i = 0; i < NS; i++) {
        const uint32_t l = NL == 1 ? 0 : part + 2 * i;
        kc[b][i] = *reinterpret_cast<const i32x4*>(k + piece_at<FULL, true>(l, D));
        vc[b][i] = *reinterpret_cast<const i32x4*>(v + piece_at<FULL, false>(l, D));
      }
    }
    if (++at == 32) {
      at = 0;
      pages = step_pages(a, t, step + 2, 2);
    }
  };
  const auto store = [&]() {
#pragma unroll
    for (int i = 0; i < NS; i++) {
      const uint32_t l = NL == 1 ? 0 : part + 2 * i;
#pragma unroll
      for (int b = 0; b < 2; b++) kb[(b * NL + l) * 64 + lane] = kc[b][i];
#pragma unroll
      for (int j = 0; j < 4; j++) vb[(l * 4 + j) * 64 + lane] = codes_f16((uint32_t)vc[0][i][j], (uint32_t)vc[1][i][j]);
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
      ks[b] = ks_next[b];
      vs[b] = vs_next[b];
      has[b] = has_next[b];
    }
  };

  i32x4 qd[4][NL];
  uint32_t s = s0 + par;
  if (s < s1) load(s);
  const Factor qf = load_q<NL>(a, a.q + row_at(a, t, col), qd);
  // the lowest digits are in LDS: the registers hold three of four
  i32x4* q0 = reinterpret_cast<i32x4*>(lds) + 2 * (kPieces + vPieces) + part * NL * 64;
  if (par == 0) {
#pragma unroll
    for (int l = 0; l < NL; l++) q0[l * 64 + lane] = qd[0][l];
  }
  Run<NL> r;
  clear<NL>(&r);
  for (uint32_t first = s0; first < s1; first += 2, s += 2) {
    if (s < s1) store();
    if (s + 2 < s1) load(s + 2);
    __syncthreads();
    // (a step that none of the wave's columns sees: the others' barriers only)
    if (s < s1 && s - mine.step0 < mine.steps) {
      float sc[2][4];
      {
        i32x4 acc[2][4];
#pragma unroll
        for (int d = 0; d < 4; d++) acc[0][d] = acc[1][d] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int l = 0; l < NL; l++) {
          const i32x4 k0 = kb[l * 64 + lane], k1 = kb[(NL + l) * 64 + lane], low = q0[l * 64 + lane];
#pragma unroll
          for (int d = 0; d < 4; d++) {
            const i32x4 q = d == 0 ? low : qd[d][l];
            acc[0][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k0, q, acc[0][d], 0, 0, 0);
            acc[1][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k1, q, acc[1][d], 0, 0, 0);
          }
        }
        finish_scores(a, acc, ks, vs, has, qf, mine, pos, s, sc);
      }
      f16x8 x[4];  // the values' operands, one l ahead
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = vb[j * 64 + lane];
      f16x8 hi, lo;
      soft_step<NL, kLazy>(sc, vs, has, &r, &hi, &lo);
#pragma unroll
      for (int l = 0; l < NL; l++) {
        f16x8 y[4];
        if (l + 1 < NL) {
#pragma unroll
          for (int j = 0; j < 4; j++) y[j] = vb[((l + 1) * 4 + j) * 64 + lane];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) r.o[l][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[j], hi, r.o[l][j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; j++) r.o[l][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[j], lo, r.o[l][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = y[j];
      }
    }
    __syncthreads();
  }
  r.l += __shfl_xor(r.l, 16, 64);
  r.l += __shfl_xor(r.l, 32, 64);
  // the odd steps' sums come to the wave of the even ones
  float* lm = reinterpret_cast<float*>(lds) + part * (16 * NL * 64 + 192);
  float* lo = lm + 192;
  if (par == 1) {
    lm[lane] = r.m;
    lm[64 + lane] = r.l;
    lm[128 + lane] = r.E;
#pragma unroll
    for (int l = 0; l < NL; l++)
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) lo[(l * 16 + j * 4 + i) * 64 + lane] = r.o[l][j][i];
  }
  __syncthreads();
  if (par == 1) return;
  const float m1 = lm[lane], M = fmaxf(r.m, m1), d0 = r.m - M, d1 = m1 - M;
  const float E = fmaxf(fmaxf(r.E + d0, lm[128 + lane] + d1), kNoUnit);
  const float f0 = __builtin_amdgcn_exp2f(d0 + (r.E - E)), f1 = __builtin_amdgcn_exp2f(d1 + (lm[128 + lane] - E));
  const float L = r.l * __builtin_amdgcn_exp2f(d0) + lm[64 + lane] * __builtin_amdgcn_exp2f(d1);
#pragma unroll
  for (int l = 0; l < NL; l++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) r.o[l][j][i] = fmaf(lo[(l * 16 + j * 4 + i) * 64 + lane], f1, r.o[l][j][i] * f0);
  if (c0 + n > last) return;
  const float by = L == 0.f ? 0.f : 1.f / L;  // nothing visible: 0
  float* to = a.out + row_at(a, t, col);
#pragma unroll
  for (int l = 0; l < NL; l++) write_dims(r.o[l], to, 64 * l, D, by, (int)E - kTop + kLazy);
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void gh_kv8_append_p1_k(Kv8AppendArgs a) { append<1>(a); }
extern "C" __global__ __launch_bounds__(256) void gh_kv8_append_p2_k(Kv8AppendArgs a) { append<2>(a); }
extern "C" __global__ __launch_bounds__(256) void gh_kv8_append_p4_k(Kv8AppendArgs a) { append<4>(a); }

#define KV8_ATTN(NL, WAVES)                                                                                       \
  extern "C" __global__ __launch_bounds__(256, WAVES) void gh_kv8_attn_l##NL##_k(Kv8AttnArgs a) { attend<NL, true, false>(a); } \
  extern "C" __global__ __launch_bounds__(256, WAVES) void gh_kv8_attn_l##NL##r_k(Kv8AttnArgs a) { attend<NL, false, false>(a); } \
  extern "C" __global__ __launch_bounds__(256, WAVES) void gh_kv8_attn_l##NL##s_k(Kv8AttnArgs a) { attend<NL, true, true>(a); } \
  extern "C" __global__ __launch_bounds__(256, WAVES) void gh_kv8_attn_l##NL##rs_k(Kv8AttnArgs a) { attend<NL, false, true>(a); } \
  extern "C" __global__ __launch_bounds__(256, WAVES) void gh_kv8_rows_l##NL##_k(Kv8AttnArgs a) { attend_rows<NL, true>(a); } \
  extern "C" __global__ __launch_bounds__(256, WAVES) void gh_kv8_rows_l##NL##r_k(Kv8AttnArgs a) { attend_rows<NL, false>(a); }
KV8_ATTN(1, 2)
KV8_ATTN(2, 2)
KV8_ATTN(4, 2)
KV8_ATTN(8, 1)

// Joins the splits of a tile's column, in split order: the splits' factors in
// LDS, then a lane a dim.  (4 us: a chain of the sequence's length, the maxima, the sums.)  grid (tiles * columns a tile can have, kv heads, sequences)
extern "C" __global__ __launch_bounds__(256) void gh_kv8_merge_k(Kv8AttnArgs a, uint32_t cols) {
  const uint32_t tile = blockIdx.x / cols, n = blockIdx.x % cols, D = a.c.D;
  Tile t;
  if (!tile_of(a, blockIdx.z, blockIdx.y, tile, KV8_COLS, &t) || n >= t.ncol) return;
  const uint32_t per = kv8_split_steps(t.steps, a.nsplit, a.chunk);
  if (per >= t.steps) return;  // written by its only split
  const uint32_t live = (t.steps + per - 1) / per, tid = threadIdx.x;
  const uint64_t unit = ((uint64_t)blockIdx.z * a.c.nkv + t.head) * (gridDim.x / cols) + tile;
  const uint64_t row = KV8_COLS * (uint64_t)(D + KV8_PART);
  const float* p = a.part + unit * a.nsplit * row + n * (uint64_t)(D + KV8_PART);
  __shared__ float f[KV8_MAX_SPLIT], red[12];
  constexpr uint32_t N = 8;  // sums on their way at a time, the first of them before the factors
  float x[N];
#pragma unroll
  for (uint32_t i = 0; i < N; i++) x[i] = i < live && tid < D ? p[i * row + tid] : 0.f;
  float m = kNoMax, l = 0.f, e = kNoUnit;
  if (tid < live) {
    m = p[tid * row + D];
    l = p[tid * row + D + 1];
    e = p[tid * row + D + 2];
  }
  // the largest maximum, then the largest unit by it
  float M = m;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
  if ((tid & 63) == 0) red[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float x2 = (m - M) + e, L0 = wave_sum(l * __builtin_amdgcn_exp2f(m - M));
  float E = fmaxf(x2, kNoUnit);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) E = fmaxf(E, __shfl_xor(E, off, 64));
  if ((tid & 63) == 0) {
    red[4 + (tid >> 6)] = L0;
    red[8 + (tid >> 6)] = E;
  }
  __syncthreads();
  E = fmaxf(fmaxf(red[8], red[9]), fmaxf(red[10], red[11]));
  f[tid] = __builtin_amdgcn_exp2f(x2 - E);
  __syncthreads();
  const float L = (red[4] + red[5]) + (red[6] + red[7]);
  const float by = L == 0.f ? 0.f : 1.f / L;
  float* out = a.out + row_at(a, t, t.col0 + n);
  for (uint32_t d = tid; d < D; d += 256) {
    float o = 0.f;
    for (uint32_t s = 0; s < live; s += N) {
      if (s > 0 || d >= 256) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++) x[i] = s + i < live ? p[(s + i) * row + d] : 0.f;
      }
#pragma unroll
      for (uint32_t i = 0; i < N; i++) o = fmaf(x[i], s + i < live ? f[s + i] : 0.f, o);
    }
    out[d] = ldexpf(o * by, (int)E - kTop);
  }
}

namespace {
// (wide: 16-byte aligned; by the caches: 2000 rows of 8 heads of 256 8.2 us, 5.0
// TB/s; through them 9.0)
__device__ __forceinline__ void write4(float* to, f32x4 x, uint32_t wide) {
  if (wide) {
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(to));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) to[i] = x[i];
  }
}
}  // namespace

// Read-back: the rows that a batch names as the values their codes stand for;
// rows of places without a page are 0.  grid (kv heads, blocks, sequences)
extern "C" __global__ __launch_bounds__(256) void gh_kv8_read_k(Kv8ReadArgs a) {
  const uint32_t seq = blockIdx.z, head = blockIdx.x, D = a.c.D;
  uint32_t first;
  const uint32_t rows = seq_rows(a.b, seq, &first);
  const uint64_t past = a.b.past[seq], blk = past / KV8_BLOCK + blockIdx.y;
  const uint64_t p0 = max(past, blk * KV8_BLOCK), p1 = min(past + rows, (blk + 1) * KV8_BLOCK);
  if (p0 >= p1) return;
  const uint32_t o0 = (uint32_t)(p0 - blk * KV8_BLOCK), o1 = (uint32_t)(p1 - blk * KV8_BLOCK);
  const uint64_t row0 = first + (p0 - past), kv = (uint64_t)a.c.nkv * D;
  const uint32_t page = page_of(a.c, a.b, seq, blk);
  const bool has = page < a.c.num_pages;
  const uint32_t at = block_at(a.c, has ? page : 0, head, blk);
  const uint64_t bytes = (uint64_t)at * (KV8_BLOCK * D);
  // four dims of a token (K), of four tokens (V): a wave's rows of float4 in a row
  if (a.k) {
    const float s = has ? a.c.ks[at] : 0.f;
    for (uint32_t i = threadIdx.x; i < 4 * D; i += 256) {
      const uint32_t t = i / (D / 4), d = (i % (D / 4)) * 4;
      if (t < o0 || t >= o1) continue;
      char4 c{0, 0, 0, 0};
      if (has) c = *reinterpret_cast<const char4*>(a.c.k + bytes + k_place(t, d));
      write4(a.k + (row0 + t - o0) * kv + (uint64_t)head * D + d, f32x4{(float)c.x, (float)c.y, (float)c.z, (float)c.w} * s, a.wide);
    }
  }
  if (a.v) {
    const float s = has ? a.c.vs[at] : 0.f;
    for (uint32_t i = threadIdx.x; i < D; i += 256) {
      const uint32_t grp = i / (D / 4), d = (i % (D / 4)) * 4;
      union {
        int4 w;
        int8_t b[16];
      } p;
      p.w = int4{0, 0, 0, 0};
      if (has) p.w = reinterpret_cast<const int4*>(a.c.v + bytes)[i];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t t = grp * 4 + e;
        if (t < o0 || t >= o1) continue;
        write4(a.v + (row0 + t - o0) * kv + (uint64_t)head * D + d,
               f32x4{(float)p.b[e], (float)p.b[4 + e], (float)p.b[8 + e], (float)p.b[12 + e]} * s, a.wide);
      }
    }
  }
}
