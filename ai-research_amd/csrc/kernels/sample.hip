// sample.hip -- from logits to probabilities, and the verification of drafted
// tokens against them, for gfx950.
//
// Both read rows of a vocabulary once or twice and compute little: what bounds
// them is memory for a batch and latency for one row.  A row is cut into chunks of
// 256 N elements, a workgroup each, N = 16, or 4 so that one row of 262144 spreads
// over every CU; a second launch joins the chunks.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../common/sample_args.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// A thread's elements of chunk c: VEC: float4, 1 KB apart in a wave's row; else
// single floats.  Elements past the row are `none`.  STREAM: they are not read again,
// and pass by the caches.
template <bool VEC>
__device__ __forceinline__ uint32_t elem(uint32_t i) {
  return VEC ? (i >> 2) * 1024 + threadIdx.x * 4 + (i & 3) : i * 256 + threadIdx.x;
}
template <bool VEC, uint32_t N, bool STREAM>
__device__ __forceinline__ void load_chunk(const float* row, uint32_t c, uint32_t vocab, float none, float (&x)[N]) {
  const uint32_t base = c * (256 * N), left = vocab - base;
  row += base;
#pragma unroll
  for (uint32_t i = 0; i < N; i += VEC ? 4 : 1) {
    const uint32_t e = elem<VEC>(i);
    if (VEC) {  // (vocab is a multiple of 4 there)
      f32x4 v = {none, none, none, none};
      const f32x4* p = reinterpret_cast<const f32x4*>(row + e);
      if (e < left) v = STREAM ? __builtin_nontemporal_load(p) : *p;
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) x[i + j] = v[j];
    } else {
      x[i] = e < left ? row[e] : none;
    }
  }
}

// ---------------------------------------------------------------------------
// Probabilities: y = cap tanh(x / cap) (x without a cap; -inf stays), p =
// 2^((y - max) log2(e) / temperature) / sum.  The first launch leaves each chunk's
// maximum and sum, the second joins a row's and writes; it finds the logits in
// the last-level cache.  (40 rows of 262144: 19 us a call among others, 23 when the
// second's loads and stores stay in the caches; 4 bytes read and 4 written an element
// at the rate of a copy are 17.7.)
// ---------------------------------------------------------------------------
// tanh within 5 half steps, without the library's branches, which bounded the
// kernels (40 rows of 262144: 17 us a launch at 2.5 TB/s): below 0.7 y + y^3 P(y^2),
// P fitted by least squares at Chebyshev nodes (relative error 8e-10 before
// rounding), above 1 - 2 / (e^2y + 1).
__device__ __forceinline__ float tanh_low(float y) {
  const float t = y * y;
  float p = 0.00188978482f;
  p = fmaf(p, t, -0.00787458383f);
  p = fmaf(p, t, 0.0215662047f);
  p = fmaf(p, t, -0.0539197139f);
  p = fmaf(p, t, 0.13332969f);
  p = fmaf(p, t, -0.333333254f);
  return fmaf(y * t, p, y);
}
__device__ __forceinline__ float tanh_high(float y) {
  const float e = __builtin_amdgcn_exp2f(fabsf(y) * 2.885390082f);
  return copysignf(fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f), y);
}
// A thread's logits soft-capped, in units of the cap.  Most rows have nothing past 0.7
// cap: a wave without takes the first form alone.
template <uint32_t N>
__device__ __forceinline__ void soft_cap(float (&x)[N], float inv_cap) {
  if (!(inv_cap > 0.f)) return;
  float y[N], far = 0.f;
#pragma unroll
  for (uint32_t i = 0; i < N; i++) {
    y[i] = x[i] * inv_cap;
    far = fmaxf(far, fabsf(y[i]));
  }
  if (__any(!(far < 0.7f))) {
#pragma unroll
    for (uint32_t i = 0; i < N; i++)
      if (x[i] != -INFINITY) x[i] = fabsf(y[i]) < 0.7f ? tanh_low(y[i]) : tanh_high(y[i]);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; i++) x[i] = tanh_low(y[i]);
  }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// what is subtracted for a maximum (of nothing: 0)
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// The workgroup's maximum and the sum relative to it, in every thread, from its waves'
// maxima and their threads' sums relative to them.
__device__ __forceinline__ void join(float* m, float* l, float mul) {
  __shared__ float sm[4], sl[4];
  const uint32_t wave = threadIdx.x >> 6;
  const float sum = wave_sum(*l);
  if ((threadIdx.x & 63) == 0) {
    sm[wave] = *m;
    sl[wave] = sum;
  }
  __syncthreads();
  const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float L = 0.f;
#pragma unroll
  for (int w = 0; w < 4; w++) L += sl[w] * __builtin_amdgcn_exp2f((sm[w] - base_of(M)) * mul);
  *m = M;
  *l = L;
}

// grid (chunks, rows)
template <bool VEC, uint32_t N>
__device__ __forceinline__ void probs_part(const ProbsArgs& a) {
  float x[N], m = -INFINITY, l = 0.f;
  load_chunk<VEC, N, false>(a.logits + blockIdx.y * a.stride, blockIdx.x, a.vocab, -INFINITY, x);
  soft_cap<N>(x, a.inv_cap);
#pragma unroll
  for (uint32_t i = 0; i < N; i++) m = fmaxf(m, x[i]);
  m = wave_max(m);
  const float base = base_of(m);
#pragma unroll
  for (uint32_t i = 0; i < N; i++) l += __builtin_amdgcn_exp2f((x[i] - base) * a.mul);
  join(&m, &l, a.mul);
  if (threadIdx.x == 0) {
    float* p = a.part + 2 * ((uint64_t)blockIdx.y * a.chunks + blockIdx.x);
    p[0] = m;
    p[1] = l;
  }
}

template <bool VEC, uint32_t N>
__device__ __forceinline__ void probs_write(const ProbsArgs& a) {
  float x[N], m = -INFINITY, l = 0.f;
  load_chunk<VEC, N, true>(a.logits + blockIdx.y * a.stride, blockIdx.x, a.vocab, -INFINITY, x);
  const float* p = a.part + 2 * (uint64_t)blockIdx.y * a.chunks;
  for (uint32_t c = threadIdx.x; c < a.chunks; c += 256) {
    const float m2 = p[2 * c], l2 = p[2 * c + 1], mx = fmaxf(m, m2), base = base_of(mx);
    l = l * __builtin_amdgcn_exp2f((m - base) * a.mul) + l2 * __builtin_amdgcn_exp2f((m2 - base) * a.mul);
    m = mx;
  }
  soft_cap<N>(x, a.inv_cap);
  const float wm = wave_max(m);
  l *= __builtin_amdgcn_exp2f((m - base_of(wm)) * a.mul);
  m = wm;
  join(&m, &l, a.mul);
  const float base = base_of(m);
  const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;  // every logit -inf: all 0
  const uint32_t start = blockIdx.x * (256 * N), left = a.vocab - start;
  float* out = a.probs + blockIdx.y * a.stride + start;
#pragma unroll
  for (uint32_t i = 0; i < N; i++) x[i] = __builtin_amdgcn_exp2f((x[i] - base) * a.mul) * inv;
#pragma unroll
  for (uint32_t i = 0; i < N; i += VEC ? 4 : 1) {
    const uint32_t e = elem<VEC>(i);
    if (e >= left) continue;
    if (VEC) {
      __builtin_nontemporal_store(f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]}, reinterpret_cast<f32x4*>(out + e));
    } else {
      out[e] = x[i];
    }
  }
}

// ---------------------------------------------------------------------------
// Verification.  Draft i is kept while u_i q_i(x_i) < p_i(x_i) (exact in 64 bits);
// where it stops, the token is drawn from what the target has over the draft,
// max(p - q, 0), or from the target itself after the last draft.  A token is
// decided next to a border, so weights and sums are in 64 bits.  (32 sequences of 262144:
// 12.9 us for the chunks' sums, 5.2 TB/s, and 4.9 for the token, a chain of loads.)
// ---------------------------------------------------------------------------
struct Stop {
  uint32_t kept, drafts;
};

// how many drafts of sequence b are kept (every wave finds it for itself: a few
// scattered loads)
__device__ __forceinline__ Stop stop_of(const VerifyArgs& a, uint32_t b) {
  const uint32_t n = a.n_draft ? min(a.n_draft[b], a.max_draft) : a.max_draft, lane = threadIdx.x & 63;
  uint32_t kept = n;
  for (uint32_t i0 = 0; i0 < n; i0 += 64) {
    const uint32_t i = i0 + lane;
    bool fine = true;
    if (i < n) {
      const uint32_t x = a.tokens[(uint64_t)b * a.max_draft + i];
      fine = false;
      if (x < a.vocab) {
        const double p = a.target[((uint64_t)b * (a.max_draft + 1) + i) * a.vocab + x];
        const double q = a.draft ? (double)a.draft[((uint64_t)b * a.max_draft + i) * a.vocab + x] : 1.0;
        fine = (double)a.u[(uint64_t)b * a.max_draft + i] * q < p;
      }
    }
    const uint64_t bad = __ballot(!fine);
    if (bad) {
      kept = i0 + (uint32_t)__builtin_ctzll(bad);
      break;
    }
  }
  return Stop{(uint32_t)__builtin_amdgcn_readfirstlane(kept), n};
}

// weight of element v where sequence b stops: left over the draft, and the target's
struct Rows {
  const float *p, *q;  // q null: nothing is taken off, or one token is (cut)
  uint32_t cut;
};
__device__ __forceinline__ Rows rows_of(const VerifyArgs& a, uint32_t b, Stop s) {
  Rows r;
  r.p = a.target + ((uint64_t)b * (a.max_draft + 1) + s.kept) * a.vocab;
  const bool stopped = s.kept < s.drafts;
  r.q = stopped && a.draft ? a.draft + ((uint64_t)b * a.max_draft + s.kept) * a.vocab : nullptr;
  r.cut = stopped && !a.draft ? a.tokens[(uint64_t)b * a.max_draft + s.kept] : 0xffffffffu;
  return r;
}
// (comparisons, so that NaN and negative entries weigh nothing)
__device__ __forceinline__ double over(float p, float q, bool cut) {
  const double d = (double)p - (cut ? 1.0 : (double)q);
  return d > 0.0 ? d : 0.0;
}
__device__ __forceinline__ double plain(float p) { return p > 0.f ? (double)p : 0.0; }

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// grid (chunks, sequences)
template <bool VEC, uint32_t N>
__device__ __forceinline__ void verify_part(const VerifyArgs& a) {
  const uint32_t b = blockIdx.y, c = blockIdx.x;
  const Stop s = stop_of(a, b);
  const Rows r = rows_of(a, b, s);
  float p[N], q[N];
  load_chunk<VEC, N, true>(r.p, c, a.vocab, 0.f, p);
  if (r.q) {
    load_chunk<VEC, N, true>(r.q, c, a.vocab, 0.f, q);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; i++) q[i] = 0.f;
  }
  double w = 0.0, t = 0.0;
#pragma unroll
  for (uint32_t i = 0; i < N; i++) {
    w += over(p[i], q[i], c * (256 * N) + elem<VEC>(i) == r.cut);
    t += plain(p[i]);
  }
  w = wave_sum(w);
  t = wave_sum(t);
  __shared__ double sw[4], st[4];
  if ((threadIdx.x & 63) == 0) {
    sw[threadIdx.x >> 6] = w;
    st[threadIdx.x >> 6] = t;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double* out = a.part + 2 * ((uint64_t)b * a.chunks + c);
    out[0] = sw[0] + sw[1] + (sw[2] + sw[3]);
    out[1] = st[0] + st[1] + (st[2] + st[3]);
    if (c == 0) a.accepted[b] = s.kept;
  }
}

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ double wave_scan(double v) {
  const uint32_t lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double u = __shfl_up(v, off, 64);
    if (lane >= (uint32_t)off) v += u;
  }
  return v;
}

// N elements of a row from v0 on (0 past its end, or without a row).
template <bool VEC, uint32_t N>
__device__ __forceinline__ void row_part(const float* row, uint32_t v0, uint32_t vocab, float (&x)[N]) {
#pragma unroll
  for (uint32_t i = 0; i < N; i += VEC ? 4 : 1) {
    if (VEC) {
      float4 v = {0.f, 0.f, 0.f, 0.f};
      if (row && v0 + i < vocab) v = *reinterpret_cast<const float4*>(row + v0 + i);
      x[i] = v.x;
      x[i + 1] = v.y;
      x[i + 2] = v.z;
      x[i + 3] = v.w;
    } else {
      x[i] = row && v0 + i < vocab ? row[v0 + i] : 0.f;
    }
  }
}

// The token of a sequence: the chunk that the drawn share falls into (every wave
// finds it for itself, its lanes a run of chunks each), then the element.
// grid (sequences)
template <bool VEC, uint32_t N>
__device__ __forceinline__ void verify_token(const VerifyArgs& a) {
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t kept = a.accepted[b];  // (the first launch's)
  const uint32_t drafts = a.n_draft ? min(a.n_draft[b], a.max_draft) : a.max_draft;
  const Rows r = rows_of(a, b, Stop{kept, drafts});
  const double* part = a.part + 2 * (uint64_t)b * a.chunks;
  const uint32_t per = (a.chunks + 63) / 64, c0 = min(lane * per, a.chunks), c1 = min(c0 + per, a.chunks);
  double w = 0.0, t = 0.0;
  for (uint32_t c = c0; c < c1; c++) {
    w += part[2 * c];
    t += part[2 * c + 1];
  }
  const double cw = wave_scan(w), ct = wave_scan(t);
  const double total_w = __shfl(cw, 63, 64), total_t = __shfl(ct, 63, 64);
  const bool left = total_w > 0.0;  // else (the draft covers the target) the target itself
  const double total = left ? total_w : total_t, mine = left ? w : t, upto = left ? cw : ct;
  uint32_t token = 0xffffffffu;
  if (total > 0.0 && total < HUGE_VAL) {
    float u = a.pick[b];
    u = u > 0.f ? u : 0.f;
    const double goal = (double)u * total;
    // the lane whose run of chunks holds it (past the end: the last that weighs)
    const uint64_t hits = __ballot(upto > goal && mine > 0.0), some = __ballot(mine > 0.0);
    const int who = hits ? __builtin_ctzll(hits) : 63 - __builtin_clzll(some);
    double before = __shfl(upto - mine, who, 64), run = before;
    uint32_t chunk = 0;
    const uint32_t w0 = min((uint32_t)who * per, a.chunks), w1 = min(w0 + per, a.chunks);
    for (uint32_t c = w0; c < w1; c++) {
      const double x = part[2 * c + (left ? 0 : 1)];
      if (x > 0.0) {
        chunk = c;
        before = run;
        if (run + x > goal) break;
      }
      run += x;
    }
    // the chunk's elements, N in a row a thread
    const uint32_t v0 = chunk * (256 * N) + tid * N;
    double e[N], sum = 0.0;
    uint32_t last = 0xffffffffu, hit = 0xffffffffu;
    float p[N], q[N];
    row_part<VEC, N>(r.p, v0, a.vocab, p);
    row_part<VEC, N>(left ? r.q : nullptr, v0, a.vocab, q);
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
      e[i] = left ? over(p[i], q[i], v0 + i == r.cut) : plain(p[i]);
      if (e[i] > 0.0) last = v0 + i;
      sum += e[i];
    }
    __shared__ double waves[4];
    __shared__ uint32_t found[8];
    const double upto_here = wave_scan(sum);
    if (lane == 63) waves[wave] = upto_here;
    __syncthreads();
    for (uint32_t k = 0; k < wave; k++) before += waves[k];
    double here = before + (upto_here - sum);
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
      here += e[i];
      if (e[i] > 0.0 && hit == 0xffffffffu && here > goal) hit = v0 + i;
    }
    const uint64_t with_hit = __ballot(hit != 0xffffffffu), with_any = __ballot(last != 0xffffffffu);
    const uint32_t first_hit = __shfl(hit, with_hit ? __builtin_ctzll(with_hit) : 0, 64);
    const uint32_t last_any = __shfl(last, with_any ? 63 - __builtin_clzll(with_any) : 0, 64);
    if (lane == 0) {
      found[wave] = with_hit ? first_hit : 0xffffffffu;
      found[4 + wave] = with_any ? last_any : 0xffffffffu;
    }
    __syncthreads();
#pragma unroll
    for (int k = 3; k >= 0; k--)
      if (found[k] != 0xffffffffu) token = found[k];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (token == 0xffffffffu && found[7 - k] != 0xffffffffu) token = found[7 - k];
  }
  const uint32_t width = a.max_draft + 1;
  for (uint32_t i = tid; i < width; i += 256)
    a.out[(uint64_t)b * width + i] =
        i < kept ? a.tokens[(uint64_t)b * a.max_draft + i] : i == kept ? token : 0xffffffffu;
}

}  // namespace

// N elements a thread, 16-byte loads (v4) or single ones (v1)
#define SAMPLE(N)                                                                                                     \
  extern "C" __global__ __launch_bounds__(256) void gh_probs_part_n##N##_v4_k(ProbsArgs a) { probs_part<true, N>(a); }   \
  extern "C" __global__ __launch_bounds__(256) void gh_probs_part_n##N##_v1_k(ProbsArgs a) { probs_part<false, N>(a); }  \
  extern "C" __global__ __launch_bounds__(256) void gh_probs_write_n##N##_v4_k(ProbsArgs a) { probs_write<true, N>(a); } \
  extern "C" __global__ __launch_bounds__(256) void gh_probs_write_n##N##_v1_k(ProbsArgs a) { probs_write<false, N>(a); } \
  extern "C" __global__ __launch_bounds__(256) void gh_verify_part_n##N##_v4_k(VerifyArgs a) { verify_part<true, N>(a); } \
  extern "C" __global__ __launch_bounds__(256) void gh_verify_part_n##N##_v1_k(VerifyArgs a) { verify_part<false, N>(a); } \
  extern "C" __global__ __launch_bounds__(256) void gh_verify_token_n##N##_v4_k(VerifyArgs a) { verify_token<true, N>(a); } \
  extern "C" __global__ __launch_bounds__(256) void gh_verify_token_n##N##_v1_k(VerifyArgs a) { verify_token<false, N>(a); }
SAMPLE(4)
SAMPLE(16)
