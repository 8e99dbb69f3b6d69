// sample.hip -- from logits to probabilities, and the verification of drafted
// tokens against them, for gfx950.
//
// Both read rows of a vocabulary once or twice and compute little: what bounds
// them is memory for a batch and latency for one row.  A row is cut into chunks
// of SAMPLE_CHUNK elements, a workgroup each, so that one row of 262144 spreads
// over 64 CUs; a second launch joins the chunks.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../common/sample_args.h"

namespace {

constexpr uint32_t kEach = SAMPLE_CHUNK / 256;  // elements of a thread

// A thread's elements of chunk c: VEC: four float4, 1 KB apart in a wave's row;
// else single floats.  Elements past the row are `none`.
template <bool VEC>
__device__ __forceinline__ uint32_t elem(uint32_t i) {
  return VEC ? (i >> 2) * 1024 + threadIdx.x * 4 + (i & 3) : i * 256 + threadIdx.x;
}
template <bool VEC>
__device__ __forceinline__ void load_chunk(const float* row, uint32_t c, uint32_t vocab, float none, float (&x)[kEach]) {
  const uint32_t base = c * SAMPLE_CHUNK, left = vocab - base;
  row += base;
#pragma unroll
  for (uint32_t i = 0; i < kEach; i += VEC ? 4 : 1) {
    const uint32_t e = elem<VEC>(i);
    if (VEC) {  // (vocab is a multiple of 4 there)
      float4 v = {none, none, none, none};
      if (e < left) v = *reinterpret_cast<const float4*>(row + e);
      x[i] = v.x;
      x[i + 1] = v.y;
      x[i + 2] = v.z;
      x[i + 3] = v.w;
    } else {
      x[i] = e < left ? row[e] : none;
    }
  }
}

// ---------------------------------------------------------------------------
// Probabilities: y = cap tanh(x / cap) (x without a cap; -inf stays), p =
// 2^((y - max) log2(e) / temperature) / sum.  The first launch leaves each chunk's
// maximum and sum, the second joins a row's and writes; it finds the logits in
// the last-level cache.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float capped(float x, float cap) {
  return cap > 0.f && x != -INFINITY ? cap * tanhf(x / cap) : x;
}

// the workgroup's maximum and the sum relative to it, in every thread
__device__ __forceinline__ void join(float* m, float* l, float mul) {
  __shared__ float sm[4], sl[4];
  float M = *m, L = *l;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float m2 = __shfl_xor(M, off, 64), l2 = __shfl_xor(L, off, 64), mx = fmaxf(M, m2);
    const float base = mx == -INFINITY ? 0.f : mx;
    // in the order of the lanes, so that both of a pair get the same sum
    const float a = L * exp2f((M - base) * mul), b = l2 * exp2f((m2 - base) * mul);
    L = a + b;
    M = mx;
  }
  const uint32_t wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    sm[wave] = M;
    sl[wave] = L;
  }
  __syncthreads();
  M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float base = M == -INFINITY ? 0.f : M;
  L = 0.f;
#pragma unroll
  for (int w = 0; w < 4; w++) L += sl[w] * exp2f((sm[w] - base) * mul);
  *m = M;
  *l = L;
}

// grid (chunks, rows)
template <bool VEC>
__device__ __forceinline__ void probs_part(const ProbsArgs& a) {
  float x[kEach], m = -INFINITY, l = 0.f;
  load_chunk<VEC>(a.logits + blockIdx.y * a.stride, blockIdx.x, a.vocab, -INFINITY, x);
#pragma unroll
  for (uint32_t i = 0; i < kEach; i++) {
    x[i] = capped(x[i], a.cap);
    m = fmaxf(m, x[i]);
  }
  const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (uint32_t i = 0; i < kEach; i++) l += exp2f((x[i] - base) * a.mul);
  join(&m, &l, a.mul);
  if (threadIdx.x == 0) {
    float* p = a.part + 2 * ((uint64_t)blockIdx.y * a.chunks + blockIdx.x);
    p[0] = m;
    p[1] = l;
  }
}

template <bool VEC>
__device__ __forceinline__ void probs_write(const ProbsArgs& a) {
  float x[kEach], m = -INFINITY, l = 0.f;
  load_chunk<VEC>(a.logits + blockIdx.y * a.stride, blockIdx.x, a.vocab, -INFINITY, x);
  const float* p = a.part + 2 * (uint64_t)blockIdx.y * a.chunks;
  for (uint32_t c = threadIdx.x; c < a.chunks; c += 256) {
    const float m2 = p[2 * c], l2 = p[2 * c + 1], mx = fmaxf(m, m2), base = mx == -INFINITY ? 0.f : mx;
    l = l * exp2f((m - base) * a.mul) + l2 * exp2f((m2 - base) * a.mul);
    m = mx;
  }
  join(&m, &l, a.mul);
  const float base = m == -INFINITY ? 0.f : m;
  const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;  // every logit -inf: all 0
  const uint32_t start = blockIdx.x * SAMPLE_CHUNK, left = a.vocab - start;
  float* out = a.probs + blockIdx.y * a.stride + start;
#pragma unroll
  for (uint32_t i = 0; i < kEach; i++) x[i] = exp2f((capped(x[i], a.cap) - base) * a.mul) * inv;
#pragma unroll
  for (uint32_t i = 0; i < kEach; i += VEC ? 4 : 1) {
    const uint32_t e = elem<VEC>(i);
    if (e >= left) continue;
    if (VEC) {
      *reinterpret_cast<float4*>(out + e) = float4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    } else {
      out[e] = x[i];
    }
  }
}

// ---------------------------------------------------------------------------
// Verification.  Draft i is kept while u_i q_i(x_i) < p_i(x_i) (exact in 64 bits);
// where it stops, the token is drawn from what the target has over the draft,
// max(p - q, 0), or from the target itself after the last draft.  A token is
// decided next to a border, so weights and sums are in 64 bits.
// ---------------------------------------------------------------------------
struct Stop {
  uint32_t kept, drafts;
};

// how many drafts of sequence b are kept (every workgroup finds it for itself:
// a few scattered loads)
__device__ __forceinline__ Stop stop_of(const VerifyArgs& a, uint32_t b) {
  __shared__ uint32_t s;
  const uint32_t n = a.n_draft ? min(a.n_draft[b], a.max_draft) : a.max_draft;
  if (threadIdx.x < 64) {
    uint32_t kept = n;
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {
      const uint32_t i = i0 + threadIdx.x;
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
    if (threadIdx.x == 0) s = kept;
  }
  __syncthreads();
  return Stop{s, n};
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
template <bool VEC>
__device__ __forceinline__ void verify_part(const VerifyArgs& a) {
  const uint32_t b = blockIdx.y, c = blockIdx.x;
  const Rows r = rows_of(a, b, stop_of(a, b));
  float p[kEach], q[kEach];
  load_chunk<VEC>(r.p, c, a.vocab, 0.f, p);
  if (r.q) {
    load_chunk<VEC>(r.q, c, a.vocab, 0.f, q);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) q[i] = 0.f;
  }
  double w = 0.0, t = 0.0;
#pragma unroll
  for (uint32_t i = 0; i < kEach; i++) {
    w += over(p[i], q[i], c * SAMPLE_CHUNK + elem<VEC>(i) == r.cut);
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
  }
}

// Inclusive sums over the workgroup's threads, in their order.
__device__ __forceinline__ double scan(double v, double* total) {
  __shared__ double s[4];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double u = __shfl_up(v, off, 64);
    if (lane >= (uint32_t)off) v += u;
  }
  __syncthreads();
  if (lane == 63) s[wave] = v;
  __syncthreads();
  double before = 0.0;
  for (uint32_t w = 0; w < wave; w++) before += s[w];
  *total = s[0] + s[1] + s[2] + s[3];
  return before + v;
}

// The least index whose mark is set, 0xffffffff if there is none; `last`: the greatest.
__device__ __forceinline__ uint32_t pick_index(bool mark, uint32_t index, bool last) {
  __shared__ uint32_t s[4];
  uint32_t v = mark ? (last ? 0xfffffffeu - index : index) : 0xffffffffu;  // (index below 2^31)
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = min(v, (uint32_t)__shfl_xor((int)v, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = min(min(s[0], s[1]), min(s[2], s[3]));
  return v == 0xffffffffu ? v : last ? 0xfffffffeu - v : v;
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void gh_probs_part_v4_k(ProbsArgs a) { probs_part<true>(a); }
extern "C" __global__ __launch_bounds__(256) void gh_probs_part_v1_k(ProbsArgs a) { probs_part<false>(a); }
extern "C" __global__ __launch_bounds__(256) void gh_probs_write_v4_k(ProbsArgs a) { probs_write<true>(a); }
extern "C" __global__ __launch_bounds__(256) void gh_probs_write_v1_k(ProbsArgs a) { probs_write<false>(a); }
extern "C" __global__ __launch_bounds__(256) void gh_verify_part_v4_k(VerifyArgs a) { verify_part<true>(a); }
extern "C" __global__ __launch_bounds__(256) void gh_verify_part_v1_k(VerifyArgs a) { verify_part<false>(a); }

// The token of each sequence: the chunk that the drawn share falls into, then the
// element.  grid (sequences)
extern "C" __global__ __launch_bounds__(256) void gh_verify_token_k(VerifyArgs a) {
  const uint32_t b = blockIdx.x, tid = threadIdx.x;
  const Stop st = stop_of(a, b);
  const Rows r = rows_of(a, b, st);
  const double* part = a.part + 2 * (uint64_t)b * a.chunks;
  // the sums of a thread's run of chunks
  const uint32_t per = (a.chunks + 255) / 256, c0 = min(tid * per, a.chunks), c1 = min(c0 + per, a.chunks);
  double w = 0.0, t = 0.0;
  for (uint32_t c = c0; c < c1; c++) {
    w += part[2 * c];
    t += part[2 * c + 1];
  }
  double total_w, total_t;
  const double cw = scan(w, &total_w), ct = scan(t, &total_t);
  const bool left = total_w > 0.0;  // else (the draft covers the target) the target itself
  const double total = left ? total_w : total_t, mine = left ? w : t;
  uint32_t token = 0xffffffffu;
  if (total > 0.0 && total < HUGE_VAL) {
    float u = a.pick[b];
    u = u > 0.f ? u : 0.f;
    const double goal = (double)u * total;
    // the thread whose run of chunks holds it (past the end: the last that weighs)
    const double upto = left ? cw : ct;
    uint32_t who = pick_index(upto > goal && mine > 0.0, tid, false);
    if (who == 0xffffffffu) who = pick_index(mine > 0.0, tid, true);
    __shared__ double s_before;
    __shared__ uint32_t s_chunk;
    if (tid == who) {
      double before = upto - mine;
      uint32_t c = c0, last = c0;
      double last_before = before;
      for (; c < c1; c++) {
        const double x = part[2 * c + (left ? 0 : 1)];
        if (x > 0.0) {
          last = c;
          last_before = before;
          if (before + x > goal) break;
        }
        before += x;
      }
      s_chunk = last;
      s_before = last_before;
    }
    __syncthreads();
    const uint32_t c = s_chunk, base = c * SAMPLE_CHUNK, v0 = base + tid * kEach;
    const double before = s_before;
    double e[kEach], sum = 0.0, chunk_total;
    bool any = false;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
      const uint32_t v = v0 + i;
      e[i] = 0.0;
      if (v < a.vocab) e[i] = left ? over(r.p[v], r.q ? r.q[v] : 0.f, v == r.cut) : plain(r.p[v]);
      any |= e[i] > 0.0;
      sum += e[i];
    }
    double run = before + (scan(sum, &chunk_total) - sum);
    uint32_t hit = 0xffffffffu, last = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
      run += e[i];
      if (e[i] > 0.0) {
        last = v0 + i;
        if (hit == 0xffffffffu && run > goal) hit = v0 + i;
      }
    }
    token = pick_index(hit != 0xffffffffu, hit, false);
    if (token == 0xffffffffu) token = pick_index(any, last, true);
  }
  const uint32_t width = a.max_draft + 1;
  for (uint32_t i = tid; i < width; i += 256)
    a.out[(uint64_t)b * width + i] =
        i < st.kept ? a.tokens[(uint64_t)b * a.max_draft + i] : i == st.kept ? token : 0xffffffffu;
  if (tid == 0) a.accepted[b] = st.kept;
}
