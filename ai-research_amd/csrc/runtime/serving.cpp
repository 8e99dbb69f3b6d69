// serving.cpp -- entry points of batched serving: the paged 8-bit K/V cache
// (append, read-back, attention), probabilities from logits, and the verification
// of drafted tokens.  Argument checks, launch shapes, and the launch on the
// context stream.  Nothing here allocates: a caller gives the workspace.
#include <float.h>
#include <math.h>

#include <new>
#include <string>

#include "../common/kv8_args.h"
#include "../common/sample_args.h"
#include "runtime.hpp"

using gh::fail;

namespace {

// No exception leaves a C entry.
template <typename F>
gh_status guarded(const char* who, F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(GH_ERR_ALLOC, "out of host memory");
  } catch (...) {
    return fail(GH_ERR_INVALID, who);
  }
}

gh_status invalid(const char* who, const char* what) { return fail(GH_ERR_INVALID, std::string(who) + ": " + what); }
gh_status unsupported(const char* who, const char* what) {
  return fail(GH_ERR_UNSUPPORTED, std::string(who) + ": " + what);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The first launch of a kernel asks the code objects for it in turn; the answer
// "not found" of one stays behind as HIP's last error, which a host's other HIP
// code in this thread would take for its own.  An error that was pending before is the
// host's, and stays.
gh_status launch(gh_context* ctx, const char* name, dim3 grid, dim3 block, unsigned lds, void** args) {
  const bool clean = hipPeekAtLastError() == hipSuccess;
  const hipFunction_t f = ctx->fn(name);
  if (clean && hipPeekAtLastError() == hipErrorNotFound) (void)hipGetLastError();
  if (!f) return fail(GH_ERR_CODE_OBJECT, std::string("kernel not found in the code objects: ") + name);
  return ctx->launch(name, grid, block, lds, args);
}

constexpr uint32_t kMaxRows = 1000000u, kMaxGrid = 65535u;

gh_status check_cache(const char* who, const gh_kv8_cache* c, Kv8View* v) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return invalid(who, "cache is null or has a null pointer");
  if (c->num_pages == 0 || c->num_kv == 0 || c->head_dim == 0) return invalid(who, "cache has a zero size");
  if (c->num_pages == 0xffffffffu) return unsupported(who, "num_pages must be below 2^32 - 1");
  if (c->page_tokens < KV8_BLOCK || c->page_tokens > 256 || (c->page_tokens & (c->page_tokens - 1)))
    return unsupported(who, "page_tokens must be 16, 32, 64, 128 or 256");
  if (c->head_dim % 16 || c->head_dim > 512) return unsupported(who, "head_dim must be a multiple of 16 up to 512");
  if (c->num_kv > 4096) return unsupported(who, "more than 4096 kv heads");
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
    return invalid(who, "cache codes must be 16-byte aligned, scales 4-byte");
  if ((uint64_t)c->num_pages * c->num_kv * (c->page_tokens / KV8_BLOCK) >= 1ull << 32)
    return unsupported(who, "the cache has 2^32 blocks or more");
  uint32_t shift = 4;
  while ((1u << shift) < c->page_tokens) shift++;
  *v = Kv8View{static_cast<int8_t*>(c->k), static_cast<int8_t*>(c->v), c->k_scale, c->v_scale, c->num_pages, shift,
               c->num_kv, c->head_dim};
  return GH_OK;
}

gh_status check_batch(const char* who, const gh_kv8_batch* b, Kv8Rows* r) {
  if (!b) return invalid(who, "batch is null");
  *r = Kv8Rows{b->seq_start, b->past, b->pages, b->num_seqs, b->max_pages, b->num_rows, b->max_rows};
  if (b->num_seqs == 0 || b->num_rows == 0 || b->max_rows == 0) return GH_OK;  // nothing to do
  if (!b->seq_start || !b->past || !b->pages) return invalid(who, "batch has a null pointer");
  if (b->max_pages == 0) return invalid(who, "max_pages is zero");
  if (!aligned(b->seq_start, 4) || !aligned(b->past, 4) || !aligned(b->pages, 4))
    return invalid(who, "batch arrays must be 4-byte aligned");
  if (b->num_seqs > kMaxGrid) return unsupported(who, "more than 65535 sequences");
  if (b->num_rows > kMaxRows) return unsupported(who, "more than 1000000 rows");
  r->max_rows = std::min(b->max_rows, b->num_rows);
  return GH_OK;
}

bool empty(const Kv8Rows& r) { return r.num_seqs == 0 || r.num_rows == 0 || r.max_rows == 0; }

// Blocks that a sequence's rows can touch.
uint32_t touched(const Kv8Rows& r) { return (r.max_rows + KV8_BLOCK - 2) / KV8_BLOCK + 1; }

// Of heads of up to 64 nl dims the kernels have variants.
uint32_t dims64(const Kv8View& c) { return c.D <= 64 ? 1 : c.D <= 128 ? 2 : c.D <= 256 ? 4 : 8; }

struct AttnPlan {
  bool rows = false;  // the kernel of many columns
  bool stream = false;
  uint32_t tiles = 0, nsplit = 1, chunk = 1;
  size_t bytes = 0;
};

// Which kernel, and into how many parts each sequence's tokens are split.
//
// The kernel of many columns halves what is read and converted a column, and wants many
// workgroups: it is taken where several tiles of 16 columns a sequence alone give every CU
// two of them.
// (us with it and with the other one, 8 key heads of 256 under 16 query heads: prompts
// of 2000 tokens 107 / 121, 700: 32 / 32, 8 of 64 rows over 1000: 45 / 49, over 4000: 133
// / 169; with fewer tiles, a prompt of 500: 26 / 20, 8 of 32 over 2000: 71 / 44; with one
// tile, 100 single rows over 500 - 3000: 176 / 135.)
//
// The other one splits the tokens where that shortens the whole: its four waves take
// steps of 32 tokens in turn, 2.3 us for a step each (256 dims; 0.6 more of that for
// every workgroup that some CU has beyond one), and the splits' sums cost a launch and their
// way through memory, 4 us and 3 TB/s.  (One token over 544, 8 heads: 5 splits 11.2 us,
// none 13.6; 8 sequences of 32 rows over 2000, 256 tiles: none 44, 2 61; a prompt of 256
// tokens, 256 tiles: none 11, 2 23; 32 sequences of 20 - 4000 tokens, 256 tiles: 2 60,
// none 70; 8 of 5 rows over 1000 - 3000, 64 tiles: 8 24, none 47.  The estimate is for loads
// through the caches, and can be a tenth off for those by them: the 32 sequences take 57
// with 3, and of 4000 tokens each 87 with none against 92.)  Parts are of equal
// length in tokens, so that long sequences of a batch take more of them than short ones.
// They are at most as many as two workgroups a CU, which even out lengths that differ; one
// a CU where there is one sequence and tile (one row over 120000 tokens: 85 us with one, 89
// with two; over 30000: 31 and 32).
//
// Codes that one tile reads once, and that are too many to be in the last-level cache
// (256 MB) at the next call, pass by the caches: from 96 MB on, going by the bounds.  (One
// row over 120000, 492 MB: 85 us by them and 98 through them; 16 sequences over 2000,
// 131 MB: 30 and 34; 8 over 2000, 65 MB, the same three caches in turn: 21 and 20.)
gh_status plan_attn(const char* who, const gh_context* ctx, const Kv8View& c, const Kv8Rows& r, uint32_t num_q,
                    uint32_t window, uint32_t max_kv, AttnPlan* p) {
  if (num_q == 0 || num_q % c.nkv) return invalid(who, "num_q must be a positive multiple of the kv heads");
  if (num_q > 65536) return unsupported(who, "more than 65536 query heads");
  *p = AttnPlan{};
  if (empty(r)) return GH_OK;
  const uint64_t G = num_q / c.nkv, cols = r.max_rows * G, cus = std::max(ctx->num_cus, 1);
  uint64_t tiles = (cols + KV8_COLS - 1) / KV8_COLS, units = tiles * c.nkv * r.num_seqs;
  p->rows = tiles > 1 && units >= 2 * cus;
  if (p->rows) tiles = (cols + KV8_ROW_COLS - 1) / KV8_ROW_COLS;
  // (a grid holds less than 2^32 threads along x)
  if (tiles * c.nkv >= 1ull << 24) return unsupported(who, "2^29 or more query columns");
  p->tiles = (uint32_t)tiles;
  if (p->rows) return GH_OK;
  // (tokens are numbered in 32 bits: a table of more pages has no use for them, and the parts'
  // steps are counted in as many)
  uint64_t tokens = std::min<uint64_t>((uint64_t)r.max_pages << c.page_shift, (1ull << 32) + r.max_rows);
  if (max_kv) tokens = std::min<uint64_t>(tokens, max_kv);
  if (window) tokens = std::min<uint64_t>(tokens, (uint64_t)window + (KV8_COLS + G - 1) / G);
  const uint64_t steps = tokens / KV8_STEP + 1;
  const uint64_t a_cu = tiles == 1 && r.num_seqs == 1 ? 1 : 2;
  const uint64_t most = std::min<uint64_t>({(steps + 3) / 4, a_cu * cus / units, KV8_MAX_SPLIT});
  double least = INFINITY;
  for (uint64_t n = 1; n <= std::max<uint64_t>(most, 1); n++) {
    const double turns = (double)(((steps + n - 1) / n + 3) / 4), each = 2.3 * std::max(0.5, c.D / 256.0);
    const double load = 1 + 0.6 * (double)((units * n - 1) / cus);
    const double join = n > 1 ? 4 + (double)(units * n) * c.D * (2 * sizeof(float) * KV8_COLS) / 3e6 : 0;
    const double us = turns * each * load + join;
    if (us < least) {
      least = us;
      p->nsplit = (uint32_t)n;
    }
  }
  p->chunk = (uint32_t)((steps + p->nsplit - 1) / p->nsplit);
  p->stream = tiles == 1 && units * steps >= (96ull << 20) / (2 * KV8_STEP * c.D);
  if (p->nsplit > 1) p->bytes = (size_t)units * p->nsplit * KV8_COLS * (c.D + KV8_PART) * sizeof(float);
  return GH_OK;
}

// Elements of a thread in the sampling kernels: 16, or 4 while that gives fewer
// workgroups than CUs (one row of 262144, least times of the two launches: probabilities
// 2.7 + 3.0 us with 4 a thread, 3.1 + 4.0 with 16; verification 3.2 + 2.6 and 3.5 + 4.3;
// the calls take 7 and 8 us, what a host needs to launch them.  40 rows: 26 us with 4, 20 with
// 16; verification of 32: 22 and 18).
uint32_t sample_each(const gh_context* ctx, uint32_t rows, uint32_t vocab) {
  const uint64_t many = (vocab + 256ull * SAMPLE_MANY - 1) / (256 * SAMPLE_MANY);
  return rows * many < (uint64_t)ctx->num_cus ? SAMPLE_FEW : SAMPLE_MANY;
}
uint32_t chunks_of(uint32_t vocab, uint32_t each) { return (uint32_t)((vocab + 256ull * each - 1) / (256 * each)); }

gh_status check_work(const char* who, const void* work, size_t have, size_t need) {
  if (need == 0) return GH_OK;
  if (!work || have < need) return invalid(who, "workspace is null or smaller than the workspace function says");
  if (!aligned(work, 16)) return invalid(who, "workspace must be 16-byte aligned");
  return GH_OK;
}

}  // namespace

extern "C" {

size_t gh_kv8_code_bytes(const gh_kv8_cache* c) {
  return c ? (size_t)c->num_pages * c->page_tokens * c->num_kv * c->head_dim : 0;
}
size_t gh_kv8_scale_bytes(const gh_kv8_cache* c) {
  return c ? (size_t)c->num_pages * (c->page_tokens / KV8_BLOCK) * c->num_kv * sizeof(float) : 0;
}

gh_status gh_kv8_append(gh_context* ctx, const gh_kv8_cache* cache, const gh_kv8_batch* batch, const float* Q_in,
                        const float* K_in, const float* V_in, uint32_t q_stride, uint32_t kv_stride,
                        const float* Q_norm, const float* K_norm, float* Q_out, uint32_t num_q, uint32_t rotary_dim,
                        uint32_t k_eq_v, float theta, float eps) {
  return guarded("gh_kv8_append", [&]() -> gh_status {
    const char* who = "gh_kv8_append";
    if (!ctx) return invalid(who, "ctx is null");
    Kv8AppendArgs a{};
    gh_status st = check_cache(who, cache, &a.c);
    if (st != GH_OK) return st;
    if ((st = check_batch(who, batch, &a.b)) != GH_OK) return st;
    if (rotary_dim > a.c.D || rotary_dim % 2) return invalid(who, "rotary_dim must be even and at most head_dim");
    if (!(theta > 0.f) || !(theta < INFINITY)) return invalid(who, "theta must be positive");
    if (!(eps >= 0.f) || !(eps < INFINITY)) return invalid(who, "eps must not be negative");
    if (num_q > 65536) return unsupported(who, "more than 65536 query heads");
    if (empty(a.b)) return GH_OK;
    if (!K_in || !K_norm || (!V_in && !k_eq_v)) return invalid(who, "K_in, V_in or K_norm is null");
    if (num_q && (!Q_in || !Q_norm || !Q_out)) return invalid(who, "Q_in, Q_norm or Q_out is null");
    if (kv_stride < (uint64_t)a.c.nkv * a.c.D || (num_q && q_stride < (uint64_t)num_q * a.c.D))
      return invalid(who, "a row stride is shorter than its heads");
    if (num_q && Q_out == Q_in && q_stride != (uint64_t)num_q * a.c.D && a.b.num_rows > 1)
      return invalid(who, "Q_out is Q_in with rows that are not num_q * head_dim apart");
    if (num_q && (Q_out == K_in || (Q_out == V_in && !k_eq_v))) return invalid(who, "Q_out is K_in or V_in");
    for (const void* p : {(const void*)Q_in, (const void*)K_in, (const void*)V_in, (const void*)Q_norm,
                          (const void*)K_norm, (const void*)Q_out})
      if (!aligned(p, 4)) return invalid(who, "rows and norms must be 4-byte aligned");
    a.q = Q_in;
    a.k = K_in;
    a.v = V_in ? V_in : K_in;
    a.qn = Q_norm;
    a.kn = K_norm;
    a.qo = Q_out;
    a.qs = q_stride;
    a.kvs = kv_stride;
    a.nq = num_q;
    a.rot = rotary_dim;
    a.k_eq_v = k_eq_v ? 1 : 0;
    a.eps = eps;
    const long double log = rotary_dim ? -2 * log2l((long double)theta) / rotary_dim : 0;
    a.log_hi = (double)log;
    a.log_lo = (double)(log - a.log_hi);
    const uint32_t rows = std::min(a.b.max_rows, KV8_BLOCK);
    const unsigned lds = 32 + KV8_BLOCK * a.c.D + rows * (rotary_dim / 2) * 16;
    const dim3 grid(2 * a.c.nkv + (num_q + KV8_Q_HEADS - 1) / KV8_Q_HEADS, touched(a.b), a.b.num_seqs);
    const char* name = a.c.D <= 128 ? "gh_kv8_append_p1_k" : a.c.D <= 256 ? "gh_kv8_append_p2_k" : "gh_kv8_append_p4_k";
    void* args[] = {&a};
    return launch(ctx, name, grid, dim3(256), lds, args);
  });
}

gh_status gh_kv8_read(gh_context* ctx, const gh_kv8_cache* cache, const gh_kv8_batch* batch, float* K_out,
                      float* V_out) {
  return guarded("gh_kv8_read", [&]() -> gh_status {
    const char* who = "gh_kv8_read";
    if (!ctx) return invalid(who, "ctx is null");
    Kv8ReadArgs a{};
    gh_status st = check_cache(who, cache, &a.c);
    if (st != GH_OK) return st;
    if ((st = check_batch(who, batch, &a.b)) != GH_OK) return st;
    if (!K_out && !V_out) return invalid(who, "K_out and V_out are null");
    if (!aligned(K_out, 4) || !aligned(V_out, 4)) return invalid(who, "rows must be 4-byte aligned");
    if (empty(a.b)) return GH_OK;
    a.k = K_out;
    a.v = V_out;
    a.wide = aligned(K_out, 16) && aligned(V_out, 16);
    void* args[] = {&a};
    return launch(ctx, "gh_kv8_read_k", dim3(a.c.nkv, touched(a.b), a.b.num_seqs), dim3(256), 0, args);
  });
}

size_t gh_kv8_attn_workspace(const gh_context* ctx, const gh_kv8_cache* cache, const gh_kv8_batch* batch,
                             uint32_t num_q, uint32_t window, uint32_t max_kv) {
  size_t bytes = 0;
  guarded("gh_kv8_attn_workspace", [&]() -> gh_status {
    const char* who = "gh_kv8_attn_workspace";
    if (!ctx) return invalid(who, "ctx is null");
    Kv8View c;
    Kv8Rows r;
    AttnPlan p;
    gh_status st = check_cache(who, cache, &c);
    if (st == GH_OK) st = check_batch(who, batch, &r);
    if (st == GH_OK) st = plan_attn(who, ctx, c, r, num_q, window, max_kv, &p);
    bytes = p.bytes;
    return st;
  });
  return bytes;
}

gh_status gh_kv8_attn(gh_context* ctx, const gh_kv8_cache* cache, const gh_kv8_batch* batch, const float* Q,
                      float* out, uint32_t num_q, float scale, uint32_t window, uint32_t max_kv, void* work,
                      size_t work_bytes) {
  return guarded("gh_kv8_attn", [&]() -> gh_status {
    const char* who = "gh_kv8_attn";
    if (!ctx) return invalid(who, "ctx is null");
    Kv8AttnArgs a{};
    AttnPlan p;
    gh_status st = check_cache(who, cache, &a.c);
    if (st != GH_OK) return st;
    if ((st = check_batch(who, batch, &a.b)) != GH_OK) return st;
    if ((st = plan_attn(who, ctx, a.c, a.b, num_q, window, max_kv, &p)) != GH_OK) return st;
    if (!(fabsf(scale) < INFINITY)) return invalid(who, "scale must be finite");
    if (empty(a.b)) return GH_OK;
    if (!Q || !out) return invalid(who, "Q or out is null");
    if (!aligned(Q, 16) || !aligned(out, 16)) return invalid(who, "Q and out must be 16-byte aligned");
    if ((st = check_work(who, work, work_bytes, p.bytes)) != GH_OK) return st;
    a.q = Q;
    a.out = out;
    a.part = static_cast<float*>(work);
    a.nq = num_q;
    a.window = window;
    a.nsplit = p.nsplit;
    a.chunk = p.chunk;
    a.scale = scale;
    const uint32_t nl = dims64(a.c);
    // r: heads of fewer dims than the kernel's 64 nl; s: codes by the caches
    const std::string name = std::string(p.rows ? "gh_kv8_rows_l" : "gh_kv8_attn_l") + std::to_string(nl) +
                             (a.c.D == 64 * nl ? "" : "r") + (p.stream ? "s_k" : "_k");
    void* args[] = {&a};
    if (p.rows) return launch(ctx, name.c_str(), dim3(p.tiles * a.c.nkv, 1, a.b.num_seqs), dim3(256), 14336 * nl, args);
    st = launch(ctx, name.c_str(), dim3(p.tiles * p.nsplit, a.c.nkv, a.b.num_seqs), dim3(256),
                KV8_ATTN_HEAD + 16384 * nl, args);
    if (st != GH_OK || p.nsplit == 1) return st;
    uint32_t cols = (uint32_t)std::min<uint64_t>(KV8_COLS, (uint64_t)a.b.max_rows * (num_q / a.c.nkv));
    void* margs[] = {&a, &cols};
    return launch(ctx, "gh_kv8_merge_k", dim3(p.tiles * cols, a.c.nkv, a.b.num_seqs), dim3(256), 0, margs);
  });
}

size_t gh_logit_probs_workspace(const gh_context* ctx, uint32_t rows, uint32_t vocab) {
  return ctx ? (size_t)rows * chunks_of(vocab, sample_each(ctx, rows, vocab)) * 2 * sizeof(float) : 0;
}

gh_status gh_logit_probs(gh_context* ctx, const float* logits, float* probs, uint32_t rows, uint32_t vocab,
                         uint32_t stride, float softcap, float temperature, void* work, size_t work_bytes) {
  return guarded("gh_logit_probs", [&]() -> gh_status {
    const char* who = "gh_logit_probs";
    if (!ctx) return invalid(who, "ctx is null");
    if (stride < vocab) return invalid(who, "stride is shorter than a row");
    if (!(softcap >= 0.f) || !(softcap < INFINITY)) return invalid(who, "softcap must be 0 (none) or positive");
    if (!(temperature > 0.f) || !(temperature < INFINITY)) return invalid(who, "temperature must be positive");
    if (rows > kMaxGrid) return unsupported(who, "more than 65535 rows");
    // (the second launch's workgroups each join all chunks of their row)
    if (vocab > 1u << 24) return unsupported(who, "vocab above 2^24");
    if (rows == 0 || vocab == 0) return GH_OK;
    if (!logits || !probs) return invalid(who, "logits or probs is null");
    if (!aligned(logits, 4) || !aligned(probs, 4)) return invalid(who, "rows must be 4-byte aligned");
    gh_status st = check_work(who, work, work_bytes, gh_logit_probs_workspace(ctx, rows, vocab));
    if (st != GH_OK) return st;
    const uint32_t each = sample_each(ctx, rows, vocab);
    double mul = 1.4426950408889634 / (double)temperature * (softcap > 0.f ? (double)softcap : 1.0);
    // (soft-capped logits lie within 2 of each other in units of the cap: a factor below f32's
    // normal range makes them all even, as that range's least does; 0 would make masked ones NaN)
    if (softcap > 0.f) mul = std::max(mul, (double)FLT_MIN);
    ProbsArgs a{logits, probs, static_cast<float*>(work), stride, vocab, chunks_of(vocab, each),
                softcap > 0.f ? 1.f / softcap : 0.f, (float)mul};
    if (!(a.mul < INFINITY)) return invalid(who, "softcap / temperature is too large");
    if (!(a.inv_cap < INFINITY)) return invalid(who, "softcap is too small");
    const bool vec = vocab % 4 == 0 && stride % 4 == 0 && aligned(logits, 16) && aligned(probs, 16);
    void* args[] = {&a};
    const dim3 grid(a.chunks, rows);
    const std::string form = "_n" + std::to_string(each) + (vec ? "_v4_k" : "_v1_k");
    st = launch(ctx, ("gh_probs_part" + form).c_str(), grid, dim3(256), 0, args);
    if (st != GH_OK) return st;
    return launch(ctx, ("gh_probs_write" + form).c_str(), grid, dim3(256), 0, args);
  });
}

size_t gh_spec_verify_workspace(const gh_context* ctx, uint32_t num_seqs, uint32_t vocab) {
  return ctx ? (size_t)num_seqs * chunks_of(vocab, sample_each(ctx, num_seqs, vocab)) * 2 * sizeof(double) : 0;
}

gh_status gh_spec_verify(gh_context* ctx, const float* target, const float* draft, const uint32_t* tokens,
                         const uint32_t* n_draft, const float* u, const float* pick, uint32_t* out_tokens,
                         uint32_t* accepted, uint32_t num_seqs, uint32_t max_draft, uint32_t vocab, void* work,
                         size_t work_bytes) {
  return guarded("gh_spec_verify", [&]() -> gh_status {
    const char* who = "gh_spec_verify";
    if (!ctx) return invalid(who, "ctx is null");
    if (num_seqs > kMaxGrid) return unsupported(who, "more than 65535 sequences");
    if (max_draft > 65535) return unsupported(who, "more than 65535 drafted tokens");
    if (vocab == 0) return invalid(who, "vocab is zero");
    if (vocab > 0x7fffffffu) return unsupported(who, "vocab must be below 2^31");
    if (num_seqs == 0) return GH_OK;
    if (!target || !pick || !out_tokens || !accepted || (max_draft && (!tokens || !u)))
      return invalid(who, "null pointer");
    if (accepted == n_draft || out_tokens == tokens) return invalid(who, "accepted is n_draft, or out_tokens tokens");
    for (const void* p : {(const void*)target, (const void*)draft, (const void*)tokens, (const void*)n_draft,
                          (const void*)u, (const void*)pick, (const void*)out_tokens, (const void*)accepted})
      if (!aligned(p, 4)) return invalid(who, "arrays must be 4-byte aligned");
    gh_status st = check_work(who, work, work_bytes, gh_spec_verify_workspace(ctx, num_seqs, vocab));
    if (st != GH_OK) return st;
    const uint32_t each = sample_each(ctx, num_seqs, vocab);
    VerifyArgs a{target, draft, tokens, n_draft, u, pick, out_tokens, accepted, static_cast<double*>(work),
                 max_draft, vocab, chunks_of(vocab, each)};
    const bool vec = vocab % 4 == 0 && aligned(target, 16) && aligned(draft, 16);
    void* args[] = {&a};
    const std::string form = "_n" + std::to_string(each) + (vec ? "_v4_k" : "_v1_k");
    st = launch(ctx, ("gh_verify_part" + form).c_str(), dim3(a.chunks, num_seqs), dim3(256), 0, args);
    if (st != GH_OK) return st;
    return launch(ctx, ("gh_verify_token" + form).c_str(), dim3(num_seqs), dim3(256), 0, args);
  });
}

}  // extern "C"
