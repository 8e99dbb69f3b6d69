// kv8_args.h -- argument blocks of the paged 8-bit K/V kernels (kv8.hip),
// shared with the host launcher (passed by value), and the split rule that the
// attention and its merge both apply.
#pragma once
#include <stdint.h>

#define KV8_BLOCK 16u      // tokens that share a scale, and rows of one matrix tile
#define KV8_STEP 32u       // tokens of one step of the attention
#define KV8_COLS 16u       // query columns of a wave (a row's heads of one kv head, row after row)
#define KV8_ROW_COLS 32u   // and of a workgroup of many columns
#define KV8_MAX_SPLIT 256u // parts of one tile's token range
#define KV8_PART 4u        // floats of a part's row behind its D sums: maximum, sum, unit, and one unused
#define KV8_ATTN_HEAD 768u // bytes of LDS before the few-column kernel's digits: maxima, sums and units
#define KV8_Q_HEADS 4u     // query heads of one append workgroup

// The cache (gh_kv8_cache); page_tokens = 1 << page_shift.
struct Kv8View {
  int8_t *k, *v;   // codes of a page's head: block after block, 16 D bytes each
  float *ks, *vs;  // [page][head][block]
  uint32_t num_pages, page_shift, nkv, D;
};

// The batch (gh_kv8_batch).
struct Kv8Rows {
  const uint32_t *seq_start, *past, *pages;
  uint32_t num_seqs, max_pages, num_rows, max_rows;
};

struct Kv8AppendArgs {
  Kv8View c;
  Kv8Rows b;
  const float *q, *k, *v, *qn, *kn;  // row strides: qs floats (q), kvs floats (k, v)
  float* qo;                         // [num_rows][nq D]
  uint64_t qs, kvs;
  uint32_t nq, rot, k_eq_v;
  float eps;
  double log_hi, log_lo;  // -2 log2(theta) / rot as the sum of two
};

struct Kv8ReadArgs {
  Kv8View c;
  Kv8Rows b;
  float *k, *v;  // [num_rows][nkv D], either may be null
  uint32_t wide;  // both 16-byte aligned
};

struct Kv8AttnArgs {
  Kv8View c;
  Kv8Rows b;
  const float* q;  // [num_rows][nq D]
  float* out;      // [num_rows][nq D]
  float* part;     // [tile][split][column][D + KV8_PART]; unused with one split
  uint32_t nq, window, nsplit, chunk;  // chunk: steps of a split at least
  float scale;
};

// Steps of a tile's token range that one split takes, so that at most nsplit
// splits (of at least `chunk` steps) cover it.
static inline
#ifdef __HIPCC__
    __host__ __device__
#endif
    uint32_t
    kv8_split_steps(uint32_t steps, uint32_t nsplit, uint32_t chunk) {
  const uint32_t even = (steps + nsplit - 1) / nsplit;
  return even > chunk ? even : chunk;
}
