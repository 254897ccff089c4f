// Attention over a paged key-value cache: arguments of the kernels and their launchers (host interface of
// lw_attn_decode.hip and lw_attn_prompt.hip; the C-ABI in lw_attn_api.cpp checks what a caller gives and fills these).
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <string>

namespace lw {

// Sets lw_last_error() of the calling thread.
void set_error(const std::string& m);

// The cache and the batch, as every kernel takes them. Key j of sequence s is row j & (2^page_shift - 1) of page
// table[s * tstride + (j >> page_shift)]; a page outside [0, pages) holds no keys. The batch's rows are its new tokens:
// those of sequence s are [q_start[s], q_start[s + 1]), its last ones, so row t has position kv_len[s] - q_start[s + 1] + t.
struct KvView {
  uint16_t *k, *v;
  int64_t pstride, hstride, rstride;  // elements from a page, a head, a row to the next
  const int32_t *q_start, *kv_len, *table;
  int64_t tstride;
  uint32_t pages;
  int page_shift, table_pages;
  int kv_heads, seqs, tokens;
};

struct AppendArgs {
  KvView c;
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv, ldo;
  uint16_t* q_out;
  const float *cos, *sin;  // [rope_rows][rot / 2]
  int heads, rot, rope_rows, neighbours;
};

// x / d for 0 <= x < 2^31 as a product and a shift: the product of x and ceil(2^(31 + k) / d), 2^k the power of two at or
// above d, is less than 2^31 too large
struct Divisor {
  uint64_t mul;
  int shift;
  __host__ __device__ int operator()(int x) const { return (int)(((uint64_t)(uint32_t)x * mul) >> shift); }
};
inline Divisor divisor(int d) {
  int k = 0;
  while ((1u << k) < (uint32_t)d) ++k;
  return {(((uint64_t)1 << (31 + k)) + d - 1) / d, 31 + k};
}

struct AttnArgs {
  KvView c;
  const uint16_t* q;
  void* out;
  int64_t ldq, ldo;
  int out_type;
  int heads, group;  // group = heads / kv_heads
  Divisor by_group;
  float scale;       // of the scores, times log2(e) (weights are powers of two), positive
  uint32_t q_flip;   // the sign bits of two elements where the caller's scale is negative: q is negated instead
  int window;        // > 0: a row sees its last `window` positions
  // the decode kernel's workspace and division (DecodePlan)
  float* part;
  uint32_t* count;
  int row_blocks, blocks_log2, most_keys, whole;
  // the prompt kernel's
  int splits;    // blocks that share the keys of a row tile, their sums in `part`
  int most_run;  // about as many keys as one block goes through, at most
};

// How the decode kernel divides a batch: row_tiles tiles of 16 (token, head) rows per item, row_blocks items for a
// sequence's key-value head, and a power of two of blocks. The list of all items' tiles of 32 keys is counted in 32 bits:
// most_keys is the most of a sequence that keeps it there (2^31 tiles in all).
struct DecodePlan {
  int row_tiles, row_blocks, blocks, blocks_log2, most_keys;
  bool whole;  // a block per item, of 8 waves
  size_t count_bytes, part_bytes;  // workspace: counters (zero before and after a launch), then partials
};
DecodePlan decode_plan(int seqs, int kv_heads, int group, int head_dim, int max_new, int max_kv);

// The prompt kernel's row tiles of 128 (token, head) rows of a key-value head, and into how many blocks the keys of each are shared
// out, with a workspace of `slots` slots of prompt_slot_bytes() each (kPromptSlots are of use).
// Runs of more than kLongRun keys are summed with more care for fp32 outputs.
constexpr int kPromptSlots = 512, kLongRun = 16384;
int64_t prompt_items(int seqs, int kv_heads, int group, int tokens);
size_t prompt_slot_bytes(int head_dim);
int prompt_splits(int seqs, int kv_heads, int group, int tokens, int max_kv, int64_t slots);

hipError_t launch_append(const AppendArgs& a, int head_dim, int type, int x_type, hipStream_t s);
hipError_t launch_attn_decode(const AttnArgs& a, const DecodePlan& p, int head_dim, int type, hipStream_t s);
hipError_t launch_attn_prompt(const AttnArgs& a, int head_dim, int type, hipStream_t s);

}  // namespace lw
