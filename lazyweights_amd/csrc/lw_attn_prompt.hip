// Attention of whole prompts, or chunks of them, over a paged key-value cache.
#include <algorithm>

#include "lw_attn_prompt.h"

namespace lw {

namespace {

// Parts of the weights: all of them for fp32 outputs; one for 16-bit ones, whose own rounding is larger than what a row's average
// shows of its weights' (1000 tokens after 9001, fp16: 2.2e-4 from 64 bits, 2.1e-4 where only the output is rounded; 15999 in bf16
// 1.8e-3 and 1.7e-3). 9000 tokens of 32 heads of 128: fp16 756 us with one, 998 with two, bf16 653 with one, 1114 with three.
template <int D, bool BF, int W>
hipError_t prompt_w(const AttnArgs& a, int splits, hipStream_t s) {
  const dim3 grid((uint32_t)(((int64_t)a.c.tokens * a.group / (32 * W) + a.c.seqs) * a.c.kv_heads * splits));
  if (a.out_type == 0 && a.most_run > kLongRun) k_attn_prompt<D, BF, BF ? 3 : 2, W, true, AttnArgs><<<grid, 64 * W, 0, s>>>(a);
  else if (a.out_type == 0) k_attn_prompt<D, BF, BF ? 3 : 2, W, false, AttnArgs><<<grid, 64 * W, 0, s>>>(a);
  else k_attn_prompt<D, BF, 1, W, false, AttnArgs><<<grid, 64 * W, 0, s>>>(a);
  return hipGetLastError();
}
template <int D, bool BF>
hipError_t prompt_d(const AttnArgs& a, hipStream_t s) {
  // 8 waves read each key tile for twice as many rows, but are twice as coarse: 5 % faster where there are at least 4 such
  // blocks for every CU (15999 tokens of 32 heads 2137 us against 2241), slower below (766 blocks of ragged prompts 148
  // against 133, 125 blocks 133 against 107)
  const int64_t blocks = (int64_t)a.c.tokens * a.group / 256 * a.c.kv_heads;
  if (blocks >= 1024) return prompt_w<D, BF, 8>(a, 1, s);
  hipError_t e = prompt_w<D, BF, 4>(a, a.splits, s);
  if (e == hipSuccess && a.splits > 1) {
    k_attn_join<D><<<dim3((uint32_t)prompt_items(a.c.seqs, a.c.kv_heads, a.group, a.c.tokens) * (D / 32)), 256, 0, s>>>(a);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace

int64_t prompt_items(int seqs, int kv_heads, int group, int tokens) {
  return ((int64_t)tokens * group / 128 + seqs) * kv_heads;
}

size_t prompt_slot_bytes(int head_dim) { return (size_t)128 * (head_dim + 4) * 4; }

int prompt_splits(int seqs, int kv_heads, int group, int tokens, int max_kv, int64_t slots, int least) {
  // Two blocks per CU, of 1024 keys and more, where that makes `least` at least of every row tile's, three of 16 bits: us with / without, the join
  // included, 64 tokens after 20000 59 / 504, 500 after 3000 52 / 89; two shares of 256 row tiles gain nothing (1000 tokens
  // after 9001 100 / 106, their sums' way through memory takes 13), nor do few keys (700 tokens 27 / 25). Of 8 bits, whose tiles pass through registers and are longer on their way, two do:
  // the same 103 / 127.
  const int64_t items = prompt_items(seqs, kv_heads, group, tokens);
  const int64_t splits = std::min<int64_t>(std::min<int64_t>(kPromptSlots, slots) / items, max_kv / 1024);
  return splits < least ? 1 : (int)splits;
}

hipError_t launch_attn_prompt(const AttnArgs& a, int head_dim, int type, hipStream_t s) {
  if (head_dim == 64) return type == 2 ? prompt_d<64, true>(a, s) : prompt_d<64, false>(a, s);
  if (head_dim == 96) return type == 2 ? prompt_d<96, true>(a, s) : prompt_d<96, false>(a, s);
  return type == 2 ? prompt_d<128, true>(a, s) : prompt_d<128, false>(a, s);
}

}  // namespace lw
