// Attention of whole prompts, or chunks of them, over a paged key-value cache held in 8 bits.
#include "lw_attn_prompt.h"

namespace lw {

namespace {

// Parts of the weights as for 16 bits: two (22 bits) for fp32 outputs, one for 16-bit ones, of fp16 whatever q's type.
template <int D, bool BF, int W>
hipError_t prompt8_w(const Attn8Args& args, int splits, hipStream_t s) {
  const AttnArgs& a = args.a;
  const dim3 grid((uint32_t)(((int64_t)a.c.tokens * a.group / (32 * W) + a.c.seqs) * a.c.kv_heads * splits));
  if (a.out_type == 0 && a.most_run > kLongRun) k_attn_prompt<D, BF, 2, W, true, Attn8Args><<<grid, 64 * W, 0, s>>>(args);
  else if (a.out_type == 0) k_attn_prompt<D, BF, 2, W, false, Attn8Args><<<grid, 64 * W, 0, s>>>(args);
  else k_attn_prompt<D, BF, 1, W, false, Attn8Args><<<grid, 64 * W, 0, s>>>(args);
  return hipGetLastError();
}
template <int D, bool BF>
hipError_t prompt8_d(const Attn8Args& args, hipStream_t s) {
  const AttnArgs& a = args.a;
  // 8 waves where there is such a block for most of the CUs: a tile is converted for twice as many rows (us with 8 / 4 waves: 712 blocks
  // of ragged prompts, 32 heads of 96, fp32 out 135 / 149; 500 of 4000 tokens, fp32 out 198 / 248; 187 of 1500 tokens 51 / 56; 175
  // of 1400 after 3000 129 / 140; 225 of 1800, fp32 out 77 / 73)
  const int64_t blocks = (int64_t)a.c.tokens * a.group / 256 * a.c.kv_heads;
  if (blocks >= 160) return prompt8_w<D, BF, 8>(args, 1, s);
  hipError_t e = prompt8_w<D, BF, 4>(args, a.splits, s);
  if (e == hipSuccess && a.splits > 1) {
    k_attn_join<D><<<dim3((uint32_t)prompt_items(a.c.seqs, a.c.kv_heads, a.group, a.c.tokens) * (D / 32)), 256, 0, s>>>(a);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace

hipError_t launch_attn8_prompt(const Attn8Args& a, int head_dim, int q_type, hipStream_t s) {
  if (head_dim == 64) return q_type == 2 ? prompt8_d<64, true>(a, s) : prompt8_d<64, false>(a, s);
  if (head_dim == 96) return q_type == 2 ? prompt8_d<96, true>(a, s) : prompt8_d<96, false>(a, s);
  return q_type == 2 ? prompt8_d<128, true>(a, s) : prompt8_d<128, false>(a, s);
}

}  // namespace lw
