// Attention of whole prompts, or chunks of them, over a paged key-value cache held in 8 bits.
#include "lw_attn_prompt.h"

namespace lw {

namespace {

// Parts of the weights as for 16 bits: two (22 bits) for fp32 outputs, one (11 bits) for 16-bit ones, whose own rounding is larger than what
// a row's average shows of its weights' (1000 tokens after 9001, fp16: 2.14e-4 from 64 bits, 2.07e-4 where only the output is rounded;
// 15999 in bf16 1.650e-3 and 1.648e-3). Of fp16 whatever q's type, as V is: fp32 outputs with q in bf16 have 22 bits, where a bf16 cache has
// three parts, 24.
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
  // 8 waves where there is such a block for most of the CUs: a tile is converted for twice as many rows. us with 8 / 4 waves, 8 heads of 128
  // for 32, one prompt: 160 blocks (1300 tokens) 46 / 49, 224 60 / 62, 320 85 / 92, 496 152 / 180; 168 of 1400 after 3000 130 / 140; 7 ragged
  // prompts, 232 blocks 24.1 / 25.2; heads of 96, 224 blocks 56 / 62, of 64 46.5 / 46.9. fp32 outputs, whose products take longer than a
  // tile's conversion: 160 blocks 58 / 58, 320 113 / 112, 496 202 / 236, 712 of ragged prompts and heads of 96 135 / 149; the rule loses from
  // 224 (78 / 73) to 256 (94 / 89), where a second turn of large blocks begins.
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
