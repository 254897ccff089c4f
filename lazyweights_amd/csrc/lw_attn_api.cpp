// C-ABI of the attention over a paged key-value cache (include/lazyweights_amd.h): checks of what a caller gives, kernel
// arguments, launches. The lengths and pages a batch's arrays hold are known on the GPU only; the kernels keep them in
// range.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/lazyweights_amd.h"
#include "lw_attention.h"

namespace {

int refuse(const char* fn, const std::string& why) {
  lw::set_error(std::string(fn) + ": " + why);
  return -1;
}

constexpr long long kMostBlocks = 0xFFFFFFFFll / 256;  // of 256 threads, along one dimension of a launch
constexpr long long kMostRows = 1 << 30;             // rows of a batch, (row, head) pairs, positions of a sequence

bool aligned(const void* p, long long stride) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0; }

// the cache's and the batch's own members, and heads; "" if they are fine
std::string check(const lw_kv_cache* c, const lw_batch* b, int heads) {
  if (!c || !b) return "no cache or no batch";
  if (c->type != LW_F16 && c->type != LW_BF16) return "the cache's type must be LW_F16 or LW_BF16";
  if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128) return "head_dim must be 64, 96 or 128";
  if (c->page_size < 1 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
    return "page_size must be a power of two up to 65536";
  if (c->pages < 0 || c->pages > 0x7FFFFFFF) return "pages out of range";
  if (c->kv_heads < 1 || heads < 1 || heads % c->kv_heads || heads > 65535) return "heads must be a multiple of kv_heads";
  if (c->pages > 0 && (!c->k || !c->v)) return "no cache memory";
  if (!aligned(c->k, c->page_stride) || !aligned(c->v, c->head_stride) || c->row_stride % 8)
    return "the cache must be aligned to 16 bytes, with strides of multiples of 8 elements";
  if (c->page_stride < 0 || c->head_stride < 0 || c->row_stride < 0) return "negative cache stride";
  if (b->seqs < 0 || b->seqs > 65535 || b->tokens < 0 || b->max_new < 0 || b->max_kv < 0 || b->table_pages < 0)
    return "negative batch size, or more than 65535 sequences";
  if (b->reserved) return "reserved must be 0";
  if (b->seqs > 0 && (!b->q_start || !b->kv_len || (b->table_pages > 0 && !b->page_table))) return "null batch array";
  if ((long long)b->tokens * heads > kMostRows) return "more than 2^30 rows and heads";
  if ((long long)b->table_pages * c->page_size > kMostRows) return "the page table holds more than 2^30 positions";
  if (b->table_stride < b->table_pages) return "table_stride is less than table_pages";
  if (b->max_kv > (long long)b->table_pages * c->page_size) return "max_kv is more than the page table holds";
  return "";
}

lw::KvView view(const lw_kv_cache& c, const lw_batch& b) {
  lw::KvView v;
  v.k = static_cast<uint16_t*>(c.k);
  v.v = static_cast<uint16_t*>(c.v);
  v.pstride = c.page_stride;
  v.hstride = c.head_stride;
  v.rstride = c.row_stride;
  v.q_start = b.q_start;
  v.kv_len = b.kv_len;
  v.table = b.page_table;
  v.tstride = b.table_stride;
  v.pages = (uint32_t)c.pages;
  v.page_shift = __builtin_ctz((unsigned)c.page_size);
  v.table_pages = b.table_pages;
  v.kv_heads = c.kv_heads;
  v.seqs = b.seqs;
  v.tokens = b.tokens;
  return v;
}

int launched(const char* fn, hipError_t e) {
  return e == hipSuccess ? 0 : refuse(fn, std::string("launch failed: ") + hipGetErrorString(e));
}

// decode and prompt alike; 1: nothing to do
int attention_args(const char* fn, const lw_kv_cache* cache, const lw_batch* batch, int heads, const void* q, long long ldq,
                   void* out, int out_type, long long ldo, float scale, int window, lw::AttnArgs& a) {
  const std::string bad = check(cache, batch, heads);
  if (!bad.empty()) return refuse(fn, bad);
  if (out_type != LW_F32 && out_type != LW_F16 && out_type != LW_BF16) return refuse(fn, "unknown type of out");
  if (!std::isfinite(scale)) return refuse(fn, "scale is not finite");
  if (window < 0) return refuse(fn, "negative window");
  if (batch->seqs == 0 || batch->tokens == 0) return 1;
  if (!q || !out) return refuse(fn, "null buffer");
  if (!aligned(q, ldq) || !aligned(out, ldo) || ldq < (long long)heads * cache->head_dim ||
      ldo < (long long)heads * cache->head_dim)
    return refuse(fn, "q and out must be aligned to 16 bytes, with row strides of multiples of 8 that hold their heads");
  a.c = view(*cache, *batch);
  // (where a page is not there the kernels load the first page's keys instead and leave them out: of no pages there is no first, so
  // no sequence has keys, and all rows are zeros)
  if (cache->pages == 0) a.c.table_pages = 0;
  a.q = static_cast<const uint16_t*>(q);
  a.out = out;
  a.ldq = ldq;
  a.ldo = ldo;
  a.out_type = out_type;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.by_group = lw::divisor(a.group);
  // (0 stands for the least normal number and more: products with it are 0 to any purpose, and -infinity, which marks what a
  // row does not see, stays what it is)
  a.scale = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-37f);
  a.q_flip = scale < 0 ? 0x80008000u : 0;
  a.window = (int)std::min<long long>(window, kMostRows);
  a.part = nullptr;
  a.count = nullptr;
  a.row_blocks = a.blocks_log2 = a.most_keys = a.whole = 0;
  a.splits = 1;
  a.most_run = 0;
  return 0;
}

}  // namespace

extern "C" {

long long lw_attn_workspace(const lw_kv_cache* cache, const lw_batch* batch, int heads) {
  const std::string bad = check(cache, batch, heads);
  if (!bad.empty()) return refuse("lw_attn_workspace", bad);
  if (batch->seqs == 0) return 0;
  if (batch->max_new > 16)  // (a row tile's keys are shared out where there are three times 1024 and more)
    return batch->max_kv < 3 * 1024 ? 0 : (long long)(lw::kPromptSlots * lw::prompt_slot_bytes(cache->head_dim));
  const lw::DecodePlan p = lw::decode_plan(batch->seqs, cache->kv_heads, heads / cache->kv_heads, cache->head_dim,
                                           batch->max_new, batch->max_kv);
  return (long long)(p.count_bytes + p.part_bytes);
}

int lw_kv_append(const lw_kv_cache* cache, const lw_batch* batch, int heads, const void* q, const void* k, const void* v,
                 int x_type, long long ldq, long long ldk, long long ldv, const float* cos, const float* sin, int rot,
                 int rope_rows, int neighbours, void* q_out, long long ldo, void* stream) {
  const char* fn = "lw_kv_append";
  const std::string bad = check(cache, batch, heads);
  if (!bad.empty()) return refuse(fn, bad);
  if (x_type != LW_F32 && x_type != LW_F16 && x_type != LW_BF16) return refuse(fn, "unknown type of q, k and v");
  if (neighbours != 0 && neighbours != 1) return refuse(fn, "neighbours must be 0 or 1");
  if (rot < 0 || rot > cache->head_dim || rot % 8) return refuse(fn, "rot must be a multiple of 8 up to head_dim");
  if (rot > 0 && (!cos || !sin || !aligned(cos, 0) || !aligned(sin, 0)))
    return refuse(fn, "cos and sin must be given, aligned to 16 bytes");
  if (rot > 0 && rope_rows < batch->max_kv) return refuse(fn, "cos and sin have fewer rows than max_kv");
  if (batch->seqs == 0 || batch->tokens == 0) return 0;
  const long long kd = (long long)cache->kv_heads * cache->head_dim, qd = (long long)heads * cache->head_dim;
  if (!k || !v || (q && !q_out)) return refuse(fn, "null buffer");
  if (!aligned(k, ldk) || !aligned(v, ldv) || ldk < kd || ldv < kd ||
      (q && (!aligned(q, ldq) || !aligned(q_out, ldo) || ldq < qd || ldo < qd)))
    return refuse(fn, "q, k, v and q_out must be aligned to 16 bytes, with row strides of multiples of 8 that hold their heads");
  const long long parts = (qd + 2 * kd + 8 * 256 - 1) / (8 * 256);
  if (parts * batch->tokens > kMostBlocks) return refuse(fn, "more tokens than a launch can take");
  lw::AppendArgs a;
  a.c = view(*cache, *batch);
  a.q = q;
  a.k = k;
  a.v = v;
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.ldo = ldo;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.cos = cos;
  a.sin = sin;
  a.heads = heads;
  a.rot = rot;
  a.rope_rows = rope_rows > 0 ? rope_rows : 1;
  a.neighbours = neighbours;
  return launched(fn, lw::launch_append(a, cache->head_dim, cache->type, x_type, static_cast<hipStream_t>(stream)));
}

int lw_attn_decode(const lw_kv_cache* cache, const lw_batch* batch, int heads, const void* q, long long ldq, void* out,
                   int out_type, long long ldo, float scale, int window, void* stream) {
  const char* fn = "lw_attn_decode";
  lw::AttnArgs a;
  const int rc = attention_args(fn, cache, batch, heads, q, ldq, out, out_type, ldo, scale, window, a);
  if (rc) return rc < 0 ? -1 : 0;
  if (batch->max_new < 1) return 0;
  if (batch->max_new > 16) return refuse(fn, "max_new is more than 16 (lw_attn_prompt takes any number)");
  const lw::DecodePlan p = lw::decode_plan(batch->seqs, cache->kv_heads, a.group, cache->head_dim, batch->max_new,
                                           batch->max_kv);
  if (p.most_keys < batch->max_kv) return refuse(fn, "more sequences, heads and positions than a launch can take");
  if (!batch->workspace || (reinterpret_cast<uintptr_t>(batch->workspace) & 15) ||
      batch->workspace_bytes < (long long)(p.count_bytes + p.part_bytes))
    return refuse(fn, "needs a workspace of " + std::to_string(p.count_bytes + p.part_bytes) + " bytes, aligned to 16");
  a.count = static_cast<uint32_t*>(batch->workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(batch->workspace) + p.count_bytes);
  a.row_blocks = p.row_blocks;
  a.blocks_log2 = p.blocks_log2;
  a.whole = p.whole;
  a.most_keys = p.most_keys;
  return launched(fn, lw::launch_attn_decode(a, p, cache->head_dim, cache->type, static_cast<hipStream_t>(stream)));
}

int lw_attn_prompt(const lw_kv_cache* cache, const lw_batch* batch, int heads, const void* q, long long ldq, void* out,
                   int out_type, long long ldo, float scale, int window, void* stream) {
  const char* fn = "lw_attn_prompt";
  lw::AttnArgs a;
  const int rc = attention_args(fn, cache, batch, heads, q, ldq, out, out_type, ldo, scale, window, a);
  if (rc) return rc < 0 ? -1 : 0;
  if (((long long)batch->tokens * a.group / 128 + batch->seqs) * cache->kv_heads > kMostBlocks)
    return refuse(fn, "more tokens than a launch can take");
  if (batch->workspace && (reinterpret_cast<uintptr_t>(batch->workspace) & 15)) return refuse(fn, "workspace not aligned to 16");
  if (batch->workspace) {  // (past the counters of lw_attn_decode, if the batch may go there)
    size_t skip = 0;
    if (batch->max_new <= 16)
      skip = lw::decode_plan(batch->seqs, cache->kv_heads, a.group, cache->head_dim, std::max(batch->max_new, 1), batch->max_kv)
                 .count_bytes;
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(batch->workspace) + skip);
    const long long bytes = batch->workspace_bytes - (long long)skip;
    if (bytes > 0)
      a.splits = lw::prompt_splits(batch->seqs, cache->kv_heads, a.group, batch->tokens, batch->max_kv,
                                   bytes / (long long)lw::prompt_slot_bytes(cache->head_dim));
  }
  const int most_kv = a.window > 0 ? std::min(batch->max_kv, a.window) : batch->max_kv;
  a.most_run = most_kv / a.splits;
  return launched(fn, lw::launch_attn_prompt(a, cache->head_dim, cache->type, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
