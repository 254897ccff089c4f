// Attention of whole prompts, or chunks of them, over a paged key-value cache.
#include "lw_attn_device.h"

namespace lw {

namespace {

// ── prompt ──────────────────────────────────────────────────────────────────────────────────────────────────────────

// A block: 128 rows (token, head) of one key-value head of a sequence, 32 per wave, over the keys they see in tiles of 64.
// K and V tiles lie in LDS as [16-key block][D / 8 chunks][16 slots][8 dims], key k of a block in slot (k + 4 chunk) & 15:
// the score product's operand reads (32 keys of a chunk) and the transposed reads of V (4 keys of 4 chunks) are both free
// of bank conflicts. The next tile is loaded into registers while one is worked on.
template <int D, bool BF, int NP>
__global__ __launch_bounds__(256, 2) void k_attn_prompt(const AttnArgs a) {
  constexpr int C = D / 32, ROWS = 128, BLK = D * 16;  // BLK: elements of a 16-key block
  __shared__ __align__(16) uint16_t kl[2][4 * BLK], vl[2][4 * BLK];
  __shared__ uint16_t seen_l[2][4];
  __shared__ float care[4][16 * 32];  // weights of 16 keys x 32 rows of each wave, in the second pass
  __shared__ int any_bad;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, g = lane >> 5;
  const KvView& c = a.c;
  const int kvh = blockIdx.x % c.kv_heads, tile = (int)(gridDim.x / c.kv_heads) - 1 - (int)(blockIdx.x / c.kv_heads);
  // sequence s owns tiles from q_start[s] group / ROWS + s on: at least as many as its rows take
  auto first_tile = [&](int i) {
    return (int)((int64_t)clampi(c.q_start[i], 0, c.tokens) * a.group / ROWS) + i;
  };
  const int s = __builtin_amdgcn_readfirstlane(last_at_most(c.seqs, tile, first_tile));
  const Seq sq = sequence(c, s);
  const int R = sq.rows * a.group, r0 = (tile - first_tile(s)) * ROWS;
  if (r0 < 0 || r0 >= R) return;
  const int past = sq.len - sq.rows;
  const int pos_last = past + (min(r0 + ROWS, R) - 1) / a.group, pos_first = past + r0 / a.group;
  const int hi = min(pos_last + 1, sq.len);
  const int lo = a.window > 0 ? max(0, pos_first - a.window + 1) & ~63 : 0;
  const int tiles = hi > lo ? (hi - lo + 63) / 64 : 0;

  // this wave's rows
  const int row = r0 + 32 * w + n, tok = row / a.group, head = kvh * a.group + row % a.group;
  const int pos = row < R ? past + tok : -1;
  const int wlo = past + min(r0 + 32 * w, R - 1) / a.group, whi = past + min(r0 + 32 * w + 31, R - 1) / a.group;
  const bool full = r0 + 32 * w + 32 <= R, empty = r0 + 32 * w >= R;
  u32x4 qf[2 * C];
#pragma unroll
  for (int i = 0; i < 2 * C; ++i)
    qf[i] = row < R ? *reinterpret_cast<const u32x4*>(a.q + (int64_t)(sq.row0 + tok) * a.ldq + (int64_t)head * D + 16 * i + 8 * g) ^
                          a.q_flip
                    : (u32x4)0;

  // staging: wave w loads the 16 keys of block w, lane l row (l - 4 (l >> 4)) & 15, chunks 4 i + (l >> 4)
  const int lrow = ((lane & 15) - 4 * (lane >> 4)) & 15;
  const int32_t* table = c.table + s * c.tstride;
  const uint16_t* kb = c.k + kvh * c.hstride + 8 * (lane >> 4);
  const uint16_t* vb = c.v + kvh * c.hstride + 8 * (lane >> 4);
  uint32_t pg = 0;
  bool there = false;
  u32x4 ks[C], vs[C];
  auto key_of = [&](int t) { return min(lo + 64 * t + 16 * w + lrow, hi - 1); };
  auto ask_page = [&](int t) { pg = (uint32_t)table[key_of(t) >> c.page_shift]; };
  auto ask = [&](int t) {
    const int64_t off = key_offset(c, pg, key_of(t), there);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      ks[i] = *reinterpret_cast<const u32x4*>(kb + off + 32 * i);
      vs[i] = *reinterpret_cast<const u32x4*>(vb + off + 32 * i);
    }
  };
  auto stage = [&](int b) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      *reinterpret_cast<u32x4*>(&kl[b][w * BLK + 512 * i + 8 * lane]) = ks[i];
      *reinterpret_cast<u32x4*>(&vl[b][w * BLK + 512 * i + 8 * lane]) = vs[i];
    }
    const uint32_t bits = (uint32_t)__ballot(there) & 0xFFFFu;  // lanes 0..15 hold rows 0..15
    if (lane == 0) seen_l[b][w] = (uint16_t)bits;
  };

  float m, l;
  f16x16 o[C];  // dims 32 d + 8 j + 4 g + i in element 4 j + i
  auto pass = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < C; ++d) o[d] = (f16x16)0.f;
    ask_page(0);
    ask(0);
    ask_page(min(1, tiles - 1));
    stage(0);
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
      const int b = t & 1, t0 = lo + 64 * t;
      if (t + 1 < tiles) {
        ask(t + 1);
        ask_page(min(t + 2, tiles - 1));
      }
      // keys that this wave's rows see
      if (!empty && t0 <= whi && (a.window <= 0 || t0 + 63 > wlo - a.window)) {
        const uint64_t seen = *reinterpret_cast<const uint64_t*>(seen_l[b]);
        f16x16 sc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sc[h] = (f16x16)0.f;
#pragma unroll
          for (int i = 0; i < 2 * C; ++i) {
            const int ch = 2 * i + g;
            const u32x4 kf = *reinterpret_cast<const u32x4*>(
                &kl[b][(2 * h + (n >> 4)) * BLK + ch * 128 + (((n & 15) + 4 * ch) & 15) * 8]);
            sc[h] = mfma32<BF>(kf, qf[i], sc[h]);
          }
        }
        if (!(seen == ~0ull && full && t0 + 64 <= min(wlo + 1, hi) && (a.window <= 0 || t0 > whi - a.window))) {
          // bit k: this lane's row sees key t0 + k
          const int end = min(min(pos + 1, hi) - t0, 64), begin = a.window > 0 ? max(pos - a.window + 1 - t0, 0) : 0;
          uint64_t bits = end > begin && begin < 64 ? (~0ull >> (64 - end + begin)) << begin & seen : 0;
          bits >>= 4 * g;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((uint32_t)(bits >> (e & 16 ? 32 : 0)) & (1u << (8 * ((e >> 2) & 3) + (e & 3))))) sc[e >> 4][e & 15] = -INFINITY;
        }
        float mx = sc[0][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) mx = fmaxf(mx, sc[e >> 4][e & 15]);
        mx = max32(mx) * a.scale;
        // weights are 2^(score - m); m follows the largest score only when that is far ahead of it (a weight is at most 2^8
        // then: no range is lost), since moving it costs a product of every sum
        if (__any(mx > m + 8.f)) {
          const float up = fmaxf(m, mx), down = m == -INFINITY ? 0.f : pow2(m - up);
          m = up;
          l *= down;
#pragma unroll
          for (int d = 0; d < C; ++d) o[d] *= down;
        }
        const float base = m == -INFINITY ? 0.f : m;
        float p[32], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = sc[e >> 4][e & 15], v = pow2(__builtin_fmaf(x, a.scale, -base));
          sum += v;
          p[e] = CAREFUL && x == -INFINITY ? -1.f : v;  // (-1: not seen)
        }
        l += sum;
        if constexpr (CAREFUL) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int e = 0; e < 8; ++e) care[w][(8 * (e >> 2) + 4 * g + (e & 3)) * 32 + n] = p[8 * q + e];
#pragma unroll 1
            for (int k = 0; k < 16; ++k) {
              const float pk = care[w][k * 32 + n];
#pragma unroll
              for (int d = 0; d < C; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // dims 32 d + 8 j + 4 g + i: chunk 4 d + j
                  const int ch = 4 * d + j;
                  const uint2 u = *reinterpret_cast<const uint2*>(&vl[b][q * BLK + ch * 128 + ((k + 4 * ch) & 15) * 8 + 4 * g]);
                  const f4v v = {wide<BF>((uint16_t)u.x), wide<BF>((uint16_t)(u.x >> 16)), wide<BF>((uint16_t)u.y),
                                 wide<BF>((uint16_t)(u.y >> 16))};
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[d][4 * j + i] = pk < 0.f ? o[d][4 * j + i] : o[d][4 * j + i] + pk * v[i];
                }
            }
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {  // 16 keys: 16 q + 4 g + i and 16 q + 8 + 4 g + i
            u32x4 part[NP];
            split8<BF, NP>(p + 8 * q, part);
#pragma unroll
            for (int d = 0; d < C; ++d) {
              // 16 lanes: dims 32 d + 16 (lane >> 4 & 1) ..; lane n & 15 of them points at key n / 4 & 3, 4 dims
              const int ch = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
              u32x4 vt;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = 8 * e + 4 * g + ((lane >> 2) & 3);
                const uint2 u = read_tr(&vl[b][q * BLK + ch * 128 + ((key + 4 * ch) & 15) * 8 + 4 * (lane & 1)]);
                vt[2 * e] = u.x;
                vt[2 * e + 1] = u.y;
              }
#pragma unroll
              for (int i = 0; i < NP; ++i) o[d] = mfma32<BF>(vt, part[i], o[d]);
            }
          }
        }
      }
      if (t + 1 < tiles) stage(b ^ 1);
      __syncthreads();
    }
  };
  if (tiles) {
    if (threadIdx.x == 0) any_bad = 0;
    pass(std::false_type{});
    bool bad = false;
#pragma unroll
    for (int d = 0; d < C; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) bad |= !finite(o[d][i]);
    if (bad) any_bad = 1;
    __syncthreads();
    if (any_bad) pass(std::true_type{});
    l = add32(l);
  } else {
    l = 0.f;
#pragma unroll
    for (int d = 0; d < C; ++d) o[d] = (f16x16)0.f;
  }
  if (row >= R) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = (int64_t)(sq.row0 + tok) * a.ldo + (int64_t)head * D + 4 * g;
#pragma unroll
  for (int d = 0; d < C; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f4v v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = l == 0.f ? 0.f : o[d][4 * j + i] * inv;
      store4(a.out_type, a.out, at + 32 * d + 8 * j, v);
    }
}

template <int D, bool BF>
hipError_t prompt_d(const AttnArgs& a, hipStream_t s) {
  const int64_t tiles = (int64_t)a.c.tokens * a.group / 128 + a.c.seqs;
  const dim3 grid((uint32_t)(tiles * a.c.kv_heads));
  if (a.out_type == 0) k_attn_prompt<D, BF, BF ? 3 : 2><<<grid, 256, 0, s>>>(a);
  else k_attn_prompt<D, BF, 1><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attn_prompt(const AttnArgs& a, int head_dim, int type, hipStream_t s) {
  if (head_dim == 64) return type == 2 ? prompt_d<64, true>(a, s) : prompt_d<64, false>(a, s);
  if (head_dim == 96) return type == 2 ? prompt_d<96, true>(a, s) : prompt_d<96, false>(a, s);
  return type == 2 ? prompt_d<128, true>(a, s) : prompt_d<128, false>(a, s);
}

}  // namespace lw
