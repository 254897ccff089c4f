// Attention of a few new tokens per sequence over a paged key-value cache held in 8 bits.
#include <algorithm>

#include "lw_attn8_device.h"
#include "lw_attn_list.h"

namespace lw {

namespace {

// Tiles [t_from, t_to) of 16 H keys of the item (s, kvh, rb), as decode_item's of a 16-bit cache.
template <int D, bool BF, int RT, int NW, int H>
__device__ __forceinline__ void decode8_item(const Attn8Args& args, uint8_t* smem, float* ml, float* pcare, int* last_block, int s,
                                             const Seq& sq, int kvh, int rb, int lo, int t_from, int t_to, uint32_t item0, int T,
                                             uint32_t run, int lane, int w, int n, int g) {
  constexpr int KEYS = 16 * H, C = D / 32, DT = D / 16, NP = 2, FULL = D / 64, TAIL = C % 2;
  constexpr float LIFT = lift<false>(0);
  const AttnArgs& a = args.a;
  const KvView& c = a.c;
  const Divisor by_group = a.by_group;
  const int R = sq.rows * a.group, r0 = rb * RT * 16;
  const int past = sq.len - sq.rows;  // row r has position past + r / group
  const int rn = max(min(r0 + RT * 16, R) - 1, r0), pos_lo = past + by_group(r0), pos_hi = past + by_group(rn);
  const int k0 = lo + KEYS * t_from, k1 = min(lo + KEYS * t_to, sq.len), tiles = k1 > k0 && r0 < R ? t_to - t_from : 0;
  const int last = (k1 - 1) & ~15, mask = (1 << c.page_shift) - 1;  // the last block of 16 keys

  const u32x4 flip = (u32x4)(uint32_t)__builtin_amdgcn_readfirstlane(a.q_flip);
  int pos[RT];
  // q's operands: of one row tile in registers, of two in LDS, each wave's own. A lane's 16 bytes of a key are 16 dims
  // 64 i + 16 g on, operands 2 i and 2 i + 1 (a tail of 32 dims: 8 bytes), and q's are of the same dims.
  constexpr bool QL = RT > 1;
  u32x4 qr[QL ? 1 : C];
  u32x4* ql = reinterpret_cast<u32x4*>(smem + NW * KEYS * D + w * RT * 16 * D * 2) + lane;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    // (past the last row: that row's q, for which nothing is written)
    const int r = min(r0 + 16 * t + n, R - 1), tok = by_group(r);
    pos[t] = r0 + 16 * t + n < R ? past + tok : 1 << 30;
    const uint16_t* q = a.q + (int64_t)(sq.row0 + tok) * a.ldq + (int64_t)(kvh * a.group + r - tok * a.group) * D;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int dim = TAIL && i == C - 1 ? 64 * FULL + 8 * g : 64 * (i >> 1) + 16 * g + 8 * (i & 1);
      const u32x4 x = !QL || r0 + 16 * t + n < R ? *reinterpret_cast<const u32x4*>(q + dim) ^ flip : (u32x4)0;
      if (QL) ql[64 * (t * C + i)] = x;
      else qr[QL ? 0 : i] = x;
    }
  }
  auto qf = [&](int t, int i) { return QL ? ql[64 * (t * C + i)] : qr[QL ? 0 : i]; };
  const int32_t* table = c.table + s * c.tstride;
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(c.k) + kvh * c.hstride;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(c.v) + kvh * c.hstride;
  // a lane asks for the page, and for the exponent of K (lanes 0 .. of 8) or V (4 .. of 8), of block `lane & (H - 1)` of a tile
  const int8_t* eb = (lane & 4 ? args.e.v : args.e.k) + kvh * args.e.hstride;
  // V of a tile, each wave's own: [H][D / 16 chunks][16 keys][16 dims], the keys of odd blocks turned by 8, so that the keys
  // 4 g .. 4 g + 3 of two blocks lie in other banks
  uint8_t* vl = smem + w * KEYS * D;

  float m[RT], l[RT];  // m: the largest score plus its value's exponent, the power of two that weights are measured against
  f4v o[RT][DT];
  // careful: products with V only where a row sees the key, so that NaN elsewhere stay out of it (0 times them is NaN), on the vector
  // units; taken when a first pass ends with a sum that is not finite
  auto pass = [&](auto mode) {
    constexpr bool careful = decltype(mode)::value;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[t][d] = (f4v)0.f;
    }
    uint32_t pg;
    int ex;
    u32x4 kf[H][FULL], vf[H][FULL];
    uint2 kt[H], vt8[H];
    uint32_t there = 0;
    auto ask_page = [&](int t) { pg = (uint32_t)table[min(k0 + KEYS * t + 16 * (lane & (H - 1)), last) >> c.page_shift]; };
    auto ask = [&](int t) {
      const int mine = min(k0 + KEYS * t + 16 * (lane & (H - 1)), last) & mask;
      ex = eb[(pg < c.pages ? pg * args.e.pstride : 0) + mine / kExpBlock];
      there = 0;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint32_t page = __builtin_amdgcn_readlane(pg, h);
        const int b = min(k0 + KEYS * t + 16 * h, last);
        there |= (page < c.pages ? 1u : 0u) << h;
        const int64_t off = (page < c.pages ? (int64_t)page * c.pstride : 0) + (int64_t)(b & mask) * c.rstride;
        const uint32_t row = (uint32_t)min(n, k1 - 1 - b) * (uint32_t)c.rstride;
#pragma unroll
        for (int i = 0; i < FULL; ++i) {
          kf[h][i] = *reinterpret_cast<const u32x4*>(kb + off + (row + 64 * i + 16 * g));
          vf[h][i] = *reinterpret_cast<const u32x4*>(vb + off + (row + 64 * i + 16 * g));
        }
        if (TAIL) {
          kt[h] = *reinterpret_cast<const uint2*>(kb + off + (row + 64 * FULL + 8 * g));
          vt8[h] = *reinterpret_cast<const uint2*>(vb + off + (row + 64 * FULL + 8 * g));
        }
      }
    };
    if (w >= tiles) return;
    ask_page(w);
    ask(w);
    ask_page(min(w + NW, tiles - 1));
    int t = w;
    do {
      const int t0 = k0 + KEYS * t;
      f4v sc[RT][H];
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int r = 0; r < RT; ++r) sc[r][h] = (f4v)0.f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const u32x4 k = TAIL && i == C - 1 ? widen8<BF>(kt[h].x, kt[h].y) : widen8<BF>(kf[h][i / 2][2 * (i & 1)], kf[h][i / 2][2 * (i & 1) + 1]);
#pragma unroll
          for (int r = 0; r < RT; ++r) sc[r][h] = mfma16<BF>(k, qf(r, i), sc[r][h]);
        }
      }
      int ke[H], ve[H];
      const int e = clampi(ex, -kMostExp, kMostExp);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        ke[h] = __builtin_amdgcn_readlane(e, h);
        ve[h] = __builtin_amdgcn_readlane(e, 4 + h);
        const int at = n ^ (h & 1 ? 8 : 0);
#pragma unroll
        for (int i = 0; i < FULL; ++i) *reinterpret_cast<u32x4*>(vl + ((h * DT + 4 * i + g) * 16 + at) * 16) = vf[h][i];
        if (TAIL) *reinterpret_cast<uint2*>(vl + ((h * DT + 4 * FULL + (g >> 1)) * 16 + at) * 16 + 8 * (g & 1)) = vt8[h];
      }
      const uint32_t seen = there;
      if (t + NW < tiles) {
        ask(t + NW);
        ask_page(min(t + 2 * NW, tiles - 1));
      }
      const bool all = seen == (1u << H) - 1 && t0 + KEYS <= min(pos_lo + 1, k1) && (a.window <= 0 || t0 > pos_hi - a.window);
      u32x4 part[RT][H / 2][NP];
      float p[RT][4 * H];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        // score and value's exponent together, in powers of two
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float ks = a.scale * two_to(ke[h]), vs = (float)ve[h];
#pragma unroll
          for (int i = 0; i < 4; ++i) p[r][4 * h + i] = __builtin_fmaf(sc[r][h][i], ks, vs);
        }
        if (!all) {
          const int first = a.window > 0 ? pos[r] - a.window : -1;
#pragma unroll
          for (int i = 0; i < 4 * H; ++i) {
            const int h = i >> 2, key = t0 + 16 * h + 4 * g + (i & 3);
            if (!(key <= pos[r] && key > first && key < k1 && ((seen >> h) & 1u))) p[r][i] = -INFINITY;
          }
        }
        float mx = p[r][0];
#pragma unroll
        for (int i = 1; i < 4 * H; ++i) mx = fmaxf(mx, p[r][i]);
        mx = fmaxf(max32(max16(mx)), m[r]);
        const float top = mx == -INFINITY ? 0.f : mx, down = pow2(m[r] - top), base = top - LIFT;
        m[r] = mx;
        l[r] *= down;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = p[r][4 * h + i], v = pow2(x - base);
            sum += v;
            p[r][4 * h + i] = careful && x == -INFINITY ? -1.f : v;  // (-1: not seen)
          }
          l[r] = __builtin_fmaf(sum, two_to(-ve[h]), l[r]);  // the weights themselves
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] *= down;
        if constexpr (!careful)
#pragma unroll
          for (int x = 0; x < H / 2; ++x) split8<false, NP>(p[r] + 8 * x, part[r][x]);
      }
      if constexpr (careful) {
        float* pl = pcare + w * 32 * 16;  // [32 keys][16 rows]
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int x = 0; x < H / 2; ++x) {
#pragma unroll
            for (int i = 0; i < 8; ++i) pl[(16 * (i >> 2) + 4 * g + (i & 3)) * 16 + n] = p[r][8 * x + i];
#pragma unroll 1
            for (int k = 0; k < 32; ++k) {
              const float pk = pl[k * 16 + n];
              const int h = 2 * x + (k >> 4), at = (k & 15) ^ (h & 1 ? 8 : 0);
#pragma unroll
              for (int d = 0; d < DT; ++d) {
                const f4v v = from8(*reinterpret_cast<const uint32_t*>(vl + ((h * DT + d) * 16 + at) * 16 + 4 * g));
#pragma unroll
                for (int i = 0; i < 4; ++i) o[r][d][i] = pk < 0.f ? o[r][d][i] : o[r][d][i] + pk * v[i];
              }
            }
          }
      } else {
        // V's operand: of two blocks x, the keys 4 g .. 4 g + 3 of each, as the weights lie
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int x = 0; x < H / 2; ++x) {
            const int key = n >> 1, h = key >> 2, at = (4 * g + (key & 3)) ^ (8 * h);
            const uint2 u = read_tr8(vl + (((2 * x + h) * DT + d) * 16 + at) * 16 + 8 * (n & 1));
            const u32x4 v = widen8<false>(u.x, u.y);
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
              for (int i = 0; i < NP; ++i) o[r][d] = mfma16<false>(v, part[r][x][i], o[r][d]);
          }
      }
    } while ((t += NW) < tiles);
  };
  pass(std::false_type{});
  bool bad = false;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) bad |= !finite(o[r][d][i]);
  if (__any(bad)) pass(std::true_type{});

  join_item<D, RT, NW>(a, smem, ml, last_block, m, l, o, s, sq, kvh, rb, item0, T, run, w, n, g);
}

template <int D, bool BF, int RT, int NW, int H>
__global__ __launch_bounds__(64 * NW, 2) void k_attn8_decode(const Attn8Args args) {
  // V tiles of the waves (after the loop their sums), then, of more than one row tile, q
  __shared__ __align__(16) uint8_t smem[NW * D * std::max(16 * H, 64) + (RT > 1 ? NW * RT * 16 * D * 2 : 0)];
  __shared__ float ml[NW * 16 * RT * 2];
  __shared__ float pcare[NW * 32 * 16];
  __shared__ uint32_t csum[1024];  // tiles of the sequences up to each 64th
  __shared__ int last_block;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  walk_items<NW, 16 * H>(args.a, csum, lane, w, [&](int s, const Seq& sq, int kvh, int rb, int lo, int t_from, int t_to, uint32_t item0,
                                                    int T, uint32_t run) __attribute__((always_inline)) {
    decode8_item<D, BF, RT, NW, H>(args, smem, ml, pcare, &last_block, s, sq, kvh, rb, lo, t_from, t_to, item0, T, run, lane, w, n, g);
  });
}

template <int D, bool BF>
hipError_t decode8_d(const Attn8Args& a, const DecodePlan& p, hipStream_t s) {
  const dim3 grid((uint32_t)p.blocks);
  if (p.row_tiles == 1 && p.whole) k_attn8_decode<D, BF, 1, 8, 4><<<grid, 512, 0, s>>>(a);
  else if (p.row_tiles == 1) k_attn8_decode<D, BF, 1, 4, 4><<<grid, 256, 0, s>>>(a);
  else k_attn8_decode<D, BF, 2, 4, 4><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

DecodePlan decode8_plan(int seqs, int kv_heads, int group, int head_dim, int max_new, int max_kv) {
  DecodePlan p;
  const int rows = group * max_new;
  p.row_tiles = rows <= 16 || (int64_t)seqs * kv_heads * max_kv < 1 << 18 ? 1 : 2;
  p.row_blocks = (rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles);
  const int64_t items = (int64_t)seqs * kv_heads * p.row_blocks, tiles = items * (max_kv / 64 + 2);
  const int most = items > 256 ? 9 : 8;
  p.whole = p.row_tiles == 1 && items <= 1 << 20 && (max_kv <= 512 || (items >= 1024 && max_kv <= 8192));
  p.blocks_log2 = 0;
  while (p.blocks_log2 < most && ((int64_t)4 << p.blocks_log2) < tiles) ++p.blocks_log2;
  p.blocks = p.whole ? (int)items : 1 << p.blocks_log2;
  p.count_bytes = ((size_t)items * 4 + 255) & ~(size_t)255;
  p.part_bytes = ((size_t)1 << p.blocks_log2) * 2 * p.row_tiles * 16 * (head_dim + 2) * 4;
  p.most_keys = (int)std::min<int64_t>(1 << 30, ((int64_t)1 << 37) / std::max<int64_t>(items, 1) / 2 - 128);
  return p;
}

hipError_t launch_attn8_decode(const Attn8Args& a, const DecodePlan& p, int head_dim, int q_type, hipStream_t s) {
  if (head_dim == 64) return q_type == 2 ? decode8_d<64, true>(a, p, s) : decode8_d<64, false>(a, p, s);
  if (head_dim == 96) return q_type == 2 ? decode8_d<96, true>(a, p, s) : decode8_d<96, false>(a, p, s);
  return q_type == 2 ? decode8_d<128, true>(a, p, s) : decode8_d<128, false>(a, p, s);
}

}  // namespace lw
