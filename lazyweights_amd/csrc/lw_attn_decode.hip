// Appending to a paged key-value cache with the position rotation, and attention of a few new tokens per sequence over it.
#include <algorithm>

#include "lw_attn_list.h"

namespace lw {

namespace {

// ── append ──────────────────────────────────────────────────────────────────────────────────────────────────────────

// q_out = R_i q, cache k = R_i k, cache v = v for the batch's new tokens, position i; R_i rotates pairs of the first `rot`
// elements by the angles of row i of cos / sin: (x, y) -> (x c - y s, y c + x s), in 32 bits, rounded once when stored.
// Pairs are elements j and j + rot / 2 ("halves") or 2 j and 2 j + 1 ("neighbours"). A thread takes 8 elements of a head:
// 4 pairs, or 8 that are only copied, so that every load and store is 8 or 16 bytes and neighbouring threads' are adjacent.
// Bound by memory: 16383 tokens of 32 + 8 + 8 heads of 128, fp32 in, 612 MB in 109 us (5.6 TB/s, two thirds of it read; a copy of
// 1 GiB reaches 5.0). A few tokens are one pass of loads that depend on each other (the sequence, its length, the page):
// 2.5 us for one token, 3.4 for 48 sequences, less than the 8 us that the host takes to make the call.
template <int D, int X, bool BF>
__global__ __launch_bounds__(256) void k_kv_append(const AppendArgs a) {
  constexpr int U = D / 8;
  const int heads = a.q ? a.heads : 0, units = (heads + 2 * a.c.kv_heads) * U, parts = (units + 255) / 256;
  const int row = blockIdx.x / parts, unit = (blockIdx.x - row * parts) * 256 + threadIdx.x;
  // the common case first: one new token per sequence
  int s = min(row, a.c.seqs - 1);
  if (!(a.c.q_start[s] <= row && row < a.c.q_start[s + 1]))
    s = last_at_most(a.c.seqs, row, [&](int i) { return a.c.q_start[i]; });
  const Seq sq = sequence(a.c, s);
  const int pos = sq.len - sq.rows + (row - sq.row0);
  if (unit >= units || row < sq.row0 || row >= sq.row0 + sq.rows || pos < 0) return;
  const int hs = unit / U, u = unit - hs * U;  // head slot: queries, keys, values
  const int h = hs < heads ? hs : (hs - heads) % a.c.kv_heads;
  const int what = hs < heads ? 0 : hs < heads + a.c.kv_heads ? 1 : 2;
  const void* src = what == 0 ? a.q : what == 1 ? a.k : a.v;
  const int64_t at = (what == 0 ? a.ldq : what == 1 ? a.ldk : a.ldv) * row + (int64_t)h * D;
  const bool turn = what < 2 && 8 * u < a.rot;
  const int e0 = turn && !a.neighbours ? 4 * u : 8 * u, e1 = turn && !a.neighbours ? a.rot / 2 + 4 * u : 8 * u + 4;
  f4v x = load4<X>(src, at + e0), y = load4<X>(src, at + e1);
  if (turn) {
    const int64_t r = (int64_t)min(pos, a.rope_rows - 1) * (a.rot / 2) + 4 * u;
    const f4v c = *reinterpret_cast<const f4v*>(a.cos + r), n = *reinterpret_cast<const f4v*>(a.sin + r);
    if (a.neighbours) {
      const f4v p = {x[0], x[2], y[0], y[2]}, q = {x[1], x[3], y[1], y[3]};
      f4v t, w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t[i] = p[i] * c[i] - q[i] * n[i];
        w[i] = q[i] * c[i] + p[i] * n[i];
      }
      x = (f4v){t[0], w[0], t[1], w[1]};
      y = (f4v){t[2], w[2], t[3], w[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = x[i], q = y[i];
        x[i] = p * c[i] - q * n[i];
        y[i] = q * c[i] + p * n[i];
      }
    }
  }
  uint16_t* dst;
  if (what == 0) {
    dst = a.q_out + a.ldo * row + (int64_t)h * D;
  } else {
    const uint32_t page = (uint32_t)a.c.table[s * a.c.tstride + (pos >> a.c.page_shift)];
    if (page >= a.c.pages) return;
    dst = (what == 1 ? a.c.k : a.c.v) + page * a.c.pstride + h * a.c.hstride +
          (pos & ((1 << a.c.page_shift) - 1)) * a.c.rstride;
  }
  *reinterpret_cast<uint2*>(dst + e0) = make_uint2(narrow2<BF>(x[0], x[1]), narrow2<BF>(x[2], x[3]));
  *reinterpret_cast<uint2*>(dst + e1) = make_uint2(narrow2<BF>(y[0], y[1]), narrow2<BF>(y[2], y[3]));
}

// ── decode ──────────────────────────────────────────────────────────────────────────────────────────────────────────

// Tiles [t_from, t_to) of the item (s, kvh, rb), whose keys start at `lo` and whose T tiles are the list's from item0 on; a block
// has `run` tiles of the list (or a whole item, which is joined by nobody else).
template <int D, bool BF, int RT, int NW>
__device__ __forceinline__ void decode_item(const AttnArgs& a, uint8_t* smem, float* ml, float* pcare, int* last_block, int s, const Seq& sq,
                                            int kvh, int rb, int lo, int t_from, int t_to, uint32_t item0, int T,
                                            uint32_t run, int lane, int w, int n, int g) {
  constexpr int C = D / 32, DT = D / 16, NP = BF ? 3 : 2;
  constexpr float LIFT = lift<BF>(0);
  const KvView& c = a.c;
  const Divisor by_group = a.by_group;
  const int R = sq.rows * a.group, r0 = rb * RT * 16;
  const int past = sq.len - sq.rows;  // row r has position past + r / group
  const int rn = max(min(r0 + RT * 16, R) - 1, r0), pos_lo = past + by_group(r0), pos_hi = past + by_group(rn);
  const int k0 = lo + 32 * t_from, k1 = min(lo + 32 * t_to, sq.len), tiles = k1 > k0 && r0 < R ? t_to - t_from : 0;

  const u32x4 flip = (u32x4)(uint32_t)__builtin_amdgcn_readfirstlane(a.q_flip);
  int pos[RT];
  // q's operands: of one row tile in registers; of two in LDS (each wave's own, read per tile), since no registers for a second
  // block per CU would be left (64 sequences of 100-3000 keys, 20 rows each: 115 us against 140)
  constexpr bool QL = RT > 1;
  u32x4 qr[QL ? 1 : C];
  u32x4* ql = reinterpret_cast<u32x4*>(smem + (NW * 32 + w * RT * 16) * D * 2) + lane;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    // Past the last row: that row's q and any keys, nothing is written. (A branch has each load waited for by itself: one sequence of
    // 778 keys 13.3 us against 12.7; with q in LDS it is the faster form, 64 sequences of 8 tokens 117 against 124.)
    const int r = min(r0 + 16 * t + n, R - 1), tok = by_group(r);
    pos[t] = r0 + 16 * t + n < R ? past + tok : 1 << 30;
    const uint16_t* q = a.q + (int64_t)(sq.row0 + tok) * a.ldq + (int64_t)(kvh * a.group + r - tok * a.group) * D + 8 * g;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const u32x4 x = !QL || r0 + 16 * t + n < R ? *reinterpret_cast<const u32x4*>(q + 32 * i) ^ flip : (u32x4)0;
      if (QL) ql[64 * (t * C + i)] = x;
      else qr[QL ? 0 : i] = x;
    }
  }
  auto qf = [&](int t, int i) { return QL ? ql[64 * (t * C + i)] : qr[QL ? 0 : i]; };
  const int32_t* table = c.table + s * c.tstride;
  const uint16_t* kb = c.k + kvh * c.hstride + 8 * g;
  const uint16_t* vb = c.v + kvh * c.hstride + 8 * g;
  uint16_t* vl = reinterpret_cast<uint16_t*>(smem) + w * 32 * D;  // [half][D / 8 chunks][16 keys][8 dims]

  float m[RT], l[RT];
  f4v o[RT][DT];
  // careful: products with V only where a row sees the key, so that infinities and NaN elsewhere stay out of it (0 times
  // them is NaN), on the vector units; taken when a first pass ends with a sum that is not finite
  auto pass = [&](auto mode) {
    constexpr bool careful = decltype(mode)::value;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[t][d] = (f4v)0.f;
    }
    uint32_t pg[2];
    u32x4 kf[2][C], vf[2][C];
    bool there[2];
    auto key_of = [&](int t, int h) { return min(k0 + 32 * t + 16 * h + n, k1 - 1); };
    auto ask_page = [&](int t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) pg[h] = (uint32_t)table[key_of(t, h) >> c.page_shift];
    };
    auto ask = [&](int t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t off = key_offset(c, pg[h], key_of(t, h), there[h]);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          kf[h][i] = *reinterpret_cast<const u32x4*>(kb + off + 32 * i);
          vf[h][i] = *reinterpret_cast<const u32x4*>(vb + off + 32 * i);
        }
      }
    };
    if (w < tiles) {
      ask_page(w);
      ask(w);
      ask_page(min(w + NW, tiles - 1));
    }
    for (int t = w; t < tiles; t += NW) {
      const int t0 = k0 + 32 * t;
      f4v sc[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f4v acc = (f4v)0.f;
#pragma unroll
          for (int i = 0; i < C; ++i) acc = mfma16<BF>(kf[h][i], qf(r, i), acc);
          sc[r][h] = acc;
        }
      uint32_t seen[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        seen[h] = (uint32_t)__ballot(there[h]) & 0xFFFFu;
#pragma unroll
        for (int i = 0; i < C; ++i)
          *reinterpret_cast<u32x4*>(vl + ((h * (D / 8) + 4 * i + g) * 16 + n) * 8) = vf[h][i];
      }
      if (t + NW < tiles) {
        ask(t + NW);
        ask_page(min(t + 2 * NW, tiles - 1));
      }
      const bool all = (seen[0] & seen[1]) == 0xFFFFu && t0 + 32 <= min(pos_lo + 1, k1) &&
                       (a.window <= 0 || t0 > pos_hi - a.window);
      u32x4 part[RT][NP];
      float p[RT][8];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) p[r][4 * h + i] = sc[r][h][i] * a.scale;
        if (!all) {
          const int first = a.window > 0 ? pos[r] - a.window : -1;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int h = e >> 2, key = t0 + 16 * h + 4 * g + (e & 3);
            const bool ok = key <= pos[r] && key > first && key < k1 && ((seen[h] >> (4 * g + (e & 3))) & 1u);
            if (!ok) p[r][e] = -INFINITY;
          }
        }
        float mx = p[r][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, p[r][e]);
        mx = fmaxf(max32(max16(mx)), m[r]);
        const float top = mx == -INFINITY ? 0.f : mx, down = pow2(m[r] - top), base = top - LIFT;
        m[r] = mx;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = pow2(p[r][e] - base);
          sum += v;
          p[r][e] = careful && p[r][e] == -INFINITY ? -1.f : v;  // (-1: not seen)
        }
        l[r] = l[r] * down + sum;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] *= down;
        split8<BF, NP>(p[r], part[r]);
      }
      if constexpr (careful) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          float* pl = pcare + w * 32 * 16;  // [32 keys][16 rows]
#pragma unroll
          for (int e = 0; e < 8; ++e) pl[(16 * (e >> 2) + 4 * g + (e & 3)) * 16 + n] = p[r][e];
#pragma unroll 1
          for (int k = 0; k < 32; ++k) {
            const float pk = pl[k * 16 + n];
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              const uint2 u = *reinterpret_cast<const uint2*>(
                  vl + (((k >> 4) * (D / 8) + 2 * d + (g >> 1)) * 16 + (k & 15)) * 8 + 4 * (g & 1));
              const f4v v = {wide<BF>((uint16_t)u.x), wide<BF>((uint16_t)(u.x >> 16)), wide<BF>((uint16_t)u.y),
                             wide<BF>((uint16_t)(u.y >> 16))};
#pragma unroll
              for (int i = 0; i < 4; ++i) o[r][d][i] = pk < 0.f ? o[r][d][i] : o[r][d][i] + pk * v[i];
            }
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          u32x4 vt;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint2 u = read_tr(vl + ((h * (D / 8) + 2 * d + ((n & 3) >> 1)) * 16 + 4 * g + (n >> 2)) * 8 + 4 * (n & 1));
            vt[2 * h] = u.x;
            vt[2 * h + 1] = u.y;
          }
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < NP; ++i) o[r][d] = mfma16<BF>(vt, part[r][i], o[r][d]);
        }
      }
    }
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

  // (a block's number is that of its run in the list)
  const int b0 = (int)(item0 / run), b1 = (int)((item0 + T - 1) / run);
  join_item<D, RT, NW>(a, smem, ml, last_block, m, l, o, s, sq, kvh, rb, b0, (int)blockIdx.x - b0, b1 - b0 + 1, w, n, g);
}

// Work is divided by walk_items, in tiles of 32 keys.
//
// Each key and value is read once, for all rows of its key-value head: 2 x 2 x D bytes a key against 4 x D x rows operations, so
// a few tens of rows are bound by memory and the matrix cores are used for their layout (an item of 4 rows fills a quarter of a
// tile's columns, the matrix cores busy 5 % of the time). A wave has a tile's 32 keys and values in flight to registers (16 KB at D = 128)
// while it works on the one before; V goes through LDS, its own, for the transposed reads. Times (us, and of what bytes):
// 64 sequences of 500-16000 keys, 8 heads of 128: 194 (1.05 GB: 5.4 TB/s, of the 6.7 that a stream of reads reaches); one of
// 131071: 97 (537 MB: 5.5); 4 x 5 tokens of 32 heads of 96 over 301-5003: 28 (101 MB); one of 778: 12.7. What separates the
// first two from that stream are mostly the launch's ends, and the others are little else: the XCDs start up to 4 us after one
// another, then come the lengths, a page number, its keys, and at the end the join of runs, each waiting for the one before.
template <int D, bool BF, int RT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void k_attn_decode(const AttnArgs a) {
  // V tiles of the waves (after the loop their sums), then, of more than one row tile, q
  __shared__ __align__(16) uint8_t smem[NW * (RT > 1 ? 32 + RT * 16 : 32) * D * 2];
  __shared__ float ml[NW * 16 * RT * 2];
  __shared__ float pcare[NW * 32 * 16];
  __shared__ uint32_t csum[1024];  // tiles of the sequences up to each 64th
  __shared__ int last_block;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  walk_items<NW, 32, true>(a, csum, lane, w, [&](int s, const Seq& sq, int kvh, int rb, int lo, int t_from, int t_to, uint32_t item0, int T,
                                           uint32_t run) __attribute__((always_inline)) {
    decode_item<D, BF, RT, NW>(a, smem, ml, pcare, &last_block, s, sq, kvh, rb, lo, t_from, t_to, item0, T, run, lane, w, n, g);
  });
}

template <int D, int X>
hipError_t append_d(const AppendArgs& a, int type, hipStream_t s) {
  const int units = ((a.q ? a.heads : 0) + 2 * a.c.kv_heads) * (D / 8), parts = (units + 255) / 256;
  const dim3 grid((uint32_t)a.c.tokens * (uint32_t)parts);
  if (type == 2) k_kv_append<D, X, true><<<grid, 256, 0, s>>>(a);
  else k_kv_append<D, X, false><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}
template <int D>
hipError_t append_x(const AppendArgs& a, int type, int x_type, hipStream_t s) {
  return x_type == 0 ? append_d<D, 0>(a, type, s) : x_type == 1 ? append_d<D, 1>(a, type, s) : append_d<D, 2>(a, type, s);
}

template <int D, bool BF>
hipError_t decode_d(const AttnArgs& a, const DecodePlan& p, hipStream_t s) {
  const dim3 grid((uint32_t)p.blocks);
  if (p.row_tiles == 1 && p.whole) k_attn_decode<D, BF, 1, 8><<<grid, 512, 0, s>>>(a);
  else if (p.row_tiles == 1) k_attn_decode<D, BF, 1, 4><<<grid, 256, 0, s>>>(a);
  else k_attn_decode<D, BF, 2, 4><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

DecodePlan decode_plan(int seqs, int kv_heads, int group, int head_dim, int max_new, int max_kv) {
  DecodePlan p;
  const int rows = group * max_new;
  // More than 16 rows: two row tiles per item, which share what is read, where there is much to read; else one, and more items,
  // each sooner done (us with two / one: 8 sequences of 1000-8000 keys, 8 heads of 128, 20 rows 40 / 55, one of 20000, 64 rows
  // 52 / 65; one of 500, 64 rows 22 / 15, 4 of 300-5000, 4 heads, 64 rows 33 / 29; at 160000 keys of all heads from 52 / 65 to
  // 34 / 32). Four row tiles took 54 and 97 in the cases of 500 and 20000 keys: no registers for a second block, and a join of
  // all their sums by one.
  p.row_tiles = rows <= 16 || (int64_t)seqs * kv_heads * max_kv < 1 << 17 ? 1 : 2;
  p.row_blocks = (rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles);
  // A block per CU, or two where a block would have more than one item to go through: the second works while the first goes from
  // one item to the next, but an item in more parts takes longer to join. us with one / two: 512 items of 500-16000 keys
  // 208 / 196, 2048 items (dim 64) 437 / 382, 1600 items of 100-3000 keys 216 / 182, 512 of 100-3000 and two row tiles 130 / 115;
  // 128 items 29 / 29 and 51 / 52, 8 items of 131071 keys 98 / 107, 1 item of a million 109 / 126. Fewer (a power of two) where
  // they would not have a tile per wave.
  const int64_t items = (int64_t)seqs * kv_heads * p.row_blocks, tiles = items * (max_kv / 32 + 2);
  const int most = items > 256 ? 9 : 8;
  // A block of 8 waves per item: where every wave has one tile at most, nothing is left to join between blocks (us against
  // runs: 201 keys 8.4 / 13.7, but 778 keys, four tiles after another, 15.6 / 12.9); and where there are many items, none long
  // (1600 items of 100-3000 keys 175 / 182, 1024 of 628-3033 130 / 141; 512 of 500-16000 270 / 198).
  p.whole = p.row_tiles == 1 && items <= 1 << 20 && (max_kv <= 256 || (items >= 1024 && max_kv <= 4096));
  p.blocks_log2 = 0;
  while (p.blocks_log2 < most && ((int64_t)4 << p.blocks_log2) < tiles) ++p.blocks_log2;
  p.blocks = p.whole ? (int)items : 1 << p.blocks_log2;
  p.count_bytes = ((size_t)items * 4 + 255) & ~(size_t)255;
  p.part_bytes = ((size_t)1 << p.blocks_log2) * 2 * p.row_tiles * 16 * (head_dim + 2) * 4;
  p.most_keys = (int)std::min<int64_t>(1 << 30, ((int64_t)1 << 36) / std::max<int64_t>(items, 1) / 2 - 64);
  return p;
}

hipError_t launch_append(const AppendArgs& a, int head_dim, int type, int x_type, hipStream_t s) {
  if (head_dim == 64) return append_x<64>(a, type, x_type, s);
  if (head_dim == 96) return append_x<96>(a, type, x_type, s);
  return append_x<128>(a, type, x_type, s);
}

hipError_t launch_attn_decode(const AttnArgs& a, const DecodePlan& p, int head_dim, int type, hipStream_t s) {
  if (head_dim == 64) return type == 2 ? decode_d<64, true>(a, p, s) : decode_d<64, false>(a, p, s);
  if (head_dim == 96) return type == 2 ? decode_d<96, true>(a, p, s) : decode_d<96, false>(a, p, s);
  return type == 2 ? decode_d<128, true>(a, p, s) : decode_d<128, false>(a, p, s);
}

}  // namespace lw
