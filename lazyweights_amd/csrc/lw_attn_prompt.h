// Attention of whole prompts, or chunks of them, over a paged key-value cache of 16 bits (lw_attn_prompt.hip) or 8 (lw_attn8_prompt.hip).
#pragma once
#include <algorithm>
#include <type_traits>

#include "lw_attn8_device.h"

namespace lw {

namespace {

// every wave's copies have arrived (of 8 bits they are stores to LDS, which the barrier waits for), and every wave is done with what it
// read
template <bool F8>
__device__ __forceinline__ void arrived() {
  if (!F8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

__device__ __forceinline__ const AttnArgs& attn_args(const AttnArgs& a) { return a; }
__device__ __forceinline__ const AttnArgs& attn_args(const Attn8Args& a) { return a.a; }

// The ROWS rows (token, head) of a sequence that a block has, and the keys [lo, hi) that they see together, in `tiles` tiles of 64.
struct RowTile {
  Seq sq;
  int s, r0, rows, lo, hi, tiles;
  // the tiles that each of `splits` blocks takes (eight at least): the first one has some wherever there are any
  __device__ __forceinline__ int tiles_each(int splits) const { return splits > 1 ? max((tiles + splits - 1) / splits, 8) : tiles; }
};
template <int ROWS>
__device__ __forceinline__ RowTile row_tile(const AttnArgs& a, int tile) {
  const KvView& c = a.c;
  const int tokens = c.tokens, group = a.group;
  // sequence s owns tiles from q_start[s] group / ROWS + s on: at least as many as its rows take
  auto first_tile = [&](int i) { return (int)((int64_t)clampi(c.q_start[i], 0, tokens) * group / ROWS) + i; };
  RowTile t;
  t.s = __builtin_amdgcn_readfirstlane(last_at_most(c.seqs, tile, first_tile));
  t.sq = sequence(c, t.s);
  const int R = t.sq.rows * group, past = t.sq.len - t.sq.rows;
  t.r0 = (tile - first_tile(t.s)) * ROWS;
  t.rows = t.r0 < 0 ? 0 : min(R - t.r0, ROWS);
  t.lo = t.hi = t.tiles = 0;
  if (t.rows > 0) {
    const Divisor by_group = a.by_group;
    const int first = past + by_group(t.r0), last = past + by_group(t.r0 + t.rows - 1);
    t.hi = min(last + 1, t.sq.len);
    t.lo = a.window > 0 ? max(0, first - a.window + 1) & ~63 : 0;
    t.tiles = t.hi > t.lo ? (t.hi - t.lo + 63) / 64 : 0;
  }
  return t;
}

// A block: W waves, each 32 rows (token, head) of one key-value head of a sequence, over the keys they see in tiles of 64.
// K and V tiles lie in LDS as [16-key block][D / 8 chunks][16 slots][8 dims], key k of a block in slot (k + 4 chunk) & 15:
// the score product's operand reads (32 keys of a chunk) and the transposed reads of V (4 keys of 4 chunks) are both free
// of bank conflicts. The next tile is copied by loads that go to LDS directly (a wave copies a block of 16 keys, lane l
// its 16 bytes of chunk 4 i + (l >> 4)) while one is worked on.
//
// Of 8 waves, two share a SIMD, and all meet once per tile: so that one's softmax runs beside the other's products, the
// last four work through a tile in another order, the second product of the tile before first (V has four buffers).
// 4 waves leave room for a second block on the CU, which runs at its own pace.
//
// Per 64 keys and 32 rows a wave has 32 matrix instructions of 32 cycles (D = 128, one-part weights) and some 170 vector
// instructions (a score's scaling, exponential, conversion; its share of maximum and sum), 32 of them exponentials at a
// quarter of the rate: 1024 cycles beside about 1100, which the SIMD's two waves run against each other. 15999 tokens of
// 32 heads of 128, bf16: 2.10 TFLOP in 1960 us, 1070 TFLOP/s (a library product of 16384 in each direction reaches 1338);
// the matrix cores are busy half of the cycles, and the card holds its clock at 1.75 to 1.95 of 2.4 GHz meanwhile. fp32
// outputs take two- or three-part weights, half as many or as many matrix instructions more: 9 ragged prompts of 17-2500
// tokens, 32 heads of 96, 55 GFLOP (83 with both parts) in 127 us. Row tiles with the most keys first over all sequences (they
// are so within each) lost 5 to 14 %: neighbouring tiles then no longer share keys in an XCD's L2, and each block has to
// find its tile.
//
// Where there are few rows (AttnArgs::splits > 1), the key tiles of a block's rows are shared out to up to `splits` blocks, which
// leave their maxima and sums in slots of the workspace, lane by lane, for k_attn_join.
//
// LONG (fp32 outputs, more than kLongRun keys in a block's run): a tile's products are summed from zero, its smallest parts first,
// and then added to the rows' sums, and l by add_exactly(): what a weight's later parts add is near the last bit of a long sum,
// and where many weights are alike every addition loses the same of it (40000 like keys: 4.3e-5 of the output without,
// 1.3e-6 with). It takes an addition per sum and tile: 9000 tokens of 32 heads of 128 in fp16 1010 us against 982, 1000 tokens of 32
// heads of 96 after 12000 375 against 303, so that shorter runs, whose sums have a few hundred steps a part, go without. (Over 8 bits,
// heads of 128, and of 96 with 4 waves, have some of these sums' registers in memory within the loop; no other form of 8 bits has.)
//
// A cache in 8 bits (ARGS = Attn8Args): a wave's share of the tile after the next comes to registers while one is worked on, and goes to
// LDS as 16-bit numbers, K's of q's type and V's fp16, which hold 8 bits exactly: converted once per block, since every wave reads all
// of a tile (converting where operands are read would take a wave 256 instructions a tile, of some 230 in all). The powers of two of a
// block of 16 keys enter the scores: K's as a factor, V's as an addend, since weights are measured against the largest product of a
// weight and its value's power of two; for the sum of weights that is taken off again.
template <int D, bool BF, int NP, int W, bool LONG, class ARGS>
__global__ __launch_bounds__(64 * W, 2) void k_attn_prompt(const ARGS args) {
  constexpr bool F8 = std::is_same<ARGS, Attn8Args>::value, VBF = BF && !F8;  // VBF: V and weights in bf16
  const AttnArgs& a = attn_args(args);
  constexpr int C = D / 32, ROWS = 32 * W, BLK = D * 16;  // BLK: elements of a 16-key block
  // fp16: 4 costs 1 to 2 % of a call against 8 (9 ragged prompts 126 us against 124), 1 would cost 4 %
  constexpr float AHEAD = VBF ? 8.f : 4.f, LIFT = lift<VBF>(AHEAD);
  // (separate arrays, and a loop over all of them, so that the compiler sees which copies a read has to wait for)
  __shared__ __align__(16) uint16_t k0[4 * BLK], k1[4 * BLK], v0[4 * BLK], v1[4 * BLK], v2[W == 8 ? 4 * BLK : 8],
      v3[W == 8 ? 4 * BLK : 8];
  __shared__ __align__(8) uint16_t seen_l[2][4];
  __shared__ __align__(16) float ks_l[F8 ? 2 : 1][4], ve_l[F8 ? 2 : 1][4], iv_l[F8 ? 2 : 1][4];  // scale 2^e of K, e and 2^-e of V
  __shared__ float care[W][16 * 32];  // weights of 16 keys x 32 rows of each wave, in the second pass
  __shared__ int any_bad;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, g = lane >> 5;
  const KvView& c = a.c;
  const int splits = W == 4 ? a.splits : 1, unit = blockIdx.x / c.kv_heads, kvh = blockIdx.x - unit * c.kv_heads;
  const int tile = (int)(gridDim.x / c.kv_heads) / splits - 1 - unit / splits, share = unit % splits;
  const RowTile rt = row_tile<ROWS>(a, tile);
  if (rt.rows <= 0) return;
  const Seq& sq = rt.sq;
  const int s = rt.s, R = sq.rows * a.group, r0 = rt.r0;
  const int past = sq.len - sq.rows;
  const Divisor by_group = a.by_group;
  const int each = W == 4 ? rt.tiles_each(splits) : rt.tiles;
  const int lo = rt.lo + 64 * each * share, hi = min(rt.hi, lo + 64 * each);
  const int tiles = hi > lo ? (hi - lo + 63) / 64 : 0;
  if (share > 0 && tiles == 0) return;

  // this wave's rows
  const int row = r0 + 32 * w + n, tok = by_group(row), head = kvh * a.group + row - tok * a.group;
  const int pos = row < R ? past + tok : -1;
  const int wlo = past + by_group(min(r0 + 32 * w, R - 1)), whi = past + by_group(min(r0 + 32 * w + 31, R - 1));
  const bool full = r0 + 32 * w + 32 <= R, empty = r0 + 32 * w >= R;
  const u32x4 flip = (u32x4)(uint32_t)__builtin_amdgcn_readfirstlane(a.q_flip);
  // (past the last row: that row's q, for which nothing is seen or written; a branch would have each load waited for by itself)
  const int q_row = min(row, R - 1), q_tok = by_group(q_row);
  const uint16_t* q_from = a.q + (int64_t)(sq.row0 + q_tok) * a.ldq + (int64_t)(kvh * a.group + q_row - q_tok * a.group) * D + 8 * g;
  u32x4 qf[2 * C];
#pragma unroll
  for (int i = 0; i < 2 * C; ++i) qf[i] = *reinterpret_cast<const u32x4*>(q_from + 16 * i) ^ flip;

  const int lrow = ((lane & 15) - 4 * (lane >> 4)) & 15;  // the row of its block that this lane copies
  const int32_t* table = c.table + s * c.tstride;
  const uint16_t* kb = c.k + kvh * c.hstride + 8 * (lane >> 4);
  const uint16_t* vb = c.v + kvh * c.hstride + 8 * (lane >> 4);
  const int wb = w & 3;  // the 16 keys that this wave copies; of 8 waves, the first four copy K and the others V
  uint32_t pg = 0;
  auto key_of = [&](int t) { return min(lo + 64 * t + 16 * wb + lrow, hi - 1); };
  auto ask_page = [&](int t) { pg = (uint32_t)table[key_of(t) >> c.page_shift]; };
  // a wave's share of a tile's copy, in PIECES instructions of 1 KB: where from, then piece by piece (a run of them would
  // keep every wave waiting for the address units at the start of a tile)
  // (of 8 bits: keys 8 u .. 8 u + 7 of K and of V for each unit u = w, and w + 4 of 4 waves, a lane 16 bytes of row lane & 7)
  constexpr int UNITS = 8 / W, PIECES = F8 ? 2 * UNITS : W == 4 ? 2 * C : C;
  const uint16_t *k_from = nullptr, *v_from = nullptr;
  // where a lane's 16 bytes go, two chunks
  int put_at[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int ch = 2 * (lane >> 3) + i, row = 8 * (w & 1) + (lane & 7);
    put_at[i] = 2 * ((w >> 1) * BLK + ch * 128 + ((row + 4 * ch) & 15) * 8);
  }
  // Of 8 waves, those of even units see to K's exponents and those of odd ones, the other halves of the same blocks, to V's; of 4 each
  // sees to both, since a branch costs more there (15999 tokens 2074 us against 2173, but 2000 tokens 77 / 68).
  constexpr bool PARITY = W == 8;
  const uint8_t* kb8 = reinterpret_cast<const uint8_t*>(c.k) + kvh * c.hstride;
  const uint8_t* vb8 = reinterpret_cast<const uint8_t*>(c.v) + kvh * c.hstride;
  const int8_t *ke8 = nullptr, *ve8 = nullptr;
  if constexpr (F8) {
    ve8 = args.e.v + kvh * args.e.hstride;
    ke8 = PARITY && w & 1 ? ve8 : args.e.k + kvh * args.e.hstride;
  }
  const uint32_t lane_off = (uint32_t)(lane & 7) * (uint32_t)c.rstride + 16 * min(lane >> 3, D / 16 - 1);
  u32x4 raw[F8 ? PIECES : 1];
  int raw_e[F8 ? PIECES : 1];
  uint32_t raw_pg[UNITS];
  bool raw_there[UNITS];
  // the first key of a unit of tile t (past the last key: of the unit that holds it)
  auto unit_key = [&](int t, int u) { return min(lo + 64 * t + 8 * (w + 4 * u), (hi - 1) & ~7); };
  auto ask_pages = [&](int t) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) raw_pg[u] = (uint32_t)table[unit_key(t, u) >> c.page_shift];
  };
  // unit u of tile t on its way
  auto load_unit = [&](int t, int u) {
    if constexpr (F8) {
      const uint32_t page = __builtin_amdgcn_readfirstlane(raw_pg[u]);
      const int key = unit_key(t, u), in_page = key & ((1 << c.page_shift) - 1);
      raw_there[u] = page < c.pages;
      const int64_t at = raw_there[u] ? page : 0;
      const int64_t off = at * c.pstride + (int64_t)((uint64_t)(uint32_t)in_page * (uint32_t)c.rstride);
      const int64_t eoff = at * args.e.pstride + in_page / kExpBlock;
      uint32_t mine = lane_off;
      if (W == 4 || hi - key < 8) mine = (uint32_t)min(lane & 7, hi - 1 - key) * (uint32_t)c.rstride + 16 * min(lane >> 3, D / 16 - 1);
      raw[2 * u] = *reinterpret_cast<const u32x4*>(kb8 + off + mine);
      raw[2 * u + 1] = *reinterpret_cast<const u32x4*>(vb8 + off + mine);
      raw_e[2 * u] = ke8[eoff];
      if (!PARITY) raw_e[2 * u + 1] = ve8[eoff];
    }
  };
  auto load = [&](int t) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) load_unit(t, u);
  };
  auto locate = [&](int t) {
    bool there;
    const int64_t off = key_offset(c, pg, key_of(t), there);
    k_from = kb + off;
    v_from = vb + off;
    const uint32_t bits = (uint32_t)__ballot(there) & 0xFFFFu;  // lanes 0..15 hold rows 0..15
    if (lane == 0 && w < 4) seen_l[t & 1][w] = (uint16_t)bits;
  };
  // (t: the tile that is worked on, the one before the piece's)
  auto piece = [&](int j, uint16_t* kt, uint16_t* vt, int t) {
    if constexpr (F8) {
      const int u = j >> 1, block = (w >> 1) + 2 * u;
      uint16_t* to = (j & 1 ? vt : kt) + 2 * u * BLK;
      asm("" : "+v"(put_at[0]), "+v"(put_at[1]));  // (or the compiler keeps the address in every buffer)
      if (D == 128 || (lane >> 3) < D / 16)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<u32x4*>(reinterpret_cast<uint8_t*>(to) + put_at[i]) =
              j & 1 ? widen8<false>(raw[j][2 * i], raw[j][2 * i + 1]) : widen8<BF>(raw[j][2 * i], raw[j][2 * i + 1]);
      if (PARITY && j & 1) return;
      const int to_tile = (t + 1) & 1;
      const int e = clampi(PARITY ? __builtin_amdgcn_readfirstlane(raw_e[j]) : raw_e[j], -kMostExp, kMostExp);
      if (PARITY ? w & 1 : j & 1) {  // (the same values from every lane; of 4 waves from the two units of a block)
        ve_l[to_tile][block] = (float)e;
        iv_l[to_tile][block] = two_to(-e);
      } else {
        seen_l[to_tile][block] = raw_there[u] ? 0xFFFF : 0;
        ks_l[to_tile][block] = fmaxf(a.scale * two_to(e), 1e-37f);
      }
      return;
    }
    if (W == 4 ? j < C : w < 4) copy_lds16(k_from + 32 * (j % C), kt + wb * BLK + 512 * (j % C));
    else copy_lds16(v_from + 32 * (j % C), vt + wb * BLK + 512 * (j % C));
  };
  // (offsets in bytes of 8 bits)
  auto in_tile = [](const uint16_t* buf, int at) {
    return F8 ? reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(buf) + at) : buf + at;
  };
  // where a lane reads: K, chunk 2 i + g of key n & 15 of block 2 h + (n >> 4), by the parity of i; V, 4 dims of chunk
  // 4 d + c0 of key 8 e + 4 g + (lane >> 2 & 3) of block q
  const int c0 = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  int kr[2], vr[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    kr[i] = (F8 ? 2 : 1) * ((n >> 4) * BLK + g * 128 + (((n & 15) + 8 * i + 4 * g) & 15) * 8);
    vr[i] = (F8 ? 2 : 1) * (c0 * 128 + ((8 * i + 4 * g + ((lane >> 2) & 3) + 4 * c0) & 15) * 8 + 4 * (lane & 1));
  }

  float m, l, lost;  // lost: what rounding has added to l
  f16x16 o[C];  // dims 32 d + 8 j + 4 g + i in element 4 j + i
  auto pass = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
    m = -INFINITY;
    l = lost = 0.f;
#pragma unroll
    for (int d = 0; d < C; ++d) o[d] = (f16x16)0.f;
    float p[CAREFUL ? 32 : 1];
    u32x4 part[4][NP];  // weights of 16 keys: 16 q + 4 g + i and 16 q + 8 + 4 g + i
    // keys that this wave's rows see
    auto needed = [&](int t) {
      const int t0 = lo + 64 * t;
      return !empty && t0 <= whi && (a.window <= 0 || t0 + 63 > wlo - a.window);
    };
    auto scores = [&](int t, const uint16_t* buf, auto between) {
      const int t0 = lo + 64 * t;
      f16x16 sc[2];
      if (F8 && W == 4) asm("" : "+v"(kr[0]), "+v"(kr[1]));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h] = (f16x16)0.f;
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) {
          sc[h] = mfma32<BF>(*reinterpret_cast<const u32x4*>(in_tile(buf, kr[i & 1]) + 2 * h * BLK + 256 * i), qf[i], sc[h]);
          between(2 * C * h + i);
        }
      }
      const uint64_t seen = *reinterpret_cast<const uint64_t*>(seen_l[t & 1]);
      if (!(seen == ~0ull && full && t0 + 64 <= min(wlo + 1, hi) && (a.window <= 0 || t0 > whi - a.window))) {
        // bit k: this lane's row sees key t0 + k
        const int end = min(min(pos + 1, hi) - t0, 64), begin = a.window > 0 ? max(pos - a.window + 1 - t0, 0) : 0;
        uint64_t bits = end > begin && begin < 64 ? (~0ull >> (64 - end + begin)) << begin & seen : 0;
        bits >>= 4 * g;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const uint32_t there = __builtin_amdgcn_sbfe((uint32_t)(bits >> (e & 16 ? 32 : 0)), 8 * ((e >> 2) & 3) + (e & 3), 1);
          // (or -infinity)
          sc[e >> 4][e & 15] = __uint_as_float((__float_as_uint(sc[e >> 4][e & 15]) & there) | (0xFF800000u & ~there));
        }
      }
      f4v ks, ve, iv;
      float mx;
      if constexpr (F8) {
        ks = *reinterpret_cast<const f4v*>(ks_l[t & 1]);
        ve = *reinterpret_cast<const f4v*>(ve_l[t & 1]);
        iv = *reinterpret_cast<const f4v*>(iv_l[t & 1]);
        mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float most = sc[q >> 1][8 * (q & 1)];
#pragma unroll
          for (int e = 1; e < 8; ++e) most = fmaxf(most, sc[q >> 1][8 * (q & 1) + e]);
          mx = fmaxf(mx, __builtin_fmaf(most, ks[q], ve[q]));
        }
        mx = max32(mx);
      } else {
        mx = sc[0][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) mx = fmaxf(mx, sc[e >> 4][e & 15]);
        mx = max32(mx) * a.scale;
      }
      // weights are 2^(score - m); m follows the largest score only when that is far ahead of it (a weight is at most
      // 2^AHEAD times the lift then), since moving it costs a product of every sum
      if (__any(mx > m + AHEAD)) {
        const float up = fmaxf(m, mx), down = m == -INFINITY ? 0.f : pow2(m - up);
        m = up;
        l *= down;
        if (LONG) lost *= down;
#pragma unroll
        for (int d = 0; d < C; ++d) o[d] *= down;
      }
      const float base = (m == -INFINITY ? 0.f : m) - LIFT;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[8], some = 0.f;
        const float by = F8 ? ks[q] : a.scale, less = F8 ? ve[q] - base : -base;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = sc[q >> 1][8 * (q & 1) + e];
          v[e] = pow2(__builtin_fmaf(x, by, less));
          if (F8) some += v[e];
          else sum += v[e];
          if constexpr (CAREFUL) p[8 * q + e] = x == -INFINITY ? -1.f : v[e];  // (-1: not seen)
        }
        if (F8) sum = __builtin_fmaf(some, iv[q], sum);
        if constexpr (!CAREFUL) split8<VBF, NP>(v, part[q]);
      }
      if (LONG) add_exactly(l, lost, sum);
      else l += sum;
    };
    auto v_operand = [&](const uint16_t* buf, int q, int d) {
      u32x4 vt;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint2 u = read_tr(in_tile(buf, vr[e]) + q * BLK + 512 * d);
        vt[2 * e] = u.x;
        vt[2 * e + 1] = u.y;
      }
      return vt;
    };
    auto values_with = [&](const uint16_t* buf, auto between) {
      if (F8 && W == 4) asm("" : "+v"(vr[0]), "+v"(vr[1]));
      if constexpr (LONG && !CAREFUL) {
#pragma unroll
        for (int d = 0; d < C; ++d) {
          f16x16 t = (f16x16)0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const u32x4 vt = v_operand(buf, q, d);
#pragma unroll
            for (int i = NP - 1; i >= 0; --i) t = mfma32<VBF>(vt, part[q][i], t);
          }
          o[d] += t;
        }
        for (int q = 0; q < 4; ++q) between(q);
        return;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (CAREFUL) {
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
                const uint2 u = *reinterpret_cast<const uint2*>(buf + q * BLK + ch * 128 + ((k + 4 * ch) & 15) * 8 + 4 * g);
                const f4v v = {wide<VBF>((uint16_t)u.x), wide<VBF>((uint16_t)(u.x >> 16)), wide<VBF>((uint16_t)u.y),
                               wide<VBF>((uint16_t)(u.y >> 16))};
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][4 * j + i] = pk < 0.f ? o[d][4 * j + i] : o[d][4 * j + i] + pk * v[i];
              }
          }
        } else {
#pragma unroll
          for (int d = 0; d < C; ++d) {
            const u32x4 vt = v_operand(buf, q, d);
#pragma unroll
            for (int i = 0; i < NP; ++i) o[d] = mfma32<VBF>(vt, part[q][i], o[d]);
          }
        }
        between(q);
      }
    };
    auto values = [&](const uint16_t* buf) { values_with(buf, [](int) {}); };
    auto ask = [&](int t) {  // (the last tile is copied twice: no branch between the products)
      if (F8) return;
      locate(min(t + 1, tiles - 1));
      ask_page(min(t + 2, tiles - 1));
    };
    auto ask_after = [&](int t) {  // 8 bits: when the next tile is out of the registers
      if (!F8) return;
      load(min(t + 2, tiles - 1));
      ask_pages(min(t + 3, tiles - 1));
    };
    auto step = [&](int t, const uint16_t* kt, uint16_t* k_next, uint16_t* v_next) {
      constexpr int EVERY = 4 * C / PIECES;
      scores(t, kt, [&](int i) {
        if (i % EVERY == 0) piece(i / EVERY, k_next, v_next, t);
        if (i == (PIECES - 1) * EVERY) ask_after(t);
      });
    };
    auto only_copy = [&](int t, uint16_t* k_next, uint16_t* v_next) {
#pragma unroll
      for (int j = 0; j < PIECES; ++j) piece(j, k_next, v_next, t);
      ask_after(t);
    };
    // one tile after the other, the products of those that its rows see
    auto run = [&] {
      auto one = [&](int t, const uint16_t* kt, const uint16_t* vt, uint16_t* k_next, uint16_t* v_next) {
        ask(t);
        if (needed(t)) {
          step(t, kt, k_next, v_next);
          values(vt);
        } else {
          only_copy(t, k_next, v_next);
        }
        arrived<F8>();
      };
      for (int t = 0; t < tiles; t += 2) {
        one(t, k0, v0, k1, v1);
        if (t + 1 < tiles) one(t + 1, k1, v1, k0, v0);
      }
    };
    // the same with four buffers of V, and the tiles before and after those that its rows see in loops of their own: a branch
    // around the products has their sums moved from register to register (15999 tokens 2070 us against 2140 then; of two buffers
    // the branch is up to 3 % faster, but of 8 bits leaves too few registers)
    auto run4 = [&] {
      auto copies = [&](int t, int end) {
        for (; t < end; ++t) {
          ask(t);
          const int b = (t + 1) & 3;
          if constexpr (W == 8) only_copy(t, t & 1 ? k0 : k1, b == 0 ? v0 : b == 1 ? v1 : b == 2 ? v2 : v3);
          else only_copy(t, t & 1 ? k0 : k1, t & 1 ? v0 : v1);
          arrived<F8>();
        }
      };
      auto one = [&](int t, const uint16_t* kt, const uint16_t* vt, uint16_t* k_next, uint16_t* v_next) {
        ask(t);
        if constexpr (F8 && W == 4) {  // (beside the first product there are no registers for the next tile's way)
          scores(t, kt, [](int) {});
          values_with(vt, [&](int q) {
            piece(q, k_next, v_next, t);
            if (q & 1) load_unit(min(t + 2, tiles - 1), q >> 1);
            if (q == 3) ask_pages(min(t + 3, tiles - 1));
          });
        } else {
          step(t, kt, k_next, v_next);
          values(vt);
        }
        arrived<F8>();
      };
      // (from a multiple of the buffers on: what is seen of the tiles up to three before is masked)
      const int end = empty ? 0 : max(min((whi - lo + 64) >> 6, tiles), 0);
      int t = a.window > 0 ? min(max((wlo - a.window - lo + 1) >> 6, 0) & (W == 8 ? ~3 : ~1), end) : 0;
      copies(0, t);
      while (t < end) {
        one(t, k0, v0, k1, v1);
        if (++t == end) break;
        if constexpr (W == 8) {
          one(t, k1, v1, k0, v2);
          if (++t == end) break;
          one(t, k0, v2, k1, v3);
          if (++t == end) break;
          one(t, k1, v3, k0, v0);
        } else {
          one(t, k1, v1, k0, v0);
        }
        ++t;
      }
      copies(t, tiles);
    };
    // the second product of the tile before first
    auto run_late = [&] {
      auto late = [&](int t, const uint16_t* kt, const uint16_t* v_before, uint16_t* k_next, uint16_t* v_next) {
        ask(t);
        if (t > 0 && needed(t - 1)) values(v_before);
        if (needed(t)) step(t, kt, k_next, v_next);
        else only_copy(t, k_next, v_next);
        arrived<F8>();
      };
      for (int t = 0; t < tiles; t += 4) {
        late(t, k0, v3, k1, v1);
        if (t + 1 < tiles) late(t + 1, k1, v0, k0, v2);
        if (t + 2 < tiles) late(t + 2, k0, v1, k1, v3);
        if (t + 3 < tiles) late(t + 3, k1, v2, k0, v0);
      }
      if (needed(tiles - 1)) {
        const int b = (tiles - 1) & 3;
        values(b == 0 ? v0 : b == 1 ? v1 : b == 2 ? v2 : v3);
      }
    };
    if (F8) {
      ask_pages(0);
      load(0);
      ask_pages(min(1, tiles - 1));
    } else {
      ask_page(0);
      locate(0);
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) piece(j, k0, v0, -1);
    if (F8) ask_after(-1);
    else ask_page(min(1, tiles - 1));
    arrived<F8>();
    if constexpr (W == 4 && !F8) {
      run();
    } else if constexpr (W == 4 || CAREFUL) {
      run4();
    } else {
      if (w < 4) run4();
      else run_late();
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
  if (W == 4 && rt.tiles > each) {  // its share: m, l, then four sums at a time, lane by lane
    float* z = a.part + ((int64_t)(tile * c.kv_heads + kvh) * splits + share) * (ROWS * (D + 4)) + w * 32 * (D + 4) + lane;
    z[0] = m;
    z[64] = l;
    f4v* zo = reinterpret_cast<f4v*>(z - lane + 128) + lane;
#pragma unroll
    for (int d = 0; d < C; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        zo[64 * (4 * d + j)] = (f4v){o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
    return;
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

// Joins the shares of row tiles that k_attn_prompt left in the workspace: block (item, d) the dims 32 d .. 32 d + 31 of a row tile
// of a key-value head, its waves and lanes as there.
template <int D>
__global__ __launch_bounds__(256) void k_attn_join(const AttnArgs a) {
  constexpr int C = D / 32;
  const KvView& c = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, g = lane >> 5;
  const int item = blockIdx.x / C, d = blockIdx.x - item * C, tile = item / c.kv_heads, kvh = item - tile * c.kv_heads;
  const RowTile rt = row_tile<128>(a, tile);
  const int each = rt.tiles_each(a.splits), row = 32 * w + n;
  if (rt.tiles <= each || row >= rt.rows) return;
  const int shares = (rt.tiles + each - 1) / each;
  const float* z = a.part + (int64_t)item * a.splits * (128 * (D + 4)) + w * 32 * (D + 4) + lane;
  float m = -INFINITY, l = 0.f;
  f4v o[4] = {(f4v)0.f, (f4v)0.f, (f4v)0.f, (f4v)0.f};
#pragma unroll 4
  for (int i = 0; i < shares; ++i) {
    const float* p = z + (int64_t)i * (128 * (D + 4));
    const f4v* po = reinterpret_cast<const f4v*>(p - lane + 128) + lane + 64 * 4 * d;
    const float m2 = p[0], up = fmaxf(m, m2), base = up == -INFINITY ? 0.f : up, x = pow2(m - base), y = pow2(m2 - base);
    m = up;
    l = l * x + p[64] * y;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = o[j] * x + po[64 * j] * y;
  }
  const int tok = a.by_group(rt.r0 + row), head = kvh * a.group + rt.r0 + row - tok * a.group;
  const int64_t at = (int64_t)(rt.sq.row0 + tok) * a.ldo + (int64_t)head * D + 32 * d + 4 * g;
#pragma unroll
  for (int j = 0; j < 4; ++j) store4(a.out_type, a.out, at + 8 * j, normal(o[j], l));
}

}  // namespace

}  // namespace lw
