// Attention of a few new tokens per sequence over a paged key-value cache held in 8 bits.
#include <algorithm>

#include "lw_attn8_device.h"
#include "lw_attn_list.h"

namespace lw {

namespace {

constexpr int H = 2, KEYS = 16 * H;  // of a tile: blocks of 16 keys that share an exponent, keys

// LDS of a wave: its V tile and the weights of 32 keys, then [D][16] sums
constexpr int decode8_wave(int dim) { return std::max(KEYS * dim + 32 * 16 * 4, 64 * dim); }

// The part of an item that a block has. Items are (sequence, key-value head, block of RT tiles of 16 (token, head) rows), each as
// many tiles of KEYS keys as the sequence's rows see together. A part takes `run` tiles at most, the tiles of all items / spare, so that
// items + spare blocks are enough whatever the lengths; parts are of one item alone, so that a block has one pass, one join and is
// done, and what it waits for in turn is covered by the blocks beside it. (With equal runs of the list of all items a block goes
// from item to item, each waited for anew: us with runs / parts, 256 sequences of 100-2000 keys, 8 heads of 128: 119 / 91, 30 of
// them 29 / 19, one of 30000 26 / 20.)
struct Part {
  Seq sq;
  int s, kvh, rb, lo, t_from, t_to;
  int base_slot, part, active;
};
template <int NW>
__device__ __forceinline__ bool find_part(const Attn8Args& args, uint32_t* tiles_l, uint32_t* parts_l, int lane, int w, Part& p) {
  const AttnArgs& a = args.a;
  const KvView& c = a.c;
  const int seqs = c.seqs, kv_heads = c.kv_heads, of_seq = kv_heads * a.row_blocks, chunks = (seqs + 63) >> 6;
  // tiles of each of a sequence's items: those of the keys [lo, len) that its rows see; one where they see none, to write
  // the zeros
  auto first_key = [&](const Seq& q) { return a.window > 0 ? max(0, q.len - q.rows - a.window + 1) & ~(KEYS - 1) : 0; };
  auto tiles_of = [&](const Seq& q) { return q.rows ? max((q.len - first_key(q) + KEYS - 1) / KEYS, 1) : 0; };
  p.base_slot = p.part = 0;
  p.active = 1;
  if (a.whole) {
    p.s = (int)blockIdx.x / of_seq;
    const int hb = (int)blockIdx.x - p.s * of_seq;
    p.rb = hb / kv_heads;
    p.kvh = hb - p.rb * kv_heads;
    p.sq = sequence(c, p.s);
    p.lo = first_key(p.sq);
    p.t_from = 0;
    p.t_to = tiles_of(p.sq);
    return p.t_to > 0;
  }
  // the sequences are held 64 at a time, one per lane, with their tiles and parts and those up to theirs
  Seq mine = {0, 0, 0};
  uint32_t T = 0, tiles = 0, parts = 0;
  auto hold = [&](int chunk) __attribute__((always_inline)) {
    mine = {0, 0, 0};
    if (64 * chunk + lane < seqs) {
      mine = sequence(c, 64 * chunk + lane);
      mine.len = min(mine.len, a.most_keys);
    }
    T = tiles_of(mine);
  };
  auto upto = [&](uint32_t v) __attribute__((always_inline)) {
    for (int d = 1; d < min(64, seqs); d *= 2) {
      const uint32_t o = __shfl_up(v, d);
      if (lane >= d) v += o;
    }
    return v;
  };
  auto run_of = [&](uint32_t total) { return max((uint32_t)args.by_spare((int)total + args.by_spare.of - 1), (uint32_t)NW); };
  uint32_t run, tiles_before = 0, parts_before = 0, at = blockIdx.x;
  int chunk = 0;
  if (chunks == 1) {
    hold(0);
    tiles = upto(T * of_seq);
    run = run_of(__builtin_amdgcn_readlane(tiles, min(seqs, 64) - 1));
    parts = upto((T + run - 1) / run * of_seq);
  } else {
    // sums up to each 64th sequence, of tiles and then, with the run that these give, of parts
    auto sums = [&](uint32_t* l, auto value) __attribute__((always_inline)) {
      for (int i = w; i < chunks; i += NW) {
        hold(i);
        const uint32_t v = upto(value());
        if (lane == 63) l[i] = v;
      }
      __syncthreads();
      if (w == 0) {
        uint32_t base = 0;
        for (int i = 0; i < chunks; i += 64) {
          uint32_t t = i + lane < chunks ? l[i + lane] : 0;
#pragma unroll
          for (int d = 1; d < 64; d *= 2) {
            const uint32_t o = __shfl_up(t, d);
            if (lane >= d) t += o;
          }
          t += base;
          if (i + lane < chunks) l[i + lane] = t;
          base = __builtin_amdgcn_readlane(t, 63);
        }
      }
      __syncthreads();
    };
    sums(tiles_l, [&] { return T * of_seq; });
    run = run_of(__builtin_amdgcn_readfirstlane(tiles_l[chunks - 1]));
    sums(parts_l, [&] { return (T + run - 1) / run * of_seq; });
    for (int i = 0; i < chunks; i += 64) chunk += __popcll(__ballot(i + lane < chunks && parts_l[min(i + lane, chunks - 1)] <= at));
    if (chunk && chunk < chunks) {
      tiles_before = __builtin_amdgcn_readfirstlane(tiles_l[chunk - 1]);
      parts_before = __builtin_amdgcn_readfirstlane(parts_l[chunk - 1]);
    }
    __syncthreads();  // (the memory is used again)
    if (chunk >= chunks) return false;
    hold(chunk);
    tiles = upto(T * of_seq);
    parts = upto((T + run - 1) / run * of_seq);
  }
  at -= parts_before;
  const int j = __ffsll((unsigned long long)__ballot(parts > at)) - 1;
  if (j < 0) return false;
  auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane(v, j); };
  p.sq = Seq{(int)of(mine.row0), (int)of(mine.rows), (int)of(mine.len)};
  p.s = 64 * chunk + j;
  const uint32_t t = of(T), each = (t + run - 1) / run;
  at -= of(parts) - each * of_seq;
  tiles_before += of(tiles) - t * of_seq;
  const uint32_t hb = at / each;
  p.rb = hb / kv_heads;
  p.kvh = hb - p.rb * kv_heads;
  p.part = at - hb * each;
  p.active = each;
  p.base_slot = (tiles_before + hb * t) / run;  // (two items' first parts, of runs at least, have not one number)
  p.lo = first_key(p.sq);
  p.t_from = p.part * run;
  p.t_to = min(p.t_from + run, t);
  return true;
}

template <int D, bool BF, int RT, int NW>
__device__ __forceinline__ void decode8_part(const Attn8Args& args, uint8_t* smem, float* ml, int* last_block, const Part& p0, int lane,
                                             int w, int n, int g) {
  constexpr int C = D / 32, DT = D / 16, NP = 2, FULL = D / 64, TAIL = C % 2;
  constexpr float LIFT = lift<false>(0);
  constexpr int WAVE = decode8_wave(D);
  const AttnArgs& a = args.a;
  const KvView& c = a.c;
  const Seq& sq = p0.sq;
  const int s = p0.s, kvh = p0.kvh, rb = p0.rb, lo = p0.lo, t_from = p0.t_from, t_to = p0.t_to;
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
  u32x4* ql = reinterpret_cast<u32x4*>(smem + NW * WAVE + w * RT * 16 * D * 2) + lane;
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
  uint8_t* vl = smem + w * WAVE;

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
        float* pl = reinterpret_cast<float*>(vl + KEYS * D);  // [32 keys][16 rows]
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

  join_item<D, RT, NW>(a, smem, ml, last_block, m, l, o, s, sq, kvh, rb, p0.base_slot, p0.part, p0.active, w, n, g);
}

// Attention over 8 bits: scores S^T = K Q^T of 16 rows and 32 keys of each wave's tiles, O^T = V^T P^T, numbers made 16 bits of
// q's type (K) and fp16 (V) in registers, where both are exact: an instruction for two numbers, at the full rate. K's power of two is a
// factor of a block's scores; V's enters the weight, 2^(score + e - m) with m the largest score + e, so that weights need no more range
// than before, and the sum of weights takes it off again by the block. Bytes of V go to LDS as they are and come back transposed
// (ds_read_b64_tr_b8), eight keys of a dim per lane.
//
// Bound by memory: 2 D + 1/8 bytes a key and key-value head. A wave has a tile of 32 keys (8 KB at D = 128) on its way while it works on the
// one before; 128 registers leave room for 16 waves a CU (64 keys a tile and 8 waves: 64 sequences of 500-16000 keys 127 us against
// 123, 256 of 100-2000 94 against 91). us, and of the bytes: 64 sequences of 500-16000 keys, 8 heads of 128: 120 (580 MB: 4.8
// TB/s); one of 131071: 55 (268 MB: 4.9, 5.4 in the loop); 4 x 5 tokens of 32 heads of 96 over 301-5003: 11.7 (50 MB); one of 778: 8.2.
// A launch without its bytes is 6 us (200 keys: 6.7): start, lengths 1, page and first tile 1.5, stores of a part until they are
// counted 2; the last part's join 2 to 4 more.
//
// RUNS: a block has an equal run of the list of all items' tiles (walk_items) instead of a part.
template <int D, bool BF, int RT, int NW, bool RUNS>
__global__ __launch_bounds__(64 * NW, RT == 1 && !RUNS ? 4 : 2) void k_attn8_decode(const Attn8Args args) {
  // the waves' V tiles, and behind each the weights of 32 keys of the careful pass (after the loop their sums); then, of more than one
  // row tile, q
  __shared__ __align__(16) uint8_t smem[NW * decode8_wave(D) + (RT > 1 ? NW * RT * 16 * D * 2 : 0)];
  __shared__ float ml[NW * 16 * RT * 2];
  __shared__ uint32_t csum[RUNS ? 1024 : 1];
  __shared__ int last_block;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  if constexpr (RUNS) {
    walk_items<NW, KEYS, false>(args.a, csum, lane, w, [&](int s, const Seq& sq, int kvh, int rb, int lo, int t_from, int t_to, uint32_t item0,
                                                      int T, uint32_t run) __attribute__((always_inline)) {
      // (a block's number is that of its run in the list)
      const int b0 = (int)(item0 / run), b1 = (int)((item0 + T - 1) / run);
      const Part p = {sq, s, kvh, rb, lo, t_from, t_to, b0, (int)blockIdx.x - b0, b1 - b0 + 1};
      decode8_part<D, BF, RT, NW>(args, smem, ml, &last_block, p, lane, w, n, g);
    });
  } else {
    Part p = {};
    uint32_t* sums_l = reinterpret_cast<uint32_t*>(smem);  // of tiles and of parts of the sequences up to each 64th
    if (find_part<NW>(args, sums_l, sums_l + 1024, lane, w, p))
      decode8_part<D, BF, RT, NW>(args, smem, ml, &last_block, p, lane, w, n, g);
  }
}

template <int D, bool BF>
hipError_t decode8_d(const Attn8Args& a, const DecodePlan& p, hipStream_t s) {
  const dim3 grid((uint32_t)p.blocks);
  if (p.row_tiles == 2) k_attn8_decode<D, BF, 2, 4, false><<<grid, 256, 0, s>>>(a);
  else if (D == 128 && p.runs) k_attn8_decode<128, BF, 1, 4, true><<<grid, 256, 0, s>>>(a);
  else if (p.waves == 8) k_attn8_decode<D, BF, 1, 8, false><<<grid, 512, 0, s>>>(a);
  else k_attn8_decode<D, BF, 1, 4, false><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

DecodePlan decode8_plan(int seqs, int kv_heads, int group, int head_dim, int max_new, int max_kv) {
  DecodePlan p;
  const int rows = group * max_new;
  // Two row tiles per item share what is read, where there is much to read (us with two / one: 8 sequences of 1000-8000 keys, 8 heads of
  // 128, 20 rows 29 / 34, 64 of 500-16000 194 / 242; one of 500, 64 rows 15 / 10, 4 of 300-5000 23 / 22).
  p.row_tiles = rows <= 16 || (int64_t)seqs * kv_heads * max_kv < 1 << 18 ? 1 : 2;
  p.row_blocks = (rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles);
  const int64_t items = (int64_t)seqs * kv_heads * p.row_blocks, tiles = items * (max_kv / 32 + 2);
  // A block per item, which has nothing to find out and nothing to join: where an item is one or two tiles for each wave (200 keys 6.7
  // us), and where there are many, none long (us against parts: 1024 items of 300-1000 keys 42 / 44, 2048 of 100-2000 91 / 95; 512 of
  // two row tiles and 100-3000 keys 53 / 62; but 240 of 100-2000 20 / 18).
  p.whole = items <= 1 << 20 && (max_kv <= 256 || (p.row_tiles == 2 ? items >= 512 && max_kv <= 4096 : items >= 1024 && max_kv <= 2048));
  // Equal runs of the list of all items, for 512 blocks, where there are many and not short ones: what a CU has to read is then the same
  // everywhere, and a CU takes little more than its share of the card's rate (parts end unevenly, whatever their number). us with runs
  // / parts: 512 items of 500-16000 keys 144 / 148, of 8000 182 / 189, of 1500-3500 74 / 101, of 500-4000 62 / 75, 2048 of 1500-3500 235 /
  // 306; 248 of 500-16000 67 / 84, 192 of 1500-3500 29 / 33; 128 of 20000-60000 207 / 228, of 8000 60 / 61, of 1500-3500 24 / 23; but
  // 2048 of 100-2000 119 / 88. Heads of 96, whose tiles are smaller, need more waves beside one another: 512 of 500-16000 124 / 101.
  // All of these with the longest length as the bound. The host knows bounds alone, and under a bound far above the lengths short items go in
  // runs too: 512 items of 100-2000 keys 34 with a bound of 8192 and more, 25 of 2000; of 30-500 23 and 14; 2048 of 100-2000 113 and 86, of
  // 200-800 62 and 44; 1024 of 300-1500 48 and 40 (1500-3500 are 62 with any).
  p.runs = !p.whole && p.row_tiles == 1 && head_dim == 128 && (items > 128 ? max_kv > 2048 : items >= 64 && max_kv > 16384);
  p.blocks_log2 = 9;
  // Parts: few items in about as many blocks as there are CUs (the more parts of an item, the longer its join: one of 131071 keys with
  // 248 spare blocks 58 us, 504 60, 1016 82; one of 30000 19, 25, 41), some more for items that are shorter (128 of 1000-3000 keys with
  // 248 24, 504 20); many items so that a part is of some 100 tiles at the bounds (512 of two row tiles, 500-16000 keys, with 1024
  // 183, 2048 194; 248 items, us with many / few: heads of 64, 500-16000 keys 36 / 48, of 128, 300-1500 20 / 21; but 160 of heads
  // of 96, 1500-3500 24 / 21, and 248 of two row tiles 71 / 59).
  const int64_t few = items <= 64 ? 256 - items : std::max<int64_t>(512 - items, 256);
  const int64_t many = std::min<int64_t>(std::max<int64_t>(tiles / 96, 512), p.row_tiles == 2 ? 1024 : 2048);
  p.spare = (int)std::max<int64_t>(1, std::min<int64_t>(items > (p.row_tiles == 2 ? 256 : 192) ? many : few, (tiles + 3) / 4));
  p.blocks = p.runs ? 1 << p.blocks_log2 : (int)std::min<int64_t>(items + (p.whole ? 0 : p.spare), 1 << 30);
  // 8 waves where one block of a CU has a long part: half as many parts would leave half of the CUs idle, and 4 waves ask for too little
  // at a time (one of 131071 keys 55 / 58; one of 778 10.4 / 8.2)
  p.waves = !p.whole && items <= 64 && tiles / p.spare >= 64 ? 8 : 4;
  p.count_bytes = ((size_t)items * 4 + 255) & ~(size_t)255;
  // (two slots for every run of the list: blocks of runs have one each, parts as many as there are spare blocks, and one begun)
  p.part_bytes = (size_t)(p.runs ? p.blocks : p.spare + 1) * 2 * p.row_tiles * 16 * (head_dim + 2) * 4;
  // (and 2^13 fewer, so that a run of the list of all of them, rounded up, is counted in 31 bits)
  p.most_keys = (int)std::min<int64_t>(1 << 30, (((int64_t)1 << 36) - (1 << 18)) / std::max<int64_t>(items, 1) - 128);
  return p;
}

hipError_t launch_attn8_decode(const Attn8Args& args, const DecodePlan& p, int head_dim, int q_type, hipStream_t s) {
  Attn8Args a = args;
  a.by_spare = divisor(p.spare);
  if (head_dim == 64) return q_type == 2 ? decode8_d<64, true>(a, p, s) : decode8_d<64, false>(a, p, s);
  if (head_dim == 96) return q_type == 2 ? decode8_d<96, true>(a, p, s) : decode8_d<96, false>(a, p, s);
  return q_type == 2 ? decode8_d<128, true>(a, p, s) : decode8_d<128, false>(a, p, s);
}

}  // namespace lw
