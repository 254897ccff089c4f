// The division of decode attention's work into equal runs of a list and the join of an item's parts (lw_attn_decode.hip, and
// lw_attn8_decode.hip, which has parts of another division too).
//
// Work is a list of items (sequence, key-value head, block of RT tiles of 16 (token, head) rows), each as many tiles of KEYS
// keys as the sequence's rows see together; the launch's blocks take equal runs of the list's tiles, whatever the lengths.
// Within a run, a block's waves take the tiles of an item in turn, each on its own (no barrier in the loop), and join at
// the item's end. An item that lies in several runs is joined, in their order, by the block that ends last.
#pragma once
#include "lw_attn_device.h"

namespace lw {

namespace {

// Calls item(s, sequence, key-value head, row block, first key, first tile, end tile, item's first tile in the list, its
// tiles, tiles of a run) for the tiles of every item that this block has. csum: [1024] in LDS. WHOLE: a block may have an
// item of its own (AttnArgs::whole).
template <int NW, int KEYS, bool WHOLE, class Item>
__device__ __forceinline__ void walk_items(const AttnArgs& a, uint32_t* csum, int lane, int w, Item&& item) {
  const KvView& c = a.c;
  const int seqs = c.seqs, kv_heads = c.kv_heads, H = kv_heads * a.row_blocks, chunks = (seqs + 63) >> 6;
  // tiles of each of a sequence's items: those of the keys [lo, len) that its rows see; one where they see none, to write
  // the zeros
  auto first_key = [&](const Seq& q) { return a.window > 0 ? max(0, q.len - q.rows - a.window + 1) & ~(KEYS - 1) : 0; };
  auto tiles_of = [&](const Seq& q) { return q.rows ? max((q.len - first_key(q) + KEYS - 1) / KEYS, 1) : 0; };
  if (WHOLE && a.whole) {
    const int s = (int)blockIdx.x / H, hb = (int)blockIdx.x - s * H, rb = hb / kv_heads;
    const Seq sq = sequence(c, s);
    const int T = tiles_of(sq);
    if (T) item(s, sq, hb - rb * kv_heads, rb, first_key(sq), 0, T, 0u, T, (uint32_t)T);
    return;
  }
  // the sequences are held 64 at a time, one per lane, with their tiles and those up to theirs (none yet: of two or three times 64,
  // a block's last waves hold none before the run's first)
  Seq mine = {0, 0, 0};
  uint32_t own = 0, upto = 0;
  int held = -1;
  auto hold = [&](int chunk) __attribute__((always_inline)) {
    held = chunk;
    mine = {0, 0, 0};
    if (64 * chunk + lane < seqs) {
      mine = sequence(c, 64 * chunk + lane);
      mine.len = min(mine.len, a.most_keys);
    }
    upto = own = tiles_of(mine) * H;
    for (int d = 1; d < min(64, seqs); d *= 2) {
      const uint32_t o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
  };
  auto held_seq = [&](int j) __attribute__((always_inline)) {
    return Seq{__builtin_amdgcn_readlane(mine.row0, j), __builtin_amdgcn_readlane(mine.rows, j),
               __builtin_amdgcn_readlane(mine.len, j)};
  };
  uint32_t total;
  if (chunks == 1) {
    hold(0);
    total = __builtin_amdgcn_readlane(upto, min(seqs, 64) - 1);
  } else {
    for (int i = w; i < chunks; i += NW) {
      hold(i);
      if (lane == 63) csum[i] = upto;
    }
    __syncthreads();
    if (w == 0) {
      uint32_t base = 0;
      for (int i = 0; i < chunks; i += 64) {
        uint32_t t = i + lane < chunks ? csum[i + lane] : 0;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const uint32_t o = __shfl_up(t, d);
          if (lane >= d) t += o;
        }
        t += base;
        if (i + lane < chunks) csum[i + lane] = t;
        base = __builtin_amdgcn_readlane(t, 63);
      }
    }
    __syncthreads();
    total = __builtin_amdgcn_readfirstlane(csum[chunks - 1]);
  }
  const uint32_t run = max((total + gridDim.x - 1) >> a.blocks_log2, (uint32_t)NW);
  uint32_t at = min(run * blockIdx.x, total);
  const uint32_t to = min(at + run, total);
  if (at >= to) return;
  // the sequence that holds the run's first tile, and the list's tiles before it
  uint32_t before = 0;
  if (chunks > 1) {
    int ch = 0;
    for (int i = 0; i < chunks; i += 64) ch += __popcll(__ballot(i + lane < chunks && csum[min(i + lane, chunks - 1)] <= at));
    if (ch) before = __builtin_amdgcn_readfirstlane(csum[ch - 1]);
    if (ch != held) hold(ch);
  }
  int j = __ffsll((unsigned long long)__ballot(before + upto > at)) - 1;
  before += __builtin_amdgcn_readlane(upto, j) - __builtin_amdgcn_readlane(own, j);
  Seq sq = held_seq(j);
  int s = 64 * held + j, T = tiles_of(sq), hb = (int)((at - before) / T);
  uint32_t item0 = before + hb * T;  // the item's first tile in the list
  for (;;) {
    int rb = 0, kvh = hb;
    while (kvh >= kv_heads) {
      kvh -= kv_heads;
      ++rb;
    }
    item(s, sq, kvh, rb, first_key(sq), (int)(at - item0), (int)(min(item0 + T, to) - item0), item0, T, run);
    at = item0 = item0 + T;
    if (at >= to) break;
    if (++hb < H) continue;
    hb = 0;
    do {  // (a later sequence has tiles, since the list goes on)
      if ((++s >> 6) != held) hold(s >> 6);
      sq = held_seq(s & 63);
      T = tiles_of(sq);
    } while (T == 0);
  }
}

// The end of an item's tiles in a block: the waves' maxima m, sums l of weights (each lane its own) and sums o of products (dims
// 16 d + 4 g + i of row 16 r + n) become outputs, or this block's part of them; the block that ends an item last joins its
// `active` parts, of which this is number `part`. Each has a slot in the workspace, [RW] (m, l), [RW][D], two for each number from
// base on: the first part's is 2 base + 1, part i's 2 (base + i), so that an item may begin at the number where another ends.
// smem: NW [D][16] floats, done with by every wave itself; ml: [NW][RT][16][2].
template <int D, int RT, int NW>
__device__ __forceinline__ void join_item(const AttnArgs& a, uint8_t* smem, float* ml, int* last_block, const float (&m)[RT],
                                          float (&l)[RT], const f4v (&o)[RT][D / 16], int s, const Seq& sq, int kvh, int rb,
                                          int base_slot, int part, int active, int w, int n, int g) {
  constexpr int DT = D / 16;
  const KvView& c = a.c;
  const Divisor by_group = a.by_group;
  const int R = sq.rows * a.group, r0 = rb * RT * 16;
  // The waves join: each scales its sums to the rows' maxima over the block and lays them in LDS; then thread x of a row tile
  // adds those of row x & 15, dims 4 (x >> 4) .. (and 64 on), in the waves' order.
  constexpr int RW = 16 * RT, TH = 64 * NW, Q = (4 * D + TH - 1) / TH;  // Q: groups of 4 dims per thread
  const int64_t item = ((int64_t)s * a.row_blocks + rb) * c.kv_heads + kvh;
  constexpr int SLOT = RW * (D + 2);
  auto slot = [&](int i) { return a.part + (int64_t)(2 * (base_slot + i) + (i == 0)) * SLOT; };
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] = add32(add16(l[r]));
    if (g == 0) {
      ml[(w * RW + 16 * r + n) * 2] = m[r];
      ml[(w * RW + 16 * r + n) * 2 + 1] = l[r];
    }
  }
  __syncthreads();
  float* ob = reinterpret_cast<float*>(smem);  // [NW waves][D / 4][16 rows][4]
  const int n2 = threadIdx.x & 15, q2 = threadIdx.x >> 4;
  float* my_slot = slot(part);
  auto out_at = [&](int row, int dim) {
    const int tok = by_group(row);
    return (int64_t)(sq.row0 + tok) * a.ldo + (int64_t)(kvh * a.group + row - tok * a.group) * D + dim;
  };
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    auto top = [&](int row) {
      float mx = ml[row * 2];
#pragma unroll
      for (int i = 1; i < NW; ++i) mx = fmaxf(mx, ml[(i * RW + row) * 2]);
      return mx;
    };
    {
      const float mx = top(16 * r + n), x = pow2(m[r] - (mx == -INFINITY ? 0.f : mx));
      if (r) __syncthreads();
#pragma unroll
      for (int d = 0; d < DT; ++d)
        *reinterpret_cast<f4v*>(ob + ((w * (D / 4) + 4 * d + g) * 16 + n) * 4) = o[r][d] * x;
    }
    __syncthreads();
    const int lr = 16 * r + n2, row = r0 + lr;
    const float mx = top(lr), base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) sum += ml[(i * RW + lr) * 2 + 1] * pow2(ml[(i * RW + lr) * 2] - base);
    if (row < R) {
      if (active > 1 && q2 == 0) put2(my_slot + lr * 2, mx, sum);
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        const int dq = q2 + TH / 16 * k;
        if (4 * dq < D) {
          f4v v = *reinterpret_cast<const f4v*>(ob + (dq * 16 + n2) * 4);
#pragma unroll
          for (int i = 1; i < NW; ++i) v += *reinterpret_cast<const f4v*>(ob + ((i * (D / 4) + dq) * 16 + n2) * 4);
          if (active > 1) {
            float* p = my_slot + 2 * RW + lr * D + 4 * dq;
            put2(p, v[0], v[1]);
            put2(p + 2, v[2], v[3]);
          } else {
            store4(a.out_type, a.out, out_at(row, 4 * dq), normal(v, sum));
          }
        }
      }
    }
  }
  if (active == 1) {
    __syncthreads();  // (the next item reuses the memory)
    return;
  }
  // The block that ends last joins the chunks. A block is counted when all its stores (write-through) have arrived: every
  // wave waits for its own, then they meet.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = __hip_atomic_fetch_add(a.count + item, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *last_block = before == (uint32_t)active - 1;
    if (*last_block) __hip_atomic_store(a.count + item, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!*last_block) return;  // (the barriers between this and its next use: at least one per item)
  // Thread x takes 4 dims of a row and, where there are few rows, one of `groups` interleaved shares of the parts, 8 parts'
  // loads in flight; the shares meet in LDS.
  const int rows = min(R - r0, RW), units = rows * (D / 4);
  const int width = units <= 32 ? 32 : units <= 64 ? 64 : units <= 128 ? 128 : TH, groups = TH / width;
  const int cg = threadIdx.x / width;
  for (int u0 = 0; u0 < units; u0 += width) {  // (one turn where groups > 1)
    const int u = u0 + threadIdx.x % width, rr = min(u, units - 1) / (D / 4), dq = min(u, units - 1) - rr * (D / 4);
    float mx = -INFINITY, sum = 0.f;
    f4v acc = (f4v)0.f;
    constexpr int NB = 8;
    for (int i0 = cg; i0 < active; i0 += NB * groups) {
      f2v h[NB], x[NB], y[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {  // (past the last part: the first of the turn again, with no weight)
        const float* p = slot(i0 + i * groups < active ? i0 + i * groups : i0);
        h[i] = get2(p + rr * 2);
        x[i] = get2(p + 2 * RW + rr * D + 4 * dq);
        y[i] = get2(p + 2 * RW + rr * D + 4 * dq + 2);
      }
      float top = mx;
#pragma unroll
      for (int i = 0; i < NB; ++i) top = fmaxf(top, h[i][0]);
      const float base = top == -INFINITY ? 0.f : top, down = pow2(mx - base);
      mx = top;
      sum *= down;
      acc *= down;
#pragma unroll
      for (int i = 0; i < NB; ++i)
        if (i0 + i * groups < active) {
          const float f = pow2(h[i][0] - base);
          sum += h[i][1] * f;
          acc += (f4v){x[i][0], x[i][1], y[i][0], y[i][1]} * f;
        }
    }
    if (groups > 1) {
      float* z = ob + threadIdx.x * 6;
      z[0] = mx;
      z[1] = sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) z[2 + i] = acc[i];
      __syncthreads();
      if (cg == 0) {
        float top = mx;
        for (int i = 1; i < groups; ++i) top = fmaxf(top, ob[(i * width + threadIdx.x) * 6]);
        const float base = top == -INFINITY ? 0.f : top, f0 = pow2(mx - base);
        sum *= f0;
        acc *= f0;
        for (int i = 1; i < groups; ++i) {
          const float* p = ob + (i * width + threadIdx.x) * 6;
          const float f = pow2(p[0] - base);
          sum += p[1] * f;
          acc += (f4v){p[2], p[3], p[4], p[5]} * f;
        }
      }
    }
    if (u < units && cg == 0) store4(a.out_type, a.out, out_at(r0 + rr, 4 * dq), normal(acc, sum));
  }
  __syncthreads();
}

}  // namespace

}  // namespace lw
