// Appending to a paged key-value cache with the position rotation, and attention of a few new tokens per sequence over it.
#include <algorithm>

#include "lw_attn_device.h"

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
template <int X, bool BF>  // X: type of q, k, v (LW_F32, LW_F16, LW_BF16)
__device__ __forceinline__ f4v load4(const void* p, int64_t i) {
  if (X == 0) return *reinterpret_cast<const f4v*>(static_cast<const float*>(p) + i);
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  return (f4v){wide<X == 2>((uint16_t)u.x), wide<X == 2>((uint16_t)(u.x >> 16)), wide<X == 2>((uint16_t)u.y),
               wide<X == 2>((uint16_t)(u.y >> 16))};
}

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
  f4v x = load4<X, BF>(src, at + e0), y = load4<X, BF>(src, at + e1);
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

  // The waves join: each scales its sums to the rows' maxima over the block and lays them in LDS; then thread x of a row tile
  // adds those of row x & 15, dims 4 (x >> 4) .. (and 64 on), in the waves' order.
  constexpr int RW = 16 * RT, TH = 64 * NW, Q = (4 * D + TH - 1) / TH;  // Q: groups of 4 dims per thread
  const int64_t item = ((int64_t)s * a.row_blocks + rb) * c.kv_heads + kvh;
  const int b0 = (int)(item0 / run), b1 = (int)((item0 + T - 1) / run), active = b1 - b0 + 1;
  // a block has two slots for its parts of items, [RW] (m, l), [RW][D]: 2 b for one that began in an earlier run, and 2 b + 1
  constexpr int SLOT = RW * (D + 2);
  auto slot = [&](int b) { return a.part + (int64_t)(2 * b + (b == b0)) * SLOT; };
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
  float* my_slot = slot(blockIdx.x);
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
    for (int i0 = b0 + cg; i0 <= b1; i0 += NB * groups) {
      f2v h[NB], x[NB], y[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {  // (past the last part: the first of the turn again, with no weight)
        const int b = i0 + i * groups <= b1 ? i0 + i * groups : i0;
        const float* p = slot(b);
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
        if (i0 + i * groups <= b1) {
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

// Work is a list of items (sequence, key-value head, block of RT tiles of 16 (token, head) rows), each as many tiles of 32
// keys as the sequence's rows see together; the launch's blocks take equal runs of the list's tiles, whatever the lengths.
// Within a run, a block's waves take the tiles of an item in turn, each on its own (no barrier in the loop), and join at
// the item's end. An item that lies in several runs is joined, in their order, by the block that ends last.
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
  const KvView& c = a.c;
  const int seqs = c.seqs, kv_heads = c.kv_heads, H = kv_heads * a.row_blocks, chunks = (seqs + 63) >> 6;
  // tiles of each of a sequence's items: those of the keys [lo, len) that its rows see; one where they see none, to write
  // the zeros
  auto first_key = [&](const Seq& q) { return a.window > 0 ? max(0, q.len - q.rows - a.window + 1) & ~31 : 0; };
  auto tiles_of = [&](const Seq& q) { return q.rows ? max((q.len - first_key(q) + 31) >> 5, 1) : 0; };
  if (a.whole) {
    const int s = (int)blockIdx.x / H, hb = (int)blockIdx.x - s * H, rb = hb / kv_heads;
    const Seq sq = sequence(c, s);
    const int T = tiles_of(sq);
    if (T) decode_item<D, BF, RT, NW>(a, smem, ml, pcare, &last_block, s, sq, hb - rb * kv_heads, rb, first_key(sq), 0, T, 0, T, T, lane, w, n, g);
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
    decode_item<D, BF, RT, NW>(a, smem, ml, pcare, &last_block, s, sq, kvh, rb, first_key(sq), (int)(at - item0),
                           (int)(min(item0 + T, to) - item0), item0, T, run, lane, w, n, g);
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
