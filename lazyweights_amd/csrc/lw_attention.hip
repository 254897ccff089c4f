// Attention over a paged key-value cache: appending with the position rotation, a few new tokens per sequence (decode),
// whole prompts.
//
// Both attention kernels form the scores transposed, S^T = K Q^T: a lane of the product holds several keys of one row (a
// row is a new token's query head; the heads that share a key-value head are rows of the same tile), so the maximum, the
// sum and the rescaling of a row are per-lane scalars, and the weights P^T lie in a lane as the second product's operand
// O^T = V^T P^T takes them. The contraction runs over keys in whatever order the score product left them; V^T's operand,
// read transposed from LDS (ds_read_b64_tr_b16: 16 lanes give 4 keys x 16 dims and get 4 keys of one dim each), follows
// that order.
#include <algorithm>
#include <cmath>

#include "lw_attention.h"
#include "lw_device.h"

namespace lw {

namespace {

typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v LdsS4;
typedef __attribute__((address_space(3))) const u32x4 LdsU4;
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// 16-bit conversions, rounded to nearest even
template <bool BF>
__device__ __forceinline__ float wide(uint16_t h) {
  if (BF) return __uint_as_float((uint32_t)h << 16);
  return (float)__builtin_bit_cast(_Float16, h);
}
template <bool BF>
__device__ __forceinline__ uint32_t narrow2(float x, float y) {  // x in the low half
  if (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v){x, y}, b2v));
  return __builtin_bit_cast(uint32_t, (h2v){(_Float16)x, (_Float16)y});
}

template <bool BF>
__device__ __forceinline__ f4v mfma16(u32x4 a, u32x4 b, f4v c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ f16x16 mfma32(u32x4 a, u32x4 b, f16x16 c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}

// 4 keys x 16 dims of 16 lanes, transposed: lane l of the 16 gets dim l of the 4 keys
__device__ __forceinline__ uint2 read_tr(const uint16_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)p));
}

// v combined with lane ^ 32's (and ^ 16's)
__device__ __forceinline__ uint2 swap32(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return make_uint2(r[0], r[1]);
}
__device__ __forceinline__ uint2 swap16(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return make_uint2(r[0], r[1]);
}
__device__ __forceinline__ float max32(float v) {
  const uint2 r = swap32(__float_as_uint(v));
  return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float max16(float v) {
  const uint2 r = swap16(__float_as_uint(v));
  return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float add32(float v) {
  const uint2 r = swap32(__float_as_uint(v));
  return __uint_as_float(r.x) + __uint_as_float(r.y);
}
__device__ __forceinline__ float add16(float v) {
  const uint2 r = swap16(__float_as_uint(v));
  return __uint_as_float(r.x) + __uint_as_float(r.y);
}

// 2^v by the hardware's instruction (results below 2^-126 are 0: weights are at most 1 and sums at least that of a row's
// largest)
__device__ __forceinline__ float pow2(float v) { return __builtin_amdgcn_exp2f(v); }

__device__ __forceinline__ bool finite(float v) { return __builtin_fabsf(v) < INFINITY; }

// The last s in [0, n) with first(s) <= x, first non-decreasing (0 if there is none): 64 candidates at a time.
template <class F>
__device__ __forceinline__ int last_at_most(int n, int x, F first) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = lane * step;
    const int c = __popcll(__ballot(at < n && first(lo + at) <= x));
    const int skip = max(c - 1, 0) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// a sequence's rows and keys, whatever the arrays hold: rows lie in [0, tokens), keys in the page table
struct Seq {
  int row0, rows, len;
};
__device__ __forceinline__ Seq sequence(const KvView& c, int s) {
  Seq q;
  q.row0 = clampi(c.q_start[s], 0, c.tokens);
  q.rows = clampi(c.q_start[s + 1], q.row0, c.tokens) - q.row0;
  q.len = clampi(c.kv_len[s], 0, c.table_pages << c.page_shift);  // (the host keeps that within 2^30)
  return q;
}

// ── append ──────────────────────────────────────────────────────────────────────────────────────────────────────────

// q_out = R_i q, cache k = R_i k, cache v = v for the batch's new tokens, position i; R_i rotates pairs of the first `rot`
// elements by the angles of row i of cos / sin: (x, y) -> (x c - y s, y c + x s), in 32 bits, rounded once when stored.
// Pairs are elements j and j + rot / 2 ("halves") or 2 j and 2 j + 1 ("neighbours"). A thread takes 8 elements of a head:
// 4 pairs, or 8 that are only copied.
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

// ── shared by the attention kernels ─────────────────────────────────────────────────────────────────────────────────

// element offset of key `key` of the sequence whose table row is `table`, and whether it is there
__device__ __forceinline__ int64_t key_offset(const KvView& c, uint32_t page, int key, bool& there) {
  there = page < c.pages;
  return (there ? (int64_t)page * c.pstride : 0) + (int64_t)(key & ((1 << c.page_shift) - 1)) * c.rstride;
}

template <int OUT>
__device__ __forceinline__ void store4(void* out, int64_t i, f4v v) {
  if (OUT == 0)
    *reinterpret_cast<f4v*>(static_cast<float*>(out) + i) = v;
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) =
        make_uint2(narrow2<OUT == 2>(v[0], v[1]), narrow2<OUT == 2>(v[2], v[3]));
}
__device__ __forceinline__ void store4(int type, void* out, int64_t i, f4v v) {
  if (type == 0) store4<0>(out, i, v);
  else if (type == 1) store4<1>(out, i, v);
  else store4<2>(out, i, v);
}

// weights p as the operand of the second product, in NP 16-bit parts that add up to p (two of fp16: 22 bits, three of
// bf16: 24; one: rounded)
template <bool BF, int NP>
__device__ __forceinline__ void split8(const float* p, u32x4* part) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = p[i];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = narrow2<BF>(r[2 * i], r[2 * i + 1]);
      part[n][i] = w;
      if (n + 1 < NP) {
        r[2 * i] -= wide<BF>((uint16_t)w);
        r[2 * i + 1] -= wide<BF>((uint16_t)(w >> 16));
      }
    }
  }
}

// ── decode ──────────────────────────────────────────────────────────────────────────────────────────────────────────

// A block: one key-value head of a sequence, RT tiles of 16 rows (token, head), one chunk of keys; its 4 waves take the
// chunk's tiles of 32 keys in turn, each on its own (no barrier in the loop), and join at the end. Chunks of a sequence
// that has more than one are joined, in their order, by the block that ends last.
template <int D, bool BF, int RT>
__global__ __launch_bounds__(256) void k_attn_decode(const AttnArgs a) {
  constexpr int C = D / 32, DT = D / 16, NP = BF ? 3 : 2, REGS = 4 * DT + 2;  // REGS: a row tile's state per lane
  constexpr int VB = 4 * 32 * D * 2, MB = 2 * RT * REGS * 64 * 4;
  __shared__ __align__(16) uint8_t smem[VB > MB ? VB : MB];
  __shared__ int last_block;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const KvView& c = a.c;
  const int s = blockIdx.z, kvh = blockIdx.y % c.kv_heads, rb = blockIdx.y / c.kv_heads;
  const Seq sq = sequence(c, s);
  const int R = sq.rows * a.group, r0 = rb * RT * 16;
  if (r0 >= R) return;
  const int past = sq.len - sq.rows;  // row r has position past + r / group
  const int rn = min(r0 + RT * 16, R) - 1, pos_lo = past + r0 / a.group, pos_hi = past + rn / a.group;
  const int hi = min(pos_hi + 1, sq.len);  // keys some row may see: [lo, hi)
  const int lo = a.window > 0 ? max(0, pos_lo - a.window + 1) & ~31 : 0;
  const int keys = max(hi - lo, 0);
  int chunk = a.chunk;
  if ((int64_t)chunk * gridDim.x < keys) chunk = ((keys + gridDim.x - 1) / gridDim.x + 127) & ~127;
  const int active = max((keys + chunk - 1) / chunk, 1), split = blockIdx.x;
  if (split >= active) return;
  const int k0 = lo + split * chunk, k1 = min(hi, k0 + chunk), tiles = (max(k1 - k0, 0) + 31) / 32;

  int pos[RT];
  u32x4 qf[RT][C];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + 16 * t + n;
    pos[t] = r < R ? past + r / a.group : -1;
    const uint16_t* q = a.q + (int64_t)(sq.row0 + r / a.group) * a.ldq + (int64_t)(kvh * a.group + r % a.group) * D + 8 * g;
#pragma unroll
    for (int i = 0; i < C; ++i) qf[t][i] = r < R ? *reinterpret_cast<const u32x4*>(q + 32 * i) : (u32x4)0;
  }
  const int32_t* table = c.table + s * c.tstride;
  const uint16_t* kb = c.k + kvh * c.hstride + 8 * g;
  const uint16_t* vb = c.v + kvh * c.hstride + 8 * g;
  uint16_t* vl = reinterpret_cast<uint16_t*>(smem) + w * 32 * D;  // [half][D / 8 chunks][16 keys][8 dims]

  float m[RT], l[RT];
  f4v o[RT][DT];
  // CAREFUL: products with V only where a row sees the key, so that infinities and NaN elsewhere stay out of it (0 times
  // them is NaN); taken when the first pass ends with a value that is not finite
  auto pass = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
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
      ask_page(min(w + 4, tiles - 1));
    }
    for (int t = w; t < tiles; t += 4) {
      const int t0 = k0 + 32 * t;
      f4v sc[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f4v acc = (f4v)0.f;
#pragma unroll
          for (int i = 0; i < C; ++i) acc = mfma16<BF>(kf[h][i], qf[r][i], acc);
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
      if (t + 4 < tiles) {
        ask(t + 4);
        ask_page(min(t + 8, tiles - 1));
      }
      const bool all = (seen[0] & seen[1]) == 0xFFFFu && t0 + 32 <= min(pos_lo + 1, k1) && r0 + RT * 16 <= R &&
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
        const float base = mx == -INFINITY ? 0.f : mx, down = pow2(m[r] - base);
        m[r] = mx;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = pow2(p[r][e] - base);
          sum += v;
          if (CAREFUL && p[r][e] == -INFINITY) p[r][e] = -1.f;  // not seen: no product
          else p[r][e] = v;
        }
        l[r] = l[r] * down + sum;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] *= down;
        if (!CAREFUL) split8<BF, NP>(p[r], part[r]);
      }
      if (CAREFUL) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          for (int kg = 0; kg < 4; ++kg)
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const float pk = __shfl(p[r][e], 16 * kg + n);
#pragma unroll
              for (int d = 0; d < DT; ++d) {
                const uint2 u = *reinterpret_cast<const uint2*>(
                    vl + (((e >> 2) * (D / 8) + 2 * d + (g >> 1)) * 16 + 4 * kg + (e & 3)) * 8 + 4 * (g & 1));
                const f4v v = {wide<BF>((uint16_t)u.x), wide<BF>((uint16_t)(u.x >> 16)), wide<BF>((uint16_t)u.y),
                               wide<BF>((uint16_t)(u.y >> 16))};
                if (!(pk < 0.f))
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[r][d][i] += pk * v[i];
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
#pragma unroll
  for (int r = 0; r < RT; ++r) l[r] = add32(add16(l[r]));

  // the waves' states, joined pairwise through LDS
  float* mb = reinterpret_cast<float*>(smem);  // [2][RT][REGS][64]
  auto put = [&](int slot) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float* p = mb + (slot * RT + r) * REGS * 64 + lane;
      p[0] = m[r];
      p[64] = l[r];
#pragma unroll
      for (int i = 0; i < 4 * DT; ++i) p[64 * (2 + i)] = o[r][i >> 2][i & 3];
    }
  };
  auto join = [&](int slot) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float* p = mb + (slot * RT + r) * REGS * 64 + lane;
      const float m2 = p[0], mx = fmaxf(m[r], m2), base = mx == -INFINITY ? 0.f : mx;
      const float x = pow2(m[r] - base), y = pow2(m2 - base);
      m[r] = mx;
      l[r] = l[r] * x + p[64] * y;
#pragma unroll
      for (int i = 0; i < 4 * DT; ++i) o[r][i >> 2][i & 3] = o[r][i >> 2][i & 3] * x + p[64 * (2 + i)] * y;
    }
  };
  __syncthreads();
  if (w >= 2) put(w - 2);
  __syncthreads();
  if (w < 2) join(w);
  __syncthreads();
  if (w == 1) put(0);
  __syncthreads();

  auto write = [&](int r, int d, f4v v, float sum) {
    const int row = r0 + 16 * r + n;
    if (row >= R) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = sum == 0.f ? 0.f : v[i] * inv;
    store4(a.out_type, a.out,
           (int64_t)(sq.row0 + row / a.group) * a.ldo + (int64_t)(kvh * a.group + row % a.group) * D + 16 * d + 4 * g, v);
  };
  const int64_t item = ((int64_t)s * c.kv_heads + kvh) * a.row_blocks + rb;
  float* part = a.part + (item * a.splits) * (RT * REGS * 64);
  if (w == 0) {
    join(0);
    if (active == 1) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int d = 0; d < DT; ++d) write(r, d, o[r][d], l[r]);
    } else {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float* p = part + ((int64_t)split * RT + r) * (REGS * 64) + lane;
        p[0] = m[r];
        p[64] = l[r];
#pragma unroll
        for (int i = 0; i < 4 * DT; ++i) p[64 * (2 + i)] = o[r][i >> 2][i & 3];
      }
    }
  }
  if (active == 1) return;
  // the stores above are wave 0's, which counts them
  if (threadIdx.x == 0) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
    const uint32_t before = __hip_atomic_fetch_add(a.count + item, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last_block = before == (uint32_t)active - 1;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  }
  __syncthreads();
  if (!last_block) return;
  if (threadIdx.x == 0) __hip_atomic_store(a.count + item, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // each wave joins its share of the dims, every row's splits in their order
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float* p = part + r * (REGS * 64) + lane;
    float mx = -INFINITY, sum = 0.f;
    for (int i = 0; i < active; ++i) mx = fmaxf(mx, p[(int64_t)i * (RT * REGS * 64)]);
    const float base = mx == -INFINITY ? 0.f : mx;
    f4v acc[(DT + 3) / 4];
#pragma unroll
    for (int d = 0; d < (DT + 3) / 4; ++d) acc[d] = (f4v)0.f;
    for (int i = 0; i < active; ++i) {
      const float* q = p + (int64_t)i * (RT * REGS * 64);
      const float x = pow2(q[0] - base);
      sum += q[64] * x;
#pragma unroll
      for (int d = 0; d < (DT + 3) / 4; ++d)
        if (4 * d + w < DT)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[d][e] += q[64 * (2 + 4 * (4 * d + w) + e)] * x;
    }
#pragma unroll
    for (int d = 0; d < (DT + 3) / 4; ++d)
      if (4 * d + w < DT) write(r, 4 * d + w, acc[d], sum);
  }
}

// ── prompt ──────────────────────────────────────────────────────────────────────────────────────────────────────────

// A block: 128 rows (token, head) of one key-value head of a sequence, 32 per wave, over the keys they see in tiles of 64.
// K and V tiles lie in LDS as [16-key block][D / 8 chunks][16 slots][8 dims], key k of a block in slot (k + 4 chunk) & 15:
// the score product's operand reads (32 keys of a chunk) and the transposed reads of V (4 keys of 4 chunks) are both free
// of bank conflicts. The next tile is loaded into registers while one is worked on.
template <int D, bool BF, int NP>
__global__ __launch_bounds__(256) void k_attn_prompt(const AttnArgs a) {
  constexpr int C = D / 32, ROWS = 128, BLK = D * 16;  // BLK: elements of a 16-key block
  __shared__ __align__(16) uint16_t kl[2][4 * BLK], vl[2][4 * BLK];
  __shared__ uint16_t seen_l[2][4];
  __shared__ int any_bad;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 31, g = lane >> 5;
  const KvView& c = a.c;
  const int kvh = blockIdx.x % c.kv_heads, tile = (int)(gridDim.x / c.kv_heads) - 1 - (int)(blockIdx.x / c.kv_heads);
  // sequence s owns tiles from q_start[s] group / ROWS + s on: at least as many as its rows take
  auto first_tile = [&](int i) {
    return (int)((int64_t)clampi(c.q_start[i], 0, c.tokens) * a.group / ROWS) + i;
  };
  const int s = last_at_most(c.seqs, tile, first_tile);
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
    qf[i] = row < R ? *reinterpret_cast<const u32x4*>(a.q + (int64_t)(sq.row0 + tok) * a.ldq + (int64_t)head * D + 16 * i + 8 * g)
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
        const bool all = seen == ~0ull && full && t0 + 64 <= min(wlo + 1, hi) && (a.window <= 0 || t0 > whi - a.window);
        float p[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) p[e] = sc[e >> 4][e & 15] * a.scale;
        if (!all) {
          const int first = a.window > 0 ? pos - a.window : -1;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int k = 32 * (e >> 4) + 8 * ((e >> 2) & 3) + 4 * g + (e & 3), key = t0 + k;
            if (!(key <= pos && key > first && key < hi && ((seen >> k) & 1))) p[e] = -INFINITY;
          }
        }
        float mx = p[0];
#pragma unroll
        for (int e = 1; e < 32; ++e) mx = fmaxf(mx, p[e]);
        mx = fmaxf(max32(mx), m);
        const float base = mx == -INFINITY ? 0.f : mx, down = pow2(m - base);
        m = mx;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float v = pow2(p[e] - base);
          sum += v;
          if (CAREFUL && p[e] == -INFINITY) p[e] = -1.f;
          else p[e] = v;
        }
        l = l * down + sum;
#pragma unroll
        for (int d = 0; d < C; ++d) o[d] *= down;
        if (CAREFUL) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            for (int kg = 0; kg < 2; ++kg) {
              const float pk = __shfl(p[e], 32 * kg + n);
              const int k = 32 * (e >> 4) + 8 * ((e >> 2) & 3) + 4 * kg + (e & 3);
#pragma unroll
              for (int d = 0; d < C; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // dims 32 d + 8 j + 4 g + i: chunk 4 d + j
                  const int ch = 4 * d + j;
                  const uint2 u = *reinterpret_cast<const uint2*>(
                      &vl[b][(k >> 4) * BLK + ch * 128 + (((k & 15) + 4 * ch) & 15) * 8 + 4 * g]);
                  const f4v v = {wide<BF>((uint16_t)u.x), wide<BF>((uint16_t)(u.x >> 16)), wide<BF>((uint16_t)u.y),
                                 wide<BF>((uint16_t)(u.y >> 16))};
                  if (!(pk < 0.f))
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][4 * j + i] += pk * v[i];
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
  const dim3 grid((uint32_t)p.splits, (uint32_t)(a.c.kv_heads * p.row_blocks), (uint32_t)a.c.seqs);
  if (p.row_tiles == 1) k_attn_decode<D, BF, 1><<<grid, 256, 0, s>>>(a);
  else if (p.row_tiles == 2) k_attn_decode<D, BF, 2><<<grid, 256, 0, s>>>(a);
  else k_attn_decode<D, BF, 4><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
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

DecodePlan decode_plan(int seqs, int kv_heads, int group, int head_dim, int max_new, int max_kv) {
  DecodePlan p;
  const int rows = group * max_new;
  p.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  p.row_blocks = (rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles);
  // chunks so that the launch has about 4 blocks per CU where the keys allow it, of 128 keys (a tile per wave) at least
  const int64_t items = (int64_t)seqs * kv_heads * p.row_blocks, keys = max_kv > 0 ? max_kv : 1;
  const int64_t want = std::max<int64_t>(1, 1024 / items);
  p.chunk = (int)std::max<int64_t>(128, ((keys + want - 1) / want + 127) / 128 * 128);
  p.chunk = std::min(p.chunk, 2048);
  p.splits = (int)((keys + p.chunk - 1) / p.chunk) + 1;  // (a window's first key lies anywhere in a tile of 32)
  p.count_bytes = ((size_t)items * 4 + 255) & ~(size_t)255;
  p.part_bytes = (size_t)items * p.splits * p.row_tiles * (head_dim / 4 + 2) * 64 * 4;
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

hipError_t launch_attn_prompt(const AttnArgs& a, int head_dim, int type, hipStream_t s) {
  if (head_dim == 64) return type == 2 ? prompt_d<64, true>(a, s) : prompt_d<64, false>(a, s);
  if (head_dim == 96) return type == 2 ? prompt_d<96, true>(a, s) : prompt_d<96, false>(a, s);
  return type == 2 ? prompt_d<128, true>(a, s) : prompt_d<128, false>(a, s);
}

}  // namespace lw
