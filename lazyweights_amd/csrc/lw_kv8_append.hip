// Appending to a paged key-value cache held in 8 bits.
#include <algorithm>

#include "lw_attn8_device.h"

namespace lw {

namespace {

__device__ __forceinline__ int exponent(int8_t e) { return clampi(e, -kMostExp, kMostExp); }

// The least e with most <= 448 2^e, 448 = 1.75 * 2^8: of a magnitude 1.f 2^k that is k - 8, and one more past 1.75
__device__ __forceinline__ int exponent_of(float most) {
  return clampi((int)((__float_as_uint(most) + 0x1FFFFFu) >> 23) - 127 - 8, -kMostExp, kMostExp);
}

// four numbers of 8 bits, v in the lowest first, rounded to nearest even; what is not finite is NaN
__device__ __forceinline__ uint32_t to8(f4v v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = finite(v[i]) ? fminf(fmaxf(v[i], -448.f), 448.f) : NAN;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
}

// x and y, pairs (x, y) or, as neighbours, pairs within each, by the angles c, n: every product and sum rounded for itself
__device__ __forceinline__ void rotate(f4v& x, f4v& y, f4v c, f4v n, bool neighbours) {
#pragma clang fp contract(off)
  const f4v p = neighbours ? (f4v){x[0], x[2], y[0], y[2]} : x, q = neighbours ? (f4v){x[1], x[3], y[1], y[3]} : y;
  const f4v pc = p * c, qn = q * n, qc = q * c, pn = p * n;
  const f4v t = pc - qn, w = qc + pn;
  x = neighbours ? (f4v){t[0], w[0], t[1], w[1]} : t;
  y = neighbours ? (f4v){t[2], w[2], t[3], w[3]} : w;
}

// As k_kv_append, with keys and values quantized: a block of 2 D threads has the 16 rows that share an exponent, of the keys and
// the values of a head, a thread 8 elements of a row of each: the largest magnitude of the new rows gives the exponent, and rows from
// before, if there are any and it has grown, are rounded to it. The rows of a sequence lie in at most
// rows / 16 + 2 such blocks, so that sequence s has the items from q_start[s] / 16 + 2 s on. The last blocks of the launch rotate q, a
// thread 8 elements.
//
// One pass: what is rounded to an exponent stays in registers while it is found (a block of threads has all of a block of rows; a
// barrier between). Bound by memory where there is much of it (16383 tokens of 32 q and 8 kv heads of 128, fp32 in: 579 MB in 100 us,
// 5.8 TB/s, seven tenths of it read), else by latency: sequence, then page and rows, then old rows and exponents, each asked for at once
// (one token 3.9 us; 1009 tokens of 7 prompts, 32 and 32 heads of 64, bf16 in, 21 MB: 8.6; with blocks for keys and for values apart, and
// a sequence's numbers, its page and the rows waited for in turn, 4.1, 9.7 and the long one 114).
template <int D, int X, bool BF>
__global__ __launch_bounds__(2 * D) void k_kv8_append(const Append8Args args, uint32_t kv_blocks) {
  constexpr int U = D / 8, WAVES = 2 * D / 64;
  const AppendArgs& a = args.a;
  const KvView& c = a.c;
  __shared__ float most_l[WAVES][2];
  const int unit = threadIdx.x % U;
  auto pieces = [&](int u, bool turn, int& e0, int& e1) {
    e0 = turn && !a.neighbours ? 4 * u : 8 * u;
    e1 = turn && !a.neighbours ? a.rot / 2 + 4 * u : 8 * u + 4;
  };
  auto angles = [&](int u, int pos, f4v& cs, f4v& sn) {
    const int64_t r = (int64_t)min(pos, a.rope_rows - 1) * (a.rot / 2) + 4 * u;
    cs = *reinterpret_cast<const f4v*>(a.cos + r);
    sn = *reinterpret_cast<const f4v*>(a.sin + r);
  };
  // the sequence s that has `at` of what first(s, q_start[s]) counts, `s` if that is right: start, end and length in one load
  auto find = [&](int& s, int at, auto first) {
    const int lane = threadIdx.x & 63;
    int from, to, len;
    auto read = [&] {
      const int v = *(lane == 2 ? c.kv_len + s : c.q_start + s + (lane == 1));
      from = __builtin_amdgcn_readlane(v, 0), to = __builtin_amdgcn_readlane(v, 1), len = __builtin_amdgcn_readlane(v, 2);
    };
    read();
    if (!((first(s, from) <= at) & (at < first(s + 1, to)))) {
      s = last_at_most(c.seqs, at, [&](int i) { return first(i, c.q_start[i]); });
      read();
    }
    return sequence(c, from, to, len);
  };
  if (blockIdx.x >= kv_blocks) {
    const int parts = (a.heads + 15) / 16, b = blockIdx.x - kv_blocks, row = b / parts;
    const int head = (b - row * parts) * 16 + threadIdx.x / U, h = min(head, a.heads - 1);  // (all lanes search)
    const bool turn = 8 * unit < a.rot;
    int e0, e1;
    pieces(unit, turn, e0, e1);
    const int64_t at = a.ldq * row + (int64_t)h * D;
    f4v x = load4<X>(a.q, at + e0), y = load4<X>(a.q, at + e1), cs, sn;
    int s = min(row, c.seqs - 1);
    const Seq sq = find(s, row, [&](int, int from) { return from; });
    const int pos = sq.len - sq.rows + (row - sq.row0);
    if (head >= a.heads || row < sq.row0 || row >= sq.row0 + sq.rows || pos < 0) return;
    if (turn) {
      angles(unit, pos, cs, sn);
      rotate(x, y, cs, sn, a.neighbours);
    }
    uint16_t* dst = a.q_out + a.ldo * row + (int64_t)h * D;
    *reinterpret_cast<uint2*>(dst + e0) = make_uint2(narrow2<BF>(x[0], x[1]), narrow2<BF>(x[2], x[3]));
    *reinterpret_cast<uint2*>(dst + e1) = make_uint2(narrow2<BF>(y[0], y[1]), narrow2<BF>(y[2], y[3]));
    return;
  }
  const int item = blockIdx.x / c.kv_heads, h = blockIdx.x - item * c.kv_heads;
  auto first_item = [&](int i, int from) { return clampi(from, 0, c.tokens) / kExpBlock + 2 * i; };
  int s = min((int)((int64_t)item * 16 / 33), c.seqs - 1);  // one new token per sequence first: 33 items for 16 of them
  const Seq sq = find(s, item, first_item);
  // (items of no sequence: those before the first one's, whose rows may begin behind others)
  const int past = sq.len - sq.rows, p0 = max(past, 0), nth = item - first_item(s, sq.row0);
  const int64_t block = (int64_t)p0 / kExpBlock + nth;
  if (sq.rows == 0 || nth < 0 || block * kExpBlock >= sq.len) return;
  const int begin = (int)block * kExpBlock, mask = (1 << c.page_shift) - 1;
  const int pos = begin + (int)threadIdx.x / U;
  const bool fresh = pos >= p0 && pos < sq.len, older = pos < p0, turn = 8 * unit < a.rot;
  int e0[2], e1[2];  // of keys, of values
  pieces(unit, turn, e0[0], e1[0]);
  pieces(unit, false, e0[1], e1[1]);
  // the page, the new rows and their angles on their way together (a number that the compiler takes for one of each lane: it would
  // wait for the page of all lanes at once), then the old rows and exponents
  int at_page = begin >> c.page_shift;
  asm("" : "+v"(at_page));
  const uint32_t of_lane = (uint32_t)c.table[s * c.tstride + at_page];
  f4v x[2], y[2], cs = (f4v)1.f, sn = (f4v)0.f;
  x[0] = x[1] = y[0] = y[1] = (f4v)0.f;
  if (fresh) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = (i ? a.ldv : a.ldk) * (sq.row0 + pos - past) + (int64_t)h * D;
      x[i] = load4<X>(i ? a.v : a.k, at + e0[i]);
      y[i] = load4<X>(i ? a.v : a.k, at + e1[i]);
    }
    if (turn) angles(unit, pos, cs, sn);
  }
  const uint32_t page = (uint32_t)__builtin_amdgcn_readfirstlane((int)of_lane);
  if (page >= c.pages) return;
  uint8_t* dst[2];
  int8_t* ex[2];
  uint32_t was0[2] = {0, 0}, was1[2] = {0, 0};
  int e_old[2] = {-kMostExp, -kMostExp};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    dst[i] = reinterpret_cast<uint8_t*>(i ? c.v : c.k) + page * c.pstride + h * c.hstride + (pos & mask) * c.rstride;
    ex[i] = (i ? args.e.v : args.e.k) + page * args.e.pstride + h * args.e.hstride + (begin & mask) / kExpBlock;
  }
  if (begin < p0) {
    e_old[0] = *ex[0];
    e_old[1] = *ex[1];
    if (older) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        was0[i] = *reinterpret_cast<const uint32_t*>(dst[i] + e0[i]);
        was1[i] = *reinterpret_cast<const uint32_t*>(dst[i] + e1[i]);
      }
    }
  }
  if (fresh && turn) rotate(x[0], y[0], cs, sn, a.neighbours);
  float most[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      most[i] = fmaxf(most[i], finite(x[i][j]) ? fabsf(x[i][j]) : 0.f);
      most[i] = fmaxf(most[i], finite(y[i][j]) ? fabsf(y[i][j]) : 0.f);
    }
#pragma unroll
    for (int d = 32; d; d /= 2) most[i] = fmaxf(most[i], __shfl_xor(most[i], d));
  }
  if ((threadIdx.x & 63) == 0) {
    most_l[threadIdx.x >> 6][0] = most[0];
    most_l[threadIdx.x >> 6][1] = most[1];
  }
  __syncthreads();
  uint32_t to0[2], to1[2];
  int e[2];
  bool put[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int w = 0; w < WAVES; ++w) most[i] = fmaxf(most[i], most_l[w][i]);
    const int old = exponent((int8_t)e_old[i]);
    e[i] = max(exponent_of(most[i]), old);
    put[i] = fresh || (older && e[i] > old);
    const float down = two_to(fresh ? -e[i] : old - e[i]);  // (-96 at least)
    to0[i] = to8((fresh ? x[i] : from8(was0[i])) * down);
    to1[i] = to8((fresh ? y[i] : from8(was1[i])) * down);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // (all loads are here: none is waited for behind a store)
    if (threadIdx.x == 0) *ex[i] = (int8_t)e[i];
    if (put[i]) {
      *reinterpret_cast<uint32_t*>(dst[i] + e0[i]) = to0[i];
      *reinterpret_cast<uint32_t*>(dst[i] + e1[i]) = to1[i];
    }
  }
}

template <int D, int X>
hipError_t append8_d(const Append8Args& a, int q_type, hipStream_t s) {
  const uint32_t items = (uint32_t)(a.a.c.tokens / kExpBlock + 2 * a.a.c.seqs), kv_blocks = items * (uint32_t)a.a.c.kv_heads;
  const dim3 grid(kv_blocks + (a.a.q ? (uint32_t)a.a.c.tokens * (uint32_t)((a.a.heads + 15) / 16) : 0));
  if (q_type == 2) k_kv8_append<D, X, true><<<grid, 2 * D, 0, s>>>(a, kv_blocks);
  else k_kv8_append<D, X, false><<<grid, 2 * D, 0, s>>>(a, kv_blocks);
  return hipGetLastError();
}
template <int D>
hipError_t append8_x(const Append8Args& a, int q_type, int x_type, hipStream_t s) {
  return x_type == 0 ? append8_d<D, 0>(a, q_type, s) : x_type == 1 ? append8_d<D, 1>(a, q_type, s) : append8_d<D, 2>(a, q_type, s);
}

}  // namespace

hipError_t launch_append8(const Append8Args& a, int head_dim, int q_type, int x_type, hipStream_t s) {
  if (head_dim == 64) return append8_x<64>(a, q_type, x_type, s);
  if (head_dim == 96) return append8_x<96>(a, q_type, x_type, s);
  return append8_x<128>(a, q_type, x_type, s);
}

}  // namespace lw
