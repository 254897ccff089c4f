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

// As k_kv_append, with keys and values quantized: a block of 2 D threads has the 16 rows that share an exponent, of the keys or
// the values of a head, a thread 8 elements of a row: the largest magnitude of the new rows gives the exponent, and rows from
// before, if there are any and it has grown, are rounded to it. The rows of a sequence lie in at most
// rows / 16 + 2 such blocks, so that sequence s has the items from q_start[s] / 16 + 2 s on. The last blocks of the launch rotate q, a
// thread 8 elements.
//
// One pass: what is rounded to an exponent stays in registers while it is found (a block of threads has all of a block of rows; a
// barrier between). Bound by memory where there is much of it (16383 tokens of 32 q and 8 kv heads of 128, fp32 in: 579 MB in 114 us,
// 5.1 TB/s, where a copy of 1 GiB reaches 5.2), else by latency: sequence, length, page, old rows and exponent, one after the other
// (one token 4.1 us; 1009 tokens of 7 prompts, 32 and 32 heads of 64, bf16 in, 21 MB: 9.7).
template <int D, int X, bool BF>
__global__ __launch_bounds__(2 * D) void k_kv8_append(const Append8Args args, uint32_t kv_blocks) {
  constexpr int U = D / 8, WAVES = 2 * D / 64;
  const AppendArgs& a = args.a;
  const KvView& c = a.c;
  __shared__ float most_l[WAVES];
  const int unit = threadIdx.x % U;
  auto pieces = [&](int u, bool turn, int& e0, int& e1) {
    e0 = turn && !a.neighbours ? 4 * u : 8 * u;
    e1 = turn && !a.neighbours ? a.rot / 2 + 4 * u : 8 * u + 4;
  };
  auto turned = [&](f4v& x, f4v& y, int u, int pos) {
    const int64_t r = (int64_t)min(pos, a.rope_rows - 1) * (a.rot / 2) + 4 * u;
    rotate(x, y, *reinterpret_cast<const f4v*>(a.cos + r), *reinterpret_cast<const f4v*>(a.sin + r), a.neighbours);
  };
  if (blockIdx.x >= kv_blocks) {
    const int parts = (a.heads + 15) / 16, b = blockIdx.x - kv_blocks, row = b / parts;
    const int h = (b - row * parts) * 16 + threadIdx.x / U;
    int s = min(row, c.seqs - 1);
    if (!(c.q_start[s] <= row && row < c.q_start[s + 1])) s = last_at_most(c.seqs, row, [&](int i) { return c.q_start[i]; });
    const Seq sq = sequence(c, s);
    const int pos = sq.len - sq.rows + (row - sq.row0);
    if (h >= a.heads || row < sq.row0 || row >= sq.row0 + sq.rows || pos < 0) return;
    const bool turn = 8 * unit < a.rot;
    int e0, e1;
    pieces(unit, turn, e0, e1);
    const int64_t at = a.ldq * row + (int64_t)h * D;
    f4v x = load4<X>(a.q, at + e0), y = load4<X>(a.q, at + e1);
    if (turn) turned(x, y, unit, pos);
    uint16_t* dst = a.q_out + a.ldo * row + (int64_t)h * D;
    *reinterpret_cast<uint2*>(dst + e0) = make_uint2(narrow2<BF>(x[0], x[1]), narrow2<BF>(x[2], x[3]));
    *reinterpret_cast<uint2*>(dst + e1) = make_uint2(narrow2<BF>(y[0], y[1]), narrow2<BF>(y[2], y[3]));
    return;
  }
  const int slots = 2 * c.kv_heads, item = blockIdx.x / slots, hs = blockIdx.x - item * slots;
  const bool value = hs >= c.kv_heads;
  const int h = value ? hs - c.kv_heads : hs;
  auto first_item = [&](int i) { return clampi(c.q_start[i], 0, c.tokens) / kExpBlock + 2 * i; };
  // one new token per sequence first: 33 items for 16 of them
  int s = min((int)((int64_t)item * 16 / 33), c.seqs - 1);
  if (!(first_item(s) <= item && item < first_item(s + 1))) s = last_at_most(c.seqs, item, first_item);
  const Seq sq = sequence(c, s);
  const int past = sq.len - sq.rows, p0 = max(past, 0);
  const int64_t block = (int64_t)p0 / kExpBlock + item - first_item(s);
  if (sq.rows == 0 || block * kExpBlock >= sq.len) return;
  const int begin = (int)block * kExpBlock, mask = (1 << c.page_shift) - 1;
  const uint32_t page = (uint32_t)c.table[s * c.tstride + (begin >> c.page_shift)];
  if (page >= c.pages) return;
  const int pos = begin + (int)threadIdx.x / U;
  const bool fresh = pos >= p0 && pos < sq.len, older = pos < p0, turn = !value && 8 * unit < a.rot;
  int e0, e1;
  pieces(unit, turn, e0, e1);
  uint8_t* dst = reinterpret_cast<uint8_t*>(value ? c.v : c.k) + page * c.pstride + h * c.hstride + (pos & mask) * c.rstride;
  int8_t* ex = (value ? args.e.v : args.e.k) + page * args.e.pstride + h * args.e.hstride + (begin & mask) / kExpBlock;
  f4v x = (f4v)0.f, y = (f4v)0.f;
  uint32_t was0 = 0, was1 = 0;
  int e_old = -kMostExp;
  if (begin < p0) e_old = exponent(*ex);
  if (older) {
    was0 = *reinterpret_cast<const uint32_t*>(dst + e0);
    was1 = *reinterpret_cast<const uint32_t*>(dst + e1);
  }
  if (fresh) {
    const int64_t at = (value ? a.ldv : a.ldk) * (sq.row0 + pos - past) + (int64_t)h * D;
    const void* src = value ? a.v : a.k;
    x = load4<X>(src, at + e0);
    y = load4<X>(src, at + e1);
    if (turn) turned(x, y, unit, pos);
  }
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    most = fmaxf(most, finite(x[i]) ? fabsf(x[i]) : 0.f);
    most = fmaxf(most, finite(y[i]) ? fabsf(y[i]) : 0.f);
  }
#pragma unroll
  for (int d = 32; d; d /= 2) most = fmaxf(most, __shfl_xor(most, d));
  if ((threadIdx.x & 63) == 0) most_l[threadIdx.x >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) most = fmaxf(most, most_l[i]);
  const int e = max(exponent_of(most), e_old);
  if (threadIdx.x == 0) *ex = (int8_t)e;
  if (fresh) {
    const float down = two_to(-e);
    *reinterpret_cast<uint32_t*>(dst + e0) = to8(x * down);
    *reinterpret_cast<uint32_t*>(dst + e1) = to8(y * down);
  } else if (older && e > e_old) {
    const float down = two_to(e_old - e);  // (-96 at least)
    *reinterpret_cast<uint32_t*>(dst + e0) = to8(from8(was0) * down);
    *reinterpret_cast<uint32_t*>(dst + e1) = to8(from8(was1) * down);
  }
}

template <int D, int X>
hipError_t append8_d(const Append8Args& a, int q_type, hipStream_t s) {
  const uint32_t items = (uint32_t)(a.a.c.tokens / kExpBlock + 2 * a.a.c.seqs), kv_blocks = items * 2 * (uint32_t)a.a.c.kv_heads;
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
