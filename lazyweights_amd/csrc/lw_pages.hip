// A step of sequences over their pages: lengths, page tables, the pool of free pages, and the rows' positions and slots, made on
// the GPU from the tokens that each sequence keeps and gets (lw_pages_advance).
#include <algorithm>

#include "lw_attn_device.h"

namespace lw {

namespace {

constexpr int kMost = 1 << 30;  // sums are counted up to here, so that they fit 32 bits whatever the arrays hold
constexpr int kPageThreads = 512, kGroups = 16;

__device__ __forceinline__ int add_up(int x, int y) { return min(x + y, kMost); }

// the last i in [0, n) with first[i] <= x, first non-decreasing and first[0] <= x
__device__ __forceinline__ int find(const int* first, int n, int x) {
  int lo = 0;
  while (n > 1) {
    const int half = n >> 1;
    if (first[lo + half] <= x) lo += half, n -= half;
    else n = half;
  }
  return lo;
}

// Every block adds up all sequences' new rows, pages taken and pages given (sums before each in LDS), so that one launch needs
// no exchange between blocks; then the blocks share the rows and the pages that change hands, each found by
// bisection. What the step reads (table entries up to the old lengths, the pool up to its count) it does not write (entries
// and places behind these): only lengths and count may be given in place, and then the block that has read them last writes those. It
// is found by counters in two levels, since additions to one take 65 ns each, one after the other (500 sequences with 216000 rows in
// 422 blocks; kGroups counters on lines of their own).
//
// Bound by latency: the arrays, the sums, a bisection, a page: a few thousand cycles in turn, over as many threads as there are rows
// (a row per thread: 500 sequences, 216000 rows 7.5 us, four rows 13; 64 sequences 4.5).
template <int SEQS>
__global__ __launch_bounds__(kPageThreads) void k_pages(const PagesArgs a) {
  constexpr int T = kPageThreads, PER = (SEQS + T - 1) / T, WAVES = T / 64;
  __shared__ int rows_l[SEQS], take_l[SEQS], give_l[SEQS], keep_l[SEQS];
  __shared__ int part[WAVES][3], lacks, last;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, shift = a.page_shift, room = a.table_pages << shift;
  const int left = clampi(a.left[0], 0, a.pages);
  auto pages_of = [&](int n) { return (int)(((int64_t)n + (1 << shift) - 1) >> shift); };
  struct Step {
    int len, keep, add;
  };
  auto step_of = [&](int s) {
    Step p;
    p.len = clampi(a.kv_len[s], 0, room);
    p.keep = a.keep ? clampi(a.keep[s], 0, p.len) : p.len;
    p.add = clampi(a.add[s], 0, kMost);
    return p;
  };
  if (t == 0) lacks = 0;
  __syncthreads();
  int rows = 0, take = 0, give = 0;
  bool table_lacks = false;
  for (int i = 0; i < PER; ++i) {
    const int s = t * PER + i;
    if (s >= a.seqs) break;
    const Step p = step_of(s);
    const int had = pages_of(p.len), need = pages_of(min(p.keep + p.add, kMost));
    table_lacks |= p.keep + p.add > room;
    rows_l[s] = rows;  // (of this thread's sequences so far)
    take_l[s] = take;
    give_l[s] = give;
    keep_l[s] = p.keep;
    rows = add_up(rows, p.add);
    take = add_up(take, max(need - had, 0));
    give = add_up(give, max(had - need, 0));
  }
  int up[3] = {rows, take, give};
#pragma unroll
  for (int d = 1; d < 64; d *= 2)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int o = __shfl_up(up[i], d);
      if (lane >= d) up[i] = add_up(up[i], o);
    }
  if (lane == 63)
    for (int i = 0; i < 3; ++i) part[w][i] = up[i];
  if (table_lacks) lacks = 2;
  __syncthreads();
  int total[3] = {0, 0, 0}, before[3] = {0, 0, 0};
  for (int j = 0; j < WAVES; ++j)
    for (int i = 0; i < 3; ++i) {
      if (j == w) before[i] = total[i];
      total[i] = add_up(total[i], part[j][i]);
    }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const int o = __shfl_up(up[i], 1);
    if (lane > 0) before[i] = add_up(before[i], o);
  }
  for (int i = 0; i < PER; ++i) {
    const int s = t * PER + i;
    if (s >= a.seqs) break;
    rows_l[s] = add_up(rows_l[s], before[0]);
    take_l[s] = add_up(take_l[s], before[1]);
    give_l[s] = add_up(give_l[s], before[2]);
  }
  const int all = total[0], taken = total[1], given = total[2];
  const int lack = lacks | (taken - given > left ? 1 : 0) | (all > a.rows ? 4 : 0);
  __syncthreads();
  // this block is done with what may be overwritten
  if (t == 0) {
    auto arrive = [&](int counter, uint32_t of) {  // whether this is the last of so many; the counter is 0 again then
      int32_t* count = a.count + 16 * counter;
      const bool end = (uint32_t)__hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
      if (end) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return end;
    };
    const uint32_t group = blockIdx.x % kGroups;
    if (gridDim.x == 1 || !a.in_place) last = blockIdx.x == 0;
    else last = arrive(1 + group, (gridDim.x - group + kGroups - 1) / kGroups) && arrive(0, min(gridDim.x, (uint32_t)kGroups));
  }
  __syncthreads();
  if (last) {
    for (int s = t; s < a.seqs; s += T) {
      const Step p = step_of(s);
      a.kv_len_out[s] = lack ? p.len : p.keep + p.add;
    }
    if (t == 0) {
      a.left_out[0] = lack ? left : min(left - taken + given, a.pages);
      a.left_out[1] = lack;
    }
  }
  const int me = blockIdx.x * T + t, threads = gridDim.x * T;
  for (int s = me; s <= a.seqs; s += threads) a.q_start[s] = lack ? 0 : s < a.seqs ? rows_l[s] : all;
  if (lack) return;
  const int n = a.seqs;
  // the i-th page taken, or given
  auto given_page = [&](int i) {
    const int s = find(give_l, n, i);
    const int need = pages_of(keep_l[s] + ((s + 1 < n ? rows_l[s + 1] : all) - rows_l[s]));
    return a.table[s * a.tstride + need + i - give_l[s]];
  };
  auto page = [&](int i) { return i < given ? given_page(i) : a.free[left - 1 - (i - given)]; };
  // pages of s before the step (those it needs now are as many, with what it takes and without what it gives)
  auto had_of = [&](int s) {
    const int need = pages_of(keep_l[s] + ((s + 1 < n ? rows_l[s + 1] : all) - rows_l[s]));
    return need - ((s + 1 < n ? take_l[s + 1] : taken) - take_l[s]) + ((s + 1 < n ? give_l[s + 1] : given) - give_l[s]);
  };
  for (int i = me; i < taken; i += threads) {
    const int s = find(take_l, n, i);
    a.table[s * a.tstride + had_of(s) + i - take_l[s]] = page(i);
  }
  for (int i = taken + me; i < given; i += threads)
    if (left + i - taken < a.pages) a.free[left + i - taken] = given_page(i);
  if (a.position || a.slot)
    for (int i = me; i < all; i += threads) {
      const int s = find(rows_l, n, i), at = keep_l[s] + i - rows_l[s], j = at >> shift, had = had_of(s);
      const int p = j < had ? a.table[s * a.tstride + j] : page(take_l[s] + j - had);
      if (a.position) a.position[i] = at;
      if (a.slot) a.slot[i] = (uint32_t)p < (uint32_t)a.pages ? ((int64_t)p << shift) + (at & ((1 << shift) - 1)) : -1;
    }
}

}  // namespace

hipError_t launch_pages(const PagesArgs& a, hipStream_t s) {
  // (as many as are on the card at once: of 8192 sequences, with 128 KB of LDS, one per CU)
  const int blocks = std::max(1, std::min(a.seqs <= kPageThreads ? 1024 : 256, (a.rows + kPageThreads - 1) / kPageThreads));
  if (a.seqs <= kPageThreads) k_pages<kPageThreads><<<blocks, kPageThreads, 0, s>>>(a);
  else k_pages<kMostPageSeqs><<<blocks, kPageThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace lw
