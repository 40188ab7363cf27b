// Score of a row's pages for a query, from the bounds of each page's keys: no key k with lo <= k <= hi (dimension by
// dimension, as given) gives a head more than sum_d max(q_d lo_d, q_d hi_d), and
//   score[t, g, c] = max over the query heads of KV head g of that sum for the page in column c of the query's table row,
// -inf past the row's pages and on invalid ones; a product with a query element of 0 is 0, and a head whose sum is NaN counts
// only where all of them are. As max(q lo, q hi) is q hi for q >= 0 and q lo for q <= 0, the sum is the
// product of the page's [lo, hi] with [min(q, 0), max(q, 0)]: 2 D long, on the matrix cores.
//
// Work: one wave per 16 pages of a (query, KV head), 4 waves a workgroup. v_mfma_f32_16x16x32_bf16 with M = 16 pages, N =
// 16 heads (the group's), K = 2 D: lane (g4, li) feeds page li's 8 elements from 32 s + 8 g4 in step s and head li's of the
// same dimensions, and gets pages 4 g4 + r of head li; the heads' maximum is taken over the 16 lanes of a row.
//
// What bounds it: reads of 512 bytes (head dim 128) at random places, the query's length and the table before them. 64 rows of
// 16384 keys in pages of 64, 8 KV heads: 12.9-14.1 us, 68 MB, 4.8-5.3 TB/s; one row of 131071 in pages of 32, 17 MB, 6.2. Two or
// four groups of 16 pages a wave, all asked for at once: the same, and slower for one row (P = 128: 3.9, 5.7 and 8.1).
#include "sna_device.h"
#include "sna_host.h"

namespace sna {

struct BlockScoreArgs {
  const uint16_t* q;       // [T, H, D] bf16
  const uint16_t* bounds;  // [num_blocks, G, 2, D] bf16
  const int32_t* table;
  int64_t table_stride;
  int32_t table_width, table_rows;
  const int32_t* rows;      // [T] or null
  const int32_t* seq_lens;  // [T]
  float* scores;            // [T, G, table_width]
  int32_t* counts;          // [T]
  int32_t T, H, G, group, P;
  int32_t runs;  // workgroups of a (query, KV head)
  int64_t num_blocks;
};

// The sums of a lane's pages (4 g4 + r, whose bounds are at the lanes' `at`) and head (elements qp) by their definition, one
// element after the other: where bounds are infinite (infinite keys; lo = inf, hi = -inf: a dimension whose keys are all NaN),
// as their products with the zeros of [min(q, 0), max(q, 0)] are NaN.
// Its loads wait for each other: 64 rows of 16384 keys, 15 us, take 65 with such a bound in every 16th page, 75 in every page; as
// products of cleaned bounds and of counts of the infinite ones it took 95 registers, where 58 keep 8 waves a SIMD for all calls.
template <int D>
__device__ __forceinline__ f32x4_t block_scores_defined(const uint16_t* bounds, int64_t at, const uint16_t* qp) {
  const int lane = threadIdx.x & 63, g4 = lane >> 4;
  f32x4_t sums = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int r = 0; r < 4; ++r) {
    const int src = 16 * g4 + 4 * g4 + r;
    const uint16_t* b = bounds + __shfl((long long)at, src);
    float sum = 0.0f;
#pragma unroll 1
    for (int d = 0; d < D; d += 8) {
      const uint4 wl = ld16(b + d), wh = ld16(b + D + d), wq = ld16(qp + d);
      const uint32_t l[4] = {wl.x, wl.y, wl.z, wl.w}, h[4] = {wh.x, wh.y, wh.z, wh.w}, q[4] = {wq.x, wq.y, wq.z, wq.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int up = e & 1 ? 0 : 16;  // an element's bits to the upper half
        const float f = __uint_as_float(q[e >> 1] << up & 0xffff0000u);
        const float lo = __uint_as_float(l[e >> 1] << up & 0xffff0000u), hi = __uint_as_float(h[e >> 1] << up & 0xffff0000u);
        sum += f == 0.0f ? 0.0f : fmaxf(f * lo, f * hi);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[k] = r == k ? sum : sums[k];
  }
  return sums;
}

template <int D>
__global__ __launch_bounds__(256) void block_scores_kernel(BlockScoreArgs a) {
  constexpr int HS = D / 32, STEPS = 2 * HS;  // steps of the lower bounds, then as many of the upper ones
  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, li = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // eight (query, run of columns) items' first heads, then their second ones, ..: an item's heads run on one XCD at about one
  // time. Their bounds lie side by side, so that the reads in flight fall on every memory channel
  const uint32_t run = 8u * (uint32_t)a.G, in = blockIdx.x % run, item = blockIdx.x / run * 8 + in % 8;
  const int32_t g = (int32_t)(in / 8), t = (int32_t)(item / (uint32_t)a.runs);
  if (t >= a.T) return;
  const int32_t cx = (int32_t)(item - (uint32_t)t * (uint32_t)a.runs);
  const int32_t c0 = cx * 64 + 16 * wave, col = c0 + li;  // this wave's first column, this lane's
  const int32_t row = a.rows ? a.rows[t] : t;
  const int32_t len = a.seq_lens[t];
  const uint16_t* qp = a.q + ((int64_t)t * a.H + g * a.group + min(li, a.group - 1)) * D + 8 * g4;
  uint4 qw[HS];
#pragma unroll
  for (int s = 0; s < HS; ++s) qw[s] = ld16(qp + 32 * s);
  if (c0 >= a.table_width) return;
  const bool row_ok = row >= 0 && row < a.table_rows;
  const int32_t* trow = a.table + (int64_t)(row_ok ? row : 0) * a.table_stride;
  const int32_t page = trow[min(col, a.table_width - 1)];
  const int32_t count = (int32_t)(((int64_t)max(len, 0) + a.P - 1) / a.P);
  if (cx == 0 && g == 0 && tid == 0) a.counts[t] = count;
  const bool ok = row_ok && col < count && col < a.table_width && page >= 0 && (int64_t)page < a.num_blocks;
  const uint16_t* b = a.bounds + ((int64_t)(ok ? page : 0) * a.G + g) * 2 * D + 8 * g4;
  uint32_t bv[STEPS][4];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const uint4 w = ld16(b + 32 * s);  // (two loads a 128-byte line: non-temporal ones 17.2 us where these take 13.9)
    bv[s][0] = w.x, bv[s][1] = w.y, bv[s][2] = w.z, bv[s][3] = w.w;
  }
  uint32_t neg[HS][4], pos[HS][4];
#pragma unroll
  for (int s = 0; s < HS; ++s) {
    const uint32_t ww[4] = {qw[s].x, qw[s].y, qw[s].z, qw[s].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // as 16-bit integers bf16 values have their sign
      const s16x2_t z = {0, 0}, v = __builtin_bit_cast(s16x2_t, ww[i]);
      neg[s][i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(v, z));
      pos[s][i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(v, z));
    }
  }
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < HS; ++s) {
    acc = mfma_16x16x32_bf16(bv[s], neg[s], acc);
    acc = mfma_16x16x32_bf16(bv[HS + s], pos[s], acc);
  }
  const uint64_t okm = __ballot(ok);  // (bit li of each 16: column c0 + li)
  bool infinite = false;
#pragma unroll
  for (int r = 0; r < 4; ++r) infinite |= !(fabsf(acc[r]) < INFINITY) && (okm >> (4 * g4 + r) & 1);
  if (__any(infinite)) acc = block_scores_defined<D>(a.bounds, b - a.bounds - 8 * g4, qp - 8 * g4);
  // (a lane past the group repeats its last head)
  float best[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) best[r] = row16_max(acc[r]);
  const float mine = li == 0 ? best[0] : (li == 1 ? best[1] : (li == 2 ? best[2] : best[3]));
  const int32_t at = 4 * g4 + li;
  if (li < 4 && c0 + at < a.table_width)
    a.scores[((int64_t)t * a.G + g) * a.table_width + c0 + at] = (okm >> at) & 1 ? mine : -INFINITY;
}

template <int D>
static void launch_block_scores(const BlockScoreArgs& a, hipStream_t s) {
  const uint32_t items = (uint32_t)(a.T * a.runs);
  hipLaunchKernelGGL((block_scores_kernel<D>), dim3((items + 7) / 8 * 8 * a.G), dim3(256), 0, s, a);
}

}  // namespace sna

using namespace sna;

extern "C" int sna_block_scores(const void* q, const void* k_bounds, const int32_t* block_table, int64_t table_stride,
                                int32_t table_width, int32_t table_rows, const int32_t* rows, const int32_t* seq_lens,
                                float* scores, int32_t* counts, int32_t T, int32_t num_q_heads, int32_t num_kv_heads,
                                int32_t head_dim, int32_t page_size, int64_t num_blocks, void* stream) {
  ApiGuard guard;
  const char* what = "block_scores";
  if (T < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads || num_blocks < 1 || table_width < 1 ||
      table_rows < 0 || table_stride < table_width || page_size < 1)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: bad sizes (T %d, heads %d / %d, blocks %lld, table %d x %d, stride %lld, "
                "page %d)", what, T, num_q_heads, num_kv_heads, (long long)num_blocks, table_rows, table_width,
                (long long)table_stride, page_size);
  const int32_t group = num_q_heads / num_kv_heads;
  if (group > 16) return fail(SNA_ERR_UNSUPPORTED, "%s: GQA group %d > 16", what, group);
  if (head_dim != 64 && head_dim != 128)
    return fail(SNA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  if (T == 0) return SNA_OK;
  if (!q || !k_bounds || !block_table || !seq_lens || !scores || !counts)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(q, 16) || !aligned(k_bounds, 16))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: q and k_bounds must be 16-byte aligned", what);
  if (table_rows < 1) return fail(SNA_ERR_INVALID_ARGUMENT, "%s: a table of no rows", what);
  if (!rows && table_rows < T)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d queries over a table of %d rows", what, T, table_rows);
  BlockScoreArgs a;
  a.q = (const uint16_t*)q;
  a.bounds = (const uint16_t*)k_bounds;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.table_rows = table_rows;
  a.rows = rows;
  a.seq_lens = seq_lens;
  a.scores = scores;
  a.counts = counts;
  a.H = num_q_heads;
  a.G = num_kv_heads;
  a.group = group;
  a.P = page_size;
  a.num_blocks = num_blocks;
  a.T = T;
  a.runs = (int32_t)(((int64_t)table_width + 63) / 64);
  if (((int64_t)T * a.runs + 8) * num_kv_heads >= 1 << 24)  // (a grid has under 2^32 threads)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d queries over %d columns, %d KV heads exceed the grid", what, T, table_width,
                num_kv_heads);
  if (head_dim == 128) launch_block_scores<128>(a, (hipStream_t)stream);
  else launch_block_scores<64>(a, (hipStream_t)stream);
  return check_launch(what);
}
