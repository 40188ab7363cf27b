// Score of a row's pages for a query, from the bounds of each page's keys: no key k with lo <= k <= hi (dimension by
// dimension) gives a head more than sum_d max(q_d lo_d, q_d hi_d), and
//   score[t, g, c] = max over the query heads of KV head g of that sum for the page in column c of the query's table row,
// -inf past the row's pages and on invalid ones. As max(q lo, q hi) is q hi for q >= 0 and q lo for q <= 0, the sum is the
// product of the page's [lo, hi] with [min(q, 0), max(q, 0)]: 2 D long, on the matrix cores.
//
// Work: one wave per 16 pages of a (query, KV head), 4 waves a workgroup. v_mfma_f32_16x16x32_bf16 with M = 16 pages, N =
// 16 heads (the group's), K = 2 D: lane (g4, li) feeds page li's 8 elements from 32 s + 8 g4 in step s and head li's of the
// same dimensions, and gets pages 4 g4 + r of head li; the heads' maximum is taken over the 16 lanes of a row.
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
  int32_t H, G, group, P;
  int64_t num_blocks;
};

template <int D>
__global__ __launch_bounds__(256) void block_scores_kernel(BlockScoreArgs a) {
  constexpr int HS = D / 32, STEPS = 2 * HS;  // steps of the lower bounds, then as many of the upper ones
  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, li = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t t = blockIdx.y, g = blockIdx.z;
  const int32_t c0 = (int32_t)blockIdx.x * 64 + 16 * wave;  // this wave's first column
  const int32_t row = a.rows ? a.rows[t] : t;
  const int32_t len = a.seq_lens[t], L = max(len, 0);
  const int32_t count = (int32_t)(((int64_t)L + a.P - 1) / a.P);
  if (blockIdx.x == 0 && g == 0 && tid == 0) a.counts[t] = count;
  if (c0 >= a.table_width) return;
  const bool row_ok = row >= 0 && row < a.table_rows;
  const int32_t col = c0 + li;
  int32_t page = row_ok && col < count && col < a.table_width ? a.table[(int64_t)row * a.table_stride + col] : -1;
  const bool ok = page >= 0 && (int64_t)page < a.num_blocks;
  float* dst = a.scores + ((int64_t)t * a.G + g) * a.table_width + c0;
  if (!__any(ok)) {
    if (lane < 16 && col < a.table_width) dst[li] = -INFINITY;
    return;
  }
  const uint16_t* b = a.bounds + ((int64_t)(ok ? page : 0) * a.G + g) * 2 * D + 8 * g4;
  uint32_t bv[STEPS][4];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const uint4 w = ld16_stream(b + 32 * s);
    bv[s][0] = w.x, bv[s][1] = w.y, bv[s][2] = w.z, bv[s][3] = w.w;
  }
  const uint16_t* qp = a.q + ((int64_t)t * a.H + g * a.group + min(li, a.group - 1)) * D + 8 * g4;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < HS; ++s) {
    const uint4 w = ld16(qp + 32 * s);
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
    uint32_t neg[4], pos[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // as 16-bit integers bf16 values have their sign
      const s16x2_t z = {0, 0}, v = __builtin_bit_cast(s16x2_t, ww[i]);
      neg[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(v, z));
      pos[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(v, z));
    }
    acc = mfma_16x16x32_bf16(bv[s], neg, acc);
    acc = mfma_16x16x32_bf16(bv[HS + s], pos, acc);
  }
  // (a lane past the group repeats its last head)
  float best[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) best[r] = row16_max(acc[r]);
  const float mine = li == 0 ? best[0] : (li == 1 ? best[1] : (li == 2 ? best[2] : best[3]));
  const uint64_t okm = __ballot(ok);  // (bit li of each 16: column c0 + li)
  const int32_t at = 4 * g4 + li;
  if (li < 4 && c0 + at < a.table_width) dst[at] = (okm >> at) & 1 ? mine : -INFINITY;
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
  if (!rows && table_rows < T)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d queries over a table of %d rows", what, T, table_rows);
  if (T > 65535 || num_kv_heads > 65535)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d queries x %d KV heads exceed the grid", what, T, num_kv_heads);
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
  const dim3 grid((uint32_t)(table_width / 64 + (table_width % 64 ? 1 : 0)), T, num_kv_heads);
  if (grid.x >= 1u << 24) return fail(SNA_ERR_INVALID_ARGUMENT, "%s: a table of %d columns exceeds the grid", what, table_width);
  if (head_dim == 128) hipLaunchKernelGGL((block_scores_kernel<128>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((block_scores_kernel<64>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(what);
}
