// Eviction of cached tokens by weight: which tokens of a row each KV head keeps (select), and their K/V rows moved
// together (compact). The pool's pages are head-major, so every KV head keeps a set of its own: the heads of a row share
// the block table and the count, not the tokens.
//
//   select   Row r of L tokens keeps, where L > keep, its first `first` tokens, its last `recent` ones, and of the rest
//            the keep - first - recent of the largest weights (ties: the lowest position; a NaN ranks above every
//            number), in ascending order; else all L. One workgroup per (row, KV head) finds the threshold weight exactly
//            by three histogram passes over the weights' order-preserving 32-bit keys (11, 11 and 10 bits, integer
//            counts), then writes the positions at or above it by prefix counts.
//   compact  Kept token i goes to position i of the row's (or another table's) pages. In place a target lies at or before
//            its source, and at or after every earlier target, so one workgroup may walk a row's tokens in order,
//            reading a whole tile before it writes it, without a copy elsewhere; the columns of a head's rows are
//            independent, so several workgroups share a row by columns, and K and V are apart. To other pages nothing
//            orders the tokens and the tiles go to workgroups of their own.
// Both are bound by memory (latency for few rows): select reads 4 bytes a token and head, compact reads and writes the
// kept rows.
#include <algorithm>

#include "sna_device.h"
#include "sna_host.h"

namespace sna {

struct SelectArgs {
  const float* weights;  // [R, G, width]
  int64_t w_row, w_head;
  int32_t width;
  const int32_t* lens;  // [R]
  int32_t R, G, keep, first, recent;
  int32_t* kept;      // [R, G, keep]
  int32_t* new_lens;  // [R]
  float* out;         // [R, G, out_width] the kept tokens' weights, then zeros; or null (may be `weights` itself)
  int64_t o_row, o_head;
  int32_t out_width;
};

// Order-preserving key of a weight: unsigned order is the floats', -0 equals 0, NaN is above infinity.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const float x = w + 0.0f;
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectBins = 2048;

__global__ __launch_bounds__(kSelectThreads) void select_tokens_kernel(SelectArgs a) {
  __shared__ uint32_t hist[kSelectBins];
  __shared__ uint32_t wtot[16], wtie[16], pick[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t g = blockIdx.x, r = blockIdx.y;
  const int32_t L = min(max(a.lens[r], 0), a.width);
  const float* const w = a.weights + r * a.w_row + g * a.w_head;
  int32_t* const kept = a.kept + ((int64_t)r * a.G + g) * a.keep;
  if (g == 0 && tid == 0) a.new_lens[r] = min(L, a.keep);
  if (L <= a.keep) {  // uniform
    for (int32_t i = tid; i < a.keep; i += kSelectThreads) kept[i] = i < L ? i : -1;
  } else {
    const int32_t lo = a.first, hi = L - a.recent;  // the candidates
    uint32_t need = (uint32_t)(a.keep - a.first - a.recent);
    for (int32_t i = tid; i < a.first; i += kSelectThreads) kept[i] = i;
    for (int32_t i = tid; i < a.recent; i += kSelectThreads) kept[a.keep - a.recent + i] = hi + i;
    uint32_t T = 0;  // the key of the last weight taken: bits found so far
    if (need > 0) {
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < kSelectBins; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        for (int32_t i = lo + tid; i < hi; i += kSelectThreads) {
          const uint32_t key = weight_key(w[i]);
          // (the bits above this pass's are T's)
          if (pass == 0 || (key ^ T) >> (shift + bits) == 0) atomicAdd(&hist[key >> shift & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // the bin that holds the need-th largest: thread i owns bins top - 2 i and the one below it, largest first
        const int top = kSelectBins - 1 - 2 * tid;
        const uint32_t h0 = hist[top], h1 = hist[top - 1];
        int32_t total;
        const uint32_t incl = (uint32_t)wave_incl_scan_i32((int32_t)(h0 + h1), &total);
        if (lane == 0) wtot[wave] = (uint32_t)total;
        __syncthreads();
        uint32_t before = incl - (h0 + h1);
        for (int i = 0; i < wave; ++i) before += wtot[i];
        if (before < need && need <= before + h0) pick[0] = (uint32_t)top, pick[1] = before;
        if (before + h0 < need && need <= before + h0 + h1) pick[0] = (uint32_t)top - 1, pick[1] = before + h0;
        __syncthreads();
        T |= pick[0] << shift;
        need -= pick[1];
      }
      // T is the key of the last weight taken, `need` how many of its ties are; each wave takes a run of the candidates
      const int32_t per = ((hi - lo + 15) / 16 + 63) & ~63;
      const int32_t a0 = min(lo + wave * per, hi), a1 = min(a0 + per, hi);
      uint32_t above = 0, ties = 0;
      for (int32_t i = a0 + lane; i < a1; i += 64) {
        const uint32_t key = weight_key(w[i]);
        above += key > T, ties += key == T;
      }
      int32_t n_above, n_ties;
      wave_incl_scan_i32((int32_t)above, &n_above);
      wave_incl_scan_i32((int32_t)ties, &n_ties);
      if (lane == 0) wtot[wave] = (uint32_t)n_above, wtie[wave] = (uint32_t)n_ties;
      __syncthreads();
      uint32_t run_above = 0, run_ties = 0;
      for (int i = 0; i < wave; ++i) run_above += wtot[i], run_ties += wtie[i];
      const uint64_t below = (1ull << lane) - 1;
      for (int32_t i0 = a0; i0 < a1; i0 += 64) {
        const int32_t i = i0 + lane;
        const uint32_t key = i < a1 ? weight_key(w[i]) : 0;
        const bool gt = i < a1 && key > T, eq = i < a1 && key == T;
        const uint64_t mg = __ballot(gt), me = __ballot(eq);
        const uint32_t ranked = run_ties + (uint32_t)__popcll(me & below);  // ties before this one
        const uint32_t at = run_above + (uint32_t)__popcll(mg & below) + min(ranked, need);
        if (gt || (eq && ranked < need)) kept[a.first + at] = i;
        run_above += (uint32_t)__popcll(mg), run_ties += (uint32_t)__popcll(me);
      }
    }
  }
  if (!a.out) return;
  // The kept tokens' weights, in order: a tile is read before it is written, for `out` may be `weights` itself.
  float* const out = a.out + r * a.o_row + g * a.o_head;
  const int32_t n = min(L, a.keep);
  __syncthreads();
  for (int32_t i0 = 0; i0 < n; i0 += kSelectThreads) {  // uniform
    const int32_t i = i0 + tid;
    const float v = i < n ? w[kept[i]] : 0.0f;
    wait_vmcnt<0>();
    __syncthreads();
    if (i < n) out[i] = v;
  }
  for (int32_t i = n + tid; i < a.out_width; i += kSelectThreads) out[i] = 0.0f;
}

struct CompactArgs {
  uint8_t* k_cache;  // [num_blocks, G, P, row_bytes]
  uint8_t* v_cache;
  int64_t num_blocks;
  int32_t G, P, row_bytes;
  const int32_t* table;  // [R, table_width]
  int64_t table_stride;
  int32_t table_width;
  const int32_t* dst;  // [R, dst_width], or `table`
  int64_t dst_stride;
  int32_t dst_width;
  const int32_t* kept;  // [R, G, keep], -1 where there is none
  int32_t R, keep;
  int32_t slices;  // a row's columns are cut into so many
  int32_t chunks;  // workgroups that share a row's tokens (1 in place)
};

constexpr int kCompactThreads = 256;
constexpr int kCompactUnroll = 4;  // 16-byte pieces a thread holds

__global__ __launch_bounds__(kCompactThreads) void compact_tokens_kernel(CompactArgs a) {
  const int32_t chunk = blockIdx.x;
  const int32_t slice = blockIdx.y % a.slices, g = blockIdx.y / a.slices % a.G, kv = blockIdx.y / a.slices / a.G;
  const int32_t r = blockIdx.z;
  const int32_t pieces = a.row_bytes / a.slices / 16;  // 16-byte pieces of a token (a power of two)
  const int32_t sh = __builtin_ctz((uint32_t)pieces);
  uint8_t* const cache = kv ? a.v_cache : a.k_cache;
  const int32_t* const kept = a.kept + ((int64_t)r * a.G + g) * a.keep;
  const int32_t* const src_row = a.table + r * a.table_stride;
  const int32_t* const dst_row = a.dst + r * a.dst_stride;
  const int32_t col = (threadIdx.x & (pieces - 1)) * 16 + slice * (a.row_bytes / a.slices);
  const int32_t per = kCompactThreads * kCompactUnroll >> sh;  // tokens of a tile
  for (int32_t i0 = chunk * per; i0 < a.keep; i0 += a.chunks * per) {  // uniform
    uint4 v[kCompactUnroll];
    uint8_t* to[kCompactUnroll];
#pragma unroll
    for (int u = 0; u < kCompactUnroll; ++u) {
      const int32_t i = i0 + ((u * kCompactThreads + (int32_t)threadIdx.x) >> sh);
      to[u] = nullptr;
      v[u] = make_uint4(0, 0, 0, 0);
      const int32_t from = i < a.keep ? kept[i] : -1;
      if (from < 0) continue;
      const int32_t sc = from / a.P, dc = i / a.P;
      if (sc >= a.table_width || dc >= a.dst_width) continue;
      const int64_t sp = src_row[sc], dp = dst_row[dc];
      if (sp < 0 || sp >= a.num_blocks || dp < 0 || dp >= a.num_blocks) continue;
      const uint8_t* src = cache + ((sp * a.G + g) * a.P + (from - sc * a.P)) * (int64_t)a.row_bytes + col;
      uint8_t* dst = cache + ((dp * a.G + g) * a.P + (i - dc * a.P)) * (int64_t)a.row_bytes + col;
      if (src == dst) continue;
      to[u] = dst;
      v[u] = ld16(src);
    }
    if (a.chunks == 1) {  // in place: the tile is read before any of it is written
      wait_vmcnt<0>();
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kCompactUnroll; ++u)
      if (to[u]) *reinterpret_cast<uint4*>(to[u]) = v[u];
  }
}

}  // namespace sna

using namespace sna;

extern "C" int sna_select_tokens(const float* weights, int64_t row_stride, int64_t head_stride, int32_t width,
                                 const int32_t* seq_lens, int32_t R, int32_t num_kv_heads, int32_t keep, int32_t first,
                                 int32_t recent, int32_t* kept, int32_t* new_lens, float* weights_out,
                                 int64_t out_row_stride, int64_t out_head_stride, int32_t out_width, void* stream) {
  ApiGuard guard;
  if (R < 0 || num_kv_heads < 1 || width < 1 || keep < 1 || first < 0 || recent < 0 || (int64_t)first + recent > keep ||
      row_stride < width || head_stride < width)
    return fail(SNA_ERR_INVALID_ARGUMENT,
                "select_tokens: bad sizes (R %d, KV heads %d, width %d, strides %lld / %lld, keep %d of which first %d "
                "and recent %d)", R, num_kv_heads, width, (long long)row_stride, (long long)head_stride, keep, first,
                recent);
  if (weights_out && (out_width < keep || out_row_stride < out_width || out_head_stride < out_width))
    return fail(SNA_ERR_INVALID_ARGUMENT, "select_tokens: weights_out of %d columns (strides %lld / %lld) for %d tokens",
                out_width, (long long)out_row_stride, (long long)out_head_stride, keep);
  if (R == 0) return SNA_OK;
  if (!weights || !seq_lens || !kept || !new_lens)
    return fail(SNA_ERR_INVALID_ARGUMENT, "select_tokens: null pointer");
  if (R > 65535) return fail(SNA_ERR_INVALID_ARGUMENT, "select_tokens: %d rows exceed the grid", R);
  SelectArgs a;
  a.weights = weights;
  a.w_row = row_stride;
  a.w_head = head_stride;
  a.width = width;
  a.lens = seq_lens;
  a.R = R;
  a.G = num_kv_heads;
  a.keep = keep;
  a.first = first;
  a.recent = recent;
  a.kept = kept;
  a.new_lens = new_lens;
  a.out = weights_out;
  a.o_row = out_row_stride;
  a.o_head = out_head_stride;
  a.out_width = out_width;
  hipLaunchKernelGGL(select_tokens_kernel, dim3(num_kv_heads, R), dim3(kSelectThreads), 0, (hipStream_t)stream, a);
  return check_launch("select_tokens");
}

extern "C" int sna_compact_tokens(void* k_cache, void* v_cache, int64_t num_blocks, int32_t num_kv_heads,
                                  int32_t page_size, int32_t head_dim, int32_t cache_dtype, const int32_t* block_table,
                                  int64_t table_stride, int32_t table_width, const int32_t* dst_table,
                                  int64_t dst_stride, int32_t dst_width, const int32_t* kept, int32_t R, int32_t keep,
                                  void* stream) {
  ApiGuard guard;
  if (R < 0 || num_kv_heads < 1 || num_blocks < 1 || page_size < 1 || keep < 1 || table_width < 1 ||
      table_stride < table_width || (dst_table && (dst_width < 1 || dst_stride < dst_width)))
    return fail(SNA_ERR_INVALID_ARGUMENT,
                "compact_tokens: bad sizes (R %d, KV heads %d, blocks %lld, page %d, keep %d, tables %d and %d wide, "
                "strides %lld and %lld)", R, num_kv_heads, (long long)num_blocks, page_size, keep, table_width,
                dst_width, (long long)table_stride, (long long)dst_stride);
  if (dst_table == block_table) dst_table = nullptr;  // in place
  if (head_dim != 64 && head_dim != 128)
    return fail(SNA_ERR_UNSUPPORTED, "compact_tokens: head_dim %d (64 or 128)", head_dim);
  if (cache_dtype != SNA_DTYPE_BF16 && cache_dtype != SNA_DTYPE_FP8_E4M3FN && cache_dtype != SNA_DTYPE_FP8_E4M3FN_MUL)
    return fail(SNA_ERR_UNSUPPORTED, "compact_tokens: KV dtype %d (FP8 e4m3fn or bf16)", cache_dtype);
  if (R == 0) return SNA_OK;
  if (!k_cache || !v_cache || !block_table || !kept)
    return fail(SNA_ERR_INVALID_ARGUMENT, "compact_tokens: null pointer");
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(SNA_ERR_INVALID_ARGUMENT, "compact_tokens: the caches must be 16-byte aligned");
  CompactArgs a;
  a.k_cache = (uint8_t*)k_cache;
  a.v_cache = (uint8_t*)v_cache;
  a.num_blocks = num_blocks;
  a.G = num_kv_heads;
  a.P = page_size;
  a.row_bytes = head_dim * (cache_dtype == SNA_DTYPE_BF16 ? 2 : 1);
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.dst = dst_table ? dst_table : block_table;
  a.dst_stride = dst_table ? dst_stride : table_stride;
  a.dst_width = dst_table ? dst_width : table_width;
  a.kept = kept;
  a.R = R;
  a.keep = keep;
  a.slices = dst_table ? 1 : a.row_bytes / 64;
  const int32_t per = kCompactThreads * kCompactUnroll / (a.row_bytes / a.slices / 16);
  a.chunks = dst_table ? (int32_t)std::min<int64_t>(((int64_t)keep + per - 1) / per, 65535) : 1;
  const int64_t y = (int64_t)a.slices * num_kv_heads * 2;
  if (R > 65535 || y > 65535)
    return fail(SNA_ERR_INVALID_ARGUMENT, "compact_tokens: %d rows x %d KV heads exceed the grid", R, num_kv_heads);
  hipLaunchKernelGGL(compact_tokens_kernel, dim3(a.chunks, (unsigned)y, R), dim3(kCompactThreads), 0, (hipStream_t)stream,
                     a);
  return check_launch("compact_tokens");
}
