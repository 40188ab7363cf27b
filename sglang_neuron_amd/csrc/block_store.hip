// Writer of a cache whose blocks of tokens carry a scale each: a call's tokens join their requests' pages [blocks, G, P, D]
// (e4m3fn or int8 codes with a scale for every `bt` tokens of a page and KV head; bf16 without scales), and, where asked
// for, the pages' key bounds (the least and the largest value of each dimension over a page's keys).
//
// For a block (bt tokens, one KV head, K or V apart) that the call writes from its token `lo` on:
//   fresh = max(max |x| / top, 2^-100) over the call's tokens of the block (infinities not counted; a NaN makes it NaN)
//   scale = fresh where lo = 0 (the block starts anew), else max(fresh, the scale it had)
//   code  = round(clamp(x / scale)) of the new tokens; where the scale grew, the tokens before lo are rounded again,
//           round(code * had / scale), so that one scale holds for the block.
// top is 448 (e4m3fn) or 127 (int8), quotients are correctly rounded, codes rounded to nearest even.
//
// Work: one workgroup per (page that a request writes, KV head). A wave takes a block of K or of V at a time, all of it: its
// rows in 16-byte pieces, D / 8 lanes a row, held in registers between the maximum and the rounding where they fit.
#include "sna_device.h"
#include "sna_host.h"

namespace sna {

struct BlockStoreArgs {
  const uint16_t* x[2];  // the new tokens' K and V, [T, G, D] bf16, rows x_row elements apart
  int64_t x_row[2];
  uint8_t* cache[2];     // K, V [num_blocks, G, P, D]
  float* scale[2];       // [num_blocks, G, P / bt]
  uint16_t* bounds;      // [num_blocks, G, 2, D] bf16, or null
  const int32_t* table;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* q_start;  // [R + 1], or null: token r is request r's
  const int32_t* prior;    // [R]
  int32_t T, G, P, bt, max_q, pages;  // pages: the most that a request's tokens can touch
  int64_t num_blocks;
};

// The correctly rounded quotient x / s from rs, the rounded 1 / s, held to the range that the clamp to the top leaves
// open (see quantize_pair_e4m3fn_hw).
__device__ __forceinline__ float block_quotient(float x, float s, float rs) {
  const float q = __builtin_amdgcn_fmed3f(x * rs, -1024.0f, 1024.0f);
  return fmaf(fmaf(-q, s, x), rs, q);
}

// Four elements to four codes of a format, the first in the low byte.
template <int FMT>
__device__ __forceinline__ uint32_t block_codes(const float (&x)[4], float s, float rs) {
  if constexpr (FMT == kBlockFp8) {
    return quantize_pair_e4m3fn_hw_nonan(x[0], x[1], s, rs) | quantize_pair_e4m3fn_hw_nonan(x[2], x[3], s, rs) << 16;
  } else {
    // adding 1.5 * 2^23 rounds to a whole number, to nearest even, whose low byte is the code
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b[i] = __float_as_uint(__builtin_amdgcn_fmed3f(block_quotient(x[i], s, rs), -kInt8Max, kInt8Max) + 12582912.0f);
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    return lo | hi;
  }
}
template <int FMT>
__device__ __forceinline__ void block_values(uint32_t w, float (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = FMT == kBlockFp8 ? e4m3fn_to_f32((w >> (8 * i)) & 0xffu) : (float)(int8_t)(w >> (8 * i));
}

template <int D, int FMT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void kv_store_blocks_kernel(BlockStoreArgs a) {
  constexpr int LR = D / 8;     // lanes a row, 8 elements each
  constexpr int RP = 64 / LR;   // rows a wave holds in a piece
  constexpr int HELD = 8;       // pieces held in registers
  constexpr int ESZ = FMT == kBlockBf16 ? 2 : 1;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col8 = lane % LR, row0 = lane / LR;
  const int32_t r = blockIdx.x / a.pages, j = blockIdx.x - r * a.pages, g = blockIdx.y;

  // the request's tokens: rows [t0, t0 + n) of the call at positions prior ..
  int32_t t0 = r, n = 1;
  if (a.q_start) {
    t0 = a.q_start[r];
    const int32_t t1 = min(a.q_start[r + 1], a.T);
    if (t0 < 0 || t1 <= t0) return;
    n = min(t1 - t0, a.max_q);
  }
  const int32_t prior = a.prior[r];
  if (prior < 0) return;
  // this workgroup's page and the positions [lo, hi) in it that the call writes
  const int64_t col = prior / a.P + (int64_t)j;
  const int64_t first = col * a.P;
  const int32_t lo = (int32_t)max((int64_t)prior - first, (int64_t)0);
  const int32_t hi = (int32_t)min((int64_t)prior + n - first, (int64_t)a.P);
  if (hi <= lo || col >= a.table_width) return;
  const int32_t page = a.table[(int64_t)r * a.table_stride + col];
  if (page < 0 || (int64_t)page >= a.num_blocks) return;
  const int64_t ph = (int64_t)page * a.G + g;
  // token `at` of the page is row src + at of the call
  const int64_t src = (int64_t)t0 + (first - prior);

  float mn[8], mx[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) mn[e] = INFINITY, mx[e] = -INFINITY;
  const int32_t nblk = a.P / a.bt, b0 = lo / a.bt, b1 = (hi - 1) / a.bt + 1;
  for (int32_t task = wave; task < 2 * (b1 - b0); task += WAVES) {  // uniform in the wave
    const int which = task & 1;  // K or V
    const int32_t blk = b0 + (task >> 1), head = blk * a.bt;
    const int32_t from = max(lo, head), to = min(hi, head + a.bt);
    const int64_t x_row = a.x_row[which];
    const uint16_t* x = a.x[which] + src * x_row + g * D + 8 * col8;
    uint8_t* cache = a.cache[which] + (ph * a.P * D + 8 * col8) * ESZ;
    float* sp = FMT == kBlockBf16 ? nullptr : a.scale[which] + ph * nblk + blk;
    const float had = FMT != kBlockBf16 && from > head ? *sp : 0.0f;
    const int32_t pieces = (to - from + RP - 1) / RP;
    uint4 w[HELD];
    auto load = [&](int32_t p0) {
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        const int32_t at = from + (p0 + i) * RP + row0;
        if (p0 + i < pieces) w[i] = at < to ? ld16(x + at * x_row) : make_uint4(0, 0, 0, 0);
      }
    };
    // the largest magnitude, and the keys' bounds
    float most = 0.0f;
    bool nan = false;
    for (int32_t p0 = 0; p0 < pieces; p0 += HELD) {
      load(p0);
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        if (p0 + i >= pieces) break;
        const bool live = from + (p0 + i) * RP + row0 < to;
        const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = __uint_as_float(e & 1 ? ww[e >> 1] & 0xffff0000u : ww[e >> 1] << 16);
          if (FMT != kBlockBf16) {
            const float m = fabsf(f);
            nan |= m != m;
            most = fmaxf(most, m < INFINITY ? m : 0.0f);
          }
          if (a.bounds && which == 0 && live) mn[e] = fminf(mn[e], f), mx[e] = fmaxf(mx[e], f);
        }
      }
    }
    float s = 1.0f, rs = 1.0f;
    if (FMT != kBlockBf16) {
      constexpr float top = FMT == kBlockFp8 ? kFp8Max : kInt8Max;
      most = wave_max(most);
      s = __any(nan) ? __uint_as_float(0x7fc00000u) : fmaxf(most / top, kLeastBlockScale);
      if (from > head) s = s != s || had != had ? __uint_as_float(0x7fc00000u) : fmaxf(s, had);
      rs = 1.0f / s;
      // the block's earlier tokens, where the scale grew
      if (from > head && s > had) {
        for (int32_t at = head + row0; at < from; at += RP) {
          uint2 c = ld8(cache + (int64_t)at * D);
          float y[4];
          block_values<FMT>(c.x, y);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] *= had;
          c.x = block_codes<FMT>(y, s, rs);
          block_values<FMT>(c.y, y);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] *= had;
          c.y = block_codes<FMT>(y, s, rs);
          *reinterpret_cast<uint2*>(cache + (int64_t)at * D) = c;
        }
      }
      if (lane == 0) *sp = s;
    }
    for (int32_t p0 = 0; p0 < pieces; p0 += HELD) {
      if (pieces > HELD) load(p0);
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        const int32_t at = from + (p0 + i) * RP + row0;
        if (p0 + i >= pieces || at >= to) continue;
        if constexpr (FMT == kBlockBf16) {
          *reinterpret_cast<uint4*>(cache + (int64_t)at * D * 2) = w[i];
        } else {
          const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          uint32_t c[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float y[4] = {__uint_as_float(ww[2 * h] << 16), __uint_as_float(ww[2 * h] & 0xffff0000u),
                                __uint_as_float(ww[2 * h + 1] << 16), __uint_as_float(ww[2 * h + 1] & 0xffff0000u)};
            c[h] = block_codes<FMT>(y, s, rs);
          }
          *reinterpret_cast<uint2*>(cache + (int64_t)at * D) = make_uint2(c[0], c[1]);
        }
      }
    }
  }

  // ---- the page's key bounds: over the wave's rows, over the waves, and with what the page had ----
  if (!a.bounds) return;
  __shared__ float sm[WAVES][2][D];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int off = LR; off < 64; off <<= 1) {
      mn[e] = fminf(mn[e], __shfl_xor(mn[e], off));
      mx[e] = fmaxf(mx[e], __shfl_xor(mx[e], off));
    }
    if (row0 == 0) sm[wave][0][8 * col8 + e] = mn[e], sm[wave][1][8 * col8 + e] = mx[e];
  }
  __syncthreads();
  for (int32_t i = tid; i < 2 * D; i += 64 * WAVES) {
    const bool upper = i >= D;
    uint16_t* b = a.bounds + ph * 2 * D + i;
    float f = lo > 0 ? bf16_bits_to_f32(*b) : (upper ? -INFINITY : INFINITY);
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
      const float o = sm[v][upper][upper ? i - D : i];
      f = upper ? fmaxf(f, o) : fminf(f, o);
    }
    *b = (uint16_t)(__float_as_uint(f) >> 16);  // a bf16 value already
  }
}

template <int D, int FMT>
static void launch_block_store(const BlockStoreArgs& a, int32_t R, hipStream_t s) {
  const dim3 grid((uint32_t)(R * a.pages), a.G);
  // one block of K and one of V at the most: two waves
  if (a.bt == a.P || a.max_q == 1) hipLaunchKernelGGL((kv_store_blocks_kernel<D, FMT, 2>), grid, dim3(128), 0, s, a);
  else hipLaunchKernelGGL((kv_store_blocks_kernel<D, FMT, 4>), grid, dim3(256), 0, s, a);
}

template <int D>
static void launch_block_store_format(const BlockStoreArgs& a, int32_t R, int32_t dtype, hipStream_t s) {
  if (dtype == SNA_DTYPE_BF16) launch_block_store<D, kBlockBf16>(a, R, s);
  else if (dtype == SNA_DTYPE_INT8) launch_block_store<D, kBlockInt8>(a, R, s);
  else launch_block_store<D, kBlockFp8>(a, R, s);
}

}  // namespace sna

using namespace sna;

extern "C" int sna_kv_store_blocks(const void* k, const void* v, int64_t k_row_stride,
                                   int64_t v_row_stride, int32_t n_tokens, const int32_t* block_table,
                                   int64_t table_stride, int32_t table_width, const int32_t* q_start,
                                   const int32_t* prior_lens, int32_t R, int32_t max_q_len, void* k_cache, void* v_cache,
                                   float* k_scale, float* v_scale, int32_t scale_tokens, void* k_bounds,
                                   int64_t num_blocks, int32_t num_kv_heads, int32_t page_size, int32_t head_dim,
                                   int32_t cache_dtype, void* stream) {
  ApiGuard guard;
  const char* what = "kv_store_blocks";
  if (n_tokens < 0 || R < 0 || max_q_len < 0 || num_kv_heads < 1 || num_blocks < 1 || table_width < 1 ||
      table_stride < table_width)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: bad sizes (tokens %d, R %d, max_q_len %d, heads %d, blocks %lld, table %d "
                "wide, stride %lld)", what, n_tokens, R, max_q_len, num_kv_heads, (long long)num_blocks, table_width,
                (long long)table_stride);
  if (cache_dtype != SNA_DTYPE_BF16 && cache_dtype != SNA_DTYPE_FP8_E4M3FN && cache_dtype != SNA_DTYPE_INT8)
    return fail(SNA_ERR_UNSUPPORTED, "%s: cache dtype %d (bf16, FP8 e4m3fn or int8)", what, cache_dtype);
  if (head_dim != 64 && head_dim != 128)
    return fail(SNA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  if (page_size < 16 || page_size % 16 || page_size > SNA_MAX_BLOCK_PAGE)
    return fail(SNA_ERR_UNSUPPORTED, "%s: page_size %d (a multiple of 16, at most %d)", what, page_size,
                SNA_MAX_BLOCK_PAGE);
  const bool scaled = cache_dtype != SNA_DTYPE_BF16;
  if (scaled && (scale_tokens < 16 || scale_tokens % 16 || page_size % scale_tokens))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: a scale for every %d tokens (a multiple of 16 that divides the page of %d)",
                what, scale_tokens, page_size);
  if (!q_start && (max_q_len != 1 || n_tokens != R))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: without q_start each request has one token (%d tokens, R %d, max_q_len %d)",
                what, n_tokens, R, max_q_len);
  const int64_t width = (int64_t)num_kv_heads * head_dim;
  if (k_row_stride < width || v_row_stride < width || k_row_stride % 8 || v_row_stride % 8)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: rows of %lld elements, %lld and %lld apart (multiples of 8)", what,
                (long long)width, (long long)k_row_stride, (long long)v_row_stride);
  if (n_tokens == 0 || R == 0 || max_q_len == 0) return SNA_OK;
  if (!k || !v || !block_table || !prior_lens || !k_cache || !v_cache || (scaled && (!k_scale || !v_scale)))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: k, v and the caches must be 16-byte aligned", what);
  BlockStoreArgs a;
  a.x[0] = (const uint16_t*)k, a.x[1] = (const uint16_t*)v;
  a.x_row[0] = k_row_stride, a.x_row[1] = v_row_stride;
  a.cache[0] = (uint8_t*)k_cache, a.cache[1] = (uint8_t*)v_cache;
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.bounds = (uint16_t*)k_bounds;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.q_start = q_start;
  a.prior = prior_lens;
  a.T = n_tokens;
  a.G = num_kv_heads;
  a.P = page_size;
  a.bt = scaled ? scale_tokens : page_size % 32 ? 16 : 32;  // (bf16: what a wave holds at a time)
  a.max_q = max_q_len < n_tokens ? max_q_len : n_tokens;
  a.pages = (int32_t)(((int64_t)a.max_q + page_size - 2) / page_size + 1);
  a.num_blocks = num_blocks;
  if ((int64_t)R * a.pages >= 1 << 24 || num_kv_heads > 65535)  // (a grid has under 2^32 threads)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d requests of up to %d pages, %d heads exceed the grid", what, R, a.pages,
                num_kv_heads);
  if (head_dim == 128) launch_block_store_format<128>(a, R, cache_dtype, (hipStream_t)stream);
  else launch_block_store_format<64>(a, R, cache_dtype, (hipStream_t)stream);
  return check_launch(what);
}
