// Writer of a cache whose blocks of tokens carry a scale each: a call's tokens join their requests' pages [blocks, G, P, D]
// (e4m3fn or int8 codes with a scale for every `bt` tokens of a page and KV head; bf16 without scales), and, where asked
// for, the pages' key bounds (the least and the largest value of each dimension over a page's keys).
//
// For a block (bt tokens, one KV head, K or V apart) that the call writes from its token `lo` on:
//   fresh = max(max |x| * (1 / top), 2^-100) over the call's tokens of the block (infinities not counted; a NaN makes it NaN;
//           the reciprocal rounded, so no division)
//   scale = fresh where lo = 0 (the block starts anew), else max(fresh, the scale it had)
//   code  = round(clamp(x / scale)) of the new tokens; where the scale grew, the tokens before lo are rounded again,
//           round(code * had / scale), so that one scale holds for the block.
// top is 448 (e4m3fn) or 127 (int8), quotients are correctly rounded, codes rounded to nearest even.
//
// Work: one workgroup per (page that a request writes, KV head). A block of K or of V is a task, taken by one wave, or by a
// team of 2 or 4 where the block is longer than a wave's registers hold (8 pieces of 1 KB: 32 rows of 128); the rows, 16 bytes a
// lane, stay in registers between the maximum and the rounding. Their loads go out before the page is looked up.
//
// What bounds it: one round of waves that all load, then compute, then store, so neither memory nor the vector units are busy
// throughout. Four requests of 2048 tokens, 8 KV heads of 128, FP8, pages of 64 with bounds, blocks of 32: 15.5 us (51 MB, 3.3
// TB/s; without bounds 14.0; bf16, 67 MB, 13.4). From 22.2: magnitudes as packed 16-bit integers, quotients without clamps
// where no element is infinite (VALU an element 16 -> 8) 17.7; rows past the end clamped instead of masked, bounds through LDS,
// 5 waves a SIMD (one round) 15.5. Blocks of 128: one wave a block 31.6, teams 17.8.
#include <algorithm>
#include <type_traits>

#include "sna_device.h"
#include "sna_host.h"

namespace sna {

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

struct BlockStoreArgs {
  const uint16_t* x[2];  // the new tokens' K and V, [T, G, D] bf16, rows x_row elements apart
  uint32_t x_row[2];
  uint8_t* cache[2];     // K, V [num_blocks, G, P, D]
  float* scale[2];       // [num_blocks, G, P / bt]
  uint16_t* bounds;      // [num_blocks, G, 2, D] bf16, or null
  const int32_t* table;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* q_start;  // [R + 1], or null: token r is request r's
  const int32_t* prior;    // [R]
  int32_t R, T, G, P, bt, max_q, pages;  // pages: the most that a request's tokens can touch
  int32_t items;  // workgroups of a KV head: R * pages, or (less) as many pages as the call can touch, found by block_item
  int64_t num_blocks;
};

// Four elements over s, rounded to four codes of a format, the first in the low byte. The quotient comes from rs, the rounded
// 1 / s, corrected once by its exact residual (correctly rounded so). TAME: no |x| is past top * s, so no quotient rounds past
// the top; else quotients are held to the range that the clamp leaves open (see quantize_pair_e4m3fn_hw) and clamped.
// sign: the elements' sign bits, in the codes' places (e4m3fn: the residual of -0 is +0).
template <int FMT, bool TAME>
__device__ __forceinline__ uint32_t block_codes(const float (&x)[4], float s, float rs, uint32_t sign) {
  constexpr float top = FMT == kBlockFp8 ? kFp8Max : kInt8Max;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float q = x[i] * rs;
    if (!TAME) q = __builtin_amdgcn_fmed3f(q, -1024.0f, 1024.0f);
    y[i] = fmaf(fmaf(-q, s, x[i]), rs, q);
    if (!TAME) y[i] = __builtin_amdgcn_fmed3f(y[i], -top, top);
  }
  if constexpr (FMT == kBlockFp8) {
    uint32_t c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], (int)c, true);
    return (c & 0x7f7f7f7fu) | (sign & 0x80808080u);
  } else {
    // adding 1.5 * 2^23 rounds to a whole number, to nearest even, whose low byte is the code
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(y[i] + 12582912.0f);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
  }
}
// The same of four bf16 elements, two a word.
template <int FMT, bool TAME>
__device__ __forceinline__ uint32_t block_codes_bf16(uint32_t w0, uint32_t w1, float s, float rs) {
  const float x[4] = {__uint_as_float(w0 << 16), __uint_as_float(w0 & 0xffff0000u), __uint_as_float(w1 << 16),
                      __uint_as_float(w1 & 0xffff0000u)};
  return block_codes<FMT, TAME>(x, s, rs, __builtin_amdgcn_perm(w1, w0, 0x07050301u));
}
template <int FMT>
__device__ __forceinline__ void block_values(uint32_t w, float (&x)[4]) {
  if constexpr (FMT == kBlockFp8) {
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
}

// Request r's tokens: rows [t0, t0 + n) of the call (n = 0: none).
__device__ __forceinline__ void block_request(const BlockStoreArgs& a, int32_t r, int32_t& t0, int32_t& n, int32_t& prior) {
  t0 = r, n = 1;
  if (a.q_start) {
    t0 = a.q_start[r];
    const int32_t t1 = min(a.q_start[r + 1], a.T);
    n = t0 >= 0 && t1 > t0 ? min(t1 - t0, a.max_q) : 0;
  }
  prior = a.prior[r];
  if (prior < 0) n = 0;
}

// The item'th page that the call touches, request by request: its request and its place among the request's pages (every lane
// of the wave gets the same; false past the last).
__device__ bool block_item(const BlockStoreArgs& a, int32_t item, int32_t& r_out, int32_t& j_out) {
  const int lane = threadIdx.x & 63;
  int32_t base = 0;
  for (int32_t r0 = 0; r0 < a.R; r0 += 64) {  // uniform
    int32_t t0, n = 0, prior = 0;
    if (r0 + lane < a.R) block_request(a, r0 + lane, t0, n, prior);
    const int32_t pages = n > 0 ? (int32_t)(((int64_t)prior + n - 1) / a.P) - prior / a.P + 1 : 0;
    int32_t part;
    const int32_t incl = wave_incl_scan_i32(pages, &part);
    if (item < base + part) {
      const uint64_t mine = __ballot(item >= base + incl - pages && item < base + incl);
      const int32_t src = (int32_t)__builtin_amdgcn_readfirstlane(__ffsll((long long)mine) - 1);
      r_out = r0 + src;
      j_out = item - base - __builtin_amdgcn_readlane(incl - pages, src);
      return true;
    }
    base += part;
  }
  return false;
}

template <int D, int FMT, int WAVES, int TEAM>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(5)))
void kv_store_blocks_kernel(BlockStoreArgs a) {
  constexpr int LR = D / 8;     // lanes a row, 8 elements each
  constexpr int RP = 64 / LR;   // rows a wave holds in a piece
  constexpr int HELD = 8;       // pieces held in registers
  constexpr int ESZ = FMT == kBlockBf16 ? 2 : 1;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col8 = lane % LR, row0 = lane / LR;
  const int team = wave / TEAM, part = wave % TEAM;
  // (KV head fastest: a page's heads, whose rows of the call lie side by side, at one time: bf16 15.2 -> 13.5 us)
  const uint32_t pj = blockIdx.x / (uint32_t)a.G;
  const int32_t g = (int32_t)(blockIdx.x - pj * a.G);
  int32_t r = (int32_t)(pj / (uint32_t)a.pages), j = (int32_t)pj - r * a.pages;
  if (a.items != a.R * a.pages && !__builtin_amdgcn_readfirstlane((int)block_item(a, (int32_t)pj, r, j))) return;
  r = __builtin_amdgcn_readfirstlane(r), j = __builtin_amdgcn_readfirstlane(j);

  int32_t t0, n, prior;
  block_request(a, r, t0, n, prior);
  if (n == 0) return;
  // this workgroup's page and the positions [lo, hi) in it that the call writes
  const int64_t col = prior / a.P + (int64_t)j;
  const int64_t first = col * a.P;
  const int32_t lo = (int32_t)max((int64_t)prior - first, (int64_t)0);
  const int32_t hi = (int32_t)min((int64_t)prior + n - first, (int64_t)a.P);
  if (hi <= lo || col >= a.table_width) return;
  const int32_t page = a.table[(int64_t)r * a.table_stride + col];  // (on its way while the rows are asked for)
  // token `at` of the page is row src + at of the call
  const int64_t src = (int64_t)t0 + (first - prior);
  const int32_t nblk = a.P / a.bt, b0 = lo / a.bt, b1 = (hi - 1) / a.bt + 1, tasks = 2 * (b1 - b0);

  // A task: block b0 + task / 2 of K (even) or V, taken by the TEAM waves of a team, HELD pieces each in turn: piece i of a
  // wave's from p0 on. A workgroup's teams take TEAMS tasks at a time.
  constexpr int TEAMS = WAVES / TEAM;
  static_assert(TEAMS % 2 == 0, "a team keeps to K or to V");
  const int which = team & 1;
  const uint16_t* x = a.x[which] + src * (int64_t)a.x_row[which] + g * D + 8 * col8;
  const uint32_t x_row = a.x_row[which];
  int32_t head = 0, from = 0, to = 0, pieces = 0;
  uint4 w[HELD];
  auto take = [&](int32_t task) {
    head = (b0 + (task >> 1)) * a.bt;
    from = max(lo, head), to = min(hi, head + a.bt);
    pieces = task < tasks ? (to - from + RP - 1) / RP : 0;
  };
  auto load = [&](int32_t p0) {  // (a lane past the last row takes that row again)
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (p0 + i < pieces) w[i] = ld16_stream(x + (uint64_t)(uint32_t)min(from + (p0 + i) * RP + row0, to - 1) * x_row);
  };
  take(team);
  load(part * HELD);
  if (page < 0 || (int64_t)page >= a.num_blocks) return;
  const int64_t ph = (int64_t)page * a.G + g;

  __shared__ int32_t sm_most[WAVES];
  float low[8], high[8];  // K: the negated least and the largest of this lane's 8 dimensions
#pragma unroll
  for (int e = 0; e < 8; ++e) low[e] = high[e] = -INFINITY;
  for (int32_t task0 = 0; task0 < tasks; task0 += TEAMS) {  // uniform in the workgroup
    if (task0 > 0) take(task0 + team);  // (past the last task: no pieces)
    uint8_t* cache = a.cache[which] + (ph * a.P * D + 8 * col8) * ESZ;
    float* sp = FMT == kBlockBf16 ? nullptr : a.scale[which] + ph * nblk + head / a.bt;
    const float had = FMT != kBlockBf16 && pieces > 0 && from > head ? *sp : 0.0f;
    // the largest magnitude, as bf16 bits without the sign (NaN's are above infinity's), and the keys' bounds
    u16x2_t bits = {0, 0};
    for (int32_t p0 = part * HELD; p0 < pieces; p0 += TEAM * HELD) {
      if (p0 >= TEAM * HELD || task0 > 0) load(p0);
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        if (p0 + i >= pieces) break;
        const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        if constexpr (FMT != kBlockBf16) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            bits = __builtin_elementwise_max(bits, __builtin_bit_cast(u16x2_t, ww[e] & 0x7fff7fffu));
        }
        if (a.bounds && which == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = __uint_as_float(e & 1 ? ww[e >> 1] & 0xffff0000u : ww[e >> 1] << 16);
            low[e] = fmaxf(low[e], -f), high[e] = fmaxf(high[e], f);
          }
        }
      }
    }
    float s = 1.0f, rs = 1.0f;
    bool tame = true;
    if constexpr (FMT != kBlockBf16) {
      constexpr float top = FMT == kBlockFp8 ? kFp8Max : kInt8Max;
      constexpr int32_t kWild = 1 << 16;  // the block holds an infinity or a NaN
      int32_t most = wave_max_nonneg_i32(max((int32_t)bits[0], (int32_t)bits[1]));
      if (most >= 0x7f80) {  // (uniform) the largest of the others
        int32_t other = 0;
        bool nan = false;
#pragma unroll 1
        for (int32_t at = from + part * RP + row0; at < to; at += TEAM * RP) {
          const uint4 v = ld16(x + (uint64_t)(uint32_t)at * x_row);
          const uint32_t ww[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int32_t u = (int32_t)((ww[e >> 1] >> (16 * (e & 1))) & 0x7fffu);
            nan |= u > 0x7f80;
            other = max(other, u < 0x7f80 ? u : 0);
          }
        }
        most = kWild | (__any(nan) ? 0x7fc0 : wave_max_nonneg_i32(other));
      }
      if constexpr (TEAM > 1) {  // the team's
        if (task0 > 0) __syncthreads();
        if (lane == 0) sm_most[wave] = most;
        __syncthreads();
        int32_t wild = 0;
        most = 0;
#pragma unroll
        for (int i = 0; i < TEAM; ++i) {
          const int32_t m = sm_most[team * TEAM + i];
          wild |= m & kWild, most = max(most, m & 0xffff);
        }
        most = __builtin_amdgcn_readfirstlane(most | wild);
      }
      if (pieces == 0) continue;
      const float amax = bf16_bits_to_f32((uint32_t)most & 0xffffu);
      const float nan_f = __uint_as_float(0x7fc00000u);
      s = amax != amax ? nan_f : fmaxf(amax * (1.0f / top), kLeastBlockScale);
      if (from > head) s = s != s || had != had ? nan_f : fmaxf(s, had);
      rs = 1.0f / s;
      // (a block whose scale was no number gives quotients that are none: clamped they are codes that are numbers, which a
      // probability of 0 times gives 0, so that the block reaches nobody who does not see it)
      tame = most < kWild && s < INFINITY;
      // the block's earlier tokens, where the scale grew, four rows' loads in flight
      if (from > head && s > had) {
        for (int32_t at0 = head + part * RP + row0; at0 < from; at0 += 4 * TEAM * RP) {
          uint2 c[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) c[i] = ld8(cache + (int64_t)min(at0 + i * TEAM * RP, from - 1) * D);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            asm volatile("" : "+v"(c[i].x), "+v"(c[i].y));  // (one row after the other)
            const int32_t at = at0 + i * TEAM * RP;
            float y[4];
            block_values<FMT>(c[i].x, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] *= had;
            c[i].x = block_codes<FMT, false>(y, s, rs, c[i].x);
            block_values<FMT>(c[i].y, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] *= had;
            c[i].y = block_codes<FMT, false>(y, s, rs, c[i].y);
            if (at < from) *reinterpret_cast<uint2*>(cache + (int64_t)at * D) = c[i];
          }
        }
      }
      if (part == 0 && lane == 0) *sp = s;
    }
    if (!tame) {
      if constexpr (FMT != kBlockBf16) {
#pragma unroll 1
        for (int32_t at = from + part * RP + row0; at < to; at += TEAM * RP) {
          const uint4 v = ld16(x + (uint64_t)(uint32_t)at * x_row);
          *reinterpret_cast<uint2*>(cache + (int64_t)at * D) = make_uint2(block_codes_bf16<FMT, false>(v.x, v.y, s, rs),
                                                                          block_codes_bf16<FMT, false>(v.z, v.w, s, rs));
        }
      }
      continue;
    }
    // (new values to the compiler, which would else hold every element as a float from the maximum to the rounding: twice the
    // registers)
#pragma unroll
    for (int i = 0; i < HELD; ++i) asm volatile("" : "+v"(w[i].x), "+v"(w[i].y), "+v"(w[i].z), "+v"(w[i].w));
    for (int32_t p0 = part * HELD; p0 < pieces; p0 += TEAM * HELD) {
      if (pieces > TEAM * HELD) load(p0);
      const int32_t left = to - (from + p0 * RP + row0);  // rows from this lane's first one on
      uint8_t* dst = cache + (int64_t)(from + p0 * RP + row0) * D * ESZ;
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        if (p0 + i >= pieces) break;
        const uint4 v = w[i];
        if constexpr (FMT == kBlockBf16) {
          if (i * RP < left) *reinterpret_cast<uint4*>(dst + i * RP * D * 2) = v;
        } else {
          const uint2 c = make_uint2(block_codes_bf16<FMT, true>(v.x, v.y, s, rs), block_codes_bf16<FMT, true>(v.z, v.w, s, rs));
          if (i * RP < left) *reinterpret_cast<uint2*>(dst + i * RP * D) = c;
        }
      }
    }
  }

  // ---- the page's key bounds: over the wave's rows, over the waves, and with what the page had ----
  if (!a.bounds) return;
  __shared__ __attribute__((aligned(16))) float sm[WAVES / 2][RP][2][D];  // of the waves that take K
  if (which == 0) {
    float* own = &sm[team / 2 * TEAM + part][row0][0][8 * col8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      *reinterpret_cast<f32x4_t*>(own + e) = f32x4_t{-low[e], -low[e + 1], -low[e + 2], -low[e + 3]};
      *reinterpret_cast<f32x4_t*>(own + D + e) = f32x4_t{high[e], high[e + 1], high[e + 2], high[e + 3]};
    }
  }
  __syncthreads();
  for (int32_t i = tid; i < 2 * D; i += 64 * WAVES) {
    const bool upper = i >= D;
    uint16_t* b = a.bounds + ph * 2 * D + i;
    float f = lo > 0 ? bf16_bits_to_f32(*b) : (upper ? -INFINITY : INFINITY);
#pragma unroll
    for (int v = 0; v < WAVES / 2; ++v)
#pragma unroll
      for (int u = 0; u < RP; ++u) {
        const float o = (&sm[v][u][0][0])[i];
        f = upper ? fmaxf(f, o) : fminf(f, o);
      }
    *b = (uint16_t)(__float_as_uint(f) >> 16);  // a bf16 value already
  }
}

template <int D, int FMT>
static void launch_block_store(const BlockStoreArgs& a, hipStream_t s) {
  const dim3 grid((uint32_t)(a.items * a.G));
  // a wave holds 8 pieces of 64 * 8 elements: so many waves share a block of tokens; a workgroup takes K's and V's at once
  const int32_t waves = (a.bt * D + 8 * 512 - 1) / (8 * 512);
  if (FMT == kBlockBf16 || waves <= 1) {
    // a page of one block, or of one token's, is two tasks: two waves; else four (2 | 4 waves, us; 4 x 2048 tokens, 8 heads of 128,
    // FP8: pages of 64 of blocks of 16 20.2 | 15.4, of 32 17.8 | 13.6, of 64 14.4 | 14.3; of 32 of blocks of 16 16.2 | 15.6, of 32
    // 14.6 | 17.9; of 16 16.1 | 21.9; bf16 pages of 64 17.8 | 14.2; 256 rows of one token, FP8 7.1 | 9.5, of 64 5.4 | 5.4)
    if (a.bt == a.P || a.max_q == 1) hipLaunchKernelGGL((kv_store_blocks_kernel<D, FMT, 2, 1>), grid, dim3(128), 0, s, a);
    else hipLaunchKernelGGL((kv_store_blocks_kernel<D, FMT, 4, 1>), grid, dim3(256), 0, s, a);
  } else if (waves <= 2) {
    hipLaunchKernelGGL((kv_store_blocks_kernel<D, FMT == kBlockBf16 ? kBlockFp8 : FMT, 4, 2>), grid, dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((kv_store_blocks_kernel<D, FMT == kBlockBf16 ? kBlockFp8 : FMT, 8, 4>), grid, dim3(512), 0, s, a);
  }
}

template <int D>
static void launch_block_store_format(const BlockStoreArgs& a, int32_t dtype, hipStream_t s) {
  if (dtype == SNA_DTYPE_BF16) launch_block_store<D, kBlockBf16>(a, s);
  else if (dtype == SNA_DTYPE_INT8) launch_block_store<D, kBlockInt8>(a, s);
  else launch_block_store<D, kBlockFp8>(a, s);
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
  if (k_row_stride < width || v_row_stride < width || k_row_stride % 8 || v_row_stride % 8 ||
      std::max(k_row_stride, v_row_stride) > INT32_MAX)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: rows of %lld elements, %lld and %lld apart (multiples of 8 below 2^31)", what,
                (long long)width, (long long)k_row_stride, (long long)v_row_stride);
  if (n_tokens == 0 || R == 0 || max_q_len == 0) return SNA_OK;
  if (!k || !v || !block_table || !prior_lens || !k_cache || !v_cache || (scaled && (!k_scale || !v_scale)))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: k, v and the caches must be 16-byte aligned", what);
  BlockStoreArgs a;
  a.x[0] = (const uint16_t*)k, a.x[1] = (const uint16_t*)v;
  a.x_row[0] = (uint32_t)k_row_stride, a.x_row[1] = (uint32_t)v_row_stride;
  a.cache[0] = (uint8_t*)k_cache, a.cache[1] = (uint8_t*)v_cache;
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.bounds = (uint16_t*)k_bounds;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.q_start = q_start;
  a.prior = prior_lens;
  a.R = R;
  a.T = n_tokens;
  a.G = num_kv_heads;
  a.P = page_size;
  a.bt = scaled ? scale_tokens : page_size % 32 ? 16 : 32;  // (bf16: what a wave holds at a time)
  a.max_q = max_q_len < n_tokens ? max_q_len : n_tokens;
  a.pages = (int32_t)(((int64_t)a.max_q + page_size - 2) / page_size + 1);
  a.num_blocks = num_blocks;
  // A batch of one long chunk and many short ones (a chunk between decode steps): most of R * pages workgroups would find no
  // page, so the pages there are, at most one for every page_size tokens and two a request, are counted out instead.
  const int64_t direct = (int64_t)R * a.pages, touched = (int64_t)n_tokens / page_size + 2 * (int64_t)R;
  const int64_t items = direct > 4 * touched ? touched : direct;
  if (items * num_kv_heads >= 1 << 23 || direct > INT32_MAX)  // (a grid has under 2^32 threads)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d requests of up to %d pages, %d heads exceed the grid", what, R, a.pages,
                num_kv_heads);
  a.items = (int32_t)items;
  if (head_dim == 128) launch_block_store_format<128>(a, cache_dtype, (hipStream_t)stream);
  else launch_block_store_format<64>(a, cache_dtype, (hipStream_t)stream);
  return check_launch(what);
}
