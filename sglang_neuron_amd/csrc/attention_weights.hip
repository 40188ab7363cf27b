// The attention weight that each cached key of a GQA layer receives: for request r, KV head g and key j
//   W[r, g, j] (+)= sum over the request's queries i and the group's heads h of p(i, h, j),
//   p(i, h, j) = exp(s(i, h, j)) / (sum over the keys that i sees of exp(s(i, h, .)) + exp(sink_h)),
// s = sm_scale * q . k with K read from the paged pool (bf16, or e4m3fn with per-KV-head scales). A query at position p
// sees the keys (p - window, p] (all up to p without a window) that lie on valid pages; a query that sees none adds
// nothing. It is what an eviction by accumulated weight ranks the keys by.
//
// A probability needs its row's sum over all keys before it can be added to its key's. Three forms, by the number of query
// rows ((query token, head) pairs of one KV head, token-major: row = t * group + j) and how the batch fills the chip:
//   many rows   the scores are computed twice, key-stationary:
//     weights_tile_kernel<kStats>  per block of 256 keys and query row: the largest score, the sum of exp(score - largest)
//     weights_merge_kernel         per query row: the blocks merged to the row's largest score and 1 / its whole sum
//     weights_tile_kernel<kSum>    per key: the probabilities summed over a run of the rows
//     weights_reduce_kernel        per key: the runs' sums added, where the queries are cut into runs
//   up to 16 rows, as in a decode step: the keys are read once
//     weights_score_kernel         the scores to a workspace, and each block's (largest, sum)
//     weights_from_scores_kernel   the blocks merged, the probabilities of a key summed
//   the same, with (request, KV head) pairs enough to fill the chip:
//     weights_row_kernel           a pair's scores in the LDS of one workgroup: one launch
// Scores are fp32, exponentials in the log2 domain, every sum fp32; sums run in a fixed order, without atomics.
//
// Measured (us of kernels; heads 32/8 of 128, e4m3fn, pages of 16, where not said): 64 rows of 4096 keys 66, 273 MB of
// keys at 4.2 TB/s (HBM: a plain copy reaches 4.8); 8 rows of 128-1024 bf16 keys, heads 16/8, 5.0 + 4.1 (two launches and
// their chains of round trips); 128 rows of 2048-8192 keys, heads 8/1 of 64, 17 + 8 (the same, ragged, and 22 MB of scores
// written and read beside 43 MB of keys); 32 queries over each of 3001 to 16384 keys 22 + 5 + 26 (three launches' chains of
// loads) and 64 over 131071 bf16 keys 214-224 in all (products 28-31% and VALU 49-56% of the cycles, the keys read twice at 2.6
// TB/s); 4 x 2048 queries after 2048 each 470-490 in all, the first pass a little over half: products take 36% (40% in the second
// pass) of a SIMD's cycles and VALU instructions 59% (54%). These are two pipes that different waves could keep busy at once;
// that their shares add up to 95% says that the three waves of a SIMD hardly overlap them here, not that they cannot.
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "sna_device.h"
#include "sna_host.h"

namespace sna {

struct WeightsArgs {
  const uint16_t* q;       // [T, H, D] bf16
  const uint8_t* k_cache;  // [num_blocks, G, P, D]
  const float* k_scale;    // [G] dequantization scales, or (mul_scale) multipliers m: a byte is worth byte / m
  bool mul_scale;
  const int32_t* table;  // [R, table_width] (row stride table_stride)
  int64_t table_stride;
  int32_t table_width;
  const int32_t* q_start;  // [R + 1], or null: request r has the one query r
  const int32_t* lens;     // [R] prior tokens (q_start), or keys with the query's own
  const float* sinks;      // [H] natural-log sink logits, or null
  float* weights;          // [R, G, width], strides below
  int64_t w_row, w_head;
  int32_t width;
  bool add;  // add to what is there instead of writing every column
  int32_t T, R, H, G, P, group, max_q;
  uint64_t magic;  // ceil(2^32 / group): row / group = row * magic >> 32 while rows * group <= 2^32
  int64_t num_blocks;
  float sm_scale;
  int32_t window;
  int32_t blocks;    // key blocks that the table's keys (and, when every column is written, the width) take
  float2* ws_part;   // [G, blocks, T * group] a block's (largest score in the log2 domain, sum)
  float2* ws_row;    // [G, T * group] a row's (largest score in the log2 domain, 1 / sum)
  int32_t splits, split_tokens;  // the queries are cut into so many runs of so many tokens (a multiple of 32)
  float* ws_sum;     // [splits, R, G, blocks * 256] the runs' sums, with more than one
  // few rows instead: ws_part is [R, G, blocks, max_q * group], and
  float* ws_score;   // [R, G, max_q * group, blocks * score_keys] scores in the log2 domain, -inf where unseen
  int32_t span, score_keys;  // chunks of a workgroup, and their keys (weights_row_kernel: a row's keys in LDS)
};

constexpr int kWeightKeys = 256;  // keys of a workgroup, 64 to a wave
constexpr int kWeightRows = 32;   // query rows of a tile

// A request's queries and keys: rows 0 .. S - 1 are tokens qa .. of q at positions prior + t; keys 0 .. n - 1.
struct WeightsRequest {
  int32_t qa, S;
  int64_t prior;
  int32_t n;
};
__device__ __forceinline__ WeightsRequest weights_request(const WeightsArgs& a, int32_t r) {
  WeightsRequest q;
  if (a.q_start) {
    // (offsets outside q, or a chunk past max_q, are cut: no row past q is read)
    q.qa = min(max(ld_const(a.q_start + r), 0), a.T);
    q.S = min(min(max(ld_const(a.q_start + r + 1), q.qa), a.T) - q.qa, a.max_q);
    q.prior = ld_const(a.lens + r);
  } else {
    q.qa = r, q.S = 1;
    q.prior = (int64_t)ld_const(a.lens + r) - 1;
  }
  q.n = (int32_t)min(max(q.prior + q.S, (int64_t)0), (int64_t)a.table_width * a.P);
  return q;
}

template <int D, int ESZ>
struct WeightsGeo {
  static constexpr int NS = D / 16;            // matrix steps of a score
  static constexpr int ROWB = D * ESZ;         // bytes of a key
  static constexpr int KCH = ROWB / 16;        // its 16-byte chunks
  static constexpr int KEYB = 64 * ROWB;       // bytes of a wave's keys
  static constexpr int QCH = D * 2 / 16;       // 16-byte chunks of a query row
  static constexpr int TILE = kWeightRows * QCH;
  // Rows of N chunks lie in LDS with chunk c of row r at c ^ swz(r), so that 16 lanes which read one chunk of 16
  // consecutive rows touch every bank once.
  static __device__ __forceinline__ int swz(int r, int n) { return (n >= 16 ? r : r / (16 / n)) & (n - 1); }
};

// The wave's 64 keys from k0 on, lane i's being key k0 + i: its first byte in the cache, or -1 where there is none.
__device__ __forceinline__ int64_t weights_key_at(const WeightsArgs& a, int32_t r, int32_t g, int32_t key, int32_t n,
                                                  int32_t row_bytes) {
  if (key >= n) return -1;
  const int32_t col = key / a.P;
  const int64_t page = a.table[r * a.table_stride + col];
  if (page < 0 || page >= a.num_blocks) return -1;
  return ((page * a.G + g) * a.P + (key - col * a.P)) * (int64_t)row_bytes;
}

// Loads straight into LDS (lane i's bytes at LDS address m0 + size * i) from an address per lane, kept in the caches: other
// workgroups and the second pass read them again. Assembly, as the DMAs of sna_device.h are; waited for by wait_vmcnt.
__device__ __forceinline__ void dma_global16_cached(const void* src, uint32_t lds) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(m0), "v"(src) : "memory");
}
__device__ __forceinline__ void dma_global4(const void* src, uint32_t lds) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(m0), "v"(src) : "memory");
}

// N keys of a wave (lane i holding the place of key i mod N) into LDS: whole rows by DMA, 1024 bytes an instruction, chunk
// c of row r to c ^ swz(r). A key that is not there reads the cache's first row; what comes of it is masked or dropped.
template <int D, int ESZ, int N>
__device__ __forceinline__ void weights_stage(const WeightsArgs& a, int64_t at, uint8_t* lds) {
  using Geo = WeightsGeo<D, ESZ>;
  constexpr int RPD = 1024 / Geo::ROWB;
  const int lane = threadIdx.x & 63;
  const int64_t from = at < 0 ? 0 : at;
  const uint32_t base = lds_address((lds_ptr_t*)lds);
#pragma unroll
  for (int j = 0; j < N / RPD; ++j) {
    const int row = j * RPD + lane / Geo::KCH, ch = lane % Geo::KCH ^ Geo::swz(row, Geo::KCH);
    const uint32_t lo = __shfl((uint32_t)from, row, 64), hi = __shfl((uint32_t)(from >> 32), row, 64);
    dma_global16_cached(a.k_cache + (int64_t)((uint64_t)hi << 32 | lo) + 16 * ch, base + 1024 * j);
  }
}

// The wave's 64 keys through LDS (STEP at a time) to A operands in registers: lane (g2, i) feeds key 32 s + i, dims 16 c + 8
// g2 .. of step c (bf16) or 32 (c / 2) + 16 g2 + 8 (c & 1) .. (FP8, as its 16-byte chunks hold them).
template <int D, int ESZ, int STEP>
__device__ __forceinline__ void weights_keys(const WeightsArgs& a, int64_t at, uint8_t* lds, uint32_t (&kf)[2][D / 16][4]) {
  using Geo = WeightsGeo<D, ESZ>;
  const int lane = threadIdx.x & 63, g2 = lane >> 5, i32 = lane & 31;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (STEP == 64 ? s == 0 : true) {
      int64_t from = at;
      if constexpr (STEP == 32) {  // keys 32 s .. 32 s + 31, in both halves of the wave
        const uint32_t lo = __shfl((uint32_t)at, 32 * s + i32, 64), hi = __shfl((uint32_t)(at >> 32), 32 * s + i32, 64);
        from = (int64_t)((uint64_t)hi << 32 | lo);
        if (s > 0) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the first ones are read
      }
      weights_stage<D, ESZ, STEP>(a, from, lds);
      wait_vmcnt<0>();
    }
    const int row = STEP == 64 ? 32 * s + i32 : i32;
    const uint8_t* mine = lds + row * Geo::ROWB;
    if constexpr (ESZ == 1) {
#pragma unroll
      for (int c = 0; c < Geo::NS / 2; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(mine + 16 * ((2 * c + g2) ^ Geo::swz(row, Geo::KCH)));
        fp8x4_to_bf16x4(w.x, kf[s][2 * c][0], kf[s][2 * c][1]);
        fp8x4_to_bf16x4(w.y, kf[s][2 * c][2], kf[s][2 * c][3]);
        fp8x4_to_bf16x4(w.z, kf[s][2 * c + 1][0], kf[s][2 * c + 1][1]);
        fp8x4_to_bf16x4(w.w, kf[s][2 * c + 1][2], kf[s][2 * c + 1][3]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < Geo::NS; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(mine + 16 * ((2 * c + g2) ^ Geo::swz(row, Geo::KCH)));
        kf[s][c][0] = w.x, kf[s][c][1] = w.y, kf[s][c][2] = w.z, kf[s][c][3] = w.w;
      }
    }
  }
}
// The query chunk (8 dims) that meets lane group g2's K operand of step c.
template <int ESZ>
__device__ __forceinline__ int weights_chunk(int c, int g2) {
  return ESZ == 1 ? 4 * (c / 2) + 2 * g2 + (c & 1) : 2 * c + g2;
}

// Log2-domain factor of a score.
template <int ESZ>
__device__ __forceinline__ float weights_scale(const WeightsArgs& a, int32_t g) {
  double scale = (double)a.sm_scale * 1.4426950408889634;
  if (ESZ == 1) scale = a.mul_scale ? scale / (double)a.k_scale[g] : scale * (double)a.k_scale[g];
  return (float)scale;
}

// The keys of the wave's 64 (from kw on) that a row at position pos sees, as bits.
__device__ __forceinline__ uint64_t weights_seen(const WeightsArgs& a, uint64_t valid, int64_t pos, int32_t kw) {
  const int64_t hi = pos - kw;  // keys 0 .. hi
  uint64_t seen = hi < 0 ? 0 : hi < 63 ? valid & ((2ull << hi) - 1) : valid;
  if (a.window > 0) {
    const int64_t lo = pos - a.window + 1 - kw;  // from key lo
    seen = lo > 63 ? 0 : lo > 0 ? seen & (~0ull << lo) : seen;
  }
  return seen;
}
// The lane's share of such bits: bit 8 q + r of word s is element 4 q + r of sub-tile s.
__device__ __forceinline__ uint32_t weights_bits(uint64_t seen, int s, int g2) { return (uint32_t)(seen >> 32 * s) >> 4 * g2; }
__device__ __forceinline__ constexpr uint32_t weights_bit(int e) { return 1u << (8 * (e / 4) + e % 4); }
// Key of element e of lane group g2's sub-tile s.
__device__ __forceinline__ constexpr int weights_key(int s, int e, int g2) { return 32 * s + 8 * (e / 4) + 4 * g2 + e % 4; }

// Head h's sink in the log2 domain. One past the largest number takes its rows whole, as the largest does: infinity less
// itself would be NaN.
__device__ __forceinline__ float weights_sink(const WeightsArgs& a, int32_t h) {
  const float x = a.sinks[h] * kLog2e;
  return x > FLT_MAX ? FLT_MAX : x;
}

// (largest, sum of 2^(x - largest)) of two sets merged.
__device__ __forceinline__ float2 weights_join(float2 p, float2 o) {
  const float b = fmaxf(p.x, o.x);
  return make_float2(b, p.y * __builtin_amdgcn_exp2f(p.x - b) + o.y * __builtin_amdgcn_exp2f(o.x - b));
}

// The lane's 32 scores x * c2 of one row as (largest, sum), with the lane's 32 away, which holds the row's other 32 keys.
// ALL: every key is seen and c2 > 0; else the scores are left in x, scaled and -inf where unseen.
template <bool ALL>
__device__ __forceinline__ float2 weights_stats(f32x16_t (&x)[2], float c2, uint64_t seen, int g2) {
  float mx = ALL ? -INFINITY : kNegBig, sum = 0.0f;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint32_t bits = ALL ? 0 : weights_bits(seen, s, g2);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (!ALL) x[s][e] = bits & weights_bit(e) ? x[s][e] * c2 : -INFINITY;
      mx = fmaxf(mx, x[s][e]);
    }
  }
  if (ALL) mx = fmaxf(mx * c2, kNegBig);  // (32 scores of -inf have the sum 0, as where there are masks)
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f(ALL ? fmaf(x[s][e], c2, -mx) : x[s][e] - mx);
  const float both = xor32_partner_max(mx);
  return make_float2(both, xor32_partner_sum(sum * __builtin_amdgcn_exp2f(mx - both)));
}

// Many rows. A workgroup of 4 waves owns 256 keys of one (request, KV head), 64 to a wave, held as bf16 matrix operands in
// registers (an e4m3fn value is a bf16 value); the rows of its run pass in tiles of 32 through a ring of two pairs of tiles
// in LDS that the waves share, filled by DMA, one barrier a pair. The product is S^T[key, row] = K[key, :] . Q[row, :] by
// v_mfma_f32_32x32x16_bf16, so a lane holds 16 keys of one row twice: the row's maximum, sum and normalization are values of
// the lane, and a key's sum over the rows stays in the lane's registers until the end, where it is added across the lanes
// once. A tile costs a wave 32 exponentials a lane (8 cycles each), as many fused multiply-adds, and at head_dim 128 16
// products of 32 cycles. Products and exponentials of one wave take turns, on three waves a SIMD. (The next tile's products
// among the exponentials, on two waves a SIMD, took 620 us for 4 x 2048 after 2048 where this took 590.) Pairs of tiles whose
// rows see all of the wave's keys take a path without masks.
enum WeightsPass { kStats, kSum };
template <int D, int ESZ>
struct WeightsRing {
  using Geo = WeightsGeo<D, ESZ>;
  static constexpr int SLOTS = 4;               // row tiles in LDS: a pair that is read, a pair on its way
  static constexpr int SLOTB = Geo::TILE * 16;  // bytes of a tile
  static constexpr int LD = SLOTB / 4096;       // DMAs of a tile that a wave issues
  // The keys pass through the second pair's slots (and beyond) while the first pair is on its way.
  static constexpr int STEP = Geo::ROWB > 128 ? 32 : 64;  // keys of a wave at a time: three workgroups fit a CU's LDS
  static constexpr int STAGE = STEP * Geo::ROWB;
  static constexpr int BYTES = 2 * SLOTB + (4 * STAGE > 2 * SLOTB ? 4 * STAGE : 2 * SLOTB);
};
template <int D, int ESZ, WeightsPass PASS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3)))
void weights_tile_kernel(WeightsArgs a) {
  using Geo = WeightsGeo<D, ESZ>;
  using Ring = WeightsRing<D, ESZ>;
  constexpr int NS = Geo::NS, CH = Geo::QCH, SLOTS = Ring::SLOTS, LD = Ring::LD;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[Ring::BYTES];
  __shared__ float2 sm_row[PASS == kSum ? SLOTS : 1][kWeightRows];  // the tiles' rows of ws_row
  __shared__ float sm_out[PASS == kSum ? kWeightKeys : 1];
  __shared__ float2 sm_part[PASS == kStats ? 4 : 1][4][kWeightRows];
  const int tid = threadIdx.x, lane = tid & 63, g2 = lane >> 5, i32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t lin = xcd_order(blockIdx.x, gridDim.x);
  const int32_t kb = (int32_t)(lin % a.blocks);
  lin /= a.blocks;
  const int32_t run = (int32_t)(lin % a.splits), r = (int32_t)(lin / a.splits % a.R), g = (int32_t)(lin / a.splits / a.R);
  const WeightsRequest rq = weights_request(a, r);
  const int32_t k0 = kb * kWeightKeys;
  // the run's rows that see any of the block's keys: tokens [t0, t1)
  const int64_t last = (int64_t)min(k0 + kWeightKeys, rq.n) - 1;
  // (the runs' tokens count from the 32 with the first one that sees the block)
  const int64_t run0 = (min(max(k0 - rq.prior, (int64_t)0), (int64_t)rq.S) & ~31) + (int64_t)run * a.split_tokens;
  const int32_t s0 = (int32_t)min(run0, (int64_t)rq.S), s1 = (int32_t)min(run0 + a.split_tokens, (int64_t)rq.S);
  int32_t t0 = (int32_t)min(max(k0 - rq.prior, (int64_t)s0), (int64_t)s1), t1 = s1;
  if (a.window > 0) t1 = (int32_t)min(max(last + a.window - rq.prior, (int64_t)s0), (int64_t)s1);
  if (k0 >= rq.n) t1 = t0;
  // where the block's sums go: the weights, or the run's part of them
  const bool parts = a.splits > 1;
  float* const out = parts ? a.ws_sum + (((int64_t)run * a.R + r) * a.G + g) * a.blocks * kWeightKeys
                           : a.weights + r * a.w_row + g * a.w_head;
  const int32_t width = parts ? a.blocks * kWeightKeys : a.width;
  const bool add = a.add && !parts;
  if (t1 <= t0) {  // uniform
    if (PASS == kSum && !add && k0 + tid < width) out[k0 + tid] = 0.0f;
    return;
  }
  auto token_of = [&](int32_t row) -> int32_t { return (int32_t)((uint64_t)(uint32_t)row * a.magic >> 32); };
  const int32_t m_end = t1 * a.group;
  const int32_t m0 = (t0 * a.group) & ~(kWeightRows - 1);
  const int32_t tiles = (m_end - m0 + kWeightRows - 1) / kWeightRows;
  const int64_t rows = (int64_t)a.T * a.group;  // rows of a KV head
  float2* const part = a.ws_part + ((int64_t)g * a.blocks + kb) * rows + (int64_t)rq.qa * a.group;
  const float2* const row_of = a.ws_row + (int64_t)g * rows + (int64_t)rq.qa * a.group;
  // Tile i (in order) to its slot by whole-row DMAs, chunk c of row r to c ^ swz(r). Where the heads of a token never
  // straddle two tiles, every tile but the last lies a scalar step behind the one before; else, and in the last (rows past
  // its end repeat the last one; they are dropped), the rows' tokens are found again.
  const bool whole = kWeightRows % a.group == 0;
  const uint16_t* const q0 = a.q + ((int64_t)rq.qa * a.H + g * a.group) * D;
  const uint32_t ring = lds_address((lds_ptr_t*)sm), ring_row = lds_address((lds_ptr_t*)sm_row);
  constexpr int RPD = 64 / CH;  // rows a DMA fills
  const int64_t q_step = (int64_t)(kWeightRows / a.group) * a.H * D;
  const uint16_t* q_tile = q0 + (int64_t)token_of(m0) * a.H * D;  // tile i's first row, where they are whole
  uint32_t ld_off[LD];
#pragma unroll
  for (int l = 0; l < LD; ++l) {
    const int32_t row = (LD * wave + l) * RPD + lane / CH, t = token_of(row);
    ld_off[l] = (uint32_t)(t * a.H + row - t * a.group) * (2 * D) + 16 * (lane % CH ^ Geo::swz(row, CH));
  }
  auto load = [&](int32_t i) {
    const uint32_t slot = ring + (i & (SLOTS - 1)) * Ring::SLOTB + LD * wave * 1024;
    if (whole && i < tiles - 1) {  // uniform
#pragma unroll
      for (int l = 0; l < LD; ++l) dma_saddr16_cached(q_tile, ld_off[l], slot + 1024 * l);
    } else {
#pragma unroll
      for (int l = 0; l < LD; ++l) {
        const int32_t at = (LD * wave + l) * RPD + lane / CH;
        const int32_t row = min(m0 + kWeightRows * i + at, m_end - 1), t = token_of(row);
        dma_global16_cached(q0 + ((int64_t)t * a.H + row - t * a.group) * D + 8 * (lane % CH ^ Geo::swz(at, CH)),
                            slot + 1024 * l);
      }
    }
    q_tile += q_step;
    if constexpr (PASS == kSum) {  // 8 of the tile's rows, two dwords each
      if (lane < 16) {
        const int32_t row = min(m0 + kWeightRows * i + 8 * wave + lane / 2, m_end - 1);
        dma_global4(reinterpret_cast<const float*>(row_of + row) + (lane & 1),
                    ring_row + (i & (SLOTS - 1)) * (kWeightRows * 8) + 64 * wave);
      }
    }
  };
  load(0);
  if (tiles > 1) load(1);
  const int64_t at = weights_key_at(a, r, g, k0 + tid, rq.n, Geo::ROWB);
  const uint64_t valid = __ballot(at >= 0);
  uint32_t kf[2][NS][4];
  weights_keys<D, ESZ, Ring::STEP>(a, at, sm + 2 * Ring::SLOTB + wave * Ring::STAGE, kf);
  const float c2 = weights_scale<ESZ>(a, g);
  const int32_t kw = k0 + 64 * wave;  // the wave's first key
  float acc[2][16];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[s][e] = 0.0f;
  // The pairs of tiles [f0, f1) whose every row sees all of the wave's keys (SUM does not mind keys that are not there:
  // their sums are dropped): from the pair whose first token reaches the last key, to the one before a row past the end, or
  // past the first key's window.
  const int32_t pairs = (tiles + 1) / 2;
  // the first `unseen` pairs see none of the wave's keys
  int32_t unseen = (int32_t)(max((min(kw - rq.prior, (int64_t)t1) * a.group - m0), (int64_t)0) / (2 * kWeightRows));
  unseen = __builtin_amdgcn_readfirstlane(unseen);
  int32_t f0 = pairs, f1 = 0;
  if (c2 > 0.0f && (PASS == kSum || valid == ~0ull)) {  // uniform
    auto pair_from = [&](int64_t token) -> int32_t {  // the first pair that starts at or behind a token's first row
      const int64_t row = min(max(token, (int64_t)t0), (int64_t)t1) * a.group - m0;
      return (int32_t)((row + 2 * kWeightRows - 1) / (2 * kWeightRows));
    };
    f0 = max(pair_from(kw + 63 - rq.prior), 0);
    f1 = (m_end - m0) / (2 * kWeightRows);
    if (a.window > 0) {  // whole pairs of tokens below the first one that no longer sees key kw
      const int64_t end = min(max((int64_t)kw + a.window - rq.prior, (int64_t)t0), (int64_t)t1) * a.group - m0;
      f1 = min(f1, (int32_t)(max(end, (int64_t)0) / (2 * kWeightRows)));
    }
  }
  f0 = __builtin_amdgcn_readfirstlane(f0), f1 = __builtin_amdgcn_readfirstlane(f1);
  // the four waves' parts of tile i merged and written
  auto write_part = [&](int32_t i) {
    const int32_t m = m0 + kWeightRows * i + i32;
    if (wave == (i & 3) && g2 == 0 && m < m_end) {
      const float2(*p)[kWeightRows] = sm_part[i & 3];
      part[m] = weights_join(weights_join(p[0][i32], p[1][i32]), weights_join(p[2][i32], p[3][i32]));
    }
  };
  float2 rw = make_float2(0.0f, 0.0f);  // the lane's row's (largest, 1 / sum) of a tile
  f32x16_t x[2];                        // and its scores
  // The products of tile i (past the last tile: of stale rows, dropped).
  auto products = [&](int32_t i) {
    const uint4* const slot = reinterpret_cast<const uint4*>(sm + (i & (SLOTS - 1)) * Ring::SLOTB);
    if (PASS == kSum) rw = sm_row[i & (SLOTS - 1)][i32];
    x[0] = x[1] = f32x16_t{};
#pragma unroll
    for (int c = 0; c < NS; ++c) {
      const uint4 w = slot[i32 * CH + (weights_chunk<ESZ>(c, g2) ^ Geo::swz(i32, CH))];
      const uint32_t qf[4] = {w.x, w.y, w.z, w.w};
      x[0] = mfma_32x32x16_bf16(kf[0][c], qf, x[0]);
      x[1] = mfma_32x32x16_bf16(kf[1][c], qf, x[1]);
    }
  };
  // Tile i's scores, all of them seen, or those that weights_seen says.
  auto work = [&](auto all, int32_t i) {
    constexpr bool ALL = decltype(all)::value;
    const int32_t m = m0 + kWeightRows * i + i32;
    const uint64_t seen = ALL || m >= m_end ? 0 : weights_seen(a, valid, rq.prior + token_of(m), kw);
    if constexpr (PASS == kStats) {
      const float2 p = weights_stats<ALL>(x, c2, seen, g2);
      if (g2 == 0) sm_part[i & 3][wave][i32] = p;
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t bits = weights_bits(seen, s, g2);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(x[s][e], c2, -rw.x));
          // (an unseen key keeps its sum, whatever the row's is: NaN, or stale past the last tile)
          const float sum = fmaf(p, rw.y, acc[s][e]);
          acc[s][e] = ALL || bits & weights_bit(e) ? sum : acc[s][e];
        }
      }
      // (here, not after the next tile's products: or both tiles' scores would be held)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 16; ++e) asm volatile("" : "+v"(acc[s][e]));
    }
  };
  // Before a pair of tiles, 2 p and 2 p + 1: they are in their slots once this wave's DMAs and the others' are; the barrier
  // also says that the pair before, whose slots the next pair takes, is read (and, at first, every wave's keys are).
  auto ready = [&](int32_t p) {
    wait_vmcnt<0>();
    __syncthreads();
    if (2 * p + 2 < tiles) load(2 * p + 2);
    if (2 * p + 3 < tiles) load(2 * p + 3);
    if (PASS == kStats && p > 0) {
      write_part(2 * p - 2);
      write_part(2 * p - 1);
    }
  };
  auto pair = [&](auto all, int32_t p) {
    ready(p);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      products(2 * p + b);
      work(all, 2 * p + b);
    }
  };
  int32_t p = 0;
  for (; p < unseen; ++p) {
    ready(p);
    if (PASS == kStats && g2 == 0) {
      const float2 none = make_float2(kNegBig, 0.0f);
      sm_part[2 * p & 3][wave][i32] = sm_part[(2 * p + 1) & 3][wave][i32] = none;
    }
  }
  for (; p < min(f0, pairs); ++p) pair(std::false_type{}, p);
  for (; p < f1; ++p) pair(std::true_type{}, p);
  for (; p < pairs; ++p) pair(std::false_type{}, p);
  if constexpr (PASS == kStats) {
    __syncthreads();
    write_part(2 * pairs - 2);
    write_part(2 * pairs - 1);
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float v = row16_sum(acc[s][e]);
        const float both = v + __shfl_xor(v, 16, 64);
        if (i32 == 0) sm_out[64 * wave + weights_key(s, e, g2)] = both;
      }
    __syncthreads();
    const int32_t key = k0 + tid;
    if (key < width) {
      const float v = at >= 0 ? sm_out[tid] : 0.0f;
      if (!add) out[key] = v;
      else if (at >= 0) out[key] += v;
    }
  }
}

// The runs' sums of a key added in their order.
__global__ __launch_bounds__(256) void weights_reduce_kernel(WeightsArgs a) {
  const int32_t r = blockIdx.z, g = blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
  const WeightsRequest rq = weights_request(a, r);
  if (key >= a.width || (a.add && key >= rq.n)) return;
  const int64_t step = (int64_t)a.R * a.G * a.blocks * kWeightKeys;
  const float* src = a.ws_sum + ((int64_t)r * a.G + g) * a.blocks * kWeightKeys + key;
  float v = 0.0f;
#pragma unroll 4
  for (int32_t s = 0; s < a.splits; ++s) v += src[s * step];
  float* out = a.weights + r * a.w_row + g * a.w_head + key;
  *out = a.add ? *out + v : v;
}

// A row's blocks merged: (its largest score M in the log2 domain, 1 / sum of 2^(score - M) with the sink's). ROWS rows a
// workgroup, a row's blocks dealt to 256 / ROWS threads.
template <int ROWS>
__global__ __launch_bounds__(256) void weights_merge_kernel(WeightsArgs a) {
  constexpr int SLICES = 256 / ROWS;
  __shared__ float2 sm[SLICES][ROWS];
  const int32_t r = blockIdx.z, g = blockIdx.y;
  const WeightsRequest rq = weights_request(a, r);
  const int i = threadIdx.x % ROWS, slice = threadIdx.x / ROWS;
  if ((int32_t)blockIdx.x * ROWS >= rq.S * a.group) return;  // uniform
  const int32_t m = min((int32_t)blockIdx.x * ROWS + i, rq.S * a.group - 1);
  const int32_t t = m / a.group, h = g * a.group + m - t * a.group;
  const int64_t pos = rq.prior + t;
  const int64_t rows = (int64_t)a.T * a.group;
  const int64_t row = (int64_t)rq.qa * a.group + m;
  // the blocks that hold keys it sees: each has written this row
  const int64_t hi = min(pos, (int64_t)rq.n - 1), lo = a.window > 0 ? max(pos - a.window + 1, (int64_t)0) : 0;
  float2 p = make_float2(kNegBig, 0.0f);
  if (hi >= lo) {
    const int32_t b1 = (int32_t)(hi / kWeightKeys);
#pragma unroll 4
    for (int32_t b = (int32_t)(lo / kWeightKeys) + slice; b <= b1; b += SLICES)
      p = weights_join(p, a.ws_part[((int64_t)g * a.blocks + b) * rows + row]);
  }
  sm[slice][i] = p;
  __syncthreads();
  if (slice == 0 && (int32_t)blockIdx.x * ROWS + i < rq.S * a.group) {
    for (int s = 1; s < SLICES; ++s) p = weights_join(p, sm[s][i]);
    if (a.sinks) p = weights_join(p, make_float2(weights_sink(a, h), 1.0f));
    // (a row that sees nothing: every score is dropped)
    a.ws_row[(int64_t)g * rows + row] = p.y == 0.0f ? make_float2(-kNegBig, 0.0f) : make_float2(p.x, 1.0f / p.y);
  }
}

// Few rows (at most kScoreRows a request and KV head: a decode step): the scores themselves go to the workspace, so that
// the keys are read once, and a second launch sums the probabilities from them.
constexpr int kScoreRows = 16;
// A workgroup of 4 waves takes `span` chunks of 4 x CK consecutive keys, CK to a wave; a wave's next chunk is on its way to
// LDS while it works on one. (Keys of 64 bytes: one chunk a workgroup, whose 16 KB leave room for more workgroups: 128 rows
// of 2048-8192 keys took 16 us so and 21 in spans; of 128 bytes, 64 rows of 4096, 72 and 64.) By v_mfma_f32_16x16x32_bf16:
// lane (g4, i) feeds key 16 s + i's dims 32 c + 8 g4 .. of step c (FP8: 64 (c / 2) + 16 g4 + 8 (c & 1) ..) and holds the
// scores of row i and keys 16 s + 4 g4 + e.
constexpr int score_chunk(int row_bytes) { return row_bytes > 128 ? 32 : 64; }  // keys of a wave's chunk: at most 8 KB
constexpr int score_span(int row_bytes) { return row_bytes > 64 ? 8 : 1; }      // most chunks
template <int D, int ESZ>
__global__ __launch_bounds__(256) void weights_score_kernel(WeightsArgs a) {
  using Geo = WeightsGeo<D, ESZ>;
  constexpr int NS = D / 32;                     // matrix steps
  constexpr int CK = score_chunk(Geo::ROWB), SPAN = score_span(Geo::ROWB), SLOTS = SPAN > 1 ? 2 : 1, NT = CK / 16;
  constexpr int DMAS = CK * Geo::ROWB / 1024;    // of a chunk
  __shared__ __attribute__((aligned(1024))) uint8_t sm[4][SLOTS][CK * Geo::ROWB];
  __shared__ int32_t sm_page[4][SPAN][CK];  // the keys' pages, -1 where there is none
  __shared__ float2 sm_part[4][kScoreRows];
  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, i16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t kb = (int32_t)(blockIdx.x % a.blocks), r = (int32_t)(blockIdx.x / a.blocks % a.R);
  const int32_t g = (int32_t)(blockIdx.x / a.blocks / a.R);
  const WeightsRequest rq = weights_request(a, r);
  const int32_t keys = 4 * CK * a.span, k0 = kb * keys;
  // (a block before every row's window, or past the keys, is not read by the second launch)
  if (k0 >= rq.n || rq.S == 0 || (a.window > 0 && (int64_t)k0 + keys - 1 <= rq.prior - a.window)) return;  // uniform
  const int32_t chunks = SPAN == 1 ? 1 : min(a.span, (rq.n - k0 + 4 * CK - 1) / (4 * CK));
  auto key_of = [&](int32_t q) -> int32_t { return k0 + (4 * q + wave) * CK; };  // chunk q's first key
  for (int32_t q = 0; q < chunks; ++q) {
    const int32_t key = key_of(q) + lane % CK;
    int32_t page = -1;
    if (key < rq.n) {
      page = a.table[r * a.table_stride + key / a.P];
      if (page < 0 || page >= a.num_blocks) page = -1;
    }
    if (lane < CK) sm_page[wave][q][lane] = page;
  }
  auto stage = [&](int32_t q) -> uint64_t {
    const int32_t key = key_of(q) + lane % CK, page = sm_page[wave][q][lane % CK];
    const int64_t at = page < 0 ? -1 : (((int64_t)page * a.G + g) * a.P + key % a.P) * (int64_t)Geo::ROWB;
    weights_stage<D, ESZ, CK>(a, at, sm[wave][q & (SLOTS - 1)]);
    return __ballot(page >= 0);
  };
  uint64_t valid = stage(0), next = 0;
  const int32_t m = i16, M = rq.S * a.group;
  const int32_t t = m / a.group, j = m - t * a.group;
  const uint16_t* row = a.q + ((int64_t)(rq.qa + min(t, rq.S - 1)) * a.H + g * a.group + j) * D;
  uint4 qw[NS];
#pragma unroll
  for (int c = 0; c < NS; ++c) qw[c] = ld16(row + 8 * (ESZ == 1 ? 8 * (c / 2) + 2 * g4 + (c & 1) : 4 * c + g4));
  const float c2 = weights_scale<ESZ>(a, g);
  const int32_t width = a.blocks * keys, rows = a.max_q * a.group;
  float* const dst = a.ws_score + (((int64_t)r * a.G + g) * rows + min(m, rows - 1)) * width + 4 * g4;
  float2 best = make_float2(kNegBig, 0.0f);
  for (int32_t q = 0; q < chunks; ++q) {
    if (SPAN > 1 && q + 1 < chunks) {
      next = stage(q + 1);  // its slot's last chunk is read: this wave's own
      wait_vmcnt<DMAS>();
    } else {
      wait_vmcnt<0>();
    }
    const int32_t kw = key_of(q);
    f32x4_t x[NT];
#pragma unroll
    for (int s = 0; s < NT; ++s) {
      const int key = 16 * s + i16;
      const uint8_t* k = sm[wave][q & (SLOTS - 1)] + key * Geo::ROWB;
      x[s] = f32x4_t{};
#pragma unroll
      for (int c = 0; c < NS; c += ESZ == 1 ? 2 : 1) {
        const uint4 w = *reinterpret_cast<const uint4*>(k + 16 * ((4 * (ESZ == 1 ? c / 2 : c) + g4) ^ Geo::swz(key, Geo::KCH)));
        const uint32_t q0[4] = {qw[c].x, qw[c].y, qw[c].z, qw[c].w};
        if constexpr (ESZ == 1) {
          const uint32_t q1[4] = {qw[c + 1].x, qw[c + 1].y, qw[c + 1].z, qw[c + 1].w};
          uint32_t ka[4], kc[4];
          fp8x4_to_bf16x4(w.x, ka[0], ka[1]);
          fp8x4_to_bf16x4(w.y, ka[2], ka[3]);
          fp8x4_to_bf16x4(w.z, kc[0], kc[1]);
          fp8x4_to_bf16x4(w.w, kc[2], kc[3]);
          x[s] = mfma_16x16x32_bf16(ka, q0, x[s]);
          x[s] = mfma_16x16x32_bf16(kc, q1, x[s]);
        } else {
          const uint32_t ka[4] = {w.x, w.y, w.z, w.w};
          x[s] = mfma_16x16x32_bf16(ka, q0, x[s]);
        }
      }
    }
    // scaled, -inf where unseen
    constexpr uint64_t kAll = CK == 64 ? ~0ull : (1ull << CK % 64) - 1;
    const bool all = (valid & kAll) == kAll && rq.prior >= kw + CK - 1 &&
                     (a.window <= 0 || rq.prior + rq.S - 1 - a.window < kw);  // uniform
    const uint64_t seen = all ? 0 : weights_seen(a, valid, rq.prior + t, kw) >> 4 * g4;
    float mx = kNegBig, sum = 0.0f;
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[s][e] *= c2;
        if (!all) x[s][e] = seen >> (16 * s + e) & 1 ? x[s][e] : -INFINITY;
        mx = fmaxf(mx, x[s][e]);
      }
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f(x[s][e] - mx);
    best = weights_join(best, make_float2(mx, sum));
    if (m < M) {
#pragma unroll
      for (int s = 0; s < NT; ++s) *reinterpret_cast<f32x4_t*>(dst + kw + 16 * s) = x[s];
    }
    valid = next;
  }
  const float mx = max_across_groups(best.x);
  const float sum = sum_across_groups(best.y * __builtin_amdgcn_exp2f(best.x - mx));
  if (g4 == 0) sm_part[wave][m] = make_float2(mx, sum);
  __syncthreads();
  if (tid < M)
    a.ws_part[(((int64_t)r * a.G + g) * a.blocks + kb) * rows + tid] =
        weights_join(weights_join(sm_part[0][tid], sm_part[1][tid]), weights_join(sm_part[2][tid], sm_part[3][tid]));
}

// A score's probability by its row's (largest, 1 / sum): none for an unseen one, whatever the row's sum is.
__device__ __forceinline__ float weights_p(float x, float2 row) {
  return x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - row.x) * row.y;
}

// 1024 keys a workgroup, 4 to a thread: the rows' blocks merged (16 threads a row), then every key's probabilities summed.
__global__ __launch_bounds__(256) void weights_from_scores_kernel(WeightsArgs a) {
  __shared__ float2 sm[16][kScoreRows], sm_row[kScoreRows];
  const int tid = threadIdx.x;
  const int32_t r = blockIdx.z, g = blockIdx.y, k0 = blockIdx.x * 1024;
  const WeightsRequest rq = weights_request(a, r);
  const int32_t M = rq.S * a.group, rows = a.max_q * a.group;
  float* const out = a.weights + r * a.w_row + g * a.w_head;
  // the blocks that any row sees
  const int64_t first = a.window > 0 ? max(rq.prior - a.window + 1, (int64_t)0) : 0;
  const int32_t keys = a.score_keys;
  const int32_t b0 = (int32_t)min(first / keys, (int64_t)a.blocks), b1 = (rq.n + keys - 1) / keys;
  if (k0 >= rq.n || M == 0 || (int64_t)k0 + 1023 < first) {  // uniform
    if (!a.add)
      for (int32_t k = k0 + tid; k < min(k0 + 1024, a.width); k += 256) out[k] = 0.0f;
    return;
  }
  {
    const int m = tid & (kScoreRows - 1), slice = tid / kScoreRows;
    float2 p = make_float2(kNegBig, 0.0f);
    if (m < M) {
      const float2* part = a.ws_part + ((int64_t)r * a.G + g) * a.blocks * rows + m;
#pragma unroll 4
      for (int32_t b = b0 + slice; b < b1; b += 16) p = weights_join(p, part[(int64_t)b * rows]);
    }
    sm[slice][m] = p;
    __syncthreads();
    if (tid < M) {
      for (int s = 1; s < 16; ++s) p = weights_join(p, sm[s][tid]);
      if (a.sinks) p = weights_join(p, make_float2(weights_sink(a, g * a.group + tid % a.group), 1.0f));
      sm_row[tid] = p.y == 0.0f ? make_float2(-kNegBig, 0.0f) : make_float2(p.x, 1.0f / p.y);
    }
    __syncthreads();
  }
  const int32_t key = k0 + 4 * tid;
  if (key >= a.width) return;
  float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (key >= (int64_t)b0 * keys && key < rq.n) {
    const int64_t width = (int64_t)a.blocks * keys;
    const float* src = a.ws_score + ((int64_t)r * a.G + g) * rows * width + key;
#pragma unroll 4
    for (int32_t m = 0; m < M; ++m) {
      const float4 x = *reinterpret_cast<const float4*>(src + m * width);
      const float2 rw = sm_row[m];
      w.x += weights_p(x.x, rw);
      w.y += weights_p(x.y, rw);
      w.z += weights_p(x.z, rw);
      w.w += weights_p(x.w, rw);
    }
  }
  const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (key + e >= a.width) break;
    if (!a.add) out[key + e] = v[e];
    else if (key + e < rq.n) out[key + e] += v[e];
  }
}

// Few rows whose scores fit LDS (FLOATS of them, with the row's page ids): one workgroup of 16 waves reads all of a (request,
// KV head)'s keys, straight to registers, 64 (or 32) to a wave at a time and the next ones on their way, keeps the scores in
// LDS, and turns them into the keys' weights there: one launch, every key read once and nothing else but the weights moved.
// Lanes as in weights_score_kernel.
constexpr int kRowThreads = 1024;
constexpr int kRowPad = 16;  // floats between two rows of scores, on top of their keys: 16 banks apart
template <int D, int ESZ, int FLOATS>
__global__ __launch_bounds__(kRowThreads) void weights_row_kernel(WeightsArgs a) {
  using Geo = WeightsGeo<D, ESZ>;
  constexpr int NS = D / 32, CK = score_chunk(Geo::ROWB), NT = CK / 16, NL = Geo::KCH / 4, WAVES = kRowThreads / 64;
  __shared__ __attribute__((aligned(16))) float sm[FLOATS];
  __shared__ float sm_wave[WAVES][kScoreRows];
  __shared__ float2 sm_row[kScoreRows];
  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, i16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t r = (int32_t)(blockIdx.x / a.G), g = (int32_t)(blockIdx.x % a.G);
  const WeightsRequest rq = weights_request(a, r);
  const int32_t M = rq.S * a.group, rows = a.max_q * a.group;
  float* const out = a.weights + r * a.w_row + g * a.w_head;
  // keys [lo, n): from the 64 that hold the first one that any row sees
  const int32_t lo = a.window > 0 ? (int32_t)min(max(rq.prior - a.window + 1, (int64_t)0), (int64_t)rq.n) & ~63 : 0;
  if (M == 0 || rq.n <= lo) {  // uniform
    if (!a.add)
      for (int32_t k = tid; k < a.width; k += kRowThreads) out[k] = 0.0f;
    return;
  }
  const int32_t cols = (rq.n - lo + 63) & ~63;
  float* const score = sm;  // [rows, pitch]
  const int32_t pitch = a.score_keys + kRowPad;
  int32_t* const page_of = reinterpret_cast<int32_t*>(sm + rows * pitch);  // of the pages from lo's on, -1 where invalid
  const int32_t c0 = lo / a.P;
  for (int32_t c = tid; c <= (rq.n - 1) / a.P - c0; c += kRowThreads) {
    const int32_t page = a.table[r * a.table_stride + c0 + c];
    page_of[c] = page >= 0 && page < a.num_blocks ? page : -1;
  }
  const int32_t m = i16, t = m / a.group, j = m - t * a.group;
  const uint16_t* const row = a.q + ((int64_t)(rq.qa + min(t, rq.S - 1)) * a.H + g * a.group + j) * D;
  uint32_t qf[NS][4];
#pragma unroll
  for (int c = 0; c < NS; ++c) {
    const uint4 w = ld16(row + 8 * (ESZ == 1 ? 8 * (c / 2) + 2 * g4 + (c & 1) : 4 * c + g4));
    qf[c][0] = w.x, qf[c][1] = w.y, qf[c][2] = w.z, qf[c][3] = w.w;
  }
  const float c2 = weights_scale<ESZ>(a, g);
  const uint64_t p_magic = ((1ull << 32) + a.P - 1) / a.P;  // key / P = key * magic >> 32: keys * P < 2^32 here
  __syncthreads();
  // (One copy of each step's code, none unrolled over the rows: a launch this short pays for every line of code it fetches.)
  uint4 cur[NT][NL], next[NT][NL];
  uint64_t valid = 0, valid_next = 0;
  float best = kNegBig;
  const int32_t end = lo + cols;
  for (int32_t kw = lo + (wave - WAVES) * CK; kw < end; kw += WAVES * CK) {  // (the first round only loads)
    const int32_t ahead = kw + WAVES * CK;
    if (ahead < end) {  // uniform: the wave's next keys to registers, and which of them are there
      valid_next = 0;
#pragma unroll
      for (int s = 0; s < NT; ++s) {
        const int32_t key = ahead + 16 * s + i16;
        const int32_t col = (int32_t)((uint32_t)key * p_magic >> 32);
        const int32_t page = key < rq.n ? page_of[col - c0] : -1;
        valid_next |= (uint64_t)(__ballot(page >= 0) & 0xffff) << 16 * s;
        // (a key that is not there reads the cache's first row: masked)
        const int64_t at = page < 0 ? 0 : (((int64_t)page * a.G + g) * a.P + (key - col * a.P)) * (int64_t)Geo::ROWB;
#pragma unroll
        for (int c = 0; c < NL; ++c) next[s][c] = ld16_stream(a.k_cache + at + 16 * (4 * c + g4));
      }
    }
    if (kw >= lo) {
      constexpr uint64_t kAll = CK == 64 ? ~0ull : (1ull << CK % 64) - 1;
      const bool all = valid == kAll && rq.prior >= kw + CK - 1 &&
                       (a.window <= 0 || rq.prior + rq.S - 1 - a.window < kw);  // uniform
      const uint64_t seen = all ? ~0ull : weights_seen(a, valid, rq.prior + t, kw) >> 4 * g4;
#pragma unroll
      for (int s = 0; s < NT; ++s) {
        f32x4_t x = {};
#pragma unroll
        for (int c = 0; c < NL; ++c) {
          const uint4 w = cur[s][c];
          if constexpr (ESZ == 1) {
            uint32_t ka[4], kb[4];
            fp8x4_to_bf16x4(w.x, ka[0], ka[1]);
            fp8x4_to_bf16x4(w.y, ka[2], ka[3]);
            fp8x4_to_bf16x4(w.z, kb[0], kb[1]);
            fp8x4_to_bf16x4(w.w, kb[2], kb[3]);
            x = mfma_16x16x32_bf16(ka, qf[2 * c], x);
            x = mfma_16x16x32_bf16(kb, qf[2 * c + 1], x);
          } else {
            const uint32_t ka[4] = {w.x, w.y, w.z, w.w};
            x = mfma_16x16x32_bf16(ka, qf[c], x);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = seen >> (16 * s + e) & 1 ? x[e] * c2 : -INFINITY;
          best = fmaxf(best, x[e]);
        }
        if (m < M) *reinterpret_cast<f32x4_t*>(score + m * pitch + (kw - lo) + 16 * s + 4 * g4) = x;
      }
    }
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
      for (int c = 0; c < NL; ++c) cur[s][c] = next[s][c];
    valid = valid_next;
  }
  best = max_across_groups(best);
  if (g4 == 0) sm_wave[wave][m] = best;
  __syncthreads();
  if (tid < M) {  // the rows' largest, and their sinks' share of the sum
    const float sink = a.sinks ? weights_sink(a, g * a.group + tid % a.group) : -INFINITY;
    float v = a.sinks ? sink : kNegBig;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v = fmaxf(v, sm_wave[w][tid]);
    sm_row[tid] = make_float2(v, __builtin_amdgcn_exp2f(sink - v));
  }
  __syncthreads();
  // Exponentials in place, four keys a thread, and the rows' sums.
#pragma unroll 1
  for (int i = 0; i < M; ++i) {
    const float top = sm_row[i].x;
    float sum = 0.0f;
#pragma unroll 1
    for (int32_t c = 4 * tid; c < cols; c += 4 * kRowThreads) {
      float4* const at = reinterpret_cast<float4*>(score + i * pitch + c);
      float4 x = *at;
      const float4 p = make_float4(__builtin_amdgcn_exp2f(x.x - top), __builtin_amdgcn_exp2f(x.y - top),
                                   __builtin_amdgcn_exp2f(x.z - top), __builtin_amdgcn_exp2f(x.w - top));
      sum += (p.x + p.y) + (p.z + p.w);
      // (an unseen key's is kept as -1: it adds nothing, whatever the row's sum is)
      x.x = x.x == -INFINITY ? -1.0f : p.x, x.y = x.y == -INFINITY ? -1.0f : p.y;
      x.z = x.z == -INFINITY ? -1.0f : p.z, x.w = x.w == -INFINITY ? -1.0f : p.w;
      *at = x;
    }
    sum = wave_sum(sum);
    if (lane == 0) sm_wave[wave][i] = sum;
  }
  __syncthreads();
  if (tid < M) {
    float v = sm_row[tid].y;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += sm_wave[w][tid];
    sm_row[tid].y = v == 0.0f ? 0.0f : 1.0f / v;
  }
  __syncthreads();
#pragma unroll 1
  for (int32_t c = 4 * tid; c < cols; c += 4 * kRowThreads) {
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int i = 0; i < M; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(score + i * pitch + c);
      const float inv = sm_row[i].y;
      w[0] += x.x < 0.0f ? 0.0f : x.x * inv, w[1] += x.y < 0.0f ? 0.0f : x.y * inv;
      w[2] += x.z < 0.0f ? 0.0f : x.z * inv, w[3] += x.w < 0.0f ? 0.0f : x.w * inv;
    }
    const int32_t key = lo + c;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (key + e < min(rq.n, a.width)) out[key + e] = a.add ? out[key + e] + w[e] : w[e];
  }
  if (!a.add) {
    for (int32_t k = tid; k < min(lo, a.width); k += kRowThreads) out[k] = 0.0f;
    for (int32_t k = rq.n + tid; k < a.width; k += kRowThreads) out[k] = 0.0f;
  }
}

}  // namespace sna

using namespace sna;

namespace {

constexpr int64_t kGridMax = (1 << 24) - 1;  // workgroups of 256 threads: 32 bits number a launch's threads

int64_t weights_blocks(int32_t page_size, int32_t table_width, int32_t width, int32_t keys) {
  return (std::max<int64_t>((int64_t)table_width * page_size, width) + keys - 1) / keys;
}

// How a launch works, and its workspace: few rows a request keep their scores while these take 512 MB at most, others
// compute them twice.
constexpr int64_t kScoreBytes = (int64_t)1 << 29;
struct WeightsPlan {
  int64_t blocks, part, rest, bytes;
  int32_t splits, split_tokens, span, score_keys;
  bool scores;
  int32_t row_floats;  // the LDS of weights_row_kernel where that serves, else 0
};
// weights_row_kernel serves where the scores fit LDS, the (request, KV head) pairs leave at most a quarter of its
// workgroups' places on the chip empty, and the tables are long enough that a workgroup of 16 waves is worth starting.
// Against two launches (us, heads 32/8 of 128, e4m3fn, all keys full): 256 pairs of 2048 keys 21.8 : 24.5, 512 of 8192
// 132 : 156, 256 of 4096 with heads 8/1 of 64 21 : 29; without these bounds 264 pairs of 4096 would take 60 : 46 (the last
// 8 a second turn), 1024 of 100 to 1024 bf16 keys 58 : 47 and 64 of 2048 13 : 9 (a CU alone reads 256 KB in 8 us).
constexpr int64_t kRowPairs = 256, kRowKeys = 2048;  // the CUs, and the least keys of a table
constexpr int32_t kRowFloats[2] = {18432, 36864};    // LDS of two workgroups a CU, or one
constexpr int64_t kScoreWorkgroups = 1024;  // a score launch has so many at least before one takes several chunks
// Queries are cut into runs of at least so many rows while that makes no more than so many workgroups: by 4 tiles up to two
// rounds of the 3 workgroups that a CU holds, by 8 up to ten a CU. One run each: 635 queries of 8 heads over 2270 keys 100 us
// (29 cut), 300 of a window of 128 86 (39), 1024 of 32 heads over 8192 keys 327 (295), 4 x 2048 over 4096 keys 497 (479).
constexpr int64_t kRunRows[2] = {128, 256}, kRunWorkgroups[2] = {1536, 2560};
WeightsPlan weights_plan(int64_t T, int64_t R, int64_t max_q, int32_t H, int32_t G, int32_t page_size,
                         int32_t table_width, int32_t width, int32_t head_dim, int32_t esz, int32_t window) {
  WeightsPlan p;
  p.score_keys = 0;
  p.row_floats = 0;
  p.splits = 1, p.split_tokens = (int32_t)max_q;
  const int64_t table_keys = ((int64_t)table_width * page_size + 63) / 64 * 64;
  const int64_t group = H / G, rows = max_q * group, pairs = R * G;
  if (rows <= kScoreRows && table_keys >= kRowKeys && rows * (table_keys + kRowPad) + table_width <= kRowFloats[1]) {
    const bool half = rows * (table_keys + kRowPad) + table_width <= kRowFloats[0];
    const int64_t slots = half ? 2 * kRowPairs : kRowPairs, turns = (pairs + slots - 1) / slots;
    if (pairs >= kRowPairs && (turns == 1 || 4 * pairs >= 3 * turns * slots)) {
      p.row_floats = kRowFloats[half ? 0 : 1];
      p.blocks = 1, p.span = 1, p.part = p.rest = p.bytes = 0, p.scores = false;
      p.score_keys = (int32_t)table_keys;
      return p;
    }
  }
  p.blocks = weights_blocks(page_size, table_width, width, kWeightKeys);
  p.span = 1;
  int64_t score = INT64_MAX;
  if (rows <= kScoreRows) {
    const int32_t chunk = 4 * score_chunk(head_dim * esz);
    const int64_t chunks = weights_blocks(page_size, table_width, 0, chunk);
    p.span = (int32_t)std::min<int64_t>(score_span(head_dim * esz), std::max<int64_t>(1, chunks * R * G / kScoreWorkgroups));
    p.score_keys = chunk * p.span;
    const int64_t blocks = (chunks + p.span - 1) / p.span;
    score = R * G * rows * blocks * p.score_keys * (int64_t)sizeof(float);
    if (score <= kScoreBytes) p.blocks = blocks;
  }
  p.scores = score <= kScoreBytes;
  p.part = (p.scores ? R * G * rows : T * H) * p.blocks * (int64_t)sizeof(float2);
  p.rest = p.scores ? score : T * H * (int64_t)sizeof(float2);
  int64_t sum = 0;
  if (!p.scores) {
    // the tokens that can see one block, from a multiple of 32 on, and the blocks that any can see
    const int64_t most_tokens = window > 0 ? std::min<int64_t>(max_q, (int64_t)kWeightKeys + window + 31) : max_q;
    const int64_t seen = window > 0 ? std::min<int64_t>(p.blocks, (max_q + window) / kWeightKeys + 2) : p.blocks;
    auto runs = [&](int64_t fewest, int64_t workgroups) {
      const int64_t least = ((fewest + group - 1) / group + kWeightRows - 1) / kWeightRows * kWeightRows;
      return std::min((most_tokens + least - 1) / least, workgroups / (seen * R * G));
    };
    const int64_t most = std::max<int64_t>({1, runs(kRunRows[0], kRunWorkgroups[0]), runs(kRunRows[1], kRunWorkgroups[1])});
    p.split_tokens = (int32_t)(((most_tokens + most - 1) / most + kWeightRows - 1) / kWeightRows * kWeightRows);
    p.splits = (int32_t)((most_tokens + p.split_tokens - 1) / p.split_tokens);
    if (p.splits > 1) sum = p.splits * R * G * p.blocks * kWeightKeys * (int64_t)sizeof(float);
  }
  p.part = (p.part + 15) / 16 * 16;
  p.rest = (p.rest + 15) / 16 * 16;
  p.bytes = p.part + p.rest + sum;
  return p;
}

// Up to so many rows (of all requests and KV heads) are merged 8 to a workgroup, a row's blocks by 32 threads, else 32 and by
// 8. In us by 8 / 32, rows of 512 blocks: 2048 rows 5.8 / 10.2, 4096 8.4 / 10.8, 6144 11.2 / 11.2, 8192 13.5 / 11.3, 16384
// 23 / 15; of 64 blocks 4 to 5 both up to 6144 rows, 16384 6.1 / 5.2, 65536 13.7 / 7.4; of 8 blocks 4 to 5 both up to 16384,
// 32768 6.9 / 5.2.
constexpr int64_t kMergeFewRows = 6144;
template <int D, int ESZ>
void launch_weights(const WeightsArgs& a, uint32_t wgs, int32_t row_floats, hipStream_t s) {
  if (row_floats > 0) {
    if (row_floats == kRowFloats[0])
      hipLaunchKernelGGL((weights_row_kernel<D, ESZ, kRowFloats[0]>), dim3(a.R * a.G), dim3(kRowThreads), 0, s, a);
    else
      hipLaunchKernelGGL((weights_row_kernel<D, ESZ, kRowFloats[1]>), dim3(a.R * a.G), dim3(kRowThreads), 0, s, a);
    return;
  }
  if (a.ws_score) {
    hipLaunchKernelGGL((weights_score_kernel<D, ESZ>), dim3(wgs), dim3(256), 0, s, a);
    const int64_t cols = a.add ? (int64_t)a.blocks * a.score_keys : a.width;  // (every column is written, or the keys')
    hipLaunchKernelGGL(weights_from_scores_kernel, dim3((unsigned)((cols + 1023) / 1024), a.G, a.R), dim3(256), 0, s, a);
    return;
  }
  hipLaunchKernelGGL((weights_tile_kernel<D, ESZ, kStats>), dim3(wgs), dim3(256), 0, s, a);
  const int64_t rows = (int64_t)a.max_q * a.group;
  if (rows * a.G * a.R <= kMergeFewRows)
    hipLaunchKernelGGL((weights_merge_kernel<8>), dim3((unsigned)((rows + 7) / 8), a.G, a.R), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((weights_merge_kernel<32>), dim3((unsigned)((rows + 31) / 32), a.G, a.R), dim3(256), 0, s, a);
  hipLaunchKernelGGL((weights_tile_kernel<D, ESZ, kSum>), dim3(wgs), dim3(256), 0, s, a);
  if (a.splits > 1)
    hipLaunchKernelGGL(weights_reduce_kernel, dim3((unsigned)((a.width + 255) / 256), a.G, a.R), dim3(256), 0, s, a);
}

int attention_weights(const char* what, const void* q, const void* k_cache, const float* k_scale,
                      const int32_t* block_table, int64_t table_stride, int32_t table_width, const int32_t* q_start,
                      const int32_t* lens, int32_t T, int32_t R, int32_t max_q_len, const float* sinks, float sm_scale,
                      int32_t window, float* weights, int64_t row_stride, int64_t head_stride, int32_t width,
                      int32_t accumulate, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                      int32_t page_size, int64_t num_blocks, int32_t kv_dtype, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  if (T < 0 || R < 0 || max_q_len < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads != 0 ||
      window < 0 || num_blocks < 1 || table_width < 1 || table_stride < table_width || width < 0 || page_size < 1)
    return fail(SNA_ERR_INVALID_ARGUMENT,
                "%s: bad sizes (tokens %d, R %d, max_q_len %d, heads %d / %d, window %d, blocks %lld, table %d wide, "
                "stride %lld, width %d, page %d)", what, T, R, max_q_len, num_q_heads, num_kv_heads, window,
                (long long)num_blocks, table_width, (long long)table_stride, width, page_size);
  max_q_len = std::max(std::min(max_q_len, T), 1);
  const int32_t group = num_q_heads / num_kv_heads;
  if (head_dim != 64 && head_dim != 128)
    return fail(SNA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  if (group > 128) return fail(SNA_ERR_UNSUPPORTED, "%s: %d query heads per KV head (at most 128)", what, group);
  if (kv_dtype != SNA_DTYPE_FP8_E4M3FN && kv_dtype != SNA_DTYPE_FP8_E4M3FN_MUL && kv_dtype != SNA_DTYPE_BF16)
    return fail(SNA_ERR_UNSUPPORTED, "%s: KV dtype %d (FP8 e4m3fn or bf16)", what, kv_dtype);
  if ((int64_t)table_width * page_size > INT32_MAX - (1 << 16) || width > INT32_MAX - (1 << 16))
    return fail(SNA_ERR_UNSUPPORTED, "%s: a table of %d pages of %d, a width of %d (under 2^31 keys)", what, table_width,
                page_size, width);
  if (R == 0 || width == 0) return SNA_OK;
  if ((T > 0 && !q) || !k_cache || (kv_dtype != SNA_DTYPE_BF16 && !k_scale) || !block_table || !lens || !weights)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(weights, 4))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: q and the cache must be 16-byte aligned", what);
  if (R > 65535 || num_kv_heads > 65535)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d requests x %d KV heads exceed the grid", what, R, num_kv_heads);
  if ((int64_t)T * group > INT32_MAX - kWeightRows)
    return fail(SNA_ERR_UNSUPPORTED, "%s: %d tokens of %d heads a KV head (split the batch)", what, T, group);
  if ((int64_t)max_q_len * group * group > (int64_t)1 << 32)  // (the kernels' row / group is exact up to there)
    return fail(SNA_ERR_UNSUPPORTED, "%s: chunks of up to %d tokens of %d heads a KV head (split them)", what, max_q_len,
                group);
  if (head_stride < width || row_stride < width)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: weight strides %lld / %lld for %d columns", what, (long long)row_stride,
                (long long)head_stride, width);
  if (((int64_t)max_q_len * group + kWeightRows - 1) / kWeightRows > kGridMax)
    return fail(SNA_ERR_UNSUPPORTED, "%s: chunks of up to %d tokens of %d heads a KV head exceed the grid (split them)",
                what, max_q_len, group);
  const WeightsPlan plan = weights_plan(T, R, max_q_len, num_q_heads, num_kv_heads, page_size, table_width, width,
                                        head_dim, kv_dtype == SNA_DTYPE_BF16 ? 2 : 1, window);
  const int64_t blocks = plan.blocks;
  const int64_t wgs = blocks * R * num_kv_heads * plan.splits;
  if (wgs > kGridMax / 4)
    return fail(SNA_ERR_UNSUPPORTED, "%s: %lld key blocks x %d requests x %d KV heads exceed the grid (split the batch)",
                what, (long long)blocks, R, num_kv_heads);
  const int64_t need = plan.bytes;
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(SNA_ERR_WORKSPACE, "%s: workspace of %lld bytes, need %lld", what, (long long)workspace_bytes,
                (long long)need);
  if (!aligned(workspace, 16)) return fail(SNA_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
  WeightsArgs a;
  a.q = (const uint16_t*)q;
  a.k_cache = (const uint8_t*)k_cache;
  a.k_scale = k_scale;
  a.mul_scale = kv_dtype == SNA_DTYPE_FP8_E4M3FN_MUL;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.q_start = q_start;
  a.lens = lens;
  a.sinks = sinks;
  a.weights = weights;
  a.w_row = row_stride;
  a.w_head = head_stride;
  a.width = width;
  a.add = accumulate != 0;
  a.T = T;
  a.R = R;
  a.H = num_q_heads;
  a.G = num_kv_heads;
  a.P = page_size;
  a.group = group;
  a.magic = ((1ull << 32) + group - 1) / group;
  a.max_q = max_q_len;
  a.num_blocks = num_blocks;
  a.sm_scale = sm_scale;
  a.window = window;
  a.blocks = (int32_t)blocks;
  a.ws_part = (float2*)workspace;
  a.ws_row = plan.scores ? nullptr : (float2*)((uint8_t*)workspace + plan.part);
  a.splits = plan.splits;
  a.split_tokens = plan.split_tokens;
  a.span = plan.span;
  a.score_keys = plan.score_keys;
  a.ws_sum = (float*)((uint8_t*)workspace + plan.part + plan.rest);
  a.ws_score = plan.scores ? (float*)((uint8_t*)workspace + plan.part) : nullptr;
  const hipStream_t s = (hipStream_t)stream;
  if (kv_dtype != SNA_DTYPE_BF16) {
    if (head_dim == 128) launch_weights<128, 1>(a, (uint32_t)wgs, plan.row_floats, s);
    else launch_weights<64, 1>(a, (uint32_t)wgs, plan.row_floats, s);
  } else {
    if (head_dim == 128) launch_weights<128, 2>(a, (uint32_t)wgs, plan.row_floats, s);
    else launch_weights<64, 2>(a, (uint32_t)wgs, plan.row_floats, s);
  }
  return check_launch(what);
}

}  // namespace

extern "C" int64_t sna_attention_weights_workspace_bytes(int32_t n_tokens, int32_t R, int32_t max_q_len,
                                                         int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                         int32_t page_size, int32_t table_width, int32_t width,
                                                         int32_t kv_dtype, int32_t window) {
  if (n_tokens < 0 || R < 1 || max_q_len < 0 || num_q_heads < 1 || num_kv_heads < 1 ||
      num_q_heads % num_kv_heads != 0 || page_size < 1 || table_width < 1 || width < 0)
    return 0;
  return weights_plan(n_tokens, R, std::max(std::min(max_q_len, n_tokens), 1), num_q_heads, num_kv_heads, page_size,
                      table_width, width, head_dim, kv_dtype == SNA_DTYPE_BF16 ? 2 : 1, window).bytes;
}

extern "C" int sna_prefill_attention_weights(const void* q, const void* k_cache, const float* k_scale,
                                             const int32_t* block_table, int64_t table_stride, int32_t table_width,
                                             const int32_t* q_start, const int32_t* prior_lens, int32_t n_tokens,
                                             int32_t R, int32_t max_q_len, const float* sinks, float sm_scale,
                                             int32_t window, float* weights, int64_t row_stride, int64_t head_stride,
                                             int32_t width, int32_t accumulate, int32_t num_q_heads,
                                             int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                             int64_t num_blocks, int32_t kv_dtype, void* workspace,
                                             int64_t workspace_bytes, void* stream) {
  ApiGuard guard;
  if (R > 0 && !q_start) return fail(SNA_ERR_INVALID_ARGUMENT, "prefill_attention_weights: null pointer");
  return attention_weights("prefill_attention_weights", q, k_cache, k_scale, block_table, table_stride, table_width,
                           q_start, prior_lens, n_tokens, R, max_q_len, sinks, sm_scale, window, weights, row_stride,
                           head_stride, width, accumulate, num_q_heads, num_kv_heads, head_dim, page_size, num_blocks,
                           kv_dtype, workspace, workspace_bytes, stream);
}

extern "C" int sna_decode_attention_weights(const void* q, const void* k_cache, const float* k_scale,
                                            const int32_t* block_table, int64_t table_stride, int32_t table_width,
                                            const int32_t* seq_lens, int32_t B, const float* sinks, float sm_scale,
                                            int32_t window, float* weights, int64_t row_stride, int64_t head_stride,
                                            int32_t width, int32_t accumulate, int32_t num_q_heads,
                                            int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                            int64_t num_blocks, int32_t kv_dtype, void* workspace,
                                            int64_t workspace_bytes, void* stream) {
  ApiGuard guard;
  return attention_weights("decode_attention_weights", q, k_cache, k_scale, block_table, table_stride, table_width,
                           nullptr, seq_lens, B, B, 1, sinks, sm_scale, window, weights, row_stride, head_stride,
                           width, accumulate, num_q_heads, num_kv_heads, head_dim, page_size, num_blocks, kv_dtype,
                           workspace, workspace_bytes, stream);
}
