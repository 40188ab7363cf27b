// The attention weight that each cached key of a GQA layer receives: for request r, KV head g and key j
//   W[r, g, j] (+)= sum over the request's queries i and the group's heads h of p(i, h, j),
//   p(i, h, j) = exp(s(i, h, j)) / (sum over the keys that i sees of exp(s(i, h, .)) + exp(sink_h)),
// s = sm_scale * q . k with K read from the paged pool (bf16, or e4m3fn with per-KV-head scales). A query at position p
// sees the keys (p - window, p] (all up to p without a window) that lie on valid pages; a query that sees none adds
// nothing. It is what an eviction by accumulated weight ranks the keys by.
//
// A probability needs its row's sum over all keys before it can be added to its key's, so the scores are computed twice:
//   weights_tile_kernel<STATS>  per block of 256 keys and query row: the largest score and the sum of exp(score - largest)
//   weights_merge_kernel        per query row: the blocks merged to the row's largest score and 1 / its whole sum
//   weights_tile_kernel<SUM>    per key: the probabilities summed over the rows
// Rows are (query token, head) pairs of one KV head, token-major (row = t * group + j). A workgroup of 4 waves owns 256
// keys of one (request, KV head), 64 to a wave, held as bf16 matrix operands in registers (an e4m3fn value is a bf16
// value); the rows pass in tiles of 32 through a 2-slot LDS ring that the waves share. The product is S^T[key, row] =
// K[key, :] . Q[row, :] by v_mfma_f32_32x32x16_bf16, so a lane holds 16 keys of one row: the row's maximum, sum and
// normalization are values of the lane, and a key's sum over the rows stays in the lane's registers until the end.
// Scores are fp32, exponentials in the log2 domain, every sum fp32; a key's rows are added in a fixed order.
#include <algorithm>

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
  int64_t num_blocks;
  float sm_scale;
  int32_t window;
  int32_t blocks;    // key blocks that the table's keys (and, when every column is written, the width) take
  float2* ws_part;   // [G, blocks, T * group] a block's (largest score in the log2 domain, sum)
  float2* ws_row;    // [G, T * group] a row's (largest score in the log2 domain, 1 / sum)
};

constexpr int kWeightKeys = 256;  // keys of a workgroup
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

enum WeightsPass { kStats, kSum };
template <int D, int ESZ, WeightsPass PASS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void weights_tile_kernel(WeightsArgs a) {
  constexpr bool FP8 = ESZ == 1;
  constexpr int NS = D / 16;          // matrix steps of a score
  constexpr int CH = D * 2 / 16;      // 16-byte chunks of a query row
  constexpr int TILE = kWeightRows * CH;
  constexpr int LD = TILE / 256;      // chunks of a tile that a thread moves
  __shared__ uint4 sm_q[2][TILE];
  __shared__ int64_t sm_key[kWeightKeys];  // a key's first byte in the cache, -1 where there is none
  __shared__ float sm_out[kWeightKeys];
  __shared__ float2 sm_part[2][4][kWeightRows];
  const int tid = threadIdx.x, lane = tid & 63, g2 = lane >> 5, i32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lin = xcd_order(blockIdx.x, gridDim.x);
  const int32_t kb = (int32_t)(lin % a.blocks), r = (int32_t)(lin / a.blocks % a.R), g = (int32_t)(lin / a.blocks / a.R);
  const WeightsRequest rq = weights_request(a, r);
  const int32_t k0 = kb * kWeightKeys;
  // the rows that see any of the block's keys: tokens [t0, t1)
  const int64_t last = (int64_t)min(k0 + kWeightKeys, rq.n) - 1;
  int32_t t0 = (int32_t)min(max(k0 - rq.prior, (int64_t)0), (int64_t)rq.S), t1 = rq.S;
  if (a.window > 0) t1 = (int32_t)min(max(last + a.window - rq.prior, (int64_t)0), (int64_t)rq.S);
  if (k0 >= rq.n) t1 = t0;
  float* const out = a.weights + r * a.w_row + g * a.w_head;
  if (t1 <= t0) {  // uniform
    if (PASS == kSum && !a.add && k0 + tid < a.width) out[k0 + tid] = 0.0f;
    return;
  }
  {
    const int32_t key = k0 + tid;
    int64_t at = -1;
    if (key < rq.n) {
      const int32_t col = key / a.P;
      const int64_t page = a.table[r * a.table_stride + col];
      if (page >= 0 && page < a.num_blocks) at = ((page * a.G + g) * a.P + (key - col * a.P)) * (int64_t)(D * ESZ);
    }
    sm_key[tid] = at;
  }
  const int32_t m_end = t1 * a.group;
  const int32_t m0 = (t0 * a.group) & ~(kWeightRows - 1);
  const int32_t tiles = (m_end - m0 + kWeightRows - 1) / kWeightRows;
  // this thread's chunks of a tile: row (tid + 256 l) / CH, chunk (tid + 256 l) % CH; the row's token and head move on by
  // 32 rows a tile
  const int32_t step_t = kWeightRows / a.group, step_j = kWeightRows - step_t * a.group;
  int32_t ld_t[LD], ld_j[LD];
  uint4 ld[LD];
#pragma unroll
  for (int l = 0; l < LD; ++l) {
    const int32_t m = m0 + (tid + 256 * l) / CH;
    ld_t[l] = m / a.group, ld_j[l] = m - ld_t[l] * a.group;
  }
  auto load = [&]() {
#pragma unroll
    for (int l = 0; l < LD; ++l) {
      ld[l] = make_uint4(0, 0, 0, 0);
      if (ld_t[l] < t1)
        ld[l] = ld16(a.q + ((int64_t)(rq.qa + ld_t[l]) * a.H + g * a.group + ld_j[l]) * D + 8 * (tid % CH));
      ld_t[l] += step_t, ld_j[l] += step_j;
      if (ld_j[l] >= a.group) ld_j[l] -= a.group, ++ld_t[l];
    }
  };
  load();
  __syncthreads();
  // the wave's keys as A operands: lane (g2, i) feeds key 32 s + i
  uint32_t kf[2][NS][4];
  uint64_t valid = 0;  // bit i: key 64 wave + i is there
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int64_t at = sm_key[64 * wave + 32 * s + i32];
    valid |= (__ballot(at >= 0) & 0xffffffffull) << (32 * s);
    const uint8_t* row = a.k_cache + at;
    if constexpr (FP8) {
#pragma unroll
      for (int c = 0; c < NS / 2; ++c) {
        const uint4 w = at >= 0 ? ld16(row + 32 * c + 16 * g2) : make_uint4(0, 0, 0, 0);
        fp8x4_to_bf16x4(w.x, kf[s][2 * c][0], kf[s][2 * c][1]);
        fp8x4_to_bf16x4(w.y, kf[s][2 * c][2], kf[s][2 * c][3]);
        fp8x4_to_bf16x4(w.z, kf[s][2 * c + 1][0], kf[s][2 * c + 1][1]);
        fp8x4_to_bf16x4(w.w, kf[s][2 * c + 1][2], kf[s][2 * c + 1][3]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NS; ++c) {
        const uint4 w = at >= 0 ? ld16(row + 32 * c + 16 * g2) : make_uint4(0, 0, 0, 0);
        kf[s][c][0] = w.x, kf[s][c][1] = w.y, kf[s][c][2] = w.z, kf[s][c][3] = w.w;
      }
    }
  }
  double scale = (double)a.sm_scale * 1.4426950408889634;
  if (FP8) scale = a.mul_scale ? scale / (double)a.k_scale[g] : scale * (double)a.k_scale[g];
  const float c2 = (float)scale;
  const int64_t rows = (int64_t)a.T * a.group;  // rows of a KV head
  float2* const part = a.ws_part + ((int64_t)g * a.blocks + kb) * rows + (int64_t)rq.qa * a.group;
  const float2* const row_of = a.ws_row + (int64_t)g * rows + (int64_t)rq.qa * a.group;
  const int32_t kw = k0 + 64 * wave;  // the wave's first key
  float acc[2][16];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[s][e] = 0.0f;

  for (int32_t i = 0; i < tiles; ++i) {
    uint4* const slot = sm_q[i & 1];
#pragma unroll
    for (int l = 0; l < LD; ++l) {
      const int row = (tid + 256 * l) / CH, ch = tid % CH;
      slot[row * CH + (ch ^ (row & (CH - 1)))] = ld[l];
    }
    __syncthreads();  // the slot was read two tiles ago: the barrier between covers it
    if (i + 1 < tiles) load();
    const int32_t m = m0 + kWeightRows * i + i32;  // this lane's row
    float2 rw = make_float2(0.0f, 0.0f);
    if (PASS == kSum && m < m_end) rw = row_of[m];
    const int32_t t = m / a.group;
    const int64_t pos = rq.prior + t;
    f32x16_t x[2] = {};
#pragma unroll
    for (int c = 0; c < NS; ++c) {
      // chunk of 8 dims that the lane's K operand of step c holds
      const int ch = FP8 ? 4 * (c / 2) + 2 * g2 + (c & 1) : 2 * c + g2;
      const uint4 w = slot[i32 * CH + (ch ^ (i32 & (CH - 1)))];
      const uint32_t qf[4] = {w.x, w.y, w.z, w.w};
      x[0] = mfma_32x32x16_bf16(kf[0][c], qf, x[0]);
      x[1] = mfma_32x32x16_bf16(kf[1][c], qf, x[1]);
    }
    // the keys that the lane's row sees, of the wave's 64
    uint64_t seen = valid;
    {
      const int64_t hi = pos - kw;  // keys 0 .. hi of the wave
      seen = m >= m_end || hi < 0 ? 0 : hi < 63 ? seen & ((2ull << hi) - 1) : seen;
      if (a.window > 0) {
        const int64_t lo = pos - a.window + 1 - kw;  // from key lo
        seen = lo > 63 ? 0 : lo > 0 ? seen & (~0ull << lo) : seen;
      }
    }
    const bool all = __all(seen == ~0ull);
    if constexpr (PASS == kStats) {
      float mx = kNegBig, sum = 0.0f;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool on = all || (seen >> (32 * s + 8 * (e / 4) + 4 * g2 + e % 4) & 1);
          x[s][e] = on ? x[s][e] * c2 : -INFINITY;
          mx = fmaxf(mx, x[s][e]);
        }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f(x[s][e] - mx);
      // the row's other keys of the wave are the lane 32 away
      const float om = __shfl_xor(mx, 32, 64), os = __shfl_xor(sum, 32, 64);
      const float bm = fmaxf(mx, om);
      sum = sum * __builtin_amdgcn_exp2f(mx - bm) + os * __builtin_amdgcn_exp2f(om - bm);
      if (g2 == 0) sm_part[i & 1][wave][i32] = make_float2(bm, sum);
      __syncthreads();
      if (tid < kWeightRows && m0 + kWeightRows * i + tid < m_end) {
        float2 p = sm_part[i & 1][0][tid];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float2 o = sm_part[i & 1][w][tid];
          const float b = fmaxf(p.x, o.x);
          p.y = p.y * __builtin_amdgcn_exp2f(p.x - b) + o.y * __builtin_amdgcn_exp2f(o.x - b);
          p.x = b;
        }
        part[m0 + kWeightRows * i + tid] = p;
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool on = all || (seen >> (32 * s + 8 * (e / 4) + 4 * g2 + e % 4) & 1);
          const float p = __builtin_amdgcn_exp2f(x[s][e] * c2 - rw.x) * rw.y;
          acc[s][e] += on ? p : 0.0f;
        }
    }
  }
  if constexpr (PASS == kSum) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float v = acc[s][e];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
        if (i32 == 0) sm_out[64 * wave + 32 * s + 8 * (e / 4) + 4 * g2 + e % 4] = v;
      }
    __syncthreads();
    const int32_t key = k0 + tid;
    if (key < a.width) {
      const float v = sm_key[tid] >= 0 ? sm_out[tid] : 0.0f;
      if (!a.add) out[key] = v;
      else if (sm_key[tid] >= 0) out[key] += v;
    }
  }
}

// A row's blocks merged: (its largest score M in the log2 domain, 1 / sum of 2^(score - M) with the sink's).
__global__ __launch_bounds__(256) void weights_merge_kernel(WeightsArgs a) {
  const int32_t r = blockIdx.z, g = blockIdx.y;
  const WeightsRequest rq = weights_request(a, r);
  const int32_t m = blockIdx.x * 256 + threadIdx.x;
  if (m >= rq.S * a.group) return;
  const int32_t t = m / a.group, h = g * a.group + m - t * a.group;
  const int64_t pos = rq.prior + t;
  const int64_t rows = (int64_t)a.T * a.group;
  const int64_t row = (int64_t)rq.qa * a.group + m;
  // the blocks that hold keys it sees: each has written this row
  const int64_t hi = min(pos, (int64_t)rq.n - 1), lo = a.window > 0 ? max(pos - a.window + 1, (int64_t)0) : 0;
  float M = kNegBig, S = 0.0f;
  if (a.sinks) M = a.sinks[h] * kLog2e, S = 1.0f;
  for (int32_t b = (int32_t)(lo / kWeightKeys); hi >= lo && b <= hi / kWeightKeys; ++b) {
    const float2 p = a.ws_part[((int64_t)g * a.blocks + b) * rows + row];
    const float n = fmaxf(M, p.x);
    S = S * __builtin_amdgcn_exp2f(M - n) + p.y * __builtin_amdgcn_exp2f(p.x - n);
    M = n;
  }
  a.ws_row[(int64_t)g * rows + row] = make_float2(M, S == 0.0f ? 0.0f : 1.0f / S);
}

}  // namespace sna

using namespace sna;

namespace {

constexpr int64_t kGridMax = (1 << 24) - 1;  // workgroups of 256 threads: 32 bits number a launch's threads

int64_t weights_blocks(int32_t page_size, int32_t table_width, int32_t width) {
  const int64_t keys = std::max<int64_t>((int64_t)table_width * page_size, width);
  return (keys + kWeightKeys - 1) / kWeightKeys;
}

int64_t weights_bytes(int64_t T, int32_t H, int64_t blocks) { return (blocks + 1) * T * H * (int64_t)sizeof(float2); }

template <int D, int ESZ>
void launch_weights(const WeightsArgs& a, uint32_t wgs, hipStream_t s) {
  hipLaunchKernelGGL((weights_tile_kernel<D, ESZ, kStats>), dim3(wgs), dim3(256), 0, s, a);
  hipLaunchKernelGGL(weights_merge_kernel, dim3((unsigned)(((int64_t)a.max_q * a.group + 255) / 256), a.G, a.R), dim3(256),
                     0, s, a);
  hipLaunchKernelGGL((weights_tile_kernel<D, ESZ, kSum>), dim3(wgs), dim3(256), 0, s, a);
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
  const int32_t group = num_q_heads / num_kv_heads;
  if (head_dim != 64 && head_dim != 128)
    return fail(SNA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  if (group > 128) return fail(SNA_ERR_UNSUPPORTED, "%s: %d query heads per KV head (at most 128)", what, group);
  if (kv_dtype != SNA_DTYPE_FP8_E4M3FN && kv_dtype != SNA_DTYPE_FP8_E4M3FN_MUL && kv_dtype != SNA_DTYPE_BF16)
    return fail(SNA_ERR_UNSUPPORTED, "%s: KV dtype %d (FP8 e4m3fn or bf16)", what, kv_dtype);
  if ((int64_t)table_width * page_size > INT32_MAX - kWeightKeys || width > INT32_MAX - kWeightKeys)
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
  if (head_stride < width || row_stride < width)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: weight strides %lld / %lld for %d columns", what, (long long)row_stride,
                (long long)head_stride, width);
  const int64_t blocks = weights_blocks(page_size, table_width, width);
  const int64_t wgs = blocks * R * num_kv_heads;
  if (wgs > kGridMax)
    return fail(SNA_ERR_UNSUPPORTED, "%s: %lld key blocks x %d requests x %d KV heads exceed the grid (split the batch)",
                what, (long long)blocks, R, num_kv_heads);
  const int64_t need = weights_bytes(T, num_q_heads, blocks);
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
  a.max_q = std::max(max_q_len, 1);
  a.num_blocks = num_blocks;
  a.sm_scale = sm_scale;
  a.window = window;
  a.blocks = (int32_t)blocks;
  a.ws_row = (float2*)workspace;
  a.ws_part = a.ws_row + (int64_t)T * num_q_heads;
  const hipStream_t s = (hipStream_t)stream;
  if (kv_dtype != SNA_DTYPE_BF16) {
    if (head_dim == 128) launch_weights<128, 1>(a, (uint32_t)wgs, s); else launch_weights<64, 1>(a, (uint32_t)wgs, s);
  } else {
    if (head_dim == 128) launch_weights<128, 2>(a, (uint32_t)wgs, s); else launch_weights<64, 2>(a, (uint32_t)wgs, s);
  }
  return check_launch(what);
}

}  // namespace

extern "C" int64_t sna_attention_weights_workspace_bytes(int32_t n_tokens, int32_t R, int32_t max_q_len,
                                                         int32_t num_q_heads, int32_t num_kv_heads, int32_t page_size,
                                                         int32_t table_width, int32_t width) {
  if (n_tokens < 1 || R < 1 || max_q_len < 1 || num_q_heads < 1 || num_kv_heads < 1 ||
      num_q_heads % num_kv_heads != 0 || page_size < 1 || table_width < 1 || width < 0)
    return 0;
  return weights_bytes(n_tokens, num_q_heads, weights_blocks(page_size, table_width, width));
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
