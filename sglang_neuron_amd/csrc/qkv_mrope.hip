// The QKV writer for rotary positions with several axes (time, height, width of images and video): per-head RMSNorm of Q
// and K (optional), the rotation of pair i (elements i and i + rot / 2 of a head's first rot) by the angle
//   positions[axis(i), t] * inv_freq[i],
// Q written out and K / V stored into the paged MHA pool (bf16, or e4m3fn with per-KV-head scales), in one pass over the
// projection's output.
//
// Angles are formed in turns (position * (inv_freq / 2 pi), less its whole part) in 64 bits, far ones in twice as many, so
// every int64 position keeps the fraction that fewer would lose; sine and cosine of the fraction are fp32. The norm and the
// rotation are fp32 and each output is rounded once: Q and a bf16 pool to bf16, an FP8 pool to e4m3fn(x / s). (The one-axis
// writer rounds its intermediate steps to bf16 as the reference's torch path does; this operator has no such path to follow.)
//
// A workgroup takes 8 tokens, two to a wave, and a run of heads, 64 / (D / 8) at a time: lane j of a head holds its elements
// 8 j .. 8 j + 7 (one 16-byte load), the next heads' rows are on their way while these are worked on. The tokens' sines and
// cosines are computed once by the workgroup's threads (one each for two pairs of a token at D = 128) and handed round
// through LDS; a lane keeps its own in registers for every head. Bound by memory: every projection row is read once, every
// Q, K and V row written once: 185 MB for 8192 tokens of heads 32/8 of 128 to an e4m3fn pool in 42 us, 4.4 TB/s, where a
// plain copy reaches 4.8; few tokens by one launch's round trips (4.5 us).
#include <algorithm>

#include "sna_device.h"
#include "sna_host.h"

namespace sna {

struct MropeArgs {
  const uint16_t* qkv;  // [T, (Hq + 2 Hkv) D]
  int64_t qkv_stride, T;
  int32_t Hq, Hkv;
  const uint16_t* q_norm;  // [D], or both null
  const uint16_t* k_norm;
  float eps;
  const int64_t* positions;  // [A, T]
  int64_t pos_stride;
  const float* inv_freq;  // [half]
  int32_t half;           // rotated pairs
  uint64_t axes[2];       // 2 bits a pair
  const int64_t* slots;
  uint16_t* q_out;  // [T, Hq, D]
  uint8_t* k_cache;
  uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  int64_t num_slots;
  int32_t P;
  int32_t groups;  // head groups (of 64 / (D / 8) heads) that a workgroup takes
};

constexpr int kMropeTokens = 8;  // of a workgroup

// e4m3fn(clamp(x / s)) of two floats, as a 16-bit pair of bytes.
__device__ __forceinline__ uint32_t mrope_fp8_pair(float x0, float x1, float s, float rs, bool rcp_ok) {
  uint32_t b;
  if (rcp_ok) b = quantize_pair_e4m3fn_hw_nonan(x0, x1, s, rs);
  else b = f32_to_e4m3fn(clamp_fp8(x0 / s)) | f32_to_e4m3fn(clamp_fp8(x1 / s)) << 8;
  if (x0 != x0) b = (b & 0xff00u) | (__float_as_uint(x0) >> 24 & 0x80u) | 0x7fu;
  if (x1 != x1) b = (b & 0x00ffu) | ((__float_as_uint(x1) >> 24 & 0x80u) | 0x7fu) << 8;
  return b;
}

// 1 / sqrt(v), v >= eps, to 1 ulp. The instruction takes numbers below 2^-126 as 0, so where eps leaves room for them (a
// uniform branch; for every row 8192 tokens took 41.6 us instead of 41.2) small ones are scaled.
__device__ __forceinline__ float mrope_rsqrt(float v, float eps) {
  float up = 1.0f;
  if (__builtin_expect(eps < 0x1p-100f, 0)) {
    asm volatile("");  // (a branch: selects would be paid for by every row)
    if (v < 0x1p-100f) v *= 0x1p100f, up = 0x1p50f;
  }
  return __builtin_amdgcn_rsqf(v) * up;
}

// The angle position * inv_freq in half turns, in [-1, 1]. Up to 2^24 turns one double holds them: the constant's rounding, the
// position's and those of two products are 2^-27 of a turn at most, and the fraction's rounding to fp32 is 2^-26. Farther ones take
// 1 / (2 pi) as two doubles, its product with inv_freq as the rounded one (hi) and what is left of it (lo), and the position as
// two halves that are exact doubles; of each half's product with hi the whole part is dropped and the rounding's remainder, which
// an fma gives exactly, is kept: 2^-105 of the turns is left out. (All angles so: 8192 tokens 43.4 us instead of 42.2.)
__device__ __forceinline__ float mrope_half_turns(int64_t position, float inv_freq) {
#pragma clang fp contract(off)  // (a contracted p - rint(p) would take the remainder twice)
  constexpr double kInv2PiHi = 0x1.45f306dc9c883p-3, kInv2PiLo = -0x1.6b01ec5417056p-57;
  const double f = (double)inv_freq, hi = f * kInv2PiHi;
  double turns = (double)position * hi;
  if (!(fabs(turns) < 0x1p24)) {
    const double lo = fma(f, kInv2PiLo, fma(f, kInv2PiHi, -hi));
    const double half[2] = {(double)(int32_t)(position >> 32) * 0x1p32, (double)(uint32_t)position};
    turns = 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double p = half[i] * hi;
      turns += (p - rint(p)) + fma(half[i], lo, fma(half[i], hi, -p));
    }
  }
  return 2.0f * (float)(turns - rint(turns));
}

// FULL: every element of a head is rotated (its partner is the lane half a head away).
template <bool FP8, int D, bool FULL>
__global__ __launch_bounds__(256) void qkv_norm_mrope_store_kernel(MropeArgs a) {
  constexpr int LPH = D / 8, HPW = 64 / LPH, U = kMropeTokens / 4;
  __shared__ __attribute__((aligned(16))) float sm_cos[kMropeTokens][D / 2], sm_sin[kMropeTokens][D / 2];
  const int tid = threadIdx.x, lane = tid & 63, sub = lane % LPH;
  const int32_t wave = __builtin_amdgcn_readfirstlane((int32_t)(tid >> 6));
  const int32_t heads = a.Hq + 2 * a.Hkv;
  const int64_t tb = (int64_t)blockIdx.x * kMropeTokens, t0 = tb + wave * U;
  const int32_t g0 = blockIdx.y * a.groups, g1 = min(g0 + a.groups, (heads + HPW - 1) / HPW);
  const int32_t half = FULL ? D / 2 : a.half;
  uint4 w[U];
  auto load = [&](int32_t grp) {
    const int32_t head = grp * HPW + lane / LPH;
#pragma unroll
    for (int k = 0; k < U; ++k)
      w[k] = t0 + k < a.T && head < heads ? ld16_stream(a.qkv + (t0 + k) * a.qkv_stride + (int64_t)head * D + 8 * sub)
                                          : make_uint4(0, 0, 0, 0);
  };
  load(g0);
  int64_t kv_at[U];  // the tokens' elements in a pool of one KV head (redirected as the pool's store redirects)
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int64_t slot = t0 + k < a.T ? redirect_slot(a.slots[t0 + k], a.num_slots) : 0;
    const int64_t page = slot / a.P;
    kv_at[k] = (page * a.Hkv * a.P + (slot - page * a.P)) * D + 8 * sub;
  }
  for (int p = tid; p < kMropeTokens * half; p += 256) {
    const int k = p / half, i = p - k * half;
    if (tb + k >= a.T) break;
    const int axis = (int)(a.axes[i >> 5] >> (2 * (i & 31)) & 3);
    const float f = mrope_half_turns(a.positions[axis * a.pos_stride + tb + k], a.inv_freq[i]);
    sm_cos[k][i] = cospif(f);
    sm_sin[k][i] = sinpif(f);
  }
  __syncthreads();
  // the rotation partner of the lane's elements, half elements away; the lane's cosines and signed sines
  const bool rotated = FULL || 8 * sub < 2 * half, first = 8 * sub < half;
  const int partner = rotated ? lane + (first ? half / 8 : -(half / 8)) : lane;
  const int pair0 = rotated ? (first ? 8 * sub : 8 * sub - half) : 0;  // (one that is not rotated: any pair's, unused)
  float cs[U][8], sn[U][8];
#pragma unroll
  for (int k = 0; k < U; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = sm_sin[wave * U + k][pair0 + e];
      cs[k][e] = sm_cos[wave * U + k][pair0 + e];
      sn[k][e] = first ? -v : v;
    }
  for (int32_t grp = g0; grp < g1; ++grp) {  // uniform
    const int32_t head = grp * HPW + lane / LPH;
    const bool head_ok = head < heads;
    const bool is_q = head < a.Hq, is_k = !is_q && head < a.Hq + a.Hkv, roped = head < a.Hq + a.Hkv;
    const int32_t h = head - a.Hq - (is_k ? 0 : a.Hkv);  // the KV head (K and V lanes)
    uint4 cur[U];
#pragma unroll
    for (int k = 0; k < U; ++k) cur[k] = w[k];
    if (grp + 1 < g1) load(grp + 1);
    float gf[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) gf[e] = 1.0f;
    if (a.q_norm && head_ok && roped) {
      const uint4 gw = ld16((is_q ? a.q_norm : a.k_norm) + 8 * sub);
      const uint32_t gg[4] = {gw.x, gw.y, gw.z, gw.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) gf[e] = bf16_bits_to_f32(gg[e / 2] >> (16 * (e & 1)) & 0xffffu);
    }
    float scl = 1.0f, rs = 1.0f;
    bool rcp_ok = false;
    if (FP8 && head_ok && !is_q) {
      scl = is_k ? a.k_scale[h] : a.v_scale[h];
      rcp_ok = rcp_scale_ok(scl);
      rs = rcp_ok ? 1.0f / scl : 1.0f;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t t = t0 + k;
      if (t >= a.T) break;  // uniform
      const uint32_t ww[4] = {cur[k].x, cur[k].y, cur[k].z, cur[k].w};
      float x[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = e & 1 ? __uint_as_float(ww[e / 2] & 0xffff0000u) : bf16_bits_to_f32(ww[e / 2]);
      if (a.q_norm) {  // uniform
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        if constexpr (LPH == 16) {
          ss = row16_sum(ss);
        } else {
#pragma unroll
          for (int off = LPH / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, 64);
        }
        if (roped) {
          const float inv = mrope_rsqrt(ss * (1.0f / D) + a.eps, a.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * gf[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float o;
        if constexpr (FULL && LPH == 16)
          o = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x[e]), 0x128, 0xf, 0xf, true));  // row_ror:8
        else
          o = __shfl(x[e], partner, 64);
        y[e] = roped && rotated ? fmaf(x[e], cs[k][e], o * sn[k][e]) : x[e];  // (an infinite x * 0 would be NaN)
      }
      if (!head_ok) continue;
      const uint4 b16 = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                                   pack_bf16x2(y[6], y[7]));
      if (is_q) {
        *reinterpret_cast<uint4*>(a.q_out + (t * a.Hq + head) * D + 8 * sub) = b16;
        continue;
      }
      uint8_t* const cache = is_k ? a.k_cache : a.v_cache;
      const int64_t dst = kv_at[k] + (int64_t)h * a.P * D;
      if constexpr (FP8) {
        *reinterpret_cast<uint2*>(cache + dst) =
            make_uint2(mrope_fp8_pair(y[0], y[1], scl, rs, rcp_ok) | mrope_fp8_pair(y[2], y[3], scl, rs, rcp_ok) << 16,
                       mrope_fp8_pair(y[4], y[5], scl, rs, rcp_ok) | mrope_fp8_pair(y[6], y[7], scl, rs, rcp_ok) << 16);
      } else {
        *reinterpret_cast<uint4*>(cache + 2 * dst) = b16;
      }
    }
  }
}

// A token block's heads are shared out until a launch has so many workgroups: 8 tokens of heads 16/8 of 128 take 4.7 us so and
// 10.4 with a workgroup for all heads, 1531 of heads 24/4 of 64 6.0 and 7.9; 8192 tokens of heads 32/8 of 128 take 42 with
// their heads in one workgroup and 56 with one a head group, which computes their angles each time.
constexpr int64_t kMropeWorkgroups = 1024;

}  // namespace sna

using namespace sna;

extern "C" int sna_qkv_norm_mrope_store(const void* qkv, int64_t qkv_stride, int64_t n_tokens, int32_t num_q_heads,
                                        int32_t num_kv_heads, int32_t head_dim, const void* q_norm, const void* k_norm,
                                        float eps, const int64_t* positions, int64_t pos_stride, int32_t n_axes,
                                        const float* inv_freq, int32_t n_pairs, const uint8_t* axes,
                                        const int64_t* slots, void* q_out, void* k_cache, void* v_cache,
                                        const float* k_scale, const float* v_scale, int64_t num_blocks,
                                        int32_t page_size, int32_t cache_dtype, void* stream) {
  ApiGuard guard;
  if (n_tokens < 0 || num_q_heads < 1 || num_kv_heads < 1 || page_size < 1 || num_blocks < 1)
    return fail(SNA_ERR_INVALID_ARGUMENT,
                "qkv_norm_mrope_store: bad sizes (tokens %lld, heads %d/%d, head_dim %d, page %d, blocks %lld)",
                (long long)n_tokens, num_q_heads, num_kv_heads, head_dim, page_size, (long long)num_blocks);
  if (head_dim != 64 && head_dim != 128)
    return fail(SNA_ERR_UNSUPPORTED, "qkv_norm_mrope_store: head_dim %d (64 or 128 are built)", head_dim);
  if (n_axes < 1 || n_axes > 4)
    return fail(SNA_ERR_UNSUPPORTED, "qkv_norm_mrope_store: %d position axes (1 to 4)", n_axes);
  if (n_pairs < 8 || n_pairs % 8 != 0 || 2 * n_pairs > head_dim)
    return fail(SNA_ERR_UNSUPPORTED, "qkv_norm_mrope_store: %d rotated pairs (a multiple of 8, at most head_dim / 2 = %d)",
                n_pairs, head_dim / 2);
  if (qkv_stride < (int64_t)(num_q_heads + 2 * (int64_t)num_kv_heads) * head_dim || pos_stride < n_tokens)
    return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: row strides %lld / %lld are shorter than a row",
                (long long)qkv_stride, (long long)pos_stride);
  if ((q_norm == nullptr) != (k_norm == nullptr))
    return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: give both QK-norm gammas or neither");
  if (cache_dtype == SNA_DTYPE_FP8_E4M3FN_MUL)
    return fail(SNA_ERR_UNSUPPORTED, "qkv_norm_mrope_store: the writer divides by dequantization scales; for a pool of "
                "multipliers m pass SNA_DTYPE_FP8_E4M3FN with the scales bf16(1 / m)");
  if (cache_dtype != SNA_DTYPE_BF16 && cache_dtype != SNA_DTYPE_FP8_E4M3FN)
    return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: unknown cache dtype %d", cache_dtype);
  if (!axes) return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: null pointer");
  MropeArgs a;
  a.axes[0] = a.axes[1] = 0;
  for (int32_t i = 0; i < n_pairs; ++i) {
    if (axes[i] >= n_axes)
      return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: pair %d on axis %d of %d", i, axes[i], n_axes);
    a.axes[i >> 5] |= (uint64_t)axes[i] << (2 * (i & 31));
  }
  const bool fp8 = cache_dtype == SNA_DTYPE_FP8_E4M3FN;
  if (n_tokens == 0) return SNA_OK;
  if (!qkv || !positions || !inv_freq || !slots || !q_out || !k_cache || !v_cache || (fp8 && (!k_scale || !v_scale)))
    return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: null pointer");
  if (!(eps >= 0.0f)) return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: eps %g", (double)eps);
  if (!aligned(qkv, 16) || qkv_stride % 8 || !aligned(q_out, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) ||
      (q_norm && (!aligned(q_norm, 16) || !aligned(k_norm, 16))))
    return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: tensors and row strides must be 16-byte aligned");
  const int32_t hpw = 64 / (head_dim / 8);
  // (32 bits number a launch's threads along a grid axis)
  const int64_t token_blocks = (n_tokens + kMropeTokens - 1) / kMropeTokens;
  const int64_t head_groups = (num_q_heads + 2 * (int64_t)num_kv_heads + hpw - 1) / hpw;
  if (token_blocks >= 1 << 24 || head_groups > 65535)
    return fail(SNA_ERR_INVALID_ARGUMENT, "qkv_norm_mrope_store: %lld tokens of %lld heads are too many for one launch",
                (long long)n_tokens, num_q_heads + 2ll * num_kv_heads);
  a.qkv = (const uint16_t*)qkv;
  a.qkv_stride = qkv_stride;
  a.T = n_tokens;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.q_norm = (const uint16_t*)q_norm;
  a.k_norm = (const uint16_t*)k_norm;
  a.eps = eps;
  a.positions = positions;
  a.pos_stride = pos_stride;
  a.inv_freq = inv_freq;
  a.half = n_pairs;
  a.slots = slots;
  a.q_out = (uint16_t*)q_out;
  a.k_cache = (uint8_t*)k_cache;
  a.v_cache = (uint8_t*)v_cache;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.num_slots = num_blocks * page_size;
  a.P = page_size;
  const int64_t parts = std::min(head_groups, (kMropeWorkgroups + token_blocks - 1) / token_blocks);
  a.groups = (int32_t)((head_groups + parts - 1) / parts);
  const dim3 grid((unsigned)token_blocks, (unsigned)((head_groups + a.groups - 1) / a.groups));
  const hipStream_t s = (hipStream_t)stream;
  const bool full = 2 * n_pairs == head_dim;
#define SNA_MROPE_LAUNCH(F, DD)                                                                                        \
  if (full) hipLaunchKernelGGL((qkv_norm_mrope_store_kernel<F, DD, true>), grid, dim3(256), 0, s, a);                  \
  else hipLaunchKernelGGL((qkv_norm_mrope_store_kernel<F, DD, false>), grid, dim3(256), 0, s, a)
  if (fp8 && head_dim == 128) { SNA_MROPE_LAUNCH(true, 128); }
  else if (fp8) { SNA_MROPE_LAUNCH(true, 64); }
  else if (head_dim == 128) { SNA_MROPE_LAUNCH(false, 128); }
  else { SNA_MROPE_LAUNCH(false, 64); }
#undef SNA_MROPE_LAUNCH
  return check_launch("qkv_norm_mrope_store");
}
