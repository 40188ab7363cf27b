// Attention of single query tokens over a paged GQA cache whose blocks of tokens carry scales (e4m3fn or int8 codes; bf16
// without scales): over all of a row's keys, or over the pages that a list names for each query and KV head.
//
//   out[t, h] = sum_j p_j v_j / (sum_j p_j + e^(sink_h - m)),  p_j = e^(sm_scale q[t, h] . k_j - m),
// over the keys j < seq_lens[t] of table row rows[t] (inside the window; on the listed pages), with k_j = code * its
// block's K scale and v_j = code * its block's V scale. A block's scales are the same for 16 keys at a time, so K's joins
// the score's factor and V's the probability: codes go into the matrix products as they are, exact in bf16.
//
// Work: one workgroup per (query, KV head), or, where those do not fill the card, per (split of a query, KV head): a
// query's splits divide its tiles evenly, and a second launch merges them. A wave takes tiles round-robin, the next one's
// loads in flight while it computes one.
// A tile is two half-tiles of 16 keys, each inside one page and one block. Lane roles (lane = 16 g4 + li):
//   QK   S^T[key, head] = K[key, :] . Q[head, :], v_mfma_f32_16x16x32_bf16 with M = 16 keys, N = 16 heads (the group's,
//        zero-padded): lane (g4, li) feeds key li's 16-byte chunks 4 c + g4 and head li's elements of the same dims, and
//        gets S^T[4 g4 + r, li].
//   PV   O^T[d, head] = V^T[d, keys] . P^T[keys, head] over the tile's 32 keys, lane (g4, *) supplying keys 4 g4 .. + 3 of
//        both halves, which are the probabilities it holds: only V is transposed, in registers (lane (g4, li) loads D / 16
//        contiguous elements from D / 16 * li of its 8 keys).
//   acc  lane (g4, j), d-tile t, row r: O[head j, D / 16 * (4 g4 + r) + t].
// The softmax state is (m, l, acc) in the log2 domain, m moved only when a tile's maximum passes it by more than 8.
//
// What bounds it: HBM where the rows fill the card (64 rows of 4096 e4m3fn keys, 32 / 8 heads of 128, pages of 16: 87 us, 539 MB,
// 6.2 TB/s; one row of 131071 int8 keys 48 us, the first launch at 6.0; matrix pipe 7%, VALU 38% of the cycles); the longest
// row's share and the merge where they are ragged (128 rows of 2048 to 8192, 8 heads on one of 64, int8: 22 + 3 us for 84 MB).
// Many queries of few rows with pages of their own go another way, block_pages_kernel.
#include <algorithm>

#include "sna_device.h"
#include "sna_host.h"

namespace sna {

struct BlockDecodeArgs {
  const uint16_t* q;  // [T, H, D] bf16
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;  // [num_blocks, G, P / bt], page and head strides below
  const float* v_scale;
  int64_t scale_page, scale_head;
  int32_t sub_magic;  // ceil(2^16 / (bt / 16)): a 16-key half's block in its page (0: one block a page)
  const int32_t* table;
  int64_t table_stride;
  int32_t table_width, table_rows;
  const int32_t* rows;      // [T] each query's table row, or null: query t's is t
  const int32_t* seq_lens;  // [T]
  const int32_t* blocks;    // SEL: [T, G, n_blocks] table columns
  int32_t n_blocks;
  const float* sinks;  // [H] or null
  int32_t T, H, G, group, P, halves;  // halves: 16-key halves a page
  int64_t num_blocks;
  int32_t window;
  float sm_scale;
  int32_t splits;  // of a query's tiles; of a launch page by page n_blocks * segs: a partial for each listed page's 64 keys
  int32_t segs;    // page by page: runs of 64 keys of a page
  float* ws_o;     // [T, splits, H, D] unnormalized partials
  float* ws_ml;    // [T, splits, H, 2] reference max (log2 domain) and softmax sum
  uint16_t* out;
};

// The 32-key tiles of a query of L keys: [first, first + n). Dense: tile i is positions 32 i ..; SEL: the listed pages'
// halves two by two, whatever they name.
template <bool SEL>
__device__ __forceinline__ void block_tiles_of(const BlockDecodeArgs& a, int32_t L, int32_t& first, int32_t& n) {
  const int32_t lo = a.window > 0 ? max(0, L - a.window) : 0;
  first = SEL ? 0 : lo / 32;
  n = L <= 0 ? 0 : SEL ? (a.n_blocks * a.halves + 1) / 2 : (int32_t)(((int64_t)L + 31) / 32) - first;
}
// (keys past the table have no page)
__device__ __forceinline__ int32_t block_len(const BlockDecodeArgs& a, int32_t len) {
  return (int32_t)min((int64_t)max(len, 0), (int64_t)a.table_width * a.P);
}

constexpr float kBlockRescaleSlack = 8.0f;

// NB bytes of a V row; STREAM: non-temporal (see below).
template <int NB, bool STREAM>
__device__ __forceinline__ void load_run(const uint8_t* p, uint32_t (&dst)[NB / 4]) {
  if constexpr (NB % 16 == 0) {
#pragma unroll
    for (int i = 0; i < NB / 16; ++i) {
      const uint4 w = STREAM ? ld16_stream(p + 16 * i) : ld16(p + 16 * i);
      dst[4 * i] = w.x, dst[4 * i + 1] = w.y, dst[4 * i + 2] = w.z, dst[4 * i + 3] = w.w;
    }
  } else if constexpr (NB == 8) {
    const uint2 w = STREAM ? ld8_stream(p) : ld8(p);
    dst[0] = w.x, dst[1] = w.y;
  } else {
    static_assert(NB == 4, "4, 8 or a multiple of 16 bytes");
    dst[0] = STREAM ? ld4_stream(p) : *reinterpret_cast<const uint32_t*>(p);
  }
}

// Four codes of a dword to four bf16 values.
template <int FMT>
__device__ __forceinline__ void codes_to_bf16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == kBlockFp8) fp8x4_to_bf16x4(w, lo, hi);
  else int8x4_to_bf16x4(w, lo, hi);
}

template <int D, int FMT>
struct BlockTile {
  static constexpr int ESZ = FMT == kBlockBf16 ? 2 : 1;
  static constexpr int KB = D / 4 * ESZ;   // K bytes per lane and key
  static constexpr int VB = D / 16 * ESZ;  // V bytes per lane and key
  uint32_t k[2][KB / 4];
  uint32_t v[8][VB / 4];
  float scale;     // lane group 0: K's of half 0, 1: K's of half 1, 2 and 3: V's
  int32_t pos[2];  // the halves' first positions
  bool valid[2];   // on a page of the pool, below the table's width
};

// The operand of a 16-wide d-tile of V^T over a tile's 32 keys, regrouped in registers: byte or element dt of each key's run.
template <int D, int FMT>
__device__ __forceinline__ void block_v_op(const BlockTile<D, FMT>& T, int dt, uint32_t (&op)[4]) {
  if constexpr (FMT == kBlockBf16) {
#pragma unroll
    for (int pr = 0; pr < 4; ++pr) {
      const uint32_t e0 = (T.v[2 * pr][dt >> 1] >> (16 * (dt & 1))) & 0xffffu;
      const uint32_t e1 = (T.v[2 * pr + 1][dt >> 1] >> (16 * (dt & 1))) & 0xffffu;
      op[pr] = e0 | (e1 << 16);
    }
  } else {
    uint32_t c0 = 0, c1 = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c0 |= ((T.v[e][dt >> 2] >> (8 * (dt & 3))) & 0xffu) << (8 * e);
      c1 |= ((T.v[e + 4][dt >> 2] >> (8 * (dt & 3))) & 0xffu) << (8 * e);
    }
    codes_to_bf16x4<FMT>(c0, op[0], op[1]);
    codes_to_bf16x4<FMT>(c1, op[2], op[3]);
  }
}

// SHARED: queries of one row, which read the same pages, may be among the call's (`rows`). V then stays in the L2 (2 x 256
// queries of 1024 selected keys, bf16, one by one: 178 -> 152 us); else it is read once, past it (64 rows of 4096 FP8 keys 87.5
// us, through the L2 97). K, two loads a 128-byte line, always goes through it (past it 90; the 2 x 256 queries 244).
template <int D, int FMT, bool SEL, bool SPLIT, int WAVES, bool SHARED>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2)))
void block_decode_kernel(BlockDecodeArgs a) {
  using Tile = BlockTile<D, FMT>;
  constexpr int ESZ = Tile::ESZ, KB = Tile::KB, VB = Tile::VB;
  constexpr int STEPS = D / 32;  // QK products of a half-tile
  constexpr int VE = D / 16;     // V elements per lane and key
  constexpr int DT = D / 16;     // d-tiles
  constexpr int CE = 16 / ESZ;   // elements of a 16-byte chunk
  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, li = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t items = (uint32_t)(SPLIT ? a.T * a.splits : a.T);  // of a KV head
  // Queries of one row with the KV head fastest: a head's are found in one L2 (the 2 x 256: 290 -> 244 us, non-temporal then).
  // Rows of their own gain nothing by that and lose where a head's rows of a page are a few KB, which one head alone reads
  // through a part of its L2's channels (64 rows of 4096 FP8 keys: 90 -> 101 us).
  const uint32_t v = SHARED ? blockIdx.x / (uint32_t)a.G : blockIdx.x % items;
  const int32_t g = (int32_t)(SHARED ? blockIdx.x - v * a.G : blockIdx.x / items);
  const int32_t t = (int32_t)(SPLIT ? v / (uint32_t)a.splits : v), split = SPLIT ? (int32_t)v - t * a.splits : 0;
  const int32_t len_v = a.seq_lens[t];
  const int32_t row_v = a.rows ? a.rows[t] : t;

  // query operand: step s, lane (g4, li): head li's 8 elements from dim CE (4 c + g4) + w, 8 s = CE c + w
  uint32_t qv[STEPS][4];
  {
    const uint16_t* qp = a.q + ((int64_t)t * a.H + g * a.group + min(li, a.group - 1)) * D;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const uint4 w = ld16(qp + CE * (4 * (8 * s / CE) + g4) + (8 * s) % CE);
      const bool live = li < a.group;
      qv[s][0] = live ? w.x : 0u, qv[s][1] = live ? w.y : 0u, qv[s][2] = live ? w.z : 0u, qv[s][3] = live ? w.w : 0u;
    }
  }
  const float sink_pre = a.sinks && tid < a.group ? a.sinks[g * a.group + tid] : 0.0f;

  const int32_t row = __builtin_amdgcn_readfirstlane(row_v);
  const bool row_ok = row >= 0 && row < a.table_rows;
  const int32_t L = row_ok ? block_len(a, __builtin_amdgcn_readfirstlane(len_v)) : 0;
  const int32_t lo = a.window > 0 ? max(0, L - a.window) : 0;  // visible: [lo, L)
  const int32_t* trow = a.table + (int64_t)(row_ok ? row : 0) * a.table_stride;
  const int32_t* list = SEL ? a.blocks + ((int64_t)t * a.G + g) * a.n_blocks : nullptr;
  int32_t t_first, t_last;
  block_tiles_of<SEL>(a, L, t_first, t_last);
  t_last += t_first;
  if constexpr (SPLIT) {
    const int32_t n = t_last - t_first, per = n / a.splits, extra = n - per * a.splits;
    t_first += split * per + min(split, extra);
    t_last = t_first + per + (split < extra ? 1 : 0);
  }

  const int32_t ncol = SEL ? a.n_blocks : a.table_width;
  const bool pow2 = (a.P & (a.P - 1)) == 0;
  const int p_shift = __builtin_ctz((uint32_t)a.P);
  // entry (table column, or place in the list) of a half, and its place in the page
  auto entry_of = [&](int32_t half) -> int32_t { return pow2 ? half >> (p_shift - 4) : half / a.halves; };
  // The pages of 256 entries from col0 on, entry col0 + 64 i + lane in pg[i] (-1: none); SEL: their table columns in bk.
  // A wave's entries ascend: it loads the next 256 when it gets there.
  int32_t col0 = 0, pg[4], bk[4];
  auto stage = [&](int32_t c0) {
    col0 = c0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t c = c0 + 64 * i + lane;
      int32_t b = c;
      if (SEL) b = c < ncol ? list[c] : -1;
      pg[i] = b >= 0 && b < a.table_width && c < ncol ? trow[b] : -1;
      if (pg[i] >= a.num_blocks) pg[i] = -1;
      bk[i] = pg[i] >= 0 ? b : 0;
    }
  };
  auto pick = [&](const int32_t (&v)[4], int32_t c) -> int32_t {
    return __builtin_amdgcn_readlane(c < 64 ? v[0] : (c < 128 ? v[1] : (c < 192 ? v[2] : v[3])), c & 63);
  };

  const int64_t head_bytes = (int64_t)a.P * D * ESZ;
  const float* scale_base = FMT == kBlockBf16 ? nullptr : (g4 < 2 ? a.k_scale : a.v_scale) + g * a.scale_head;
  const uint32_t k_off = (uint32_t)(li * D * ESZ + 16 * g4), v_off = (uint32_t)(4 * g4 * D * ESZ + VB * li);
  auto load_tile = [&](Tile& T, int32_t tile) {
    int32_t page[2], sub[2];
    const int32_t half0 = __builtin_amdgcn_readfirstlane(2 * tile);
    if (entry_of(half0 + 1) - col0 >= 256) stage(entry_of(half0));
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int32_t half = half0 + hf, e = entry_of(half), in16 = half - e * a.halves;  // the half's place in its page
      const bool inside = e < ncol;
      const int32_t c = inside ? e - col0 : 0;
      const int32_t p = pick(pg, c);
      const int32_t b = SEL ? pick(bk, c) : e;
      T.pos[hf] = b * a.P + 16 * in16;
      T.valid[hf] = inside && p >= 0 && T.pos[hf] < L && T.pos[hf] + 16 > lo;
      page[hf] = T.valid[hf] ? p : 0;
      sub[hf] = T.valid[hf] ? (int32_t)((uint32_t)in16 * (uint32_t)a.sub_magic >> 16) : 0;
      // (uniform bases and 32-bit offsets of the lane: addresses take no vector arithmetic)
      const int64_t blk = ((int64_t)page[hf] * a.G + g) * head_bytes + (int64_t)(16 * in16) * D * ESZ;
      const uint8_t* kp = a.k_cache + blk;
      const uint8_t* vp = a.v_cache + blk;
#pragma unroll
      for (int c4 = 0; c4 < KB / 16; ++c4) {
        const uint4 w = ld16(kp + k_off + 64 * c4);
        T.k[hf][4 * c4] = w.x, T.k[hf][4 * c4 + 1] = w.y, T.k[hf][4 * c4 + 2] = w.z, T.k[hf][4 * c4 + 3] = w.w;
      }
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4)
        load_run<VB, !SHARED>(vp + v_off + e4 * D * ESZ, T.v[4 * hf + e4]);
    }
    if constexpr (FMT != kBlockBf16) {
      const bool second = g4 & 1;
      T.scale = scale_base[(int64_t)(second ? page[1] : page[0]) * a.scale_page + (second ? sub[1] : sub[0])];
    }
  };

  float m_ref = kNegBig, l_run = 0.0f;
  f32x4_t acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float qk_scale = a.sm_scale * kLog2e;

  auto compute_tile = [&](Tile& T) {
    float ks[2] = {qk_scale, qk_scale}, vs[2] = {1.0f, 1.0f};
    if constexpr (FMT != kBlockBf16) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        ks[hf] = qk_scale * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(T.scale), 16 * hf));
        vs[hf] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(T.scale), 32 + 16 * hf));
      }
    }
    float x[8];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        uint32_t op[4];
        if constexpr (FMT == kBlockBf16) {
#pragma unroll
          for (int i = 0; i < 4; ++i) op[i] = T.k[hf][4 * st + i];
        } else {
          codes_to_bf16x4<FMT>(T.k[hf][2 * st], op[0], op[1]);
          codes_to_bf16x4<FMT>(T.k[hf][2 * st + 1], op[2], op[3]);
        }
        s = mfma_16x16x32_bf16(op, qv[st], s);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x[4 * hf + r] = s[r] * ks[hf];
    }
    // a tile that is not wholly visible: hidden keys score -inf and their V (which may be anything) is zero
    const bool full = T.valid[0] && T.valid[1] && T.pos[0] >= lo && T.pos[1] >= lo && T.pos[0] + 16 <= L && T.pos[1] + 16 <= L;
    if (!full) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        bool any = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int32_t pos = T.pos[hf] + 4 * g4 + r;
          const bool ok = T.valid[hf] && pos >= lo && pos < L;
          any |= ok;
          x[4 * hf + r] = ok ? x[4 * hf + r] : -INFINITY;
#pragma unroll
          for (int i = 0; i < VB / 4; ++i) T.v[4 * hf + r][i] = ok ? T.v[4 * hf + r][i] : 0u;
        }
        vs[hf] = any ? vs[hf] : 1.0f;  // (a block with no visible key here: its scale may be anything)
      }
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) tmax = fmaxf(tmax, x[i]);
    tmax = max_across_groups(tmax);
    const bool bump = tmax > m_ref + kBlockRescaleSlack;
    if (__any(bump)) {
      const float m_new = bump ? tmax : m_ref;
      const float alpha = __builtin_amdgcn_exp2f(m_ref - m_new);
      m_ref = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] *= alpha;
    }
    // The probabilities, times V's scale, go into the product as bf16, off by at most 2^-8 of themselves; their sum is of the
    // same rounded values (over the scale again), so that a row which one key carries is off by nothing (8 rows of 128 to 1024
    // keys: 2.5e-3 of the result, norm by norm, with the unrounded sum, 2.0e-3 so; the rounding of the result alone 1.6e-3).
    uint32_t pop[4];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float part = 0.0f;
      // (a scale under the least one of a block is taken for that; NaN stays)
      const float v = vs[hf] < kLeastBlockScale ? kLeastBlockScale : vs[hf];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float p0 = __builtin_amdgcn_exp2f(x[4 * hf + 2 * k] - m_ref), p1 = __builtin_amdgcn_exp2f(x[4 * hf + 2 * k + 1] - m_ref);
        if constexpr (FMT != kBlockBf16) p0 *= v, p1 *= v;
        pop[2 * hf + k] = pack_bf16x2(p0, p1);
        float& sum = FMT != kBlockBf16 ? part : l_run;
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pop[2 * hf + k]),
                                              __builtin_bit_cast(bf16x2_t, 0x3f803f80u), sum, false);
      }
      if constexpr (FMT != kBlockBf16) l_run = fmaf(part, __builtin_amdgcn_rcpf(v), l_run);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      uint32_t op[4];
      block_v_op<D, FMT>(T, dt, op);
      acc[dt] = mfma_16x16x32_bf16(op, pop, acc[dt]);
    }
  };

  // ---- the tile loop: two register tiles, one in flight ----
  {
    Tile ring[2];
    const int32_t first = t_first + wave;
    if (first < t_last) {
      stage(entry_of(2 * first));
      load_tile(ring[0], first);
    }
    for (int32_t cur = first; cur < t_last;) {
      if (cur + WAVES < t_last) load_tile(ring[1], cur + WAVES);
      compute_tile(ring[0]);
      cur += WAVES;
      if (cur >= t_last) break;
      if (cur + WAVES < t_last) load_tile(ring[0], cur + WAVES);
      compute_tile(ring[1]);
      cur += WAVES;
    }
  }

  // ---- merge the waves in LDS; write the output, or this split's partial ----
  __shared__ float sm_o[WAVES][16][D + 1];
  __shared__ float sm_m[WAVES][16], sm_l[WAVES][16], sm_sink[16];
  if (tid < a.group) sm_sink[tid] = sink_pre;
  const float l_tot = sum_across_groups(l_run);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) sm_o[wave][li][VE * (4 * g4 + r) + dt] = acc[dt][r];
  if (g4 == 0) sm_m[wave][li] = m_ref, sm_l[wave][li] = l_tot;
  __syncthreads();
  for (int32_t idx = tid; idx < a.group * D; idx += 64 * WAVES) {
    const int32_t j = idx / D, d = idx % D;
    float M = kNegBig;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M = fmaxf(M, sm_m[w][j]);
    float o = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float e = __builtin_amdgcn_exp2f(sm_m[w][j] - M);
      o += e * sm_o[w][j][d];
      l += e * sm_l[w][j];
    }
    if constexpr (SPLIT) {
      const int64_t at = (int64_t)v * a.H + g * a.group + j;
      a.ws_o[at * D + d] = o;
      if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * at) = make_float2(M, l);
    } else {
      if (a.sinks) l += __builtin_amdgcn_exp2f(sm_sink[j] * kLog2e - M);
      a.out[((int64_t)t * a.H + g * a.group + j) * D + d] = (uint16_t)f32_to_bf16_bits(l == 0.0f ? 0.0f : o / l);
    }
  }
}

// Page by page, for many queries of few rows (a prompt's, each with pages of its own choice): a workgroup finds the queries
// whose lists name one of four pages of a row, for one KV head and 64 keys of the page, keeps a page's keys as operands in
// registers and attends 16 / group queries at a time to them, so a page is read once, not once a query, and the columns are full.
// A partial is written for each entry of the lists and merged as splits are. Latency bounds it: a page's operands take all the
// registers that two waves a SIMD have, and each batch waits for its queries (2 x 256 queries of 16 pages of 64, bf16, group 2:
// 94 us, of which the search 20 and the merge 13; with one page a workgroup 30 more, the lists searched once for each; the first
// and last pages, which most lists name, before the others 9 more).
constexpr int kPageWaves = 4;  // and pages
constexpr int kPageScan = 8;   // entries that a thread reads at a time
constexpr int kPageStep = kPageScan * 64 * kPageWaves, kPageList = kPageStep + 1024;
template <int D, int FMT>
__global__ __launch_bounds__(64 * kPageWaves) __attribute__((amdgpu_waves_per_eu(2)))
void block_pages_kernel(BlockDecodeArgs a) {
  using Tile = BlockTile<D, FMT>;
  constexpr int ESZ = Tile::ESZ, KB = Tile::KB, VB = Tile::VB, STEPS = D / 32, VE = D / 16, DT = D / 16, CE = 16 / ESZ;
  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, li = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t idx = blockIdx.x;
  const int32_t g = (int32_t)(idx % (uint32_t)a.G);
  idx /= (uint32_t)a.G;
  const int32_t seg = (int32_t)(idx % (uint32_t)a.segs);
  idx /= (uint32_t)a.segs;
  const uint32_t quads = ((uint32_t)a.table_width + kPageWaves - 1) / kPageWaves;
  const int32_t c0 = (int32_t)(idx % quads) * kPageWaves, row = (int32_t)(idx / quads);
  const int32_t keys = min(a.P - 64 * seg, 64);  // of a page's, this workgroup's

  // By page: the entries t * n_blocks + i of the lists that name it, of queries that see all of the keys from the front, of
  // queries that see some of them from the end; how many, how many of them waves have taken, the most keys that one of the
  // latter sees.
  __shared__ int32_t sm_e[kPageWaves][kPageList], sm_n[kPageWaves][2], sm_taken[kPageWaves][2], sm_vis[kPageWaves];
  __shared__ int32_t sm_hit[kPageStep], sm_page[kPageWaves], sm_hits, sm_first, sm_end;
  if (tid < kPageWaves) {
    int32_t page = c0 + tid < a.table_width ? a.table[(int64_t)row * a.table_stride + c0 + tid] : -1;
    if ((int64_t)page >= a.num_blocks) page = -1;
    sm_page[tid] = page;
    sm_n[tid][0] = sm_n[tid][1] = sm_taken[tid][0] = sm_taken[tid][1] = sm_vis[tid] = 0;
    if (tid == 0) sm_hits = 0, sm_first = INT32_MAX, sm_end = 0;
  }
  __syncthreads();
  {  // the row's queries lie in [sm_first, sm_end)
    int32_t lo = INT32_MAX, hi = 0;
    for (int32_t t = tid; t < a.T; t += 64 * kPageWaves)
      if (a.rows[t] == row) lo = min(lo, t), hi = t + 1;
    if (hi > 0) atomicMin(&sm_first, lo), atomicMax(&sm_end, hi);
  }
  __syncthreads();
  const int32_t t_first = sm_first, t_end = sm_end;
  if (t_end == 0) return;
  auto seen = [&](int32_t t, int32_t c) { return block_len(a, a.seq_lens[t]) - (c0 + c) * a.P - 64 * seg; };

  // The keys as operands in bf16: 16 keys (rows) of K by 32 of D, 16 of D by 32 keys of V. V of keys from `vis` on is zero (what
  // was never stored may be anything).
  struct Keys {
    uint32_t k_op[4][STEPS][4], v_op[2][DT][4];
    float scales[2];
  };
  // scales: of both tiles, in the lanes of the format's decode: K's at 0 and 16, V's at 32 and 48
  const uint32_t k_off = (uint32_t)(li * D * ESZ + 16 * g4), v_off = (uint32_t)(4 * g4 * D * ESZ + VB * li);
  const float* scale_base = FMT == kBlockBf16 ? nullptr : (g4 < 2 ? a.k_scale : a.v_scale) + g * a.scale_head;
  auto load = [&](Keys& o, int32_t c, int32_t vis) {
    const int32_t page = __builtin_amdgcn_readfirstlane(sm_page[c]);
    const int64_t at0 = (((int64_t)page * a.G + g) * a.P + 64 * seg) * D * ESZ;
    Tile T[2];
#pragma unroll
    for (int tl = 0; tl < 2; ++tl) {
      int32_t sub[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int32_t half = 2 * tl + hf;
        const bool in = 16 * half < keys;  // (uniform; past the page: the first half again, which is masked)
        const uint8_t* kp = a.k_cache + at0 + (int64_t)(in ? 16 * half : 0) * D * ESZ;
        const uint8_t* vp = a.v_cache + at0 + (int64_t)(in ? 16 * half : 0) * D * ESZ;
        sub[hf] = (int32_t)((uint32_t)(4 * seg + (in ? half : 0)) * (uint32_t)a.sub_magic >> 16);
#pragma unroll
        for (int c4 = 0; c4 < KB / 16; ++c4) {
          const uint4 w = ld16(kp + k_off + 64 * c4);
          T[tl].k[hf][4 * c4] = w.x, T[tl].k[hf][4 * c4 + 1] = w.y, T[tl].k[hf][4 * c4 + 2] = w.z, T[tl].k[hf][4 * c4 + 3] = w.w;
        }
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) load_run<VB, false>(vp + v_off + e4 * D * ESZ, T[tl].v[4 * hf + e4]);
      }
      if constexpr (FMT != kBlockBf16)
        o.scales[tl] = scale_base[(int64_t)page * a.scale_page + (g4 & 1 ? sub[1] : sub[0])];
    }
#pragma unroll
    for (int tl = 0; tl < 2; ++tl) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < VB / 4; ++i)
            T[tl].v[4 * hf + r][i] = 32 * tl + 16 * hf + 4 * g4 + r < vis ? T[tl].v[4 * hf + r][i] : 0u;
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          uint32_t(&op)[4] = o.k_op[2 * tl + hf][st];
          if constexpr (FMT == kBlockBf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) op[i] = T[tl].k[hf][4 * st + i];
          } else {
            codes_to_bf16x4<FMT>(T[tl].k[hf][2 * st], op[0], op[1]);
            codes_to_bf16x4<FMT>(T[tl].k[hf][2 * st + 1], op[2], op[3]);
          }
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) block_v_op<D, FMT>(T[tl], dt, o.v_op[tl][dt]);
    }
  };

  const float qk_scale = a.sm_scale * kLog2e;
  // Columns [0, tpi * group): n entries from e0 on. What a query does not see counts nothing, except that a NaN or an infinity
  // among it becomes NaN: false, and nothing is written, if `check` and the result holds one.
  auto attend = [&](const Keys& o, int32_t c, int part, int32_t e0, int32_t n, bool check) -> bool {
    const int32_t ce = li / a.group, hc = li - ce * a.group;
    const bool live = ce < n;
    const int32_t e = sm_e[c][part ? kPageList - 1 - e0 - (live ? ce : 0) : e0 + (live ? ce : 0)], t = e / a.n_blocks;
    const int32_t vis = part ? seen(t, c) : keys;
    uint32_t qv[STEPS][4];
    const uint16_t* qp = a.q + ((int64_t)t * a.H + g * a.group + hc) * D;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const uint4 w = ld16(qp + CE * (4 * (8 * s / CE) + g4) + (8 * s) % CE);
      qv[s][0] = w.x, qv[s][1] = w.y, qv[s][2] = w.z, qv[s][3] = w.w;
    }
    float x[2][8], m = kNegBig;
#pragma unroll
    for (int h4 = 0; h4 < 4; ++h4) {
      float ks = qk_scale;
      if constexpr (FMT != kBlockBf16)
        ks *= __int_as_float(__builtin_amdgcn_readlane(__float_as_int(o.scales[h4 / 2]), 16 * (h4 & 1)));
      f32x4_t sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < STEPS; ++st) sc = mfma_16x16x32_bf16(o.k_op[h4][st], qv[st], sc);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float& y = x[h4 / 2][4 * (h4 & 1) + r];
        y = 16 * h4 + 4 * g4 + r < vis ? sc[r] * ks : -INFINITY;
        m = fmaxf(m, y);
      }
    }
    m = max_across_groups(m);
    float l = 0.0f;
    f32x4_t acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int tl = 0; tl < 2; ++tl) {
      uint32_t pop[4];  // (rounded and summed as in block_decode_kernel)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float v = 1.0f, part_l = 0.0f;
        if constexpr (FMT != kBlockBf16) {
          v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(o.scales[tl]), 32 + 16 * hf));
          v = 32 * tl + 16 * hf >= vis ? 1.0f : v < kLeastBlockScale ? kLeastBlockScale : v;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float p0 = __builtin_amdgcn_exp2f(x[tl][4 * hf + 2 * k] - m);
          float p1 = __builtin_amdgcn_exp2f(x[tl][4 * hf + 2 * k + 1] - m);
          if constexpr (FMT != kBlockBf16) p0 *= v, p1 *= v;
          pop[2 * hf + k] = pack_bf16x2(p0, p1);
          part_l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pop[2 * hf + k]),
                                                   __builtin_bit_cast(bf16x2_t, 0x3f803f80u), part_l, false);
        }
        l = FMT != kBlockBf16 ? fmaf(part_l, __builtin_amdgcn_rcpf(v), l) : l + part_l;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma_16x16x32_bf16(o.v_op[tl][dt], pop, acc[dt]);
    }
    l = sum_across_groups(l);
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) nan = nan || acc[dt][r] != acc[dt][r];
    const bool redo = __builtin_amdgcn_readfirstlane((int)(check && __any(nan && live)));
    if (live && !redo) {
      const int64_t at = ((int64_t)e * a.segs + seg) * a.H + g * a.group + hc;
      // A lane holds D / 4 elements in a row, so that a store of all lanes' quarters would touch 64 lines: four lane groups
      // transpose their quads of elements among each other, and each stores one of four that follow each other (107 -> 102 us).
      float* wo = a.ws_o + at * D;
#pragma unroll
      for (int c0 = 0; c0 < D / 16; c0 += 4) {
        uint32_t y[4][4];  // [quad c0 + o of the lane's, its element], then [quad c0 + g4 of lane group o's, ..]
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
          for (int o = 0; o < 4; ++o) y[o][w] = __float_as_uint(acc[(4 * (c0 + o) + w) % VE][(4 * (c0 + o) + w) / VE]);
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const auto z = __builtin_amdgcn_permlane32_swap(y[o][w], y[o + 2][w], false, false);
            y[o][w] = (uint32_t)z[0], y[o + 2][w] = (uint32_t)z[1];
          }
#pragma unroll
          for (int o = 0; o < 4; o += 2) {
            const auto z = __builtin_amdgcn_permlane16_swap(y[o][w], y[o + 1][w], false, false);
            y[o][w] = (uint32_t)z[0], y[o + 1][w] = (uint32_t)z[1];
          }
        }
#pragma unroll
        for (int o = 0; o < 4; ++o)
          *reinterpret_cast<uint4*>(wo + D / 4 * o + 4 * (c0 + g4)) = make_uint4(y[o][0], y[o][1], y[o][2], y[o][3]);
      }
      if (g4 == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * at) = make_float2(m, l);
    }
    return !redo;
  };

  const int32_t tpi = 16 / a.group;
  constexpr int kStep = 64 * kPageWaves;
  const int32_t entries = t_end * a.n_blocks, step_t = kStep / a.n_blocks, step_i = kStep % a.n_blocks;
  int32_t t = t_first + tid / a.n_blocks, i = tid % a.n_blocks;
  for (int32_t e0 = t_first * a.n_blocks; e0 < entries; e0 += kPageStep) {  // uniform in the workgroup
    int32_t named[kPageScan];
#pragma unroll
    for (int u = 0; u < kPageScan; ++u) {
      named[u] = t < t_end ? a.blocks[((int64_t)t * a.G + g) * a.n_blocks + i] : -1;
      t += step_t, i += step_i;
      if (i >= a.n_blocks) i -= a.n_blocks, ++t;
    }
#pragma unroll
    for (int u = 0; u < kPageScan; ++u)
      if (named[u] >= c0 && named[u] < c0 + kPageWaves)
        sm_hit[atomicAdd(&sm_hits, 1)] = (u * kStep + tid) * kPageWaves + named[u] - c0;
    __syncthreads();
    for (int32_t h = tid; h < sm_hits; h += kStep) {
      const int32_t c = sm_hit[h] % kPageWaves, e = e0 + sm_hit[h] / kPageWaves, th = e / a.n_blocks;
      const int32_t r = a.rows[th], vis = seen(th, c);
      if (r != row || vis <= 0 || sm_page[c] < 0) continue;
      if (vis >= keys) {
        sm_e[c][atomicAdd(&sm_n[c][0], 1)] = e;
      } else {
        sm_e[c][kPageList - 1 - atomicAdd(&sm_n[c][1], 1)] = e;
        atomicMax(&sm_vis[c], vis);
      }
    }
    __syncthreads();
    bool flush = e0 + kPageStep >= entries;
#pragma unroll
    for (int c = 0; c < kPageWaves; ++c) flush = flush || sm_n[c][0] + sm_n[c][1] > kPageList - kPageStep;
    if (tid == 0) sm_hits = 0;
    if (flush) {
      // The wave's next batch, of its own page first, then of the others: page c, its keys that V holds, entries from f on. After
      // one with a NaN the same entry by entry (alone >= 0).
      int32_t k = 0, c = 0, vis = 0, part = 0, f = 0, n = 0, alone = -1;
      auto next = [&](bool ok) {
        if (!ok) {
          alone = 0;
        } else if (alone < 0 || ++alone >= n) {
          alone = -1, n = 0;
          for (; k < 2 * kPageWaves; ++k) {
            c = (wave + k / 2) % kPageWaves, part = k & 1;
            const int32_t count = __builtin_amdgcn_readfirstlane(sm_n[c][part]);
            if (count == 0) continue;
            f = __builtin_amdgcn_readfirstlane(lane == 0 ? atomicAdd(&sm_taken[c][part], tpi) : 0);
            n = min(tpi, count - f);
            if (n > 0) break;
          }
          if (k == 2 * kPageWaves) return;
        }
        vis = __builtin_amdgcn_readfirstlane(alone >= 0 ? seen(sm_e[c][kPageList - 1 - f - alone] / a.n_blocks, c)
                                             : part     ? sm_vis[c]
                                                        : keys);
      };
      next(true);
      while (k < 2 * kPageWaves) {
        Keys o;
        const int32_t at_c = c, at_vis = vis;
        load(o, c, vis);
        do {
          next(attend(o, c, part, f + max(alone, 0), alone < 0 ? n : 1, part > 0 && alone < 0));
        } while (k < 2 * kPageWaves && c == at_c && vis == at_vis);
      }
      __syncthreads();
      if (tid < 2 * kPageWaves) (&sm_n[0][0])[tid] = 0, (&sm_taken[0][0])[tid] = 0;
      if (tid < kPageWaves) sm_vis[tid] = 0;
    }
    __syncthreads();
  }
}

// Merge of a query's splits, one workgroup per (query, head): out = sum_s e_s o_s / (sum_s e_s l_s + e_sink), e_s =
// exp2(m_s - M). D / 4 lanes take a split's row in 16-byte pieces, 1024 / D splits at a time, each such group of lanes with a
// running (M, l, o) of its own; the groups are merged in LDS.
template <int D>
__global__ __launch_bounds__(256) void block_combine_kernel(BlockDecodeArgs a) {
  constexpr int LR = D / 4, NG = 256 / LR, CH = 4;
  const int32_t t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, gi = tid / LR, d = 4 * (tid % LR);
  const int32_t ns = a.splits;
  const int64_t at0 = (int64_t)t * ns * a.H + h;
  const float* wo = a.ws_o + at0 * D + d;
  const float* ml = a.ws_ml + 2 * at0;
  float M = kNegBig, l = 0.0f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int32_t s0 = gi; s0 < ns; s0 += NG * CH) {
    f32x4_t x[CH];
    float2 w[CH];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int64_t s = (int64_t)min(s0 + NG * k, ns - 1) * a.H;
      x[k] = *reinterpret_cast<const f32x4_t*>(wo + s * D);
      w[k] = *reinterpret_cast<const float2*>(ml + 2 * s);
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (s0 + NG * k < ns) {
        const float m = fmaxf(M, w[k].x), e0 = __builtin_amdgcn_exp2f(M - m), e1 = __builtin_amdgcn_exp2f(w[k].x - m);
        l = l * e0 + w[k].y * e1;
        o = o * e0 + x[k] * e1;
        M = m;
      }
    }
  }
  __shared__ __attribute__((aligned(16))) float sm_o[NG][D];
  __shared__ float sm_m[NG], sm_l[NG];
  *reinterpret_cast<f32x4_t*>(&sm_o[gi][d]) = o;
  if (tid % LR == 0) sm_m[gi] = M, sm_l[gi] = l;
  __syncthreads();
  if (tid >= D / 2) return;
  float T = kNegBig, den = 0.0f, a0 = 0.0f, a1 = 0.0f;
#pragma unroll
  for (int k = 0; k < NG; ++k) T = fmaxf(T, sm_m[k]);
#pragma unroll
  for (int k = 0; k < NG; ++k) {
    const float e = __builtin_amdgcn_exp2f(sm_m[k] - T);
    den += e * sm_l[k];
    a0 += e * sm_o[k][2 * tid], a1 += e * sm_o[k][2 * tid + 1];
  }
  if (a.sinks) den += __builtin_amdgcn_exp2f(a.sinks[h] * kLog2e - T);
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  reinterpret_cast<uint32_t*>(a.out + ((int64_t)t * a.H + h) * D)[tid] =
      f32_to_bf16_bits(a0 * inv) | f32_to_bf16_bits(a1 * inv) << 16;
}

// The same of the partials page by page, one wave per (query, head): split s is the keys 64 (s % segs) .. of the page that entry
// s / segs of the list names, and was written where the query sees some of them. 64 splits at a time, each lane looks one up;
// D / 4 lanes take a split's row. (2 x 256 queries of 16 pages, 16 heads of 128: a workgroup per (query, head), each lane with
// look-ups of its own, 22 us; 13 so.)
template <int D>
__global__ __launch_bounds__(256) void block_pages_combine_kernel(BlockDecodeArgs a) {
  constexpr int LR = D / 4, NG = 64 / LR, CH = 8;
  const int lane = threadIdx.x & 63, gi = lane / LR, d = 4 * (lane % LR);
  const int32_t item = (int32_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (item >= a.T * a.H) return;
  const int32_t t = item / a.H, h = item - t * a.H, ns = a.splits, row = a.rows[t];
  const int32_t L = row >= 0 && row < a.table_rows ? block_len(a, a.seq_lens[t]) : 0;
  const int32_t* list = a.blocks + ((int64_t)t * a.G + h / a.group) * a.n_blocks;
  const int64_t at0 = (int64_t)t * ns * a.H + h;
  const float* wo = a.ws_o + at0 * D + d;
  const float* ml = a.ws_ml + 2 * at0;
  float M = kNegBig, l = 0.0f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int32_t s0 = 0; s0 < ns; s0 += 64) {  // uniform
    const int32_t s = s0 + lane, e = s / a.segs;
    float m = kNegBig, sum = 0.0f;
    bool written = false;
    if (s < ns) {
      const int32_t c = list[e];
      const float2 w = *reinterpret_cast<const float2*>(ml + (int64_t)2 * s * a.H);
      if (c >= 0 && c < a.table_width && L - c * a.P - 64 * (s - e * a.segs) > 0) {
        const int32_t page = a.table[(int64_t)row * a.table_stride + c];
        written = page >= 0 && (int64_t)page < a.num_blocks && w.y != 0.0f;
        if (written) m = w.x, sum = w.y;
      }
    }
    const float m_new = fmaxf(M, wave_max(m)), keep = __builtin_amdgcn_exp2f(M - m_new);
    const float f = __builtin_amdgcn_exp2f(m - m_new);
    M = m_new;
    l = l * keep + wave_sum(sum * f);
    o *= keep;
    const uint64_t some = __ballot(written);
    for (int32_t i0 = 0; i0 < min(ns - s0, 64); i0 += NG * CH) {
      f32x4_t x[CH];
#pragma unroll
      for (int k = 0; k < CH; ++k)
        x[k] = *reinterpret_cast<const f32x4_t*>(wo + (int64_t)min(s0 + i0 + NG * k + gi, ns - 1) * a.H * D);
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int32_t i = i0 + NG * k + gi;  // below 64 + NG * CH
        const float fi = __shfl(f, i & 63);
        if (i < 64 && (some >> (i & 63) & 1)) o += x[k] * fi;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = D == 128 ? xor32_partner_sum(o[r]) : sum_across_groups(o[r]);
  if (a.sinks) l += __builtin_amdgcn_exp2f(a.sinks[h] * kLog2e - M);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (gi == 0)
    *reinterpret_cast<uint2*>(a.out + ((int64_t)t * a.H + h) * D + d) =
        make_uint2(f32_to_bf16_bits(o[0] * inv) | f32_to_bf16_bits(o[1] * inv) << 16,
                   f32_to_bf16_bits(o[2] * inv) | f32_to_bf16_bits(o[3] * inv) << 16);
}

template <int D, int FMT, bool SEL, bool SHARED>
static void launch_block_decode(const BlockDecodeArgs& a, int32_t waves, hipStream_t s) {
  const dim3 grid((uint32_t)(a.T * a.splits * a.G));
  if (a.splits > 1) {
    if (waves == 4) hipLaunchKernelGGL((block_decode_kernel<D, FMT, SEL, true, 4, SHARED>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((block_decode_kernel<D, FMT, SEL, true, 8, SHARED>), grid, dim3(512), 0, s, a);
    hipLaunchKernelGGL((block_combine_kernel<D>), dim3(a.T, a.H), dim3(256), 0, s, a);
  } else {
    if (waves == 4) hipLaunchKernelGGL((block_decode_kernel<D, FMT, SEL, false, 4, SHARED>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((block_decode_kernel<D, FMT, SEL, false, 8, SHARED>), grid, dim3(512), 0, s, a);
  }
}

template <int D, int FMT>
static void launch_block_decode_form(const BlockDecodeArgs& a, int32_t waves, hipStream_t s) {
  if (a.segs > 0) {
    const int32_t quads = (a.table_width + kPageWaves - 1) / kPageWaves;
    hipLaunchKernelGGL((block_pages_kernel<D, FMT>), dim3((uint32_t)(a.table_rows * quads * a.segs * a.G)), dim3(64 * kPageWaves),
                       0, s, a);
    hipLaunchKernelGGL((block_pages_combine_kernel<D>), dim3((uint32_t)((a.T * a.H + 3) / 4)), dim3(256), 0, s, a);
  } else if (a.rows) {
    if (a.blocks) launch_block_decode<D, FMT, true, true>(a, waves, s);
    else launch_block_decode<D, FMT, false, true>(a, waves, s);
  } else {
    if (a.blocks) launch_block_decode<D, FMT, true, false>(a, waves, s);
    else launch_block_decode<D, FMT, false, false>(a, waves, s);
  }
}

template <int D>
static void launch_block_decode_format(const BlockDecodeArgs& a, int32_t dtype, int32_t waves, hipStream_t s) {
  if (dtype == SNA_DTYPE_BF16) launch_block_decode_form<D, kBlockBf16>(a, waves, s);
  else if (dtype == SNA_DTYPE_INT8) launch_block_decode_form<D, kBlockInt8>(a, waves, s);
  else launch_block_decode_form<D, kBlockFp8>(a, waves, s);
}

// How a launch shares its keys out: waves a workgroup, and the splits of a query, each an even share of its own tiles (the
// table's width says little about them: it is what a graph is captured for).
//   Queries of equal work (lists of one length; a single query): 8 waves and one round of workgroups, so the fewest partials
//   (32 queries of 2048 selected FP8 keys, 32 / 8 heads of 128: whole rows on 8 waves 27.0 us, two splits on 4 waves 32.3, on
//   8 32.3; one row of 131071 int8 keys: 32 splits on 8 waves 48.6, 64 on 4 50.0, 32 on 4 60.0; both sides before K went
//   through the L2, 24.7 and 47.8 since).
//   Rows of unequal lengths: 4 waves, some 1024 workgroups, so that the short ones even the long ones out (24 rows of 1000 to
//   4096 keys: 2, 4 and 8 splits on 4 waves 40.5, 33.3, 34.6 us, on 8 waves 43.2, 40.4, 47.7; 40 of 200 to 8000: whole 128, 3
//   splits 85, 6 78; 16 of 4096: 2, 4, 8, 16 splits 31.6, 28.5, 28.9, 33.5). Where whole rows fill the card they stay whole (64
//   rows of 4096: 82.4, two splits 85.7, four 84.9; 56 such rows 74.0, 80.4, 75.1; of 1024 keys 25.7, 29.8, 30.5), above that up to
//   three rounds of them are halved (70 of 100 to 6000: 131 and 103; 100 of 500 to 2000: 61.8 and 60.8). Ragged rows pay for
//   staying whole: 64 of 100 to 6000 whole, two and four splits 91.2, 91.5, 77.7, in bf16 158, 145, 134; 63 of 500 and one of 16384
//   217, 160, 87. What a launch knows beforehand does not tell the two kinds apart.
// The card holds 512 workgroups of 4 waves at head dim 128 (FP8 768), 1024 at 64. A split has 4 tiles at the least.
// table_rows: of a call whose queries share rows and take listed pages (rows and blocks given), else 0.
struct BlockShape {
  int32_t waves, splits, segs;
};
static BlockShape block_shape(int32_t T, int32_t H, int32_t G, int32_t head_dim, int32_t page_size, int32_t table_width,
                              int32_t table_rows, int32_t window, int32_t n_blocks, int32_t esz) {
  if (table_rows > 0 && n_blocks > 0) {
    // Page by page: for many queries, which a page is worth finding them for, with groups of three at most, since a partial is
    // written for each head but K and V are read once a group. One by one | page by page, us, each query 16 pages of 64, heads
    // of 128, rows of up to 16384 keys:
    //   bf16, 8 KV heads, group 2: 2 x 64 queries 44 | 54, 2 x 128 80 | 70, 2 x 256 151 | 94, 2 x 1024 579 | 247, 4 x 64 86 | 90,
    //   8 x 128 307 | 200, 1 x 1024 of 65536 keys 447 | 217; 2 KV heads, 2 x 512 77 | 77;
    //   8 KV heads, group 1 at 2 x 256 150 | 74; group 3 at 2 x 128 80 | 81, 2 x 256 152 | 119; group 4 at 2 x 1024 292 | 321;
    //   FP8, group 2: 2 x 256 100 | 81, 2 x 1024 373 | 231, 2 KV heads at 2 x 512 54 | 72, group 3 at 2 x 256 100 | 106, 2 x 1024
    //   377 | 356; int8 at 2 x 1024: group 2 507 | 231, group 3 511 | 359;
    //   pages of 128 at 2 x 512 294 | 139, of 32 at 2 x 256 86 | 111; heads of 64 at 2 x 512 176 | 90.
    // A workgroup reads all of a row's lists for four pages: not for tables much wider than a page's keys are worth. The partials
    // stay within 1 GiB.
    const int64_t segs = (page_size + 63) / 64, listed = (int64_t)T * n_blocks;
    const int64_t partials = listed * segs * H * (head_dim + 2) * 4;
    if (H <= 3 * G && page_size >= 64 && listed * G * esz >= (H <= 2 * G ? 1 : 2) << 16 &&
        listed >= 8 * (int64_t)table_rows * table_width && table_width <= 16 * (int64_t)page_size && partials <= 1 << 30)
      return {4, (int32_t)(n_blocks * segs), (int32_t)segs};
  }
  const int64_t keys = (int64_t)(n_blocks > 0 ? n_blocks : table_width) * page_size;
  const int64_t tiles = ((window > 0 ? std::min<int64_t>(keys, (int64_t)window + 31) : keys) + 31) / 32;
  const int64_t base = (int64_t)T * G, slots = head_dim == 64 ? 1024 : 512;
  const bool even = n_blocks > 0 || T == 1, full = base >= slots * 7 / 8;
  int64_t n = 1;
  if (even) n = slots / 2 / base;
  else if (!full) n = 1024 / base;
  else if (base > slots && base < 3 * slots) n = 2;
  n = std::max<int64_t>(1, std::min<int64_t>({n, tiles / 4, (int64_t)256}));
  return {even && !full ? 8 : 4, (int32_t)n, 0};
}

}  // namespace sna

using namespace sna;

extern "C" int64_t sna_block_decode_workspace_bytes(int32_t T, int32_t num_q_heads, int32_t num_kv_heads,
                                                    int32_t head_dim, int32_t page_size, int32_t table_width,
                                                    int32_t table_rows, int32_t window, int32_t n_blocks,
                                                    int32_t cache_dtype) {
  if (T < 1 || num_q_heads < 1 || num_kv_heads < 1 || head_dim < 1 || page_size < 1 || table_width < 1 || window < 0 ||
      n_blocks < 0 || table_rows < 0)
    return 0;
  const BlockShape b = block_shape(T, num_q_heads, num_kv_heads, head_dim, page_size, table_width, table_rows, window, n_blocks,
                                   cache_dtype == SNA_DTYPE_BF16 ? 2 : 1);
  return b.splits > 1 || b.segs > 0 ? (int64_t)T * b.splits * num_q_heads * (head_dim + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int sna_paged_decode_blocks(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                                       const float* v_scale, int64_t scale_page_stride, int64_t scale_head_stride,
                                       int32_t scale_tokens, const int32_t* block_table, int64_t table_stride,
                                       int32_t table_width, int32_t table_rows, const int32_t* rows,
                                       const int32_t* seq_lens, const int32_t* blocks, int32_t n_blocks,
                                       const float* sinks, int32_t window, float sm_scale, void* out, int32_t T,
                                       int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                       int64_t num_blocks, int32_t cache_dtype, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  ApiGuard guard;
  const char* what = blocks ? "paged_decode_selected" : "paged_decode_blocks";
  if (T < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads || window < 0 || num_blocks < 1 ||
      table_width < 1 || table_rows < 0 || table_stride < table_width || n_blocks < 0 || !(sm_scale > 0.0f))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: bad sizes (T %d, heads %d / %d, window %d, blocks %lld, table %d x %d, "
                "stride %lld, list %d) or scale %g", what, T, num_q_heads, num_kv_heads, window, (long long)num_blocks,
                table_rows, table_width, (long long)table_stride, n_blocks, (double)sm_scale);
  const int32_t group = num_q_heads / num_kv_heads;
  if (group > 16) return fail(SNA_ERR_UNSUPPORTED, "%s: GQA group %d > 16 (a workgroup covers 16 query heads)", what, group);
  if (head_dim != 64 && head_dim != 128)
    return fail(SNA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  if (page_size < 16 || page_size % 16 || page_size > SNA_MAX_BLOCK_PAGE)
    return fail(SNA_ERR_UNSUPPORTED, "%s: page_size %d (a multiple of 16, at most %d)", what, page_size,
                SNA_MAX_BLOCK_PAGE);
  if (cache_dtype != SNA_DTYPE_BF16 && cache_dtype != SNA_DTYPE_FP8_E4M3FN && cache_dtype != SNA_DTYPE_INT8)
    return fail(SNA_ERR_UNSUPPORTED, "%s: cache dtype %d (bf16, FP8 e4m3fn or int8)", what, cache_dtype);
  const bool scaled = cache_dtype != SNA_DTYPE_BF16;
  if (scaled && (scale_tokens < 16 || scale_tokens % 16 || page_size % scale_tokens || scale_page_stride < 0 ||
                 scale_head_stride < 0))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: a scale for every %d tokens (a multiple of 16 that divides the page of "
                "%d), strides %lld and %lld", what, scale_tokens, page_size, (long long)scale_page_stride,
                (long long)scale_head_stride);
  if (blocks && (n_blocks < 1 || window > 0))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: a list of %d pages, window %d (none)", what, n_blocks, window);
  const int64_t keys = (int64_t)(blocks ? n_blocks : table_width) * page_size;
  if (keys > INT32_MAX - 4096 || (int64_t)table_width * page_size > INT32_MAX - 4096)
    return fail(SNA_ERR_UNSUPPORTED, "%s: %lld keys of a query, a table of %lld (positions are 32 bits)", what,
                (long long)keys, (long long)table_width * page_size);
  if (T == 0) return SNA_OK;
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !out || (scaled && (!k_scale || !v_scale)))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(out, 4))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: q and the caches must be 16-byte aligned, out 4-byte", what);
  if (table_rows < 1) return fail(SNA_ERR_INVALID_ARGUMENT, "%s: a table of no rows", what);
  if (!rows && table_rows < T)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d queries over a table of %d rows", what, T, table_rows);
  if (num_q_heads > 65535) return fail(SNA_ERR_INVALID_ARGUMENT, "%s: grid too large", what);

  BlockDecodeArgs a;
  a.q = (const uint16_t*)q;
  a.k_cache = (const uint8_t*)k_cache;
  a.v_cache = (const uint8_t*)v_cache;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.scale_page = scale_page_stride;
  a.scale_head = scale_head_stride;
  const int32_t per = scaled ? scale_tokens / 16 : page_size / 16;
  a.sub_magic = scaled && scale_tokens < page_size ? (65536 + per - 1) / per : 0;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.table_rows = table_rows;
  a.rows = rows;
  a.seq_lens = seq_lens;
  a.blocks = blocks;
  a.n_blocks = blocks ? n_blocks : 0;
  a.sinks = sinks;
  a.T = T;
  a.H = num_q_heads;
  a.G = num_kv_heads;
  a.group = group;
  a.P = page_size;
  a.halves = page_size / 16;
  a.num_blocks = num_blocks;
  a.window = window;
  a.sm_scale = sm_scale;
  const BlockShape shape = block_shape(T, num_q_heads, num_kv_heads, head_dim, page_size, table_width,
                                       rows && blocks ? table_rows : 0, window, a.n_blocks, scaled ? 1 : 2);
  a.splits = shape.splits;
  a.segs = shape.segs;
  a.ws_o = a.ws_ml = nullptr;
  if (a.splits > 1 || a.segs > 0) {
    const int64_t rows_n = (int64_t)T * a.splits * num_q_heads, need = rows_n * (head_dim + 2) * (int64_t)sizeof(float);
    if (!workspace || workspace_bytes < need)
      return fail(SNA_ERR_WORKSPACE, "%s: workspace of %lld bytes, the splits need %lld", what,
                  (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!aligned(workspace, 16))
      return fail(SNA_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
    a.ws_o = (float*)workspace;
    a.ws_ml = a.ws_o + rows_n * head_dim;
  }
  const int64_t items = a.segs > 0 ? (int64_t)table_rows * table_width * a.segs : (int64_t)T * a.splits;
  if (items * num_kv_heads >= 1 << 23)  // (a grid has under 2^32 threads)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d queries exceed the grid", what, T);
  a.out = (uint16_t*)out;
  const hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) launch_block_decode_format<128>(a, cache_dtype, shape.waves, s);
  else launch_block_decode_format<64>(a, cache_dtype, shape.waves, s);
  return check_launch(what);
}
