// Eviction of cached tokens by weight: which tokens of a row each KV head keeps (select), and their K/V rows moved
// together (compact). The pool's pages are head-major, so every KV head keeps a set of its own: the heads of a row share
// the block table and the count, not the tokens.
//
//   select   Row r of L tokens keeps, where L > keep, its first `first` tokens, its last `recent` ones, and of the rest
//            the keep - first - recent of the largest weights (ties: the lowest position; a NaN ranks above every number),
//            in ascending order; else all L. The threshold weight is found exactly, by three histogram passes over the
//            weights' order-preserving 32-bit keys (11, 11 and 10 bits, integer counts); the positions at or above it are
//            then written by prefix counts. One workgroup per (row, KV head) does it all while it holds the row's
//            candidates in registers (16384); a longer row takes one for every 16384, and a launch a pass.
//   compact  Kept token i goes to position i of the row's (or another table's) pages. In place a target lies at or before
//            its source, and at or after every earlier target, so one workgroup may walk a row's tokens in order,
//            reading a whole tile before it writes it, without a copy elsewhere; the columns of a head's rows are
//            independent, so several workgroups share a row by columns, and K and V are apart. To other pages nothing
//            orders the tokens and the tiles go to workgroups of their own.
// Both are bound by memory (latency for few rows): select reads 4 bytes a token and head, compact reads and writes the
// kept rows. Measured (us, 8 KV heads): select of one row of 1000 tokens 7.6 (a chain of 3 histograms on one CU), of 32 rows
// of up to 8192 13-14, of 4 rows of 50001 to 131072 7 + 9 + 10 + 14 (three passes and the writer, each one round trip and the
// row's histograms; in place 10 more for the weights' way back); compact to other pages of 32 x 1024 e4m3fn tokens of 128
// 24-26, 5.2-5.6 TB/s read and written, of 4 x 8192 bf16 62, 4.3 TB/s (a plain copy: 4.8), in place 26-28 and 94-99 (a
// workgroup reads a tile, waits, writes it, and only then asks for the next).
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
constexpr int kSelectBins = 2048, kSelectCopies = 4;  // a pass's histogram: a copy for every 4th lane,
constexpr int kSelectCopy = kSelectBins + 16;         // 16 banks apart
constexpr int kSelectMost = 16;                       // keys a thread holds, at most
constexpr int32_t kSelectSegment = kSelectThreads * kSelectMost;  // candidates of a workgroup
// Pass p looks at a key's bits [kSelectShift[p], kSelectShift[p - 1]).
__device__ constexpr int kSelectShift[3] = {21, 10, 0};
__device__ constexpr int kSelectBits[3] = {11, 11, 10};

// A row's candidates [lo, hi) (whole: there is nothing to choose).
struct SelectRow {
  const float* w;
  int32_t L, n, lo, hi;
  bool whole;  // every token is kept
};
__device__ __forceinline__ SelectRow select_row(const SelectArgs& a, int32_t g, int32_t r) {
  SelectRow s;
  s.w = a.weights + r * a.w_row + g * a.w_head;
  s.L = min(max(a.lens[r], 0), a.width);
  s.n = min(s.L, a.keep);
  s.whole = s.L <= a.keep;
  s.lo = a.first, s.hi = s.L - a.recent;
  return s;
}
// The segment of them that a workgroup holds: E a thread, in position order wave by wave, 64 at a time. A place past the
// candidates has key 0, below that of every weight: it is never among the largest.
template <int E>
struct SelectKeys {
  float x[E];
  uint32_t key[E];
  int32_t first;  // the lane's first place
  __device__ __forceinline__ void load(const SelectRow& s, int32_t segment) {
    first = s.lo + (segment * (kSelectThreads / 64) + (int)(threadIdx.x >> 6)) * (64 * E) + (int)(threadIdx.x & 63);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = first + 64 * e < s.hi ? s.w[first + 64 * e] : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = first + 64 * e < s.hi ? weight_key(x[e]) : 0u;
  }
};

struct SelectShared {
  uint32_t hist[kSelectCopies * kSelectCopy];
  uint32_t wave[16], other[16], third[16], pick[3];
};
__device__ __forceinline__ void select_clear(SelectShared& sm) {
  for (int i = threadIdx.x; i < kSelectCopies * kSelectCopy / 4; i += kSelectThreads)
    reinterpret_cast<uint4*>(sm.hist)[i] = make_uint4(0, 0, 0, 0);
}
template <int E>
__device__ __forceinline__ void select_count(SelectShared& sm, const SelectKeys<E>& k, int pass, uint32_t T) {
  uint32_t* const mine = sm.hist + (threadIdx.x & (kSelectCopies - 1)) * kSelectCopy;
  const int shift = kSelectShift[pass], bits = kSelectBits[pass];
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (pass == 0 ? k.key[e] != 0 : k.key[e] >> (shift + bits) == T)
      atomicAdd(&mine[k.key[e] >> shift & ((1u << bits) - 1)], 1u);
}
// Thread t's bins of the histogram, 2047 - 2 t and the one below it, copies added.
__device__ __forceinline__ uint2 select_bins(const SelectShared& sm) {
  uint2 h = make_uint2(0, 0);
#pragma unroll
  for (int c = 0; c < kSelectCopies; ++c) {
    const uint2 v = *reinterpret_cast<const uint2*>(sm.hist + c * kSelectCopy + kSelectBins - 2 - 2 * (int)threadIdx.x);
    h.x += v.y, h.y += v.x;
  }
  return h;
}
// Over the workgroup's bins, thread t holding counts h of bins 2047 - 2 t and below: the bin of the need-th largest key, the
// keys in bins above it and its own, in sm.pick after the next barrier.
__device__ __forceinline__ void select_find(SelectShared& sm, uint2 h, uint32_t need) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t total;
  const uint32_t incl = (uint32_t)wave_incl_scan_i32((int32_t)(h.x + h.y), &total);
  if (lane == 0) sm.wave[wave] = (uint32_t)total;
  __syncthreads();
  uint32_t before = incl - (h.x + h.y);
#pragma unroll
  for (int i = 0; i < 16; ++i) before += i < wave ? sm.wave[i] : 0u;
  const uint32_t top = (uint32_t)(kSelectBins - 1 - 2 * tid);
  if (before < need && need <= before + h.x) sm.pick[0] = top, sm.pick[1] = before, sm.pick[2] = h.x;
  before += h.x;
  if (before < need && need <= before + h.y) sm.pick[0] = top - 1, sm.pick[1] = before, sm.pick[2] = h.y;
}
// Keys whose bits from `shift` on are above T, and the first `need` of those equal to it (`above` and `equal` of either lie
// in segments before), go to kept from a.first on in position order, their weights to out (where there is one).
template <int E>
__device__ __forceinline__ void select_write(SelectShared& sm, const SelectArgs& a, const SelectKeys<E>& k, uint32_t T,
                                             int shift, uint32_t need, uint32_t above, uint32_t equal, int32_t* kept,
                                             float* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t n_above = 0, n_equal = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    n_above += (uint32_t)__popcll(__ballot(k.key[e] >> shift > T));
    n_equal += (uint32_t)__popcll(__ballot(k.key[e] >> shift == T));
  }
  if (lane == 0) sm.wave[wave] = n_above, sm.other[wave] = n_equal;
  __syncthreads();  // (also: the segment is read, so its places may be written)
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < wave) above += sm.wave[i], equal += sm.other[i];
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool gt = k.key[e] >> shift > T, eq = k.key[e] >> shift == T;
    const uint64_t mg = __ballot(gt), me = __ballot(eq);
    const uint32_t pe = equal + (uint32_t)__popcll(me & below);
    if (gt || (eq && pe < need)) {
      const uint32_t to = (uint32_t)a.first + above + (uint32_t)__popcll(mg & below) + min(pe, need);
      kept[to] = k.first + 64 * e;
      if (out) out[to] = k.x[e];
    }
    above += (uint32_t)__popcll(mg), equal += (uint32_t)__popcll(me);
  }
}
// What a row keeps without choosing: all of a short row, the first tokens of another. (out may be the weights themselves:
// then these weights are in place.)
__device__ __forceinline__ void select_first(const SelectArgs& a, const SelectRow& s, int32_t* kept, float* out) {
  for (int32_t i = threadIdx.x; i < (s.whole ? a.keep : a.first); i += kSelectThreads) {
    kept[i] = i < s.L ? i : -1;
    if (out && out != s.w && i < s.L) out[i] = s.w[i];
  }
}
// ... and the last ones: a tile is read before it is written, for out may be the weights themselves, and their candidates
// have been read.
__device__ __forceinline__ void select_recent(const SelectArgs& a, const SelectRow& s, int32_t* kept, float* out) {
  const int32_t to = a.keep - a.recent;
  for (int32_t i0 = 0; i0 < a.recent; i0 += kSelectThreads) {  // uniform
    const int32_t i = i0 + threadIdx.x;
    const float v = i < a.recent && out ? s.w[s.hi + i] : 0.0f;
    wait_vmcnt<0>();
    __syncthreads();
    if (i < a.recent) {
      kept[to + i] = s.hi + i;
      if (out) out[to + i] = v;
    }
  }
}

// A row whose candidates one workgroup holds.
template <int E>
__global__ __launch_bounds__(kSelectThreads) void select_row_kernel(SelectArgs a) {
  __shared__ SelectShared sm;
  const int32_t g = blockIdx.x, r = blockIdx.y;
  const SelectRow s = select_row(a, g, r);
  int32_t* const kept = a.kept + ((int64_t)r * a.G + g) * a.keep;
  float* const out = a.out ? a.out + r * a.o_row + g * a.o_head : nullptr;
  if (g == 0 && threadIdx.x == 0) a.new_lens[r] = s.n;
  select_first(a, s, kept, out);
  uint32_t need = (uint32_t)(a.keep - a.first - a.recent);
  if (!s.whole) {  // uniform
    if (need > 0) {
      SelectKeys<E> x;
      x.load(s, 0);
      select_clear(sm);
      uint32_t T = 0;  // the threshold key's bits found so far
      int pass = 0;
      for (;; ++pass) {
        __syncthreads();  // the histogram is clear
        select_count(sm, x, pass, T);
        __syncthreads();
        const uint2 h = select_bins(sm);
        select_find(sm, h, need);  // (its barrier: the bins are read)
        select_clear(sm);
        __syncthreads();
        T = T << kSelectBits[pass] | sm.pick[0];
        need -= sm.pick[1];
        // (a bin that is taken whole: what is left of its bits does not matter)
        if (pass == 2 || sm.pick[2] == need) break;
      }
      select_write(sm, a, x, T, kSelectShift[pass], need, 0, 0, kept, out);
    }
    select_recent(a, s, kept, out);
  }
  if (out) {
    __syncthreads();
    for (int32_t i = s.n + threadIdx.x; i < a.out_width; i += kSelectThreads) out[i] = 0.0f;
  }
}

// A longer row takes S workgroups of kSelectSegment candidates, one launch a pass: a segment's histogram goes to the
// workspace, the next launch adds the row's up.
struct SelectLong {
  uint32_t* hist[3];  // [R, G, S, 2048]
  uint32_t* above;    // [R, G, S] a segment's keys above the bits found before the last pass
  uint32_t* state;    // [3, R, G, 2] the bits found before each pass, and how many keys are still to be found
  float* kept_w;      // [R, G, keep] the kept weights of a row that is thinned in place, or null
  int32_t S;
};
// The row's histogram of pass `pass` added over its segments (thread t's bins), the threshold's bits and count brought up to
// it, and this segment's keys above its bin added to what is above already. prior: the same of the segments before this one.
struct SelectFound {
  uint32_t T, need, above, prior_above, prior_equal;
};
__device__ __forceinline__ SelectFound select_fold(SelectShared& sm, const SelectArgs& a, const SelectLong& b, int32_t row,
                                                   int32_t seg, int pass) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  SelectFound f;
  const uint32_t* const state = b.state + 2 * ((int64_t)pass * a.R * a.G + row);
  f.T = pass > 0 ? state[0] : 0u;
  f.need = pass > 0 ? state[1] : (uint32_t)(a.keep - a.first - a.recent);
  const uint2* h = reinterpret_cast<const uint2*>(b.hist[pass]) + (int64_t)row * b.S * (kSelectBins / 2) + tid;
  uint2 all = make_uint2(0, 0), mine = make_uint2(0, 0), prior = make_uint2(0, 0);
#pragma unroll 8
  for (int32_t i = 0; i < b.S; ++i) {
    const uint2 v = h[(int64_t)i * (kSelectBins / 2)];
    all.x += v.x, all.y += v.y;
    if (i < seg) prior.x += v.x, prior.y += v.y;
    if (i == seg) mine = v;
  }
  select_find(sm, all, f.need);
  __syncthreads();
  const uint32_t bin = sm.pick[0], top = (uint32_t)(kSelectBins - 1 - 2 * tid);
  f.T = f.T << kSelectBits[pass] | bin;
  f.need -= sm.pick[1];
  // counts above the bin, and in it, of this segment and of those before
  const uint32_t mine_above = (top > bin ? mine.x : 0u) + (top - 1 > bin && top > 0 ? mine.y : 0u);
  const uint32_t prior_above = (top > bin ? prior.x : 0u) + (top - 1 > bin && top > 0 ? prior.y : 0u);
  const uint32_t prior_equal = top == bin ? prior.x : top - 1 == bin ? prior.y : 0u;
  int32_t m, p, e;
  wave_incl_scan_i32((int32_t)mine_above, &m);
  wave_incl_scan_i32((int32_t)prior_above, &p);
  wave_incl_scan_i32((int32_t)prior_equal, &e);
  __syncthreads();  // sm.wave is read
  if (lane == 0) sm.wave[wave] = (uint32_t)m, sm.other[wave] = (uint32_t)p, sm.third[wave] = (uint32_t)e;
  __syncthreads();
  f.above = f.prior_above = f.prior_equal = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) f.above += sm.wave[i], f.prior_above += sm.other[i], f.prior_equal += sm.third[i];
  __syncthreads();
  return f;
}

template <int PASS>
__global__ __launch_bounds__(kSelectThreads) void select_hist_kernel(SelectArgs a, SelectLong b) {
  __shared__ SelectShared sm;
  const int32_t seg = blockIdx.x, g = blockIdx.y, r = blockIdx.z, row = r * a.G + g;
  const SelectRow s = select_row(a, g, r);
  if (s.whole || a.keep == a.first + a.recent) return;  // uniform
  SelectKeys<kSelectMost> x;
  x.load(s, seg);
  uint32_t T = 0;
  if constexpr (PASS > 0) {
    const SelectFound f = select_fold(sm, a, b, row, seg, PASS - 1);
    T = f.T;
    if (threadIdx.x == 0) {
      uint32_t* const above = b.above + (int64_t)row * b.S + seg;
      *above = PASS == 1 ? f.above : *above + f.above;
      uint32_t* const state = b.state + 2 * ((int64_t)PASS * a.R * a.G + row);
      if (seg == 0) state[0] = f.T, state[1] = f.need;
    }
  }
  select_clear(sm);
  __syncthreads();
  select_count(sm, x, PASS, T);
  __syncthreads();
  reinterpret_cast<uint2*>(b.hist[PASS])[((int64_t)row * b.S + seg) * (kSelectBins / 2) + threadIdx.x] = select_bins(sm);
}

__global__ __launch_bounds__(kSelectThreads) void select_write_kernel(SelectArgs a, SelectLong b) {
  __shared__ SelectShared sm;
  const int32_t seg = blockIdx.x, g = blockIdx.y, r = blockIdx.z, row = r * a.G + g;
  const SelectRow s = select_row(a, g, r);
  int32_t* const kept = a.kept + (int64_t)row * a.keep;
  float* out = a.out ? a.out + r * a.o_row + g * a.o_head : nullptr;
  // a row that is thinned in place: its weights go by the workspace, for other workgroups still read them
  if (b.kept_w && !s.whole) out = b.kept_w + (int64_t)row * a.keep;
  if (seg == 0) {
    if (g == 0 && threadIdx.x == 0) a.new_lens[r] = s.n;
    select_first(a, s, kept, out);
  }
  if (seg == 1 && !s.whole) select_recent(a, s, kept, out);  // (there are two at least; another than the first's)
  if (!s.whole && a.keep > a.first + a.recent) {  // uniform
    SelectKeys<kSelectMost> x;
    x.load(s, seg);
    const SelectFound f = select_fold(sm, a, b, row, seg, 2);
    uint32_t above = f.prior_above;
    const uint32_t* const counts = b.above + (int64_t)row * b.S;
#pragma unroll 8
    for (int32_t i = 0; i < seg; ++i) above += counts[i];
    select_write(sm, a, x, f.T, 0, f.need, above, f.prior_equal, kept, out);
  }
  if (out && !(b.kept_w && !s.whole))
    for (int32_t i = s.n + seg * kSelectThreads + threadIdx.x; i < a.out_width; i += b.S * kSelectThreads) out[i] = 0.0f;
}

// The rows thinned in place: their kept weights, then zeros.
__global__ __launch_bounds__(kSelectThreads) void select_place_kernel(SelectArgs a, SelectLong b) {
  const int32_t g = blockIdx.y, r = blockIdx.z;
  const SelectRow s = select_row(a, g, r);
  if (s.whole) return;
  float* const out = a.out + r * a.o_row + g * a.o_head;
  const float* const from = b.kept_w + ((int64_t)r * a.G + g) * a.keep;
  for (int32_t i = blockIdx.x * kSelectThreads + threadIdx.x; i < a.out_width; i += gridDim.x * kSelectThreads)
    out[i] = i < a.keep ? from[i] : 0.0f;
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

// In place a workgroup walks all of a row's tokens (of some columns), and large tiles make it few round trips: 4096 tokens of
// 16384 (one row, 8 KV heads of 128, bf16) took 58 us by 256 threads and 28 by 1024, 8192 of 32768 (4 rows) 142 and 94. To
// other pages the tiles are shared out, and small ones start sooner.
constexpr int kCompactThreads = 256, kCompactInPlace = 1024;
constexpr int kCompactUnroll = 4;  // 16-byte pieces a thread holds
// In place a workgroup takes 128 bytes of a token's row where that makes so many workgroups at least, else 64 where that makes
// so few, else 32. In us by 32 / 64 / 128 (heads of 128): 1024 workgroups of 128 bytes (32 rows, 1024 of 8192 tokens, bf16)
// 134 / 88 / 69, 512 (the same, e4m3fn) 63 / 36 / 26, 128 (4 rows, 8192 of 32768, bf16) 123 / 93 / 126, 128 (8 rows, e4m3fn)
// 18 / 12 / 16, 32 (one row) 21 / 28 / 46. (Whole rows of 256 bytes: 66 where 128 take 69, and 81 where 32 take 21.)
constexpr int64_t kCompactWide = 512, kCompactFew = 128;

template <int THREADS>
__global__ __launch_bounds__(THREADS) void compact_tokens_kernel(CompactArgs a) {
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
  const int32_t per = THREADS * kCompactUnroll >> sh;  // tokens of a tile
  for (int32_t i0 = chunk * per; i0 < a.keep; i0 += a.chunks * per) {  // uniform
    uint4 v[kCompactUnroll];
    uint8_t* to[kCompactUnroll];
#pragma unroll
    for (int u = 0; u < kCompactUnroll; ++u) {
      const int32_t i = i0 + ((u * THREADS + (int32_t)threadIdx.x) >> sh);
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
    if (THREADS == kCompactInPlace) {  // in place: the tile is read before any of it is written
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

namespace {

// The kernels number a row's places by 32 bits: a segment's start behind the first tokens, and a loop's place a step past its
// end, stay below 2^31 with so many.
constexpr int32_t kMostTokens = (1 << 30) - (1 << 15);

// The workspace of a launch whose rows may be longer than one workgroup holds: histograms, counts and thresholds, and the
// kept weights where rows are thinned in place.
int64_t select_segments(int32_t width) { return ((int64_t)width + kSelectSegment - 1) / kSelectSegment; }
int64_t select_bytes(int64_t rows, int32_t width, int32_t keep, bool in_place) {
  if (width <= kSelectSegment) return 0;
  return rows * (select_segments(width) * (3 * kSelectBins + 1) + 3 * 2 + (in_place ? keep : 0)) * 4;
}

}  // namespace

extern "C" int64_t sna_select_workspace_bytes(int32_t R, int32_t num_kv_heads, int32_t width, int32_t keep,
                                              int32_t in_place) {
  if (R < 1 || num_kv_heads < 1 || width < 1 || keep < 1) return 0;
  return select_bytes((int64_t)R * num_kv_heads, width, keep, in_place != 0);
}

namespace {

// Both operators' arguments are checked, and their launches laid out, before either is launched.
struct SelectLaunch {
  SelectArgs a;
  SelectLong b;
  void run(hipStream_t s) const {
    const dim3 block(kSelectThreads), grid(a.G, a.R);
    // (no more keys a thread than the widest row can need: 32 rows of 8192 took 11.7 us with 8 and 14.1 with 16, 64 of 2048
    // 8.9 with 4 and 13.1 with 16)
    if (a.width <= kSelectSegment / 4) {
      hipLaunchKernelGGL((select_row_kernel<kSelectMost / 4>), grid, block, 0, s, a);
    } else if (a.width <= kSelectSegment / 2) {
      hipLaunchKernelGGL((select_row_kernel<kSelectMost / 2>), grid, block, 0, s, a);
    } else if (a.width <= kSelectSegment) {
      hipLaunchKernelGGL((select_row_kernel<kSelectMost>), grid, block, 0, s, a);
    } else {
      const dim3 parts(b.S, a.G, a.R);
      hipLaunchKernelGGL((select_hist_kernel<0>), parts, block, 0, s, a, b);
      hipLaunchKernelGGL((select_hist_kernel<1>), parts, block, 0, s, a, b);
      hipLaunchKernelGGL((select_hist_kernel<2>), parts, block, 0, s, a, b);
      hipLaunchKernelGGL(select_write_kernel, parts, block, 0, s, a, b);
      if (b.kept_w) hipLaunchKernelGGL(select_place_kernel, parts, block, 0, s, a, b);
    }
  }
};

int plan_select(const char* what, const float* weights, int64_t row_stride, int64_t head_stride, int32_t width,
                const int32_t* seq_lens, int32_t R, int32_t num_kv_heads, int32_t keep, int32_t first, int32_t recent,
                int32_t* kept, int32_t* new_lens, float* weights_out, int64_t out_row_stride, int64_t out_head_stride,
                int32_t out_width, void* workspace, int64_t workspace_bytes, SelectLaunch* to) {
  if (R < 0 || num_kv_heads < 1 || width < 1 || keep < 1 || first < 0 || recent < 0 || (int64_t)first + recent > keep ||
      row_stride < width || head_stride < width)
    return fail(SNA_ERR_INVALID_ARGUMENT,
                "%s: bad sizes (R %d, KV heads %d, width %d, strides %lld / %lld, keep %d of which first %d "
                "and recent %d)", what, R, num_kv_heads, width, (long long)row_stride, (long long)head_stride, keep, first,
                recent);
  if (weights_out && (out_width < keep || out_row_stride < out_width || out_head_stride < out_width))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: weights_out of %d columns (strides %lld / %lld) for %d tokens", what,
                out_width, (long long)out_row_stride, (long long)out_head_stride, keep);
  if (width > kMostTokens || keep > kMostTokens || (weights_out && out_width > kMostTokens))
    return fail(SNA_ERR_UNSUPPORTED, "%s: %d columns, %d kept, %d out (at most %d)", what, width, keep, out_width,
                kMostTokens);
  if (R == 0) return SNA_OK;
  if (!weights || !seq_lens || !kept || !new_lens)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (R > 65535 || num_kv_heads > 65535)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d rows x %d KV heads exceed the grid", what, R, num_kv_heads);
  const bool in_place = weights_out == weights && weights_out;
  if (in_place && (out_row_stride != row_stride || out_head_stride != head_stride))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: weights_out is weights with other strides", what);
  const int64_t rows = (int64_t)R * num_kv_heads, need = select_bytes(rows, width, keep, in_place);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(SNA_ERR_WORKSPACE, "%s: workspace of %lld bytes, need %lld", what, (long long)workspace_bytes,
                (long long)need);
  if (need > 0 && !aligned(workspace, 16))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
  SelectArgs& a = to->a;
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
  SelectLong& b = to->b;
  b = {};
  if (need > 0) {
    b.S = (int32_t)select_segments(width);
    const int64_t bins = rows * b.S * kSelectBins;
    b.hist[0] = (uint32_t*)workspace;
    b.hist[1] = b.hist[0] + bins;
    b.hist[2] = b.hist[1] + bins;
    b.above = b.hist[2] + bins;
    b.state = b.above + rows * b.S;
    b.kept_w = in_place ? (float*)(b.state + rows * 6) : nullptr;
  }
  return SNA_OK;
}

struct CompactLaunch {
  CompactArgs a;
  dim3 grid;
  void run(hipStream_t s) const {
    if (a.dst == a.table) hipLaunchKernelGGL((compact_tokens_kernel<kCompactInPlace>), grid, dim3(kCompactInPlace), 0, s, a);
    else hipLaunchKernelGGL((compact_tokens_kernel<kCompactThreads>), grid, dim3(kCompactThreads), 0, s, a);
  }
};

int plan_compact(const char* what, void* k_cache, void* v_cache, int64_t num_blocks, int32_t num_kv_heads,
                 int32_t page_size, int32_t head_dim, int32_t cache_dtype, const int32_t* block_table,
                 int64_t table_stride, int32_t table_width, const int32_t* dst_table, int64_t dst_stride,
                 int32_t dst_width, const int32_t* kept, int32_t R, int32_t keep, CompactLaunch* to) {
  if (R < 0 || num_kv_heads < 1 || num_blocks < 1 || page_size < 1 || keep < 1 || table_width < 1 ||
      table_stride < table_width || (dst_table && (dst_width < 1 || dst_stride < dst_width)))
    return fail(SNA_ERR_INVALID_ARGUMENT,
                "%s: bad sizes (R %d, KV heads %d, blocks %lld, page %d, keep %d, tables %d and %d wide, "
                "strides %lld and %lld)", what, R, num_kv_heads, (long long)num_blocks, page_size, keep, table_width,
                dst_width, (long long)table_stride, (long long)dst_stride);
  if (dst_table == block_table && dst_table) {
    if (R > 1 && dst_stride != table_stride)
      return fail(SNA_ERR_INVALID_ARGUMENT, "%s: dst_table is block_table with another stride", what);
    dst_table = nullptr;  // in place
  }
  if (head_dim != 64 && head_dim != 128)
    return fail(SNA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  if (cache_dtype != SNA_DTYPE_BF16 && cache_dtype != SNA_DTYPE_FP8_E4M3FN && cache_dtype != SNA_DTYPE_FP8_E4M3FN_MUL)
    return fail(SNA_ERR_UNSUPPORTED, "%s: KV dtype %d (FP8 e4m3fn or bf16)", what, cache_dtype);
  if (keep > kMostTokens)
    return fail(SNA_ERR_UNSUPPORTED, "%s: %d kept tokens (at most %d)", what, keep, kMostTokens);
  if (R == 0) return SNA_OK;
  if (!k_cache || !v_cache || !block_table || !kept)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: the caches must be 16-byte aligned", what);
  CompactArgs& a = to->a;
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
  if (dst_table) {
    const int32_t per = kCompactThreads * kCompactUnroll / (a.row_bytes / 16);
    a.slices = 1;
    a.chunks = (int32_t)std::min<int64_t>(((int64_t)keep + per - 1) / per, 65535);
  } else {
    const int64_t columns = 2 * (int64_t)R * num_kv_heads * a.row_bytes;
    const int32_t bytes = columns >= 128 * kCompactWide ? 128 : columns >= 64 * kCompactFew ? 64 : 32;
    a.slices = std::max(a.row_bytes / bytes, 1);
    a.chunks = 1;
  }
  const int64_t y = (int64_t)a.slices * num_kv_heads * 2;
  if (R > 65535 || y > 65535)
    return fail(SNA_ERR_INVALID_ARGUMENT, "%s: %d rows x %d KV heads exceed the grid", what, R, num_kv_heads);
  to->grid = dim3(a.chunks, (unsigned)y, R);
  return SNA_OK;
}

}  // namespace

extern "C" int sna_select_tokens(const float* weights, int64_t row_stride, int64_t head_stride, int32_t width,
                                 const int32_t* seq_lens, int32_t R, int32_t num_kv_heads, int32_t keep, int32_t first,
                                 int32_t recent, int32_t* kept, int32_t* new_lens, float* weights_out,
                                 int64_t out_row_stride, int64_t out_head_stride, int32_t out_width, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  ApiGuard guard;
  SelectLaunch select;
  const int rc = plan_select("select_tokens", weights, row_stride, head_stride, width, seq_lens, R, num_kv_heads, keep,
                             first, recent, kept, new_lens, weights_out, out_row_stride, out_head_stride, out_width,
                             workspace, workspace_bytes, &select);
  if (rc || R == 0) return rc;
  select.run((hipStream_t)stream);
  return check_launch("select_tokens");
}

extern "C" int sna_compact_tokens(void* k_cache, void* v_cache, int64_t num_blocks, int32_t num_kv_heads,
                                  int32_t page_size, int32_t head_dim, int32_t cache_dtype, const int32_t* block_table,
                                  int64_t table_stride, int32_t table_width, const int32_t* dst_table,
                                  int64_t dst_stride, int32_t dst_width, const int32_t* kept, int32_t R, int32_t keep,
                                  void* stream) {
  ApiGuard guard;
  CompactLaunch compact;
  const int rc = plan_compact("compact_tokens", k_cache, v_cache, num_blocks, num_kv_heads, page_size, head_dim,
                              cache_dtype, block_table, table_stride, table_width, dst_table, dst_stride, dst_width,
                              kept, R, keep, &compact);
  if (rc || R == 0) return rc;
  compact.run((hipStream_t)stream);
  return check_launch("compact_tokens");
}

extern "C" int sna_evict_tokens(void* k_cache, void* v_cache, int64_t num_blocks, int32_t num_kv_heads,
                                int32_t page_size, int32_t head_dim, int32_t cache_dtype, const int32_t* block_table,
                                int64_t table_stride, int32_t table_width, const int32_t* dst_table, int64_t dst_stride,
                                int32_t dst_width, const float* weights, int64_t row_stride, int64_t head_stride,
                                int32_t width, const int32_t* seq_lens, int32_t R, int32_t keep, int32_t first,
                                int32_t recent, int32_t* kept, int32_t* new_lens, float* weights_out,
                                int64_t out_row_stride, int64_t out_head_stride, int32_t out_width, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  ApiGuard guard;
  SelectLaunch select;
  CompactLaunch compact;
  int rc = plan_select("evict_tokens", weights, row_stride, head_stride, width, seq_lens, R, num_kv_heads, keep, first,
                       recent, kept, new_lens, weights_out, out_row_stride, out_head_stride, out_width, workspace,
                       workspace_bytes, &select);
  if (rc == SNA_OK)
    rc = plan_compact("evict_tokens", k_cache, v_cache, num_blocks, num_kv_heads, page_size, head_dim, cache_dtype,
                      block_table, table_stride, table_width, dst_table, dst_stride, dst_width, kept, R, keep, &compact);
  if (rc || R == 0) return rc;
  select.run((hipStream_t)stream);
  compact.run((hipStream_t)stream);
  return check_launch("evict_tokens");
}
