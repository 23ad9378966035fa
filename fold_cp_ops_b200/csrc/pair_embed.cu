// Embedding lookup into the pair stream, and the gradient of its table by sorted tokens.
//
// Mathematics.  out[t] = base[t] + scale E[x_t];  dE[v] = scale sum_{t: x_t = v} d_out[t].  An index outside
// [0, rows) stands for "no embedding": it adds nothing and receives no gradient.
//
// Bound.  Forward: HBM, base read and out written once; the table (tens of rows for position bins) stays in L1 and L2.
// Gradient: HBM, d_out read once.  Position bins give some 10^6 tokens to each of a few dozen rows, vocabularies give
// one or two, so the sum is organised by sorted tokens: a stable counting sort of the token numbers by index (up to
// 2048 bins a pass, no comparison, int32 numbers only), then every group of lanes sums the d_out rows of an equal share
// of the SORTED tokens.  A run of equal indices inside one share goes straight to the table; a run that crosses
// shares leaves its pieces in the workspace, and the share in which it begins adds them up afterwards.  No atomics: the
// same bits every time, whatever the distribution.
// Few tokens (or few tokens per table row) skip the sort: one CTA per table row looks through all indices.
#include "pair_stream.cuh"

namespace pair {
namespace {

constexpr int kSlabOcts = 32;            // octs (256 channels) of a row that one warp covers
constexpr int kSortWarps = 4;            // warps per CTA of the sorting kernels
constexpr int kMaxDigitBits = 11;        // bins of one sorting pass: 2^11 counters of 4 bytes per warp
constexpr uint32_t kNone = 0xffffffffu;  // key of a token without an embedding

struct IndexView {
  const void* p;
  int bits;
  uint32_t rows;
  // the table row, or kNone
  __device__ __forceinline__ uint32_t at(uint32_t t) const {
    if (bits == 32) {
      const uint32_t v = static_cast<const uint32_t*>(p)[t];  // negative values are above every row
      return v < rows ? v : kNone;
    }
    const uint64_t v = static_cast<const uint64_t*>(p)[t];
    return v < rows ? static_cast<uint32_t>(v) : kNone;
  }
};

template <bool kWide>
__device__ __forceinline__ void load_table(const void* table, int dtype, int64_t at, int n, float (&f)[8]) {
  if constexpr (kWide) {
    if (dtype == PAIR_FP32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(table) + at);
      const float4 x = __ldg(p), y = __ldg(p + 1);
      f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w, f[4] = y.x, f[5] = y.y, f[6] = y.z, f[7] = y.w;
    } else {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(table) + at));
      if (dtype == PAIR_FP16)
        unpack(reinterpret_cast<const Oct<__half>&>(x), f);
      else
        unpack(reinterpret_cast<const Oct<__nv_bfloat16>&>(x), f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = k < n ? load_any(table, at + k, dtype) : 0.f;
  }
}

template <bool kWide>
__device__ __forceinline__ void store_table(void* table, int dtype, int64_t at, int n, const float (&f)[8]) {
  if constexpr (kWide) {
    if (dtype == PAIR_FP32)
      store_oct<true>(static_cast<float*>(table) + at, pack<float>(f), 8);
    else if (dtype == PAIR_FP16)
      store_oct<true>(static_cast<__half*>(table) + at, pack<__half>(f), 8);
    else
      store_oct<true>(static_cast<__nv_bfloat16*>(table) + at, pack<__nv_bfloat16>(f), 8);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) store_any(table, at + k, dtype, f[k]);
  }
}

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------
template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads) embed_kernel(IndexView index, const void* table, int table_dtype, const T* base,
                                                         T* out, uint32_t tokens, int d, int octs, FastDiv by_octs, float scale) {
  const int64_t total = static_cast<int64_t>(tokens) * octs;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t n = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; n < total; n += step) {
    uint32_t t, v;
    if (total <= 0x7fffffff) {
      t = by_octs.div(static_cast<uint32_t>(n));
      v = static_cast<uint32_t>(n) - t * by_octs.d;
    } else {
      t = static_cast<uint32_t>(n / octs);
      v = static_cast<uint32_t>(n - static_cast<int64_t>(t) * octs);
    }
    const int left = d - static_cast<int>(v) * 8;
    const int64_t at = static_cast<int64_t>(t) * d + v * 8;
    const uint32_t row = index.at(t);
    Oct<T> b;
    if (base != nullptr) b = load_oct<kWide>(base + at, left);
    float f[8], g[8];
    if (row != kNone) {
      load_table<kWide>(table, table_dtype, static_cast<int64_t>(row) * d + v * 8, left, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= scale;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
    }
    if (base != nullptr) {
      unpack(b, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += g[e];
    }
    store_oct<kWide>(out + at, pack<T>(f), left);
  }
}

// ---------------------------------------------------------------------------------------------
// gradient without a sort
// ---------------------------------------------------------------------------------------------
// One CTA per table row (x) and slab of 256 channels (y): its eight warps look through an eighth of the indices each and
// add the rows that match, in ascending order; the warps' sums are joined in order.
template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads) embed_grad_few_kernel(IndexView index, const T* d_out, void* d_table,
                                                                  int table_dtype, uint32_t tokens, int d, int octs, float scale) {
  __shared__ float sums[kThreads / 32][kSlabOcts * 8 + 8];
  const uint32_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int v = blockIdx.y * kSlabOcts + lane;
  const bool on = v < octs;
  const uint32_t share = ((tokens + 8 * 32 - 1) / (8 * 32)) * 32;
  const uint32_t lo = warp * share, hi = min(tokens, lo + share);
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (uint32_t t0 = lo; t0 < hi; t0 += 32) {
    const uint32_t t = t0 + lane;
    uint32_t hit = __ballot_sync(0xffffffffu, t < hi && index.at(t) == row);
    while (hit != 0) {
      Oct<T> o[4];
      int n = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (hit != 0) {
          const uint32_t at = t0 + __ffs(hit) - 1;
          hit &= hit - 1;
          o[k] = on ? load_oct<kWide>(d_out + static_cast<int64_t>(at) * d + v * 8, d - v * 8) : zero_oct<T>();
          n = k + 1;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n) {
          float f[8];
          unpack(o[k], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += f[e];
        }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[warp][lane * 8 + e] = acc[e];
  __syncthreads();
  if (warp != 0 || !on) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) acc[e] += sums[w][lane * 8 + e];
    acc[e] *= scale;
  }
  store_table<kWide>(d_table, table_dtype, static_cast<int64_t>(row) * d + v * 8, d - v * 8, acc);
}

// ---------------------------------------------------------------------------------------------
// stable counting sort of the token numbers
// ---------------------------------------------------------------------------------------------
// The tokens are cut into `tiles` equal tiles, one per warp.  Pass: count each tile's digits (counts[bin][tile]), scan
// every bin over the tiles, then place each token behind its bin's, its tile's and its own predecessors.
struct SortArgs {
  IndexView index;
  const uint32_t* in;  // token numbers in the order of the passes so far; nullptr: 0, 1, 2, ...
  uint32_t* out;
  uint32_t* counts;  // (bins, tiles)
  uint32_t* totals;  // (bins)
  uint32_t tokens, tiles, tile;
  int shift, bins;
};

// Tokens without an embedding sort behind all others: their key is the number of rows.
__device__ __forceinline__ uint32_t digit_of(const SortArgs& a, uint32_t t) {
  const uint32_t key = a.index.at(t);
  return ((key == kNone ? a.index.rows : key) >> a.shift) & (a.bins - 1);
}

__global__ void __launch_bounds__(kSortWarps * 32) sort_count_kernel(const SortArgs a) {
  extern __shared__ uint32_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* mine = smem + warp * a.bins;
  const uint32_t w = blockIdx.x * kSortWarps + warp;
  for (int k = lane; k < a.bins; k += 32) mine[k] = 0;
  __syncwarp();
  if (w >= a.tiles) return;
  const uint32_t lo = min(a.tokens, w * a.tile), hi = min(a.tokens, lo + a.tile);
  for (uint32_t p0 = lo; p0 < hi; p0 += 128) {
    uint32_t digit[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t p = p0 + k * 32 + lane;
      digit[k] = p < hi ? digit_of(a, a.in != nullptr ? a.in[p] : p) : kNone;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t same = __match_any_sync(0xffffffffu, digit[k]);
      if (digit[k] != kNone && lane == __ffs(same) - 1) mine[digit[k]] += __popc(same);
      __syncwarp();
    }
  }
  for (int k = lane; k < a.bins; k += 32) a.counts[static_cast<int64_t>(k) * a.tiles + w] = mine[k];
}

// Exclusive scan of one bin's counts over the tiles; the bin's total beside it.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(uint32_t* counts, uint32_t* totals, uint32_t tiles) {
  __shared__ uint32_t part[kThreads / 32];
  uint32_t* c = counts + static_cast<int64_t>(blockIdx.x) * tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t carry = 0;
  for (uint32_t base = 0; base < tiles; base += kThreads) {
    const uint32_t at = base + threadIdx.x;
    const uint32_t own = at < tiles ? c[at] : 0;
    uint32_t x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += up;
    }
    if (lane == 31) part[warp] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int k = 0; k < kThreads / 32; ++k) {
      if (k < warp) before += part[k];
      all += part[k];
    }
    if (at < tiles) c[at] = carry + before + x - own;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

__global__ void __launch_bounds__(kSortWarps * 32) sort_place_kernel(const SortArgs a) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t part[kSortWarps];
  uint32_t* first = smem + kSortWarps * a.bins;  // where each bin begins
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t carry = 0;
  for (int base = 0; base < a.bins; base += kSortWarps * 32) {
    const int at = base + threadIdx.x;
    const uint32_t own = at < a.bins ? a.totals[at] : 0;
    uint32_t x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += up;
    }
    if (lane == 31) part[warp] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int k = 0; k < kSortWarps; ++k) {
      if (k < warp) before += part[k];
      all += part[k];
    }
    if (at < a.bins) first[at] = carry + before + x - own;
    carry += all;
    __syncthreads();
  }
  const uint32_t w = blockIdx.x * kSortWarps + warp;
  if (w >= a.tiles) return;
  uint32_t* next = smem + warp * a.bins;
  for (int k = lane; k < a.bins; k += 32) next[k] = first[k] + a.counts[static_cast<int64_t>(k) * a.tiles + w];
  __syncwarp();
  const uint32_t lo = min(a.tokens, w * a.tile), hi = min(a.tokens, lo + a.tile);
  for (uint32_t p0 = lo; p0 < hi; p0 += 128) {
    uint32_t token[4], digit[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t p = p0 + k * 32 + lane;
      token[k] = p < hi ? (a.in != nullptr ? a.in[p] : p) : kNone;
      digit[k] = p < hi ? digit_of(a, token[k]) : kNone;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t same = __match_any_sync(0xffffffffu, digit[k]);
      const uint32_t at = digit[k] != kNone ? next[digit[k]] : 0;
      __syncwarp();
      if (digit[k] != kNone) {
        a.out[at + __popc(same & ((1u << lane) - 1))] = token[k];
        if (lane == __ffs(same) - 1) next[digit[k]] = at + __popc(same);
      }
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------------------------------------
// sums over the sorted tokens
// ---------------------------------------------------------------------------------------------
template <typename T>
struct SumArgs {
  IndexView index;
  const uint32_t* sorted;
  const T* d_out;
  void* d_table;
  float* pieces;  // (shares, 2, padded width): sums of runs that cross into [0] / out of [1] the share
  uint32_t tokens, share, shares;
  int d, octs, table_dtype;
  float scale;
  __device__ __forceinline__ uint32_t key(uint32_t p) const { return index.at(sorted[p]); }
};

// kGroup lanes sum one share of sorted tokens over one slab of channels (blockIdx.y).
template <typename T, int kGroup, bool kWide>
__global__ void __launch_bounds__(kThreads) sum_runs_kernel(const SumArgs<T> a) {
  constexpr int kAhead = 8;  // rows of d_out in flight per lane
  const int lane = threadIdx.x % kGroup;
  const uint32_t mask = kGroup == 32 ? 0xffffffffu : ((1u << kGroup) - 1) << ((threadIdx.x & 31) / kGroup * kGroup);
  const uint32_t share = blockIdx.x * (kThreads / kGroup) + threadIdx.x / kGroup;
  if (share >= a.shares) return;
  const int v = blockIdx.y * kSlabOcts + lane;
  const bool on = v < a.octs;
  const uint32_t lo = share * a.share, hi = min(a.tokens, lo + a.share);

  double total[8];
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) total[e] = 0.0, acc[e] = 0.f;
  uint32_t run = a.key(lo);  // index of the run at hand
  bool from_left = lo > 0 && a.key(lo - 1) == run;

  auto flush = [&](bool to_right) {
    if (run == kNone || !on) return;
    float f[8];
    if (from_left || to_right) {
      float* p = a.pieces + (static_cast<int64_t>(share) * 2 + (from_left ? 0 : 1)) * (a.octs * 8) + v * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(total[e] + acc[e]);
      reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(total[e] + acc[e]) * a.scale;
      store_table<kWide>(a.d_table, a.table_dtype, static_cast<int64_t>(run) * a.d + v * 8, a.d - v * 8, f);
    }
  };

  for (uint32_t p0 = lo; p0 < hi; p0 += kGroup) {
    const uint32_t p = p0 + lane;
    const uint32_t my_token = p < hi ? a.sorted[p] : 0;
    const uint32_t my_key = p < hi ? a.index.at(my_token) : kNone;
    const int here = min(static_cast<uint32_t>(kGroup), hi - p0);
    for (int e0 = 0; e0 < here; e0 += kAhead) {
      Oct<T> o[kAhead];
      uint32_t key[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint32_t t = __shfl_sync(mask, my_token, e0 + k, kGroup);
        key[k] = __shfl_sync(mask, my_key, e0 + k, kGroup);
        o[k] = on && e0 + k < here && key[k] != kNone
                   ? load_oct<kWide>(a.d_out + static_cast<int64_t>(t) * a.d + v * 8, a.d - v * 8)
                   : zero_oct<T>();
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (e0 + k < here) {
          if (key[k] != run) {
            flush(false);
            run = key[k];
            from_left = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) total[e] = 0.0, acc[e] = 0.f;
          }
          float f[8];
          unpack(o[k], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += f[e];
        }
      }
    }
    // fp32 sums of at most 32 terms are carried over to 64 bits
#pragma unroll
    for (int e = 0; e < 8; ++e) total[e] += acc[e], acc[e] = 0.f;
  }
  flush(hi < a.tokens && a.key(hi) == run);
}

// The share in which a crossing run begins adds up its pieces: its own [1], then [0] of the shares that follow.
template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads) join_runs_kernel(const SumArgs<T> a) {
  __shared__ double sums[kThreads / 32][kSlabOcts * 8];
  __shared__ uint32_t last;
  const uint32_t share = blockIdx.x;
  const uint32_t lo = share * a.share, hi = lo + a.share;
  if (hi >= a.tokens) return;
  const uint32_t run = a.key(hi - 1);
  if (run == kNone || a.key(hi) != run) return;
  if (lo > 0 && a.key(lo - 1) == run) return;  // the run began before this share
  // the last share that the run reaches: the first keys of the shares are sorted
  if (threadIdx.x == 0) last = share;
  __syncthreads();
  uint32_t from = share + 1, until = a.shares;  // shares [from, until) may begin with the run
  while (from < until) {
    const uint32_t step = (until - from + kThreads - 1) / kThreads;
    const uint32_t at = from + threadIdx.x * step;
    const bool mine = at < until && a.key(at * a.share) == run;
    const int n = __syncthreads_count(mine);  // a prefix of the probes
    if (n == 0) break;
    const uint32_t reached = from + (n - 1) * step;
    if (threadIdx.x == 0) last = reached;
    from = reached + 1;
    until = min(until, reached + step);
  }
  __syncthreads();
  const uint32_t end = last + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t width = a.octs * 8;
  // eight warps, each an equal part of the pieces in order
  const uint32_t pieces = end - share, per = (pieces + 7) / 8;
  const uint32_t p_lo = share + min(pieces, warp * per), p_hi = share + min(pieces, (warp + 1) * per);
  for (int slab = 0; slab * kSlabOcts < a.octs; ++slab) {
    const int v = slab * kSlabOcts + lane;
    double acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (v < a.octs) {
#pragma unroll 4
      for (uint32_t s = p_lo; s < p_hi; ++s) {
        const float4* p = reinterpret_cast<const float4*>(a.pieces + (static_cast<int64_t>(s) * 2 + (s == share ? 1 : 0)) * width + v * 8);
        const float4 x = p[0], y = p[1];
        acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
        acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[warp][lane * 8 + e] = acc[e];
    __syncthreads();
    if (warp == 0 && v < a.octs) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int w = 1; w < kThreads / 32; ++w) acc[e] += sums[w][lane * 8 + e];
        f[e] = static_cast<float>(acc[e]) * a.scale;
      }
      store_table<kWide>(a.d_table, a.table_dtype, static_cast<int64_t>(run) * a.d + v * 8, a.d - v * 8, f);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
struct Plan {
  bool few;
  int octs, passes, digit_bits, bins;
  uint32_t tiles, tile, share, shares;
  uint64_t sorted_at[2], counts_at, totals_at, pieces_at, bytes;
};

inline uint64_t up256(uint64_t n) { return (n + 255) & ~255ull; }

// Lanes that cover a row (of at most one slab).
inline int group_of(int octs) { return octs <= 8 ? 8 : octs <= 16 ? 16 : 32; }

Plan make_plan(const pair_embed_desc_t* d, int sms) {
  Plan p = {};
  const uint64_t tokens = static_cast<uint64_t>(d->tokens);
  p.octs = (d->d + 7) / 8;
  p.few = tokens <= 2048 && tokens * static_cast<uint64_t>(d->rows) <= (1u << 22);
  if (p.few) {
    p.bytes = 256;
    return p;
  }
  int bits = 1;
  while ((1ull << bits) <= static_cast<uint64_t>(d->rows)) ++bits;  // keys 0 .. rows
  p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  p.bins = 1 << p.digit_bits;
  // tiles of at least 256 tokens, at most 16 warps an SM, and no more counters than tokens (one SM's worth aside)
  uint64_t most = tokens / p.bins > static_cast<uint64_t>(sms) ? tokens / p.bins : sms;
  if (most > static_cast<uint64_t>(sms) * 16) most = static_cast<uint64_t>(sms) * 16;
  uint64_t tiles = (tokens + 255) / 256;
  if (tiles > most) tiles = most;
  p.tile = static_cast<uint32_t>(((tokens + tiles - 1) / tiles + 31) / 32 * 32);
  p.tiles = static_cast<uint32_t>((tokens + p.tile - 1) / p.tile);
  // shares: one wave of resident groups, of at least 32 tokens
  const uint64_t groups = static_cast<uint64_t>(sms) * (4 * kThreads / group_of(p.octs));
  uint64_t share = (tokens + groups - 1) / groups;
  if (share < 32) share = 32;
  p.share = static_cast<uint32_t>(share);
  p.shares = static_cast<uint32_t>((tokens + share - 1) / share);
  uint64_t at = 0;
  p.sorted_at[0] = at, at += up256(tokens * 4);
  p.sorted_at[1] = at, at += p.passes > 1 ? up256(tokens * 4) : 0;
  p.counts_at = at, at += up256(static_cast<uint64_t>(p.bins) * p.tiles * 4);
  p.totals_at = at, at += up256(static_cast<uint64_t>(p.bins) * 4);
  p.pieces_at = at, at += up256(static_cast<uint64_t>(p.shares) * 2 * p.octs * 8 * 4);
  p.bytes = at;
  return p;
}

template <typename T, bool kWide>
cudaError_t embed_run(const pair_embed_desc_t* d, const IndexView& index, const void* table, const void* base, void* out,
                      int sms, cudaStream_t s) {
  const int octs = (d->d + 7) / 8;
  const int64_t need = (d->tokens * octs + kThreads - 1) / kThreads, most = static_cast<int64_t>(sms) * 8;
  embed_kernel<T, kWide><<<static_cast<unsigned>(need < most ? need : most), kThreads, 0, s>>>(
      index, table, d->table_dtype, static_cast<const T*>(base), static_cast<T*>(out), static_cast<uint32_t>(d->tokens), d->d,
      octs, make_fast_div(octs), d->scale);
  return cudaGetLastError();
}

template <typename T, bool kWide>
cudaError_t grad_run(const pair_embed_desc_t* d, const IndexView& index, const void* d_out, void* d_table, void* workspace,
                     int sms, cudaStream_t s) {
  const Plan p = make_plan(d, sms);
  const uint32_t tokens = static_cast<uint32_t>(d->tokens);
  const int slabs = (p.octs + kSlabOcts - 1) / kSlabOcts;
  if (p.few) {
    embed_grad_few_kernel<T, kWide><<<dim3(d->rows, slabs), kThreads, 0, s>>>(
        index, static_cast<const T*>(d_out), d_table, d->table_dtype, tokens, d->d, p.octs, d->scale);
    return cudaGetLastError();
  }
  char* ws = static_cast<char*>(workspace);
  // rows that no token names; the others are written afterwards
  cudaError_t e = cudaMemsetAsync(d_table, 0, static_cast<size_t>(d->rows) * d->d * type_bytes(d->table_dtype), s);
  if (e != cudaSuccess) return e;
  SortArgs a;
  a.index = index;
  a.counts = reinterpret_cast<uint32_t*>(ws + p.counts_at);
  a.totals = reinterpret_cast<uint32_t*>(ws + p.totals_at);
  a.tokens = tokens;
  a.tiles = p.tiles;
  a.tile = p.tile;
  a.bins = p.bins;
  a.in = nullptr;
  const int count_smem = kSortWarps * p.bins * 4, place_smem = (kSortWarps + 1) * p.bins * 4;
  const unsigned grid = (p.tiles + kSortWarps - 1) / kSortWarps;
  for (int pass = 0; pass < p.passes; ++pass) {
    // the last pass ends in buffer 0
    a.out = reinterpret_cast<uint32_t*>(ws + p.sorted_at[(p.passes - 1 - pass) & 1]);
    a.shift = pass * p.digit_bits;
    sort_count_kernel<<<grid, kSortWarps * 32, count_smem, s>>>(a);
    sort_scan_kernel<<<p.bins, kThreads, 0, s>>>(a.counts, a.totals, a.tiles);
    sort_place_kernel<<<grid, kSortWarps * 32, place_smem, s>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    a.in = a.out;
  }
  SumArgs<T> m;
  m.index = index;
  m.sorted = a.in;
  m.d_out = static_cast<const T*>(d_out);
  m.d_table = d_table;
  m.pieces = reinterpret_cast<float*>(ws + p.pieces_at);
  m.tokens = tokens;
  m.share = p.share;
  m.shares = p.shares;
  m.d = d->d;
  m.octs = p.octs;
  m.table_dtype = d->table_dtype;
  m.scale = d->scale;
  const int group = group_of(p.octs);
  const int held = kThreads / group;
  const dim3 sum_grid((p.shares + held - 1) / held, slabs);
  if (group == 8)
    sum_runs_kernel<T, 8, kWide><<<sum_grid, kThreads, 0, s>>>(m);
  else if (group == 16)
    sum_runs_kernel<T, 16, kWide><<<sum_grid, kThreads, 0, s>>>(m);
  else
    sum_runs_kernel<T, 32, kWide><<<sum_grid, kThreads, 0, s>>>(m);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  join_runs_kernel<T, kWide><<<p.shares, kThreads, 0, s>>>(m);
  return cudaGetLastError();
}

int check_embed_desc(const pair_embed_desc_t* d, const char* who) {
  using trimul::report_error;
  if (d == nullptr) return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: desc is NULL", who);
  if (d->tokens < 0 || d->d < 1 || d->rows < 1)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: %lld tokens of width %d and %d table rows", who,
                        static_cast<long long>(d->tokens), d->d, d->rows);
  if (d->tokens > 0x7fffffffLL)
    return report_error(TRIMUL_ERR_UNSUPPORTED_SHAPE, "%s: %lld tokens are above 2^31 - 1", who, static_cast<long long>(d->tokens));
  if (d->d > PAIR_MAX_WIDTH)
    return report_error(TRIMUL_ERR_UNSUPPORTED_SHAPE, "%s: width d=%d is above %d", who, d->d, PAIR_MAX_WIDTH);
  if (d->index_bits != 32 && d->index_bits != 64)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: index_bits=%d is neither 32 nor 64", who, d->index_bits);
  if (int rc = check_dtype(d->dtype, "the activation", who)) return rc;
  return check_dtype(d->table_dtype, "the table", who);
}

}  // namespace
}  // namespace pair

extern "C" int pair_sm100_embed(const pair_embed_desc_t* desc, const void* index, const void* table, const void* base,
                                void* out, trimul_stream_t cuda_stream) {
  using namespace pair;
  using trimul::report_error;
  const char* who = "pair_sm100_embed";
  if (int rc = check_embed_desc(desc, who)) return rc;
  if (desc->tokens == 0) return TRIMUL_OK;
  if (index == nullptr || table == nullptr || out == nullptr)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: index, table and out must not be NULL", who);
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  const IndexView view{index, desc->index_bits, static_cast<uint32_t>(desc->rows)};
  const bool wide = desc->d % 8 == 0 && aligned16(table) && aligned16(base) && aligned16(out);
  cudaError_t e;
  if (desc->dtype == PAIR_FP32)
    e = wide ? embed_run<float, true>(desc, view, table, base, out, sms, cuda_stream)
             : embed_run<float, false>(desc, view, table, base, out, sms, cuda_stream);
  else if (desc->dtype == PAIR_FP16)
    e = wide ? embed_run<__half, true>(desc, view, table, base, out, sms, cuda_stream)
             : embed_run<__half, false>(desc, view, table, base, out, sms, cuda_stream);
  else
    e = wide ? embed_run<__nv_bfloat16, true>(desc, view, table, base, out, sms, cuda_stream)
             : embed_run<__nv_bfloat16, false>(desc, view, table, base, out, sms, cuda_stream);
  if (e != cudaSuccess) return report_error(TRIMUL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return TRIMUL_OK;
}

extern "C" int pair_sm100_embed_grad_workspace(const pair_embed_desc_t* desc, uint64_t* bytes) {
  using namespace pair;
  const char* who = "pair_sm100_embed_grad_workspace";
  if (int rc = check_embed_desc(desc, who)) return rc;
  if (bytes == nullptr) return trimul::report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: bytes is NULL", who);
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return trimul::report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  *bytes = desc->tokens == 0 ? 0 : make_plan(desc, sms).bytes;
  return TRIMUL_OK;
}

extern "C" int pair_sm100_embed_grad(const pair_embed_desc_t* desc, const void* index, const void* d_out, void* d_table,
                                     void* workspace, trimul_stream_t cuda_stream) {
  using namespace pair;
  using trimul::report_error;
  const char* who = "pair_sm100_embed_grad";
  if (int rc = check_embed_desc(desc, who)) return rc;
  if (d_table == nullptr) return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: d_table is NULL", who);
  cudaError_t e;
  if (desc->tokens == 0) {
    e = cudaMemsetAsync(d_table, 0, static_cast<size_t>(desc->rows) * desc->d * type_bytes(desc->table_dtype), cuda_stream);
    if (e != cudaSuccess) return report_error(TRIMUL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return TRIMUL_OK;
  }
  if (index == nullptr || d_out == nullptr) return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: index and d_out must not be NULL", who);
  if (workspace == nullptr || !aligned16(workspace))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace", who);
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  const IndexView view{index, desc->index_bits, static_cast<uint32_t>(desc->rows)};
  const bool wide = desc->d % 8 == 0 && aligned16(d_out) && aligned16(d_table);
  if (desc->dtype == PAIR_FP32)
    e = wide ? grad_run<float, true>(desc, view, d_out, d_table, workspace, sms, cuda_stream)
             : grad_run<float, false>(desc, view, d_out, d_table, workspace, sms, cuda_stream);
  else if (desc->dtype == PAIR_FP16)
    e = wide ? grad_run<__half, true>(desc, view, d_out, d_table, workspace, sms, cuda_stream)
             : grad_run<__half, false>(desc, view, d_out, d_table, workspace, sms, cuda_stream);
  else
    e = wide ? grad_run<__nv_bfloat16, true>(desc, view, d_out, d_table, workspace, sms, cuda_stream)
             : grad_run<__nv_bfloat16, false>(desc, view, d_out, d_table, workspace, sms, cuda_stream);
  if (e != cudaSuccess) return report_error(TRIMUL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return TRIMUL_OK;
}
