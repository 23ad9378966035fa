// Embedding lookup into the pair stream, and the gradient of its table.
//
// Mathematics.  out[t] = base[t] + scale E[x_t];  dE[v] = scale sum_{t: x_t = v} d_out[t].  An index outside
// [0, rows) stands for "no embedding": it adds nothing and receives no gradient.
//
// Bound.  Forward: HBM, base read and out written once; the table (tens of rows for position bins) stays in L1 and L2.
// Gradient: HBM, d_out read once.  Position bins give some 10^6 tokens to each of a few dozen rows, vocabularies give
// one or two, so the sum is organised by sorted tokens: a stable counting sort of the token numbers by index (up to
// 256 bins a pass, no comparison, pairs of int32 only), then every group of lanes sums the d_out rows of an equal share
// of the SORTED tokens.  A run of equal indices inside one share goes straight to the table; a run that crosses
// shares leaves its pieces in the workspace, and the share in which it begins adds them up afterwards.  No atomics: the
// same bits every time, whatever the distribution.
// Few tokens skip the sort: one CTA per table row looks through all indices.  So do small tables, of which every warp of an SM has one of its
// own in shared memory.
#include "pair_stream.cuh"

namespace pair {
namespace {

constexpr int kSlab = 256;               // channels of a row that one warp covers
constexpr int kSortWarps = 4;            // warps per CTA of the sorting kernels
// Bits of one sorting pass: 2^8 counters of 4 bytes per warp.  (More bits save passes and cost more than that in counters: 16384 tokens into
// 1024 rows take 28 us with 8 bits, 41 with 11; into 100000 rows 39 against 73; with 5 bits 33 and 45.)
constexpr int kMaxDigitBits = 8;
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

// Eight channels of a row per lane: whole octs of aligned rows (kWide), or channels that lie kGroup apart, so that the accesses of
// the lanes are contiguous either way.
template <bool kWide, int kGroup>
__device__ __forceinline__ int channel_of(int lane, int e) { return kWide ? lane * 8 + e : lane + e * kGroup; }

template <bool kWide, int kGroup, typename T>
__device__ __forceinline__ Unit<T, 8> load_eight(const T* row, int lane, int left) {
  if constexpr (kWide) {
    return lane * 8 < left ? load_unit<T, 8>(row + lane * 8) : zero_unit<T, 8>();
  } else {
    Unit<T, 8> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.e[e] = lane + e * kGroup < left ? load_unit<T, 1>(row + lane + e * kGroup).e[0] : from_f32<T>(0.f);
    return o;
  }
}

template <bool kWide, int kGroup>
__device__ __forceinline__ void store_eight(void* table, int dtype, int64_t at, int lane, int left, const float (&f)[8]) {
  if constexpr (kWide) {
    if (lane * 8 >= left) return;
    Lane<8, 1> v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v.p[e] = make_float2(f[2 * e], f[2 * e + 1]);
    at += lane * 8;
    if (dtype == PAIR_FP32)
      store_unit<float, 8>(static_cast<float*>(table) + at, pack<float>(v));
    else if (dtype == PAIR_FP16)
      store_unit<__half, 8>(static_cast<__half*>(table) + at, pack<__half>(v));
    else
      store_unit<__nv_bfloat16, 8>(static_cast<__nv_bfloat16*>(table) + at, pack<__nv_bfloat16>(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + e * kGroup < left) store_any(table, at + lane + e * kGroup, dtype, f[e]);
  }
}

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------
struct EmbedArgs {
  IndexView index;
  const void* table;
  const void* base;
  void* out;
  uint32_t tokens;
  int d, octs, table_dtype;
  float scale;
};

__device__ __forceinline__ Lane<8, 1> table_oct(const void* table, int dtype, int64_t at) {
  if (dtype == PAIR_FP32) {
    Unit<float, 8> x;
    reinterpret_cast<uint4*>(&x)[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(table) + at));
    reinterpret_cast<uint4*>(&x)[1] = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(table) + at) + 1);
    return unpack(x);
  }
  const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(table) + at));
  return dtype == PAIR_FP16 ? unpack(reinterpret_cast<const Unit<__half, 8>&>(x)) : unpack(reinterpret_cast<const Unit<__nv_bfloat16, 8>&>(x));
}

// Whole octs: one per thread and step.
template <typename T>
__global__ void __launch_bounds__(kThreads) embed_octs_kernel(const EmbedArgs a, const FastDiv by_octs) {
  const T* base = static_cast<const T*>(a.base);
  const int64_t total = static_cast<int64_t>(a.tokens) * a.octs;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t n = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; n < total; n += step) {
    uint32_t t, v;
    if (total <= 0x7fffffff) {
      t = by_octs.div(static_cast<uint32_t>(n));
      v = static_cast<uint32_t>(n) - t * by_octs.d;
    } else {
      t = static_cast<uint32_t>(n / a.octs);
      v = static_cast<uint32_t>(n - static_cast<int64_t>(t) * a.octs);
    }
    const uint32_t row = a.index.at(t);
    Unit<T, 8> b = zero_unit<T, 8>();
    if (base != nullptr) b = load_unit<T, 8>(base + n * 8);
    Lane<8, 1> f = unpack(b);
    if (row != kNone) {
      const Lane<8, 1> x = table_oct(a.table, a.table_dtype, static_cast<int64_t>(row) * a.d + v * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) f.p[e] = fma_whole(x.p[e], both(a.scale), f.p[e]);
    }
    store_unit<T, 8>(static_cast<T*>(a.out) + n * 8, pack<T>(f));
  }
}

// Other rows: a warp takes 256 channels of a token at a time, 32 apart.
template <typename T>
__global__ void __launch_bounds__(kThreads) embed_pieces_kernel(const EmbedArgs a, const FastDiv by_pieces) {
  const int lane = threadIdx.x & 31;
  const int64_t total = static_cast<int64_t>(a.tokens) * by_pieces.d;
  const int64_t span = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  for (int64_t n = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); n < total; n += span) {
    uint32_t t, piece;
    if (total <= 0x7fffffff) {
      t = by_pieces.div(static_cast<uint32_t>(n));
      piece = static_cast<uint32_t>(n) - t * by_pieces.d;
    } else {
      t = static_cast<uint32_t>(n / by_pieces.d);
      piece = static_cast<uint32_t>(n - static_cast<int64_t>(t) * by_pieces.d);
    }
    const uint32_t row = a.index.at(t);
    const int c0 = piece * 256 + lane;
    const int64_t at = static_cast<int64_t>(t) * a.d + c0, from = static_cast<int64_t>(row) * a.d + c0;
    const int left = a.d - c0;  // channels from the lane's first one on
    Unit<T, 1> b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      b[k] = zero_unit<T, 1>();
      if (a.base != nullptr && k * 32 < left) b[k] = load_unit<T, 1>(static_cast<const T*>(a.base) + at + k * 32);
    }
    auto add = [&](const auto* table) {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = k * 32 < left ? to_f32(table[from + k * 32]) : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) b[k].e[0] = from_f32<T>(fma_whole(f[k], a.scale, to_f32(b[k].e[0])));
    };
    if (row != kNone) {
      if (a.table_dtype == PAIR_FP32)
        add(static_cast<const float*>(a.table));
      else if (a.table_dtype == PAIR_FP16)
        add(static_cast<const __half*>(a.table));
      else
        add(static_cast<const __nv_bfloat16*>(a.table));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k * 32 < left) store_unit<T, 1>(static_cast<T*>(a.out) + at + k * 32, b[k]);
  }
}

// ---------------------------------------------------------------------------------------------
// gradient without a sort
// ---------------------------------------------------------------------------------------------
// One CTA per table row (x) and slab of 256 channels (y): each warp looks through its part of the indices and adds the rows that
// match, in ascending order; the warps' sums are joined in order.  The fewer rows there are, the more warps each takes (4096 tokens
// into 21 rows: 7.4 us with 32, 12.7 with eight; into 2048 rows 22 and 13).  Of a table with more rows than there are tokens
// (kByToken), each token's CTA takes the token's row, unless an earlier token has named it; the other rows are cleared before.
template <typename T, bool kWide, bool kByToken>
__global__ void __launch_bounds__(1024) embed_grad_few_kernel(IndexView index, const T* d_out, void* d_table, int table_dtype,
                                                              uint32_t tokens, uint32_t share, int d, float scale) {
  constexpr int kAhead = 4, kLook = 4;  // rows of d_out and blocks of 32 indices in flight
  extern __shared__ float sums[];       // (warps, kSlab)
  const int threads = blockDim.x;
  uint32_t row = blockIdx.x;
  if constexpr (kByToken) {
    row = index.at(blockIdx.x);
    if (row == kNone) return;
    int named = 0;
    for (uint32_t t = threadIdx.x; t < blockIdx.x; t += threads) named |= index.at(t) == row;
    if (__syncthreads_or(named)) return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slab = blockIdx.y * kSlab, left = d - slab;
  float* mine = sums + warp * kSlab + lane;
  const uint32_t lo = min(tokens, warp * share), hi = min(tokens, lo + share);
#pragma unroll
  for (int e = 0; e < 8; ++e) mine[e * 32] = 0.f;
  for (uint32_t block = lo; block < hi; block += 32 * kLook) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // of a block first: at most 128 terms, then at most 32
    uint32_t hits[kLook];
#pragma unroll
    for (int k = 0; k < kLook; ++k) {
      const uint32_t t = block + k * 32 + lane;
      hits[k] = t < hi && index.at(t) == row;
    }
#pragma unroll
    for (int k = 0; k < kLook; ++k) hits[k] = __ballot_sync(0xffffffffu, hits[k]);
#pragma unroll 1
    for (int look = 0; look < kLook && block + look * 32 < hi; ++look) {
      uint32_t hit = hits[0];
#pragma unroll
      for (int k = 0; k + 1 < kLook; ++k) hits[k] = hits[k + 1];
      const uint32_t t0 = block + look * 32;
      while (hit != 0) {
        Unit<T, 8> o[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          o[k] = zero_unit<T, 8>();
          if (hit != 0) {
            o[k] = load_eight<kWide, 32>(d_out + static_cast<int64_t>(t0 + __ffs(hit) - 1) * d + slab, lane, left);
            hit &= hit - 1;
          }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += to_f32(o[k].e[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[e * 32] += acc[e];
  }
  __syncthreads();
  if (threadIdx.x >= kSlab) return;
  const int c = channel_of<kWide, 32>(lane, warp);  // thread 32 e + lane joins value e of the lanes
  float sum = 0.f;
#pragma unroll 8
  for (int w = 0; w < threads / 32; ++w) sum += sums[w * kSlab + threadIdx.x];
  if (c < left) store_any(d_table, static_cast<int64_t>(row) * d + slab + c, table_dtype, sum * scale);
}

// ---------------------------------------------------------------------------------------------
// gradient of a small table
// ---------------------------------------------------------------------------------------------
// The fp32 sums of up to 74 rows and 64 channels fit an SM's shared memory a dozen times: each warp walks over an equal share of the tokens
// in order, two channels per lane, and adds them to a table of its own.  No sort, no gather: d_out streams in as it lies, a
// batch at hand and one on its way.  The CTA's tables are joined in order, and a second kernel joins the CTAs'.
// Measured beside the sort, 768 x 768 positions of 128 bf16 channels: 66 relative-position bins 47 us against 62, 66 random bins 60
// against 63, 21 rows 39 and 45 against 60; 64 x 64 positions into 21 rows 8 against 15.  110 rows (eight warps' tables): 67 against 63.
// (Four channels per lane take as long: 47 and 60 us.)
constexpr int kTableSlab = 64, kTableWarps = 16, kTableRows = 74;
constexpr int kTableSmem = 227 * 1024;
constexpr uint32_t kTableShare = 1024;  // most tokens of a warp: the terms of an fp32 sum

template <int kBytes>
struct RawOf {
  using type = uint16_t;
};
template <>
struct RawOf<4> {
  using type = uint32_t;
};
template <>
struct RawOf<8> {
  using type = uint2;  // a pair of fp32
};

template <typename T>
struct TableArgs {
  IndexView index;
  const T* d_out;
  float* partial;  // (parts, rows, d)
  uint32_t tokens, share;
  int d;
};

// kU channels per access: a lane's two neighbours, or two channels that lie 32 apart.
template <typename T, int kU>
__global__ void __launch_bounds__(kTableWarps * 32) embed_grad_table_kernel(const TableArgs<T> a) {
  next_may_start();
  constexpr int kUnits = 2 / kU;
  constexpr int kBatch = sizeof(T) == 2 && kU == 2 ? 32 : 16;  // tokens on their way
  using Raw = typename RawOf<sizeof(T) * kU>::type;
  extern __shared__ float2 tables[];  // [warp][row][lane]; a row behind the last one takes tokens without an embedding
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
  const uint32_t rows = a.index.rows;
  float2* const mine = tables + warp * (rows + 1) * 32 + lane;
  for (uint32_t r = 0; r <= rows; ++r) mine[r * 32] = both(0.f);
  const int slab = blockIdx.y * kTableSlab;
  const int c0 = slab + lane * kU;  // the lane's first channel
  const uint64_t begin = (static_cast<uint64_t>(blockIdx.x) * warps + warp) * a.share;
  const uint32_t lo = begin < a.tokens ? static_cast<uint32_t>(begin) : a.tokens, hi = min(a.tokens, lo + a.share);

  // lanes behind the row's end read its first channels, and nothing that they add is written
  int at[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) at[u] = c0 + u * 32 < a.d ? c0 + u * 32 : slab;
  struct Batch {
    uint32_t key;  // of token `lane` of the batch
    Raw x[kBatch][kUnits];
  };
  // The batch of tokens t0 ...; what lies behind the share has no embedding and is read as its last token.
  auto fetch = [&](uint32_t t0, Batch& b) {
    b.key = lane < kBatch && t0 + lane < hi ? min(a.index.at(t0 + lane), rows) : rows;
    if (t0 >= hi) return;
    const T* p = a.d_out + static_cast<int64_t>(t0) * a.d;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) b.x[k][u] = __ldcs(reinterpret_cast<const Raw*>(p + at[u]));
      if (t0 + k + 1 < hi) p += a.d;
    }
  };
  auto value = [](const Raw (&x)[kUnits]) {
    Unit<T, kU> o[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) o[u] = reinterpret_cast<const Unit<T, kU>&>(x[u]);
    return unpack_all<T, kU, kUnits>(o).p[0];
  };
  auto take = [&](const Batch& b) {
    // a batch of one bin (far positions, padding) is summed in registers
    const uint32_t first = __shfl_sync(0xffffffffu, b.key, 0);
    if (__all_sync(0xffffffffu, b.key == first || lane >= kBatch)) {
      float2 sum = value(b.x[0]);
#pragma unroll
      for (int k = 1; k < kBatch; ++k) sum = __fadd2_rn(sum, value(b.x[k]));
      mine[first * 32] = __fadd2_rn(mine[first * 32], sum);
      return;
    }
    // Four tokens at a time: their rows of the table are read together, and where two are the same row the later one adds to
    // what the earlier one made of it and is written after it.  (One by one, with equal neighbours joined: 98 us for 768 x 768 random
    // bins of 66 against 60.)
#pragma unroll
    for (int k = 0; k < kBatch; k += 4) {
      uint32_t key[4];
      float2 sum[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) key[e] = __shfl_sync(0xffffffffu, b.key, k + e);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = mine[key[e] * 32];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int f = 0; f < e; ++f) sum[e] = key[f] == key[e] ? sum[f] : sum[e];
        sum[e] = __fadd2_rn(sum[e], value(b.x[k + e]));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[key[e] * 32] = sum[e];
    }
  };
  Batch x, y;
  fetch(lo, x);
  for (uint32_t t = lo; t < hi; t += 2 * kBatch) {
    fetch(t + kBatch, y);
    take(x);
    fetch(t + 2 * kBatch, x);
    take(y);
  }
  __syncthreads();
  for (uint32_t n = threadIdx.x; n < rows * 32; n += blockDim.x) {
    double s0 = 0.0, s1 = 0.0;
    for (int w = 0; w < warps; ++w) {
      const float2 v = tables[w * (rows + 1) * 32 + n];
      s0 += v.x, s1 += v.y;
    }
    float* to = a.partial + (static_cast<int64_t>(blockIdx.x) * rows + (n >> 5)) * a.d;
    const int c = slab + (n & 31) * kU, other = c + (kU == 2 ? 1 : 32);
    if (c < a.d) to[c] = static_cast<float>(s0);
    if (other < a.d) to[other] = static_cast<float>(s1);
  }
}

// d_table[n] = scale x the sum over the CTAs' tables: 32 values and 32 tables per CTA.
__global__ void __launch_bounds__(1024) join_tables_kernel(const float* partial, int parts, int64_t size, void* d_table, int dtype,
                                                          float scale) {
  behind_previous();
  __shared__ double s[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 32 + x;
  double sum = 0.0;
  if (n < size) {
#pragma unroll 4
    for (int r = y; r < parts; r += 32) sum += partial[r * size + n];
  }
  s[y][x] = sum;
#pragma unroll
  for (int half = 16; half > 0; half /= 2) {
    __syncthreads();
    if (y < half) s[y][x] += s[y + half][x];
  }
  if (y == 0 && n < size) store_any(d_table, n, dtype, static_cast<float>(s[0][x]) * scale);
}

// ---------------------------------------------------------------------------------------------
// stable counting sort of the token numbers
// ---------------------------------------------------------------------------------------------
// The tokens are cut into `tiles` equal tiles, one per warp.  Pass: count each tile's digits (counts[bin][tile]), scan
// every bin over the tiles, then place each token behind its bin's, its tile's and its own predecessors.
struct Entry {
  uint32_t token, key;  // key: the token's table row, or the number of rows where it has none
};

struct SortArgs {
  IndexView index;
  const Entry* in;  // the order of the passes so far; nullptr: tokens 0, 1, 2, ...
  Entry* out;
  uint32_t* counts;  // (bins, tiles)
  uint32_t* totals;  // (bins)
  uint32_t tokens, tiles, tile;
  int shift, bins;
  uint4* clear;  // nullable: the first pass also clears the table's gradient, for the rows that no token names
  int64_t clear_vecs;
};

// Tokens without an embedding sort behind all others: their key is the number of rows.
__device__ __forceinline__ Entry entry_of(const SortArgs& a, uint32_t p) {
  if (a.in != nullptr) {
    const uint2 e = __ldcg(reinterpret_cast<const uint2*>(a.in) + p);
    return Entry{e.x, e.y};
  }
  const uint32_t row = a.index.at(p);
  return Entry{p, row == kNone ? a.index.rows : row};
}

__global__ void __launch_bounds__(kSortWarps * 32) sort_count_kernel(const SortArgs a) {
  next_may_start();
  behind_previous();
  extern __shared__ uint32_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* mine = smem + warp * a.bins;
  const uint32_t w = blockIdx.x * kSortWarps + warp;
  if (a.clear != nullptr)
    for (int64_t n = static_cast<int64_t>(blockIdx.x) * (kSortWarps * 32) + threadIdx.x; n < a.clear_vecs;
         n += static_cast<int64_t>(gridDim.x) * (kSortWarps * 32))
      a.clear[n] = make_uint4(0, 0, 0, 0);
  for (int k = lane; k < a.bins; k += 32) mine[k] = 0;
  __syncwarp();
  if (w >= a.tiles) return;
  const uint32_t lo = min(a.tokens, w * a.tile), hi = min(a.tokens, lo + a.tile);
  for (uint32_t p0 = lo; p0 < hi; p0 += 128) {
    uint32_t digit[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t p = p0 + k * 32 + lane;
      digit[k] = p < hi ? (entry_of(a, p).key >> a.shift) & (a.bins - 1) : kNone;
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

// Exclusive scan of one bin's counts over the tiles, a run of neighbours per thread; the bin's total beside it.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(uint32_t* counts, uint32_t* totals, uint32_t tiles) {
  next_may_start();
  behind_previous();
  __shared__ uint32_t part[kThreads / 32];
  uint32_t* c = counts + static_cast<int64_t>(blockIdx.x) * tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t per = (tiles + kThreads - 1) / kThreads;
  const uint32_t lo = min(tiles, threadIdx.x * per), hi = min(tiles, lo + per);
  uint32_t own = 0;
#pragma unroll 8
  for (uint32_t k = lo; k < hi; ++k) own += c[k];
  uint32_t x = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += up;
  }
  if (lane == 31) part[warp] = x;
  __syncthreads();
  uint32_t before = x - own, all = 0;
#pragma unroll
  for (int k = 0; k < kThreads / 32; ++k) {
    if (k < warp) before += part[k];
    all += part[k];
  }
#pragma unroll 8
  for (uint32_t k = lo; k < hi; ++k) {
    const uint32_t n = c[k];
    c[k] = before;
    before += n;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = all;
}

__global__ void __launch_bounds__(kSortWarps * 32) sort_place_kernel(const SortArgs a) {
  next_may_start();
  behind_previous();
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
    Entry entry[4];
    uint32_t digit[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t p = p0 + k * 32 + lane;
      digit[k] = kNone;
      if (p < hi) {
        entry[k] = entry_of(a, p);
        digit[k] = (entry[k].key >> a.shift) & (a.bins - 1);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t same = __match_any_sync(0xffffffffu, digit[k]);
      const uint32_t at = digit[k] != kNone ? next[digit[k]] : 0;
      __syncwarp();
      if (digit[k] != kNone) {
        a.out[at + __popc(same & ((1u << lane) - 1))] = entry[k];
        if (lane == __ffs(same) - 1) next[digit[k]] = at + __popc(same);
      }
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------------------------------------
// sums over the sorted tokens
// ---------------------------------------------------------------------------------------------
// The sorted tokens are cut into equal shares, one per group of lanes; the shares of a CTA are neighbours.  A run (equal
// indices) inside one share goes straight to the table.  A run that crosses shares leaves a piece in each: the CTA joins the pieces of
// its own shares, and what crosses CTAs is left in the workspace with the CTA's edges, for the second kernel.
struct Edge {
  uint32_t first, last;  // index of the first and last run
  uint32_t bits;
  uint32_t pad;
};
constexpr uint32_t kFromLeft = 1, kToRight = 2, kOneRun = 4;

template <typename T>
struct SumArgs {
  const Entry* sorted;
  const T* d_out;
  void* d_table;
  float* pieces;  // (CTAs, 2, width): what crosses into the CTA, and what begins in it and crosses out
  Edge* edges;    // (CTAs)
  uint32_t tokens, rows, share, ctas;
  int d, width, table_dtype;
  float scale;
};

// Four entries at a time are a batch.  The rows of octs of 16-bit types travel through a ring of two batches of asynchronous
// copies per lane; others are loaded when their batch is at hand.  Four CTAs an SM with two batches take 30 us for 768 x 768
// positions of 128 channels, three CTAs with three 34, two with four 40 (and two waves of any more than one).
constexpr int kBatch = 4, kSumRing = 2, kSumCtas = 4;
template <typename T, bool kWide>
constexpr bool kSumStaged = kWide && sizeof(T) == 2;

template <typename T, int kGroup, bool kWide>
__global__ void __launch_bounds__(kThreads, kSumCtas) sum_runs_kernel(const SumArgs<T> a) {
  next_may_start();
  behind_previous();
  constexpr int kGroups = kThreads / kGroup;
  constexpr int kChannels = kGroup * 8;
  constexpr bool kStaged = kSumStaged<T, kWide>;
  __shared__ float piece[2][kGroups][kChannels];
  __shared__ Edge edge[kGroups];
  extern __shared__ uint4 ring[];
  const int lane = threadIdx.x % kGroup, group = threadIdx.x / kGroup;
  const uint32_t share = blockIdx.x * kGroups + group;
  const int slab = blockIdx.y * kSlab, left = a.d - slab;
  // 64 bits: the last CTA's shares may begin behind 2^32
  const uint64_t begin = static_cast<uint64_t>(share) * a.share;
  const uint32_t lo = begin < a.tokens ? static_cast<uint32_t>(begin) : a.tokens;
  const uint32_t hi = min(a.tokens, lo + a.share);

  // The groups of a warp stay together: the loop is as long for a group whose share is short or empty (its entries have no table
  // row then), and only what a run's end writes is done by some groups alone.
  struct Batch {
    uint32_t token[kBatch], key[kBatch];
  };
  auto entries_of = [&](uint32_t q) {  // of the share's entries q .. q + 3; q, the share and its begin are multiples of 4
    Batch b;
    uint4 x = make_uint4(0, a.rows, 0, a.rows), y = x;
    if (q < a.share && lo + q < hi) {  // (behind the last token there is padding)
      x = __ldcg(reinterpret_cast<const uint4*>(a.sorted + lo + q));
      y = __ldcg(reinterpret_cast<const uint4*>(a.sorted + lo + q) + 1);
      if (hi - (lo + q) < kBatch) {
        y.w = a.rows;
        if (hi - (lo + q) < 3) y.y = a.rows;
        if (hi - (lo + q) < 2) x.w = a.rows;
      }
    }
    b.token[0] = x.x, b.token[1] = x.z, b.token[2] = y.x, b.token[3] = y.z;
    b.key[0] = x.y, b.key[1] = x.w, b.key[2] = y.y, b.key[3] = y.w;
    return b;
  };
  const T* const d_out = a.d_out + slab;
  auto fetch = [&](const Batch& b, int stage) {
    if constexpr (kStaged) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (b.key[k] != a.rows && lane * 8 < left)
          stage_unit<T, 8>(ring + (stage * kBatch + k) * kThreads + threadIdx.x,
                           d_out + static_cast<int64_t>(b.token[k]) * a.d + lane * 8);
      stage_commit();
    }
  };

  // keys of the batches whose copies are under way, the one at hand first, and the entries of the batch after them
  constexpr int kAhead = kStaged ? kSumRing - 1 : 1;
  uint32_t key[kAhead][kBatch];
  Batch next;
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    next = entries_of(k * kBatch);
    fetch(next, k);
#pragma unroll
    for (int e = 0; e < kBatch; ++e) key[k][e] = next.key[e];
  }
  if constexpr (kStaged) next = entries_of(kAhead * kBatch);

  float2 total[4], acc[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) total[e] = acc[e] = both(0.f);
  const uint32_t before = lo > 0 && lo < hi ? a.sorted[lo - 1].key : a.rows;
  const uint32_t after = lo < hi && hi < a.tokens ? a.sorted[hi].key : a.rows;
  const uint32_t first = key[0][0];
  const bool crosses_in = first != a.rows && before == first;
  uint32_t run = first;  // the run at hand
  bool from_left = crosses_in, one = true;

  auto end_run = [&] {
    if (from_left) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        piece[0][group][channel_of<kWide, kGroup>(lane, 2 * e)] = total[e].x + acc[e].x;
        piece[0][group][channel_of<kWide, kGroup>(lane, 2 * e + 1)] = total[e].y + acc[e].y;
      }
    } else {
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = (total[e].x + acc[e].x) * a.scale;
        f[2 * e + 1] = (total[e].y + acc[e].y) * a.scale;
      }
      store_eight<kWide, kGroup>(a.d_table, a.table_dtype, static_cast<int64_t>(run) * a.d + slab, lane, left, f);
    }
  };
  auto add = [&](const Unit<T, 8>& o) {
    const Lane<8, 1> v = unpack(o);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = __fadd2_rn(acc[e], v.p[e]);
  };

  int stage = 0;
#pragma unroll 1
  for (uint32_t q = 0; q < a.share; q += kBatch) {
    if constexpr (kStaged) {
      fetch(next, stage == 0 ? kSumRing - 1 : stage - 1);
      stage_wait<kSumRing - 1>();
    }
    const uint4* slot = ring + stage * kBatch * kThreads + threadIdx.x;
    bool same = true;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) same = same && key[0][k] == run;
    if (__all_sync(0xffffffffu, same)) {
      if (run != a.rows) {
        Unit<T, 8> o[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if constexpr (kStaged)  // (lanes behind the row's end add what their slot holds: those sums go nowhere)
            o[k] = staged_unit<T, 8>(slot + k * kThreads);
          else
            o[k] = load_eight<kWide, kGroup>(d_out + static_cast<int64_t>(next.token[k]) * a.d, lane, left);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) add(o[k]);
      }
    } else {
#pragma unroll 1
      for (uint32_t k = 0; k < kBatch && lo + q + k < hi; ++k) {
        const Entry e = a.sorted[lo + q + k];
        if (e.key != run) {
          if (run != a.rows) end_run();
          run = e.key;
          from_left = one = false;
#pragma unroll
          for (int c = 0; c < 4; ++c) total[c] = acc[c] = both(0.f);
        }
        if (run != a.rows) {
          if constexpr (kStaged)
            add(staged_unit<T, 8>(slot + k * kThreads));
          else
            add(load_eight<kWide, kGroup>(d_out + static_cast<int64_t>(e.token) * a.d, lane, left));
        }
      }
    }
    // sums of at most 32 terms first: the error grows with the root of either count
    if ((q / kBatch & 7) == 7) {
#pragma unroll
      for (int e = 0; e < 4; ++e) total[e] = __fadd2_rn(total[e], acc[e]), acc[e] = both(0.f);
    }
    if constexpr (kStaged) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int e = 0; e < kBatch; ++e) key[k][e] = k + 1 < kAhead ? key[k + 1 < kAhead ? k + 1 : 0][e] : next.key[e];
      next = entries_of(q + (kAhead + 1) * kBatch);
      stage = stage == kSumRing - 1 ? 0 : stage + 1;
    } else {
      next = entries_of(q + kBatch);
#pragma unroll
      for (int e = 0; e < kBatch; ++e) key[0][e] = next.key[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) total[e] = __fadd2_rn(total[e], acc[e]), acc[e] = both(0.f);
  if (lo < hi) {
    const bool to_right = run != a.rows && after == run;
    if (to_right && !from_left) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        piece[1][group][channel_of<kWide, kGroup>(lane, 2 * e)] = total[e].x;
        piece[1][group][channel_of<kWide, kGroup>(lane, 2 * e + 1)] = total[e].y;
      }
    } else if (run != a.rows) {
      end_run();
    }
    if (lane == 0) edge[group] = Edge{first, run, (crosses_in ? kFromLeft : 0) | (to_right ? kToRight : 0) | (one ? kOneRun : 0), 0};
  } else if (lane == 0) {
    edge[group] = Edge{a.rows, a.rows, kOneRun, 0};
  }
  __syncthreads();

  // Join the pieces of neighbouring shares, one channel per thread.
  const int c = threadIdx.x;
  if (c < kChannels && c < left) {
    double sum = 0.0;
    bool before = false;  // the run at hand began before this CTA
    bool open = false;
    for (int g = 0; g < kGroups; ++g) {
      const Edge s = edge[g];
      if (s.first == a.rows) break;  // tokens without an embedding, or behind the last one
      if (s.bits & kFromLeft) {
        if (g == 0) before = true;
        sum += piece[0][g][c];
        open = (s.bits & kOneRun) && (s.bits & kToRight);
        if (!open) {
          if (before)
            a.pieces[static_cast<int64_t>(blockIdx.x) * 2 * a.width + slab + c] = static_cast<float>(sum);
          else
            store_any(a.d_table, static_cast<int64_t>(s.first) * a.d + slab + c, a.table_dtype, static_cast<float>(sum) * a.scale);
          before = false;
        }
      }
      if ((s.bits & kToRight) && !((s.bits & kOneRun) && (s.bits & kFromLeft))) {
        sum = piece[1][g][c];
        open = true;
      }
    }
    if (open) a.pieces[(static_cast<int64_t>(blockIdx.x) * 2 + (before ? 0 : 1)) * a.width + slab + c] = static_cast<float>(sum);
  }
  if (threadIdx.x == 0 && blockIdx.y == 0) {
    // the CTA's own edges: it is one run when every share that has tokens is, and is entered or left as its outer shares are
    Edge out = edge[0];
    bool one = true;
    for (int g = 0; g < kGroups; ++g) {
      if (static_cast<uint64_t>(blockIdx.x * kGroups + g) * a.share >= a.tokens) break;
      one = one && (edge[g].bits & kOneRun) && edge[g].first == out.first;
      out.last = edge[g].last;
      out.bits = (out.bits & kFromLeft) | (edge[g].bits & kToRight);
    }
    out.bits |= one ? kOneRun : 0;
    a.edges[blockIdx.x] = out;
  }
}

// The CTA in which a crossing run begins adds up its pieces: its own [1], then [0] of the CTAs that follow.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_runs_kernel(const SumArgs<T> a) {
  behind_previous();
  __shared__ float4 sums[kThreads / 32][32];
  const uint32_t cta = blockIdx.x;
  const Edge own = a.edges[cta];
  if (!(own.bits & kToRight) || ((own.bits & kOneRun) && (own.bits & kFromLeft))) return;
  // the run ends in the first CTA that it does not fill and leave (the last CTA is left by none)
  __shared__ uint32_t stop;
  if (threadIdx.x == 0) stop = 0xffffffffu;
  for (uint32_t from = cta + 1;; from += kThreads) {
    __syncthreads();
    const uint32_t at = from + threadIdx.x;
    if (at >= a.ctas || (a.edges[at].bits & (kOneRun | kToRight)) != (kOneRun | kToRight)) atomicMin(&stop, at);
    __syncthreads();
    if (stop != 0xffffffffu) break;
  }
  const uint32_t end = stop + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // eight warps, each an equal part of the pieces in order; 128 channels at a time
  const uint32_t pieces = end - cta, per = (pieces + 7) / 8;
  const uint32_t p_lo = min(pieces, warp * per), p_hi = min(pieces, (warp + 1) * per);
  for (int c0 = blockIdx.y * 128; c0 < a.width; c0 += gridDim.y * 128) {
    const int c = c0 + lane * 4;
    double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
    if (c < a.width) {
#pragma unroll 8
      for (uint32_t k = p_lo; k < p_hi; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(a.pieces + (static_cast<int64_t>(cta + k) * 2 + (k == 0 ? 1 : 0)) * a.width + c);
        s0 += x.x, s1 += x.y, s2 += x.z, s3 += x.w;
      }
    }
    sums[warp][lane] = make_float4(static_cast<float>(s0), static_cast<float>(s1), static_cast<float>(s2), static_cast<float>(s3));
    __syncthreads();
    if (threadIdx.x < 128 && c0 + threadIdx.x < a.d) {
      double sum = 0.0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) sum += reinterpret_cast<const float*>(sums[w])[threadIdx.x];
      store_any(a.d_table, static_cast<int64_t>(own.last) * a.d + c0 + threadIdx.x, a.table_dtype, static_cast<float>(sum) * a.scale);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
struct Plan {
  bool few, by_token, small;
  int passes, digit_bits, bins, group, slabs, width;
  int warps;        // of a small table
  uint32_t parts;   // of a small table
  uint32_t tiles, tile, share, ctas;
  uint64_t sorted_at[2], counts_at, totals_at, pieces_at, edges_at, bytes;
};

inline uint64_t up256(uint64_t n) { return (n + 255) & ~255ull; }

Plan make_plan(const pair_embed_desc_t* d, int sms) {
  Plan p = {};
  const uint64_t tokens = static_cast<uint64_t>(d->tokens);
  p.slabs = (d->d + kSlab - 1) / kSlab;
  // Few tokens: looking through all indices once per table row (or, of a larger table, per token) and slab takes about 1.3 ns +
  // 0.8 ps a token for each of them, the sort 15 to 30 us whatever its size.  Up to 4096 tokens, so that a row that takes most
  // of them stays short too.  (Looking against sorting: 128 channels, 1024 tokens into 100 rows 2.4 against 15 us, 4096 into
  // 2048 rows 19 against 23, 2048 into 16384 rows 19 by token against 31; 512 channels, 4096 into 2048 rows 37 against 27.)
  // By token of tables with more rows than that, where clearing the table is worth its launch; a token's look costs about two rows'.
  p.by_token = static_cast<uint64_t>(d->rows) > tokens && static_cast<uint64_t>(d->rows) * p.slabs > 1024;
  p.few = tokens <= 4096 && (p.by_token ? 2 * tokens : d->rows) * p.slabs * (tokens + 1600) <= (1u << 24);
  // A small table takes longer by row than by a walk where most tokens share a row: 2304 tokens into 21 rows 23 us against 8.
  p.small = d->rows <= kTableRows && !(p.few && (tokens <= 1024 || tokens <= 64ull * d->rows));
  if (p.few && !p.small) {
    p.bytes = 256;
    return p;
  }
  p.few = false;
  if (p.small) {
    p.warps = kTableSmem / ((d->rows + 1) * kTableSlab * 4);
    if (p.warps > kTableWarps) p.warps = kTableWarps;
    const int slabs = (d->d + kTableSlab - 1) / kTableSlab;
    const uint64_t ctas = sms > slabs ? sms / slabs : 1;  // one CTA an SM
    const uint64_t wave = ctas * p.warps, waves = (tokens + wave * kTableShare - 1) / (wave * kTableShare);
    p.share = static_cast<uint32_t>(((tokens + waves * wave - 1) / (waves * wave) + 31) / 32 * 32);
    const uint64_t held = static_cast<uint64_t>(p.share) * p.warps;
    p.parts = static_cast<uint32_t>((tokens + held - 1) / held);
    p.bytes = up256(static_cast<uint64_t>(p.parts) * d->rows * d->d * 4);
    return p;
  }
  int bits = 1;
  while ((1ull << bits) <= static_cast<uint64_t>(d->rows)) ++bits;  // keys 0 .. rows
  p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  p.bins = 1 << p.digit_bits;
  // tiles of at least 64 tokens, at most 16 warps an SM, and at most two counters a token (one SM's worth of tiles aside)
  uint64_t most = 2 * tokens / p.bins > static_cast<uint64_t>(sms) ? 2 * tokens / p.bins : sms;
  if (most > static_cast<uint64_t>(sms) * 16) most = static_cast<uint64_t>(sms) * 16;
  uint64_t tiles = (tokens + 63) / 64;
  if (tiles > most) tiles = most;
  p.tile = static_cast<uint32_t>(((tokens + tiles - 1) / tiles + 31) / 32 * 32);
  p.tiles = static_cast<uint32_t>((tokens + p.tile - 1) / p.tile);
  // shares: one wave of resident groups over all slabs, of at least 8 tokens, in whole batches
  p.group = d->d <= 64 ? 8 : d->d <= 128 ? 16 : 32;
  p.width = (d->d + 7) / 8 * 8;
  const int groups = kThreads / p.group;
  uint64_t ctas = static_cast<uint64_t>(sms) * kSumCtas / p.slabs;
  if (ctas < 1) ctas = 1;
  uint64_t share = (tokens + ctas * groups - 1) / (ctas * groups);
  if (share < 8) share = 8;
  share = (share + kBatch - 1) / kBatch * kBatch;
  p.share = static_cast<uint32_t>(share);
  p.ctas = static_cast<uint32_t>((tokens + share * groups - 1) / (share * groups));
  uint64_t at = 0;
  p.sorted_at[0] = at, at += up256(tokens * sizeof(Entry));
  p.sorted_at[1] = at, at += p.passes > 1 ? up256(tokens * sizeof(Entry)) : 0;
  p.counts_at = at, at += up256(static_cast<uint64_t>(p.bins) * p.tiles * 4);
  p.totals_at = at, at += up256(static_cast<uint64_t>(p.bins) * 4);
  p.pieces_at = at, at += up256(static_cast<uint64_t>(p.ctas) * 2 * p.width * 4);
  p.edges_at = at, at += up256(static_cast<uint64_t>(p.ctas) * sizeof(Edge));
  p.bytes = at;
  return p;
}

template <typename T>
cudaError_t embed_run(const pair_embed_desc_t* d, const IndexView& index, const void* table, const void* base, void* out,
                      bool wide, int sms, cudaStream_t s) {
  EmbedArgs a;
  a.index = index;
  a.table = table;
  a.base = base;
  a.out = out;
  a.tokens = static_cast<uint32_t>(d->tokens);
  a.d = d->d;
  a.octs = (d->d + 7) / 8;
  a.table_dtype = d->table_dtype;
  a.scale = d->scale;
  if (wide) {
    static const int resident = resident_ctas(embed_octs_kernel<T>, kThreads, 0);
    const uint64_t need = (static_cast<uint64_t>(d->tokens) * a.octs + kThreads - 1) / kThreads;
    return launch(embed_octs_kernel<T>, walk_grid(need, sms, resident, 4), kThreads, 0, s, a, make_fast_div(a.octs));
  }
  static const int resident = resident_ctas(embed_pieces_kernel<T>, kThreads, 0);
  const uint32_t pieces = (a.d + 255) / 256;
  const uint64_t need = (static_cast<uint64_t>(d->tokens) * pieces + kThreads / 32 - 1) / (kThreads / 32);
  return launch(embed_pieces_kernel<T>, walk_grid(need, sms, resident, 4), kThreads, 0, s, a, make_fast_div(pieces));
}

template <typename T, bool kWide>
cudaError_t grad_run(const pair_embed_desc_t* d, const IndexView& index, const void* d_out, void* d_table, void* workspace,
                     int sms, cudaStream_t s) {
  const Plan p = make_plan(d, sms);
  const uint32_t tokens = static_cast<uint32_t>(d->tokens);
  if (p.few) {
    const int64_t ctas = (p.by_token ? d->tokens : d->rows) * p.slabs;
    const int warps = ctas <= 2 * sms ? 32 : ctas <= 4096 ? 16 : 8;
    if (p.by_token) {
      const cudaError_t e = cudaMemsetAsync(d_table, 0, static_cast<size_t>(d->rows) * d->d * type_bytes(d->table_dtype), s);
      if (e != cudaSuccess) return e;
    }
    return launch(p.by_token ? embed_grad_few_kernel<T, kWide, true> : embed_grad_few_kernel<T, kWide, false>,
                  dim3(static_cast<unsigned>(p.by_token ? d->tokens : d->rows), p.slabs), warps * 32, warps * kSlab * sizeof(float), s,
                  index, static_cast<const T*>(d_out), d_table, static_cast<int>(d->table_dtype), tokens,
                  (tokens + warps * 32 - 1) / (warps * 32) * 32, static_cast<int>(d->d), d->scale);
  }
  if (p.small) {
    TableArgs<T> a{index, static_cast<const T*>(d_out), static_cast<float*>(workspace), tokens, p.share, static_cast<int>(d->d)};
    const bool pairs = d->d % 2 == 0 && aligned(d_out, 2 * sizeof(T));
    auto kernel = pairs ? embed_grad_table_kernel<T, 2> : embed_grad_table_kernel<T, 1>;
    const int smem = p.warps * (d->rows + 1) * kTableSlab * 4;
    // all that any table takes: the attribute is the kernel's, and another thread's smaller table must not lower it before this launch
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTableSmem);
    if (e == cudaSuccess) e = launch(kernel, dim3(p.parts, (d->d + kTableSlab - 1) / kTableSlab), p.warps * 32, smem, s, a);
    if (e != cudaSuccess) return e;
    const int64_t size = static_cast<int64_t>(d->rows) * d->d;
    return launch_behind(join_tables_kernel, static_cast<unsigned>((size + 31) / 32), 1024, 0, s, static_cast<const float*>(a.partial), static_cast<int>(p.parts), size,
                         d_table, static_cast<int>(d->table_dtype), d->scale);
  }
  char* ws = static_cast<char*>(workspace);
  cudaError_t e;
  SortArgs a;
  a.index = index;
  a.counts = reinterpret_cast<uint32_t*>(ws + p.counts_at);
  a.totals = reinterpret_cast<uint32_t*>(ws + p.totals_at);
  a.tokens = tokens;
  a.tiles = p.tiles;
  a.tile = p.tile;
  a.bins = p.bins;
  a.in = nullptr;
  // rows that no token names become 0; the others are written afterwards
  const uint64_t table_bytes = static_cast<uint64_t>(d->rows) * d->d * type_bytes(d->table_dtype);
  a.clear = nullptr;
  a.clear_vecs = static_cast<int64_t>(table_bytes / 16);
  if (aligned(d_table, 16) && table_bytes % 16 == 0) {
    a.clear = static_cast<uint4*>(d_table);
  } else {
    e = cudaMemsetAsync(d_table, 0, table_bytes, s);
    if (e != cudaSuccess) return e;
  }
  const int count_smem = kSortWarps * p.bins * 4, place_smem = (kSortWarps + 1) * p.bins * 4;
  const unsigned grid = (p.tiles + kSortWarps - 1) / kSortWarps;
  for (int pass = 0; pass < p.passes; ++pass) {
    // the last pass ends in buffer 0
    a.out = reinterpret_cast<Entry*>(ws + p.sorted_at[(p.passes - 1 - pass) & 1]);
    a.shift = pass * p.digit_bits;
    // clearing takes every SM, whatever the tiles need
    const unsigned busy = a.clear != nullptr && grid < 4u * sms ? 4u * sms : grid;
    e = pass == 0 ? launch(sort_count_kernel, busy, kSortWarps * 32, count_smem, s, a)
                  : launch_behind(sort_count_kernel, busy, kSortWarps * 32, count_smem, s, a);
    if (e == cudaSuccess) e = launch_behind(sort_scan_kernel, p.bins, kThreads, 0, s, a.counts, a.totals, a.tiles);
    if (e == cudaSuccess) e = launch_behind(sort_place_kernel, grid, kSortWarps * 32, place_smem, s, a);
    if (e != cudaSuccess) return e;
    a.in = a.out;
    a.clear = nullptr;
  }
  SumArgs<T> m;
  m.sorted = a.in;
  m.rows = static_cast<uint32_t>(d->rows);
  m.d_out = static_cast<const T*>(d_out);
  m.d_table = d_table;
  m.pieces = reinterpret_cast<float*>(ws + p.pieces_at);
  m.edges = reinterpret_cast<Edge*>(ws + p.edges_at);
  m.tokens = tokens;
  m.share = p.share;
  m.ctas = p.ctas;
  m.d = d->d;
  m.width = p.width;
  m.table_dtype = d->table_dtype;
  m.scale = d->scale;
  const dim3 sum_grid(p.ctas, p.slabs);
  const int smem = kSumStaged<T, kWide> ? kSumRing * kBatch * kThreads * 16 : 0;
  auto kernel = p.group == 8 ? sum_runs_kernel<T, 8, kWide> : p.group == 16 ? sum_runs_kernel<T, 16, kWide> : sum_runs_kernel<T, 32, kWide>;
  if (smem > 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  e = launch_behind(kernel, sum_grid, kThreads, smem, s, m);
  if (e != cudaSuccess) return e;
  const int quads = (p.width + 127) / 128;
  return launch_behind(join_runs_kernel<T>, dim3(p.ctas, quads < 4 ? quads : 4), kThreads, 0, s, m);
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
  if (!elements_aligned(type_bytes(desc->dtype), {}, {base, out}) || !aligned(index, desc->index_bits / 8) ||
      !aligned(table, type_bytes(desc->table_dtype)))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: a buffer is not aligned to its elements", who);
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  const IndexView view{index, desc->index_bits, static_cast<uint32_t>(desc->rows)};
  const bool wide = desc->d % 8 == 0 && aligned(table, 16) && aligned(base, 16) && aligned(out, 16);
  cudaError_t e;
  if (desc->dtype == PAIR_FP32)
    e = embed_run<float>(desc, view, table, base, out, wide, sms, cuda_stream);
  else if (desc->dtype == PAIR_FP16)
    e = embed_run<__half>(desc, view, table, base, out, wide, sms, cuda_stream);
  else
    e = embed_run<__nv_bfloat16>(desc, view, table, base, out, wide, sms, cuda_stream);
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
  if (workspace == nullptr || !aligned(workspace, 16))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace", who);
  if (!aligned(d_out, type_bytes(desc->dtype)) || !aligned(index, desc->index_bits / 8) ||
      !aligned(d_table, type_bytes(desc->table_dtype)))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: a buffer is not aligned to its elements", who);
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  const IndexView view{index, desc->index_bits, static_cast<uint32_t>(desc->rows)};
  const bool wide = desc->d % 8 == 0 && aligned(d_out, 16) && aligned(d_table, 16);
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
