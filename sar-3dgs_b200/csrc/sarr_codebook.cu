// Codebook rows: Gaussians whose parameter rows (SH) are taken from a shared
// table by index, and the gradient of that table.
//
//   lookup    rows[i,:] = scale * table[index[i],:], zeros where index[i] is
//             outside [0, codes) (a Gaussian without a code)
//   sort      the stable order of the Gaussians by code: order, the code at each
//             place, and where each code's places begin
//   gradient  grad_table[c,:] = scale * sum of grad_rows[i,:] over the Gaussians
//             i with index[i] = c, zeros for a code that none has
//
// Sums are in 32 bits and in a fixed order (the sort is stable and nothing is
// added by atomics), so the same inputs give the same bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>

#include "sarr.h"
#include "sarr_launch.cuh"

namespace sarr {
void count_launches(int k);  // the library's launch counter (sarr_abi.cu)
}

namespace {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// A word of rows that are used again (kAgain: kept in L1) or once (from L2).
template <bool kAgain, typename W>
__device__ __forceinline__ W load_word(const W* p) {
  return kAgain ? __ldg(p) : __ldcg(p);
}

// kV consecutive elements as floats; p is aligned to min(16, kV * sizeof(T)) bytes.
template <bool kAgain, typename T, int kV>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[kV]) {
  constexpr int kBytes = kV * (int)sizeof(T);
  T t[kV];
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int k = 0; k < kBytes / 16; ++k) {
      const uint4 q = load_word<kAgain>(reinterpret_cast<const uint4*>(p) + k);
      memcpy(reinterpret_cast<char*>(t) + 16 * k, &q, 16);
    }
  } else if constexpr (kBytes == 8) {
    const uint2 q = load_word<kAgain>(reinterpret_cast<const uint2*>(p));
    memcpy(t, &q, 8);
  } else if constexpr (kBytes == 4) {
    const unsigned q = load_word<kAgain>(reinterpret_cast<const unsigned*>(p));
    memcpy(t, &q, 4);
  } else {
    const unsigned short q = load_word<kAgain>(reinterpret_cast<const unsigned short*>(p));
    memcpy(t, &q, 2);
  }
#pragma unroll
  for (int k = 0; k < kV; ++k) x[k] = to_float(t[k]);
}

template <typename T, int kV>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[kV]) {
  constexpr int kBytes = kV * (int)sizeof(T);
  T t[kV];
#pragma unroll
  for (int k = 0; k < kV; ++k) t[k] = from_float<T>(x[k]);
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int k = 0; k < kBytes / 16; ++k) {
      uint4 q;
      memcpy(&q, reinterpret_cast<const char*>(t) + 16 * k, 16);
      reinterpret_cast<uint4*>(p)[k] = q;
    }
  } else if constexpr (kBytes == 8) {
    uint2 q;
    memcpy(&q, t, 8);
    *reinterpret_cast<uint2*>(p) = q;
  } else if constexpr (kBytes == 4) {
    uint32_t q;
    memcpy(&q, t, 4);
    *reinterpret_cast<uint32_t*>(p) = q;
  } else {
    p[0] = t[0];
  }
}

// index[i], or `codes` where it is outside [0, codes).
__device__ __forceinline__ uint32_t code_of(const void* index, bool wide, int64_t i, uint32_t codes) {
  const int64_t v = wide ? __ldg(static_cast<const long long*>(index) + i)
                         : (int64_t)__ldg(static_cast<const int*>(index) + i);
  return v >= 0 && v < (int64_t)codes ? (uint32_t)v : codes;
}

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------
constexpr int kLookupThreads = 256;
constexpr int kLookupRows = 4;  // rows per thread, their loads in flight together

struct LookupArgs {
  int64_t n;
  uint32_t codes;
  int vecs;    // vectors per row
  int lanes;   // threads per row (a power of two)
  bool wide;   // 64-bit indexes
  float scale;
  const void* index;
  const void* table;
  void* rows;
  int64_t table_stride, rows_stride;
};

template <typename TT, typename TR, int kV>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(const LookupArgs a) {
  const int lane = threadIdx.x & (a.lanes - 1), at_once = kLookupThreads / a.lanes;
  const int64_t i0 = (int64_t)blockIdx.x * at_once * kLookupRows + threadIdx.x / a.lanes;
  uint32_t code[kLookupRows];
#pragma unroll
  for (int k = 0; k < kLookupRows; ++k) {
    const int64_t i = i0 + (int64_t)k * at_once;
    code[k] = i < a.n ? code_of(a.index, a.wide, i, a.codes) : a.codes;
  }
  for (int v = lane; v < a.vecs; v += a.lanes) {
    float x[kLookupRows][kV];
#pragma unroll
    for (int k = 0; k < kLookupRows; ++k) {
      if (code[k] < a.codes) {
        load_vec<true, TT, kV>(static_cast<const TT*>(a.table) + code[k] * a.table_stride + (int64_t)v * kV, x[k]);
      } else {
#pragma unroll
        for (int j = 0; j < kV; ++j) x[k][j] = 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < kLookupRows; ++k) {
      const int64_t i = i0 + (int64_t)k * at_once;
      if (i >= a.n) continue;
      if (code[k] < a.codes) {  // a row without a code is zeros whatever the scale
#pragma unroll
        for (int j = 0; j < kV; ++j) x[k][j] *= a.scale;
      }
      store_vec<TR, kV>(static_cast<TR*>(a.rows) + i * a.rows_stride + (int64_t)v * kV, x[k]);
    }
  }
}

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------
// A stable sort of the keys (the codes, `codes` for none). The unit is a tile of
// up to 8192 keys that one CTA sorts in registers and shared memory: each warp
// holds a contiguous part of the tile, 32 keys a round; a key's rank among the
// warp's keys of its digit is a running count plus the lower lanes that vote for
// the same digit (one vote per bit, so a digit of 7 bits costs 7 votes whatever
// the keys are), and one scan over (digit, warp) gives every rank its place.
//
// Up to 8192 keys: one CTA, every digit, and the offsets (sort_tile_kernel).
//
// More: passes over digits of up to 13 bits (so one pass up to 8191 codes), of
// three kernels each, which the scheduler may overlap:
//   histogram  each tile's count of every digit, [tiles][bins]
//   prefix     per digit the counts of the earlier tiles, and the total
//   scatter    the tile sorted by the digit, written out behind the smaller digits
//              and the earlier tiles (in runs, since the tile is in order). The
//              first pass sorts its tile before it waits for the other two.
// With one pass the scan over the totals is the offsets.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kTileRounds = 8, kTile = kSortThreads * kTileRounds;
constexpr int kLocalBits = 7;                          // of a pass inside a tile
constexpr int kMaxDigitBits = 13, kMaxBins = 1 << kMaxDigitBits;
constexpr int kCountPitch = kSortWarps + 1;            // [digit][warp], padded against bank conflicts
constexpr int kCountWords = kCountPitch << kLocalBits;
constexpr int kPrefixThreads = 256, kPrefixBins = 32;  // bins of a CTA; its threads split the tiles 8 ways

struct SortArgs {
  int n;
  uint32_t codes;
  bool wide;
  const void* index;
  const uint32_t* key_in;  // null: the indexes
  const int32_t* place_in;
  uint32_t* key_out;
  int32_t* place_out;
  int32_t *counts, *totals;  // [tiles][bins], [bins]
  int shift, bits;           // of this pass's digit
  int tiles;
  int32_t* offsets;          // written by the scatter of a sort of one pass, else null
};

struct TileShared {
  uint32_t key[kTile];
  int32_t place[kTile];
  int32_t count[kCountWords];
  int32_t warp_sum[kSortWarps];
};

// Exclusive scan over the CTA's threads.
__device__ __forceinline__ int block_scan(int x, int32_t* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int before = lane < warp ? warp_sum[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  __syncthreads();
  return before + incl - x;
}

// One stable pass over the tile's keys, which the threads hold: element
// (warp * rounds + r) * 32 + lane in key[r]. On return S holds the tile in order
// and so do the threads.
__device__ __forceinline__ void tile_pass(TileShared& S, uint32_t (&key)[kTileRounds], int32_t (&place)[kTileRounds],
                                          int rounds, int len, int shift, int bits) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = 1 << bits;
  for (int i = tid; i < bins * kCountPitch; i += kSortThreads) S.count[i] = 0;
  __syncthreads();
  int rank[kTileRounds];
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    if (r < rounds) {
      const bool have = (warp * rounds + r) * 32 + lane < len;
      const uint32_t digit = (key[r] >> shift) & (bins - 1);
      uint32_t peers = __ballot_sync(0xffffffffu, have);
#pragma unroll
      for (int b = 0; b < kLocalBits; ++b) {  // the bits above `bits` are 0 in every lane
        const bool one = (digit >> b) & 1;
        const uint32_t ones = __ballot_sync(0xffffffffu, one);
        peers &= one ? ones : ~ones;
      }
      const uint32_t below = peers & ((1u << lane) - 1);
      int32_t* at = S.count + digit * kCountPitch + warp;
      const int before = have ? *at : 0;
      __syncwarp();
      if (have && below == 0) *at = before + __popc(peers);
      __syncwarp();
      rank[r] = before + __popc(below);
    }
  }
  __syncthreads();
  {  // scan in the order (digit, warp): bins / 32 entries per thread, at least one
    const int each = bins >= 32 ? bins / 32 : 1, first = tid * each;
    int x[(1 << kLocalBits) / 32], sum = 0;
#pragma unroll
    for (int k = 0; k < (1 << kLocalBits) / 32; ++k) {
      const int e = first + k;
      x[k] = k < each && e < bins * 32 ? S.count[(e >> 5) * kCountPitch + (e & 31)] : 0;
      sum += x[k];
    }
    int at = block_scan(sum, S.warp_sum);
#pragma unroll
    for (int k = 0; k < (1 << kLocalBits) / 32; ++k) {
      const int e = first + k;
      if (k < each && e < bins * 32) S.count[(e >> 5) * kCountPitch + (e & 31)] = at;
      at += x[k];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    if (r < rounds && (warp * rounds + r) * 32 + lane < len) {
      const int to = S.count[((key[r] >> shift) & (bins - 1)) * kCountPitch + warp] + rank[r];
      S.key[to] = key[r];
      S.place[to] = place[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int e = (warp * rounds + r) * 32 + lane;
    if (r < rounds && e < len) {
      key[r] = S.key[e];
      place[r] = S.place[e];
    }
  }
}

// The tile's keys into the threads, then sorted by `bits` bits from `shift`.
__device__ __forceinline__ void sort_tile(const SortArgs& a, TileShared& S, uint32_t (&key)[kTileRounds],
                                          int32_t (&place)[kTileRounds], int tile0, int len, int rounds, int shift,
                                          int bits) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int e = (warp * rounds + r) * 32 + lane;
    key[r] = 0;
    place[r] = 0;
    if (r < rounds && e < len) {
      const int i = tile0 + e;
      key[r] = a.key_in ? __ldcg(a.key_in + i) : code_of(a.index, a.wide, i, a.codes);
      place[r] = a.key_in ? __ldcg(a.place_in + i) : i;
    }
  }
  const int passes = (bits + kLocalBits - 1) / kLocalBits, each = (bits + passes - 1) / passes;
  for (int p = 0; p < passes; ++p)
    tile_pass(S, key, place, rounds, len, shift + p * each, min(each, bits - p * each));
}

extern __shared__ __align__(16) unsigned char s_sort[];

__global__ void __launch_bounds__(kSortThreads) sort_tile_kernel(const SortArgs a) {
  TileShared& S = *reinterpret_cast<TileShared*>(s_sort);
  uint32_t key[kTileRounds];
  int32_t place[kTileRounds];
  sarr::dependents_may_start();
  const int rounds = (a.n + kSortThreads - 1) / kSortThreads;
  sort_tile(a, S, key, place, 0, a.n, rounds, 0, a.bits);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int e = (warp * rounds + r) * 32 + lane;
    if (r < rounds && e < a.n) {
      a.key_out[e] = key[r];
      a.place_out[e] = place[r];
    }
  }
  // the first place whose key is >= c
#pragma unroll 4
  for (int64_t c = threadIdx.x; c <= a.codes; c += kSortThreads) {
    int lo = 0, hi = a.n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (S.key[mid] < (uint32_t)c) lo = mid + 1;
      else hi = mid;
    }
    a.offsets[c] = lo;
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_histogram_kernel(const SortArgs a) {
  __shared__ int32_t s_bin[kMaxBins];
  sarr::dependents_may_start();
  sarr::wait_for_previous();
  const int bins = 1 << a.bits, tile0 = blockIdx.x * kTile, len = min(kTile, a.n - tile0);
  for (int d = threadIdx.x; d < bins; d += kSortThreads) s_bin[d] = 0;
  uint32_t key[kTileRounds];
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int e = r * kSortThreads + threadIdx.x;
    if (e < len) key[r] = a.key_in ? __ldcg(a.key_in + tile0 + e) : code_of(a.index, a.wide, tile0 + e, a.codes);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r)
    if (r * kSortThreads + threadIdx.x < len) atomicAdd(s_bin + ((key[r] >> a.shift) & (bins - 1)), 1);
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) a.counts[(int64_t)blockIdx.x * bins + d] = s_bin[d];
}

// counts[t][d] becomes the sum of counts[0 .. t-1][d], totals[d] the sum of all.
__global__ void __launch_bounds__(kPrefixThreads) sort_prefix_kernel(const SortArgs a) {
  constexpr int kSplit = kPrefixThreads / kPrefixBins;
  __shared__ int32_t s_sum[kSplit][kPrefixBins];
  sarr::dependents_may_start();
  sarr::wait_for_previous();
  const int bins = 1 << a.bits, d = blockIdx.x * kPrefixBins + (threadIdx.x & (kPrefixBins - 1));
  const int part = threadIdx.x / kPrefixBins, per = (a.tiles + kSplit - 1) / kSplit;
  const int t0 = min(part * per, a.tiles), t1 = min(t0 + per, a.tiles);
  int32_t* c = a.counts + d;
  int sum = 0;
  if (d < bins) {
#pragma unroll 16
    for (int t = t0; t < t1; ++t) sum += __ldcg(c + (int64_t)t * bins);
  }
  s_sum[part][threadIdx.x & (kPrefixBins - 1)] = sum;
  __syncthreads();
  if (d >= bins) return;
  int at = 0, all = 0;
#pragma unroll
  for (int k = 0; k < kSplit; ++k) {
    const int x = s_sum[k][threadIdx.x & (kPrefixBins - 1)];
    if (k < part) at += x;
    all += x;
  }
  if (part == 0) a.totals[d] = all;
  for (int t = t0; t < t1; t += 16) {
    int x[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = t + k < t1 ? __ldcg(c + (int64_t)(t + k) * bins) : 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      if (t + k < t1) c[(int64_t)(t + k) * bins] = at;
      at += x[k];
    }
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const SortArgs a) {
  TileShared& S = *reinterpret_cast<TileShared*>(s_sort);
  int32_t* s_base = reinterpret_cast<int32_t*>(s_sort + sizeof(TileShared));  // [bins]
  uint32_t key[kTileRounds];
  int32_t place[kTileRounds];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bins = 1 << a.bits, tile0 = blockIdx.x * kTile, len = min(kTile, a.n - tile0);
  const int rounds = (len + kSortThreads - 1) / kSortThreads;
  sarr::dependents_may_start();
  if (a.key_in) sarr::wait_for_previous();  // the first pass's keys are the caller's
  sort_tile(a, S, key, place, tile0, len, rounds, a.shift, a.bits);
  if (!a.key_in) sarr::wait_for_previous();
  // where each digit begins, and in it this tile's keys
  {
    const int each = max(bins / kSortThreads, 1), first = tid * each;
    int x[kMaxBins / kSortThreads], sum = 0;
#pragma unroll
    for (int k = 0; k < kMaxBins / kSortThreads; ++k) {
      x[k] = k < each && first + k < bins ? __ldcg(a.totals + first + k) : 0;
      sum += x[k];
    }
    int before[kMaxBins / kSortThreads];
#pragma unroll
    for (int k = 0; k < kMaxBins / kSortThreads; ++k)
      before[k] = k < each && first + k < bins ? __ldcg(a.counts + (int64_t)blockIdx.x * bins + first + k) : 0;
    int at = block_scan(sum, S.warp_sum);
#pragma unroll
    for (int k = 0; k < kMaxBins / kSortThreads; ++k) {
      const int d = first + k;
      if (k < each && d < bins) {
        s_base[d] = at + before[k];
        if (a.offsets && blockIdx.x == 0 && d <= (int)a.codes) a.offsets[d] = at;
      }
      at += x[k];
    }
  }
  __syncthreads();
  // less the place in the tile where the digit begins
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int e = (warp * rounds + r) * 32 + lane;
    if (r < rounds && e < len) {
      const uint32_t d = (key[r] >> a.shift) & (bins - 1);
      if (e == 0 || ((S.key[e - 1] >> a.shift) & (bins - 1)) != d) s_base[d] -= e;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int e = (warp * rounds + r) * 32 + lane;
    if (r < rounds && e < len) {
      const int to = s_base[(key[r] >> a.shift) & (bins - 1)] + e;
      a.key_out[to] = key[r];
      a.place_out[to] = place[r];
    }
  }
}

// The first place whose code is >= c, for each c.
__global__ void __launch_bounds__(256) sort_offsets_kernel(int n, uint32_t codes, const int32_t* sorted,
                                                           int32_t* offsets) {
  sarr::dependents_may_start();
  sarr::wait_for_previous();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c > codes) return;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if ((uint32_t)sorted[mid] < (uint32_t)c) lo = mid + 1;
    else hi = mid;
  }
  offsets[c] = lo;
}

// ---------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------
// The places of the sorted order are cut into equal spans, one per CTA, and
// each span into equal parts, one per group of `lanes` threads that hold a row
// side by side: equal work whatever the codes' lengths. A group adds the rows
// of its part in order and writes the codes that lie inside it; the sums of
// codes that cross a part's border are joined through shared memory, those of
// codes that cross a span's border through the workspace, by grad_finish_kernel,
// which also writes the zeros of codes without Gaussians.
constexpr int kGradThreads = 256;
constexpr int kGradRows = 8;     // rows of a group loaded together
constexpr int kMaxPart = 64;     // places of a group, at most
constexpr int kMaxSpan = 2048;   // places of a CTA, at most
constexpr int kLongSpans = 16;   // spans from which a code's partials are added by a whole CTA

struct GradArgs {
  int64_t cols;
  uint32_t codes;
  int vecs, lanes, part;  // vectors per row; threads per row; places per group
  int span;               // places per CTA: part * (kGradThreads / lanes)
  float scale;
  const void* rows;
  int64_t rows_stride;
  const int32_t *order, *sorted, *offsets;
  void* table;
  int64_t table_stride;
  float* partial;  // [spans][2][cols]: a span's sum of the code open at its start (0) and at its end (1)
};

template <typename TT, int kV>
__device__ __forceinline__ void write_row(const GradArgs& a, uint32_t code, int v, const float (&sum)[kV]) {
  float x[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) x[j] = sum[j] * a.scale;
  store_vec<TT, kV>(static_cast<TT*>(a.table) + code * a.table_stride + (int64_t)v * kV, x);
}

template <int kV>
__device__ __forceinline__ void write_partial(const GradArgs& a, int span, int slot, int v, const float (&x)[kV]) {
  float* p = a.partial + ((int64_t)span * 2 + slot) * a.cols + (int64_t)v * kV;
#pragma unroll
  for (int j = 0; j < kV; ++j) p[j] = x[j];
}

template <typename TG, typename TT, int kV>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(const GradArgs a) {
  __shared__ int32_t s_code[kMaxSpan + 2];  // codes of the span, with its neighbours
  __shared__ int32_t s_row[kMaxSpan];
  __shared__ float s_head[kV][kGradThreads], s_tail[kV][kGradThreads];
  __shared__ uint8_t s_state[kGradThreads];  // per group
  enum : uint8_t { kHead = 1, kTail = 2, kThrough = 4 };
  sarr::dependents_may_start();
  sarr::wait_for_previous();

  const int tid = threadIdx.x, lane = tid & (a.lanes - 1), group = tid / a.lanes;
  const int groups = kGradThreads / a.lanes;
  const int n = a.offsets[a.codes];  // places with a code
  const int64_t p0 = (int64_t)blockIdx.x * a.span;
  if (p0 >= n) return;
  const int len = (int)(n - p0 < a.span ? n - p0 : a.span);
  for (int i = tid; i < len + 2; i += kGradThreads) {
    const int64_t p = p0 + i - 1;
    s_code[i] = p >= 0 && p < n ? a.sorted[p] : -1;
  }
  for (int i = tid; i < len; i += kGradThreads) s_row[i] = a.order[p0 + i];
  if (lane == 0) s_state[group] = 0;
  __syncthreads();

  const int v = blockIdx.y * a.lanes + lane;
  const bool active = v < a.vecs;
  const TG* rows = static_cast<const TG*>(a.rows) + (int64_t)v * kV;
  const int q0 = group * a.part, q1 = min(q0 + a.part, len);
  float acc[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
  if (q0 < q1) {
    int cur = s_code[q0 + 1];
    bool open = s_code[q0] == cur;  // the code began before this part
    uint8_t state = 0;
    for (int q = q0; q < q1; q += kGradRows) {
      float x[kGradRows][kV];
#pragma unroll
      for (int k = 0; k < kGradRows; ++k)
        if (q + k < q1 && active) load_vec<false, TG, kV>(rows + s_row[q + k] * a.rows_stride, x[k]);
#pragma unroll
      for (int k = 0; k < kGradRows; ++k) {
        if (q + k < q1) {
          const int c = s_code[q + k + 1];
          if (c != cur) {
            if (open) {
              state |= kHead;
#pragma unroll
              for (int j = 0; j < kV; ++j) s_head[j][tid] = acc[j];
            } else if (active) {
              write_row<TT, kV>(a, (uint32_t)cur, v, acc);
            }
            open = false;
            cur = c;
#pragma unroll
            for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
          }
          if (active) {
#pragma unroll
            for (int j = 0; j < kV; ++j) acc[j] += x[k][j];
          }
        }
      }
    }
    if (s_code[q1 + 1] == cur) {  // goes on behind this part
      state |= open ? kThrough : kTail;
#pragma unroll
      for (int j = 0; j < kV; ++j) s_tail[j][tid] = acc[j];
    } else if (open) {
      state |= kHead;
#pragma unroll
      for (int j = 0; j < kV; ++j) s_head[j][tid] = acc[j];
    } else if (active) {
      write_row<TT, kV>(a, (uint32_t)cur, v, acc);
    }
    if (lane == 0) s_state[group] = state;
  }
  __syncthreads();
  if (q0 >= q1 || !active) return;
  const uint8_t state = s_state[group];
  if (group == 0 && (state & kHead)) {  // the code open at the span's start ends in its first part
    float x[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) x[j] = s_head[j][tid];
    write_partial<kV>(a, blockIdx.x, 0, v, x);
  }
  // the group where an open code begins (or the span's first) adds its pieces
  if ((state & kTail) || (group == 0 && (state & kThrough))) {
#pragma unroll
    for (int j = 0; j < kV; ++j) acc[j] = s_tail[j][tid];
    bool closed = false;
    for (int h = group + 1; h < groups && !closed; ++h) {
      const uint8_t sh = s_state[h];
      if (!sh) break;  // behind the span's last place
      closed = (sh & kThrough) == 0;
      const int from = h * a.lanes + lane;
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[j] += closed ? s_head[j][from] : s_tail[j][from];
    }
    const bool from_start = (state & kThrough) != 0;
    if (!closed) write_partial<kV>(a, blockIdx.x, 1, v, acc);
    else if (from_start) write_partial<kV>(a, blockIdx.x, 0, v, acc);
    else write_row<TT, kV>(a, (uint32_t)s_code[q1], v, acc);
  }
}

// Codes without Gaussians (zeros) and codes over several spans (the sum of
// their partials, in the order of the spans).
template <typename TT, int kV>
__global__ void __launch_bounds__(kGradThreads) grad_finish_kernel(const GradArgs a) {
  __shared__ int s_long[kGradThreads];
  __shared__ int s_n_long;
  __shared__ float s_sum[kV][kGradThreads];
  sarr::wait_for_previous();
  const int tid = threadIdx.x, lane = tid & (a.lanes - 1), group = tid / a.lanes;
  const int groups = kGradThreads / a.lanes;
  const int v = blockIdx.y * a.lanes + lane;
  const bool active = v < a.vecs;
  if (tid == 0) s_n_long = 0;
  __syncthreads();
  const int64_t c = (int64_t)blockIdx.x * groups + group;
  if (c < a.codes) {
    const int begin = a.offsets[c], end = a.offsets[c + 1];
    float acc[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
    if (begin == end) {
      if (active) store_vec<TT, kV>(static_cast<TT*>(a.table) + c * a.table_stride + (int64_t)v * kV, acc);
    } else {
      const int first = begin / a.span, last = (end - 1) / a.span;
      if (last - first >= kLongSpans) {
        if (lane == 0) s_long[atomicAdd(&s_n_long, 1)] = group;
      } else if (last > first && active) {
        for (int s = first; s <= last; ++s) {
          const float* p = a.partial + ((int64_t)s * 2 + (s < last)) * a.cols + (int64_t)v * kV;
#pragma unroll
          for (int j = 0; j < kV; ++j) acc[j] += p[j];
        }
        write_row<TT, kV>(a, (uint32_t)c, v, acc);
      }
    }
  }
  __syncthreads();
  for (int k = 0; k < s_n_long; ++k) {  // the order of these codes does not matter
    const int64_t code = (int64_t)blockIdx.x * groups + s_long[k];
    const int begin = a.offsets[code], end = a.offsets[code + 1];
    const int first = begin / a.span, last = (end - 1) / a.span;
    float acc[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
    if (active) {
#pragma unroll 4
      for (int s = first + group; s <= last; s += groups) {
        const float* p = a.partial + ((int64_t)s * 2 + (s < last)) * a.cols + (int64_t)v * kV;
#pragma unroll
        for (int j = 0; j < kV; ++j) acc[j] += p[j];
      }
    }
#pragma unroll
    for (int j = 0; j < kV; ++j) s_sum[j][tid] = acc[j];
    for (int half = groups / 2; half > 0; half /= 2) {
      __syncthreads();
      if (group < half) {
#pragma unroll
        for (int j = 0; j < kV; ++j) s_sum[j][tid] += s_sum[j][tid + half * a.lanes];
      }
    }
    __syncthreads();
    if (group == 0 && active) {
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[j] = s_sum[j][tid];
      write_row<TT, kV>(a, (uint32_t)code, v, acc);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int cuda_status(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  else cudaGetLastError();
  return e == cudaSuccess ? SARR_OK : SARR_ERR_CUDA;
}

constexpr int64_t kMaxCols = 1 << 22;
constexpr int64_t kMaxCount = 2147483647 - (1 << 19);  // Gaussians and codes

size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }
int type_size(int type) { return type == SARR_F32 ? 4 : 2; }
bool type_ok(int type) { return type == SARR_F32 || type == SARR_BF16 || type == SARR_F16; }
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int pow2_at_least(int64_t x, int most) {
  int p = 1;
  while (p < x && p < most) p *= 2;
  return p;
}

// Elements of a vector access that rows of both arrays allow: 16 bytes of the
// first, else two elements, else one.
int vector_of(int64_t cols, const void* a, int a_size, int64_t a_stride, const void* b, int b_size,
              int64_t b_stride) {
  for (const int v : {16 / a_size, 2}) {
    const size_t wa = (size_t)std::min(16, v * a_size), wb = (size_t)std::min(16, v * b_size);
    if (cols % v == 0 && aligned(a, wa) && aligned(b, wb) && (a_stride * a_size) % wa == 0 &&
        (b_stride * b_size) % wb == 0)
      return v;
  }
  return 1;
}

template <typename TT, typename TR>
cudaError_t launch_lookup(LookupArgs a, int v, cudaStream_t s) {
  const int64_t per_cta = (int64_t)(kLookupThreads / a.lanes) * kLookupRows;
  const sarr::LaunchShape shape{dim3((unsigned)((a.n + per_cta - 1) / per_cta)), kLookupThreads, 0, false, 1};
  sarr::count_launches(1);
  if (v == 16 / (int)sizeof(TT)) return sarr::launch(lookup_kernel<TT, TR, 16 / (int)sizeof(TT)>, shape, s, a);
  if (v == 2) return sarr::launch(lookup_kernel<TT, TR, 2>, shape, s, a);
  return sarr::launch(lookup_kernel<TT, TR, 1>, shape, s, a);
}

struct SortPlan {
  int bits, passes, digit_bits, tiles;
  size_t key_bytes, counts_at, totals_at, bytes;
};

SortPlan sort_plan(int64_t n, int64_t codes) {
  SortPlan P;
  P.bits = 1;
  while (((int64_t)1 << P.bits) <= codes) ++P.bits;  // keys 0 .. codes
  P.passes = (P.bits + kMaxDigitBits - 1) / kMaxDigitBits;
  P.digit_bits = (P.bits + P.passes - 1) / P.passes;
  P.tiles = (int)((n + kTile - 1) / kTile);
  P.key_bytes = P.counts_at = P.totals_at = 0;
  P.bytes = 0;  // one tile: shared memory holds it all
  if (P.tiles > 1) {
    P.key_bytes = round256((size_t)n * 4);
    const int buffers = std::min(P.passes - 1, 2);
    P.counts_at = (size_t)buffers * 2 * P.key_bytes;
    P.totals_at = P.counts_at + round256((size_t)P.tiles * (4u << P.digit_bits));
    P.bytes = P.totals_at + round256(4u << P.digit_bits);
  }
  return P;
}

// The tile kernels use more than 48 KB of shared memory; the permission is per
// device, asked for once.
constexpr size_t kTileSmem = sizeof(TileShared);
cudaError_t allow_sort_smem() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (bit & done.load(std::memory_order_acquire)) return cudaSuccess;
  e = cudaFuncSetAttribute(sort_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTileSmem);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(sort_scatter_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)(kTileSmem + 4 * kMaxBins));
  if (e != cudaSuccess) return e;
  done.fetch_or(bit, std::memory_order_release);
  return cudaSuccess;
}

cudaError_t run_sort(SortArgs a, const SortPlan& P, char* w, int32_t* order, int32_t* sorted, int32_t* offsets,
                     cudaStream_t s) {
  if (P.tiles <= 1) {
    a.key_out = reinterpret_cast<uint32_t*>(sorted);
    a.place_out = order;
    a.offsets = offsets;
    a.bits = P.bits;
    sarr::count_launches(1);
    return sarr::launch(sort_tile_kernel, {dim3(1), kSortThreads, kTileSmem, false, 1}, s, a);
  }
  a.tiles = P.tiles;
  a.counts = reinterpret_cast<int32_t*>(w + P.counts_at);
  a.totals = reinterpret_cast<int32_t*>(w + P.totals_at);
  cudaError_t e;
  for (int p = 0; p < P.passes; ++p) {
    const bool last = p == P.passes - 1;
    uint32_t* key = last ? reinterpret_cast<uint32_t*>(sorted)
                         : reinterpret_cast<uint32_t*>(w + (size_t)(2 * (p & 1)) * P.key_bytes);
    int32_t* place = last ? order : reinterpret_cast<int32_t*>(w + (size_t)(2 * (p & 1) + 1) * P.key_bytes);
    a.shift = p * P.digit_bits;
    a.bits = std::min(P.digit_bits, P.bits - a.shift);
    a.key_out = key;
    a.place_out = place;
    a.offsets = P.passes == 1 ? offsets : nullptr;
    const unsigned bins = 1u << a.bits;
    sarr::count_launches(3);
    e = sarr::launch(sort_histogram_kernel, {dim3((unsigned)P.tiles), kSortThreads, 0, p > 0, 1}, s, a);
    if (e != cudaSuccess) return e;
    e = sarr::launch(sort_prefix_kernel, {dim3((bins + kPrefixBins - 1) / kPrefixBins), kPrefixThreads, 0, true, 1}, s, a);
    if (e != cudaSuccess) return e;
    e = sarr::launch(sort_scatter_kernel, {dim3((unsigned)P.tiles), kSortThreads, kTileSmem + 4 * bins, true, 1}, s, a);
    if (e != cudaSuccess) return e;
    a.key_in = key;
    a.place_in = place;
  }
  if (P.passes == 1) return cudaSuccess;
  sarr::count_launches(1);
  return sarr::launch(sort_offsets_kernel, {dim3((unsigned)(((int64_t)a.codes + 256) / 256)), 256, 0, true, 1}, s, a.n,
                      a.codes, sorted, offsets);
}

struct GradPlan {
  int lanes, part, span;
  int64_t spans, tiles;
  size_t bytes;
};

// Widths of a group and a part from the sizes alone (the workspace's size is
// asked for without the arrays): 4 rows wide at least, and parts short enough
// to fill the GPU with CTAs.
GradPlan grad_plan(int64_t n, int64_t cols, int64_t vecs) {
  GradPlan P;
  P.lanes = pow2_at_least(vecs, kGradThreads);
  P.tiles = (vecs + P.lanes - 1) / P.lanes;
  const int groups = kGradThreads / P.lanes;
  P.part = kGradRows;
  while (P.part < kMaxPart && P.part * 2 * groups <= kMaxSpan &&
         n / ((int64_t)P.part * 2 * groups) * P.tiles >= 148 * 6)
    P.part *= 2;
  P.span = P.part * groups;
  P.spans = (n + P.span - 1) / P.span;
  P.bytes = round256((size_t)P.spans * 2 * (size_t)cols * 4) + 256;
  return P;
}

// What the two gradient entry points check alike.
int check_gradient(int64_t n, int64_t codes, int64_t cols, const void* grad_rows, int rows_type, int64_t rows_stride,
                   const void* grad_table, int table_type, int64_t table_stride) {
  if (n < 0 || n > kMaxCount || codes < 0 || codes > kMaxCount || cols < 0 || cols > kMaxCols) return SARR_ERR_ARG;
  if (!type_ok(rows_type) || !type_ok(table_type)) return SARR_ERR_ARG;
  if (rows_type != SARR_F32 && table_type != SARR_F32 && table_type != rows_type) return SARR_ERR_ARG;
  if (rows_stride < cols || table_stride < cols) return SARR_ERR_ARG;
  if (codes == 0 || cols == 0) return SARR_OK;
  if (!grad_table || (n > 0 && !grad_rows)) return SARR_ERR_ARG;
  if (!aligned(grad_rows, type_size(rows_type)) || !aligned(grad_table, type_size(table_type))) return SARR_ERR_ARG;
  return SARR_OK;
}

template <typename TG, typename TT, int kV>
cudaError_t launch_grad_v(const GradArgs& a, const GradPlan& P, cudaStream_t s) {
  if (P.spans > 0) {
    sarr::count_launches(1);
    const cudaError_t e = sarr::launch(grad_kernel<TG, TT, kV>,
                                       {dim3((unsigned)P.spans, (unsigned)P.tiles), kGradThreads, 0, true, 1}, s, a);
    if (e != cudaSuccess) return e;
  }
  const int groups = kGradThreads / P.lanes;
  sarr::count_launches(1);
  return sarr::launch(grad_finish_kernel<TT, kV>,
                      {dim3((unsigned)((a.codes + groups - 1) / groups), (unsigned)P.tiles), kGradThreads, 0, true, 1},
                      s, a);
}

template <typename TG, typename TT>
cudaError_t launch_grad(const GradArgs& a, const GradPlan& P, int v, cudaStream_t s) {
  if (v == 16 / (int)sizeof(TG)) return launch_grad_v<TG, TT, 16 / (int)sizeof(TG)>(a, P, s);
  if (v == 2) return launch_grad_v<TG, TT, 2>(a, P, s);
  return launch_grad_v<TG, TT, 1>(a, P, s);
}

}  // namespace

extern "C" int sarr_codebook_lookup(int64_t n, int64_t codes, int64_t cols, const void* index, int index_bits,
                                    const void* table, int table_type, int64_t table_stride, float scale,
                                    void* rows, int rows_type, int64_t rows_stride, sarr_stream_t stream) {
  if (n < 0 || n > kMaxCount || codes < 0 || codes > kMaxCount || cols < 0 || cols > kMaxCols) return SARR_ERR_ARG;
  if ((index_bits != 32 && index_bits != 64) || !type_ok(table_type) || !type_ok(rows_type)) return SARR_ERR_ARG;
  if (rows_type != table_type && rows_type != SARR_F32) return SARR_ERR_ARG;
  if (table_stride < cols || rows_stride < cols) return SARR_ERR_ARG;
  if (n == 0 || cols == 0) return SARR_OK;
  if (!index || !rows || (codes > 0 && !table)) return SARR_ERR_ARG;
  if (!aligned(index, index_bits / 8) || !aligned(table, type_size(table_type)) ||
      !aligned(rows, type_size(rows_type)))
    return SARR_ERR_ARG;
  const int v = vector_of(cols, table, type_size(table_type), table_stride, rows, type_size(rows_type), rows_stride);
  LookupArgs a;
  memset(&a, 0, sizeof(a));
  a.n = n;
  a.codes = (uint32_t)codes;
  a.vecs = (int)(cols / v);
  a.lanes = pow2_at_least(a.vecs, kLookupThreads);
  a.wide = index_bits == 64;
  a.scale = scale;
  a.index = index;
  a.table = table;
  a.rows = rows;
  a.table_stride = table_stride;
  a.rows_stride = rows_stride;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (table_type == SARR_F32) e = launch_lookup<float, float>(a, v, s);
  else if (table_type == SARR_BF16)
    e = rows_type == SARR_F32 ? launch_lookup<__nv_bfloat16, float>(a, v, s)
                              : launch_lookup<__nv_bfloat16, __nv_bfloat16>(a, v, s);
  else
    e = rows_type == SARR_F32 ? launch_lookup<__half, float>(a, v, s) : launch_lookup<__half, __half>(a, v, s);
  return cuda_status(e);
}

extern "C" int sarr_codebook_sort_workspace_size(int64_t n, int64_t codes, size_t* bytes) {
  if (!bytes || n < 0 || n > kMaxCount || codes < 0 || codes > kMaxCount) return SARR_ERR_ARG;
  *bytes = sort_plan(n, codes).bytes;
  return SARR_OK;
}

extern "C" int sarr_codebook_sort(int64_t n, int64_t codes, const void* index, int index_bits, int32_t* order,
                                  int32_t* sorted_codes, int32_t* offsets, void* ws, size_t ws_bytes,
                                  sarr_stream_t stream) {
  size_t need = 0;
  if (sarr_codebook_sort_workspace_size(n, codes, &need) != SARR_OK) return SARR_ERR_ARG;
  if (index_bits != 32 && index_bits != 64) return SARR_ERR_ARG;
  if (!offsets || (n > 0 && (!index || !order || !sorted_codes))) return SARR_ERR_ARG;
  if (!aligned(index, index_bits / 8) || !aligned(order, 4) || !aligned(sorted_codes, 4) || !aligned(offsets, 4))
    return SARR_ERR_ARG;
  if (ws_bytes < need || (need > 0 && (!ws || !aligned(ws, 256)))) return SARR_ERR_WORKSPACE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = allow_sort_smem();
  if (e != cudaSuccess) return cuda_status(e);
  SortArgs a;
  memset(&a, 0, sizeof(a));
  a.n = (int)n;
  a.codes = (uint32_t)codes;
  a.wide = index_bits == 64;
  a.index = index;
  return cuda_status(run_sort(a, sort_plan(n, codes), static_cast<char*>(ws), order, sorted_codes, offsets, s));
}

extern "C" int sarr_codebook_grad_workspace_size(int64_t n, int64_t cols, size_t* bytes) {
  if (!bytes || n < 0 || n > kMaxCount || cols < 0 || cols > kMaxCols) return SARR_ERR_ARG;
  // the shortest spans that any vector width of these columns gives
  size_t most = 256;
  for (const int v : {1, 2, 4, 8})
    if (cols % v == 0) most = std::max(most, grad_plan(n, cols, std::max<int64_t>(cols / v, 1)).bytes);
  *bytes = most;
  return SARR_OK;
}

extern "C" int sarr_codebook_grad(int64_t n, int64_t codes, int64_t cols, const void* grad_rows, int rows_type,
                                  int64_t rows_stride, const int32_t* order, const int32_t* sorted_codes,
                                  const int32_t* offsets, float scale, void* grad_table, int table_type,
                                  int64_t table_stride, void* ws, size_t ws_bytes, sarr_stream_t stream) {
  size_t need = 0;
  const int st = check_gradient(n, codes, cols, grad_rows, rows_type, rows_stride, grad_table, table_type, table_stride);
  if (st != SARR_OK) return st;
  if (sarr_codebook_grad_workspace_size(n, cols, &need) != SARR_OK) return SARR_ERR_ARG;
  if (codes == 0 || cols == 0) return SARR_OK;
  if (!offsets || (n > 0 && (!order || !sorted_codes))) return SARR_ERR_ARG;
  if (!aligned(order, 4) || !aligned(sorted_codes, 4) || !aligned(offsets, 4)) return SARR_ERR_ARG;
  if (!ws || ws_bytes < need || !aligned(ws, 256)) return SARR_ERR_WORKSPACE;
  const int v = vector_of(cols, grad_rows, type_size(rows_type), rows_stride, grad_table, type_size(table_type),
                          table_stride);
  const GradPlan P = grad_plan(n, cols, cols / v);
  GradArgs a;
  memset(&a, 0, sizeof(a));
  a.cols = cols;
  a.codes = (uint32_t)codes;
  a.vecs = (int)(cols / v);
  a.lanes = P.lanes;
  a.part = P.part;
  a.span = P.span;
  a.scale = scale;
  a.rows = grad_rows;
  a.rows_stride = rows_stride;
  a.order = order;
  a.sorted = sorted_codes;
  a.offsets = offsets;
  a.table = grad_table;
  a.table_stride = table_stride;
  a.partial = static_cast<float*>(ws);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (rows_type == SARR_F32)
    e = table_type == SARR_F32    ? launch_grad<float, float>(a, P, v, s)
        : table_type == SARR_BF16 ? launch_grad<float, __nv_bfloat16>(a, P, v, s)
                                  : launch_grad<float, __half>(a, P, v, s);
  else if (rows_type == SARR_BF16)
    e = table_type == SARR_F32 ? launch_grad<__nv_bfloat16, float>(a, P, v, s)
                               : launch_grad<__nv_bfloat16, __nv_bfloat16>(a, P, v, s);
  else
    e = table_type == SARR_F32 ? launch_grad<__half, float>(a, P, v, s) : launch_grad<__half, __half>(a, P, v, s);
  return cuda_status(e);
}

extern "C" int sarr_codebook_gradient_workspace_size(int64_t n, int64_t codes, int64_t cols, size_t* bytes) {
  size_t sort = 0, grad = 0;
  if (!bytes || sarr_codebook_sort_workspace_size(n, codes, &sort) != SARR_OK ||
      sarr_codebook_grad_workspace_size(n, cols, &grad) != SARR_OK)
    return SARR_ERR_ARG;
  // the order, the sorted codes and the offsets, then the two parts' own
  // workspaces, which are not needed at the same time
  *bytes = 2 * round256((size_t)n * 4) + round256((size_t)(codes + 1) * 4) + std::max(round256(sort), grad);
  return SARR_OK;
}

extern "C" int sarr_codebook_gradient(int64_t n, int64_t codes, int64_t cols, const void* grad_rows, int rows_type,
                                      int64_t rows_stride, const void* index, int index_bits, float scale,
                                      void* grad_table, int table_type, int64_t table_stride, void* ws,
                                      size_t ws_bytes, sarr_stream_t stream) {
  size_t need = 0;
  if (sarr_codebook_gradient_workspace_size(n, codes, cols, &need) != SARR_OK) return SARR_ERR_ARG;
  int st = check_gradient(n, codes, cols, grad_rows, rows_type, rows_stride, grad_table, table_type, table_stride);
  if (st != SARR_OK) return st;
  if ((index_bits != 32 && index_bits != 64) || (n > 0 && !index) || !aligned(index, index_bits / 8)) return SARR_ERR_ARG;
  if (codes == 0 || cols == 0) return SARR_OK;
  if (!ws || ws_bytes < need || !aligned(ws, 256)) return SARR_ERR_WORKSPACE;
  char* w = static_cast<char*>(ws);
  int32_t* order = reinterpret_cast<int32_t*>(w);
  int32_t* sorted = reinterpret_cast<int32_t*>(w + round256((size_t)n * 4));
  int32_t* offsets = reinterpret_cast<int32_t*>(w + 2 * round256((size_t)n * 4));
  char* rest = w + 2 * round256((size_t)n * 4) + round256((size_t)(codes + 1) * 4);
  const size_t rest_bytes = ws_bytes - (size_t)(rest - w);
  st = sarr_codebook_sort(n, codes, index, index_bits, order, sorted, offsets, rest, rest_bytes, stream);
  if (st != SARR_OK) return st;
  return sarr_codebook_grad(n, codes, cols, grad_rows, rows_type, rows_stride, order, sorted, offsets, scale, grad_table,
                            table_type, table_stride, rest, rest_bytes, stream);
}
