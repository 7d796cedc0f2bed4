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
// added by atomics): the same inputs at the same offsets from a 16-byte boundary
// give the same bits. Rows that are not aligned are read in narrower vectors, which
// cut the sums into other parts; parts that do not depend on the alignment were
// tried, and made such rows slower (16,381 of 1024 bf16, one element behind a
// boundary: 65 to 114 us against 61).
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

// kV consecutive elements as they lie in memory (floats of them only where they
// are used: half the registers of a 16-bit row in flight).
template <typename T, int kV>
struct Raw {
  static constexpr int kBytes = kV * (int)sizeof(T), kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];
};

// p is aligned to min(16, kV * sizeof(T)) bytes.
template <bool kAgain, typename T, int kV>
__device__ __forceinline__ Raw<T, kV> load_raw(const T* p) {
  constexpr int kBytes = Raw<T, kV>::kBytes;
  Raw<T, kV> x;
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int k = 0; k < kBytes / 16; ++k) {
      const uint4 q = load_word<kAgain>(reinterpret_cast<const uint4*>(p) + k);
      x.w[4 * k] = q.x, x.w[4 * k + 1] = q.y, x.w[4 * k + 2] = q.z, x.w[4 * k + 3] = q.w;
    }
  } else if constexpr (kBytes == 8) {
    const uint2 q = load_word<kAgain>(reinterpret_cast<const uint2*>(p));
    x.w[0] = q.x, x.w[1] = q.y;
  } else if constexpr (kBytes == 4) {
    x.w[0] = load_word<kAgain>(reinterpret_cast<const unsigned*>(p));
  } else {
    x.w[0] = load_word<kAgain>(reinterpret_cast<const unsigned short*>(p));
  }
  return x;
}

template <int kV>
__device__ __forceinline__ void to_floats(const Raw<float, kV>& r, float (&x)[kV]) {
#pragma unroll
  for (int k = 0; k < kV; ++k) x[k] = __uint_as_float(r.w[k]);
}
template <int kV>
__device__ __forceinline__ void to_floats(const Raw<__nv_bfloat16, kV>& r, float (&x)[kV]) {
#pragma unroll
  for (int k = 0; k < kV; ++k) x[k] = __uint_as_float(k & 1 ? r.w[k / 2] & 0xffff0000u : r.w[k / 2] << 16);
}
template <int kV>
__device__ __forceinline__ void to_floats(const Raw<__half, kV>& r, float (&x)[kV]) {
#pragma unroll
  for (int k = 0; k < kV; ++k) x[k] = __half2float(__ushort_as_half((unsigned short)(r.w[k / 2] >> (16 * (k & 1)))));
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
template <typename TI>
__device__ __forceinline__ uint32_t code_of(const TI* index, int i, uint32_t codes) {
  const TI v = __ldg(index + i);
  return v >= 0 && v < (TI)codes ? (uint32_t)v : codes;
}
__device__ __forceinline__ uint32_t code_of(const void* index, bool wide, int64_t i, uint32_t codes) {
  const int64_t v = wide ? __ldg(static_cast<const long long*>(index) + i)
                         : (int64_t)__ldg(static_cast<const int*>(index) + i);
  return v >= 0 && v < (int64_t)codes ? (uint32_t)v : codes;
}

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------
// A row is held by `lanes` threads, 16 bytes of the result each, so a warp writes
// whole lines. Bound by the writes to HBM: 1M rows of 16 floats from 4096 bf16
// rows take 13.0 us (68 MB, 5.3 TB/s, 0.80 of the measured copy bandwidth), 16,381
// rows of 1000 bf16 11.9 us (5.5 TB/s). Six rows a thread and CTAs of 64 threads:
// 12.9 us against 14.1 with 4 and 256 and 15.6 with 8 and 256 (short CTAs fill the
// tail), 27 where a lane wrote 32 bytes in two halves; 1000 rows take 2 us, a launch.
// Columns that are no whole number of vectors are read and written one or two at a
// time: 1M rows of 3 floats take 8.6 us (16 MB), the first 9 of 16 columns 42 (rows
// of 64 bytes written in part), the first 4 13.5.
constexpr int kLookupThreads = 64;
constexpr int kLookupRows = 6;  // rows per thread, their loads in flight together

struct LookupArgs {
  int64_t n;
  uint32_t codes;
  int vecs;    // vectors per row
  int lanes;   // threads per row (a power of two)
  float scale;
  const void* index;
  const void* table;
  void* rows;
  int64_t table_stride, rows_stride;  // bytes
};

template <typename TI, typename TT, typename TR, int kV>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(const LookupArgs a) {
  const int lane = threadIdx.x & (a.lanes - 1), at_once = kLookupThreads / a.lanes;
  const int64_t i0 = (int64_t)blockIdx.x * at_once * kLookupRows + threadIdx.x / a.lanes;
  const int left = (int)min(a.n - i0, (int64_t)kLookupRows * at_once);  // row k is there where k * at_once < left
  const TI* index = static_cast<const TI*>(a.index) + i0;
  uint32_t code[kLookupRows];
#pragma unroll
  for (int k = 0; k < kLookupRows; ++k) code[k] = k * at_once < left ? code_of(index, k * at_once, a.codes) : a.codes;
  const int64_t step = a.rows_stride * at_once;
  for (int v = lane; v < a.vecs; v += a.lanes) {
    const char* from = static_cast<const char*>(a.table) + v * (kV * (int)sizeof(TT));
    char* to = static_cast<char*>(a.rows) + i0 * a.rows_stride + v * (kV * (int)sizeof(TR));
    Raw<TT, kV> raw[kLookupRows];
#pragma unroll
    for (int k = 0; k < kLookupRows; ++k) {
#pragma unroll
      for (int j = 0; j < Raw<TT, kV>::kWords; ++j) raw[k].w[j] = 0;
      if (code[k] < a.codes) raw[k] = load_raw<true, TT, kV>(reinterpret_cast<const TT*>(from + code[k] * a.table_stride));
    }
#pragma unroll
    for (int k = 0; k < kLookupRows; ++k, to += step) {
      const float scale = code[k] < a.codes ? a.scale : 0.0f;  // zeros whatever the scale is
      float x[kV];
      to_floats(raw[k], x);
#pragma unroll
      for (int j = 0; j < kV; ++j) x[j] *= scale;
      if (k * at_once < left) store_vec<TR, kV>(reinterpret_cast<TR*>(to), x);
    }
  }
}

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------
// A stable sort of the keys (the codes, `codes` for none). The unit is a tile of
// 1024 to 8192 keys that one CTA sorts in registers and shared memory, as words
// key << 13 | place in the tile (the digit alone of a key over 19 bits): each warp
// holds a contiguous part of the tile, 32 words a round; a word's rank among the warp's words of its digit is a running
// count plus the lower lanes that vote for the same digit (one vote per bit, so a
// digit costs the same whatever the keys are), and a scan over the warps' counts
// and the digits gives every rank its place. Counts are 16 bits wide, two digits
// to a word.
//
// One tile: one CTA sorts by every digit and finds the offsets (sort_tile_kernel).
//
// More: passes over digits of up to 13 bits (so one pass up to 8191 codes), of
// three kernels each, which overlap (their CTAs fit on an SM together):
//   histogram  each tile's count of every digit, [tiles][bins]
//   prefix     per digit the counts of the earlier tiles, and the total
//   scatter    the tile sorted by the digit, written out behind the smaller digits
//              and the earlier tiles (in runs, since the tile is in order). The
//              first pass sorts its tile before it waits for the other two.
// With one pass the scan over the totals is the offsets.
//
// Bound by integer instructions and latency, not by its 12 bytes a key: 1M keys
// take 14.4 us for 256 codes (one pass in the tile), 22.5 for 4096 (two), 37 for
// 65,536 (two passes over all tiles); 50,000 keys of 1024 codes 9 us, 1000 keys 4 to
// 7. For 1M keys of 4096 codes: votes 30 us where a match over the lanes took 36, then
// 22 with kernels small enough to share an SM where they were not 29.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kMaxRounds = 8;                          // words per thread
constexpr int kPlaceBits = 13;                         // of a place in a tile
constexpr int kLocalBits = 9, kLocalBins = 1 << kLocalBits;  // of a pass inside a tile, at most
constexpr int kMaxDigitBits = 13, kMaxBins = 1 << kMaxDigitBits;
constexpr int kWholeBits = 32 - kPlaceBits;            // of a key that fits a word
constexpr int kOneTile = 4;                            // up to 4096 such keys in one tile (8192: 19 us against 10 in 8 tiles)
constexpr int kPrefixThreads = 256;                    // of the prefix kernel: 16 bins a CTA, or 32 where that is over a CTA per SM
constexpr int kDirectCounts = 16384;                   // counts that each scatter CTA adds itself, without the prefix kernel
constexpr int kManyTiles = 148;                        // tiles grow until there are no more of them than SMs
static_assert(kSortThreads * kMaxRounds <= 1 << kPlaceBits, "a place fits its bits");
static_assert(kSortWarps * kLocalBins * sizeof(uint16_t) >= kMaxBins * sizeof(int32_t), "a row of counts fits the warps' counts");

struct SortArgs {
  int n;
  uint32_t codes;
  bool wide;
  const void* index;
  const uint32_t* key_in;  // null: the indexes
  const int32_t* place_in;
  uint32_t* key_out;
  int32_t* place_out;
  int32_t *counts, *totals;  // [tiles][bins], [bins]; no totals: counts as the histogram left them
  int shift, bits, bins;     // of this pass's digit; with one pass bins = codes + 1, else 2^bits
  int tiles;
  bool whole;                // words hold the whole key (of up to 19 bits), else the digit
  int32_t* starts;           // null, or [bins]: where each digit's keys begin (with one pass: the offsets)
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int i) {
  return a.key_in ? a.key_in[i] : code_of(a.index, a.wide, i, a.codes);
}

// Where the pass's digit is in a word.
__device__ __forceinline__ int digit_shift(const SortArgs& a) { return kPlaceBits + (a.whole ? a.shift : 0); }

template <int kRounds>
struct TileShared {
  uint32_t word[kSortThreads * kRounds];
  uint16_t count[kSortWarps][kLocalBins];  // as many bytes as kMaxBins words
  int32_t digit[kLocalBins];
  int32_t warp_sum[kSortWarps];
};

__device__ __forceinline__ int warp_inclusive(int x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// Sum of warp_sum over the warps before this one.
__device__ __forceinline__ int warps_before(const int32_t* warp_sum, int lane, int warp) {
  return __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
}

// One stable pass over the tile's words, which the threads hold: element
// (warp * kRounds + r) * 32 + lane in word[r]. Elements behind the keys are all ones:
// last in every digit, they stay behind. On return S holds the tile in order and so
// do the threads.
template <int kRounds>
__device__ __forceinline__ void tile_pass(TileShared<kRounds>& S, uint32_t (&word)[kRounds], int shift, int bits) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = 1 << bits;
  const int first = warp * kRounds * 32 + lane;
  uint16_t* count = S.count[warp];
  for (int i = lane; i < (bins + 1) / 2; i += 32) reinterpret_cast<uint32_t*>(count)[i] = 0;
  uint32_t peers[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) peers[r] = 0xffffffffu;
  uint32_t bit = 1u << shift;
  for (int b = 0; b < bits; ++b, bit += bit) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const bool one = (word[r] & bit) != 0;
      const uint32_t ones = __ballot_sync(0xffffffffu, one);
      peers[r] &= one ? ones : ~ones;
    }
  }
  __syncwarp();
  const uint32_t lower = (1u << lane) - 1;
  int rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t digit = (word[r] >> shift) & (bins - 1), below = peers[r] & lower;
    const int before = count[digit];
    __syncwarp();
    if (below == 0) count[digit] = (uint16_t)(before + __popc(peers[r]));
    __syncwarp();
    rank[r] = before + __popc(below);
  }
  __syncthreads();
  // per digit (two to a thread): the counts of the earlier warps, and the digits before
  const int pairs = (bins + 1) / 2;
  int lo = 0, incl = 0;
  if (tid < ((pairs + 31) & ~31)) {
    uint32_t sum = 0;
    if (tid < pairs) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        uint32_t* c = reinterpret_cast<uint32_t*>(S.count[w]) + tid;
        const uint32_t x = *c;
        *c = sum;
        sum += x;
      }
    }
    lo = sum & 0xffffu;
    const int both = lo + (int)(sum >> 16);
    incl = warp_inclusive(both, lane);
    if (lane == 31) S.warp_sum[warp] = incl;
    incl -= both;
  }
  __syncthreads();
  if (tid < ((pairs + 31) & ~31)) {
    const int at = incl + warps_before(S.warp_sum, lane, warp);
    if (tid < pairs) {
      S.digit[2 * tid] = at;
      if (2 * tid + 1 < bins) S.digit[2 * tid + 1] = at + lo;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t digit = (word[r] >> shift) & (bins - 1);
    S.word[S.digit[digit] + count[digit] + rank[r]] = word[r];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) word[r] = S.word[first + 32 * r];
}

// The tile's words into the threads, then sorted by the `bits` bits of the digit.
template <int kRounds>
__device__ __forceinline__ void sort_tile(const SortArgs& a, TileShared<kRounds>& S, uint32_t (&word)[kRounds],
                                          int tile0, int len) {
  const int first = (threadIdx.x >> 5) * kRounds * 32 + (threadIdx.x & 31);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int e = first + 32 * r;
    word[r] = e < len ? sort_key(a, tile0 + e) : 0;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int e = first + 32 * r;
    word[r] = (a.whole ? word[r] : (word[r] >> a.shift) & ((1u << a.bits) - 1)) << kPlaceBits | e;
    if (e >= len) word[r] = 0xffffffffu;
  }
  const int passes = (a.bits + kLocalBits - 1) / kLocalBits, each = (a.bits + passes - 1) / passes;
#pragma unroll 1
  for (int p = 0; p < passes; ++p)
    tile_pass<kRounds>(S, word, digit_shift(a) + p * each, min(each, a.bits - p * each));
}

extern __shared__ __align__(16) unsigned char s_sort[];

template <int kRounds>
__global__ void __launch_bounds__(kSortThreads) sort_tile_kernel(const SortArgs a) {
  TileShared<kRounds>& S = *reinterpret_cast<TileShared<kRounds>*>(s_sort);
  uint32_t word[kRounds];
  sarr::dependents_may_start();
  sort_tile<kRounds>(a, S, word, 0, a.n);
  const int first = (threadIdx.x >> 5) * kRounds * 32 + (threadIdx.x & 31);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int e = first + 32 * r;
    if (e < a.n) {
      a.key_out[e] = word[r] >> kPlaceBits;
      a.place_out[e] = word[r] & ((1 << kPlaceBits) - 1);
    }
  }
  if (!a.starts) return;
  // the first place whose key is >= c
  for (int64_t c = threadIdx.x; c <= a.codes; c += kSortThreads) {
    int lo = 0, hi = a.n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (S.word[mid] >> kPlaceBits < (uint32_t)c) lo = mid + 1;
      else hi = mid;
    }
    a.starts[c] = lo;
  }
}

// Threads of the histogram: few enough for its CTA beside the other two kernels'.
template <int kRounds>
constexpr int kCountThreads = kRounds >= 8 ? 512 : 256;

template <int kRounds>
__global__ void __launch_bounds__(kCountThreads<kRounds>, 2048 / kCountThreads<kRounds>)
    sort_histogram_kernel(const SortArgs a) {
  constexpr int kTile = kSortThreads * kRounds, kThreads = kCountThreads<kRounds>, kBatch = 8;
  __shared__ int32_t s_bin[kMaxBins];
  sarr::dependents_may_start();
  sarr::wait_for_previous();
  const int bins = a.bins, mask = (1 << a.bits) - 1, tile0 = blockIdx.x * kTile, len = min(kTile, a.n - tile0);
  for (int d = threadIdx.x; d < bins; d += kThreads) s_bin[d] = 0;
  __syncthreads();
  for (int e0 = threadIdx.x; e0 < len; e0 += kBatch * kThreads) {
    uint32_t key[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (e0 + k * kThreads < len) key[k] = sort_key(a, tile0 + e0 + k * kThreads);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (e0 + k * kThreads < len) atomicAdd(s_bin + ((key[k] >> a.shift) & mask), 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kThreads) a.counts[(int64_t)blockIdx.x * bins + d] = s_bin[d];
}

// counts[t][d] becomes the sum of counts[0 .. t-1][d], totals[d] the sum of all. A
// CTA takes kBins digits; its threads split the tiles. Of 1M keys, 65,536 codes take
// 41 us with 32 digits a CTA and 37 with 16; 4096 codes 22.5 with 32 and 25.7 with
// 16, two CTAs per SM beside the scatter's.
template <int kBins>
__global__ void __launch_bounds__(kPrefixThreads, 8) sort_prefix_kernel(const SortArgs a) {
  constexpr int kSplit = kPrefixThreads / kBins;
  __shared__ int32_t s_sum[kSplit][kBins];
  sarr::dependents_may_start();
  sarr::wait_for_previous();
  const int bins = a.bins, d = blockIdx.x * kBins + (threadIdx.x & (kBins - 1));
  const int part = threadIdx.x / kBins, per = (a.tiles + kSplit - 1) / kSplit;
  const int t0 = min(part * per, a.tiles), t1 = min(t0 + per, a.tiles);
  int32_t* c = a.counts + d;
  int sum = 0;
  if (d < bins) {
#pragma unroll 8
    for (int t = t0; t < t1; ++t) sum += __ldcg(c + (int64_t)t * bins);
  }
  s_sum[part][threadIdx.x & (kBins - 1)] = sum;
  __syncthreads();
  if (d >= bins) return;
  int at = 0, all = 0;
#pragma unroll
  for (int k = 0; k < kSplit; ++k) {
    const int x = s_sum[k][threadIdx.x & (kBins - 1)];
    if (k < part) at += x;
    all += x;
  }
  if (part == 0) a.totals[d] = all;
  for (int t = t0; t < t1; t += 8) {
    int x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = t + k < t1 ? __ldcg(c + (int64_t)(t + k) * bins) : 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (t + k < t1) c[(int64_t)(t + k) * bins] = at;
      at += x[k];
    }
  }
}

template <int kRounds>
__global__ void __maxnreg__(kRounds <= 4 ? 32 : 40) sort_scatter_kernel(const SortArgs a) {
  constexpr int kTile = kSortThreads * kRounds;
  TileShared<kRounds>& S = *reinterpret_cast<TileShared<kRounds>*>(s_sort);
  int32_t* s_base = reinterpret_cast<int32_t*>(s_sort + sizeof(TileShared<kRounds>));  // [bins]
  uint32_t word[kRounds];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, begin = warp * kRounds * 32 + lane;
  const int bins = a.bins, tile0 = blockIdx.x * kTile, len = min(kTile, a.n - tile0);
  const int shift = digit_shift(a), mask = (1 << a.bits) - 1;
  sarr::dependents_may_start();
  if (a.key_in) sarr::wait_for_previous();  // the first pass's keys are the caller's
  sort_tile<kRounds>(a, S, word, tile0, len);
  if (!a.key_in) sarr::wait_for_previous();
  // where each digit begins, and in it this tile's keys
  {
    // (the warps' counts are not needed any more: the tile's row of the counts goes there)
    int32_t* s_before = reinterpret_cast<int32_t*>(S.count);
    const int32_t* before = a.counts + (int64_t)blockIdx.x * bins;
    if (a.totals) {
#pragma unroll 4
      for (int d = tid; d < bins; d += kSortThreads) {
        s_base[d] = __ldcg(a.totals + d);
        s_before[d] = __ldcg(before + d);
      }
    } else {
      for (int d = tid; d < bins; d += kSortThreads) {
        int total = 0, earlier = 0;
#pragma unroll 8
        for (int t = 0; t < a.tiles; ++t) {
          const int x = __ldcg(a.counts + (int64_t)t * bins + d);
          total += x;
          if (t < (int)blockIdx.x) earlier += x;
        }
        s_base[d] = total;
        s_before[d] = earlier;
      }
    }
    __syncthreads();
    const int each = (bins + kSortThreads - 1) / kSortThreads, first = min(tid * each, bins), end = min(first + each, bins);
    int sum = 0;
    for (int d = first; d < end; ++d) sum += s_base[d];
    const int incl = warp_inclusive(sum, lane);
    if (lane == 31) S.warp_sum[warp] = incl;
    __syncthreads();
    int at = incl - sum + warps_before(S.warp_sum, lane, warp);
    for (int d = first; d < end; ++d) {
      const int x = s_base[d];
      s_base[d] = at + s_before[d];
      if (a.starts && blockIdx.x == 0) a.starts[d] = at;
      at += x;
    }
  }
  __syncthreads();
  // less the place in the tile where the digit begins
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int e = begin + 32 * r;
    if (e < len) {
      const uint32_t d = (word[r] >> shift) & mask;
      if (e == 0 || ((S.word[e - 1] >> shift) & mask) != d) s_base[d] -= e;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int e = begin + 32 * r;
    if (e < len) {
      const int from = tile0 + (int)(word[r] & ((1 << kPlaceBits) - 1)), to = s_base[(word[r] >> shift) & mask] + e;
      a.key_out[to] = a.whole ? word[r] >> kPlaceBits : sort_key(a, from);
      a.place_out[to] = a.key_in ? a.place_in[from] : from;
    }
  }
}

// The first place whose code is >= c, for each c: a search among the keys of its
// last digit (starts: where each digit's keys begin), or among all.
__global__ void __launch_bounds__(256) sort_offsets_kernel(int n, uint32_t codes, const int32_t* sorted,
                                                           const int32_t* starts, int shift, int bins,
                                                           int32_t* offsets) {
  sarr::dependents_may_start();
  sarr::wait_for_previous();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c > codes) return;
  int lo = 0, hi = n;
  if (starts) {
    const int digit = (int)(c >> shift);
    lo = starts[digit];
    if (digit + 1 < bins) hi = starts[digit + 1];
  }
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
// codes that cross a span's border through the workspace, by grad_finish_kernel.
// CTAs behind the spans' write the zeros of the codes without Gaussians, while the
// others wait for their rows (evenly among them they hold the spans up: 39 us
// against 31 for 16,381 rows of 1024 bf16 into 32,000).
//
// Rows of 1024 bf16 are bound by their reads: 31 us for 165 MB (5.3 TB/s, 0.81 of
// the measured copy bandwidth). Rows of 16 floats are bound by latency: 1M of them
// take 20.6 us for 72 MB from HBM, 24 where one code has 6 % of them and 26 where one
// has all (14, 16 and 19 with the rows in L2). With one code the rows are read one
// after another, so it is not their random places: there is one wave of CTAs, each
// of which waits for its codes and its order, then loads eight rows when the eight
// before are added; a code over all spans has its 489 partials added by one CTA.
constexpr int kGradThreads = 256;
constexpr int kGradRows = 8;     // rows of a group loaded together
constexpr int kMaxPart = 64;     // places of a group, at most; a multiple of kGradRows
// Places of a group up to which one CTA takes them all, without a kernel behind it:
// 1000 rows of 16 4.5 us against 5.5 in several, 2048 of 8 5.4 against 6.2, 256 of 64
// 3.8 against 4.1. With up to 32 places 2048 rows of 16 take 6.4 us in one CTA against
// 5.9 in several, 4096 of 8 7.7 against 6.4, 512 of 64 5.6 against 5.0.
constexpr int kOneSpanPart = 16;
constexpr int kMaxSpan = 2048;   // places of a CTA, at most
constexpr int kFinishThreads = 64;
constexpr int kFillCodes = 8;    // codes of a group in a zero-writing CTA
constexpr int kLongSpans = 16;   // spans from which a code's partials are added by a whole CTA

struct GradArgs {
  int n;
  int64_t cols;
  uint32_t codes;
  int vecs, lanes, part;  // vectors per row; threads per row; places per group
  int span, spans;        // places per CTA: part * (kGradThreads / lanes); CTAs with places
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

// Partials are at [span][slot][v][j]: kV floats side by side.
template <int kV>
__device__ __forceinline__ float* partial_at(const GradArgs& a, int span, int slot, int v) {
  return a.partial + ((int64_t)span * 2 + slot) * a.cols + (int64_t)v * kV;
}

template <typename TG, typename TT, int kV>
__global__ void __launch_bounds__(kGradThreads, kV >= 8 ? 3 : 4) grad_kernel(const GradArgs a) {
  // codes and rows of the parts, each part kPad words behind the one before, so
  // that groups at the same place of their parts use different banks
  constexpr int kPad = 4, kWords = kMaxSpan + kMaxSpan / kGradRows * kPad;
  __shared__ __align__(16) int32_t s_code[kWords], s_row[kWords];
  __shared__ float s_head[kV][kGradThreads], s_tail[kV][kGradThreads];
  __shared__ uint8_t s_state[kGradThreads];  // per group
  __shared__ int32_t s_edge[2];              // codes before and behind the span
  enum : uint8_t { kHead = 1, kTail = 2, kThrough = 4 };
  sarr::dependents_may_start();
  sarr::wait_for_previous();

  const int tid = threadIdx.x, lane = tid & (a.lanes - 1), group = tid / a.lanes;
  const int groups = kGradThreads / a.lanes;
  const int v = blockIdx.y * a.lanes + lane;
  const bool active = v < a.vecs;
  const int span = blockIdx.x;
  if (span >= a.spans) {  // zeros of the codes without Gaussians
    const int64_t c0 = ((int64_t)span - a.spans) * groups * kFillCodes + group;
    bool none[kFillCodes];
#pragma unroll
    for (int k = 0; k < kFillCodes; ++k) {
      const int64_t c = c0 + (int64_t)k * groups;
      none[k] = c < a.codes && a.offsets[c] == a.offsets[c + 1];
    }
    if constexpr (kV * sizeof(TT) >= 16) {  // 16 bytes a lane side by side
      constexpr int kPer = 16 / (int)sizeof(TT), kSteps = kV / kPer;
      const int64_t col0 = (int64_t)blockIdx.y * a.lanes * kV + lane * kPer;
#pragma unroll
      for (int k = 0; k < kFillCodes; ++k) {
        TT* row = static_cast<TT*>(a.table) + (c0 + (int64_t)k * groups) * a.table_stride;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const int64_t col = col0 + j * a.lanes * kPer;
          if (none[k] && col < a.cols) *reinterpret_cast<uint4*>(row + col) = make_uint4(0, 0, 0, 0);
        }
      }
    } else {
      const float zero[kV] = {};
#pragma unroll
      for (int k = 0; k < kFillCodes; ++k)
        if (none[k] && active)
          store_vec<TT, kV>(static_cast<TT*>(a.table) + (c0 + (int64_t)k * groups) * a.table_stride + (int64_t)v * kV, zero);
    }
    return;
  }
  const int none = (int)a.codes;  // places from the first of this code on are without
  const int64_t p0 = (int64_t)span * a.span;
  const int pitch = a.part + kPad;
#pragma unroll 2
  for (int i = 4 * lane; i < a.part; i += 4 * a.lanes) {
    const int64_t p = p0 + group * a.part + i;
    int c[4], r[4];
    if (p + 4 <= a.n) {
      const int4 c4 = *reinterpret_cast<const int4*>(a.sorted + p), r4 = *reinterpret_cast<const int4*>(a.order + p);
      c[0] = c4.x, c[1] = c4.y, c[2] = c4.z, c[3] = c4.w;
      r[0] = r4.x, r[1] = r4.y, r[2] = r4.z, r[3] = r4.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        c[k] = p + k < a.n ? a.sorted[p + k] : none;
        r[k] = p + k < a.n ? a.order[p + k] : 0;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // whatever the caller's arrays hold, inside the table and the rows
      c[k] = min((uint32_t)c[k], a.codes);
      r[k] = min((uint32_t)r[k], (uint32_t)a.n - 1);
    }
    *reinterpret_cast<int4*>(s_code + group * pitch + i) = make_int4(c[0], c[1], c[2], c[3]);
    *reinterpret_cast<int4*>(s_row + group * pitch + i) = make_int4(r[0], r[1], r[2], r[3]);
  }
  if (tid < 2) {
    const int64_t p = tid == 0 ? p0 - 1 : p0 + a.span;
    s_edge[tid] = p >= 0 && p < a.n ? a.sorted[p] : none;
  }
  if (lane == 0) s_state[group] = 0;
  __syncthreads();

  const TG* rows = static_cast<const TG*>(a.rows) + (int64_t)v * kV;
  const int32_t* my_code = s_code + group * pitch;
  const int32_t* my_row = s_row + group * pitch;
  float acc[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
  int cur = my_code[0];
  const bool work = cur != none;
  if (work) {
    bool open = (group > 0 ? my_code[a.part - 1 - pitch] : s_edge[0]) == cur;  // the code began before this part
    uint8_t state = 0;
    for (int q = 0; q < a.part && cur != none; q += kGradRows) {
      Raw<TG, kV> x[kGradRows];  // of places without a code too: their rows are there, and not added
#pragma unroll
      for (int k = 0; k < kGradRows; k += 4) {
        const int4 r = *reinterpret_cast<const int4*>(my_row + q + k);
        if (active) {
          x[k] = load_raw<false, TG, kV>(rows + r.x * a.rows_stride);
          x[k + 1] = load_raw<false, TG, kV>(rows + r.y * a.rows_stride);
          x[k + 2] = load_raw<false, TG, kV>(rows + r.z * a.rows_stride);
          x[k + 3] = load_raw<false, TG, kV>(rows + r.w * a.rows_stride);
        }
      }
      if (my_code[q + kGradRows - 1] == cur) {  // in order: all of one code
#pragma unroll
        for (int k = 0; k < kGradRows; ++k) {
          float f[kV];
          to_floats(x[k], f);
#pragma unroll
          for (int j = 0; j < kV; ++j) acc[j] += f[j];
        }
        continue;
      }
#pragma unroll
      for (int k = 0; k < kGradRows; ++k) {
        const int c = my_code[q + k];
        if (c != cur) {
          if (open) {
            state |= kHead;
#pragma unroll
            for (int j = 0; j < kV; ++j) s_head[j][tid] = acc[j];
          } else if (active && cur != none) {
            write_row<TT, kV>(a, (uint32_t)cur, v, acc);
          }
          open = false;
          cur = c;
#pragma unroll
          for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
        }
        if (cur != none) {
          float f[kV];
          to_floats(x[k], f);
#pragma unroll
          for (int j = 0; j < kV; ++j) acc[j] += f[j];
        }
      }
    }
    if (cur != none) {
      if ((group + 1 < groups ? my_code[pitch] : s_edge[1]) == cur) {  // goes on behind this part
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
    }
    if (lane == 0) s_state[group] = state;
  }
  __syncthreads();
  if (!work || !active) return;
  const uint8_t state = s_state[group];
  if (group == 0 && (state & kHead)) {  // the code open at the span's start ends in its first part
    float x[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) x[j] = s_head[j][tid];
    store_vec<float, kV>(partial_at<kV>(a, span, 0, v), x);
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
    if (closed && !(state & kThrough)) {
      write_row<TT, kV>(a, (uint32_t)cur, v, acc);
    } else {
      store_vec<float, kV>(partial_at<kV>(a, span, closed ? 0 : 1, v), acc);
    }
  }
}

// Adds the partials of the spans from, from + step, ... of a code whose last span
// is `last` (where it is the one open at the start).
template <int kAtOnce, int kV>
__device__ __forceinline__ void add_partials(const GradArgs& a, int from, int step, int last, int v,
                                             float (&acc)[kV]) {
  for (int s0 = from; s0 <= last; s0 += kAtOnce * step) {
    Raw<float, kV> x[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int s = s0 + k * step;
      x[k] = load_raw<false, float, kV>(partial_at<kV>(a, min(s, last), s < last ? 1 : 0, v));
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (s0 + k * step <= last) {
#pragma unroll
        for (int j = 0; j < kV; ++j) acc[j] += __uint_as_float(x[k].w[j]);
      }
  }
}

__device__ __forceinline__ int last_span(const GradArgs& a, int code) {
  return min((a.offsets[code + 1] - 1) / a.span, a.spans - 1);
}

// Codes over several spans: the sum of their partials, in the order of the
// spans. Each is found at the border behind the span where it begins; a group
// takes one, and codes over many spans are taken by the whole CTA, group g the
// spans g, g + groups, ..., then a tree over the groups.
template <typename TT, int kV>
__global__ void __launch_bounds__(kFinishThreads) grad_finish_kernel(const GradArgs a) {
  __shared__ int s_long[kFinishThreads];
  __shared__ int s_n_long;
  __shared__ float s_sum[kV][kFinishThreads];
  sarr::wait_for_previous();
  const int lanes = min(a.lanes, kFinishThreads);
  const int tid = threadIdx.x, lane = tid & (lanes - 1), group = tid / lanes;
  const int groups = kFinishThreads / lanes;
  const int v = blockIdx.y * lanes + lane;
  const bool active = v < a.vecs;
  if (tid == 0) s_n_long = 0;
  int first = blockIdx.x * groups + group, last = first, code = (int)a.codes;
  if (first < a.spans - 1) {
    const int64_t border = (int64_t)(first + 1) * a.span;
    code = a.sorted[border - 1];
    if ((uint32_t)code < a.codes && a.sorted[border] == code && a.offsets[code] / a.span == first)
      last = last_span(a, code);
  }
  const bool is_long = last - first >= kLongSpans;
  if (__syncthreads_or(is_long)) {
    if (is_long && lane == 0) s_long[atomicAdd(&s_n_long, 1)] = code;
    __syncthreads();
  }
  float acc[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
  if (last > first && !is_long && active) {
    add_partials<4, kV>(a, first, 1, last, v, acc);
    write_row<TT, kV>(a, (uint32_t)code, v, acc);
  }
  const int n_long = s_n_long;
  for (int k = 0; k < n_long; ++k) {  // the order of these codes does not matter
    code = s_long[k];
    first = a.offsets[code] / a.span;
    last = last_span(a, code);
#pragma unroll
    for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
    if (active) add_partials<8, kV>(a, first + group, groups, last, v, acc);
#pragma unroll
    for (int j = 0; j < kV; ++j) s_sum[j][tid] = acc[j];
    for (int half = groups / 2; half > 0; half /= 2) {
      __syncthreads();
      if (group < half) {
#pragma unroll
        for (int j = 0; j < kV; ++j) s_sum[j][tid] += s_sum[j][tid + half * lanes];
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

constexpr int64_t kMaxCols = 1 << 21;
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

template <typename TI, typename TT, typename TR>
cudaError_t launch_lookup(const LookupArgs& a, int v, cudaStream_t s) {
  const int64_t per_cta = (int64_t)(kLookupThreads / a.lanes) * kLookupRows;
  const sarr::LaunchShape shape{dim3((unsigned)((a.n + per_cta - 1) / per_cta)), kLookupThreads, 0, false};
  sarr::count_launches(1);
  if (v == 16 / (int)sizeof(TR)) return sarr::launch(lookup_kernel<TI, TT, TR, 16 / (int)sizeof(TR)>, shape, s, a);
  if (v == 2) return sarr::launch(lookup_kernel<TI, TT, TR, 2>, shape, s, a);
  return sarr::launch(lookup_kernel<TI, TT, TR, 1>, shape, s, a);
}

template <typename TT, typename TR>
cudaError_t launch_lookup(const LookupArgs& a, bool wide, int v, cudaStream_t s) {
  return wide ? launch_lookup<long long, TT, TR>(a, v, s) : launch_lookup<int, TT, TR>(a, v, s);
}

struct SortPlan {
  int bits, passes, digit_bits, rounds, tiles;
  bool one;  // one tile sorts it
  size_t key_bytes, counts_at, totals_at, starts_at, bytes;
};

SortPlan sort_plan(int64_t n, int64_t codes) {
  SortPlan P;
  P.bits = 1;
  while (((int64_t)1 << P.bits) <= codes) ++P.bits;  // keys 0 .. codes
  P.passes = (P.bits + kMaxDigitBits - 1) / kMaxDigitBits;
  P.digit_bits = (P.bits + P.passes - 1) / P.passes;
  const int64_t thousands = (n + kSortThreads - 1) / kSortThreads;
  const bool one = thousands <= kOneTile && P.bits <= kWholeBits;
  const int64_t least = one ? thousands : (thousands + kManyTiles - 1) / kManyTiles;
  P.rounds = 1;
  while (P.rounds < least && P.rounds < kMaxRounds) P.rounds *= 2;
  P.tiles = (int)((thousands + P.rounds - 1) / P.rounds);
  P.key_bytes = P.counts_at = P.totals_at = P.starts_at = 0;
  P.bytes = 0;  // one tile: shared memory holds it all
  P.one = one || n == 0;
  if (!P.one) {
    P.key_bytes = round256((size_t)n * 4);
    const int buffers = std::min(P.passes - 1, 2);
    P.counts_at = (size_t)buffers * 2 * P.key_bytes;
    P.totals_at = P.counts_at + round256((size_t)P.tiles * (4u << P.digit_bits));
    P.starts_at = P.totals_at + round256(4u << P.digit_bits);
    P.bytes = P.starts_at + round256(4u << P.digit_bits);
  }
  return P;
}

// The tile kernels use more than 48 KB of shared memory; the permission is per
// device, asked for once.
template <int kRounds>
cudaError_t allow_tile_smem() {
  if constexpr (kRounds <= kOneTile) {
    const cudaError_t e = cudaFuncSetAttribute(sort_tile_kernel<kRounds>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)sizeof(TileShared<kRounds>));
    if (e != cudaSuccess) return e;
  }
  return cudaFuncSetAttribute(sort_scatter_kernel<kRounds>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)(sizeof(TileShared<kRounds>) + 4 * kMaxBins));
}

cudaError_t allow_sort_smem() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (bit & done.load(std::memory_order_acquire)) return cudaSuccess;
  if ((e = allow_tile_smem<1>()) != cudaSuccess || (e = allow_tile_smem<2>()) != cudaSuccess ||
      (e = allow_tile_smem<4>()) != cudaSuccess || (e = allow_tile_smem<8>()) != cudaSuccess)
    return e;
  done.fetch_or(bit, std::memory_order_release);
  return cudaSuccess;
}

cudaError_t launch_offsets(const SortArgs& a, const int32_t* sorted, int32_t* offsets, cudaStream_t s) {
  sarr::count_launches(1);
  return sarr::launch(sort_offsets_kernel, {dim3((unsigned)(((int64_t)a.codes + 256) / 256)), 256, 0, true}, s, a.n,
                      a.codes, sorted, a.starts, a.shift, a.bins, offsets);
}

template <int kRounds>
cudaError_t run_sort(SortArgs a, const SortPlan& P, char* w, int32_t* order, int32_t* sorted, int32_t* offsets,
                     cudaStream_t s) {
  constexpr size_t kSmem = sizeof(TileShared<kRounds>);
  a.whole = P.bits <= kWholeBits;
  if constexpr (kRounds <= kOneTile) {
    if (P.one) {
      a.key_out = reinterpret_cast<uint32_t*>(sorted);
      a.place_out = order;
      a.starts = P.passes == 1 ? offsets : nullptr;  // more codes than one CTA finds quickly: below
      a.bits = P.bits;
      sarr::count_launches(1);
      const cudaError_t e = sarr::launch(sort_tile_kernel<kRounds>, {dim3(1), kSortThreads, kSmem, false}, s, a);
      return e != cudaSuccess || P.passes == 1 ? e : launch_offsets(a, sorted, offsets, s);
    }
  }
  a.tiles = P.tiles;
  a.counts = reinterpret_cast<int32_t*>(w + P.counts_at);
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
    a.starts = !last ? nullptr : P.passes == 1 ? offsets : reinterpret_cast<int32_t*>(w + P.starts_at);
    a.bins = P.passes == 1 ? (int)a.codes + 1 : 1 << a.bits;
    const unsigned bins = (unsigned)a.bins, tiles = (unsigned)P.tiles;
    sarr::count_launches(2);
    e = sarr::launch(sort_histogram_kernel<kRounds>, {dim3(tiles), (unsigned)kCountThreads<kRounds>, 0, p > 0}, s, a);
    if (e != cudaSuccess) return e;
    a.totals = nullptr;
    if ((int64_t)tiles * bins > kDirectCounts) {
      a.totals = reinterpret_cast<int32_t*>(w + P.totals_at);
      sarr::count_launches(1);
      e = bins <= 148 * 16 ? sarr::launch(sort_prefix_kernel<16>, {dim3((bins + 15) / 16), kPrefixThreads, 0, true}, s, a)
                           : sarr::launch(sort_prefix_kernel<32>, {dim3((bins + 31) / 32), kPrefixThreads, 0, true}, s, a);
      if (e != cudaSuccess) return e;
    }
    e = sarr::launch(sort_scatter_kernel<kRounds>, {dim3(tiles), kSortThreads, kSmem + 4 * bins, true}, s, a);
    if (e != cudaSuccess) return e;
    a.key_in = key;
    a.place_in = place;
  }
  return P.passes == 1 ? cudaSuccess : launch_offsets(a, sorted, offsets, s);
}

struct GradPlan {
  int lanes, part, span;
  int64_t spans, tiles;
  size_t bytes;
};

// Widths of a group and a part from the sizes alone (the workspace's size is
// asked for without the arrays): parts as short as the CTAs that the GPU holds
// at once can share, so that all spans run side by side, up to kMaxPart.
constexpr int grad_ctas(int v) { return 148 * (v >= 8 ? 3 : 4); }  // of grad_kernel's launch bounds

GradPlan grad_plan(int64_t n, int64_t cols, int v) {
  GradPlan P;
  const int64_t vecs = std::max<int64_t>(cols / v, 1);
  P.lanes = pow2_at_least(vecs, kGradThreads);
  P.tiles = (vecs + P.lanes - 1) / P.lanes;
  const int64_t groups = kGradThreads / P.lanes, spans = std::max<int64_t>(grad_ctas(v) / P.tiles, 1);
  const bool one = n <= groups * kOneSpanPart;
  const int64_t share = (n + groups * (one ? 1 : spans) - 1) / (groups * (one ? 1 : spans)), most = std::min<int64_t>(kMaxPart, kMaxSpan / groups);
  P.part = (int)std::max<int64_t>(std::min((share + kGradRows - 1) / kGradRows * kGradRows, most), kGradRows);
  P.span = P.part * (int)groups;
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
  const int groups = kGradThreads / P.lanes;
  const int64_t fills = ((int64_t)a.codes + groups * kFillCodes - 1) / (groups * kFillCodes);
  sarr::count_launches(1);
  const cudaError_t e = sarr::launch(
      grad_kernel<TG, TT, kV>, {dim3((unsigned)(P.spans + fills), (unsigned)P.tiles), kGradThreads, 0, true}, s, a);
  if (e != cudaSuccess || P.spans <= 1) return e;  // one span: nothing crosses its border
  const int lanes = std::min(P.lanes, kFinishThreads), at_once = kFinishThreads / lanes;
  const int64_t borders = P.spans - 1;
  sarr::count_launches(1);
  return sarr::launch(grad_finish_kernel<TT, kV>,
                      {dim3((unsigned)((borders + at_once - 1) / at_once), (unsigned)((a.vecs + lanes - 1) / lanes)),
                       kFinishThreads, 0, true},
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
  const int v = vector_of(cols, rows, type_size(rows_type), rows_stride, table, type_size(table_type), table_stride);
  LookupArgs a;
  memset(&a, 0, sizeof(a));
  a.n = n;
  a.codes = (uint32_t)codes;
  a.vecs = (int)(cols / v);
  a.lanes = pow2_at_least(a.vecs, kLookupThreads);
  a.scale = scale;
  a.index = index;
  a.table = table;
  a.rows = rows;
  a.table_stride = table_stride * type_size(table_type);
  a.rows_stride = rows_stride * type_size(rows_type);
  const bool wide = index_bits == 64;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (table_type == SARR_F32) e = launch_lookup<float, float>(a, wide, v, s);
  else if (table_type == SARR_BF16)
    e = rows_type == SARR_F32 ? launch_lookup<__nv_bfloat16, float>(a, wide, v, s)
                              : launch_lookup<__nv_bfloat16, __nv_bfloat16>(a, wide, v, s);
  else
    e = rows_type == SARR_F32 ? launch_lookup<__half, float>(a, wide, v, s)
                              : launch_lookup<__half, __half>(a, wide, v, s);
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
  const SortPlan P = sort_plan(n, codes);
  const auto run = P.rounds == 1 ? run_sort<1> : P.rounds == 2 ? run_sort<2> : P.rounds == 4 ? run_sort<4> : run_sort<8>;
  return cuda_status(run(a, P, static_cast<char*>(ws), order, sorted_codes, offsets, s));
}

extern "C" int sarr_codebook_grad_workspace_size(int64_t n, int64_t cols, size_t* bytes) {
  if (!bytes || n < 0 || n > kMaxCount || cols < 0 || cols > kMaxCols) return SARR_ERR_ARG;
  // the shortest spans that any vector width of these columns gives
  size_t most = 256;
  for (const int v : {1, 2, 4, 8})
    if (cols % v == 0) most = std::max(most, grad_plan(n, cols, v).bytes);
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
  if (!aligned(order, 16) || !aligned(sorted_codes, 16) || !aligned(offsets, 4)) return SARR_ERR_ARG;
  if (!ws || ws_bytes < need || !aligned(ws, 256)) return SARR_ERR_WORKSPACE;
  const int v = vector_of(cols, grad_rows, type_size(rows_type), rows_stride, grad_table, type_size(table_type),
                          table_stride);
  const GradPlan P = grad_plan(n, cols, v);
  GradArgs a;
  memset(&a, 0, sizeof(a));
  a.n = (int)n;
  a.cols = cols;
  a.codes = (uint32_t)codes;
  a.vecs = (int)(cols / v);
  a.lanes = P.lanes;
  a.spans = (int)P.spans;
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
