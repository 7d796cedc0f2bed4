// Global gradient norm over many tensors, clipping by it, and the Adam update
// with clipped gradients.
//
//   N = sqrt(sum_t sum_j g_t[j]^2)      (or N = max |g_t[j]|)
//   c = min(1, max_norm / (N + 1e-6))   (torch.nn.utils.clip_grad_norm_)
//   clip:  out_t[j] = c g_t[j]
//   Adam:  torch.optim.Adam's update with c g in the place of g
//
// The gradients of all tensors are cut into pieces of a few KB, whatever tensors
// they belong to, and dealt to the CTAs round robin (neighbouring CTAs read
// neighbouring pieces; with a contiguous run per CTA 40M parameters took 3 % longer,
// 1M a quarter), so a list of many small tensors costs little more than one buffer.
//
//   norm_kernel    one partial sum (or maximum) per CTA, in 64 bits: a square
//                  neither overflows nor underflows, and the sum keeps the
//                  accuracy of its terms; written to the workspace in CTA order.
//                  At the copy rate: 468 MB in 74 us (6.3 TB/s); the largest
//                  magnitude in 100 (two 64-bit compares an element);
//   finish_kernel  adds the partials and writes N (norm only);
//   clip_kernel,   every CTA adds the partials itself, in the same fixed order
//   adam_kernel    (so that all get the same c without another launch), then
//                  makes its elements, from the last piece down, newest in L2
//                  first. Bound by HBM: clip_kernel 936 MB in 172 us (5.4 TB/s; with
//                  two loads a thread norm and clip of 160 odd tensors take 243 us
//                  into others and 248 in place, with one 239 and 251),
//                  900 MB of one tensor in 151 us (6.0 TB/s), adam_kernel
//                  1.12 GB in 168 us (6.7 TB/s; a grid of 96 CTAs per SM, 184 us
//                  with 6).
//
// No atomics: the same inputs at the same offsets from a 16-byte boundary give the
// same bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "sarr.h"
#include "sarr_launch.cuh"

namespace sarr {
void count_launches(int k);  // the library's launch counter (sarr_abi.cu)
}

namespace {

// A piece is what a CTA takes at a time: 16-byte loads, kNormVecs and so on, of each
// of its threads.
constexpr int kNormThreads = 256, kNormVecs = 4, kNormCtas = 148 * 8;  // kNormCtas: the most partials of a launch
constexpr int kThreads = 256;                                          // of the clip and Adam kernels
constexpr int kClipVecs = 2, kClipCtas = 148 * 8;
constexpr int kAdamVecs = 1, kAdamCtas = 148 * 96;
// Tensors of one launch: the list travels as kernel parameters, so there is a short
// one for a scene's few tensors (0.7 KB instead of 20).
constexpr int kSmallList = 16, kMediumList = 96, kLargeList = 512;
constexpr int kAdamRanges = 64;

// One tensor of a list. Elements are numbered from the 16-byte boundary at or
// below its first one ("lead" elements before it, which are never touched), so
// that a piece's vectors are aligned in every tensor.
struct Entry {
  const void* in;
  void* out;          // clip: destination
  int64_t count;
  int64_t piece_end;  // pieces of this launch up to and including this tensor's
  uint8_t type, out_type, lead;
  bool vec;           // out's vectors are aligned where in's are
};

template <int kMax>
struct TensorList {
  int n;
  int64_t pieces;
  Entry e[kMax];
};

__device__ __forceinline__ float load_as_float(const void* p, int type, int64_t i) {
  if (type == SARR_F32) return static_cast<const float*>(p)[i];
  if (type == SARR_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_float(void* p, int type, int64_t i, float x) {
  if (type == SARR_F32) static_cast<float*>(p)[i] = x;
  else if (type == SARR_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

// 16 bytes as 4 or 8 floats.
__device__ __forceinline__ void unpack(const uint4& q, int type, float* x) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if (type == SARR_F32) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(w[k]);
  } else if (type == SARR_BF16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = __uint_as_float(w[k] << 16);
      x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      __half2 h;
      memcpy(&h, &w[k], 4);
      const float2 f = __half22float2(h);
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
  }
}

// ---------------------------------------------------------------------------
// norm
// ---------------------------------------------------------------------------
// Maximum that keeps a NaN (fmax drops it).
__device__ __forceinline__ double max_nan(double a, double b) { return (b > a || isnan(b)) ? b : a; }

template <bool kInf>
__device__ __forceinline__ double norm_add(double acc, float x) {
  if (kInf) return max_nan(acc, (double)fabsf(x));
  return fma((double)x, (double)x, acc);
}

template <bool kInf>
__device__ __forceinline__ double norm_join(double a, double b) {
  return kInf ? max_nan(a, b) : a + b;
}

// Over the CTA, in a fixed order; every thread gets the result.
template <int kCta, bool kInf>
__device__ __forceinline__ double block_join(double x) {
  __shared__ double s[kCta / 32];
  __shared__ double s_all;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = norm_join<kInf>(x, __shfl_xor_sync(0xffffffffu, x, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = s[0];
#pragma unroll
    for (int k = 1; k < kCta / 32; ++k) t = norm_join<kInf>(t, s[k]);
    s_all = t;
  }
  __syncthreads();
  return s_all;
}

template <int kMax>
__device__ __forceinline__ int64_t first_piece(const TensorList<kMax>& L, int t) {
  return t > 0 ? L.e[t - 1].piece_end : 0;
}

// Pieces inside a tensor are read 16 bytes at a time, its first and last one (which
// begin or end between 16-byte boundaries) element by element.
template <int kType, bool kInf>
__device__ __forceinline__ double piece_norm(const Entry& E, int64_t piece, double acc) {
  constexpr int kPer = kType == SARR_F32 ? 4 : 8, kElems = kNormThreads * kNormVecs * kPer;  // of 16 bytes, of a piece
  const int64_t at = piece * kElems - E.lead;
  if (at >= 0 && at + kElems <= E.count) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(E.in) + at * (16 / kPer));
    uint4 q[kNormVecs];
#pragma unroll
    for (int k = 0; k < kNormVecs; ++k) q[k] = p[k * kNormThreads + threadIdx.x];
#pragma unroll
    for (int k = 0; k < kNormVecs; ++k) {
      float x[8];
      unpack(q[k], kType, x);
#pragma unroll
      for (int j = 0; j < kPer; ++j) acc = norm_add<kInf>(acc, x[j]);
    }
  } else {
    const int64_t end = min(at + kElems, E.count);
#pragma unroll 4
    for (int64_t i = max(at, (int64_t)0) + threadIdx.x; i < end; i += kNormThreads)
      acc = norm_add<kInf>(acc, load_as_float(E.in, kType, i));
  }
  return acc;
}

template <int kMax, bool kInf>
__global__ void __launch_bounds__(kNormThreads, 8) norm_kernel(const __grid_constant__ TensorList<kMax> L,
                                                        double* __restrict__ partial) {
  sarr::dependents_may_start();
  sarr::wait_for_previous();
  double acc = 0.0;
  int t = 0;
  int64_t first = 0, stop = L.e[0].piece_end;
  for (int64_t p = blockIdx.x; p < L.pieces; p += gridDim.x) {
    while (p >= stop) first = stop, stop = L.e[++t].piece_end;
    const Entry& E = L.e[t];
    if (E.type == SARR_F32) acc = piece_norm<SARR_F32, kInf>(E, p - first, acc);
    else if (E.type == SARR_BF16) acc = piece_norm<SARR_BF16, kInf>(E, p - first, acc);
    else acc = piece_norm<SARR_F16, kInf>(E, p - first, acc);
  }
  acc = block_join<kNormThreads, kInf>(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// The norm of `n` partials (every thread gets it).
template <bool kInf>
__device__ __forceinline__ double total_norm(const double* __restrict__ partial, int n) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) acc = norm_join<kInf>(acc, partial[i]);
  acc = block_join<kThreads, kInf>(acc);
  return kInf ? acc : sqrt(acc);
}

template <bool kInf>
__global__ void __launch_bounds__(kThreads) finish_kernel(const double* __restrict__ partial, int n,
                                                          float* __restrict__ norm_out) {
  sarr::wait_for_previous();
  const double norm = total_norm<kInf>(partial, n);
  if (threadIdx.x == 0) *norm_out = (float)norm;
}

// c = min(1, max_norm / (N + 1e-6)), NaN kept, rounded once to 32 bits.
__device__ __forceinline__ float clip_coef(double norm, double max_norm) {
  const double c = max_norm / (norm + 1e-6);
  return c > 1.0 ? 1.0f : (float)c;
}

// ---------------------------------------------------------------------------
// clip
// ---------------------------------------------------------------------------
template <int kOut>
__device__ __forceinline__ void store_scaled(char* o, const float* x, int n, float c) {
  uint32_t w[8];
  if (kOut == SARR_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) w[k] = __float_as_uint(x[k] * c);
  } else if (kOut == SARR_BF16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * k] * c, x[2 * k + 1] * c);
      memcpy(&w[k], &h, 4);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __half2 h = __floats2half2_rn(x[2 * k] * c, x[2 * k + 1] * c);
      memcpy(&w[k], &h, 4);
    }
  }
  reinterpret_cast<uint4*>(o)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  if (kOut == SARR_F32 && n == 8) reinterpret_cast<uint4*>(o)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

template <int kIn, int kOut>
__device__ __forceinline__ void piece_clip(const Entry& E, int64_t piece, float c) {
  constexpr int kPer = kIn == SARR_F32 ? 4 : 8, kOutSize = kOut == SARR_F32 ? 4 : 2;
  constexpr int kElems = kThreads * kClipVecs * kPer;
  const int64_t at = piece * kElems - E.lead;
  if (E.vec && at >= 0 && at + kElems <= E.count) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(E.in) + at * (16 / kPer));
    char* o = static_cast<char*>(E.out) + at * kOutSize;
    uint4 q[kClipVecs];
#pragma unroll
    for (int k = 0; k < kClipVecs; ++k) q[k] = p[k * kThreads + threadIdx.x];
#pragma unroll
    for (int k = 0; k < kClipVecs; ++k) {
      float x[8];
      unpack(q[k], kIn, x);
      store_scaled<kOut>(o + (k * kThreads + (int)threadIdx.x) * kPer * kOutSize, x, kPer, c);
    }
  } else {  // a tensor's first or last piece, or out is aligned otherwise than in
    const int64_t end = min(at + kElems, E.count);
#pragma unroll 4
    for (int64_t i = max(at, (int64_t)0) + threadIdx.x; i < end; i += kThreads)
      store_float(E.out, kOut, i, load_as_float(E.in, kIn, i) * c);
  }
}

template <int kMax, bool kInf>
__global__ void __launch_bounds__(kThreads, 8) clip_kernel(const __grid_constant__ TensorList<kMax> L,
                                                        const double* __restrict__ partial, int n_partial,
                                                        double max_norm, float* __restrict__ norm_out) {
  sarr::wait_for_previous();
  const double norm = total_norm<kInf>(partial, n_partial);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const float c = clip_coef(norm, max_norm);
  int t = L.n - 1;
  int64_t first = first_piece(L, t);
  for (int64_t p = L.pieces - 1 - blockIdx.x; p >= 0; p -= gridDim.x) {
    while (p < first) first = first_piece(L, --t);
    const Entry& E = L.e[t];
    if (c == 1.0f && E.out == E.in) {  // in place and nothing to clip, c x is x: on to the tensor before
      p -= (p - first) / gridDim.x * gridDim.x;
      continue;
    }
    const int64_t piece = p - first;
    if (E.type == SARR_F32) piece_clip<SARR_F32, SARR_F32>(E, piece, c);
    else if (E.type == SARR_BF16 && E.out_type == SARR_BF16) piece_clip<SARR_BF16, SARR_BF16>(E, piece, c);
    else if (E.type == SARR_BF16) piece_clip<SARR_BF16, SARR_F32>(E, piece, c);
    else if (E.out_type == SARR_F16) piece_clip<SARR_F16, SARR_F16>(E, piece, c);
    else piece_clip<SARR_F16, SARR_F32>(E, piece, c);
  }
}

// ---------------------------------------------------------------------------
// Adam
// ---------------------------------------------------------------------------
constexpr int kAdamPiece = kThreads * kAdamVecs * 4;  // elements

struct AdamRange {
  int64_t begin, count;  // elements of param / exp_avg / exp_avg_sq
  int64_t grad_begin;
  int64_t piece_end;
  float step_size;       // lr / (1 - beta1^step)
  uint8_t lead;          // elements between the 16-byte boundary below param + begin and it
  bool vec;              // all four arrays are aligned alike there
};

struct AdamList {
  int n;
  int64_t pieces;
  float one_m_beta1, beta2, one_m_beta2, bc2_sqrt, eps;
  AdamRange r[kAdamRanges];
};

// torch.optim.Adam's update of one element (no weight decay, no amsgrad), in
// the same operations as sarr_adam_step's.
__device__ __forceinline__ float adam_one(const AdamList& A, float step_size, float p, float g, float& m,
                                          float& v) {
  m = __fmaf_rn(A.one_m_beta1, __fsub_rn(g, m), m);
  v = __fadd_rn(__fmul_rn(v, A.beta2), __fmul_rn(__fmul_rn(A.one_m_beta2, g), g));
  const float denom = __fadd_rn(__fdiv_rn(__fsqrt_rn(v), A.bc2_sqrt), A.eps);
  return __fadd_rn(p, __fmul_rn(-step_size, __fdiv_rn(m, denom)));
}

__global__ void __launch_bounds__(kThreads, 6) adam_kernel(const __grid_constant__ AdamList A,
                                                        const double* __restrict__ partial, int n_partial,
                                                        double max_norm, float* __restrict__ param,
                                                        const float* __restrict__ grad,
                                                        float* __restrict__ exp_avg,
                                                        float* __restrict__ exp_avg_sq,
                                                        float* __restrict__ norm_out) {
  sarr::wait_for_previous();
  const double norm = total_norm<false>(partial, n_partial);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const float c = clip_coef(norm, max_norm);
  int t = A.n - 1;
  for (int64_t p = A.pieces - 1 - blockIdx.x; p >= 0; p -= gridDim.x) {
    while (t > 0 && p < A.r[t - 1].piece_end) --t;
    const AdamRange& R = A.r[t];
    const int64_t at = (p - (t > 0 ? A.r[t - 1].piece_end : 0)) * kAdamPiece - R.lead, count = R.count;
    float* P = param + R.begin;
    float* M = exp_avg + R.begin;
    float* V = exp_avg_sq + R.begin;
    const float* G = grad + R.grad_begin;
    const float step_size = R.step_size;
    if (R.vec) {
      float4 p4[kAdamVecs], g4[kAdamVecs], m4[kAdamVecs], v4[kAdamVecs];
#pragma unroll
      for (int k = 0; k < kAdamVecs; ++k) {
        const int64_t i = at + 4 * (k * kThreads + (int)threadIdx.x);
        if (i >= 0 && i + 4 <= count) {
          g4[k] = *reinterpret_cast<const float4*>(G + i);
          p4[k] = __ldcs(reinterpret_cast<const float4*>(P + i));
          m4[k] = __ldcs(reinterpret_cast<const float4*>(M + i));
          v4[k] = __ldcs(reinterpret_cast<const float4*>(V + i));
        }
      }
#pragma unroll
      for (int k = 0; k < kAdamVecs; ++k) {
        const int64_t i = at + 4 * (k * kThreads + (int)threadIdx.x);
        if (i >= 0 && i + 4 <= count) {
          p4[k].x = adam_one(A, step_size, p4[k].x, g4[k].x * c, m4[k].x, v4[k].x);
          p4[k].y = adam_one(A, step_size, p4[k].y, g4[k].y * c, m4[k].y, v4[k].y);
          p4[k].z = adam_one(A, step_size, p4[k].z, g4[k].z * c, m4[k].z, v4[k].z);
          p4[k].w = adam_one(A, step_size, p4[k].w, g4[k].w * c, m4[k].w, v4[k].w);
          __stcs(reinterpret_cast<float4*>(P + i), p4[k]);
          __stcs(reinterpret_cast<float4*>(M + i), m4[k]);
          __stcs(reinterpret_cast<float4*>(V + i), v4[k]);
        } else {
          for (int64_t e = max(i, (int64_t)0); e < min(i + 4, count); ++e) {
            float m = M[e], w = V[e];
            P[e] = adam_one(A, step_size, P[e], G[e] * c, m, w);
            M[e] = m;
            V[e] = w;
          }
        }
      }
    } else {
      for (int v = threadIdx.x; v < kAdamPiece; v += kThreads) {
        const int64_t i = at + v;
        if (i >= 0 && i < count) {
          float m = M[i], w = V[i];
          P[i] = adam_one(A, step_size, P[i], G[i] * c, m, w);
          M[i] = m;
          V[i] = w;
        }
      }
    }
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

int type_size(int type) { return type == SARR_F32 ? 4 : 2; }
bool type_ok(int type) { return type == SARR_F32 || type == SARR_BF16 || type == SARR_F16; }
unsigned lead_of(const void* p, int size) { return (unsigned)((reinterpret_cast<uintptr_t>(p) & 15) / size); }

int64_t ctas_for(int64_t pieces) { return pieces < kNormCtas ? (pieces > 0 ? pieces : 1) : kNormCtas; }

size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }

struct ListArgs {
  int n;
  const void* const* grads;
  const int64_t* counts;
  const int32_t* types;
  void* const* outs;
  const int32_t* out_types;
};

int check_list(const ListArgs& a) {
  if (a.n < 0 || (a.n > 0 && (!a.grads || !a.counts || !a.types))) return SARR_ERR_ARG;
  for (int i = 0; i < a.n; ++i) {
    if (a.counts[i] < 0 || a.counts[i] > (int64_t)1 << 48 || !type_ok(a.types[i])) return SARR_ERR_ARG;
    if (a.counts[i] == 0) continue;
    if (!a.grads[i] || reinterpret_cast<uintptr_t>(a.grads[i]) % type_size(a.types[i])) return SARR_ERR_ARG;
    if (a.outs) {
      const int ot = a.out_types ? a.out_types[i] : a.types[i];
      if (!type_ok(ot) || (ot != a.types[i] && ot != SARR_F32)) return SARR_ERR_ARG;
      if (!a.outs[i] || reinterpret_cast<uintptr_t>(a.outs[i]) % type_size(ot)) return SARR_ERR_ARG;
      if (a.outs[i] == a.grads[i] && ot != a.types[i]) return SARR_ERR_ARG;
    }
  }
  return SARR_OK;
}

// Whether no destination shares memory with another destination or with
// another tensor's source (its own source it may be, exactly).
int check_overlap(const ListArgs& a) {
  struct Span {
    uintptr_t begin, end;
  };
  if (a.n == 0) return SARR_OK;
  Span* out = new (std::nothrow) Span[2 * (size_t)a.n];
  if (!out) return SARR_ERR_WORKSPACE;
  Span* in = out + a.n;
  size_t n_out = 0, n_in = 0;
  for (int i = 0; i < a.n; ++i) {
    if (a.counts[i] == 0) continue;
    const uintptr_t g = reinterpret_cast<uintptr_t>(a.grads[i]), o = reinterpret_cast<uintptr_t>(a.outs[i]);
    const int ot = a.out_types ? a.out_types[i] : a.types[i];
    out[n_out++] = Span{o, o + (uintptr_t)a.counts[i] * type_size(ot)};
    if (g != o) in[n_in++] = Span{g, g + (uintptr_t)a.counts[i] * type_size(a.types[i])};
  }
  const auto before = [](const Span& x, const Span& y) { return x.begin < y.begin; };
  if (!std::is_sorted(out, out + n_out, before)) std::sort(out, out + n_out, before);
  if (!std::is_sorted(in, in + n_in, before)) std::sort(in, in + n_in, before);
  bool ok = true;
  for (size_t i = 1; i < n_out && ok; ++i) ok = out[i - 1].end <= out[i].begin;
  // the destinations are disjoint now: each source is held against those that
  // end behind its begin
  for (size_t i = 0, j = 0; i < n_in && ok; ++i) {
    while (j < n_out && out[j].end <= in[i].begin) ++j;
    ok = j == n_out || out[j].begin >= in[i].end;
  }
  delete[] out;
  return ok ? SARR_OK : SARR_ERR_ARG;
}

template <int kMax>
void fill_list(TensorList<kMax>& L, const ListArgs& a, int begin, int end, int piece_bytes) {
  L.n = 0;
  L.pieces = 0;
  for (int i = begin; i < end; ++i) {
    if (a.counts[i] == 0) continue;
    Entry& E = L.e[L.n++];
    E.in = a.grads[i];
    E.type = (uint8_t)a.types[i];
    E.count = a.counts[i];
    E.lead = (uint8_t)lead_of(E.in, type_size(E.type));
    E.out = nullptr;
    E.out_type = E.type;
    E.vec = false;
    if (a.outs) {
      E.out = a.outs[i];
      E.out_type = (uint8_t)(a.out_types ? a.out_types[i] : a.types[i]);
      E.vec = ((reinterpret_cast<uintptr_t>(E.out) - (uintptr_t)E.lead * type_size(E.out_type)) & 15) == 0;
    }
    const int64_t piece = piece_bytes / type_size(E.type);
    L.pieces += (E.lead + E.count + piece - 1) / piece;
    E.piece_end = L.pieces;
  }
}

template <int kMax, bool kInf>
cudaError_t norm_group(const ListArgs& a, int begin, int end, bool dependent, double* partial, int* n_partial,
                       cudaStream_t s) {
  TensorList<kMax> L;
  fill_list(L, a, begin, end, kNormThreads * kNormVecs * 16);
  if (L.n == 0) return cudaSuccess;
  const unsigned ctas = (unsigned)ctas_for(L.pieces);
  const cudaError_t e = sarr::launch(norm_kernel<kMax, kInf>, {dim3(ctas), kNormThreads, 0, dependent}, s, L,
                                     partial + *n_partial);
  *n_partial += (int)ctas;
  sarr::count_launches(1);
  return e;
}

template <int kMax, bool kInf>
cudaError_t clip_group(const ListArgs& a, int begin, int end, const double* partial, int n_partial,
                       double max_norm, float* norm_out, cudaStream_t s) {
  TensorList<kMax> L;
  fill_list(L, a, begin, end, kThreads * kClipVecs * 16);
  if (L.n == 0) return cudaSuccess;
  const unsigned ctas = (unsigned)std::min<int64_t>(L.pieces, kClipCtas);
  sarr::count_launches(1);
  return sarr::launch(clip_kernel<kMax, kInf>, {dim3(ctas), kThreads, 0, true}, s, L, partial, n_partial,
                      max_norm, norm_out);
}

// The partials of all tensors, then (outs) the clipped gradients and the norm,
// or the norm alone. Lists of more than kLargeList tensors take several launches.
template <bool kInf>
cudaError_t run_list(const ListArgs& a, double max_norm, float* norm_out, double* partial, cudaStream_t s) {
  int n_partial = 0;
  bool dependent = false;
  for (int b = 0; b < a.n; b += kLargeList) {
    const int e = std::min(a.n, b + kLargeList), before = n_partial;
    const cudaError_t st =
        e - b <= kSmallList    ? norm_group<kSmallList, kInf>(a, b, e, dependent, partial, &n_partial, s)
        : e - b <= kMediumList ? norm_group<kMediumList, kInf>(a, b, e, dependent, partial, &n_partial, s)
                               : norm_group<kLargeList, kInf>(a, b, e, dependent, partial, &n_partial, s);
    if (st != cudaSuccess) return st;
    dependent = dependent || n_partial > before;
  }
  if (!a.outs || n_partial == 0) {
    if (!norm_out) return cudaSuccess;
    sarr::count_launches(1);
    return sarr::launch(finish_kernel<kInf>, {dim3(1), kThreads, 0, dependent}, s, partial, n_partial, norm_out);
  }
  float* out = norm_out;
  for (int b = 0; b < a.n; b += kLargeList) {
    const int e = std::min(a.n, b + kLargeList);
    bool any = false;
    for (int i = b; i < e; ++i) any = any || a.counts[i] > 0;
    if (!any) continue;
    const cudaError_t st =
        e - b <= kSmallList    ? clip_group<kSmallList, kInf>(a, b, e, partial, n_partial, max_norm, out, s)
        : e - b <= kMediumList ? clip_group<kMediumList, kInf>(a, b, e, partial, n_partial, max_norm, out, s)
                               : clip_group<kLargeList, kInf>(a, b, e, partial, n_partial, max_norm, out, s);
    if (st != cudaSuccess) return st;
    out = nullptr;
  }
  return cudaSuccess;
}

int run_norm(const ListArgs& a, int norm_kind, double max_norm, float* norm_out, void* ws, size_t ws_bytes,
             sarr_stream_t stream) {
  size_t need = 0;
  if (norm_kind != SARR_NORM_2 && norm_kind != SARR_NORM_INF) return SARR_ERR_ARG;
  int st = check_list(a);
  if (st != SARR_OK) return st;
  if (sarr_grad_norm_workspace_size(a.n, &need) != SARR_OK) return SARR_ERR_ARG;
  if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)) return SARR_ERR_WORKSPACE;
  if (a.outs && (st = check_overlap(a)) != SARR_OK) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(ws);
  return cuda_status(norm_kind == SARR_NORM_INF ? run_list<true>(a, max_norm, norm_out, partial, s)
                                                : run_list<false>(a, max_norm, norm_out, partial, s));
}

}  // namespace

extern "C" int sarr_grad_norm_workspace_size(int n_tensors, size_t* bytes) {
  if (!bytes || n_tensors < 0) return SARR_ERR_ARG;
  const size_t launches = ((size_t)n_tensors + kLargeList - 1) / kLargeList;
  *bytes = round256((launches > 0 ? launches : 1) * kNormCtas * sizeof(double));
  return SARR_OK;
}

extern "C" int sarr_grad_norm(int n_tensors, const void* const* grads, const int64_t* counts,
                              const int32_t* types, int norm_kind, float* norm_out, void* ws,
                              size_t ws_bytes, sarr_stream_t stream) {
  if (!norm_out) return SARR_ERR_ARG;
  return run_norm(ListArgs{n_tensors, grads, counts, types, nullptr, nullptr}, norm_kind, 0.0, norm_out, ws,
                  ws_bytes, stream);
}

extern "C" int sarr_clip_grads(int n_tensors, const void* const* grads, const int64_t* counts,
                               const int32_t* types, void* const* outs, const int32_t* out_types,
                               int norm_kind, double max_norm, float* norm_out, void* ws, size_t ws_bytes,
                               sarr_stream_t stream) {
  if (!(max_norm >= 0.0) || (n_tensors > 0 && !outs)) return SARR_ERR_ARG;
  return run_norm(ListArgs{n_tensors, grads, counts, types, outs, out_types}, norm_kind, max_norm, norm_out,
                  ws, ws_bytes, stream);
}

extern "C" int sarr_adam_step_clipped(int n_ranges, const int64_t* range_begin, const int64_t* range_end,
                                      const int64_t* grad_begin, const double* range_lr, float* param,
                                      const float* grad, float* exp_avg, float* exp_avg_sq, double beta1,
                                      double beta2, double eps, int64_t step, double max_norm,
                                      float* norm_out, void* ws, size_t ws_bytes, sarr_stream_t stream) {
  if (n_ranges < 0 || n_ranges > kAdamRanges || step < 1 || !(max_norm >= 0.0)) return SARR_ERR_ARG;
  if (n_ranges > 0 && (!range_begin || !range_end || !grad_begin || !range_lr)) return SARR_ERR_ARG;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return SARR_ERR_ARG;
  size_t need = 0;
  if (sarr_grad_norm_workspace_size(kAdamRanges, &need) != SARR_OK) return SARR_ERR_ARG;
  if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)) return SARR_ERR_WORKSPACE;
  AdamList A;
  memset(&A, 0, sizeof(A));
  const void* grads[kAdamRanges];
  int64_t counts[kAdamRanges];
  int32_t types[kAdamRanges];
  int64_t sorted[kAdamRanges][2];
  const double bc1 = 1.0 - pow(beta1, (double)step), bc2 = 1.0 - pow(beta2, (double)step);
  for (int k = 0; k < n_ranges; ++k) {
    if (range_begin[k] < 0 || range_end[k] < range_begin[k] || grad_begin[k] < 0) return SARR_ERR_ARG;
    const int64_t count = range_end[k] - range_begin[k];
    if (count > (int64_t)1 << 48) return SARR_ERR_ARG;
    if (count == 0) continue;
    if (!param || !grad || !exp_avg || !exp_avg_sq) return SARR_ERR_ARG;
    AdamRange& R = A.r[A.n];
    R.begin = range_begin[k];
    R.count = count;
    R.grad_begin = grad_begin[k];
    R.step_size = (float)(range_lr[k] / bc1);
    R.lead = (uint8_t)lead_of(param + R.begin, 4);
    R.vec = lead_of(grad + R.grad_begin, 4) == R.lead && lead_of(exp_avg + R.begin, 4) == R.lead &&
            lead_of(exp_avg_sq + R.begin, 4) == R.lead;
    A.pieces += (R.lead + count + kAdamPiece - 1) / kAdamPiece;
    R.piece_end = A.pieces;
    grads[A.n] = grad + R.grad_begin;
    counts[A.n] = count;
    types[A.n] = SARR_F32;
    sorted[A.n][0] = range_begin[k];
    sorted[A.n][1] = range_end[k];
    ++A.n;
  }
  for (int i = 0; i < A.n; ++i)  // ranges are disjoint
    for (int j = 0; j < i; ++j)
      if (sorted[i][0] < sorted[j][1] && sorted[j][0] < sorted[i][1]) return SARR_ERR_ARG;
  A.one_m_beta1 = (float)(1.0 - beta1);
  A.beta2 = (float)beta2;
  A.one_m_beta2 = (float)(1.0 - beta2);
  A.bc2_sqrt = (float)sqrt(bc2);
  A.eps = (float)eps;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(ws);
  const ListArgs list{A.n, grads, counts, types, nullptr, nullptr};
  if (A.n == 0) return cuda_status(run_list<false>(list, max_norm, norm_out, partial, s));
  int n_partial = 0;
  cudaError_t e = A.n <= kSmallList ? norm_group<kSmallList, false>(list, 0, A.n, false, partial, &n_partial, s)
                                    : norm_group<kMediumList, false>(list, 0, A.n, false, partial, &n_partial, s);
  if (e != cudaSuccess) return cuda_status(e);
  const unsigned ctas = (unsigned)std::min<int64_t>(A.pieces, kAdamCtas);
  sarr::count_launches(1);
  return cuda_status(sarr::launch(adam_kernel, {dim3(ctas), kThreads, 0, true}, s, A, partial, n_partial,
                                  max_norm, param, grad, exp_avg, exp_avg_sq, norm_out));
}
