// The global norm of many gradient tensors, and their clipping, for gfx950.
//
//   norm = sqrt(sum over all tensors of g^2),  coef = min(1, max_norm / (norm + 1e-6)),  out = clamp(coef g, -v, v)
// (torch.nn.utils.clip_grad_norm_ and clip_grad_value_ as the reference calls them, src/models/for_training.py:98-109), for
// gradients that lie in tensors of their own; the flat buffer of the framework's own engine has vpt_grad_sumsq.
//
// The tensors are cut into pieces of at most kPiece values beforehand (a table in device memory, one entry per piece), so that
// one launch covers any number of them, tiny and large. Pass 1: block b takes pieces b, b + blocks, ... and leaves the sum of
// their squares in part[b] (a fixed order: the same bits every time). Pass 2: every block adds all of part in the same order
// and scales its pieces, last pieces first (they are still in the cache). Squares are added in 64 bits: f32 squares leave the
// range for values past 1.8e19 or below 1e-23.
// Bound by HBM. 87 M f32 values into buffers of their own: 59 us for the norm (5.8 TB/s), 112 for the clipping (6.2 TB/s with
// what the cache holds); in place and over the limit 176 for both. 42 M bf16 values in 1400 tensors, in place and under the
// limit: 15 us (5.7 TB/s) and 4, the second pass reading the sums and no gradient; over the limit 43 for both. 1024 blocks:
// 2048 are level, 512 lose 40 % of the first pass.
#include "common.h"

namespace {

enum { GC_BF16 = 0, GC_F32 = 1, GC_F16 = 2 };
constexpr int kPiece = 16384;
constexpr int kBlocks = 1024;

struct Piece {  // include/vpt_hip.h VptGradPiece
  const void* g;
  void* out;
  int n, dtype;
};

template <int T> constexpr int gc_size() { return T == GC_F32 ? 4 : 2; }
template <int T> constexpr int gc_vec() { return 16 / gc_size<T>(); }  // values of 16 bytes

template <int T>
__device__ __forceinline__ float gc_get(const void* p, int i) {
  return T == GC_F32    ? reinterpret_cast<const float*>(p)[i]
         : T == GC_BF16 ? bf2f(reinterpret_cast<const bf16_t*>(p)[i])
                        : h2f(reinterpret_cast<const unsigned short*>(p)[i]);
}
template <int T>
__device__ __forceinline__ void gc_put(void* p, int i, float v) {
  if (T == GC_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (T == GC_BF16) reinterpret_cast<bf16_t*>(p)[i] = f2bf(v);
  else reinterpret_cast<unsigned short*>(p)[i] = f2h(v);
}
template <int T>
__device__ __forceinline__ void gc_unpack(uint4 v, float (&f)[gc_vec<T>()]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (T == GC_F32) f[e] = __uint_as_float(w[e]);
    else if constexpr (T == GC_BF16) f[2 * e] = __uint_as_float(w[e] << 16), f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    else f[2 * e] = h2f(w[e] & 0xffff), f[2 * e + 1] = h2f(w[e] >> 16);
  }
}
template <int T>
__device__ __forceinline__ uint4 gc_pack(const float (&f)[gc_vec<T>()]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (T == GC_F32) w[e] = __float_as_uint(f[e]);
    else if constexpr (T == GC_BF16) w[e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
    else w[e] = f2h(f[2 * e]) | (uint32_t)f2h(f[2 * e + 1]) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Values before the first 16-byte boundary of p (at most n).
template <int T>
__device__ __forceinline__ int gc_head(const void* p, int n) {
  const int k = (int)((-(uintptr_t)p & 15) / gc_size<T>());
  return k < n ? k : n;
}

__device__ __forceinline__ double block_sum(double v) {  // 256 threads; the result in every thread
  __shared__ double red[4];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// 16-byte loads, four per thread in flight; the values before the first boundary and behind the last one apart.
template <int T>
__device__ __forceinline__ double piece_sumsq(const Piece& p) {
  constexpr int V = gc_vec<T>(), U = 4;
  const int head = gc_head<T>(p.g, p.n), nv = (p.n - head) / V, tail = head + nv * V;
  double s = 0.;
  if ((int)threadIdx.x < head) {
    const double v = gc_get<T>(p.g, threadIdx.x);
    s += v * v;
  }
  if (tail + (int)threadIdx.x < p.n) {
    const double v = gc_get<T>(p.g, tail + threadIdx.x);
    s += v * v;
  }
  const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p.g) + head * gc_size<T>());
  for (int i = threadIdx.x; i < nv; i += 256 * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = i + 256 * u < nv ? q[i + 256 * u] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[V];
      gc_unpack<T>(w[u], f);
#pragma unroll
      for (int e = 0; e < V; ++e) s = fma((double)f[e], (double)f[e], s);
    }
  }
  return s;
}

__global__ __launch_bounds__(256) void grad_list_sumsq_kernel(const Piece* __restrict__ pieces, int count,
                                                              double* __restrict__ part) {
  double s = 0.;
  for (int i = blockIdx.x; i < count; i += gridDim.x) {
    const Piece p = pieces[i];
    s += p.dtype == GC_F32 ? piece_sumsq<GC_F32>(p) : p.dtype == GC_BF16 ? piece_sumsq<GC_BF16>(p) : piece_sumsq<GC_F16>(p);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double parts_norm(const double* part, int n) {
  double s = 0.;
  for (int i = threadIdx.x; i < n; i += 256) s += part[i];
  return sqrt(block_sum(s));
}

__device__ __forceinline__ float gc_clip(float v, float coef, float limit) {
  v *= coef;
  return limit > 0.f ? (v < -limit ? -limit : v > limit ? limit : v) : v;  // a NaN stays one
}
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
// STREAM: stores that leave no copy in the caches.
template <int T, bool STREAM>
__device__ __forceinline__ void piece_clip(const Piece& p, float coef, float limit) {
  constexpr int V = gc_vec<T>(), U = 4;
  int head = gc_head<T>(p.g, p.n), nv = (p.n - head) / V;
  if (((uintptr_t)p.g ^ (uintptr_t)p.out) & 15) head = p.n, nv = 0;  // no 16-byte pieces in common: value by value
  const int tail = head + nv * V;
  for (int i = threadIdx.x; i < head; i += 256) gc_put<T>(p.out, i, gc_clip(gc_get<T>(p.g, i), coef, limit));
  for (int i = tail + threadIdx.x; i < p.n; i += 256) gc_put<T>(p.out, i, gc_clip(gc_get<T>(p.g, i), coef, limit));
  const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p.g) + (long)head * gc_size<T>());
  uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<char*>(p.out) + (long)head * gc_size<T>());
  for (int i = threadIdx.x; i < nv; i += 256 * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = i + 256 * u < nv ? q[i + 256 * u] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[V];
      gc_unpack<T>(w[u], f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = gc_clip(f[e], coef, limit);
      w[u] = gc_pack<T>(f);
      if (i + 256 * u < nv) {
        if (STREAM) __builtin_nontemporal_store(u32x4_t{w[u].x, w[u].y, w[u].z, w[u].w}, reinterpret_cast<u32x4_t*>(o + i + 256 * u));
        else o[i + 256 * u] = w[u];
      }
    }
  }
}

// max_norm <= 0: no norm clipping (part is not read, norm not written); limit <= 0: no value clipping.
template <bool STREAM>
__global__ __launch_bounds__(256) void grad_list_clip_kernel(const Piece* __restrict__ pieces, int count,
                                                             const double* __restrict__ part, int parts, float max_norm,
                                                             float limit, float* __restrict__ norm_out) {
  float coef = 1.f;
  if (part) {
    const double norm = parts_norm(part, parts);
    if (max_norm > 0.f) {
      const double c = (double)max_norm / (norm + 1e-6);
      coef = c < 1. ? (float)c : c != c ? (float)c : 1.f;  // a NaN norm makes every gradient NaN
    }
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  }
  for (int i = count - 1 - (int)blockIdx.x; i >= 0; i -= gridDim.x) {  // last read, first again: what the caches still hold
    const Piece p = pieces[i];
    if (coef == 1.f && limit <= 0.f && p.out == p.g) continue;  // in place and nothing changes
    if (p.dtype == GC_F32) piece_clip<GC_F32, STREAM>(p, coef, limit);
    else if (p.dtype == GC_BF16) piece_clip<GC_BF16, STREAM>(p, coef, limit);
    else piece_clip<GC_F16, STREAM>(p, coef, limit);
  }
}

}  // namespace

extern "C" int vpt_grad_list_piece(void) { return kPiece; }
extern "C" int vpt_grad_list_parts(int count) { return count < 1 ? 1 : count < kBlocks ? count : kBlocks; }

extern "C" int vpt_grad_list_norm(const void* pieces, int count, double* part, void* stream) {
  VPT_CHECK_ARG(count >= 0 && part && ((uintptr_t)part & 7) == 0 && (count == 0 || pieces),
                "vpt_grad_list_norm: pieces, part of vpt_grad_list_parts(count) doubles");
  hipLaunchKernelGGL(grad_list_sumsq_kernel, dim3(vpt_grad_list_parts(count)), dim3(256), 0, (hipStream_t)stream,
                     (const Piece*)pieces, count, part);
  VPT_LAUNCH_CHECK();
  return VPT_OK;
}

extern "C" int vpt_grad_list_clip(const void* pieces, int count, int cached, const double* part, int parts, float max_norm,
                                  float clip_value, float* norm_out, void* stream) {
  VPT_CHECK_ARG(count >= 0 && (count == 0 || pieces), "vpt_grad_list_clip: bad table");
  VPT_CHECK_ARG(max_norm >= 0.f && clip_value >= 0.f, "vpt_grad_list_clip: max_norm, clip_value >= 0 (0: off)");
  VPT_CHECK_ARG((part && parts >= 1 && parts <= kBlocks && ((uintptr_t)part & 7) == 0) || (!part && max_norm == 0.f && !norm_out),
                "vpt_grad_list_clip: a norm needs part, the parts doubles that vpt_grad_list_norm wrote");
  const dim3 grid(vpt_grad_list_parts(count));
  if (cached)
    hipLaunchKernelGGL(grad_list_clip_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, (const Piece*)pieces, count, part,
                       parts, max_norm, clip_value, norm_out);
  else
    hipLaunchKernelGGL(grad_list_clip_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, (const Piece*)pieces, count, part,
                       parts, max_norm, clip_value, norm_out);
  VPT_LAUNCH_CHECK();
  return VPT_OK;
}
