// The global norm of many gradient tensors, and their clipping, for gfx950.
//
//   norm = sqrt(sum over all tensors of g^2),  coef = min(1, max_norm / (norm + 1e-6)),  out = clamp(coef g, -v, v)
// (torch.nn.utils.clip_grad_norm_ and clip_grad_value_ as the reference calls them, src/models/for_training.py:98-109), for
// gradients that lie in tensors of their own; the flat buffer of the framework's own engine has vpt_grad_sumsq.
//
// The tensors are cut into pieces of at most kPiece values beforehand (a table in device memory, one entry per piece), so that
// one launch covers any number of them, tiny and large. Pass 1: block b takes pieces b, b + blocks, ... and leaves the sum of
// their squares in part[b] (a fixed order: the same bits every time). Pass 2: every block adds all of part in the same order
// and scales its pieces. Squares are added in 64 bits: f32 squares leave the range for values past 1.8e19 or below 1e-23.
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

__device__ __forceinline__ double block_sum(double v) {  // 256 threads; the result in every thread
  __shared__ double red[4];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <int T>
__device__ __forceinline__ double piece_sumsq(const Piece& p) {
  double s = 0.;
  for (int i = threadIdx.x; i < p.n; i += 256) {
    const double v = gc_get<T>(p.g, i);
    s += v * v;
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

template <int T>
__device__ __forceinline__ void piece_clip(const Piece& p, float coef, float limit) {
  for (int i = threadIdx.x; i < p.n; i += 256) {
    float v = gc_get<T>(p.g, i) * coef;
    if (limit > 0.f) v = v < -limit ? -limit : v > limit ? limit : v;  // a NaN stays one
    gc_put<T>(p.out, i, v);
  }
}

// max_norm <= 0: no norm clipping (part is not read, norm not written); limit <= 0: no value clipping.
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
  for (int i = blockIdx.x; i < count; i += gridDim.x) {
    const Piece p = pieces[i];
    if (coef == 1.f && limit <= 0.f && p.out == p.g) continue;  // in place and nothing changes
    if (p.dtype == GC_F32) piece_clip<GC_F32>(p, coef, limit);
    else if (p.dtype == GC_BF16) piece_clip<GC_BF16>(p, coef, limit);
    else piece_clip<GC_F16>(p, coef, limit);
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

extern "C" int vpt_grad_list_clip(const void* pieces, int count, const double* part, int parts, float max_norm,
                                  float clip_value, float* norm_out, void* stream) {
  VPT_CHECK_ARG(count >= 0 && (count == 0 || pieces), "vpt_grad_list_clip: bad table");
  VPT_CHECK_ARG(max_norm >= 0.f && clip_value >= 0.f, "vpt_grad_list_clip: max_norm, clip_value >= 0 (0: off)");
  VPT_CHECK_ARG((part && parts >= 1 && parts <= kBlocks && ((uintptr_t)part & 7) == 0) || (!part && max_norm == 0.f && !norm_out),
                "vpt_grad_list_clip: a norm needs part, the parts doubles that vpt_grad_list_norm wrote");
  hipLaunchKernelGGL(grad_list_clip_kernel, dim3(vpt_grad_list_parts(count)), dim3(256), 0, (hipStream_t)stream,
                     (const Piece*)pieces, count, part, parts, max_norm, clip_value, norm_out);
  VPT_LAUNCH_CHECK();
  return VPT_OK;
}
