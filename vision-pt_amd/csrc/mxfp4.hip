// Microscaled 4-bit floating point (MXFP4) for gfx950: quantisation, dequantisation and the product of two such matrices.
//
// Format (the OCP microscaling formats' MXFP4): a row of K values, padded with zeros to a multiple of 128, in blocks of
// 32 consecutive ones. A block has the scale 2^(s - 127), s one byte, and 32 codes e2m1: sign and
// {0, 0.5, 1, 1.5, 2, 3, 4, 6}. s = max(floor(log2 max|x|) + 125, 0), the exponent that brings the largest value into
// [4, 8); code = x / 2^(s - 127) rounded to the nearest, ties to the even code, and saturated at 6. A block with an
// infinity or a NaN gets s = 255, which makes all its values NaN. Every step but that rounding is exact (the scales are
// powers of two), so codes and scales do not depend on how the work is split.
// Codes: row r, byte i of [M][64 c] holds the values 2 i (low half) and 2 i + 1, c = ceil(K / 128); scales [M][4 c].
//
// A 16x16x128 scaled MFMA takes from each lane 32 codes of one row (16 bytes) and that block's scale byte: lane l holds
// row l & 15, block l >> 4 of the 128-deep step. These are the byte positions of the bf16 16x16x32 MFMA (16 bytes per
// lane, 64-byte rows per step), at four times the values per byte.
#include "gemm_common.h"

namespace {

using namespace vptg;

typedef int intx8 __attribute__((ext_vector_type(8)));

enum { MX_BF16 = 0, MX_F32 = 1, MX_F16 = 2 };

__device__ __forceinline__ uint32_t dpp_xor1(uint32_t v) {  // quad_perm [1, 0, 3, 2]
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t dpp_xor2(uint32_t v) {  // quad_perm [2, 3, 0, 1]
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);
}

// Eight values of one row from column c0 on, as f32; columns at or past K are zero. VEC: K % 8 == 0 and 16-byte rows.
template <int T, bool VEC>
__device__ __forceinline__ void mx_load8(const void* x, long at, int c0, int K, float (&f)[8]) {
  if (VEC) {
    if (c0 >= K) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
    } else if (T == MX_F32) {
      const floatx4 a = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(x) + at);
      const floatx4 b = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(x) + at + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned short*>(x) + at);
      if (T == MX_BF16) {
        unpack8(v, f);
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) f[2 * e] = h2f(w[e] & 0xffff), f[2 * e + 1] = h2f(w[e] >> 16);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = 0.f;
      if (c0 + e < K)
        f[e] = T == MX_F32    ? reinterpret_cast<const float*>(x)[at + e]
               : T == MX_BF16 ? bf2f(reinterpret_cast<const bf16_t*>(x)[at + e])
                              : h2f(reinterpret_cast<const unsigned short*>(x)[at + e]);
    }
  }
}

// The scale byte of a block whose largest magnitude has these f32 bits (sign cleared).
__device__ __forceinline__ uint32_t mx_scale(uint32_t top) {
  const uint32_t be = top >> 23;
  return be == 255u ? 255u : be > 2u ? be - 2u : 0u;
}

// Eight codes of the values f under scale byte s: e2m1 by comparisons with the seven midpoints.
__device__ __forceinline__ uint32_t mx_codes8(const float (&f)[8], uint32_t s) {
  if (s == 255u) return 0u;
  const float inv = __uint_as_float((254u - s) << 23);  // 2^(127 - s), s <= 252
  uint32_t out = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = fabsf(f[e]) * inv;
    const uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
    out |= (c | (__float_as_uint(f[e]) >> 31 << 3)) << (4 * e);
  }
  return out;
}

// One thread per 8 values: four neighbouring lanes share a block. Bound by HBM: 2 (or 4) bytes in, 17 / 32 out per value.
template <int T, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const void* __restrict__ x, long ldx, unsigned total,
                                                          unsigned nch, int K, uint8_t* __restrict__ codes, long ldc,
                                                          uint8_t* __restrict__ scales, long lds) {
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= total) return;  // total % 16 == 0: the lanes of a block leave together
  const unsigned row = idx / nch, c = idx - row * nch;
  float f[8];
  mx_load8<T, VEC>(x, (long)row * ldx + c * 8, c * 8, K, f);
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
  top = max(top, dpp_xor1(top));
  top = max(top, dpp_xor2(top));
  const uint32_t s = mx_scale(top);
  *reinterpret_cast<uint32_t*>(codes + (long)row * ldc + c * 4) = mx_codes8(f, s);
  if ((c & 3) == 0) scales[(long)row * lds + (c >> 2)] = (uint8_t)s;
}

__device__ __forceinline__ float mx_value(uint32_t code, float unit) {
  const uint32_t m = code & 7u;  // 0, 0.5, then 1.m x 2^(m / 2 - 1)
  const float v = m < 2u ? 0.5f * (float)m : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1u) << 22);
  return (code & 8u ? -v : v) * unit;
}
__device__ __forceinline__ float mx_unit(uint32_t s) {  // 2^(s - 127); NaN for 255
  return __uint_as_float(s == 255u ? 0x7fc00000u : s ? s << 23 : 1u << 22);
}

// One thread per 8 values. VEC: K % 8 == 0 and 16-byte rows.
template <bool F32OUT, bool VEC>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, long ldc,
                                                            const uint8_t* __restrict__ scales, long lds, unsigned total,
                                                            unsigned nch, int K, void* __restrict__ out, long ldo) {
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= total) return;
  const unsigned row = idx / nch, c = idx - row * nch;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + (long)row * ldc + c * 4);
  const float unit = mx_unit(scales[(long)row * lds + (c >> 2)]);
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = mx_value(w >> (4 * e), unit);
  const long at = (long)row * ldo + c * 8;
  if (VEC) {
    if (F32OUT) {
      *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(out) + at) = floatx4{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(out) + at + 4) = floatx4{f[4], f[5], f[6], f[7]};
    } else {
      *reinterpret_cast<uint4*>(reinterpret_cast<bf16_t*>(out) + at) = pack8(f);  // exact: two significant bits
    }
  } else {
    for (int e = 0; e < 8 && (int)(c * 8) + e < K; ++e) {
      if (F32OUT) reinterpret_cast<float*>(out)[at + e] = f[e];
      else reinterpret_cast<bf16_t*>(out)[at + e] = f2bf(f[e]);
    }
  }
}

struct MxArgs {
  const uint8_t* A; long lda;    // codes [M][64 steps], bytes per row
  const uint8_t* AS; long ldas;  // scales [M][4 steps]
  const uint8_t* B; long ldb;
  const uint8_t* BS; long ldbs;
  void* C; long ldc;
  const bf16_t* bias;
  const bf16_t* resid; long ldr;
  int M, N, steps;  // steps of 128 along K
  int f32out;
};

__device__ __forceinline__ intx8 mx_frag(uint4 v) { return intx8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }

__device__ __forceinline__ floatx4 mx_mfma(uint4 a, uint4 b, floatx4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_frag(a), mx_frag(b), c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// 128 x 128 tile, 4 waves of 64 x 64, one 128-deep step at a time through LDS.
__global__ __launch_bounds__(256) void mx_gemm_kernel(MxArgs g) {
  __shared__ __attribute__((aligned(16))) char as[128 * 64], bs[128 * 64];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid >> 1, wn = wid & 1;
  const int tiles_n = (g.N + 127) / 128;
  const int m0 = blockIdx.x / tiles_n * 128, n0 = blockIdx.x % tiles_n * 128;
  floatx4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int t = 0; t < g.steps; ++t) {
    uint4 va[2], vb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // rows past the edge: the last one (its results are not stored)
      const int row = (tid >> 2) + 64 * i, ch = tid & 3;
      va[i] = *reinterpret_cast<const uint4*>(g.A + (long)min(m0 + row, g.M - 1) * g.lda + t * 64 + ch * 16);
      vb[i] = *reinterpret_cast<const uint4*>(g.B + (long)min(n0 + row, g.N - 1) * g.ldb + t * 64 + ch * 16);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = (tid >> 2) + 64 * i, ch = tid & 3;
      *reinterpret_cast<uint4*>(as + kmaj32_off(row, ch)) = va[i];
      *reinterpret_cast<uint4*>(bs + kmaj32_off(row, ch)) = vb[i];
    }
    __syncthreads();
    uint4 af[4], bf[4];
    uint32_t sa[4], sb[4];
    const int r = lane & 15, blk = lane >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ra = wm * 64 + i * 16 + r, rb = wn * 64 + i * 16 + r;
      af[i] = *reinterpret_cast<const uint4*>(as + kmaj32_off(ra, blk));
      bf[i] = *reinterpret_cast<const uint4*>(bs + kmaj32_off(rb, blk));
      sa[i] = g.AS[(long)min(m0 + ra, g.M - 1) * g.ldas + t * 4 + blk];
      sb[i] = g.BS[(long)min(n0 + rb, g.N - 1) * g.ldbs + t * 4 + blk];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mx_mfma(af[i], bf[j], acc[i][j], sa[i], sb[j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + wm * 64 + i * 16 + (lane >> 4) * 4 + r, n = n0 + wn * 64 + j * 16 + (lane & 15);
        if (m >= g.M || n >= g.N) continue;
        float v = acc[i][j][r];
        if (g.bias) v += bf2f(g.bias[n]);
        if (g.resid) v += bf2f(g.resid[(long)m * g.ldr + n]);
        if (g.f32out) reinterpret_cast<float*>(g.C)[(long)m * g.ldc + n] = v;
        else reinterpret_cast<bf16_t*>(g.C)[(long)m * g.ldc + n] = f2bf(v);
      }
}

bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

template <int T, bool VEC>
void mx_quantize_launch(const void* x, long ldx, long rows, unsigned nch, int K, uint8_t* codes, long ldc, uint8_t* scales,
                        long lds, hipStream_t s) {
  const unsigned total = (unsigned)(rows * nch);
  hipLaunchKernelGGL((mx_quantize_kernel<T, VEC>), dim3((total + 255u) / 256u), dim3(256), 0, s, x, ldx, total, nch, K,
                     codes, ldc, scales, lds);
}

}  // namespace

extern "C" int vpt_mxfp4_quantize(const void* x, int dtype, long ldx, long M, int K, void* codes, long ldc, void* scales,
                                  long lds, void* stream) {
  VPT_CHECK_ARG(dtype >= MX_BF16 && dtype <= MX_F16, "vpt_mxfp4_quantize: dtype 0 bf16, 1 f32, 2 f16");
  VPT_CHECK_ARG(M >= 0 && K > 0 && K <= (1 << 30), "vpt_mxfp4_quantize: M >= 0, 0 < K <= 2^30");
  if (M == 0) return VPT_OK;
  VPT_CHECK_ARG(x && codes && scales, "vpt_mxfp4_quantize: null pointer");
  const long steps = (K + 127) / 128;
  VPT_CHECK_ARG(ldx >= K || M == 1, "vpt_mxfp4_quantize: ldx >= K");
  VPT_CHECK_ARG(ldc >= 64 * steps && ldc % 16 == 0 && aligned(codes, 16),
                "vpt_mxfp4_quantize: code rows of 64 ceil(K / 128) bytes at multiples of 16 bytes");
  VPT_CHECK_ARG(lds >= 4 * steps && lds % 4 == 0 && aligned(scales, 4),
                "vpt_mxfp4_quantize: scale rows of 4 ceil(K / 128) bytes at multiples of 4 bytes");
  const int es = dtype == MX_F32 ? 4 : 2;
  VPT_CHECK_ARG(aligned(x, es), "vpt_mxfp4_quantize: x is not aligned to its type");
  const bool vec = K % 8 == 0 && aligned(x, 16) && ldx * es % 16 == 0;
  const unsigned nch = (unsigned)(steps * 16);
  const long slab = (1L << 31) / nch;  // rows of a launch: its chunk index stays in 32 bits
  for (long r = 0; r < M; r += slab) {
    const long n = M - r < slab ? M - r : slab;
    const void* xr = (const char*)x + r * ldx * es;
    uint8_t* cr = (uint8_t*)codes + r * ldc;
    uint8_t* sr = (uint8_t*)scales + r * lds;
    hipStream_t st = (hipStream_t)stream;
#define VPT_MXQ(T)                                                              \
  vec ? mx_quantize_launch<T, true>(xr, ldx, n, nch, K, cr, ldc, sr, lds, st)   \
      : mx_quantize_launch<T, false>(xr, ldx, n, nch, K, cr, ldc, sr, lds, st)
    if (dtype == MX_BF16) VPT_MXQ(MX_BF16);
    else if (dtype == MX_F32) VPT_MXQ(MX_F32);
    else VPT_MXQ(MX_F16);
#undef VPT_MXQ
    VPT_LAUNCH_CHECK();
  }
  return VPT_OK;
}

extern "C" int vpt_mxfp4_dequantize(const void* codes, long ldc, const void* scales, long lds, long M, int K, void* out,
                                    long ldo, int f32_out, void* stream) {
  VPT_CHECK_ARG(M >= 0 && K > 0 && K <= (1 << 30), "vpt_mxfp4_dequantize: M >= 0, 0 < K <= 2^30");
  if (M == 0) return VPT_OK;
  VPT_CHECK_ARG(codes && scales && out, "vpt_mxfp4_dequantize: null pointer");
  const long steps = (K + 127) / 128;
  VPT_CHECK_ARG(ldc >= 64 * steps && ldc % 16 == 0 && aligned(codes, 16),
                "vpt_mxfp4_dequantize: code rows of 64 ceil(K / 128) bytes at multiples of 16 bytes");
  VPT_CHECK_ARG(lds >= 4 * steps && lds % 4 == 0 && aligned(scales, 4),
                "vpt_mxfp4_dequantize: scale rows of 4 ceil(K / 128) bytes at multiples of 4 bytes");
  const int es = f32_out ? 4 : 2;
  VPT_CHECK_ARG((ldo >= K || M == 1) && aligned(out, es), "vpt_mxfp4_dequantize: ldo >= K, out aligned to its type");
  const bool vec = K % 8 == 0 && aligned(out, 16) && ldo * es % 16 == 0;
  const unsigned nch = (unsigned)((K + 7) / 8);
  const long slab = (1L << 31) / nch;
  for (long r = 0; r < M; r += slab) {
    const long n = M - r < slab ? M - r : slab;
    const unsigned total = (unsigned)(n * nch);
    const uint8_t* cr = (const uint8_t*)codes + r * ldc;
    const uint8_t* sr = (const uint8_t*)scales + r * lds;
    void* o = (char*)out + r * ldo * es;
    const dim3 grid((total + 255u) / 256u), block(256);
    hipStream_t st = (hipStream_t)stream;
    if (f32_out && vec) hipLaunchKernelGGL((mx_dequantize_kernel<true, true>), grid, block, 0, st, cr, ldc, sr, lds, total, nch, K, o, ldo);
    else if (f32_out) hipLaunchKernelGGL((mx_dequantize_kernel<true, false>), grid, block, 0, st, cr, ldc, sr, lds, total, nch, K, o, ldo);
    else if (vec) hipLaunchKernelGGL((mx_dequantize_kernel<false, true>), grid, block, 0, st, cr, ldc, sr, lds, total, nch, K, o, ldo);
    else hipLaunchKernelGGL((mx_dequantize_kernel<false, false>), grid, block, 0, st, cr, ldc, sr, lds, total, nch, K, o, ldo);
    VPT_LAUNCH_CHECK();
  }
  return VPT_OK;
}

extern "C" int vpt_gemm_mxfp4(const void* a_codes, long lda, const void* a_scales, long ldas, const void* b_codes,
                              long ldb, const void* b_scales, long ldbs, void* C, long ldc, int M, int N, int K,
                              const void* bias, const void* resid, long ldr, int f32_out, void* stream) {
  VPT_CHECK_ARG(M >= 0 && N > 0 && K > 0 && K <= (1 << 30), "vpt_gemm_mxfp4: M >= 0, N > 0, 0 < K <= 2^30");
  if (M == 0) return VPT_OK;
  VPT_CHECK_ARG(a_codes && a_scales && b_codes && b_scales && C, "vpt_gemm_mxfp4: null pointer");
  const int steps = (K + 127) / 128;
  VPT_CHECK_ARG(lda >= 64L * steps && lda % 16 == 0 && aligned(a_codes, 16) && ldb >= 64L * steps && ldb % 16 == 0 &&
                    aligned(b_codes, 16),
                "vpt_gemm_mxfp4: code rows of 64 ceil(K / 128) bytes at multiples of 16 bytes");
  VPT_CHECK_ARG(ldas >= 4L * steps && ldas % 4 == 0 && aligned(a_scales, 4) && ldbs >= 4L * steps && ldbs % 4 == 0 &&
                    aligned(b_scales, 4),
                "vpt_gemm_mxfp4: scale rows of 4 ceil(K / 128) bytes at multiples of 4 bytes");
  VPT_CHECK_ARG((ldc >= N || M == 1) && aligned(C, f32_out ? 4 : 2), "vpt_gemm_mxfp4: ldc >= N, C aligned to its type");
  VPT_CHECK_ARG((!bias || aligned(bias, 2)) && (!resid || (aligned(resid, 2) && (ldr >= N || M == 1))),
                "vpt_gemm_mxfp4: bf16 bias and residual, ldr >= N");
  const long tiles = ((M + 127L) / 128) * ((N + 127L) / 128);
  VPT_CHECK_ARG(tiles < (1L << 31), "vpt_gemm_mxfp4: too many tiles");
  const MxArgs g{(const uint8_t*)a_codes, lda, (const uint8_t*)a_scales, ldas, (const uint8_t*)b_codes, ldb,
                 (const uint8_t*)b_scales, ldbs, C, ldc, (const bf16_t*)bias, (const bf16_t*)resid, ldr, M, N, steps, f32_out};
  hipLaunchKernelGGL(mx_gemm_kernel, dim3((unsigned)tiles), dim3(256), 0, (hipStream_t)stream, g);
  VPT_LAUNCH_CHECK();
  return VPT_OK;
}
