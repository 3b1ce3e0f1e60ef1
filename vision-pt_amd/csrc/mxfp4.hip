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

#include <type_traits>

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

// Eight codes of the values f under scale byte s: v_cvt_scalef32_pk_fp4_f32 rounds to the nearest code, ties to even, and
// saturates; the values are brought to the block's unit by an exact product first (s <= 252: the factor is a normal number).
__device__ __forceinline__ uint32_t mx_codes8(const float (&f)[8], uint32_t s) {
  if (s == 255u) return 0u;
  const float inv = __uint_as_float((254u - s) << 23);  // 2^(127 - s)
  uint32_t out = 0;
  out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, f[0] * inv, f[1] * inv, 1.f, 0);
  out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, f[2] * inv, f[3] * inv, 1.f, 1);
  out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, f[4] * inv, f[5] * inv, 1.f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, f[6] * inv, f[7] * inv, 1.f, 3);
}

// One thread per 8 values: four neighbouring lanes share a block, its largest magnitude by two DPP exchanges. Bound by HBM:
// 2 (or 4) bytes in, 17 / 32 out per value; 33360 x 2048 bf16 in 35 us, 4.9 TB/s (a 4-GB copy runs at 4.6).
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

// One thread per 8 values. VEC: K % 8 == 0 and 16-byte rows. Bound by HBM as the quantisation: 33360 x 2048 to bf16 in 34 us.
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

// ---- the tile product: TM x 128 tiles, 4 waves (2 x 2) of TM / 2 x 64, two blocks per CU -----------------------------
// The pipeline of the bf16 256x128 ring (gemm_r2.hip), whose stages hold the same bytes here: a 3-stage LDS ring of 128-deep
// K steps (64-byte rows of codes) filled by LDS-DMA two steps ahead with counted waits. Per step and wave TM / 64 + 2 pieces of
// 1 KB, TM / 32 + 4 fragment reads of 16 bytes and TM / 8 MFMAs.
// Scales: 16 bytes per row, those of 4 steps, in one piece of 16 bytes per lane (rows of 4 bytes per step cost as many cache
// accesses as the codes: 1.39x the time at 33360 x 4096 x 3840). They have one buffer: a wave takes its rows' bytes of all 4
// steps into registers at the first of them, and the next 4 steps' piece is fetched from the second on.
// The product is taken transposed, W's fragment first, so that a lane holds 4 consecutive columns of one output row; W's rows
// lie in LDS in an order (mx_wrow) that makes the columns of two fragments neighbours: 16-byte stores from registers.
// What bounds it: 1.27 us per step of a CU's two blocks, of which the MFMAs need 0.6 at the 7.0 PFLOP/s that the instruction
// reaches on random operands (9.8 on zeros). No unit is full: counters at 33360 x 4096 x 768 give MFMA busy 0.22, LDS reads
// 0.11 without bank conflicts, and waves that wait 0.39 of their time to issue and 0.29 for memory and barriers. Short
// reductions are bound by the stores: that product takes 101 us (105 to 114 with a bias), 67 without its 273 MB of
// stores, which as half lines past the cache write 398 MB. 17568 x 2304 x 768 34 us; 4224 x 1280 x 5120 (128-row
// tiles) 31 us, 36 with a residual: its loads wait behind the stores of the fragment before (17568 x 2304 x 768 with one 71,
// 33360 x 4096 x 768 198).
constexpr int MXST = 3;
template <int TM> constexpr int mx_stage() { return (TM + 128) * 64; }               // 24 / 16 KB
template <int TM> constexpr int mx_lds() { return MXST * mx_stage<TM>() + (TM + 128) * 16; }  // 78 / 52 KB

// Position p of a wave's 64 rows of W in LDS holds row mx_wrow(p): fragment j = p >> 4, row i = p & 15 of the MFMA operand;
// output rows 4 g + e of fragments 2 q, 2 q + 1 become columns 32 q + 8 g + 0 .. 7.
__device__ __forceinline__ int mx_wrow(int p) {
  return (p >> 5) * 32 + ((p >> 2) & 3) * 8 + ((p >> 4) & 1) * 4 + (p & 3);
}

struct MxOffs {  // loop-invariant per-lane byte offsets of a tile's pieces
  uint32_t a[4], b[2], as, bs;
};

template <int TM>
__device__ __forceinline__ void mx_issue(const MxArgs& g, const MxOffs& o, int m0, int n0, int t, uint32_t smem0, int wid) {
  const uint32_t st = smem0 + (uint32_t)(t % MXST) * mx_stage<TM>();
  const void* ab = uniform_ptr(g.A + (long)m0 * g.lda + t * 64);
  const void* bb = uniform_ptr(g.B + (long)n0 * g.ldb + t * 64);
  const uint32_t la = __builtin_amdgcn_readfirstlane(st + wid * (TM * 16));
  const uint32_t lb = __builtin_amdgcn_readfirstlane(st + TM * 64 + wid * 2048);
  if constexpr (TM == 256) {
    glds_step(ab, bb, o.a[0], o.a[1], o.b[0], o.b[1], la, la + 1024, lb, lb + 1024);
    glds16(ab, o.a[2], la + 2 * 1024);
    glds16(ab, o.a[3], la + 3 * 1024);
  } else {
    glds_step(ab, bb, o.a[0], o.a[1], o.b[0], o.b[1], la, la + 1024, lb, lb + 1024);
  }
}

// The scale bytes from `at` on, 16 per row (waves 2, 3 repeat what 0, 1 fetch of a 128-row operand: every wave counts alike).
template <int TM>
__device__ __forceinline__ void mx_issue_scales(const MxArgs& g, const MxOffs& o, int m0, int n0, int at, uint32_t smem0, int wid) {
  const uint32_t ls = smem0 + MXST * mx_stage<TM>();
  glds16(uniform_ptr(g.AS + (long)m0 * g.ldas + at), o.as,
         __builtin_amdgcn_readfirstlane(ls + (TM == 256 ? wid : wid & 1) * 1024));
  glds16(uniform_ptr(g.BS + (long)n0 * g.ldbs + at), o.bs, __builtin_amdgcn_readfirstlane(ls + TM * 16 + (wid & 1) * 1024));
}

// The scale bytes of block blk in the 4 steps whose 16 bytes lie at p: byte s of the result is step s's. `first` > 0: the steps
// are the last 4 - first of the row, at the end of the 16 bytes.
__device__ __forceinline__ uint32_t mx_scale4(const char* p, uint32_t sel_lo, uint32_t sel_hi, int first) {
  const uint4 d = *reinterpret_cast<const uint4*>(p);
  return (__builtin_amdgcn_perm(d.y, d.x, sel_lo) | __builtin_amdgcn_perm(d.w, d.z, sel_hi)) >> (8 * first);
}

template <int S>
__device__ __forceinline__ floatx4 mx_mfma_at(uint4 a, uint4 b, floatx4 c, uint32_t sa, uint32_t sb) {  // scale byte S
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_frag(a), mx_frag(b), c, 4, 4, S, (int)sa, S, (int)sb);
}

// acc[i][j][e]: row 16 i + (lane & 15), column 32 (j >> 1) + 8 (lane >> 4) + 4 (j & 1) + e of the wave's tile, which starts at
// (row0, col0) of the block's at (m0, n0). VEC (N % 8 == 0, 16-byte rows): 16-byte buffer stores whose per-store part is one
// scalar; rows past M lie behind the buffer's end, columns past N get an offset there, and the hardware drops them (the
// tests frame results of every kernel by more rows than a tile has, with last tiles of 4 and 8 rows). Otherwise element by
// element.
template <bool VEC, int AUX, int MI, int NP>
__device__ __forceinline__ void mx_epilogue(const MxArgs& g, const floatx4 (&acc)[MI][2 * NP], int lane, int m0, int n0, int row0,
                                            int col0, const float (&bias)[NP][8]) {
  const int lr = row0 + (lane & 15), lc = col0 + (lane >> 4) * 8;
  if (VEC) {
    const int es = g.f32out ? 4 : 2, rows_here = min(256, g.M - m0);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (char*)g.C + ((long)m0 * g.ldc + n0) * es, (short)0, rows_here * (int)g.ldc * es, 0x00020000);
    const bf16_t* rbase = g.resid ? g.resid + (long)m0 * g.ldr + n0 : nullptr;
    const __amdgpu_buffer_rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)rbase, (short)0, g.resid ? rows_here * (int)g.ldr * 2 : 0, 0x00020000);
    uint32_t vo[NP], vr[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const bool in = n0 + lc + q * 32 < g.N;
      vo[q] = in ? (uint32_t)((lr * (int)g.ldc + lc + q * 32) * es) : 0x80000000u;
      vr[q] = in ? (uint32_t)((lr * (int)g.ldr + lc + q * 32) * 2) : 0x80000000u;
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      u32x4 res[NP];
      if (g.resid) {
#pragma unroll
        for (int q = 0; q < NP; ++q) res[q] = __builtin_amdgcn_raw_buffer_load_b128(rr, (int)vr[q], i * 32 * (int)g.ldr, 0);
      }
      const int so = i * 16 * (int)g.ldc * es;
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = acc[i][2 * q + (e >> 2)][e & 3] + bias[q][e];
        if (g.resid) {
          float rv[8];
          unpack8(make_uint4(res[q][0], res[q][1], res[q][2], res[q][3]), rv);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] += rv[e];
        }
        if (g.f32out) {
          store_b128_padded<AUX>(u32x4{__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])},
                                 rs, (int)vo[q], so);
          store_b128_padded<AUX>(u32x4{__float_as_uint(o[4]), __float_as_uint(o[5]), __float_as_uint(o[6]), __float_as_uint(o[7])},
                                 rs, (int)vo[q], so + 16);
        } else {
          const uint4 w = pack8(o);
          store_b128_padded<AUX>(u32x4{w.x, w.y, w.z, w.w}, rs, (int)vo[q], so);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int row = m0 + lr + i * 16;
    if (row >= g.M) continue;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = n0 + lc + q * 32 + e;
        if (col >= g.N) break;
        float o = acc[i][2 * q + (e >> 2)][e & 3] + bias[q][e];
        if (g.resid) o += bf2f(g.resid[(long)row * g.ldr + col]);
        if (g.f32out) reinterpret_cast<float*>(g.C)[(long)row * g.ldc + col] = o;
        else reinterpret_cast<bf16_t*>(g.C)[(long)row * g.ldc + col] = f2bf(o);
      }
  }
}

// The bias of a lane's columns c0 .. c0 + 7 and 32 on, in registers before the first DMA (a later wait for these loads would
// drain the ring). 16-byte loads where the bias lies so: value by value they cost 12 us of 33360 x 4096 x 768,
// by LDS-DMA with the first pieces as much as this.
template <bool VEC>
__device__ __forceinline__ void mx_bias(const MxArgs& g, int c0, float (&bias)[2][8]) {
  const bool vec = VEC && ((uintptr_t)g.bias & 15) == 0;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int c = c0 + q * 32;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (vec && g.bias && c < g.N) v = *reinterpret_cast<const uint4*>(g.bias + c);
    unpack8(v, bias[q]);
    if (!vec)
#pragma unroll
      for (int e = 0; e < 8; ++e) bias[q][e] = g.bias && c + e < g.N ? bf2f(g.bias[c + e]) : 0.f;
  }
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(bias[q][e]));
}

template <int TM, bool VEC, int AUX>
__global__ __launch_bounds__(256, 2) void mx_tile_kernel(MxArgs g) {
  constexpr int MI = TM / 32, STG = mx_stage<TM>(), PCS = TM / 64 + 2;
  static_assert(PCS == 6 || PCS == 4, "the counted waits below");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid >> 1, wn = wid & 1;
  const int tiles_n = (g.N + 127) / 128, items = (g.M + TM - 1) / TM * tiles_n;
  // XCD-contiguous order: the dispatcher deals block ids round-robin to the 8 XCDs, each of which runs one range of tiles
  const int q8 = items >> 3, r8 = items & 7, xcd = blockIdx.x & 7;
  const int tile = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
  const int m0 = tile / tiles_n * TM, n0 = tile % tiles_n * 128;
  const uint32_t smem0 = (uint32_t)(uintptr_t)(VPT_LDS char*)smem;
  const int nk = g.steps, r = lane & 15, blk = lane >> 4;
  // v_perm selectors: byte blk of one dword into byte 0 (2), of the next into byte 1 (3), zeros elsewhere
  const uint32_t sel_lo = 0x0c0c0400u + blk * 0x0101u, sel_hi = 0x04000c0cu + blk * 0x01010000u;
  MxOffs o;  // rows past the edge: the last one (its results are not stored)
#pragma unroll
  for (int i = 0; i < TM / 64; ++i) o.a[i] = tile_voff<true, TM, 4>(g.lda >> 1, m0, g.M, RBK, wid, lane, i);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = (wid * 2 + i) * 16 + (lane >> 2), row = (p & 64) | mx_wrow(p & 63);
    o.b[i] = (uint32_t)(min(row, g.N - 1 - n0) * (int)g.ldb + ((lane & 3) ^ (((p >> 2) & 1) << 1)) * 16);
  }
  o.as = (uint32_t)(min((TM == 256 ? wid : wid & 1) * 64 + lane, g.M - 1 - m0) * (int)g.ldas);
  o.bs = (uint32_t)(min((wid & 1) * 64 + mx_wrow(lane), g.N - 1 - n0) * (int)g.ldbs);

  float bias[2][8];
  mx_bias<VEC>(g, n0 + wn * 64 + blk * 8, bias);
  uint32_t sa[MI], sb[4];
#pragma unroll
  for (int i = 0; i < MI; ++i) sa[i] = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) sb[j] = 0;
  if (nk < 4) {  // no 16 bytes of scales in a row: straight into registers
    for (int t = 0; t < nk; ++t) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
        sa[i] |= (uint32_t)g.AS[(long)min(m0 + wm * (TM / 2) + i * 16 + r, g.M - 1) * g.ldas + t * 4 + blk] << (8 * t);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sb[j] |= (uint32_t)g.BS[(long)min(n0 + wn * 64 + mx_wrow(j * 16 + r), g.N - 1) * g.ldbs + t * 4 + blk] << (8 * t);
    }
  }
  floatx4 acc[MI][4];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  if (nk >= 4) mx_issue_scales<TM>(g, o, m0, n0, 0, smem0, wid);
  mx_issue<TM>(g, o, m0, n0, 0, smem0, wid);
  if (nk > 1) {
    mx_issue<TM>(g, o, m0, n0, 1, smem0, wid);
    if constexpr (PCS == 6) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  __syncthreads();

  // Step kt = 4 c + S.
  auto step = [&](int kt, auto S_) {
    constexpr int S = decltype(S_)::value;
    // the next 4 steps' scales: the buffer was read at step 4 c; a last group of fewer than 4 ends with the row
    const bool fetch = S == 1 && kt + 3 < nk;
    if (fetch) mx_issue_scales<TM>(g, o, m0, n0, min(4 * (kt + 3), 4 * nk - 16), smem0, wid);
    // step kt + 2 into the stage of step kt - 1, which every wave finished reading before the last barrier
    if (kt + 2 < nk) mx_issue<TM>(g, o, m0, n0, kt + 2, smem0, wid);
    const char* st = smem + (kt % MXST) * STG;
    if (S == 0 && nk >= 4) {
      const char* sc = smem + MXST * STG;
      const int rem = nk - kt, first = rem < 4 ? 4 - rem : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sb[j] = mx_scale4(sc + TM * 16 + (wn * 64 + j * 16 + r) * 16, sel_lo, sel_hi, first);
#pragma unroll
      for (int i = 0; i < MI; ++i) sa[i] = mx_scale4(sc + (wm * (TM / 2) + i * 16 + r) * 16, sel_lo, sel_hi, first);
    }
    uint4 af[MI], bf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      bf[j] = *reinterpret_cast<const uint4*>(st + TM * 64 + kmaj32_off(wn * 64 + j * 16 + r, blk));
#pragma unroll
    for (int i = 0; i < MI; ++i) af[i] = *reinterpret_cast<const uint4*>(st + kmaj32_off(wm * (TM / 2) + i * 16 + r, blk));
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mx_mfma_at<S>(bf[j], af[i], acc[i][j], sb[j], sa[i]);
    __builtin_amdgcn_s_setprio(0);
    if (kt + 1 < nk) {
      // this wave's pieces of step kt + 1 landed (those of step kt + 2, and scales issued with them, may still fly), then
      // every wave's
      if (kt + 2 >= nk) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      } else if (fetch) {
        if constexpr (PCS == 6) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
      } else {
        if constexpr (PCS == 6) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      }
      __syncthreads();
    }
  };
  for (int kt = 0; kt < nk; kt += 4) {
    step(kt, std::integral_constant<int, 0>{});
    if (kt + 1 < nk) step(kt + 1, std::integral_constant<int, 1>{});
    if (kt + 2 < nk) step(kt + 2, std::integral_constant<int, 2>{});
    if (kt + 3 < nk) step(kt + 3, std::integral_constant<int, 3>{});
  }
  mx_epilogue<VEC, AUX, MI, 2>(g, acc, lane, m0, n0, wm * (TM / 2), wn * 64, bias);
}

// ---- large products: 256 x 256 tiles, 8 waves (2 x 4) of 128 x 64, one block per CU -----------------------------------
// The same wave tile as the 256 x 128 form with two thirds of its LDS-DMA per product, four stages (three steps ahead), and the
// phases of the bf16 256x256 ring (gemm.hip): waves 4-7 run one barrier behind waves 0-3, so that on every SIMD one wave
// multiplies while the other reads its fragments.
//   L_t: DMA of step t + 3 into the stage of step t - 1; fragments of step t into registers; this wave's pieces of step
//        t + 1 have landed; barrier      C_t: 32 MFMAs; barrier
// A stage is refilled in L_t, after both groups' L_t-1 closed with lgkmcnt(0) and a barrier; a step's pieces of all waves have
// landed one barrier before the first group reads them. The scales' buffer (one, 16 bytes per row) is read in L_4c and
// refilled from L_4c+1 on; its piece has landed where step 4c + 4's are waited for.
// 1.02 us per step: 8192^3 in 286 to 307 us, 3.6 to 3.8 PFLOP/s, MFMA busy 0.48, LDS reads 0.23. Wider waves (four of 128 x 128, a third less LDS reading, fragments a step
// ahead in registers) took 1.16: one wave per SIMD leaves its waits uncovered.
constexpr int MXR_ST = 4, MXR_STG = 512 * 64;
constexpr int mx_ring_lds() { return MXR_ST * MXR_STG + 512 * 16; }  // 136 KB

__device__ __forceinline__ void mxr_issue(const MxArgs& g, const uint32_t (&va)[2], const uint32_t (&vb)[2], int m0, int n0, int t,
                                          uint32_t smem0, int wid) {
  const uint32_t la = __builtin_amdgcn_readfirstlane(smem0 + (uint32_t)(t % MXR_ST) * MXR_STG + wid * 2048);
  glds_step(uniform_ptr(g.A + (long)m0 * g.lda + t * 64), uniform_ptr(g.B + (long)n0 * g.ldb + t * 64), va[0], va[1], vb[0],
            vb[1], la, la + 1024, la + 16384, la + 16384 + 1024);
}

template <bool VEC, int AUX>
__global__ __launch_bounds__(512, 1) void mx_ring_kernel(MxArgs g) {
  constexpr int MI = 8;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wid >> 2, wn = wid & 3;
  const int tiles_n = (g.N + 255) / 256, items = (g.M + 255) / 256 * tiles_n;
  const int q8 = items >> 3, r8 = items & 7, xcd = blockIdx.x & 7;
  const int tile = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
  const int m0 = tile / tiles_n * 256, n0 = tile % tiles_n * 256;
  const uint32_t smem0 = (uint32_t)(uintptr_t)(VPT_LDS char*)smem;
  const int nk = g.steps, r = lane & 15, blk = lane >> 4;
  // v_perm selectors: byte blk of one dword into byte 0 (2), of the next into byte 1 (3), zeros elsewhere
  const uint32_t sel_lo = 0x0c0c0400u + blk * 0x0101u, sel_hi = 0x04000c0cu + blk * 0x01010000u;
  uint32_t va[2], vb[2];  // rows past the edge: the last one (its results are not stored)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    va[i] = tile_voff<true, 256, 8>(g.lda >> 1, m0, g.M, RBK, wid, lane, i);
    const int p = (wid * 2 + i) * 16 + (lane >> 2), row = (p & ~63) | mx_wrow(p & 63);
    vb[i] = (uint32_t)(min(row, g.N - 1 - n0) * (int)g.ldb + ((lane & 3) ^ (((p >> 2) & 1) << 1)) * 16);
  }
  // scales: waves 0-3 fetch A's rows, 4-7 B's
  const uint32_t vs = wid < 4 ? (uint32_t)(min(wid * 64 + lane, g.M - 1 - m0) * (int)g.ldas)
                              : (uint32_t)(min((wid - 4) * 64 + mx_wrow(lane), g.N - 1 - n0) * (int)g.ldbs);
  const uint8_t* sbase = wid < 4 ? g.AS + (long)m0 * g.ldas : g.BS + (long)n0 * g.ldbs;
  const uint32_t ls = __builtin_amdgcn_readfirstlane(smem0 + MXR_ST * MXR_STG + wid * 1024);

  float bias[2][8];
  mx_bias<VEC>(g, n0 + wn * 64 + blk * 8, bias);
  uint32_t sa[MI], sb[4];
  glds16(uniform_ptr(sbase), vs, ls);  // the host takes this kernel for 24 steps and more: every row has 16 bytes of scales
  floatx4 acc[MI][4];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  for (int t = 0; t < 3; ++t) mxr_issue(g, va, vb, m0, n0, t, smem0, wid);
  wait_younger(2);  // step 0 and the scales landed: the two younger steps' 4 pieces each may fly
  raw_barrier();
  if (wid >= 4) bare_barrier();

  auto step = [&](int kt, auto S_) {
    constexpr int S = decltype(S_)::value;
    const bool fetch = S == 1 && kt + 3 < nk;  // a last group of fewer than 4 steps' scales ends with the row
    if (fetch) glds16(uniform_ptr(sbase + min(4 * (kt + 3), 4 * nk - 16)), vs, ls);
    if (kt + 3 < nk) mxr_issue(g, va, vb, m0, n0, kt + 3, smem0, wid);
    const char* st = smem + (kt % MXR_ST) * MXR_STG;
    if (S == 0) {
      const char* sc = smem + MXR_ST * MXR_STG;
      const int rem = nk - kt, first = rem < 4 ? 4 - rem : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sb[j] = mx_scale4(sc + 4096 + (wn * 64 + j * 16 + r) * 16, sel_lo, sel_hi, first);
#pragma unroll
      for (int i = 0; i < MI; ++i) sa[i] = mx_scale4(sc + (wm * 128 + i * 16 + r) * 16, sel_lo, sel_hi, first);
    }
    uint4 af[MI], bf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) bf[j] = *reinterpret_cast<const uint4*>(st + 16384 + kmaj32_off(wn * 64 + j * 16 + r, blk));
#pragma unroll
    for (int i = 0; i < MI; ++i) af[i] = *reinterpret_cast<const uint4*>(st + kmaj32_off(wm * 128 + i * 16 + r, blk));
    // this wave's pieces of step kt + 1 landed; steps kt + 2, kt + 3 (4 pieces each) and a scale piece issued at S = 1 fly
    const bool scale_flies = (S == 1 && fetch) || (S == 2 && kt + 2 < nk);
    if (kt + 3 < nk) {
      if (scale_flies) asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else if (kt + 2 < nk) {
      if (scale_flies) asm volatile("s_waitcnt vmcnt(5)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    raw_barrier();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mx_mfma_at<S>(bf[j], af[i], acc[i][j], sb[j], sa[i]);
    __builtin_amdgcn_s_setprio(0);
    bare_barrier();
  };
  for (int kt = 0; kt < nk; kt += 4) {
    step(kt, std::integral_constant<int, 0>{});
    if (kt + 1 < nk) step(kt + 1, std::integral_constant<int, 1>{});
    if (kt + 2 < nk) step(kt + 2, std::integral_constant<int, 2>{});
    if (kt + 3 < nk) step(kt + 3, std::integral_constant<int, 3>{});
  }
  if (wid < 4) bare_barrier();
  mx_epilogue<VEC, AUX, MI, 2>(g, acc, lane, m0, n0, wm * 128, wn * 64, bias);
}

// ---- few rows: 16 MI rows x 16 columns per block, its 4 waves share the steps along K --------------------------------
// With few rows the product is a pass over W: each wave takes every fourth 128-deep step, its 16 rows of W straight from
// memory into registers (four steps' loads in flight), and the four partial sums meet in LDS in a fixed order. FUSE: the block
// quantises its rows of x itself, into LDS (M <= 16; the same codes as mx_quantize_kernel), and saves a launch. One row
// of 2304 x 768: 2.5 us in a graph; of 10240 x 5120: 10 us, 2.8 TB/s of codes, its waves waiting for memory 0.68 of their
// time with few loads in flight, each of half a line of its row (8 loads instead of 4 per wave, or the first ones before x is
// quantised, were slower).
struct MxX {
  const void* x; long ldx;
  int K;
};
constexpr int kMxSkinnyLoads = 4;

template <int MI, int FUSE, bool XVEC>  // FUSE: 0 no, else 1 + the type of x
__global__ __launch_bounds__(256) void mx_skinny_kernel(MxArgs g, MxX x) {
  __shared__ float red[4][16 * MI][17];
  extern __shared__ __attribute__((aligned(16))) char smem[];  // FUSE: codes [M][64 steps + 16], scales [M][4 steps]
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * MI);
  const int pitch = 64 * g.steps + 16;
  char* lscale = smem + (long)g.M * pitch;
  const int r = lane & 15, blk = lane >> 4;
  const long wrow = min(n0 + r, g.N - 1);  // rows past the edge: the last one (its results are not stored)
  const uint8_t* wb = g.B + wrow * g.ldb + blk * 16;
  const uint8_t* ws = g.BS + wrow * g.ldbs + blk;
  uint4 bf[kMxSkinnyLoads];
  uint32_t sb[kMxSkinnyLoads];
  auto load_w = [&](int t0) {
#pragma unroll
    for (int u = 0; u < kMxSkinnyLoads; ++u) {
      const int t = t0 + 4 * u;  // wave-uniform
      if (t >= g.steps) break;
      bf[u] = *reinterpret_cast<const uint4*>(wb + (long)t * 64);
      sb[u] = ws[(long)t * 4];
    }
  };
  if (FUSE) {
    const int nch = 16 * g.steps, total = g.M * nch;
    for (int idx = tid; idx < total; idx += 256) {  // total % 16 == 0: the four lanes of a block stay together
      const int row = idx / nch, c = idx - row * nch;
      float f[8];
      mx_load8<FUSE - 1, XVEC>(x.x, (long)row * x.ldx + c * 8, c * 8, x.K, f);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
      top = max(top, dpp_xor1(top));
      top = max(top, dpp_xor2(top));
      const uint32_t sc = mx_scale(top);
      *reinterpret_cast<uint32_t*>(smem + row * pitch + c * 4) = mx_codes8(f, sc);
      if ((c & 3) == 0) lscale[row * 4 * g.steps + (c >> 2)] = (char)sc;
    }
    __syncthreads();
  }
  const uint8_t* ab[MI];
  const uint8_t* as[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const long row = min(m0 + i * 16 + r, g.M - 1);
    ab[i] = FUSE ? (const uint8_t*)smem + row * pitch + blk * 16 : g.A + row * g.lda + blk * 16;
    as[i] = FUSE ? (const uint8_t*)lscale + row * 4 * g.steps + blk : g.AS + row * g.ldas + blk;
  }
  floatx4 acc[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int t0 = wid; t0 < g.steps; t0 += 4 * kMxSkinnyLoads) {
    load_w(t0);
#pragma unroll
    for (int u = 0; u < kMxSkinnyLoads; ++u) {
      const int t = t0 + 4 * u;  // wave-uniform
      if (t >= g.steps) break;
#pragma unroll
      for (int i = 0; i < MI; ++i)
        acc[i] = mx_mfma(*reinterpret_cast<const uint4*>(ab[i] + (long)t * 64), bf[u], acc[i], as[i][(long)t * 4], sb[u]);
    }
  }
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) red[wid][i * 16 + blk * 4 + q][r] = acc[i][q];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int lr = i * 16 + (tid >> 4), c = tid & 15, m = m0 + lr, n = n0 + c;
    if (m >= g.M || n >= g.N) continue;
    float v = (red[0][lr][c] + red[1][lr][c]) + (red[2][lr][c] + red[3][lr][c]);
    if (g.bias) v += bf2f(g.bias[n]);
    if (g.resid) v += bf2f(g.resid[(long)m * g.ldr + n]);
    if (g.f32out) reinterpret_cast<float*>(g.C)[(long)m * g.ldc + n] = v;
    else reinterpret_cast<bf16_t*>(g.C)[(long)m * g.ldc + n] = f2bf(v);
  }
}

// Rows too far apart for the tile kernels' 32-bit offsets: 128 x 128 tile, 4 waves of 64 x 64, one 128-deep step at a time
// through LDS with 64-bit addresses (505 us where the tile kernels take 112 for x, quantised, of 33360 x 4096 x 768).
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

// W, the output, bias and residual of a product.
int mx_check_product(const void* b_codes, long ldb, const void* b_scales, long ldbs, const void* C, long ldc, int M, int N, int K,
                     const void* bias, const void* resid, long ldr, int f32_out) {
  const long steps = (K + 127) / 128;
  VPT_CHECK_ARG(b_codes && b_scales && C, "mxfp4 product: null pointer");
  VPT_CHECK_ARG(ldb >= 64 * steps && ldb % 16 == 0 && aligned(b_codes, 16),
                "mxfp4 product: code rows of 64 ceil(K / 128) bytes at multiples of 16 bytes");
  VPT_CHECK_ARG(ldbs >= 4 * steps && ldbs % 4 == 0 && aligned(b_scales, 4),
                "mxfp4 product: scale rows of 4 ceil(K / 128) bytes at multiples of 4 bytes");
  VPT_CHECK_ARG((ldc >= N || M == 1) && aligned(C, f32_out ? 4 : 2), "mxfp4 product: output rows of N values, aligned to their type");
  VPT_CHECK_ARG((!bias || aligned(bias, 2)) && (!resid || (aligned(resid, 2) && (ldr >= N || M == 1))),
                "mxfp4 product: bf16 bias and residual, rows of N values");
  VPT_CHECK_ARG(((M + 127L) / 128) * ((N + 127L) / 128) < (1L << 24), "mxfp4 product: too many tiles");  // a grid has under 2^32 threads
  return VPT_OK;
}

// Cache policy of the tile kernels' 16-byte stores (buffer instruction aux bits): sc1 (16: the line leaves the XCD's L2, which
// the weight's rows keep) where the output fits the 256-MB cache, nt (2) where it does not. Measured (default / sc1 / nt):
// 17568 x 2304 x 768 32.0 / 30.2 / 34.7 us, 24000 x 5120 x 768 (246 MB) - / 88.7 / 93.5, 33360 x 4096 x 768 (273 MB)
// 124 / 109 / 93, 33360 x 4096 x 1536 - / 202 / 147.
constexpr int kMxKeep = 16, kMxStream = 2;
constexpr int kMxRingSteps = 24;  // mx_ring_kernel takes at least 4

template <int MI>
void mx_skinny_launch(const MxArgs& g, hipStream_t s) {
  hipLaunchKernelGGL((mx_skinny_kernel<MI, 0, false>), dim3((g.N + 15) / 16, (g.M + 16 * MI - 1) / (16 * MI)), dim3(256), 0, s, g,
                     MxX{nullptr, 0, 0});
}

// The product of checked arguments.
void mx_product(const MxArgs& g, hipStream_t st) {
  const long tiles = ((g.M + 127L) / 128) * ((g.N + 127L) / 128);
  // Few rows: also while blocks of 64 rows x 16 columns do not outnumber the CUs (65 x 1280 x 5120 13.6 us against 19.8 of the
  // 128 x 128 tiles, 192 rows 13.9 : 20.1, 256 rows, 320 blocks, 24.6 : 20.3; 384 x 640 x 2048 7.7 : 10.2, 512 rows 11.6 : 10.2).
  if (g.M <= 64 || ((g.M + 63L) / 64) * ((g.N + 15L) / 16) <= 256) {
    if (g.M <= 16) mx_skinny_launch<1>(g, st);
    else if (g.M <= 32) mx_skinny_launch<2>(g, st);
    else mx_skinny_launch<4>(g, st);
    return;
  }
  // the tile kernels keep 32-bit offsets within a tile of at most 256 rows
  const long es = g.f32out ? 4 : 2, far = 1L << 22;
  if (g.lda >= far || g.ldb >= far || g.ldas >= far || g.ldbs >= far || g.ldc * es >= far || (g.resid && g.ldr * 2 >= far)) {
    hipLaunchKernelGGL(mx_gemm_kernel, dim3((unsigned)tiles), dim3(256), 0, st, g);
    return;
  }
  const bool vec = g.N % 8 == 0 && aligned(g.C, 16) && g.ldc * es % 16 == 0 &&
                   (!g.resid || (aligned(g.resid, 16) && g.ldr % 8 == 0));
  const bool stream = (long)g.M * g.N * es >= 256L << 20;
  const long tiles256 = ((g.M + 255L) / 256) * ((g.N + 127L) / 128), tiles2 = ((g.M + 255L) / 256) * ((g.N + 255L) / 256);
  // A step of a round of 256 x 256 tiles (one per CU) takes 1.02 us, of 256 x 128 tiles (two per CU) 1.27 us, whose blocks
  // overlap their ends and waste less of a last round; short reductions are ends for the most part. Measured, 256 x 256 :
  // 256 x 128: 4096^3 38.5 : 44.1 us, 8448 x 1280 x 5120 40.4 : 48.6, 33360 x 4096 x 3840 316 : 353, 8192^3 294 : 335; but
  // 16384 x 1280 x 5120 (1.25 rounds) 82.8 : 76.8, 16384 x 2560 x 2560 74.5 : 68.7, 33360 x 4096 x 768 116 : 93.
  const long rounds = (tiles2 + 255) / 256;
  if (g.steps >= kMxRingSteps && tiles2 > 128 && rounds * 102 < tiles2 * 127 / 256 + 20) {
    const dim3 grid((unsigned)tiles2);
    if (!vec) hipLaunchKernelGGL((mx_ring_kernel<false, 0>), grid, dim3(512), mx_ring_lds(), st, g);
    else if (stream) hipLaunchKernelGGL((mx_ring_kernel<true, kMxStream>), grid, dim3(512), mx_ring_lds(), st, g);
    else hipLaunchKernelGGL((mx_ring_kernel<true, kMxKeep>), grid, dim3(512), mx_ring_lds(), st, g);
  } else if (tiles256 >= 768) {  // 1.5 rounds. 256 : 128 rows per tile: 33360 x 768 x 2048 (786) 40.4 : 42.7 us, 17568 x 2304 x
                                 // 768 30.2 : 32.0; 8440 x 4096 x 768 29.7 : 27.7, 4224 x 1280 x 5120 (170) 30.5 : 29.4
    const dim3 grid((unsigned)tiles256);
    if (!vec) hipLaunchKernelGGL((mx_tile_kernel<256, false, 0>), grid, dim3(256), mx_lds<256>(), st, g);
    else if (stream) hipLaunchKernelGGL((mx_tile_kernel<256, true, kMxStream>), grid, dim3(256), mx_lds<256>(), st, g);
    else hipLaunchKernelGGL((mx_tile_kernel<256, true, kMxKeep>), grid, dim3(256), mx_lds<256>(), st, g);
  } else {
    const dim3 grid((unsigned)tiles);
    if (!vec) hipLaunchKernelGGL((mx_tile_kernel<128, false, 0>), grid, dim3(256), mx_lds<128>(), st, g);
    else hipLaunchKernelGGL((mx_tile_kernel<128, true, kMxKeep>), grid, dim3(256), mx_lds<128>(), st, g);
  }
}

// LDS of the fused form, 0 where it is not taken: up to 16384 values of x, which every block quantises anew. Fused : two
// launches, in a graph, K x M (N = 2304): 768 x 1 2.5 : 4.0 us, 768 x 16 4.5 : 4.5, 2048 x 8 5.9 : 5.4, 2048 x 16 8.9 : 5.8,
// 5120 x 2 6.0 : 7.2, 5120 x 4 7.9 : 7.4 (outside a graph the second launch costs about 4 us of the host more).
size_t mx_fused_lds(long M, int K) {
  const long steps = (K + 127) / 128;
  return M <= 16 && M * steps <= 128 ? (size_t)(M * (68 * steps + 16)) : 0;
}

template <int T>
void mx_fused_launch(const MxArgs& g, const MxX& x, bool vec, size_t lds, hipStream_t s) {
  const dim3 grid((g.N + 15) / 16, 1);
  if (vec) hipLaunchKernelGGL((mx_skinny_kernel<1, T + 1, true>), grid, dim3(256), lds, s, g, x);
  else hipLaunchKernelGGL((mx_skinny_kernel<1, T + 1, false>), grid, dim3(256), lds, s, g, x);
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
  VPT_CHECK_ARG(M >= 0 && M <= (1 << 30) && N > 0 && N <= (1 << 27) && K > 0 && K <= (1 << 30), "vpt_gemm_mxfp4: 0 <= M <= 2^30, 0 < N <= 2^27, 0 < K <= 2^30");
  if (M == 0) return VPT_OK;
  const int steps = (K + 127) / 128;
  VPT_CHECK_ARG(a_codes && a_scales, "vpt_gemm_mxfp4: null pointer");
  VPT_CHECK_ARG(lda >= 64L * steps && lda % 16 == 0 && aligned(a_codes, 16),
                "vpt_gemm_mxfp4: code rows of 64 ceil(K / 128) bytes at multiples of 16 bytes");
  VPT_CHECK_ARG(ldas >= 4L * steps && ldas % 4 == 0 && aligned(a_scales, 4),
                "vpt_gemm_mxfp4: scale rows of 4 ceil(K / 128) bytes at multiples of 4 bytes");
  const int rc = mx_check_product(b_codes, ldb, b_scales, ldbs, C, ldc, M, N, K, bias, resid, ldr, f32_out);
  if (rc) return rc;
  const MxArgs g{(const uint8_t*)a_codes, lda, (const uint8_t*)a_scales, ldas, (const uint8_t*)b_codes, ldb,
                 (const uint8_t*)b_scales, ldbs, C, ldc, (const bf16_t*)bias, (const bf16_t*)resid, ldr, M, N, steps, f32_out};
  mx_product(g, (hipStream_t)stream);
  VPT_LAUNCH_CHECK();
  return VPT_OK;
}

extern "C" long vpt_linear_mxfp4_workspace(int M, int K) {
  if (M <= 0 || K <= 0 || K > (1 << 30) || mx_fused_lds(M, K)) return 0;
  return M * 68L * ((K + 127) / 128);
}

extern "C" int vpt_linear_mxfp4(const void* x, int dtype, long ldx, const void* w_codes, long ldw, const void* w_scales,
                                long ldws, void* y, long ldy, int M, int N, int K, const void* bias, const void* resid, long ldr,
                                int f32_out, void* workspace, void* stream) {
  VPT_CHECK_ARG(dtype >= MX_BF16 && dtype <= MX_F16, "vpt_linear_mxfp4: dtype 0 bf16, 1 f32, 2 f16");
  VPT_CHECK_ARG(M >= 0 && M <= (1 << 30) && N > 0 && N <= (1 << 27) && K > 0 && K <= (1 << 30), "vpt_linear_mxfp4: 0 <= M <= 2^30, 0 < N <= 2^27, 0 < K <= 2^30");
  if (M == 0) return VPT_OK;
  const int es = dtype == MX_F32 ? 4 : 2;
  VPT_CHECK_ARG(x && aligned(x, es) && (ldx >= K || M == 1), "vpt_linear_mxfp4: x aligned to its type, ldx >= K");
  const long steps = (K + 127) / 128;
  const int rc = mx_check_product(w_codes, ldw, w_scales, ldws, y, ldy, M, N, K, bias, resid, ldr, f32_out);
  if (rc) return rc;
  const size_t lds = mx_fused_lds(M, K);
  uint8_t* codes = (uint8_t*)workspace;
  uint8_t* scales = codes + M * 64L * steps;
  if (!lds) {
    VPT_CHECK_ARG(workspace && aligned(workspace, 16), "vpt_linear_mxfp4: workspace of vpt_linear_mxfp4_workspace bytes");
    const int qrc = vpt_mxfp4_quantize(x, dtype, ldx, M, K, codes, 64 * steps, scales, 4 * steps, stream);
    if (qrc) return qrc;
    return vpt_gemm_mxfp4(codes, 64 * steps, scales, 4 * steps, w_codes, ldw, w_scales, ldws, y, ldy, M, N, K, bias, resid, ldr,
                          f32_out, stream);
  }
  const MxArgs g{nullptr, 0, nullptr, 0, (const uint8_t*)w_codes, ldw, (const uint8_t*)w_scales, ldws, y, ldy,
                 (const bf16_t*)bias, (const bf16_t*)resid, ldr, M, N, (int)steps, f32_out};
  const MxX xx{x, ldx, K};
  const bool vec = K % 8 == 0 && aligned(x, 16) && (M == 1 || ldx * es % 16 == 0);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MX_BF16) mx_fused_launch<MX_BF16>(g, xx, vec, lds, st);
  else if (dtype == MX_F32) mx_fused_launch<MX_F32>(g, xx, vec, lds, st);
  else mx_fused_launch<MX_F16>(g, xx, vec, lds, st);
  VPT_LAUNCH_CHECK();
  return VPT_OK;
}
