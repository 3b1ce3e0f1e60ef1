// The end of a gated transformer block and the norm of the next one, fused, forward and backward, for gfx950.
//
//   u  = h r_h w_post,  r_h = rsqrt(mean h^2 + eps)      (the norm behind the block; u = h without w_post)
//   x' = x + s gate u                                    (gate: one vector, one per group of rows, or none)
//   n  = x' r_x,        r_x = rsqrt(mean x'^2 + eps)     (the next block's norm, of x' as it is stored)
//   y  = n w_pre (1 + scale) + shift                     (modulation: one vector, one per group of rows, or none)
// Backward, from dy and the gradient dx' that the stream brings from later blocks:
//   dn = dy (1 + scale) w_pre,  dX = dx' + r_x (dn - n mean(dn n)),  dx = dX
//   v  = h r_h,  du = s gate dX,  dv = du w_post,  dh = r_h (dv - v mean(dv v))
// and, per group, the column sums S = sum dy, P = sum dy n, Q = sum dX v, from which
//   dshift = S, dscale = w_pre P, dw_pre = sum over groups (1 + scale) P,
//   dgate = s w_post Q, dw_post = s sum over groups gate Q.
// Beside RMSNorm (norm.hip; FP32RMSNorm, reference src/modules/norm.py:20-27), which has neither gate nor modulation.
//
// Both directions are bound by HBM: h, x, x', y once each forward; dy, dx', h, x', dx, dh once each backward. A row is held
// in registers by TPR lanes, NC chunks of 8 columns per lane, so nothing is read twice; the means are sums of f32 squares
// over at most 8 NC values per lane and then a tree over the lanes. Measured at 8 x 4170 rows of 768, bf16, gate and
// modulation per group: forward 43 us (4.7 TB/s; a 4-GB copy runs at 4.6), backward 64 us (4.8 TB/s) and 6.8 us for the
// vectors' gradients; on an f32 stream 65 us (4.7 TB/s) and 98 (4.7). At 4 x 1025 x 1280 the backward takes 20 and 6 us
// (3.1 TB/s: three passes of a block do not cover their latency).
#include "common.h"

namespace {

struct GnArgs {
  const bf16_t* h; long ldh;
  const void* x; long ldx;        // forward: x; backward: x'
  void* xo; long ldxo;            // forward: x'; backward: dx
  bf16_t* y; long ldy;            // forward: y; backward: dh
  const bf16_t* dy; long lddy;    // backward
  const void* dxn; long lddxn;    // backward: dx' (may be null: zero)
  const bf16_t* w_post; const bf16_t* w_pre;
  const bf16_t* gate; long ldg;   // row stride per group; 0: one vector for all
  const bf16_t* scale; long lds;
  const bf16_t* shift; long ldsh;
  float* rstd_post; float* rstd_pre;
  float* part;                    // backward: [groups * bpg][3][D]
  int rows, D;                    // rows per group
  int bpg, rpb;                   // blocks per group, rows per block
  float s, eps;
};

template <bool F32>
__device__ __forceinline__ void gn_load8(const void* p, long at, float (&f)[8]) {
  if (F32) {
    const floatx4 a = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(p) + at);
    const floatx4 b = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(p) + at + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
  } else {
    unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const bf16_t*>(p) + at), f);
  }
}
// Stores f and leaves in f the stored values.
template <bool F32>
__device__ __forceinline__ void gn_store8(void* p, long at, float (&f)[8]) {
  if (F32) {
    *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(p) + at) = floatx4{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(p) + at + 4) = floatx4{f[4], f[5], f[6], f[7]};
  } else {
    const uint4 v = pack8(f);
    *reinterpret_cast<uint4*>(reinterpret_cast<bf16_t*>(p) + at) = v;
    unpack8(v, f);
  }
}

// Eight values as they lie in memory, so that all loads of a row are under way before the first is used.
template <bool F32> struct Raw8;
template <> struct Raw8<false> {
  uint4 v;
  __device__ __forceinline__ void load(const void* p, long at, bool on) {
    v = on ? *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16_t*>(p) + at) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const { unpack8(v, f); }
};
template <> struct Raw8<true> {
  floatx4 a, b;
  __device__ __forceinline__ void load(const void* p, long at, bool on) {
    const float* q = reinterpret_cast<const float*>(p) + at;
    a = on ? *reinterpret_cast<const floatx4*>(q) : floatx4{0.f, 0.f, 0.f, 0.f};
    b = on ? *reinterpret_cast<const floatx4*>(q + 4) : floatx4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
  }
};

// Sum over the TPR lanes (a power of two, at most 64) of a row, or over the whole block (TPR = 256) through `red`.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) v += __shfl_xor(v, o, 64);
  if (TPR > 64) {
    __syncthreads();  // the previous sum's readers are done with red
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

template <int TPR, int NC, bool XF32>
__global__ __launch_bounds__(256) void gated_norm_fwd_kernel(GnArgs g) {
  __shared__ float red[4];
  constexpr int RPB = 256 / TPR;  // rows a block works on at once
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int group = blockIdx.x / g.bpg, r0 = (blockIdx.x % g.bpg) * g.rpb;
  const int nch = g.D >> 3;
  const float inv = 1.f / (float)g.D;
  const int r1 = min(g.rows, r0 + g.rpb);
  for (int rb = r0; rb < r1; rb += RPB) {  // the same trip count for the whole block (row_sum's barriers)
    const bool ok = rb + sub < r1;
    const long row = (long)group * g.rows + rb + sub;
    Raw8<false> wh[NC];
    Raw8<XF32> wx[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + TPR * i;
      wh[i].load(g.h, row * g.ldh + c * 8, ok && c < nch);
      wx[i].load(g.x, row * g.ldx + c * 8, ok && c < nch);
    }
    float ss = 0.f, r = g.s;
    if (g.w_post) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float u[8];
        wh[i].get(u);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += u[e] * u[e];
      }
      const float rh = rsqrtf(row_sum<TPR>(ss, red) * inv + g.eps);
      if (lane == 0 && ok && g.rstd_post) g.rstd_post[row] = rh;
      r *= rh;
    }
    float f[NC][8];
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + TPR * i, cv = min(c, nch - 1);  // past the row (in the last chunk): no value, no part in the mean
      float u[8], t[8];
      wh[i].get(u);
      wx[i].get(f[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] *= r;
      if (g.w_post) {
        gn_load8<false>(g.w_post, cv * 8, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] *= t[e];
      }
      if (g.gate) {
        gn_load8<false>(g.gate, group * g.ldg + cv * 8, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] *= t[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = i == NC - 1 && c >= nch ? 0.f : f[i][e] + u[e];
      if (ok && c < nch) gn_store8<XF32>(g.xo, row * g.ldxo + c * 8, f[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += f[i][e] * f[i][e];
    }
    if (!g.w_pre) continue;
    const float rx = rsqrtf(row_sum<TPR>(ss, red) * inv + g.eps);
    if (lane == 0 && ok && g.rstd_pre) g.rstd_pre[row] = rx;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + TPR * i;
      if (ok && c < nch) {
        float t[8];
        gn_load8<false>(g.w_pre, c * 8, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * rx * t[e];
        if (g.scale) {
          float b[8];
          gn_load8<false>(g.scale, group * g.lds + c * 8, t);
          gn_load8<false>(g.shift, group * g.ldsh + c * 8, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * (1.f + t[e]) + b[e];
        }
        gn_store8<false>(g.y, row * g.ldy + c * 8, f[i]);
      }
    }
  }
}

constexpr int gn_bwd_occ(int nc) { return nc == 1 ? 4 : nc == 2 ? 3 : nc == 3 ? 2 : 1; }  // blocks per CU

// The rows of a block belong to one group; each lane keeps the sums S, P, Q of its columns and the block leaves one partial
// row of each in g.part (no atomics: the same bits every time).
template <int TPR, int NC, bool XF32>
__global__ __launch_bounds__(256, gn_bwd_occ(NC)) void gated_norm_bwd_kernel(GnArgs g) {
  extern __shared__ __attribute__((aligned(16))) float cols[];  // the rows' factors [2][D], then column sums [4][D]
  __shared__ float red[4];
  constexpr int RPB = 256 / TPR;
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int group = blockIdx.x / g.bpg, r0 = (blockIdx.x % g.bpg) * g.rpb;
  const int nch = g.D >> 3;
  const float inv = 1.f / (float)g.D;
  const int r1 = min(g.rows, r0 + g.rpb);
  // what the rows of the group share: (1 + scale) w_pre and s gate w_post, f32
  float* cw = cols;
  float* gw = cols + g.D;
  for (int c = threadIdx.x; c < nch; c += 256) {
    float a[8], b[8], t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = 1.f, b[e] = g.s;
    if (g.scale) {
      gn_load8<false>(g.scale, group * g.lds + c * 8, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] += t[e];
    }
    if (g.w_pre) {
      gn_load8<false>(g.w_pre, c * 8, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] *= t[e];
    }
    if (g.gate) {
      gn_load8<false>(g.gate, group * g.ldg + c * 8, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] *= t[e];
    }
    if (g.w_post) {
      gn_load8<false>(g.w_post, c * 8, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] *= t[e];
    }
    gn_store8<true>(cw, c * 8, a);
    gn_store8<true>(gw, c * 8, b);
  }
  __syncthreads();
  float S[NC][8], P[NC][8], Q[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) S[i][e] = P[i][e] = Q[i][e] = 0.f;
  for (int rb = r0; rb < r1; rb += RPB) {
    const bool ok = rb + sub < r1;
    const long row = (long)group * g.rows + rb + sub;
    Raw8<XF32> wx[NC], wd[NC];
    Raw8<false> wy[NC], wh[NC];
    const float rx = ok && g.w_pre ? g.rstd_pre[row] : 0.f, rh = g.w_post ? (ok ? g.rstd_post[row] : 0.f) : 1.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + TPR * i;
      const bool on = ok && c < nch, pre = on && g.w_pre;
      wx[i].load(g.x, row * g.ldx + c * 8, pre);
      wy[i].load(g.dy, row * g.lddy + c * 8, pre);
      wd[i].load(g.dxn, row * g.lddxn + c * 8, on && g.dxn);
      wh[i].load(g.h, row * g.ldh + c * 8, on);
    }
    float dX[NC][8], dn[NC][8];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = min(lane + TPR * i, nch - 1);
      const bool on = ok && (i < NC - 1 || lane + TPR * i < nch);  // else no value: a factor may be infinite
      wd[i].get(dX[i]);
      if (g.w_pre) {
        float n[8], t[8];
        wx[i].get(n);
        gn_load8<true>(cw, c * 8, t);
        wy[i].get(dn[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          n[e] *= rx;
          S[i][e] += dn[i][e];
          P[i][e] += dn[i][e] * n[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dn[i][e] = on ? dn[i][e] * t[e] : 0.f;
          dot += dn[i][e] * n[e];
        }
      }
    }
    if (g.w_pre) {
      const float mean = row_sum<TPR>(dot, red) * inv;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float n[8];
        wx[i].get(n);
#pragma unroll
        for (int e = 0; e < 8; ++e) dX[i][e] += rx * (dn[i][e] - n[e] * rx * mean);
      }
    }
    dot = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + TPR * i, cv = min(c, nch - 1);
      float v[8], t[8];
      wh[i].get(v);
      gn_load8<true>(gw, cv * 8, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] *= rh;
        Q[i][e] += dX[i][e] * v[e];
        dn[i][e] = i == NC - 1 && c >= nch ? 0.f : dX[i][e] * t[e];  // from here on dn holds dv
        dot += dn[i][e] * v[e];
      }
      if (g.xo && ok && c < nch) gn_store8<XF32>(g.xo, row * g.ldxo + c * 8, dX[i]);
    }
    const float mean = g.w_post ? row_sum<TPR>(dot, red) * inv : 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + TPR * i;
      if (ok && c < nch) {
        if (g.w_post) {
          float v[8];
          wh[i].get(v);
#pragma unroll
          for (int e = 0; e < 8; ++e) dn[i][e] = rh * (dn[i][e] - v[e] * rh * mean);
        }
        gn_store8<false>(g.y, row * g.ldy + c * 8, dn[i]);
      }
    }
  }
  if (!g.part) return;
  // column sums: the lanes of a wave that hold the same columns, then the four waves in order through LDS (cols [4][8 nch],
  // value e of chunk c at e * nch + c: neighbouring lanes at neighbouring addresses)
  float* out = g.part + (long)blockIdx.x * 3 * g.D;
  constexpr int WPR = TPR > 64 ? TPR / 64 : 1;  // waves per row: with more than one, every column has one lane
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    float(&A)[NC][8] = k == 0 ? S : k == 1 ? P : Q;
    if (WPR > 1) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = lane + TPR * i;
        if (c < nch) {
          *reinterpret_cast<floatx4*>(out + k * g.D + c * 8) = floatx4{A[i][0], A[i][1], A[i][2], A[i][3]};
          *reinterpret_cast<floatx4*>(out + k * g.D + c * 8 + 4) = floatx4{A[i][4], A[i][5], A[i][6], A[i][7]};
        }
      }
      continue;
    }
    __syncthreads();
    float* mine = cols + (threadIdx.x >> 6) * g.D;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + TPR * i;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int o = TPR; o < 64; o <<= 1) A[i][e] += __shfl_xor(A[i][e], o, 64);
        if ((threadIdx.x & 63) < TPR && c < nch) mine[e * nch + c] = A[i][e];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < nch; c += 256) {
      float t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float* q = cols + e * nch + c;
        t[e] = (q[0] + q[g.D]) + (q[2 * g.D] + q[3 * g.D]);
      }
      *reinterpret_cast<floatx4*>(out + k * g.D + c * 8) = floatx4{t[0], t[1], t[2], t[3]};
      *reinterpret_cast<floatx4*>(out + k * g.D + c * 8 + 4) = floatx4{t[4], t[5], t[6], t[7]};
    }
  }
}

struct GnSum {
  const float* part;  // [groups * bpg][3][D]
  const bf16_t* w_post; const bf16_t* w_pre;
  const bf16_t* gate; long ldg;
  const bf16_t* scale; long lds;
  float* dw_post; float* dw_pre;
  float* dgate; float* dscale; float* dshift;
  int groups, bpg, per, D, gate_each, scale_each, shift_each;  // *_each: a gradient row per group
  float s;
};

// The gradients of the vectors from the blocks' partial rows: block (x, k) takes 16 columns of sum k (0 S: dshift; 1 P: dscale,
// dw_pre; 2 Q: dgate, dw_post), its 256 slots of 4 threads x 4 columns over (group, partial row). `per` slots (a power of two)
// share a group, 256 / per groups go at once; the slots of a group meet in a tree, the groups one after the other: a fixed
// order throughout.
__global__ __launch_bounds__(1024) void gated_norm_vec_kernel(GnSum g) {
  __shared__ floatx4 red[256][4];
  const int k = blockIdx.y, cl = threadIdx.x & 3, slot = threadIdx.x >> 2;
  float* each = k == 0 ? (g.shift_each ? g.dshift : nullptr) : k == 1 ? (g.scale_each ? g.dscale : nullptr)
                                                                       : (g.gate_each ? g.dgate : nullptr);
  float* sum = k == 0 ? (g.shift_each ? nullptr : g.dshift) : k == 1 ? (g.scale_each ? nullptr : g.dscale)
                                                                      : (g.gate_each ? nullptr : g.dgate);
  float* w = k == 0 ? nullptr : k == 1 ? g.dw_pre : g.dw_post;
  if (!each && !sum && !w) return;
  const int c = blockIdx.x * 16 + cl * 4;
  const bool on = c < g.D;  // D % 8 == 0: all four columns or none
  const int per = g.per, at_once = 256 / per, rank = slot & (per - 1);
  // d(vector of each group) = mul * sum; d(norm weight) = sum over groups of fac * sum, fac = 1 + scale or s * gate
  float mul[4] = {1.f, 1.f, 1.f, 1.f};
  const bf16_t* wv = k == 1 ? g.w_pre : k == 2 ? g.w_post : nullptr;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (on && wv) mul[e] = bf2f(wv[c + e]);
    if (k == 2) mul[e] *= g.s;
  }
  const bf16_t* fv = k == 1 ? g.scale : k == 2 ? g.gate : nullptr;
  const long fld = k == 1 ? g.lds : g.ldg;
  float a_sum[4] = {0.f, 0.f, 0.f, 0.f}, a_w[4] = {0.f, 0.f, 0.f, 0.f};
  for (int g0 = 0; g0 < g.groups; g0 += at_once) {
    const int i = g0 + slot / per;
    floatx4 s = {0.f, 0.f, 0.f, 0.f};
    if (on && i < g.groups) {
      const float* p = g.part + ((long)i * g.bpg * 3 + k) * g.D + c;
#pragma unroll 4
      for (int b = rank; b < g.bpg; b += per) s += *reinterpret_cast<const floatx4*>(p + (long)b * 3 * g.D);
    }
    red[slot][cl] = s;
    __syncthreads();
    for (int st = per >> 1; st >= 1; st >>= 1) {
      if (rank < st) red[slot][cl] += red[slot + st][cl];
      __syncthreads();
    }
    if (rank == 0 && on && i < g.groups) {
      s = red[slot][cl];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = fv ? bf2f(fv[i * fld + c + e]) : k == 1 ? 0.f : 1.f;
        const float d = mul[e] * s[e];
        if (each) each[(long)i * g.D + c + e] = d;
        a_sum[e] += d;
        a_w[e] += (k == 1 ? 1.f + f : g.s * f) * s[e];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    float* out = t == 0 ? sum : w;
    if (!out) continue;  // the same for the whole block
    if (rank == 0) red[slot / per][cl] = t == 0 ? floatx4{a_sum[0], a_sum[1], a_sum[2], a_sum[3]}
                                                : floatx4{a_w[0], a_w[1], a_w[2], a_w[3]};
    __syncthreads();
    if (slot == 0 && on) {
      floatx4 v = {0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < at_once; ++i) v += red[i][cl];
      *reinterpret_cast<floatx4*>(out + c) = v;
    }
    __syncthreads();
  }
}

constexpr int kGnMaxD = 10240;

// Lanes per row of the forward: the fewest of 16, 32, 64, 256 that hold the row in at most 5 chunks each, so that few lanes
// idle (768 columns: 32 lanes of 3 chunks).
int gn_tpr(int D) {
  const int nch = D / 8;
  return nch <= 80 ? 16 : nch <= 160 ? 32 : nch <= 320 ? 64 : 256;
}

// The backward keeps three sums for each of a lane's columns, so at most 3 chunks per lane below 1536 columns (5 took 256
// registers and one wave per SIMD).
int gn_bwd_tpr(int D) { return D <= 384 ? 16 : D <= 1536 ? 64 : 256; }
// Rows per block of the backward: whole passes of the block's rows, as many blocks as fit on the 256 CUs at once where there
// are enough rows.
int gn_rows_per_block(int groups, int rows, int D) {
  const int tpr = gn_bwd_tpr(D), nc = (D / 8 + tpr - 1) / tpr;
  const long rpb = 256 / tpr, at_once = 256L * gn_bwd_occ(nc) * rpb;
  const long passes = ((long)groups * rows + at_once - 1) / at_once;
  return (int)(rpb * (passes < 1 ? 1 : passes));
}
int gn_blocks_per_group(int groups, int rows, int D) {
  const int rpb = gn_rows_per_block(groups, rows, D);
  return (rows + rpb - 1) / rpb;
}

template <int TPR, int NC>
void gn_fwd_launch(const GnArgs& g, int blocks, bool xf32, hipStream_t s) {
  if (xf32) hipLaunchKernelGGL((gated_norm_fwd_kernel<TPR, NC, true>), dim3(blocks), dim3(256), 0, s, g);
  else hipLaunchKernelGGL((gated_norm_fwd_kernel<TPR, NC, false>), dim3(blocks), dim3(256), 0, s, g);
}
template <int TPR, int NC>
void gn_bwd_launch(const GnArgs& g, int blocks, bool xf32, hipStream_t s) {
  const size_t lds = (size_t)g.D * (TPR > 64 ? 2 : 4) * sizeof(float);
  if (xf32) hipLaunchKernelGGL((gated_norm_bwd_kernel<TPR, NC, true>), dim3(blocks), dim3(256), lds, s, g);
  else hipLaunchKernelGGL((gated_norm_bwd_kernel<TPR, NC, false>), dim3(blocks), dim3(256), lds, s, g);
}

template <int TPR>
void gn_fwd(const GnArgs& g, int blocks, bool xf32, hipStream_t s) {
  switch ((g.D / 8 + TPR - 1) / TPR) {
    case 1: gn_fwd_launch<TPR, 1>(g, blocks, xf32, s); break;
    case 2: gn_fwd_launch<TPR, 2>(g, blocks, xf32, s); break;
    case 3: gn_fwd_launch<TPR, 3>(g, blocks, xf32, s); break;
    case 4: gn_fwd_launch<TPR, 4>(g, blocks, xf32, s); break;
    default: gn_fwd_launch<TPR, 5>(g, blocks, xf32, s);
  }
}
template <int TPR>
void gn_bwd(const GnArgs& g, int blocks, bool xf32, hipStream_t s) {
  switch ((g.D / 8 + TPR - 1) / TPR) {
    case 1: gn_bwd_launch<TPR, 1>(g, blocks, xf32, s); break;
    case 2: gn_bwd_launch<TPR, 2>(g, blocks, xf32, s); break;
    case 3: gn_bwd_launch<TPR, 3>(g, blocks, xf32, s); break;
    default:
      if constexpr (TPR == 256) {
        if (g.D <= 8192) gn_bwd_launch<TPR, 4>(g, blocks, xf32, s);
        else gn_bwd_launch<TPR, 5>(g, blocks, xf32, s);
      }
  }
}

void gn_fwd_dispatch(const GnArgs& g, int blocks, bool xf32, hipStream_t s) {
  switch (gn_tpr(g.D)) {
    case 16: gn_fwd<16>(g, blocks, xf32, s); break;
    case 32: gn_fwd<32>(g, blocks, xf32, s); break;
    case 64: gn_fwd<64>(g, blocks, xf32, s); break;
    default: gn_fwd<256>(g, blocks, xf32, s);
  }
}
void gn_bwd_dispatch(const GnArgs& g, int blocks, bool xf32, hipStream_t s) {
  switch (gn_bwd_tpr(g.D)) {
    case 16: gn_bwd<16>(g, blocks, xf32, s); break;
    case 64: gn_bwd<64>(g, blocks, xf32, s); break;
    default: gn_bwd<256>(g, blocks, xf32, s);
  }
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// Rows of D elements of es bytes at multiples of 16 bytes; a null p is no tensor.
bool rows_ok(const void* p, long ld, int D, int es, long rows) {
  return !p || (al16(p) && (rows <= 1 || (ld >= D && ld * es % 16 == 0)));
}
bool vec_ok(const void* p, long ld, int D) { return !p || (al16(p) && (ld == 0 || (ld >= D && ld % 8 == 0))); }

}  // namespace

extern "C" long vpt_gated_norm_bwd_workspace(int groups, int rows, int D) {
  if (groups <= 0 || rows <= 0 || D <= 0 || D % 8 || D > kGnMaxD) return 0;
  return (long)groups * gn_blocks_per_group(groups, rows, D) * 3 * D * (long)sizeof(float);
}

#define VPT_GN_SHAPE(name)                                                                                             \
  VPT_CHECK_ARG(groups >= 0 && rows >= 0 && groups < (1 << 24) && (long)groups * rows <= (1L << 30),                   \
                name ": 0 <= groups < 2^24, 0 <= rows, groups * rows <= 2^30");                                         \
  VPT_CHECK_ARG(D > 0 && D % 8 == 0 && D <= kGnMaxD, name ": D a multiple of 8, at most 10240");                       \
  VPT_CHECK_ARG(!scale == !shift, name ": scale and shift go together");                                               \
  VPT_CHECK_ARG(w_pre || !scale, name ": a modulation needs w_pre")

extern "C" int vpt_gated_norm_fwd(const void* h, long ldh, const void* x, int x_f32, long ldx, const void* w_post,
                                  const void* w_pre, const void* gate, long ldg, const void* scale, long lds,
                                  const void* shift, long ldsh, void* x_out, long ldxo, void* y, long ldy,
                                  float* rstd_post, float* rstd_pre, int groups, int rows, int D, float resid_scale,
                                  float eps, void* stream) {
  VPT_GN_SHAPE("vpt_gated_norm_fwd");
  const long M = (long)groups * rows;
  if (M == 0) return VPT_OK;
  const int es = x_f32 ? 4 : 2;
  VPT_CHECK_ARG(h && x && x_out && (!w_pre == !y), "vpt_gated_norm_fwd: h, x, x_out, and y with w_pre");
  VPT_CHECK_ARG(rows_ok(h, ldh, D, 2, M) && rows_ok(x, ldx, D, es, M) && rows_ok(x_out, ldxo, D, es, M) &&
                    rows_ok(y, ldy, D, 2, M),
                "vpt_gated_norm_fwd: rows of D elements at multiples of 16 bytes");
  VPT_CHECK_ARG(vec_ok(w_post, 0, D) && vec_ok(w_pre, 0, D) && vec_ok(gate, ldg, D) && vec_ok(scale, lds, D) &&
                    vec_ok(shift, ldsh, D),
                "vpt_gated_norm_fwd: vectors at multiples of 16 bytes");
  GnArgs g{};
  g.h = (const bf16_t*)h; g.ldh = ldh;
  g.x = x; g.ldx = ldx;
  g.xo = x_out; g.ldxo = ldxo;
  g.y = (bf16_t*)y; g.ldy = ldy;
  g.w_post = (const bf16_t*)w_post; g.w_pre = (const bf16_t*)w_pre;
  g.gate = (const bf16_t*)gate; g.ldg = ldg;
  g.scale = (const bf16_t*)scale; g.lds = lds;
  g.shift = (const bf16_t*)shift; g.ldsh = ldsh;
  g.rstd_post = rstd_post; g.rstd_pre = rstd_pre;
  g.rows = rows; g.D = D;
  g.rpb = 256 / gn_tpr(D);
  while ((long)groups * ((rows + g.rpb - 1) / g.rpb) >= 1L << 24) g.rpb *= 2;  // a grid has under 2^32 threads
  g.bpg = (rows + g.rpb - 1) / g.rpb;
  g.s = resid_scale; g.eps = eps;
  gn_fwd_dispatch(g, groups * g.bpg, x_f32 != 0, (hipStream_t)stream);
  VPT_LAUNCH_CHECK();
  return VPT_OK;
}

extern "C" int vpt_gated_norm_bwd(const void* dy, long lddy, const void* dx_new, long lddxn, const void* h, long ldh,
                                  const void* x_new, int x_f32, long ldxn, const float* rstd_post, const float* rstd_pre,
                                  const void* w_post, const void* w_pre, const void* gate, long ldg, const void* scale,
                                  long lds, const void* shift, long ldsh, void* dh, long lddh, void* dx, long lddx,
                                  float* dw_post, float* dw_pre, float* dgate, float* dscale, float* dshift, void* workspace,
                                  int groups, int rows, int D, float resid_scale, void* stream) {
  VPT_GN_SHAPE("vpt_gated_norm_bwd");
  const long M = (long)groups * rows;
  const int es = x_f32 ? 4 : 2;
  VPT_CHECK_ARG((w_post || !dw_post) && (w_pre || !dw_pre) && (gate || !dgate) && (scale || (!dscale && !dshift)),
                "vpt_gated_norm_bwd: a gradient of a vector that is not there");
  VPT_CHECK_ARG(vec_ok(w_post, 0, D) && vec_ok(w_pre, 0, D) && vec_ok(gate, ldg, D) && vec_ok(scale, lds, D) &&
                    vec_ok(shift, ldsh, D),
                "vpt_gated_norm_bwd: vectors at multiples of 16 bytes");
  const bool sums = dw_post || dw_pre || dgate || dscale || dshift;
  hipStream_t st = (hipStream_t)stream;
  GnSum z{};
  z.w_post = (const bf16_t*)w_post; z.w_pre = (const bf16_t*)w_pre;
  z.gate = (const bf16_t*)gate; z.ldg = ldg;
  z.scale = (const bf16_t*)scale; z.lds = lds;
  z.dw_post = dw_post; z.dw_pre = dw_pre;
  z.dgate = dgate; z.dscale = dscale; z.dshift = dshift;
  z.groups = groups; z.D = D;
  z.gate_each = ldg != 0; z.scale_each = lds != 0; z.shift_each = ldsh != 0;
  z.s = resid_scale;
  VPT_CHECK_ARG(M > 0 || !sums, "vpt_gated_norm_bwd: no rows to sum over");
  if (M == 0) return VPT_OK;
  VPT_CHECK_ARG(h && dh && (!w_post || rstd_post) && (!w_pre || (dy && x_new && rstd_pre && dx)) && (w_pre || dx_new),
                "vpt_gated_norm_bwd: h, dh; rstd_post with w_post; dy, x_new, rstd_pre and dx with w_pre, dx_new without");
  VPT_CHECK_ARG(rows_ok(dy, lddy, D, 2, M) && rows_ok(dx_new, lddxn, D, es, M) && rows_ok(h, ldh, D, 2, M) &&
                    rows_ok(x_new, ldxn, D, es, M) && rows_ok(dh, lddh, D, 2, M) && rows_ok(dx, lddx, D, es, M),
                "vpt_gated_norm_bwd: rows of D elements at multiples of 16 bytes");
  VPT_CHECK_ARG(!sums || (workspace && al16(workspace)), "vpt_gated_norm_bwd: the vectors' gradients need the workspace");
  GnArgs g{};
  g.h = (const bf16_t*)h; g.ldh = ldh;
  g.x = x_new; g.ldx = ldxn;
  g.xo = w_pre ? dx : nullptr; g.ldxo = lddx;  // without a next norm dx is dx_new itself
  g.y = (bf16_t*)dh; g.ldy = lddh;
  g.dy = (const bf16_t*)dy; g.lddy = lddy;
  g.dxn = dx_new; g.lddxn = lddxn;
  g.w_post = z.w_post; g.w_pre = z.w_pre;
  g.gate = z.gate; g.ldg = ldg;
  g.scale = z.scale; g.lds = lds;
  g.rstd_post = const_cast<float*>(rstd_post); g.rstd_pre = const_cast<float*>(rstd_pre);
  g.rows = rows; g.D = D; g.s = resid_scale;
  g.bpg = gn_blocks_per_group(groups, rows, D);
  g.rpb = gn_rows_per_block(groups, rows, D);
  g.part = sums ? (float*)workspace : nullptr;
  const int blocks = groups * g.bpg;
  gn_bwd_dispatch(g, blocks, x_f32 != 0, st);
  VPT_LAUNCH_CHECK();
  if (!sums) return VPT_OK;
  z.bpg = g.bpg;
  z.part = g.part;
  z.per = 1;
  while (z.per < 256 && z.per * 2 * groups <= 256) z.per *= 2;
  hipLaunchKernelGGL(gated_norm_vec_kernel, dim3((D + 15) / 16, 3), dim3(1024), 0, st, z);
  VPT_LAUNCH_CHECK();
  return VPT_OK;
}
