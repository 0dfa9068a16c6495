// Layer norm with modulation, and the backward pass of layer and RMS norm with modulation (gfx950).
//
//   n = (x - mean) * rstd (layer) or x * rstd (RMS);  y = (n * w + b) * (1 + scale[seg]) + shift[seg]
//
// Backward, with g = dy * w * (1 + scale[seg]) and row means over the D columns:
//   dx = rstd * (g - mean(g) - n * mean(g * n))        (RMS: no mean(g) term)
// and, from the two column sums of each segment S0 = sum dy and S1 = sum dy * n, every small gradient:
//   dshift[seg] = S0, dscale[seg] = w * S1 + b * S0, dw = sum_seg (1 + scale) * S1, db = sum_seg (1 + scale) * S0.
//
// Bound by HBM: x and dy are read once (mean and rstd are made again from the row in registers, so the forward pass
// keeps nothing), dx is written once. One thread holds 8 consecutive columns of a row (16-B bf16 accesses).
#include <math.h>

#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace flite {

namespace {

constexpr int kMaxThreads = 512;  // threads per row: 8 columns each, so one pass covers 4096 columns
constexpr int kMaxDim = 8192;

struct NormTrainDev {
  NormTrainParams p;
  int strips;      // row strips per segment (backward)
  int strip_rows;  // rows per strip
};

template <bool BF>
__device__ __forceinline__ void load8(const void* base, long off, float (&v)[8]) {
  if constexpr (BF) {
    const u32x4 w = *(const u32x4*)((const bf16_t*)base + off);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  } else {
    const f32x4 a = *(const f32x4*)((const float*)base + off), b = *(const f32x4*)((const float*)base + off + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  }
}

template <bool BF>
__device__ __forceinline__ void store8(void* base, long off, const float (&v)[8]) {
  if constexpr (BF) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack2bf(v[2 * j], v[2 * j + 1]);
    *(u32x4*)((bf16_t*)base + off) = w;
  } else {
    *(f32x4*)((float*)base + off) = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)((float*)base + off + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}

// Sums of N values over the row's threads (all of the workgroup), the same on every thread: a wave sum, then one LDS
// slot per wave. `buf` holds N * 8 floats; consecutive calls alternate between two of them, so one barrier per call
// is enough (a wave can be at most one call ahead of the slowest reader).
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* buf, int waves) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if (waves == 1) return;
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[i * 8 + wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = 0; w < waves; ++w) s += buf[i * 8 + w];
    v[i] = s;
  }
}

// ---- forward: one workgroup per row (D <= 512: one wave) ----
template <bool XBF, int NCH>
__global__ __launch_bounds__(kMaxThreads) void layernorm_mod_kernel(NormTrainParams p) {
  __shared__ float buf[2][8];
  const int waves = blockDim.x >> 6;
  const long row = blockIdx.x;
  const long seg = p.seg_rows > 0 ? row / p.seg_rows : 0;
  float x[NCH][8];
  float s[1] = {0.f};
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * blockDim.x + threadIdx.x) * 8;
    if (col < p.D) {
      load8<XBF>(p.x, row * p.ldx + col, x[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[c][j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[0] += x[c][j];
  }
  row_sums<1>(s, buf[0], waves);
  const float mean = s[0] / (float)p.D;
  s[0] = 0.f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const bool live = (c * (int)blockDim.x + (int)threadIdx.x) * 8 < p.D;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[c][j] = live ? x[c][j] - mean : 0.f;
      s[0] += x[c][j] * x[c][j];
    }
  }
  row_sums<1>(s, buf[1], waves);
  const float r = 1.f / sqrtf(s[0] / (float)p.D + p.eps);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * blockDim.x + threadIdx.x) * 8;
    if (col >= p.D) continue;
    float a[8], y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = x[c][j] * r;
    if (p.w) {
      load8<true>(p.w, col, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= a[j];
    }
    if (p.b) {
      load8<true>(p.b, col, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] += a[j];
    }
    if (p.scale) {
      load8<false>(p.scale, seg * p.mod_seg_stride + col, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= 1.f + a[j];
    }
    if (p.shift) {
      load8<false>(p.shift, seg * p.mod_seg_stride + col, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] += a[j];
    }
    store8<true>(p.y, row * p.ldy + col, y);
  }
}

// ---- backward: one workgroup per strip of rows of one segment; S0 and S1 of the strip to the workspace ----
template <bool XBF, bool RMS, int NCH, bool SUMS>
__global__ __launch_bounds__(kMaxThreads) void norm_bwd_kernel(NormTrainDev d) {
  const NormTrainParams& p = d.p;
  __shared__ float buf[2][3 * 8];
  const int waves = blockDim.x >> 6;
  const int strip = blockIdx.x % d.strips;
  const long seg = blockIdx.x / d.strips;
  const long seg_rows = p.seg_rows > 0 ? p.seg_rows : p.rows;
  const long seg_end = min((seg + 1) * seg_rows, p.rows);
  const long r0 = seg * seg_rows + (long)strip * d.strip_rows;
  const long r1 = min(r0 + d.strip_rows, seg_end);

  float a[NCH][8], s0[NCH][8], s1[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[c][j] = 1.f;
      s0[c][j] = s1[c][j] = 0.f;
    }
    if (col >= p.D) continue;
    float t[8];
    if (p.w) load8<true>(p.w, col, a[c]);
    if (p.scale) {
      load8<false>(p.scale, seg * p.mod_seg_stride + col, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[c][j] *= 1.f + t[j];
    }
  }
  const float inv_d = 1.f / (float)p.D;
  for (long row = r0; row < r1; ++row) {
    float x[NCH][8], dy[NCH][8];
    float mean = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * 8;
      if (col < p.D) {
        load8<XBF>(p.x, row * p.ldx + col, x[c]);
        load8<true>(p.dy, row * p.lddy + col, dy[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[c][j] = dy[c][j] = 0.f;
      }
    }
    if constexpr (!RMS) {
      float s[1] = {0.f};
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] += x[c][j];
      row_sums<1>(s, buf[0], waves);
      mean = s[0] * inv_d;
    }
    float s[3] = {0.f, 0.f, 0.f};  // sum (x - mean)^2, sum g, sum g (x - mean)
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const bool live = (c * (int)blockDim.x + (int)threadIdx.x) * 8 < p.D;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (!RMS) x[c][j] = live ? x[c][j] - mean : 0.f;
        const float g = dy[c][j] * a[c][j];
        s[0] += x[c][j] * x[c][j];
        s[1] += g;
        s[2] += g * x[c][j];
      }
    }
    row_sums<3>(s, buf[RMS ? (int)(row & 1) : 1], waves);
    const float r = 1.f / sqrtf(s[0] * inv_d + p.eps);
    const float c1 = RMS ? 0.f : s[1] * inv_d;
    const float c2 = s[2] * inv_d * r;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * 8;
      if (col >= p.D) continue;
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = x[c][j] * r;
        if constexpr (SUMS) {
          s0[c][j] += dy[c][j];
          s1[c][j] += dy[c][j] * n;
        }
        o[j] = r * (dy[c][j] * a[c][j] - c1 - n * c2);
      }
      store8<XBF>(p.dx, row * p.lddx + col, o);
    }
  }
  if constexpr (SUMS) {
    float* ws = p.ws + (long)blockIdx.x * 2 * p.D;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * 8;
      if (col >= p.D) continue;
      store8<false>(ws, col, s0[c]);
      store8<false>(ws, p.D + col, s1[c]);
    }
  }
}

// ---- the column sums over the strips, in strip and segment order, and the small gradients ----
// A workgroup has 16 columns (64 B of a partial row) and 32 lanes per column: lp of them share a segment's strips, the
// others take other segments. The lanes' sums are added in lane order, so a result does not depend on timing.
constexpr int RC = 16, RL = 32;
__global__ __launch_bounds__(RC* RL) void norm_sums_kernel(NormTrainDev d, long segs, int lp) {
  const NormTrainParams& p = d.p;
  __shared__ float sh[2][RL][RC + 1];
  const int c = threadIdx.x % RC, l = threadIdx.x / RC;
  const int col = blockIdx.x * RC + c;
  const bool live = col < p.D;
  const int ls = RL / lp, li = l % lp;
  const float w = live && p.w ? bf2f(p.w[col]) : 1.f, b = live && p.b ? bf2f(p.b[col]) : 0.f;
  float dw = 0.f, db = 0.f;
  for (long base = 0; base < segs; base += ls) {
    const long seg = base + l / lp;
    float t0 = 0.f, t1 = 0.f;
    if (live && seg < segs) {
      const float* ws = p.ws + seg * d.strips * 2 * p.D + col;
#pragma unroll 4
      for (int s = li; s < d.strips; s += lp) {
        t0 += ws[(long)s * 2 * p.D];
        t1 += ws[(long)s * 2 * p.D + p.D];
      }
    }
    sh[0][l][c] = t0;
    sh[1][l][c] = t1;
    __syncthreads();
    if (live && li == 0 && seg < segs) {
      t0 = t1 = 0.f;
      for (int i = 0; i < lp; ++i) {
        t0 += sh[0][l + i][c];
        t1 += sh[1][l + i][c];
      }
      const float g = p.scale ? 1.f + p.scale[seg * p.mod_seg_stride + col] : 1.f;
      dw += g * t1;
      db += g * t0;
      if (p.dshift) p.dshift[seg * p.D + col] = t0;
      if (p.dscale) p.dscale[seg * p.D + col] = w * t1 + b * t0;
    }
    __syncthreads();
  }
  sh[0][l][c] = li == 0 ? dw : 0.f;
  sh[1][l][c] = li == 0 ? db : 0.f;
  __syncthreads();
  if (l == 0 && live) {
    dw = db = 0.f;
    for (int i = 0; i < RL; i += lp) {
      dw += sh[0][i][c];
      db += sh[1][i][c];
    }
    if (p.dw) p.dw[col] = dw;
    if (p.db) p.db[col] = db;
  }
}

int threads_of(int D, int* nch) {
  *nch = D > kMaxThreads * 8 ? 2 : 1;
  const int per = (D / 8 + *nch - 1) / *nch;
  return (per + 63) / 64 * 64;
}

int check_common(const NormTrainParams& p) {
  FLITE_REQUIRE(p.D > 0 && p.D % 8 == 0 && p.D <= kMaxDim, "norm: dim must be a multiple of 8, at most 8192");
  FLITE_REQUIRE(p.rows >= 0 && p.rows <= 0x7fffffffL, "norm: rows outside 0 .. 2^31 - 1");
  FLITE_REQUIRE(p.seg_rows >= 0, "norm: seg_rows < 0");
  FLITE_REQUIRE((p.x || p.rows == 0) && ((uintptr_t)p.x & 15) == 0 && p.ldx % 8 == 0 && p.ldx >= p.D,
                "norm: x must be 16-byte aligned rows, their stride a multiple of 8 and at least dim");
  FLITE_REQUIRE(((uintptr_t)p.w & 15) == 0 && ((uintptr_t)p.b & 15) == 0, "norm: w and b must be 16-byte aligned");
  FLITE_REQUIRE(((uintptr_t)p.scale & 15) == 0 && ((uintptr_t)p.shift & 15) == 0 && p.mod_seg_stride % 4 == 0 &&
                    p.mod_seg_stride >= 0,
                "norm: shift and scale must be 16-byte aligned rows");
  return 0;
}

// Strips of the backward pass: enough workgroups for the chip (two per CU), none under 4 rows, one segment each.
void plan(const NormTrainParams& p, long* segs, int* strips, int* strip_rows) {
  const long seg_rows = p.seg_rows > 0 ? std::min(p.seg_rows, p.rows) : p.rows;
  *segs = p.rows > 0 ? (p.rows + seg_rows - 1) / seg_rows : 0;
  if (*segs == 0) {
    *strips = *strip_rows = 0;
    return;
  }
  const long want = std::max(1L, 512 / *segs);
  const long most = std::max(1L, seg_rows / 4);
  const long n = std::min(want, most);
  *strip_rows = (int)((seg_rows + n - 1) / n);
  *strips = (int)((seg_rows + *strip_rows - 1) / *strip_rows);
}

using BwdKernel = void (*)(NormTrainDev);
template <bool X, bool R, int N>
BwdKernel pick(bool sums) {
  return sums ? (BwdKernel)norm_bwd_kernel<X, R, N, true> : (BwdKernel)norm_bwd_kernel<X, R, N, false>;
}
template <bool X, bool R>
BwdKernel pick(int nch, bool sums) {
  return nch == 1 ? pick<X, R, 1>(sums) : pick<X, R, 2>(sums);
}
BwdKernel bwd_kernel(bool x_bf16, bool rms, int nch, bool sums) {
  if (x_bf16) return rms ? pick<true, true>(nch, sums) : pick<true, false>(nch, sums);
  return rms ? pick<false, true>(nch, sums) : pick<false, false>(nch, sums);
}

}  // namespace

long norm_bwd_workspace_bytes(long rows, long seg_rows, int D) {
  if (rows <= 0 || D <= 0 || seg_rows < 0) return 0;
  NormTrainParams p;
  p.rows = rows;
  p.seg_rows = seg_rows;
  long segs;
  int strips, strip_rows;
  plan(p, &segs, &strips, &strip_rows);
  return segs * strips * 2 * D * 4;
}

int layernorm_mod(const NormTrainParams& p, bool x_bf16, hipStream_t s) {
  if (int rc = check_common(p)) return rc;
  FLITE_REQUIRE((p.y || p.rows == 0) && ((uintptr_t)p.y & 15) == 0 && p.ldy % 8 == 0 && p.ldy >= p.D,
                "layernorm: y must be 16-byte aligned rows, their stride a multiple of 8 and at least dim");
  if (p.rows == 0) return 0;
  int nch;
  const dim3 block(threads_of(p.D, &nch)), grid((unsigned)p.rows);
  if (x_bf16 && nch == 1) hipLaunchKernelGGL((layernorm_mod_kernel<true, 1>), grid, block, 0, s, p);
  if (x_bf16 && nch == 2) hipLaunchKernelGGL((layernorm_mod_kernel<true, 2>), grid, block, 0, s, p);
  if (!x_bf16 && nch == 1) hipLaunchKernelGGL((layernorm_mod_kernel<false, 1>), grid, block, 0, s, p);
  if (!x_bf16 && nch == 2) hipLaunchKernelGGL((layernorm_mod_kernel<false, 2>), grid, block, 0, s, p);
  FLITE_HIP_CHECK(hipGetLastError());
  return 0;
}

int norm_bwd(const NormTrainParams& p, bool x_bf16, bool rms, hipStream_t s) {
  if (int rc = check_common(p)) return rc;
  FLITE_REQUIRE((p.dy || p.rows == 0) && ((uintptr_t)p.dy & 15) == 0 && p.lddy % 8 == 0 && p.lddy >= p.D,
                "norm backward: dy must be 16-byte aligned rows, their stride a multiple of 8 and at least dim");
  FLITE_REQUIRE((p.dx || p.rows == 0) && ((uintptr_t)p.dx & 15) == 0 && p.lddx % 8 == 0 && p.lddx >= p.D,
                "norm backward: dx must be 16-byte aligned rows, their stride a multiple of 8 and at least dim");
  FLITE_REQUIRE(!rms || !p.b, "norm backward: the RMS norm has no bias");
  FLITE_REQUIRE((!p.dw || p.w) && (!p.db || p.b) && (!p.dscale || p.scale),
                "norm backward: a gradient was asked for a weight, bias or scale that is not given");
  const bool sums = p.dw || p.db || p.dshift || p.dscale;
  NormTrainDev d;
  d.p = p;
  long segs;
  plan(p, &segs, &d.strips, &d.strip_rows);
  FLITE_REQUIRE(!sums || p.rows == 0 || (p.ws && ((uintptr_t)p.ws & 15) == 0 &&
                                         p.ws_bytes >= norm_bwd_workspace_bytes(p.rows, p.seg_rows, p.D)),
                "norm backward: workspace missing or too small");
  FLITE_REQUIRE(segs * d.strips <= 0x7fffffffL, "norm backward: too many segments");
  if (p.rows > 0) {
    int nch;
    const dim3 block(threads_of(p.D, &nch)), grid((unsigned)(segs * d.strips));
    hipLaunchKernelGGL(bwd_kernel(x_bf16, rms, nch, sums), grid, block, 0, s, d);
    FLITE_HIP_CHECK(hipGetLastError());
  }
  if (sums) {
    int lp = 1;
    while (lp < RL && lp < d.strips) lp *= 2;
    hipLaunchKernelGGL(norm_sums_kernel, dim3((p.D + RC - 1) / RC), dim3(RC * RL), 0, s, d, segs, lp);
    FLITE_HIP_CHECK(hipGetLastError());
  }
  return 0;
}

}  // namespace flite
