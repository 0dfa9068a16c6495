// Rotary positions over several axes (time, height, width, ...) with an optional per-head RMS norm, forward and
// backward (gfx950).
//
// Pair i of an axis with n pairs turns by a = position * base^(-i / n); the sign is the framework's (rotate-half,
// reference f_lite/model.py:403-414): (x1, x2) -> (x1 cos a + x2 sin a, x2 cos a - x1 sin a). The pairs of all axes
// follow one another; dimensions past the last pair are not turned. Then, as QKNorm does after the rotation
// (model.py:115-126,180,197), y = r * rot(x) with r = rsqrt(mean(x^2) + eps) per head.
// Backward, from y and r: dx = rot^-1(r * (dy - y * mean(y * dy))); a rotation keeps lengths, so nothing else of the
// forward pass is needed and y is the tensor that attention keeps anyway.
//
// Bound by HBM: every element is read once (backward with the norm: dy and y) and written once. The angles cost no
// traffic but the positions: a workgroup makes the sines of its rows once, in LDS, for all their heads. An angle is
// position * frequency in turns in 64 bits, less its whole turns, so a far position keeps a full fp32 sine.
// Measured, with the norm: 8224 rows of 24 heads of 256 in bf16, 202 MB forward, 33 us where the rows are in the last-level
// cache and 43 (4.7 TB/s) where they are not; backward 304 MB in 57 us (5.3 TB/s). A large copy reaches 5.2 TB/s.
#include <cmath>

#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace flite {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;

struct RopeAxesDev {
  RopeAxesParams p;
  double turns[kMaxPairs];  // base^(-i / n) / (2 pi) of pair j
  unsigned char axis[kMaxPairs];
  int pairs;     // all axes'
  int lanes_lg;  // lanes of one head: 16 elements each, a power of two of them
  int rows_lg;   // rows of a workgroup
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

// Turns the 8 pairs of a lane: rotate-half holds the x1 of its pairs in u and the x2 in v, interleaved holds pair j in
// elements 2j, 2j + 1 of (u, v). INV turns back.
template <bool INTER, bool INV>
__device__ __forceinline__ void turn(float (&u)[8], float (&v)[8], const f32x2 (&cs)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float& a = INTER ? (j < 4 ? u[2 * j] : v[2 * j - 8]) : u[j];
    float& b = INTER ? (j < 4 ? u[2 * j + 1] : v[2 * j - 7]) : v[j];
    const float c = cs[j][0], s = INV ? -cs[j][1] : cs[j][1];
    const float x1 = a, x2 = b;
    a = x1 * c + x2 * s;
    b = x2 * c - x1 * s;
  }
}

template <bool BF, bool INTER, bool NORM, bool BWD>
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(RopeAxesDev d) {
  extern __shared__ __attribute__((aligned(16))) f32x2 cs_tab[];  // [rows of the workgroup][pairs] (cos, sin)
  const RopeAxesParams& p = d.p;
  const int n_rows = 1 << d.rows_lg;
  const long row0 = (long)blockIdx.x << d.rows_lg;
  for (int i = threadIdx.x; i < n_rows * d.pairs; i += kThreads) {
    const int r = i / d.pairs, j = i - r * d.pairs;
    const long row = row0 + r;
    if (row >= p.rows) break;
    const long at = (row % p.tokens) * p.axes + d.axis[j];
    const double pos = p.pos_is_f32 ? (double)((const float*)p.positions)[at] : (double)((const int*)p.positions)[at];
    const double t = pos * d.turns[j];
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    cs_tab[i] = f32x2{c, s};
  }
  __syncthreads();

  const int lane = threadIdx.x & ((1 << d.lanes_lg) - 1);
  const int group = threadIdx.x >> d.lanes_lg, groups = kThreads >> d.lanes_lg;
  const int r = group & (n_rows - 1);
  const long row = row0 + r;
  const bool unit = lane * 16 < p.dim;         // this lane has elements
  const bool turned = unit && lane * 8 < d.pairs;
  int e1, e2;                                  // where its two runs of 8 elements start
  if (turned) {
    e1 = INTER ? 16 * lane : 8 * lane;
    e2 = INTER ? e1 + 8 : e1 + d.pairs;
  } else {
    e1 = 2 * d.pairs + 16 * (lane - (d.pairs >> 3));
    e2 = e1 + 8;
  }
  f32x2 cs[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cs[j] = turned ? cs_tab[r * d.pairs + 8 * lane + j] : f32x2{1.f, 0.f};

  const int step = groups >> d.rows_lg;
  for (int h = group >> d.rows_lg; h < p.heads; h += step) {
    const bool live = unit && row < p.rows;
    float u[8], v[8], y1[8], y2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = v[j] = y1[j] = y2[j] = 0.f;
    float rstd = 1.f;
    if (live) {
      const long at = row * p.x_row + (long)h * p.x_head;
      load8<BF>(p.x, at + e1, u);
      load8<BF>(p.x, at + e2, v);
      if constexpr (BWD && NORM) {
        const long yat = row * p.y_row + (long)h * p.y_head;
        load8<BF>(p.y, yat + e1, y1);
        load8<BF>(p.y, yat + e2, y2);
        rstd = p.rstd[row * p.heads + h];
      }
    }
    const bool rot = turned && h < p.rope_heads;
    if constexpr (!BWD) {
      if (rot) turn<INTER, false>(u, v, cs);
    }
    if constexpr (NORM) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += BWD ? u[j] * y1[j] + v[j] * y2[j] : u[j] * u[j] + v[j] * v[j];
      for (int o = 1; o < (1 << d.lanes_lg); o <<= 1) s += __shfl_xor(s, o, 64);
      s /= (float)p.dim;
      if constexpr (BWD) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[j] = rstd * (u[j] - y1[j] * s);
          v[j] = rstd * (v[j] - y2[j] * s);
        }
      } else {
        rstd = 1.f / sqrtf(s + p.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[j] *= rstd;
          v[j] *= rstd;
        }
        if (live && lane == 0) p.rstd[row * p.heads + h] = rstd;
      }
    }
    if constexpr (BWD) {
      if (rot) turn<INTER, true>(u, v, cs);
    }
    if (live) {
      const long at = row * p.o_row + (long)h * p.o_head;
      store8<BF>(p.out, at + e1, u);
      store8<BF>(p.out, at + e2, v);
    }
  }
}

using Kernel = void (*)(RopeAxesDev);
template <bool B, bool I>
Kernel pick(bool norm, bool bwd) {
  if (norm) return bwd ? (Kernel)rope_axes_kernel<B, I, true, true> : (Kernel)rope_axes_kernel<B, I, true, false>;
  return bwd ? (Kernel)rope_axes_kernel<B, I, false, true> : (Kernel)rope_axes_kernel<B, I, false, false>;
}

}  // namespace

int rope_axes(const RopeAxesParams& p, const int* axis_pairs, const double* bases, bool x_bf16, bool interleaved,
              bool norm, bool bwd, hipStream_t s) {
  FLITE_REQUIRE(p.dim > 0 && p.dim % 16 == 0 && p.dim <= 256, "rope_axes: head size must be a multiple of 16, at most 256");
  FLITE_REQUIRE(p.axes >= 1 && p.axes <= 8, "rope_axes: 1 to 8 axes");
  RopeAxesDev d;
  d.p = p;
  int n = 0;
  for (int a = 0; a < p.axes; ++a) {
    FLITE_REQUIRE(axis_pairs[a] >= 0 && axis_pairs[a] <= p.dim / 2 - n, "rope_axes: more pairs than the head holds");
    FLITE_REQUIRE(bases[a] > 0.0 && std::isfinite(bases[a]), "rope_axes: bases must be positive");
    // base^(-i / n) as a product of two powers, 3 ulp: a pow per pair would cost more host time than the launch
    double low[8], high = 0.;
    for (int i = 0; i < std::min(axis_pairs[a], 8); ++i) low[i] = pow(bases[a], -(double)i / axis_pairs[a]);
    for (int i = 0; i < axis_pairs[a]; ++i, ++n) {
      if (i % 8 == 0) high = pow(bases[a], -(double)i / axis_pairs[a]) * 0.15915494309189533577;  // 1 / (2 pi)
      d.turns[n] = high * low[i % 8];
      d.axis[n] = (unsigned char)a;
    }
  }
  d.pairs = n;
  FLITE_REQUIRE(n % 8 == 0 && n > 0, "rope_axes: the pairs of all axes must add up to a multiple of 8");
  FLITE_REQUIRE(p.rows >= 0 && p.heads > 0 && p.rope_heads >= 0 && p.rope_heads <= p.heads,
                "rope_axes: rows >= 0, heads > 0 and 0 <= rope_heads <= heads");
  if (p.rows == 0) return 0;
  FLITE_REQUIRE(p.positions && p.tokens > 0, "rope_axes: positions missing");
  FLITE_REQUIRE(p.x && p.out && ((uintptr_t)p.x & 15) == 0 && ((uintptr_t)p.out & 15) == 0 && p.x_row % 8 == 0 &&
                    p.x_head % 8 == 0 && p.o_row % 8 == 0 && p.o_head % 8 == 0,
                "rope_axes: tensors must be 16-byte aligned, their row and head strides multiples of 8");
  FLITE_REQUIRE(!norm || p.rstd, "rope_axes: the norm needs rstd");
  FLITE_REQUIRE(!(norm && bwd) || (p.y && ((uintptr_t)p.y & 15) == 0 && p.y_row % 8 == 0 && p.y_head % 8 == 0),
                "rope_axes: the norm's backward pass needs the forward pass's 16-byte aligned output");
  d.lanes_lg = 0;
  while ((16 << d.lanes_lg) < p.dim) ++d.lanes_lg;
  const int groups = kThreads >> d.lanes_lg;
  d.rows_lg = 0;
  while ((1 << d.rows_lg) < groups && ((long)p.heads << d.rows_lg) < groups) ++d.rows_lg;
  const long blocks = (p.rows + (1 << d.rows_lg) - 1) >> d.rows_lg;
  FLITE_REQUIRE(blocks <= 0x7fffffffL, "rope_axes: too many rows");
  const size_t lds = (size_t)(d.pairs << d.rows_lg) * sizeof(f32x2);
  const dim3 grid((unsigned)blocks), block(kThreads);
  const Kernel k = x_bf16 ? (interleaved ? pick<true, true>(norm, bwd) : pick<true, false>(norm, bwd))
                          : (interleaved ? pick<false, true>(norm, bwd) : pick<false, false>(norm, bwd));
  hipLaunchKernelGGL(k, grid, block, lds, s, d);
  FLITE_HIP_CHECK(hipGetLastError());
  return 0;
}

}  // namespace flite
