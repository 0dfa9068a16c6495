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
// keeps nothing), dx is written once. A wave holds a row of up to 3072 columns, 8 consecutive ones a lane and chunk (16-B
// bf16 accesses), so that its sums need neither LDS nor barriers; longer rows take two or four waves. A workgroup of four
// waves walks over a strip of rows, the next row of each wave on its way, and keeps what the rows share in LDS.
// Measured at 8224 x 3072 bf16, two segments: forward 24.8 us (101 MB, 4.1 TB/s; a workgroup per row, which reads the
// shared rows anew, 32.4), backward 37 us (151 MB, 4.1 TB/s; a workgroup per row at a time 59.6, four at a time 66) and
// 8.4 for the sums of its 12.6 MB of partial sums. A large copy reaches 5.2 TB/s.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace flite {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxDim = 8192;
// Workgroups wanted, and rows of a strip at least. Backward, both kernels: 256 strips 48.5 us, 384 46.5, 512 46.2, 1024 57
// (each strip writes 2 D partial sums, which the second kernel reads); forward 256 to 2056: the same.
constexpr int kFwdStrips = 1024, kBwdStrips = 512, kBwdRows = 8;

struct NormTrainDev {
  NormTrainParams p;
  int strips;      // row strips per segment
  int strip_rows;  // rows per strip
  int row_waves;   // waves per row: 1, 2 or 4
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

// Eight values as they lie in memory
template <bool BF>
struct Raw8 {
  u32x4 w[BF ? 1 : 2];
  __device__ __forceinline__ void load(const void* base, long off) {
    const char* at = (const char*)base + off * (BF ? 2 : 4);
    w[0] = *(const u32x4*)at;
    if constexpr (!BF) w[1] = *(const u32x4*)(at + 16);
  }
  __device__ __forceinline__ void zero() {
    w[0] = u32x4{0, 0, 0, 0};
    if constexpr (!BF) w[1] = w[0];
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (BF)
      return __uint_as_float(j & 1 ? w[0][j >> 1] & 0xffff0000u : w[0][j >> 1] << 16);
    else
      return __uint_as_float(w[j >> 2][j & 3]);
  }
};

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

// Sum over a wave, the same on every lane: neighbours, pairs, quads and rows of 16 by lane moves of the vector unit (a
// shuffle through LDS takes several times as long)
template <int CTRL>
__device__ __forceinline__ float lanes(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum64(float v) {
  v += lanes<0xB1>(v);   // lane ^ 1
  v += lanes<0x4E>(v);   // lane ^ 2
  v += lanes<0x141>(v);  // mirrored within 8
  v += lanes<0x140>(v);  // mirrored within 16
  auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// A thread's place: its row group of the workgroup, its place in the row
struct Place {
  int group, groups, t, threads;  // threads: per row
  __device__ __forceinline__ Place(int row_waves) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    groups = kWaves / row_waves;
    group = wave / row_waves;
    threads = 64 * row_waves;
    t = threadIdx.x - group * threads;
  }
  __device__ __forceinline__ int col(int c) const { return (c * threads + t) * 8; }
};

// Sums of N values over the row's threads, the same on each. Rows of several waves go through N LDS slots a wave;
// consecutive calls alternate between two buffers, so one barrier per call is enough (a wave can be at most one call ahead
// of the slowest reader). All waves of the workgroup make the same calls.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* buf, int row_waves) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = sum64(v[i]);
  if (row_waves == 1) return;
  const int wave = threadIdx.x >> 6, first = wave & ~(row_waves - 1);
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[wave * N + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int w = 0; w < row_waves; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += buf[(first + w) * N + i];
}

// Eight columns of a table in LDS: two planes of 16 B a lane, without bank conflicts
struct Table {
  float* base;
  int threads, t;
  __device__ __forceinline__ f32x4* at(int c, int half) const { return (f32x4*)base + (2 * c + half) * threads + t; }
  __device__ __forceinline__ void put(int c, const float (&v)[8]) const {
    *at(c, 0) = f32x4{v[0], v[1], v[2], v[3]};
    *at(c, 1) = f32x4{v[4], v[5], v[6], v[7]};
  }
  __device__ __forceinline__ void get(int c, float (&v)[8]) const {
    const f32x4 a = *at(c, 0), b = *at(c, 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  }
};

// Rows r0 .. r1 of the workgroup's strip
struct Strip {
  long seg, r0, r1;
  __device__ __forceinline__ explicit Strip(const NormTrainDev& d) {
    const NormTrainParams& p = d.p;
    seg = blockIdx.x / d.strips;
    const long seg_rows = p.seg_rows > 0 ? p.seg_rows : p.rows;
    r0 = seg * seg_rows + (long)(blockIdx.x % d.strips) * d.strip_rows;
    r1 = min(min(r0 + d.strip_rows, (seg + 1) * seg_rows), p.rows);
  }
};

// a = w (1 + scale) of the eight columns at col
__device__ __forceinline__ void factor8(const NormTrainParams& p, long seg, int col, float (&a)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = 1.f;
  if (p.w) load8<true>(p.w, col, a);
  if (p.scale) {
    float t[8];
    load8<false>(p.scale, seg * p.mod_seg_stride + col, t);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] *= 1.f + t[j];
  }
}

// ---- forward: y = n a + c with a = w (1 + scale) and c = b (1 + scale) + shift of the segment ----
template <bool XBF, int NCH>
__global__ __launch_bounds__(kThreads) void layernorm_mod_kernel(NormTrainDev d) {
  extern __shared__ __attribute__((aligned(16))) float smem[];
  __shared__ float buf[2][kWaves];
  const NormTrainParams& p = d.p;
  const Place at(d.row_waves);
  const Strip st(d);
  if (st.r0 >= st.r1) return;
  const Table ta{smem, at.threads, at.t}, tc{smem + at.threads * NCH * 8, at.threads, at.t};

  Raw8<XBF> nx[NCH];
  auto fetch = [&](long row) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (at.col(c) < p.D)
        nx[c].load(p.x, row * p.ldx + at.col(c));
      else
        nx[c].zero();
    }
  };
  fetch(min(st.r0 + at.group, st.r1 - 1));
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = at.col(c);
    if (c % at.groups != at.group || col >= p.D) continue;  // the groups share the work
    float a[8], b[8], t[8];
    factor8(p, st.seg, col, a);
    ta.put(c, a);
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = 0.f;
    if (p.b) {
      load8<true>(p.b, col, b);
      if (p.scale) {
        load8<false>(p.scale, st.seg * p.mod_seg_stride + col, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] *= 1.f + t[j];
      }
    }
    if (p.shift) {
      load8<false>(p.shift, st.seg * p.mod_seg_stride + col, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] += t[j];
    }
    tc.put(c, b);
  }
  __syncthreads();
  const float inv_d = 1.f / (float)p.D;
  for (long first = st.r0; first < st.r1; first += at.groups) {
    const long row = first + at.group;
    Raw8<XBF> x[NCH];
    float s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      x[c] = nx[c];
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += x[c].get(j);
    }
    if (first + at.groups < st.r1) fetch(min(row + at.groups, st.r1 - 1));
    row_sums<1>(s, buf[0], d.row_waves);
    const float mean = s[0] * inv_d;
    s[0] = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const bool live = at.col(c) < p.D;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = live ? x[c].get(j) - mean : 0.f;
        s[0] += v * v;
      }
    }
    row_sums<1>(s, buf[1], d.row_waves);
    const float r = 1.f / sqrtf(s[0] * inv_d + p.eps);
    if (row >= st.r1) continue;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (at.col(c) >= p.D) continue;
      float a[8], b[8], y[8];
      ta.get(c, a);
      tc.get(c, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = (x[c].get(j) - mean) * r * a[j] + b[j];
      store8<true>(p.y, row * p.ldy + at.col(c), y);
    }
  }
}

// ---- backward: S0 and S1 of the strip to the workspace ----
// (two waves a SIMD for bf16: with one, where it takes 264 registers, 8224 x 3072 take 56 us in place of 46)
template <bool XBF, bool RMS, int NCH, bool SUMS>
__global__ __launch_bounds__(kThreads, XBF ? 2 : 1) void norm_bwd_kernel(NormTrainDev d) {
  extern __shared__ __attribute__((aligned(16))) float smem[];
  __shared__ float buf[2][kWaves * 3];
  const NormTrainParams& p = d.p;
  const Place at(d.row_waves);
  const Strip st(d);
  const Table ta{smem, at.threads, at.t};

  Raw8<XBF> nx[NCH];
  Raw8<true> ndy[NCH];
  auto fetch = [&](long row) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (at.col(c) < p.D) {
        nx[c].load(p.x, row * p.ldx + at.col(c));
        ndy[c].load(p.dy, row * p.lddy + at.col(c));
      } else {
        nx[c].zero();
        ndy[c].zero();
      }
    }
  };
  if (st.r0 < st.r1) fetch(min(st.r0 + at.group, st.r1 - 1));
  float s0[NCH][8], s1[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s0[c][j] = s1[c][j] = 0.f;
    if (c % at.groups != at.group || at.col(c) >= p.D) continue;  // the groups share the work
    float a[8];
    factor8(p, st.seg, at.col(c), a);
    ta.put(c, a);
  }
  __syncthreads();
  const float inv_d = 1.f / (float)p.D;
  int turn = 0;
  for (long first = st.r0; first < st.r1; first += at.groups) {
    const long row = first + at.group;
    Raw8<XBF> x[NCH];
    Raw8<true> dy[NCH];
    float mean = 0.f, m[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      x[c] = nx[c];
      dy[c] = ndy[c];
      if constexpr (!RMS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) m[0] += x[c].get(j);
      }
    }
    if (first + at.groups < st.r1) fetch(min(row + at.groups, st.r1 - 1));
    if constexpr (!RMS) {
      row_sums<1>(m, buf[turn], d.row_waves);
      turn ^= 1;
      mean = m[0] * inv_d;
    }
    float s[3] = {0.f, 0.f, 0.f};  // sum (x - mean)^2, sum g, sum g (x - mean)
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const bool live = at.col(c) < p.D;
      float a[8];
      if (live) {
        ta.get(c, a);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = x[c].get(j) - mean;
          const float g = dy[c].get(j) * a[j];
          s[0] += v * v;
          if constexpr (!RMS) s[1] += g;
          s[2] += g * v;
        }
      }
    }
    row_sums<3>(s, buf[turn], d.row_waves);
    turn ^= 1;
    if (row >= st.r1) continue;
    const float r = 1.f / sqrtf(s[0] * inv_d + p.eps);
    const float c1 = RMS ? 0.f : s[1] * inv_d;
    const float c2 = s[2] * inv_d * r;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (at.col(c) >= p.D) continue;
      float a[8], o[8];
      ta.get(c, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = (x[c].get(j) - mean) * r, g = dy[c].get(j);
        if constexpr (SUMS) {
          s0[c][j] += g;
          s1[c][j] += g * n;
        }
        o[j] = r * (g * a[j] - c1 - n * c2);
      }
      store8<XBF>(p.dx, row * p.lddx + at.col(c), o);
    }
  }
  if constexpr (SUMS) {
    // the groups' sums, in group order, through the table's place
    for (int g = 1; g < at.groups; ++g) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __syncthreads();
        if (at.group == g) {
#pragma unroll
          for (int c = 0; c < NCH; ++c) ta.put(c, k ? s1[c] : s0[c]);
        }
        __syncthreads();
        if (at.group == 0) {
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            float v[8];
            ta.get(c, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) (k ? s1[c][j] : s0[c][j]) += v[j];
          }
        }
      }
    }
    if (at.group != 0) return;
    float* ws = p.ws + (long)blockIdx.x * 2 * p.D;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (at.col(c) >= p.D) continue;
      store8<false>(ws, at.col(c), s0[c]);
      store8<false>(ws, p.D + at.col(c), s1[c]);
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

// Waves per row and chunks per lane (1, 2, 4 or 6)
struct Shape {
  int row_waves, chunks, table;  // table: bytes of one table
};
Shape shape_of(int D) {
  Shape x;
  x.row_waves = D <= 64 * 48 ? 1 : D <= 128 * 48 ? 2 : 4;
  const int need = (D + 512 * x.row_waves - 1) / (512 * x.row_waves);
  x.chunks = need <= 2 ? need : need <= 4 ? 4 : 6;
  x.table = 64 * x.row_waves * x.chunks * 8 * 4;
  return x;
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

// Strips of one segment each: `want` workgroups in all, none under `least` rows
void plan(const NormTrainParams& p, int wanted, int least, long* segs, int* strips, int* strip_rows) {
  const long seg_rows = p.seg_rows > 0 ? std::min(p.seg_rows, p.rows) : p.rows;
  *segs = p.rows > 0 ? (p.rows + seg_rows - 1) / seg_rows : 0;
  if (*segs == 0) {
    *strips = *strip_rows = 0;
    return;
  }
  const long want = std::max(1L, wanted / *segs);
  const long most = std::max(1L, (seg_rows + least - 1) / least);
  const long n = std::min(want, most);
  *strip_rows = (int)((seg_rows + n - 1) / n);
  *strips = (int)((seg_rows + *strip_rows - 1) / *strip_rows);
}

using Kernel = void (*)(NormTrainDev);
template <bool X, bool R, bool S>
Kernel pick(int chunks) {
  return chunks == 1   ? (Kernel)norm_bwd_kernel<X, R, 1, S>
         : chunks == 2 ? (Kernel)norm_bwd_kernel<X, R, 2, S>
         : chunks == 4 ? (Kernel)norm_bwd_kernel<X, R, 4, S>
                       : (Kernel)norm_bwd_kernel<X, R, 6, S>;
}
template <bool X>
Kernel pick(int chunks, bool rms, bool sums) {
  if (rms) return sums ? pick<X, true, true>(chunks) : pick<X, true, false>(chunks);
  return sums ? pick<X, false, true>(chunks) : pick<X, false, false>(chunks);
}
template <bool X>
Kernel pick_fwd(int chunks) {
  return chunks == 1   ? (Kernel)layernorm_mod_kernel<X, 1>
         : chunks == 2 ? (Kernel)layernorm_mod_kernel<X, 2>
         : chunks == 4 ? (Kernel)layernorm_mod_kernel<X, 4>
                       : (Kernel)layernorm_mod_kernel<X, 6>;
}

}  // namespace

long norm_bwd_workspace_bytes(long rows, long seg_rows, int D) {
  if (rows <= 0 || D <= 0 || seg_rows < 0) return 0;
  NormTrainParams p;
  p.rows = rows;
  p.seg_rows = seg_rows;
  long segs;
  int strips, strip_rows;
  plan(p, kBwdStrips, kBwdRows, &segs, &strips, &strip_rows);
  return segs * strips * 2 * D * 4;
}

int layernorm_mod(const NormTrainParams& p, bool x_bf16, hipStream_t s) {
  if (int rc = check_common(p)) return rc;
  FLITE_REQUIRE((p.y || p.rows == 0) && ((uintptr_t)p.y & 15) == 0 && p.ldy % 8 == 0 && p.ldy >= p.D,
                "layernorm: y must be 16-byte aligned rows, their stride a multiple of 8 and at least dim");
  if (p.rows == 0) return 0;
  const Shape x = shape_of(p.D);
  NormTrainDev d;
  d.p = p;
  d.row_waves = x.row_waves;
  long segs;
  plan(p, kFwdStrips, kWaves / x.row_waves, &segs, &d.strips, &d.strip_rows);
  FLITE_REQUIRE(segs * d.strips <= 0x7fffffffL, "layernorm: too many segments");
  const Kernel k = x_bf16 ? pick_fwd<true>(x.chunks) : pick_fwd<false>(x.chunks);
  if (2 * x.table > 48 * 1024)
    FLITE_HIP_CHECK(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * x.table));
  hipLaunchKernelGGL(k, dim3((unsigned)(segs * d.strips)), dim3(kThreads), 2 * x.table, s, d);
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
  plan(p, kBwdStrips, kBwdRows, &segs, &d.strips, &d.strip_rows);
  FLITE_REQUIRE(!sums || p.rows == 0 || (p.ws && ((uintptr_t)p.ws & 15) == 0 &&
                                         p.ws_bytes >= norm_bwd_workspace_bytes(p.rows, p.seg_rows, p.D)),
                "norm backward: workspace missing or too small");
  FLITE_REQUIRE(segs * d.strips <= 0x7fffffffL, "norm backward: too many segments");
  if (p.rows > 0) {
    const Shape x = shape_of(p.D);
    d.row_waves = x.row_waves;
    const Kernel k = x_bf16 ? pick<true>(x.chunks, rms, sums) : pick<false>(x.chunks, rms, sums);
    hipLaunchKernelGGL(k, dim3((unsigned)(segs * d.strips)), dim3(kThreads), x.table, s, d);
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
