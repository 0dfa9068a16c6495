// Attention for training on gfx950: the forward pass that keeps its log-sum-exp, and the backward pass that makes the
// probabilities again from it. Packed sequences (cu_seqlens), no mask, head sizes 64, 128 and 256, bf16, K/V heads
// shared by groups of query heads.
//
//   S = scale q k^T, lse = log sum exp S, P = exp(S - lse), out = P v
//   delta = sum_d dout * out,  dP = dout v^T,  dS = P * (dP - delta)
//   dv = P^T dout,  dk = scale dS^T q,  dq = scale dS k
//
// Forward: a workgroup owns 256 queries of one head and sweeps the keys, two products; where units are few or long, the
// sweeps are cut into ranges and joined (attn_lse_kernel).
//
// Backward = three launches. (1) delta and lse * log2(e) per query row, and the work list. (2) Two kinds of workgroups in
// one launch: a "key" workgroup owns 128 keys of one K/V head and sweeps the queries of its group of heads (4 products:
// S, dP, dv, dk); a "query" workgroup owns 128 queries of one head and sweeps the keys (S, dP, and dq twice: its dS counts
// in two bf16 parts). That is 8 products, where 5 would do if S and dP were made once; in return every gradient is summed
// by one workgroup in registers, in a fixed order: no atomics, no fp32 dq in memory. (3) Where too few workgroups would
// run, the sweeps are cut into ranges whose fp32 partial gradients a last kernel adds in range order.
//
// Two waves share 64 of the workgroup's rows ("stationary": fragments in registers, row on the lane) and split the
// products between them: an accumulator of 64 x 256 takes 256 registers, so a wave of its 512 holds one. They read tiles
// of 32 swept rows from LDS, where copies bring them several steps ahead: row-wise (ds_read_b128, A operand of S and dP)
// and transposed (ds_read_b64_tr_b16, A operand of the gradients); P and dS go straight into the B operand of their own
// wave, and through LDS to the other.
//
// Bound by the matrix cores. Measured: backward of 2 x 4112 tokens, 12 heads of 256 (8 products, 1.66 TFLOP): 1340 us =
// 1.24 PFLOP/s, where an 8192^3 matrix product reaches 1.38 and the card lowers its clock under either. With head size 128
// (4 x 4096 tokens, 16 heads) 1921 us = 1.14 PFLOP/s, with 64 1490 us = 0.74: the scores' exp2 and products take as long
// as the MFMAs there. Forward, two products: 390 us = 1.07, 510 = 1.08 and 325 = 0.85 PFLOP/s.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "attn_common.h"
#include "common.h"
#include "kernels.h"

namespace flite {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
// The backward pass works with 2^15 P (and 2^15 dS), taken back when the gradients are stored: P goes from wave to wave
// in fp16 (2^-12, against the 2^-9 of the rounding that follows), where 2^15 P <= 2^15 fits and stays normal down to
// P = 2^-29.
constexpr float kShift = 15.f, kUnshift = 1.f / 32768.f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int WROWS = 128;  // stationary rows of a workgroup
constexpr int kThreads = 256;
constexpr int kMaxRanges = 16;
constexpr int kMinRange = 8;  // stages: what a workgroup's start and end cost
constexpr int kCus = 256;
constexpr int kFullShare = 2;  // ranges of full tiles that make up a CU's share of the work, where little else fills it

// How a launch cuts its work. A unit is one 128-row tile ("full", or the rest of a sequence, "part") of one head with
// its whole sweep; where units are few or long, a sweep is cut into ranges, whose fp32 partial gradients a last kernel
// adds in range order.
struct Cut {
  int full;            // upper bound of the batch's full tiles
  int heads;
  int max_full, max_part;  // ranges that the workspace has room for
  float* ws_full;      // [max_full][total][heads][D], with max_full > 1
  float* ws_part;      // [max_part][B][128][heads][D], with max_part > 1
  __host__ __device__ int full_blocks() const { return full * heads * max_full; }
  __host__ __device__ int blocks(int B) const { return full_blocks() + B * heads * max_part; }
};

struct TrainDev {
  AttnTrainParams p;
  // forward
  int tiles;               // upper bound of the 256-row tiles
  int most, stages;        // ranges of a sweep, at most; stages of a range
  float* part_o;           // [most][total_q][H][D] with most > 1: sums of 2^(S - m) v
  float2* part_ml;         // [most][H][total_q]: m and the sum of 2^(S - m), S in units of log2
  int* starts;             // [B + 1] units of a head before each sequence, for batches of more than 64
  // backward
  Cut q, k;
  int* target;             // stages per range: of a full tile, of a part; [2]: groups, [3]: blocks that have work
  int4* groups;            // [4 B] (Group)
  float* lse2;             // [H][total_q] lse * log2 e - kShift
  float* delta;            // [H][total_q]
};

// One sequence's rows [start, start + len) of `total`, from a cumulative array that a caller may have filled wrongly:
// clamped, so that nothing outside the tensors is touched.
__device__ __forceinline__ void seq_range(const int* cu, int b, int total, int* start, int* len) {
  const int s = min(max(cu[b], 0), total);
  const int e = min(max(cu[b + 1], s), total);
  *start = s;
  *len = e - s;
}

// Sequence that holds `row`, -1: none
__device__ __forceinline__ int find_seq(const int* cu, int B, int total, int row) {
  int lo = 0, hi = B;  // the last b with cu[b] <= row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (cu[mid] <= row ? lo : hi) = mid;
  }
  int s, len;
  seq_range(cu, lo, total, &s, &len);
  return row >= s && row < s + len ? lo : -1;
}

// Ranges of a sweep of `stages`
__device__ __forceinline__ int ranges_of(int stages, int target, int most) {
  return min(max((stages + target - 1) / target, 1), most);
}

// The last of `start`'s n ascending entries (STEP ints apart) that is at most v; start[0] is. A wave looks at 64 at a time.
template <int STEP>
__device__ __forceinline__ int last_at_most(const int* start, int n, int v) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const int found = __popcll(__ballot(at < hi && start[(long)min(at, hi - 1) * STEP] <= v));
    lo += max(found - 1, 0) * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

// The backward pass's work list: groups of equal units (the full tiles of a sequence, or its part, as keys or as queries),
// the longest ranges first. Made on the device, which alone knows the lengths; the launch has an upper bound of blocks.
struct Group {
  static constexpr int PART = 1, QUERY = 2;
  static __device__ int4 make(int first, int b, int kind, int ranges, int tiles) {
    return make_int4(first, b * 4 + kind, ranges, tiles);
  }
};
// One unit and range of the sweep over it
struct Unit {
  int b, h, tile, part, ranges;
  bool full, query;
};
// Block v -> its unit; false: nothing to do
__device__ __forceinline__ bool find_unit(const TrainDev& d, int v, Unit* u) {
  const int n = d.target[2], blocks = d.target[3];
  if (v >= blocks) return false;
  const int e = __builtin_amdgcn_readfirstlane(last_at_most<4>((const int*)d.groups, n, v));
  const int4 g = d.groups[e];
  const int size = (e + 1 < n ? d.groups[e + 1].x : blocks) - g.x;
  u->ranges = g.z;
  u->b = g.y >> 2;
  u->full = !(g.y & Group::PART);
  u->query = (g.y & Group::QUERY) != 0;
  v = xcd_remap(v - g.x, size);  // neighbours in the group (tiles of a head) on one XCD
  u->part = v % g.z;
  v /= g.z;
  u->tile = v % g.w;
  u->h = v / g.w;
  return true;
}

// Row `row` of sequence b, head h, range 0 in the partial gradients; *step: floats from range to range
template <int D>
__device__ __forceinline__ float* part_row(const Cut& c, bool full, int B, int total, int start, int b, int row, int h,
                                           long* step) {
  *step = (long)(full ? total : B * WROWS) * c.heads * D;
  const long r = full ? (long)start + row : (long)b * WROWS + row % WROWS;
  return (full ? c.ws_full : c.ws_part) + (r * c.heads + h) * D;
}

// XOR of the 16-B chunk index of tile row r. The low 4 bits of a row map one to one onto the XOR (row reads of 16 lanes
// hit 16 different chunks), and rows 0..3 of a group land in different 64-B blocks (transposed reads). 128-B rows
// (D = 64): two rows share the 256 B of banks, so bit 0 of the row needs no XOR.
template <int D>
__device__ __forceinline__ int swz(int r) {
  if constexpr (D == 64)
    return ((r & 2) << 1) | ((r >> 2) & 3);
  else
    return ((r & 3) << 2) | ((r >> 2) & 3);
}

// Fragments of the stationary rows: lane (row lq, half hh) holds elements 16 s + 8 hh .. + 7
template <int D>
__device__ __forceinline__ void load_frags(const bf16_t* row, int hh, bf16x8 (&f)[D / 16]) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) f[s] = *(const bf16x8*)(row + 16 * s + 8 * hh);
}

// Scores are made of the stationary rows with the scale's sign, and scaled by its magnitude (score_scale): the largest
// product is the largest score, and a masked one, -inf, stays so. A scale of zero takes rows of zeros.
template <int D>
__device__ __forceinline__ void take_sign(bf16x8 (&f)[D / 16], float scale) {
  const unsigned keep = scale == 0.f ? 0u : ~0u, flip = scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    u32x4 w = __builtin_bit_cast(u32x4, f[s]);
    w = (w & keep) ^ flip;
    f[s] = __builtin_bit_cast(bf16x8, w);
  }
}
__device__ __forceinline__ float score_scale(float scale) { return scale == 0.f ? 1.f : fabsf(scale) * kLog2e; }

// The lane's stationary row of acc[D x rows], times f: bf16 to `dst` (the row's start)
template <int D>
__device__ __forceinline__ void store_row(bf16_t* dst, const f32x16 (&acc)[D / 32], float f, int hh, bool live) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int rp = 0; rp < 2; ++rp) {
      const int a = 8 * rp, b = 8 * rp + 4;
      const auto x0 = __builtin_amdgcn_permlane32_swap(pack2bf(acc[i][a] * f, acc[i][a + 1] * f),
                                                       pack2bf(acc[i][b] * f, acc[i][b + 1] * f), false, false);
      const auto x1 = __builtin_amdgcn_permlane32_swap(pack2bf(acc[i][a + 2] * f, acc[i][a + 3] * f),
                                                       pack2bf(acc[i][b + 2] * f, acc[i][b + 3] * f), false, false);
      const u32x4 w = {x0[0], x1[0], x0[1], x1[1]};
      if (live) *(u32x4*)(dst + i * 32 + 16 * rp + 8 * hh) = w;
    }
}

// the same as an fp32 partial
template <int D>
__device__ __forceinline__ void store_part(float* dst, const f32x16 (&acc)[D / 32], float f, int hh, bool live) {
  if (!live) return;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4)
      *(f32x4*)(dst + i * 32 + 8 * r4 + 4 * hh) =
          f32x4{acc[i][4 * r4] * f, acc[i][4 * r4 + 1] * f, acc[i][4 * r4 + 2] * f, acc[i][4 * r4 + 3] * f};
}

// Zeros (lse: -inf) in the rows before the first and behind the last sequence, by `blocks` workgroups of which this is
// number i
__device__ __forceinline__ void zero_outside(bf16_t* out, long row_stride, long head_stride, const int* cu, int B, int total,
                                             int H, int D, float* lse, int i, int blocks) {
  const int first = min(max(cu[0], 0), total), behind = min(max(cu[B], first), total);
  const long n = (long)(first + total - behind) * H * (D / 8);
  for (long e = (long)i * kThreads + threadIdx.x; e < n; e += (long)blocks * kThreads) {
    const int c = (int)(e % (D / 8)) * 8, h = (int)(e / (D / 8) % H), r = (int)(e / (D / 8) / H);
    const int row = r < first ? r : behind + r - first;
    *(u32x4*)(out + (long)row * row_stride + (long)h * head_stride + c) = u32x4{0u, 0u, 0u, 0u};
    if (lse != nullptr && c == 0) lse[(long)h * total + row] = -INFINITY;
  }
}

// ------------------------------------------------------------------------------------------------ backward
// One workgroup: the ranges' lengths and the work list
__device__ __forceinline__ void make_groups(const TrainDev& d) {
  const AttnTrainParams& p = d.p;
  __shared__ double sums[kThreads / 64];
  __shared__ int cost[kThreads], count[kThreads], waves[kThreads / 64];
  const int tid = threadIdx.x;
  // Stages of all units, over the CUs: a range of a full tile is at most half of a CU's share of them, one of a part (they
  // fill the end of the launch) a 32nd; none is shorter than kMinRange. Where units of under a third of the share make up a
  // third of the work, they fill what longer ranges leave open, and ranges are as long as the share: fewer partial
  // gradients (4112 queries on 512 and 77 keys, 12 heads of 256: 210 -> 188 us; a ragged batch with long units alone took
  // 147 us in place of 126).
  auto total = [&](double most) {  // stages of the units of at most `most`
    double sum = 0.;
    for (int b = tid; b < p.B; b += kThreads) {
      int s, ql, kl;
      seq_range(p.cu_q, b, p.total_q, &s, &ql);
      seq_range(p.cu_k, b, p.total_k, &s, &kl);
      const int qs = (kl + 31) / 32, ks = (ql + 31) / 32 * (p.H / p.HK);
      if (qs <= most) sum += (double)((ql + WROWS - 1) / WROWS) * qs * p.H;
      if (ks <= most) sum += (double)((kl + WROWS - 1) / WROWS) * ks * p.HK;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    __syncthreads();
    if ((tid & 63) == 0) sums[tid >> 6] = sum;
    __syncthreads();
    sum = 0.;
    for (int w = 0; w < kThreads / 64; ++w) sum += sums[w];
    return sum;
  };
  const double work = total(1e18), share = fmin(work / kCus, 1e9);
  const bool fill = share > kMinRange && total(share / 3.) > work / 3.;
  const int t_full = max((int)(fill ? share : share / kFullShare), kMinRange), t_part = max((int)(share / 32), kMinRange);
  // entry e: kind e / B (keys full, keys part, queries full, queries part) of sequence e % B
  const int n = 4 * p.B;
  int first = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int e = base + tid;
    int b = 0, kind = 0, ranges = 1, tiles = 0, blocks = 0, len = 0;
    if (e < n) {
      kind = e / p.B;
      b = e % p.B;
      const bool query = (kind & Group::QUERY) != 0, part = (kind & Group::PART) != 0;
      int s, ql, kl;
      seq_range(p.cu_q, b, p.total_q, &s, &ql);
      seq_range(p.cu_k, b, p.total_k, &s, &kl);
      const Cut& c = query ? d.q : d.k;
      const int own = query ? ql : kl, stages = ((query ? kl : ql) + 31) / 32 * (query ? 1 : p.H / p.HK);
      tiles = part ? (own % WROWS ? 1 : 0) : own / WROWS;
      ranges = ranges_of(stages, part ? t_part : t_full, part ? c.max_part : c.max_full);
      blocks = tiles * c.heads * ranges;
      len = (stages + ranges - 1) / ranges;
    }
    // rank: by length, then by number (only where all groups fit one round of threads: else they keep their order)
    int rank = tid;
    __syncthreads();
    if (n <= kThreads) {
      cost[tid] = e < n && blocks > 0 ? len : -1;
      __syncthreads();
      const int mine = cost[tid];
      rank = e < n ? 0 : tid;
      for (int i = 0; e < n && i < n; ++i) rank += cost[i] > mine || (cost[i] == mine && i < tid);
    }
    count[rank] = blocks;
    __syncthreads();
    int upto = count[tid];  // blocks of the ranks up to tid
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(upto, o, 64);
      if ((tid & 63) >= o) upto += up;
    }
    if ((tid & 63) == 63) waves[tid >> 6] = upto;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
      if (w < (tid >> 6)) upto += waves[w];
      all += waves[w];
    }
    count[tid] = upto;
    __syncthreads();
    if (e < n) d.groups[base + rank] = Group::make(first + count[rank] - blocks, b, kind, ranges, max(tiles, 1));
    first += all;
    __syncthreads();
  }
  if (tid == 0) {
    d.target[0] = t_full;
    d.target[1] = t_part;
    d.target[2] = n;
    d.target[3] = first;
  }
}

// First launch of the backward pass: lse * log2 e and delta of every query row (those outside all sequences are read by
// nobody); the work list; zeros outside. Bound by HBM: 101 MB (8224 rows, 12 heads of 256) in 23 us = 4.4 TB/s.
template <int D>
__global__ __launch_bounds__(kThreads) void attn_delta_kernel(TrainDev d, int n) {  // the first n workgroups: the rest
  const AttnTrainParams& p = d.p;
  constexpr int LANES = D / 8;
  if ((int)blockIdx.x < n) {
    const int i = blockIdx.x;
    if (i == 0) make_groups(d);
    if (p.zero_outside) {
      zero_outside(p.dq, p.dq_row, p.dq_head, p.cu_q, p.B, p.total_q, p.H, D, nullptr, i, n);
      zero_outside(p.dk, p.dk_row, p.dk_head, p.cu_k, p.B, p.total_k, p.HK, D, nullptr, i, n);
      zero_outside(p.dv, p.dv_row, p.dv_head, p.cu_k, p.B, p.total_k, p.HK, D, nullptr, i, n);
    }
    return;
  }
  const long item = ((long)(blockIdx.x - n) * kThreads + threadIdx.x) / LANES;
  const int c = threadIdx.x % LANES;
  if (item >= (long)p.total_q * p.H) return;
  const int row = (int)(item / p.H), h = (int)(item % p.H);
  const bf16x8 a = *(const bf16x8*)(p.dout + (long)row * p.do_row + (long)h * p.do_head + 8 * c);
  const bf16x8 b = *(const bf16x8*)(p.o + (long)row * p.o_row + (long)h * p.o_head + 8 * c);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s += (float)a[j] * (float)b[j];
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) s += __shfl_xor(s, o, 64);
  if (c == 0) {
    const long at = (long)h * p.total_q + row;
    const float lse = p.lse[at];
    // a row without keys (or with -inf scores alone) has P = 0: exp2(x - inf)
    d.lse2[at] = lse == -INFINITY ? INFINITY : lse * kLog2e - kShift;
    d.delta[at] = s;
  }
}

// Two kinds of waves. A wave with 32 stationary rows would read every LDS byte for one MFMA; with 64 rows the gradients
// take twice the registers. So the waves of a pair share 64 stationary rows (two blocks of 32) and split the products:
// each A fragment read from LDS feeds both blocks.
//   key workgroup:   wave 0: S, P, dv    wave 1: dP, dS = P (dP - delta), dk      (P handed over)
//   query workgroup: wave 0: S, dP, dS   wave 1: dq                               (dS handed over)
// All four have 64 MFMAs per 32 swept rows. dS enters dq as a bf16 pair hi + lo (2^-17): its rows sum to 0, so where
// keys share a direction, that direction cancels in dq and a single rounding's error would stay (dq 1.7 times as far
// from the exact gradient as one final rounding to bf16 is, against 1.4 for dk and dv).
//
// Everything is made a step (32 swept rows) or more ahead, so that between two barriers no wave waits: a step's tiles
// have been in LDS before its barrier, the first fragments of a step are read where MFMAs cover them, scores are turned
// into P or dS in the step after their products. Measured (one sequence of 4096, 4 heads): 3140 cycles a step of a key
// workgroup and 2710 of a query workgroup with D = 256, of which the MFMAs take 2048; 2090 and 1770 with D = 128 (1024),
// 1650 and 1400 with 64 (512). The scores' vector work, about 900 cycles, hides behind D = 256's MFMAs; what is left is
// the barrier and the waits on LDS and on copies around it. A workgroup starts in 5.1 us with D = 128 and 7.5 with 256
// (stationary rows: 32 rows a load, 32 B of each) and ends in 3.5 and 9. Of a whole launch shorter waits give back less:
// the card lowers its clock under this load (query steps 6 % shorter: 2 x 4112 tokens 1349 -> 1330 us).

// Steps that a copy may take beyond the one it is issued in. A copy takes 1.2 to 2 us (L2 or HBM), a step 1.6 us with
// D = 256, 1.0 with 128 and 0.8 with 64, and LDS has room for more stages where they are small. Without one more a step of
// D = 64 takes 3 % longer (4 x 4096 tokens, 16 heads: 1550 us against 1500), with four as long; D = 128: 1 to 3 alike.
template <int D>
constexpr int kExtra = D == 256 ? 0 : D == 128 ? 2 : 1;

template <int D>
struct Stage {
  static constexpr int BYTES = 32 * D * 2;      // 32 swept rows
  static constexpr int PIECES = D / 64;         // 1-KiB copies per wave: pieces wave, wave + 4, ...
  static constexpr int ROWS = 1024 / (D * 2);   // rows of a piece
  int voff[PIECES > 1 ? 2 : 1];                 // this lane's source bytes, even and odd pieces (less the rows before)
  int step;                                     // bytes of 4 pieces' rows
  __device__ __forceinline__ void init(long stride, int wave, int lane) {
    constexpr int CPR = D / 8;
    step = (int)(4 * ROWS * stride * 2);
#pragma unroll
    for (int i = 0; i < (PIECES > 1 ? 2 : 1); ++i) {
      const int row = wave * ROWS + lane / CPR;  // 4 pieces further: the same XOR but for bit 3 of the row
      voff[i] = (int)(row * stride * 2) + (((lane % CPR) ^ swz<D>(row + 4 * ROWS * i)) << 4);
    }
  }
  __device__ __forceinline__ unsigned src(int i) const { return (unsigned)(voff[PIECES > 1 ? i & 1 : 0] + i * step); }
  static __device__ __forceinline__ unsigned dst(int i) { return i * 4096; }
};

// Buffer range of the rows left in a sequence (0: the stage becomes zeros)
__device__ __forceinline__ unsigned rows_bytes(int rows_left, long stride) {
  return (unsigned)min((long)max(rows_left, 0) * stride * 2, 0x7fffffffL);
}

// LDS copies, 16 B or 4 B per lane (0 where voff is past the range). Inline asm for the reason given at blds16
// (attn_common.h): the compiler would wait for a builtin copy before every later LDS read. m0 is named as clobbered
// instead of kept: two scalar instructions fewer per copy.
__device__ __forceinline__ void copy16(const i32x4& rsrc, unsigned voff, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(voff), "s"(rsrc), "s"(lds_addr)
               : "memory", "m0");
}
__device__ __forceinline__ void copy4(const i32x4& rsrc, unsigned voff, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
               :
               : "v"(voff), "s"(rsrc), "s"(lds_addr)
               : "memory", "m0");
}

// A stream of 32-row stages over a tensor: descriptor of the next one, zeros after the last. One head's rows [0, len)
// follow those of the head before; all in scalar registers.
struct Stream {
  i32x4 rs;          // descriptor of the current stage
  const char* ptr;   // first byte of the next one
  int left;          // rows from there to the sequence end
  int stages;        // stages that are still to come
  int len, row_b;    // rows of a sequence, bytes of a row
  long step, wrap;   // bytes to the next stage, and what moves past a head's last stage to the next head's first
  // len > 0; the first stage is number t of the sweep, `stages` follow
  __device__ __forceinline__ void init(const void* base, int t, int tiles, int len_, int stages_, long row_bytes,
                                       long head_bytes) {
    const int h = t / tiles, r = (t - h * tiles) * 32;
    len = len_;
    row_b = (int)row_bytes;
    left = len - r;
    stages = stages_;
    step = 32 * row_bytes;
    wrap = head_bytes - (long)(tiles - 1) * step;
    ptr = (const char*)base + (long)h * head_bytes + (long)r * row_bytes;
  }
  // rows_of: bytes per row that the range counts (the whole stride: offsets are row * stride + column)
  __device__ __forceinline__ void next() {
    const int live = stages > 0 ? min(left, 32) : 0;
    rs = make_rsrc(ptr, (unsigned)(live * row_b));
    --stages;
    left -= 32;
    const bool w = left <= 0;
    ptr += stages > 0 ? (w ? wrap : step) : 0;
    left = w ? len : left;
  }
};

// Slots of a ring of N stages, in bytes: where a copy goes, or what moves a reader on
template <int N, int BYTES>
struct Ring {
  int at;
  __device__ __forceinline__ void next() {
    at += BYTES;
    at = at == N * BYTES ? 0 : at;
  }
  __device__ __forceinline__ int move() {
    at += BYTES;
    const bool end = at == N * BYTES;
    at = end ? 0 : at;
    return end ? (1 - N) * BYTES : BYTES;
  }
};

// The step barrier: own LDS writes done, own copies but the last N (those of the last kExtra steps); then everyone's
template <int N = 0>
__device__ __forceinline__ void step_sync() {
  static_assert(N < 64, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// LDS addresses of a lane's reads in a stage, moved along from stage to stage in place (no registers for sums); k-steps
// s >= 8 and column tiles dt >= 4 are 256 B further (the XOR stays within 16 chunks)
template <int D>
struct RowReader {
  static constexpr int NR = D / 16 < 8 ? D / 16 : 8;
  unsigned at[NR];
  __device__ __forceinline__ void init(int lane, unsigned st) {
    const int lq = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int s = 0; s < NR; ++s) at[s] = st + lq * D * 2 + (((2 * s + hh) ^ swz<D>(lq)) << 4);
  }
  __device__ __forceinline__ void move(int by) {
#pragma unroll
    for (int s = 0; s < NR; ++s) at[s] += by;
  }
  __device__ __forceinline__ bf16x8 read(int s) const {
    return *(const LDS_AS bf16x8*)(unsigned long)(at[s % NR] + 256 * (s / NR));
  }
};
template <int D>
struct TrReader {
  static constexpr int NT = D / 32 < 4 ? D / 32 : 4;
  unsigned at[2][NT];
  __device__ __forceinline__ void init(int lane, unsigned st) {
    const int G = lane >> 4, vq = (lane & 15) >> 2, vp = lane & 3;
    const int r0 = 4 * (G >> 1) + vq;
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int dt = 0; dt < NT; ++dt)
        at[o][dt] = st + (r0 + 8 * o) * D * 2 +
                    (((4 * dt + 2 * (G & 1) + (vp >> 1)) ^ swz<D>(r0 + 8 * o)) << 4) + (vp & 1) * 8;
  }
  __device__ __forceinline__ void move(int by) {
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int dt = 0; dt < NT; ++dt) at[o][dt] += by;
  }
  __device__ __forceinline__ bf16x8 read(int ks, int dt) const {
    const int by = ks * 16 * D * 2 + 256 * (dt / NT);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(unsigned long)(at[0][dt % NT] + by));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(unsigned long)(at[1][dt % NT] + by));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

#define FENCE() __builtin_amdgcn_sched_barrier(0)

// The phases below fix the instruction order by hand. Waves issue in order and a 32x32x16 MFMA holds its pipe for 32
// cycles, so a second MFMA right behind the first blocks the wave until the first is done: other work overlaps only
// where it stands BETWEEN MFMAs, at most 28 cycles of it (7 VALU instructions, or a v_exp and 3) per MFMA. With the VALU
// work behind pairs of MFMAs a step took the sum of both. Score products are builtins, so that the compiler keeps the
// wait states before the VALU reads them (built with -amdgpu-mfma-vgpr-form: scores stay in VGPRs); the gradients' are
// asm with the accumulators pinned to AGPRs (attn_common.h, mfma_o).

// MFMAs of the next phase that are issued before the VALU reads a phase's scores: an 8-pass MFMA's result may be read 72
// cycles after its start, and the third MFMA behind it starts after 96
constexpr int SKIP = 2;

__device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// The first reads of a phase, made before it starts
template <int D>
struct RowAhead {
  static constexpr int N = 4;
  bf16x8 a[N];
  __device__ __forceinline__ void read(const RowReader<D>& o) {
#pragma unroll
    for (int s = 0; s < N; ++s) a[s] = o.read(s);
  }
};
template <int D>
struct TrAhead {
  static constexpr int N = 3;
  bf16x8 a[N];
  __device__ __forceinline__ void read(const TrReader<D>& o) {
#pragma unroll
    for (int m = 0; m < N; ++m) a[m] = o.read(m / (D / 32), m % (D / 32));
  }
};

// acc[n] (VGPRs) = stage rows . stationary block n. hook(m) after each of the D / 8 MFMAs; last(): reads of the next phase
template <int D, typename Hook, typename Last>
__device__ __forceinline__ void row_phase(const RowReader<D>& o, const RowAhead<D>& first,
                                          const bf16x8 (&f)[2][D / 16], f32x16 (&acc)[2], Hook hook, Last last) {
  constexpr int NS = D / 16, AHEAD = RowAhead<D>::N;
  bf16x8 a[NS];
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) a[s] = first.a[s];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    acc[0] = mfma(a[s], f[0][s], s == 0 ? zero16() : acc[0]);
    FENCE();
    if (s + AHEAD < NS) a[s + AHEAD] = o.read(s + AHEAD);
    if (s + AHEAD == NS) last();
    hook(2 * s);
    FENCE();
    acc[1] = mfma(a[s], f[1][s], s == 0 ? zero16() : acc[1]);
    FENCE();
    hook(2 * s + 1);
    FENCE();
  }
}

// acc[n][dt] (AGPRs) += (stage columns)^T . b[n]. hook(m) after each of the 4 D / 32 MFMAs; last(): reads of the next
// phase
template <int D, typename Hook, typename Last>
__device__ __forceinline__ void tr_phase(const TrReader<D>& o, const TrAhead<D>& first,
                                         bf16x8 (&b)[2][2], f32x16 (&acc)[2][D / 32], Hook hook, Last last) {
  constexpr int ND = D / 32, AHEAD = TrAhead<D>::N;
  bf16x8 a[2 * ND];
#pragma unroll
  for (int m = 0; m < AHEAD; ++m) a[m] = first.a[m];
#pragma unroll
  for (int m = 0; m < 2 * ND; ++m) {
    mfma_o<false>(acc[0][m % ND], a[m], b[0][m / ND]);
    FENCE();
    if (m + AHEAD < 2 * ND) a[m + AHEAD] = o.read((m + AHEAD) / ND, (m + AHEAD) % ND);
    if (m + AHEAD == 2 * ND) last();
    hook(2 * m);
    FENCE();
    mfma_o<false>(acc[1][m % ND], a[m], b[1][m / ND]);
    FENCE();
    hook(2 * m + 1);
    FENCE();
  }
}

// A softmax has 32 scores a lane and stage. With D = 256 they fit between the 32 MFMAs of the tr phase behind their row
// phase. With fewer columns the last kLate of them get their exp2 between the MFMAs of the next row phase (which makes
// the next stage's scores: their arguments move out of its way in the tr phase).
template <int D>
constexpr int kLate = D == 256 ? 0 : D == 128 ? 20 : 16;
// MFMA of the tr phase that score e is done behind: 6 parts of work for a whole one, 1 for an argument
template <int D>
constexpr int slot_of(int e) {
  constexpr int M = D / 8 - SKIP, T = 32 - kLate<D>, W = 6 * T + kLate<D>;
  return SKIP + (e < T ? 6 * e : 6 * T + e - T) * M / W;
}

template <int ND>
__device__ __forceinline__ void acc_zero(f32x16 (&acc)[2][ND]) {
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[n][i][r] = 0.f;
}

// MFMA writes of the accumulators -> their readers
template <int ND>
__device__ __forceinline__ void acc_fence(f32x16 (&acc)[2][ND]) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" ::: "memory");
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < ND; ++i) asm volatile("" : "+a"(acc[n][i]));
}

__device__ __forceinline__ unsigned pack_bf(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  const bf16x2 v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(unsigned, v);
}

// What bf16 dropped of the pair whose rounded halves are `hi`, as bf16
__device__ __forceinline__ unsigned dropped(float a, float b, unsigned hi) {
  return pack_bf(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}

// P and dS are rounded to bf16 for their products. Over many roundings and results that averages out: dv, dk and out are
// sqrt(2) times as far (in the mean square) from the exact ones as one rounding of the result is. Where a sequence has few
// of them, or few that matter, chance takes that far up (one query's P rounds alike for all columns: up to 2), so there a
// second run of MFMAs adds what the rounding dropped. Few: for out at most 2048 P or 8192 results, for dk and dv, whose
// terms vary more, 2^17 P or 32768 results. In 800 batches of up to five sequences of 1 to 4720 tokens, with keys that
// many queries share: out 1.43 at most, dk and dv 1.50, against 1.46 and 1.54 in 100 without.
__device__ __forceinline__ bool few(long pairs, long results, bool gradient) {
  return pairs <= (gradient ? 1 << 17 : 2048) || results <= (gradient ? 32768 : 8192);
}

// VALU write -> asm MFMA read (the compiler does not look into asm): two wait states before a run of MFMAs
__device__ __forceinline__ void settle() {
  FENCE();
  asm volatile("s_nop 1");
  FENCE();
}

// LDS of a key workgroup: q ring of 5 stages, dout ring of 3, P double-buffered, lse and delta rings; of a query
// workgroup: k ring of 5, v ring of 3, dS double-buffered (D = 256: all 160 KB). Rings are kExtra stages longer.
template <int D>
struct Lds {
  static constexpr int RA = 5 + kExtra<D>, RB = 3 + kExtra<D>;
  static constexpr int A = 0, B = RA * Stage<D>::BYTES, X = B + RB * Stage<D>::BYTES;
  static constexpr int PBYTES = 8192, SBYTES = 16384;  // one buffer of P, of dS
  static constexpr int LSE = X + 2 * PBYTES, DELTA = LSE + 8 * 256, LOW = DELTA + 8 * 256, TOTAL = X + 2 * SBYTES;
  static_assert(LOW + PBYTES <= TOTAL, "lse, delta and the low parts of dS lie behind P, where a query workgroup has dS");
  static_assert(TOTAL <= 160 * 1024 && 3 + kExtra<D> < 8, "LDS of a CU; the rings of lse and delta");
};

// First of the `all` pieces of work that stand behind MFMA m of M, of which the first SKIP have none
__device__ __forceinline__ constexpr int share(int m, int M, int all) {
  return m <= SKIP ? 0 : ((m - SKIP) * all + (M - SKIP) - 1) / (M - SKIP);
}

// A key workgroup: dk and dv of 128 keys of K/V head hk. Step i: wave 0 makes S(i + 1), then (behind the barrier) adds
// dout(i)^T P(i) to dv while it turns S(i + 1) into P(i + 1); wave 1 makes dP(i), then adds q(i - 1)^T dS(i - 1) to dk
// while it makes dS(i) from dP(i) and P(i).
template <int D, bool FEW>
__device__ __forceinline__ void key_block(const TrainDev& d, const Unit& u, char* smem) {
  const AttnTrainParams& p = d.p;
  using L = Lds<D>;
  constexpr int ND = D / 32, SB = Stage<D>::BYTES, P = Stage<D>::PIECES, E = kExtra<D>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lq = lane & 31, hh = lane >> 5, pair = wave >> 1;
  const int hk = u.h, b = u.b;
  int q_start, q_len, k_start, k_len;
  seq_range(p.cu_q, b, p.total_q, &q_start, &q_len);
  seq_range(p.cu_k, b, p.total_k, &k_start, &k_len);
  const int row0 = u.full ? u.tile * WROWS : k_len - k_len % WROWS;
  const int group = p.H / p.HK;
  const int tiles = (q_len + 31) / 32;  // stages of one head
  const int all = tiles * group, ranges = u.ranges;
  const int per = (all + ranges - 1) / ranges, t0 = min(u.part * per, all), n = min(per, all - t0);

  f32x16 acc[2][ND];
  acc_zero<ND>(acc);
  if (n > 0) {
    Stage<D> sq, sd;
    sq.init(p.q_row, wave, lane);
    sd.init(p.do_row, wave, lane);
    const unsigned lds0 = (unsigned)__builtin_amdgcn_readfirstlane((int)lds_addr_of(smem));
    const unsigned wlds = lds0 + wave * 1024;
    const unsigned ld_off = lane < 32 ? lane * 4 : 0x7ffffff0u;
    // Stages: rows of the group's heads in turn. Rows past the sequence end and stages past the last are zeros, lse and
    // delta included: P = exp2(0 - 0) = 1 meets zero rows
    Stream st_q, st_d, st_x;  // st_x: lse for wave 0, delta for the others (wave 1 copies it)
    const long h0 = (long)hk * group;
    st_q.init(p.q + (long)q_start * p.q_row + h0 * p.q_head, t0, tiles, q_len, n, p.q_row * 2, p.q_head * 2);
    st_d.init(p.dout + (long)q_start * p.do_row + h0 * p.do_head, t0, tiles, q_len, n, p.do_row * 2, p.do_head * 2);
    st_x.init((wave == 0 ? d.lse2 : d.delta) + h0 * p.total_q + q_start, t0, tiles, q_len, n, 4, (long)p.total_q * 4);
    Ring<L::RA, SB> to_a{(3 + E) * SB};  // where step i's copies go
    Ring<L::RB, SB> to_b{(2 + E) * SB};
    // stages i + 3 + E of q and i + 2 + E of dout, in 2 P + 1 pieces: issued behind step i's barrier, in place E + 1
    // barriers later
    auto open = [&]() {
      st_q.next();
      st_d.next();
      st_x.next();
    };
    auto copy = [&](int i, int k) {
      if (k < P)
        copy16(st_q.rs, sq.src(k), wlds + L::A + to_a.at + sq.dst(k));
      else if (k < 2 * P)
        copy16(st_d.rs, sd.src(k - P), wlds + L::B + to_b.at + sd.dst(k - P));
      else if (k == 2 * P && wave < 2)
        copy4(st_x.rs, ld_off, lds0 + (wave == 0 ? L::LSE + ((i + 3 + E) & 7) * 256 : L::DELTA + ((i + 2 + E) & 7) * 256));
    };
    RowReader<D> rr;
    TrReader<D> tr;
    // before step 0: q stages -1 (zeros: dk(-1) adds nothing), 0 .. 2 + E; dout stages 0 .. 1 + E
    {
      const i32x4 zero = make_rsrc(p.q, 0);
#pragma unroll
      for (int k = 0; k < P; ++k) copy16(zero, sq.src(k), wlds + L::A + (L::RA - 1) * SB + sq.dst(k));
#pragma unroll
      for (int j = 0; j < 3 + E; ++j) {
        st_q.next();
#pragma unroll
        for (int k = 0; k < P; ++k) copy16(st_q.rs, sq.src(k), wlds + L::A + j * SB + sq.dst(k));
      }
#pragma unroll
      for (int j = 0; j < 2 + E; ++j) {
        st_d.next();
#pragma unroll
        for (int k = 0; k < P; ++k) copy16(st_d.rs, sd.src(k), wlds + L::B + j * SB + sd.dst(k));
      }
      for (int j = 0; j < (wave == 0 ? 3 : 2) + E; ++j) {
        st_x.next();
        if (wave < 2) copy4(st_x.rs, ld_off, lds0 + (wave == 0 ? L::LSE : L::DELTA) + j * 256);
      }
    }
    // stationary rows: k for wave 0, v for wave 1
    bf16x8 f[2][D / 16];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const long rc = k_start + min(row0 + pair * 64 + nb * 32 + lq, k_len - 1);
      load_frags<D>(wave & 1 ? p.v + rc * p.v_row + (long)hk * p.v_head : p.k + rc * p.k_row + (long)hk * p.k_head, hh,
                    f[nb]);
      if (!(wave & 1)) take_sign<D>(f[nb], p.scale);
    }
    bf16x8 bc[2][2];  // P (wave 0) or dS (wave 1) of the stage that the tr phase takes, B operands
    u32x4 bn[2][2];   // of the next
    f32x16 s[2];
    RowAhead<D> ra;
    TrAhead<D> ta;
    const float sl2 = score_scale(p.scale);
    // P of stage j, fp16: [j & 1][pair][r4][block][lane] 8 B
    char* const xch = smem + L::X + pair * (L::PBYTES / 2) + lane * 8;
    auto none = [](int) {};
    auto nothing = []() {};
    // work behind MFMA m of the tr phase: copies of step i, and the 32 scores spread over the MFMAs m >= SKIP
    auto spread_copies = [&](int i, int m) {
      constexpr int GAP = (4 * ND) / (2 * P + 1);
      if (m % GAP == 0 && m / GAP <= 2 * P) copy(i, m / GAP);
    };
    auto spread = [&](int i, int m, auto one) {
      spread_copies(i, m);
#pragma unroll
      for (int e = share(m, 4 * ND, 32); e < share(m + 1, 4 * ND, 32); ++e) one(e);
    };
    auto next = [&]() {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) bc[nb][ks] = __builtin_bit_cast(bf16x8, bn[nb][ks]);
    };
    step_sync();
    if ((wave & 1) == 0) {
      // score e of stage j: group r4 = e >> 3 (rows 8 r4 + 4 hh + 0..3), block (e >> 2) & 1. Each call does the exp2 of
      // its score, the argument of the next and the stores of the ones before, so that nothing waits on the exp2
      constexpr int LATE = kLate<D>, T = 32 - LATE;
      f32x4 lse, lse_n;
      float x, late[LATE > 0 ? LATE : 1];
      auto val = [&](int e) { return e < T ? s[(e >> 2) & 1][4 * (e >> 3) + (e & 3)] : late[e < T ? 0 : e - T]; };
      auto arg = [&](int j, int e) {
        const int r4 = e >> 3, nb = (e >> 2) & 1, i = e & 3;
        if ((e & 7) == 0) lse = lse_n;
        const float y = __builtin_fmaf(s[nb][4 * r4 + i], sl2, -lse[i]);
        if (e < T)
          x = y;
        else
          late[e - T] = y;
        if ((e & 7) == 0 && r4 < 3)
          lse_n = *(const f32x4*)(smem + L::LSE + (j & 7) * 256 + (8 * (r4 + 1) + 4 * hh) * 4);
      };
      auto store = [&](int j, int e) {  // P of score e is there
        const int r4 = e >> 3, nb = (e >> 2) & 1, i = e & 3, r = 4 * r4 + i;
        if (i & 1) bn[nb][r >> 3][(r & 7) >> 1] = pack_bf(val(e - 1), val(e));
        if (i == 3) {
          typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
          *(f16x4*)(xch + (j & 1) * L::PBYTES + (r4 * 2 + nb) * 512) =
              f16x4{(_Float16)val(e - 3), (_Float16)val(e - 2), (_Float16)val(e - 1), (_Float16)val(e)};
        }
      };
      auto begin = [&](int j) { lse_n = *(const f32x4*)(smem + L::LSE + (j & 7) * 256 + 4 * hh * 4); };
      auto prob = [&](int j, int e) {  // in the tr phase
        if (e == 0) arg(j, 0);
        if (e < T) s[(e >> 2) & 1][4 * (e >> 3) + (e & 3)] = __builtin_amdgcn_exp2f(x);
        if (e < 31) arg(j, e + 1);
        if (e > 0 && e <= T) store(j, e - 1);
        if (e == 31 && T == 32) store(j, 31);
      };
      auto prob_late = [&](int j, int m) {  // behind MFMA m of the next row phase
#pragma unroll
        for (int e = T + m * LATE / (D / 8); e < T + (m + 1) * LATE / (D / 8); ++e) {
          late[e - T] = __builtin_amdgcn_exp2f(late[e - T]);
          if (e > T) store(j, e - 1);
          if (e == 31) store(j, 31);
        }
      };
      rr.init(lane, lds0 + L::A);
      tr.init(lane, lds0 + L::B);
      begin(0);
      ra.read(rr);
      row_phase<D>(rr, ra, f, s, none, nothing);
#pragma unroll
      for (int e = 0; e < 32; ++e) prob(0, e);
      if constexpr (LATE == 0) next();
      rr.move(SB);  // q stage i + 1
      ra.read(rr);
      Ring<L::RA, SB> at_r{SB};
      Ring<L::RB, SB> at_t{0};
      for (int i = 0; i < n; ++i) {
        open();
        begin(i + 1);
        row_phase<D>(rr, ra, f, s, [&](int m) { prob_late(i, m); }, [&]() { ta.read(tr); });
        if constexpr (LATE > 0) next();
        rr.move(at_r.move());
        if (wave == 0)
          step_sync<E*(2 * P + 1)>();
        else
          step_sync<E * 2 * P>();
        tr_phase<D>(
            tr, ta, bc, acc,
            [&](int m) {
              spread_copies(i, m);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (slot_of<D>(e) == m) prob(i + 1, e);
            },
            [&]() { ra.read(rr); });
        if constexpr (FEW) {  // P(i) lies in LDS with three more bits
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const int nb = g & 1, ks = g >> 2, w = g & 2;
            typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
            const f16x4 y = *(const f16x4*)(xch + (i & 1) * L::PBYTES + g * 512);
            u32x4 b = __builtin_bit_cast(u32x4, bc[nb][ks]);
            b[w] = dropped((float)y[0], (float)y[1], b[w]);
            b[w + 1] = dropped((float)y[2], (float)y[3], b[w + 1]);
            bc[nb][ks] = __builtin_bit_cast(bf16x8, b);
          }
          ta.read(tr);
          settle();
          tr_phase<D>(tr, ta, bc, acc, none, nothing);
        }
        if constexpr (LATE == 0) next();
        tr.move(at_t.move());
        to_a.next();
        to_b.next();
      }
      step_sync();
    } else {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) bc[nb][ks] = __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
      rr.init(lane, lds0 + L::B);           // dout stage i
      tr.init(lane, lds0 + L::A + (L::RA - 1) * SB);  // q stage i - 1
      ra.read(rr);
      f32x4 del, del_n;
      typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
      f16x4 pr, pr_n;
      Ring<L::RB, SB> at_r{0};
      Ring<L::RA, SB> at_t{(L::RA - 1) * SB};
      char* const low = smem + L::LOW + pair * (L::PBYTES / 2) + lane * 16;  // of dS(i - 1): [block][k-step][lane] 16 B
      if constexpr (FEW) {
#pragma unroll
        for (int g = 0; g < 4; ++g) *(u32x4*)(low + g * 1024) = u32x4{0u, 0u, 0u, 0u};
      }
      for (int i = 0; i <= n; ++i) {
        auto rd = [&](int e) {  // delta and P of the 4 scores from e on
          const int r4 = e >> 3, nb = (e >> 2) & 1;
          if (nb == 0) del_n = *(const f32x4*)(smem + L::DELTA + (i & 7) * 256 + (8 * r4 + 4 * hh) * 4);
          pr_n = *(const f16x4*)(xch + (i & 1) * L::PBYTES + (r4 * 2 + nb) * 512);
        };
        open();  // after the last stage: zeros
        row_phase<D>(rr, ra, f, s, none, [&]() { ta.read(tr); });
        rr.move(at_r.move());
        if (wave == 1)
          step_sync<E*(2 * P + 1)>();
        else
          step_sync<E * 2 * P>();
        rd(0);
        tr_phase<D>(
            tr, ta, bc, acc,
            [&](int m) {
              spread(i, m, [&](int e) {
                const int nb = (e >> 2) & 1, k = e & 3, r = 4 * (e >> 3) + k;
                if (k == 0) {
                  pr = pr_n;
                  if (nb == 0) del = del_n;
                  if (e + 4 < 32) rd(e + 4);
                }
                s[nb][r] = (float)pr[k] * (s[nb][r] - del[k]);
                if (k & 1) bn[nb][r >> 3][(r & 7) >> 1] = pack_bf(s[nb][r - 1], s[nb][r]);
              });
            },
            [&]() { ra.read(rr); });
        if constexpr (FEW) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int nb = g >> 1, ks = g & 1;
            bc[nb][ks] = *(const bf16x8*)(low + g * 1024);
            u32x4 w;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              w[c] = dropped(s[nb][8 * ks + 2 * c], s[nb][8 * ks + 2 * c + 1], bn[nb][ks][c]);
            *(u32x4*)(low + g * 1024) = w;
          }
          ta.read(tr);
          settle();
          tr_phase<D>(tr, ta, bc, acc, none, nothing);
        }
        next();
        tr.move(at_t.move());
        to_a.next();
        to_b.next();
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy may outlive the workgroup
  }
  acc_fence<ND>(acc);
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int row = row0 + pair * 64 + nb * 32 + lq;
    const bool live = row < k_len;
    const long rc = k_start + min(row, k_len - 1);
    const float f = wave & 1 ? p.scale * kUnshift : kUnshift;
    if (ranges > 1) {
      // dv's partials follow all of dk's
      long step;
      float* to = part_row<D>(d.k, u.full, p.B, p.total_k, k_start, b, min(row, k_len - 1), hk, &step);
      to += (u.part + (wave & 1 ? 0 : u.full ? d.k.max_full : d.k.max_part)) * step;
      store_part<D>(to, acc[nb], f, hh, live);
    } else if (wave & 1) {
      store_row<D>(p.dk + rc * p.dk_row + (long)hk * p.dk_head, acc[nb], f, hh, live);
    } else {
      store_row<D>(p.dv + rc * p.dv_row + (long)hk * p.dv_head, acc[nb], f, hh, live);
    }
  }
}

// A query workgroup: dq of 128 queries of head h. Step i: wave 0 makes S and dP of stage i + 1 while it makes dS(i);
// wave 1 adds k(i - 1)^T dS(i - 1) to dq.
template <int D>
__device__ __forceinline__ void query_block(const TrainDev& d, const Unit& u, char* smem) {
  const AttnTrainParams& p = d.p;
  using L = Lds<D>;
  constexpr int ND = D / 32, NS = D / 16, SB = Stage<D>::BYTES, P = Stage<D>::PIECES, E = kExtra<D>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lq = lane & 31, hh = lane >> 5, pair = wave >> 1;
  const int h = u.h, b = u.b;
  int q_start, q_len, k_start, k_len;
  seq_range(p.cu_q, b, p.total_q, &q_start, &q_len);
  seq_range(p.cu_k, b, p.total_k, &k_start, &k_len);
  const int row0 = u.full ? u.tile * WROWS : q_len - q_len % WROWS;
  const int hk = h / (p.H / p.HK);
  const int all = (k_len + 31) / 32, ranges = u.ranges;
  const int per = (all + ranges - 1) / ranges, t0 = min(u.part * per, all), n = min(per, all - t0);

  Stage<D> sk, sv;
  sk.init(p.k_row, wave, lane);
  sv.init(p.v_row, wave, lane);
  const unsigned lds0 = (unsigned)__builtin_amdgcn_readfirstlane((int)lds_addr_of(smem));
  const unsigned wlds = lds0 + wave * 1024;
  Stream st_k, st_v;
  if (n > 0) {
    st_k.init(p.k + (long)k_start * p.k_row + (long)hk * p.k_head, t0, all, k_len, n, p.k_row * 2, 0);
    st_v.init(p.v + (long)k_start * p.v_row + (long)hk * p.v_head, t0, all, k_len, n, p.v_row * 2, 0);
  }
  // stages i + 3 + E of k and v
  Ring<L::RA, SB> to_a{0};
  Ring<L::RB, SB> to_b{0};
  auto open = [&]() {
    st_k.next();
    st_v.next();
  };
  auto copy = [&](int k) {  // piece k
    if (k < P)
      copy16(st_k.rs, sk.src(k), wlds + L::A + to_a.at + sk.dst(k));
    else if (k < 2 * P)
      copy16(st_v.rs, sv.src(k - P), wlds + L::B + to_b.at + sv.dst(k - P));
  };
  auto advance = [&]() {
    to_a.next();
    to_b.next();
  };
  auto copy_all = [&]() {
    open();
#pragma unroll
    for (int k = 0; k < 2 * P; ++k) copy(k);
    advance();
  };

  // dS of stage j: [j & 1][pair][block][r4][lane] f32x4
  char* const xch = smem + L::X + pair * (L::SBYTES / 2) + lane * 16;
  if ((wave & 1) == 0) {
    if (n <= 0) return;  // wave 1 stores the zeros
#pragma unroll
    for (int j = 0; j < 3 + E; ++j) copy_all();
    bf16x8 qf[2][NS], df[2][NS];
    float lse[2], del[2];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const long rc = q_start + min(row0 + pair * 64 + nb * 32 + lq, q_len - 1);
      load_frags<D>(p.q + rc * p.q_row + (long)h * p.q_head, hh, qf[nb]);
      take_sign<D>(qf[nb], p.scale);
      load_frags<D>(p.dout + rc * p.do_row + (long)h * p.do_head, hh, df[nb]);
      lse[nb] = d.lse2[(long)h * p.total_q + rc];
      del[nb] = d.delta[(long)h * p.total_q + rc];
    }
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        asm volatile("" : "+a"(qf[nb][s]));
        asm volatile("" : "+a"(df[nb][s]));
      }
    asm volatile("s_nop 4" ::: "memory");
    const float sl2 = score_scale(p.scale);
    f32x16 sa[2], da[2], sb[2], db[2];
    // Half u of the 64 that make stage j's dS from its S and dP: element e = u >> 1 (block e >> 4, score e & 15); even
    // halves do an exp2 and the next one's argument, odd ones the product
    // dP starts from -delta where there are registers for it: a subtraction less per score
    constexpr bool FROM = D < 256;
    f32x16 from[FROM ? 2 : 1];
    if constexpr (FROM) {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) from[nb][r] = -del[nb];
    }
    float x, pe;
    auto ds_half = [&](int j, f32x16 (&s)[2], f32x16 (&dp)[2], int u) {
      const int e = u >> 1, nb = e >> 4, r = e & 15;
      if ((u & 1) == 0) {
        if (e == 0) x = __builtin_fmaf(s[0][0], sl2, -lse[0]);
        pe = __builtin_amdgcn_exp2f(x);
        if (e < 31) x = __builtin_fmaf(s[(e + 1) >> 4][(e + 1) & 15], sl2, -lse[(e + 1) >> 4]);
      } else {
        s[nb][r] = pe * (FROM ? dp[nb][r] : dp[nb][r] - del[nb]);
        if ((r & 3) == 3)
          *(f32x4*)(xch + (j & 1) * L::SBYTES + (nb * 4 + (r >> 2)) * 1024) =
              f32x4{s[nb][r - 3], s[nb][r - 2], s[nb][r - 1], s[nb][r]};
      }
    };
    constexpr int AHEAD = 5;
    bf16x8 first[AHEAD];
    RowReader<D> kr, vr;
    kr.init(lane, lds0 + L::A);
    vr.init(lane, lds0 + L::B);
    auto rd = [&](int m) { return m & 1 ? vr.read(m >> 1) : kr.read(m >> 1); };
    auto read_first = [&]() {
#pragma unroll
      for (int m = 0; m < AHEAD; ++m) first[m] = rd(m);
    };
    // S and dP of the readers' stage into (s, dp); hook(u) after each of the 4 NS MFMAs. last() may move the readers on
    auto products = [&](f32x16 (&s)[2], f32x16 (&dp)[2], auto hook, auto last) {
      bf16x8 a[2 * NS];
#pragma unroll
      for (int m = 0; m < AHEAD; ++m) a[m] = first[m];
#pragma unroll
      for (int m = 0; m < 2 * NS; ++m) {
        f32x16(&acc)[2] = m & 1 ? dp : s;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          const bf16x8& f = m & 1 ? df[nb][m >> 1] : qf[nb][m >> 1];
          acc[nb] = mfma(a[m], f, m == 1 && FROM ? from[FROM ? nb : 0] : m < 2 ? zero16() : acc[nb]);
          FENCE();
          if (nb == 0 && m + AHEAD < 2 * NS) a[m + AHEAD] = rd(m + AHEAD);
          if (nb == 0 && m + AHEAD == 2 * NS) last();
          hook(2 * m + nb);
          FENCE();
        }
      }
    };
    Ring<L::RA, SB> at_k{SB};
    Ring<L::RB, SB> at_v{SB};
    auto mask = [&](int j, f32x16 (&s)[2]) {  // keys past the end: P = 0 (their exp2(-lse) may overflow)
      const int left = k_len - (t0 + j) * 32;
      if (left >= 32) return;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[nb][r] = 8 * (r >> 2) + 4 * hh + (r & 3) < left ? s[nb][r] : -INFINITY;
    };
    auto step = [&](int i, f32x16 (&s)[2], f32x16 (&dp)[2], f32x16 (&s2)[2], f32x16 (&dp2)[2]) {
      read_first();  // behind the barrier: before it, the stage's copies had a step less to arrive
      open();
      mask(i, s);
      products(
          s2, dp2,
          [&](int m) {
#pragma unroll
            for (int u = share(m, 4 * NS, 64); u < share(m + 1, 4 * NS, 64); ++u) ds_half(i, s, dp, u);
            if ((m & 1) && (m >> 1) < 2 * P) copy(m >> 1);
          },
          [&]() {
            kr.move(at_k.move());
            vr.move(at_v.move());
          });
      advance();
      step_sync<(E + 1) * 2 * P>();
    };
    step_sync();
    read_first();
    products(sa, da, [](int) {}, []() {});
    kr.move(SB);
    vr.move(SB);
    step_sync();
    int i = 0;
    for (; i + 1 < n; i += 2) {
      step(i, sa, da, sb, db);
      step(i + 1, sb, db, sa, da);
    }
    if (i < n) step(i, sa, da, sb, db);
    step_sync();  // wave 1's last one; no copy may outlive the workgroup
    return;
  }
  f32x16 acc[2][ND];
  acc_zero<ND>(acc);
  if (n > 0) {
#pragma unroll
    for (int j = 0; j < 3 + E; ++j) copy_all();
    step_sync();
    step_sync();
    copy_all();
    bf16x8 a[ND];
    TrReader<D> tr;  // k stage i - 1
    tr.init(lane, lds0 + L::A);
    auto rd = [&](int s, int dt) { a[dt] = tr.read(s, dt); };
    Ring<L::RA, SB> at_t{0};
    f32x4 w[2][4];
    u32x4 hi[2][2], lo[2][2];
    auto load = [&](int j) {  // dS of stage j
      const char* x = xch + (j & 1) * L::SBYTES;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) w[nb][r4] = *(const f32x4*)(x + (nb * 4 + r4) * 1024);
    };
    auto split_hi = [&](int s, int q) {  // pair q of 8: block q >> 2, scores 8 s + 2 (q & 3), + 1
      const int nb = q >> 2, c = q & 3;
      const f32x4& y = w[nb][2 * s + (c >> 1)];
      hi[nb][s][c] = pack_bf(y[2 * (c & 1)], y[2 * (c & 1) + 1]);
    };
    auto split_lo = [&](int s, int q) {
      const int nb = q >> 2, c = q & 3;
      const f32x4& y = w[nb][2 * s + (c >> 1)];
      lo[nb][s][c] = dropped(y[2 * (c & 1)], y[2 * (c & 1) + 1], hi[nb][s][c]);
    };
    // 2 ND MFMAs with one half of the stage's rows; hook(m) behind each
    auto run = [&](const u32x4 (&b)[2][2], int s, auto hook) {
      settle();
#pragma unroll
      for (int m = 0; m < 2 * ND; ++m) {
        bf16x8 bb = __builtin_bit_cast(bf16x8, b[m & 1][s]);
        mfma_o<false>(acc[m & 1][m >> 1], a[m >> 1], bb);
        FENCE();
        hook(m);
        FENCE();
      }
    };
    auto begin = [&]() {
#pragma unroll
      for (int q = 0; q < 8; ++q) split_hi(0, q);
      FENCE();
    };
    step_sync<(E + 1) * 2 * P>();
    load(0);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) rd(0, dt);
    begin();
    for (int i = 1; i <= n; ++i) {
      open();  // after the last stage: zeros
      run(hi, 0, [&](int m) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q * ND / 4 == m) split_lo(0, q);
        if (m & 1) copy(m >> 1);
      });
      // the fragments once more, then their place takes the next half's; beside them the next half's split
      run(lo, 0, [&](int m) {
        if (m & 1) rd(1, m >> 1);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q * ND / 4 == m) {
            split_hi(1, q);
            split_lo(1, q);
          }
      });
      run(hi, 1, [](int) {});
      // The barrier stands before the last MFMAs, which cover the next step's first reads (behind the last one they are
      // of no use; wave 0 has one barrier more for it)
      advance();
      tr.move(at_t.move());
      step_sync<(E + 1) * 2 * P>();
      load(i);
      run(lo, 1, [&](int m) {
        if (m & 1) rd(0, m >> 1);
      });
      begin();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy may outlive the workgroup
  }
  acc_fence<ND>(acc);
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int row = row0 + pair * 64 + nb * 32 + lq;
    const bool live = row < q_len;
    const long rc = q_start + min(row, q_len - 1);
    const float f = p.scale * kUnshift;
    if (ranges > 1) {
      long step;
      float* to = part_row<D>(d.q, u.full, p.B, p.total_q, q_start, b, min(row, q_len - 1), h, &step);
      store_part<D>(to + u.part * step, acc[nb], f, hh, live);
    } else
      store_row<D>(p.dq + rc * p.dq_row + (long)h * p.dq_head, acc[nb], f, hh, live);
  }
}

template <int D>
__global__ __launch_bounds__(kThreads, 1) void attn_bwd_kernel(TrainDev d) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Unit u;
  if (!find_unit(d, blockIdx.x, &u)) return;
  const AttnTrainParams& p = d.p;
  int start, q_len, k_len;
  seq_range(p.cu_q, u.b, p.total_q, &start, &q_len);
  seq_range(p.cu_k, u.b, p.total_k, &start, &k_len);
  if (u.query)
    query_block<D>(d, u, smem);
  else if (few((long)q_len * k_len * p.H, (long)k_len * p.HK * D, true))
    key_block<D, true>(d, u, smem);
  else
    key_block<D, false>(d, u, smem);
}

// Adds the ranges' partial gradients in order: one item = 8 columns of a row and head, of all rows (full tiles) or of the
// 128-row slots of the sequences' parts. Bound by memory: three ranges of 589 keys, 12 heads of 256, and their like 15 us.
struct JoinItems {
  int q_full, q_part, k_full, k_part;  // workgroups; 0: that kind has no ranges
};
template <int D>
__global__ __launch_bounds__(kThreads) void attn_join_kernel(TrainDev d, JoinItems n) {
  const AttnTrainParams& p = d.p;
  constexpr int LANES = D / 8;
  int blk = blockIdx.x;
  const bool is_q = blk < n.q_full + n.q_part;
  blk -= is_q ? 0 : n.q_full + n.q_part;
  const bool full = blk < (is_q ? n.q_full : n.k_full);
  blk -= full ? 0 : is_q ? n.q_full : n.k_full;
  const Cut& c = is_q ? d.q : d.k;
  const long item = ((long)blk * kThreads + threadIdx.x) / LANES;
  const int col = threadIdx.x % LANES * 8;
  const int total = is_q ? p.total_q : p.total_k;
  const int* own = is_q ? p.cu_q : p.cu_k;
  const long slot = item / c.heads;
  const int h = (int)(item % c.heads);
  int b, start, len, row;
  if (full) {
    if (slot >= total) return;
    b = find_seq(own, p.B, total, (int)slot);
    if (b < 0) return;
    seq_range(own, b, total, &start, &len);
    row = (int)slot - start;
    if (row >= len - len % WROWS) return;
  } else {
    if (slot >= (long)p.B * WROWS) return;
    b = (int)(slot / WROWS);
    seq_range(own, b, total, &start, &len);
    row = len - len % WROWS + (int)(slot % WROWS);
    if (row >= len) return;
  }
  int s2, swept;
  seq_range(is_q ? p.cu_k : p.cu_q, b, is_q ? p.total_k : p.total_q, &s2, &swept);
  const int most = full ? c.max_full : c.max_part;
  const int ranges = ranges_of((swept + 31) / 32 * (is_q ? 1 : p.H / p.HK), d.target[full ? 0 : 1], most);
  if (ranges < 2) return;
  long step;
  const float* src = part_row<D>(c, full, p.B, total, start, b, row, h, &step) + col;
  const long r = (long)start + row;
  for (int out = 0; out < (is_q ? 1 : 2); ++out, src += most * step) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
    for (int i = 0; i < ranges; ++i) {
      x += *(const f32x4*)(src + i * step);
      y += *(const f32x4*)(src + i * step + 4);
    }
    bf16_t* to = is_q ? p.dq + r * p.dq_row + (long)h * p.dq_head
                 : out ? p.dv + r * p.dv_row + (long)h * p.dv_head
                       : p.dk + r * p.dk_row + (long)h * p.dk_head;
    *(u32x4*)(to + col) = u32x4{pack2bf(x[0], x[1]), pack2bf(x[2], x[3]), pack2bf(y[0], y[1]), pack2bf(y[2], y[3])};
  }
}

// ------------------------------------------------------------------------------------------------ forward
// A workgroup owns 256 queries of one head, a wave 64 of them and both products: S = k . q^T row-wise, out^T = v^T . P
// transposed, as a key workgroup's wave 0 does. P = 2^(S - m) with m the largest score of the query's first 32 keys: any m
// will do while P and the sums stay in fp32's range, which they do up to S = m + 40 (bf16 rounds P to the same relative
// 2^-9 there), so the accumulators are never scaled anew. Where a later score is larger still, the workgroup sweeps its
// keys once more, with m the largest score of them all, which it then knows. (Scaling the accumulators where a maximum
// grows took 300 registers' spills: a branch that multiplies pulls them out of the AGPRs.) Measured: 2970 cycles a step
// with D = 256 (2048 of MFMAs), 1900 with 128 (1024), 1500 with 64 (512), where two workgroups share a CU instead: 4 x 4096
// tokens, 16 heads 384 -> 321 us.
template <int D>
struct FwdLds {
  static constexpr int E = D == 256 ? 1 : D == 128 ? 3 : 4;  // steps that a copy may take beyond its own
  static constexpr int R = 3 + E, A = 0, B = R * Stage<D>::BYTES, LOW = 2 * R * Stage<D>::BYTES, FLAG = LOW + 16384,
                       TOTAL = FLAG + 16;
};

// The forward pass's units: a tile of 256 queries and a range of its sequence's keys, tiles in order, ranges within
__device__ __forceinline__ int units_of(const TrainDev& d, int b, int* ranges) {
  const AttnTrainParams& p = d.p;
  *ranges = 1;
  if (b >= p.B) return 0;
  int s, q_len, k_len;
  seq_range(p.cu_q, b, p.total_q, &s, &q_len);
  seq_range(p.cu_k, b, p.total_k, &s, &k_len);
  *ranges = ranges_of((k_len + 31) / 32, d.stages, d.most);
  return (q_len + 255) / 256 * *ranges;
}
// Block v -> its unit, heads in turn; false: nothing to do. The launch has an upper bound of blocks, and those without
// a unit come last (between the others they kept units from starting: ragged batch 63 -> 55 us).
struct FwdUnit {
  int b, h, row0, part, ranges;
};
__device__ __forceinline__ bool find_fwd_unit(const TrainDev& d, FwdUnit* u) {
  const int lane = threadIdx.x & 63, B = d.p.B;
  int v = blockIdx.x, units, own;
  if (B <= 64) {
    const int n = units_of(d, lane, &own);
    int sum = n;  // units up to and with sequence `lane`
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(sum, o, 64);
      if (lane >= o) sum += up;
    }
    units = min(__builtin_amdgcn_readlane(sum, 63), d.tiles * d.most);  // more: the cumulative lengths are wrong
    if (v >= units * d.p.H) return false;
    v = xcd_remap(v, units * d.p.H);
    u->h = v / units;
    v %= units;
    u->b = __builtin_ctzll(__ballot(v < sum));
    v -= __builtin_amdgcn_readlane(sum, u->b) - __builtin_amdgcn_readlane(n, u->b);
    u->ranges = __builtin_amdgcn_readlane(own, u->b);
  } else {
    units = min(__builtin_amdgcn_readfirstlane(d.starts[B]), d.tiles * d.most);
    if (v >= units * d.p.H) return false;
    v = xcd_remap(v, units * d.p.H);
    u->h = v / units;
    v %= units;
    u->b = __builtin_amdgcn_readfirstlane(last_at_most<1>(d.starts, B, v));
    v -= __builtin_amdgcn_readfirstlane(d.starts[u->b]);
    units_of(d, u->b, &own);
    u->ranges = __builtin_amdgcn_readfirstlane(own);
  }
  u->row0 = v / u->ranges * 256;
  u->part = v % u->ranges;
  return true;
}

// Units before each sequence, in one workgroup: a block that counted them itself would read all lengths (1024 sequences
// of 64 tokens, 16 heads: 702 us)
__global__ __launch_bounds__(kThreads) void attn_lse_units_kernel(TrainDev d) {
  __shared__ int waves[kThreads / 64];
  const int tid = threadIdx.x;
  int before = 0;
  for (int base = 0; base < d.p.B; base += kThreads) {
    int own;
    const int n = units_of(d, base + tid, &own);
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(sum, o, 64);
      if ((tid & 63) >= o) sum += up;
    }
    if ((tid & 63) == 63) waves[tid >> 6] = sum;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
      if (w < (tid >> 6)) sum += waves[w];
      all += waves[w];
    }
    if (base + tid < d.p.B) d.starts[base + tid] = before + sum - n;
    before += all;
    __syncthreads();
  }
  if (tid == 0) d.starts[d.p.B] = before;
}

template <int D, bool FEW>
__device__ __forceinline__ void lse_unit(const TrainDev& d, const FwdUnit& u, char* smem) {
  const AttnTrainParams& p = d.p;
  const int b = u.b, h = u.h, row0 = u.row0, part = u.part, ranges = u.ranges;
  using L = FwdLds<D>;
  constexpr int ND = D / 32, SB = Stage<D>::BYTES, P = Stage<D>::PIECES, E = L::E;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lq = lane & 31, hh = lane >> 5;
  int q_start, q_len, k_start, k_len;
  seq_range(p.cu_q, b, p.total_q, &q_start, &q_len);
  seq_range(p.cu_k, b, p.total_k, &k_start, &k_len);
  const int hk = h / (p.H / p.HK);
  const int all = (k_len + 31) / 32;
  const int per = (all + ranges - 1) / ranges, t0 = min(part * per, all), n = min(per, all - t0);

  f32x16 acc[2][ND];
  float m[2] = {-INFINITY, -INFINITY}, l[2], largest[2];
  bool again = false;
  do {
    acc_zero<ND>(acc);
    l[0] = l[1] = 0.f;
    if (n <= 0) break;
    const unsigned lds0 = (unsigned)__builtin_amdgcn_readfirstlane((int)lds_addr_of(smem));
    const unsigned wlds = lds0 + wave * 1024;
    Stage<D> sk, sv;
    sk.init(p.k_row, wave, lane);
    sv.init(p.v_row, wave, lane);
    Stream st_k, st_v;
    st_k.init(p.k + (long)k_start * p.k_row + (long)hk * p.k_head, t0, all, k_len, n, p.k_row * 2, 0);
    st_v.init(p.v + (long)k_start * p.v_row + (long)hk * p.v_head, t0, all, k_len, n, p.v_row * 2, 0);
    Ring<L::R, SB> to_a{0}, to_b{(L::R - 1) * SB}, at_r{SB}, at_t{0};
    // stages i + 3 + E of k and i + 2 + E of v: issued behind step i's barrier, in place E + 1 barriers later
    auto open = [&]() {
      st_k.next();
      st_v.next();
    };
    auto copy = [&](int k) {
      if (k < P)
        copy16(st_k.rs, sk.src(k), wlds + L::A + to_a.at + sk.dst(k));
      else if (k < 2 * P)
        copy16(st_v.rs, sv.src(k - P), wlds + L::B + to_b.at + sv.dst(k - P));
    };
#pragma unroll
    for (int j = 0; j < L::R; ++j) {
      st_k.next();
#pragma unroll
      for (int k = 0; k < P; ++k) copy16(st_k.rs, sk.src(k), wlds + L::A + j * SB + sk.dst(k));
    }
#pragma unroll
    for (int j = 0; j < L::R - 1; ++j) {
      st_v.next();
#pragma unroll
      for (int k = 0; k < P; ++k) copy16(st_v.rs, sv.src(k), wlds + L::B + j * SB + sv.dst(k));
    }
    bf16x8 f[2][D / 16];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const long rc = q_start + min(row0 + wave * 64 + nb * 32 + lq, q_len - 1);
      load_frags<D>(p.q + rc * p.q_row + (long)h * p.q_head, hh, f[nb]);
      take_sign<D>(f[nb], p.scale);
    }
    const float sl2 = score_scale(p.scale);
    bf16x8 bc[2][2];
    u32x4 bn[2][2];
    f32x16 s[2];
    RowReader<D> rr;
    TrReader<D> tr;
    RowAhead<D> ra;
    TrAhead<D> ta;
    rr.init(lane, lds0 + L::A);
    tr.init(lane, lds0 + L::B);
    auto none = [](int) {};
    auto nothing = []() {};
    auto next = [&]() {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) bc[nb][ks] = __builtin_bit_cast(bf16x8, bn[nb][ks]);
    };
    auto mask = [&](int j) {  // keys past the end of the sequence or the range
      const int left = j < n ? k_len - (t0 + j) * 32 : 0;
      if (left >= 32) return;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[nb][r] = 8 * (r >> 2) + 4 * hh + (r & 3) < left ? s[nb][r] : -INFINITY;
    };
    constexpr int LATE = kLate<D>, T = 32 - LATE;
    float most[2];  // largest exponent (score less m)
    float sub[2], x, last, late[LATE > 0 ? LATE : 1];
    auto val = [&](int e) { return e < T ? s[(e >> 2) & 1][4 * (e >> 3) + (e & 3)] : late[e < T ? 0 : e - T]; };
    auto arg = [&](int e) {
      const int nb = (e >> 2) & 1, r = 4 * (e >> 3) + (e & 3);
      const float y = __builtin_fmaf(s[nb][r], sl2, -sub[nb]);
      if (e < T)
        x = y;
      else
        late[e - T] = y;
      if (e & 1)
        most[nb] = fmaxf(fmaxf(most[nb], last), y);
      else
        last = y;
    };
    auto add = [&](int e) {  // P of score e is there
      const int nb = (e >> 2) & 1, r = 4 * (e >> 3) + (e & 3);
      l[nb] += val(e);
      if (r & 1) bn[nb][r >> 3][(r & 7) >> 1] = pack_bf(val(e - 1), val(e));
    };
    auto prob = [&](int e) {  // in the tr phase
      if (e == 0) arg(0);
      if (e < T) s[(e >> 2) & 1][4 * (e >> 3) + (e & 3)] = __builtin_amdgcn_exp2f(x);
      if (e < 31) arg(e + 1);
      if (e > 0 && e <= T) add(e - 1);
      if (e == 31 && T == 32) add(31);
    };
    auto prob_late = [&](int m) {  // behind MFMA m of the next row phase
#pragma unroll
      for (int e = T + m * LATE / (D / 8); e < T + (m + 1) * LATE / (D / 8); ++e) {
        late[e - T] = __builtin_amdgcn_exp2f(late[e - T]);
        asm volatile("" : "+v"(late[e - T]));  // not behind the branch of the mask
        if (e > T) add(e - 1);
        if (e == 31) add(31);
      }
    };
    // largest score of the query: the lane halves hold different keys
    auto both = [&](float v) {
      const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
    };
    step_sync();
    ra.read(rr);
    row_phase<D>(rr, ra, f, s, none, nothing);
    mask(0);
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      if (!again) {
        float x = s[nb][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) x = fmaxf(x, s[nb][r]);
        m[nb] = both(x) * sl2;
      }
      sub[nb] = m[nb] == -INFINITY ? 0.f : m[nb];  // only -inf scores so far: P = exp2(-inf) = 0
      most[nb] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) prob(e);
    // what bf16 drops of P, in 4s of scores: [wave][group][lane] 8 B
    char* const low = smem + L::LOW + wave * 4096 + lane * 8;
    auto save = [&](int from, int to) {
#pragma unroll
      for (int e = from; e < to; e += 4) {
        const int nb = (e >> 2) & 1, r = 4 * (e >> 3), w = (r & 7) >> 1;
        *(uint2*)(low + (e >> 2) * 512) = make_uint2(dropped(val(e), val(e + 1), bn[nb][r >> 3][w]),
                                                     dropped(val(e + 2), val(e + 3), bn[nb][r >> 3][w + 1]));
      }
    };
    if constexpr (FEW) save(0, T);
    if constexpr (LATE == 0) next();
    rr.move(SB);  // k stage i + 1
    ra.read(rr);
    for (int i = 0; i < n; ++i) {
      open();
      row_phase<D>(rr, ra, f, s, [&](int k) { prob_late(k); }, [&]() { ta.read(tr); });
      if constexpr (FEW && LATE > 0) save(T, 32);
      if constexpr (LATE > 0) next();
      rr.move(at_r.move());
      mask(i + 1);
      step_sync<E * 2 * P>();
      tr_phase<D>(
          tr, ta, bc, acc,
          [&](int k) {
            constexpr int GAP = (4 * ND) / (2 * P);
            if (k % GAP == 0 && k / GAP < 2 * P) copy(k / GAP);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (slot_of<D>(e) == k) prob(e);
          },
          [&]() { ra.read(rr); });
      if constexpr (FEW) {
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const uint2 y = *(const uint2*)(low + g * 512);
          u32x4 b = __builtin_bit_cast(u32x4, bc[g & 1][g >> 2]);
          b[g & 2] = y.x;
          b[(g & 2) + 1] = y.y;
          bc[g & 1][g >> 2] = __builtin_bit_cast(bf16x8, b);
        }
        save(0, T);
        ta.read(tr);
        settle();
        tr_phase<D>(tr, ta, bc, acc, none, nothing);
      }
      if constexpr (LATE == 0) next();
      tr.move(at_t.move());
      to_a.next();
      to_b.next();
    }
    // a score far above m in any wave (all copies land here, too: none may outlive the sweep)
    bool far = false;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const float x = both(most[nb]);
      far |= x > 40.f || (m[nb] == -INFINITY && x > m[nb]);
      largest[nb] = x + sub[nb];
    }
    far = __any(far);
    volatile LDS_AS unsigned char* flag = (volatile LDS_AS unsigned char*)(unsigned long)(lds0 + L::FLAG);
    if (lane == 0) flag[wave] = far && !again;
    step_sync();
    again = (flag[0] | flag[1] | flag[2] | flag[3]) != 0;
    if (again) {
      m[0] = largest[0];
      m[1] = largest[1];
    }
    step_sync();
  } while (again);
  acc_fence<ND>(acc);
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int row = row0 + wave * 64 + nb * 32 + lq;
    const bool live = row < q_len;
    const long rc = q_start + min(row, q_len - 1);
    const float sum = l[nb] + __shfl_xor(l[nb], 32, 64);  // the lane halves hold complementary keys
    if (ranges > 1) {
      store_part<D>(d.part_o + (((long)part * p.total_q + rc) * p.H + h) * D, acc[nb], 1.f, hh, live);
      if (live && hh == 0) d.part_ml[((long)part * p.H + h) * p.total_q + rc] = make_float2(m[nb], sum);
      continue;
    }
    store_row<D>(p.o + rc * p.o_row + (long)h * p.o_head, acc[nb], sum == 0.f ? 0.f : 1.f / sum, hh, live);
    if (live && hh == 0) p.lse[(long)h * p.total_q + rc] = sum == 0.f ? -INFINITY : (m[nb] + log2f(sum)) * kLn2;
  }
}

template <int D>
__global__ __launch_bounds__(kThreads, D == 64 ? 2 : 1) void attn_lse_kernel(TrainDev d, int blocks) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const AttnTrainParams& p = d.p;
  if ((int)blockIdx.x >= blocks) {
    zero_outside(p.o, p.o_row, p.o_head, p.cu_q, p.B, p.total_q, p.H, D, p.lse, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  FwdUnit u;
  if (!find_fwd_unit(d, &u)) return;
  int start, q_len, k_len;
  seq_range(p.cu_q, u.b, p.total_q, &start, &q_len);
  seq_range(p.cu_k, u.b, p.total_k, &start, &k_len);
  if (few((long)q_len * k_len * p.H, (long)q_len * p.H * D, false))
    lse_unit<D, true>(d, u, smem);
  else
    lse_unit<D, false>(d, u, smem);
}

// Joins the ranges of rows that were cut: out and lse from their sums, in range order
template <int D>
__global__ __launch_bounds__(kThreads) void attn_lse_join_kernel(TrainDev d) {
  const AttnTrainParams& p = d.p;
  constexpr int LANES = D / 8;
  const long item = ((long)blockIdx.x * kThreads + threadIdx.x) / LANES;
  const int col = threadIdx.x % LANES * 8;
  if (item >= (long)p.total_q * p.H) return;
  const int row = (int)(item / p.H), h = (int)(item % p.H);
  const int b = find_seq(p.cu_q, p.B, p.total_q, row);
  if (b < 0) return;
  int s, k_len;
  seq_range(p.cu_k, b, p.total_k, &s, &k_len);
  const int ranges = ranges_of((k_len + 31) / 32, d.stages, d.most);
  if (ranges < 2) return;
  const float2* ml = d.part_ml + (long)h * p.total_q + row;
  const long ml_step = (long)p.H * p.total_q, step = (long)p.total_q * p.H * D;
  float m = -INFINITY;
  for (int i = 0; i < ranges; ++i) m = fmaxf(m, ml[i * ml_step].x);
  const float sub = m == -INFINITY ? 0.f : m;
  const float* src = d.part_o + item * D + col;
  f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
  float sum = 0.f;
  for (int i = 0; i < ranges; ++i) {
    const float2 r = ml[i * ml_step];
    const float w = __builtin_amdgcn_exp2f(r.x - sub);
    sum += r.y * w;
    x += *(const f32x4*)(src + i * step) * w;
    y += *(const f32x4*)(src + i * step + 4) * w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  x *= inv;
  y *= inv;
  *(u32x4*)(p.o + (long)row * p.o_row + (long)h * p.o_head + col) =
      u32x4{pack2bf(x[0], x[1]), pack2bf(x[2], x[3]), pack2bf(y[0], y[1]), pack2bf(y[2], y[3])};
  if (col == 0) p.lse[(long)h * p.total_q + row] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
}

struct Plan {
  Cut q, k;
  long head_bytes, lse_bytes, qf_bytes, qp_bytes, kf_bytes, kp_bytes;  // kf, kp: dk and dv
  long total() const { return head_bytes + lse_bytes + qf_bytes + qp_bytes + kf_bytes + kp_bytes; }
};

// Room for ranges, from the average lengths (attn_delta_kernel knows the real ones and uses what it needs of it): three
// times what the average unit would take, none where that is under one, and none shorter than kMinRange stages in a
// sequence four times the average.
Plan make_plan(const AttnTrainParams& p) {
  Plan x;
  auto pad = [](long n) { return (n + 255) / 256 * 256; };
  const double sweep_q = p.total_k / 32. / p.B, sweep_k = p.total_q / 32. / p.B * (p.H / p.HK);
  const double units_q = ((double)(p.total_q / WROWS) + p.B) * p.H, units_k = ((double)(p.total_k / WROWS) + p.B) * p.HK;
  const double share = std::max(1., (units_q * sweep_q + units_k * sweep_k) / kCus);
  auto cut = [&](int total, int heads, double sweep) {
    Cut c{};
    c.full = total / WROWS;
    c.heads = heads;
    const double longest = std::min(sweep * 4, sweep * p.B) / kMinRange;
    auto ranges = [&](double want) { return (int)std::max(1., std::min({(double)kMaxRanges, want, longest})); };
    c.max_full = ranges(3 * sweep / (share / kFullShare));
    c.max_part = ranges((double)kCus / ((double)p.B * heads));
    return c;
  };
  x.q = cut(p.total_q, p.H, sweep_q);
  x.k = cut(p.total_k, p.HK, sweep_k);
  auto full_bytes = [&](const Cut& c, int total) {
    return c.max_full > 1 ? pad((long)c.max_full * total * c.heads * p.dim * 4) : 0;
  };
  auto part_bytes = [&](const Cut& c) {
    return c.max_part > 1 ? pad((long)c.max_part * p.B * WROWS * c.heads * p.dim * 4) : 0;
  };
  x.head_bytes = pad(256 + (long)p.B * 4 * 16);
  x.lse_bytes = pad((long)p.H * p.total_q * 8);
  x.qf_bytes = full_bytes(x.q, p.total_q);
  x.qp_bytes = part_bytes(x.q);
  x.kf_bytes = 2 * full_bytes(x.k, p.total_k);
  x.kp_bytes = 2 * part_bytes(x.k);
  return x;
}

// The forward pass's ranges, from the average lengths: as long as a CU's share of the work, in sequences up to four times the
// average, and none shorter than kFwdRange stages: a short batch of 512 keys takes 74 us in all in ranges of 8, 69 whole
// (each range costs its start and its share of the join). A sequence of 7 queries and 3000 keys between longer ones: 101 us
// whole, 59 + 6.5 in ranges.
constexpr int kFwdRange = 16;
struct FwdPlan {
  int tiles, most, stages;
  long o_bytes, ml_bytes, starts_bytes;
  long total() const { return o_bytes + ml_bytes + starts_bytes; }
};
FwdPlan make_fwd_plan(const AttnTrainParams& p) {
  FwdPlan x;
  x.tiles = p.total_q / 256 + p.B;
  const double sweep = p.total_k / 32. / p.B, units = (double)x.tiles * p.H;
  x.stages = (int)std::max((double)kFwdRange, std::min(units * sweep / kCus, 1e9));
  const double longest = std::min(sweep * 4, sweep * p.B) / x.stages;
  x.most = (int)std::max(1., std::min((double)kMaxRanges, longest));
  auto pad = [](long n) { return (n + 255) / 256 * 256; };
  x.o_bytes = x.most > 1 ? pad((long)x.most * p.total_q * p.H * p.dim * 4) : 0;
  x.ml_bytes = x.most > 1 ? pad((long)x.most * p.total_q * p.H * 8) : 0;
  x.starts_bytes = p.B > 64 ? pad((p.B + 1L) * 4) : 0;
  return x;
}

int check(const AttnTrainParams& p) {
  FLITE_REQUIRE(p.dim == 64 || p.dim == 128 || p.dim == 256, "attention: head size must be 64, 128 or 256");
  FLITE_REQUIRE(p.B > 0 && p.H > 0 && p.HK > 0 && p.H % p.HK == 0,
                "attention: batch, heads and kv heads must be positive, heads a multiple of kv heads");
  FLITE_REQUIRE(p.total_q >= 0 && p.total_k >= 0, "attention: rows must not be negative");
  FLITE_REQUIRE(((long)p.total_q / WROWS + p.B) * p.H < (1L << 29) / kMaxRanges &&
                    ((long)p.total_k / WROWS + p.B) * p.HK < (1L << 29) / kMaxRanges,
                "attention: too many rows, sequences or heads");
  FLITE_REQUIRE(p.cu_q && p.cu_k, "attention: cu_seqlens missing");
  return 0;
}

int check_rows(const void* ptr, long row, long head, int dim, bool any, const char* what) {
  FLITE_REQUIRE(!any || ptr, std::string("attention: missing ") + what);
  FLITE_REQUIRE(((uintptr_t)ptr & 15) == 0 && row % 8 == 0 && head % 8 == 0 && row >= dim && head >= 0 && row <= (1 << 22),
                std::string("attention: ") + what +
                    " must be 16-byte aligned, its row and head strides multiples of 8, the row stride dim to 2^22");
  return 0;
}

template <typename F>
int lds_limit(F* f, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  FLITE_HIP_CHECK(hipGetDevice(&dev));
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load() & bit) return 0;
  FLITE_HIP_CHECK(hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit);
  return 0;
}

constexpr int kZeroBlocks = 32;

template <int D>
int launch_fwd(const TrainDev& d, hipStream_t s) {
  constexpr int lds = FwdLds<D>::TOTAL;
  static std::atomic<unsigned long long> done{0};
  if (lds_limit(attn_lse_kernel<D>, lds, done)) return 1;
  const AttnTrainParams& p = d.p;
  const int blocks = d.tiles * p.H * d.most;
  if (p.B > 64) hipLaunchKernelGGL(attn_lse_units_kernel, dim3(1), dim3(kThreads), 0, s, d);
  FLITE_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(attn_lse_kernel<D>, dim3(blocks + (p.zero_outside ? kZeroBlocks : 0)), dim3(kThreads), lds, s, d, blocks);
  FLITE_HIP_CHECK(hipGetLastError());
  if (d.most > 1)
    hipLaunchKernelGGL(attn_lse_join_kernel<D>, dim3((unsigned)(((long)p.total_q * p.H * (D / 8) + kThreads - 1) / kThreads)),
                       dim3(kThreads), 0, s, d);
  FLITE_HIP_CHECK(hipGetLastError());
  return 0;
}

template <int D>
int launch_bwd(const TrainDev& d, hipStream_t s) {
  const AttnTrainParams& p = d.p;
  constexpr int lds = Lds<D>::TOTAL;
  static std::atomic<unsigned long long> done{0};
  if (lds_limit(attn_bwd_kernel<D>, lds, done)) return 1;
  auto blocks = [](long rows_heads) { return (int)((rows_heads * (D / 8) + kThreads - 1) / kThreads); };
  const int q_rows = blocks((long)p.total_q * p.H);
  const int extra = p.zero_outside ? kZeroBlocks : 1;
  hipLaunchKernelGGL(attn_delta_kernel<D>, dim3(extra + q_rows), dim3(kThreads), 0, s, d, extra);
  FLITE_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(attn_bwd_kernel<D>, dim3(d.k.blocks(p.B) + d.q.blocks(p.B)), dim3(kThreads), lds, s, d);
  FLITE_HIP_CHECK(hipGetLastError());
  JoinItems j;
  j.q_full = d.q.max_full > 1 ? q_rows : 0;
  j.q_part = d.q.max_part > 1 ? blocks((long)p.B * WROWS * p.H) : 0;
  j.k_full = d.k.max_full > 1 ? blocks((long)p.total_k * p.HK) : 0;
  j.k_part = d.k.max_part > 1 ? blocks((long)p.B * WROWS * p.HK) : 0;
  const int join = j.q_full + j.q_part + j.k_full + j.k_part;
  if (join > 0) hipLaunchKernelGGL(attn_join_kernel<D>, dim3(join), dim3(kThreads), 0, s, d, j);
  FLITE_HIP_CHECK(hipGetLastError());
  return 0;
}

}  // namespace

long attn_train_workspace_bytes(const AttnTrainParams& p) {
  if (check(p)) return -1;
  return make_plan(p).total();
}

long attn_train_fwd_workspace_bytes(const AttnTrainParams& p) {
  if (check(p)) return -1;
  return make_fwd_plan(p).total();
}

int attn_train_fwd(const AttnTrainParams& p, void* ws, long ws_bytes, hipStream_t s) {
  if (int rc = check(p)) return rc;
  const bool any_q = p.total_q > 0, any_k = p.total_k > 0;
  if (int rc = check_rows(p.q, p.q_row, p.q_head, p.dim, any_q, "q")) return rc;
  if (int rc = check_rows(p.k, p.k_row, p.k_head, p.dim, any_k, "k")) return rc;
  if (int rc = check_rows(p.v, p.v_row, p.v_head, p.dim, any_k, "v")) return rc;
  if (int rc = check_rows(p.o, p.o_row, p.o_head, p.dim, any_q, "out")) return rc;
  FLITE_REQUIRE(p.lse || !any_q, "attention: missing lse");
  if (!any_q) return 0;
  const FwdPlan x = make_fwd_plan(p);
  FLITE_REQUIRE(x.total() == 0 || (ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= x.total()),
                "attention: workspace missing, not 256-byte aligned, or too small");
  TrainDev d{};
  d.p = p;
  d.tiles = x.tiles;
  d.most = x.most;
  d.stages = x.stages;
  d.part_o = (float*)ws;
  d.part_ml = (float2*)((char*)ws + x.o_bytes);
  d.starts = (int*)((char*)ws + x.o_bytes + x.ml_bytes);
  if (p.dim == 64) return launch_fwd<64>(d, s);
  if (p.dim == 128) return launch_fwd<128>(d, s);
  return launch_fwd<256>(d, s);
}

int attn_train_bwd(const AttnTrainParams& p, void* ws, long ws_bytes, hipStream_t s) {
  if (int rc = check(p)) return rc;
  const bool any_q = p.total_q > 0, any_k = p.total_k > 0;
  if (int rc = check_rows(p.q, p.q_row, p.q_head, p.dim, any_q, "q")) return rc;
  if (int rc = check_rows(p.k, p.k_row, p.k_head, p.dim, any_k, "k")) return rc;
  if (int rc = check_rows(p.v, p.v_row, p.v_head, p.dim, any_k, "v")) return rc;
  if (int rc = check_rows(p.o, p.o_row, p.o_head, p.dim, any_q, "out")) return rc;
  if (int rc = check_rows(p.dout, p.do_row, p.do_head, p.dim, any_q, "dout")) return rc;
  if (int rc = check_rows(p.dq, p.dq_row, p.dq_head, p.dim, any_q, "dq")) return rc;
  if (int rc = check_rows(p.dk, p.dk_row, p.dk_head, p.dim, any_k, "dk")) return rc;
  if (int rc = check_rows(p.dv, p.dv_row, p.dv_head, p.dim, any_k, "dv")) return rc;
  FLITE_REQUIRE(p.lse || !any_q, "attention: missing lse");
  const Plan x = make_plan(p);
  FLITE_REQUIRE(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= x.total(),
                "attention backward: workspace missing, not 256-byte aligned, or too small");
  TrainDev d{};
  d.p = p;
  d.q = x.q;
  d.k = x.k;
  char* at = (char*)ws;
  auto take = [&](long n) {
    char* r = at;
    at += n;
    return r;
  };
  d.target = (int*)take(x.head_bytes);
  d.groups = (int4*)(d.target + 64);
  d.lse2 = (float*)take(x.lse_bytes);
  d.delta = d.lse2 + (long)p.H * p.total_q;
  d.q.ws_full = (float*)take(x.qf_bytes);
  d.q.ws_part = (float*)take(x.qp_bytes);
  d.k.ws_full = (float*)take(x.kf_bytes);
  d.k.ws_part = (float*)take(x.kp_bytes);
  if (p.dim == 64) return launch_bwd<64>(d, s);
  if (p.dim == 128) return launch_bwd<128>(d, s);
  return launch_bwd<256>(d, s);
}

}  // namespace flite
