// Group normalisation with an activation over node features [N, C], channels last:
//   y = act((x - mean) / sqrt(var + eps) * weight[c] + bias[c])
// with mean and (biased) variance over the C / groups channels of a group, either
// of each node on its own, or of all nodes of a graph of a batch (graph_ptr, ragged).
//
// Statistics: each lane folds a batch of rows' mean and squared deviations about it
// into its running ones (the pairwise update of mean and M2), so nothing is
// subtracted from a large sum; lanes, warps, then pieces, are joined the same way.
// The result is the same every time: no floating-point atomics.
//
// Batch mode: rows are cut into windows, one block each. A graph of at most kShort
// nodes belongs to the block in whose window it starts and is finished there, from
// registers where its rows fit them (8 warps x U rows), else with a second read from
// L1 / L2; so is a longer one that lies inside the window. Another graph leaves a piece
// per window in the workspace; a second kernel joins the pieces, a third reads x again
// and writes. So a long graph costs three passes over its rows where x exceeds the L2.
//
// Measured on one B200: 232,965 nodes x 256 on their own, SiLU, 84-88 us = 0.83 of copy
// bandwidth; one graph of 2,449,029 x 128 602 us, three passes at 0.95 of it (joining its
// pieces 11 us); 8,192 ragged graphs, 200,003 x 100, GELU, 114 us (108 on the device), bound by
// latency: 24 warps an SM, each of which waits for a graph's statistics before it writes its rows.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"

namespace gnnb200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kSmallGroup = 4;    // channels per group for which a mean rounded to 32 bits is not good enough
constexpr int kShort = 64;        // the longest graph that one block finishes
constexpr int kTile = 1024;       // channels per column tile at most (whole groups)
constexpr int kFewPieces = 64;    // pieces that one warp joins
constexpr int kMaxWindow = 512;   // rows per block at most
constexpr int kMaxLongs = kMaxWindow / kShort + 2;  // long graphs that meet a window

struct NormArgs {
  const float* x;
  const float* weight;
  const float* bias;
  float* out;
  const void* ptr;    // graph offsets, batch mode
  int wide_ptr;       // they are int64
  int64_t graphs;
  int64_t n;
  int c, groups, cg;  // channels, groups, channels per group
  int tile_groups;    // groups per column tile
  float eps;
  int act;
  int window;         // rows per block (a multiple of kShort)
  int64_t windows;
  float2* part;       // [windows, 2, groups]: (mean, M2) of a split graph's piece: it began earlier / it begins here
  float2* fin;        // [windows, groups]: (mean, 1 / sqrt(var + eps)) of the split graph that begins in the window
};

// y * Phi(y), Phi being the normal distribution function, as max(y, 0) - |y| * Phi(-|y|): nothing
// cancels for negative y. Phi(-z) = exp(-z^2 / 2) * P(z) / Q(z), a rational function fitted to the
// ratio by weighted least squares on [0, 8]: off by 1.4e-7 of itself there, 1.5e-5 at 14. The
// exponential's argument is rounded to 32 bits, which adds z^2 * 1e-7. Against 1 + erf, whose
// error is 1e-5 of the result at -3. Past 20 Phi(-z) is 0.
__device__ __forceinline__ float gelu(float y) {
  const float z = fminf(fabsf(y), 20.0f);
  const float p = fmaf(fmaf(fmaf(0.014852066524326801f, z, 0.11001348495483398f), z, 0.34495601058006287f), z,
                       0.4999999403953552f);
  const float r = fmaf(fmaf(0.037241388112306595f, z, 0.2753705382347107f), z, 0.9071747064590454f);
  const float q = fmaf(fmaf(r, z, 1.4877893924713135f), z, 1.0f);
  return (y < 0.0f ? 0.0f : y) - z * __fdividef(p, q) * __expf(-0.5f * z * z);
}

template <int ACT>
__device__ __forceinline__ float activate(float y) {
  if constexpr (ACT == GNN_ACT_RELU) return y < 0.0f ? 0.0f : y;
  // the exponential's argument is rounded to 32 bits: |y| * 1e-7 of the result (a correct division and
  // exponential cost 7 to 20 % of a node norm); below -87, where less than 1e-36 is left, it is 0
  if constexpr (ACT == GNN_ACT_SILU) return __fdividef(y, 1.0f + __expf(-y));
  if constexpr (ACT == GNN_ACT_GELU) return gelu(y);
  return y;
}

// Calls f with the activation as a compile-time constant.
template <class F>
__device__ __forceinline__ void with_activation(int act, F f) {
  switch (act) {
    case GNN_ACT_RELU: f(std::integral_constant<int, GNN_ACT_RELU>{}); break;
    case GNN_ACT_SILU: f(std::integral_constant<int, GNN_ACT_SILU>{}); break;
    case GNN_ACT_GELU: f(std::integral_constant<int, GNN_ACT_GELU>{}); break;
    default: f(std::integral_constant<int, GNN_ACT_NONE>{}); break;
  }
}

__device__ __forceinline__ int64_t ptr_at(const NormArgs& a, int64_t g) {
  const int64_t v = a.wide_ptr ? __ldg(static_cast<const int64_t*>(a.ptr) + g)
                               : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(a.ptr) + g));
  return v < 0 ? 0 : (v > a.n ? a.n : v);
}

// The first graph whose end lies past `row` (graphs where there is none): every lane
// of the warp asks at another place, five bits a round.
__device__ __forceinline__ int64_t graph_of(const NormArgs& a, int64_t row) {
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, hi = a.graphs;  // the answer is in [lo, hi]
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32;
    const int64_t at = min(lo + lane * step + step - 1, hi - 1);
    const unsigned past = __ballot_sync(kFull, ptr_at(a, at + 1) > row);
    if (past == 0) return hi;
    const int first = __ffs(past) - 1;
    hi = min(lo + first * step + step - 1, hi - 1);
    lo = min(lo + first * step, hi);
    if (step == 1) return hi;
  }
  return lo;
}

// A warp's view of one column tile: lane l holds the channels
// c0 + CH * (l + 32 j) .. + CH, j < NV. WHOLE: a chunk of CH channels lies in one
// group. What belongs to a group is kept once a chunk (WHOLE) or once a channel.
template <int CH, int NV, bool WHOLE>
struct Tile {
  static constexpr int E = WHOLE ? 1 : CH;
  int c0, cols;     // first channel, channels
  int g0, groups;   // first group, groups
  int cg;           // channels per group
  int lane;
  int gsize;        // WHOLE: chunks per group
  bool pow2;        // WHOLE: a group is an aligned power of two of at most 32 lanes
  int grp[NV];      // group (in the tile) of chunk lane + 32 j (of its first channel)
  uint32_t delta[NV];  // !WHOLE: how many groups further channel e is, two bits each
  float* sh;        // this warp's scratch: partials, totals

  __device__ __forceinline__ bool live(int j) const { return (lane + 32 * j) * CH < cols; }
  __device__ __forceinline__ int channel(int j) const { return c0 + CH * (lane + 32 * j); }
  __device__ __forceinline__ int group(int j, int e) const {
    return WHOLE ? grp[j] : grp[j] + static_cast<int>((delta[j] >> (2 * e)) & 3u);
  }
  // channel e of chunk j is the first of its group
  __device__ __forceinline__ bool leads(int j, int e) const {
    return WHOLE ? (lane + 32 * j) % gsize == 0 : CH * (lane + 32 * j) + e == group(j, e) * cg;
  }

  __device__ __forceinline__ void init(const NormArgs& a, float* scratch) {
    lane = threadIdx.x & 31;
    g0 = static_cast<int>(blockIdx.y) * a.tile_groups;
    groups = min(a.tile_groups, a.groups - g0);
    cg = a.cg;
    c0 = g0 * cg;
    cols = groups * cg;
    gsize = WHOLE ? cg / CH : 1;
    pow2 = gsize <= 32 && (gsize & (gsize - 1)) == 0;
    sh = scratch;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int ch = CH * (lane + 32 * j);
      grp[j] = ch / cg;
      delta[j] = 0;
      if constexpr (!WHOLE) {
#pragma unroll
        for (int e = 1; e < CH; ++e) delta[j] |= static_cast<uint32_t>((ch + e) / cg - grp[j]) << (2 * e);
      }
    }
  }

  // Takes the mean of its group off each value of a row, for groups of 2 to kSmallGroup channels.
  // These often lie close together, and rstd (up to 316) then magnifies a mean rounded to 32 bits;
  // counted from the group's first value it is rounded in proportion to their spread.
  __device__ __forceinline__ void center_small(float (&v)[NV][CH]) const {
    const float inv = 1.0f / static_cast<float>(cg);
    if constexpr (WHOLE) {
      float from[NV], sum[NV][1];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        from[j] = v[j][0];  // a chunk of kSmallGroup channels is its group
        if constexpr (CH < kSmallGroup) {
          if (pow2) {
            from[j] = __shfl_sync(kFull, from[j], lane & ~(gsize - 1));
          } else if (live(j) && leads(j, 0)) {
            sh[grp[j]] = from[j];
          }
        }
      }
      if (CH < kSmallGroup && !pow2) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NV; ++j) from[j] = live(j) ? sh[grp[j]] : 0.0f;
        __syncwarp();
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        sum[j][0] = 0.0f;
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          v[j][e] -= from[j];
          if (live(j)) sum[j][0] += v[j][e];
        }
      }
      if constexpr (CH < kSmallGroup) group_sum(sum);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < CH; ++e) v[j][e] = fmaf(-sum[j][0], inv, v[j][e]);
      }
    } else {
      // a lane per group: its first value and the mean from there (at most a group for every two channels)
      float2* tot = reinterpret_cast<float2*>(sh + 32 * NV * CH);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < CH; ++e) sh[(lane + 32 * j) * CH + e] = v[j][e];
      }
      __syncwarp();
      for (int g = lane; g < groups; g += 32) {
        const float from = sh[g * cg];
        float s = 0.0f;
        for (int i = 1; i < cg; ++i) s += sh[g * cg + i] - from;
        tot[g] = make_float2(from, s * inv);
      }
      __syncwarp();
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          const float2 m = live(j) ? tot[group(j, e)] : make_float2(0.0f, 0.0f);
          v[j][e] = v[j][e] - m.x - m.y;
        }
      }
      __syncwarp();
    }
  }

  // p[j][e]: this lane's partials -> the totals of their groups
  __device__ __forceinline__ void group_sum(float (&p)[NV][E]) const {
    if (WHOLE && pow2) {
      for (int o = 1; o < gsize; o <<= 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) p[j][0] += __shfl_xor_sync(kFull, p[j][0], o);
      }
      return;
    }
    if (groups == 1) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < E; ++e) s += live(j) ? p[j][e] : 0.0f;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < E; ++e) p[j][e] = s;
      }
      return;
    }
    const int each = WHOLE ? gsize : cg;  // partials per group
    float* tot = sh + 32 * NV * E;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) sh[(lane + 32 * j) * E + e] = p[j][e];
    }
    __syncwarp();
    int per = 1;  // lanes per group
    while (per * 2 * min(groups, 32) <= 32) per *= 2;
    const int at = lane / per, t = lane & (per - 1);
    for (int base = 0; base < groups; base += 32 / per) {
      const int g = base + at;
      float s = 0.0f;
      if (g < groups) {
        for (int i = t; i < each; i += per) s += sh[g * each + i];
      }
      for (int o = 1; o < per; o <<= 1) s += __shfl_xor_sync(kFull, s, o);
      if (t == 0 && g < groups) tot[g] = s;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) p[j][e] = live(j) ? tot[group(j, e)] : 0.0f;
    }
    __syncwarp();
  }
};

// partials and totals of group_sum (at most a group per partial), per warp
template <int CH, int NV, bool WHOLE>
constexpr int scratch_floats() {
  return 2 * 32 * NV * (WHOLE ? 1 : CH);
}

template <int CH>
__device__ __forceinline__ void load_chunk(const float* p, float (&v)[CH]) {
  if constexpr (CH == 4) {
    const float4 t = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = t.x;
    v[1] = t.y;
    v[2] = t.z;
    v[3] = t.w;
  } else if constexpr (CH == 2) {
    const float2 t = __ldg(reinterpret_cast<const float2*>(p));
    v[0] = t.x;
    v[1] = t.y;
  } else {
    v[0] = __ldg(p);
  }
}

template <int CH>
__device__ __forceinline__ void store_chunk(float* p, const float (&v)[CH]) {
  if constexpr (CH == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else if constexpr (CH == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else {
    *p = v[0];
  }
}

template <int CH, int NV, bool WHOLE>
__device__ __forceinline__ void load_affine(const NormArgs& a, const Tile<CH, NV, WHOLE>& t, float (&w)[NV][CH],
                                            float (&b)[NV][CH]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      w[j][e] = (a.weight != nullptr && t.live(j)) ? __ldg(a.weight + t.channel(j) + e) : 1.0f;
      b[j][e] = (a.bias != nullptr && t.live(j)) ? __ldg(a.bias + t.channel(j) + e) : 0.0f;
    }
  }
}

// Rows of a warp in flight, and blocks per SM that the registers have to allow. Measured
// on the ragged batch (200,003 rows, 8,192 graphs): where a chunk lies in one group (C =
// 128, no activation) 8 rows and 3 blocks 82 us, 4 rows and 3 blocks 89 us, 8 rows and 2
// blocks 90 us; where it does not (C = 100, GELU), which takes more registers, 4 rows and
// 3 blocks 119 us, 8 rows and 3 blocks (spilling) 165 us, 8 rows and 2 blocks 145 us.
template <int CH, int NV, bool WHOLE>
constexpr int batch_rows() {
  return NV * CH <= 4 ? (WHOLE ? 8 : 4) : (NV * CH <= 8 ? 4 : (NV * CH <= 16 ? 2 : 1));
}
template <int CH, int NV, bool WHOLE>
constexpr int min_blocks() {
  return CH * NV <= 4 ? 3 : (CH * NV <= 8 ? 2 : 1);
}

// ---- each node on its own: one warp per row, R rows in flight ----------------
//
// SMALL: groups of 2 to kSmallGroup channels. Measured with it and without: 300 channels in 100
// groups 302 and 339 us, 192 in 96 265 and 290 us, 512 in 128 80.6 and 82.0 us (200,000, 300,000
// and 100,000 nodes); for wider groups, whose spread is seldom so small, it is left out (16 of
// 256: 3 % slower).
template <int CH, int NV, bool WHOLE, bool SMALL>
__global__ void __launch_bounds__(kThreads, CH * NV <= 8 ? 4 : (CH * NV <= 16 ? 2 : 1)) norm_rows_kernel(NormArgs a) {
  constexpr int R = NV * CH <= 4 ? 4 : (NV * CH <= 8 ? 2 : 1);
  constexpr int E = WHOLE ? 1 : CH;
  extern __shared__ float scratch[];
  Tile<CH, NV, WHOLE> t;
  t.init(a, scratch + (threadIdx.x >> 5) * scratch_floats<CH, NV, WHOLE>());
  float w[NV][CH], b[NV][CH];
  load_affine(a, t, w, b);
  const float inv = 1.0f / static_cast<float>(a.cg);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps * R;
  for (int64_t r0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * R; r0 < a.n; r0 += step) {
    float v[R][NV][CH];
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (t.live(j) && r0 + i < a.n) load_chunk<CH>(a.x + (r0 + i) * a.c + t.channel(j), v[i][j]);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (r0 + i >= a.n) break;
      if constexpr (SMALL) {
        t.center_small(v[i]);
      } else {
        float p[NV][E];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
          for (int e = 0; e < E; ++e) p[j][e] = 0.0f;
          if (t.live(j)) {
#pragma unroll
            for (int e = 0; e < CH; ++e) p[j][e % E] += v[i][j][e];
          }
        }
        t.group_sum(p);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
          for (int e = 0; e < CH; ++e) v[i][j][e] -= p[j][e % E] * inv;
        }
      }
      float q[NV][E];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < E; ++e) q[j][e] = 0.0f;
        if (t.live(j)) {
#pragma unroll
          for (int e = 0; e < CH; ++e) q[j][e % E] = fmaf(v[i][j][e], v[i][j][e], q[j][e % E]);
        }
      }
      t.group_sum(q);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (t.live(j)) {
#pragma unroll
          for (int e = 0; e < E; ++e) q[j][e] = rsqrtf(fmaf(q[j][e], inv, a.eps));
#pragma unroll
          for (int e = 0; e < CH; ++e) v[i][j][e] = fmaf(v[i][j][e] * q[j][e % E], w[j][e], b[j][e]);
        }
      }
      with_activation(a.act, [&](auto act) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (t.live(j)) {
#pragma unroll
            for (int e = 0; e < CH; ++e) v[i][j][e] = activate<decltype(act)::value>(v[i][j][e]);
            store_chunk<CH>(a.out + (r0 + i) * a.c + t.channel(j), v[i][j]);
          }
        }
      });
    }
  }
}

// ---- each node on its own, few channels: a thread per group ------------------
//
// A warp per row would leave most lanes idle (or join groups through shared memory row
// by row), so a block takes a tile of whole rows into shared memory, a thread
// normalises one group of one row there, and the tile is written back. Measured: 1,187,608
// nodes x 27 in 3 groups 467 us with a warp per row, 91 us here; 316,025 x 32 in 32 groups
// 116 and 66 us. Bound by instructions and shared memory: two passes over a group's values
// and one back, one word at a time.
constexpr int kNarrowFloats = 8192;  // a tile: 32 KB
constexpr int kNarrowChannels = 128;
constexpr int kNarrowGroup = 32;     // channels per group at most

__global__ void __launch_bounds__(kThreads) norm_narrow_kernel(NormArgs a, int tile_rows, int vec) {
  extern __shared__ float4 tile4[];
  float* const tile = reinterpret_cast<float*>(tile4);
  const float inv = 1.0f / static_cast<float>(a.cg);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * tile_rows; r0 < a.n;
       r0 += static_cast<int64_t>(gridDim.x) * tile_rows) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(tile_rows), a.n - r0));
    const int count = rows * a.c;
    const float* src = a.x + r0 * a.c;
    float* dst = a.out + r0 * a.c;
    const int whole = vec ? count / 4 : 0;  // 16-byte pieces
    for (int i = threadIdx.x; i < whole; i += kThreads) tile4[i] = __ldcs(reinterpret_cast<const float4*>(src) + i);
    for (int i = whole * 4 + threadIdx.x; i < count; i += kThreads) tile[i] = __ldcs(src + i);
    __syncthreads();
    with_activation(a.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      // pair p is group p % groups of row p / groups: its values start at p * cg
      for (int p = threadIdx.x; p < rows * a.groups; p += kThreads) {
        float* v = tile + p * a.cg;
        const int ch = (p % a.groups) * a.cg;
        // each thread starts at another place of its group, so that groups whose size shares
        // factors with the 32 banks do not meet in one
        const int first = p % a.cg;
        auto next = [&](int i) { return i + 1 == a.cg ? 0 : i + 1; };
        const float from = v[0];  // the mean is counted from the first value (center_small)
        float sum = 0.0f, dev = 0.0f;
        for (int k = 0, i = first; k < a.cg; ++k, i = next(i)) sum += v[i] - from;
        const float mean = sum * inv;
        for (int k = 0, i = first; k < a.cg; ++k, i = next(i)) {
          const float d = v[i] - from - mean;
          dev = fmaf(d, d, dev);
        }
        const float rstd = rsqrtf(fmaf(dev, inv, a.eps));
        for (int k = 0, i = first; k < a.cg; ++k, i = next(i)) {
          const float w = a.weight != nullptr ? __ldg(a.weight + ch + i) : 1.0f;
          const float b = a.bias != nullptr ? __ldg(a.bias + ch + i) : 0.0f;
          v[i] = activate<ACT>(fmaf((v[i] - from - mean) * rstd, w, b));
        }
      }
    });
    __syncthreads();
    for (int i = threadIdx.x; i < whole; i += kThreads) __stcs(reinterpret_cast<float4*>(dst) + i, tile4[i]);
    for (int i = whole * 4 + threadIdx.x; i < count; i += kThreads) __stcs(dst + i, tile[i]);
    __syncthreads();
  }
}

// ---- graphs of a batch ------------------------------------------------------

// The rows of a span, shared by a team: warp i of `size` takes rows i, i + size, ...
// The team is the block, or a warp by itself.
template <int CH, int NV, bool WHOLE>
struct Team {
  static constexpr int E = WHOLE ? 1 : CH;
  static constexpr int U = batch_rows<CH, NV, WHOLE>();
  Tile<CH, NV, WHOLE> t;
  float2* joint;  // [2][kWarps][groups in the tile]: (mean, M2) of the warps' rows
  int flip;       // which half of `joint` is next
  int size;       // kWarps or 1
  int warp;       // this warp's place in the team
  float v[U][NV][CH];

  __device__ __forceinline__ int keep() const { return size * U; }  // rows that stay in registers

  // every size-th of `rows` rows
  __device__ __forceinline__ int count(int rows) const { return size == 1 ? rows : (rows + kWarps - 1) / kWarps; }

  // `cnt` rows (U of them where FULL), `step` floats apart, the first at p
  template <bool FULL>
  __device__ __forceinline__ void load(const float* p, int64_t step, int cnt) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if ((FULL || u < cnt) && t.live(j)) load_chunk<CH>(p + u * step + 32 * CH * j, v[u][j]);
      }
    }
  }

  // folds the rows in v into the running (m, s) of n rows a channel; the quick divisions are good to two
  // units in the last place, like the sums around them
  template <bool FULL>
  __device__ __forceinline__ void fold(int cnt, float& n, float (&m)[NV][CH], float (&s)[NV][CH]) {
    const float cf = FULL ? static_cast<float>(U) : static_cast<float>(cnt);
    const float icf = FULL ? 1.0f / U : __fdividef(1.0f, cf);
    const float nn = n + cf;
    const float share = __fdividef(cf, nn);
    const float both = n * share;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!t.live(j)) continue;
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (FULL || u < cnt) sum += v[u][j][e];
        }
        const float mb = sum * icf;
        float dev = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (FULL || u < cnt) {
            const float d = v[u][j][e] - mb;
            dev = fmaf(d, d, dev);
          }
        }
        const float d = mb - m[j][e];
        m[j][e] = fmaf(d, share, m[j][e]);
        s[j][e] += fmaf(d * d, both, dev);
      }
    }
    n = nn;
  }

  // (mean, M2) of the groups over `rows` rows from row beg, the same in every warp; the
  // last batch of rows is left in v
  __device__ __forceinline__ void stats(const NormArgs& a, int64_t beg, int rows, float (&mean)[NV][E],
                                        float (&m2)[NV][E]) {
    float m[NV][CH], s[NV][CH];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < CH; ++e) m[j][e] = s[j][e] = 0.0f;
    }
    float n = 0.0f;
    const int64_t step = static_cast<int64_t>(size) * a.c;
    const float* p = a.x + (beg + warp) * a.c + t.channel(0);
    int left = rows > warp ? count(rows - warp) : 0;
    for (; left >= U; left -= U, p += U * step) {
      load<true>(p, step, U);
      fold<true>(U, n, m, s);
    }
    if (left > 0) {
      load<false>(p, step, left);
      fold<false>(left, n, m, s);
    }
    // the channels of a group: n values each
    const float icg = 1.0f / static_cast<float>(a.cg);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) mean[j][e] = 0.0f;
      if (t.live(j)) {
#pragma unroll
        for (int e = 0; e < CH; ++e) mean[j][e % E] += m[j][e];
      }
    }
    t.group_sum(mean);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        mean[j][e] *= icg;
        m2[j][e] = 0.0f;
      }
      if (t.live(j)) {
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          const float d = m[j][e] - mean[j][e % E];
          m2[j][e % E] += fmaf(d * d, n, s[j][e]);
        }
      }
    }
    t.group_sum(m2);
    if (size == 1) return;
    // the warps: warp i has the rows beg + i, beg + i + 8, ...
    const int stride = a.tile_groups;
    float2* half = joint + flip * kWarps * stride;
    flip ^= 1;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (t.live(j) && t.leads(j, e)) half[warp * stride + t.group(j, e)] = make_float2(mean[j][e], m2[j][e]);
      }
    }
    __syncthreads();
    const float inv = 1.0f / static_cast<float>(rows);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (!t.live(j)) continue;
        const float2* p = half + t.group(j, e);
        float sum = 0.0f, dev = 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          const float ni = static_cast<float>((rows - i + kWarps - 1) / kWarps);
          if (i < rows) sum = fmaf(ni, p[i * stride].x, sum);
        }
        const float mu = sum * inv;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          const float ni = static_cast<float>((rows - i + kWarps - 1) / kWarps) * static_cast<float>(a.cg);
          const float d = p[i * stride].x - mu;
          if (i < rows) dev += fmaf(d * d, ni, p[i * stride].y);
        }
        mean[j][e] = mu;
        m2[j][e] = dev;
      }
    }
  }

  // act((v - mean) * scale + shift) of the batch in v, stored at q, q + step, ...
  template <int ACT, bool FULL>
  __device__ __forceinline__ void put(float* q, int64_t step, int cnt, const float (&mean)[NV][E],
                                      const float (&scale)[NV][CH], const float (&shift)[NV][CH]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!FULL && u >= cnt) break;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (t.live(j)) {
#pragma unroll
          for (int e = 0; e < CH; ++e) {
            v[u][j][e] = activate<ACT>(fmaf(v[u][j][e] - mean[j][e % E], scale[j][e], shift[j][e]));
          }
          store_chunk<CH>(q + u * step + 32 * CH * j, v[u][j]);
        }
      }
    }
  }

  // Normalises `rows` rows from row beg, which are still in v where `kept`. The mean is taken
  // off first: folded into the affine part, it was rounded once more (a group of equal
  // values far from 0 was off by 316 of its units), for 1 % of the time of a ragged batch.
  __device__ __forceinline__ void apply(const NormArgs& a, int64_t beg, int rows, bool kept, const float (&mean)[NV][E],
                                        const float (&rstd)[NV][E], const float (&w)[NV][CH],
                                        const float (&b)[NV][CH]) {
    float scale[NV][CH];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        scale[j][e] = rstd[j][e % E] * w[j][e];
      }
    }
    const int64_t step = static_cast<int64_t>(size) * a.c;
    const int64_t at = (beg + warp) * a.c + t.channel(0);
    const int mine = rows > warp ? count(rows - warp) : 0;
    with_activation(a.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      const float* p = a.x + at;
      float* q = a.out + at;
      int left = mine;
      for (; left >= U; left -= U, p += U * step, q += U * step) {
        if (!kept) load<true>(p, step, U);
        put<ACT, true>(q, step, U, mean, scale, b);
      }
      if (left > 0) {
        if (!kept) load<false>(p, step, left);
        put<ACT, false>(q, step, left, mean, scale, b);
      }
    });
  }

  __device__ __forceinline__ void init(const NormArgs& a, float* shared) {
    warp = threadIdx.x >> 5;
    size = kWarps;
    flip = 0;
    joint = reinterpret_cast<float2*>(shared);
    t.init(a, shared + 4 * kWarps * a.tile_groups + warp * scratch_floats<CH, NV, WHOLE>());
  }
};

// The graphs of a window. Short: at most kShort rows, starts here (and may run on into
// the next window). Long: more rows; whole ones lie inside the window, split ones
// (at most two of them) do not.
struct Window {
  int shorts, longs, next;
  int item[kMaxWindow];  // short: first row from r0 << 8 | rows
  int64_t begin[kMaxLongs], end[kMaxLongs];
};

__device__ __forceinline__ bool is_split(const NormArgs& a, int64_t s, int64_t e) {
  return e - s > kShort && s / a.window != (e - 1) / a.window;
}

// Asks the L2 for rows [r0, r1), whatever graphs they belong to.
__device__ __forceinline__ void prefetch_rows(const NormArgs& a, int64_t r0, int64_t r1) {
  const uintptr_t first = (reinterpret_cast<uintptr_t>(a.x + r0 * a.c) + 15) & ~uintptr_t(15);
  const uintptr_t last = reinterpret_cast<uintptr_t>(a.x + r1 * a.c) & ~uintptr_t(15);
  // (a few huge graphs stream anyway: no look-up to hide behind)
  if (threadIdx.x == 0 && blockIdx.y == 0 && first < last && a.graphs * 8 >= a.windows) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(first), "r"(static_cast<uint32_t>(last - first))
                 : "memory");
  }
}

// Lists the graphs of rows [r0, r1) (in any order: no result depends on it); of the
// long ones only the split ones where `split_only`.
__device__ __forceinline__ void list_graphs(const NormArgs& a, int64_t r0, int64_t r1, bool split_only, Window& w) {
  if (threadIdx.x == 0) w.shorts = w.longs = w.next = 0;
  __syncthreads();
  const int64_t last = graph_of(a, r1 - 1);
  for (int64_t g = graph_of(a, r0) + threadIdx.x; g <= last && g < a.graphs; g += kThreads) {
    const int64_t s = ptr_at(a, g), e = ptr_at(a, g + 1);
    if (e - s > kShort && s < r1 && e > r0) {
      if (split_only && !is_split(a, s, e)) continue;
      const int i = atomicAdd(&w.longs, 1);
      if (i < kMaxLongs) {
        w.begin[i] = s;
        w.end[i] = e;
      }
    } else if (!split_only && e > s && e - s <= kShort && s >= r0 && s < r1) {
      const int i = atomicAdd(&w.shorts, 1);
      if (i < kMaxWindow) w.item[i] = static_cast<int>(s - r0) << 8 | static_cast<int>(e - s);
    }
  }
  __syncthreads();
}

template <int CH, int NV, bool WHOLE>
__global__ void __launch_bounds__(kThreads, min_blocks<CH, NV, WHOLE>()) norm_windows_kernel(NormArgs a) {
  constexpr int E = WHOLE ? 1 : CH;
  extern __shared__ float shared[];
  __shared__ Window list;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.window, r1 = min(r0 + a.window, a.n);
  prefetch_rows(a, r0, r1);
  list_graphs(a, r0, r1, false, list);
  Team<CH, NV, WHOLE> team;
  team.init(a, shared);
  const int me = team.warp;
  float w[NV][CH], b[NV][CH];
  load_affine(a, team.t, w, b);
  float mean[NV][E], m2[NV][E];
  // normalises `rows` rows from row s, whose statistics are (mean, m2)
  auto finish = [&](int64_t s, int rows) {
    const float inv = 1.0f / (static_cast<float>(rows) * static_cast<float>(a.cg));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < E; ++k) m2[j][k] = rsqrtf(fmaf(m2[j][k], inv, a.eps));
    }
    team.apply(a, s, rows, rows <= team.keep(), mean, m2, w, b);
  };
  // Several short graphs: each warp takes one after the other by itself. Few: all
  // warps work on each.
  const int shorts = min(list.shorts, kMaxWindow);
  const bool solo = shorts >= kWarps / 2;
  if (solo) {
    team.size = 1;
    team.warp = 0;
  }
  for (int i = 0;; ++i) {
    if (solo) {
      if (team.t.lane == 0) i = atomicAdd(&list.next, 1);
      i = __shfl_sync(kFull, i, 0);
    }
    if (i >= shorts) break;
    const int item = list.item[i];
    const int64_t s = r0 + (item >> 8);
    team.stats(a, s, item & 0xff, mean, m2);
    finish(s, item & 0xff);
  }
  team.size = kWarps;
  team.warp = me;
  const int longs = min(list.longs, kMaxLongs);
  for (int i = 0; i < longs; ++i) {
    const int64_t s = list.begin[i], e = list.end[i];
    const int64_t beg = max(s, r0);
    team.stats(a, beg, static_cast<int>(min(e, r1) - beg), mean, m2);
    if (!is_split(a, s, e)) {
      finish(s, static_cast<int>(e - s));
    } else if (me == 0) {
      float2* slot = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (s >= r0 ? 1 : 0)) * a.groups + team.t.g0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
          if (team.t.live(j) && team.t.leads(j, k)) slot[team.t.group(j, k)] = make_float2(mean[j][k], m2[j][k]);
        }
      }
    }
  }
}

// The pieces of a split graph, one per window.
struct Pieces {
  int64_t s, e, first, last;  // rows [s, e), windows first .. last
  double total;               // values per group
  __device__ __forceinline__ Pieces(const NormArgs& a, int64_t g)
      : s(ptr_at(a, g)), e(ptr_at(a, g + 1)), first(s / a.window), last((e - 1) / a.window),
        total(static_cast<double>(e - s) * a.cg) {}
  // values per group of piece k
  __device__ __forceinline__ double size(const NormArgs& a, int64_t k) const {
    return static_cast<double>(min(e, (k + 1) * a.window) - max(s, k * a.window)) * a.cg;
  }
  __device__ __forceinline__ float2 at(const NormArgs& a, int64_t k, int grp) const {
    return a.part[(k * 2 + (k == first ? 1 : 0)) * a.groups + grp];
  }
  __device__ __forceinline__ void put(const NormArgs& a, int grp, double mean, double m2) const {
    a.fin[first * a.groups + grp] =
        make_float2(static_cast<float>(mean), static_cast<float>(1.0 / sqrt(m2 / total + a.eps)));
  }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// Joins the pieces of split graphs in 64 bits, always in the same order. Blocks with
// blockIdx.y == 0 join graphs of few pieces, a warp each; the others take the graphs of
// many pieces, a block per group.
__global__ void __launch_bounds__(kThreads) norm_join_kernel(NormArgs a) {
  __shared__ double sh[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.y == 0) {
    // lane l of warp w looks at graph w + l * warps, so that neighbours go to different warps
    const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarps;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
    // the lanes are `parts` pieces times 32 / parts groups
    int parts = 32;
    while (parts > 1 && (32 / parts) < a.groups) parts /= 2;
    const int width = 32 / parts, part = lane / width, col = lane & (width - 1);
    for (int64_t base = 0; base < a.graphs; base += 32 * warps) {
      const int64_t mine = base + w + lane * warps;
      bool take = false;
      if (mine < a.graphs) {
        const int64_t s = ptr_at(a, mine), e = ptr_at(a, mine + 1);
        take = is_split(a, s, e) && e - s <= static_cast<int64_t>(kFewPieces - 2) * a.window;
      }
      for (unsigned todo = __ballot_sync(kFull, take); todo != 0; todo &= todo - 1) {
        const Pieces p(a, base + w + (__ffs(todo) - 1) * warps);
        for (int g0 = 0; g0 < a.groups; g0 += width) {
          const int grp = g0 + col;
          const bool live = grp < a.groups;
          double sum = 0.0, m2 = 0.0;
#pragma unroll 4
          for (int64_t k = p.first + part; k <= p.last; k += parts) {
            if (live) sum += p.size(a, k) * p.at(a, k, grp).x;
          }
          for (int o = width; o < 32; o <<= 1) sum += __shfl_xor_sync(kFull, sum, o);
          const double mean = sum / p.total;
#pragma unroll 4
          for (int64_t k = p.first + part; k <= p.last; k += parts) {
            if (live) {
              const float2 v = p.at(a, k, grp);
              m2 += v.y + p.size(a, k) * (v.x - mean) * (v.x - mean);
            }
          }
          for (int o = width; o < 32; o <<= 1) m2 += __shfl_xor_sync(kFull, m2, o);
          if (live && part == 0) p.put(a, grp, mean, m2);
        }
      }
    }
    return;
  }
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * 32; base < a.graphs;
       base += static_cast<int64_t>(gridDim.x) * 32) {
    bool take = false;
    if (base + lane < a.graphs) {
      const int64_t s = ptr_at(a, base + lane), e = ptr_at(a, base + lane + 1);
      take = e - s > static_cast<int64_t>(kFewPieces - 2) * a.window;
    }
    for (unsigned todo = __ballot_sync(kFull, take); todo != 0; todo &= todo - 1) {  // the same in every warp
      const Pieces p(a, base + __ffs(todo) - 1);
      auto block_sum = [&](double v) {
        v = warp_sum(v);
        if (lane == 0) sh[warp] = v;
        __syncthreads();
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) t += sh[i];
        __syncthreads();
        return t;
      };
      for (int grp = blockIdx.y - 1; grp < a.groups; grp += gridDim.y - 1) {
        double sum = 0.0, m2 = 0.0;
#pragma unroll 4
        for (int64_t k = p.first + threadIdx.x; k <= p.last; k += kThreads) sum += p.size(a, k) * p.at(a, k, grp).x;
        const double mean = block_sum(sum) / p.total;
#pragma unroll 4
        for (int64_t k = p.first + threadIdx.x; k <= p.last; k += kThreads) {
          const float2 v = p.at(a, k, grp);
          m2 += v.y + p.size(a, k) * (v.x - mean) * (v.x - mean);
        }
        m2 = block_sum(m2);
        if (threadIdx.x == 0) p.put(a, grp, mean, m2);
      }
    }
  }
}

// The rows of split graphs; the last windows first, whose rows the L2 may still hold.
template <int CH, int NV, bool WHOLE>
__global__ void __launch_bounds__(kThreads, min_blocks<CH, NV, WHOLE>()) norm_apply_kernel(NormArgs a) {
  constexpr int E = WHOLE ? 1 : CH;
  extern __shared__ float shared[];
  __shared__ Window list;
  const int64_t r0 = (a.windows - 1 - blockIdx.x) * a.window, r1 = min(r0 + a.window, a.n);
  list_graphs(a, r0, r1, true, list);
  if (list.longs == 0) return;
  Team<CH, NV, WHOLE> team;
  team.init(a, shared);
  float w[NV][CH], b[NV][CH];
  load_affine(a, team.t, w, b);
  for (int i = 0; i < min(list.longs, kMaxLongs); ++i) {
    const int64_t s = list.begin[i];
    const float2* fin = a.fin + (s / a.window) * a.groups + team.t.g0;
    float mean[NV][E], rstd[NV][E];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float2 f = team.t.live(j) ? fin[team.t.group(j, k)] : make_float2(0.0f, 0.0f);
        mean[j][k] = f.x;
        rstd[j][k] = f.y;
      }
    }
    const int64_t beg = max(s, r0);
    team.apply(a, beg, static_cast<int>(min(list.end[i], r1) - beg), false, mean, rstd, w, b);
  }
}

// Opts a kernel in to more than 48 KB of dynamic shared memory where a call needs it: once
// per device, to the most that any call can need, so that no thread takes away what
// another is about to launch with.
template <auto Kernel>
int allow_shared(size_t bytes, size_t most) {
  if (bytes <= 48 * 1024) return GNN_OK;
  static bool configured[64] = {};
  static std::mutex mu;
  int dev = 0;
  GNN_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    GNN_CUDA_TRY(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)),
                 "group norm: shared memory opt-in");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return GNN_OK;
}

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Rows per block: about eight graphs of average length, so that each warp has one to
// itself (or, of long graphs, few pieces to join), as long as the SMs get a few blocks each.
int window_for(int64_t n, int64_t graphs) {
  int window = kShort;
  while (window < kMaxWindow && window < 8 * (n / graphs) && n / (2 * window) >= 2 * sm_count()) window *= 2;
  return window;
}

size_t workspace_for(int64_t n, int64_t graphs, int64_t groups) {
  if (n <= kShort) return 0;  // every graph is finished by one block
  const int64_t window = window_for(n, graphs);
  return static_cast<size_t>(round_up((n + window - 1) / window * 3 * groups * 8, 256));
}

template <int CH, int NV, bool WHOLE>
int run(const NormArgs& a, bool rows, unsigned tiles, cudaStream_t s) {
  const size_t warps = sizeof(float) * kWarps * scratch_floats<CH, NV, WHOLE>();
  if (rows) {
    constexpr int R = NV * CH <= 4 ? 4 : (NV * CH <= 8 ? 2 : 1);
    const int64_t want = (a.n + kWarps * R - 1) / (kWarps * R);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(want, 16LL * sm_count())), tiles);
    if (a.cg > 1 && a.cg <= kSmallGroup) {
      if (int rc = allow_shared<norm_rows_kernel<CH, NV, WHOLE, true>>(warps, warps)) return rc;
      norm_rows_kernel<CH, NV, WHOLE, true><<<grid, kThreads, warps, s>>>(a);
    } else {
      if (int rc = allow_shared<norm_rows_kernel<CH, NV, WHOLE, false>>(warps, warps)) return rc;
      norm_rows_kernel<CH, NV, WHOLE, false><<<grid, kThreads, warps, s>>>(a);
    }
    GNN_LAUNCH_CHECK("norm_rows_kernel launch");
    return GNN_OK;
  }
  const size_t smem = warps + sizeof(float2) * 2 * kWarps * a.tile_groups;
  constexpr size_t most =
      sizeof(float) * kWarps * scratch_floats<CH, NV, WHOLE>() + sizeof(float2) * 2 * kWarps * kTile;
  static_assert(most + sizeof(Window) + 1024 <= 227 * 1024, "the largest call has to fit");
  const dim3 grid(static_cast<unsigned>(a.windows), tiles);
  if (int rc = allow_shared<norm_windows_kernel<CH, NV, WHOLE>>(smem, most)) return rc;
  norm_windows_kernel<CH, NV, WHOLE><<<grid, kThreads, smem, s>>>(a);
  GNN_LAUNCH_CHECK("norm_windows_kernel launch");
  if (a.n <= kShort) return GNN_OK;
  const int64_t batches = (a.graphs + kWarps - 1) / kWarps;  // a warp per graph
  const bool many = a.n > static_cast<int64_t>(kFewPieces - 2) * a.window;  // some graph may have many pieces
  const dim3 jgrid(static_cast<unsigned>(std::min<int64_t>(batches, 4LL * sm_count())),
                   many ? 1u + static_cast<unsigned>(std::min(a.groups, 64)) : 1u);
  norm_join_kernel<<<jgrid, kThreads, 0, s>>>(a);
  GNN_LAUNCH_CHECK("norm_join_kernel launch");
  if (int rc = allow_shared<norm_apply_kernel<CH, NV, WHOLE>>(smem, most)) return rc;
  norm_apply_kernel<CH, NV, WHOLE><<<grid, kThreads, smem, s>>>(a);
  GNN_LAUNCH_CHECK("norm_apply_kernel launch");
  return GNN_OK;
}

int run_narrow(const NormArgs& a, cudaStream_t s) {
  const int tile_rows = std::max(4, kNarrowFloats / a.c / 4 * 4);  // a multiple of 4: tiles start on 16 bytes
  const int64_t want = (a.n + tile_rows - 1) / tile_rows;
  const int vec = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0;
  const size_t smem = static_cast<size_t>(std::min<int64_t>(tile_rows, a.n)) * a.c * 4;
  norm_narrow_kernel<<<static_cast<unsigned>(std::min<int64_t>(want, 28LL * sm_count())), kThreads, smem, s>>>(
      a, tile_rows, vec);
  GNN_LAUNCH_CHECK("norm_narrow_kernel launch");
  return GNN_OK;
}

template <int CH, bool WHOLE>
int run_width(const NormArgs& a, bool rows, int64_t cols, unsigned tiles, cudaStream_t s) {
  if (cols <= 32 * CH) return run<CH, 1, WHOLE>(a, rows, tiles, s);
  if (cols <= 64 * CH) return run<CH, 2, WHOLE>(a, rows, tiles, s);
  if (cols <= 128 * CH) return run<CH, 4, WHOLE>(a, rows, tiles, s);
  if (cols <= 256 * CH) return run<CH, 8, WHOLE>(a, rows, tiles, s);
  if constexpr (CH <= 2) {
    if (cols <= 512 * CH) return run<CH, 16, WHOLE>(a, rows, tiles, s);
  }
  if constexpr (CH == 1) return run<CH, 32, WHOLE>(a, rows, tiles, s);
  return fail(GNN_ERR_UNSUPPORTED, "group norm: column tile too wide");
}

}  // namespace
}  // namespace gnnb200

using namespace gnnb200;

extern "C" size_t gnn_group_norm_workspace_bytes(int64_t num_nodes, int64_t num_graphs, int64_t groups) {
  if (num_nodes <= 0 || num_graphs <= 0 || groups <= 0) return 0;
  return workspace_for(num_nodes, num_graphs, groups);
}

extern "C" int gnn_group_norm_forward(const float* x, const void* graph_ptr, int graph_ptr_type, int64_t num_graphs,
                                      const float* weight, const float* bias, float* out, int64_t num_nodes,
                                      int64_t channels, int64_t groups, float eps, int activation, void* workspace,
                                      size_t workspace_bytes, gnn_stream_t stream) {
  GNN_REQUIRE(num_nodes >= 0 && channels >= 0 && num_graphs >= 0, GNN_ERR_INVALID_ARGUMENT,
              "num_nodes, channels and num_graphs must be >= 0");
  GNN_REQUIRE(groups >= 1 && channels % groups == 0, GNN_ERR_INVALID_ARGUMENT,
              "groups must be >= 1 and divide the number of channels");
  GNN_REQUIRE(activation >= GNN_ACT_NONE && activation <= GNN_ACT_GELU, GNN_ERR_INVALID_ARGUMENT,
              "activation must be one of gnn_activation");
  GNN_REQUIRE(eps >= 0.0f, GNN_ERR_INVALID_ARGUMENT, "eps must be >= 0");
  GNN_REQUIRE(graph_ptr == nullptr || graph_ptr_type == GNN_INDEX_INT32 || graph_ptr_type == GNN_INDEX_INT64,
              GNN_ERR_INVALID_ARGUMENT, "graph_ptr must be int32 or int64");
  if (num_nodes == 0 || channels == 0 || (graph_ptr != nullptr && num_graphs == 0)) {
    clear_error();
    return GNN_OK;
  }
  const int64_t cg = channels / groups;
  GNN_REQUIRE(cg <= kTile, GNN_ERR_UNSUPPORTED, "at most 1024 channels per group");
  const int64_t tile_groups = std::min(groups, kTile / cg);
  const int64_t tiles = (groups + tile_groups - 1) / tile_groups;
  GNN_REQUIRE(channels <= 0x7fffffffLL && tiles <= 65535, GNN_ERR_UNSUPPORTED, "too many channels");
  GNN_REQUIRE(num_nodes <= (int64_t(1) << 36), GNN_ERR_UNSUPPORTED, "too many nodes");
  GNN_REQUIRE(x != nullptr && out != nullptr, GNN_ERR_NULL_POINTER, "x and out must not be NULL");
  const size_t need = graph_ptr != nullptr ? workspace_for(num_nodes, num_graphs, groups) : 0;
  GNN_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), GNN_ERR_WORKSPACE,
              "workspace missing or too small (gnn_group_norm_workspace_bytes)");
  GNN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, GNN_ERR_WORKSPACE,
              "workspace must be 16-byte aligned");
  NormArgs a{};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.out = out;
  a.ptr = graph_ptr;
  a.graphs = num_graphs;
  a.n = num_nodes;
  a.c = static_cast<int>(channels);
  a.groups = static_cast<int>(groups);
  a.cg = static_cast<int>(cg);
  a.tile_groups = static_cast<int>(tile_groups);
  a.eps = eps;
  a.act = activation;
  a.wide_ptr = graph_ptr_type == GNN_INDEX_INT64 ? 1 : 0;
  const bool rows = graph_ptr == nullptr;
  if (!rows) {
    a.window = window_for(num_nodes, num_graphs);
    a.windows = (num_nodes + a.window - 1) / a.window;
    a.part = static_cast<float2*>(workspace);
    a.fin = a.part + a.windows * 2 * groups;
  }
  // 16- or 8-byte pieces of rows: in several column tiles only where each starts on one
  const uintptr_t base = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out);
  const bool vec4 = channels % 4 == 0 && (tiles == 1 || cg % 4 == 0) && base % 16 == 0;
  const bool vec2 = channels % 2 == 0 && (tiles == 1 || cg % 2 == 0) && base % 8 == 0;
  const int64_t cols = tile_groups * cg;
  const unsigned ty = static_cast<unsigned>(tiles);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int rc;
  // where a row is short or its groups are no aligned powers of two of a warp's lanes
  const bool lanes = vec4 && cg % 4 == 0 && (cg / 4 & (cg / 4 - 1)) == 0 && channels >= 64;
  if (rows && channels <= kNarrowChannels && cg <= kNarrowGroup && !lanes) {
    rc = run_narrow(a, s);
  } else if (vec4) {
    rc = cg % 4 == 0 ? run_width<4, true>(a, rows, cols, ty, s) : run_width<4, false>(a, rows, cols, ty, s);
  } else if (vec2) {
    rc = cg % 2 == 0 ? run_width<2, true>(a, rows, cols, ty, s) : run_width<2, false>(a, rows, cols, ty, s);
  } else {
    rc = run_width<1, true>(a, rows, cols, ty, s);
  }
  if (rc == GNN_OK) clear_error();
  return rc;
}
