// Group normalisation with an activation over node features [N, C], channels last:
//   y = act((x - mean) / sqrt(var + eps) * weight[c] + bias[c])
// with mean and (biased) variance over the C / groups channels of a group, either
// of each node on its own, or of all nodes of a graph of a batch (graph_ptr, ragged).
//
// Statistics: a warp reads rows in batches of U; each lane folds a batch's mean and
// squared deviations about it into its running ones (the pairwise update of mean and
// M2), so nothing is subtracted from a large sum; lanes, then pieces, are joined the
// same way. The result is the same every time: no atomics.
//
// Batch mode: rows are cut into chunks of kChunk, one warp each. A graph of at most
// kChunk nodes belongs to the warp in whose chunk it starts and is finished there
// (its second read comes from L1 / L2). A longer graph leaves a piece per chunk in
// the workspace; a second kernel joins the pieces, a third reads x again and writes.
// So a long graph costs three passes over its rows where x exceeds the L2.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"

namespace gnnb200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kChunk = 64;        // rows per warp; the longest graph that one warp finishes
constexpr int kTile = 1024;       // channels per column tile at most (whole groups)
constexpr int kJoinThreads = 512;

struct NormArgs {
  const float* x;
  const float* weight;
  const float* bias;
  float* out;
  const void* ptr;    // graph offsets, batch mode
  int64_t graphs;
  int64_t n;
  int c, groups, cg;  // channels, groups, channels per group
  int tile_groups;    // groups per column tile
  float eps;
  int act;
  float2* part;       // [chunks, 2, groups]: (mean, M2) of a long graph's piece: it began earlier / it begins here
  float2* fin;        // [chunks, groups]: (mean, 1 / sqrt(var + eps)) of the long graph that begins in the chunk
  int64_t chunks;
};

__device__ __forceinline__ float activate(float y, int act) {
  switch (act) {
    case GNN_ACT_RELU: return y < 0.0f ? 0.0f : y;
    case GNN_ACT_SILU: return __fdividef(y, 1.0f + __expf(-y));
    case GNN_ACT_GELU: return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    default: return y;
  }
}

template <class IdxT>
__device__ __forceinline__ int64_t ptr_at(const NormArgs& a, int64_t g) {
  const int64_t v = static_cast<int64_t>(__ldg(static_cast<const IdxT*>(a.ptr) + g));
  return v < 0 ? 0 : (v > a.n ? a.n : v);
}

// The first graph whose end lies past `row` (graphs where there is none).
template <class IdxT>
__device__ __forceinline__ int64_t graph_of(const NormArgs& a, int64_t row) {
  int64_t lo = 0, hi = a.graphs;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (ptr_at<IdxT>(a, mid + 1) > row) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo;
}

// A warp's view of one column tile: lane l holds the channels
// c0 + CH * (l + 32 j) .. + CH, j < NV.
template <int CH, int NV>
struct Tile {
  int c0, cols;     // first channel, channels
  int g0, groups;   // first group, groups
  int cg;           // channels per group
  int gsize;        // chunks of CH channels per group
  int lane;
  bool pow2;        // a group is an aligned power of two of at most 32 lanes
  int grp[NV];      // group (in the tile) of chunk lane + 32 j
  float* sh;        // this warp's scratch: 32 NV partials and up to kTile totals

  __device__ __forceinline__ bool live(int j) const { return (lane + 32 * j) * CH < cols; }
  __device__ __forceinline__ int channel(int j) const { return c0 + CH * (lane + 32 * j); }

  __device__ __forceinline__ void init(const NormArgs& a, float* scratch) {
    lane = threadIdx.x & 31;
    g0 = static_cast<int>(blockIdx.y) * a.tile_groups;
    groups = min(a.tile_groups, a.groups - g0);
    cg = a.cg;
    c0 = g0 * cg;
    cols = groups * cg;
    gsize = cg / CH;
    pow2 = gsize <= 32 && (gsize & (gsize - 1)) == 0;
    sh = scratch;
#pragma unroll
    for (int j = 0; j < NV; ++j) grp[j] = (lane + 32 * j) / gsize;
  }

  // p[j]: this lane's partial of chunk j -> the total of the chunk's group
  __device__ __forceinline__ void group_sum(float (&p)[NV]) const {
    if (pow2) {
      for (int o = 1; o < gsize; o <<= 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) p[j] += __shfl_xor_sync(kFull, p[j], o);
      }
      return;
    }
    if (groups == 1) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j) s += live(j) ? p[j] : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
#pragma unroll
      for (int j = 0; j < NV; ++j) p[j] = s;
      return;
    }
    float* tot = sh + 32 * NV;
#pragma unroll
    for (int j = 0; j < NV; ++j) sh[lane + 32 * j] = p[j];
    __syncwarp();
    int per = 1;  // lanes per group
    while (per * 2 * min(groups, 32) <= 32) per *= 2;
    const int at = lane / per, t = lane & (per - 1);
    for (int base = 0; base < groups; base += 32 / per) {
      const int g = base + at;
      float s = 0.0f;
      if (g < groups) {
        for (int i = t; i < gsize; i += per) s += sh[g * gsize + i];
      }
      for (int o = 1; o < per; o <<= 1) s += __shfl_xor_sync(kFull, s, o);
      if (t == 0 && g < groups) tot[g] = s;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NV; ++j) p[j] = live(j) ? tot[grp[j]] : 0.0f;
    __syncwarp();
  }
};

template <int CH>
__device__ __forceinline__ void load_chunk(const float* p, float (&v)[CH]) {
  if constexpr (CH == 4) {
    const float4 t = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = t.x;
    v[1] = t.y;
    v[2] = t.z;
    v[3] = t.w;
  } else {
    v[0] = __ldg(p);
  }
}

template <int CH>
__device__ __forceinline__ void store_chunk(float* p, const float (&v)[CH]) {
  if constexpr (CH == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *p = v[0];
  }
}

template <int CH, int NV>
__device__ __forceinline__ void load_affine(const NormArgs& a, const Tile<CH, NV>& t, float (&w)[NV][CH],
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

// 8 warps a block; 4 where their scratch would not fit the static 48 KB
template <int NV>
constexpr int block_warps() {
  return NV >= 32 ? 4 : 8;
}

template <int CH, int NV>
constexpr int scratch_floats() {
  return 32 * NV + 32 * NV;  // partials, totals (at most one group per chunk)
}

// ---- each node on its own: one warp per row --------------------------------
template <int CH, int NV>
__global__ void __launch_bounds__(32 * block_warps<NV>()) norm_rows_kernel(NormArgs a) {
  constexpr int kWarps = block_warps<NV>();
  __shared__ float scratch[kWarps][scratch_floats<CH, NV>()];
  Tile<CH, NV> t;
  t.init(a, scratch[threadIdx.x >> 5]);
  float w[NV][CH], b[NV][CH];
  load_affine(a, t, w, b);
  const float inv = 1.0f / static_cast<float>(a.cg);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); r < a.n; r += step) {
    const float* src = a.x + r * a.c;
    float v[NV][CH], p[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      p[j] = 0.0f;
      if (t.live(j)) {
        load_chunk<CH>(src + t.channel(j), v[j]);
#pragma unroll
        for (int e = 0; e < CH; ++e) p[j] += v[j][e];
      }
    }
    t.group_sum(p);
    float q[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q[j] = 0.0f;
      if (t.live(j)) {
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          v[j][e] -= p[j] * inv;
          q[j] = fmaf(v[j][e], v[j][e], q[j]);
        }
      }
    }
    t.group_sum(q);
    float* dst = a.out + r * a.c;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (t.live(j)) {
        const float rstd = __frcp_rn(__fsqrt_rn(fmaf(q[j], inv, a.eps)));
#pragma unroll
        for (int e = 0; e < CH; ++e) v[j][e] = activate(fmaf(v[j][e] * rstd, w[j][e], b[j][e]), a.act);
        store_chunk<CH>(dst + t.channel(j), v[j]);
      }
    }
  }
}

// ---- graphs of a batch ------------------------------------------------------

template <int NV>
constexpr int batch_rows() {
  return NV == 1 ? 8 : (NV == 2 ? 4 : (NV <= 8 ? 2 : 1));
}

// (mean, M2) per group of rows [beg, end), in the lanes of the group's chunks.
template <int CH, int NV>
__device__ __forceinline__ void piece_stats(const NormArgs& a, const Tile<CH, NV>& t, int64_t beg, int64_t end,
                                            float (&mean)[NV], float (&m2)[NV]) {
  constexpr int U = batch_rows<NV>();
  float m[NV][CH], s[NV][CH];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int e = 0; e < CH; ++e) m[j][e] = s[j][e] = 0.0f;
  }
  float n = 0.0f;
  for (int64_t r = beg; r < end; r += U) {
    float v[U][NV][CH];
    const int cnt = static_cast<int>(min(static_cast<int64_t>(U), end - r));
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (u < cnt && t.live(j)) {
          load_chunk<CH>(a.x + (r + u) * a.c + t.channel(j), v[u][j]);
        } else {
#pragma unroll
          for (int e = 0; e < CH; ++e) v[u][j][e] = 0.0f;
        }
      }
    }
    const float cf = static_cast<float>(cnt);
    const float icf = __frcp_rn(cf);
    const float nn = n + cf;
    const float share = __fdividef(cf, nn);
    const float both = n * share;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) sum += v[u][j][e];
        const float mb = sum * icf;
        float dev = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float d = v[u][j][e] - mb;
          if (u < cnt) dev = fmaf(d, d, dev);
        }
        const float delta = mb - m[j][e];
        m[j][e] = fmaf(delta, share, m[j][e]);
        s[j][e] += fmaf(delta * delta, both, dev);
      }
    }
    n = nn;
  }
  // channels of a group: n values each
  const float icg = 1.0f / static_cast<float>(a.cg);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    mean[j] = 0.0f;
    if (t.live(j)) {
#pragma unroll
      for (int e = 0; e < CH; ++e) mean[j] += m[j][e];
    }
  }
  t.group_sum(mean);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    mean[j] *= icg;
    m2[j] = 0.0f;
    if (t.live(j)) {
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float d = m[j][e] - mean[j];
        m2[j] += fmaf(d * d, n, s[j][e]);
      }
    }
  }
  t.group_sum(m2);
}

// Rows [beg, end) with the statistics of their groups.
template <int CH, int NV>
__device__ __forceinline__ void apply_rows(const NormArgs& a, const Tile<CH, NV>& t, int64_t beg, int64_t end,
                                           const float (&mean)[NV], const float (&rstd)[NV]) {
  constexpr int U = batch_rows<NV>() >= 4 ? 4 : batch_rows<NV>();
  float w[NV][CH], b[NV][CH];
  load_affine(a, t, w, b);
  for (int64_t r = beg; r < end; r += U) {
    float v[U][NV][CH];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (r + u < end && t.live(j)) load_chunk<CH>(a.x + (r + u) * a.c + t.channel(j), v[u][j]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (r + u < end && t.live(j)) {
#pragma unroll
          for (int e = 0; e < CH; ++e) {
            v[u][j][e] = activate(fmaf((v[u][j][e] - mean[j]) * rstd[j], w[j][e], b[j][e]), a.act);
          }
          store_chunk<CH>(a.out + (r + u) * a.c + t.channel(j), v[u][j]);
        }
      }
    }
  }
}

template <int CH, int NV, class IdxT>
__global__ void __launch_bounds__(32 * block_warps<NV>()) norm_pieces_kernel(NormArgs a) {
  constexpr int kWarps = block_warps<NV>();
  __shared__ float scratch[kWarps][scratch_floats<CH, NV>()];
  Tile<CH, NV> t;
  t.init(a, scratch[threadIdx.x >> 5]);
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (chunk >= a.chunks) return;
  const int64_t r0 = chunk * kChunk, r1 = min(r0 + kChunk, a.n);
  for (int64_t g = graph_of<IdxT>(a, r0); g < a.graphs;) {
    const int64_t s = ptr_at<IdxT>(a, g), e = ptr_at<IdxT>(a, g + 1);
    if (s >= r1) break;
    float mean[NV], m2[NV];
    if (e - s <= kChunk) {
      if (s >= r0 && e > s) {
        piece_stats<CH, NV>(a, t, s, e, mean, m2);
        const float inv = 1.0f / (static_cast<float>(e - s) * static_cast<float>(a.cg));
#pragma unroll
        for (int j = 0; j < NV; ++j) m2[j] = __frcp_rn(__fsqrt_rn(fmaf(m2[j], inv, a.eps)));
        apply_rows<CH, NV>(a, t, s, e, mean, m2);
      }
    } else {
      piece_stats<CH, NV>(a, t, max(s, r0), min(e, r1), mean, m2);
      float2* slot = a.part + (chunk * 2 + (s >= r0 ? 1 : 0)) * a.groups + t.g0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        // the first chunk of a group writes for all of it
        if (t.live(j) && (t.lane + 32 * j) % t.gsize == 0) slot[t.grp[j]] = make_float2(mean[j], m2[j]);
      }
    }
    ++g;
    // a run of empty graphs is passed in one search
    if (g < a.graphs && ptr_at<IdxT>(a, g + 1) <= e) g = max(g, graph_of<IdxT>(a, max(e, r0)));
  }
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) s += sh[i];
  __syncthreads();
  return s;
}

// Joins the pieces of long graphs, in 64 bits and in piece order per thread:
// blocks take graphs in batches of kJoinThreads, group by group (blockIdx.y, striding).
template <class IdxT>
__global__ void __launch_bounds__(kJoinThreads) norm_join_kernel(NormArgs a) {
  __shared__ double sh[kJoinThreads / 32];
  __shared__ int todo[kJoinThreads];
  __shared__ int count;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kJoinThreads; base < a.graphs;
       base += static_cast<int64_t>(gridDim.x) * kJoinThreads) {
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const int64_t mine = base + threadIdx.x;
    if (mine < a.graphs && ptr_at<IdxT>(a, mine + 1) - ptr_at<IdxT>(a, mine) > kChunk) {
      todo[atomicAdd(&count, 1)] = threadIdx.x;  // the order of graphs does not touch their results
    }
    __syncthreads();
    for (int i = 0; i < count; ++i) {
      const int64_t g = base + todo[i];
      const int64_t s = ptr_at<IdxT>(a, g), e = ptr_at<IdxT>(a, g + 1);
      const int64_t first = s / kChunk, last = (e - 1) / kChunk;
      const double total = static_cast<double>(e - s) * a.cg;
      for (int grp = blockIdx.y; grp < a.groups; grp += gridDim.y) {
        double sum = 0.0;
        for (int64_t k = first + threadIdx.x; k <= last; k += kJoinThreads) {
          const int64_t rows = min(e, (k + 1) * kChunk) - max(s, k * kChunk);
          const float2 p = a.part[(k * 2 + (k == first ? 1 : 0)) * a.groups + grp];
          sum += static_cast<double>(rows) * a.cg * p.x;
        }
        const double mean = block_sum(sum, sh) / total;
        double m2 = 0.0;
        for (int64_t k = first + threadIdx.x; k <= last; k += kJoinThreads) {
          const int64_t rows = min(e, (k + 1) * kChunk) - max(s, k * kChunk);
          const float2 p = a.part[(k * 2 + (k == first ? 1 : 0)) * a.groups + grp];
          const double d = p.x - mean;
          m2 += p.y + static_cast<double>(rows) * a.cg * d * d;
        }
        m2 = block_sum(m2, sh);
        if (threadIdx.x == 0) {
          a.fin[first * a.groups + grp] =
              make_float2(static_cast<float>(mean), static_cast<float>(1.0 / sqrt(m2 / total + a.eps)));
        }
      }
    }
    __syncthreads();
  }
}

// The rows of long graphs. A chunk holds at most two of them: the graph of its first
// row and that of its last.
template <int CH, int NV, class IdxT>
__global__ void __launch_bounds__(32 * block_warps<NV>()) norm_apply_kernel(NormArgs a) {
  constexpr int kWarps = block_warps<NV>();
  __shared__ float scratch[kWarps][scratch_floats<CH, NV>()];
  Tile<CH, NV> t;
  t.init(a, scratch[threadIdx.x >> 5]);
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (chunk >= a.chunks) return;
  const int64_t r0 = chunk * kChunk, r1 = min(r0 + kChunk, a.n);
  int64_t before = -1;
  for (int i = 0; i < 2; ++i) {
    const int64_t g = graph_of<IdxT>(a, i == 0 ? r0 : r1 - 1);
    if (g >= a.graphs || g == before) continue;
    before = g;
    const int64_t s = ptr_at<IdxT>(a, g), e = ptr_at<IdxT>(a, g + 1);
    if (e - s <= kChunk || s >= r1 || e <= r0) continue;
    const float2* fin = a.fin + (s / kChunk) * a.groups + t.g0;
    float mean[NV], rstd[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float2 f = t.live(j) ? fin[t.grp[j]] : make_float2(0.0f, 0.0f);
      mean[j] = f.x;
      rstd[j] = f.y;
    }
    apply_rows<CH, NV>(a, t, max(s, r0), min(e, r1), mean, rstd);
  }
}

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t chunks_for(int64_t n) { return (n + kChunk - 1) / kChunk; }

size_t workspace_for(int64_t n, int64_t groups) {
  if (n <= kChunk) return 0;  // every graph is finished by one warp
  return static_cast<size_t>(round_up(chunks_for(n) * 3 * groups * 8, 256));
}

template <int CH, int NV, class IdxT>
int run_batch(const NormArgs& a, unsigned tiles, cudaStream_t s) {
  constexpr int kWarps = block_warps<NV>();
  const dim3 grid(static_cast<unsigned>((a.chunks + kWarps - 1) / kWarps), tiles);
  norm_pieces_kernel<CH, NV, IdxT><<<grid, 32 * kWarps, 0, s>>>(a);
  GNN_LAUNCH_CHECK("norm_pieces_kernel launch");
  if (a.n <= kChunk) return GNN_OK;
  const int64_t batches = (a.graphs + kJoinThreads - 1) / kJoinThreads;
  const dim3 jgrid(static_cast<unsigned>(std::min<int64_t>(batches, 4LL * sm_count())),
                   static_cast<unsigned>(std::min(a.groups, 32)));
  norm_join_kernel<IdxT><<<jgrid, kJoinThreads, 0, s>>>(a);
  GNN_LAUNCH_CHECK("norm_join_kernel launch");
  norm_apply_kernel<CH, NV, IdxT><<<grid, 32 * kWarps, 0, s>>>(a);
  GNN_LAUNCH_CHECK("norm_apply_kernel launch");
  return GNN_OK;
}

template <int CH, int NV>
int run(const NormArgs& a, bool rows, bool wide_index, unsigned tiles, cudaStream_t s) {
  if (rows) {
    constexpr int kWarps = block_warps<NV>();
    const int64_t want = (a.n + kWarps - 1) / kWarps;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(want, 16LL * sm_count())), tiles);
    norm_rows_kernel<CH, NV><<<grid, 32 * kWarps, 0, s>>>(a);
    GNN_LAUNCH_CHECK("norm_rows_kernel launch");
    return GNN_OK;
  }
  return wide_index ? run_batch<CH, NV, int64_t>(a, tiles, s) : run_batch<CH, NV, int32_t>(a, tiles, s);
}

}  // namespace
}  // namespace gnnb200

using namespace gnnb200;

extern "C" size_t gnn_group_norm_workspace_bytes(int64_t num_nodes, int64_t num_graphs, int64_t groups) {
  if (num_nodes <= 0 || num_graphs <= 0 || groups <= 0) return 0;
  return workspace_for(num_nodes, groups);
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
  const size_t need = graph_ptr != nullptr ? workspace_for(num_nodes, groups) : 0;
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
  a.chunks = chunks_for(num_nodes);
  a.part = static_cast<float2*>(workspace);
  a.fin = a.part + a.chunks * 2 * groups;
  const bool vec = cg % 4 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int64_t cols = tile_groups * cg;
  const bool rows = graph_ptr == nullptr;
  const bool wide = graph_ptr_type == GNN_INDEX_INT64;
  const unsigned ty = static_cast<unsigned>(tiles);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int rc;
  if (vec) {
    if (cols <= 128) {
      rc = run<4, 1>(a, rows, wide, ty, s);
    } else if (cols <= 256) {
      rc = run<4, 2>(a, rows, wide, ty, s);
    } else if (cols <= 512) {
      rc = run<4, 4>(a, rows, wide, ty, s);
    } else {
      rc = run<4, 8>(a, rows, wide, ty, s);
    }
  } else {
    if (cols <= 128) {
      rc = run<1, 4>(a, rows, wide, ty, s);
    } else if (cols <= 512) {
      rc = run<1, 16>(a, rows, wide, ty, s);
    } else {
      rc = run<1, 32>(a, rows, wide, ty, s);
    }
  }
  if (rc == GNN_OK) clear_error();
  return rc;
}
