// CSR aggregation over 8-bit feature rows with one fp32 scale each:
//   out[r, :] = f_r * sum_e w_e * scale[c_e] * q[c_e, :]
// with (f_r, w_e) = (dis[r], dis[c_e]) for GCN, (1, edge_weight[e]) weighted,
// (1, 1) sum and (1 / deg r, 1) mean; sums in fp32.
//
// Split: the merged sequence of row ends and entries is cut into equal shares, one
// per warp (the cut points are found by a binary search on row_ptr), so hubs, short
// and empty rows all balance. A warp stores the rows that lie wholly in its share;
// what it holds of a row that began earlier, or ends later, goes to a workspace
// slot, and a second small kernel adds those pieces in share order: no float
// atomics, the same bits every time.
//
// Inside a warp a row takes L lanes of 16 columns each (one 128-bit load a lane), so
// 32 / L entries are in flight per load; their sums are joined by a
// reduce-scatter over the lane groups when the row ends.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"

namespace gnnb200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTileCols = 512;  // columns of one pass (32 lanes x 16)

enum Mode : int { kSum = GNN_WEIGHT_SUM, kMean = GNN_WEIGHT_MEAN, kGcn = GNN_WEIGHT_GCN, kWeighted = GNN_WEIGHT_EDGE };

struct I8SpmmArgs {
  const void* row_ptr;
  const int32_t* col;
  const float* dis;
  const float* ew;
  const int8_t* x;
  int64_t ldx;
  const float* scale;
  float* out;
  int64_t n, nnz;
  int f;
  int64_t share;    // row ends + entries per warp
  int64_t shares;   // number of shares
  float* part;      // [2 * shares, f]: head (row began earlier), tail (row ends later)
  int64_t* part_row;  // [shares] row of the tail piece, -1 none
};

// Four packed signed bytes as floats: each byte becomes the low mantissa bits of
// 2^23 + 128 + q, from which 2^23 + 128 is taken off again (exact, no conversion unit).
__device__ __forceinline__ void bytes_to_float(uint32_t v, float (&f)[4]) {
  v ^= 0x80808080u;
  constexpr float kBase = 8388736.0f;  // 2^23 + 128
  f[0] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7540)) - kBase;
  f[1] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7541)) - kBase;
  f[2] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7542)) - kBase;
  f[3] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7543)) - kBase;
}

// 16 bytes of row data starting at column c of a row of `f` columns.
// VEC: rows start on 16-byte boundaries and the load may run past f within the
// row's stride; `edge` marks the matrix's last row, whose stride may not be there.
template <bool VEC>
__device__ __forceinline__ uint4 load16(const int8_t* row, int c, int f, bool edge) {
  if (VEC && (!edge || c + 16 <= f)) return __ldg(reinterpret_cast<const uint4*>(row + c));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (c + i < f) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(row + c + i))) << (8 * (i & 3));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <class IdxT>
__device__ __forceinline__ int64_t rp(const I8SpmmArgs& a, int64_t r) {
  return static_cast<int64_t>(__ldg(static_cast<const IdxT*>(a.row_ptr) + r));
}

// Number of row ends among the first `d` items of the merged sequence (row r's end
// comes after its entries): the smallest r with row_ptr[r + 1] + r + 1 > d.
template <class IdxT>
__device__ __forceinline__ int64_t row_at(const I8SpmmArgs& a, int64_t d) {
  int64_t lo = 0, hi = a.n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (rp<IdxT>(a, mid + 1) + mid + 1 > d) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo;
}

template <int MODE, class IdxT>
__device__ __forceinline__ float row_factor(const I8SpmmArgs& a, int64_t r) {
  if constexpr (MODE == kGcn) {
    return __ldg(a.dis + r);
  } else if constexpr (MODE == kMean) {
    const int64_t deg = rp<IdxT>(a, r + 1) - rp<IdxT>(a, r);
    return deg > 0 ? __fdiv_rn(1.0f, static_cast<float>(deg)) : 0.0f;
  } else {
    return 1.0f;
  }
}

// L lanes per row (a power of two), 32 / L entries at a time.
template <int MODE, int L, bool VEC, class IdxT>
__global__ void __launch_bounds__(kThreads) spmm_i8_kernel(I8SpmmArgs a) {
  constexpr int G = 32 / L;                    // lane groups
  constexpr int KEEP = G >= 16 ? 1 : 16 / G;   // columns a lane holds after the reduce-scatter
  const int lane = threadIdx.x & 31;
  const int grp = lane / L;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (w >= a.shares) return;
  const int cbase = blockIdx.y * kTileCols;    // L == 32 where f > 512, else 0
  const int c0 = cbase + (lane % L) * 16;      // this lane's 16 columns
  const bool have = c0 < a.f;
  const int64_t total = a.n + a.nnz;
  const int64_t d0 = w * a.share, d1 = min(d0 + a.share, total);
  int64_t row = row_at<IdxT>(a, d0);
  const int64_t row_end = row_at<IdxT>(a, d1);  // rows [row, row_end) end in this share
  int64_t e = d0 - row;
  const int64_t e_end = d1 - row_end;
  bool head = row < a.n && rp<IdxT>(a, row) < e;  // the first row began in an earlier share
  // column of the matrix that this lane keeps after the reduce-scatter
  int keep_col = c0;
#pragma unroll
  for (int o = 16, half = 8; o >= L && half >= 1; o >>= 1, half >>= 1) keep_col += (lane & o) ? half : 0;

  while (row < row_end || e < e_end) {
    const bool ends = row < row_end;
    const int64_t stop = ends ? rp<IdxT>(a, row + 1) : e_end;
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    for (; e < stop; e += 32) {
      const int cnt = static_cast<int>(min(static_cast<int64_t>(32), stop - e));
      int c = 0;
      float wt = 0.0f;
      if (lane < cnt) {
        c = ld_stream_i32(a.col + e + lane);
        wt = __ldg(a.scale + c);
        if constexpr (MODE == kGcn) wt = __fmul_rn(wt, __ldg(a.dis + c));
        if constexpr (MODE == kWeighted) wt = __fmul_rn(wt, ld_stream_f32(a.ew + e + lane));
      }
      for (int j = 0; j < cnt; j += G) {
        const int src = j + grp;
        const int cj = __shfl_sync(kFull, c, src & 31);
        const float wj = __shfl_sync(kFull, wt, src & 31);
        if (src < cnt && have) {
          const uint4 v = load16<VEC>(a.x + static_cast<int64_t>(cj) * a.ldx, c0, a.f, cj == a.n - 1);
          const uint32_t b[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f4[4];
            bytes_to_float(b[i], f4);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[4 * i + k] = __fmaf_rn(wj, f4[k], acc[4 * i + k]);
          }
        }
      }
    }
    e = stop;
    // reduce-scatter over the lane groups: halves of the columns are exchanged until a
    // lane holds KEEP of them; past 16 groups the last sums are taken whole
    int width = 16;
#pragma unroll
    for (int o = 16; o >= L; o >>= 1) {
      if (width > 1) {
        const int half = width / 2;
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i < half) {
            const float give = up ? acc[i] : acc[i + half];
            const float keep = up ? acc[i + half] : acc[i];
            acc[i] = keep + __shfl_xor_sync(kFull, give, o);
          }
        }
        width = half;
      } else {
        acc[0] += __shfl_xor_sync(kFull, acc[0], o);
      }
    }
    const bool whole = ends && !head;
    float* dst;
    if (whole) {
      const float fr = row_factor<MODE, IdxT>(a, row);
#pragma unroll
      for (int i = 0; i < KEEP; ++i) acc[i] = __fmul_rn(acc[i], fr);
      dst = a.out + row * a.f;
    } else {
      dst = a.part + (head ? 2 * w : 2 * w + 1) * a.f;
    }
    if (keep_col < a.f) {
      if (KEEP >= 4 && keep_col + KEEP <= a.f && (a.f & 3) == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
        for (int i = 0; i + 3 < KEEP; i += 4) {
          *reinterpret_cast<float4*>(dst + keep_col + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < KEEP; ++i) {
          if (keep_col + i < a.f) dst[keep_col + i] = acc[i];
        }
      }
    }
    if (!ends) break;
    head = false;
    ++row;
  }
  // the row that this share began but did not end (its piece is the tail slot), if any
  if (lane == 0 && blockIdx.y == 0) {
    const bool tail = row_end < a.n && rp<IdxT>(a, row_end) < e_end && rp<IdxT>(a, row_end) + row_end >= d0;
    a.part_row[w] = tail ? row_end : -1;
  }
}

// One warp per share whose tail piece begins a row: adds the head pieces of the
// following shares up to the row's end.
template <int MODE, class IdxT>
__global__ void __launch_bounds__(kThreads) spmm_i8_join_kernel(I8SpmmArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (w >= a.shares) return;
  const int64_t row = a.part_row[w];
  if (row < 0) return;
  // the row's end is item row_ptr[row + 1] + row of the merged sequence
  const int64_t last = (rp<IdxT>(a, row + 1) + row) / a.share;
  const float fr = row_factor<MODE, IdxT>(a, row);
  for (int c = lane; c < a.f; c += 32) {
    float s = a.part[(2 * w + 1) * a.f + c];
    for (int64_t k = w + 1; k <= last; ++k) s += a.part[2 * k * a.f + c];
    a.out[row * a.f + c] = __fmul_rn(s, fr);
  }
}

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Items (row ends and entries) per warp: about 8 shares for each warp slot of the
// device, at least 64 so that a share's pieces do not outweigh its rows.
int64_t share_for(int64_t n, int64_t nnz) {
  const int64_t slots = static_cast<int64_t>(sm_count()) * 48 * 4;
  return std::max<int64_t>(64, std::min<int64_t>(2048, (n + nnz + slots - 1) / slots));
}

size_t workspace_for(int64_t n, int64_t nnz, int64_t f) {
  const int64_t share = share_for(n, nnz);
  const int64_t shares = (n + nnz + share - 1) / share;
  return static_cast<size_t>(round_up(shares * 8, 256) + round_up(2 * shares * f * 4, 256));
}

template <int MODE, bool VEC, class IdxT>
void launch_lanes(const I8SpmmArgs& a, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>((a.shares + kWarps - 1) / kWarps);
  const unsigned tiles = static_cast<unsigned>((a.f + kTileCols - 1) / kTileCols);
  const dim3 grid(blocks, tiles);
  if (a.f <= 16) {
    spmm_i8_kernel<MODE, 1, VEC, IdxT><<<grid, kThreads, 0, s>>>(a);
  } else if (a.f <= 32) {
    spmm_i8_kernel<MODE, 2, VEC, IdxT><<<grid, kThreads, 0, s>>>(a);
  } else if (a.f <= 64) {
    spmm_i8_kernel<MODE, 4, VEC, IdxT><<<grid, kThreads, 0, s>>>(a);
  } else if (a.f <= 128) {
    spmm_i8_kernel<MODE, 8, VEC, IdxT><<<grid, kThreads, 0, s>>>(a);
  } else if (a.f <= 256) {
    spmm_i8_kernel<MODE, 16, VEC, IdxT><<<grid, kThreads, 0, s>>>(a);
  } else {
    spmm_i8_kernel<MODE, 32, VEC, IdxT><<<grid, kThreads, 0, s>>>(a);
  }
}

template <int MODE, class IdxT>
int run(const I8SpmmArgs& a, bool vec, cudaStream_t s) {
  if (vec) {
    launch_lanes<MODE, true, IdxT>(a, s);
  } else {
    launch_lanes<MODE, false, IdxT>(a, s);
  }
  GNN_LAUNCH_CHECK("spmm_i8_kernel launch");
  spmm_i8_join_kernel<MODE, IdxT>
      <<<static_cast<unsigned>((a.shares + kWarps - 1) / kWarps), kThreads, 0, s>>>(a);
  GNN_LAUNCH_CHECK("spmm_i8_join_kernel launch");
  return GNN_OK;
}

template <class IdxT>
int run_mode(int mode, const I8SpmmArgs& a, bool vec, cudaStream_t s) {
  switch (mode) {
    case kSum: return run<kSum, IdxT>(a, vec, s);
    case kMean: return run<kMean, IdxT>(a, vec, s);
    case kGcn: return run<kGcn, IdxT>(a, vec, s);
    default: return run<kWeighted, IdxT>(a, vec, s);
  }
}

}  // namespace
}  // namespace gnnb200

using namespace gnnb200;

extern "C" size_t gnn_spmm_int8_workspace_bytes(int64_t num_nodes, int64_t num_edges, int64_t feat_dim) {
  if (num_nodes <= 0 || num_edges < 0 || feat_dim <= 0) return 0;
  return workspace_for(num_nodes, num_edges, feat_dim);
}

extern "C" int gnn_spmm_int8_forward(const void* row_ptr, int row_ptr_type, const int32_t* col_ind, int weighting,
                                     const float* deg_inv_sqrt, const float* edge_weight, const int8_t* x, int64_t ldx,
                                     const float* x_scale, float* out, int64_t num_nodes, int64_t num_edges,
                                     int64_t feat_dim, void* workspace, size_t workspace_bytes, gnn_stream_t stream) {
  GNN_REQUIRE(num_nodes >= 0 && num_edges >= 0 && feat_dim >= 0, GNN_ERR_INVALID_ARGUMENT,
              "num_nodes, num_edges and feat_dim must be >= 0");
  GNN_REQUIRE(row_ptr_type == GNN_INDEX_INT32 || row_ptr_type == GNN_INDEX_INT64, GNN_ERR_INVALID_ARGUMENT,
              "row_ptr must be int32 or int64");
  GNN_REQUIRE(row_ptr_type == GNN_INDEX_INT64 || num_edges <= 0x7fffffffLL, GNN_ERR_INVALID_ARGUMENT,
              "more than 2^31 - 1 entries need an int64 row_ptr");
  GNN_REQUIRE(weighting >= GNN_WEIGHT_SUM && weighting <= GNN_WEIGHT_EDGE, GNN_ERR_INVALID_ARGUMENT,
              "weighting must be one of gnn_weighting");
  if (num_nodes == 0 || feat_dim == 0) {
    clear_error();
    return GNN_OK;
  }
  GNN_REQUIRE(num_nodes <= 0x7fffffffLL, GNN_ERR_UNSUPPORTED, "num_nodes must be <= 2^31 - 1");
  GNN_REQUIRE(feat_dim <= 65535LL * kTileCols, GNN_ERR_UNSUPPORTED, "feat_dim too large");
  GNN_REQUIRE(ldx >= feat_dim, GNN_ERR_INVALID_ARGUMENT, "row stride of x must be >= feat_dim");
  GNN_REQUIRE(row_ptr != nullptr && out != nullptr, GNN_ERR_NULL_POINTER, "row_ptr and out must not be NULL");
  GNN_REQUIRE(num_edges == 0 || (col_ind != nullptr && x != nullptr && x_scale != nullptr), GNN_ERR_NULL_POINTER,
              "col_ind, x and x_scale must not be NULL");
  GNN_REQUIRE(weighting != GNN_WEIGHT_GCN || deg_inv_sqrt != nullptr, GNN_ERR_NULL_POINTER,
              "deg_inv_sqrt must not be NULL");
  GNN_REQUIRE(weighting != GNN_WEIGHT_EDGE || edge_weight != nullptr || num_edges == 0, GNN_ERR_NULL_POINTER,
              "edge_weight must not be NULL");
  const size_t need = workspace_for(num_nodes, num_edges, feat_dim);
  GNN_REQUIRE(workspace != nullptr && workspace_bytes >= need, GNN_ERR_WORKSPACE,
              "workspace missing or too small (gnn_spmm_int8_workspace_bytes)");
  GNN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, GNN_ERR_WORKSPACE,
              "workspace must be 256-byte aligned");
  I8SpmmArgs a{};
  a.row_ptr = row_ptr;
  a.col = col_ind;
  a.dis = deg_inv_sqrt;
  a.ew = edge_weight;
  a.x = x;
  a.ldx = ldx;
  a.scale = x_scale;
  a.out = out;
  a.n = num_nodes;
  a.nnz = num_edges;
  a.f = static_cast<int>(feat_dim);
  a.share = share_for(num_nodes, num_edges);
  a.shares = (num_nodes + num_edges + a.share - 1) / a.share;
  a.part_row = static_cast<int64_t*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + round_up(a.shares * 8, 256));
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 16 == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rc = row_ptr_type == GNN_INDEX_INT32 ? run_mode<int32_t>(weighting, a, vec, s)
                                                 : run_mode<int64_t>(weighting, a, vec, s);
  if (rc == GNN_OK) clear_error();
  return rc;
}
