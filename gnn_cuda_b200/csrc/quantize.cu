// fp32 rows to signed 8-bit rows with one scale each (int8_rows.cuh holds the
// rule), the same for the columns of a weight matrix, and a repack of 8-bit rows
// whose stride or base does not suit TMA.
//
// All three move each byte once. quantize_rows keeps a row's values in registers
// between the maximum and the rounding (4 to 32 lanes a row up to 2,048 columns, a
// block a row up to 4,096); wider rows are read a second time, from L1 / L2.
// Bound by HBM: 232,965 x 256 takes 52 us, 299 MB at 0.88 of the measured copy
// bandwidth. Narrow rows are bound by instructions (about 12 an element with the loads):
// a whole warp for each row of 27 columns took 48 us for 274,063 rows; with eight lanes a
// row the MLP around it went from 102 to 73 us.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "int8_rows.cuh"

namespace gnnb200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;

__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_abs_nan(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// LANES lanes per row, up to LANES * NV * 4 columns: lane l of them holds the columns
// 4 (l + LANES j) .. + 4, so narrow rows share a warp. VEC: cols % 4 == 0, x 16-byte and
// q 4-byte aligned, row by row. R warps' worth of rows are in flight.
template <int LANES, int NV, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const float* __restrict__ x, int64_t ldx,
                                                                 int64_t rows, int cols, int8_t* __restrict__ q,
                                                                 int64_t ldq, float* __restrict__ scale,
                                                                 int word_store) {
  constexpr int R = NV == 1 ? 4 : (NV == 2 ? 2 : 1);
  constexpr int G = 32 / LANES;  // rows side by side in a warp
  const int sub = threadIdx.x & (LANES - 1), side = (threadIdx.x & 31) / LANES;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  for (int64_t r0 = warp * R * G; r0 < rows; r0 += warps * R * G) {
    float v[R][NV * 4];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t row = r0 + i * G + side;
      const float* src = x + row * ldx;
      const bool live = row < rows;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (sub + LANES * j) * 4;
        if constexpr (VEC) {
          float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
          if (live && c < cols) t = __ldcs(reinterpret_cast<const float4*>(src + c));
          v[i][4 * j] = t.x;
          v[i][4 * j + 1] = t.y;
          v[i][4 * j + 2] = t.z;
          v[i][4 * j + 3] = t.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][4 * j + e] = (live && c + e < cols) ? __ldg(src + c + e) : 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t row = r0 + i * G + side;
      float amax = 0.0f;
#pragma unroll
      for (int j = 0; j < NV * 4; ++j) amax = max_abs_nan(amax, v[i][j]);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) amax = max_abs_nan(amax, __shfl_xor_sync(kFull, amax, o));
      const RowQuant rq = row_quant(amax);
      if (row < rows) {
        int8_t* dst = q + row * ldq;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const uint32_t p = quant4(rq, v[i][4 * j], v[i][4 * j + 1], v[i][4 * j + 2], v[i][4 * j + 3]);
          const int c = (sub + LANES * j) * 4;
          if (VEC ? c < cols : (word_store && c + 4 <= cols)) {
            *reinterpret_cast<uint32_t*>(dst + c) = p;
          } else if (!VEC) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (c + e < cols) dst[c + e] = static_cast<int8_t>((p >> (8 * e)) & 0xffu);
            }
          }
        }
        if (sub == 0) scale[row] = rq.s;
      }
    }
  }
}

// One block per row. Rows of up to kThreads * 16 columns stay in registers between the
// maximum and the rounding; wider ones are read again. VEC as above.
template <bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_wide_rows_kernel(const float* __restrict__ x, int64_t ldx,
                                                                      int64_t rows, int64_t cols,
                                                                      int8_t* __restrict__ q, int64_t ldq,
                                                                      float* __restrict__ scale) {
  constexpr int kKeep = 4;  // groups of four columns a thread keeps
  __shared__ float part[kThreads / 32];
  // column e of this thread's group g: four neighbours, or four a block apart
  auto column = [](int64_t g, int e) -> int64_t {
    return VEC ? (g * kThreads + threadIdx.x) * 4 + e : (g * 4 + e) * kThreads + threadIdx.x;
  };
  const int64_t groups = (cols + kThreads * 4 - 1) / (kThreads * 4);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* src = x + r * ldx;
    auto load = [&](int64_t g, float (&v)[4]) {
      if constexpr (VEC) {
        const int64_t c = column(g, 0);
        const float4 t = c < cols ? __ldg(reinterpret_cast<const float4*>(src + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[0] = t.x;
        v[1] = t.y;
        v[2] = t.z;
        v[3] = t.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = column(g, e) < cols ? __ldg(src + column(g, e)) : 0.0f;
      }
    };
    float v[kKeep][4];
    float amax = 0.0f;
#pragma unroll
    for (int g = 0; g < kKeep; ++g) {
      if (g < groups) {
        load(g, v[g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) amax = max_abs_nan(amax, v[g][e]);
      }
    }
    for (int64_t g = kKeep; g < groups; ++g) {
      float t[4];
      load(g, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) amax = max_abs_nan(amax, t[e]);
    }
    amax = warp_max_nan(amax);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
    __syncthreads();
    amax = 0.0f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) amax = max_abs_nan(amax, part[w]);
    const RowQuant rq = row_quant(amax);
    int8_t* dst = q + r * ldq;
    auto store = [&](int64_t g, const float (&t)[4]) {
      const uint32_t p = quant4(rq, t[0], t[1], t[2], t[3]);
      if constexpr (VEC) {
        if (column(g, 0) < cols) *reinterpret_cast<uint32_t*>(dst + column(g, 0)) = p;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (column(g, e) < cols) dst[column(g, e)] = static_cast<int8_t>((p >> (8 * e)) & 0xffu);
        }
      }
    };
#pragma unroll
    for (int g = 0; g < kKeep; ++g) {
      if (g < groups) store(g, v[g]);
    }
    for (int64_t g = kKeep; g < groups; ++g) {
      float t[4];
      load(g, t);
      store(g, t);
    }
    if (threadIdx.x == 0) scale[r] = rq.s;
    __syncthreads();
  }
}

// weight [k, n] -> q [n, k] and one scale per column: 32 columns a block, the
// maximum over k first, then 32 x 32 tiles turned round through shared memory.
__global__ void __launch_bounds__(kThreads) quantize_weight_kernel(const float* __restrict__ w, int64_t k, int64_t n,
                                                                   int8_t* __restrict__ q, int64_t ldq,
                                                                   float* __restrict__ scale) {
  __shared__ float red[8][32];
  __shared__ int8_t tile[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  float amax = 0.0f;
  if (c < n) {
    for (int64_t r = ty; r < k; r += 8) amax = max_abs_nan(amax, __ldg(w + r * n + c));
  }
  red[ty][tx] = amax;
  __syncthreads();
  amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max_abs_nan(amax, red[i][tx]);
  const RowQuant rq = row_quant(amax);
  if (ty == 0 && c < n) scale[c] = rq.s;
  for (int64_t r0 = 0; r0 < k; r0 += 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = r0 + ty + 8 * i;
      tile[tx][ty + 8 * i] = (c < n && r < k) ? quant1(rq, __ldg(w + r * n + c)) : int8_t(0);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + ty + 8 * i;
      if (col < n && r0 + tx < k) q[col * ldq + r0 + tx] = tile[ty + 8 * i][tx];
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads) repack_rows_kernel(const int8_t* __restrict__ x, int64_t ldx, int64_t rows,
                                                               int64_t cols, int8_t* __restrict__ out, int64_t ldo) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); r < rows; r += warps) {
    for (int64_t c = lane; c < cols; c += 32) out[r * ldo + c] = x[r * ldx + c];
  }
}

unsigned grid_for(int64_t units) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(units, 16LL * sm_count())));
}

template <int LANES, int NV>
void launch_rows(bool vec, const float* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* q, int64_t ldq,
                 float* scale, cudaStream_t stream) {
  constexpr int per_block = (NV == 1 ? 4 : (NV == 2 ? 2 : 1)) * (32 / LANES) * (kThreads / 32);
  const unsigned grid = grid_for((rows + per_block - 1) / per_block);
  const int word_store = ldq % 4 == 0 && reinterpret_cast<uintptr_t>(q) % 4 == 0;
  if (vec) {
    quantize_rows_kernel<LANES, NV, true>
        <<<grid, kThreads, 0, stream>>>(x, ldx, rows, static_cast<int>(cols), q, ldq, scale, word_store);
  } else {
    quantize_rows_kernel<LANES, NV, false>
        <<<grid, kThreads, 0, stream>>>(x, ldx, rows, static_cast<int>(cols), q, ldq, scale, word_store);
  }
}

}  // namespace

int quantize_rows(const float* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* q, int64_t ldq, float* scale,
                  cudaStream_t stream) {
  const bool vec = cols % 4 == 0 && ldx % 4 == 0 && ldq % 4 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(q) % 4 == 0;
  if (cols <= 16) {
    launch_rows<4, 1>(vec, x, ldx, rows, cols, q, ldq, scale, stream);
  } else if (cols <= 32) {
    launch_rows<8, 1>(vec, x, ldx, rows, cols, q, ldq, scale, stream);
  } else if (cols <= 64) {
    launch_rows<16, 1>(vec, x, ldx, rows, cols, q, ldq, scale, stream);
  } else if (cols <= 128) {
    launch_rows<32, 1>(vec, x, ldx, rows, cols, q, ldq, scale, stream);
  } else if (cols <= 256) {
    launch_rows<32, 2>(vec, x, ldx, rows, cols, q, ldq, scale, stream);
  } else if (cols <= 512) {
    launch_rows<32, 4>(vec, x, ldx, rows, cols, q, ldq, scale, stream);
  } else if (cols <= 1024) {
    launch_rows<32, 8>(vec, x, ldx, rows, cols, q, ldq, scale, stream);
  } else if (cols <= 2048) {
    launch_rows<32, 16>(vec, x, ldx, rows, cols, q, ldq, scale, stream);
  } else if (vec) {
    quantize_wide_rows_kernel<true><<<grid_for(rows), kThreads, 0, stream>>>(x, ldx, rows, cols, q, ldq, scale);
  } else {
    quantize_wide_rows_kernel<false><<<grid_for(rows), kThreads, 0, stream>>>(x, ldx, rows, cols, q, ldq, scale);
  }
  GNN_LAUNCH_CHECK("quantize_rows launch");
  return GNN_OK;
}

int repack_rows(const int8_t* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* out, int64_t ldo,
                cudaStream_t stream) {
  repack_rows_kernel<<<grid_for((rows + 7) / 8), kThreads, 0, stream>>>(x, ldx, rows, cols, out, ldo);
  GNN_LAUNCH_CHECK("repack_rows launch");
  return GNN_OK;
}

}  // namespace gnnb200

using namespace gnnb200;

extern "C" int gnn_quantize_rows(const float* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* q, int64_t ldq,
                                 float* scale, gnn_stream_t stream) {
  GNN_REQUIRE(rows >= 0 && cols >= 0, GNN_ERR_INVALID_ARGUMENT, "rows and cols must be >= 0");
  if (rows == 0) {
    clear_error();
    return GNN_OK;
  }
  GNN_REQUIRE(scale != nullptr && (cols == 0 || (x != nullptr && q != nullptr)), GNN_ERR_NULL_POINTER,
              "x, q and scale must not be NULL");
  GNN_REQUIRE(ldx >= cols && ldq >= cols, GNN_ERR_INVALID_ARGUMENT, "row strides must be >= cols");
  const int rc = quantize_rows(x, ldx, rows, cols, q, ldq, scale, reinterpret_cast<cudaStream_t>(stream));
  if (rc == GNN_OK) clear_error();
  return rc;
}

extern "C" int gnn_quantize_weight(const float* weight, int64_t k, int64_t n, int8_t* q, int64_t ldq, float* scale,
                                   gnn_stream_t stream) {
  GNN_REQUIRE(k >= 0 && n >= 0, GNN_ERR_INVALID_ARGUMENT, "k and n must be >= 0");
  if (n == 0) {
    clear_error();
    return GNN_OK;
  }
  GNN_REQUIRE(scale != nullptr && (k == 0 || (weight != nullptr && q != nullptr)), GNN_ERR_NULL_POINTER,
              "weight, q and scale must not be NULL");
  GNN_REQUIRE(ldq >= k, GNN_ERR_INVALID_ARGUMENT, "row stride of q must be >= k");
  GNN_REQUIRE((n + 31) / 32 <= 0x7fffffffLL, GNN_ERR_UNSUPPORTED, "weight too wide");
  quantize_weight_kernel<<<static_cast<unsigned>((n + 31) / 32), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      weight, k, n, q, ldq, scale);
  GNN_LAUNCH_CHECK("quantize_weight launch");
  clear_error();
  return GNN_OK;
}
