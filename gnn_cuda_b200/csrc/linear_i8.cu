// Dense transform over 8-bit rows on the tcgen05 tensor cores:
//   acc[i, j] = sum_k x[i, k] * w[j, k]                    (int32, exact)
//   y[i, j]   = relu?((float(acc) * x_scale[i]) * w_scale[j] + bias[j])
// with x [M, K] and w [N, K] in signed 8-bit integers, one fp32 scale per row of
// each; every step of the second line is rounded to fp32. The output is y, or y
// quantised row by row again (int8_rows.cuh) as the next layer's input. fp32 input
// rows are quantised into the workspace first.
//
// Kernel: persistent CTAs walk 128 x BN output tiles. Warp 0 streams 128-byte K
// slices of x and w through a ring of TMA stages (128-byte swizzle; rows, columns
// and K past the edges are zero-filled, which adds nothing to an integer sum);
// warp 1 issues tcgen05.mma kind::i8 (K = 32 per instruction) into one of two TMEM
// accumulators; the other warps drain the other accumulator, apply the scales, bias
// and ReLU, and store fp32 blocks by TMA (or row by row where the output's rows are
// not 16-byte aligned). For an 8-bit output one tile holds whole rows (N <= BN):
// the first pass over TMEM finds each row's largest value, the second rounds.
// Every mbarrier wait is bounded by a clock deadline and records a status code.
//
// Measured on one B200. 2,449,029 x 128 x 128, 8-bit in, fp32 out: 278 us = 0.87 of copy
// bandwidth (HBM-bound; 383 us with four epilogue warps and one staging buffer, 319 with
// eight, 293 with sixteen, then the row scales a tile ahead). 16,384 x 4096 x 4096: 193 us
// alone = 2,850 TOP/s, 237 us back to back under the power cap (tensor-bound).
// 232,965 x 256 x 256 with 8-bit output: 94 us, bound by the epilogue, whose warps meet
// between a row's maximum and its rounding (43 % of the issue slots used).
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "common.cuh"
#include "int8_rows.cuh"
#include "tc_core.cuh"
#include "tma_host.cuh"

namespace gnnb200 {

int quantize_rows(const float* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* q, int64_t ldq, float* scale,
                  cudaStream_t stream);
int repack_rows(const int8_t* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* out, int64_t ldo,
                cudaStream_t stream);

namespace {

using namespace tc;

constexpr unsigned kFull = 0xffffffffu;
constexpr int BM = 128;        // rows per tile (TMEM lanes)
constexpr int KB = 128;        // K bytes per stage: one 128-byte swizzle row
constexpr int kMaxStages = 8;
constexpr size_t kSmemLimit = 227 * 1024;  // per CTA
constexpr size_t kSmemPerSm = 228 * 1024;
constexpr int kBlockBytes = 32 * 32 * 4;  // one epilogue warp's staging: 32 rows x 128 bytes
constexpr int64_t kMaxK = 131071;         // 128 * 128 * K stays below 2^31

// device status word: 0 ok, otherwise the role that gave up waiting
__device__ int g_i8_status = 0;
__device__ __forceinline__ void record_timeout(int code) { atomicCAS(&g_i8_status, 0, code); }

struct I8Params {
  int64_t m, n;
  int64_t m_tiles;
  int n_tiles;
  int k_slices;
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  float* out;        // fp32 output (FP32 kernels)
  int8_t* out8;      // 8-bit output
  float* out_scale;  // its row scales
  int64_t ldo;       // output row stride in elements
  int relu;
  int tma_store;     // fp32 output rows are 16-byte aligned: whole blocks by TMA
  int vec_store;     // 8-bit output rows are 16-byte aligned
};

// y of one element, rounded after each step. Without a bias b is -0, which adds nothing
// to any value; without ReLU `floor` is minus infinity, below which nothing lies.
__device__ __forceinline__ float scaled(int acc, float sx, float sw, float b, float floor) {
  const float y = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(acc), sx), sw), b);
  return y < floor ? 0.0f : y;
}
__device__ __forceinline__ float floor_of(int relu) { return relu ? 0.0f : __int_as_float(0xff800000); }

// Barrier 1 over `threads` threads; true where all of them came with true.
__device__ __forceinline__ bool all_of_barrier(int threads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.aligned.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(v ? 1u : 0u), "r"(threads)
      : "memory");
  return r != 0;
}

// This CTA's tiles, column tiles first: tile blockIdx.x, then every gridDim.x-th.
struct Walk {
  int m, n;            // row tile, column tile
  int dm, dn, n_tiles;
  int64_t left;
  __device__ __forceinline__ Walk(const I8Params& p) {
    n_tiles = p.n_tiles;
    const int grid = static_cast<int>(gridDim.x), first = static_cast<int>(blockIdx.x);
    m = first / n_tiles;
    n = first - m * n_tiles;
    dm = grid / n_tiles;
    dn = grid - dm * n_tiles;
    left = (p.m_tiles * n_tiles - first + grid - 1) / grid;
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next() {
    --left;
    m += dm;
    n += dn;
    if (n >= n_tiles) {
      n -= n_tiles;
      ++m;
    }
  }
};

// One tile kernel: BN columns, 8-bit or fp32 output, EW epilogue warps.
template <int BN, bool OUT8, int EW>
struct Shape {
  static constexpr int kHalves = EW / 4;  // epilogue warps per TMEM lane quarter
  static constexpr int kCols = BN / kHalves >= 32 ? BN / kHalves : 32;  // columns per epilogue warp
  // staging buffers per warp: with two, a block is written while the last one leaves
  static constexpr int kBuffers = OUT8 || EW == 16 || BN == 64 || (BN == 256 && EW == 4) ? 1 : 2;
  // CTAs per SM: narrow tiles move little each, so their latencies are overlapped instead
  static constexpr int kCtas = BN <= 32 ? 3 : (BN <= 64 ? 2 : 1);
  static constexpr size_t fixed() {
    return 1024 /* alignment */ + EW * (kBuffers * kBlockBytes + kCols * 8) + (OUT8 ? kHalves * BM * 4 : 0) + 64;
  }
  static constexpr size_t bytes(int stages) { return fixed() + static_cast<size_t>(stages) * ((BM + BN) * KB + 16); }
  static constexpr int stages() {
    int s = kMaxStages;
    while (bytes(s) + 1024 > kSmemPerSm / kCtas || bytes(s) > kSmemLimit) --s;  // 1 KB a CTA is the system's
    return s;
  }
};

template <int BN, bool OUT8, int EW>
__global__ void __launch_bounds__(64 + 32 * EW, Shape<BN, OUT8, EW>::kCtas)
    linear_i8_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                     const __grid_constant__ CUtensorMap tmap_out, I8Params p) {
  using Sh = Shape<BN, OUT8, EW>;
  constexpr int HALVES = Sh::kHalves;
  constexpr int COLS = Sh::kCols;
  constexpr int S = Sh::stages();
  constexpr uint32_t A_BYTES = BM * KB;
  constexpr uint32_t B_BYTES = BN * KB;
  constexpr uint32_t kTmemCols = 2 * BN;    // two accumulators; BN in {32, 64, 128, 256}
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S * A_BYTES;
  uint8_t* sOut = sB + S * B_BYTES;                                   // staging of the epilogue warps
  float* sCol = reinterpret_cast<float*>(sOut + EW * Sh::kBuffers * kBlockBytes);  // EW x (scales, biases)
  float* sMax = sCol + EW * 2 * COLS;                                 // OUT8: [HALVES][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sMax + (OUT8 ? HALVES * BM : 0));
  uint64_t* full = bars;
  uint64_t* empty = bars + S;
  uint64_t* acc_full = bars + 2 * S;
  uint64_t* acc_empty = bars + 2 * S + 2;
  uint64_t* drain = bars + 2 * S + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  Walk at(p);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], EW);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer ----------------
      int stage = 0;
      uint32_t phase = 0;
      int64_t issued = 0;
      bool ok = true;
      for (; at.more() && ok; at.next()) {
        const int row = at.m * BM;
        const int col = at.n * BN;
        for (int ks = 0; ks < p.k_slices; ++ks) {
          if (!mbar_wait(&empty[stage], phase ^ 1)) {
            record_timeout(33);
            ok = false;
            break;
          }
          mbar_expect_tx(&full[stage], A_BYTES + B_BYTES);
          tma_load_2d(sA + stage * A_BYTES, &tmap_x, &full[stage], ks * KB, row);
          tma_load_2d(sB + stage * B_BYTES, &tmap_w, &full[stage], ks * KB, col);
          ++issued;
          if (++stage == S) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // the last min(issued, S) copies must have landed before exit
      const int64_t pending = issued < S ? issued : S;
      for (int64_t i = 0; i < pending; ++i) {
        if (--stage < 0) {
          stage = S - 1;
          phase ^= 1;
        }
        if (!mbar_wait(&full[stage], phase)) record_timeout(37);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t idesc = idesc_s8(BM, BN);
      const uint32_t sa_base = smem_u32(sA);
      const uint32_t sb_base = smem_u32(sB);
      bool ok = true;
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      for (; at.more() && ok; at.next()) {
        if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1)) {
          record_timeout(34);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int ks = 0; ks < p.k_slices; ++ks) {
          if (!mbar_wait(&full[stage], phase)) {
            record_timeout(34);
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < KB / 32; ++kk) {
            const uint64_t a_desc = sw128_desc(sa_base + stage * A_BYTES + kk * 32, 16, 1024);
            const uint64_t b_desc = sw128_desc(sb_base + stage * B_BYTES + kk * 32, 16, 1024);
            mma_s8(d_tmem, a_desc, b_desc, idesc, (ks | kk) != 0 ? 1u : 0u);
          }
          mma_commit(&empty[stage]);
          if (++stage == S) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit(&acc_full[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      mma_commit(drain);  // all MMAs complete before TMEM is released
      if (!mbar_wait(drain, 0)) record_timeout(38);
    }
  } else {
    // ---------------- epilogue ----------------
    const int ew = warp - 2;
    const int q = warp & 3;          // TMEM lane quarter this warp may access
    const int half = ew / 4;
    const int cbeg = half * COLS;    // this warp's columns of the tile: [cbeg, cend)
    const int cend = cbeg + COLS <= BN ? cbeg + COLS : (cbeg < BN ? BN : cbeg);
    uint8_t* staging = sOut + ew * (Sh::kBuffers * kBlockBytes);
    float* scales = sCol + ew * 2 * COLS;  // of this warp's columns, read by all lanes as broadcasts
    float* biases = scales + COLS;
    const float floor = floor_of(p.relu);
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t blocks = 0;      // blocks staged so far
    int have_cols = -1;       // the column tile whose scales are there
    auto load_scale = [&]() -> float {
      const int64_t r = static_cast<int64_t>(at.m) * BM + 32 * q + lane;
      return at.more() && r < p.m ? __ldg(p.x_scale + r) : 0.0f;
    };
    float sx_next = load_scale();
    while (at.more()) {
      const int64_t row0 = static_cast<int64_t>(at.m) * BM + 32 * q;  // first row of this warp's lane quarter
      const int n_tile = at.n;
      const int64_t n0 = static_cast<int64_t>(n_tile) * BN;
      const float sx = sx_next;
      at.next();
      sx_next = load_scale();  // a tile ahead of its use
      if (n_tile != have_cols) {
        have_cols = n_tile;
        __syncwarp();
#pragma unroll
        for (int c0 = 0; c0 < COLS; c0 += 32) {
          const int64_t c = n0 + cbeg + c0 + lane;
          scales[c0 + lane] = c < p.n ? __ldg(p.w_scale + c) : 0.0f;
          biases[c0 + lane] = (p.bias != nullptr && c < p.n) ? __ldg(p.bias + c) : -0.0f;
        }
        __syncwarp();
      }
      // warp-uniform decision: the tcgen05.ld below is .sync.aligned. An 8-bit output's warps
      // meet at a barrier, so they decide together; that meeting also orders the last tile's
      // reads of sMax before this tile's writes.
      bool ready = __all_sync(kFull, mbar_wait(&acc_full[acc], acc_phase));
      if constexpr (OUT8) ready = all_of_barrier(EW * 32, ready);
      if (!ready) {
        if (lane == 0) record_timeout(35);
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + static_cast<uint32_t>(acc * BN) + (static_cast<uint32_t>(32 * q) << 16);
      // y of columns [c0, c0 + 32) of this warp's share
      auto transform = [&](int c0, uint32_t (&r)[32]) {
        tmem_ld32(taddr + static_cast<uint32_t>(cbeg + c0), r);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 sw = *reinterpret_cast<const float4*>(scales + c0 + j);
          const float4 sb = *reinterpret_cast<const float4*>(biases + c0 + j);
          r[j] = __float_as_uint(scaled(static_cast<int>(r[j]), sx, sw.x, sb.x, floor));
          r[j + 1] = __float_as_uint(scaled(static_cast<int>(r[j + 1]), sx, sw.y, sb.y, floor));
          r[j + 2] = __float_as_uint(scaled(static_cast<int>(r[j + 2]), sx, sw.z, sb.z, floor));
          r[j + 3] = __float_as_uint(scaled(static_cast<int>(r[j + 3]), sx, sw.w, sb.w, floor));
        }
      };
      if constexpr (!OUT8) {
        const bool has_rows = row0 < p.m;
#pragma unroll 1
        for (int c0 = 0; c0 < COLS && has_rows; c0 += 32) {
          if (cbeg + c0 >= BN || n0 + cbeg + c0 >= p.n) break;
          uint32_t r[32];
          transform(c0, r);
          uint8_t* buf = staging + (Sh::kBuffers == 2 ? (blocks & 1) * kBlockBytes : 0);
          ++blocks;
          if (p.tma_store) {
            if (lane == 0) {  // the store that last used this buffer has read it
              if constexpr (Sh::kBuffers == 2) {
                bulk_wait_read_1();
              } else {
                bulk_wait_read_0();
              }
            }
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            *reinterpret_cast<uint4*>(buf + lane * 128 + ((((j >> 2) ^ (lane & 7))) << 4)) =
                make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
          }
          if (p.tma_store) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmap_out, buf, static_cast<int>(n0 + cbeg + c0), static_cast<int>(row0));
              bulk_commit();
            }
          } else {
            __syncwarp();
            const int64_t c = n0 + cbeg + c0 + lane;
            const int rows = static_cast<int>(p.m - row0 < 32 ? p.m - row0 : 32);
            if (c < p.n) {
              float* dst = p.out + row0 * p.ldo + c;
#pragma unroll 8
              for (int j = 0; j < rows; ++j) {
                dst[j * p.ldo] = *reinterpret_cast<const float*>(buf + j * 128 + (((lane >> 2) ^ (j & 7)) << 4) +
                                                                ((lane & 3) << 2));
              }
            }
            __syncwarp();
          }
        }
      } else {
        // one tile holds whole rows; a lane keeps its row's values in registers between
        // the largest of them and the rounding
        uint32_t r[COLS / 32][32];
        float amax = 0.0f;
#pragma unroll
        for (int b = 0; b < COLS / 32; ++b) {
          if (cbeg + b * 32 < BN) {
            transform(b * 32, r[b]);
            if (p.n < BN) {  // columns past n are 0 * x_scale, which an infinite or NaN scale makes NaN
              const int live = static_cast<int>(p.n) - cbeg - b * 32;
#pragma unroll
              for (int j = 0; j < 32; ++j) r[b][j] = j < live ? r[b][j] : 0u;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) amax = max_abs_nan(amax, __uint_as_float(r[b][j]));
          }
        }
        sMax[half * BM + 32 * q + lane] = amax;
        asm volatile("bar.sync 1, %0;" ::"n"(EW * 32) : "memory");
#pragma unroll
        for (int h = 0; h < HALVES; ++h) amax = max_abs_nan(amax, sMax[h * BM + 32 * q + lane]);
        const RowQuant rq = row_quant(amax);
        if (half == 0 && row0 + lane < p.m) p.out_scale[row0 + lane] = rq.s;
#pragma unroll
        for (int b = 0; b < COLS / 32; ++b) {
          if (cbeg + b * 32 < BN) {
            // 32 columns are 32 bytes: two 16-byte chunks of this row's up to 128 staged bytes
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t* y = &r[b][h * 16 + i * 4];
                w[i] = quant4(rq, __uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]),
                              __uint_as_float(y[3]));
              }
              const int chunk = b * 2 + h;
              *reinterpret_cast<uint4*>(staging + lane * 128 + ((chunk ^ (lane & 7)) << 4)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        __syncwarp();
        // 8 lanes a row, 16 bytes each, 4 rows a pass
        const int chunk = lane & 7;
        const int64_t c = cbeg + chunk * 16;
        if (chunk * 16 < cend - cbeg && c < p.n) {
          const int bytes = static_cast<int>(p.n - c < 16 ? p.n - c : 16);
#pragma unroll
          for (int pass = 0; pass < 8; ++pass) {
            const int j = pass * 4 + (lane >> 3);
            if (row0 + j >= p.m) break;
            const uint4 v = *reinterpret_cast<const uint4*>(staging + j * 128 + ((chunk ^ (j & 7)) << 4));
            int8_t* dst = p.out8 + (row0 + j) * p.ldo + c;
            if (p.vec_store && bytes == 16) {
              *reinterpret_cast<uint4*>(dst) = v;
            } else {
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                if (i < bytes) dst[i] = static_cast<int8_t>((w[i >> 2] >> (8 * (i & 3))) & 0xffu);
              }
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (!OUT8) {
      if (lane == 0) bulk_wait_all();  // shared staging must outlive the stores reading it
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// ---- a few rows ----------------------------------------------------------------
//
// Up to kSmallRows rows are bound by latency and by reading w once, so no tensor core
// is set up: one kernel quantises the rows (fp32 input; every block for itself, they
// are small) into shared memory, zero-padded to 16 columns, and a warp takes an output
// channel, 16 bytes of w a lane, with four-way 8-bit dot products.
constexpr int kSmallRows = 16;
constexpr int kSmallBytes = 40 * 1024;  // shared memory for the rows
constexpr int kSmallThreads = 256;

struct SmallParams {
  const void* x;
  int64_t ldx;
  const float* x_scale;  // NULL: x is fp32
  const int8_t* w;
  int64_t ldw;
  const float* w_scale;
  const float* bias;
  float* out;
  int64_t ldo;
  int m, k, n;
  int relu;
};

template <int MR>
__global__ void __launch_bounds__(kSmallThreads) linear_i8_small_kernel(SmallParams p) {
  extern __shared__ __align__(16) int8_t sx[];  // [m][pitch]
  __shared__ float sscale[kSmallRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = (p.k + 15) / 16;
  const int pitch = chunks * 16;
  int64_t j = static_cast<int64_t>(blockIdx.x) * (kSmallThreads / 32) + warp;
  // 16 bytes of row j of w; its last piece byte by byte where the last row may end
  auto load_w = [&](int64_t row, int c) -> uint4 {
    const int8_t* src = p.w + row * p.ldw + c * 16;
    if (c * 16 + 16 <= p.k || row < p.n - 1) return __ldg(reinterpret_cast<const uint4*>(src));
    uint32_t v[4] = {0, 0, 0, 0};
    for (int i = 0; c * 16 + i < p.k; ++i) {
      v[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(src + i))) << (8 * (i & 3));
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  };
  uint4 first = make_uint4(0, 0, 0, 0);  // on its way while the rows are quantised
  if (j < p.n && lane < chunks) first = load_w(j, lane);

  for (int r = warp; r < p.m; r += kSmallThreads / 32) {
    int8_t* dst = sx + r * pitch;
    if (p.x_scale == nullptr) {
      const float* src = static_cast<const float*>(p.x) + r * p.ldx;
      float amax = 0.0f;
      for (int c = lane; c < p.k; c += 32) amax = max_abs_nan(amax, __ldg(src + c));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = max_abs_nan(amax, __shfl_xor_sync(kFull, amax, o));
      const RowQuant rq = row_quant(amax);
      for (int c = lane; c < pitch; c += 32) dst[c] = c < p.k ? quant1(rq, __ldg(src + c)) : int8_t(0);
      if (lane == 0) sscale[r] = rq.s;
    } else {
      const int8_t* src = static_cast<const int8_t*>(p.x) + r * p.ldx;
      for (int c = lane; c < pitch; c += 32) dst[c] = c < p.k ? __ldg(src + c) : int8_t(0);
      if (lane == 0) sscale[r] = __ldg(p.x_scale + r);
    }
  }
  __syncthreads();

  const int64_t step = static_cast<int64_t>(gridDim.x) * (kSmallThreads / 32);
  for (bool again = false; j < p.n; j += step, again = true) {
    int acc[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) acc[r] = 0;
    for (int c = lane; c < chunks; c += 32) {
      const uint4 w = (c == lane && !again) ? first : load_w(j, c);
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        if (r < p.m) {
          const uint4 v = *reinterpret_cast<const uint4*>(sx + r * pitch + c * 16);
          acc[r] = __dp4a(static_cast<int>(v.x), static_cast<int>(w.x), acc[r]);
          acc[r] = __dp4a(static_cast<int>(v.y), static_cast<int>(w.y), acc[r]);
          acc[r] = __dp4a(static_cast<int>(v.z), static_cast<int>(w.z), acc[r]);
          acc[r] = __dp4a(static_cast<int>(v.w), static_cast<int>(w.w), acc[r]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < MR; ++r) acc[r] = __reduce_add_sync(kFull, acc[r]);
    if (lane < p.m) {
      int mine = acc[0];
#pragma unroll
      for (int r = 1; r < MR; ++r) mine = lane == r ? acc[r] : mine;
      p.out[lane * p.ldo + j] = scaled(mine, sscale[lane], __ldg(p.w_scale + j),
                                       p.bias != nullptr ? __ldg(p.bias + j) : -0.0f, floor_of(p.relu));
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

bool aligned_rows(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 16 == 0; }

int encode_rows(CUtensorMap* map, const int8_t* p, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {KB, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dims, strides, box,
                                 estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(GNN_ERR_CUDA, "cuTensorMapEncodeTiled(int8 rows) failed: " + std::to_string(r));
  return GNN_OK;
}

template <int BN, bool OUT8, int EW>
int launch_bn(const int8_t* x, int64_t ldx, const int8_t* w, int64_t ldw, int64_t k, I8Params p, cudaStream_t stream) {
  CUtensorMap tx{}, tw{}, to{};
  int rc = encode_rows(&tx, x, p.m, k, ldx, BM);
  if (rc == GNN_OK) rc = encode_rows(&tw, w, p.n, k, ldw, BN);
  if (rc != GNN_OK) return rc;
  if (!OUT8 && p.tma_store) {
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.n), static_cast<cuuint64_t>(p.m)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.ldo) * 4};
    cuuint32_t box[2] = {32, 32};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = encode_fn()(&to, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, p.out, dims, strides, box, estr,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GNN_ERR_CUDA, "cuTensorMapEncodeTiled(out) failed: " + std::to_string(r));
  }
  p.m_tiles = (p.m + BM - 1) / BM;
  p.n_tiles = static_cast<int>((p.n + BN - 1) / BN);
  p.k_slices = static_cast<int>((k + KB - 1) / KB);
  constexpr int stages = Shape<BN, OUT8, EW>::stages();
  constexpr size_t smem = Shape<BN, OUT8, EW>::bytes(stages);
  static_assert(stages >= 2, "at least two stages have to fit");
  // the opt-in is a per-device function attribute
  static bool configured[64] = {};
  static std::mutex mu;
  int dev = 0;
  GNN_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
      GNN_CUDA_TRY(cudaFuncSetAttribute(linear_i8_kernel<BN, OUT8, EW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(smem)),
                   "linear_i8_kernel: shared memory opt-in");
      if (dev >= 0 && dev < 64) configured[dev] = true;
    }
  }
  const int64_t ctas = std::min<int64_t>(p.m_tiles * p.n_tiles, static_cast<int64_t>(Shape<BN, OUT8, EW>::kCtas) * sm_count());
  linear_i8_kernel<BN, OUT8, EW><<<static_cast<unsigned>(ctas), 64 + 32 * EW, smem, stream>>>(
      tx, tw, to, p);
  GNN_LAUNCH_CHECK("linear_i8_kernel launch");
  return GNN_OK;
}

template <bool OUT8>
int launch(const int8_t* x, int64_t ldx, const int8_t* w, int64_t ldw, int64_t k, const I8Params& p,
           cudaStream_t stream) {
  if (p.n <= 32) return launch_bn<32, OUT8, 4>(x, ldx, w, ldw, k, p, stream);
  if (p.n <= 64) return launch_bn<64, OUT8, 8>(x, ldx, w, ldw, k, p, stream);
  if (p.n <= 128) return launch_bn<128, OUT8, 16>(x, ldx, w, ldw, k, p, stream);
  if constexpr (!OUT8) {
    // Long K: the MMAs are the bottleneck, and a fourth stage is worth more than a faster epilogue.
    if (k >= 1024) return launch_bn<256, OUT8, 4>(x, ldx, w, ldw, k, p, stream);
  }
  return launch_bn<256, OUT8, 16>(x, ldx, w, ldw, k, p, stream);
}

// Whether the few-rows kernel takes the call: fp32 output, aligned w, and rows so small
// together that every block can quantise or copy them for itself, a warp a row. Measured
// against the tile kernel (with the quantiser for fp32 rows), us on the device, K x N:
//   fp32 rows   512 x 512, 1 row 4.6 / 8.0, 16 rows 8.0 / 8.5; 512 x 4096, 16 rows 11.9 / 8.6;
//               1024 x 4096, 8 rows 11.2 / 10.9 (whole calls 12.7 / 18.7); 2048 x 512, 1 row 12.6 / 13.6;
//               4096 x 512, 1 row 23.4 / 17.8; 40,960 x 512, 1 row 405 / 106
//   8-bit rows  4096 x 512, 1 row 11.2 / 15.3, 2 rows 15.8 / 15.3; 40,960 x 512, 1 row 95.3 / 95.0
constexpr int64_t kSmallK = 2048;  // the longest row that is quantised, or stands beside others

bool small_call(int x_type, const int8_t* w, int64_t ldw, int out_type, int64_t m, int64_t k) {
  const bool alone = m == 1 && x_type == GNN_ROWS_INT8;
  return out_type == GNN_ROWS_FP32 && m <= kSmallRows && (alone || (k <= kSmallK && m * k <= 8192)) &&
         m * round_up(k, 16) <= kSmallBytes && aligned_rows(w, ldw);
}

int launch_small(const SmallParams& p, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(p.m) * round_up(p.k, 16);
  const unsigned grid = static_cast<unsigned>(
      std::min<int64_t>((p.n + kSmallThreads / 32 - 1) / (kSmallThreads / 32), 8LL * sm_count()));
  if (p.m <= 1) {
    linear_i8_small_kernel<1><<<grid, kSmallThreads, smem, stream>>>(p);
  } else if (p.m <= 2) {
    linear_i8_small_kernel<2><<<grid, kSmallThreads, smem, stream>>>(p);
  } else if (p.m <= 4) {
    linear_i8_small_kernel<4><<<grid, kSmallThreads, smem, stream>>>(p);
  } else if (p.m <= 8) {
    linear_i8_small_kernel<8><<<grid, kSmallThreads, smem, stream>>>(p);
  } else {
    linear_i8_small_kernel<16><<<grid, kSmallThreads, smem, stream>>>(p);
  }
  GNN_LAUNCH_CHECK("linear_i8_small_kernel launch");
  return GNN_OK;
}

constexpr int64_t kMaxRow8 = 256;  // widest 8-bit output row that one tile holds

// Workspace: [quantised or repacked x][its scales][repacked w][fp32 rows of a wide 8-bit output]
struct Plan {
  int64_t x_bytes = 0, scale_bytes = 0, w_bytes = 0, y_bytes = 0;
  size_t total() const { return static_cast<size_t>(x_bytes + scale_bytes + w_bytes + y_bytes); }
};

Plan plan_for(const void* x, int x_type, int64_t ldx, const int8_t* w, int64_t ldw, int out_type, int64_t m, int64_t k,
              int64_t n) {
  Plan p;
  if (small_call(x_type, w, ldw, out_type, m, k)) return p;
  const int64_t pitch = round_up(std::max<int64_t>(k, 1), 16);
  if (x_type == GNN_ROWS_FP32) {
    p.x_bytes = round_up(m * pitch, 256);
    p.scale_bytes = round_up(m * 4, 256);
  } else if (!aligned_rows(x, ldx)) {
    p.x_bytes = round_up(m * pitch, 256);
  }
  if (!aligned_rows(w, ldw)) p.w_bytes = round_up(n * pitch, 256);
  if (out_type == GNN_ROWS_INT8 && n > kMaxRow8) p.y_bytes = round_up(m * n * 4, 256);
  return p;
}

}  // namespace

int i8_status_read(int reset, int* status) {
  GNN_CUDA_TRY(cudaMemcpyFromSymbol(status, g_i8_status, sizeof(int)), "read 8-bit transform status word");
  if (reset) {
    const int zero = 0;
    GNN_CUDA_TRY(cudaMemcpyToSymbol(g_i8_status, &zero, sizeof(int)), "reset 8-bit transform status word");
  }
  return GNN_OK;
}

}  // namespace gnnb200

using namespace gnnb200;

extern "C" size_t gnn_linear_int8_workspace_bytes(const void* x, int x_type, int64_t ldx, const int8_t* weight,
                                                  int64_t ldw, int out_type, int64_t m, int64_t k, int64_t n) {
  if (m <= 0 || k < 0 || n <= 0) return 0;
  return plan_for(x, x_type, ldx, weight, ldw, out_type, m, k, n).total();
}

extern "C" int gnn_linear_int8_forward(const void* x, int x_type, int64_t ldx, const float* x_scale,
                                       const int8_t* weight, int64_t ldw, const float* weight_scale, const float* bias,
                                       void* out, int out_type, int64_t ldo, float* out_scale, int64_t m, int64_t k,
                                       int64_t n, int relu, void* workspace, size_t workspace_bytes,
                                       gnn_stream_t stream) {
  GNN_REQUIRE(m >= 0 && k >= 1 && n >= 0, GNN_ERR_INVALID_ARGUMENT, "m and n must be >= 0, k >= 1");
  GNN_REQUIRE((x_type == GNN_ROWS_FP32 || x_type == GNN_ROWS_INT8) &&
                  (out_type == GNN_ROWS_FP32 || out_type == GNN_ROWS_INT8),
              GNN_ERR_INVALID_ARGUMENT, "row types must be GNN_ROWS_FP32 or GNN_ROWS_INT8");
  GNN_REQUIRE(k <= kMaxK, GNN_ERR_UNSUPPORTED, "k must be <= 131071 (32-bit sums of 8-bit products)");
  GNN_REQUIRE(m <= (int64_t(1) << 31) - BM && n <= (int64_t(1) << 31) - 256, GNN_ERR_UNSUPPORTED,
              "int8 linear: too many rows or columns");
  GNN_REQUIRE(ldx >= k && ldw >= k && ldo >= n, GNN_ERR_INVALID_ARGUMENT, "row strides must hold a whole row");
  if (m == 0 || n == 0) {
    clear_error();
    return GNN_OK;
  }
  GNN_REQUIRE(x != nullptr && weight != nullptr && weight_scale != nullptr && out != nullptr, GNN_ERR_NULL_POINTER,
              "x, weight, weight_scale and out must not be NULL");
  GNN_REQUIRE(x_type == GNN_ROWS_FP32 || x_scale != nullptr, GNN_ERR_NULL_POINTER,
              "x_scale must not be NULL for 8-bit x");
  GNN_REQUIRE(out_type == GNN_ROWS_FP32 || out_scale != nullptr, GNN_ERR_NULL_POINTER,
              "out_scale must not be NULL for 8-bit out");
  GNN_REQUIRE(device_is_sm100() && encode_fn() != nullptr, GNN_ERR_DEVICE, "int8 linear needs an sm_100 device");
  const Plan plan = plan_for(x, x_type, ldx, weight, ldw, out_type, m, k, n);
  GNN_REQUIRE(plan.total() == 0 || (workspace != nullptr && workspace_bytes >= plan.total()), GNN_ERR_WORKSPACE,
              "workspace missing or too small (gnn_linear_int8_workspace_bytes)");
  GNN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, GNN_ERR_WORKSPACE,
              "workspace must be 256-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (small_call(x_type, weight, ldw, out_type, m, k)) {
    const SmallParams sp{x, ldx, x_type == GNN_ROWS_FP32 ? nullptr : x_scale, weight, ldw, weight_scale, bias,
                         static_cast<float*>(out), ldo, static_cast<int>(m), static_cast<int>(k), static_cast<int>(n),
                         relu ? 1 : 0};
    const int rc = launch_small(sp, s);
    if (rc == GNN_OK) clear_error();
    return rc;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t pitch = round_up(k, 16);
  int rc = GNN_OK;
  const int8_t* xq = static_cast<const int8_t*>(x);
  if (x_type == GNN_ROWS_FP32) {
    int8_t* q = reinterpret_cast<int8_t*>(ws);
    float* sc = reinterpret_cast<float*>(ws + plan.x_bytes);
    rc = quantize_rows(static_cast<const float*>(x), ldx, m, k, q, pitch, sc, s);
    xq = q;
    x_scale = sc;
    ldx = pitch;
  } else if (plan.x_bytes) {
    rc = repack_rows(xq, ldx, m, k, reinterpret_cast<int8_t*>(ws), pitch, s);
    xq = reinterpret_cast<int8_t*>(ws);
    ldx = pitch;
  }
  if (rc == GNN_OK && plan.w_bytes) {
    int8_t* q = reinterpret_cast<int8_t*>(ws + plan.x_bytes + plan.scale_bytes);
    rc = repack_rows(weight, ldw, n, k, q, pitch, s);
    weight = q;
    ldw = pitch;
  }
  if (rc != GNN_OK) return rc;
  I8Params p{};
  p.m = m;
  p.n = n;
  p.x_scale = x_scale;
  p.w_scale = weight_scale;
  p.bias = bias;
  p.relu = relu ? 1 : 0;
  if (out_type == GNN_ROWS_FP32 || plan.y_bytes) {
    p.out = out_type == GNN_ROWS_FP32 ? static_cast<float*>(out)
                                      : reinterpret_cast<float*>(ws + plan.x_bytes + plan.scale_bytes + plan.w_bytes);
    p.ldo = out_type == GNN_ROWS_FP32 ? ldo : n;
    p.tma_store = aligned_rows(p.out, p.ldo * 4) ? 1 : 0;
    rc = launch<false>(xq, ldx, weight, ldw, k, p, s);
    if (rc == GNN_OK && plan.y_bytes) {
      rc = quantize_rows(p.out, n, m, n, static_cast<int8_t*>(out), ldo, out_scale, s);
    }
  } else {
    p.out8 = static_cast<int8_t*>(out);
    p.out_scale = out_scale;
    p.ldo = ldo;
    p.vec_store = aligned_rows(out, ldo) ? 1 : 0;
    rc = launch<true>(xq, ldx, weight, ldw, k, p, s);
  }
  if (rc == GNN_OK) clear_error();
  return rc;
}
