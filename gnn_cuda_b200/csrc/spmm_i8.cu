// CSR aggregation over 8-bit feature rows with one fp32 scale each:
//   out[r, :] = f_r * sum_e w_e * scale[c_e] * q[c_e, :]
// with (f_r, w_e) = (dis[r], dis[c_e]) for GCN, (1, edge_weight[e]) weighted,
// (1, 1) sum and (1 / deg r, 1) mean; sums in fp32.
//
// Split: the merged sequence of row ends and entries is cut into equal shares (the
// cut points are found by a binary search on row_ptr), so hubs, short and empty rows
// all balance. A share is summed by a group of L lanes, 16 columns a lane: a warp
// works on 32 / L shares at once, each load instruction brings 32 / L feature rows,
// and nothing is joined across lanes. A group stores the rows that lie wholly in its
// share; what it holds of a row that began earlier, or ends later, goes to a
// workspace slot, and a second small kernel adds those pieces in share order: no
// float atomics, the same bits every time.
//
// The entries are those that row_ptr spans, [row_ptr[0], row_ptr[n]), whatever the host
// gives as their number: that one sizes the grid and the scratch and is the length of
// col_ind and edge_weight, so entries past it count as absent and are recorded as a status.
//
// Measured on one B200 (612,257 nodes, 16,077,042 entries, GCN, F = 128): 448 us, the pieces
// among them. Bound by instructions (0.66 a cycle and scheduler; unpacking and adding
// 16 columns of an entry takes 36) and by the L2's gathers (2.06 GB of rows at 4.6 TB/s).
// Against it: a whole warp per share with four columns a lane 684-790 us, lane groups on
// one share joined at row ends 712 us, two rows in flight instead of four 521 us. The loop is
// sensitive to registers: row ends clamped to the span in it 467 us, degrees taken from the
// row ends 479 us, the first entry's place in 64 bits 468 us. Byte loads, of 100,000
// contiguous rows of 100 columns with 1,500,000 entries: 175 us.
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

// device status word: 0 ok, 39 row_ptr spans entries outside [0, num_edges)
__device__ int g_spmm_i8_status = 0;
constexpr int kSpanOutside = 39;

enum Mode : int { kSum = GNN_WEIGHT_SUM, kMean = GNN_WEIGHT_MEAN, kGcn = GNN_WEIGHT_GCN, kWeighted = GNN_WEIGHT_EDGE };

struct I8SpmmArgs {
  const void* row_ptr;
  const int32_t* col;
  const float* dis;      // GCN row factors
  const float* dis_col;  // GCN column factors; NULL where `scale` has them in already
  const float* ew;
  const int8_t* x;
  int64_t ldx;
  const float* scale;
  float* out;
  int64_t n, nnz;
  int f;
  int mode;
  int64_t share;    // row ends + entries per lane group
  int64_t shares;   // number of shares
  float* part;      // [2 * shares, f]: head (row began earlier), tail (row ends later)
  int64_t* part_row;  // [shares] row of the tail piece, -1 none
};

// How feature rows can be read.
enum Kind : int {
  kWhole = 0,   // 16-byte aligned rows, f % 16 == 0
  kRagged = 1,  // 16-byte aligned rows; the last lane's load runs past f within the stride
  kBytes = 2    // any base and stride
};

// 16 columns of row c; xl: the matrix's base plus this lane's first column c0. The
// last row of the matrix may lack the storage behind its last column.
template <int KIND>
__device__ __forceinline__ uint4 load_row(const int8_t* xl, uint32_t ldx, int c, int c0, int f, int last_row) {
  const int8_t* p = xl + static_cast<uint64_t>(static_cast<uint32_t>(c)) * ldx;
  if (KIND == kWhole || (KIND == kRagged && (c0 + 16 <= f || c != last_row))) {
    return __ldg(reinterpret_cast<const uint4*>(p));
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (c0 + i < f) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(p + i))) << (8 * (i & 3));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// acc += w * the four signed bytes of v, two columns an instruction. Each byte
// becomes the low mantissa bits of 2^23 + 128 + q, from which 2^23 + 128 is taken off
// again: exact, and without the conversion unit.
__device__ __forceinline__ void fma_word(uint64_t ww, uint32_t v, uint64_t& a01, uint64_t& a23) {
  v ^= 0x80808080u;
  const uint32_t b0 = __byte_perm(v, 0x4b000000u, 0x7540), b1 = __byte_perm(v, 0x4b000000u, 0x7541);
  const uint32_t b2 = __byte_perm(v, 0x4b000000u, 0x7542), b3 = __byte_perm(v, 0x4b000000u, 0x7543);
  asm("{\n\t.reg .b64 p, q, m;\n\t"
      "mov.b64 p, {%2, %3};\n\t"
      "mov.b64 q, {%4, %5};\n\t"
      "mov.b64 m, {%7, %7};\n\t"
      "add.rn.f32x2 p, p, m;\n\t"
      "add.rn.f32x2 q, q, m;\n\t"
      "fma.rn.f32x2 %0, %6, p, %0;\n\t"
      "fma.rn.f32x2 %1, %6, q, %1;\n\t}"
      : "+l"(a01), "+l"(a23)
      : "r"(b0), "r"(b1), "r"(b2), "r"(b3), "l"(ww), "r"(0xcb000080u));  // -(2^23 + 128)
}

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}

// eight floats, one 32-byte sector, not to be kept in the caches
__device__ __forceinline__ void store8(float* p, const float* f) {
  asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(__float_as_uint(f[0])),
               "r"(__float_as_uint(f[1])), "r"(__float_as_uint(f[2])), "r"(__float_as_uint(f[3])),
               "r"(__float_as_uint(f[4])), "r"(__float_as_uint(f[5])), "r"(__float_as_uint(f[6])),
               "r"(__float_as_uint(f[7]))
               : "memory");
}

template <class IdxT>
__device__ __forceinline__ int64_t rp(const I8SpmmArgs& a, int64_t r) {
  return static_cast<int64_t>(__ldg(static_cast<const IdxT*>(a.row_ptr) + r));
}

// The rows of the CSR over the entries that exist: row r begins at(row_ptr[r]), counted from
// the first entry, `base`; never below 0 nor past `span`, whatever row_ptr holds.
template <class IdxT>
struct Rows {
  const IdxT* ptr;
  IdxT base, end;
  bool cut;  // row_ptr reaches outside the entries
  __device__ __forceinline__ explicit Rows(const I8SpmmArgs& a) : ptr(static_cast<const IdxT*>(a.row_ptr)) {
    const IdxT limit = static_cast<IdxT>(a.nnz), first = __ldg(ptr), last = __ldg(ptr + a.n);
    base = min(max(first, IdxT(0)), limit);
    end = min(max(last, base), limit);
    cut = base != first || end != last;
  }
  __device__ __forceinline__ int64_t span() const { return static_cast<int64_t>(end - base); }
  __device__ __forceinline__ int64_t at(IdxT v) const { return static_cast<int64_t>(min(max(v, base), end) - base); }
  __device__ __forceinline__ int64_t begin(int64_t r) const { return at(__ldg(ptr + r)); }
};

// Number of row ends among the first `d` items of the merged sequence (row r's end
// comes after its entries): the smallest r with begin(r + 1) + r + 1 > d. The L
// lanes of a group ask at L places a round; all groups of the warp take part. Past the
// sequence's end it is n; the answer never exceeds d.
template <int L, class IdxT>
struct Search {
  int64_t lo, hi;  // the answer is in [lo, hi]
  __device__ __forceinline__ int64_t step() const { return (hi - lo + L - 1) / L; }
  // the row at which this lane asks
  __device__ __forceinline__ int64_t place() const {
    return min(lo + ((threadIdx.x & (L - 1)) + 1) * step() - 1, hi - 1);
  }
  __device__ __forceinline__ void narrow(bool past) {
    const unsigned all = __ballot_sync(kFull, lo < hi && past);
    const unsigned found = (all >> (threadIdx.x & 31 & ~(L - 1))) & (L == 32 ? kFull : (1u << (L & 31)) - 1u);
    if (lo >= hi) return;
    const int64_t s = step();
    if (found == 0) {
      lo = hi;
    } else {
      const int64_t first = lo + (__ffs(found) - 1) * s;
      hi = min(first + s - 1, hi - 1);
      lo = s == 1 ? hi : min(first, hi);
    }
  }
};

template <class IdxT>
__device__ __forceinline__ float row_factor(const I8SpmmArgs& a, int64_t r) {
  if (a.mode == kGcn) return __ldg(a.dis + r);
  if (a.mode == kMean) {
    const int64_t deg = rp<IdxT>(a, r + 1) - rp<IdxT>(a, r);
    return deg > 0 ? __fdiv_rn(1.0f, static_cast<float>(deg)) : 0.0f;
  }
  return 1.0f;
}

// The weight of an entry whose column is c.
__device__ __forceinline__ float entry_weight(const I8SpmmArgs& a, int c, int64_t e) {
  float w = __ldg(a.scale + c);
  if (a.dis_col != nullptr) w = __fmul_rn(w, __ldg(a.dis_col + c));
  if (a.ew != nullptr) w = __fmul_rn(w, ld_stream_f32(a.ew + e));
  return w;
}

// L lanes (4, 8, 16 or 32) per share. Entries are taken in chunks of L, one per
// lane, whatever rows they belong to; the next chunk's weights and the columns of the
// one after it are on their way while a chunk is summed, U feature rows in flight.
template <int L, int KIND, class IdxT>
__global__ void __launch_bounds__(kThreads, 4) spmm_i8_kernel(I8SpmmArgs a) {
  constexpr int U = 4;
  const int sub = threadIdx.x & (L - 1);
  const int64_t w = static_cast<int64_t>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;  // share
  // this lane's 16 columns; a lane past the last one reads the first ones and stores nothing
  const int c0 = blockIdx.y * kTileCols + sub * 16;  // f > 512: column tiles
  const bool have = c0 < a.f;
  const int cl = have ? c0 : 0;
  const int8_t* const xl = a.x + cl;
  const uint32_t ldx = static_cast<uint32_t>(a.ldx);
  const int last_row = static_cast<int>(a.n - 1);
  const Rows<IdxT> rows(a);
  if (rows.cut && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    atomicCAS(&g_spmm_i8_status, 0, kSpanOutside);
  }
  // a group past the last share, or past the entries that row_ptr spans, takes an empty one
  const int64_t d0 = w * a.share, d1 = d0 + a.share;
  Search<L, IdxT> begins{0, a.n}, ends{0, a.n};  // both at once: their loads are on their way together
  while (__any_sync(kFull, begins.lo < begins.hi || ends.lo < ends.hi)) {
    const int64_t r0 = begins.place(), r1 = ends.place();
    const int64_t v0 = rows.begin(r0 + 1), v1 = rows.begin(r1 + 1);
    begins.narrow(v0 + r0 + 1 > d0);
    ends.narrow(v1 + r1 + 1 > d1);
  }
  int row = static_cast<int>(begins.lo);
  const int row_end = max(row, static_cast<int>(ends.lo));  // rows [row, row_end) end in this share
  const int64_t e0 = min(d0 - row, rows.span());
  // entries; positions are relative to e0
  const int len = static_cast<int>(max(min(d1 - row_end, rows.span()) - e0, int64_t(0)));
  bool head = row < a.n && rows.begin(row) < e0;            // the first row began in an earlier share
  const bool open = e0 + len > max(e0, rows.begin(row_end));  // the last entries' row ends in a later share
  if (sub == 0 && blockIdx.y == 0 && w < a.shares) {
    // the row that this share begins but does not end: its piece is the tail slot
    a.part_row[w] = open && !(head && row == row_end) ? row_end : -1;
  }
  const IdxT entry = rows.base + static_cast<IdxT>(e0);  // the share's first entry
  const int32_t* const cp = a.col + entry + sub;
  auto load_col = [&](int p) -> int { return p + sub < len ? ld_stream_i32(cp + p) : 0; };
  // past the share: weight 0 on row 0
  auto load_weight = [&](int p, int c) -> float {
    return p + sub < len ? entry_weight(a, c, static_cast<int64_t>(entry) + p + sub) : 0.0f;
  };
  // (past len, so that the row ends behind the loop, where the entries are cut off)
  // (r unsigned: one past the last of 2^31 - 1 rows is no negative place)
  auto load_stop = [&](uint32_t r) -> int {
    return r < static_cast<uint32_t>(row_end)
               ? static_cast<int>(__ldg(static_cast<const IdxT*>(a.row_ptr) + r + 1) - entry)
               : 0x7fffffff;
  };
  auto load_factor = [&](uint32_t r) -> float {
    return r < static_cast<uint32_t>(row_end) ? row_factor<IdxT>(a, r) : 0.0f;
  };
  float* const partl = a.part + 2 * w * a.f + c0;
  const bool vec = (a.f & 7) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
  uint64_t acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0;
  // stores what was summed and starts anew
  auto store = [&](float* dst, float fr) {
    float f[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      unpair(acc[i], f[2 * i], f[2 * i + 1]);
      acc[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = __fmul_rn(f[i], fr);
    if (have) {
      if (vec) {
        store8(dst, f);
        if (c0 + 8 < a.f) store8(dst + 8, f + 8);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (c0 + i < a.f) __stcs(dst + i, f[i]);
        }
      }
    }
  };
  // where the current row and the next one end, and their factors; a row without entries is 0,
  // also where its factor is no number (the GCN factor of degree 0)
  int stop = load_stop(row), stop_nxt = load_stop(row + 1u);
  float factor = min(stop, len) > 0 || head ? load_factor(row) : 0.0f, factor_nxt = load_factor(row + 1u);
  auto finish_row = [&](bool any) {
    // the row's sums, or the piece of a row that began earlier
    store(head ? partl : a.out + static_cast<int64_t>(row) * a.f + c0, head ? 1.0f : (any ? factor : 0.0f));
    head = false;
    ++row;
    stop = stop_nxt;
    factor = factor_nxt;
    stop_nxt = load_stop(row + 1u);
    factor_nxt = load_factor(row + 1u);
  };

  int c_cur = load_col(0);
  float w_cur = load_weight(0, c_cur);
  int c_nxt = load_col(L);
  for (int base = 0; __any_sync(kFull, base < len); base += L) {
    const float w_nxt = load_weight(base + L, c_nxt);
    const int c_far = load_col(base + 2 * L);
#pragma unroll
    for (int j = 0; j < L; j += U) {
      if (L > 8 && !__any_sync(kFull, base + j < len)) break;
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u] = load_row<KIND>(xl, ldx, __shfl_sync(kFull, c_cur, j + u, L), cl, a.f, last_row);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float wt = __shfl_sync(kFull, w_cur, j + u, L);
        for (bool any = true; stop == base + j + u && row < row_end; any = false) finish_row(any);
        const uint64_t ww = pair(wt, wt);
        fma_word(ww, v[u].x, acc[0], acc[1]);
        fma_word(ww, v[u].y, acc[2], acc[3]);
        fma_word(ww, v[u].z, acc[4], acc[5]);
        fma_word(ww, v[u].w, acc[6], acc[7]);
      }
    }
    c_cur = c_nxt;
    w_cur = w_nxt;
    c_nxt = c_far;
  }
  for (bool any = true; row < row_end; any = false) finish_row(any);  // rows that end with the share's last entry
  if (open) store(head ? partl : partl + a.f, 1.0f);  // entries of a row that ends in a later share
}

// One warp per 32 columns of a share whose tail piece begins a row: adds the head
// pieces of the following shares up to the row's end, eight loads in flight.
template <class IdxT>
__global__ void __launch_bounds__(kThreads) spmm_i8_join_kernel(I8SpmmArgs a) {
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (w >= a.shares) return;
  const int64_t row = a.part_row[w];
  const Rows<IdxT> rows(a);
  const int c = blockIdx.y * 32 + (threadIdx.x & 31);
  if (row < 0 || row >= a.n || c >= a.f) return;
  const int64_t end = rows.begin(row + 1);
  const int64_t last = (end + row) / a.share;  // the row's end is item end + row of the merged sequence
  const float* p = a.part + 2 * w * a.f + c;
  float s = p[a.f];
  int64_t k = w + 1;
  for (; k + 8 <= last + 1; k += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = a.part[2 * (k + i) * a.f + c];
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
  }
  for (; k <= last; ++k) s += a.part[2 * k * a.f + c];
  a.out[row * a.f + c] = __fmul_rn(s, row_factor<IdxT>(a, row));
}

__global__ void __launch_bounds__(kThreads) scale_table_kernel(const float* __restrict__ scale,
                                                               const float* __restrict__ dis,
                                                               float* __restrict__ table, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i < n) table[i] = __fmul_rn(scale[i], dis[i]);
}

// GCN: scale[c] * dis[c] is tabulated first where the entries are many, which saves
// one random 32-byte sector per entry; below, the extra launch costs more.
bool use_table(int weighting, int64_t nnz) { return weighting == kGcn && nnz >= (int64_t(1) << 20); }

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

int lanes_for(int64_t f) { return f <= 64 ? 4 : (f <= 128 ? 8 : (f <= 256 ? 16 : 32)); }

// Items (row ends and entries) per share: about one share for each lane group that the
// device holds at once, at least kMinShare so that a share's pieces do not outweigh its
// rows. Measured: two and four shares per group 521 / 568 us against 506 us (a quarter of
// the products-shaped graph, GCN, F = 128, two rows in flight); kMinShare 64 / 32 / 16 on
// the Pubmed-shaped graph 31.8 / 27.4 / 27.3 us.
constexpr int64_t kMinShare = 32;

int64_t share_for(int64_t n, int64_t nnz, int64_t f) {
  const int64_t groups = static_cast<int64_t>(sm_count()) * (1024 / lanes_for(f));
  return std::max<int64_t>(kMinShare, std::min<int64_t>(4096, (n + nnz + groups - 1) / groups));
}

// [tail rows][pieces][table]
size_t workspace_for(int64_t n, int64_t nnz, int64_t f) {
  const int64_t share = share_for(n, nnz, f);
  const int64_t shares = (n + nnz + share - 1) / share;
  return static_cast<size_t>(round_up(shares * 8, 256) + round_up(2 * shares * f * 4, 256) +
                             (use_table(kGcn, nnz) ? round_up(n * 4, 256) : 0));
}

template <int L, class IdxT>
void launch(const I8SpmmArgs& a, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.shares * L + kThreads - 1) / kThreads),
                  static_cast<unsigned>((a.f + kTileCols - 1) / kTileCols));
  if (((reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.ldx)) & 15) != 0) {
    spmm_i8_kernel<L, kBytes, IdxT><<<grid, kThreads, 0, s>>>(a);
  } else if (a.f % 16 != 0) {
    spmm_i8_kernel<L, kRagged, IdxT><<<grid, kThreads, 0, s>>>(a);
  } else {
    spmm_i8_kernel<L, kWhole, IdxT><<<grid, kThreads, 0, s>>>(a);
  }
}

template <class IdxT>
int run(const I8SpmmArgs& a, cudaStream_t s) {
  switch (lanes_for(a.f)) {
    case 4: launch<4, IdxT>(a, s); break;
    case 8: launch<8, IdxT>(a, s); break;
    case 16: launch<16, IdxT>(a, s); break;
    default: launch<32, IdxT>(a, s); break;
  }
  GNN_LAUNCH_CHECK("spmm_i8_kernel launch");
  const dim3 grid(static_cast<unsigned>((a.shares + kWarps - 1) / kWarps), static_cast<unsigned>((a.f + 31) / 32));
  spmm_i8_join_kernel<IdxT><<<grid, kThreads, 0, s>>>(a);
  GNN_LAUNCH_CHECK("spmm_i8_join_kernel launch");
  return GNN_OK;
}

}  // namespace

int spmm_i8_status_read(int reset, int* status) {
  GNN_CUDA_TRY(cudaMemcpyFromSymbol(status, g_spmm_i8_status, sizeof(int)), "read 8-bit aggregation status word");
  if (reset) {
    const int zero = 0;
    GNN_CUDA_TRY(cudaMemcpyToSymbol(g_spmm_i8_status, &zero, sizeof(int)), "reset 8-bit aggregation status word");
  }
  return GNN_OK;
}

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
  GNN_REQUIRE(feat_dim <= 65535LL * 32, GNN_ERR_UNSUPPORTED, "feat_dim too large");
  GNN_REQUIRE(ldx <= 0xffffffffLL, GNN_ERR_UNSUPPORTED, "row stride of x must be below 2^32");
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
  a.mode = weighting;
  a.dis = weighting == GNN_WEIGHT_GCN ? deg_inv_sqrt : nullptr;
  a.dis_col = a.dis;
  a.ew = weighting == GNN_WEIGHT_EDGE ? edge_weight : nullptr;
  a.x = x;
  a.ldx = ldx;
  a.scale = x_scale;
  a.out = out;
  a.n = num_nodes;
  a.nnz = num_edges;
  a.f = static_cast<int>(feat_dim);
  a.share = share_for(num_nodes, num_edges, feat_dim);
  a.shares = (num_nodes + num_edges + a.share - 1) / a.share;
  a.part_row = static_cast<int64_t*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + round_up(a.shares * 8, 256));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (use_table(weighting, num_edges)) {
    float* table = a.part + round_up(2 * a.shares * feat_dim * 4, 256) / 4;
    scale_table_kernel<<<static_cast<unsigned>((num_nodes + kThreads - 1) / kThreads), kThreads, 0, s>>>(
        x_scale, deg_inv_sqrt, table, num_nodes);
    GNN_LAUNCH_CHECK("scale_table_kernel launch");
    a.scale = table;
    a.dis_col = nullptr;
  }
  const int rc = row_ptr_type == GNN_INDEX_INT32 ? run<int32_t>(a, s) : run<int64_t>(a, s);
  if (rc == GNN_OK) clear_error();
  return rc;
}
