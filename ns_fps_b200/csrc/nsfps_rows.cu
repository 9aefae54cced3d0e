// nsfps_rows.cu -- lookup of feature rows by index, and its gradient.
//
// Forward: out[p] = scale * table[idx[p]], a copy bound by memory: the index,
// the row and the output move once.  2^21 rows of 128 bytes out of 32 tables
// take 73 us, 352 MB at 4.8 TB/s.
//
// Gradient: dtable[n] = scale * sum of dout[p] over idx[p] == n.  The entries
// are sorted by index, stably, so a row's entries are consecutive and ascending
// in p, and every row is written once by one owner: no atomics, the same bits
// every time.  In a batch the index alone is the key: positions ascend with the
// batch entry, so the entries of (n, b) are consecutive too, and the sort needs
// the bits of N and not those of B * N.
#include <algorithm>
#include <cmath>

#include "nsfps_feature.cuh"
#include "nsfps_sort.cuh"

namespace nsfps {
namespace {

// A vector of VB bytes.
template <int VB> struct VecOf;
template <> struct VecOf<16> { using type = uint4; };
template <> struct VecOf<8> { using type = uint2; };
template <> struct VecOf<4> { using type = uint32_t; };
template <> struct VecOf<2> { using type = uint16_t; };

template <class T, int VB>
struct Pack {
  static constexpr int E = VB / (int)sizeof(T);
  union {
    typename VecOf<VB>::type v;
    T e[E];
  };
  __device__ Pack() {}
};

struct RowsArgs {
  const char *table;       // forward: table; gradient: dout
  char *out;
  const int64_t *idx;
  uint64_t batch_stride, row_stride;  // bytes
  uint32_t rows, count, batch;
  uint32_t vecs;           // vectors per row
  uint32_t total;          // batch * count
  float scale;
};

// Rows a group of lanes copies at once: loads in flight per lane behind the
// index -> row -> store chain.  2 and 4 are level (74 and 73 us for 352 MB), 8
// takes 80.
constexpr int kRowsFlight = 4;

// LANES lanes (a power of two up to 32) copy one row, 32 / LANES rows per warp
// side by side, kRowsFlight such steps at once.
template <class T, int VB>
__global__ void __launch_bounds__(256)
gather_rows_kernel(const RowsArgs a, const int lanes_log2) {
  const uint32_t lanes = 1u << lanes_log2;
  const uint32_t per_block = 256u >> lanes_log2;
  const uint32_t sub = threadIdx.x & (lanes - 1u);
  const uint32_t first = blockIdx.x * (per_block * kRowsFlight) + (threadIdx.x >> lanes_log2);
  const char *src[kRowsFlight];
  bool live[kRowsFlight], bad[kRowsFlight];
#pragma unroll
  for (int u = 0; u < kRowsFlight; ++u) {
    const uint32_t p = first + u * per_block;
    live[u] = p < a.total;
    const int64_t i = live[u] ? a.idx[p] : -1;
    bad[u] = i >= (int64_t)a.rows;
    src[u] = (i < 0 || bad[u]) ? nullptr
                               : a.table + (uint64_t)(p / a.count) * a.batch_stride +
                                     (uint64_t)i * a.row_stride;
  }
  for (uint32_t j = sub; j < a.vecs; j += lanes) {
    Pack<T, VB> x[kRowsFlight];
#pragma unroll
    for (int u = 0; u < kRowsFlight; ++u) {
      if (src[u]) {
        x[u].v = *reinterpret_cast<const typename VecOf<VB>::type *>(src[u] + (uint64_t)j * VB);
      } else {
#pragma unroll
        for (int e = 0; e < Pack<T, VB>::E; ++e)
          x[u].e[e] = from_f32<T>(bad[u] ? __int_as_float(0x7fc00000) : 0.0f);
      }
    }
#pragma unroll
    for (int u = 0; u < kRowsFlight; ++u) {
      if (!live[u]) continue;
      if (a.scale != 1.0f) {
#pragma unroll
        for (int e = 0; e < Pack<T, VB>::E; ++e)
          x[u].e[e] = from_f32<T>(to_f32(x[u].e[e]) * a.scale);
      }
      const uint64_t p = first + u * per_block;
      // written once and not read here: kept out of the way of the table's rows
      __stcs(reinterpret_cast<typename VecOf<VB>::type *>(a.out + (p * a.vecs + j) * VB), x[u].v);
    }
  }
}

// Sort keys: the indices; `rows` for an entry without a row, which is dropped.
struct IndexKeys {
  const int64_t *idx;
  uint32_t rows;
  static constexpr bool kFirst = true;
  __device__ __forceinline__ uint32_t count(uint32_t n) const { return n; }
  __device__ __forceinline__ uint32_t key(uint32_t i) const {
    const int64_t v = idx[i];
    return v >= 0 && v < (int64_t)rows ? (uint32_t)v : rows;
  }
  __device__ __forceinline__ uint32_t value(uint32_t i) const { return i; }
};

// The sum walks the sorted list in tiles of kWalk entries, one group of lanes
// each: whatever the rows' lengths, a group has the same work, and its loads
// depend on the list alone, eight in flight (one group per table row waited for
// run -> entry -> row: 123 us for 2^20 entries of 192 bytes; this takes 87, 3.5
// TB/s of rows read out of order and written).  A row inside the
// tile is written by it.  Of a row that the tile's border cuts, the tile leaves
// a partial sum: slot 0 for a row that began before the tile, slot 1 for one
// that begins in it and goes on.  rows_join adds those in order.
constexpr uint32_t kWalk = 32;
constexpr int kWalkFlight = 8;

// Table row of a sorted entry.
__device__ __forceinline__ uint32_t entry_row(const SortedList &list, uint32_t i, uint32_t count,
                                              uint32_t rows) {
  return list.vals[i] / count * rows + list.keys[i];
}

template <class T, int VB>
__device__ __forceinline__ void store_row(char *out, uint64_t r, uint32_t vecs, uint32_t j,
                                          float scale, const float (&acc)[Pack<T, VB>::E]) {
  Pack<T, VB> y;
#pragma unroll
  for (int k = 0; k < Pack<T, VB>::E; ++k) y.e[k] = from_f32<T>(acc[k] * scale);
  *reinterpret_cast<typename VecOf<VB>::type *>(out + (r * vecs + j) * VB) = y.v;
}

struct WalkArgs {
  const char *dout;
  char *out;
  SortedList list;
  float *part;      // [2 * tile + slot][width]
  uint32_t count, rows, vecs;
  float scale;
  int lanes_log2;   // 4 or 5: 16 or 32 lanes per tile, one vector each
};

// grid.y: runs of 1 << lanes_log2 vectors of the rows.
template <class T, int VB>
__global__ void __launch_bounds__(256)
rows_walk(const WalkArgs a) {
  after_previous();
  constexpr int E = Pack<T, VB>::E;
  using V = typename VecOf<VB>::type;
  const uint32_t lanes = 1u << a.lanes_log2, sub = threadIdx.x & (lanes - 1u);
  const uint32_t tile = blockIdx.x * (256u >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2);
  const uint32_t n = *a.list.kept, b = tile * kWalk;
  const uint32_t warp_tile = blockIdx.x * (256u >> a.lanes_log2) +
                             ((threadIdx.x & ~31u) >> a.lanes_log2);
  if (warp_tile * kWalk >= n) return;  // the whole warp
  const uint32_t m = b < n ? min(kWalk, n - b) : 0u;
  const uint32_t j = blockIdx.y * lanes + sub;
  const bool mine = j < a.vecs;
  // the tile's entries over its lanes: two per lane of 16, one per lane of 32
  uint32_t val[2], row[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t e = sub + i * lanes;
    val[i] = row[i] = 0xffffffffu;
    if (e < m) {
      val[i] = a.list.vals[b + e];
      row[i] = val[i] / a.count * a.rows + a.list.keys[b + e];
    }
  }
  const uint32_t before = m && b ? entry_row(a.list, b - 1u, a.count, a.rows) : 0xffffffffu;
  const uint32_t after = b + m < n && m ? entry_row(a.list, b + m, a.count, a.rows) : 0xffffffffu;
  uint32_t cur = __shfl_sync(0xffffffffu, row[0], 0, (int)lanes);
  bool begun = m && cur == before;  // the current row began in an earlier tile
  float acc[E] = {};
  auto flush = [&](bool goes_on) {
    if (!mine) return;
    if (begun || goes_on) {
      float *o = a.part + ((uint64_t)(2u * tile + (begun ? 0u : 1u)) * a.vecs + j) * E;
#pragma unroll
      for (int k = 0; k < E; ++k) o[k] = acc[k];
    } else {
      store_row<T, VB>(a.out, cur, a.vecs, j, a.scale, acc);
    }
  };
#pragma unroll 1
  for (uint32_t i = 0; i < kWalk; i += kWalkFlight) {
    uint32_t r[kWalkFlight];
    Pack<T, VB> x[kWalkFlight];
#pragma unroll
    for (int u = 0; u < kWalkFlight; ++u) {
      const uint32_t e = i + u;
      const uint32_t v0 = __shfl_sync(0xffffffffu, val[0], e & (lanes - 1u), (int)lanes);
      const uint32_t v1 = __shfl_sync(0xffffffffu, val[1], e & (lanes - 1u), (int)lanes);
      const uint32_t r0 = __shfl_sync(0xffffffffu, row[0], e & (lanes - 1u), (int)lanes);
      const uint32_t r1 = __shfl_sync(0xffffffffu, row[1], e & (lanes - 1u), (int)lanes);
      const uint32_t v = e < lanes ? v0 : v1;
      r[u] = e < lanes ? r0 : r1;
      if (e < m && mine)
        x[u].v = __ldcs(reinterpret_cast<const V *>(a.dout + ((uint64_t)v * a.vecs + j) * VB));
    }
#pragma unroll
    for (int u = 0; u < kWalkFlight; ++u) {
      if (i + u >= m) continue;
      if (r[u] != cur) {
        flush(false);
        cur = r[u];
        begun = false;
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] = 0.f;
      }
      if (mine)
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] += to_f32(x[u].e[k]);
    }
  }
  if (m) flush(cur == after);
}

// One warp per tile: the row that begins in it and goes on.  A long chain of
// tiles (a row that thousands of entries name) is shared by the CTA's warps.
constexpr uint32_t kLongChain = 32;

template <class T, int VB>
__global__ void __launch_bounds__(256)
rows_join(const WalkArgs a) {
  after_previous();
  constexpr int E = Pack<T, VB>::E;
  __shared__ float s_acc[8][32][E];
  __shared__ uint32_t s_row[8], s_len[8];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t n = *a.list.kept, t = blockIdx.x * 8u + warp, e = (t + 1u) * kWalk;
  if (blockIdx.x * 8u * kWalk >= n) return;
  uint32_t row = 0xffffffffu, len = 0;  // tiles behind t that the row reaches
  if (e < n) {
    const uint32_t r = entry_row(a.list, e - 1u, a.count, a.rows);
    const uint32_t head = t ? entry_row(a.list, t * kWalk - 1u, a.count, a.rows) : 0xffffffffu;
    if (r == entry_row(a.list, e, a.count, a.rows) && r != head) {
      row = r;
      // tile t + 1 + i holds a part while its first entry is the row's
      for (;; len += 32u) {
        const uint64_t first = ((uint64_t)t + 1u + len + lane) * kWalk;
        const bool in = first < n && entry_row(a.list, (uint32_t)first, a.count, a.rows) == r;
        const uint32_t out = ~__ballot_sync(0xffffffffu, in);
        if (out) {
          len += __ffs(out) - 1;
          break;
        }
      }
    }
  }
  if (row != 0xffffffffu && len <= kLongChain) {
    for (uint32_t j = lane; j < a.vecs; j += 32u) {
      float acc[E];
      const float *o = a.part + ((uint64_t)(2u * t + 1u) * a.vecs + j) * E;
#pragma unroll
      for (int k = 0; k < E; ++k) acc[k] = o[k];
#pragma unroll 4
      for (uint32_t i = 1; i <= len; ++i)
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] += (o + (uint64_t)(2u * i - 1u) * a.vecs * E)[k];
      store_row<T, VB>(a.out, row, a.vecs, j, a.scale, acc);
    }
    row = 0xffffffffu;
  }
  if (lane == 0) s_row[warp] = row, s_len[warp] = len;
  __syncthreads();
  for (uint32_t c = 0; c < 8u; ++c) {
    if (s_row[c] == 0xffffffffu) continue;
    const uint32_t tc = blockIdx.x * 8u + c, per = (s_len[c] + 7u) / 8u;
    const uint32_t i0 = 1u + warp * per, i1 = min(s_len[c] + 1u, i0 + per);
    for (uint32_t j0 = 0; j0 < a.vecs; j0 += 32u) {
      const uint32_t j = j0 + lane;
      float acc[E] = {};
      if (j < a.vecs) {
        const float *o = a.part + ((uint64_t)(2u * tc + 1u) * a.vecs + j) * E;
        if (warp == 0)
#pragma unroll
          for (int k = 0; k < E; ++k) acc[k] = o[k];
#pragma unroll 8
        for (uint32_t i = i0; i < i1; ++i)
#pragma unroll
          for (int k = 0; k < E; ++k) acc[k] += (o + (uint64_t)(2u * i - 1u) * a.vecs * E)[k];
      }
#pragma unroll
      for (int k = 0; k < E; ++k) s_acc[warp][lane][k] = acc[k];
      __syncthreads();
      if (warp == 0 && j < a.vecs) {
        for (int w = 1; w < 8; ++w)
#pragma unroll
          for (int k = 0; k < E; ++k) acc[k] += s_acc[w][lane][k];
        store_row<T, VB>(a.out, s_row[c], a.vecs, j, a.scale, acc);
      }
      __syncthreads();
    }
  }
}

// Widest vector (up to 16 bytes) that divides every one of the given byte
// counts and addresses.
int vec_bytes(uint64_t all_or, int elem) {
  int v = 16;
  while (v > elem && (all_or & (uint64_t)(v - 1))) v >>= 1;
  return v;
}

int lanes_log2_for(uint32_t vecs) {
  int l = 0;
  while (l < 5 && (1u << l) < vecs) ++l;
  return l;
}

int check_rows(const nsfps_rows_desc *d) {
  if (!d) return set_error(NSFPS_ERR_ARG, "desc is NULL");
  if (d->dtype != NSFPS_F32 && d->dtype != NSFPS_F16 && d->dtype != NSFPS_BF16)
    return set_error(NSFPS_ERR_ARG, "dtype must be float32, float16 or bfloat16");
  const uint64_t lim = 1ull << 31;
  if (d->batch >= lim || d->rows >= lim || d->count >= lim || d->width >= (1ull << 20) ||
      d->batch * d->rows >= lim || d->batch * d->count >= lim)
    return set_error(NSFPS_ERR_UNSUPPORTED,
                     "batch * rows and batch * count must be below 2^31, width below 2^20");
  if (!std::isfinite(d->scale)) return set_error(NSFPS_ERR_ARG, "scale must be finite");
  return NSFPS_OK;
}

struct RowsGradWork {
  SortScratch sort;
  float *part;
  uint64_t bytes;
};

RowsGradWork carve_rows_grad(const nsfps_rows_desc &d, void *base) {
  RowsGradWork w{};
  WorkCarver c(base);
  const uint32_t n = (uint32_t)(d.batch * d.count);
  w.sort.carve(c, n);
  w.part = c.take<float>(2 * ceil_div(n, kWalk) * d.width);
  w.bytes = c.off;
  return w;
}

// Calls f with the element type and vector width as types.
template <class F>
cudaError_t with_vec(int dtype, int vb, F &&f) {
#define NSFPS_ROWS_CASE(T, VB) return f.template operator()<T, VB>()
  if (dtype == NSFPS_F32) {
    if (vb == 16) NSFPS_ROWS_CASE(float, 16);
    if (vb == 8) NSFPS_ROWS_CASE(float, 8);
    NSFPS_ROWS_CASE(float, 4);
  }
  if (dtype == NSFPS_F16) {
    if (vb == 16) NSFPS_ROWS_CASE(__half, 16);
    if (vb == 8) NSFPS_ROWS_CASE(__half, 8);
    if (vb == 4) NSFPS_ROWS_CASE(__half, 4);
    NSFPS_ROWS_CASE(__half, 2);
  }
  if (vb == 16) NSFPS_ROWS_CASE(__nv_bfloat16, 16);
  if (vb == 8) NSFPS_ROWS_CASE(__nv_bfloat16, 8);
  if (vb == 4) NSFPS_ROWS_CASE(__nv_bfloat16, 4);
  NSFPS_ROWS_CASE(__nv_bfloat16, 2);
#undef NSFPS_ROWS_CASE
}

struct LaunchGather {
  RowsArgs a;
  int lanes_log2;
  cudaStream_t st;
  template <class T, int VB>
  cudaError_t operator()() const {
    const uint64_t per_block = (uint64_t)(256u >> lanes_log2) * kRowsFlight;
    gather_rows_kernel<T, VB><<<(uint32_t)ceil_div(a.total, per_block), 256, 0, st>>>(a, lanes_log2);
    return cudaGetLastError();
  }
};

struct LaunchWalk {
  WalkArgs a;
  uint32_t n;
  cudaStream_t st;
  template <class T, int VB>
  cudaError_t operator()() const {
    const uint32_t tiles = (uint32_t)ceil_div(n, kWalk);
    const dim3 grid((uint32_t)ceil_div(tiles, 256u >> a.lanes_log2),
                    (uint32_t)ceil_div(a.vecs, 1u << a.lanes_log2));
    const cudaError_t err = launch_next(rows_walk<T, VB>, grid, 256, 0, st, a);
    if (err || n <= kWalk) return err;
    return launch_next(rows_join<T, VB>, (uint32_t)ceil_div(tiles, 8), 256, 0, st, a);
  }
};

}  // namespace
}  // namespace nsfps

using namespace nsfps;

extern "C" {

int nsfps_gather_rows_device(const nsfps_rows_desc *desc, const void *d_table,
                             const int64_t *d_idx, void *d_out, void *stream) {
  clear_error();
  int rc = check_rows(desc);
  if (rc) return rc;
  const nsfps_rows_desc &d = *desc;
  const uint64_t total = d.batch * d.count;
  if (total == 0 || d.width == 0) return NSFPS_OK;
  if (!d_idx || !d_out || (d.rows && !d_table)) return set_error(NSFPS_ERR_ARG, "NULL argument");
  if (d.batch_stride < 0 || d.row_stride < 0)
    return set_error(NSFPS_ERR_ARG, "strides must not be negative");
  const int elem = d.dtype == NSFPS_F32 ? 4 : 2;
  if (((uint64_t)d_table | (uint64_t)d_out) % elem || (uint64_t)d_idx % 8)
    return set_error(NSFPS_ERR_ARG, "a pointer is not aligned to its elements");
  RowsArgs a{};
  a.table = (const char *)d_table;
  a.out = (char *)d_out;
  a.idx = d_idx;
  a.batch_stride = (uint64_t)d.batch_stride * elem;
  a.row_stride = (uint64_t)d.row_stride * elem;
  a.rows = (uint32_t)d.rows;
  a.count = (uint32_t)d.count;
  a.batch = (uint32_t)d.batch;
  a.total = (uint32_t)total;
  a.scale = d.scale;
  const int vb = vec_bytes((uint64_t)d_table | (uint64_t)d_out | a.batch_stride | a.row_stride |
                               d.width * elem, elem);
  a.vecs = (uint32_t)(d.width * elem / vb);
  NSFPS_FEATURE_CUDA(with_vec(d.dtype, vb,
                              LaunchGather{a, lanes_log2_for(a.vecs), (cudaStream_t)stream}));
  return NSFPS_OK;
}

int nsfps_gather_rows_grad_workspace(const nsfps_rows_desc *desc, uint64_t *bytes) {
  clear_error();
  int rc = check_rows(desc);
  if (rc) return rc;
  if (!bytes) return set_error(NSFPS_ERR_ARG, "bytes is NULL");
  *bytes = carve_rows_grad(*desc, nullptr).bytes;
  return NSFPS_OK;
}

int nsfps_gather_rows_grad_device(const nsfps_rows_desc *desc, const void *d_dout,
                                  const int64_t *d_idx, void *d_dtable, void *d_work,
                                  uint64_t work_bytes, void *stream) {
  clear_error();
  int rc = check_rows(desc);
  if (rc) return rc;
  const nsfps_rows_desc &d = *desc;
  const uint32_t rows = (uint32_t)(d.batch * d.rows), n = (uint32_t)(d.batch * d.count);
  if (rows == 0 || d.width == 0) return NSFPS_OK;
  const int elem = d.dtype == NSFPS_F32 ? 4 : 2;
  if (!d_dtable || (n && (!d_dout || !d_idx))) return set_error(NSFPS_ERR_ARG, "NULL argument");
  if (((uint64_t)d_dout | (uint64_t)d_dtable) % elem || (uint64_t)d_idx % 8)
    return set_error(NSFPS_ERR_ARG, "a pointer is not aligned to its elements");
  cudaStream_t st = (cudaStream_t)stream;
  if (n == 0) {
    NSFPS_FEATURE_CUDA(cudaMemsetAsync(d_dtable, 0, (uint64_t)rows * d.width * elem, st));
    return NSFPS_OK;
  }
  if (!d_work || (uint64_t)d_work % 256)
    return set_error(NSFPS_ERR_ARG, "d_work must be 256-byte aligned");
  const RowsGradWork w = carve_rows_grad(d, d_work);
  if (work_bytes < w.bytes)
    return set_error(NSFPS_ERR_ARG, "d_work holds %llu bytes, %llu are needed",
                     (unsigned long long)work_bytes, (unsigned long long)w.bytes);
  SortedList list;
  NSFPS_FEATURE_CUDA(run_sort(IndexKeys{d_idx, (uint32_t)d.rows}, n, (uint32_t)d.rows, w.sort,
                              &list, st));
  // Zeros everywhere first: the memset writes a table of 100 MB in 16 us;
  // marking the rows that entries name and clearing the others took 25.
  NSFPS_FEATURE_CUDA(cudaMemsetAsync(d_dtable, 0, (uint64_t)rows * d.width * elem, st));
  const int vb = vec_bytes((uint64_t)d_dout | (uint64_t)d_dtable | d.width * elem, elem);
  WalkArgs a{};
  a.dout = (const char *)d_dout;
  a.out = (char *)d_dtable;
  a.list = list;
  a.part = w.part;
  a.count = (uint32_t)d.count;
  a.rows = (uint32_t)d.rows;
  a.vecs = (uint32_t)(d.width * elem / vb);
  a.scale = d.scale;
  a.lanes_log2 = a.vecs <= 16 ? 4 : 5;
  NSFPS_FEATURE_CUDA(with_vec(d.dtype, vb, LaunchWalk{a, n, st}));
  return NSFPS_OK;
}

}  // extern "C"
