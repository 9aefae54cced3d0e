// nsfps_rows.cu -- lookup of feature rows by index, and its gradient.
//
// Forward: out[p] = scale * table[idx[p]], a copy bound by memory: the index,
// the row and the output move once.
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

// Rows a group of lanes copies at once.  Four row loads in flight per lane
// cover the latency of the dependent index -> row -> store chain.
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
      *reinterpret_cast<typename VecOf<VB>::type *>(a.out + (p * a.vecs + j) * VB) = x[u].v;
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

// Where each table row's entries lie in the sorted list: its first and last
// entry write their ends (rows without an entry keep the zeros written before).
__global__ void __launch_bounds__(256)
rows_runs(const SortedList list, uint32_t count, uint32_t rows, uint2 *__restrict__ run) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, n = *list.kept;
  if (i >= n) return;
  const uint32_t key = list.keys[i], b = list.vals[i] / count;
  const uint32_t row = b * rows + key;
  if (i == 0 || list.keys[i - 1] != key || list.vals[i - 1] / count != b) run[row].x = i;
  if (i + 1 == n || list.keys[i + 1] != key || list.vals[i + 1] / count != b) run[row].y = i + 1;
}

// A row with more entries than a tile is summed tile by tile (rows_hot_tiles,
// rows_hot_join): one warp's serial walk would hold up the launch.  64 entries
// are 16 steps of four loads.
constexpr uint32_t kHotTile = 64;

template <class T, int VB>
__device__ __forceinline__ void add_entries(const char *__restrict__ dout,
                                            const uint32_t *__restrict__ vals, uint32_t b,
                                            uint32_t e, uint32_t vecs, uint32_t j,
                                            float (&acc)[Pack<T, VB>::E]) {
  using V = typename VecOf<VB>::type;
  uint32_t i = b;
  for (; i + 4u <= e; i += 4u) {
    Pack<T, VB> x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      x[u].v = *reinterpret_cast<const V *>(dout + ((uint64_t)vals[i + u] * vecs + j) * VB);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < Pack<T, VB>::E; ++k) acc[k] += to_f32(x[u].e[k]);
  }
  for (; i < e; ++i) {
    Pack<T, VB> x;
    x.v = *reinterpret_cast<const V *>(dout + ((uint64_t)vals[i] * vecs + j) * VB);
#pragma unroll
    for (int k = 0; k < Pack<T, VB>::E; ++k) acc[k] += to_f32(x.e[k]);
  }
}

template <class T, int VB>
__device__ __forceinline__ void store_row(char *out, uint64_t r, uint32_t vecs, uint32_t j,
                                          float scale, const float (&acc)[Pack<T, VB>::E]) {
  Pack<T, VB> y;
#pragma unroll
  for (int k = 0; k < Pack<T, VB>::E; ++k) y.e[k] = from_f32<T>(acc[k] * scale);
  *reinterpret_cast<typename VecOf<VB>::type *>(out + (r * vecs + j) * VB) = y.v;
}

// Rows that a group of lanes sums side by side, two entries of each at a time:
// eight loads in flight behind the run -> entry -> row chain.
constexpr int kSumFlight = 4;

// LANES lanes per table row.
template <class T, int VB>
__global__ void __launch_bounds__(256)
rows_sum(const char *__restrict__ dout, const uint32_t *__restrict__ vals,
         const uint2 *__restrict__ run, uint32_t rows, uint32_t vecs, float scale,
         char *__restrict__ out, const int lanes_log2) {
  constexpr int E = Pack<T, VB>::E;
  using V = typename VecOf<VB>::type;
  const uint32_t lanes = 1u << lanes_log2, per_block = 256u >> lanes_log2;
  const uint32_t first = blockIdx.x * (per_block * kSumFlight) + (threadIdx.x >> lanes_log2);
  uint32_t b[kSumFlight], n[kSumFlight], most = 0;
#pragma unroll
  for (int u = 0; u < kSumFlight; ++u) {
    const uint32_t r = first + u * per_block;
    const uint2 x = r < rows ? run[r] : make_uint2(0u, 0u);
    b[u] = x.x;
    n[u] = x.y - x.x > kHotTile ? 0u : x.y - x.x;  // a hot row is written elsewhere
    most = max(most, n[u]);
  }
  for (uint32_t j = threadIdx.x & (lanes - 1u); j < vecs; j += lanes) {
    float acc[kSumFlight][E] = {};
    for (uint32_t i = 0; i < most; i += 2u) {
      uint32_t v[kSumFlight][2];
      Pack<T, VB> x[kSumFlight][2];
#pragma unroll
      for (int u = 0; u < kSumFlight; ++u)
#pragma unroll
        for (int k = 0; k < 2; ++k) v[u][k] = i + k < n[u] ? vals[b[u] + i + k] : 0u;
#pragma unroll
      for (int u = 0; u < kSumFlight; ++u)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (i + k < n[u])
            x[u][k].v = *reinterpret_cast<const V *>(dout + ((uint64_t)v[u][k] * vecs + j) * VB);
#pragma unroll
      for (int u = 0; u < kSumFlight; ++u)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (i + k < n[u])
#pragma unroll
            for (int e = 0; e < E; ++e) acc[u][e] += to_f32(x[u][k].e[e]);
    }
#pragma unroll
    for (int u = 0; u < kSumFlight; ++u) {
      const uint32_t r = first + u * per_block;
      if (r < rows && (n[u] || run[r].x == run[r].y))
        store_row<T, VB>(out, r, vecs, j, scale, acc[u]);
    }
  }
}

// Tiles of the sorted list, one warp each.  A tile meets at most two hot rows,
// that of its first entry and that of its last (any row between them is
// shorter than the tile); slot 0 / 1 of part[] takes their sums over the tile.
struct TileRow {
  uint32_t row, lo, hi;  // table row (all ones: none), its entries
};

__device__ __forceinline__ TileRow row_of_entry(const SortedList &list, const uint2 *run,
                                                uint32_t i, uint32_t count, uint32_t rows) {
  TileRow t;
  t.row = list.vals[i] / count * rows + list.keys[i];
  const uint2 x = run[t.row];
  t.lo = x.x;
  t.hi = x.y;
  if (t.hi - t.lo <= kHotTile) t.row = 0xffffffffu;
  return t;
}

template <class T, int VB>
__global__ void __launch_bounds__(256)
rows_hot_tiles(const char *__restrict__ dout, const SortedList list,
               const uint2 *__restrict__ run, uint32_t count, uint32_t rows, uint32_t vecs,
               float *__restrict__ part) {
  constexpr int E = Pack<T, VB>::E;
  const uint32_t t = blockIdx.x * 8u + (threadIdx.x >> 5), lane = threadIdx.x & 31u;
  const uint32_t n = *list.kept, b = t * kHotTile, e = min(n, b + kHotTile);
  if (b >= n) return;
  const TileRow first = row_of_entry(list, run, b, count, rows);
  const TileRow last = row_of_entry(list, run, e - 1u, count, rows);
  for (int s = 0; s < 2; ++s) {
    const TileRow r = s ? last : first;
    if (r.row == 0xffffffffu || (s && last.row == first.row)) continue;
    for (uint32_t j = lane; j < vecs; j += 32u) {
      float acc[E] = {};
      add_entries<T, VB>(dout, list.vals, max(b, r.lo), min(e, r.hi), vecs, j, acc);
      float *o = part + ((uint64_t)(2u * t + s) * vecs + j) * E;
#pragma unroll
      for (int k = 0; k < E; ++k) o[k] = acc[k];
    }
  }
}

// The hot row that starts in a tile (at most one: it reaches the tile's end)
// adds its tile sums in order: eight warps a share each, then the shares.
template <class T, int VB>
__global__ void __launch_bounds__(256)
rows_hot_join(const SortedList list, const uint2 *__restrict__ run, uint32_t count,
              uint32_t rows, uint32_t vecs, float scale, const float *__restrict__ part,
              char *__restrict__ out) {
  constexpr int E = Pack<T, VB>::E;
  __shared__ float s_acc[8][32][E];
  __shared__ TileRow s_row[8];
  __shared__ uint32_t s_slot[8];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, n = *list.kept;
  if (blockIdx.x * 8u * kHotTile >= n) return;
  {
    const uint32_t t = blockIdx.x * 8u + warp, b = t * kHotTile, e = min(n, b + kHotTile);
    TileRow r{0xffffffffu, 0u, 0u};
    uint32_t slot = 0;
    if (b < n) {
      r = row_of_entry(list, run, e - 1u, count, rows);
      if (r.row != 0xffffffffu && r.lo < b) r.row = 0xffffffffu;
      slot = 2u * t + (r.lo == b ? 0u : 1u);
    }
    if (lane == 0) s_row[warp] = r, s_slot[warp] = slot;
  }
  __syncthreads();
  for (uint32_t i = 0; i < 8u; ++i) {
    const TileRow r = s_row[i];
    if (r.row == 0xffffffffu) continue;
    const uint32_t t = blockIdx.x * 8u + i, last = (r.hi - 1u) / kHotTile;  // tiles t .. last
    const uint32_t per = (last - t + 8u) / 8u;
    const uint32_t wb = min(last + 1u, t + warp * per), we = min(last + 1u, wb + per);
    for (uint32_t j0 = 0; j0 < vecs; j0 += 32u) {
      float acc[E] = {};
      if (j0 + lane < vecs)
#pragma unroll 4
        for (uint32_t x = wb; x < we; ++x) {
          const uint32_t slot = x == t ? s_slot[i] : 2u * x;
          const float *o = part + ((uint64_t)slot * vecs + j0 + lane) * E;
#pragma unroll
          for (int k = 0; k < E; ++k) acc[k] += o[k];
        }
#pragma unroll
      for (int k = 0; k < E; ++k) s_acc[warp][lane][k] = acc[k];
      __syncthreads();
      if (warp == 0 && j0 + lane < vecs) {
        for (int w = 1; w < 8; ++w)
#pragma unroll
          for (int k = 0; k < E; ++k) acc[k] += s_acc[w][lane][k];
        store_row<T, VB>(out, r.row, vecs, j0 + lane, scale, acc);
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
  if (d->batch >= lim || d->rows >= lim || d->count >= lim || d->width >= (1ull << 24) ||
      d->batch * d->rows >= lim || d->batch * d->count >= lim)
    return set_error(NSFPS_ERR_UNSUPPORTED,
                     "batch * rows and batch * count must be below 2^31, width below 2^24");
  if (!std::isfinite(d->scale)) return set_error(NSFPS_ERR_ARG, "scale must be finite");
  return NSFPS_OK;
}

struct RowsGradWork {
  SortScratch sort;
  uint2 *run;
  float *part;
  uint64_t bytes;
};

RowsGradWork carve_rows_grad(const nsfps_rows_desc &d, void *base) {
  RowsGradWork w{};
  WorkCarver c(base);
  const uint32_t n = (uint32_t)(d.batch * d.count);
  w.sort.carve(c, n);
  w.run = c.take<uint2>(d.batch * d.rows);
  w.part = c.take<float>(2 * ceil_div(n, kHotTile) * d.width);
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

struct LaunchRowsSum {
  const char *dout;
  char *out;
  SortedList list;
  const uint2 *run;
  float *part;
  uint32_t n, count, all_rows, rows, vecs;
  float scale;
  int lanes_log2;
  cudaStream_t st;
  template <class T, int VB>
  cudaError_t operator()() const {
    rows_sum<T, VB><<<(uint32_t)ceil_div(all_rows, (256u >> lanes_log2) * kSumFlight), 256, 0,
                      st>>>(dout, list.vals, run, all_rows, vecs, scale, out, lanes_log2);
    if (n > kHotTile) {  // fewer entries make no hot row
      const uint32_t grid = (uint32_t)ceil_div(n, 8u * kHotTile);
      rows_hot_tiles<T, VB><<<grid, 256, 0, st>>>(dout, list, run, count, rows, vecs, part);
      rows_hot_join<T, VB><<<grid, 256, 0, st>>>(list, run, count, rows, vecs, scale, part, out);
    }
    return cudaGetLastError();
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
  NSFPS_FEATURE_CUDA(cudaMemsetAsync(w.run, 0, (uint64_t)rows * sizeof(uint2), st));
  rows_runs<<<(uint32_t)ceil_div(n, 256), 256, 0, st>>>(list, (uint32_t)d.count, (uint32_t)d.rows,
                                                        w.run);
  NSFPS_FEATURE_CUDA(cudaGetLastError());
  const int vb = vec_bytes((uint64_t)d_dout | (uint64_t)d_dtable | d.width * elem, elem);
  const uint32_t vecs = (uint32_t)(d.width * elem / vb);
  NSFPS_FEATURE_CUDA(with_vec(
      d.dtype, vb,
      LaunchRowsSum{(const char *)d_dout, (char *)d_dtable, list, w.run, w.part, n,
                    (uint32_t)d.count, rows, (uint32_t)d.rows, vecs, d.scale,
                    lanes_log2_for(vecs), st}));
  return NSFPS_OK;
}

}  // extern "C"
