// nsfps_rows.cu -- lookup of feature rows by index, and its gradient.
//
// Forward: out[p] = scale * table[idx[p]], a copy bound by memory: the index,
// the row and the output move once.
//
// Gradient: dtable[n] = scale * sum of dout[p] over idx[p] == n.  The entries
// (n, p) are sorted by n with the engine's stable radix sort, so each row's
// entries are consecutive and ascending in p, and every row is written once
// by one owner: no atomics, the same bits every time.
#include <algorithm>
#include <cmath>

#include "nsfps_feature.cuh"

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

// Sort keys: the table row over all batch entries; `none` (batch * rows) for
// entries without a row, which sort behind every row.
__global__ void __launch_bounds__(256)
rows_keys(const int64_t *__restrict__ idx, uint32_t total, uint32_t count, uint32_t rows,
          uint32_t none, uint32_t *__restrict__ keys, uint32_t *__restrict__ vals) {
  const uint32_t p = blockIdx.x * 256u + threadIdx.x;
  if (p >= total) return;
  const int64_t i = idx[p];
  keys[p] = (i >= 0 && i < (int64_t)rows) ? (p / count) * rows + (uint32_t)i : none;
  vals[p] = p;
}

// start[r] = first sorted entry of row r; start[rows] = entries with a row.
__global__ void __launch_bounds__(256)
rows_starts(const uint32_t *__restrict__ keys, uint32_t n, uint32_t rows,
            uint32_t *__restrict__ start) {
  const uint32_t r = blockIdx.x * 256u + threadIdx.x;
  if (r <= rows) start[r] = lower_bound(keys, n, r);
}

// A row with more entries than this is summed in tiles of the sorted list by
// rows_hot_tiles / rows_hot_join: one warp's serial walk would otherwise hold
// up the launch (a row that every entry names).
constexpr uint32_t kHotTile = 256;

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

// LANES lanes per table row.
template <class T, int VB>
__global__ void __launch_bounds__(256)
rows_sum(const char *__restrict__ dout, const uint32_t *__restrict__ vals,
         const uint32_t *__restrict__ start, uint32_t rows, uint32_t vecs, float scale,
         char *__restrict__ out, const int lanes_log2) {
  const uint32_t lanes = 1u << lanes_log2;
  const uint32_t r = blockIdx.x * (256u >> lanes_log2) + (threadIdx.x >> lanes_log2);
  if (r >= rows) return;
  const uint32_t b = start[r], e = start[r + 1];
  if (e - b > kHotTile) return;
  for (uint32_t j = threadIdx.x & (lanes - 1u); j < vecs; j += lanes) {
    float acc[Pack<T, VB>::E] = {};
    add_entries<T, VB>(dout, vals, b, e, vecs, j, acc);
    store_row<T, VB>(out, r, vecs, j, scale, acc);
  }
}

// Tile t: sorted entries [t * kHotTile, ...).  It meets at most two hot rows,
// that of its first entry and that of its last (any row between them is
// shorter than the tile); slot 0 / 1 of part[] takes their sums over the tile.
template <class T, int VB>
__global__ void __launch_bounds__(256)
rows_hot_tiles(const char *__restrict__ dout, const uint32_t *__restrict__ keys,
               const uint32_t *__restrict__ vals, const uint32_t *__restrict__ start,
               uint32_t n, uint32_t none, uint32_t vecs, float *__restrict__ part) {
  constexpr int E = Pack<T, VB>::E;
  __shared__ float s_acc[8][32][E];
  const uint32_t b = blockIdx.x * kHotTile, e = min(n, b + kHotTile);
  const uint32_t r0 = keys[b], r1 = keys[e - 1];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  for (int s = 0; s < 2; ++s) {
    const uint32_t r = s ? r1 : r0;
    if (r == none || (s && r1 == r0)) continue;
    const uint32_t rb = start[r], re = start[r + 1];
    if (re - rb <= kHotTile) continue;
    const uint32_t lo = max(b, rb), hi = min(e, re);
    const uint32_t per = (hi - lo + 7u) / 8u;
    const uint32_t wb = min(hi, lo + warp * per), we = min(hi, wb + per);
    for (uint32_t j0 = 0; j0 < vecs; j0 += 32u) {
      float acc[E] = {};
      if (j0 + lane < vecs) add_entries<T, VB>(dout, vals, wb, we, vecs, j0 + lane, acc);
#pragma unroll
      for (int k = 0; k < E; ++k) s_acc[warp][lane][k] = acc[k];
      __syncthreads();
      if (warp == 0 && j0 + lane < vecs) {
        for (int w = 1; w < 8; ++w)
#pragma unroll
          for (int k = 0; k < E; ++k) acc[k] += s_acc[w][lane][k];
        float *o = part + ((uint64_t)(2u * blockIdx.x + s) * vecs + j0 + lane) * E;
#pragma unroll
        for (int k = 0; k < E; ++k) o[k] = acc[k];
      }
      __syncthreads();
    }
  }
}

// The tile in which a hot row starts adds that row's tile sums in order.
template <class T, int VB>
__global__ void __launch_bounds__(256)
rows_hot_join(const uint32_t *__restrict__ keys, const uint32_t *__restrict__ start, uint32_t n,
              uint32_t none, uint32_t vecs, float scale, const float *__restrict__ part,
              char *__restrict__ out) {
  constexpr int E = Pack<T, VB>::E;
  __shared__ float s_acc[8][32][E];
  const uint32_t t = blockIdx.x, b = t * kHotTile, e = min(n, b + kHotTile);
  const uint32_t r = keys[e - 1];
  if (r == none) return;
  const uint32_t rb = start[r], re = start[r + 1];
  if (re - rb <= kHotTile || rb < b) return;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t last = (re - 1u) / kHotTile;         // tiles t .. last
  const uint32_t s0 = keys[b] == r ? 0u : 1u;         // its slot in tile t
  const uint32_t per = (last - t + 8u) / 8u;
  const uint32_t wb = t + warp * per, we = min(last + 1u, wb + per);
  for (uint32_t j0 = 0; j0 < vecs; j0 += 32u) {
    float acc[E] = {};
    if (j0 + lane < vecs)
      for (uint32_t i = wb; i < we; ++i) {
        const uint32_t slot = 2u * i + (i == t ? s0 : 0u);
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
      store_row<T, VB>(out, r, vecs, j0 + lane, scale, acc);
    }
    __syncthreads();
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
  uint32_t *start;
  float *part;
  uint64_t bytes;
};

RowsGradWork carve_rows_grad(const nsfps_rows_desc &d, void *base) {
  RowsGradWork w{};
  WorkCarver c(base);
  const uint32_t n = (uint32_t)(d.batch * d.count);
  w.sort.carve(c, n);
  w.start = c.take<uint32_t>(d.batch * d.rows + 1);
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
  const uint32_t *keys, *vals, *start;
  float *part;
  uint32_t n, rows, vecs;
  float scale;
  int lanes_log2;
  cudaStream_t st;
  template <class T, int VB>
  cudaError_t operator()() const {
    rows_sum<T, VB><<<(uint32_t)ceil_div(rows, 256u >> lanes_log2), 256, 0, st>>>(
        dout, vals, start, rows, vecs, scale, out, lanes_log2);
    if (n > kHotTile) {  // fewer entries make no hot row
      const uint32_t tiles = (uint32_t)ceil_div(n, kHotTile);
      rows_hot_tiles<T, VB><<<tiles, 256, 0, st>>>(dout, keys, vals, start, n, rows, vecs, part);
      rows_hot_join<T, VB><<<tiles, 256, 0, st>>>(keys, start, n, rows, vecs, scale, part, out);
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
  rows_keys<<<(uint32_t)ceil_div(n, 256), 256, 0, st>>>(d_idx, n, (uint32_t)d.count,
                                                        (uint32_t)d.rows, rows, w.sort.keys0,
                                                        w.sort.vals0);
  NSFPS_FEATURE_CUDA(cudaGetLastError());
  uint32_t *keys = w.sort.keys0, *vals = w.sort.vals0, launches = 0;
  NSFPS_FEATURE_CUDA(run_sort_pairs(&keys, &vals, w.sort.keys1, w.sort.vals1, n, rows,
                                    w.sort.hist, w.sort.partial, st, launches));
  rows_starts<<<(uint32_t)ceil_div((uint64_t)rows + 1, 256), 256, 0, st>>>(keys, n, rows, w.start);
  NSFPS_FEATURE_CUDA(cudaGetLastError());
  const int vb = vec_bytes((uint64_t)d_dout | (uint64_t)d_dtable | d.width * elem, elem);
  const uint32_t vecs = (uint32_t)(d.width * elem / vb);
  NSFPS_FEATURE_CUDA(with_vec(
      d.dtype, vb,
      LaunchRowsSum{(const char *)d_dout, (char *)d_dtable, keys, vals, w.start, w.part, n, rows,
                    vecs, d.scale, lanes_log2_for(vecs), st}));
  return NSFPS_OK;
}

}  // extern "C"
