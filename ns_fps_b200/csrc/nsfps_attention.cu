// nsfps_attention.cu -- attention over the blocks of keys chosen for each
// query, and its gradient.
#include <algorithm>
#include <cmath>

#include "nsfps_feature.cuh"

namespace nsfps {
namespace {

constexpr uint32_t kFullMask = 0xffffffffu;

struct AttnArgs {
  const void *q, *k, *v, *dout;
  const void *out_in;
  void *out, *dq, *dk, *dv;
  float *lse;              // forward: may be null
  const float *lse_in;
  const int64_t *blocks;
  const int32_t *lengths;  // or null
  uint32_t B, M, N, H, G, D, block_log2, top, nb;
  int64_t qs[3], ks[3], vs[3];
  float scale;
};

__device__ __forceinline__ uint32_t cloud_length(const int32_t *lengths, uint32_t b, uint32_t n) {
  return lengths ? (uint32_t)min(max(lengths[b], 0), (int)n) : n;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFullMask, x, o);
  return x;
}

// One warp per (b, m, h); lane l holds elements l, l + 32, ...
template <class T>
__global__ void __launch_bounds__(256)
attend_forward(const AttnArgs a) {
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t w = (uint64_t)blockIdx.x * 8u + (threadIdx.x >> 5);
  if (w >= (uint64_t)a.B * a.M * a.H) return;
  const uint32_t h = w % a.H;
  const uint64_t bm = w / a.H;
  const uint32_t m = bm % a.M, b = bm / a.M, g = h / (a.H / a.G);
  const T *q = (const T *)a.q + b * a.qs[0] + m * a.qs[1] + h * a.qs[2];
  const T *k = (const T *)a.k + b * a.ks[0] + g * a.ks[2];
  const T *v = (const T *)a.v + b * a.vs[0] + g * a.vs[2];
  const int64_t *list = a.blocks + bm * a.top;
  const uint32_t len = cloud_length(a.lengths, b, a.N);
  float qf[4], acc[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) qf[i] = lane + 32 * i < a.D ? to_f32(q[lane + 32 * i]) * a.scale : 0.f;
  float mx = -INFINITY, sum = 0.f;
  for (uint32_t s = 0; s < a.top; ++s) {
    const int64_t j = list[s];
    bool use = j >= 0 && j < (int64_t)a.nb;
    for (uint32_t e = 0; e < s; ++e) use = use && list[e] != j;
    if (!use) continue;
    const uint32_t t0 = (uint32_t)j << a.block_log2;
    const uint32_t t1 = (uint32_t)min((uint64_t)len, ((uint64_t)j + 1) << a.block_log2);
    for (uint32_t t = t0; t < t1; ++t) {
      float d = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < a.D) d += qf[i] * to_f32(k[(int64_t)t * a.ks[1] + lane + 32 * i]);
      d = warp_sum(d);
      const float nm = fmaxf(mx, d), c = expf(mx - nm), p = expf(d - nm);
      mx = nm;
      sum = sum * c + p;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < a.D)
          acc[i] = acc[i] * c + p * to_f32(v[(int64_t)t * a.vs[1] + lane + 32 * i]);
    }
  }
  T *o = (T *)a.out + w * a.D;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < a.D) o[lane + 32 * i] = from_f32<T>(sum > 0.f ? acc[i] / sum : 0.f);
  if (a.lse && lane == 0) a.lse[w] = sum > 0.f ? mx + logf(sum) : -INFINITY;
}

template <class T>
__device__ __forceinline__ float row_dot(const T *x, const T *y, uint32_t D, uint32_t lane) {
  float d = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < D) d += to_f32(x[lane + 32 * i]) * to_f32(y[lane + 32 * i]);
  return warp_sum(d);
}

template <class T>
__global__ void __launch_bounds__(256)
attend_dq(const AttnArgs a, float *delta) {
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t w = (uint64_t)blockIdx.x * 8u + (threadIdx.x >> 5);
  if (w >= (uint64_t)a.B * a.M * a.H) return;
  const uint32_t h = w % a.H;
  const uint64_t bm = w / a.H;
  const uint32_t m = bm % a.M, b = bm / a.M, g = h / (a.H / a.G);
  const T *q = (const T *)a.q + b * a.qs[0] + m * a.qs[1] + h * a.qs[2];
  const T *k = (const T *)a.k + b * a.ks[0] + g * a.ks[2];
  const T *v = (const T *)a.v + b * a.vs[0] + g * a.vs[2];
  const T *dout = (const T *)a.dout + w * a.D, *out = (const T *)a.out_in + w * a.D;
  const int64_t *list = a.blocks + bm * a.top;
  const uint32_t len = cloud_length(a.lengths, b, a.N);
  const float dl = row_dot(dout, out, a.D, lane), lse = a.lse_in[w];
  if (lane == 0) delta[w] = dl;
  float acc[4] = {};
  for (uint32_t s = 0; s < a.top; ++s) {
    const int64_t j = list[s];
    bool use = j >= 0 && j < (int64_t)a.nb;
    for (uint32_t e = 0; e < s; ++e) use = use && list[e] != j;
    if (!use) continue;
    const uint32_t t0 = (uint32_t)j << a.block_log2;
    const uint32_t t1 = (uint32_t)min((uint64_t)len, ((uint64_t)j + 1) << a.block_log2);
    for (uint32_t t = t0; t < t1; ++t) {
      const T *kt = k + (int64_t)t * a.ks[1];
      const float p = expf(row_dot(q, kt, a.D, lane) * a.scale - lse);
      const float ds = p * (row_dot(dout, v + (int64_t)t * a.vs[1], a.D, lane) - dl) * a.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < a.D) acc[i] += ds * to_f32(kt[lane + 32 * i]);
    }
  }
  T *o = (T *)a.dq + w * a.D;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < a.D) o[lane + 32 * i] = from_f32<T>(acc[i]);
}

// (block of keys, query slot) pairs for the sort; `none` for a slot that
// counts for nothing.
__global__ void __launch_bounds__(256)
pair_keys(const AttnArgs a, uint32_t none, uint32_t *__restrict__ keys,
          uint32_t *__restrict__ vals) {
  const uint32_t p = blockIdx.x * 256u + threadIdx.x;
  if (p >= a.B * a.M * a.top) return;
  const uint32_t bm = p / a.top, s = p - bm * a.top, b = bm / a.M;
  const int64_t *list = a.blocks + (uint64_t)bm * a.top;
  const int64_t j = list[s];
  bool use = j >= 0 && j < (int64_t)a.nb;
  for (uint32_t e = 0; e < s; ++e) use = use && list[e] != j;
  keys[p] = use ? b * a.nb + (uint32_t)j : none;
  vals[p] = p;
}

__global__ void __launch_bounds__(256)
pair_starts(const uint32_t *__restrict__ keys, uint32_t n, uint32_t groups,
            uint32_t *__restrict__ start) {
  const uint32_t r = blockIdx.x * 256u + threadIdx.x;
  if (r <= groups) start[r] = lower_bound(keys, n, r);
}

// One warp per (b, key, kv head): every query that chose the key's block, in
// ascending order.
template <class T>
__global__ void __launch_bounds__(256)
attend_dkv(const AttnArgs a, const float *delta, const uint32_t *vals, const uint32_t *start) {
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t w = (uint64_t)blockIdx.x * 8u + (threadIdx.x >> 5);
  if (w >= (uint64_t)a.B * a.N * a.G) return;
  const uint32_t g = w % a.G;
  const uint64_t bt = w / a.G;
  const uint32_t t = bt % a.N, b = bt / a.N, r = a.H / a.G;
  const T *kt = (const T *)a.k + b * a.ks[0] + t * a.ks[1] + g * a.ks[2];
  const T *vt = (const T *)a.v + b * a.vs[0] + t * a.vs[1] + g * a.vs[2];
  float dk[4] = {}, dv[4] = {};
  const uint32_t j = b * a.nb + (t >> a.block_log2);
  if (t < cloud_length(a.lengths, b, a.N))
    for (uint32_t e = start[j]; e < start[j + 1]; ++e) {
      const uint32_t bm = vals[e] / a.top, m = bm % a.M;
      for (uint32_t h = g * r; h < (g + 1) * r; ++h) {
        const uint64_t row = (uint64_t)bm * a.H + h;
        const T *q = (const T *)a.q + b * a.qs[0] + m * a.qs[1] + h * a.qs[2];
        const T *dout = (const T *)a.dout + row * a.D;
        const float p = expf(row_dot(q, kt, a.D, lane) * a.scale - a.lse_in[row]);
        const float ds = p * (row_dot(dout, vt, a.D, lane) - delta[row]) * a.scale;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (lane + 32 * i < a.D) {
            dk[i] += ds * to_f32(q[lane + 32 * i]);
            dv[i] += p * to_f32(dout[lane + 32 * i]);
          }
      }
    }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < a.D) {
      ((T *)a.dk)[w * a.D + lane + 32 * i] = from_f32<T>(dk[i]);
      ((T *)a.dv)[w * a.D + lane + 32 * i] = from_f32<T>(dv[i]);
    }
}

int check_attention(const nsfps_attention_desc *d) {
  if (!d) return set_error(NSFPS_ERR_ARG, "desc is NULL");
  if (d->reserved) return set_error(NSFPS_ERR_ARG, "reserved must be 0");
  if (d->dtype != NSFPS_F16 && d->dtype != NSFPS_BF16)
    return set_error(NSFPS_ERR_ARG, "dtype must be float16 or bfloat16");
  if (d->head_dim == 0 || d->head_dim > 128 || d->head_dim % 8)
    return set_error(NSFPS_ERR_ARG, "head_dim must be a multiple of 8 in 8..128");
  if (d->kv_heads == 0 || d->heads == 0 || d->heads > 256 || d->heads % d->kv_heads)
    return set_error(NSFPS_ERR_ARG, "heads must be a multiple of kv_heads, at most 256");
  if (d->block != 16 && d->block != 32 && d->block != 64 && d->block != 128)
    return set_error(NSFPS_ERR_ARG, "block must be 16, 32, 64 or 128");
  if (d->top == 0 || d->top > NSFPS_MAX_TOP)
    return set_error(NSFPS_ERR_ARG, "top must be in 1..%u", NSFPS_MAX_TOP);
  if (!std::isfinite(d->scale)) return set_error(NSFPS_ERR_ARG, "scale must be finite");
  const uint64_t lim = 1ull << 30;
  if (d->batch >= lim || d->queries >= lim || d->keys >= lim || d->batch * d->keys >= lim ||
      d->batch * d->queries >= lim || d->batch * d->queries * d->top >= lim)
    return set_error(NSFPS_ERR_UNSUPPORTED,
                     "batch * queries * top and batch * keys must be below 2^30");
  for (int i = 0; i < 3; ++i)
    if (d->q_stride[i] < 0 || d->k_stride[i] < 0 || d->v_stride[i] < 0 || d->q_stride[i] % 8 ||
        d->k_stride[i] % 8 || d->v_stride[i] % 8)
      return set_error(NSFPS_ERR_ARG, "strides must be multiples of 8 elements, not negative");
  return NSFPS_OK;
}

struct AttnWork {
  SortScratch sort;
  uint32_t *start;
  float *delta;
  uint64_t bytes;
};

AttnWork carve_attention(const nsfps_attention_desc &d, bool backward, void *base) {
  AttnWork w{};
  WorkCarver c(base);
  if (backward) {
    w.sort.carve(c, (uint32_t)(d.batch * d.queries * d.top));
    w.start = c.take<uint32_t>(d.batch * ceil_div(d.keys, d.block) + 1);
    w.delta = c.take<float>(d.batch * d.queries * d.heads);
  }
  w.bytes = c.off + 256;
  return w;
}

AttnArgs common_args(const nsfps_attention_desc &d, const void *q, const void *k, const void *v,
                     const int64_t *blocks, const int32_t *lengths) {
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.blocks = blocks; a.lengths = lengths;
  a.B = (uint32_t)d.batch; a.M = (uint32_t)d.queries; a.N = (uint32_t)d.keys;
  a.H = d.heads; a.G = d.kv_heads; a.D = d.head_dim; a.top = d.top;
  a.block_log2 = d.block == 16 ? 4 : d.block == 32 ? 5 : d.block == 64 ? 6 : 7;
  a.nb = (uint32_t)ceil_div(d.keys, d.block);
  for (int i = 0; i < 3; ++i) a.qs[i] = d.q_stride[i], a.ks[i] = d.k_stride[i], a.vs[i] = d.v_stride[i];
  a.scale = d.scale;
  return a;
}

int check_work(const void *d_work, uint64_t have, uint64_t need) {
  if (!d_work || (uint64_t)d_work % 256)
    return set_error(NSFPS_ERR_ARG, "d_work must be 256-byte aligned");
  if (have < need)
    return set_error(NSFPS_ERR_ARG, "d_work holds %llu bytes, %llu are needed",
                     (unsigned long long)have, (unsigned long long)need);
  return NSFPS_OK;
}

}  // namespace
}  // namespace nsfps

using namespace nsfps;

extern "C" {

int nsfps_block_attention_workspace(const nsfps_attention_desc *desc, int backward,
                                    uint64_t *bytes) {
  clear_error();
  int rc = check_attention(desc);
  if (rc) return rc;
  if (!bytes) return set_error(NSFPS_ERR_ARG, "bytes is NULL");
  *bytes = carve_attention(*desc, backward != 0, nullptr).bytes;
  return NSFPS_OK;
}

int nsfps_block_attention_device(const nsfps_attention_desc *desc, const void *d_q,
                                 const void *d_k, const void *d_v, const int64_t *d_blocks,
                                 const int32_t *d_lengths, void *d_out, float *d_lse,
                                 void *d_work, uint64_t work_bytes, void *stream) {
  clear_error();
  int rc = check_attention(desc);
  if (rc) return rc;
  const nsfps_attention_desc &d = *desc;
  if (d.batch * d.queries == 0) return NSFPS_OK;
  if (!d_q || !d_out || !d_blocks || (d.keys && (!d_k || !d_v)))
    return set_error(NSFPS_ERR_ARG, "NULL argument");
  if (((uint64_t)d_q | (uint64_t)d_k | (uint64_t)d_v | (uint64_t)d_out) % 16)
    return set_error(NSFPS_ERR_ARG, "q, k, v and out must be 16-byte aligned");
  if ((uint64_t)d_blocks % 8 || ((uint64_t)d_lse | (uint64_t)d_lengths) % 4)
    return set_error(NSFPS_ERR_ARG, "a pointer is not aligned to its elements");
  const AttnWork w = carve_attention(d, false, d_work);
  rc = check_work(d_work, work_bytes, w.bytes);
  if (rc) return rc;
  AttnArgs a = common_args(d, d_q, d_k, d_v, d_blocks, d_lengths);
  a.out = d_out;
  a.lse = d_lse;
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t grid = (uint32_t)ceil_div(d.batch * d.queries * d.heads, 8);
  if (d.dtype == NSFPS_F16) attend_forward<__half><<<grid, 256, 0, st>>>(a);
  else attend_forward<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  NSFPS_FEATURE_CUDA(cudaGetLastError());
  return NSFPS_OK;
}

int nsfps_block_attention_grad_device(const nsfps_attention_desc *desc, const void *d_q,
                                      const void *d_k, const void *d_v, const int64_t *d_blocks,
                                      const int32_t *d_lengths, const void *d_out,
                                      const float *d_lse, const void *d_dout, void *d_dq,
                                      void *d_dk, void *d_dv, void *d_work, uint64_t work_bytes,
                                      void *stream) {
  clear_error();
  int rc = check_attention(desc);
  if (rc) return rc;
  const nsfps_attention_desc &d = *desc;
  const uint64_t nq = d.batch * d.queries, nk = d.batch * d.keys;
  if (nq + nk == 0) return NSFPS_OK;
  if ((nq && (!d_q || !d_blocks || !d_out || !d_lse || !d_dout || !d_dq)) ||
      (nk && (!d_k || !d_v || !d_dk || !d_dv)))
    return set_error(NSFPS_ERR_ARG, "NULL argument");
  if (((uint64_t)d_q | (uint64_t)d_k | (uint64_t)d_v | (uint64_t)d_out | (uint64_t)d_dout |
       (uint64_t)d_dq | (uint64_t)d_dk | (uint64_t)d_dv) % 16)
    return set_error(NSFPS_ERR_ARG, "q, k, v, out and the gradients must be 16-byte aligned");
  if ((uint64_t)d_blocks % 8 || ((uint64_t)d_lse | (uint64_t)d_lengths) % 4)
    return set_error(NSFPS_ERR_ARG, "a pointer is not aligned to its elements");
  const AttnWork w = carve_attention(d, true, d_work);
  rc = check_work(d_work, work_bytes, w.bytes);
  if (rc) return rc;
  AttnArgs a = common_args(d, d_q, d_k, d_v, d_blocks, d_lengths);
  a.out_in = d_out; a.lse_in = d_lse; a.dout = d_dout;
  a.dq = d_dq; a.dk = d_dk; a.dv = d_dv;
  cudaStream_t st = (cudaStream_t)stream;
  const bool half = d.dtype == NSFPS_F16;
  if (nq) {
    const uint32_t grid = (uint32_t)ceil_div(nq * d.heads, 8);
    if (half) attend_dq<__half><<<grid, 256, 0, st>>>(a, w.delta);
    else attend_dq<__nv_bfloat16><<<grid, 256, 0, st>>>(a, w.delta);
    NSFPS_FEATURE_CUDA(cudaGetLastError());
  }
  if (nk) {
    const uint32_t n = (uint32_t)(nq * d.top), groups = a.B * a.nb;
    uint32_t *keys = w.sort.keys0, *vals = w.sort.vals0, launches = 0;
    if (n) {
      pair_keys<<<(uint32_t)ceil_div(n, 256), 256, 0, st>>>(a, groups, keys, vals);
      NSFPS_FEATURE_CUDA(cudaGetLastError());
      NSFPS_FEATURE_CUDA(run_sort_pairs(&keys, &vals, w.sort.keys1, w.sort.vals1, n, groups,
                                        w.sort.hist, w.sort.partial, st, launches));
    }
    pair_starts<<<(uint32_t)ceil_div((uint64_t)groups + 1, 256), 256, 0, st>>>(keys, n, groups,
                                                                              w.start);
    NSFPS_FEATURE_CUDA(cudaGetLastError());
    const uint32_t grid = (uint32_t)ceil_div(nk * d.kv_heads, 8);
    if (half) attend_dkv<__half><<<grid, 256, 0, st>>>(a, w.delta, vals, w.start);
    else attend_dkv<__nv_bfloat16><<<grid, 256, 0, st>>>(a, w.delta, vals, w.start);
    NSFPS_FEATURE_CUDA(cudaGetLastError());
  }
  return NSFPS_OK;
}

}  // extern "C"
