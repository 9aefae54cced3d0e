// nsfps_select.cu -- for every centre the nearest blocks of its cloud, by the
// squared distance to a block's bounding box (the bound that the sampler skips
// leaves with), exact in fp32.
//
// block_boxes reduces each block of points to its box.  choose_blocks scans
// the boxes of a cloud in index order, 32 per step and warp, and keeps the
// best `top` in registers, sorted over the lanes.  Distances are never
// negative or NaN, so their bits order as integers; the scan runs upwards, so
// a later block of equal distance never displaces an earlier one and a strict
// comparison gives the (d2, index) order.
#include <algorithm>

#include "nsfps_feature.cuh"

namespace nsfps {
namespace {

constexpr uint32_t kFullMask = 0xffffffffu;
constexpr uint32_t kNoDist = 0x7f800001u;  // above +inf: an empty slot of a list

struct SelectArgs {
  const float *xyz, *centers;
  const int32_t *lengths;  // or null
  uint32_t B, n, m, nb;    // nb: blocks of a cloud of n points
  uint32_t block_log2, top;
  float *box;              // 6 arrays of B * nb: lo x, y, z, hi x, y, z
  int64_t *out;
  float *out_d2;           // or null
};

__device__ __forceinline__ uint32_t cloud_length(const int32_t *lengths, uint32_t b, uint32_t n) {
  return lengths ? (uint32_t)min(max(lengths[b], 0), (int)n) : n;
}

// 16 lanes per block of points.
__global__ void __launch_bounds__(256)
block_boxes(const SelectArgs a) {
  const uint32_t g = blockIdx.x * 16u + (threadIdx.x >> 4), lane = threadIdx.x & 15u;
  const uint32_t all = a.B * a.nb;
  const float inf = __int_as_float(0x7f800000);
  float lo[3] = {inf, inf, inf}, hi[3] = {-inf, -inf, -inf};
  if (g < all) {
    const uint32_t b = g / a.nb, j = g - b * a.nb;
    const uint32_t len = cloud_length(a.lengths, b, a.n);
    const uint64_t end = min((uint64_t)len, ((uint64_t)j + 1) << a.block_log2);
    const float *p = a.xyz + 3 * (uint64_t)b * a.n;
    for (uint64_t i = ((uint64_t)j << a.block_log2) + lane; i < end; i += 16u)
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const float v = p[3 * i + k];
        lo[k] = fminf(lo[k], v);  // fminf / fmaxf drop a NaN
        hi[k] = fmaxf(hi[k], v);
      }
  }
#pragma unroll
  for (int o = 8; o; o >>= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      lo[k] = fminf(lo[k], __shfl_xor_sync(kFullMask, lo[k], o));
      hi[k] = fmaxf(hi[k], __shfl_xor_sync(kFullMask, hi[k], o));
    }
  if (g < all && lane < 6u) {
    const float v = lane == 0u ? lo[0] : lane == 1u ? lo[1] : lane == 2u ? lo[2]
                  : lane == 3u ? hi[0] : lane == 4u ? hi[1] : hi[2];
    a.box[(uint64_t)lane * all + g] = v;
  }
}

__device__ __forceinline__ float axis_gap(float lo, float hi, float c) {
  return fmaxf(fmaxf(__fsub_rn(lo, c), __fsub_rn(c, hi)), 0.0f);
}

// The `top` smallest (distance bits, block) seen so far, ascending over lane
// + 32 * slot.
template <int SLOTS>
struct BestList {
  uint32_t d[SLOTS], j[SLOTS];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) d[s] = kNoDist, j[s] = 0u;
  }
  __device__ __forceinline__ uint32_t limit(uint32_t top) const {
    return __shfl_sync(kFullMask, d[SLOTS - 1], (top - 1u) & 31u);
  }
  // (all lanes) puts (cd, cj) behind every entry of distance <= cd
  __device__ __forceinline__ void insert(uint32_t cd, uint32_t cj, uint32_t lane) {
    uint32_t at = 0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) at += __popc(__ballot_sync(kFullMask, d[s] <= cd));
    uint32_t carry_d = 0, carry_j = 0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const uint32_t last_d = __shfl_sync(kFullMask, d[s], 31);
      const uint32_t last_j = __shfl_sync(kFullMask, j[s], 31);
      uint32_t up_d = __shfl_up_sync(kFullMask, d[s], 1);
      uint32_t up_j = __shfl_up_sync(kFullMask, j[s], 1);
      if (lane == 0u) up_d = carry_d, up_j = carry_j;
      const uint32_t me = lane + 32u * s;
      if (me > at) d[s] = up_d, j[s] = up_j;
      else if (me == at) d[s] = cd, j[s] = cj;
      carry_d = last_d;
      carry_j = last_j;
    }
  }
  // (all lanes) offers every lane's (cd, cj), lower lanes first
  __device__ __forceinline__ void offer(uint32_t cd, uint32_t cj, uint32_t top, uint32_t lane,
                                        uint32_t &lim) {
    uint32_t want = __ballot_sync(kFullMask, cd < lim);
    while (want) {
      const int src = __ffs(want) - 1;
      insert(__shfl_sync(kFullMask, cd, src), __shfl_sync(kFullMask, cj, src), lane);
      lim = limit(top);
      want &= __ballot_sync(kFullMask, cd < lim) & ~((2u << src) - 1u);
    }
  }
};

// WARPS warps per centre (8 / WARPS centres per CTA); each scans a contiguous
// share of the blocks and the first joins the lists in share order.
template <int SLOTS, int WARPS>
__global__ void __launch_bounds__(256)
choose_blocks(const SelectArgs a) {
  __shared__ uint32_t s_d[WARPS > 1 ? 8 : 1][SLOTS * 32], s_j[WARPS > 1 ? 8 : 1][SLOTS * 32];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint32_t c = blockIdx.x * (8u / WARPS) + warp / WARPS;
  const bool live = c < a.B * a.m;
  BestList<SLOTS> best;
  best.clear();
  uint32_t lim = kNoDist;
  if (live) {
    const uint32_t b = c / a.m;
    const uint32_t len = cloud_length(a.lengths, b, a.n);
    const uint32_t nv = (uint32_t)(((uint64_t)len + (1u << a.block_log2) - 1u) >> a.block_log2);
    const uint32_t share = (nv + WARPS - 1u) / WARPS;
    const uint32_t j0 = min(nv, (warp % WARPS) * share), j1 = min(nv, j0 + share);
    const float cx = a.centers[3 * (uint64_t)c], cy = a.centers[3 * (uint64_t)c + 1],
                cz = a.centers[3 * (uint64_t)c + 2];
    const uint64_t all = (uint64_t)a.B * a.nb;
    const float *box = a.box + (uint64_t)b * a.nb;
    for (uint32_t j = j0; j < j1; j += 32u) {
      uint32_t d = kNoDist;
      if (j + lane < j1) {
        const float *p = box + j + lane;
        const float dx = axis_gap(p[0], p[3 * all], cx), dy = axis_gap(p[all], p[4 * all], cy),
                    dz = axis_gap(p[2 * all], p[5 * all], cz);
        d = __float_as_uint(
            __fadd_rn(__fadd_rn(__fmul_rn(dx, dx), __fmul_rn(dy, dy)), __fmul_rn(dz, dz)));
      }
      best.offer(d, j + lane, a.top, lane, lim);
    }
  }
  if (WARPS > 1) {
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      s_d[warp][lane + 32 * s] = best.d[s], s_j[warp][lane + 32 * s] = best.j[s];
    __syncthreads();
    if (!live || warp % WARPS) return;
    for (int w = 1; w < WARPS; ++w)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
        best.offer(s_d[warp + w][lane + 32 * s], s_j[warp + w][lane + 32 * s], a.top, lane, lim);
  }
  if (!live) return;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const uint32_t i = lane + 32u * s;
    if (i >= a.top) continue;
    const bool some = best.d[s] != kNoDist;
    const uint64_t o = (uint64_t)c * a.top + i;
    a.out[o] = some ? (int64_t)best.j[s] : -1;
    if (a.out_d2) a.out_d2[o] = __uint_as_float(some ? best.d[s] : 0x7f800000u);
  }
}

template <int SLOTS>
cudaError_t launch_choose(const SelectArgs &a, cudaStream_t st) {
  const uint32_t centres = a.B * a.m;
  // Few centres leave SMs idle at a warp each: below two waves of warps a
  // whole CTA scans for one centre.
  if (centres < 148u * 16u)
    choose_blocks<SLOTS, 8><<<centres, 256, 0, st>>>(a);
  else
    choose_blocks<SLOTS, 1><<<(uint32_t)ceil_div(centres, 8), 256, 0, st>>>(a);
  return cudaGetLastError();
}

int check_select(const nsfps_select_desc *d) {
  if (!d) return set_error(NSFPS_ERR_ARG, "desc is NULL");
  if (d->block != 16 && d->block != 32 && d->block != 64 && d->block != 128)
    return set_error(NSFPS_ERR_ARG, "block must be 16, 32, 64 or 128");
  if (d->top == 0 || d->top > NSFPS_MAX_TOP)
    return set_error(NSFPS_ERR_ARG, "top must be in 1..%u", NSFPS_MAX_TOP);
  const uint64_t lim = 1ull << 31;
  if (d->batch >= lim || d->points >= lim || d->centers >= lim || d->batch * d->points >= lim ||
      d->batch * d->centers >= lim)
    return set_error(NSFPS_ERR_UNSUPPORTED,
                     "batch * points and batch * centers must be below 2^31");
  return NSFPS_OK;
}

uint64_t select_work_bytes(const nsfps_select_desc &d) {
  return d.batch * ceil_div(d.points, d.block) * 6 * sizeof(float) + 256;
}

}  // namespace
}  // namespace nsfps

using namespace nsfps;

extern "C" {

int nsfps_select_blocks_workspace(const nsfps_select_desc *desc, uint64_t *bytes) {
  clear_error();
  int rc = check_select(desc);
  if (rc) return rc;
  if (!bytes) return set_error(NSFPS_ERR_ARG, "bytes is NULL");
  *bytes = select_work_bytes(*desc);
  return NSFPS_OK;
}

int nsfps_select_blocks_device(const nsfps_select_desc *desc, const float *d_xyz,
                               const int32_t *d_lengths, const float *d_centers,
                               int64_t *d_blocks, float *d_d2, void *d_work, uint64_t work_bytes,
                               void *stream) {
  clear_error();
  int rc = check_select(desc);
  if (rc) return rc;
  const nsfps_select_desc &d = *desc;
  if (d.batch * d.centers == 0) return NSFPS_OK;
  if (!d_centers || !d_blocks || (d.points && !d_xyz))
    return set_error(NSFPS_ERR_ARG, "NULL argument");
  if (((uint64_t)d_xyz | (uint64_t)d_centers | (uint64_t)d_lengths | (uint64_t)d_d2) % 4 ||
      (uint64_t)d_blocks % 8)
    return set_error(NSFPS_ERR_ARG, "a pointer is not aligned to its elements");
  if (!d_work || (uint64_t)d_work % 256)
    return set_error(NSFPS_ERR_ARG, "d_work must be 256-byte aligned");
  if (work_bytes < select_work_bytes(d))
    return set_error(NSFPS_ERR_ARG, "d_work holds %llu bytes, %llu are needed",
                     (unsigned long long)work_bytes, (unsigned long long)select_work_bytes(d));
  cudaStream_t st = (cudaStream_t)stream;
  SelectArgs a{};
  a.xyz = d_xyz;
  a.centers = d_centers;
  a.lengths = d_lengths;
  a.B = (uint32_t)d.batch;
  a.n = (uint32_t)d.points;
  a.m = (uint32_t)d.centers;
  a.nb = (uint32_t)ceil_div(d.points, d.block);
  a.block_log2 = d.block == 16 ? 4 : d.block == 32 ? 5 : d.block == 64 ? 6 : 7;
  a.top = d.top;
  a.box = (float *)d_work;
  a.out = d_blocks;
  a.out_d2 = d_d2;
  if (a.nb) {
    block_boxes<<<(uint32_t)ceil_div((uint64_t)a.B * a.nb, 16), 256, 0, st>>>(a);
    NSFPS_FEATURE_CUDA(cudaGetLastError());
  }
  NSFPS_FEATURE_CUDA(d.top <= 32 ? launch_choose<1>(a, st) : launch_choose<2>(a, st));
  return NSFPS_OK;
}

}  // extern "C"
