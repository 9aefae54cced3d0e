// nsfps_select.cu -- for every centre the nearest blocks of its cloud, by the
// squared distance to a block's bounding box (the bound that the sampler skips
// leaves with), exact in fp32.
//
// block_boxes reduces each block of points to its box, and each group of 32
// blocks to one box around theirs.  choose_blocks, one warp per centre, looks
// at the groups first: rounding is monotone, so a group's distance is never
// above a block's of it, exactly.  It takes the nearest group for a first list
// of `top`, then every group that is not beyond the list's last distance, and
// keeps the list sorted over the lanes.  Distances are never negative or NaN,
// so (distance bits, index) order as one 64-bit key, lower indices first among
// equals.  (Scanning every block cost 3.6 ns of the machine per centre over 512
// blocks, most of it insertions; the order by groups leaves few.)
#include <algorithm>

#include "nsfps_feature.cuh"

namespace nsfps {
namespace {

constexpr uint32_t kFullMask = 0xffffffffu;
constexpr uint64_t kNoKey = (uint64_t)0x7f800001u << 32;  // above +inf: an empty slot

struct SelectArgs {
  const float *xyz, *centers;
  const int32_t *lengths;  // or null
  uint32_t B, n, m;
  uint32_t block_log2, top;
  uint32_t ng;             // groups of 32 blocks of a cloud
  float *box;              // 6 arrays of B * ng * 32: lo x, y, z, hi x, y, z
  float *group;            // 6 arrays of B * ng, likewise
  int64_t *out;
  float *out_d2;           // or null
};

__device__ __forceinline__ uint32_t cloud_length(const int32_t *lengths, uint32_t b, uint32_t n) {
  return lengths ? (uint32_t)min(max(lengths[b], 0), (int)n) : n;
}

// One CTA per group of 32 blocks, 16 lanes per block.
__global__ void __launch_bounds__(512)
block_boxes(const SelectArgs a) {
  __shared__ float s_box[32][6];
  const uint32_t g = blockIdx.x, k = threadIdx.x >> 4, lane = threadIdx.x & 15u;
  const uint32_t b = g / a.ng, j = (g - b * a.ng) * 32u + k;
  const uint64_t groups = (uint64_t)a.B * a.ng;
  const float inf = __int_as_float(0x7f800000);
  float lo[3] = {inf, inf, inf}, hi[3] = {-inf, -inf, -inf};
  const uint32_t len = cloud_length(a.lengths, b, a.n);
  const uint64_t end = min((uint64_t)len, ((uint64_t)j + 1) << a.block_log2);
  const float *p = a.xyz + 3 * (uint64_t)b * a.n;
  for (uint64_t i = ((uint64_t)j << a.block_log2) + lane; i < end; i += 16u)
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      const float v = p[3 * i + x];
      lo[x] = fminf(lo[x], v);  // fminf / fmaxf drop a NaN
      hi[x] = fmaxf(hi[x], v);
    }
#pragma unroll
  for (int o = 8; o; o >>= 1)
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      lo[x] = fminf(lo[x], __shfl_xor_sync(kFullMask, lo[x], o));
      hi[x] = fmaxf(hi[x], __shfl_xor_sync(kFullMask, hi[x], o));
    }
  if (lane < 6u) {
    const float v = lane == 0u ? lo[0] : lane == 1u ? lo[1] : lane == 2u ? lo[2]
                  : lane == 3u ? hi[0] : lane == 4u ? hi[1] : hi[2];
    s_box[k][lane] = v;
    a.box[lane * groups * 32u + (uint64_t)g * 32u + k] = v;
  }
  __syncthreads();
  if (threadIdx.x < 32u) {
#pragma unroll
    for (int x = 0; x < 6; ++x) {
      float v = s_box[threadIdx.x][x];
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const float y = __shfl_xor_sync(kFullMask, v, o);
        v = x < 3 ? fminf(v, y) : fmaxf(v, y);
      }
      if (threadIdx.x == 0) a.group[x * groups + g] = v;
    }
  }
}

__device__ __forceinline__ float axis_gap(float lo, float hi, float c) {
  return fmaxf(fmaxf(__fsub_rn(lo, c), __fsub_rn(c, hi)), 0.0f);
}

// Bits of the squared distance from (x, y, z) to box `at` of six arrays.
__device__ __forceinline__ uint32_t box_distance(const float *__restrict__ box, uint64_t stride,
                                                 uint64_t at, float x, float y, float z) {
  const float *p = box + at;
  const float dx = axis_gap(p[0], p[3 * stride], x), dy = axis_gap(p[stride], p[4 * stride], y),
              dz = axis_gap(p[2 * stride], p[5 * stride], z);
  return __float_as_uint(
      __fadd_rn(__fadd_rn(__fmul_rn(dx, dx), __fmul_rn(dy, dy)), __fmul_rn(dz, dz)));
}

__device__ __forceinline__ uint64_t min64(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a < b ? b : a; }

// Ascending sort of one key per lane; from_stage 32 merges a sequence that
// rises and then falls.
template <int FROM>
__device__ __forceinline__ uint64_t sort_lanes(uint64_t v, uint32_t lane) {
#pragma unroll
  for (uint32_t k = FROM; k <= 32u; k <<= 1)
#pragma unroll
    for (uint32_t j = k >> 1; j; j >>= 1) {
      const uint64_t o = __shfl_xor_sync(kFullMask, v, j);
      const bool up = (lane & k) == 0u, low = (lane & j) == 0u;
      v = (low == up) ? min64(v, o) : max64(v, o);
    }
  return v;
}

// The smallest keys so far, ascending over lane + 32 * slot.
template <int SLOTS>
struct BestList {
  uint64_t v[SLOTS];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) v[s] = kNoKey;
  }
  __device__ __forceinline__ uint64_t limit(uint32_t top) const {
    return __shfl_sync(kFullMask, v[SLOTS - 1], (top - 1u) & 31u);
  }
  __device__ __forceinline__ void insert(uint64_t c, uint32_t lane) {
    uint32_t at = 0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) at += __popc(__ballot_sync(kFullMask, v[s] < c));
    uint64_t carry = 0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const uint64_t last = __shfl_sync(kFullMask, v[s], 31);
      uint64_t up = __shfl_up_sync(kFullMask, v[s], 1);
      if (lane == 0u) up = carry;
      const uint32_t me = lane + 32u * s;
      v[s] = me > at ? up : me == at ? c : v[s];
      carry = last;
    }
  }
  // One key per lane (kNoKey: none), all different from the list's.  Few are
  // inserted one by one (about 15 instructions each); many are sorted and
  // merged (about 200).
  __device__ __forceinline__ void offer(uint64_t c, uint32_t top, uint32_t lane, uint64_t &lim) {
    uint32_t want = __ballot_sync(kFullMask, c < lim);
    if (__popc(want) > 10) {
      uint64_t x = sort_lanes<2>(c, lane);
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const uint64_t y = __shfl_sync(kFullMask, x, 31u - lane);
        const uint64_t lo = min64(v[s], y), hi = max64(v[s], y);
        v[s] = sort_lanes<32>(lo, lane);
        if (s + 1 < SLOTS) x = sort_lanes<32>(hi, lane);
      }
      lim = limit(top);
      return;
    }
    while (want) {
      const int src = __ffs(want) - 1;
      insert(__shfl_sync(kFullMask, c, src), lane);
      lim = limit(top);
      want &= __ballot_sync(kFullMask, c < lim) & ~((2u << src) - 1u);
    }
  }
};

constexpr int kAhead = 4;  // group distances in flight per lane

template <int SLOTS>
__global__ void __launch_bounds__(256)
choose_blocks(const SelectArgs a) {
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t c = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (c >= a.B * a.m) return;
  const uint32_t b = c / a.m;
  const uint32_t len = cloud_length(a.lengths, b, a.n);
  const uint32_t nv = (uint32_t)(((uint64_t)len + (1u << a.block_log2) - 1u) >> a.block_log2);
  const uint32_t ng = (nv + 31u) / 32u;
  const float x = a.centers[3 * (uint64_t)c], y = a.centers[3 * (uint64_t)c + 1],
              z = a.centers[3 * (uint64_t)c + 2];
  const uint64_t groups = (uint64_t)a.B * a.ng;
  const float *gbox = a.group + (uint64_t)b * a.ng, *bbox = a.box + (uint64_t)b * a.ng * 32u;
  BestList<SLOTS> best;
  best.clear();
  uint64_t lim = kNoKey;
  auto take = [&](uint32_t g) {
    const uint32_t j = g * 32u + lane;
    uint64_t key = kNoKey;
    if (j < nv) key = (uint64_t)box_distance(bbox, groups * 32u, j, x, y, z) << 32 | j;
    best.offer(key, a.top, lane, lim);
  };
  // the nearest groups, until the list is full
  uint32_t done[SLOTS + 1];
#pragma unroll
  for (int i = 0; i <= SLOTS; ++i) {
    done[i] = 0xffffffffu;
    if (i && lim != kNoKey) continue;
    uint64_t near = ~0ull;
    for (uint32_t g0 = 0; g0 < ng; g0 += 32u * kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t g = g0 + u * 32u + lane;
        bool free = g < ng;
#pragma unroll
        for (int k = 0; k < i; ++k) free = free && g != done[k];
        if (free) near = min64(near, (uint64_t)box_distance(gbox, groups, g, x, y, z) << 32 | g);
      }
    }
    const uint32_t d = __reduce_min_sync(kFullMask, (uint32_t)(near >> 32));
    if (d == 0xffffffffu) continue;  // no group is left
    done[i] = __reduce_min_sync(kFullMask, (uint32_t)(near >> 32) == d ? (uint32_t)near : ~0u);
    take(done[i]);
  }
  // every other group that may hold a nearer block
  for (uint32_t g0 = 0; g0 < ng; g0 += 32u * kAhead) {
    uint32_t d[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t g = g0 + u * 32u + lane;
      d[u] = 0xffffffffu;
      bool free = g < ng;
#pragma unroll
      for (int k = 0; k <= SLOTS; ++k) free = free && g != done[k];
      if (free) d[u] = box_distance(gbox, groups, g, x, y, z);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      // (an equal distance may go with a lower index)
      uint32_t want = __ballot_sync(kFullMask, d[u] <= (uint32_t)(lim >> 32));
      while (want) {
        const int src = __ffs(want) - 1;
        take(g0 + u * 32u + src);
        want &= __ballot_sync(kFullMask, d[u] <= (uint32_t)(lim >> 32)) & ~((2u << src) - 1u);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const uint32_t i = lane + 32u * s;
    if (i >= a.top) continue;
    const bool some = best.v[s] < kNoKey;
    const uint64_t o = (uint64_t)c * a.top + i;
    a.out[o] = some ? (int64_t)(uint32_t)best.v[s] : -1;
    if (a.out_d2) a.out_d2[o] = __uint_as_float(some ? (uint32_t)(best.v[s] >> 32) : 0x7f800000u);
  }
}

template <int SLOTS>
cudaError_t launch_choose(const SelectArgs &a, cudaStream_t st) {
  // one warp per CTA while there is an SM for each centre, up to eight
  const uint32_t centres = a.B * a.m;
  const uint32_t warps = std::min(8u, std::max(1u, centres / (uint32_t)sm_count()));
  choose_blocks<SLOTS><<<(uint32_t)ceil_div(centres, warps), warps * 32u, 0, st>>>(a);
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
  return d.batch * ceil_div(d.points, 32ull * d.block) * 33 * 6 * sizeof(float) + 256;
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
  a.ng = (uint32_t)ceil_div(d.points, 32ull * d.block);
  a.block_log2 = d.block == 16 ? 4 : d.block == 32 ? 5 : d.block == 64 ? 6 : 7;
  a.top = d.top;
  a.box = (float *)d_work;
  a.group = a.box + (uint64_t)a.B * a.ng * 32 * 6;
  a.out = d_blocks;
  a.out_d2 = d_d2;
  if (a.ng) {
    block_boxes<<<a.B * a.ng, 512, 0, st>>>(a);
    NSFPS_FEATURE_CUDA(cudaGetLastError());
  }
  NSFPS_FEATURE_CUDA(d.top <= 32 ? launch_choose<1>(a, st) : launch_choose<2>(a, st));
  return NSFPS_OK;
}

}  // extern "C"
