// nsfps_select.cu -- for every centre the nearest blocks of its cloud, by the
// squared distance to a block's bounding box (the bound that the sampler skips
// leaves with), exact in fp32.
//
// block_boxes reduces each block of points to its box, and each group of 32
// blocks to one box around theirs.  choose_blocks, one warp per centre, looks
// at the groups first: rounding is monotone, so a group's distance is never
// above a block's of it, exactly.  The nearest groups give a bound on the
// `top`-th distance; the blocks of all groups within it are looked at in index
// order, and those within it are listed and ranked by comparison.  Distances
// are never negative or NaN, so their bits order as integers, and a list in
// index order gives the lower index among equals first.  What bounds it is
// instructions (73 % of the issue slots) and the wait for boxes out of
// the L1: 131,072 centres over 512 blocks of padded clouds and top 16 take 158 us
// (a list kept sorted by insertion over all blocks 469, by groups 260), 16,384
// centres over 1,920 blocks 54 (203, 76).
#include <algorithm>

#include "nsfps_feature.cuh"

namespace nsfps {
namespace {

constexpr uint32_t kFullMask = 0xffffffffu;
constexpr uint32_t kNoDist = 0xffffffffu;  // above every distance

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

constexpr int kAhead = 4;            // group distances in flight per lane
constexpr int kNear = 4;             // groups that the bound is taken from
constexpr uint32_t kListMax = 128;   // candidates listed per centre

// The candidates of a centre, in shared memory: distance bits and block, in an
// order that has the lower block first among equal distances.
struct Candidates {
  uint32_t *d, *j;
  uint32_t n;

  // Calls f(rank, distance, block) for every candidate, one per lane and turn;
  // the rank is the number of candidates before it in (distance, place) order,
  // found by comparing with all of them, which for the usual 25 is cheaper than
  // any sort.
  template <class F>
  __device__ __forceinline__ void ranked(uint32_t lane, F f) const {
    for (uint32_t base = 0; base < n; base += 32u) {
      const uint32_t me = base + lane;
      const bool some = me < n;
      const uint32_t mine = some ? d[me] : kNoDist, block = some ? j[me] : 0u;
      uint32_t rank = 0;
      for (uint32_t k = 0; k < n; k += 4u) {
        const uint4 o = *reinterpret_cast<const uint4 *>(d + k);  // (unused places hold kNoDist)
        rank += o.x < mine + (k < me) ? 1u : 0u;
        rank += o.y < mine + (k + 1u < me) ? 1u : 0u;
        rank += o.z < mine + (k + 2u < me) ? 1u : 0u;
        rank += o.w < mine + (k + 3u < me) ? 1u : 0u;
      }
      f(some, rank, mine, block);
    }
  }
  // Fills the places up to a multiple of four.
  __device__ __forceinline__ void pad(uint32_t lane) {
    if (lane < 4u) d[n + lane] = kNoDist;
    __syncwarp();
  }
};

// Clouds of at most this many blocks: every distance is computed once and held
// in registers, without groups.  32 clouds of 4,096 centres and top 16 take, so
// and by groups, 108 and 169 us with 128 blocks, 132 and 185 with 256, 182 and
// 207 with 512; eight clouds of 2,048 and top 48 with 512 53 and 87, one centre
// 10 and 6.  Twice the registers, for 1,024 blocks, cost occupancy: 252 us with
// 512, 292 with 700 and 357 with 1,024, by groups 238 and 259.
constexpr int kHeldRegs = 16;
constexpr uint32_t kHeldBlocks = 32 * kHeldRegs;

// SLOTS: 32-entry parts of the result.
template <int SLOTS, bool HELD>
__global__ void __launch_bounds__(256)
choose_blocks(const SelectArgs a) {
  after_previous();
  __shared__ __align__(16) uint32_t s_d[8][kListMax + 4], s_j[8][kListMax];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint32_t c = blockIdx.x * (blockDim.x >> 5) + warp;
  if (c >= a.B * a.m) return;
  const uint32_t b = c / a.m;
  const uint32_t len = cloud_length(a.lengths, b, a.n);
  const uint32_t nv = (uint32_t)(((uint64_t)len + (1u << a.block_log2) - 1u) >> a.block_log2);
  const uint32_t ng = (nv + 31u) / 32u;
  const float x = a.centers[3 * (uint64_t)c], y = a.centers[3 * (uint64_t)c + 1],
              z = a.centers[3 * (uint64_t)c + 2];
  const uint64_t groups = (uint64_t)a.B * a.ng;
  const float *gbox = a.group + (uint64_t)b * a.ng, *bbox = a.box + (uint64_t)b * a.ng * 32u;
  auto block_distance = [&](uint32_t j) {
    return j < nv ? box_distance(bbox, groups * 32u, j, x, y, z) : kNoDist;
  };

  // A bound on the top-th distance: of the nearest groups' blocks each lane
  // keeps its smallest distance (with SLOTS 2 the smallest of every other
  // group); `top` of these are as many blocks within their top-th.
  uint32_t limit = 0x7f800000u;
  uint32_t held[HELD ? kHeldRegs : 1];
  if (HELD) {
#pragma unroll
    for (int r = 0; r < kHeldRegs; ++r) {
      held[r] = kNoDist;
      if (32u * r < nv) held[r] = block_distance(32u * r + lane);
    }
  }
  if (nv > a.top) {
    uint32_t done[kNear], v[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) v[s] = kNoDist;
    if (HELD) {
#pragma unroll
      for (int r = 0; r < kHeldRegs; ++r) v[r % SLOTS] = min(v[r % SLOTS], held[r]);
    }
#pragma unroll
    for (int i = 0; i < (HELD ? 0 : kNear); ++i) {
      uint32_t near = kNoDist, who = kNoDist;
      for (uint32_t g0 = 0; g0 < ng; g0 += 32u) {
        const uint32_t g = g0 + lane;
        uint32_t d = g < ng ? box_distance(gbox, groups, g, x, y, z) : kNoDist;
#pragma unroll
        for (int k = 0; k < i; ++k)
          if (g == done[k]) d = kNoDist;
        if (d < near) near = d, who = g;
      }
      const uint32_t d = __reduce_min_sync(kFullMask, near);
      done[i] = __reduce_min_sync(kFullMask, near == d ? who : kNoDist);
      if (d == kNoDist) continue;  // no group is left
      v[i % SLOTS] = min(v[i % SLOTS], block_distance(done[i] * 32u + lane));
    }
    // the smallest 15-bit prefix that `top` of the lanes do not exceed (all
    // bits set where fewer have a block)
    uint32_t prefix = 0;
#pragma unroll
    for (int bit = 30; bit >= 16; --bit) {
      const uint32_t below = prefix | (1u << bit);  // first value with this bit
      uint32_t count = 0;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) count += __popc(__ballot_sync(kFullMask, v[s] < below));
      if (count < a.top) prefix = below;
    }
    limit = min(prefix | 0xffffu, limit);
  }

  // The blocks within the bound, in index order.
  Candidates list{s_d[warp], s_j[warp], 0u};
  bool open = true;  // false: nothing further can be nearer
  auto add = [&](uint32_t d, uint32_t j0) {  // blocks j0 .. j0 + 31
    const uint32_t in = __ballot_sync(kFullMask, d <= limit);
    if (!in) return;
    if (d <= limit) {
      const uint32_t at = list.n + __popc(in & ((1u << lane) - 1u));
      list.d[at] = d;
      list.j[at] = j0 + lane;
    }
    list.n += __popc(in);
    __syncwarp();
    if (list.n + 32u <= kListMax) return;
    // the list is full: keep its best, in order (what follows has higher
    // indices, so from here on only smaller distances matter)
    list.pad(lane);
    uint32_t rank[kListMax / 32], dist[kListMax / 32], block[kListMax / 32];
    int turn = 0;
    list.ranked(lane, [&](bool some, uint32_t r, uint32_t d, uint32_t j) {
      rank[turn] = some ? r : kNoDist;
      dist[turn] = d;
      block[turn++] = j;
    });
    __syncwarp();
#pragma unroll
    for (int i = 0; i < (int)kListMax / 32; ++i)
      if (i < turn && rank[i] < a.top) list.d[rank[i]] = dist[i], list.j[rank[i]] = block[i];
    __syncwarp();
    list.n = a.top;
    const uint32_t last = list.d[a.top - 1u];
    open = last != 0u;
    limit = last - 1u;
  };
  if (HELD) {
#pragma unroll
    for (int r = 0; r < kHeldRegs; ++r)
      if (32u * r < nv && open) add(held[r], 32u * r);
  }
  for (uint32_t g0 = 0; !HELD && g0 < ng && open; g0 += 32u * kAhead) {
    uint32_t gd[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t g = g0 + u * 32u + lane;
      gd[u] = kNoDist;
      if (g0 + u * 32u >= ng) continue;
      gd[u] = g < ng ? box_distance(gbox, groups, g, x, y, z) : kNoDist;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (g0 + u * 32u >= ng) break;
      uint32_t want = __ballot_sync(kFullMask, gd[u] <= limit);
      while (want && open) {
        const uint32_t g = g0 + u * 32u + __ffs(want) - 1u;
        want &= want - 1u;
        add(block_distance(g * 32u + lane), g * 32u);
        want &= __ballot_sync(kFullMask, gd[u] <= limit);
      }
    }
  }
  const uint32_t found = min(a.top, list.n);
  const uint64_t to = (uint64_t)c * a.top;
  list.pad(lane);
  list.ranked(lane, [&](bool some, uint32_t rank, uint32_t d, uint32_t j) {
    if (!some || rank >= a.top) return;
    a.out[to + rank] = (int64_t)j;
    if (a.out_d2) a.out_d2[to + rank] = __uint_as_float(d);
  });
  for (uint32_t i = found + lane; i < a.top; i += 32u) {
    a.out[to + i] = -1;
    if (a.out_d2) a.out_d2[to + i] = __uint_as_float(0x7f800000u);
  }
}

template <int SLOTS>
cudaError_t launch_choose(const SelectArgs &a, cudaStream_t st) {
  // one warp per CTA while there is an SM for each centre, up to eight
  const uint32_t centres = a.B * a.m;
  const uint32_t warps = std::min(8u, std::max(1u, centres / (uint32_t)sm_count()));
  const uint32_t grid = (uint32_t)ceil_div(centres, warps);
  if (ceil_div(a.n, 1ull << a.block_log2) <= kHeldBlocks)
    return launch_next(choose_blocks<SLOTS, true>, grid, warps * 32u, 0, st, a);
  return launch_next(choose_blocks<SLOTS, false>, grid, warps * 32u, 0, st, a);
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
