// nsfps_sort.cuh -- stable sort of the positions 0 .. n - 1 by a 32-bit key,
// for the feature operators' lists (row lookups by row, query and span pairs
// by span).  Positions whose key is `none` are dropped.
//
// Least significant digit first, digits of up to 8 bits over the bits that
// the keys use, three launches per digit: per-tile digit counts; one CTA per
// digit turns its counts into offsets; each tile ranks its keys, orders them
// in shared memory and writes runs.  The first digit reads the keys from a
// source object and takes a position's value to be the position itself.
// Where a list has ten million entries this moves 20 bytes per entry and
// digit; at the usual hundred thousand it is bound by its launches.  So the
// offsets of few tiles are summed where they are used (two launches per
// digit), and a list that fits one CTA takes one launch in all.  (The sampler's
// setup has a sort of its own, by an array of keys that it keeps whole; here keys
// come from what a caller has, entries are dropped on the way, and the short
// lists of a call count.)
#pragma once

#include "nsfps_feature.cuh"

namespace nsfps {

constexpr uint32_t kSortThreads = 256, kSortWarps = kSortThreads / 32;

// Lists up to this long are sorted by one CTA in shared memory.  On the GPU
// alone that is within a tenth of the launches per digit at 4,096 keys (a whole
// row gradient of 4,000 entries, 25 us and 23; of 8,000, 35 and 23); in a
// program that waits for its launches it saves three to five of them.
constexpr uint32_t kSortSmall = 4096, kSmallItems = kSortSmall / 1024;
constexpr uint32_t kSmallSmem = kSortSmall * 8u + 32u * 256u * 2u;

// Tiles whose counts each CTA of the scatter sums itself.  On the GPU alone that
// is ahead up to some 24 tiles (two digits of 24,576 keys 14.5 us and 16.3 with
// an offsets launch, of 65,536 keys 29.9 and 17.2); in a program that waits for
// its launches it saves one per digit (a training lookup of 30,011 ids 100 us and
// 104 to 107).
constexpr uint32_t kSumTiles = 64;

// Keys per tile.  Tiles of 4,096 are no faster for any list: two digits of 2^17
// keys take 17 us in tiles of 1,024 and 34 in those, 2^20 43 and 43, 2^24 470
// and 548.
constexpr int kSortItems = 4;
constexpr uint32_t kSortTile = kSortThreads * kSortItems;

// Scratch for any list of up to n keys.
struct SortScratch {
  uint32_t *keys0, *vals0, *keys1, *vals1, *hist, *total, *kept;
  uint32_t tiles;  // for which hist has room
  void carve(WorkCarver &w, uint32_t n) {
    tiles = (uint32_t)ceil_div(n, kSortTile);
    keys0 = w.take<uint32_t>(n);
    vals0 = w.take<uint32_t>(n);
    keys1 = w.take<uint32_t>(n);
    vals1 = w.take<uint32_t>(n);
    hist = w.take<uint32_t>(256ull * tiles);
    total = w.take<uint32_t>(256);
    kept = w.take<uint32_t>(1);
  }
};

// The sorted list: keys and positions, and their number (device).
struct SortedList {
  const uint32_t *keys, *vals, *kept;
};

// Key source of the digits after the first.
struct StoredKeys {
  const uint32_t *keys, *vals, *kept;
  static constexpr bool kFirst = false;
  __device__ __forceinline__ uint32_t count(uint32_t) const { return *kept; }
  __device__ __forceinline__ uint32_t key(uint32_t i) const { return keys[i]; }
  __device__ __forceinline__ uint32_t value(uint32_t i) const { return vals[i]; }
};

template <class Source>
__global__ void __launch_bounds__(kSortThreads)
sort_count(const Source src, uint32_t n, uint32_t none, uint32_t shift, uint32_t digit_mask,
           uint32_t *__restrict__ hist, uint32_t tiles) {
  after_previous();
  __shared__ uint32_t s_hist[256];
  s_hist[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t m = src.count(n), first = blockIdx.x * kSortTile + threadIdx.x;
  uint32_t key[kSortItems];
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const uint32_t at = first + i * kSortThreads;
    key[i] = at < m ? src.key(at) : none;
  }
#pragma unroll
  for (int i = 0; i < kSortItems; ++i)
    if (key[i] != none) atomicAdd(&s_hist[(key[i] >> shift) & digit_mask], 1u);
  __syncthreads();
  if (threadIdx.x <= digit_mask) hist[(size_t)threadIdx.x * tiles + blockIdx.x] = s_hist[threadIdx.x];
}

// Exclusive sum over the 256 threads of a CTA; `all` gets the total.
__device__ __forceinline__ uint32_t sort_cta_sum(uint32_t v, uint32_t *s_warp, uint32_t &all) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (uint32_t o = 1; o < 32u; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31u) s_warp[warp] = x;
  __syncthreads();
  uint32_t before = 0, sum = 0;
#pragma unroll
  for (uint32_t w = 0; w < kSortWarps; ++w) {
    const uint32_t s = s_warp[w];
    before += w < warp ? s : 0u;
    sum += s;
  }
  __syncthreads();
  all = sum;
  return before + x - v;
}

// One CTA per digit: its counts per tile become offsets within the digit.
static __global__ void __launch_bounds__(kSortThreads)
sort_offsets(uint32_t *__restrict__ hist, uint32_t tiles, uint32_t *__restrict__ total) {
  after_previous();
  __shared__ uint32_t s_warp[kSortWarps];
  uint32_t *h = hist + (size_t)blockIdx.x * tiles;
  uint32_t base = 0;
  for (uint32_t t0 = 0; t0 < tiles; t0 += kSortThreads) {
    const uint32_t t = t0 + threadIdx.x;
    uint32_t all;
    const uint32_t v = t < tiles ? h[t] : 0u;
    const uint32_t x = sort_cta_sum(v, s_warp, all);
    if (t < tiles) h[t] = base + x;
    base += all;
  }
  if (threadIdx.x == 0) total[blockIdx.x] = base;
}

template <class Source>
__global__ void __launch_bounds__(kSortThreads)
sort_scatter(const Source src, uint32_t n, uint32_t none, uint32_t shift, uint32_t digit_mask,
             const uint32_t *hist, uint32_t tiles,
             const uint32_t *total,  // null: hist holds counts, not offsets
             uint32_t *__restrict__ out_keys,
             uint32_t *__restrict__ out_vals, uint32_t *__restrict__ kept) {
  after_previous();
  __shared__ uint32_t s_count[kSortWarps][256];
  __shared__ uint32_t s_base[256], s_global[256], s_warp[kSortWarps];
  __shared__ uint32_t s_key[kSortTile], s_val[kSortTile];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
#pragma unroll
  for (uint32_t w = 0; w < kSortWarps; ++w) s_count[w][tid] = 0;
  const uint32_t m = src.count(n);
  // a warp's keys are consecutive, lanes first: the order the ranks keep
  const uint32_t first = blockIdx.x * kSortTile + warp * (32u * kSortItems) + lane;
  uint32_t key[kSortItems], val[kSortItems], rank[kSortItems];
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const uint32_t at = first + i * 32u;
    key[i] = at < m ? src.key(at) : none;
    val[i] = at < m ? src.value(at) : 0u;
  }
  __syncthreads();
  uint32_t *cnt = s_count[warp];
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const bool some = key[i] != none;
    const uint32_t d = some ? (key[i] >> shift) & digit_mask : 256u;
    const uint32_t peers = __match_any_sync(0xffffffffu, d);
    rank[i] = __popc(peers & ((1u << lane) - 1u));
    if (some) rank[i] += cnt[d];
    __syncwarp();
    if (some && (peers >> lane) == 1u) cnt[d] += __popc(peers);  // the last peer
    __syncwarp();
  }
  __syncthreads();
  // thread d: digit d's counts over the warps, its place in the tile and in
  // the output
  uint32_t sum = 0;
#pragma unroll
  for (uint32_t w = 0; w < kSortWarps; ++w) {
    const uint32_t c = s_count[w][tid];
    s_count[w][tid] = sum;
    sum += c;
  }
  uint32_t in_tile, all;
  const uint32_t base = sort_cta_sum(sum, s_warp, in_tile);
  uint32_t digits = 0, earlier = 0;  // thread d: keys of digit d, those of earlier tiles
  if (tid <= digit_mask) {
    const uint32_t *h = hist + (size_t)tid * tiles;
    if (total) {
      digits = total[tid];
      earlier = h[blockIdx.x];
    } else {
#pragma unroll 8
      for (uint32_t t = 0; t < tiles; ++t) {
        const uint32_t c = h[t];
        digits += c;
        earlier += t < blockIdx.x ? c : 0u;
      }
    }
  }
  const uint32_t before = sort_cta_sum(digits, s_warp, all);
  s_base[tid] = base;
  s_global[tid] = before + earlier;
  if (blockIdx.x == 0 && tid == 0 && Source::kFirst) *kept = all;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    if (key[i] == none) continue;
    const uint32_t d = (key[i] >> shift) & digit_mask;
    const uint32_t at = s_base[d] + cnt[d] + rank[i];
    s_key[at] = key[i];
    s_val[at] = val[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const uint32_t at = tid + i * kSortThreads;
    if (at >= in_tile) continue;
    const uint32_t k = s_key[at], d = (k >> shift) & digit_mask;
    const uint32_t to = s_global[d] + at - s_base[d];
    out_keys[to] = k;
    out_vals[to] = s_val[at];
  }
}

// All digits of a list of at most kSortSmall keys.
template <class Source>
__global__ void __launch_bounds__(1024)
sort_small(const Source src, uint32_t n, uint32_t none, uint32_t passes, uint32_t digit,
           uint32_t *__restrict__ out_keys, uint32_t *__restrict__ out_vals,
           uint32_t *__restrict__ kept) {
  after_previous();
  extern __shared__ uint32_t s_small[];
  uint32_t *s_key = s_small, *s_val = s_small + kSortSmall;
  uint16_t(*s_count)[256] = reinterpret_cast<uint16_t(*)[256]>(s_small + 2u * kSortSmall);
  __shared__ uint32_t s_base[256], s_warp[kSortWarps], s_m;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t dm = (1u << digit) - 1u;
  uint32_t key[kSmallItems], val[kSmallItems], rank[kSmallItems];
  const uint32_t first = warp * (32u * kSmallItems) + lane;
#pragma unroll
  for (uint32_t i = 0; i < kSmallItems; ++i) {
    const uint32_t at = first + i * 32u;
    key[i] = at < n ? src.key(at) : none;
    val[i] = at < n ? src.value(at) : 0u;
  }
  uint32_t m = n;
  for (uint32_t p = 0; p < passes; ++p) {
    const uint32_t shift = p * digit;
    if (p) {
#pragma unroll
      for (uint32_t i = 0; i < kSmallItems; ++i) {
        const uint32_t at = first + i * 32u;
        key[i] = at < m ? s_key[at] : none;
        val[i] = at < m ? s_val[at] : 0u;
      }
    }
    for (uint32_t x = tid; x < 32u * 256u / 2u; x += 1024u) reinterpret_cast<uint32_t *>(s_count)[x] = 0;
    __syncthreads();
    uint16_t *cnt = s_count[warp];
#pragma unroll
    for (uint32_t i = 0; i < kSmallItems; ++i) {
      const bool some = key[i] != none;
      const uint32_t d = some ? (key[i] >> shift) & dm : 256u;
      const uint32_t peers = __match_any_sync(0xffffffffu, d);
      rank[i] = __popc(peers & ((1u << lane) - 1u));
      if (some) rank[i] += cnt[d];
      __syncwarp();
      if (some && (peers >> lane) == 1u) cnt[d] += (uint16_t)__popc(peers);  // the last peer
      __syncwarp();
    }
    __syncthreads();
    if (tid < 256u) {  // (whole warps; the barriers of the sum are theirs)
      uint32_t sum = 0;
#pragma unroll 8
      for (uint32_t w = 0; w < 32u; ++w) {
        const uint32_t c = s_count[w][tid];
        s_count[w][tid] = (uint16_t)sum;
        sum += c;
      }
      uint32_t x = sum;
#pragma unroll
      for (uint32_t o = 1; o < 32u; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31u) s_warp[warp] = x;
      s_base[tid] = x - sum;
    }
    __syncthreads();
    if (tid < 256u) {
      uint32_t before = 0;
      for (uint32_t w = 0; w < warp; ++w) before += s_warp[w];
      s_base[tid] += before;
    }
    if (tid == 0) {
      uint32_t all = 0;
      for (uint32_t w = 0; w < kSortWarps; ++w) all += s_warp[w];
      s_m = all;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kSmallItems; ++i) {
      if (key[i] == none) continue;
      const uint32_t d = (key[i] >> shift) & dm, at = s_base[d] + cnt[d] + rank[i];
      s_key[at] = key[i];
      s_val[at] = val[i];
    }
    m = s_m;
    __syncthreads();
  }
  for (uint32_t at = tid; at < m; at += 1024u) {
    out_keys[at] = s_key[at];
    out_vals[at] = s_val[at];
  }
  if (tid == 0) *kept = m;
}

// Sorts the positions of src (n of them; keys below `none`, or `none` to be
// dropped; none > 0) in scratch carved for n keys or more.
template <class Source>
cudaError_t run_sort(const Source &src, uint32_t n, uint32_t none, const SortScratch &w,
                     SortedList *out, cudaStream_t st) {
  uint32_t bits = 1;
  while (bits < 32 && ((none - 1u) >> bits)) ++bits;
  const uint32_t passes = (bits + 7u) / 8u, digit = (bits + passes - 1u) / passes;
  const uint32_t tiles = (uint32_t)ceil_div(n, kSortTile);
  const uint32_t dm = (1u << digit) - 1u;
  if (n <= kSortSmall) {
    const cudaError_t err = opt_in<sort_small<Source>>(kSmallSmem);
    if (err) return err;
    *out = SortedList{w.keys1, w.vals1, w.kept};
    return launch_next(sort_small<Source>, 1, 1024, kSmallSmem, st, src, n, none, passes, digit,
                       w.keys1, w.vals1, w.kept);
  }
  if (tiles > w.tiles) return cudaErrorInvalidValue;
  const bool few = tiles <= kSumTiles;
  uint32_t *keys = w.keys0, *vals = w.vals0, *keys_next = w.keys1, *vals_next = w.vals1;
  for (uint32_t p = 0; p < passes; ++p) {
    const uint32_t shift = p * digit;
    const StoredKeys stored{keys, vals, w.kept};
    auto pass = [&](auto count, auto scatter, const auto &from) {
      cudaError_t err = launch_next(count, tiles, kSortThreads, 0, st, from, n, none, shift, dm,
                                    w.hist, tiles);
      if (!err && !few)
        err = launch_next(sort_offsets, dm + 1u, kSortThreads, 0, st, w.hist, tiles, w.total);
      if (!err)
        err = launch_next(scatter, tiles, kSortThreads, 0, st, from, n, none, shift, dm, w.hist,
                          tiles, few ? (uint32_t *)nullptr : w.total, keys_next, vals_next, w.kept);
      return err;
    };
    const cudaError_t err = p == 0 ? pass(sort_count<Source>, sort_scatter<Source>, src)
                                   : pass(sort_count<StoredKeys>, sort_scatter<StoredKeys>, stored);
    if (err) return err;
    std::swap(keys, keys_next);
    std::swap(vals, vals_next);
  }
  *out = SortedList{keys, vals, w.kept};
  return cudaSuccess;
}

// (one warp) First position in the ascending keys[0 .. n) whose key is >= v:
// 32 probes per step.
__device__ __forceinline__ uint32_t warp_lower_bound(const uint32_t *__restrict__ keys,
                                                     uint32_t n, uint32_t v) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t lo = 0, len = n;  // the answer lies in [lo, lo + len]
  while (len) {
    const uint32_t step = (len + 31u) / 32u;
    const uint32_t off = lane * step;  // probes lo, lo + step, ...
    const bool below = off < len && keys[lo + off] < v;
    const uint32_t c = __popc(__ballot_sync(0xffffffffu, below));
    if (c == 0) break;  // keys[lo] >= v
    // keys[lo + (c - 1) * step] < v, and the next probe, if any, is >= v
    const uint32_t from = (c - 1u) * step + 1u;
    const uint32_t to = min(len, c * step);
    lo += from;
    len = to - from;
  }
  return lo;
}

}  // namespace nsfps
