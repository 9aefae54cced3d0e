// nsfps_attention.cu -- attention over the blocks of keys chosen for each
// query, and its gradient.
//
// A query reads few keys, and neighbouring queries read the same ones, so the
// work is turned round: the keys are cut into spans of 256 consecutive keys (of
// 128 in the gradient), and every (query, span) pair that shares a key is
// sorted by span.  A CTA takes a run of pairs of one span, gathers their query
// rows into a matrix tile, and meets the span's keys once for all of them
// (tcgen05.mma on 16-bit operands, fp32 in tensor memory).  Each pair leaves a
// partial result in fp32 (its normalised output and log-sum-exp; in the
// gradient its share of dq), and a last kernel joins the partials of a query.
// No atomics in a sum: every partial has one writer, and the sort is stable, so
// dk and dv add up in one order.
//
// What bounds it: per pair and head the tile products cost 4 * D * keys
// operations against 8 * D bytes of partials (written and read), so the
// partials, the softmax and the way to the tiles, not the matrix unit, set the
// pace (its share of the time is 13 % forward, 15 % in the gradient).  Of a
// scan's 170 us (16,384 queries, 4 heads of 64, 512 of 122,880 keys each) the
// tiles take 107, the join 36 (132 MB of partials, 3.7 TB/s), the plan 33; the
// floor is 22 by bytes.  Spans of 128 keys make more pairs (186 us); spans of 512
// make that call 3 % faster, not enough for the second plan that the smaller
// calls would then want.
//
// A handful of queries does not fill tiles and would wait for the sort; they
// take a direct path, which splits each query's own keys over CTAs (mma.sync,
// whose 16-row tiles suit a query's few heads; the keys' bytes bound it).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nsfps_feature.cuh"
#include "nsfps_sort.cuh"
#include "nsfps_tmem.cuh"

namespace nsfps {
namespace {

constexpr uint32_t kFullMask = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnArgs {
  const char *q, *k, *v, *dout, *out_in, *rest_in;
  char *out, *rest, *dq, *dk, *dv;  // rest: may be null, as rest_in
  float *lse;              // forward: may be null
  const float *lse_in;
  const int64_t *blocks;
  const int32_t *lengths;  // or null
  uint32_t B, M, N, H, G, R, D;  // R = H / G query heads per key head
  uint32_t block_log2, top, nb;
  int64_t qs[3], ks[3], vs[3];   // element strides: batch, row, head
  float scale;
  // plan of the (query, span) pairs
  uint32_t nsb;            // spans per cloud
  const uint32_t *vals;    // sorted pairs: query * top + leading slot
  const uint32_t *mask;    // per query slot: blocks of the span that are listed
  const unsigned long long *lead;  // per query: bit s = slot s leads a pair
  const uint32_t *skeys;   // their sort keys: span, then the chunks read
  const uint4 *listed;     // per span: 16 bytes, 1 for each block that some query lists
  const uint4 *span;       // per span: first pair, end, first share, tiles
  const uint4 *tiles;      // by cost: (span, tile within it, first pair, pairs of the span)
  uint32_t tile_stride;    // places per cost class
  const uint32_t *tile_count;
  // waits: their limit; set when one ran out; a CTA that does not announce a
  // product (tests), or -1, and which
  unsigned long long wait_ns;
  uint32_t *gave_up;
  int hold_cta;
  uint32_t hold_step;
  // partials of key heads g0 .. g0 + gc - 1
  uint32_t g0, gc;
  float *part;             // [pair][gc * R][D]
  float *part_lse;         // [pair][gc * R], base 2
  float *delta;            // [query][H]
  uint32_t *most;          // [cloud][G][2], float bits: |dout|^2 and |delta| at most
  float *part_kv;          // [share][gc][2][span][D]
  // direct path: partials per query, rounds per partial, 16-row parts of R
  uint32_t splits, rounds, row_parts;
};

__device__ __forceinline__ uint32_t cloud_length(const int32_t *lengths, uint32_t b, uint32_t n) {
  return lengths ? (uint32_t)min(max(lengths[b], 0), (int)n) : n;
}

// ------------------------------------------------------------ matrix tiles

template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4],
                                                 uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&x);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 x = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&x);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// 16-byte asynchronous copy; zeros where `some` is false (the source is then
// not read).
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool some) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(some ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two at once: one instruction each.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;"
      : "=f"(d)
      : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

// Shared tiles of 16-bit rows of DP elements: byte offset of 16-byte chunk c
// of row r.  The chunks of a row are permuted by the row, so that the eight
// rows of a matrix load fall into different banks.
template <int DP>
__device__ __forceinline__ uint32_t tile_off(uint32_t r, uint32_t c) {
  if (DP == 32) return r * 64u + ((c ^ ((r >> 1) & 3u)) << 4);
  return r * (DP * 2u) + ((c ^ (r & 7u)) << 4);
}

// ------------------------------------------------------------- the plan

constexpr uint32_t kTileClasses = 5;  // of cost: 4 quarters .. 0

// Blocks (as bits of a pair's mask) of the 64-key chunk c of a span.
__device__ __forceinline__ uint32_t chunk_blocks(uint32_t c, uint32_t block_log2) {
  const uint32_t n = block_log2 >= 6u ? 1u : 64u >> block_log2;
  return ((1u << n) - 1u) << ((c << 6) >> block_log2);
}

// LANES lanes per query: which slots lead a pair, and the blocks of each pair.
// A pair's leading slot is the first slot that lists a block of its span; a
// repeated block sets the same bit again.  The sort key is the span and, as
// its place in a Gray code, the set of 64-key chunks that are read: neighbours
// in that order differ in few chunks, so the rows of a tile read alike.
template <int SLOTS, int LANES>  // slots per lane, LANES apart
__global__ void __launch_bounds__(256)
plan_pairs(const AttnArgs a, uint32_t span_log2, uint32_t *__restrict__ keys,
           uint32_t *__restrict__ mask, unsigned long long *__restrict__ lead,
           uint8_t *__restrict__ listed) {
  after_previous();
  const uint32_t lane = threadIdx.x & (LANES - 1u), here = (threadIdx.x & 31u) - lane;
  const uint32_t bm = blockIdx.x * (256u / LANES) + threadIdx.x / LANES;
  const bool some = bm < a.B * a.M;  // (all lanes of a warp take part in its shuffles)
  const uint32_t top = some ? a.top : 0u, b = some ? bm / a.M : 0u;
  const uint32_t len = cloud_length(a.lengths, b, a.N);
  const uint32_t live = (uint32_t)(((uint64_t)len + (1u << a.block_log2) - 1u) >> a.block_log2);
  const uint32_t in_log2 = span_log2 - a.block_log2;  // blocks per span, log2
  const uint32_t none = 0xffffffffu;
  uint32_t sb[SLOTS], bit[SLOTS], m[SLOTS], lead_of[SLOTS];
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const uint32_t s = lane + LANES * i;
    const int64_t j = s < top ? a.blocks[(uint64_t)bm * a.top + s] : -1;
    const bool use = j >= 0 && j < (int64_t)live;
    sb[i] = use ? (uint32_t)j >> in_log2 : none;
    bit[i] = use ? 1u << ((uint32_t)j & ((1u << in_log2) - 1u)) : 0u;
    m[i] = 0u;
    lead_of[i] = none;
    // (every query that lists the block stores the same byte)
    if (use) listed[16u * (b * a.nsb + sb[i]) + ((uint32_t)j & ((1u << in_log2) - 1u))] = 1u;
  }
#pragma unroll
  for (int part = SLOTS - 1; part >= 0; --part) {
    const uint32_t n = min((uint32_t)LANES, a.top > LANES * part ? a.top - LANES * part : 0u);
#pragma unroll 4
    for (uint32_t s = n; s-- > 0u;) {  // downwards: the last match is the first slot
      const uint32_t osb = __shfl_sync(kFullMask, sb[part], s, LANES);
      const uint32_t obit = __shfl_sync(kFullMask, bit[part], s, LANES);
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
        if (osb == sb[i]) {
          m[i] |= obit;
          lead_of[i] = s + LANES * part;
        }
    }
  }
  unsigned long long leaders = 0;
  const uint32_t chunks = 1u << (span_log2 - 6u);
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const uint32_t s = lane + LANES * i;
    const bool first = sb[i] != none && lead_of[i] == s;
    const uint32_t firsts = __ballot_sync(kFullMask, first) >> here;
    leaders |= (unsigned long long)(firsts & (kFullMask >> (32 - LANES))) << (LANES * i);
    if (s >= top) continue;
    uint32_t read = 0;
    for (uint32_t c = 0; c < chunks; ++c)
      read |= (m[i] & chunk_blocks(c, a.block_log2)) ? 1u << c : 0u;
    uint32_t rank = read;  // the inverse of r ^ (r >> 1), over up to 4 bits
    rank ^= rank >> 1;
    rank ^= rank >> 2;
    const uint64_t p = (uint64_t)bm * a.top + s;
    keys[p] = first ? ((b * a.nsb + sb[i]) << chunks) | rank : (a.B * a.nsb) << chunks;
    mask[p] = m[i];
  }
  if (some && lane == 0) lead[bm] = leaders;
}

// Keys of the sort: one per query slot, in slot order.
struct PairKeys {
  const uint32_t *keys;
  static constexpr bool kFirst = true;
  __device__ __forceinline__ uint32_t count(uint32_t n) const { return n; }
  __device__ __forceinline__ uint32_t key(uint32_t i) const { return keys[i]; }
  __device__ __forceinline__ uint32_t value(uint32_t i) const { return i; }
};

// One warp per span: its pairs, and its tiles of tile_rows rows (at least
// `least`), listed by cost.  CTAs take the tiles in turns, so with the dear
// ones first the turns come out even (the gradient of shared heads took 53 us
// unsorted, 38 sorted).  A tile's place in its class comes from a
// counter and differs from run to run; no result depends on it.  Spans of
// several tiles get places for their tiles' shares of dk and dv, in order.
__global__ void __launch_bounds__(256)
plan_spans(const SortedList list, uint32_t spans, uint32_t shift, uint32_t R, uint32_t tile_rows,
           uint32_t least, bool by_chunks, uint4 *__restrict__ span, uint4 *__restrict__ tiles,
           uint32_t tile_stride, uint32_t *__restrict__ tile_count) {
  after_previous();
  const uint32_t s = blockIdx.x * 8u + (threadIdx.x >> 5), lane = threadIdx.x & 31u;
  if (s >= spans) return;
  const uint32_t n = *list.kept;
  const uint32_t b = warp_lower_bound(list.keys, n, s << shift);
  const uint32_t e = b + warp_lower_bound(list.keys + b, n - b, (s + 1u) << shift);
  const uint32_t rows = (e - b) * R, count = max(least, (rows + tile_rows - 1u) / tile_rows);
  uint32_t first = 0;
  if (lane == 0 && count > 1u) first = atomicAdd(tile_count + kTileClasses, count);
  first = __shfl_sync(kFullMask, first, 0);
  if (lane == 0) span[s] = make_uint4(b, e, first, count);
  for (uint32_t i = lane; i < count; i += 32u) {
    const uint32_t r0 = i * tile_rows, r1 = min(rows, r0 + tile_rows);
    uint32_t cost = 0;  // 0 .. 4
    if (by_chunks && r0 < r1) {
      // the chunks between the Gray ranks of the first and the last row
      const uint32_t low = (1u << shift) - 1u;
      const uint32_t g0 = list.keys[b + r0 / R] & low, g1 = list.keys[b + (r1 - 1u) / R] & low;
      uint32_t read = 0;
      for (uint32_t g = g0; g <= g1; ++g) read |= g ^ (g >> 1);
      cost = __popc(read);
    } else if (r0 < r1) {
      cost = (4u * (r1 - r0) + tile_rows - 1u) / tile_rows;
    }
    const uint32_t c = kTileClasses - 1u - min(cost, kTileClasses - 1u);
    tiles[(uint64_t)c * tile_stride + atomicAdd(tile_count + c, 1u)] = make_uint4(s, i, b, e - b);
  }
}

// A span's marks as bits.
__device__ __forceinline__ uint32_t marked(const uint4 &x) {
  auto four = [](uint32_t y) { return (y * 0x10204080u) >> 28; };  // bytes of 0 or 1
  return four(x.x) | four(x.y) << 4 | four(x.z) << 8 | four(x.w) << 12;
}

// The tiles, dear ones first.
struct TileOrder {
  const uint4 *tiles;
  uint32_t stride, end[kTileClasses];
  __device__ __forceinline__ explicit TileOrder(const AttnArgs &a)
      : tiles(a.tiles), stride(a.tile_stride) {
    uint32_t sum = 0;
#pragma unroll
    for (uint32_t c = 0; c < kTileClasses; ++c) end[c] = sum += a.tile_count[c];
  }
  __device__ __forceinline__ uint32_t size() const { return end[kTileClasses - 1u]; }
  __device__ __forceinline__ uint4 operator[](uint32_t i) const {
    const uint4 *p = tiles + i;
#pragma unroll
    for (uint32_t c = 1; c < kTileClasses; ++c)
      if (i >= end[c - 1u]) p = tiles + ((uint64_t)c * stride + (i - end[c - 1u]));
    return *p;
  }
};

// -------------------------------------------------------------- forward

constexpr uint32_t kSpanLog2 = 8;      // keys per span of the forward pass
constexpr uint32_t kTileRows = 128;    // query rows per tile

// Copies keys [key0, key0 + ROWS) of one head into a shared tile; zeros behind
// the cloud's end and behind the head's elements.
template <int DP, int ROWS, int THREADS>
__device__ __forceinline__ void load_keys(uint32_t dst, const char *src, int64_t row_stride,
                                          uint32_t key0, uint32_t len, uint32_t D, uint32_t tid) {
  constexpr uint32_t kChunks = DP / 8;
#pragma unroll
  for (uint32_t i = tid; i < ROWS * kChunks; i += THREADS) {
    const uint32_t r = i / kChunks, c = i % kChunks;
    const bool some = key0 + r < len && c * 8u < D;
    copy16(dst + tile_off<DP>(r, c), some ? src + ((int64_t)(key0 + r) * row_stride + c * 8) * 2 : src,
           some);
  }
}

// The A fragments (16 rows x DP) of two query rows per lane, straight from
// memory.
template <int DP>
__device__ __forceinline__ void load_rows(uint32_t (&f)[DP / 16][4], const char *r0,
                                          const char *r1, uint32_t D, uint32_t t) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t d = kk * 16 + h * 8 + 2 * t;
      const bool in = d < D;
      f[kk][2 * h] = r0 && in ? *reinterpret_cast<const uint32_t *>(r0 + 2 * d) : 0u;
      f[kk][2 * h + 1] = r1 && in ? *reinterpret_cast<const uint32_t *>(r1 + 2 * d) : 0u;
    }
}

// What turns a raw score into base-2 exponents: exp2(s * c2).  The factor is
// kept positive, so that the maximum of the raw scores is that of the scaled
// ones: a negative scale flips the signs of q, a scale of zero makes q zero.
struct ScoreScale {
  float c2;
  uint32_t flip, keep;  // on two packed elements of q
  __device__ __forceinline__ explicit ScoreScale(float scale) {
    c2 = scale == 0.f ? 1.f : fabsf(scale) * kLog2e;
    flip = scale < 0.f ? 0x80008000u : 0u;
    keep = scale == 0.f ? 0u : 0xffffffffu;
  }
  template <int N>
  __device__ __forceinline__ void apply(uint32_t (&f)[N][4]) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) f[i][j] = (f[i][j] & keep) ^ flip;
  }
};

// Running softmax state and output of 16 rows (two per lane).
template <class T, int DP>
struct RowsState {
  float o[DP / 8][4];
  float mx[2], sum[2];  // maximum of the raw scores; this lane's share of the sum
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    mx[0] = mx[1] = -INFINITY;
    sum[0] = sum[1] = 0.f;
  }

  // 16 * KP keys at rows key_row.. of the tiles sk, sv; key0 is the first.
  // For its 16 keys kp: sel(kp) tells whether any row of the warp reads them,
  // all(kp) whether every one does, row(kp, h) whether row h of this lane
  // does.  Instructions per score, not the matrix products, are what this
  // costs, so the masks are looked at only where a warp's rows differ or the
  // cloud ends.  The weights are rounded to T for the product with v: half a
  // step of T each, as the output's own rounding.
  template <int KP, class Sel, class All, class Row>
  __device__ __forceinline__ void add(const uint32_t (&qf)[DP / 16][4], uint32_t sk, uint32_t sv,
                                      uint32_t key_row, uint32_t key0, uint32_t len, float c2,
                                      uint32_t lane, Sel sel, All all, Row row) {
    const uint32_t t = lane & 3u;
    float s[2 * KP][4];
    float nm[2] = {mx[0], mx[1]};
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      if (!sel(kp)) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) s[2 * kp][i] = s[2 * kp + 1][i] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t b[4];
        ldsm4(b, sk + tile_off<DP>(key_row + kp * 16 + (lane & 7u) + ((lane >> 4) << 3),
                                   kk * 2 + ((lane >> 3) & 1u)));
        mma16816<T>(s[2 * kp], qf[kk], b[0], b[1]);
        mma16816<T>(s[2 * kp + 1], qf[kk], b[2], b[3]);
      }
      if (!all(kp) || key0 + kp * 16 + 16u > len) {
        const bool r0 = row(kp, 0), r1 = row(kp, 1);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool in = (i < 2 ? r0 : r1) && key0 + kp * 16 + n * 8 + 2 * t + (i & 1) < len;
            s[2 * kp + n][i] = in ? s[2 * kp + n][i] : -INFINITY;
          }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          nm[h] = fmaxf(nm[h], fmaxf(s[2 * kp + n][2 * h], s[2 * kp + n][2 * h + 1]));
    }
    float base[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      nm[h] = fmaxf(nm[h], __shfl_xor_sync(kFullMask, nm[h], 1));
      nm[h] = fmaxf(nm[h], __shfl_xor_sync(kFullMask, nm[h], 2));
      base[h] = nm[h] == -INFINITY ? 0.f : nm[h] * c2;  // no key yet: exp2(-inf) = 0
    }
    if (__any_sync(kFullMask, nm[0] > mx[0] || nm[1] > mx[1])) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float c = exp2_fast(fmaf(mx[h], c2, -base[h]));
        mx[h] = nm[h];
        sum[h] *= c;
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) o[j][2 * h] *= c, o[j][2 * h + 1] *= c;
      }
    }
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      if (!sel(kp)) continue;
      uint32_t a[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float *x = s[2 * kp + n];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = exp2_fast(fmaf(x[i], c2, -base[i >> 1]));
        sum[0] += x[0] + x[1];
        sum[1] += x[2] + x[3];
        a[2 * n] = pack2<T>(x[0], x[1]);
        a[2 * n + 1] = pack2<T>(x[2], x[3]);
      }
#pragma unroll
      for (int jj = 0; jj < DP / 16; ++jj) {
        uint32_t b[4];
        ldsm4t(b, sv + tile_off<DP>(key_row + kp * 16 + (lane & 15u), jj * 2 + (lane >> 4)));
        mma16816<T>(o[2 * jj], a, b[0], b[1]);
        mma16816<T>(o[2 * jj + 1], a, b[2], b[3]);
      }
    }
  }

  // Sums over the lanes of a row, and the maximum in base 2.
  __device__ __forceinline__ void finish(float c2) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(kFullMask, sum[h], 1);
      sum[h] += __shfl_xor_sync(kFullMask, sum[h], 2);
      mx[h] *= c2;
    }
  }
};

// A tile of 128 rows against one span: thread r owns row r.  Per 64-key chunk
// that some row reads: s = q k^T (128 x 64) by the tensor core into tensor
// memory, the thread takes its row's scores out, makes the weights, puts them
// back as 16-bit values over the scores, and o += p v takes them from there.
// Nothing but the operands' tiles passes through shared memory.  Four CTAs an
// SM (two with heads of 128): while one waits for its products or its loads,
// the others compute.  Smaller heads go through tiles of 64 elements, zeros
// behind their own (the scan's tiles take 92 us with heads of 16, 94 with 32, 99
// with 48, 105 with 64; 190 with 96, 228 with 128): the softmax does not depend
// on them.  A scan's 5,104 tiles take 107 us, 4,200 cycles each and
// SM, of which the instructions of the softmax and the loads are 45 %; with
// mma.sync and scores in registers it was 182.
constexpr uint32_t kTileThreads = 128;

// The reference maximum moves only when a row's maximum outgrows it by this
// much (in base 2): weights up to 2^8 sum exactly as well, and the output in
// tensor memory is rescaled about once per tile instead of once per chunk.
constexpr float kLazy = 8.f;

template <int DP>  // 64 or 128
struct TileShape {
  static constexpr uint32_t kQ = kTileRows * DP * 2u, kChunk = 64u * DP * 2u;
  static constexpr uint32_t kSmem = kQ + 4u * kChunk + 1024u;  // two chunks of k and v
  static constexpr uint32_t kTmem = DP == 64 ? 128u : 256u;    // scores, then output
  static constexpr uint32_t kCtas = DP == 64 ? 4 : 2;          // per SM
};

// ROWS rows of DP elements into shared tiles of 64 columns each; src(r) gives
// the row (null: zeros).
template <int DP, uint32_t ROWS, uint32_t THREADS, class Src>
__device__ __forceinline__ void load_rows_by(uint32_t dst, uint32_t D, uint32_t tid,
                                             const char *any, Src src) {
  constexpr uint32_t kChunks = DP / 8, kStep = THREADS / kChunks;
  const uint32_t c = tid % kChunks, r0 = tid / kChunks;
  const uint32_t at = dst + (c >> 3) * (ROWS * 128u) + swizzled(r0, c & 7u);
  const bool in = c * 8u < D;
#pragma unroll
  for (uint32_t i = 0; i < ROWS / kStep; ++i) {  // (kStep is a multiple of 8 rows)
    const char *p = src(r0 + i * kStep);
    const bool some = p && in;
    copy16(at + i * kStep * 128u, some ? p + c * 16u : any, some);
  }
}

// The same for keys `stride` bytes apart: those below `live` of the blocks that
// `blocks` names (bit r >> block_log2), zeros for the others.  Whatever lies in
// a block that no query lists meets weights of zero, and must not be a NaN.
template <int DP, uint32_t ROWS, uint32_t THREADS>
__device__ __forceinline__ void load_strided(uint32_t dst, uint32_t D, uint32_t tid,
                                             const char *first, int64_t stride, uint32_t live,
                                             uint32_t blocks, uint32_t block_log2) {
  const uint32_t n = ROWS >> block_log2, every = n ? (1u << n) - 1u : 1u;
  const bool all = (blocks & every) == every;
  constexpr uint32_t kChunks = DP / 8, kStep = THREADS / kChunks;
  const uint32_t c = tid % kChunks, r0 = tid / kChunks;
  const uint32_t at = dst + (c >> 3) * (ROWS * 128u) + swizzled(r0, c & 7u);
  const char *p = first + (int64_t)r0 * stride + c * 16u;
  const bool in = c * 8u < D;
#pragma unroll
  for (uint32_t i = 0; i < ROWS / kStep; ++i) {
    const uint32_t r = r0 + i * kStep;
    const bool some = in && r < live && (all || ((blocks >> (r >> block_log2)) & 1u));
    copy16(at + i * kStep * 128u, some ? p : first, some);
    p += (int64_t)kStep * stride;
  }
}

// Eight accumulators times f: 32 bytes, a whole sector per thread.
__device__ __forceinline__ void store8(float *to, const uint32_t *x, float f) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(x[i]) * f;
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "f"(y[0]), "f"(y[1]),
               "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7])
               : "memory");
}

template <class T, int DP>
__global__ void __launch_bounds__(kTileThreads, TileShape<DP>::kCtas)
attend_tiles(const AttnArgs a) {
  after_previous();
  using Shape = TileShape<DP>;
  extern __shared__ char smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[3];
  __shared__ uint32_t s_tmem, s_any[4];
  __shared__ volatile uint32_t s_gave_up;
  __shared__ const char *s_q[kTileRows];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = warp_value(tid >> 5);
  const uint32_t sq = (smem_u32(smem_raw) + 1023u) & ~1023u;  // the swizzle's pattern
  const uint32_t sk = sq + Shape::kQ, sv = sk + 2u * Shape::kChunk;
  const uint32_t bar_s = smem_u32(&s_bar[0]), bar_o = smem_u32(&s_bar[1]);
  const uint32_t bar_end = smem_u32(&s_bar[2]);
  constexpr uint32_t kChunkBits = 1u << (kSpanLog2 - 6u);
  if (warp == 0) tmem_alloc<Shape::kTmem>(smem_u32(&s_tmem));
  if (tid == 0) {
    bar_init(bar_s);
    bar_init(bar_o);
    bar_init(bar_end);
    s_gave_up = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  const uint32_t tm = warp_value(s_tmem), tm_s = tm, tm_o = tm + 64u;
  const uint32_t my = (warp * 32u) << 16;  // this warp's lanes
  constexpr uint32_t kScores = mma_desc<T>(128, 64, false, false);
  constexpr uint32_t kOutput = mma_desc<T>(128, DP, false, true);
  const float c2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  const float sign = a.scale == 0.f ? 0.f : a.scale < 0.f ? -1.f : 1.f;
  uint32_t phase = 0;     // of both barriers: each completes once per chunk
  // A thread whose wait runs out goes on without waiting, so that the CTA ends;
  // what it overwrites may be in use, for any row of its tiles.  So the mark is
  // for the whole turn, and the join gives NaN.
  bool failed = false;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (failed || bar_wait(bar, parity, a.wait_ns)) return;
    failed = true;
    *(volatile uint32_t *)a.gave_up = 1u;
    s_gave_up = 1u;
  };
  const TileOrder order(a);
  const uint32_t work = order.size() * a.gc;
  // What this thread's row of a tile is: asked for one tile ahead, the tile
  // itself two, as each waits for the one before.
  struct Row {
    uint32_t pair, head, read;
    bool live;
    uint32_t listed;  // of the tile's span
  };
  auto row_of = [&](const uint4 &tile) {
    Row x{0xffffffffu, 0u, 0u, false, 0u};
    if (tile.w) x.listed = marked(a.listed[tile.x]);
    const uint32_t r = tile.y * kTileRows + tid;
    x.live = r < tile.w * a.R;
    if (x.live) {
      const uint32_t e = r / a.R;
      x.head = r - e * a.R;
      x.pair = a.vals[tile.z + e];
      x.read = a.skeys[tile.z + e];
    }
    return x;
  };
  const uint32_t step = gridDim.x;
  uint4 tile = make_uint4(0u, 0u, 0u, 0u), tile_next = tile;
  if (blockIdx.x < work) tile = order[blockIdx.x / a.gc];
  if (blockIdx.x + step < work) tile_next = order[(blockIdx.x + step) / a.gc];
  Row mine = row_of(tile);
  struct Tile {
    uint32_t gi, key0, len, listed, todo;  // todo: chunks that some row reads
    const char *kh, *vh;
    uint32_t pair, head, mask;             // this thread's row
    bool live;
  };
  // Takes the next tile: puts its rows' places and chunks into shared memory
  // (todo is known behind a barrier) and asks for the one after it.
  auto open = [&](uint32_t w) {
    Tile x;
    const uint32_t b = tile.x / a.nsb, g = a.g0 + w % a.gc;
    x.gi = w % a.gc;
    x.key0 = (tile.x - b * a.nsb) << kSpanLog2;
    x.len = cloud_length(a.lengths, b, a.N);
    x.listed = mine.listed;
    x.kh = a.k + 2 * ((int64_t)b * a.ks[0] + (int64_t)g * a.ks[2]);
    x.vh = a.v + 2 * ((int64_t)b * a.vs[0] + (int64_t)g * a.vs[2]);
    x.pair = mine.pair;
    x.head = mine.head;
    x.live = mine.live;
    x.mask = 0u;
    uint32_t read = mine.read & ((1u << kChunkBits) - 1u);
    read ^= read >> 1;  // from the place in the Gray code
    const char *q = nullptr;
    if (x.live) {
      x.mask = a.mask[x.pair];
      const uint32_t m = x.pair / a.top - b * a.M;
      q = a.q + 2 * ((int64_t)b * a.qs[0] + (int64_t)m * a.qs[1] +
                     (int64_t)(g * a.R + x.head) * a.qs[2]);
    }
    read = __reduce_or_sync(kFullMask, read);
    if (lane == 0) s_any[warp] = read;
    s_q[tid] = q;
    tile = tile_next;
    mine = row_of(tile);
    if (w + 2u * step < work) tile_next = order[(w + 2u * step) / a.gc];
    return x;
  };
  auto fetch = [&](const Tile &x, uint32_t c, uint32_t buf, bool some) {
    if (some) {
      const uint32_t key = x.key0 + c * 64u, live = key < x.len ? x.len - key : 0u;
      const uint32_t blocks = x.listed >> ((c * 64u) >> a.block_log2);
      const int64_t ks = a.ks[1] * 2, vs = a.vs[1] * 2;
      // (a chunk wholly behind the end reads nothing, but its address is formed)
      load_strided<DP, 64, kTileThreads>(sk + buf * Shape::kChunk, a.D, tid,
                                         x.kh + (live ? (int64_t)key * ks : 0), ks, live, blocks,
                                         a.block_log2);
      load_strided<DP, 64, kTileThreads>(sv + buf * Shape::kChunk, a.D, tid,
                                         x.vh + (live ? (int64_t)key * vs : 0), vs, live, blocks,
                                         a.block_log2);
    }
    copy_commit();
  };
  // (behind a barrier) the tile's q and first chunk, one group; then the second
  uint32_t ahead = 0;  // chunks not yet asked for
  auto load_first = [&](Tile &x, uint32_t buf) {
    x.todo = warp_value(s_any[0] | s_any[1] | s_any[2] | s_any[3]);
    ahead = x.todo;
    load_rows_by<DP, kTileRows, kTileThreads>(sq, a.D, tid, a.q, [&](uint32_t r) { return s_q[r]; });
    fetch(x, __ffs(ahead) - 1, buf, ahead != 0);
    ahead &= ahead - 1u;
  };
  auto load_second = [&](const Tile &x, uint32_t buf) {
    fetch(x, __ffs(ahead) - 1, buf, ahead != 0);
    ahead &= ahead - 1u;
  };
  Tile now{}, coming{};
  uint32_t buf = 0;  // of the chunk at hand
  if (blockIdx.x < work) {
    now = open(blockIdx.x);
    __syncthreads();
    load_first(now, 0u);
    load_second(now, 1u);
  }
  for (uint32_t w = blockIdx.x; w < work; w += step) {
    const bool another = w + step < work;
    const uint32_t key0 = now.key0, len = now.len, mask = now.mask;
    const uint32_t warp_any = __reduce_or_sync(kFullMask, mask);
    const uint32_t warp_all = __reduce_and_sync(kFullMask, now.live ? mask : ~0u);
    float ref = -INFINITY, sum = 0.f;  // reference maximum of the signed raw scores
    for (uint32_t i = 0; now.todo; ++i) {
      const uint32_t c = __ffs(now.todo) - 1;
      now.todo &= now.todo - 1u;
      if (i) {
        // the chunk before is used up: its buffers take the next but one
        buf ^= 1u;
        wait(bar_o, phase ^ 1u);
        __syncwarp();
        tmem_after_sync();
        load_second(now, buf ^ 1u);
      }
      copy_wait<1>();
      smem_to_mma();
      tmem_before_sync();
      __syncthreads();
      if (warp == 0) {
        tmem_after_sync();
        const uint64_t q_desc = tile_desc(sq, 16u), k_desc = tile_desc(sk + buf * Shape::kChunk, 16u);
#pragma unroll
        for (uint32_t kk = 0; kk < DP / 16; ++kk)
          mma_ss(tm_s, further(q_desc, (kk >> 2) * (kTileRows * 128u) + (kk & 3u) * 32u),
                 further(k_desc, (kk >> 2) * (64u * 128u) + (kk & 3u) * 32u), kScores, kk != 0u);
        if (a.hold_cta != (int)blockIdx.x || a.hold_step || w != blockIdx.x || i)
          mma_commit(bar_s);
      }
      __syncwarp();
      wait(bar_s, phase);
      __syncwarp();
      tmem_after_sync();
      uint32_t s[2][32];
      tmem_ld32(s[0], tm_s + my);
      tmem_ld32(s[1], tm_s + my + 32u);
      tmem_ld_wait();
      // scores that the row does not read are -inf; 16 keys that no row of the
      // warp reads are not looked at
      float mx = -INFINITY;
      auto bit = [&](uint32_t x) { return (c * 64u + x * 16u) >> a.block_log2; };
#pragma unroll
      for (uint32_t x = 0; x < 4u; ++x) {
        if (!((warp_any >> bit(x)) & 1u)) continue;
        uint32_t *v = &s[x >> 1][(x & 1u) * 16u];
        const uint32_t key = key0 + c * 64u + x * 16u;
        if (sign != 1.f) {
#pragma unroll
          for (uint32_t y = 0; y < 16u; ++y) v[y] = __float_as_uint(__uint_as_float(v[y]) * sign);
        }
        if (!((warp_all >> bit(x)) & 1u) || key + 16u > len) {
          const uint32_t n = (mask >> bit(x)) & 1u && key < len ? len - key : 0u;
#pragma unroll
          for (uint32_t y = 0; y < 16u; ++y) v[y] = y < n ? v[y] : 0xff800000u;
        }
        // a tree: a chain of maxima would wait for each
        float m0 = max3(v[0], v[1], v[2]), m1 = max3(v[3], v[4], v[5]);
        float m2 = max3(v[6], v[7], v[8]), m3 = max3(v[9], v[10], v[11]);
        m0 = fmaxf(m0, max3(v[12], v[13], v[14]));
        m1 = fmaxf(m1, __uint_as_float(v[15]));
        mx = fmaxf(mx, fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)));
      }
      // A row whose first keys these are has nothing to rescale; without a key
      // the reference stays -inf and the weights come out 0.
      const bool grow = mx * c2 > ref * c2 + kLazy;
      const float next = grow ? mx : ref;
      const float base = next == -INFINITY ? 0.f : next * c2;
      if (__any_sync(kFullMask, grow && ref != -INFINITY)) {
        const float f = ref == -INFINITY ? 0.f : exp2_fast(fmaf(ref, c2, -base));
        sum *= f;
#pragma unroll 1
        for (uint32_t j = 0; j < DP / 16; ++j) {
          uint32_t o[16];
          tmem_ld16(o, tm_o + my + j * 16u);
          tmem_ld_wait();
#pragma unroll
          for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
          tmem_st16(tm_o + my + j * 16u, o);
        }
      }
      ref = next;
      // weights, rounded to T for the product with v: half a step of T each,
      // like the output's own rounding
      float2 part[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
      const float2 scale2 = make_float2(c2, c2), base2 = make_float2(-base, -base);
#pragma unroll
      for (uint32_t x = 0; x < 4u; ++x) {
        const uint32_t *v = &s[x >> 1][(x & 1u) * 16u];
        uint32_t *p = &s[0][x * 8u];  // the packed weights move up over the scores
        if ((warp_any >> bit(x)) & 1u) {
#pragma unroll
          for (uint32_t y = 0; y < 16u; y += 2) {
            float2 f = fma2(make_float2(__uint_as_float(v[y]), __uint_as_float(v[y + 1])), scale2,
                            base2);
            f.x = exp2_fast(f.x);
            f.y = exp2_fast(f.y);
            part[(y / 2u) & 3u] = add2(part[(y / 2u) & 3u], f);
            p[y / 2u] = pack2<T>(f.x, f.y);
          }
        } else {
#pragma unroll
          for (uint32_t y = 0; y < 8u; ++y) p[y] = 0u;
        }
      }
      part[0] = add2(add2(part[0], part[1]), add2(part[2], part[3]));
      sum += part[0].x + part[0].y;
      tmem_st32(tm_s + my, s[0]);
      const bool last = another && !now.todo;
      if (last) coming = open(w + step);
      tmem_st_wait();
      tmem_before_sync();
      __syncthreads();
      if (warp == 0) {
        tmem_after_sync();
        const uint64_t v_desc = tile_desc(sv + buf * Shape::kChunk, 64u * 128u);
#pragma unroll
        for (uint32_t kk = 0; kk < 4u; ++kk)
          mma_ts(tm_o, tm_s + kk * 8u, further(v_desc, kk * 2048u), kOutput, i != 0u || kk != 0u);
        mma_commit(bar_o);
      }
      __syncwarp();
      phase ^= 1u;
      // the next tile's loads go before this one's results: q is used up, and
      // so is the other buffer
      if (last) load_first(coming, buf ^ 1u);
    }
    wait(bar_o, phase ^ 1u);
    __syncwarp();
    tmem_after_sync();
    if (another) load_second(coming, buf);
    buf ^= 1u;
    const bool live_row = now.live;
    const uint64_t row = (uint64_t)now.pair * (a.gc * a.R) + now.gi * a.R + now.head;
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (uint32_t j = 0; j < DP / 32; ++j) {
      uint32_t o[32];
      tmem_ld32(o, tm_o + my + j * 32u);
      tmem_ld_wait();
      if (live_row)
#pragma unroll
        for (uint32_t y = 0; y < 32u; y += 8u)
          if (j * 32u + y < a.D) store8(a.part + row * a.D + j * 32u + y, &o[y], inv);
      __syncwarp();
    }
    if (live_row) a.part_lse[row] = sum > 0.f ? fmaf(ref, c2, log2f(sum)) : -INFINITY;
    now = coming;  // (the output is read before the barriers of the next chunk)
  }
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  if (warp == 0) {
    if (s_gave_up) {  // nothing may write tensor memory that is given back
      mma_commit(bar_end);
      bar_wait(bar_end, 0u, a.wait_ns);
      __syncwarp();
    }
    tmem_free<Shape::kTmem>(tm);
  }
}

// Four consecutive elements of the output, rounded, and what the rounding left.
template <class T>
__device__ __forceinline__ void store_out(const AttnArgs &a, uint64_t at, float4 x) {
  const uint2 y = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
  *reinterpret_cast<uint2 *>(a.out + at * 2) = y;
  if (!a.rest) return;
  const T *e = reinterpret_cast<const T *>(&y);
  *reinterpret_cast<uint2 *>(a.rest + at * 2) =
      make_uint2(pack2<T>(x.x - to_f32(e[0]), x.y - to_f32(e[1])),
                 pack2<T>(x.z - to_f32(e[2]), x.w - to_f32(e[3])));
}

// In the joins.  (Asked for at their beginning, and as a volatile, it took 1 us
// of each.)
__device__ __forceinline__ bool some_gave_up(const AttnArgs &a) { return *a.gave_up != 0u; }

// Joins a query's partials: out = sum_s w_s o_s, w_s = exp2(lse_s - lse), over
// its leading slots.  A warp takes 128 consecutive elements of a query's heads,
// four per lane: the slots are the same for all lanes, and what a slot's
// partial holds of them is consecutive too.  A scan's 132 MB of partials, read
// in the queries' order, take 36 us (the logs and the weights in a pass of their
// own first: 42).
constexpr int kJoinFlight = 8;  // partials in flight per lane

template <class T>
__global__ void __launch_bounds__(256)
attend_join(const AttnArgs a, uint32_t parts) {
  after_previous();
  const uint32_t lane = threadIdx.x & 31u, hc = a.gc * a.R;
  const uint64_t w = (uint64_t)blockIdx.x * 8u + (threadIdx.x >> 5);
  const uint32_t bm = (uint32_t)(w / parts);
  if (bm >= a.B * a.M) return;
  const uint32_t d = (uint32_t)(w - (uint64_t)bm * parts) * 128u + lane * 4u;
  if (d >= hc * a.D) return;
  const uint32_t hh = d / a.D;
  const unsigned long long lead = a.lead[bm];
  const float *lse = a.part_lse + (uint64_t)bm * a.top * hc + hh;
  const float *part = a.part + (uint64_t)bm * a.top * hc * a.D + d;
  const uint64_t step = (uint64_t)hc * a.D;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float mx = -INFINITY, total = 0.f;  // the sums so far are relative to mx
  for (unsigned long long l = lead; l;) {
    float c[kJoinFlight];
    float4 x[kJoinFlight];
    float next = mx;
#pragma unroll
    for (int u = 0; u < kJoinFlight; ++u) {
      const uint32_t s = l ? __ffsll(l) - 1 : 0u;
      c[u] = l ? lse[(uint64_t)s * hc] : -INFINITY;
      x[u] = l ? __ldcs(reinterpret_cast<const float4 *>(part + s * step))
               : make_float4(0.f, 0.f, 0.f, 0.f);
      l &= l - 1ull;
    }
#pragma unroll
    for (int u = 0; u < kJoinFlight; ++u) next = fmaxf(next, c[u]);
    const float base = next == -INFINITY ? 0.f : next, old = exp2_fast(mx - base);
    mx = next;
    total *= old;
    acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
    for (int u = 0; u < kJoinFlight; ++u) {
      const float y = exp2_fast(c[u] - base);
      total += y;
      acc.x += y * x[u].x; acc.y += y * x[u].y; acc.z += y * x[u].z; acc.w += y * x[u].w;
    }
  }
  const bool gave_up = some_gave_up(a);
  const float inv = gave_up ? NAN : total > 0.f ? 1.f / total : 0.f;
  const uint64_t out = ((uint64_t)bm * a.H + a.g0 * a.R) * a.D + d;
  store_out<T>(a, out, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  if (a.lse && d == hh * a.D)
    a.lse[(uint64_t)bm * a.H + a.g0 * a.R + hh] =
        gave_up ? NAN : total > 0.f ? (mx + log2f(total)) * kLn2 : -INFINITY;
}

// The same for the direct path, one CTA per row: groups of LANES lanes take
// the splits in turns, and their sums meet in shared memory.
template <class T, int LANES>
__global__ void __launch_bounds__(256)
attend_join_direct(const AttnArgs a) {
  after_previous();
  constexpr uint32_t kGroups = 256 / LANES;
  __shared__ float s_mx[8];
  __shared__ float4 s_acc[kGroups][LANES];
  __shared__ float s_total[kGroups];
  const uint32_t tid = threadIdx.x, sub = tid & (LANES - 1u), grp = tid / LANES;
  const uint64_t row = blockIdx.x, first = row * a.splits;
  float mx = -INFINITY;
  for (uint32_t s = tid; s < a.splits; s += 256u) mx = fmaxf(mx, a.part_lse[first + s]);
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, o));
  if ((tid & 31u) == 0) s_mx[tid >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) mx = fmaxf(mx, s_mx[w]);
  const float base = mx == -INFINITY ? 0.f : mx;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
#pragma unroll 4
  for (uint32_t s = grp; s < a.splits; s += kGroups) {
    const float w = exp2_fast(a.part_lse[first + s] - base);
    total += w;
    if (4u * sub < a.D) {
      const float4 x = *reinterpret_cast<const float4 *>(a.part + (first + s) * a.D + 4 * sub);
      acc.x += w * x.x; acc.y += w * x.y; acc.z += w * x.z; acc.w += w * x.w;
    }
  }
  s_acc[grp][sub] = acc;
  if (sub == 0) s_total[grp] = total;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (uint32_t g = 1; g < kGroups; ++g) {
    const float4 x = s_acc[g][sub];
    acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    total += s_total[g];
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  if (4u * sub < a.D)
    store_out<T>(a, row * a.D + 4 * sub,
                 make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  if (a.lse && sub == 0) a.lse[row] = total > 0.f ? (mx + log2f(total)) * kLn2 : -INFINITY;
}

// Direct path: a CTA takes `rounds` times kDirectKeys of one query's listed
// keys and one key head, the next round's keys in flight; each warp has 16 of
// a round's keys.  The warps' rows meet in shared memory at the end.
constexpr uint32_t kDirectKeys = 64;
constexpr uint32_t kDirectWarps = 4;

template <int DP>
struct DirectShape {
  static constexpr uint32_t kSlice = 16u * DP * 2u;            // k or v of a warp's round
  static constexpr uint32_t kTiles = kDirectWarps * 4u * kSlice;  // two rounds
  static constexpr uint32_t kJoin = kDirectWarps * 16u * DP * 4u;
  // (the join lies over the tiles)
  static constexpr uint32_t kSmem = kTiles > kJoin ? kTiles : kJoin;
};

template <class T, int DP>
__global__ void __launch_bounds__(kDirectWarps * 32)
attend_direct(const AttnArgs a) {
  after_previous();
  using Shape = DirectShape<DP>;
  extern __shared__ __align__(128) char smem[];
  __shared__ float s_stat[kDirectWarps][2][16];
  __shared__ int64_t s_list[64];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t split = blockIdx.x, bm = blockIdx.y;
  const uint32_t g = blockIdx.z / a.row_parts, h0 = (blockIdx.z % a.row_parts) * 16u;
  const uint32_t b = bm / a.M, m = bm - b * a.M;
  const uint32_t len = cloud_length(a.lengths, b, a.N);
  const char *kh = a.k + 2 * ((int64_t)b * a.ks[0] + (int64_t)g * a.ks[2]);
  const char *vh = a.v + 2 * ((int64_t)b * a.vs[0] + (int64_t)g * a.vs[2]);
  const uint32_t tiles = smem_u32(smem) + warp * 4u * Shape::kSlice;
  if (tid < 64u) s_list[tid] = tid < a.top ? a.blocks[(uint64_t)bm * a.top + tid] : -1;
  uint32_t qf[DP / 16][4];
  {
    const char *qrow[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t hh = h0 + (lane >> 2) + 8u * h;
      qrow[h] = hh < a.R ? a.q + 2 * ((int64_t)b * a.qs[0] + (int64_t)m * a.qs[1] +
                                      (int64_t)(g * a.R + hh) * a.qs[2])
                         : nullptr;
    }
    load_rows<DP>(qf, qrow[0], qrow[1], a.D, lane & 3u);
  }
  const ScoreScale sc(a.scale);
  sc.apply(qf);
  __syncthreads();

  // the warp's first key of round i, or none
  constexpr uint32_t kNone = 0xffffffffu;
  auto key_of = [&](uint32_t i) {
    const uint32_t at = (split * a.rounds + i) * kDirectKeys + warp * 16u;  // of the listed keys
    const uint32_t s = at >> a.block_log2;
    if (i >= a.rounds || s >= a.top) return kNone;
    const int64_t j = s_list[s];
    // an entry that an earlier slot holds already counts for nothing
    const bool again = __any_sync(kFullMask, (lane < s && s_list[lane] == j) ||
                                                 (lane + 32u < s && s_list[lane + 32u] == j));
    if (again || j < 0 || j >= (int64_t)a.nb) return kNone;
    const uint32_t key = ((uint32_t)j << a.block_log2) + (at & ((1u << a.block_log2) - 1u));
    return key < len ? key : kNone;
  };
  auto fetch = [&](uint32_t i) {
    const uint32_t key = key_of(i), to = tiles + (i & 1u) * 2u * Shape::kSlice;
    if (key != kNone) {
      load_keys<DP, 16, 32>(to, kh, a.ks[1], key, len, a.D, lane);
      load_keys<DP, 16, 32>(to + Shape::kSlice, vh, a.vs[1], key, len, a.D, lane);
    }
    copy_commit();
    return key;
  };
  RowsState<T, DP> st;
  st.clear();
  uint32_t key = fetch(0);
  for (uint32_t i = 0; i < a.rounds; ++i) {
    const uint32_t next = fetch(i + 1u);
    copy_wait<1>();
    __syncwarp();
    if (key != kNone) {
      const uint32_t at = tiles + (i & 1u) * 2u * Shape::kSlice;
      st.template add<1>(qf, at, at + Shape::kSlice, 0u, key, len, sc.c2, lane,
                         [](int) { return true; }, [](int) { return true; },
                         [](int, int) { return true; });
    }
    __syncwarp();
    key = next;
  }
  copy_wait<0>();
  st.finish(sc.c2);
  const uint32_t t = lane & 3u;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (t == 0) {
      s_stat[warp][0][(lane >> 2) + 8 * h] = st.mx[h];
      s_stat[warp][1][(lane >> 2) + 8 * h] = st.sum[h];
    }
  __syncthreads();  // statistics written, and every warp is done with its tiles
  float *s_o = reinterpret_cast<float *>(smem);  // [warp][16][DP]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t r = (lane >> 2) + 8u * h;
    if (h0 + r >= a.R) continue;
    float mx = -INFINITY;
    for (uint32_t w = 0; w < kDirectWarps; ++w) mx = fmaxf(mx, s_stat[w][0][r]);
    const float c = st.mx[h] == -INFINITY ? 0.f : exp2_fast(st.mx[h] - mx);
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
      *reinterpret_cast<float2 *>(s_o + (warp * 16u + r) * DP + j * 8 + 2 * t) =
          make_float2(st.o[j][2 * h] * c, st.o[j][2 * h + 1] * c);
  }
  __syncthreads();
  const uint32_t live = min(16u, a.R - h0);
  for (uint32_t i = tid; i < live * (DP / 4); i += kDirectWarps * 32) {
    const uint32_t r = i / (DP / 4), d = (i % (DP / 4)) * 4;
    if (d >= a.D) continue;
    float mx = -INFINITY, sum = 0.f;
    for (uint32_t w = 0; w < kDirectWarps; ++w) mx = fmaxf(mx, s_stat[w][0][r]);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t w = 0; w < kDirectWarps; ++w) {
      if (s_stat[w][0][r] == -INFINITY) continue;
      sum += s_stat[w][1][r] * exp2_fast(s_stat[w][0][r] - mx);
      const float4 y = *reinterpret_cast<const float4 *>(s_o + (w * 16u + r) * DP + d);
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const uint64_t row = (uint64_t)bm * a.H + g * a.R + h0 + r;
    if (a.splits == 1u) {
      store_out<T>(a, row * a.D + d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
      if (a.lse && d == 0) a.lse[row] = sum > 0.f ? (mx + log2f(sum)) * kLn2 : -INFINITY;
    } else {
      *reinterpret_cast<float4 *>(a.part + (row * a.splits + split) * a.D + d) =
          make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
      if (d == 0) a.part_lse[row * a.splits + split] = sum > 0.f ? mx + log2f(sum) : -INFINITY;
    }
  }
}

// -------------------------------------------------------------- gradient

// Whether a query reads one key: the first of the cloud's last block, alone.
__device__ __forceinline__ bool one_key(const AttnArgs &a, uint32_t bm) {
  const unsigned long long lead = a.lead[bm];
  if (__popcll(lead) != 1) return false;
  const uint64_t slot = (uint64_t)bm * a.top + __ffsll(lead) - 1;
  return __popc(a.mask[slot]) == 1 &&
         ((uint64_t)a.blocks[slot] << a.block_log2) + 1u == cloud_length(a.lengths, bm / a.M, a.N);
}

// In half precision p and ds would lie among the smallest numbers, where few
// bits are left, for a usual gradient without a scaled loss (ds is 10^-6 with
// dout of 10^-4 and 512 keys: dk was off four times as far as its own rounding
// puts it), and ds beyond the largest one for a large gradient and few keys.  So
// p is taken times 2^15, which p <= 1 allows, and ds times a power of two per
// item, undone on the fp32 sums.  By |dp| <= |dout| |v| the factor of
//   bound = max |dout| over the queries of the cloud and key head
//           * max |v| over the item's keys + max |delta| likewise
// keeps every ds below 2^15, half the largest number, whatever the inputs; the
// rows' maxima come from grad_delta, |v| from the item's keys in shared memory.
template <class T>
constexpr bool kScaled = std::is_same_v<T, __half>;
constexpr float kUp = 32768.f;  // 2^15

// The exponent of the factor (the bound's parts squared: dout, v; delta).
__device__ __forceinline__ int ds_exponent(float dout2, float v2, float delta) {
  const float bound = sqrtf(dout2 * v2) + delta;  // < 2^(e + 1)
  const int e = (int)(__float_as_uint(bound) >> 23) - 127;
  return min(max(14 - e, -100), 100);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// *to = max(*to, x), x >= 0.  Most rows find a larger one there already.
__device__ __forceinline__ void raise(uint32_t *to, float x) {
  const uint32_t bits = __float_as_uint(x);
  if (bits > *reinterpret_cast<volatile uint32_t *>(to)) atomicMax(to, bits);
}

// delta = sum_d dout * out per row; 8 lanes per row, 8 elements per step; bound
// by the bytes read.  out comes with what its rounding left: ds = p (dp - delta)
// is a difference of like numbers where few keys have the weight, and with the
// rounded out alone dq and dk were off 2.3 times as far as their own rounding
// puts them (two keys).  With one key the difference is zero by definition, not
// nearly: delta = inf stands for that.
template <class T>
__global__ void __launch_bounds__(256)
grad_delta(const AttnArgs a) {
  after_previous();
  const uint64_t row = (uint64_t)blockIdx.x * 32u + (threadIdx.x >> 3);
  const uint32_t sub = threadIdx.x & 7u;
  float s = 0.f, dout2 = 0.f;
  if (row < (uint64_t)a.B * a.M * a.H)
    for (uint32_t d = sub * 8; d < a.D; d += 64) {
      const uint4 x = *reinterpret_cast<const uint4 *>(a.dout + (row * a.D + d) * 2);
      const uint4 y = *reinterpret_cast<const uint4 *>(a.out_in + (row * a.D + d) * 2);
      const uint4 z = a.rest_in
                          ? *reinterpret_cast<const uint4 *>(a.rest_in + (row * a.D + d) * 2)
                          : make_uint4(0u, 0u, 0u, 0u);
      const T *xe = reinterpret_cast<const T *>(&x), *ye = reinterpret_cast<const T *>(&y);
      const T *ze = reinterpret_cast<const T *>(&z);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s += to_f32(xe[i]) * (to_f32(ye[i]) + to_f32(ze[i]));
        if (kScaled<T>) dout2 += to_f32(xe[i]) * to_f32(xe[i]);
      }
    }
#pragma unroll
  for (int o = 4; o; o >>= 1) {
    s += __shfl_xor_sync(kFullMask, s, o);
    if (kScaled<T>) dout2 += __shfl_xor_sync(kFullMask, dout2, o);
  }
  const uint32_t bm = (uint32_t)(row / a.H);
  const bool some = row < (uint64_t)a.B * a.M * a.H, one = some && one_key(a, bm);
  if (some && sub == 0) a.delta[row] = one ? INFINITY : s;
  if (!kScaled<T>) return;
  // The rows' maxima: first among the CTA's 32 rows, so that a word of a key
  // head is raised by few (by every row, this kernel took 31 us of a training
  // step of four clouds; so it takes 9, and 6 without the maxima).  Rows that
  // move no score do not count, nor do those that are not finite: they spoil
  // their own results, not the others' factor.
  __shared__ uint32_t s_word[32];
  __shared__ float2 s_most[32];
  if (sub == 0) {
    const bool counts = some && !one && a.lead[bm] && dout2 < INFINITY && fabsf(s) < INFINITY;
    const uint32_t g = (uint32_t)(row - (uint64_t)bm * a.H) / a.R;
    s_word[threadIdx.x >> 3] = counts ? bm / a.M * a.G + g : 0xffffffffu;
    s_most[threadIdx.x >> 3] = make_float2(dout2, fabsf(s));
  }
  __syncthreads();
  if (threadIdx.x >= 32u) return;
  const uint32_t mine = s_word[threadIdx.x];
  bool first = mine != 0xffffffffu;
  float2 most = make_float2(0.f, 0.f);
#pragma unroll 8
  for (uint32_t r = 0; r < 32u; ++r) {
    if (s_word[r] != mine) continue;
    const float2 x = s_most[r];
    most = make_float2(fmaxf(most.x, x.x), fmaxf(most.y, x.y));
    if (r < threadIdx.x) first = false;
  }
  if (first) {
    raise(a.most + 2ull * mine, most.x);
    raise(a.most + 2ull * mine + 1u, most.y);
  }
}

constexpr uint32_t kGradItem = 512;    // query rows per item
// Warps by role: weights, results, products (one warp), loads (one warp per
// stage).
constexpr uint32_t kWeightWarps = 16, kResultWarps = 4, kGradStages = 3;
constexpr uint32_t kGradThreads = 32 * (kWeightWarps + kResultWarps + 1 + kGradStages);

template <int DP>  // 64 or 128
struct GradShape {
  static constexpr uint32_t kRows = DP == 64 ? 128u : 64u;  // query rows per step
  static constexpr uint32_t kStages = kGradStages;          // steps' rows in shared memory
  static constexpr uint32_t kKv = DP == 64 ? 2u : 1u;       // items' keys in shared memory
  static constexpr uint32_t kKeyTile = 128u * DP * 2u, kRowTile = kRows * DP * 2u;
  static constexpr uint32_t kStage = 2u * kRowTile;         // q, dout
  static constexpr uint32_t kRowsAt = kKv * 2u * kKeyTile, kDsAt = kRowsAt + kStages * kStage;
  static constexpr uint32_t kInfoAt = kDsAt + 128u * kRows * 2u;
  // per stage: (lse, delta) of the rows; which rows read block j, j < 8; the
  // rows' places among the partials
  static constexpr uint32_t kBitsAt = 1024u, kPlaceAt = 1152u, kInfo = 1664u;
  // per stage, for the loads: where the rows of q and dout begin
  static constexpr uint32_t kFromAt = kInfoAt + kStages * kInfo, kFrom = kRows * 16u;
  static constexpr uint32_t kSmem = kFromAt + kStages * kFrom + 1024u;
  // tensor memory columns: s^T, dp^T, dv, dk, dq, p^T
  static constexpr uint32_t kDp = kRows, kDv = 2u * kRows, kDk = kDv + DP, kDq = 384u, kP = 448u;
};

// What the roles of the gradient kernel know of an item.
struct GradItem {
  uint32_t gi, g, span, index, b, key0, len, e0, row0, rows, all_rows, steps;
};

// Items of up to kGradItem rows of one span of 128 keys and key head, CTAs
// taking them in turns; dk and dv of the item stay in tensor memory.  Per step
// of rows the tensor core forms s^T = k q^T and dp^T = v dout^T (keys over the
// lanes, rows over the columns); a thread takes one key and half the rows, and
// puts p^T back into tensor memory and ds^T into shared memory, rows
// consecutive.  That tile is dk's left operand as it lies (dk += ds^T q) and
// an operand of dq read down its rows (dq = ds k, or with heads of 128
// elements dq^T = k^T ds^T, so that 64 rows a step suffice); dv += p^T dout
// takes p from tensor memory.  p and ds are rounded to T for these products,
// half a step each (in half precision clear of its ends: kScaled, which costs
// the four clouds below 7 us here).
//
// Done in turns by all warps, the stages of a step took 11,000 cycles, of
// which the weights were 2,500.  So the warps have roles and meet at barriers:
// sixteen make weights, three load a step's rows each (the loads of three steps
// are in the air), four take dq, dk and dv out, and one issues the products,
// the next step's scores before this step's gradients.  Four clouds (16,384
// queries, 4 heads of 64) took 210 us without roles and take 131 (the matrix
// unit 15 % busy, memory 19 %: what is left is the way of a step from barrier to
// barrier, with the gather of 128 rows of q and dout in it), shared heads
// (2,046 queries, 8 heads of 128 over 2) 62 and 38.  At 24 warps a thread has 80
// registers; heads of 128 and half precision spill 8 to 20 bytes of them.  A call
// of few queries pays for its whole cloud here: one query of 122,880 keys and 8
// heads 162 us, most of it zeros written to dk and dv (252 MB).
template <class T, int DP>
__global__ void __launch_bounds__(kGradThreads, 1)
attend_grad(const AttnArgs a) {
  after_previous();
  using Shape = GradShape<DP>;
  constexpr uint32_t kRows = Shape::kRows, kStages = Shape::kStages, kChunks = DP / 8;
  extern __shared__ char smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[kStages * 2 + 4 + 7];
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_gave_up;
  // |v|^2 at most, per warp that loads them, of items k & 3 (a warp that is a
  // step behind another may still read those of the item before)
  __shared__ float s_v2[4][kResultWarps];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = warp_value(tid >> 5);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  char *smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = smem_u32(s_bar);
  auto full = [&](uint32_t st) { return bars + 8u * st; };                // rows loaded
  auto empty = [&](uint32_t st) { return bars + 8u * (kStages + st); };   // and used up
  // (of item k; in turns even where there is one buffer, as a loader may be
  // three steps ahead and must not take one phase for another)
  auto kv_full = [&](uint32_t k) { return bars + 8u * (2 * kStages + (k & 1u)); };
  auto kv_empty = [&](uint32_t k) { return bars + 8u * (2 * kStages + 2 + (k & 1u)); };
  constexpr uint32_t kRest = 8u * (2 * kStages + 4);
  const uint32_t s_ready = bars + kRest, s_free = s_ready + 8u;   // scores made, taken out
  const uint32_t p_ready = s_free + 8u, g_done = p_ready + 8u;    // weights there; products done
  const uint32_t dq_free = g_done + 8u, acc_free = dq_free + 8u;  // dq, dk and dv taken out
  const uint32_t bar_end = acc_free + 8u;
  if (warp == 0) tmem_alloc<512>(smem_u32(&s_tmem));
  if (tid == 0) {
    for (uint32_t i = 0; i < kStages; ++i) {
      bar_init(full(i));
      bar_init(empty(i), 1u + kResultWarps);  // the products, and four warps' reading of the places
    }
    for (uint32_t i = 0; i < 2u; ++i) {
      bar_init(kv_full(i), kResultWarps);
      bar_init(kv_empty(i));
    }
    bar_init(s_ready);
    bar_init(s_free, kWeightWarps);
    bar_init(p_ready, kWeightWarps);
    bar_init(g_done);
    bar_init(dq_free, kResultWarps);
    bar_init(acc_free, kResultWarps);
    bar_init(bar_end);
    s_gave_up = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  const uint32_t tm = warp_value(s_tmem);
  const TileOrder order(a);
  const uint32_t work = warp_value(order.size() * a.gc);
  // Every role walks the same items; the next one's tile is asked for ahead.
  struct Items {
    uint32_t w;
    uint4 tile, next;
  };
  auto tile_at = [&](uint32_t w) {
    return w < work ? order[w / a.gc] : make_uint4(0u, 0u, 0u, 0u);
  };
  auto items = [&]() {
    return Items{blockIdx.x, tile_at(blockIdx.x), tile_at(blockIdx.x + gridDim.x)};
  };
  auto advance = [&](Items &x) {
    x.w += gridDim.x;
    x.tile = x.next;
    x.next = tile_at(x.w + gridDim.x);
  };
  auto steps_of = [&](const uint4 &tile) {
    const uint32_t all = tile.w * a.R, row0 = tile.y * kGradItem;
    return all > row0 ? (min(all - row0, kGradItem) + kRows - 1u) / kRows : 0u;
  };
  auto item_of = [&](const Items &y) {
    GradItem x;
    x.gi = y.w % a.gc;
    x.g = a.g0 + x.gi;
    x.span = y.tile.x;
    x.index = y.tile.y;
    x.b = y.tile.x / a.nsb;
    x.key0 = (y.tile.x - x.b * a.nsb) * 128u;
    x.len = cloud_length(a.lengths, x.b, a.N);
    x.e0 = y.tile.z;
    x.all_rows = y.tile.w * a.R;
    x.row0 = y.tile.y * kGradItem;
    x.rows = x.all_rows > x.row0 ? min(x.all_rows - x.row0, kGradItem) : 0u;
    x.steps = steps_of(y.tile);
    return x;
  };
  // A thread whose wait runs out goes on without waiting, so that the CTA ends.
  // It says so before it touches what may be in use: dk and dv that this CTA
  // writes from then on are NaN, and by the joins all of the turn that shares
  // make, dq among it.
  bool failed = false;
  auto wait = [&](uint32_t bar, uint32_t phase) {
    if (failed || bar_wait(bar, phase, a.wait_ns)) return;
    failed = true;
    *(volatile uint32_t *)a.gave_up = 1u;
    s_gave_up = 1u;
  };
  // The exponent of an item's factor of ds; `most` is asked for before the keys
  // are waited for.
  auto most_of = [&](const GradItem &x) {
    return kScaled<T>
               ? *reinterpret_cast<const float2 *>(a.most + 2ull * ((uint64_t)x.b * a.G + x.g))
               : make_float2(0.f, 0.f);
  };
  auto exponent_of = [&](uint32_t k, const float2 &most) {
    wait(kv_full(k), (k >> 1) & 1u);
    const float *v2 = s_v2[k & 3u];
    return ds_exponent(most.x, fmaxf(fmaxf(v2[0], v2[1]), fmaxf(v2[2], v2[3])), most.y);
  };
  // n counts the steps, k the items
  // with steps.  Use u of a buffer or result waits for completion u - 1 of its
  // release, whose parity is (u - 1) & 1.
  if (warp < kWeightWarps) {
    // ---- weights: lanes 32 quad.. of tensor memory, a quarter of the columns
    const uint32_t quad = warp & 3u, my = (quad * 32u) << 16;
    constexpr uint32_t kCols = kRows / (kWeightWarps / 4u);
    const uint32_t col0 = (warp >> 2) * kCols;
    const uint32_t key_in = quad * 32u + lane, block = key_in >> a.block_log2;
    const float c2 = a.scale * kLog2e;
    uint32_t n = 0, k = 0;
    for (Items y = items(); y.w < work; advance(y)) {
      const GradItem it = item_of(y);
      const float2 most = most_of(it);
      float f_ds = 1.f;  // of ds, over p's
      if (kScaled<T> && it.steps) f_ds = pow2(exponent_of(k++, most) - 15);
      // rows that may read this key; kLone: it is a block's only key
      constexpr uint32_t kLone = 0x10000u;
      const uint32_t key = it.key0 + key_in;
      const uint32_t live = key >= it.len ? 0u
                            : key + 1u == it.len && !(key & ((1u << a.block_log2) - 1u))
                                ? 0xffffu | kLone
                                : 0xffffu;
      for (uint32_t i = 0; i < it.steps; ++i, ++n) {
        const uint32_t st = n % kStages;
        const char *info = smem + Shape::kInfoAt + st * Shape::kInfo;
        wait(full(st), (n / kStages) & 1u);
        wait(s_ready, n & 1u);
        __syncwarp();
        tmem_after_sync();
        constexpr uint32_t kPieces = kCols / 16u;  // of 16 rows
        uint32_t p[kPieces][8], e[kPieces][8];
#pragma unroll
        for (uint32_t x = 0; x < kPieces; ++x) {
          const uint32_t col = col0 + x * 16u;
          uint32_t sx[16], dx[16];
          tmem_ld16(sx, tm + my + col);
          tmem_ld16(dx, tm + Shape::kDp + my + col);
          // which of the 16 rows read this key
          uint32_t in = reinterpret_cast<const uint16_t *>(info + Shape::kBitsAt)[block * 8u + col / 16u];
          in &= live;
          tmem_ld_wait();
          if (x + 1u == kPieces) {
            tmem_before_sync();
            __syncwarp();
            if (lane == 0) bar_arrive(s_free);
          }
          uint32_t *p16 = p[x], *e16 = e[x];
          const bool all = __all_sync(kFullMask, in == 0xffffu);
          if (__any_sync(kFullMask, in != 0u)) {
#pragma unroll
            for (uint32_t y = 0; y < 16u; y += 2u) {
              // (lse, delta) of two rows
              const float4 z = reinterpret_cast<const float4 *>(info)[col / 2u + y / 2u];
              float2 f = fma2(make_float2(__uint_as_float(sx[y]), __uint_as_float(sx[y + 1])),
                              make_float2(c2, c2), make_float2(-z.x, -z.z));
              f.x = exp2_fast(f.x);
              f.y = exp2_fast(f.y);
              float2 g = add2(make_float2(__uint_as_float(dx[y]), __uint_as_float(dx[y + 1])),
                              make_float2(-z.y, -z.w));
              if (kScaled<T>) g = mul2(g, make_float2(f_ds, f_ds));
              g = mul2(f, g);
              if (!all) {
                const bool in0 = (in >> y) & 1u, in1 = (in >> (y + 1u)) & 1u;
                f.x = in0 ? f.x : 0.f, g.x = in0 ? g.x : 0.f;
                f.y = in1 ? f.y : 0.f, g.y = in1 ? g.y : 0.f;
              }
              p16[y / 2u] = pack2<T>(f.x, f.y);
              e16[y / 2u] = pack2<T>(g.x, g.y);
            }
          } else {
#pragma unroll
            for (uint32_t y = 0; y < 8u; ++y) p16[y] = e16[y] = 0u;
          }
        }
        if (n) {  // the step before is done with p and ds
          wait(g_done, (n - 1u) & 1u);
          __syncwarp();
          tmem_after_sync();
        }
#pragma unroll
        for (uint32_t x = 0; x < kPieces; ++x) {
          const uint32_t col = col0 + x * 16u;
          tmem_st8(tm + Shape::kP + my + col / 2u, p[x]);
#pragma unroll
          for (uint32_t c = 0; c < 2u; ++c)
            *reinterpret_cast<uint4 *>(smem + Shape::kDsAt + (col / 64u) * 16384u +
                                       swizzled(key_in, (col % 64u) / 8u + c)) =
                make_uint4(e[x][4 * c], e[x][4 * c + 1], e[x][4 * c + 2], e[x][4 * c + 3]);
        }
        if (live & kLone)  // rows of one key are here only (tested per element: 11 us of 140)
#pragma unroll 1
          for (uint32_t col = col0; col < col0 + kCols; ++col)
            if (reinterpret_cast<const float2 *>(info)[col].y == INFINITY)
              *reinterpret_cast<uint16_t *>(smem + Shape::kDsAt + (col / 64u) * 16384u +
                                            swizzled(key_in, (col % 64u) / 8u) + (col % 8u) * 2u) = 0u;
        tmem_st_wait();
        smem_to_mma();
        tmem_before_sync();
        __syncwarp();
        if (lane == 0) bar_arrive(p_ready);
      }
    }
  } else if (warp < kWeightWarps + kResultWarps) {
    // ---- results: lanes 32 (warp & 3).. of tensor memory
    const uint32_t at_lane = (warp & 3u) * 32u + lane, my = (at_lane & ~31u) << 16;
    const uint32_t role_tid = tid - 32u * kWeightWarps;
    uint32_t n = 0;
    // These warps also load the items' keys: item k's at the beginning, then
    // one ahead where there are two buffers.
    Items later = items();
    uint32_t loaded = 0;
    auto load_next = [&]() {  // the next item with steps, if any
      for (; later.w < work; advance(later)) {
        if (!steps_of(later.tile)) continue;
        const GradItem x = item_of(later);
        if (loaded >= Shape::kKv)
          wait(kv_empty(loaded - Shape::kKv), ((loaded - Shape::kKv) >> 1) & 1u);
        __syncwarp();
        const uint32_t sk = base + (loaded % Shape::kKv) * 2u * Shape::kKeyTile;
        const int64_t ks = a.ks[1] * 2, vs = a.vs[1] * 2;
        const char *kh = a.k + 2 * ((int64_t)x.b * a.ks[0] + (int64_t)x.g * a.ks[2]) + x.key0 * ks;
        const char *vh = a.v + 2 * ((int64_t)x.b * a.vs[0] + (int64_t)x.g * a.vs[2]) + x.key0 * vs;
        const uint32_t blocks = marked(a.listed[x.span]), live = x.len - x.key0;
        load_strided<DP, 128, 128>(sk, a.D, role_tid, kh, ks, live, blocks, a.block_log2);
        load_strided<DP, 128, 128>(sk + Shape::kKeyTile, a.D, role_tid, vh, vs, live, blocks,
                                   a.block_log2);
        copy_commit();
        advance(later);
        return true;
      }
      return false;
    };
    auto finish_load = [&]() {
      copy_wait<0>();
      smem_to_mma();
      if (kScaled<T>) {
        // of the chunks of 8 elements that this thread loaded (load_strided),
        // the longest in each place of a row, and those of a row together
        constexpr uint32_t kStep = 128u / kChunks;
        const uint32_t c = role_tid % kChunks, r0 = role_tid / kChunks;
        const char *v = smem + ((loaded % Shape::kKv) * 2u + 1u) * Shape::kKeyTile +
                        (c >> 3) * (128u * 128u) + swizzled(r0, c & 7u);
        float most = 0.f;
#pragma unroll 4
        for (uint32_t i = 0; i < 128u / kStep; ++i) {
          const uint4 x = *reinterpret_cast<const uint4 *>(v + i * kStep * 128u);
          const T *e = reinterpret_cast<const T *>(&x);
          float v2 = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) v2 = fmaf(to_f32(e[j]), to_f32(e[j]), v2);
          most = fmaxf(most, v2 < INFINITY ? v2 : 0.f);
        }
#pragma unroll
        for (uint32_t o = 16u; o >= kChunks; o >>= 1)
          most = fmaxf(most, __shfl_xor_sync(kFullMask, most, o));
#pragma unroll
        for (uint32_t o = kChunks / 2u; o; o >>= 1) most += __shfl_xor_sync(kFullMask, most, o);
        if (lane == 0) s_v2[loaded & 3u][warp & 3u] = most;
      }
      __syncwarp();
      if (lane == 0) bar_arrive(kv_full(loaded));
      ++loaded;
    };
    if (load_next()) finish_load();
    uint32_t k = 0;
    for (Items y = items(); y.w < work; advance(y)) {
      const GradItem it = item_of(y);
      const float2 most = most_of(it);
      float down_ds = 1.f;
      if (kScaled<T> && it.steps) down_ds = pow2(-exponent_of(k++, most));
      constexpr float kDownP = kScaled<T> ? 1.f / kUp : 1.f;
      // (waited for here: the products of this item's last step come after the
      // next item's scores)
      if (it.steps && Shape::kKv == 2u && load_next()) finish_load();
      const uint32_t key = it.key0 + at_lane;
      const uint64_t key_row = ((uint64_t)it.b * a.N + key) * a.G + it.g;
      for (uint32_t i = 0; i < it.steps; ++i, ++n) {
        const uint32_t st = n % kStages;
        const uint32_t *place = reinterpret_cast<const uint32_t *>(
            smem + Shape::kInfoAt + st * Shape::kInfo + Shape::kPlaceAt);
        wait(full(st), (n / kStages) & 1u);
        wait(g_done, n & 1u);
        __syncwarp();
        tmem_after_sync();
        const float f = down_ds;
        // (places first: behind the second half the stage is given back)
        const uint32_t mine = DP == 64 ? place[at_lane] : 0u;
#pragma unroll
        for (uint32_t h = 0; h < 2u; ++h) {
          uint32_t o[32];
          tmem_ld32(o, tm + Shape::kDq + my + h * 32u);
          tmem_ld_wait();
          if (h) {
            tmem_before_sync();
            __syncwarp();
            if (lane == 0) bar_arrive(dq_free);
          }
          if (DP == 64) {  // a lane has a row
            if (mine != 0xffffffffu) {
              float *to = a.part + (uint64_t)mine * a.D + h * 32u;
#pragma unroll
              for (uint32_t y = 0; y < 32u; y += 8u)
                if (h * 32u + y < a.D) store8(to + y, &o[y], f);
            }
          } else {         // a lane has one element of 32 rows
#pragma unroll
            for (uint32_t y = 0; y < 32u; ++y) {
              const uint32_t to = place[h * 32u + y];
              if (to != 0xffffffffu && at_lane < a.D)
                a.part[(uint64_t)to * a.D + at_lane] = __uint_as_float(o[y]) * f;
            }
          }
          __syncwarp();
        }
        if (lane == 0) bar_arrive(empty(st));
      }
      // the span's dk and dv, or this item's share of them: a lane has a key
      const bool whole = it.all_rows <= kGradItem, some = key < a.N;
      if (it.steps) {
        const uint64_t place = whole ? 0u : a.span[it.span].z + it.index;
        float *share = a.part_kv + ((place * a.gc + it.gi) * 256u + at_lane) * a.D;
#pragma unroll
        for (uint32_t j = 0; j < DP / 16; ++j) {
          const bool is_k = j >= DP / 32;
          const uint32_t col = (j % (DP / 32)) * 32u;
          uint32_t o[32];
          tmem_ld32(o, tm + (is_k ? Shape::kDk : Shape::kDv) + my + col);
          tmem_ld_wait();
          if (j + 1u == DP / 16) {
            tmem_before_sync();
            __syncwarp();
            if (lane == 0) bar_arrive(acc_free);
          }
          const float f = !is_k ? kDownP : whole ? down_ds * a.scale : down_ds;
          const float g = s_gave_up ? NAN : f;  // (looked at behind the values)
          if (some) {
#pragma unroll
            for (uint32_t y = 0; y < 32u; y += 8u) {
              if (col + y >= a.D) continue;
              if (whole) {
                uint32_t h[4];
#pragma unroll
                for (uint32_t z = 0; z < 4u; ++z)
                  h[z] = pack2<T>(__uint_as_float(o[y + 2 * z]) * g,
                                  __uint_as_float(o[y + 2 * z + 1]) * g);
                *reinterpret_cast<uint4 *>((is_k ? a.dk : a.dv) + 2 * (key_row * a.D + col + y)) =
                    make_uint4(h[0], h[1], h[2], h[3]);
              } else {
                store8(share + (is_k ? 0 : 128 * (uint64_t)a.D) + col + y, &o[y], g);
              }
            }
          }
          __syncwarp();
        }
        if (Shape::kKv == 1u && load_next()) finish_load();
      } else if (some) {  // a span that nobody reads
        for (uint32_t j = 0; j < a.D; j += 8u) {
          *reinterpret_cast<uint4 *>(a.dk + 2 * (key_row * a.D + j)) = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4 *>(a.dv + 2 * (key_row * a.D + j)) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
    }
  } else if (warp == kWeightWarps + kResultWarps) {
    // ---- products: the warp in step
    {
      constexpr uint32_t kScores = mma_desc<T>(128, kRows, false, false);
      constexpr uint32_t kRowsBy = mma_desc<T>(128, DP, false, true);  // dv, dk
      constexpr uint32_t kDqBy = mma_desc<T>(128, 64, true, true);
      struct Walk {  // steps in order
        Items y;
        uint32_t i, steps, n, k;
      };
      auto settle = [&](Walk &x) {  // on the next item with steps
        for (; x.y.w < work; advance(x.y))
          if ((x.steps = warp_value(steps_of(x.y.tile)))) return;
      };
      auto next = [&](Walk &x) {
        ++x.n;
        if (++x.i < x.steps) return;
        x.i = 0;
        ++x.k;
        advance(x.y);
        settle(x);
      };
      const bool hold = a.hold_cta == (int)blockIdx.x;
      // (the distance of further columns means nothing where there are none)
      const uint64_t ds_desc = tile_desc(base + Shape::kDsAt, 16384u);
      auto keys_at = [&](uint32_t k) { return base + (k % Shape::kKv) * 2u * Shape::kKeyTile; };
      auto rows_at = [&](uint32_t n) { return base + Shape::kRowsAt + (n % kStages) * Shape::kStage; };
      auto scores = [&](Walk &x) {
        wait(full(x.n % kStages), (x.n / kStages) & 1u);
        if (x.i == 0) wait(kv_full(x.k), (x.k >> 1) & 1u);
        if (x.n) wait(s_free, (x.n - 1u) & 1u);
        __syncwarp();
        tmem_after_sync();
        const uint64_t k_desc = tile_desc(keys_at(x.k), 16u), q_desc = tile_desc(rows_at(x.n), 16u);
#pragma unroll
        for (uint32_t kk = 0; kk < DP / 16; ++kk)
          mma_ss(tm, further(k_desc, (kk >> 2) * 16384u + (kk & 3u) * 32u),
                 further(q_desc, (kk >> 2) * (kRows * 128u) + (kk & 3u) * 32u), kScores, kk != 0u);
#pragma unroll
        for (uint32_t kk = 0; kk < DP / 16; ++kk)
          mma_ss(tm + Shape::kDp,
                 further(k_desc, Shape::kKeyTile + (kk >> 2) * 16384u + (kk & 3u) * 32u),
                 further(q_desc, Shape::kRowTile + (kk >> 2) * (kRows * 128u) + (kk & 3u) * 32u),
                 kScores, kk != 0u);
        if (!(hold && x.n == 0u && a.hold_step == 0u)) mma_commit(s_ready);
        next(x);
      };
      auto grads = [&](Walk &x) {
        wait(p_ready, x.n & 1u);
        if (x.n) wait(dq_free, (x.n - 1u) & 1u);
        if (x.i == 0 && x.k) wait(acc_free, (x.k - 1u) & 1u);
        __syncwarp();
        tmem_after_sync();
        const uint64_t k_desc = tile_desc(keys_at(x.k), 16384u);
        const uint64_t q_desc = tile_desc(rows_at(x.n), kRows * 128u);
        const bool add = x.i != 0u;
#pragma unroll
        for (uint32_t kk = 0; kk < kRows / 16; ++kk)
          mma_ts(tm + Shape::kDv, tm + Shape::kP + kk * 8u,
                 further(q_desc, Shape::kRowTile + kk * 2048u), kRowsBy, add || kk != 0u);
#pragma unroll
        for (uint32_t kk = 0; kk < kRows / 16; ++kk)
          mma_ss(tm + Shape::kDk, further(ds_desc, (kk >> 2) * 16384u + (kk & 3u) * 32u),
                 further(q_desc, kk * 2048u), kRowsBy, add || kk != 0u);
#pragma unroll
        for (uint32_t kk = 0; kk < 8u; ++kk) {
          const uint64_t ds = further(ds_desc, kk * 2048u), ky = further(k_desc, kk * 2048u);
          mma_ss(tm + Shape::kDq, DP == 64 ? ds : ky, DP == 64 ? ky : ds, kDqBy, kk != 0u);
        }
        if (!(hold && x.n == 0u && a.hold_step == 1u)) mma_commit(g_done);
        mma_commit(empty(x.n % kStages));
        if (x.i + 1u == x.steps) mma_commit(kv_empty(x.k));
        next(x);
      };
      Walk ahead{items(), 0u, 0u, 0u, 0u};
      settle(ahead);
      Walk now = ahead;
      if (ahead.y.w < work) scores(ahead);
      while (now.y.w < work) {
        // (with one buffer of keys the next item's wait for this one's products)
        const bool early = ahead.y.w < work && (Shape::kKv == 2u || ahead.i != 0u);
        if (early) scores(ahead);
        grads(now);
        if (!early && ahead.y.w < work) scores(ahead);
      }
    }
    __syncwarp();
  } else {
    // ---- loads: steps n with n % kStages == stage
    const uint32_t stage = warp - (kWeightWarps + kResultWarps + 1u);
    char *info = smem + Shape::kInfoAt + stage * Shape::kInfo;
    longlong2 *from = reinterpret_cast<longlong2 *>(smem + Shape::kFromAt + stage * Shape::kFrom);
    const uint32_t at = base + Shape::kRowsAt + stage * Shape::kStage;
    uint32_t n = 0;
    for (Items y = items(); y.w < work; advance(y)) {
      const GradItem it = item_of(y);
      for (uint32_t i = 0; i < it.steps; ++i, ++n) {
        if (n % kStages != stage) continue;
        const uint32_t use = n / kStages;
        // the rows: lane, lane + 32, ... (asked for before the stage is free);
        // rows behind the last repeat it, and no weight of theirs is kept
        constexpr uint32_t kHeld = kRows / 32u;
        float lse[kHeld], delta[kHeld];
        uint32_t mask[kHeld], place[kHeld];
#pragma unroll
        for (uint32_t j = 0; j < kHeld; ++j) {
          const uint32_t r0 = i * kRows + j * 32u + lane, r = min(r0, it.rows - 1u);
          const uint32_t e = (it.row0 + r) / a.R, head = it.row0 + r - e * a.R;
          const uint32_t pair = a.vals[it.e0 + e];
          const uint32_t bm = pair / a.top, m = bm - it.b * a.M, h = it.g * a.R + head;
          const uint32_t row = bm * a.H + h;
          lse[j] = a.lse_in[row] * kLog2e - (kScaled<T> ? 15.f : 0.f);
          delta[j] = a.delta[row];
          mask[j] = r0 < it.rows ? a.mask[pair] : 0u;
          place[j] = r0 < it.rows ? pair * (a.gc * a.R) + it.gi * a.R + head : 0xffffffffu;
          from[j * 32u + lane] = make_longlong2(
              2 * ((int64_t)it.b * a.qs[0] + (int64_t)m * a.qs[1] + (int64_t)h * a.qs[2]),
              2 * (int64_t)((uint64_t)row * a.D));
        }
        if (use) wait(empty(stage), (use - 1u) & 1u);
        __syncwarp();
        {
          constexpr uint32_t kTogether = 32u / kChunks;  // rows per turn
          const uint32_t c = lane % kChunks, r0 = lane / kChunks;
          const bool in = c * 8u < a.D;
          const char *q = a.q + (in ? c * 16u : 0u), *o = a.dout + (in ? c * 16u : 0u);
          const uint32_t to = at + (c >> 3) * (kRows * 128u);
#pragma unroll 8
          for (uint32_t y = 0; y < kRows / kTogether; ++y) {
            const uint32_t r = y * kTogether + r0;
            const longlong2 x = from[r];
            const uint32_t dst = to + swizzled(r, c & 7u);
            copy16(dst, q + x.x, in);
            copy16(dst + Shape::kRowTile, o + x.y, in);
          }
        }
        copy_commit();
#pragma unroll
        for (uint32_t j = 0; j < kHeld; ++j) {
          reinterpret_cast<float2 *>(info)[j * 32u + lane] = make_float2(lse[j], delta[j]);
          reinterpret_cast<uint32_t *>(info + Shape::kPlaceAt)[j * 32u + lane] = place[j];
#pragma unroll
          for (uint32_t x = 0; x < 8u; ++x) {
            const uint32_t bits = __ballot_sync(kFullMask, (mask[j] >> x) & 1u);
            if (lane == x) reinterpret_cast<uint32_t *>(info + Shape::kBitsAt)[x * 4u + j] = bits;
          }
        }
        copy_wait<0>();
        smem_to_mma();
        __syncwarp();
        if (lane == 0) bar_arrive(full(stage));
      }
    }
  }
  __syncwarp();
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  if (s_gave_up) {  // nothing may write tensor memory that is given back
    if (warp == kWeightWarps + kResultWarps) {
      mma_commit(bar_end);
      bar_wait(bar_end, 0u, a.wait_ns);
    }
    __syncthreads();
  }
  if (warp == 0) tmem_free<512>(tm);
}

// dk and dv of the spans that several items share, their shares in order.
template <class T>
__global__ void __launch_bounds__(256)
grad_join_keys(const AttnArgs a, uint32_t span) {
  after_previous();
  const uint32_t s = blockIdx.x, gi = blockIdx.y, g = a.g0 + gi;
  const uint4 sp = a.span[s];
  const uint32_t i0 = sp.z, i1 = sp.z + sp.w;
  if (sp.w < 2u) return;
  const uint32_t b = s / a.nsb, key0 = (s - b * a.nsb) * span;
  const uint32_t keys = min(span, a.N - key0);
  for (uint32_t x = blockIdx.z * 256u + threadIdx.x; x < keys * a.D / 2u; x += 256u * gridDim.z) {
    const uint32_t r = x / (a.D / 2u), d = (x - r * (a.D / 2u)) * 2u;
    float2 k = make_float2(0.f, 0.f), v = k;
    for (uint32_t i = i0; i < i1; ++i) {
      const float *o = a.part_kv + (((uint64_t)i * a.gc + gi) * 2 * span + r) * a.D + d;
      const float2 y = *reinterpret_cast<const float2 *>(o);
      const float2 z = *reinterpret_cast<const float2 *>(o + (uint64_t)span * a.D);
      k.x += y.x; k.y += y.y; v.x += z.x; v.y += z.y;
    }
    const uint64_t o = 2 * ((((uint64_t)b * a.N + key0 + r) * a.G + g) * a.D + d);
    if (some_gave_up(a)) k.x = k.y = v.x = v.y = NAN;
    *reinterpret_cast<uint32_t *>(a.dk + o) = pack2<T>(k.x * a.scale, k.y * a.scale);
    *reinterpret_cast<uint32_t *>(a.dv + o) = pack2<T>(v.x, v.y);
  }
}

// dq of a query: the shares of its pairs, slots in order; lanes as in
// attend_join, and bound as it is (24 us for the four clouds).
template <class T>
__global__ void __launch_bounds__(256)
grad_join_queries(const AttnArgs a, uint32_t parts) {
  after_previous();
  const uint32_t lane = threadIdx.x & 31u, hc = a.gc * a.R;
  const uint64_t w = (uint64_t)blockIdx.x * 8u + (threadIdx.x >> 5);
  const uint32_t bm = (uint32_t)(w / parts);
  if (bm >= a.B * a.M) return;
  const uint32_t d = (uint32_t)(w - (uint64_t)bm * parts) * 128u + lane * 4u;
  if (d >= hc * a.D) return;
  const float *part = a.part + (uint64_t)bm * a.top * hc * a.D + d;
  const uint64_t step = (uint64_t)hc * a.D;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (unsigned long long l = a.lead[bm]; l;) {
    float4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      x[u] = l ? __ldcs(reinterpret_cast<const float4 *>(part + (uint64_t)(__ffsll(l) - 1) * step))
               : make_float4(0.f, 0.f, 0.f, 0.f);
      l &= l - 1ull;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      acc.x += x[u].x; acc.y += x[u].y; acc.z += x[u].z; acc.w += x[u].w;
    }
  }
  const uint64_t out = ((uint64_t)bm * a.H + a.g0 * a.R) * a.D + d;
  const float f = some_gave_up(a) ? NAN : a.scale;
  *reinterpret_cast<uint2 *>(a.dq + out * 2) =
      make_uint2(pack2<T>(acc.x * f, acc.y * f), pack2<T>(acc.z * f, acc.w * f));
}

// ------------------------------------------------------------- host side

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
  if (!std::isfinite(d->scale * kLog2e))
    return set_error(NSFPS_ERR_ARG, "scale must be finite, times log2(e) too");
  const uint64_t lim = 1ull << 30;
  if (d->batch >= lim / 8 || d->queries >= lim || d->keys >= lim || d->batch * d->keys >= lim ||
      d->batch * d->queries >= lim || d->batch * d->queries * d->top >= lim ||
      d->queries * d->top * (d->heads / d->kv_heads) >= 2 * lim)
    return set_error(NSFPS_ERR_UNSUPPORTED,
                     "batch must be below 2^27, batch * queries * top and batch * keys below "
                     "2^30, queries * top * heads / kv_heads below 2^31");
  for (int i = 0; i < 3; ++i)
    if (d->q_stride[i] < 0 || d->k_stride[i] < 0 || d->v_stride[i] < 0 || d->q_stride[i] % 8 ||
        d->k_stride[i] % 8 || d->v_stride[i] % 8)
      return set_error(NSFPS_ERR_ARG, "strides must be multiples of 8 elements, not negative");
  return NSFPS_OK;
}

uint32_t log2_of(uint32_t block) { return block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7; }

int padded_dim(uint32_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// Keys per span of the gradient.
constexpr uint32_t kGradSpanLog2 = 7;  // one key per lane of tensor memory

// Partials of a pass stay below this where taking the key heads, then the clouds
// of a call, in turns brings them there.  A turn has at least one cloud and one
// key head, with all their queries: dk and dv of a key add up over those, and the
// gradient has no place to keep such sums between turns.  So one cloud of 65,536
// queries, lists of 16 and eight query heads of 128 on one key head takes 4.3 GB,
// every slot counted, as the plan cannot know how many lead a pair.  Turns small
// enough to keep their partials in L2 cost more in launches and half-empty waves
// than they save: a scan's attention took 199 us in one turn, 207 in two, 267 in
// four.
constexpr uint64_t kMaxPartBytes = 1ull << 30;

// How a call is cut up, and its scratch.
struct AttnPlan {
  bool direct;
  uint32_t bc;             // clouds per turn
  uint32_t gc;             // key heads per turn
  uint32_t span_log2, tile_rows, least, splits, rounds;
  uint64_t pairs, spans, max_tiles;  // of one turn
  SortScratch sort;
  uint32_t *mask, *tile_count, *most;
  uint64_t most_bytes;
  uint8_t *listed;
  uint4 *span;
  unsigned long long *lead;
  uint4 *tiles;
  float *part, *part_lse, *delta, *part_kv;
  uint64_t bytes;
};

// The direct path reads each query's keys once per query, the tiles once per
// 128 of them, behind a sort.  Up to some 200 MB of keys the former is less:
// 64 queries of 8 heads and 1,024 keys of 64 (134 MB) took 28 us direct and 34
// by tiles, 128 queries (268 MB) 37 and 38, 512 queries 135 and 47; 1,024
// queries of 4 heads and 64 keys (67 MB) 23 and 31, 4,096 (268 MB) 84 and 39;
// one query 4 and 24.
bool takes_direct(const nsfps_attention_desc &d) {
  const uint64_t keys = std::min<uint64_t>((uint64_t)d.top * d.block, d.keys);
  return d.batch * d.queries <= 65535 &&
         d.batch * d.queries * d.kv_heads * keys * d.head_dim * 4 <= 200000000;
}

AttnPlan plan_attention(const nsfps_attention_desc &d, bool backward, void *base) {
  AttnPlan w{};
  WorkCarver c(base);
  const uint64_t R = d.heads / d.kv_heads;
  w.direct = !backward && takes_direct(d);
  w.bc = (uint32_t)d.batch;
  w.gc = d.kv_heads;
  if (w.direct) {
    // as many rounds per CTA as leave six CTAs for every SM: one query of 1,024
    // keys takes a round each, 16 of 8,192 keys and heads of 128 four (40 us in
    // all, with a round each 61: a partial costs its write, its read and a
    // CTA's start; 134 MB of keys come at 4.2 TB/s)
    const uint64_t all = ceil_div((uint64_t)d.top * d.block, kDirectKeys);
    const uint64_t ctas = all * d.batch * d.queries * d.kv_heads * ceil_div(R, 16);
    w.rounds = (uint32_t)std::min(all, std::max<uint64_t>(1, ctas / (148 * 6)));
    w.splits = (uint32_t)ceil_div(all, w.rounds);
    if (w.splits > 1) {
      const uint64_t rows = d.batch * d.queries * d.heads * w.splits;
      w.part = c.take<float>(rows * d.head_dim);
      w.part_lse = c.take<float>(rows);
    }
    w.bytes = c.off + 256;
    return w;
  }
  w.span_log2 = backward ? kGradSpanLog2 : kSpanLog2;
  w.tile_rows = backward ? kGradItem : kTileRows;
  w.least = backward ? 1 : 0;
  const uint64_t span = 1ull << w.span_log2, nsb = ceil_div(d.keys, span);
  auto part_bytes = [&](uint64_t clouds, uint64_t heads) {
    const uint64_t pairs = clouds * d.queries * d.top, spans = clouds * nsb;
    uint64_t b = pairs * R * heads * (d.head_dim + 1) * 4;
    if (backward)
      b += (pairs * R / w.tile_rows + spans) * heads * 2 * span * d.head_dim * 4;
    return b;
  };
  while (w.gc > 1 && part_bytes(w.bc, w.gc) > kMaxPartBytes) w.gc = (w.gc + 1) / 2;
  while (w.bc > 1 && part_bytes(w.bc, w.gc) > kMaxPartBytes) w.bc = (w.bc + 1) / 2;
  w.pairs = w.bc * d.queries * d.top;
  w.spans = w.bc * nsb;
  w.max_tiles = w.pairs * R / w.tile_rows + w.spans;
  w.sort.carve(c, (uint32_t)w.pairs);
  w.mask = c.take<uint32_t>(w.pairs);
  w.lead = c.take<unsigned long long>(w.bc * d.queries);
  w.span = c.take<uint4>(w.spans);
  static_assert(4 * (kTileClasses + 2) <= 32, "the marks begin 32 bytes behind");
  // (cleared together, before a turn)
  w.most_bytes = backward && d.dtype == NSFPS_F16 ? ceil_div(w.bc * (uint64_t)d.kv_heads, 2) * 16 : 0;
  w.tile_count = (uint32_t *)c.take<char>(32 + w.most_bytes + 16 * w.spans);
  w.most = w.tile_count + (base ? 8 : 0);
  w.listed = (uint8_t *)w.most + (base ? w.most_bytes : 0);
  w.tiles = c.take<uint4>(kTileClasses * w.max_tiles);
  w.part = c.take<float>(w.pairs * R * w.gc * d.head_dim);
  if (backward) {
    w.delta = c.take<float>(w.bc * d.queries * d.heads);
    w.part_kv = c.take<float>(w.max_tiles * w.gc * 2 * span * d.head_dim);
  } else {
    w.part_lse = c.take<float>(w.pairs * R * w.gc);
  }
  w.bytes = c.off + 256;
  return w;
}

AttnArgs common_args(const nsfps_attention_desc &d, const void *q, const void *k, const void *v,
                     const int64_t *blocks, const int32_t *lengths, const AttnPlan &w) {
  AttnArgs a{};
  a.q = (const char *)q; a.k = (const char *)k; a.v = (const char *)v;
  a.blocks = blocks; a.lengths = lengths;
  a.B = (uint32_t)d.batch; a.M = (uint32_t)d.queries; a.N = (uint32_t)d.keys;
  a.H = d.heads; a.G = d.kv_heads; a.R = d.heads / d.kv_heads; a.D = d.head_dim; a.top = d.top;
  a.block_log2 = log2_of(d.block);
  a.nb = (uint32_t)ceil_div(d.keys, d.block);
  for (int i = 0; i < 3; ++i) a.qs[i] = d.q_stride[i], a.ks[i] = d.k_stride[i], a.vs[i] = d.v_stride[i];
  a.scale = d.scale;
  a.nsb = w.direct ? 0 : (uint32_t)ceil_div(d.keys, 1ull << w.span_log2);
  a.most = w.most;
  a.mask = w.mask; a.lead = w.lead; a.span = w.span; a.tile_count = w.tile_count;
  a.gave_up = w.tile_count + kTileClasses + 1;
  const WaitHooks hooks = wait_hooks();
  a.wait_ns = (unsigned long long)hooks.limit_ns;
  a.hold_cta = hooks.hold_cta;
  a.hold_step = hooks.hold_step;
  a.listed = (const uint4 *)w.listed;
  a.tile_stride = (uint32_t)w.max_tiles;
  a.tiles = w.tiles; a.part = w.part; a.part_lse = w.part_lse; a.delta = w.delta;
  a.part_kv = w.part_kv; a.splits = w.splits; a.rounds = w.rounds;
  a.row_parts = (uint32_t)ceil_div(a.R, 16); a.gc = w.gc;
  return a;
}

// The turn that starts with cloud b0.
AttnArgs turn_args(const AttnArgs &all, uint32_t b0, uint32_t bc) {
  AttnArgs a = all;
  a.B = std::min(bc, all.B - b0);
  const uint64_t rows = (uint64_t)b0 * a.M;
  a.q += 2 * (int64_t)b0 * a.qs[0];
  a.k += 2 * (int64_t)b0 * a.ks[0];
  a.v += 2 * (int64_t)b0 * a.vs[0];
  a.blocks += rows * a.top;
  if (a.lengths) a.lengths += b0;
  const uint64_t ro = 2 * rows * a.H * a.D, ko = 2 * (uint64_t)b0 * a.N * a.G * a.D;
  if (a.out) a.out += ro;
  if (a.rest) a.rest += ro;
  if (a.rest_in) a.rest_in += ro;
  if (a.lse) a.lse += rows * a.H;
  if (a.dout) a.dout += ro, a.out_in += ro, a.dq += ro, a.lse_in += rows * a.H;
  if (a.dk) a.dk += ko, a.dv += ko;
  return a;
}

// Sorts a turn's pairs by span and lists its tiles.
cudaError_t run_plan(AttnArgs &a, const AttnPlan &w, cudaStream_t st) {
  const uint32_t n = a.B * a.M * a.top, spans = a.B * a.nsb;
  const uint32_t shift = 1u << (w.span_log2 - 6);  // key bits of the chunks read
  SortedList list{w.sort.keys0, w.sort.vals0, w.sort.kept};
  cudaError_t err;
  // (the tile counters and gave_up, the rows' maxima, the spans' marks)
  if ((err = cudaMemsetAsync(w.tile_count, 0, 32 + w.most_bytes + 16 * (uint64_t)spans, st)))
    return err;
  if (n && spans) {
    // a power of two of lanes that holds the list, up to a warp with two slots each
    const uint32_t lanes = a.top <= 8 ? 8 : a.top <= 16 ? 16 : 32;
    const auto kernel = a.top <= 8    ? plan_pairs<1, 8>
                        : a.top <= 16 ? plan_pairs<1, 16>
                        : a.top <= 32 ? plan_pairs<1, 32>
                                      : plan_pairs<2, 32>;
    if ((err = launch_next(kernel, (uint32_t)ceil_div((uint64_t)a.B * a.M * lanes, 256), 256, 0, st,
                           a, w.span_log2, w.sort.keys0, w.mask, w.lead, w.listed)))
      return err;
    if ((err = run_sort(PairKeys{w.sort.keys0}, n, spans << shift, w.sort, &list, st))) return err;
  } else {  // no pair, or no key to form one with
    if ((err = cudaMemsetAsync(w.sort.kept, 0, 4, st))) return err;
    if (a.B * a.M &&
        (err = cudaMemsetAsync(w.lead, 0, sizeof(*w.lead) * (uint64_t)a.B * a.M, st)))
      return err;
  }
  a.vals = list.vals;
  a.skeys = list.keys;
  if (!spans) return cudaSuccess;
  return launch_next(plan_spans, (uint32_t)ceil_div(spans, 8), 256, 0, st, list, spans, shift, a.R,
                     w.tile_rows, w.least, w.least == 0u, w.span, w.tiles, a.tile_stride,
                     w.tile_count);
}

template <class T, int DP>
cudaError_t launch_forward(const AttnArgs &all, const AttnPlan &w, cudaStream_t st) {
  cudaError_t err;
  if (w.direct) {
    AttnArgs a = all;
    const uint32_t smem = DirectShape<DP>::kSmem;
    if ((err = opt_in<attend_direct<T, DP>>(smem))) return err;
    const dim3 grid(w.splits, a.B * a.M, a.G * a.row_parts);
    err = launch_next(attend_direct<T, DP>, grid, kDirectWarps * 32, smem, st, a);
    if (err || w.splits == 1) return err;
    return launch_next(attend_join_direct<T, DP / 4>, a.B * a.M * a.H, 256, 0, st, a);
  }
  constexpr int TP = DP < 64 ? 64 : DP;  // the tiles' rows are 64 or 128 elements
  const uint32_t smem = TileShape<TP>::kSmem;
  if ((err = opt_in<attend_tiles<T, TP>>(smem))) return err;
  const uint64_t resident = (uint64_t)sm_count() * TileShape<TP>::kCtas;
  for (uint32_t b0 = 0; b0 < all.B; b0 += w.bc) {
    AttnArgs a = turn_args(all, b0, w.bc);
    if ((err = run_plan(a, w, st))) return err;
    const uint64_t tiles = (uint64_t)a.B * a.M * a.top * a.R / w.tile_rows + (uint64_t)a.B * a.nsb;
    for (a.g0 = 0; a.g0 < a.G; a.g0 += w.gc) {
      a.gc = std::min(w.gc, a.G - a.g0);
      if (tiles && (err = launch_next(attend_tiles<T, TP>,
                                      (uint32_t)std::min(tiles * a.gc, resident), kTileThreads,
                                      smem, st, a)))
        return err;
      const uint64_t rows = (uint64_t)a.B * a.M;
      const uint32_t parts = (uint32_t)ceil_div((uint64_t)a.gc * a.R * a.D, 128);
      if ((err = launch_next(attend_join<T>, (uint32_t)ceil_div(rows * parts, 8), 256, 0, st, a,
                             parts)))
        return err;
    }
  }
  return cudaSuccess;
}

template <class T, int DP>
cudaError_t launch_backward(const AttnArgs &all, const AttnPlan &w, cudaStream_t st) {
  cudaError_t err;
  const uint32_t smem = GradShape<DP>::kSmem;
  if ((err = opt_in<attend_grad<T, DP>>(smem))) return err;
  const uint64_t resident = (uint64_t)sm_count();
  for (uint32_t b0 = 0; b0 < all.B; b0 += w.bc) {
    AttnArgs a = turn_args(all, b0, w.bc);
    const uint64_t nq = (uint64_t)a.B * a.M;
    if ((err = run_plan(a, w, st))) return err;
    if (nq && (err = launch_next(grad_delta<T>, (uint32_t)ceil_div(nq * a.H, 32), 256, 0, st, a)))
      return err;
    const uint32_t spans = a.B * a.nsb;
    const uint64_t tiles = nq * a.top * a.R / w.tile_rows + spans;
    for (a.g0 = 0; a.g0 < a.G; a.g0 += w.gc) {
      a.gc = std::min(w.gc, a.G - a.g0);
      if (tiles && (err = launch_next(attend_grad<T, DP>,
                                      (uint32_t)std::min(tiles * a.gc, resident), kGradThreads,
                                      smem, st, a)))
        return err;
      if (nq * a.top * a.R > w.tile_rows && spans &&
          (err = launch_next(grad_join_keys<T>, dim3(spans, a.gc, 4), 256, 0, st, a,
                             1u << kGradSpanLog2)))
        return err;
      if (nq) {
        const uint32_t parts = (uint32_t)ceil_div((uint64_t)a.gc * a.R * a.D, 128);
        if ((err = launch_next(grad_join_queries<T>, (uint32_t)ceil_div(nq * parts, 8), 256, 0, st,
                               a, parts)))
          return err;
      }
    }
  }
  return cudaSuccess;
}

template <class T>
cudaError_t forward_of(const AttnArgs &a, const AttnPlan &w, cudaStream_t st) {
  switch (padded_dim(a.D)) {
    case 32: return launch_forward<T, 32>(a, w, st);
    case 64: return launch_forward<T, 64>(a, w, st);
    default: return launch_forward<T, 128>(a, w, st);
  }
}

template <class T>
cudaError_t backward_of(const AttnArgs &a, const AttnPlan &w, cudaStream_t st) {
  switch (padded_dim(a.D)) {
    case 32:
    case 64: return launch_backward<T, 64>(a, w, st);
    default: return launch_backward<T, 128>(a, w, st);
  }
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
  *bytes = plan_attention(*desc, backward != 0, nullptr).bytes;
  return NSFPS_OK;
}

int nsfps_block_attention_device(const nsfps_attention_desc *desc, const void *d_q,
                                 const void *d_k, const void *d_v, const int64_t *d_blocks,
                                 const int32_t *d_lengths, void *d_out, float *d_lse,
                                 void *d_rest, void *d_work, uint64_t work_bytes, void *stream) {
  clear_error();
  int rc = check_attention(desc);
  if (rc) return rc;
  const nsfps_attention_desc &d = *desc;
  if (d.batch * d.queries == 0) return NSFPS_OK;
  if (!d_q || !d_out || !d_blocks || (d.keys && (!d_k || !d_v)))
    return set_error(NSFPS_ERR_ARG, "NULL argument");
  if (((uint64_t)d_q | (uint64_t)d_k | (uint64_t)d_v | (uint64_t)d_out | (uint64_t)d_rest) % 16)
    return set_error(NSFPS_ERR_ARG, "q, k, v, out and rest must be 16-byte aligned");
  if ((uint64_t)d_blocks % 8 || ((uint64_t)d_lse | (uint64_t)d_lengths) % 4)
    return set_error(NSFPS_ERR_ARG, "a pointer is not aligned to its elements");
  const AttnPlan w = plan_attention(d, false, d_work);
  rc = check_work(d_work, work_bytes, w.bytes);
  if (rc) return rc;
  AttnArgs a = common_args(d, d_q, d_k, d_v, d_blocks, d_lengths, w);
  a.out = (char *)d_out;
  a.lse = d_lse;
  a.rest = (char *)d_rest;
  cudaStream_t st = (cudaStream_t)stream;
  NSFPS_FEATURE_CUDA(d.dtype == NSFPS_F16 ? forward_of<__half>(a, w, st)
                                          : forward_of<__nv_bfloat16>(a, w, st));
  return NSFPS_OK;
}

int nsfps_block_attention_grad_device(const nsfps_attention_desc *desc, const void *d_q,
                                      const void *d_k, const void *d_v, const int64_t *d_blocks,
                                      const int32_t *d_lengths, const void *d_out,
                                      const float *d_lse, const void *d_rest,
                                      const void *d_dout, void *d_dq,
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
       (uint64_t)d_rest | (uint64_t)d_dq | (uint64_t)d_dk | (uint64_t)d_dv) % 16)
    return set_error(NSFPS_ERR_ARG, "q, k, v, out, rest and the gradients must be 16-byte aligned");
  if ((uint64_t)d_blocks % 8 || ((uint64_t)d_lse | (uint64_t)d_lengths) % 4)
    return set_error(NSFPS_ERR_ARG, "a pointer is not aligned to its elements");
  const AttnPlan w = plan_attention(d, true, d_work);
  rc = check_work(d_work, work_bytes, w.bytes);
  if (rc) return rc;
  AttnArgs a = common_args(d, d_q, d_k, d_v, d_blocks, d_lengths, w);
  a.out_in = (const char *)d_out; a.lse_in = d_lse; a.dout = (const char *)d_dout;
  a.rest_in = (const char *)d_rest;
  a.dq = (char *)d_dq; a.dk = (char *)d_dk; a.dv = (char *)d_dv;
  cudaStream_t st = (cudaStream_t)stream;
  NSFPS_FEATURE_CUDA(d.dtype == NSFPS_F16 ? backward_of<__half>(a, w, st)
                                          : backward_of<__nv_bfloat16>(a, w, st));
  return NSFPS_OK;
}

}  // extern "C"
