/*
 * nsfps.h -- C ABI of the B200-native farthest-point-sampling engine
 * (ns_fps_b200).  Drop-in for the sampling path of satreeby/ns_fps
 * (`yuezu_fps()` and its pybind11 surface `yuezu_fps.yuezu_fps_module`).
 *
 * Plain pointers and sizes only.  Every entry point returns NSFPS_OK (0) or an
 * NSFPS_ERR_* code; nsfps_last_error() then describes the failure (the text is
 * thread-local).  The caller owns every buffer.  Calls are thread-safe; calls
 * on the same device are serialised internally.
 *
 * Results are bit-exact with the reference `yuezu_fps()` built without
 * multiply-add contraction: the same sample indices, in the same order, with
 * the same early stop.
 */
#ifndef NSFPS_H_
#define NSFPS_H_

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define NSFPS_API __attribute__((visibility("default")))
#else
#define NSFPS_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Compile-time constants of the reference (src/yuezu_fps.h:20-50), exposed
 * with the same names by the pybind11 module.  MORTON_BLOCK_SIZE and
 * CACHE_BLOCK_SIZE only shape the reference's internal tree; neither changes
 * which points are sampled. */
#define NSFPS_MORTON_BLOCK_SIZE 16
#define NSFPS_CACHE_BLOCK_SIZE 16
#define NSFPS_DEFAULT_X_BLOCKS 16
#define NSFPS_DEFAULT_Y_BLOCKS 16
#define NSFPS_DEFAULT_Z_BLOCKS 16
#define NSFPS_BOUNDARY_EPS 1e-6f

/* Limits of this engine (the reference allocates its bucket table up front
 * and is bounded by host memory instead). */
#define NSFPS_MAX_BLOCKS_PER_AXIS 1024u

enum nsfps_status {
  NSFPS_OK = 0,
  NSFPS_ERR_ARG = 1,         /* invalid argument (shape, range, pointer) */
  NSFPS_ERR_CUDA = 2,        /* a CUDA runtime call failed */
  NSFPS_ERR_OOM = 3,         /* device or host allocation failed */
  NSFPS_ERR_TIMEOUT = 4,     /* a bounded in-kernel wait gave up */
  NSFPS_ERR_UNSUPPORTED = 5  /* input beyond this engine's limits */
};

/* The user-facing part of the reference's SpaceRange (src/yuezu_fps.h:56-83):
 * bounds and per-axis block counts.  The derived fields (inv_bs, bit counts,
 * Morton LUTs) are recomputed from these exactly as make_range() does
 * (src/yuezu_fps.cpp:136-161) every time the range is used. */
typedef struct nsfps_range {
  float min_x, max_x;
  float min_y, max_y;
  float min_z, max_z;
  uint32_t x_blocks, y_blocks, z_blocks;
} nsfps_range;

/* Derived fields of a range, as the reference computes them. */
typedef struct nsfps_range_info {
  float inv_bs[3];       /* 1.0f / ((max - min) / (float)blocks)   src/yuezu_fps.cpp:140-142 */
  float block_size[3];   /* (max - min) / blocks                    src/yuezu_fps.cpp:7-11 */
  uint32_t bits[3];      /* max(1, ceil(log2(blocks)))              src/yuezu_fps.cpp:13-32 */
  uint32_t total_bits;   /* bits[0] + bits[1] + bits[2]             src/yuezu_fps.cpp:34-36 */
  uint64_t total_blocks; /* x_blocks * y_blocks * z_blocks          src/yuezu_fps.cpp:38-40 */
} nsfps_range_info;

/* Text of the last error on this thread ("" when none). */
NSFPS_API const char *nsfps_last_error(void);

/* Library version (major * 10000 + minor * 100 + patch). */
NSFPS_API int nsfps_version(void);

/* Number of CUDA devices visible to the library. */
NSFPS_API int nsfps_device_count(int *count);

/* make_range(): fills *out (replaces src/yuezu_fps.cpp:136-161 and the
 * pybind11 binding yuezu_fps/yuezu_fps_pybind.cpp:128-130). */
NSFPS_API int nsfps_make_range(float min_x, float max_x, float min_y, float max_y,
                     float min_z, float max_z, uint32_t x_blocks,
                     uint32_t y_blocks, uint32_t z_blocks, nsfps_range *out);

/* make_uniform_range(): blocks_per_dim on every axis (replaces
 * src/yuezu_fps.cpp:98-134, binding yuezu_fps_pybind.cpp:132-134). */
NSFPS_API int nsfps_make_uniform_range(float min_x, float max_x, float min_y,
                             float max_y, float min_z, float max_z,
                             uint32_t blocks_per_dim, nsfps_range *out);

/* SpaceRange::block_size_* / *_bits / total_bits / total_blocks and the
 * inv_bs fields (replaces src/yuezu_fps.cpp:7-40, yuezu_fps_pybind.cpp:118-125).
 * Fails with NSFPS_ERR_ARG for zero block counts. */
NSFPS_API int nsfps_range_get_info(const nsfps_range *r, nsfps_range_info *info);

/* Per-axis Morton LUT (x_lut_/y_lut_/z_lut_, src/yuezu_fps.cpp:52-97).
 * axis 0..2; lut receives 2^bits entries when cap allows; *len gets 2^bits. */
NSFPS_API int nsfps_range_get_lut(const nsfps_range *r, int axis, uint32_t *lut,
                        uint64_t cap, uint64_t *len);

/* compute_bbox(points, xb, yb, zb): bounds of the cloud widened by
 * BOUNDARY_EPS; an empty cloud gives [0,1]^3 with 1x1x1 blocks (replaces
 * src/yuezu_fps.cpp:643-670).  Runs on the host. */
NSFPS_API int nsfps_compute_bbox(const float *xyz, uint64_t n, uint32_t x_blocks,
                       uint32_t y_blocks, uint32_t z_blocks, nsfps_range *out);

/* Farthest point sampling of one cloud (replaces yuezu_fps(),
 * src/yuezu_fps.h:211-212 / src/yuezu_fps.cpp:676-730, as bound by
 * fps_numpy, yuezu_fps/yuezu_fps_pybind.cpp:67-86).
 *   xyz     n x 3 floats, dense, HOST memory
 *   range   NULL selects compute_bbox(points, 16, 16, 16) like fps(range=None)
 *   out     HOST buffer of capacity min(k, n) receiving original indices
 *   out_len receives the number of samples (< k when every remaining point is
 *           at distance 0 from the samples, as in the reference)
 *   device  CUDA device ordinal */
NSFPS_API int nsfps_fps(const float *xyz, uint64_t n, uint64_t k,
              const nsfps_range *range, uint64_t *out, uint64_t *out_len,
              int device);

/* fps_with_bbox(points, k, xb, yb, zb) (replaces
 * yuezu_fps/yuezu_fps_pybind.cpp:88-101). */
NSFPS_API int nsfps_fps_with_bbox(const float *xyz, uint64_t n, uint64_t k,
                        uint32_t x_blocks, uint32_t y_blocks,
                        uint32_t z_blocks, uint64_t *out, uint64_t *out_len,
                        int device);

/* Batched sampling: `count` independent clouds, the same k for each, whole
 * clouds sharded across `ndev` devices (one host thread per device, no
 * inter-GPU traffic).  Each cloud i is n[i] x 3 host floats; ranges holds one
 * range shared by all clouds (per_cloud_ranges == 0) or `count` ranges;
 * a NULL ranges selects compute_bbox(cloud, 16, 16, 16) per cloud.  out[i]
 * has capacity min(k, n[i]); out_len[i] receives each length.  devices == NULL
 * uses devices 0..ndev-1.  The reference has no batched entry point; this
 * replaces a loop of fps() calls (yuezu_fps_pybind.cpp:67-86). */
NSFPS_API int nsfps_fps_batched(const float *const *clouds, const uint64_t *n,
                      uint64_t count, uint64_t k, const nsfps_range *ranges,
                      int per_cloud_ranges, uint64_t *const *out,
                      uint64_t *out_len, const int *devices, int ndev);

/* Device-resident sampling for callers that keep clouds in HBM: `count`
 * clouds packed back to back in d_xyz (offsets[i]..offsets[i+1] points,
 * offsets in HOST memory, count + 1 entries), ranges as in
 * nsfps_fps_batched (host memory; NULL selects compute_bbox(cloud, 16, 16,
 * 16) per cloud, like fps(range=None), with the min/max reduction done on the
 * device, src/yuezu_fps.cpp:643-670), d_out a DEVICE buffer of
 * count * k uint64 (cloud i at d_out + i * k), out_len a HOST array of
 * `count` lengths.  Work is issued on `stream` (a cudaStream_t; NULL = the
 * legacy default stream) of the current device; the call returns after the
 * lengths are known (it synchronises `stream`).  No reference counterpart
 * (the reference is host-only); it exists so callers avoid a host round trip
 * per call. */
NSFPS_API int nsfps_fps_device(const float *d_xyz, const uint64_t *offsets,
                     uint64_t count, uint64_t k, const nsfps_range *ranges,
                     int per_cloud_ranges, uint64_t *d_out, uint64_t *out_len,
                     void *stream);

/* fps_with_bbox() for device-resident clouds: nsfps_fps_device with every
 * cloud's bounding box (reduced on the device, widened by BOUNDARY_EPS as in
 * compute_bbox) and x_blocks x y_blocks x z_blocks blocks (replaces the
 * binding yuezu_fps/yuezu_fps_pybind.cpp:88-101 and src/yuezu_fps.cpp:
 * 643-670 for clouds in HBM; it is also the range the reference's KITTI
 * benchmark builds, eval/src_cpu/compare_cpu_test_kitti.cpp:230-245). */
NSFPS_API int nsfps_fps_device_with_bbox(const float *d_xyz, const uint64_t *offsets,
                               uint64_t count, uint64_t k, uint32_t x_blocks,
                               uint32_t y_blocks, uint32_t z_blocks, uint64_t *d_out,
                               uint64_t *out_len, void *stream);

/* Limits of nsfps_fps_device_static(): points per call, and the size of the
 * fixed device scratch array that holds every intermediate buffer. */
#define NSFPS_STATIC_MAX_POINTS 65536u
#define NSFPS_STATIC_SCRATCH_BYTES (8u << 20)

/* No counterpart in the reference (which is host-only).  One device-resident
 * cloud, sampled without allocating any device memory: for callers that
 * cannot allocate mid-run, such as a host that has given all device memory to
 * its own pool, or a latency-bound loop where cudaMalloc / cudaFree would
 * synchronise the device.  Every intermediate buffer lives in one fixed
 * scratch array of NSFPS_STATIC_SCRATCH_BYTES per device, reserved with the
 * library's device code.
 *   d_xyz   n x 3 floats in DEVICE memory of the current device
 *   n       1 <= k < n <= NSFPS_STATIC_MAX_POINTS; larger n fails with
 *           NSFPS_ERR_ARG before any device work (k >= n or k == 0 fail with
 *           NSFPS_ERR_UNSUPPORTED, as in nsfps_fps_device)
 *   range   HOST memory, non-NULL
 *   d_out   DEVICE buffer of k uint64 (original indices)
 *   out_len HOST; receives the number of samples
 *   stream  cudaStream_t of the current device (NULL = legacy default stream)
 * Samples are identical to nsfps_fps_device() on the same input.  The first
 * call on a device resolves the array's address (cudaGetSymbolAddress, with
 * that device current) and creates the device's timing events; make that
 * first call before any stream capture.  The array is shared by all calls on
 * a device, so overlapping calls would race on it: calls take a per-device
 * lock and return only after their work on `stream` has finished, which runs
 * them one at a time.  Each call clears the counters that must start at zero
 * itself (cudaMemsetAsync on `stream`). */
NSFPS_API int nsfps_fps_device_static(const float *d_xyz, uint64_t n, uint64_t k,
                            const nsfps_range *range, uint64_t *d_out,
                            uint64_t *out_len, void *stream);

/* ---- Grouping after sampling.  No counterpart in the reference, which stops
 * at the sample indices (src/yuezu_fps.cpp:676-730, yuezu_fps_pybind.cpp:
 * 137-143); these are the operators a PointNet++-style pipeline applies to
 * them next.
 *
 * Ball query (PointNet++ query_ball_point semantics): for centre j, the first
 * `nsample` points k of its cloud in index order with d2 < radius * radius,
 * d2 = (dx*dx + dy*dy) + dz*dz, dx = x_k - cx, every operation fp32 rounded
 * to nearest with no multiply-add contraction (the sampler's distance,
 * src/yuezu_fps.cpp:205-209).  idx[j * nsample + s] holds point indices
 * within the cloud, ascending; slots past the hits repeat the first hit; a
 * centre with no hit gets 0 in every slot.  hits[j] = min(number of hits,
 * nsample).  Points with a non-finite coordinate are never hits; a negative
 * radius acts as its magnitude, a NaN or zero radius finds nothing. */
#define NSFPS_MAX_NSAMPLE 1024u

/* Device-resident, batched: `count` clouds packed in d_xyz
 * (point_offsets[i]..point_offsets[i+1]) and their centres packed in
 * d_centers (center_offsets[i]..center_offsets[i+1]); offsets in HOST memory
 * (count + 1 entries each).  d_idx (m x nsample int64) and d_hits (m uint32,
 * may be NULL) are DEVICE buffers indexed from the first centre of the call.
 * Work is issued on `stream` of the current device; the call returns after
 * the stream has drained (the per-device workspace is reused by the next
 * call).  Inputs are not modified. */
NSFPS_API int nsfps_ball_query_device(const float *d_xyz, const uint64_t *point_offsets,
                            const float *d_centers, const uint64_t *center_offsets,
                            uint64_t count, float radius, uint32_t nsample, int64_t *d_idx,
                            uint32_t *d_hits, void *stream);

/* The same for one cloud in HOST memory (n x 3 points, m x 3 centres);
 * idx (m x nsample) and hits (m, may be NULL) are HOST buffers. */
NSFPS_API int nsfps_ball_query(const float *xyz, uint64_t n, const float *centers, uint64_t m,
                     float radius, uint32_t nsample, int64_t *idx, uint32_t *hits,
                     int device);

/* Gather of sampled points (PointNet++ gather_operation on coordinates):
 * d_out[3j + a] = coordinate a of point d_idx[j] of entry j's cloud; entries
 * packed per cloud by idx_offsets (HOST, count + 1), points by point_offsets.
 * Device buffers, current device, returns after `stream` drained.  An index
 * outside its cloud gives NaNs at its entry and NSFPS_ERR_ARG. */
NSFPS_API int nsfps_gather_points_device(const float *d_xyz, const uint64_t *point_offsets,
                               const int64_t *d_idx, const uint64_t *idx_offsets,
                               uint64_t count, float *d_out, void *stream);

/* Grouped coordinates relative to each centre (PointNet++ grouping of
 * xyz followed by the subtraction of the centre): d_out[((j * nsample) + s)
 * * 3 + a] = xyz[d_idx[j * nsample + s]][a] - centers[j][a] (fp32, round to
 * nearest), d_idx as written by nsfps_ball_query_device.  Errors as in
 * nsfps_gather_points_device. */
NSFPS_API int nsfps_group_points_device(const float *d_xyz, const uint64_t *point_offsets,
                              const float *d_centers, const uint64_t *center_offsets,
                              uint64_t count, uint32_t nsample, const int64_t *d_idx,
                              float *d_out, void *stream);

/* ---- Features of sampled clouds: row lookup by index with its gradient, the
 * choice of the nearest blocks of a cloud, and attention over chosen blocks
 * with its gradient.  No counterpart in the reference, which stops at the
 * sample indices; these are what a point network does with them next.
 *
 * All of these calls are asynchronous: they issue kernels on `stream` of the
 * current device and return.  They keep no state and allocate nothing; scratch
 * comes from the caller (`d_work`, at least the bytes the matching _workspace
 * call gives, 256-byte aligned), so calls on different streams, or captured
 * into different graphs, need only have different scratch.  Results do not
 * depend on how the work is scheduled: the same inputs give the same bits.
 * Waits inside the attention kernels are bounded (2 s; no working call comes
 * near).  A call that does not wait cannot report one that runs out: the out and
 * lse of its clouds are then NaN, and of a gradient dq and every part of dk and
 * dv that the CTA in question had in hand. */
enum nsfps_dtype { NSFPS_F32 = 0, NSFPS_F16 = 1, NSFPS_BF16 = 2 };

/* Lookup of `count` rows per batch entry in a table of `rows` rows of `width`
 * elements, times `scale` (the product taken in fp32 and rounded once):
 *   out[b][p][:] = scale * table[b][idx[b][p]][:]
 * A negative index stands for no row: zeros, and no gradient.  An index of
 * `rows` or more reads nothing: its output row is NaN, its gradient goes
 * nowhere.  The table's elements are contiguous within a row; batch_stride
 * and row_stride are in elements.  idx (batch x count int64) and out are
 * dense. */
typedef struct nsfps_rows_desc {
  uint64_t batch, rows, width, count;
  int64_t batch_stride, row_stride;
  float scale;
  int32_t dtype; /* nsfps_dtype of table and out */
} nsfps_rows_desc;

NSFPS_API int nsfps_gather_rows_device(const nsfps_rows_desc *desc, const void *d_table,
                                       const int64_t *d_idx, void *d_out, void *stream);

/* Gradient of the lookup with respect to the table (dense, batch x rows x
 * width; the strides of `desc` are not used):
 *   dtable[b][n][:] = scale * sum over p with idx[b][p] == n of dout[b][p][:]
 * summed in fp32 in a fixed order of p and rounded once; rows that no index
 * names are written as zeros.  batch * count and batch * rows below 2^31, width
 * below 2^20. */
NSFPS_API int nsfps_gather_rows_grad_workspace(const nsfps_rows_desc *desc, uint64_t *bytes);
NSFPS_API int nsfps_gather_rows_grad_device(const nsfps_rows_desc *desc, const void *d_dout,
                                            const int64_t *d_idx, void *d_dtable, void *d_work,
                                            uint64_t work_bytes, void *stream);

/* Nearest blocks of a cloud.  Block j of a cloud is its points [j * block,
 * (j + 1) * block) below the cloud's length; its distance to a centre is that
 * of the block's bounding box, squared, in the sampler's arithmetic:
 *   dx = max(max(lo_x - c_x, c_x - hi_x), 0), ...  d2 = (dx*dx + dy*dy) + dz*dz
 * every operation fp32 rounded to nearest without contraction.  d_blocks
 * receives, per centre, the `top` blocks of smallest (d2, j), ascending, and
 * d_d2 (may be NULL) their d2; slots beyond the cloud's blocks get -1 and
 * +inf.  d_xyz: batch x n x 3 and d_centers: batch x m x 3 floats, dense;
 * d_lengths: batch int32 (clamped to 0..n), or NULL when every cloud has n
 * points.  A NaN point coordinate is left out of its box, a NaN centre
 * coordinate counts as inside every box.  block: 16, 32, 64 or 128; top:
 * 1..NSFPS_MAX_TOP; batch * m and batch * n below 2^31. */
#define NSFPS_MAX_TOP 64u
typedef struct nsfps_select_desc {
  uint64_t batch, points, centers;
  uint32_t block, top;
} nsfps_select_desc;

NSFPS_API int nsfps_select_blocks_workspace(const nsfps_select_desc *desc, uint64_t *bytes);
NSFPS_API int nsfps_select_blocks_device(const nsfps_select_desc *desc, const float *d_xyz,
                                         const int32_t *d_lengths, const float *d_centers,
                                         int64_t *d_blocks, float *d_d2, void *d_work,
                                         uint64_t work_bytes, void *stream);

/* Attention of every query over the blocks chosen for it:
 *   out[b][m][h] = sum_t p_t v[b][t][g], p = softmax_t(scale * q[b][m][h] . k[b][t][g]),
 * g = h / (heads / kv_heads), t over the keys below the cloud's length of the
 * blocks that blocks[b][m][0 .. top) lists.  The list is a set: an entry that
 * occurs again, is negative or names no block of the cloud counts for nothing.
 * A query without a key gets zeros (and no gradient).  What lies behind a
 * cloud's length, in blocks that no query of the cloud lists, or in rows of
 * queries that list nothing, is never part of a result, whatever its value;
 * what is listed has to be finite (a value that is not may also reach results
 * of queries and keys nearby that do not list it), and so have its products:
 * q . k, and that times scale * log2(e), in fp32.
 * q, k and v: F16 or BF16, elements of a head contiguous, 16-byte aligned, the
 * strides (batch, row, head, in elements) multiples of 8.  blocks (batch x
 * queries x top int64), out (batch x queries x heads x head_dim) and lse
 * (batch x queries x heads fp32: log of the softmax sum, -inf without a key;
 * may be NULL) are dense; so is rest (like out; may be NULL), which takes what
 * the rounding of out left, for the gradient.  head_dim: a multiple of 8 up to 128; block: 16, 32,
 * 64 or 128; top: 1..NSFPS_MAX_TOP; heads a multiple of kv_heads, at most 256.
 * batch below 2^27, batch * queries * top and batch * keys below 2^30, queries *
 * top * heads / kv_heads below 2^31. */
typedef struct nsfps_attention_desc {
  uint64_t batch, queries, keys;
  uint32_t heads, kv_heads, head_dim, block, top;
  int32_t dtype;
  int64_t q_stride[3], k_stride[3], v_stride[3];
  float scale;
  uint32_t reserved; /* 0 */
} nsfps_attention_desc;

/* Scratch of the forward (backward == 0) or the gradient call.  Most of it are
 * partial results: for each cloud and key head
 *   queries * top * heads / kv_heads * 4 * (head_dim + 1) bytes
 * (the gradient half as much again, and keys * 8 * head_dim).  Key heads and
 * clouds are taken in turns while these pass 1 GiB; the queries of one cloud are
 * not, so one cloud and key head may take more than that: split such a call by
 * queries where it does not fit (the gradient's dk and dv of the parts add up). */
NSFPS_API int nsfps_block_attention_workspace(const nsfps_attention_desc *desc, int backward,
                                              uint64_t *bytes);
NSFPS_API int nsfps_block_attention_device(const nsfps_attention_desc *desc, const void *d_q,
                                           const void *d_k, const void *d_v,
                                           const int64_t *d_blocks, const int32_t *d_lengths,
                                           void *d_out, float *d_lse, void *d_rest,
                                           void *d_work, uint64_t work_bytes, void *stream);

/* Gradient: dq (dense, like out), dk and dv (dense, batch x keys x kv_heads x
 * head_dim; keys that no query reads get zeros) from dout (dense, like out,
 * 16-byte aligned) and the forward's out, lse and rest.  Without rest (NULL)
 * the gradient takes out as it is rounded, which dq and dk of queries with few
 * weighty keys feel.  The weights p and the score gradients ds are rounded to
 * the inputs' type for the products; in F16 both are first multiplied by powers
 * of two (ds by one that follows the sizes of dout and v), so neither overflows
 * nor sinks among the smallest numbers where the results do not. */
NSFPS_API int nsfps_block_attention_grad_device(const nsfps_attention_desc *desc, const void *d_q,
                                                const void *d_k, const void *d_v,
                                                const int64_t *d_blocks,
                                                const int32_t *d_lengths, const void *d_out,
                                                const float *d_lse, const void *d_rest,
                                                const void *d_dout,
                                                void *d_dq, void *d_dk, void *d_dv, void *d_work,
                                                uint64_t work_bytes, void *stream);

/* Timing and work counters of the last call on this thread: stage times in
 * milliseconds measured with CUDA events on the launching stream (setup =
 * binning, sort and leaf build; loop = the persistent sampling kernel;
 * total = first to last event), the number of kernel launches, and the work
 * counters of the sampling loop: points in the buckets the reference updates
 * (summed over iterations), points actually re-evaluated after the exact
 * bounding-box skip, and the loop configuration (CTAs per cloud and mode:
 * 0 = per-step cluster loop, 2 = round-based cluster loop, 3 = round-based
 * loop over co-resident CTAs: 64 or 128 for a single cloud of at least 4,096
 * points, groups of up to 16 for a batch when the device cannot hold a
 * cluster per cloud).  After a ball query (mode 4): setup = the grid build,
 * loop = the query kernel, launches = its kernel launches; the work counters
 * are 0.
 * Enabled by nsfps_set_profiling. */
typedef struct nsfps_profile {
  float setup_ms, loop_ms, total_ms;
  uint32_t launches;
  uint32_t ctas_per_cloud;
  uint32_t mode;
  uint32_t leaves;
  uint64_t ref_points_updated;
  uint64_t points_evaluated;
  uint64_t iterations;
} nsfps_profile;

NSFPS_API int nsfps_set_profiling(int enable);
NSFPS_API int nsfps_last_profile(nsfps_profile *out);

/* ---- Test hooks.  No counterpart in the reference, whose GPU prototype
 * ignores CUDA errors (eval/src_gpu/yuezu_fps_gpu_optimized.cu:904-910) and
 * whose CPU path has no failure mode to test.  They drive this engine's error
 * paths without faulting the GPU:
 *   wait_limit_ns      limit of every bounded in-kernel wait (0 = the default,
 *                      2 s; the queue polling of worker warps gets twice it)
 *   withhold_cta       rank, among the CTAs of cloud 0, of one CTA that does
 *                      not publish its round-`withhold_step` candidate list
 *                      (round loops) or its step-`withhold_step` proposals
 *                      (per-step loop); every wait for it then runs out and
 *                      the call returns NSFPS_ERR_TIMEOUT with the device
 *                      still usable.  -1 = none.  In the attention kernels on
 *                      tiles: the CTA of the grid that does not announce a
 *                      product of its first tile or item; the results are then
 *                      NaN, as said above.
 *   withhold_step      the round (round loops, from 0) or step (per-step loop,
 *                      from 1) at which it withholds; attention: 0 the scores,
 *                      1 (gradient only) the products behind them
 *   fail_alloc_device  the next workspace request of an allocating entry point
 *                      on this device fails as if cudaMalloc had run out of
 *                      memory (NSFPS_ERR_OOM); it fires once.  -1 = none.
 * The hooks are process-wide and stay set until replaced; NULL restores the
 * defaults.  Not for production use. */
typedef struct nsfps_test_hooks {
  uint64_t wait_limit_ns;
  int32_t withhold_cta;
  uint32_t withhold_step;
  int32_t fail_alloc_device;
  int32_t reserved;
} nsfps_test_hooks;

NSFPS_API int nsfps_set_test_hooks(const nsfps_test_hooks *hooks);

#ifdef __cplusplus
}
#endif

#endif /* NSFPS_H_ */
