// ilqr_gradclip.h -- launch records of the gradient norm and clipping kernels
// (ilqr_gradclip.cu), filled by the entry points in ilqr_gradclip_abi.cu.
#ifndef ILQR_GRADCLIP_H
#define ILQR_GRADCLIP_H

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace ilqr {

// One dense tensor of a list: its values are cut into chunks of chunk_bytes,
// numbered through the list; chunk0 is its first. Every tensor has at least
// one chunk (an empty one, a chunk without values).
struct GradEntry {
  const void* in;
  void* out;
  int64_t numel;
  uint32_t chunk0;
  uint32_t dtype;
};

// Kernel parameters hold at most 32764 bytes: longer lists take several
// launches. Shorter tables keep the parameter copy of shorter lists small (host
// time of a launch with 2 KB of them 2.4 us, 8 KB 3.1 us, 32 KB 5.5 us).
constexpr int GRAD_CAP_SHORT = 60;
constexpr int GRAD_CAP_MIDDLE = 240;
constexpr int GRAD_CAP_LONG = 1000;

template <int CAP>
struct GradTable {
  int32_t n;
  uint32_t chunks;
  uint32_t chunk_bytes;
  uint32_t in_place;  // whether every out is its in
  GradEntry e[CAP];
};

// A wave: four blocks of 256 threads on each SM.
constexpr int GRAD_MAX_GRID = 148 * 4;
constexpr uint32_t GRAD_CHUNK_BYTES = 16384;

// A list beyond this size does not stay in L2 between the two passes (300 MB,
// us as a shorter list | as a long one: 155 | 140; 80 MB 42 | 40, 48 MB 26 | 27).
// Its first pass leaves the last GRAD_KEEP_BYTES for the second to find; its
// scaling takes GRAD_LONG_STEP chunks a block at a time, GRAD_LONG_GRID blocks at
// most: with fewer of them, each with a larger share, the last to end is waited
// for (a wave of eight on an SM: 137 us for 275 MB, two 135, three 131, four 129,
// one for every step 129). Beyond GRAD_CAP_LONG tensors both passes go through
// the list's tables from the first to the last, and the sums of each table leave
// its own last GRAD_KEEP_BYTES: the scaling finds less in L2 then (200 MB bf16 of
// 200 tensors 99 us, of 1500, with two launches more, 113).
constexpr int64_t GRAD_LONG_BYTES = 64 << 20;
constexpr int64_t GRAD_KEEP_BYTES = 90 << 20;
constexpr uint32_t GRAD_LONG_STEP = 2;
constexpr unsigned GRAD_LONG_GRID = 148 * 8 * 4;

// A list up to this size is short: one cluster takes it, in one launch instead
// of two (two | one, us of GPU time and of an eager call: clipping 128 KB
// 4.1 | 4.3 and 8.4 | 6.9; 512 KB 4.2 | 6.2 and 8.5 | 8.5).
constexpr int64_t GRAD_SMALL_BYTES = 128 << 10;
constexpr uint32_t GRAD_SMALL_CHUNK_BYTES = 4096;
constexpr int GRAD_SMALL_BLOCKS = 8;

struct GradNormOut {
  float* norm;          // may be null
  float* tensor_norms;  // may be null
  double* total;        // may be null
};

struct GradScale {
  double max_norm;
  double eps;
  int32_t max_type;  // 1: largest magnitude, 0: 2-norm
};

// One tensor of the per-element form: row b is n_seg segments of seg_vecs
// vectors of vec_bytes; strides in bytes.
struct RowTensor {
  const char* in;
  char* out;
  int64_t in_row, in_seg, out_row, out_seg;
  uint32_t n_seg, seg_vecs;
  uint32_t vec_bytes, dtype;
  uint32_t magic, shift;  // i / seg_vecs = i magic >> (32 + shift)
  uint32_t staged;        // where the slice is staged, from the element's place
  uint32_t staged_vecs;   // 16-byte words that it takes there
  uint32_t seg_bytes;
  uint32_t place;         // bytes from one staged segment to the next
  uint32_t bulk;          // what moves it
  uint32_t pad;
};

constexpr uint32_t ROW_THREADS = 0;    // the threads, a vector each
constexpr uint32_t ROW_BULK = 1;       // bulk copies: its segments are whole 16-byte words
constexpr uint32_t ROW_BULK_ENDS = 2;  // bulk copies, and the threads at the segments' ends

constexpr int ROW_MAX_TENSORS = 8;

struct RowTable {
  RowTensor t[ROW_MAX_TENSORS];
  int32_t n;
  int32_t zero_nonfinite;
  int64_t B;
  double max_norm, eps;
  float* norms;
  uint32_t staged_bytes;  // of an element, every slice from a multiple of 16
  uint32_t bulk;          // whether bulk copies move any of it
  uint32_t one_dtype;
  uint32_t pad;
};

// Of the 227 KB of shared memory that a block can have.
constexpr uint32_t GRAD_MAX_STAGED = 224 * 1024;
// Segments from this many bytes on move by bulk copies.
constexpr uint32_t GRAD_MIN_BULK = 256;

// Partial sums of a launch: one for each block. keep_chunks > 0: what lies before
// that many of the last chunks will not be found in L2 and leaves it first.
template <int CAP>
cudaError_t launch_grad_sum(const GradTable<CAP>& tab, int grid, bool max_type, uint32_t keep_chunks, double* slots,
                            cudaStream_t stream);
// One for each (block, tensor) that meet, at slot block + tensor.
template <int CAP>
cudaError_t launch_grad_each(const GradTable<CAP>& tab, int grid, bool max_type, double* slots, cudaStream_t stream);
// Joins n_slots partials into the norm; with tab != nullptr also the norms of
// its tensors from the launch's own slots (tab_slots, grid).
template <int CAP>
cudaError_t launch_grad_join(const GradTable<CAP>* tab, int grid, const double* tab_slots, bool max_type,
                             const double* slots, int64_t n_slots, const GradNormOut& out, bool want_global,
                             cudaStream_t stream);
template <int CAP>
cudaError_t launch_grad_scale(const GradTable<CAP>& tab, int grid, const GradScale& s, const double* slots,
                              int64_t n_slots, float* norm, bool dependent, cudaStream_t stream);
template <int CAP>
cudaError_t launch_grad_scale_long(const GradTable<CAP>& tab, const GradScale& s, const double* total, float* norm,
                                   bool dependent, cudaStream_t stream);
// A short list in one launch; s == nullptr: its norm only.
template <int CAP>
cudaError_t launch_grad_small(const GradTable<CAP>& tab, bool max_type, const GradScale* s, const GradNormOut& out,
                              cudaStream_t stream);
cudaError_t launch_grad_rows(const RowTable& tab, cudaStream_t stream);

}  // namespace ilqr

#endif
