// ilqr_gradclip_abi.cu -- extern "C" entry points of the gradient norms and
// clipping (include/ilqr_b200.h). The host arrays that describe the tensors
// are read during the call only: what the kernels need of them travels in the
// launch parameters, so a captured call keeps nothing of the caller's.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <vector>

#include "ilqr_b200.h"
#include "ilqr_gradclip.h"
#include "ilqr_overlap.h"

namespace {

using ilqr::GradEntry;
using ilqr::GradTable;

int status_of(cudaError_t e) { return e == cudaSuccess ? ILQR_OK : ILQR_ERR_CUDA; }

bool aligned(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

int64_t size_of(int32_t dtype) { return dtype == ILQR_DTYPE_F32 ? 4 : 2; }

constexpr int64_t MAX_VALUES = (int64_t)1 << 40;  // of a list: chunk numbers stay in 32 bits

struct List {
  const void* const* in;
  void* const* out;  // nullptr: norm only
  const int64_t* numel;
  const int32_t* dtype;
  int32_t n;
};

int check_list(const List& l, int32_t norm_type) {
  if (l.n < 0 || (norm_type != ILQR_NORM_L2 && norm_type != ILQR_NORM_MAX)) return ILQR_ERR_INVALID_ARGUMENT;
  if (l.n > 0 && (l.in == nullptr || l.numel == nullptr || l.dtype == nullptr)) return ILQR_ERR_INVALID_ARGUMENT;
  int64_t values = 0;
  for (int32_t i = 0; i < l.n; ++i) {
    if (l.dtype[i] < ILQR_DTYPE_F32 || l.dtype[i] > ILQR_DTYPE_BF16) return ILQR_ERR_INVALID_ARGUMENT;
    if (l.numel[i] < 0 || l.numel[i] > MAX_VALUES) return ILQR_ERR_INVALID_ARGUMENT;
    values += l.numel[i];
    if (values > MAX_VALUES) return ILQR_ERR_INVALID_ARGUMENT;
    if (l.numel[i] == 0) continue;
    const uintptr_t low = (uintptr_t)size_of(l.dtype[i]) - 1;
    if (l.in[i] == nullptr || (l.out != nullptr && l.out[i] == nullptr)) return ILQR_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)l.in[i] & low) || (l.out != nullptr && ((uintptr_t)l.out[i] & low))) return ILQR_ERR_MISALIGNED;
  }
  return ILQR_OK;
}

struct Span {
  uintptr_t lo, hi;
};

void sort_spans(std::vector<Span>& s) {
  const auto before = [](const Span& a, const Span& b) { return a.lo < b.lo; };
  if (!std::is_sorted(s.begin(), s.end(), before)) std::sort(s.begin(), s.end(), before);
}

bool any_meets(const std::vector<Span>& s, const void* p, size_t bytes) {
  const uintptr_t lo = (uintptr_t)p, hi = lo + bytes;
  return p != nullptr && std::any_of(s.begin(), s.end(), [=](const Span& x) { return x.lo < hi && lo < x.hi; });
}

// Whether a value that the call writes is also one that it writes or reads
// elsewhere: blocks run in no order, so only a tensor's own input may be its
// output, whole.
bool overlaps(const List& l, const double* total, const float* norm) {
  std::vector<Span> outs, ins;  // of those that are not in place
  outs.reserve((size_t)l.n);
  for (int32_t i = 0; i < l.n; ++i) {
    if (l.numel[i] == 0) continue;
    const uintptr_t bytes = (uintptr_t)(l.numel[i] * size_of(l.dtype[i]));
    const uintptr_t q = (uintptr_t)l.out[i], p = (uintptr_t)l.in[i];
    outs.push_back({q, q + bytes});
    if (p != q) ins.push_back({p, p + bytes});
  }
  sort_spans(outs);
  for (size_t k = 1; k < outs.size(); ++k)
    if (outs[k].lo < outs[k - 1].hi) return true;
  sort_spans(ins);
  size_t k = 0;
  for (const Span& x : ins) {
    while (k < outs.size() && outs[k].hi <= x.lo) ++k;
    if (k < outs.size() && outs[k].lo < x.hi) return true;
  }
  // the first block writes the norm while others may still read
  if (total != nullptr) ins.push_back({(uintptr_t)total, (uintptr_t)(total + 1)});
  return any_meets(outs, total, sizeof(*total)) || any_meets(outs, norm, sizeof(*norm)) ||
         any_meets(ins, norm, sizeof(*norm));
}

uint64_t chunks_of(int64_t numel, int32_t dtype, uint32_t chunk_bytes) {
  const uint64_t c = ((uint64_t)(numel * size_of(dtype)) + chunk_bytes - 1) / chunk_bytes;
  return c > 0 ? c : 1;
}

int64_t bytes_of(const List& l) {
  int64_t bytes = 0;
  for (int32_t i = 0; i < l.n; ++i) bytes += l.numel[i] * size_of(l.dtype[i]);
  return bytes;
}

// Whether a list is short enough for the one-launch form.
bool is_small(const List& l) { return l.n <= ilqr::GRAD_CAP_SHORT && bytes_of(l) <= ilqr::GRAD_SMALL_BYTES; }

template <int CAP>
void fill(GradTable<CAP>& tab, const List& l, int32_t first, int32_t n,
          uint32_t chunk_bytes = ilqr::GRAD_CHUNK_BYTES) {
  tab.n = n;
  tab.chunk_bytes = chunk_bytes;
  tab.in_place = 1;
  uint64_t at = 0;
  for (int32_t i = 0; i < n; ++i) {
    const int32_t k = first + i;
    tab.e[i] = GradEntry{l.in[k], l.out != nullptr ? l.out[k] : nullptr, l.numel[k], (uint32_t)at,
                         (uint32_t)l.dtype[k]};
    if (tab.e[i].in != tab.e[i].out) tab.in_place = 0;
    at += chunks_of(l.numel[k], l.dtype[k], chunk_bytes);
  }
  tab.chunks = (uint32_t)at;
}

int grid_of(uint32_t chunks) { return (int)std::min<uint32_t>(chunks, (uint32_t)ilqr::GRAD_MAX_GRID); }

// Slots that the partial sums of a list take, at most.
size_t slots_of(int32_t n) {
  const size_t launches = ((size_t)n + ilqr::GRAD_CAP_LONG - 1) / ilqr::GRAD_CAP_LONG;
  return launches * ilqr::GRAD_MAX_GRID + (size_t)n + 1;  // and one for the joined total
}

constexpr int64_t MANY_SLOTS = 4096;  // beyond this the blocks of the scaling do not each join them

// The join of partial sums alone (no tensors' norms, so no table of them).
cudaError_t join_all(bool max_type, const double* slots, int64_t n_slots, const ilqr::GradNormOut& o,
                     cudaStream_t stream) {
  return ilqr::launch_grad_join<ilqr::GRAD_CAP_SHORT>(nullptr, 0, nullptr, max_type, slots, n_slots, o, true, stream);
}

template <int CAP>
int norm_impl(const List& l, bool max_type, const ilqr::GradNormOut& o, double* slots, cudaStream_t stream) {
  const std::unique_ptr<GradTable<CAP>> tab(new GradTable<CAP>);
  const bool per = o.tensor_norms != nullptr;
  int64_t used = 0;
  for (int32_t first = 0; first < l.n; first += CAP) {
    const int32_t n = std::min<int32_t>(CAP, l.n - first);
    fill(*tab, l, first, n);
    const int grid = grid_of(tab->chunks);
    cudaError_t e = per ? ilqr::launch_grad_each(*tab, grid, max_type, slots + used, stream)
                        : ilqr::launch_grad_sum(*tab, grid, max_type, 0u, slots + used, stream);
    if (e != cudaSuccess) return ILQR_ERR_CUDA;
    const double* mine = slots + used;
    used += grid + (per ? n - 1 : 0);
    const bool last = first + n == l.n;
    if (per || last) {
      ilqr::GradNormOut part = o;
      if (per) part.tensor_norms = o.tensor_norms + first;
      e = per ? ilqr::launch_grad_join(tab.get(), grid, mine, max_type, slots, used, part, last, stream)
              : join_all(max_type, slots, used, part, stream);
      if (e != cudaSuccess) return ILQR_ERR_CUDA;
    }
  }
  return ILQR_OK;
}

template <int CAP>
int clip_impl(const List& l, const ilqr::GradScale& s, const double* total, float* norm, double* slots,
              cudaStream_t stream) {
  const std::unique_ptr<GradTable<CAP>> tab(new GradTable<CAP>);
  const bool is_long = bytes_of(l) > ilqr::GRAD_LONG_BYTES;
  const uint32_t keep = is_long ? (uint32_t)(ilqr::GRAD_KEEP_BYTES / ilqr::GRAD_CHUNK_BYTES) : 0;
  const bool mx = s.max_type != 0;
  const double* from = total;
  int64_t used = 1;
  if (total == nullptr) {
    used = 0;
    for (int32_t first = 0; first < l.n; first += CAP) {
      fill(*tab, l, first, std::min<int32_t>(CAP, l.n - first));
      const int grid = grid_of(tab->chunks);
      if (ilqr::launch_grad_sum(*tab, grid, mx, keep, slots + used, stream) != cudaSuccess) return ILQR_ERR_CUDA;
      used += grid;
    }
    from = slots;
    if (is_long || used > MANY_SLOTS) {
      const ilqr::GradNormOut o{nullptr, nullptr, slots + used};
      if (join_all(mx, slots, used, o, stream) != cudaSuccess) return ILQR_ERR_CUDA;
      from = slots + used;
      used = 1;
    }
  }
  const bool dependent = total == nullptr;
  for (int32_t first = 0; first < l.n; first += CAP) {
    if (l.n > CAP || total != nullptr) fill(*tab, l, first, std::min<int32_t>(CAP, l.n - first));
    float* out = first == 0 ? norm : nullptr;
    const cudaError_t e =
        is_long ? ilqr::launch_grad_scale_long(*tab, s, from, out, dependent, stream)
                : ilqr::launch_grad_scale(*tab, grid_of(tab->chunks), s, from, used, out, dependent, stream);
    if (e != cudaSuccess) return ILQR_ERR_CUDA;
  }
  return ILQR_OK;
}

int small_impl(const List& l, bool max_type, const ilqr::GradScale* s, const ilqr::GradNormOut& o,
               cudaStream_t stream) {
  GradTable<ilqr::GRAD_CAP_SHORT> tab;
  fill(tab, l, 0, l.n, ilqr::GRAD_SMALL_CHUNK_BYTES);
  return status_of(ilqr::launch_grad_small(tab, max_type, s, o, stream));
}

uint64_t magnitude(int64_t v) { return v < 0 ? 0 - (uint64_t)v : (uint64_t)v; }

}  // namespace

extern "C" {

int ilqr_b200_grad_workspace_size(int32_t n_tensors, size_t* bytes) {
  if (bytes == nullptr || n_tensors < 0) return ILQR_ERR_INVALID_ARGUMENT;
  *bytes = slots_of(n_tensors) * sizeof(double);
  return ILQR_OK;
}

int ilqr_b200_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int32_t n_tensors,
                        int32_t norm_type, float* norm, float* tensor_norms, double* total, void* workspace,
                        size_t workspace_bytes, cudaStream_t stream) {
  const List l{grads, nullptr, numel, dtypes, n_tensors};
  if (const int st = check_list(l, norm_type); st != ILQR_OK) return st;
  if (norm == nullptr && tensor_norms == nullptr && total == nullptr) return ILQR_ERR_INVALID_ARGUMENT;
  if (!aligned(norm, sizeof(float)) || !aligned(tensor_norms, sizeof(float)) || !aligned(total, sizeof(double)))
    return ILQR_ERR_MISALIGNED;
  if (n_tensors == 0) {
    cudaError_t e = cudaSuccess;
    if (norm != nullptr) e = cudaMemsetAsync(norm, 0, sizeof(float), stream);
    if (e == cudaSuccess && total != nullptr) e = cudaMemsetAsync(total, 0, sizeof(double), stream);
    return status_of(e);
  }
  if (workspace == nullptr || workspace_bytes < slots_of(n_tensors) * sizeof(double)) return ILQR_ERR_WORKSPACE;
  if (!aligned(workspace, sizeof(double))) return ILQR_ERR_MISALIGNED;
  try {
    const ilqr::GradNormOut o{norm, tensor_norms, total};
    double* slots = static_cast<double*>(workspace);
    const bool mx = norm_type == ILQR_NORM_MAX;
    if (tensor_norms == nullptr && is_small(l)) return small_impl(l, mx, nullptr, o, stream);
    if (n_tensors <= ilqr::GRAD_CAP_SHORT) return norm_impl<ilqr::GRAD_CAP_SHORT>(l, mx, o, slots, stream);
    if (n_tensors <= ilqr::GRAD_CAP_MIDDLE) return norm_impl<ilqr::GRAD_CAP_MIDDLE>(l, mx, o, slots, stream);
    return norm_impl<ilqr::GRAD_CAP_LONG>(l, mx, o, slots, stream);
  } catch (...) {
    return ILQR_ERR_HOST_MEMORY;
  }
}

int ilqr_b200_grad_clip(const void* const* grads, void* const* out, const int64_t* numel, const int32_t* dtypes,
                        int32_t n_tensors, int32_t norm_type, double max_norm, double eps, const double* total,
                        float* norm, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (n_tensors > 0 && out == nullptr) return ILQR_ERR_INVALID_ARGUMENT;
  const List l{grads, out, numel, dtypes, n_tensors};
  if (const int st = check_list(l, norm_type); st != ILQR_OK) return st;
  if (!(max_norm >= 0.0) || !(eps >= 0.0) || std::isinf(eps)) return ILQR_ERR_INVALID_ARGUMENT;
  if (!aligned(total, sizeof(double)) || !aligned(norm, sizeof(float))) return ILQR_ERR_MISALIGNED;
  if (workspace == nullptr || workspace_bytes < slots_of(n_tensors) * sizeof(double)) return ILQR_ERR_WORKSPACE;
  if (!aligned(workspace, sizeof(double))) return ILQR_ERR_MISALIGNED;
  double* slots = static_cast<double*>(workspace);
  const ilqr::GradScale s{max_norm, eps, norm_type == ILQR_NORM_MAX ? 1 : 0};
  if (n_tensors == 0) {
    if (norm == nullptr) return ILQR_OK;
    if (total == nullptr) return status_of(cudaMemsetAsync(norm, 0, sizeof(float), stream));
    const ilqr::GradNormOut o{norm, nullptr, nullptr};
    return status_of(join_all(s.max_type != 0, total, 1, o, stream));
  }
  try {
    if (overlaps(l, total, norm)) return ILQR_ERR_OVERLAP;
    if (total == nullptr && is_small(l))
      return small_impl(l, s.max_type != 0, &s, ilqr::GradNormOut{norm, nullptr, nullptr}, stream);
    if (n_tensors <= ilqr::GRAD_CAP_SHORT) return clip_impl<ilqr::GRAD_CAP_SHORT>(l, s, total, norm, slots, stream);
    if (n_tensors <= ilqr::GRAD_CAP_MIDDLE) return clip_impl<ilqr::GRAD_CAP_MIDDLE>(l, s, total, norm, slots, stream);
    return clip_impl<ilqr::GRAD_CAP_LONG>(l, s, total, norm, slots, stream);
  } catch (...) {
    return ILQR_ERR_HOST_MEMORY;
  }
}

}  // extern "C"

namespace {

// Where the slices of one tensor lie, in bytes.
struct Rows {
  uintptr_t base;
  int64_t row, seg, len, n_seg, B;
};

// Whether no two of its values share memory: one of the two strides steps over
// all that the other spans.
bool apart(const Rows& r) {
  if (r.row < 0 || r.seg < 0) return false;
  const bool one_row = r.B == 1, one_seg = r.n_seg == 1;
  if (!one_row && r.row < r.len) return false;
  if (!one_seg && r.seg < r.len) return false;
  if (one_row || one_seg) return true;
  return r.row >= (r.n_seg - 1) * r.seg + r.len || r.seg >= (r.B - 1) * r.row + r.len;
}

// Whether two sets of slices share no memory: interleaved ones (columns of one
// packed array, in either layout) are told apart.
bool disjoint(const Rows& a, const Rows& b) {
  const ilqr::Every da[2] = {{a.B, a.row}, {a.n_seg, a.seg}}, db[2] = {{b.B, b.row}, {b.n_seg, b.seg}};
  return !ilqr::Meeting::of({a.base, a.len, da, 2}, {b.base, b.len, db, 2});
}

// i / d = i magic >> (32 + shift) for 0 <= i < 2^31 and d >= 2: with
// 2^shift < d <= 2^(shift + 1) and magic = ceil(2^(32 + shift) / d) < 2^32 the
// error magic d - 2^(32 + shift) is below d, and i times it below 2^(32 + shift).
void reciprocal(uint32_t d, uint32_t* magic, uint32_t* shift) {
  *magic = *shift = 0;
  if (d < 2) return;
  while (((uint64_t)2 << *shift) < d) ++*shift;
  *magic = (uint32_t)((((uint64_t)1 << (32 + *shift)) + d - 1) / d);
}

bool same(const Rows& a, const Rows& b) {
  return a.base == b.base && (a.B == 1 || a.row == b.row) && (a.n_seg == 1 || a.seg == b.seg);
}

}  // namespace

extern "C" {

int ilqr_b200_grad_clip_elements(const void* const* grads, void* const* out, const int32_t* dtypes,
                                 const int64_t* layout, int32_t n_tensors, int64_t B, double max_norm, double eps,
                                 int32_t zero_nonfinite, float* norms, cudaStream_t stream) {
  if (n_tensors < 1 || n_tensors > ILQR_MAX_ELEMENT_TENSORS || B < 0 || B > ILQR_MAX_BATCH)
    return ILQR_ERR_INVALID_ARGUMENT;
  if (grads == nullptr || out == nullptr || dtypes == nullptr || layout == nullptr) return ILQR_ERR_INVALID_ARGUMENT;
  if (!(max_norm >= 0.0) || !(eps >= 0.0) || std::isinf(eps)) return ILQR_ERR_INVALID_ARGUMENT;
  if (!aligned(norms, sizeof(float))) return ILQR_ERR_MISALIGNED;
  if (B == 0) return ILQR_OK;
  constexpr int64_t FAR = (int64_t)1 << 44;  // bytes: no address arithmetic below can wrap
  ilqr::RowTable tab;
  std::memset(&tab, 0, sizeof(tab));
  Rows ins[ILQR_MAX_ELEMENT_TENSORS], outs[ILQR_MAX_ELEMENT_TENSORS];
  int64_t row_bytes = 0;
  tab.one_dtype = 1;
  for (int32_t i = 0; i < n_tensors; ++i) {
    const int64_t* g = layout + 6 * i;
    const int64_t n_seg = g[0], len = g[1];
    if (dtypes[i] < ILQR_DTYPE_F32 || dtypes[i] > ILQR_DTYPE_BF16) return ILQR_ERR_INVALID_ARGUMENT;
    if (n_seg < 0 || len < 0) return ILQR_ERR_INVALID_ARGUMENT;
    if (n_seg == 0 || len == 0) continue;
    const int64_t sz = size_of(dtypes[i]);
    if (n_seg > INT32_MAX || len > INT32_MAX || n_seg * len > INT32_MAX) return ILQR_ERR_INVALID_ARGUMENT;
    for (int k = 2; k < 6; ++k) {
      const int64_t times = (k & 1) ? B : n_seg;  // [2] in_seg, [3] in_row, [4] out_seg, [5] out_row
      if (magnitude(g[k]) > (uint64_t)(FAR / sz / std::max<int64_t>(times, 1)))
        return ILQR_ERR_INVALID_ARGUMENT;
    }
    if (grads[i] == nullptr || out[i] == nullptr) return ILQR_ERR_INVALID_ARGUMENT;
    const uintptr_t p = (uintptr_t)grads[i], q = (uintptr_t)out[i];
    if ((p | q) & (uintptr_t)(sz - 1)) return ILQR_ERR_MISALIGNED;
    const int k = tab.n++;
    ins[k] = Rows{p, g[3] * sz, g[2] * sz, len * sz, n_seg, B};
    outs[k] = Rows{q, g[5] * sz, g[4] * sz, len * sz, n_seg, B};
    if (ins[k].row < 0 || ins[k].seg < 0) return ILQR_ERR_INVALID_ARGUMENT;
    if (!apart(outs[k])) return ILQR_ERR_OVERLAP;
    // the widest vector that divides every address and length
    uintptr_t all = p | q | (uintptr_t)(len * sz) | 16u;
    if (n_seg > 1) all |= (uintptr_t)ins[k].seg | (uintptr_t)outs[k].seg;
    if (B > 1) all |= (uintptr_t)ins[k].row | (uintptr_t)outs[k].row;
    const uint32_t vec = (uint32_t)(all & (~all + 1));
    ilqr::RowTensor& r = tab.t[k];
    r.in = static_cast<const char*>(grads[i]);
    r.out = static_cast<char*>(out[i]);
    r.in_row = ins[k].row, r.in_seg = ins[k].seg;
    r.out_row = outs[k].row, r.out_seg = outs[k].seg;
    r.n_seg = (uint32_t)n_seg, r.seg_vecs = (uint32_t)(len * sz / vec);
    r.vec_bytes = vec, r.dtype = (uint32_t)dtypes[i];
    reciprocal(r.seg_vecs, &r.magic, &r.shift);
    r.staged = (uint32_t)std::min<int64_t>(row_bytes, UINT32_MAX);
    r.seg_bytes = (uint32_t)std::min<int64_t>(len * sz, UINT32_MAX);
    // what every address of the input has in common with the output's
    uintptr_t off = p ^ q;
    if (n_seg > 1) off |= (uintptr_t)(ins[k].seg - outs[k].seg);
    if (B > 1) off |= (uintptr_t)(ins[k].row - outs[k].row);
    int64_t place = len * sz;
    if (len * sz >= ilqr::GRAD_MIN_BULK && (off & 15u) == 0) {
      r.bulk = vec == 16 ? ilqr::ROW_BULK : ilqr::ROW_BULK_ENDS;
      if (vec != 16) place = (place + 30) / 16 * 16;
      tab.bulk = 1;
    }
    r.place = (uint32_t)std::min<int64_t>(place, UINT32_MAX);
    const int64_t words = (n_seg * place + 15) / 16;
    r.staged_vecs = (uint32_t)std::min<int64_t>(words, UINT32_MAX);
    row_bytes += words * 16;
    if (r.dtype != tab.t[0].dtype) tab.one_dtype = 0;
  }
  const Rows all_norms{(uintptr_t)norms, 0, 0, norms != nullptr ? B * (int64_t)sizeof(float) : 0, 1, 1};
  for (int a = 0; a < tab.n; ++a) {
    if (!disjoint(outs[a], all_norms) || !disjoint(ins[a], all_norms)) return ILQR_ERR_OVERLAP;
    for (int b = 0; b < tab.n; ++b) {
      if (a != b && (!disjoint(outs[a], outs[b]) || !disjoint(outs[a], ins[b]))) return ILQR_ERR_OVERLAP;
      if (a == b && !same(ins[a], outs[a]) && !disjoint(outs[a], ins[a])) return ILQR_ERR_OVERLAP;
    }
  }
  // in place is told by the address alone in the kernel
  tab.B = B;
  tab.max_norm = max_norm;
  tab.eps = eps;
  tab.zero_nonfinite = zero_nonfinite != 0 ? 1 : 0;
  tab.norms = norms;
  tab.staged_bytes = (uint32_t)std::min<int64_t>(row_bytes, UINT32_MAX);
  return status_of(ilqr::launch_grad_rows(tab, stream));
}

}  // extern "C"
