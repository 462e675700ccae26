// ilqr_gradclip.cu -- norms of gradients and clipping by them.
//
// Over a list of tensors: n = sqrt(sum g^2) (or max |g|), c = min(1, m / (n + eps)),
// out = c g. Per batch element: the same over each element's slices of up to
// eight tensors.
//
// Sums: up to 32 values are squared and added in 32 bits, in four or eight
// chains that are joined in pairs, and those sums in 64 bits. No value passes
// through more than eight roundings of relative size 2^-24 on the way: they move
// a sum of squares by 2^-21 at most, its root by 2^-22, whatever the length. (A
// conversion and an addition in 64 bits for every four values instead cost as
// much as everything else: the per-element kernel was bound by instructions.)
// Squares that leave the range of a float (|g| above 2^63, or so small that the
// group's sum is under 2^-100) are formed again in 64 bits, so a norm is right
// wherever it is a float itself. The order of every sum is fixed by sizes and
// grid: no atomics, the same bits each time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ilqr_b200.h"
#include "ilqr_gradclip.h"

namespace ilqr {

namespace {

constexpr int NT = 256;  // threads of a block
constexpr int UN = 4;    // 16-byte loads that a thread has in flight

// ---- values ----------------------------------------------------------------

template <int DT> struct Type;
template <> struct Type<ILQR_DTYPE_F32> {
  static constexpr int SIZE = 4;
  static constexpr bool WIDE = true;  // squares can leave the range of a float
};
template <> struct Type<ILQR_DTYPE_F16> {
  static constexpr int SIZE = 2;
  static constexpr bool WIDE = false;
};
template <> struct Type<ILQR_DTYPE_BF16> {
  static constexpr int SIZE = 2;
  static constexpr bool WIDE = true;
};

// the values of one 32-bit word
template <int DT>
__device__ __forceinline__ void unpack(uint32_t w, float* x) {
  if constexpr (DT == ILQR_DTYPE_F32) {
    x[0] = __uint_as_float(w);
  } else if constexpr (DT == ILQR_DTYPE_BF16) {
    x[0] = __uint_as_float(w << 16);
    x[1] = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x[0] = f.x;
    x[1] = f.y;
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack(const float* x) {
  if constexpr (DT == ILQR_DTYPE_F32) {
    return __float_as_uint(x[0]);
  } else if constexpr (DT == ILQR_DTYPE_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[0], x[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(x[0], x[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <int DT>
__device__ __forceinline__ float load_one(const char* p) {
  if constexpr (DT == ILQR_DTYPE_F32) return *reinterpret_cast<const float*>(p);
  if constexpr (DT == ILQR_DTYPE_BF16) return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
  return __half2float(*reinterpret_cast<const __half*>(p));
}

template <int DT>
__device__ __forceinline__ void store_one(char* p, float x) {
  if constexpr (DT == ILQR_DTYPE_F32) *reinterpret_cast<float*>(p) = x;
  else if constexpr (DT == ILQR_DTYPE_BF16) *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(x);
  else *reinterpret_cast<__half*>(p) = __float2half_rn(x);
}

// ---- sums ------------------------------------------------------------------

// MAX: the largest magnitude, kept as its bits: those order magnitudes as
// integers, with NaN above infinity, so a NaN stays the largest.
template <bool MAX> struct Acc {
  double s = 0.0;
};
template <> struct Acc<true> {
  uint32_t m = 0u;
};

// whether a value is not zero
template <int N>
__device__ __forceinline__ bool any_of(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m |= __float_as_uint(x[i]) << 1;
  return m != 0;
}

// N values (a power of two, 32 at most)
template <int DT, int N>
__device__ __forceinline__ void add(Acc<false>& a, const float* x) {
  constexpr int NC = N >= 32 ? 8 : N >= 4 ? 4 : N;
  float c[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) c[i] = __fmul_rn(x[i], x[i]);
#pragma unroll
  for (int i = NC; i < N; ++i) c[i % NC] = __fmaf_rn(x[i], x[i], c[i % NC]);
#pragma unroll
  for (int o = NC / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) c[i] = __fadd_rn(c[i], c[i + o]);
  const float s = c[0];
  if (!Type<DT>::WIDE || (s >= 0x1p-100f && s < __int_as_float(0x7f800000))) {
    a.s += (double)s;
  } else if (s != 0.0f || any_of<N>(x)) {
#pragma unroll
    for (int i = 0; i < N; ++i) a.s = __fma_rn((double)x[i], (double)x[i], a.s);
  }
}

template <int DT, int N>
__device__ __forceinline__ void add(Acc<true>& a, const float* x) {
#pragma unroll
  for (int i = 0; i < N; ++i) a.m = max(a.m, __float_as_uint(x[i]) & 0x7fffffffu);
}

__device__ __forceinline__ double value(const Acc<false>& a) { return a.s; }
__device__ __forceinline__ double value(const Acc<true>& a) { return (double)__uint_as_float(a.m); }

template <bool MAX>
__device__ __forceinline__ double join(double a, double b) {
  if constexpr (!MAX) return a + b;
  return a != a ? a : (b != b || b > a ? b : a);
}

template <bool MAX>
__device__ __forceinline__ double warp_join(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join<MAX>(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The join over a block, for every thread; sh has a place for each warp.
template <bool MAX>
__device__ __forceinline__ double block_join(double v, double* sh) {
  v = warp_join<MAX>(v);
  __syncthreads();  // sh may still be read from the join before
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < (blockDim.x >> 5) ? sh[threadIdx.x & 31] : 0.0;
  return warp_join<MAX>(v);
}

__device__ __forceinline__ double norm_of(double total, bool max_type) { return max_type ? total : sqrt(total); }

// WIDE: the coefficient is so small that as a float it has lost bits; the
// product is formed in 64 bits.
struct Coef {
  float f;
  double d;
  bool wide;
};

__device__ __forceinline__ Coef coef_of(double norm, double max_norm, double eps) {
  Coef c;
  c.d = max_norm / (norm + eps);
  if (c.d >= 1.0 || isinf(max_norm)) c.d = 1.0;  // NaN stays
  c.f = (float)c.d;
  c.wide = c.d < 0x1p-100;
  return c;
}

template <bool WIDE>
__device__ __forceinline__ float scaled(float x, const Coef& c) {
  if constexpr (WIDE) return (float)((double)x * c.d);
  return x * c.f;
}

// ---- vectors ---------------------------------------------------------------

template <int VB> struct Vec;
template <> struct Vec<16> { uint4 w; };
template <> struct Vec<8> { uint2 w; };
template <> struct Vec<4> { uint32_t w; };
template <> struct Vec<2> { uint16_t w; };

template <int VB>
__device__ __forceinline__ Vec<VB> load_vec(const char* p) {
  return *reinterpret_cast<const Vec<VB>*>(p);
}

template <int DT, int VB>
__device__ __forceinline__ void unpack_vec(const Vec<VB>& v, float* x) {
  if constexpr (VB == 2) {
    float two[2];
    unpack<DT>((uint32_t)v.w, two);
    x[0] = two[0];
  } else {
    constexpr int K = 4 / Type<DT>::SIZE;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int k = 0; k < VB / 4; ++k) unpack<DT>(w[k], x + k * K);
  }
}

template <int DT, int VB>
__device__ __forceinline__ Vec<VB> pack_vec(const float* x) {
  Vec<VB> v;
  if constexpr (VB == 2) {
    const float two[2] = {x[0], 0.0f};
    v.w = (uint16_t)pack<DT>(two);
  } else {
    constexpr int K = 4 / Type<DT>::SIZE;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int k = 0; k < VB / 4; ++k) w[k] = pack<DT>(x + k * K);
  }
  return v;
}

// U vectors into a sum
template <int DT, int VB, int U, bool MAX>
__device__ __forceinline__ void add_vecs(Acc<MAX>& a, const Vec<VB>* v) {
  constexpr int NV = VB / Type<DT>::SIZE;
  float x[U * NV];
#pragma unroll
  for (int u = 0; u < U; ++u) unpack_vec<DT, VB>(v[u], x + u * NV);
  add<DT, U * NV>(a, x);
}

template <int DT, int VB, bool WIDE>
__device__ __forceinline__ Vec<VB> scale_vec(const Vec<VB>& v, const Coef& c) {
  constexpr int NV = VB / Type<DT>::SIZE;
  float x[NV];
  unpack_vec<DT, VB>(v, x);
#pragma unroll
  for (int j = 0; j < NV; ++j) x[j] = scaled<WIDE>(x[j], c);
  return pack_vec<DT, VB>(x);
}

// ---- a range of a dense tensor ---------------------------------------------

template <int DT>
__device__ __forceinline__ int head_of(const char* p, int64_t n) {
  const int h = (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / Type<DT>::SIZE;
  return n < h ? (int)n : h;
}

template <int DT, bool MAX>
__device__ __forceinline__ void range_sum(Acc<MAX>& a, const char* p, int64_t n) {
  constexpr int SZ = Type<DT>::SIZE, VE = 16 / SZ;
  const int tid = threadIdx.x;
  const int h = head_of<DT>(p, n);
  const int tail = (int)((n - h) % VE);
  if (tid < h + tail) {
    const float x = load_one<DT>(p + (tid < h ? tid : n - tail + (tid - h)) * SZ);
    add<DT, 1>(a, &x);
  }
  p += h * SZ + tid * 16;
  int64_t left = (n - h) / VE - tid;  // vectors from this thread's first on
  for (; left > (UN - 1) * NT; left -= UN * NT, p += UN * NT * 16) {
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) v[u] = load_vec<16>(p + u * NT * 16);
    add_vecs<DT, 16, UN, MAX>(a, v);
  }
  if (left > 0) {
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      v[u].w = make_uint4(0, 0, 0, 0);
      if (left > u * NT) v[u] = load_vec<16>(p + u * NT * 16);
    }
    add_vecs<DT, 16, UN, MAX>(a, v);
  }
}

// out = c in; `in` may be `out`
template <int DT>
__device__ __forceinline__ void range_scale(const char* p, char* q, int64_t n, const Coef& c) {
  constexpr int SZ = Type<DT>::SIZE, VE = 16 / SZ;
  const int tid = threadIdx.x;
  const int h = head_of<DT>(p, n);
  const int tail = (int)((n - h) % VE);
  if (tid < h + tail) {
    const int64_t at = (tid < h ? tid : n - tail + (tid - h)) * SZ;
    store_one<DT>(q + at, scaled<false>(load_one<DT>(p + at), c));
  }
  // from the end: what the sums read last is still in L2
  const int64_t nv = (n - h) / VE, full = nv / (UN * NT) * (UN * NT);
  int64_t left = nv - full - tid;
  p += h * SZ + (full + tid) * 16;
  q += h * SZ + (full + tid) * 16;
  if (left > 0) {
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (left > u * NT) v[u] = load_vec<16>(p + u * NT * 16);
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (left > u * NT) *reinterpret_cast<Vec<16>*>(q + u * NT * 16) = scale_vec<DT, 16, false>(v[u], c);
  }
  for (left = full; left > 0; left -= UN * NT) {
    p -= UN * NT * 16;
    q -= UN * NT * 16;
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) v[u] = load_vec<16>(p + u * NT * 16);
#pragma unroll
    for (int u = 0; u < UN; ++u) *reinterpret_cast<Vec<16>*>(q + u * NT * 16) = scale_vec<DT, 16, false>(v[u], c);
  }
}

// ---- lists -----------------------------------------------------------------

// The tensor that chunk k belongs to.
template <int CAP>
__device__ __forceinline__ int find(const GradTable<CAP>& tab, uint32_t k) {
  int lo = 0, hi = tab.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.e[mid].chunk0 <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t first_chunk(uint32_t block, uint32_t chunks, uint32_t grid) {
  return (uint32_t)((uint64_t)block * chunks / grid);
}

// the block whose chunks [first_chunk(b), first_chunk(b + 1)) hold chunk k
__device__ __forceinline__ uint32_t block_of(uint32_t k, uint32_t chunks, uint32_t grid) {
  return (uint32_t)((((uint64_t)k + 1) * grid - 1) / chunks);
}

template <int CAP>
__device__ __forceinline__ void span(const GradTable<CAP>& tab, int t, uint32_t k0, uint32_t k1, int64_t* at,
                                     int64_t* n) {
  const GradEntry& e = tab.e[t];
  const int64_t per = tab.chunk_bytes / (e.dtype == ILQR_DTYPE_F32 ? 4 : 2);
  const int64_t a = (int64_t)(k0 - e.chunk0) * per, b = (int64_t)(k1 - e.chunk0) * per;
  *at = a;
  *n = (b < e.numel ? b : e.numel) - a;
}

template <bool MAX>
__device__ __forceinline__ void entry_sum(Acc<MAX>& a, uint32_t dtype, const void* in, int64_t at, int64_t n) {
  const char* p = static_cast<const char*>(in);
  if (dtype == ILQR_DTYPE_F32) range_sum<ILQR_DTYPE_F32, MAX>(a, p + at * 4, n);
  else if (dtype == ILQR_DTYPE_BF16) range_sum<ILQR_DTYPE_BF16, MAX>(a, p + at * 2, n);
  else range_sum<ILQR_DTYPE_F16, MAX>(a, p + at * 2, n);
}

// Value by value: for coefficients below the floats' range, and for `in` and
// `out` that lie differently in their 16-byte words.
__device__ __forceinline__ void entry_scale_apart(uint32_t dtype, const char* p, char* q, int64_t n, const Coef& c) {
  const int sz = dtype == ILQR_DTYPE_F32 ? 4 : 2;
#pragma unroll 1
  for (int64_t i = threadIdx.x; i < n; i += NT) {
    const char* from = p + i * sz;
    float x = dtype == ILQR_DTYPE_F32    ? load_one<ILQR_DTYPE_F32>(from)
              : dtype == ILQR_DTYPE_BF16 ? load_one<ILQR_DTYPE_BF16>(from)
                                         : load_one<ILQR_DTYPE_F16>(from);
    x = c.wide ? scaled<true>(x, c) : scaled<false>(x, c);
    char* to = q + i * sz;
    if (dtype == ILQR_DTYPE_F32) store_one<ILQR_DTYPE_F32>(to, x);
    else if (dtype == ILQR_DTYPE_BF16) store_one<ILQR_DTYPE_BF16>(to, x);
    else store_one<ILQR_DTYPE_F16>(to, x);
  }
}

__device__ __forceinline__ void entry_scale(uint32_t dtype, const void* in, void* out, int64_t at, int64_t n,
                                            const Coef& c) {
  const int sz = dtype == ILQR_DTYPE_F32 ? 4 : 2;
  const char* p = static_cast<const char*>(in) + at * sz;
  char* q = static_cast<char*>(out) + at * sz;
  if (c.wide || ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15u))
    entry_scale_apart(dtype, p, q, n, c);
  else if (dtype == ILQR_DTYPE_F32) range_scale<ILQR_DTYPE_F32>(p, q, n, c);
  else if (dtype == ILQR_DTYPE_BF16) range_scale<ILQR_DTYPE_BF16>(p, q, n, c);
  else range_scale<ILQR_DTYPE_F16>(p, q, n, c);
}

// Partial sums. Each block takes a contiguous run of chunks; with PER one sum
// for each tensor in it, at slot block + tensor: slots of neighbours are
// neighbours, and where a block ends with its tensor the one slot that falls
// out is set to 0, the identity of both joins.
template <int CAP, bool MAX, bool PER>
__global__ void __launch_bounds__(NT) grad_sum_kernel(const __grid_constant__ GradTable<CAP> tab, double* slots) {
  __shared__ double sh[32];
  asm volatile("griddepcontrol.launch_dependents;");
  uint32_t k = first_chunk(blockIdx.x, tab.chunks, gridDim.x);
  const uint32_t k1 = first_chunk(blockIdx.x + 1, tab.chunks, gridDim.x);
  int t = find(tab, k);
  if (PER && blockIdx.x > 0 && k == tab.e[t].chunk0 && threadIdx.x == 0) slots[blockIdx.x + t - 1] = 0.0;
  Acc<MAX> a;
  for (; k < k1; ++t) {
    const uint32_t end = t + 1 < tab.n ? min(k1, tab.e[t + 1].chunk0) : k1;
    int64_t at, n;
    span(tab, t, k, end, &at, &n);
    entry_sum<MAX>(a, tab.e[t].dtype, tab.e[t].in, at, n);
    if (PER) {
      const double v = block_join<MAX>(value(a), sh);
      if (threadIdx.x == 0) slots[blockIdx.x + t] = v;
      a = Acc<MAX>();
    }
    k = end;
  }
  if (!PER) {
    const double v = block_join<MAX>(value(a), sh);
    if (threadIdx.x == 0) slots[blockIdx.x] = v;
  }
}

template <bool MAX>
__device__ __forceinline__ double join_slots(const double* slots, int64_t n, double* sh) {
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) v = join<MAX>(v, slots[i]);
  return block_join<MAX>(v, sh);
}

// Block 0: the norm of the whole list. The others: a warp for each tensor.
template <int CAP, bool MAX>
__global__ void __launch_bounds__(NT) grad_join_kernel(const __grid_constant__ GradTable<CAP> tab, uint32_t grid,
                                                       const double* tab_slots, const double* slots, int64_t n_slots,
                                                       GradNormOut out, int want_global) {
  __shared__ double sh[32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == 0) {
    if (!want_global) return;
    const double v = join_slots<MAX>(slots, n_slots, sh);
    if (threadIdx.x == 0) {
      if (out.norm != nullptr) *out.norm = (float)norm_of(v, MAX);
      if (out.total != nullptr) *out.total = v;
    }
    return;
  }
  const int t = (int)(blockIdx.x - 1) * (NT / 32) + (int)(threadIdx.x >> 5);
  if (t >= tab.n) return;
  const uint32_t c0 = tab.e[t].chunk0, c1 = t + 1 < tab.n ? tab.e[t + 1].chunk0 : tab.chunks;
  const uint32_t lo = block_of(c0, tab.chunks, grid) + t, hi = block_of(c1 - 1, tab.chunks, grid) + t;
  double v = 0.0;
  for (uint32_t i = lo + (threadIdx.x & 31); i <= hi; i += 32) v = join<MAX>(v, tab_slots[i]);
  v = warp_join<MAX>(v);
  if ((threadIdx.x & 31) == 0) out.tensor_norms[t] = (float)norm_of(v, MAX);
}

// out = c in over the list; every block joins the partial sums for itself, in
// the same order. In place a coefficient of 1 leaves the values where they are.
template <int CAP>
__global__ void __launch_bounds__(NT, 4) grad_scale_kernel(const __grid_constant__ GradTable<CAP> tab, GradScale s,
                                                        const double* slots, int64_t n_slots, float* norm) {
  __shared__ double sh[32];
  const uint32_t k0 = first_chunk(blockIdx.x, tab.chunks, gridDim.x);
  uint32_t k1 = first_chunk(blockIdx.x + 1, tab.chunks, gridDim.x);
  int t = find(tab, k1 - 1);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double total = s.max_type ? join_slots<true>(slots, n_slots, sh) : join_slots<false>(slots, n_slots, sh);
  const double nrm = norm_of(total, s.max_type);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nrm;
  const Coef c = coef_of(nrm, s.max_norm, s.eps);
  for (; k1 > k0; --t) {
    const GradEntry& e = tab.e[t];
    const uint32_t begin = max(k0, e.chunk0);
    if (!(c.d == 1.0 && e.in == e.out)) {
      int64_t at, n;
      span(tab, t, begin, k1, &at, &n);
      entry_scale(e.dtype, e.in, e.out, at, n, c);
    }
    k1 = begin;
  }
}

// ---- batch elements ---------------------------------------------------------

// Vector i of a slice lies in segment i / seg_vecs: by a multiplication with
// the reciprocal rounded up to 2^(31 + shift), exact for i < 2^31.
__device__ __forceinline__ int64_t vec_at(const RowTensor& r, uint32_t i, uint32_t vb, int64_t seg_stride) {
  if (r.n_seg == 1) return (int64_t)i * vb;
  const uint32_t s = r.seg_vecs == 1 ? i : __umulhi(i, r.magic) >> r.shift;
  return s * seg_stride + (int64_t)(i - s * r.seg_vecs) * vb;
}

template <int VB>
__device__ __forceinline__ void copy_async(uint32_t to, const char* from) {
  if constexpr (VB == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  } else if constexpr (VB == 2) {
    const uint16_t w = *reinterpret_cast<const uint16_t*>(from);
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(w) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(VB) : "memory");
  }
}

// The three steps of a slice. Each thread copies, adds and scales the same
// vectors: no thread reads what another copied, so the copies need no barrier.
template <int VB>
__device__ __forceinline__ void row_copy(const RowTensor& r, int64_t b, uint32_t to, uint32_t lane, uint32_t step) {
  const char* p = r.in + b * r.in_row;
  const uint32_t n = r.n_seg * r.seg_vecs;
#pragma unroll 4
  for (uint32_t i = lane; i < n; i += step) copy_async<VB>(to + i * VB, p + vec_at(r, i, VB, r.in_seg));
}

template <int DT, int VB, bool STAGED>
__device__ __forceinline__ void row_sum(Acc<false>& a, const RowTensor& r, int64_t b, const char* staged, uint32_t lane,
                                        uint32_t step) {
  const char* p = r.in + b * r.in_row;
  const uint32_t n = r.n_seg * r.seg_vecs;
  for (uint32_t i = lane; i < n; i += UN * step) {
    Vec<VB> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const uint32_t k = i + u * step;
      v[u] = Vec<VB>{};
      if (k < n) v[u] = load_vec<VB>(STAGED ? staged + k * VB : p + vec_at(r, k, VB, r.in_seg));
    }
    add_vecs<DT, VB, UN, false>(a, v);
  }
}

template <int DT, int VB, bool STAGED>
__device__ __forceinline__ void row_scale(const RowTensor& r, int64_t b, const char* staged, const Coef& c,
                                          uint32_t lane, uint32_t step) {
  const char* p = r.in + b * r.in_row;
  char* q = r.out + b * r.out_row;
  const uint32_t n = r.n_seg * r.seg_vecs;
#pragma unroll 4
  for (uint32_t i = lane; i < n; i += step) {
    const Vec<VB> v = load_vec<VB>(STAGED ? staged + i * VB : p + vec_at(r, i, VB, r.in_seg));
    *reinterpret_cast<Vec<VB>*>(q + vec_at(r, i, VB, r.out_seg)) = scale_vec<DT, VB, false>(v, c);
  }
}

// Value by value: zeros in the place of a slice, or coefficients below the
// floats' range.
__device__ __noinline__ void row_apart(const RowTensor& r, int64_t b, const Coef& c, bool zero, uint32_t lane,
                                       uint32_t step) {
  const uint32_t sz = r.dtype == ILQR_DTYPE_F32 ? 4 : 2, per = r.vec_bytes / sz;
  const char* p = r.in + b * r.in_row;
  char* q = r.out + b * r.out_row;
  const uint32_t n = r.n_seg * r.seg_vecs;
#pragma unroll 1
  for (uint32_t i = lane; i < n; i += step) {
    const char* from = p + vec_at(r, i, r.vec_bytes, r.in_seg);
    char* to = q + vec_at(r, i, r.vec_bytes, r.out_seg);
#pragma unroll 1
    for (uint32_t k = 0; k < per; ++k, from += sz, to += sz) {
      if (r.dtype == ILQR_DTYPE_F32)
        store_one<ILQR_DTYPE_F32>(to, zero ? 0.0f : scaled<true>(load_one<ILQR_DTYPE_F32>(from), c));
      else if (r.dtype == ILQR_DTYPE_BF16)
        store_one<ILQR_DTYPE_BF16>(to, zero ? 0.0f : scaled<true>(load_one<ILQR_DTYPE_BF16>(from), c));
      else
        store_one<ILQR_DTYPE_F16>(to, zero ? 0.0f : scaled<true>(load_one<ILQR_DTYPE_F16>(from), c));
    }
  }
}

#define ROW_DISPATCH(r, CALL)                                                       \
  switch ((r).dtype * 32 + (r).vec_bytes) {                                         \
    case ILQR_DTYPE_F32 * 32 + 16: CALL(ILQR_DTYPE_F32, 16); break;                 \
    case ILQR_DTYPE_F32 * 32 + 8: CALL(ILQR_DTYPE_F32, 8); break;                   \
    case ILQR_DTYPE_F32 * 32 + 4: CALL(ILQR_DTYPE_F32, 4); break;                   \
    case ILQR_DTYPE_F16 * 32 + 16: CALL(ILQR_DTYPE_F16, 16); break;                 \
    case ILQR_DTYPE_F16 * 32 + 8: CALL(ILQR_DTYPE_F16, 8); break;                   \
    case ILQR_DTYPE_F16 * 32 + 4: CALL(ILQR_DTYPE_F16, 4); break;                   \
    case ILQR_DTYPE_F16 * 32 + 2: CALL(ILQR_DTYPE_F16, 2); break;                   \
    case ILQR_DTYPE_BF16 * 32 + 16: CALL(ILQR_DTYPE_BF16, 16); break;               \
    case ILQR_DTYPE_BF16 * 32 + 8: CALL(ILQR_DTYPE_BF16, 8); break;                 \
    case ILQR_DTYPE_BF16 * 32 + 4: CALL(ILQR_DTYPE_BF16, 4); break;                 \
    default: CALL(ILQR_DTYPE_BF16, 2); break;                                       \
  }

// G threads (a warp or the block) for each element. STAGED: its slices are
// copied to shared memory, read from there twice and written once, so global
// memory is read once; without, both passes read global memory.
template <int G, int THREADS, bool STAGED>
__global__ void __launch_bounds__(THREADS) grad_rows_kernel(const __grid_constant__ RowTable tab) {
  extern __shared__ __align__(16) char staged[];
  __shared__ double sh[32];
  constexpr int PER = THREADS / G;
  const int64_t b = PER == 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * PER + threadIdx.x / G;
  if (b >= tab.B) return;  // of a whole warp, or not at all
  const uint32_t lane = threadIdx.x % G;
  const char* mine = staged + (PER == 1 ? 0 : (threadIdx.x / G) * tab.staged_bytes);
  if (STAGED) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(mine);
    for (int k = 0; k < tab.n; ++k) {
      const RowTensor& r = tab.t[k];
      if (r.vec_bytes == 16) row_copy<16>(r, b, to + r.staged, lane, G);
      else if (r.vec_bytes == 8) row_copy<8>(r, b, to + r.staged, lane, G);
      else if (r.vec_bytes == 4) row_copy<4>(r, b, to + r.staged, lane, G);
      else row_copy<2>(r, b, to + r.staged, lane, G);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  Acc<false> a;
  for (int k = 0; k < tab.n; ++k) {
    const RowTensor& r = tab.t[k];
#define CALL(DT, VB) row_sum<DT, VB, STAGED>(a, r, b, mine + r.staged, lane, G)
    ROW_DISPATCH(r, CALL)
#undef CALL
  }
  const double nrm = sqrt(G == 32 ? warp_join<false>(a.s) : block_join<false>(a.s, sh));
  if (lane == 0 && tab.norms != nullptr) tab.norms[b] = (float)nrm;
  const Coef c = coef_of(nrm, tab.max_norm, tab.eps);
  const bool zero = tab.zero_nonfinite && !isfinite(nrm);
  for (int k = 0; k < tab.n; ++k) {
    const RowTensor& r = tab.t[k];
    if (c.d == 1.0 && !zero && r.in == r.out) continue;
    if (zero || c.wide) {
      row_apart(r, b, c, zero, lane, G);
      continue;
    }
#define CALL(DT, VB) row_scale<DT, VB, STAGED>(r, b, mine + r.staged, c, lane, G)
    ROW_DISPATCH(r, CALL)
#undef CALL
  }
}

// ---- launches ---------------------------------------------------------------

template <typename... K, typename... A>
cudaError_t launch(void (*kernel)(K...), unsigned grid, bool dependent, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(NT);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<A&&>(args)...);
}

}  // namespace

template <int CAP>
cudaError_t launch_grad_sum(const GradTable<CAP>& tab, int grid, bool max_type, bool per_tensor, double* slots,
                            cudaStream_t stream) {
  if (max_type)
    return per_tensor ? launch(grad_sum_kernel<CAP, true, true>, grid, false, stream, tab, slots)
                      : launch(grad_sum_kernel<CAP, true, false>, grid, false, stream, tab, slots);
  return per_tensor ? launch(grad_sum_kernel<CAP, false, true>, grid, false, stream, tab, slots)
                    : launch(grad_sum_kernel<CAP, false, false>, grid, false, stream, tab, slots);
}

template <int CAP>
cudaError_t launch_grad_join(const GradTable<CAP>* tab, int grid, const double* tab_slots, bool max_type,
                             const double* slots, int64_t n_slots, const GradNormOut& out, bool want_global,
                             cudaStream_t stream) {
  static const GradTable<CAP> none{};
  const unsigned blocks = 1 + (tab != nullptr ? (unsigned)(tab->n + NT / 32 - 1) / (NT / 32) : 0);
  const GradTable<CAP>& use = tab != nullptr ? *tab : none;
  return max_type ? launch(grad_join_kernel<CAP, true>, blocks, true, stream, use, (uint32_t)grid, tab_slots, slots,
                           n_slots, out, want_global ? 1 : 0)
                  : launch(grad_join_kernel<CAP, false>, blocks, true, stream, use, (uint32_t)grid, tab_slots, slots,
                           n_slots, out, want_global ? 1 : 0);
}

template <int CAP>
cudaError_t launch_grad_scale(const GradTable<CAP>& tab, int grid, const GradScale& s, const double* slots,
                              int64_t n_slots, float* norm, bool dependent, cudaStream_t stream) {
  return launch(grad_scale_kernel<CAP>, grid, dependent, stream, tab, s, slots, n_slots, norm);
}

#define INSTANTIATE(CAP)                                                                                              \
  template cudaError_t launch_grad_sum<CAP>(const GradTable<CAP>&, int, bool, bool, double*, cudaStream_t);           \
  template cudaError_t launch_grad_join<CAP>(const GradTable<CAP>*, int, const double*, bool, const double*, int64_t, \
                                             const GradNormOut&, bool, cudaStream_t);                                 \
  template cudaError_t launch_grad_scale<CAP>(const GradTable<CAP>&, int, const GradScale&, const double*, int64_t,   \
                                              float*, bool, cudaStream_t);
INSTANTIATE(GRAD_CAP_SHORT)
INSTANTIATE(GRAD_CAP_LONG)
#undef INSTANTIATE

namespace {

template <int G, int THREADS, bool STAGED>
cudaError_t launch_rows(const RowTable& tab, cudaStream_t stream) {
  constexpr int PER = THREADS / G;
  const size_t smem = STAGED ? (size_t)tab.staged_bytes * PER : 0;
  const auto kernel = grad_rows_kernel<G, THREADS, STAGED>;
  if (STAGED) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((tab.B + PER - 1) / PER));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, kernel, tab);
}

}  // namespace

cudaError_t launch_grad_rows(const RowTable& tab, cudaStream_t stream) {
  if (tab.staged_bytes <= 4096) return launch_rows<32, 128, true>(tab, stream);
  if (tab.staged_bytes <= 20480) return launch_rows<128, 128, true>(tab, stream);
  if (tab.staged_bytes <= 220000) return launch_rows<256, 256, true>(tab, stream);
  return launch_rows<256, 256, false>(tab, stream);
}

}  // namespace ilqr
