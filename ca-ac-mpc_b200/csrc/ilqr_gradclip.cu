// ilqr_gradclip.cu -- norms of gradients and clipping by them.
//
// Over a list of tensors: n = sqrt(sum g^2) (or max |g|), c = min(1, m / (n + eps)),
// out = c g. Per batch element: the same over each element's slices of up to
// eight tensors.
//
// Sums: up to 32 values are squared and added in 32 bits, in four or eight
// chains that are joined in pairs, and those sums in 64 bits. No value passes
// through more than eight roundings of relative size 2^-24 on the way: they move
// a sum of squares by 2^-21 at most, its root by 2^-22, whatever the length.
// (Joined in 64 bits after every four values instead, the per-element kernel was
// bound by instructions: 1079 us for the 5.5 GB of B = 65536, T = 50 against 939.)
// Squares that leave the range of a float (|g| above 2^63, or so small that the
// group's sum is under 2^-100) are formed again in 64 bits, so a norm is right
// wherever it is a float itself. The order of every sum is fixed by sizes,
// alignment and grid: no atomics, the same bits each time.
//
// Measured on one B200 (times of a captured call, inputs alternating between
// three sets; the copy rate is 6551 GB/s): see each kernel.
#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ilqr_b200.h"
#include "ilqr_device.cuh"
#include "ilqr_gradclip.h"

namespace ilqr {

namespace {

constexpr int BLK = 256;        // threads of a block
constexpr int LONG_BLK = 1024;  // and of one that shares an element beyond shared memory
constexpr int UN = 4;     // 16-byte loads that a thread has in flight

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

// ---- clusters ---------------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The join of one value of each block of a cluster, in the order of their
// ranks. Ends with an arrival that the caller has to wait for before it returns.
template <bool MAX>
__device__ __forceinline__ double cluster_join(double v, double* mine) {
  if (threadIdx.x == 0) *mine = v;
  cluster_arrive();
  cluster_wait();
  double all = 0.0;
  for (uint32_t k = 0, n = cluster_size(); k < n; ++k) {
    uint32_t at;
    double x;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(mine)), "r"(k));
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(at) : "memory");
    all = join<MAX>(all, x);
  }
  cluster_arrive();
  return all;
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

// What L2 does with a line: a long list's two passes read it from L2 where they
// can, and what will not be read again leaves it first.
enum class Keep { USUAL, POLICY };

__device__ __forceinline__ uint64_t policy_first_out() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}

__device__ __forceinline__ uint64_t policy_usual() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}

template <Keep K>
__device__ __forceinline__ Vec<16> load_16(const char* p, uint64_t policy) {
  if constexpr (K == Keep::USUAL) {
    return load_vec<16>(p);
  } else {
    Vec<16> v;
    asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(v.w.x), "=r"(v.w.y), "=r"(v.w.z), "=r"(v.w.w)
                 : "l"(p), "l"(policy)
                 : "memory");
    return v;
  }
}

template <Keep K>
__device__ __forceinline__ void store_16(char* p, const Vec<16>& v, uint64_t policy) {
  if constexpr (K == Keep::USUAL)
    *reinterpret_cast<Vec<16>*>(p) = v;
  else
    asm volatile("st.global.L2::cache_hint.v4.u32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(p), "r"(v.w.x), "r"(v.w.y),
                 "r"(v.w.z), "r"(v.w.w), "l"(policy)
                 : "memory");
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

template <int DT, bool MAX, Keep K>
__device__ __forceinline__ void range_sum(Acc<MAX>& a, const char* p, int64_t n, uint64_t policy) {
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
  for (; left > (UN - 1) * BLK; left -= UN * BLK, p += UN * BLK * 16) {
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) v[u] = load_16<K>(p + u * BLK * 16, policy);
    add_vecs<DT, 16, UN, MAX>(a, v);
  }
  if (left > 0) {
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      v[u].w = make_uint4(0, 0, 0, 0);
      if (left > u * BLK) v[u] = load_16<K>(p + u * BLK * 16, policy);
    }
    add_vecs<DT, 16, UN, MAX>(a, v);
  }
}

// out = c in; `in` may be `out`
template <int DT, Keep K, int UN>
__device__ __forceinline__ void range_scale(const char* p, char* q, int64_t n, const Coef& c, uint64_t policy) {
  constexpr int SZ = Type<DT>::SIZE, VE = 16 / SZ;
  const int tid = threadIdx.x;
  const int h = head_of<DT>(p, n);
  const int tail = (int)((n - h) % VE);
  if (tid < h + tail) {
    const int64_t at = (tid < h ? tid : n - tail + (tid - h)) * SZ;
    store_one<DT>(q + at, scaled<false>(load_one<DT>(p + at), c));
  }
  // from the end: what the sums read last is still in L2
  const int64_t nv = (n - h) / VE, full = nv / (UN * BLK) * (UN * BLK);
  int64_t left = nv - full - tid;
  p += h * SZ + (full + tid) * 16;
  q += h * SZ + (full + tid) * 16;
  if (left > 0) {
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (left > u * BLK) v[u] = load_16<K>(p + u * BLK * 16, policy);
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (left > u * BLK) store_16<K>(q + u * BLK * 16, scale_vec<DT, 16, false>(v[u], c), policy);
  }
  for (left = full; left > 0; left -= UN * BLK) {
    p -= UN * BLK * 16;
    q -= UN * BLK * 16;
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) v[u] = load_16<K>(p + u * BLK * 16, policy);
#pragma unroll
    for (int u = 0; u < UN; ++u) store_16<K>(q + u * BLK * 16, scale_vec<DT, 16, false>(v[u], c), policy);
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

template <bool MAX, Keep K>
__device__ __forceinline__ void entry_sum(Acc<MAX>& a, uint32_t dtype, const void* in, int64_t at, int64_t n,
                                          uint64_t policy) {
  const char* p = static_cast<const char*>(in);
  if (dtype == ILQR_DTYPE_F32) range_sum<ILQR_DTYPE_F32, MAX, K>(a, p + at * 4, n, policy);
  else if (dtype == ILQR_DTYPE_BF16) range_sum<ILQR_DTYPE_BF16, MAX, K>(a, p + at * 2, n, policy);
  else range_sum<ILQR_DTYPE_F16, MAX, K>(a, p + at * 2, n, policy);
}

// Value by value: for coefficients below the floats' range, and for `in` and
// `out` that lie differently in their 16-byte words (new outputs of views packed
// at odd offsets). A thread has one load in flight: 200 MB of bf16 in 200 such
// views 231 us where the vectors take 99 (both passes), 200 MB of f32 147 and 99.
// The scaling alone runs at 21 % of DRAM's rate, its warps waiting for that load.
__device__ __forceinline__ void entry_scale_apart(uint32_t dtype, const char* p, char* q, int64_t n, const Coef& c) {
  const int sz = dtype == ILQR_DTYPE_F32 ? 4 : 2;
#pragma unroll 1
  for (int64_t i = threadIdx.x; i < n; i += BLK) {
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

template <Keep K, int UN>
__device__ __forceinline__ void entry_scale(uint32_t dtype, const void* in, void* out, int64_t at, int64_t n,
                                            const Coef& c, uint64_t policy) {
  const int sz = dtype == ILQR_DTYPE_F32 ? 4 : 2;
  const char* p = static_cast<const char*>(in) + at * sz;
  char* q = static_cast<char*>(out) + at * sz;
  if (c.wide || ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15u))
    entry_scale_apart(dtype, p, q, n, c);
  else if (dtype == ILQR_DTYPE_F32) range_scale<ILQR_DTYPE_F32, K, UN>(p, q, n, c, policy);
  else if (dtype == ILQR_DTYPE_BF16) range_scale<ILQR_DTYPE_BF16, K, UN>(p, q, n, c, policy);
  else range_scale<ILQR_DTYPE_F16, K, UN>(p, q, n, c, policy);
}

// Chunks [k, end) of the list into a sum, t the tensor of chunk k.
template <int CAP, bool MAX, Keep K>
__device__ __forceinline__ void chunks_sum(Acc<MAX>& a, const GradTable<CAP>& tab, uint32_t k, uint32_t end, int t,
                                           uint64_t policy) {
  for (; k < end; ++t) {
    const uint32_t stop = t + 1 < tab.n ? min(end, tab.e[t + 1].chunk0) : end;
    int64_t at, n;
    span(tab, t, k, stop, &at, &n);
    entry_sum<MAX, K>(a, tab.e[t].dtype, tab.e[t].in, at, n, policy);
    k = stop;
  }
}

// Partial sums, one for each block, of equal contiguous runs of chunks. Bound by
// DRAM: with the join 47.5 us for 300 MB, 143 us for 1 GB (7.0 TB/s, more than a
// copy's rate), of which 2 us are the two launches. Four blocks of 256 threads on
// an SM keep 64 KB of loads in flight; five to eight blocks, or eight loads a
// thread instead of four, were within 2 % either way.
template <int CAP, bool MAX>
__global__ void __launch_bounds__(BLK) grad_sum_kernel(const __grid_constant__ GradTable<CAP> tab, double* slots) {
  __shared__ double sh[32];
  asm volatile("griddepcontrol.launch_dependents;");
  const uint32_t k = first_chunk(blockIdx.x, tab.chunks, gridDim.x);
  Acc<MAX> a;
  chunks_sum<CAP, MAX, Keep::USUAL>(a, tab, k, first_chunk(blockIdx.x + 1, tab.chunks, gridDim.x), find(tab, k), 0);
  const double v = block_join<MAX>(value(a), sh);
  if (threadIdx.x == 0) slots[blockIdx.x] = v;
}

// The same before the scaling of a long list: the blocks go through it together,
// four chunks each at a time, so that its last part is read last; what lies
// before the last keep_chunks leaves L2 first (300 MB, both passes, in runs and
// so: 143 | 140 us; the sums alone are 47 | 49 us).
template <int CAP, bool MAX>
__global__ void __launch_bounds__(BLK) grad_sum_long_kernel(const __grid_constant__ GradTable<CAP> tab,
                                                            uint32_t keep_chunks, double* slots) {
  __shared__ double sh[32];
  asm volatile("griddepcontrol.launch_dependents;");
  const uint64_t first = policy_first_out(), usual = policy_usual();
  Acc<MAX> a;
  for (uint32_t k = blockIdx.x * 4; k < tab.chunks; k += gridDim.x * 4)
    chunks_sum<CAP, MAX, Keep::POLICY>(a, tab, k, min(k + 4, tab.chunks), find(tab, k),
                                       tab.chunks - k > keep_chunks ? first : usual);
  const double v = block_join<MAX>(value(a), sh);
  if (threadIdx.x == 0) slots[blockIdx.x] = v;
}

// Partial sums for each tensor. Each block takes a contiguous run of chunks and
// leaves one sum for each tensor in it at slot block + tensor: slots of
// neighbours are neighbours, and where a block ends with its tensor the one slot
// that falls out is set to 0, the identity of both joins. 400 bf16 tensors,
// 600 MB: 96 us with the join (6.2 TB/s).
template <int CAP, bool MAX>
__global__ void __launch_bounds__(BLK) grad_each_kernel(const __grid_constant__ GradTable<CAP> tab, double* slots) {
  __shared__ double sh[32];
  asm volatile("griddepcontrol.launch_dependents;");
  uint32_t k = first_chunk(blockIdx.x, tab.chunks, gridDim.x);
  const uint32_t k1 = first_chunk(blockIdx.x + 1, tab.chunks, gridDim.x);
  int t = find(tab, k);
  if (blockIdx.x > 0 && k == tab.e[t].chunk0 && threadIdx.x == 0) slots[blockIdx.x + t - 1] = 0.0;
  for (; k < k1; ++t) {
    const uint32_t end = t + 1 < tab.n ? min(k1, tab.e[t + 1].chunk0) : k1;
    Acc<MAX> a;
    chunks_sum<CAP, MAX, Keep::USUAL>(a, tab, k, end, t, 0);
    const double v = block_join<MAX>(value(a), sh);
    if (threadIdx.x == 0) slots[blockIdx.x + t] = v;
    k = end;
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
__global__ void __launch_bounds__(BLK) grad_join_kernel(const __grid_constant__ GradTable<CAP> tab, uint32_t grid,
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
  const int t = (int)(blockIdx.x - 1) * (BLK / 32) + (int)(threadIdx.x >> 5);
  if (t >= tab.n) return;
  const uint32_t c0 = tab.e[t].chunk0, c1 = t + 1 < tab.n ? tab.e[t + 1].chunk0 : tab.chunks;
  const uint32_t lo = block_of(c0, tab.chunks, grid) + t, hi = block_of(c1 - 1, tab.chunks, grid) + t;
  double v = 0.0;
  for (uint32_t i = lo + (threadIdx.x & 31); i <= hi; i += 32) v = join<MAX>(v, tab_slots[i]);
  v = warp_join<MAX>(v);
  if ((threadIdx.x & 31) == 0) out.tensor_norms[t] = (float)norm_of(v, MAX);
}

// out = c in over chunks [k0, k1), from the end (what the sums read last is still
// in L2), t the tensor of chunk k1 - 1. In place a coefficient of 1 leaves the
// values where they are.
template <int CAP, Keep K, int UN>
__device__ __forceinline__ void chunks_scale(const GradTable<CAP>& tab, uint32_t k0, uint32_t k1, int t, const Coef& c,
                                             uint64_t policy) {
  if (c.d == 1.0 && tab.in_place) return;
  for (; k1 > k0; --t) {
    const GradEntry& e = tab.e[t];
    const uint32_t begin = max(k0, e.chunk0);
    if (!(c.d == 1.0 && e.in == e.out)) {
      int64_t at, n;
      span(tab, t, begin, k1, &at, &n);
      entry_scale<K, UN>(e.dtype, e.in, e.out, at, n, c, policy);
    }
    k1 = begin;
  }
}

// A wave of blocks with a run of chunks each; every block joins the partial sums
// for itself, in the same order, instead of a launch between the two. For lists
// that L2 holds: 20 MB of bf16 16.1 us out of place with the sums; 32 MB below
// the bound and in place 9.4 us. Four blocks on an SM leave a thread 64 registers,
// of which the vectors in flight take most: 40 bytes of the rest are spilled.
template <int CAP>
__global__ void __launch_bounds__(BLK, 4) grad_scale_kernel(const __grid_constant__ GradTable<CAP> tab, GradScale s,
                                                            const double* slots, int64_t n_slots, float* norm) {
  __shared__ double sh[32];
  const uint32_t k0 = first_chunk(blockIdx.x, tab.chunks, gridDim.x);
  const uint32_t k1 = first_chunk(blockIdx.x + 1, tab.chunks, gridDim.x);
  const int t = find(tab, k1 - 1);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double total = s.max_type ? join_slots<true>(slots, n_slots, sh) : join_slots<false>(slots, n_slots, sh);
  const double nrm = norm_of(total, s.max_type);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nrm;
  chunks_scale<CAP, Keep::USUAL, UN>(tab, k0, k1, t, coef_of(nrm, s.max_norm, s.eps), 0);
}

// A long list: the blocks go through it together from the end, GRAD_LONG_STEP
// chunks at a time. The total is one value. 276 MB (x0, C, c of B = 16384, T = 20)
// out of place: 129 us, 47 of them the sums, 82 this: the rate of a plain product
// of the same tensors (82 us). DRAM brings 214 MB of the second reading, L2 the
// rest; without the policies 136 us.
template <int CAP>
__global__ void __launch_bounds__(BLK, 8) grad_scale_long_kernel(const __grid_constant__ GradTable<CAP> tab,
                                                                 GradScale s, const double* total, float* norm) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double nrm = norm_of(*total, s.max_type);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nrm;
  const Coef c = coef_of(nrm, s.max_norm, s.eps);
  if (c.d == 1.0 && tab.in_place) return;
  const uint64_t policy = policy_first_out();
  for (uint32_t past = blockIdx.x * GRAD_LONG_STEP; past < tab.chunks; past += gridDim.x * GRAD_LONG_STEP) {
    const uint32_t k1 = tab.chunks - past, k0 = k1 > GRAD_LONG_STEP ? k1 - GRAD_LONG_STEP : 0;
    chunks_scale<CAP, Keep::POLICY, 2>(tab, k0, k1, find(tab, k1 - 1), c, policy);
  }
}

// A short list by one cluster, in one launch and without a workspace: the
// blocks' sums meet in shared memory, and what they read again is in L1 or L2.
template <int CAP, bool MAX, bool SCALE>
__global__ void __launch_bounds__(BLK) grad_small_kernel(const __grid_constant__ GradTable<CAP> tab, GradScale s,
                                                         GradNormOut out) {
  __shared__ double sh[33];
  const uint32_t rank = cluster_rank(), n_blocks = cluster_size();
  const uint32_t k0 = first_chunk(rank, tab.chunks, n_blocks), k1 = first_chunk(rank + 1, tab.chunks, n_blocks);
  Acc<MAX> a;
  if (k0 < k1) chunks_sum<CAP, MAX, Keep::USUAL>(a, tab, k0, k1, find(tab, k0), 0);
  const double total = cluster_join<MAX>(block_join<MAX>(value(a), sh), sh + 32);
  const double nrm = norm_of(total, MAX);
  if (rank == 0 && threadIdx.x == 0) {
    if (out.norm != nullptr) *out.norm = (float)nrm;
    if (out.total != nullptr) *out.total = total;
  }
  if constexpr (SCALE) {
    if (k0 < k1)
      chunks_scale<CAP, Keep::USUAL, UN>(tab, k0, k1, find(tab, k1 - 1), coef_of(nrm, s.max_norm, s.eps), 0);
  }
  cluster_wait();
}

// ---- batch elements ---------------------------------------------------------

// Vector i of a slice lies in segment i / seg_vecs: a multiplication by the
// reciprocal, rounded up at 2^-(32 + shift), exact for i < 2^31.
__device__ __forceinline__ int64_t vec_at(const RowTensor& r, uint32_t i, uint32_t vb, int64_t seg_stride) {
  if (r.n_seg == 1) return (int64_t)i * vb;
  const uint32_t s = r.seg_vecs == 1 ? i : __umulhi(i, r.magic) >> r.shift;
  return s * seg_stride + (int64_t)(i - s * r.seg_vecs) * vb;
}

template <int VB>
__device__ __forceinline__ void copy_async(uint32_t to, const char* from) {
  if constexpr (VB == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(VB) : "memory");
  }
}

// How a slice gets to shared memory and back. Long segments move by bulk
// copies, one each, issued by all threads: each segment has a place of
// whole 16-byte words, lies there at its address modulo 16, and the copy takes
// its whole words. What is left at its two ends moves value by value, and zeros
// fill the place, so that sums and products run over whole words. Other slices
// move by the threads, a vector each.
struct Piece {
  uint32_t off;    // of the segment in its place: its address modulo 16
  uint32_t lead;   // bytes before the first whole word
  uint32_t whole;  // bytes of whole words
};

__device__ __forceinline__ Piece piece_of(const RowTensor& r, const char* p) {
  Piece c;
  c.off = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u);
  c.lead = -c.off & 15u;
  c.whole = (r.seg_bytes - c.lead) & ~15u;
  return c;
}

// Every `issuers`-th segment from the issuer's own; returns the bytes that these
// copies bring.
__device__ __forceinline__ uint32_t bulk_in(const RowTensor& r, int64_t b, uint32_t to, uint64_t* bar, uint32_t issuer,
                                            uint32_t issuers) {
  const char* p = r.in + b * r.in_row;
  uint32_t bytes = 0;
  for (uint32_t s = issuer; s < r.n_seg; s += issuers) {
    const char* from = p + s * r.in_seg;
    const Piece c = piece_of(r, from);
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            to + s * r.place + c.off + c.lead),
        "l"(from + c.lead), "r"(c.whole), "r"(smem_u32(bar))
        : "memory");
    bytes += c.whole;
  }
  return bytes;
}

__device__ __forceinline__ void bulk_out(const RowTensor& r, int64_t b, uint32_t at, uint32_t issuer,
                                         uint32_t issuers) {
  char* q = r.out + b * r.out_row;
  for (uint32_t s = issuer; s < r.n_seg; s += issuers) {
    char* to = q + s * r.out_seg;
    const Piece c = piece_of(r, to);
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to + c.lead),
                 "r"(at + s * r.place + c.off + c.lead), "r"(c.whole)
                 : "memory");
  }
}

// The ends of the segments, one for each thread: the first word of a place, where
// the segment begins within it, and what follows the last whole one.
template <int VB, bool OUT>
__device__ __forceinline__ void ends(const RowTensor& r, int64_t b, char* staged, uint32_t lane, uint32_t step) {
  constexpr uint32_t N = 16 / VB;
  char* g = OUT ? r.out + b * r.out_row : const_cast<char*>(r.in) + b * r.in_row;
  const int64_t seg = OUT ? r.out_seg : r.in_seg;
  for (uint32_t i = lane; i < 2 * r.n_seg; i += step) {
    const uint32_t s = i >> 1;
    char* q = g + s * seg;
    const Piece c = piece_of(r, q);
    const bool first = (i & 1) == 0;
    if (first && c.lead == 0) continue;  // it begins with a whole word
    const uint32_t at = first ? 0 : c.off + c.lead + c.whole;
    const uint32_t from = first ? c.off : 0, to = first ? 16 : c.off + r.seg_bytes - at;
    char* mine = staged + s * r.place + at;
    char* theirs = q + ((int64_t)at - c.off);
    __align__(16) Vec<VB> w[N];
    if constexpr (OUT) {
      if (from < to) *reinterpret_cast<Vec<16>*>(w) = load_vec<16>(mine);
#pragma unroll
      for (uint32_t u = 0; u < N; ++u)
        if (u * VB >= from && u * VB < to) *reinterpret_cast<Vec<VB>*>(theirs + u * VB) = w[u];
    } else {
#pragma unroll
      for (uint32_t u = 0; u < N; ++u) {
        w[u] = Vec<VB>{};
        if (u * VB >= from && u * VB < to) w[u] = load_vec<VB>(theirs + u * VB);
      }
      const uint32_t room = first ? 16 : r.place - at;
      if (room > 0) *reinterpret_cast<Vec<16>*>(mine) = *reinterpret_cast<const Vec<16>*>(w);
      for (uint32_t x = 16; x < room; x += 16) *reinterpret_cast<Vec<16>*>(mine + x) = Vec<16>{};
    }
  }
}

template <bool OUT>
__device__ __forceinline__ void ends(const RowTensor& r, int64_t b, char* staged, uint32_t lane, uint32_t step) {
  if (r.vec_bytes == 8) ends<8, OUT>(r, b, staged, lane, step);
  else if (r.vec_bytes == 4) ends<4, OUT>(r, b, staged, lane, step);
  else ends<2, OUT>(r, b, staged, lane, step);
}

template <int VB>
__device__ __forceinline__ void threads_in(const RowTensor& r, int64_t b, uint32_t to, uint32_t lane, uint32_t step) {
  const char* p = r.in + b * r.in_row;
  const uint32_t n = r.n_seg * r.seg_vecs;
  if constexpr (VB > 2) {
    for (uint32_t i = lane; i < n; i += step) copy_async<VB>(to + i * VB, p + vec_at(r, i, VB, r.in_seg));
  } else {  // through registers: there is no asynchronous copy of two bytes
    for (uint32_t i = lane; i < n; i += UN * step) {
      uint16_t w[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (i + u * step < n) w[u] = *reinterpret_cast<const uint16_t*>(p + vec_at(r, i + u * step, 2, r.in_seg));
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (i + u * step < n) asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + (i + u * step) * 2), "h"(w[u]) : "memory");
    }
  }
}

template <int VB>
__device__ __forceinline__ void threads_out(const RowTensor& r, int64_t b, const char* from, uint32_t lane,
                                            uint32_t step) {
  char* q = r.out + b * r.out_row;
  const uint32_t n = r.n_seg * r.seg_vecs;
  for (uint32_t i = lane; i < n; i += step)
    *reinterpret_cast<Vec<VB>*>(q + vec_at(r, i, VB, r.out_seg)) = load_vec<VB>(from + i * VB);
}

// n 16-byte vectors of shared memory into a sum, and scaled where they are
template <int DT>
__device__ __forceinline__ void staged_sum(Acc<false>& a, const char* p, uint32_t n, uint32_t lane, uint32_t step) {
  for (uint32_t i = lane; i < n; i += UN * step) {
    Vec<16> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      v[u] = Vec<16>{};
      if (i + u * step < n) v[u] = load_vec<16>(p + (i + u * step) * 16);
    }
    add_vecs<DT, 16, UN, false>(a, v);
  }
}

template <int DT>
__device__ __forceinline__ void staged_scale(char* p, uint32_t n, const Coef& c, uint32_t lane, uint32_t step) {
#pragma unroll 4
  for (uint32_t i = lane; i < n; i += step) {
    Vec<16>* v = reinterpret_cast<Vec<16>*>(p + i * 16);
    *v = scale_vec<DT, 16, false>(*v, c);
  }
}

__device__ __forceinline__ void staged_sum(Acc<false>& a, uint32_t dtype, const char* p, uint32_t n, uint32_t lane,
                                           uint32_t step) {
  if (dtype == ILQR_DTYPE_F32) staged_sum<ILQR_DTYPE_F32>(a, p, n, lane, step);
  else if (dtype == ILQR_DTYPE_BF16) staged_sum<ILQR_DTYPE_BF16>(a, p, n, lane, step);
  else staged_sum<ILQR_DTYPE_F16>(a, p, n, lane, step);
}

__device__ __forceinline__ void staged_scale(uint32_t dtype, char* p, uint32_t n, const Coef& c, uint32_t lane,
                                             uint32_t step) {
  if (dtype == ILQR_DTYPE_F32) staged_scale<ILQR_DTYPE_F32>(p, n, c, lane, step);
  else if (dtype == ILQR_DTYPE_BF16) staged_scale<ILQR_DTYPE_BF16>(p, n, c, lane, step);
  else staged_scale<ILQR_DTYPE_F16>(p, n, c, lane, step);
}

// Zeros in their place, or scaled by a coefficient below the floats' range.
__device__ __noinline__ void staged_apart(uint32_t dtype, char* p, uint32_t n, const Coef& c, bool zero, uint32_t lane,
                                          uint32_t step) {
  if (zero) {
#pragma unroll 1
    for (uint32_t i = lane; i < n; i += step) *reinterpret_cast<Vec<16>*>(p + i * 16) = Vec<16>{};
  } else if (dtype == ILQR_DTYPE_F32) {
#pragma unroll 1
    for (uint32_t i = lane; i < n * 4; i += step) {
      float* x = reinterpret_cast<float*>(p) + i;
      *x = scaled<true>(*x, c);
    }
  } else {
#pragma unroll 1
    for (uint32_t i = lane; i < n * 8; i += step) {
      char* at = p + i * 2;
      if (dtype == ILQR_DTYPE_BF16)
        store_one<ILQR_DTYPE_BF16>(at, scaled<true>(load_one<ILQR_DTYPE_BF16>(at), c));
      else
        store_one<ILQR_DTYPE_F16>(at, scaled<true>(load_one<ILQR_DTYPE_F16>(at), c));
    }
  }
}

// The same from global memory, for slices that shared memory cannot hold.
template <int DT, int VB>
__device__ __forceinline__ void row_sum(Acc<false>& a, const RowTensor& r, int64_t b, uint32_t lane, uint32_t step) {
  const char* p = r.in + b * r.in_row;
  const uint32_t n = r.n_seg * r.seg_vecs;
  for (uint32_t i = lane; i < n; i += UN * step) {
    Vec<VB> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const uint32_t k = i + u * step;
      v[u] = Vec<VB>{};
      if (k < n) v[u] = load_vec<VB>(p + vec_at(r, k, VB, r.in_seg));
    }
    add_vecs<DT, VB, UN, false>(a, v);
  }
}

template <int DT, int VB>
__device__ __forceinline__ void row_scale(const RowTensor& r, int64_t b, const Coef& c, uint32_t lane, uint32_t step) {
  const char* p = r.in + b * r.in_row;
  char* q = r.out + b * r.out_row;
  const uint32_t n = r.n_seg * r.seg_vecs;
#pragma unroll 4
  for (uint32_t i = lane; i < n; i += step) {
    const Vec<VB> v = load_vec<VB>(p + vec_at(r, i, VB, r.in_seg));
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

// The threads of a group: a part of a warp, a warp, or the block.
template <int G>
__device__ __forceinline__ uint32_t group_mask() {
  if constexpr (G >= 32) return 0xffffffffu;
  else return ((1u << G) - 1u) << (threadIdx.x % 32 / G * G);
}

template <int G>
__device__ __forceinline__ void group_sync() {
  if constexpr (G <= 32) __syncwarp(group_mask<G>());
  else __syncthreads();
}

template <int G>
__device__ __forceinline__ double group_sum(double v, double* sh) {
  if constexpr (G > 32) {
    return block_join<false>(v, sh);
  } else {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(group_mask<G>(), v, o);
    return v;
  }
}

// The part of a slice that one of several blocks takes: segments, or of a
// single segment a run of whole 16-byte words.
__device__ __forceinline__ RowTensor part_of(const RowTensor& r, uint32_t rank, uint32_t parts) {
  RowTensor x = r;
  if (r.n_seg > 1) {
    const uint32_t s0 = (uint32_t)((uint64_t)r.n_seg * rank / parts);
    const uint32_t s1 = (uint32_t)((uint64_t)r.n_seg * (rank + 1) / parts);
    x.in += s0 * r.in_seg;
    x.out += s0 * r.out_seg;
    x.n_seg = s1 - s0;
  } else {
    const uint32_t words = (r.seg_bytes + 15) / 16;
    const uint32_t o0 = (uint32_t)((uint64_t)words * rank / parts) * 16;
    const uint32_t o1 = min((uint32_t)((uint64_t)words * (rank + 1) / parts) * 16, r.seg_bytes);
    x.in += o0;
    x.out += o0;
    x.seg_bytes = o1 - o0;
    x.seg_vecs = x.seg_bytes / r.vec_bytes;
    x.n_seg = x.seg_bytes > 0 ? 1 : 0;
    x.place = x.seg_bytes;
    if (r.bulk == ROW_BULK_ENDS) x.place = (x.seg_bytes + 30) / 16 * 16;
    if (x.seg_bytes < GRAD_MIN_BULK) x.bulk = ROW_THREADS, x.place = x.seg_bytes;
  }
  x.staged_vecs = (x.n_seg * x.place + 15) / 16;
  return x;
}

// G threads for each element, whose slices are staged in shared memory: global
// memory is read once and written once. CLUSTER: the blocks of a cluster share
// one element. Bound by DRAM for elements of some KB and more: B = 65536, T = 50
// time-major 878 us for 5.5 GB (6.28 TB/s, 96 % of the copy rate); B = 16384,
// T = 20 94 us time-major, 87 us batch-major for 552 MB; the 13-state model,
// B = 4096, T = 20 33 us for 201 MB. What the time-major layout costs it costs in
// writing (reading alone 112 us against 109, T = 50, 0.8 GB; with writing 250
// against 230), and the more the more segments an element has. Segments of 16-bit
// values that are no whole 16-byte words (392 bytes, and 28) cost instructions
// besides: 2490 of a warp for each element of 8.4 KB, issued in 55 % of the
// cycles, 70 us for 276 MB. Shorter elements are bound by instructions and by the
// wait of a warp for its few loads: B = 16384 sigmoid rows of 2.3 KB 15 us for
// 75 MB; B = 65536 rows of 300 bytes of bf16 1290 instructions for a warp's eight,
// 16.6 us for 39 MB (of 600 bytes of f32 1000, 18.5 us for 79 MB).
template <int G, int THREADS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, G <= 32 ? 1280 / THREADS : 1)
    grad_rows_kernel(const __grid_constant__ RowTable tab) {
  extern __shared__ __align__(16) char staged[];
  __shared__ double sh[33];
  __shared__ uint64_t bars[THREADS / G];
  __shared__ RowTensor parts[CLUSTER ? ROW_MAX_TENSORS : 1];
  constexpr int PER = THREADS / G;
  // Every thread issues bulk copies, neighbouring segments by different warps: a
  // warp issues those of its lanes one after the other (one warp for all: reading
  // 0.8 GB of 784-byte segments took 137 us instead of 112).
  constexpr uint32_t WARPS = G > 32 ? G / 32 : 1;
  const uint32_t group = threadIdx.x / G, lane = threadIdx.x % G;
  int64_t b = (int64_t)blockIdx.x * PER + group;
  uint32_t staged_bytes = tab.staged_bytes;
  const RowTensor* tensors = tab.t;
  if constexpr (CLUSTER) {
    const uint32_t rank = cluster_rank(), n = cluster_size();
    b = blockIdx.x / n;
    if (threadIdx.x < tab.n) parts[threadIdx.x] = part_of(tab.t[threadIdx.x], rank, n);
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t at = 0;
      for (int k = 0; k < tab.n; ++k) {
        parts[k].staged = at;
        at += parts[k].staged_vecs * 16;
      }
    }
    __syncthreads();
    tensors = parts;
    staged_bytes = parts[tab.n - 1].staged + parts[tab.n - 1].staged_vecs * 16;
  }
  if (b >= tab.B) return;  // of a whole group, or not at all
  char* mine = staged + group * staged_bytes;
  const uint32_t to = smem_u32(mine);
  uint64_t* bar = bars + group;
  const uint32_t issuer = lane % 32 * WARPS + lane / 32;
  if (tab.bulk) {
    if (lane == 0) {
      mbar_init(bar, G);
      fence_mbar_init();
    }
    group_sync<G>();
    uint32_t bytes = 0;
    for (int k = 0; k < tab.n; ++k)
      if (tensors[k].bulk) bytes += bulk_in(tensors[k], b, to + tensors[k].staged, bar, issuer, G);
    mbar_expect_tx(bar, bytes);
  }
  for (int k = 0; k < tab.n; ++k) {
    const RowTensor& r = tensors[k];
    if (r.bulk) {
      if (r.bulk == ROW_BULK_ENDS) ends<false>(r, b, mine + r.staged, lane, G);
      continue;
    }
    if (r.vec_bytes == 16) threads_in<16>(r, b, to + r.staged, lane, G);
    else if (r.vec_bytes == 8) threads_in<8>(r, b, to + r.staged, lane, G);
    else if (r.vec_bytes == 4) threads_in<4>(r, b, to + r.staged, lane, G);
    else threads_in<2>(r, b, to + r.staged, lane, G);
    // zeros after it, to a whole word
    const uint32_t end = r.n_seg * r.seg_bytes;
    for (uint32_t x = lane * 2; x < (-end & 15u); x += G * 2)
      *reinterpret_cast<uint16_t*>(mine + r.staged + end + x) = 0;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  group_sync<G>();  // the threads' copies and the barrier's set-up
  Acc<false> a;
  // copies that never come (after a second, as bounded, wait) make the
  // element's norm NaN
  if (tab.bulk && !mbar_wait(bar, 0) && !mbar_wait(bar, 0)) a.s = __longlong_as_double(0x7ff8000000000000ll);
  if (tab.one_dtype) {
    staged_sum(a, tab.t[0].dtype, mine, staged_bytes / 16, lane, G);
  } else {
    for (int k = 0; k < tab.n; ++k)
      staged_sum(a, tensors[k].dtype, mine + tensors[k].staged, tensors[k].staged_vecs, lane, G);
  }
  double total = group_sum<G>(a.s, sh);
  if constexpr (CLUSTER) total = cluster_join<false>(total, sh + 32);
  const double nrm = sqrt(total);
  if (lane == 0 && tab.norms != nullptr && (!CLUSTER || cluster_rank() == 0)) tab.norms[b] = (float)nrm;
  const Coef c = coef_of(nrm, tab.max_norm, tab.eps);
  const bool zero = tab.zero_nonfinite && !isfinite(nrm);
  const bool changed = c.d != 1.0 || zero;
  if (changed) {
    if (zero || c.wide) {
      for (int k = 0; k < tab.n; ++k)
        staged_apart(tensors[k].dtype, mine + tensors[k].staged, tensors[k].staged_vecs, c, zero, lane, G);
    } else if (tab.one_dtype) {
      staged_scale(tab.t[0].dtype, mine, staged_bytes / 16, c, lane, G);
    } else {
      for (int k = 0; k < tab.n; ++k)
        staged_scale(tensors[k].dtype, mine + tensors[k].staged, tensors[k].staged_vecs, c, lane, G);
    }
    fence_proxy_async();
    group_sync<G>();
  }
  if (tab.bulk) {
    for (int k = 0; k < tab.n; ++k) {
      const RowTensor& r = tensors[k];
      if (r.bulk && (changed || r.in != r.out)) bulk_out(r, b, to + r.staged, issuer, G);
    }
    bulk_commit();
  }
  for (int k = 0; k < tab.n; ++k) {
    const RowTensor& r = tensors[k];
    if (!changed && r.in == r.out) continue;
    if (r.bulk) {
      if (r.bulk == ROW_BULK_ENDS) ends<true>(r, b, mine + r.staged, lane, G);
      continue;
    }
    if (r.vec_bytes == 16) threads_out<16>(r, b, mine + r.staged, lane, G);
    else if (r.vec_bytes == 8) threads_out<8>(r, b, mine + r.staged, lane, G);
    else if (r.vec_bytes == 4) threads_out<4>(r, b, mine + r.staged, lane, G);
    else threads_out<2>(r, b, mine + r.staged, lane, G);
  }
  if (tab.bulk) bulk_wait_read<0>();      // the copies read this block's memory
  if constexpr (CLUSTER) cluster_wait();  // and the cluster's blocks their sums
}

// Elements that the shared memory of a cluster cannot hold: its blocks share one,
// and both passes read global memory. 64 elements of 2.8 MB 100 us, 300 of 2 MB
// 310 us (3.9 TB/s of what must move); a single one of 52 MB 248 us, what eight SMs
// can read and write.
__global__ void __launch_bounds__(LONG_BLK) grad_long_rows_kernel(const __grid_constant__ RowTable tab) {
  __shared__ double sh[33];
  const uint32_t n_blocks = cluster_size();
  const int64_t b = blockIdx.x / n_blocks;
  const uint32_t lane = cluster_rank() * LONG_BLK + threadIdx.x, step = n_blocks * LONG_BLK;
  Acc<false> a;
  for (int k = 0; k < tab.n; ++k) {
    const RowTensor& r = tab.t[k];
#define CALL(DT, VB) row_sum<DT, VB>(a, r, b, lane, step)
    ROW_DISPATCH(r, CALL)
#undef CALL
  }
  const double nrm = sqrt(cluster_join<false>(block_join<false>(a.s, sh), sh + 32));
  if (lane == 0 && tab.norms != nullptr) tab.norms[b] = (float)nrm;
  const Coef c = coef_of(nrm, tab.max_norm, tab.eps);
  const bool zero = tab.zero_nonfinite && !isfinite(nrm);
  for (int k = 0; k < tab.n; ++k) {
    const RowTensor& r = tab.t[k];
    if (c.d == 1.0 && !zero && r.in == r.out) continue;
    if (zero || c.wide) {
      row_apart(r, b, c, zero, lane, step);
      continue;
    }
#define CALL(DT, VB) row_scale<DT, VB>(r, b, c, lane, step)
    ROW_DISPATCH(r, CALL)
#undef CALL
  }
  cluster_wait();
}

// ---- launches ---------------------------------------------------------------

template <typename... K, typename... A>
cudaError_t launch(void (*kernel)(K...), unsigned grid, bool dependent, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(BLK);
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
cudaError_t launch_grad_sum(const GradTable<CAP>& tab, int grid, bool max_type, uint32_t keep_chunks, double* slots,
                            cudaStream_t stream) {
  if (keep_chunks > 0)
    return max_type ? launch(grad_sum_long_kernel<CAP, true>, grid, false, stream, tab, keep_chunks, slots)
                    : launch(grad_sum_long_kernel<CAP, false>, grid, false, stream, tab, keep_chunks, slots);
  return max_type ? launch(grad_sum_kernel<CAP, true>, grid, false, stream, tab, slots)
                  : launch(grad_sum_kernel<CAP, false>, grid, false, stream, tab, slots);
}

template <int CAP>
cudaError_t launch_grad_each(const GradTable<CAP>& tab, int grid, bool max_type, double* slots, cudaStream_t stream) {
  return max_type ? launch(grad_each_kernel<CAP, true>, grid, false, stream, tab, slots)
                  : launch(grad_each_kernel<CAP, false>, grid, false, stream, tab, slots);
}

template <int CAP>
cudaError_t launch_grad_join(const GradTable<CAP>* tab, int grid, const double* tab_slots, bool max_type,
                             const double* slots, int64_t n_slots, const GradNormOut& out, bool want_global,
                             cudaStream_t stream) {
  static const GradTable<CAP> none{};
  const unsigned blocks = 1 + (tab != nullptr ? (unsigned)(tab->n + BLK / 32 - 1) / (BLK / 32) : 0);
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

template <int CAP>
cudaError_t launch_grad_scale_long(const GradTable<CAP>& tab, const GradScale& s, const double* total, float* norm,
                                   bool dependent, cudaStream_t stream) {
  const unsigned grid = min((tab.chunks + GRAD_LONG_STEP - 1) / GRAD_LONG_STEP, GRAD_LONG_GRID);
  return launch(grad_scale_long_kernel<CAP>, grid, dependent, stream, tab, s, total, norm);
}

template <int CAP, bool MAX, bool SCALE>
static cudaError_t launch_small(const GradTable<CAP>& tab, const GradScale& s, const GradNormOut& out,
                                cudaStream_t stream) {
  unsigned blocks = 1;
  while (blocks < (unsigned)GRAD_SMALL_BLOCKS && blocks < tab.chunks) blocks *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(BLK);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {blocks, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, grad_small_kernel<CAP, MAX, SCALE>, tab, s, out);
}

template <int CAP>
cudaError_t launch_grad_small(const GradTable<CAP>& tab, bool max_type, const GradScale* s, const GradNormOut& out,
                              cudaStream_t stream) {
  const GradScale none{};
  if (s != nullptr)
    return max_type ? launch_small<CAP, true, true>(tab, *s, out, stream)
                    : launch_small<CAP, false, true>(tab, *s, out, stream);
  return max_type ? launch_small<CAP, true, false>(tab, none, out, stream)
                  : launch_small<CAP, false, false>(tab, none, out, stream);
}

#define INSTANTIATE(CAP)                                                                                              \
  template cudaError_t launch_grad_sum<CAP>(const GradTable<CAP>&, int, bool, uint32_t, double*, cudaStream_t);       \
  template cudaError_t launch_grad_each<CAP>(const GradTable<CAP>&, int, bool, double*, cudaStream_t);                \
  template cudaError_t launch_grad_join<CAP>(const GradTable<CAP>*, int, const double*, bool, const double*, int64_t, \
                                             const GradNormOut&, bool, cudaStream_t);                                 \
  template cudaError_t launch_grad_scale<CAP>(const GradTable<CAP>&, int, const GradScale&, const double*, int64_t,   \
                                              float*, bool, cudaStream_t);                                            \
  template cudaError_t launch_grad_scale_long<CAP>(const GradTable<CAP>&, const GradScale&, const double*, float*,    \
                                                   bool, cudaStream_t);
template cudaError_t launch_grad_small<GRAD_CAP_SHORT>(const GradTable<GRAD_CAP_SHORT>&, bool, const GradScale*,
                                                       const GradNormOut&, cudaStream_t);
INSTANTIATE(GRAD_CAP_SHORT)
INSTANTIATE(GRAD_CAP_MIDDLE)
INSTANTIATE(GRAD_CAP_LONG)
#undef INSTANTIATE

namespace {

// The most that one of `parts` blocks stages of an element: up to a segment and
// the words' ends of each tensor beyond the even share.
size_t part_bytes(const RowTable& tab, size_t parts) {
  size_t bytes = 0;
  for (int k = 0; k < tab.n; ++k) {
    const RowTensor& r = tab.t[k];
    bytes += r.n_seg > 1 ? ((r.n_seg + parts - 1) / parts * r.place + 15) / 16 * 16
                         : (r.staged_vecs + parts - 1) / parts * 16 + 48;
  }
  return bytes;
}

// cluster: blocks of a cluster, which share an element (CLUSTER) or have one each
// and are together only to run on neighbouring SMs.
template <int G, int THREADS, bool CLUSTER = false>
cudaError_t launch_rows(const RowTable& tab, cudaStream_t stream, unsigned cluster = 1) {
  constexpr int PER = THREADS / G;
  const size_t smem = CLUSTER ? part_bytes(tab, cluster) : (size_t)tab.staged_bytes * PER;
  const auto kernel = grad_rows_kernel<G, THREADS, CLUSTER>;
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may have all shared memory
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)GRAD_MAX_STAGED);
    if (e != cudaSuccess) return e;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  const int64_t blocks = CLUSTER ? tab.B * cluster : (tab.B + PER - 1) / PER;
  cfg.gridDim = dim3((unsigned)((blocks + cluster - 1) / cluster * cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {cluster, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, tab);
}

}  // namespace

cudaError_t launch_grad_rows(const RowTable& tab, cudaStream_t stream) {
  // Threads for an element by what it stages. More threads cost instructions
  // that every element repeats (its records, the join, square root and quotient),
  // fewer leave the additions of long elements to few: us by threads, bytes of an
  // element of float32 and number of elements (without the pairs below):
  //     bytes (elements)    4     8    16    32    64   128   256
  //       264 (100000)     15    19    31    55   120   205
  //       600  (60000)     16    18    25    40    82   141
  //      1720  (40000)     30    25    28    39    75   129
  //      2280  (65536)     53    49    48    52    93   161
  //      4240  (16384)     40    36    28    27    39    60
  //      8440  (16384)    117    82    58    49    49    70   129
  //     16840  (16384)                 113    86    86    86   121
  //     24532   (4096)                  93    64    52    49    56
  //     42040  (65536)                      1409   877   887   873
  //     84040   (2048)                              92    76    72
  //    210040   (1024)                             157   119   111
  // 16-bit elements go by the same bytes; theirs were not swept.
  if (tab.staged_bytes <= 640) return launch_rows<4, 64>(tab, stream);
  if (tab.staged_bytes <= 2048) return launch_rows<8, 128>(tab, stream);
  if (tab.staged_bytes <= 4096) return launch_rows<16, 128>(tab, stream);
  if (tab.staged_bytes <= 12288) return launch_rows<32, 128>(tab, stream);
  if (tab.staged_bytes <= 20480) return launch_rows<64, 64>(tab, stream);
  // Blocks of neighbouring elements in pairs, whose segments' ends meet in a line
  // of L2: with up to twelve of them on an SM 42040 bytes 887 -> 869 us, 24532
  // time-major 48.5 -> 44.6, batch-major 35.0 -> 33.4; with more (16840 bytes) the
  // scheduling of pairs costs more than that, 95 -> 110.
  if (tab.staged_bytes <= 65536) return launch_rows<128, 128>(tab, stream, 2);
  if (tab.staged_bytes <= 114688) return launch_rows<256, 256>(tab, stream);
  // Longer ones leave an SM one block, whose copies, sums and stores take turns:
  // blocks of a cluster share them. us in one block | 2 | 4 | 8:
  //  84040 (2048)  72 | 79 | 90 | 134      210040 (1024)  111 | 105 | 103 | 104
  for (unsigned parts = 2; parts <= 8; parts *= 2)
    if (part_bytes(tab, parts) <= (parts < 8 ? 57344 : GRAD_MAX_STAGED))
      return launch_rows<128, 128, true>(tab, stream, parts);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)tab.B * 8);
  cfg.blockDim = dim3(LONG_BLK);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {8, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, grad_long_rows_kernel, tab);
}

}  // namespace ilqr
