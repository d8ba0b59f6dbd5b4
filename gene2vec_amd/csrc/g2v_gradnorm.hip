// g2v_gradnorm.hip -- the global norm of a list of gradients, and clipping.
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   clip: dst = g * (clip / max(norm, clip)); NaN everywhere when an element is
//         not finite (an overflow is not hidden).  A finite norm beyond fp32 is
//         returned as infinity, and its elements are clipped.
//
// The squares are formed and added in fp64: an fp32 sum would overflow from
// elements of 1.8e19 on and lose the small tensors beside the large ones, and
// gfx950 adds fp64 far faster than memory delivers the elements.  Memory bound:
// 10^9 bf16 elements in 48 tensors 314 us (6.4 TB/s), clipping 3 * 10^8 elements
// of two types in 600 tensors 586 us (1 GB read twice and written).  No atomics:
// every workgroup writes one partial sum, and they are added in a fixed order,
// so the same gradients give the same bits.
//
// The tensors' addresses travel in the kernel arguments, kTensors a launch: no
// copy from the host, nothing that a captured graph would have to keep alive.
// Longer lists are first written to the workspace by small launches, so that
// the tensors themselves are always read by one launch, and clipped by one.
#include <algorithm>
#include <vector>

#include "g2v_ops.h"

namespace {

using g2v::bf16;
using g2v::f16;

constexpr int kThreads = 256;
constexpr int kTensors = 128;       // per launch: 3.7 KB of arguments
constexpr int kMaxPartials = 2048;  // workgroups: 8 per CU
// all of them resident: 8 waves a SIMD, so at most 64 registers.  At the 66 and 73
// that the compiler takes unasked only 7 or 6 of a CU's 8 fit, and the rest of
// the equal shares begin when the first have ended: the norm of 10^9 bf16
// elements 314 us against 339, clipping 3 * 10^8 in 600 tensors 586 against 590
constexpr int kWaves = 8;
constexpr int64_t kChunk = 8192;    // elements a workgroup takes at a time
constexpr int kAlign = 64;          // bytes: where a tensor's chunks begin

struct Tensors {  // in the kernel arguments
  const void* src[kTensors];
  void* dst[kTensors];
  int64_t numel[kTensors];
  int32_t first[kTensors + 1];  // chunks before tensor t
  int8_t type[kTensors];
  int32_t n;
};

struct TensorList {  // the same in the workspace
  const void** src;
  void** dst;
  int64_t* numel;
  int32_t* first;
  int8_t* type;
  int32_t n;
};

// A tensor's first chunk also takes the elements before the first aligned
// address: the rest is read in whole cache lines.
__host__ __device__ __forceinline__ int64_t head_of(const void* p, int64_t numel, int bytes) {
  const int64_t h = (int64_t)((0 - (uintptr_t)p) % kAlign) / bytes;
  return h < numel ? h : numel;
}

inline int64_t chunks_of(const void* p, int64_t numel, int type) {
  if (numel == 0) return 0;
  const int64_t n = numel - head_of(p, numel, (int)g2v::type_bytes(type));
  return n > kChunk ? (n + kChunk - 1) / kChunk : 1;
}

__global__ __launch_bounds__(kTensors) void k_list(Tensors a, TensorList to, int at,
                                                   int chunks_before) {
  const int t = threadIdx.x;
  if (t < a.n) {
    to.src[at + t] = a.src[t];
    to.dst[at + t] = a.dst[t];
    to.numel[at + t] = a.numel[t];
    to.type[at + t] = a.type[t];
    to.first[at + t + 1] = chunks_before + a.first[t + 1];
  }
  if (t == 0 && at == 0) to.first[0] = 0;
}

template <class F>
__device__ __forceinline__ void by_type_dev(int type, F f) {
  if (type == G2V_F32) f(float{});
  else if (type == G2V_F16) f(f16{});
  else f(bf16{});
}

// the sum over the workgroup, in every thread, always in the same order
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[kThreads / 64];
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = x;
  __syncthreads();
  double s = part[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) s += part[w];
  __syncthreads();
  return s;
}

// n elements at p by the workgroup, 16 bytes an access: f(first element,
// values).  A full chunk is unrolled, all its loads in flight at once; a tail
// goes element by element.
template <class T, bool NT, class F>
__device__ __forceinline__ void for_vectors(const T* p, int n, F f) {
  constexpr int VEC = 16 / sizeof(T), kStep = kThreads * VEC;
  if (n == kChunk) {
    float x[kChunk / kStep][VEC];
#pragma unroll
    for (int k = 0; k < kChunk / kStep; ++k)
      if (NT) g2v::load_vec_nt<T, VEC>(p + k * kStep + threadIdx.x * VEC, x[k]);
      else g2v::load_vec<T, VEC>(p + k * kStep + threadIdx.x * VEC, x[k]);
#pragma unroll
    for (int k = 0; k < kChunk / kStep; ++k) f(k * kStep + threadIdx.x * VEC, x[k]);
    return;
  }
  int i = threadIdx.x * VEC;
  for (; i + VEC <= n; i += kStep) {
    float x[VEC];
    g2v::load_vec<T, VEC>(p + i, x);
    f(i, x);
  }
  for (int e = i; e < n && e < i + VEC; ++e) {
    float x[1] = {(float)p[e]};
    f(e, x);
  }
}

// f(tensor, first element, values) for this workgroup's share of the chunks
template <bool NT, class A, class F>
__device__ __forceinline__ void for_elements(const A& a, F f) {
  const int64_t chunks = a.first[a.n];
  const int c0 = (int)(chunks * blockIdx.x / gridDim.x);
  const int c1 = (int)(chunks * (blockIdx.x + 1) / gridDim.x);
  int lo = 0, hi = a.n;  // the tensor of chunk c0: first[lo] <= c0 < first[lo + 1]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (a.first[m] <= c0) lo = m;
    else hi = m;
  }
  for (int c = c0, t = lo; c < c1; ++t) {
    const int t0 = a.first[t], t1 = a.first[t + 1] < c1 ? a.first[t + 1] : c1;
    const int64_t numel = a.numel[t];
    by_type_dev(a.type[t], [&](auto z) {
      using T = decltype(z);
      const T* p = static_cast<const T*>(a.src[t]);
      const int head = (int)head_of(p, numel, sizeof(T));
      if (c == t0 && (int)threadIdx.x < head) {
        float x[1] = {(float)p[threadIdx.x]};
        f(t, z, (int64_t)threadIdx.x, x);
      }
      for (; c < t1; ++c) {
        const int64_t e = head + (int64_t)(c - t0) * kChunk, left = numel - e;
        for_vectors<T, NT>(p + e, (int)(left < kChunk ? left : kChunk),
                           [&](int i, auto& x) { f(t, z, e + i, x); });
      }
    });
  }
}

template <bool NT, class A>
__global__ __launch_bounds__(kThreads, kWaves) void k_square_sum(A a, double* __restrict__ partial) {
  double s0 = 0.0, s1 = 0.0;
  for_elements<NT>(a, [&](int, auto, int64_t, auto& x) {
    constexpr int N = sizeof x / sizeof x[0];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double d = (double)x[i];
      if (i & 1) s1 = fma(d, d, s1);
      else s0 = fma(d, d, s0);
    }
  });
  const double s = block_sum(s0 + s1);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double sum_partials(const double* __restrict__ partial, int np) {
  double s = 0.0;
  for (int i = threadIdx.x; i < np; i += kThreads) s += partial[i];
  return block_sum(s);
}

__global__ __launch_bounds__(kThreads) void k_norm(const double* __restrict__ partial, int np,
                                                   float* __restrict__ norm) {
  const double s = sum_partials(partial, np);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// Every workgroup adds the partial sums for itself (the same order, the same
// factor everywhere): 16 KB from the L2 instead of a launch in between.  What
// is read here for the last time and what is written go past the caches, and
// the norm's pass leaves them the gradients: of 400 MB fp32 clipped to another
// buffer 190 us, 243 with ordinary accesses, 211 with the norm's pass past them.
template <class A>
__global__ __launch_bounds__(kThreads, kWaves) void k_clip(A a, const double* __restrict__ partial, int np,
                                                   double clip, bool in_place,
                                                   float* __restrict__ norm) {
  const double nrm = sqrt(sum_partials(partial, np));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nrm;
  const double factor = nrm < INFINITY ? clip / (nrm > clip ? nrm : clip) : NAN;
  // a factor below fp32's normal numbers (a norm 10^38 times the bound) would keep
  // few of its bits there: its exponent is applied apart, after the product
  int e = 0;
  const float f = (float)(factor < 0x1p-126 ? frexp(factor, &e) : factor);
  if (in_place && f == 1.f && e == 0) return;  // within the bound
  for_elements<true>(a, [&](int t, auto z, int64_t at, auto& x) {
    using T = decltype(z);
    constexpr int N = sizeof x / sizeof x[0];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = ldexpf(x[i] * f, e);
    g2v::store_vec_nt<T, N>(static_cast<T*>(a.dst[t]) + at, x);
  });
}

struct Range {
  uintptr_t a, b;
  int64_t t;
  bool operator<(const Range& o) const { return a < o.a; }
};

int check_list(const char* what, int device, const void* const* src, const int64_t* numel,
               const int32_t* types, int64_t n, const void* norm, const void* ws,
               int64_t ws_bytes) {
  OP_REQUIRE(device >= 0, G2V_EINVAL, "%s: device %d", what, device);
  OP_REQUIRE(n >= 0 && (n == 0 || (src && numel && types)), G2V_EINVAL, "%s: null list", what);
  OP_REQUIRE(norm && (uintptr_t)norm % 4 == 0, G2V_EINVAL, "%s: norm is null or not aligned", what);
  int64_t need = 0;
  const int rc = g2v_global_norm_workspace(n, &need);
  if (rc != G2V_OK) return rc;
  OP_REQUIRE(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, G2V_EINVAL,
             "%s: a 16-byte aligned workspace of %lld bytes is needed (got %lld)", what,
             (long long)need, (long long)ws_bytes);
  int64_t chunks = 0;
  for (int64_t t = 0; t < n; ++t) {
    const int64_t b = g2v::type_bytes(types[t]);
    OP_REQUIRE(b != 0, G2V_EINVAL, "%s: tensor %lld has the unknown type %d", what, (long long)t,
               (int)types[t]);
    OP_REQUIRE(numel[t] >= 0 && numel[t] <= (int64_t)1 << 40, G2V_ERANGE,
               "%s: tensor %lld has %lld elements (at most 2^40)", what, (long long)t,
               (long long)numel[t]);
    OP_REQUIRE(numel[t] == 0 || (src[t] && (uintptr_t)src[t] % b == 0), G2V_EINVAL,
               "%s: tensor %lld is null or not aligned to its type", what, (long long)t);
    chunks += chunks_of(src[t], numel[t], types[t]);
    OP_REQUIRE(chunks <= INT32_MAX, G2V_ERANGE, "%s: more than 2^44 elements in all", what);
  }
  return G2V_OK;
}

// no element is written twice, and none is written that another tensor reads
int check_apart(const char* what, const void* const* src, void* const* dst, const int64_t* numel,
                const int32_t* types, int64_t n) {
  std::vector<Range> r;
  r.reserve((size_t)n);
  for (int64_t t = 0; t < n; ++t) {
    const int64_t b = g2v::type_bytes(types[t]);
    if (numel[t] == 0) continue;
    OP_REQUIRE(dst[t] && (uintptr_t)dst[t] % b == 0, G2V_EINVAL,
               "%s: output %lld is null or not aligned to its type", what, (long long)t);
    r.push_back({(uintptr_t)dst[t], (uintptr_t)dst[t] + (uintptr_t)(numel[t] * b), t});
  }
  std::sort(r.begin(), r.end());
  for (size_t k = 1; k < r.size(); ++k)
    OP_REQUIRE(r[k].a >= r[k - 1].b, G2V_EINVAL, "%s: outputs %lld and %lld overlap", what,
               (long long)r[k - 1].t, (long long)r[k].t);
  for (int64_t t = 0; t < n; ++t) {
    if (numel[t] == 0) continue;
    const uintptr_t a = (uintptr_t)src[t],
                    b = a + (uintptr_t)(numel[t] * g2v::type_bytes(types[t]));
    // the outputs are apart and in order: those that meet [a, b) follow the
    // last one that begins at or before a
    size_t k = (size_t)(std::upper_bound(r.begin(), r.end(), Range{a, 0, 0}) - r.begin());
    for (k = k ? k - 1 : 0; k < r.size() && r[k].a < b; ++k) {
      if (r[k].b <= a) continue;
      OP_REQUIRE(r[k].t == t && r[k].a == a, G2V_EINVAL,
                 "%s: output %lld overlaps input %lld (in place means the same address)", what,
                 (long long)r[k].t, (long long)t);
    }
  }
  return G2V_OK;
}

// where the parts of the workspace lie: partial sums, then the list where it
// does not fit the kernel arguments
struct Plan {
  int64_t src, dst, numel, first, type, bytes;
};

Plan plan(int64_t n) {
  Plan p{};
  const auto take = [&](int64_t count, int64_t size) {
    const int64_t o = p.bytes;
    p.bytes += (count * size + 15) / 16 * 16;
    return o;
  };
  take(kMaxPartials, sizeof(double));
  const int64_t k = n > kTensors ? n : 0;
  p.src = take(k, 8);
  p.dst = take(k, 8);
  p.numel = take(k, 8);
  p.first = take(k + 1, 4);
  p.type = take(k, 1);
  return p;
}

// f(the list as a kernel takes it, workgroups), once; not at all for a list
// that holds no element
template <class F>
int with_tensors(const void* const* src, void* const* dst, const int64_t* numel,
                 const int32_t* types, int64_t n, char* ws, hipStream_t st, F f) {
  int64_t full = 0;
  for (int64_t t = 0; t < n; ++t) full += numel[t] > 0;
  if (full == 0) return G2V_OK;
  const Plan p = plan(n);
  const TensorList list{reinterpret_cast<const void**>(ws + p.src),
                        reinterpret_cast<void**>(ws + p.dst),
                        reinterpret_cast<int64_t*>(ws + p.numel),
                        reinterpret_cast<int32_t*>(ws + p.first),
                        reinterpret_cast<int8_t*>(ws + p.type), (int32_t)full};
  Tensors a;
  a.n = 0;
  a.first[0] = 0;
  int64_t listed = 0, chunks = 0;
  for (int64_t t = 0; t < n; ++t) {
    if (numel[t] == 0) continue;
    a.src[a.n] = src[t];
    a.dst[a.n] = dst ? dst[t] : nullptr;
    a.numel[a.n] = numel[t];
    a.type[a.n] = (int8_t)types[t];
    a.first[a.n + 1] = a.first[a.n] + (int32_t)chunks_of(src[t], numel[t], types[t]);
    ++a.n;
    if (full > kTensors && (a.n == kTensors || listed + a.n == full)) {
      hipLaunchKernelGGL(k_list, dim3(1), dim3(kTensors), 0, st, a, list, (int)listed, (int)chunks);
      OP_HIP(hipGetLastError(), "g2v_global_norm");
      listed += a.n;
      chunks += a.first[a.n];
      a.n = 0;
    }
  }
  if (full <= kTensors) chunks = a.first[a.n];
  const unsigned g = (unsigned)(chunks < kMaxPartials ? chunks : kMaxPartials);
  if (full <= kTensors) f(a, g);
  else f(list, g);
  OP_HIP(hipGetLastError(), "g2v_global_norm");
  return G2V_OK;
}

}  // namespace

extern "C" int g2v_global_norm_workspace(int64_t n, int64_t* bytes) {
  OP_REQUIRE(bytes && n >= 0, G2V_EINVAL, "g2v_global_norm_workspace: bad arguments");
  OP_REQUIRE(n <= INT32_MAX, G2V_ERANGE, "g2v_global_norm_workspace: %lld tensors", (long long)n);
  *bytes = plan(n).bytes;
  return G2V_OK;
}

extern "C" int g2v_global_norm(int device, const void* const* tensors, const int64_t* numel,
                               const int32_t* types, int64_t n, float* norm, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  const char* what = "g2v_global_norm";
  int rc = check_list(what, device, tensors, numel, types, n, norm, workspace, workspace_bytes);
  if (rc != G2V_OK) return rc;
  g2v::DeviceScope scope(device);
  OP_HIP(scope.error(), what);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  // beyond the Infinity Cache's 256 MB nothing stays for the next reader, and
  // loads past the caches are faster (1 GB of fp32: 149 us against 170, 400 MB 63
  // against 72); what fits may still lie there (250 MB: 41.5 us against 40)
  double bytes = 0.0;
  for (int64_t t = 0; t < n; ++t) bytes += (double)(numel[t] * g2v::type_bytes(types[t]));
  const bool large = bytes > 256e6;
  int np = 0;
  rc = with_tensors(tensors, nullptr, numel, types, n, static_cast<char*>(workspace), st,
                    [&](const auto& a, unsigned g) {
                      using A = std::decay_t<decltype(a)>;
                      hipLaunchKernelGGL((large ? k_square_sum<true, A> : k_square_sum<false, A>),
                                         dim3(g), dim3(kThreads), 0, st, a, partial);
                      np = (int)g;
                    });
  if (rc != G2V_OK) return rc;
  hipLaunchKernelGGL(k_norm, dim3(1), dim3(kThreads), 0, st, partial, np, norm);
  OP_HIP(hipGetLastError(), what);
  return G2V_OK;
}

extern "C" int g2v_clip_global_norm(int device, const void* const* src, void* const* dst,
                                    const int64_t* numel, const int32_t* types, int64_t n,
                                    double clip_norm, float* norm, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  const char* what = "g2v_clip_global_norm";
  int rc = check_list(what, device, src, numel, types, n, norm, workspace, workspace_bytes);
  if (rc != G2V_OK) return rc;
  OP_REQUIRE(n == 0 || dst, G2V_EINVAL, "%s: null list", what);
  OP_REQUIRE(clip_norm > 0 && clip_norm < INFINITY, G2V_EINVAL,
             "%s: clip_norm must be positive and finite (got %g)", what, clip_norm);
  try {
    rc = check_apart(what, src, dst, numel, types, n);
  } catch (...) {
    return g2v::op_fail(G2V_ENOMEM, "%s: no host memory for %lld tensors", what, (long long)n);
  }
  if (rc != G2V_OK) return rc;
  bool in_place = true;
  for (int64_t t = 0; t < n; ++t) in_place = in_place && (numel[t] == 0 || src[t] == dst[t]);
  g2v::DeviceScope scope(device);
  OP_HIP(scope.error(), what);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  bool any = false;
  rc = with_tensors(src, dst, numel, types, n, static_cast<char*>(workspace), st,
                    [&](const auto& a, unsigned g) {
                      using A = std::decay_t<decltype(a)>;
                      hipLaunchKernelGGL((k_square_sum<false, A>), dim3(g), dim3(kThreads), 0, st,
                                         a, partial);
                      hipLaunchKernelGGL(k_clip<A>, dim3(g), dim3(kThreads), 0, st, a, partial,
                                         (int)g, clip_norm, in_place, norm);
                      any = true;
                    });
  if (rc != G2V_OK || any) return rc;
  // nothing to clip: the norm of nothing is 0
  hipLaunchKernelGGL(k_norm, dim3(1), dim3(kThreads), 0, st, partial, 0, norm);
  OP_HIP(hipGetLastError(), what);
  return G2V_OK;
}
