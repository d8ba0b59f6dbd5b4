// g2v_gradnorm.hip -- the global norm of a list of gradients, and clipping.
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   clip: dst = g * (clip / max(norm, clip)); NaN everywhere when the norm is
//         not finite (tf.clip_by_global_norm's rule: an overflow is not hidden)
//
// The squares are formed and added in fp64: an fp32 sum would overflow from
// elements of 1.8e19 on and lose the small tensors beside the large ones, and
// the fp64 rate of gfx950 equals its fp32 rate per lane, far above what the
// memory delivers.  No atomics: every workgroup writes one partial sum, and
// they are added in a fixed order, so the same gradients give the same bits.
//
// The tensors' addresses travel in the kernel arguments, kTensors a launch: no
// copy to the device, nothing that a captured graph would have to keep alive.
#include <algorithm>
#include <vector>

#include "g2v_ops.h"

namespace {

using g2v::bf16;
using g2v::f16;

constexpr int kThreads = 256;
constexpr int kTensors = 128;      // per launch: 3.6 KB of arguments
constexpr int kMaxPartials = 2048; // workgroups of all launches, less one a launch
constexpr int64_t kChunk = 8192;   // elements a workgroup takes at a time

struct Tensors {
  const void* src[kTensors];
  void* dst[kTensors];
  int64_t numel[kTensors];
  int32_t first[kTensors + 1];  // chunks before tensor t
  int8_t type[kTensors];
  int32_t n;
};

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

// calls f(tensor, first element, elements) for the chunks [c0, c1)
template <class F>
__device__ __forceinline__ void for_chunks(const Tensors& a, int c0, int c1, F f) {
  int lo = 0, hi = a.n;  // the tensor of chunk c0: first[lo] <= c0 < first[lo + 1]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (a.first[m] <= c0) lo = m;
    else hi = m;
  }
  for (int c = c0, t = lo; c < c1; ++c) {
    while (c >= a.first[t + 1]) ++t;
    const int64_t e = (int64_t)(c - a.first[t]) * kChunk;
    const int64_t left = a.numel[t] - e;
    f(t, e, (int)(left < kChunk ? left : kChunk));
  }
}

__device__ __forceinline__ void my_chunks(const Tensors& a, int& c0, int& c1) {
  const int64_t chunks = a.first[a.n];
  c0 = (int)(chunks * blockIdx.x / gridDim.x);
  c1 = (int)(chunks * (blockIdx.x + 1) / gridDim.x);
}

// x[0 .. n) of p by the workgroup's threads, 16 bytes an access; f(first
// element, values, their number).  A full chunk is unrolled: all its loads are
// in flight at once.  The tail goes element by element.
template <class T, class F>
__device__ __forceinline__ void for_vectors(const T* p, int n, F f) {
  constexpr int VEC = 16 / sizeof(T), kStep = kThreads * VEC;
  if (n == kChunk) {
    float x[kChunk / kStep][VEC];
#pragma unroll
    for (int k = 0; k < kChunk / kStep; ++k)
      g2v::load_vec<T, VEC>(p + k * kStep + threadIdx.x * VEC, x[k]);
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

__global__ __launch_bounds__(kThreads) void k_square_sum(Tensors a, double* __restrict__ partial) {
  int c0, c1;
  my_chunks(a, c0, c1);
  double s0 = 0.0, s1 = 0.0;
  for_chunks(a, c0, c1, [&](int t, int64_t e, int n) {
    by_type_dev(a.type[t], [&](auto z) {
      using T = decltype(z);
      for_vectors(static_cast<const T*>(a.src[t]) + e, n, [&](int, auto& x) {
        constexpr int N = sizeof x / sizeof x[0];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const double d = (double)x[i];
          if (i & 1) s1 = fma(d, d, s1);
          else s0 = fma(d, d, s0);
        }
      });
    });
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

// every workgroup adds the partial sums for itself (the same order, the same
// factor everywhere): 16 KB from the L2 instead of a launch in between
__global__ __launch_bounds__(kThreads) void k_clip(Tensors a, const double* __restrict__ partial,
                                                   int np, double clip, float* __restrict__ norm) {
  const double nrm = sqrt(sum_partials(partial, np));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nrm;
  const float f = (float)(nrm < INFINITY ? clip / (nrm > clip ? nrm : clip) : NAN);
  int c0, c1;
  my_chunks(a, c0, c1);
  for_chunks(a, c0, c1, [&](int t, int64_t e, int n) {
    if (f == 1.f && a.src[t] == a.dst[t]) return;  // in place and within the bound
    by_type_dev(a.type[t], [&](auto z) {
      using T = decltype(z);
      T* q = static_cast<T*>(a.dst[t]) + e;
      for_vectors(static_cast<const T*>(a.src[t]) + e, n, [&](int at, auto& x) {
        constexpr int N = sizeof x / sizeof x[0];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= f;
        g2v::store_vec<T, N>(q + at, x);
      });
    });
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
    chunks += (numel[t] + kChunk - 1) / kChunk;
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

// f(arguments, workgroups, is it the first) for every kTensors tensors that
// hold something; the workgroups of all calls are at most kMaxPartials + calls
template <class F>
int for_launches(const void* const* src, void* const* dst, const int64_t* numel,
                 const int32_t* types, int64_t n, F f) {
  int64_t total = 0;
  for (int64_t t = 0; t < n; ++t) total += (numel[t] + kChunk - 1) / kChunk;
  bool first = true;
  Tensors a;
  a.n = 0;
  a.first[0] = 0;
  for (int64_t t = 0; t < n; ++t) {
    if (numel[t] > 0) {
      a.src[a.n] = src[t];
      a.dst[a.n] = dst ? dst[t] : nullptr;
      a.numel[a.n] = numel[t];
      a.type[a.n] = (int8_t)types[t];
      a.first[a.n + 1] = a.first[a.n] + (int32_t)((numel[t] + kChunk - 1) / kChunk);
      ++a.n;
    }
    if (a.n == kTensors || (t == n - 1 && a.n > 0)) {
      const int64_t c = a.first[a.n];
      const int64_t g = total <= kMaxPartials ? c : (c * kMaxPartials + total - 1) / total;
      f(a, (unsigned)g, first);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return g2v::op_fail(G2V_EHIP, "launch: %s", hipGetErrorString(e));
      first = false;
      a.n = 0;
    }
  }
  return G2V_OK;
}

int square_sums(const void* const* src, const int64_t* numel, const int32_t* types, int64_t n,
                double* partial, int* np, hipStream_t st) {
  int used = 0;
  const int rc = for_launches(src, nullptr, numel, types, n,
                              [&](const Tensors& a, unsigned g, bool) {
                                hipLaunchKernelGGL(k_square_sum, dim3(g), dim3(kThreads), 0, st, a,
                                                   partial + used);
                                used += (int)g;
                              });
  *np = used;
  return rc;
}

}  // namespace

extern "C" int g2v_global_norm_workspace(int64_t n, int64_t* bytes) {
  OP_REQUIRE(bytes && n >= 0, G2V_EINVAL, "g2v_global_norm_workspace: bad arguments");
  *bytes = (int64_t)sizeof(double) * (kMaxPartials + 1 + n / kTensors + 1);
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
  int np = 0;
  rc = square_sums(tensors, numel, types, n, partial, &np, st);
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
  g2v::DeviceScope scope(device);
  OP_HIP(scope.error(), what);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  int np = 0;
  rc = square_sums(src, numel, types, n, partial, &np, st);
  if (rc != G2V_OK) return rc;
  if (np == 0) {  // nothing to clip: the norm of nothing is 0
    hipLaunchKernelGGL(k_norm, dim3(1), dim3(kThreads), 0, st, partial, 0, norm);
    OP_HIP(hipGetLastError(), what);
    return G2V_OK;
  }
  return for_launches(src, dst, numel, types, n, [&](const Tensors& a, unsigned g, bool first) {
    hipLaunchKernelGGL(k_clip, dim3(g), dim3(kThreads), 0, st, a, partial, np, clip_norm,
                       first ? norm : nullptr);
  });
}
