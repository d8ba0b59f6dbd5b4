// g2v_embed.hip -- embedding lookup with scaling, and its gradient.
//
//   y[i]  = scale * W[ids[i]]                       (zero row: ids[i] not in [0, V))
//   dW[v] = scale * sum over i with ids[i] == v of dy[i], added in token order
//
// GGIPNN's lookup (src/GGIPNN.py:19-25, tf.nn.embedding_lookup) and, for
// train_embedding=True there, the gradient of its table.
#include <type_traits>

#include "g2v_ops.h"

namespace {

using g2v::bf16;
using g2v::f16;

constexpr int kThreads = 256;

constexpr int kUnits = 4;  // vectors a thread of the lookup moves

// The elements of a vector: 16 bytes of the narrower of the two types.  A row
// of D elements is ceil(D / VEC) vectors; the last one ends with the row and
// overlaps the one before where VEC does not divide D (the same values are
// written twice), so that no width needs a scalar tail.  Rows narrower than a
// vector go element by element.
template <class A, class B>
constexpr int vec_of() {
  return 16 / (sizeof(A) < sizeof(B) ? sizeof(A) : sizeof(B));
}

// Memory bound: a row read and a row written per token, no reuse.  Vectors of
// all rows are numbered through and dealt out 1024 to a workgroup, so every
// width fills the lanes and one row is spread over as many threads as it has
// vectors; kUnits independent id -> row chains per thread cover the latency.
template <class TW, class TY, class I, int VEC>
__global__ __launch_bounds__(kThreads) void k_embed_lookup(
    const TW* __restrict__ W, int64_t V, int D, int64_t ld, const I* __restrict__ ids,
    int64_t units, int nv, float scale, TY* __restrict__ out) {
  const int64_t u0 = (int64_t)blockIdx.x * (kThreads * kUnits);
  const int64_t row0 = u0 / nv;
  const uint32_t r0 = (uint32_t)(u0 - row0 * nv) + threadIdx.x;  // < nv + 1024
  const int64_t left = units - u0;
  int64_t id[kUnits], at[kUnits];
  int col[kUnits];
  float x[kUnits][VEC];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const uint32_t l = r0 + k * kThreads, q = l / (uint32_t)nv;
    const int c = (int)(l - q * nv) * VEC;
    col[k] = c + VEC <= D ? c : D - VEC;
    at[k] = row0 + q;
    id[k] = (int)threadIdx.x + k * kThreads < left ? (int64_t)ids[at[k]] : -1;
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[k][i] = 0.f;
    if (id[k] >= 0 && id[k] < V) {
      g2v::load_vec<TW, VEC>(W + id[k] * ld + col[k], x[k]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[k][i] *= scale;
    }
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k)
    if ((int)threadIdx.x + k * kThreads < left)
      g2v::store_vec<TY, VEC>(out + at[k] * D + col[k], x[k]);
}

// one wave per row and 64 columns: the ids in order, 64 at a time, and the
// rows of dy whose id is this one
template <class TY, class TG, class I>
__global__ __launch_bounds__(kThreads) void k_embed_grad_direct(
    const TY* __restrict__ dy, int64_t dy_ld, const I* __restrict__ ids, int64_t n, int64_t V,
    int64_t D, float scale, int64_t pad, TG* __restrict__ grad) {
  const int lane = threadIdx.x & 63;
  const int64_t tiles = (D + 63) / 64, items = V * tiles;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t it = (int64_t)blockIdx.x * (kThreads / 64) + threadIdx.x / 64; it < items;
       it += step) {
    const int64_t v = it / tiles, col = (it - v * tiles) * 64 + lane;
    float acc = 0.f;
    if (v != pad) {
      for (int64_t b = 0; b < n; b += 64) {
        uint64_t m = __ballot(b + lane < n && (int64_t)ids[b + lane < n ? b + lane : 0] == v);
        while (m) {
          const int64_t i = b + __builtin_ctzll(m);
          m &= m - 1;
          if (col < D) acc += (float)dy[i * dy_ld + col];
        }
      }
    }
    if (col < D) grad[v * D + col] = (TG)(acc * scale);
  }
}

template <class F>
int by_type(int type, F f) {
  switch (type) {
    case G2V_F32: return f(float{});
    case G2V_F16: return f(f16{});
    default: return f(bf16{});
  }
}

template <class F>
int by_id(int id_bytes, F f) {
  return id_bytes == 4 ? f(int32_t{}) : f(int64_t{});
}

int check_common(const char* what, int device, int64_t V, int64_t D, const void* ids,
                 int id_bytes, int64_t n) {
  OP_REQUIRE(device >= 0, G2V_EINVAL, "%s: device %d", what, device);
  OP_REQUIRE(V >= 1 && D >= 1 && n >= 0, G2V_EINVAL, "%s: V = %lld, D = %lld, n = %lld", what,
             (long long)V, (long long)D, (long long)n);
  OP_REQUIRE(V <= INT32_MAX && n <= INT32_MAX && D <= G2V_EMBED_MAX_DIM, G2V_ERANGE,
             "%s: V = %lld and n = %lld are at most 2^31 - 1, D = %lld at most %d", what,
             (long long)V, (long long)n, (long long)D, G2V_EMBED_MAX_DIM);
  OP_REQUIRE(id_bytes == 4 || id_bytes == 8, G2V_EINVAL, "%s: ids of %d bytes", what, id_bytes);
  OP_REQUIRE(n == 0 || (ids && (uintptr_t)ids % id_bytes == 0), G2V_EINVAL,
             "%s: ids are null or not aligned to their size", what);
  return G2V_OK;
}

int check_matrix(const char* what, const char* name, const void* p, int type, int64_t rows,
                 int64_t ld, int64_t D) {
  OP_REQUIRE(g2v::type_bytes(type) != 0, G2V_EINVAL, "%s: %s has the unknown type %d", what, name,
             type);
  OP_REQUIRE(rows == 0 || (p && (uintptr_t)p % g2v::type_bytes(type) == 0), G2V_EINVAL,
             "%s: %s is null or not aligned to its type", what, name);
  OP_REQUIRE(ld >= D, G2V_EINVAL, "%s: %s has rows of %lld elements every %lld", what, name,
             (long long)D, (long long)ld);
  OP_REQUIRE(ld <= (INT64_MAX / 4) / (rows > 1 ? rows : 1), G2V_ERANGE,
             "%s: %s spans more than 2^63 bytes", what, name);
  return G2V_OK;
}

unsigned grid_for(int64_t items, int64_t per_block) {
  const int64_t g = (items + per_block - 1) / per_block;
  return (unsigned)(g < 1 ? 1 : g > 8192 ? 8192 : g);
}

}  // namespace

extern "C" int g2v_embed_lookup(int device, const void* table, int table_type, int64_t V,
                                int64_t D, int64_t ld, const void* ids, int id_bytes, int64_t n,
                                float scale, void* out, int out_type, void* stream) {
  const char* what = "g2v_embed_lookup";
  int rc = check_common(what, device, V, D, ids, id_bytes, n);
  if (rc == G2V_OK) rc = check_matrix(what, "table", table, table_type, V, ld, D);
  if (rc == G2V_OK) rc = check_matrix(what, "out", out, out_type, n, D, D);
  if (rc != G2V_OK || n == 0) return rc;
  g2v::DeviceScope scope(device);
  OP_HIP(scope.error(), what);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  rc = by_type(table_type, [&](auto w) {
    return by_type(out_type, [&](auto y) {
      return by_id(id_bytes, [&](auto i) {
        using TW = decltype(w);
        using TY = decltype(y);
        using I = decltype(i);
        constexpr int VEC = vec_of<TW, TY>();
        const int64_t nv = D >= VEC ? (D + VEC - 1) / VEC : D;
        const int64_t blocks = (n * nv + kThreads * kUnits - 1) / (kThreads * kUnits);
        // a launch is limited to 2^32 threads
        OP_REQUIRE(blocks < (int64_t)1 << 24, G2V_ERANGE, "%s: %lld x %lld elements in one call",
                   what, (long long)n, (long long)D);
        hipLaunchKernelGGL((D >= VEC ? k_embed_lookup<TW, TY, I, VEC> : k_embed_lookup<TW, TY, I, 1>),
                           dim3((unsigned)blocks), dim3(kThreads), 0, st,
                           static_cast<const TW*>(table), V, (int)D, ld,
                           static_cast<const I*>(ids), n * nv, (int)nv, scale,
                           static_cast<TY*>(out));
        return (int)G2V_OK;
      });
    });
  });
  if (rc != G2V_OK) return rc;
  OP_HIP(hipGetLastError(), what);
  return G2V_OK;
}

extern "C" int g2v_embed_grad_workspace(int64_t n, int64_t V, int64_t D, int64_t* bytes) {
  const char* what = "g2v_embed_grad_workspace";
  OP_REQUIRE(bytes, G2V_EINVAL, "%s: null output", what);
  *bytes = 0;
  const int rc = check_common(what, 0, V, D, nullptr, 4, 0);
  if (rc != G2V_OK) return rc;
  OP_REQUIRE(n >= 0 && n <= INT32_MAX, G2V_ERANGE, "%s: n = %lld", what, (long long)n);
  return G2V_OK;
}

extern "C" int g2v_embed_grad(int device, const void* dy, int dy_type, int64_t dy_ld,
                              const void* ids, int id_bytes, int64_t n, int64_t V, int64_t D,
                              float scale, int64_t padding_id, void* grad, int grad_type,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "g2v_embed_grad";
  int rc = check_common(what, device, V, D, ids, id_bytes, n);
  if (rc == G2V_OK) rc = check_matrix(what, "dy", dy, dy_type, n, dy_ld, D);
  if (rc == G2V_OK) rc = check_matrix(what, "grad", grad, grad_type, V, D, D);
  if (rc != G2V_OK) return rc;
  OP_REQUIRE(padding_id >= -1 && padding_id < V, G2V_EINVAL, "%s: padding id %lld outside [-1, %lld)",
             what, (long long)padding_id, (long long)V);
  int64_t need = 0;
  rc = g2v_embed_grad_workspace(n, V, D, &need);
  if (rc != G2V_OK) return rc;
  OP_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 16 == 0)),
             G2V_EINVAL, "%s: a 16-byte aligned workspace of %lld bytes is needed (got %lld)", what,
             (long long)need, (long long)workspace_bytes);
  g2v::DeviceScope scope(device);
  OP_HIP(scope.error(), what);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dy_type, [&](auto y) {
    return by_type(grad_type, [&](auto g) {
      return by_id(id_bytes, [&](auto i) {
        using TY = decltype(y);
        using TG = decltype(g);
        using I = decltype(i);
        hipLaunchKernelGGL((k_embed_grad_direct<TY, TG, I>),
                           dim3(grid_for(V * ((D + 63) / 64), kThreads / 64)), dim3(kThreads), 0,
                           st, static_cast<const TY*>(dy), dy_ld, static_cast<const I*>(ids), n, V,
                           D, scale, padding_id, static_cast<TG*>(grad));
        return 0;
      });
    });
  });
  OP_HIP(hipGetLastError(), what);
  return G2V_OK;
}
