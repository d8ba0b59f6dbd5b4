// g2v_ops.h -- what the tensor operators (g2v_embed.hip, g2v_gradnorm.hip)
// share: element types, vector access at element alignment, argument checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <type_traits>

#include "g2v.h"
#include "g2v_internal.h"

namespace g2v {

using f16 = _Float16;
using bf16 = __bf16;

// VEC elements at the alignment of one element.  gfx950 serves a 16-byte
// global access at any element address, so rows of odd width keep full-width
// accesses and no kernel needs a second path for them.
template <class T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[VEC]) {
  T t[VEC];
  __builtin_memcpy(t, p, sizeof t);
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = (float)t[i];
}

// one rounding, to nearest even, from fp32 to the type stored
template <class T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[VEC]) {
  T t[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) t[i] = (T)x[i];
  __builtin_memcpy(p, t, sizeof t);
}

typedef uint32_t word4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t word4_at4 __attribute__((ext_vector_type(4), aligned(4)));

// the same, past the caches: for results larger than they hold
template <class T, int VEC>
__device__ __forceinline__ void store_vec_nt(T* p, const float (&x)[VEC]) {
  if constexpr (sizeof(T) * VEC % 16 == 0) {
    using word4 = std::conditional_t<sizeof(T) == 2, word4_at2, word4_at4>;
    T t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = (T)x[i];
    word4 w[sizeof(T) * VEC / 16];
    __builtin_memcpy(w, t, sizeof t);
#pragma unroll
    for (unsigned k = 0; k < sizeof(T) * VEC / 16; ++k)
      __builtin_nontemporal_store(w[k], reinterpret_cast<word4*>(p) + k);
  } else {
    store_vec<T, VEC>(p, x);
  }
}

template <class T, int VEC>
__device__ __forceinline__ void load_vec_nt(const T* p, float (&x)[VEC]) {
  if constexpr (sizeof(T) * VEC % 16 == 0) {
    using word4 = std::conditional_t<sizeof(T) == 2, word4_at2, word4_at4>;
    word4 w[sizeof(T) * VEC / 16];
#pragma unroll
    for (unsigned k = 0; k < sizeof(T) * VEC / 16; ++k)
      w[k] = __builtin_nontemporal_load(reinterpret_cast<const word4*>(p) + k);
    T t[VEC];
    __builtin_memcpy(t, w, sizeof t);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = (float)t[i];
  } else {
    load_vec<T, VEC>(p, x);
  }
}

inline int64_t type_bytes(int type) {
  return type == G2V_F32 ? 4 : type == G2V_F16 || type == G2V_BF16 ? 2 : 0;
}

inline int op_fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  try {
    return set_error(code, buf);
  } catch (...) {  // no memory for the message: the code alone
    return code;
  }
}

// the caller's current device is the same after the call
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    err_ = hipGetDevice(&old_);
    if (err_ == hipSuccess && old_ != device) {
      err_ = hipSetDevice(device);
      moved_ = err_ == hipSuccess;
    }
  }
  ~DeviceScope() {
    if (moved_) (void)hipSetDevice(old_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  hipError_t error() const { return err_; }

 private:
  int old_ = 0;
  bool moved_ = false;
  hipError_t err_ = hipSuccess;
};

}  // namespace g2v

#define OP_REQUIRE(cond, code, ...)                       \
  do {                                                    \
    if (!(cond)) return g2v::op_fail((code), __VA_ARGS__); \
  } while (0)

#define OP_HIP(x, what)                                                             \
  do {                                                                              \
    hipError_t e_ = (x);                                                            \
    if (e_ != hipSuccess)                                                           \
      return g2v::op_fail(G2V_EHIP, "%s: %s", (what), hipGetErrorString(e_));       \
  } while (0)
