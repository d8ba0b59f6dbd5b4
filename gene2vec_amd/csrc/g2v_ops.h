// g2v_ops.h -- what the tensor operators (g2v_embed.hip, g2v_gradnorm.hip)
// share: element types, vector access at element alignment, argument checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

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

// words of an access past the caches, at the alignment of an element
template <int ALIGN, int BYTES>
struct Words;
#define G2V_WORDS(ALIGN, BYTES)                                                              \
  template <>                                                                                \
  struct Words<ALIGN, BYTES> {                                                               \
    typedef uint32_t type                                                                    \
        __attribute__((ext_vector_type(BYTES / 4), aligned(ALIGN), may_alias));              \
  };
G2V_WORDS(2, 8) G2V_WORDS(2, 16) G2V_WORDS(4, 8) G2V_WORDS(4, 16)
#undef G2V_WORDS

// how vectors of N bytes are split: 16 bytes an access, 8 where there are no
// more; 0: single elements take ordinary accesses
template <int N>
constexpr int access_bytes() {
  return N % 16 == 0 ? 16 : N % 8 == 0 ? 8 : 0;
}

// the same past the caches, for what is not read again soon
template <class T, int VEC>
__device__ __forceinline__ void store_vec_nt(T* p, const float (&x)[VEC]) {
  constexpr int A = access_bytes<sizeof(T) * VEC>();
  if constexpr (A != 0) {
    using W = typename Words<sizeof(T), A>::type;
    T t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = (T)x[i];
    W w[sizeof t / A];
    __builtin_memcpy(w, t, sizeof t);
#pragma unroll
    for (unsigned k = 0; k < sizeof t / A; ++k)
      __builtin_nontemporal_store(w[k], reinterpret_cast<W*>(p) + k);
  } else {
    store_vec<T, VEC>(p, x);
  }
}

template <class T, int VEC>
__device__ __forceinline__ void load_vec_nt(const T* p, float (&x)[VEC]) {
  constexpr int A = access_bytes<sizeof(T) * VEC>();
  if constexpr (A != 0) {
    using W = typename Words<sizeof(T), A>::type;
    T t[VEC];
    W w[sizeof t / A];
#pragma unroll
    for (unsigned k = 0; k < sizeof t / A; ++k)
      w[k] = __builtin_nontemporal_load(reinterpret_cast<const W*>(p) + k);
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

// the error is reported here: it does not stay behind for the thread's next check
#define OP_HIP(x, what)                                                             \
  do {                                                                              \
    hipError_t e_ = (x);                                                            \
    if (e_ != hipSuccess) {                                                         \
      (void)hipGetLastError();                                                      \
      return g2v::op_fail(G2V_EHIP, "%s: %s", (what), hipGetErrorString(e_));       \
    }                                                                               \
  } while (0)
