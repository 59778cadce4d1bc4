// 16-byte vectors of the three storage types (fp32, bf16, fp16), with all
// arithmetic in fp32.
//
// Loads and stores are declared with the alignment of one element, so a row
// may start anywhere (an odd row length, a view into a larger tensor);
// gfx950 takes such addresses in its widest accesses, and the compiler
// emits global_load_dwordx4 / global_store_dwordx4 for them.
#pragma once

#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
  struct __attribute__((packed, aligned(sizeof(T)))) Unaligned {
    V v;
  };
  static __device__ __forceinline__ V load(const T* p) {
    return reinterpret_cast<const Unaligned*>(p)->v;
  }
  static __device__ __forceinline__ void store(T* p, V v) {
    reinterpret_cast<Unaligned*>(p)->v = v;
  }
  // For what is read or written once and is larger than the caches: it does
  // not displace what they hold.
  static __device__ __forceinline__ V load_once(const T* p) {
    return __builtin_nontemporal_load(
        &reinterpret_cast<const Unaligned*>(p)->v);
  }
  static __device__ __forceinline__ void store_once(T* p, V v) {
    __builtin_nontemporal_store(v, &reinterpret_cast<Unaligned*>(p)->v);
  }
};

// Calls f(T()) with the kernel's type for a tensor's dtype.
template <typename F>
static inline void for_dtype(c10::ScalarType t, const char* name, F&& f) {
  if (t == c10::kFloat) {
    f(float());
  } else if (t == c10::kBFloat16) {
    f(bf16_t());
  } else {
    TORCH_CHECK(t == c10::kHalf, name, " must be fp32, bf16 or fp16, got ",
                t);
    f(f16_t());
  }
}

template <typename T>
static inline T* ptr(const torch::Tensor& t) {
  return reinterpret_cast<T*>(t.data_ptr());
}

// The blocks of a launch, whose threads are counted in 32 bits.
static inline dim3 grid_of(long blocks, int threads, const char* name) {
  TORCH_CHECK(blocks * threads < (1l << 32), name, ": too many rows");
  return dim3((unsigned)blocks);
}

// After a launch: a refused launch becomes an exception at the call.
#define LAUNCH_OK()                                                     \
  do {                                                                  \
    const hipError_t _e = hipGetLastError();                            \
    TORCH_CHECK(_e == hipSuccess, "kernel launch failed: ",             \
                hipGetErrorString(_e));                                 \
  } while (0)
