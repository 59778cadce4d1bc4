// Dropout whose mask is a function of (seed, offset, element) and is never
// stored: the backward pass draws it again.
//
//   y_i = x_i * s   if w_i <= last, else 0        s = 1 / (1 - p)
//
// w_i is word i % 4 of Philox4x32 with 10 rounds (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter
// (i / 4, offset) under key seed, 64 bits each; last = round((1-p) 2^32) - 1.
// The mask depends on the element's index alone, not on the type or on how
// the work is split.  A dropped element is selected away, not multiplied,
// so an infinity or NaN in it is gone.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "vec.h"

struct Philox {
  unsigned w[4];
};

// 20 products of 32 x 32 bits a block of four words; each high half takes
// its two exclusive-ors in one three-input operation.
__device__ __forceinline__ Philox philox10(unsigned long block,
                                           unsigned long offset,
                                           unsigned long seed) {
  unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32);
  unsigned c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long p0 = 0xD2511F53ul * c0;
    const unsigned long p1 = 0xCD9E8D57ul * c2;
    c0 = (unsigned)(p1 >> 32) ^ c1 ^ k0;
    c2 = (unsigned)(p0 >> 32) ^ c3 ^ k1;
    c1 = (unsigned)p1;
    c3 = (unsigned)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

template <typename T>
__device__ __forceinline__ T drop(T x, unsigned w, unsigned last, float s) {
  float y = (float)x * s;
  // Keeps the product and the rounding to fp16 apart, which the compiler
  // would otherwise do in one instruction with one rounding: two roundings
  // are what the CPU path does, and the results stay the same bits.
  asm("" : "+v"(y));
  return w <= last ? (T)y : (T)0.0f;
}

// One vector of 16 bytes a thread: more of them (2: 47.6 us for 45.4, 4: 50.9
// at 8192 x 8192 bf16) only lengthen a block.  That is 5.9 TB/s, 94% of what
// a plain copy reaches; two Philox blocks for every eight elements of 16 bits
// stay hidden behind it.
template <typename T, bool LARGE>
__global__ void __launch_bounds__(256)
    dropout_kernel(const T* __restrict__ x, T* __restrict__ y,
                   const long* __restrict__ state, long n, unsigned last,
                   float scale) {
  constexpr int N = Vec<T>::N;
  const unsigned long seed = (unsigned long)state[0];
  const unsigned long offset = (unsigned long)state[1];
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * N;
  if (i + N <= n) {
    typename Vec<T>::V v =
        LARGE ? Vec<T>::load_once(x + i) : Vec<T>::load(x + i);
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      const Philox r = philox10((unsigned long)(i / 4 + q), offset, seed);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[4 * q + j] = drop(v[4 * q + j], r.w[j], last, scale);
    }
    if (LARGE)
      Vec<T>::store_once(y + i, v);
    else
      Vec<T>::store(y + i, v);
    return;
  }
  for (long e = i; e < n; ++e) {
    const Philox r = philox10((unsigned long)(e / 4), offset, seed);
    const unsigned w = e % 4 == 0   ? r.w[0]
                       : e % 4 == 1 ? r.w[1]
                       : e % 4 == 2 ? r.w[2]
                                    : r.w[3];
    y[e] = drop(x[e], w, last, scale);
  }
}

// The state of one draw, and the state stepped on for the next one.
__global__ void dropout_next_kernel(long* __restrict__ state,
                                    long* __restrict__ out) {
  out[0] = state[0];
  out[1] = state[1];
  state[1] = (long)((unsigned long)state[1] + 1);
}

static void check_state(const torch::Tensor& state) {
  TORCH_CHECK(state.is_cuda() && state.scalar_type() == torch::kInt64 &&
                  state.is_contiguous() && state.numel() == 2,
              "state must be two contiguous int64 on GPU");
}

// keep: how many of the 2^32 words keep an element, 1 .. 2^32.
torch::Tensor dropout(torch::Tensor x, torch::Tensor state, int64_t keep,
                      double scale) {
  check_state(state);
  TORCH_CHECK(x.is_cuda() && x.is_contiguous(),
              "x must be contiguous on GPU");
  TORCH_CHECK(x.device() == state.device(),
              "x and state must be on one device");
  TORCH_CHECK(keep >= 1 && keep <= (1l << 32), "keep must be 1 .. 2^32");
  const at::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty_like(x);
  const long n = x.numel();
  if (n == 0) return y;
  auto stream = at::cuda::getCurrentCUDAStream();
  for_dtype(x.scalar_type(), "x", [&](auto t) {
    using T = decltype(t);
    const long vecs = (n + Vec<T>::N - 1) / Vec<T>::N;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid_of((vecs + 255) / 256, 256, "dropout"),
                         dim3(256), 0, stream, ptr<T>(x), ptr<T>(y),
                         state.data_ptr<int64_t>(), n,
                         (unsigned)(keep - 1), (float)scale);
    };
    // Beyond the 256 MB of the last cache nothing of x or y would be found
    // there again (8192 x 8192 bf16: 45.4 us for 47.5).
    if (2 * n * (long)sizeof(T) >= 256l << 20)
      go(dropout_kernel<T, true>);
    else
      go(dropout_kernel<T, false>);
  });
  LAUNCH_OK();
  return y;
}

torch::Tensor dropout_next(torch::Tensor state) {
  check_state(state);
  const at::cuda::CUDAGuard guard(state.device());
  auto out = torch::empty_like(state);
  hipLaunchKernelGGL(dropout_next_kernel, dim3(1), dim3(1), 0,
                     at::cuda::getCurrentCUDAStream(),
                     state.data_ptr<int64_t>(), out.data_ptr<int64_t>());
  LAUNCH_OK();
  // a change in place, which autograd has to notice in what it saved
  state.unsafeGetTensorImpl()->bump_version();
  return out;
}
