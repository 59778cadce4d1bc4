// fp32 MFMA GEMM with fused bias + activation epilogue, plus the dgrad /
// wgrad / bias-grad companions — the MI355X replacement for the
// reference's TF dense layers (reference examples/simple_dnn.py:16-18;
// SURVEY.md §2.2 "Dense layer: GEMM + bias add").
//
// Design: 64x64 output tile per 256-thread workgroup (4 waves, each a
// 32x32 subtile of 2x2 v_mfma_f32_16x16x4_f32 fragments — exact fp32 at
// the 157 TF matrix rate, cdna_hip_programming.md §3), K staged through
// LDS in 16-deep chunks, bias+activation fused into the accumulator
// store.  Transpose handling for the backward GEMMs is done at the LDS
// staging step (coalesced global reads either way), so dgrad
// (dy @ W^T) and wgrad (x^T @ dy) reuse the same MFMA pipeline.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>

#include "common.h"

#define BM 64
#define BN 64
#define BK 16

// Logical C[M,N] = act(A'[M,K] @ B'[K,N] + bias).
// TA=0: A' = A_phys[M,K] (lda=K);  TA=1: A' = A_phys[K,M]^T (lda=M).
// TB=0: B' = B_phys[K,N] (ldb=N);  TB=1: B' = B_phys[N,K]^T (ldb=K).
//
// SPLITK mode (blockIdx.z slices the K range): the async-PS workloads are
// small-M GEMMs whose M/N tiling alone fills a fraction of the 256 CUs —
// K-slicing multiplies resident workgroups (the "decomposition first"
// rule for sampling-regime GEMMs).  Each K-slice writes its partial tile
// to a [splitk, M, N] workspace with plain stores (no zero-fill pass, no
// atomics, deterministic); a small reduce epilogue sums the slices and
// applies bias+activation.
// DPRE_A / DPRE_B: the A (TA=0) or B (TB=0) operand is the activation
// backward dpre = act_grad(preY, A_phys) computed AT LOAD TIME — fusing
// the standalone act_bwd kernel (and its dpre HBM round trip) into the
// dgrad / wgrad GEMMs that consume it.
template <bool TA, bool TB, bool HAS_BIAS, bool SPLITK,
          bool BIASROW = false, bool DPRE_A = false, bool DPRE_B = false>
__global__ __launch_bounds__(256) void gemm_f32_kernel(
    const float* __restrict__ A, const float* __restrict__ B,
    const float* __restrict__ bias, float* __restrict__ C, int M, int N,
    int K, int lda, int ldb, int act, int k_chunk,
    const float* __restrict__ preY = nullptr, int pre_act = 0) {
  __shared__ float As[BM][BK + 1];
  __shared__ float Bs[BK][BN + 4];

  const int t = threadIdx.x;
  const int lane = t & 63;
  const int w = t >> 6;       // wave 0..3
  const int wm = (w >> 1) * 32;
  const int wn = (w & 1) * 32;
  const int m0 = blockIdx.y * BM;
  const int n0 = blockIdx.x * BN;

  f32x4 acc[2][2] = {};

  int k_begin = 0, k_end = K;
  if (SPLITK) {
    k_begin = blockIdx.z * k_chunk;
    k_end = min(K, k_begin + k_chunk);
  }

  // Per-thread load/store split so the NEXT chunk's global loads issue
  // during the CURRENT chunk's MFMAs (register prefetch — the K loop is
  // load-latency-bound at these sizes, cdna_hip_programming.md "overlap
  // global with MFMA").  Each thread owns one float4 of A and one of B
  // per chunk.
  const int a_row = t >> 2, a_c4 = (t & 3) * 4;       // TA=0 path
  const int a_kk = t >> 4, a_m4 = (t & 15) * 4;       // TA=1 path
  const int b_kk = t >> 4, b_n4 = (t & 15) * 4;       // TB=0 path
  const int b_row = t >> 2, b_c4 = (t & 3) * 4;       // TB=1 path

  auto load_a = [&](int k0) -> float4 {
    float4 r;
    if (!TA) {
      const int gm = m0 + a_row;
      if (gm < M && k0 + BK <= K) {
        r = *reinterpret_cast<const float4*>(&A[(long)gm * lda + k0 + a_c4]);
        if (DPRE_A) {
          const float4 y4 = *reinterpret_cast<const float4*>(
              &preY[(long)gm * lda + k0 + a_c4]);
          float* rr = reinterpret_cast<float*>(&r);
          const float* yy = reinterpret_cast<const float*>(&y4);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            rr[i] = act_grad_from_out(yy[i], rr[i], pre_act);
        }
      } else {
        float* rr = reinterpret_cast<float*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int gk = k0 + a_c4 + i;
          const bool ok = gm < M && gk < K;
          float v = ok ? A[(long)gm * lda + gk] : 0.0f;
          if (DPRE_A && ok)
            v = act_grad_from_out(preY[(long)gm * lda + gk], v, pre_act);
          rr[i] = v;
        }
      }
    } else {
      const int gk = k0 + a_kk;
      // BIASROW: logical row M-1 is a virtual all-ones row (bias grad
      // rides the wgrad GEMM); the fast path must not read it.
      const int m_phys = BIASROW ? M - 1 : M;
      if (gk < K && m0 + BM <= m_phys) {
        r = *reinterpret_cast<const float4*>(&A[(long)gk * lda + m0 + a_m4]);
      } else {
        float* rr = reinterpret_cast<float*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int gm = m0 + a_m4 + i;
          float val = 0.0f;
          if (gk < K && gm < M) {
            val = (BIASROW && gm == M - 1) ? 1.0f : A[(long)gk * lda + gm];
          }
          rr[i] = val;
        }
      }
    }
    return r;
  };

  auto load_b = [&](int k0) -> float4 {
    float4 r;
    if (!TB) {
      const int gk = k0 + b_kk;
      if (gk < K && n0 + BN <= N) {
        r = *reinterpret_cast<const float4*>(&B[(long)gk * ldb + n0 + b_n4]);
        if (DPRE_B) {
          const float4 y4 = *reinterpret_cast<const float4*>(
              &preY[(long)gk * ldb + n0 + b_n4]);
          float* rr = reinterpret_cast<float*>(&r);
          const float* yy = reinterpret_cast<const float*>(&y4);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            rr[i] = act_grad_from_out(yy[i], rr[i], pre_act);
        }
      } else {
        float* rr = reinterpret_cast<float*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int gn = n0 + b_n4 + i;
          const bool ok = gk < K && gn < N;
          float v = ok ? B[(long)gk * ldb + gn] : 0.0f;
          if (DPRE_B && ok)
            v = act_grad_from_out(preY[(long)gk * ldb + gn], v, pre_act);
          rr[i] = v;
        }
      }
    } else {
      const int gn = n0 + b_row;
      if (gn < N && k0 + BK <= K) {
        r = *reinterpret_cast<const float4*>(&B[(long)gn * ldb + k0 + b_c4]);
      } else {
        float* rr = reinterpret_cast<float*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int gk = k0 + b_c4 + i;
          rr[i] = (gn < N && gk < K) ? B[(long)gn * ldb + gk] : 0.0f;
        }
      }
    }
    return r;
  };

  auto store_lds = [&](float4 ra, float4 rb) {
    const float* pa = reinterpret_cast<const float*>(&ra);
    const float* pb = reinterpret_cast<const float*>(&rb);
    if (!TA) {
#pragma unroll
      for (int i = 0; i < 4; ++i) As[a_row][a_c4 + i] = pa[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) As[a_m4 + i][a_kk] = pa[i];
    }
    if (!TB) {
#pragma unroll
      for (int i = 0; i < 4; ++i) Bs[b_kk][b_n4 + i] = pb[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) Bs[b_c4 + i][b_row] = pb[i];
    }
  };

  const int fr = lane & 15;   // fragment row/col position
  const int fk = lane >> 4;   // k sub-index 0..3

  float4 ra = load_a(k_begin);
  float4 rb = load_b(k_begin);
  for (int k0 = k_begin; k0 < k_end; k0 += BK) {
    store_lds(ra, rb);
    __syncthreads();
    if (k0 + BK < k_end) {  // prefetch next chunk over this chunk's MFMAs
      ra = load_a(k0 + BK);
      rb = load_b(k0 + BK);
    }
    // ---- 16x16x4 MFMA over the 16-deep chunk ----
#pragma unroll
    for (int kk = 0; kk < BK / 4; ++kk) {
      const float a0 = As[wm + fr][kk * 4 + fk];
      const float a1 = As[wm + 16 + fr][kk * 4 + fk];
      const float b0 = Bs[kk * 4 + fk][wn + fr];
      const float b1 = Bs[kk * 4 + fk][wn + 16 + fr];
      acc[0][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a0, b0, acc[0][0], 0, 0, 0);
      acc[0][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(a0, b1, acc[0][1], 0, 0, 0);
      acc[1][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a1, b0, acc[1][0], 0, 0, 0);
      acc[1][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(a1, b1, acc[1][1], 0, 0, 0);
    }
    __syncthreads();
  }

  // ---- epilogue ----
  // C/D fragment map (16x16 shapes): col = lane&15, row = (lane>>4)*4 + i.
  const int fcol = lane & 15;
  const int frow = (lane >> 4) * 4;
#pragma unroll
  for (int mi = 0; mi < 2; ++mi) {
#pragma unroll
    for (int ni = 0; ni < 2; ++ni) {
      const int col = n0 + wn + ni * 16 + fcol;
      if (col >= N) continue;
      const float bv = (!SPLITK && HAS_BIAS) ? bias[col] : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = m0 + wm + mi * 16 + frow + i;
        if (row < M) {
          if (SPLITK) {
            // C points at the workspace; slice z owns plane z*M*N
            C[(long)blockIdx.z * M * N + (long)row * N + col] =
                acc[mi][ni][i];
          } else {
            C[(long)row * N + col] = act_apply(acc[mi][ni][i] + bv, act);
          }
        }
      }
    }
  }
}

// Split-K reduce epilogue: C = act(sum_z W[z] + bias).
template <bool HAS_BIAS>
__global__ void splitk_reduce_kernel(const float* __restrict__ W,
                                     const float* __restrict__ bias,
                                     float* __restrict__ C, long n, int N,
                                     int splitk, int act) {
  const long stride = (long)gridDim.x * blockDim.x;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += stride) {
    float s = HAS_BIAS ? bias[i % N] : 0.0f;
    for (int z = 0; z < splitk; ++z) s += W[(long)z * n + i];
    C[i] = act_apply(s, act);
  }
}

// float4 variant (n % 4 == 0, and N % 4 == 0 when biased, so a bias
// float4 never straddles a row boundary).
template <bool HAS_BIAS>
__global__ void splitk_reduce4_kernel(const float4* __restrict__ W,
                                      const float* __restrict__ bias,
                                      float4* __restrict__ C, long n4, int N,
                                      int splitk, int act) {
  const long stride = (long)gridDim.x * blockDim.x;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n4;
       i += stride) {
    float4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (HAS_BIAS) {
      const int col = (int)((i * 4) % N);
      s = *reinterpret_cast<const float4*>(&bias[col]);
    }
    for (int z = 0; z < splitk; ++z) {
      const float4 w = W[(long)z * n4 + i];
      s.x += w.x; s.y += w.y; s.z += w.z; s.w += w.w;
    }
    s.x = act_apply(s.x, act);
    s.y = act_apply(s.y, act);
    s.z = act_apply(s.z, act);
    s.w = act_apply(s.w, act);
    C[i] = s;
  }
}

// Column sums with 2D parallelism: blockIdx.y owns a row chunk so narrow
// layers (N=10..256) still fill more than one CU; partial sums combine
// with one atomicAdd per (col, chunk).  db must arrive zeroed.
#define BG_ROWS 8
__global__ void bias_grad_kernel(const float* __restrict__ dy,
                                 float* __restrict__ db, int M, int N) {
  const int n = blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= N) return;
  const int m0 = blockIdx.y * BG_ROWS;
  const int m1 = min(M, m0 + BG_ROWS);
  float s = 0.0f;
  for (int m = m0; m < m1; ++m) s += dy[(long)m * N + n];
  if (gridDim.y == 1) {
    db[n] = s;
  } else {
    atomicAdd(&db[n], s);
  }
}

// ---------------------------------------------------------------------------

static inline void check_f32(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32, name, " must be fp32");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

int sf_splitk_env_max() {
  static int cached = -1;
  if (cached < 0) {
    const char* e = getenv("SPARKFLOW_SPLITK_MAX");
    cached = e ? atoi(e) : 1 << 20;  // unset: no env cap, structural
    if (cached < 1) cached = 1;      // limits at the call sites govern
  }
  return cached;
}

// Pick a K split so the grid approaches the 256-CU mark (a launch needs
// many more workgroups than the M/N tiling of a 300x256 layer provides).
// Measured (profiles/w4_kernels.md): shrinking the split under multi-
// stream contention makes each GEMM slower without removing the reduce
// launch, so the target stays at 512 regardless of the hint; the env cap
// remains for experiments.
// Small-output direct mode: once the wgrad reduces are fused into the
// optimizer apply (reduce_apply_adam), the per-GEMM split-K reduce
// launch (~5 us) costs more than the split buys for small-M*N,
// shallow-K outputs (the 300x256 dgrad / L2-L3 fwd shapes) — below the
// threshold the GEMM goes direct and its reduce launch disappears.
static long sf_splitk_direct_mn() {
  static long cached = -1;
  if (cached < 0) {
    const char* e = getenv("SPARKFLOW_SPLITK_DIRECT_MN");
    cached = e ? atol(e) : 0;  // default off until measured
    if (cached < 0) cached = 0;
  }
  return cached;
}

static int pick_splitk(int M, int N, int K) {
  if ((long)M * N <= sf_splitk_direct_mn() && K <= 256) return 1;
  const int base = ceil_div(M, BM) * ceil_div(N, BN);
  const int max_by_k = std::max(1, K / 64);  // keep >=64-deep slices
  const int cap = sf_splitk_env_max();
  int splitk = 1;
  while (splitk < 8 && splitk < cap && base * splitk * 2 <= 512 &&
         splitk * 2 <= max_by_k) {
    splitk *= 2;
  }
  return splitk;
}

template <bool TA, bool TB, bool DPRE_A = false, bool DPRE_B = false>
static void launch_gemm(const torch::Tensor& A, const torch::Tensor& B,
                        const torch::Tensor& bias, torch::Tensor& C, int M,
                        int N, int K, int lda, int ldb, int act,
                        const float* preY = nullptr, int pre_act = 0) {
  // an empty batch: a launch without blocks would leave an error behind,
  // which the next operator reports
  if (M == 0 || N == 0) return;
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool has_bias = bias.numel() > 0;
  const int splitk = pick_splitk(M, N, K);
  if (splitk > 1) {
    const int k_chunk = ceil_div(K, splitk * BK) * BK;
    auto ws = torch::empty({splitk, M, N}, C.options());
    dim3 grid(ceil_div(N, BN), ceil_div(M, BM), splitk);
    hipLaunchKernelGGL(
        (gemm_f32_kernel<TA, TB, false, true, false, DPRE_A, DPRE_B>), grid,
        dim3(256), 0, stream, A.data_ptr<float>(), B.data_ptr<float>(),
        nullptr, ws.data_ptr<float>(), M, N, K, lda, ldb, act, k_chunk,
        preY, pre_act);
    const long n = (long)M * N;
    const bool v4 = (n & 3) == 0 && (!has_bias || (N & 3) == 0);
    if (v4) {
      const long n4 = n >> 2;
      const int blocks = (int)std::min<long>(2048, (n4 + 255) / 256);
      auto* w4 = reinterpret_cast<const float4*>(ws.data_ptr<float>());
      auto* c4 = reinterpret_cast<float4*>(C.data_ptr<float>());
      if (has_bias) {
        hipLaunchKernelGGL((splitk_reduce4_kernel<true>), dim3(blocks),
                           dim3(256), 0, stream, w4,
                           bias.data_ptr<float>(), c4, n4, N, splitk, act);
      } else {
        hipLaunchKernelGGL((splitk_reduce4_kernel<false>), dim3(blocks),
                           dim3(256), 0, stream, w4, nullptr, c4, n4, N,
                           splitk, act);
      }
      return;
    }
    const int blocks = (int)std::min<long>(2048, (n + 255) / 256);
    if (has_bias) {
      hipLaunchKernelGGL((splitk_reduce_kernel<true>), dim3(blocks),
                         dim3(256), 0, stream, ws.data_ptr<float>(),
                         bias.data_ptr<float>(), C.data_ptr<float>(), n, N,
                         splitk, act);
    } else {
      hipLaunchKernelGGL((splitk_reduce_kernel<false>), dim3(blocks),
                         dim3(256), 0, stream, ws.data_ptr<float>(), nullptr,
                         C.data_ptr<float>(), n, N, splitk, act);
    }
    return;
  }
  dim3 grid(ceil_div(N, BN), ceil_div(M, BM));
  if (has_bias) {
    hipLaunchKernelGGL(
        (gemm_f32_kernel<TA, TB, true, false, false, DPRE_A, DPRE_B>), grid,
        dim3(256), 0, stream, A.data_ptr<float>(), B.data_ptr<float>(),
        bias.data_ptr<float>(), C.data_ptr<float>(), M, N, K, lda, ldb, act,
        K, preY, pre_act);
  } else {
    hipLaunchKernelGGL(
        (gemm_f32_kernel<TA, TB, false, false, false, DPRE_A, DPRE_B>),
        grid, dim3(256), 0, stream, A.data_ptr<float>(),
        B.data_ptr<float>(), nullptr, C.data_ptr<float>(), M, N, K, lda,
        ldb, act, K, preY, pre_act);
  }
}

torch::Tensor gemm_act(torch::Tensor x, torch::Tensor w, torch::Tensor bias,
                       int64_t act) {
  check_f32(x, "x");
  check_f32(w, "w");
  const int M = x.size(0), K = x.size(1), N = w.size(1);
  TORCH_CHECK(w.size(0) == K, "shape mismatch x@w");
  auto y = torch::empty({M, N}, x.options());
  launch_gemm<false, false>(x, w, bias, y, M, N, K, K, N, (int)act);
  return y;
}

torch::Tensor gemm_dgrad(torch::Tensor dy, torch::Tensor w) {
  check_f32(dy, "dy");
  check_f32(w, "w");
  const int M = dy.size(0), Nout = dy.size(1), Kin = w.size(0);
  TORCH_CHECK(w.size(1) == Nout, "shape mismatch dgrad");
  auto dx = torch::empty({M, Kin}, dy.options());
  auto empty = torch::empty({0}, dy.options());
  // dx[M,Kin] = dy[M,Nout] @ w^T  (B' = w^T via TB=1)
  launch_gemm<false, true>(dy, w, empty, dx, M, Kin, Nout, Nout, Nout,
                           ACT_NONE);
  return dx;
}

torch::Tensor gemm_dgrad_act(torch::Tensor dy, torch::Tensor y,
                             torch::Tensor w, int64_t act) {
  // dx = act_grad(y, dy) @ w^T with the activation backward fused into
  // the A-operand load (no standalone act_bwd pass or dpre buffer).
  check_f32(dy, "dy");
  check_f32(y, "y");
  check_f32(w, "w");
  const int M = dy.size(0), Nout = dy.size(1), Kin = w.size(0);
  TORCH_CHECK(w.size(1) == Nout, "shape mismatch dgrad");
  auto dx = torch::empty({M, Kin}, dy.options());
  auto empty = torch::empty({0}, dy.options());
  launch_gemm<false, true, true, false>(dy, w, empty, dx, M, Kin, Nout,
                                        Nout, Nout, ACT_NONE,
                                        y.data_ptr<float>(), (int)act);
  return dx;
}

torch::Tensor gemm_wgrad(torch::Tensor x, torch::Tensor dy) {
  check_f32(x, "x");
  check_f32(dy, "dy");
  const int Mb = x.size(0), Kin = x.size(1), Nout = dy.size(1);
  TORCH_CHECK(dy.size(0) == Mb, "shape mismatch wgrad");
  auto dw = torch::empty({Kin, Nout}, x.options());
  auto empty = torch::empty({0}, x.options());
  // dw[Kin,Nout] = x^T @ dy  (A' = x^T via TA=1)
  launch_gemm<true, false>(x, dy, empty, dw, Kin, Nout, Mb, Kin, Nout,
                           ACT_NONE);
  return dw;
}

template <bool DPRE_B>
static torch::Tensor wgrad_bias_impl(torch::Tensor x, torch::Tensor dy,
                                     const float* preY, int pre_act) {
  // dwb[Kin+1, Nout] = [x; ones]^T @ dpre : rows 0..Kin-1 are dW, row
  // Kin is the bias gradient (column sums) — one GEMM instead of a GEMM
  // plus a separate reduction kernel; with DPRE_B the activation
  // backward is fused into the B-operand load as well.
  check_f32(x, "x");
  check_f32(dy, "dy");
  const int Mb = x.size(0), Kin = x.size(1), Nout = dy.size(1);
  TORCH_CHECK(dy.size(0) == Mb, "shape mismatch wgrad_bias");
  const int M = Kin + 1;
  auto dwb = torch::empty({M, Nout}, x.options());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int splitk = pick_splitk(M, Nout, Mb);
  if (splitk > 1) {
    const int k_chunk = ceil_div(Mb, splitk * BK) * BK;
    auto ws = torch::empty({splitk, M, Nout}, x.options());
    dim3 grid(ceil_div(Nout, BN), ceil_div(M, BM), splitk);
    hipLaunchKernelGGL(
        (gemm_f32_kernel<true, false, false, true, true, false, DPRE_B>),
        grid, dim3(256), 0, stream, x.data_ptr<float>(),
        dy.data_ptr<float>(), nullptr, ws.data_ptr<float>(), M, Nout, Mb,
        Kin, Nout, ACT_NONE, k_chunk, preY, pre_act);
    const long n = (long)M * Nout;
    if ((n & 3) == 0) {
      const long n4 = n >> 2;
      const int blocks = (int)std::min<long>(2048, (n4 + 255) / 256);
      hipLaunchKernelGGL(
          (splitk_reduce4_kernel<false>), dim3(blocks), dim3(256), 0,
          stream, reinterpret_cast<const float4*>(ws.data_ptr<float>()),
          nullptr, reinterpret_cast<float4*>(dwb.data_ptr<float>()), n4,
          Nout, splitk, ACT_NONE);
    } else {
      const int blocks = (int)std::min<long>(2048, (n + 255) / 256);
      hipLaunchKernelGGL((splitk_reduce_kernel<false>), dim3(blocks),
                         dim3(256), 0, stream, ws.data_ptr<float>(), nullptr,
                         dwb.data_ptr<float>(), n, Nout, splitk, ACT_NONE);
    }
  } else {
    dim3 grid(ceil_div(Nout, BN), ceil_div(M, BM));
    hipLaunchKernelGGL(
        (gemm_f32_kernel<true, false, false, false, true, false, DPRE_B>),
        grid, dim3(256), 0, stream, x.data_ptr<float>(),
        dy.data_ptr<float>(), nullptr, dwb.data_ptr<float>(), M, Nout, Mb,
        Kin, Nout, ACT_NONE, Mb, preY, pre_act);
  }
  return dwb;
}

// Deferred-reduce variant: return the raw [splitk, Kin+1, Nout] split-K
// workspace WITHOUT the reduce epilogue.  The fused reduce+Adam apply
// (optim.hip reduce_apply_adam) consumes the partials of every layer in
// one launch; a plane of this workspace is exactly the layer's
// contiguous (weight, bias) slice of the flat buffer.  splitk == 1
// degenerates to the direct GEMM writing plane 0.
template <bool DPRE_B>
static torch::Tensor wgrad_bias_ws_impl(torch::Tensor x, torch::Tensor dy,
                                        const float* preY, int pre_act) {
  check_f32(x, "x");
  check_f32(dy, "dy");
  const int Mb = x.size(0), Kin = x.size(1), Nout = dy.size(1);
  TORCH_CHECK(dy.size(0) == Mb, "shape mismatch wgrad_bias_ws");
  const int M = Kin + 1;
  auto stream = at::cuda::getCurrentCUDAStream();
  const int splitk = pick_splitk(M, Nout, Mb);
  auto ws = torch::empty({splitk, M, Nout}, x.options());
  if (splitk > 1) {
    const int k_chunk = ceil_div(Mb, splitk * BK) * BK;
    dim3 grid(ceil_div(Nout, BN), ceil_div(M, BM), splitk);
    hipLaunchKernelGGL(
        (gemm_f32_kernel<true, false, false, true, true, false, DPRE_B>),
        grid, dim3(256), 0, stream, x.data_ptr<float>(),
        dy.data_ptr<float>(), nullptr, ws.data_ptr<float>(), M, Nout, Mb,
        Kin, Nout, ACT_NONE, k_chunk, preY, pre_act);
  } else {
    dim3 grid(ceil_div(Nout, BN), ceil_div(M, BM));
    hipLaunchKernelGGL(
        (gemm_f32_kernel<true, false, false, false, true, false, DPRE_B>),
        grid, dim3(256), 0, stream, x.data_ptr<float>(),
        dy.data_ptr<float>(), nullptr, ws.data_ptr<float>(), M, Nout, Mb,
        Kin, Nout, ACT_NONE, Mb, preY, pre_act);
  }
  return ws;
}

torch::Tensor gemm_wgrad_bias_ws(torch::Tensor x, torch::Tensor dy) {
  return wgrad_bias_ws_impl<false>(x, dy, nullptr, 0);
}

torch::Tensor gemm_wgrad_bias_act_ws(torch::Tensor x, torch::Tensor dy,
                                     torch::Tensor y, int64_t act) {
  check_f32(y, "y");
  return wgrad_bias_ws_impl<true>(x, dy, y.data_ptr<float>(), (int)act);
}

torch::Tensor gemm_wgrad_bias(torch::Tensor x, torch::Tensor dy) {
  return wgrad_bias_impl<false>(x, dy, nullptr, 0);
}

torch::Tensor gemm_wgrad_bias_act(torch::Tensor x, torch::Tensor dy,
                                  torch::Tensor y, int64_t act) {
  check_f32(y, "y");
  return wgrad_bias_impl<true>(x, dy, y.data_ptr<float>(), (int)act);
}

torch::Tensor bias_grad(torch::Tensor dy) {
  check_f32(dy, "dy");
  const int M = dy.size(0), N = dy.size(1);
  const int chunks = ceil_div(M, BG_ROWS);
  auto db = chunks > 1 ? torch::zeros({N}, dy.options())
                       : torch::empty({N}, dy.options());
  auto stream = at::cuda::getCurrentCUDAStream();
  hipLaunchKernelGGL(bias_grad_kernel, dim3(ceil_div(N, 256), chunks),
                     dim3(256), 0, stream, dy.data_ptr<float>(),
                     db.data_ptr<float>(), M, N);
  return db;
}
