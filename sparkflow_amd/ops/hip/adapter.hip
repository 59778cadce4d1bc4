// Low-rank adapters of many requests beside a shared projection.
//
//   out_m = act(base_m + s_e (x_m A_e^T) B_e^T),  e = ids[m]
//   A [E, R, K], B [E, N, R], R small
//
//   dz_m = s_e dy_m B_e          dx_m = dz_m A_e
//   dA_e = sum_m dz_m^T x_m      dB_e = sum_m dy_m^T z_m,  z_m = s_e x_m A_e^T
//
// Rows are grouped by adapter first (adapter_plan), and every other kernel
// works on tiles of up to 16 rows of one adapter, so an adapter is read once
// a tile and not once a row.  z and dz stay in fp32, [M, Rp] in the grouped
// order with R padded to whole blocks of 16: every output is rounded once.
//
// Four kernels do all the products:
//   shrink  z = s x A^T, dz = s dy B     long sums, few columns
//   expand  out = act(base + z B^T), dx = dz A
//   outer   dA, dB: sums over the rows of an adapter
//   reduce  joins outer's partial sums
// A row with a negative id has no adapter and comes through as act(base);
// an id of E or more cannot be refused without waiting for the device and
// gives a row of NaN.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "vec.h"

#define TILE 16
#define RANK_MAX 128
#define ADAPTERS_MAX 1024

typedef float f32x4v __attribute__((ext_vector_type(4)));

// -- rows by adapter ----------------------------------------------------------

// Groups: 0 .. E-1 the adapters, E rows without one, E + 1 rows whose id
// names none.
__device__ __forceinline__ int group_of(long id, int E) {
  return id < 0 ? E : id < E ? (int)id : E + 1;
}

struct Plan {
  int* perm;        // [M] the row at each place of the grouped order
  int* seg;         // [E + 3] where a group's rows begin
  int* tbase;       // [E + 3] where a group's tiles begin
  int* tile_group;  // [tiles] -1 behind the last
  int* tile_place;  // [tiles] first place
};

// A stable counting sort in one block.  Each of 8 waves owns a stretch of
// the rows and counts it for itself, so that no order depends on timing.
__global__ void __launch_bounds__(512)
    adapter_plan_kernel(const long* __restrict__ ids, Plan p, int M, int E,
                        int tiles) {
  extern __shared__ int hist[];  // [8][E + 2] and [E + 3]
  const int G = E + 2;
  int* total = hist + 8 * G;
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid & (WAVE - 1);
  for (int i = tid; i < 8 * G; i += 512) hist[i] = 0;
  __syncthreads();
  const int stretch = (M + 8 * WAVE - 1) / (8 * WAVE) * WAVE;
  const int lo = wave * stretch;
  const int hi = min(M, lo + stretch);
  int* mine = hist + wave * G;
  for (int i = lo + lane; i < hi; i += WAVE)
    atomicAdd(&mine[group_of(ids[i], E)], 1);
  __syncthreads();
  // per group: the waves' counts become offsets, their sum the total
  for (int g = tid; g < G; g += 512) {
    int sum = 0;
    for (int w = 0; w < 8; ++w) {
      const int c = hist[w * G + g];
      hist[w * G + g] = sum;
      sum += c;
    }
    total[g] = sum;
  }
  __syncthreads();
  // the first wave sums over the groups, 64 at a time
  if (wave == 0) {
    int rows = 0, blocks = 0;
    for (int g0 = 0; g0 < G; g0 += WAVE) {
      const int g = g0 + lane;
      const int c = g < G ? total[g] : 0;
      const int b = (c + TILE - 1) / TILE;
      int cs = c, bs = b;
#pragma unroll
      for (int off = 1; off < WAVE; off <<= 1) {
        const int cu = __shfl_up(cs, off, WAVE);
        const int bu = __shfl_up(bs, off, WAVE);
        if (lane >= off) {
          cs += cu;
          bs += bu;
        }
      }
      const int r0 = rows + cs - c, b0 = blocks + bs - b;
      if (g < G) {
        p.seg[g] = r0;
        p.tbase[g] = b0;
        total[g] = r0;
        for (int j = 0; j < b; ++j) {
          p.tile_group[b0 + j] = g;
          p.tile_place[b0 + j] = r0 + j * TILE;
        }
      }
      rows += __shfl(cs, WAVE - 1, WAVE);
      blocks += __shfl(bs, WAVE - 1, WAVE);
    }
    if (lane == 0) {
      p.seg[G] = rows;
      p.tbase[G] = blocks;
    }
    for (int t = blocks + lane; t < tiles; t += WAVE) p.tile_group[t] = -1;
  }
  __syncthreads();
  // each wave places its stretch in order
  for (int i0 = lo; i0 < hi; i0 += WAVE) {
    const int i = i0 + lane;
    const int g = i < hi ? group_of(ids[i], E) : -1;
    unsigned long left = __ballot(g >= 0);
    while (left) {
      const int first = __ffsll((unsigned long long)left) - 1;
      const int of = __shfl(g, first, WAVE);
      const unsigned long same = __ballot(g == of);
      int at = 0;
      if (lane == first) at = total[of] + atomicAdd(&mine[of], __popcll(same));
      at = __shfl(at, first, WAVE);
      if (g == of)
        p.perm[at + __popcll(same & ((1ul << lane) - 1))] = i;
      left &= ~same;
    }
  }
}

// -- matrix instructions ------------------------------------------------------

// D[i][j] += sum_k a[i][k] b[j][k] over 16 x 16: lane l gives row l % 16 of
// both operands, 16 bytes of k from the lane's quarter l / 16, and holds
// D[4 (l / 16) + q][l % 16].  In the 16-bit types one instruction takes the
// 32 k of a wave, its products exact and its sums fp32; in fp32 four take
// its 16.
__device__ __forceinline__ f32x4 mma(Vec<float>::V a, Vec<float>::V b,
                                     f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x4 mma(Vec<bf16_t>::V a, Vec<bf16_t>::V b,
                                     f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(Vec<f16_t>::V a, Vec<f16_t>::V b,
                                     f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// -- shrink -------------------------------------------------------------------

// z[place][r] = s_e sum_k x[row][k] W_e(r, k).  W is [R, K] (KMAJOR) or
// [K, R].  One block a tile; its waves take turns along k, and meet in LDS.
template <typename T, int RB, bool KMAJOR, int WAVES, int U>
__global__ void __launch_bounds__(WAVES * WAVE)
    adapter_shrink_kernel(const T* __restrict__ x, long xstride,
                          const T* __restrict__ w, Plan p,
                          const float* __restrict__ scales, float scale,
                          float* __restrict__ z, int K, int R, int E) {
  constexpr int N = Vec<T>::N;
  constexpr int STEP = 4 * N;  // k of one wave
  typedef typename Vec<T>::V V;
  __shared__ f32x4 part[WAVES][RB][WAVE];
  const int g = p.tile_group[blockIdx.x];
  if (g < 0 || g >= E) return;
  const int place = p.tile_place[blockIdx.x];
  const int rows = min(TILE, p.seg[g + 1] - place);
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int i = lane & 15, quarter = lane >> 4;
  // rows behind the tile's last repeat it, ranks behind R the last rank;
  // neither is written
  const T* xr = x + (long)p.perm[place + min(i, rows - 1)] * xstride;
  const T* we = w + (long)g * R * K;
  auto load_w = [&](int rb, int k) -> V {
    const int r = min(rb * 16 + i, R - 1);
    if (KMAJOR) return Vec<T>::load(we + (long)r * K + k);
    V v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = we[(long)(k + j) * R + r];
    return v;
  };
  f32x4 acc[RB] = {};
  const int whole = K / (STEP * U);
  for (int c = wave; c < whole; c += WAVES) {
    V xv[U], wv[U][RB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (c * U + u) * STEP + quarter * N;
      xv[u] = Vec<T>::load(xr + k);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) wv[u][rb] = load_w(rb, k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        acc[rb] = mma(xv[u], wv[u][rb], acc[rb]);
  }
  for (int k0 = whole * (STEP * U) + wave * STEP; k0 < K;
       k0 += WAVES * STEP) {
    const int k = k0 + quarter * N;
    V xv, wv[RB];
    if (k + N <= K) {
      xv = Vec<T>::load(xr + k);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) wv[rb] = load_w(rb, k);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        xv[j] = k + j < K ? xr[k + j] : (T)0.0f;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const int r = min(rb * 16 + i, R - 1);
          wv[rb][j] = k + j < K ? (KMAJOR ? we[(long)r * K + k + j]
                                          : we[(long)(k + j) * R + r])
                                : (T)0.0f;
        }
      }
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) acc[rb] = mma(xv, wv[rb], acc[rb]);
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) part[wave][rb][lane] = acc[rb];
  __syncthreads();
  const float s = scales ? scales[g] : scale;
  for (int at = threadIdx.x; at < RB * WAVE; at += WAVES * WAVE) {
    const int rb = at / WAVE, l = at % WAVE;
    f32x4 sum = part[0][rb][l];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) sum += part[v][rb][l];
    const int r = rb * 16 + (l & 15);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = (l >> 4) * 4 + q;
      if (m < rows)
        z[(long)(place + m) * (RB * 16) + r] = r < R ? s * sum[q] : 0.0f;
    }
  }
}

// The activations, a NaN staying one.
__device__ __forceinline__ float act_keep_nan(float x, int act) {
  if (act == ACT_RELU) return x < 0.0f ? 0.0f : x;
  return act_apply(x, act);
}

// -- expand -------------------------------------------------------------------

// out[row][n] = act(base[row][n] + sum_r z[place][r] W_e(n, r)), W [N, R]
// (RMAJOR) or [R, N].  The product is taken as D[n][m], in fp32, with the 16
// columns of an instruction chosen so that a lane ends up with 16 bytes of
// adjacent outputs: instruction j's row 4 h + q is column N h + 4 j + q of
// the chunk.  base enters as the sum's first term.
template <typename T, int RB, bool RMAJOR>
__global__ void __launch_bounds__(256)
    adapter_expand_kernel(const T* __restrict__ base, long bstride,
                          const float* __restrict__ z,
                          const T* __restrict__ w, Plan p,
                          T* __restrict__ out, int N, int R, int E, int act) {
  constexpr int V = Vec<T>::N;
  constexpr int CHUNK = 4 * V;
  const int g = p.tile_group[blockIdx.x];
  if (g < 0) return;
  const int place = p.tile_place[blockIdx.x];
  const int rows = min(TILE, p.seg[g + 1] - place);
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int i = lane & 15, quarter = lane >> 4;
  const bool mine = i < rows;
  const long row = p.perm[place + min(i, rows - 1)];
  const T* we = w + (long)min(g, E - 1) * N * R;
  f32x4v zv[RB];
#pragma unroll
  for (int c = 0; c < RB; ++c) {
    zv[c] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
    if (g < E)
      zv[c] = *reinterpret_cast<const f32x4v*>(
          z + (long)(place + min(i, rows - 1)) * (RB * 16) + 16 * c +
          4 * quarter);
  }
  for (int n0 = (blockIdx.y * 4 + wave) * CHUNK; n0 < N;
       n0 += gridDim.y * 4 * CHUNK) {
    const int n = n0 + quarter * V;
    f32x4 acc[V / 4] = {};
    if (base != nullptr) {
      const T* br = base + row * bstride + n;
      if (n + V <= N) {
        const typename Vec<T>::V b = Vec<T>::load(br);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j / 4][j % 4] = (float)b[j];
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (n + j < N) acc[j / 4][j % 4] = (float)br[j];
      }
    }
    if (g < E) {
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        const int col = min(n0 + (i >> 2) * V + 4 * j + (i & 3), N - 1);
#pragma unroll
        for (int c = 0; c < RB; ++c) {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int r = 16 * c + 4 * quarter + s;
            float wf = 0.0f;
            if (r < R)
              wf = (float)(RMAJOR ? we[(long)col * R + r]
                                  : we[(long)r * N + col]);
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(wf, zv[c][s],
                                                          acc[j], 0, 0, 0);
          }
        }
      }
    } else if (g > E) {
#pragma unroll
      for (int j = 0; j < V / 4; ++j)
        acc[j] = f32x4{NAN, NAN, NAN, NAN};
    }
    if (!mine) continue;
    T* o = out + row * N + n;
    typename Vec<T>::V v;
#pragma unroll
    for (int j = 0; j < V; ++j)
      v[j] = (T)act_keep_nan(acc[j / 4][j % 4], act);
    if (n + V <= N) {
      Vec<T>::store(o, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (n + j < N) o[j] = v[j];
    }
  }
}

// -- outer --------------------------------------------------------------------

// sum over the rows of a stretch of one adapter: z[place][r] x[row][k], with
// fp32 products.  A lane loads 16 bytes of a row; instruction j takes
// element j of all lanes, so its 16 columns are k0 + V (l % 16) + j and its
// four k are four rows.  KMAJOR: the result is [R, K] (dA), else [K, R]
// (dB).  DIRECT: one block an adapter, rounded into out; else one block a
// stretch of `stretch` tiles, into fp32 partial sums that reduce joins.
template <typename T, int RB, bool KMAJOR, bool DIRECT>
__global__ void __launch_bounds__(256)
    adapter_outer_kernel(const T* __restrict__ x, long xstride,
                         const float* __restrict__ z, int zstride, Plan p,
                         T* __restrict__ out, float* __restrict__ partial,
                         int K, int R, int E, int stretch) {
  constexpr int V = Vec<T>::N;
  __shared__ f32x4 part[2][RB * V][WAVE];
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int i = lane & 15, quarter = lane >> 4;
  int g, place, end;
  long slot;
  if (DIRECT) {
    g = blockIdx.x;
    place = p.seg[g];
    end = p.seg[g + 1];
    slot = g;
  } else {
    const int t = blockIdx.x;
    g = p.tile_group[t];
    if (g < 0 || g >= E || (t - p.tbase[g]) % stretch != 0) return;
    place = p.tile_place[t];
    end = min(p.seg[g + 1], place + stretch * TILE);
    slot = t / stretch + g;
  }
  const int r0 = blockIdx.z * (RB * 16);
  const int k0 = blockIdx.y * (16 * V);
  const int k = k0 + i * V;
  f32x4 acc[RB][V] = {};
  for (int m0 = place + wave * 4; m0 < end; m0 += 16) {
    const int at = m0 + quarter;
    typename Vec<T>::V xv;
    float zv[RB];
#pragma unroll
    for (int j = 0; j < V; ++j) xv[j] = (T)0.0f;
#pragma unroll
    for (int c = 0; c < RB; ++c) zv[c] = 0.0f;
    if (at < end) {
      const T* xr = x + (long)p.perm[at] * xstride;
      if (k + V <= K) {
        xv = Vec<T>::load(xr + k);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (k + j < K) xv[j] = xr[k + j];
      }
#pragma unroll
      for (int c = 0; c < RB; ++c)
        zv[c] = z[(long)at * zstride + r0 + 16 * c + i];
    }
#pragma unroll
    for (int c = 0; c < RB; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j)
        acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
            zv[c], (float)xv[j], acc[c][j], 0, 0, 0);
  }
  // the four waves' sums meet in the first
#pragma unroll
  for (int half = 2; half > 0; half >>= 1) {
    __syncthreads();
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int c = 0; c < RB; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) part[wave - half][c * V + j][lane] =
            acc[c][j];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int c = 0; c < RB; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[c][j] += part[wave][c * V + j][lane];
    }
  }
  if (wave != 0) return;
#pragma unroll
  for (int c = 0; c < RB; ++c)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = r0 + 16 * c + 4 * quarter + q;
      if (r >= R) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (k + j >= K) continue;
        const long o = slot * R * K + (KMAJOR ? (long)r * K + k + j
                                              : (long)(k + j) * R + r);
        if (DIRECT)
          out[o] = (T)acc[c][j][q];
        else
          partial[o] = acc[c][j][q];
      }
    }
}

// out_e = the sum of adapter e's partial sums, in their order; zero for an
// adapter without rows.
template <typename T>
__global__ void __launch_bounds__(256)
    adapter_reduce_kernel(const float* __restrict__ partial, Plan p,
                          T* __restrict__ out, long n, int stretch) {
  const int e = blockIdx.y;
  const int t0 = p.tbase[e], t1 = p.tbase[e + 1];
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (long)gridDim.x * 256) {
    float sum = 0.0f;
    for (int t = t0; t < t1; t += stretch)
      sum += partial[(long)(t / stretch + e) * n + i];
    out[e * n + i] = (T)sum;
  }
}

// d(act) from the output, in the operand's own type.
template <typename T>
__global__ void __launch_bounds__(256)
    adapter_act_bwd_kernel(const T* __restrict__ y, const T* __restrict__ dy,
                           T* __restrict__ dx, long n, int act) {
  const long stride = (long)gridDim.x * 256;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += stride)
    dx[i] = (T)act_grad_from_out((float)y[i], (float)dy[i], act);
}

// -- host ---------------------------------------------------------------------

static long max_tiles(long M, long E) {
  return M / TILE + std::min(E + 2, M);
}

// perm, seg, tbase, tile_group, tile_place in one int32 tensor.
static Plan plan_of(const torch::Tensor& plan, long M, long E) {
  TORCH_CHECK(plan.is_cuda() && plan.is_contiguous() &&
                  plan.scalar_type() == torch::kInt32 &&
                  plan.numel() == M + 2 * (E + 3) + 2 * max_tiles(M, E),
              "plan does not belong to these rows and adapters");
  int* p = plan.data_ptr<int>();
  Plan r;
  r.perm = p;
  r.seg = p + M;
  r.tbase = r.seg + E + 3;
  r.tile_group = r.tbase + E + 3;
  r.tile_place = r.tile_group + max_tiles(M, E);
  return r;
}

torch::Tensor adapter_plan(torch::Tensor ids, int64_t E) {
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() && ids.dim() == 1 &&
                  ids.scalar_type() == torch::kInt64,
              "ids must be contiguous int64 [rows] on GPU");
  const long M = ids.size(0);
  TORCH_CHECK(M < (1l << 30), "ids: too many rows");
  TORCH_CHECK(E >= 1 && E <= ADAPTERS_MAX, "1 .. 1024 adapters");
  const at::cuda::CUDAGuard guard(ids.device());
  const long tiles = max_tiles(M, E);
  auto plan = torch::empty({M + 2 * (E + 3) + 2 * tiles},
                           ids.options().dtype(torch::kInt32));
  const int lds = (int)((8 * (E + 2) + E + 3) * sizeof(int));
  hipLaunchKernelGGL(adapter_plan_kernel, dim3(1), dim3(512), lds,
                     at::cuda::getCurrentCUDAStream(),
                     ids.data_ptr<int64_t>(), plan_of(plan, M, E), (int)M,
                     (int)E, (int)tiles);
  LAUNCH_OK();
  return plan;
}

static void check_rows(const torch::Tensor& t, const char* name, long M,
                       long n, const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.dim() == 2 &&
                  t.size(0) == M && t.size(1) == n &&
                  t.scalar_type() == like.scalar_type() &&
                  (n == 1 || t.stride(1) == 1),
              name, " must be rows beside the weights, of their type");
}

// Calls f with the number of 16-wide blocks of the rank, as a constant of
// 1, 2, 4 or 8.
template <typename F>
static void for_rank(long R, F&& f) {
  if (R <= 16)
    f(std::integral_constant<int, 1>());
  else if (R <= 32)
    f(std::integral_constant<int, 2>());
  else if (R <= 64)
    f(std::integral_constant<int, 4>());
  else
    f(std::integral_constant<int, 8>());
}

static long padded_rank(long R) {
  return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128;
}

static void check_weight(const torch::Tensor& w, long E) {
  TORCH_CHECK(w.is_cuda() && w.is_contiguous() && w.dim() == 3 &&
                  w.size(0) == E,
              "adapters must be contiguous [adapters, ., .] on GPU");
}

// z [M, Rp]: x [M, K] through w, [E, R, K] (kmajor) or [E, K, R].
torch::Tensor adapter_shrink(torch::Tensor x, torch::Tensor w,
                             torch::Tensor plan,
                             c10::optional<torch::Tensor> scales,
                             double scale, bool kmajor) {
  const long M = x.size(0), E = w.size(0);
  const long R = kmajor ? w.size(1) : w.size(2);
  const long K = kmajor ? w.size(2) : w.size(1);
  check_weight(w, E);
  check_rows(x, "x", M, K, w);
  TORCH_CHECK(R >= 1 && R <= RANK_MAX && K >= 1 && K < (1l << 30),
              "rank must be 1 .. 128");
  const Plan p = plan_of(plan, M, E);
  const float* sp = nullptr;
  if (scales.has_value()) {
    TORCH_CHECK(scales->device() == x.device() && scales->is_contiguous() &&
                    scales->scalar_type() == torch::kFloat32 &&
                    scales->numel() == E,
                "scale must be contiguous fp32 [adapters]");
    sp = scales->data_ptr<float>();
  }
  const at::cuda::CUDAGuard guard(x.device());
  auto z = torch::empty({M, padded_rank(R)},
                        x.options().dtype(torch::kFloat32));
  if (M == 0) return z;
  auto stream = at::cuda::getCurrentCUDAStream();
  const long tiles = max_tiles(M, E);
  for_dtype(x.scalar_type(), "x", [&](auto t) {
    using T = decltype(t);
    for_rank(R, [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      constexpr int U = RB <= 2 ? 4 : 2;
      auto go = [&](auto kernel, int waves) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)tiles),
                           dim3(waves * WAVE), 0, stream, ptr<T>(x),
                           (long)x.stride(0), ptr<T>(w), p, sp, (float)scale,
                           z.data_ptr<float>(), (int)K, (int)R, (int)E);
      };
      if (kmajor)
        go(adapter_shrink_kernel<T, RB, true, 8, U>, 8);
      else
        go(adapter_shrink_kernel<T, RB, false, 8, U>, 8);
    });
  });
  LAUNCH_OK();
  return z;
}

// act(base + z w): w [E, N, R] (rmajor) or [E, R, N]; no base: zero.
torch::Tensor adapter_expand(c10::optional<torch::Tensor> base,
                             torch::Tensor z, torch::Tensor w,
                             torch::Tensor plan, int64_t act, bool rmajor) {
  const long M = z.size(0), E = w.size(0);
  const long N = rmajor ? w.size(1) : w.size(2);
  const long R = rmajor ? w.size(2) : w.size(1);
  check_weight(w, E);
  TORCH_CHECK(R >= 1 && R <= RANK_MAX && N >= 1 && N < (1l << 30),
              "rank must be 1 .. 128");
  TORCH_CHECK(z.device() == w.device() && z.is_contiguous() &&
                  z.scalar_type() == torch::kFloat32 && z.dim() == 2 &&
                  z.size(1) == padded_rank(R),
              "z must be what adapter_shrink gave");
  if (base.has_value()) check_rows(*base, "base", M, N, w);
  const Plan p = plan_of(plan, M, E);
  const at::cuda::CUDAGuard guard(w.device());
  auto out = torch::empty({M, N}, w.options());
  if (M == 0) return out;
  auto stream = at::cuda::getCurrentCUDAStream();
  const long tiles = max_tiles(M, E);
  for_dtype(w.scalar_type(), "adapters", [&](auto t) {
    using T = decltype(t);
    const long cols = 4 * 4 * Vec<T>::N;
    for_rank(R, [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(
            kernel, dim3((unsigned)tiles, (unsigned)((N + cols - 1) / cols)),
            dim3(256), 0, stream, base.has_value() ? ptr<T>(*base) : nullptr,
            base.has_value() ? (long)base->stride(0) : 0l,
            z.data_ptr<float>(), ptr<T>(w), p, ptr<T>(out), (int)N, (int)R,
            (int)E, (int)act);
      };
      if (rmajor)
        go(adapter_expand_kernel<T, RB, true>);
      else
        go(adapter_expand_kernel<T, RB, false>);
    });
  });
  LAUNCH_OK();
  return out;
}

// [E, R, K] (kmajor) or [E, K, R]: the sums of z^T x over each adapter's
// rows.
torch::Tensor adapter_outer(torch::Tensor x, torch::Tensor z,
                            torch::Tensor plan, int64_t E, int64_t R,
                            bool kmajor) {
  const long M = z.size(0), K = x.size(1);
  check_rows(x, "x", M, K, x);
  TORCH_CHECK(R >= 1 && R <= RANK_MAX && K >= 1 && K < (1l << 30),
              "rank must be 1 .. 128");
  TORCH_CHECK(z.device() == x.device() && z.is_contiguous() &&
                  z.scalar_type() == torch::kFloat32 && z.dim() == 2 &&
                  z.size(1) == padded_rank(R),
              "z must be what adapter_shrink gave");
  const Plan p = plan_of(plan, M, E);
  const at::cuda::CUDAGuard guard(x.device());
  auto out = kmajor ? torch::empty({E, R, K}, x.options())
                    : torch::empty({E, K, R}, x.options());
  auto stream = at::cuda::getCurrentCUDAStream();
  const long tiles = max_tiles(M, E);
  // Up to 1024 rows one block adds all of an adapter's; above, stretches
  // that give about 1024 blocks, so that one busy adapter is not one block.
  const bool direct = M <= 1024;
  const long cols = 16 * (x.element_size() == 4 ? 4 : 8);
  const long chunks = (K + cols - 1) / cols;
  long stretch = 1;
  if (!direct)
    stretch = std::max<long>(4, M / TILE * chunks / 1024);
  torch::Tensor partial;
  if (!direct)
    partial = torch::empty({tiles / stretch + E + 1, R, K},
                           x.options().dtype(torch::kFloat32));
  for_dtype(x.scalar_type(), "x", [&](auto t) {
    using T = decltype(t);
    for_rank(R, [&](auto rb) {
      // ranks above 32 take turns of 32: more sums than that do not fit
      // the registers beside their operands
      constexpr int RB = decltype(rb)::value < 2 ? 1 : 2;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(
            kernel,
            dim3((unsigned)(direct ? E : tiles), (unsigned)chunks,
                 (unsigned)(padded_rank(R) / (16 * RB))),
            dim3(256), 0, stream, ptr<T>(x), (long)x.stride(0),
            z.data_ptr<float>(), (int)z.size(1), p, ptr<T>(out),
            direct ? nullptr : partial.data_ptr<float>(), (int)K, (int)R,
            (int)E, (int)stretch);
      };
      if (kmajor && direct)
        go(adapter_outer_kernel<T, RB, true, true>);
      else if (kmajor)
        go(adapter_outer_kernel<T, RB, true, false>);
      else if (direct)
        go(adapter_outer_kernel<T, RB, false, true>);
      else
        go(adapter_outer_kernel<T, RB, false, false>);
    });
    LAUNCH_OK();
    if (!direct) {
      const long n = R * K;
      hipLaunchKernelGGL((adapter_reduce_kernel<T>),
                         dim3((unsigned)std::min<long>(256, (n + 255) / 256),
                              (unsigned)E),
                         dim3(256), 0, stream, partial.data_ptr<float>(), p,
                         ptr<T>(out), n, (int)stretch);
      LAUNCH_OK();
    }
  });
  return out;
}

torch::Tensor adapter_act_bwd(torch::Tensor y, torch::Tensor dy,
                              int64_t act) {
  TORCH_CHECK(y.is_cuda() && y.is_contiguous() && dy.is_contiguous() &&
                  y.device() == dy.device() && y.sizes() == dy.sizes() &&
                  y.scalar_type() == dy.scalar_type(),
              "y and dy must be contiguous and alike on GPU");
  const at::cuda::CUDAGuard guard(y.device());
  auto dx = torch::empty_like(dy);
  const long n = dy.numel();
  if (n == 0) return dx;
  const int blocks = (int)std::min<long>(4096, (n + 255) / 256);
  for_dtype(y.scalar_type(), "y", [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((adapter_act_bwd_kernel<T>), dim3(blocks), dim3(256),
                       0, at::cuda::getCurrentCUDAStream(), ptr<T>(y),
                       ptr<T>(dy), ptr<T>(dx), n, (int)act);
  });
  LAUNCH_OK();
  return dx;
}
