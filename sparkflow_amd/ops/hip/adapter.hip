// Low-rank adapters of many requests beside a shared projection.
//
//   out_m = act(base_m + s_e (x_m A_e^T) B_e^T),  e = ids[m]
//   A [E, R, K], B [E, N, R], R small
//
//   dz_m = s_e dy_m B_e          dx_m = dz_m A_e
//   dA_e = sum_m dz_m^T x_m      dB_e = sum_m dy_m^T z_m,  z_m = s_e x_m A_e^T
//
// Rows are grouped by adapter (adapter_plan; up to 64 rows each wave does it
// by itself), and every kernel works on tiles of up to 16 rows of one
// adapter, so an adapter is read once a tile and not once a row.  z and dz
// stay in fp32, [M, Rp] in the grouped order with R padded to 16, 32, 64 or
// 128: every output is rounded once.
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

// -- rows by adapter ----------------------------------------------------------

// Groups: 0 .. E-1 the adapters, E rows without one, E + 1 rows whose id
// names none.
__device__ __forceinline__ int group_of(long id, int E) {
  return id < 0 ? E : id < E ? (int)id : E + 1;
}

// The rows in grouped order and its tiles.  Up to 64 rows nothing is
// prepared (perm is null): one wave sees all ids at once and finds the rows
// of a tile by itself, and a place is the row.
struct Plan {
  const long* ids;  // [M]
  int M, E;
  int* perm;        // [M] the row at each place of the grouped order
  int* seg;         // [E + 3] where a group's rows begin
  int* tbase;       // [E + 3] where a group's tiles begin
  int* tile_group;  // [tiles] -1 behind the last
  int* tile_place;  // [tiles] first place
};

#define SMALL_ROWS 64

// What a lane needs of a tile: its group (-1: no tile), how many rows it
// has, and the place and row of tile row lane % 16 (rows behind the last
// repeat it).
struct Tile {
  int g, rows, place, row;
};

// Tile t of a prepared plan, moved on by `sub` tiles of its group; the
// caller makes sure that the group has them.
__device__ __forceinline__ Tile plan_tile(const Plan& p, int t, int sub,
                                          int lane) {
  Tile r = {p.tile_group[t], 0, 0, 0};
  if (r.g < 0) return r;
  const int first = p.tile_place[t] + sub * TILE;
  r.rows = min(TILE, p.seg[r.g + 1] - first);
  r.place = first + min(lane & 15, r.rows - 1);
  r.row = p.perm[r.place];
  return r;
}

// The tile that begins with row t, if one does: of the rows with t's group,
// every sixteenth begins a tile.
__device__ __forceinline__ Tile small_tile(const Plan& p, int t, int lane) {
  const int of = lane < p.M ? group_of(p.ids[lane], p.E) : -1;
  Tile r = {__shfl(of, t, WAVE), 0, 0, 0};
  unsigned long same = __ballot(of == r.g);
  if (__popcll(same & ((1ul << t) - 1)) % TILE != 0) {
    r.g = -1;
    return r;
  }
  same = same >> t << t;
  r.rows = min(TILE, (int)__popcll(same));
  const int i = min(lane & 15, r.rows - 1);
  for (int j = 0; j < TILE - 1; ++j)
    if (j < i) same &= same - 1;
  r.row = r.place = __ffsll((unsigned long long)same) - 1;
  return r;
}

// Lanes of the wave with this lane's group: one ballot for each bit.
__device__ __forceinline__ unsigned long same_group(int g, int bits) {
  unsigned long same = ~0ul;
  for (int b = 0; b < bits; ++b) {
    const bool set = (g >> b) & 1;
    const unsigned long with = __ballot(set);
    same &= set ? with : ~with;
  }
  return same;
}

#define PLAN_WAVES 16
#define PLAN_BATCH 8

// A stable counting sort in one block.  Each wave owns a stretch of the
// rows and counts it for itself, so that no order depends on timing.  It is
// bound by latency: a wave loads 8 x 64 ids ahead of using them, and ranks
// 64 rows at once (8192 rows of 8 or 32 adapters, shuffled or in runs: one
// batch a wave).
__global__ void __launch_bounds__(PLAN_WAVES* WAVE)
    adapter_plan_kernel(Plan p, int tiles, int waves) {
  extern __shared__ int hist[];  // [waves][E + 2] and [E + 3]
  const int M = p.M, E = p.E, G = E + 2;
  int* total = hist + waves * G;
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid & (WAVE - 1);
  const int threads = waves * WAVE;
  const int bits = 32 - __clz(G);
  for (int i = tid; i < waves * G; i += threads) hist[i] = 0;
  const int stretch = (M + threads - 1) / threads * WAVE;
  const int lo = wave * stretch;
  const int hi = min(M, lo + stretch);
  int* mine = hist + wave * G;
  int of[PLAN_BATCH], peer[PLAN_BATCH];  // group; first lane and rank in it
  auto fetch = [&](int i0) {
    long id[PLAN_BATCH];
#pragma unroll
    for (int u = 0; u < PLAN_BATCH; ++u) {
      const int i = i0 + u * WAVE + lane;
      id[u] = i < hi ? p.ids[i] : 0;
    }
#pragma unroll
    for (int u = 0; u < PLAN_BATCH; ++u)
      of[u] = i0 + u * WAVE + lane < hi ? group_of(id[u], E) : -1;
#pragma unroll
    for (int u = 0; u < PLAN_BATCH; ++u) {
      if (i0 + u * WAVE >= hi) break;
      const unsigned long same = same_group(of[u], bits);
      peer[u] = (__ffsll((unsigned long long)same) - 1) |
                __popcll(same & ((1ul << lane) - 1)) << 8 |
                __popcll(same) << 16;
    }
  };
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += PLAN_BATCH * WAVE) {
    fetch(i0);
#pragma unroll
    for (int u = 0; u < PLAN_BATCH; ++u) {
      if (i0 + u * WAVE >= hi) break;
      if (of[u] >= 0 && (peer[u] & 255) == lane)
        atomicAdd(&mine[of[u]], peer[u] >> 16);
    }
  }
  __syncthreads();
  // per group: the waves' counts become offsets, their sum the total
  for (int g = tid; g < G; g += threads) {
    int sum = 0;
    for (int w = 0; w < waves; ++w) {
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
      if (g < G) {
        p.seg[g] = total[g] = rows + cs - c;
        p.tbase[g] = blocks + bs - b;
      }
      rows += __shfl(cs, WAVE - 1, WAVE);
      blocks += __shfl(bs, WAVE - 1, WAVE);
    }
    if (lane == 0) {
      p.seg[G] = total[G] = rows;
      p.tbase[G] = blocks;
    }
    for (int t = blocks + lane; t < tiles; t += WAVE) p.tile_group[t] = -1;
  }
  __syncthreads();
  // a wave a group writes its tiles
  for (int g = wave; g < G; g += waves) {
    const int r0 = total[g], b0 = p.tbase[g];
    const int b = (total[g + 1] - r0 + TILE - 1) / TILE;
    for (int j = lane; j < b; j += WAVE) {
      p.tile_group[b0 + j] = g;
      p.tile_place[b0 + j] = r0 + j * TILE;
    }
  }
  // each wave places its stretch in order
  for (int i0 = lo; i0 < hi; i0 += PLAN_BATCH * WAVE) {
    if (hi - lo > PLAN_BATCH * WAVE) fetch(i0);  // else it holds them yet
#pragma unroll
    for (int u = 0; u < PLAN_BATCH; ++u) {
      if (i0 + u * WAVE >= hi) break;
      const int first = peer[u] & 255;
      int at = 0;
      if (of[u] >= 0 && first == lane)
        at = total[of[u]] + atomicAdd(&mine[of[u]], peer[u] >> 16);
      at = __shfl(at, first, WAVE);
      if (of[u] >= 0)
        p.perm[at + (peer[u] >> 8 & 255)] = i0 + u * WAVE + lane;
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
// [K, R].  One block takes SUB tiles of an adapter, which share its loads of
// W; its waves take turns along k and meet in LDS.
template <typename T, int RB, bool KMAJOR, bool SMALL, int WAVES, int SUB,
          int U>
__global__ void __launch_bounds__(WAVES * WAVE)
    adapter_shrink_kernel(const T* __restrict__ x, long xstride,
                          const T* __restrict__ w, Plan p,
                          const float* __restrict__ scales, float scale,
                          float* __restrict__ z, int K, int R) {
  constexpr int N = Vec<T>::N;
  constexpr int STEP = 4 * N;  // k of one wave
  typedef typename Vec<T>::V V;
  __shared__ f32x4 part[WAVES][SUB * RB][WAVE];
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  Tile t[SUB];
  if (SMALL) {
    t[0] = small_tile(p, blockIdx.x, lane);
    if (t[0].g < 0 || t[0].g >= p.E) return;
  } else {
    const int g = p.tile_group[blockIdx.x];
    if (g < 0 || g >= p.E) return;
    const int at = blockIdx.x - p.tbase[g];
    if (at % SUB != 0) return;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      // a tile that the group does not have repeats the first, unwritten
      const bool has = (int)blockIdx.x + s < p.tbase[g + 1];
      t[s] = plan_tile(p, blockIdx.x, has ? s : 0, lane);
      if (!has) t[s].rows = 0;
    }
  }
  const int g = t[0].g;
  const int i = lane & 15, quarter = lane >> 4;
  // ranks behind R repeat the last; they are written as zero
  const T* xr[SUB];
#pragma unroll
  for (int s = 0; s < SUB; ++s) xr[s] = x + (long)t[s].row * xstride;
  const T* we = w + (long)g * R * K;
  auto load_w = [&](int rb, int k) -> V {
    const int r = min(rb * 16 + i, R - 1);
    if (KMAJOR) return Vec<T>::load(we + (long)r * K + k);
    V v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = we[(long)(k + j) * R + r];
    return v;
  };
  f32x4 acc[SUB][RB] = {};
  const int whole = K / (STEP * U);
  for (int c = wave; c < whole; c += WAVES) {
    V xv[U][SUB], wv[U][RB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (c * U + u) * STEP + quarter * N;
#pragma unroll
      for (int s = 0; s < SUB; ++s) xv[u][s] = Vec<T>::load(xr[s] + k);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) wv[u][rb] = load_w(rb, k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          acc[s][rb] = mma(xv[u][s], wv[u][rb], acc[s][rb]);
  }
  for (int k0 = whole * (STEP * U) + wave * STEP; k0 < K;
       k0 += WAVES * STEP) {
    const int k = k0 + quarter * N;
    V xv[SUB], wv[RB];
    if (k + N <= K) {
#pragma unroll
      for (int s = 0; s < SUB; ++s) xv[s] = Vec<T>::load(xr[s] + k);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) wv[rb] = load_w(rb, k);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int s = 0; s < SUB; ++s)
          xv[s][j] = k + j < K ? xr[s][k + j] : (T)0.0f;
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
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        acc[s][rb] = mma(xv[s], wv[rb], acc[s][rb]);
  }
#pragma unroll
  for (int s = 0; s < SUB; ++s)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      part[wave][s * RB + rb][lane] = acc[s][rb];
  __syncthreads();
  const float f = scales ? scales[g] : scale;
  // whole waves: a wave's 64 lanes finish the 16 x 16 of one (s, rb)
  for (int b = wave; b < SUB * RB; b += WAVES) {
    f32x4 sum = part[0][b][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) sum += part[v][b][lane];
    const int r = b % RB * 16 + i;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      if (b / RB != s) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = quarter * 4 + q;
        const long place = __shfl(t[s].place, m, WAVE);
        if (m < t[s].rows)
          z[place * (RB * 16) + r] = r < R ? f * sum[q] : 0.0f;
      }
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
// (RMAJOR) or [R, N].  One block takes 16 V columns of up to WAVES tiles of
// an adapter, a wave a tile, and lays its part of W into LDS once as [n][r].
// The product is taken as D[n][m], in fp32; instruction j's row 4 h + q is
// column 4 V a + V h + e of the block's, where j = a V / 4 + e / 4 and
// q = e % 4, so that a lane ends up with 16 bytes of adjacent outputs and
// its row's four lanes with 64.  base enters as the sum's first term.
template <typename T, int RB, bool RMAJOR, int WAVES>
__global__ void __launch_bounds__(WAVES * WAVE)
    adapter_expand_kernel(const T* __restrict__ base, long bstride,
                          const float* __restrict__ z,
                          const T* __restrict__ w, Plan p,
                          T* __restrict__ out, int N, int R, int act) {
  constexpr int V = Vec<T>::N;
  constexpr int COLS = 16 * V;
  constexpr int PITCH = 16 * RB + 16 / sizeof(T);  // of a column in LDS
  constexpr bool SMALL = WAVES == 1;
  typedef typename Vec<T>::V VT;
  typedef T T4 __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) T wl[COLS * PITCH];
  const int tid = threadIdx.x;
  const int lane = tid & (WAVE - 1), wave = tid / WAVE;
  const int i = lane & 15, quarter = lane >> 4;
  const int n0 = blockIdx.y * COLS;
  Tile t;
  int g;
  bool has = true;
  if (SMALL) {
    t = small_tile(p, blockIdx.x, lane);
    g = t.g;
    if (g < 0) return;
  } else {
    g = p.tile_group[blockIdx.x];
    if (g < 0 || (blockIdx.x - p.tbase[g]) % WAVES != 0) return;
    has = (int)blockIdx.x + wave < p.tbase[g + 1];
    t = plan_tile(p, blockIdx.x, has ? wave : 0, lane);
  }
  const bool mine = has && i < t.rows;
  const int out0 = n0 + V * quarter;
  VT bv[4];
  if (base != nullptr && mine) {
    const T* br = base + (long)t.row * bstride + out0;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (out0 + 4 * V * a + V <= N) {
        bv[a] = Vec<T>::load(br + 4 * V * a);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          bv[a][e] = out0 + 4 * V * a + e < N ? br[4 * V * a + e] : (T)0.0f;
      }
    }
  }
  f32x4 zv[RB];
  if (g < p.E) {
#pragma unroll
    for (int c = 0; c < RB; ++c)
      zv[c] = *reinterpret_cast<const f32x4*>(
          z + (long)t.place * (RB * 16) + 16 * c + 4 * quarter);
    const T* we = w + (long)g * N * R;
    if (RMAJOR) {
      // ranks in fours: a vector where the rank has all four
      for (int at = tid; at < COLS * 4 * RB; at += WAVES * WAVE) {
        const int c = at / (4 * RB), r = at % (4 * RB) * 4;
        const T* wr = we + (long)min(n0 + c, N - 1) * R + r;
        T4 v;
        if (r + 4 <= R) {
          struct __attribute__((packed, aligned(sizeof(T)))) U4 {
            T4 v;
          };
          v = reinterpret_cast<const U4*>(wr)->v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = r + e < R ? wr[e] : (T)0.0f;
        }
        *reinterpret_cast<T4*>(&wl[c * PITCH + r]) = v;
      }
    } else {
      for (int at = tid; at < 16 * RB * 16; at += WAVES * WAVE) {
        const int r = at / 16, c = at % 16 * V;
        const T* wr = we + (long)min(r, R - 1) * N + n0 + c;
        VT v;
        if (n0 + c + V <= N) {
          v = Vec<T>::load(wr);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            v[e] = n0 + c + e < N ? wr[e] : (T)0.0f;
        }
#pragma unroll
        for (int e = 0; e < V; ++e)
          wl[(c + e) * PITCH + r] = r < R ? v[e] : (T)0.0f;
      }
    }
  }
  __syncthreads();
  f32x4 acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    constexpr int H = V / 4;  // instructions to a vector of the output
#pragma unroll
    for (int q = 0; q < 4; ++q)
      acc[j][q] = base != nullptr ? (float)bv[j / H][4 * (j % H) + q] : 0.0f;
    if (g < p.E) {
      const int c = 4 * V * (j / H) + V * (i >> 2) + 4 * (j % H) + (i & 3);
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const T4 v = *reinterpret_cast<const T4*>(
            &wl[c * PITCH + 16 * b + 4 * quarter]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
              (float)v[e], zv[b][e], acc[j], 0, 0, 0);
      }
    }
  }
  if (!mine) return;
  T* o = out + (long)t.row * N + out0;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    VT v;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float y = g > p.E ? NAN : acc[a * (V / 4) + e / 4][e % 4];
      v[e] = (T)act_keep_nan(y, act);
    }
    if (out0 + 4 * V * a + V <= N) {
      Vec<T>::store(o + 4 * V * a, v);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (out0 + 4 * V * a + e < N) o[4 * V * a + e] = v[e];
    }
  }
}

// -- outer --------------------------------------------------------------------

enum OuterWork { SMALL_OUTER, DIRECT_OUTER, SPLIT_OUTER };

// Where adapter e's stretches of `stretch` tiles begin among all stretches.
// (t / stretch + e is another one for each stretch's first tile t.)
__device__ __forceinline__ int first_slot(const Plan& p, int e,
                                          int stretch) {
  return p.tbase[e] / stretch + e;
}

// sum over the rows of a stretch of one adapter: z[place][r] x[row][k], with
// fp32 products.  A lane loads 16 bytes of a row; instruction j takes
// element j of all lanes, so its 16 columns are k0 + V (l % 16) + j and its
// four k are four rows.  KMAJOR: the result is [R, K] (dA), else [K, R]
// (dB).  SMALL_OUTER, DIRECT_OUTER: one block an adapter, rounded into out;
// SPLIT_OUTER: one block a stretch, into fp32 sums that reduce joins.
template <typename T, int RB, bool KMAJOR, OuterWork WORK>
__global__ void __launch_bounds__(256)
    adapter_outer_kernel(const T* __restrict__ x, long xstride,
                         const float* __restrict__ z, int zstride, Plan p,
                         T* __restrict__ out, float* __restrict__ partial,
                         int K, int R, int stretch) {
  constexpr int V = Vec<T>::N;
  constexpr int U = 4;
  __shared__ f32x4 part[2][RB * V][WAVE];
  __shared__ int list[SMALL_ROWS];
  __shared__ int found;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int i = lane & 15, quarter = lane >> 4;
  int begin = 0, end = 0;
  if (WORK == SMALL_OUTER) {
    const bool here = lane < p.M && p.ids[lane] == (long)blockIdx.x;
    const unsigned long all = __ballot(here);
    if (here && wave == 0) list[__popcll(all & ((1ul << lane) - 1))] = lane;
    end = __popcll(all);
    __syncthreads();
  } else if (WORK == DIRECT_OUTER) {
    begin = p.seg[blockIdx.x];
    end = p.seg[blockIdx.x + 1];
  } else {
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += 256) {
      const int c = (int)blockIdx.x - first_slot(p, e, stretch);
      const int n = p.tbase[e + 1] - p.tbase[e];
      if (c >= 0 && c * stretch < n) {
        found = e;
        list[0] = p.tile_place[p.tbase[e] + c * stretch];
      }
    }
    __syncthreads();
    if (found < 0) return;
    begin = list[0];
    end = min(p.seg[found + 1], begin + stretch * TILE);
  }
  const int r0 = blockIdx.z * (RB * 16);
  const int k0 = blockIdx.y * (16 * V);
  const int k = k0 + i * V;
  f32x4 acc[RB][V] = {};
  // Four rows an instruction, U times four a step.  The next step's rows
  // are loaded before this one's products, and their numbers a step before
  // that.
  int place[U], row[U];
  auto number = [&](int m0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(m0 + 4 * u + quarter, end - 1);
      place[u] = WORK == SMALL_OUTER ? list[at] : at;
      row[u] = WORK == SMALL_OUTER ? place[u] : p.perm[at];
    }
  };
  typename Vec<T>::V xv[U], xn[U];
  float zv[U][RB], zn[U][RB];
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* xr = x + (long)row[u] * xstride;
      if (k + V <= K) {
        xn[u] = Vec<T>::load(xr + k);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          xn[u][j] = k + j < K ? xr[k + j] : (T)0.0f;
      }
#pragma unroll
      for (int c = 0; c < RB; ++c)
        zn[u][c] = z[(long)place[u] * zstride + r0 + 16 * c + i];
    }
  };
  constexpr int STEP = 16 * U;
  int m0 = begin + wave * 4 * U;
  if (m0 < end) {
    number(m0);
    load();
    number(m0 + STEP);
  }
  for (; m0 < end; m0 += STEP) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = m0 + 4 * u + quarter < end;
      // rows behind the last: both factors, since 0 x NaN is not 0
#pragma unroll
      for (int j = 0; j < V; ++j) xv[u][j] = in ? xn[u][j] : (T)0.0f;
#pragma unroll
      for (int c = 0; c < RB; ++c) zv[u][c] = in ? zn[u][c] : 0.0f;
    }
    if (m0 + STEP < end) {
      load();
      number(m0 + 2 * STEP);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < RB; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j)
          acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
              zv[u][c], (float)xv[u][j], acc[c][j], 0, 0, 0);
  }
  // the four waves' sums meet in the first
#pragma unroll
  for (int half = 2; half > 0; half >>= 1) {
    __syncthreads();
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int c = 0; c < RB; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j)
          part[wave - half][c * V + j][lane] = acc[c][j];
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
  const long o0 = (long)blockIdx.x * R * K;
#pragma unroll
  for (int c = 0; c < RB; ++c)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = r0 + 16 * c + 4 * quarter + q;
      if (r >= R) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (k + j >= K) continue;
        const long o = o0 + (KMAJOR ? (long)r * K + k + j
                                    : (long)(k + j) * R + r);
        if (WORK == SPLIT_OUTER)
          partial[o] = acc[c][j][q];
        else
          out[o] = (T)acc[c][j][q];
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
  const int tiles = p.tbase[e + 1] - p.tbase[e];
  const int slots = (tiles + stretch - 1) / stretch;
  const float* from = partial + (long)first_slot(p, e, stretch) * n;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (long)gridDim.x * 256) {
    float sum = 0.0f;
    for (int s = 0; s < slots; ++s) sum += from[s * n + i];
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

static long plan_size(long M, long E) {
  return M <= SMALL_ROWS ? 0 : M + 2 * (E + 3) + 2 * max_tiles(M, E);
}

// perm, seg, tbase, tile_group, tile_place in one int32 tensor.
static Plan plan_of(const torch::Tensor& ids, const torch::Tensor& plan,
                    long E) {
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() && ids.dim() == 1 &&
                  ids.scalar_type() == torch::kInt64 &&
                  ids.size(0) < (1l << 30),
              "ids must be contiguous int64 [rows] on GPU");
  TORCH_CHECK(E >= 1 && E <= ADAPTERS_MAX, "1 .. 1024 adapters");
  const long M = ids.size(0);
  TORCH_CHECK(plan.device() == ids.device() && plan.is_contiguous() &&
                  plan.scalar_type() == torch::kInt32 &&
                  plan.numel() == plan_size(M, E),
              "plan does not belong to these rows and adapters");
  Plan r = {ids.data_ptr<int64_t>(), (int)M, (int)E, nullptr, nullptr,
            nullptr, nullptr, nullptr};
  if (M > SMALL_ROWS) {
    r.perm = plan.data_ptr<int>();
    r.seg = r.perm + M;
    r.tbase = r.seg + E + 3;
    r.tile_group = r.tbase + E + 3;
    r.tile_place = r.tile_group + max_tiles(M, E);
  }
  return r;
}

// Empty up to 64 rows.
torch::Tensor adapter_plan(torch::Tensor ids, int64_t E) {
  const long M = ids.size(0);
  const at::cuda::CUDAGuard guard(ids.device());
  TORCH_CHECK(E >= 1 && E <= ADAPTERS_MAX, "1 .. 1024 adapters");
  auto plan = torch::empty({plan_size(M, E)},
                           ids.options().dtype(torch::kInt32));
  const Plan p = plan_of(ids, plan, E);
  if (M <= SMALL_ROWS) return plan;
  // 16 waves while their counts fit 48 KB of LDS, else 8
  const int waves = PLAN_WAVES * (E + 2) + E + 3 <= 12288 ? PLAN_WAVES : 8;
  const int lds = (int)((waves * (E + 2) + E + 3) * sizeof(int));
  hipLaunchKernelGGL(adapter_plan_kernel, dim3(1), dim3(waves * WAVE), lds,
                     at::cuda::getCurrentCUDAStream(), p,
                     (int)max_tiles(M, E), waves);
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

static float* check_z(const torch::Tensor& z, const torch::Tensor& like,
                      long M, long R) {
  TORCH_CHECK(R >= 1 && R <= RANK_MAX, "rank must be 1 .. 128");
  TORCH_CHECK(z.device() == like.device() && z.is_contiguous() &&
                  z.scalar_type() == torch::kFloat32 && z.dim() == 2 &&
                  z.size(0) == M && z.size(1) == padded_rank(R),
              "z must be what adapter_shrink gave");
  return z.data_ptr<float>();
}

// z [M, Rp]: x [M, K] through w, [E, R, K] (kmajor) or [E, K, R].
torch::Tensor adapter_shrink(torch::Tensor x, torch::Tensor w,
                             torch::Tensor ids, torch::Tensor plan,
                             c10::optional<torch::Tensor> scales,
                             double scale, bool kmajor) {
  const long M = x.size(0), E = w.size(0);
  check_weight(w, E);
  const long R = kmajor ? w.size(1) : w.size(2);
  const long K = kmajor ? w.size(2) : w.size(1);
  check_rows(x, "x", M, K, w);
  TORCH_CHECK(R >= 1 && R <= RANK_MAX, "rank must be 1 .. 128");
  TORCH_CHECK(K >= 1 && K < (1l << 30), "inputs must be 1 .. 2^30");
  const Plan p = plan_of(ids, plan, E);
  TORCH_CHECK(p.M == M && ids.device() == x.device(),
              "ids must be one a row beside x");
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
  const bool small = M <= SMALL_ROWS;
  const long tiles = small ? M : max_tiles(M, E);
  for_dtype(x.scalar_type(), "x", [&](auto t) {
    using T = decltype(t);
    for_rank(R, [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      // loads of 16 bytes that a lane has in flight: U (SUB + RB)
      constexpr int U = RB == 1 ? 8 : RB == 2 ? 4 : 2;
      constexpr int MANY = RB <= 4 ? 16 : 8;  // waves whose sums fit the LDS
      auto go = [&](auto kernel, int waves) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)tiles),
                           dim3(waves * WAVE), 0, stream, ptr<T>(x),
                           (long)x.stride(0), ptr<T>(w), p, sp, (float)scale,
                           z.data_ptr<float>(), (int)K, (int)R);
      };
      auto pick = [&](auto major) {
        constexpr bool KM = decltype(major)::value;
        if (small)
          go(adapter_shrink_kernel<T, RB, KM, true, MANY, 1, U>, MANY);
        else
          go(adapter_shrink_kernel<T, RB, KM, false, 8, 1, U>, 8);
      };
      if (kmajor)
        pick(std::true_type());
      else
        pick(std::false_type());
    });
  });
  LAUNCH_OK();
  return z;
}

// act(base + z w): w [E, N, R] (rmajor) or [E, R, N]; no base: zero.
torch::Tensor adapter_expand(c10::optional<torch::Tensor> base,
                             torch::Tensor z, torch::Tensor w,
                             torch::Tensor ids, torch::Tensor plan,
                             int64_t act, bool rmajor) {
  const long M = z.size(0), E = w.size(0);
  check_weight(w, E);
  const long N = rmajor ? w.size(1) : w.size(2);
  const long R = rmajor ? w.size(2) : w.size(1);
  TORCH_CHECK(N >= 1 && N < (1l << 30), "outputs must be 1 .. 2^30");
  const float* zp = check_z(z, w, M, R);
  if (base.has_value()) check_rows(*base, "base", M, N, w);
  const Plan p = plan_of(ids, plan, E);
  TORCH_CHECK(p.M == M && ids.device() == w.device(),
              "ids must be one a row beside the adapters");
  const at::cuda::CUDAGuard guard(w.device());
  auto out = torch::empty({M, N}, w.options());
  if (M == 0) return out;
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool small = M <= SMALL_ROWS;
  const long tiles = small ? M : max_tiles(M, E);
  for_dtype(w.scalar_type(), "adapters", [&](auto t) {
    using T = decltype(t);
    const long cols = 16 * Vec<T>::N;
    for_rank(R, [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      auto go = [&](auto kernel, int waves) {
        hipLaunchKernelGGL(
            kernel,
            dim3((unsigned)tiles, (unsigned)((N + cols - 1) / cols)),
            dim3(waves * WAVE), 0, stream,
            base.has_value() ? ptr<T>(*base) : nullptr,
            base.has_value() ? (long)base->stride(0) : 0l, zp, ptr<T>(w), p,
            ptr<T>(out), (int)N, (int)R, (int)act);
      };
      if (rmajor && small)
        go(adapter_expand_kernel<T, RB, true, 1>, 1);
      else if (rmajor)
        go(adapter_expand_kernel<T, RB, true, 4>, 4);
      else if (small)
        go(adapter_expand_kernel<T, RB, false, 1>, 1);
      else
        go(adapter_expand_kernel<T, RB, false, 4>, 4);
    });
  });
  LAUNCH_OK();
  return out;
}

// [E, R, K] (kmajor) or [E, K, R]: the sums of z^T x over each adapter's
// rows.
torch::Tensor adapter_outer(torch::Tensor x, torch::Tensor z,
                            torch::Tensor ids, torch::Tensor plan, int64_t E,
                            int64_t R, bool kmajor) {
  const long M = z.size(0), K = x.size(1);
  check_rows(x, "x", M, K, x);
  TORCH_CHECK(K >= 1 && K < (1l << 30), "inputs must be 1 .. 2^30");
  const float* zp = check_z(z, x, M, R);
  const Plan p = plan_of(ids, plan, E);
  TORCH_CHECK(p.M == M && ids.device() == x.device(),
              "ids must be one a row beside x");
  const at::cuda::CUDAGuard guard(x.device());
  auto out = kmajor ? torch::empty({E, R, K}, x.options())
                    : torch::empty({E, K, R}, x.options());
  auto stream = at::cuda::getCurrentCUDAStream();
  const long tiles = max_tiles(M, E);
  // Up to 1024 rows one block adds all of an adapter's; above, stretches
  // that give about 1024 blocks, so that one busy adapter is not one block.
  const bool small = M <= SMALL_ROWS, direct = M <= 1024;
  const long cols = 16 * (x.element_size() == 4 ? 4 : 8);
  const long chunks = (K + cols - 1) / cols;
  const long stretch =
      direct ? 1 : std::max<long>(4, M / TILE * chunks / 1024);
  const long slots = direct ? E : tiles / stretch + E;
  torch::Tensor partial;
  if (!direct)
    partial = torch::empty({slots, R, K}, x.options().dtype(torch::kFloat32));
  for_dtype(x.scalar_type(), "x", [&](auto t) {
    using T = decltype(t);
    for_rank(R, [&](auto rb) {
      // ranks above 32 take turns of 32: more sums than that do not fit
      // the registers beside their operands
      constexpr int RB = decltype(rb)::value < 2 ? 1 : 2;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(
            kernel,
            dim3((unsigned)slots, (unsigned)chunks,
                 (unsigned)(padded_rank(R) / (16 * RB))),
            dim3(256), 0, stream, ptr<T>(x), (long)x.stride(0), zp,
            (int)z.size(1), p, ptr<T>(out),
            direct ? nullptr : partial.data_ptr<float>(), (int)K, (int)R,
            (int)stretch);
      };
      auto pick = [&](auto major) {
        constexpr bool KM = decltype(major)::value;
        if (small)
          go(adapter_outer_kernel<T, RB, KM, SMALL_OUTER>);
        else if (direct)
          go(adapter_outer_kernel<T, RB, KM, DIRECT_OUTER>);
        else
          go(adapter_outer_kernel<T, RB, KM, SPLIT_OUTER>);
      };
      if (kmajor)
        pick(std::true_type());
      else
        pick(std::false_type());
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
