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
// 128: every output is rounded once (what an activation adds to that is at
// adapter_act_bwd).
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
// so that no launch has 2^32 threads: 512 for each tile
#define ROWS_MAX (1l << 26)

// -- rows by adapter ----------------------------------------------------------

// Groups: 0 .. E-1 the adapters, E rows without one, E + 1 rows whose id
// names none.
__device__ __forceinline__ int group_of(long id, int E) {
  const int high = (int)(id >> 32);
  const unsigned low = (unsigned)id;
  return high < 0 ? E : high == 0 && low < (unsigned)E ? (int)low : E + 1;
}

// The rows in grouped order and its tiles.  Up to 64 rows nothing is
// prepared (perm is null): one wave sees all ids at once and finds the rows
// of a tile by itself, and a place is the row.
struct Plan {
  const long* ids;  // [M]
  int M, E;
  int4* tiles;   // up to 16 rows: group (-1 behind the last), first place, rows
  int4* blocks;  // up to 64 rows, the same
  int* perm;     // [M] the row at each place of the grouped order
  int* seg;      // [E + 3] where a group's rows begin
  int* tbase;    // [E + 3] where its tiles begin
};

#define BLOCK_TILES 4  // tiles of a block

#define SMALL_ROWS 64

// What a lane needs of a tile: its group (-1: no tile), how many rows it
// has, and the place and row of tile row lane % 16 (rows behind the last
// repeat it).
struct Tile {
  int g, rows, place, row;
};

// Tile `sub` of the rows that an entry of the plan names.
__device__ __forceinline__ Tile plan_tile(const Plan& p, int4 of, int sub,
                                          int lane) {
  Tile r = {of.x, min(TILE, of.z - sub * TILE), 0, 0};
  r.place = of.y + sub * TILE + min(lane & 15, r.rows - 1);
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
  unsigned low = ~0u, high = ~0u;
  for (int b = 0; b < bits; ++b) {
    const unsigned set = (unsigned)(-((g >> b) & 1));
    const unsigned long with = __ballot(set != 0);
    low &= ~((unsigned)with ^ set);
    high &= ~((unsigned)(with >> 32) ^ set);
  }
  return (unsigned long)high << 32 | low;
}

#define PLAN_WAVES 16
#define PLAN_BATCH 8

// A stable counting sort in one block.  Each wave owns a stretch of the
// rows and counts it for itself, so that no order depends on timing.  It is
// bound by latency on its one CU: a wave loads 8 x 64 ids ahead of using
// them, and ranks 64 rows at once, by a ballot for each bit of the group (a
// loop over the groups present: 38 us for 9.9 at 8192 rows of 8 adapters;
// 300 rows: 4.2 us).  A wave holds the ranks of 8 x 64 rows; from 8193 rows
// on every id is loaded and ranked a second time (8256 rows 14.3 us, 65536
// 72, 2^20 1.1 ms).  Layers that share their rows share it: adapter_groups.
__global__ void __launch_bounds__(PLAN_WAVES* WAVE)
    adapter_plan_kernel(Plan p, int tiles, int blocks, int waves) {
  extern __shared__ int hist[];  // [waves][E + 2] and three of [E + 3]
  const int M = p.M, E = p.E, G = E + 2;
  int* total = hist + waves * G;
  int* tbase = total + G + 1;
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
      const unsigned rank = __builtin_amdgcn_mbcnt_hi(
          (unsigned)(same >> 32),
          __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
      peer[u] = (__ffsll((unsigned long long)same) - 1) | rank << 8 |
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
  int* bbase = tbase + G + 1;
  if (wave == 0) {
    int rows = 0, nt = 0, nb = 0;
    for (int g0 = 0; g0 < G; g0 += WAVE) {
      const int g = g0 + lane;
      const int c = g < G ? total[g] : 0;
      const int t = (c + TILE - 1) / TILE;
      const int b = (t + BLOCK_TILES - 1) / BLOCK_TILES;
      int cs = c, ts = t, bs = b;
#pragma unroll
      for (int off = 1; off < WAVE; off <<= 1) {
        const int cu = __shfl_up(cs, off, WAVE);
        const int tu = __shfl_up(ts, off, WAVE);
        const int bu = __shfl_up(bs, off, WAVE);
        if (lane >= off) {
          cs += cu;
          ts += tu;
          bs += bu;
        }
      }
      if (g < G) {
        p.seg[g] = total[g] = rows + cs - c;
        p.tbase[g] = tbase[g] = nt + ts - t;
        bbase[g] = nb + bs - b;
      }
      rows += __shfl(cs, WAVE - 1, WAVE);
      nt += __shfl(ts, WAVE - 1, WAVE);
      nb += __shfl(bs, WAVE - 1, WAVE);
    }
    if (lane == 0) {
      p.seg[G] = total[G] = rows;
      p.tbase[G] = tbase[G] = nt;
      bbase[G] = nb;
    }
  }
  __syncthreads();
  // a wave a group writes its tiles and blocks
  for (int g = wave; g < G; g += waves) {
    const int r0 = total[g], n = total[g + 1] - r0;
    for (int j = lane; j * TILE < n; j += WAVE)
      p.tiles[tbase[g] + j] =
          make_int4(g, r0 + j * TILE, min(TILE, n - j * TILE), 0);
    constexpr int ROWS = BLOCK_TILES * TILE;
    for (int j = lane; j * ROWS < n; j += WAVE)
      p.blocks[bbase[g] + j] =
          make_int4(g, r0 + j * ROWS, min(ROWS, n - j * ROWS), 0);
  }
  for (int t = tbase[G] + tid; t < tiles; t += threads)
    p.tiles[t] = make_int4(-1, 0, 0, 0);
  for (int t = bbase[G] + tid; t < blocks; t += threads)
    p.blocks[t] = make_int4(-1, 0, 0, 0);
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

// bf16 has the exponents of fp32, so three of them hold an fp32 number's 24
// bits exactly: products of z with bf16 weights or rows go through the bf16
// instruction three times at an eighth of the fp32 instruction's time each.
// (fp16 has not the exponents: three of them would hold z only after a
// scaling of each row, and its products are taken in fp32.)
struct Split {
  Vec<bf16_t>::V high, mid, low;
};

__device__ __forceinline__ Split split(const float (&x)[8]) {
  Split s;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    s.high[j] = (bf16_t)x[j];
    // an infinity has no rest: inf - inf would make it NaN
    const float a = fabsf(x[j]) <= 3.0e38f ? x[j] - (float)s.high[j] : 0.0f;
    s.mid[j] = (bf16_t)a;
    s.low[j] = (bf16_t)(a - (float)s.mid[j]);
  }
  return s;
}

// -- shrink -------------------------------------------------------------------

// z[place][r] = s_e sum_k x[row][k] W_e(r, k).  W is [R, K] (KMAJOR) or
// [K, R].  One block takes SUB tiles of an adapter, which share its loads of
// W; its waves take turns along k and meet in LDS.  Both factors go from
// memory to the matrix instruction without LDS: 16 bytes of a lane are its
// operand.  Bound by what is under way: 8192 rows of 4096 bf16 (67 MB) at a
// rank of 16 take 18 us, 3.7 TB/s, of which 4 are the way from the plan to
// the first row; a plain read of as much takes 12.  A few rows may be split
// over blocks along k too (gridDim.y): each writes a plane of z of its own,
// and expand adds them up.
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
  } else if (SUB == 1) {
    const int4 of = p.tiles[blockIdx.x];
    if (of.x < 0 || of.x >= p.E) return;
    t[0] = plan_tile(p, of, 0, lane);
  } else {
    constexpr int PARTS = BLOCK_TILES / SUB;
    const int4 of = p.blocks[blockIdx.x / PARTS];
    const int first = blockIdx.x % PARTS * SUB;
    if (of.x < 0 || of.x >= p.E || first * TILE >= of.z) return;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      // a tile that is not there repeats the first and is not written
      const bool has = (first + s) * TILE < of.z;
      t[s] = plan_tile(p, of, has ? first + s : first, lane);
      if (!has) t[s].rows = 0;
    }
  }
  const int i = lane & 15, quarter = lane >> 4;
  // ranks behind R repeat the last; they are written as zero
  const T* xr[SUB];
#pragma unroll
  for (int s = 0; s < SUB; ++s) xr[s] = x + (long)t[s].row * xstride;
  const T* we = w + (long)t[0].g * R * K;
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
  // Every block starts elsewhere in its rows: rows lie a power of two apart
  // as a rule, and blocks that walk them in step meet in a few channels of
  // the memory.
  const int turn = whole > 0 ? (int)blockIdx.x * WAVES % whole : 0;
  const int from = wave + WAVES * blockIdx.y, stride = WAVES * gridDim.y;
  for (int c0 = from; c0 < whole; c0 += stride) {
    const int c = c0 + turn < whole ? c0 + turn : c0 + turn - whole;
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
  for (int k0 = whole * (STEP * U) + from * STEP; k0 < K;
       k0 += stride * STEP) {
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
  const float f = scales ? scales[t[0].g] : scale;
  float* plane = z + (long)blockIdx.y * p.M * (RB * 16);
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
          plane[place * (RB * 16) + r] = r < R ? f * sum[q] : 0.0f;
      }
    }
  }
}

// -- expand -------------------------------------------------------------------

// out[row][n] = act(base[row][n] + sum_r z[place][r] W_e(n, r)), W [N, R]
// (RMAJOR), or without base and act, W [R, N].  One block takes up to WAVES
// tiles of an adapter, a wave a tile, through chunks of 16 V columns; a
// chunk's part of W is laid into LDS (in bf16 [R, N] is turned round there),
// and the loads of the next chunk are under way during this one's products.
// The product is taken as D[n][m], in fp32, or in bf16 with z in three parts;
// instruction j's row 4 h + q is the chunk's column
// 4 V a + V h + e, where j = a V / 4 + e / 4 and q = e % 4, so that a lane
// ends up with 16 bytes of adjacent outputs and its row's four lanes with
// 64.  base enters as the sum's first term.  8192 rows of 4096 bf16 at a rank
// of 16 (base read, out written: 134 MB): 28.7 us, 4.7 TB/s; a plain copy
// takes 21.  What only one of the forms needs is left out of the others at
// compile time: 32 divisions of a sigmoid and the base are registers of a
// fourth wave a SIMD (out of 8192 rows of 4096 alone, 67 MB, at a rank of 32:
// 21.1 us for 25.4).  Lanes that trade places, for 128 bytes of a
// row an instruction, and 1024 or 4096 blocks measured no better.  Few rows
// at high ranks: a wave alone keeps a whole chunk of W in registers, up to
// 480, so one wave a SIMD is left (32 rows x 4096 of 64 adapters, ranks of
// 16, 32, 64 and 128: bf16 5.6, 5.7, 7.9 and 15 us, fp32 5.2, 6.5, 17 and
// 30).
template <typename T, int RB, bool RMAJOR, bool SIGMOID, int WAVES>
__global__ void __launch_bounds__(WAVES * WAVE)
    adapter_expand_kernel(const T* __restrict__ base, long bstride,
                          const float* __restrict__ z,
                          const T* __restrict__ w, Plan p,
                          T* __restrict__ out, int N, int R, bool relu,
                          int across, int planes) {
  constexpr int V = Vec<T>::N;
  constexpr int COLS = 16 * V;
  constexpr int THREADS = WAVES * WAVE;
  constexpr bool SMALL = WAVES == 1;
  typedef typename Vec<T>::V VT;
  typedef T T4 __attribute__((ext_vector_type(4)));
  struct __attribute__((packed, aligned(sizeof(T)))) U4 {
    T4 v;
  };
  // bf16: 16 bytes of ranks an operand, so [R, N] is turned round on its
  // way into LDS
  constexpr bool BF16 = std::is_same<T, bf16_t>::value;
  constexpr bool TURN = BF16 && !RMAJOR;
  // LDS: a column's ranks side by side, or a rank's columns; the pitch
  // spreads a wave's quarters over the banks
  constexpr int PITCH = RMAJOR || TURN ? 16 * RB + 16 / sizeof(T)
                                       : COLS + 16 / sizeof(T);
  constexpr int PART = RMAJOR || TURN ? COLS * PITCH : 16 * RB * PITCH;
  constexpr int BUFFERS = 2 * PART * sizeof(T) <= 49152 ? 2 : 1;
  // vectors of W that a thread takes: 4 ranks; V columns; V columns of four
  // ranks
  constexpr int ALL = RMAJOR ? COLS * 4 * RB : TURN ? 64 * RB : 256 * RB;
  constexpr int TAKE = ALL < THREADS ? 1 : ALL / THREADS;
  constexpr int WIDE = TURN ? 4 : 1;
  __shared__ __attribute__((aligned(16))) T wl[BUFFERS][PART];
  const int tid = threadIdx.x;
  const int lane = tid & (WAVE - 1), wave = tid / WAVE;
  const int i = lane & 15, quarter = lane >> 4;
  // the columns' blocks are neighbours: blocks of different rows that run
  // side by side would write the same channels of the memory
  const int block = blockIdx.x / across, first = blockIdx.x % across;
  Tile t;
  bool has = true;
  if (SMALL) {
    t = small_tile(p, block, lane);
    if (t.g < 0) return;
  } else {
    const int4 of = p.blocks[block];
    if (of.x < 0) return;
    has = wave * TILE < of.z;
    t = plan_tile(p, of, has ? wave : 0, lane);
  }
  const int g = t.g;
  const bool adapted = g < p.E;
  const bool mine = has && i < t.rows;
  const T* br = base + (long)t.row * bstride;
  T* orow = out + (long)t.row * N;
  const T* we = w + (long)(adapted ? g : 0) * N * R;

  VT bv[4], bn[4];
  // Only the last chunk has vectors to cut: the others load without
  // branches.
  auto load_base = [&](int n0) {
    if (!RMAJOR) return;
    const int c0 = n0 + V * quarter;
    if (n0 + COLS <= N) {
#pragma unroll
      for (int a = 0; a < 4; ++a) bn[a] = Vec<T>::load(br + c0 + 4 * V * a);
      return;
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = c0 + 4 * V * a + e;
        bn[a][e] = c < N ? br[c] : (T)0.0f;
      }
  };
  // [R, N]: neighbouring lanes take neighbouring columns; turned round,
  // neighbouring ranks, which lie side by side in LDS (the other way round
  // eight lanes meet in a bank)
  auto rank_of = [](int at) { return TURN ? at % (4 * RB) * 4 : at / 16; };
  auto column_of = [](int at) {
    return (TURN ? at / (4 * RB) : at % 16) * V;
  };
  T4 w4[RMAJOR ? TAKE : 1];
  VT wv[RMAJOR ? 1 : TAKE][WIDE];
  auto load_w = [&](int n0) {
    if (!adapted) return;
    if (n0 + COLS <= N && R == 16 * RB) {
#pragma unroll
      for (int u = 0; u < TAKE; ++u) {
        const int at = tid + u * THREADS;
        if (RMAJOR) {  // the chunk is one piece of memory
          w4[u] = reinterpret_cast<const U4*>(we + (long)n0 * R + at * 4)->v;
        } else if (at < ALL) {
#pragma unroll
          for (int q = 0; q < WIDE; ++q)
            wv[u][q] = Vec<T>::load(we + (long)(rank_of(at) + q) * N + n0 +
                                    column_of(at));
        }
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < TAKE; ++u) {
      const int at = tid + u * THREADS;
      if (RMAJOR) {
        const int c = at / (4 * RB), r = at % (4 * RB) * 4;
        const T* wr = we + (long)min(n0 + c, N - 1) * R + r;
#pragma unroll
        for (int e = 0; e < 4; ++e) w4[u][e] = r + e < R ? wr[e] : (T)0.0f;
      } else {
#pragma unroll
        for (int q = 0; q < WIDE; ++q) {
          const int r = rank_of(at) + q, c = n0 + column_of(at);
          const T* wr = we + (long)r * N + c;
          if (r < R && c + V <= N) {
            wv[u][q] = Vec<T>::load(wr);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
              wv[u][q][e] = r < R && c + e < N ? wr[e] : (T)0.0f;
          }
        }
      }
    }
  };

  const int step = across * COLS;
  int n0 = first * COLS;
  load_base(n0);
  load_w(n0);
  // z: fp32 four at a time; bf16 in parts, eight at a time.  A rank of 16
  // fills only half of the 32 that a bf16 instruction sums over: there the
  // high parts take one half and the middle parts the other.
  constexpr int ZB = BF16 ? 1 : RB, ZP = BF16 ? (RB + 1) / 2 : 1;
  const float* zr = z + (long)t.place * (RB * 16);
  auto load_z = [&](int r) {
    f32x4 sum = *reinterpret_cast<const f32x4*>(zr + r);
    if (SMALL) {
#pragma unroll 4
      for (int s = 1; s < planes; ++s)
        sum += *reinterpret_cast<const f32x4*>(
            zr + (long)s * p.M * (RB * 16) + r);
    }
    return sum;
  };
  f32x4 zv[ZB];
  Vec<bf16_t>::V zh[ZP], zm[ZP], zl[ZP];
  if (adapted && BF16) {
#pragma unroll
    for (int b = 0; b < ZP; ++b) {
      const int r = 32 * b + 8 * (RB == 1 ? quarter & 1 : quarter);
      const f32x4 lo = load_z(r), hi = load_z(r + 4);
      const float f[8] = {lo[0], lo[1], lo[2], lo[3],
                          hi[0], hi[1], hi[2], hi[3]};
      const Split s = split(f);
      zh[b] = s.high;
      zm[b] = s.mid;
      zl[b] = s.low;
      if (RB == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          zh[b][e] = quarter < 2 ? s.high[e] : s.mid[e];
          zl[b][e] = quarter < 2 ? s.low[e] : (bf16_t)0.0f;
        }
      }
    }
  } else if (adapted) {
#pragma unroll
    for (int c = 0; c < ZB; ++c) zv[c] = load_z(16 * c + 4 * quarter);
  }
  for (int turn = 0; n0 < N; n0 += step, ++turn) {
    T* const part = wl[turn % BUFFERS];
    if (BUFFERS == 1) __syncthreads();  // the last chunk's part was read
    if (adapted) {
#pragma unroll
      for (int u = 0; u < TAKE; ++u) {
        const int at = tid + u * THREADS;
        if (RMAJOR) {
          *reinterpret_cast<T4*>(
              &part[at / (4 * RB) * PITCH + at % (4 * RB) * 4]) = w4[u];
        } else if (TURN) {
          if (at < ALL) {
#pragma unroll
            for (int e = 0; e < V; ++e)
              *reinterpret_cast<T4*>(
                  &part[(column_of(at) + e) * PITCH + rank_of(at)]) =
                  T4{wv[u][0][e], wv[u][1 % WIDE][e], wv[u][2 % WIDE][e],
                     wv[u][3 % WIDE][e]};
          }
        } else {
          *reinterpret_cast<VT*>(
              &part[rank_of(at) * PITCH + column_of(at)]) = wv[u][0];
        }
      }
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) bv[a] = bn[a];
    __syncthreads();
    if (n0 + step < N) {
      load_base(n0 + step);
      load_w(n0 + step);
    }
    f32x4 acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      constexpr int H = V / 4;  // instructions to a vector of the output
#pragma unroll
      for (int q = 0; q < 4; ++q)
        acc[j][q] = RMAJOR ? (float)bv[j / H][4 * (j % H) + q] : 0.0f;
      if (adapted) {
        const int c = 4 * V * (j / H) + V * (i >> 2) + 4 * (j % H) + (i & 3);
        if constexpr (BF16) {
#pragma unroll
          for (int b = 0; b < ZP; ++b) {
            const VT v = *reinterpret_cast<const VT*>(
                &part[c * PITCH + 32 * b +
                      8 * (RB == 1 ? quarter & 1 : quarter)]);
            acc[j] = mma(v, zl[b], acc[j]);
            if (RB > 1) acc[j] = mma(v, zm[b], acc[j]);
            acc[j] = mma(v, zh[b], acc[j]);
          }
          continue;
        }
#pragma unroll
        for (int b = 0; b < ZB; ++b) {
          const int r = 16 * b + 4 * quarter;
          T4 v;
          if (RMAJOR) {
            v = *reinterpret_cast<const T4*>(&part[c * PITCH + r]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = part[(r + e) * PITCH + c];
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                (float)v[e], zv[b][e], acc[j], 0, 0, 0);
        }
      }
    }
    const int c0 = n0 + V * quarter;
    if (g > p.E) {
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = f32x4{NAN, NAN, NAN, NAN};
    } else if (RMAJOR && relu) {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[j][q] = acc[j][q] < 0.0f ? 0.0f : acc[j][q];  // NaN stays
    } else if (SIGMOID) {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[j][q] = act_apply(acc[j][q], ACT_SIGMOID);
    }
    VT v[4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int e = 0; e < V; ++e)
        v[a][e] = (T)acc[a * (V / 4) + e / 4][e % 4];
    if (!mine) continue;
    if (n0 + COLS <= N) {
#pragma unroll
      for (int a = 0; a < 4; ++a) Vec<T>::store(orow + c0 + 4 * V * a, v[a]);
    } else {
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c0 + 4 * V * a + e < N) orow[c0 + 4 * V * a + e] = v[a][e];
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

// One of the two: dA from x and dz, or dB from dy and z.
template <typename T>
struct OuterSide {
  const T* x;
  long xstride;
  const float* z;
  T* out;
  float* partial;
  int K, chunks, stretch;  // chunks of 16 V columns; 0: not wanted
};

// sum over the rows of a stretch of one adapter: z[place][r] x[row][k].  A
// lane loads 16 bytes of a row; instruction j takes element j of all lanes,
// so its 16 columns are k0 + V (l % 16) + j.  Its sum runs over four rows in
// fp32; in bf16 over 32, of which a lane has every fourth: eight loads, whose
// elements j are one operand, beside z in three parts.  KMAJOR: the result
// is [R, K] (dA), else [K, R] (dB).  SMALL_OUTER, DIRECT_OUTER: one block an
// adapter, rounded into out; SPLIT_OUTER: one block a stretch, into fp32
// sums that reduce joins.
template <typename T, int RB, bool KMAJOR, OuterWork WORK>
__device__ __forceinline__ void outer_block(
    const OuterSide<T>& side, const Plan& p, int zstride, int R, int column,
    f32x4 (&part)[2][RB * Vec<T>::N][WAVE], int (&list)[SMALL_ROWS],
    int& found) {
  constexpr int V = Vec<T>::N;
  constexpr bool BF16 = std::is_same<T, bf16_t>::value;
  constexpr int U = BF16 ? 8 : 4;
  const T* __restrict__ x = side.x;
  const float* __restrict__ z = side.z;
  const long xstride = side.xstride;
  const int K = side.K, stretch = side.stretch;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int i = lane & 15, quarter = lane >> 4;
  int begin = 0, end = 0;
  if (WORK == SMALL_OUTER) {
    const bool here = lane < p.M && p.ids[lane] == (long)blockIdx.y;
    const unsigned long all = __ballot(here);
    if (here && wave == 0) list[__popcll(all & ((1ul << lane) - 1))] = lane;
    end = __popcll(all);
    __syncthreads();
  } else if (WORK == DIRECT_OUTER) {
    begin = p.seg[blockIdx.y];
    end = p.seg[blockIdx.y + 1];
  } else {
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += 256) {
      const int c = (int)blockIdx.y - first_slot(p, e, stretch);
      const int n = p.tbase[e + 1] - p.tbase[e];
      if (c >= 0 && (long)c * stretch < n) {
        found = e;
        list[0] = p.seg[e] + c * stretch * TILE;
      }
    }
    __syncthreads();
    if (found < 0) return;
    begin = list[0];
    end = min(p.seg[found + 1], begin + stretch * TILE);
  }
  const int r0 = blockIdx.z * (RB * 16);
  const int k0 = column * (16 * V);
  const int k = k0 + i * V;
  f32x4 acc[RB][V] = {};
  // The bf16 loop: 32 rows a step.  Nothing but the rows' numbers is loaded
  // a step ahead: with the rows too the loop took 268 registers, one wave a
  // SIMD, for 204, two (dA of 8192 rows x 4096: 34.9 us for 24.4).
  auto steps32 = [&](auto whole) {
    if constexpr (BF16) {
      constexpr bool WHOLE = decltype(whole)::value;
      constexpr int STEP = 4 * 32;  // of the four waves
      int row[U];
      auto place = [&](int m0, int u) {
        const int at = min(m0 + 4 * u + quarter, end - 1);
        return WORK == SMALL_OUTER ? list[at] : at;
      };
      auto number = [&](int m0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          row[u] = WORK == SMALL_OUTER ? place(m0, u) : p.perm[place(m0, u)];
      };
      int m0 = begin + wave * 32;
      if (m0 < end) number(m0);
      for (; m0 < end; m0 += STEP) {
        typename Vec<T>::V xv[U];
        float zv[RB][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const T* xr = x + (long)row[u] * xstride;
          if (WHOLE) {
            xv[u] = Vec<T>::load(xr + k);
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
              xv[u][j] = k + j < K ? xr[k + j] : (T)0.0f;
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int c = 0; c < RB; ++c)
            zv[c][u] = z[(long)place(m0, u) * zstride + r0 + 16 * c + i];
        number(m0 + STEP);
        if (m0 + 32 > end) {
          // rows behind the last: both factors, since 0 x NaN is not 0
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const bool in = m0 + 4 * u + quarter < end;
#pragma unroll
            for (int j = 0; j < V; ++j) xv[u][j] = in ? xv[u][j] : (T)0.0f;
#pragma unroll
            for (int c = 0; c < RB; ++c) zv[c][u] = in ? zv[c][u] : 0.0f;
          }
        }
        Split zs[RB];
#pragma unroll
        for (int c = 0; c < RB; ++c) zs[c] = split(zv[c]);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          typename Vec<T>::V col[2];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            col[0][u] = xv[u][j];
            col[1][u] = xv[u][j + 1];
          }
#pragma unroll
          for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int c = 0; c < RB; ++c)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                acc[c][j + h] = mma(part == 0   ? zs[c].low
                                    : part == 1 ? zs[c].mid
                                                : zs[c].high,
                                    col[h], acc[c][j + h]);
        }
      }
    }
  };
  // Four rows an instruction, U times four a step.  The next step's rows
  // are loaded before this one's products, and their numbers a step before
  // that.  Only the last columns' block has vectors to cut: the others take
  // a loop without branches.
  auto steps = [&](auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
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
        if (WHOLE) {
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
      load();  // behind the last step: rows that are there, not used
      number(m0 + 2 * STEP);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < RB; ++c)
#pragma unroll
          for (int j = 0; j < V; ++j)
            acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                zv[u][c], (float)xv[u][j], acc[c][j], 0, 0, 0);
    }
  };
  auto run = [&](auto whole) {
    if constexpr (BF16)
      steps32(whole);
    else
      steps(whole);
  };
  if (k0 + 16 * V <= K)
    run(std::true_type());
  else
    run(std::false_type());
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
  const long o0 = (long)blockIdx.y * R * K;
  // KMAJOR: a lane has V adjacent columns of four ranks; else four adjacent
  // ranks of V columns
#pragma unroll
  for (int c = 0; c < RB; ++c) {
    const int r = r0 + 16 * c + 4 * quarter;
    if (k + V <= K && r + 4 <= R && WORK == SPLIT_OUTER) {
#pragma unroll
      for (int q = 0; KMAJOR && q < 4; ++q)
#pragma unroll
        for (int h = 0; h < V / 4; ++h)
          Vec<float>::store(side.partial + o0 + (long)(r + q) * K + k + 4 * h,
                            f32x4{acc[c][4 * h][q], acc[c][4 * h + 1][q],
                                  acc[c][4 * h + 2][q],
                                  acc[c][4 * h + 3][q]});
#pragma unroll
      for (int j = 0; !KMAJOR && j < V; ++j)
        Vec<float>::store(side.partial + o0 + (long)(k + j) * R + r, acc[c][j]);
      continue;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (k + j >= K || r + q >= R) continue;
        const long o = o0 + (KMAJOR ? (long)(r + q) * K + k + j
                                    : (long)(k + j) * R + r + q);
        if (WORK == SPLIT_OUTER)
          side.partial[o] = acc[c][j][q];
        else
          side.out[o] = (T)acc[c][j][q];
      }
  }
}

// Both gradients in one launch: the first chunks of columns are dA's.  8192
// rows of 4096 and of 2048 bf16 at a rank of 32 (101 MB): 24.6 us, 4.1 TB/s
// (one after the other 34).  What bounds it are rows under way: 200
// registers leave two waves a SIMD, and with fewer they spill (32 us).
template <typename T, int RB, OuterWork WORK>
__global__ void __launch_bounds__(256)
    adapter_outer_kernel(OuterSide<T> da, OuterSide<T> db, Plan p,
                         int zstride, int R) {
  __shared__ f32x4 part[2][RB * Vec<T>::N][WAVE];
  __shared__ int list[SMALL_ROWS];
  __shared__ int found;
  const int column = blockIdx.x;
  if (column < da.chunks)
    outer_block<T, RB, true, WORK>(da, p, zstride, R, column, part, list,
                                   found);
  else
    outer_block<T, RB, false, WORK>(db, p, zstride, R, column - da.chunks,
                                    part, list, found);
}

// out_e = the sum of adapter e's partial sums, in their order; zero for an
// adapter without rows.  5.2 us for 8 adapters of 32 x (4096 + 2048).
template <typename T>
__global__ void __launch_bounds__(256)
    adapter_reduce_kernel(OuterSide<T> da, OuterSide<T> db, Plan p, int R) {
  const OuterSide<T>& side = blockIdx.z == 0 ? da : db;
  const long n = side.chunks ? (long)side.K * R : 0;
  const int e = blockIdx.y;
  const int tiles = p.tbase[e + 1] - p.tbase[e];
  const int slots = (tiles + side.stretch - 1) / side.stretch;
  const float* from = side.partial + (long)first_slot(p, e, side.stretch) * n;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (long)gridDim.x * 256) {
    float sum = 0.0f;
    for (int s = 0; s < slots; ++s) sum += from[s * n + i];
    side.out[e * n + i] = (T)sum;
  }
}

// d(act) from the output, in the operand's own type.  Two roundings that
// other outputs do not have: the slope is that of the rounded y (the sum
// before it would be another tensor to keep; a sigmoid's slope y (1 - y) is
// off by up to half a step of y, which is all of it where y rounds to 1),
// and dy is rounded to the type before dz, dA and dB are taken from it (it is
// base's gradient, wanted in that type, and the matrix instructions' operand).
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

static long max_blocks(long M, long E) {
  return M / (BLOCK_TILES * TILE) + std::min(E + 2, M);
}

static long plan_size(long M, long E) {
  if (M <= SMALL_ROWS) return 0;
  return 4 * (max_tiles(M, E) + max_blocks(M, E)) + M + 2 * (E + 3);
}

// tiles, blocks, perm, seg and tbase in one int32 tensor.
static Plan plan_of(const torch::Tensor& ids, const torch::Tensor& plan,
                    long E) {
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() && ids.dim() == 1 &&
                  ids.scalar_type() == torch::kInt64 &&
                  ids.size(0) < ROWS_MAX,
              "ids must be contiguous int64 [rows] on GPU, less than 2^26");
  TORCH_CHECK(E >= 1 && E <= ADAPTERS_MAX, "1 .. 1024 adapters");
  const long M = ids.size(0);
  TORCH_CHECK(plan.device() == ids.device() && plan.is_contiguous() &&
                  plan.scalar_type() == torch::kInt32 &&
                  plan.numel() == plan_size(M, E),
              "plan does not belong to these rows and adapters");
  Plan r = {ids.data_ptr<int64_t>(), (int)M, (int)E, nullptr, nullptr,
            nullptr, nullptr, nullptr};
  if (M > SMALL_ROWS) {
    r.tiles = reinterpret_cast<int4*>(plan.data_ptr<int>());
    r.blocks = r.tiles + max_tiles(M, E);
    r.perm = reinterpret_cast<int*>(r.blocks + max_blocks(M, E));
    r.seg = r.perm + M;
    r.tbase = r.seg + E + 3;
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
  const long each = 3 * (E + 3);
  const int waves = PLAN_WAVES * (E + 2) + each <= 12288 ? PLAN_WAVES : 8;
  const int lds = (int)((waves * (E + 2) + each) * sizeof(int));
  hipLaunchKernelGGL(adapter_plan_kernel, dim3(1), dim3(waves * WAVE), lds,
                     at::cuda::getCurrentCUDAStream(), p,
                     (int)max_tiles(M, E), (int)max_blocks(M, E), waves);
  LAUNCH_OK();
  return plan;
}

// (No rows may have any strides: contiguous() leaves those of an expanded
// gradient as they are.)
static void check_rows(const torch::Tensor& t, const char* name, long M,
                       long n, const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.dim() == 2 &&
                  t.size(0) == M && t.size(1) == n &&
                  t.scalar_type() == like.scalar_type() &&
                  (M == 0 || n == 1 || t.stride(1) == 1),
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
                  z.scalar_type() == torch::kFloat32 && z.dim() == 3 &&
                  z.size(0) >= 1 && z.size(1) == M &&
                  z.size(2) == padded_rank(R),
              "z must be what adapter_shrink gave");
  return z.data_ptr<float>();
}

// z [planes, M, Rp], whose sum is x [M, K] through w, [E, R, K] (kmajor) or
// [E, K, R].  More than one plane only where split allows it.
torch::Tensor adapter_shrink(torch::Tensor x, torch::Tensor w,
                             torch::Tensor ids, torch::Tensor plan,
                             c10::optional<torch::Tensor> scales,
                             double scale, bool kmajor, bool split) {
  const long M = x.size(0), E = w.size(0);
  check_weight(w, E);
  const long R = kmajor ? w.size(1) : w.size(2);
  const long K = kmajor ? w.size(2) : w.size(1);
  check_rows(x, "x", M, K, w);
  TORCH_CHECK(R >= 1 && R <= RANK_MAX, "rank must be 1 .. 128");
  TORCH_CHECK(K >= 1 && K < (1l << 28), "inputs must be 1 .. 2^28");
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
  const bool small = M <= SMALL_ROWS;
  // Few rows: split along k, so that reading the adapters is spread over the
  // chip.  32 rows of 4096 bf16 with as many adapters, shrink and expand
  // together: 12.5 us with one plane, 10.5 with 2, 9.9 with 4 or 8 (expand
  // has to add them), 10.9 with 16.
  const long bite = 2048 / x.element_size();
  const long planes =
      small && split ? std::max<long>(1, std::min<long>(16, K / bite)) : 1;
  auto z = torch::empty({planes, M, padded_rank(R)},
                        x.options().dtype(torch::kFloat32));
  if (M == 0) return z;
  auto stream = at::cuda::getCurrentCUDAStream();
  for_dtype(x.scalar_type(), "x", [&](auto t) {
    using T = decltype(t);
    for_rank(R, [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      // Loads of 16 bytes that a lane has in flight: U (1 + RB).  Two tiles
      // a block halve the reads of W, and the blocks: at 8192 rows of 4096
      // bf16 and a rank of 32 that is 18.8 us for 25.5, at 16 25.8 for 17.9
      // (what a CU has under way is what bounds it).  At ranks of 17 to 64
      // it gains from 4096 rows on, where the tiles are more than the 256
      // CUs.  z of 4096 inputs, 8 adapters, two tiles for one, us: 3000 rows
      // bf16 18.9 for 15.0 (rank 32) and 26.7 for 23.1 (64), fp32 36 for 26
      // and 59 for 47; 4096 rows 18.7 for 24.4, 29 for 42, 38 for 50 and 62
      // for 91; 16384 rows 58 for 65, 77 for 101, 112 for 116 and 183 for
      // 207.  It loses where 4096 rows are 256 tiles and no more (one
      // adapter, rank 32: bf16 18.7 for 16.0, fp32 35 for 26), and in fp32
      // at 8192 rows and a rank of 32 (79 for 74).
      constexpr int U = RB == 1 ? 8 : RB == 2 ? 4 : 2;
      constexpr int MANY = RB <= 4 ? 16 : 8;  // waves whose sums fit the LDS
      auto go = [&](auto kernel, int waves, long blocks) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)planes),
                           dim3(waves * WAVE), 0, stream, ptr<T>(x),
                           (long)x.stride(0), ptr<T>(w), p, sp, (float)scale,
                           z.data_ptr<float>(), (int)K, (int)R);
      };
      auto pick = [&](auto major) {
        constexpr bool KM = decltype(major)::value;
        if (planes > 1)
          go(adapter_shrink_kernel<T, RB, KM, true, 4, 1, RB <= 2 ? 4 : 2>, 4,
             M);
        else if (small)
          go(adapter_shrink_kernel<T, RB, KM, true, MANY, 1, U>, MANY, M);
        else if (M >= 4096 && (RB == 2 || RB == 4))
          go(adapter_shrink_kernel<T, RB, KM, false, 8, RB <= 4 ? 2 : 1,
                                   RB <= 4 ? 4 / RB : 1>,
             8, BLOCK_TILES / 2 * max_blocks(M, E));
        else
          go(adapter_shrink_kernel<T, RB, KM, false, 8, 1, U>, 8,
             max_tiles(M, E));
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

// act(base + z w) with w [E, N, R] (rmajor), or z w with w [E, R, N].
torch::Tensor adapter_expand(c10::optional<torch::Tensor> base,
                             torch::Tensor z, torch::Tensor w,
                             torch::Tensor ids, torch::Tensor plan,
                             int64_t act, bool rmajor) {
  const long M = z.size(1), E = w.size(0);
  check_weight(w, E);
  const long N = rmajor ? w.size(1) : w.size(2);
  const long R = rmajor ? w.size(2) : w.size(1);
  TORCH_CHECK(N >= 1 && N < (1l << 28), "outputs must be 1 .. 2^28");
  const float* zp = check_z(z, w, M, R);
  if (base.has_value()) check_rows(*base, "base", M, N, w);
  TORCH_CHECK(base.has_value() == rmajor && (rmajor || act == ACT_NONE),
              "a base and an activation belong to [outputs, rank]");
  TORCH_CHECK(z.size(0) == 1 || M <= SMALL_ROWS, "z: one plane");
  const Plan p = plan_of(ids, plan, E);
  TORCH_CHECK(p.M == M && ids.device() == w.device(),
              "ids must be one a row beside the adapters");
  const at::cuda::CUDAGuard guard(w.device());
  auto out = torch::empty({M, N}, w.options());
  if (M == 0) return out;
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool small = M <= SMALL_ROWS;
  const long blocks = small ? M : max_blocks(M, E);
  for_dtype(w.scalar_type(), "adapters", [&](auto t) {
    using T = decltype(t);
    const long cols = 16 * Vec<T>::N;
    for_rank(R, [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      auto go = [&](auto kernel, int waves) {
        // as many blocks across as leave 2048 in all: what is left of the
        // columns a block takes in turns
        const long chunks = (N + cols - 1) / cols;
        long turns = std::max<long>(1, chunks * blocks / 2048);
        const long across = (chunks + turns - 1) / turns;
        hipLaunchKernelGGL(
            kernel, grid_of(blocks * across, waves * WAVE, "adapters"),
            dim3(waves * WAVE), 0, stream,
            base.has_value() ? ptr<T>(*base) : nullptr,
            base.has_value() ? (long)base->stride(0) : 0l, zp, ptr<T>(w), p,
            ptr<T>(out), (int)N, (int)R, act == ACT_RELU, (int)across,
            (int)z.size(0));
      };
      auto pick = [&](auto major, auto sigmoid) {
        constexpr bool RM = decltype(major)::value;
        constexpr bool SG = decltype(sigmoid)::value;
        if (small)
          go(adapter_expand_kernel<T, RB, RM, SG, 1>, 1);
        else
          go(adapter_expand_kernel<T, RB, RM, SG, 4>, 4);
      };
      const std::true_type yes;
      const std::false_type no;
      if (!rmajor)
        pick(no, no);
      else if (act == ACT_SIGMOID)
        pick(yes, yes);
      else
        pick(yes, no);
    });
  });
  LAUNCH_OK();
  return out;
}

// dA [E, R, K] = the sums of dz^T x over each adapter's rows, and dB
// [E, N, R] those of dy^T z; either without its rows is not wanted.
std::vector<torch::Tensor> adapter_outer(c10::optional<torch::Tensor> x,
                                         c10::optional<torch::Tensor> dz,
                                         c10::optional<torch::Tensor> dy,
                                         c10::optional<torch::Tensor> z,
                                         torch::Tensor ids,
                                         torch::Tensor plan, int64_t E,
                                         int64_t R) {
  const c10::optional<torch::Tensor> from[2] = {x, dy}, of[2] = {dz, z};
  TORCH_CHECK(x.has_value() || dy.has_value(), "nothing is wanted");
  const torch::Tensor& like = x.has_value() ? *x : *dy;
  const Plan p = plan_of(ids, plan, E);
  TORCH_CHECK(ids.device() == like.device(), "ids must be beside x");
  const long M = p.M;
  const at::cuda::CUDAGuard guard(like.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  // Up to 1024 rows one block adds all of an adapter's, a column chunk each;
  // above, stretches that give about 512 blocks, so that one busy adapter is
  // not one block (8192 rows of 4096 fp16: 44 us, with 256 blocks 54); in
  // bf16, whose products take less time than its rows' loads, 256 (22 us,
  // with 512 24).  Both weights' gradients, one block for stretches and
  // their reduce, us.  8 adapters, 784 -> 256 at a rank of 8, fp32: 1024
  // rows 8.3 for 9.3, 2048 11.8 for 13.0, 4096 19 for 15; 4096 -> 2048 at
  // 32, bf16: 1024 rows 11 for 21, 4096 17 for 25.  What decides is an
  // adapter's rows, and a limit by all rows is late for one adapter (784 ->
  // 256 fp32: 256 rows 7.5 for 8.4, 512 11.0 for 9.4, 1024 29 for 12) and
  // early for many (64 of them, 4096 rows: 9.8 for 16).
  const bool small = M <= SMALL_ROWS, direct = M <= 1024;
  const long wanted = like.scalar_type() == torch::kBFloat16 ? 256 : 512;
  const long cols = 16 * (like.element_size() == 4 ? 4 : 8);
  std::vector<torch::Tensor> out(2), partial(2);
  long stretch[2] = {1, 1}, chunks[2] = {0, 0}, K[2] = {0, 0}, slots = E;
  const auto f32 = like.options().dtype(torch::kFloat32);
  for (int i = 0; i < 2; ++i) {
    if (!from[i].has_value()) continue;
    K[i] = from[i]->size(1);
    check_rows(*from[i], "rows", M, K[i], like);
    TORCH_CHECK(K[i] >= 1 && K[i] < (1l << 28), "rows must be 1 .. 2^28 wide");
    TORCH_CHECK(of[i].has_value() && of[i]->size(0) == 1, "z: one plane");
    check_z(*of[i], like, M, R);
    out[i] = torch::empty(i == 0 ? at::IntArrayRef({E, R, K[i]})
                                 : at::IntArrayRef({E, K[i], R}),
                          like.options());
    chunks[i] = (K[i] + cols - 1) / cols;
    if (direct) continue;
    stretch[i] = std::max<long>(4, M / TILE * chunks[i] / wanted);
    const long n = max_tiles(M, E) / stretch[i] + E;
    partial[i] = torch::empty({n, R, K[i]}, f32);
    slots = std::max(slots, n);
  }
  for_dtype(like.scalar_type(), "rows", [&](auto t) {
    using T = decltype(t);
    OuterSide<T> side[2] = {};
    for (int i = 0; i < 2; ++i) {
      side[i].stretch = (int)stretch[i];
      if (!from[i].has_value()) continue;
      side[i] = {ptr<T>(*from[i]),
                 (long)from[i]->stride(0),
                 of[i]->data_ptr<float>(),
                 ptr<T>(out[i]),
                 direct ? nullptr : partial[i].data_ptr<float>(),
                 (int)K[i],
                 (int)chunks[i],
                 (int)stretch[i]};
    }
    for_rank(R, [&](auto rb) {
      // ranks above 32 take turns of 32: more sums than that do not fit
      // the registers beside their operands
      constexpr int RB = decltype(rb)::value < 2 ? 1 : 2;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(
            kernel,
            dim3((unsigned)(chunks[0] + chunks[1]), (unsigned)slots,
                 (unsigned)(padded_rank(R) / (16 * RB))),
            dim3(256), 0, stream, side[0], side[1], p, (int)padded_rank(R),
            (int)R);
      };
      if (small)
        go(adapter_outer_kernel<T, RB, SMALL_OUTER>);
      else if (direct)
        go(adapter_outer_kernel<T, RB, DIRECT_OUTER>);
      else
        go(adapter_outer_kernel<T, RB, SPLIT_OUTER>);
    });
    LAUNCH_OK();
    if (!direct) {
      const long n = R * std::max(K[0], K[1]);
      hipLaunchKernelGGL((adapter_reduce_kernel<T>),
                         dim3((unsigned)std::min<long>(256, (n + 255) / 256),
                              (unsigned)E, 2),
                         dim3(256), 0, stream, side[0], side[1], p, (int)R);
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
