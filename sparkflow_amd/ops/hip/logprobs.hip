// Log-probabilities of given tokens with the entropy of their rows and the
// k best alternatives, and the gradient of all three.
//
//   m = max x      s = sum e^(x-m)      t = sum e^(x-m) (x-m)
//   l = log s                           logp_c = (x_c - m) - l
//   H = -sum p log p = l - t / s        (l >= 0 and t <= 0)
//   dx_c = g_logp [c = token] + sum_j g_j [c = id_j]
//          - p_c (g_logp + sum_j g_j) - g_H p_c (logp_c + H)
//
// m and l are kept apart: their sum in 32 bits would lose l beside a large
// m (a row masked by the type's lowest value, far-off logits).
//
// Forward reads the logits once: every thread keeps its own (m, s, t), a
// block joins them, and a row may be split over blocks that a second kernel
// joins.  The alternatives need no second pass over the row: of 64 groups
// of threads, the k-th largest maximum is a value that k elements reach, so
// only the threads whose own maximum reaches it, hardly more than k, read
// their elements again.
//
// All sums and statistics are fp32; outputs are fp32.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <climits>

#include "vec.h"

#define TOP_MAX 32

// (m, s, t) of a set of elements.  An empty set, or one of -inf alone, has
// s = t = 0.  NaN and +inf end up in s as NaN.
struct Stat {
  float m, s, t;
};

// The set moved to the larger maximum m.  The distance is bounded where its
// exponential has long been 0: a set of nothing but the type's lowest value
// would make s d infinite, and 0 times that NaN.
__device__ __forceinline__ Stat stat_at(Stat a, float m) {
  if (a.m == m || a.m == -INFINITY) return {m, a.s, a.t};
  const float d = fmaxf(a.m - m, -1000.0f);
  const float f = __expf(d);
  return {m, a.s * f, (a.t + a.s * d) * f};
}

__device__ __forceinline__ Stat stat_join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  a = stat_at(a, m);
  b = stat_at(b, m);
  return {m, a.s + b.s, a.t + b.t};
}

// A value in an order that whole numbers keep; both zeros are one.  0 is
// below every number and stands for NaN, whose row has no alternatives.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned b = __float_as_uint(x + 0.0f);
  if (x != x) return 0;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// The join of all lanes, in every lane: one change of maximum, then sums.
__device__ __forceinline__ Stat wave_join(Stat a) {
  a = stat_at(a, wave_max(a.m));
  return {a.m, wave_sum(a.s), wave_sum(a.t)};
}

// A thread's own running sums, in steps of log 2 and about a whole number of
// them, `shift`: e^x / 2^shift is one exponential of one fused product, with
// one rounding and two instructions less than e^(x - m), and instructions
// are what bounds the pass in the 16-bit types.  The sums move to another
// shift only when a value is 2.5 above `ref`, where they were put last: some
// lane of a wave has a new maximum almost every time, and seldom one that
// far.  Two sums each, for shorter chains.
//
// ref log2 e is rounded before it becomes a whole number, by half a step of
// fp32: 1/16 at 2^20, but 512 at a mask of -1e10, whose exponential would be
// infinite or 0.  From 2^20 on, and for an infinity, the sums are therefore
// about ref itself, at one instruction more an element (4096 rows of 32000
// bf16, all but 100 of them masked: 52.7 us for 45.9 if the mask is -1e9 and
// not -1e5; half of them 49.0 for 46.3).
struct Run {
  float m, ref, limit, shift, s0, s1, t0, t1;

  __device__ __forceinline__ void clear() {
    m = ref = limit = shift = -INFINITY;
    s0 = s1 = t0 = t1 = 0.0f;
  }

  static __device__ __forceinline__ bool far(float ref) {
    return !(fabsf(ref) < 0x1p20f);
  }

  // Adds 2^d to the sums of j's parity.
  __device__ __forceinline__ void add(int j, float d) {
    const float e = __builtin_amdgcn_exp2f(d);
    // -inf: e is 0 and must meet a finite factor
    const float f = fmaxf(d, -1000.0f);
    if (j % 2 == 0) {
      s0 += e;
      t0 = fmaf(e, f, t0);
    } else {
      s1 += e;
      t1 = fmaf(e, f, t1);
    }
  }

  // Adds n values.
  template <int n>
  __device__ __forceinline__ void take(const float (&x)[n]) {
    constexpr float LOG2E = 1.44269504089f;
    float gm = x[0];
#pragma unroll
    for (int j = 1; j < n; ++j) gm = fmaxf(gm, x[j]);
    m = fmaxf(m, gm);
    if (gm > limit) {
      const float old = ref, from = shift;
      ref = gm;
      shift = rintf(gm * LOG2E);
      limit = far(ref) ? ref : ref + 2.5f;
      if (old != -INFINITY) {
        // from what the sums were about to what they are about now
        const float d = far(old)   ? (far(ref) ? (old - ref) * LOG2E
                                               : fmaf(old, LOG2E, -shift))
                        : far(ref) ? -fmaf(ref, LOG2E, -from)
                                   : from - shift;
        const float f = __builtin_amdgcn_exp2f(d);
        // a reference of infinite distance leaves nothing of the old sums
        const float g = fmaxf(d, -1000.0f);
        t0 = (t0 + s0 * g) * f;
        t1 = (t1 + s1 * g) * f;
        s0 *= f;
        s1 *= f;
      }
    }
    if (far(ref)) {
      // nothing but -inf so far: it stays -inf, and a NaN a NaN
      const float about = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
      for (int j = 0; j < n; ++j) add(j, (x[j] - about) * LOG2E);
      return;
    }
#pragma unroll
    for (int j = 0; j < n; ++j) add(j, fmaf(x[j], LOG2E, -shift));
  }

  // The same about m, in natural steps.  t - s d takes the distance from
  // `shift` to m, up to 4.2 steps, out of every term: where one value is
  // nearly all of the sum, what is left of t is off by some 2^-21 s, in
  // either direction.  The maximum's own term is 1 and no term of t is above
  // 0, so s and t are held to that: no log-probability comes out above 0 and
  // no entropy below.  A NaN passes both comparisons.
  __device__ __forceinline__ Stat stat() const {
    constexpr float LOG2E = 1.44269504089f, LN2 = 0.69314718056f;
    float s = s0 + s1, t = t0 + t1;
    if (!far(ref)) {  // else m is ref
      const float d = fmaf(m, LOG2E, -shift);
      const float f = __builtin_amdgcn_exp2f(-d);
      t = (t - s * d) * f;
      s *= f;
    }
    if (m > -INFINITY && s < 1.0f) s = 1.0f;
    if (t > 0.0f) t = 0.0f;
    return {m, s, t * LN2};
  }
};

// An element in the order of the alternatives: larger values first, equal
// ones by the lower index.  0 is no element.
__device__ __forceinline__ unsigned long order_key(unsigned order,
                                                   unsigned idx) {
  return order ? ((unsigned long)order << 32) | (0xFFFFFFFFu - idx) : 0;
}

__device__ __forceinline__ float key_value(unsigned long key) {
  const unsigned o = (unsigned)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

__device__ __forceinline__ long key_index(unsigned long key) {
  return (long)(0xFFFFFFFFu - (unsigned)key);
}

__device__ __forceinline__ unsigned long key_max(unsigned long a,
                                                 unsigned long b) {
  return a > b ? a : b;
}

// The wave's largest, in every lane: six steps within the vector unit, where
// a shuffle goes through LDS.
__device__ __forceinline__ unsigned wave_max_u32(unsigned v) {
#define STEP(ctrl, rows)                                                    \
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows,   \
                                                   0xf, false))
  STEP(0x111, 0xf);  // from one lane lower, of 16
  STEP(0x112, 0xf);
  STEP(0x114, 0xf);
  STEP(0x118, 0xf);
  STEP(0x142, 0xa);  // the last of 16 to the next 16
  STEP(0x143, 0xc);  // the last of 32 to the next 32
#undef STEP
  return (unsigned)__builtin_amdgcn_readlane((int)v, WAVE - 1);
}

// The same of keys: the larger halves first, then the others among equals.
__device__ __forceinline__ unsigned long wave_key_max(unsigned long key) {
  const unsigned high = (unsigned)(key >> 32);
  const unsigned top = wave_max_u32(high);
  const unsigned low = wave_max_u32(high == top ? (unsigned)key : 0);
  return ((unsigned long)top << 32) | low;
}

// Labels are int64, or fp32 that hold whole numbers (the engine's labels).
struct Tokens {
  const long* i64;
  const float* f32;
  long ignore;
};

// What does not fit 64 bits, a NaN among it, is no token (the conversion
// has no defined result).
__device__ __forceinline__ long token_of(const Tokens& t, long row) {
  if (t.i64) return t.i64[row];
  const float x = t.f32[row];
  return fabsf(x) < 0x1p62f ? (long)x : LONG_MIN;
}

struct RowOut {
  float* logp;
  float* entropy;
  float* stat;  // [M, 2]: m and log s
  float* top;   // [M, k]
  long* ids;    // [M, k]
};

// What a row says when it is not to be read.
__device__ __forceinline__ void write_ignored(const RowOut& o, long row,
                                              int k, int tid, int nt) {
  if (tid == 0) {
    o.logp[row] = 0.0f;
    o.entropy[row] = 0.0f;
    o.stat[2 * row] = 0.0f;
    o.stat[2 * row + 1] = 0.0f;
  }
  for (int j = tid; j < k; j += nt) {
    o.top[row * k + j] = 0.0f;
    o.ids[row * k + j] = -1;
  }
}

// x: the token's logit, NaN for a token that the row does not have.
__device__ __forceinline__ void write_stats(const RowOut& o, long row,
                                            Stat a, float x) {
  const float l = a.s == 0.0f ? 0.0f : logf(a.s);
  float lp;
  if (x != x) {
    lp = NAN;
  } else if (a.s == 0.0f) {
    lp = -INFINITY;  // every token of the row is impossible
  } else {
    lp = (x - a.m) - l;
  }
  o.logp[row] = lp;
  o.entropy[row] = a.s == 0.0f ? 0.0f : l - a.t / a.s;
  o.stat[2 * row] = a.m;
  o.stat[2 * row + 1] = l;
}

__device__ __forceinline__ void write_top(const RowOut& o, long row, int k,
                                          int j, unsigned long key, Stat a) {
  const bool none = a.s != a.s;  // a NaN or +inf: no distribution
  float lp = NAN;
  long id = -1;
  if (!none && key != 0) {
    const float x = key_value(key);
    lp = x == -INFINITY ? -INFINITY : (x - a.m) - logf(a.s);
    id = key_index(key);
  }
  o.top[row * k + j] = lp;
  o.ids[row * k + j] = id;
}

// One block per (row, split).  Thread t of NT owns the vectors t, t + NT,
// t + 2 NT ... of the split and, if it is the last thread, the elements
// behind the last whole vector.
//
// In bf16 about nine instructions and an exponential an element keep the
// vector units 73% busy: 3277 rows of 32000 (210 MB) take 56 us, 3.7 TB/s,
// where a plain read takes 33; fp32, 461 rows of 50001 with 5 alternatives
// (92 MB): 21 us, 4.4 TB/s.  Longer rounds, blocks of 128, 512 or 1024
// threads and loads before the row's token is known change that by less
// than 3%.
template <typename T, int NT, int UNROLL, bool TOP>
__global__ void __launch_bounds__(NT)
    logprobs_fwd_kernel(const T* __restrict__ logits, long stride,
                        Tokens tokens, RowOut out, float* __restrict__ pstat,
                        unsigned long* __restrict__ pkeys, long C, int splits,
                        long span, int k) {
  constexpr int N = Vec<T>::N;
  constexpr int CAP = 512;
  typedef typename Vec<T>::V V;
  __shared__ Stat wstat[NT / WAVE];
  __shared__ __attribute__((aligned(16))) unsigned groups[WAVE];
  __shared__ unsigned long cand[TOP ? CAP : 1];
  __shared__ int owners[NT];
  __shared__ unsigned bar;
  __shared__ int nown, count;

  const int tid = threadIdx.x;
  const int lane = tid & (WAVE - 1), wave = tid / WAVE;
  const long row = blockIdx.x / splits;
  const int split = blockIdx.x % splits;
  const long token = token_of(tokens, row);
  if (token == tokens.ignore) {
    if (splits == 1) write_ignored(out, row, k, tid, NT);
    return;
  }
  const T* xr = logits + row * stride;
  const float chosen = token >= 0 && token < C ? (float)xr[token] : NAN;
  const long lo = split * span;
  const long hi = lo + span < C ? lo + span : C;
  const T* part = xr + lo;
  const int vecs = (int)((hi - lo) / N);  // whole vectors
  const int tail = (int)((hi - lo) % N);

  // -- one pass
  Run run;
  run.clear();
  // rounds of the block, the next one's loads under way; only the last is
  // cut, and filled up with what has no weight
  constexpr int ROUND = NT * UNROLL;
  const int rounds = (vecs + ROUND - 1) / ROUND;
  V v[UNROLL];
  auto load = [&](int r) {
    const int at = r * ROUND + tid;
    if ((r + 1) * ROUND <= vecs) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        v[u] = Vec<T>::load(part + (long)(at + u * NT) * N);
      return;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[u][j] = (T)-INFINITY;
      if (at + u * NT < vecs)
        v[u] = Vec<T>::load(part + (long)(at + u * NT) * N);
    }
  };
  if (rounds > 0) load(0);
  for (int r = 0; r < rounds; ++r) {
    float x[UNROLL * N];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int j = 0; j < N; ++j) x[u * N + j] = (float)v[u][j];
    if (r + 1 < rounds) load(r + 1);
    run.take(x);
  }
  if (tid == NT - 1)
    for (int j = 0; j < tail; ++j) {
      const float x[1] = {(float)part[(long)vecs * N + j]};
      run.take(x);
    }
  Stat a = run.stat();

  // the thread's maximum, and that of its group
  const bool any = tid < vecs || (tid == NT - 1 && tail > 0);
  const unsigned own = any ? order_of(a.m) : 0;
  if (TOP) {
    constexpr int G = NT / WAVE;  // threads of a group: 1 or 4
    unsigned g = own;
#pragma unroll
    for (int off = 1; off < G; off <<= 1)
      g = max(g, (unsigned)__shfl_xor((int)g, off, WAVE));
    if (tid % G == 0) groups[tid / G] = g;
    if (tid == 0) {
      bar = 0xFFFFFFFFu;
      nown = count = 0;
    }
  }

  // -- the block's (m, s, t)
  a = wave_join(a);
  if (lane == 0) wstat[wave] = a;
  __syncthreads();
  a = wstat[0];
#pragma unroll
  for (int w = 1; w < NT / WAVE; ++w) a = stat_join(a, wstat[w]);
  if (tid == 0) {
    if (splits == 1) {
      write_stats(out, row, a, chosen);
    } else {
      float* p = pstat + ((long)row * splits + split) * 3;
      p[0] = a.m;
      p[1] = a.s;
      p[2] = a.t;
    }
  }
  if (!TOP) return;

  // -- the bar: the smallest of the groups' k largest maxima (0, which
  // every element reaches, if there are not k groups that hold anything)
  if (wave == 0) {
    const unsigned mine = groups[lane];
    int above = 0;
#pragma unroll
    for (int i = 0; i < WAVE; i += 4) {
      const uint4 g = *reinterpret_cast<const uint4*>(&groups[i]);
      above += (g.x > mine) + (g.y > mine) + (g.z > mine) + (g.w > mine);
    }
    if (above < k) atomicMin(&bar, mine);
  }
  __syncthreads();
  const unsigned least = max(bar, 1u);
  if (own >= least) owners[atomicAdd(&nown, 1)] = tid;
  __syncthreads();

  // -- every element that reaches it, from the threads that have one
  const int n_own = nown;
  const int per = (vecs + NT - 1) / NT;  // vectors of one thread, at most
  for (int w = tid; w < n_own * per; w += NT) {
    const int at = owners[w / per] + (w % per) * NT;
    if (at >= vecs) continue;
    const V x = Vec<T>::load(part + (long)at * N);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const unsigned o = order_of((float)x[j]);
      if (o >= least) {
        const int i = atomicAdd(&count, 1);
        if (i < CAP)
          cand[i] = order_key(o, (unsigned)(lo + (long)at * N + j));
      }
    }
  }
  if (tid < tail) {
    const unsigned o = order_of((float)part[(long)vecs * N + tid]);
    if (o >= least) {
      const int i = atomicAdd(&count, 1);
      if (i < CAP)
        cand[i] = order_key(o, (unsigned)(lo + (long)vecs * N + tid));
    }
  }
  __syncthreads();
  const int n = count;
  unsigned long* pk =
      splits == 1 ? nullptr : pkeys + ((long)row * splits + split) * k;
  auto emit = [&](int j, unsigned long key) {
    if (splits == 1)
      write_top(out, row, k, j, key, a);
    else
      pk[j] = key;
  };
  if (n <= CAP) {
    for (int i = tid; i < n; i += NT) {
      const unsigned long key = cand[i];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) r += cand[j] > key ? 1 : 0;
      if (r < k) emit(r, key);
    }
    for (int j = n + tid; j < k; j += NT) emit(j, 0);
    return;
  }
  // More than the list holds: many equal values, or the large ones together
  // in few threads' vectors.  Take them one after another, the largest below
  // the last: a pass over the owners' elements each (512 rows of 50001 equal
  // fp32 logits 214 us with 5 alternatives and 666 with 20, where different
  // ones take 21 and 26, and whole numbers up to 4 52 and 58).
  unsigned long last = ~0ul;
  for (int j = 0; j < k; ++j) {
    unsigned long top = 0;
    for (int w = tid; w < n_own * per; w += NT) {
      const int at = owners[w / per] + (w % per) * NT;
      if (at >= vecs) continue;
      const V x = Vec<T>::load(part + (long)at * N);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned long key =
            order_key(order_of((float)x[i]),
                      (unsigned)(lo + (long)at * N + i));
        if (key < last) top = key_max(top, key);
      }
    }
    if (tid < tail) {
      const unsigned long key =
          order_key(order_of((float)part[(long)vecs * N + tid]),
                    (unsigned)(lo + (long)vecs * N + tid));
      if (key < last) top = key_max(top, key);
    }
    top = wave_key_max(top);
    __syncthreads();  // the list, or the last turn's maxima, were read
    if (lane == 0) cand[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / WAVE; ++w) top = key_max(top, cand[w]);
    if (tid == 0) emit(j, top);
    last = top;
  }
}

#define SPLITS_MAX 64

// Joins the splits of a row, one wave a row: latency alone (16 rows of 32
// splits with 20 alternatives 6.9 us, 9.1 before its loads were made to wait
// together).  Lane l holds split l and its
// sorted list.  If q is how many a list has to give on average, c lists
// whose q-th elements are the largest hold k elements that reach the
// smallest of those c: only what reaches that bar is ranked.
template <typename T>
__global__ void __launch_bounds__(WAVE)
    logprobs_join_kernel(const T* __restrict__ logits, long stride,
                         Tokens tokens, RowOut out,
                         const float* __restrict__ pstat,
                         const unsigned long* __restrict__ pkeys, long C,
                         int splits, int k) {
  __shared__ unsigned long list[SPLITS_MAX * TOP_MAX];
  __shared__ unsigned long cand[SPLITS_MAX * TOP_MAX];
  __shared__ __attribute__((aligned(16))) unsigned probes[WAVE];
  __shared__ unsigned bar;
  __shared__ int count;
  const long row = blockIdx.x;
  const int lane = threadIdx.x;
  const long token = token_of(tokens, row);
  // (what an ignored row's splits left unwritten is loaded and not used)
  const unsigned long* from = pkeys + row * splits * k;
  for (int i0 = lane; i0 < splits * k; i0 += 8 * WAVE) {
    unsigned long some[8];  // eight loads under way
#pragma unroll
    for (int u = 0; u < 8; ++u)
      some[u] = i0 + u * WAVE < splits * k ? from[i0 + u * WAVE] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u * WAVE < splits * k) list[i0 + u * WAVE] = some[u];
  }
  Stat a = {-INFINITY, 0.0f, 0.0f};
  if (lane < splits) {
    const float* p = pstat + (row * splits + lane) * 3;
    a = {p[0], p[1], p[2]};
  }
  if (lane == 0) {
    bar = 0xFFFFFFFFu;
    count = 0;
  }
  if (token == tokens.ignore) {
    write_ignored(out, row, k, lane, WAVE);
    return;
  }
  const float chosen =
      token >= 0 && token < C ? (float)logits[row * stride + token] : NAN;
  a = wave_join(a);
  if (lane == 0) write_stats(out, row, a, chosen);
  if (k == 0) return;
  __syncthreads();
  const int q = (k + splits - 1) / splits, c = (k + q - 1) / q;
  const unsigned mine =
      lane < splits ? (unsigned)(list[lane * k + q - 1] >> 32) : 0;
  probes[lane] = mine;  // 0 behind the last split: above no one
  __syncthreads();
  int above = 0;
#pragma unroll
  for (int i = 0; i < WAVE; i += 4) {
    const uint4 g = *reinterpret_cast<const uint4*>(&probes[i]);
    above += (g.x > mine) + (g.y > mine) + (g.z > mine) + (g.w > mine);
  }
  if (lane < splits && above < c) atomicMin(&bar, mine);
  __syncthreads();
  const unsigned least = max(bar, 1u);
  if (lane < splits)
    for (int j = 0; j < k; ++j) {
      const unsigned long key = list[lane * k + j];
      if ((unsigned)(key >> 32) < least) break;
      cand[atomicAdd(&count, 1)] = key;
    }
  __syncthreads();
  const int n = count;
  for (int i = lane; i < n; i += WAVE) {
    const unsigned long key = cand[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += cand[j] > key ? 1 : 0;
    if (r < k) write_top(out, row, k, r, key, a);
  }
  for (int j = n + lane; j < k; j += WAVE) write_top(out, row, k, j, 0, a);
}

struct RowGrad {
  const float* logp;     // each may be null: no gradient from there
  const float* entropy;
  const float* top;
};

// One block per (row, span).  The few places that take a gradient of their
// own (the token, the alternatives) are listed first; a vector without one
// of them costs one comparison per listed place, and a span that holds none
// costs nothing.  Bound by memory: bf16 4096 x 32000, a fifth of the rows
// ignored (read 210 MB, written 262) 71 us, 6.6 TB/s; fp32 512 x 50001
// 32 us, 6.1 TB/s.
template <typename T, int NT>
__global__ void __launch_bounds__(NT)
    logprobs_bwd_kernel(const T* __restrict__ logits, long stride,
                        Tokens tokens, const float* __restrict__ stat,
                        const float* __restrict__ entropy,
                        const long* __restrict__ ids, RowGrad grad,
                        T* __restrict__ dx, long C, int spans, long span,
                        int k) {
  constexpr int N = Vec<T>::N;
  __shared__ long place[TOP_MAX + 1];
  __shared__ float add[TOP_MAX + 1];
  __shared__ int count;
  const int tid = threadIdx.x;
  const long row = blockIdx.x / spans;
  const long lo = (long)(blockIdx.x % spans) * span;
  const long hi = lo + span < C ? lo + span : C;
  const T* xr = logits + row * stride;
  T* dr = dx + row * C;
  const long token = token_of(tokens, row);
  const long vecs = (hi - lo) / N;

  if (token == tokens.ignore) {
    typename Vec<T>::V zero;
#pragma unroll
    for (int j = 0; j < N; ++j) zero[j] = (T)0.0f;
    for (long v = tid; v < vecs; v += NT) Vec<T>::store(dr + lo + v * N, zero);
    for (long c = lo + vecs * N + tid; c < hi; c += NT) dr[c] = (T)0.0f;
    return;
  }
  const float m = stat[2 * row], l = stat[2 * row + 1];
  const float H = entropy[row];
  const float gp = grad.logp ? grad.logp[row] : 0.0f;
  const float gh = grad.entropy ? grad.entropy[row] : 0.0f;
  float share = gp;
  if (grad.top)
    for (int j = 0; j < k; ++j) share += grad.top[row * k + j];
  const bool bad = grad.logp && (token < 0 || token >= C);  // no such token
  if (bad) share = NAN;
  // a row of -inf alone is constant
  const bool constant = m == -INFINITY && l == 0.0f && !bad;
  if (tid < WAVE) {  // k + 1 <= 33 places, listed in their order
    long c = -1;
    float g = 0.0f;
    if (tid < k && grad.top) {
      c = ids[row * k + tid];
      g = grad.top[row * k + tid];
    } else if (tid == k) {
      c = token;
      g = gp;
    }
    const bool here = !constant && c >= lo && c < hi && g != 0.0f;
    const unsigned long all = __ballot(here);
    if (here) {
      const int i = __popcll(all & ((1ul << tid) - 1));
      place[i] = c;
      add[i] = g;
    }
    if (tid == 0) count = __popcll(all);
  }
  __syncthreads();
  const int n = count;
  auto at = [&](float x) -> float {
    if (constant) return 0.0f;
    const float d = (x - m) - l;
    const float p = __expf(d);
    // -inf: p is 0 and must meet a finite factor
    return -p * fmaf(gh, fmaxf(d, -1000.0f) + H, share);
  };
  for (long v = tid; v < vecs; v += NT) {
    const long c0 = lo + v * N;
    const typename Vec<T>::V in = Vec<T>::load(xr + c0);
    float d[N];
#pragma unroll
    for (int j = 0; j < N; ++j) d[j] = at((float)in[j]);
    for (int i = 0; i < n; ++i) {
      const long p = place[i] - c0;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (p == j) d[j] += add[i];
    }
    typename Vec<T>::V o;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = (T)d[j];
    Vec<T>::store(dr + c0, o);
  }
  for (long c = lo + vecs * N + tid; c < hi; c += NT) {
    float d = at((float)xr[c]);
    for (int i = 0; i < n; ++i)
      if (place[i] == c) d += add[i];
    dr[c] = (T)d;
  }
}

static Tokens check_logits(const torch::Tensor& logits,
                           const torch::Tensor& tokens, int64_t ignore) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) >= 1 &&
                  (logits.size(0) == 0 || logits.size(1) == 1 ||
                   logits.stride(1) == 1) &&
                  logits.size(1) < (1l << 31),
              "logits must be [rows, classes] on GPU with classes side by "
              "side");
  TORCH_CHECK(tokens.device() == logits.device() && tokens.dim() == 1 &&
                  tokens.is_contiguous() &&
                  tokens.size(0) == logits.size(0) &&
                  (tokens.scalar_type() == torch::kInt64 ||
                   tokens.scalar_type() == torch::kFloat32),
              "tokens must be contiguous int64 or fp32 [rows] beside logits");
  const bool whole = tokens.scalar_type() == torch::kInt64;
  return {whole ? tokens.data_ptr<int64_t>() : nullptr,
          whole ? nullptr : tokens.data_ptr<float>(), ignore};
}

std::vector<torch::Tensor> logprobs_fwd(torch::Tensor logits,
                                        torch::Tensor tokens, int64_t k,
                                        int64_t ignore) {
  const Tokens tok = check_logits(logits, tokens, ignore);
  TORCH_CHECK(k >= 0 && k <= TOP_MAX && k <= logits.size(1),
              "top_k must be 0 .. min(32, classes)");
  const at::cuda::CUDAGuard guard(logits.device());
  const long M = logits.size(0), C = logits.size(1);
  const auto f32 = logits.options().dtype(torch::kFloat32);
  const auto i64 = logits.options().dtype(torch::kInt64);
  auto logp = torch::empty({M}, f32), entropy = torch::empty({M}, f32),
       stat = torch::empty({M, 2}, f32), top = torch::empty({M, k}, f32);
  auto ids = torch::empty({M, k}, i64);
  if (M == 0) return {logp, entropy, stat, top, ids};
  const RowOut out = {logp.data_ptr<float>(), entropy.data_ptr<float>(),
                      stat.data_ptr<float>(), top.data_ptr<float>(),
                      ids.data_ptr<int64_t>()};
  auto stream = at::cuda::getCurrentCUDAStream();
  for_dtype(logits.scalar_type(), "logits", [&](auto t) {
    using T = decltype(t);
    constexpr int N = Vec<T>::N;
    // Split rows until the blocks fill the 256 CUs twice, in spans of
    // 4096 elements at least.
    long splits = 1;
    if (M < 512)
      splits = std::min<long>(SPLITS_MAX, std::min((512 + M - 1) / M,
                                                   (C + 4095) / 4096));
    long span = (C + splits - 1) / splits;
    span = (span + N - 1) / N * N;
    splits = (C + span - 1) / span;
    torch::Tensor pstat, pkeys;
    if (splits > 1) {
      pstat = torch::empty({M, splits, 3}, f32);
      pkeys = torch::empty({M, splits, k}, i64);
    }
    float* ps = splits > 1 ? pstat.data_ptr<float>() : nullptr;
    auto* pk = splits > 1
                   ? reinterpret_cast<unsigned long*>(pkeys.data_ptr())
                   : nullptr;
    const T* x = ptr<T>(logits);
    auto go = [&](auto kernel, int nt) {
      hipLaunchKernelGGL(kernel, grid_of(M * splits, nt, "logits"), dim3(nt),
                         0, stream, x, (long)logits.stride(0), tok, out, ps,
                         pk, C, (int)splits, span, (int)k);
    };
    // One wave a row while a row gives a wave no more than 4 vectors a
    // lane; more rows are in flight then and nothing waits at a barrier.
    if (span <= 4 * WAVE * N) {
      if (k)
        go(logprobs_fwd_kernel<T, 64, 1, true>, 64);
      else
        go(logprobs_fwd_kernel<T, 64, 1, false>, 64);
    } else if (k) {
      go(logprobs_fwd_kernel<T, 256, 16 / N, true>, 256);
    } else {
      go(logprobs_fwd_kernel<T, 256, 16 / N, false>, 256);
    }
    LAUNCH_OK();
    if (splits > 1) {
      hipLaunchKernelGGL((logprobs_join_kernel<T>),
                         dim3((unsigned)M), dim3(WAVE), 0, stream, x,
                         (long)logits.stride(0), tok, out, ps, pk, C,
                         (int)splits, (int)k);
      LAUNCH_OK();
    }
  });
  return {logp, entropy, stat, top, ids};
}

static const float* row_grad(const c10::optional<torch::Tensor>& g,
                             const torch::Tensor& logits, long n) {
  if (!g.has_value()) return nullptr;
  TORCH_CHECK(g->device() == logits.device() && g->is_contiguous() &&
                  g->scalar_type() == torch::kFloat32 && g->numel() == n,
              "row gradients must be contiguous fp32 beside logits");
  return g->data_ptr<float>();
}

torch::Tensor logprobs_bwd(torch::Tensor logits, torch::Tensor tokens,
                           torch::Tensor stat, torch::Tensor entropy,
                           torch::Tensor ids,
                           c10::optional<torch::Tensor> g_logp,
                           c10::optional<torch::Tensor> g_entropy,
                           c10::optional<torch::Tensor> g_top,
                           int64_t ignore) {
  const Tokens tok = check_logits(logits, tokens, ignore);
  const long M = logits.size(0), C = logits.size(1);
  TORCH_CHECK(ids.device() == logits.device() && ids.is_contiguous() &&
                  ids.scalar_type() == torch::kInt64 && ids.dim() == 2 &&
                  ids.size(0) == M && ids.size(1) <= TOP_MAX,
              "ids must be contiguous int64 [rows, k]");
  const int k = (int)ids.size(1);
  const float* pl = row_grad(stat, logits, 2 * M);
  const float* pe = row_grad(entropy, logits, M);
  const RowGrad grad = {row_grad(g_logp, logits, M),
                        row_grad(g_entropy, logits, M),
                        row_grad(g_top, logits, M * k)};
  const at::cuda::CUDAGuard guard(logits.device());
  auto dx = torch::empty({M, C}, logits.options());
  if (M == 0) return dx;
  auto stream = at::cuda::getCurrentCUDAStream();
  for_dtype(logits.scalar_type(), "logits", [&](auto t) {
    using T = decltype(t);
    constexpr int N = Vec<T>::N;
    auto go = [&](auto kernel, int nt, long span) {
      const long spans = (C + span - 1) / span;
      hipLaunchKernelGGL(kernel, grid_of(M * spans, nt, "logits"), dim3(nt),
                         0, stream, ptr<T>(logits), (long)logits.stride(0),
                         tok, pl, pe, ids.data_ptr<int64_t>(), grad,
                         ptr<T>(dx), C, (int)spans, span, k);
    };
    if (C <= 4 * WAVE * N) {
      go(logprobs_bwd_kernel<T, 64>, 64, 4 * WAVE * N);
    } else {
      go(logprobs_bwd_kernel<T, 256>, 256, 256 * N * 4);
    }
  });
  LAUNCH_OK();
  return dx;
}
