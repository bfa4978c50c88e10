// The selection step of a beam search: of a sequence's beams and all their next tokens, the n continuations of the highest
// log-probability.  (The reference keeps one continuation and has no such step; its softmax over a row is
// src/sampler/mod.rs:119-143.)
//
//   v(b, t) = c_b + x_bt - log sum_u exp x_bu        the n largest of all (b, t) in falling order; ties: lowest (b, t) first
//
// Two kernels.  The first reads every row once, a block per part of a row.  Within a row the constant c_b - lse does not matter, so
// a part's n largest x are all that can become a candidate.  An entry that reaches a bound that n entries are known to reach is
// collected in shared memory, any other is added to the sum of exp(x - bound), in which nothing can overflow.  The first bound comes of
// the part's first 4096 entries (the threads form groups, and the n-th largest of the groups' maxima is reached by n entries and, for n = 16,
// by 22 in all); whenever the tiles read have doubled, the n-th largest of those collected becomes the next, so that ever fewer
// are collected (some 20 in each doubling) and the threads hardly ever wait for each other.  In the end the collected entries are added
// in 64 bits and ranked by counting.  The second kernel, a block per sequence, joins the parts of each row and takes the n
// largest of their candidates the same way.
//
// Candidates are compared by sums in 64 bits, and the logarithm is taken in 64.  What goes into it is less exact: the collected entries' exp
// runs in 64 bits, that of the others in 32, and their results are added without rounding (below).  An entry d = bound - x below the bound
// has an exponent d log2 e, rounded (with the difference and the constant) by less than 1.5 x 2^-20 for d up to 11, and ex2 and a change of the
// bound add 2^-22 each; entries further below have no weight beside the bound's n unless there are more than 2^17 of them.  So a row's
// logarithm is off by less than 2^-19 where it has up to 2^18 entries (2^-20.9 was the most that rows made for it gave), the same for all
// candidates of a beam: their order is that of the logits, and candidates of different beams that are closer than 2^-18 may change places.
//
// What bounds it: for many rows the reading of the logits, for few the chain of small steps (loads, barriers, 64-bit exp and log).
// Measured: 64 sequences x 8 beams x 131072 entries, 268 MB: 58 us (4.6 TB/s); 8 x 4 x 32000: 9 us; 1 x 2 x 256: 7 us, 4 of them the
// second kernel.  One kernel, a cluster of blocks per sequence, took 0 to 1 us more for few rows and 4 to 5 more for 512 (a cluster
// waits for its slowest block).
//
// An entry that is NaN counts as -inf, +inf as the largest finite number; an entry of -inf is no candidate.
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "pdl.cuh"

#define BS_THREADS 256
#define BS_CAP 1024        // entries that may reach the bound before the slow way is taken
#define BS_MAX_N 128
#define LOG2E 1.4426950408889634f

typedef unsigned long long u64;

// larger number -> larger key
__device__ __forceinline__ uint32_t bs_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float bs_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// a number that does not order as one (NaN) as -inf, +inf as the largest finite one
__device__ __forceinline__ float bs_clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }
// two 32-bit numbers in one register pair, and sm_100's arithmetic on them
__device__ __forceinline__ u64 bs_pair(float a, float b) {
  u64 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void bs_unpair(u64 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ u64 bs_add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ u64 bs_mul2(u64 a, u64 b) {
  u64 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ u64 bs_fma2(u64 a, u64 b, u64 c) {
  u64 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float bs_max3(float a, float b, float c) {     // (passes over NaN)
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ u64 max_u64(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 bs_warp_max(u64 w) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) w = max_u64(w, __shfl_xor_sync(0xffffffffu, w, o));
  return w;
}

// What the first kernel leaves for the second, per (row, part): the largest entry M, the sum of exp(x - M), how many candidates follow.
struct BsPart {
  double sum;
  float max;
  int count;
};

#define BS_TILE (BS_THREADS * 16)
#define BS_MAX_TILES 32
#define BS_PER_SM 4                // resident blocks

// GS threads form a group (256 / GS >= 2 n groups, or as many as there are threads).
//
// ALIKE: all rows begin at the same place between two 16-byte boundaries of memory (their distance is a multiple of 16 bytes, or there is
// one): entries are read in fours on those boundaries.  Otherwise they are read one by one, a row's first by the first thread.  Either way
// an entry's place in its row alone says which thread adds it, and when, so rows with the same entries have the same sum to the last bit, and
// beams that are alike tie.  (Fours on the boundaries of every row instead: 64 x 8 x 131071 entries 66 us against 61.5, 64 x 8 x 50257 34.7 against
// 35.5, 64 x 4 x 32003 18.0 against 18.5.)
template <int GS, bool ALIKE>
__global__ void __launch_bounds__(BS_THREADS, BS_PER_SM)
beam_rows_kernel(const float* __restrict__ logits, long long ld, int V, const float* __restrict__ scores, int n, int chunk,
                 BsPart* __restrict__ part, uint2* __restrict__ cand) {
  constexpr int GROUPS = BS_THREADS / GS;
  __shared__ u64 gm[GROUPS];
  __shared__ u64 buf[BS_CAP];
  __shared__ u64 bound;
  __shared__ u64 wmax[BS_THREADS / 32];
  __shared__ double wsum[BS_THREADS / 32];
  __shared__ u64 wfixed[BS_THREADS / 32];
  __shared__ int count;
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t slot = (size_t)row * gridDim.x + blockIdx.x;
  const float score = scores[row];
  // In fours: `shift` entries before the row's first belong to the row before.
  const float* x0 = logits + (size_t)row * ld;
  const int shift = ALIKE ? (int)(((uintptr_t)x0 >> 2) & 3) : 0;
  const int first = blockIdx.x * chunk - shift, end = min(first + chunk, V);
  // Entry j of this thread in the tile that begins at i0.
  auto index = [&](int i0, int j) { return ALIKE ? i0 + ((j >> 2) * BS_THREADS + tid) * 4 + (j & 3) : i0 + j * BS_THREADS + tid; };
  const float* mine0 = x0 + first + (ALIKE ? tid * 4 : tid);
  bool nans = false;              // entries that are NaN were met: they become -inf as they are loaded
  auto load = [&](int i0, float (&x)[16]) {
    if (i0 >= 0 && i0 + BS_TILE <= end) {              // (a whole tile)
      const float* p = mine0 + (i0 - first);
      if constexpr (ALIKE) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 v = __ldcs(reinterpret_cast<const float4*>(p + k * BS_THREADS * 4));
          x[4 * k] = v.x; x[4 * k + 1] = v.y; x[4 * k + 2] = v.z; x[4 * k + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = __ldcs(p + j * BS_THREADS);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int i = index(i0, j);
        x[j] = i >= 0 && i < end ? x0[i] : -INFINITY;
      }
    }
    if (nans) {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = fmaxf(x[j], -INFINITY);
    }
  };
  // A word orders entries by value, equal ones (zeros of either sign among them) by index, lowest first.
  auto word = [&](float x, int i) { return ((u64)bs_key(x + 0.0f) << 32) | (uint32_t)~i; };

  float x[16];
  load(first, x);
  if (!(score > -INFINITY)) {     // no beam: its row does not matter (but its first tile is on its way while the score is)
    if (tid == 0) part[slot] = {0.0, -INFINITY, 0};
    return;
  }
  u64 top;                        // the largest entry that this thread knows
  {
    float best = -INFINITY;
    int best_j = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (x[j] > best) { best = x[j]; best_j = j; }
    top = best > -INFINITY ? word(fminf(best, FLT_MAX), index(first, best_j)) : 0;
  }

  // Each exp lies in [0, 1]; 1536 has a last place of 2^-13, so (e + 1536) - 1536 is e's part above that and what is left is exact too.
  // The upper parts of up to 2048 entries add without rounding, and the lower ones' roundings are below 2^-34.  (Another bound
  // scales both sums, which rounds a thread's share of them by 2^-24.)
  float ref = 0.0f, bv;
  u64 b, hi, lo;                  // (sums of two kinds of places)
  const u64 log2e = bs_pair(LOG2E, LOG2E), up = bs_pair(1536.0f, 1536.0f), down = bs_pair(-1536.0f, -1536.0f), minus = bs_pair(-1.0f, -1.0f);
  auto take_bound = [&] {         // 0: fewer than n entries so far, all of which are collected
    b = bound;
    const float now = b ? bs_value((uint32_t)(b >> 32)) : 0.0f;
    bv = b ? now : -INFINITY;
    float f;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(fminf((ref - now) * LOG2E, 0.0f)));
    hi = bs_mul2(hi, bs_pair(f, f));
    lo = bs_mul2(lo, bs_pair(f, f));
    ref = now;
  };
  auto take = [&](int i0, float (&v)[16]) {
    const u64 neg_ref = bs_pair(-ref, -ref);
#pragma unroll
    for (int k = 0; k < 16; k += 8) {
      const float m8 = bs_max3(bs_max3(v[k], v[k + 1], v[k + 2]), bs_max3(v[k + 3], v[k + 4], v[k + 5]), fmaxf(v[k + 6], v[k + 7]));
      if (__any_sync(0xffffffffu, m8 >= bv)) {       // (a vote, so that this is a branch)
#pragma unroll
        for (int e = k; e < k + 8; ++e) {
          if (v[e] >= bv && v[e] > -INFINITY) {
            v[e] = fminf(v[e], FLT_MAX);     // (+inf comes here under every bound; one behind the bound's place is summed as what it counts as)
            const u64 w = word(v[e], index(i0, e));
            if (w >= b) {
              const int at = atomicAdd(&count, 1);
              if (at < BS_CAP) buf[at] = w;
              v[e] = -INFINITY;
            }
          }
        }
      }
#pragma unroll
      for (int e = k; e < k + 8; e += 2) {
        float p0, p1;
        bs_unpair(bs_mul2(bs_add2(bs_pair(v[e], v[e + 1]), neg_ref), log2e), p0, p1);
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(p0));
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(p1));
        const u64 p = bs_pair(p0, p1), h = bs_add2(bs_add2(p, up), down);
        hi = bs_add2(hi, h);
        lo = bs_add2(lo, bs_fma2(h, minus, p));
      }
    }
  };
  b = 0;
  bool groups = true, scanned = false;
  for (;;) {
    if (groups) {                 // the n-th largest of the groups' maxima (but for empty groups they all differ: an index is part of each)
      u64 w = top;
#pragma unroll
      for (int o = 1; o < GS; o <<= 1) w = max_u64(w, __shfl_xor_sync(0xffffffffu, w, o));
      if (tid % GS == 0) gm[tid / GS] = w;
      if (tid == 0) count = 0;
      __syncthreads();
      if (tid < GROUPS) {
        const u64 mine = gm[tid];
        int rank = 0;
#pragma unroll 8
        for (int k = 0; k < GROUPS; ++k) rank += gm[k] > mine || (gm[k] == mine && k < tid) ? 1 : 0;
        if (rank == (n < GROUPS ? n : GROUPS) - 1) bound = max_u64(mine, b);
      }
      __syncthreads();
    }
    hi = lo = bs_pair(0.0f, 0.0f);
    take_bound();
    int next = first + BS_TILE;   // where the bound is looked at again: after 1, 2, 4, ... tiles
    auto look = [&](int i0) -> bool {      // true: more were collected than there is room for
      if (i0 != next || next >= end) return false;
      next = first + 2 * (next - first);
      __syncthreads();
      const int c = count;
      if (c > BS_CAP) return true;
      for (int i = tid; i < c; i += BS_THREADS) {
        const u64 mine = buf[i];
        int rank = 0;
#pragma unroll 8
        for (int k = 0; k < c; ++k) rank += buf[k] > mine ? 1 : 0;
        if (rank == n - 1) bound = mine;
      }
      __syncthreads();
      take_bound();
      return false;
    };
#pragma unroll 1
    for (int i0 = first; i0 < end; i0 += 2 * BS_TILE) {
      float y[16];
      if (i0 + BS_TILE < end) load(i0 + BS_TILE, y);           // the next tile is on its way while one is summed
      take(i0, x);
      if (look(i0 + BS_TILE) || i0 + BS_TILE >= end) break;
      if (i0 + 2 * BS_TILE < end) load(i0 + 2 * BS_TILE, x);
      take(i0 + BS_TILE, y);
      if (look(i0 + 2 * BS_TILE)) break;
    }
    // a NaN has come into a sum: once more without, and with the bound that has been found
    float h0, h1;
    bs_unpair(hi, h0, h1);
    if (__syncthreads_or(!nans && h0 + h1 != h0 + h1)) {
      nans = true;
      groups = false;
      if (tid == 0) count = 0;
      load(first, x);
      __syncthreads();
      continue;
    }
    if (count <= BS_CAP) break;
    // More entries were collected than there is room for: they rise along the row, so the bound is looked for again among all of the part
    // (the largest entries of a vocabulary at its end, 64 x 8 x 131072: 4.1 ms without this,
    // 0.35 so; it costs others 2 %).
    if (!scanned) {
      scanned = groups = true;
      top = 0;
#pragma unroll 4
      for (int i = first + tid; i < end; i += BS_THREADS) {
        const float v = i >= 0 ? bs_clean(x0[i]) : -INFINITY;
        if (v > -INFINITY) top = max_u64(top, word(v, i));
      }
      load(first, x);
      __syncthreads();            // (everyone has read the count)
      continue;
    }
    // Or they bunch in few groups: the n-th largest of the part, found one after the other, each the largest below the one before;
    // then the same again with that as the bound.
    groups = false;
    u64 last = ~0ull;
    for (int r = 0; r < n; ++r) {
      u64 w = 0;
#pragma unroll 1
      for (int i = first + tid; i < end; i += BS_THREADS) {
        const float v = i >= 0 ? bs_clean(x0[i]) : -INFINITY;
        const u64 wi = word(v, i);
        if (v > -INFINITY && wi < last) w = max_u64(w, wi);
      }
      w = bs_warp_max(w);
      if (lane == 0) wmax[warp] = w;
      __syncthreads();
      for (int k = 0; k < BS_THREADS / 32; ++k) w = max_u64(w, wmax[k]);
      __syncthreads();
      last = w;                   // more than BS_CAP >= n entries are there, so w is one
    }
    if (tid == 0) { bound = last; count = 0; }
    __syncthreads();
    load(first, x);
  }

  // ---- the part's maximum, its sum, its n largest
  const int c = count;
  if (c == 0) {                   // nothing here can follow
    if (tid == 0) part[slot] = {0.0, -INFINITY, 0};
    return;
  }
  u64 w = 0;
  for (int i = tid; i < c; i += BS_THREADS) w = max_u64(w, buf[i]);
  w = bs_warp_max(w);
  if (lane == 0) wmax[warp] = w;
  __syncthreads();
  const float M = bs_value((uint32_t)(bs_warp_max(wmax[lane & (BS_THREADS / 32 - 1)]) >> 32));
  // the entries that were not collected, then the collected ones
  double rest;
  {
    float h0, h1, l0, l1;
    bs_unpair(hi, h0, h1);
    bs_unpair(lo, l0, l1);
    rest = ((double)h0 + (double)h1) + ((double)l0 + (double)l1);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
  // The collected ones lie in no particular order: they are added as whole multiples of 2^-52, so that the sum does not depend on it (at
  // most 1024 of at most 1).  (Lane 0 of a warp has the warp's rest beside its entries.)
  double sum = 0.0;
  u64 fixed = 0;
  for (int i = lane == 0 ? tid - BS_THREADS : tid; i < c; i += BS_THREADS) {
    const double at = i < 0 ? (double)ref : (double)bs_value((uint32_t)(buf[i] >> 32));
    if (i < 0 && rest == 0.0) continue;
    const double e = exp(at - (double)M);
    if (i < 0) sum = rest * e; else fixed += (u64)(e * 4503599627370496.0);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) fixed += __shfl_xor_sync(0xffffffffu, fixed, o);
  if (lane == 0) {
    wsum[warp] = sum;
    wfixed[warp] = fixed;
  }
  uint2* out = cand + slot * n;
  for (int i = tid; i < c; i += BS_THREADS) {
    const u64 mine = buf[i];
    if (mine < b) continue;       // (n entries reach the last bound)
    int rank = 0;
#pragma unroll 8
    for (int k = 0; k < c; ++k) rank += buf[k] > mine ? 1 : 0;
    if (rank < n) out[rank] = make_uint2((uint32_t)(mine >> 32), ~(uint32_t)mine);
  }
  __syncthreads();
  if (warp == 0) {
    sum = lane < BS_THREADS / 32 ? wsum[lane] : 0.0;
    fixed = lane < BS_THREADS / 32 ? wfixed[lane] : 0;
#pragma unroll
    for (int o = BS_THREADS / 64; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      fixed += __shfl_xor_sync(0xffffffffu, fixed, o);
    }
    if (lane == 0) part[slot] = {sum + (double)fixed * 2.220446049250313e-16, M, c < n ? c : n};
  }
}

// A candidate's value as a word that orders as it does (0: none; both zeros are one), and what comes first where values are equal: the lower
// beam (10 bits), its larger logit (32 bits; sums far from zero may be equal where logits are not), the lower token (22 bits: the place in the beam's lists of
// candidates, which have equal logits in the order of their tokens).
struct __align__(16) BsCand {
  u64 v;
  u64 tie;
};
#define BS_NONE ~0ull
#define BS_PLACE_BITS 22
#define BS_BEAM_SHIFT (32 + BS_PLACE_BITS)
__device__ __forceinline__ u64 bs_key64(double x) {
  const u64 u = (u64)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double bs_value64(u64 k) { return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k)); }
// 1 where a comes before b: the borrow of (b.v, a.tie) - (a.v, b.tie) as numbers of 128 bits.  (As an expression it becomes a branch where the
// first half ties: 64 x 8 x 50257 entries 39.2 us.)
__device__ __forceinline__ int bs_before(const BsCand& a, const BsCand& b) {
  int borrow;
  asm("{\n\t.reg .u64 t;\n\t"
      "sub.cc.u64 t, %1, %2;\n\t"
      "subc.cc.u64 t, %3, %4;\n\t"
      "subc.u32 %0, 0, 0;\n\t}"
      : "=r"(borrow)
      : "l"(a.tie), "l"(b.tie), "l"(b.v), "l"(a.v));
  return -borrow;
}
// How many of list[0 .. c) come before `mine`.  (Eight loads, then comparisons without branches: taken one by one, with the second half of a
// comparison only where the first ties, 32 of them took 7000 cycles and the whole selection half as long again.)
__device__ __forceinline__ int bs_rank(const BsCand* list, int c, const BsCand& mine) {
  int rank = 0, k = 0;
  for (; k + 8 <= c; k += 8) {
    BsCand o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = list[k + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) rank += bs_before(o[i], mine);
  }
#pragma unroll 1
  for (; k < c; ++k) rank += bs_before(list[k], mine);
  return rank;
}
__device__ __forceinline__ BsCand bs_shfl(const BsCand& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.v, o), __shfl_xor_sync(0xffffffffu, a.tie, o)};
}

// CAND: candidates of a sequence per thread that are held in registers; 0: any number, read again for every look at them.  (The bound on
// registers is for the order of the code: without it 64 sequences of 8 beams take 4 us more.)
template <int GS, int CAND>
__global__ void __launch_bounds__(BS_THREADS, 4)
beam_merge_kernel(const BsPart* __restrict__ part, const uint2* __restrict__ cand, const float* __restrict__ scores, int B,
                  int n, int parts, float* __restrict__ values, int* __restrict__ beams, int* __restrict__ tokens) {
  constexpr int GROUPS = BS_THREADS / GS, HELD = CAND ? CAND : 1;
  extern __shared__ double lse[];         // [B]
  __shared__ BsCand gm[GROUPS];
  __shared__ BsCand buf[BS_CAP];
  __shared__ uint32_t token_of[BS_CAP];
  __shared__ BsCand bound;
  __shared__ int count;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row0 = (size_t)s * B;
  const int total = B * parts * n;
  const BsCand none = {0, BS_NONE};
  if (tid == 0) count = 0;
  pdl_wait();
  pdl_launch_dependents();
  // candidate i: its value without its beam's share, and which beam's; everything is on its way before the first is waited for
  struct Raw {
    uint32_t key, token;
    float score;
    int beam, left;                       // left: how many follow it and itself; none if it is not positive
  };
  auto raw = [&](int i) -> Raw {
    if (i >= total) return {0u, 0u, 0.0f, 0, 0};
    const int k = i / n, b = k / parts;
    const uint2 c = cand[row0 * parts * n + i];
    return {c.x, c.y, scores[row0 + b], b, part[row0 * parts + k].count - (i - k * n)};
  };
  auto value = [&](const Raw& r, int i) -> BsCand {
    if (r.left <= 0) return none;
    return {bs_key64((double)r.score + ((double)bs_value(r.key) - lse[r.beam])),
            (u64)r.beam << BS_BEAM_SHIFT | (u64)~r.key << BS_PLACE_BITS | (uint32_t)(i - r.beam * parts * n)};
  };
  auto part_of = [&](int b) -> BsPart {
    if (b < B && lane < parts) return part[(row0 + b) * parts + lane];
    return {0.0, -INFINITY, 0};
  };
  BsPart q = part_of(warp);
  Raw held[HELD];
  if (CAND) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) held[j] = raw(tid + j * BS_THREADS);
  }
  // a warp per row: its maximum, its sum
  for (int b = warp; b < B; b += BS_THREADS / 32) {
    const BsPart* p = part + (row0 + b) * parts;
    float M = q.max;
    for (int i = lane + 32; i < parts; i += 32) M = fmaxf(M, p[i].max);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    double sum = 0.0;
    for (int i = lane; i < parts; i += 32) {
      if (i >= 32) q = p[i];
      if (q.count) sum += q.max == M ? q.sum : q.sum * exp((double)q.max - (double)M);
    }
    if (parts > 1) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane == 0) lse[b] = (double)M + log(sum);       // (a row without entries: not used)
    q = part_of(b + BS_THREADS / 32);
  }
  __syncthreads();
  BsCand mine[HELD], best = none;
  if (CAND) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      mine[j] = value(held[j], tid + j * BS_THREADS);
      if (bs_before(mine[j], best)) best = mine[j];
    }
  } else {
    for (int i = tid; i < total; i += BS_THREADS) {
      const BsCand e = value(raw(i), i);
      if (bs_before(e, best)) best = e;
    }
  }
#pragma unroll
  for (int o = 1; o < GS; o <<= 1) {
    const BsCand other = bs_shfl(best, o);
    if (bs_before(other, best)) best = other;
  }
  if (best.v == 0) best.tie = BS_NONE - tid / GS;          // (empty groups come one after the other)
  if (tid % GS == 0) gm[tid / GS] = best;
  __syncthreads();
  if (tid < GROUPS) {
    const BsCand of = gm[tid];
    const int rank = bs_rank(gm, GROUPS, of);
    if (rank == (n < GROUPS ? n : GROUPS) - 1) bound = of;
  }
  __syncthreads();
  BsCand bd = bound;
  auto collect = [&](const BsCand& e, uint32_t token) {
    if (e.tie != BS_NONE && !bs_before(bd, e)) {
      const int at = atomicAdd(&count, 1);
      if (at < BS_CAP) {
        buf[at] = e;
        token_of[at] = token;
      }
    }
  };
  if (CAND) {                             // (held candidates are at most as many as there is room for)
#pragma unroll
    for (int j = 0; j < HELD; ++j) collect(mine[j], held[j].token);
    __syncthreads();
  } else {
    for (;;) {
      for (int i = tid; i < total; i += BS_THREADS) {
        const Raw r = raw(i);
        collect(value(r, i), r.token);
      }
      __syncthreads();
      if (count <= BS_CAP) break;
      // more reach the bound than there is room for: the n-th of those collected is the next one (which leaves out all but n of them)
      for (int i = tid; i < BS_CAP; i += BS_THREADS) {
        const BsCand e = buf[i];
        if (bs_rank(buf, BS_CAP, e) == n - 1) bound = e;
      }
      __syncthreads();
      bd = bound;
      if (tid == 0) count = 0;
      __syncthreads();
    }
  }
  const int c = count;
  const size_t o0 = (size_t)s * n;
  auto put = [&](int r, const BsCand& e, int token) {
    const double v = bs_value64(e.v);
    const bool got = e.tie != BS_NONE && v > -INFINITY;
    values[o0 + r] = got ? (float)v : -INFINITY;
    beams[o0 + r] = got ? (int)(e.tie >> BS_BEAM_SHIFT) : -1;
    tokens[o0 + r] = got ? token : -1;
  };
  for (int i = tid; i < max(c, n); i += BS_THREADS) {
    BsCand e = none;
    int rank = i, token = -1;             // places without a candidate
    if (i < c) {
      e = buf[i];
      token = (int)token_of[i];
      rank = bs_rank(buf, c, e);
    }
    if (rank < n) put(rank, e, token);
  }
}

// Entries of a row per block: the fewest tiles (the most blocks) that leave at most as many blocks as run at once on 148 SMs; BS_MAX_TILES at
// most.
static int bs_chunk(int rows, int V) {
  for (int tiles = 1; tiles < BS_MAX_TILES; tiles *= 2)
    if ((long long)rows * ((V + BS_TILE * tiles - 1) / (BS_TILE * tiles)) <= 148 * BS_PER_SM) return BS_TILE * tiles;
  return BS_TILE * BS_MAX_TILES;
}
// (rows that do not begin on 16-byte boundaries are shifted by up to three entries)
static int bs_parts(int V, int chunk, bool shifted) { return (int)(((long long)V + (shifted ? 3 : 0) + chunk - 1) / chunk); }

extern "C" long long tl_beam_scratch_bytes(int rows, int V, int n) {
  return (long long)rows * bs_parts(V, bs_chunk(rows, V), true) * ((long long)sizeof(BsPart) + 8 * n);
}

template <int GS>
static int bs_run(const float* logits, long long ld, int S, int B, int V, const float* scores, int n, void* scratch, float* values,
                  int* beams, int* tokens, cudaStream_t stream) {
  const int rows = S * B;
  const bool alike = rows == 1 || ld % 4 == 0, shifted = alike && ((uintptr_t)logits & 15);
  int chunk = bs_chunk(rows, V);
  // Longer parts where they leave no more candidates than the second kernel's threads hold: one sequence of 8 beams, 16 continuations, 262144
  // entries: parts of one tile 33 us, of 8 tiles 19 us; 16 beams, 32 continuations, 131072 entries 146 and 33.  (More than 8
  // tiles gain no more.)
  while ((long long)B * bs_parts(V, chunk, shifted) * n > 4 * BS_THREADS && chunk < 8 * BS_TILE && chunk < V) chunk *= 2;
  const int parts = bs_parts(V, chunk, shifted);
  if ((long long)parts * n >= 1ll << BS_PLACE_BITS) return -2;     // (2^30 entries have some 2^13 parts)
  BsPart* part = (BsPart*)scratch;
  uint2* cand = (uint2*)(part + (size_t)rows * parts);
  const int st = alike ? tl_launch(beam_rows_kernel<GS, true>, dim3(parts, rows), dim3(BS_THREADS), 0, stream, logits, ld, V, scores, n, chunk, part, cand)
                       : tl_launch(beam_rows_kernel<GS, false>, dim3(parts, rows), dim3(BS_THREADS), 0, stream, logits, ld, V, scores, n, chunk, part, cand);
  if (st) return st;
  const long long total = (long long)B * parts * n;
  auto merge = [&](auto kernel) {
    return tl_launch(kernel, dim3(S), dim3(BS_THREADS), (size_t)B * sizeof(double), stream, (const BsPart*)part, (const uint2*)cand, scores, B,
                     n, parts, values, beams, tokens);
  };
  return total <= BS_THREADS ? merge(beam_merge_kernel<GS, 1>) : total <= 4 * BS_THREADS ? merge(beam_merge_kernel<GS, 4>) : merge(beam_merge_kernel<GS, 0>);
}

// logits [S * B] rows of V entries, `ld` apart; scores [S * B]; values, beams, tokens [S * n].  `scratch`: tl_beam_scratch_bytes,
// 16-byte aligned.
extern "C" int tl_beam_select(const float* logits, long long ld, int S, int B, int V, const float* scores, int n, void* scratch,
                              float* values, int* beams, int* tokens, cudaStream_t stream) {
  if (S <= 0) return 0;
  if (B <= 0 || V <= 0 || n <= 0 || ld < V || ((uintptr_t)logits & 3)) return -1;
  if (V > (1 << 30)) return -2;
  if (n > BS_MAX_N || B > 1 << (64 - BS_BEAM_SHIFT) || (long long)S * B > 65535 || (long long)B * V >= 0x7fffffffLL ||
      (long long)B * bs_parts(V, BS_TILE, true) * n >= 0x7fffffffLL)
    return -2;
  // twice as many groups as entries are asked for, where there are
  if (n <= 16) return bs_run<8>(logits, ld, S, B, V, scores, n, scratch, values, beams, tokens, stream);
  if (n <= 32) return bs_run<4>(logits, ld, S, B, V, scores, n, scratch, values, beams, tokens, stream);
  if (n <= 64) return bs_run<2>(logits, ld, S, B, V, scores, n, scratch, values, beams, tokens, stream);
  return bs_run<1>(logits, ld, S, B, V, scores, n, scratch, values, beams, tokens, stream);
}
