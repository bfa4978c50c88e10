// The selection step of a beam search: of a sequence's beams and all their next tokens, the n continuations of the highest
// log-probability.  (The reference keeps one continuation and has no such step; its softmax over a row is
// src/sampler/mod.rs:119-143.)
//
//   v(b, t) = c_b + x_bt - log sum_u exp x_bu        the n largest of all (b, t) in falling order; ties: lowest (b, t) first
//
// Two kernels.  The first reads every row once: a block holds a part of a row in registers, takes its maximum M and the
// sum of exp(x - M), and keeps its n largest entries.  Within a row the constant c_b - lse does not matter, so a part's n
// largest x are all that can become a candidate.  Which those are: the threads form groups, and the n-th largest of the
// groups' maxima is a bound that at least n entries reach; few others do (22 for n = 16), those go to shared memory and are
// ranked by counting.  The second kernel, a block per sequence, joins the parts of each row and takes the n
// largest of the parts' candidates the same way.
//
// Candidates of different beams are compared by sums of 32-bit numbers whose logarithm is rounded too, so which comes first is decided
// in 64 bits: exp runs in 32 bits, but its results are added without rounding (below), the parts' sums are joined in 64 bits, and the
// entries with weight (each part's n largest) are then exchanged for their exp in 64 bits.
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
__device__ __forceinline__ float bs_exp(float x, float m) {   // 0 for x = -inf; m is finite
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((x - m) * LOG2E));
  return e;
}
__device__ __forceinline__ u64 max_u64(u64 a, u64 b) { return a > b ? a : b; }

// What the first kernel leaves for the second, per (row, part): the part's maximum and sum, how many candidates follow.
struct BsPart {
  double sum;
  float max;
  int count;
};

// E entries per thread; GS threads form a group (256 / GS >= 2 n groups, or as many as there are threads).
template <int E, int GS>
__global__ void __launch_bounds__(BS_THREADS)
beam_rows_kernel(const float* __restrict__ logits, long long ld, int V, const float* __restrict__ scores, int n, int parts,
                 BsPart* __restrict__ part, uint2* __restrict__ cand) {
  constexpr int GROUPS = BS_THREADS / GS;
  __shared__ u64 gm[GROUPS];
  __shared__ u64 buf[BS_CAP];
  __shared__ u64 bound;
  __shared__ u64 wmax[BS_THREADS / 32];
  __shared__ double wsum[BS_THREADS / 32];
  __shared__ int count;
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t slot = (size_t)row * parts + blockIdx.x;
  const float score = scores[row];
  if (!(score > -INFINITY)) {     // no beam: its row is not read
    if (tid == 0) part[slot] = {0.0, -INFINITY, 0};
    return;
  }
  // The entries in fours on 16-byte boundaries of memory: `shift` entries before the row's first belong to the row before.
  const float* x0 = logits + (size_t)row * ld;
  const int shift = (int)(((uintptr_t)x0 >> 2) & 3);
  const int first = blockIdx.x * (BS_THREADS * E) - shift;
  float x[E];
#pragma unroll
  for (int k = 0; k < E / 4; ++k) {
    const int i = first + (k * BS_THREADS + tid) * 4;
    if (i >= 0 && i + 3 < V) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(x0 + i));
      x[4 * k] = v.x; x[4 * k + 1] = v.y; x[4 * k + 2] = v.z; x[4 * k + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * k + e] = i + e >= 0 && i + e < V ? x0[i + e] : -INFINITY;
    }
  }
  // entry number k * 4 + e of this thread; a word orders entries by value, equal ones by index, lowest first
  auto index = [&](int j) { return first + ((j >> 2) * BS_THREADS + tid) * 4 + (j & 3); };
  auto word = [&](int j) { return ((u64)bs_key(x[j]) << 32) | (uint32_t)~index(j); };
  float best = -INFINITY;
  int best_j = 0;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    x[j] = bs_clean(x[j]);
    if (x[j] > best) { best = x[j]; best_j = j; }
  }
  u64 w = ((u64)bs_key(best) << 32) | (uint32_t)~index(best_j);
#pragma unroll
  for (int o = 1; o < GS; o <<= 1) w = max_u64(w, __shfl_xor_sync(0xffffffffu, w, o));
  if (tid % GS == 0) gm[tid / GS] = w;
  if (tid == 0) count = 0;
  __syncthreads();
  // the block's maximum, in every warp
  u64 top = 0;
#pragma unroll
  for (int k = 0; k < GROUPS; k += 32) top = max_u64(top, gm[k + lane]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_u64(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float M = bs_value((uint32_t)(top >> 32));
  if (M == -INFINITY) {           // nothing here can follow (the same in all threads)
    if (tid == 0) part[slot] = {0.0, -INFINITY, 0};
    return;
  }
  if (tid < GROUPS) {             // the n-th largest of the groups' maxima (they all differ: an index is part of each)
    const u64 mine = gm[tid];
    int rank = 0;
#pragma unroll 8
    for (int k = 0; k < GROUPS; ++k) rank += gm[k] > mine ? 1 : 0;
    if (rank == (n < GROUPS ? n : GROUPS) - 1) bound = mine;
  }
  // Each exp lies in [0, 1]; 1536 has a last place of 2^-13, so (e + 1536) - 1536 is e's part above that and what is left is exact too.
  // Up to 32 upper parts add without rounding, and the lower ones' roundings are below 2^-37.
  float hi = 0.0f, lo = 0.0f;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const float e = bs_exp(x[j], M);
    const float h = __fsub_rn(__fadd_rn(e, 1536.0f), 1536.0f);
    hi += h;
    lo += e - h;
  }
  double sum = (double)hi + (double)lo;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) wsum[warp] = sum;
  __syncthreads();
  const u64 b = bound;
  const float bv = bs_value((uint32_t)(b >> 32));
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if (x[j] >= bv && x[j] > -INFINITY) {
      const u64 wj = word(j);
      if (wj >= b) {
        const int at = atomicAdd(&count, 1);
        if (at < BS_CAP) buf[at] = wj;
      }
    }
  }
  __syncthreads();
  const int c = count;
  uint2* out = cand + slot * n;
  if (c <= BS_CAP) {
    for (int i = tid; i < c; i += BS_THREADS) {
      const u64 mine = buf[i];
      int rank = 0;
      for (int k = 0; k < c; ++k) rank += buf[k] > mine ? 1 : 0;
      if (rank < n) out[rank] = make_uint2((uint32_t)(mine >> 32), ~(uint32_t)mine);
    }
  } else {
    // entries bunch in fewer than n groups: one after the other, each the largest below the one before
    u64 last = ~0ull;
    for (int r = 0; r < n; ++r) {
      u64 m = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const u64 wj = word(j);
        if (x[j] > -INFINITY && wj < last) m = max_u64(m, wj);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = max_u64(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (lane == 0) wmax[warp] = m;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < BS_THREADS / 32; ++k) m = max_u64(m, wmax[k]);
      __syncthreads();
      last = m;                   // more than BS_CAP >= n entries are there, so m is one
      if (tid == 0) out[r] = make_uint2((uint32_t)(m >> 32), ~(uint32_t)m);
    }
  }
  if (tid == 0) {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < BS_THREADS / 32; ++k) s += wsum[k];
    part[slot] = {s, M, c < n ? c : n};
  }
}

struct BsCand {
  double v;
  uint32_t at;          // beam * V + token
};
__device__ __forceinline__ bool bs_before(const BsCand& a, const BsCand& b) { return a.v > b.v || (a.v == b.v && a.at < b.at); }
__device__ __forceinline__ BsCand bs_shfl(const BsCand& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.v, o), __shfl_xor_sync(0xffffffffu, a.at, o)};
}

template <int GS>
__global__ void __launch_bounds__(BS_THREADS)
beam_merge_kernel(const BsPart* __restrict__ part, const uint2* __restrict__ cand, const float* __restrict__ scores, int B, int V,
                  int n, int parts, float* __restrict__ values, int* __restrict__ beams, int* __restrict__ tokens) {
  constexpr int GROUPS = BS_THREADS / GS;
  extern __shared__ double base[];        // [B]: c_b - lse_b
  __shared__ BsCand gm[GROUPS];
  __shared__ BsCand buf[BS_CAP];
  __shared__ BsCand bound;
  __shared__ BsCand wbest[BS_THREADS / 32];
  __shared__ int count;
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row0 = (size_t)s * B;
  const BsCand none = {-INFINITY, 0xffffffffu};
  // a warp per row: its maximum, its sum, the entries with weight exchanged for their exp in 64 bits
  for (int b = warp; b < B; b += BS_THREADS / 32) {
    const BsPart* p = part + (row0 + b) * parts;
    float M = -INFINITY;
    for (int i = lane; i < parts; i += 32) M = fmaxf(M, p[i].max);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (M == -INFINITY) {
      if (lane == 0) base[b] = -INFINITY;
      continue;
    }
    double sum = 0.0;
    for (int i = lane; i < parts; i += 32)
      if (p[i].count) sum += p[i].sum * exp((double)p[i].max - (double)M);
    const uint2* c = cand + (row0 + b) * parts * n;
    for (int i = lane; i < parts * n; i += 32) {
      const int k = i / n;
      const BsPart q = p[k];
      if (i - k * n < q.count) {
        const float x = bs_value(c[i].x);
        // (a part far below the row's maximum has no weight; neither has an entry 2^-20 of it)
        if (x - M > -14.0f) sum += exp((double)x - (double)M) - (double)bs_exp(x, q.max) * exp((double)q.max - (double)M);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) base[b] = (double)M + log(sum);      // lse
  }
  if (tid == 0) count = 0;
  __syncthreads();
  const int total = B * parts * n;
  auto entry = [&](int i) -> BsCand {
    const int k = i / n, b = k / parts;
    if (i - k * n >= part[row0 * parts + k].count) return none;
    const uint2 c = cand[row0 * parts * n + i];
    return {(double)scores[row0 + b] + ((double)bs_value(c.x) - base[b]), (uint32_t)b * (uint32_t)V + c.y};
  };
  BsCand best = none;
  for (int i = tid; i < total; i += BS_THREADS) {
    const BsCand e = entry(i);
    if (bs_before(e, best)) best = e;
  }
#pragma unroll
  for (int o = 1; o < GS; o <<= 1) {
    const BsCand other = bs_shfl(best, o);
    if (bs_before(other, best)) best = other;
  }
  if (tid % GS == 0) gm[tid / GS] = best;
  __syncthreads();
  if (tid < GROUPS) {
    const BsCand mine = gm[tid];
    int rank = 0;
#pragma unroll 4
    for (int k = 0; k < GROUPS; ++k) rank += bs_before(gm[k], mine) || (k < tid && gm[k].at == mine.at) ? 1 : 0;   // (empty groups are equal)
    if (rank == (n < GROUPS ? n : GROUPS) - 1) bound = mine;
  }
  __syncthreads();
  const BsCand bd = bound;
  for (int i = tid; i < total; i += BS_THREADS) {
    const BsCand e = entry(i);
    if (e.at != 0xffffffffu && !bs_before(bd, e)) {
      const int at = atomicAdd(&count, 1);
      if (at < BS_CAP) buf[at] = e;
    }
  }
  __syncthreads();
  const int c = count;
  const size_t o0 = (size_t)s * n;
  auto put = [&](int r, const BsCand& e) {
    const bool got = e.at != 0xffffffffu && e.v > -INFINITY;
    values[o0 + r] = got ? (float)e.v : -INFINITY;
    beams[o0 + r] = got ? (int)(e.at / (uint32_t)V) : -1;
    tokens[o0 + r] = got ? (int)(e.at % (uint32_t)V) : -1;
  };
  if (c <= BS_CAP) {
    for (int i = tid; i < c; i += BS_THREADS) {
      const BsCand mine = buf[i];
      int rank = 0;
      for (int k = 0; k < c; ++k) rank += bs_before(buf[k], mine) ? 1 : 0;
      if (rank < n) put(rank, mine);
    }
    for (int r = c + tid; r < n; r += BS_THREADS) put(r, none);
  } else {
    BsCand last = {INFINITY, 0u};
    for (int r = 0; r < n; ++r) {
      BsCand m = none;
      for (int i = tid; i < total; i += BS_THREADS) {
        const BsCand e = entry(i);
        if (e.at != 0xffffffffu && (r == 0 || bs_before(last, e)) && bs_before(e, m)) m = e;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const BsCand other = bs_shfl(m, o);
        if (bs_before(other, m)) m = other;
      }
      if (lane == 0) wbest[warp] = m;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < BS_THREADS / 32; ++k)
        if (bs_before(wbest[k], m)) m = wbest[k];
      __syncthreads();
      last = m;
      if (tid == 0) put(r, m);
    }
  }
}

// Entries per thread: the fewest (the most blocks) that leave at most eight blocks of a row or so on each of 148 SMs.
static int bs_entries(int rows, int V) {
  for (int e = 4; e < 32; e *= 2)
    if ((long long)rows * ((V + BS_THREADS * e - 1) / (BS_THREADS * e)) <= 148 * 8) return e;
  return 32;
}
static int bs_parts(int V, int e) { return (int)(((long long)V + 3 + BS_THREADS * e - 1) / (BS_THREADS * e)); }   // + 3: a shifted row

extern "C" long long tl_beam_scratch_bytes(int rows, int V, int n) {
  return (long long)rows * bs_parts(V, bs_entries(rows, V)) * ((long long)sizeof(BsPart) + 8 * n);
}

template <int GS>
static int bs_run(const float* logits, long long ld, int S, int B, int V, const float* scores, int n, void* scratch, float* values,
                  int* beams, int* tokens, cudaStream_t stream) {
  const int rows = S * B, e = bs_entries(rows, V), parts = bs_parts(V, e);
  BsPart* part = (BsPart*)scratch;
  uint2* cand = (uint2*)(part + (size_t)rows * parts);
  const dim3 grid(parts, rows), block(BS_THREADS);
  const int st = e == 4    ? tl_launch(beam_rows_kernel<4, GS>, grid, block, 0, stream, logits, ld, V, scores, n, parts, part, cand)
                 : e == 8  ? tl_launch(beam_rows_kernel<8, GS>, grid, block, 0, stream, logits, ld, V, scores, n, parts, part, cand)
                 : e == 16 ? tl_launch(beam_rows_kernel<16, GS>, grid, block, 0, stream, logits, ld, V, scores, n, parts, part, cand)
                           : tl_launch(beam_rows_kernel<32, GS>, grid, block, 0, stream, logits, ld, V, scores, n, parts, part, cand);
  if (st) return st;
  return tl_launch(beam_merge_kernel<GS>, dim3(S), block, (size_t)B * sizeof(double), stream, (const BsPart*)part, (const uint2*)cand,
                   scores, B, V, n, parts, values, beams, tokens);
}

// logits [S * B] rows of V entries, `ld` apart; scores [S * B]; values, beams, tokens [S * n].  `scratch`: tl_beam_scratch_bytes,
// 16-byte aligned.
extern "C" int tl_beam_select(const float* logits, long long ld, int S, int B, int V, const float* scores, int n, void* scratch,
                              float* values, int* beams, int* tokens, cudaStream_t stream) {
  if (S <= 0) return 0;
  if (B <= 0 || V <= 0 || n <= 0 || ld < V || ((uintptr_t)logits & 3)) return -1;
  if (V > (1 << 30)) return -2;
  if (n > BS_MAX_N || B > 1024 || (long long)S * B > 65535 || (long long)B * V >= 0x7fffffffLL ||
      (long long)B * bs_parts(V, 4) * n >= 0x7fffffffLL)
    return -2;
  // twice as many groups as entries are asked for, where there are
  if (n <= 16) return bs_run<8>(logits, ld, S, B, V, scores, n, scratch, values, beams, tokens, stream);
  if (n <= 32) return bs_run<4>(logits, ld, S, B, V, scores, n, scratch, values, beams, tokens, stream);
  if (n <= 64) return bs_run<2>(logits, ld, S, B, V, scores, n, scratch, values, beams, tokens, stream);
  return bs_run<1>(logits, ld, S, B, V, scores, n, scratch, values, beams, tokens, stream);
}
