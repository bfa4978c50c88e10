// Decode attention of rows that share the leading pages of their cache: the beams of a search, which have one prompt.
// (Per row and head as everywhere: scores of the cached keys times the scale, softmax, weighted sum of the cached values;
// reference src/model/modules/attention.rs:186-226.)
//
//   o[r, h] = sum_j p_j v[j, h'] / sum_j p_j,   p_j = exp(scale q[r, h] . k[j, h'] - max),   j in [len - window, len)
//
// Consecutive rows form groups.  The page tables of a group's rows agree in their first `group_pages[g]` columns, so those
// keys and values are read once for all of them.  A unit of work is a group and kv head: its rows times query heads (R of them, padded to
// N = 16, 32 or 64; more rows take several units) against the shared pages and then each row's own.  On the fifth-generation
// tensor cores keys take the 128 lanes and rows the columns, so that few rows cost little:
//   S^T[128 keys, N]  = K . Q^T      two pages of keys, Q in shared memory, S^T in tensor memory (two buffers)
//   softmax           a key and half of the columns per thread; a column's reference is the score of the first key of the stretch and
//                     moves only when another exceeds it by 2^60, so that a tile needs no barrier and no maxima; P^T
//                     rounded to bfloat16 (by at most 2^-8 of each weight: the products take bfloat16) to shared memory
//   O^T[hd, N]       += V^T . P^T    the transposed value slab as it lies in the cache, O^T in tensor memory
// A row's own page is multiplied with all rows of the unit; the others' weights are zero there, as all weights of keys that are not seen
// are.  Where such a value is no number (0 x NaN is NaN) the second kernel finds a result that is none and computes it again,
// from the keys that the row sees alone.
//
// The tiles of all units lie in one line, which the blocks (one per SM) cut into equal stretches: nobody waits for the longest
// sequence, and loads run on across units.  A stretch of a unit leaves a reference, a sum and a weighted sum per row and head, and a
// second kernel merges them in the order of the keys.
//
// What bounds this is the memory: a tile of head size 128 is 64 KB and takes an SM 1.5 us at the copy rate; the softmax of 16 columns
// takes a third of that, of 64 columns 1.1 us.  Measured (L2 cold): 4 prompts of 6000 to 16000 tokens x 8 beams, 48 over 8 heads of 128, 206 MB:
// 46 us, 1.55 us a tile between a start of 5 us (the line, the lists of pages, the first pages) and an end of 5 (a unit's results 2, the
// merge 3); 8 prompts of 300 to 4000 tokens x 4, 32 over 8 heads, 84 MB: 24 us; one prompt of 2000 x 4: 10 us, all of it start and
// end; heads of 64, 6 prompts x 16 beams: 18 us, its tiles 32 KB with a softmax of 64 columns.  Sixteen warps of softmax for 64 columns
// instead of eight: 2 us more (registers).
//
// Nothing is read before the wait for the kernels before: a page may have been copied by one of them.  Every wait on an mbarrier
// is bounded; when a bound is hit the block records a code in tl_attn_shared_error, waits (bounded) for its copies in flight, frees its tensor
// memory and returns.
#include <cuda.h>
#include <stdlib.h>
#include <type_traits>

#include "attention_bf16_common.cuh"
#include "attention_shared.cuh"

#define SH_SOFT 256                                 // threads of the softmax: warps 0-3 the lower half of the columns, 4-7 the upper
#define SH_THREADS (SH_SOFT + 96)                   // warp 8 TMA of keys, warp 9 of values, warp 10 tcgen05.mma
#define SH_KSUB (HEAD_DIM / 64)                     // 64-column boxes of a K slab
#define SH_PAGE_K (PAGE * HEAD_DIM * 2)
#define SH_PAGE_V (HEAD_DIM * PAGE * 2)
#define SH_STRIDE (HEAD_DIM + 2)                    // floats of a partial result: weighted sum, maximum, sum
#define SH_MAX_HEADS 16                             // query heads per key/value head
// A column's reference moves two tiles after a score has exceeded it by 2^60 (in between weights reach what the two tiles' scores exceed it
// by; where one weight or their sum comes to 2^128 the result is none and is computed again), so that no tile waits for a maximum; rounding to
// bfloat16 is relative.  A sum of weights below 2^-60 is not taken either: what is lost below 2^-126 is then no more than 2^-66 of it.
#define SH_SLACK 60.0f
#define SH_LEAST 8.67361737988403547e-19f            // 2^-60

__device__ int tl_attn_shared_error = 0;

__device__ __forceinline__ bool sh_park(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code) {
  return tl_mbar_park(bar, parity, abort_flag, code, &tl_attn_shared_error);
}
__device__ __forceinline__ void sh_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float sh_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void sh_async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// C columns of this thread's lane: 8 at a time
template <int C>
__device__ __forceinline__ void sh_tmem_ld(uint32_t taddr, float (&v)[C]) {
  static_assert(C % 8 == 0, "");
#pragma unroll
  for (int c = 0; c < C; c += 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[c]), "=f"(v[c + 1]), "=f"(v[c + 2]), "=f"(v[c + 3]), "=f"(v[c + 4]), "=f"(v[c + 5]), "=f"(v[c + 6]), "=f"(v[c + 7])
                 : "r"(taddr + c));
  tmem_ld_wait();
  // (the values are there from here on, whatever order the compiler would like)
#pragma unroll
  for (int c = 0; c < C; ++c) asm volatile("" : "+f"(v[c]));
}
__device__ __forceinline__ void sh_tmem_st8(uint32_t taddr, const float* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void sh_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ constexpr uint32_t sh_idesc(int n) {   // bf16 x bf16 -> f32, M = 128, both K-major
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// A weight at its place of P^T, by an address of shared memory (no clobber: the loop's loads and arithmetic may run past it).
__device__ __forceinline__ void sh_store_bf16(uint32_t addr, float v) {
  const unsigned short b = __bfloat16_as_ushort(__float2bfloat16_rn(v));
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(b));
}

// Bits c0 to c1 - 1.
__device__ __forceinline__ uint32_t sh_mask(int c0, int c1) {
  return (uint32_t)(((1ull << c1) - 1ull) & ~((1ull << c0) - 1ull));
}
// s <- s scale - reference in the columns that see this thread's key, -inf in the others; returns the largest.
template <bool MASKED, int N>
__device__ __forceinline__ float sh_shift(float (&s)[N], uint32_t columns, const float* neg_ref, float scale) {
  float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
  for (int c4 = 0; c4 < N; c4 += 4) {
    const float4 v = *reinterpret_cast<const float4*>(neg_ref + c4);
    const float neg[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = c4 + e;
      s[c] = fmaf(s[c], scale, neg[e]);
      if (MASKED) s[c] = (columns >> c & 1u) ? s[c] : -INFINITY;
      if (c & 1) m1 = fmaxf(m1, s[c]); else m0 = fmaxf(m0, s[c]);
    }
  }
  return fmaxf(m0, m1);
}

// Joins v[0 .. N) over the lanes of a warp into out[0 .. N): each exchange halves the columns that a lane holds.
template <int N, typename F>
__device__ __forceinline__ void sh_columns(const float (&v)[N], int lane, float* out, F join) {
  float x[N / 2];
  {
    const bool up = (lane & 16) != 0;
#pragma unroll
    for (int c = 0; c < N / 2; ++c) {
      const float send = up ? v[c] : v[c + N / 2], keep = up ? v[c + N / 2] : v[c];
      x[c] = join(keep, __shfl_xor_sync(0xffffffffu, send, 16));
    }
  }
  int cnt = N / 2;
#pragma unroll
  for (int mask = 8; mask > 0; mask >>= 1) {
    const bool up = (lane & mask) != 0;
    if (cnt > 1) {
      cnt >>= 1;
#pragma unroll
      for (int c = 0; c < N / 4; ++c)
        if (c < cnt) {
          const float send = up ? x[c] : x[c + cnt], keep = up ? x[c + cnt] : x[c];
          x[c] = join(keep, __shfl_xor_sync(0xffffffffu, send, mask));
        }
    } else {
      x[0] = join(x[0], __shfl_xor_sync(0xffffffffu, x[0], mask));
    }
  }
#pragma unroll
  for (int c = 0; c < (N >= 32 ? N / 32 : 1); ++c) out[lane * N / 32 + c] = x[c];
}

template <int N>
struct ShSizes {
  static constexpr int KS = HEAD_DIM == 64 ? (N == 64 ? 4 : 6) : (N == 64 ? 2 : 3), VS = HEAD_DIM == 64 ? 4 : 2;   // ring slots of two pages
  static constexpr int K = 2 * SH_PAGE_K, V = 2 * SH_PAGE_V, Q = N * HEAD_DIM * 2, P = 2 * N * 128;
  static constexpr int aux = SH_MAX_GROUPS * (int)sizeof(ShGroup) + 7 * N * 4 + 512;
  static constexpr int smem = KS * K + VS * V + 2 * Q + 2 * P + aux;
  static constexpr uint32_t tmem = N == 16 ? 64 : N == 32 ? 128 : 256;                             // S^T twice, O^T
};

template <int N>
__global__ void __launch_bounds__(SH_THREADS, 1)
FN(attn_shared_kernel)(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const ShArgs<__nv_bfloat16> a) {
  using Z = ShSizes<N>;
  // Swizzled tiles need 1024-byte alignment, which dynamic shared memory has when there is no static one (checked below).
  extern __shared__ __align__(1024) uint8_t sh_smem[];
  uint8_t* k_s = sh_smem;
  uint8_t* v_s = k_s + Z::KS * Z::K;
  uint8_t* q_s = v_s + Z::VS * Z::V;                   // [2][Q]
  uint8_t* p_s = q_s + 2 * Z::Q;                       // [2][P]
  ShGroup* table = (ShGroup*)(p_s + 2 * Z::P);
  float* red_s = (float*)(table + SH_MAX_GROUPS);      // [4][N]
  float* ref_s = red_s + 4 * N;                        // [N]
  float* neg_s = ref_s + N;                            // [N]: the negated references
  float* al_s = neg_s + N;                             // [N]: square roots of the factors by which what is summed so far shrinks
  uint64_t* k_full = (uint64_t*)(al_s + N);
  uint64_t* k_empty = k_full + Z::KS;
  uint64_t* v_full = k_empty + Z::KS;
  uint64_t* v_empty = v_full + Z::VS;
  uint64_t* s_full = v_empty + Z::VS;                  // [2]
  uint64_t* p_full = s_full + 2;                       // [2]
  uint64_t* pv_done = p_full + 2;                      // [2]
  uint64_t* q_full = pv_done + 2;                      // [2]
  uint64_t* o_free = q_full + 2;
  uint64_t* half_bar = o_free + 1;                     // [2]
  uint32_t* tmem_slot = (uint32_t*)(half_bar + 2);
  int* total_s = (int*)(tmem_slot + 1);                // [3]
  volatile int* abort_flag = (volatile int*)(total_s + 3);
  // [2][8]: a reference in this half of the columns has to move.  By tile number modulo 8: written in tile n, read in tile n + 2 when
  // its wait has shown that every warp is through with tile n, cleared in tile n + 6 (then every warp has read it, and none is as far
  // as tile n + 8).
  volatile int* moved_s = abort_flag + 1;
  ShPiece* first_s = (ShPiece*)(abort_flag + 1 + 16);   // the stretch's first unit

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(sh_smem) & 1023u) {                     // nothing has been allocated yet
    if (tid == 0) atomicCAS(&tl_attn_shared_error, 0, 9);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < Z::KS; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
    for (int s = 0; s < Z::VS; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
    for (int u = 0; u < 2; ++u) {
      mbar_init(&s_full[u], 1);
      mbar_init(&p_full[u], SH_SOFT);
      mbar_init(&pv_done[u], 1);
      mbar_init(&q_full[u], SH_SOFT);
      mbar_init(&half_bar[u], SH_SOFT / 2);
    }
    for (int u = 0; u < 16; ++u) moved_s[u] = 0;
    mbar_init(o_free, SH_SOFT);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_v) : "memory");
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, Z::tmem);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch_dependents();
  // The next piece with tiles from place t on; without, if there is none.  (The first one is found once for all roles: this is much code,
  // and every copy of it that runs is fetched from afar.)
  int gap = 0, share = 0, t0 = 0, t1 = 0;
  auto piece = [&](int t) {
    ShPiece p = {};
    while (t < t1) {
      p = sh_locate(table, a, gap, t, t1);
      t = p.next;
      if (p.tile < p.last) break;
    }
    return p;
  };
  auto stretch = [&] {
    gap = total_s[2];
    share = sh_share(total_s, gridDim.x, a.parts);
    t0 = min((int)blockIdx.x * share, total_s[0]);
    t1 = min(t0 + share, total_s[0]);
  };
  if (warp == 8) {
    sh_make_line<2>(table, total_s, a, gridDim.x, lane);
    __syncwarp();
    stretch();
    const ShPiece p = piece(t0);
    if (lane == 0) *first_s = p;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + 2 * N;
  stretch();
  const int G = a.nh / a.nkv;

  // ---- TMA: a warp for the keys of every tile of the stretch, one for the values.  The lanes look up 32 pages at a time:
  // with one lookup (two reads, each waiting for the one before) before every tile, and values that wait for their slot in front of the next
  // keys, 4 prompts x 8 beams of the 22B sizes took 4 us more.
  auto produce = [&](auto which) {
    constexpr bool VALUES = decltype(which)::value;
    constexpr int SLOTS = VALUES ? Z::VS : Z::KS, BYTES = VALUES ? SH_PAGE_V : SH_PAGE_K;
    uint64_t *full = VALUES ? v_full : k_full, *empty = VALUES ? v_empty : k_empty;
    bool ok = true;
    int n = 0;
    ShPiece p = *first_s;
    for (int i0 = 2 * p.tile; p.tile < p.last && ok;) {
      const int end = min(min(2 * p.last, p.pages), i0 + 32);
      int slab = 0;
      if (i0 + lane < end) {
        int owner, col;
        sh_page(p, i0 + lane, owner, col);
        slab = a.page_table[(size_t)a.seq_slot[p.row0 + max(owner, 0)] * a.table_stride + col] * a.nkv + p.kvh;
      }
      for (int i = 0; i0 + i < end; i += 2, ++n) {
        const int s = n % SLOTS, slab0 = __shfl_sync(0xffffffffu, slab, i), slab1 = __shfl_sync(0xffffffffu, slab, i + 1);
        ok = __all_sync(0xffffffffu, sh_park(&empty[s], ((uint32_t)(n / SLOTS) & 1u) ^ 1u, abort_flag, VALUES ? 2 : 1));
        if (!ok) break;
        if (lane == 0) {
          const int pages = min(2, end - i0 - i);
          mbar_expect_tx(&full[s], pages * BYTES);
          for (int h = 0; h < pages; ++h) {
            const int at = h ? slab1 : slab0;
            if constexpr (VALUES) {
              tma_load_2d(v_s + s * Z::V + h * SH_PAGE_V, &tm_v, &full[s], 0, at * HEAD_DIM);
            } else {
#pragma unroll
              for (int sub = 0; sub < SH_KSUB; ++sub)
                tma_load_2d(k_s + s * Z::K + sub * (2 * PAGE * 128) + h * (PAGE * 128), &tm_k, &full[s], sub * 64, at * PAGE);
            }
          }
        }
        __syncwarp();
      }
      i0 += 32;
      if (i0 >= 2 * p.last) {
        p = piece(p.next);
        i0 = 2 * p.tile;
      }
    }
    if (!ok && lane == 0) {
      // given up: what is in flight lands before the block ends, or for as long as a wait may take
      for (int i = 0; i < SLOTS && i < n; ++i)
        for (uint32_t k = 0; k < TL_WAIT_LIMIT / 64 && !tl_mbar_try_wait(&full[(n - 1 - i) % SLOTS], (uint32_t)((n - 1 - i) / SLOTS) & 1u); ++k) {}
    }
  };

  if (t0 < t1) {
    if (warp == 8) {
      produce(std::false_type());
    } else if (warp == 9) {
      produce(std::true_type());
    } else if (warp == 10 && elect_one()) {
      // ---- the products: S^T of tile n + 1 before O^T of tile n
      constexpr uint32_t idesc = sh_idesc(N);
      const uint32_t desc_hi = (uint32_t)(smem_desc_k128(0) >> 32);
      auto lo_of = [](const uint8_t* s) { return ((smem_u32(s) & 0x3FFFFu) >> 4) | (1u << 16); };
      auto desc = [&](uint32_t lo) { return ((uint64_t)desc_hi << 32) | lo; };
      const uint32_t k_lo = lo_of(k_s), v_lo = lo_of(v_s), q_lo = lo_of(q_s), p_lo = lo_of(p_s);
      // tile n + 1's unit runs ahead of tile n's
      ShPiece s_piece = *first_s, o_piece = s_piece;
      int s_unit = 0, s_left = s_piece.last - s_piece.tile;            // for S^T: units begun, tiles left of the current one
      int o_unit = 0, o_tile = o_piece.tile;
      bool s_begins = true, o_first = true;
      // 1: issued, 0: there is no further tile, -1: given up
      auto scores = [&](int n) {
        if (s_left == 0) {
          s_piece = piece(s_piece.next);
          s_left = s_piece.last - s_piece.tile;
          if (s_left == 0) return 0;
          s_begins = true;
        }
        if (s_begins) {
          s_begins = false;
          if (!sh_park(&q_full[s_unit & 1], (uint32_t)(s_unit >> 1) & 1u, abort_flag, 3)) return -1;
          ++s_unit;
        }
        --s_left;
        if (!sh_park(&k_full[n % Z::KS], (uint32_t)(n / Z::KS) & 1u, abort_flag, 4)) return -1;
        tc_fence_after();
        const uint32_t ka = k_lo + (uint32_t)(n % Z::KS) * (Z::K >> 4), qa = q_lo + (uint32_t)((s_unit - 1) & 1) * (Z::Q >> 4);
#pragma unroll
        for (int kk = 0; kk < HEAD_DIM / 16; ++kk)
          umma_bf16(tmem + (uint32_t)(n & 1) * N, desc(ka + (kk >> 2) * ((2 * PAGE * 128) >> 4) + (kk & 3) * 2),
                    desc(qa + (kk >> 2) * ((N * 128) >> 4) + (kk & 3) * 2), idesc, kk > 0 ? 1u : 0u);
        umma_commit(&s_full[n & 1]);
        umma_commit(&k_empty[n % Z::KS]);
        return 1;
      };
      for (int n = -1; s_piece.tile < s_piece.last || n >= 0; ++n) {
        const int next = scores(n + 1);           // (its buffer was read before P of tile n - 1 was there)
        if (next < 0) break;
        if (n < 0) continue;
        if (o_first) {
          // O^T is free when the unit before has been written out
          if (o_unit > 0 && !sh_park(o_free, (uint32_t)(o_unit - 1) & 1u, abort_flag, 5)) break;
          ++o_unit;
        }
        if (!sh_park(&v_full[n % Z::VS], (uint32_t)(n / Z::VS) & 1u, abort_flag, 6) ||
            !sh_park(&p_full[n & 1], (uint32_t)(n >> 1) & 1u, abort_flag, 7))
          break;
        tc_fence_after();
        const uint32_t va = v_lo + (uint32_t)(n % Z::VS) * (Z::V >> 4), pa = p_lo + (uint32_t)(n & 1) * (Z::P >> 4);
        const int pages = min(2, o_piece.pages - 2 * o_tile);
        for (int h = 0; h < pages; ++h)        // a second page that is not there is not multiplied
#pragma unroll
          for (int kk = 0; kk < PAGE / 16; ++kk) {
            umma_bf16(tmem_o, desc(va + h * (SH_PAGE_V >> 4) + kk * 2), desc(pa + h * ((N * 128) >> 4) + kk * 2), idesc, o_first ? 0u : 1u);
            o_first = false;
          }
        umma_commit(&pv_done[n & 1]);
        umma_commit(&v_empty[n % Z::VS]);
        if (next == 0) break;
        if (++o_tile == o_piece.last) {
          o_piece = piece(o_piece.next);
          o_tile = o_piece.tile;
          o_first = true;
        }
      }
    } else if (warp < 8) {
      // ---- softmax: key `key` of a tile, columns first_col to first_col + NC - 1.  After a wait that runs out the warps go through the loop
      // to the end (every later wait returns at once), and what they write is not valid.
      constexpr int NC = N / 2;
      const int upper = warp >> 2, key = tid & 127, page_of = key >> 6, first_col = upper * NC, quad = warp & 3;
      const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
      volatile int* moved = moved_s + 8 * upper;
      uint32_t met_before = 0;
      auto meet = [&] {                        // the four warps of this half, by a wait that is bounded too
        sh_arrive(&half_bar[upper]);
        sh_park(&half_bar[upper], met_before, abort_flag, 14);
        met_before ^= 1u;
      };
      const int my_col = first_col + (key & (NC - 1)), my_beam = my_col / G, my_head = my_col - my_beam * G;
      const int first_beam = first_col / G, first_head = first_col - first_beam * G;
      const ShRow q_row(tid / (HEAD_DIM / 8), G);
      auto load_q = [&](const ShPiece& p, int buf) {
        uint8_t* dst = q_s + buf * Z::Q;
        constexpr int C = HEAD_DIM / 8;        // 16-byte pieces of a row
        const int c = tid % C;
        constexpr int STEP = SH_SOFT / C, PASSES = (N + STEP - 1) / STEP;
        ShRow at = q_row;
        uint4 v[PASSES];                       // (all on their way before the first is waited for)
#pragma unroll
        for (int k = 0; k < PASSES; ++k) {
          v[k] = make_uint4(0, 0, 0, 0);
          if (tid / C + k * STEP < p.beams * G)
            v[k] = ldg16(a.q + ((size_t)(p.row0 + at.beam) * a.nh + p.kvh * G + at.head) * HEAD_DIM + c * 8);
          at.step(STEP);
        }
#pragma unroll
        for (int k = 0; k < PASSES; ++k) {
          const int r = tid / C + k * STEP;
          if (r < N) *reinterpret_cast<uint4*>(dst + (c >> 3) * (N * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[k];
        }
        sh_async_fence();
        sh_arrive(&q_full[buf]);
      };
      int n = 0, unit = 0;
      float l[NC];                             // sums of this thread's weights
      const float* neg = neg_s + first_col;    // (the negated references stay in shared memory: 32 columns of them are registers too many)
      ShPiece p = *first_s;
      if (p.tile < p.last) load_q(p, 0);
      for (; p.tile < p.last; ++unit) {
        const int last = p.last, R = p.beams * G;
        ShPiece np = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) l[c] = 0.0f;
        const uint32_t all = sh_mask(0, min(max(R - first_col, 0), NC));
        // the columns of this half that see a page
        auto seen_by = [&](int owner) {
          return owner < 0 ? all : sh_mask(min(max(owner * G - first_col, 0), NC), min(max(owner * G + G - first_col, 0), NC));
        };
        // this thread's page of the tile, step by step
        int owner = -1, in_own = 0, col = p.first + 2 * p.tile + page_of;
        if (2 * p.tile + page_of >= p.common) {
          owner = p.own ? (2 * p.tile + page_of - p.common) / p.own : 0;
          in_own = 2 * p.tile + page_of - p.common - owner * p.own;
          col = p.first + p.common + in_own;
        }
        uint32_t columns = seen_by(owner);
        for (int j = p.tile; j < last; ++j, ++n) {
          const int buf = n & 1;
          const bool there = 2 * j + page_of < p.pages;
          const int at = col * PAGE + (key & 63);
          const bool seen = there && at >= p.lo && at < p.len;
          const bool plain = there && owner < 0 && col * PAGE >= p.lo && col * PAGE + PAGE <= p.len;
          sh_park(&s_full[buf], (uint32_t)(n >> 1) & 1u, abort_flag, 9);
          tc_fence_after();
          float s[NC];                         // scores, then weights
          const uint32_t t_s = tmem + t_lane + (uint32_t)buf * N + first_col;
          sh_tmem_ld<NC>(t_s, s);
          if (j == p.tile) {
            // The references: every column's score of the first key that the tile has to see, whoever sees it.  (A row's own keys may lie far
            // from it: where its weights come to nothing, its result is computed again.)
            if (key == max(p.lo - col * PAGE, 0)) {
#pragma unroll
              for (int c = 0; c < NC; c += 4) {
                float r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = fminf(fmaxf(s[c + e] * a.scale, -1e30f), 1e30f);       // (no number: -1e30)
                *reinterpret_cast<float4*>(ref_s + first_col + c) = make_float4(r[0], r[1], r[2], r[3]);
                *reinterpret_cast<float4*>(neg_s + first_col + c) = make_float4(-r[0], -r[1], -r[2], -r[3]);
              }
            }
            meet();
          }
          const float largest = plain ? sh_shift<false>(s, columns, neg, a.scale) : sh_shift<true>(s, seen ? columns : 0u, neg, a.scale);
          // (These scores were issued after the product with P^T of two tiles ago and are done after it: its buffer is free, and every warp is
          // through with that tile, so they agree on what it noted.)
          if (__any_sync(0xffffffffu, largest > SH_SLACK) && lane == 0) moved[n & 7] = 1;
          if (key == 0) moved[(n + 2) & 7] = 0;
          if (n >= 2 && moved[(n - 2) & 7]) {
            // another reference for the columns that need one: the maximum of this tile's scores
            sh_tmem_ld<NC>(t_s, s);
#pragma unroll
            for (int c = 0; c < NC; ++c) s[c] = seen && (columns >> c & 1u) ? s[c] * a.scale : -INFINITY;
            sh_columns<NC>(s, lane, red_s + quad * N + first_col, [](float x, float y) { return fmaxf(x, y); });
            meet();
            if (key < NC) {
              const float* r = red_s + first_col + key;
              const float m = fmaxf(fmaxf(r[0], r[N]), fmaxf(r[2 * N], r[3 * N])), old = ref_s[first_col + key];
              const float now = m > old + SH_SLACK ? m : old;
              ref_s[first_col + key] = now;
              neg_s[first_col + key] = -now;
              // (the root of the factor, which is taken twice: the sums so far may have come to 2^128 against the old reference and
              // weigh something below it, where the factor itself, from 2^-127 on, would be flushed to zero)
              al_s[first_col + key] = now == old ? 1.0f : sh_ex2(0.5f * (old - now));
            }
            meet();
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const float root = al_s[first_col + c];
              l[c] = l[c] * root * root;
              s[c] += neg[c];
            }
            if (j > p.tile) {
              // O^T so far, once the product before is done (the next one waits for this tile's weights)
              sh_park(&pv_done[buf ^ 1], (uint32_t)((n - 1) >> 1) & 1u, abort_flag, 10);
              tc_fence_after();
              float o[NC];
              sh_tmem_ld<NC>(tmem_o + t_lane + first_col, o);
#pragma unroll
              for (int c = 0; c < NC; ++c) {
                const float root = al_s[first_col + c];
                o[c] = o[c] * root * root;
              }
#pragma unroll
              for (int c = 0; c < NC; c += 8) sh_tmem_st8(tmem_o + t_lane + first_col + c, o + c);
              sh_tmem_st_wait();
            }
          }
          // weights
          const uint32_t pw = smem_u32(p_s + buf * Z::P + page_of * (N * 128) + first_col * 128), k2 = (uint32_t)(key & 63) * 2;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            s[c] = sh_ex2(s[c]);
            l[c] += s[c];
          }
#pragma unroll
          for (int c = 0; c < NC; ++c) sh_store_bf16(pw + c * 128 + (k2 ^ ((c & 7) << 4)), s[c]);
          sh_async_fence();
          tc_fence_before();
          sh_arrive(&p_full[buf]);
          if (j == p.tile) {
            // the next unit's queries: its buffer's scores were all read a unit ago
            np = piece(p.next);
            if (np.tile < np.last) load_q(np, (unit + 1) & 1);
          }
          // two pages on
          const int before = owner;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ++col;
            if (owner < 0) {
              if (col == p.first + p.common) owner = 0;
            } else if (++in_own >= p.own) {
              in_own = 0;
              ++owner;
              col = p.first + p.common;
            }
          }
          if (owner != before) columns = seen_by(owner);
        }
        // ---- the unit's end: sums over the keys, O^T out
        sh_columns<NC>(l, lane, red_s + quad * N + first_col, [](float x, float y) { return x + y; });
        meet();
        const int first_block = p.start / share, pieces = (p.start + p.tiles - 1) / share - first_block + 1;
        const int slot = (int)blockIdx.x - first_block;
        if (tid == 0 && slot == 0) a.unit_parts[p.unit] = pieces;
        // (What runs once per unit is fetched from afar, some ten cycles an instruction: it is written as loops, without divisions.)
        const int heads = a.parts * SH_STRIDE;
        if (key < NC && my_col < R) {
          float* dst = a.part + ((size_t)(p.row0 + my_beam) * a.nh + p.kvh * G + my_head) * heads + slot * SH_STRIDE + HEAD_DIM;
          const float sum = (red_s[my_col] + red_s[N + my_col]) + (red_s[2 * N + my_col] + red_s[3 * N + my_col]);
          // (the columns that have seen a key: all, or those of the rows whose own pages these were)
          const int from = 2 * p.tile - p.common, to = min(2 * last, p.pages) - 1 - p.common;
          const bool any = from < 0 || (my_beam >= from / p.own && my_beam <= to / p.own);
          dst[0] = any ? ref_s[my_col] : -INFINITY;
          dst[1] = any && !(sum >= SH_LEAST && sum < INFINITY) ? NAN : sum;     // (too little of it is left, or it overflowed)
        }
        sh_park(&pv_done[(n - 1) & 1], (uint32_t)((n - 1) >> 1) & 1u, abort_flag, 13);
        tc_fence_after();
        if (key < HEAD_DIM) {                  // (whole warps)
          float* dst = a.part + ((size_t)(p.row0 + first_beam) * a.nh + p.kvh * G + first_head) * heads + slot * SH_STRIDE + key;
          int left = G - first_head;           // heads to the end of the beam
          const int n_col = min(R - first_col, NC);
#pragma unroll 1
          for (int c = 0; c < n_col; c += 8) {
            float o[8];
            sh_tmem_ld<8>(tmem_o + t_lane + first_col + c, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (c + e < n_col) *dst = o[e];
              dst += heads;
              if (--left == 0) { left = G; dst += (size_t)(a.nh - G) * heads; }
            }
          }
        }
        tc_fence_before();
        sh_arrive(o_free);
        meet();                         // red_s and ref_s are written again
        p = np;
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, Z::tmem);
  }
}

template <int N>
static int sh_run(const CUtensorMap& tk, const CUtensorMap& tv, const ShArgs<__nv_bfloat16>& a, int blocks, cudaStream_t stream) {
  constexpr int smem = ShSizes<N>::smem;
  static_assert(smem <= 232448, "a block's shared memory");
  const cudaError_t set = tl_allow_smem<FN(attn_shared_kernel)<N>>(smem);
  if (set != cudaSuccess) return (int)set;
  return tl_launch(FN(attn_shared_kernel)<N>, dim3(blocks), dim3(SH_THREADS), (size_t)smem, stream, tk, tv, a);
}

// q, out [rows][nh][HEAD_DIM]; the rows of group g are group_start[g] to group_start[g + 1] - 1, at most `group_rows` of them, of one
// length.  `row_blocks`: units that a group's rows are split into, at most 64 / (nh / nkv) rows each; `part`: rows * nh * parts *
// (HEAD_DIM + 2) floats, `parts` pieces of a unit at most (2 to 160); `unit_parts`: groups * row_blocks * nkv ints; `blocks`: blocks to launch.
// Returns 0, a CUDA error, or -1 / -2 for arguments that are refused / sizes that are not taken.
extern "C" int FN(tl_attn_shared)(const void* q, const void* k_pages, const void* v_pages, long long n_pages, void* out, float* part,
                                  int* unit_parts, const int* seq_len, const int* seq_slot, const int* page_table, int table_stride,
                                  const int* group_start, const int* group_pages, int groups, int rows, int group_rows, int nh, int nkv,
                                  int window, float scale, int row_blocks, int parts, int blocks, cudaStream_t stream) {
  if (rows <= 0 || groups <= 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || row_blocks < 1 || parts < 2 || blocks < 1 || group_rows < 1 || window < 0) return -1;
  const int G = nh / nkv, beams = (group_rows + row_blocks - 1) / row_blocks, R = beams * G;
  if (G > SH_MAX_HEADS || R > 64 || parts > SH_MAX_PARTS || groups > SH_MAX_GROUPS || nkv > 65535 || group_rows > 65535 ||
      n_pages * nkv * (HEAD_DIM > PAGE ? HEAD_DIM : PAGE) > 0x7fffffffLL || ((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15))
    return -2;
  CUtensorMap tk, tv;
  if (!sh_make_map(&tk, k_pages, n_pages * nkv * PAGE, HEAD_DIM, PAGE, 2)) return -2;
  if (!sh_make_map(&tv, v_pages, n_pages * nkv * HEAD_DIM, PAGE, HEAD_DIM, 2)) return -2;
  const ShArgs<__nv_bfloat16> a = {(const __nv_bfloat16*)q, (__nv_bfloat16*)out, part, unit_parts, seq_len, seq_slot, page_table, group_start, group_pages,
                    table_stride, groups, nh, nkv, window, scale * 1.4426950408889634f, parts, row_blocks, beams};
  const int st = R <= 16 ? sh_run<16>(tk, tv, a, blocks, stream) : R <= 32 ? sh_run<32>(tk, tv, a, blocks, stream) : sh_run<64>(tk, tv, a, blocks, stream);
  if (st) return st;
  return tl_launch(attn_shared_merge_kernel<HEAD_DIM, true, true, __nv_bfloat16>, dim3((nh * (HEAD_DIM / 64) + 3) / 4, group_rows, groups), dim3(SH_MERGE_THREADS), 0, stream, a,
                   (const __nv_bfloat16*)k_pages, (const __nv_bfloat16*)v_pages);
}

extern "C" int FN(tl_attn_shared_take_error)() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, tl_attn_shared_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(tl_attn_shared_error, &zero, sizeof(int));
  return v;
}
