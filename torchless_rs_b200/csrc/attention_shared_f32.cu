// The 32-bit form of attention_shared.cu: decode attention of rows that share the leading pages of their cache, with true 32-bit
// products on the CUDA cores (reference: src/model/modules/attention.rs:186-226).
//
// Units, the line of tiles (of one page) and the merge are those of attention_shared.cuh.  A unit holds up to 32 rows (rows of a group times
// query heads).  S = Q K^T in registers, 8 rows x 4 keys per thread over a share of the dimensions (the shares are
// added by shuffles), softmax through shared memory, O += P V in registers, 8 rows x 4 dimensions per thread over a share of the keys.
// A tile of 8 x 4 takes 12 reads of 16 bytes for 128 multiply-adds, which keeps the multiply-adds the bound and not shared memory.
// What bounds the kernel: a page of head size 128 is 64 KB and takes an SM 1.5 us at the copy rate; its products take 16 rows
// 1.1 us at the SM's full rate, 32 rows 2.1 us.  Pages come by TMA, keys in boxes of 32 dimensions and values in boxes of 32 keys,
// whose 128-byte swizzle keeps the reads of neighbouring rows in different banks.  Two blocks share an SM (one's barriers and
// softmax under the other's products); the next page's keys are requested when the scores are done, its values after the products.
// Measured: 4 prompts of 500 to 2000 tokens x 4 beams, 32 over 8 heads of 128, 51 MB: 30 us.  A page takes 13900 instructions of a warp, 8200 of
// them multiply-adds; the busiest SM issues 62 % of what it could (eight warps of 128 registers do not hide the reads of shared memory
// and the four barriers of a page), and it has a third more pages than the mean, since pages are dealt whole.  One block per SM with two
// buffers for pages: 35 us.  Weights against a reference instead of maxima (a barrier less), stretches that differ by a page at most: 29.5 to 30 us.
//
// Nothing is read before the wait for the kernels before: a page may have been copied by one of them.  Every wait on an mbarrier
// is bounded; when a bound is hit the block records a code in tl_attn_shared_f32_error, waits (bounded) for its copies in flight and returns.
#include "attention_shared.cuh"

#define SF_THREADS 256
#define SF_PLD (PAGE + 4)       // floats of a row of weights

__device__ int tl_attn_shared_f32_error = 0;

template <int HD>
struct SfSizes {
  static constexpr int K = PAGE * HD * 4, V = HD * PAGE * 4;
  // a page's keys, a page's values (and the shares of the keys of a unit's output: 64 rows), queries, weights, factors, the groups
  static constexpr int smem(int rg) { return K + V + 8 * rg * (HD + SF_PLD + 1) * 4 + SH_MAX_GROUPS * (int)sizeof(ShGroup) + 128; }
};

// RG: eights of rows that a unit holds: 1, 2 or 4.
template <int HD, int RG>
__global__ void __launch_bounds__(SF_THREADS, 2)
attn_shared_f32_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const ShArgs<float> a) {
  using Z = SfSizes<HD>;
  constexpr int ROWS = 8 * RG;
  constexpr int KS = 16 / RG;              // threads that share the dimensions of a tile of scores
  constexpr int DG = HD / 4, KV = SF_THREADS / (DG * RG);   // groups of dimensions; threads that share the keys of a tile of O
  static_assert(KV * ROWS == 64 * 128 / HD, "");
  extern __shared__ __align__(1024) uint8_t sf_smem[];
  uint8_t* kb = sf_smem;
  uint8_t* vb = kb + Z::K;
  float* o_s = (float*)vb;                                  // [KV][ROWS][HD] (head size 64: in two halves)
  float* q_s = (float*)(vb + Z::V);                         // [ROWS][HD]
  float* p_s = q_s + ROWS * HD;                             // [ROWS][SF_PLD]
  float* al_s = p_s + ROWS * SF_PLD;                        // [ROWS]
  ShGroup* table = (ShGroup*)(al_s + ROWS);
  uint64_t* k_full = (uint64_t*)(table + SH_MAX_GROUPS);
  uint64_t* v_full = k_full + 1;
  int* total_s = (int*)(v_full + 1);                        // [3]
  volatile int* abort_flag = (volatile int*)(total_s + 3);
  const int tid = threadIdx.x;
  if (smem_u32(sf_smem) & 1023u) {         // swizzled tiles need that alignment
    if (tid == 0) atomicCAS(&tl_attn_shared_f32_error, 0, 9);
    return;
  }
  if (tid == 0) {
    mbar_init(k_full, 1);
    mbar_init(v_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  if (tid < 32) sh_make_line<1>(table, total_s, a, gridDim.x, tid);
  __syncthreads();
  const int total = total_s[0], gap = total_s[2], share = sh_share(total_s, gridDim.x, a.parts);
  const int t0 = min((int)blockIdx.x * share, total), t1 = min(t0 + share, total);
  const int G = a.nh / a.nkv;
  if (t0 >= t1) return;

  // One thread requests pages; it looks a page's place up a tile before it is wanted.
  ShPiece ahead;
  ahead.next = t0;
  int ahead_j = 0;
  bool more = false;               // `ahead` has another page
  auto advance = [&] {             // to the next piece with tiles
    do {
      ahead = sh_locate(table, a, gap, ahead.next, t1);
    } while (ahead.tile == ahead.last && ahead.next < t1);
    ahead_j = ahead.tile;
    more = ahead_j < ahead.last;
  };
  auto next_slab = [&]() -> int {
    int owner, col;
    sh_page(ahead, ahead_j, owner, col);
    const int slab = a.page_table[(size_t)a.seq_slot[ahead.row0 + max(owner, 0)] * a.table_stride + col] * a.nkv + ahead.kvh;
    if (++ahead_j == ahead.last) {
      more = false;
      if (ahead.next < t1) advance();
    }
    return slab;
  };
  auto issue_k = [&](int slab) {
    mbar_expect_tx(k_full, Z::K);
#pragma unroll
    for (int sub = 0; sub < HD / 32; ++sub) tma_load_2d(kb + sub * (PAGE * 128), &tm_k, k_full, sub * 32, slab * PAGE);
  };
  auto issue_v = [&](int slab) {
    mbar_expect_tx(v_full, Z::V);
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) tma_load_2d(vb + sub * (HD * 128), &tm_v, v_full, sub * 32, slab * HD);
  };
  int slab = 0;
  bool pending = false;            // `slab` is that of a page that has not been requested
  if (tid == 0) {
    advance();
    if (more) {
      slab = next_slab();
      issue_k(slab);
      issue_v(slab);
    }
  }

  // scores: this thread's share of the dimensions, its keys kg + 16 i, its rows 8 rs + j.  Where four threads share the
  // dimensions, two neighbouring groups of keys lie four rows apart: their 16-byte pieces then fill all banks.
  const int ks = tid % KS, x = (tid / KS) & 15, rs = tid / (KS * 16);
  const int kg = KS == 4 ? ((x & 1) << 2) | ((x >> 1) & 3) | (x & 8) : x;
  // softmax: 32 / RG threads per row, each 2 RG keys
  constexpr int TR = 32 / RG;
  const int sr = tid / TR, sk = tid % TR;
  // output: dimensions dg + DG i, keys of share kv, rows 8 ro + j
  const int dg = tid % DG, kv = (tid / DG) % KV, ro = tid / (DG * KV);
  const ShRow row_of(tid / DG, G), soft_row(sr, G), out_row(tid / HD, G);
  auto load_q = [&](const ShPiece& p) {
    constexpr int STEP = SF_THREADS / DG, PASSES = (ROWS + STEP - 1) / STEP;
    ShRow at = row_of;
    float4 v[PASSES];              // (all on their way before the first is waited for)
#pragma unroll
    for (int k = 0; k < PASSES; ++k) {
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (tid / DG + k * STEP < p.beams * G)
        v[k] = reinterpret_cast<const float4*>(a.q + ((size_t)(p.row0 + at.beam) * a.nh + p.kvh * G + at.head) * HD)[dg];
      at.step(STEP);
    }
#pragma unroll
    for (int k = 0; k < PASSES; ++k)
      if (tid / DG + k * STEP < ROWS) reinterpret_cast<float4*>(q_s)[(tid / DG + k * STEP) * DG + dg] = v[k];
  };
  // A wait that runs out leaves the loop's barriers in place: the warps go through them to the end (every later wait returns at
  // once), and what they write is not valid.
  int n = 0;
  for (int t = t0; t < t1;) {
    const ShPiece p = sh_locate(table, a, gap, t, t1);
    const int last = p.last, R = p.beams * G;
    t = p.next;
    if (p.tile == last) continue;
    load_q(p);
    float m = -INFINITY, l = 0.0f;           // of row sr, the sum of this thread's keys
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
    __syncthreads();                         // the queries are there
    for (int i = p.tile; i < last; ++i, ++n) {
      if (tid == 0) {
        pending = more;
        if (more) slab = next_slab();
      }
      tl_mbar_park(k_full, (uint32_t)n & 1u, abort_flag, 1, &tl_attn_shared_f32_error);
      int owner, col;
      sh_page(p, i, owner, col);
      const int key0 = col * PAGE, r0 = owner > 0 ? owner * G : 0, r1 = owner >= 0 ? r0 + G : R;   // the rows that see the page
      const bool whole = key0 >= p.lo && key0 + PAGE <= p.len;
      if (8 * rs < r1 && 8 * rs + 8 > r0) {
        float sc[32];                        // [8 rows][4 keys]
#pragma unroll
        for (int j = 0; j < 32; ++j) sc[j] = 0.0f;
#pragma unroll
        for (int c = 0; c < DG / KS; ++c) {
          const int chunk = c * KS + ks;
          float4 kk[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = kg + 16 * e;
            kk[e] = *reinterpret_cast<const float4*>(kb + (chunk >> 3) * (PAGE * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
          }
          float4 qq[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) qq[j] = reinterpret_cast<const float4*>(q_s + (8 * rs + j) * HD)[chunk];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float& v = sc[4 * j + e];
              v = fmaf(qq[j].x, kk[e].x, v);
              v = fmaf(qq[j].y, kk[e].y, v);
              v = fmaf(qq[j].z, kk[e].z, v);
              v = fmaf(qq[j].w, kk[e].w, v);
            }
          }
        }
        // the KS shares: every exchange halves how many scores a thread holds; thread ks ends with those from ks * 32 / KS on
        // (rs is one for a warp)
        int half = 16;
#pragma unroll
        for (int mask = KS / 2; mask > 0; mask >>= 1, half >>= 1) {
          const bool up = (ks & mask) != 0;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (j < half) {
              const float send = up ? sc[j] : sc[j + half], keep = up ? sc[j + half] : sc[j];
              sc[j] = keep + __shfl_xor_sync(0xffffffffu, send, mask);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 32 / KS; ++j) {
          const int id = ks * (32 / KS) + j;
          p_s[(8 * rs + (id >> 2)) * SF_PLD + kg + 16 * (id & 3)] = sc[j];
        }
      }
      __syncthreads();
      if (tid == 0 && pending) issue_k(slab);
      {
        const bool in = sr >= r0 && sr < r1;
        float v[2 * RG], mx = m;
#pragma unroll
        for (int j = 0; j < 2 * RG; ++j) {
          const int k = sk + TR * j, at = key0 + k;
          v[j] = in && (whole || (at >= p.lo && at < p.len)) ? p_s[sr * SF_PLD + k] * a.scale : -INFINITY;
          mx = fmaxf(mx, v[j]);
        }
#pragma unroll
        for (int d = TR / 2; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float ref = mx == -INFINITY ? 0.0f : mx, alpha = expf(m - ref);
        l *= alpha;
#pragma unroll
        for (int j = 0; j < 2 * RG; ++j) {
          const float w = expf(v[j] - ref);
          l += w;
          p_s[sr * SF_PLD + sk + TR * j] = w;
        }
        m = mx;
        if (sk == 0) al_s[sr] = alpha;
      }
      tl_mbar_park(v_full, (uint32_t)n & 1u, abort_flag, 2, &tl_attn_shared_f32_error);
      __syncthreads();
      if (8 * ro < r1 && 8 * ro + 8 > r0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = 8 * ro + j;
          const float al = r >= r0 && r < r1 ? al_s[r] : 1.0f;
          acc[j][0] *= al; acc[j][1] *= al; acc[j][2] *= al; acc[j][3] *= al;
        }
#pragma unroll
        for (int c = 0; c < 16 / KV; ++c) {
          const int chunk = kv * (16 / KV) + c;
          float4 vv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = dg + DG * e;
            vv[e] = *reinterpret_cast<const float4*>(vb + (chunk >> 3) * (HD * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
          }
          if (!whole) {            // values of keys that are not seen stay out whatever they are
            const int at = key0 + 4 * chunk;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (at < p.lo || at >= p.len) vv[e].x = 0.0f;
              if (at + 1 < p.lo || at + 1 >= p.len) vv[e].y = 0.0f;
              if (at + 2 < p.lo || at + 2 >= p.len) vv[e].z = 0.0f;
              if (at + 3 < p.lo || at + 3 >= p.len) vv[e].w = 0.0f;
            }
          }
          float4 pp[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) pp[j] = *reinterpret_cast<const float4*>(p_s + (8 * ro + j) * SF_PLD + 4 * chunk);
          auto row = [&](int j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              acc[j][e] = fmaf(pp[j].x, vv[e].x, acc[j][e]);
              acc[j][e] = fmaf(pp[j].y, vv[e].y, acc[j][e]);
              acc[j][e] = fmaf(pp[j].z, vv[e].z, acc[j][e]);
              acc[j][e] = fmaf(pp[j].w, vv[e].w, acc[j][e]);
            }
          };
          if (owner < 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) row(j);
          } else {                 // a row that does not see the page stays as it is, whatever the values are
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (8 * ro + j >= r0 && 8 * ro + j < r1) row(j);
          }
        }
      }
      __syncthreads();           // the page and its weights are used up
      if (tid == 0 && i + 1 < last) issue_v(slab);
    }
    // ---- the unit's end: the shares of the keys
    const int first_block = p.start / share, pieces = (p.start + p.tiles - 1) / share - first_block + 1;
    const int slot = (int)blockIdx.x - first_block;
    if (tid == 0 && slot == 0) a.unit_parts[p.unit] = pieces;
#pragma unroll
    for (int d = TR / 2; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    // (What runs once per unit is fetched from afar, some ten cycles an instruction: it is written as loops, without divisions.)
    const int heads = a.parts * (HD + 2);
    auto part_of = [&](const ShRow& at) {
      return a.part + ((size_t)(p.row0 + at.beam) * a.nh + p.kvh * G + at.head) * heads + slot * (HD + 2);
    };
    if (sk == 0 && sr < R) {
      float* dst = part_of(soft_row) + HD;
      dst[0] = m;
      dst[1] = l;
    }
    constexpr int HALVES = 128 / HD;         // head size 64: twice as many shares as there is room for
#pragma unroll
    for (int h = HALVES - 1; h >= 0; --h) {
      if (kv / (KV / HALVES) == h) {
        float* o = o_s + ((kv % (KV / HALVES)) * ROWS + 8 * ro) * HD + dg;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j * HD + DG * e] = h == HALVES - 1 ? acc[j][e] : o[j * HD + DG * e] + acc[j][e];
      }
      __syncthreads();
    }
    ShRow at = out_row;
#pragma unroll 1
    for (int r = tid / HD; r < R; r += SF_THREADS / HD) {
      float o = 0.0f;
#pragma unroll
      for (int k = 0; k < KV / HALVES; ++k) o += o_s[(k * ROWS + r) * HD + tid % HD];
      part_of(at)[tid % HD] = o;
      at.step(SF_THREADS / HD);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the next values come where the shares lay
    __syncthreads();
    if (tid == 0 && pending) issue_v(slab);
  }
  // (if a wait ran out: what is in flight lands before the block ends, or for as long as a wait may take)
  if (*abort_flag && tid == 0) {
    const uint32_t parity = (uint32_t)(n - 1) & 1u;
    for (uint32_t k = 0; k < TL_WAIT_LIMIT / 64 && !(tl_mbar_try_wait(k_full, parity) && tl_mbar_try_wait(v_full, parity)); ++k) {}
  }
  __syncthreads();
}

template <int HD, int RG>
static int sf_launch(const CUtensorMap& tk, const CUtensorMap& tv, const ShArgs<float>& a, int blocks, cudaStream_t stream) {
  constexpr int smem = SfSizes<HD>::smem(RG);
  static_assert(smem <= 115 * 1024, "a block's shared memory");
  const cudaError_t set = tl_allow_smem<attn_shared_f32_kernel<HD, RG>>(smem);
  if (set != cudaSuccess) return (int)set;
  return tl_launch(attn_shared_f32_kernel<HD, RG>, dim3(blocks), dim3(SF_THREADS), (size_t)smem, stream, tk, tv, a);
}
template <int HD>
static int sf_run(const void* k_pages, const void* v_pages, long long n_pages, const ShArgs<float>& a, int blocks, int group_rows,
                  cudaStream_t stream) {
  CUtensorMap tk, tv;
  if (!sh_make_map(&tk, k_pages, n_pages * a.nkv * PAGE, HD, PAGE, 4)) return -2;
  if (!sh_make_map(&tv, v_pages, n_pages * a.nkv * HD, PAGE, HD, 4)) return -2;
  const int R = a.beams * (a.nh / a.nkv);
  const int st = R <= 8    ? sf_launch<HD, 1>(tk, tv, a, blocks, stream)
                 : R <= 16 ? sf_launch<HD, 2>(tk, tv, a, blocks, stream)
                           : sf_launch<HD, 4>(tk, tv, a, blocks, stream);
  if (st) return st;
  return tl_launch(attn_shared_merge_kernel<HD, false, false, float>, dim3((a.nh * (HD / 64) + 3) / 4, group_rows, a.groups), dim3(SH_MERGE_THREADS), 0, stream, a,
                   (const float*)nullptr, (const float*)nullptr);
}

// As tl_attn_shared_hd<N> (attention_shared.cu), with the head size as an argument (64 or 128) and at most 32 / (nh / nkv) rows of a group
// in a unit.
extern "C" int tl_attn_shared_f32(const void* q, const void* k_pages, const void* v_pages, long long n_pages, void* out, float* part,
                                  int* unit_parts, const int* seq_len, const int* seq_slot, const int* page_table, int table_stride,
                                  const int* group_start, const int* group_pages, int groups, int rows, int group_rows, int nh, int nkv,
                                  int hd, int window, float scale, int row_blocks, int parts, int blocks, cudaStream_t stream) {
  if (rows <= 0 || groups <= 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || row_blocks < 1 || parts < 2 || blocks < 1 || group_rows < 1 || window < 0) return -1;
  const int beams = (group_rows + row_blocks - 1) / row_blocks;
  if (beams * (nh / nkv) > 32 || parts > SH_MAX_PARTS || groups > SH_MAX_GROUPS || nkv > 65535 || group_rows > 65535 ||
      n_pages * nkv * 128 > 0x7fffffffLL || ((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15))
    return -2;
  const ShArgs<float> a = {(const float*)q, (float*)out, part, unit_parts, seq_len, seq_slot, page_table, group_start, group_pages,
                           table_stride, groups, nh, nkv, window, scale, parts, row_blocks, beams};
  if (hd == 64) return sf_run<64>(k_pages, v_pages, n_pages, a, blocks, group_rows, stream);
  if (hd == 128) return sf_run<128>(k_pages, v_pages, n_pages, a, blocks, group_rows, stream);
  return -2;
}

extern "C" int tl_attn_shared_f32_take_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, tl_attn_shared_f32_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(tl_attn_shared_f32_error, &zero, sizeof(int));
  return v;
}
