// The 32-bit form of attention_shared.cu: decode attention of rows that share the leading pages of their cache, with true 32-bit
// products on the CUDA cores (reference: src/model/modules/attention.rs:186-226).
//
// Units, the line of tiles (of one page) and the merge are those of attention_shared.cuh.  A unit holds up to 32 rows (rows of a group times
// query heads).  S = Q K^T in registers, 8 rows x 4 keys per thread over a share of the dimensions (the shares are
// added by shuffles), softmax through shared memory, O += P V in registers, 8 rows x 4 dimensions per thread over a share of the keys.
// A tile of 8 x 4 takes 12 reads of 16 bytes for 128 multiply-adds, which keeps the multiply-adds the bound and not shared memory.
// What bounds the kernel: a page of head size 128 is 64 KB and takes an SM 1.5 us at the copy rate; its products take 16 rows
// 1.1 us at the SM's full rate, 32 rows 2.1 us.  Pages come by TMA, keys in boxes of 32 dimensions and values in boxes of 32 keys,
// whose 128-byte swizzle keeps the reads of neighbouring rows in different banks.
//
// Nothing is read before the wait for the kernels before: a page may have been copied by one of them.  Every wait on an mbarrier
// is bounded; when a bound is hit the block records a code in tl_attn_shared_f32_error, waits (bounded) for its copies in flight and returns.
#include "attention_shared.cuh"

#define SF_THREADS 256          // that compute; a warp more brings the pages
#define SF_PLD (PAGE + 4)       // floats of a row of weights

__device__ int tl_attn_shared_f32_error = 0;

__device__ __forceinline__ void sf_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }   // the computing warps

template <int HD>
struct SfSizes {
  static constexpr int K = PAGE * HD * 4, V = HD * PAGE * 4, STAGE = K + V, STAGES = HD == 64 ? 4 : 2;
  // stages, the shares of the keys of one unit's output (64 rows in all), queries of two units, weights, references and factors
  static constexpr int smem(int rg) {
    return STAGES * STAGE + 64 * HD * 4 + 8 * rg * (2 * HD + SF_PLD + 1) * 4 + SH_MAX_GROUPS * (int)sizeof(ShGroup) + 256;
  }
};

// RG: eights of rows that a unit holds: 1, 2 or 4.
template <int HD, int RG>
__global__ void __launch_bounds__(SF_THREADS + 32, 1)
attn_shared_f32_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const ShArgs<float> a) {
  using Z = SfSizes<HD>;
  constexpr int ROWS = 8 * RG;
  constexpr int KS = 16 / RG;              // threads that share the dimensions of a tile of scores
  constexpr int DG = HD / 4, KV = SF_THREADS / (DG * RG);   // groups of dimensions; threads that share the keys of a tile of O
  static_assert(KV * ROWS == 64 * 128 / HD, "");
  extern __shared__ __align__(1024) uint8_t sf_smem[];
  uint8_t* smem = sf_smem;
  float* o_s = (float*)(smem + Z::STAGES * Z::STAGE);       // [KV][ROWS][HD] (head size 64: in two halves)
  float* q_s = o_s + 64 * HD;                               // [2][ROWS][HD]
  float* p_s = q_s + 2 * ROWS * HD;                         // [ROWS][SF_PLD]
  float* al_s = p_s + ROWS * SF_PLD;                        // [ROWS]
  ShGroup* table = (ShGroup*)(al_s + ROWS);
  uint64_t* full_bar = (uint64_t*)(table + SH_MAX_GROUPS);
  uint64_t* empty_bar = full_bar + Z::STAGES;
  int* total_s = (int*)(empty_bar + Z::STAGES);             // [2]
  volatile int* abort_flag = (volatile int*)(total_s + 2);
  const int tid = threadIdx.x, warp = tid >> 5;
  if (smem_u32(sf_smem) & 1023u) {         // swizzled tiles need that alignment
    if (tid == 0) atomicCAS(&tl_attn_shared_f32_error, 0, 9);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < Z::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], SF_THREADS / 32); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  if (warp == SF_THREADS / 32) sh_make_line<1>(table, total_s, a, tid & 31);
  __syncthreads();
  const int total = total_s[0], share = sh_share(total_s, gridDim.x, a.parts);
  const int t0 = min((int)blockIdx.x * share, total), t1 = min(t0 + share, total);
  const int G = a.nh / a.nkv;
  if (t0 >= t1) return;

  if (warp == SF_THREADS / 32) {
    if (!elect_one()) return;
    bool ok = true;
    int n = 0;
    for (int t = t0; t < t1 && ok;) {
      const ShPiece p = sh_locate<1>(table, a, t);
      const int last = min(p.tiles, p.tile + t1 - t);
      for (int j = p.tile; j < last; ++j, ++t, ++n) {
        int owner, col;
        sh_page(p, j, owner, col);
        const int slab = a.page_table[(size_t)a.seq_slot[p.row0 + max(owner, 0)] * a.table_stride + col] * a.nkv + p.kvh;
        const int s = n % Z::STAGES;
        ok = tl_mbar_park(&empty_bar[s], ((uint32_t)(n / Z::STAGES) & 1u) ^ 1u, abort_flag, 1, &tl_attn_shared_f32_error);
        if (!ok) break;
        uint8_t* st = smem + (size_t)s * Z::STAGE;
        mbar_expect_tx(&full_bar[s], Z::STAGE);
#pragma unroll
        for (int sub = 0; sub < HD / 32; ++sub) tma_load_2d(st + sub * (PAGE * 128), &tm_k, &full_bar[s], sub * 32, slab * PAGE);
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) tma_load_2d(st + Z::K + sub * (HD * 128), &tm_v, &full_bar[s], sub * 32, slab * HD);
      }
    }
    if (!ok)             // given up: what is in flight lands before the block ends, or for as long as a wait may take
      for (int i = max(0, n - Z::STAGES); i < n; ++i)
        for (uint32_t k = 0; k < TL_WAIT_LIMIT / 64 && !tl_mbar_try_wait(&full_bar[i % Z::STAGES], (uint32_t)(i / Z::STAGES) & 1u); ++k) {}
    return;
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
  auto load_q = [&](const ShPiece& p, int buf) {
    for (int i = tid; i < ROWS * DG; i += SF_THREADS) {
      const int r = i / DG, c = i % DG;
      reinterpret_cast<float4*>(q_s + buf * ROWS * HD)[i] =
          r < p.beams * G ? reinterpret_cast<const float4*>(a.q + ((size_t)(p.row0 + r / G) * a.nh + p.kvh * G + r % G) * HD)[c]
                          : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  // A wait that runs out leaves the loop's barriers in place: the warps go through them to the end (every later wait returns at
  // once), and what they write is not valid.
  int n = 0, unit = 0;
  ShPiece p = sh_locate<1>(table, a, t0);
  load_q(p, 0);
  for (int t = t0; t < t1; ++unit) {
    const int last = min(p.tiles, p.tile + t1 - t), R = p.beams * G, next = t + last - p.tile;
    ShPiece np = p;
    if (next < t1) {
      np = sh_locate<1>(table, a, next);
      load_q(np, (unit + 1) & 1);
    }
    const float* qq_s = q_s + (unit & 1) * ROWS * HD;
    float m = -INFINITY, l = 0.0f;           // of row sr, the sum of this thread's keys
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
    sf_bar();                                // the queries are there, the unit before has left shared memory
    for (int i = p.tile; i < last; ++i, ++n) {
      const int s = n % Z::STAGES;
      tl_mbar_wait(&full_bar[s], (uint32_t)(n / Z::STAGES) & 1u, abort_flag, 2, &tl_attn_shared_f32_error);
      const uint8_t* kb = smem + (size_t)s * Z::STAGE;
      const uint8_t* vb = kb + Z::K;
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
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 qq = reinterpret_cast<const float4*>(qq_s + (8 * rs + j) * HD)[chunk];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float& v = sc[4 * j + e];
              v = fmaf(qq.x, kk[e].x, v);
              v = fmaf(qq.y, kk[e].y, v);
              v = fmaf(qq.z, kk[e].z, v);
              v = fmaf(qq.w, kk[e].w, v);
            }
          }
        }
        // the KS shares: every exchange halves how many scores a thread holds; thread ks ends with those from ks * 32 / KS on
        // (the lanes that exchange have one rs)
        int half = 16;
        const unsigned lanes = __activemask();
#pragma unroll
        for (int mask = KS / 2; mask > 0; mask >>= 1, half >>= 1) {
          const bool up = (ks & mask) != 0;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (j < half) {
              const float send = up ? sc[j] : sc[j + half], keep = up ? sc[j + half] : sc[j];
              sc[j] = keep + __shfl_xor_sync(lanes, send, mask);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 32 / KS; ++j) {
          const int id = ks * (32 / KS) + j;
          p_s[(8 * rs + (id >> 2)) * SF_PLD + kg + 16 * (id & 3)] = sc[j];
        }
      }
      sf_bar();
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
      sf_bar();
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
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            // (a row that does not see the page stays as it is, whatever the values are)
            if (owner >= 0 && (8 * ro + j < r0 || 8 * ro + j >= r1)) continue;
            const float4 pp = *reinterpret_cast<const float4*>(p_s + (8 * ro + j) * SF_PLD + 4 * chunk);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              acc[j][e] = fmaf(pp.x, vv[e].x, acc[j][e]);
              acc[j][e] = fmaf(pp.y, vv[e].y, acc[j][e]);
              acc[j][e] = fmaf(pp.z, vv[e].z, acc[j][e]);
              acc[j][e] = fmaf(pp.w, vv[e].w, acc[j][e]);
            }
          }
        }
      }
      sf_bar();                  // the page and its weights are used up
      if ((tid & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty_bar[s])) : "memory");
    }
    // ---- the unit's end: the shares of the keys
    const int first_block = p.start / share, pieces = (p.start + p.tiles - 1) / share - first_block + 1;
    const int slot = (int)blockIdx.x - first_block;
    if (tid == 0 && slot == 0) a.unit_parts[p.unit] = pieces;
#pragma unroll
    for (int d = TR / 2; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    auto head_of = [&](int r) { return (size_t)(p.row0 + r / G) * a.nh + p.kvh * G + r % G; };
    if (sk == 0 && sr < R) {
      float* dst = a.part + (head_of(sr) * a.parts + slot) * (HD + 2) + HD;
      dst[0] = m;
      dst[1] = l;
    }
    constexpr int HALVES = 128 / HD;         // head size 64: twice as many shares as there is room for
#pragma unroll
    for (int h = HALVES - 1; h >= 0; --h) {
      if (kv / (KV / HALVES) == h) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float* o = o_s + ((kv % (KV / HALVES)) * ROWS + 8 * ro + j) * HD + dg + DG * e;
            *o = h == HALVES - 1 ? acc[j][e] : *o + acc[j][e];
          }
      }
      sf_bar();
    }
    for (int i = tid; i < R * HD; i += SF_THREADS) {
      float o = 0.0f;
#pragma unroll
      for (int k = 0; k < KV / HALVES; ++k) o += o_s[k * ROWS * HD + i];
      a.part[(head_of(i / HD) * a.parts + slot) * (HD + 2) + i % HD] = o;
    }
    t = next;
    p = np;
  }
}

template <int HD, int RG>
static int sf_launch(const CUtensorMap& tk, const CUtensorMap& tv, const ShArgs<float>& a, int blocks, cudaStream_t stream) {
  constexpr int smem = SfSizes<HD>::smem(RG);
  static_assert(smem <= 232448, "a block's shared memory");
  const cudaError_t set = tl_allow_smem<attn_shared_f32_kernel<HD, RG>>(smem);
  if (set != cudaSuccess) return (int)set;
  return tl_launch(attn_shared_f32_kernel<HD, RG>, dim3(blocks), dim3(SF_THREADS + 32), (size_t)smem, stream, tk, tv, a);
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
  return tl_launch(attn_shared_merge_kernel<HD, false, false, float>, dim3(a.nh, group_rows, a.groups), dim3(HD), 0, stream, a,
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
      n_pages * nkv * 128 > 0x7fffffffLL || ((uintptr_t)q & 15) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15))
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
