// Decode attention of rows that share the leading pages of their cache: the beams of a search, which have one prompt.
// (Per row and head as everywhere: scores of the cached keys times the scale, softmax, weighted sum of the cached values;
// reference src/model/modules/attention.rs:186-226.)
//
//   o[r, h] = sum_j p_j v[j, h'] / sum_j p_j,   p_j = exp(scale q[r, h] . k[j, h'] - max),   j in [len - window, len)
//
// Consecutive rows form groups.  The page tables of a group's rows agree in their first `group_pages[g]` columns, so those
// keys and values are read once for all of them: a block takes some of these pages for the rows x query heads of
// one group and kv head, as the rows of one product.  Other blocks take the pages that are a row's own.  Every block leaves, per row and head, a maximum, a
// sum and a weighted sum; a second kernel merges them in the order of the keys.  What bounds this is the memory: a page
// of head size 128 is 32 KB per kv head and takes an SM 0.75 us at the copy rate, in which its rows' products are done.
//
// Pages come by TMA (128-byte swizzle) into a ring of three stages; each of the four warps takes 16 keys of a page for all
// rows, with mma.m16n8k16 on fragments read from shared memory.  Contraction slots are mapped to whatever dimensions (K) or keys
// (V) a 16-byte or 8-byte read delivers, the same for both operands.  Scores, sums and accumulators are 32-bit; the weights are
// rounded to bfloat16 before the second product (2^-9 of each, as the decode attention's).  Head sizes 64 and 128.
//
// Nothing is read before the wait for the kernels before: a page may have been copied by one of them.  Every wait on an mbarrier
// is bounded; when a bound is hit the block records a code in tl_attn_shared_error and stops.
#include <cuda.h>
#include <stdlib.h>

#include "attention_bf16_common.cuh"
#include "per_device.cuh"
#include "umma.cuh"

#include <map>
#include <mutex>
#include <tuple>

#define SH_WARPS 4
#define SH_STAGES 3
#define SH_KSUB (HEAD_DIM / 64)                     // 64-column boxes of a K slab
#define SH_K_BYTES (PAGE * HEAD_DIM * 2)
#define SH_V_BYTES (HEAD_DIM * PAGE * 2)
#define SH_STAGE_BYTES (SH_K_BYTES + SH_V_BYTES)
#define SH_STRIDE (HEAD_DIM + 2)                    // floats of a partial result: weighted sum, maximum, sum
#define SH_SMEM (1024 + SH_STAGES * SH_STAGE_BYTES + 256)
#define SH_MAX_PARTS 64

__device__ int tl_attn_shared_error = 0;

__device__ __forceinline__ bool sh_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code) {
  return tl_mbar_wait(bar, parity, abort_flag, code, &tl_attn_shared_error);
}
__device__ __forceinline__ void sh_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint4 sh_lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 sh_lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

struct ShArgs {
  const __nv_bfloat16* q;      // [rows][nh][HEAD_DIM]
  float* part;                 // [rows][nh][parts][SH_STRIDE]
  const int* seq_len;
  const int* seq_slot;
  const int* page_table;
  const int* group_start;      // [groups + 1]
  const int* group_pages;      // [groups]
  int table_stride, nh, nkv, window;
  float scale_log2;
  int splits, quantum;         // of the shared pages: blocks, and the pages of each (the last takes what is left)
  int tails;                   // blocks for the pages of a row's own
  int row_blocks, beams;       // blocks that share the rows of a group, the group's rows of each
};

// R8: eights of rows (rows of the group times query heads) that a block holds: 1, 2 or 4.
template <int R8>
__global__ void __launch_bounds__(SH_WARPS * 32, 2)
FN(attn_shared_kernel)(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const ShArgs a) {
  constexpr int MT = (R8 + 1) / 2;
  constexpr bool HI = R8 > 1;
  extern __shared__ uint8_t sh_smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)sh_smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full_bar = (uint64_t*)(smem + SH_STAGES * SH_STAGE_BYTES);
  uint64_t* empty_bar = full_bar + SH_STAGES;
  volatile int* abort_flag = (volatile int*)(empty_bar + SH_STAGES);
  // the merge of the four warps reuses the stages after the loop
  float* sm_o = (float*)smem;                                   // [warps][16 * MT][HEAD_DIM]
  float* sm_m = sm_o + SH_WARPS * 16 * MT * HEAD_DIM;           // [warps][16 * MT]
  float* sm_l = sm_m + SH_WARPS * 16 * MT;

  const int kvh = blockIdx.y, grp = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = a.nh / a.nkv, parts = a.splits + a.tails;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SH_STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], SH_WARPS); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  // ---- which rows and which pages
  const int g0 = a.group_start[grp], group_rows = a.group_start[grp + 1] - g0;
  const int shared_blocks = a.splits * a.row_blocks;
  const bool shared = (int)blockIdx.x < shared_blocks;
  int row0, n_beams, slot;
  if (shared) {
    const int rb = blockIdx.x % a.row_blocks;
    slot = blockIdx.x / a.row_blocks;
    row0 = g0 + rb * a.beams;
    n_beams = min(a.beams, group_rows - rb * a.beams);
  } else {
    const int y = blockIdx.x - shared_blocks;
    row0 = g0 + y / a.tails;
    n_beams = y / a.tails < group_rows ? 1 : 0;
    slot = a.splits + y % a.tails;
  }
  if (n_beams <= 0) return;
  const int R = n_beams * G;                 // rows of this block's products
  const int len = a.seq_len[row0];           // of all rows of the group
  const int lo = (a.window > 0 && len - a.window > 0) ? len - a.window : 0;
  const int* table = a.page_table + (size_t)a.seq_slot[row0] * a.table_stride;
  const int first = lo / PAGE, end = (len + PAGE - 1) / PAGE;      // columns that hold seen keys
  const int border = min(max(a.group_pages[grp], first), end);     // columns before it are shared
  int ps, pe;
  if (shared) {
    ps = first + slot * a.quantum;
    pe = slot == a.splits - 1 ? border : min(ps + a.quantum, border);
  } else {
    const int per = (end - border + a.tails - 1) / a.tails;
    ps = border + (slot - a.splits) * per;
    pe = min(ps + per, end);
  }
  const int n_pg = max(0, pe - ps);
  auto part_of = [&](int r) {      // row r of this block: its partial result
    return a.part + (((size_t)(row0 + r / G) * a.nh + kvh * G + r % G) * parts + slot) * SH_STRIDE;
  };
  if (n_pg == 0) {                 // nothing here: a sum of zero marks it
    for (int r = threadIdx.x; r < R; r += SH_WARPS * 32) {
      float* dst = part_of(r);
      dst[HEAD_DIM] = -INFINITY;
      dst[HEAD_DIM + 1] = 0.0f;
    }
    return;
  }

  // one thread requests pages; `issue(i)` brings page ps + i into stage i % SH_STAGES
  auto issue = [&](int i) {
    const int s = i % SH_STAGES;
    if (!sh_wait(&empty_bar[s], ((uint32_t)(i / SH_STAGES) & 1u) ^ 1u, abort_flag, 1)) return;
    const int slab = table[ps + i] * a.nkv + kvh;
    uint8_t* st = smem + (size_t)s * SH_STAGE_BYTES;
    mbar_expect_tx(&full_bar[s], SH_STAGE_BYTES);
#pragma unroll
    for (int sub = 0; sub < SH_KSUB; ++sub)
      tma_load_2d(st + sub * (PAGE * 128), &tm_k, &full_bar[s], sub * 64, slab * PAGE);
    tma_load_2d(st + SH_K_BYTES, &tm_v, &full_bar[s], 0, slab * HEAD_DIM);
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < SH_STAGES - 1 && i < n_pg; ++i) issue(i);

  // query fragments
  uint32_t qa[MT][NCHUNK][4], qb[MT][NCHUNK][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int ra = mt * 16 + g, rb = ra + 8;
    const __nv_bfloat16* pa = a.q + ((size_t)(row0 + ra / G) * a.nh + kvh * G + ra % G) * HEAD_DIM;
    const __nv_bfloat16* pb = a.q + ((size_t)(row0 + rb / G) * a.nh + kvh * G + rb % G) * HEAD_DIM;
#pragma unroll
    for (int j = 0; j < NCHUNK; ++j) {
      uint4 va = make_uint4(0, 0, 0, 0), vb = make_uint4(0, 0, 0, 0);
      if (ra < R) va = ldg16(pa + (4 * j + t) * 8);
      if (HI && rb < R) vb = ldg16(pb + (4 * j + t) * 8);
      qa[mt][j][0] = va.x; qa[mt][j][1] = va.y; qa[mt][j][2] = va.z; qa[mt][j][3] = va.w;
      qb[mt][j][0] = vb.x; qb[mt][j][1] = vb.y; qb[mt][j][2] = vb.z; qb[mt][j][3] = vb.w;
    }
  }
  float o[MT][NDT][4], m[MT][2], l[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int i = 0; i < NDT; ++i) o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.0f;
    m[mt][0] = m[mt][1] = -INFINITY;
    l[mt][0] = l[mt][1] = 0.0f;
  }

  for (int i = 0; i < n_pg; ++i) {
    if (threadIdx.x == 0 && i + SH_STAGES - 1 < n_pg) issue(i + SH_STAGES - 1);
    __syncwarp();
    const int s = i % SH_STAGES;
    if (!sh_wait(&full_bar[s], (uint32_t)(i / SH_STAGES) & 1u, abort_flag, 2)) break;
    const uint32_t kb = smem_u32(smem + (size_t)s * SH_STAGE_BYTES);
    const uint32_t vb_ = kb + SH_K_BYTES;
    const int key0 = (ps + i) * PAGE + 16 * warp;   // first of this warp's 16 keys
    const bool whole = key0 >= lo && key0 + 16 <= len;
    // ---- scores: 2 tiles of 8 keys; column c of tile jt is key 4*(c>>1) + 2*jt + (c&1)
    float sc[MT][2][4];
#pragma unroll
    for (int jt = 0; jt < 2; ++jt) {
      const int r = 16 * warp + 4 * (g >> 1) + 2 * jt + (g & 1);   // row of the K slab
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) sc[mt][jt][0] = sc[mt][jt][1] = sc[mt][jt][2] = sc[mt][jt][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < NCHUNK; ++j) {
        const int chunk = 4 * j + t;
        const uint4 kv = sh_lds128(kb + (uint32_t)(chunk >> 3) * (PAGE * 128) + (uint32_t)r * 128 +
                                   (uint32_t)(((chunk & 7) ^ (r & 7)) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t f[4];
          f[0] = qa[mt][j][0]; f[1] = qb[mt][j][0]; f[2] = qa[mt][j][1]; f[3] = qb[mt][j][1];
          mma_bf16(sc[mt][jt], f, kv.x, kv.y);
          f[0] = qa[mt][j][2]; f[1] = qb[mt][j][2]; f[2] = qa[mt][j][3]; f[3] = qb[mt][j][3];
          mma_bf16(sc[mt][jt], f, kv.z, kv.w);
        }
      }
    }
    // ---- mask, running maximum, weights; column 2t+e of tile jt is key 4t + 2jt + e
    uint32_t pa[MT][4];
    float al[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int jt = 0; jt < 2; ++jt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int idx = key0 + 4 * t + 2 * jt + e;
          const bool ok = whole || (idx >= lo && idx < len);
          sc[mt][jt][e] = ok ? sc[mt][jt][e] * a.scale_log2 : -INFINITY;
          sc[mt][jt][2 + e] = ok ? sc[mt][jt][2 + e] * a.scale_log2 : -INFINITY;
          mx0 = fmaxf(mx0, sc[mt][jt][e]);
          mx1 = fmaxf(mx1, sc[mt][jt][2 + e]);
        }
      }
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
      if (HI) {
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
      }
      const float n0 = fmaxf(m[mt][0], mx0), n1 = fmaxf(m[mt][1], mx1);
      // the 16 keys of a warp may all lie outside the sequence or the window
      const float ref0 = n0 == -INFINITY ? 0.0f : n0, ref1 = n1 == -INFINITY ? 0.0f : n1;
      al[mt][0] = exp2f(m[mt][0] - ref0);
      al[mt][1] = HI ? exp2f(m[mt][1] - ref1) : 0.0f;
      m[mt][0] = n0;
      m[mt][1] = n1;
      float r0 = 0.0f, r1 = 0.0f;
#pragma unroll
      for (int jt = 0; jt < 2; ++jt) {
        const float p0 = exp2f(sc[mt][jt][0] - ref0), p1 = exp2f(sc[mt][jt][1] - ref0);
        const float p2 = HI ? exp2f(sc[mt][jt][2] - ref1) : 0.0f, p3 = HI ? exp2f(sc[mt][jt][3] - ref1) : 0.0f;
        r0 += p0 + p1;
        r1 += p2 + p3;
        pa[mt][2 * jt] = pack_bf16(p0, p1);
        pa[mt][2 * jt + 1] = pack_bf16(p2, p3);
      }
      l[mt][0] = l[mt][0] * al[mt][0] + r0;
      l[mt][1] = l[mt][1] * al[mt][1] + r1;
    }
    // ---- o = o * alpha + p . v; thread (g, t) reads v^T[dim 8i + g][keys 16*warp + 4t .. +3].  Values of keys that
    // are not seen stay out whatever they are (0 x NaN is NaN).
    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
    if (!whole) {
      const int k = key0 + 4 * t;
      keep0 = (k >= lo && k < len ? 0xffffu : 0u) | (k + 1 >= lo && k + 1 < len ? 0xffff0000u : 0u);
      keep1 = (k + 2 >= lo && k + 2 < len ? 0xffffu : 0u) | (k + 3 >= lo && k + 3 < len ? 0xffff0000u : 0u);
    }
#pragma unroll
    for (int i2 = 0; i2 < NDT; ++i2) {
      const int row = 8 * i2 + g;
      const uint2 vv = sh_lds64(vb_ + (uint32_t)row * 128 + (uint32_t)(((2 * warp + (t >> 1)) ^ (row & 7)) << 4) +
                                (uint32_t)(t & 1) * 8);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        o[mt][i2][0] *= al[mt][0]; o[mt][i2][1] *= al[mt][0]; o[mt][i2][2] *= al[mt][1]; o[mt][i2][3] *= al[mt][1];
        mma_bf16(o[mt][i2], pa[mt], vv.x & keep0, vv.y & keep1);
      }
    }
    __syncwarp();
    if (lane == 0) sh_arrive(&empty_bar[s]);
  }

  __syncthreads();   // every warp is done with the stages; unless a wait ran out, every requested page has arrived
  if (*abort_flag) {
    // no result; the block stays until its copies in flight have landed (a stage's last request is that of the last page
    // with its number), or for as long as a wait may take
    if (threadIdx.x == 0)
      for (int i = max(0, n_pg - SH_STAGES); i < n_pg; ++i)
        for (uint32_t k = 0; k < TL_WAIT_LIMIT / 64 && !tl_mbar_try_wait(&full_bar[i % SH_STAGES], (uint32_t)(i / SH_STAGES) & 1u); ++k) {}
    __syncthreads();
    return;
  }
  // ---- merge the four warps of the block (their keys are disjoint)
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 1);
      l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 2);
    }
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int base = warp * 16 * MT + mt * 16 + g;
    if (t == 0) {
      sm_m[base] = m[mt][0]; sm_l[base] = l[mt][0];
      sm_m[base + 8] = m[mt][1]; sm_l[base + 8] = l[mt][1];
    }
#pragma unroll
    for (int i = 0; i < NDT; ++i) {
      float* ro = sm_o + (size_t)base * HEAD_DIM + 8 * i + 2 * t;
      *reinterpret_cast<float2*>(ro) = make_float2(o[mt][i][0], o[mt][i][1]);
      if (HI) *reinterpret_cast<float2*>(ro + 8 * HEAD_DIM) = make_float2(o[mt][i][2], o[mt][i][3]);
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < R * HEAD_DIM; idx += SH_WARPS * 32) {
    const int r = idx / HEAD_DIM, d = idx - r * HEAD_DIM;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < SH_WARPS; ++w) mm = fmaxf(mm, sm_m[w * 16 * MT + r]);
    float acc = 0.0f, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < SH_WARPS; ++w) {
      const float wm = sm_m[w * 16 * MT + r];
      const float f = wm == -INFINITY ? 0.0f : exp2f(wm - mm);
      acc += f * sm_o[(size_t)(w * 16 * MT + r) * HEAD_DIM + d];
      ll += f * sm_l[w * 16 * MT + r];
    }
    float* dst = part_of(r);
    dst[d] = acc;
    if (d == 0) { dst[HEAD_DIM] = mm; dst[HEAD_DIM + 1] = ll; }
  }
}

// Merges the partial results of one (row, head), a thread per dimension, in the order of the keys.  A row without any key
// (of length 0) gives zero.
__global__ void __launch_bounds__(HEAD_DIM)
FN(attn_shared_merge_kernel)(const float* __restrict__ part, __nv_bfloat16* __restrict__ out, int nh, int parts) {
  __shared__ float f_s[SH_MAX_PARTS], l_s[SH_MAX_PARTS];
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const float* src = part + ((size_t)b * nh + h) * parts * SH_STRIDE;
  constexpr int AHEAD = 16;        // of the first parts this thread's number is fetched before their weights are known
  float v[AHEAD];
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) v[s] = s < parts ? src[s * SH_STRIDE + d] : 0.0f;
  if (d < parts) {
    f_s[d] = src[d * SH_STRIDE + HEAD_DIM];
    l_s[d] = src[d * SH_STRIDE + HEAD_DIM + 1];
  }
  __syncthreads();
  float m = -INFINITY;
  for (int s = 0; s < parts; ++s) m = fmaxf(m, f_s[s]);
  float acc = 0.0f, l = 0.0f;
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) {
    if (s < parts && l_s[s] != 0.0f) {       // (an empty part's weighted sum was never written)
      const float f = exp2f(f_s[s] - m);
      acc += f * v[s];
      l += f * l_s[s];
    }
  }
#pragma unroll 4
  for (int s = AHEAD; s < parts; ++s) {
    if (l_s[s] != 0.0f) {
      const float f = exp2f(f_s[s] - m);
      acc += f * src[s * SH_STRIDE + d];
      l += f * l_s[s];
    }
  }
  out[((size_t)b * nh + h) * HEAD_DIM + d] = __float2bfloat16_rn(l != 0.0f ? acc / l : 0.0f);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
typedef CUresult (*ShEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// rows x cols bfloat16, contiguous rows; boxes of 64 columns (128 bytes) x box_rows, 128-byte swizzle.  What is kept by address is the
// map, which is a function of the address and the sizes alone.
static bool sh_make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, int box_rows) {
  typedef std::tuple<const void*, long long, long long, int> Key;
  static std::map<Key, CUtensorMap> cache;
  static std::mutex mu;
  static ShEncodeFn fn = nullptr;
  std::lock_guard<std::mutex> lock(mu);
  const Key key(ptr, rows, cols, box_rows);
  auto it = cache.find(key);
  if (it != cache.end()) { *map = it->second; return true; }
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return false;
    fn = (ShEncodeFn)p;
  }
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUtensorMap m;
  if (fn(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return false;
  if (cache.size() > 4096) cache.clear();
  cache[key] = m;
  *map = m;
  return true;
}

template <int R8>
static int sh_run(const CUtensorMap& tk, const CUtensorMap& tv, const ShArgs& a, dim3 grid, cudaStream_t stream) {
  const cudaError_t set = tl_allow_smem<FN(attn_shared_kernel)<R8>>(SH_SMEM);
  if (set != cudaSuccess) return (int)set;
  return tl_launch(FN(attn_shared_kernel)<R8>, grid, dim3(SH_WARPS * 32), (size_t)SH_SMEM, stream, tk, tv, a);
}

// q, out [rows][nh][HEAD_DIM]; the rows of group g are group_start[g] to group_start[g + 1] - 1, at most `group_rows` of them, of one
// length; `part`: rows * nh * (splits + tails) * (HEAD_DIM + 2) floats.  `splits`, `quantum`, `tails`: see ShArgs.
// Returns 0, a CUDA error, or -1 / -2 for arguments that are refused / sizes that are not taken.
extern "C" int FN(tl_attn_shared)(const void* q, const void* k_pages, const void* v_pages, long long n_pages, void* out, float* part,
                                  const int* seq_len, const int* seq_slot, const int* page_table, int table_stride,
                                  const int* group_start, const int* group_pages, int groups, int rows, int group_rows, int nh, int nkv,
                                  int window, float scale, int splits, int quantum, int tails, cudaStream_t stream) {
  if (rows <= 0 || groups <= 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || splits < 1 || quantum < 1 || tails < 1 || group_rows < 1 || window < 0) return -1;
  const int G = nh / nkv;
  if (G > 16 || splits + tails > SH_MAX_PARTS || nkv > 65535 || groups > 65535 || rows > 65535 ||
      n_pages * nkv * (HEAD_DIM > PAGE ? HEAD_DIM : PAGE) > 0x7fffffffLL || ((uintptr_t)q & 15) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15))
    return -2;
  CUtensorMap tk, tv;
  if (!sh_make_map(&tk, k_pages, n_pages * nkv * PAGE, HEAD_DIM, PAGE)) return -2;
  if (!sh_make_map(&tv, v_pages, n_pages * nkv * HEAD_DIM, PAGE, HEAD_DIM)) return -2;
  // as few blocks as hold a group's rows, 32 products' rows each, evenly
  const int row_blocks = (group_rows * G + 32 / G * G - 1) / (32 / G * G), beams = (group_rows + row_blocks - 1) / row_blocks;
  ShArgs a = {(const __nv_bfloat16*)q, part, seq_len, seq_slot, page_table, group_start, group_pages, table_stride, nh, nkv, window,
              scale * 1.4426950408889634f, splits, quantum, tails, row_blocks, beams};
  const dim3 grid(splits * row_blocks + group_rows * tails, nkv, groups);
  const int R = beams * G;
  const int st = R <= 8 ? sh_run<1>(tk, tv, a, grid, stream) : R <= 16 ? sh_run<2>(tk, tv, a, grid, stream) : sh_run<4>(tk, tv, a, grid, stream);
  if (st) return st;
  return tl_launch(FN(attn_shared_merge_kernel), dim3(nh, rows), dim3(HEAD_DIM), 0, stream, (const float*)part, (__nv_bfloat16*)out, nh,
                   splits + tails);
}

extern "C" int FN(tl_attn_shared_take_error)() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, tl_attn_shared_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(tl_attn_shared_error, &zero, sizeof(int));
  return v;
}
