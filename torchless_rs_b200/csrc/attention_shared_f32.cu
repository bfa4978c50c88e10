// The 32-bit form of attention_shared.cu: decode attention of rows that share the leading pages of their cache, with true 32-bit
// products on the CUDA cores (reference: src/model/modules/attention.rs:186-226).
//
// Grid, shared and own pages, partial results and merge as there.  A block holds up to 32 rows (rows of a group times query heads)
// and walks over its pages: S = Q K^T in registers, 8 rows x 4 keys per thread over a share of the dimensions (the shares are
// added by shuffles), softmax through shared memory, O += P V in registers, 8 rows x 4 dimensions per thread over a share of the keys.
// A tile of 8 x 4 takes 12 reads of 16 bytes for 128 multiply-adds, which keeps the multiply-adds the bound and not shared memory.
// What bounds the kernel: a page of head size 128 is 64 KB and takes an SM 1.5 us at the copy rate; its products take 16 rows
// 1.1 us at the SM's full rate, 32 rows 2.1 us.  Pages come by TMA, keys in boxes of 32 dimensions and values in boxes of 32 keys,
// whose 128-byte swizzle keeps the reads of neighbouring rows in different banks.
//
// Nothing is read before the wait for the kernels before: a page may have been copied by one of them.  Every wait on an mbarrier
// is bounded; when a bound is hit the block records a code in tl_attn_shared_f32_error and stops.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"
#include "per_device.cuh"
#include "umma.cuh"

#include <map>
#include <mutex>
#include <tuple>

#define PAGE TL_PAGE
static_assert(PAGE == 64, "the tiles are laid out for pages of 64 tokens");
#define SF_THREADS 256
#define SF_STAGES 3
#define SF_MAX_PARTS 64
#define SF_PLD (PAGE + 4)       // floats of a row of weights

__device__ int tl_attn_shared_f32_error = 0;

struct SfArgs {
  const float* q;              // [rows][nh][HD]
  float* part;                 // [rows][nh][parts][HD + 2]
  const int* seq_len;
  const int* seq_slot;
  const int* page_table;
  const int* group_start;
  const int* group_pages;
  int table_stride, nh, nkv, window;
  float scale;
  int splits, quantum, tails, row_blocks, beams;
};

template <int HD>
struct SfSizes {
  static constexpr int K = PAGE * HD * 4, V = HD * PAGE * 4, STAGE = K + V;
  static constexpr int smem(int rg) { return 1024 + SF_STAGES * STAGE + 8 * rg * (HD + SF_PLD + 1) * 4 + 128; }
};

// RG: eights of rows that a block holds: 1, 2 or 4.
template <int HD, int RG>
__global__ void __launch_bounds__(SF_THREADS)
attn_shared_f32_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const SfArgs a) {
  constexpr int K_BYTES = SfSizes<HD>::K, STAGE = SfSizes<HD>::STAGE, ROWS = 8 * RG, STRIDE = HD + 2;
  constexpr int KS = 16 / RG;              // threads that share the dimensions of a tile of scores
  constexpr int DG = HD / 4, KV = SF_THREADS / (DG * RG);   // groups of dimensions; threads that share the keys of a tile of O
  extern __shared__ uint8_t sf_smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)sf_smem_raw + 1023) & ~(uintptr_t)1023);
  float* q_s = (float*)(smem + SF_STAGES * STAGE);          // [ROWS][HD]
  float* p_s = q_s + ROWS * HD;                             // [ROWS][SF_PLD]
  float* al_s = p_s + ROWS * SF_PLD;                        // [ROWS]
  uint64_t* full_bar = (uint64_t*)(al_s + ROWS);
  volatile int* abort_flag = (volatile int*)(full_bar + SF_STAGES);
  const int kvh = blockIdx.y, grp = blockIdx.z, tid = threadIdx.x;
  const int G = a.nh / a.nkv, parts = a.splits + a.tails;
  if (tid == 0) {
    for (int s = 0; s < SF_STAGES; ++s) mbar_init(&full_bar[s], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  // ---- which rows and which pages (as in attention_shared.cu)
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
  const int R = n_beams * G;
  const int len = a.seq_len[row0];
  const int lo = (a.window > 0 && len - a.window > 0) ? len - a.window : 0;
  const int* table = a.page_table + (size_t)a.seq_slot[row0] * a.table_stride;
  const int first = lo / PAGE, end = (len + PAGE - 1) / PAGE;
  const int border = min(max(a.group_pages[grp], first), end);
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
  auto part_of = [&](int r) {
    return a.part + (((size_t)(row0 + r / G) * a.nh + kvh * G + r % G) * parts + slot) * STRIDE;
  };
  if (n_pg == 0) {
    for (int r = tid; r < R; r += SF_THREADS) {
      float* dst = part_of(r);
      dst[HD] = -INFINITY;
      dst[HD + 1] = 0.0f;
    }
    return;
  }
  auto issue = [&](int i) {      // by one thread, after all have left the stage
    const int s = i % SF_STAGES, slab = table[ps + i] * a.nkv + kvh;
    uint8_t* st = smem + (size_t)s * STAGE;
    mbar_expect_tx(&full_bar[s], STAGE);
#pragma unroll
    for (int sub = 0; sub < HD / 32; ++sub) tma_load_2d(st + sub * (PAGE * 128), &tm_k, &full_bar[s], sub * 32, slab * PAGE);
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) tma_load_2d(st + K_BYTES + sub * (HD * 128), &tm_v, &full_bar[s], sub * 32, slab * HD);
  };
  if (tid == 0)
    for (int i = 0; i < SF_STAGES && i < n_pg; ++i) issue(i);
  for (int i = tid; i < ROWS * DG; i += SF_THREADS) {
    const int r = i / DG, c = i % DG;
    reinterpret_cast<float4*>(q_s)[i] = r < R ? reinterpret_cast<const float4*>(a.q + ((size_t)(row0 + r / G) * a.nh + kvh * G + r % G) * HD)[c]
                                              : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();

  // scores: this thread's share of the dimensions, its keys kg + 16 i, its rows 8 rs + j.  Where four threads share the
  // dimensions, two neighbouring groups of keys lie four rows apart: their 16-byte pieces then fill all banks.
  const int ks = tid % KS, x = (tid / KS) & 15, rs = tid / (KS * 16);
  const int kg = KS == 4 ? ((x & 1) << 2) | ((x >> 1) & 3) | (x & 8) : x;
  // softmax: 32 / RG threads per row, each 2 RG keys
  constexpr int TR = 32 / RG;
  const int sr = tid / TR, sk = tid % TR;
  float m = -INFINITY, l = 0.0f;           // of row sr, the sum of this thread's keys
  // output: dimensions dg + DG i, keys of share kv, rows 8 ro + j
  const int dg = tid % DG, kv = (tid / DG) % KV, ro = tid / (DG * KV);
  float acc[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;

  bool ok = true;
  for (int i = 0; i < n_pg; ++i) {
    const int s = i % SF_STAGES;
    ok = tl_mbar_wait(&full_bar[s], (uint32_t)(i / SF_STAGES) & 1u, abort_flag, 2, &tl_attn_shared_f32_error);
    if (!__syncthreads_and(ok)) break;
    const uint8_t* kb = smem + (size_t)s * STAGE;
    const uint8_t* vb = kb + K_BYTES;
    const int key0 = (ps + i) * PAGE;
    const bool whole = key0 >= lo && key0 + PAGE <= len;
    {
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
          const float4 qq = reinterpret_cast<const float4*>(q_s + (8 * rs + j) * HD)[chunk];
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
    {
      float v[2 * RG], mx = m;
#pragma unroll
      for (int j = 0; j < 2 * RG; ++j) {
        const int k = sk + TR * j, at = key0 + k;
        v[j] = whole || (at >= lo && at < len) ? p_s[sr * SF_PLD + k] * a.scale : -INFINITY;
        mx = fmaxf(mx, v[j]);
      }
#pragma unroll
      for (int d = TR / 2; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float ref = mx == -INFINITY ? 0.0f : mx, alpha = expf(m - ref);
      l *= alpha;
#pragma unroll
      for (int j = 0; j < 2 * RG; ++j) {
        const float p = expf(v[j] - ref);
        l += p;
        p_s[sr * SF_PLD + sk + TR * j] = p;
      }
      m = mx;
      if (sk == 0) al_s[sr] = alpha;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float al = al_s[8 * ro + j];
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
          if (at < lo || at >= len) vv[e].x = 0.0f;
          if (at + 1 < lo || at + 1 >= len) vv[e].y = 0.0f;
          if (at + 2 < lo || at + 2 >= len) vv[e].z = 0.0f;
          if (at + 3 < lo || at + 3 >= len) vv[e].w = 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
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
    __syncthreads();           // the page and its weights are used up
    if (tid == 0 && i + SF_STAGES < n_pg) issue(i + SF_STAGES);
  }
  if (*abort_flag) {
    // no result; the block stays until its copies in flight have landed, or for as long as a wait may take
    if (tid == 0)
      for (int i = max(0, n_pg - SF_STAGES); i < n_pg; ++i)
        for (uint32_t k = 0; k < TL_WAIT_LIMIT / 64 && !tl_mbar_try_wait(&full_bar[i % SF_STAGES], (uint32_t)(i / SF_STAGES) & 1u); ++k) {}
    __syncthreads();
    return;
  }
  // ---- the shares of the keys, through the stages
  float* o_s = (float*)smem;   // [KV][ROWS][HD]
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o_s[(kv * ROWS + 8 * ro + j) * HD + dg + DG * e] = acc[j][e];
#pragma unroll
  for (int d = TR / 2; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  if (sk == 0 && sr < R) {
    float* dst = part_of(sr);
    dst[HD] = m;
    dst[HD + 1] = l;
  }
  __syncthreads();
  for (int i = tid; i < R * HD; i += SF_THREADS) {
    float o = 0.0f;
#pragma unroll
    for (int k = 0; k < KV; ++k) o += o_s[k * ROWS * HD + i];
    part_of(i / HD)[i % HD] = o;
  }

}

// Merges the partial results of one (row, head), a thread per dimension, in the order of the keys.  A row without any key
// (of length 0) gives zero.
template <int HD>
__global__ void __launch_bounds__(HD)
attn_shared_f32_merge_kernel(const float* __restrict__ part, float* __restrict__ out, int nh, int parts) {
  __shared__ float f_s[SF_MAX_PARTS], l_s[SF_MAX_PARTS];
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const float* src = part + ((size_t)b * nh + h) * parts * (HD + 2);
  if (d < parts) {
    f_s[d] = src[d * (HD + 2) + HD];
    l_s[d] = src[d * (HD + 2) + HD + 1];
  }
  __syncthreads();
  float m = -INFINITY;
  for (int s = 0; s < parts; ++s) m = fmaxf(m, f_s[s]);
  float acc = 0.0f, l = 0.0f;
#pragma unroll 8
  for (int s = 0; s < parts; ++s) {
    if (l_s[s] != 0.0f) {      // (an empty part's weighted sum was never written)
      const float f = expf(f_s[s] - m);
      acc = fmaf(f, src[s * (HD + 2) + d], acc);
      l = fmaf(f, l_s[s], l);
    }
  }
  out[((size_t)b * nh + h) * HD + d] = l != 0.0f ? acc / l : 0.0f;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
typedef CUresult (*SfEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// rows x cols 32-bit floats, contiguous rows; boxes of 32 columns (128 bytes) x box_rows, 128-byte swizzle.  What is kept by address
// is the map, which is a function of the address and the sizes alone.
static bool sf_make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, int box_rows) {
  typedef std::tuple<const void*, long long, long long, int> Key;
  static std::map<Key, CUtensorMap> cache;
  static std::mutex mu;
  static SfEncodeFn fn = nullptr;
  std::lock_guard<std::mutex> lock(mu);
  const Key key(ptr, rows, cols, box_rows);
  auto it = cache.find(key);
  if (it != cache.end()) { *map = it->second; return true; }
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return false;
    fn = (SfEncodeFn)p;
  }
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols * 4};
  cuuint32_t box[2] = {32, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUtensorMap m;
  if (fn(&m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return false;
  if (cache.size() > 4096) cache.clear();
  cache[key] = m;
  *map = m;
  return true;
}

template <int HD, int RG>
static int sf_launch(const CUtensorMap& tk, const CUtensorMap& tv, const SfArgs& a, dim3 grid, cudaStream_t stream) {
  constexpr int smem = SfSizes<HD>::smem(RG);
  const cudaError_t set = tl_allow_smem<attn_shared_f32_kernel<HD, RG>>(smem);
  if (set != cudaSuccess) return (int)set;
  return tl_launch(attn_shared_f32_kernel<HD, RG>, grid, dim3(SF_THREADS), (size_t)smem, stream, tk, tv, a);
}
template <int HD>
static int sf_run(const void* k_pages, const void* v_pages, long long n_pages, const SfArgs& a, dim3 grid, int R, int rows, float* out,
                  cudaStream_t stream) {
  CUtensorMap tk, tv;
  if (!sf_make_map(&tk, k_pages, n_pages * a.nkv * PAGE, HD, PAGE)) return -2;
  if (!sf_make_map(&tv, v_pages, n_pages * a.nkv * HD, PAGE, HD)) return -2;
  const int st = R <= 8    ? sf_launch<HD, 1>(tk, tv, a, grid, stream)
                 : R <= 16 ? sf_launch<HD, 2>(tk, tv, a, grid, stream)
                           : sf_launch<HD, 4>(tk, tv, a, grid, stream);
  if (st) return st;
  return tl_launch(attn_shared_f32_merge_kernel<HD>, dim3(a.nh, rows), dim3(HD), 0, stream, (const float*)a.part, out, a.nh,
                   a.splits + a.tails);
}

// As tl_attn_shared_hd<N> (attention_shared.cu), with the head size as an argument: 64 or 128.
extern "C" int tl_attn_shared_f32(const void* q, const void* k_pages, const void* v_pages, long long n_pages, void* out, float* part,
                                  const int* seq_len, const int* seq_slot, const int* page_table, int table_stride,
                                  const int* group_start, const int* group_pages, int groups, int rows, int group_rows, int nh, int nkv,
                                  int hd, int window, float scale, int splits, int quantum, int tails, cudaStream_t stream) {
  if (rows <= 0 || groups <= 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || splits < 1 || quantum < 1 || tails < 1 || group_rows < 1 || window < 0) return -1;
  const int G = nh / nkv;
  if (G > 32 || splits + tails > SF_MAX_PARTS || nkv > 65535 || groups > 65535 || rows > 65535 ||
      n_pages * nkv * 128 > 0x7fffffffLL || ((uintptr_t)q & 15) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15))
    return -2;
  const int row_blocks = (group_rows * G + 32 / G * G - 1) / (32 / G * G), beams = (group_rows + row_blocks - 1) / row_blocks;
  const SfArgs a = {(const float*)q, part, seq_len, seq_slot, page_table, group_start, group_pages, table_stride, nh, nkv, window, scale,
                    splits, quantum, tails, row_blocks, beams};
  const dim3 grid(splits * row_blocks + group_rows * tails, nkv, groups);
  if (hd == 64) return sf_run<64>(k_pages, v_pages, n_pages, a, grid, beams * G, rows, (float*)out, stream);
  if (hd == 128) return sf_run<128>(k_pages, v_pages, n_pages, a, grid, beams * G, rows, (float*)out, stream);
  return -2;
}

extern "C" int tl_attn_shared_f32_take_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, tl_attn_shared_f32_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(tl_attn_shared_f32_error, &zero, sizeof(int));
  return v;
}
