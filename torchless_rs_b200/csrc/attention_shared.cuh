// What the two forms of decode attention over shared pages have in common (attention_shared.cu, attention_shared_f32.cu): the units of
// work, the line of their tiles that the blocks cut into equal stretches, the merge of a unit's pieces, tensor maps.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "per_device.cuh"
#include "umma.cuh"

#ifndef PAGE
#define PAGE TL_PAGE
#endif
static_assert(PAGE == 64, "the tiles are laid out for pages of 64 tokens");

#define SH_MAX_PARTS 160
#define SH_MAX_GROUPS 256
#define SH_PART_TAIL 2                 // floats behind a piece's weighted sum: its reference and sum
#define SH_MERGE_THREADS 128
#define SH_UNIT_TILES 4

template <typename T>
struct ShArgs {
  const T* q;                  // [rows][nh][head size]
  T* out;                      // the same
  float* part;                 // [rows][nh][parts][head size + 2]: weighted sum, maximum, sum
  int* unit_parts;             // [groups][row_blocks][nkv]: pieces of a unit
  const int* seq_len;
  const int* seq_slot;
  const int* page_table;
  const int* group_start;      // [groups + 1]
  const int* group_pages;      // [groups]
  int table_stride, groups, nh, nkv, window;
  float scale;                 // (bfloat16: times log2 e)
  int parts;                   // room for pieces of a unit
  int row_blocks, beams;       // units that share the rows of a group, the group's rows of each
};

// The pages that the rows of a group see: `first` column, how many are common, how many are each row's own.
struct ShSpan {
  int len, lo, first, common, own;
};
__device__ __forceinline__ ShSpan sh_span(int len, int window, int shared) {
  ShSpan s;
  s.len = len;
  s.lo = (window > 0 && len - window > 0) ? len - window : 0;
  s.first = s.lo / PAGE;
  const int end = (len + PAGE - 1) / PAGE, border = min(max(shared, s.first), end);
  s.common = border - s.first;
  s.own = end - border;
  return s;
}
struct ShGroup {
  int before;                  // tiles of the groups before
  int row0, len, lo, first, common, own;
  int full, rest;              // units with all their rows (per kv head), rows of a last one with fewer
  int t_full, t_rest, per_kv;  // tiles of either; places that a kv head takes in the line
};
// What a stretch has of a unit.
struct ShPiece {
  int kvh, row0, beams, len, lo, first, common, own, pages;
  int tile, last, tiles;       // tiles [tile, last) of the unit's `tiles`; none if tile == last
  int unit, start, next;       // the unit's number; the places in the line of its first tile and of what follows this piece
};

// TP: pages of a tile
template <int TP>
__device__ __forceinline__ int sh_tiles(int common, int own, int beams) { return (common + own * beams + TP - 1) / TP; }

// One warp: the groups' places in the line.  Every unit begins with `totals[2]` places without a tile: that is what beginning a unit and
// writing one out takes a block, in tiles, so that equal stretches take equal time (4 prompts x 8 beams of the 22B
// sizes: 57.8 us without them, 55.8 with 2, 53.6 with 4, 52.5 with 6; 8 x 4 of the 7B sizes 27.4, 26.5, 26.9,
// 27.2).  Where a stretch is a few tiles long there are fewer: more, shorter stretches are then faster.  totals[0], [1]: places in the
// line, tiles of the longest unit.
template <int TP, typename T>
__device__ __forceinline__ void sh_make_line(ShGroup* table, int* totals, const ShArgs<T>& a, int blocks, int lane) {
  int tiles = 0, units = 0, longest = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const int g = g0 + lane;
    ShGroup e = {};
    int n = 0, u = 0;
    if (g < a.groups) {
      e.row0 = a.group_start[g];
      const int rows = min(a.group_start[g + 1] - e.row0, a.beams * a.row_blocks);
      if (rows > 0) {
        const ShSpan s = sh_span(a.seq_len[e.row0], a.window, a.group_pages[g]);
        e.len = s.len; e.lo = s.lo; e.first = s.first; e.common = s.common; e.own = s.own;
        if (s.common + s.own > 0) {
          e.full = a.row_blocks == 1 && rows == a.beams ? 1 : rows / a.beams;
          e.rest = rows - e.full * a.beams;
          e.t_full = sh_tiles<TP>(s.common, s.own, a.beams);
          e.t_rest = e.rest ? sh_tiles<TP>(s.common, s.own, e.rest) : 0;
          n = a.nkv * (e.full * e.t_full + e.t_rest);
          u = a.nkv * (e.full + (e.rest ? 1 : 0));
          longest = max(longest, e.full ? e.t_full : e.t_rest);
        }
      }
    }
    int sum = n, sum_u = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o), w = __shfl_up_sync(0xffffffffu, sum_u, o);
      if (lane >= o) { sum += v; sum_u += w; }
    }
    e.before = tiles + sum - n;
    e.per_kv = units + sum_u - u;         // (units before, for now)
    if (g < a.groups) table[g] = e;
    tiles += __shfl_sync(0xffffffffu, sum, 31);
    units += __shfl_sync(0xffffffffu, sum_u, 31);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  const int gap = min(SH_UNIT_TILES, (tiles + blocks - 1) / blocks / 3);
  for (int g = lane; g < a.groups; g += 32) {
    ShGroup& e = table[g];
    e.before += gap * e.per_kv;
    e.per_kv = e.full * (e.t_full + gap) + (e.rest ? e.t_rest + gap : 0);
  }
  if (lane == 0) { totals[0] = tiles + gap * units; totals[1] = longest; totals[2] = gap; }
}
// The length of a stretch: an equal share, but no unit in more pieces than there is room for.
__device__ __forceinline__ int sh_share(const int* totals, int blocks, int parts) {
  return max((totals[0] + blocks - 1) / blocks, (totals[1] + parts - 2) / (parts - 1));
}

// The rows of a unit one after the other, as a row of the group and a query head of the kv head's.
struct ShRow {
  int beam, head, G;
  __device__ __forceinline__ ShRow(int r, int G_) : G(G_) { beam = r / G; head = r - beam * G; }
  __device__ __forceinline__ void step(int k) {
    head += k;
    while (head >= G) { head -= G; ++beam; }
  }
};

// What the stretch that ends at t1 has at place t.
template <typename T>
__device__ ShPiece sh_locate(const ShGroup* table, const ShArgs<T>& a, int gap, int t, int t1) {
  int lo = 0, hi = a.groups - 1;
  while (lo < hi) {            // the last group that begins at or before t and has tiles
    const int mid = (lo + hi + 1) >> 1;
    if (table[mid].before <= t) lo = mid; else hi = mid - 1;
  }
  const ShGroup& g = table[lo];
  const int in_group = t - g.before, kvh = in_group / g.per_kv, r = in_group - kvh * g.per_kv;
  const int rb = a.row_blocks == 1 ? 0 : min(r / (g.t_full + gap), g.full), j = r - rb * (g.t_full + gap);
  const bool whole = rb < g.full;
  ShPiece p;
  p.kvh = kvh;
  p.row0 = g.row0 + rb * a.beams;
  p.beams = whole ? a.beams : g.rest;
  p.len = g.len; p.lo = g.lo; p.first = g.first; p.common = g.common; p.own = g.own;
  p.pages = g.common + g.own * p.beams;
  p.tiles = whole ? g.t_full : g.t_rest;
  p.unit = (lo * a.row_blocks + rb) * a.nkv + kvh;
  p.start = t - j + gap;
  p.tile = max(j - gap, 0);
  p.next = min(p.start + p.tiles, t1);
  p.last = max(p.next - p.start, p.tile);
  return p;
}
// Page i of a unit: the row (of the unit) whose table and weights it takes, -1 for a common one, and the table's column.
__device__ __forceinline__ void sh_page(const ShPiece& p, int i, int& owner, int& col) {
  if (i < p.common) {
    owner = -1;
    col = p.first + i;
  } else {
    owner = (i - p.common) / p.own;
    col = p.first + p.common + (i - p.common) - owner * p.own;
  }
}

// Merges the pieces of (row, head) pairs in the order of the keys, 64 of a head's numbers a warp, two a lane.  A row without any key (of
// length 0) gives zero.  EXP2: the references are logarithms to the base 2.  (Little code and no barriers: this runs when everything
// else is done, so that each step of it is waited for.  A block per pair with a thread per number took 1 us more at 8 prompts x 4 beams of the
// 7B sizes and 2 us more in 32-bit.)
//
// AGAIN: a result that is no number is computed again from the keys that the row sees, one page after the other (the first kernel
// multiplies values that it does not see by zero, and gives a sum that is none where a row's weights left their range).  That is slow, a
// thread per key, and rare.
template <int HD, bool EXP2, bool AGAIN, typename T>
__global__ void __launch_bounds__(SH_MERGE_THREADS)
attn_shared_merge_kernel(const ShArgs<T> a, const T* __restrict__ k_pages, const T* __restrict__ v_pages) {
  constexpr int E = 2, SPLIT = HD / 64, AHEAD = 24, STRIDE = HD + SH_PART_TAIL;
  // what the call was given may be read before the wait: the kernel before this one has waited for those that wrote it
  const int lane = threadIdx.x & 31, w = blockIdx.x * (SH_MERGE_THREADS / 32) + (threadIdx.x >> 5);
  const int h = w / SPLIT, d0 = w % SPLIT * 64 + E * lane, in_group = blockIdx.y, g = blockIdx.z;
  const int row0 = a.group_start[g], row = row0 + in_group;
  const bool there = row < a.group_start[g + 1] && h < a.nh;
  const ShSpan span = sh_span(there ? a.seq_len[row0] : 0, a.window, a.group_pages[g]);
  const int kvh = h / (a.nh / a.nkv);
  pdl_wait();
  pdl_launch_dependents();
  if (!there) return;
  const size_t head = (size_t)row * a.nh + h;
  float acc[E] = {}, l = 0.0f, m = -INFINITY;
  auto store = [&](float by) {
    T* dst = a.out + head * HD + d0;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<__nv_bfloat162*>(dst + e) = __floats2bfloat162_rn(acc[e] / by, acc[e + 1] / by);
      else
        *reinterpret_cast<float2*>(dst + e) = make_float2(acc[e] / by, acc[e + 1] / by);
    }
  };
  if (span.common + span.own == 0) {
    store(1.0f);
    return;
  }
  const float* src = a.part + head * a.parts * STRIDE;
  float v[AHEAD][E];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 x = s0 + k < a.parts ? *reinterpret_cast<const float2*>(src + (s0 + k) * STRIDE + d0 + e) : make_float2(0.0f, 0.0f);
        v[k][e] = x.x; v[k][e + 1] = x.y;
      }
  };
  fetch(0);                        // the first pieces' numbers, before it is known how many there are
  const int parts = a.unit_parts[((size_t)g * a.row_blocks + in_group / a.beams) * a.nkv + kvh];
  for (int s0 = 0; s0 < parts; s0 += 32) {
    // references and sums of 32 pieces (a piece in which this row sees no key has a reference of -inf)
    const float2 rs = s0 + lane < parts ? *reinterpret_cast<const float2*>(src + (s0 + lane) * STRIDE + HD) : make_float2(-INFINITY, 0.0f);
    // What a piece weighs is its sum against its reference.  Where the reference is not the maximum, the sum (2^-60 to 2^128) says
    // as much as the reference, and its power of two counts with it: a piece's factor then is 2^-127 at the least where the piece
    // matters, which 32 bits hold (not flushed) to 2^-22.
    float top = fmaxf(m, EXP2 && rs.x > -INFINITY ? rs.x + (float)((int)(__float_as_uint(rs.y) >> 23 & 255u) - 127) : rs.x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    auto weight = [&](float ref) { return ref == -INFINITY ? 0.0f : EXP2 ? exp2f(ref - top) : expf(ref - top); };
    const float f = weight(rs.x), old = weight(m);
    float sum = f * rs.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * old + sum;
    m = top;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= old;
    const int end = min(s0 + 32, parts);
    for (int s = s0; s < end; s += AHEAD) {
      if (s > 0) fetch(s);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, s - s0 + k);
        if (s + k < end)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += fk * v[k][e];
      }
    }
  }
  store(l);
  if constexpr (AGAIN) {
    bool bad = !isfinite(l);       // (a sum that overflowed would make zeros of a weighted sum that did not)
#pragma unroll
    for (int e = 0; e < E; ++e) bad |= !isfinite(acc[e] / l);
    if (!__any_sync(0xffffffffu, bad)) return;
    const int* table = a.page_table + (size_t)a.seq_slot[row] * a.table_stride;
    const float scale = EXP2 ? a.scale * 0.6931471805599453f : a.scale;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll 1
    for (int col = span.first; col < span.first + span.common + span.own; ++col) {
      const size_t slab = (size_t)table[col] * a.nkv + kvh;
      const int from = max(span.lo - col * PAGE, 0), to = min(span.len - col * PAGE, PAGE);
      float sc[2], top = m;        // the scores of keys `lane` and `lane` + 32
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = lane + 32 * i;
        sc[i] = -INFINITY;
        if (k < from || k >= to) continue;
        const T* key = k_pages + (slab * PAGE + k) * HD;
        float x = 0.0f;
#pragma unroll 1
        for (int d = 0; d < HD; ++d) x = fmaf(to_f32(a.q[head * HD + d]), to_f32(key[d]), x);
        sc[i] = x * scale;
        top = fmaxf(top, sc[i]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float old = m == top ? 1.0f : expf(m - top);
      m = top;
      l *= old;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= old;
      const T* value = v_pages + (slab * HD + d0) * PAGE;
#pragma unroll 1
      for (int k = from; k < to; ++k) {
        const float w = expf(__shfl_sync(0xffffffffu, k < 32 ? sc[0] : sc[1], k & 31) - m);
        l += w;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(w, to_f32(value[e * PAGE + k]), acc[e]);
      }
    }
    store(l);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
typedef CUresult (*ShEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// rows x cols numbers of `size` bytes (2: bfloat16, 4: 32-bit), contiguous rows; boxes of 128 bytes x box_rows, 128-byte swizzle.
static bool sh_make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, int box_rows, int size) {
  static const ShEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (ShEncodeFn)p;
  }();
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols * size};
  cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn && fn(map, size == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(ptr), dims, strides,
                  box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
