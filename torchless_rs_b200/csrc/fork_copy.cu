// Copies by which a sequence goes on from another one's cache: state of fixed size from slot to slot, and the filled
// part of a page into a page that the sequence may write to.  (The reference has one sequence and never copies its cache,
// src/model/kv_cache.rs:23-53.)
//
// Nothing is computed: the bound is the memory's copy rate, twice the bytes that move.  A block moves up to 16 KB of a slot, or one head's
// keys or values of one layer's page; a thread has four 16-byte loads in flight before its first store (two and two where
// values end inside a sector: with one or three and three of them the copy below takes 60 and 56 us).  The pairs travel as kernel
// arguments, so that nothing has to be brought to the device first.  Sources are never destinations (the caller's rule, checked there), so
// blocks may run in any order.  The next kernel is not let go early: attention kernels read pages that "earlier steps" have filled before they
// wait, and a copied page is one of those.
//
// Measured: 32 layers x 24 pages, 8 heads of 128 in bfloat16: whole pages 62 us (6.5 TB/s read and written); 1 to 63 positions, 32 in the
// mean, 56 us (3.4 TB/s of what is asked for: keys go at 6.1, but a part of a value row of 128 bytes costs whole 64-byte units of
// memory, read and written); half the keys alone 32 us.
#include "common.cuh"

#define FORK_PAIRS 256
#define FORK_THREADS 256
#define FORK_AHEAD 4
#define FORK_BLEND 2

struct ForkPairs {
  int src[FORK_PAIRS];
  int dst[FORK_PAIRS];
  unsigned char count[FORK_PAIRS];   // pages: positions to copy, 1 to TL_PAGE
};

// storage [layers][slots][row_bytes]; V: the widest unit that divides a row
template <typename V>
__global__ void __launch_bounds__(FORK_THREADS)
TL_NAME(copy_slots_kernel)(unsigned char* __restrict__ storage, const __grid_constant__ ForkPairs p, long long layer_bytes,
                           long long row_bytes) {
  pdl_wait();
  unsigned char* layer = storage + (size_t)blockIdx.z * layer_bytes;
  const V* src = reinterpret_cast<const V*>(layer + (size_t)p.src[blockIdx.y] * row_bytes);
  V* dst = reinterpret_cast<V*>(layer + (size_t)p.dst[blockIdx.y] * row_bytes);
  const long long n = row_bytes / (long long)sizeof(V);
  const long long i0 = (long long)blockIdx.x * (FORK_THREADS * FORK_AHEAD) + threadIdx.x;
  V v[FORK_AHEAD];
#pragma unroll
  for (int k = 0; k < FORK_AHEAD; ++k)
    if (i0 + k * FORK_THREADS < n) v[k] = __ldcs(src + i0 + k * FORK_THREADS);
#pragma unroll
  for (int k = 0; k < FORK_AHEAD; ++k)
    if (i0 + k * FORK_THREADS < n) __stcs(dst + i0 + k * FORK_THREADS, v[k]);
}

// One layer's key pages [pages][heads][TL_PAGE][dim] and after them its value pages [pages][heads][vdim][TL_PAGE] (vdim 0: none):
// of a head, the first `count` positions.  Those are the first count * dim numbers of its keys, and the first `count` numbers
// of every row of its values; what lies beyond is not written.  A block copies a head's keys (blockIdx.x < heads) or its values.
template <typename T>
__global__ void __launch_bounds__(FORK_THREADS)
TL_NAME(copy_pages_kernel)(T* __restrict__ storage, const __grid_constant__ ForkPairs p, long long layer_elems, long long v_off,
                           int heads, int dim, int vdim) {
  constexpr int W = 16 / sizeof(T);                 // numbers in 16 bytes
  pdl_wait();
  const int bx = blockIdx.x;
  const bool values = bx >= heads;
  const int head = values ? bx - heads : bx, c = p.count[blockIdx.y], tid = threadIdx.x;
  T* layer = storage + (size_t)blockIdx.z * layer_elems;
  const size_t from = (size_t)p.src[blockIdx.y] * heads + head, to = (size_t)p.dst[blockIdx.y] * heads + head;
  if (!values) {
    const T* src = layer + from * TL_PAGE * dim;
    T* dst = layer + to * TL_PAGE * dim;
    const int n = c * dim / W;
    for (int i0 = tid; i0 < n; i0 += FORK_THREADS * FORK_AHEAD) {
      uint4 v[FORK_AHEAD];
#pragma unroll
      for (int k = 0; k < FORK_AHEAD; ++k)
        if (i0 + k * FORK_THREADS < n) v[k] = __ldcs(reinterpret_cast<const uint4*>(src) + i0 + k * FORK_THREADS);
#pragma unroll
      for (int k = 0; k < FORK_AHEAD; ++k)
        if (i0 + k * FORK_THREADS < n) __stcs(reinterpret_cast<uint4*>(dst) + i0 + k * FORK_THREADS, v[k]);
    }
    for (int i = n * W + tid; i < c * dim; i += FORK_THREADS) dst[i] = src[i];   // a key of no multiple of 16 bytes
    return;
  }
  const T* src = layer + v_off + from * vdim * TL_PAGE;
  T* dst = layer + v_off + to * vdim * TL_PAGE;
  // 16-byte pieces of a row up to the end of the 32-byte sector in which the copied positions end.  That sector is read from the
  // destination too and written whole: memory takes whole sectors, and one written in part is fetched by the cache first, at
  // half the rate (the copy above with 17 positions each: 62 us written in part, 48 so).
  const int per = (c + 2 * W - 1) / (2 * W) * 2, n = vdim * per;
  const float inv = 1.f / per;
  for (int i0 = tid; i0 < n; i0 += FORK_THREADS * FORK_BLEND) {
    uint4 v[FORK_BLEND], w[FORK_BLEND];
    int at[FORK_BLEND], left[FORK_BLEND];
#pragma unroll
    for (int k = 0; k < FORK_BLEND; ++k) {
      // i / per by a product: i + 1/2 is at least 1 / (2 per) >= 1/32 away from the next whole row, and with rows below 2^16 the two
      // roundings move the result by less than 2^16 * 2^-22 = 1/64
      const int i = i0 + k * FORK_THREADS, row = (int)((i + 0.5f) * inv), piece = i - row * per;
      at[k] = row * TL_PAGE + piece * W;
      left[k] = i < n ? c - piece * W : W + 1;      // (W + 1: nothing to read or write)
      if (i < n && left[k] > 0) v[k] = __ldcs(reinterpret_cast<const uint4*>(src + at[k]));
      if (left[k] < W) w[k] = __ldcs(reinterpret_cast<const uint4*>(dst + at[k]));
    }
#pragma unroll
    for (int k = 0; k < FORK_BLEND; ++k) {
      if (i0 + k * FORK_THREADS >= n) break;
      if (left[k] < W) {
        const T* e = reinterpret_cast<const T*>(&v[k]);
        T* f = reinterpret_cast<T*>(&w[k]);
#pragma unroll
        for (int j = 0; j < W; ++j)
          if (j < left[k]) f[j] = e[j];
        v[k] = w[k];
      }
      __stcs(reinterpret_cast<uint4*>(dst + at[k]), v[k]);
    }
  }
}

static void TL_NAME(fork_pairs)(ForkPairs& p, const int* src, const int* dst, const int* count, int n) {
  for (int i = 0; i < n; ++i) {
    p.src[i] = src[i];
    p.dst[i] = dst[i];
    p.count[i] = count ? (unsigned char)count[i] : 0;
  }
}

// storage [layers][slots][row_bytes]: row dst[i] of every layer := row src[i].  The lists lie on the host.
extern "C" int TL_NAME(tl_copy_slots)(void* storage, int layers, int slots, long long row_bytes, const int* src,
                                      const int* dst, int n, cudaStream_t stream) {
  if (n <= 0 || layers <= 0 || row_bytes <= 0) return 0;
  if (layers > 65535) return TL_ERR_UNSUPPORTED;
  const unsigned long long unit = (unsigned long long)(uintptr_t)storage | (unsigned long long)row_bytes;
  const int size = !(unit & 15) ? 16 : !(unit & 3) ? 4 : !(unit & 1) ? 2 : 1;
  const long long per = (long long)size * FORK_THREADS * FORK_AHEAD, blocks = (row_bytes + per - 1) / per;
  if (blocks > 0x7fffffffLL) return TL_ERR_UNSUPPORTED;
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= slots || dst[i] < 0 || dst[i] >= slots) return TL_ERR_BAD_ARG;
  for (int i0 = 0; i0 < n; i0 += FORK_PAIRS) {
    const int m = n - i0 < FORK_PAIRS ? n - i0 : FORK_PAIRS;
    ForkPairs p;
    TL_NAME(fork_pairs)(p, src + i0, dst + i0, nullptr, m);
    const dim3 grid((unsigned)blocks, m, layers);
    const long long layer_bytes = (long long)slots * row_bytes;
    unsigned char* at = (unsigned char*)storage;
    const int st = size == 16 ? tl_launch(TL_NAME(copy_slots_kernel)<uint4>, grid, dim3(FORK_THREADS), 0, stream, at, p, layer_bytes, row_bytes)
                 : size == 4  ? tl_launch(TL_NAME(copy_slots_kernel)<unsigned int>, grid, dim3(FORK_THREADS), 0, stream, at, p, layer_bytes, row_bytes)
                 : size == 2  ? tl_launch(TL_NAME(copy_slots_kernel)<unsigned short>, grid, dim3(FORK_THREADS), 0, stream, at, p, layer_bytes, row_bytes)
                              : tl_launch(TL_NAME(copy_slots_kernel)<unsigned char>, grid, dim3(FORK_THREADS), 0, stream, at, p, layer_bytes, row_bytes);
    if (st) return st;
  }
  return 0;
}

// storage [layers][layer_elems] of numbers of the activation type: in every layer the first count[i] positions of page dst[i] := those of
// page src[i].  The lists lie on the host.
extern "C" int TL_NAME(tl_copy_pages)(void* storage, int layers, long long layer_elems, int pages, int heads, int dim,
                                      int vdim, const int* src, const int* dst, const int* count, int n,
                                      cudaStream_t stream) {
  if (n <= 0 || layers <= 0) return 0;
  if (heads <= 0 || heads > 65536 || dim <= 0 || vdim < 0 || pages <= 0 || ((uintptr_t)storage & 15) ||
      layer_elems < (long long)pages * heads * TL_PAGE * (dim + vdim))
    return TL_ERR_BAD_ARG;
  if (layers > 65535 || dim > 65536 || vdim > 65536 || (layer_elems * (long long)sizeof(act_t)) % 16) return TL_ERR_UNSUPPORTED;
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages || count[i] < 1 || count[i] > TL_PAGE)
      return TL_ERR_BAD_ARG;
  const long long v_off = (long long)pages * heads * TL_PAGE * dim;
  for (int i0 = 0; i0 < n; i0 += FORK_PAIRS) {
    const int m = n - i0 < FORK_PAIRS ? n - i0 : FORK_PAIRS;
    ForkPairs p;
    TL_NAME(fork_pairs)(p, src + i0, dst + i0, count + i0, m);
    const int st = tl_launch(TL_NAME(copy_pages_kernel)<act_t>, dim3(vdim ? 2 * heads : heads, m, layers), dim3(FORK_THREADS), 0, stream,
                             (act_t*)storage, p, layer_elems, v_off, heads, dim, vdim);
    if (st) return st;
  }
  return 0;
}
