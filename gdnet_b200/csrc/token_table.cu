// Token table: lookup with scaling, and its gradient by sorted tokens.
//
//   lookup     out[t, :] = scale * W[tok_t, :]
//   gradient   dW[v, :] (+)= scale * sum over {t : tok_t = v} of dY[t, :]
//
// The gradient sorts the token positions by id (stable, so the rows of one id stay in the order of the batch), then
// walks the sorted list in chunks and sums the rows of each id in fp32 registers. No atomics: the same inputs give
// the same bits. Both directions move every row once and are bound by memory bandwidth; the sort moves 16 bytes a
// token and is bound by the latency of its few dependent steps.
#include "kernels.h"

#include <cuda_fp16.h>

#include "common.cuh"

namespace gd {

// ---------------------------------------------------------------------------------------
// element types
// ---------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V elements moved as one access
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

__device__ __forceinline__ int64_t token_at(const void* tokens, int wide, int64_t i) {
  return wide ? reinterpret_cast<const int64_t*>(tokens)[i] : (int64_t)reinterpret_cast<const int32_t*>(tokens)[i];
}

// ---------------------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------------------
// A row is covered by `tpr` threads (a power of two) in steps of V elements; a block of 256 threads holds 256 / tpr
// row slots and each slot fetches four rows at a time, so that four ids and then four row pieces are in flight per
// thread. An id outside [0, vocab) is never used as an index: its row is zero and the status word records it.
constexpr int LOOKUP_THREADS = 256;
constexpr int LOOKUP_ROWS = 4;

template <typename T, int V, bool SCALED>
__global__ void __launch_bounds__(LOOKUP_THREADS)
token_lookup_kernel(const void* __restrict__ tokens, int wide, int64_t n, const T* __restrict__ table, int64_t ld,
                    int64_t vocab, int vecs, int tpr_log2, float scale, T* __restrict__ out, Status* status) {
  const int tpr = 1 << tpr_log2;
  const int slot = threadIdx.x >> tpr_log2, slots = LOOKUP_THREADS >> tpr_log2;
  const int v0 = threadIdx.x & (tpr - 1);
  const int64_t row0 = (int64_t)blockIdx.x * slots * LOOKUP_ROWS + slot;
  int64_t id[LOOKUP_ROWS];
#pragma unroll
  for (int r = 0; r < LOOKUP_ROWS; ++r) {
    const int64_t row = row0 + (int64_t)r * slots;
    id[r] = row < n ? token_at(tokens, wide, row) : 0;
    if (row < n && (id[r] < 0 || id[r] >= vocab)) {
      if (v0 == 0) report(status, STATUS_BAD_ARGUMENT, 70, (int)row);
      id[r] = -1;
    }
  }
  for (int v = v0; v < vecs; v += tpr) {
    Vec<T, V> x[LOOKUP_ROWS];
#pragma unroll
    for (int r = 0; r < LOOKUP_ROWS; ++r) {
      const int64_t row = row0 + (int64_t)r * slots;
      if (row < n && id[r] >= 0) {
        x[r] = *reinterpret_cast<const Vec<T, V>*>(table + id[r] * ld + (int64_t)v * V);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[r].e[i] = from_f32<T>(0.0f);
      }
    }
#pragma unroll
    for (int r = 0; r < LOOKUP_ROWS; ++r) {
      const int64_t row = row0 + (int64_t)r * slots;
      if (row >= n) continue;
      if (SCALED) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[r].e[i] = from_f32<T>(to_f32(x[r].e[i]) * scale);
      }
      *reinterpret_cast<Vec<T, V>*>(out + (row * vecs + v) * V) = x[r];
    }
  }
}

// Elements per access: the widest of 16, 8, 4 bytes (or one element) that divides the width and the addresses.
static int vec_elems(int elem_bytes, int64_t width, uint64_t address_bits) {
  for (int bytes = 16; bytes > elem_bytes; bytes >>= 1)
    if ((width * elem_bytes) % bytes == 0 && address_bits % bytes == 0) return bytes / elem_bytes;
  return 1;
}

static int tpr_log2_for(int vecs, int most_log2) {
  int l = 0;
  while (l < most_log2 && (1 << l) < vecs) ++l;
  return l;
}

template <typename T, int V>
static const char* lookup_as(const TokenLookupArgs& a, Status* status, cudaStream_t st) {
  const int vecs = (int)(a.width / V);
  const int l = tpr_log2_for(vecs, 8);
  const int64_t rows_per_block = (int64_t)(LOOKUP_THREADS >> l) * LOOKUP_ROWS;
  const int64_t blocks = (a.n + rows_per_block - 1) / rows_per_block;
  if (blocks > 0x7fffffff) return "token_lookup: too many tokens";
  const T* table = reinterpret_cast<const T*>(a.table);
  T* out = reinterpret_cast<T*>(a.out);
  if (a.scale == 1.0f)
    token_lookup_kernel<T, V, false><<<(unsigned)blocks, LOOKUP_THREADS, 0, st>>>(a.tokens, a.wide, a.n, table, a.ld, a.vocab, vecs, l, a.scale, out, status);
  else
    token_lookup_kernel<T, V, true><<<(unsigned)blocks, LOOKUP_THREADS, 0, st>>>(a.tokens, a.wide, a.n, table, a.ld, a.vocab, vecs, l, a.scale, out, status);
  return cudaGetLastError() == cudaSuccess ? nullptr : "token_lookup launch failed";
}

template <typename T>
static const char* lookup_typed(const TokenLookupArgs& a, Status* status, cudaStream_t st) {
  const uint64_t bits = (uint64_t)(uintptr_t)a.table | (uint64_t)(uintptr_t)a.out | (uint64_t)(a.ld * (int64_t)sizeof(T));
  switch (vec_elems(sizeof(T), a.width, bits)) {
    case 8: if constexpr (sizeof(T) == 2) return lookup_as<T, 8>(a, status, st); break;
    case 4: return lookup_as<T, 4>(a, status, st);
    case 2: return lookup_as<T, 2>(a, status, st);
    default: break;
  }
  return lookup_as<T, 1>(a, status, st);
}

const char* launch_token_lookup(const TokenLookupArgs& a, Status* status, cudaStream_t st) {
  if (a.n == 0 || a.width == 0) return nullptr;
  if (a.width > (1 << 30)) return "token_lookup: rows too wide";
  switch (a.dtype) {
    case ELEM_BF16: return lookup_typed<__nv_bfloat16>(a, status, st);
    case ELEM_F16: return lookup_typed<__half>(a, status, st);
    case ELEM_F32: return lookup_typed<float>(a, status, st);
  }
  return "token_lookup: unknown element type";
}

// ---------------------------------------------------------------------------------------
// stable sort of the token positions by id
// ---------------------------------------------------------------------------------------
// Least-significant-digit radix sort by one cluster of eight blocks (256 warps), so that a pass needs no launch of
// its own: every warp owns one contiguous slice of the list, counts its digits in a histogram of its own, and after
// one exchange of the blocks' totals through distributed shared memory knows where each of its digits goes. Digits
// are at most 9 bits (two passes up to a vocabulary of 2^18). A token outside [0, vocab) gets the key `vocab` and
// sorts to the end, where the sums leave it out.
constexpr int SORT_CTAS = 8;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_MAX_BITS = 9;
constexpr int SORT_UNROLL = 4;

__device__ __forceinline__ uint32_t ld_dsmem_u32(uint32_t addr, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(addr, rank)) : "memory");
  return v;
}

__global__ void __cluster_dims__(SORT_CTAS, 1, 1) __launch_bounds__(SORT_THREADS)
token_sort_kernel(const void* __restrict__ tokens, int wide, int n, uint32_t vocab, int bits, int passes,
                  uint32_t* key0, uint32_t* pos0, uint32_t* key1, uint32_t* pos1, Status* status) {
  extern __shared__ uint32_t hist[];                 // [SORT_WARPS][bins]
  __shared__ uint32_t total[1 << SORT_MAX_BITS];     // this block's count of every digit
  __shared__ uint32_t warp_tot[SORT_WARPS];
  const int bins = 1 << bits;
  const uint32_t mask = (uint32_t)bins - 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster_ctarank();
  const int slice = ((n + SORT_CTAS * SORT_WARPS - 1) / (SORT_CTAS * SORT_WARPS) + 31) & ~31;
  const int64_t begin = (int64_t)(rank * SORT_WARPS + warp) * slice;
  const int lo = (int)(begin < n ? begin : n), hi = (int)(begin + slice < n ? begin + slice : n);
  uint32_t* mine = hist + warp * bins;

  for (int p = 0; p < passes; ++p) {
    const uint32_t* src_k = (p & 1) ? key0 : key1;   // pass p writes buffer p & 1; pass 0 reads the tokens
    const uint32_t* src_p = (p & 1) ? pos0 : pos1;
    uint32_t* dst_k = (p & 1) ? key1 : key0;
    uint32_t* dst_p = (p & 1) ? pos1 : pos0;
    const int shift = p * bits;
    auto key_at = [&](int i) -> uint32_t {
      if (p != 0) return __ldcg(src_k + i);
      const int64_t t = token_at(tokens, wide, i);
      return (t < 0 || t >= (int64_t)vocab) ? vocab : (uint32_t)t;
    };
    for (int b = lane; b < bins; b += 32) mine[b] = 0;
    __syncwarp();
    for (int i0 = lo; i0 < hi; i0 += 32 * SORT_UNROLL) {
      uint32_t k[SORT_UNROLL];
#pragma unroll
      for (int u = 0; u < SORT_UNROLL; ++u) {
        const int i = i0 + u * 32 + lane;
        k[u] = i < hi ? key_at(i) : 0;
        if (p == 0 && i < hi && k[u] == vocab) report(status, STATUS_BAD_ARGUMENT, 71, i);
      }
#pragma unroll
      for (int u = 0; u < SORT_UNROLL; ++u)
        if (i0 + u * 32 + lane < hi) atomicAdd(&mine[(k[u] >> shift) & mask], 1u);
    }
    __syncthreads();
    // per digit: counts of the block's warps -> exclusive prefix, and the block's total
    for (int b = threadIdx.x; b < bins; b += SORT_THREADS) {
      uint32_t run = 0;
      for (int w = 0; w < SORT_WARPS; ++w) {
        const uint32_t c = hist[w * bins + b];
        hist[w * bins + b] = run;
        run += c;
      }
      total[b] = run;
    }
    cluster_sync_all();
    // digit b starts at (all smaller digits of all blocks) + (digit b of the blocks before this one)
    uint32_t all = 0, before = 0;
    if ((int)threadIdx.x < bins) {
      for (uint32_t c = 0; c < SORT_CTAS; ++c) {
        const uint32_t t = ld_dsmem_u32(smem_u32(&total[threadIdx.x]), c);
        if (c < rank) before += t;
        all += t;
      }
    }
    uint32_t incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    uint32_t base = incl - all + before;
    for (int w = 0; w < warp; ++w) base += warp_tot[w];
    if ((int)threadIdx.x < bins)
      for (int w = 0; w < SORT_WARPS; ++w) hist[w * bins + threadIdx.x] += base;
    __syncthreads();
    // place: equal digits of a warp's 32 keys keep their order (rank among the lower lanes)
    for (int i0 = lo; i0 < hi; i0 += 32 * SORT_UNROLL) {
      uint32_t k[SORT_UNROLL], at[SORT_UNROLL];
#pragma unroll
      for (int u = 0; u < SORT_UNROLL; ++u) {
        const int i = i0 + u * 32 + lane;
        k[u] = i < hi ? key_at(i) : 0;
        at[u] = p == 0 ? (uint32_t)i : (i < hi ? __ldcg(src_p + i) : 0);
      }
#pragma unroll
      for (int u = 0; u < SORT_UNROLL; ++u) {
        const bool live = i0 + u * 32 + lane < hi;
        const uint32_t d = live ? (k[u] >> shift) & mask : 0xffffffffu;
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        const int before_me = __popc(same & ((1u << lane) - 1));
        if (live) {
          const uint32_t to = mine[d] + before_me;
          dst_k[to] = k[u];
          dst_p[to] = at[u];
        }
        __syncwarp();
        if (live && before_me == 0) mine[d] += __popc(same);
        __syncwarp();
      }
    }
    __threadfence();
    cluster_sync_all();      // the list and the totals are free for the next pass
  }
}

// ---------------------------------------------------------------------------------------
// sums over equal ids
// ---------------------------------------------------------------------------------------
// The sorted list is cut into chunks of `chunk` rows; `tpr` threads cover a row and walk one chunk, eight rows in
// flight. An id whose rows all lie in one chunk is finished there. An id that runs over a chunk's end leaves partial
// sums: slot 0 of a chunk holds the sum of the id that was already running when the chunk began, slot 1 the sum of the
// id that runs on. token_grad_join_kernel adds those up in the order of the chunks.
constexpr int GRAD_THREADS = 128;
constexpr int GRAD_INFLIGHT = 8;
constexpr uint32_t NO_KEY = 0xffffffffu;

template <typename T, int V, bool ADD>
__device__ __forceinline__ void emit_row(void* out, int64_t at, const float (&acc)[V], float scale) {
  if (ADD) {
    Vec<float, V>* o = reinterpret_cast<Vec<float, V>*>(reinterpret_cast<float*>(out) + at);
    if constexpr (V == 8) {      // 32 bytes: two accesses of 16
      Vec<float, 4>* h = reinterpret_cast<Vec<float, 4>*>(o);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        Vec<float, 4> w = h[q];
#pragma unroll
        for (int i = 0; i < 4; ++i) w.e[i] += acc[q * 4 + i] * scale;
        h[q] = w;
      }
    } else {
      Vec<float, V> w = *o;
#pragma unroll
      for (int i = 0; i < V; ++i) w.e[i] += acc[i] * scale;
      *o = w;
    }
  } else {
    Vec<T, V> w;
#pragma unroll
    for (int i = 0; i < V; ++i) w.e[i] = from_f32<T>(acc[i] * scale);
    *reinterpret_cast<Vec<T, V>*>(reinterpret_cast<T*>(out) + at) = w;
  }
}

template <int V>
__device__ __forceinline__ void put_partial(float* dst, const float (&acc)[V]) {
  constexpr int W = V < 4 ? V : 4;          // V floats in accesses of at most 16 bytes (the buffer is aligned)
#pragma unroll
  for (int q = 0; q < V; q += W) {
    Vec<float, W> w;
#pragma unroll
    for (int i = 0; i < W; ++i) w.e[i] = acc[q + i];
    *reinterpret_cast<Vec<float, W>*>(dst + q) = w;
  }
}

template <typename T, int V, bool ADD>
__global__ void __launch_bounds__(GRAD_THREADS)
token_grad_sum_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos, int n, uint32_t vocab,
                      const T* __restrict__ grad, int64_t grad_ld, int vecs, int tpr_log2, int chunk, int n_chunks,
                      float scale, void* __restrict__ out, float* __restrict__ partial) {
  const int tpr = 1 << tpr_log2;
  const int v = blockIdx.y * tpr + (threadIdx.x & (tpr - 1));
  const int c = blockIdx.x * (GRAD_THREADS >> tpr_log2) + (threadIdx.x >> tpr_log2);
  if (c >= n_chunks || v >= vecs) return;
  const int64_t width = (int64_t)vecs * V, col = (int64_t)v * V;
  const int lo = c * chunk, hi = min(n, lo + chunk);
  const uint32_t key_before = lo > 0 ? key[lo - 1] : NO_KEY;
  const uint32_t key_after = hi < n ? key[hi] : NO_KEY;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
  uint32_t cur = key[lo];
  bool open_left = cur == key_before;       // the running id began in an earlier chunk
  for (int j0 = lo; j0 < hi && cur < vocab; j0 += GRAD_INFLIGHT) {
    uint32_t k[GRAD_INFLIGHT];
    Vec<T, V> x[GRAD_INFLIGHT];
#pragma unroll
    for (int u = 0; u < GRAD_INFLIGHT; ++u) {
      k[u] = j0 + u < hi ? key[j0 + u] : NO_KEY;
      if (k[u] < vocab) x[u] = *reinterpret_cast<const Vec<T, V>*>(grad + (int64_t)pos[j0 + u] * grad_ld + col);
    }
#pragma unroll
    for (int u = 0; u < GRAD_INFLIGHT; ++u) {
      if (k[u] != cur && cur < vocab && k[u] != NO_KEY) {       // the running id ends inside this chunk
        if (open_left) put_partial<V>(partial + ((int64_t)c * 2) * width + col, acc);
        else emit_row<T, V, ADD>(out, (int64_t)cur * width + col, acc, scale);
        open_left = false;
        cur = k[u];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
      }
      if (k[u] < vocab) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += to_f32(x[u].e[i]);
      }
    }
  }
  if (cur >= vocab) return;
  if (open_left) put_partial<V>(partial + ((int64_t)c * 2) * width + col, acc);
  else if (cur == key_after) put_partial<V>(partial + ((int64_t)c * 2 + 1) * width + col, acc);
  else emit_row<T, V, ADD>(out, (int64_t)cur * width + col, acc, scale);
}

// For every chunk whose last id runs on into the next chunk and began in this one: its partial sums, in order. The
// number of partial sums of an id is known from the ends of its run, found by bisection in the sorted list.
template <typename T, int V, bool ADD>
__global__ void __launch_bounds__(GRAD_THREADS)
token_grad_join_kernel(const uint32_t* __restrict__ key, int n, uint32_t vocab, int vecs, int tpr_log2, int chunk,
                       int n_chunks, float scale, void* __restrict__ out, const float* __restrict__ partial) {
  const int tpr = 1 << tpr_log2;
  const int v = blockIdx.y * tpr + (threadIdx.x & (tpr - 1));
  const int c = blockIdx.x * (GRAD_THREADS >> tpr_log2) + (threadIdx.x >> tpr_log2);
  if (c >= n_chunks - 1 || v >= vecs) return;
  const int lo = c * chunk, hi = lo + chunk;                    // a full chunk: it is not the last one
  const uint32_t id = key[hi - 1];
  if (id >= vocab || key[hi] != id) return;                     // nothing runs on
  if (lo > 0 && key[lo] == id && key[lo - 1] == id) return;     // the id began before this chunk
  int a = hi, b = n;                                            // first position >= hi with another id
  while (a < b) {
    const int m = a + ((b - a) >> 1);
    if (key[m] == id) a = m + 1;
    else b = m;
  }
  const int last = (a - 1) / chunk;                             // chunk of the id's last row
  const int64_t width = (int64_t)vecs * V, col = (int64_t)v * V;
  float acc[V];
  const float* p = partial + ((int64_t)c * 2 + 1) * width + col;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = p[i];
  for (int j0 = c + 1; j0 <= last; j0 += 4) {
    float x[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* q = partial + ((int64_t)(j0 + u) * 2) * width + col;
#pragma unroll
      for (int i = 0; i < V; ++i) x[u][i] = j0 + u <= last ? q[i] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += x[u][i];
  }
  emit_row<T, V, ADD>(out, (int64_t)id * width + col, acc, scale);
}

static int grad_chunk(int64_t n) {
  // rows per chunk: about a thousand chunks, between 16 (short lists still fill the GPU) and 128 rows
  int c = 16;
  while (c < 128 && n / c > 1536) c *= 2;
  return c;
}

int64_t token_grad_partial_floats(int64_t n, int64_t width) {
  const int c = grad_chunk(n);
  return ((n + c - 1) / c) * 2 * width;
}

template <typename T, int V, bool ADD>
static const char* grad_as(const TokenGradArgs& a, const uint32_t* key, const uint32_t* pos, cudaStream_t st) {
  const int vecs = (int)(a.width / V);
  const int l = tpr_log2_for(vecs, 7);
  const int chunk = grad_chunk(a.n);
  const int n_chunks = (int)((a.n + chunk - 1) / chunk);
  const int per_block = GRAD_THREADS >> l;
  const dim3 grid((unsigned)((n_chunks + per_block - 1) / per_block), (unsigned)((vecs + (1 << l) - 1) >> l));
  if (grid.y > 65535) return "token_grad: rows too wide";
  token_grad_sum_kernel<T, V, ADD><<<grid, GRAD_THREADS, 0, st>>>(key, pos, (int)a.n, (uint32_t)a.vocab,
      reinterpret_cast<const T*>(a.grad), a.grad_ld, vecs, l, chunk, n_chunks, a.scale, a.out, a.partial);
  if (n_chunks > 1)
    token_grad_join_kernel<T, V, ADD><<<grid, GRAD_THREADS, 0, st>>>(key, (int)a.n, (uint32_t)a.vocab, vecs, l, chunk, n_chunks,
                                                                    a.scale, a.out, a.partial);
  return cudaGetLastError() == cudaSuccess ? nullptr : "token_grad launch failed";
}

template <typename T, bool ADD>
static const char* grad_typed(const TokenGradArgs& a, const uint32_t* key, const uint32_t* pos, cudaStream_t st) {
  // adding, the destination's elements have four bytes: twice a 16-bit row's, in accesses of at most 16
  const uint64_t out_bits = (uint64_t)(uintptr_t)a.out & 15;
  const uint64_t bits = (uint64_t)(uintptr_t)a.grad | (uint64_t)(a.grad_ld * (int64_t)sizeof(T)) |
                        (ADD && sizeof(T) == 2 ? out_bits >> 1 : out_bits);
  switch (vec_elems(sizeof(T), a.width, bits)) {
    case 8: if constexpr (sizeof(T) == 2) return grad_as<T, 8, ADD>(a, key, pos, st); break;
    case 4: return grad_as<T, 4, ADD>(a, key, pos, st);
    case 2: return grad_as<T, 2, ADD>(a, key, pos, st);
    default: break;
  }
  return grad_as<T, 1, ADD>(a, key, pos, st);
}

const char* launch_token_grad(const TokenGradArgs& a, Status* status, cudaStream_t st) {
  if (a.n == 0 || a.width == 0) return nullptr;
  if (a.n >= (1ll << 30) || a.vocab >= (1ll << 31) || a.width > (1 << 30)) return "token_grad: sizes out of range";
  int need = 0;
  while (need < 31 && (a.vocab >> need) != 0) ++need;           // keys are 0..vocab
  const int passes = need == 0 ? 1 : (need + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
  const int bits = need == 0 ? 1 : (need + passes - 1) / passes;
  const size_t smem = (size_t)SORT_WARPS * (1u << bits) * sizeof(uint32_t);
  if (cudaFuncSetAttribute(token_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           SORT_WARPS * (1 << SORT_MAX_BITS) * (int)sizeof(uint32_t)) != cudaSuccess)
    return "token_sort: shared memory";
  uint32_t* key0 = a.sort;
  uint32_t* pos0 = key0 + a.n;
  uint32_t* key1 = pos0 + a.n;
  uint32_t* pos1 = key1 + a.n;
  token_sort_kernel<<<SORT_CTAS, SORT_THREADS, smem, st>>>(a.tokens, a.wide, (int)a.n, (uint32_t)a.vocab, bits, passes, key0, pos0,
                                                          key1, pos1, status);
  if (cudaGetLastError() != cudaSuccess) return "token_sort launch failed";
  const uint32_t* key = (passes & 1) ? key0 : key1;             // pass p wrote buffer p & 1
  const uint32_t* pos = (passes & 1) ? pos0 : pos1;
  switch (a.dtype) {
    case ELEM_BF16: return a.add ? grad_typed<__nv_bfloat16, true>(a, key, pos, st) : grad_typed<__nv_bfloat16, false>(a, key, pos, st);
    case ELEM_F16: return a.add ? grad_typed<__half, true>(a, key, pos, st) : grad_typed<__half, false>(a, key, pos, st);
    case ELEM_F32: return a.add ? grad_typed<float, true>(a, key, pos, st) : grad_typed<float, false>(a, key, pos, st);
  }
  return "token_grad: unknown element type";
}

}  // namespace gd
