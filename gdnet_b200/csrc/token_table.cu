// Token table: lookup with scaling, and its gradient by sorted tokens.
//
//   lookup     out[t, :] = scale * W[tok_t, :]
//   gradient   dW[v, :] (+)= scale * sum over {t : tok_t = v} of dY[t, :]
//
// The gradient sorts the token positions by id (stable, so the rows of one id stay in the order of the batch), then
// walks the sorted list in chunks and sums the rows of each id in fp32 registers. An element is written once, or added once to
// what stood there: the same inputs give the same bits. Both directions move every row once and are bound by memory bandwidth; the sort moves 16 bytes a
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
// row slots and each slot fetches two rows at a time: two ids, then two row pieces in flight per thread (with four or eight a
// batch of 32768 x 1024 bf16 took 22.5 and 30.7 us instead of 18.4, whose bytes need 13: too few blocks to spread). The rows
// written are not kept in cache before others, so the table stays there. An id outside [0, vocab) is never used as an
// index: its row is zero and the status word records it.
constexpr int LOOKUP_THREADS = 256;
constexpr int LOOKUP_ROWS = 2;

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
      Vec<T, V>* to = reinterpret_cast<Vec<T, V>*>(out + (row * vecs + v) * V);
      if constexpr (sizeof(Vec<T, V>) == 16) __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(&x[r]));
      else *to = x[r];
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
// Least-significant-digit radix sort by one cluster of sixteen blocks (512 warps), so that a pass needs no launch of
// its own: every warp owns one contiguous slice of the list, counts its digits in a histogram of its own, and after
// one exchange of the blocks' totals through distributed shared memory knows where each of its digits goes. Digits
// are at most 9 bits (two passes up to a vocabulary of 2^18). Key and position travel as one 8-byte word: a pass of few SMs is
// bound by its stores and by the latency of its steps (32768 tokens: 8 blocks and two words 27 us, 16 blocks and one word 19).
// A token outside [0, vocab) gets the key `vocab` and sorts to the end, where the sums leave it out. The blocks behind the
// first cluster clear the dense gradient meanwhile.
constexpr int SORT_CTAS = 16;       // more than 8 need leave (cudaFuncAttributeNonPortableClusterSizeAllowed)
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_MAX_BITS = 9;
constexpr int SORT_ROW = SORT_WARPS + 1;
constexpr int SORT_UNROLL = 4;        // keys a lane has in flight

__device__ __forceinline__ uint32_t ld_dsmem_u32(uint32_t addr, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(addr, rank)) : "memory");
  return v;
}

__global__ void __cluster_dims__(SORT_CTAS, 1, 1) __launch_bounds__(SORT_THREADS)
token_sort_kernel(const void* __restrict__ tokens, int wide, int n, uint32_t vocab, int bits, int passes,
                  uint2* list0, uint2* list1, uint8_t* clear, int64_t clear_bytes,
                  Status* status) {
  if (blockIdx.x >= SORT_CTAS) {      // the destination is 16-byte aligned
    const int64_t step = (int64_t)(gridDim.x - SORT_CTAS) * SORT_THREADS, me = (int64_t)(blockIdx.x - SORT_CTAS) * SORT_THREADS + threadIdx.x;
    for (int64_t i = me; i < clear_bytes / 16; i += step) reinterpret_cast<uint4*>(clear)[i] = make_uint4(0, 0, 0, 0);
    if (me < clear_bytes % 16) clear[clear_bytes / 16 * 16 + me] = 0;
    return;
  }
  extern __shared__ uint32_t hist[];                 // [bins][SORT_WARPS], rows of 33 words: no bank is hit twice by a digit's
                                                     // warps, nor by a warp's neighbouring digits
  __shared__ uint32_t total[1 << SORT_MAX_BITS];     // this block's count of every digit
  __shared__ uint32_t first[1 << SORT_MAX_BITS];     // where this block's share of a digit begins
  __shared__ uint32_t warp_tot[SORT_WARPS];
  const int bins = 1 << bits;
  const uint32_t mask = (uint32_t)bins - 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster_ctarank();
  const int slice = ((n + SORT_CTAS * SORT_WARPS - 1) / (SORT_CTAS * SORT_WARPS) + 31) & ~31;
  const int64_t begin = (int64_t)(rank * SORT_WARPS + warp) * slice;
  const int lo = (int)(begin < n ? begin : n), hi = (int)(begin + slice < n ? begin + slice : n);
  const bool in_regs = slice <= 32 * SORT_UNROLL;    // one round: counted and placed without reading twice
  uint32_t* mine = hist + warp;

  for (int p = 0; p < passes; ++p) {
    const uint2* src = (p & 1) ? list0 : list1;      // pass p writes list p & 1; pass 0 reads the tokens
    uint2* dst = (p & 1) ? list1 : list0;
    const int shift = p * bits;
    uint32_t k[SORT_UNROLL], at[SORT_UNROLL];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int u = 0; u < SORT_UNROLL; ++u) {
        const int i = i0 + u * 32 + lane;
        k[u] = 0;
        at[u] = (uint32_t)i;
        if (i >= hi) continue;
        if (p != 0) {
          const uint2 w = __ldcg(src + i);
          k[u] = w.x;
          at[u] = w.y;
        } else {
          const int64_t t = token_at(tokens, wide, i);
          k[u] = (t < 0 || t >= (int64_t)vocab) ? vocab : (uint32_t)t;
        }
      }
    };
    for (int b = lane; b < bins; b += 32) mine[b * SORT_ROW] = 0;
    __syncwarp();
    for (int i0 = lo; i0 < hi; i0 += 32 * SORT_UNROLL) {
      fetch(i0);
#pragma unroll
      for (int u = 0; u < SORT_UNROLL; ++u) {
        const int i = i0 + u * 32 + lane;
        if (i >= hi) continue;
        if (p == 0 && k[u] == vocab) report(status, STATUS_BAD_ARGUMENT, 71, i);
        atomicAdd(&mine[((k[u] >> shift) & mask) * SORT_ROW], 1u);
      }
    }
    __syncthreads();
    // per digit: counts of the block's warps -> exclusive prefix, and the block's total. 2^split neighbouring lanes share a digit,
    // each with an equal range of the warps (a warp per digit and a scan across its lanes took three times as long).
    const int split = bins >= 512 ? 1 : 2, per = SORT_WARPS >> split;
    for (int t = threadIdx.x; t < bins << split; t += SORT_THREADS) {
      const int d = t >> split, piece = t & ((1 << split) - 1);
      uint32_t* at = hist + d * SORT_ROW + piece * per;
      uint32_t run = 0;
      for (int w0 = 0; w0 < per; w0 += 8) {
        uint32_t c[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) c[w] = at[w0 + w];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          at[w0 + w] = run;
          run += c[w];
        }
      }
      uint32_t before = 0, sum = run;
      for (int o = 1; o < 1 << split; o <<= 1) {
        const uint32_t other = __shfl_xor_sync(__activemask(), sum, o);
        if (piece & o) before += other;
        sum += other;
      }
      if (piece != 0)
        for (int w = 0; w < per; ++w) at[w] += before;
      if (piece == 0) total[d] = sum;
    }
    cluster_sync_all();
    // digit b starts at (all smaller digits of all blocks) + (digit b of the blocks before this one)
    uint32_t all = 0, before = 0;
    if ((int)threadIdx.x < bins) {
#pragma unroll
      for (uint32_t c = 0; c < SORT_CTAS; ++c) {
        const uint32_t t = ld_dsmem_u32(smem_u32(&total[threadIdx.x]), c);
        if (c < rank) before += t;
        all += t;
      }
    }
    uint32_t incl = all;
    if (warp * 32 < bins) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      if (lane == 31) warp_tot[warp] = incl;
    }
    __syncthreads();
    if ((int)threadIdx.x < bins) {
      uint32_t base = incl - all + before;
      for (int w = 0; w < warp; ++w) base += warp_tot[w];
      first[threadIdx.x] = base;
    }
    __syncthreads();
    // Place: equal digits of a warp's 32 keys keep their order (rank among the lower lanes). Neither ballots of the digit's bits
    // instead of the match, nor ordering the block's keys in shared memory before they are written, was faster.
    for (int i0 = lo; i0 < hi; i0 += 32 * SORT_UNROLL) {
      if (!in_regs) fetch(i0);
      uint32_t same[SORT_UNROLL];                      // lanes with the same digit
#pragma unroll
      for (int u = 0; u < SORT_UNROLL; ++u)
        same[u] = __match_any_sync(0xffffffffu, i0 + u * 32 + lane < hi ? (k[u] >> shift) & mask : 0xffffffffu);
#pragma unroll
      for (int u = 0; u < SORT_UNROLL; ++u) {
        const bool live = i0 + u * 32 + lane < hi;
        const uint32_t d = (k[u] >> shift) & mask;
        const int before_me = __popc(same[u] & ((1u << lane) - 1));
        if (live) dst[first[d] + mine[d * SORT_ROW] + before_me] = make_uint2(k[u], at[u]);
        __syncwarp();
        if (live && before_me == 0) mine[d * SORT_ROW] += __popc(same[u]);
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
// The sorted list is cut into chunks of `chunk` rows; `tpr` threads cover a row and walk one chunk. Each
// thread's pieces of the next GRAD_RING rows are on their way into shared memory (asynchronous copies that only this thread
// reads: no synchronisation), so the loop is short; with the rows in registers and unrolled, the code that ends an id was
// there 8 or 16 times and fetching it took longer than the rows (35 and 90 us against 30 for 32768 x 1024, whose bytes need 21).
// An id whose rows all lie in one chunk is finished there. An id that runs over a chunk's end leaves partial sums: slot 0
// of a chunk holds the sum of the id that was already running when the chunk began, slot 1 the sum of the id that runs
// on. token_grad_join_kernel adds those up in the order of the chunks.
constexpr int GRAD_THREADS = 128;
constexpr int GRAD_INFLIGHT = 8;
constexpr int GRAD_MAX_CHUNK = 64;
constexpr int GRAD_RING = 16;
constexpr uint32_t NO_KEY = 0xffffffffu;

template <int BYTES>
__device__ __forceinline__ void cp_async_bytes(void* smem_dst, const void* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem_dst)), "l"(src) : "memory");
  else if constexpr (BYTES >= 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(smem_dst)), "l"(src), "n"(BYTES) : "memory");
}

// The sum of an id, scaled, to its row. Adding, each element of a call gets exactly one addition, so a reduction in L2 gives
// the same bits as reading, adding and storing, without waiting for the row.
template <typename T, int V, bool ADD>
__device__ __forceinline__ void emit_row(void* out, int64_t at, const float (&acc)[V], float scale) {
  if (ADD) {
    float* o = reinterpret_cast<float*>(out) + at;
    if constexpr (V % 4 == 0) {
#pragma unroll
      for (int q = 0; q < V; q += 4) red_add_v4(o + q, acc[q] * scale, acc[q + 1] * scale, acc[q + 2] * scale, acc[q + 3] * scale);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) atomicAdd(o + i, acc[i] * scale);
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
token_grad_sum_kernel(const uint2* __restrict__ sorted, int n, uint32_t vocab,
                      const T* __restrict__ grad, int64_t grad_ld, int vecs, int tpr_log2, int chunk, int n_chunks,
                      float scale, void* __restrict__ out, float* __restrict__ partial) {
  extern __shared__ uint2 entries[];                    // this block's part of the list: chunks back to back, one entry more
  const int tpr = 1 << tpr_log2, per_block = GRAD_THREADS >> tpr_log2;
  const int v = blockIdx.y * tpr + (threadIdx.x & (tpr - 1));
  const int64_t block_lo = (int64_t)blockIdx.x * per_block * chunk;
  for (int i = threadIdx.x; i <= per_block * chunk; i += GRAD_THREADS)
    entries[i] = block_lo + i < n ? sorted[block_lo + i] : make_uint2(NO_KEY, 0);
  __syncthreads();
  const int c = blockIdx.x * per_block + (threadIdx.x >> tpr_log2);
  if (c >= n_chunks || v >= vecs) return;
  const int64_t width = (int64_t)vecs * V, col = (int64_t)v * V;
  const int lo = c * chunk, count = min(n - lo, chunk);
  const uint2* mine = entries + (threadIdx.x >> tpr_log2) * chunk;
  const uint32_t key_before = lo > 0 ? sorted[lo - 1].x : NO_KEY, key_after = mine[count].x;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
  uint32_t cur = mine[0].x;
  bool open_left = cur == key_before;       // the running id began in an earlier chunk
  constexpr int BYTES = V * (int)sizeof(T);
  constexpr bool ASYNC = BYTES >= 4;        // odd widths of 16-bit elements are read where they are needed
  uint8_t* ring = reinterpret_cast<uint8_t*>(entries) + ((per_block * chunk + 1) * 8 + 15) / 16 * 16 + threadIdx.x * BYTES;
  auto fetch = [&](int j) {
    if (ASYNC) {
      if (j < count) {
        const uint2 w = mine[j];
        if (w.x < vocab) cp_async_bytes<BYTES>(ring + (j & (GRAD_RING - 1)) * (GRAD_THREADS * BYTES), grad + (int64_t)w.y * grad_ld + col);
      }
      cp_async_commit();
    }
  };
  for (int j = 0; j < GRAD_RING - 1; ++j) fetch(j);
#pragma unroll 1
  for (int j = 0; j < count; ++j) {
    const uint2 w = mine[j];
    fetch(j + GRAD_RING - 1);
    if (w.x != cur) {                       // the running id ends inside this chunk
      if (open_left) put_partial<V>(partial + ((int64_t)c * 2) * width + col, acc);
      else emit_row<T, V, ADD>(out, (int64_t)cur * width + col, acc, scale);
      open_left = false;
      cur = w.x;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    }
    if (w.x >= vocab) break;                // ids outside the table come last
    Vec<T, V> x;
    if (ASYNC) {
      cp_async_wait_but<GRAD_RING - 1>();
      x = *reinterpret_cast<const Vec<T, V>*>(ring + (j & (GRAD_RING - 1)) * (GRAD_THREADS * BYTES));
    } else {
      x = *reinterpret_cast<const Vec<T, V>*>(grad + (int64_t)w.y * grad_ld + col);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += to_f32(x.e[i]);
  }
  cp_async_wait_but<0>();
  if (cur >= vocab) return;
  if (open_left) put_partial<V>(partial + ((int64_t)c * 2) * width + col, acc);
  else if (cur == key_after) put_partial<V>(partial + ((int64_t)c * 2 + 1) * width + col, acc);
  else emit_row<T, V, ADD>(out, (int64_t)cur * width + col, acc, scale);
}

// For every chunk whose last id runs on into the next chunk and began in this one: its partial sums, in order. A block looks
// at one chunk; its groups of tpr threads take equal ranges of the partial sums, which are then added up in order.
constexpr int JOIN_THREADS = 512;

template <typename T, int V, bool ADD>
__global__ void __launch_bounds__(JOIN_THREADS)
token_grad_join_kernel(const uint2* __restrict__ sorted, uint32_t vocab, int vecs, int tpr_log2, int chunk,
                       int n_chunks, float scale, void* __restrict__ out, const float* __restrict__ partial) {
  __shared__ float part[JOIN_THREADS * V];
  const int tpr = 1 << tpr_log2, groups = JOIN_THREADS >> tpr_log2, group = threadIdx.x >> tpr_log2;
  const int v = blockIdx.y * tpr + (threadIdx.x & (tpr - 1));
  const int c = blockIdx.x;
  const int lo = c * chunk, hi = lo + chunk;                    // a full chunk: it is not the last one
  const uint32_t id = sorted[hi - 1].x, before = lo > 0 ? sorted[lo - 1].x : NO_KEY, at_lo = sorted[lo].x, after = sorted[hi].x;
  if (id >= vocab || after != id) return;                       // nothing runs on
  if (at_lo == id && before == id) return;                      // the id began before this chunk
  // last chunk that the id reaches: every lane looks at one chunk's end
  int last = c + 1;
  for (;; last += 32) {
    const int j = last + (threadIdx.x & 31);                    // does the id run on past chunk j?
    const bool on = j < n_chunks - 1 && sorted[(j + 1) * chunk - 1].x == id && sorted[(j + 1) * chunk].x == id;
    const uint32_t stop = __ballot_sync(0xffffffffu, !on);
    if (stop != 0) {
      last += __ffs(stop) - 1;
      break;
    }
  }
  const int64_t width = (int64_t)vecs * V, col = (int64_t)v * V;
  const int count = last - c + 1, per = (count + groups - 1) / groups;      // partial sums c (slot 1), c + 1 ... last (slot 0)
  const int g0 = group * per, g1 = min(count, g0 + per);
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
  if (v < vecs) {
    for (int j0 = g0; j0 < g1; j0 += 4) {
      Vec<float, (V < 4 ? V : 4)> x[4][V < 4 ? 1 : V / 4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j0 + u >= g1) continue;
        const float* q = partial + ((int64_t)(c + j0 + u) * 2 + (j0 + u == 0 ? 1 : 0)) * width + col;
#pragma unroll
        for (int i = 0; i < (V < 4 ? 1 : V / 4); ++i) x[u][i] = reinterpret_cast<const Vec<float, (V < 4 ? V : 4)>*>(q)[i];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j0 + u >= g1) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += x[u][i / (V < 4 ? V : 4)].e[i % (V < 4 ? V : 4)];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) part[i * JOIN_THREADS + threadIdx.x] = acc[i];
  __syncthreads();
  if (group != 0 || v >= vecs) return;
  for (int w = 1; w < groups && w * per < count; ++w)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += part[i * JOIN_THREADS + w * tpr + threadIdx.x];
  emit_row<T, V, ADD>(out, (int64_t)id * width + col, acc, scale);
}

// ---------------------------------------------------------------------------------------
// short lists: no sort
// ---------------------------------------------------------------------------------------
// Each block owns every gridDim.x-th row of the table (frequent ids are neighbours in most vocabularies) and 32 accesses of
// their columns. It reads the whole list of tokens, keeps those of its rows in order, and sums every row (or clears it): one
// launch instead of three dependent ones. Rows with up to 32 tokens take one warp, others all eight.
constexpr int DIRECT_THREADS = 256;
constexpr int DIRECT_WARPS = DIRECT_THREADS / 32;
constexpr int DIRECT_MAX = 2048;         // tokens
constexpr int DIRECT_ROWS = 256;         // most table rows per block

template <typename T, int V, bool ADD>
__global__ void __launch_bounds__(DIRECT_THREADS)
token_grad_direct_kernel(const void* __restrict__ tokens, int wide, int n, uint32_t vocab, const T* __restrict__ grad,
                         int64_t grad_ld, int vecs, float scale, void* __restrict__ out, Status* status) {
  __shared__ uint32_t found[DIRECT_MAX];                 // row of this block << 16 | token, in the order of the list
  __shared__ uint16_t list[DIRECT_MAX];                  // tokens by row
  __shared__ int start[DIRECT_ROWS + 1], fill[DIRECT_ROWS];
  __shared__ int warp_count[DIRECT_WARPS];
  __shared__ int n_long;
  __shared__ uint8_t long_rows[DIRECT_ROWS];             // rows with more than 32 tokens
  __shared__ float part[DIRECT_WARPS][32 * V + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t stride = gridDim.x;                     // row r of this block is row blockIdx.x + r * stride of the table
  const int here = (int)((vocab - blockIdx.x + stride - 1) / stride);
  const int v = blockIdx.y * 32 + lane;
  const int64_t width = (int64_t)vecs * V, col = (int64_t)v * V;

  for (int r = threadIdx.x; r < here; r += DIRECT_THREADS) fill[r] = 0;
  __syncthreads();
  int count = 0;
  for (int t0 = 0; t0 < n; t0 += DIRECT_THREADS * 4) {      // four tokens a thread in flight, kept in the order of the list
    int mine[4];                                            // row of this block, or -1
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + u * DIRECT_THREADS + threadIdx.x;
      const int64_t id = t < n ? token_at(tokens, wide, t) : 0;
      const bool good = id >= 0 && id < (int64_t)vocab;
      if (!good && blockIdx.x == 0 && blockIdx.y == 0) report(status, STATUS_BAD_ARGUMENT, 71, t);
      const uint32_t r = (uint32_t)id / stride;
      mine[u] = t < n && good && (uint32_t)id - r * stride == blockIdx.x ? (int)r : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (t0 + u * DIRECT_THREADS >= n) break;
      const bool hit = mine[u] >= 0;
      const uint32_t ball = __ballot_sync(0xffffffffu, hit);
      if (lane == 0) warp_count[warp] = __popc(ball);
      __syncthreads();
      int before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < DIRECT_WARPS; ++w) {
        const int c = warp_count[w];
        if (w < warp) before += c;
        all += c;
      }
      if (hit) {
        found[count + before + __popc(ball & ((1u << lane) - 1))] =
            (uint32_t)mine[u] << 16 | (uint32_t)(t0 + u * DIRECT_THREADS + threadIdx.x);
        atomicAdd(&fill[mine[u]], 1);
      }
      count += all;
      __syncthreads();
    }
  }
  // where each row's tokens begin, and the tokens by row, each row's in order (one warp: few of the tokens are this block's)
  if (warp == 0) {
    int run = 0, longs = 0;
    for (int r0 = 0; r0 < here; r0 += 32) {
      const int c = r0 + lane < here ? fill[r0 + lane] : 0;
      const uint32_t big = __ballot_sync(0xffffffffu, c > 32);
      if (c > 32) long_rows[longs + __popc(big & ((1u << lane) - 1))] = (uint8_t)(r0 + lane);
      longs += __popc(big);
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      if (r0 + lane < here) {
        start[r0 + lane] = run + incl - c;
        fill[r0 + lane] = run + incl - c;
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      start[here] = run;
      n_long = longs;
    }
    __syncwarp();
    for (int i0 = 0; i0 < count; i0 += 32) {
      const bool live = i0 + lane < count;
      const uint32_t f = live ? found[i0 + lane] : 0xffffffffu;
      const uint32_t same = __match_any_sync(0xffffffffu, f >> 16);
      const int rank = __popc(same & ((1u << lane) - 1));
      if (live) list[fill[f >> 16] + rank] = (uint16_t)(f & 0xffffu);
      __syncwarp();
      if (live && rank == 0) fill[f >> 16] += __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();

  // sum of list[i0 .. i1) in order, eight rows in flight
  auto sum_range = [&](int i0, int i1, float (&acc)[V]) {
    for (int i = i0; i < i1; i += GRAD_INFLIGHT) {
      Vec<T, V> x[GRAD_INFLIGHT];
#pragma unroll
      for (int u = 0; u < GRAD_INFLIGHT; ++u)
        if (i + u < i1) x[u] = *reinterpret_cast<const Vec<T, V>*>(grad + (int64_t)list[i + u] * grad_ld + col);
#pragma unroll
      for (int u = 0; u < GRAD_INFLIGHT; ++u)
        if (i + u < i1) {
#pragma unroll
          for (int q = 0; q < V; ++q) acc[q] += to_f32(x[u].e[q]);
        }
    }
  };
  for (int r = warp; r < here; r += DIRECT_WARPS) {
    const int i0 = start[r], i1 = start[r + 1];
    if (v >= vecs || i1 - i0 > 32 || (ADD && i0 == i1)) continue;
    float acc[V];
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] = 0.0f;
    sum_range(i0, i1, acc);
    emit_row<T, V, ADD>(out, ((int64_t)blockIdx.x + (int64_t)r * stride) * width + col, acc, scale);
  }
  for (int l = 0; l < n_long; ++l) {
    const int r = long_rows[l];
    const int i0 = start[r], i1 = start[r + 1];
    const int per = (i1 - i0 + DIRECT_WARPS - 1) / DIRECT_WARPS;
    float acc[V];
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] = 0.0f;
    if (v < vecs) sum_range(i0 + warp * per, min(i1, i0 + (warp + 1) * per), acc);
    __syncthreads();                  // the sums of the row before have been read
#pragma unroll
    for (int q = 0; q < V; ++q) part[warp][q * 32 + lane] = acc[q];
    __syncthreads();
    if (warp == 0 && v < vecs) {
      for (int w = 1; w < DIRECT_WARPS; ++w)
#pragma unroll
        for (int q = 0; q < V; ++q) acc[q] += part[w][q * 32 + lane];
      emit_row<T, V, ADD>(out, ((int64_t)blockIdx.x + (int64_t)r * stride) * width + col, acc, scale);
    }
  }
}

// Rows per chunk: as many as leave 480 blocks of 128 threads (three to four an SM), between 16 and 64. 32768 x 1024: 62 us with
// 64 rows, 67 with 32, 78 with 128; 8192 x 1024: 35 us with 16, 43 with 64.
static int grad_chunk(int64_t n, int vecs) {
  const int l = tpr_log2_for(vecs, 7);
  const int64_t row_blocks = (n >> (7 - l)) * ((vecs + (1 << l) - 1) >> l);      // blocks with one row per chunk
  int c = 16;
  while (c < GRAD_MAX_CHUNK && row_blocks / (2 * c) >= 480) c *= 2;
  return c;
}

int64_t token_grad_partial_floats(int64_t n, int64_t width) {
  if (n <= DIRECT_MAX) return 0;
  return ((n + 15) / 16) * 2 * width;      // chunks have 16 rows or more
}

// Up to 2048 tokens the sort is left out: 2048 tokens add up in 12 to 25 us (vocabulary 4096 to 100288) without it, 25 to 27 with
// it; 4096 tokens in 17 to 33 us without it, 25 to 30 with it.
static bool grad_is_direct(int64_t n) { return n <= DIRECT_MAX; }

template <typename T, int V, bool ADD>
static const char* grad_as(const TokenGradArgs& a, const uint2* sorted, Status* status, cudaStream_t st) {
  const int vecs = (int)(a.width / V);
  if (grad_is_direct(a.n)) {
    const unsigned slabs = (unsigned)((vecs + 31) / 32);
    if (slabs > 65535) return "token_grad: rows too wide";
    // about 600 blocks, of at most DIRECT_ROWS rows
    int64_t rows = (a.vocab * slabs + 591) / 592;
    rows = rows < 1 ? 1 : (rows > DIRECT_ROWS ? DIRECT_ROWS : rows);
    const dim3 grid((unsigned)((a.vocab + rows - 1) / rows), slabs);
    token_grad_direct_kernel<T, V, ADD><<<grid, DIRECT_THREADS, 0, st>>>(a.tokens, a.wide, (int)a.n, (uint32_t)a.vocab,
        reinterpret_cast<const T*>(a.grad), a.grad_ld, vecs, a.scale, a.out, status);
    return cudaGetLastError() == cudaSuccess ? nullptr : "token_grad launch failed";
  }
  const int l = tpr_log2_for(vecs, 7);
  const int chunk = grad_chunk(a.n, vecs);
  const int n_chunks = (int)((a.n + chunk - 1) / chunk);
  const int per_block = GRAD_THREADS >> l;
  const dim3 grid((unsigned)((n_chunks + per_block - 1) / per_block), (unsigned)((vecs + (1 << l) - 1) >> l));
  if (grid.y > 65535) return "token_grad: rows too wide";
  const int smem = ((per_block * chunk + 1) * 8 + 15) / 16 * 16 + GRAD_RING * GRAD_THREADS * V * (int)sizeof(T);
  if (cudaFuncSetAttribute(token_grad_sum_kernel<T, V, ADD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (GRAD_THREADS * GRAD_MAX_CHUNK + 2) * 8 + GRAD_RING * GRAD_THREADS * 16) != cudaSuccess)
    return "token_grad: shared memory";
  token_grad_sum_kernel<T, V, ADD><<<grid, GRAD_THREADS, smem, st>>>(sorted, (int)a.n, (uint32_t)a.vocab,
      reinterpret_cast<const T*>(a.grad), a.grad_ld, vecs, l, chunk, n_chunks, a.scale, a.out, a.partial);
  if (n_chunks > 1)
    token_grad_join_kernel<T, V, ADD><<<dim3((unsigned)(n_chunks - 1), grid.y), JOIN_THREADS, 0, st>>>(sorted, (uint32_t)a.vocab, vecs, l,
                                                                                          chunk, n_chunks, a.scale, a.out, a.partial);
  return cudaGetLastError() == cudaSuccess ? nullptr : "token_grad launch failed";
}

template <typename T, bool ADD>
static const char* grad_typed(const TokenGradArgs& a, const uint2* sorted, Status* status, cudaStream_t st) {
  // adding, the destination's elements have four bytes: twice a 16-bit row's, in accesses of at most 16
  const uint64_t out_bits = (uint64_t)(uintptr_t)a.out & 15;
  const uint64_t bits = (uint64_t)(uintptr_t)a.grad | (uint64_t)(a.grad_ld * (int64_t)sizeof(T)) |
                        (ADD && sizeof(T) == 2 ? out_bits >> 1 : out_bits);
  switch (vec_elems(sizeof(T), a.width, bits)) {
    case 8: if constexpr (sizeof(T) == 2) return grad_as<T, 8, ADD>(a, sorted, status, st); break;
    case 4: return grad_as<T, 4, ADD>(a, sorted, status, st);
    case 2: return grad_as<T, 2, ADD>(a, sorted, status, st);
    default: break;
  }
  return grad_as<T, 1, ADD>(a, sorted, status, st);
}

static size_t sort_smem(int bits) {
  return (size_t)SORT_ROW * (1u << bits) * sizeof(uint32_t);
}

int64_t token_grad_sort_words(int64_t n) { return grad_is_direct(n) ? 0 : 4 * n; }

const char* launch_token_grad(const TokenGradArgs& a, Status* status, cudaStream_t st) {
  if (a.width == 0 || a.vocab == 0) return nullptr;
  if (a.n >= (1ll << 30) || a.vocab >= (1ll << 31) || a.width > (1 << 30)) return "token_grad: sizes out of range";
  if (a.n == 0 && a.add) return nullptr;
  const uint2* sorted = nullptr;
  if (!grad_is_direct(a.n)) {
    int need = 0;
    while (need < 31 && (a.vocab >> need) != 0) ++need;           // keys are 0..vocab
    const int passes = (need + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
    const int bits = (need + passes - 1) / passes;
    const size_t smem = sort_smem(bits);
    if (cudaFuncSetAttribute(token_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)sort_smem(SORT_MAX_BITS)) != cudaSuccess ||
        cudaFuncSetAttribute(token_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return "token_sort: shared memory";
    uint2* list0 = reinterpret_cast<uint2*>(a.sort);
    uint2* list1 = list0 + a.n;
    const int64_t size = a.dtype == ELEM_F32 ? 4 : 2;
    const int64_t clear = a.add ? 0 : a.vocab * a.width * size;
    if (clear != 0 && reinterpret_cast<uintptr_t>(a.out) % 16 != 0) return "token_grad: a dense gradient must be 16-byte aligned";
    const unsigned others = clear == 0 ? 0 : (unsigned)(clear / (1 << 20) < 7 ? clear / (1 << 20) + 1 : 7);      // clusters that clear
    token_sort_kernel<<<SORT_CTAS * (1 + others), SORT_THREADS, smem, st>>>(a.tokens, a.wide, (int)a.n, (uint32_t)a.vocab, bits, passes,
        list0, list1, reinterpret_cast<uint8_t*>(a.out), clear, status);
    if (cudaGetLastError() != cudaSuccess) return "token_sort launch failed";
    sorted = (passes & 1) ? list0 : list1;                        // pass p wrote list p & 1
  }
  switch (a.dtype) {
    case ELEM_BF16: return a.add ? grad_typed<__nv_bfloat16, true>(a, sorted, status, st) : grad_typed<__nv_bfloat16, false>(a, sorted, status, st);
    case ELEM_F16: return a.add ? grad_typed<__half, true>(a, sorted, status, st) : grad_typed<__half, false>(a, sorted, status, st);
    case ELEM_F32: return a.add ? grad_typed<float, true>(a, sorted, status, st) : grad_typed<float, false>(a, sorted, status, st);
  }
  return "token_grad: unknown element type";
}

}  // namespace gd
