// Orthogonalising matrices by Newton-Schulz products, and the momentum update built on it.
//
// For a batch of matrices X (r x c), each divided by its Frobenius norm, `steps` times
//
//     A = X X^T,   B = b A + c A^2,   X <- a X + B X          (r <= c; otherwise A = X^T X and X <- a X + X B)
//
// which moves every singular value s to s (a + b s^2 + c s^4) and keeps the singular vectors. Three products a step, the
// first two symmetric: only the tiles on and above the diagonal are computed and their transposes stored from the same
// registers, so a step costs k (k + 1) w + k (k + 1) k + 2 k^2 w operations with k = min(r, c), w = max(r, c), against
// 4 k^2 w + 2 k^3 without. Bound by the tensor cores from about k = 1024 on, by the latency of 3 x steps dependent
// products below.
//
// Number format. Operands are fp16, scaled by 2^14: with the coefficients that the host admits the spectral norms of X, A
// and B, and so their entries, stay below 3.9, and 3.9 * 2^14 < 65504, so entries down to 2^-28 keep all 11 bits.
// X is held as hi + lo, two fp16 values (22 bits). With `pairs` off the products read the high parts only and the
// linear term a X reads both: rounding errors then enter through B X alone, in the directions whose singular values
// are already large (error of the result 5e-4 to 1.7e-3 of its norm, below the 1.7e-3 of rounding it to bf16; without the
// low part in a X the noise of the large directions is amplified into the small ones, 3e-3 to 1e-1). With `pairs` on
// every operand is a pair and a product is the three partial products hi hi + hi lo + lo hi (the result is as exact
// as in fp32 arithmetic), at three times the tensor-core work and on single-CTA tiles, whose sums fit the registers. Sums are fp32 in TMEM; the norm is summed in fp64.
#include "orthogonalize.h"

#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.h"

namespace gd {

constexpr float NS_SCALE = 16384.0f;            // 2^14
constexpr float NS_UNSCALE = 1.0f / NS_SCALE;

// ---------------------------------------------------------------------------------------
// three-dimensional bulk copies (batch = slowest coordinate)
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* m, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(m)), "r"(src), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// ---------------------------------------------------------------------------------------
// one product over the batch
// ---------------------------------------------------------------------------------------
// D = acc_scale * P Q^T + aux_scale * aux, P (M x K), Q (N x K). Same structure as the GEMM kernels: a producer warp, an
// MMA warp, eight epilogue warps, two accumulators in TMEM. PAIR: a pair of CTAs (two SMs) shares a 256 x 256
// tile, each loading its half of both operands; otherwise a CTA has a 128 x 128 tile of its own (small matrices: more
// tiles, shorter chain).
constexpr int NS_BK = 64;                       // K elements per stage: one 128-byte swizzle row
constexpr int NS_EPI_WARPS = 8;
constexpr int NS_THREADS = 64 + NS_EPI_WARPS * 32;
constexpr int NS_OPERAND_BYTES = 128 * 128;     // 128 rows x 64 fp16 per CTA and operand
constexpr int NS_STAGE_BYTES = 2 * NS_OPERAND_BYTES;
constexpr int NS_STAGES = 5;
constexpr int NS_BOX = 32;                      // epilogue chunk: 32 x 32
constexpr int NS_STAGING_BYTES = NS_BOX * NS_BOX * 2;                 // 2 KB
constexpr int NS_STAGING_PER_WARP = 2 * NS_STAGING_BYTES;             // the chunk and its transpose
constexpr int NS_ACC = 2;
constexpr int NS_SPLIT_KBLOCKS = 2;             // pairs: K blocks summed in TMEM before the sum moves to registers

struct __align__(8) NsBars {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t acc_full[NS_ACC];
  uint64_t acc_empty[NS_ACC];
  uint32_t tmem_base;
  int abort;
};

constexpr int NS_SMEM = NS_STAGES * NS_STAGE_BYTES + NS_EPI_WARPS * NS_STAGING_PER_WARP + (int)sizeof(NsBars) + 1024;

__device__ __forceinline__ bool ns_aborted(const NsBars* b) { return *((volatile const int*)&b->abort) != 0; }
__device__ __forceinline__ void ns_abort(NsBars* b, Status* st, int code, int site, int detail) {
  report(st, code, site, detail);
  *((volatile int*)&b->abort) = 1;
}
__device__ __noinline__ bool ns_wait_slow(uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity); }
__device__ __forceinline__ bool ns_wait(uint32_t bar, uint32_t parity) {
  return mbar_try_wait(bar, parity) ? true : ns_wait_slow(bar, parity);
}
__device__ __forceinline__ uint64_t ns_desc(uint32_t hi, uint32_t lo) { return ((uint64_t)hi << 32) | (uint64_t)lo; }

// work item -> (matrix, row block, column block). Symmetric products list only column block >= row block.
__device__ __forceinline__ void ns_tile(const NsProduct& g, int item, int& z, int& mb, int& nb) {
  z = item / g.tiles;
  int t = item - z * g.tiles;
  if (!g.symmetric) {
    nb = t / g.tiles_m;          // neighbours share a column block
    mb = t - nb * g.tiles_m;
    return;
  }
  // column block nb holds the nb + 1 tiles t = nb (nb + 1) / 2 ... (blocks per side are few: count up)
  nb = 0;
  while (t > nb) { t -= nb + 1; ++nb; }
  mb = t;
}

// 16-byte piece `slot` (0..3) of row `row` of a 32 x 64-byte box in the 64-byte swizzle order of the bulk copies
__device__ __forceinline__ uint32_t ns_box_off(int row, int slot) {
  return (uint32_t)(row * 64 + ((slot ^ ((row >> 1) & 3)) << 4));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The staging boxes may still be the source of a bulk store of this warp: wait until it has been read. Warp-collective.
__device__ __forceinline__ void stage_drain() {
  if (elect_one()) bulk_wait_read_all();
  __syncwarp();
}

// One 32 x 32 chunk (this lane's row in w) to the box at column x, row y of matrix z. Warp-collective.
__device__ __forceinline__ void ns_put_box(uint8_t* stage, int lane, const uint32_t (&w)[16], const CUtensorMap* map, int x,
                                           int y, int z) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<uint4*>(stage + ns_box_off(lane, q)) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
  fence_proxy_async_smem();
  __syncwarp();
  if (elect_one()) {
    tma_store_3d(map, smem_u32(stage), x, y, z);
    bulk_commit_group();
  }
  __syncwarp();
}

// The transpose of the same chunk to column x, row y: column j of the chunk becomes row j of the box.
__device__ __forceinline__ void ns_put_box_t(uint8_t* stage, int lane, const uint32_t (&w)[16], const CUtensorMap* map, int x,
                                             int y, int z) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    *reinterpret_cast<uint16_t*>(stage + ns_box_off(2 * j, lane >> 3) + (lane & 7) * 2) = (uint16_t)(w[j] & 0xffffu);
    *reinterpret_cast<uint16_t*>(stage + ns_box_off(2 * j + 1, lane >> 3) + (lane & 7) * 2) = (uint16_t)(w[j] >> 16);
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (elect_one()) {
    tma_store_3d(map, smem_u32(stage), x, y, z);
    bulk_commit_group();
  }
  __syncwarp();
}

// rows [0, rows_valid) x 32 fp16 of a row-major matrix -> this lane's row (coalesced: 8 rows x 64 bytes at a time)
__device__ __forceinline__ void ns_get_rows(uint8_t* stage, int lane, uint32_t (&w)[16], const __half* base, int64_t ld,
                                            int rows_valid) {
  const int r_in = lane >> 2, slot = lane & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = r_in + 8 * j;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (row < rows_valid) u = *reinterpret_cast<const uint4*>(base + (int64_t)row * ld + slot * 8);
    *reinterpret_cast<uint4*>(stage + ns_box_off(row, slot)) = u;
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint4 u = *reinterpret_cast<const uint4*>(stage + ns_box_off(lane, q));
    w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w;
  }
  __syncwarp();
}

__device__ __forceinline__ float2 unpack_half2(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

template <bool PAIR, bool SPLIT>
__device__ __forceinline__ void ns_product_body(const NsMaps& maps, const NsProduct& g, Status* status) {
  constexpr int TILE_M = PAIR ? 256 : 128, TILE_N = PAIR ? 256 : 128;
  constexpr int ACC_COLS = TILE_N;
  constexpr int CHUNKS = TILE_N / 64;            // 32-column chunks per epilogue warp (two warps share a lane quarter)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + NS_STAGES * NS_STAGE_BYTES;
  NsBars* bars = reinterpret_cast<NsBars*>(staging + NS_EPI_WARPS * NS_STAGING_PER_WARP);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, units = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < NS_STAGES; ++s) {
      mbar_init(smem_u32(&bars->full[s]), 1);
      mbar_init(smem_u32(&bars->empty[s]), 1);
    }
    for (int a = 0; a < NS_ACC; ++a) {
      mbar_init(smem_u32(&bars->acc_full[a]), 1);
      mbar_init(smem_u32(&bars->acc_empty[a]), (PAIR ? 2 : 1) * NS_EPI_WARPS);
    }
    bars->abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(smem_u32(&bars->tmem_base), NS_ACC * ACC_COLS); tmem_relinquish_pair(); }
    else { tmem_alloc(smem_u32(&bars->tmem_base), NS_ACC * ACC_COLS); tmem_relinquish(); }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  tc_fence_after_sync();
  pdl_enter();
  const uint32_t tmem_base = bars->tmem_base;

  const int n_work = g.batch * g.tiles;
  const int kblocks = (g.K + NS_BK - 1) / NS_BK;
  constexpr int SEGS = SPLIT ? 3 : 1;
  // K blocks that one accumulator in TMEM takes: all of them, or, with pairs, few enough for the sum to stay as exact as fp32
  const int per_acc = SPLIT ? NS_SPLIT_KBLOCKS : kblocks;
  const int n_acc = (kblocks * SEGS + per_acc - 1) / per_acc;
  const uint32_t smem0 = smem_u32(smem);
  const uint32_t full0 = smem_u32(&bars->full[0]), empty0 = smem_u32(&bars->empty[0]);
  const uint32_t afull0 = smem_u32(&bars->acc_full[0]), aempty0 = smem_u32(&bars->acc_empty[0]);

  if (warp == 0) {
    const uint32_t full_lead0 = PAIR ? map_to_cta(full0, 0) : full0;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int work = unit; work < n_work && ok; work += units) {
      int z, mb, nb;
      ns_tile(g, work, z, mb, nb);
      const int m0 = mb * TILE_M + (int)rank * 128, n0 = nb * TILE_N + (int)rank * 128;
      for (int seg = 0; seg < SEGS && ok; ++seg) {
        // hi lo, lo hi, hi hi: the small partial products first
        const CUtensorMap* ma = (SPLIT && seg == 1) ? &maps.p_lo : &maps.p_hi;
        const CUtensorMap* mq = (SPLIT && seg == 0) ? &maps.q_lo : &maps.q_hi;
        for (int kb = 0, kx = 0; kb < kblocks; ++kb, kx += NS_BK) {
          if (!__all_sync(0xffffffffu, ns_wait(empty0 + 8 * s, ph ^ 1))) {
            if (lane == 0) ns_abort(bars, status, STATUS_TIMEOUT_SMEM_EMPTY, 80, s);
            ok = false;
            break;
          }
          const uint32_t full = full_lead0 + 8 * s;
          const uint32_t a_dst = smem0 + s * NS_STAGE_BYTES, q_dst = a_dst + NS_OPERAND_BYTES;
          if (elect_one()) {
            if (!PAIR || rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, (PAIR ? 2 : 1) * NS_STAGE_BYTES);
            auto load = [&](uint32_t dst, const CUtensorMap* m, int x, int y) {
              if (PAIR) tma_load_3d_pair(dst, m, full, x, y, z);
              else tma_load_3d(dst, m, full, x, y, z);
            };
            if (!g.p_mn) load(a_dst, ma, kx, m0);
            else {
#pragma unroll
              for (int i = 0; i < 2; ++i) load(a_dst + i * (NS_BK * 128), ma, m0 + i * 64, kx);
            }
            if (!g.q_mn) load(q_dst, mq, kx, n0);
            else {
#pragma unroll
              for (int i = 0; i < 2; ++i) load(q_dst + i * (NS_BK * 128), mq, n0 + i * 64, kx);
            }
          }
          __syncwarp();
          if (++s == NS_STAGES) { s = 0; ph ^= 1; }
        }
      }
      if (ns_aborted(bars)) break;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = make_instr_desc(0, 0, g.p_mn ? 1 : 0, g.q_mn ? 1 : 0, TILE_M, TILE_N);
      const uint32_t p_lbo = g.p_mn ? NS_BK * 128 : 16, q_lbo = g.q_mn ? NS_BK * 128 : 16;
      const uint32_t p_step = g.p_mn ? (16 * 128) >> 4 : 2, q_step = g.q_mn ? (16 * 128) >> 4 : 2;
      const uint64_t p_tmpl = make_smem_desc(smem0, p_lbo, 1024), q_tmpl = make_smem_desc(smem0 + NS_OPERAND_BYTES, q_lbo, 1024);
      const uint32_t p_hi = (uint32_t)(p_tmpl >> 32), p_lo0 = (uint32_t)p_tmpl;
      const uint32_t q_hi = (uint32_t)(q_tmpl >> 32), q_lo0 = (uint32_t)q_tmpl;
      int s = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int work = unit; work < n_work && ok; work += units) {
        for (int part = 0; part < n_acc && ok; ++part) {
          if (!__all_sync(0xffffffffu, ns_wait(aempty0 + 8 * acc, acc_ph ^ 1))) {
            if (lane == 0) ns_abort(bars, status, STATUS_TIMEOUT_TMEM_EMPTY, 81, acc);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + acc * ACC_COLS;
          const int count = min(per_acc, kblocks * SEGS - part * per_acc);
          uint32_t accumulate = 0;
          for (int i = 0; i < count; ++i) {
            if (!__all_sync(0xffffffffu, ns_wait(full0 + 8 * s, ph))) {
              if (lane == 0) ns_abort(bars, status, STATUS_TIMEOUT_SMEM_FULL, 82, s);
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const uint32_t p_lo = p_lo0 + s * (NS_STAGE_BYTES >> 4), q_lo = q_lo0 + s * (NS_STAGE_BYTES >> 4);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < NS_BK / 16; ++k) {
                const uint64_t dp = ns_desc(p_hi, p_lo + k * p_step), dq = ns_desc(q_hi, q_lo + k * q_step);
                const uint32_t on = k == 0 ? accumulate : 1u;
                if (PAIR) mma_bf16_pair(d_tmem, dp, dq, idesc, on);      // kind::f16; idesc says fp16
                else mma_bf16(d_tmem, dp, dq, idesc, on);
              }
              if (PAIR) mma_commit_pair(empty0 + 8 * s);
              else mma_commit(empty0 + 8 * s);
            }
            __syncwarp();
            accumulate = 1;
            if (++s == NS_STAGES) { s = 0; ph ^= 1; }
          }
          if (!ok || ns_aborted(bars)) { ok = false; break; }
          if (elect_one()) {
            if (PAIR) mma_commit_pair(afull0 + 8 * acc);
            else mma_commit(afull0 + 8 * acc);
          }
          __syncwarp();
          if (++acc == NS_ACC) { acc = 0; acc_ph ^= 1; }
        }
      }
    }
  } else {
    const int ew = warp - 2;
    uint8_t* box = staging + ew * NS_STAGING_PER_WARP;
    uint8_t* box_t = box + NS_STAGING_BYTES;
    const int quarter = warp & 3, half = ew >> 2;
    const uint32_t aempty_lead0 = PAIR ? map_to_cta(aempty0, 0) : aempty0;
    int acc = 0;
    uint32_t acc_ph = 0;
    for (int work = unit; work < n_work && !ns_aborted(bars); work += units) {
      int z, mb, nb;
      ns_tile(g, work, z, mb, nb);
      const int m_warp = mb * TILE_M + (int)rank * 128 + quarter * 32;
      const int n_half = nb * TILE_N + half * (TILE_N / 2);
      const bool mirror = g.symmetric && mb != nb;
      const int rows_valid = min(32, g.M - m_warp);
      auto acc_wait = [&]() -> bool {
        if (mbar_wait_warp(afull0 + 8 * acc, acc_ph)) {
          tc_fence_after_sync();
          return true;
        }
        ns_abort(bars, status, STATUS_TIMEOUT_TMEM_FULL, 83, acc);
        return false;
      };
      auto acc_release = [&]() {      // everything of this accumulator is in registers
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster(aempty_lead0 + 8 * acc);
          else mbar_arrive(aempty0 + 8 * acc);
        }
      };
      auto acc_row = [&]() { return tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * ACC_COLS + half * (TILE_N / 2); };
      // Pairs: the tensor core cuts a running sum where fp32 rounds it, an error of one sign that grows with the number of
      // additions, so every few K blocks the sum moves to registers and is continued there.
      float sum[SPLIT ? CHUNKS : 1][32];
      if (SPLIT) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[SPLIT ? c : 0][j] = 0.0f;
        bool ok = true;
        for (int part = 0; part < n_acc; ++part) {
          if (!(ok = acc_wait())) break;
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            uint32_t raw[32];
            tmem_ld_32x32(acc_row() + c * 32, raw);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[SPLIT ? c : 0][j] += __uint_as_float(raw[j]);
          }
          acc_release();
          if (++acc == NS_ACC) { acc = 0; acc_ph ^= 1; }
        }
        if (!ok) break;
      } else if (!acc_wait()) {
        break;
      }
#pragma unroll(SPLIT ? CHUNKS : 1)
      for (int c = 0; c < CHUNKS; ++c) {
        uint32_t raw[32];
        if (!SPLIT) tmem_ld_32x32(acc_row() + c * 32, raw);
        const int n0 = n_half + c * 32;
        const bool live = m_warp < g.M && n0 < g.N;      // warp-uniform
        float aux[32];
        if (live && g.aux_hi != nullptr) {
          const int64_t off = (int64_t)z * g.aux_stride + (int64_t)m_warp * g.aux_ld + n0;
          uint32_t w[16];
          stage_drain();
          ns_get_rows(box, lane, w, g.aux_hi + off, g.aux_ld, rows_valid);
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const float2 f = unpack_half2(w[t]);
            aux[2 * t] = f.x; aux[2 * t + 1] = f.y;
          }
          if (g.aux_lo != nullptr) {
            ns_get_rows(box, lane, w, g.aux_lo + off, g.aux_ld, rows_valid);
#pragma unroll
            for (int t = 0; t < 16; ++t) {
              const float2 f = unpack_half2(w[t]);
              aux[2 * t] += f.x; aux[2 * t + 1] += f.y;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) aux[j] = 0.0f;
        }
        if (SPLIT) {
#pragma unroll
          for (int j = 0; j < 32; ++j) raw[j] = __float_as_uint(sum[SPLIT ? c : 0][j]);
        } else {
          tmem_ld_wait();
          if (c == CHUNKS - 1) acc_release();
        }
        if (!live) continue;
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          const float v0 = fmaf(g.aux_scale, aux[2 * t], g.acc_scale * __uint_as_float(raw[2 * t]));
          const float v1 = fmaf(g.aux_scale, aux[2 * t + 1], g.acc_scale * __uint_as_float(raw[2 * t + 1]));
          hi[t] = pack_half2(v0, v1);
          const float2 h = unpack_half2(hi[t]);
          lo[t] = pack_half2(v0 - h.x, v1 - h.y);
        }
        stage_drain();
        ns_put_box(box, lane, hi, &maps.out_hi, n0, m_warp, z);
        if (mirror) ns_put_box_t(box_t, lane, hi, &maps.out_hi, m_warp, n0, z);
        if (g.store_lo) {
          stage_drain();
          ns_put_box(box, lane, lo, &maps.out_lo, n0, m_warp, z);
          if (mirror) ns_put_box_t(box_t, lane, lo, &maps.out_lo, m_warp, n0, z);
        }
      }
      if (!SPLIT && ++acc == NS_ACC) { acc = 0; acc_ph ^= 1; }
    }
    if (elect_one()) bulk_wait_all();      // the stores are complete before the kernel ends
    __syncwarp();
  }

  tc_fence_before_sync();
  __syncthreads();
  if (ns_aborted(bars)) {        // give copies in flight time to land before the shared memory is handed on (100 us)
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 100000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem_base, NS_ACC * ACC_COLS);
    else tmem_dealloc(tmem_base, NS_ACC * ACC_COLS);
  }
}

__global__ void __launch_bounds__(NS_THREADS, 1)
ns_product_kernel(const __grid_constant__ NsMaps maps, const __grid_constant__ NsProduct g, Status* status) {
  ns_product_body<false, false>(maps, g, status);
}

__global__ void __launch_bounds__(NS_THREADS, 1)
ns_product_split_kernel(const __grid_constant__ NsMaps maps, const __grid_constant__ NsProduct g, Status* status) {
  ns_product_body<false, true>(maps, g, status);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NS_THREADS, 1)
ns_product_pair_kernel(const __grid_constant__ NsMaps maps, const __grid_constant__ NsProduct g, Status* status) {
  ns_product_body<true, false>(maps, g, status);
}

// ---------------------------------------------------------------------------------------
// element-wise ends: momentum, norm, scaling into the operand format, result
// ---------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float ns_f32(T v);
template <>
__device__ __forceinline__ float ns_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float ns_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float ns_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
  if (dtype == ELEM_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == ELEM_BF16) return ns_f32(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return ns_f32(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int dtype, int64_t i, float v) {
  if (dtype == ELEM_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == ELEM_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += red[w];
  return s;
}

// u (fp32, row pitch ld) of every matrix and the blocks' partial sums of u^2. Without momentum u is the input itself.
//   g = scalars[1] * ((1 - beta * scalars[0]) * gt + beta * gi);   m <- mu m + g;   u = nesterov ? g + mu m : m
__global__ void __launch_bounds__(256)
ns_begin_kernel(const __grid_constant__ NsEnds e) {
  __shared__ double red[8];
  const int z = blockIdx.y;
  const int64_t numel = (int64_t)e.rows * e.cols;
  float kt = 1.0f, ki = 0.0f;
  if (e.scalars != nullptr) {
    kt = (1.0f - e.beta * e.scalars[0]) * e.scalars[1];
    ki = e.beta * e.scalars[1];
  }
  double ssq = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < numel; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / e.cols, c = i - r * e.cols;
    float u;
    if (e.momentum) {
      float g = load_elem(e.grad[z], e.grad_dtype, i);
      if (e.scalars != nullptr) {
        g *= kt;
        if (e.info[z] != nullptr) g = fmaf(ki, load_elem(e.info[z], e.grad_dtype, i), g);
      }
      float* mp = reinterpret_cast<float*>(e.moment[z]);
      const float m = fmaf(e.mu, mp[i], g);
      mp[i] = m;
      u = e.nesterov ? fmaf(e.mu, m, g) : m;
    } else {
      u = load_elem(e.grad[z], e.grad_dtype, r * e.grad_ld + c);
    }
    e.u[(int64_t)z * e.plane + r * e.ld + c] = u;
    ssq += (double)u * (double)u;
  }
  const double s = block_sum(ssq, red);
  if (threadIdx.x == 0) e.partial[(int64_t)z * gridDim.x + blockIdx.x] = s;
}

// u / (norm + eps) * 2^14 as hi + lo
__global__ void __launch_bounds__(256)
ns_scale_kernel(const __grid_constant__ NsEnds e, int n_partial) {
  const int z = blockIdx.y;
  double s = 0.0;
  for (int i = 0; i < n_partial; ++i) s += e.partial[(int64_t)z * n_partial + i];
  const double inv = (double)NS_SCALE / (sqrt(s) + (double)e.eps);
  const int64_t numel = (int64_t)e.rows * e.ld;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < numel; i += (int64_t)gridDim.x * 256) {
    if (i % e.ld >= e.cols) continue;
    const int64_t at = (int64_t)z * e.plane + i;
    const float v = (float)((double)e.u[at] * inv);
    const __half h = __float2half_rn(v);
    e.x_hi[at] = h;
    e.x_lo[at] = __float2half_rn(v - __half2float(h));
  }
}

// the result, or the parameter update p <- p * decay - step * x
__global__ void __launch_bounds__(256)
ns_end_kernel(const __grid_constant__ NsEnds e) {
  const int z = blockIdx.y;
  const int64_t numel = (int64_t)e.rows * e.cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < numel; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / e.cols, c = i - r * e.cols;
    const int64_t at = (int64_t)z * e.plane + r * e.ld + c;
    const float x = (__half2float(e.x_hi[at]) + __half2float(e.x_lo[at])) * NS_UNSCALE;
    if (e.momentum) store_elem(e.out[z], e.out_dtype, i, fmaf(-e.step, x, load_elem(e.out[z], e.out_dtype, i) * e.decay));
    else store_elem(e.out[z], e.out_dtype, i, x);
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn ns_encode_fn() {
  static EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// fp16 matrices [batch][rows][cols], row pitch ld, as boxes of box_rows x box_cols. Elements outside read as zero.
static bool ns_map(CUtensorMap* out, const __half* base, int64_t batch, int64_t rows, int64_t cols, int64_t ld, int64_t plane,
                   int box_rows, int box_cols, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = ns_encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(plane * 2)};
  cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int64_t ns_ld(int64_t cols) { return (cols + 31) / 32 * 32; }   // the epilogue reads whole 32-column chunks

// Layout of the workspace for `batch` matrices: X twice (hi and lo planes), A and B (hi and lo), norms.
struct NsSpace {
  int64_t ld_x, plane_x, ld_k, plane_k, x, k, partial, total;   // elements; x, k = one buffer's hi + lo
};
static NsSpace ns_space(int64_t batch, int64_t rows, int64_t cols) {
  NsSpace w;
  const int64_t k = rows < cols ? rows : cols;
  w.ld_x = ns_ld(cols);
  w.plane_x = rows * w.ld_x;
  w.ld_k = ns_ld(k);
  w.plane_k = k * w.ld_k;
  w.x = 2 * batch * w.plane_x;
  w.k = 2 * batch * w.plane_k;
  w.partial = 2 * w.x + 2 * w.k;                                // byte offset = 2 * elements, a multiple of 64
  w.total = 2 * w.partial + batch * NS_NORM_BLOCKS * (int64_t)sizeof(double);
  return w;
}

int64_t ns_workspace_bytes(int64_t batch, int64_t rows, int64_t cols) { return ns_space(batch, rows, cols).total; }

static const char* ns_launch_product(const NsMaps& maps, const NsProduct& g, bool pair, int sms, Status* status, cudaStream_t st) {
  const int work = g.batch * g.tiles;
  if (pair) {
    const int units = sms / 2 < work ? sms / 2 : work;
    if (launch_pdl(ns_product_pair_kernel, dim3(2 * units), dim3(NS_THREADS), NS_SMEM, st, maps, g, status) != cudaSuccess)
      return "ns_product_pair launch failed";
  } else {
    const int units = sms < work ? sms : work;
    if (launch_pdl(g.pairs ? ns_product_split_kernel : ns_product_kernel, dim3(units), dim3(NS_THREADS), NS_SMEM, st, maps, g, status) != cudaSuccess)
      return "ns_product launch failed";
  }
  return nullptr;
}

const char* launch_orthogonalize(const NsCall& call, Status* status, cudaStream_t st) {
  const int64_t batch = call.ends.batch, rows = call.ends.rows, cols = call.ends.cols;
  if (batch < 1 || batch > NS_MAX_BATCH || rows < 1 || cols < 1) return "orthogonalize: sizes";
  if (rows > (1 << 20) || cols > (1 << 20)) return "orthogonalize: matrix too large";
  const NsSpace w = ns_space(batch, rows, cols);
  __half* base = reinterpret_cast<__half*>(call.workspace);
  __half* x[2] = {base, base + w.x};                       // each: hi planes of the batch, then lo planes
  __half* A = base + 2 * w.x;
  __half* B = A + w.k;
  const int64_t lo_x = w.x / 2, lo_k = w.k / 2;
  const bool tall = rows > cols;
  const int k = (int)(tall ? cols : rows);

  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return "orthogonalize: device";

  NsEnds e = call.ends;
  e.ld = (int)w.ld_x;
  e.plane = w.plane_x;
  e.u = reinterpret_cast<float*>(x[1]);                    // hi and lo planes of the other X buffer: four bytes an element
  e.x_hi = x[0];
  e.x_lo = x[0] + lo_x;
  e.partial = reinterpret_cast<double*>(reinterpret_cast<uint8_t*>(call.workspace) + 2 * w.partial);
  const int64_t numel = rows * cols;
  int64_t blocks = (numel + 2047) / 2048;
  const int norm_blocks = (int)(blocks < NS_NORM_BLOCKS ? blocks : NS_NORM_BLOCKS);
  blocks = blocks < 1024 ? blocks : 1024;
  ns_begin_kernel<<<dim3(norm_blocks, (unsigned)batch), 256, 0, st>>>(e);
  ns_scale_kernel<<<dim3((unsigned)blocks, (unsigned)batch), 256, 0, st>>>(e, norm_blocks);

  if (cudaFuncSetAttribute(ns_product_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM) != cudaSuccess ||
      cudaFuncSetAttribute(ns_product_split_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM) != cudaSuccess ||
      cudaFuncSetAttribute(ns_product_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM) != cudaSuccess)
    return "orthogonalize: shared memory";

  // A pair's 256 x 256 tile needs half the operand traffic of a 128 x 128 one; with a side of 256 or less it would leave one
  // or two pairs to work on each matrix.
  const bool pair = k > 256 && !call.pairs;
  const int tile = pair ? 256 : 128;
  auto load_map = [&](CUtensorMap* m, const __half* p, int64_t r, int64_t c, int64_t ld, int64_t plane, bool mn) {
    return ns_map(m, p, batch, r, c, ld, plane, mn ? NS_BK : 128, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  auto store_map = [&](CUtensorMap* m, const __half* p, int64_t r, int64_t c, int64_t ld, int64_t plane) {
    return ns_map(m, p, batch, r, c, ld, plane, NS_BOX, NS_BOX, CU_TENSOR_MAP_SWIZZLE_64B);
  };
  const int kt = (k + tile - 1) / tile, wt = (int)(((tall ? rows : cols) + tile - 1) / tile);
  int cur = 0;
  for (int step = 0; step < call.steps; ++step) {
    __half* xin = x[cur];
    __half* xout = x[cur ^ 1];
    NsMaps m1, m2, m3;
    bool ok = true;
    // A = X X^T (wide: X rows are K-major; tall: A = X^T X, both operands MN-major)
    ok &= load_map(&m1.p_hi, xin, rows, cols, w.ld_x, w.plane_x, tall);
    ok &= load_map(&m1.p_lo, xin + lo_x, rows, cols, w.ld_x, w.plane_x, tall);
    m1.q_hi = m1.p_hi;
    m1.q_lo = m1.p_lo;
    ok &= store_map(&m1.out_hi, A, k, k, w.ld_k, w.plane_k);
    ok &= store_map(&m1.out_lo, A + lo_k, k, k, w.ld_k, w.plane_k);
    // B = b A + c A A^T
    ok &= load_map(&m2.p_hi, A, k, k, w.ld_k, w.plane_k, false);
    ok &= load_map(&m2.p_lo, A + lo_k, k, k, w.ld_k, w.plane_k, false);
    m2.q_hi = m2.p_hi;
    m2.q_lo = m2.p_lo;
    ok &= store_map(&m2.out_hi, B, k, k, w.ld_k, w.plane_k);
    ok &= store_map(&m2.out_lo, B + lo_k, k, k, w.ld_k, w.plane_k);
    // X' = a X + B X (wide: X is the MN-major second operand) or a X + X B^T (tall)
    CUtensorMap b_hi, b_lo;
    ok &= load_map(&b_hi, B, k, k, w.ld_k, w.plane_k, false);
    ok &= load_map(&b_lo, B + lo_k, k, k, w.ld_k, w.plane_k, false);
    CUtensorMap x_hi, x_lo;
    ok &= load_map(&x_hi, xin, rows, cols, w.ld_x, w.plane_x, !tall);
    ok &= load_map(&x_lo, xin + lo_x, rows, cols, w.ld_x, w.plane_x, !tall);
    m3.p_hi = tall ? x_hi : b_hi;
    m3.p_lo = tall ? x_lo : b_lo;
    m3.q_hi = tall ? b_hi : x_hi;
    m3.q_lo = tall ? b_lo : x_lo;
    ok &= store_map(&m3.out_hi, xout, rows, cols, w.ld_x, w.plane_x);
    ok &= store_map(&m3.out_lo, xout + lo_x, rows, cols, w.ld_x, w.plane_x);
    if (!ok) return "orthogonalize: cuTensorMapEncodeTiled failed";

    NsProduct g{};
    g.batch = (int)batch;
    g.pairs = call.pairs;
    g.M = g.N = k;
    g.K = (int)(tall ? rows : cols);
    g.symmetric = 1;
    g.p_mn = g.q_mn = tall;
    g.store_lo = call.pairs;
    g.acc_scale = NS_UNSCALE;
    g.tiles_m = kt;
    g.tiles = kt * (kt + 1) / 2;
    const char* err = ns_launch_product(m1, g, pair, sms, status, st);
    if (err) return err;
    g.K = k;
    g.p_mn = g.q_mn = 0;
    g.acc_scale = call.c[2] * NS_UNSCALE;
    g.aux_scale = call.c[1];
    g.aux_hi = A;
    g.aux_lo = call.pairs ? A + lo_k : nullptr;
    g.aux_ld = w.ld_k;
    g.aux_stride = w.plane_k;
    err = ns_launch_product(m2, g, pair, sms, status, st);
    if (err) return err;
    g.M = (int)rows;
    g.N = (int)cols;
    g.symmetric = 0;
    g.q_mn = !tall;
    g.store_lo = 1;
    g.acc_scale = NS_UNSCALE;
    g.aux_scale = call.c[0];
    g.aux_hi = xin;
    g.aux_lo = xin + lo_x;
    g.aux_ld = w.ld_x;
    g.aux_stride = w.plane_x;
    g.tiles_m = tall ? wt : kt;
    g.tiles = kt * wt;
    err = ns_launch_product(m3, g, pair, sms, status, st);
    if (err) return err;
    cur ^= 1;
  }
  e.x_hi = x[cur];
  e.x_lo = x[cur] + lo_x;
  ns_end_kernel<<<dim3((unsigned)blocks, (unsigned)batch), 256, 0, st>>>(e);
  return cudaGetLastError() == cudaSuccess ? nullptr : "orthogonalize launch failed";
}

}  // namespace gd
