// Orthogonalising matrices by Newton-Schulz products, and the momentum update built on it.
//
// For a batch of matrices X (r x c), each divided by its Frobenius norm, `steps` times
//
//     A = X X^T,   B = b A + c A^2,   X <- a X + B X          (r <= c; otherwise A = X^T X and X <- a X + X B)
//
// which moves every singular value s to s (a + b s^2 + c s^4) and keeps the singular vectors. Three products a step, the
// first two symmetric: only the tiles on and above the diagonal of A and B are computed and stored, and what lies below is
// read from above with the operand's other major order (a bit of the MMA instruction). A step then costs
// k (k + 1) w + k (k + 1) k + 2 k^2 w operations with k = min(r, c), w = max(r, c), against 4 k^2 w + 2 k^3.
//
// Matrices with a side of at most 256 (pairs: 128) stay in one cluster for the whole call (ns_small_kernel); larger ones go
// tile by tile through one persistent kernel (ns_chain_body) between element-wise ends. Few matrices are bound by the
// latency of 3 x steps dependent products (one 1024 x 1024: 0.16 ms), many by the tensor cores under the power cap and by the
// epilogue of X <- a X + B X, which reads and writes X twice over (48 of 1024 x 1024: 1.5 ms, 0.69 PFLOP/s of the
// operations above; four of 2048 x 4096: 1.3 ms, 0.92 PFLOP/s).
//
// Number format. Operands are fp16, scaled by 2^14: with the coefficients that the host admits the spectral norms of X, A
// and B, and so their entries, stay below 3.9, and 3.9 * 2^14 < 65504, so entries down to 2^-28 keep all 11 bits.
// X is held as hi + lo, two fp16 values (22 bits). With `pairs` off the products read the high parts only and the
// linear term a X reads both: rounding errors then enter through B X alone, in the directions whose singular values
// are already large (error of the result 5e-4 to 1.7e-3 of its norm, at most that of rounding it to bf16; without the
// low part in a X the noise of the large directions is amplified into the small ones, 3e-3 to 1e-1). With `pairs` on
// every operand is a pair and a product is the three partial products hi hi + hi lo + lo hi (the result is as exact
// as in fp32 arithmetic), at three times the tensor-core work and on single-CTA tiles, whose sums fit the registers. Sums are
// fp32 in TMEM; the norm is summed in fp64.
#include "orthogonalize.h"

#include <cuda_fp16.h>

#include <cstring>

#include "common.cuh"

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
// all products of a call in one kernel
// ---------------------------------------------------------------------------------------
// An item is one output tile of one product of one matrix. Items are handed out in order by a counter in memory, and an
// item waits only for items before it: the products of a matrix follow one another, and a count of the finished
// tiles per matrix says how far it is. So any number of resident blocks makes progress (two calls on two streams may share
// the GPU), nothing is launched between the 3 x steps products, and the tiles of one product fill the gaps that
// the end of another leaves. The order is: product by product, all matrices. (Windows of as many matrices as stay in L2 from
// one product to the next were slower: 48 matrices of 1024 x 1024 took 1.69 ms as one window, 2.07 in windows of 8, whose ends
// waited on one another.)
//
// A block: warp 10 fetches items, waits until what they read is written and hands them to the others; warp 0 loads operands
// with bulk tensor copies into a ring of stages; warp 1 issues the MMAs into two accumulators in TMEM; warps 2..9
// read the accumulator, add the linear term (its boxes are copied in while the MMAs run) and send 32 x 32 boxes
// out with bulk stores. A diagonal tile of a symmetric product reads the same rows twice and loads them once.
// PAIR: a pair of CTAs on two SMs shares a
// 256 x 256 tile, each loading its half of both operands; otherwise a CTA has a 128 x 128 tile of its own.
constexpr int NS_BK = 64;                       // K elements per stage: one 128-byte swizzle row
constexpr int NS_EPI_WARPS = 8;
constexpr int NS_THREADS = 96 + NS_EPI_WARPS * 32;
constexpr int NS_OPERAND_BYTES = 128 * 128;     // 128 rows x 64 fp16 per CTA and operand
constexpr int NS_BOX = 32;                      // epilogue chunk: 32 x 32
constexpr int NS_BOX_BYTES = NS_BOX * NS_BOX * 2;
constexpr int NS_SLOTS = 2;                     // chunks of the linear term in flight per epilogue warp
constexpr int NS_MAX_ACC = 4;
// Items on their way through a block: two are handed out ahead of the loads, which run at most the stages (4) ahead of the
// MMAs, these two accumulators ahead of the epilogue; a ring of 16 is never overwritten before it is read.
constexpr int NS_RING = 16;

template <bool SPLIT>
struct NsShape {
  static constexpr int PLANES = SPLIT ? 2 : 1;                                // hi, lo: a stage holds both of both operands
  static constexpr int STAGES = SPLIT ? 2 : 4;
  static constexpr int P_BYTES = PLANES * NS_OPERAND_BYTES;
  static constexpr int STAGE_BYTES = 2 * P_BYTES;
  static constexpr int ACC = SPLIT ? 4 : 2;                                   // accumulators in TMEM; with pairs they change hands more often
  static constexpr int AUX_BYTES = 2 * NS_BOX_BYTES;                          // hi and lo
  static constexpr int OUT_BYTES = 2 * NS_BOX_BYTES;
  static constexpr int WARP_BYTES = NS_SLOTS * AUX_BYTES + OUT_BYTES;
  static constexpr int SMEM = STAGES * STAGE_BYTES + NS_EPI_WARPS * WARP_BYTES + 1024 + 1024;   // barriers; alignment
};

struct __align__(16) NsBars {
  uint64_t full[4];
  uint64_t empty[4];
  uint64_t acc_full[NS_MAX_ACC];
  uint64_t acc_empty[NS_MAX_ACC];
  uint64_t aux_full[NS_EPI_WARPS * NS_SLOTS];
  uint64_t item_full[NS_RING];
  uint64_t taken[2];                 // the loads have begun item it (barrier it & 1)
  uint4 item[NS_RING];               // see NsItem::pack
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(NsBars) <= 1024, "barrier area");
constexpr int NS_MAPS = 24;                     // tensor maps at the start of NsPlan

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

// The same wait for a word that the other CTA of the pair wrote before it arrived (acquire at cluster scope).
__device__ __forceinline__ uint32_t ns_try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
// Without the time that a try_wait may be suspended for.
__device__ __forceinline__ uint32_t ns_test_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
__device__ __forceinline__ void ns_put_remote(uint32_t cluster_addr, uint4 v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void ns_arrive_remote(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

struct NsItem {
  int live;                          // 0: the list has ended
  int step, phase, z, mb, nb;        // phase 0: A, 1: B, 2: X
  __device__ __forceinline__ uint4 pack() const {
    return make_uint4((uint32_t)z, (uint32_t)(step | phase << 16), (uint32_t)mb, (uint32_t)nb | (uint32_t)live << 31);
  }
};

// Item `slot_no` of this block's list; not live at its end or when the wait ran out. Warp-collective.
__device__ __forceinline__ NsItem ns_next_item(NsBars* bars, int slot_no, Status* status) {
  const uint32_t bar = smem_u32(&bars->item_full[slot_no & (NS_RING - 1)]);
  const uint32_t parity = (slot_no / NS_RING) & 1;
  bool ok = false;
  if ((threadIdx.x & 31) == 0) {
    for (int i = 0; i < 256 && !ok; ++i) ok = ns_try_wait_cluster(bar, parity);
    if (!ok) {
      const uint64_t t0 = globaltimer_ns();
      while (!(ok = ns_try_wait_cluster(bar, parity))) {
        __nanosleep(32);
        if (ns_aborted(bars)) break;
        if (globaltimer_ns() - t0 > GD_WAIT_BUDGET_NS) {
          ns_abort(bars, status, STATUS_TIMEOUT_SMEM_FULL, 87, slot_no);
          break;
        }
      }
    }
  }
  ok = __shfl_sync(0xffffffffu, ok, 0);
  NsItem t;
  t.live = 0;
  if (!ok) return t;
  const volatile uint4* at = &bars->item[slot_no & (NS_RING - 1)];
  const uint32_t x = at->x, y = at->y, m = at->z, n = at->w;
  t.z = (int)x;
  t.step = (int)(y & 0xffffu);
  t.phase = (int)(y >> 16);
  t.mb = (int)m;
  t.nb = (int)(n & 0x7fffffffu);
  t.live = (int)(n >> 31);
  return t;
}

// Whether ns_next_item(slot_no) would return at once. Warp-collective.
__device__ __forceinline__ bool ns_item_there(NsBars* bars, int slot_no) {
  uint32_t ok = 0;
  if ((threadIdx.x & 31) == 0)
    ok = ns_test_wait_cluster(smem_u32(&bars->item_full[slot_no & (NS_RING - 1)]), (slot_no / NS_RING) & 1);
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// `need`: finished tiles of matrix z that this one reads (counted in epilogue warps)
__device__ __forceinline__ NsItem ns_decode(const NsPlan& g, int item, uint32_t warps_per_tile, uint32_t& need) {
  NsItem t;
  t.live = 1;
  const int per_step = 2 * g.tiles_sym + g.tiles_x;
  t.step = item / (g.batch * per_step);
  int r = item - t.step * g.batch * per_step;
  const int sym = g.batch * g.tiles_sym;
  int tiles = g.tiles_sym;
  t.phase = 0;
  if (r >= 2 * sym) { t.phase = 2; r -= 2 * sym; tiles = g.tiles_x; }
  else if (r >= sym) { t.phase = 1; r -= sym; }
  t.z = r / tiles;
  r -= t.z * tiles;
  need = (uint32_t)(t.step * per_step + t.phase * g.tiles_sym) * warps_per_tile;
  if (t.phase == 2) {
    t.nb = r / g.tiles_xm;           // neighbours share a column block
    t.mb = r - t.nb * g.tiles_xm;
  } else {
    int nb = 0;                      // column block nb holds the nb + 1 tiles on and above the diagonal
    while (r > nb) { r -= nb + 1; ++nb; }
    t.nb = nb;
    t.mb = r;
  }
  return t;
}

// 16-byte piece `slot` (0..3) of row `row` of a 32 x 64-byte box in the 64-byte swizzle order of the bulk copies
__device__ __forceinline__ uint32_t ns_box_off(int row, int slot) {
  return (uint32_t)(row * 64 + ((slot ^ ((row >> 1) & 3)) << 4));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

// This lane's row of a box, in registers <-> shared memory
__device__ __forceinline__ void ns_write_row(uint8_t* box, int lane, const uint32_t (&w)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<uint4*>(box + ns_box_off(lane, q)) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
}
__device__ __forceinline__ void ns_read_row(const uint8_t* box, int lane, uint32_t (&w)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint4 u = *reinterpret_cast<const uint4*>(box + ns_box_off(lane, q));
    w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w;
  }
}
// Whether K block kb (64 columns) of row block `block` of a symmetric factor lies below the diagonal, in tiles that are not
// stored: it is then read as the transpose of the tile above.
template <int TILE>
__device__ __forceinline__ bool ns_below(int kb, int block) { return kb * NS_BK / TILE < block; }

template <bool PAIR, bool SPLIT>
__device__ __forceinline__ void ns_chain_body(const NsPlan& g, Status* status) {
  constexpr int TILE = PAIR ? 256 : 128;
  constexpr int CHUNKS = TILE / 64;              // 32-column chunks per epilogue warp (two warps share a lane quarter)
  constexpr int STAGES = NsShape<SPLIT>::STAGES, ACC = NsShape<SPLIT>::ACC, PLANES = NsShape<SPLIT>::PLANES;
  constexpr int P_BYTES = NsShape<SPLIT>::P_BYTES, STAGE_BYTES = NsShape<SPLIT>::STAGE_BYTES;
  constexpr uint32_t WARPS_PER_TILE = (PAIR ? 2 : 1) * NS_EPI_WARPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* boxes = smem + STAGES * STAGE_BYTES;
  NsBars* bars = reinterpret_cast<NsBars*>(boxes + NS_EPI_WARPS * NsShape<SPLIT>::WARP_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&bars->full[s]), 1);
      mbar_init(smem_u32(&bars->empty[s]), 1);
    }
    for (int a = 0; a < ACC; ++a) {
      mbar_init(smem_u32(&bars->acc_full[a]), 1);
      mbar_init(smem_u32(&bars->acc_empty[a]), WARPS_PER_TILE);
    }
    for (int a = 0; a < NS_EPI_WARPS * NS_SLOTS; ++a) mbar_init(smem_u32(&bars->aux_full[a]), 1);
    for (int a = 0; a < NS_RING; ++a) mbar_init(smem_u32(&bars->item_full[a]), 1);
    for (int a = 0; a < 2; ++a) mbar_init(smem_u32(&bars->taken[a]), 1);
    bars->abort = 0;
    fence_barrier_init();
  }
  // the tensor maps of the first items are fetched while the block starts
  if (warp >= 2) {
    const CUtensorMap* maps = &g.x_gram[0][0];
    for (int i = (warp - 2) * 32 + lane; i < (int)(NS_MAPS); i += (NS_THREADS - 64)) tma_prefetch_desc(maps + i);
  }
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(smem_u32(&bars->tmem_base), ACC * TILE); tmem_relinquish_pair(); }
    else { tmem_alloc(smem_u32(&bars->tmem_base), ACC * TILE); tmem_relinquish(); }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  tc_fence_after_sync();
  pdl_enter();
  const uint32_t tmem_base = bars->tmem_base;

  const int kb_x = (g.wide + NS_BK - 1) / NS_BK, kb_k = (g.k + NS_BK - 1) / NS_BK;   // K blocks of product A; of B and X
  const uint32_t smem0 = smem_u32(smem);
  const uint32_t full0 = smem_u32(&bars->full[0]), empty0 = smem_u32(&bars->empty[0]);
  const uint32_t afull0 = smem_u32(&bars->acc_full[0]), aempty0 = smem_u32(&bars->acc_empty[0]);

  if (warp == 0) {
    const uint32_t full_lead0 = PAIR ? map_to_cta(full0, 0) : full0;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const NsItem t = ns_next_item(bars, it, status);
      if (!t.live) break;
      if (rank == 0 && lane == 0) mbar_arrive(smem_u32(&bars->taken[it & 1]));
      fence_proxy_async_global();      // what other blocks wrote before they counted up is read by bulk copies below
      const int cur = t.step & 1;
      const int m0 = t.mb * TILE + (int)rank * 128, n0 = t.nb * TILE + (int)rank * 128;
      const int kblocks = t.phase == 0 ? kb_x : kb_k;
      const bool once = t.phase != 2 && t.mb == t.nb;      // both operands are the same rows
      // the symmetric factor (A, or B) [plane][major order] and, but for B = b A + c A A, the X operand [plane]
      const CUtensorMap (*f)[2] = t.phase == 1 ? g.a_load : g.b_load;
      const CUtensorMap* x = t.phase == 0 ? g.x_gram[cur] : g.x_apply[cur];
      for (int kb = 0, kx = 0; kb < kblocks; ++kb, kx += NS_BK) {
        if (!__all_sync(0xffffffffu, ns_wait(empty0 + 8 * s, ph ^ 1))) {
          if (lane == 0) ns_abort(bars, status, STATUS_TIMEOUT_SMEM_EMPTY, 80, s);
          ok = false;
          break;
        }
        const uint32_t full = full_lead0 + 8 * s;
        const uint32_t p_dst = smem0 + s * STAGE_BYTES, q_dst = p_dst + P_BYTES;
        if (elect_one()) {
          if (!PAIR || rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, (PAIR ? 2 : 1) * (once ? P_BYTES : STAGE_BYTES));
          auto load = [&](uint32_t dst, const CUtensorMap* m, bool mn, int row) {      // rows row .. row + 127, this K block
            auto copy = [&](uint32_t d, int x, int y) {
              if (PAIR) tma_load_3d_pair(d, m, full, x, y, t.z);
              else tma_load_3d(d, m, full, x, y, t.z);
            };
            if (!mn) {
              copy(dst, kx, row);
            } else {
#pragma unroll
              for (int i = 0; i < 2; ++i) copy(dst + i * (NS_BK * 128), row + i * 64, kx);
            }
          };
          auto factor = [&](uint32_t dst, int block, int row) {
            const bool mn = ns_below<TILE>(kb, block);
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl) load(dst + pl * NS_OPERAND_BYTES, &f[pl][mn], mn, row);
          };
          auto x_rows = [&](uint32_t dst, bool mn, int row) {
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl) load(dst + pl * NS_OPERAND_BYTES, &x[pl], mn, row);
          };
          if (t.phase == 0) {
            x_rows(p_dst, g.tall, m0);
            if (!once) x_rows(q_dst, g.tall, n0);
          } else if (t.phase == 1) {
            factor(p_dst, t.mb, m0);
            if (!once) factor(q_dst, t.nb, n0);
          } else if (g.tall) {
            x_rows(p_dst, false, m0);
            factor(q_dst, t.nb, n0);
          } else {
            factor(p_dst, t.mb, m0);
            x_rows(q_dst, true, n0);
          }
        }
        __syncwarp();
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      int s = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const NsItem t = ns_next_item(bars, it, status);
        if (!t.live) break;
        const int kblocks = t.phase == 0 ? kb_x : kb_k;
        const bool diagonal = t.phase != 2 && t.mb == t.nb;
        // An operand is MN-major for its first K blocks: X all the way or not at all, a symmetric factor up to the diagonal.
        constexpr int ALL = 0x7fffffff, PER_TILE = TILE / NS_BK;
        const int p_mn_until = t.phase == 0 ? (g.tall ? ALL : 0) : (t.phase == 2 && g.tall ? 0 : t.mb * PER_TILE);
        const int q_mn_until = t.phase == 0 ? (g.tall ? ALL : 0) : (t.phase == 2 && !g.tall ? ALL : t.nb * PER_TILE);
        const uint64_t k_tmpl = make_smem_desc(smem0, 16, 1024), mn_tmpl = make_smem_desc(smem0, NS_BK * 128, 1024);
        // K blocks that one accumulator takes: all of them, or, with pairs, one, for the sum to stay as exact as fp32
        const int per_acc = SPLIT ? 1 : kblocks;
        for (int b0 = 0; b0 < kblocks && ok; b0 += per_acc) {
          if (!__all_sync(0xffffffffu, ns_wait(aempty0 + 8 * acc, acc_ph ^ 1))) {
            if (lane == 0) ns_abort(bars, status, STATUS_TIMEOUT_TMEM_EMPTY, 81, acc);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + acc * TILE;
          const int count = min(per_acc, kblocks - b0);
          uint32_t accumulate = 0;
          for (int i = 0; i < count; ++i) {
            if (!__all_sync(0xffffffffu, ns_wait(full0 + 8 * s, ph))) {
              if (lane == 0) ns_abort(bars, status, STATUS_TIMEOUT_SMEM_FULL, 82, s);
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const bool p_mn = b0 + i < p_mn_until, q_mn = b0 + i < q_mn_until;
            const uint32_t idesc = make_instr_desc(0, 0, 0, 0, TILE, TILE) | (p_mn ? 1u << 15 : 0u) | (q_mn ? 1u << 16 : 0u);
            const uint32_t p_step = p_mn ? (16 * 128) >> 4 : 2, q_step = q_mn ? (16 * 128) >> 4 : 2;
            const uint32_t d_hi = (uint32_t)(k_tmpl >> 32);                       // the strides that differ are in the low word
            const uint32_t p_lo = (uint32_t)(p_mn ? mn_tmpl : k_tmpl) + s * (STAGE_BYTES >> 4);
            const uint32_t q_lo = (uint32_t)(q_mn ? mn_tmpl : k_tmpl) + s * (STAGE_BYTES >> 4) + (diagonal ? 0 : P_BYTES >> 4);
            if (elect_one()) {
#pragma unroll
              for (int part = SPLIT ? 0 : 2; part < 3; ++part) {                 // hi lo, lo hi, hi hi
                const uint32_t p_at = p_lo + (part == 1 ? NS_OPERAND_BYTES >> 4 : 0), q_at = q_lo + (part == 0 ? NS_OPERAND_BYTES >> 4 : 0);
#pragma unroll
                for (int k = 0; k < NS_BK / 16; ++k) {
                  const uint64_t dp = ns_desc(d_hi, p_at + k * p_step), dq = ns_desc(d_hi, q_at + k * q_step);
                  const uint32_t on = k == 0 && part == (SPLIT ? 0 : 2) ? accumulate : 1u;
                  if (PAIR) mma_bf16_pair(d_tmem, dp, dq, idesc, on);      // kind::f16; idesc says fp16
                  else mma_bf16(d_tmem, dp, dq, idesc, on);
                }
              }
              if (PAIR) mma_commit_pair(empty0 + 8 * s);
              else mma_commit(empty0 + 8 * s);
            }
            __syncwarp();
            accumulate = 1;
            if (++s == STAGES) { s = 0; ph ^= 1; }
          }
          if (!ok || ns_aborted(bars)) { ok = false; break; }
          if (elect_one()) {
            if (PAIR) mma_commit_pair(afull0 + 8 * acc);
            else mma_commit(afull0 + 8 * acc);
          }
          __syncwarp();
          if (++acc == ACC) { acc = 0; acc_ph ^= 1; }
        }
      }
    }
  } else if (warp == 2 + NS_EPI_WARPS) {
    if (rank == 0) {
      const uint32_t peer_item0 = PAIR ? map_to_cta(smem_u32(&bars->item[0]), 1) : 0;
      const uint32_t peer_bar0 = PAIR ? map_to_cta(smem_u32(&bars->item_full[0]), 1) : 0;
      if (lane == 0) {
        int ahead = (int)atomicAdd(g.next_item, 1u);
        NsItem t{};
        for (int it = 0;; ++it) {
          t.live = 0;
          if (ahead < g.items) {
            uint32_t need;
            t = ns_decode(g, ahead, WARPS_PER_TILE, need);
            ahead = (int)atomicAdd(g.next_item, 1u);      // needed one item later
            if (need != 0 && !wait_flag_ge_gpu(g.done + t.z, need, GD_WAIT_BUDGET_NS)) {
              ns_abort(bars, status, STATUS_TIMEOUT_PEER_FLAG, 84, t.z);
              t.live = 0;
            }
            if (it >= 2 && !ns_wait(smem_u32(&bars->taken[it & 1]), ((it >> 1) - 1) & 1)) {
              if (!ns_aborted(bars)) ns_abort(bars, status, STATUS_TIMEOUT_SMEM_EMPTY, 85, it);
              t.live = 0;
            }
            if (ns_aborted(bars)) t.live = 0;
          }
          const int slot = it & (NS_RING - 1);
          const uint4 w = t.pack();
          bars->item[slot] = w;
          mbar_arrive(smem_u32(&bars->item_full[slot]));
          if (PAIR) {
            ns_put_remote(peer_item0 + 16 * slot, w);
            ns_arrive_remote(peer_bar0 + 8 * slot);
          }
          if (!t.live) break;
        }
      }
      __syncwarp();
    }
  } else {
    const int ew = warp - 2;
    uint8_t* aux_slots = boxes + ew * NsShape<SPLIT>::WARP_BYTES;
    uint8_t* out_box = aux_slots + NS_SLOTS * NsShape<SPLIT>::AUX_BYTES;
    const uint32_t aux_bar0 = smem_u32(&bars->aux_full[ew * NS_SLOTS]);
    const int quarter = warp & 3, half = ew >> 2;
    const uint32_t aempty_lead0 = PAIR ? map_to_cta(aempty0, 0) : aempty0;
    int acc = 0;
    uint32_t acc_ph = 0, aux_ph = 0;             // aux_ph: bit s = phase of slot s
    bool ok = true;

    NsItem t{};
    int m_warp, n_half, chunks;                  // this warp's corner of the tile; chunks that hold anything of the matrix
    auto corner = [&]() {
      const int M = t.phase == 2 ? g.rows : g.k, N = t.phase == 2 ? g.cols : g.k;
      m_warp = t.mb * TILE + (int)rank * 128 + quarter * 32;
      n_half = t.nb * TILE + half * (TILE / 2);
      chunks = m_warp < M ? max(0, min(CHUNKS, (N - n_half + 31) / 32)) : 0;
    };
    // chunk c of the linear term (the old X, or A) into its slot, which every lane has finished reading
    auto aux_request = [&](int c) {
      if (elect_one()) {
        const CUtensorMap* aux = t.phase == 1 ? g.a_box : g.x_box[t.step & 1];
        const bool lo = SPLIT || t.phase == 2;
        const int sl = c & (NS_SLOTS - 1);
        const uint32_t bar = aux_bar0 + 8 * sl, dst = smem_u32(aux_slots) + sl * NsShape<SPLIT>::AUX_BYTES;
        mbar_arrive_expect_tx(bar, (lo ? 2 : 1) * NS_BOX_BYTES);
        tma_load_3d(dst, &aux[0], bar, n_half + c * 32, m_warp, t.z);
        if (lo) tma_load_3d(dst + NS_BOX_BYTES, &aux[1], bar, n_half + c * 32, m_warp, t.z);
      }
      __syncwarp();
    };
    // This warp's part of a tile of matrix z is written: count it. `behind`: stores of a later tile may still be on their way.
    int uncounted = -1;
    auto count_tile = [&](int z, bool behind) {
      if (elect_one()) {
        if (behind) bulk_wait_but_one();
        else bulk_wait_all();
        fence_proxy_async_global();
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(g.done + z) : "memory");
      }
      __syncwarp();
    };
    auto aux_begin = [&]() {
      if (t.phase == 0) return;
      fence_proxy_async_global();      // the item was handed out after what it reads was written
      for (int c = 0; c < min(chunks, NS_SLOTS); ++c) aux_request(c);
    };

    t = ns_next_item(bars, 0, status);
    if (t.live) {
      corner();
      aux_begin();
    }
    for (int it = 0; t.live && ok; ++it) {
      const CUtensorMap* out = t.phase == 0 ? g.a_box : (t.phase == 1 ? g.b_box : g.x_box[(t.step & 1) ^ 1]);
      const bool with_lo = SPLIT || t.phase == 2;
      const float aux_scale = t.phase == 1 ? g.b : g.a, acc_scale = (t.phase == 1 ? g.c : 1.0f) * NS_UNSCALE;
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
        if (++acc == ACC) { acc = 0; acc_ph ^= 1; }
      };
      auto acc_row = [&]() { return tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * TILE + half * (TILE / 2); };

      // one 32 x 32 chunk: linear term, result as hi + lo, out. `ready` waits for the accumulator values in `raw`
      auto do_chunk = [&](int c, uint32_t (&raw)[32], auto ready) {
        float v[32];
        if (t.phase != 0) {
          const int sl = c & (NS_SLOTS - 1);
          if (!mbar_wait_warp(aux_bar0 + 8 * sl, (aux_ph >> sl) & 1)) {
            ns_abort(bars, status, STATUS_TIMEOUT_SMEM_FULL, 86, ew);
            ok = false;
            return;
          }
          aux_ph ^= 1u << sl;
          const uint8_t* slot = aux_slots + sl * NsShape<SPLIT>::AUX_BYTES;
          uint32_t w[16];
          ns_read_row(slot, lane, w);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 f = unpack_half2(w[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
          }
          if (with_lo) {
            ns_read_row(slot + NS_BOX_BYTES, lane, w);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 f = unpack_half2(w[i]);
              v[2 * i] += f.x; v[2 * i + 1] += f.y;
            }
          }
          __syncwarp();
          if (c + NS_SLOTS < chunks) aux_request(c + NS_SLOTS);
          ready();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = fmaf(aux_scale, v[j], acc_scale * __uint_as_float(raw[j]));
        } else {
          ready();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = acc_scale * __uint_as_float(raw[j]);
        }
        uint32_t hi[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) hi[i] = pack_half2(v[2 * i], v[2 * i + 1]);
        if (elect_one()) bulk_wait_read_all();      // the stores of the chunk before have left the boxes
        __syncwarp();
        ns_write_row(out_box, lane, hi);
        if (with_lo) {
          uint32_t lo[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 h = unpack_half2(hi[i]);
            lo[i] = pack_half2(v[2 * i] - h.x, v[2 * i + 1] - h.y);
          }
          ns_write_row(out_box + NS_BOX_BYTES, lane, lo);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one()) {
          const int n0 = n_half + c * 32;
          tma_store_3d(&out[0], smem_u32(out_box), n0, m_warp, t.z);
          if (with_lo) tma_store_3d(&out[1], smem_u32(out_box + NS_BOX_BYTES), n0, m_warp, t.z);
          bulk_commit_group();
        }
        __syncwarp();
        if (uncounted >= 0) {
          count_tile(uncounted, true);
          uncounted = -1;
        }
      };

      if constexpr (SPLIT) {
        // Pairs: the tensor core cuts a running sum where fp32 rounds it, an error of one sign that grows with the number of
        // additions, so after every K block the sum moves to registers and is continued there.
        float sum[CHUNKS][32];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[c][j] = 0.0f;
        const int kblocks = t.phase == 0 ? kb_x : kb_k;
        for (int b0 = 0; b0 < kblocks && ok; ++b0) {
          if (!(ok = acc_wait())) break;
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            uint32_t raw[32];
            tmem_ld_32x32(acc_row() + c * 32, raw);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[c][j] += __uint_as_float(raw[j]);
          }
          acc_release();
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          if (c >= chunks || !ok) continue;
          uint32_t raw[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) raw[j] = __float_as_uint(sum[c][j]);
          do_chunk(c, raw, []() {});
        }
      } else {
        if (!(ok = acc_wait())) break;
        if (chunks == 0) acc_release();
        // two register buffers: the accumulator's next chunk is on its way while this one is worked on
        uint32_t raw0[32], raw1[32];
        if (chunks > 0) tmem_ld_32x32(acc_row(), raw0);
#pragma unroll 1
        for (int c = 0; c < chunks && ok; c += 2) {
          do_chunk(c, raw0, [&]() {
            tmem_ld_wait();
            if (c + 1 < chunks) tmem_ld_32x32(acc_row() + (c + 1) * 32, raw1);
            else acc_release();
          });
          if (c + 1 >= chunks || !ok) break;
          do_chunk(c + 1, raw1, [&]() {
            tmem_ld_wait();
            if (c + 2 < chunks) tmem_ld_32x32(acc_row() + (c + 2) * 32, raw0);
            else acc_release();
          });
        }
      }
      if (!ok) break;
      // The next item's linear term can be asked for before this one's stores are complete, but an item that is not handed out
      // yet cannot be waited for: what it reads may depend on the count below. If the next item is there and its
      // accumulator too, this tile is counted after the next one's first chunk, when its stores have long completed.
      const int z_done = t.z;
      bool there = ns_item_there(bars, it + 1), busy = false;
      if (there) {
        t = ns_next_item(bars, it + 1, status);
        if (t.live) {
          corner();
          aux_begin();
          busy = chunks > 0 && __shfl_sync(0xffffffffu, lane == 0 ? mbar_test_wait(afull0 + 8 * acc, acc_ph) : 0u, 0) != 0;
        }
      }
      if (busy) uncounted = z_done;
      else count_tile(z_done, false);
      if (!there) {
        t = ns_next_item(bars, it + 1, status);
        if (t.live) {
          corner();
          aux_begin();
        }
      }
    }
    if (elect_one()) bulk_wait_all();
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
    if (PAIR) tmem_dealloc_pair(tmem_base, ACC * TILE);
    else tmem_dealloc(tmem_base, ACC * TILE);
  }
}

__global__ void __launch_bounds__(NS_THREADS, 1)
ns_chain_kernel(const __grid_constant__ NsPlan g, Status* status) {
  ns_chain_body<false, false>(g, status);
}

__global__ void __launch_bounds__(NS_THREADS, 1)
ns_chain_split_kernel(const __grid_constant__ NsPlan g, Status* status) {
  ns_chain_body<false, true>(g, status);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NS_THREADS, 1)
ns_chain_pair_kernel(const __grid_constant__ NsPlan g, Status* status) {
  ns_chain_body<true, false>(g, status);
}

// ---------------------------------------------------------------------------------------
// element-wise ends: momentum, norm, scaling into the operand format, result
// ---------------------------------------------------------------------------------------
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

// Rows are covered by 2^tpr_log2 threads in steps of V elements, so no index is divided; a block takes ENDS_ROWS rows per
// thread group at a time, whose loads are in flight together.
constexpr int ENDS_THREADS = 256;
constexpr int ENDS_ROWS = 4;

template <int V>
struct alignas(V < 4 ? V * 4 : 16) VecF { float e[V]; };
template <int V>
struct alignas(V * 2) VecH { uint16_t e[V]; };

template <int V>
__device__ __forceinline__ VecF<V> load_vec(const void* p, int dtype, int64_t i) {
  VecF<V> v;
  if (dtype == ELEM_F32) return *reinterpret_cast<const VecF<V>*>(reinterpret_cast<const float*>(p) + i);
  const VecH<V> h = *reinterpret_cast<const VecH<V>*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
  for (int q = 0; q < V; ++q)
    v.e[q] = dtype == ELEM_BF16 ? __uint_as_float((uint32_t)h.e[q] << 16) : __half2float(__ushort_as_half(h.e[q]));
  return v;
}
template <int V>
__device__ __forceinline__ void store_vec(void* p, int dtype, int64_t i, const VecF<V>& v) {
  if (dtype == ELEM_F32) {
    *reinterpret_cast<VecF<V>*>(reinterpret_cast<float*>(p) + i) = v;
    return;
  }
  VecH<V> h;
#pragma unroll
  for (int q = 0; q < V; ++q)
    h.e[q] = dtype == ELEM_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v.e[q])) : __half_as_ushort(__float2half_rn(v.e[q]));
  *reinterpret_cast<VecH<V>*>(reinterpret_cast<uint16_t*>(p) + i) = h;
}

// Sum of squares without overflow or underflow: fp32 where the largest of the values allows it, fp64 otherwise.
template <int V>
__device__ __forceinline__ void add_squares(double& ssq, const VecF<V>& u) {
  float top = 0.0f, s = 0.0f;
#pragma unroll
  for (int q = 0; q < V; ++q) {
    top = fmaxf(top, fabsf(u.e[q]));
    s = fmaf(u.e[q], u.e[q], s);
  }
  if (top > 1e-16f && top < 1e18f) {
    ssq += (double)s;
  } else {
#pragma unroll
    for (int q = 0; q < V; ++q) ssq += (double)u.e[q] * (double)u.e[q];
  }
}

// u: the gradient, in place the matrix to orthogonalise; f: information gradient; m: momentum, updated
//   g = scalars[1] * ((1 - beta * scalars[0]) * gt + beta * gi);   m <- mu m + g;   u = nesterov ? g + mu m : m
template <int V>
__device__ __forceinline__ void momentum_step(const NsEnds& e, float kt, float ki, bool info, VecF<V>& u, const VecF<V>& f, VecF<V>& m) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float x = u.e[i];
    if (e.scalars != nullptr) {
      x *= kt;
      if (info) x = fmaf(ki, f.e[i], x);
    }
    m.e[i] = fmaf(e.mu, m.e[i], x);
    u.e[i] = e.nesterov ? fmaf(e.mu, m.e[i], x) : m.e[i];
  }
}

// u (fp32, row pitch ld) of every matrix and the blocks' partial sums of u^2. Without momentum u is the input itself.
// (MOMENTUM is a parameter of the code because the loads of its inputs cost registers, and those cost blocks per SM.)
template <int V, bool MOMENTUM>
__global__ void __launch_bounds__(ENDS_THREADS)
ns_begin_kernel(const __grid_constant__ NsEnds e) {
  __shared__ double red[ENDS_THREADS / 32];
  const int z = blockIdx.y;
  const int group = threadIdx.x >> e.tpr_log2, groups = ENDS_THREADS >> e.tpr_log2;
  const int c0 = (threadIdx.x & ((1 << e.tpr_log2) - 1)) * V;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    e.done[z] = 0;
    if (z == 0) *e.next_item = 0;
  }
  float kt = 1.0f, ki = 0.0f;
  if (e.scalars != nullptr) {
    kt = (1.0f - e.beta * e.scalars[0]) * e.scalars[1];
    ki = e.beta * e.scalars[1];
  }
  const void* gt = e.grad[z];
  const void* gi = e.info[z];
  float* mom = reinterpret_cast<float*>(e.moment[z]);
  float* up = e.u + (int64_t)z * e.plane;
  double ssq = 0.0;
  for (int r0 = blockIdx.x * groups * ENDS_ROWS; r0 < e.rows; r0 += gridDim.x * groups * ENDS_ROWS) {
    for (int c = c0; c < e.cols; c += V << e.tpr_log2) {
      VecF<V> g[ENDS_ROWS], f[ENDS_ROWS], m[ENDS_ROWS];
#pragma unroll
      for (int q = 0; q < ENDS_ROWS; ++q) {
        const int r = r0 + q * groups + group;
        if (r >= e.rows) continue;
        g[q] = load_vec<V>(gt, e.grad_dtype, (int64_t)r * e.grad_ld + c);
        if (MOMENTUM) {
          m[q] = *reinterpret_cast<const VecF<V>*>(mom + (int64_t)r * e.cols + c);
          if (gi != nullptr) f[q] = load_vec<V>(gi, e.grad_dtype, (int64_t)r * e.grad_ld + c);
        }
      }
#pragma unroll
      for (int q = 0; q < ENDS_ROWS; ++q) {
        const int r = r0 + q * groups + group;
        if (r >= e.rows) continue;
        VecF<V> u = g[q];
        if (MOMENTUM) {
          momentum_step<V>(e, kt, ki, gi != nullptr, u, f[q], m[q]);
          *reinterpret_cast<VecF<V>*>(mom + (int64_t)r * e.cols + c) = m[q];
        }
        *reinterpret_cast<VecF<V>*>(up + (int64_t)r * e.ld + c) = u;
        add_squares<V>(ssq, u);
      }
    }
  }
  const double s = block_sum(ssq, red);
  if (threadIdx.x == 0) e.partial[(int64_t)z * gridDim.x + blockIdx.x] = s;
}

// u / (norm + eps) * 2^14 as hi + lo
template <int V>
__global__ void __launch_bounds__(ENDS_THREADS)
ns_scale_kernel(const __grid_constant__ NsEnds e, int n_partial) {
  const int z = blockIdx.y;
  const int group = threadIdx.x >> e.tpr_log2, groups = ENDS_THREADS >> e.tpr_log2;
  const int c0 = (threadIdx.x & ((1 << e.tpr_log2) - 1)) * V;
  double s = 0.0;
  for (int i = threadIdx.x & 31; i < n_partial; i += 32) s += e.partial[(int64_t)z * n_partial + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const double inv = (double)NS_SCALE / (sqrt(s) + (double)e.eps);
  const float finv = (float)inv;
  const bool fine = finv > 1e-30f && finv < 1e30f;      // else the factor itself does not fit fp32
  const float* up = e.u + (int64_t)z * e.plane;
  __half* hi = e.x_hi + (int64_t)z * e.plane;
  __half* lo = e.x_lo + (int64_t)z * e.plane;
  for (int r0 = blockIdx.x * groups * ENDS_ROWS; r0 < e.rows; r0 += gridDim.x * groups * ENDS_ROWS) {
    for (int c = c0; c < e.cols; c += V << e.tpr_log2) {
      VecF<V> u[ENDS_ROWS];
#pragma unroll
      for (int q = 0; q < ENDS_ROWS; ++q) {
        const int r = r0 + q * groups + group;
        if (r < e.rows) u[q] = *reinterpret_cast<const VecF<V>*>(up + (int64_t)r * e.ld + c);
      }
#pragma unroll
      for (int q = 0; q < ENDS_ROWS; ++q) {
        const int r = r0 + q * groups + group;
        if (r >= e.rows) continue;
        VecH<V> h, l;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float v = fine ? u[q].e[i] * finv : (float)((double)u[q].e[i] * inv);
          const __half a = __float2half_rn(v);
          h.e[i] = __half_as_ushort(a);
          l.e[i] = __half_as_ushort(__float2half_rn(v - __half2float(a)));
        }
        *reinterpret_cast<VecH<V>*>(hi + (int64_t)r * e.ld + c) = h;
        *reinterpret_cast<VecH<V>*>(lo + (int64_t)r * e.ld + c) = l;
      }
    }
  }
}

// the result, or the parameter update p <- p * decay - step * x
template <int V>
__global__ void __launch_bounds__(ENDS_THREADS)
ns_end_kernel(const __grid_constant__ NsEnds e) {
  const int z = blockIdx.y;
  const int group = threadIdx.x >> e.tpr_log2, groups = ENDS_THREADS >> e.tpr_log2;
  const int c0 = (threadIdx.x & ((1 << e.tpr_log2) - 1)) * V;
  const __half* hi = e.x_hi + (int64_t)z * e.plane;
  const __half* lo = e.x_lo + (int64_t)z * e.plane;
  void* out = e.out[z];
  for (int r0 = blockIdx.x * groups * ENDS_ROWS; r0 < e.rows; r0 += gridDim.x * groups * ENDS_ROWS) {
    for (int c = c0; c < e.cols; c += V << e.tpr_log2) {
      VecF<V> p[ENDS_ROWS];
      VecH<V> h[ENDS_ROWS], l[ENDS_ROWS];
#pragma unroll
      for (int q = 0; q < ENDS_ROWS; ++q) {
        const int r = r0 + q * groups + group;
        if (r >= e.rows) continue;
        h[q] = *reinterpret_cast<const VecH<V>*>(hi + (int64_t)r * e.ld + c);
        l[q] = *reinterpret_cast<const VecH<V>*>(lo + (int64_t)r * e.ld + c);
        if (e.momentum) p[q] = load_vec<V>(out, e.out_dtype, (int64_t)r * e.cols + c);
      }
#pragma unroll
      for (int q = 0; q < ENDS_ROWS; ++q) {
        const int r = r0 + q * groups + group;
        if (r >= e.rows) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float x = (__half2float(__ushort_as_half(h[q].e[i])) + __half2float(__ushort_as_half(l[q].e[i]))) * NS_UNSCALE;
          p[q].e[i] = e.momentum ? fmaf(-e.step, x, p[q].e[i] * e.decay) : x;
        }
        store_vec<V>(out, e.out_dtype, (int64_t)r * e.cols + c, p[q]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// matrices with a side of at most 256: a whole call in one kernel
// ---------------------------------------------------------------------------------------
// One cluster per matrix; each of its 1 to 16 CTAs keeps a slice of the long side (64 n columns of X, RB blocks of 128 rows) for the
// whole call:
// the fp32 X in TMEM, its fp16 operands in shared memory. A tile of X lies as k rows of 128-byte pieces, which is the K-major
// operand of A = X X^T and, read as rows of the reduction, the MN-major operand of B X. X in TMEM is stored times a, so that
// the MMAs of B X add to the linear term in place (with pairs B X has columns of its own and is added in registers: the
// tensor core cuts a sum where fp32 rounds it, and a X is several times the result).
// The slices' shares of A are summed through distributed shared memory:
// every CTA adds up some of the rows, in the order of the CTAs, and hands them to all. What bounds this kernel is the chain of
// 3 x steps products with an exchange of operands between them (128 x 256: 35 us a call, 4 us a step; 256 x 256: 98 us, 17 us
// a step, most of it the exchange of A), not work or traffic; as tiles handed out by ns_chain_body one 128 x 512 matrix
// took 111 us instead of 50.
constexpr int SM_THREADS = 512;                      // 16 warps: four share the rows of a lane quarter and split its columns
constexpr int SM_PANEL = 128 * 128;                 // 128 rows x 64 fp16

template <int RB, bool SPLIT>
struct SmShape {
  static constexpr int SLICE = RB == 2 ? 64 : (SPLIT ? 128 : 256);   // columns a CTA holds at most
  static constexpr int PLANES = SPLIT ? 2 : 1;                       // hi, lo
  static constexpr int BLOCKS = RB * (RB + 1) / 2;                   // 128 x 128 blocks of A and B on and above the diagonal
  static constexpr int X_BYTES = RB * SLICE / 64 * SM_PANEL;         // one plane of X
  static constexpr int F_BYTES = 2 * SM_PANEL;                       // one plane of a block of A or B
  static constexpr int PART_BYTES = 128 * 128 * 4;                   // this CTA's share of a block of A in fp32
  // The shares lie where B does, which is not in use between B X and the next B (one block of B alone is too small for them).
  static constexpr bool PART_IN_B = PLANES * BLOCKS * F_BYTES >= PART_BYTES;
  static constexpr int SMEM = PLANES * (X_BYTES + 2 * BLOCKS * F_BYTES) + (PART_IN_B ? 0 : PART_BYTES) + 1024;
  static constexpr int X_COL = 0, ACC_COL = RB * SLICE;              // TMEM columns
  static constexpr int BX_COL = SPLIT ? SLICE + 128 : X_COL;
  static constexpr int TMEM_COLS = 512;
};
static_assert(SmShape<2, false>::ACC_COL + 128 * SmShape<2, false>::BLOCKS <= 512 && SmShape<2, false>::SMEM <= 231424, "two row blocks");

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float4 ld_dsmem_f4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(map_to_cta(addr, rank))
               : "memory");
  return v;
}
__device__ __forceinline__ double ld_dsmem_f64(uint32_t addr, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(map_to_cta(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void st_dsmem_u2(uint32_t addr, uint32_t rank, uint2 v) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(map_to_cta(addr, rank)), "r"(v.x), "r"(v.y) : "memory");
}

// byte of (row, 16-byte piece) in a panel: 128-byte rows, pieces XOR-ed with the row
__device__ __forceinline__ int sm_piece(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

// 32 values of row `row`, columns col .. col + 31 of an operand, as hi (and lo, `plane` bytes further)
template <bool SPLIT>
__device__ __forceinline__ void sm_put_operand(uint8_t* base, int plane, int row, int col, const float (&v)[32]) {
  uint8_t* panel = base + (col >> 6) * SM_PANEL;
  const int piece0 = (col & 63) >> 3;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = pack_half2(v[8 * q + 2 * i], v[8 * q + 2 * i + 1]);
      if (SPLIT) {
        const float2 h = unpack_half2(hi[i]);
        lo[i] = pack_half2(v[8 * q + 2 * i] - h.x, v[8 * q + 2 * i + 1] - h.y);
      }
    }
    *reinterpret_cast<uint4*>(panel + sm_piece(row, piece0 + q)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (SPLIT) *reinterpret_cast<uint4*>(panel + plane + sm_piece(row, piece0 + q)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// V elements an access (neighbouring along the memory's rows). RB: blocks of 128 rows (1 or 2).
template <int RB, bool SPLIT, int V>
__global__ void __launch_bounds__(SM_THREADS, 1)
ns_small_kernel(const __grid_constant__ NsEnds e, const __grid_constant__ NsSmall g, Status* status) {
  using S = SmShape<RB, SPLIT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  __shared__ double red[SM_THREADS / 32];
  __shared__ double ssq_cta;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* xs = smem;                                          // panels of 64 columns; with two row blocks one panel of each
  uint8_t* as = xs + S::PLANES * S::X_BYTES;                   // blocks (0, 0), (0, 1), (1, 1), each with its planes
  uint8_t* bs = as + S::PLANES * S::BLOCKS * S::F_BYTES;
  uint8_t* part = S::PART_IN_B ? bs : bs + S::F_BYTES;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quarter = warp & 3, part4 = warp >> 2, row = quarter * 32 + lane;
  const uint32_t ctas = g.ctas, rank = ctas > 1 ? cluster_ctarank() : 0;
  const int z = blockIdx.x / ctas;
  const int slice = g.slice, s0 = (int)rank * slice;
  const uint32_t mma_bar = smem_u32(&bar);

  if (tid == 0) {
    mbar_init(mma_bar, 1);
    failed = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_slot), S::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_row = tmem_slot + ((uint32_t)(quarter * 32) << 16);
  uint32_t phase = 0;

  // ---- the matrix (or the momentum update that makes it) -> TMEM, and its sum of squares
  float kt = 1.0f, ki = 0.0f;
  if (e.scalars != nullptr) {
    kt = (1.0f - e.beta * e.scalars[0]) * e.scalars[1];
    ki = e.beta * e.scalars[1];
  }
  const void* gt = e.grad[z];
  const void* gi = e.info[z];
  float* mom = reinterpret_cast<float*>(e.moment[z]);
  // Chunk c0 of X's columns in TMEM (slice columns of each row block): a thread holds row i, columns j .. j + 31 of X, which are
  // 32 elements of a row of the matrix, or, when it is tall, of a column, where neighbouring lanes read neighbouring addresses.
  // Sixteen elements at a time: in row-major order a lane's accesses fill whole sectors.
  auto chunk_at = [&](int c0, int& i, int& j) {
    i = RB == 2 ? (c0 >> 6) * 128 + row : row;
    j = s0 + (RB == 2 ? (c0 & 63) : c0);
  };
  auto for_pieces = [&](int i, int j, auto body) {      // body(first element, address offset given the row pitch)
#pragma unroll
    for (int q = 0; q < 16 / V; ++q)
      if (i < g.k && j + q * V < g.wide) body(q);
  };
  auto offset = [&](int i, int j, int64_t ld) { return g.tall ? (int64_t)j * ld + i : (int64_t)i * ld + j; };
  auto load16 = [&](const void* p, int dtype, int64_t ld, int i, int j, float (&v)[16]) {
    for_pieces(i, j, [&](int q) {
      if (V > 1 && !g.tall) {
        const VecF<V> x = load_vec<V>(p, dtype, offset(i, j + q * V, ld));
#pragma unroll
        for (int n = 0; n < V; ++n) v[q * V + n] = x.e[n];
      } else {
#pragma unroll
        for (int n = 0; n < V; ++n)
          if (j + q * V + n < g.wide) v[q * V + n] = load_vec<1>(p, dtype, offset(i, j + q * V + n, ld)).e[0];
      }
    });
  };
  auto store16 = [&](void* p, int dtype, int64_t ld, int i, int j, const float (&v)[16]) {
    for_pieces(i, j, [&](int q) {
      if (V > 1 && !g.tall) {
        VecF<V> x;
#pragma unroll
        for (int n = 0; n < V; ++n) x.e[n] = v[q * V + n];
        store_vec<V>(p, dtype, offset(i, j + q * V, ld), x);
      } else {
#pragma unroll
        for (int n = 0; n < V; ++n)
          if (j + q * V + n < g.wide) {
            VecF<1> x;
            x.e[0] = v[q * V + n];
            store_vec<1>(p, dtype, offset(i, j + q * V + n, ld), x);
          }
      }
    });
  };
  double ssq = 0.0;
  for (int c0 = part4 * 32; c0 < RB * slice; c0 += 128) {
    int i, j0;
    chunk_at(c0, i, j0);
    VecF<16> u[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < 16; ++n) u[h].e[n] = 0.0f;
      load16(gt, e.grad_dtype, e.grad_ld, i, j0 + 16 * h, u[h].e);
    }
    if (e.momentum) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        VecF<16> f, m;
#pragma unroll
        for (int n = 0; n < 16; ++n) f.e[n] = m.e[n] = 0.0f;
        if (gi != nullptr) load16(gi, e.grad_dtype, e.grad_ld, i, j0 + 16 * h, f.e);
        load16(mom, ELEM_F32, e.cols, i, j0 + 16 * h, m.e);
        momentum_step<16>(e, kt, ki, gi != nullptr, u[h], f, m);      // zeros outside the matrix stay zeros
        store16(mom, ELEM_F32, e.cols, i, j0 + 16 * h, m.e);
      }
    }
    add_squares<16>(ssq, u[0]);
    add_squares<16>(ssq, u[1]);
    uint32_t w[32];
#pragma unroll
    for (int n = 0; n < 32; ++n) w[n] = __float_as_uint(u[n >> 4].e[n & 15]);
    tmem_st_32x32(tmem_row + S::X_COL + c0, w);
  }
  tmem_st_wait();
  tc_fence_before_sync();
  double total = block_sum(ssq, red);
  if (ctas > 1) {
    if (tid == 0) ssq_cta = total;
    cluster_sync_all();
    total = 0.0;
    for (uint32_t c = 0; c < ctas; ++c) total += ld_dsmem_f64(smem_u32(&ssq_cta), c);
  }
  const double inv = (double)NS_SCALE / (sqrt(total) + (double)e.eps);
  const float finv = (float)inv;
  const bool fine = finv > 1e-30f && finv < 1e30f;      // else the factor itself does not fit fp32

  tc_fence_after_sync();

  // all MMAs issued so far are done: their results can be read
  auto mma_wait = [&]() {
    if (!*((volatile int*)&failed) && !mbar_wait(mma_bar, phase)) {
      report(status, STATUS_TIMEOUT_TMEM_FULL, 88, z);
      *((volatile int*)&failed) = 1;
    }
    phase ^= 1;
    tc_fence_after_sync();
  };
  // operands written by all threads (of all CTAs) -> the issuing thread's MMAs
  auto publish = [&](bool cluster) {
    fence_proxy_async_smem();
    tc_fence_before_sync();
    if (cluster) {
      asm volatile("fence.proxy.async;" ::: "memory");      // the other CTAs' shared memory as well
      cluster_sync_all();
      fence_proxy_async_smem();
    } else {
      __syncthreads();
    }
    tc_fence_after_sync();
  };
  const uint32_t xs_addr = smem_u32(xs), as_addr = smem_u32(as), bs_addr = smem_u32(bs);
  // One thread: acc (+)= P Q^T over k_steps x 16 of the reduction; hi lo, lo hi, hi hi. An MN-major operand lies as rows of the
  // reduction in panels of 64 columns.
  auto mma_run = [&](uint32_t acc_col, uint32_t p0, int p_plane, bool p_mn, uint32_t q0, int q_plane, bool q_mn, int k_steps, int n, bool add) {
    const uint32_t idesc = make_instr_desc(0, 0, p_mn ? 1 : 0, q_mn ? 1 : 0, 128, (uint32_t)n);
    uint32_t on = add ? 1u : 0u;
    for (int seg = SPLIT ? 0 : 2; seg < 3; ++seg) {
      const uint32_t pb = p0 + (seg == 1 ? p_plane : 0), qb = q0 + (seg == 0 ? q_plane : 0);
      for (int s = 0; s < k_steps; ++s) {
        const uint32_t k_off = (s >> 2) * SM_PANEL + (s & 3) * 32, mn_off = s * (16 * 128);
        const uint64_t dp = p_mn ? make_smem_desc(pb + mn_off, SM_PANEL, 1024) : make_smem_desc(pb + k_off, 16, 1024);
        const uint64_t dq = q_mn ? make_smem_desc(qb + mn_off, SM_PANEL, 1024) : make_smem_desc(qb + k_off, 16, 1024);
        mma_bf16(tmem_slot + acc_col, dp, dq, idesc, on);
        on = 1u;
      }
    }
  };
  // block (i, j) of a symmetric factor: stored at and above the diagonal, read below it in the other major order
  auto block_of = [](int i, int j) { return i <= j ? i * (RB - 1) + j : j * (RB - 1) + i; };
  constexpr int BLOCK_BYTES = S::PLANES * S::F_BYTES;

  // ---- X scaled: operands, and a X for the products to add to
  // columns of X in TMEM: slice columns of each row block
  for (int c0 = part4 * 32; c0 < RB * slice; c0 += 128) {
    uint32_t w[32];
    float v[32];
    tmem_ld_32x32(tmem_row + S::X_COL + c0, w);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      v[i] = fine ? __uint_as_float(w[i]) * finv : (float)((double)__uint_as_float(w[i]) * inv);
      w[i] = __float_as_uint(SPLIT ? v[i] : v[i] * (g.a * NS_SCALE));
    }
    sm_put_operand<SPLIT>(xs, S::X_BYTES, row, c0, v);      // with two row blocks c0 / 64 is the block, which is also the panel
    tmem_st_32x32(tmem_row + S::X_COL + c0, w);
  }
  tmem_st_wait();

  for (int step = 0; step < g.steps; ++step) {
    // A = X X^T
    publish(false);
    if (warp == 0 && elect_one()) {
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = i; j < RB; ++j)
          mma_run(S::ACC_COL + 128 * block_of(i, j), xs_addr + i * SM_PANEL, S::X_BYTES, false, xs_addr + j * SM_PANEL, S::X_BYTES, false,
                  slice >> 4, 128, false);
      mma_commit(mma_bar);
    }
    __syncwarp();
    mma_wait();
    if (RB == 1 && ctas == 1) {
      uint32_t w[32];
      float v[32];
      tmem_ld_32x32(tmem_row + S::ACC_COL + part4 * 32, w);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(w[i]) * NS_UNSCALE;
      sm_put_operand<SPLIT>(as, S::F_BYTES, row, part4 * 32, v);
      publish(false);
    } else {
      for (int blk = 0; blk < S::BLOCKS; ++blk) {
      // this CTA's share as 512-byte rows of 16-byte pieces, XOR-ed with the row
      uint32_t w[32];
      tmem_ld_32x32(tmem_row + S::ACC_COL + 128 * blk + part4 * 32, w);
      tmem_ld_wait();
#pragma unroll
      for (int q = 0; q < 8; ++q)
        *reinterpret_cast<uint4*>(part + row * 512 + (((part4 * 8 + q) ^ (row & 7)) << 4)) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
      tc_fence_before_sync();
      cluster_sync_all();
      // rows rank * 128 / ctas ...: sum over the CTAs, result to all of them
      const int rows_here = 128 / (int)ctas;
      for (int t0 = tid; t0 < rows_here * 32; t0 += 2 * SM_THREADS) {      // two 16-byte pieces a thread in flight, of up to four CTAs each
        float4 sum[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) sum[h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto piece = [&](int h, int& r, int& q) {
          const int t = t0 + h * SM_THREADS;
          r = (int)rank * rows_here + (t >> 5);
          q = t & 31;
          return t < rows_here * 32;
        };
        for (uint32_t c0 = 0; c0 < ctas; c0 += 4) {
          float4 v[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            int r, q;
            const bool live = piece(h, r, q);
            const uint32_t at = smem_u32(part + r * 512 + ((q ^ (r & 7)) << 4));
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c)
              if (live && c0 + c < ctas) v[h][c] = ld_dsmem_f4(at, c0 + c);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c)
              if (c0 + c < ctas) { sum[h].x += v[h][c].x; sum[h].y += v[h][c].y; sum[h].z += v[h][c].z; sum[h].w += v[h][c].w; }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int r, q;
          if (!piece(h, r, q)) continue;
          const float s0_ = sum[h].x * NS_UNSCALE, s1_ = sum[h].y * NS_UNSCALE, s2_ = sum[h].z * NS_UNSCALE, s3_ = sum[h].w * NS_UNSCALE;
          const uint2 hi = make_uint2(pack_half2(s0_, s1_), pack_half2(s2_, s3_));
          const float2 h0 = unpack_half2(hi.x), h1 = unpack_half2(hi.y);
          const uint2 lo = make_uint2(pack_half2(s0_ - h0.x, s1_ - h0.y), pack_half2(s2_ - h1.x, s3_ - h1.y));
          const int col = q * 4;
          const uint32_t to = smem_u32(as + blk * BLOCK_BYTES + (col >> 6) * SM_PANEL + sm_piece(r, (col & 63) >> 3) + (col & 7) * 2);
          for (uint32_t c = 0; c < ctas; ++c) {
            st_dsmem_u2(to, c, hi);
            if (SPLIT) st_dsmem_u2(to + S::F_BYTES, c, lo);
          }
        }
      }
      if (blk + 1 < S::BLOCKS) cluster_sync_all();      // the shares have been read
      else publish(true);
      }
    }
    // B = b A + c A A
    if (warp == 0 && elect_one()) {
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = i; j < RB; ++j)
#pragma unroll
          for (int m = 0; m < RB; ++m)
            mma_run(S::ACC_COL + 128 * block_of(i, j), as_addr + block_of(i, m) * BLOCK_BYTES, S::F_BYTES, i > m,
                    as_addr + block_of(j, m) * BLOCK_BYTES, S::F_BYTES, j > m, 8, 128, m > 0);
      mma_commit(mma_bar);
    }
    __syncwarp();
    mma_wait();
#pragma unroll 1
    for (int blk = 0; blk < S::BLOCKS; ++blk) {
      const int c0 = part4 * 32;
      uint32_t w[32];
      float v[32];
      tmem_ld_32x32(tmem_row + S::ACC_COL + 128 * blk + c0, w);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint8_t* at = as + blk * BLOCK_BYTES + (c0 >> 6) * SM_PANEL + sm_piece(row, ((c0 & 63) >> 3) + q);
        const uint4 hi = *reinterpret_cast<const uint4*>(at);
        const uint32_t hw[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack_half2(hw[i]);
          v[8 * q + 2 * i] = f.x; v[8 * q + 2 * i + 1] = f.y;
        }
        if (SPLIT) {
          const uint4 lo = *reinterpret_cast<const uint4*>(at + S::F_BYTES);
          const uint32_t lw[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_half2(lw[i]);
            v[8 * q + 2 * i] += f.x; v[8 * q + 2 * i + 1] += f.y;
          }
        }
      }
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = fmaf(g.b, v[i], (g.c * NS_UNSCALE) * __uint_as_float(w[i]));
      sm_put_operand<SPLIT>(bs + blk * BLOCK_BYTES, S::F_BYTES, row, c0, v);
    }
    publish(false);
    // X <- a X + B X
    if (warp == 0 && elect_one()) {
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int m = 0; m < RB; ++m)
          mma_run(S::BX_COL + i * slice, bs_addr + block_of(i, m) * BLOCK_BYTES, S::F_BYTES, i > m, xs_addr + m * SM_PANEL, S::X_BYTES, true, 8,
                  slice, !SPLIT || m > 0);
      mma_commit(mma_bar);
    }
    __syncwarp();
    mma_wait();
    if (!SPLIT && step + 1 == g.steps) break;
#pragma unroll 1
    for (int c0 = part4 * 32; c0 < RB * slice; c0 += 128) {
      uint32_t w[32];
      float v[32];
      tmem_ld_32x32(tmem_row + S::X_COL + c0, w);
      if constexpr (SPLIT) {
        uint32_t bx[32];
        tmem_ld_32x32(tmem_row + S::BX_COL + c0, bx);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          v[i] = fmaf(g.a, __uint_as_float(w[i]), __uint_as_float(bx[i]) * NS_UNSCALE);
          w[i] = __float_as_uint(v[i]);
        }
      } else {
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          v[i] = __uint_as_float(w[i]) * NS_UNSCALE;
          w[i] = __float_as_uint(__uint_as_float(w[i]) * g.a);
        }
      }
      sm_put_operand<SPLIT>(xs, S::X_BYTES, row, c0, v);
      tmem_st_32x32(tmem_row + S::X_COL + c0, w);
    }
    tmem_st_wait();
  }

  // ---- the result, or the parameter update
  void* out = e.out[z];
  for (int c0 = part4 * 32; c0 < RB * slice; c0 += 128) {
    int i, j0;
    chunk_at(c0, i, j0);
    uint32_t w[32];
    tmem_ld_32x32(tmem_row + S::X_COL + c0, w);
    float p[2][16];
    if (e.momentum) {
#pragma unroll
      for (int h = 0; h < 2; ++h) load16(out, e.out_dtype, e.cols, i, j0 + 16 * h, p[h]);
    }
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const float o = __uint_as_float(w[16 * h + n]) * (SPLIT ? NS_UNSCALE : NS_UNSCALE * NS_UNSCALE);
        p[h][n] = e.momentum ? fmaf(-e.step, o, p[h][n] * e.decay) : o;
      }
      store16(out, e.out_dtype, e.cols, i, j0 + 16 * h, p[h]);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_slot, S::TMEM_COLS);
  }
  if (ctas > 1) cluster_sync_all();
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

// Layout of the workspace for `batch` matrices: X twice (hi and lo planes), A and B (hi and lo), norms, tile counts.
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
  w.total = 2 * w.partial + batch * NS_NORM_BLOCKS * (int64_t)sizeof(double) + (batch + 1) * (int64_t)sizeof(uint32_t);
  return w;
}


template <int V>
static void ns_begin(const NsEnds& e, int norm_blocks, int blocks, cudaStream_t st) {
  if (e.momentum) ns_begin_kernel<V, true><<<dim3(norm_blocks, e.batch), ENDS_THREADS, 0, st>>>(e);
  else ns_begin_kernel<V, false><<<dim3(norm_blocks, e.batch), ENDS_THREADS, 0, st>>>(e);
  ns_scale_kernel<V><<<dim3(blocks, e.batch), ENDS_THREADS, 0, st>>>(e, norm_blocks);
}

// Whether four elements an access fit every row of every matrix.
static bool ns_vec4(const NsEnds& e) {
  const int in_size = e.grad_dtype == ELEM_F32 ? 4 : 2, out_size = e.out_dtype == ELEM_F32 ? 4 : 2;
  bool vec = e.cols % 4 == 0 && e.grad_ld % 4 == 0;
  for (int z = 0; z < e.batch && vec; ++z) {
    vec = reinterpret_cast<uintptr_t>(e.grad[z]) % (4 * in_size) == 0 && reinterpret_cast<uintptr_t>(e.out[z]) % (4 * out_size) == 0 &&
          reinterpret_cast<uintptr_t>(e.info[z]) % (4 * in_size) == 0 && reinterpret_cast<uintptr_t>(e.moment[z]) % 16 == 0;
  }
  return vec;
}

template <int RB, bool SPLIT, int V>
static const char* launch_small(const NsCall& call, Status* status, cudaStream_t st) {
  using S = SmShape<RB, SPLIT>;
  NsSmall g;
  g.tall = call.ends.rows > call.ends.cols;
  g.k = g.tall ? call.ends.cols : call.ends.rows;
  g.wide = g.tall ? call.ends.rows : call.ends.cols;
  g.steps = call.steps;
  g.a = call.c[0];
  g.b = call.c[1];
  g.c = call.c[2];
  g.ctas = 1;
  // As few CTAs as hold the matrix: one 128 x 512 matrix takes 50 us on 2 CTAs and 43 us on 8, 48 of them 51 and 168 us.
  while (g.ctas * S::SLICE < g.wide) g.ctas *= 2;
  g.slice = ((g.wide + g.ctas - 1) / g.ctas + 63) / 64 * 64;
  auto kernel = ns_small_kernel<RB, SPLIT, V>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess) return "orthogonalize: shared memory";
  if (g.ctas > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return "orthogonalize: cluster size";
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(call.ends.batch * g.ctas));
  cfg.blockDim = dim3(SM_THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)g.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, call.ends, g, status) == cudaSuccess ? nullptr : "ns_small launch failed";
}

// Row blocks of a matrix that one cluster keeps, 0 for the others. One block of 128 rows: 8 CTAs with slices of 256 columns, or, with
// pairs, 16 with slices of 128. Two blocks: 4 CTAs with slices of 64 columns; pairs do not fit.
// With two blocks the exchange of A weighs more, so they are worth it only up to 256 x 256 and while all clusters run at once: 32
// matrices 107 us against 131 in ns_chain_body, one of them 99 against 100, 64 of them 198 against 157; in 8 CTAs one of 256 x 512
// took 111 against 107, 8 of them 113 against 112.
static int ns_small_blocks(int64_t batch, int64_t rows, int64_t cols, int steps, int pairs) {
  const int64_t k = rows < cols ? rows : cols, wide = rows < cols ? cols : rows;
  if (steps == 0) return 0;
  if (k <= 128 && wide <= 2048) return 1;
  return wide <= 256 && batch <= 32 && !pairs ? 2 : 0;
}

int64_t ns_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int steps, int pairs) {
  return ns_small_blocks(batch, rows, cols, steps, pairs) != 0 ? 0 : ns_space(batch, rows, cols).total;
}

const char* launch_orthogonalize(const NsCall& call, Status* status, cudaStream_t st) {
  const int64_t batch = call.ends.batch, rows = call.ends.rows, cols = call.ends.cols;
  if (batch < 1 || batch > NS_MAX_BATCH || rows < 1 || cols < 1) return "orthogonalize: sizes";
  if (rows > (1 << 20) || cols > (1 << 20)) return "orthogonalize: matrix too large";
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return "orthogonalize: device";
  const bool vec = ns_vec4(call.ends);
  switch (ns_small_blocks(batch, rows, cols, call.steps, call.pairs)) {
    case 1:
      if (call.pairs) return vec ? launch_small<1, true, 4>(call, status, st) : launch_small<1, true, 1>(call, status, st);
      return vec ? launch_small<1, false, 4>(call, status, st) : launch_small<1, false, 1>(call, status, st);
    case 2: return vec ? launch_small<2, false, 4>(call, status, st) : launch_small<2, false, 1>(call, status, st);
    default: break;
  }
  const NsSpace w = ns_space(batch, rows, cols);
  __half* base = reinterpret_cast<__half*>(call.workspace);
  __half* x[2] = {base, base + w.x};                       // each: hi planes of the batch, then lo planes
  __half* A = base + 2 * w.x;
  __half* B = A + w.k;
  const int64_t lo_x = w.x / 2, lo_k = w.k / 2;
  uint8_t* tail = reinterpret_cast<uint8_t*>(call.workspace) + 2 * w.partial;
  const bool tall = rows > cols;

  NsPlan g;
  memset(&g, 0, sizeof(g));
  NsEnds e = call.ends;
  e.ld = (int)w.ld_x;
  e.plane = w.plane_x;
  e.u = reinterpret_cast<float*>(x[1]);                    // hi and lo planes of the other X buffer: four bytes an element
  e.x_hi = x[0];
  e.x_lo = x[0] + lo_x;
  e.partial = reinterpret_cast<double*>(tail);
  e.done = reinterpret_cast<uint32_t*>(tail + batch * NS_NORM_BLOCKS * sizeof(double));
  e.next_item = e.done + batch;
  const int64_t per_row = (cols + (vec ? 3 : 0)) / (vec ? 4 : 1);
  e.tpr_log2 = 0;
  while (e.tpr_log2 < 8 && (1 << e.tpr_log2) < per_row) ++e.tpr_log2;
  const int64_t rows_per_block = (ENDS_THREADS >> e.tpr_log2) * ENDS_ROWS;
  const int64_t blocks = (rows + rows_per_block - 1) / rows_per_block;
  const int norm_blocks = (int)(blocks < NS_NORM_BLOCKS ? blocks : NS_NORM_BLOCKS);
  const int all_blocks = (int)(blocks < 4096 ? blocks : 4096);
  if (vec) ns_begin<4>(e, norm_blocks, all_blocks, st);
  else ns_begin<1>(e, norm_blocks, all_blocks, st);

  g.batch = (int)batch;
  g.steps = call.steps;
  g.rows = (int)rows;
  g.cols = (int)cols;
  g.tall = tall;
  g.k = (int)(tall ? cols : rows);
  g.wide = (int)(tall ? rows : cols);
  g.a = call.c[0];
  g.b = call.c[1];
  g.c = call.c[2];
  g.done = e.done;
  g.next_item = e.next_item;
  // A pair's 256 x 256 tile needs half the operand traffic of a 128 x 128 one, but has four times its latency: worth it where a step
  // has some three tiles for every pair (32 of 512 x 512: 238 us against 255 with single tiles, 16 of 512 x 2048: 364 against 416,
  // six of 1024 x 1024: 244 against 250; ten of 768 x 768: 233 against 219, 20 of 512 x 512: 211 against 187) or where the sums
  // are long (one 1400 x 1400: 228 against 251, one 1536 x 1536: 237 against 270; one 1024 x 1024: 191 against 157).
  const int64_t k256 = (g.k + 255) / 256, wide256 = (g.wide + 255) / 256;
  const bool pair = !call.pairs && g.k > 256 && (batch * (k256 * (k256 + 1) + k256 * wide256) >= 210 || g.k >= 1280);
  const int tile = pair ? 256 : 128;
  const int kt = (g.k + tile - 1) / tile, wt = (g.wide + tile - 1) / tile;
  g.tiles_sym = kt * (kt + 1) / 2;
  g.tiles_x = kt * wt;
  g.tiles_xm = tall ? wt : kt;
  const int units = pair ? sms / 2 : sms;
  const int64_t items = batch * g.steps * (2 * g.tiles_sym + g.tiles_x);
  if (items > (1ll << 30)) return "orthogonalize: too many tiles";
  g.items = (int)items;

  bool ok = true;
  auto load_map = [&](CUtensorMap* m, const __half* p, int64_t r, int64_t c, int64_t ld, int64_t plane, bool mn) {
    ok &= ns_map(m, p, batch, r, c, ld, plane, mn ? NS_BK : 128, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  auto box_map = [&](CUtensorMap* m, const __half* p, int64_t r, int64_t c, int64_t ld, int64_t plane) {
    ok &= ns_map(m, p, batch, r, c, ld, plane, NS_BOX, NS_BOX, CU_TENSOR_MAP_SWIZZLE_64B);
  };
  for (int lo = 0; lo < 2; ++lo) {
    for (int i = 0; i < 2; ++i) {
      const __half* p = x[i] + lo * lo_x;
      load_map(&g.x_gram[i][lo], p, rows, cols, w.ld_x, w.plane_x, tall);      // A = X X^T; tall: X^T X, both operands MN-major
      load_map(&g.x_apply[i][lo], p, rows, cols, w.ld_x, w.plane_x, !tall);    // B X: X is the MN-major second operand; tall: X B^T
      box_map(&g.x_box[i][lo], p, rows, cols, w.ld_x, w.plane_x);
    }
    for (int mn = 0; mn < 2; ++mn) {
      load_map(&g.a_load[lo][mn], A + lo * lo_k, g.k, g.k, w.ld_k, w.plane_k, mn);
      load_map(&g.b_load[lo][mn], B + lo * lo_k, g.k, g.k, w.ld_k, w.plane_k, mn);
    }
    box_map(&g.a_box[lo], A + lo * lo_k, g.k, g.k, w.ld_k, w.plane_k);
    box_map(&g.b_box[lo], B + lo * lo_k, g.k, g.k, w.ld_k, w.plane_k);
  }
  if (!ok) return "orthogonalize: cuTensorMapEncodeTiled failed";
  if (g.items > 0) {
    auto kernel = call.pairs ? ns_chain_split_kernel : (pair ? ns_chain_pair_kernel : ns_chain_kernel);
    const int smem = call.pairs ? NsShape<true>::SMEM : NsShape<false>::SMEM;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return "orthogonalize: shared memory";
    // No product has more tiles at once than batch x tiles_x, but a CTA that finishes one has its next item, of a later
    // product, in hand already, and its loads wait while others stand idle: with four CTAs a tile the next product's items
    // are with CTAs that have nothing else to do (one 1024 x 1024: 206 us with one a tile, 164 with two, 156 with four, 156
    // with the whole device; 1030 x 515 in pairs of fp16: 271, 232, 232, 232). What is left stays free for a second shape.
    const int64_t most = 4 * batch * g.tiles_x;
    const int count = (int)(most < units ? most : units);
    kernel<<<(pair ? 2 : 1) * count, NS_THREADS, smem, st>>>(g, status);
  }
  e.x_hi = x[g.steps & 1];
  e.x_lo = x[g.steps & 1] + lo_x;
  if (vec) ns_end_kernel<4><<<dim3(all_blocks, (unsigned)batch), ENDS_THREADS, 0, st>>>(e);
  else ns_end_kernel<1><<<dim3(all_blocks, (unsigned)batch), ENDS_THREADS, 0, st>>>(e);
  return cudaGetLastError() == cudaSuccess ? nullptr : "orthogonalize launch failed";
}

}  // namespace gd
