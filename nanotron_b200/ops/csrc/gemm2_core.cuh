// The kernel of the bf16 GEMM on CTA pairs (tcgen05 cta_group::2 + TMEM + TMA), persistent and warp-specialised (sm_100a).
//
//   D[M,N] (=|+=) sum_k A(m,k) * B(n,k)          same operand-storage and output conventions as gemm_tcgen05.cu
//
// Two CTAs of a cluster (one per SM of a pair) work on one 256 x 256 output tile.  Each CTA keeps in its own shared memory the
// 128 rows of A that it owns and HALF of the B tile (128 of the 256 output columns); one thread of the leader CTA issues
// tcgen05.mma.cta_group::2 (256 x 256 x 16), the hardware reads both halves of B for both SMs, and each CTA's TMEM receives its
// 128 rows x 256 columns of accumulators.  Per MMA each SM reads 8 KB of operands instead of the 12 KB of the one-CTA 128 x 256
// tile, and its shared memory holds 32 KB per stage instead of 48, so six stages fit.
//
// Warp roles per CTA: warp 0 TMA producer (own A rows + own half of B into the CTA's own shared memory; the loads are the
// cta_group::2 form of cp.async.bulk.tensor, whose completion bytes are counted on the LEADER's stage barrier, so the leader's MMA
// thread waits on one barrier for both halves); warp 1: the MMA issuer in the leader, idle in the peer; warps 2..5 epilogue
// (tcgen05.ld -> swizzled staging -> TMA store / reduce-add of the CTA's own rows).  Epilogues that compute take EW = 8 warps, four to
// each half of the columns: 2..9, or 4..11 with warps 2 and 3 idle where warp groups exchange registers (statistics).
// Cross-CTA signals besides the loads are plain remote mbarrier arrives: the leader's producer forwards every "stage free" to the
// peer's producer, one leader epilogue warp forwards "accumulator ready" to the peer's epilogue, and the peer's epilogue warps hand
// accumulators back to the leader's MMA thread.  All waits are bounded; the two CTAs meet in a cluster barrier before TMEM is freed.
#pragma once
#include "common.cuh"
#include "sm100_ptx.cuh"
#include <type_traits>

namespace {

constexpr int P_BLOCK_M = 128;   // rows per CTA (256 per pair)
constexpr int P_BLOCK_N = 256;   // columns per pair; each CTA stages 128 of them
constexpr int P_HALF_N = 128;
constexpr int P_BLOCK_K = 64;
constexpr int P_UMMA_K = 16;
constexpr int P_MAX_STAGES = 6;
constexpr int P_A_BYTES = P_BLOCK_M * P_BLOCK_K * 2;  // 16 KiB
constexpr int P_B_BYTES = P_HALF_N * P_BLOCK_K * 2;   // 16 KiB
constexpr int P_STAGE_BYTES = P_A_BYTES + P_B_BYTES;
constexpr int P_EPI_WARPS = 4;
constexpr int P_EPI_BUF = 32 * 128;
constexpr int P_THREADS = 32 * (2 + P_EPI_WARPS);
constexpr int P_SMEM = P_MAX_STAGES * P_STAGE_BYTES + P_EPI_WARPS * 2 * P_EPI_BUF + 1024 + 512;

enum POut { P_OUT_BF16 = 0, P_OUT_F32 = 1, P_OUT_F32_ACCUM = 2, P_OUT_PEER_BF16 = 3, P_OUT_CE_STATS = 4, P_OUT_CE_GRAD = 5, P_OUT_CE_STATS_T = 6 };
constexpr bool p_ce_stats(int out) { return out == P_OUT_CE_STATS || out == P_OUT_CE_STATS_T; }

// What an epilogue needs beside the accumulator.  PPlain: nothing.
struct PPlain {};
// D = *alpha * (A B^T): a device scalar applied to the fp32 accumulator before it is rounded or added.
struct PAlpha {
  const float* alpha = nullptr;
};
// Cross entropy over the product's columns (linear_ce.cu): A = hidden states, B = rows of the head weight, so an accumulator row
// holds 256 consecutive scores of one token.
struct PCeArgs {
  const int64_t* target = nullptr;  // [M] class of every row, in the numbering in which column 0 of this product is `col0`
  int64_t col0 = 0;
  // P_OUT_CE_STATS: nothing but these leaves the kernel
  float2* part = nullptr;           // [tiles_n * EW / 4][M] (largest score, sum exp(score - largest)) of every 1024 / EW columns
  float* tgt = nullptr;             // [M] the target's score, written where the target is one of this product's columns
  // P_OUT_CE_STATS_T: the product the other way around, A = rows of the head weight, B = hidden states, so that a tile's width follows the
  // number of tokens (`tile_n`, a multiple of 32 up to 256; `part` is then [2 pairs of a token tile][N], `target` and `tgt` are [N])
  int tile_n = P_BLOCK_N;
  // P_OUT_CE_GRAD: D = coef * exp(score - logz) - g * [column is the target], zero in the padding columns of D
  const float* logz = nullptr;
  const float* coef = nullptr;
  const float* g = nullptr;
  int a_rows = P_BLOCK_M;           // rows per load of A: P_BLOCK_M, or all there are in steps of 8
};

// P_OUT_CE_STATS_T: BLOCKS = tile_n / 64, rounded up.
template <int BLOCKS_> struct PCeTurned : PCeArgs {
  static constexpr int BLOCKS = BLOCKS_;
};

// The tensor cores cut what does not fit when they add to an accumulator: a sum over K comes out small by about 2^-26 of its value per 16
// products (measured: 9e-10 K).  For the loss that is the largest error (4e-6 of every score at K = 4096), so its scores are accumulated
// over at most this many k-blocks (1024 products) and the pieces added in registers, rounding to nearest: the loss (of
// scores with a standard deviation of 1.5) is then off by 2.7e-7 of its value instead of 1.1e-6 (K = 4096) or 2.4e-6 (8192).  us, one
// accumulator -> pieces: 4096 x 2048 x 128256 1265 -> 1290, 16384 x 2048 x 128256 5650 -> 5795.
constexpr int P_CE_SEGMENT = 16;

constexpr float P_LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float p_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// In a kernel that may have been launched before the one in front of it in the stream is complete: waits until it is, and its writes are seen.
// Returns at once after an ordinary launch.
__device__ __forceinline__ void p_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Tensor-parallel fusion on the pair kernel (same protocol as the one-CTA kernel in gemm_tcgen05.cu; all off when world == 0):
//  * all-gather -> GEMM: A is a gathered buffer of `world` row blocks of `ag_rows` rows that peers fill with plain stores;
//    block r is valid once ag_flags[r] >= epoch.  Each CTA's TMA producer polls the word of the block its 128 rows belong to
//    (bounded) before its first load from it; tile rows are visited starting with this rank's own block.
//  * GEMM -> reduce-scatter (P_OUT_PEER_BF16): the epilogue TMA-stores every bf16 chunk into slot `me` of the staging area of the
//    rank that owns those rows (one tensor map per owner); the last CTA of the grid to finish raises rs_flags[owner][me] everywhere.
constexpr int P_TP_MAX = 8;
struct PFuse {
  int world = 0, me = 0;
  uint32_t epoch = 0;
  int m_rot = 0;                        // rotation of the tile rows, in 256-row pair tiles
  const uint32_t* ag_flags = nullptr;   // local flag words [world]
  int ag_rows = 0;                      // rows per gathered block (multiple of 128)
  int ag_local = 0;                     // 1: this rank's own block is read through tmap_al (its source tensor) and needs no flag
  uint32_t* rs_flags[P_TP_MAX] = {};    // per-owner flag words [world]
  int rs_rows = 0;                      // rows per owner (multiple of 32)
  unsigned int* done_counter = nullptr; // local counter, zero before launch
};
struct PPeerMaps {
  CUtensorMap m[P_TP_MAX];
};

// Work units of a launch.  Tiles are dealt to the CTA pairs round robin; when the last round would leave most pairs idle, the
// tiles of that round are cut along K into `split` chunks each, one unit per chunk, so the tail of the launch is shared by all
// pairs.  A chunk stores its fp32 partial sums into a slab of its own in a workspace (no zero fill, no atomics); a small pass
// then sums the slabs of a tile in chunk order and writes D (bf16 / fp32 store, or fp32 accumulate), so the result does not
// depend on which chunk finished first.
struct PSched {
  int total_units = 0;  // grid-stride loop bound
  int full_units = 0;   // units [0, full_units) are whole tiles with the same index
  int split = 1;        // chunks per tile of the last round (1: nothing is split)
  int kb_per = 0;       // k-blocks per chunk
};
struct PUnit {
  int tile, kb0, kbs, ws;  // ws: workspace slab of this chunk (unit index within the last round), -1 for a whole tile
};
__device__ __forceinline__ PUnit decode_unit(int u, const PSched& sc, int k_blocks) {
  if (u < sc.full_units || sc.split <= 1) return {u, 0, k_blocks, -1};
  const int v = u - sc.full_units;
  const int rt = v / sc.split, ch = v - rt * sc.split;
  const int kb0 = ch * sc.kb_per;
  return {sc.full_units + rt, kb0, min(sc.kb_per, k_blocks - kb0), v};
}

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared::cta address of this CTA -> shared::cluster address of the same location in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_to_cta(uint32_t local_addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local_addr), "r"(rank));
  return a;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Forwarding a hardware completion (nothing this thread wrote has to become visible): no release fence on the hot path.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void tmem_alloc2(uint32_t* smem_dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(smem_dst)), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish2() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void umma2_f16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrive on the barrier at shared::cluster address `addr` once every tcgen05.mma issued so far by this thread has completed
__device__ __forceinline__ void umma2_commit(uint32_t addr) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(addr) : "memory");
}

// Tiled loads whose mbarrier may live in the other CTA of the pair (`bar_cluster_addr` is a shared::cluster address).
__device__ __forceinline__ void tma2_load_2d(void* smem_dst, const CUtensorMap* m, uint32_t bar_cluster_addr, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(ptx::smem_u32(smem_dst)),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster_addr), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tma2_load_3d(void* smem_dst, const CUtensorMap* m, uint32_t bar_cluster_addr, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(ptx::smem_u32(smem_dst)),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
               : "memory");
}

struct PTile {
  int m_blk, n_blk;  // in units of 256 x 256 pair tiles
};
// Tiles are visited column by column inside bands of `BAND` tile rows: the band's rows of A stay in L2 while B streams through
// once per band.  The host picks the band so that its A rows take about a third of L2, i.e. B is re-read as rarely as possible.
__device__ __forceinline__ PTile pair_tile(int t, int tiles_m, int tiles_n, int BAND) {
  const int band_size = BAND * tiles_n;
  const int band = t / band_size;
  const int first_m = band * BAND;
  const int rows = min(BAND, tiles_m - first_m);
  const int r = t - band * band_size;
  return {first_m + r % rows, r / rows};
}

// Running (largest, sum of exponentials) of a row over 32 more scores.  One pass: when the largest grows, the sum so far is rescaled
// once per 32 scores, not per score.  Scores are folded as 2^(score log2 e - largest log2 e): one FMA and one ex2 each.
template <int W>
__device__ __forceinline__ void p_ce_accumulate(const uint32_t (&r)[W], int valid, float& m, float& s) {
  float cm = -INFINITY;
  if (valid >= W) {
#pragma unroll
    for (int j = 0; j < W; j++) cm = fmaxf(cm, __uint_as_float(r[j]));
  } else {
#pragma unroll
    for (int j = 0; j < W; j++)
      if (j < valid) cm = fmaxf(cm, __uint_as_float(r[j]));
  }
  const float nm = fmaxf(m, cm);
  const float base = nm == -INFINITY ? 0.f : nm * P_LOG2E;  // a row of -inf scores keeps the sum 0 instead of inf - inf
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (valid >= W) {
#pragma unroll
    for (int j = 0; j < W; j++) a[j & 3] += p_ex2(fmaf(__uint_as_float(r[j]), P_LOG2E, -base));
  } else {
#pragma unroll
    for (int j = 0; j < W; j++)
      if (j < valid) a[j & 3] += p_ex2(fmaf(__uint_as_float(r[j]), P_LOG2E, -base));
  }
  s = s * p_ex2(fmaf(m, P_LOG2E, -base)) + ((a[0] + a[1]) + (a[2] + a[3]));
  m = nm;
}

// 32 scores of a row -> 32 entries of the loss gradient; `valid` columns exist, `tj` is the target's position among them (or outside).
__device__ __forceinline__ void p_ce_gradient(uint32_t (&r)[32], int valid, int tj, float lz, float coef, float g) {
#pragma unroll
  for (int j = 0; j < 32; j++) r[j] = __float_as_uint(coef * p_ex2(fmaf(__uint_as_float(r[j]), P_LOG2E, -lz)));
  if (__any_sync(0xffffffffu, tj >= 0 && tj < 32)) {
#pragma unroll
    for (int j = 0; j < 32; j++)
      if (j == tj) r[j] = __float_as_uint(__uint_as_float(r[j]) - g);
  }
  if (valid < 32) {
#pragma unroll
    for (int j = 0; j < 32; j++)
      if (j >= valid) r[j] = 0u;
  }
}

// The statistics keep 128 scores of a row in every epilogue thread.  Its warps come in groups of four that exchange registers: the
// first group (producer, MMA issuer, two idle warps) hands most of its own to the two epilogue groups.  The shares add up to what the
// block is launched with (168 x 384); the host checks that before the launch.  (Without the exchange the scores spill, 168 registers at
// eight or 96 at sixteen epilogue warps, and the pass takes 1.3 times as long.)
constexpr int P_SPLIT_REGS = 168, P_SPLIT_REGS_LOAD = 72, P_SPLIT_REGS_EPI = 216;
static_assert(4 * P_SPLIT_REGS_LOAD + 8 * P_SPLIT_REGS_EPI == 12 * P_SPLIT_REGS, "register shares of the warp groups");
constexpr int p_first_epilogue_warp(int out) { return p_ce_stats(out) ? 4 : 2; }
constexpr int p_threads(int out, int ew) { return 32 * (p_first_epilogue_warp(out) + ew); }

// EW: epilogue warps per CTA, 4 (each takes 32 rows), or in the cross entropy modes 8 (each takes 32 rows and half of the columns; where
// the epilogue stages its output, P_OUT_CE_GRAD, the staging of the other four takes the memory of one operand stage).
template <bool A_MN, bool B_MN, int OUT, int P_STAGES, class EXT = PPlain, int EW = P_EPI_WARPS>
__global__ void __launch_bounds__(p_threads(OUT, EW), 1)
gemm2_tcgen05_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_d,
                     int M, int N, int K, int band, int* __restrict__ status, const __grid_constant__ PFuse fuse, const __grid_constant__ PPeerMaps pmaps,
                     const __grid_constant__ PSched sched, const __grid_constant__ CUtensorMap tmap_ws, const __grid_constant__ CUtensorMap tmap_al,
                     const __grid_constant__ EXT ext) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr bool TURNED = OUT == P_OUT_CE_STATS_T;  // more stages where they are smaller
  constexpr int STAGE = TURNED ? P_MAX_STAGES * P_STAGE_BYTES / P_STAGES : P_STAGE_BYTES;
  constexpr int EPI_BYTES = OUT == P_OUT_CE_STATS ? 0 : TURNED ? EW * P_EPI_BUF : EW * 2 * P_EPI_BUF;
  static_assert(P_STAGES * STAGE + EPI_BYTES + 1024 + 512 <= P_SMEM && P_STAGES <= 2 * P_MAX_STAGES && STAGE % 1024 == 0 &&
                    (EW == 4 || (EW == 8 && (p_ce_stats(OUT) || OUT == P_OUT_CE_GRAD))),
                "shared memory of a launch");
  uint8_t* epi_smem = smem + P_STAGES * STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi_smem + EPI_BYTES);
  uint64_t* full_bar = bars;                       // [STAGES]  (leader) both CTAs' loads of the stage have landed
  uint64_t* empty_bar = bars + 2 * P_MAX_STAGES;       // [STAGES]  the MMAs that read this stage are done
  uint64_t* tmem_full = bars + 4 * P_MAX_STAGES;       // [2]
  uint64_t* tmem_empty = tmem_full + 2;            // [2]  (leader) both CTAs' epilogues have drained the accumulator
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  constexpr int EPI0 = p_first_epilogue_warp(OUT);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();  // 0 = leader
  const int pair = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;
  const int tiles_m = (M + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M);
  int block_n = P_BLOCK_N;
  if constexpr (TURNED) block_n = ext.tile_n;
  const int tiles_n = (N + block_n - 1) / block_n;
  const int k_blocks = (K + P_BLOCK_K - 1) / P_BLOCK_K;

  if (threadIdx.x == 0) {
    for (int s = 0; s < P_STAGES; s++) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      ptx::mbar_init(&tmem_full[b], 1);  // leader: the MMA commit; peer: the remote arrive that forwards it
      ptx::mbar_init(&tmem_empty[b], 2 * EW);
    }
    *abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tmap(&tmap_a);
    ptx::prefetch_tmap(&tmap_b);
    ptx::prefetch_tmap(&tmap_d);
  }
  if constexpr (OUT == P_OUT_CE_GRAD) {
    if (M <= P_BLOCK_M) {  // rows of A that no load fills
      for (int i = threadIdx.x; i < P_STAGES * (P_A_BYTES / 16); i += blockDim.x)
        *reinterpret_cast<uint4*>(smem + (i / (P_A_BYTES / 16)) * P_STAGE_BYTES + (i % (P_A_BYTES / 16)) * 16) = make_uint4(0, 0, 0, 0);
      ptx::fence_proxy_async();
    }
  }
  if (warp == 1) {
    tmem_alloc2(tmem_base_slot, 512);
    tmem_relinquish2();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (!std::is_same_v<EXT, PPlain>) p_wait_for_previous();
  cluster_sync_all();  // both CTAs' barriers are initialised before any remote arrive or commit can reach them
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;

  if (warp < EPI0) {
  if constexpr (p_ce_stats(OUT)) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P_SPLIT_REGS_LOAD));
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    if (ptx::elect_one()) {
      int it = 0;
      bool ok = true;
      uint32_t ag_ready = 0;
      // A of up to 128 rows: only those are loaded (a load fills rows past the end with zeros, but slowly), the rest of the operand stays zero
      bool a_none = false;  // this CTA has no rows of A
      uint32_t stage_bytes = 2 * P_STAGE_BYTES;
      if constexpr (TURNED) {
        stage_bytes = 2 * P_A_BYTES + block_n * P_BLOCK_K * 2;
      } else if constexpr (OUT == P_OUT_CE_GRAD) {
        a_none = M <= P_BLOCK_M && cta == 1;
        stage_bytes = 2 * P_B_BYTES + (M <= P_BLOCK_M ? 1 : 2) * ext.a_rows * P_BLOCK_K * 2;
      }
      for (int u = pair; u < sched.total_units && ok; u += num_pairs) {
        const PUnit un = decode_unit(u, sched, k_blocks);
        if (un.kbs <= 0) continue;
        PTile tc = TURNED ? PTile{un.tile / tiles_n, un.tile % tiles_n} : pair_tile(un.tile, tiles_m, tiles_n, band);
        tc.m_blk = (tc.m_blk + fuse.m_rot) % tiles_m;
        const int m0 = (tc.m_blk * 2 + static_cast<int>(cta)) * P_BLOCK_M;           // this CTA's rows of A
        const int n0 = tc.n_blk * block_n + static_cast<int>(cta) * (block_n / 2);   // this CTA's half of B
        bool a_local = false;
        if (fuse.ag_flags != nullptr && m0 < M) {
          const int src = min(fuse.world - 1, m0 / fuse.ag_rows);  // ag_rows is a multiple of 128: one source per CTA row block
          if (fuse.ag_local && src == fuse.me) {
            a_local = true;  // own rows come straight from the tensor they were pushed from: nothing to wait for
          } else if (!(ag_ready & (1u << src))) {
            const uint64_t t0 = ptx::globaltimer();
            while (true) {
              uint32_t v;
              asm volatile("ld.acquire.sys.global.u32 %0, [%1];" : "=r"(v) : "l"(fuse.ag_flags + src) : "memory");
              if (static_cast<int32_t>(v - fuse.epoch) >= 0) { ag_ready |= 1u << src; break; }
              if (*abort_flag || ptx::globaltimer() - t0 > NTB_WAIT_LIMIT_NS) { *abort_flag = 1; ok = false; break; }
              __nanosleep(100);
            }
            if (!ok) break;
            // the block was written by peers with generic stores: make it visible to the async (TMA) proxy
            asm volatile("fence.proxy.async.global;" ::: "memory");
          }
        }
        for (int kb = un.kb0; kb < un.kb0 + un.kbs; kb++, it++) {
          const int s = it % P_STAGES;
          const uint32_t ph = (it / P_STAGES) & 1;
          if (!ptx::mbar_wait(&empty_bar[s], ph ^ 1, abort_flag, 200)) { ok = false; break; }
          uint8_t* sa = smem + s * STAGE;
          uint8_t* sb = sa + P_A_BYTES;
          if (cta == 0) {
            // the stage is free in both CTAs (the MMAs that read it are complete): tell the peer's producer, then expect both halves
            if (it >= P_STAGES) mbar_arrive_cluster_relaxed(map_to_cta(ptx::smem_u32(&empty_bar[s]), 1));
            ptx::mbar_expect_tx(&full_bar[s], stage_bytes);
          }
          const uint32_t fb = map_to_cta(ptx::smem_u32(&full_bar[s]), 0);  // bytes of both CTAs are counted on the leader's barrier
          if (A_MN) tma2_load_3d(sa, &tmap_a, fb, 0, kb * P_BLOCK_K, m0 / 64);
          else if (a_local) tma2_load_2d(sa, &tmap_al, fb, kb * P_BLOCK_K, m0 - fuse.me * fuse.ag_rows);
          else if (!a_none) tma2_load_2d(sa, &tmap_a, fb, kb * P_BLOCK_K, m0);
          if (B_MN) tma2_load_3d(sb, &tmap_b, fb, 0, kb * P_BLOCK_K, n0 / 64);
          else      tma2_load_2d(sb, &tmap_b, fb, kb * P_BLOCK_K, n0);
        }
      }
      if (!ok && cta == 1) {
        // this CTA's loads in flight are counted on the leader's barrier: give them time to land before the shared memory goes away
        const uint64_t t0 = ptx::globaltimer();
        while (ptx::globaltimer() - t0 < 100000ull) {}
      }
      if (!ok && cta == 0) {
        const uint64_t t0 = ptx::globaltimer();
        for (int s = 0; s < P_STAGES; s++) {
          const int last = it - 1 - ((it - 1 - s) % P_STAGES + P_STAGES) % P_STAGES;
          if (it == 0 || last < 0) continue;
          const uint32_t ph = (last / P_STAGES) & 1;
          while (!ptx::mbar_try_wait(&full_bar[s], ph) && ptx::globaltimer() - t0 < NTB_WAIT_LIMIT_NS) {}
        }
      }
    }
  } else if (warp == 1) {
    if (ptx::elect_one()) {
      if (cta == 0) {
        // ---------------------------------------------------------------- MMA issuer (leader)
        const uint32_t idesc = ptx::make_idesc_bf16(2 * P_BLOCK_M, block_n, A_MN, B_MN);
        int it = 0, tile_it = 0;
        bool ok = true;
        for (int u = pair; u < sched.total_units && ok; u += num_pairs) {
          const PUnit un = decode_unit(u, sched, k_blocks);
          if (un.kbs <= 0) continue;
          int kb = 0;
          do {  // one accumulator per tile; statistics: one per P_CE_SEGMENT k-blocks of a tile
            const int kb0 = kb, kb1 = p_ce_stats(OUT) ? min(kb + P_CE_SEGMENT, un.kbs) : un.kbs;
            const int acc = tile_it & 1;
            const uint32_t acc_ph = (tile_it >> 1) & 1;
            tile_it++;
            if (!ptx::mbar_wait(&tmem_empty[acc], acc_ph ^ 1, abort_flag)) { ok = false; break; }
            ptx::tc_fence_after();
            const uint32_t tmem_d = tmem_base + acc * P_BLOCK_N;
            for (; kb < kb1; kb++, it++) {
              const int s = it % P_STAGES;
              const uint32_t ph = (it / P_STAGES) & 1;
              if (!ptx::mbar_wait(&full_bar[s], ph, abort_flag)) { ok = false; break; }
              ptx::tc_fence_after();
              const uint32_t sa = ptx::smem_u32(smem + s * STAGE);
              const uint32_t sb = sa + P_A_BYTES;
#pragma unroll
              for (int k = 0; k < P_BLOCK_K / P_UMMA_K; k++) {
                const uint64_t adesc = A_MN ? ptx::make_smem_desc(sa + k * P_UMMA_K * 128, P_BLOCK_K * 128, 1024) : ptx::make_smem_desc(sa + k * P_UMMA_K * 2, 16, 1024);
                const uint64_t bdesc = B_MN ? ptx::make_smem_desc(sb + k * P_UMMA_K * 128, P_BLOCK_K * 128, 1024) : ptx::make_smem_desc(sb + k * P_UMMA_K * 2, 16, 1024);
                umma2_f16(tmem_d, adesc, bdesc, idesc, ((kb - kb0) | k) != 0 ? 1u : 0u);
              }
              umma2_commit(ptx::smem_u32(&empty_bar[s]));  // the stage is free once these MMAs (in both SMs) have read it
            }
            if (ok) umma2_commit(ptx::smem_u32(&tmem_full[acc]));
          } while (p_ce_stats(OUT) && ok && kb < un.kbs);
        }
      }
    }
  }
  } else {
    if constexpr (p_ce_stats(OUT)) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P_SPLIT_REGS_EPI));
    // ------------------------------------------------------------------ epilogue warps (both CTAs, own 128 rows)
    constexpr uint32_t POLL_NS = p_ce_stats(OUT) ? 100 : 1000;  // pieces of a tile follow one another in 4 us
    const int q = warp & 3;
    const int half = EW == 8 ? (warp - EPI0) >> 2 : 0;  // of the columns
    uint8_t* my_epi = epi_smem + (warp - EPI0) * 2 * P_EPI_BUF;
    constexpr bool BF16_OUT = (OUT == P_OUT_BF16 || OUT == P_OUT_PEER_BF16 || OUT == P_OUT_CE_GRAD);
    float alpha = 1.f;
    if constexpr (std::is_same_v<EXT, PAlpha>) alpha = ext.alpha ? *ext.alpha : 1.f;
    int tile_it = 0, buf = 0;
    bool ok = true;
    if constexpr (TURNED) {
      // A warp has 32 vocabulary entries (lanes) of up to 128 tokens (columns), always the same tokens: the grid is a multiple of the token
      // tiles.  Blocks of 32 x 32 scores are turned around in shared memory, so that a lane folds 32 scores of its own token into running
      // statistics that stay in registers until the CTA's last tile.
      constexpr int NB = EXT::BLOCKS;  // blocks of 32 columns; the second half of the warps may have one without tokens at its end
      const int n_blk = pair % tiles_n, c0 = half * NB * 32;
      float* turn = reinterpret_cast<float*>(epi_smem + (warp - EPI0) * P_EPI_BUF);
      float m[NB], s[NB];
      int tl[NB];  // the token's target among this product's rows, or far from any row
#pragma unroll
      for (int b = 0; b < NB; b++) {
        m[b] = -INFINITY;
        s[b] = 0.f;
        tl[b] = -(1 << 30);
        const int col = c0 + b * 32 + lane, token = n_blk * block_n + col;
        if (col < block_n && token < N) {
          const int64_t rel = ext.target[token] - ext.col0;
          if (rel >= 0 && rel < M) tl[b] = static_cast<int>(rel);
        }
      }
      auto hand_back = [&](int a) {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (cta == 0) ptx::mbar_arrive(&tmem_empty[a]);
          else mbar_arrive_cluster(map_to_cta(ptx::smem_u32(&tmem_empty[a]), 0));
        }
      };
      for (int u = pair; u < sched.total_units && ok; u += num_pairs) {
        const int row0 = (u / tiles_n * 2 + static_cast<int>(cta)) * P_BLOCK_M + q * 32;
        const int valid = M - row0;  // rows that exist: the others are zeros of the load
        auto fold = [&](int b, const uint32_t (&r)[32]) {
#pragma unroll
          for (int j = 0; j < 8; j++)
            *reinterpret_cast<uint4*>(turn + lane * 32 + ((j ^ (lane & 7)) << 2)) = make_uint4(r[j * 4], r[j * 4 + 1], r[j * 4 + 2], r[j * 4 + 3]);
          __syncwarp();
          auto at = [&](int i) { return turn + i * 32 + (((lane >> 2) ^ (i & 7)) << 2) + (lane & 3); };
          const int i = tl[b] - row0;
          if (i >= 0 && i < 32) ext.tgt[n_blk * block_n + c0 + b * 32 + lane] = *at(i);
#pragma unroll 1
          for (int h = 0; h < 32; h += 16) {
            uint32_t own[16];
#pragma unroll
            for (int i = 0; i < 16; i++) own[i] = __float_as_uint(*at(h + i));
            p_ce_accumulate(own, valid - h, m[b], s[b]);
          }
          __syncwarp();
        };
        uint32_t sums[NB][32];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int j = 0; j < 32; j++) sums[b][j] = 0u;
        for (int kb = 0; kb < k_blocks; kb += P_CE_SEGMENT) {
          const int a = tile_it & 1;
          if (!ptx::mbar_wait(&tmem_full[a], (tile_it >> 1) & 1, abort_flag, POLL_NS)) { ok = false; break; }
          tile_it++;
          if (cta == 0 && warp == EPI0 && lane == 0) mbar_arrive_cluster(map_to_cta(ptx::smem_u32(&tmem_full[a]), 1));  // forward to the peer's epilogue
          ptx::tc_fence_after();
          const uint32_t ta = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + a * P_BLOCK_N + c0;
#pragma unroll
          for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int c = 0; c < 4; c++) {
              uint32_t r0[8];
              ptx::tmem_ld_32x8(ta + b * 32 + c * 8, r0);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 8; j++) sums[b][c * 8 + j] = __float_as_uint(__uint_as_float(sums[b][c * 8 + j]) + __uint_as_float(r0[j]));
            }
          }
          hand_back(a);
        }
        if (!ok) break;
#pragma unroll
        for (int b = 0; b < NB; b++) fold(b, sums[b]);
      }
      // the four row groups of the CTA
      float2* all = reinterpret_cast<float2*>(epi_smem);  // [4][256]
      asm volatile("bar.sync 1, %0;" ::"n"(32 * EW) : "memory");
#pragma unroll
      for (int b = 0; b < NB; b++) all[q * 256 + c0 + b * 32 + lane] = make_float2(m[b], s[b]);
      asm volatile("bar.sync 1, %0;" ::"n"(32 * EW) : "memory");
      const int e = threadIdx.x - EPI0 * 32, token = n_blk * block_n + e;
      if (e < block_n && token < N) {
        float gm = -INFINITY, gs = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) gm = fmaxf(gm, all[i * 256 + e].x);
        const float base = gm == -INFINITY ? 0.f : gm * P_LOG2E;
#pragma unroll
        for (int i = 0; i < 4; i++) gs += all[i * 256 + e].y * p_ex2(fmaf(all[i * 256 + e].x, P_LOG2E, -base));
        ext.part[static_cast<int64_t>(pair / tiles_n * 2 + static_cast<int>(cta)) * N + token] = make_float2(gm, gs);
      }
    } else
    for (int u = pair; u < sched.total_units && ok; u += num_pairs) {
      const PUnit un = decode_unit(u, sched, k_blocks);
      if (un.kbs <= 0) continue;
      PTile tc = pair_tile(un.tile, tiles_m, tiles_n, band);
      tc.m_blk = (tc.m_blk + fuse.m_rot) % tiles_m;
      const int acc = tile_it & 1;
      const uint32_t acc_ph = (tile_it >> 1) & 1;
      tile_it++;
      // a chunk of a split tile leaves as fp32 partial sums in its workspace slab, whatever the type of D
      const bool to_ws = un.ws >= 0;
      const bool bf16_path = BF16_OUT && !to_ws;
      const int CHUNK_COLS = bf16_path ? 64 : 32;
      const int CHUNKS = P_BLOCK_N / CHUNK_COLS;
      if (!ptx::mbar_wait(&tmem_full[acc], acc_ph, abort_flag, POLL_NS)) { ok = false; break; }
      if (cta == 0 && warp == EPI0 && lane == 0) mbar_arrive_cluster(map_to_cta(ptx::smem_u32(&tmem_full[acc]), 1));  // forward to the peer's epilogue
      ptx::tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * P_BLOCK_N;
      const int row0 = (tc.m_blk * 2 + static_cast<int>(cta)) * P_BLOCK_M + q * 32;
      if constexpr (OUT == P_OUT_CE_STATS) {
        const int row = row0 + lane;
        const int cols = min(P_BLOCK_N, N - tc.n_blk * P_BLOCK_N);  // columns of this tile that exist: the others are zeros of the load
        int t = -1;  // the target's column in this tile, or -1
        if (row < M) {
          const int64_t rel = ext.target[row] - ext.col0 - static_cast<int64_t>(tc.n_blk) * P_BLOCK_N;
          if (rel >= 0 && rel < cols) t = static_cast<int>(rel);
        }
        constexpr int PARTS = EW / 4, PART_COLS = P_BLOCK_N / PARTS;
        const int c0 = half * PART_COLS;  // this warp's columns
        float m = -INFINITY, s = 0.f;
        auto hand_back = [&](int a) {  // to the leader's MMA thread (a remote arrive from the peer CTA)
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (cta == 0) ptx::mbar_arrive(&tmem_empty[a]);
            else mbar_arrive_cluster(map_to_cta(ptx::smem_u32(&tmem_empty[a]), 0));
          }
        };
        if (un.kbs <= P_CE_SEGMENT) {
#pragma unroll 1
          for (int c = c0; c < c0 + PART_COLS && c < cols; c += 32) {
            uint32_t r0[32];
            ptx::tmem_ld_32x32(taddr + c, r0);
            ptx::tmem_ld_wait();
            p_ce_accumulate(r0, cols - c, m, s);
            const int tj = t - c;
            if (__any_sync(0xffffffffu, tj >= 0 && tj < 32)) {  // rare: 32 rows against a whole vocabulary
#pragma unroll
              for (int j = 0; j < 32; j++)
                if (j == tj) ext.tgt[row] = __uint_as_float(r0[j]);
            }
          }
          hand_back(acc);
        } else {
          // several accumulators: their sum is built in registers, eight columns at a time, and each goes back as soon as it is read
          uint32_t sums[PART_COLS / 8][8];
          int a = acc;
          for (int kb = P_CE_SEGMENT;; kb += P_CE_SEGMENT) {
            const uint32_t ta = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + a * P_BLOCK_N + c0;
            const bool first = kb == P_CE_SEGMENT;
#pragma unroll
            for (int c = 0; c < PART_COLS / 8; c++) {
              uint32_t r0[8];
              ptx::tmem_ld_32x8(ta + c * 8, r0);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 8; j++) sums[c][j] = first ? r0[j] : __float_as_uint(__uint_as_float(sums[c][j]) + __uint_as_float(r0[j]));
            }
            hand_back(a);
            if (kb >= un.kbs) break;
            a = tile_it & 1;
            if (!ptx::mbar_wait(&tmem_full[a], (tile_it >> 1) & 1, abort_flag, POLL_NS)) { ok = false; break; }
            tile_it++;
            if (cta == 0 && warp == EPI0 && lane == 0) mbar_arrive_cluster(map_to_cta(ptx::smem_u32(&tmem_full[a]), 1));
            ptx::tc_fence_after();
          }
          if (!ok) break;
#pragma unroll
          for (int c = 0; c < PART_COLS / 8; c++) {
            if (c0 + c * 8 < cols) {
              p_ce_accumulate(sums[c], cols - c0 - c * 8, m, s);
              const int tj = t - c0 - c * 8;
              if (__any_sync(0xffffffffu, tj >= 0 && tj < 8)) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                  if (j == tj) ext.tgt[row] = __uint_as_float(sums[c][j]);
              }
            }
          }
        }
        if (row < M) ext.part[static_cast<int64_t>(tc.n_blk * PARTS + half) * M + row] = make_float2(m, s);
      } else {
      float ce_lz = 0.f, ce_coef = 0.f, ce_g = 0.f;
      int ce_t = -1, ce_cols = 0;
      if constexpr (OUT == P_OUT_CE_GRAD) {
        const int row = row0 + lane;
        ce_cols = min(P_BLOCK_N, N - tc.n_blk * P_BLOCK_N);
        if (row < M) {
          ce_lz = ext.logz[row] * P_LOG2E;
          ce_coef = ext.coef[row];
          ce_g = ext.g[row];
          const int64_t rel = ext.target[row] - ext.col0 - static_cast<int64_t>(tc.n_blk) * P_BLOCK_N;
          if (rel >= 0 && rel < ce_cols) ce_t = static_cast<int>(rel);
        }
      }
#pragma unroll 1
      for (int c = EW == 8 ? half * (CHUNKS / 2) : 0; c < (EW == 8 ? (half + 1) * (CHUNKS / 2) : CHUNKS); c++) {
        uint8_t* stage_buf = my_epi + buf * P_EPI_BUF;
        if (lane == 0) ptx::tma_wait_group_read<1>();
        __syncwarp();
        uint8_t* my_row = stage_buf + lane * 128;
        if (bf16_path) {
          uint32_t r0[32], r1[32];
          ptx::tmem_ld_32x32(taddr + c * 64, r0);
          ptx::tmem_ld_32x32(taddr + c * 64 + 32, r1);
          ptx::tmem_ld_wait();
          if constexpr (OUT == P_OUT_CE_GRAD) {
            p_ce_gradient(r0, ce_cols - c * 64, ce_t - c * 64, ce_lz, ce_coef, ce_g);
            p_ce_gradient(r1, ce_cols - c * 64 - 32, ce_t - c * 64 - 32, ce_lz, ce_coef, ce_g);
          }
          if constexpr (std::is_same_v<EXT, PAlpha>) {
#pragma unroll
            for (int j = 0; j < 32; j++) {
              r0[j] = __float_as_uint(__uint_as_float(r0[j]) * alpha);
              r1[j] = __float_as_uint(__uint_as_float(r1[j]) * alpha);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const uint32_t* src = (j < 4) ? &r0[j * 8] : &r1[(j - 4) * 8];
            uint4 pk;
            __nv_bfloat162 h0 = __floats2bfloat162_rn(__uint_as_float(src[0]), __uint_as_float(src[1]));
            __nv_bfloat162 h1 = __floats2bfloat162_rn(__uint_as_float(src[2]), __uint_as_float(src[3]));
            __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(src[4]), __uint_as_float(src[5]));
            __nv_bfloat162 h3 = __floats2bfloat162_rn(__uint_as_float(src[6]), __uint_as_float(src[7]));
            pk.x = *reinterpret_cast<uint32_t*>(&h0);
            pk.y = *reinterpret_cast<uint32_t*>(&h1);
            pk.z = *reinterpret_cast<uint32_t*>(&h2);
            pk.w = *reinterpret_cast<uint32_t*>(&h3);
            *reinterpret_cast<uint4*>(my_row + ((j ^ (lane & 7)) << 4)) = pk;
          }
        } else {
          uint32_t r0[32];
          ptx::tmem_ld_32x32(taddr + c * 32, r0);
          ptx::tmem_ld_wait();
          if constexpr (std::is_same_v<EXT, PAlpha>) {
            if (!to_ws) {  // a chunk of a split tile is scaled once, when the chunks are summed
#pragma unroll
              for (int j = 0; j < 32; j++) r0[j] = __float_as_uint(__uint_as_float(r0[j]) * alpha);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; j++) {
            uint4 pk = make_uint4(r0[j * 4], r0[j * 4 + 1], r0[j * 4 + 2], r0[j * 4 + 3]);
            *reinterpret_cast<uint4*>(my_row + ((j ^ (lane & 7)) << 4)) = pk;
          }
        }
        ptx::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          const int x = tc.n_blk * P_BLOCK_N + c * CHUNK_COLS;
          if (to_ws) {
            ptx::tma_store_2d(&tmap_ws, stage_buf, c * 32, un.ws * (2 * P_BLOCK_M) + static_cast<int>(cta) * P_BLOCK_M + q * 32);
          } else if (x < N && row0 < M) {
            if (OUT == P_OUT_PEER_BF16) {
              const int owner = row0 / fuse.rs_rows;  // rs_rows is a multiple of 32: the 32 rows of this warp share an owner
              ptx::tma_store_2d(&pmaps.m[owner], stage_buf, x, fuse.me * fuse.rs_rows + (row0 - owner * fuse.rs_rows));
            } else if (OUT == P_OUT_F32_ACCUM) ptx::tma_reduce_add_2d(&tmap_d, stage_buf, x, row0);
            else ptx::tma_store_2d(&tmap_d, stage_buf, x, row0);
          }
          ptx::tma_commit_group();
        }
        buf ^= 1;
      }
      }
      if constexpr (!p_ce_stats(OUT)) {
        // accumulator fully read: hand it back to the leader's MMA thread (a remote arrive from the peer CTA)
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (cta == 0) ptx::mbar_arrive(&tmem_empty[acc]);
          else mbar_arrive_cluster(map_to_cta(ptx::smem_u32(&tmem_empty[acc]), 0));
        }
      }
    }
    if (lane == 0) {
      ptx::tma_wait_group<0>();
      if (OUT == P_OUT_PEER_BF16) {
        // the peer stores were made by the async proxy: order them before the generic-proxy flag store that follows the CTA barrier
        asm volatile("fence.proxy.async.global;" ::: "memory");
        __threadfence_system();
      }
    }
    __syncwarp();
  }

  ptx::tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the leader's MMAs write the peer's TMEM and read its shared memory: nobody leaves or frees before both are done
  if (warp == 1) {
    ptx::tc_fence_after();
    tmem_dealloc2(tmem_base, 512);
  }
  if (OUT == P_OUT_PEER_BF16 && fuse.done_counter != nullptr && threadIdx.x == 0) {
    // every store of this CTA is complete and fenced (epilogue warps, before the barrier above); the last CTA of the grid to get
    // here tells every owner that this rank's partial sums are in place
    __threadfence_system();
    const unsigned int prev = atomicAdd(fuse.done_counter, 1u);
    if (prev == gridDim.x - 1) {
      __threadfence_system();
      for (int r = 0; r < fuse.world; r++)
        asm volatile("st.release.sys.global.u32 [%0], %1;" ::"l"(fuse.rs_flags[r] + fuse.me), "r"(fuse.epoch) : "memory");
      *fuse.done_counter = 0;
    }
  }
  if (threadIdx.x == 0 && *abort_flag && status) atomicExch(status, NTB_ERR_TIMEOUT);
}

// Split tiles: D tile = (D tile +) the sum, in chunk order, of the tile's workspace slabs (256 x 256 fp32 each, complete once the
// GEMM kernel has finished).  One block per split tile and 32-row group.  OUT as in the GEMM kernel.
template <int OUT>
__global__ void gemm2_split_fixup_kernel(const float* __restrict__ ws, void* __restrict__ d_, int64_t ldd, int M, int N, int k_blocks, PSched sched, int tiles_m,
                                         int tiles_n, int band, int m_rot) {
  const int rt = blockIdx.x >> 3, rg = blockIdx.x & 7;
  PTile tc = pair_tile(sched.full_units + rt, tiles_m, tiles_n, band);
  tc.m_blk = (tc.m_blk + m_rot) % tiles_m;
  const int chunks = min(sched.split, (k_blocks + sched.kb_per - 1) / sched.kb_per);  // chunks past the end of K wrote nothing
  const int64_t slab = static_cast<int64_t>(2 * P_BLOCK_M) * P_BLOCK_N;
  const float* src = ws + static_cast<int64_t>(rt) * sched.split * slab + static_cast<int64_t>(rg) * 32 * P_BLOCK_N;
  for (int i = threadIdx.x; i < 32 * P_BLOCK_N / 8; i += blockDim.x) {
    const int r = i / (P_BLOCK_N / 8), c8 = (i % (P_BLOCK_N / 8)) * 8;
    const int row = tc.m_blk * 2 * P_BLOCK_M + rg * 32 + r, col = tc.n_blk * P_BLOCK_N + c8;
    if (row >= M || col >= N) continue;  // N is a multiple of 8 and rows of D start 16-byte aligned (checked by the host)
    float f[8];
    if (OUT == P_OUT_F32_ACCUM) {
      const float* dp = reinterpret_cast<const float*>(d_) + static_cast<int64_t>(row) * ldd + col;
      *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(dp);
      *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(dp + 4);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = 0.f;
    }
    for (int ch = 0; ch < chunks; ch++) {
      const float* p = src + ch * slab + r * P_BLOCK_N + c8;
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w;
      f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
    }
    if (OUT == P_OUT_BF16) {
      Vec8<__nv_bfloat16> o;
      o.from_float(f);
      o.store(reinterpret_cast<__nv_bfloat16*>(d_) + static_cast<int64_t>(row) * ldd + col);
    } else {
      float* dp = reinterpret_cast<float*>(d_) + static_cast<int64_t>(row) * ldd + col;
      *reinterpret_cast<float4*>(dp) = *reinterpret_cast<float4*>(f);
      *reinterpret_cast<float4*>(dp + 4) = *reinterpret_cast<float4*>(f + 4);
    }
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn p_get_encode() {
  ntb_bind_context_to_thread();
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

bool p_map_kmajor(CUtensorMap* m, const void* ptr, int64_t rows, int64_t k, int64_t ld, int box_rows = P_BLOCK_M) {
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1, 1};
  return p_get_encode()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool p_map_mnmajor(CUtensorMap* m, const void* ptr, int64_t mn, int64_t k, int64_t ld) {
  cuuint64_t dims[3] = {64, (cuuint64_t)k, (cuuint64_t)((mn + 63) / 64)};
  cuuint64_t strides[2] = {(cuuint64_t)ld * 2, 128};
  cuuint32_t box[3] = {64, (cuuint32_t)P_BLOCK_K, 2};
  cuuint32_t es[3] = {1, 1, 1};
  return p_get_encode()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool p_map_out(CUtensorMap* m, void* ptr, int64_t rows, int64_t cols, int64_t ld, bool f32) {
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * (f32 ? 4 : 2)};
  cuuint32_t box[2] = {(cuuint32_t)(f32 ? 32 : 64), 32};
  cuuint32_t es[2] = {1, 1};
  return p_get_encode()(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
