// Cross entropy of a linear head without its logits (sm_100a).
//
//   l[t,v] = sum_h x[t,h] w[v,h]      logZ[t] = log sum_v exp l[t,v]      loss[t] = logZ[t] - l[t, y_t]
//   d[t,v] = coef[t] exp(l[t,v] - logZ[t]) - g[t] [v == y_t]             dx = d w        dw = d^T x
//
// Forward: one GEMM over the whole vocabulary on CTA pairs (gemm2_core.cuh) whose epilogue keeps, per token and 256-column tile, only
// (largest score, sum of exponentials); a small kernel joins the half tiles of a token.  With few tokens the operands change places (up to
// 1024, see ce_turned_tile) or the weight is only streamed (up to 8, ce_few_kernel).  Scores never leave the tensor memory, and they
// are used in fp32 (logits written in bf16 are off by up to 2^-8 of their value, several percent of a probability).  They are accumulated
// 1024 products at a time and the pieces added in registers, because the tensor cores cut when they add to an accumulator: a score comes
// out small by 1e-6 of its value at any H (in one accumulator by 9e-10 H), the loss of scores with a standard deviation of 1.5 by 3e-7 (in
// one accumulator 1.1e-6 at H = 4096, 2.4e-6 at 8192).  That takes 1 .. 3 % of the forward pass.
// Backward: the vocabulary is cut into pieces; for each piece the scores are computed again, the epilogue turns them into d (bf16,
// one rounding), and two plain products take d to dx (summed over the pieces in fp32) and to the piece's rows of dw.  Only one
// piece of d is alive.  d is kept in units of the largest |g| (`ce_row_coefficients`) and the products are scaled back by that one
// number in fp32: with a masked mean every g is the same number, and rounding -g (1 - p) to bf16 would shift the dominant entry of
// every row by the same relative amount (up to 2^-8), an error that no summation averages out; in units of g it is -(1 - p).
#include "gemm2_core.cuh"

namespace {

constexpr int CE_JOIN_ROWS = 32;
constexpr int CE_JOIN_PARTS = 16;

// One block per 32 tokens; 16 groups of threads share the tiles of a token.  Reads of `part` are contiguous over the tokens.
__global__ void __launch_bounds__(CE_JOIN_ROWS * CE_JOIN_PARTS)
ce_join_kernel(const float2* __restrict__ part, const float* __restrict__ tgt, const int64_t* __restrict__ target, int64_t vocab_start, int vocab, int tiles,
               int rows, float* __restrict__ out_max, float* __restrict__ out_sum, float* __restrict__ out_tgt, float* __restrict__ logz,
               float* __restrict__ loss, float* __restrict__ z, float z_coef) {
  __shared__ float sm[CE_JOIN_PARTS][CE_JOIN_ROWS], ss[CE_JOIN_PARTS][CE_JOIN_ROWS];
  p_wait_for_previous();
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int row = blockIdx.x * CE_JOIN_ROWS + lane;
  float m = -INFINITY, s = 0.f;
  if (row < rows) {
    for (int i = grp; i < tiles; i += CE_JOIN_PARTS) {
      const float2 p = part[static_cast<int64_t>(i) * rows + row];
      const float nm = fmaxf(m, p.x);
      const float base = nm == -INFINITY ? 0.f : nm * P_LOG2E;
      s = s * p_ex2(fmaf(m, P_LOG2E, -base)) + p.y * p_ex2(fmaf(p.x, P_LOG2E, -base));
      m = nm;
    }
  }
  sm[grp][lane] = m;
  ss[grp][lane] = s;
  __syncthreads();
  if (grp != 0 || row >= rows) return;
  float gm = -INFINITY, gs = 0.f;
#pragma unroll
  for (int i = 0; i < CE_JOIN_PARTS; i++) gm = fmaxf(gm, sm[i][lane]);
  const float base = gm == -INFINITY ? 0.f : gm * P_LOG2E;
#pragma unroll
  for (int i = 0; i < CE_JOIN_PARTS; i++) gs += ss[i][lane] * p_ex2(fmaf(sm[i][lane], P_LOG2E, -base));
  const int64_t rel = target[row] - vocab_start;
  const float t = (rel >= 0 && rel < vocab) ? tgt[row] : 0.f;
  if (out_max != nullptr) {
    out_max[row] = gm;
    out_sum[row] = gs;
    out_tgt[row] = t;
  }
  if (logz != nullptr) {
    const float lz = gm + logf(gs);
    logz[row] = lz;
    loss[row] = lz - t;
    if (z != nullptr) z[row] = z_coef * (lz * lz);
  }
}

// coef = (g + 2 z_coef logz gz) / unit, g = g / unit with unit = the largest |g| or |g + 2 z_coef logz gz| (1 where that is no use as a
// divisor).  One block: a reduction over the tokens, then a second look at values that are in the cache.
__global__ void __launch_bounds__(1024) ce_row_coefficients_kernel(const float* __restrict__ g, const float* __restrict__ gz, const float* __restrict__ logz, float z_coef,
                                                                    int rows, float* __restrict__ coef, float* __restrict__ gn, float* __restrict__ unit) {
  __shared__ float scratch[32];
  float m = 0.f;
  for (int i = threadIdx.x; i < rows; i += blockDim.x) m = fmaxf(m, fmaxf(fabsf(g[i]), gz ? fabsf(g[i] + 2.f * z_coef * logz[i] * gz[i]) : 0.f));
  m = block_max(m, scratch);
  const float u = (m > 1e-30f && m < 1e30f) ? m : 1.f;
  if (threadIdx.x == 0) *unit = u;
  for (int i = threadIdx.x; i < rows; i += blockDim.x) {
    coef[i] = (gz ? g[i] + 2.f * z_coef * logz[i] * gz[i] : g[i]) / u;
    gn[i] = g[i] / u;
  }
}

// out = bf16(*unit * acc), eight elements a thread.
__global__ void __launch_bounds__(256) ce_scale_cast_kernel(const float* __restrict__ acc, const float* __restrict__ unit, __nv_bfloat16* __restrict__ out, int64_t n8) {
  p_wait_for_previous();
  const float u = *unit;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n8; i += static_cast<int64_t>(gridDim.x) * 256) {
    Vec8<float> a;
    float f[8];
    a.load(acc + i * 8);
    a.to_float(f);
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] *= u;
    Vec8<__nv_bfloat16> o;
    o.from_float(f);
    o.store(out + i * 8);
  }
}

// ------------------------------------------------------------------------------------------------ a few tokens
// Scores of up to 8 tokens: the work is reading the weight once.  A CTA takes 32 whole rows at a time, one contiguous piece of the weight,
// and neighbouring CTAs neighbouring pieces; the 64-column blocks of the rows are dealt to eight warps, each with a ring of TMA loads of
// its own, so no warp waits for another but at the end of the 32 rows.  1 x 2048 x 128256: 85 us, 6.2 TB/s; blocks of
// 16 rows took 129 us, bound by the turn of a warp's loop (wait, read, four dependent products, next load) rather than by memory.
//
// With so few tokens the products are small: mma.sync m16n8k16, 16 weight rows x 8 tokens (bound by the
// loads, not by this tensor path).  A lane reads 16 consecutive columns of a row
// as two 16-byte words and feeds them to four products; the columns of a product are then a permutation of the block's, the same one
// for weight and tokens, which a sum over columns does not see.  With the 128-byte swizzle of the loads these reads are free of bank
// conflicts (lane t of a row takes words 2t, 2t + 1; eight lanes cover two rows and, after the swizzle, all eight word columns).
constexpr int FEW_WARPS = 8;
constexpr int FEW_ROWS = 32;
constexpr int FEW_SLOT = FEW_ROWS * 128;  // bytes of one 32 x 64 block
constexpr int FEW_TOKENS = 8;
constexpr int FEW_MAX_STAGES = 8;
constexpr int FEW_SMEM = 227 * 1024;

struct FewLayout {  // of the dynamic shared memory, from a 1024-byte boundary on
  int x_bytes, red_bytes, stages;
};
// Partial sums of the warps go through two buffers (one CTA barrier per 32 rows).
__host__ __device__ inline FewLayout few_layout(int k_blocks) {
  FewLayout l;
  l.x_bytes = k_blocks * FEW_TOKENS * 128;
  l.red_bytes = 2 * FEW_WARPS * FEW_ROWS * FEW_TOKENS * 4;
  const int left = FEW_SMEM - 2048 - l.x_bytes - l.red_bytes;
  l.stages = left / (FEW_WARPS * FEW_SLOT);
  if (l.stages > FEW_MAX_STAGES) l.stages = FEW_MAX_STAGES;
  return l;
}

__device__ __forceinline__ void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16-byte word `word` of row `row` of a block whose rows are 128 bytes, swizzled by the load
__device__ __forceinline__ uint4 few_word(const uint8_t* block, int row, int word) {
  return *reinterpret_cast<const uint4*>(block + row * 128 + ((word ^ (row & 7)) << 4));
}

// GRAD false: part[blockIdx.x][T] = (largest, sum of exponentials) of the rows this CTA saw, and the targets' scores.  GRAD true:
// d [T, V] at pitch ldd, columns up to `width` written.
template <bool GRAD>
__global__ void __launch_bounds__(FEW_WARPS * 32, 1)
ce_few_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, int T, int V, int k_blocks, PCeArgs args, __nv_bfloat16* __restrict__ d,
              int64_t ldd, int width, int* __restrict__ status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const FewLayout lay = few_layout(k_blocks);
  uint8_t* xs = smem;
  uint8_t* ring = xs + lay.x_bytes;
  float* red = reinterpret_cast<float*>(ring + lay.stages * FEW_WARPS * FEW_SLOT);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(red) + lay.red_bytes);  // [0]: tokens; then [warp][stage]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 1 + FEW_WARPS * FEW_MAX_STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int groups = ((GRAD ? width : V) + FEW_ROWS - 1) / FEW_ROWS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 1 + FEW_WARPS * FEW_MAX_STAGES; i++) ptx::mbar_init(&bars[i], 1);
    *abort_flag = 0;
    ptx::fence_barrier_init();
  }
  p_wait_for_previous();
  __syncthreads();
  if (threadIdx.x == 0) {
    ptx::mbar_expect_tx(&bars[0], lay.x_bytes);
    for (int kb = 0; kb < k_blocks; kb++) ptx::tma_load_2d(xs + kb * FEW_TOKENS * 128, &tmap_x, &bars[0], kb * 64, 0);
  }
  // this warp's blocks, in order: for each of the CTA's groups, blocks warp, warp + 8, ...
  const int per_group = k_blocks > warp ? (k_blocks - warp + FEW_WARPS - 1) / FEW_WARPS : 0;
  const int my_groups = groups > static_cast<int>(blockIdx.x) ? (groups - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x) : 0;
  const int total = per_group * my_groups;
  uint64_t* my_bars = bars + 1 + warp * FEW_MAX_STAGES;
  uint8_t* my_ring = ring + warp * lay.stages * FEW_SLOT;
  int next = 0, next_slot = 0, next_kb = warp, next_group = blockIdx.x;  // the next block to load (lane 0)
  auto issue = [&]() {
    ptx::mbar_expect_tx(&my_bars[next_slot], FEW_SLOT);
    ptx::tma_load_2d(my_ring + next_slot * FEW_SLOT, &tmap_w, &my_bars[next_slot], next_kb * 64, next_group * FEW_ROWS);
    next++;
    if (++next_slot == lay.stages) next_slot = 0;
    next_kb += FEW_WARPS;
    if (next_kb >= k_blocks) next_kb = warp, next_group += gridDim.x;
  };
  if (lane == 0)
    while (next < total && next < lay.stages) issue();
  bool ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars[0], 0, abort_flag));

  // the epilogue gives every thread one of the 32 x 8 scores: a warp has the 32 rows of a token
  static_assert(FEW_WARPS == FEW_TOKENS && FEW_ROWS == 32, "threads of the epilogue");
  const int token = warp;
  float run_m = -INFINITY, run_s = 0.f, e_lz = 0.f, e_coef = 0.f, e_g = 0.f;
  int e_t = -1;
  if (token < T) {
    const int64_t rel = args.target[token] - args.col0;
    if (rel >= 0 && rel < V) e_t = static_cast<int>(rel);
    if (GRAD) {
      e_lz = args.logz[token] * P_LOG2E;
      e_coef = args.coef[token];
      e_g = args.g[token];
    }
  }

  int slot = 0, buf = 0;
  uint32_t phase = 0;
  for (int group = blockIdx.x; group < groups; group += gridDim.x) {
    float acc[2][4];
#pragma unroll
    for (int j = 0; j < 4; j++) acc[0][j] = acc[1][j] = 0.f;
    for (int kb = warp; kb < k_blocks && ok; kb += FEW_WARPS) {
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&my_bars[slot], phase, abort_flag))) { ok = false; break; }
      const uint8_t* blk = my_ring + slot * FEW_SLOT;
      uint4 w[2][4];  // [rows 0..15 | 16..31][row g: words 2t, 2t + 1; row g + 8: the same]
#pragma unroll
      for (int m = 0; m < 2; m++) {
        w[m][0] = few_word(blk, m * 16 + g, 2 * t);
        w[m][1] = few_word(blk, m * 16 + g, 2 * t + 1);
        w[m][2] = few_word(blk, m * 16 + g + 8, 2 * t);
        w[m][3] = few_word(blk, m * 16 + g + 8, 2 * t + 1);
      }
      const uint8_t* xb = xs + kb * FEW_TOKENS * 128;
      const uint4 b0 = few_word(xb, g, 2 * t), b1 = few_word(xb, g, 2 * t + 1);
#pragma unroll
      for (int m = 0; m < 2; m++) few_mma(acc[m], w[m][0].x, w[m][2].x, w[m][0].y, w[m][2].y, b0.x, b0.y);
#pragma unroll
      for (int m = 0; m < 2; m++) few_mma(acc[m], w[m][0].z, w[m][2].z, w[m][0].w, w[m][2].w, b0.z, b0.w);
#pragma unroll
      for (int m = 0; m < 2; m++) few_mma(acc[m], w[m][1].x, w[m][3].x, w[m][1].y, w[m][3].y, b1.x, b1.y);
#pragma unroll
      for (int m = 0; m < 2; m++) few_mma(acc[m], w[m][1].z, w[m][3].z, w[m][1].w, w[m][3].w, b1.z, b1.w);
      __syncwarp();  // every lane's reads of the block have been consumed by the products above
      if (lane == 0 && next < total) issue();
      if (++slot == lay.stages) slot = 0, phase ^= 1;
    }
    // the warps' shares of the 32 x 8 scores, [token][row]
    float* out = red + (buf * FEW_WARPS + warp) * FEW_ROWS * FEW_TOKENS;
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
      for (int j = 0; j < 4; j++) out[(2 * t + (j & 1)) * FEW_ROWS + m * 16 + g + (j & 2) * 4] = acc[m][j];
    if (__syncthreads_or(!ok)) {  // the same answer in every thread
      ok = false;
      break;
    }
    if (token < T) {
      const int v = group * FEW_ROWS + lane;
      float sc = 0.f;
#pragma unroll
      for (int w = 0; w < FEW_WARPS; w++) sc += red[(buf * FEW_WARPS + w) * FEW_ROWS * FEW_TOKENS + threadIdx.x];
      if (GRAD) {
        if (v < width) {
          float p = v < V ? e_coef * p_ex2(fmaf(sc, P_LOG2E, -e_lz)) : 0.f;
          if (v == e_t) p -= e_g;
          d[token * ldd + v] = __float2bfloat16_rn(p);
        }
      } else if (v < V) {
        if (v == e_t) args.tgt[token] = sc;
        const float nm = fmaxf(run_m, sc);
        const float base = nm == -INFINITY ? 0.f : nm * P_LOG2E;
        run_s = run_s * p_ex2(fmaf(run_m, P_LOG2E, -base)) + p_ex2(fmaf(sc, P_LOG2E, -base));
        run_m = nm;
      }
    }
    buf ^= 1;
  }
  if (!ok) {  // leave no load in flight behind (bounded)
    if (lane == 0) {
      const uint64_t t0 = ptx::globaltimer();
      for (int j = next > lay.stages ? next - lay.stages : 0; j < next; j++)
        while (!ptx::mbar_try_wait(&my_bars[j % lay.stages], (j / lay.stages) & 1) && ptx::globaltimer() - t0 < NTB_WAIT_LIMIT_NS) {}
      if (warp == 0)
        while (!ptx::mbar_try_wait(&bars[0], 0) && ptx::globaltimer() - t0 < NTB_WAIT_LIMIT_NS) {}
    }
    if (threadIdx.x == 0 && status) atomicExch(status, NTB_ERR_TIMEOUT);
    return;
  }
  if (!GRAD) {
    float m = run_m, s = run_s;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, k), os = __shfl_xor_sync(0xffffffffu, s, k);
      const float nm = fmaxf(m, om);
      const float base = nm == -INFINITY ? 0.f : nm * P_LOG2E;
      s = s * p_ex2(fmaf(m, P_LOG2E, -base)) + os * p_ex2(fmaf(om, P_LOG2E, -base));
      m = nm;
    }
    if (lane == 0 && token < T) args.part[static_cast<int64_t>(blockIdx.x) * T + token] = make_float2(m, s);
  }
}

// Launches a kernel that starts with `p_wait_for_previous`: it may be set up while the kernel before it in the stream runs out (saves 1 to 2 us
// between two kernels of an eager call).  Only behind a kernel that the same entry point has launched: what came before that one is
// complete by then.
template <class... P, class... A>
int ce_launch_next(void (*kern)(P...), int64_t grid, int block, int smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(block), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...) != cudaSuccess) {
    cudaGetLastError();
    return NTB_ERR_LAUNCH;
  }
  return ntb_check_launch();
}

template <class K>
int ce_configure(K kern, bool (&done)[64], int smem) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NTB_ERR_LAUNCH;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
      cudaGetLastError();
      return NTB_ERR_LAUNCH;
    }
    done[dev] = true;
  }
  return NTB_OK;
}

int ce_band(int M, int K) {
  const int tiles_m = (M + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M);
  int band = static_cast<int>(40000000ll / (512ll * K));  // rows of A that stay in L2 while B streams: about 40 MB
  if (band < 2) band = 2;
  return band > tiles_m ? tiles_m : band;
}

// The epilogues that take an exponential per score get eight warps; with a short product four of them are what a tile waits for.  Four |
// eight warps, us: statistics of 2048 x 256 x 32000 60 | 51, 2047 x 768 x 50257 115 | 109; gradient (one operand stage less) 72 | 59, 127 |
// 123; level from H = 1024 on.  The plain products' epilogues gain nothing and keep four.
constexpr int CE_WARPS = 8;

template <bool A_MN, bool B_MN, int OUT, int ST = 0, class EXT>
int ce_launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& td, int M, int N, int K, const PSched& sched, const CUtensorMap& tws, const EXT& ext,
              int* status, int num_sms, cudaStream_t stream) {
  constexpr int EW = p_ce_stats(OUT) || OUT == P_OUT_CE_GRAD ? CE_WARPS : P_EPI_WARPS;
  constexpr int STAGES = ST ? ST : OUT == P_OUT_CE_GRAD ? P_MAX_STAGES - 1 : P_MAX_STAGES;
  auto kern = gemm2_tcgen05_kernel<A_MN, B_MN, OUT, STAGES, EXT, EW>;
  static bool done[64] = {};
  if (int rc = ce_configure(kern, done, P_SMEM)) return rc;
  if (p_ce_stats(OUT)) {  // its warp groups exchange registers: the block has to be launched with as many as they share out
    static int regs = -1;
    if (regs < 0) {
      cudaFuncAttributes fa;
      if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess) return NTB_ERR_LAUNCH;
      regs = fa.numRegs;
    }
    if (regs < P_SPLIT_REGS) return NTB_ERR_LAUNCH;
  }
  static const PPeerMaps no_maps = {};
  int pairs = num_sms / 2;
  if (sched.total_units < pairs) pairs = sched.total_units;
  if constexpr (OUT == P_OUT_CE_STATS_T) pairs = pairs / ((N + ext.tile_n - 1) / ext.tile_n) * ((N + ext.tile_n - 1) / ext.tile_n);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs), 1, 1);
  cfg.blockDim = dim3(p_threads(OUT, EW), 1, 1);
  cfg.dynamicSmemBytes = P_SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see ce_launch_next
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p_ce_stats(OUT) ? 1 : 2;  // the statistics are their entry point's first kernel
  if (cudaLaunchKernelEx(&cfg, kern, ta, tb, td, M, N, K, ce_band(M, K), status, PFuse(), no_maps, sched, tws, ta, ext) != cudaSuccess) {
    cudaGetLastError();
    return NTB_ERR_LAUNCH;
  }
  return ntb_check_launch();
}

PSched ce_whole_tiles(int M, int N, int K, bool& fits) {
  const long long tiles = static_cast<long long>((M + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M)) * ((N + P_BLOCK_N - 1) / P_BLOCK_N);
  fits = tiles < (1ll << 30);
  PSched sc;
  sc.total_units = sc.full_units = static_cast<int>(tiles);
  sc.split = 1;
  sc.kb_per = (K + P_BLOCK_K - 1) / P_BLOCK_K;
  return sc;
}

// Whether the few-token kernel takes the call.  The tokens' padded copy takes shared memory from the rings.  Forward pass, us, this kernel | the turned
// product (ce_turned_tile): 1 x 256 x 32000 10 | 12, 1 x 2048 x 128256 85 | 89, 8 x 4096 x 128256 161 | 175, 1 x 8192 x 128256 367 | 338.
bool ce_few(int T, int H) { return T <= FEW_TOKENS && H <= 4096; }

// Rows of a load of the tokens: no more than there are, in steps of the swizzle's 8 rows.  A load fills rows past the end with zeros, but
// slowly: gradient of the scores, us, loads of 128 rows | of the tokens: 17 x 1024 x 128256 61 | 56, 17 x 2048 x 128256 109 | 98, level from 64
// tokens on.  What is not loaded has to be zero all the same: leftovers in its place took 4 % (power, not work).
int ce_a_rows(int T) { return T < P_BLOCK_M ? (T + 7) / 8 * 8 : P_BLOCK_M; }

bool few_map(CUtensorMap* m, const void* ptr, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1, 1};
  return p_get_encode()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int few_grid(int rows, int num_sms) {
  const int groups = (rows + FEW_ROWS - 1) / FEW_ROWS;
  return groups < num_sms ? groups : num_sms;
}

template <bool GRAD>
int few_launch(const void* x, int64_t ldx, const void* w, int64_t ldw, int T, int V, int H, const PCeArgs& a, void* d, int64_t ldd, int width, int* status, int num_sms,
               cudaStream_t stream) {
  auto kern = ce_few_kernel<GRAD>;
  static bool done[64] = {};
  if (int rc = ce_configure(kern, done, FEW_SMEM)) return rc;
  CUtensorMap tx, tw;
  if (!few_map(&tx, x, T, H, ldx, FEW_TOKENS) || !few_map(&tw, w, V, H, ldw, FEW_ROWS)) return NTB_ERR_ARG;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(d);
  if (GRAD) return ce_launch_next(kern, few_grid(width, num_sms), FEW_WARPS * 32, FEW_SMEM, stream, tx, tw, T, V, H / 64, a, out, ldd, width, status);
  kern<<<few_grid(V, num_sms), FEW_WARPS * 32, FEW_SMEM, stream>>>(tx, tw, T, V, H / 64, a, out, ldd, width, status);
  return ntb_check_launch();
}

bool ce_operand_ok(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 64 == 0; }

// Tokens per tile where the product is turned around (P_OUT_CE_STATS_T: weight rows in the place of A), 0: not turned.  A tile of the product as it
// stands has 256 tokens, empty rows and all; turned around its width is what there is, in steps of 32.  With up to 128 tokens that leaves the
// tensor cores half idle and room for two more stages of the weight, and the pass runs at the rate of the memory.  Forward pass, us, as it stands |
// turned: 32 x 1024 x 128256 66 | 49, 64 x 2048 x 128256 112 | 84 (6.25 TB/s), 128 x 4096 x 128256 211 | 175, 333 x 768 x 50257 39 | 36, 256 x 2048 x
// 128256 149 | 127, 448 x 2048 x 128256 260 | 211, 1024 x 2048 x 128256 448 | 423, 1024 x 8192 x 128256 1741 | 1686.  The epilogue does more for a
// score (it is turned back in shared memory), which wide tiles show where the products are short: 256 x 512 x 32000 18 | 20, 768 x 1024 x 128256
// 168 | 174.  Behind 1024 tokens the two are level at best (1536 x 4096 x 128256 1300 | 1304), and token tiles that do not divide the pairs leave
// some idle: 4096 x 2048 x 128256 1500 | 1700.
int ce_turned_tile(int T, int H, int num_sms) {
  const int tiles = (T + P_BLOCK_N - 1) / P_BLOCK_N;
  const int tile = ((T + tiles - 1) / tiles + 31) / 32 * 32;
  return T <= 1024 && tiles <= num_sms / 2 && (tile <= 192 || H >= (T <= P_BLOCK_N ? 1024 : 2048)) ? tile : 0;
}
// Pairs of CTAs that share the vocabulary for one of the token tiles.
int ce_turned_pairs(int T, int V, int tile, int num_sms) {
  const int token_tiles = (T + tile - 1) / tile, pairs = num_sms / 2 / token_tiles, v_tiles = (V + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M);
  return pairs < v_tiles ? pairs : v_tiles;
}

int ce_stats(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target, int64_t vocab_start, int T, int V, int H, void* part, float* tgt, int* status,
             int num_sms, cudaStream_t stream) {
  PCeArgs a;
  a.target = target;
  a.col0 = vocab_start;
  a.part = static_cast<float2*>(part);
  a.tgt = tgt;
  if (ce_few(T, H)) return few_launch<false>(x, ldx, w, ldw, T, V, H, a, nullptr, 0, 0, status, num_sms, stream);
  bool fits;
  CUtensorMap ta, tb;
  if (const int tile = ce_turned_tile(T, H, num_sms)) {
    const int token_tiles = (T + tile - 1) / tile;
    PSched sched;
    sched.total_units = sched.full_units = (V + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M) * token_tiles;
    a.tile_n = tile;
    if (!p_map_kmajor(&ta, w, V, H, ldw) || !p_map_kmajor(&tb, x, T, H, ldx, tile / 2)) return NTB_ERR_ARG;
    switch ((tile + 63) / 64) {
      case 1: return ce_launch<false, false, P_OUT_CE_STATS_T, 8>(ta, tb, ta, V, T, H, sched, ta, PCeTurned<1>{a}, status, num_sms, stream);
      case 2: return ce_launch<false, false, P_OUT_CE_STATS_T, 8>(ta, tb, ta, V, T, H, sched, ta, PCeTurned<2>{a}, status, num_sms, stream);
      case 3: return ce_launch<false, false, P_OUT_CE_STATS_T>(ta, tb, ta, V, T, H, sched, ta, PCeTurned<3>{a}, status, num_sms, stream);
      default: return ce_launch<false, false, P_OUT_CE_STATS_T>(ta, tb, ta, V, T, H, sched, ta, PCeTurned<4>{a}, status, num_sms, stream);
    }
  }
  const PSched sched = ce_whole_tiles(T, V, H, fits);
  if (!fits || !p_map_kmajor(&ta, x, T, H, ldx) || !p_map_kmajor(&tb, w, V, H, ldw)) return NTB_ERR_ARG;
  return ce_launch<false, false, P_OUT_CE_STATS>(ta, tb, ta, T, V, H, sched, ta, a, status, num_sms, stream);
}

// d [T, V] at pitch ldd; the columns up to V rounded up to 64 are written (zeros behind V).
int ce_dlogits(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target, int64_t vocab_start, const float* logz, const float* coef, const float* gn,
               int T, int V, int H, void* d, int64_t ldd, int* status, int num_sms, cudaStream_t stream) {
  const int64_t width = (static_cast<int64_t>(V) + 63) / 64 * 64;
  PCeArgs a;
  a.target = target;
  a.col0 = vocab_start;
  a.logz = logz;
  a.coef = coef;
  a.g = gn;
  if (ce_few(T, H)) return few_launch<true>(x, ldx, w, ldw, T, V, H, a, d, ldd, static_cast<int>(width), status, num_sms, stream);
  bool fits;
  const PSched sched = ce_whole_tiles(T, V, H, fits);
  CUtensorMap ta, tb, td;
  a.a_rows = ce_a_rows(T);
  if (!fits || !p_map_kmajor(&ta, x, T, H, ldx, a.a_rows) || !p_map_kmajor(&tb, w, V, H, ldw) || !p_map_out(&td, d, T, width, ldd, false)) return NTB_ERR_ARG;
  return ce_launch<false, false, P_OUT_CE_GRAD>(ta, tb, td, T, V, H, sched, ta, a, status, num_sms, stream);
}

// D tile = the sum, in chunk order, of the tile's workspace slabs (see PSched); bf16: scaled by *unit and rounded; fp32: stored, or added
// with `accumulate`.  One thread per eight columns, one block per tile and 8 rows: a product cut for lack of tiles has few tiles, so
// the sum takes its parallelism from the rows.
__global__ void __launch_bounds__(256) ce_split_sum_kernel(const float* __restrict__ ws, void* __restrict__ out, int64_t ldo, int M, int N, int split, int chunks, int tiles_m,
                                                            int tiles_n, int band, int bf16_out, int accumulate, const float* __restrict__ unit) {
  p_wait_for_previous();
  const int tile = blockIdx.x >> 5;
  const PTile tc = pair_tile(tile, tiles_m, tiles_n, band);
  const int r = (blockIdx.x & 31) * 8 + (threadIdx.x >> 5), c8 = (threadIdx.x & 31) * 8;
  const int row = tc.m_blk * 2 * P_BLOCK_M + r, col = tc.n_blk * P_BLOCK_N + c8;
  if (row >= M || col >= N) return;
  constexpr int64_t slab = static_cast<int64_t>(2 * P_BLOCK_M) * P_BLOCK_N;
  const float* src = ws + static_cast<int64_t>(tile) * split * slab + r * P_BLOCK_N + c8;
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int ch = 0; ch < chunks; ch++) {
    Vec8<float> a;
    float v[8];
    a.load(src + ch * slab);
    a.to_float(v);
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] += v[j];
  }
  if (bf16_out) {
    const float u = *unit;
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] *= u;
    Vec8<__nv_bfloat16> o;
    o.from_float(f);
    o.store(static_cast<__nv_bfloat16*>(out) + static_cast<int64_t>(row) * ldo + col);
  } else {
    float* dst = static_cast<float*>(out) + static_cast<int64_t>(row) * ldo + col;
    Vec8<float> o;
    if (accumulate) {
      float v[8];
      o.load(dst);
      o.to_float(v);
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] += v[j];
    }
    o.from_float(f);
    o.store(dst);
  }
}

// dx (+)= d w over the V columns of d.  mode 0: dx bf16 = unit * sum; 1: dx fp32 = sum; 2: dx fp32 += sum.  ws: fp32, split * tiles slabs
// of 65536 when split > 1.
int ce_dx(const void* d, int64_t ldd, const void* w, int64_t ldw, void* dx, int64_t lddx, int T, int V, int H, int mode, const float* unit, int split, float* ws,
          int* status, int num_sms, cudaStream_t stream) {
  bool fits;
  PSched sched = ce_whole_tiles(T, H, V, fits);
  const int tiles = sched.total_units, kb = sched.kb_per;
  CUtensorMap ta, tb, td;
  if (!fits || !p_map_kmajor(&ta, d, T, V, ldd) || !p_map_mnmajor(&tb, w, H, V, ldw) || !p_map_out(&td, dx, T, H, lddx, mode != 0)) return NTB_ERR_ARG;
  CUtensorMap tws = td;
  if (split > 1) {
    sched.full_units = 0;
    sched.split = split;
    sched.kb_per = (kb + split - 1) / split;
    sched.total_units = tiles * split;
    if (!p_map_out(&tws, ws, static_cast<int64_t>(tiles) * split * 2 * P_BLOCK_M, P_BLOCK_N, P_BLOCK_N, true)) return NTB_ERR_ARG;
  }
  PAlpha a;
  a.alpha = mode == 0 ? unit : nullptr;
  int rc;
  if (mode == 0) rc = ce_launch<false, true, P_OUT_BF16>(ta, tb, td, T, H, V, sched, tws, a, status, num_sms, stream);
  else if (mode == 1) rc = ce_launch<false, true, P_OUT_F32>(ta, tb, td, T, H, V, sched, tws, a, status, num_sms, stream);
  else rc = ce_launch<false, true, P_OUT_F32_ACCUM>(ta, tb, td, T, H, V, sched, tws, a, status, num_sms, stream);
  if (rc != NTB_OK || split == 1) return rc;
  const int chunks = (kb + sched.kb_per - 1) / sched.kb_per;  // chunks past the end of K wrote nothing
  return ce_launch_next(ce_split_sum_kernel, tiles * 32, 256, 0, stream, ws, dx, lddx, T, H, split, chunks, (T + 255) / 256, (H + 255) / 256, ce_band(T, V), mode == 0, mode == 2,
                        unit);
}

// Rows of the weight gradient: dw [V, H] = unit * d^T x (accumulate 0: bf16 store; 1: added to fp32 dw).
int ce_dw(const void* d, int64_t ldd, const void* x, int64_t ldx, void* dw, int64_t lddw, int T, int V, int H, int accumulate, const float* unit, int* status, int num_sms,
          cudaStream_t stream) {
  bool fits;
  const PSched sched = ce_whole_tiles(V, H, T, fits);
  CUtensorMap ta, tb, td;
  if (!fits || !p_map_mnmajor(&ta, d, V, T, ldd) || !p_map_mnmajor(&tb, x, H, T, ldx) || !p_map_out(&td, dw, V, H, lddw, accumulate != 0)) return NTB_ERR_ARG;
  PAlpha a;
  a.alpha = unit;
  if (accumulate) return ce_launch<true, true, P_OUT_F32_ACCUM>(ta, tb, td, V, H, T, sched, ta, a, status, num_sms, stream);
  return ce_launch<true, true, P_OUT_BF16>(ta, tb, td, V, H, T, sched, ta, a, status, num_sms, stream);
}

}  // namespace

// x [T, H] and w [V, H] bf16, rows 16-byte aligned at pitches ldx, ldw (multiples of 64), H a multiple of 64; target int64 [T]; this
// rank's rows of the vocabulary start at vocab_start.  part: fp32 scratch, (max(ceil(V / 256) * 4, 2 * min(ceil(V / 32), num_sms)) + 1) * T elements, 8-byte aligned.
// out0..2: fp32 [T]: with finish, logZ, loss and (z_coef > 0) z_coef logZ^2; without, the three numbers that vocabulary shards exchange:
// largest score, sum of exp(score - largest), the target's score or 0.
NTB_EXPORT int ntb_linear_ce_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target, int64_t vocab_start, int T, int V, int H, float* part,
                                     float* out0, float* out1, float* out2, int finish, float z_coef, int* status, int num_sms, cudaStream_t stream) {
  if (T <= 0 || V <= 0 || H <= 0 || H % 64 || !ce_operand_ok(x, ldx) || !ce_operand_ok(w, ldw) || (reinterpret_cast<uintptr_t>(part) & 7) || num_sms < 2 || !out0 || !out1 || (!out2 && (!finish || z_coef > 0.f)) ||
      !p_get_encode())
    return NTB_ERR_ARG;
  // partial statistics per token: one of every CTA, or one of every half tile (the last may have no columns: (-inf, 0))
  const int turned = ce_turned_tile(T, H, num_sms);
  const int tiles = ce_few(T, H) ? few_grid(V, num_sms) : turned ? 2 * ce_turned_pairs(T, V, turned, num_sms) : (V + P_BLOCK_N - 1) / P_BLOCK_N * (CE_WARPS / 4);
  float* tgt = part + static_cast<int64_t>(tiles) * 2 * T;
  const int rc = ce_stats(x, ldx, w, ldw, target, vocab_start, T, V, H, part, tgt, status, num_sms, stream);
  if (rc != NTB_OK) return rc;
  return ce_launch_next(ce_join_kernel, (T + CE_JOIN_ROWS - 1) / CE_JOIN_ROWS, CE_JOIN_ROWS * CE_JOIN_PARTS, 0, stream, reinterpret_cast<const float2*>(part), tgt, target,
                        vocab_start, V, tiles, T, finish ? nullptr : out0, finish ? nullptr : out1, finish ? nullptr : out2, finish ? out0 : nullptr, finish ? out1 : nullptr,
                        finish && z_coef > 0.f ? out2 : nullptr, z_coef);
}

// How the dx product [T, H] over V is cut along V: with fewer tiles than CTA pairs (few tokens) every tile becomes `split` chunks
// whose fp32 partial sums go through a workspace and are added in chunk order.  Returns the chunks per tile (1: not cut).
NTB_EXPORT int ntb_linear_ce_dx_split(int T, int V, int H, int num_sms) {
  const int pairs = num_sms / 2;
  const long long tiles = ((T + 255ll) / 256) * ((H + 255) / 256);
  const int kb = (V + P_BLOCK_K - 1) / P_BLOCK_K;
  if (tiles >= 2 * pairs) return 1;
  // fewest rounds of (chunk length + a fixed share for the start and the hand-over of a chunk, about eight k-blocks)
  int best = 1;
  long long best_cost = -1;
  for (int s = 1; s <= 64 && s * 8 <= kb + 7 && tiles * s <= 4 * pairs; s++) {
    const long long rounds = (tiles * s + pairs - 1) / pairs;
    const long long cost = rounds * ((kb + s - 1) / s + 8);
    if (best_cost < 0 || cost < best_cost) best = s, best_cost = cost;
  }
  return best;
}

// Gradients, in pieces of `width` vocabulary entries.  g, gz (null without a z term), logz: fp32 [T].
// d: bf16 [T, ldd], ldd a multiple of 64 and at least min(width, V); rows: fp32 scratch, 2 T + 1; acc: fp32 [T, H] when there are
// several pieces and dx is wanted; ws: fp32, split * ceil(T / 256) * ceil(H / 256) * 65536 when split (ntb_linear_ce_dx_split of a
// piece) > 1.  dx: bf16 [T, H] or null; dw: [V, H] at pitch lddw or null, bf16 (dw_accumulate 0) or fp32 that is added to (1).
NTB_EXPORT int ntb_linear_ce_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target, int64_t vocab_start, const float* logz, const float* g,
                                      const float* gz, float z_coef, int T, int V, int H, int width, void* d, int64_t ldd, float* rows, void* dx, float* acc, int split,
                                      float* ws, void* dw, int64_t lddw, int dw_accumulate, int* status, int num_sms, cudaStream_t stream) {
  if (T <= 0 || V <= 0 || H <= 0 || H % 64 || width <= 0 || width % 64 || !ce_operand_ok(x, ldx) || !ce_operand_ok(w, ldw) || !ce_operand_ok(d, ldd) || num_sms < 2 ||
      ldd < (static_cast<int64_t>(width < V ? width : V) + 63) / 64 * 64 || !p_get_encode())
    return NTB_ERR_ARG;
  if (dx != nullptr && (!ce_operand_ok(dx, H) || (width < V && (acc == nullptr || !ce_operand_ok(acc, H))) || split < 1 || (split > 1 && (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 127)))))
    return NTB_ERR_ARG;
  if (dw != nullptr && ((reinterpret_cast<uintptr_t>(dw) & 15) || lddw % 8 || lddw < H)) return NTB_ERR_ARG;
  float *coef = rows, *gn = rows + T, *unit = rows + 2 * static_cast<int64_t>(T);
  ce_row_coefficients_kernel<<<1, 1024, 0, stream>>>(g, gz, logz, z_coef, T, coef, gn, unit);
  for (int64_t v0 = 0; v0 < V; v0 += width) {
    const int n = static_cast<int>(V - v0 < width ? V - v0 : width);
    const char* wp = static_cast<const char*>(w) + v0 * ldw * 2;
    int rc = ce_dlogits(x, ldx, wp, ldw, target, vocab_start + v0, logz, coef, gn, T, n, H, d, ldd, status, num_sms, stream);
    if (rc != NTB_OK) return rc;
    if (dx != nullptr) {
      rc = width >= V ? ce_dx(d, ldd, wp, ldw, dx, H, T, n, H, 0, unit, split, ws, status, num_sms, stream)
                      : ce_dx(d, ldd, wp, ldw, acc, H, T, n, H, v0 == 0 ? 1 : 2, unit, split, ws, status, num_sms, stream);
      if (rc != NTB_OK) return rc;
    }
    if (dw != nullptr) {
      rc = ce_dw(d, ldd, x, ldx, static_cast<char*>(dw) + v0 * lddw * (dw_accumulate ? 4 : 2), lddw, T, n, H, dw_accumulate, unit, status, num_sms, stream);
      if (rc != NTB_OK) return rc;
    }
  }
  if (dx != nullptr && width < V) {
    const int64_t n8 = static_cast<int64_t>(T) * H / 8;
    const int64_t blocks = (n8 + 255) / 256;
    return ce_launch_next(ce_scale_cast_kernel, blocks < 148 * 8 ? blocks : 148 * 8, 256, 0, stream, acc, unit, static_cast<__nv_bfloat16*>(dx), n8);
  }
  return ntb_check_launch();
}
