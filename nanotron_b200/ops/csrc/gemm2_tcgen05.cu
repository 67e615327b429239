// Entry points of the bf16 GEMM on CTA pairs (kernel: gemm2_core.cuh): plain, all-gather-gated and peer-store products, and the
// optional cut of a launch's last round along K.
#include "gemm2_core.cuh"

namespace {

// Per-device fp32 workspace for split tiles (caller-owned, ws_tiles slabs of 256 x 256 floats); see ntb_gemm2_set_workspace.
static float* g_p_ws[64] = {};
static int g_p_ws_tiles[64] = {};
static cudaStream_t g_p_ws_stream[64] = {};
static int g_p_split_enabled = 0;  // off by default: measured within +-5 % of whole tiles on Llama shapes (the step is power-bound, not round-bound)

// How the tiles of a launch are dealt out (see PSched).  `ws_tiles`: workspace slabs available (0: never split).
static PSched p_schedule(int num_tiles, int pairs_max, int k_blocks, int ws_tiles) {
  PSched sc;
  sc.total_units = sc.full_units = num_tiles;
  sc.split = 1;
  sc.kb_per = k_blocks;
  if (!g_p_split_enabled || ws_tiles <= 0 || num_tiles <= 0) return sc;
  const int rounds = num_tiles / pairs_max, rem = num_tiles % pairs_max;
  if (rem == 0 || rem * 100 >= pairs_max * 85) return sc;  // the last round is (nearly) full already
  int split = pairs_max / rem;
  if (split > k_blocks / 4) split = k_blocks / 4;  // at least four k-blocks per chunk
  if (split < 2) return sc;
  if (rem * split > ws_tiles) return sc;
  sc.full_units = rounds * pairs_max;
  sc.split = split;
  sc.kb_per = (k_blocks + split - 1) / split;
  sc.total_units = sc.full_units + rem * split;
  return sc;
}

template <bool A_MN, bool B_MN, int OUT, int ST = P_MAX_STAGES>
int p_launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& td, int M, int N, int K, int* status, int num_sms, cudaStream_t stream,
             const PFuse& fuse = PFuse(), const PPeerMaps* pmaps = nullptr, void* d_out = nullptr, int64_t ldd = 0, const CUtensorMap* tal = nullptr) {
  static const PPeerMaps no_maps = {};
  const PPeerMaps& pm = pmaps ? *pmaps : no_maps;
  auto kern = gemm2_tcgen05_kernel<A_MN, B_MN, OUT, ST>;
  static bool configured = false;
  if (!configured) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P_SMEM) != cudaSuccess) return NTB_ERR_LAUNCH;
    configured = true;
  }
  const long long tiles = static_cast<long long>((M + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M)) * ((N + P_BLOCK_N - 1) / P_BLOCK_N);
  const int k_blocks = (K + P_BLOCK_K - 1) / P_BLOCK_K;
  // every output mode but the peer stores of the reduce-scatter mode may cut the tiles of its last round along K, if a workspace
  // was registered for this device and stream and D is known as a plain pointer (16-byte aligned rows for the fix-up pass)
  int dev = 0, ws_tiles = 0;
  float* ws = nullptr;
  if (OUT != P_OUT_PEER_BF16 && d_out != nullptr && N % 8 == 0 && (OUT == P_OUT_BF16 || (ldd % 4 == 0 && (reinterpret_cast<uintptr_t>(d_out) & 15) == 0)) &&
      cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 && g_p_ws[dev] != nullptr && g_p_ws_stream[dev] == stream) {
    ws = g_p_ws[dev];
    ws_tiles = g_p_ws_tiles[dev];
  }
  const PSched sched = p_schedule(static_cast<int>(tiles), num_sms / 2, k_blocks, tiles > (1 << 30) ? 0 : ws_tiles);
  CUtensorMap tws = td;  // placeholder when nothing goes through the workspace
  const bool uses_ws = sched.split > 1;
  if (uses_ws && !p_map_out(&tws, ws, static_cast<int64_t>(ws_tiles) * 2 * P_BLOCK_M, P_BLOCK_N, P_BLOCK_N, true)) return NTB_ERR_ARG;
  long long pairs = num_sms / 2;
  if (sched.total_units < pairs) pairs = sched.total_units;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs), 1, 1);
  cfg.blockDim = dim3(P_THREADS, 1, 1);
  cfg.dynamicSmemBytes = P_SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // rows of A (256 per tile row, K deep, bf16) that should stay resident in the 126 MB L2 while B streams: about 40 MB
  int band = static_cast<int>(40000000ll / (512ll * (K > 0 ? K : 1)));
  const int tiles_m = (M + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M);
  if (band < 2) band = 2;
  if (band > tiles_m) band = tiles_m;
  if (cudaLaunchKernelEx(&cfg, kern, ta, tb, td, M, N, K, band, status, fuse, pm, sched, tws, tal ? *tal : ta, PPlain()) != cudaSuccess) {
    cudaGetLastError();
    return NTB_ERR_LAUNCH;
  }
  if (uses_ws) {
    const int split_tiles = static_cast<int>(tiles) - sched.full_units;
    const int tiles_n = (N + P_BLOCK_N - 1) / P_BLOCK_N;
    gemm2_split_fixup_kernel<OUT><<<split_tiles * 8, 256, 0, stream>>>(ws, d_out, ldd, M, N, k_blocks, sched, tiles_m, tiles_n, band, fuse.m_rot);
  }
  return ntb_check_launch();
}

}  // namespace

// Same contract as ntb_gemm_bf16 (gemm_tcgen05.cu); additionally M-major / N-major operands need M % 128 == 0 / N % 128 == 0 is NOT
// required: edges are clipped by TMA.  a_mn / b_mn: 0 = K-major, 1 = MN-major.  out_mode: 0 bf16 store, 1 fp32 store, 2 fp32 accumulate.
// Which argument check rejected the last ntb_gemm2_bf16 call of this thread (0: none; for error messages).
static thread_local int g_p_reject = 0;
NTB_EXPORT int ntb_gemm2_last_reject() { return g_p_reject; }

NTB_EXPORT int ntb_gemm2_bf16(const void* a, const void* b, void* d, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldd, int a_mn, int b_mn, int out_mode,
                              int* status, int num_sms, cudaStream_t stream) {
  g_p_reject = 0;
#define NTB_P_REJECT(code) do { g_p_reject = (code); return NTB_ERR_ARG; } while (0)
  if (M <= 0 || N <= 0 || K <= 0) NTB_P_REJECT(1);
  if (!p_get_encode()) NTB_P_REJECT(2);
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(d)) & 15) NTB_P_REJECT(3);
  if (a_mn ? (lda % 64 || M % 64) : (lda % 8)) NTB_P_REJECT(4);
  if (b_mn ? (ldb % 64 || N % 64) : (ldb % 8)) NTB_P_REJECT(5);
  if (out_mode == P_OUT_BF16 ? (ldd % 8) : (ldd % 4)) NTB_P_REJECT(6);
  if (num_sms <= 1) num_sms = 148;
  CUtensorMap ta, tb, td;
  if (!(a_mn ? p_map_mnmajor(&ta, a, M, K, lda) : p_map_kmajor(&ta, a, M, K, lda))) NTB_P_REJECT(7);
  if (!(b_mn ? p_map_mnmajor(&tb, b, N, K, ldb) : p_map_kmajor(&tb, b, N, K, ldb))) NTB_P_REJECT(8);
  if (!p_map_out(&td, d, M, N, ldd, out_mode != P_OUT_BF16)) NTB_P_REJECT(9);
#define NTB_P_CASE(AM, BM, OM) \
  if (a_mn == AM && b_mn == BM && out_mode == OM) return p_launch<AM != 0, BM != 0, OM>(ta, tb, td, M, N, K, status, num_sms, stream, PFuse(), nullptr, d, ldd);
  NTB_P_CASE(0, 0, 0) NTB_P_CASE(0, 0, 1) NTB_P_CASE(0, 0, 2)
  NTB_P_CASE(0, 1, 0) NTB_P_CASE(0, 1, 1) NTB_P_CASE(0, 1, 2)
  NTB_P_CASE(1, 1, 0) NTB_P_CASE(1, 1, 1) NTB_P_CASE(1, 1, 2)
  NTB_P_CASE(1, 0, 0) NTB_P_CASE(1, 0, 1) NTB_P_CASE(1, 0, 2)
#undef NTB_P_CASE
  NTB_P_REJECT(10);
#undef NTB_P_REJECT
}

// D = gathered_A @ B^T (or @ B when b_mn) where gathered_A = [world * ag_rows, K] is filled by ntb_tp_allgather_push on every rank
// (same contract as ntb_gemm_bf16_ag; ag_rows must be a multiple of 128 here).
static int p_gemm_ag(const void* a_gathered, const void* a_local, int64_t lda_local, const void* b, void* d, int M, int N, int K, int64_t lda, int64_t ldb,
                     int64_t ldd, int b_mn, const uint32_t* ag_flags, int ag_rows, int me, int world, uint32_t epoch, int* status, int num_sms,
                     cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || !p_get_encode() || world < 1 || world > P_TP_MAX || ag_rows <= 0 || ag_rows % P_BLOCK_M || ag_flags == nullptr) return NTB_ERR_ARG;
  if (me < 0 || me >= world || static_cast<int64_t>(ag_rows) * world != M) return NTB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(a_gathered) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(d) | reinterpret_cast<uintptr_t>(a_local)) & 15) return NTB_ERR_ARG;
  if (lda % 8 || (b_mn ? (ldb % 64 || N % 64) : (ldb % 8)) || ldd % 8 || (a_local != nullptr && lda_local % 8)) return NTB_ERR_ARG;
  if (num_sms <= 1) num_sms = 148;
  CUtensorMap ta, tb, td, tal;
  if (!p_map_kmajor(&ta, a_gathered, M, K, lda)) return NTB_ERR_ARG;
  if (a_local != nullptr && !p_map_kmajor(&tal, a_local, ag_rows, K, lda_local)) return NTB_ERR_ARG;
  if (!(b_mn ? p_map_mnmajor(&tb, b, N, K, ldb) : p_map_kmajor(&tb, b, N, K, ldb))) return NTB_ERR_ARG;
  if (!p_map_out(&td, d, M, N, ldd, false)) return NTB_ERR_ARG;
  PFuse f;
  f.world = world;
  f.me = me;
  f.epoch = epoch;
  f.ag_flags = ag_flags;
  f.ag_rows = ag_rows;
  f.ag_local = a_local != nullptr ? 1 : 0;
  const int tiles_m = (M + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M);
  f.m_rot = ((me * ag_rows) / (2 * P_BLOCK_M)) % tiles_m;  // start with the rows this rank contributed itself
  const CUtensorMap* pl = a_local != nullptr ? &tal : nullptr;
  return b_mn ? p_launch<false, true, P_OUT_BF16>(ta, tb, td, M, N, K, status, num_sms, stream, f, nullptr, d, ldd, pl)
              : p_launch<false, false, P_OUT_BF16>(ta, tb, td, M, N, K, status, num_sms, stream, f, nullptr, d, ldd, pl);
}

// D = gathered_A @ B^T (or @ B when b_mn) where gathered_A = [world * ag_rows, K] is filled by ntb_tp_allgather_push on every rank.
NTB_EXPORT int ntb_gemm2_bf16_ag(const void* a_gathered, const void* b, void* d, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldd, int b_mn,
                                 const uint32_t* ag_flags, int ag_rows, int me, int world, uint32_t epoch, int* status, int num_sms, cudaStream_t stream) {
  return p_gemm_ag(a_gathered, nullptr, 0, b, d, M, N, K, lda, ldb, ldd, b_mn, ag_flags, ag_rows, me, world, epoch, status, num_sms, stream);
}

// Same product, but rows [me * ag_rows, (me + 1) * ag_rows) are read from `a_local` (the tensor this rank pushes, row pitch
// lda_local) instead of from the gather buffer.  The launch then depends on no kernel of its own GPU, so the caller may run this
// rank's push on another stream at the same time; only the peers' blocks are waited for (bounded).
NTB_EXPORT int ntb_gemm2_bf16_ag_local(const void* a_gathered, const void* a_local, int64_t lda_local, const void* b, void* d, int M, int N, int K, int64_t lda,
                                       int64_t ldb, int64_t ldd, int b_mn, const uint32_t* ag_flags, int ag_rows, int me, int world, uint32_t epoch, int* status,
                                       int num_sms, cudaStream_t stream) {
  if (a_local == nullptr) return NTB_ERR_ARG;
  return p_gemm_ag(a_gathered, a_local, lda_local, b, d, M, N, K, lda, ldb, ldd, b_mn, ag_flags, ag_rows, me, world, epoch, status, num_sms, stream);
}

// Registers (ws != nullptr) or removes the fp32 workspace that lets launches on the CURRENT device cut the tiles of
// their last round along K: `tiles` slabs of 256 x 256 floats (contents do not matter), owned by the caller for as long as it is
// registered.  Only launches on `stream` use it (launches on other streams run unsplit), so two launches never write it at once.
// Returns 0, or NTB_ERR_ARG.
NTB_EXPORT int ntb_gemm2_set_workspace(float* ws, int tiles, cudaStream_t stream) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || (ws != nullptr && (tiles <= 0 || (reinterpret_cast<uintptr_t>(ws) & 127)))) return NTB_ERR_ARG;
  g_p_ws[dev] = ws;
  g_p_ws_tiles[dev] = ws ? tiles : 0;
  g_p_ws_stream[dev] = stream;
  return NTB_OK;
}

// Non-zero switches the split of the last round on for every launch that has a workspace, 0 (the default) off.
NTB_EXPORT void ntb_gemm2_enable_split(int on) { g_p_split_enabled = on != 0; }

// Partial product A @ B^T (or A @ B when b_mn) whose rows [r*rs_rows, (r+1)*rs_rows) are stored (bf16) into rank r's staging slot `me`
// (same contract as ntb_gemm_bf16_rs).
NTB_EXPORT int ntb_gemm2_bf16_rs(const void* a, const void* b, int M, int N, int K, int64_t lda, int64_t ldb, int b_mn, const uint64_t* staging_ptrs,
                                 const uint64_t* flag_ptrs, int rs_rows, int me, int world, uint32_t epoch, unsigned int* done_counter, int* status, int num_sms,
                                 cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || !p_get_encode() || world < 1 || world > P_TP_MAX || rs_rows * world != M || rs_rows % 32 || N % 8 || done_counter == nullptr) return NTB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) return NTB_ERR_ARG;
  if (lda % 8 || (b_mn ? (ldb % 64 || N % 64) : (ldb % 8))) return NTB_ERR_ARG;
  if (num_sms <= 1) num_sms = 148;
  CUtensorMap ta, tb;
  if (!p_map_kmajor(&ta, a, M, K, lda)) return NTB_ERR_ARG;
  if (!(b_mn ? p_map_mnmajor(&tb, b, N, K, ldb) : p_map_kmajor(&tb, b, N, K, ldb))) return NTB_ERR_ARG;
  PFuse f;
  f.world = world;
  f.me = me;
  f.epoch = epoch;
  f.rs_rows = rs_rows;
  f.done_counter = done_counter;
  PPeerMaps pm = {};
  for (int r = 0; r < world; r++) {
    if (staging_ptrs[r] & 15) return NTB_ERR_ARG;
    if (!p_map_out(&pm.m[r], reinterpret_cast<void*>(staging_ptrs[r]), static_cast<int64_t>(world) * rs_rows, N, N, false)) return NTB_ERR_ARG;
    f.rs_flags[r] = reinterpret_cast<uint32_t*>(flag_ptrs[r]);
  }
  const int tiles_m = (M + 2 * P_BLOCK_M - 1) / (2 * P_BLOCK_M);
  f.m_rot = ((((me + 1) % world) * rs_rows) / (2 * P_BLOCK_M)) % tiles_m;  // the next rank's rows first, our own last
  return b_mn ? p_launch<false, true, P_OUT_PEER_BF16>(ta, tb, ta, M, N, K, status, num_sms, stream, f, &pm)
              : p_launch<false, false, P_OUT_PEER_BF16>(ta, tb, ta, M, N, K, status, num_sms, stream, f, &pm);
}
