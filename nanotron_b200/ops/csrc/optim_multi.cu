// One AdamW step over many tensors in one launch, running averages in fp32 or in 8-bit blocks (sm_100a).
//
//   g' = s g      m = b1 m + (1 - b1) g'      v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit blocks.  128 consecutive elements of a tensor share one byte E, the fp32 exponent field of the block's largest magnitude.
// Code c > 0 counts eighths of binades from the lower end of the window below 2^(E - 127): for m a sign and 7 bits (15 binades and
// 3 mantissa bits), for v, which is never negative, 8 bits (31 binades of the square, 15.5 of the root the step divides by).  With t
// = the fp32 bit pattern >> 20, c = t - 8 E + 120 (m) or + 248 (v), so encoding and decoding are integer additions.  Code 0 is zero.
//  * Rounding is stochastic: the 20 cut mantissa bits round up with the probability they stand for.  The averages move by at most
//    (1 - b) of their value per step, for b2 = 0.95 .. 0.999 less than half a code, where rounding to nearest would never move them.
//    The random bits are a hash of (seed of the call, tensor number, element number): a step is a function of its inputs.
//  * m below the window becomes zero, v below it the smallest code: v = 0 beside m > 0 would make the step m / eps.
//  * A block with a value that is not finite stores E = 255 and reads back as NaN throughout.
// The step itself uses the unrounded m and v.  In the 8-bit form m and v are computed with separately rounded operations (no fused
// multiply-add), so the codes do not depend on how a compiler contracts them: any other fp32 evaluation of the formulas, the PyTorch
// one among them, gives the same bytes.
//
// Bound by HBM: 18 bytes an element with a bf16 copy, fp32 gradients and 8-bit states, 30 with fp32 states.  A warp takes blocks of 128
// elements as 32 lanes x 4 (every access of a warp is one contiguous 128 .. 512 byte segment), so the largest magnitude of a block is
// one redux over the warp; four blocks per warp are loaded before the first is used.
#include "common.cuh"

namespace {

constexpr int AM_THREADS = 256;
constexpr int AM_BLOCK = 128;                                       // elements per state block: one warp, four elements a lane
constexpr int AM_UNROLL = 4;                                        // blocks a warp holds in flight
constexpr int AM_WARP_ELEMS = AM_BLOCK * AM_UNROLL;
constexpr int AM_CHUNK = AM_WARP_ELEMS * (AM_THREADS / 32);        // 4096 elements per CTA and iteration

struct AmTensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  __nv_bfloat16* half;  // bf16 copy of the result, or null
  uint8_t* me;          // block exponents of m and v (8-bit states)
  uint8_t* ve;
  int64_t n;
  float lr, wd;
  uint32_t key;         // of the random bits
  uint32_t vec;         // 1: every pointer is aligned for four elements at a time
};
static_assert(sizeof(AmTensor) == 80, "layout shared with the Python side");

// The table travels as a kernel parameter: no copy to the device, nothing to keep alive, and a captured graph owns its table.  Two
// sizes, because a parameter is copied whole at every launch.
template <int CAP> struct AmTable {
  AmTensor t[CAP];
  uint32_t first[CAP + 1];  // first chunk of every tensor, then the number of chunks
  int count;
};
constexpr int AM_SMALL = 24, AM_LARGE = 384;
static_assert(sizeof(AmTable<AM_LARGE>) < 32700, "kernel parameters end at 32764 bytes");

struct AmHyper {
  float b1, omb1, b2, omb2, eps, inv_bc1, inv_sqrt_bc2;  // omb: 1 - b, rounded once from 64 bits (1.f - 0.999f is off by 2^-16); bc: 1 - b^t
  const float* grad_scale;
};

__device__ __forceinline__ float mul_rn(float a, float b) {
  float c;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ float add_rn(float a, float b) {
  float c;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// Integer mixing (xor-shift, multiply, twice), constants of C. Wellons' published low-bias 32-bit hash.
__host__ __device__ __forceinline__ uint32_t am_mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

template <bool SIGNED> struct Q8 {
  static constexpr int TOP = SIGNED ? 127 : 255;
  // e8: 8 * E - (TOP - 7); nan: E == 255
  static __device__ __forceinline__ float decode(uint32_t c, int e8, bool nan) {
    const int mag = static_cast<int>(c & TOP) + e8;
    float f = ((c & TOP) == 0 || mag < 8) ? 0.f : __int_as_float(mag << 20);
    if (SIGNED) f = __uint_as_float(__float_as_uint(f) | ((c & 128u) << 24));
    return nan ? __int_as_float(0x7fffffff) : f;
  }
  // size: magnitude bits; r16: 16 random bits
  static __device__ __forceinline__ uint32_t encode(float x, uint32_t r16, int e8, bool nan) {
    const uint32_t bits = __float_as_uint(x), size = bits & 0x7fffffffu;
    int c = static_cast<int>((size + (r16 << 4) + 8u) >> 20) - e8;
    c = min(max(c, SIGNED ? 0 : 1), TOP);
    if (size < 0x800000u || nan) c = 0;
    if (SIGNED && c > 0) c |= static_cast<int>((bits >> 24) & 128u);
    return static_cast<uint32_t>(c);
  }
  static __device__ __forceinline__ int window(uint32_t E) { return static_cast<int>(8 * E) - (TOP - 7); }
};

// Four consecutive elements of a tensor from element i on; `vec`: all four exist and the address is aligned for them.
template <typename T> __device__ __forceinline__ void load4(const T* p, int64_t i, int64_t n, bool vec, float (&f)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p + i);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(p + i);
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&a.x)), y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&a.y));
      f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = i + j < n ? to_f<T>(p[i + j]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store4(T* p, int64_t i, int64_t n, bool vec, const float (&f)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p + i) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      __nv_bfloat162 x = __floats2bfloat162_rn(f[0], f[1]), y = __floats2bfloat162_rn(f[2], f[3]);
      *reinterpret_cast<uint2*>(p + i) = make_uint2(*reinterpret_cast<uint32_t*>(&x), *reinterpret_cast<uint32_t*>(&y));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j < n) p[i + j] = from_f<T>(f[j]);
  }
}
__device__ __forceinline__ uint32_t load4(const uint8_t* p, int64_t i, int64_t n, bool vec) {
  if (vec) return *reinterpret_cast<const uint32_t*>(p + i);
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (i + j < n) c |= static_cast<uint32_t>(p[i + j]) << (8 * j);
  return c;
}
__device__ __forceinline__ void store4(uint8_t* p, int64_t i, int64_t n, bool vec, uint32_t c) {
  if (vec) {
    *reinterpret_cast<uint32_t*>(p + i) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j < n) p[i + j] = static_cast<uint8_t>(c >> (8 * j));
  }
}

template <typename P, typename G, int BITS, int CAP>
__global__ void __launch_bounds__(AM_THREADS) adamw_multi_kernel(const __grid_constant__ AmTable<CAP> tab, const __grid_constant__ AmHyper hy) {
  const float gs = hy.grad_scale ? *hy.grad_scale : 1.f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t chunks = tab.first[tab.count];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    int lo = 0, hi = tab.count - 1;  // the last tensor that starts at or before this chunk
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tab.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    const AmTensor& t = tab.t[lo];
    const int64_t n = t.n;
    const int64_t base = static_cast<int64_t>(chunk - tab.first[lo]) * AM_CHUNK + warp * AM_WARP_ELEMS;
    if (base >= n) continue;
    P* p = static_cast<P*>(t.p);
    const G* g = static_cast<const G*>(t.g);
    float pv[AM_UNROLL][4], gv[AM_UNROLL][4];
    float mf[BITS == 32 ? AM_UNROLL : 1][4], vf[BITS == 32 ? AM_UNROLL : 1][4];
    uint32_t mc[AM_UNROLL], vc[AM_UNROLL], me[AM_UNROLL], ve[AM_UNROLL];
#pragma unroll
    for (int u = 0; u < AM_UNROLL; u++) {
      const int64_t i = base + u * AM_BLOCK + lane * 4;
      const bool vec = t.vec && i + 3 < n;
      load4<P>(p, i, n, vec, pv[u]);
      load4<G>(g, i, n, vec, gv[u]);
      if constexpr (BITS == 32) {
        load4<float>(static_cast<const float*>(t.m), i, n, vec, mf[u]);
        load4<float>(static_cast<const float*>(t.v), i, n, vec, vf[u]);
      } else {
        mc[u] = load4(static_cast<const uint8_t*>(t.m), i, n, vec);
        vc[u] = load4(static_cast<const uint8_t*>(t.v), i, n, vec);
        const int64_t b = base / AM_BLOCK + u;
        const bool in = b * AM_BLOCK < n;
        me[u] = in ? t.me[b] : 0u;
        ve[u] = in ? t.ve[b] : 0u;
      }
    }
#pragma unroll
    for (int u = 0; u < AM_UNROLL; u++) {
      const int64_t i = base + u * AM_BLOCK + lane * 4;
      if (base + u * AM_BLOCK >= n) break;  // the whole warp
      const bool vec = t.vec && i + 3 < n;
      float m[4], v[4];
      if constexpr (BITS == 32) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float gj = gv[u][j] * gs;
          m[j] = hy.b1 * mf[u][j] + hy.omb1 * gj;
          v[j] = hy.b2 * vf[u][j] + hy.omb2 * gj * gj;
        }
      } else {
        const int m8 = Q8<true>::window(me[u]), v8 = Q8<false>::window(ve[u]);
        const bool mnan = me[u] == 255u, vnan = ve[u] == 255u;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float gj = mul_rn(gv[u][j], gs);
          m[j] = add_rn(mul_rn(Q8<true>::decode((mc[u] >> (8 * j)) & 255u, m8, mnan), hy.b1), mul_rn(gj, hy.omb1));
          v[j] = add_rn(mul_rn(Q8<false>::decode((vc[u] >> (8 * j)) & 255u, v8, vnan), hy.b2), mul_rn(mul_rn(gj, gj), hy.omb2));
        }
      }
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float denom = sqrtf(v[j]) * hy.inv_sqrt_bc2 + hy.eps;
        o[j] = pv[u][j] * (1.f - t.lr * t.wd);
        o[j] -= t.lr * hy.inv_bc1 * m[j] / denom;
      }
      store4<P>(p, i, n, vec, o);
      if (t.half != nullptr) store4<__nv_bfloat16>(t.half, i, n, vec, o);
      if constexpr (BITS == 32) {
        store4<float>(static_cast<float*>(t.m), i, n, vec, m);
        store4<float>(static_cast<float*>(t.v), i, n, vec, v);
      } else {
        uint32_t mx = 0, vx = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (i + j < n) {
            mx = max(mx, __float_as_uint(m[j]) & 0x7fffffffu);
            vx = max(vx, __float_as_uint(v[j]) & 0x7fffffffu);
          }
        }
        const uint32_t Em = __reduce_max_sync(0xffffffffu, mx) >> 23, Ev = __reduce_max_sync(0xffffffffu, vx) >> 23;
        const int m8 = Q8<true>::window(Em), v8 = Q8<false>::window(Ev);
        const bool mnan = Em == 255u, vnan = Ev == 255u;
        uint32_t mo = 0, vo = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint64_t e = static_cast<uint64_t>(i + j);
          const uint32_t r = am_mix(static_cast<uint32_t>(e) ^ (t.key + static_cast<uint32_t>(e >> 32) * 0x9e3779b9u));
          mo |= Q8<true>::encode(m[j], r & 0xffffu, m8, mnan) << (8 * j);
          vo |= Q8<false>::encode(v[j], r >> 16, v8, vnan) << (8 * j);
        }
        store4(static_cast<uint8_t*>(t.m), i, n, vec, mo);
        store4(static_cast<uint8_t*>(t.v), i, n, vec, vo);
        if (lane == 0) {
          const int64_t b = base / AM_BLOCK + u;
          t.me[b] = static_cast<uint8_t>(Em);
          t.ve[b] = static_cast<uint8_t>(Ev);
        }
      }
    }
  }
}

// One warp per block of 128.
template <typename T, bool SIGNED>
__global__ void __launch_bounds__(256) q8_decode_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, T* __restrict__ out, int64_t n, int aligned) {
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (n + AM_BLOCK - 1) / AM_BLOCK;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); b < blocks; b += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t i = b * AM_BLOCK + lane * 4;
    const bool vec = aligned && i + 3 < n;
    const uint32_t c = load4(codes, i, n, vec), E = exps[b];
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = Q8<SIGNED>::decode((c >> (8 * j)) & 255u, Q8<SIGNED>::window(E), E == 255u);
    store4<T>(out, i, n, vec, f);
  }
}

// To the nearest code (ties away from zero): what a decoded block encodes to is the block itself.
template <bool SIGNED>
__global__ void __launch_bounds__(256) q8_encode_kernel(const float* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ exps, int64_t n, int aligned) {
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (n + AM_BLOCK - 1) / AM_BLOCK;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); b < blocks; b += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t i = b * AM_BLOCK + lane * 4;
    const bool vec = aligned && i + 3 < n;
    float f[4];
    load4<float>(x, i, n, vec, f);
    uint32_t mx = 0, c = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) mx = max(mx, __float_as_uint(f[j]) & 0x7fffffffu);
    const uint32_t E = __reduce_max_sync(0xffffffffu, mx) >> 23;
#pragma unroll
    for (int j = 0; j < 4; j++) c |= Q8<SIGNED>::encode(f[j], 0x8000u, Q8<SIGNED>::window(E), E == 255u) << (8 * j);
    store4(codes, i, n, vec, c);
    if (lane == 0) exps[b] = static_cast<uint8_t>(E);
  }
}

template <typename P, typename G, int BITS, int CAP>
int am_launch(const AmTensor* t, int count, const AmHyper& hy, int num_sms, cudaStream_t stream) {
  AmTable<CAP> tab;  // copied by the launch
  uint64_t chunks = 0;
  for (int i = 0; i < count; i++) {
    tab.t[i] = t[i];
    tab.first[i] = static_cast<uint32_t>(chunks);
    chunks += static_cast<uint64_t>((t[i].n + AM_CHUNK - 1) / AM_CHUNK);
    if (chunks > 0x7fffffffull) return NTB_ERR_ARG;
  }
  tab.first[count] = static_cast<uint32_t>(chunks);
  tab.count = count;
  const uint64_t cap = static_cast<uint64_t>(num_sms) * 8;
  adamw_multi_kernel<P, G, BITS, CAP><<<static_cast<unsigned>(chunks < cap ? chunks : cap), AM_THREADS, 0, stream>>>(tab, hy);
  return ntb_check_launch();
}

template <typename P, typename G>
int am_dispatch(const AmTensor* t, int count, int bits, const AmHyper& hy, int num_sms, cudaStream_t stream) {
  for (int at = 0; at < count; at += AM_LARGE) {
    const int k = count - at < AM_LARGE ? count - at : AM_LARGE;
    int rc;
    if (k <= AM_SMALL) rc = bits == 8 ? am_launch<P, G, 8, AM_SMALL>(t + at, k, hy, num_sms, stream) : am_launch<P, G, 32, AM_SMALL>(t + at, k, hy, num_sms, stream);
    else rc = bits == 8 ? am_launch<P, G, 8, AM_LARGE>(t + at, k, hy, num_sms, stream) : am_launch<P, G, 32, AM_LARGE>(t + at, k, hy, num_sms, stream);
    if (rc != NTB_OK) return rc;
  }
  return NTB_OK;
}

}  // namespace

// table: `count` AmTensor records in host memory (every n > 0; `vec` is set here).  p_dtype / g_dtype: NTB_F32 or NTB_BF16.  bits: 32 or 8.
NTB_EXPORT int ntb_adamw_multi(void* table, int count, int p_dtype, int g_dtype, int bits, float b1, float omb1, float b2, float omb2, float eps, float bias_correction1,
                               float bias_correction2, const float* grad_scale, int num_sms, cudaStream_t stream) {
  if (count <= 0 || table == nullptr || (bits != 8 && bits != 32) || num_sms <= 0) return NTB_ERR_ARG;
  AmTensor* t = static_cast<AmTensor*>(table);
  for (int i = 0; i < count; i++) {
    if (t[i].n <= 0 || !t[i].p || !t[i].g || !t[i].m || !t[i].v || (bits == 8 && (!t[i].me || !t[i].ve))) return NTB_ERR_ARG;
    const uintptr_t p = reinterpret_cast<uintptr_t>(t[i].p), g = reinterpret_cast<uintptr_t>(t[i].g), s = reinterpret_cast<uintptr_t>(t[i].m) | reinterpret_cast<uintptr_t>(t[i].v);
    t[i].vec = p % (p_dtype == NTB_F32 ? 16 : 8) == 0 && g % (g_dtype == NTB_F32 ? 16 : 8) == 0 && s % (bits == 32 ? 16 : 4) == 0 && reinterpret_cast<uintptr_t>(t[i].half) % 8 == 0;
  }
  AmHyper hy = {b1, omb1, b2, omb2, eps, 1.f / bias_correction1, rsqrtf(bias_correction2), grad_scale};
  if (p_dtype == NTB_F32 && g_dtype == NTB_F32) return am_dispatch<float, float>(t, count, bits, hy, num_sms, stream);
  if (p_dtype == NTB_F32 && g_dtype == NTB_BF16) return am_dispatch<float, __nv_bfloat16>(t, count, bits, hy, num_sms, stream);
  if (p_dtype == NTB_BF16 && g_dtype == NTB_F32) return am_dispatch<__nv_bfloat16, float>(t, count, bits, hy, num_sms, stream);
  if (p_dtype == NTB_BF16 && g_dtype == NTB_BF16) return am_dispatch<__nv_bfloat16, __nv_bfloat16>(t, count, bits, hy, num_sms, stream);
  return NTB_ERR_ARG;
}

// codes [n], exps [ceil(n / 128)] -> out [n] (fp32 or bf16; both hold every value exactly).
NTB_EXPORT int ntb_q8_decode(const void* codes, const void* exps, void* out, int64_t n, int is_signed, int out_dtype, cudaStream_t stream) {
  if (n <= 0) return NTB_ERR_ARG;
  const int64_t want = ((n + AM_BLOCK - 1) / AM_BLOCK + 7) / 8;
  const unsigned grid = static_cast<unsigned>(want < 148 * 32 ? want : 148 * 32);
  const uint8_t *c = static_cast<const uint8_t*>(codes), *e = static_cast<const uint8_t*>(exps);
  const int aligned = reinterpret_cast<uintptr_t>(c) % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (out_dtype == NTB_F32 ? 16 : 8) == 0;
  if (out_dtype == NTB_F32) {
    if (is_signed) q8_decode_kernel<float, true><<<grid, 256, 0, stream>>>(c, e, static_cast<float*>(out), n, aligned);
    else q8_decode_kernel<float, false><<<grid, 256, 0, stream>>>(c, e, static_cast<float*>(out), n, aligned);
  } else if (out_dtype == NTB_BF16) {
    if (is_signed) q8_decode_kernel<__nv_bfloat16, true><<<grid, 256, 0, stream>>>(c, e, static_cast<__nv_bfloat16*>(out), n, aligned);
    else q8_decode_kernel<__nv_bfloat16, false><<<grid, 256, 0, stream>>>(c, e, static_cast<__nv_bfloat16*>(out), n, aligned);
  } else {
    return NTB_ERR_ARG;
  }
  return ntb_check_launch();
}

NTB_EXPORT int ntb_q8_encode(const float* x, void* codes, void* exps, int64_t n, int is_signed, cudaStream_t stream) {
  if (n <= 0) return NTB_ERR_ARG;
  const int64_t want = ((n + AM_BLOCK - 1) / AM_BLOCK + 7) / 8;
  const unsigned grid = static_cast<unsigned>(want < 148 * 32 ? want : 148 * 32);
  uint8_t *c = static_cast<uint8_t*>(codes), *e = static_cast<uint8_t*>(exps);
  const int aligned = reinterpret_cast<uintptr_t>(c) % 4 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  if (is_signed) q8_encode_kernel<true><<<grid, 256, 0, stream>>>(x, c, e, n, aligned);
  else q8_encode_kernel<false><<<grid, 256, 0, stream>>>(x, c, e, n, aligned);
  return ntb_check_launch();
}
