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
// A warp takes blocks of 128 elements as 32 lanes x 4 (every access of a warp is one contiguous 128 .. 512 byte segment), so the largest
// magnitude of a block is one redux over the warp.  32-bit states are bound by HBM: 243 M elements at 30 bytes in 1.13 ms, 6.4 TB/s, the
// copy rate.  With 8-bit states (18 bytes with fp32 master, gradient and bf16 copy; 10 with bf16 parameters and gradients) the integer
// work of the codes shows: about 40 of 70 instructions an element are for the ALU pipe, which takes one every two cycles.  436 M elements
// at 18 bytes in 1.34 ms, 5.9 TB/s; 112 M at 10 bytes in 0.32 ms, 3.5 TB/s, the ALU pipe busy 79 % of the time.  What led there from 1.91
// and 0.68 ms: exponents written for four blocks at once (two byte stores per block alone held the kernel to 2.1 G blocks a second), codes
// and signs placed by byte permutes, shifts as multiply-adds, clamps in one instruction, a path without edge tests for whole chunks.
#include "common.cuh"

namespace {

constexpr int AM_THREADS = 256;
constexpr int AM_BLOCK = 128;                                       // elements per state block: one warp, four elements a lane
constexpr int AM_WARP_BLOCKS = 4;                                   // consecutive blocks of a warp: their exponents are one access of four lanes
constexpr int AM_UNROLL = 2;                                        // of these, in flight
constexpr int AM_CTAS = 4;                                          // resident CTAs per SM
constexpr int AM_WARP_ELEMS = AM_BLOCK * AM_WARP_BLOCKS;
constexpr int AM_CHUNK = AM_WARP_ELEMS * (AM_THREADS / 32);        // elements per CTA and iteration

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
  uint32_t key;         // of the random bits; in: the tensor's position in the list
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
  uint32_t by4, by8;  // AmShift
  float one;
};

// Two fp32 operations at a time, each rounded by itself.  The sum is written as a fused multiply-add with a factor of 1 that the
// compiler does not know: ptxas contracts mul.rn.f32x2 + add.rn.f32x2 into one fused operation (a quarter of the sums then differ in
// their last bit from separately rounded ones, and some 3e-7 of the codes with them); a product by 1 leaves it nothing to contract.
struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 mul_rn(F2 a, F2 b) {
  F2 c;
  asm("{ .reg .b64 a, b, c; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 c, a, b; mov.b64 {%0, %1}, c; }" : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return c;
}
__device__ __forceinline__ F2 add_rn(F2 a, F2 b, float one) {
  F2 c;
  asm("{ .reg .b64 a, b, c, o; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 o, {%6, %6}; fma.rn.f32x2 c, a, o, b; mov.b64 {%0, %1}, c; }"
      : "=f"(c.x), "=f"(c.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(one));
  return c;
}

// Integer mixing (xor-shift, multiply, twice), constants of C. Wellons' published low-bias 32-bit hash.
__host__ __device__ __forceinline__ uint32_t am_mix_early(uint32_t x) {  // all but the last exchange of halves
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  return x * 0x846ca68bu;
}
__host__ __device__ __forceinline__ uint32_t am_mix(uint32_t x) {
  x = am_mix_early(x);
  return x ^ (x >> 16);
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Powers of two as kernel parameters: a multiplication by a value that the compiler does not know is an integer multiply-add on the
// FMA pipe, where a shift or a shift-add would go to the ALU pipe that bounds the 8-bit form (see the kernel).
struct AmShift {
  uint32_t by4, by8;  // 16, 256
};

// Four codes at a time; the window of a block is fixed once per block.
template <bool SIGNED> struct Q8 {
  static constexpr int TOP = SIGNED ? 127 : 255;
  uint32_t E;
  __device__ __forceinline__ explicit Q8(uint32_t E_) : E(E_) {}
  __device__ __forceinline__ int e8() const { return static_cast<int>(8 * E) - (TOP - 7); }  // code + e8 = fp32 bit pattern >> 20
  __device__ __forceinline__ bool nan() const { return E == 255u; }
  __device__ __forceinline__ float factor(float b) const { return nan() ? __int_as_float(0x7fffffff) : b; }

  // without the NaN of a block that is not finite: the caller multiplies by `factor(...)`
  __device__ __forceinline__ void decode(uint32_t c, const AmShift& sh, float (&f)[4]) const {
    const uint32_t lo = static_cast<uint32_t>(max(1, 8 - e8())) << 16;  // the first code of a normal number: 1, or more where the window ends below 2^-126
    const uint32_t low = static_cast<uint32_t>(e8()) << 20;
    const uint32_t mag = SIGNED ? c & 0x7f7f7f7fu : c, sign = c & 0x80808080u;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t k = __byte_perm(mag, 0, 0x4044 | (j << 8));  // code << 16
      uint32_t bits = k * sh.by4 + low;
      bits = k < lo ? 0u : bits;
      if (SIGNED) bits = __byte_perm(sign, 0, 0x4044 | (j << 8)) * sh.by8 + bits;
      f[j] = __uint_as_float(bits);
    }
  }

  // share[j]: 16 random bits << 4 | 8
  __device__ __forceinline__ uint32_t encode(const float (&f)[4], const uint32_t (&share)[4], const AmShift& sh) const {
    uint32_t w[4];  // the code in the top byte
    if (E - (SIGNED ? 16u : 32u) < 255u - (SIGNED ? 16u : 32u)) {
      // finite, and the whole window is normal numbers: what is below it (zero too, for m) comes out negative.  The clamp to the largest
      // code and to zero is one instruction; v's smallest code is 1, so its window is shifted by one around the clamp.
      const uint32_t low = (static_cast<uint32_t>(e8()) + (SIGNED ? 0u : 1u)) << 20;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t size = SIGNED ? __float_as_uint(f[j]) & 0x7fffffffu : __float_as_uint(f[j]);  // a mean of squares has no sign
        const int u = __vimin_s32_relu(static_cast<int>(size + share[j] - low), ((TOP - (SIGNED ? 0 : 1)) << 20) | 0xfffff);
        w[j] = static_cast<uint32_t>(u) * sh.by4 + (SIGNED ? 0u : 1u << 24);
        if (!SIGNED) w[j] = size < 0x800000u ? 0u : w[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t size = __float_as_uint(f[j]) & 0x7fffffffu;
        const int c = min(max(static_cast<int>((size + share[j]) >> 20) - e8(), SIGNED ? 0 : 1), TOP);
        w[j] = (size < 0x800000u || nan()) ? 0u : static_cast<uint32_t>(c) << 24;
      }
    }
    uint32_t codes = __byte_perm(__byte_perm(w[0], w[1], 0x0073), __byte_perm(w[2], w[3], 0x0073), 0x5410);
    if (SIGNED) {
      // the signs, where the code is not zero (bytes hold at most 127, so adding 127 carries into a byte's top bit exactly there)
      const uint32_t sign = __byte_perm(__byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x0073), __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x0073), 0x5410);
      codes |= sign & (codes + 0x7f7f7f7fu) & 0x80808080u;
    }
    return codes;
  }

  static __device__ __forceinline__ uint32_t largest(const float (&f)[4]) {  // exponent field of the warp's 128 values
    uint32_t a[4];
#pragma unroll
    for (int j = 0; j < 4; j++) a[j] = __float_as_uint(f[j]) & 0x7fffffffu;
    return __reduce_max_sync(0xffffffffu, max(__vimax3_u32(a[0], a[1], a[2]), a[3])) >> 23;
  }
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

// One block of 128 elements, four a lane: element i0 + 4 lane .. of a tensor of n elements (32-bit offsets from the block's own
// pointers).  FULL: all of them exist and every pointer is aligned for four at a time.
template <typename P, typename G, int BITS> struct AmBlock {
  float p[4], g[4], m[4], v[4];
  uint32_t mc, vc, me, ve;

  template <bool FULL> __device__ __forceinline__ void load(const AmTensor& t, int64_t b0, int lane) {
    const int64_t i = b0 + lane * 4;
    const bool vec = FULL || (t.vec && i + 3 < t.n);
    load4<P>(static_cast<const P*>(t.p), i, t.n, vec, p);
    load4<G>(static_cast<const G*>(t.g), i, t.n, vec, g);
    if constexpr (BITS == 32) {
      load4<float>(static_cast<const float*>(t.m), i, t.n, vec, m);
      load4<float>(static_cast<const float*>(t.v), i, t.n, vec, v);
    } else {
      mc = load4(static_cast<const uint8_t*>(t.m), i, t.n, vec);
      vc = load4(static_cast<const uint8_t*>(t.v), i, t.n, vec);
    }
  }

  // 8-bit states: me, ve are the block's exponents, replaced by the new ones (not stored).
  template <bool FULL> __device__ __forceinline__ void step(const AmTensor& t, const AmHyper& hy, float gs, int64_t b0, int lane) {
    const int64_t i = b0 + lane * 4;
    const bool vec = FULL || (t.vec && i + 3 < t.n);
    if constexpr (BITS == 32) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float gj = g[j] * gs;
        m[j] = hy.b1 * m[j] + hy.omb1 * gj;
        v[j] = hy.b2 * v[j] + hy.omb2 * gj * gj;
      }
    } else {
      const AmShift sh = {hy.by4, hy.by8};
      const Q8<true> qm(me);
      const Q8<false> qv(ve);
      qm.decode(mc, sh, m);
      qv.decode(vc, sh, v);
      const float b1 = qm.factor(hy.b1), b2 = qv.factor(hy.b2);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const F2 gj = mul_rn(F2{g[j], g[j + 1]}, F2{gs, gs});
        const F2 mj = add_rn(mul_rn(F2{m[j], m[j + 1]}, F2{b1, b1}), mul_rn(gj, F2{hy.omb1, hy.omb1}), hy.one);
        const F2 vj = add_rn(mul_rn(F2{v[j], v[j + 1]}, F2{b2, b2}), mul_rn(mul_rn(gj, gj), F2{hy.omb2, hy.omb2}), hy.one);
        m[j] = mj.x; m[j + 1] = mj.y;
        v[j] = vj.x; v[j + 1] = vj.y;
      }
    }
    const float keep = 1.f - t.lr * t.wd, size = t.lr * hy.inv_bc1;
#pragma unroll
    for (int j = 0; j < 4; j++) p[j] = p[j] * keep - size * m[j] * rcp(sqrtf(v[j]) * hy.inv_sqrt_bc2 + hy.eps);
    store4<P>(static_cast<P*>(t.p), i, t.n, vec, p);
    if (t.half != nullptr) store4<__nv_bfloat16>(t.half, i, t.n, vec, p);
    if constexpr (BITS == 32) {
      store4<float>(static_cast<float*>(t.m), i, t.n, vec, m);
      store4<float>(static_cast<float*>(t.v), i, t.n, vec, v);
    } else {
      if constexpr (!FULL) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (i + j >= t.n) m[j] = v[j] = 0.f;  // what lies behind the tensor has no part in the block's largest
      }
      const uint32_t Em = Q8<true>::largest(m), Ev = Q8<false>::largest(v);
      uint32_t rm[4], rv[4];
      const uint32_t at = static_cast<uint32_t>(i) ^ (t.key + static_cast<uint32_t>(static_cast<uint64_t>(i) >> 32) * 0x9e3779b9u);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t r = am_mix_early(at ^ static_cast<uint32_t>(j));  // i is a multiple of four
        rm[j] = ((r ^ (r >> 16)) & 0xffffu) * hy.by4 + 8u;                // the last step of the mix changes only the lower half
        rv[j] = ((r >> 12) & 0xffff0u) | 8u;
      }
      const AmShift sh = {hy.by4, hy.by8};
      store4(static_cast<uint8_t*>(t.m), i, t.n, vec, Q8<true>(Em).encode(m, rm, sh));
      store4(static_cast<uint8_t*>(t.v), i, t.n, vec, Q8<false>(Ev).encode(v, rv, sh));
      me = Em;
      ve = Ev;
    }
  }
};

template <typename P, typename G, int BITS, int CAP>
__global__ void __launch_bounds__(AM_THREADS, AM_CTAS) adamw_multi_kernel(const __grid_constant__ AmTable<CAP> tab, const __grid_constant__ AmHyper hy) {
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
    const int64_t base = static_cast<int64_t>(chunk - tab.first[lo]) * AM_CHUNK + warp * AM_WARP_ELEMS;
    if (t.vec && base + AM_WARP_ELEMS <= t.n) {
      uint32_t me = 0, ve = 0, men = 0, ven = 0;
      if constexpr (BITS == 8) {
        me = t.me[base / AM_BLOCK + lane % AM_WARP_BLOCKS];
        ve = t.ve[base / AM_BLOCK + lane % AM_WARP_BLOCKS];
      }
#pragma unroll
      for (int h = 0; h < AM_WARP_BLOCKS; h += AM_UNROLL) {
        AmBlock<P, G, BITS> b[AM_UNROLL];
#pragma unroll
        for (int u = 0; u < AM_UNROLL; u++) b[u].template load<true>(t, base + (h + u) * AM_BLOCK, lane);
#pragma unroll
        for (int u = 0; u < AM_UNROLL; u++) {
          if constexpr (BITS == 8) {
            b[u].me = __shfl_sync(0xffffffffu, me, h + u);
            b[u].ve = __shfl_sync(0xffffffffu, ve, h + u);
          }
          b[u].template step<true>(t, hy, gs, base + (h + u) * AM_BLOCK, lane);
          if (lane == h + u) men = b[u].me, ven = b[u].ve;
        }
      }
      if (BITS == 8 && lane < AM_WARP_BLOCKS) {
        t.me[base / AM_BLOCK + lane] = static_cast<uint8_t>(men);
        t.ve[base / AM_BLOCK + lane] = static_cast<uint8_t>(ven);
      }
    } else {
#pragma unroll 1
      for (int u = 0; u < AM_WARP_BLOCKS; u++) {
        const int64_t b0 = base + u * AM_BLOCK;
        if (b0 >= t.n) break;  // the whole warp
        AmBlock<P, G, BITS> b;
        b.template load<false>(t, b0, lane);
        if constexpr (BITS == 8) b.me = t.me[b0 / AM_BLOCK], b.ve = t.ve[b0 / AM_BLOCK];
        b.template step<false>(t, hy, gs, b0, lane);
        __syncwarp();  // every lane has read the exponents
        if (BITS == 8 && lane == 0) t.me[b0 / AM_BLOCK] = static_cast<uint8_t>(b.me), t.ve[b0 / AM_BLOCK] = static_cast<uint8_t>(b.ve);
      }
    }
  }
}

// Eight codes a thread (sixteen threads share a block), two such groups in flight.
template <typename T, bool SIGNED>
__global__ void __launch_bounds__(256) q8_decode_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, T* __restrict__ out, int64_t n, int aligned, AmShift sh) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256 * 8;
  for (int64_t i0 = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; i0 < n; i0 += 2 * stride) {
    uint2 c[2];
    uint32_t E[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int64_t i = i0 + u * stride;
      if (i >= n) continue;
      E[u] = exps[i / AM_BLOCK];
      if (aligned && i + 7 < n) c[u] = *reinterpret_cast<const uint2*>(codes + i);
      else c[u] = make_uint2(load4(codes, i, n, false), load4(codes, i + 4, n, false));
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int64_t i = i0 + u * stride;
      if (i >= n) continue;
      const Q8<SIGNED> q(E[u]);
      float a[4], b[4], f[8];
      q.decode(c[u].x, sh, a);
      q.decode(c[u].y, sh, b);
#pragma unroll
      for (int j = 0; j < 4; j++) f[j] = q.nan() ? q.factor(0.f) : a[j], f[j + 4] = q.nan() ? q.factor(0.f) : b[j];
      if (aligned && i + 7 < n) {
        Vec8<T> o;
        o.from_float(f);
        o.store(out + i);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (i + j < n) out[i + j] = from_f<T>(f[j]);
      }
    }
  }
}

// One warp per block of 128.  To the nearest code (ties away from zero): what a decoded block encodes to is the block itself.
template <bool SIGNED>
__global__ void __launch_bounds__(256) q8_encode_kernel(const float* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ exps, int64_t n, int aligned) {
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (n + AM_BLOCK - 1) / AM_BLOCK;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); b < blocks; b += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t i = b * AM_BLOCK + lane * 4;
    const bool vec = aligned && i + 3 < n;
    float f[4];
    load4<float>(x, i, n, vec, f);
    const uint32_t E = Q8<SIGNED>::largest(f), half[4] = {0x80008u, 0x80008u, 0x80008u, 0x80008u};
    if (!SIGNED) {
#pragma unroll
      for (int j = 0; j < 4; j++) f[j] = fabsf(f[j]);
    }
    store4(codes, i, n, vec, Q8<SIGNED>(E).encode(f, half, AmShift{16u, 256u}));
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
  const uint64_t cap = static_cast<uint64_t>(num_sms) * AM_CTAS * 4;
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

// table: `count` AmTensor records in host memory (every n > 0; `key` and `vec` are filled in here).  p_dtype / g_dtype: NTB_F32 or NTB_BF16.  bits: 32 or 8.
NTB_EXPORT int ntb_adamw_multi(void* table, int count, int p_dtype, int g_dtype, int bits, float b1, float omb1, float b2, float omb2, float eps, float bias_correction1,
                               float bias_correction2, const float* grad_scale, uint32_t seed, int num_sms, cudaStream_t stream) {
  if (count <= 0 || table == nullptr || (bits != 8 && bits != 32) || num_sms <= 0) return NTB_ERR_ARG;
  AmTensor* t = static_cast<AmTensor*>(table);
  for (int i = 0; i < count; i++) {
    if (t[i].n <= 0 || !t[i].p || !t[i].g || !t[i].m || !t[i].v || (bits == 8 && (!t[i].me || !t[i].ve))) return NTB_ERR_ARG;
    t[i].key = am_mix(seed + 0x9e3779b9u * (t[i].key + 1u));
    const uintptr_t p = reinterpret_cast<uintptr_t>(t[i].p), g = reinterpret_cast<uintptr_t>(t[i].g), s = reinterpret_cast<uintptr_t>(t[i].m) | reinterpret_cast<uintptr_t>(t[i].v);
    t[i].vec = p % (p_dtype == NTB_F32 ? 16 : 8) == 0 && g % (g_dtype == NTB_F32 ? 16 : 8) == 0 && s % (bits == 32 ? 16 : 4) == 0 && reinterpret_cast<uintptr_t>(t[i].half) % 8 == 0;
  }
  AmHyper hy = {b1, omb1, b2, omb2, eps, 1.f / bias_correction1, rsqrtf(bias_correction2), grad_scale, 16u, 256u, 1.f};
  if (p_dtype == NTB_F32 && g_dtype == NTB_F32) return am_dispatch<float, float>(t, count, bits, hy, num_sms, stream);
  if (p_dtype == NTB_F32 && g_dtype == NTB_BF16) return am_dispatch<float, __nv_bfloat16>(t, count, bits, hy, num_sms, stream);
  if (p_dtype == NTB_BF16 && g_dtype == NTB_F32) return am_dispatch<__nv_bfloat16, float>(t, count, bits, hy, num_sms, stream);
  if (p_dtype == NTB_BF16 && g_dtype == NTB_BF16) return am_dispatch<__nv_bfloat16, __nv_bfloat16>(t, count, bits, hy, num_sms, stream);
  return NTB_ERR_ARG;
}

// codes [n], exps [ceil(n / 128)] -> out [n] (fp32 or bf16; both hold every value exactly).
NTB_EXPORT int ntb_q8_decode(const void* codes, const void* exps, void* out, int64_t n, int is_signed, int out_dtype, cudaStream_t stream) {
  if (n <= 0) return NTB_ERR_ARG;
  const int64_t want = (n + 4095) / 4096;
  const unsigned grid = static_cast<unsigned>(want < 148 * 16 ? want : 148 * 16);
  const uint8_t *c = static_cast<const uint8_t*>(codes), *e = static_cast<const uint8_t*>(exps);
  const int aligned = reinterpret_cast<uintptr_t>(c) % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const AmShift sh = {16u, 256u};
  if (out_dtype == NTB_F32) {
    if (is_signed) q8_decode_kernel<float, true><<<grid, 256, 0, stream>>>(c, e, static_cast<float*>(out), n, aligned, sh);
    else q8_decode_kernel<float, false><<<grid, 256, 0, stream>>>(c, e, static_cast<float*>(out), n, aligned, sh);
  } else if (out_dtype == NTB_BF16) {
    if (is_signed) q8_decode_kernel<__nv_bfloat16, true><<<grid, 256, 0, stream>>>(c, e, static_cast<__nv_bfloat16*>(out), n, aligned, sh);
    else q8_decode_kernel<__nv_bfloat16, false><<<grid, 256, 0, stream>>>(c, e, static_cast<__nv_bfloat16*>(out), n, aligned, sh);
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
