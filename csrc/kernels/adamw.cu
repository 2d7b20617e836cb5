// An AdamW step over many tensors in one launch, with states in 32 or 8 bits.
//
//   g = c g;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p - lr ((m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps) + wd p)
//
// with c the clipping factor of a given norm.  The reference's workers computed their updates in the (absent) Caffe application;
// this is the worker-side optimizer beside the shards' momentum SGD (ps_fabric.cu).
//
// States in 8 bits: a block of 128 values has an exponent byte E for m and one for v, and each value the upper bits of an fp32
// number relative to it: code = (bits >> 20) - base, which keeps three bits of the mantissa.  v: 8 bits, base = 8 E - 248, so the
// block's largest value has a code of 248 to 255 and the smallest is 2^-31 of it; m: a sign and 7 bits, base = 8 E - 120, down to
// 2^-15.  Code 0 is zero.  A v that is not zero gets code 1 at least: a zero would leave eps alone under the quotient.  Without
// subnormals every code costs an addition and a shift each way, and infinities and NaN go through as they are (with them in a block,
// E is 255 and its finite values vanish or become v's least).
// An exponential mean moves by (1 - b) of its value a step, less than half of the distance between two codes, so nearest rounding
// leaves it where it is.  Stochastic rounding adds 16 random bits below the last one that is kept: from code 1 on the mean of the
// rounded values is the value.  Below, m has less: from 2^-15 (of the power of two at or below the block's largest) to code 1, 9/8 of that,
// it becomes 0 or code 1 by the distance from the two, and under 2^-15 always 0, where v becomes code 1.  A parameter whose
// gradients are that much smaller than those of its 128 neighbours so moves by its decay alone.
// The bits come from a hash of seed, step and place (the finaliser of the splittable generator of Steele, Lea and Flood, as in the
// dropout kernel), 64 for two neighbours.
// m and v are rounded after every operation (no fused multiply-add), so that their codes do not depend on how they are compiled.
//
// Bound by memory with states in 32 bits (28 bytes a value with fp32 parameters and gradients); with 8 by the latency of some 76 instructions a
// value, at 2.3 of 4 a cycle from 24 warps an SM (61 M fp32 216 us, floor 149).
// A warp takes a block of 128 a step, four neighbouring values a lane where the tensors' addresses allow vectors, else every 32nd:
// both are whole lines, and a block's largest value is one reduction over the warp.  The tensors' table travels in the launch
// arguments.  The step's number is on the device and is moved on by the last block to finish, so a captured step can be replayed.
#include <math.h>

#include "common.cuh"
#include "tensor_list.h"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kUnit = 2;                       // blocks of 128 that a warp has in flight
constexpr int resident(bool bits8, bool sr) { return bits8 || sr ? 3 : 4; }      // blocks of threads an SM

struct Entry { void* p; const void* g; void* out; long long n; int place, first; };     // place: blocks of 128 before its states; first: units before it
template <int MAX>
struct Table {
  Entry e[MAX + 1];                // the last one has the number of units
  unsigned char type[MAX];         // bit 0: p is fp32, 1: g is, 2: out is, 3: decays, 4: vectors
  int n;
};
struct Args {
  void *m, *v;
  unsigned char* exponents;
  unsigned long long* steps;       // steps taken, blocks that are through
  const float *lr_ref, *norm;
  double ln1, ln2;                 // logarithms of the betas
  unsigned long long seed;
  float b1, a1, b2, a2, lr, eps, decay, max_norm;
  int last;                        // the last launch of the step
};
__host__ __device__ inline long long units_of(long long n) { return (n + 128 * kUnit - 1) / (128 * kUnit); }

constexpr uint64_t kGamma = 0x9E3779B97F4A7C15ull;
__device__ __forceinline__ uint64_t mix64_added(uint64_t z) {        // of a z that kGamma has been added to
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
__device__ __forceinline__ uint64_t mix64(uint64_t z) { return mix64_added(z + kGamma); }

struct Step { float c, c1, c2, lr, lr_decay; uint64_t key, key_p; };       // of a launch (lr_decay: of a tensor; keys with kGamma added)

// What a lane has of a block of 128: four values
struct Values { float p[4], g[4], m[4], v[4]; };

// The codes of four values and the exponent of their block.  TOP: the largest code.  r: random bits << 4, + 8, or nearest (even).
// Most instructions of a step in 8 bits are integer ones: sums with limits are one, bytes move by permutations, the multiplications by
// powers of two are IMADs, and what only zeros need stands behind a branch.
template <int TOP, bool SR>
__device__ __forceinline__ uint32_t encode(const float (&f)[4], const uint32_t (&r)[4], uint32_t& exponent) {
  uint32_t mag[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) mag[j] = TOP == 255 ? __float_as_uint(f[j]) : __float_as_uint(f[j]) & 0x7fffffffu;
  const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(mag[0], mag[1]), max(mag[2], mag[3])));
  exponent = min(max((top + 0xFFFFFu) >> 23, 32u), 255u);
  const uint32_t base = ((TOP - 7) - 8 * exponent) << 20, up = base + 8u;      // of (bits >> 20) - base, and half of the last random bit
  int c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // the bits as they are added: r holds 16 of them in its lower (m) or upper half (v)
    const uint32_t add = SR ? (TOP == 255 ? r[j] >> 16 : r[j] & 0xffffu) * 16u + up : 0x7FFFFu + base + ((mag[j] >> 20) & 1u);
    c[j] = __vimin_s32_relu((int)(mag[j] + add) >> 20, TOP);
  }
  if (TOP == 255 && __any_sync(0xffffffffu, min(min(c[0], c[1]), min(c[2], c[3])) == 0)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = mag[j] ? max(c[j], 1) : c[j];
  }
  const uint32_t codes = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  if (TOP == 255) return codes;
  const uint32_t high = __byte_perm(__byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x0073),
                                    __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x0073), 0x5410);
  return codes | (high & 0x80808080u);           // a zero may get a sign
}
// WARP: all lanes of a warp call it together
template <int TOP, bool WARP>
__device__ __forceinline__ void decode(uint32_t codes, uint32_t exponent, float (&f)[4]) {
  const uint32_t mags = TOP == 255 ? codes : codes & 0x7f7f7f7fu, base = (8 * exponent - (TOP - 7)) << 20;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t at16 = __byte_perm(mags, 0, 0x4044 | (j << 8));       // the byte at bits 16 to 23
    uint32_t w = at16 * 16u + base;
    if (TOP != 255) w |= __byte_perm(codes, 0, 0x0444 | (j << 12)) & 0x80000000u;
    f[j] = __uint_as_float(w);
  }
  const bool zeros = TOP == 255 ? ((codes - 0x01010101u) & ~codes & 0x80808080u) != 0 : ((mags + 0x7f7f7f7fu) & 0x80808080u) != 0x80808080u;
  if (WARP ? __any_sync(0xffffffffu, zeros) : zeros) {          // by the whole warp: as selections for each lane it would be done always
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = (mags >> (8 * j) & 255u) ? f[j] : 0.f;
  }
}

// Below this a root that .ftz takes for zero (1.1e-19) shows in its sum with eps.  Kernels of their own: as a branch in the others 181 -> 187 us
// for 33.6 M bf16 in 8 bits
constexpr float kSmallEps = 1e-12f;
// one value: the new states and the parameter's change.  SMALL: beside an eps below kSmallEps roots and sums of every size count, which are
// brought to where the approximations have all their bits by powers of two
template <bool SMALL>
__device__ __forceinline__ float advance(const Args& a, const Step& s, float p, float g, float& m, float& v) {
  g = __fmul_rn(g, s.c);
  m = __fadd_rn(__fmul_rn(m, a.b1), __fmul_rn(g, a.a1));
  v = __fadd_rn(__fmul_rn(v, a.b2), __fmul_rn(__fmul_rn(g, g), a.a2));
  const float d = v * s.c2, up = SMALL && d < 0x1p-60f ? 0x1p64f : 1.f;
  float root, inverse;
  // a step or two of 2^-23 off, as the quotient: a change has 20 bits at least
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(d * up));
  if (SMALL && d < 0x1p-60f) root *= 0x1p-32f;
  const float sum = root + a.eps, far = SMALL && sum < 0x1p-60f ? 0x1p64f : 1.f;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(sum * far));
  const float q = m * s.c1 * inverse;
  return fmaf(-s.lr, SMALL ? q * far : q, -s.lr_decay * p);
}
// 32 random bits of each of a lane's four values, the first of which has the number i: neighbours, or every 32nd
template <bool VEC>
__device__ __forceinline__ void random4(uint64_t key, uint64_t i, uint32_t (&r)[4]) {
  key += i >> 1;
  if (VEC) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint64_t z = mix64_added(key + (j >> 1));
      r[j] = (uint32_t)z;
      r[j + 1] = (uint32_t)(z >> 32);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t z = mix64_added(key + 16 * j);
      r[j] = (uint32_t)(i & 1 ? z >> 32 : z);
    }
  }
}

template <bool F32>
__device__ __forceinline__ void load_vector(const void* p, long long i, float (&f)[4]) {
  if (F32) {
    const float4 v = ld_f4_nc_stream((const float*)p + i);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else {
    uint2 w;
    asm volatile("ld.global.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(w.x), "=r"(w.y) : "l"((const bf16*)p + i));
    f[0] = __uint_as_float(w.x << 16); f[1] = __uint_as_float(w.x & 0xffff0000u);
    f[2] = __uint_as_float(w.y << 16); f[3] = __uint_as_float(w.y & 0xffff0000u);
  }
}
// Four values as bf16: to the nearest, or by random bits below the last one that is kept
template <bool SR>
__device__ __forceinline__ uint2 to_bf16(const float (&f)[4], const uint32_t (&r)[4]) {
  if (SR) {
    const float sum = (f[0] + f[1]) + (f[2] + f[3]);           // not finite if one is not (or if it overflows: then they are looked at)
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(f[j]) + (r[j] & 0xffffu);
    if (__any_sync(0xffffffffu, (__float_as_uint(sum) & 0x7f800000u) == 0x7f800000u)) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((__float_as_uint(f[j]) & 0x7f800000u) == 0x7f800000u) w[j] = (__float_as_uint(f[j]) & 0xffff0000u) | (f[j] != f[j] ? 0x400000u : 0u);
    }
    return make_uint2(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
  }
  return make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
}

// Blocks [b, b + COUNT) of a tensor by a warp.  VEC: whole blocks, vectors.
template <bool BITS8, bool SR, bool SMALL, bool P32, bool G32, bool VEC, int COUNT>
__device__ __forceinline__ void take(const Entry& e, unsigned type, const Args& a, const Step& s, long long b, int lane) {
  Values x[COUNT];
  uint32_t mc[COUNT], vc[COUNT], ex[COUNT];
  const long long left = e.n - b * 128;         // values from the first block's on
  const long long at = b * 128 + (VEC ? lane * 4 : lane), state = (long long)e.place * 128 + at;
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    if (VEC) {
      load_vector<P32>(e.p, at + k * 128, x[k].p);
      load_vector<G32>(e.g, at + k * 128, x[k].g);
      if (BITS8) {
        mc[k] = *(const uint32_t*)((const unsigned char*)a.m + state + k * 128);
        vc[k] = *(const uint32_t*)((const unsigned char*)a.v + state + k * 128);
      } else {
        load_vector<true>(a.m, state + k * 128, x[k].m);
        load_vector<true>(a.v, state + k * 128, x[k].v);
      }
    } else {
      mc[k] = vc[k] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long i = at + k * 128 + 32 * j;
        const bool in = k * 128 + 32 * j + lane < left;
        x[k].p[j] = in ? (P32 ? ((const float*)e.p)[i] : __bfloat162float(((const bf16*)e.p)[i])) : 0.f;
        x[k].g[j] = in ? (G32 ? ((const float*)e.g)[i] : __bfloat162float(((const bf16*)e.g)[i])) : 0.f;
        if (BITS8) {
          mc[k] |= (uint32_t)((const unsigned char*)a.m)[state + k * 128 + 32 * j] << (8 * j);
          vc[k] |= (uint32_t)((const unsigned char*)a.v)[state + k * 128 + 32 * j] << (8 * j);
        } else {
          x[k].m[j] = ((const float*)a.m)[state + k * 128 + 32 * j];
          x[k].v[j] = ((const float*)a.v)[state + k * 128 + 32 * j];
        }
      }
    }
    if (BITS8) ex[k] = ((const unsigned short*)a.exponents)[e.place + b + k];
  }
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    Values& y = x[k];
    if (BITS8) {
      decode<127, true>(mc[k], ex[k] & 255u, y.m);
      decode<255, true>(vc[k], ex[k] >> 8, y.v);
    }
    float change[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) change[j] = advance<SMALL>(a, s, y.p[j], y.g[j], y.m[j], y.v[j]);
    uint32_t r[4] = {};
    if (BITS8) {
      if (SR) {
        random4<VEC>(s.key, (uint64_t)(state + k * 128), r);
      }
      uint32_t em, ev;
      mc[k] = encode<127, SR>(y.m, r, em);
      vc[k] = encode<255, SR>(y.v, r, ev);
      if (lane == 0) ((unsigned short*)a.exponents)[e.place + b + k] = (unsigned short)(em | ev << 8);
    }
    if (!P32 && SR && e.out == nullptr) random4<VEC>(s.key_p, (uint64_t)(state + k * 128), r);
    if (VEC) {
      if (BITS8) {
        *(uint32_t*)((unsigned char*)a.m + state + k * 128) = mc[k];
        *(uint32_t*)((unsigned char*)a.v + state + k * 128) = vc[k];
      } else {
        st_f4((float*)a.m + state + k * 128, make_float4(y.m[0], y.m[1], y.m[2], y.m[3]));
        st_f4((float*)a.v + state + k * 128, make_float4(y.v[0], y.v[1], y.v[2], y.v[3]));
      }
      const long long i = at + k * 128;
      if (e.out != nullptr) {
        if (type & 4) st_f4((float*)e.out + i, make_float4(change[0], change[1], change[2], change[3]));
        else *(uint2*)((bf16*)e.out + i) = make_uint2(pack_bf16x2(change[0], change[1]), pack_bf16x2(change[2], change[3]));
      } else if (P32) {
        st_f4((float*)e.p + i, make_float4(y.p[0] + change[0], y.p[1] + change[1], y.p[2] + change[2], y.p[3] + change[3]));
      } else {
        const float f[4] = {y.p[0] + change[0], y.p[1] + change[1], y.p[2] + change[2], y.p[3] + change[3]};
        *(uint2*)((bf16*)e.p + i) = to_bf16<SR>(f, r);
      }
    } else {
      const float f[4] = {y.p[0] + change[0], y.p[1] + change[1], y.p[2] + change[2], y.p[3] + change[3]};
      uint2 half = make_uint2(0, 0);
      if (!P32 && e.out == nullptr) half = to_bf16<SR>(f, r);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long i = at + k * 128 + 32 * j, si = state + k * 128 + 32 * j;
        if (BITS8) {
          ((unsigned char*)a.m)[si] = (unsigned char)(mc[k] >> (8 * j));
          ((unsigned char*)a.v)[si] = (unsigned char)(vc[k] >> (8 * j));
        } else {
          ((float*)a.m)[si] = y.m[j];
          ((float*)a.v)[si] = y.v[j];
        }
        if (k * 128 + 32 * j + lane < left) {
          if (e.out != nullptr) {
            if (type & 4) ((float*)e.out)[i] = change[j]; else ((bf16*)e.out)[i] = __float2bfloat16(change[j]);
          } else if (P32) {
            ((float*)e.p)[i] = f[j];
          } else {
            ((unsigned short*)e.p)[i] = (unsigned short)((j < 2 ? half.x : half.y) >> (16 * (j & 1)));
          }
        }
      }
    }
  }
}
template <bool BITS8, bool SR, bool SMALL, bool P32, bool G32>
__device__ __forceinline__ void unit(const Entry& e, unsigned type, const Args& a, const Step& s, long long b, int lane) {
  if ((type & 16) && (b + kUnit) * 128 <= e.n) {
    take<BITS8, SR, SMALL, P32, G32, true, kUnit>(e, type, a, s, b, lane);
  } else if ((b + kUnit - 1) * 128 < e.n) {
    take<BITS8, SR, SMALL, P32, G32, false, kUnit>(e, type, a, s, b, lane);
  } else {
    const long long end = (e.n + 127) >> 7;
#pragma unroll 1
    for (; b < end; ++b) take<BITS8, SR, SMALL, P32, G32, false, 1>(e, type, a, s, b, lane);
  }
}

template <bool BITS8, bool SR, bool SMALL, int MAX>
__global__ void __launch_bounds__(kThreads, resident(BITS8, SR))
adamw_kernel(const __grid_constant__ Table<MAX> t, const __grid_constant__ Args a) {
  geeps_pdl_enter();
  __shared__ float correction[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned long long step = a.steps[0] + 1;
  if (threadIdx.x < 2) correction[threadIdx.x] = (float)(-1.0 / expm1((double)step * (threadIdx.x ? a.ln2 : a.ln1)));
  __syncthreads();
  Step s;
  s.c = 1.f;
  if (a.norm != nullptr) {
    const float n = *a.norm;
    if (n > a.max_norm) s.c = __fdiv_rn(a.max_norm, n);
  }
  s.c1 = correction[0];
  s.c2 = correction[1];
  s.lr = a.lr_ref != nullptr ? *a.lr_ref : a.lr;
  const uint64_t key = mix64(a.seed * 0x100000001B3ull + step);
  s.key = key + kGamma;
  s.key_p = mix64(key) + kGamma;
  // all blocks go through the tensors side by side: with a range of its own for each (330 us, 274 for 61M fp32 in 8 bits with the
  // moments' cast; 134M packed 642, 598) memory has five times as many places open
  const int units = t.e[t.n].first;
  int i = 0;
  for (int u = blockIdx.x * kWarps + warp; u < units; u += gridDim.x * kWarps) {
    while (t.e[i + 1].first <= u) ++i;
    const Entry& e = t.e[i];
    const unsigned type = t.type[i];
    const long long b = (long long)(u - e.first) * kUnit;
    s.lr_decay = type & 8 ? s.lr * a.decay : 0.f;
    switch (type & 3) {
      case 0: unit<BITS8, SR, SMALL, false, false>(e, type, a, s, b, lane); break;
      case 1: unit<BITS8, SR, SMALL, true, false>(e, type, a, s, b, lane); break;
      case 2: unit<BITS8, SR, SMALL, false, true>(e, type, a, s, b, lane); break;
      default: unit<BITS8, SR, SMALL, true, true>(e, type, a, s, b, lane); break;
    }
  }
  // every block has read the step's number before it arrives here
  __syncthreads();
  if (a.last && threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(&a.steps[1], 1ull) == gridDim.x - 1) { a.steps[0] = step; a.steps[1] = 0; }
  }
}

// Two codes (bytes 2 i and 2 i + 1) as a pair of bf16, which hold them exactly: upper halves of what decode() makes
template <int TOP>
__device__ __forceinline__ uint32_t decode_pair(uint32_t codes, uint32_t base, int i) {
  const uint32_t two = __byte_perm(codes, 0, i ? 0x4342 : 0x4140);
  if (TOP == 255) return two * 16u + base;
  return ((two & 0x007f007fu) * 16u + base) | (two & 0x00800080u) << 8;
}
// What the codes stand for: 16 of them a thread
template <bool F32, int TOP>
__global__ void __launch_bounds__(256)
moments_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exponents, void* __restrict__ out, long long n16) {
  geeps_pdl_enter();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n16; i += (long long)gridDim.x * 256) {
    const uint4 w = ((const uint4*)codes)[i];
    const uint32_t c[4] = {w.x, w.y, w.z, w.w}, e = exponents[(i >> 3) * 2 + (TOP == 255 ? 1 : 0)];
    if (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[4];
        decode<TOP, false>(c[j], e, f);
        st_f4((float*)out + i * 16 + 4 * j, make_float4(f[0], f[1], f[2], f[3]));
      }
    } else {
      const uint32_t base = ((8 * e - (TOP - 7)) << 4) * 0x10001u;
      uint32_t o[8];
      bool zeros = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t mags = TOP == 255 ? c[j] : c[j] & 0x7f7f7f7fu;
        zeros |= TOP == 255 ? ((c[j] - 0x01010101u) & ~c[j] & 0x80808080u) != 0 : ((mags + 0x7f7f7f7fu) & 0x80808080u) != 0x80808080u;
        o[2 * j] = decode_pair<TOP>(c[j], base, 0);
        o[2 * j + 1] = decode_pair<TOP>(c[j], base, 1);
      }
      if (zeros) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (!(c[j >> 2] >> (8 * (j & 3)) & (TOP == 255 ? 255u : 127u))) o[j >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
      }
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"((uint4*)out + 2 * i), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]),
                   "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");       // a whole sector
    }
  }
}

template <bool SMALL, int MAX>
int run(const GeepsAdamW& k, cudaStream_t st) {
  const GeepsTensors &p = *k.params, &g = *k.grads;
  Table<MAX> t;
  Args a = {};
  a.m = k.m; a.v = k.v; a.exponents = k.exponents; a.steps = k.steps; a.lr_ref = k.lr_ref; a.norm = k.norm;
  a.ln1 = log(k.beta1); a.ln2 = log(k.beta2); a.seed = k.seed;
  a.b1 = (float)k.beta1; a.a1 = (float)(1.0 - k.beta1); a.b2 = (float)k.beta2; a.a2 = (float)(1.0 - k.beta2);
  a.lr = k.lr; a.eps = k.eps; a.decay = k.weight_decay; a.max_norm = k.max_norm;
  long long place = 0;
  for (long long from = 0; from == 0 || from < p.n; from += MAX) {
    t.n = (int)(p.n - from < MAX ? p.n - from : MAX);
    long long units = 0;
    for (int i = 0; i < t.n; ++i) {
      const long long j = from + i, n = p.count[j];
      Entry& e = t.e[i];
      e.p = p.ptr[j]; e.g = g.ptr[j]; e.out = k.out ? k.out->ptr[j] : nullptr; e.n = n;
      e.place = (int)place; e.first = (int)units;
      const bool out32 = k.out && k.out->fp32[j];
      const bool vec = (((uintptr_t)e.p & (p.fp32[j] ? 15 : 7)) | ((uintptr_t)e.g & (g.fp32[j] ? 15 : 7)) | ((uintptr_t)e.out & (out32 ? 15 : 7))) == 0;
      t.type[i] = (p.fp32[j] ? 1 : 0) | (g.fp32[j] ? 2 : 0) | (out32 ? 4 : 0) | (k.decay[j] ? 8 : 0) | (vec ? 16 : 0);
      place += (n + 127) >> 7;
      units += units_of(n);
      if (place > 0x7fffffffLL || units > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    }
    t.e[t.n].first = (int)units;
    a.last = from + MAX >= p.n;
    const long long most = (long long)geeps_sm_count() * resident(k.bits == 8, k.stochastic), want = (units + kWarps - 1) / kWarps;
    const int blocks = (int)(want < 1 ? 1 : want < most ? want : most);
    auto kernel = k.bits == 8 ? (k.stochastic ? adamw_kernel<true, true, SMALL, MAX> : adamw_kernel<true, false, SMALL, MAX>)
                              : (k.stochastic ? adamw_kernel<false, true, SMALL, MAX> : adamw_kernel<false, false, SMALL, MAX>);
    geeps_launch(kernel, dim3(blocks), dim3(kThreads), 0, st, t, a);
  }
  return (int)cudaGetLastError();
}

}  // namespace

extern "C" int geeps_adamw(const GeepsAdamW* k, void* stream) {
  if (!k || !k->params || !k->grads || !k->steps || !k->decay || (k->bits != 8 && k->bits != 32)) return (int)cudaErrorInvalidValue;
  const GeepsTensors &p = *k->params, &g = *k->grads;
  if (p.n < 0 || g.n != p.n || (k->out && k->out->n != p.n)) return (int)cudaErrorInvalidValue;
  if (!(k->beta1 >= 0 && k->beta1 < 1 && k->beta2 >= 0 && k->beta2 < 1 && k->eps >= 0)) return (int)cudaErrorInvalidValue;
  long long blocks = 0;
  for (long long i = 0; i < p.n; ++i) {
    if (p.count[i] < 0 || g.count[i] != p.count[i] || (k->out && k->out->count[i] != p.count[i])) return (int)cudaErrorInvalidValue;
    if (p.count[i] && (!p.ptr[i] || !g.ptr[i] || (k->out && !k->out->ptr[i]))) return (int)cudaErrorInvalidValue;
    blocks += (p.count[i] + 127) >> 7;
  }
  if (blocks > k->blocks || (blocks && (!k->m || !k->v || (k->bits == 8 && !k->exponents)))) return (int)cudaErrorInvalidValue;
  const int size = k->bits / 8;
  if ((((uintptr_t)k->m | (uintptr_t)k->v) & (size == 4 ? 15 : 3)) || ((uintptr_t)k->exponents & 1) || ((uintptr_t)k->steps & 7) ||
      ((uintptr_t)k->lr_ref & 3) || ((uintptr_t)k->norm & 3) || tensors_between(p) || tensors_between(g) || (k->out && tensors_between(*k->out)))
    return GEEPS_ERR_CLIP_ALIGN;
  if (tensors_overlap(p) || tensors_overlap(g)) return GEEPS_ERR_CLIP_OVERLAP;
  // out[i] may be grads[i]; parameters share memory with nothing
  auto apart = [](const GeepsTensors& x, const GeepsTensors& y) {
    for (long long i = 0; i < x.n; ++i)
      if (tensors_meet(y, x.ptr[i], (unsigned long long)x.count[i] * (x.fp32[i] ? 4 : 2))) return false;
    return true;
  };
  if (!apart(p, g) || (k->out && (tensors_overlap(*k->out) || !apart(p, *k->out) || tensors_overlap(g, *k->out)))) return GEEPS_ERR_CLIP_OVERLAP;
  const struct { const void* at; unsigned long long bytes; bool written; } own[] = {
      {k->m, (unsigned long long)blocks * 128 * size, true}, {k->v, (unsigned long long)blocks * 128 * size, true},
      {k->bits == 8 ? k->exponents : nullptr, (unsigned long long)blocks * 2, true}, {k->steps, 16, true}, {k->lr_ref, 4, false}, {k->norm, 4, false}};
  for (const auto& o : own)
    if (tensors_meet(p, o.at, o.bytes) || (k->out && tensors_meet(*k->out, o.at, o.bytes)) || (o.written && tensors_meet(g, o.at, o.bytes)))
      return GEEPS_ERR_CLIP_OVERLAP;
  for (const auto& x : own)
    for (const auto& y : own)
      if (&x != &y && x.written && x.at && y.at && x.bytes && (uintptr_t)x.at < (uintptr_t)y.at + y.bytes && (uintptr_t)y.at < (uintptr_t)x.at + x.bytes)
        return GEEPS_ERR_CLIP_OVERLAP;
  cudaStream_t st = (cudaStream_t)stream;
  return k->eps < kSmallEps ? run<true, 512>(*k, st) : p.n <= 32 ? run<false, 32>(*k, st) : run<false, 512>(*k, st);
}

extern "C" int geeps_adamw_moments(const unsigned char* codes, const unsigned char* exponents, void* out, int second, int fp32, long long blocks, void* stream) {
  if (blocks == 0) return 0;
  if (blocks < 0 || !codes || !exponents || !out || ((uintptr_t)codes & 15) || ((uintptr_t)out & 31)) return (int)cudaErrorInvalidValue;
  const long long n16 = blocks * 8, want = (n16 + 255) / 256, most = (long long)geeps_sm_count() * 8;
  auto kernel = second ? (fp32 ? moments_kernel<true, 255> : moments_kernel<false, 255>) : (fp32 ? moments_kernel<true, 127> : moments_kernel<false, 127>);
  geeps_launch(kernel, dim3((unsigned)(want < most ? want : most)), dim3(256), 0, (cudaStream_t)stream, codes, exponents, out, n16);
  return (int)cudaGetLastError();
}
