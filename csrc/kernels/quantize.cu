// Casts to e4m3 with a scale 2^e for each block of 128: e = the smallest with max |x| 2^-e <= 448, q = x 2^-e to nearest even.
//
// With a power of two x 2^-e is exact, so q is the one rounding of the cast and the same wherever it is computed; the scale loses
// nothing, since the relative error of a float does not depend on where in its range it lies.
//
// Two kernels, both bound by memory.  Rows: a warp takes 512 columns of a row, 16 a lane, eight lanes a block.  Tiles: a
// block of 256 threads keeps 128 x 128 values in registers as they are in memory (8 rows x 8 columns a thread, 16 bytes a load), from
// which it makes the cast of x, that of x transposed (through shared memory) or both, so that a training step reads its gradient once
// for its two products.  With one scale for the tile the bytes of the cast are those of its transpose, turned by byte permutations.
// 4096 x 4096 bf16 in a captured chain (floor, of reads and writes at 6.54 TB/s): rows 12.1 us (7.7), tile 10.5 (7.7), both 17.6
// (10.3), tile with its transpose 14.3 (10.3); values kept in fp32 (117 registers, two blocks an SM) 27.9, 38.0 and 32.3.
#include "common.cuh"
#include "kernels.h"
#include "nn_ops.h"
#include "tensor_list.h"

namespace {

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// E8M0 byte of a block's scale from the bits of its largest magnitude, and 1 / scale
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7F800000u) return 255u;
  const int e = (int)(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);      // + 127
  return (uint32_t)(e < 0 ? 0 : e);
}
__device__ __forceinline__ float inverse(uint32_t byte) { return __uint_as_float((byte == 255u ? 127u : 254u - byte) << 23); }

__device__ __forceinline__ size_t scale_at(long long r, long long block, long long quads) {
  return ((size_t)(r >> 7) * quads + (block >> 2)) * 512 + ((r & 31) << 4) + (((r & 127) >> 5) << 2) + (block & 3);
}

// V values of a row from column c on, zeros behind the last
template <bool F32, int V, bool VEC>
__device__ __forceinline__ void load(const void* row, long long c, long long cols, float (&f)[V]) {
  if (VEC && c + V <= cols) {
    if (F32) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 v = ld_f4_nc_stream((const float*)row + c + i);
        f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 8) {
        const uint4 v = __ldg((const uint4*)((const __nv_bfloat16*)row + c + i));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[i + 2 * e] = __uint_as_float(w[e] << 16); f[i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
      }
    }
  } else if (!F32 && c + V <= cols) {          // words where there are whole ones
    const __nv_bfloat16* at = (const __nv_bfloat16*)row + c;
    const int odd = (int)((uintptr_t)at >> 1 & 1);
    const uint32_t* words = (const uint32_t*)(at + odd);
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = i < V / 2 - 1 || !odd ? __ldg(words + i) : (uint32_t)__ldg((const unsigned short*)at + V - 1);
    const uint32_t first = odd ? (uint32_t)__ldg((const unsigned short*)at) << 16 : 0u;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const uint32_t pair = odd ? __funnelshift_l(i ? w[i - 1] : first, w[i], 16) : w[i];
      f[2 * i] = __uint_as_float(pair << 16);
      f[2 * i + 1] = __uint_as_float(pair & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      f[i] = c + i < cols ? (F32 ? ((const float*)row)[c + i] : __bfloat162float(((const __nv_bfloat16*)row)[c + i])) : 0.f;
  }
}
__device__ __forceinline__ uint32_t bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

template <bool F32, bool VEC>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const void* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ scale, long long rows, long long cols,
                     long long ldx, long long ldq, long long quads) {
  geeps_pdl_enter();
  const int lane = threadIdx.x & 31;
  const long long ldq_used = (cols + 15) & ~15LL;        // of a row of q, with its padding
  const long long units = rows * quads, step = (long long)gridDim.x * 8;
  for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += step) {
    const long long r = u / quads, qd = u - r * quads;
    if (VEC || !F32) {
      const long long c = qd * 512 + lane * 16;
      float f[16];
      load<F32, 16, VEC>((const char*)x + r * ldx * (F32 ? 4 : 2), c, cols, f);
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, bits(f[i]));
#pragma unroll
      for (int o = 4; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const uint32_t byte = scale_byte(top);
      const float inv = inverse(byte);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = e4m3x2(f[4 * i] * inv, f[4 * i + 1] * inv) | e4m3x2(f[4 * i + 2] * inv, f[4 * i + 3] * inv) << 16;
      if (c < cols) *reinterpret_cast<uint4*>(q + r * ldq + c) = make_uint4(w[0], w[1], w[2], w[3]);
      if ((lane & 7) == 0 && c < cols) scale[scale_at(r, qd * 4 + (lane >> 3), quads)] = (uint8_t)byte;
    } else {
      // fp32 rows that begin anywhere: lanes take neighbours, value i of a lane is column 32 i + lane (4000 x 4003 24.8 us; 16 neighbours a
      // lane 39.5.  In bf16 27.5 and, by words, 15.8.)
      const float* row = (const float*)x + r * ldx + qd * 512 + lane;
      const long long left = cols - qd * 512 - lane;
      float f[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = i * 32 < left ? __ldg(row + i * 32) : 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t byte = scale_byte(__reduce_max_sync(0xffffffffu, max(max(bits(f[4 * b]), bits(f[4 * b + 1])), max(bits(f[4 * b + 2]), bits(f[4 * b + 3])))));
        const float inv = inverse(byte);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long c = qd * 512 + (4 * b + i) * 32 + lane;
          if (c < ldq_used) q[r * ldq + c] = (uint8_t)e4m3x2(f[4 * b + i] * inv, 0.f);
        }
        if (lane == 0 && qd * 512 + b * 128 < cols) scale[scale_at(r, qd * 4 + b, quads)] = (uint8_t)byte;
      }
    }
  }
}

// Eight values of a row as they were loaded, and their magnitudes in 16 bits: sign and lower half of an fp32 number cut off, what is cut
// rounded up, so that a scale formed from the largest one is that of the values.  A finite one stays finite.
template <bool F32>
struct Eight;
template <>
struct Eight<false> {
  uint4 w;
  __device__ __forceinline__ void load(const void* p) {
    const float4 f = ld_f4_nc_stream((const float*)p);
    w = make_uint4(__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w));
  }
  __device__ __forceinline__ void load_any(const void* p) {          // on any two bytes: words where there are whole ones
    const unsigned short* at = (const unsigned short*)p;
    const int odd = (int)((uintptr_t)p >> 1 & 1);
    const uint32_t* words = (const uint32_t*)(at + odd);
    const uint32_t first = odd ? (uint32_t)__ldg(at) << 16 : 0u;
    const uint32_t a = __ldg(words), b = __ldg(words + 1), c = __ldg(words + 2), d = odd ? (uint32_t)__ldg(at + 7) : __ldg(words + 3);
    w = odd ? make_uint4(__funnelshift_l(first, a, 16), __funnelshift_l(a, b, 16), __funnelshift_l(b, c, 16), __funnelshift_l(c, d, 16)) : make_uint4(a, b, c, d);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    w = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
  __device__ __forceinline__ uint32_t word(int j) const { return j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w; }
  __device__ __forceinline__ float get(int j) const { return __uint_as_float(j & 1 ? word(j >> 1) & 0xffff0000u : word(j >> 1) << 16); }
  // of values 2 j and 2 j + 1
  __device__ __forceinline__ uint32_t sizes(int j) const { return word(j) & 0x7fff7fffu; }
};
template <>
struct Eight<true> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* p) { a = ld_f4_nc_stream((const float*)p); b = ld_f4_nc_stream((const float*)p + 4); }
  __device__ __forceinline__ void load_any(const void* p) {
    const float* f = (const float*)p;
    a = make_float4(__ldg(f), __ldg(f + 1), __ldg(f + 2), __ldg(f + 3));
    b = make_float4(__ldg(f + 4), __ldg(f + 5), __ldg(f + 6), __ldg(f + 7));
  }
  __device__ __forceinline__ void set(const float (&f)[8]) { a = make_float4(f[0], f[1], f[2], f[3]); b = make_float4(f[4], f[5], f[6], f[7]); }
  __device__ __forceinline__ float get(int j) const { return j == 0 ? a.x : j == 1 ? a.y : j == 2 ? a.z : j == 3 ? a.w : j == 4 ? b.x : j == 5 ? b.y : j == 6 ? b.z : b.w; }
  static __device__ __forceinline__ uint32_t up(uint32_t b) { return (b < 0x7f800000u ? min(b + 0xffffu, 0x7f7fffffu) : b) >> 16; }
  __device__ __forceinline__ uint32_t sizes(int j) const { return up(bits(get(2 * j))) | up(bits(get(2 * j + 1))) << 16; }
};
// E8M0 byte from the largest magnitude in 16 bits
__device__ __forceinline__ uint32_t scale_byte16(uint32_t top) {
  if (top >= 0x7f80u) return 255u;
  const int e = (int)(top >> 7) - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0);
  return (uint32_t)(e < 0 ? 0 : e);
}
// Bytes of column c (0 to 3) of four rows of four bytes
__device__ __forceinline__ void turn4(const uint32_t (&r)[4], uint32_t (&c)[4]) {
  const uint32_t a = __byte_perm(r[0], r[1], 0x5140), b = __byte_perm(r[0], r[1], 0x7362), d = __byte_perm(r[2], r[3], 0x5140), e = __byte_perm(r[2], r[3], 0x7362);
  c[0] = __byte_perm(a, d, 0x5410); c[1] = __byte_perm(a, d, 0x7632); c[2] = __byte_perm(b, e, 0x5410); c[3] = __byte_perm(b, e, 0x7632);
}

// One block of 128 x 128 values.  Thread: columns 8 (tid % 16) to + 7 of rows 8 (tid / 16) to + 7, kept as loaded.
template <bool F32, bool VEC, bool TILE>
__global__ void __launch_bounds__(256, F32 ? 2 : 3)
quantize_tile_kernel(const GeepsQuantizeFp8 p, unsigned tiles_c, long long quads, long long quads_t) {
  geeps_pdl_enter();
  __shared__ __align__(16) uint2 turned[128 * 16];       // columns of the tile, 16 pieces of eight rows, piece ^ (column / 8)
  __shared__ __align__(16) uint32_t tops[8][64];         // of a warp's columns, in pairs
  __shared__ uint8_t col_byte[128];
  const int tid = threadIdx.x, c8 = tid & 15, rg = tid >> 4, warp = tid >> 5;
  const long long bc = blockIdx.x % tiles_c, br = blockIdx.x / tiles_c;
  const long long r0 = br * 128 + rg * 8, c0 = bc * 128 + c8 * 8;
  Eight<F32> x[8];
  {
    constexpr int SIZE = F32 ? 4 : 2;
    const char* from = (const char*)p.x + (r0 * p.ldx + c0) * SIZE;
    if ((br + 1) * 128 <= p.rows && (bc + 1) * 128 <= p.cols) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (VEC) x[i].load(from + i * p.ldx * SIZE); else x[i].load_any(from + i * p.ldx * SIZE);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f[8];
        if (r0 + i < p.rows) {
          load<F32, 8, VEC>(from + (i * p.ldx - c0) * SIZE, c0, p.cols, f);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = 0.f;
        }
        x[i].set(f);
      }
    }
  }
  // largest magnitudes of a row, of two rows a word, and of columns, likewise
  uint32_t byte = 0, rows[4];
  if (TILE || p.q != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      uint32_t t[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        t[e] = __vimax3_u16x2(x[i + e].sizes(0), x[i + e].sizes(1), __vmaxu2(x[i + e].sizes(2), x[i + e].sizes(3)));
        t[e] = max(t[e] & 0xffffu, t[e] >> 16);
      }
      rows[i >> 1] = t[0] | t[1] << 16;
    }
  }
  if (TILE) {
    uint32_t top = __vimax3_u16x2(rows[0], rows[1], __vmaxu2(rows[2], rows[3]));
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
    if ((tid & 31) == 0) tops[0][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = max(top, tops[0][w]);
    byte = scale_byte16(top);
    if (tid < 128) {
      if (p.q != nullptr) p.scale[scale_at(br * 128 + tid, bc, quads)] = (uint8_t)byte;
      if (p.qt != nullptr) p.scale_t[scale_at(bc * 128 + tid, br, quads_t)] = (uint8_t)byte;
    }
  } else {
    uint32_t cols[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cols[j] = __vmaxu2(x[0].sizes(j), x[1].sizes(j));
#pragma unroll
      for (int i = 2; i < 8; i += 2) cols[j] = __vimax3_u16x2(cols[j], x[i].sizes(j), x[i + 1].sizes(j));
      cols[j] = __vmaxu2(cols[j], __shfl_xor_sync(0xffffffffu, cols[j], 16));
    }
    if ((tid & 16) == 0) *reinterpret_cast<uint4*>(&tops[warp][c8 * 4]) = make_uint4(cols[0], cols[1], cols[2], cols[3]);
    if (p.q != nullptr) {
#pragma unroll
      for (int o = 8; o; o >>= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) rows[i] = __vmaxu2(rows[i], __shfl_xor_sync(0xffffffffu, rows[i], o));
      }
    }
    __syncthreads();
    if (tid < 64) {
      uint32_t t = tops[0][tid];
#pragma unroll
      for (int w = 1; w < 8; ++w) t = __vmaxu2(t, tops[w][tid]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t b = scale_byte16(e ? t >> 16 : t & 0xffffu);
        col_byte[2 * tid + e] = (uint8_t)b;
        p.scale_t[scale_at(bc * 128 + 2 * tid + e, br, quads_t)] = (uint8_t)b;
      }
    }
    __syncthreads();
  }
  uint2 q[8];                      // the rows' bytes, which with one scale are the columns' too
  const long long pitch = (p.cols + 15) & ~15LL;         // what a row has, with its padding: others may lie behind it
  if (TILE || p.q != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t b = byte;
      if (!TILE) {
        b = scale_byte16(i & 1 ? rows[i >> 1] >> 16 : rows[i >> 1] & 0xffffu);
        if (c8 == 0) p.scale[scale_at(r0 + i, bc, quads)] = (uint8_t)b;
      }
      const float inv = inverse(b);
      q[i].x = e4m3x2(x[i].get(0) * inv, x[i].get(1) * inv) | e4m3x2(x[i].get(2) * inv, x[i].get(3) * inv) << 16;
      q[i].y = e4m3x2(x[i].get(4) * inv, x[i].get(5) * inv) | e4m3x2(x[i].get(6) * inv, x[i].get(7) * inv) << 16;
      if (p.q != nullptr && r0 + i < p.rows && c0 < pitch) *reinterpret_cast<uint2*>((uint8_t*)p.q + (r0 + i) * p.ldq + c0) = q[i];
    }
  }
  if (p.qt != nullptr) {
    uint2* to = turned + c8 * 128 + (rg ^ c8);
    if (TILE) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {          // four columns each
        uint32_t r[2][4], c[2][4];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i >> 2][i & 3] = h ? q[i].y : q[i].x;
        turn4(r[0], c[0]);
        turn4(r[1], c[1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) to[(4 * h + j) * 16] = make_uint2(c[0][j], c[1][j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float inv = inverse(col_byte[c8 * 8 + j]);
        const uint32_t lo = e4m3x2(x[0].get(j) * inv, x[1].get(j) * inv) | e4m3x2(x[2].get(j) * inv, x[3].get(j) * inv) << 16;
        const uint32_t hi = e4m3x2(x[4].get(j) * inv, x[5].get(j) * inv) | e4m3x2(x[6].get(j) * inv, x[7].get(j) * inv) << 16;
        to[j * 16] = make_uint2(lo, hi);
      }
    }
    __syncthreads();
    // eight lanes write the 128 bytes of a column, 16 each
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int c = s * 32 + (tid >> 3), piece = (tid & 7) * 2, k = c >> 3;
      const uint2 a = turned[c * 16 + (piece ^ k)], b = turned[c * 16 + ((piece + 1) ^ k)];
      const long long row = bc * 128 + c, at = br * 128 + piece * 8;
      if (row < p.cols && at < ((p.rows + 15) & ~15LL)) *reinterpret_cast<uint4*>((uint8_t*)p.qt + row * p.ldqt + at) = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
}

}  // namespace

extern "C" int geeps_quantize_fp8(const GeepsQuantizeFp8* p, void* stream) {
  const int size = p->fp32 ? 4 : 2;
  if (p->rows < 0 || p->cols < 0 || p->rows > 0x3fffffffLL || p->cols > 0x3fffffffLL) return (int)cudaErrorInvalidValue;
  if (p->rows == 0 || p->cols == 0 || (p->q == nullptr && p->qt == nullptr)) return 0;
  if (p->x == nullptr || ((uintptr_t)p->x & (size - 1)) || p->ldx < p->cols) return (int)cudaErrorInvalidValue;
  if (p->q != nullptr && (((uintptr_t)p->q & 15) || (p->ldq & 15) || p->ldq < p->cols || p->scale == nullptr)) return (int)cudaErrorInvalidValue;
  if (p->qt != nullptr && (((uintptr_t)p->qt & 15) || (p->ldqt & 15) || p->ldqt < p->rows || p->scale_t == nullptr)) return (int)cudaErrorInvalidValue;
  const long long quads = (p->cols + 511) / 512, quads_t = (p->rows + 511) / 512;
  auto bytes = [](long long rows, long long ld, long long cols) { return (rows - 1) * ld + cols; };
  const MemoryRange ranges[] = {{p->q, p->q ? bytes(p->rows, p->ldq, (p->cols + 15) & ~15LL) : 0}, {p->scale, p->q ? (p->rows + 127) / 128 * quads * 512 : 0},
                                {p->qt, p->qt ? bytes(p->cols, p->ldqt, (p->rows + 15) & ~15LL) : 0}, {p->scale_t, p->qt ? (p->cols + 127) / 128 * quads_t * 512 : 0},
                                {p->x, bytes(p->rows, p->ldx, p->cols) * size}};
  if (ranges_overlap(ranges, 4, 5)) return GEEPS_ERR_NORM_OVERLAP;
  const bool vec = ((uintptr_t)p->x & 15) == 0 && p->ldx * size % 16 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (p->qt == nullptr && !p->tile) {
    const long long units = p->rows * quads, most = (long long)geeps_sm_count() * 8, want = (units + 7) / 8;
    auto k = p->fp32 ? (vec ? quantize_rows_kernel<true, true> : quantize_rows_kernel<true, false>)
                     : (vec ? quantize_rows_kernel<false, true> : quantize_rows_kernel<false, false>);
    geeps_launch(k, dim3((unsigned)(want < most ? want : most)), 256, 0, st, p->x, (uint8_t*)p->q, (uint8_t*)p->scale, p->rows, p->cols, p->ldx, p->ldq, quads);
    return (int)cudaGetLastError();
  }
  const long long bc = (p->cols + 127) / 128, br = (p->rows + 127) / 128;
  if (bc * br > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  auto k = p->tile ? (p->fp32 ? (vec ? quantize_tile_kernel<true, true, true> : quantize_tile_kernel<true, false, true>)
                              : (vec ? quantize_tile_kernel<false, true, true> : quantize_tile_kernel<false, false, true>))
                   : (p->fp32 ? (vec ? quantize_tile_kernel<true, true, false> : quantize_tile_kernel<true, false, false>)
                              : (vec ? quantize_tile_kernel<false, true, false> : quantize_tile_kernel<false, false, false>));
  geeps_launch_plain(k, dim3((unsigned)(bc * br)), 256, 0, st, *p, (unsigned)bc, quads, quads_t);
  return (int)cudaGetLastError();
}
