// Casts to e4m3 with a scale 2^e for each block of 128: e = the smallest with max |x| 2^-e <= 448, q = x 2^-e to nearest even.
//
// With a power of two x 2^-e is exact, so q is the one rounding of the cast and the same wherever it is computed; the scale loses
// nothing, since the relative error of a float does not depend on where in its range it lies.
//
// Two kernels, both bound by memory.  Rows: a warp takes 512 columns of a row, 16 a lane, eight lanes a block.  Tiles: a
// block of 256 threads keeps 128 x 128 values in registers (8 rows x 8 columns a thread), from which it makes the cast of x, that of
// x transposed (through shared memory) or both, so that a training step reads its gradient once for its two products.
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
  const long long units = rows * quads, step = (long long)gridDim.x * 8;
  for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += step) {
    const long long r = u / quads, qd = u - r * quads, c = qd * 512 + lane * 16;
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
  }
}

// One block of 128 x 128 values.  Thread: columns 8 (tid % 16) to + 7 of rows 8 (tid / 16) to + 7.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256)
quantize_tile_kernel(const GeepsQuantizeFp8 p, unsigned tiles_c, long long quads, long long quads_t) {
  geeps_pdl_enter();
  __shared__ __align__(16) uint2 turned[128 * 16];       // columns of the tile, 16 pieces of eight rows, piece ^ (column / 8)
  __shared__ uint32_t tops[8][128];
  __shared__ uint8_t col_byte[128];
  const int tid = threadIdx.x, c8 = tid & 15, rg = tid >> 4, warp = tid >> 5;
  const long long bc = blockIdx.x % tiles_c, br = blockIdx.x / tiles_c;
  const long long r0 = br * 128 + rg * 8, c0 = bc * 128 + c8 * 8;
  float f[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (r0 + i < p.rows) {
      load<F32, 8, VEC>((const char*)p.x + (r0 + i) * p.ldx * (F32 ? 4 : 2), c0, p.cols, f[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
    }
  }
  uint32_t byte = 0;
  if (p.tile) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, bits(f[i][j]));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((tid & 31) == 0) tops[0][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = max(top, tops[0][w]);
    byte = scale_byte(top);
    if (tid < 128) {
      if (p.q != nullptr) p.scale[scale_at(br * 128 + tid, bc, quads)] = (uint8_t)byte;
      if (p.qt != nullptr) p.scale_t[scale_at(bc * 128 + tid, br, quads_t)] = (uint8_t)byte;
    }
  } else if (p.qt != nullptr) {
    uint32_t top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      top[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top[j] = max(top[j], bits(f[i][j]));
      top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], 16));
    }
    if ((tid & 16) == 0) {
      *reinterpret_cast<uint4*>(&tops[warp][c8 * 8]) = make_uint4(top[0], top[1], top[2], top[3]);
      *reinterpret_cast<uint4*>(&tops[warp][c8 * 8 + 4]) = make_uint4(top[4], top[5], top[6], top[7]);
    }
    __syncthreads();
    if (tid < 128) {
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) t = max(t, tops[w][tid]);
      const uint32_t b = scale_byte(t);
      col_byte[tid] = (uint8_t)b;
      p.scale_t[scale_at(bc * 128 + tid, br, quads_t)] = (uint8_t)b;
    }
    __syncthreads();
  }
  if (p.q != nullptr) {
    const long long pitch = (p.cols + 15) & ~15LL;         // what a row has, with its padding: others may lie behind it
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t b = byte;
      if (!p.tile) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, bits(f[i][j]));
#pragma unroll
        for (int o = 8; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        b = scale_byte(top);
        if (c8 == 0) p.scale[scale_at(r0 + i, bc, quads)] = (uint8_t)b;
      }
      const float inv = inverse(b);
      const uint32_t lo = e4m3x2(f[i][0] * inv, f[i][1] * inv) | e4m3x2(f[i][2] * inv, f[i][3] * inv) << 16;
      const uint32_t hi = e4m3x2(f[i][4] * inv, f[i][5] * inv) | e4m3x2(f[i][6] * inv, f[i][7] * inv) << 16;
      if (r0 + i < p.rows && c0 < pitch) *reinterpret_cast<uint2*>((uint8_t*)p.q + (r0 + i) * p.ldq + c0) = make_uint2(lo, hi);
    }
  }
  if (p.qt != nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float inv = inverse(p.tile ? byte : col_byte[c8 * 8 + j]);
      const uint32_t lo = e4m3x2(f[0][j] * inv, f[1][j] * inv) | e4m3x2(f[2][j] * inv, f[3][j] * inv) << 16;
      const uint32_t hi = e4m3x2(f[4][j] * inv, f[5][j] * inv) | e4m3x2(f[6][j] * inv, f[7][j] * inv) << 16;
      turned[(c8 * 8 + j) * 16 + (rg ^ c8)] = make_uint2(lo, hi);
    }
    __syncthreads();
    // eight lanes write the 128 bytes of a column, 16 each
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int c = s * 32 + (tid >> 3), piece = (tid & 7) * 2, x = c >> 3;
      const uint2 a = turned[c * 16 + (piece ^ x)], b = turned[c * 16 + ((piece + 1) ^ x)];
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
  auto k = p->fp32 ? (vec ? quantize_tile_kernel<true, true> : quantize_tile_kernel<true, false>)
                   : (vec ? quantize_tile_kernel<false, true> : quantize_tile_kernel<false, false>);
  geeps_launch_plain(k, dim3((unsigned)(bc * br)), 256, 0, st, *p, (unsigned)bc, quads, quads_t);
  return (int)cudaGetLastError();
}
