// Clipping of gradients by their global norm: N = sqrt(sum g^2) over all tensors, g = c g with c = max / N where N > max.
//
// The reference's solver had this (clip_gradients of a solver definition) in its Caffe application, which is not part of
// the reference's tree.
//
// Two launches over the same chunks: the first adds the squares, in 64 bits (fp32 squares leave the range from 1.8e19 up and
// from 1e-19 down; the sum of all chunks keeps no rounding that shows in an fp32 norm), the second adds the blocks' sums, in
// block order in every block, and scales.  The second goes through the chunks backwards: what the first read last is still in
// L2.  A tensor table travels in the launch arguments, so a call keeps nothing on the device.
#include "common.cuh"
#include "nn_ops.h"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;                                  // vectors of eight a thread has in flight
constexpr long long kChunk = 8LL * kThreads * kUnits;      // elements a block takes at a time
constexpr int kTensors = 1024;                             // tensors a launch

struct Entry { const void* src; void* dst; long long n; };
template <int MAX>
struct Table {
  Entry e[MAX];
  int first[MAX + 1];              // number of chunks before tensor i
  unsigned char type[MAX];         // bit 0: src is fp32, bit 1: dst is fp32
  int n;
};

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) { f[2 * e] = __uint_as_float(w[e] << 16); f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
}
template <bool F32>
__device__ __forceinline__ void load8(const void* p, float (&f)[8]) {
  if (F32) {
    const float4 lo = ld_f4((const float*)p), hi = ld_f4((const float*)p + 4);
    f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w; f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
  } else {
    unpack8(*(const uint4*)p, f);
  }
}
template <bool F32>
__device__ __forceinline__ float load1(const void* p, long long i) {
  return F32 ? ((const float*)p)[i] : (float)((const bf16*)p)[i];
}

// Chunk k of a tensor of n elements: vectors of eight from the first 16-byte boundary on; the elements before it and behind
// the last whole vector go with chunk 0.
struct Chunk { long long head, from, to, tail; };
template <bool F32>
__device__ __forceinline__ Chunk chunk_of(const void* src, long long n, long long k) {
  Chunk c;
  c.head = ((16 - ((uintptr_t)src & 15)) & 15) / (F32 ? 4 : 2);
  if (c.head > n) c.head = n;
  const long long units = (n - c.head) >> 3, per = kChunk >> 3;
  c.from = k * per;
  c.to = c.from + per < units ? c.from + per : units;
  c.tail = c.head + (units << 3);
  return c;
}

template <int MAX>
__device__ __forceinline__ int tensor_of(const Table<MAX>& t, int chunk) {
  int lo = 0, hi = t.n;             // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

template <bool F32>
__device__ __forceinline__ double squares(const void* src, long long n, long long k) {
  const Chunk c = chunk_of<F32>(src, n, k);
  const char* base = (const char*)src + c.head * (F32 ? 4 : 2);
  double a = 0.0;
  for (long long u = c.from + threadIdx.x; u < c.to; u += kThreads) {
    float f[8];
    load8<F32>(base + u * (F32 ? 32 : 16), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fma((double)f[e], (double)f[e], a);
  }
  if (k == 0) {
    const long long odd = c.head + (n - c.tail);
    if (threadIdx.x < odd) {
      const double f = load1<F32>(src, threadIdx.x < c.head ? threadIdx.x : c.tail + threadIdx.x - c.head);
      a = fma(f, f, a);
    }
  }
  return a;
}

// sum over the block, in thread 0
__device__ __forceinline__ double block_sum(double a) {
  __shared__ double sh[kThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    a = 0.0;
    for (int w = 0; w < kThreads / 32; ++w) a += sh[w];
  }
  return a;
}

template <int MAX>
__global__ void __launch_bounds__(kThreads)
square_sums_kernel(const __grid_constant__ Table<MAX> t, double* partial) {
  geeps_pdl_enter();
  double a = 0.0;
  for (int chunk = blockIdx.x; chunk < t.first[t.n]; chunk += gridDim.x) {
    const int i = tensor_of(t, chunk);
    const Entry& e = t.e[i];
    a += t.type[i] & 1 ? squares<true>(e.src, e.n, chunk - t.first[i]) : squares<false>(e.src, e.n, chunk - t.first[i]);
  }
  a = block_sum(a);
  if (threadIdx.x == 0) partial[blockIdx.x] = a;
}

template <bool F32, bool OUT32>
__device__ __forceinline__ void scale(const void* src, void* dst, long long n, long long k, float c) {
  const Chunk q = chunk_of<F32>(src, n, k);
  const char* base = (const char*)src + q.head * (F32 ? 4 : 2);
  char* to = (char*)dst + q.head * (OUT32 ? 4 : 2);
  const bool wide = ((uintptr_t)to & 15) == 0;
  for (long long u = q.from + threadIdx.x; u < q.to; u += kThreads) {
    float f[8];
    load8<F32>(base + u * (F32 ? 32 : 16), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= c;
    if (OUT32) {
      float* d = (float*)to + 8 * u;
      if (wide) { st_f4(d, make_float4(f[0], f[1], f[2], f[3])); st_f4(d + 4, make_float4(f[4], f[5], f[6], f[7])); }
      else for (int e = 0; e < 8; ++e) d[e] = f[e];
    } else {
      bf16* d = (bf16*)to + 8 * u;
      if (wide) *(uint4*)d = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
      else for (int e = 0; e < 8; ++e) d[e] = __float2bfloat16(f[e]);
    }
  }
  if (k == 0) {
    const long long odd = q.head + (n - q.tail);
    if (threadIdx.x < odd) {
      const long long i = threadIdx.x < q.head ? threadIdx.x : q.tail + threadIdx.x - q.head;
      const float f = load1<F32>(src, i) * c;
      if (OUT32) ((float*)dst)[i] = f; else ((bf16*)dst)[i] = __float2bfloat16(f);
    }
  }
}

// {norm, coefficient} of the blocks' sums, the same in every block
__device__ __forceinline__ float finish(const double* partial, int count, double max_norm, float* result) {
  __shared__ float coef;
  double a = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) a += partial[i];
  a = block_sum(a);
  if (threadIdx.x == 0) {
    const double norm = sqrt(a);
    const float c = norm > max_norm ? (float)(max_norm / norm) : 1.f;
    coef = c;
    if (result && blockIdx.x == 0) { result[0] = (float)norm; result[1] = c; }
  }
  __syncthreads();
  return coef;
}

template <int MAX>
__global__ void __launch_bounds__(kThreads)
clip_scale_kernel(const __grid_constant__ Table<MAX> t, const double* partial, int count, double max_norm, float* result,
                  int in_place) {
  geeps_pdl_enter();
  const float c = finish(partial, count, max_norm, result);
  if (in_place && c == 1.f) return;
  for (int chunk = t.first[t.n] - 1 - (int)blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    const int i = tensor_of(t, chunk);
    const Entry& e = t.e[i];
    const int k = chunk - t.first[i];
    switch (t.type[i] & 3) {
      case 0: scale<false, false>(e.src, e.dst, e.n, k, c); break;
      case 1: scale<true, false>(e.src, e.dst, e.n, k, c); break;
      case 2: scale<false, true>(e.src, e.dst, e.n, k, c); break;
      default: scale<true, true>(e.src, e.dst, e.n, k, c); break;
    }
  }
}

int most_blocks() { return geeps_sm_count() * 8; }
long long chunks_of(long long n) { return n <= 0 ? 0 : (n + kChunk - 1) / kChunk; }
long long pieces(long long n) { return (n + kTensors - 1) / kTensors; }

template <int MAX>
int clip(const GeepsTensors& src, const GeepsTensors* dst, double max_norm, float* result, double* work, cudaStream_t st) {
  const long long n = src.n;
  const int launches = n ? (int)((n + MAX - 1) / MAX) : 1;
  Table<MAX> t;
  int sums = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int l = 0; l < launches; ++l) {
      const long long from = (long long)l * MAX;
      t.n = (int)(n - from < MAX ? n - from : MAX);
      long long chunks = 0;
      for (int i = 0; i < t.n; ++i) {
        const long long j = from + i;
        t.e[i].src = src.ptr[j];
        t.e[i].dst = dst ? dst->ptr[j] : src.ptr[j];
        t.e[i].n = src.count[j];
        t.type[i] = (src.fp32[j] ? 1 : 0) | ((dst ? dst->fp32[j] : src.fp32[j]) ? 2 : 0);
        t.first[i] = (int)chunks;
        chunks += chunks_of(src.count[j]);
        if (chunks > 0x7fffffffLL - most_blocks()) return (int)cudaErrorInvalidValue;
      }
      t.first[t.n] = (int)chunks;
      const int blocks = chunks < 1 ? 1 : (int)(chunks < most_blocks() ? chunks : most_blocks());
      if (pass == 0) {
        geeps_launch(square_sums_kernel<MAX>, dim3(blocks), dim3(kThreads), 0, st, t, work + sums);
        sums += blocks;
      } else {
        geeps_launch(clip_scale_kernel<MAX>, dim3(blocks), dim3(kThreads), 0, st, t, (const double*)work, sums, max_norm,
                     l ? nullptr : result, dst ? 0 : 1);
      }
    }
  }
  return (int)cudaGetLastError();
}

// Is there a tensor of `a` that shares memory with one of `b` (a itself: with another of its own)?  Both are sorted by address
// and each without overlaps, so one merge finds it.  dst[i] may be src[i].
struct Range { uintptr_t from, to; };
Range range(const GeepsTensors& t, long long i) {
  const uintptr_t p = (uintptr_t)t.ptr[i];
  return {p, p + (uintptr_t)t.count[i] * (t.fp32[i] ? 4 : 2)};
}
bool overlaps_itself(const GeepsTensors& t) {
  uintptr_t end = 0;
  for (long long k = 0; k < t.n; ++k) {
    const Range r = range(t, t.order[k]);
    if (r.from == r.to) continue;
    if (r.from < end) return true;
    end = r.to;
  }
  return false;
}
bool overlaps(const GeepsTensors& a, const GeepsTensors& b) {
  long long i = 0, j = 0;
  while (i < a.n && j < b.n) {
    const long long x = a.order[i], y = b.order[j];
    const Range p = range(a, x), q = range(b, y);
    const bool same = x == y && p.from == q.from && a.fp32[x] == b.fp32[y];
    if (p.from < q.to && q.from < p.to && p.from != p.to && q.from != q.to && !same) return true;
    if (p.to < q.to) ++i; else ++j;
  }
  return false;
}

}  // namespace

extern "C" long long geeps_clip_work(const GeepsTensors* src) { return (pieces(src->n) + 1) * most_blocks(); }

extern "C" int geeps_clip_gradients(const GeepsTensors* src, const GeepsTensors* dst, double max_norm, float* result, double* work,
                                    void* stream) {
  if (!src || src->n < 0 || !result || !work || !(max_norm >= 0.0) || (dst && dst->n != src->n)) return (int)cudaErrorInvalidValue;
  for (long long i = 0; i < src->n; ++i) {
    if (src->count[i] < 0 || (dst && dst->count[i] != src->count[i])) return (int)cudaErrorInvalidValue;
    if (src->count[i] && (!src->ptr[i] || (dst && !dst->ptr[i]))) return (int)cudaErrorInvalidValue;
  }
  if (overlaps_itself(*src) || (dst && (overlaps_itself(*dst) || overlaps(*src, *dst)))) return GEEPS_ERR_CLIP_OVERLAP;
  cudaStream_t st = (cudaStream_t)stream;
  return src->n <= 64 ? clip<64>(*src, dst, max_norm, result, work, st) : clip<kTensors>(*src, dst, max_norm, result, work, st);
}
