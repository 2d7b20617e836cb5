// Clipping of gradients by their global norm: N = sqrt(sum g^2) over all tensors, g = c g with c = max / N where N > max.
//
// The reference's solver had this (clip_gradients of a solver definition) in its Caffe application, which is not part of
// the reference's tree.
//
// Two launches over the same ranges: the first adds the squares, in 64 bits (fp32 squares leave the range from 1.8e19 up and
// from 1e-19 down; the sum of all keeps no rounding that shows in an fp32 norm), the second adds the blocks' sums, in block
// order in every block, and scales.  The second goes through a block's range backwards and marks what it reads and writes as the
// first to leave L2, where the end of every range is then still found (268M bf16 315 us without the marks, 289 with).
// Up to kOneBlock values take one launch of one block, which keeps them in registers.  The tensors' table travels in the launch
// arguments, so a call keeps nothing on the device.
#include "common.cuh"
#include "nn_ops.h"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int kThreads = 256;
constexpr int kFlight = 4;                     // vectors of eight a thread has in flight
constexpr int kRow = 8 * kThreads;             // elements of a row: a vector for every thread
constexpr int kTensors = 1024;                 // tensors a launch
constexpr int kSquareBlocks = 5, kScaleBlocks = 3;      // blocks an SM: as many as are resident, each with its range
constexpr int kBlocks = 1024;                  // blocks a launch, at the most
constexpr int kOneThreads = 1024, kOneVectors = 4, kOneBlock = 8 * kOneThreads * kOneVectors, kOneTensors = 64;

struct Entry { const void* src; void* dst; long long n; };
template <int MAX>
struct Table {
  Entry e[MAX];
  int first[MAX + 1];              // rows before tensor i
  unsigned short start[kBlocks];   // the tensor that block b starts in (a search in here was a tenth of a short call)
  unsigned char type[MAX];         // bit 0: src is fp32, bit 1: dst is fp32
  int n;
};
// rows of a tensor; the vectors start at its first boundary of their size, what lies before it and behind the last goes with row 0
__host__ __device__ inline long long rows_of(long long n) { return (n + kRow - 1) / kRow; }

__device__ __forceinline__ uint64_t leaves_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
// Eight values from and to a boundary of their size: whole 32-byte sectors of fp32
template <bool F32, bool LAST>
__device__ __forceinline__ void load8(const void* p, uint64_t policy, uint32_t (&w)[8]) {
  if (F32) {
    if (LAST)
      asm volatile("ld.global.L1::no_allocate.L2::evict_first.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
    else
      asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
  } else if (LAST) {
    asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.b32 {%0,%1,%2,%3}, [%4], %5;"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p), "l"(policy) : "memory");
  } else {
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p) : "memory");
  }
}
template <bool F32>
__device__ __forceinline__ void unpack8(const uint32_t (&w)[8], float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(F32 ? w[e] : e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
}
// c * f, to an address that may be any (`wide`: such a boundary)
template <bool OUT32>
__device__ __forceinline__ void store8(void* p, bool wide, const float (&g)[8], float c, uint64_t policy) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = g[e] * c;
  if (OUT32) {
    if (wide) {
      asm volatile("st.global.L2::evict_first.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]),
                   "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]) : "memory");
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) ((float*)p)[e] = f[e];
    }
  } else if (wide) {
    asm volatile("st.global.L2::cache_hint.v4.b32 [%0], {%1,%2,%3,%4}, %5;" ::"l"(p), "r"(pack_bf16x2(f[0], f[1])), "r"(pack_bf16x2(f[2], f[3])),
                 "r"(pack_bf16x2(f[4], f[5])), "r"(pack_bf16x2(f[6], f[7])), "l"(policy) : "memory");
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) ((bf16*)p)[e] = __float2bfloat16(f[e]);
  }
}
template <bool OUT32>
__device__ __forceinline__ bool at_boundary(const void* p) { return ((uintptr_t)p & (OUT32 ? 31 : 15)) == 0; }
__device__ __forceinline__ float load1(const void* p, bool f32, long long i) { return f32 ? ((const float*)p)[i] : (float)((const bf16*)p)[i]; }
__device__ __forceinline__ void store1(void* p, bool f32, long long i, float f) {
  if (f32) ((float*)p)[i] = f; else ((bf16*)p)[i] = __float2bfloat16(f);
}
__device__ __forceinline__ double add_squares(const float (&f)[8], double a) {
  double b = 0.0;
#pragma unroll
  for (int e = 0; e < 8; e += 2) { a = fma((double)f[e], (double)f[e], a); b = fma((double)f[e + 1], (double)f[e + 1], b); }
  return a + b;
}

// Where the vectors of a tensor start, how many there are and which single elements lie outside: thread i < odd has at(i).
struct Parts {
  long long head, units, tail;
  int odd;
  __device__ __forceinline__ Parts(const void* src, long long n, bool f32) {
    const int line = f32 ? 32 : 16;
    head = (long long)((line - ((uintptr_t)src & (line - 1))) & (line - 1)) >> (f32 ? 2 : 1);
    if (head > n) head = n;
    units = (n - head) >> 3;
    tail = head + (units << 3);
    odd = (int)(head + n - tail);
  }
  __device__ __forceinline__ long long at(int i) const { return i < head ? i : tail + i - head; }
};

// rows [share(b), share(b + 1)) are block b's
__host__ __device__ __forceinline__ int share(int rows, int blocks, int b) { return (int)((long long)rows * b / blocks); }

// squares of rows [from, to) of a tensor
template <bool F32>
__device__ __forceinline__ double squares(const void* src, long long n, int from, int to, double a) {
  const Parts q(src, n, F32);
  const char* base = (const char*)src + q.head * (F32 ? 4 : 2);
  const long long end = (long long)to * kThreads < q.units ? (long long)to * kThreads : q.units;
  long long u = (long long)from * kThreads + threadIdx.x;
  for (; u - threadIdx.x + kFlight * kThreads <= end; u += kFlight * kThreads) {
    uint32_t v[kFlight][8];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) load8<F32, false>(base + (u + i * kThreads) * (F32 ? 32 : 16), 0, v[i]);
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      float f[8];
      unpack8<F32>(v[i], f);
      a = add_squares(f, a);
    }
  }
  for (; u < end; u += kThreads) {
    float f[8];
    uint32_t v[8];
    load8<F32, false>(base + u * (F32 ? 32 : 16), 0, v);
    unpack8<F32>(v, f);
    a = add_squares(f, a);
  }
  if (from == 0 && threadIdx.x < q.odd) {
    const double f = load1(src, F32, q.at(threadIdx.x));
    a = fma(f, f, a);
  }
  return a;
}
// ... and c times them, from the last row to the first
template <bool F32, bool OUT32>
__device__ __forceinline__ void scale(const void* src, void* dst, long long n, int from, int to, float c, uint64_t policy) {
  const Parts q(src, n, F32);
  const char* base = (const char*)src + q.head * (F32 ? 4 : 2);
  char* out = (char*)dst + q.head * (OUT32 ? 4 : 2);
  const bool wide = at_boundary<OUT32>(out);
  const long long first = (long long)from * kThreads, end = (long long)to * kThreads < q.units ? (long long)to * kThreads : q.units;
  long long u = end - 1 - threadIdx.x;
  for (; u + threadIdx.x + 1 - kFlight * kThreads >= first; u -= kFlight * kThreads) {
    uint32_t v[kFlight][8];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) load8<F32, true>(base + (u - i * kThreads) * (F32 ? 32 : 16), policy, v[i]);
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      float f[8];
      unpack8<F32>(v[i], f);
      store8<OUT32>(out + (u - i * kThreads) * (OUT32 ? 32 : 16), wide, f, c, policy);
    }
  }
  for (; u >= first; u -= kThreads) {
    float f[8];
    uint32_t v[8];
    load8<F32, true>(base + u * (F32 ? 32 : 16), policy, v);
    unpack8<F32>(v, f);
    store8<OUT32>(out + u * (OUT32 ? 32 : 16), wide, f, c, policy);
  }
  if (from == 0 && threadIdx.x < q.odd) store1(dst, OUT32, q.at(threadIdx.x), load1(src, F32, q.at(threadIdx.x)) * c);
}

// sum over the block, in thread 0
template <int THREADS>
__device__ __forceinline__ double block_sum(double a) {
  __shared__ double sh[THREADS / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    a = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) a += sh[w];
  }
  return a;
}
// the coefficient of a sum that thread 0 has, in every thread; block 0 writes the result
__device__ __forceinline__ float finish(double a, double max_norm, float* result) {
  __shared__ float coef;
  if (threadIdx.x == 0) {
    const double norm = sqrt(a);
    coef = norm > max_norm ? (float)(max_norm / norm) : 1.f;
    if (result && blockIdx.x == 0) { result[0] = (float)norm; result[1] = coef; }
  }
  __syncthreads();
  return coef;
}

template <int MAX>
__global__ void __launch_bounds__(kThreads, kSquareBlocks)
square_sums_kernel(const __grid_constant__ Table<MAX> t, double* partial) {
  geeps_pdl_enter();
  const int end = share(t.first[t.n], gridDim.x, blockIdx.x + 1);
  int row = share(t.first[t.n], gridDim.x, blockIdx.x);
  double a = 0.0;
  for (int i = t.start[blockIdx.x]; row < end; ++i) {
    const int to = t.first[i + 1] < end ? t.first[i + 1] : end, base = t.first[i];
    if (to <= row) continue;
    a = t.type[i] & 1 ? squares<true>(t.e[i].src, t.e[i].n, row - base, to - base, a) : squares<false>(t.e[i].src, t.e[i].n, row - base, to - base, a);
    row = to;
  }
  a = block_sum<kThreads>(a);
  if (threadIdx.x == 0) partial[blockIdx.x] = a;
}

template <int MAX>
__global__ void __launch_bounds__(kThreads, kScaleBlocks)
clip_scale_kernel(const __grid_constant__ Table<MAX> t, const double* partial, int count, double max_norm, float* result,
                  int in_place) {
  geeps_pdl_enter();
  double a = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) a += partial[i];
  const float c = finish(block_sum<kThreads>(a), max_norm, result);
  if (in_place && c == 1.f) return;
  const uint64_t policy = leaves_first();
  const int begin = share(t.first[t.n], gridDim.x, blockIdx.x);
  int row = share(t.first[t.n], gridDim.x, blockIdx.x + 1);
  for (int i = t.start[blockIdx.x]; row > begin; --i) {
    const int base = t.first[i], from = base > begin ? base : begin;
    if (from >= row) continue;
    const Entry& e = t.e[i];
    switch (t.type[i] & 3) {
      case 0: scale<false, false>(e.src, e.dst, e.n, from - base, row - base, c, policy); break;
      case 1: scale<true, false>(e.src, e.dst, e.n, from - base, row - base, c, policy); break;
      case 2: scale<false, true>(e.src, e.dst, e.n, from - base, row - base, c, policy); break;
      default: scale<true, true>(e.src, e.dst, e.n, from - base, row - base, c, policy); break;
    }
    row = from;
  }
}

// One block for everything: a warp takes vector after vector of the tensors in turn and keeps what it took.
__global__ void __launch_bounds__(kOneThreads)
clip_one_block_kernel(const __grid_constant__ Table<kOneTensors> t, double max_norm, float* result, int in_place) {
  geeps_pdl_enter();
  double a = 0.0;
  float f[kOneVectors][8], odd = 0.f;
  int tensor[kOneVectors], odd_tensor = -1, at = threadIdx.x;     // `at`: a vector's number among those of all tensors
  long long unit[kOneVectors], odd_at = 0;
  // vectors of tensor i are numbered from before[i]; the search over a few tensors is a walk
  __shared__ int before[kOneTensors + 1], odd_before[kOneTensors + 1];
  if (threadIdx.x == 0) {
    int v = 0, o = 0;
    for (int i = 0; i < t.n; ++i) {
      const Parts q(t.e[i].src, t.e[i].n, t.type[i] & 1);
      before[i] = v; odd_before[i] = o;
      v += (int)q.units; o += q.odd;
    }
    before[t.n] = v; odd_before[t.n] = o;
  }
  __syncthreads();
  auto find = [&](const int* b, int x) {
    int i = 0;
    while (x >= b[i + 1]) ++i;
    return i;
  };
#pragma unroll
  for (int k = 0; k < kOneVectors; ++k, at += kOneThreads) {
    tensor[k] = -1;
    if (at >= before[t.n]) continue;
    const int i = tensor[k] = find(before, at);
    const bool f32 = t.type[i] & 1;
    const Parts q(t.e[i].src, t.e[i].n, f32);
    unit[k] = at - before[i];
    const char* p = (const char*)t.e[i].src + (q.head + 8 * unit[k]) * (f32 ? 4 : 2);
    uint32_t v[8];
    if (f32) { load8<true, false>(p, 0, v); unpack8<true>(v, f[k]); } else { load8<false, false>(p, 0, v); unpack8<false>(v, f[k]); }
  }
#pragma unroll
  for (int k = 0; k < kOneVectors; ++k) if (tensor[k] >= 0) a = add_squares(f[k], a);
  if (threadIdx.x < odd_before[t.n]) {                           // at most 14 a tensor
    const int i = odd_tensor = find(odd_before, threadIdx.x);
    odd_at = Parts(t.e[i].src, t.e[i].n, t.type[i] & 1).at(threadIdx.x - odd_before[i]);
    odd = load1(t.e[i].src, t.type[i] & 1, odd_at);
    a = fma((double)odd, (double)odd, a);
  }
  const float c = finish(block_sum<kOneThreads>(a), max_norm, result);
  if (in_place && c == 1.f) return;
#pragma unroll
  for (int k = 0; k < kOneVectors; ++k) {
    if (tensor[k] < 0) continue;
    const int i = tensor[k];
    const bool out32 = t.type[i] & 2;
    const Parts q(t.e[i].src, t.e[i].n, t.type[i] & 1);
    char* p = (char*)t.e[i].dst + (q.head + 8 * unit[k]) * (out32 ? 4 : 2);
    const uint64_t policy = leaves_first();
    if (out32) store8<true>(p, at_boundary<true>(p), f[k], c, policy); else store8<false>(p, at_boundary<false>(p), f[k], c, policy);
  }
  if (odd_tensor >= 0) store1(t.e[odd_tensor].dst, t.type[odd_tensor] & 2, odd_at, odd * c);
}

int blocks_of(int rows, int per_sm) {
  const int sms = geeps_sm_count() * per_sm, most = sms < kBlocks ? sms : kBlocks;
  return rows < 1 ? 1 : rows < most ? rows : most;
}
long long pieces(long long n) { return (n + kTensors - 1) / kTensors; }

// the table of tensors [from, from + MAX) of a call; false: too many rows for one
template <int MAX>
bool fill(Table<MAX>& t, const GeepsTensors& src, const GeepsTensors* dst, long long from) {
  const long long n = src.n - from < MAX ? src.n - from : MAX;
  long long rows = 0;
  t.n = (int)n;
  for (int i = 0; i < t.n; ++i) {
    const long long j = from + i;
    t.e[i].src = src.ptr[j];
    t.e[i].dst = dst ? dst->ptr[j] : src.ptr[j];
    t.e[i].n = src.count[j];
    t.type[i] = (src.fp32[j] ? 1 : 0) | ((dst ? dst->fp32[j] : src.fp32[j]) ? 2 : 0);
    t.first[i] = (int)rows;
    rows += rows_of(src.count[j]);
    if (rows > 0x7fffffffLL) return false;
  }
  t.first[t.n] = (int)rows;
  return true;
}

// the tensors that the blocks start in: with the first row of their share, or going backwards the last
template <int MAX>
void starts(Table<MAX>& t, int blocks, bool backwards) {
  const int rows = t.first[t.n];
  for (int b = 0, i = 0; b < blocks; ++b) {
    const int row = backwards ? share(rows, blocks, b + 1) - 1 : share(rows, blocks, b);
    while (i + 1 < t.n && t.first[i + 1] <= row) ++i;
    t.start[b] = (unsigned short)i;
  }
}

template <int MAX>
int clip(const GeepsTensors& src, const GeepsTensors* dst, double max_norm, float* result, double* work, cudaStream_t st) {
  const int launches = src.n ? (int)((src.n + MAX - 1) / MAX) : 1;
  Table<MAX> t;
  int sums = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int l = 0; l < launches; ++l) {
      if ((launches > 1 || pass == 0) && !fill(t, src, dst, (long long)l * MAX)) return (int)cudaErrorInvalidValue;
      const int blocks = blocks_of(t.first[t.n], pass == 0 ? kSquareBlocks : kScaleBlocks);
      starts(t, blocks, pass == 1);
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

extern "C" long long geeps_clip_work(const GeepsTensors* src) { return (pieces(src->n) + 1) * geeps_sm_count() * kSquareBlocks; }

extern "C" int geeps_clip_gradients(const GeepsTensors* src, const GeepsTensors* dst, double max_norm, float* result, double* work,
                                    void* stream) {
  if (!src || src->n < 0 || !result || !work || !(max_norm >= 0.0) || (dst && dst->n != src->n)) return (int)cudaErrorInvalidValue;
  for (long long i = 0; i < src->n; ++i) {
    if (src->count[i] < 0 || (dst && dst->count[i] != src->count[i])) return (int)cudaErrorInvalidValue;
    if (src->count[i] && (!src->ptr[i] || (dst && !dst->ptr[i]))) return (int)cudaErrorInvalidValue;
  }
  bool between = ((uintptr_t)result & 3) || ((uintptr_t)work & 7);
  for (long long i = 0; i < src->n; ++i)
    if (src->count[i]) between |= ((uintptr_t)src->ptr[i] & (src->fp32[i] ? 3 : 1)) || (dst && ((uintptr_t)dst->ptr[i] & (dst->fp32[i] ? 3 : 1)));
  if (between) return GEEPS_ERR_CLIP_ALIGN;
  if (overlaps_itself(*src) || (dst && (overlaps_itself(*dst) || overlaps(*src, *dst)))) return GEEPS_ERR_CLIP_OVERLAP;
  const uintptr_t r = (uintptr_t)result, w = (uintptr_t)work, we = w + geeps_clip_work(src) * sizeof(double);
  auto meets = [&](const Range& q) { return q.from != q.to && ((q.from < r + 8 && r < q.to) || (q.from < we && w < q.to)); };
  for (long long i = 0; i < src->n; ++i) if (meets(range(*src, i)) || (dst && meets(range(*dst, i)))) return GEEPS_ERR_CLIP_OVERLAP;
  if (r < we && w < r + 8) return GEEPS_ERR_CLIP_OVERLAP;
  cudaStream_t st = (cudaStream_t)stream;
  long long total = 0;
  for (long long i = 0; i < src->n && total <= kOneBlock; ++i) total += src->count[i];
  if (src->n <= kOneTensors && total <= kOneBlock) {
    Table<kOneTensors> t;
    fill(t, *src, dst, 0);
    geeps_launch(clip_one_block_kernel, dim3(1), dim3(kOneThreads), 0, st, t, max_norm, result, dst ? 0 : 1);
    return (int)cudaGetLastError();
  }
  return src->n <= 64 ? clip<64>(*src, dst, max_norm, result, work, st) : src->n <= 256 ? clip<256>(*src, dst, max_norm, result, work, st)
                      : clip<kTensors>(*src, dst, max_norm, result, work, st);
}
