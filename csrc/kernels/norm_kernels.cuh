// The kernels of norm.cu, which has the mathematics and the checks: one translation unit for each pair of types.
#pragma once
#include "common.cuh"
#include "nn_ops.h"

typedef __nv_bfloat16 bf16;

namespace rownorm {

constexpr int kMaxChannels = 16384;
constexpr int kVec = 8;                 // channels a vector
constexpr int kRingBytes = 200 * 1024;  // shared memory of an SM for rows on their way
enum { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };
enum { MODE_NORM = 1, MODE_JOIN = 2, MODE_BOTH = 3 };     // the next norm alone, a join alone, a join and the norm behind it

// ---- launch shape ----
struct Shape {
  int vectors;       // vectors a thread
  int slot;          // threads a row: a power of two up to 32, or whole warps
  int slots;         // rows a block works on at a time
  int blocks, per_sm;
  int threads() const { return slot * slots; }
};
// K vectors a thread: as few as the threads of a block allow, since what a thread keeps for its columns is in registers.  A
// block of the backward pass has up to 384 (rows of up to 384 vectors, but of more than 16) or 512 threads and an SM to itself,
// so that few blocks leave column sums behind; forward several blocks of 256 share an SM.
inline Shape plan(long long rows, int C, bool backward, int mode) {
  Shape s;
  const int vec = (C + kVec - 1) / kVec;
  const int narrow = vec <= 16, one = backward ? 384 : 256;
  s.vectors = vec <= one ? 1 : vec <= 1024 ? 2 : 4;
  const int need = (vec + s.vectors - 1) / s.vectors, most = s.vectors > 1 ? 512 : backward ? narrow ? 512 : 384 : 256;
  s.slot = 1;
  if (need <= 32) while (s.slot < need) s.slot <<= 1;
  else s.slot = (need + 31) / 32 * 32;
  s.slots = s.slot > most / 2 ? 1 : most / s.slot;
  s.per_sm = backward || s.vectors > 1 ? 1 : mode == MODE_NORM ? 3 : 2;
  const long long room = (long long)geeps_sm_count() * s.per_sm, want = (rows + s.slots - 1) / s.slots;
  s.blocks = (int)(want < room ? want : room);
  return s;
}
// rows [first_row(i), first_row(i + 1)) are slot i's, of all slots of all blocks; rows are less than 2^31
__host__ __device__ inline int first_row(int rows, int slots, int i) {
  return rows / slots * i + (rows % slots < i ? rows % slots : i);
}
// An operand as a thread sees it: where its first column of row 0 is (without VEC: where row 0 is), and bytes to the next row.
template <typename T>
struct Rows {
  char* first;
  int pitch;
  __device__ __forceinline__ Rows(const void* base, long long ld, int column) : first((char*)((T*)base + column)), pitch((int)ld * (int)sizeof(T)) {}
  __device__ __forceinline__ T* at(int row) const { return (T*)(first + (long long)row * pitch); }
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until at most depth - 1 of this thread's groups are under way
__device__ __forceinline__ void copy_wait(int depth) {
  if (depth == 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (depth == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (depth == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---- pairs of fp32 ----
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(r))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(r))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(r))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ uint4 ld_shared16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ float ld_shared1(uint32_t a) {
  if (sizeof(T) == 2) {
    unsigned short h;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(a) : "memory");
    return __uint_as_float((uint32_t)h << 16);
  }
  float f;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
  return f;
}

// ---- a thread's columns ----
// Eight a vector, held as pairs.  VEC: vectors t, t + slot, ...: 16- or 32-byte accesses.  Otherwise (odd widths, pitches or
// addresses) single columns t, t + slot, ...: neighbouring threads on neighbouring columns.  A thread without a column at some
// place has zeros there.
// Rows come through a ring of `depth` stages in shared memory, so that what is on its way takes no registers.  With VEC a thread
// copies what it reads itself and nobody waits for anybody; otherwise the slot copies the 16-byte pieces that hold the row (up
// to 15 bytes before and behind it in the same pieces come along) and meets before and after reading them.  The ring starts as
// zeros, so what has no column or no operand is read from it like the rest.  Rows of more than two vectors a thread do not
// fit and are read where they lie.
// THREADS: as many as a block may have; a thread's places in the ring are then the same for every launch.
template <int K, bool VEC, int THREADS>
struct Columns {
  static constexpr int N = 4 * K;      // pairs
  static constexpr bool RING = K <= 2;
  int t, slot, C, slots;
  __device__ __forceinline__ int first() const { return VEC ? at(0) : 0; }
  __device__ __forceinline__ static constexpr int threads() { return THREADS; }
  __device__ __forceinline__ int at(int j) const { return VEC ? (t + (j >> 3) * slot) * 8 + (j & 7) : t + j * slot; }
  __device__ __forceinline__ bool on(int j) const { return at(VEC ? j & ~7 : j) < C; }

  // bytes of a row of a slot without VEC, and of a stage for one stream of T
  template <typename T>
  __device__ __forceinline__ int pieces() const { return ((C * (int)sizeof(T) + 15) / 16 + 1) * 16; }
  template <typename T>
  __device__ __forceinline__ int stage() const { return VEC ? K * 8 * (int)sizeof(T) * THREADS : pieces<T>() * slots; }
  // `from` is what Rows::at() gives; `to` has the thread's 16 * threadIdx.x with VEC, the slot's share without
  template <typename T>
  __device__ __forceinline__ void copy(const T* from, uint32_t to) const {
    if (VEC) {
      constexpr int Q = 8 * sizeof(T) / 16;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (K > 1 && !on(8 * k)) continue;         // K = 1: the caller has asked
#pragma unroll
        for (int q = 0; q < Q; ++q) copy16(to + (k * Q + q) * THREADS * 16, from + k * slot * 8 + q * (8 / Q));
      }
    } else {
      const uintptr_t start = (uintptr_t)from & ~(uintptr_t)15, end = (uintptr_t)(from + C);
      const uint32_t mine = to + (threadIdx.x / slot) * pieces<T>();
      for (uintptr_t a = start + 16 * t; a < end; a += 16 * slot) copy16(mine + (uint32_t)(a - start), (const void*)a);
    }
  }
  template <typename T>
  __device__ __forceinline__ static void unpack(const uint4& v, float2* o) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) o[e] = make_float2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
    }
  }
  // a row from where it lies
  template <typename T>
  __device__ __forceinline__ void fetch(const T* row, bool there, float2 (&f)[N]) const {
    constexpr int Q = 8 * sizeof(T) / 16;
    if (VEC) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int q = 0; q < Q; ++q)
          unpack<T>(there && on(8 * k) ? *reinterpret_cast<const uint4*>(row + k * slot * 8 + q * (8 / Q)) : make_uint4(0u, 0u, 0u, 0u),
                    f + 4 * k + q * (4 / Q));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        f[i] = make_float2(there && on(2 * i) ? (float)row[at(2 * i)] : 0.f, there && on(2 * i + 1) ? (float)row[at(2 * i + 1)] : 0.f);
    }
  }
  // zeros in the place of a row that the slot does not have
  template <typename T>
  __device__ __forceinline__ void no_row(uint32_t to) const {
    if (!VEC) return;
#pragma unroll
    for (int q = 0; q < K * 8 * (int)sizeof(T) / 16; ++q)
      asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(to + q * THREADS * 16), "r"(0) : "memory");
  }
  // a row from the ring if there is one; zeros where the slot has no such row
  template <typename T>
  __device__ __forceinline__ void load(const Rows<T>& rows, int row, bool active, bool there, uint32_t from, float2 (&f)[N]) const {
    if (!RING) {
      fetch(rows.at(row), active && there, f);
    } else if (VEC) {
      constexpr int Q = 8 * sizeof(T) / 16;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int q = 0; q < Q; ++q)
          unpack<T>(ld_shared16(from + (k * Q + q) * THREADS * 16), f + 4 * k + q * (4 / Q));
    } else {
      const uint32_t r = from + (threadIdx.x / slot) * pieces<T>() + (uint32_t)((uintptr_t)rows.at(row) & 15);
      const bool any = active && there;
#pragma unroll
      for (int i = 0; i < N; ++i)
        f[i] = make_float2(any && on(2 * i) ? ld_shared1<T>(r + at(2 * i) * (int)sizeof(T)) : 0.f,
                           any && on(2 * i + 1) ? ld_shared1<T>(r + at(2 * i + 1) * (int)sizeof(T)) : 0.f);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, bool active, const float2 (&f)[N]) const {
    if (!active) return;
    if (VEC) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!on(8 * k)) continue;
        const int c = k * slot * 8;
        const float2* v = f + 4 * k;
        if (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(row + c) = make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y),
                                                          pack_bf16x2(v[2].x, v[2].y), pack_bf16x2(v[3].x, v[3].y));
        } else {
          float* r = reinterpret_cast<float*>(row) + c;
          st_f4(r, make_float4(v[0].x, v[0].y, v[1].x, v[1].y));
          st_f4(r + 4, make_float4(v[2].x, v[2].y, v[3].x, v[3].y));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2 * N; ++j) if (on(j)) row[at(j)] = (T)(j & 1 ? f[j >> 1].y : f[j >> 1].x);
    }
  }
  // a parameter of every column; `other` where there is none
  __device__ __forceinline__ void param(const float* p, float other, float2 (&f)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      f[i] = make_float2(!on(2 * i) ? 0.f : p ? p[at(2 * i)] : other, !on(2 * i + 1) ? 0.f : p ? p[at(2 * i + 1)] : other);
  }
  // f - mean, zero where there is no column
  __device__ __forceinline__ void subtract(float2 (&f)[N], float mean) const {
    if (VEC) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float2 m = both(on(8 * k) ? -mean : 0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[4 * k + e] = add2(f[4 * k + e], m);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float2 v = add2(f[i], both(-mean));
        f[i] = make_float2(on(2 * i) ? v.x : 0.f, on(2 * i + 1) ? v.y : 0.f);
      }
    }
  }
};

struct Slot {
  int id, t, size;
  float* red;        // 128 floats of shared memory: two turns of 64, zero where no warp writes
  int turn;
  __device__ __forceinline__ void sync() const {
    if (size > 32) asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(size) : "memory");
    else __syncwarp();
  }
};

// Sums of M values (1, 2 or 4) over the threads of a slot, the same in each.  In a warp each step halves the values a lane
// goes on with, until it is one: four sums take six shuffles.  Warps meet in shared memory at the slot's named barrier; the two
// turns of `red` alternate, so the next sums may be written while these are still being read.
template <bool WIDE, int M>
__device__ __forceinline__ void slot_sum(float (&v)[M], Slot& s) {
  if (!WIDE) {
    for (int o = s.size >> 1; o; o >>= 1) {
#pragma unroll
      for (int i = 0; i < M; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    return;
  }
  float one;
  if (M == 4) {
    const bool a = threadIdx.x & 16, b = threadIdx.x & 8;
    float x = a ? v[2 % M] : v[0], y = a ? v[3 % M] : v[1 % M];
    x += __shfl_xor_sync(0xffffffffu, a ? v[0] : v[2 % M], 16);
    y += __shfl_xor_sync(0xffffffffu, a ? v[1 % M] : v[3 % M], 16);
    one = b ? y : x;
    one += __shfl_xor_sync(0xffffffffu, b ? x : y, 8);
  } else if (M == 2) {
    const bool a = threadIdx.x & 16;
    one = a ? v[1 % M] : v[0];
    one += __shfl_xor_sync(0xffffffffu, a ? v[0] : v[1 % M], 16);
    one += __shfl_xor_sync(0xffffffffu, one, 8);
  } else {
    one = v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
    one += __shfl_xor_sync(0xffffffffu, one, 8);
  }
#pragma unroll
  for (int o = 4; o; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
  float* r = s.red + s.turn;
  s.turn ^= 64;
  constexpr int L = 32 / M;           // lanes that hold the same sum
  if (s.t % L == 0) r[s.t / L] = one;
  s.sync();
  // four values at a time, values of more warps than four (M = 4), eight or sixteen in a loop
  constexpr int Q = M == 4 ? 4 : M == 2 ? 2 : 1;
#pragma unroll
  for (int i = 0; i < M; ++i) v[i] = 0.f;
  auto add = [&](int w) {
    const float4 q = ld_f4(r + 4 * w);
    if (M == 4) { v[0] += q.x; v[1 % M] += q.y; v[2 % M] += q.z; v[3 % M] += q.w; }
    else if (M == 2) { v[0] += q.x + q.z; v[1 % M] += q.y + q.w; }
    else v[0] += (q.x + q.y) + (q.z + q.w);
  };
#pragma unroll
  for (int w = 0; w < Q; ++w) add(w);
  for (int w = 4; w < s.size >> 5; w += 4) {
#pragma unroll
    for (int u = 0; u < Q; ++u) add(w * Q / 4 + u);
  }
}
template <int N>
__device__ __forceinline__ float total(const float2 (&f)[N]) {
  float2 v = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) v = add2(v, f[i]);
  return v.x + v.y;
}
template <int N>
__device__ __forceinline__ float dot(const float2 (&f)[N], const float2 (&g)[N]) {
  float2 v = mul2(f[0], g[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) v = fma2(f[i], g[i], v);
  return v.x + v.y;
}

// n = (f - mean) * rstd of R rows in place; mean and rstd go to stats
template <bool WIDE, int R, int K, bool VEC, int THREADS>
__device__ __forceinline__ void normalise(const Columns<K, VEC, THREADS>& cols, Slot& s, const GeepsNorm& norm, int row, int end,
                                          float inv_c, float2 (&f)[R][4 * K]) {
  float mean[R], v[R];
#pragma unroll
  for (int r = 0; r < R; ++r) mean[r] = 0.f;
  if (norm.kind == NORM_LAYER) {
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] = total(f[r]);
    slot_sum<WIDE>(mean, s);
#pragma unroll
    for (int r = 0; r < R; ++r) { mean[r] *= inv_c; cols.subtract(f[r], mean[r]); }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = dot(f[r], f[r]);
  slot_sum<WIDE>(v, s);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float rstd = 1.f / sqrtf(fmaf(v[r], inv_c, norm.eps));
#pragma unroll
    for (int i = 0; i < 4 * K; ++i) f[r][i] = mul2(f[r][i], both(rstd));
    if (norm.stats && row + r < end && s.t == 0) *reinterpret_cast<float2*>(norm.stats + 2LL * (row + r)) = make_float2(mean[r], rstd);
  }
}

// n = (f - mean) * rstd with the statistics at hand.  Not zero where there is no column, but whatever it meets there is.
template <int N>
__device__ __forceinline__ void normalised(float2 (&f)[N], float2 st) {
  const float2 r = both(st.y), m = both(-st.x * st.y);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = fma2(f[i], r, m);
}

// Gradients of R rows n * w + b by their inputs, for a = dz * w: rstd * (a - mean a - n mean(a n)), added to `to`
template <bool WIDE, int R, int N>
__device__ __forceinline__ void norm_gradient(Slot& s, int kind, const float2 (&st)[R], float inv_c, const float2 (&n)[R][N],
                                              const float2 (&a)[R][N], float2 (&to)[R][N]) {
  float v[2 * R];
#pragma unroll
  for (int r = 0; r < R; ++r) { v[2 * r] = total(a[r]); v[2 * r + 1] = dot(a[r], n[r]); }
  slot_sum<WIDE>(v, s);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float scale = -inv_c * st[r].y;
    const float2 m0 = both(kind == NORM_LAYER ? v[2 * r] * scale : 0.f), m1 = both(v[2 * r + 1] * scale), rs = both(st[r].y);
#pragma unroll
    for (int i = 0; i < N; ++i) to[r][i] = fma2(n[r][i], m1, fma2(a[r][i], rs, add2(to[r][i], m0)));
  }
}

__device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + expf(-g)); }
template <int N>
__device__ __forceinline__ void gate_factor(int through_sigmoid, float2 (&g)[N]) {
  if (!through_sigmoid) return;
#pragma unroll
  for (int i = 0; i < N; ++i) g[i] = make_float2(sigmoid(g[i].x), sigmoid(g[i].y));
}
__device__ __forceinline__ float2 gate_slope(int through_sigmoid, float2 g) {       // of the factor g by the gate
  return through_sigmoid ? make_float2(g.x * (1.f - g.x), g.y * (1.f - g.y)) : both(1.f);
}

// zeros to the ring, before any copy
__device__ __forceinline__ void clear_ring(unsigned char* ring, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<uint4*>(ring + i) = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
}

// The rows of a slot, R a turn.  Slots that share a warp take the same number of turns, since its lanes meet in sums: some have
// no row in the last.
struct Walk {
  int lo, hi, step, turns;
  __device__ __forceinline__ Walk(const GeepsResidual& p, int slots, int id, bool wide, int R, bool ranges) {
    const int rows = (int)p.rows, all = gridDim.x * slots, me = blockIdx.x * slots + id;
    lo = ranges ? first_row(rows, all, me) : me * R;
    hi = ranges ? first_row(rows, all, me + 1) : rows;
    step = ranges ? R : all * R;
    const int most = ranges ? (rows + all - 1) / all : (rows + step - 1) / step;
    turns = !wide ? most : lo < hi ? (hi - lo + step - 1) / step : 0;
  }
};

// What kernels of K vectors a thread are like.  Two rows a turn where a turn's overhead counts most and registers allow: bf16
// rows of up to 384 vectors; blocks have 384 threads then backward (168 registers a thread).
template <typename TB, int K, bool VEC, bool WIDE>
struct Form {
  static constexpr int R = WIDE && K == 1 && VEC && sizeof(TB) == 2 ? 2 : 1;
  static constexpr int forward_threads = K == 1 ? 256 : 512;
  static constexpr int backward_threads = K == 1 && WIDE ? 384 : 512;
};

// WIDE: a slot is whole warps.  PIXEL: a gate for every row.
template <typename TR, typename TB, int K, bool VEC, bool WIDE, int MODE, bool PIXEL>
__global__ void __launch_bounds__(Form<TB, K, VEC, WIDE>::forward_threads, K == 1 ? MODE == MODE_NORM ? 3 : 2 : 1)
residual_forward_kernel(const __grid_constant__ GeepsResidual p, int slot, int slots, int depth) {
  geeps_pdl_enter();
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ __align__(16) float red[16][128];
  constexpr int N = 4 * K, R = Form<TB, K, VEC, WIDE>::R;
  for (int i = threadIdx.x; i < 16 * 128; i += blockDim.x) red[0][i] = 0.f;
  __syncthreads();
  Slot s;
  s.id = threadIdx.x / slot; s.t = threadIdx.x % slot; s.size = slot; s.red = red[WIDE ? s.id : 0]; s.turn = 0;
  const Columns<K, VEC, Form<TB, K, VEC, WIDE>::forward_threads> cols = {s.t, slot, p.C, slots};
  const float inv_c = 1.f / (float)p.C;
  const bool by_image = (MODE & MODE_JOIN) && !PIXEL && p.gate;
  float2 sw[N], sb[N], w2[N], b2[N];           // scale * weight and scale * bias, times the gate where an image has one
  auto join_params = [&]() {
    float2 sc[N];
    cols.param(p.scale, 1.f, sc); cols.param(p.post.weight, 1.f, sw); cols.param(p.post.bias, 0.f, sb);
#pragma unroll
    for (int i = 0; i < N; ++i) { sw[i] = mul2(sw[i], sc[i]); sb[i] = mul2(sb[i], sc[i]); }
  };
  if ((MODE & MODE_JOIN) && !by_image) join_params();
  if (MODE & MODE_NORM) { cols.param(p.pre.weight, 1.f, w2); cols.param(p.pre.bias, 0.f, b2); }
  const Walk w(p, slots, s.id, WIDE, R, by_image);
  const int per_gate = by_image ? (int)(p.rows / p.gate_rows) : 1;
  int left = 0;                                // rows to go with the gate at hand

  const bool live = !VEC || cols.on(0);        // K = 1: a thread has its one vector or nothing
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(ring) + (VEC ? threadIdx.x * 16 : 0);
  const int at_x = cols.template stage<TR>(), at_g = at_x + (MODE & MODE_JOIN ? cols.template stage<TB>() : 0);
  const int one = at_g + (PIXEL ? cols.template stage<TB>() : 0), last = (depth - 1) * R * one;
  const Rows<TR> res(p.res, p.ldres, cols.first()), h_out(p.out, p.ldout, cols.first());
  const Rows<TB> x(p.x, p.ldx, cols.first()), gate(p.gate, p.ldgate, cols.first()), y_out(p.y, p.ldy, cols.first());
  int ahead = w.lo, in = 0, out = 0;           // the row that is copied next, stages that are filled and read next
  auto copy = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = ahead + r;
      if (row < w.hi && live) {
        const uint32_t to = base + in + r * one;
        cols.copy(res.at(row), to);
        if (MODE & MODE_JOIN) cols.copy(x.at(row), to + at_x);
        if (PIXEL) cols.copy(gate.at(row), to + at_g);
      }
    }
    ahead += w.step;
    in = in == last ? 0 : in + R * one;
    copy_commit();
  };
  if (cols.RING) {
    clear_ring(ring, depth * R * one);
    for (int i = 0; i < depth - 1; ++i) copy();
  }
  for (int i = 0; i < w.turns; ++i) {
    const int row = w.lo + i * w.step;
    if (cols.RING) {
      if (!VEC) s.sync();
      copy();
      copy_wait(depth);
      if (!VEC) s.sync();
    }
    const uint32_t from = base + out;
    if (cols.RING) out = out == last ? 0 : out + R * one;
    float2 h[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r) cols.load(res, row + r, row + r < w.hi, true, from + r * one, h[r]);
    if (MODE & MODE_JOIN) {
      float2 z[R][N];
#pragma unroll
      for (int r = 0; r < R; ++r) cols.load(x, row + r, row + r < w.hi, true, from + r * one + at_x, z[r]);
      if (p.post.kind) normalise<WIDE>(cols, s, p.post, row, w.hi, inv_c, z);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float2 g[N];
        const bool active = row + r < w.hi;
        if (by_image && left-- == 0 && active) {
          const int image = (row + r) / per_gate;
          left = (image + 1) * per_gate - (row + r) - 1;
          cols.fetch(gate.at(image), true, g);
          gate_factor(p.sigmoid, g);
          join_params();
#pragma unroll
          for (int j = 0; j < N; ++j) { sw[j] = mul2(sw[j], g[j]); sb[j] = mul2(sb[j], g[j]); }
        }
        if (PIXEL) { cols.load(gate, row + r, active, true, from + r * one + at_g, g); gate_factor(p.sigmoid, g); }
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (PIXEL) h[r][j] = fma2(fma2(z[r][j], sw[j], sb[j]), g[j], h[r][j]);
          else h[r][j] = add2(h[r][j], fma2(z[r][j], sw[j], sb[j]));
        }
        cols.store(h_out.at(row + r), active, h[r]);
      }
    }
    if (MODE & MODE_NORM) {
      normalise<WIDE>(cols, s, p.pre, row, w.hi, inv_c, h);
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < N; ++j) h[r][j] = fma2(h[r][j], w2[j], b2[j]);
        cols.store(y_out.at(row + r), row + r < w.hi, h[r]);
      }
    }
  }
}

// Sums kept per block in the workspace: [block][sums][C], A and B of the join, then dweight and dbias of the next norm;
// behind them a row of the gate's gradient for each (slot, image) pair that shares rows, number slot + image.
__host__ __device__ inline int sums_of(int mode) { return mode == MODE_BOTH ? 4 : 2; }

// dw, db, dscale from a column's sums
__device__ __forceinline__ void write_sums(const GeepsResidual& p, int mode, int c, const float* v) {
  if (mode & MODE_JOIN) {
    const float sc = p.scale ? p.scale[c] : 1.f;
    if (p.dscale) p.dscale[c] = (p.post.weight ? p.post.weight[c] : 1.f) * v[0] + (p.post.bias ? p.post.bias[c] : 0.f) * v[1];
    if (p.post.dweight) p.post.dweight[c] = sc * v[0];
    if (p.post.dbias) p.post.dbias[c] = sc * v[1];
    v += 2;
  }
  if (mode & MODE_NORM) {
    if (p.pre.dweight) p.pre.dweight[c] = v[0];
    if (p.pre.dbias) p.pre.dbias[c] = v[1];
  }
}

template <typename TR, typename TB, int K, bool VEC, bool WIDE, int MODE, bool PIXEL>
__global__ void __launch_bounds__(Form<TB, K, VEC, WIDE>::backward_threads)
residual_backward_kernel(const __grid_constant__ GeepsResidual p, int slot, int slots, int depth) {
  geeps_pdl_enter();
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 stats[2][512];
  __shared__ __align__(16) float red[16][128];
  constexpr int N = 4 * K, R = Form<TB, K, VEC, WIDE>::R;
  for (int i = threadIdx.x; i < 16 * 128; i += blockDim.x) red[0][i] = 0.f;
  for (int i = threadIdx.x; i < 2 * 512; i += blockDim.x) stats[0][i] = both(0.f);
  __syncthreads();
  Slot s;
  s.id = threadIdx.x / slot; s.t = threadIdx.x % slot; s.size = slot; s.red = red[WIDE ? s.id : 0]; s.turn = 0;
  const Columns<K, VEC, Form<TB, K, VEC, WIDE>::backward_threads> cols = {s.t, slot, p.C, slots};
  const float inv_c = 1.f / (float)p.C;
  const bool by_image = (MODE & MODE_JOIN) && !PIXEL && p.gate;
  float2 sw[N], sb[N], w2[N], a0[N], a1[N], n0[N], n1[N];     // sw: scale * weight, times the gate where an image has one
  auto scaled = [&](const float* of, float other, float2 (&f)[N]) {
    float2 sc[N];
    cols.param(p.scale, 1.f, sc); cols.param(of, other, f);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = mul2(f[i], sc[i]);
  };
  if (MODE & MODE_JOIN) {
    scaled(p.post.weight, 1.f, sw);
    if (PIXEL) scaled(p.post.bias, 0.f, sb);
#pragma unroll
    for (int i = 0; i < N; ++i) a0[i] = a1[i] = both(0.f);
  }
  if (MODE & MODE_NORM) {
    cols.param(p.pre.weight, 1.f, w2);
#pragma unroll
    for (int i = 0; i < N; ++i) n0[i] = n1[i] = both(0.f);
  }
  const Walk w(p, slots, s.id, WIDE, R, by_image);
  const int per_gate = by_image ? (int)(p.rows / p.gate_rows) : 1;
  int image = -1, left = 0;

  const bool live = !VEC || cols.on(0);        // K = 1: a thread has its one vector or nothing
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(ring) + (VEC ? threadIdx.x * 16 : 0);
  const int at_o = cols.template stage<TR>(), at_y = at_o + (MODE & MODE_NORM ? cols.template stage<TR>() : 0);
  const int at_x = at_y + (MODE & MODE_NORM ? cols.template stage<TB>() : 0);
  const int at_g = at_x + (MODE & MODE_JOIN ? cols.template stage<TB>() : 0);
  const int one = at_g + (PIXEL ? cols.template stage<TB>() : 0), last = (depth - 1) * R * one;
  const Rows<TR> dout(p.dout, p.lddout, cols.first()), h(p.out, p.ldout, cols.first()), dres(p.dres, p.lddres, cols.first());
  const Rows<TB> dy(p.dy, p.lddy, cols.first()), x(p.x, p.ldx, cols.first()), gate(p.gate, p.ldgate, cols.first());
  const Rows<TB> dx(p.dx, p.lddx, cols.first()), dgate(p.dgate, p.lddgate, cols.first());
  const bool has_dout = p.dout != nullptr;
  int ahead = w.lo, in = 0, out = 0;
  auto copy = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = ahead + r;
      const uint32_t to = base + in + r * one;
      if (row < w.hi) {
        if (live) {
          if (has_dout) cols.copy(dout.at(row), to);
          if (MODE & MODE_NORM) { cols.copy(h.at(row), to + at_o); cols.copy(dy.at(row), to + at_y); }
          if (MODE & MODE_JOIN) cols.copy(x.at(row), to + at_x);
          if (PIXEL) cols.copy(gate.at(row), to + at_g);
        }
      } else if (R > 1 || !WIDE) {             // rows that are read and are none: they add nothing to the sums
        cols.template no_row<TR>(to);
        if (MODE & MODE_NORM) { cols.template no_row<TR>(to + at_o); cols.template no_row<TB>(to + at_y); }
        if (MODE & MODE_JOIN) cols.template no_row<TB>(to + at_x);
        if (PIXEL) cols.template no_row<TB>(to + at_g);
      }
    }
    ahead += w.step;
    in = in == last ? 0 : in + R * one;
    copy_commit();
  };
  // with a gate per image a0 and a1 are the sums u and v of the image at hand; A and B of all images are kept behind the ring
  float* all_images = reinterpret_cast<float*>(ring + depth * R * one) + threadIdx.x;
  auto kept = [&](int i) -> float& { return all_images[i * slot * slots]; };
  if (by_image) {
    for (int i = 0; i < 4 * N; ++i) kept(i) = 0.f;
  }
  // the rows of an image that this slot has are done: its part of the gate's gradient, all of it if no other slot has any
  auto image_done = [&]() {
    float2 g[N], d[N], b[N];
    cols.fetch(gate.at(image), true, g);
    gate_factor(p.sigmoid, g);
    scaled(p.post.weight, 1.f, d); scaled(p.post.bias, 0.f, b);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      d[i] = mul2(fma2(d[i], a0[i], mul2(b[i], a1[i])), gate_slope(p.sigmoid, g[i]));
      kept(4 * i) = fmaf(g[i].x, a0[i].x, kept(4 * i)); kept(4 * i + 1) = fmaf(g[i].y, a0[i].y, kept(4 * i + 1));
      kept(4 * i + 2) = fmaf(g[i].x, a1[i].x, kept(4 * i + 2)); kept(4 * i + 3) = fmaf(g[i].y, a1[i].y, kept(4 * i + 3));
      a0[i] = a1[i] = both(0.f);
    }
    if (!p.dgate) return;
    if (image * per_gate >= w.lo && (image + 1) * per_gate <= w.hi) cols.store(dgate.at(image), true, d);
    else {
      float* to = p.work + ((long long)gridDim.x * sums_of(MODE) + (long long)blockIdx.x * slots + s.id + image) * p.C;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (cols.on(2 * i)) to[cols.at(2 * i)] = d[i].x;
        if (cols.on(2 * i + 1)) to[cols.at(2 * i + 1)] = d[i].y;
      }
    }
  };
  if (cols.RING) {
    clear_ring(ring, depth * R * one);
    for (int i = 0; i < depth - 1; ++i) copy();
  }
  for (int i = 0; i < w.turns; ++i) {
    const int row = w.lo + i * w.step;
    if (cols.RING) {
      if (!VEC) s.sync();
      copy();
      copy_wait(depth);
      if (!VEC) s.sync();
    }
    const uint32_t from = base + out;
    if (cols.RING) out = out == last ? 0 : out + R * one;
    // Statistics of the rows of several turns at a time, a row a lane: a load for every turn was waited for in the turn that
    // issued it, with the loads from shared memory that share its scoreboard (50176 x 576: 36 % of the time).
    const int chunk = WIDE ? 32 : slot, k = i * R & (chunk - 1);
    if (k == 0) {
      const int turn = i + (s.t & (chunk - 1)) / R, q = w.lo + turn * w.step + (s.t & (R - 1));
      __syncwarp();
      if (turn < w.turns && q < w.hi) {
        if ((MODE & MODE_JOIN) && p.post.kind) stats[0][threadIdx.x] = *reinterpret_cast<const float2*>(p.post.stats + 2LL * q);
        if (MODE & MODE_NORM) stats[1][threadIdx.x] = *reinterpret_cast<const float2*>(p.pre.stats + 2LL * q);
      }
      __syncwarp();
    }
    float2 now1[R], now2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int lane = (threadIdx.x & ~(chunk - 1)) + k + r;
      now1[r] = MODE & MODE_JOIN ? stats[0][lane] : both(0.f);
      now2[r] = MODE & MODE_NORM ? stats[1][lane] : both(0.f);
    }
    // an output may lie where an operand does: without a ring everything of the row is read before its first output is written
    float2 dh[R][N], z[R][N], g[R][N];
    auto load_branch = [&]() {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool active = WIDE && R == 1 || row + r < w.hi;
        if (MODE & MODE_JOIN) cols.load(x, row + r, active, true, from + r * one + at_x, z[r]);
        if (PIXEL) { cols.load(gate, row + r, active, true, from + r * one + at_g, g[r]); gate_factor(p.sigmoid, g[r]); }
      }
    };
    if (!cols.RING) load_branch();
#pragma unroll
    for (int r = 0; r < R; ++r) cols.load(dout, row + r, WIDE && R == 1 || row + r < w.hi, has_dout, from + r * one, dh[r]);
    if (MODE & MODE_NORM) {
      float2 n[R][N], a[R][N];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool active = WIDE && R == 1 || row + r < w.hi;
        cols.load(h, row + r, active, true, from + r * one + at_o, n[r]);
        cols.load(dy, row + r, active, true, from + r * one + at_y, a[r]);
        normalised(n[r], now2[r]);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          n0[j] = fma2(a[r][j], n[r][j], n0[j]); n1[j] = add2(n1[j], a[r][j]);
          a[r][j] = mul2(a[r][j], w2[j]);
        }
      }
      norm_gradient<WIDE>(s, p.pre.kind, now2, inv_c, n, a, dh);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) cols.store(dres.at(row + r), WIDE && R == 1 || row + r < w.hi, dh[r]);
    if (MODE & MODE_JOIN) {
      if (cols.RING) load_branch();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool active = WIDE && R == 1 || row + r < w.hi;
        if (by_image && left == 0 && active) {
          if (image >= 0) image_done();
          image = (row + r) / per_gate;
          left = (image + 1) * per_gate - (row + r);
          float2 factor[N];
          cols.fetch(gate.at(image), true, factor);
          gate_factor(p.sigmoid, factor);
          scaled(p.post.weight, 1.f, sw);
#pragma unroll
          for (int j = 0; j < N; ++j) sw[j] = mul2(sw[j], factor[j]);
        }
        --left;
        if (p.post.kind) normalised(z[r], now1[r]);
        float2 dg[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          float2 d = dh[r][j];
          if (PIXEL) {
            dg[j] = mul2(mul2(d, fma2(sw[j], z[r][j], sb[j])), gate_slope(p.sigmoid, g[r][j]));
            d = mul2(d, g[r][j]);
          }
          a0[j] = fma2(d, z[r][j], a0[j]); a1[j] = add2(a1[j], d);
          dh[r][j] = mul2(d, sw[j]);
        }
        if (PIXEL && p.dgate) cols.store(dgate.at(row + r), active, dg);
      }
      if (p.post.kind) {
        float2 e[R][N];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int j = 0; j < N; ++j) e[r][j] = both(0.f);
        }
        norm_gradient<WIDE>(s, p.post.kind, now1, inv_c, z, dh, e);
#pragma unroll
        for (int r = 0; r < R; ++r) cols.store(dx.at(row + r), WIDE && R == 1 || row + r < w.hi, e[r]);
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) cols.store(dx.at(row + r), WIDE && R == 1 || row + r < w.hi, dh[r]);
      }
    }
  }
  if (by_image && image >= 0) image_done();
  // the slots' sums, in slot order, in the threads of slot 0
  if (by_image) {
#pragma unroll
    for (int i = 0; i < N; ++i) { a0[i] = make_float2(kept(4 * i), kept(4 * i + 1)); a1[i] = make_float2(kept(4 * i + 2), kept(4 * i + 3)); }
  }
  __syncthreads();
  float2* meet = reinterpret_cast<float2*>(ring);
  auto over_slots = [&](float2 (&v)[N]) {
    if (slots == 1) return;
#pragma unroll
    for (int j = 0; j < N; ++j) meet[(s.id * N + j) * slot + s.t] = v[j];
    __syncthreads();
    if (s.id == 0) {
      for (int i = 1; i < slots; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = add2(v[j], meet[(i * N + j) * slot + s.t]);
      }
    }
    __syncthreads();
  };
  if (MODE & MODE_JOIN) { over_slots(a0); over_slots(a1); }
  if (MODE & MODE_NORM) { over_slots(n0); over_slots(n1); }
  if (s.id != 0) return;
#pragma unroll
  for (int j = 0; j < 2 * N; ++j) {
    if (!cols.on(j)) continue;
    const int c = cols.at(j);
    auto of = [&](const float2 (&f)[N]) { return j & 1 ? f[j >> 1].y : f[j >> 1].x; };
    float v[4];
    int k = 0;
    if (MODE & MODE_JOIN) { v[k++] = of(a0); v[k++] = of(a1); }
    if (MODE & MODE_NORM) { v[k++] = of(n0); v[k++] = of(n1); }
    if (gridDim.x == 1) write_sums(p, MODE, c, v);
    else for (int i = 0; i < sums_of(MODE); ++i) p.work[((long long)blockIdx.x * sums_of(MODE) + i) * p.C + c] = v[i];
  }
}

// Second launch: the blocks' sums in block order (blockIdx.y = 0), and the gate's gradient of the images whose rows several
// slots had: blockIdx.y - 1, by gridDim.y - 1, goes through the slots that begin inside of an image and are its first cut.
template <typename TB>
__global__ void __launch_bounds__(256)
residual_sums_kernel(const __grid_constant__ GeepsResidual p, int mode, int blocks, int slots) {
  geeps_pdl_enter();
  const int lane = threadIdx.x & 7, part = threadIdx.x >> 3, c = blockIdx.x * 8 + lane, sums = sums_of(mode);
  if (blockIdx.y == 0) {
    if (blocks == 1) return;
    __shared__ float sh[32][4][8];
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < p.C) {
      for (int b = part; b < blocks; b += 32)
        for (int i = 0; i < sums; ++i) v[i] += p.work[((long long)b * sums + i) * p.C + c];
    }
    for (int i = 0; i < 4; ++i) sh[part][i][lane] = v[i];
    __syncthreads();
    if (part != 0 || c >= p.C) return;
    for (int i = 0; i < sums; ++i) { v[i] = 0.f; for (int q = 0; q < 32; ++q) v[i] += sh[q][i][lane]; }
    write_sums(p, mode, c, v);
    return;
  }
  if (c >= p.C) return;
  const int rows = (int)p.rows, per_gate = (int)(p.rows / p.gate_rows);
  const int all = blocks * slots;
  const float* w = p.work + (long long)blocks * sums * p.C;
  for (int b = 1 + (blockIdx.y - 1) * 32 + part; b < all; b += (gridDim.y - 1) * 32) {
    const int cut = first_row(rows, all, b);
    if (cut >= rows) break;
    const int image = cut / per_gate, start = image * per_gate;
    if (cut == start || first_row(rows, all, b - 1) > start) continue;
    float v = 0.f;
    for (int q = b - 1; q < all && first_row(rows, all, q) - start < per_gate && first_row(rows, all, q) < rows; ++q)
      v += w[((long long)q + image) * p.C + c];
    ((TB*)p.dgate)[image * p.lddgate + c] = (TB)v;
  }
}

// ---- launches ----
// stages of the ring: what fits, up to four (kRingBytes holds one of every kind of call with a ring)
template <typename TR, typename TB, int K, bool VEC, bool WIDE>
int ring_depth(const GeepsResidual& p, const Shape& s, bool backward, size_t* bytes) {
  typedef Form<TB, K, VEC, WIDE> F;
  const bool norm = p.mode & MODE_NORM, join = p.mode & MODE_JOIN, by_pixel = p.gate && p.gate_rows == p.rows, by_image = p.gate && !by_pixel;
  const int r = backward ? (norm ? 2 : 1) : 1, b = (backward && norm ? 1 : 0) + (join ? 1 : 0) + (by_pixel ? 1 : 0);
  const size_t threads = backward ? F::backward_threads : F::forward_threads;
  auto stage = [&](int size) { return F::R * (VEC ? K * 8 * size * threads : (size_t)((p.C * size + 15) / 16 + 1) * 16 * s.slots); };
  const size_t one = r * stage(sizeof(TR)) + b * stage(sizeof(TB)), kept = backward && by_image ? (size_t)s.threads() * 16 * K * sizeof(float) : 0;
  const size_t room = kRingBytes / s.per_sm - kept;
  const int depth = !Columns<K, VEC, 512>::RING ? 0 : one * 4 <= room ? 4 : (int)(room / one);
  *bytes = depth * one + kept;
  return depth;
}

// done: one a kernel
template <typename F>
void allow_shared(F kernel, size_t bytes, bool (&done)[64]) {
  if (bytes <= 24 * 1024) return;             // the default limit, 48 KB, less what the kernels have statically
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 && done[dev]) return;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024) == cudaSuccess && dev >= 0 && dev < 64)
    done[dev] = true;
}

template <typename TR, typename TB, int K, bool VEC, bool WIDE, int MODE, bool PIXEL>
void launch_kernel(const GeepsResidual& p, const Shape& s, bool backward, cudaStream_t st) {
  static bool forward_done[64] = {false}, backward_done[64] = {false};
  size_t smem = 0;
  const int depth = ring_depth<TR, TB, K, VEC, WIDE>(p, s, backward, &smem);
  if (backward) {
    const size_t meet = s.slots > 1 ? (size_t)s.threads() * 8 * K * sizeof(float) : 0;
    if (smem < meet) smem = meet;
    const auto kernel = residual_backward_kernel<TR, TB, K, VEC, WIDE, MODE, PIXEL>;
    allow_shared(kernel, smem, backward_done);
    geeps_launch(kernel, dim3(s.blocks), dim3(s.threads()), smem, st, p, s.slot, s.slots, depth);
  } else {
    const auto kernel = residual_forward_kernel<TR, TB, K, VEC, WIDE, MODE, PIXEL>;
    allow_shared(kernel, smem, forward_done);
    geeps_launch(kernel, dim3(s.blocks), dim3(s.threads()), smem, st, p, s.slot, s.slots, depth);
  }
}
template <typename TR, typename TB, int K, bool VEC, bool WIDE>
void launch(const GeepsResidual& p, const Shape& s, bool backward, cudaStream_t st) {
  const bool by_pixel = p.gate && p.gate_rows == p.rows;
  if (p.mode == MODE_NORM) launch_kernel<TR, TB, K, VEC, WIDE, MODE_NORM, false>(p, s, backward, st);
  else if (p.mode == MODE_JOIN && by_pixel) launch_kernel<TR, TB, K, VEC, WIDE, MODE_JOIN, true>(p, s, backward, st);
  else if (p.mode == MODE_JOIN) launch_kernel<TR, TB, K, VEC, WIDE, MODE_JOIN, false>(p, s, backward, st);
  else if (by_pixel) launch_kernel<TR, TB, K, VEC, WIDE, MODE_BOTH, true>(p, s, backward, st);
  else launch_kernel<TR, TB, K, VEC, WIDE, MODE_BOTH, false>(p, s, backward, st);
}
template <typename TR, typename TB, bool VEC>
void run_vec(const GeepsResidual& p, const Shape& s, bool backward, cudaStream_t st) {
  if (s.slot < 32) launch<TR, TB, 1, VEC, false>(p, s, backward, st);
  else if (s.vectors == 1) launch<TR, TB, 1, VEC, true>(p, s, backward, st);
  else if (s.vectors == 2) launch<TR, TB, 2, VEC, true>(p, s, backward, st);
  else launch<TR, TB, 4, VEC, true>(p, s, backward, st);
}
template <typename TR, typename TB>
void run(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st) {
  const Shape s = plan(p.rows, p.C, backward, p.mode);
  (vec ? run_vec<TR, TB, true> : run_vec<TR, TB, false>)(p, s, backward, st);
  const bool cuts = p.gate && p.gate_rows < p.rows && p.dgate;
  if (!backward || (s.blocks == 1 && !(cuts && s.slots > 1))) return;
  int y = cuts ? (s.blocks * s.slots + 31) / 32 : 0;
  if (y > 64) y = 64;
  geeps_launch(residual_sums_kernel<TB>, dim3((p.C + 7) / 8, 1 + y), dim3(256), 0, st, p, p.mode, s.blocks, s.slots);
}

void run_bf16(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st);
void run_mixed(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st);
void run_fp32(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st);

}  // namespace rownorm
