// The kernels of norm.cu, which has the mathematics and the checks: one translation unit for each pair of types.
#pragma once
#include "common.cuh"
#include "nn_ops.h"

#include <type_traits>

typedef __nv_bfloat16 bf16;

namespace rownorm {

constexpr int kMaxChannels = 16384;
constexpr int kVec = 8;                 // channels a vector
constexpr int kRingBytes = 200 * 1024;  // shared memory of an SM for parameters and rows on their way
enum { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };
enum { MODE_NORM = 1, MODE_JOIN = 2, MODE_BOTH = 3 };     // the next norm alone, a join alone, a join and the norm behind it

// ---- launch shape ----
// VEC: rows of whole, aligned vectors.  large (forward): rows that registers and shared memory do not hold; wide (forward): rows
// that one block an SM works on, so that the parameters lie there once; tiles (backward): rows cut into ranges of `width` columns.
struct Shape {
  int vectors;       // vectors a thread
  int slot;          // threads a row: a power of two up to 32, or whole warps
  int slots;         // rows a block works on at a time
  int blocks, per_sm, depth;
  bool large, wide;
  int tiles, width;
  size_t ring, smem;      // bytes before the ring, and of all
  int threads() const { return slot * slots; }
};
// Threads of a block.  Backward a block has an SM to itself, so that few blocks leave column sums behind, and as many threads as
// their column sums leave registers for; forward several blocks of 256 share an SM, and from 4096 channels on blocks of 512
// (us, blocks of 256 / 512, 4000 x 6144: bf16 norm 40 / 32, join and norm without a gate 44 / 37, fp32 84 / 60; 16250 x 1536, bf16:
// 22.8 / 22.7, 46.5 / 48.3; single columns, 3332 x 6001 join 376 / 70).
__host__ __device__ constexpr int block_threads(bool backward, bool vec, bool large, bool wide, int vectors, int mode) {
  return large || wide ? 512 : !backward ? 256 : !vec ? 512 : vectors > 2 && mode != MODE_NORM ? 256 : 384;
}
// ... and blocks an SM that registers allow forward
__host__ __device__ constexpr int blocks_forward(bool large, bool wide, int mode) {
  return large ? 1 : (mode == MODE_NORM ? 4 : 2) / (wide ? 2 : 1);
}

// What a call keeps in shared memory: parameters of the columns (one vector a thread keeps them in registers), with a gate per
// image its factors, and the ring.
struct Call {
  bool backward, vec, by_pixel, by_image, tile;
  int mode, stream, block;                 // sizes of the two types
  int threads(const Shape& s) const { return block_threads(backward, vec, s.large, s.wide, s.vectors, mode); }
};
inline size_t fixed_bytes(const Call& c, const Shape& s) {
  const bool norm = c.mode & MODE_NORM, join = c.mode & MODE_JOIN;
  const int params = c.backward ? (norm ? 1 : 0) + (join ? c.by_pixel || c.by_image ? 2 : 1 : 0) : (norm ? 2 : 0) + (join ? 2 : 0);
  const size_t thread = (size_t)8 * s.vectors * sizeof(float);         // a value for each of a thread's columns
  return (s.large || s.vectors == 1 ? 0 : params * thread * s.slot) + (c.by_image ? thread * c.threads(s) : 0);
}
inline size_t stage_bytes(const Call& c, const Shape& s) {
  const bool norm = c.mode & MODE_NORM, join = c.mode & MODE_JOIN;
  const int r = c.backward ? (norm ? 2 : 1) : 1, b = (c.backward && norm ? 1 : 0) + (join ? 1 : 0) + (c.by_pixel ? 1 : 0);
  auto stage = [&](int size) {
    return c.vec ? (size_t)s.vectors * 8 * size * c.threads(s) : (size_t)(8 * s.vectors * s.slot * size + 16) * s.slots;
  };
  return r * stage(c.stream) + b * stage(c.block);
}
// Backward, rows that no thread count holds with their column sums are cut into tiles of columns, with the row's means taken by a
// launch of its own: it reads once more, but nothing spills (3325 x 8972 bf16, join and norm: 1765 us by one block a row; 2230 x
// 8968: 147).
// Rows that fit stay whole (2441 x 4096: 55 us, two tiles 85; 1220 x 8192: 89, 96), but for single columns of a join with a norm
// behind it and no gate for every pixel, where 16 columns a thread do not fit in 128 registers (2438 x 4101 240 us, 149; 1249 x
// 8001 169, 154).  A tile is as wide as a block has columns: narrower ones lose (8192 in eight: 184).
constexpr int tile_columns(bool vec) { return vec ? 2 * kVec * 384 : kVec * 512; }
constexpr bool spills(bool backward, int mode, bool by_pixel) { return backward && mode == MODE_BOTH && !by_pixel; }
// How many vectors a thread has: more save what every thread does once a row, fewer leave no lane without work.  The costs are
// instructions a row.  Eight threads a row at least, where there is so much: pieces of rows in a warp's access are whole lines then
// (50176 x 64 backward 12 us, 21 with four).  A join with a norm behind it has four column sums: two vectors while they do
// (50176 x 1024 backward 115 us, four vectors by half the threads 180).
inline Shape plan(long long rows, int C, const Call& c) {
  Shape best = {};
  best.tiles = 1;
  best.width = C;
  const int vec = (C + kVec - 1) / kVec, most = c.tile ? (c.vec ? 2 : 1) : c.vec ? 4 : spills(c.backward, c.mode, c.by_pixel) ? 1 : 2;
  long long least = -1;
  const bool wide = !c.backward && vec >= (c.vec ? 512 : 513);
  for (int k = wide ? 0 : c.tile ? most : 1; k <= (c.backward ? most : most + 1); ++k) {   // 0: blocks of 512, the rest where these do not fit
    Shape s = best;
    s.large = k > most;
    s.wide = k == 0;
    s.vectors = s.wide || s.large ? 4 : k;
    if (least >= 0 && best.wide) break;
    const int need = (vec + s.vectors - 1) / s.vectors, limit = c.threads(s);
    if (need > limit || ((s.large || (c.backward && c.mode == MODE_BOTH && k > 2)) && least >= 0)) continue;
    s.slot = 1;
    while (s.slot < 32 && (s.slot < need || (s.slot < 8 && s.slot < vec))) s.slot <<= 1;
    if (need > 32 || s.large || c.tile) s.slot = (need + 31) / 32 * 32;
    if (s.slot >= 32 && s.vectors == 1 && c.vec) continue;
    if (s.slot < 32 && s.vectors == 2 && !c.vec) continue;
    s.slots = limit / s.slot;
    s.ring = fixed_bytes(c, s);
    const size_t stage = stage_bytes(c, s);
    s.depth = 0;
    // a row of single columns by a block of 512 is read where it lies if its parameters leave no room for it (2493 x 8021, join and
    // norm 160 us, 455 with the parameters read again for every row)
    for (s.per_sm = c.backward ? 1 : blocks_forward(s.large, s.wide, c.mode); s.per_sm >= 1 && s.depth < 1; --s.per_sm) {
      const size_t room = kRingBytes / s.per_sm;
      s.depth = s.ring > room ? 0 : s.ring + 4 * stage <= room ? 4 : (int)((room - s.ring) / stage);
    }
    ++s.per_sm;
    if (!s.large && s.depth < 1 && !(s.wide && !c.vec && s.ring <= kRingBytes)) continue;
    s.smem = s.ring + s.depth * stage;
    const long long cost = (long long)s.slot * (100 + 45 * s.vectors + (s.slot > 32 ? 60 : 0));
    if (least < 0 || (cost < least && c.vec)) { least = cost; best = s; }       // single columns cost the same for any k
  }
  if (least < 0 && !c.tile) {               // backward only
    Call t = c;
    t.tile = true;
    const int most_columns = tile_columns(c.vec), tiles = (C + most_columns - 1) / most_columns, width = ((C + tiles - 1) / tiles + kVec - 1) / kVec * kVec;
    best = plan(rows, width, t);
    best.tiles = tiles;
    return best;
  }
  const long long room = (long long)geeps_sm_count() * best.per_sm, want = (rows + best.slots - 1) / best.slots;
  best.blocks = (int)(want < room ? want : room);
  return best;
}
// The kernels that plan() asks for, besides those for large rows and tiles; no others are built.  `big`: blocks of 512 forward.  Of
// whole vectors one a thread never fills a warp, and two or three are dearer than four from there on unless four column sums leave
// no registers for them (then three are not cheapest anywhere).  A gate for every row in fp32 leaves no shared memory for a ring
// beside four vectors of 512 threads' parameters, nor for rows of four vectors beside four column sums.
constexpr bool planned(bool backward, bool vec, bool wide, bool big, int vectors, int mode, bool by_pixel, int block) {
  const bool both = mode == MODE_BOTH, room = !(by_pixel && block == 4);
  if (!vec) return vectors == 4 ? big && (room || !both) : vectors == 1 || !spills(backward, mode, by_pixel);
  if (big) return vectors == 4 && room;
  if (!backward) return vectors > 2 || !wide;
  return vectors == 1 ? !wide : vectors == 2 ? !wide || both : vectors == 3 ? !both : !both || (wide && room);
}
// rows [first_row(i), first_row(i + 1)) are slot i's, of all slots of all blocks; rows are at most 2^30
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
// ... a piece whose other half of a 32-byte sector comes with another copy
__device__ __forceinline__ void copy16_half(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void st_f8(float* p, float2 a, float2 b, float2 c, float2 d) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y),
               "f"(d.x), "f"(d.y) : "memory");
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
// K vectors of eight, held as pairs.  VEC: vectors t, t + slot, ...: 16- or 32-byte accesses.  Otherwise (odd widths, pitches or
// addresses) single columns t, t + slot, ...: neighbouring threads on neighbouring columns.  A thread without a column at some
// place has zeros there.
// Rows come through a ring of `depth` stages in shared memory, so that what is on its way takes no registers.  With VEC a thread
// copies what it reads itself and nobody waits for anybody; otherwise the slot copies the 16-byte pieces that hold the row (up
// to 15 bytes before and behind it in the same pieces come along) and meets before and after reading them.  The ring starts as
// zeros where no copy goes, so what has no column or no operand is read from it like the rest.  LARGE rows take more threads,
// leave no room for parameters, and are read where they lie if they do not fit the ring.  THREADS: as many as a block may have; a
// thread's places in the ring are then the same for every launch.
// DIRECT: without a ring, if `ring` says so.
template <int K, bool VEC, bool DIRECT, int THREADS>
struct Columns {
  static constexpr int N = 4 * K;      // pairs
  int t, slot, C, slots;
  bool ring;
  __device__ __forceinline__ int first() const { return VEC ? at(0) : 0; }
  __device__ __forceinline__ int at(int j) const { return VEC ? (t + (j >> 3) * slot) * 8 + (j & 7) : t + j * slot; }
  __device__ __forceinline__ bool on(int j) const { return at(VEC ? j & ~7 : j) < C; }

  // bytes of a row of a slot without VEC, and of a stage for one stream of T
  template <typename T>
  __device__ __forceinline__ int pieces() const { return 8 * K * slot * (int)sizeof(T) + 16; }
  template <typename T>
  __device__ __forceinline__ int stage() const { return VEC ? K * 8 * (int)sizeof(T) * THREADS : pieces<T>() * slots; }
  // `from` is what Rows::at() gives; `to` has the thread's 16 * threadIdx.x with VEC, the slot's share without
  template <typename T>
  __device__ __forceinline__ void copy(const T* from, uint32_t to) const {
    if (VEC) {
      constexpr int Q = 8 * sizeof(T) / 16;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!on(8 * k)) continue;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          if (Q == 1) copy16(to + k * THREADS * 16, from + k * slot * 8);
          else copy16_half(to + (k * Q + q) * THREADS * 16, from + k * slot * 8 + q * (8 / Q));
        }
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
  // zeros in the place of what no copy fills: vectors behind the row, or all of a row that is not there
  template <typename T>
  __device__ __forceinline__ void no_copy(uint32_t to, bool all) const {
    if (!VEC) return;
    constexpr int Q = 8 * sizeof(T) / 16;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!all && on(8 * k)) continue;
#pragma unroll
      for (int q = 0; q < Q; ++q)
        asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(to + (k * Q + q) * THREADS * 16), "r"(0) : "memory");
    }
  }
  // a row from the ring if there is one; zeros where the slot has no such row
  template <typename T>
  __device__ __forceinline__ void load(const Rows<T>& rows, int row, bool active, bool there, uint32_t from, float2 (&f)[N]) const {
    if (DIRECT && !ring) {
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
      float v[2 * N];              // without branches: what lies behind the row is read and dropped
#pragma unroll
      for (int j = 0; j < 2 * N; ++j) v[j] = ld_shared1<T>(r + at(j) * (int)sizeof(T));
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = make_float2(any && on(2 * i) ? v[2 * i] : 0.f, any && on(2 * i + 1) ? v[2 * i + 1] : 0.f);
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
          st_f8(reinterpret_cast<float*>(row) + c, v[0], v[1], v[2], v[3]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2 * N; ++j) if (on(j)) row[at(j)] = (T)(j & 1 ? f[j >> 1].y : f[j >> 1].x);
    }
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

// A parameter of every column: one, times another, or `other` where there is none.  In registers for one vector a thread, else
// in shared memory (16 bytes of a vector's half beside those of the next thread), read for every row; rows that do not fit read
// it where it lies.
template <typename C_, int K, bool VEC, bool LARGE>
struct Param {
  static constexpr bool REG = K == 1, SHARED = K > 1 && !LARGE;
  float2 reg[REG ? 4 * K : 1];
  uint32_t at;
  const float *one, *two;
  float other;
  __device__ __forceinline__ float value(int c) const { return (one ? one[c] : other) * (two ? two[c] : 1.f); }
  // `area` moves on behind what is taken; the block meets before the first get()
  __device__ __forceinline__ void set(const C_& cols, const float* a, float b, const float* c, unsigned char*& area) {
    one = a; two = c; other = b;
    if (REG) {
#pragma unroll
      for (int i = 0; i < C_::N; ++i)
        reg[REG ? i : 0] = make_float2(cols.on(2 * i) ? value(cols.at(2 * i)) : 0.f, cols.on(2 * i + 1) ? value(cols.at(2 * i + 1)) : 0.f);
    } else if (SHARED) {
      // eight loads are under way at a time: one after the other they were a fifth of a short call
      float* to = reinterpret_cast<float*>(area);
      const int all = 8 * K * cols.slot, step = blockDim.x;
      for (int i0 = threadIdx.x; i0 < all; i0 += 8 * step) {
        float v[8], w[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = i0 + u * step;
          int col = i;
          if (VEC) {       // [k][half][thread][4]
            const int e = i & 3, q = i >> 2, t = q % cols.slot, h = q / cols.slot;
            col = (t + (h >> 1) * cols.slot) * 8 + (h & 1) * 4 + e;
          }
          const bool there = i < all && col < cols.C;
          v[u] = !there ? 0.f : one ? one[col] : other;
          w[u] = there && two ? two[col] : 1.f;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) if (i0 + u * step < all) to[i0 + u * step] = v[u] * w[u];
      }
      at = (uint32_t)__cvta_generic_to_shared(area) + cols.t * (VEC ? 16 : 4);
      area += 8 * K * cols.slot * sizeof(float);
    }
  }
  // pairs 4 k to 4 k + 3
  __device__ __forceinline__ void get(const C_& cols, int k, float2 (&f)[4]) const {
    if (REG) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = reg[REG ? 4 * k + e : 0];
    } else if (SHARED && VEC) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 v = ld_shared16(at + (2 * k + h) * cols.slot * 16);
        f[2 * h] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        f[2 * h + 1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
      }
    } else if (SHARED) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = make_float2(ld_shared1<float>(at + (8 * k + 2 * e) * cols.slot * 4), ld_shared1<float>(at + (8 * k + 2 * e + 1) * cols.slot * 4));
    } else {
      const int c = cols.at(8 * k);
      if (VEC && (((uintptr_t)one | (uintptr_t)two) & 15) == 0) {
        float v[8], w[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool on = cols.on(8 * k);
          const float4 a = on && one ? ld_f4(one + c + 4 * h) : make_float4(on ? other : 0.f, on ? other : 0.f, on ? other : 0.f, on ? other : 0.f);
          const float4 b = on && two ? ld_f4(two + c + 4 * h) : make_float4(1.f, 1.f, 1.f, 1.f);
          v[4 * h] = a.x; v[4 * h + 1] = a.y; v[4 * h + 2] = a.z; v[4 * h + 3] = a.w;
          w[4 * h] = b.x; w[4 * h + 1] = b.y; w[4 * h + 2] = b.z; w[4 * h + 3] = b.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = make_float2(v[2 * e] * w[2 * e], v[2 * e + 1] * w[2 * e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 8 * k + 2 * e;
          f[e] = make_float2(cols.on(j) ? value(cols.at(j)) : 0.f, cols.on(j + 1) ? value(cols.at(j + 1)) : 0.f);
        }
      }
    }
  }
};
// A thread's own values of its columns in shared memory: 16 bytes beside those of the next thread
template <int K, int THREADS>
struct Own {
  uint32_t at;
  __device__ __forceinline__ void set(unsigned char*& area) {
    at = (uint32_t)__cvta_generic_to_shared(area) + threadIdx.x * 16;
    area += 8 * K * THREADS * sizeof(float);
  }
  __device__ __forceinline__ void get(int k, float2 (&f)[4]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 v = ld_shared16(at + (2 * k + h) * THREADS * 16);
      f[2 * h] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
      f[2 * h + 1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
  }
  __device__ __forceinline__ void put(int k, const float2 (&f)[4]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(at + (2 * k + h) * THREADS * 16), "f"(f[2 * h].x), "f"(f[2 * h].y),
                   "f"(f[2 * h + 1].x), "f"(f[2 * h + 1].y) : "memory");
  }
};

struct Slot {
  int id, t, size;
  float* red;        // 64 floats of shared memory: two turns of 32, zero where no warp writes
  int turn;
  __device__ __forceinline__ void sync() const {
    if (size > 32) asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(size) : "memory");
    else __syncwarp();
  }
};

// Sums of one or two values over the threads of a slot, the same in each.  Of two, a half of the warp goes on with each after
// the first step.  Warps meet in shared memory at the slot's named barrier; the two turns of `red` alternate, so the next sums
// may be written while these are still being read.
template <bool WIDE>
__device__ __forceinline__ float slot_sum(float v, Slot& s) {
  if (!WIDE) {
    for (int o = s.size >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (s.size == 32) return v;
  float* r = s.red + s.turn;
  s.turn ^= 32;
  if ((s.t & 31) == 0) r[s.t >> 5] = v;
  s.sync();
  float4 q = ld_f4(r);
  v = (q.x + q.y) + (q.z + q.w);
  for (int w = 128; w < s.size; w += 128) { q = ld_f4(r + (w >> 5)); v += (q.x + q.y) + (q.z + q.w); }
  return v;
}
template <bool WIDE>
__device__ __forceinline__ float2 slot_sum(float2 v, Slot& s) {
  if (!WIDE) {
    for (int o = s.size >> 1; o; o >>= 1) { v.x += __shfl_xor_sync(0xffffffffu, v.x, o); v.y += __shfl_xor_sync(0xffffffffu, v.y, o); }
    return v;
  }
  const bool upper = threadIdx.x & 16;
  float one = upper ? v.y : v.x;
  one += __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
  if (s.size == 32) {
    const float other = __shfl_xor_sync(0xffffffffu, one, 16);
    return upper ? make_float2(other, one) : make_float2(one, other);
  }
  float* r = s.red + s.turn;
  s.turn ^= 32;
  if ((s.t & 15) == 0) r[s.t >> 4] = one;
  s.sync();
  float4 q = ld_f4(r);
  v = make_float2(q.x + q.z, q.y + q.w);
  for (int w = 64; w < s.size; w += 64) { q = ld_f4(r + (w >> 4)); v.x += q.x + q.z; v.y += q.y + q.w; }
  return v;
}
// 1 / sqrt(v): the approximation and a step of Newton's, which leaves it within two roundings
__device__ __forceinline__ float inverse_root(float v) {
  const float y = rsqrtf(v);
  return v > 0.f && v < 3e38f ? fmaf(y * fmaf(-v * y, y, 1.f), 0.5f, y) : y;
}
// Sums over a thread's pairs, in up to four chains: few warps share a scheduler
template <int N>
__device__ __forceinline__ float total(const float2 (&f)[N]) {
  constexpr int W = N >= 16 ? 4 : N >= 8 ? 2 : 1;
  float2 v[W];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i % W] = i < W ? f[i] : add2(v[i % W], f[i]);
#pragma unroll
  for (int i = W >> 1; i; i >>= 1)
#pragma unroll
    for (int u = 0; u < i; ++u) v[u] = add2(v[u], v[u + i]);
  return v[0].x + v[0].y;
}
template <int N>
__device__ __forceinline__ float dot(const float2 (&f)[N], const float2 (&g)[N]) {
  constexpr int W = N >= 16 ? 4 : N >= 8 ? 2 : 1;
  float2 v[W];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i % W] = i < W ? mul2(f[i], g[i]) : fma2(f[i], g[i], v[i % W]);
#pragma unroll
  for (int i = W >> 1; i; i >>= 1)
#pragma unroll
    for (int u = 0; u < i; ++u) v[u] = add2(v[u], v[u + i]);
  return v[0].x + v[0].y;
}

// n = (f - mean) * rstd in place; mean and rstd go to stats.  used(): called when the first sum of f is there
template <bool WIDE, typename C_, int N, typename U_>
__device__ __forceinline__ void normalise(const C_& cols, Slot& s, const GeepsNorm& norm, int row, bool active, float inv_c, float2 (&f)[N],
                                          U_ used) {
  float mean = 0.f, squares;
  if (norm.kind == NORM_LAYER) {
    mean = slot_sum<WIDE>(total(f), s) * inv_c;
    used();
    cols.subtract(f, mean);
    squares = slot_sum<WIDE>(dot(f, f), s);
  } else {
    squares = slot_sum<WIDE>(dot(f, f), s);
    used();
  }
  const float rstd = inverse_root(fmaf(squares, inv_c, norm.eps));
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = mul2(f[i], both(rstd));
  if (norm.stats && active && s.t == 0) *reinterpret_cast<float2*>(norm.stats + 2LL * row) = make_float2(mean, rstd);
}
// n = (f - mean) * rstd with the statistics at hand, the difference first: f * rstd - mean * rstd takes an instruction less (a norm of
// 4882 x 4096 backward 44.5 us, 46.6), but is off by the rounding of mean * rstd, however small n is.  Not zero where there is no
// column, but whatever it meets there is.
template <int N>
__device__ __forceinline__ void normalised(float2 (&f)[N], float2 st) {
  const float2 r = both(st.y), m = both(-st.x);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = mul2(add2(f[i], m), r);
}
// Gradient of n * w + b by its input is rstd * (a - mean a - n mean(a n)), for a = dz * w: what stands in the brackets, in place.
// rstd comes last, so what cancels in there cancels before anything is rounded to rstd's steps.
__device__ __forceinline__ float2 norm_means(int kind, float inv_c, float2 v) {       // of sums of a and a n, both negative
  return make_float2(kind == NORM_LAYER ? v.x * -inv_c : 0.f, v.y * -inv_c);
}
template <bool WIDE, bool TILE, int N>
__device__ __forceinline__ void norm_gradient(Slot& s, int kind, float inv_c, float2 known, const float2 (&n)[N], float2 (&a)[N]) {
  const float2 m = TILE ? known : norm_means(kind, inv_c, slot_sum<WIDE>(make_float2(total(a), dot(a, n)), s));
  const float2 m0 = both(m.x), m1 = both(m.y);
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = fma2(n[i], m1, add2(a[i], m0));
}

// A gate's factor and its slope.  A sigmoid is kept as q = min(f, 1 - f), negative where that is 1 - f: its slope q (1 - q) has
// then all bits of q.  f (1 - f) lost those that 1 - f has not (84 steps of fp32 at a gate of 5).
__device__ __forceinline__ float sigmoid(float g) {
  const float e = expf(-fabsf(g));
  return copysignf(__fdividef(e, 1.f + e), -g);
}
__device__ __forceinline__ float factor_of(float q) { return __float_as_int(q) < 0 ? 1.f + q : q; }
template <int N>
__device__ __forceinline__ void gate_keep(int through_sigmoid, float2 (&g)[N]) {
  if (!through_sigmoid) return;
#pragma unroll
  for (int i = 0; i < N; ++i) g[i] = make_float2(sigmoid(g[i].x), sigmoid(g[i].y));
}
__device__ __forceinline__ float2 gate_factor(int through_sigmoid, float2 q) {
  return through_sigmoid ? make_float2(factor_of(q.x), factor_of(q.y)) : q;
}
__device__ __forceinline__ float2 gate_slope(int through_sigmoid, float2 q) {
  return through_sigmoid ? make_float2(fmaf(-q.x, q.x, fabsf(q.x)), fmaf(-q.y, q.y, fabsf(q.y))) : both(1.f);
}
template <int N>
__device__ __forceinline__ void gate_factor(int through_sigmoid, float2 (&g)[N]) {
  gate_keep(through_sigmoid, g);
#pragma unroll
  for (int i = 0; i < N; ++i) g[i] = gate_factor(through_sigmoid, g[i]);
}

// The rows of a slot: a range of its own with a gate per image, else every `step`-th of all.  Slots that share a warp take the
// same number of turns, since its lanes meet in sums: some have no row in the last.
struct Walk {
  int lo, hi, step, turns;
  __device__ __forceinline__ Walk(const GeepsResidual& p, int slots, int id, bool wide, bool ranges) {
    const int rows = (int)p.rows, all = gridDim.x * slots, me = blockIdx.x * slots + id;
    lo = ranges ? first_row(rows, all, me) : me;
    hi = ranges ? first_row(rows, all, me + 1) : rows;
    step = ranges ? 1 : all;
    turns = !wide ? (rows + all - 1) / all : lo < hi ? (hi - lo + step - 1) / step : 0;
  }
};

// WIDE: a slot is whole warps.  BIG: blocks of 512 threads; with LARGE the parameters leave no room for a ring.  PIXEL: a gate for
// every row.
template <typename TR, typename TB, int K, bool VEC, bool WIDE, bool LARGE, bool BIG, int MODE, bool PIXEL>
__global__ void __launch_bounds__(block_threads(false, VEC, LARGE, BIG, K, MODE), blocks_forward(LARGE, BIG, MODE))
residual_forward_kernel(const __grid_constant__ GeepsResidual p, int slot, int slots, int depth, int ring) {
  geeps_pdl_enter();
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ __align__(16) float red[16][64];
  constexpr int N = 4 * K, THREADS = block_threads(false, VEC, LARGE, BIG, K, MODE);
  typedef Columns<K, VEC, LARGE, THREADS> Cols;
  for (int i = threadIdx.x; i < 16 * 64; i += blockDim.x) red[0][i] = 0.f;
  Slot s;
  s.id = threadIdx.x / slot; s.t = threadIdx.x % slot; s.size = slot; s.red = red[WIDE ? s.id : 0]; s.turn = 0;
  const Cols cols = {s.t, slot, p.C, slots, !LARGE || (!BIG && depth > 0)};
  const float inv_c = 1.f / (float)p.C;
  const bool by_image = (MODE & MODE_JOIN) && !PIXEL && p.gate;
  const Walk w(p, slots, s.id, WIDE, by_image);
  const int per_gate = by_image ? (int)(p.rows / p.gate_rows) : 1;
  int image = 0, left = 0;                     // rows to go with the gate at hand

  const uint32_t base = (uint32_t)__cvta_generic_to_shared(shared + ring) + (VEC ? threadIdx.x * 16 : 0);
  const int at_x = cols.template stage<TR>(), at_g = at_x + (MODE & MODE_JOIN ? cols.template stage<TB>() : 0);
  const int one = at_g + (PIXEL ? cols.template stage<TB>() : 0), last = (depth - 1) * one;
  const Rows<TR> res(p.res, p.ldres, cols.first()), h_out(p.out, p.ldout, cols.first());
  const Rows<TB> x(p.x, p.ldx, cols.first()), gate(p.gate, p.ldgate, cols.first()), y_out(p.y, p.ldy, cols.first());
  // The row that is copied next and the stage that is read and then filled with it: a row's copies start when what lay there is
  // in registers, so a ring of one stage has a row on its way for most of a turn, too.
  int ahead = w.lo, now = 0;
  auto copy = [&]() {
    if (!cols.ring) return;
    if (!VEC) s.sync();
    if (ahead < w.hi) {
      const uint32_t to = base + now;
      cols.copy(res.at(ahead), to);
      if (MODE & MODE_JOIN) cols.copy(x.at(ahead), to + at_x);
      if (PIXEL) cols.copy(gate.at(ahead), to + at_g);
    }
    ahead += w.step;
    now = now == last ? 0 : now + one;
    copy_commit();
  };
  if (cols.ring) {
    for (int i = 0; i < depth; ++i) {
      const uint32_t to = base + i * one;
      cols.template no_copy<TR>(to, false);
      if (MODE & MODE_JOIN) cols.template no_copy<TB>(to + at_x, false);
      if (PIXEL) cols.template no_copy<TB>(to + at_g, false);
      copy();
    }
  }
  unsigned char* area = shared;
  Param<Cols, K, VEC, LARGE && !BIG> sw, sb, w2, b2;          // scale * weight and scale * bias of the join, weight and bias of the next norm
  Own<K, THREADS> factor;                      // the gate of the image at hand
  if (MODE & MODE_JOIN) { sw.set(cols, p.post.weight, 1.f, p.scale, area); sb.set(cols, p.post.bias, 0.f, p.scale, area); }
  if (MODE & MODE_NORM) { w2.set(cols, p.pre.weight, 1.f, nullptr, area); b2.set(cols, p.pre.bias, 0.f, nullptr, area); }
  if (by_image) factor.set(area);
  __syncthreads();
  for (int i = 0; i < w.turns; ++i) {
    const int row = w.lo + i * w.step;
    const bool active = WIDE || row < w.hi;
    if (cols.ring) {
      copy_wait(depth);
      if (!VEC) s.sync();
    }
    const uint32_t from = base + now;
    float2 h[N];
    if (MODE & MODE_JOIN) {
      float2 z[N];
      cols.load(x, row, active, true, from + at_x, z);
      if (by_image && left-- == 0 && active) {
        image = row / per_gate;
        left = (image + 1) * per_gate - row - 1;
        float2 g[N];
        cols.fetch(gate.at(image), true, g);
        gate_factor(p.sigmoid, g);
#pragma unroll
        for (int k = 0; k < K; ++k) factor.put(k, reinterpret_cast<float2(&)[4]>(g[4 * k]));
      }
      if (p.post.kind) normalise<WIDE>(cols, s, p.post, row, active, inv_c, z, [] {});
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 a[4], b[4];
        sw.get(cols, k, a); sb.get(cols, k, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[4 * k + e] = fma2(z[4 * k + e], a[e], b[e]);
      }
      if (by_image) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float2 g[4];
          factor.get(k, g);
#pragma unroll
          for (int e = 0; e < 4; ++e) z[4 * k + e] = mul2(z[4 * k + e], g[e]);
        }
      } else if (PIXEL) {
        float2 g[N];
        cols.load(gate, row, active, true, from + at_g, g);
        gate_factor(p.sigmoid, g);
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = mul2(z[j], g[j]);
      }
      cols.load(res, row, active, true, from, h);
#pragma unroll
      for (int j = 0; j < N; ++j) h[j] = add2(h[j], z[j]);
      copy();
      cols.store(h_out.at(row), active, h);
    } else {
      cols.load(res, row, active, true, from, h);
    }
    if (MODE & MODE_NORM) {
      normalise<WIDE>(cols, s, p.pre, row, active, inv_c, h, [&] { if (!(MODE & MODE_JOIN)) copy(); });
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 a[4], b[4];
        w2.get(cols, k, a); b2.get(cols, k, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[4 * k + e] = fma2(h[4 * k + e], a[e], b[e]);
      }
      cols.store(y_out.at(row), active, h);
    }
  }
}

// The workspace: sums of every block, [block][sums][C], A and B of the join, then dweight and dbias of the next norm; with a
// gate per image {A, B} of every slot's images, [slot][C][2], and a row of the gate's gradient for each (slot, image) pair that
// shares rows, number slot + image.
__host__ __device__ inline int sums_of(int mode) { return mode == MODE_BOTH ? 4 : 2; }
// How many slots have one share of an image that they alone have rows of: those of a warp, where every slot has rows (125552 x 32 as
// one image 91 us with a share a slot, 39 with one a warp; 160000 x 8 as four 91, 22)
__host__ __device__ __forceinline__ int merged_slots(long long rows, long long all, int slot) { return slot < 32 && rows >= all ? 32 / slot : 1; }
inline long long work_floats(const Shape& s, int C, int mode, long long images) {
  return ((long long)s.blocks * sums_of(mode) + (images ? 3LL * s.blocks * s.slots + images : 0)) * C;
}
__device__ __forceinline__ float* sums_of_images(const GeepsResidual& p, int mode, long long slot) {
  return p.work + ((long long)gridDim.x * sums_of(mode) + 2 * slot) * p.C;
}
__device__ __forceinline__ float* image_share(const GeepsResidual& p, int mode, int blocks, long long all, long long slot, int image) {
  return p.work + (blocks * sums_of(mode) + 2 * all + slot + image) * p.C;
}

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

// TILE: the operands are a range of the columns of wider rows, whose means a launch before this one has put into `means`, two pairs
// a row.
template <typename TR, typename TB, int K, bool VEC, bool WIDE, bool TILE, int MODE, bool PIXEL>
__global__ void __launch_bounds__(block_threads(true, VEC, false, false, K, MODE))
residual_backward_kernel(const __grid_constant__ GeepsResidual p, int slot, int slots, int depth, int ring, const float2* means) {
  geeps_pdl_enter();
  extern __shared__ __align__(16) unsigned char shared[];
  constexpr int N = 4 * K, THREADS = block_threads(true, VEC, false, false, K, MODE);
  typedef Columns<K, VEC, false, THREADS> Cols;
  __shared__ float2 stats[TILE ? 4 : 2][THREADS];      // and the means
  __shared__ __align__(16) float red[16][64];
  for (int i = threadIdx.x; i < 16 * 64; i += blockDim.x) red[0][i] = 0.f;
  Slot s;
  s.id = threadIdx.x / slot; s.t = threadIdx.x % slot; s.size = slot; s.red = red[WIDE ? s.id : 0]; s.turn = 0;
  stats[0][threadIdx.x] = stats[1][threadIdx.x] = both(0.f);
  const Cols cols = {s.t, slot, p.C, slots, true};
  const float inv_c = 1.f / (float)p.C;
  const bool by_image = (MODE & MODE_JOIN) && !PIXEL && p.gate;
  Param<Cols, K, VEC, false> sw, sb, w2;              // scale * weight, scale * bias (for a gate's gradient), the next norm's weight
  Own<K, THREADS> factor;                      // the gate of the image at hand
  float2 a0[N], a1[N], n0[N], n1[N];
#pragma unroll
  for (int i = 0; i < N; ++i) a0[i] = a1[i] = n0[i] = n1[i] = both(0.f);
  const Walk w(p, slots, s.id, WIDE, by_image);
  const int per_gate = by_image ? (int)(p.rows / p.gate_rows) : 1;
  int image = -1, left = 0;

  const uint32_t base = (uint32_t)__cvta_generic_to_shared(shared + ring) + (VEC ? threadIdx.x * 16 : 0);
  const int at_o = cols.template stage<TR>(), at_y = at_o + (MODE & MODE_NORM ? cols.template stage<TR>() : 0);
  const int at_x = at_y + (MODE & MODE_NORM ? cols.template stage<TB>() : 0);
  const int at_g = at_x + (MODE & MODE_JOIN ? cols.template stage<TB>() : 0);
  const int one = at_g + (PIXEL ? cols.template stage<TB>() : 0), last = (depth - 1) * one;
  const Rows<TR> dout(p.dout, p.lddout, cols.first()), h(p.out, p.ldout, cols.first()), dres(p.dres, p.lddres, cols.first());
  const Rows<TB> dy(p.dy, p.lddy, cols.first()), x(p.x, p.ldx, cols.first()), gate(p.gate, p.ldgate, cols.first());
  const Rows<TB> dx(p.dx, p.lddx, cols.first()), dgate(p.dgate, p.lddgate, cols.first());
  const bool has_dout = p.dout != nullptr;
  int ahead = w.lo, now = 0;                   // as in the forward pass, the branch's share of a row later than the rest
  auto copy_stream = [&]() {
    if (!VEC) s.sync();
    const uint32_t to = base + now;
    if (ahead < w.hi) {
      if (has_dout) cols.copy(dout.at(ahead), to);
      if (MODE & MODE_NORM) { cols.copy(h.at(ahead), to + at_o); cols.copy(dy.at(ahead), to + at_y); }
    } else if (!WIDE) {                        // rows that are read and are none: they add nothing to the sums
      cols.template no_copy<TR>(to, true);
      if (MODE & MODE_NORM) { cols.template no_copy<TR>(to + at_o, true); cols.template no_copy<TB>(to + at_y, true); }
    }
  };
  auto copy_branch = [&]() {
    if (!VEC && (MODE & MODE_JOIN)) s.sync();
    const uint32_t to = base + now;
    if (ahead < w.hi) {
      if (MODE & MODE_JOIN) cols.copy(x.at(ahead), to + at_x);
      if (PIXEL) cols.copy(gate.at(ahead), to + at_g);
    } else if (!WIDE) {
      if (MODE & MODE_JOIN) cols.template no_copy<TB>(to + at_x, true);
      if (PIXEL) cols.template no_copy<TB>(to + at_g, true);
    }
    ahead += w.step;
    now = now == last ? 0 : now + one;
    copy_commit();
  };
  // The rows of an image that this slot has are done: its part of the gate's gradient, all of it if no other slot has any.  With
  // a gate per image a0 and a1 are the sums u and v of the image at hand; A and B of the images before it are in the workspace,
  // every thread its own columns.
  float2* before = by_image ? reinterpret_cast<float2*>(sums_of_images(p, MODE, blockIdx.x * slots + s.id)) : nullptr;
  bool none_before = true, merge = false;
  if (!WIDE && by_image) {
    const int a = blockIdx.x * slots + s.id & -(32 / slot), all = gridDim.x * slots;
    merge = merged_slots(p.rows, all, slot) > 1 && first_row((int)p.rows, all, a) / per_gate == (first_row((int)p.rows, all, a + 32 / slot) - 1) / per_gate;
  }
  auto image_done = [&](bool end) {
    float2 d[N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 m[4], b[4], g[4];
      sw.get(cols, k, m); sb.get(cols, k, b); factor.get(k, g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * k + e;
        d[i] = mul2(fma2(m[e], a0[i], mul2(b[e], a1[i])), gate_slope(p.sigmoid, g[e]));
        g[e] = gate_factor(p.sigmoid, g[e]);
        float2 sum = mul2(g[e], a0[i]), sum1 = mul2(g[e], a1[i]);
        float2 *x = before + cols.at(2 * i), *y = before + cols.at(2 * i + 1);           // [column]{A, B}
        if (!none_before) {
          const float2 v = cols.on(2 * i) ? *x : both(0.f), u = cols.on(2 * i + 1) ? *y : both(0.f);
          sum = add2(sum, make_float2(v.x, u.x)); sum1 = add2(sum1, make_float2(v.y, u.y));
        }
        if (!end && cols.on(2 * i)) *x = make_float2(sum.x, sum1.x);
        if (!end && cols.on(2 * i + 1)) *y = make_float2(sum.y, sum1.y);
        a0[i] = end ? sum : both(0.f); a1[i] = end ? sum1 : both(0.f);
      }
    }
    none_before = false;
    if (!p.dgate) return;
    if (end && merge) {                        // the slots of this warp had rows of this image alone, in the end: one share
      for (int o = slot; o < 32; o <<= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) { d[i].x += __shfl_xor_sync(0xffffffffu, d[i].x, o); d[i].y += __shfl_xor_sync(0xffffffffu, d[i].y, o); }
      }
      if ((threadIdx.x & 31) >= slot) return;
    }
    if (image * per_gate >= w.lo && (image + 1) * per_gate <= w.hi) cols.store(dgate.at(image), true, d);
    else {
      float* to = image_share(p, MODE, gridDim.x, (long long)gridDim.x * slots, blockIdx.x * slots + s.id, image);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (cols.on(2 * i)) to[cols.at(2 * i)] = d[i].x;
        if (cols.on(2 * i + 1)) to[cols.at(2 * i + 1)] = d[i].y;
      }
    }
  };
  for (int i = 0; i < depth; ++i) {
    const uint32_t to = base + i * one;
    cols.template no_copy<TR>(to, !has_dout);
    if (MODE & MODE_NORM) { cols.template no_copy<TR>(to + at_o, false); cols.template no_copy<TB>(to + at_y, false); }
    if (MODE & MODE_JOIN) cols.template no_copy<TB>(to + at_x, false);
    if (PIXEL) cols.template no_copy<TB>(to + at_g, false);
    copy_stream();
    copy_branch();
  }
  unsigned char* area = shared;
  if (MODE & MODE_JOIN) {
    sw.set(cols, p.post.weight, 1.f, p.scale, area);
    if (p.gate) sb.set(cols, p.post.bias, 0.f, p.scale, area);
  }
  if (MODE & MODE_NORM) w2.set(cols, p.pre.weight, 1.f, nullptr, area);
  if (by_image) factor.set(area);
  __syncthreads();
  for (int i = 0; i < w.turns; ++i) {
    const int row = w.lo + i * w.step;
    const bool active = WIDE || row < w.hi;
    copy_wait(depth);
    if (!VEC) s.sync();
    const uint32_t from = base + now;
    // Statistics of the rows of several turns at a time, a row a lane: a load for every turn was waited for in the turn that
    // issued it, with the loads from shared memory that share its scoreboard (50176 x 576: 36 % of the time).
    const int chunk = WIDE ? 32 : slot, k0 = i & (chunk - 1);
    if (k0 == 0) {
      const int turn = i + (s.t & (chunk - 1)), q = w.lo + turn * w.step;
      __syncwarp();
      if (turn < w.turns && q < w.hi) {
        if ((MODE & MODE_JOIN) && p.post.kind) stats[0][threadIdx.x] = *reinterpret_cast<const float2*>(p.post.stats + 2LL * q);
        if (MODE & MODE_NORM) stats[1][threadIdx.x] = *reinterpret_cast<const float2*>(p.pre.stats + 2LL * q);
        if (TILE && (MODE & MODE_JOIN) && p.post.kind) stats[TILE ? 2 : 0][threadIdx.x] = means[2LL * q];
        if (TILE && (MODE & MODE_NORM)) stats[TILE ? 3 : 0][threadIdx.x] = means[2LL * q + 1];
      } else if (!WIDE) {          // a row that is none must not be normalised as one of an image before, which may not be finite
        stats[0][threadIdx.x] = stats[1][threadIdx.x] = both(0.f);
      }
      __syncwarp();
    }
    const int lane = (threadIdx.x & ~(chunk - 1)) + k0;
    const float2 st1 = stats[0][lane], st2 = stats[1][lane], known1 = stats[TILE ? 2 : 0][lane], known2 = stats[TILE ? 3 : 0][lane];
    float2 dh[N], z[N], g[N];
    auto load_branch = [&]() {
      if (MODE & MODE_JOIN) cols.load(x, row, active, true, from + at_x, z);
      if (PIXEL) { cols.load(gate, row, active, true, from + at_g, g); gate_keep(p.sigmoid, g); }
    };
    if (MODE & MODE_NORM) {
      float2 n[N], a[N];
      cols.load(h, row, active, true, from + at_o, n);
      cols.load(dy, row, active, true, from + at_y, a);
      normalised(n, st2);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 m[4];
        w2.get(cols, k, m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 4 * k + e;
          n0[j] = fma2(a[j], n[j], n0[j]); n1[j] = add2(n1[j], a[j]);
          a[j] = mul2(a[j], m[e]);
        }
      }
      norm_gradient<WIDE, TILE>(s, p.pre.kind, inv_c, known2, n, a);
      cols.load(dout, row, active, has_dout, from, dh);
#pragma unroll
      for (int j = 0; j < N; ++j) dh[j] = fma2(a[j], both(st2.y), dh[j]);
    } else {
      cols.load(dout, row, active, has_dout, from, dh);
    }
    if (MODE & MODE_NORM) copy_stream();       // what it overwrites has gone into sums that are there
    cols.store(dres.at(row), active, dh);
    if (MODE & MODE_JOIN) {
      load_branch();
      if (by_image && left == 0 && active) {
        if (image >= 0) image_done(false);
        image = row / per_gate;
        left = (image + 1) * per_gate - row;
        float2 f[N];
        cols.fetch(gate.at(image), true, f);
        gate_keep(p.sigmoid, f);
#pragma unroll
        for (int k = 0; k < K; ++k) factor.put(k, reinterpret_cast<float2(&)[4]>(f[4 * k]));
      }
      --left;
      if (p.post.kind) normalised(z, st1);
      float2 dg[N];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 m[4], f[4], b[4];
        sw.get(cols, k, m);
        if (PIXEL) sb.get(cols, k, b);
        if (by_image) factor.get(k, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 4 * k + e;
          float2 d = dh[j];
          if (PIXEL) {
            dg[j] = mul2(mul2(d, fma2(m[e], z[j], b[e])), gate_slope(p.sigmoid, g[j]));
            d = mul2(d, gate_factor(p.sigmoid, g[j]));
          }
          a0[j] = fma2(d, z[j], a0[j]); a1[j] = add2(a1[j], d);
          if (by_image) d = mul2(d, gate_factor(p.sigmoid, f[e]));
          dh[j] = mul2(d, m[e]);
        }
      }
      if (PIXEL && p.dgate) cols.store(dgate.at(row), active, dg);
      if (p.post.kind) {
        norm_gradient<WIDE, TILE>(s, p.post.kind, inv_c, known1, z, dh);
#pragma unroll
        for (int j = 0; j < N; ++j) dh[j] = mul2(dh[j], both(st1.y));
      }
      if (!(MODE & MODE_NORM)) copy_stream();
      copy_branch();
      cols.store(dx.at(row), active, dh);
    } else copy_branch();
  }
  if (by_image && image >= 0) image_done(true);      // and a0, a1 are A and B
  // the slots' sums, in slot order, in the threads of slot 0
  __syncthreads();
  float2* meet = reinterpret_cast<float2*>(shared);
  auto over_slots = [&](float2 (&v)[N]) {
    if (slots == 1) return;
    int shares = slots, share = s.id;
    if (!WIDE) {                       // slots of a warp first
      for (int o = slot; o < 32; o <<= 1) {
#pragma unroll
        for (int j = 0; j < N; ++j) { v[j].x += __shfl_xor_sync(0xffffffffu, v[j].x, o); v[j].y += __shfl_xor_sync(0xffffffffu, v[j].y, o); }
      }
      shares = blockDim.x >> 5; share = threadIdx.x >> 5;
    }
    if (WIDE || (threadIdx.x & 31) < slot) {
#pragma unroll
      for (int j = 0; j < N; ++j) meet[(share * N + j) * slot + s.t] = v[j];
    }
    __syncthreads();
    if (s.id == 0) {
      for (int i = 1; i < shares; ++i) {
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

template <int W>
__device__ __forceinline__ void four(float4 v, float (&f)[W], int e) {
  if (W >= 4) { f[e] = v.x; f[(e + 1) % W] = v.y; f[(e + 2) % W] = v.z; f[(e + 3) % W] = v.w; }
}
// W columns of a row from where they lie
template <int W, typename T>
__device__ __forceinline__ void columns(const T* p, float (&f)[W]) {
  if (W == 1) {
    f[0] = (float)*p;
  } else if (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < W; e += 4) four(ld_f4((const float*)p + e), f, e);
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < W; ++e) f[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
}
// The means of rows that are worked on in tiles: for each norm {-mean a, -mean (a n)}, what norm_gradient() adds.  A block
// reads a row twice, the second time from L2: the join's sums are of the gradient that the next norm's means are part of.
constexpr int kMeansThreads = 256;
template <typename TR, typename TB, bool VEC, int MODE, bool PIXEL>
__global__ void __launch_bounds__(kMeansThreads, 4)
residual_means_kernel(const __grid_constant__ GeepsResidual p, float2* means) {
  geeps_pdl_enter();
  constexpr int W = VEC ? kVec : 1, WARPS = kMeansThreads / 32;
  __shared__ float2 sh[2][WARPS];
  const float inv_c = 1.f / (float)p.C;
  const int rows = (int)p.rows, per_gate = p.gate ? (int)(p.rows / p.gate_rows) : 1;
  int turn = 0;
  auto block_sum = [&](float2 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) { v.x += __shfl_xor_sync(0xffffffffu, v.x, o); v.y += __shfl_xor_sync(0xffffffffu, v.y, o); }
    if ((threadIdx.x & 31) == 0) sh[turn][threadIdx.x >> 5] = v;
    __syncthreads();
    v = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { v.x += sh[turn][w].x; v.y += sh[turn][w].y; }
    turn ^= 1;
    return v;
  };
  const bool wide = (((uintptr_t)p.pre.weight | (uintptr_t)p.post.weight | (uintptr_t)p.scale) & 15) == 0;
  auto param = [&](const float* from, int c, float (&v)[W]) {
    if (!from) {
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = 1.f;
    } else if (VEC && wide) {
#pragma unroll
      for (int e = 0; e < W; e += 4) four(ld_f4(from + c + e), v, e);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = from[c + e];
    }
  };
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const TR *h = (const TR*)p.out + row * p.ldout, *dout = (const TR*)p.dout + row * p.lddout;
    const TB *dy = (const TB*)p.dy + row * p.lddy, *x = (const TB*)p.x + row * p.ldx, *gate = (const TB*)p.gate + row / per_gate * p.ldgate;
    float2 st1 = both(0.f), st2 = both(0.f), known = both(0.f);
    if ((MODE & MODE_JOIN) && p.post.kind) st1 = *reinterpret_cast<const float2*>(p.post.stats + 2LL * row);
    if (MODE & MODE_NORM) {
      st2 = *reinterpret_cast<const float2*>(p.pre.stats + 2LL * row);
      float2 v = both(0.f);
#pragma unroll 2
      for (int c = threadIdx.x * W; c < p.C; c += kMeansThreads * W) {
        float n[W], a[W], w[W];
        columns<W>(h + c, n); columns<W>(dy + c, a); param(p.pre.weight, c, w);
#pragma unroll
        for (int e = 0; e < W; ++e) { a[e] *= w[e]; v.x += a[e]; v.y = fmaf(a[e], (n[e] - st2.x) * st2.y, v.y); }
      }
      known = norm_means(p.pre.kind, inv_c, block_sum(v));
      if (threadIdx.x == 0) means[2LL * row + 1] = known;
    }
    if ((MODE & MODE_JOIN) && p.post.kind) {
      float2 v = both(0.f);
#pragma unroll 2
      for (int c = threadIdx.x * W; c < p.C; c += kMeansThreads * W) {
        float d[W], z[W], w[W], f[W];
        columns<W>(x + c, z);
        if (p.dout) columns<W>(dout + c, d);
        else {
#pragma unroll
          for (int e = 0; e < W; ++e) d[e] = 0.f;
        }
        if (MODE & MODE_NORM) {
          float n[W], a[W];
          columns<W>(h + c, n); columns<W>(dy + c, a); param(p.pre.weight, c, w);
#pragma unroll
          for (int e = 0; e < W; ++e) d[e] = fmaf(fmaf((n[e] - st2.x) * st2.y, known.y, a[e] * w[e] + known.x), st2.y, d[e]);
        }
        param(p.post.weight, c, w); param(p.scale, c, f);
#pragma unroll
        for (int e = 0; e < W; ++e) d[e] *= w[e] * f[e];
        if (p.gate) {
          columns<W>(gate + c, f);
#pragma unroll
          for (int e = 0; e < W; ++e) d[e] *= p.sigmoid ? factor_of(sigmoid(f[e])) : f[e];
        }
#pragma unroll
        for (int e = 0; e < W; ++e) { v.x += d[e]; v.y = fmaf(d[e], (z[e] - st1.x) * st1.y, v.y); }
      }
      v = block_sum(v);
      if (threadIdx.x == 0) means[2LL * row] = norm_means(p.post.kind, inv_c, v);
    }
  }
}

// The slot whose rows have row i
__device__ __forceinline__ int slot_of(int rows, int slots, int i) {
  const int base = rows / slots, longer = rows % slots, split = longer * (base + 1);
  return i < split ? i / (base + 1) : longer + (i - split) / base;
}
// Second launch: the blocks' sums, and the gate's gradient of the images whose rows several slots had, each in the order of the
// blocks or slots.  A block has 32 columns at the most and 32 shares: blockIdx.y 0 to 3 a quarter of the columns each and every
// 32nd block's sums a share; then 32 / `parts` images, or, where there are more images than slots, slots that begin inside of
// one and are its first cut.
constexpr int kSumsThreads = 256;
template <typename TB, bool MERGED>
__global__ void __launch_bounds__(kSumsThreads)
residual_sums_kernel(const __grid_constant__ GeepsResidual p, int mode, int blocks, int slots, int parts, int merged) {
  geeps_pdl_enter();
  __shared__ float sh[32][4][8];
  const int lane = threadIdx.x & 7, share = threadIdx.x >> 3, sums = sums_of(mode);
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (blockIdx.y < 4) {
    const int c = blockIdx.x * 32 + blockIdx.y * 8 + lane;
    if (blocks == 1 || c - lane >= p.C) return;
    if (c < p.C) {
#pragma unroll 5
      for (int b = share; b < blocks; b += 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < sums) v[i] += p.work[((long long)b * sums + i) * p.C + c];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] += __shfl_xor_sync(0xffffffffu, v[i], 8);
      v[i] += __shfl_xor_sync(0xffffffffu, v[i], 16);
      if ((threadIdx.x & 24) == 0) sh[threadIdx.x >> 5][i][lane] = v[i];
    }
    __syncthreads();
    if (share != 0 || c >= p.C) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v[i] += sh[w][i][lane];
    }
    write_sums(p, mode, c, v);
    return;
  }
  const int rows = (int)p.rows, images = (int)p.gate_rows, per_gate = rows / images, all = blocks * slots;
  const int item = (blockIdx.y - 4) * (32 / parts) + share / parts, part = share % parts;
  int image = item, first = 0, end = 0;               // slots [first, end) have rows of the image
  if (images <= all) {
    if (item < images) {
      first = slot_of(rows, all, item * per_gate);
      end = slot_of(rows, all, (item + 1) * per_gate - 1) + 1;
    }
  } else if (item + 1 < all && first_row(rows, all, item + 1) < rows) {
    const int cut = first_row(rows, all, item + 1), start = cut / per_gate * per_gate;
    image = cut / per_gate;
    if (cut != start && first_row(rows, all, item) <= start) {
      first = item;
      end = slot_of(rows, all, start + per_gate - 1) + 1;
    }
  }
  if (end - first < 2) end = first;                   // one slot had it all
  auto add = [&](int q, int until, int step) {
#pragma unroll 4
    for (q += part * step; q < until; q += parts * step) {
      const float* w = image_share(p, mode, blocks, all, q, image);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = blockIdx.x * 32 + u * 8 + lane;
        if (c < p.C) v[u] += w[c];
      }
    }
  };
  if (!MERGED) {
    add(first, end, 1);
  } else if (end > first) {                  // warps [from, to) have the image alone: one share of each, before and behind them one a slot
    int from = (first + merged - 1) / merged, to = end / merged;
    if (from * merged < all && first_row(rows, all, from * merged) < image * per_gate) ++from;
    if (first_row(rows, all, to * merged) > (image + 1) * per_gate) --to;
    if (to < from) from = to = (end + merged - 1) / merged;
    const int head = min(from * merged, end);
    add(first, head, 1);
    add(from * merged, to * merged, merged);
    add(max(to * merged, head), end, 1);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) sh[share][u][lane] = v[u];
  __syncthreads();
  if (part != 0 || end == first) return;
  for (int u = 0; u < 4; ++u) {
    const int c = blockIdx.x * 32 + u * 8 + lane;
    float t = 0.f;
    for (int q = 0; q < parts; ++q) t += sh[share + q][u][lane];
    if (c < p.C) ((TB*)p.dgate)[image * p.lddgate + c] = (TB)t;
  }
}

// ---- launches ----
// done: one a kernel
template <typename F>
void allow_shared(F kernel, size_t bytes, bool (&done)[64]) {
  if (bytes <= 24 * 1024) return;             // the default limit, 48 KB, less what the kernels have statically
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 && done[dev]) return;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024) == cudaSuccess && dev >= 0 && dev < 64)
    done[dev] = true;
}

template <typename TR, typename TB, int K, bool VEC, bool WIDE, bool LARGE, bool BIG, int MODE, bool PIXEL>
void launch_forward(const GeepsResidual& p, const Shape& s, cudaStream_t st) {
  static bool done[64] = {false};
  const auto kernel = residual_forward_kernel<TR, TB, K, VEC, WIDE, LARGE, BIG, MODE, PIXEL>;
  allow_shared(kernel, s.smem, done);
  geeps_launch(kernel, dim3(s.blocks), dim3(s.threads()), s.smem, st, p, s.slot, s.slots, s.depth, (int)s.ring);
}
template <typename TR, typename TB, int K, bool VEC, bool WIDE, bool TILE, int MODE, bool PIXEL>
void launch_backward(const GeepsResidual& p, const Shape& s, const float2* means, cudaStream_t st) {
  static bool done[64] = {false};
  const size_t meet = s.slots > 1 ? (size_t)s.threads() * 8 * K * sizeof(float) : 0, smem = s.smem < meet ? meet : s.smem;
  const auto kernel = residual_backward_kernel<TR, TB, K, VEC, WIDE, TILE, MODE, PIXEL>;
  allow_shared(kernel, smem, done);
  geeps_launch(kernel, dim3(s.blocks), dim3(s.threads()), smem, st, p, s.slot, s.slots, s.depth, (int)s.ring, means);
}
// ... false: there is no such kernel
template <typename TR, typename TB, int K, bool VEC, bool WIDE, int MODE, bool PIXEL>
bool launch_kernel(const GeepsResidual& p, const Shape& s, bool backward, cudaStream_t st) {
  constexpr int B = sizeof(TB);
  if (backward) {
    if constexpr (planned(true, VEC, WIDE, false, K, MODE, PIXEL, B)) {
      launch_backward<TR, TB, K, VEC, WIDE, false, MODE, PIXEL>(p, s, nullptr, st);
      return true;
    }
  } else if (s.wide) {
    if constexpr (K == 4 && WIDE && planned(false, VEC, WIDE, true, K, MODE, PIXEL, B)) {
      launch_forward<TR, TB, K, VEC, WIDE, false, true, MODE, PIXEL>(p, s, st);
      return true;
    }
  } else {
    if constexpr (planned(false, VEC, WIDE, false, K, MODE, PIXEL, B)) {
      launch_forward<TR, TB, K, VEC, WIDE, false, false, MODE, PIXEL>(p, s, st);
      return true;
    }
  }
  return false;
}
template <typename TR, typename TB, int MODE, bool PIXEL>
bool launch(const GeepsResidual& p, const Shape& s, bool backward, bool vec, cudaStream_t st) {
  const bool wide = s.slot >= 32;
  if (!vec) {
    if constexpr (MODE == MODE_BOTH) {         // the others' two parameters always fit
      if (s.large) { launch_forward<TR, TB, 4, false, true, true, false, MODE, PIXEL>(p, s, st); return true; }
    }
    if constexpr (MODE != MODE_NORM) {
      if (s.wide && s.depth == 0) { launch_forward<TR, TB, 4, false, true, true, true, MODE, PIXEL>(p, s, st); return true; }
    }
    if (s.wide) return launch_kernel<TR, TB, 4, false, true, MODE, PIXEL>(p, s, backward, st);
    if (s.vectors == 2) return launch_kernel<TR, TB, 2, false, true, MODE, PIXEL>(p, s, backward, st);
    if (wide) return launch_kernel<TR, TB, 1, false, true, MODE, PIXEL>(p, s, backward, st);
    return launch_kernel<TR, TB, 1, false, false, MODE, PIXEL>(p, s, backward, st);
  }
  if constexpr (MODE != MODE_NORM) {
    if (s.large) { launch_forward<TR, TB, 4, true, true, true, false, MODE, PIXEL>(p, s, st); return true; }
  }
  if (s.vectors == 1) return launch_kernel<TR, TB, 1, true, false, MODE, PIXEL>(p, s, backward, st);
  if (s.vectors == 2 && wide) return launch_kernel<TR, TB, 2, true, true, MODE, PIXEL>(p, s, backward, st);
  if (s.vectors == 2) return launch_kernel<TR, TB, 2, true, false, MODE, PIXEL>(p, s, backward, st);
  if (s.vectors == 3 && wide) return launch_kernel<TR, TB, 3, true, true, MODE, PIXEL>(p, s, backward, st);
  if (s.vectors == 3) return launch_kernel<TR, TB, 3, true, false, MODE, PIXEL>(p, s, backward, st);
  if (wide) return launch_kernel<TR, TB, 4, true, true, MODE, PIXEL>(p, s, backward, st);
  return launch_kernel<TR, TB, 4, true, false, MODE, PIXEL>(p, s, backward, st);
}
inline Call call_of(const GeepsResidual& p, bool backward, bool vec) {
  const bool by_pixel = p.gate && p.gate_rows == p.rows;
  return {backward, vec, by_pixel, p.gate && !by_pixel, false, p.mode, p.stream_fp32 ? 4 : 2, p.block_fp32 ? 4 : 2};
}
// The second launch of a backward pass, where blocks or slots share sums: x = 0 if there is none
struct SumsShape { int x, y, parts, merged; };
inline SumsShape plan_sums(long long rows, long long images, int C, bool cuts, const Shape& s) {
  if (s.blocks == 1 && !(cuts && s.slots > 1)) return {0, 0, 1, 1};
  SumsShape q = {(C + 31) / 32, 4, 1, 1};
  if (cuts) {
    q.merged = merged_slots(rows, (long long)s.blocks * s.slots, s.slot);
    // Shares that an image has: one of each slot, or of each warp between those of its first and its last slots.  With no more
    // parts than that y stays below 6 / 32 of the slots, 76000 of which are the most: a grid has 65535 blocks along y (with parts for
    // the merged shares alone 70000 images of two pixels and 4 channels took 70004).
    const long long all = (long long)s.blocks * s.slots, by_slot = all / images + 2, by_warp = all / q.merged / images + 2 * q.merged;
    while (q.parts < 32 && q.parts < by_slot && q.parts < by_warp) q.parts <<= 1;
    const long long items = images <= all ? images : all - 1;
    q.y += (int)((items + 32 / q.parts - 1) / (32 / q.parts));
  }
  return q;
}
template <typename TB>
void join_sums(const GeepsResidual& p, const Shape& s, cudaStream_t st) {
  const SumsShape q = plan_sums(p.rows, p.gate_rows, p.C, p.gate && p.gate_rows < p.rows && p.dgate, s);
  if (!q.x) return;
  geeps_launch(q.merged > 1 ? residual_sums_kernel<TB, true> : residual_sums_kernel<TB, false>, dim3(q.x, q.y), dim3(kSumsThreads), 0, st, p, p.mode,
               s.blocks, s.slots, q.parts, q.merged);
}
// columns [c, c + width) of the operands
template <typename TR, typename TB>
GeepsResidual columns_of(const GeepsResidual& p, int c, int width) {
  GeepsResidual q = p;
  auto move = [&](auto& at, size_t size) { if (at) at = (std::remove_reference_t<decltype(at)>)((uintptr_t)at + c * size); };
  move(q.x, sizeof(TB)); move(q.gate, sizeof(TB)); move(q.dy, sizeof(TB)); move(q.dx, sizeof(TB)); move(q.dgate, sizeof(TB));
  move(q.out, sizeof(TR)); move(q.dout, sizeof(TR)); move(q.dres, sizeof(TR));
  move(q.scale, 4); move(q.dscale, 4);
  for (GeepsNorm* n : {&q.post, &q.pre}) { move(n->weight, 4); move(n->bias, 4); move(n->dweight, 4); move(n->dbias, 4); }
  q.C = p.C - c < width ? p.C - c : width;
  return q;
}
template <typename TR, typename TB, int MODE, bool PIXEL>
void run_tiles(const GeepsResidual& p, const Shape& s, Call c, cudaStream_t st) {
  float2* means = reinterpret_cast<float2*>(p.work);
  const int room = geeps_sm_count() * 4, grid = p.rows < room ? (int)p.rows : room;
  if ((MODE & MODE_NORM) || p.post.kind) {
    if (c.vec) geeps_launch(residual_means_kernel<TR, TB, true, MODE, PIXEL>, dim3(grid), dim3(kMeansThreads), 0, st, p, means);
    else geeps_launch(residual_means_kernel<TR, TB, false, MODE, PIXEL>, dim3(grid), dim3(kMeansThreads), 0, st, p, means);
  }
  c.tile = true;
  for (int i = 0; i < s.tiles; ++i) {
    GeepsResidual q = columns_of<TR, TB>(p, i * s.width, s.width);
    q.work = p.work + 4 * p.rows;
    const Shape t = plan(p.rows, q.C, c);
    if (c.vec) launch_backward<TR, TB, 2, true, true, true, MODE, PIXEL>(q, t, means, st);
    else launch_backward<TR, TB, 1, false, true, true, MODE, PIXEL>(q, t, means, st);
    join_sums<TB>(q, t, st);
  }
}
template <typename TR, typename TB, int MODE, bool PIXEL>
bool run_mode(const GeepsResidual& p, const Call& c, cudaStream_t st) {
  const Shape s = plan(p.rows, p.C, c);
  if (s.tiles > 1) { run_tiles<TR, TB, MODE, PIXEL>(p, s, c, st); return true; }
  if (!launch<TR, TB, MODE, PIXEL>(p, s, c.backward, c.vec, st)) return false;
  if (c.backward) join_sums<TB>(p, s, st);
  return true;
}
template <typename TR, typename TB>
bool run(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st) {
  const Call c = call_of(p, backward, vec);
  if (p.mode == MODE_NORM) return run_mode<TR, TB, MODE_NORM, false>(p, c, st);
  if (p.mode == MODE_JOIN) return c.by_pixel ? run_mode<TR, TB, MODE_JOIN, true>(p, c, st) : run_mode<TR, TB, MODE_JOIN, false>(p, c, st);
  return c.by_pixel ? run_mode<TR, TB, MODE_BOTH, true>(p, c, st) : run_mode<TR, TB, MODE_BOTH, false>(p, c, st);
}

bool run_bf16(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st);
bool run_mixed(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st);
bool run_fp32(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st);

}  // namespace rownorm
