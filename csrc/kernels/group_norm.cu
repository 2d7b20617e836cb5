// Group norm with its activation, channels last: statistics of the pixels x channels of a group of an image.
//
//   z = ((x - mean) rstd) w + b,  y = act(z)                     act: none, ReLU, SiLU
//   dz = dy act'(z);  db = sum dz;  dw = sum dz n;  dx = rstd (dz w - mean_g(dz w) - n mean_g(dz w n)),  n = (x - mean) rstd
//
// No counterpart in the reference, whose (absent) Caffe application normalised over batches.
//
// An item is an image and a slice of its channels, whole groups and whole vectors of eight.  The CTAs of a cluster share an item's
// pixels.  A thread owns the eight channels of a vector in every R-th pixel of its CTA: its sums need no other thread until the
// end, and what it reads it keeps in shared memory of its own (asynchronous copies, no barrier) for the second pass, so an item is
// read from memory once.  The CTAs' sums meet over distributed shared memory in the order of their ranks.  Images that are too few
// for the machine as items are cut over many CTAs in two launches (sums, then the rest), which meet in a workspace.
// Forward reads x and writes y, backward reads x and dy and writes dx.  A block's life is a chain of waits (its pixels, the column sums,
// the group sums, the stores: some 6 us; nothing is loaded while it sums), of which as many run side by side as shared memory holds slices: 0.45 to 0.55 of the copy
// rate (32 x 3136 x 192 forward 26 us, 256 x 196 x 576 backward 52.6).  Neither taking turns at the start (55 to 57 of 56 at the time), nor
// four groups of copies with sums between them, nor reading again from L2 instead of keeping (121) does better.
//
// Variance: values less the first of every 32 of a thread's pixels are added and squared, and such parts meet as count, mean and
// sum of squared differences, so a mean far from zero costs nothing.  A first value far from the others does: squares about it are at most
// 32 times those about a part's mean, which leaves 1/std up to 1e-5 off (of 64-bit arithmetic; 2e-7 otherwise).
// The backward pass, and with a ReLU the forward pass, form z in the four rounded operations above, so that the border of the ReLU is one and
// does not depend on how it is compiled (forward by a subtraction and a fused operation 32 x 3136 x 192 26.0 us, so 26.2; 37 x 113 x 1003 15.4, 15.8).
#include <math.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "nn_ops.h"
#include "tc05.cuh"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int kMostParts = 256;            // chunks of an image in two launches
constexpr int kMostChannels = 16384;       // for which a slice of a single group fits in shared memory, both ways
constexpr int kPart = 32;                  // pixels of a part of the variance
// One launch with the pixels kept in shared memory, or read again; or two launches; or kept, the first of a thread in registers
enum Phase { KEPT = 0, TWICE = 1, SUMS = 2, APPLY = 3, MIXED = 4 };
// Backward, bf16: pixels of a thread in registers, where that lets another block onto an SM (256 x 196 x 576 56.4 -> 52.6 us, 64 x 196 x 1024
// 29.1 -> 24.9).  Four spill (112 bytes, three 64).
constexpr int kInRegisters = 3;
// Threads of a block.  Where a slice's pixels stay in the block, 128: more blocks then share an SM, each in another step.  With 256, us,
// bf16: 512 x 64 x 96 forward 7.1 -> 11.4, 256 x 196 x 576 backward 56.5 -> 75.8, 8 x 12544 x 128 18.2 -> 31.1; only some forward passes of
// many channels gain (256 x 196 x 576 35.2 -> 31.2).
constexpr int threads_of(int phase) { return phase == SUMS || phase == APPLY ? 256 : 128; }

// n / d for n below 2^31 by a multiplication (Granlund and Montgomery)
struct Divide {
  unsigned m, s;
  int d;
  Divide() = default;
  explicit Divide(int by) : s(0), d(by) {
    while ((1ull << s) < (unsigned)by) ++s;
    m = (unsigned)(((1ull << 32) * ((1ull << s) - (unsigned)by)) / (unsigned)by + 1);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(m, (unsigned)n) + (unsigned)n) >> s); }
};

struct Dev {
  const void *x, *dy;
  void* out;                               // y or dx
  const float *w, *b;
  float *stats, *sums;                     // sums: workspace
  long long ldx, lddy, ldo;
  int pixels, C, groups, slice, slices, rows, act, keep, V, R, entries;    // rows: pixels of a chunk; keep: pixels a thread keeps
  Divide by_chunks, by_slices, by_V, by_cg;                               // by_V: of a thread's number, or one that gives 0
  float eps, one;                          // one: 1
};

// ---- pairs of fp32 ----
__device__ __forceinline__ unsigned long long word(float2 a) { return reinterpret_cast<unsigned long long&>(a); }
__device__ __forceinline__ float2 pair(unsigned long long a) { return reinterpret_cast<float2&>(a); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(word(a)), "l"(word(b)));
  return pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(word(a)), "l"(word(b)));
  return pair(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(word(a)), "l"(word(b)), "l"(word(c)));
  return pair(r);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// ---- vectors of eight (or single) values, as pairs ----
template <typename T, int W>
struct Vec;
template <>
struct Vec<bf16, 8> {
  uint4 a;
  __device__ __forceinline__ void load(const bf16* p) { a = *(const uint4*)p; }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  __device__ __forceinline__ void set(const float2 (&f)[4]) {
    a = make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y), pack_bf16x2(f[3].x, f[3].y));
  }
  __device__ __forceinline__ void store(bf16* p) const { *(uint4*)p = a; }
  __device__ __forceinline__ void relu() {           // a NaN stays one
    __nv_bfloat162* h = (__nv_bfloat162*)&a;
    const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], zero);
  }
  __device__ __forceinline__ void mask(const float2 (&z)[4]) {      // zero where z is not above zero
    uint32_t* w = (uint32_t*)&a;
    const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= __hgt2_mask(__floats2bfloat162_rn(z[i].x, z[i].y), zero);
  }
};
template <>
struct Vec<float, 8> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = ld_f4(p); b = ld_f4(p + 4); }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    f[0] = make_float2(a.x, a.y); f[1] = make_float2(a.z, a.w); f[2] = make_float2(b.x, b.y); f[3] = make_float2(b.z, b.w);
  }
  __device__ __forceinline__ void set(const float2 (&f)[4]) { a = make_float4(f[0].x, f[0].y, f[1].x, f[1].y); b = make_float4(f[2].x, f[2].y, f[3].x, f[3].y); }
  __device__ __forceinline__ void store(float* p) const { st_f4(p, a); st_f4(p + 4, b); }
  __device__ __forceinline__ void relu() {
    float* f = (float*)this;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = f[i] < 0.f ? 0.f : f[i];
  }
  __device__ __forceinline__ void mask(const float2 (&z)[4]) {
    float2* f = (float2*)this;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(z[i].x > 0.f ? f[i].x : 0.f, z[i].y > 0.f ? f[i].y : 0.f);
  }
};
template <>
struct Vec<bf16, 1> {
  bf16 a;
  __device__ __forceinline__ void load(const bf16* p) { a = *p; }
  __device__ __forceinline__ void get(float2 (&f)[1]) const { f[0] = make_float2(__bfloat162float(a), 0.f); }
  __device__ __forceinline__ void set(const float2 (&f)[1]) { a = __float2bfloat16(f[0].x); }
  __device__ __forceinline__ void store(bf16* p) const { *p = a; }
  __device__ __forceinline__ void relu() { a = __hmax_nan(a, __float2bfloat16(0.f)); }
  __device__ __forceinline__ void mask(const float2 (&z)[1]) { if (!(z[0].x > 0.f)) a = __float2bfloat16(0.f); }
};
template <>
struct Vec<float, 1> {
  float a;
  __device__ __forceinline__ void load(const float* p) { a = *p; }
  __device__ __forceinline__ void get(float2 (&f)[1]) const { f[0] = make_float2(a, 0.f); }
  __device__ __forceinline__ void set(const float2 (&f)[1]) { a = f[0].x; }
  __device__ __forceinline__ void store(float* p) const { *p = a; }
  __device__ __forceinline__ void relu() { a = a < 0.f ? 0.f : a; }
  __device__ __forceinline__ void mask(const float2 (&z)[1]) { if (!(z[0].x > 0.f)) a = 0.f; }
};
template <int W>
__device__ __forceinline__ float& value(float2 (&f)[(W + 1) / 2], int i) { return i & 1 ? f[i >> 1].y : f[i >> 1].x; }

// W values of the channels of column v
template <int W>
__device__ __forceinline__ void channel_values(const float* of, int v, float2 (&f)[(W + 1) / 2]) {
  if constexpr (W == 8) {
    const float4 a = ((const float4*)of)[2 * v], b = ((const float4*)of)[2 * v + 1];
    f[0] = make_float2(a.x, a.y); f[1] = make_float2(a.z, a.w); f[2] = make_float2(b.x, b.y); f[3] = make_float2(b.z, b.w);
  } else {
    f[0] = both(of[v]);
  }
}

__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A thread's own rows of vectors in shared memory, 16 bytes of every thread side by side.  By addresses of the shared window: through
// pointers that lambdas carry the accesses are generic ones
template <typename T>
struct Kept {
  static constexpr int kThreads = threads_of(KEPT);
  uint32_t base;                                            // of this thread
  static constexpr int kPieces = (int)sizeof(T) / 2;        // of 16 bytes
  static constexpr int kBytes = kThreads * 16 * kPieces;    // of a row
  __device__ __forceinline__ void fetch(int k, const T* src) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) copy_async(base + k * kBytes + i * kThreads * 16, (const uint8_t*)src + 16 * i);
  }
  __device__ __forceinline__ Vec<T, 8> get(int k) const {
    Vec<T, 8> v;
    uint32_t* w = (uint32_t*)&v;
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3]) : "r"(base + k * kBytes + i * kThreads * 16));
    return v;
  }
  __device__ __forceinline__ void put(int k, const Vec<T, 8>& v) const {
    const uint32_t* w = (const uint32_t*)&v;
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                   ::"r"(base + k * kBytes + i * kThreads * 16), "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3]) : "memory");
  }
};
// Rows of a column as a thread reads them: from its own shared memory or where they lie
template <typename T, int W, bool KEEP>
struct Rows {
  const T* at;
  long long step;
  Kept<T> kept;
  __device__ __forceinline__ Vec<T, W> get(int k) const {
    if constexpr (KEEP) {
      return kept.get(k);
    } else {
      Vec<T, W> v;
      v.load(at + k * step);
      return v;
    }
  }
};

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// What a CTA works on and which part of it a thread has
template <int W>
struct Place {
  int image, slice, chunk, rows, c0, v, r, most, extra;        // rows: pixels of the chunk; c0: channel of the slice
  long long pixel;                                             // of the chunk, among all images
  bool works;
  __device__ __forceinline__ Place(const Dev& d) {
    int i = d.by_chunks((int)blockIdx.x);
    chunk = (int)blockIdx.x - i * d.by_chunks.d;
    image = d.by_slices(i);
    slice = i - image * d.slices;
    const int first = chunk * d.rows;
    rows = max(0, min(d.rows, d.pixels - first));
    c0 = slice * d.slice;
    r = d.by_V((int)threadIdx.x);
    v = (int)threadIdx.x - r * d.V;
    works = r < d.R;
    pixel = (long long)image * d.pixels + first;
    most = rows / d.R;
    extra = rows - most * d.R;
  }
  // rows of this thread
  __device__ __forceinline__ int mine() const { return works ? most + (r < extra ? 1 : 0) : 0; }
};

// Sum over `lanes` neighbouring lanes (a power of two), in all of them
__device__ __forceinline__ float lane_sum(float a, int lanes) {
  for (int o = lanes >> 1; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  return a;
}
// Power of two from n up, at most 32
__device__ __forceinline__ int lanes_for(int n) { return n >= 32 ? 32 : n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }
// f(g, lane of the group, whether there is such a group) for every group of the slice, `lanes` lanes of a warp a group; lanes
// without a group get the last one
template <int kThreads, typename F>
__device__ __forceinline__ void each_group(int gs, int lanes, F f) {
  const int at = threadIdx.x & (lanes - 1), per = kThreads / lanes;
  for (int g0 = 0; g0 < gs; g0 += per) {
    const int g = g0 + (int)threadIdx.x / lanes;
    if (g0 + ((int)threadIdx.x & ~31) / lanes < gs) f(min(g, gs - 1), at, g < gs);
  }
}

// finish(c, sum over the R threads of channel c of entry[i][r][v], the first of those), c = W v + i, by one thread a channel.
// Every thread of the block calls it; no barrier behind it.
template <int kThreads, int W, typename F>
__device__ __forceinline__ void column_sums(const Dev& d, float2* entry, F finish) {
  __syncthreads();
  const int all = d.R * d.V;
  for (int i = threadIdx.x; i < d.slice; i += kThreads) {
    // threads go through a vector's place i by columns: neighbours read neighbours
    const int e = W > 1 ? d.by_V(i) : 0, v = i - e * d.V;
    const float2* at = entry + e * all + v;
    float2 s = at[0];
#pragma unroll 4
    for (int r = 1; r < d.R; ++r) s = add2(s, at[r * d.V]);
    finish(v * W + e, s, at);
  }
}

// The exponential is off by up to 2 + 1.2 |z| units in the last place, the quotient by 2, where results are fp32 too: far below zero, where that is
// much, the result itself is some z e^z
__device__ __forceinline__ float silu(float z) { return __fdividef(z, 1.f + __expf(-z)); }
__device__ __forceinline__ float silu_slope(float z, float dy) {
  const float g = __fdividef(1.f, 1.f + __expf(-z));
  return dy * (g * fmaf(z, 1.f - g, 1.f));
}

template <typename XT, typename YT, bool VEC, int PHASE>
__global__ void __launch_bounds__(threads_of(PHASE), PHASE == KEPT ? 6 : PHASE == TWICE ? 4 : 2)
group_forward_kernel(const __grid_constant__ Dev d) {
  constexpr int W = VEC ? 8 : 1, H = (W + 1) / 2, FLIGHT = PHASE == KEPT ? 4 : sizeof(XT) * W > 16 ? 4 : 8;      // FLIGHT: rows of a thread in flight
  constexpr int kThreads = threads_of(PHASE);
  constexpr bool KEEP = PHASE == KEPT, ONE = PHASE == KEPT || PHASE == TWICE;
  extern __shared__ __align__(16) uint8_t smem[];
  const Place<W> p(d);
  const int cg = d.by_cg.d, gs = d.slice / cg, chunks = d.by_chunks.d;
  const bool narrow = d.V <= kThreads;                   // one column a thread
  float* mean_of = (float*)smem;                         // [slice], each: minus the mean, 1/std times weight (with a ReLU the weight), bias of a channel
  float* a_of = mean_of + d.slice;
  float* b_of = a_of + d.slice;
  float2* column = (float2*)smem;                        // [slice], before those: mean and squared differences of a channel
  float2* part = (float2*)(smem + ((d.slice * (narrow ? 12 : 8) + 15) & ~15));     // [gs]: the CTA's, then [gs] mean and 1/std of all
  float2* stat = part + gs;
  float* base_of = (float*)(stat + gs);                  // [slice], unless a thread has several columns
  float2* entry = (float2*)(base_of + (narrow ? (d.slice + 3) & ~3 : 0));          // [W][R][V]: sums of the threads about a column's base
  const int mine = p.mine();
  const long long at = (p.pixel + p.r) * d.ldx + p.c0 + p.v * W;
  Rows<XT, W, KEEP> x = {(const XT*)d.x + at, (long long)d.R * d.ldx, {tc05::smem_u32(entry) + (uint32_t)d.entries + threadIdx.x * 16}};
  geeps_pdl_enter();

  if (PHASE != APPLY) {
    if constexpr (KEEP) {
      const XT* from = x.at;
#pragma unroll 4
      for (int k = 0; k < mine; ++k, from += x.step) x.kept.fetch(k, from);
      copies_done();
    }
    float2 mean[H], m2[H];
    auto pass = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < H; ++i) mean[i] = m2[i] = both(0.f);
      int n = 0;
      for (int k = 0; k < mine;) {
        const int end = min(mine, k + kPart), count = end - k;
        float2 s[H], q[H], base[H];
        auto begin = [&](const Vec<XT, W>& in) {
          in.get(base);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            s[i] = q[i] = both(0.f);
            base[i] = make_float2(-base[i].x, -base[i].y);
          }
        };
        auto add = [&](const Vec<XT, W>& in) {
          float2 f[H];
          in.get(f);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            const float2 e = add2(f[i], base[i]);
            s[i] = add2(s[i], e);
            q[i] = fma2(e, e, q[i]);
          }
        };
        if constexpr (KEEP) {
          begin(x.get(k));
          int j = k + 1;
          for (; j + FLIGHT <= end; j += FLIGHT) {
            Vec<XT, W> in[FLIGHT];
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) in[u] = x.get(j + u);
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) add(in[u]);
          }
#pragma unroll 1
          for (; j < end; ++j) add(x.get(j));
        } else {             // no load waits by itself: the first row, which adds nothing about itself, and the last ones come with others
          for (int j = k; j < end; j += FLIGHT) {
            Vec<XT, W> in[FLIGHT];
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) in[u] = x.get(min(j + u, end - 1));
            if (j == k) begin(in[0]);
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u)
              if (j + u < end) add(in[u]);
          }
        }
        const float inv = __frcp_rn((float)count), share = n ? (float)count / (n + count) : 1.f, weight = n * share;
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const float2 away = mul2(s[i], both(inv)), delta = make_float2(away.x - base[i].x - mean[i].x, away.y - base[i].y - mean[i].y);
          m2[i].x += fmaxf(q[i].x - s[i].x * away.x, 0.f) + delta.x * delta.x * weight;
          m2[i].y += fmaxf(q[i].y - s[i].y * away.y, 0.f) + delta.y * delta.y * weight;
          mean[i] = fma2(delta, both(share), mean[i]);
        }
        n += count;
        k = end;
      }
    };
    if (narrow) {
      pass();
      if (p.r == 0) {
#pragma unroll
        for (int i = 0; i < W; ++i) base_of[p.v * W + i] = value<W>(mean, i);
      }
      // the threads of a column about its base, the mean of the first of them
      __syncthreads();
      if (p.works) {
        const float n = (float)mine;
        float2* to = entry + p.r * d.V + p.v;
#pragma unroll
        for (int i = 0; i < W; ++i, to += d.R * d.V) {
          const float e = value<W>(mean, i) - base_of[p.v * W + i];
          *to = mine ? make_float2(n * e, fmaf(n * e, e, value<W>(m2, i))) : both(0.f);
        }
      }
      const float inv = p.rows ? __frcp_rn((float)p.rows) : 0.f;
      column_sums<kThreads, W>(d, entry, [&](int c, float2 t, const float2* at) {
        const float away = t.x * inv;
        float sq = fmaxf(t.y - t.x * away, 0.f);
        // A base far from the mean, as of a first pixel far from the others, leaves a small difference of large sums (1/std 8e-5 off for 119 pixels):
        // beyond five standard deviations, which a few pixels' mean seldom is by chance, the squares are formed again about the mean.  (Beyond
        // two 1 x 196 x 576 5.45 us -> 6.0; for every channel 256 x 196 x 576 35.0 -> 36.4.)
        if (t.x * away > 25.f * sq) {
          sq = 0.f;
#pragma unroll 1
          for (int r = 0; r < d.R; ++r) {
            const float2 u = at[r * d.V];
            const float n = (float)(p.most + (r < p.extra)), e = n > 0.f ? __fdividef(u.x, n) : 0.f;
            sq += fmaxf(u.y - u.x * e, 0.f) + n * (e - away) * (e - away);
          }
        }
        column[c] = make_float2(base_of[c] + away, sq);
      });
    } else {
      for (int v = threadIdx.x; v < d.V; v += kThreads, x.at += kThreads * W) {
        pass();
#pragma unroll
        for (int i = 0; i < W; ++i) column[v * W + i] = make_float2(value<W>(mean, i), value<W>(m2, i));
      }
      x.at = (const XT*)d.x + at;
    }
    __syncthreads();
    const int lanes = lanes_for(cg);
    const float each = __frcp_rn((float)cg);
    each_group<kThreads>(gs, lanes, [&](int g, int l, bool mine_g) {
      const float2* of = column + g * cg;
      float s = 0.f, sq = 0.f;
      for (int c = l; c < cg; c += lanes) s += of[c].x;
      const float m = lane_sum(s, lanes) * each;
      for (int c = l; c < cg; c += lanes) {
        const float e = of[c].x - m;
        sq += of[c].y + p.rows * (e * e);
      }
      sq = lane_sum(sq, lanes);
      if (l == 0 && mine_g) part[g] = make_float2(p.rows ? m : 0.f, p.rows ? sq : 0.f);
    });
  }
  if (PHASE == SUMS) {
    __syncthreads();
    for (int g = threadIdx.x; g < gs; g += kThreads)
      ((float2*)d.sums)[((long long)p.image * chunks + p.chunk) * d.groups + p.slice * gs + g] = part[g];
    return;
  }
  const float total = (float)d.pixels * cg;
  if (ONE) { if (chunks > 1) tc05::cluster_sync(); else __syncthreads(); }
  constexpr int MOST = ONE ? 1 : kMostParts / 32;       // entries of a lane
  const int lanes = lanes_for(chunks);
  each_group<kThreads>(gs, lanes, [&](int g, int l, bool) {
    auto get = [&](int i) {
      if (ONE) return ld_cluster_f2(tc05::map_to_cta(tc05::smem_u32(part + g), i));
      return ((const float2*)d.sums)[((long long)p.image * chunks + i) * d.groups + p.slice * gs + g];
    };
    auto n_of = [&](int i) { return (float)max(0, min(d.rows, d.pixels - i * d.rows)) * cg; };
    float2 t[MOST];
#pragma unroll
    for (int u = 0; u < MOST; ++u) { const int i = l + lanes * u; t[u] = i < chunks ? get(i) : both(0.f); }
    float s = 0.f, sq = 0.f;
#pragma unroll
    for (int u = 0; u < MOST; ++u) s = fmaf(n_of(l + lanes * u), t[u].x, s);
    const float m = lane_sum(s, lanes) / total;
#pragma unroll
    for (int u = 0; u < MOST; ++u) sq += t[u].y + n_of(l + lanes * u) * (t[u].x - m) * (t[u].x - m);
    sq = lane_sum(sq, lanes);
    if (l == 0) stat[g] = make_float2(m, __frcp_rn(__fsqrt_rn(sq / total + d.eps)));
  });
  __syncthreads();
  if (ONE && chunks > 1) tc05::cluster_arrive();      // nobody leaves while a peer still reads its sums
  if (d.stats != nullptr && p.chunk == 0)
    for (int g = threadIdx.x; g < gs; g += kThreads) ((float2*)d.stats)[(long long)p.image * d.groups + p.slice * gs + g] = stat[g];
  auto constant = [&](int c, float& mean, float& a, float& b) {
    const float2 s = stat[d.by_cg(c)];
    mean = -s.x;
    const float w = d.w != nullptr ? __ldg(d.w + p.c0 + c) : 1.f;
    a = d.act == 1 ? w : s.y * w;
    b = d.b != nullptr ? __ldg(d.b + p.c0 + c) : 0.f;
  };
  if (narrow) {
    for (int c = threadIdx.x; c < d.slice; c += kThreads) constant(c, mean_of[c], a_of[c], b_of[c]);
    __syncthreads();
  }
  const long long ostep = (long long)d.R * d.ldo;
  YT* y = (YT*)d.out + (p.pixel + p.r) * d.ldo + p.c0 + p.v * W;
  auto pass = [&](int v, auto act) __attribute__((always_inline)) {
    constexpr int ACT = decltype(act)::value;
    float2 mean[H], a[H], b[H], rstd[H];
    if (ACT == 1) {
#pragma unroll
      for (int i = 0; i < 2 * H; ++i) value<W>(rstd, i) = stat[d.by_cg(v * W + (i < W ? i : 0))].y;
    }
    if (narrow) {
      channel_values<W>(mean_of, v, mean);
      channel_values<W>(a_of, v, a);
      channel_values<W>(b_of, v, b);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * H; ++i) constant(v * W + (i < W ? i : 0), value<W>(mean, i), value<W>(a, i), value<W>(b, i));
    }
    YT* to = y;
    auto finish = [&](const Vec<XT, W>& in) {
      float2 f[H];
      in.get(f);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        f[i] = add2(f[i], mean[i]);
        // z of a ReLU is rounded after each operation, as in the backward pass, so that both have the same border.  A product of pairs goes
        // into an fma with a factor that is known at run time only: a sum would be contracted with it
        if (ACT != 1) f[i] = fma2(f[i], a[i], b[i]);
        else if (W > 1) f[i] = fma2(mul2(mul2(f[i], rstd[i]), a[i]), both(d.one), b[i]);
        else f[i].x = __fadd_rn(__fmul_rn(__fmul_rn(f[i].x, rstd[i].x), a[i].x), b[i].x);
        if (ACT == 2) f[i] = make_float2(silu(f[i].x), W > 1 ? silu(f[i].y) : 0.f);
      }
      Vec<YT, W> o;
      o.set(f);
      if (ACT == 1) o.relu();
      o.store(to);
      to += ostep;
    };
    int k = 0;
    for (; k + FLIGHT <= mine; k += FLIGHT) {
      Vec<XT, W> in[FLIGHT];
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) in[u] = x.get(k + u);
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) finish(in[u]);
    }
    if constexpr (KEEP) {
#pragma unroll 1
      for (; k < mine; ++k) finish(x.get(k));
    } else if (k < mine) {
      Vec<XT, W> in[FLIGHT];
#pragma unroll
      for (int u = 0; u < FLIGHT - 1; ++u) in[u] = x.get(min(k + u, mine - 1));
#pragma unroll
      for (int u = 0; u < FLIGHT - 1; ++u)
        if (k + u < mine) finish(in[u]);
    }
  };
  auto by_act = [&](int v) __attribute__((always_inline)) {
    if (d.act == 0) pass(v, std::integral_constant<int, 0>());
    else if (d.act == 1) pass(v, std::integral_constant<int, 1>());
    else pass(v, std::integral_constant<int, 2>());
  };
  if (narrow) {
    if (p.works) by_act(p.v);
  } else {
    for (int v = threadIdx.x; v < d.V; v += kThreads, x.at += kThreads * W, y += kThreads * W) by_act(v);
  }
  if (ONE && chunks > 1) tc05::cluster_wait();
}

template <typename XT, typename YT, bool VEC, int PHASE>
__global__ void __launch_bounds__(threads_of(PHASE), PHASE == KEPT && sizeof(XT) == 2 ? 5 : threads_of(PHASE) == 128 ? 4 : 2)
group_backward_kernel(const __grid_constant__ Dev d, float* channel_sums) {
  constexpr bool KEEP = PHASE == KEPT || PHASE == MIXED, ONE = KEEP || PHASE == TWICE;
  constexpr int W = VEC ? 8 : 1, H = (W + 1) / 2, FLIGHT = KEEP ? 2 : W == 1 ? 8 : sizeof(XT) > 2 ? 2 : 4;
  constexpr int kThreads = threads_of(PHASE), REG = PHASE == MIXED ? kInRegisters : 0;
  extern __shared__ __align__(16) uint8_t smem[];
  const Place<W> p(d);
  const int cg = d.by_cg.d, gs = d.slice / cg, chunks = d.by_chunks.d;
  const bool narrow = d.V <= kThreads;
  // [slice], each: minus the mean, 1/std, weight and bias of a channel; then the factors of dz and of x - mean in dx, and the rest
  float* mean_of = (float*)smem;
  float *rstd_of = mean_of + d.slice, *w_of = rstd_of + d.slice, *b_of = w_of + d.slice, *dz_of = b_of + d.slice, *x_of = dz_of + d.slice, *one_of = x_of + d.slice;
  float2* column = (float2*)(smem + (narrow ? (d.slice * 28 + 15) & ~15 : 0));     // [slice]: sums of dz and dz n of a channel
  float2* part = column + d.slice;                       // [gs]: sums of dz w and dz w n of the CTA's pixels, then of all
  float2* whole = part + gs;
  float2* entry = (float2*)(((uintptr_t)(whole + gs) + 15) & ~(uintptr_t)15);      // [W][R][V], unless there is one thread a column
  const int mine = p.mine();
  const long long x_at = (p.pixel + p.r) * d.ldx + p.c0 + p.v * W, dy_at = (p.pixel + p.r) * d.lddy + p.c0 + p.v * W;
  Rows<XT, W, KEEP> x = {(const XT*)d.x + x_at, (long long)d.R * d.ldx, {tc05::smem_u32(entry) + (uint32_t)d.entries + threadIdx.x * 16}};
  Rows<YT, W, KEEP> dy = {(const YT*)d.dy + dy_at, (long long)d.R * d.lddy, {x.kept.base + (uint32_t)(d.keep * Kept<XT>::kBytes)}};
  geeps_pdl_enter();
  Vec<XT, W> xr[REG + 1];                // (an array has one element at least)
  Vec<YT, W> dr[REG + 1];
  if constexpr (KEEP) {
    const XT* xs = x.at;
    const YT* ds = dy.at;
#pragma unroll
    for (int k = 0; k < REG; ++k, xs += x.step, ds += dy.step)
      if (k < mine) { xr[k].load(xs); dr[k].load(ds); }
#pragma unroll 4
    for (int k = 0; k < mine - REG; ++k, xs += x.step, ds += dy.step) {
      x.kept.fetch(k, xs);
      dy.kept.fetch(k, ds);
    }
  }
  const float2* stats = (const float2*)d.stats + (long long)p.image * d.groups + p.slice * gs;
  auto constant = [&](int c, float& mean, float& rstd, float& w, float& b) {
    const float2 s = stats[d.by_cg(c)];
    mean = -s.x;
    rstd = s.y;
    w = d.w != nullptr ? __ldg(d.w + p.c0 + c) : 1.f;
    b = d.b != nullptr ? __ldg(d.b + p.c0 + c) : 0.f;
  };
  if (narrow) {          // else a thread has several columns, and shared memory no room for all of theirs
    for (int c = threadIdx.x; c < d.slice; c += kThreads) constant(c, mean_of[c], rstd_of[c], w_of[c], b_of[c]);
    __syncthreads();
  }
  // f(x, dy) for all rows of a column, FLIGHT of them in flight.  keep: dy as f leaves it is kept for the next time
  auto rows = [&](auto f, auto keep) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < REG; ++k)
      if (k < mine) {
        Vec<YT, W> d = dr[k];
        f(xr[k], d);
        if (decltype(keep)::value) dr[k] = d;
      }
    const int end = mine - REG;
    int k = 0;
    auto one = [&](int k, const Vec<XT, W>& xi, Vec<YT, W>& di) {
      f(xi, di);
      if constexpr (KEEP) { if (decltype(keep)::value) dy.kept.put(k, di); }
    };
    for (; k + FLIGHT <= end; k += FLIGHT) {
      Vec<XT, W> xi[FLIGHT];
      Vec<YT, W> di[FLIGHT];
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) { xi[u] = x.get(k + u); di[u] = dy.get(k + u); }
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) one(k + u, xi[u], di[u]);
    }
    if (KEEP || k + 1 == end) {
#pragma unroll 1
      for (; k < end; ++k) {
        Vec<YT, W> d = dy.get(k);
        one(k, x.get(k), d);
      }
    } else if (k < end) {
      Vec<XT, W> xi[FLIGHT];
      Vec<YT, W> di[FLIGHT];
#pragma unroll
      for (int u = 0; u < FLIGHT - 1; ++u) { xi[u] = x.get(min(k + u, end - 1)); di[u] = dy.get(min(k + u, end - 1)); }
#pragma unroll
      for (int u = 0; u < FLIGHT - 1; ++u)
        if (k + u < end) one(k + u, xi[u], di[u]);
    }
  };
  // z, rounded after each operation: not in pairs, which are contracted to fused multiply-adds
  auto border = [&](const float2& n, const float2& w, const float2& b) {
    return make_float2(__fadd_rn(__fmul_rn(n.x, w.x), b.x), W > 1 ? __fadd_rn(__fmul_rn(n.y, w.y), b.y) : 0.f);
  };
  if (PHASE != APPLY) {
    if constexpr (KEEP) copies_done();
    auto pass = [&](int v, auto act) __attribute__((always_inline)) {
      constexpr int ACT = decltype(act)::value;
      float2 mean[H], rstd[H], w[H], b[H], sa[H], sb[H];
      if (narrow) {
        channel_values<W>(mean_of, v, mean);
        channel_values<W>(rstd_of, v, rstd);
        if (ACT) { channel_values<W>(w_of, v, w); channel_values<W>(b_of, v, b); }
      } else {
#pragma unroll
        for (int i = 0; i < 2 * H; ++i) constant(v * W + (i < W ? i : 0), value<W>(mean, i), value<W>(rstd, i), value<W>(w, i), value<W>(b, i));
      }
#pragma unroll
      for (int i = 0; i < H; ++i) sa[i] = sb[i] = both(0.f);
      rows([&](const Vec<XT, W>& xi, Vec<YT, W>& di) {
        float2 dz[H], n[H], z[H];
        xi.get(n);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          n[i] = mul2(add2(n[i], mean[i]), rstd[i]);
          if (ACT) z[i] = border(n[i], w[i], b[i]);
        }
        if (ACT == 1) di.mask(z);                        // kept for the second pass, which needs no z then
        di.get(dz);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          if (ACT == 2) dz[i] = make_float2(silu_slope(z[i].x, dz[i].x), W > 1 ? silu_slope(z[i].y, dz[i].y) : 0.f);
          sa[i] = add2(sa[i], dz[i]);
          sb[i] = fma2(dz[i], n[i], sb[i]);
        }
      }, std::integral_constant<bool, ACT == 1>());
      float2* to = d.R == 1 ? column + v * W : entry + p.r * d.V + v;
      const int next = d.R == 1 ? 1 : d.R * d.V;
#pragma unroll
      for (int i = 0; i < W; ++i, to += next) *to = make_float2(value<W>(sa, i), value<W>(sb, i));
    };
    auto by_act = [&](int v) __attribute__((always_inline)) {
      if (d.act == 0) pass(v, std::integral_constant<int, 0>());
      else if (d.act == 1) pass(v, std::integral_constant<int, 1>());
      else pass(v, std::integral_constant<int, 2>());
    };
    if (narrow) {
      if (p.works) by_act(p.v);
    } else {
      for (int v = threadIdx.x; v < d.V; v += kThreads, x.at += kThreads * W, dy.at += kThreads * W) by_act(v);
      x.at = (const XT*)d.x + x_at;
      dy.at = (const YT*)d.dy + dy_at;
    }
    if (d.R > 1) column_sums<kThreads, W>(d, entry, [&](int c, float2 t, const float2*) { column[c] = t; });
    __syncthreads();
    const int lanes = lanes_for(cg);
    each_group<kThreads>(gs, lanes, [&](int g, int l, bool mine_g) {
      float2 s = both(0.f);
      for (int c = l; c < cg; c += lanes) s = fma2(column[g * cg + c], both(narrow ? w_of[g * cg + c] : d.w != nullptr ? __ldg(d.w + p.c0 + g * cg + c) : 1.f), s);
      s.x = lane_sum(s.x, lanes);
      s.y = lane_sum(s.y, lanes);
      if (l == 0 && mine_g) part[g] = s;
    });
  }
  if (PHASE == SUMS) {
    __syncthreads();
    const long long at = (long long)p.image * chunks + p.chunk;
    for (int g = threadIdx.x; g < gs; g += kThreads) ((float2*)d.sums)[at * d.groups + p.slice * gs + g] = part[g];
    if (channel_sums != nullptr)
      for (int c = threadIdx.x; c < d.slice; c += kThreads) ((float2*)channel_sums)[at * d.C + p.c0 + c] = column[c];
    return;
  }
  const float scale = 1.f / ((float)d.pixels * cg);
  if (ONE) { if (chunks > 1) tc05::cluster_sync(); else __syncthreads(); }
  constexpr int MOST = ONE ? 1 : kMostParts / 32;       // entries of a lane
  const int lanes = lanes_for(chunks);
  each_group<kThreads>(gs, lanes, [&](int g, int l, bool) {
    float2 s = both(0.f);
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
      const int i = l + lanes * u;
      if (i >= chunks) continue;
      if (ONE) s = add2(s, ld_cluster_f2(tc05::map_to_cta(tc05::smem_u32(part + g), i)));
      else s = add2(s, ((const float2*)d.sums)[((long long)p.image * chunks + i) * d.groups + p.slice * gs + g]);
    }
    s.x = lane_sum(s.x, lanes);
    s.y = lane_sum(s.y, lanes);
    if (l == 0) whole[g] = make_float2(-s.x * scale, -s.y * scale);
  });
  // the image's sums of a channel: each CTA joins its share of the slice's
  if (ONE && channel_sums != nullptr)
    for (int c = p.chunk * kThreads + threadIdx.x; c < d.slice; c += chunks * kThreads) {
      float2 s = both(0.f);
      for (int i = 0; i < chunks; ++i) s = add2(s, ld_cluster_f2(tc05::map_to_cta(tc05::smem_u32(column + c), i)));
      ((float2*)channel_sums)[(long long)p.image * d.C + p.c0 + c] = s;
    }
  __syncthreads();
  if (ONE && chunks > 1) tc05::cluster_arrive();      // nobody leaves while a peer still reads its sums
  // dx = dz (w rstd) + (x - mean) (-mean(dz w n) rstd^2) - mean(dz w) rstd
  auto factors = [&](int c, float w, float rstd, float& dz, float& x, float& one) {
    const float2 s = whole[d.by_cg(c)];
    dz = w * rstd;
    x = s.y * rstd * rstd;
    one = s.x * rstd;
  };
  if (narrow) {
    for (int c = threadIdx.x; c < d.slice; c += kThreads) factors(c, w_of[c], rstd_of[c], dz_of[c], x_of[c], one_of[c]);
    __syncthreads();
  }
  const long long ostep = (long long)d.R * d.ldo;
  XT* dx = (XT*)d.out + (p.pixel + p.r) * d.ldo + p.c0 + p.v * W;
  auto pass = [&](int v, auto act) __attribute__((always_inline)) {
    constexpr int ACT = decltype(act)::value;
    constexpr bool AGAIN = ACT == 2 || (ACT == 1 && !KEEP);      // z is needed again
    float2 mean[H], rstd[H], w[H], b[H], fz[H], fx[H], f1[H];
    if (narrow) {
      channel_values<W>(mean_of, v, mean);
      if (AGAIN) { channel_values<W>(rstd_of, v, rstd); channel_values<W>(w_of, v, w); channel_values<W>(b_of, v, b); }
      channel_values<W>(dz_of, v, fz);
      channel_values<W>(x_of, v, fx);
      channel_values<W>(one_of, v, f1);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * H; ++i) {
        const int c = v * W + (i < W ? i : 0);
        constant(c, value<W>(mean, i), value<W>(rstd, i), value<W>(w, i), value<W>(b, i));
        factors(c, value<W>(w, i), value<W>(rstd, i), value<W>(fz, i), value<W>(fx, i), value<W>(f1, i));
      }
    }
    XT* to = dx;
    rows([&](const Vec<XT, W>& xi, Vec<YT, W>& di) {
      float2 dz[H], e[H], z[H];
      xi.get(e);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        e[i] = add2(e[i], mean[i]);
        if (AGAIN) z[i] = border(mul2(e[i], rstd[i]), w[i], b[i]);
      }
      if (AGAIN && ACT == 1) di.mask(z);
      di.get(dz);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        if (ACT == 2) dz[i] = make_float2(silu_slope(z[i].x, dz[i].x), W > 1 ? silu_slope(z[i].y, dz[i].y) : 0.f);
        dz[i] = fma2(dz[i], fz[i], fma2(e[i], fx[i], f1[i]));
      }
      Vec<XT, W> o;
      o.set(dz);
      o.store(to);
      to += ostep;
    }, std::false_type());
  };
  auto by_act = [&](int v) __attribute__((always_inline)) {
    if (d.act == 0) pass(v, std::integral_constant<int, 0>());
    else if (d.act == 1) pass(v, std::integral_constant<int, 1>());
    else pass(v, std::integral_constant<int, 2>());
  };
  if (narrow) {
    if (p.works) by_act(p.v);
  } else {
    for (int v = threadIdx.x; v < d.V; v += kThreads, x.at += kThreads * W, dy.at += kThreads * W, dx += kThreads * W) by_act(v);
  }
  if (ONE && chunks > 1) tc05::cluster_wait();
}

// Sums over `parts` rows of {dz, dz n} of the channels: 8 channels a block, 32 of them in flight for each
__global__ void __launch_bounds__(256)
group_parameters_kernel(const float2* __restrict__ sums, long long parts, int C, float* dw, float* db) {
  geeps_pdl_enter();
  __shared__ float2 sh[32][9];
  const int i = threadIdx.x >> 3, c = blockIdx.x * 8 + (threadIdx.x & 7);
  float2 s = both(0.f);
  if (c < C) {
#pragma unroll 4
    for (long long r = i; r < parts; r += 32) s = add2(s, sums[r * C + c]);
  }
  sh[i][threadIdx.x & 7] = s;
  __syncthreads();
  if (i == 0 && c < C) {
#pragma unroll
    for (int r = 1; r < 32; ++r) s = add2(s, sh[r][threadIdx.x]);
    if (db != nullptr) db[c] = s.x;
    if (dw != nullptr) dw[c] = s.y;
  }
}

// ---------------- host side ----------------
struct Shape { int vec, threads, in_registers, fused, slice, slices, chunks, rows, keep, blocks, V, R, entries; size_t smem; };

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

constexpr int kMostChunks = 8;             // CTAs of a cluster
constexpr size_t kSmem = 200 * 1024;

// Shared memory that does not depend on the pixels kept
size_t fixed_bytes(const Shape& s, int cg, bool backward) {
  const size_t gs = s.slice / cg, narrow = s.V <= s.threads;
  if (backward) return (narrow ? (s.slice * 28 + 15) & ~15 : 0) + (size_t)s.slice * 8 + gs * 16 + 16;
  return ((s.slice * (narrow ? 12 : 8) + 15) & ~15) + gs * 16 + (narrow ? ((s.slice + 3) & ~3) * 4 : 0);
}

Shape plan(int images, int pixels, int C, int groups, bool backward, bool vec, int xsize, int ysize) {
  Shape s = {};
  const int cg = C / groups, W = vec ? 8 : 1, sms = geeps_sm_count();
  const int unit = cg / gcd(cg, W) * W;          // channels of the narrowest slice
  s.vec = vec;
  s.threads = threads_of(KEPT);
  const int row_bytes = s.threads * 16 * (vec ? (xsize / 2 + (backward ? ysize / 2 : 0)) : 0);      // of all threads' kept rows
  // One launch: slices of 32 channels (whole sectors of a pixel) and more, and up to eight CTAs for an item.  The cost in us: 6 for each
  // time that the SMs' room is filled (a CTA's steps follow one another, and CTAs that began together rarely overlap; narrow slices
  // have fewer channels a thread to join), and the bytes that an SM reads (as many are written).  Measured, bf16 forward,
  // slice / CTAs of a cluster: 32 x 784 x 256: 32/1 9.0 us, 64/1 9.1, 32/3 10.8, 64/7 (just over one filling) 13.8, 32/8 21.8;
  // 64 x 49 x 1024: 128/1 7.4, 512/1 9.1, 128/6 25.8; backward, 256 x 196 x 576, all pixels in shared memory:
  // 72/1 56.5, 72/2 65.9, 288/3 88.
  auto cut = [&](Shape& t) {             // what a thread has of a slice
    t.V = t.slice / W;
    t.R = t.V < t.threads ? t.threads / t.V : 1;
    t.entries = (((backward ? t.R > 1 : t.V <= t.threads) ? t.R * t.slice * 8 : 0) + 15) & ~15;
  };
  double best = 1e300;
  int chunks = 0;
  // ... narrower ones only where the channels have no such divisor
  const int limit = W * s.threads < C ? W * s.threads : C;
  int least = C < 32 ? 1 : 32;
  while (least > 1) {
    int n = (least + unit - 1) / unit;
    while (unit * n <= limit && C / unit % n) ++n;
    if (unit * n <= limit || unit >= least) break;
    least = 1;
  }
  for (int n = 1; n == 1 || unit * n <= limit; ++n) {
    if (C / unit % n || unit * n < least) continue;
    Shape t = s;
    t.slice = unit * n;
    t.slices = C / t.slice;
    cut(t);
    if (vec && t.V > t.threads) continue;
    for (int k = 1; k <= kMostChunks; ++k) {
      const int rows = (pixels + k - 1) / k, keep = (rows + t.R - 1) / t.R;
      if (k > 1 && rows < t.R) continue;
      int fewer = 0;                       // blocks an SM without pixels in registers
      for (int held = 0; held <= (vec && backward && xsize == 2 ? kInRegisters : 0); held += kInRegisters) {
        const size_t smem = fixed_bytes(t, cg, backward) + t.entries + (size_t)(keep > held ? keep - held : 0) * row_bytes;
        if (smem > kSmem) continue;
        const int fit = (int)(228 * 1024 / (smem + 1024)), most = !vec || held ? 4 : !backward ? 6 : xsize == 2 ? 5 : 4, resident = fit < most ? fit : most;
        if (held && (resident < 3 || resident <= fewer)) continue;
        fewer = resident;
        const double ctas = (double)images * t.slices * k, filled = ctas / ((double)sms * resident);
        const double kb = (double)rows * t.slice * (xsize + (backward ? ysize : 0)) / 1024, join = k > 1 ? 0.5 : 0.0;
        const double cost = vec ? ceil(filled) * (6.0 + 0.4 * t.slice / t.threads) + ceil(ctas / sms) * (0.15 + kb / (xsize == 2 ? 21.0 : 18.0)) + join
                                : (filled > 1.0 ? filled : 1.0) * (6.0 + kb / 2.7 + join);
        if (cost < best) { best = cost; s = t; s.in_registers = held; chunks = k; }
      }
    }
  }
  // Two launches, at best of one filling of two blocks an SM.  32 x 784 x 256: 9 x 32 = 288 blocks 13.1 us, 12 x 32 = 384 20.5.  Against one
  // launch (two / one): bf16 32 x 784 x 256 forward 13.1 / 9.0, 32 x 3136 x 192 forward 31.5 / 25.9, backward 44.1 / 45.5, in fp32 75 / 122.
  Shape u = s;
  int n = 1;
  while (unit * n < C && (unit * n < 64 || C / unit % n)) ++n;
  u.threads = threads_of(SUMS);
  for (;; --n) {                             // down to a width that fits (one group does, of kMostChannels channels too)
    if (C / unit % n) continue;
    u.slice = unit * n;
    u.slices = C / u.slice;
    cut(u);
    if (n == 1 || fixed_bytes(u, cg, backward) + u.entries <= kSmem) break;
  }
  const long long parts = (long long)images * u.slices, most = (pixels + u.R - 1) / u.R;
  const int cuts = (int)std::max(1LL, std::min({2LL * sms / parts, most, (long long)kMostParts}));
  const double kb = (double)images * pixels * C * (xsize + (backward ? ysize : 0)) / 1024 / sms;
  const double twice = (backward ? 4.5 : 2.0) + 6.0 * ceil(parts * cuts / (2.0 * sms)) + kb / (!vec ? 2.0 : backward ? 16.0 : 11.6);
  s.fused = chunks > 0 && best <= twice;
  if (!s.fused) {
    s = u;
    s.in_registers = 0;
    chunks = cuts;
  }
  const long long items = (long long)images * s.slices;
  s.rows = (pixels + chunks - 1) / chunks;
  s.chunks = s.fused ? chunks : (pixels + s.rows - 1) / s.rows;
  s.keep = vec && s.fused ? std::max(0, (s.rows + s.R - 1) / s.R - s.in_registers) : 0;
  s.smem = fixed_bytes(s, cg, backward) + s.entries + (size_t)s.keep * row_bytes;
  s.blocks = items * s.chunks > 0x7fffffffLL ? 0 : (int)(items * s.chunks);
  return s;
}

// plan() of the sizes that this thread has met last: a network's layers ask again in every step
Shape choose(int images, int pixels, int C, int groups, bool backward, bool vec, int xsize, int ysize) {
  struct Met { int key[8]; Shape s; };
  static thread_local Met met[64] = {};
  const int key[8] = {images, pixels, C, groups, geeps_sm_count(), (backward ? 1 : 0) | (vec ? 2 : 0), xsize, ysize};
  unsigned h = 0;
  for (int k : key) h = (h ^ (unsigned)k) * 0x9E3779B1u;
  Met& m = met[h >> 26];
  if (memcmp(m.key, key, sizeof(key))) {
    m.s = plan(images, pixels, C, groups, backward, vec, xsize, ysize);
    memcpy(m.key, key, sizeof(key));
  }
  return m.s;
}

// Dependent launches (us in a captured chain of 12, ordinary / dependent): 1 x 196 x 576 6.0 / 5.6, 8 x 196 x 512 5.8 / 5.4, backward of
// 4 x 784 x 256 8.1 / 7.8 and of 16 x 1024 x 640 in fp32 (two launches) 46.4 / 45.3.  Forward with several blocks an SM in one launch
// they come up where the predecessor leaves room, and SMs run dry: 64 x 49 x 1024 7.4 / 7.9, 37 x 113 x 1003 14.3 / 15.2.
template <auto kernel, typename... A>
int launch(const Shape& s, bool cluster, bool dependent, cudaStream_t st, A&&... args) {
  static std::atomic<unsigned long long> ready{0};           // devices on which the kernel may have all shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(ready >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    ready |= 1ull << (dev & 63);
  }
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)s.blocks);
  cfg.blockDim = dim3(s.threads);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)s.chunks;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = dependent ? at : at + 1;
  cfg.numAttrs = (dependent ? 1 : 0) + (cluster && s.chunks > 1 ? 1 : 0);
  return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<A&&>(args)...);
}

template <typename XT, typename YT, bool VEC>
int run(const GeepsGroupNorm& k, const Shape& s, const Dev& d, bool backward, cudaStream_t st) {
  constexpr int ONE = VEC ? KEPT : TWICE;
  int e;
  if (!backward) {
    if (s.fused) return launch<group_forward_kernel<XT, YT, VEC, ONE>>(s, true, s.blocks <= geeps_sm_count(), st, d);
    e = launch<group_forward_kernel<XT, YT, VEC, SUMS>>(s, false, true, st, d);
    return e ? e : launch<group_forward_kernel<XT, YT, VEC, APPLY>>(s, false, true, st, d);
  }
  const bool want = k.dweight != nullptr || k.dbias != nullptr;
  // group sums of the chunks (two launches only), then the channels' sums of the images or chunks
  const long long parts = (long long)k.images * (s.fused ? 1 : s.chunks);
  float* channel = want ? k.work + (s.fused ? 0 : parts * k.groups * 2) : nullptr;
  if (s.fused && s.in_registers) {
    if constexpr (VEC && sizeof(XT) == 2) e = launch<group_backward_kernel<XT, YT, VEC, MIXED>>(s, true, true, st, d, channel);
    else e = (int)cudaErrorInvalidValue;
  } else if (s.fused) {
    e = launch<group_backward_kernel<XT, YT, VEC, ONE>>(s, true, true, st, d, channel);
  } else {
    e = launch<group_backward_kernel<XT, YT, VEC, SUMS>>(s, false, true, st, d, channel);
    if (!e) e = launch<group_backward_kernel<XT, YT, VEC, APPLY>>(s, false, true, st, d, channel);
  }
  if (e || !want) return e;
  geeps_launch(group_parameters_kernel, dim3((unsigned)((k.C + 7) / 8)), dim3(256), 0, st, (const float2*)channel, parts, k.C, k.dweight, k.dbias);
  return (int)cudaGetLastError();
}

bool vectors(const GeepsGroupNorm& k, bool backward) {
  const int xs = k.x_fp32 ? 4 : 2, ys = k.y_fp32 ? 4 : 2;
  auto ok = [](const void* p, long long ld, int size) { return ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0; };
  return k.C % 8 == 0 && ok(k.x, k.ldx, xs) && (backward ? ok(k.dy, k.lddy, ys) && ok(k.dx, k.lddx, xs) : ok(k.y, k.ldy, ys));
}

int check(const GeepsGroupNorm* k, bool backward) {
  if (!k || k->images < 0 || k->pixels < 0 || (k->y_fp32 && !k->x_fp32) || !(k->eps >= 0.f) || k->act < 0 || k->act > 2) return (int)cudaErrorInvalidValue;
  if (k->C < 1 || k->C > kMostChannels) return GEEPS_ERR_NORM_CHANNELS;
  if (k->groups < 1 || k->C % k->groups) return GEEPS_ERR_GROUPS;
  if (k->images > (1LL << 30) || k->pixels > (1LL << 30) || k->images * k->pixels > (1LL << 30)) return (int)cudaErrorInvalidValue;
  const long long rows = k->images * k->pixels;
  const int xs = k->x_fp32 ? 4 : 2, ys = k->y_fp32 ? 4 : 2;
  struct Range { const void* at; long long bytes; bool written; long long pitch; int align; };      // pitch: of rows, in bytes; 0: none
  auto span = [&](long long ld, int size) { return rows ? ((rows - 1) * ld + k->C) * size : 0; };
  if (k->ldx < k->C || (backward ? k->lddy < k->C || k->lddx < k->C : k->ldy < k->C)) return (int)cudaErrorInvalidValue;
  const long long stats = k->images * k->groups * 8, work = geeps_group_norm_work(k->images, k->pixels, k->C, k->groups, backward) * 4;
  const Range all[] = {
      {k->x, span(k->ldx, xs), false, k->ldx * xs, xs},
      {backward ? k->dy : nullptr, span(k->lddy, ys), false, k->lddy * ys, ys},
      {backward ? k->dx : k->y, backward ? span(k->lddx, xs) : span(k->ldy, ys), true, backward ? k->lddx * xs : k->ldy * ys, backward ? xs : ys},
      {k->weight, 4LL * k->C, false, 0, 4}, {k->bias, 4LL * k->C, false, 0, 4},
      {k->stats, stats, !backward, 0, 8}, {k->work, work, true, 0, 8},
      {backward ? k->dweight : nullptr, 4LL * k->C, true, 0, 4}, {backward ? k->dbias : nullptr, 4LL * k->C, true, 0, 4}};
  if (rows && (!k->x || !(backward ? (const void*)k->dx : k->y) || (backward && (!k->dy || !k->stats)) || (work && !k->work))) return (int)cudaErrorInvalidValue;
  for (const auto& r : all) if (r.at && ((uintptr_t)r.at & (r.align - 1))) return GEEPS_ERR_NORM_ALIGN;
  for (const auto& a : all) {
    if (!a.at || !a.written || !a.bytes) continue;
    for (const auto& b : all) {
      if (&a == &b || !b.at || !b.bytes) continue;
      // an output may be the very same rows as an input of its size
      const bool same = a.pitch && a.pitch == b.pitch && a.at == b.at && a.align == b.align && !b.written;
      // ... or other channels of the same wider rows
      const long long off = a.pitch && a.pitch == b.pitch ? (((long long)((uintptr_t)b.at - (uintptr_t)a.at)) % a.pitch + a.pitch) % a.pitch : 0;
      const bool beside = off >= (long long)k->C * a.align && off + (long long)k->C * b.align <= a.pitch;
      if (!same && !beside && (uintptr_t)a.at < (uintptr_t)b.at + b.bytes && (uintptr_t)b.at < (uintptr_t)a.at + a.bytes) return GEEPS_ERR_NORM_OVERLAP;
    }
  }
  return 0;
}

int call(const GeepsGroupNorm* k, bool backward, void* stream) {
  const int e = check(k, backward);
  if (e) return e;
  cudaStream_t st = (cudaStream_t)stream;
  if (k->images == 0 || k->pixels == 0) {
    if (backward && k->dweight) geeps_clear_f32(k->dweight, k->C, stream);
    if (backward && k->dbias) geeps_clear_f32(k->dbias, k->C, stream);
    return (int)cudaGetLastError();
  }
  const bool vec = vectors(*k, backward);
  const Shape s = choose((int)k->images, (int)k->pixels, k->C, k->groups, backward, vec, k->x_fp32 ? 4 : 2, k->y_fp32 ? 4 : 2);
  if (!s.blocks) return (int)cudaErrorInvalidValue;
  Dev d = {};
  d.x = k->x; d.dy = k->dy; d.out = backward ? k->dx : k->y; d.w = k->weight; d.b = k->bias; d.stats = k->stats; d.sums = k->work;
  d.ldx = k->ldx; d.lddy = k->lddy; d.ldo = backward ? k->lddx : k->ldy;
  d.pixels = (int)k->pixels; d.C = k->C; d.groups = k->groups; d.slice = s.slice; d.slices = s.slices; d.rows = s.rows; d.act = k->act;
  d.keep = s.keep; d.V = s.V; d.R = s.R; d.entries = s.entries; d.eps = k->eps; d.one = 1.f;
  d.by_chunks = Divide(s.chunks); d.by_slices = Divide(s.slices); d.by_V = Divide(s.V); d.by_cg = Divide(k->C / k->groups);
  if (k->y_fp32) return vec ? run<float, float, true>(*k, s, d, backward, st) : run<float, float, false>(*k, s, d, backward, st);
  if (k->x_fp32) return vec ? run<float, bf16, true>(*k, s, d, backward, st) : run<float, bf16, false>(*k, s, d, backward, st);
  return vec ? run<bf16, bf16, true>(*k, s, d, backward, st) : run<bf16, bf16, false>(*k, s, d, backward, st);
}

}  // namespace

extern "C" {

long long geeps_group_norm_work(long long images, long long pixels, int C, int groups, int backward) {
  if (images < 1 || pixels < 1 || C < 1 || C > kMostChannels || groups < 1 || C % groups || images > (1LL << 30) || pixels > (1LL << 30) || images * pixels > (1LL << 30))
    return 0;                              // the call itself says why
  // of two launches for vectors or single values, whichever the addresses will allow, of any type: the chunks' group sums; backward
  // also the channels' sums of the chunks or images
  long long most = 0;
  for (int vec = 0; vec < (C % 8 ? 1 : 2); ++vec)
    for (int type = 0; type < 3; ++type) {
      const Shape s = choose((int)images, (int)pixels, C, groups, backward, vec, type ? 4 : 2, type == 2 ? 4 : 2);
      const long long parts = images * (s.fused ? 1 : s.chunks);
      const long long n = (s.fused ? 0 : parts * groups * 2) + (backward ? parts * C * 2 : 0);
      most = n > most ? n : most;
    }
  return most;
}

int geeps_group_norm_forward(const GeepsGroupNorm* p, void* stream) { return call(p, false, stream); }
int geeps_group_norm_backward(const GeepsGroupNorm* p, void* stream) { return call(p, true, stream); }

int geeps_group_norm_shape(long long images, long long pixels, int C, int groups, int backward, int vec, int x_fp32, int y_fp32, int* out) {
  if (C < 1 || C > kMostChannels) return GEEPS_ERR_NORM_CHANNELS;
  if (images < 1 || pixels < 1 || groups < 1 || C % groups || (vec && C % 8) || images > (1LL << 30) || pixels > (1LL << 30) || images * pixels > (1LL << 30))
    return (int)cudaErrorInvalidValue;
  const Shape s = choose((int)images, (int)pixels, C, groups, backward, vec, x_fp32 ? 4 : 2, y_fp32 ? 4 : 2);
  out[0] = s.fused; out[1] = s.slice; out[2] = s.chunks; out[3] = s.rows; out[4] = s.keep; out[5] = s.blocks; out[6] = (int)s.smem; out[7] = s.threads; out[8] = s.in_registers;
  return 0;
}

}  // extern "C"
