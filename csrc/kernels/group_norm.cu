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
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.
//
// Variance: values less the first of every 32 of a thread's pixels are added and squared, and such parts meet as count, mean and
// sum of squared differences, so a mean far from zero costs nothing (a part's error is at most 32 x 2^-24 of its variance).
// The backward pass forms z in the four rounded operations above, so that the border of the ReLU does not depend on how it is compiled.
#include <stdlib.h>
#include <type_traits>
#include "common.cuh"
#include "kernels.h"
#include "nn_ops.h"
#include "tc05.cuh"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int kThreads = 128;
constexpr int kPart = 32;                  // pixels of a part of the variance
enum Phase { FUSED = 0, SUMS = 1, APPLY = 2 };

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
  float eps;
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
};
template <>
struct Vec<bf16, 1> {
  bf16 a;
  __device__ __forceinline__ void load(const bf16* p) { a = *p; }
  __device__ __forceinline__ void get(float2 (&f)[1]) const { f[0] = make_float2(__bfloat162float(a), 0.f); }
  __device__ __forceinline__ void set(const float2 (&f)[1]) { a = __float2bfloat16(f[0].x); }
  __device__ __forceinline__ void store(bf16* p) const { *p = a; }
  __device__ __forceinline__ void relu() { a = __hmax_nan(a, __float2bfloat16(0.f)); }
};
template <>
struct Vec<float, 1> {
  float a;
  __device__ __forceinline__ void load(const float* p) { a = *p; }
  __device__ __forceinline__ void get(float2 (&f)[1]) const { f[0] = make_float2(a, 0.f); }
  __device__ __forceinline__ void set(const float2 (&f)[1]) { a = f[0].x; }
  __device__ __forceinline__ void store(float* p) const { *p = a; }
  __device__ __forceinline__ void relu() { a = a < 0.f ? 0.f : a; }
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

// A thread's own rows of vectors in shared memory, 16 bytes of every thread side by side
template <typename T>
struct Kept {
  uint8_t* base;
  static constexpr int kPieces = (int)sizeof(T) / 2;        // of 16 bytes
  static constexpr int kBytes = kThreads * 16 * kPieces;    // of a row
  __device__ __forceinline__ void fetch(int k, const T* src) const {
    const uint32_t at = tc05::smem_u32(base) + k * kBytes + threadIdx.x * 16;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) copy_async(at + i * kThreads * 16, (const uint8_t*)src + 16 * i);
  }
  __device__ __forceinline__ Vec<T, 8> get(int k) const {
    Vec<T, 8> v;
    uint4* w = (uint4*)&v;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) w[i] = *(const uint4*)(base + k * kBytes + i * kThreads * 16 + threadIdx.x * 16);
    return v;
  }
};
// Rows of a column as a thread reads them: from its own shared memory (ALL), or the first `keep` from there and the others
// where they lie
template <typename T, int W>
struct Rows {
  const T* at;
  long long step;
  Kept<T> kept;
  int keep;
  template <bool ALL>
  __device__ __forceinline__ Vec<T, W> get(int k) const {
    Vec<T, W> v;
    if constexpr (W == 8) {
      if (ALL || k < keep) v = kept.get(k); else v.load(at + k * step);
    } else {
      v.load(at + k * step);
    }
    return v;
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
template <typename F>
__device__ __forceinline__ void each_group(int gs, int lanes, F f) {
  const int at = threadIdx.x & (lanes - 1), per = kThreads / lanes;
  for (int g0 = 0; g0 < gs; g0 += per) {
    const int g = g0 + (int)threadIdx.x / lanes;
    if (g0 + ((int)threadIdx.x & ~31) / lanes < gs) f(min(g, gs - 1), at, g < gs);
  }
}

// finish(c, sum over the R threads of channel c of entry[i][r][v]), c = W v + i, by one thread a channel; entry is overwritten.
// Every thread of the block calls it; no barrier behind it.
template <int W, typename F>
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
    finish(v * W + e, s);
  }
}

__device__ __forceinline__ float silu(float z) { return __fdividef(z, 1.f + __expf(-z)); }

constexpr int kFlight = 4;                 // rows of a thread in flight

template <typename XT, typename YT, bool VEC, int PHASE>
__global__ void __launch_bounds__(kThreads, 4)
group_forward_kernel(const __grid_constant__ Dev d) {
  constexpr int W = VEC ? 8 : 1, H = (W + 1) / 2;
  extern __shared__ __align__(16) uint8_t smem[];
  const Place<W> p(d);
  const int cg = d.by_cg.d, gs = d.slice / cg, chunks = d.by_chunks.d;
  const bool narrow = d.V <= kThreads;                   // one column a thread
  float* mean_of = (float*)smem;                         // [slice], each: minus the mean, 1/std times weight and bias of a channel
  float* a_of = mean_of + d.slice;
  float* b_of = a_of + d.slice;
  float2* column = (float2*)smem;                        // [slice], before those: mean and squared differences of a channel
  float2* part = (float2*)(smem + ((d.slice * (narrow ? 12 : 8) + 15) & ~15));     // [gs]: the CTA's, then [gs] mean and 1/std of all
  float2* stat = part + gs;
  float* base_of = (float*)(stat + gs);                  // [slice], unless a thread has several columns
  float2* entry = (float2*)(base_of + (narrow ? (d.slice + 3) & ~3 : 0));          // [W][R][V]: sums of the threads about a column's base
  const int mine = p.mine();
  const long long at = (p.pixel + p.r) * d.ldx + p.c0 + p.v * W, step = (long long)d.R * d.ldx;
  Rows<XT, W> x = {(const XT*)d.x + at, step, {(uint8_t*)entry + d.entries}, 0};
  geeps_pdl_enter();

  if (PHASE != APPLY) {
    if (VEC && PHASE == FUSED) {
      x.keep = min(d.keep, mine);
      const XT* from = x.at;
      for (int k = 0; k < x.keep; ++k, from += step) x.kept.fetch(k, from);
      copies_done();
    }
    float2 mean[H], m2[H];
    auto pass = [&](auto all) {
      constexpr bool ALL = decltype(all)::value;
#pragma unroll
      for (int i = 0; i < H; ++i) mean[i] = m2[i] = both(0.f);
      int n = 0;
      for (int k = 0; k < mine;) {
        const int end = min(mine, k + kPart), count = end - k;
        float2 s[H], q[H], base[H];
        x.template get<ALL>(k).get(base);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          s[i] = q[i] = both(0.f);
          base[i] = make_float2(-base[i].x, -base[i].y);
        }
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
        int j = k + 1;
        for (; j + kFlight <= end; j += kFlight) {
          Vec<XT, W> in[kFlight];
#pragma unroll
          for (int u = 0; u < kFlight; ++u) in[u] = x.template get<ALL>(j + u);
#pragma unroll
          for (int u = 0; u < kFlight; ++u) add(in[u]);
        }
        for (; j < end; ++j) add(x.template get<ALL>(j));
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
      if (VEC && PHASE == FUSED && x.keep == mine) pass(std::true_type()); else pass(std::false_type());
      if (p.r == 0) {
#pragma unroll
        for (int i = 0; i < W; ++i) base_of[p.v * W + i] = value<W>(mean, i);
      }
      // the threads of a column about its base, the mean of the first of them
      __syncthreads();
      if (p.works) {
        const float n = (float)mine;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float e = value<W>(mean, i) - base_of[p.v * W + i];
          entry[(i * d.R + p.r) * d.V + p.v] = mine ? make_float2(n * e, fmaf(n * e, e, value<W>(m2, i))) : both(0.f);
        }
      }
      const float inv = p.rows ? __frcp_rn((float)p.rows) : 0.f;
      column_sums<W>(d, entry, [&](int c, float2 t) {
        column[c] = make_float2(fmaf(t.x, inv, base_of[c]), fmaxf(t.y - t.x * t.x * inv, 0.f));
      });
    } else {
      for (int v = threadIdx.x; v < d.V; v += kThreads, x.at += kThreads * W) {
        pass(std::false_type());
#pragma unroll
        for (int i = 0; i < W; ++i) column[v * W + i] = make_float2(value<W>(mean, i), value<W>(m2, i));
      }
      x.at = (const XT*)d.x + at;
    }
    __syncthreads();
    const int lanes = lanes_for(cg);
    const float each = __frcp_rn((float)cg);
    each_group(gs, lanes, [&](int g, int l, bool mine_g) {
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
  if (PHASE == FUSED) { if (chunks > 1) tc05::cluster_sync(); else __syncthreads(); }
  const int lanes = lanes_for(chunks);
  each_group(gs, lanes, [&](int g, int l, bool) {
    auto get = [&](int i) {
      if (PHASE == FUSED) return ld_cluster_f2(tc05::map_to_cta(tc05::smem_u32(part + g), i));
      return ((const float2*)d.sums)[((long long)p.image * chunks + i) * d.groups + p.slice * gs + g];
    };
    auto n_of = [&](int i) { return (float)max(0, min(d.rows, d.pixels - i * d.rows)) * cg; };
    float2 first = both(0.f);
    if (l < chunks) first = get(l);
    float s = n_of(l) * first.x;
    for (int i = l + lanes; i < chunks; i += lanes) s = fmaf(n_of(i), get(i).x, s);
    const float m = lane_sum(s, lanes) / total;
    float sq = first.y + n_of(l) * (first.x - m) * (first.x - m);
    for (int i = l + lanes; i < chunks; i += lanes) {
      const float2 t = get(i);
      sq += t.y + n_of(i) * (t.x - m) * (t.x - m);
    }
    sq = lane_sum(sq, lanes);
    if (l == 0) stat[g] = make_float2(m, __frcp_rn(__fsqrt_rn(sq / total + d.eps)));
  });
  __syncthreads();
  if (PHASE == FUSED && chunks > 1) tc05::cluster_arrive();      // nobody leaves while a peer still reads its sums
  if (d.stats != nullptr && p.chunk == 0)
    for (int g = threadIdx.x; g < gs; g += kThreads) ((float2*)d.stats)[(long long)p.image * d.groups + p.slice * gs + g] = stat[g];
  auto constant = [&](int c, float& mean, float& a, float& b) {
    const float2 s = stat[d.by_cg(c)];
    mean = -s.x;
    a = d.w != nullptr ? s.y * __ldg(d.w + p.c0 + c) : s.y;
    b = d.b != nullptr ? __ldg(d.b + p.c0 + c) : 0.f;
  };
  if (narrow) {
    for (int c = threadIdx.x; c < d.slice; c += kThreads) constant(c, mean_of[c], a_of[c], b_of[c]);
    __syncthreads();
  }
  const long long ostep = (long long)d.R * d.ldo;
  YT* y = (YT*)d.out + (p.pixel + p.r) * d.ldo + p.c0 + p.v * W;
  auto pass = [&](auto all, int v) {
    constexpr bool ALL = decltype(all)::value;
    float2 mean[H], a[H], b[H];
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
        f[i] = fma2(add2(f[i], mean[i]), a[i], b[i]);
        if (d.act == 2) f[i] = make_float2(silu(f[i].x), W > 1 ? silu(f[i].y) : 0.f);
      }
      Vec<YT, W> o;
      o.set(f);
      if (d.act == 1) o.relu();
      o.store(to);
      to += ostep;
    };
    int k = 0;
    for (; k + kFlight <= mine; k += kFlight) {
      Vec<XT, W> in[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) in[u] = x.template get<ALL>(k + u);
#pragma unroll
      for (int u = 0; u < kFlight; ++u) finish(in[u]);
    }
    for (; k < mine; ++k) finish(x.template get<ALL>(k));
  };
  if (narrow) {
    if (p.works) { if (VEC && PHASE == FUSED && x.keep == mine) pass(std::true_type(), p.v); else pass(std::false_type(), p.v); }
  } else {
    for (int v = threadIdx.x; v < d.V; v += kThreads, x.at += kThreads * W, y += kThreads * W) pass(std::false_type(), v);
  }
  if (PHASE == FUSED && chunks > 1) tc05::cluster_wait();
}

// act'(z) dy
__device__ __forceinline__ float slope(float z, float dy, int act) {
  if (act == 1) return z > 0.f ? dy : (z == z ? 0.f : z);
  const float g = __fdividef(1.f, 1.f + __expf(-z));
  return dy * (g * fmaf(z, 1.f - g, 1.f));
}

template <typename XT, typename YT, bool VEC, int PHASE>
__global__ void __launch_bounds__(kThreads, 4)
group_backward_kernel(const __grid_constant__ Dev d, float* channel_sums) {
  constexpr int W = VEC ? 8 : 1, H = (W + 1) / 2;
  constexpr int FLIGHT = kFlight / 2;
  extern __shared__ __align__(16) uint8_t smem[];
  const Place<W> p(d);
  const int cg = d.by_cg.d, gs = d.slice / cg, chunks = d.by_chunks.d;
  const bool narrow = d.V <= kThreads;
  float* mean_of = (float*)smem;                         // [slice], each: minus the mean, 1/std, weight and bias of a channel
  float* rstd_of = mean_of + d.slice;
  float* w_of = rstd_of + d.slice;
  float* b_of = w_of + d.slice;
  float2* column = (float2*)(smem + (narrow ? d.slice * 16 : 0));    // [slice]: sums of dz and dz n of a channel
  float2* part = column + d.slice;                       // [gs]: sums of dz w and dz w n of the CTA's pixels, then of all
  float2* whole = part + gs;
  float2* entry = (float2*)(((uintptr_t)(whole + gs) + 15) & ~(uintptr_t)15);      // [W][R][V], unless there is one thread a column
  const int mine = p.mine();
  const long long x_at = (p.pixel + p.r) * d.ldx + p.c0 + p.v * W, dy_at = (p.pixel + p.r) * d.lddy + p.c0 + p.v * W;
  Rows<XT, W> x = {(const XT*)d.x + x_at, (long long)d.R * d.ldx, {(uint8_t*)entry + d.entries}, 0};
  Rows<YT, W> dy = {(const YT*)d.dy + dy_at, (long long)d.R * d.lddy, {x.kept.base + (size_t)d.keep * Kept<XT>::kBytes}, 0};
  geeps_pdl_enter();
  if (VEC && PHASE == FUSED) {
    x.keep = dy.keep = min(d.keep, mine);
    const XT* xs = x.at;
    const YT* ds = dy.at;
    for (int k = 0; k < x.keep; ++k, xs += x.step, ds += dy.step) {
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
  float2 mean[H], rstd[H], w[H], b[H];
  auto constants = [&](int v) {
    if (narrow) {
      channel_values<W>(mean_of, v, mean);
      channel_values<W>(rstd_of, v, rstd);
      channel_values<W>(w_of, v, w);
      channel_values<W>(b_of, v, b);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * H; ++i) constant(v * W + (i < W ? i : 0), value<W>(mean, i), value<W>(rstd, i), value<W>(w, i), value<W>(b, i));
    }
  };
  // dz and n of a row
  auto row = [&](const Vec<XT, W>& xi, const Vec<YT, W>& di, float2 (&dz)[H], float2 (&n)[H]) {
    xi.get(n);
    di.get(dz);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      n[i] = mul2(add2(n[i], mean[i]), rstd[i]);
      if (d.act) {
        const float2 z = add2(mul2(n[i], w[i]), b[i]);
        dz[i] = make_float2(slope(z.x, dz[i].x, d.act), W > 1 ? slope(z.y, dz[i].y, d.act) : 0.f);
      }
    }
  };
  // f(x, dy) for all rows of a column, FLIGHT of them in flight
  auto rows = [&](auto all, auto f) {
    constexpr bool ALL = decltype(all)::value;
    int k = 0;
    for (; k + FLIGHT <= mine; k += FLIGHT) {
      Vec<XT, W> xi[FLIGHT];
      Vec<YT, W> di[FLIGHT];
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) { xi[u] = x.template get<ALL>(k + u); di[u] = dy.template get<ALL>(k + u); }
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) f(xi[u], di[u]);
    }
    for (; k < mine; ++k) f(x.template get<ALL>(k), dy.template get<ALL>(k));
  };
  const bool all_kept = VEC && PHASE == FUSED && x.keep == mine && narrow;
  if (PHASE != APPLY) {
    if (VEC && PHASE == FUSED) copies_done();
    auto pass = [&](auto all, int v) {
      constants(v);
      float2 sa[H], sb[H];
#pragma unroll
      for (int i = 0; i < H; ++i) sa[i] = sb[i] = both(0.f);
      rows(all, [&](const Vec<XT, W>& xi, const Vec<YT, W>& di) {
        float2 dz[H], n[H];
        row(xi, di, dz, n);
#pragma unroll
        for (int i = 0; i < H; ++i) { sa[i] = add2(sa[i], dz[i]); sb[i] = fma2(dz[i], n[i], sb[i]); }
      });
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float2 t = make_float2(value<W>(sa, i), value<W>(sb, i));
        if (d.R == 1) column[v * W + i] = t;
        else entry[(i * d.R + p.r) * d.V + v] = t;
      }
    };
    if (narrow) {
      if (p.works) { if (all_kept) pass(std::true_type(), p.v); else pass(std::false_type(), p.v); }
    } else {
      for (int v = threadIdx.x; v < d.V; v += kThreads, x.at += kThreads * W, dy.at += kThreads * W) pass(std::false_type(), v);
      x.at = (const XT*)d.x + x_at;
      dy.at = (const YT*)d.dy + dy_at;
    }
    if (d.R > 1) column_sums<W>(d, entry, [&](int c, float2 t) { column[c] = t; });
    __syncthreads();
    const int lanes = lanes_for(cg);
    each_group(gs, lanes, [&](int g, int l, bool mine_g) {
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
  if (PHASE == FUSED) { if (chunks > 1) tc05::cluster_sync(); else __syncthreads(); }
  const int lanes = lanes_for(chunks);
  each_group(gs, lanes, [&](int g, int l, bool) {
    float2 s = both(0.f);
    for (int i = l; i < chunks; i += lanes) {
      if (PHASE == FUSED) s = add2(s, ld_cluster_f2(tc05::map_to_cta(tc05::smem_u32(part + g), i)));
      else s = add2(s, ((const float2*)d.sums)[((long long)p.image * chunks + i) * d.groups + p.slice * gs + g]);
    }
    s.x = lane_sum(s.x, lanes);
    s.y = lane_sum(s.y, lanes);
    if (l == 0) whole[g] = make_float2(-s.x * scale, -s.y * scale);
  });
  // the image's sums of a channel: each CTA joins its share of the slice's
  if (PHASE == FUSED && channel_sums != nullptr)
    for (int c = p.chunk * kThreads + threadIdx.x; c < d.slice; c += chunks * kThreads) {
      float2 s = both(0.f);
      for (int i = 0; i < chunks; ++i) s = add2(s, ld_cluster_f2(tc05::map_to_cta(tc05::smem_u32(column + c), i)));
      ((float2*)channel_sums)[(long long)p.image * d.C + p.c0 + c] = s;
    }
  __syncthreads();
  if (PHASE == FUSED && chunks > 1) tc05::cluster_arrive();      // nobody leaves while a peer still reads its sums
  const long long ostep = (long long)d.R * d.ldo;
  XT* dx = (XT*)d.out + (p.pixel + p.r) * d.ldo + p.c0 + p.v * W;
  auto pass = [&](auto all, int v) {
    if (PHASE == APPLY || !narrow) constants(v);
    float2 ca[H], cb[H], wr[H];
#pragma unroll
    for (int i = 0; i < 2 * H; ++i) {
      const float2 s = whole[d.by_cg(v * W + (i < W ? i : 0))];
      value<W>(ca, i) = s.x * value<W>(rstd, i);
      value<W>(cb, i) = s.y * value<W>(rstd, i);
      value<W>(wr, i) = value<W>(w, i) * value<W>(rstd, i);
    }
    XT* to = dx;
    rows(all, [&](const Vec<XT, W>& xi, const Vec<YT, W>& di) {
      float2 dz[H], n[H];
      row(xi, di, dz, n);
#pragma unroll
      for (int i = 0; i < H; ++i) dz[i] = fma2(dz[i], wr[i], fma2(n[i], cb[i], ca[i]));
      Vec<XT, W> o;
      o.set(dz);
      o.store(to);
      to += ostep;
    });
  };
  if (narrow) {
    if (p.works) { if (all_kept) pass(std::true_type(), p.v); else pass(std::false_type(), p.v); }
  } else {
    for (int v = threadIdx.x; v < d.V; v += kThreads, x.at += kThreads * W, dy.at += kThreads * W, dx += kThreads * W) pass(std::false_type(), v);
  }
  if (PHASE == FUSED && chunks > 1) tc05::cluster_wait();
}

// Sums over `parts` rows of {dz, dz n} of the channels: 32 channels a block, its eight warps take every eighth row
__global__ void __launch_bounds__(256)
group_parameters_kernel(const float2* __restrict__ sums, long long parts, int C, float* dw, float* db) {
  geeps_pdl_enter();
  constexpr int WARPS = 8;
  __shared__ float2 sh[WARPS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float2 s = make_float2(0.f, 0.f);
  if (c < C)
    for (long long i = warp; i < parts; i += WARPS) {
      const float2 t = sums[i * C + c];
      s.x += t.x;
      s.y += t.y;
    }
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < WARPS; ++i) { s.x += sh[i][lane].x; s.y += sh[i][lane].y; }
    if (db != nullptr) db[c] = s.x;
    if (dw != nullptr) dw[c] = s.y;
  }
}

// ---------------- host side ----------------
struct Shape { int vec, fused, slice, slices, chunks, rows, keep, blocks, V, R, entries; size_t smem; };

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

constexpr int kMostChunks = 8;             // CTAs of a cluster
constexpr size_t kSmem = 200 * 1024;

// Shared memory that does not depend on the pixels kept
size_t fixed_bytes(const Shape& s, int cg, bool backward) {
  const size_t gs = s.slice / cg, narrow = s.V <= kThreads;
  if (backward) return (size_t)s.slice * (narrow ? 24 : 8) + gs * 16 + 16;
  return ((s.slice * (narrow ? 12 : 8) + 15) & ~15) + gs * 16 + (narrow ? ((s.slice + 3) & ~3) * 4 : 0);
}

Shape choose(int images, int pixels, int C, int groups, bool backward, bool vec, int xsize, int ysize) {
  Shape s = {};
  const int cg = C / groups, W = vec ? 8 : 1, sms = geeps_sm_count();
  const int unit = cg / gcd(cg, W) * W;          // channels of the narrowest slice
  const char* kbs = getenv("GN_KB"); const int kb = kbs ? atoi(kbs) : 48; const char* fz = getenv("GN_FUSED"); const char* bl = getenv("GN_BLOCKS"); const char* sl = getenv("GN_SLICE");  // DEV
  s.vec = vec;
  // slices of 64 channels and more: whole sectors of a pixel
  const int least = vec ? (sl ? atoi(sl) : 64) : 64;
  int n = 1;
  while (unit * n < C && (unit * n < least || C / unit % n)) ++n;
  s.slice = unit * n;
  s.slices = C / s.slice;
  s.V = s.slice / W;
  s.R = s.V < kThreads ? kThreads / s.V : 1;
  s.entries = (backward ? s.R > 1 : s.V <= kThreads) ? s.R * s.slice * 8 : 0;
  s.entries = (s.entries + 15) & ~15;
  const int row_bytes = kThreads * 16 * (vec ? (xsize / 2 + (backward ? ysize / 2 : 0)) : 0);      // of all threads' kept rows
  const long long items = (long long)images * s.slices;
  const long long bytes = (long long)pixels * s.slice * (xsize + (backward ? ysize : 0));
  int chunks = 1;
  while (chunks < kMostChunks && bytes / chunks > kb * 1024) ++chunks;
  while (chunks < kMostChunks && items * chunks < sms && pixels / (chunks * 2) >= s.R) chunks *= 2;
  if (chunks > kMostChunks) chunks = kMostChunks;
  s.fused = 1;
  if (fz ? !atoi(fz) : items * chunks < sms / 2 && pixels > chunks * 4LL * s.R) {
    // too few items: two launches over as many chunks as fill the machine
    s.fused = 0;
    long long want = ((bl ? atoi(bl) : 4LL) * sms + items - 1) / items, most = (pixels + s.R - 1) / s.R;
    chunks = (int)(want < most ? want : most);
  }
  s.rows = (pixels + chunks - 1) / chunks;
  s.chunks = s.fused ? chunks : (pixels + s.rows - 1) / s.rows;
  const size_t fixed = fixed_bytes(s, cg, backward) + s.entries;
  int keep = vec && s.V <= kThreads && s.fused ? (s.rows + s.R - 1) / s.R : 0;
  while (keep > 0 && fixed + (size_t)keep * row_bytes > kSmem) --keep;
  s.keep = keep;
  s.smem = fixed + (size_t)keep * row_bytes;
  s.blocks = items * s.chunks > 0x7fffffffLL ? 0 : (int)(items * s.chunks);
  return s;
}

template <typename K, typename... A>
int launch(K kernel, const Shape& s, bool cluster, cudaStream_t st, A&&... args) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)s.blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)s.chunks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster && s.chunks > 1 ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<A&&>(args)...);
}

template <typename XT, typename YT, bool VEC>
int run(const GeepsGroupNorm& k, const Shape& s, const Dev& d, bool backward, cudaStream_t st) {
  int e;
  if (!backward) {
    if (s.fused) return launch(group_forward_kernel<XT, YT, VEC, FUSED>, s, true, st, d);
    e = launch(group_forward_kernel<XT, YT, VEC, SUMS>, s, false, st, d);
    return e ? e : launch(group_forward_kernel<XT, YT, VEC, APPLY>, s, false, st, d);
  }
  const bool want = k.dweight != nullptr || k.dbias != nullptr;
  // group sums of the chunks (two launches only), then the channels' sums of the images or chunks
  const long long parts = (long long)k.images * (s.fused ? 1 : s.chunks);
  float* channel = want ? k.work + (s.fused ? 0 : parts * k.groups * 2) : nullptr;
  if (s.fused) {
    e = launch(group_backward_kernel<XT, YT, VEC, FUSED>, s, true, st, d, channel);
  } else {
    e = launch(group_backward_kernel<XT, YT, VEC, SUMS>, s, false, st, d, channel);
    if (!e) e = launch(group_backward_kernel<XT, YT, VEC, APPLY>, s, false, st, d, channel);
  }
  if (e || !want) return e;
  geeps_launch(group_parameters_kernel, dim3((unsigned)((k.C + 31) / 32)), dim3(256), 0, st, (const float2*)channel, parts, k.C, k.dweight, k.dbias);
  return (int)cudaGetLastError();
}

bool vectors(const GeepsGroupNorm& k, bool backward) {
  const int xs = k.x_fp32 ? 4 : 2, ys = k.y_fp32 ? 4 : 2;
  auto ok = [](const void* p, long long ld, int size) { return ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0; };
  return k.C % 8 == 0 && ok(k.x, k.ldx, xs) && (backward ? ok(k.dy, k.lddy, ys) && ok(k.dx, k.lddx, xs) : ok(k.y, k.ldy, ys));
}

int check(const GeepsGroupNorm* k, bool backward) {
  if (!k || k->images < 0 || k->pixels < 0 || (k->y_fp32 && !k->x_fp32) || !(k->eps >= 0.f) || k->act < 0 || k->act > 2) return (int)cudaErrorInvalidValue;
  if (k->C < 1 || k->C > 16384) return GEEPS_ERR_NORM_CHANNELS;
  if (k->groups < 1 || k->C % k->groups) return GEEPS_ERR_GROUPS;
  if (k->images * k->pixels > (1LL << 30)) return (int)cudaErrorInvalidValue;
  const long long rows = k->images * k->pixels;
  const int xs = k->x_fp32 ? 4 : 2, ys = k->y_fp32 ? 4 : 2;
  struct Range { const void* at; long long bytes; bool written; long long pitch; int align; };      // pitch: of rows, in bytes; 0: none
  auto span = [&](long long ld, int size) { return rows ? ((rows - 1) * ld + k->C) * size : 0; };
  if (k->ldx < k->C || (backward ? k->lddy < k->C || k->lddx < k->C : k->ldy < k->C)) return (int)cudaErrorInvalidValue;
  const long long stats = k->images * k->groups * 8, work = geeps_group_norm_work(k->images, k->pixels, k->C, k->groups) * 4;
  const Range all[] = {
      {k->x, span(k->ldx, xs), false, k->ldx * xs, xs},
      {backward ? k->dy : nullptr, span(k->lddy, ys), false, k->lddy * ys, ys},
      {backward ? k->dx : k->y, backward ? span(k->lddx, xs) : span(k->ldy, ys), true, backward ? k->lddx * xs : k->ldy * ys, backward ? xs : ys},
      {k->weight, 4LL * k->C, false, 0, 4}, {k->bias, 4LL * k->C, false, 0, 4},
      {k->stats, stats, !backward, 0, 8}, {k->work, work, true, 0, 8},
      {backward ? k->dweight : nullptr, 4LL * k->C, true, 0, 4}, {backward ? k->dbias : nullptr, 4LL * k->C, true, 0, 4}};
  if (rows && (!k->x || !(backward ? (const void*)k->dx : k->y) || (backward && (!k->dy || !k->stats)) || !k->work)) return (int)cudaErrorInvalidValue;
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
  d.keep = s.keep; d.V = s.V; d.R = s.R; d.entries = s.entries; d.eps = k->eps;
  d.by_chunks = Divide(s.chunks); d.by_slices = Divide(s.slices); d.by_V = Divide(s.V); d.by_cg = Divide(k->C / k->groups);
  if (k->y_fp32) return vec ? run<float, float, true>(*k, s, d, backward, st) : run<float, float, false>(*k, s, d, backward, st);
  if (k->x_fp32) return vec ? run<float, bf16, true>(*k, s, d, backward, st) : run<float, bf16, false>(*k, s, d, backward, st);
  return vec ? run<bf16, bf16, true>(*k, s, d, backward, st) : run<bf16, bf16, false>(*k, s, d, backward, st);
}

}  // namespace

extern "C" {

long long geeps_group_norm_work(long long images, long long pixels, int C, int groups) {
  // at most 2 SMs' worth of chunks beyond one an image, each with its groups' and channels' sums
  if (images <= 0 || pixels <= 0 || C <= 0 || groups <= 0) return 2;
  return (images + 20LL * geeps_sm_count() + 2) * 2 * ((long long)C + groups);
}

int geeps_group_norm_forward(const GeepsGroupNorm* p, void* stream) { return call(p, false, stream); }
int geeps_group_norm_backward(const GeepsGroupNorm* p, void* stream) { return call(p, true, stream); }

int geeps_group_norm_shape(long long images, long long pixels, int C, int groups, int backward, int vec, int x_fp32, int y_fp32, int* out) {
  if (images < 1 || pixels < 1 || C < 1 || groups < 1 || C % groups || (vec && C % 8)) return (int)cudaErrorInvalidValue;
  const Shape s = choose((int)images, (int)pixels, C, groups, backward, vec, x_fp32 ? 4 : 2, y_fp32 ? 4 : 2);
  out[0] = s.fused; out[1] = s.slice; out[2] = s.chunks; out[3] = s.rows; out[4] = s.keep; out[5] = s.blocks; out[6] = (int)s.smem; out[7] = kThreads;
  return 0;
}

}  // extern "C"
