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
#include "common.cuh"
#include "kernels.h"
#include "nn_ops.h"
#include "tc05.cuh"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPart = 32;                  // pixels of a part of the variance
enum Phase { FUSED = 0, SUMS = 1, APPLY = 2 };

struct Dev {
  const void *x, *dy;
  void* out;                               // y or dx
  const float *w, *b;
  float *stats, *sums;                     // sums: workspace
  long long ldx, lddy, ldo;
  int pixels, C, groups, cg, slice, slices, chunks, rows, act, keep;      // rows: pixels of a chunk; keep: pixels a thread keeps
  float eps;
};

// ---- vectors of eight (or single) values ----
template <typename T, int W>
struct Vec;
template <>
struct Vec<bf16, 8> {
  uint4 a;
  __device__ __forceinline__ void load(const bf16* p) { a = *(const uint4*)p; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    a = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
  __device__ __forceinline__ void store(bf16* p) const { *(uint4*)p = a; }
};
template <>
struct Vec<float, 8> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = ld_f4(p); b = ld_f4(p + 4); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&f)[8]) { a = make_float4(f[0], f[1], f[2], f[3]); b = make_float4(f[4], f[5], f[6], f[7]); }
  __device__ __forceinline__ void store(float* p) const { st_f4(p, a); st_f4(p + 4, b); }
};
template <>
struct Vec<bf16, 1> {
  bf16 a;
  __device__ __forceinline__ void load(const bf16* p) { a = *p; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = __bfloat162float(a); }
  __device__ __forceinline__ void set(const float (&f)[1]) { a = __float2bfloat16(f[0]); }
  __device__ __forceinline__ void store(bf16* p) const { *p = a; }
};
template <>
struct Vec<float, 1> {
  float a;
  __device__ __forceinline__ void load(const float* p) { a = *p; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = a; }
  __device__ __forceinline__ void set(const float (&f)[1]) { a = f[0]; }
  __device__ __forceinline__ void store(float* p) const { *p = a; }
};
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

__device__ __forceinline__ float ld_cluster_f(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// What a CTA works on and which part of it a thread has
template <int W>
struct Place {
  int image, slice, chunk, first, rows, c0, V, R, v, r;        // first: pixel of the chunk; c0: channel of the slice
  long long pixel;                                             // of the chunk, among all images
  __device__ __forceinline__ Place(const Dev& d) {
    int i = (int)blockIdx.x;
    chunk = i % d.chunks; i /= d.chunks;
    slice = i % d.slices;
    image = i / d.slices;
    first = chunk * d.rows;
    rows = min(d.rows, d.pixels - first);
    if (rows < 0) rows = 0;
    c0 = slice * d.slice;
    V = d.slice / W;
    R = V < kThreads ? kThreads / V : 1;
    v = V < kThreads ? (int)threadIdx.x % V : (int)threadIdx.x;
    r = V < kThreads ? (int)threadIdx.x / V : 0;
    pixel = (long long)image * d.pixels + first;
  }
  __device__ __forceinline__ bool works() const { return r < R; }
  // rows of the thread that is the r-th of a column
  __device__ __forceinline__ int count(int of) const { return of < rows ? (rows - of + R - 1) / R : 0; }
};

__device__ __forceinline__ float warp_sum(float a) {
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  return a;
}

// Mean and 1/std of every group of the slice from those of the parts: part i of `parts` has n(i) values, get(i, g) its mean
// and squared differences.  One thread a group.
template <typename N, typename G>
__device__ __forceinline__ float2 join(int parts, float total, float eps, N n, G get) {
  float mean = 0.f, m2 = 0.f;
  for (int i = 0; i < parts; ++i) mean += n(i) * get(i).x;
  mean /= total;
  for (int i = 0; i < parts; ++i) {
    const float2 p = get(i);
    m2 += p.y + n(i) * (p.x - mean) * (p.x - mean);
  }
  return make_float2(mean, __frcp_rn(__fsqrt_rn(m2 / total + eps)));
}

__device__ __forceinline__ float activate(float z, int act) {
  if (act == 1) return z < 0.f ? 0.f : z;               // a NaN stays one
  if (act == 2) return __fdividef(z, 1.f + __expf(-z));
  return z;
}

template <typename XT, typename YT, bool VEC, int PHASE>
__global__ void __launch_bounds__(kThreads)
group_forward_kernel(const Dev d) {
  constexpr int W = VEC ? 8 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  const Place<W> p(d);
  const int gs = d.slice / d.cg, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wide = p.R * d.slice;                        // entries of the threads' parts
  float2* part = (float2*)smem;                          // [gs]: the CTA's, then [gs] mean and 1/std of all
  float2* stat = part + gs;
  float* mean_of = (float*)(stat + gs);                  // [R][slice], and so the squared differences
  float* m2_of = mean_of + wide;
  Kept<XT> kept = {(uint8_t*)(((uintptr_t)(m2_of + wide) + 15) & ~(uintptr_t)15)};
  const int mine = p.works() ? p.count(p.r) : 0, keep = VEC ? min(d.keep, mine) : 0;
  const XT* x = (const XT*)d.x + (p.pixel + p.r) * d.ldx + p.c0;
  YT* y = (YT*)d.out + (p.pixel + p.r) * d.ldo + p.c0;
  const long long step = (long long)p.R * d.ldx, ostep = (long long)p.R * d.ldo;
  geeps_pdl_enter();

  if (PHASE != APPLY) {
    if (VEC) {
      for (int k = 0; k < keep; ++k) kept.fetch(k, (const XT*)x + k * step + p.v * 8);
      copies_done();
    }
    for (int v = p.v; v < p.V && p.works(); v += kThreads) {
      float mean[W], m2[W];
#pragma unroll
      for (int i = 0; i < W; ++i) mean[i] = m2[i] = 0.f;
      int n = 0;
      for (int k = 0; k < mine;) {
        const int end = min(mine, k + kPart), count = end - k;
        float s[W], q[W], base[W];
#pragma unroll
        for (int i = 0; i < W; ++i) s[i] = q[i] = base[i] = 0.f;
        for (int j = k; j < end; ++j) {
          Vec<XT, W> in;
          if constexpr (VEC) { if (j < keep) in = kept.get(j); else in.load(x + j * step + v * W); } else in.load(x + j * step + v);
          float f[W];
          in.get(f);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            if (j == k) base[i] = f[i];
            const float e = f[i] - base[i];
            s[i] += e;
            q[i] = fmaf(e, e, q[i]);
          }
        }
        const float inv = 1.f / count, share = (float)count / (n + count), weight = n * share;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float m = base[i] + s[i] * inv, delta = m - mean[i];
          m2[i] += fmaxf(q[i] - s[i] * s[i] * inv, 0.f) + delta * delta * weight;
          mean[i] += delta * share;
        }
        n += count;
        k = end;
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        mean_of[p.r * d.slice + v * W + i] = mean[i];
        m2_of[p.r * d.slice + v * W + i] = m2[i];
      }
    }
    __syncthreads();
    const float total = (float)p.rows * d.cg;
    for (int g = warp; g < gs; g += kWarps) {
      float s = 0.f, m2 = 0.f;
      for (int r = 0; r < p.R; ++r) {
        const float n = (float)p.count(r);
        for (int c = lane; c < d.cg; c += 32) s = fmaf(n, mean_of[r * d.slice + g * d.cg + c], s);
      }
      const float mean = total > 0.f ? warp_sum(s) / total : 0.f;
      for (int r = 0; r < p.R; ++r) {
        const float n = (float)p.count(r);
        for (int c = lane; c < d.cg; c += 32) {
          const float e = mean_of[r * d.slice + g * d.cg + c] - mean;
          if (n > 0.f) m2 += m2_of[r * d.slice + g * d.cg + c] + n * e * e;
        }
      }
      m2 = warp_sum(m2);
      if (lane == 0) part[g] = make_float2(mean, m2);
    }
  }
  if (PHASE == SUMS) {
    __syncthreads();
    for (int g = threadIdx.x; g < gs; g += kThreads)
      ((float2*)d.sums)[((long long)p.image * d.chunks + p.chunk) * d.groups + p.slice * gs + g] = part[g];
    return;
  }
  const float total = (float)d.pixels * d.cg;
  auto n_of = [&](int i) { return (float)max(0, min(d.rows, d.pixels - i * d.rows)) * d.cg; };
  if (PHASE == FUSED) {
    tc05::cluster_sync();
    for (int g = threadIdx.x; g < gs; g += kThreads)
      stat[g] = join(d.chunks, total, d.eps, n_of, [&](int i) {
        const uint32_t at = tc05::map_to_cta(tc05::smem_u32(part + g), i);
        return make_float2(ld_cluster_f(at), ld_cluster_f(at + 4));
      });
  } else {
    for (int g = threadIdx.x; g < gs; g += kThreads)
      stat[g] = join(d.chunks, total, d.eps, n_of, [&](int i) {
        return ((const float2*)d.sums)[((long long)p.image * d.chunks + i) * d.groups + p.slice * gs + g];
      });
  }
  __syncthreads();
  if (d.stats != nullptr && p.chunk == 0)
    for (int g = threadIdx.x; g < gs; g += kThreads) ((float2*)d.stats)[(long long)p.image * d.groups + p.slice * gs + g] = stat[g];
  for (int v = p.v; v < p.V && p.works(); v += kThreads) {
    float mean[W], a[W], b[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int c = v * W + i;
      const float2 s = stat[c / d.cg];
      mean[i] = s.x;
      a[i] = d.w != nullptr ? s.y * d.w[p.c0 + c] : s.y;
      b[i] = d.b != nullptr ? d.b[p.c0 + c] : 0.f;
    }
    for (int k = 0; k < mine; ++k) {
      Vec<XT, W> in;
      if constexpr (VEC) { if (PHASE == FUSED && k < keep) in = kept.get(k); else in.load(x + k * step + v * W); } else in.load(x + k * step + v);
      float f[W];
      in.get(f);
#pragma unroll
      for (int i = 0; i < W; ++i) f[i] = activate(fmaf(f[i] - mean[i], a[i], b[i]), d.act);
      Vec<YT, W> o;
      o.set(f);
      o.store(y + k * ostep + v * W);
    }
  }
  if (PHASE == FUSED) tc05::cluster_sync();      // nobody leaves while a peer still reads its sums
}

// dz and n of a value
__device__ __forceinline__ float slope(float z, float dy, int act) {
  if (act == 1) return z > 0.f ? dy : (z == z ? 0.f : z);
  if (act == 2) {
    const float g = __fdividef(1.f, 1.f + __expf(-z));
    return dy * (g * fmaf(z, 1.f - g, 1.f));
  }
  return dy;
}

template <typename XT, typename YT, bool VEC, int PHASE>
__global__ void __launch_bounds__(kThreads)
group_backward_kernel(const Dev d, float* channel_sums) {
  constexpr int W = VEC ? 8 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  const Place<W> p(d);
  const int gs = d.slice / d.cg, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wide = p.R > 1 ? p.R * d.slice : 0;           // with one thread a column there is nothing to add
  float2* part = (float2*)smem;                          // [gs]: sums of dz w and dz w n of the CTA's pixels, then of all
  float2* whole = part + gs;
  float2* column = whole + gs;                           // [slice]: sums of dz and dz n of a channel
  float* a_of = (float*)(column + d.slice);              // [R][slice]
  float* b_of = a_of + wide;
  Kept<XT> kept_x = {(uint8_t*)(((uintptr_t)(b_of + wide) + 15) & ~(uintptr_t)15)};
  Kept<YT> kept_dy = {kept_x.base + (size_t)d.keep * Kept<XT>::kBytes};
  const int mine = p.works() ? p.count(p.r) : 0, keep = VEC ? min(d.keep, mine) : 0;
  const XT* x = (const XT*)d.x + (p.pixel + p.r) * d.ldx + p.c0;
  const YT* dy = (const YT*)d.dy + (p.pixel + p.r) * d.lddy + p.c0;
  XT* dx = (XT*)d.out + (p.pixel + p.r) * d.ldo + p.c0;
  const long long step = (long long)p.R * d.ldx, dstep = (long long)p.R * d.lddy, ostep = (long long)p.R * d.ldo;
  geeps_pdl_enter();
  if (VEC && PHASE == FUSED)
    for (int k = 0; k < keep; ++k) {
      kept_x.fetch(k, x + k * step + p.v * 8);
      kept_dy.fetch(k, dy + k * dstep + p.v * 8);
    }
  const float2* stats = (const float2*)d.stats + (long long)p.image * d.groups + p.slice * gs;
  float mean[W], rstd[W], w[W], b[W];
  auto constants = [&](int v) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int c = v * W + i;
      const float2 s = stats[c / d.cg];
      mean[i] = s.x;
      rstd[i] = s.y;
      w[i] = d.w != nullptr ? d.w[p.c0 + c] : 1.f;
      b[i] = d.b != nullptr ? d.b[p.c0 + c] : 0.f;
    }
  };
  // dz and n of row k
  auto row = [&](int k, int v, float (&dz)[W], float (&n)[W]) {
    Vec<XT, W> xi;
    Vec<YT, W> di;
    if constexpr (VEC) {
      if (PHASE == FUSED && k < keep) { xi = kept_x.get(k); di = kept_dy.get(k); }
      else { xi.load(x + k * step + v * W); di.load(dy + k * dstep + v * W); }
    } else {
      xi.load(x + k * step + v);
      di.load(dy + k * dstep + v);
    }
    xi.get(n);
    di.get(dz);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      n[i] = __fmul_rn(__fsub_rn(n[i], mean[i]), rstd[i]);
      if (d.act) dz[i] = slope(__fadd_rn(__fmul_rn(n[i], w[i]), b[i]), dz[i], d.act);
    }
  };
  if (VEC && PHASE == FUSED) copies_done();
  if (PHASE != APPLY) {
    for (int v = p.v; v < p.V && p.works(); v += kThreads) {
      constants(v);
      float sa[W], sb[W];
#pragma unroll
      for (int i = 0; i < W; ++i) sa[i] = sb[i] = 0.f;
      for (int k = 0; k < mine; ++k) {
        float dz[W], n[W];
        row(k, v, dz, n);
#pragma unroll
        for (int i = 0; i < W; ++i) { sa[i] += dz[i]; sb[i] = fmaf(dz[i], n[i], sb[i]); }
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (p.R == 1) column[v * W + i] = make_float2(sa[i], sb[i]);
        else { a_of[p.r * d.slice + v * W + i] = sa[i]; b_of[p.r * d.slice + v * W + i] = sb[i]; }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < d.slice && p.R > 1; c += kThreads) {
      float sa = 0.f, sb = 0.f;
      for (int r = 0; r < p.R; ++r) { sa += a_of[r * d.slice + c]; sb += b_of[r * d.slice + c]; }
      column[c] = make_float2(sa, sb);
    }
    __syncthreads();
    for (int g = warp; g < gs; g += kWarps) {
      float sa = 0.f, sb = 0.f;
      for (int c = lane; c < d.cg; c += 32) {
        const float2 s = column[g * d.cg + c];
        const float wc = d.w != nullptr ? d.w[p.c0 + g * d.cg + c] : 1.f;
        sa = fmaf(s.x, wc, sa);
        sb = fmaf(s.y, wc, sb);
      }
      sa = warp_sum(sa);
      sb = warp_sum(sb);
      if (lane == 0) part[g] = make_float2(sa, sb);
    }
  }
  if (PHASE == SUMS) {
    __syncthreads();
    const long long at = (long long)p.image * d.chunks + p.chunk;
    for (int g = threadIdx.x; g < gs; g += kThreads) ((float2*)d.sums)[at * d.groups + p.slice * gs + g] = part[g];
    if (channel_sums != nullptr)
      for (int c = threadIdx.x; c < d.slice; c += kThreads) ((float2*)channel_sums)[at * d.C + p.c0 + c] = column[c];
    return;
  }
  const float scale = 1.f / ((float)d.pixels * d.cg);
  if (PHASE == FUSED) {
    tc05::cluster_sync();
    for (int g = threadIdx.x; g < gs; g += kThreads) {
      float2 s = make_float2(0.f, 0.f);
      for (int i = 0; i < d.chunks; ++i) {
        const uint32_t at = tc05::map_to_cta(tc05::smem_u32(part + g), i);
        s.x += ld_cluster_f(at);
        s.y += ld_cluster_f(at + 4);
      }
      whole[g] = make_float2(s.x * scale, s.y * scale);
    }
    // the image's sums of a channel: each CTA joins its share of the slice's
    if (channel_sums != nullptr)
      for (int c = p.chunk * kThreads + threadIdx.x; c < d.slice; c += d.chunks * kThreads) {
        float2 s = make_float2(0.f, 0.f);
        for (int i = 0; i < d.chunks; ++i) {
          const uint32_t at = tc05::map_to_cta(tc05::smem_u32(column + c), i);
          s.x += ld_cluster_f(at);
          s.y += ld_cluster_f(at + 4);
        }
        ((float2*)channel_sums)[(long long)p.image * d.C + p.c0 + c] = s;
      }
  } else {
    for (int g = threadIdx.x; g < gs; g += kThreads) {
      float2 s = make_float2(0.f, 0.f);
      for (int i = 0; i < d.chunks; ++i) {
        const float2 t = ((const float2*)d.sums)[((long long)p.image * d.chunks + i) * d.groups + p.slice * gs + g];
        s.x += t.x;
        s.y += t.y;
      }
      whole[g] = make_float2(s.x * scale, s.y * scale);
    }
  }
  __syncthreads();
  for (int v = p.v; v < p.V && p.works(); v += kThreads) {
    if (PHASE == APPLY || p.V > kThreads) constants(v);
    float ca[W], cb[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float2 s = whole[(v * W + i) / d.cg];
      ca[i] = s.x;
      cb[i] = s.y;
    }
    for (int k = 0; k < mine; ++k) {
      float dz[W], n[W];
      row(k, v, dz, n);
#pragma unroll
      for (int i = 0; i < W; ++i) dz[i] = rstd[i] * (fmaf(dz[i], w[i], -ca[i]) - n[i] * cb[i]);
      Vec<XT, W> o;
      o.set(dz);
      o.store(dx + k * ostep + v * W);
    }
  }
  if (PHASE == FUSED) tc05::cluster_sync();      // nobody leaves while a peer still reads its sums
}

// Sums over `parts` rows of {dz, dz n} of the channels: 32 channels a block, its warps take every kWarps-th row
__global__ void __launch_bounds__(kThreads)
group_parameters_kernel(const float2* __restrict__ sums, long long parts, int C, float* dw, float* db) {
  geeps_pdl_enter();
  __shared__ float2 sh[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float2 s = make_float2(0.f, 0.f);
  if (c < C)
    for (long long i = warp; i < parts; i += kWarps) {
      const float2 t = sums[i * C + c];
      s.x += t.x;
      s.y += t.y;
    }
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < kWarps; ++i) { s.x += sh[i][lane].x; s.y += sh[i][lane].y; }
    if (db != nullptr) db[c] = s.x;
    if (dw != nullptr) dw[c] = s.y;
  }
}

// ---------------- host side ----------------
struct Shape { int vec, fused, slice, slices, chunks, rows, keep, blocks; size_t smem; };

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

constexpr int kMostChunks = 8;             // CTAs of a cluster
constexpr size_t kSmem = 200 * 1024;

Shape choose(int images, int pixels, int C, int groups, int backward, bool vec, int xsize, int ysize) {
  Shape s = {};
  const int cg = C / groups, W = vec ? 8 : 1, sms = geeps_sm_count();
  const int unit = cg / gcd(cg, W) * W;          // channels of the narrowest slice
  s.vec = vec;
  // slices of 64 channels and more: whole sectors of a pixel
  int n = 1;
  while (unit * n < 64 && C % (unit * (n + 1)) == 0 && unit * n < C) ++n;
  s.slice = unit * n;
  while (C % s.slice) s.slice += unit;
  s.slices = C / s.slice;
  const int V = s.slice / W, R = V < kThreads ? kThreads / V : 1;
  const int row_bytes = kThreads * 16 * (vec ? (xsize / 2 + (backward ? ysize / 2 : 0)) : 0);      // of all threads' kept rows
  const long long items = (long long)images * s.slices;
  // CTAs of 48 KB of an item
  const long long bytes = (long long)pixels * s.slice * (xsize + (backward ? ysize : 0));
  int chunks = 1;
  while (chunks < kMostChunks && bytes / chunks > 48 * 1024) chunks *= 2;
  while (chunks < kMostChunks && items * chunks < sms && pixels / (chunks * 2) >= R) chunks *= 2;
  s.fused = 1;
  if (items * chunks < sms / 2 && pixels > chunks * 4LL * R) {
    // too few items: two launches over as many chunks as fill the machine
    s.fused = 0;
    long long want = (2LL * sms + items - 1) / items, most = (pixels + R - 1) / R;
    chunks = (int)(want < most ? want : most);
  }
  s.rows = (pixels + chunks - 1) / chunks;
  s.chunks = s.fused ? chunks : (pixels + s.rows - 1) / s.rows;
  const size_t fixed = (size_t)(2 * (s.slice / cg) + (backward ? s.slice : 0)) * 8 + (backward && R == 1 ? 0 : (size_t)R * s.slice * 8) + 16;
  int keep = vec && V <= kThreads && s.fused ? (s.rows + R - 1) / R : 0;
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
  cfg.numAttrs = cluster ? 1 : 0;
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
  geeps_launch(group_parameters_kernel, dim3((unsigned)((k.C + 31) / 32)), dim3(kThreads), 0, st, (const float2*)channel, parts, k.C, k.dweight, k.dbias);
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
  d.pixels = (int)k->pixels; d.C = k->C; d.groups = k->groups; d.cg = k->C / k->groups;
  d.slice = s.slice; d.slices = s.slices; d.chunks = s.chunks; d.rows = s.rows; d.act = k->act; d.keep = s.keep; d.eps = k->eps;
  if (k->y_fp32) return vec ? run<float, float, true>(*k, s, d, backward, st) : run<float, float, false>(*k, s, d, backward, st);
  if (k->x_fp32) return vec ? run<float, bf16, true>(*k, s, d, backward, st) : run<float, bf16, false>(*k, s, d, backward, st);
  return vec ? run<bf16, bf16, true>(*k, s, d, backward, st) : run<bf16, bf16, false>(*k, s, d, backward, st);
}

}  // namespace

extern "C" {

long long geeps_group_norm_work(long long images, long long pixels, int C, int groups) {
  // at most 2 SMs' worth of chunks beyond one an image, each with its groups' and channels' sums
  if (images <= 0 || pixels <= 0 || C <= 0 || groups <= 0) return 2;
  return (images + 2LL * geeps_sm_count() + 2) * 2 * ((long long)C + groups);
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
