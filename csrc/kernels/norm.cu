// Norms over the channels of a row (a pixel or a token), before and after a residual block, and everything that stands
// between two blocks in one pass over the rows:
//
//   z = post(x)                                   LayerNorm or RMSNorm of the block's output, or x itself
//   h = res + scale * g * z                       residual connection; scale per channel, gate g per pixel or per image
//   y = pre(h)                                    the norm in front of the next block
//
//   n = (x - mean) * rstd, rstd = 1 / sqrt(mean_c (x - mean)^2 + eps), post(x) = n * weight + bias; RMSNorm has mean = 0.
//
// Backward, from dout (the gradient of h by other ways) and dy, with everything saved forward:
//   a = dy * w2,  dh = dout + rstd2 (a - mean_c a - n2 mean_c(a n2)),  dw2 = sum dy n2,  db2 = sum dy
//   e = dh g s w, dx = rstd (e - mean_c e - n mean_c(e n))              (RMSNorm: without the mean_c of a and e)
// scale, weight and bias are constants of a column, so their gradients come from two column sums,
//   A = sum_p dh g n,  B = sum_p dh g:   dw = s A,  db = s B,  dscale = w A + b B,
// and a gate per image from the same two sums over its rows without the gate, u and v: dgate = s (w u + b v), A = sum g u.
//
// A row is the work of a slot of threads that own its columns, eight a vector: the row is read once, stays in registers
// and its sums are formed there (two passes over registers for a variance: nothing cancels).  What belongs to a column is
// loaded once and column sums are kept in registers over all rows of a slot; slots meet in shared memory and blocks in a
// second launch, in a fixed order: results repeat bit for bit.  Sums, statistics and parameters are fp32; an activation is
// rounded once, when it is stored.  The norm in front of the next block is taken of h before that rounding.
#include "common.cuh"
#include "nn_ops.h"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int kMaxChannels = 16384;
constexpr int kVec = 8;                 // channels a vector
enum { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };
enum { MODE_NORM = 1, MODE_JOIN = 2, MODE_BOTH = 3 };     // the next norm alone, a join alone, a join and the norm behind it

// ---- launch shape ----
struct Shape {
  int vectors;       // vectors a thread
  int slot;          // threads a row: a power of two up to 32, or whole warps
  int slots;         // rows a block works on at a time
  int blocks;
  int threads() const { return slot * slots; }
};
// K vectors a thread: as few as 512 threads allow, since what a thread keeps for its columns is in registers
Shape plan(long long rows, int C) {
  Shape s;
  const int vec = (C + kVec - 1) / kVec;
  s.vectors = vec <= 512 ? 1 : vec <= 1024 ? 2 : 4;
  const int need = (vec + s.vectors - 1) / s.vectors;
  s.slot = 1;
  if (need <= 32) while (s.slot < need) s.slot <<= 1;
  else s.slot = (need + 31) / 32 * 32;
  s.slots = s.slot >= 256 ? 1 : 256 / s.slot;
  const long long most = (long long)geeps_sm_count() * 2;
  const long long want = (rows + s.slots - 1) / s.slots;
  s.blocks = (int)(want < most ? want : most);
  return s;
}
// rows [first, last) of block b
__host__ __device__ inline long long first_row(long long rows, int blocks, int b) {
  return rows / blocks * b + (rows % blocks < b ? rows % blocks : b);
}

// ---- a thread's columns ----
// VEC: vectors t, t + slot, ...: 16- or 32-byte accesses.  Otherwise (odd widths, pitches or addresses) single columns
// t, t + slot, ...: neighbouring threads on neighbouring columns.
template <int K, bool VEC>
struct Columns {
  int t, slot, C;
  __device__ __forceinline__ int at(int j) const { return VEC ? (t + (j >> 3) * slot) * 8 + (j & 7) : t + j * slot; }
  __device__ __forceinline__ bool on(int j) const { return at(j) < C; }

  template <typename T>
  __device__ __forceinline__ void load(const T* row, bool active, float (&f)[8 * K]) const {
#pragma unroll
    for (int j = 0; j < 8 * K; ++j) f[j] = 0.f;
    if (!active) return;
    if (VEC) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = at(8 * k);
        if (c >= C) continue;
        if (sizeof(T) == 2) {
          const uint4 q = *reinterpret_cast<const uint4*>(row + c);
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) { f[8 * k + 2 * e] = __uint_as_float(w[e] << 16); f[8 * k + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
        } else {
          const float4 lo = *reinterpret_cast<const float4*>(row + c), hi = *reinterpret_cast<const float4*>(row + c + 4);
          f[8 * k] = lo.x; f[8 * k + 1] = lo.y; f[8 * k + 2] = lo.z; f[8 * k + 3] = lo.w;
          f[8 * k + 4] = hi.x; f[8 * k + 5] = hi.y; f[8 * k + 6] = hi.z; f[8 * k + 7] = hi.w;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8 * K; ++j) if (on(j)) f[j] = (float)row[at(j)];
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, bool active, const float (&f)[8 * K]) const {
    if (!active) return;
    if (VEC) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = at(8 * k);
        if (c >= C) continue;
        if (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(row + c) = make_uint4(pack_bf16x2(f[8 * k], f[8 * k + 1]), pack_bf16x2(f[8 * k + 2], f[8 * k + 3]),
                                                          pack_bf16x2(f[8 * k + 4], f[8 * k + 5]), pack_bf16x2(f[8 * k + 6], f[8 * k + 7]));
        } else {
          float* r = reinterpret_cast<float*>(row);
          st_f4(r + c, make_float4(f[8 * k], f[8 * k + 1], f[8 * k + 2], f[8 * k + 3]));
          st_f4(r + c + 4, make_float4(f[8 * k + 4], f[8 * k + 5], f[8 * k + 6], f[8 * k + 7]));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8 * K; ++j) if (on(j)) row[at(j)] = (T)f[j];
    }
  }
  // a parameter of every column; `other` where there is none
  __device__ __forceinline__ void param(const float* p, float other, float (&f)[8 * K]) const {
#pragma unroll
    for (int j = 0; j < 8 * K; ++j) f[j] = p != nullptr && on(j) ? p[at(j)] : other;
  }
};

// Sums of N values over the threads of a slot, the same in each.  Slots of several warps meet at their named barrier; the
// two halves of `red` take turns, so the next sum may be written while this one is still being read.
template <int N>
__device__ __forceinline__ void slot_sum(float (&v)[N], int slot, int t, int slot_id, float* red, int& turn) {
  const int width = slot < 32 ? slot : 32;
  for (int o = width >> 1; o; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if (slot <= 32) return;
  const int warps = slot >> 5;
  float* r = red + turn * 32 * 2;
  turn ^= 1;
  if ((t & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[(t >> 5) * N + i] = v[i];
  }
  asm volatile("bar.sync %0, %1;" ::"r"(slot_id + 1), "r"(slot) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int w = 0; w < warps; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += r[w * N + i];
  }
}

struct Slot {
  int id, t;
  float* red;        // 128 floats of shared memory
  int turn = 0;
};

// n = (f - mean) * rstd in place; mean and rstd go to stats
template <int K, bool VEC>
__device__ __forceinline__ void normalise(const Columns<K, VEC>& cols, Slot& s, const GeepsNorm& norm, long long row, bool active,
                                          float inv_c, float (&f)[8 * K]) {
  float mean = 0.f, v[1];
  if (norm.kind == NORM_LAYER) {
    v[0] = 0.f;
#pragma unroll
    for (int j = 0; j < 8 * K; ++j) v[0] += f[j];
    slot_sum<1>(v, cols.slot, s.t, s.id, s.red, s.turn);
    mean = v[0] * inv_c;
  }
  v[0] = 0.f;
#pragma unroll
  for (int j = 0; j < 8 * K; ++j) { f[j] = cols.on(j) ? f[j] - mean : 0.f; v[0] = fmaf(f[j], f[j], v[0]); }
  slot_sum<1>(v, cols.slot, s.t, s.id, s.red, s.turn);
  const float rstd = 1.f / sqrtf(fmaf(v[0], inv_c, norm.eps));
#pragma unroll
  for (int j = 0; j < 8 * K; ++j) f[j] *= rstd;
  if (norm.stats && active && s.t == 0) { norm.stats[2 * row] = mean; norm.stats[2 * row + 1] = rstd; }
}

// gradient of n * w + b by its input, a = dz * w in place: rstd * (a - mean a - n mean(a n))
template <int K, bool VEC>
__device__ __forceinline__ void norm_gradient(const Columns<K, VEC>& cols, Slot& s, int kind, float rstd, float inv_c,
                                              const float (&n)[8 * K], float (&a)[8 * K]) {
  float v[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 8 * K; ++j) { v[0] += a[j]; v[1] = fmaf(a[j], n[j], v[1]); }
  slot_sum<2>(v, cols.slot, s.t, s.id, s.red, s.turn);
  const float m0 = kind == NORM_LAYER ? v[0] * inv_c : 0.f, m1 = v[1] * inv_c;
#pragma unroll
  for (int j = 0; j < 8 * K; ++j) a[j] = rstd * (a[j] - m0 - n[j] * m1);
}

__device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + expf(-g)); }

template <typename TR, typename TB, int K, bool VEC, int MODE>
__global__ void __launch_bounds__(512)
residual_forward_kernel(const __grid_constant__ GeepsResidual p, int slot, int slots) {
  geeps_pdl_enter();
  __shared__ float red[16][128];
  Slot s;
  s.id = threadIdx.x / slot; s.t = threadIdx.x % slot; s.red = red[slot > 32 ? s.id : 0];
  const Columns<K, VEC> cols = {s.t, slot, p.C};
  const float inv_c = 1.f / (float)p.C;
  float sw[8 * K], sb[8 * K], w2[8 * K], b2[8 * K];
  if (MODE & MODE_JOIN) {
    float sc[8 * K];
    cols.param(p.scale, 1.f, sc); cols.param(p.post.weight, 1.f, sw); cols.param(p.post.bias, 0.f, sb);
#pragma unroll
    for (int j = 0; j < 8 * K; ++j) { sw[j] *= sc[j]; sb[j] *= sc[j]; }
  }
  if (MODE & MODE_NORM) { cols.param(p.pre.weight, 1.f, w2); cols.param(p.pre.bias, 0.f, b2); }
  const long long lo = first_row(p.rows, gridDim.x, blockIdx.x), hi = first_row(p.rows, gridDim.x, blockIdx.x + 1);
  const long long per_gate = p.gate ? p.rows / p.gate_rows : 1;
  for (long long base = lo; base < hi; base += slots) {
    const long long row = base + s.id;
    const bool active = row < hi;
    float h[8 * K];
    cols.load((const TR*)p.res + row * p.ldres, active, h);
    if (MODE & MODE_JOIN) {
      float z[8 * K];
      cols.load((const TB*)p.x + row * p.ldx, active, z);
      if (p.post.kind) normalise(cols, s, p.post, row, active, inv_c, z);
#pragma unroll
      for (int j = 0; j < 8 * K; ++j) z[j] = fmaf(z[j], sw[j], sb[j]);
      if (p.gate) {
        float g[8 * K];
        cols.load((const TB*)p.gate + (row / per_gate) * p.ldgate, active, g);
#pragma unroll
        for (int j = 0; j < 8 * K; ++j) z[j] *= p.sigmoid ? sigmoid(g[j]) : g[j];
      }
#pragma unroll
      for (int j = 0; j < 8 * K; ++j) h[j] += z[j];
      cols.store((TR*)p.out + row * p.ldout, active, h);
    }
    if (MODE & MODE_NORM) {
      normalise(cols, s, p.pre, row, active, inv_c, h);
#pragma unroll
      for (int j = 0; j < 8 * K; ++j) h[j] = fmaf(h[j], w2[j], b2[j]);
      cols.store((TB*)p.y + row * p.ldy, active, h);
    }
  }
}

// Sums kept per block in the workspace: [block][sums][C], A and B of the join, then dweight and dbias of the next norm;
// behind them a row of the gate's gradient for each (block, image) pair that shares rows, number block + image.
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

template <typename TR, typename TB, int K, bool VEC, int MODE>
__global__ void __launch_bounds__(512)
residual_backward_kernel(const __grid_constant__ GeepsResidual p, int slot, int slots) {
  geeps_pdl_enter();
  extern __shared__ __align__(16) float meet[];        // [slots][8 K slot]: slots add up their column sums
  __shared__ float red[16][128];
  constexpr int N = 8 * K;
  Slot s;
  s.id = threadIdx.x / slot; s.t = threadIdx.x % slot; s.red = red[slot > 32 ? s.id : 0];
  const Columns<K, VEC> cols = {s.t, slot, p.C};
  const float inv_c = 1.f / (float)p.C;
  const bool by_image = p.gate && p.gate_rows < p.rows;
  float sw[N], w2[N], a0[N], a1[N], n0[N], n1[N], t0[N], t1[N], g[N];
  if (MODE & MODE_JOIN) {
    float sc[N];
    cols.param(p.scale, 1.f, sc); cols.param(p.post.weight, 1.f, sw);
#pragma unroll
    for (int j = 0; j < N; ++j) { sw[j] *= sc[j]; a0[j] = a1[j] = t0[j] = t1[j] = 0.f; g[j] = 1.f; }
  }
  if (MODE & MODE_NORM) {
    cols.param(p.pre.weight, 1.f, w2);
#pragma unroll
    for (int j = 0; j < N; ++j) n0[j] = n1[j] = 0.f;
  }
  const long long lo = first_row(p.rows, gridDim.x, blockIdx.x), hi = first_row(p.rows, gridDim.x, blockIdx.x + 1);
  const long long per_gate = p.gate ? p.rows / p.gate_rows : 1;
  // the sum of v over the slots, in the threads of slot 0
  auto over_slots = [&](float (&v)[N]) {
    if (slots == 1) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) meet[(s.id * N + j) * slot + s.t] = v[j];
    __syncthreads();
    if (s.id == 0) {
      for (int i = 1; i < slots; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += meet[(i * N + j) * slot + s.t];
      }
    }
  };
  for (long long from = lo; from < hi;) {
    const long long image = by_image ? from / per_gate : 0;
    const long long to = by_image && (image + 1) * per_gate < hi ? (image + 1) * per_gate : hi;
    if (by_image) {
      cols.load((const TB*)p.gate + image * p.ldgate, true, g);
      if (p.sigmoid) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] = sigmoid(g[j]);
      }
    }
    for (long long base = from; base < to; base += slots) {
      const long long row = base + s.id;
      const bool active = row < to;
      float dh[N], x[N];
      cols.load((const TR*)p.dout + row * p.lddout, active && p.dout, dh);
      if (MODE & MODE_JOIN) {              // everything is read before the first output of the row is written
        cols.load((const TB*)p.x + row * p.ldx, active, x);
        if (p.gate && !by_image) cols.load((const TB*)p.gate + row * p.ldgate, active, g);
      }
      if (MODE & MODE_NORM) {
        float n[N], a[N];
        cols.load((const TR*)p.out + row * p.ldout, active, n);
        cols.load((const TB*)p.dy + row * p.lddy, active, a);
        const float mean = active ? p.pre.stats[2 * row] : 0.f, rstd = active ? p.pre.stats[2 * row + 1] : 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          n[j] = cols.on(j) ? (n[j] - mean) * rstd : 0.f;
          n0[j] = fmaf(a[j], n[j], n0[j]); n1[j] += a[j];
          a[j] *= w2[j];
        }
        norm_gradient(cols, s, p.pre.kind, rstd, inv_c, n, a);
#pragma unroll
        for (int j = 0; j < N; ++j) dh[j] += a[j];
      }
      cols.store((TR*)p.dres + row * p.lddres, active, dh);
      if (MODE & MODE_JOIN) {
        float (&n)[N] = x;
        float e[N], rstd = 0.f;
        if (p.post.kind) {
          const float mean = active ? p.post.stats[2 * row] : 0.f;
          rstd = active ? p.post.stats[2 * row + 1] : 0.f;
#pragma unroll
          for (int j = 0; j < N; ++j) n[j] = cols.on(j) ? (n[j] - mean) * rstd : 0.f;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) if (!cols.on(j)) dh[j] = 0.f;
        if (p.gate && !by_image) {
          float dg[N], sb[N], sc[N];
          cols.param(p.post.bias, 0.f, sb); cols.param(p.scale, 1.f, sc);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            if (p.sigmoid) g[j] = sigmoid(g[j]);
            dg[j] = dh[j] * fmaf(sw[j], n[j], sb[j] * sc[j]) * (p.sigmoid ? g[j] * (1.f - g[j]) : 1.f);
          }
          if (p.dgate) cols.store((TB*)p.dgate + row * p.lddgate, active, dg);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float gd = by_image ? dh[j] : dh[j] * g[j];
          a0[j] = fmaf(gd, n[j], a0[j]); a1[j] += gd;
          e[j] = dh[j] * g[j] * sw[j];
        }
        if (p.post.kind) norm_gradient(cols, s, p.post.kind, rstd, inv_c, n, e);
        cols.store((TB*)p.dx + row * p.lddx, active, e);
      }
    }
    if ((MODE & MODE_JOIN) && by_image) {       // the image's rows of this block are done
      float d[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = cols.at(j);
        const float sc = p.scale && cols.on(j) ? p.scale[c] : 1.f, b = p.post.bias && cols.on(j) ? p.post.bias[c] : 0.f;
        d[j] = (sw[j] * a0[j] + sc * b * a1[j]) * (p.sigmoid ? g[j] * (1.f - g[j]) : 1.f);
        t0[j] = fmaf(g[j], a0[j], t0[j]); t1[j] = fmaf(g[j], a1[j], t1[j]);
        a0[j] = a1[j] = 0.f;
      }
      over_slots(d);
      if (p.dgate && s.id == 0) {
        if (image * per_gate >= lo && (image + 1) * per_gate <= hi) {
          cols.store((TB*)p.dgate + image * p.lddgate, true, d);
        } else {
          float* w = p.work + (long long)gridDim.x * sums_of(MODE) * p.C + (blockIdx.x + image) * p.C;
#pragma unroll
          for (int j = 0; j < N; ++j) if (cols.on(j)) w[cols.at(j)] = d[j];
        }
      }
    }
    from = to;
  }
  if (MODE & MODE_JOIN) {
    if (by_image) {
#pragma unroll
      for (int j = 0; j < N; ++j) { a0[j] = t0[j]; a1[j] = t1[j]; }
    }
    over_slots(a0); over_slots(a1);
  }
  if (MODE & MODE_NORM) { over_slots(n0); over_slots(n1); }
  if (s.id != 0) return;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (!cols.on(j)) continue;
    const int c = cols.at(j);
    float v[4];
    int k = 0;
    if (MODE & MODE_JOIN) { v[k++] = a0[j]; v[k++] = a1[j]; }
    if (MODE & MODE_NORM) { v[k++] = n0[j]; v[k++] = n1[j]; }
    if (gridDim.x == 1) write_sums(p, MODE, c, v);
    else for (int i = 0; i < sums_of(MODE); ++i) p.work[((long long)blockIdx.x * sums_of(MODE) + i) * p.C + c] = v[i];
  }
}

// Second launch: the blocks' sums in block order.  blockIdx.y = 0: the columns' sums; y > 0: the gate's gradient of the image
// that the rows of block y begin inside of, if they are its first cut.
template <typename TB>
__global__ void __launch_bounds__(256)
residual_sums_kernel(const __grid_constant__ GeepsResidual p, int mode, int blocks) {
  geeps_pdl_enter();
  const int lane = threadIdx.x & 7, part = threadIdx.x >> 3, c = blockIdx.x * 8 + lane, sums = sums_of(mode);
  if (blockIdx.y == 0) {
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
  const long long per_gate = p.rows / p.gate_rows;
  const int b = blockIdx.y;
  const long long cut = first_row(p.rows, blocks, b), image = cut / per_gate, start = image * per_gate;
  if (cut == start || first_row(p.rows, blocks, b - 1) > start) return;
  if (part != 0 || c >= p.C) return;
  const float* w = p.work + (long long)blocks * sums * p.C;
  float v = 0.f;
  for (int q = b - 1; q < blocks && first_row(p.rows, blocks, q) < start + per_gate; ++q) v += w[(q + image) * p.C + c];
  ((TB*)p.dgate)[image * p.lddgate + c] = (TB)v;
}

// ---- checks ----
struct Use { const void* p; long long ld, rows; int size; bool out; };
bool vectors_ok(const Use& u, int C) {
  if (!u.p) return true;
  return ((uintptr_t)u.p & 15) == 0 && (u.rows <= 1 || (u.ld * u.size & 15) == 0) && C % kVec == 0;
}
// Do two operands share memory in a way that rows of one would be overwritten before the other is read?  The very same rows
// are fine (every thread reads its columns of a row before it writes them), and so are two ranges of columns of one matrix.
bool clash(const Use& a, const Use& b, int C) {
  if (!a.p || !b.p || !a.rows || !b.rows || (!a.out && !b.out)) return false;
  const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p, wa = (uintptr_t)C * a.size, wb = (uintptr_t)C * b.size;
  const uintptr_t a1 = a0 + (uintptr_t)(a.rows - 1) * a.ld * a.size + wa, b1 = b0 + (uintptr_t)(b.rows - 1) * b.ld * b.size + wb;
  if (a1 <= b0 || b1 <= a0) return false;
  const uintptr_t pa = (uintptr_t)a.ld * a.size, pb = (uintptr_t)b.ld * b.size;
  if (!(a.out && b.out) && a0 == b0 && a.size == b.size && a.rows == b.rows && (pa == pb || a.rows == 1)) return false;
  if (pa == pb) {
    const uintptr_t d = a0 < b0 ? (b0 - a0) % pa : pa - 1 - (a0 - b0 - 1) % pa;      // b's first column behind a's
    const uintptr_t dd = d % pa;
    if (dd >= wa && dd + wb <= pa) return false;
  }
  return true;
}

int check(const GeepsResidual& p, bool backward, int mode, bool* vec) {
  if (p.C < 1 || p.C > kMaxChannels) return GEEPS_ERR_NORM_CHANNELS;
  if (p.rows < 0 || p.rows > (1LL << 40)) return (int)cudaErrorInvalidValue;
  if (p.gate && (p.gate_rows < 1 || p.gate_rows > p.rows || p.rows % p.gate_rows)) return p.rows ? GEEPS_ERR_NORM_GATE : 0;
  if (p.stream_fp32 == 0 && p.block_fp32) return (int)cudaErrorInvalidValue;
  const int r = p.stream_fp32 ? 4 : 2, b = p.block_fp32 ? 4 : 2;
  const long long n = p.rows, gr = p.gate ? p.gate_rows : 0;
  const Use fwd[] = {{p.x, p.ldx, n, b, false}, {p.res, p.ldres, n, r, false}, {p.gate, p.ldgate, gr, b, false},
                     {p.out, p.ldout, n, r, true}, {p.y, p.ldy, n, b, true}};
  const Use bwd[] = {{p.x, p.ldx, n, b, false}, {p.dout, p.lddout, n, r, false}, {p.gate, p.ldgate, gr, b, false},
                     {p.out, p.ldout, n, r, false}, {p.dy, p.lddy, n, b, false}, {p.dres, p.lddres, n, r, true},
                     {p.dx, p.lddx, n, b, true}, {p.dgate, p.lddgate, gr, b, true}};
  const Use* u = backward ? bwd : fwd;
  const int count = backward ? 8 : 5;
  *vec = true;
  for (int i = 0; i < count; ++i) {
    if (u[i].p && u[i].rows > 1 && u[i].ld < (u[i].out ? p.C : 0)) return (int)cudaErrorInvalidValue;
    *vec = *vec && vectors_ok(u[i], p.C);
    for (int j = 0; j < i; ++j) if (clash(u[i], u[j], p.C)) return GEEPS_ERR_NORM_OVERLAP;
  }
  const bool join = mode & MODE_JOIN, norm = mode & MODE_NORM;
  if (norm != (p.pre.kind != NORM_NONE) || (!join && (p.x || p.gate || p.post.kind))) return (int)cudaErrorInvalidValue;
  if (p.rows == 0) return 0;
  if (join && !p.x) return (int)cudaErrorInvalidValue;
  if (!backward) {
    if (!p.res || (join && !p.out) || (norm && !p.y)) return (int)cudaErrorInvalidValue;
  } else {
    if (!p.dres || (join && !p.dx) || (norm && (!p.out || !p.dy || !p.pre.stats)) || (!norm && !p.dout)) return (int)cudaErrorInvalidValue;
    if (join && p.post.kind && !p.post.stats) return (int)cudaErrorInvalidValue;
  }
  return 0;
}

template <typename TR, typename TB, int K, bool VEC>
void run(const GeepsResidual& p, const Shape& s, int mode, bool backward, cudaStream_t st) {
  const dim3 grid(s.blocks), block(s.threads());
  const size_t smem = backward && s.slots > 1 ? (size_t)s.threads() * 8 * K * sizeof(float) : 0;
#define GEEPS_MODE(M)                                                                                                       \
  case M:                                                                                                                   \
    if (backward) geeps_launch(residual_backward_kernel<TR, TB, K, VEC, M>, grid, block, smem, st, p, s.slot, s.slots);      \
    else geeps_launch(residual_forward_kernel<TR, TB, K, VEC, M>, grid, block, smem, st, p, s.slot, s.slots);                \
    break;
  switch (mode) { GEEPS_MODE(MODE_NORM) GEEPS_MODE(MODE_JOIN) GEEPS_MODE(MODE_BOTH) }
#undef GEEPS_MODE
}
template <typename TR, typename TB>
void run_types(const GeepsResidual& p, const Shape& s, int mode, bool backward, bool vec, cudaStream_t st) {
  if (s.vectors == 1) { if (vec) run<TR, TB, 1, true>(p, s, mode, backward, st); else run<TR, TB, 1, false>(p, s, mode, backward, st); }
  else if (s.vectors == 2) { if (vec) run<TR, TB, 2, true>(p, s, mode, backward, st); else run<TR, TB, 2, false>(p, s, mode, backward, st); }
  else { if (vec) run<TR, TB, 4, true>(p, s, mode, backward, st); else run<TR, TB, 4, false>(p, s, mode, backward, st); }
  if (!backward || s.blocks == 1) return;
  const bool cuts = p.gate && p.gate_rows < p.rows && p.dgate;
  geeps_launch(residual_sums_kernel<TB>, dim3((p.C + 7) / 8, cuts ? s.blocks : 1), dim3(256), 0, st, p, mode, s.blocks);
}

__global__ void clear_sums_kernel(const __grid_constant__ GeepsResidual p, int mode) {
  geeps_pdl_enter();
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < p.C) write_sums(p, mode, c, zero);
}

int residual(const GeepsResidual* q, bool backward, void* stream) {
  const GeepsResidual& p = *q;
  const int mode = p.mode;
  if (mode < MODE_NORM || mode > MODE_BOTH) return (int)cudaErrorInvalidValue;
  bool vec = true;
  const int bad = check(p, backward, mode, &vec);
  if (bad) return bad;
  cudaStream_t st = (cudaStream_t)stream;
  if (p.rows == 0) {
    if (!backward) return 0;
    geeps_launch(clear_sums_kernel, dim3((p.C + 255) / 256), dim3(256), 0, st, p, mode);
    return (int)cudaGetLastError();
  }
  const Shape s = plan(p.rows, p.C);
  if (backward && !p.work && geeps_residual_work(p.rows, p.gate ? p.gate_rows : 0, p.C, mode) > 0) return (int)cudaErrorInvalidValue;
  if (!p.stream_fp32) run_types<bf16, bf16>(p, s, mode, backward, vec, st);
  else if (!p.block_fp32) run_types<float, bf16>(p, s, mode, backward, vec, st);
  else run_types<float, float>(p, s, mode, backward, vec, st);
  return (int)cudaGetLastError();
}

}  // namespace

extern "C" long long geeps_residual_work(long long rows, long long gate_rows, int C, int mode) {
  if (rows <= 0 || C < 1 || C > kMaxChannels) return 0;
  const Shape s = plan(rows, C);
  if (s.blocks == 1) return 0;
  return ((long long)s.blocks * sums_of(mode) + (gate_rows > 0 && gate_rows < rows ? s.blocks + gate_rows : 0)) * C;
}
extern "C" int geeps_residual_forward(const GeepsResidual* p, void* stream) { return residual(p, false, stream); }
extern "C" int geeps_residual_backward(const GeepsResidual* p, void* stream) { return residual(p, true, stream); }
extern "C" int geeps_norm_shape(long long rows, int C, int* out) {
  const Shape s = plan(rows, C);
  out[0] = s.vectors; out[1] = s.slot; out[2] = s.slots; out[3] = s.blocks;
  return 0;
}
