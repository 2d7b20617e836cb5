// Products of 8-bit matrices on the 5th-generation tensor cores: C[M,N] = A[M,K] * B[N,K]^T + bias, optional ReLU, bf16 or fp32 out.
//
// A and B are e4m3 with a scale 2^e for every 128 columns of a row (quantize.cu makes them).  Scales that are powers of two are
// applied by the tensor core itself (kind::mxf8f6f4): an MMA of 32 columns takes one E8M0 byte for each row of A and of B, so the
// sum over K stays in TMEM in fp32 and no other instruction touches it before the epilogue.  The scales' layout in memory is the
// one that TMEM wants, 512 bytes for 128 rows x 4 blocks of K, which are copied there (tcgen05.cp) in front of every fourth k tile.
//
// As in the bf16 GEMM: TMA -> ring of stages in shared memory (128-byte swizzle, a k tile is one block of 128 columns) -> MMAs by
// one elected lane -> two accumulators in TMEM -> epilogue by two groups of four warps through swizzled slabs and TMA stores.
// Outputs with too few tiles for the machine cut K over the CTAs of a cluster, which add their slices over distributed shared
// memory in slice order.  With few rows in A the operands change places: the 128 rows of a tile are then B's (a layer's weights)
// and the tile is only as wide as A has rows.
// Every mbarrier wait is bounded; on expiry the CTA records TIMEOUT in `status`, stops issuing work, frees its TMEM and returns.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "kernels.h"
#include "nn_ops.h"
#include "tc05.cuh"
#include "tensor_list.h"

namespace {

constexpr int BM = 128;                     // rows of a tile
constexpr int BK = 128;                     // columns of a k tile: one block of the scales, one 128-byte swizzle row
constexpr int A_BYTES = BM * BK;
constexpr int ATOM = 512;                   // scales of 128 rows x 4 k tiles
constexpr int SCALE_BYTES = 2048;           // of a stage: one atom of A, up to three of B
constexpr int MAX_STAGES = 8;
constexpr int SCALE_SETS = 4;               // sets of scales in TMEM, 16 columns each, for four k tiles (the last of a tile: one to four) in turn.
                                            // A set is written anew when the MMAs that read it have been waited for, in whatever order copies
                                            // and MMAs run: with three quads or more a tile, any three that follow one another have 4 + 4 + 1 k tiles at
                                            // least, so the set was read last 10 k tiles ago, and a k tile is loaded when the one MAX_STAGES before it is done;
                                            // with one or two it was read by a tile before the last, whose accumulator has been handed back
constexpr int SLAB_BYTES = BM * 128;
constexpr uint64_t WAIT_BUDGET_NS = 2000000000ull;
constexpr int groups(bool cl) { return cl ? 1 : 2; }
constexpr int threads(bool cl) { return 64 + 128 * groups(cl); }
static_assert(SCALE_SETS == 4 && MAX_STAGES <= 10, "scales in TMEM are overwritten while MMAs may read them");

struct Dev {
  void* C; const float* bias; int* status;
  const uint8_t *scale_a, *scale_b;
  long long M, N, ldc;                      // rows of the operand with 128-row tiles, of the other one, pitch of C
  long long whole;                          // columns of C in whole pieces of 16 bytes
  int out_fp32, swap, relu;                 // swap: C is [N, M]
  int kt, quads;                            // k tiles, and atoms along K
  int bn, m_tiles, n_tiles, cluster, stages, slabs, tma_store, tmem_cols;
};

struct Ctl {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], tmem_full[2], tmem_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
// byte of the 16-byte piece q of row r in a [128][bn] fp32 tile; the XOR keeps a column of rows off a single bank
__device__ __forceinline__ uint32_t part_off(int r, int q, int bn) { return (uint32_t)(r * bn * 4 + ((q ^ (r & 7)) << 4)); }

__device__ __forceinline__ void store1(const Dev& d, long long i, float v) {
  if (d.out_fp32) ((float*)d.C)[i] = v; else ((__nv_bfloat16*)d.C)[i] = __float2bfloat16(v);
}

// The epilogue of a group of four warps (group grp of G) for its share of a tile's columns: slabs 128 bytes wide (64 bf16 or 32 fp32
// columns) leave with one TMA store each, clipped at the matrix edge, which for TMA is d.whole (store_tail).  r: the thread's row of the tile
// TWO: two slabs a group, used in turn
template <int G, bool TWO>
__device__ __forceinline__ void store_slabs(const Dev& d, const CUtensorMap& tmC, uint8_t* slabs, uint32_t tacc, int m0, int n0, int grp, int r,
                                            uint32_t& slab_i) {
  const int cols = d.out_fp32 ? 32 : 64;
  const bool issuer = threadIdx.x == 64 + 128 * grp;
  const uint32_t row_off = (uint32_t)r * 128u, rsw = (uint32_t)(r & 7);
#pragma unroll 1
  for (int c = grp * cols; c < d.bn; c += G * cols) {
    if ((long long)n0 + c >= d.whole) break;
    uint8_t* slab = slabs + (size_t)(TWO ? 2 * grp + (slab_i & 1u) : grp) * SLAB_BYTES;
    if (issuer) { if (TWO) tc05::bulk_wait_read<1>(); else tc05::bulk_wait_read<0>(); }      // the slab this group stored there has been read out
    tc05::named_bar_sync(1 + grp, 128);
    for (int h = 0; h < cols; h += 32) {
      uint32_t w[32];
      tc05::tmem_ld_32x32(tacc + (uint32_t)(c + h), w);
      tc05::tmem_ld_wait();
      const long long col0 = (long long)n0 + c + h;
      float v[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(w[j]);
      if (d.bias != nullptr) {
        if (col0 + 32 <= d.N) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += __ldg(d.bias + col0 + j);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += col0 + j < d.N ? __ldg(d.bias + col0 + j) : 0.f;
        }
      }
      if (d.relu) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];      // not fmaxf: a NaN stays one
      }
      if (d.out_fp32) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<float4*>(slab + row_off + (uint32_t)((j ^ rsw) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(slab + row_off + (uint32_t)((((h >> 3) + j) ^ rsw) << 4)) =
              make_uint4(pack_bf16x2(v[8 * j], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                         pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
      }
    }
    tc05::fence_proxy_async_smem();
    tc05::named_bar_sync(1 + grp, 128);
    if (issuer) {
      tc05::tma_store_2d(&tmC, slab, n0 + c, m0);
      tc05::bulk_commit();
    }
    ++slab_i;
  }
}

// The last columns of a row where it does not end in a whole piece of 16 bytes: a TMA store writes such a piece whole, zeros behind the last
// column, where something else may lie.  By the group that does not have to store the slab before them, each row by its thread.  (As a part of
// store_slabs 7452 x 8960, K = 256 30.0 us -> 31.3, without a tail.)
template <int G>
__device__ __forceinline__ void store_tail(const Dev& d, uint32_t tacc, int m0, int n0, int grp, int r) {
  if (d.whole == d.N || d.whole < n0 || d.whole >= n0 + d.bn) return;
  const int c = (int)(d.whole - n0) & ~31;
  if (G > 1 && grp != ((int)(d.whole - n0) / (d.out_fp32 ? 32 : 64) + 1) % G) return;
  uint32_t w[32];
  tc05::tmem_ld_32x32(tacc + (uint32_t)c, w);
  tc05::tmem_ld_wait();
  if (m0 + r >= d.M) return;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const long long col = (long long)n0 + c + j;
    if (col < d.whole || col >= d.N) continue;
    float v = __uint_as_float(w[j]) + (d.bias != nullptr ? __ldg(d.bias + col) : 0.f);
    if (d.relu) v = v < 0.f ? 0.f : v;
    store1(d, (m0 + r) * d.ldc + col, v);
  }
}

// The same for rows of any pitch and alignment: a warp turns its 32 rows from row0 on through 4 KB of shared memory, 32 columns at a
// time, so that its lanes store neighbours.  (A row a lane: 4068 x 647, K = 74 32.6 us, so 8.7.)
template <int G>
__device__ __forceinline__ void store_rows(const Dev& d, uint8_t* turned, uint32_t tacc, int row0, int n0, int grp, int lane) {
  const int rows = (int)min((long long)32, d.M - row0);
#pragma unroll 1
  for (int c = grp * 32; c < d.bn; c += G * 32) {
    if ((long long)n0 + c >= d.N) break;
    uint32_t w[32];
    tc05::tmem_ld_32x32(tacc + (uint32_t)c, w);
    tc05::tmem_ld_wait();
    __syncwarp();              // the last 32 columns have been read
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<uint4*>(turned + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    __syncwarp();
    const long long col = (long long)n0 + c + lane;
    if (col >= d.N) continue;
    const float bias = d.bias != nullptr ? __ldg(d.bias + col) : 0.f;
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
      float v = *reinterpret_cast<const float*>(turned + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) + bias;
      if (d.relu) v = v < 0.f ? 0.f : v;
      store1(d, (row0 + r) * d.ldc + col, v);
    }
  }
}

// A warp's 32 rows of an accumulator into the CTA's partial tile
__device__ __forceinline__ void leave_part(uint8_t* part, uint32_t tacc, int r, int BN) {
#pragma unroll 1
  for (int c = 0; c < BN; c += 32) {
    uint32_t v[32];
    tc05::tmem_ld_32x32(tacc + (uint32_t)c, v);
    tc05::tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<uint4*>(part + part_off(r, (c >> 2) + j, BN)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
}
// Share z of the sums of a tile's partial tiles, which the CTAs of the cluster hold, in the order of their ranks
__device__ __forceinline__ void finish_slices(const Dev& d, uint32_t part, uint32_t gave_up, int z, int m0, int n0) {
  const int BN = d.bn, quads = BN >> 2, lane = threadIdx.x & 31;
  // a CTA that gave up left no partial tile: nobody stores (the status word names it)
  const bool stop = __any_sync(0xffffffffu, ld_cluster_u32(tc05::map_to_cta(gave_up, lane % d.cluster)) != 0u);
  const long long ri = d.swap ? 1 : d.ldc, ci = d.swap ? d.ldc : 1;
  const int items = stop ? 0 : BM * quads, end = (int)((long long)items * (z + 1) / d.cluster);
  constexpr int U = 4;         // pieces of four columns that a thread has in flight of each slice: the way to another SM takes long
  for (int i0 = (int)((long long)items * z / d.cluster) + threadIdx.x; i0 < end; i0 += U * blockDim.x) {
    float4 v[U];
    uint32_t off[U];
    long long row[U], col0[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // neighbours in C are neighbouring threads
      const int i = min(i0 + u * (int)blockDim.x, items - 1), r = d.swap ? i % BM : i / quads, o = d.swap ? i / BM : i % quads;
      off[u] = part_off(r, o, BN);
      row[u] = (long long)m0 + r;
      col0[u] = i0 + u * (int)blockDim.x < end ? (long long)n0 + o * 4 : d.N;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll 2
    for (int k = 0; k < d.cluster; ++k) {
      const uint32_t at = tc05::map_to_cta(part, k);
      float4 a[U];
#pragma unroll
      for (int u = 0; u < U; ++u) a[u] = i0 + u * (int)blockDim.x < end ? ld_cluster_f4(at + off[u]) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) { v[u].x += a[u].x; v[u].y += a[u].y; v[u].z += a[u].z; v[u].w += a[u].w; }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row[u] >= d.M || col0[u] >= d.N) continue;
      const int nc = (int)min((long long)4, d.N - col0[u]);
      float w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e < nc) {
          if (d.bias != nullptr) w[e] += __ldg(d.bias + (d.swap ? row[u] : col0[u] + e));
          if (d.relu) w[e] = w[e] < 0.f ? 0.f : w[e];
        }
      }
      if (!d.swap && !d.out_fp32 && nc == 4 && (((uintptr_t)((__nv_bfloat16*)d.C + row[u] * d.ldc + col0[u])) & 7) == 0) {
        *reinterpret_cast<uint2*>((__nv_bfloat16*)d.C + row[u] * d.ldc + col0[u]) = make_uint2(pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < nc) store1(d, row[u] * ri + (col0[u] + e) * ci, w[e]);
      }
    }
  }
}

// CL: a cluster of d.cluster CTAs per tile, one slice of K each
template <bool CL>
__global__ void __launch_bounds__(threads(CL), 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmC, const Dev d) {
  extern __shared__ uint8_t smem_raw[];
  const int BN = d.bn;
  const int B_BYTES = BN * BK, STAGE = A_BYTES + B_BYTES + SCALE_BYTES;
  uint8_t* tiles = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* slabs = tiles + (size_t)d.stages * STAGE;
  Ctl* ctl = (Ctl*)(slabs + (CL ? 0 : d.slabs * SLAB_BYTES));      // a cluster stages its tile in the operand ring
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = d.stages;
  const int tiles_mn = d.m_tiles * d.n_tiles;
  // k tiles of a slice: whole atoms of scales
  const int per = CL ? (d.quads + d.cluster - 1) / d.cluster * 4 : d.kt;
  const int k_first = CL ? (int)(blockIdx.x % d.cluster) * per : 0, k_end = min(d.kt, k_first + per);
  const int t_first = CL ? (int)(blockIdx.x / d.cluster) : (int)blockIdx.x;
  const int t_step = CL ? tiles_mn : (int)gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) { tc05::mbar_init(&ctl->full[s], 1); tc05::mbar_init(&ctl->empty[s], 1); }
    for (int a = 0; a < 2; ++a) { tc05::mbar_init(&ctl->tmem_full[a], 1); tc05::mbar_init(&ctl->tmem_empty[a], 4 * groups(CL)); }
    ctl->abort_flag = 0;
    tc05::mbar_fence_init();
  }
  if (warp == 1) {
    tc05::tmem_alloc(&ctl->tmem_base, (uint32_t)d.tmem_cols);
    tc05::tmem_relinquish();
  }
  tc05::fence_before_sync();
  __syncthreads();
  tc05::fence_after_sync();
  const uint32_t tmem = ctl->tmem_base;
  geeps_pdl_wait();          // everything above touches this CTA's own memory only
  volatile int* abort_flag = &ctl->abort_flag;
  const uint32_t tiles_u = tc05::smem_u32(tiles), empty_u = tc05::smem_u32(ctl->empty);

  if (warp == 0) {
    // ---------------- loads ----------------
    const bool leader = tc05::elect_one();
    if (leader) { tc05::tma_prefetch_desc(&tmA); tc05::tma_prefetch_desc(&tmB); }
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    const int atoms_n = (int)((d.N + 127) >> 7);
    for (int t = t_first; t < tiles_mn && ok; t += t_step) {
      const int mt = t % d.m_tiles, n0 = t / d.m_tiles * BN;
      const int b_atom = n0 >> 7, b_atoms = min((n0 + BN + 127) >> 7, atoms_n) - b_atom;
      for (int kt = k_first; kt < k_end; ++kt) {
        if (!tc05::mbar_wait_warp(&ctl->empty[s], ph ^ 1u, abort_flag, WAIT_BUDGET_NS)) { ok = false; break; }
        if (leader) {
          uint8_t* sa = tiles + (size_t)s * STAGE;
          const bool scales = (kt & 3) == 0;
          tc05::mbar_expect_tx(&ctl->full[s], (uint32_t)(A_BYTES + B_BYTES + (scales ? ATOM * (1 + b_atoms) : 0)));
          tc05::tma_load_2d(sa, &tmA, &ctl->full[s], kt * BK, mt * BM);
          tc05::tma_load_2d(sa + A_BYTES, &tmB, &ctl->full[s], kt * BK, n0);
          if (scales) {
            const uint32_t at = tiles_u + (uint32_t)(s * STAGE + A_BYTES + B_BYTES);
            tc05::bulk_load(at, d.scale_a + ((size_t)mt * d.quads + (kt >> 2)) * ATOM, ATOM, &ctl->full[s]);
            for (int i = 0; i < b_atoms; ++i)
              tc05::bulk_load(at + ATOM * (1 + i), d.scale_b + ((size_t)(b_atom + i) * d.quads + (kt >> 2)) * ATOM, ATOM, &ctl->full[s]);
          }
        }
        if (++s == S) { s = 0; ph ^= 1u; }
      }
    }
    geeps_pdl_trigger();       // every operand is on its way: the rest of this CTA is its last products and stores
  } else if (warp == 1) {
    // ---------------- products ----------------
    const bool leader = tc05::elect_one();
    const uint32_t idesc = tc05::make_idesc_e4m3(BM, BN);
    uint32_t tile_i = 0, ph = 0, set = 0;
    int s = 0;
    bool ok = true;
    const int atoms_n = (int)((d.N + 127) >> 7);
    for (int t = t_first; t < tiles_mn && ok; t += t_step, ++tile_i) {
      const int n0 = t / d.m_tiles * BN;
      const int b_atom = n0 >> 7, b_atoms = min((n0 + BN + 127) >> 7, atoms_n) - b_atom;
      const uint32_t acc = tile_i & 1u, acc_ph = (tile_i >> 1) & 1u;
      if (!tc05::mbar_wait_warp(&ctl->tmem_empty[acc], acc_ph ^ 1u, abort_flag, WAIT_BUDGET_NS)) { ok = false; break; }
      tc05::fence_after_sync();
      const uint32_t tacc = tmem + acc * (uint32_t)BN;
      uint32_t sf = 0;
      for (int kt = k_first; kt < k_end; ++kt) {
        if (!tc05::mbar_wait_warp(&ctl->full[s], ph, abort_flag, WAIT_BUDGET_NS)) { ok = false; break; }
        tc05::fence_after_sync();
        const uint32_t sa = tiles_u + (uint32_t)(s * STAGE), sb = sa + A_BYTES;
        if ((kt & 3) == 0) {
          sf = tmem + 2u * (uint32_t)BN + 16u * set;
          if (++set == SCALE_SETS) set = 0;
          if (leader) {
            tc05::scale_copy(sf, sb + B_BYTES);
            for (int i = 0; i < b_atoms; ++i) tc05::scale_copy(sf + 4u + 4u * i, sb + B_BYTES + ATOM * (1 + i));
          }
        }
        tc05::mma_ktile_e4m3(tacc, tc05::desc_lo(sa, 16), tc05::desc_lo(sb, 16), tc05::desc_hi(1024),
                             idesc | tc05::idesc_scale_byte(kt & 3), sf, sf + 4u + ((uint32_t)(n0 & 127) >> 5), kt > k_first ? 1u : 0u,
                             empty_u + 8u * (uint32_t)s);
        if (++s == S) { s = 0; ph ^= 1u; }
      }
      if (ok && leader) tc05::mma_commit(&ctl->tmem_full[acc]);
    }
  } else {
    // ---------------- epilogue: TMEM -> registers -> global ----------------
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    constexpr int G = groups(CL);
    const int grp = (warp - 2) >> 2;
    uint32_t tile_i = 0, slab_i = 0;
    for (int t = t_first; t < tiles_mn; t += t_step, ++tile_i) {
      const int m0 = t % d.m_tiles * BM, n0 = t / d.m_tiles * BN;
      const uint32_t acc = tile_i & 1u, acc_ph = (tile_i >> 1) & 1u;
      if (!tc05::mbar_wait(&ctl->tmem_full[acc], acc_ph, abort_flag, WAIT_BUDGET_NS)) break;
      tc05::fence_after_sync();
      const uint32_t tacc = tmem + acc * (uint32_t)BN + ((uint32_t)(q * 32) << 16);
      const int r = q * 32 + lane;
      const long long row = (long long)m0 + r;
      if (CL) {
        // the commit behind tmem_full covers every MMA of the slice: the operand stages are free to hold the partial tile
        leave_part(tiles, tacc, r, BN);
      } else if (d.tma_store) {
        store_slabs<G, true>(d, tmC, slabs, tacc, m0, n0, grp, r, slab_i);
        store_tail<G>(d, tacc, m0, n0, grp, r);
      } else if (!d.swap) {
        store_rows<G>(d, slabs + grp * SLAB_BYTES + q * 32 * 128, tacc, m0 + q * 32, n0, grp, lane);
      } else {
        // the lanes of a warp are neighbours in C
        const float bias_row = d.bias != nullptr && row < d.M ? d.bias[row] : 0.f;
#pragma unroll 1
        for (int c = grp * 32; c < BN; c += G * 32) {
          uint32_t w[32];
          tc05::tmem_ld_32x32(tacc + (uint32_t)c, w);
          tc05::tmem_ld_wait();
          const long long col0 = (long long)n0 + c;
          if (row < d.M) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (col0 + j < d.N) {
                float v = __uint_as_float(w[j]) + bias_row;
                if (d.relu) v = v < 0.f ? 0.f : v;
                store1(d, row + (col0 + j) * d.ldc, v);
              }
            }
          }
        }
      }
      // this warp is done reading the accumulator: hand it back
      tc05::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc05::mbar_arrive(&ctl->tmem_empty[acc]);
    }
  }

  if (CL) {
    __syncwarp();
    tc05::cluster_sync();
    const int mn = (int)(blockIdx.x / d.cluster);
    finish_slices(d, tc05::smem_u32(tiles), tc05::smem_u32(&ctl->abort_flag), (int)(blockIdx.x % d.cluster), mn % d.m_tiles * BM, mn / d.m_tiles * BN);
    __syncwarp();
    tc05::cluster_sync();      // nobody leaves while a peer still reads its partial tile
  }
  if (!CL && d.tma_store && (threadIdx.x == 64 || threadIdx.x == 192)) tc05::bulk_wait<0>();   // all TMA stores of this CTA have landed
  tc05::fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && ctl->abort_flag) geeps_report(d.status, GEEPS_ERR_TIMEOUT, KID_GEMM_FP8, (int)blockIdx.x, 0);
  if (warp == 1) {
    tc05::fence_after_sync();
    tc05::tmem_dealloc(tmem, (uint32_t)d.tmem_cols);
  }
}

// Two CTAs compute a tile of 256 rows with MMAs of cta_group::2: each loads its own 128 rows of A and half of B's rows, and the scales
// of its rows of A and of all of B's.  The leader issues the copies of scales and the MMAs for both; every load signals its barrier.
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(threads(false), 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC,
                     const __grid_constant__ CUtensorMap tmScaleA, const __grid_constant__ CUtensorMap tmScaleB, const Dev d) {
  extern __shared__ uint8_t smem_raw[];
  const int BN = d.bn;
  const int B_BYTES = BN / 2 * BK, STAGE = A_BYTES + B_BYTES + SCALE_BYTES;
  uint8_t* tiles = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* slabs = tiles + (size_t)d.stages * STAGE;
  Ctl* ctl = (Ctl*)(slabs + d.slabs * SLAB_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc05::cluster_ctarank();
  const int S = d.stages, num_tiles = d.m_tiles * d.n_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int b_atoms = (BN + 127) / 128;              // tiles begin at multiples of 64: these hold 64 + 192 rows as well as 192

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) { tc05::mbar_init(&ctl->full[s], 1); tc05::mbar_init(&ctl->empty[s], 1); }
    for (int a = 0; a < 2; ++a) { tc05::mbar_init(&ctl->tmem_full[a], 1); tc05::mbar_init(&ctl->tmem_empty[a], 16); }
    ctl->abort_flag = 0;
    tc05::mbar_fence_init();
  }
  if (warp == 1) {
    tc05::tmem_alloc_pair(&ctl->tmem_base, (uint32_t)d.tmem_cols);
    tc05::tmem_relinquish_pair();
  }
  tc05::fence_before_sync();
  __syncthreads();
  tc05::cluster_sync();            // the peer's barriers are initialised before anything signals them
  tc05::fence_after_sync();
  const uint32_t tmem = ctl->tmem_base;
  geeps_pdl_wait();          // everything above touches this CTA's own memory only
  volatile int* abort_flag = &ctl->abort_flag;
  const uint32_t tiles_u = tc05::smem_u32(tiles), empty_u = tc05::smem_u32(ctl->empty);

  if (warp == 0) {
    // ---------------- loads (both CTAs) ----------------
    const bool leader = tc05::elect_one();
    if (leader) { tc05::tma_prefetch_desc(&tmA); tc05::tma_prefetch_desc(&tmB); tc05::tma_prefetch_desc(&tmScaleA); tc05::tma_prefetch_desc(&tmScaleB); }
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = first; t < num_tiles && ok; t += step) {
      const int mt = 2 * (t % d.m_tiles) + (int)rank, n0 = t / d.m_tiles * BN;
      for (int kt = 0; kt < d.kt; ++kt) {
        if (!tc05::mbar_wait_warp(&ctl->empty[s], ph ^ 1u, abort_flag, WAIT_BUDGET_NS)) { ok = false; break; }
        if (leader) {
          uint8_t* sa = tiles + (size_t)s * STAGE;
          const bool scales = (kt & 3) == 0;
          // the leader's barrier counts the bytes of both CTAs
          if (rank == 0) tc05::mbar_expect_tx(&ctl->full[s], 2u * (uint32_t)(A_BYTES + B_BYTES + (scales ? ATOM * (1 + b_atoms) : 0)));
          const uint32_t bar = tc05::map_to_cta(tc05::smem_u32(&ctl->full[s]), 0);
          tc05::tma_load_2d_pair(sa, &tmA, bar, kt * BK, mt * BM);
          tc05::tma_load_2d_pair(sa + A_BYTES, &tmB, bar, kt * BK, n0 + (int)rank * (BN / 2));
          if (scales) {
            // atoms behind the last row arrive as zeros
            uint8_t* at = sa + A_BYTES + B_BYTES;
            tc05::tma_load_2d_pair(at, &tmScaleA, bar, 0, mt * d.quads + (kt >> 2));
            for (int i = 0; i < b_atoms; ++i) tc05::tma_load_2d_pair(at + ATOM * (1 + i), &tmScaleB, bar, 0, ((n0 >> 7) + i) * d.quads + (kt >> 2));
          }
        }
        if (++s == S) { s = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ---------------- products (leader) ----------------
    if (rank == 0) {
      const bool leader = tc05::elect_one();
      const uint32_t idesc = tc05::make_idesc_e4m3(2 * BM, BN);
      uint32_t tile_i = 0, ph = 0, set = 0;
      int s = 0;
      bool ok = true;
      for (int t = first; t < num_tiles && ok; t += step, ++tile_i) {
        const int n0 = t / d.m_tiles * BN;
        const uint32_t acc = tile_i & 1u, acc_ph = (tile_i >> 1) & 1u;
        if (!tc05::mbar_wait_warp(&ctl->tmem_empty[acc], acc_ph ^ 1u, abort_flag, WAIT_BUDGET_NS)) { ok = false; break; }
        tc05::fence_after_sync();
        const uint32_t tacc = tmem + acc * (uint32_t)BN;
        uint32_t sf = 0;
        for (int kt = 0; kt < d.kt; ++kt) {
          if (!tc05::mbar_wait_warp(&ctl->full[s], ph, abort_flag, WAIT_BUDGET_NS)) { ok = false; break; }
          tc05::fence_after_sync();
          const uint32_t sa = tiles_u + (uint32_t)(s * STAGE), sb = sa + A_BYTES;
          if ((kt & 3) == 0) {
            sf = tmem + 2u * (uint32_t)BN + 16u * set;
            if (++set == SCALE_SETS) set = 0;
            if (leader) {
              tc05::scale_copy_pair(sf, sb + B_BYTES);
              for (int i = 0; i < b_atoms; ++i) tc05::scale_copy_pair(sf + 4u + 4u * i, sb + B_BYTES + ATOM * (1 + i));
            }
          }
          tc05::mma_ktile_e4m3_pair(tacc, tc05::desc_lo(sa, 16), tc05::desc_lo(sb, 16), tc05::desc_hi(1024), idesc | tc05::idesc_scale_byte(kt & 3), sf,
                                    sf + 4u + ((uint32_t)(n0 & 127) >> 5), kt > 0 ? 1u : 0u, empty_u + 8u * (uint32_t)s);
          if (++s == S) { s = 0; ph ^= 1u; }
        }
        if (ok && leader) tc05::mma_commit_pair(&ctl->tmem_full[acc], 3);
      }
    }
  } else {
    // ---------------- epilogue (both CTAs): own 128 rows ----------------
    const int q = warp & 3, grp = (warp - 2) >> 2;
    uint32_t tile_i = 0, slab_i = 0;
    for (int t = first; t < num_tiles; t += step, ++tile_i) {
      const int m0 = (2 * (t % d.m_tiles) + (int)rank) * BM, n0 = t / d.m_tiles * BN;
      const uint32_t acc = tile_i & 1u, acc_ph = (tile_i >> 1) & 1u;
      if (!tc05::mbar_wait(&ctl->tmem_full[acc], acc_ph, abort_flag, WAIT_BUDGET_NS)) break;
      tc05::fence_after_sync();
      const uint32_t tacc = tmem + acc * (uint32_t)BN + ((uint32_t)(q * 32) << 16);
      if (m0 < d.M) {
        store_slabs<2, false>(d, tmC, slabs, tacc, m0, n0, grp, q * 32 + lane, slab_i);
        store_tail<2>(d, tacc, m0, n0, grp, q * 32 + lane);
      }
      tc05::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc05::mbar_arrive_cluster(tc05::map_to_cta(tc05::smem_u32(&ctl->tmem_empty[acc]), 0));      // the warps of both report
    }
  }
  if (threadIdx.x == 64 || threadIdx.x == 192) tc05::bulk_wait<0>();
  tc05::fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && ctl->abort_flag) geeps_report(d.status, GEEPS_ERR_TIMEOUT, KID_GEMM_FP8, (int)blockIdx.x, 1);
  // neither CTA may release TMEM or exit while the peer can still signal its barriers or use the pair's TMEM
  tc05::cluster_sync();
  if (warp == 1) {
    tc05::fence_after_sync();
    tc05::tmem_dealloc_pair(tmem, (uint32_t)d.tmem_cols);
  }
}

// ---------------- host side ----------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)p;
  });
  return fn;
}
// `outer` lines of `inner` values, `pitch` bytes apart
bool make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long inner, long long outer, long long pitch,
              int box_inner, int box_outer, bool swizzle = true) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer}, one[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan { int swap, bn, cluster, pair; };        // cluster: CTAs that share K; pair: CTA pairs
// Tile widths: 64, 128 and 192 (two accumulators and the scales in 512 columns of TMEM), or 32 for a single tile.  The scales of a
// tile then begin at an even column of TMEM; an MMA whose scales begin at an odd one is a misaligned access.
bool width_ok(int bn, long long N) { return bn == 64 || bn == 128 || bn == 192 || (bn == 32 && N <= 32); }

// Whether an atom's worth of every slice is there
bool slices_ok(int quads, int cluster) { return (long long)((quads + cluster - 1) / cluster) * (cluster - 1) < quads; }

// The cut with the shortest expected time.  A k tile takes a round trip through the ring of stages (0.22 us, pairs 0.29) or what L2
// needs for its operands (128 KB/us an SM, 14.5 MB/us in all, the same line for 300 readers a us): seldom the tensor pipe's time (0.2 us
// for 128 x 192), so wide tiles and pairs win where there are enough of them, and slices of K where there are not.  A tile's stores run
// beside the next one's products.  The constants are fitted to 550 sizes of 1 to 9216; over others the chosen cut takes 0.8 % longer
// than the best one.  In a captured chain, us (width / CTAs that share K, p: pairs, t: B's rows on the tall side): 8192 x 16384, K =
// 4096 407 (192p), 482 (192/1), 588 (128/1); 1024 x 9216, K = 4096 32.2 (192p), 39.1, 39.2; 2048 x 4096, K = 4096 31.8 (192p), 34.9,
// 36.6; 512 x 4096, K = 4096 11.8 (128/1), 13.9 (192p), 14.0; 256 x 4096, K = 9216 17.8 (128/2), 19.6 (64/1), 20.0 (128/1); 7 x 4096,
// K = 4096 7 (32/4t), 8.3 (32/2t), 10.3 (32/1t); 4 x 6400, K = 2688 8.3 (128/1), 12.0 (64/1: 100 CTAs read the same lines of A); 449 x
// 6912, K = 256 5.0 (192/1), 6.8 (192p); 3913 x 1408, K = 256 in fp32 7.6, 11.6; 7451 x 8960, K = 256 30.2, 55.6 (its stores).
Plan choose(const GeepsGemmFp8* p, int sms) {
  const int quads = (int)((p->K + 511) / 512), tiles_k = (int)((p->K + BK - 1) / BK);
  const bool rows16 = ((uintptr_t)p->C & 15) == 0 && p->ldc * (p->out_fp32 ? 4 : 2) % 16 == 0;
  Plan best = {0, 64, 1, 0};
  double least = 1e300;
  for (int pair = 0; pair < 2; ++pair)
    for (int swap = 0; swap < 2 - pair; ++swap) {
      const long long M = swap ? p->N : p->M, N = swap ? p->M : p->N;
      if ((swap && p->M > 128) || (pair && M <= BM)) continue;
      const int tall = pair ? 2 * BM : BM;
      for (int bn = 32; bn <= 192; bn += 32) {
        if (pair ? bn % 64 : !width_ok(bn, N)) continue;
        const long long tiles = ((M + tall - 1) / tall) * ((N + bn - 1) / bn);
        for (int cs = 1; cs <= (pair ? 1 : 8); cs *= 2) {
          if (!slices_ok(quads, cs) || (pair && !rows16)) continue;
          const int size = pair ? 2 : cs;
          // CTAs that whole clusters find in GPCs of different sizes
          const int slots = size <= 2 ? sms : size <= 4 ? sms * 9 / 10 / size * size : sms * 5 / 6 / size * size;
          const long long rounds = (tiles * size + slots - 1) / slots;
          if (cs > 1 && rounds > 1) continue;
          const double active = (double)(tiles * size < slots ? tiles * size : slots), kt = std::min<double>(tiles_k, 4.0 * ((quads + cs - 1) / cs));
          const double kb = 16.0 + (pair ? 0.5 : 1.0) * bn / 8;
          const double m_tiles = (double)((M + tall - 1) / tall), at_once = active / size, readers = std::max(std::min(m_tiles, at_once), at_once / m_tiles);
          const double products = kt * std::max({pair ? 0.29 : 0.22, kb / 128.0, active * kb / 14500.0, 0.0033 * readers});
          // the stores of a tile, beside the next one's products
          const double store = (0.53 + 0.005 * bn) * (p->out_fp32 ? 1.25 : 1.0) * (pair ? 1.8 : 1.0) * (swap ? 2.1 : rows16 ? 1.0 : 1.6);
          const double time = cs > 1 ? products + 5.0 + 0.0275 * bn + (swap ? 0.6 : 0.0)
                                     : 2.3 + (pair ? 1.1 : 0.0) + products + store + (rounds - 1) * std::max(products, store);
          if (time < least * 0.99) { least = time; best = {swap, bn, cs, pair}; }
        }
      }
    }
  return best;
}

// Bytes of a stage of the ring
int stage_bytes(const Dev& d, const Plan& plan) { return A_BYTES + (plan.pair ? d.bn / 2 : d.bn) * BK + SCALE_BYTES; }
// Slabs of the epilogue, and as many stages as fit beside them
void give_memory(Dev& d, const Plan& plan) {
  d.slabs = d.tma_store ? (plan.pair ? 2 : d.bn > (d.out_fp32 ? 32 : 64) ? 4 : 2) : plan.cluster == 1 && !plan.swap ? 2 : 0;
  d.stages = std::min((224 * 1024 - d.slabs * SLAB_BYTES) / stage_bytes(d, plan), MAX_STAGES);
}
int ctas(const Dev& d, const Plan& plan, int sms) {
  const long long tiles = (long long)d.m_tiles * d.n_tiles;
  return (int)(plan.pair ? std::min(tiles, (long long)sms / 2) * 2 : d.cluster > 1 ? tiles * d.cluster : std::min(tiles, (long long)sms));
}
// The cut and all that follows from it without a look at the GPU
int lay_out(const GeepsGemmFp8* p, Plan& plan, Dev& d) {
  plan = p->bn ? Plan{p->swap, p->bn, p->cluster < 0 ? 1 : p->cluster, p->cluster < 0} : choose(p, geeps_sm_count());
  d = Dev{};
  d.kt = (int)((p->K + BK - 1) / BK);
  d.quads = (d.kt + 3) / 4;
  const bool pair = plan.pair != 0;
  const int size = p->out_fp32 ? 4 : 2;
  const bool rows16 = ((uintptr_t)p->C & 15) == 0 && p->ldc * size % 16 == 0;       // what TMA stores
  if (plan.cluster < 1 || plan.cluster > 8 || (plan.cluster & (plan.cluster - 1)) || !slices_ok(d.quads, plan.cluster) ||
      (pair ? plan.swap || !rows16 || (plan.bn != 64 && plan.bn != 128 && plan.bn != 192) : !width_ok(plan.bn, plan.swap ? p->M : p->N)))
    return (int)cudaErrorInvalidValue;
  d.C = p->C; d.bias = p->bias; d.status = p->status;
  d.swap = plan.swap; d.relu = p->relu; d.out_fp32 = p->out_fp32;
  d.M = plan.swap ? p->N : p->M; d.N = plan.swap ? p->M : p->N; d.ldc = p->ldc;
  d.scale_a = plan.swap ? p->scale_b : p->scale_a; d.scale_b = plan.swap ? p->scale_a : p->scale_b;
  d.tma_store = plan.cluster == 1 && !plan.swap && rows16;
  d.whole = p->N & -(16LL / size);
  d.bn = plan.bn;
  d.cluster = plan.cluster;
  d.m_tiles = (int)((d.M + (pair ? 2 : 1) * BM - 1) / ((pair ? 2 : 1) * BM));
  const long long n_tiles = (d.N + d.bn - 1) / d.bn;
  if (n_tiles * d.m_tiles > 0x3fffffffLL) return (int)cudaErrorInvalidValue;
  d.n_tiles = (int)n_tiles;
  d.tmem_cols = 32;
  while (d.tmem_cols < 2 * d.bn + 16 * SCALE_SETS) d.tmem_cols <<= 1;
  give_memory(d, plan);
  return 0;
}

// Lets a kernel have all shared memory of the current device, once
template <auto kernel>
int all_shared() {
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(ready >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    ready |= 1ull << (dev & 63);
  }
  return (int)e;
}

template <bool CL>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Dev& d, int grid, cudaStream_t st) {
  const size_t smem = (size_t)d.stages * (A_BYTES + d.bn * BK + SCALE_BYTES) + (CL ? 0 : d.slabs * SLAB_BYTES) + sizeof(Ctl) + 1024;
  const int e = all_shared<gemm_fp8_kernel<CL>>();
  if (e) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads(CL));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)d.cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CL ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, gemm_fp8_kernel<CL>, ta, tb, tc, d);
}

}  // namespace

extern "C" {

int geeps_gemm_fp8(const GeepsGemmFp8* p, void* stream) {
  if (p->M < 0 || p->N < 0 || p->K < 0 || p->M > 0x3fffffffLL || p->N > 0x3fffffffLL || p->K > 0x3fffffffLL) return (int)cudaErrorInvalidValue;
  if (p->M == 0 || p->N == 0) return 0;
  if (p->K == 0) return (int)cudaErrorInvalidValue;
  if ((((uintptr_t)p->A | (uintptr_t)p->B | (uintptr_t)p->scale_a | (uintptr_t)p->scale_b) & 15) || (p->lda & 15) || (p->ldb & 15) ||
      p->lda < p->K || p->ldb < p->K || p->ldc < p->N || !p->A || !p->B || !p->scale_a || !p->scale_b || !p->C ||
      ((uintptr_t)p->C & (p->out_fp32 ? 3 : 1)) || (((uintptr_t)p->bias | (uintptr_t)p->status) & 3))
    return (int)cudaErrorInvalidValue;
  const long long quads = (p->K + 511) / 512;
  const MemoryRange ranges[] = {{p->C, ((p->M - 1) * p->ldc + p->N) * (p->out_fp32 ? 4 : 2)}, {p->A, (p->M - 1) * p->lda + p->K}, {p->B, (p->N - 1) * p->ldb + p->K},
                                {p->scale_a, (p->M + 127) / 128 * quads * 512}, {p->scale_b, (p->N + 127) / 128 * quads * 512},
                                {p->bias, p->bias ? p->N * 4 : 0}, {p->status, p->status ? 16 : 0}};
  if (ranges_overlap(ranges, 1, 7)) return GEEPS_ERR_NORM_OVERLAP;
  Plan plan;
  Dev d;
  const int bad = lay_out(p, plan, d);
  if (bad) return bad;
  const bool pair = plan.pair != 0;
  const int size = p->out_fp32 ? 4 : 2, sms = geeps_sm_count();
  const void *A = plan.swap ? p->B : p->A, *B = plan.swap ? p->A : p->B;
  const long long lda = plan.swap ? p->ldb : p->lda, ldb = plan.swap ? p->lda : p->ldb;
  CUtensorMap ta, tb, tc;
  if (!make_map(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, p->K, d.M, lda, BK, BM) || !make_map(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, B, p->K, d.N, ldb, BK, pair ? d.bn / 2 : d.bn))
    return (int)cudaErrorInvalidValue;
  if (d.tma_store && !make_map(&tc, p->out_fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p->C,
                               d.whole ? d.whole : 16 / size, p->M, p->ldc * size, p->out_fp32 ? 32 : 64, BM)) {
    if (pair) return (int)cudaErrorInvalidValue;
    d.tma_store = 0;
    give_memory(d, plan);
  }
  if (!d.tma_store) tc = ta;   // unused by the kernel
  cudaStream_t st = (cudaStream_t)stream;
  if (pair) {
    const long long rows_a = (d.M + 127) / 128 * d.quads, rows_b = (d.N + 127) / 128 * d.quads;
    CUtensorMap sa, sb;
    if (!make_map(&sa, CU_TENSOR_MAP_DATA_TYPE_UINT32, d.scale_a, ATOM / 4, rows_a, ATOM, ATOM / 4, 1, false) ||
        !make_map(&sb, CU_TENSOR_MAP_DATA_TYPE_UINT32, d.scale_b, ATOM / 4, rows_b, ATOM, ATOM / 4, 1, false))
      return (int)cudaErrorInvalidValue;
    const int e = all_shared<gemm_fp8_pair_kernel>();
    if (e) return e;
    const size_t smem = (size_t)d.stages * stage_bytes(d, plan) + d.slabs * SLAB_BYTES + sizeof(Ctl) + 1024;
    geeps_launch(gemm_fp8_pair_kernel, ctas(d, plan, sms), threads(false), smem, st, ta, tb, tc, sa, sb, d);
    return (int)cudaGetLastError();
  }
  return d.cluster > 1 ? launch<true>(ta, tb, tc, d, ctas(d, plan, sms), st) : launch<false>(ta, tb, tc, d, ctas(d, plan, sms), st);
}

int geeps_gemm_fp8_shape(const GeepsGemmFp8* p, int* out) {
  if (p->M < 1 || p->N < 1 || p->K < 1 || p->M > 0x3fffffffLL || p->N > 0x3fffffffLL || p->K > 0x3fffffffLL) return (int)cudaErrorInvalidValue;
  Plan plan;
  Dev d;
  const int bad = lay_out(p, plan, d);
  if (bad) return bad;
  out[0] = d.bn; out[1] = plan.pair ? -2 : d.cluster; out[2] = d.swap; out[3] = ctas(d, plan, geeps_sm_count());
  out[4] = d.m_tiles * d.n_tiles; out[5] = d.kt; out[6] = d.stages; out[7] = SCALE_SETS; out[8] = d.tmem_cols;
  return 0;
}

}  // extern "C"
