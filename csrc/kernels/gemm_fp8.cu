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

#include <atomic>
#include <mutex>

#include "kernels.h"
#include "tc05.cuh"

namespace {

constexpr int BM = 128;                     // rows of a tile
constexpr int BK = 128;                     // columns of a k tile: one block of the scales, one 128-byte swizzle row
constexpr int A_BYTES = BM * BK;
constexpr int ATOM = 512;                   // scales of 128 rows x 4 k tiles
constexpr int SCALE_BYTES = 2048;           // of a stage: one atom of A, up to three of B
constexpr int MAX_STAGES = 8;
constexpr int SCALE_SETS = 3;               // sets of scales in TMEM, 16 columns each.  The set that k tiles 4q to 4q + 3 use was
                                            // read last by k tile 4q - 9; tile 4q is loaded when MAX_STAGES tiles before it are done
constexpr int SLAB_BYTES = BM * 128;
constexpr uint64_t WAIT_BUDGET_NS = 2000000000ull;
constexpr int groups(bool cl) { return cl ? 1 : 2; }
constexpr int threads(bool cl) { return 64 + 128 * groups(cl); }
static_assert(MAX_STAGES <= 4 * SCALE_SETS - 3, "scales in TMEM are overwritten while MMAs may read them");

struct Dev {
  void* C; const float* bias; int* status;
  const uint8_t *scale_a, *scale_b;
  long long M, N, ldc;                      // rows of the operand with 128-row tiles, of the other one, pitch of C
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
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// byte of the 16-byte piece q of row r in a [128][bn] fp32 tile; the XOR keeps a column of rows off a single bank
__device__ __forceinline__ uint32_t part_off(int r, int q, int bn) { return (uint32_t)(r * bn * 4 + ((q ^ (r & 7)) << 4)); }

__device__ __forceinline__ void store1(const Dev& d, long long i, float v) {
  if (d.out_fp32) ((float*)d.C)[i] = v; else ((__nv_bfloat16*)d.C)[i] = __float2bfloat16(v);
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
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          uint32_t v[32];
          tc05::tmem_ld_32x32(tacc + (uint32_t)c, v);
          tc05::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(tiles + part_off(r, (c >> 2) + j, BN)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
      } else if (d.tma_store) {
        // slabs 128 bytes wide (64 bf16 or 32 fp32 columns) leave with one TMA store each, clipped at the matrix edge
        const int cols = d.out_fp32 ? 32 : 64;
        const bool issuer = threadIdx.x == 64 + 128 * grp;
        const uint32_t row_off = (uint32_t)r * 128u, rsw = (uint32_t)(r & 7);
#pragma unroll 1
        for (int c = grp * cols; c < BN; c += G * cols) {
          if ((long long)n0 + c >= d.N) break;
          uint8_t* slab = slabs + (size_t)(2 * grp + (slab_i & 1u)) * SLAB_BYTES;
          if (issuer) tc05::bulk_wait_read<1>();   // the slab this group stored two slabs ago has been read out
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
      } else {
        // any pitch and alignment; with the operands swapped the lanes of a warp are neighbours in C
        const long long ri = d.swap ? 1 : d.ldc, ci = d.swap ? d.ldc : 1;
        const float bias_row = d.swap && d.bias != nullptr && row < d.M ? d.bias[row] : 0.f;
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
                if (!d.swap && d.bias != nullptr) v += __ldg(d.bias + col0 + j);
                if (d.relu) v = v < 0.f ? 0.f : v;
                store1(d, row * ri + (col0 + j) * ci, v);
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
    // this CTA finishes 128 / cluster rows of the tile, four columns per thread and step
    const int rank = (int)(blockIdx.x % d.cluster), mn = (int)(blockIdx.x / d.cluster);
    const int m0 = mn % d.m_tiles * BM, n0 = mn / d.m_tiles * BN;
    const int rows = BM / d.cluster, quads = BN >> 2;
    const uint32_t part = tc05::smem_u32(tiles);
    // a CTA that gave up left no partial tile: nobody stores (the status word names it)
    const uint32_t gave_up = ld_cluster_u32(tc05::map_to_cta(tc05::smem_u32(&ctl->abort_flag), lane % d.cluster));
    const int todo = __any_sync(0xffffffffu, gave_up != 0u) ? 0 : rows * quads;
    const long long ri = d.swap ? 1 : d.ldc, ci = d.swap ? d.ldc : 1;
    for (int i = threadIdx.x; i < todo; i += blockDim.x) {
      // neighbours in C are neighbouring threads
      const int rr = d.swap ? i % rows : i / quads, o = d.swap ? i / rows : i % quads;
      const int r = rank * rows + rr;
      const long long row = (long long)m0 + r, col0 = (long long)n0 + o * 4;
      if (row >= d.M || col0 >= d.N) continue;
      const uint32_t off = part_off(r, o, BN);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      for (int z = 0; z < d.cluster; ++z) {
        const float4 a = ld_cluster_f4(tc05::map_to_cta(part, z) + off);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      }
      const int nc = (int)min((long long)4, d.N - col0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e < nc) {
          if (d.bias != nullptr) v[e] += __ldg(d.bias + (d.swap ? row : col0 + e));
          if (d.relu) v[e] = v[e] < 0.f ? 0.f : v[e];
        }
      }
      if (!d.swap && !d.out_fp32 && nc == 4 && (((uintptr_t)((__nv_bfloat16*)d.C + row * d.ldc + col0)) & 7) == 0) {
        *reinterpret_cast<uint2*>((__nv_bfloat16*)d.C + row * d.ldc + col0) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < nc) store1(d, row * ri + (col0 + e) * ci, v[e]);
      }
    }
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
              int box_inner, int box_outer) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer}, one[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan { int swap, bn, cluster; };
// Tile widths: 64, 128 and 192 (two accumulators and the scales in 512 columns of TMEM), or 32 for a single tile.  The scales of a
// tile then begin at an even column of TMEM; an MMA whose scales begin at an odd one is a misaligned access.
bool width_ok(int bn, long long N) { return bn == 64 || bn == 128 || bn == 192 || (bn == 32 && N <= 32); }

// Whether an atom's worth of every slice is there
bool slices_ok(int quads, int cluster) { return (long long)((quads + cluster - 1) / cluster) * (cluster - 1) < quads; }

Plan choose(const GeepsGemmFp8* p, int sms) {
  const int quads = (int)((p->K + 511) / 512);
  Plan best = {0, 64, 1};
  double best_cost = 1e300;
  for (int swap = 0; swap < 2; ++swap) {
    const long long M = swap ? p->N : p->M, N = swap ? p->M : p->N;
    if (swap && p->M > 128) continue;
    const long long m_tiles = (M + BM - 1) / BM;
    for (int bn = 32; bn <= 192; bn += 32) {
      if (!width_ok(bn, N)) continue;
      const long long tiles = m_tiles * ((N + bn - 1) / bn);
      for (int cs = 1; cs <= 8; cs *= 2) {
        if (cs > 1 && !slices_ok(quads, cs)) continue;
        // SMs that whole clusters find in GPCs of different sizes
        const long long slots = cs <= 2 ? sms : cs == 4 ? sms * 9 / 10 / 4 * 4 : sms * 5 / 6 / 8 * 8;
        const long long rounds = (tiles * cs + slots - 1) / slots;
        if (cs > 1 && rounds > 1) continue;
        const double kt = 4.0 * ((quads + cs - 1) / cs);
        double cost = rounds * (kt * ((M < BM ? M : BM) + bn < 192 ? 192.0 : (double)((M < BM ? M : BM) + bn)) + 1200.0);
        if (cs > 1) cost += 1200.0 + 8.0 * bn;
        if (cost < best_cost * 0.98) { best_cost = cost; best = {swap, bn, cs}; }
      }
    }
  }
  return best;
}

template <bool CL>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Dev& d, int grid, cudaStream_t st) {
  const size_t smem = (size_t)d.stages * (A_BYTES + d.bn * BK + SCALE_BYTES) + (CL ? 0 : d.slabs * SLAB_BYTES) + sizeof(Ctl) + 1024;
  static std::atomic<unsigned long long> ready{0};           // devices on which the kernel may have all shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(ready >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(gemm_fp8_kernel<CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    ready |= 1ull << (dev & 63);
  }
  if (e != cudaSuccess) return (int)e;
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
      p->lda < p->K || p->ldb < p->K || p->ldc < p->N)
    return (int)cudaErrorInvalidValue;
  const int sms = geeps_sm_count();
  Plan plan = p->bn ? Plan{p->swap, p->bn, p->cluster} : choose(p, sms);
  Dev d = {};
  d.kt = (int)((p->K + BK - 1) / BK);
  d.quads = (d.kt + 3) / 4;
  if (!width_ok(plan.bn, plan.swap ? p->M : p->N) || plan.cluster < 1 || plan.cluster > 8 || (plan.cluster & (plan.cluster - 1)) ||
      !slices_ok(d.quads, plan.cluster))
    return (int)cudaErrorInvalidValue;
  d.C = p->C; d.bias = p->bias; d.status = p->status;
  d.swap = plan.swap; d.relu = p->relu; d.out_fp32 = p->out_fp32;
  d.M = plan.swap ? p->N : p->M; d.N = plan.swap ? p->M : p->N; d.ldc = p->ldc;
  d.scale_a = plan.swap ? p->scale_b : p->scale_a; d.scale_b = plan.swap ? p->scale_a : p->scale_b;
  const void *A = plan.swap ? p->B : p->A, *B = plan.swap ? p->A : p->B;
  const long long lda = plan.swap ? p->ldb : p->lda, ldb = plan.swap ? p->lda : p->ldb;
  const int size = p->out_fp32 ? 4 : 2;
  d.tma_store = plan.cluster == 1 && !plan.swap && ((uintptr_t)p->C & 15) == 0 && p->ldc * size % 16 == 0;
  d.bn = plan.bn;
  d.cluster = plan.cluster;
  d.m_tiles = (int)((d.M + BM - 1) / BM);
  const long long n_tiles = (d.N + d.bn - 1) / d.bn;
  if (n_tiles * d.m_tiles > 0x3fffffffLL) return (int)cudaErrorInvalidValue;
  d.n_tiles = (int)n_tiles;
  d.tmem_cols = 32;
  while (d.tmem_cols < 2 * d.bn + 16 * SCALE_SETS) d.tmem_cols <<= 1;
  CUtensorMap ta, tb, tc;
  if (!make_map(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, p->K, d.M, lda, BK, BM) || !make_map(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, B, p->K, d.N, ldb, BK, d.bn))
    return (int)cudaErrorInvalidValue;
  if (d.tma_store && !make_map(&tc, p->out_fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p->C, p->N, p->M,
                               p->ldc * size, p->out_fp32 ? 32 : 64, BM))
    d.tma_store = 0;
  if (!d.tma_store) tc = ta;   // unused by the kernel
  d.slabs = d.tma_store ? (d.bn > (p->out_fp32 ? 32 : 64) ? 4 : 2) : 0;
  const int stage = A_BYTES + d.bn * BK + SCALE_BYTES;
  d.stages = (224 * 1024 - d.slabs * SLAB_BYTES) / stage;
  if (d.stages > MAX_STAGES) d.stages = MAX_STAGES;
  const long long tiles = (long long)d.m_tiles * d.n_tiles;
  cudaStream_t st = (cudaStream_t)stream;
  if (d.cluster > 1) return launch<true>(ta, tb, tc, d, (int)(tiles * d.cluster), st);
  return launch<false>(ta, tb, tc, d, (int)(tiles < sms ? tiles : sms), st);
}

}  // extern "C"
