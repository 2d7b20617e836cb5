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
//
// What bounds them, in parts of the copy rate: whole, aligned rows of 1024 bf16 channels move at 0.81 forward and 0.72 backward (50176
// rows, 5.3 and 4.7 TB/s), of 576 at 0.66 and 0.76, the rest being issue slots, start and end, and the meeting of a row's warps with
// few rows on an SM, which leaves 0.43 to 0.20 of 4096 channels and more backward.  Odd widths and addresses go column by column and
// are bound by instructions (0.28 at 1003 channels backward); narrow rows with one gate for all by the launch that joins its shares
// (125552 x 32 backward 0.19); calls of a few rows by the launch and one round trip to memory.
#include "norm_kernels.cuh"

using namespace rownorm;

namespace {

struct Use { const void* p; long long ld, rows; int size; bool out; };
bool vectors_ok(const Use& u, int C) {
  if (!u.p) return true;
  const uintptr_t line = kVec * u.size - 1;
  return ((uintptr_t)u.p & line) == 0 && (u.rows <= 1 || ((uintptr_t)(u.ld * u.size) & line) == 0) && C % kVec == 0;
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
  if (pa == pb && pa) {                    // a single row may have a pitch of zero
    const uintptr_t d = a0 <= b0 ? (b0 - a0) % pa : (pa - (a0 - b0) % pa) % pa;      // bytes from a's first column to b's
    if (d >= wa && d + wb <= pa) return false;
  }
  return true;
}

// A parameter, its gradient or statistics: `n` floats
struct Column { const void* p; long long n; bool out; };
bool meet(const void* a, uintptr_t na, const void* b, uintptr_t nb) {
  return a && b && na && nb && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

int check(const GeepsResidual& p, bool backward, int mode, bool* vec) {
  if (p.C < 1 || p.C > kMaxChannels) return GEEPS_ERR_NORM_CHANNELS;
  if (p.rows < 0 || p.rows > 1LL << 30) return (int)cudaErrorInvalidValue;
  // without rows any number of images goes: each has none
  if (p.gate && (p.rows ? p.gate_rows < 1 || p.gate_rows > p.rows || p.rows % p.gate_rows : p.gate_rows < 0)) return GEEPS_ERR_NORM_GATE;
  if (p.gate && p.gate_rows > 1LL << 30) return (int)cudaErrorInvalidValue;
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
    if (u[i].p && u[i].rows > 1 && (u[i].ld < (u[i].out ? p.C : 0) || u[i].ld >= 1LL << 29)) return (int)cudaErrorInvalidValue;
    *vec = *vec && vectors_ok(u[i], p.C);
    for (int j = 0; j < i; ++j) if (clash(u[i], u[j], p.C)) return GEEPS_ERR_NORM_OVERLAP;
  }
  // the columns' gradients last: backward only
  const Column v[] = {{p.post.stats, 2 * n, !backward}, {p.pre.stats, 2 * n, !backward}, {p.scale, p.C, false},
                      {p.post.weight, p.C, false}, {p.post.bias, p.C, false}, {p.pre.weight, p.C, false}, {p.pre.bias, p.C, false},
                      {p.dscale, p.C, true}, {p.post.dweight, p.C, true}, {p.post.dbias, p.C, true}, {p.pre.dweight, p.C, true},
                      {p.pre.dbias, p.C, true}};
  const int columns = backward ? 12 : 7;
  uintptr_t off = ((uintptr_t)p.post.stats | (uintptr_t)p.pre.stats | (uintptr_t)p.work) & 7;
  for (int i = 0; i < count; ++i) off |= (uintptr_t)u[i].p & (u[i].size - 1);
  for (int i = 0; i < columns; ++i) off |= (uintptr_t)v[i].p & 3;
  if (off) return GEEPS_ERR_NORM_ALIGN;
  for (int i = 0; i < columns; ++i) {
    for (int j = 0; j < i; ++j)
      if ((v[i].out || v[j].out) && meet(v[i].p, 4 * v[i].n, v[j].p, 4 * v[j].n)) return GEEPS_ERR_NORM_OVERLAP;
    for (int j = 0; j < count; ++j)
      if ((v[i].out || u[j].out) && u[j].rows &&
          meet(v[i].p, 4 * v[i].n, u[j].p, ((uintptr_t)(u[j].rows - 1) * u[j].ld + p.C) * u[j].size)) return GEEPS_ERR_NORM_OVERLAP;
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

// Sums over no rows: the parameters' gradients, and the gate's where there are images
__global__ void clear_sums_kernel(const __grid_constant__ GeepsResidual p) {
  geeps_pdl_enter();
  const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x, step = (long long)gridDim.x * blockDim.x;
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  if (at < p.C) write_sums(p, p.mode, (int)at, zero);
  if (!p.gate || !p.dgate) return;
  for (long long i = at; i < p.gate_rows * p.C; i += step) {
    const long long to = i / p.C * p.lddgate + i % p.C;
    if (p.block_fp32) ((float*)p.dgate)[to] = 0.f;
    else ((__nv_bfloat16*)p.dgate)[to] = __float2bfloat16(0.f);
  }
}

int residual(const GeepsResidual* q, bool backward, void* stream) {
  if (!q) return (int)cudaErrorInvalidValue;
  const GeepsResidual& p = *q;
  const int mode = p.mode;
  if (mode < MODE_NORM || mode > MODE_BOTH) return (int)cudaErrorInvalidValue;
  bool vec = true;
  const int bad = check(p, backward, mode, &vec);
  if (bad) return bad;
  cudaStream_t st = (cudaStream_t)stream;
  if (p.rows == 0) {
    if (!backward) return 0;
    const long long values = p.gate && p.dgate && p.gate_rows > 1 ? p.gate_rows * p.C : p.C, blocks = (values + 255) / 256;
    geeps_launch(clear_sums_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, p);
    return (int)cudaGetLastError();
  }
  if (backward && !p.work && geeps_residual_work(p.rows, p.gate ? p.gate_rows : 0, p.C, mode) > 0) return (int)cudaErrorInvalidValue;
  if (!(!p.stream_fp32 ? run_bf16 : !p.block_fp32 ? run_mixed : run_fp32)(p, backward, vec, st)) return (int)cudaErrorNotSupported;
  return (int)cudaGetLastError();
}

}  // namespace

// The most that any layout and types of these sizes take
extern "C" long long geeps_residual_work(long long rows, long long gate_rows, int C, int mode) {
  if (rows <= 0 || C < 1 || C > kMaxChannels || mode < MODE_NORM || mode > MODE_BOTH) return 0;
  const bool by_image = gate_rows > 0 && gate_rows < rows;
  long long most = 0;
  for (int form = 0; form < 6; ++form) {
    Call c = {true, form < 3, gate_rows == rows, by_image, false, mode, form % 3 ? 4 : 2, form % 3 == 2 ? 4 : 2};
    const Shape s = plan(rows, C, c);
    c.tile = s.tiles > 1;
    // of rows in tiles the means, and what one tile takes at a time: the widest or the last, which may have more blocks
    for (int width : {s.width, C - (s.tiles - 1) * s.width}) {
      const Shape t = s.tiles > 1 ? plan(rows, width, c) : s;
      const long long n = (s.tiles > 1 ? 4 * rows : 0) + (t.blocks == 1 && !by_image ? 0 : work_floats(t, width, mode, by_image ? gate_rows : 0));
      most = n > most ? n : most;
    }
  }
  return most;
}
extern "C" int geeps_residual_forward(const GeepsResidual* p, void* stream) { return residual(p, false, stream); }
extern "C" int geeps_residual_backward(const GeepsResidual* p, void* stream) { return residual(p, true, stream); }
extern "C" int geeps_norm_shape(long long rows, long long gate_rows, int C, int mode, int backward, int vec, int stream_fp32, int block_fp32,
                                int* out) {
  const bool by_pixel = gate_rows == rows, by_image = gate_rows > 0 && gate_rows < rows;
  const Shape s = plan(rows, C, {backward != 0, vec != 0, by_pixel, by_image, false, mode, stream_fp32 ? 4 : 2, block_fp32 ? 4 : 2});
  const int v[10] = {s.vectors, s.slot, s.slots, s.blocks, s.per_sm, s.depth, (int)s.smem, s.large, s.tiles, s.width};
  for (int i = 0; i < 10; ++i) out[i] = v[i];
  const bool direct = s.large ? mode == MODE_BOTH || (vec && mode == MODE_JOIN) : !vec && s.wide && s.depth == 0 && mode != MODE_NORM;
  return s.tiles > 1 || direct || planned(backward, vec, s.slot >= 32, s.wide, s.vectors, mode, by_pixel, block_fp32 ? 4 : 2) ? 0 : (int)cudaErrorNotSupported;
}
extern "C" int geeps_norm_sums_shape(long long rows, long long gate_rows, int C, int mode, int vec, int stream_fp32, int block_fp32, int* out) {
  const bool by_image = gate_rows > 0 && gate_rows < rows;
  const Call c = {true, vec != 0, gate_rows == rows, by_image, false, mode, stream_fp32 ? 4 : 2, block_fp32 ? 4 : 2};
  Shape s = plan(rows, C, c);
  int width = C;
  if (s.tiles > 1) {
    Call t = c;
    t.tile = true;
    width = s.width;
    s = plan(rows, width, t);
  }
  const SumsShape q = plan_sums(rows, gate_rows, width, by_image, s);
  const int v[4] = {q.x, q.y, q.parts, q.merged};
  for (int i = 0; i < 4; ++i) out[i] = v[i];
  return 0;
}
