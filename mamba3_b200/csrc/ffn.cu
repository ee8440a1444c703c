// Gated feed-forward block, forward and backward (m3b_gated_ffn_fwd / _bwd).
//
//   g = x Wg^T + bg, u = x Wu^T + bu, a = silu(g) u, out = residual + s (a Wd^T + bd)
//   da = s dout Wd;  dg = da u sig(g) (1 + g (1 - sig(g)));  du = da g sig(g)
//   dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = s dout^T a
//   dbg, dbu, dbd = the column sums of dg, du, s dout
//
// Forward: one product whose tiles hold gate and up columns side by side, so the activation and the
// product are its epilogue (g and u never reach memory in inference), then the down product with
// bias, scale and residual in its epilogue.  Backward: da's product with dg and du as its epilogue;
// dx (one product over two K segments) and the three weight gradients side by side in one launch.
// Inference on at most kSmallRows rows (a decoding step) runs the matrix-vector form of ffn_small.cu.
// 18 rows d_model d_ff operations forward and backward, the least there are: g and u are kept in
// 24 bits or more (6 bytes a pair; fp32 8), because the rounding of a 16-bit copy would reach every gradient.
//
// 16384 x 768 x 2112 bf16, forward and backward, 509 us: gate | up 93 us (tensor pipe 66 % active; it writes
// 277 MB of act, g and u), down 48 us (71 %), dg and du 96 us (34 %: 12 K blocks a tile beside its g and u on
// their way in, dg and du out: 250 and 106 MB, 45 % of HBM's time), dx and the three weight gradients 192 us
// (87 %, 1.39 PFLOP/s).
#include "carve.h"
#include "ffn_small.h"
#include "gemm.cuh"

namespace m3b {

namespace {

constexpr int kMaxWidth = (1 << 22) - 64;  // column blocks of the bias gradients' grid

struct Dims {
  int64_t M;
  int D, F, np;
  bool f16, f32;
  explicit Dims(const m3b_gated_ffn_args* a)
      : M(a->rows), D(a->d_model), F(a->d_ff), np(a->dtype == M3B_F32 ? 3 : 1), f16(a->dtype == M3B_F16),
        f32(a->dtype == M3B_F32) {}
};

// A matrix as an operand: in place where the TMA can read it, else listed for packing into the workspace.
GemmOperand operand(const void* p, int64_t rows, int64_t cols, int64_t ld, const m3b_gated_ffn_args* a, Carve& ws,
                    PackList& packs) {
  if (a->dtype != M3B_F32 && tma_ok(p, ld)) return GemmOperand{p, rows, cols, ld, 0, 1};
  const int np = a->dtype == M3B_F32 ? 3 : 1;
  const int64_t ldp = up(cols, 8), plane = rows * ldp;
  void* dst = ws.take((size_t)np * plane * 2);
  packs.add(p, rows, cols, ld, dst, ldp, plane);
  return GemmOperand{dst, rows, cols, ldp, plane, np};
}

GemmOut result(void* p, int64_t ld, int dtype) {
  GemmOut o{};
  o.p = p;
  o.ld = ld;
  o.kind = dtype == M3B_BF16 ? kOutBf16 : dtype == M3B_F16 ? kOutF16 : kOutF32;
  o.vec = aligned16(p) && ld % 8 == 0;
  return o;
}

// Sums over the rows of up to three operands, times `scale`, in a fixed order.  A block takes 64 columns (two a
// lane) and kSumRows rows, its warps every eighth row, and leaves one partial; the chunks' partials
// are added by a second kernel.  dg and du of 16 bits are summed before they are rounded, by the epilogue that
// makes them (kEpiDgluSums), which leaves the partials of 32 rows: 16384 x 768 x 2112 bf16 with biases, forward and
// backward, 730 - 780 us, and 805 with the rounded dg and du read once more (2.1e-3 off, where the result's own
// rounding is 1.3e-3).
constexpr int kSumRows = 128;
struct Sums {
  struct {
    const uint16_t* x;
    int64_t plane, ld;
    int cols;
    float scale;
    const float* num;  // scale *= *num, or null
    void* out;
    float* part;       // [parts][cols]
    int parts;
  } s[3];
  int n, f16, planes, dt;
  int made;            // of the n, the first ones whose partials colsum_kernel makes
  int64_t rows;
};
__global__ void __launch_bounds__(256) colsum_kernel(const __grid_constant__ Sums a) {
  __shared__ float2 sm[8][32];
  pdl_wait_primary();
  pdl_launch_dependents();
  const auto& m = a.s[blockIdx.z];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.y * 64 + 2 * lane;
  const int64_t r0 = (int64_t)blockIdx.x * kSumRows, r1 = r0 + kSumRows < a.rows ? r0 + kSumRows : a.rows;
  float2 s = make_float2(0.f, 0.f);
  if (c < m.cols) {
#pragma unroll 8
    for (int64_t r = r0 + w; r < r1; r += 8) {
      for (int k = a.planes - 1; k >= 0; --k) {
        const uint16_t* p = m.x + k * m.plane + r * m.ld + c;
        const uint32_t v = c + 1 < m.cols ? *reinterpret_cast<const uint32_t*>(p) : (uint32_t)*p;
        const float2 f = a.f16 ? __half22float2(*reinterpret_cast<const __half2*>(&v)) : bf2_to_f2(v);
        s.x += f.x;
        s.y += f.y;
      }
    }
  }
  sm[w][lane] = s;
  __syncthreads();
  if (w != 0 || c >= m.cols) return;
  for (int k = 1; k < 8; ++k) s.x += sm[k][lane].x, s.y += sm[k][lane].y;
  float* o = m.part + (int64_t)blockIdx.x * m.cols + c;
  o[0] = s.x;
  if (c + 1 < m.cols) o[1] = s.y;
}
__global__ void __launch_bounds__(256) colsum_finish_kernel(const __grid_constant__ Sums a) {
  __shared__ float sm[8][32];
  pdl_wait_primary();
  const auto& m = a.s[blockIdx.y];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < m.cols) {
#pragma unroll 4
    for (int k = w; k < m.parts; k += 8) s += m.part[(int64_t)k * m.cols + c];
  }
  sm[w][lane] = s;
  __syncthreads();
  if (w != 0 || c >= m.cols) return;
  for (int k = 1; k < 8; ++k) s += sm[k][lane];
  stf(m.out, c, a.dt, s * (m.num ? m.scale * *m.num : m.scale));
}
int colsums(const Sums& a, cudaStream_t st) {
  if (a.n == 0) return M3B_OK;
  int cols = 0;
  for (int i = 0; i < a.n; ++i) cols = a.s[i].cols > cols ? a.s[i].cols : cols;
  int rc = M3B_OK;
  if (a.made)
    rc = launch_dependent(colsum_kernel, dim3((unsigned)((a.rows + kSumRows - 1) / kSumRows), (cols + 63) / 64, a.made), 256,
                          st, a);
  return rc != M3B_OK ? rc : launch_dependent(colsum_finish_kernel, dim3((cols + 31) / 32, a.n), 256, st, a);
}

// fp16's smallest step is 6e-8: dg and du of an unscaled mean loss, near 1e-5, would lose most of their bits.  They
// are kept divided by a power of two that brings the largest |s dout| up to 2^-8 (larger ones stay as they are),
// and the products that read them multiply it back in fp32.  Not further up: with g and u within
// fp16 themselves, dg and du can then pass 65504 only where a column of w_down has a sum of magnitudes above 100,
// so no step that was finite becomes infinite, as a loss scaler that lowers its scale in vain would see it.
// Largest finite |s dout| of each block's rows; rows start on 16 bytes.  Bound by HBM's latency: 67 MB in 16 us, 0.6 % of
// the step that has them (128 blocks: 21).
constexpr int kPeakBlocks = 296;
__global__ void __launch_bounds__(512) peak_kernel(const uint16_t* __restrict__ x, int64_t rows, int D, int64_t ld,
                                                   float scale, float* __restrict__ peaks) {
  __shared__ uint32_t sm[16];
  pdl_wait_primary();
  pdl_launch_dependents();
  uint32_t top = 0;
  auto take = [&](uint32_t h) {
    h &= 0x7fffu;
    if (h < 0x7c00u && h > top) top = h;
  };
  const int eights = D / 8, tail = D - 8 * eights, lane = threadIdx.x & 31;
  for (int64_t r = blockIdx.x * 16 + (threadIdx.x >> 5); r < rows; r += kPeakBlocks * 16) {
    const uint4* row = reinterpret_cast<const uint4*>(x + r * ld);
#pragma unroll 4
    for (int c = lane; c < eights; c += 32) {
      const uint4 w = __ldg(row + c);
      take(w.x), take(w.x >> 16), take(w.y), take(w.y >> 16), take(w.z), take(w.z >> 16), take(w.w), take(w.w >> 16);
    }
    if (lane < tail) take(x[r * ld + 8 * eights + lane]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) sm[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int k = 1; k < 16; ++k) top = sm[k] > top ? sm[k] : top;
  peaks[blockIdx.x] = __half2float(__ushort_as_half((unsigned short)top)) * fabsf(scale);
}

int check(const m3b_gated_ffn_args* a, bool bwd) {
  if (!a) return fail(M3B_ERR_INVALID_ARG, "gated_ffn: null args");
  if (a->rows < 0 || a->d_model <= 0 || a->d_ff <= 0) return fail(M3B_ERR_INVALID_ARG, "gated_ffn: bad sizes");
  if (a->rows > (int64_t(1) << 31) - 512 || a->d_model > kMaxWidth || a->d_ff > kMaxWidth)
    return fail(M3B_ERR_INVALID_ARG, "gated_ffn: sizes past the kernels' limits");
  if (a->dtype != M3B_F32 && a->dtype != M3B_BF16 && a->dtype != M3B_F16)
    return fail(M3B_ERR_INVALID_ARG, "gated_ffn: dtype");
  if (!a->w_gate || !a->w_up || !a->w_down || (a->rows && (!a->x || !a->saved_act)))
    return fail(M3B_ERR_INVALID_ARG, "gated_ffn: null pointer");
  if ((a->b_gate == nullptr) != (a->b_up == nullptr))
    return fail(M3B_ERR_INVALID_ARG, "gated_ffn: b_gate and b_up go together");
  if (a->x_stride < a->d_model || (a->residual && a->residual_stride < a->d_model))
    return fail(M3B_ERR_INVALID_ARG, "gated_ffn: row strides shorter than the rows");
  if (!aligned16(a->saved_act) || !aligned16(a->saved_gu))
    return fail(M3B_ERR_ALIGNMENT, "gated_ffn: saved buffers must be 16-byte aligned");
  if (bwd) {
    if (a->rows && (!a->dout || !a->saved_gu)) return fail(M3B_ERR_INVALID_ARG, "gated_ffn_bwd: null pointer");
    if (a->rows && a->dout_stride < a->d_model) return fail(M3B_ERR_INVALID_ARG, "gated_ffn_bwd: dout stride");
  } else if (a->rows && !a->out) {
    return fail(M3B_ERR_INVALID_ARG, "gated_ffn_fwd: null pointer");
  }
  return M3B_OK;
}

bool sizes_ok(const m3b_gated_ffn_args* a) {
  return a && a->rows >= 0 && a->d_model > 0 && a->d_ff > 0 &&
         (a->dtype == M3B_F32 || a->dtype == M3B_BF16 || a->dtype == M3B_F16);
}

GemmOperand act_operand(const m3b_gated_ffn_args* a, void* p) {
  const Dims d(a);
  const int64_t ld = up(d.F, 8);
  return GemmOperand{p, d.M, d.F, ld, d.M * ld, d.np};
}

#define M3B_MAP(...) M3B_TRY(gemm_map(__VA_ARGS__))

GemmParams params(const Dims& d, const m3b_gated_ffn_args* a, int bn) {
  GemmParams p{};
  p.bn = bn;
  p.npass = d.f32 ? 6 : 1;
  p.f16 = d.f16;
  p.err = a->err;
  return p;
}
int blocks_of(int64_t k) { return (int)((k + kGmBK - 1) / kGmBK); }

// run == false only measures the workspace.
int forward(const m3b_gated_ffn_args* a, void* workspace, size_t* need, bool run, cudaStream_t st) {
  const Dims d(a);
  // Few rows and nothing to save: 1 row of 768 x 2112 took 18 us of three tensor-core launches.
  if (d.M <= kSmallRows && !a->saved_gu) {
    *need = 0;
    if (!run) return M3B_OK;
    SmallFfn p{};
    p.M = (int)d.M, p.D = d.D, p.F = d.F;
    p.x_stride = a->x_stride, p.res_stride = a->residual_stride;
    p.ld_act = up(d.F, 8);
    p.x = a->x, p.w_gate = a->w_gate, p.w_up = a->w_up, p.w_down = a->w_down;
    p.b_gate = a->b_gate, p.b_up = a->b_up, p.b_down = a->b_down, p.residual = a->residual;
    p.act = a->saved_act, p.out = a->out;
    p.scale = a->residual_scale;
    const int v = d.f32 ? 4 : 8;
    p.vec = aligned16(a->x) && aligned16(a->w_gate) && aligned16(a->w_up) && aligned16(a->w_down) && d.D % v == 0 &&
            d.F % v == 0 && a->x_stride % v == 0;
    return launch_small_ffn(p, a->dtype, st);
  }
  Carve ws(workspace);
  PackList packs;
  const GemmOperand x = operand(a->x, d.M, d.D, a->x_stride, a, ws, packs);
  const GemmOperand wg = operand(a->w_gate, d.F, d.D, d.D, a, ws, packs);
  const GemmOperand wu = operand(a->w_up, d.F, d.D, d.D, a, ws, packs);
  const GemmOperand wd = operand(a->w_down, d.D, d.F, d.F, a, ws, packs);
  const GemmOperand act = act_operand(a, a->saved_act);
  const bool pair = d.M > 128;

  GemmParams p = params(d, a, pair ? gemm_columns(d.M, 2 * (int64_t)d.F, d.f32) : 128);
  GemmSub& s = p.sub[0];
  p.nsub = 1;
  s.M = (int)d.M;
  s.N = d.F;
  s.nk[0] = blocks_of(d.D);
  s.bias = a->b_gate;
  s.bias2 = a->b_up;
  s.dt = a->dtype;
  p.gu = static_cast<uint8_t*>(a->saved_gu);
  p.gu_ld = up(d.F, 32) / 8;
  plan_gemm(p, kEpiGlu, pair);

  GemmParams q = params(d, a, pair ? (d.f32 ? 128 : 256) : 64);
  GemmSub& t = q.sub[0];
  q.nsub = 1;
  t.M = (int)d.M;
  t.N = d.D;
  t.nk[0] = blocks_of(d.F);
  t.out = result(a->out, d.D, a->dtype);
  t.alpha = a->residual_scale;
  t.bias = a->b_down;
  t.residual = a->residual;
  t.ld_res = a->residual_stride;
  t.res_vec = aligned16(a->residual) && a->residual_stride % 4 == 0;
  t.dt = a->dtype;
  void* parts = ws.take(plan_gemm(q, kEpiFinal, pair));
  *need = ws.at;
  if (!run) return M3B_OK;
  M3B_TRY(launch_pack(packs, a->dtype, st));

  M3B_MAP(&s.a[0], x, false, 128, d.f16);
  M3B_MAP(&s.b[0], wg, false, gemm_box_b(pair, p.bn, kEpiGlu), d.f16);
  M3B_MAP(&s.b[1], wu, false, gemm_box_b(pair, p.bn, kEpiGlu), d.f16);
  M3B_TRY(gemm_out_map(&p.o[0], act, d.f16));
  M3B_TRY(launch_gemm(p, kEpiGlu, pair, nullptr, st));
  M3B_MAP(&t.a[0], act, false, 128, d.f16);
  M3B_MAP(&t.b[0], wd, false, gemm_box_b(pair, q.bn, kEpiFinal), d.f16);
  return launch_gemm(q, kEpiFinal, pair, parts, st);
}

int backward(const m3b_gated_ffn_args* a, void* workspace, size_t* need, bool run, cudaStream_t st) {
  const Dims d(a);
  Carve ws(workspace);
  PackList packs;
  const GemmOperand x = operand(a->x, d.M, d.D, a->x_stride, a, ws, packs);
  const GemmOperand wg = operand(a->w_gate, d.F, d.D, d.D, a, ws, packs);
  const GemmOperand wu = operand(a->w_up, d.F, d.D, d.D, a, ws, packs);
  const GemmOperand wd = operand(a->w_down, d.D, d.F, d.F, a, ws, packs);
  const GemmOperand dy = operand(a->dout, d.M, d.D, a->dout_stride, a, ws, packs);
  const size_t one = (size_t)act_operand(a, nullptr).plane * d.np * 2;
  const GemmOperand dg = act_operand(a, ws.take(one)), du = act_operand(a, ws.take(one));
  const GemmOperand act = act_operand(a, a->saved_act);
  Sums sums{};
  sums.f16 = d.f16, sums.planes = d.np, sums.dt = a->dtype, sums.rows = d.M;
  float* peaks = d.f16 ? static_cast<float*>(ws.take((kPeakBlocks + 1) * 4)) : nullptr;
  float* peak = peaks ? peaks + kPeakBlocks : nullptr;
  // of an operand, or of the partials that the epilogue leaves of it
  auto sum = [&](const GemmOperand& o, bool made, float scale, const float* num, void* out) {
    const int64_t rows = made ? kSumRows : 32;
    const int parts = (int)((d.M + rows - 1) / rows);
    float* part = static_cast<float*>(ws.take((size_t)parts * o.cols * 4));
    if (out) sums.s[sums.n++] = {static_cast<const uint16_t*>(o.p), o.plane, o.ld, (int)o.cols, scale, num, out, part, parts};
    if (out && made) ++sums.made;
    return part;
  };
  if (a->db_down) sum(dy, true, a->residual_scale, nullptr, a->db_down);
  const bool in_epilogue = !d.f32 && (a->db_gate || a->db_up);
  float *sum_g = nullptr, *sum_u = nullptr;
  if (in_epilogue || a->db_gate) sum_g = sum(dg, !in_epilogue, 1.f, peak, a->db_gate);
  if (in_epilogue || a->db_up) sum_u = sum(du, !in_epilogue, 1.f, peak, a->db_up);
  int* ticket = static_cast<int*>(ws.take(4));

  // dx and the three weight gradients, side by side
  GemmParams q = params(d, a, d.f32 ? 128 : 256);
  q.ticket = ticket;
  struct Product {
    void* out;
    const GemmOperand *a[2], *b[2];
    bool a_mn;
    int64_t M, N, K;
    float alpha;
    const float* num;
  };
  const Product all[4] = {{a->dx, {&dg, &du}, {&wg, &wu}, false, d.M, d.D, d.F, 1.f, peak},
                          {a->dw_gate, {&dg, nullptr}, {&x, nullptr}, true, d.F, d.D, d.M, 1.f, peak},
                          {a->dw_up, {&du, nullptr}, {&x, nullptr}, true, d.F, d.D, d.M, 1.f, peak},
                          {a->dw_down, {&dy, nullptr}, {&act, nullptr}, true, d.D, d.F, d.M, a->residual_scale, nullptr}};
  for (const Product& e : all) {
    if (!e.out) continue;
    GemmSub& s = q.sub[q.nsub++];
    for (int k = 0; k < 2 && e.a[k]; ++k) {
      if (run) {
        M3B_MAP(&s.a[k], *e.a[k], e.a_mn, 128, d.f16);
        M3B_MAP(&s.b[k], *e.b[k], true, 0, d.f16);
      }
      s.nk[k] = blocks_of(e.K);
    }
    s.a_mn = e.a_mn;
    s.b_mn = 1;
    s.M = (int)e.M;
    s.N = (int)e.N;
    s.alpha = e.alpha;
    s.alpha_num = e.num;
    s.out = result(e.out, e.N, a->dtype);
  }
  void* parts = ws.take(plan_gemm(q, kEpiStore, true));
  *need = ws.at;
  if (!run) return M3B_OK;
  M3B_TRY(launch_pack(packs, a->dtype, st));
  if (d.f16)
    M3B_TRY(launch_dependent(peak_kernel, dim3(kPeakBlocks), 512, st, static_cast<const uint16_t*>(dy.p), d.M, d.D, dy.ld,
                             a->residual_scale, peaks));
  {  // da -> dg, du
    GemmParams p = params(d, a, gemm_columns(d.M, d.F, d.f32));
    GemmSub& s = p.sub[0];
    p.nsub = 1;
    M3B_MAP(&s.a[0], dy, false, 128, d.f16);
    M3B_MAP(&s.b[0], wd, true, 0, d.f16);
    s.b_mn = 1;
    s.M = (int)d.M;
    s.N = d.F;
    s.nk[0] = blocks_of(d.D);
    s.alpha = a->residual_scale;
    M3B_TRY(gemm_out_map(&p.o[0], dg, d.f16));
    M3B_TRY(gemm_out_map(&p.o[1], du, d.f16));
    p.gu = static_cast<uint8_t*>(a->saved_gu);
    p.gu_ld = up(d.F, 32) / 8;
    p.clear = ticket;
    if (d.f16) {
      p.peaks = peaks;
      p.npeaks = kPeakBlocks;
      p.peak_out = peak;
    }
    p.sum_g = sum_g;
    p.sum_u = sum_u;
    const int epi = in_epilogue ? kEpiDgluSums : kEpiDglu;
    plan_gemm(p, epi, true);
    M3B_TRY(launch_gemm(p, epi, true, nullptr, st));
  }
  if (q.nsub) M3B_TRY(launch_gemm(q, kEpiStore, true, parts, st));
  return colsums(sums, st);
}

int check_workspace(size_t need, const void* ws, size_t bytes) {
  if (need == 0) return M3B_OK;
  if (!ws || bytes < need) return fail(M3B_ERR_WORKSPACE, "gated_ffn: workspace of %zu bytes, %zu needed", bytes, need);
  if (!aligned16(ws)) return fail(M3B_ERR_ALIGNMENT, "gated_ffn: workspace must be 16-byte aligned");
  return M3B_OK;
}

}  // namespace

}  // namespace m3b

extern "C" {

size_t m3b_gated_ffn_act_bytes(const m3b_gated_ffn_args* a) {
  if (!m3b::sizes_ok(a)) return 0;
  const m3b::GemmOperand o = m3b::act_operand(a, nullptr);
  return (size_t)o.planes * o.plane * 2;
}

size_t m3b_gated_ffn_gu_bytes(const m3b_gated_ffn_args* a) {
  if (!m3b::sizes_ok(a)) return 0;
  return (size_t)m3b::up(a->rows, 256) * m3b::up(a->d_ff, 32) * (a->dtype == M3B_F32 ? 8 : 6);
}

size_t m3b_gated_ffn_fwd_workspace(const m3b_gated_ffn_args* a) {
  size_t need = 0;
  if (m3b::sizes_ok(a) && a->rows) m3b::forward(a, nullptr, &need, false, nullptr);
  return need;
}

int m3b_gated_ffn_fwd(const m3b_gated_ffn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  m3b::clear_error();
  int rc = m3b::check(a, false);
  if (rc != M3B_OK || a->rows == 0) return rc;
  size_t need = 0;
  m3b::forward(a, nullptr, &need, false, nullptr);
  rc = m3b::check_workspace(need, workspace, workspace_bytes);
  return rc != M3B_OK ? rc : m3b::forward(a, workspace, &need, true, static_cast<cudaStream_t>(stream));
}

size_t m3b_gated_ffn_bwd_workspace(const m3b_gated_ffn_args* a) {
  size_t need = 0;
  if (m3b::sizes_ok(a) && a->rows) m3b::backward(a, nullptr, &need, false, nullptr);
  return need;
}

int m3b_gated_ffn_bwd(const m3b_gated_ffn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  m3b::clear_error();
  int rc = m3b::check(a, true);
  if (rc != M3B_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->rows == 0) {  // no rows: every sum is zero
    const size_t es = a->dtype == M3B_F32 ? 4 : 2, F = (size_t)a->d_ff, D = (size_t)a->d_model;
    const struct {
      void* p;
      size_t n;
    } z[] = {{a->dw_gate, F * D}, {a->dw_up, F * D}, {a->dw_down, F * D},
             {a->db_gate, F},     {a->db_up, F},     {a->db_down, D}};
    for (const auto& e : z)
      if (e.p && cudaMemsetAsync(e.p, 0, e.n * es, st) != cudaSuccess) return m3b::check_launch("gated_ffn_bwd");
    return M3B_OK;
  }
  size_t need = 0;
  m3b::backward(a, nullptr, &need, false, nullptr);
  rc = m3b::check_workspace(need, workspace, workspace_bytes);
  return rc != M3B_OK ? rc : m3b::backward(a, workspace, &need, true, st);
}

}  // extern "C"
