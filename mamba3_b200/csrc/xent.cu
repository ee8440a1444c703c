// Cross entropy of the language-model head from the hidden states (m3b_linear_xent_fwd / _bwd).
//
//   z = h W^T;  lse_i = log sum_v exp(z_iv);  loss_i = lse_i - z_i[t_i]
//   dz_iv = w_i (exp(z_iv - lse_i) - [v = t_i]);  dh = dz W;  dW = dz^T h
// with w_i = dloss / kept rows (mean), dloss (sum) or dloss_i.
//
// The kept rows are first gathered into a dense operand, so ignored tokens cost nothing in any
// product (and what they hold, NaN included, reaches no sum); how many remain is read on the device.
// Forward: one product over all vocabulary tiles whose epilogue keeps each row's running maximum
// and sum and the target's logit; the logits never leave the SM.  A small kernel
// joins the tiles' statistics.  Backward: a piece of the vocabulary at a time, the logits once more
// with the softmax as their epilogue, and the piece's share of both gradients; dh is summed over the
// pieces in fp32.  8 rows d_model vocab operations forward and backward, 2 more than with the
// logits kept.  At most kSmallXentRows rows take the matrix-vector form of xent_small.cu.
//
// Bound by the tensor cores, and in long runs by the power they draw.  4096 x 768 x 32000 bf16, each launch by
// itself at 1.6 - 1.7 GHz: the forward product 113 us (tensor pipe 92 % active, 1.77 PFLOP/s), softmax - onehot
// 127 us (80 %; what else it takes is its 262 MB on their way out), both gradients 244 us (87 %, 1.65 PFLOP/s); the
// kept rows' numbers, their copy, the join and the gradients' join 5, 6, 9 and 16 us.  With four tenths of the
// targets ignored 71, 85, 152 and 5, 6, 9 and 14 us, and 441 us a call of a long run, whose clock is lower.
#include "carve.h"
#include "gemm.cuh"
#include "xent_small.h"

namespace m3b {

namespace {

constexpr size_t kPieceBytes = size_t(256) << 20;  // of softmax - onehot in memory at once
constexpr int kPieceLeast = 2048;                   // columns of a piece at least

struct Saved {
  uint16_t* h;     // [planes][Tp][Dp] kept rows
  int* row;        // [Tp] where they come from
  int* target;     // [Tp]; -1 behind the last, -2 out of range
  float2* stat;    // [Tp] maximum, and log2 of the sum of exp(z - maximum)
  int* count;      // kept rows; blocks of the join kernel that are done
  size_t bytes;
};

struct Dims {
  int64_t T, Tp, Dp;
  int D, V, np;
  bool f16, f32;
  explicit Dims(const m3b_linear_xent_args* a)
      : T(a->rows), Tp(up(a->rows, 256)), Dp(up(a->d_model, 8)), D(a->d_model), V(a->vocab),
        np(a->dtype == M3B_F32 ? 3 : 1), f16(a->dtype == M3B_F16), f32(a->dtype == M3B_F32) {}
};

Saved saved_of(const m3b_linear_xent_args* a, void* p) {
  const Dims d(a);
  Carve c(p);
  Saved s{};
  s.h = static_cast<uint16_t*>(c.take((size_t)d.np * d.Tp * d.Dp * 2));
  s.row = static_cast<int*>(c.take((size_t)d.Tp * 4));
  s.target = static_cast<int*>(c.take((size_t)d.Tp * 4));
  s.stat = static_cast<float2*>(c.take((size_t)d.Tp * 8));
  s.count = static_cast<int*>(c.take(8));
  s.bytes = c.at;
  return s;
}

// One block: the kept rows' numbers and targets in order, four targets a thread at a time.  (One long
// run per thread, its loads a line each: 52 us for 16384 targets; this 8 us.)
__global__ void __launch_bounds__(1024) keep_kernel(const int64_t* __restrict__ target, int64_t ignore, int64_t T,
                                                    int64_t Tp, int V, Saved s, int* err) {
  __shared__ int sums[2][32];
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int total = 0, side = 0;
  for (int64_t base = 0; base < T; base += 4096, side ^= 1) {
    const int64_t r0 = base + tid * 4;
    int64_t t[4];
    int n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = r0 + k < T ? target[r0 + k] : ignore;
#pragma unroll
    for (int k = 0; k < 4; ++k) n += t[k] != ignore;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[side][warp] = x;
    __syncthreads();  // the other side is written next, so one barrier a turn is enough
    int w = sums[side][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    int at = total + x - n + (warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0);
    total += __shfl_sync(0xffffffffu, w, 31);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (t[k] == ignore) continue;
      const bool ok = t[k] >= 0 && t[k] < V;
      if (!ok) record_error(err, M3B_ERR_INVALID_ARG);
      s.row[at] = (int)(r0 + k);
      s.target[at] = ok ? (int)t[k] : -2;
      ++at;
    }
  }
  for (int64_t i = total + tid; i < Tp; i += 1024) {
    s.row[i] = -1;
    s.target[i] = -1;
  }
  if (tid == 0) {
    s.count[0] = total;
    s.count[1] = 0;
  }
}

// One warp per row of the dense operand; rows behind the last kept one are zero up to the tile's end.
__global__ void __launch_bounds__(256) gather_kernel(const void* __restrict__ h, int dt, int64_t ld, int D, int64_t Tp,
                                                     int64_t Dp, int vec, Saved s) {
  pdl_wait_primary();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t n = *s.count, end = (n + 255) / 256 * 256 < Tp ? (n + 255) / 256 * 256 : Tp;
  const int64_t step = (int64_t)gridDim.x * 8, plane = Tp * Dp;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < end; i += step) {
    const int64_t r = s.row[i];
    uint16_t* dst = s.h + i * Dp;
    if (dt != M3B_F32) {
      const uint16_t* src = static_cast<const uint16_t*>(h) + r * ld;
      if (vec) {
        for (int c = lane; c < D / 8; c += 32)
          reinterpret_cast<uint4*>(dst)[c] =
              r >= 0 ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0, 0, 0, 0);
      } else {
        for (int c = lane; c < Dp; c += 32) dst[c] = r >= 0 && c < D ? src[c] : 0;
      }
    } else {
      const float* src = static_cast<const float*>(h) + r * ld;
      for (int c = lane; c < Dp; c += 32) {
        uint16_t w[3];
        split_planes(r >= 0 && c < D ? src[c] : 0.f, w);
#pragma unroll
        for (int k = 0; k < 3; ++k) dst[k * plane + c] = w[k];
      }
    }
  }
}

// Join the tiles' statistics: 32 rows per block, sixteen threads per row, each with four pairs in
// flight (one after the other, their latencies and exponentials made 30 us of 16384 rows x 394 pairs).
__device__ __forceinline__ void join2(float& m, float& sum, float2 v) {
  const float top = fmaxf(m, v.x);
  sum = sum * ex2_fast((m - top) * kLog2e) + v.y * ex2_fast((v.x - top) * kLog2e);
  m = top;
}
// The block that ends last makes the loss of the rows' losses, summed in a fixed order in fp64; without
// a reduction each goes to its row's place.
__global__ void __launch_bounds__(512) join_kernel(const float2* __restrict__ part, int slots, int64_t Tp,
                                                   const float* __restrict__ target_logit, Saved s, float* row_loss,
                                                   int reduction, float* __restrict__ loss) {
  __shared__ float2 sm[16][32];
  __shared__ double sums[16];
  __shared__ int last;
  pdl_wait_primary();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = s.count[0], blocks = n > 0 ? (n + 31) / 32 : 1;
  const int row = blockIdx.x * 32 + lane;
  if (blockIdx.x >= blocks) return;
  float m[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX}, sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (row < n) {
    int k = w;
    for (; k + 48 < slots; k += 64) {
      float2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = part[(int64_t)(k + 16 * i) * Tp + row];
#pragma unroll
      for (int i = 0; i < 4; ++i) join2(m[i], sum[i], v[i]);
    }
    for (; k < slots; k += 16) join2(m[0], sum[0], part[(int64_t)k * Tp + row]);
#pragma unroll
    for (int i = 1; i < 4; ++i) join2(m[0], sum[0], make_float2(m[i], sum[i]));
  }
  sm[w][lane] = make_float2(m[0], sum[0]);
  __syncthreads();
  if (w == 0 && row < n) {
#pragma unroll
    for (int k = 1; k < 16; ++k) join2(m[0], sum[0], sm[k][lane]);
    const bool ok = s.target[row] >= 0;
    // the maximum and the logarithm apart: their sum is rounded to 2^-24 of the maximum, which a sure token's loss
    // and the probabilities of large logits do not bear
    const float l2 = ok ? log2f(sum[0]) : __int_as_float(0x7fffffff);
    const float l = fmaf(l2, kLn2, ok ? m[0] - target_logit[row] : 0.f);
    s.stat[row] = make_float2(m[0], l2);
    if (reduction == 0) loss[s.row[row]] = l;
    else __stcg(row_loss + row, l);
    __threadfence();  // before this block counts as done
  }
  if (reduction == 0) return;
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(s.count + 1, 1) == blocks - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double x = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 512) x += (double)__ldcg(row_loss + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (lane == 0) sums[w] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    x = 0.0;
    for (int k = 0; k < 16; ++k) x += sums[k];
    *loss = (float)(reduction == 1 ? x / (double)n : x);
  }
}

// The kept rows' weights, and each block's largest finite magnitude of them.
constexpr int kRowwBlocks = 64;
__global__ void __launch_bounds__(256) roww_kernel(const float* __restrict__ dloss, Saved s, float* __restrict__ roww,
                                                   float* __restrict__ peaks) {
  __shared__ float sm[8];
  const int n = *s.count;
  float top = 0.f;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += kRowwBlocks * 256) {
    const float w = dloss[s.row[i]];
    roww[i] = w;
    if (isfinite(w)) top = fmaxf(top, fabsf(w));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int k = 1; k < 8; ++k) top = fmaxf(top, sm[k]);
  peaks[blockIdx.x] = top;
}

bool sizes_ok(const m3b_linear_xent_args* a) {
  return a && a->rows >= 0 && a->d_model > 0 && a->vocab > 0 &&
         (a->dtype == M3B_F32 || a->dtype == M3B_BF16 || a->dtype == M3B_F16);
}

int check(const m3b_linear_xent_args* a, bool bwd) {
  if (!a) return fail(M3B_ERR_INVALID_ARG, "linear_xent: null args");
  if (!sizes_ok(a)) return fail(M3B_ERR_INVALID_ARG, "linear_xent: bad sizes or dtype");
  if (a->rows > (int64_t(1) << 31) - 512 || a->d_model > (1 << 24) || a->vocab > (1 << 30))
    return fail(M3B_ERR_INVALID_ARG, "linear_xent: sizes past the kernels' limits");
  if (a->reduction < 0 || a->reduction > 2) return fail(M3B_ERR_INVALID_ARG, "linear_xent: reduction");
  if (!a->weight || !a->saved) return fail(M3B_ERR_INVALID_ARG, "linear_xent: null pointer");
  if (!aligned16(a->saved)) return fail(M3B_ERR_ALIGNMENT, "linear_xent: saved must be 16-byte aligned");
  if (bwd) {
    if (!a->dloss) return fail(M3B_ERR_INVALID_ARG, "linear_xent_bwd: null pointer");
  } else {
    if ((a->rows && (!a->hidden || !a->target)) || (!a->loss && (a->rows || a->reduction)))
      return fail(M3B_ERR_INVALID_ARG, "linear_xent_fwd: null pointer");
    if (a->rows && a->hidden_stride < a->d_model)
      return fail(M3B_ERR_INVALID_ARG, "linear_xent_fwd: row stride shorter than the rows");
  }
  return M3B_OK;
}

// The weight as an operand: in place, or packed (fp32, or rows that the TMA cannot read).
GemmOperand weight_of(const m3b_linear_xent_args* a, Carve& ws, bool run, cudaStream_t st, int* rc) {
  const Dims d(a);
  if (!d.f32 && tma_ok(a->weight, d.D)) return GemmOperand{a->weight, d.V, d.D, d.D, 0, 1};
  const int64_t plane = (int64_t)d.V * d.Dp;
  void* p = ws.take((size_t)d.np * plane * 2);
  if (run && *rc == M3B_OK) {
    PackList packs;
    packs.add(a->weight, d.V, d.D, d.D, p, d.Dp, plane);
    *rc = launch_pack(packs, a->dtype, st);
  }
  return GemmOperand{p, d.V, d.D, d.Dp, plane, d.np};
}

GemmOperand piece_of(const GemmOperand& w, int64_t c0, int64_t cols) {
  GemmOperand o = w;
  o.p = static_cast<const uint16_t*>(w.p) + c0 * w.ld;
  o.rows = cols;
  if (o.planes == 1) o.plane = 0;
  return o;
}

#define M3B_MAP(...) M3B_TRY(gemm_map(__VA_ARGS__))

// K blocks of the logits' sums of 16-bit operands (kGmSums), of equal length; 0: one sum.
int group_of(const Dims& d) {
  const int nk = (d.D + kGmBK - 1) / kGmBK, groups = d.f32 ? 1 : (nk + kGmSums - 1) / kGmSums;
  return groups > 1 ? (nk + groups - 1) / groups : 0;
}

int forward(const m3b_linear_xent_args* a, void* workspace, size_t* need, bool run, cudaStream_t st) {
  const Dims d(a);
  if (d.T <= kSmallXentRows) return small_xent_fwd(a, workspace, need, run, st);
  Carve ws(workspace);
  const bool pair = d.T > 128;
  const int bn = pair ? gemm_columns(d.T, d.V, d.f32) : d.f32 ? 64 : 128;
  const int nt = (d.V + bn - 1) / bn;
  float* target_logit = static_cast<float*>(ws.take((size_t)d.Tp * 4));
  float* row_loss = static_cast<float*>(ws.take((size_t)d.Tp * 4));
  float2* part = static_cast<float2*>(ws.take((size_t)nt * 2 * d.Tp * 8));
  const Saved s = saved_of(a, a->saved);
  int rc = M3B_OK;
  if (run) {
    keep_kernel<<<1, 1024, 0, st>>>(a->target, a->ignore_index, d.T, d.Tp, d.V, s, a->err);
    const int64_t blocks = d.Tp / 8, most = (int64_t)num_sms() * 8;
    const int vec = !d.f32 && d.D % 8 == 0 && a->hidden_stride % 8 == 0 && aligned16(a->hidden);
    M3B_TRY(check_launch("linear_xent keep"));
    M3B_TRY(launch_dependent(gather_kernel, dim3((unsigned)(blocks < most ? blocks : most)), 256, st, a->hidden,
                             (int)a->dtype, a->hidden_stride, d.D, d.Tp, d.Dp, vec, s));
  }
  const GemmOperand w = weight_of(a, ws, run, st, &rc);
  *need = ws.at;
  if (!run || rc != M3B_OK) return rc;
  GemmParams p{};
  GemmSub& g = p.sub[0];
  p.nsub = 1;
  p.bn = bn;
  p.npass = d.f32 ? 6 : 1;
  p.f16 = d.f16;
  p.dyn = s.count;
  p.err = a->err;
  const GemmOperand h{s.h, d.Tp, d.D, d.Dp, d.Tp * d.Dp, d.np};
  M3B_MAP(&g.a[0], h, false, 128, d.f16);
  M3B_MAP(&g.b[0], w, false, gemm_box_b(pair, bn, kEpiLse), d.f16);
  g.M = (int)d.T;
  g.m_dyn = 1;
  g.N = d.V;
  g.nk[0] = (d.D + kGmBK - 1) / kGmBK;
  p.group = group_of(d);
  p.target = s.target;
  p.target_logit = target_logit;
  p.part = part;
  p.part_ld = d.Tp;
  const int epi = p.group ? kEpiLseSums : kEpiLse;
  plan_gemm(p, epi, pair);
  M3B_TRY(launch_gemm(p, epi, pair, nullptr, st));
  if (a->reduction == 0 && cudaMemsetAsync(a->loss, 0, (size_t)d.T * 4, st) != cudaSuccess)
    return check_launch("linear_xent loss");
  return launch_dependent(join_kernel, dim3((unsigned)(d.Tp / 32)), 512, st, (const float2*)part, nt * 2, d.Tp,
                          (const float*)target_logit, s, row_loss, (int)a->reduction, a->loss);
}

// Columns of a piece of the vocabulary.
int64_t piece_cols(const Dims& d) {
  int64_t c = (int64_t)(kPieceBytes / ((size_t)d.np * 2 * d.Tp)) / 256 * 256;
  if (c < kPieceLeast) c = kPieceLeast;
  return c < d.V ? c : d.V;
}

int backward(const m3b_linear_xent_args* a, void* workspace, size_t* need, bool run, cudaStream_t st) {
  const Dims d(a);
  if (d.T <= kSmallXentRows) return small_xent_bwd(a, workspace, need, run, st);
  Carve ws(workspace);
  const int64_t cols = piece_cols(d), ldz = up(cols, 8);
  const int bn = d.f32 ? 128 : 256, pieces = (int)((d.V + cols - 1) / cols);
  int rc = M3B_OK;
  uint16_t* dz = static_cast<uint16_t*>(ws.take((size_t)d.np * d.Tp * ldz * 2));
  float* acc = nullptr;
  if (a->dhidden && pieces > 1) acc = static_cast<float*>(ws.take((size_t)d.Tp * up(d.D, bn) * 4));
  float *roww = nullptr, *peaks = nullptr, *peak = nullptr;
  if (a->reduction == 0) {
    roww = static_cast<float*>(ws.take((size_t)d.Tp * 4));
    peaks = static_cast<float*>(ws.take((kRowwBlocks + 1) * 4));
    peak = peaks ? peaks + kRowwBlocks : nullptr;
  }
  int* ticket = static_cast<int*>(ws.take(4));
  const GemmOperand w = weight_of(a, ws, run, st, &rc);
  const Saved s = saved_of(a, a->saved);
  const GemmOperand h{s.h, d.Tp, d.D, d.Dp, d.Tp * d.Dp, d.np};
  const size_t es = d.f32 ? 4 : 2;
  const int okind = d.f32 ? kOutF32 : d.f16 ? kOutF16 : kOutBf16;
  GemmParams base{};
  base.bn = bn;
  base.npass = d.f32 ? 6 : 1;
  base.f16 = d.f16;
  base.dyn = s.count;
  base.err = a->err;
  // fp16 has nothing between 0 and 6e-8, where most of a large vocabulary's probabilities may lie: they are
  // kept times 2^15 (at most 32768).  Weights per row, which may be a loss scaler's 65536 or one token's share of
  // a mean, are divided by the power of two at or below the largest of them (then below 2, so times 2^14), and
  // the two products multiply it back in fp32.
  const bool rowf16 = d.f16 && a->reduction == 0;
  base.shift = rowf16 ? 14.f : d.f16 ? 15.f : 0.f;

  // the two gradients' shares of the piece of n columns from c0 on, side by side
  auto gradients = [&](GemmParams& p, int64_t c0, int64_t n, const GemmOperand* z, const GemmOperand* wp) {
    auto sub = [&](void* out, int M, int K) -> GemmSub& {
      GemmSub& g = p.sub[p.nsub++];
      g.M = M;
      g.N = d.D;
      g.nk[0] = K;
      g.b_mn = 1;
      g.alpha = rowf16 ? 0x1p-14f : d.f16 ? 0x1p-15f : 1.f;
      if (a->reduction != 0) g.alpha_num = a->dloss;
      else if (d.f16) g.alpha_num = peak;
      if (a->reduction == 1) g.alpha_den = s.count;
      g.out.kind = okind;
      g.out.ld = d.D;
      g.out.p = out;
      g.out.vec = aligned16(out) && d.D % 8 == 0;
      return g;
    };
    if (a->dhidden) {
      GemmSub& g = sub(a->dhidden, (int)d.T, (int)((n + kGmBK - 1) / kGmBK));
      g.m_dyn = 1;
      g.row_index = s.row;
      g.acc = acc;
      g.acc_mode = !acc ? 0 : c0 == 0 ? 1 : c0 + cols < d.V ? 2 : 3;
      if (z) {
        M3B_TRY(gemm_map(&g.a[0], *z, false, 128, d.f16));
        M3B_TRY(gemm_map(&g.b[0], *wp, true, 0, d.f16));
      }
    }
    if (a->dweight) {
      GemmSub& g = sub(static_cast<uint8_t*>(a->dweight) + (size_t)c0 * d.D * es, (int)n, (int)(d.Tp / kGmBK));
      g.k_dyn = 1;
      g.a_mn = 1;
      if (z) {
        M3B_TRY(gemm_map(&g.a[0], *z, true, 0, d.f16));
        M3B_TRY(gemm_map(&g.b[0], h, true, 0, d.f16));
      }
    }
    return (int)M3B_OK;
  };
  size_t parts_bytes = 0;
  for (int64_t c0 = 0; c0 < d.V; c0 += cols) {  // the last piece is shorter: its plan may be another one
    GemmParams p = base;
    gradients(p, c0, d.V - c0 < cols ? d.V - c0 : cols, nullptr, nullptr);
    const size_t b = plan_gemm(p, kEpiAcc, true);
    if (b > parts_bytes) parts_bytes = b;
  }
  void* parts = ws.take(parts_bytes);
  *need = ws.at;
  if (!run || rc != M3B_OK) return rc;
  if (a->dhidden && cudaMemsetAsync(a->dhidden, 0, (size_t)d.T * d.D * es, st) != cudaSuccess)
    return check_launch("linear_xent_bwd");
  if (roww) {
    roww_kernel<<<kRowwBlocks, 256, 0, st>>>(a->dloss, s, roww, peaks);
    M3B_TRY(check_launch("linear_xent roww"));
  }
  for (int64_t c0 = 0; c0 < d.V; c0 += cols) {
    const int64_t n = d.V - c0 < cols ? d.V - c0 : cols;
    const GemmOperand wp = piece_of(w, c0, n);
    const GemmOperand z{dz, d.Tp, n, ldz, d.Tp * ldz, d.np};
    {  // softmax - onehot of the piece
      GemmParams p = base;
      GemmSub& g = p.sub[0];
      p.nsub = 1;
      p.bn = gemm_columns(d.T, n, d.f32);
      M3B_MAP(&g.a[0], h, false, 128, d.f16);
      M3B_MAP(&g.b[0], wp, false, gemm_box_b(true, p.bn, kEpiDlogit), d.f16);
      g.M = (int)d.T;
      g.m_dyn = 1;
      g.N = (int)n;
      g.nk[0] = (d.D + kGmBK - 1) / kGmBK;
      M3B_TRY(gemm_out_map(&p.o[0], z, d.f16));
      p.target = s.target;
      p.stat = s.stat;
      p.roww = roww;
      if (rowf16) {
        p.peaks = peaks;
        p.npeaks = kRowwBlocks;
        p.peak_out = peak;
      }
      p.col0 = (int)c0;
      p.clear = ticket;
      p.group = group_of(d);  // the logits of the forward pass: a sure token's gradient is their difference
      const int epi = p.group ? kEpiDlogitSums : kEpiDlogit;
      plan_gemm(p, epi, true);
      M3B_TRY(launch_gemm(p, epi, true, nullptr, st));
    }
    GemmParams p = base;
    M3B_TRY(gradients(p, c0, n, &z, &wp));
    plan_gemm(p, kEpiAcc, true);
    p.ticket = ticket;
    if (p.nsub) M3B_TRY(launch_gemm(p, kEpiAcc, true, parts, st));
  }
  return M3B_OK;
}

int check_workspace(size_t need, const void* ws, size_t bytes) {
  if (!ws || bytes < need) return fail(M3B_ERR_WORKSPACE, "linear_xent: workspace of %zu bytes, %zu needed", bytes, need);
  if (!aligned16(ws)) return fail(M3B_ERR_ALIGNMENT, "linear_xent: workspace must be 16-byte aligned");
  return M3B_OK;
}

// No rows: the sum is 0, the mean 0 / 0.
__global__ void empty_loss_kernel(float* loss, int reduction) {
  *loss = reduction == 1 ? __int_as_float(0x7fffffff) : 0.f;
}

}  // namespace

}  // namespace m3b

extern "C" {

size_t m3b_linear_xent_saved(const m3b_linear_xent_args* a) {
  if (!m3b::sizes_ok(a)) return 0;
  return a->rows <= m3b::kSmallXentRows ? m3b::small_xent_saved(a) : m3b::saved_of(a, nullptr).bytes;
}

size_t m3b_linear_xent_fwd_workspace(const m3b_linear_xent_args* a) {
  size_t need = 0;
  if (m3b::sizes_ok(a) && a->rows) m3b::forward(a, nullptr, &need, false, nullptr);
  return need;
}

int m3b_linear_xent_fwd(const m3b_linear_xent_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  m3b::clear_error();
  int rc = m3b::check(a, false);
  if (rc != M3B_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->rows == 0) {
    if (a->reduction == 0) return M3B_OK;
    m3b::empty_loss_kernel<<<1, 1, 0, st>>>(a->loss, a->reduction);
    return m3b::check_launch("linear_xent_fwd");
  }
  size_t need = 0;
  m3b::forward(a, nullptr, &need, false, nullptr);
  rc = m3b::check_workspace(need, workspace, workspace_bytes);
  return rc != M3B_OK ? rc : m3b::forward(a, workspace, &need, true, st);
}

size_t m3b_linear_xent_bwd_workspace(const m3b_linear_xent_args* a) {
  size_t need = 0;
  if (m3b::sizes_ok(a) && a->rows) m3b::backward(a, nullptr, &need, false, nullptr);
  return need;
}

int m3b_linear_xent_bwd(const m3b_linear_xent_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  m3b::clear_error();
  int rc = m3b::check(a, true);
  if (rc != M3B_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->rows == 0) {
    const size_t es = a->dtype == M3B_F32 ? 4 : 2;
    if (a->dweight && cudaMemsetAsync(a->dweight, 0, (size_t)a->vocab * a->d_model * es, st) != cudaSuccess)
      return m3b::check_launch("linear_xent_bwd");
    return M3B_OK;
  }
  size_t need = 0;
  m3b::backward(a, nullptr, &need, false, nullptr);
  rc = m3b::check_workspace(need, workspace, workspace_bytes);
  return rc != M3B_OK ? rc : m3b::backward(a, workspace, &need, true, st);
}

}  // extern "C"
