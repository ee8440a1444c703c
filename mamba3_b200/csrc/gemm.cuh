// Persistent tcgen05 matrix-product kernel with operator epilogues (sm_100a), shared by the
// training and serving operators (ffn.cu, xent.cu).
//
//   C (M x N) = sum over segments of A_s (M x K_s) B_s (N x K_s)^T, fp32 accumulate in TMEM
//
// * Operands are 16-bit tiles of 64 K values moved by TMA with the 128-byte swizzle.  Either
//   operand may be stored with K along its rows (K-major) or across them (MN-major, for the
//   products of the backward passes); the tile then arrives as 64 x 64 boxes and the UMMA
//   descriptor reads it transposed.
// * fp32 operands travel as three bf16 planes whose sum is the value exactly (each plane is what the
//   planes before it leave, rounded to nearest: at most 2^-8 and 2^-17 of the value, of either sign).  The
//   product runs over six plane pairs, smallest first; each of the two largest that are left out is
//   at most 2^-25 of the product.  (Planes cut off instead of rounded leave out up to 2^-21, always of the
//   product's sign.)  The
//   tensor core cuts its sums off instead of rounding them, a bias of half a step per addition that
//   fp32 results would show (3e-6 of a 323 x 897 product): so every kGmGroup K blocks are a sum of
//   their own, and the epilogue adds them, rounded, in registers (7e-7).  The loss's logits of 16-bit operands
//   are sums of groups too (kGmSums).
// * A launch holds up to four products ("subs"), so that products that are too small to fill the
//   GPU run side by side, and a product has up to two K segments with operands of their own.
// * Row or K counts may come from device memory (`dyn`): the loss drops ignored tokens without
//   the host knowing how many remain.
//
// Three roles per CTA: warp 0 the TMA producer, warp 1 the MMA issuer, warps 2-9 the epilogue (two
// warps per 32 TMEM lanes, half of the columns each).  Two TMEM accumulators of 256 columns let a
// tile's epilogue run under the next tile's MMAs.  Jobs of one length are dealt in turn; jobs of
// several lengths (several products, or one whose long K is split) are listed longest first and drawn
// from a counter in device memory by whoever is nearly free (the first CTA's producer, a dozen K blocks
// before it has none left; it passes the job on to the other roles through a small queue), which leaves
// idle at most the last job's length.
// A split product's parts go to the workspace in fp32 and a join kernel adds them in order, so the
// result does not depend on who took which job.  PAIR: a cluster of two CTAs computes 256 x bn
// tiles with cta_group::2, each CTA staging half of the B rows; otherwise single CTAs compute
// 128 x bn tiles.
//
// Bound by the tensor pipe where K is long: 16384 x 2048 x 8192 bf16 in 1.46 - 1.50 PFLOP/s (a library product
// of that size 1.51 - 1.55).  With K short the epilogue's stores show: the pipe is 66 - 92 % active at K = 768.
#pragma once

#include <float.h>

#include "launch.h"
#include "pair.cuh"
#include "tmap.h"

namespace m3b {

constexpr int kGmThreads = 320;
constexpr int kGmSubs = 4;      // products of a launch at most
constexpr int kGmQueue = 4;     // drawn jobs that the producer may be ahead of the epilogue
constexpr int kGmBK = 64;
constexpr int kGmGroup = 4;     // K blocks of fp32 operands summed in one accumulator
// K blocks of 16-bit operands summed in one accumulator where the result is the loss.  The tensor core's cut-off
// sums make a loss too small, by 5.5e-7 of it at K = 1024, 1.06e-6 at 2048 and 2.3e-6 at 4096 (fp16; a library
// product's fp32 logits likewise); in sums of 16 blocks by 5.0e-7 at 2048 and 5.9e-7 at 4096.  16384 x 2048 x
// 50257 bf16, forward and backward, takes 10.5 ms with either.  (Sums of 8 blocks: 2.9e-7 at 2048; of 4: 1.5e-7, and
// the forward pass 2.58 ms for 2.41.)  K up to 16 blocks is one sum: the registers between cost K = 128 a tenth.
constexpr int kGmSums = 16;
constexpr uint32_t kGmStageA = 128 * kGmBK * 2;     // 16 KB
constexpr uint32_t kGmStage = 2 * kGmStageA;        // + B: at most 128 rows of 64
constexpr uint32_t kGmBox = 32 * 128;               // staging of an epilogue warp: 32 rows x 32 fp32
constexpr int kGuSlots = 4;                         // kEpiDglu: runs of 8 columns of g and u per epilogue warp
// What the forward pass keeps of g and u, in runs of 32 rows x 8 columns: in fp32, [g, u][column / 4][row][4],
// or, where 16-bit operands follow, their upper 24 bits: the upper halves of g and u beside each other,
// [column / 4][row][4], then the next 8 bits of both, [row][column][g, u].  (A 16-bit copy's rounding would
// reach every gradient; the last 8 bits of fp32 do not, and a quarter of the bytes is theirs.)
template <bool PLANES>
constexpr uint32_t kGuRun = PLANES ? 2048 : 1536;
constexpr uint32_t kGmBarOff = 6 * kGmStage + 8 * kGmBox;
constexpr uint32_t kGmSmem = kGmBarOff + 768 + 1024;  // barriers, job queue, TMEM slot; alignment
static_assert(kGmSmem <= 227 * 1024, "shared memory plan");

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// How a product's result is stored.
enum GemmOutKind { kOutBf16 = 0, kOutF16 = 1, kOutF32 = 2 };

struct GemmOut {
  void* p;
  int64_t ld;     // elements between rows
  int kind;
  int vec;        // rows and columns allow 16-byte stores
};

// (Forms of their own rather than flags: a spilled register costs an L2 round trip here, because the
// stage ring leaves the L1 cache almost nothing.)
enum GemmEpi {
  kEpiStore = 0,   // out = alpha acc
  kEpiFinal = 1,   // out = residual + alpha (acc + bias)
  kEpiAcc = 2,     // out row_index[r] = alpha (sum of several launches' accumulators)
  kEpiGlu = 3,     // gate | up accumulators -> silu(g) u, and g, u kept in fp32 for the backward pass
  kEpiDglu = 4,    // d(silu(g) u) -> dg, du
  kEpiLse = 5,     // running maximum and sum of each row, and the target's logit
  kEpiDlogit = 6,  // softmax - one-hot
  kEpiLseSums = 7,     // kEpiLse and kEpiDlogit of 16-bit operands and more than kGmSums K blocks, in sums of at
  kEpiDlogitSums = 8,  // most that many
  kEpiDgluSums = 9,    // kEpiDglu of 16-bit operands, with the column sums of dg and du before they are rounded
};
constexpr int kEpiCount = 10;

struct GemmSub {
  CUtensorMap a[2], b[2];
  int M, N;        // result rows and columns
  int nk[2];       // K blocks of each segment
  int mt, nt;      // tiles
  int a_mn, b_mn;  // operand stored MN-major
  int m_dyn, k_dyn;
  int split;       // jobs along K of each tile
  float* part;     // [split][row / 32][col / 4][row % 32][4] fp32 when split > 1
  GemmOut out;     // final results (kEpiStore, kEpiFinal, kEpiAcc)
  // kEpiStore, kEpiFinal, kEpiAcc
  float alpha;
  const float* alpha_num;  // alpha *= alpha_num[0]
  const int* alpha_den;    // alpha /= alpha_den[0] (0 rows: alpha = 0)
  const void* bias;        // N values, of `dt`
  const void* bias2;       // kEpiGlu: the up bias
  const void* residual;    // (M, N) of `dt`, rows ld_res apart
  int64_t ld_res;
  const int* row_index;    // result row r goes to row row_index[r] (negative: nowhere)
  float* acc;              // running fp32 sum, [row / 32][col / 4][row % 32][4]
  int acc_mode;            // 0 none, 1 acc = v, 2 acc += v, 3 out = acc + v
  int dt, res_vec;         // dtype code of bias and residual; the residual's rows allow vector loads
};

struct GemmParams {
  GemmSub sub[kGmSubs];
  CUtensorMap o[2];  // kEpiGlu, kEpiDglu, kEpiDlogit: the first product's results (out, out2), 32 x 32 boxes
  int nsub;
  int bn;       // accumulator columns of a tile
  int npass;    // plane pairs: 1, or 6 for fp32 operands
  int group;    // kEpiLseSums, kEpiDlogitSums: K blocks of a sum
  int f16;      // operand type: fp16 instead of bf16
  const int* dyn;
  int* ticket;  // zeroed counter that jobs are drawn from, or null: dealt in turn
  int* clear;   // a counter to zero for the launch that follows
  // kEpiGlu / kEpiDglu: g and u in runs (kGuRun), gu_ld of them (whole 32 columns) for every 32 rows
  uint8_t* gu;
  int64_t gu_ld;
  float *sum_g, *sum_u;  // kEpiDgluSums: [row / 32][column of sub[0].N], sums over 32 rows
  // kEpiLse, kEpiLseSums, kEpiDlogit
  const int* target;       // per row
  float* target_logit;
  float2* part;            // (slots, rows): maximum, and sum of exp(logit - maximum)
  int64_t part_ld;
  const float2* stat;      // per row: maximum, and log2 of the sum of exp(logit - maximum)
  const float* roww;       // weight per row or null
  float shift;             // softmax - one-hot times 2^shift
  // fp16: a power of two that brings values into its range (peak_scale), from the largest magnitude of each
  // of npeaks blocks, or null; *peak_out: that power, for the products that read the scaled values
  const float* peaks;
  int npeaks;
  float* peak_out;
  int col0;                // first vocabulary column of this piece
  int* err;
  uint64_t wait_ns;
};

static_assert(sizeof(GemmParams) <= 4096, "kernel parameters");

// ---------------------------------------------------------------------------
// jobs
// ---------------------------------------------------------------------------
struct GemmJob {
  int sub, mt, nt;
  int ks;      // part of K
  int kb, ke;  // iterations [kb, ke) of the tile's K blocks times passes
};

template <bool PAIR>
struct GemmSched {
  const GemmParams& p;
  int dyn;
  static constexpr int kTileM = PAIR ? 256 : 128;
  __device__ explicit GemmSched(const GemmParams& q) : p(q), dyn(q.dyn ? *q.dyn : 0) {}
  __device__ int mtiles(const GemmSub& s) const { return s.m_dyn ? (dyn + kTileM - 1) / kTileM : s.mt; }
  __device__ int rows(const GemmSub& s) const { return s.m_dyn ? dyn : s.M; }
  __device__ int nk0(const GemmSub& s) const { return s.k_dyn ? (dyn + kGmBK - 1) / kGmBK : s.nk[0]; }
  __device__ int jobs() const {
    int n = 0;
    for (int i = 0; i < p.nsub; ++i) n += mtiles(p.sub[i]) * p.sub[i].nt * p.sub[i].split;
    return n;
  }
  __device__ GemmJob job(int t) const {
    GemmJob o{};
    for (int i = 0; i < p.nsub; ++i) {
      const GemmSub& s = p.sub[i];
      const int mt = mtiles(s), tiles = mt * s.nt, n = tiles * s.split;
      if (t >= n) {
        t -= n;
        continue;
      }
      // the tiles of one part of K together: what is in flight then shares operands in L2
      if (s.split > 1) {
        o.ks = t / tiles;
        t -= o.ks * tiles;
      }
      // bands of 8 row tiles, walked column by column, for the same reason
      const int band = 8 * s.nt;
      const int g = t / band, first = g * 8, size = mt - first < 8 ? mt - first : 8, r = t - g * band;
      o.sub = i;
      o.mt = first + r % size;
      o.nt = r / size;
      const int all = (nk0(s) + s.nk[1]) * p.npass;
      o.ke = all;
      if (s.split > 1) {
        const int len = (all + s.split - 1) / s.split;
        o.kb = o.ks * len < all ? o.ks * len : all;
        o.ke = o.kb + len < all ? o.kb + len : all;
      }
      break;
    }
    return o;
  }
};

// ---------------------------------------------------------------------------
// element helpers
// ---------------------------------------------------------------------------

// The next bf16 plane of an fp32 value: v keeps what is left.  Infinity and NaN lie in the last plane, which
// meets only the other operand's first, beside a first plane of +-1: so their products are those of the
// value itself (in the first plane they would meet the zeros of the other's second and third).
__device__ __forceinline__ uint32_t next_plane(float& v, int plane) {
  const uint32_t b = __float_as_uint(v);
  const bool fin = (b & 0x7f800000u) != 0x7f800000u;
  uint32_t r = (b + 0x7fffu + (b >> 16 & 1u)) & 0xffff0000u;
  if ((r & 0x7f800000u) == 0x7f800000u) r = b & 0xffff0000u;  // would round to infinity: cut off
  const uint32_t last = v != v ? 0x7fffu : b >> 16;           // a NaN whose set bits are all below stays one
  const uint32_t odd = plane == 2 ? last : plane == 1 ? 0u : (b >> 16 & 0x8000u) | 0x3f80u;
  if (fin) v -= __uint_as_float(r);
  return fin ? r >> 16 : odd;
}
__device__ __forceinline__ void split_planes(float v, uint16_t (&w)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) w[k] = (uint16_t)next_plane(v, k);
}

__device__ __forceinline__ uint32_t pack16(float a, float b, bool f16) {
  if (f16) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  return pack_bf16x2(a, b);
}

// 1 / (1 + exp(-g)) of a pair: packed arithmetic and the hardware's 2^x and reciprocal (2 and 1 steps);
// 0 where exp(-g) overflows.
__device__ __forceinline__ float2 sigmoid2(float2 g) {
  const float2 t = mul2(g, make_float2(-kLog2e, -kLog2e));
  const float2 y = fma2(make_float2(ex2_fast(t.x), ex2_fast(t.y)), make_float2(1.f, 1.f), make_float2(1.f, 1.f));
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(y.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(y.y));
  return r;
}

// Results leave through a staging box per epilogue warp: a thread owns one row of the accumulator,
// but a warp's stores should cover whole 32-byte sectors of few rows.  Each thread writes its 32
// columns into the box (16-byte chunks swizzled by the row, so neither side has bank conflicts) and
// the warp reads the box back row by row.
struct GemmRows {
  int64_t row0;          // first of the warp's 32 rows
  int M;                 // rows of the result
  const int* row_index;  // or null
  __device__ __forceinline__ int64_t out_row(int r) const {
    const int64_t row = row0 + r;
    if (row >= M) return -1;
    return row_index ? (int64_t)row_index[row] : row;
  }
};

// 32 columns from `col` on of 16-bit values, packed in pairs.
__device__ __forceinline__ void put16(uint8_t* box, const GemmOut& o, uint16_t* base, const GemmRows& rows, int col, int N,
                                      const uint32_t (&w)[16]) {
  const int lane = threadIdx.x & 31;
  __syncwarp();  // the box has been read
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *reinterpret_cast<uint4*>(box + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  __syncwarp();
  const int k = lane & 3, c = col + 8 * k;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int r = it * 8 + (lane >> 2);
    const uint8_t* src = box + r * 64 + ((k ^ ((r >> 1) & 3)) << 4);
    const int64_t orow = rows.out_row(r);
    if (orow < 0 || c >= N) continue;
    uint16_t* q = base + orow * o.ld + c;
    if (o.vec && c + 8 <= N) {
      *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(src);
    } else {
#pragma unroll 1
      for (int e = 0; e < 8 && c + e < N; ++e) q[e] = reinterpret_cast<const uint16_t*>(src)[e];
    }
  }
}

// 32 columns of fp32 results.
__device__ __forceinline__ void put32(uint8_t* box, const GemmOut& o, const GemmRows& rows, int col, int N,
                                      const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int k = 0; k < 8; ++k)
    *reinterpret_cast<float4*>(box + lane * 128 + ((k ^ (lane & 7)) << 4)) =
        make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
  __syncwarp();
  const int k = lane & 7, c = col + 4 * k;
#pragma unroll 4
  for (int it = 0; it < 8; ++it) {
    const int r = it * 4 + (lane >> 3);
    const uint8_t* src = box + r * 128 + ((k ^ (r & 7)) << 4);
    const int64_t orow = rows.out_row(r);
    if (orow < 0 || c >= N) continue;
    float* q = static_cast<float*>(o.p) + orow * o.ld + c;
    if (o.vec && c + 4 <= N) {
      *reinterpret_cast<float4*>(q) = *reinterpret_cast<const float4*>(src);
    } else {
#pragma unroll 1
      for (int e = 0; e < 4 && c + e < N; ++e) q[e] = reinterpret_cast<const float*>(src)[e];
    }
  }
}

// A following product's operand leaves by TMA instead: the warp fills one of its two boxes (the same
// swizzle is the tensor map's 64-byte one) and one thread sends it, while the warp goes on.  (Stored row by
// row, dg and du cost the warp 24 us of 104 at 16384 x 768 x 2112.)
struct GemmSend {
  uint8_t* box;
  uint32_t side;
  __device__ __forceinline__ void operator()(const CUtensorMap* map, int col, int64_t row, int plane,
                                             const uint32_t (&w)[16]) {
    const int lane = threadIdx.x & 31;
    uint8_t* b = box + side * (kGmBox / 2);
    side ^= 1;
    if (lane == 0) bulk_wait_group_read<1>();  // the box sent before last has been read
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 4; ++k)
      *reinterpret_cast<uint4*>(b + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) =
          make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(col),
                   "r"((int)row), "r"(plane), "r"(smem_u32(b))
                   : "memory");
      bulk_commit_group();
    }
  }
};

// 32 columns of a following product's operand: a 16-bit type, or the planes of fp32 values.
template <bool PLANES>
__device__ __forceinline__ void put_operand(GemmSend& send, const CUtensorMap* map, bool f16, int col, int64_t row,
                                            float (&v)[32]) {
  if constexpr (!PLANES) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pack16(v[2 * i], v[2 * i + 1], f16);
    send(map, col, row, 0, w);
  } else {
#pragma unroll 1
    for (int pl = 0; pl < 3; ++pl) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const uint32_t top = next_plane(v[i], pl);
        if (i & 1) w[i >> 1] |= top << 16;
        else w[i >> 1] = top;
      }
      send(map, col, row, pl, w);
    }
  }
}
// 32 columns of a 16-bit final result.
__device__ __forceinline__ void put_narrow(uint8_t* box, const GemmOut& o, const GemmRows& rows, int col, int N,
                                           const float (&v)[32]) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack16(v[2 * i], v[2 * i + 1], o.kind == kOutF16);
  put16(box, o, static_cast<uint16_t*>(o.p), rows, col, N, w);
}

// 32 columns as final results, (v + bias) alpha + residual, fp32 until the one rounding.
struct GemmFinal {
  float alpha;
  const void *bias, *residual;
  int64_t ld_res;
  int dt, res_vec;
};
__device__ __forceinline__ float4 final4(const GemmOut& o, const GemmFinal& f, float4 b, float4 t, float4 r) {
  return make_float4(fmaf(t.x + b.x, f.alpha, r.x), fmaf(t.y + b.y, f.alpha, r.y), fmaf(t.z + b.z, f.alpha, r.z),
                     fmaf(t.w + b.w, f.alpha, r.w));
}
__device__ __forceinline__ float4 bias4(const void* bias, int dt, int c, int N) {
  float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
  if (bias) {
    if (c < N) b.x = ldf(bias, c, dt);
    if (c + 1 < N) b.y = ldf(bias, c + 1, dt);
    if (c + 2 < N) b.z = ldf(bias, c + 2, dt);
    if (c + 3 < N) b.w = ldf(bias, c + 3, dt);
  }
  return b;
}
// Four residual values of 16 bits, as they lie in memory.
__device__ __forceinline__ float4 wide4(uint2 r, int dt) {
  float2 p, q;
  if (dt == M3B_BF16) {
    p = bf2_to_f2(r.x), q = bf2_to_f2(r.y);
  } else {
    p = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
    q = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
  }
  return make_float4(p.x, p.y, q.x, q.y);
}
__device__ __forceinline__ void put_final(uint8_t* box, const GemmOut& o, const GemmFinal& f, const GemmRows& rows, int col,
                                          int N, const float (&v)[32]) {
  const int lane = threadIdx.x & 31, k = lane & 7, c = col + 4 * k;
  const bool whole = o.vec && c + 4 <= N && o.kind != kOutF32 && (!f.residual || f.res_vec);
  const int64_t first = rows.row0 + (lane >> 3);
  const int live = rows.M - first > 32 ? 8 : rows.M <= first ? 0 : (int)((rows.M - first + 3) / 4);  // of this lane's rows
  // the residual's loads of all rows are in flight while the box fills: one by one between the stores
  // each cost its whole latency
  uint2 raw[8];
  {
    const uint16_t* rp = static_cast<const uint16_t*>(f.residual) + first * f.ld_res + c;
#pragma unroll
    for (int it = 0; it < 8; ++it, rp += 4 * f.ld_res)
      raw[it] = whole && f.residual && it < live ? __ldg(reinterpret_cast<const uint2*>(rp)) : make_uint2(0u, 0u);
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<float4*>(box + lane * 128 + ((i ^ (lane & 7)) << 4)) =
        make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  __syncwarp();
  if (c >= N) return;
  if (whole) {
    const float4 b = bias4(f.bias, f.dt, c, N);
    uint16_t* op = static_cast<uint16_t*>(o.p) + first * o.ld + c;
#pragma unroll
    for (int it = 0; it < 8; ++it, op += 4 * o.ld) {
      const int r = it * 4 + (lane >> 3);
      const float4 x = final4(o, f, b, *reinterpret_cast<const float4*>(box + r * 128 + ((k ^ (r & 7)) << 4)), wide4(raw[it], f.dt));
      if (it < live)
        *reinterpret_cast<uint2*>(op) = make_uint2(pack16(x.x, x.y, o.kind == kOutF16), pack16(x.z, x.w, o.kind == kOutF16));
    }
    return;
  }
#pragma unroll 1
  for (int it = 0; it < live; ++it) {
    const int r = it * 4 + (lane >> 3);
    const int64_t row = rows.row0 + r;
    const float* src = reinterpret_cast<const float*>(box + r * 128 + ((k ^ (r & 7)) << 4));
#pragma unroll 1
    for (int e = 0; e < 4 && c + e < N; ++e) {
      float x = src[e];
      if (f.bias) x += ldf(f.bias, c + e, f.dt);
      x *= f.alpha;
      if (f.residual) x += ldf(f.residual, row * f.ld_res + c + e, f.dt);
      stf(o.p, row * o.ld + c + e, o.kind == kOutF32 ? M3B_F32 : o.kind == kOutF16 ? M3B_F16 : M3B_BF16, x);
    }
  }
}

// The power of two at or below the largest of n magnitudes, for whole warps; 2^-100 .. 2^100, so that it and
// its reciprocal are normal (all zero: 2^-100, which scales zeros).
__device__ __forceinline__ float peak_scale(const float* peaks, int n) {
  float x = 0.f;
  for (int i = threadIdx.x & 31; i < n; i += 32) x = fmaxf(x, peaks[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  x = fminf(fmaxf(x, 0x1p-100f), 0x1p100f);
  return __uint_as_float(__float_as_uint(x) & 0x7f800000u);
}

// Waits of all roles: the plain test in a loop (the sleeping form of mbar_wait may wake late for a
// stage that lasts a third of a microsecond); the clock is read only rarely.
__device__ __forceinline__ bool gm_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t = globaltimer_ns();
    if (t0 == 0) t0 = t;
    else if (t - t0 > limit_ns) return false;
  }
}
// Arrive on the first CTA's barrier from either CTA.  What it signals is that reads have ended (their
// values are in registers), so it orders no memory across the cluster: with .release.cluster it waited
// for the warp's outstanding stores.
template <bool PAIR>
__device__ __forceinline__ void gm_arrive_first(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mapa_shared(smem_u32(bar), 0)) : "memory");
  else
    mbar_arrive(bar);
}

// One thread of the (converged) warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// TMA load of one box to shared address `dst`, completing on the barrier at shared::cluster address `bar`.
template <bool PAIR>
__device__ __forceinline__ void gm_load(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
        "%4}], [%5];" ::"r"(dst),
        "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
// Arrive on the barrier, paired: on both CTAs', when the MMAs issued so far have completed.
template <bool PAIR>
__device__ __forceinline__ void gm_commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    umma_commit(bar);
}
__device__ __forceinline__ uint64_t gm_desc(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}

// ---------------------------------------------------------------------------
// the kernel
// ---------------------------------------------------------------------------
template <int EPI, bool PAIR, bool PLANES>
__global__ void __launch_bounds__(kGmThreads, 1) gemm_kernel(const __grid_constant__ GemmParams p) {
  constexpr int kTileM = PAIR ? 256 : 128;
  // six stages; kEpiDglu gives two of them to the runs of g and u
  constexpr bool kDglu = EPI == kEpiDglu || EPI == kEpiDgluSums;
  constexpr int kGmStages = kDglu ? 4 : 6;
  constexpr uint32_t kGmBoxOff = kGmStages * kGmStage, kGuOff = kGmBoxOff + 8 * kGmBox;
  static_assert(kGuOff + (kDglu ? 8 * kGuSlots * kGuRun<PLANES> : 0) <= kGmBarOff, "shared memory plan");
  constexpr bool kSums = EPI == kEpiLseSums || EPI == kEpiDlogitSums;
  constexpr bool GROUPS = PLANES || kSums;  // sums of groups of K blocks, added in registers
  constexpr int kPart = kSums ? 4 : 2;
  constexpr bool kDraws = EPI == kEpiStore || EPI == kEpiAcc;  // forms with several products a launch
  extern __shared__ uint8_t smraw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smraw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + kGmBarOff);
  uint64_t* full = bars;                  // [kGmStages]: the stage's copies landed
  uint64_t* empty = bars + kGmStages;     // [kGmStages]: the MMAs reading the stage completed
  uint64_t* accf = bars + 2 * kGmStages;  // [2]: accumulator finished
  uint64_t* acce = accf + 2;              // [2]: accumulator read
  uint64_t* jfull = acce + 2;             // [kGmQueue]: a job number is in jq
  uint64_t* jempty = jfull + kGmQueue;    // [kGmQueue]: every role of the cluster has read it (first CTA)
  uint64_t* gufull = jempty + kGmQueue;   // [8][kGuSlots]: the run landed (kEpiDglu)
  int4* jq = reinterpret_cast<int4*>(gufull + 8 * kGuSlots);  // [kGmQueue][2]: the jobs, ready to use
  uint32_t* tslot = reinterpret_cast<uint32_t*>(jq + 2 * kGmQueue);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kGmStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accf[i], 1);
      mbar_init(&acce[i], PAIR ? 16 : 8);  // one arrival per epilogue warp (of both CTAs)
    }
    for (int i = 0; i < 8 * kGuSlots; ++i) mbar_init(&gufull[i], 1);
    for (int i = 0; i < kGmQueue; ++i) {
      mbar_init(&jfull[i], 1);
      mbar_init(&jempty[i], PAIR ? 18 : 9);  // issuer, second producer, epilogue warps
    }
    fence_mbar_init();
  }
  if (warp == 0) pair_tmem_alloc<PAIR>(tslot, 512);
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // both CTAs' barriers are initialised before any remote use
  tc_fence_after();
  // so far nothing was read that another kernel writes: launched as a programmatic dependent, this part
  // ran under the end of the kernel before
  pdl_wait_primary();
  pdl_launch_dependents();
  if (p.clear && blockIdx.x == 0 && threadIdx.x == 0) *p.clear = 0;
  const uint32_t tbase = *tslot;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;
  const int worker = PAIR ? blockIdx.x / 2 : blockIdx.x, nworkers = PAIR ? gridDim.x / 2 : gridDim.x;
  const int bn = p.bn;
  const int brows = PAIR ? bn / 2 : bn;  // B rows staged by this CTA
  const GemmSched<PAIR> sched(p);
  auto give_up = [&]() { record_error(p.err, M3B_ERR_TIMEOUT); };
  // The n-th job, for a whole warp; sub < 0 when there is none left (-1) or the wait ran out (-2).  Jobs
  // that are dealt in turn, and every worker's first, each role works out for itself; drawn ones come
  // through the queue.
  const int total = sched.jobs();
  auto job_of = [&](int t) {
    GemmJob o{};
    o.sub = -1;
    if (t < total) o = sched.job(t);
    return o;
  };
  auto next_job = [&](uint32_t n) {
    if (n == 0 || !kDraws || !p.ticket) return job_of(worker + (int)n * nworkers);
    const uint32_t slot = (n - 1) % kGmQueue;
    GemmJob o{};
    o.sub = -2;
    if (!__all_sync(0xffffffffu, gm_wait(&jfull[slot], ((n - 1) / kGmQueue) & 1, p.wait_ns))) return o;
    const int4 x = jq[2 * slot], y = jq[2 * slot + 1];
    // reductions, so that the compiler knows the fields to be the same in all lanes and keeps the loops'
    // addresses in uniform registers
    auto uni = [](int v) { return (int)__reduce_or_sync(0xffffffffu, (unsigned)v); };
    o.sub = uni(x.x), o.mt = uni(x.y), o.nt = uni(x.z), o.ks = uni(x.w), o.kb = uni(y.x), o.ke = uni(y.y);
    if (lane == 0) gm_arrive_first<PAIR>(&jempty[slot]);
    return o;
  };
  auto group_end = [&](const GemmJob& j, int i) {
    const int n = PLANES ? 6 * kGmGroup : p.group, e = (i / n + 1) * n;
    return e < j.ke ? e : j.ke;
  };
  // The first CTA's producer, one thread: job n into both CTAs' queues.
  auto pass_on = [&](uint32_t n, const GemmJob& j) {
    const uint32_t slot = (n - 1) % kGmQueue;
    if (!gm_wait(&jempty[slot], (((n - 1) / kGmQueue) & 1) ^ 1, p.wait_ns)) return false;
    jq[2 * slot] = make_int4(j.sub, j.mt, j.nt, j.ks);
    jq[2 * slot + 1] = make_int4(j.kb, j.ke, 0, 0);
    mbar_arrive(&jfull[slot]);
    if constexpr (PAIR) {
      // the second CTA's copy completes on its own barrier
      const uint32_t fb = mapa_shared(smem_u32(&jfull[slot]), 1), q0 = mapa_shared(smem_u32(&jq[2 * slot]), 1);
      asm volatile("mbarrier.arrive.expect_tx.release.cluster.shared::cluster.b64 _, [%0], 24;" ::"r"(fb) : "memory");
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(q0),
                   "r"(j.sub), "r"(j.mt), "r"(j.nt), "r"(j.ks), "r"(fb)
                   : "memory");
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(q0 + 16),
                   "r"(j.kb), "r"(j.ke), "r"(fb)
                   : "memory");
    }
    return true;
  };
  // The producer's and the issuer's loops run warp-uniform, with one elected thread for the copies,
  // the MMAs and the commits: their addresses and descriptors then live in uniform registers.  As
  // single-thread loops they took 360 ns a stage whatever the stage held (MMAs: 305 ns).
  if (warp == 0) {
    const bool leader = elect_one();
    const uint32_t bytes = (PAIR ? 2u : 1u) * (kGmStageA + (uint32_t)brows * 128u);
    const uint32_t ring = smem_u32(sm);
    // the copies of both CTAs complete on the first CTA's barriers
    const uint32_t full0 = PAIR ? mapa_shared(smem_u32(full), 0) : smem_u32(full);
    uint32_t st = 0, ph = 1, it = 0, jn = 1;
    bool ok = true;
    const bool draws = kDraws && p.ticket && rank == 0;
    const int lead = __ffs(__ballot_sync(0xffffffffu, leader)) - 1;
    GemmJob job = next_job(0);
    for (; ok && job.sub >= 0; ++jn) {
      const int draw_at = job.ke - 12 > job.kb ? job.ke - 12 : job.kb;
      int drawn = 0;
      if (draws && job.ke == job.kb && leader) drawn = atomicAdd(p.ticket, 1);
      const GemmSub& s = p.sub[job.sub];
      const int nk0 = sched.nk0(s), nks = nk0 + s.nk[1];
      const int arow = job.mt * kTileM + (int)rank * 128;
      // B rows of this CTA; the gated product stages bn / 2 gate and bn / 2 up rows (paired: the
      // first CTA holds the gate's, the second the up's)
      const int brow = EPI == kEpiGlu ? job.nt * (bn / 2) : job.nt * bn + (int)rank * brows;
      // K block r; with planes, the pairs of a group of blocks from g0 on one after the other
      int r = job.kb, pass = 5, g0 = 0, gn = 1;
      if constexpr (PLANES) {
        if (job.kb < job.ke) {
          const int g = job.kb / (6 * kGmGroup), in = job.kb - g * 6 * kGmGroup;
          g0 = g * kGmGroup;
          gn = nks - g0 < kGmGroup ? nks - g0 : kGmGroup;
          pass = in / gn;
          r = g0 + in - pass * gn;
        }
      }
      for (int i = job.kb; i < job.ke; ++i, ++it) {
        ok = __all_sync(0xffffffffu, gm_wait(&empty[st], ph, p.wait_ns));
        if (!ok) break;
        const int seg = r >= nk0 ? 1 : 0, k = (seg ? r - nk0 : r) * kGmBK;
        // plane pairs, smallest first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
        const int pa = PLANES ? (0x001102 >> (4 * pass)) & 3 : 0, pb = PLANES ? (0x010120 >> (4 * pass)) & 3 : 0;
        const uint32_t dA = ring + st * kGmStage, dB = dA + kGmStageA, fb = full0 + st * 8;
        const CUtensorMap *ma = &s.a[seg], *mb = &s.b[EPI == kEpiGlu ? (PAIR ? (int)rank : 0) : seg];
        if (leader) {
          if (draws && i == draw_at) drawn = atomicAdd(p.ticket, 1);  // its latency passes under the copies
          if (rank == 0) mbar_arrive_expect_tx(&full[st], bytes);
          if (s.a_mn) {
            gm_load<PAIR>(dA, ma, arow, k, pa, fb);
            gm_load<PAIR>(dA + 8192, ma, arow + 64, k, pa, fb);
          } else {
            gm_load<PAIR>(dA, ma, k, arow, pa, fb);
          }
          if (EPI != kEpiGlu && s.b_mn) {
            gm_load<PAIR>(dB, mb, brow, k, pb, fb);
            if (brows > 64) gm_load<PAIR>(dB + 8192, mb, brow + 64, k, pb, fb);
          } else {
            gm_load<PAIR>(dB, mb, k, brow, pb, fb);
            if constexpr (EPI == kEpiGlu && !PAIR) gm_load<PAIR>(dB + (uint32_t)(bn / 2) * 128u, &s.b[1], k, brow, pb, fb);
          }
        }
        ++r;
        if constexpr (PLANES) {
          if (r == g0 + gn) {
            if (++pass == 6) {
              pass = 0;
              g0 += kGmGroup;
              gn = nks - g0 < kGmGroup ? nks - g0 : kGmGroup;
            }
            r = g0;
          }
        }
        if (++st == kGmStages) {
          st = 0;
          ph ^= 1;
        }
      }
      if (!ok) break;
      if (draws) {
        job = job_of(nworkers + __shfl_sync(0xffffffffu, drawn, lead));
        bool passed = true;
        if (leader) passed = pass_on(jn, job);
        ok = __all_sync(0xffffffffu, passed);
      } else {
        job = next_job(jn);
      }
    }
    if (job.sub == -2) ok = false;
    if (!ok) {
      give_up();
      // an aborted run leaves once the copies in flight have landed
      if (rank == 0)
        for (uint32_t n = it > kGmStages ? it - kGmStages : 0; n < it; ++n)
          mbar_wait(&full[n % kGmStages], (n / kGmStages) & 1, 10000000ull);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(sm) >> 4;
      uint32_t st = 0, ph = 0, sc = 0, jn = 0;
      bool ok = true;
      GemmJob job = next_job(0);
      for (; ok && job.sub >= 0; job = next_job(++jn)) {
        const GemmSub& s = p.sub[job.sub];
        uint32_t idesc = idesc_bf16(kTileM, bn, s.a_mn != 0, s.b_mn != 0);
        if (p.f16) idesc &= ~((1u << 7) | (1u << 10));
        // descriptors: the address in 16-byte units in the low bits, then the leading offset (MN-major:
        // 8192 bytes between 64-column blocks); a step of 16 K values is 32 bytes along a swizzled row, or
        // two 8-row groups of an MN-major tile
        const uint32_t sa = s.a_mn ? 128 : 2, sb = s.b_mn ? 128 : 2;
        const uint32_t la = (s.a_mn ? 8192u >> 4 : 1u) << 16, lb = (s.b_mn ? 8192u >> 4 : 1u) << 16;
        const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
        int i = job.kb;
        do {  // one accumulator a job, or one a group of K blocks
          const int e = GROUPS ? group_end(job, i) : job.ke;
          if (GROUPS && i == e) break;
          const uint32_t acc = sc & 1;
          ok = __all_sync(0xffffffffu, gm_wait(&acce[acc], ((sc >> 1) & 1) ^ 1, p.wait_ns));
          if (!ok) break;
          tc_fence_after();
          const uint32_t dt = tbase + acc * 256;
          uint32_t on = 0;
          for (; i < e; ++i) {
            ok = __all_sync(0xffffffffu, gm_wait(&full[st], ph, p.wait_ns));
            if (!ok) break;
            tc_fence_after();
            const uint32_t a0 = (ring + st * (kGmStage >> 4)) | la;
            const uint32_t b0 = (ring + st * (kGmStage >> 4) + (kGmStageA >> 4)) | lb;
            if (leader) {
#pragma unroll
              for (uint32_t kk = 0; kk < kGmBK / 16; ++kk) {
                const uint64_t da = gm_desc(a0 + kk * sa, hi), db = gm_desc(b0 + kk * sb, hi);
                if constexpr (PAIR) umma_bf16_pair(dt, da, db, idesc, kk == 0 ? on : 1u);
                else umma_bf16(dt, da, db, idesc, kk == 0 ? on : 1u);
              }
              gm_commit<PAIR>(&empty[st]);  // the stage is free, in both CTAs, once these MMAs have read it
            }
            on = 1;
            if (++st == kGmStages) {
              st = 0;
              ph ^= 1;
            }
          }
          if (ok && leader) gm_commit<PAIR>(&accf[acc]);
          ++sc;
        } while (GROUPS && ok && i < job.ke);
      }
      if (!ok || job.sub == -2) give_up();
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t tl = tbase + ((uint32_t)(q * 32) << 16);
    uint32_t sc = 0;
    // kEpiDglu: this warp's runs of g and u, in the order it will use them (the jobs are dealt, so the
    // next tile's are known), kGuSlots of them on their way or in shared memory
    uint64_t* gub = gufull + (warp - 2) * kGuSlots;
    const uint8_t* gus = sm + kGuOff + (uint32_t)(warp - 2) * kGuSlots * kGuRun<PLANES>;
    uint32_t gu_used = 0, gu_sent = 0, gu_tile = 0;
    int gu_run = 0, gu_runs = 0;
    const uint8_t* gu_at = nullptr;
    auto gu_enter = [&](const GemmJob& j) {  // the runs of tile j
      const int64_t row = (int64_t)j.mt * kTileM + (int64_t)rank * 128 + q * 32;
      const int col = j.nt * bn + half * (bn / 2), n = p.sub[0].N - col < bn / 2 ? p.sub[0].N - col : bn / 2;
      gu_run = 0;
      gu_runs = n > 0 ? (n + 31) / 32 * 4 : 0;
      gu_at = p.gu + ((row >> 5) * p.gu_ld + (col >> 3)) * kGuRun<PLANES>;
    };
    auto gu_send = [&]() {
      while (gu_run >= gu_runs) {
        const GemmJob j = next_job(gu_tile++);
        if (j.sub < 0) {
          --gu_tile;
          return;
        }
        gu_enter(j);
      }
      const uint32_t slot = gu_sent++ % kGuSlots;
      if (lane == 0) {
        mbar_arrive_expect_tx(&gub[slot], kGuRun<PLANES>);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                         smem_u32(gus + slot * kGuRun<PLANES>)),
                     "l"(gu_at + (int64_t)gu_run * kGuRun<PLANES>), "r"(kGuRun<PLANES>), "r"(smem_u32(&gub[slot]))
                     : "memory");
      }
      ++gu_run;
    };
    if constexpr (kDglu)
      for (int i = 0; i < kGuSlots; ++i) gu_send();
    float peak = 1.f;  // fp16: values are kept divided by it
    if constexpr (EPI == kEpiDlogit || EPI == kEpiDlogitSums || kDglu) {
      if (p.peaks) {
        peak = peak_scale(p.peaks, p.npeaks);
        if constexpr (kDglu) peak = fminf(peak * 256.f, 1.f);  // up to 2^-8, never down: see ffn.cu
        if (blockIdx.x == 0 && threadIdx.x == 64) *p.peak_out = peak;
      }
    }
    uint32_t jn = 0;
    GemmSend send{sm + kGmBoxOff + (uint32_t)(warp - 2) * kGmBox, 0};
    GemmJob job = next_job(0);
    for (; job.sub >= 0; job = next_job(++jn)) {
      const GemmSub& s = p.sub[job.sub];
      const int64_t grow = (int64_t)job.mt * kTileM + (int64_t)rank * 128 + q * 32 + lane;
      const int M = sched.rows(s);
      const bool rok = grow < M;  // grow is the row of this thread
      const bool none = job.ke == job.kb;  // no K at all: the sum is zero
      const int cfirst = half * (bn / 2), clast = cfirst + bn / 2;
      // waits for the next accumulator; tc: its columns of this warp's lanes
      uint32_t tc = 0;
      auto await = [&]() {
        const uint32_t acc = sc & 1;
        if (!__all_sync(0xffffffffu, gm_wait(&accf[acc], (sc >> 1) & 1, p.wait_ns))) return false;
        tc_fence_after();
        tc = tl + acc * 256;
        return true;
      };
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) gm_arrive_first<PAIR>(&acce[sc & 1]);
        ++sc;
      };
      float part[kPart][32];  // the columns (GLU: 32 of either half), summed over the groups
      if constexpr (GROUPS) {
#pragma unroll
        for (int k = 0; k < kPart; ++k)
#pragma unroll
          for (int i = 0; i < 32; ++i) part[k][i] = 0.f;
        bool fine = true;
        for (int i = job.kb; i < job.ke; i = group_end(job, i)) {
          fine = await();
          if (!fine) break;
#pragma unroll
          for (int k = 0; k < kPart; ++k) {
            if (EPI != kEpiGlu && 32 * k >= bn / 2) break;
            constexpr int kRun = kPart == 4 ? 16 : 32;  // beside 128 sums, 32 more registers would spill
#pragma unroll
            for (int h = 0; h < 32; h += kRun) {
              uint32_t ra[kRun];
              __syncwarp();
              const uint32_t at = tc + (EPI == kEpiGlu ? half * (bn / 4) + k * (bn / 2) : cfirst + 32 * k) + h;
              if constexpr (kRun == 16) tmem_ld16_async(at, ra);
              else tmem_ld32_async(at, ra);
              tmem_wait_ld(ra);
#pragma unroll
              for (int e = 0; e < kRun; e += 2) {
                const float2 x = add2(make_float2(part[k][h + e], part[k][h + e + 1]),
                                      make_float2(__uint_as_float(ra[e]), __uint_as_float(ra[e + 1])));
                part[k][h + e] = x.x, part[k][h + e + 1] = x.y;
              }
            }
          }
          release();
        }
        if (!fine) {
          give_up();
          break;
        }
      } else if (!await()) {
        give_up();
        break;
      }
      uint8_t* box = sm + kGmBoxOff + (uint32_t)(warp - 2) * kGmBox;
      GemmRows rows{(int64_t)job.mt * kTileM + (int64_t)rank * 128 + q * 32, M, nullptr};
      // Columns [c0, c1) of this warp, 32 at a time.  The load is waited for at once: a register that
      // an asynchronous load still writes must not be moved or spilled, and the second warp of the
      // same lanes covers the wait.
      auto columns = [&](int c0, int c1, auto&& f) {
        if constexpr (GROUPS) {
#pragma unroll
          for (int k = 0; k < kPart; ++k)
            if (c0 + 32 * k < c1) f(c0 + 32 * k, part[k]);
        } else {
          for (int c = c0; c < c1; c += 32) {
            uint32_t ra[32];
            __syncwarp();
            tmem_ld32_async(tc + c, ra);
            tmem_wait_ld(ra);
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = none ? 0.f : __uint_as_float(ra[i]);
            f(c, v);
          }
        }
      };
      auto scale_of = [&]() {
        float alpha = s.alpha;
        if (s.alpha_num) alpha *= *s.alpha_num;
        if (s.alpha_den) alpha = *s.alpha_den > 0 ? alpha / (float)*s.alpha_den : 0.f;
        return alpha;
      };
      auto put_scaled = [&](int col, float (&v)[32], float alpha) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= alpha;
        if (s.out.kind == kOutF32) put32(box, s.out, rows, col, s.N, v);
        else put_narrow(box, s.out, rows, col, s.N, v);
      };
      // a part of a split product, as it is
      auto put_part = [&](int col, const float (&v)[32]) {
        const int64_t nq = (int64_t)s.nt * bn / 4, size = (int64_t)s.mt * kTileM / 32 * nq * 32;
        float4* ap = reinterpret_cast<float4*>(s.part) + job.ks * size + ((grow >> 5) * nq + (col >> 2)) * 32 + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) ap[i * 32] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      };
      if constexpr (EPI == kEpiStore) {
        const float alpha = scale_of();
        columns(cfirst, clast, [&](int c, float (&v)[32]) {
          const int col = job.nt * bn + c;
          if (col >= s.N) return;
          if (s.split > 1) put_part(col, v);
          else put_scaled(col, v, alpha);
        });
      } else if constexpr (EPI == kEpiFinal) {
        const GemmFinal fin{s.alpha, s.bias, s.residual, s.ld_res, s.dt, s.res_vec};
        columns(cfirst, clast, [&](int c, float (&v)[32]) {
          const int col = job.nt * bn + c;
          if (col >= s.N) return;
          if (s.split > 1) put_part(col, v);
          else put_final(box, s.out, fin, rows, col, s.N, v);
        });
      } else if constexpr (EPI == kEpiAcc) {
        const float alpha = scale_of();
        rows.row_index = s.row_index;
        const int nq = s.nt * bn / 4;
        columns(cfirst, clast, [&](int c, float (&v)[32]) {
          const int col = job.nt * bn + c;
          if (col >= s.N) return;
          if (s.split > 1) {
            put_part(col, v);
            return;
          }
          if (s.acc_mode != 0) {
            float4* ap = reinterpret_cast<float4*>(s.acc) + ((grow >> 5) * nq + (col >> 2)) * 32 + lane;
            if (s.acc_mode != 1) {
              float4 o[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = ap[i * 32];
#pragma unroll
              for (int i = 0; i < 8; ++i)
                v[4 * i] += o[i].x, v[4 * i + 1] += o[i].y, v[4 * i + 2] += o[i].z, v[4 * i + 3] += o[i].w;
            }
            if (s.acc_mode != 3) {
#pragma unroll
              for (int i = 0; i < 8; ++i) ap[i * 32] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
              return;
            }
          }
          put_scaled(col, v, alpha);
        });
      } else if constexpr (EPI == kEpiGlu) {
        const int hb = bn / 2;
        for (int c = half * (hb / 2); c < (half + 1) * (hb / 2); c += 32) {
          const int col = job.nt * hb + c;
          float g[32], u[32];
          if constexpr (PLANES) {
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = part[0][i], u[i] = part[1][i];
          } else {
            uint32_t rg[32], ru[32];
            __syncwarp();
            tmem_ld32_async(tc + c, rg);
            tmem_ld32_async(tc + hb + c, ru);
            tmem_wait_ld(rg, ru);
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = __uint_as_float(rg[i]), u[i] = __uint_as_float(ru[i]);
          }
          if (col >= s.N) continue;
          if (s.bias) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 a = bias4(s.bias, s.dt, col + 4 * k, s.N), b = bias4(s.bias2, s.dt, col + 4 * k, s.N);
              g[4 * k] += a.x, g[4 * k + 1] += a.y, g[4 * k + 2] += a.z, g[4 * k + 3] += a.w;
              u[4 * k] += b.x, u[4 * k + 1] += b.y, u[4 * k + 2] += b.z, u[4 * k + 3] += b.w;
            }
          }
          if (p.gu) {
            uint8_t* run = p.gu + ((grow >> 5) * p.gu_ld + (col >> 3)) * kGuRun<PLANES> + lane * 16;
#pragma unroll
            for (int k = 0; k < 4; ++k, run += kGuRun<PLANES>) {
              if constexpr (PLANES) {
#pragma unroll
                for (int q4 = 0; q4 < 2; ++q4) {
                  const int i = 8 * k + 4 * q4;
                  *reinterpret_cast<float4*>(run + q4 * 512) = make_float4(g[i], g[i + 1], g[i + 2], g[i + 3]);
                  *reinterpret_cast<float4*>(run + 1024 + q4 * 512) = make_float4(u[i], u[i + 1], u[i + 2], u[i + 3]);
                }
              } else {
                uint32_t hi[8], lo[4];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                  const uint32_t g0 = __float_as_uint(g[8 * k + i]), g1 = __float_as_uint(g[8 * k + i + 1]);
                  const uint32_t u0 = __float_as_uint(u[8 * k + i]), u1 = __float_as_uint(u[8 * k + i + 1]);
                  hi[i] = __byte_perm(g0, u0, 0x7632);
                  hi[i + 1] = __byte_perm(g1, u1, 0x7632);
                  lo[i >> 1] = __byte_perm(__byte_perm(g0, u0, 0x0051), __byte_perm(g1, u1, 0x0051), 0x5410);
                }
                *reinterpret_cast<uint4*>(run) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(run + 512) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                *reinterpret_cast<uint4*>(run + 1024) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 g2 = make_float2(g[i], g[i + 1]);
            const float2 a = mul2(mul2(g2, sigmoid2(g2)), make_float2(u[i], u[i + 1]));
            g[i] = a.x, g[i + 1] = a.y;
          }
          if (rows.row0 < M) put_operand<PLANES>(send, &p.o[0], p.f16, col, rows.row0, g);
        }
      } else if constexpr (kDglu) {
        const float factor = s.alpha / peak;
        columns(cfirst, clast, [&](int c, float (&d)[32]) {
          const int col = job.nt * bn + c;
          if (col >= s.N) return;
          // 16-bit results are packed as they come: two packed arrays instead of two of 32
          float dg[8], du[PLANES ? 32 : 8];
          uint32_t wg[16], wu[16];
#pragma unroll
          for (int h = 0; h < 4; ++h, ++gu_used) {
            const uint32_t slot = gu_used % kGuSlots;
            if (!__all_sync(0xffffffffu, gm_wait(&gub[slot], (gu_used / kGuSlots) & 1, p.wait_ns))) give_up();
            const uint4* run = reinterpret_cast<const uint4*>(gus + slot * kGuRun<PLANES>) + lane;
            const uint4 r0 = run[0], r1 = run[32], r2 = run[64];
            uint32_t w[16];  // g and u of eight columns: fp32 words, or halves and their next bits
            w[0] = r0.x, w[1] = r0.y, w[2] = r0.z, w[3] = r0.w, w[4] = r1.x, w[5] = r1.y, w[6] = r1.z, w[7] = r1.w;
            w[8] = r2.x, w[9] = r2.y, w[10] = r2.z, w[11] = r2.w;
            if constexpr (PLANES) {
              const uint4 r3 = run[96];
              w[12] = r3.x, w[13] = r3.y, w[14] = r3.z, w[15] = r3.w;
            }
            __syncwarp();
            gu_send();
            const float2 one = make_float2(1.f, 1.f), alpha = make_float2(factor, factor);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              float2 g, u;
              if constexpr (PLANES) {
                g = make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1]));
                u = make_float2(__uint_as_float(w[8 + i]), __uint_as_float(w[9 + i]));
              } else {
                // the bits below stand twice: any do, and these need no instruction of their own
                const uint32_t lo = w[8 + (i >> 1)];
                g = make_float2(__uint_as_float(__byte_perm(w[i], lo, 0x1044)), __uint_as_float(__byte_perm(w[i + 1], lo, 0x1066)));
                u = make_float2(__uint_as_float(__byte_perm(w[i], lo, 0x3255)), __uint_as_float(__byte_perm(w[i + 1], lo, 0x3277)));
              }
              const float2 sg = sigmoid2(g);
              const float2 ds = mul2(mul2(make_float2(d[8 * h + i], d[8 * h + i + 1]), alpha), sg);
              const float2 x = mul2(mul2(ds, u), fma2(g, fma2(sg, make_float2(-1.f, -1.f), one), one)), y = mul2(ds, g);
              du[(PLANES ? 8 * h : 0) + i] = y.x, du[(PLANES ? 8 * h : 0) + i + 1] = y.y;
              if constexpr (PLANES) d[8 * h + i] = x.x, d[8 * h + i + 1] = x.y;
              else dg[i] = x.x, dg[i + 1] = x.y;
            }
            if constexpr (!PLANES) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                wg[4 * h + i] = pack16(dg[2 * i], dg[2 * i + 1], p.f16);
                wu[4 * h + i] = pack16(du[2 * i], du[2 * i + 1], p.f16);
              }
            }
            if constexpr (EPI == kEpiDgluSums) {
              // sums of 16 columns over the warp's rows in 16 shuffles: each step sends the half that the other
              // lane keeps, until lanes 2i and 2i + 1 have column i
              float a[16];
#pragma unroll
              for (int i = 0; i < 8; ++i) a[i] = rok ? dg[i] : 0.f, a[8 + i] = rok ? du[i] : 0.f;
#pragma unroll
              for (int o = 16, n = 8; n > 0; o >>= 1, n >>= 1) {
                const bool upper = (lane & o) != 0;
#pragma unroll
                for (int i = 0; i < n; ++i) {
                  const float other = __shfl_xor_sync(0xffffffffu, upper ? a[i] : a[i + n], o);
                  a[i] = (upper ? a[i + n] : a[i]) + other;
                }
              }
              a[0] += __shfl_xor_sync(0xffffffffu, a[0], 1);
              const int v = lane >> 1, c8 = col + 8 * h + (v & 7);
              if (!(lane & 1) && rows.row0 < M && c8 < s.N) (v < 8 ? p.sum_g : p.sum_u)[(rows.row0 >> 5) * s.N + c8] = a[0];
            }
          }
          if constexpr (PLANES) {
            if (rows.row0 < M) {
              put_operand<true>(send, &p.o[0], false, col, rows.row0, d);
              put_operand<true>(send, &p.o[1], false, col, rows.row0, du);
            }
          } else if (rows.row0 < M) {
            send(&p.o[0], col, rows.row0, 0, wg);
            send(&p.o[1], col, rows.row0, 0, wu);
          }
        });
      } else if constexpr (EPI == kEpiLse || EPI == kEpiLseSums) {
        const int tgt = rok ? p.target[grow] : -1;
        // the maximum as it is: a product with log2(e) would be rounded to 2^-24 of it, and with it the loss.
        // It starts at the least finite value, so that a set of -infinities has a sum of 0.
        float m = -FLT_MAX, sum = 0.f;
        columns(cfirst, clast, [&](int c, float (&v)[32]) {
          const int col = job.nt * bn + c;
          if (col >= s.N) return;
          const int to = tgt - col;
          if (to >= 0 && to < 32) {
            float x = v[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) x = to == i ? v[i] : x;
            p.target_logit[grow] = x;
          }
          if (col + 32 > s.N) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = col + i < s.N ? v[i] : -INFINITY;
          }
          float t[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int i = 4; i < 32; ++i) t[i & 3] = fmaxf(t[i & 3], v[i]);
          const float top = fmaxf(m, fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
          float e[4] = {sum * ex2_fast((m - top) * kLog2e), 0.f, 0.f, 0.f};
          m = top;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 x = mul2(add2(make_float2(v[i], v[i + 1]), make_float2(-top, -top)), make_float2(kLog2e, kLog2e));
            e[i & 3] += ex2_fast(x.x), e[(i & 3) + 1] += ex2_fast(x.y);
          }
          sum = (e[0] + e[1]) + (e[2] + e[3]);
        });
        if (rok) p.part[(int64_t)(job.nt * 2 + half) * p.part_ld + grow] = make_float2(m, sum);
      } else {
        const int tgt = rok ? p.target[grow] - p.col0 : -1;
        const float2 st = rok ? p.stat[grow] : make_float2(0.f, 0.f);
        const float ls = st.y - p.shift, one = ex2_fast(p.shift);
        const float w = rok && p.roww ? p.roww[grow] / peak : 1.f;
        // rows behind the last kept token are K values of the next products: zero
        columns(cfirst, clast, [&](int c, float (&v)[32]) {
          const int col = job.nt * bn + c;
          if (col >= s.N) return;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 t = fma2(add2(make_float2(v[i], v[i + 1]), make_float2(-st.x, -st.x)), make_float2(kLog2e, kLog2e),
                                  make_float2(-ls, -ls));
            v[i] = ex2_fast(t.x), v[i + 1] = ex2_fast(t.y);
          }
          const int to = tgt - col;
          if (to >= 0 && to < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = to == i ? v[i] - one : v[i];
          }
          if (p.roww) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= w;
          }
          if (!rok) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
          }
          put_operand<PLANES>(send, &p.o[0], p.f16, col, rows.row0, v);
        });
      }
      if constexpr (!GROUPS) release();
    }
    if (job.sub == -2) give_up();
    if (lane == 0) bulk_wait_group_all();  // boxes stay until they have been sent
    if constexpr (kDglu)  // an aborted run leaves once its copies have landed
      for (; gu_used < gu_sent; ++gu_used) mbar_wait(&gub[gu_used % kGuSlots], (gu_used / kGuSlots) & 1, 10000000ull);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // no remote arrivals or MMAs into this CTA remain
  if (warp == 0) {
    tc_fence_after();
    pair_tmem_dealloc<PAIR>(tbase, 512);
  }
}

// The split products of a launch: add the parts in order and store as the kernel's epilogue would.
// `warps` (a power of two) warps per 32 x 32 piece, lane = row, each with a run of the parts; bound by
// L2 (the parts were just written) and, with few pieces, by the latency of one load after the other.
template <int EPI>
__global__ void __launch_bounds__(256) gemm_join_kernel(const __grid_constant__ GemmParams p, int tile_m, int warps) {
  __shared__ __align__(1024) uint8_t boxes[8 * kGmBox];
  pdl_wait_primary();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp & (warps - 1);
  uint8_t* box = boxes + warp * kGmBox;
  const int dyn = p.dyn ? *p.dyn : 0;
  int64_t u = (int64_t)blockIdx.x * (8 / warps) + warp / warps;
  int i = 0;
  for (; i < p.nsub; ++i) {
    const GemmSub& s = p.sub[i];
    if (s.split <= 1) continue;
    const int64_t n = (int64_t)(((s.m_dyn ? dyn : s.M) + 31) / 32) * ((s.N + 31) / 32);
    if (u < n) break;
    u -= n;
  }
  const bool live = i < p.nsub;
  const GemmSub& s = p.sub[live ? i : 0];
  const int M = s.m_dyn ? dyn : s.M, cb = (s.N + 31) / 32;
  const int row0 = live ? (int)(u / cb) * 32 : 0, col = live ? (int)(u % cb) * 32 : 0;
  float v[32];
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = 0.f;
  if (live) {
    const int64_t nq = (int64_t)s.nt * p.bn / 4, size = (int64_t)s.mt * tile_m / 32 * nq * 32;
    const int each = (s.split + warps - 1) / warps, k0 = w * each, k1 = k0 + each < s.split ? k0 + each : s.split;
    const float4* ap = reinterpret_cast<const float4*>(s.part) + k0 * size + ((row0 >> 5) * nq + (col >> 2)) * 32 + lane;
    for (int ks = k0; ks < k1; ++ks, ap += size) {
      float4 o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = ap[k * 32];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[4 * k] += o[k].x, v[4 * k + 1] += o[k].y, v[4 * k + 2] += o[k].z, v[4 * k + 3] += o[k].w;
    }
  }
  if (warps > 1) {  // the runs' sums in order
    float4* mine = reinterpret_cast<float4*>(box);
#pragma unroll
    for (int k = 0; k < 8; ++k) mine[k * 32 + lane] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    __syncthreads();
    if (w != 0) return;
    for (int k2 = 1; k2 < warps; ++k2) {
      const float4* other = reinterpret_cast<const float4*>(box + k2 * kGmBox);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float4 o = other[k * 32 + lane];
        v[4 * k] += o.x, v[4 * k + 1] += o.y, v[4 * k + 2] += o.z, v[4 * k + 3] += o.w;
      }
    }
  }
  if (live) {
    const GemmRows rows{row0, M, s.row_index};
    if constexpr (EPI == kEpiFinal) {
      const GemmFinal fin{s.alpha, s.bias, s.residual, s.ld_res, s.dt, s.res_vec};
      put_final(box, s.out, fin, rows, col, s.N, v);
    } else {
      if (s.acc_mode != 0) {
        const int64_t nqa = (int64_t)s.nt * p.bn / 4;
        float4* acc = reinterpret_cast<float4*>(s.acc) + ((row0 >> 5) * nqa + (col >> 2)) * 32 + lane;
        if (s.acc_mode != 1) {
          float4 o[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = acc[k * 32];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[4 * k] += o[k].x, v[4 * k + 1] += o[k].y, v[4 * k + 2] += o[k].z, v[4 * k + 3] += o[k].w;
        }
        if (s.acc_mode != 3) {
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k * 32] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          return;
        }
      }
      float alpha = s.alpha;
      if (s.alpha_num) alpha *= *s.alpha_num;
      if (s.alpha_den) alpha = *s.alpha_den > 0 ? alpha / (float)*s.alpha_den : 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] *= alpha;
      if (s.out.kind == kOutF32) put32(box, s.out, rows, col, s.N, v);
      else put_narrow(box, s.out, rows, col, s.N, v);
    }
  }
}

// ---------------------------------------------------------------------------
// host side (gemm.cu)
// ---------------------------------------------------------------------------

// A 16-bit operand in memory: `planes` matrices of rows x cols, rows ld elements apart.
struct GemmOperand {
  const void* p;
  int64_t rows, cols, ld, plane;
  int planes;
};
// A matrix as the TMA can read it in place: 16-byte aligned rows.
inline bool tma_ok(const void* p, int64_t ld_elems) { return aligned16(p) && ld_elems % 8 == 0; }

// Tensor map of an operand; box_rows counts the other dimension's box when K is along the rows
// (K-major), MN-major maps always use 64 x 64 boxes.
int gemm_map(CUtensorMap* m, const GemmOperand& o, bool mn_major, int box_rows, bool f16);
// Tensor map of an operand that a kernel's epilogue writes.
int gemm_out_map(CUtensorMap* m, const GemmOperand& o, bool f16);
// Fills mt, nt and split from M, N, nk, npass and bn, and orders the products longest job first;
// returns the bytes of fp32 parts the split ones need (to be carved and given to launch_gemm).
size_t plan_gemm(GemmParams& p, int epi, bool pair);
// Launch a planned set of products on `st`; `parts`: plan_gemm's bytes; a launch with jobs of several
// lengths draws them from p.ticket (a zeroed int; null deals them in turn).
int launch_gemm(GemmParams& p, int epi, bool pair, void* parts, cudaStream_t st);
inline int gemm_tile_m(bool pair) { return pair ? 256 : 128; }
// Accumulator columns of a CTA pair's tiles for M x N columns (GLU: both halves): 256, or 128 where that
// still leaves every tile a pair of its own.  A tile of 128 takes as long over K (0.34 us a block against
// 0.36) but half as long on its way out (777 x 897 fp32: dg and du 60 us with 16 tiles, 38 us with 32).
// Planes: 128, whose 64 columns a thread can sum in registers.
int gemm_columns(int64_t M, int64_t N, bool planes);
// Rows of B per tensor-map box for `bn` accumulator columns.
inline int gemm_box_b(bool pair, int bn, int epi) { return epi == kEpiGlu || pair ? bn / 2 : bn; }

// dst planes (rows ld apart, zero from cols to ld) of src (rows src_ld apart): the operand form of a
// matrix the TMA cannot read in place, or of an fp32 one (three bf16 planes).
struct PackList {
  struct {
    const void* src;
    void* dst;
    int64_t rows, cols, src_ld, ld, plane;
  } m[5];
  int n = 0;
  void add(const void* src, int64_t rows, int64_t cols, int64_t src_ld, void* dst, int64_t ld, int64_t plane) {
    m[n++] = {src, dst, rows, cols, src_ld, ld, plane};
  }
};
int launch_pack(const PackList& l, int dtype, cudaStream_t st);

}  // namespace m3b
