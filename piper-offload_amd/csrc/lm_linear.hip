// lm_linear.hip -- products with MXFP4 weights and with one weight per group of
// rows: forward, input gradient and (dense weights) weight gradient.
//
//   forward       y[t,n]  = sum_k x[t,k] W[n,k] (+ bias[n])
//   input grad    dx[t,k] = sum_n dy[t,n] W[n,k]
//   weight grad   dW[e,n,k] = sum over the rows t of group e of dy[t,n] x[t,k]
//
// Sums are kept in fp32 by the matrix instructions and rounded once, on the
// store.  An MXFP4 value is e2m1 * 2^(scale - 127); in bf16 it is exact.
#include <algorithm>

#include "lm_impl.h"
#include "lm_linear.h"
#include "lm_linear8.h"
#include "lm_linear_few.h"
#include "lm_linear_host.h"

// ---------------------------------------------------------------------------
// 4-bit inputs: x quantised to MXFP4 (blocks of 32 along K, scale
// 2^(floor(log2 max) - 2)), and its scales and the weight's in the order the
// scaled MFMA takes them.  One launch: the first workgroups take 2048 values of a
// row of x per wave (8 a lane and load: 16 bytes in, 4 out, a block's maximum over
// 4 lanes by DPP), the others 64 rows x 16 blocks of weight scales per wave.  Bound
// by memory: 4096 rows of 4096 and the scales of [14336, 4096] 11.7 us, 50 MB moved.
// ---------------------------------------------------------------------------
// byte of (slot, block) in the packed scales: pieces of 64 slots x 4 blocks
DEV int64_t lin_packed(int64_t slot, int64_t block, int64_t nk) {
  const int f = (int)(slot >> 4) & 3, r = (int)slot & 15, g = (int)block & 3;
  return ((slot >> 6) * nk + (block >> 2)) * 256 + (16 * g + r) * 4 + f;
}
// PACK: rows in the padded order of their groups, packed scales (k_lin_mm); else
// both in row order (k_lin_few)
template <int DT, bool PACK>
__global__ __launch_bounds__(256) void k_lin_prep4(LinArgs a, uint32_t row_blocks, uint32_t segs, uint8_t* xq, uint8_t* xs, uint8_t* wsc) {
  const int lane = threadIdx.x & 63;
  const uint32_t nk = (uint32_t)((a.K + 127) >> 7), nb = (uint32_t)(a.K >> 5);
  if (!PACK || blockIdx.x < row_blocks) {
    const uint32_t item = blockIdx.x * 4 + wave_index(), t = item / segs, units = (uint32_t)(a.K >> 3);
    if (t >= a.T) return;
    const uint32_t u0 = (item - t * segs) * 256 + lane;
    const LM_GLOBAL uint16_t* x = (const LM_GLOBAL uint16_t*)a.a + t * a.lda;
    lm_u32x4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = lm_u32x4{};
      if (u0 + 64 * i < units) w[i] = *(const LM_GLOBAL lm_u32x4_any*)(x + (u0 + 64 * i) * 8);
    }
    int64_t p = t;
    if (PACK && a.ends) {
      int g = a.experts;
      lin_row(a, (int)t, g, p);
      if (g == a.experts) return;  // a row of no group
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = u0 + 64 * i;
      uint32_t s;
      const uint32_t c = lin_quant8<DT>(w[i], s);
      if (u < units) *(LM_GLOBAL uint32_t*)(xq + p * (a.K >> 1) + u * 4) = c;
      // (blocks past K, up to whole words of scales, are zeros with the smallest scale)
      if ((lane & 3) == 0 && (u >> 2) < nk * 4)
        ((LM_GLOBAL uint8_t*)xs)[PACK ? lin_packed(p, u >> 2, nk) : p * (int64_t)(nk * 4) + (u >> 2)] = (uint8_t)(u < units ? s : 0);
    }
  } else {
    // Lane 16f + r has the row of slot (f, r) and four words w[j], blocks 4j .. 4j + 3
    // of it.  The transpose of words between the lane groups gives lane group j the
    // words of all four f for piece j; a transpose of their bytes makes them the
    // words (g, r) of the piece.
    const uint32_t gj = (uint32_t)((a.N + 63) >> 6), quads = (nk + 3) >> 2;
    const int64_t item = (int64_t)(blockIdx.x - row_blocks) * 4 + wave_index(), eg = item / quads;
    if (eg >= (int64_t)gj * a.experts) return;
    const uint32_t q = (uint32_t)(item - eg * quads);
    const int64_t e = eg / gj, n = (eg - e * gj) * 64 + lane;
    const LM_GLOBAL uint8_t* src = (const LM_GLOBAL uint8_t*)a.scale + e * a.scale_stride;
    lm_u32x4 w = {};
    if (n < a.N) {
      if (a.swizzled) {
        src += blocked_offset(n, 0, nb, true);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * q + j < nk) w[j] = *(const LM_GLOBAL uint32_t*)(src + (4 * q + j) * (int64_t)512);
      } else if (16 * q + 16 <= nb) {
        w = *(const LM_GLOBAL lm_u32x4_any*)(src + n * nb + 16 * q);
      } else {
#pragma unroll
        for (int b = 0; b < 15; ++b)
          if (16 * q + b < nb) w[b >> 2] |= (uint32_t)src[n * nb + 16 * q + b] << (8 * (b & 3));
      }
    }
    if (a.swizzled && 16 * q + 16 > nb) {  // what the padding of the last tile holds
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int have = (int)nb - (int)(16 * q + 4 * j);
        if (have < 4) w[j] = have <= 0 ? 0u : w[j] & ((1u << (8 * have)) - 1);
      }
    }
    lin_transpose4(w);
    // bytes: v[g] = byte g of w[0], w[1], w[2], w[3]
    const uint32_t a0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), a1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
    const uint32_t b0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400), b1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
    const uint32_t v[4] = {(a0 & 0xffffu) | b0 << 16, a0 >> 16 | (b0 & 0xffff0000u), (a1 & 0xffffu) | b1 << 16, a1 >> 16 | (b1 & 0xffff0000u)};
    const uint32_t piece = 4 * q + (lane >> 4);
    if (piece < nk) {
#pragma unroll
      for (int g = 0; g < 4; ++g) *(LM_GLOBAL uint32_t*)(wsc + (eg * nk + piece) * 256 + (16 * g + (lane & 15)) * 4) = v[g];
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int check_lin(const lm_weight* w, int64_t T, int32_t dtype, const int32_t* ends, int32_t experts) {
  if (dtype != LM_BF16 && dtype != LM_F16) return fail(LM_EUNSUPPORTED, "products take bf16 and fp16 rows");
  if (T < 0 || T > 0x7fffffff) return fail(LM_EINVAL, "number of rows must be 0 to 2^31 - 1");
  if (experts < 1 || experts > LM_LINEAR_MAX_EXPERTS)
    return fail(LM_EINVAL, "number of groups must be 1 to %d, got %d", LM_LINEAR_MAX_EXPERTS, experts);
  if (experts > 1 && !ends) return fail(LM_EINVAL, "several groups need their ends");
  if (!w) return LM_OK;
  if (!w->q) return fail(LM_EINVAL, "weight pointer must be non-null");
  if (w->N <= 0 || w->K <= 0) return fail(LM_EINVAL, "empty weight");
  if (w->N >= (1 << 21) || w->K >= (1 << 21)) return fail(LM_EUNSUPPORTED, "products take rows and columns below 2^21");
  if (w->dtype == LM_E2M1) {
    if (!w->scale) return fail(LM_EINVAL, "MXFP4 weight without scales");
    if (w->K % 32 != 0) return fail(LM_EINVAL, "MXFP4 requires columns divisible by 32, got %lld", (long long)w->K);
    if (((uintptr_t)w->q & 15) != 0) return fail(LM_EINVAL, "MXFP4 codes must be 16-byte aligned");
  } else if (w->dtype == LM_I8) {
    if (!w->scale) return fail(LM_EINVAL, "INT8 weight without scales");
    if (w->reserved != LM_F32 && w->reserved != LM_BF16) return fail(LM_EUNSUPPORTED, "INT8 weights have fp32 or bf16 scales");
  } else if (w->dtype != dtype) {
    return fail(LM_EUNSUPPORTED, "a dense weight must have the rows' dtype");
  }
  return LM_OK;
}

static LinArgs lin_args(const lm_weight* w, const int32_t* ends, int64_t T) {
  LinArgs a{};
  a.w = w->q;
  a.scale = w->scale;
  a.N = w->N;
  a.K = w->K;
  a.swizzled = w->swizzled;
  a.experts = w->experts;
  if (w->dtype == LM_I8) {
    a.scale16 = w->reserved == LM_BF16;
    a.scale_stride = w->N * (a.scale16 ? 2 : 4);
  } else {
    a.scale_stride = lin_scale_bytes(w->N, w->K, w->swizzled);
  }
  a.ends = ends;
  a.T = T;
  return a;
}

// ---- how a product is run: a rule on its sizes, types and alignment ----------
// k_lin_few reads the operands once per 16 to 64 rows or columns and spreads over
// all CUs by splitting the contraction inside workgroups; k_lin_mm shares tiles.
// The first wins while the product is small, which is a matter of its volume T N
// K more than of any one size.  Measured, us few / mm: MXFP4 [4096, 4096] at 64 rows
// 13 / 15, at 96 rows 23 / 17; [1024, 4096] at 200 rows 12 / 14; [64, 4096] of 24
// groups at 2048 rows 13 / 18; [1000, 8192] at 300 rows 41 / 22.  4-bit inputs pay
// for the packing of the weight's scales in k_lin_mm: [4096, 14336] at 64 rows
// 31 / 37, at 128 rows 52 / 39; 32 groups [2816, 2048] of 16 rows 36 / 46, of 32 rows
// 58 / 42.  Dense: [4096, 4096] at 32 rows 14 / 15, at 64 rows 21 / 18; [64, 4096] of 24
// groups at 2048 rows 24 / 17.
static bool lin_few(int64_t T, int64_t N, int64_t K, int64_t E, bool mx, bool quant) {
  const int64_t rows = (T + E - 1) / E;
  const double volume = (double)T * (double)N * (double)K;
  if (K < 512 && T > 64) return false;  // too few units for the waves: [4096, 16] of 24 groups at 2048 rows 39 / 13
  // (k_lin_mm<SHORT>: [14336, 64] of 16 groups at 16 rows 16.5 / 5.5; [4096, 16] at one row 3.3 / 3.8)
  if (!mx && K <= 64 && T > 1) return false;
  if (!mx) return T <= 16 || volume <= 5e8;
  return rows <= 16 || volume <= 1.1e9 || (quant && T <= 64);
}

static LinPlan lin_plan(int op, int64_t T, int64_t lda, int64_t ldb, int64_t N, int64_t K, int64_t E, bool mx, bool quant,
                        bool aligned) {
  LinPlan p{};
  const int64_t rows = (T + E - 1) / E;  // of an average group
  p.few = op == LIN_FORWARD && lin_few(T, N, K, E, mx, quant);
  const int64_t inner = op == LIN_FORWARD ? K : N;  // elements of a row of a
  const bool whole = aligned && lda % 8 == 0 && lda < (1 << 21);
  const bool wwhole = aligned && K % 8 == 0;
  p.lda = lda;
  p.ldb = ldb;
  p.ldw = K;
  p.len = op == LIN_WEIGHT_GRAD ? 0 : inner;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += align256(bytes);
    return o;
  };
  if (p.few) {
    p.copy_a = lda >= (1 << 21);
  } else if (!quant) {
    p.copy_a = !whole || (op != LIN_WEIGHT_GRAD && inner % 8);
    p.copy_b = op == LIN_WEIGHT_GRAD && (!aligned || ldb % 8 || ldb >= (1 << 21));
    p.copy_w = op != LIN_WEIGHT_GRAD && !mx && !wwhole;
    if (op != LIN_WEIGHT_GRAD) p.len = round8(inner);
  }
  if (p.copy_a) {
    p.lda = round8(inner);
    p.a = take((size_t)T * p.lda * 2);
  }
  if (p.copy_b) {
    p.ldb = round8(K);
    p.b = take((size_t)T * p.ldb * 2);
  }
  if (p.copy_w) {
    p.ldw = round8(K);
    p.w = take((size_t)E * N * p.ldw * 2);
  }
  if (quant) {
    const int64_t nk = (K + 127) / 128;
    p.padded = (T + 63) / 64 + E;
    p.xq = take((size_t)(p.padded * 64) * (size_t)(K / 2));
    p.xs = take((size_t)(p.padded * nk) * 256);
    p.wsc = take((size_t)(E * ((N + 63) / 64) * nk) * 256);
  }
  p.splits = 1;
  // Contractions of at most two stages, the ranks of adapters: a write of the
  // output.  [16, 4096] of 24 groups at 2048 rows 14.8 -> 9.9 us (input gradient,
  // 1.7 TB/s), [16, 14336] of 8 groups at 4096 rows 53.5 -> 28.8 (4.1 TB/s).
  p.brief = !p.few && !mx && op != LIN_WEIGHT_GRAD && p.len <= 64;
  if (!p.few && !p.brief) {
    const int64_t I = op == LIN_WEIGHT_GRAD ? N : T, J = op == LIN_FORWARD ? N : K;
    lin_tiling(p, op, I, J, op == LIN_WEIGHT_GRAD ? rows : p.len, E, mx, quant);
    if (p.splits > 1) p.part = take((size_t)p.splits * (op == LIN_WEIGHT_GRAD ? E * N : T) * J * 4);
  }
  p.total = at;
  return p;
}

static int launch_align(const void* src, int64_t lds, int64_t rows, int64_t cols, uint8_t* dst, int64_t ldd, hipStream_t st) {
  TimedLaunch timed("linear_prep", st);
  const int64_t n = (rows * (ldd / 8) + 255) / 256;
  if (n == 0) return LM_OK;
  if (!lin_holds(n, 256)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  hipLaunchKernelGGL(k_lin_align, dim3((unsigned)n), dim3(256), 0, st, (const uint16_t*)src, lds, rows, cols, (uint16_t*)dst, ldd);
  LAUNCH_CHECK();
  return LM_OK;
}

template <int DT, int W, int MF, int CF, int NW, int UN, bool EDGE = false>
static int launch_few(const LinArgs& a, hipStream_t st) {
  TimedLaunch timed("linear_few", st);
  const int64_t n = lin_tiles<16 * MF>(a.T, a.experts, a.ends != nullptr) * ((a.N + 16 * CF - 1) / (16 * CF));
  if (!lin_holds(n, NW * 64)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  hipLaunchKernelGGL((k_lin_few<DT, W, MF, CF, NW, UN, EDGE>), dim3((unsigned)n), dim3(NW * 64), 0, st, a);
  LAUNCH_CHECK();
  return LM_OK;
}
// Workgroups of 16 columns spread a small weight over the most CUs, wider ones read
// the rows less often; loads in flight want many units a wave, short contractions
// fewer waves, so that none is left without a unit.  `wgs`: workgroups at 16 rows x
// 16 columns.  Measured, us (weights out of memory, waves x units a wave x columns):
//   MXFP4 weight [4096, 4096], 1 row      8x4x16 5.4   8x4x32 6.3    16x2x16 5.5
//   [14336, 4096], 16 rows                8x4x64 13.3  16x2x64 14.0  8x4x32 16.7
//   32 groups [2816, 2048], 16 rows       4x2x32 16.5  8x2x64 18.6   8x4x64 20.5
//   32 groups [2048, 1408], 512 rows      4x2x64 22.8  4x2x32 25.8   8x4x64 31.3
//   4-bit inputs: [14336, 4096], 1 row    8x4x16 12.6  8x4x32 13.6   8x4x64 14.0
//   [4096, 14336], 24 rows                8x4x32 21.8  8x4x16 26.4
//   [14336, 4096], 64 rows                8x1x64 on 64 rows 25.7, 8x2x64 37.0
//   32 groups [2816, 2048], 16 rows       4x4x32 18.3  4x2x32 19.9   8x2x32 20.3
//   dense [2048, 4096], 1 row             16x2x16 8.2  8x2x16 8.6    4x2x16 10.0
//   [4096, 4096], 16 rows                 8x2x32 16.3  8x2x16 18.8   4x2x32 18.2
//   64 groups [2048, 1408], 100 rows      4x2x16 52.9  8x2x32 56.5   16x2x64 71.3
template <int DT, int W>
static int run_few_dt(const LinArgs& a, hipStream_t st) {
  if constexpr (W == W_DENSE) {
    if (a.K % 8) return launch_few<DT, W, 2, 1, 8, 1, true>(a, st);
  }
  const int64_t rows = (a.T + a.experts - 1) / a.experts, units = (a.K + 127) / 128;
  const int64_t wgs = lin_tiles<16>(a.T, a.experts, a.experts > 1) * ((a.N + 15) / 16);
  if (rows > 32 && wgs > 2048) return launch_few<DT, W, 4, 4, 8, 1>(a, st);
  if constexpr (W == W_DENSE) {
    // (16 waves with nothing to do for most of them: [4096, 16] 4.9, 4 waves 3.3)
    if (wgs <= 256 && units > 8) return launch_few<DT, W, 1, 1, 16, 2>(a, st);
    return units < 32 ? launch_few<DT, W, 1, 1, 4, 2>(a, st) : launch_few<DT, W, 1, 2, 8, 2>(a, st);
  } else {
    if (wgs <= 256 || (W == W_Q4 && rows <= 8 && units >= 32)) return launch_few<DT, W, 1, 1, 8, 4>(a, st);
    if (units >= 32) return wgs <= 512 ? launch_few<DT, W, 1, 2, 8, 4>(a, st) : launch_few<DT, W, 1, 4, 8, 4>(a, st);
    if constexpr (W == W_Q4) return launch_few<DT, W, 1, 2, 4, 4>(a, st);
    else return rows > 8 ? launch_few<DT, W, 1, 4, 4, 2>(a, st) : launch_few<DT, W, 1, 2, 4, 2>(a, st);
  }
}
template <int W>
static int run_few(const LinArgs& a, int dtype, hipStream_t st) {
  return dtype == LM_F16 ? run_few_dt<F16, W>(a, st) : run_few_dt<BF16, W>(a, st);
}

// copies of rows that are not whole 16-byte pieces, and the pointers of the plan
static int lin_setup(LinArgs& a, const LinPlan& p, int op, void* workspace, size_t workspace_bytes, hipStream_t st) {
  if (p.total > 0) {
    if (!workspace || workspace_bytes < p.total)
      return fail(LM_EWORKSPACE, "workspace too small: %zu < %zu bytes", workspace ? workspace_bytes : 0, p.total);
    if (((uintptr_t)workspace & 255) != 0) return fail(LM_EINVAL, "workspace must be 256-byte aligned");
  }
  uint8_t* base = (uint8_t*)workspace;
  const int64_t inner = op == LIN_FORWARD ? a.K : a.N;
  int rc;
  if (p.copy_a) {
    if ((rc = launch_align(a.a, a.lda, a.T, inner, base + p.a, p.lda, st))) return rc;
    a.a = base + p.a;
  }
  if (p.copy_b) {
    if ((rc = launch_align(a.b, a.ldb, a.T, a.K, base + p.b, p.ldb, st))) return rc;
    a.b = base + p.b;
  }
  if (p.copy_w) {
    if ((rc = launch_align(a.w, a.K, a.experts * a.N, a.K, base + p.w, p.ldw, st))) return rc;
    a.w = base + p.w;
  }
  a.lda = p.lda;
  a.ldb = p.ldb;
  a.ldw = p.ldw;
  a.len = p.len;
  a.padded = p.padded;
  a.part = p.splits > 1 ? (float*)(base + p.part) : nullptr;
  a.xq = base + p.xq;
  a.xs = base + p.xs;
  a.wsc = base + p.wsc;
  return LM_OK;
}

extern "C" size_t lm_linear_workspace_size(int32_t op, int64_t T, int64_t lda, int64_t ldb, int64_t N, int64_t K,
                                           int32_t experts, int32_t weight_dtype, int32_t input_dtype, int32_t aligned) {
  if (T <= 0 || N <= 0 || K <= 0 || experts <= 0 || op < LM_LINEAR_FORWARD || op > LM_LINEAR_WEIGHT_GRAD) return 0;
  if (weight_dtype == LM_I8) return op == LIN_WEIGHT_GRAD ? 0 : lin8_workspace(op, T, lda, N, K, experts, input_dtype == LM_I8, aligned != 0, input_dtype != LM_BF16);
  return lin_plan(op, T, lda, ldb, N, K, experts, weight_dtype == LM_E2M1, op == LIN_FORWARD && input_dtype == LM_E2M1, aligned != 0)
      .total;
}

extern "C" int lm_linear(const void* x, int64_t ldx, const lm_weight* w, const void* bias, const int32_t* ends, void* y,
                         int64_t T, int32_t dtype, int32_t input_dtype, void* workspace, size_t workspace_bytes,
                         void* stream) {
  int rc;
  if (!w) return fail(LM_EINVAL, "lm_linear requires a weight");
  if ((rc = check_lin(w, T, dtype, ends, w->experts))) return rc;
  const bool mx = w->dtype == LM_E2M1, quant = input_dtype == LM_E2M1, i8 = w->dtype == LM_I8;
  if (!quant && input_dtype != dtype && input_dtype != LM_I8)
    return fail(LM_EUNSUPPORTED, "the product's input dtype is the rows', LM_E2M1 or LM_I8");
  if (quant && !mx) return fail(LM_EUNSUPPORTED, "4-bit inputs need an MXFP4 weight");
  if (input_dtype == LM_I8 && !i8) return fail(LM_EUNSUPPORTED, "8-bit inputs need an INT8 weight");
  if (input_dtype == LM_I8 && w->K > LIN8_MAX_SUM)
    return fail(LM_EUNSUPPORTED, "8-bit products sum up to %d columns in 32 bits, got %lld", LIN8_MAX_SUM, (long long)w->K);
  if (T == 0) return LM_OK;
  if (!x || !y) return fail(LM_EINVAL, "row pointers must be non-null");
  if (ldx < w->K) return fail(LM_EINVAL, "row stride below the row length");
  hipStream_t st = (hipStream_t)stream;
  LinArgs a = lin_args(w, ends, T);
  a.a = x;
  a.lda = ldx;
  a.bias = bias;
  a.out = y;
  if (i8) return lin8_forward(a, dtype, input_dtype == LM_I8, workspace, workspace_bytes, st);
  const LinPlan p = lin_plan(LIN_FORWARD, T, ldx, 0, a.N, a.K, a.experts, mx, quant, aligned16(x) && aligned16(w->q));
  if ((rc = lin_setup(a, p, LIN_FORWARD, workspace, workspace_bytes, st))) return rc;
  if (!quant) {
    if (p.few) return mx ? run_few<W_MX>(a, dtype, st) : run_few<W_DENSE>(a, dtype, st);
    return mx ? run_mm<LIN_FORWARD, W_MX>(a, p, dtype, st) : run_mm<LIN_FORWARD, W_DENSE>(a, p, dtype, st);
  }
  uint8_t *xq = (uint8_t*)a.xq, *xs = (uint8_t*)a.xs, *wsc = (uint8_t*)a.wsc;
  {
    TimedLaunch timed("linear_prep", st);
    const int64_t segs = (a.K + 2047) / 2048, rows = (T * segs + 3) / 4;
    const int64_t pieces = p.few ? 0 : (a.experts * ((a.N + 63) / 64) * ((a.K + 511) / 512) + 3) / 4;
    if (T * segs > 0x7fffffff || !lin_holds(rows + pieces, 256)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
    const dim3 grid((unsigned)(rows + pieces));
#define PREP(DT, PACK) hipLaunchKernelGGL((k_lin_prep4<DT, PACK>), grid, dim3(256), 0, st, a, (uint32_t)rows, (uint32_t)segs, xq, xs, wsc)
    if (p.few) {
      if (dtype == LM_F16) PREP(F16, false);
      else PREP(BF16, false);
    } else {
      if (dtype == LM_F16) PREP(F16, true);
      else PREP(BF16, true);
    }
#undef PREP
    LAUNCH_CHECK();
  }
  return p.few ? run_few<W_Q4>(a, dtype, st) : run_mm<LIN_FORWARD, W_Q4>(a, p, dtype, st);
}

extern "C" int lm_linear_input_grad(const void* dy, int64_t lddy, const lm_weight* w, const int32_t* ends, void* dx,
                                    int64_t T, int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if (!w) return fail(LM_EINVAL, "lm_linear_input_grad requires a weight");
  if ((rc = check_lin(w, T, dtype, ends, w->experts))) return rc;
  if (T == 0) return LM_OK;
  if (!dy || !dx) return fail(LM_EINVAL, "row pointers must be non-null");
  if (lddy < w->N) return fail(LM_EINVAL, "row stride below the row length");
  hipStream_t st = (hipStream_t)stream;
  const bool mx = w->dtype == LM_E2M1;
  LinArgs a = lin_args(w, ends, T);
  a.a = dy;
  a.lda = lddy;
  a.out = dx;
  if (w->dtype == LM_I8) return lin8_input_grad(a, dtype, workspace, workspace_bytes, st);
  const LinPlan p = lin_plan(LIN_INPUT_GRAD, T, lddy, 0, a.N, a.K, a.experts, mx, false, aligned16(dy) && aligned16(w->q));
  if ((rc = lin_setup(a, p, LIN_INPUT_GRAD, workspace, workspace_bytes, st))) return rc;
  return mx ? run_mm<LIN_INPUT_GRAD, W_MX>(a, p, dtype, st) : run_mm<LIN_INPUT_GRAD, W_DENSE>(a, p, dtype, st);
}

extern "C" int lm_linear_weight_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const int32_t* ends,
                                     void* dw, int64_t T, int64_t N, int64_t K, int32_t experts, int32_t dtype,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_lin(nullptr, T, dtype, ends, experts))) return rc;
  if (N <= 0 || K <= 0) return fail(LM_EINVAL, "empty weight gradient");
  if (N >= (1 << 21) || K >= (1 << 21)) return fail(LM_EUNSUPPORTED, "products take rows and columns below 2^21");
  if (!dw || (T > 0 && (!dy || !x))) return fail(LM_EINVAL, "pointers must be non-null");
  if (lddy < N || ldx < K) return fail(LM_EINVAL, "row stride below the row length");
  hipStream_t st = (hipStream_t)stream;
  LinArgs a{};
  a.a = dy;
  a.lda = lddy;
  a.b = x;
  a.ldb = ldx;
  a.ends = ends;
  a.experts = experts;
  a.out = dw;
  a.T = T;
  a.N = N;
  a.K = K;
  const LinPlan p = lin_plan(LIN_WEIGHT_GRAD, T, lddy, ldx, N, K, experts, false, false, aligned16(dy) && aligned16(x));
  if ((rc = lin_setup(a, p, LIN_WEIGHT_GRAD, workspace, workspace_bytes, st))) return rc;
  return run_mm<LIN_WEIGHT_GRAD, W_DENSE>(a, p, dtype, st);
}
