// lm_linear.hip -- products with MXFP4 weights and with one weight per group of
// rows: forward, input gradient and (dense weights) weight gradient.
//
//   forward       y[t,n]  = sum_k x[t,k] W[n,k] (+ bias[n])
//   input grad    dx[t,k] = sum_n dy[t,n] W[n,k]
//   weight grad   dW[e,n,k] = sum over the rows t of group e of dy[t,n] x[t,k]
//
// Sums are kept in fp32 by the matrix instructions and rounded once, on the
// store.  An MXFP4 value is e2m1 * 2^(scale - 127); in bf16 it is exact.
#include "lm_impl.h"
#include "lm_linear.h"
#include "lm_linear_mm.h"

// ---------------------------------------------------------------------------
// 4-bit inputs: x quantised to MXFP4 (blocks of 32 along K, scale
// 2^(floor(log2 max) - 2)), and its scales and the weight's in the order the
// scaled MFMA takes them.  One launch: the first workgroups take a row of x per
// wave (8 values a lane: 16 bytes in, 4 out, a block's maximum over 4 lanes
// by DPP), the others one packed piece of weight scales per wave.
// ---------------------------------------------------------------------------
// byte of (slot, block) in the packed scales: pieces of 64 slots x 8 blocks
DEV int64_t lin_packed(int64_t slot, int64_t block, int64_t nk) {
  const int f = (int)(slot >> 4) & 3, r = (int)slot & 15, g = (int)(block & 7) >> 1;
  return ((slot >> 6) * nk + (block >> 3)) * 512 + (16 * g + r) * 8 + 2 * f + (block & 1);
}
template <int DT>
__global__ __launch_bounds__(256) void k_lin_prep4(LinArgs a, int row_blocks, uint8_t* xq, uint8_t* xs, uint8_t* wsc) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t nk = (a.K + 255) >> 8, nb = a.K >> 5;
  if ((int)blockIdx.x < row_blocks) {
    const int64_t t = (int64_t)blockIdx.x * 4 + wave;
    if (t >= a.T) return;
    int64_t p = t;
    if (a.ends) {
      int g;
      if (!lin_row(a, (int)t, g, p) || g == a.experts) return;  // a row of no group
    }
    const uint16_t* x = (const uint16_t*)a.a + t * a.lda;
    const int64_t units = a.K >> 3, padded = nk * 32;
    for (int64_t u = lane; u < padded; u += 64) {
      float v[8] = {};
      if (u < units) {
        const lm_u32x4 w = *(const LM_GLOBAL lm_u32x4_any*)(x + u * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = val_dt<DT>(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu);
      }
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t b = f2u(v[j]) & 0x7fffffffu;
        top = b > top ? b : top;
      }
#pragma unroll
      for (int d = 1; d <= 2; ++d) {
        const uint32_t o = (uint32_t)(d == 1 ? __builtin_amdgcn_update_dpp((int)top, (int)top, 0xB1, 0xf, 0xf, false)
                                             : __builtin_amdgcn_update_dpp((int)top, (int)top, 0x4E, 0xf, 0xf, false));
        top = o > top ? o : top;
      }
      float inv;
      const uint32_t s = lin_scale4(top, inv);
      const uint32_t w = lin_codes8(v, inv);
      if (u < units) *(LM_GLOBAL uint32_t*)(xq + p * (a.K >> 1) + u * 4) = w;
      // (blocks past K are zeros with the smallest scale)
      if ((lane & 3) == 0) *(LM_GLOBAL uint8_t*)(xs + lin_packed(p, u >> 2, nk)) = (uint8_t)(u < units ? s : 0);
    }
  } else {
    const int64_t gj = (a.N + 63) >> 6, piece = (int64_t)(blockIdx.x - row_blocks) * 4 + wave;
    if (piece >= gj * nk * a.experts) return;
    const int64_t kt = piece % nk, eg = piece / nk, e = eg / gj, n0 = (eg % gj) * 64;
    const int g = lane >> 4;
    uint16_t s[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int64_t n = n0 + lin_jcol(16 * f + (lane & 15));
      s[f] = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t b = kt * 8 + 2 * g + h;
        if (n < a.N && b < nb) s[f] |= (uint16_t)(a.scale[e * a.scale_stride + blocked_offset(n, b, nb, a.swizzled)] << (8 * h));
      }
    }
    *(LM_GLOBAL lm_u32x2*)(wsc + piece * 512 + lane * 8) = lm_u32x2{s[0] | (uint32_t)s[1] << 16, s[2] | (uint32_t)s[3] << 16};
  }
}

// ---------------------------------------------------------------------------
// the general product: any sizes, strides and alignment, 64 x 64 tiles
// ---------------------------------------------------------------------------
template <int DT, bool MX>
struct LinOps {
  static constexpr bool HALF = DT == F16;
  DEV static uint16_t bits(float v) { return HALF ? f16_bits(v) : bf16_bits(v); }
  DEV static uint16_t act(const LinArgs& a, int64_t m, int64_t c) {
    return ((const uint16_t*)a.a)[m * a.lda + c];
  }
  DEV static uint16_t weight(const LinArgs& a, int64_t e, int64_t n, int64_t k) {
    if constexpr (MX) {
      const uint32_t code = ((const uint8_t*)a.w)[(e * a.N + n) * (a.K >> 1) + (k >> 1)] >> (4 * (k & 1));
      const uint8_t s = a.scale[e * a.scale_stride + blocked_offset(n, k >> 5, a.K >> 5, a.swizzled)];
      return bits(e2m1_value(code) * e8m0_value(s));
    } else {
      return ((const uint16_t*)a.w)[(e * a.N + n) * a.K + k];
    }
  }
};

template <int DT, bool MX, int OP>
__global__ __launch_bounds__(256) void k_lin_general(LinArgs a) {
  using O = LinOps<DT, MX>;
  __shared__ __attribute__((aligned(16))) uint16_t la[64 * 40], lb[64 * 40];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t e, m0, m1, i0, iend, c0 = 0, cend;
  const int64_t j0 = (int64_t)blockIdx.x * 64, jend = OP == LIN_FORWARD ? a.N : a.K;
  if constexpr (OP == LIN_WEIGHT_GRAD) {
    e = blockIdx.z;
    lin_group(a, (int)e, m0, m1);
    i0 = (int64_t)blockIdx.y * 64;
    iend = a.N;
    c0 = m0;
    cend = m1;
  } else {
    int eg;
    if (!lin_tile<64>(a, blockIdx.y, eg, i0, iend)) return;
    e = eg;
    cend = e == a.experts ? 0 : (OP == LIN_FORWARD ? a.K : a.N);  // rows of no group: zeros
  }
  v4f32 acc[4] = {};
  for (int64_t c = c0; c < cend; c += 32) {
    for (int u = tid; u < 64 * 32; u += 256) {
      const int r = u >> 5, k = u & 31;
      const int64_t i = i0 + r, j = j0 + r, cc = c + k;
      uint16_t va = 0, vb = 0;
      if (cc < cend) {
        if (i < iend) va = OP == LIN_WEIGHT_GRAD ? O::act(a, cc, i) : O::act(a, i, cc);
        if (j < jend)
          vb = OP == LIN_FORWARD ? O::weight(a, e, j, cc)
                                 : (OP == LIN_INPUT_GRAD ? O::weight(a, e, cc, j) : ((const uint16_t*)a.b)[cc * a.ldb + j]);
      }
      la[r * 40 + k] = va;
      lb[r * 40 + k] = vb;
    }
    __syncthreads();
    const lm_u32x4 fa = *(const lm_u32x4*)(la + (wave * 16 + (lane & 15)) * 40 + (lane >> 4) * 8);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const lm_u32x4 fb = *(const lm_u32x4*)(lb + (t * 16 + (lane & 15)) * 40 + (lane >> 4) * 8);
      acc[t] = lin_mfma<O::HALF>(fa, fb, acc[t]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int64_t j = j0 + t * 16 + (lane & 15);
    if (j >= jend) continue;
    const float bias = OP == LIN_FORWARD && a.bias && e < a.experts ? val_dt<DT>(((const uint16_t*)a.bias)[j]) : 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t i = i0 + wave * 16 + (lane >> 4) * 4 + r;
      if (i < iend) {
        const int64_t row = OP == LIN_WEIGHT_GRAD ? e * a.N + i : i;
        ((uint16_t*)a.out)[row * jend + j] = bits_dt<DT>(acc[t][r] + bias);
      }
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
  if (w->N >= (1 << 22) || w->K >= (1 << 22)) return fail(LM_EUNSUPPORTED, "products take rows and columns below 2^22");
  if (w->dtype == LM_E2M1) {
    if (!w->scale) return fail(LM_EINVAL, "MXFP4 weight without scales");
    if (w->K % 32 != 0) return fail(LM_EINVAL, "MXFP4 requires columns divisible by 32, got %lld", (long long)w->K);
    if (((uintptr_t)w->q & 15) != 0) return fail(LM_EINVAL, "MXFP4 codes must be 16-byte aligned");
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
  a.scale_stride = lin_scale_bytes(w->N, w->K, w->swizzled);
  a.ends = ends;
  a.T = T;
  return a;
}

// workspace of 4-bit inputs; padded: 64-row pieces that the rows of T rows in
// `experts` groups can fill
struct LinWs {
  int64_t padded;
  size_t xs, wsc, total;
};
static LinWs lin_ws(int64_t T, int64_t N, int64_t K, int64_t experts, bool grouped) {
  LinWs w;
  const int64_t nk = (K + 255) / 256;
  w.padded = (T + 63) / 64 + (grouped ? experts : 0);
  w.xs = align256((size_t)(w.padded * 64) * (size_t)(K / 2));
  w.wsc = w.xs + (size_t)(w.padded * nk) * 512;
  w.total = w.wsc + (size_t)(experts * ((N + 63) / 64) * nk) * 512;
  return w;
}

template <int DT, bool MX, int OP>
static int run_general(const LinArgs& a, hipStream_t st) {
  TimedLaunch timed("linear", st);
  const int64_t J = OP == LIN_FORWARD ? a.N : a.K;
  const int64_t gx = (J + 63) / 64;
  const int64_t gy = OP == LIN_WEIGHT_GRAD ? (a.N + 63) / 64 : lin_tiles<64>(a.T, a.experts, a.ends != nullptr);
  if (gx > 0x7fffffff || gy > 65535) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  hipLaunchKernelGGL((k_lin_general<DT, MX, OP>), dim3((unsigned)gx, (unsigned)gy, OP == LIN_WEIGHT_GRAD ? a.experts : 1),
                     dim3(256), 0, st, a);
  LAUNCH_CHECK();
  return LM_OK;
}
// Whole 16-byte pieces along every row that is read, offsets inside a tile below
// 2^31, fewer tiles than a grid holds.
static bool mm_ok(const LinArgs& a, int op, bool mx) {
  const int64_t len = op == LIN_FORWARD ? a.K : a.N;
  if (a.lda % 8 || ((uintptr_t)a.a & 15) || a.lda >= (1 << 22)) return false;
  if (op == LIN_WEIGHT_GRAD) return a.ldb % 8 == 0 && ((uintptr_t)a.b & 15) == 0 && a.ldb < (1 << 22);
  if (len % 8) return false;
  return mx || (a.K % 8 == 0 && ((uintptr_t)a.w & 15) == 0);
}

template <int DT, int OP, int MX, int B, int WM, int WN>
static int launch_mm(const LinArgs& a, hipStream_t st) {
  TimedLaunch timed("linear", st);
  const int64_t J = OP == LIN_FORWARD ? a.N : a.K, gj = (J + B - 1) / B;
  const int64_t gi = OP == LIN_WEIGHT_GRAD ? (a.N + B - 1) / B : lin_tiles<B>(a.T, a.experts, a.ends != nullptr);
  if (gi * gj > 0x7fffffff) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  hipLaunchKernelGGL((k_lin_mm<DT, OP, MX, B, B, WM, WN>), dim3((unsigned)(gi * gj), OP == LIN_WEIGHT_GRAD ? a.experts : 1),
                     dim3(WM * WN * 64), 0, st, a);
  LAUNCH_CHECK();
  return LM_OK;
}
template <int OP, int MX>
static int run_mm(const LinArgs& a, int dtype, hipStream_t st) {
  const int64_t J = OP == LIN_FORWARD ? a.N : a.K, I = OP == LIN_WEIGHT_GRAD ? a.N : a.T;
  const int64_t big = I / 256 * ((J + 255) / 256) * (OP == LIN_WEIGHT_GRAD ? a.experts : 1);
  const bool wide = big >= 192 && (OP == LIN_WEIGHT_GRAD || a.T / a.experts >= 256);
  if (dtype == LM_F16)
    return wide ? launch_mm<F16, OP, MX, 256, 2, 4>(a, st) : launch_mm<F16, OP, MX, 128, 2, 2>(a, st);
  return wide ? launch_mm<BF16, OP, MX, 256, 2, 4>(a, st) : launch_mm<BF16, OP, MX, 128, 2, 2>(a, st);
}

template <int OP>
static int run_product(const LinArgs& a, int dtype, bool mx, hipStream_t st) {
  if (mm_ok(a, OP, mx)) {
    if constexpr (OP != LIN_WEIGHT_GRAD) {
      if (mx) return run_mm<OP, W_MX>(a, dtype, st);
    }
    return run_mm<OP, W_DENSE>(a, dtype, st);
  }
  if constexpr (OP != LIN_WEIGHT_GRAD) {
    if (mx) return dtype == LM_F16 ? run_general<F16, true, OP>(a, st) : run_general<BF16, true, OP>(a, st);
  }
  return dtype == LM_F16 ? run_general<F16, false, OP>(a, st) : run_general<BF16, false, OP>(a, st);
}

extern "C" size_t lm_linear_workspace_size(int64_t T, int64_t N, int64_t K, int32_t experts, int32_t input_dtype) {
  if (T <= 0 || N <= 0 || K <= 0 || experts <= 0 || input_dtype != LM_E2M1) return 0;
  return lin_ws(T, N, K, experts, true).total;
}

extern "C" int lm_linear(const void* x, int64_t ldx, const lm_weight* w, const void* bias, const int32_t* ends, void* y,
                         int64_t T, int32_t dtype, int32_t input_dtype, void* workspace, size_t workspace_bytes,
                         void* stream) {
  int rc;
  if (!w) return fail(LM_EINVAL, "lm_linear requires a weight");
  if ((rc = check_lin(w, T, dtype, ends, w->experts))) return rc;
  const bool mx = w->dtype == LM_E2M1, quant = input_dtype == LM_E2M1;
  if (!quant && input_dtype != dtype) return fail(LM_EUNSUPPORTED, "the product's input dtype is the rows' or LM_E2M1");
  if (quant && !mx) return fail(LM_EUNSUPPORTED, "4-bit inputs need an MXFP4 weight");
  if (T == 0) return LM_OK;
  if (!x || !y) return fail(LM_EINVAL, "row pointers must be non-null");
  if (ldx < w->K) return fail(LM_EINVAL, "row stride below the row length");
  hipStream_t st = (hipStream_t)stream;
  LinArgs a = lin_args(w, ends, T);
  a.a = x;
  a.lda = ldx;
  a.bias = bias;
  a.out = y;
  if (!quant) return run_product<LIN_FORWARD>(a, dtype, mx, st);
  const LinWs ws = lin_ws(T, a.N, a.K, a.experts, ends != nullptr);
  if (!workspace || workspace_bytes < ws.total)
    return fail(LM_EWORKSPACE, "workspace too small: %zu < %zu bytes", workspace ? workspace_bytes : 0, ws.total);
  if (((uintptr_t)workspace & 255) != 0) return fail(LM_EINVAL, "workspace must be 256-byte aligned");
  uint8_t* base = (uint8_t*)workspace;
  a.xq = base;
  a.xs = base + ws.xs;
  a.wsc = base + ws.wsc;
  a.padded = ws.padded;
  {
    TimedLaunch timed("linear_prep", st);
    const int64_t rows = (T + 3) / 4, pieces = (a.experts * ((a.N + 63) / 64) * ((a.K + 255) / 256) + 3) / 4;
    if (rows + pieces > 0x7fffffff) return fail(LM_EUNSUPPORTED, "product too large for one launch");
    const dim3 grid((unsigned)(rows + pieces));
    if (dtype == LM_F16) hipLaunchKernelGGL((k_lin_prep4<F16>), grid, dim3(256), 0, st, a, (int)rows, base, base + ws.xs, base + ws.wsc);
    else hipLaunchKernelGGL((k_lin_prep4<BF16>), grid, dim3(256), 0, st, a, (int)rows, base, base + ws.xs, base + ws.wsc);
    LAUNCH_CHECK();
  }
  return run_mm<LIN_FORWARD, W_Q4>(a, dtype, st);
}

extern "C" int lm_linear_input_grad(const void* dy, int64_t lddy, const lm_weight* w, const int32_t* ends, void* dx,
                                    int64_t T, int32_t dtype, void* stream) {
  int rc;
  if (!w) return fail(LM_EINVAL, "lm_linear_input_grad requires a weight");
  if ((rc = check_lin(w, T, dtype, ends, w->experts))) return rc;
  if (T == 0) return LM_OK;
  if (!dy || !dx) return fail(LM_EINVAL, "row pointers must be non-null");
  if (lddy < w->N) return fail(LM_EINVAL, "row stride below the row length");
  LinArgs a = lin_args(w, ends, T);
  a.a = dy;
  a.lda = lddy;
  a.out = dx;
  return run_product<LIN_INPUT_GRAD>(a, dtype, w->dtype == LM_E2M1, (hipStream_t)stream);
}

extern "C" int lm_linear_weight_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const int32_t* ends,
                                     void* dw, int64_t T, int64_t N, int64_t K, int32_t experts, int32_t dtype,
                                     void* stream) {
  int rc;
  if ((rc = check_lin(nullptr, T, dtype, ends, experts))) return rc;
  if (N <= 0 || K <= 0) return fail(LM_EINVAL, "empty weight gradient");
  if (N >= (1 << 22) || K >= (1 << 22)) return fail(LM_EUNSUPPORTED, "products take rows and columns below 2^22");
  if (!dw || (T > 0 && (!dy || !x))) return fail(LM_EINVAL, "pointers must be non-null");
  if (lddy < N || ldx < K) return fail(LM_EINVAL, "row stride below the row length");
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
  return run_product<LIN_WEIGHT_GRAD>(a, dtype, false, (hipStream_t)stream);
}
