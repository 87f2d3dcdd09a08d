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
// x quantised to MXFP4: blocks of 32 along K, scale 2^(floor(log2 max) - 2)
// ---------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void k_lin_quant(const uint16_t* x, int64_t ldx, int64_t T, int64_t K, uint8_t* q,
                                                   uint8_t* s) {
  const int64_t nb = K >> 5, total = T * nb;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / nb, b = i - t * nb;
    const uint16_t* p = x + t * ldx + b * 32;
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = val_dt<DT>(p[j]);
    uint32_t w[4];
    s[i] = (uint8_t)lin_quant32(v, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) ((uint32_t*)(q + i * 16))[j] = w[j];
  }
}

// ---------------------------------------------------------------------------
// the general product: any sizes, strides and alignment, 64 x 64 tiles
// ---------------------------------------------------------------------------
template <int DT, bool MX, bool QUANT>
struct LinOps {
  static constexpr bool HALF = DT == F16 && !QUANT;  // operands in fp16; quantised ones are exact in bf16
  DEV static uint16_t bits(float v) { return HALF ? f16_bits(v) : bf16_bits(v); }
  DEV static uint16_t act(const LinArgs& a, int64_t m, int64_t c) {
    if constexpr (QUANT) {
      const uint32_t code = a.xq[m * (a.K >> 1) + (c >> 1)] >> (4 * (c & 1));
      return bits(e2m1_value(code) * e8m0_value(a.xs[m * (a.K >> 5) + (c >> 5)]));
    } else {
      return ((const uint16_t*)a.a)[m * a.lda + c];
    }
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

template <int DT, bool MX, bool QUANT, int OP>
__global__ __launch_bounds__(256) void k_lin_general(LinArgs a) {
  using O = LinOps<DT, MX, QUANT>;
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

struct LinWs {
  size_t xq, xs, total;
};
static LinWs lin_ws(int64_t T, int64_t K, bool quant) {
  LinWs w{0, 0, 0};
  if (quant) {
    w.xs = align256((size_t)T * (size_t)(K / 2));
    w.total = w.xs + align256((size_t)T * (size_t)(K / 32));
  }
  return w;
}

template <int DT, bool MX, bool QUANT, int OP>
static int run_general(const LinArgs& a, hipStream_t st) {
  TimedLaunch timed("linear", st);
  const int64_t J = OP == LIN_FORWARD ? a.N : a.K;
  const int64_t gx = (J + 63) / 64;
  const int64_t gy = OP == LIN_WEIGHT_GRAD ? (a.N + 63) / 64 : lin_tiles<64>(a.T, a.experts, a.ends != nullptr);
  if (gx > 0x7fffffff || gy > 65535) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  hipLaunchKernelGGL((k_lin_general<DT, MX, QUANT, OP>), dim3((unsigned)gx, (unsigned)gy, OP == LIN_WEIGHT_GRAD ? a.experts : 1),
                     dim3(256), 0, st, a);
  LAUNCH_CHECK();
  return LM_OK;
}
// Whole 16-byte pieces along every row that is read, offsets inside a tile below
// 2^31, fewer tiles than a grid holds.
static bool mm_ok(const LinArgs& a, int op, bool mx) {
  const int64_t len = op == LIN_FORWARD ? a.K : a.N;
  if (a.lda % 8 || ((uintptr_t)a.a & 15) || a.lda >= (1 << 22) || a.K >= (1 << 22) || a.N >= (1 << 22)) return false;
  if (op == LIN_WEIGHT_GRAD) return a.ldb % 8 == 0 && ((uintptr_t)a.b & 15) == 0 && a.ldb < (1 << 22);
  if (len % 8) return false;
  return mx || (a.K % 8 == 0 && ((uintptr_t)a.w & 15) == 0);
}

template <int DT, int OP, bool MX, int B, int WM, int WN>
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
template <int OP, bool MX>
static int run_mm(const LinArgs& a, int dtype, hipStream_t st) {
  const int64_t J = OP == LIN_FORWARD ? a.N : a.K, I = OP == LIN_WEIGHT_GRAD ? a.N : a.T;
  const int64_t big = I / 256 * ((J + 255) / 256) * (OP == LIN_WEIGHT_GRAD ? a.experts : 1);
  const bool wide = big >= 192 && (OP == LIN_WEIGHT_GRAD || a.T / a.experts >= 256);
  if (dtype == LM_F16)
    return wide ? launch_mm<F16, OP, MX, 256, 2, 4>(a, st) : launch_mm<F16, OP, MX, 128, 2, 2>(a, st);
  return wide ? launch_mm<BF16, OP, MX, 256, 2, 4>(a, st) : launch_mm<BF16, OP, MX, 128, 2, 2>(a, st);
}

template <int OP>
static int run_product(const LinArgs& a, int dtype, bool mx, bool quant, hipStream_t st) {
  if (!quant && mm_ok(a, OP, mx)) {
    if constexpr (OP != LIN_WEIGHT_GRAD) {
      if (mx) return run_mm<OP, true>(a, dtype, st);
    }
    return run_mm<OP, false>(a, dtype, st);
  }
  if constexpr (OP == LIN_FORWARD) {
    if (quant) return dtype == LM_F16 ? run_general<F16, true, true, OP>(a, st) : run_general<BF16, true, true, OP>(a, st);
  }
  if constexpr (OP != LIN_WEIGHT_GRAD) {
    if (mx) return dtype == LM_F16 ? run_general<F16, true, false, OP>(a, st) : run_general<BF16, true, false, OP>(a, st);
  }
  return dtype == LM_F16 ? run_general<F16, false, false, OP>(a, st) : run_general<BF16, false, false, OP>(a, st);
}

extern "C" size_t lm_linear_workspace_size(int64_t T, int64_t N, int64_t K, int32_t experts, int32_t input_dtype) {
  (void)N;
  (void)experts;
  if (T <= 0 || K <= 0) return 0;
  return lin_ws(T, K, input_dtype == LM_E2M1).total;
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
  if (quant) {
    const LinWs ws = lin_ws(T, a.K, true);
    if (!workspace || workspace_bytes < ws.total)
      return fail(LM_EWORKSPACE, "workspace too small: %zu < %zu bytes", workspace ? workspace_bytes : 0, ws.total);
    if (((uintptr_t)workspace & 255) != 0) return fail(LM_EINVAL, "workspace must be 256-byte aligned");
    uint8_t* q = (uint8_t*)workspace + ws.xq;
    uint8_t* s = (uint8_t*)workspace + ws.xs;
    a.xq = q;
    a.xs = s;
    const int64_t nb = (T * (a.K / 32) + 255) / 256;
    const dim3 grid((unsigned)(nb < 65536 ? nb : 65536));
    if (dtype == LM_F16) hipLaunchKernelGGL((k_lin_quant<F16>), grid, dim3(256), 0, st, (const uint16_t*)x, ldx, T, a.K, q, s);
    else hipLaunchKernelGGL((k_lin_quant<BF16>), grid, dim3(256), 0, st, (const uint16_t*)x, ldx, T, a.K, q, s);
    LAUNCH_CHECK();
  }
  return run_product<LIN_FORWARD>(a, dtype, mx, quant, st);
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
  return run_product<LIN_INPUT_GRAD>(a, dtype, w->dtype == LM_E2M1, false, (hipStream_t)stream);
}

extern "C" int lm_linear_weight_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const int32_t* ends,
                                     void* dw, int64_t T, int64_t N, int64_t K, int32_t experts, int32_t dtype,
                                     void* stream) {
  int rc;
  if ((rc = check_lin(nullptr, T, dtype, ends, experts))) return rc;
  if (N <= 0 || K <= 0) return fail(LM_EINVAL, "empty weight gradient");
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
  return run_product<LIN_WEIGHT_GRAD>(a, dtype, false, false, (hipStream_t)stream);
}
