// lm_linear8.hip -- products with INT8 weights, W[n,k] = s[n] q[n,k]:
//
//   8-bit inputs    r[t] = max_k |x[t,k]| / 127, c[t,k] = x[t,k] / r[t] to the nearest whole number
//                   y[t,n] = r[t] s[n] sum_k c[t,k] q[n,k] (+ bias[n]): whole numbers, exact in 32 bits
//   16-bit inputs   y[t,n] = s[n] sum_k x[t,k] q[n,k] (+ bias[n]): the codes are exact in 16 bits
//   input gradient  dx[t,k] = sum_n dy[t,n] W[n,k] (straight through the rounding of 8-bit inputs)
//
// The products of one weight, or of one weight per group of rows.
#include "lm_impl.h"
#include "lm_linear8.h"

DEV float lin8_scale(const LinArgs& a, int64_t i) {
  return a.scale16 ? bf16_val(((const LM_GLOBAL uint16_t*)a.scale)[i]) : ((const LM_GLOBAL float*)a.scale)[i];
}

// x / r to the nearest whole number, ties to even, as the exact quotient rounds.
// n, from the inverse, is off by one where the quotient lies next to a border; the
// remainder x - n r is exact (one fma: x is a multiple of r's last place), and says so.
DEV float lin8_round(float x, float r, float inv) {
  const float n = __builtin_rintf(x * inv), e = __builtin_fmaf(-n, r, x), d = 2.0f * __builtin_fabsf(e);
  const float to = n + (e < 0.0f ? -1.0f : 1.0f);
  const bool odd = __builtin_rintf(n * 0.5f) * 2.0f != n;
  return d > r || (d == r && odd) ? to : n;
}

// The rows' codes, at a pitch of whole 16-byte pieces that are filled up with zeros,
// and their scales.  A row of zeros has scale 0; one with an infinity or a NaN has
// the scale NaN, so its products are NaN instead of finite numbers.  A workgroup a
// row.  Bound by memory.
template <int DT>
__global__ __launch_bounds__(256) void k_lin8_rows(LinArgs a, uint8_t* codes, float* scales, int64_t pitch) {
  __shared__ uint32_t red[4];
  const int64_t t = blockIdx.x;
  const uint16_t* x = (const uint16_t*)a.a + t * a.lda;
  uint32_t top = 0;
  for (int64_t c = threadIdx.x * 8; c < a.K; c += 2048) {
    const lm_u32x4 w = lin_chunk(x + c, a.K - c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = f2u(val_dt<DT>(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu)) & 0x7fffffffu;
      top = b > top ? b : top;
    }
  }
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)top, m);
    top = o > top ? o : top;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) top = red[i] > top ? red[i] : top;
  const bool bad = top >= 0x7f800000u;
  const float r = bad ? u2f(0x7fc00000u) : u2f(top) / 127.0f;
  if (threadIdx.x == 0) scales[t] = r;
  // (rows below 2^-126 * 127, where the inverse overflows, are scaled up first: exact)
  const float up = r < 0x1p-100f ? 0x1p100f : 1.0f, rr = r * up, inv = bad || r == 0.0f ? 0.0f : 1.0f / rr;
  for (int64_t c = threadIdx.x * 8; c < pitch; c += 2048) {
    const lm_u32x4 w = lin_chunk(x + c, a.K - c);
    uint32_t q[2] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = val_dt<DT>(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu);
      const float n = inv == 0.0f ? 0.0f : __builtin_amdgcn_fmed3f(lin8_round(v * up, rr, inv), -127.0f, 127.0f);
      q[j >> 2] |= ((uint32_t)(int)n & 0xffu) << (8 * (j & 3));
    }
    *(LM_GLOBAL lm_u32x2*)(codes + t * pitch + c) = lm_u32x2{q[0], q[1]};
  }
}

// One output a thread.
template <int DT, int OP, bool QUANT>
__global__ __launch_bounds__(256) void k_lin8(LinArgs a, const int8_t* codes, int64_t pitch) {
  int group;
  int64_t r0, r1;
  if (!lin_tile<16>(a, blockIdx.x, group, r0, r1)) return;
  const int64_t J = OP == LIN_FORWARD ? a.N : a.K, t = r0 + (threadIdx.x >> 4), j = (int64_t)blockIdx.y * 16 + (threadIdx.x & 15);
  if (t >= r1 || j >= J) return;
  float sum = 0.0f;
  if (group < a.experts) {
    const int8_t* w = (const int8_t*)a.w + group * a.N * a.K;
    const uint16_t* x = (const uint16_t*)a.a + t * a.lda;
    const int64_t s0 = group * a.N;
    if constexpr (OP == LIN_INPUT_GRAD) {
      for (int64_t n = 0; n < a.N; ++n) sum += val_dt<DT>(x[n]) * (lin8_scale(a, s0 + n) * (float)w[n * a.K + j]);
    } else if constexpr (QUANT) {
      int s = 0;
      for (int64_t k = 0; k < a.K; ++k) s += (int)codes[t * pitch + k] * (int)w[j * a.K + k];
      sum = (float)s * lin8_scale(a, s0 + j) * a.row_scale[t];  // (in this order no large row overflows on the way)
    } else {
      for (int64_t k = 0; k < a.K; ++k) sum += val_dt<DT>(x[k]) * (float)w[j * a.K + k];
      sum *= lin8_scale(a, s0 + j);
    }
    if (OP == LIN_FORWARD && a.bias) sum += val_dt<DT>(((const uint16_t*)a.bias)[j]);
  }
  ((uint16_t*)a.out)[t * J + j] = bits_dt<DT>(sum);
}

struct Lin8Plan {
  int64_t pitch;
  size_t codes, scales, total;
};
static Lin8Plan lin8_plan(int op, int64_t T, int64_t K, bool quant) {
  Lin8Plan p{};
  if (op == LIN_FORWARD && quant) {
    p.pitch = (K + 15) & ~(int64_t)15;
    p.scales = align256((size_t)T * p.pitch);
    p.total = p.scales + align256((size_t)T * 4);
  }
  return p;
}

size_t lin8_workspace(int op, int64_t T, int64_t, int64_t, int64_t K, int64_t, bool quant, bool) {
  return lin8_plan(op, T, K, quant).total;
}

template <int OP, bool QUANT>
static int launch8(const LinArgs& a, int dtype, const int8_t* codes, int64_t pitch, hipStream_t st) {
  TimedLaunch timed("linear", st);
  const int64_t J = OP == LIN_FORWARD ? a.N : a.K, gj = (J + 15) / 16;
  const int64_t gi = lin_tiles<16>(a.T, a.experts, a.ends != nullptr);
  if (gj > 65535 || gi > 0x7fffffff) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  const dim3 grid((unsigned)gi, (unsigned)gj);
  if (dtype == LM_F16) hipLaunchKernelGGL((k_lin8<F16, OP, QUANT>), grid, dim3(256), 0, st, a, codes, pitch);
  else hipLaunchKernelGGL((k_lin8<BF16, OP, QUANT>), grid, dim3(256), 0, st, a, codes, pitch);
  LAUNCH_CHECK();
  return LM_OK;
}

int lin8_forward(LinArgs& a, int dtype, bool quant, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Lin8Plan p = lin8_plan(LIN_FORWARD, a.T, a.K, quant);
  if (p.total > 0) {
    if (!workspace || workspace_bytes < p.total)
      return fail(LM_EWORKSPACE, "workspace too small: %zu < %zu bytes", workspace ? workspace_bytes : 0, p.total);
    if (((uintptr_t)workspace & 255) != 0) return fail(LM_EINVAL, "workspace must be 256-byte aligned");
  }
  if (!quant) return launch8<LIN_FORWARD, false>(a, dtype, nullptr, 0, st);
  uint8_t* codes = (uint8_t*)workspace + p.codes;
  float* scales = (float*)((uint8_t*)workspace + p.scales);
  {
    TimedLaunch timed("linear_prep", st);
    const dim3 grid((unsigned)a.T);
    if (dtype == LM_F16) hipLaunchKernelGGL((k_lin8_rows<F16>), grid, dim3(256), 0, st, a, codes, scales, p.pitch);
    else hipLaunchKernelGGL((k_lin8_rows<BF16>), grid, dim3(256), 0, st, a, codes, scales, p.pitch);
    LAUNCH_CHECK();
  }
  a.row_scale = scales;
  return launch8<LIN_FORWARD, true>(a, dtype, (const int8_t*)codes, p.pitch, st);
}

int lin8_input_grad(LinArgs& a, int dtype, void*, size_t, hipStream_t st) {
  return launch8<LIN_INPUT_GRAD, false>(a, dtype, nullptr, 0, st);
}
