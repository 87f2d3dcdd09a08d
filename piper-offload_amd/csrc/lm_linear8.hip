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
#include "lm_linear8_few.h"
#include "lm_linear_host.h"

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

// Weights whose rows are not whole 16-byte pieces, copied to rows that are.
__global__ __launch_bounds__(256) void k_lin8_align(const uint8_t* src, int64_t rows, int64_t cols, uint8_t* dst, int64_t pitch) {
  const int64_t pieces = pitch >> 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * pieces) return;
  const int64_t r = i / pieces, c = (i - r * pieces) * 16;
  store_b128_guarded((LM_GLOBAL lm_u32x4*)(dst + r * pitch + c), few8_chunk(src + r * cols + c, (int)(cols - c)));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int64_t round16(int64_t x) { return (x + 15) & ~(int64_t)15; }

struct Lin8Plan {
  LinPlan mm;                // tile and splits of k_lin_mm
  bool few;                  // k_lin_few8, else k_lin_mm
  bool copy_x, copy_w;       // rows realigned in the workspace first
  int64_t pitch, lda, ldw;   // of the codes of x, of 16-bit rows, of the weight (bytes)
  size_t codes, scales, x, w, part, total;
};

// As lin_few: a matter of the product's volume.
static bool lin8_few(int64_t T, int64_t N, int64_t K, int64_t E, bool quant) {
  const int64_t rows = (T + E - 1) / E;
  const double volume = (double)T * (double)N * (double)K;
  if (K < 512 && T > 64) return false;
  return rows <= 16 || volume <= 1.1e9 || (quant && T <= 64);
}

static Lin8Plan lin8_plan(int op, int64_t T, int64_t lda, int64_t N, int64_t K, int64_t E, bool quant, bool aligned) {
  Lin8Plan p{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += align256(bytes);
    return o;
  };
  quant = quant && op == LIN_FORWARD;
  const int64_t inner = op == LIN_FORWARD ? K : N;
  p.few = op == LIN_FORWARD && lin8_few(T, N, K, E, quant);
  p.lda = lda;
  p.ldw = K;
  if (quant) {
    p.pitch = round16(K);
    p.codes = take((size_t)T * p.pitch);
    p.scales = take((size_t)T * 4);
  } else {
    p.copy_x = lda >= (1 << 21) || (!p.few && (!aligned || lda % 8 || inner % 8));
    if (p.copy_x) {
      p.lda = round8(inner);
      p.x = take((size_t)T * p.lda * 2);
    }
  }
  if (!p.few) {
    p.copy_w = !aligned || K % 16;
    if (p.copy_w) {
      p.ldw = round16(K);
      p.w = take((size_t)E * N * p.ldw);
    }
    p.mm.len = quant ? p.pitch / 2 : round8(inner);
    p.mm.splits = 1;
    const int64_t J = op == LIN_FORWARD ? N : K;
    lin_tiling(p.mm, op, T, J, p.mm.len, E, !quant, false);
    if (p.mm.splits > 1) p.part = take((size_t)p.mm.splits * T * J * 4);
  }
  p.total = at;
  return p;
}

size_t lin8_workspace(int op, int64_t T, int64_t lda, int64_t N, int64_t K, int64_t E, bool quant, bool aligned) {
  return lin8_plan(op, T, lda, N, K, E, quant, aligned).total;
}

template <int DT, bool Q8, int MF, int CF, int NW, int UN>
static int launch_few8(const LinArgs& a, const uint8_t* codes, int64_t pitch, hipStream_t st) {
  TimedLaunch timed("linear_few", st);
  const int64_t n = lin_tiles<16 * MF>(a.T, a.experts, a.ends != nullptr) * ((a.N + 16 * CF - 1) / (16 * CF));
  if (n > 0x7fffffff) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  hipLaunchKernelGGL((k_lin_few8<DT, Q8, MF, CF, NW, UN>), dim3((unsigned)n), dim3(NW * 64), 0, st, a, codes, pitch);
  LAUNCH_CHECK();
  return LM_OK;
}
template <int DT, bool Q8>
static int run_few8(const LinArgs& a, const uint8_t* codes, int64_t pitch, hipStream_t st) {
  const int64_t rows = (a.T + a.experts - 1) / a.experts, units = (a.K + 127) / 128;
  const int64_t wgs = lin_tiles<16>(a.T, a.experts, a.experts > 1) * ((a.N + 15) / 16);
  if (rows > 32 && wgs > 2048) return launch_few8<DT, Q8, 4, 4, 8, 1>(a, codes, pitch, st);
  if (wgs <= 256) return launch_few8<DT, Q8, 1, 1, 8, 4>(a, codes, pitch, st);
  if (units >= 32) return launch_few8<DT, Q8, 1, 2, 8, 4>(a, codes, pitch, st);
  return launch_few8<DT, Q8, 1, 2, 4, 2>(a, codes, pitch, st);
}

static int lin8_setup(LinArgs& a, const Lin8Plan& p, int op, void* workspace, size_t workspace_bytes, hipStream_t st) {
  if (p.total > 0) {
    if (!workspace || workspace_bytes < p.total)
      return fail(LM_EWORKSPACE, "workspace too small: %zu < %zu bytes", workspace ? workspace_bytes : 0, p.total);
    if (((uintptr_t)workspace & 255) != 0) return fail(LM_EINVAL, "workspace must be 256-byte aligned");
  }
  uint8_t* base = (uint8_t*)workspace;
  TimedLaunch timed("linear_prep", st);
  if (p.copy_x) {
    const int64_t n = (a.T * (p.lda / 8) + 255) / 256;
    if (n > 0x7fffffff) return fail(LM_EUNSUPPORTED, "product too large for one launch");
    hipLaunchKernelGGL(k_lin_align, dim3((unsigned)n), dim3(256), 0, st, (const uint16_t*)a.a, a.lda, a.T, op == LIN_FORWARD ? a.K : a.N,
                       (uint16_t*)(base + p.x), p.lda);
    LAUNCH_CHECK();
    a.a = base + p.x;
    a.lda = p.lda;
  }
  if (p.copy_w) {
    const int64_t rows = a.experts * a.N, n = (rows * (p.ldw / 16) + 255) / 256;
    if (n > 0x7fffffff) return fail(LM_EUNSUPPORTED, "product too large for one launch");
    hipLaunchKernelGGL(k_lin8_align, dim3((unsigned)n), dim3(256), 0, st, (const uint8_t*)a.w, rows, a.K, base + p.w, p.ldw);
    LAUNCH_CHECK();
    a.w = base + p.w;
  }
  a.ldw = p.ldw;
  a.len = p.mm.len;
  a.part = p.mm.splits > 1 ? (float*)(base + p.part) : nullptr;
  return LM_OK;
}

int lin8_forward(LinArgs& a, int dtype, bool quant, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Lin8Plan p = lin8_plan(LIN_FORWARD, a.T, a.lda, a.N, a.K, a.experts, quant, aligned16(a.a) && aligned16(a.w));
  int rc;
  if ((rc = lin8_setup(a, p, LIN_FORWARD, workspace, workspace_bytes, st))) return rc;
  uint8_t* codes = (uint8_t*)workspace + p.codes;
  if (quant) {
    a.row_scale = (const float*)((uint8_t*)workspace + p.scales);
    TimedLaunch timed("linear_prep", st);
    const dim3 grid((unsigned)a.T);
    if (dtype == LM_F16) hipLaunchKernelGGL((k_lin8_rows<F16>), grid, dim3(256), 0, st, a, codes, (float*)a.row_scale, p.pitch);
    else hipLaunchKernelGGL((k_lin8_rows<BF16>), grid, dim3(256), 0, st, a, codes, (float*)a.row_scale, p.pitch);
    LAUNCH_CHECK();
  }
  if (p.few) {
    if (quant) return dtype == LM_F16 ? run_few8<F16, true>(a, codes, p.pitch, st) : run_few8<BF16, true>(a, codes, p.pitch, st);
    return dtype == LM_F16 ? run_few8<F16, false>(a, nullptr, 0, st) : run_few8<BF16, false>(a, nullptr, 0, st);
  }
  if (!quant) return run_mm<LIN_FORWARD, W_I8>(a, p.mm, dtype, st);
  // (in pairs of codes from here on)
  a.a = codes;
  a.lda = p.pitch / 2;
  a.ldw = p.ldw / 2;
  return run_mm<LIN_FORWARD, W_Q8>(a, p.mm, dtype, st);
}

int lin8_input_grad(LinArgs& a, int dtype, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Lin8Plan p = lin8_plan(LIN_INPUT_GRAD, a.T, a.lda, a.N, a.K, a.experts, false, aligned16(a.a) && aligned16(a.w));
  int rc;
  if ((rc = lin8_setup(a, p, LIN_INPUT_GRAD, workspace, workspace_bytes, st))) return rc;
  return run_mm<LIN_INPUT_GRAD, W_I8>(a, p.mm, dtype, st);
}
