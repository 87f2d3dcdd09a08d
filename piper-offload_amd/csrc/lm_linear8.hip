// lm_linear8.hip -- products with INT8 weights, W[n,k] = s[n] q[n,k]:
//
//   8-bit inputs    r[t] = max_k |x[t,k]| * 127^-1, c[t,k] = x[t,k] / r[t] to the nearest whole number
//                   y[t,n] = r[t] s[n] sum_k c[t,k] q[n,k] (+ bias[n]): whole numbers, exact in 32 bits
//   16-bit inputs   y[t,n] = s[n] sum_k x[t,k] q[n,k] (+ bias[n]): the codes are exact in 16 bits
//   input gradient  dx[t,k] = sum_n dy[t,n] W[n,k] (straight through the rounding of 8-bit inputs)
//
// The products of one weight, or of one weight per group of rows.
//
// The input gradient rounds s q to 16 bits: s lies along its sum, so the product cannot be
// multiplied by it afterwards, and to round dy s instead is off by as much.  (So does a
// program that decodes the weight to 16 bits first; bf16 outputs are off by 2.3e-3 of their norm,
// 1.7e-3 of it their own rounding.  Both halves of s q would take twice the products.)  fp16 has not
// the range of the scales: there 2^f s q is rounded, f of each weight such that its largest
// scale counts as 128 to 256 (k_lin8_shift), and the sum is multiplied by 2^-f.  Weights
// whose scale is above 2^-21 of that one keep fp16's 11 bits.
//
// Many rows (k_lin_mm): codes times codes are bound by the power that the matrix unit
// may take, 4096 rows of [14336, 4096] 244 to 252 us with the rows' codes, 10 of them (2.0
// POP/s, busy 65% of the cycles; the library's product of 8192^3 reaches 2.2).  Decoded to 16
// bits, 2048 rows of the same 214 to 224 us (1.07 to 1.12 PFLOP/s), input gradient in two
// parts with their join 220 to 245 (the library's bf16 product of 8192^3: 1.33).  Calls in
// graphs on several machines; traced one by one the kernels take up to a tenth longer.
#include "lm_impl.h"
#include "lm_linear8.h"
#include "lm_linear8_few.h"
#include "lm_linear_host.h"

// The rows' codes, at a pitch of whole pieces that are filled up with zeros, and their
// scales: a workgroup a row, whose first 4096 values stay in registers between the two.
// tail: codes of the last piece of 16 at its end, as k_lin8_tail has values.
// The workgroups after those copy weights whose rows are not whole 16-byte pieces to
// rows that are (`aligned`), a wave a row.  Bound by memory: 4096 rows of 4096 10 us
// (50 MB, 5 TB/s).
template <int DT>
__global__ __launch_bounds__(256) void k_lin8_prep(LinArgs a, uint8_t* codes, float* scales, int64_t pitch, int tail, uint8_t* aligned, int64_t ldw) {
  __shared__ uint32_t red[4];
  const int64_t t = blockIdx.x, rows = scales ? a.T : 0;
  if (t >= rows) {
    const int64_t r = (t - rows) * 4 + wave_index();
    if (r >= a.experts * a.N) return;
    const uint8_t* const from = (const uint8_t*)a.w + r * a.K;
    for (int64_t c = (threadIdx.x & 63) * 16; c < ldw; c += 4096) {
      lm_u32x4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = few8_chunk(from, c + i * 1024, a.K);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i * 1024 < ldw) store_b128_guarded((LM_GLOBAL lm_u32x4*)(aligned + r * ldw + c + i * 1024), w[i]);
    }
    return;
  }
  const uint16_t* x = (const uint16_t*)a.a + t * a.lda;
  const int64_t c0 = threadIdx.x * 8;
  const lm_u32x4 w0 = lin_chunk(x + c0, a.K - c0), w1 = lin_chunk(x + c0 + 2048, a.K - c0 - 2048);
  uint32_t top = lin8_top<DT>(w1, lin8_top<DT>(w0, 0));
  for (int64_t c = c0 + 4096; c < a.K; c += 2048) top = lin8_top<DT>(lin_chunk(x + c, a.K - c), top);
  top = lin8_wave_max(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) top = red[i] > top ? red[i] : top;
  const Lin8Row r(top);
  if (threadIdx.x == 0) scales[t] = r.scale;
  LM_GLOBAL uint8_t* const to = (LM_GLOBAL uint8_t*)codes + t * pitch;
  const int64_t last = tail ? a.K & ~(int64_t)15 : pitch;  // codes up to here are in order
  if (c0 < last) *(LM_GLOBAL lm_u32x2*)(to + c0) = r.codes<DT>(w0);
  if (c0 + 2048 < last) *(LM_GLOBAL lm_u32x2*)(to + c0 + 2048) = r.codes<DT>(w1);
  for (int64_t c = c0 + 4096; c < last; c += 2048) *(LM_GLOBAL lm_u32x2*)(to + c) = r.codes<DT>(lin_chunk(x + c, a.K - c));
  if (last + c0 < pitch) {
    lm_u32x4 w = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t i = a.K - 16 + c0 + e;
      if (i >= last && i < a.K) w[e >> 1] |= (uint32_t)((const LM_GLOBAL uint16_t*)x)[i] << (16 * (e & 1));
    }
    *(LM_GLOBAL lm_u32x2*)(to + last + c0) = r.codes<DT>(w);
  }
}

// Rows of 16 bits copied for k_lin_mm, which reads the last 16 codes of a row that is no
// whole number of them in one piece: those elements of x that belong to a code of that
// piece and to none before it, at the piece's end.
__global__ __launch_bounds__(256) void k_lin8_tail(const uint16_t* src, int64_t lds, int64_t rows, int cols, uint16_t* dst, int ldd) {
  const int64_t r = (int64_t)blockIdx.x * 4 + wave_index();
  if (r >= rows) return;
  const uint16_t* const from = src + r * lds;
  for (int c = (threadIdx.x & 63) * 8; c < ldd; c += 512) {
    lm_u32x4 w;
    if (c < ldd - 16) {
      w = lin_chunk(from + c, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = c + e - (ldd - cols);  // of the last 16
        const uint32_t x = i >= ldd - 16 ? ((const LM_GLOBAL uint16_t*)from)[i] : 0u;
        w[e >> 1] = e & 1 ? w[e >> 1] | x << 16 : x;
      }
    }
    store_b128_guarded((LM_GLOBAL lm_u32x4*)(dst + r * ldd + c), w);
  }
}

// The power of two of every weight's scales, from the largest finite one, a workgroup a
// weight.  A launch, and what it takes: a gradient over [4096, 4096] in fp16 16.8 -> 19.2 us
// at one row, with 14336 scales and 2048 rows 260 either way.
__global__ __launch_bounds__(1024) void k_lin8_shift(LinArgs a, int32_t* shift) {
  __shared__ uint32_t red[16];
  const int64_t first = blockIdx.x * a.N;
  uint32_t top = 0;
  for (int64_t i = threadIdx.x; i < a.N; i += 1024) {
    const uint32_t b = f2u(lin_scale8(a, first + i)) & 0x7fffffffu;
    top = b > top && b < 0x7f800000u ? b : top;
  }
  top = lin8_wave_max(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = red[i] > top ? red[i] : top;
  shift[blockIdx.x] = top == 0 ? 0 : 8 - __builtin_amdgcn_frexp_expf(u2f(top));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Rows of codes that are copied for k_lin_mm, x's and a weight's, start on whole 64-byte
// pieces, a stage's loads of a row: the product of 777 x [2001, 2083] 14.2 us, on 16 bytes 16.8.
static int64_t round16(int64_t x) { return (x + 15) & ~(int64_t)15; }
static int64_t round64(int64_t x) { return (x + 63) & ~(int64_t)63; }
// Up to this many rows every workgroup of k_lin_few8 quantises them by itself, while its
// first weights are on their way: one row of [1024, 4096] 6.1 us, after a launch of
// k_lin8_prep 8; four rows of [4096, 4096] 10.9, as much as the two launches, but for the host.
constexpr int64_t LIN8_OWN_ROWS = 4, LIN8_OWN_BYTES = 32768;

struct Lin8Plan {
  LinPlan mm;                // tile and splits of k_lin_mm
  bool few;                  // k_lin_few8, else k_lin_mm
  bool own;                  // k_lin_few8 quantises its rows
  bool copy_x, copy_w;       // rows realigned in the workspace first
  bool tail;                 // and x's last elements as k_lin8_tail (8-bit inputs: k_lin8_prep) has them
  bool raw;                  // 8-bit inputs: codes of the weight at any address
  int64_t pitch, lda, ldw;   // of the codes of x, of 16-bit rows, of the weight (bytes)
  bool half;                 // fp16 input gradient: k_lin8_shift
  size_t codes, codes_bytes, scales, x, w, part, shift, total;
};

// As lin_few: a matter of the product's volume.  Measured in graphs, weights from memory,
// us few / mm.  16-bit inputs: [4096, 4096] at 17 rows 14.3 / 13.8, at 64 rows 14.5 / 17.2, at
// 96 rows 24.8 / 20.0; [1024, 4096] at 200 rows 14.1 / 15.2, at 300 rows 24.7 / 17.2; [256,
// 2048] at 700 rows 8.4 / 12.8; [14336, 4096] at 24 rows 27.1 / 26.3; 8 groups [2752, 9304] at
// 76 rows 77 / 94; 32 groups [2816, 2048] at 512 rows 56 / 55, at 1024 rows 82 / 56.  8-bit:
// [4096, 4096] at 32 rows 12.9 / 15.5, at 64 rows 17.8 / 17.4, at 96 rows 23.0 / 18.4; [14336,
// 4096] at 64 rows 26.7 / 32.6; 8 groups [2752, 9304] at 76 rows 56 / 79; 32 groups [2816,
// 2048] at 1024 rows 85 / 50.  The bounds are those of MXFP4, whose weights have half the
// bytes, and take the slower kernel for some: 65 rows of [4096, 4096] 24.7 / 19.5, 260 of
// [1024, 4096] 24.6 / 16.9; 8-bit 64 rows of [4096, 14336] 51.5 / 31.9, 24 of [14336, 4096]
// 29.3 / 24.2, 64 groups [2048, 1408] at 1024 rows 60 / 45.
static bool lin8_few(int64_t T, int64_t N, int64_t K, int64_t E, bool quant) {
  const int64_t rows = (T + E - 1) / E;
  const double volume = (double)T * (double)N * (double)K;
  if (K < 512 && T > 64) return false;
  return rows <= 16 || volume <= 1.1e9 || (quant && T <= 64);
}

static Lin8Plan lin8_plan(int op, int64_t T, int64_t lda, int64_t N, int64_t K, int64_t E, bool quant, bool aligned, bool half) {
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
  p.own = quant && p.few && T <= LIN8_OWN_ROWS && T * round16(K) <= LIN8_OWN_BYTES;
  if (p.own) {
    p.pitch = round16(K);
  } else if (quant) {
    p.pitch = p.few ? round16(K) : round64(K);
    p.codes_bytes = (size_t)T * p.pitch;
    p.codes = take(p.codes_bytes);
    p.scales = take((size_t)T * 4);
  } else {
    p.copy_x = lda >= (1 << 21) || (!p.few && (!aligned || lda % 8 || inner % 8 || (op == LIN_FORWARD && K % 16)));
    if (p.copy_x) p.lda = round8(inner);
    if (p.copy_x && p.few) p.x = take((size_t)T * p.lda * 2);
  }
  if (!p.few) {
    // Rows of codes may lie anywhere, if there is one piece, or tile, of them, where they go
    // through registers.  Straight to LDS go whole pieces of 16 bytes alone: weights are
    // copied to rows of such, or, while they have few rows of x each, go through registers too
    // (32 groups [6912, 1146] at 1643 rows 111 us, copied 162; 777 rows of [2001, 2083] 30, copied 24).
    const bool off = !aligned || K % 16;
    p.raw = quant && off && K >= 16 && T <= 64 * E;
    p.copy_w = quant ? off && !p.raw : K < (op == LIN_FORWARD ? 16 : 256) && K % 16;
    if (p.copy_w) {
      p.ldw = round64(K);
      p.w = take((size_t)E * N * p.ldw);
    }
    p.tail = op == LIN_FORWARD && !p.copy_w && K % 16;
    p.mm.len = quant ? round16(K) / 2 : p.tail ? round16(K) : round8(inner);
    if (p.tail && !quant) p.lda = p.mm.len;
    if (p.copy_x) p.x = take((size_t)T * p.lda * 2);
    p.mm.splits = 1;
    const int64_t J = op == LIN_FORWARD ? N : K;
    // (codes with the costs of dense products, decoded weights with those of MXFP4.  Tiles and
    // parts forced in turn over 16 shapes: the choice within 6% of the best for 13; 1590 rows of
    // [3200, 3184] 83 / 66 us and 390 of [13696, 4344] 126 / 94, both best as 256 x 256 in two
    // parts, input gradient of 1024 rows of [4096, 4096] 68 / 58 in two parts)
    lin_tiling(p.mm, op, T, J, p.mm.len, E, !quant, false);
    if (p.mm.splits > 1) p.part = take((size_t)p.mm.splits * T * J * 4);
  }
  p.half = op == LIN_INPUT_GRAD && half;
  if (p.half) p.shift = take((size_t)E * 4);
  p.total = at;
  return p;
}

size_t lin8_workspace(int op, int64_t T, int64_t lda, int64_t N, int64_t K, int64_t E, bool quant, bool aligned, bool half) {
  return lin8_plan(op, T, lda, N, K, E, quant, aligned, half).total;
}

template <int DT, bool Q8, bool OWN, int MF, int CF, int NW, int UN>
static int launch_few8(const LinArgs& a, const uint8_t* codes, int64_t pitch, hipStream_t st) {
  TimedLaunch timed("linear_few", st);
  const int64_t n = lin_tiles<16 * MF>(a.T, a.experts, a.ends != nullptr) * ((a.N + 16 * CF - 1) / (16 * CF));
  if (!lin_holds(n, NW * 64)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  const size_t lds = OWN ? (size_t)(a.T * pitch) : 0;
  // (16 fragments have no registers left for the words besides)
  const bool odd = MF == 1 && (((uintptr_t)a.w | (uintptr_t)a.K) & 3 || (!Q8 && ((uintptr_t)a.a | (uintptr_t)(a.lda * 2)) & 3));
  if (odd) hipLaunchKernelGGL((k_lin_few8<DT, Q8, OWN, MF == 1, MF, CF, NW, UN>), dim3((unsigned)n), dim3(NW * 64), lds, st, a, codes, pitch);
  else hipLaunchKernelGGL((k_lin_few8<DT, Q8, OWN, false, MF, CF, NW, UN>), dim3((unsigned)n), dim3(NW * 64), lds, st, a, codes, pitch);
  LAUNCH_CHECK();
  return LM_OK;
}
// Columns of a workgroup, its waves, units in flight, in graphs over weights from
// memory (600 MB of them in turn).  Few workgroups: 16 columns (one row of [4096, 4096] 6.6
// us, with 32 8.2; 8-bit inputs 7.3 and 8.7).  8-bit inputs: 32 columns, one unit (one row of
// [14336, 4096] 15.4 us, four units 17.1; 64 rows of 32 experts [2816, 2048] 31.7, four waves
// with two 33.9; but one row of [8192, 14336] 28.3, 16 columns with four units 26.5).  16-bit
// inputs, twice as many bytes of x for a byte of the weight: 64 columns from 9 rows on (16
// rows of [14336, 4096] 18.6 us, 32 columns 20.6), 32 below (one row 16.6, 64 columns 17.6)
// and where the contraction is long (16 rows of [8192, 14336] 31.2, 64 columns 48.3); very
// many workgroups take four waves (64 rows of 32 experts [2816, 2048] 32.0, eight 34.1).
template <int DT, bool Q8, bool OWN>
static int run_few8(const LinArgs& a, const uint8_t* codes, int64_t pitch, hipStream_t st) {
  const int64_t rows = (a.T + a.experts - 1) / a.experts;
  const int64_t wgs = lin_tiles<16>(a.T, a.experts, a.experts > 1) * ((a.N + 15) / 16);
  if constexpr (!OWN) {
    if (rows > 32 && wgs > 2048) return launch_few8<DT, Q8, OWN, 4, 4, 8, 1>(a, codes, pitch, st);
  }
  if (wgs <= 256) return launch_few8<DT, Q8, OWN, 1, 1, 8, 4>(a, codes, pitch, st);
  if constexpr (Q8) {
    return launch_few8<DT, Q8, OWN, 1, 2, 8, 1>(a, codes, pitch, st);
  } else {
    if (wgs > 2048) return launch_few8<DT, Q8, OWN, 1, 4, 4, 1>(a, codes, pitch, st);
    if (a.T > 8 && a.K < 8192) return launch_few8<DT, Q8, OWN, 1, 4, 8, 1>(a, codes, pitch, st);
    return launch_few8<DT, Q8, OWN, 1, 2, 8, 2>(a, codes, pitch, st);
  }
}

static int lin8_setup(LinArgs& a, const Lin8Plan& p, int op, int dtype, void* workspace, size_t workspace_bytes, hipStream_t st) {
  if (p.total > 0) {
    if (!workspace || workspace_bytes < p.total)
      return fail(LM_EWORKSPACE, "workspace too small: %zu < %zu bytes", workspace ? workspace_bytes : 0, p.total);
    if (((uintptr_t)workspace & 255) != 0) return fail(LM_EINVAL, "workspace must be 256-byte aligned");
  }
  uint8_t* base = (uint8_t*)workspace;
  TimedLaunch timed("linear_prep", st);
  if (p.copy_x) {
    const int64_t n = p.tail ? (a.T + 3) / 4 : (a.T * (p.lda / 8) + 255) / 256;
    if (!lin_holds(n, 256)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
    if (p.tail) hipLaunchKernelGGL(k_lin8_tail, dim3((unsigned)n), dim3(256), 0, st, (const uint16_t*)a.a, a.lda, a.T, (int)a.K, (uint16_t*)(base + p.x), (int)p.lda);
    else hipLaunchKernelGGL(k_lin_align, dim3((unsigned)n), dim3(256), 0, st, (const uint16_t*)a.a, a.lda, a.T, op == LIN_FORWARD ? a.K : a.N,
                       (uint16_t*)(base + p.x), p.lda);
    LAUNCH_CHECK();
    a.a = base + p.x;
    a.lda = p.lda;
  }
  if (p.codes_bytes > 0 || p.copy_w) {
    const int64_t rows = p.codes_bytes > 0 ? a.T : 0, n = rows + (p.copy_w ? (a.experts * a.N + 3) / 4 : 0);
    if (!lin_holds(n, 256)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
    float* const scales = rows ? (float*)(base + p.scales) : nullptr;
    if (dtype == LM_F16) hipLaunchKernelGGL((k_lin8_prep<F16>), dim3((unsigned)n), dim3(256), 0, st, a, base + p.codes, scales, p.pitch, (int)p.tail, base + p.w, p.ldw);
    else hipLaunchKernelGGL((k_lin8_prep<BF16>), dim3((unsigned)n), dim3(256), 0, st, a, base + p.codes, scales, p.pitch, (int)p.tail, base + p.w, p.ldw);
    LAUNCH_CHECK();
    a.row_scale = scales;
    if (p.copy_w) a.w = base + p.w;
  }
  if (p.half) {
    a.shift = (const int32_t*)(base + p.shift);
    hipLaunchKernelGGL(k_lin8_shift, dim3((unsigned)a.experts), dim3(1024), 0, st, a, (int32_t*)(base + p.shift));
    LAUNCH_CHECK();
  }
  a.ldw = p.ldw;
  a.len = p.mm.len;
  a.part = p.mm.splits > 1 ? (float*)(base + p.part) : nullptr;
  return LM_OK;
}

int lin8_forward(LinArgs& a, int dtype, bool quant, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Lin8Plan p = lin8_plan(LIN_FORWARD, a.T, a.lda, a.N, a.K, a.experts, quant, aligned16(a.a) && aligned16(a.w), false);
  int rc;
  if ((rc = lin8_setup(a, p, LIN_FORWARD, dtype, workspace, workspace_bytes, st))) return rc;
  uint8_t* codes = (uint8_t*)workspace + p.codes;
  if (p.few) {
    const bool half = dtype == LM_F16;
    if (p.own) return half ? run_few8<F16, true, true>(a, nullptr, p.pitch, st) : run_few8<BF16, true, true>(a, nullptr, p.pitch, st);
    if (quant) return half ? run_few8<F16, true, false>(a, codes, p.pitch, st) : run_few8<BF16, true, false>(a, codes, p.pitch, st);
    return half ? run_few8<F16, false, false>(a, nullptr, 0, st) : run_few8<BF16, false, false>(a, nullptr, 0, st);
  }
  if (!quant) return run_mm<LIN_FORWARD, W_I8>(a, p.mm, dtype, st);
  // (in pairs of codes from here on)
  a.a = codes;
  a.lda = p.pitch / 2;
  if (p.raw) return run_mm<LIN_FORWARD, W_R8>(a, p.mm, dtype, st);
  a.ldw = p.ldw / 2;
  return run_mm<LIN_FORWARD, W_Q8>(a, p.mm, dtype, st);
}

int lin8_input_grad(LinArgs& a, int dtype, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Lin8Plan p = lin8_plan(LIN_INPUT_GRAD, a.T, a.lda, a.N, a.K, a.experts, false, aligned16(a.a) && aligned16(a.w), dtype == LM_F16);
  int rc;
  if ((rc = lin8_setup(a, p, LIN_INPUT_GRAD, dtype, workspace, workspace_bytes, st))) return rc;
  return run_mm<LIN_INPUT_GRAD, W_I8>(a, p.mm, dtype, st);
}
