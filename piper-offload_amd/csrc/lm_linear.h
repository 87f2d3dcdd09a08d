// lm_linear.h -- what the product kernels share: arguments, groups of rows,
// MXFP4 values and the in-lane quantisation of activations.
#pragma once
#include "lm_impl.h"

enum : int { LIN_FORWARD = 0, LIN_INPUT_GRAD = 1, LIN_WEIGHT_GRAD = 2 };

struct LinArgs {
  const void* a;  // x, or dy in the gradients: [T, lda]
  int64_t lda;
  const void* b;  // x in the weight gradient: [T, ldb]
  int64_t ldb;
  // 4-bit inputs: codes [64 padded, K/2], scales and the weight's scales packed in
  // pieces of 64 rows x 128 of K, 256 bytes (k_lin_prep4); every group starts on a piece
  const uint8_t* xq;
  const uint8_t* xs;
  const uint8_t* wsc;
  int64_t padded;  // 64-row pieces of xq
  int64_t ldw;     // row stride of a dense w
  int64_t len;     // contraction (with zeros up to whole 16-byte pieces)
  int rounds;      // 256 x 256 tiles: whole rounds in one launch, the rest in another (lin_rounds)
  float* part;     // split contraction: fp32 sums [splits, rows, columns], or null
  const void* w;  // [experts, N, K] dense or [experts, N, K/2] codes
  const uint8_t* scale;
  int64_t scale_stride;  // bytes of one expert's scales
  // INT8 weights: `scale` has one number a row, fp32 or bf16 (scale16); 8-bit inputs: one fp32 number a row of x
  const float* row_scale;
  int scale16;
  const int32_t* shift;  // fp16 input gradient of INT8 weights: one a group, its weights count as 2^shift of themselves (k_lin8_shift)
  const void* bias;
  const int32_t* ends;  // [experts] or null: one group of all T rows
  void* out;
  int64_t T, N, K;
  int experts, swizzled;
};

static inline int64_t lin_scale_bytes(int64_t N, int64_t K, int swizzled) {
  return swizzled ? (N + 127) / 128 * ((K + 127) / 128) * 512 : N * (K / 32);
}

constexpr int64_t LIN_SPAN = 0x7fffffff;
constexpr uint32_t LIN_OUT = 0x80000000u;  // an offset past any resource

// a buffer resource over `bytes` bytes: offsets past them (any offset from 2^31
// on) read zeros
DEV __amdgpu_buffer_rsrc_t lin_rsrc(const void* p, int64_t bytes) {
  const uint32_t n = bytes < 0 ? 0u : (bytes > LIN_SPAN ? (uint32_t)LIN_SPAN : (uint32_t)bytes);
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, n, 0x00027000);
}

// a barrier of the workgroup that waits for no memory by itself
DEV void lin_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}
// wait until at most N vector-memory operations and no LDS operation are left
template <int N>
DEV void lin_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// 8 values from p, of which the first `left` exist (any alignment)
DEV lm_u32x4 lin_chunk(const uint16_t* p, int64_t left) {
  lm_u32x4 v = {};
  if (left >= 8) {
    v = *(const LM_GLOBAL lm_u32x4_any*)p;
  } else if (left > 0) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < left) v[e >> 1] |= (uint32_t)((const LM_GLOBAL uint16_t*)p)[e] << (16 * (e & 1));
  }
  return v;
}
typedef uint32_t lm_u32_any __attribute__((aligned(1)));
typedef uint32_t lm_u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// ---- groups of rows --------------------------------------------------------
// Ends that fall, are negative or pass T are clamped to what came before and to
// T, so no index leaves the tensors whatever the caller's memory holds.  A wave
// scans 64 groups at a time, one per lane (all lanes active; every wave of a
// workgroup does it for itself).

// inclusive scans over the wave by DPP (shifts inside rows of 16, then the last
// lane of a row or of half the wave to the rows after it): every workgroup of a
// grouped product starts with them, and lane shuffles through LDS took as long
// as its loads
template <int CTRL, int ROWS>
DEV int lin_dpp(int old, int x) {
  return __builtin_amdgcn_update_dpp(old, x, CTRL, ROWS, 0xf, false);
}
DEV int lin_scan_add(int x) {
  x += lin_dpp<0x111, 0xf>(0, x);
  x += lin_dpp<0x112, 0xf>(0, x);
  x += lin_dpp<0x114, 0xf>(0, x);
  x += lin_dpp<0x118, 0xf>(0, x);
  x += lin_dpp<0x142, 0xa>(0, x);
  x += lin_dpp<0x143, 0xc>(0, x);
  return x;
}
DEV int lin_max(int a, int b) { return a > b ? a : b; }
DEV int lin_scan_max(int x) {  // x >= 0
  x = lin_max(x, lin_dpp<0x111, 0xf>(0, x));
  x = lin_max(x, lin_dpp<0x112, 0xf>(0, x));
  x = lin_max(x, lin_dpp<0x114, 0xf>(0, x));
  x = lin_max(x, lin_dpp<0x118, 0xf>(0, x));
  x = lin_max(x, lin_dpp<0x142, 0xa>(0, x));
  x = lin_max(x, lin_dpp<0x143, 0xc>(0, x));
  return x;
}

// Groups c .. c + 63, one per lane: rows [b, e); `before` is the end of group
// c - 1 and becomes that of group c + 63.  Group `experts` holds the rows of no
// group, those after it nothing.
DEV void lin_groups64(const LinArgs& a, int c, int& before, int& b, int& e) {
  const int i = c + (int)(threadIdx.x & 63), T = (int)a.T;
  int x = T;
  if (i < a.experts) {
    x = ((const LM_GLOBAL int32_t*)a.ends)[i];
    x = x > T ? T : lin_max(x, 0);
  }
  e = lin_scan_max(lin_max(x, before));
  b = __builtin_amdgcn_update_dpp(before, e, 0x138, 0xf, 0xf, false);  // wave_shr:1, lane 0 keeps `before`
  before = __builtin_amdgcn_readlane(e, 63);
}
// Rows [b, e) of group g.
DEV void lin_group(const LinArgs& a, int g, int64_t& b, int64_t& e) {
  b = 0;
  e = a.T;
  if (!a.ends) return;
  int before = 0, lb = 0, le = 0;
  for (int c = 0; c <= g; c += 64) lin_groups64(a, c, before, lb, le);
  b = __builtin_amdgcn_readlane(lb, g & 63);
  e = __builtin_amdgcn_readlane(le, g & 63);
}

// Groups are tiled one after the other, BM rows a tile, each from its own first
// row.  Finds tile t: its group and rows [r0, r1), false past the last tile;
// t < 0 counts the tiles into g.  pad: r0 if every group's rows were padded to a
// multiple of 64.
DEV bool lin_find(const LinArgs& a, int BM, int t, int& g, int64_t& r0, int64_t& r1, int64_t& pad) {
  int before = 0, tiles = 0, pieces = 0;
  for (int c = 0; c <= a.experts; c += 64) {
    int b, e;
    lin_groups64(a, c, before, b, e);
    const int n = (int)((uint32_t)(e - b + BM - 1) / (uint32_t)BM), n64 = (e - b + 63) >> 6;
    const int sum = lin_scan_add(n), sum64 = lin_scan_add(n64);
    const uint64_t hit = __ballot(t >= tiles && t < tiles + sum);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      g = c + l;
      const int first = tiles + __builtin_amdgcn_readlane(sum - n, l), in = (t - first) * BM;
      r0 = __builtin_amdgcn_readlane(b, l) + in;
      r1 = __builtin_amdgcn_readlane(e, l);
      pad = (pieces + __builtin_amdgcn_readlane(sum64 - n64, l)) * (int64_t)64 + in;
      return true;
    }
    tiles += __builtin_amdgcn_readlane(sum, 63);
    pieces += __builtin_amdgcn_readlane(sum64, 63);
  }
  g = tiles;
  return false;
}
// Row t: its group, and its place if every group's rows were padded to 64.
DEV void lin_row(const LinArgs& a, int t, int& g, int64_t& p) {
  int before = 0, pieces = 0;
  for (int c = 0; c <= a.experts; c += 64) {
    int b, e;
    lin_groups64(a, c, before, b, e);
    const int n64 = (e - b + 63) >> 6, sum64 = lin_scan_add(n64);
    const uint64_t hit = __ballot(t >= b && t < e);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      g = c + l;
      p = (pieces + __builtin_amdgcn_readlane(sum64 - n64, l)) * (int64_t)64 + t - __builtin_amdgcn_readlane(b, l);
      return;
    }
    pieces += __builtin_amdgcn_readlane(sum64, 63);
  }
}
template <int BM>
DEV bool lin_tile(const LinArgs& a, int64_t t, int& g, int64_t& r0, int64_t& r1) {
  int64_t pad;
  if (a.ends) return lin_find(a, BM, (int)t, g, r0, r1, pad);
  g = 0;
  r0 = t * BM;
  r1 = a.T;
  return r0 < a.T;
}
DEV int lin_count(const LinArgs& a, int BM) {
  int g;
  int64_t r0, r1, pad;
  lin_find(a, BM, -1, g, r0, r1, pad);
  return g;
}
// at most this many tiles: of all groups with rows (the rows of none are one more
// group, but there are no more groups than rows) but one may end in a part of one
template <int BM>
static inline int64_t lin_tiles(int64_t T, int experts, bool grouped) {
  return (T + BM - 1) / BM + (!grouped || T < 1 ? 0 : experts < T - 1 ? experts : T - 1);
}

// The e8m0 scale of a block whose largest magnitude has these bits, and its
// inverse.  A block with an infinity or a NaN gets the NaN scale, so the rows it
// feeds come out NaN instead of a finite number.
DEV uint32_t lin_scale4(uint32_t top, float& inv) {
  if (top >= 0x7f800000u) {
    inv = 0.0f;
    return 255u;
  }
  return mx_scale(u2f(top), MX_FLOOR, 2, 6.0f, 1, inv);
}
DEV uint32_t lin_codes8(const float (&v)[8], float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float lo = __builtin_amdgcn_fmed3f(v[2 * t] * inv, -6.0f, 6.0f);
    const float hi = __builtin_amdgcn_fmed3f(v[2 * t + 1] * inv, -6.0f, 6.0f);
    w |= e2m1_pack2(lo, hi) << (8 * t);
  }
  return w;
}

// 8 values, the quarter that four neighbouring lanes hold of a block each: their
// codes and (in all four lanes) the block's scale
template <int DT>
DEV uint32_t lin_quant8(lm_u32x4 w, uint32_t& s) {
  float v[8];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = val_dt<DT>(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu);
    const uint32_t b = f2u(v[j]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)top, (int)top, 0xB1, 0xf, 0xf, false);  // lane xor 1
  top = o > top ? o : top;
  o = (uint32_t)__builtin_amdgcn_update_dpp((int)top, (int)top, 0x4E, 0xf, 0xf, false);  // lane xor 2
  top = o > top ? o : top;
  float inv;
  s = lin_scale4(top, inv);
  return lin_codes8(v, inv);
}

template <bool HALF>
DEV v4f32 lin_mfma(lm_u32x4 a, lm_u32x4 b, v4f32 c) {
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8f16, a), __builtin_bit_cast(v8f16, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf16, a), __builtin_bit_cast(v8bf16, b), c, 0, 0, 0);
}

// Byte b of a word of e8m0 scales, as the conversion below takes it: it reads the
// exponent field alone (0 is 2^-127, 255 NaN), whatever sign and mantissa are.
DEV float lin_e8m0(uint32_t word, int b) {
  return u2f(b == 3 ? word >> 1 : word << (23 - 8 * b));
}
// 8 codes -> 8 values of 16 bits.  Exact in bf16.  fp16 rows take fp16 products, so
// the values are rounded to fp16: exact from 2^-23 to 49152, infinite above.
template <bool HALF>
DEV lm_u32x4 lin_decode8(uint32_t codes, float scale) {
  lm_u32x4 v;
  if constexpr (HALF) {
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3));
  } else {
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  }
  return v;
}

// W_Q8: rows and weight are INT8 codes (W_R8: the weight's rows at any address); W_I8: INT8 weight, rows of 16 bits
enum : int { W_DENSE = 0, W_MX = 1, W_Q4 = 2, W_Q8 = 3, W_I8 = 4, W_R8 = 5 };

// the scale of row i of an INT8 weight
DEV float lin_scale8(const LinArgs& a, int64_t i) {
  return a.scale16 ? bf16_val(((const LM_GLOBAL uint16_t*)a.scale)[i]) : ((const LM_GLOBAL float*)a.scale)[i];
}
// 8 INT8 codes -> 8 values of 16 bits, times s or (exact) as they are
template <bool HALF, bool SCALED>
DEV lm_u32x4 lin_decode8i(uint32_t lo, uint32_t hi, float s) {
  lm_u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? lo : hi;
    float a = (float)(int8_t)(w >> (16 * (i & 1))), b = (float)(int8_t)(w >> (16 * (i & 1) + 8));
    if constexpr (SCALED) {
      a *= s;
      b *= s;
    }
    v[i] = HALF ? (uint32_t)f16_bits(a) | (uint32_t)f16_bits(b) << 16 : pack_bf16x2(a, b);
  }
  return v;
}
typedef int lin_i32x4 __attribute__((ext_vector_type(4)));
// 64 steps of whole numbers; the sums' bits lie in a v4f32
DEV v4f32 lin_mfma8(lm_u32x4 a, lm_u32x4 b, v4f32 c) {
  return __builtin_bit_cast(v4f32, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(lin_i32x4, a), __builtin_bit_cast(lin_i32x4, b),
                                                                        __builtin_bit_cast(lin_i32x4, c), 0, 0, 0));
}

// byte FA of sa and byte FB of sb are the operands' scales
template <int FA, int FB>
DEV v4f32 lin_mfma4_(lm_u32x4 a, lm_u32x4 b, v4f32 c, uint32_t sa, uint32_t sb) {
  typedef int v8i32 __attribute__((ext_vector_type(8)));
  const v8i32 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, FA, (int)sa, FB, (int)sb);
}
template <int FA>
DEV v4f32 lin_mfma4_(lm_u32x4 a, lm_u32x4 b, v4f32 c, uint32_t sa, uint32_t sb, int fb) {
  switch (fb) {
    case 0: return lin_mfma4_<FA, 0>(a, b, c, sa, sb);
    case 1: return lin_mfma4_<FA, 1>(a, b, c, sa, sb);
    case 2: return lin_mfma4_<FA, 2>(a, b, c, sa, sb);
    default: return lin_mfma4_<FA, 3>(a, b, c, sa, sb);
  }
}
// (fa, fb known at compile time once the callers' loops are unrolled)
DEV v4f32 lin_mfma4(lm_u32x4 a, lm_u32x4 b, v4f32 c, uint32_t sa, uint32_t sb, int fa, int fb) {
  switch (fa) {
    case 0: return lin_mfma4_<0>(a, b, c, sa, sb, fb);
    case 1: return lin_mfma4_<1>(a, b, c, sa, sb, fb);
    case 2: return lin_mfma4_<2>(a, b, c, sa, sb, fb);
    default: return lin_mfma4_<3>(a, b, c, sa, sb, fb);
  }
}
