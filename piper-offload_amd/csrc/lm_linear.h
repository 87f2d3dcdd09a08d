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
  const uint8_t* xq;  // x quantised: codes [T, K/2], scales [T, K/32]
  const uint8_t* xs;
  const void* w;  // [experts, N, K] dense or [experts, N, K/2] codes
  const uint8_t* scale;
  int64_t scale_stride;  // bytes of one expert's scales
  const void* bias;
  const int32_t* ends;  // [experts] or null: one group of all T rows
  void* out;
  int64_t T, N, K;
  int experts, swizzled;
};

static inline int64_t lin_scale_bytes(int64_t N, int64_t K, int swizzled) {
  return swizzled ? (N + 127) / 128 * ((K + 127) / 128) * 512 : N * (K / 32);
}

// Rows [b, e) of group g.  Ends that fall, are negative or pass T are clamped
// to what came before and to T, so no index leaves the tensors whatever the
// caller's memory holds.
DEV void lin_group(const LinArgs& a, int g, int64_t& b, int64_t& e) {
  if (!a.ends) {
    b = 0;
    e = a.T;
    return;
  }
  b = 0;
  e = 0;
  for (int i = 0; i <= g; ++i) {
    const int64_t x = a.ends[i];
    b = e;
    e = x < e ? e : (x > a.T ? a.T : x);
  }
}

// Tile t of BM rows: its group and rows [r0, r1).  Groups are tiled one after
// the other, each from its own first row; group `experts` holds the rows of no
// group.  False past the last tile.
template <int BM>
DEV bool lin_tile(const LinArgs& a, int64_t t, int& g, int64_t& r0, int64_t& r1) {
  if (!a.ends) {
    g = 0;
    r0 = t * BM;
    r1 = a.T;
    return r0 < a.T;
  }
  int64_t e = 0;
  for (g = 0; g <= a.experts; ++g) {
    const int64_t b = e;
    if (g < a.experts) {
      const int64_t x = a.ends[g];
      e = x < e ? e : (x > a.T ? a.T : x);
    } else {
      e = a.T;
    }
    const int64_t n = (e - b + BM - 1) / BM;
    if (t < n) {
      r0 = b + t * BM;
      r1 = e;
      return true;
    }
    t -= n;
  }
  return false;
}
// at most this many tiles: every group may end in a part of one
template <int BM>
static inline int64_t lin_tiles(int64_t T, int experts, bool grouped) {
  return (T + BM - 1) / BM + (grouped ? experts : 0);
}

// 32 values -> 16 bytes of e2m1 codes and the e8m0 scale.  A block with an
// infinity or a NaN gets the NaN scale, so the rows it feeds come out NaN
// instead of a finite number.
DEV uint32_t lin_quant32(const float (&v)[32], uint32_t (&w)[4]) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const uint32_t b = f2u(v[j]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  float inv;
  const uint32_t s = top >= 0x7f800000u ? 255u : mx_scale(u2f(top), MX_FLOOR, 2, 6.0f, 1, inv);
  if (s == 255u) inv = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float lo = __builtin_amdgcn_fmed3f(v[8 * k + 2 * t] * inv, -6.0f, 6.0f);
      const float hi = __builtin_amdgcn_fmed3f(v[8 * k + 2 * t + 1] * inv, -6.0f, 6.0f);
      w[k] |= e2m1_pack2(lo, hi) << (8 * t);
    }
  }
  return s;
}

template <bool HALF>
DEV v4f32 lin_mfma(lm_u32x4 a, lm_u32x4 b, v4f32 c) {
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8f16, a), __builtin_bit_cast(v8f16, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf16, a), __builtin_bit_cast(v8bf16, b), c, 0, 0, 0);
}
