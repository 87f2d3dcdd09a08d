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
  // pieces of 64 rows x 256 of K (k_lin_prep4); every group starts on a piece
  const uint8_t* xq;
  const uint8_t* xs;
  const uint8_t* wsc;
  int64_t padded;  // 64-row pieces of xq
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

// ---- groups of rows --------------------------------------------------------
// Ends that fall, are negative or pass T are clamped to what came before and to
// T, so no index leaves the tensors whatever the caller's memory holds.  A wave
// scans 64 groups at a time, one per lane (all lanes active; every wave of a
// workgroup does it for itself).

// lane i: end of group c + i, given the end of group c - 1
DEV int lin_ends64(const LinArgs& a, int c, int before) {
  const int i = c + (int)(threadIdx.x & 63);
  int x = i < a.experts ? a.ends[i] : 0;
  x = x > (int)a.T ? (int)a.T : x;
  x = x < before ? before : x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    if ((int)(threadIdx.x & 63) >= d) x = y > x ? y : x;
  }
  return x;
}
// Rows [b, e) of group g.
DEV void lin_group(const LinArgs& a, int g, int64_t& b, int64_t& e) {
  if (!a.ends) {
    b = 0;
    e = a.T;
    return;
  }
  int before = 0;
  for (int c = 0;; c += 64) {
    const int x = lin_ends64(a, c, before);
    if (g < c + 64) {
      e = __shfl(x, g - c);
      b = g == c ? before : __shfl(x, g - c > 0 ? g - c - 1 : 0);
      break;
    }
    before = __shfl(x, 63);
  }
  b = __builtin_amdgcn_readfirstlane((int)b);
  e = __builtin_amdgcn_readfirstlane((int)e);
}

// Groups are tiled one after the other, BM rows a tile, each from its own first
// row; group `experts` holds the rows of no group.  Finds tile t: its group
// and rows [r0, r1), false past the last tile; t < 0 counts the tiles into g.
// pad: r0 if every group's rows were padded to a multiple of 64.
template <int BM>
DEV bool lin_find(const LinArgs& a, int t, int& g, int64_t& r0, int64_t& r1, int64_t& pad) {
  const int lane = threadIdx.x & 63;
  int before = 0, tiles = 0, pieces = 0;
  for (int c = 0; c <= a.experts; c += 64) {
    int x = lin_ends64(a, c, before);
    if (c + lane >= a.experts) x = (int)a.T;  // the rows of no group, then empty ones
    int b = __shfl_up(x, 1);
    if (lane == 0) b = before;
    const int n = (x - b + BM - 1) / BM, n64 = (x - b + 63) >> 6;
    int sum = n, sum64 = n64;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_up(sum, d), z = __shfl_up(sum64, d);
      if (lane >= d) {
        sum += y;
        sum64 += z;
      }
    }
    const uint64_t hit = __ballot(t >= tiles && t < tiles + sum);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      g = c + l;
      const int first = tiles + __shfl(sum - n, l);
      r0 = __builtin_amdgcn_readfirstlane(__shfl(b, l) + (t - first) * BM);
      r1 = __builtin_amdgcn_readfirstlane(__shfl(x, l));
      pad = __builtin_amdgcn_readfirstlane((pieces + __shfl(sum64 - n64, l)) * 64 + (t - first) * BM);
      g = __builtin_amdgcn_readfirstlane(g);
      return true;
    }
    before = __shfl(x, 63);
    tiles += __shfl(sum, 63);
    pieces += __shfl(sum64, 63);
  }
  g = __builtin_amdgcn_readfirstlane(tiles);
  return false;
}
template <int BM>
DEV bool lin_tile(const LinArgs& a, int64_t t, int& g, int64_t& r0, int64_t& r1) {
  int64_t pad;
  if (a.ends) return lin_find<BM>(a, (int)t, g, r0, r1, pad);
  g = 0;
  r0 = t * BM;
  r1 = a.T;
  return r0 < a.T;
}
// Row t: its group, and its place if every group's rows were padded to 64.
DEV bool lin_row(const LinArgs& a, int t, int& g, int64_t& p) {
  const int lane = threadIdx.x & 63;
  int before = 0, pieces = 0;
  for (int c = 0; c <= a.experts; c += 64) {
    int x = lin_ends64(a, c, before);
    if (c + lane >= a.experts) x = (int)a.T;
    int b = __shfl_up(x, 1);
    if (lane == 0) b = before;
    const int n64 = (x - b + 63) >> 6;
    int sum64 = n64;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int z = __shfl_up(sum64, d);
      if (lane >= d) sum64 += z;
    }
    const uint64_t hit = __ballot(t >= b && t < x);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      g = c + l;
      p = (pieces + __shfl(sum64 - n64, l)) * 64 + t - __shfl(b, l);
      return true;
    }
    before = __shfl(x, 63);
    pieces += __shfl(sum64, 63);
  }
  return false;
}
template <int BM>
DEV int lin_count(const LinArgs& a) {
  int g;
  int64_t r0, r1, pad;
  lin_find<BM>(a, -1, g, r0, r1, pad);
  return g;
}
// at most this many tiles: every group may end in a part of one
template <int BM>
static inline int64_t lin_tiles(int64_t T, int experts, bool grouped) {
  return (T + BM - 1) / BM + (grouped ? experts : 0);
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

template <bool HALF>
DEV v4f32 lin_mfma(lm_u32x4 a, lm_u32x4 b, v4f32 c) {
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8f16, a), __builtin_bit_cast(v8f16, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf16, a), __builtin_bit_cast(v8bf16, b), c, 0, 0, 0);
}
