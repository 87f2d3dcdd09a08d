// lm_linear_few.h -- products with little reuse: few rows per weight, or few
// columns.
//
// Such a product is bound by the bytes of the larger operand, not by the matrix
// unit, so there are no LDS tiles: operands go from memory straight into MFMA
// registers.  A workgroup owns 16 MF rows x 16 CF columns and its NW waves split
// the contraction, 128 a unit, and add their sums up through LDS in a fixed
// order.  With 16 columns a workgroup even a 1024-row weight spreads over 64 CUs;
// every wave has UN units of loads in flight at once.
// MXFP4 [14336, 4096] at one row: 10.0 us, 3.1 TB/s of codes and scales with the
// launch's ends (5.0 us for [1024, 4096], which is latency alone); 64 groups
// [2048, 1408] at 100 rows with 4-bit inputs 18 us, 4.1 TB/s.
//
// Both operands are read in whole runs of a row: access j of a unit gives lane
// group g (lane >> 4) 16 bytes, chunk 4j + g of 8 values, and that is what MFMA
// step j contracts.  16 bytes of MXFP4 codes are 4 chunks, 4g..4g+3; a 4 x 4
// transpose of dwords between the lane groups (4 lane swaps) brings them to
// the same order.  With 4-bit inputs both sides are codes and the scaled MFMA
// takes them as they lie; the rows are quantised by a launch of their own
// (k_lin_prep4): every workgroup needs all of them, and quantising them in each
// costs more than the launch ([14336, 4096] at 1 row: 34 us in one launch).
//
// All loads are buffer loads: 32-bit offsets, and what lies past the end of the
// contraction is sent out of the resource and comes back as zeros, without a
// branch around each load.
#pragma once
#include <type_traits>

#include "lm_linear.h"

// out[j] in lane group g = in[g] in lane group j
DEV void lin_transpose4(lm_u32x4& d) {
  const auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
  const auto p = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto q = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  d = lm_u32x4{p[0], p[1], q[0], q[1]};
}
DEV lm_u32x4 few_load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(lm_u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}

// EDGE: dense rows whose length is no multiple of 8
template <int DT, int W, int MF, int CF, int NW, int UN, bool EDGE>
__global__ __launch_bounds__(NW * 64) void k_lin_few(LinArgs a) {
  constexpr bool HALF = DT == F16, Q4 = W == W_Q4, MX = W == W_MX;
  constexpr int COLS = CF * 16, ROWS = MF * 16, PITCH = COLS + 4;
  constexpr int XL = Q4 ? 1 : 4, WL = W == W_DENSE ? 4 : 1;  // 16-byte loads a unit
  constexpr int AC = MF * CF <= 2 ? 2 : 1;                   // accumulators in turn: the MFMAs of a fragment depend on each other
  __shared__ __attribute__((aligned(16))) float red[NW * ROWS * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, wave = wave_index();
  // Row tiles first, and each XCD a contiguous part: the row tiles of a group read
  // the same columns of its weight out of one L2.
  const uint32_t gn = (uint32_t)((a.N + COLS - 1) / COLS), u = (uint32_t)xcd_unit(blockIdx.x, gridDim.x);
  const uint32_t tiles = gridDim.x / gn;
  const int64_t n0 = (int64_t)(u / tiles) * COLS;
  int group;
  int64_t r0, r1;
  if (!lin_tile<ROWS>(a, u % tiles, group, r0, r1)) return;
  const bool some = group < a.experts;
  v4f32 acc[AC][MF][CF] = {};
  if (some) {
    const int nb = (int)(a.K >> 5), nb4 = (nb + 3) & ~3;
    const int64_t ldx = Q4 ? a.K >> 1 : a.lda * 2, ldw = W == W_DENSE ? a.K * 2 : a.K >> 1;  // bytes
    const int rows = (int)(r1 - r0 < ROWS ? r1 - r0 : ROWS), cols = (int)(a.N - n0 < COLS ? a.N - n0 : COLS);
    const uint8_t* xp = (Q4 ? a.xq : (const uint8_t*)a.a) + r0 * ldx;
    const uint8_t* wp = (const uint8_t*)a.w + (group * a.N + n0) * ldw;
    const __amdgpu_buffer_rsrc_t rx = lin_rsrc(xp, (rows - 1) * ldx + (Q4 ? a.K >> 1 : a.K * 2));
    const __amdgpu_buffer_rsrc_t rw = lin_rsrc(wp, cols * ldw);
    const __amdgpu_buffer_rsrc_t rxs = lin_rsrc(Q4 ? a.xs + r0 * nb4 : nullptr, Q4 ? rows * nb4 : 0);
    const uint8_t* sp = a.scale + group * a.scale_stride + (a.swizzled ? blocked_offset(n0 & ~(int64_t)127, 0, nb, true) : n0 * nb);
    uint32_t xo[MF], xso[MF], wo[CF];
    const uint8_t* so[CF];
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const int t = m * 16 + (lane & 15);
      xo[m] = (uint32_t)((t < rows ? t : rows - 1) * ldx) + 16 * g;
      xso[m] = (uint32_t)((t < rows ? t : rows - 1) * nb4);
    }
#pragma unroll
    for (int c = 0; c < CF; ++c) {
      const int n = c * 16 + (lane & 15) < cols ? c * 16 + (lane & 15) : cols - 1;
      wo[c] = (uint32_t)(n * ldw) + 16 * g;
      const int q = (int)(n0 & 127) + n;
      so[c] = sp + (a.swizzled ? (q & 31) * 16 + (q >> 5) * 4 : n * nb);
    }
    // UN units from u0; TAIL: some of them may pass the end
    auto body = [&](int u0, auto tail) {
      constexpr bool TAIL = decltype(tail)::value;
      lm_u32x4 xv[UN][MF][XL], wv[UN][CF][WL];
      uint32_t sv[UN][CF], xs[UN][MF];
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int u = u0 + i;
#pragma unroll
        for (int c = 0; c < CF; ++c) {
#pragma unroll
          for (int j = 0; j < WL; ++j) {
            if constexpr (EDGE) {
              wv[i][c][j] = lin_chunk((const uint16_t*)(wp + wo[c]) + u * 128 + 32 * j, a.K - u * 128 - 32 * j - 8 * g);
            } else {
              const uint32_t o = wo[c] + u * (W == W_DENSE ? 256 : 64) + 64 * j;
              const bool in = W == W_DENSE ? u * 128 + 32 * j + 8 * g < a.K : u * 4 + g < nb;
              wv[i][c][j] = few_load16(rw, TAIL && !in ? LIN_OUT : o);
            }
          }
          if constexpr (W != W_DENSE) {  // scales of blocks 4u .. 4u + 3, zeros past the last
            if (!TAIL && !a.swizzled) {  // (the units' words are side by side: one load)
              if (i == 0) {
                if constexpr (UN == 4) {
                  const lm_u32x4 w = *(const LM_GLOBAL lm_u32x4_any*)(so[c] + u * 4);
#pragma unroll
                  for (int k = 0; k < UN; ++k) sv[k][c] = w[k];
                } else if constexpr (UN == 2) {
                  const lm_u32x2 w = *(const LM_GLOBAL lm_u32x2_any*)(so[c] + u * 4);
                  sv[0][c] = w[0];
                  sv[1][c] = w[1];
                } else {
                  sv[0][c] = *(const LM_GLOBAL lm_u32_any*)(so[c] + u * 4);
                }
              }
              continue;
            }
            const uint8_t* s = so[c] + u * (a.swizzled ? 512 : 4);
            const int have = nb - u * 4;
            if (!TAIL || have >= 4) {
              sv[i][c] = *(const LM_GLOBAL lm_u32_any*)s;
            } else {
              sv[i][c] = 0;
#pragma unroll
              for (int b = 0; b < 3; ++b)
                if (b < have) sv[i][c] |= (uint32_t)((const LM_GLOBAL uint8_t*)s)[b] << (8 * b);
            }
          }
        }
#pragma unroll
        for (int m = 0; m < MF; ++m) {
#pragma unroll
          for (int j = 0; j < XL; ++j) {
            if constexpr (EDGE) {
              xv[i][m][j] = lin_chunk((const uint16_t*)(xp + xo[m]) + u * 128 + 32 * j, a.K - u * 128 - 32 * j - 8 * g);
            } else {
              const uint32_t o = xo[m] + u * (Q4 ? 64 : 256) + 64 * j;
              const bool in = Q4 ? u * 4 + g < nb : u * 128 + 32 * j + 8 * g < a.K;
              xv[i][m][j] = few_load16(rx, TAIL && !in ? LIN_OUT : o);
            }
          }
          if constexpr (Q4)
            xs[i][m] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rxs, (int)(TAIL && u * 4 >= nb ? LIN_OUT : xso[m] + u * 4), 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        if constexpr (Q4) {
#pragma unroll
          for (int c = 0; c < CF; ++c)
#pragma unroll
            for (int m = 0; m < MF; ++m)
              acc[i % AC][m][c] = lin_mfma4(wv[i][c][0], xv[i][m][0], acc[i % AC][m][c], sv[i][c] >> (8 * g), xs[i][m] >> (8 * g), 0, 0);
        } else {
#pragma unroll
          for (int c = 0; c < CF; ++c) {
            if constexpr (MX) lin_transpose4(wv[i][c][0]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              lm_u32x4 f;
              if constexpr (MX) f = lin_decode8<HALF>(wv[i][c][0][j], lin_e8m0(sv[i][c], j));
              else f = wv[i][c][j];
#pragma unroll
              for (int m = 0; m < MF; ++m) acc[j % AC][m][c] = lin_mfma<HALF>(f, xv[i][m][j], acc[j % AC][m][c]);
            }
          }
        }
      }
    };
    const int units = (int)((a.K + 127) >> 7), whole = (int)(a.K >> 7);
    int u0 = wave * UN;
    for (; u0 + UN <= whole; u0 += NW * UN) body(u0, std::false_type{});
    if (u0 < units) body(u0, std::true_type{});
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
      for (int c = 0; c < CF; ++c) {
        v4f32 v = acc[0][m][c];
        if constexpr (AC == 2) v += acc[1][m][c];
        *(v4f32*)(red + ((wave * ROWS) + m * 16 + (lane & 15)) * PITCH + c * 16 + 4 * g) = v;
      }
  }
  __syncthreads();
  for (int i = tid; i < ROWS * COLS; i += NW * 64) {
    const int m = i / COLS, c = i % COLS;
    const int64_t n = n0 + c;
    if (r0 + m >= r1 || n >= a.N) continue;
    float s = 0.0f;
    if (some) {
#pragma unroll
      for (int k = 0; k < NW; ++k) s += red[(k * ROWS + m) * PITCH + c];
      if (a.bias) s += val_dt<DT>(((const LM_GLOBAL uint16_t*)a.bias)[n]);
    }
    ((LM_GLOBAL uint16_t*)a.out)[(r0 + m) * a.N + n] = bits_dt<DT>(s);
  }
}
