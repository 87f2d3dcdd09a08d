// lm_linear8_few.h -- products of few rows with INT8 weights.
//
// Bound by the bytes of the weight.  As k_lin_few: no LDS tiles, operands straight
// from memory into MFMA registers; a workgroup owns 16 MF rows x 16 CF columns, its
// NW waves split the contraction, 128 codes a unit, and add their sums up through
// LDS in a fixed order; every wave has UN units of loads in flight.
//
// Lane group g (lane >> 4) reads 16 codes of a row at 64 h + 16 g, h = 0, 1.  With
// 8-bit inputs (Q8) both sides are read so and one instruction contracts the 64 of
// an h.  With 16-bit inputs the 16 codes are decoded (exactly) into two operands of
// 8, steps (h, 0) and (h, 1), and x is read in the same order: lane group g has
// elements 64 h + 16 g + 8 c at step (h, c).
//
// From memory, with the launch: one row of [14336, 4096] in 16 bits 16.6 us (3.5 TB/s; from
// the last-level cache in part, three such weights in turn, 12.4), quantised 15.4; 100 rows
// of 64 experts [2048, 1408], quantised 28.8 (4.8 TB/s for the experts that have rows); one
// row of [1024, 4096] 6.4.
#pragma once
#include <type_traits>

#include "lm_linear.h"

DEV lm_u32x4 few8_load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(lm_u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}
DEV uint32_t few8_load4(__amdgpu_buffer_rsrc_t r, uint32_t off) { return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0); }
// bytes s .. s + 15 (s < 4) of v and e after it
DEV lm_u32x4 few8_align(lm_u32x4 v, uint32_t e, uint32_t s) {
  return lm_u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], s), __builtin_amdgcn_alignbyte(v[2], v[1], s), __builtin_amdgcn_alignbyte(v[3], v[2], s),
                  __builtin_amdgcn_alignbyte(e, v[3], s)};
}
// 16 bytes without the first n (1 .. 15), zeros after them
DEV lm_u32x4 few8_drop(lm_u32x4 v, int n) {
  if (n & 4) v = lm_u32x4{v[1], v[2], v[3], 0};
  if (n & 8) v = lm_u32x4{v[2], v[3], 0, 0};
  return lm_u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], n & 3), __builtin_amdgcn_alignbyte(v[2], v[1], n & 3),
                  __builtin_amdgcn_alignbyte(v[3], v[2], n & 3), __builtin_amdgcn_alignbyte(0, v[3], n & 3)};
}
// Codes k .. k + 15 of a row of K at any address, zeros past its end.  A part of 16 comes
// from the row's last 16 (one load; byte after byte the ends of rows took longer than
// all the rest: 117 rows of 8 groups [896, 1021] 16.8 us, [896, 1024] 6.0 in the same run; like
// this, weights from memory, 10.9 and 9.4).
DEV lm_u32x4 few8_chunk(const uint8_t* row, int64_t k, int64_t K) {
  const int64_t left = K - k;
  lm_u32x4 v = {};
  if (left > 0) {
    if (K >= 16) {
      v = *(const LM_GLOBAL lm_u32x4_any*)(row + (left < 16 ? K - 16 : k));
      if (left < 16) v = few8_drop(v, 16 - (int)left);
    } else {
      uint64_t lo = 0, hi = 0;
      for (int b = 0; b < left; ++b) {
        const uint64_t c = ((const LM_GLOBAL uint8_t*)row)[k + b];
        if (b < 8) lo |= c << (8 * b);
        else hi |= c << (8 * b - 64);
      }
      v = lm_u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
  }
  return v;
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

// The largest magnitude (as its bits) of 8 values, and of a wave
template <int DT>
DEV uint32_t lin8_top(lm_u32x4 w, uint32_t top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = f2u(val_dt<DT>(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu)) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  return top;
}
DEV uint32_t lin8_wave_max(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane(lin_scan_max((int)x), 63); }
// A row, from its largest magnitude: its scale (times 1 / 127, as torch divides by a
// number on the GPU: a program that quantises by itself gets the same codes), and codes of its values.  A row of
// zeros has scale 0; one with an infinity or a NaN has the scale NaN, so its products
// are NaN instead of finite numbers.
struct Lin8Row {
  float scale, up, to, inv;
  DEV Lin8Row(uint32_t top) {
    const bool bad = top >= 0x7f800000u;
    scale = bad ? u2f(0x7fc00000u) : u2f(top) * (1.0f / 127.0f);
    // (a scale below 2^-100, whose inverse may overflow, is scaled up first: exact)
    up = scale < 0x1p-100f ? 0x1p100f : 1.0f;
    to = scale * up;
    inv = bad || scale == 0.0f ? 0.0f : 1.0f / to;
  }
  // v / r lies within 2^-17 of v inv here (|v / r| <= 127, inv is off by 2^-24 of it), so
  // its rounding is that of v / r unless that is near a half: then a wave asks lin8_round.
  // (Added to 1.5 2^23 a number is rounded, and its low byte is the code.)
  template <int DT>
  DEV lm_u32x2 codes(lm_u32x4 w) const {
    constexpr float M = 12582912.0f;
    float v[8], t[8], off = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = val_dt<DT>(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu);
    if (up != 1.0f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= up;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      t[j] = __builtin_fmaf(v[j], inv, M);
      off = __builtin_fmaxf(off, __builtin_fabsf(__builtin_fmaf(v[j], inv, M - t[j])));
    }
    if (__ballot(off > 0.5f - 0x1p-16f)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = M + (inv == 0.0f ? 0.0f : __builtin_amdgcn_fmed3f(lin8_round(v[j], to, inv), -127.0f, 127.0f));
    }
    uint32_t q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo = __builtin_amdgcn_perm(f2u(t[4 * h + 1]), f2u(t[4 * h]), 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(f2u(t[4 * h + 3]), f2u(t[4 * h + 2]), 0x0c0c0400u);
      q[h] = lo | hi << 16;
    }
    return lm_u32x2{q[0], q[1]};
  }
};

// OWN: x is not quantised yet.  Its few rows are, into LDS, by every workgroup.
// ODD: rows of codes, or of x in 16 bits, that do not start on whole words.  16 bytes at
// such an address take twice as long to load (one row of [14336, 4090] 24.5 us, [14336,
// 4092] 15.2 in the same run), so the five words that hold them are loaded instead, and
// shifted (weights from memory: 20.7 and 19.1); a piece whose fifth word would pass its row
// is left to the tail.
template <int DT, bool Q8, bool OWN, bool ODD, int MF, int CF, int NW, int UN>
__global__ __launch_bounds__(NW * 64) void k_lin_few8(LinArgs a, const uint8_t* codes, int64_t pitch) {
  constexpr bool HALF = DT == F16;
  constexpr int COLS = CF * 16, ROWS = MF * 16, PITCH = COLS + 4;
  constexpr int XL = Q8 ? 2 : 4;            // 16-byte loads of x a unit
  constexpr int AC = MF * CF <= 2 ? 2 : 1;  // accumulators in turn: the MFMAs of a fragment depend on each other
  static_assert(!OWN || (Q8 && MF == 1), "rows of its own: a few, with 8-bit inputs");
  __shared__ __attribute__((aligned(16))) uint32_t red[NW * ROWS * PITCH];
  __shared__ uint32_t tops[OWN ? 4 * NW : 1];
  __shared__ float scales[OWN ? 4 : 1];
  extern __shared__ __attribute__((aligned(16))) uint8_t mine[];  // OWN: codes of the rows
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, wave = wave_index();
  // (row tiles first, each XCD a contiguous part: as k_lin_few)
  const uint32_t gn = (uint32_t)((a.N + COLS - 1) / COLS), u = (uint32_t)xcd_unit(blockIdx.x, gridDim.x);
  const uint32_t tiles = gridDim.x / gn;
  const int64_t n0 = (int64_t)(u / tiles) * COLS;
  int group;
  int64_t r0, r1;
  if (!lin_tile<ROWS>(a, u % tiles, group, r0, r1)) return;
  const bool some = group < a.experts;
  v4f32 acc[AC][MF][CF] = {};
  if (some) {
    const int K = (int)a.K;
    const int64_t ldx = Q8 ? pitch : a.lda * 2;  // bytes
    const int rows = (int)(r1 - r0 < ROWS ? r1 - r0 : ROWS), cols = (int)(a.N - n0 < COLS ? a.N - n0 : COLS);
    const uint8_t* xp = OWN ? nullptr : (Q8 ? codes : (const uint8_t*)a.a) + r0 * ldx;
    const uint8_t* wp = (const uint8_t*)a.w + (group * a.N + n0) * a.K;
    constexpr bool ODDX = ODD && !Q8;
    const uint32_t wm = ODD ? (uint32_t)(uintptr_t)wp & 3u : 0u, xm = ODDX ? (uint32_t)(uintptr_t)xp & 3u : 0u;
    const __amdgpu_buffer_rsrc_t rx = lin_rsrc(xp - xm, OWN ? 0 : (rows - 1) * ldx + (Q8 ? pitch : a.K * 2) + xm);
    const __amdgpu_buffer_rsrc_t rw = lin_rsrc(wp - wm, cols * a.K + wm);
    uint32_t xo[MF], wo[CF];
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const int t = m * 16 + (lane & 15);
      xo[m] = (uint32_t)((t < rows ? t : rows - 1) * ldx) + (Q8 ? 16 : 32) * g;
    }
#pragma unroll
    for (int c = 0; c < CF; ++c) {
      const int n = c * 16 + (lane & 15) < cols ? c * 16 + (lane & 15) : cols - 1;
      wo[c] = (uint32_t)(n * a.K) + 16 * g;
    }
    // UN units from u0; TAIL: some of them may pass the end
    lm_u32x4 wv[UN][CF][2];
    uint32_t we[ODD ? UN : 1][ODD ? CF : 1][2];
    auto weights = [&](int u0, auto tail) {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int k0 = (u0 + i) * 128;
#pragma unroll
        for (int c = 0; c < CF; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (decltype(tail)::value) wv[i][c][h] = few8_chunk(wp + (wo[c] - 16 * g), k0 + 64 * h + 16 * g, K);
            else wv[i][c][h] = few8_load16(rw, (ODD ? (wo[c] + wm) & ~3u : wo[c]) + k0 + 64 * h);
            if constexpr (ODD && !decltype(tail)::value) we[i][c][h] = few8_load4(rw, ((wo[c] + wm) & ~3u) + k0 + 64 * h + 16);
          }
      }
    };
    auto body = [&](int u0, auto tail) {
      constexpr bool TAIL = decltype(tail)::value;
      lm_u32x4 xv[UN][MF][XL];
      uint32_t xe[ODDX ? UN : 1][ODDX ? MF : 1][XL];
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int k0 = (u0 + i) * 128;
#pragma unroll
        for (int m = 0; m < MF; ++m)
#pragma unroll
          for (int j = 0; j < XL; ++j) {
            if constexpr (OWN) {
              const int k = k0 + 64 * j + 16 * g;
              xv[i][m][j] = lm_u32x4{};
              if (!TAIL || k < K) xv[i][m][j] = *(const lm_u32x4*)(mine + xo[m] + k0 + 64 * j);
            } else if constexpr (Q8) {
              xv[i][m][j] = few8_load16(rx, TAIL && k0 + 64 * j + 16 * g >= K ? LIN_OUT : xo[m] + k0 + 64 * j);
            } else {
              const int e = k0 + 64 * (j >> 1) + 8 * (j & 1);  // (+ 16 g)
              if constexpr (TAIL) xv[i][m][j] = lin_chunk((const uint16_t*)(xp + xo[m]) + e, K - e - 16 * g);
              else xv[i][m][j] = few8_load16(rx, (ODDX ? (xo[m] + xm) & ~3u : xo[m]) + 2 * e);
              if constexpr (ODDX && !TAIL) xe[i][m][j] = few8_load4(rx, ((xo[m] + xm) & ~3u) + 2 * e + 16);
            }
          }
      }
      if constexpr (ODDX && !TAIL) {
#pragma unroll
        for (int i = 0; i < UN; ++i)
#pragma unroll
          for (int m = 0; m < MF; ++m)
#pragma unroll
            for (int j = 0; j < XL; ++j) xv[i][m][j] = few8_align(xv[i][m][j], xe[i][m][j], (xo[m] + xm) & 3u);
      }
#pragma unroll
      for (int i = 0; i < UN; ++i)
#pragma unroll
        for (int c = 0; c < CF; ++c) {
          if constexpr (ODD && !TAIL) {
#pragma unroll
            for (int h = 0; h < 2; ++h) wv[i][c][h] = few8_align(wv[i][c][h], we[i][c][h], (wo[c] + wm) & 3u);
          }
          if constexpr (Q8) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int m = 0; m < MF; ++m) acc[h % AC][m][c] = lin_mfma8(wv[i][c][h], xv[i][m][h], acc[h % AC][m][c]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const lm_u32x4 w = wv[i][c][j >> 1];
              const lm_u32x4 f = lin_decode8i<HALF, false>(j & 1 ? w[2] : w[0], j & 1 ? w[3] : w[1], 1.0f);
#pragma unroll
              for (int m = 0; m < MF; ++m) acc[j % AC][m][c] = lin_mfma<HALF>(f, xv[i][m][j], acc[j % AC][m][c]);
            }
          }
        }
    };
    const int units = (K + 127) >> 7, whole = (ODD ? K - 4 : K) >> 7;
    int u0 = wave * UN;
    if constexpr (OWN) {
      // The rows' first pieces, then the first weights (loads come back in order), and
      // while those are on their way the codes.  Barriers that wait for LDS alone.
      const uint16_t* x = (const uint16_t*)a.a + r0 * a.lda;
      const int c0 = tid * 8;
      lm_u32x4 first[4];
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (m < rows) first[m] = lin_chunk(x + m * a.lda + c0, K - c0);
      const bool ahead = u0 + UN <= whole;
      if (ahead) weights(u0, std::false_type{});
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (m >= rows) break;
        uint32_t top = lin8_top<DT>(first[m], 0);
        for (int c = c0 + NW * 512; c < K; c += NW * 512) top = lin8_top<DT>(lin_chunk(x + m * a.lda + c, K - c), top);
        top = lin8_wave_max(top);
        if (lane == 0) tops[m * NW + wave] = top;
      }
      lin_wait<63>();
      lin_barrier();
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (m >= rows) break;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) top = tops[m * NW + i] > top ? tops[m * NW + i] : top;
        const Lin8Row r(top);
        if (tid == 0) scales[m] = r.scale;
        if (c0 < pitch) *(lm_u32x2*)(mine + m * pitch + c0) = r.codes<DT>(first[m]);
        for (int c = c0 + NW * 512; c < pitch; c += NW * 512) *(lm_u32x2*)(mine + m * pitch + c) = r.codes<DT>(lin_chunk(x + m * a.lda + c, K - c));
      }
      lin_wait<63>();
      lin_barrier();
      if (ahead) {
        body(u0, std::false_type{});
        u0 += NW * UN;
      }
    }
    for (; u0 + UN <= whole; u0 += NW * UN) {
      weights(u0, std::false_type{});
      body(u0, std::false_type{});
    }
    if (u0 < units) {
      weights(u0, std::true_type{});
      body(u0, std::true_type{});
    }
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
      for (int c = 0; c < CF; ++c) {
        lm_u32x4 v = __builtin_bit_cast(lm_u32x4, acc[0][m][c]);
        if constexpr (AC == 2) {
          if constexpr (Q8) v += __builtin_bit_cast(lm_u32x4, acc[1][m][c]);
          else v = __builtin_bit_cast(lm_u32x4, acc[0][m][c] + acc[1][m][c]);
        }
        *(lm_u32x4*)(red + ((wave * ROWS) + m * 16 + (lane & 15)) * PITCH + c * 16 + 4 * g) = v;
      }
  }
  __syncthreads();
  for (int i = tid; i < ROWS * COLS; i += NW * 64) {
    const int m = i / COLS, c = i % COLS;
    const int64_t n = n0 + c;
    if (r0 + m >= r1 || n >= a.N) continue;
    float s = 0.0f;
    if (some) {
      if constexpr (Q8) {
        uint32_t sum = 0;
#pragma unroll
        for (int k = 0; k < NW; ++k) sum += red[(k * ROWS + m) * PITCH + c];
        // (in this order no large row overflows on the way)
        s = (float)(int)sum * lin_scale8(a, group * a.N + n) * (OWN ? scales[OWN ? m : 0] : a.row_scale[r0 + m]);
      } else {
#pragma unroll
        for (int k = 0; k < NW; ++k) s += u2f(red[(k * ROWS + m) * PITCH + c]);
        s *= lin_scale8(a, group * a.N + n);
      }
      if (a.bias) s += val_dt<DT>(((const LM_GLOBAL uint16_t*)a.bias)[n]);
    }
    ((LM_GLOBAL uint16_t*)a.out)[(r0 + m) * a.N + n] = bits_dt<DT>(s);
  }
}
