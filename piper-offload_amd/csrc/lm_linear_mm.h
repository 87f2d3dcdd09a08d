// lm_linear_mm.h -- products of many rows: LDS-tiled MFMA kernels.
//
// An output tile of BM rows x BN columns per workgroup, the contraction in
// tiles of 64, two LDS buffers: while the waves multiply tile k out of one, the
// loads of tile k + 1 are on their way into the other (buffer loads straight
// to LDS, no registers in between).  One barrier a tile.
//
// Operands are named by the output index they carry: I (rows) and J
// (columns).  Their tiles lie in LDS as
//   KC16  contraction contiguous in memory: a slot of 128 bytes per I/J index,
//         its eight 16-byte chunks rotated by XOR with slot & 7, so that the
//         16 lanes that read one chunk of 16 slots hit all banks
//   KS16  contraction strided (the index contiguous): a row per contraction
//         step; read transposed (ds_read_b64_tr_b16); chunks XORed with
//         4 (row & 3) for the same reason
//   KC4   MXFP4 codes as they are stored, 32 bytes per slot, decoded to 16 bits
//         after the read (v_cvt_scalef32_pk: exact products in bf16)
//   KS4   MXFP4 with the contraction strided: every code of a run of 32 shares a
//         scale but the 8 codes of an MFMA lane do not, so these are decoded on
//         their way into LDS and then are KS16
// Q4: both operands MXFP4 (x quantised beforehand), multiplied as they are by the
// scaled MFMA, 256 codes a tile, so a slot is 128 bytes here too.  Its scales
// come packed by k_lin_prep4: per 64 slots and tile 512 bytes, which hold for
// lane (r, g) the blocks 2g and 2g + 1 of slots r, r + 16, r + 32, r + 48 side by
// side: one 8-byte read gives the scales of four fragments and both steps.
// The MFMA's first operand is J, so a lane's accumulators are consecutive output
// columns; the columns of a pair of 16-column fragments are interleaved in
// fours, which makes them 8 in a row: one 16-byte store.
#pragma once
#include "lm_linear.h"

enum : int { KC16, KS16, KC4, KS4 };

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) lm_u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) lm_u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

// 16 bytes per lane to LDS at base + 16 lane; past the resource's end: zeros
DEV void lin_dma(__amdgpu_buffer_rsrc_t r, lds_u8* base, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)base, 16, (int)off, 0, 0, 0);
}

// Slot of a J tile -> column: pairs of fragments of 16 interleaved in fours
DEV int lin_jcol(int slot) { return (slot & ~31) + 8 * ((slot & 15) >> 2) + (slot & 3) + 4 * ((slot >> 4) & 1); }

// The tile of this workgroup: group, first row, end of the group's rows, number of
// the column tile.  Tiles of up to 8 row tiles x all columns, row tiles
// first, are neighbours; each XCD takes a contiguous part of them, so its L2
// holds the weight tiles that several row tiles share.
struct LinTile {
  int group;
  int64_t r0, r1, j0;
  int64_t pad;  // the first row among the rows padded to 64 a group
};
template <int BM, int BN>
DEV bool lin_pick(const LinArgs& a, int64_t jend, LinTile& t) {
  const int gn = (int)((jend + BN - 1) / BN);
  int tiles;
  if (!a.ends) tiles = (int)((a.T + BM - 1) / BM);
  else tiles = lin_count<BM>(a);
  const uint32_t total = (uint32_t)tiles * (uint32_t)gn;
  if (blockIdx.x >= total) return false;
  const uint32_t u = xcd_unit(blockIdx.x, total);
  constexpr uint32_t GM = 8;
  const uint32_t band = u / (GM * gn), in = u - band * GM * gn;
  const uint32_t left = (uint32_t)tiles - band * GM, h = left < GM ? left : GM;
  const uint32_t tm = band * GM + in % h, tn = in / h;
  t.j0 = (int64_t)tn * BN;
  if (!a.ends) {
    t.group = 0;
    t.pad = t.r0 = (int64_t)tm * BM;
    t.r1 = a.T;
    return true;
  }
  return lin_find<BM>(a, (int)tm, t.group, t.r0, t.r1, t.pad);
}

template <int DT, int OP, int W, int BM, int BN, int WM, int WN>
struct MmTraits {
  static constexpr bool Q4 = W == W_Q4, MX = W == W_MX;
  static constexpr int CT = Q4 ? 256 : 64;                        // contraction of a tile
  static constexpr int IS = Q4 ? BM * 8 : 16, JS = Q4 ? BN * 8 : 16;  // bytes of the scales of a tile
  static constexpr int NW = WM * WN, NT = NW * 64;
  static constexpr int IK = OP == LIN_WEIGHT_GRAD ? KS16 : KC16;
  static constexpr int JK = OP == LIN_FORWARD ? (MX ? KC4 : KC16) : (OP == LIN_INPUT_GRAD && MX ? KS4 : KS16);
  static constexpr int FI = BM / WM / 16, FJ = BN / WN / 16;
  static constexpr int IB = BM * 128, JB = JK == KC4 ? BN * 32 : BN * 128;  // bytes of a tile
  static constexpr int IL = IB / 1024 / NW, JL = JB / 1024 / NW;            // loads per wave
  static_assert(IL * 1024 * NW == IB && JL * 1024 * NW == JB, "tiles are whole loads of all waves");
  static_assert(JK != KS4 || NT * 32 == 64 * BN, "a run of 32 codes per thread");
  // chunk c of contraction 8-groups that lane group g takes in MFMA step s: with
  // KC4 a lane reads the codes of both steps at once, with Q4 their scales, so they
  // are neighbours
  DEV static int chunk(int s, int g) { return JK == KC4 || Q4 ? 2 * g + s : 4 * s + g; }
};

// per-lane byte offsets of the DMA loads of one operand tile
template <int KIND, int B, int L, int NW, bool PERM>
DEV void mm_offsets(uint32_t (&off)[L], int wave, int lane, int64_t ld) {
#pragma unroll
  for (int n = 0; n < L; ++n) {
    const int piece = (n * NW + wave) * 64 + lane;  // 16-byte piece of the tile
    if constexpr (KIND == KC16) {
      const int slot = piece >> 3, c = (piece & 7) ^ (slot & 7);
      off[n] = (uint32_t)((PERM ? lin_jcol(slot) : slot) * ld * 2) + c * 16;
    } else if constexpr (KIND == KC4) {
      const int slot = piece >> 1;
      off[n] = (uint32_t)(lin_jcol(slot) * (ld >> 1)) + (piece & 1) * 16;
    } else {  // KS16
      const int row = piece / (B / 8), c = (piece % (B / 8)) ^ ((row & 3) << 2);
      off[n] = (uint32_t)(row * ld * 2) + c * 16;
    }
  }
}

template <int KIND, int B>
DEV lm_u32x4 mm_frag(const lds_u8* t, int slot0, int f, int lane, int s, int c) {
  if constexpr (KIND == KC16) {
    const int slot = slot0 + f * 16 + (lane & 15);
    return *(const lds_u32x4*)(t + slot * 128 + ((c ^ (slot & 7)) << 4));
  } else {
    return lm_u32x4{};
  }
}
// 8 contraction steps x this lane's index, read transposed: two loads of 4 steps
// each.  Lane p of 16 points at 4 indices of row p >> 2.
template <int B, bool PERM>
DEV lm_u32x4 mm_frag_tr(const lds_u8* t, int col0, int f, int lane, int s) {
  const int p = lane & 15, g = lane >> 4, q = p & 3;
  const int row = 32 * s + 8 * g + (p >> 2);
  const int col = col0 + (PERM ? (f >> 1) * 32 + 8 * q + 4 * (f & 1) : f * 16 + 4 * q);
  const int at = row * (B * 2) + ((((col >> 3) ^ ((row & 3) << 2)) << 4) | ((col & 4) << 1));
  const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(t + at));
  const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(t + at + 4 * (B * 2)));  // row + 4: same XOR
  return lm_u32x4{__builtin_bit_cast(lm_u32x2, lo)[0], __builtin_bit_cast(lm_u32x2, lo)[1],
                  __builtin_bit_cast(lm_u32x2, hi)[0], __builtin_bit_cast(lm_u32x2, hi)[1]};
}

template <int DT, int OP, int W, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_lin_mm(LinArgs a) {
  using P = MmTraits<DT, OP, W, BM, BN, WM, WN>;
  constexpr bool HALF = DT == F16, Q4 = P::Q4, MX = P::MX;
  constexpr int CT = P::CT;
  constexpr int FI = P::FI, FJ = P::FJ;
  __shared__ __attribute__((aligned(1024))) uint8_t si0[P::IB], si1[P::IB], sj0[P::JB], sj1[P::JB];
  __shared__ __attribute__((aligned(1024))) uint8_t sis0[P::IS], sis1[P::IS], sjs0[P::JS], sjs1[P::JS];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave / WN, wj = wave % WN;
  const int64_t jend = OP == LIN_FORWARD ? a.N : a.K;
  LinTile t;
  int64_t len;  // of the contraction
  const uint8_t *ip, *jp;
  int64_t ibytes, jbytes, istep, jstep;  // bytes of the resources, and per tile of 64
  int64_t lda = a.lda, ldb;
  if constexpr (OP == LIN_WEIGHT_GRAD) {
    const int gm = (int)((a.N + BM - 1) / BM);
    t.group = blockIdx.y;
    t.r0 = (int64_t)(blockIdx.x % gm) * BM;
    t.r1 = a.N;
    t.j0 = (int64_t)(blockIdx.x / gm) * BN;
    int64_t b, e;
    lin_group(a, t.group, b, e);
    len = e - b;
    ldb = a.ldb;
    ip = (const uint8_t*)a.a + (b * lda + t.r0) * 2;
    jp = (const uint8_t*)a.b + (b * ldb + t.j0) * 2;
    // (whole pieces of 16 bytes: what a piece holds past the row's end goes to columns that are not stored)
    ibytes = (((len - 1) * lda + a.N - t.r0) * 2 + 15) & ~(int64_t)15;
    jbytes = (((len - 1) * ldb + a.K - t.j0) * 2 + 15) & ~(int64_t)15;
    istep = 128 * lda;
    jstep = 128 * ldb;
  } else {
    if (!lin_pick<BM, BN>(a, jend, t)) return;
    len = t.group == a.experts ? 0 : a.len;
    if constexpr (Q4) {
      lda = a.K >> 2;  // two codes a byte, in units of two bytes as the others
      ip = a.xq + t.pad * (a.K >> 1);
      ibytes = (t.r1 - t.r0) * (a.K >> 1);
    } else {
      ip = (const uint8_t*)a.a + t.r0 * lda * 2;
      ibytes = ((t.r1 - t.r0 - 1) * lda + len) * 2;
    }
    istep = 128;
    constexpr bool MX = P::MX || Q4;
    const int64_t ldw = MX ? a.K : a.ldw;
    ldb = Q4 ? a.K >> 2 : ldw;
    const int64_t first = OP == LIN_FORWARD ? (t.group * a.N + t.j0) * ldw : t.group * a.N * ldw + t.j0;
    const int64_t count = OP == LIN_FORWARD ? (a.N - t.j0) * ldw : a.N * ldw - t.j0;
    jp = (const uint8_t*)a.w + (MX ? first >> 1 : first * 2);
    jbytes = MX ? count >> 1 : count * 2;
    jstep = OP == LIN_FORWARD ? (P::MX ? 32 : 128) : 64 * (MX ? ldw >> 1 : ldw * 2);
  }
  // tiles [kb, ke) of nk: this workgroup's part where the contraction is split
  const int nk = (int)((len + CT - 1) / CT);
  const int splits = OP == LIN_WEIGHT_GRAD ? gridDim.z : gridDim.y, split = OP == LIN_WEIGHT_GRAD ? blockIdx.z : blockIdx.y;
  const int per = (nk + splits - 1) / splits, kb = split * per, ke = kb + per < nk ? kb + per : nk;
  v4f32 acc[FI][FJ] = {};

  if (kb < ke) {
    uint32_t io[P::IL], jo[P::JL];
    mm_offsets<P::IK, BM, P::IL, P::NW, false>(io, wave, lane, lda);
    if constexpr (P::JK != KS4) mm_offsets<P::JK, BN, P::JL, P::NW, true>(jo, wave, lane, ldb);
    // scales of KC4: per fragment column, the byte of block 2 kt + (g >> 1)
    const uint8_t* sp = MX ? a.scale + t.group * a.scale_stride : nullptr;
    uint32_t so[P::JK == KC4 ? FJ : 1];
    uint32_t sv[P::JK == KC4 ? FJ : 1];
    const int64_t nb = a.K >> 5;
    if constexpr (P::JK == KC4) {
#pragma unroll
      for (int f = 0; f < FJ; ++f) {
        int64_t n = t.j0 + wj * (FJ * 16) + lin_jcol(f * 16 + (lane & 15));
        if (n >= a.N) n = a.N - 1;
        so[f] = a.swizzled ? (uint32_t)((n >> 7) * ((nb + 3) >> 2) * 512 + (n & 31) * 16 + ((n & 127) >> 5) * 4) : (uint32_t)(n * nb);
      }
    }
    // Q4: packed scales of this tile's 64-slot groups, nk pieces each
    const uint8_t *isp = nullptr, *jsp = nullptr;
    int64_t isbytes = 0, jsbytes = 0;
    if constexpr (Q4) {
      const int64_t gj = (a.N + 63) >> 6;
      isp = a.xs + (t.pad >> 6) * nk * 512;
      isbytes = (a.padded - (t.pad >> 6)) * nk * 512;
      jsp = a.wsc + (t.group * gj + (t.j0 >> 6)) * nk * 512;
      jsbytes = (gj - (t.j0 >> 6)) * nk * 512;
    }
    // KS4: this thread decodes 32 codes of contraction row kr
    const int kr = tid / (BN / 32), kc = tid % (BN / 32);
    lm_u32x4 code = {};
    uint32_t code_s = 0;

    auto load = [&](int kt, lds_u8* ti, lds_u8* tj, lds_u8* tis, lds_u8* tjs) {
      const __amdgpu_buffer_rsrc_t ri = lin_rsrc(ip + kt * istep, ibytes - kt * istep);
      const bool cut = (kt + 1) * CT > len;
      constexpr int PIECE = CT / 8;  // of the contraction in a 16-byte piece of KC16
#pragma unroll
      for (int n = 0; n < P::IL; ++n) {
        uint32_t o = io[n];
        if (P::IK == KC16 && cut) {  // chunks past the row's end are zeros, not the next row
          const int piece = (n * P::NW + wave) * 64 + lane;
          const int c = (piece & 7) ^ ((piece >> 3) & 7);
          if (kt * CT + c * PIECE >= len) o = 0x80000000u;
        }
        lin_dma(ri, ti + (n * P::NW + wave) * 1024, o);
      }
      if constexpr (P::JK != KS4) {
        const __amdgpu_buffer_rsrc_t rj = lin_rsrc(jp + kt * jstep, jbytes - kt * jstep);
#pragma unroll
        for (int n = 0; n < P::JL; ++n) {
          uint32_t o = jo[n];
          if (P::JK != KS16 && cut) {
            const int piece = (n * P::NW + wave) * 64 + lane;
            const int c = P::JK == KC4 ? (piece & 1) * 4 : (piece & 7) ^ ((piece >> 3) & 7);
            if (kt * CT + c * PIECE >= len) o = 0x80000000u;
          }
          lin_dma(rj, tj + (n * P::NW + wave) * 1024, o);
        }
      }
      if constexpr (Q4) {  // 512 bytes per 64 slots: 128 slots a load, a wave each
        const int h = wave < BM / 128 ? wave : wave - BM / 128;
        if (wave < BM / 128) lin_dma(lin_rsrc(isp, isbytes), tis + h * 1024, ((2 * h + (lane >> 5)) * nk + kt) * 512 + (lane & 31) * 16);
        else if (wave < BM / 128 + BN / 128) lin_dma(lin_rsrc(jsp, jsbytes), tjs + h * 1024, ((2 * h + (lane >> 5)) * nk + kt) * 512 + (lane & 31) * 16);
      }
    };
    auto load_scales = [&](int kt) {
      if constexpr (P::JK == KC4) {
        int64_t kb = 2 * kt + (g >> 1);
        if (kb >= nb) kb = nb - 1;
        const uint32_t at = a.swizzled ? (uint32_t)((kb >> 2) * 512 + (kb & 3)) : (uint32_t)kb;
#pragma unroll
        for (int f = 0; f < FJ; ++f) sv[f] = sp[so[f] + at];
      } else if constexpr (P::JK == KS4) {
        const int64_t n = (int64_t)kt * 64 + kr, k = t.j0 + kc * 32;
        code = lm_u32x4{};
        code_s = 0;
        if (n < a.N && k < a.K) {
          code = *(const LM_GLOBAL lm_u32x4*)(jp + n * (a.K >> 1) + kc * 16);
          code_s = sp[blocked_offset(n, k >> 5, nb, a.swizzled)];
        }
      }
    };
    auto store_codes = [&](lds_u8* tj) {
      if constexpr (P::JK == KS4) {
        const float s = e8m0_value(code_s);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *(lds_u32x4*)(tj + kr * (BN * 2) + (((kc * 4 + c) ^ ((kr & 3) << 2)) << 4)) = lin_decode8<HALF>(code[c], s);
      }
    };
    auto compute = [&](const lds_u8* ti, const lds_u8* tj, const lds_u8* tis, const lds_u8* tjs, const float* scales) {
      lm_u32x2 isc[Q4 ? FI / 4 : 1], jsc[Q4 ? FJ / 4 : 1];
      if constexpr (Q4) {
#pragma unroll
        for (int f = 0; f < FI / 4; ++f) isc[f] = *(const lds_u32x2*)(tis + (wi * (FI / 4) + f) * 512 + lane * 8);
#pragma unroll
        for (int f = 0; f < FJ / 4; ++f) jsc[f] = *(const lds_u32x2*)(tjs + (wj * (FJ / 4) + f) * 512 + lane * 8);
      }
      lm_u32x2 jc[P::JK == KC4 ? FJ : 1];
      if constexpr (P::JK == KC4) {
#pragma unroll
        for (int f = 0; f < FJ; ++f)
          jc[f] = *(const lds_u32x2*)(tj + (wj * (FJ * 16) + f * 16 + (lane & 15)) * 32 + g * 8);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        lm_u32x4 fi[FI], fj[FJ];
#pragma unroll
        for (int f = 0; f < FJ; ++f) {
          if constexpr (P::JK == KC4) fj[f] = lin_decode8<HALF>(jc[f][s], scales[f]);
          else if constexpr (P::JK == KC16) fj[f] = mm_frag<KC16, BN>(tj, wj * (FJ * 16), f, lane, s, P::chunk(s, g));
          else fj[f] = mm_frag_tr<BN, true>(tj, wj * (FJ * 16), f, lane, s);
        }
#pragma unroll
        for (int f = 0; f < FI; ++f) {
          if constexpr (P::IK == KC16) fi[f] = mm_frag<KC16, BM>(ti, wi * (FI * 16), f, lane, s, P::chunk(s, g));
          else fi[f] = mm_frag_tr<BM, false>(ti, wi * (FI * 16), f, lane, s);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < FI; ++x)
#pragma unroll
          for (int y = 0; y < FJ; ++y) {
            if constexpr (Q4) acc[x][y] = lin_mfma4(fj[y], fi[x], acc[x][y], jsc[y >> 2][(y >> 1) & 1], isc[x >> 2][(x >> 1) & 1], s, y & 1, x & 1);
            else acc[x][y] = lin_mfma<HALF>(fj[y], fi[x], acc[x][y]);
          }
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    lds_u8 *i0 = (lds_u8*)si0, *i1 = (lds_u8*)si1, *j0 = (lds_u8*)sj0, *j1 = (lds_u8*)sj1;
    lds_u8 *is0 = (lds_u8*)sis0, *is1 = (lds_u8*)sis1, *js0 = (lds_u8*)sjs0, *js1 = (lds_u8*)sjs1;
    auto scales_now = [&](float(&out)[P::JK == KC4 ? FJ : 1]) {
      if constexpr (P::JK == KC4) {
#pragma unroll
        for (int f = 0; f < FJ; ++f) out[f] = e8m0_value(sv[f]);
      }
    };
    load(kb, i0, j0, is0, js0);
    load_scales(kb);
    store_codes(j0);
    float sc[P::JK == KC4 ? FJ : 1];
    int kt = kb;
    for (; kt + 1 < ke; kt += 2) {  // (no way out of the middle: it would keep two copies of the accumulators)
      __syncthreads();
      scales_now(sc);
      load(kt + 1, i1, j1, is1, js1);
      load_scales(kt + 1);
      compute(i0, j0, is0, js0, sc);
      store_codes(j1);
      __syncthreads();
      scales_now(sc);
      if (kt + 2 < ke) {
        load(kt + 2, i0, j0, is0, js0);
        load_scales(kt + 2);
      }
      compute(i1, j1, is1, js1, sc);
      if (kt + 2 < ke) store_codes(j0);
    }
    if (kt < ke) {
      __syncthreads();
      scales_now(sc);
      compute(i0, j0, is0, js0, sc);
    }
  }

  const int64_t rows0 = OP == LIN_WEIGHT_GRAD ? t.group * a.N : 0;  // of the output above this group's
  if (a.part) {  // a part of the sums: k_lin_join adds them up
    float* part = a.part + (split * (OP == LIN_WEIGHT_GRAD ? a.experts * a.N : a.T) + rows0) * jend;
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      const int64_t i = t.r0 + wi * (FI * 16) + x * 16 + (lane & 15);
#pragma unroll
      for (int y = 0; y < FJ; ++y) {
        const int64_t j = t.j0 + wj * (FJ * 16) + (y >> 1) * 32 + 8 * g + 4 * (y & 1);
        if (i < t.r1) {
          if (j + 4 <= jend) {
            *(LM_GLOBAL lm_u32x4_any*)(part + i * jend + j) = __builtin_bit_cast(lm_u32x4, acc[x][y]);
          } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
              if (j + e < jend) ((LM_GLOBAL float*)part)[i * jend + j + e] = acc[x][y][e];
          }
        }
      }
    }
    return;
  }
  uint16_t* out = (uint16_t*)a.out + rows0 * jend;
#pragma unroll
  for (int y = 0; y < FJ; y += 2) {
    const int64_t j = t.j0 + wj * (FJ * 16) + y * 16 + 8 * g;
    float bias[8] = {};
    if (OP == LIN_FORWARD && a.bias && t.group < a.experts) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        bias[e] = val_dt<DT>(((const LM_GLOBAL uint16_t*)a.bias)[j + e < jend ? j + e : jend - 1]);
    }
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      const int64_t i = t.r0 + wi * (FI * 16) + x * 16 + (lane & 15);
      lm_u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = acc[x][y + (e >> 1)][2 * (e & 1)] + bias[2 * e], hi = acc[x][y + (e >> 1)][2 * (e & 1) + 1] + bias[2 * e + 1];
        w[e] = DT == F16 ? (uint32_t)f16_bits(lo) | (uint32_t)f16_bits(hi) << 16 : pack_bf16x2(lo, hi);
      }
      uint16_t* p = out + i * jend + j;
      if (i < t.r1) {
        if (j + 8 <= jend) {
          *(LM_GLOBAL lm_u32x4_any*)p = w;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (j + e < jend) ((LM_GLOBAL uint16_t*)p)[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
}

// the sum of the parts of a split contraction, in their order, rounded
template <int DT>
__global__ __launch_bounds__(256) void k_lin_join(const float* part, int splits, int64_t n, int64_t J, const uint16_t* bias,
                                                  uint16_t* out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float s[4] = {};
  for (int k = 0; k < splits; ++k) {
    const LM_GLOBAL float* p = (const LM_GLOBAL float*)part + k * n + i;
    if (i + 4 <= n) {
      const v4f32 v = __builtin_bit_cast(v4f32, *(const LM_GLOBAL lm_u32x4_any*)p);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (i + e < n) s[e] += p[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (i + e < n) {
      if (bias) s[e] += val_dt<DT>(((const LM_GLOBAL uint16_t*)bias)[(i + e) % J]);
      ((LM_GLOBAL uint16_t*)out)[i + e] = bits_dt<DT>(s[e]);
    }
}

// rows of any stride and alignment, copied to a stride of whole 16-byte pieces
// and filled up with zeros
__global__ __launch_bounds__(256) void k_lin_align(const uint16_t* src, int64_t lds, int64_t rows, int64_t cols, uint16_t* dst,
                                                   int64_t ldd) {
  const int64_t pieces = ldd >> 3, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * pieces) return;
  const int64_t r = i / pieces, c = (i - r * pieces) * 8;
  store_b128_guarded((LM_GLOBAL lm_u32x4*)(dst + r * ldd + c), lin_chunk(src + r * lds + c, cols - c));
}
