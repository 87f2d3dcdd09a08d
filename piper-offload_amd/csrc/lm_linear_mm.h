// lm_linear_mm.h -- products of many rows: LDS-tiled MFMA kernels.
//
// An output tile of BM rows x BN columns per workgroup.  The contraction goes by
// in stages of one MFMA step (32 values; 128 with 4-bit inputs), four LDS
// buffers deep: a stage's loads (buffer loads straight to LDS, no registers in
// between) are issued three stages before its multiplication.
//
// Operands are named by the output index they carry: I (rows) and J
// (columns).  Their tiles lie in LDS as
//   KC16  contraction contiguous in memory: a slot of 64 bytes per I/J index,
//         its four 16-byte chunks in an order that depends on the slot (mm_key)
//   KS16  contraction strided (the index contiguous): a row per contraction
//         step; read transposed (ds_read_b64_tr_b16); chunks XORed with a key
//         of the row (mm_row_key)
//   KC4   MXFP4 codes as they are stored, decoded to 16 bits after the read
//         (v_cvt_scalef32_pk: exact products in bf16).  A stage is 16 bytes of a
//         row, so four stages are loaded together, in whole runs of 64 bytes
//   KS4   MXFP4 with the contraction strided: every code of a run of 32 shares a
//         scale but the 8 codes of an MFMA lane do not, so these are decoded on
//         their way into LDS and then are KS16
//   KC8   INT8 codes along the contraction, KS8 across it: decoded on their way into
//         LDS too, and then KC16 (the codes alone: the scales come with the store)
//         and KS16 (times their row's scale, which lies along the sum; in fp16 with a
//         power of two that brings a weight's scales into its range and comes out of the sums)
// Q8: both operands INT8 codes; a slot of 64 bytes has 64 of them, and all but the
// matrix instruction is as for 16 bits (the arguments count in pairs of codes).
//   KR8   the weight's codes where rows start anywhere: loads straight to LDS take whole
//         pieces of 16 bytes only, so these go through registers, and then are KC16
// Q4: both operands MXFP4 (x quantised beforehand), multiplied as they are by the
// scaled MFMA, 128 codes a stage, so a slot is 64 bytes here too.  Its scales
// come packed by k_lin_prep4: per 64 slots and stage 256 bytes, which hold for
// lane (r, g) block g of slots r, r + 16, r + 32, r + 48: one 4-byte read gives
// the scales of four fragments.
// The MFMA's first operand is J, so a lane's four accumulators are consecutive
// output columns; before the store two neighbouring fragments trade halves
// between lane groups, which makes them 8 in a row: one 16-byte store.
//
// Eight waves (256 x 256): two on a SIMD.  If both read their fragments at the
// same time and then both multiply, LDS and the matrix unit take turns
// (measured: 1.24 PFLOP/s at most).  So the waves of the second half run one
// barrier behind those of the first: while one wave of a SIMD reads, the other
// multiplies.  Four waves (128 x 128): the two workgroups of a CU do that by
// themselves.
//
// Bound by the matrix unit, on a clock that falls under it, and by the LDS reads
// beside it: bf16 [8192, 8192] at 8192 rows 1.33 PFLOP/s; MXFP4 [14336, 4096] at
// 2048 rows 1.13 forward (matrix unit busy 63% of the cycles) and 1.09 for the input
// gradient with its join, at 4096 rows with 4-bit inputs 3.4 (46%).  INT8: lm_linear8.hip.
#pragma once
#include <type_traits>

#include "lm_linear.h"

enum : int { KC16, KS16, KC4, KS4, KC8, KS8, KR8 };

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) uint32_t lds_u32;
typedef __attribute__((address_space(3))) lm_u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

// 16 bytes per lane to LDS at base + 16 lane; past the resource's end: zeros
DEV void lin_dma(__amdgpu_buffer_rsrc_t r, lds_u8* base, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)base, 16, (int)off, 0, 0, 0);
}
// LDS serves a 16-byte read of a wave 16 lanes at a time, lanes 0-3, 12-15 and
// 20-27 first, then 4-11, 16-19 and 28-31, and the same in the upper half.  A slot
// is a quarter of the 64 banks, so four slots (p & 3) share them out and the
// four groups of slots (p >> 2) that are served together have to find their
// chunks in four different places: chunk c lies at c ^ (2 (p >> 2) in GF(4)).
// With c ^ (p >> 2), right for lanes taken in order, half the cycles are
// conflicts (SQ_LDS_BANK_CONFLICT).
DEV int mm_key(int slot) { return (((slot >> 2) << 1) & 2) ^ (((slot >> 3) & 1) * 3); }
// A transposed read takes 32 bytes each of rows 0-3 and 8-11 (then 16-19 and
// 24-27) together: eight pairs of chunks, one of each in all 64 banks.  (Rows of
// 64 indices are half of the banks, two neighbours all of them.)
template <int B>
DEV int mm_row_key(int row) {
  if constexpr (B == 64) return (((row >> 1) & 1) | ((row >> 2) & 2)) << 1;
  return ((row & 3) | ((row >> 1) & 4)) << 1;
}

// Tiles of up to 8 row tiles x all columns, row tiles first, are neighbours, and
// each XCD takes a contiguous part of them, so its L2 holds the tiles of the
// other operand that several row tiles share.
DEV void lin_order(uint32_t u, uint32_t tm, uint32_t tn, uint32_t& m, uint32_t& n) {
  const uint32_t band = u / (8 * tn), in = u - band * 8 * tn, left = tm - band * 8, h = left < 8 ? left : 8;
  m = band * 8 + in % h;
  n = in / h;
}
// Of 256 x 256 tiles, those of whole rounds over the 256 CUs.  The rest, where it
// is less than half a round, is left to a second launch of 128 x 128 tiles, which
// has something for every CU: 8 groups [4096, 2048] at 4096 rows have 312 tiles.
DEV uint32_t lin_rounds(uint32_t total) {
  return total >= 256 && total % 256 <= 128 ? total - total % 256 : total;
}
// The tile of this workgroup: group, first row, end of the group's rows, first
// column.
struct LinTile {
  int group;
  int64_t r0, r1, j0;
  int64_t pad;  // the first row among the rows padded to 64 a group
};
template <int BM, int BN>
DEV bool lin_pick(const LinArgs& a, int64_t jend, LinTile& t) {
  const bool rest = BM == 128 && a.rounds;  // quarters of the 256 x 256 tiles that are left
  const int bm = rest ? 256 : BM, bn = rest ? 256 : BN;
  const uint32_t tm = a.ends ? (uint32_t)lin_count(a, bm) : (uint32_t)((a.T + bm - 1) / bm), tn = (uint32_t)((jend + bn - 1) / bn);
  const uint32_t total = tm * tn, whole = a.rounds ? lin_rounds(total) : total;
  uint32_t b = blockIdx.x, m, n;
  if (b >= (rest ? 4 * (total - whole) : whole)) return false;
  b = (uint32_t)xcd_unit(b, rest ? 4 * (total - whole) : whole);
  lin_order(rest ? whole + (b >> 2) : b, tm, tn, m, n);
  t.j0 = (int64_t)n * bn;
  if (a.ends) {
    if (!lin_find(a, bm, (int)m, t.group, t.r0, t.r1, t.pad)) return false;
  } else {
    t.group = 0;
    t.pad = t.r0 = (int64_t)m * bm;
    t.r1 = a.T;
  }
  if (rest) {
    t.r0 += (b >> 1 & 1) * 128;
    t.pad += (b >> 1 & 1) * 128;
    t.j0 += (b & 1) * 128;
  }
  return t.r0 < t.r1 && t.j0 < jend;
}

template <int DT, int OP, int W, int BM, int BN, int WM, int WN>
struct MmTraits {
  static constexpr bool Q4 = W == W_Q4, MX = W == W_MX, Q8 = W == W_Q8 || W == W_R8, I8 = W == W_I8;
  static constexpr int NW = WM * WN, NT = NW * 64;
  static constexpr int CS = Q4 ? 128 : 32;  // contraction of a stage
  static constexpr int IK = OP == LIN_WEIGHT_GRAD ? KS16 : KC16;
  static constexpr int JK = OP == LIN_FORWARD      ? (MX ? KC4 : I8 ? KC8 : W == W_R8 ? KR8 : KC16)
                            : OP == LIN_INPUT_GRAD ? (MX ? KS4 : I8 ? KS8 : KS16)
                                                   : KS16;
  static constexpr bool REG = JK == KS4 || JK == KC8 || JK == KS8 || JK == KR8;  // to LDS through registers, decoded but for KR8
  static constexpr int LK = JK == KS4 || JK == KS8 ? KS16 : JK == KC8 || JK == KR8 ? KC16 : JK;  // J's tile in LDS
  static constexpr int FI = BM / WM / 16, FJ = BN / WN / 16;
  static constexpr int IB = BM * 64, JB = BN * 64;  // bytes of a stage (KC4: of four)
  static constexpr int IL = IB / 1024 / NW;                               // loads per wave
  static constexpr int JL = JK == KC8 ? 1 : REG ? 2 : JB / 1024 / NW;
  static constexpr int SB = Q4 ? NW * 256 : 16;  // bytes of a stage's scales: I's, then J's
  static_assert(!Q4 || BM / 64 + BN / 64 <= NW, "at most a piece of scales per wave");
  static_assert(IL * 1024 * NW == IB, "tiles are whole loads of all waves");
  static_assert(REG || JL * 1024 * NW == JB, "tiles are whole loads of all waves");
  static_assert(JK != KC4 || JL == 2, "KC4: a load in each of two stages");
  static_assert(!REG || NT * 16 == 32 * BN, "16 codes of a stage per thread");
};

// per-lane byte offsets of the DMA loads of one operand's stage
template <int KIND, int B, int L, int NW>
DEV void mm_offsets(uint32_t (&off)[L], int wave, int lane, int64_t ld) {
#pragma unroll
  for (int n = 0; n < L; ++n) {
    const int piece = (n * NW + wave) * 64 + lane;  // 16-byte piece of the tile
    if constexpr (KIND == KC16) off[n] = (uint32_t)((piece >> 2) * ld * 2) + ((piece & 3) ^ mm_key(piece >> 2)) * 16;
    else if constexpr (KIND == KC4) off[n] = (uint32_t)((piece >> 2) * (ld >> 1)) + ((piece & 3) ^ ((piece >> 4) & 3)) * 16;
    else off[n] = (uint32_t)(piece / (B / 8) * ld * 2) + ((piece % (B / 8)) ^ mm_row_key<B>(piece / (B / 8))) * 16;
  }
}

// The fragments of a stage: per lane one LDS offset (mm_at), and 8 contraction
// steps (chunk g) of this lane's index of fragment f from there.  KS16 reads
// transposed, two loads of 4 steps: lane p of 16 points at 4 indices of row p >> 2.
template <int KIND, int B>
DEV uint32_t mm_at(int slot0, int lane) {
  const int p = lane & 15, g = lane >> 4;
  if constexpr (KIND == KC16) return (slot0 + p) * 64 + ((g ^ mm_key(p)) << 4);
  else if constexpr (KIND == KC4) return (slot0 + p) * 64 + ((p >> 2) << 4) + g * 4;  // ^ 16 times the stage
  const int row = 8 * g + (p >> 2), chunk = (slot0 >> 3) + ((p >> 1) & 1);
  return row * (B * 2) + ((chunk ^ mm_row_key<B>(row)) << 4 | (p & 1) << 3);
}
template <int KIND, int B>
DEV lm_u32x4 mm_frag(const lds_u8* t, uint32_t at, int f) {
  if constexpr (KIND == KC16) return *(const lds_u32x4*)(t + at + f * 1024);
  const uint32_t o = at ^ (f << 5);  // two chunks on
  const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(t + o));
  const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(t + o + 4 * (B * 2)));  // row + 4: same key
  return lm_u32x4{__builtin_bit_cast(lm_u32x2, lo)[0], __builtin_bit_cast(lm_u32x2, lo)[1],
                  __builtin_bit_cast(lm_u32x2, hi)[0], __builtin_bit_cast(lm_u32x2, hi)[1]};
}
// The compiler would keep this value plus every buffer's address in a register
// of its own across the loop; like this it adds the buffer's offset in the read.
DEV uint32_t mm_hide(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// SHORT: a contraction of at most two stages (a LoRA's rank).  All of it is loaded
// at once, so two buffers do and twice as many workgroups fit on a CU: such a
// product is a write of its output, and a workgroup mostly waits.
template <int DT, int OP, int W, int BM, int BN, int WM, int WN, bool SHORT = false>
__global__ __launch_bounds__(WM* WN * 64, SHORT ? 5 : 2) void k_lin_mm(LinArgs a) {
  using P = MmTraits<DT, OP, W, BM, BN, WM, WN>;
  constexpr bool HALF = DT == F16, Q4 = P::Q4, Q8 = P::Q8, I8 = P::I8, REG = P::REG, PP = P::NW == 8;
  constexpr int CS = P::CS, FI = P::FI, FJ = P::FJ, IK = P::IK, JK = P::JK;
  // (separate arrays: the compiler then knows that a read of one stage need not
  // wait for the loads of another)
  __shared__ __attribute__((aligned(1024))) uint8_t si0[P::IB], si1[P::IB], si2[SHORT ? 16 : P::IB], si3[SHORT ? 16 : P::IB];
  __shared__ __attribute__((aligned(1024))) uint8_t sj0[P::JB], sj1[P::JB], sj2[JK == KC4 || SHORT ? 16 : P::JB], sj3[JK == KC4 || SHORT ? 16 : P::JB];
  __shared__ __attribute__((aligned(1024))) uint8_t ss0[P::SB], ss1[P::SB], ss2[P::SB], ss3[P::SB];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
  const int wave = wave_index();
  const int wi = wave / WN, wj = wave % WN;
  const int64_t jend = OP == LIN_FORWARD ? a.N : a.K;
  LinTile t;
  int64_t len;  // of the contraction
  const uint8_t *ip, *jp;
  int64_t ibytes, jbytes, istep, jstep;  // bytes of the resources, and per stage
  int64_t lda = a.lda, ldb;
  if constexpr (OP == LIN_WEIGHT_GRAD) {
    uint32_t m, n;
    const uint32_t tm = (uint32_t)((a.N + BM - 1) / BM), tn = (uint32_t)((a.K + BN - 1) / BN);
    lin_order((uint32_t)xcd_unit(blockIdx.x, tm * tn), tm, tn, m, n);
    t.group = blockIdx.y;
    t.r0 = (int64_t)m * BM;
    t.r1 = a.N;
    t.j0 = (int64_t)n * BN;
    int64_t b, e;
    lin_group(a, t.group, b, e);
    len = e - b;
    ldb = a.ldb;
    ip = (const uint8_t*)a.a + (b * lda + t.r0) * 2;
    jp = (const uint8_t*)a.b + (b * ldb + t.j0) * 2;
    // (whole pieces of 16 bytes: what a piece holds past the row's end goes to columns that are not stored)
    ibytes = (((len - 1) * lda + a.N - t.r0) * 2 + 15) & ~(int64_t)15;
    jbytes = (((len - 1) * ldb + a.K - t.j0) * 2 + 15) & ~(int64_t)15;
    istep = 2 * CS * lda;
    jstep = 2 * CS * ldb;
  } else {
    if (!lin_pick<BM, BN>(a, jend, t)) return;
    // KS8, rows of no whole 16-byte pieces: the last tile ends where they end, so no
    // piece of 16 codes passes a row's end (the columns that two tiles have are computed alike)
    if (JK == KS8 && a.ldw == a.K && a.K % 16 != 0 && t.j0 + BN > a.K) t.j0 = a.K - BN;
    len = t.group == a.experts ? 0 : a.len;
    if constexpr (Q4) {
      lda = a.K >> 2;  // two codes a byte, in units of two bytes as the others
      ip = a.xq + t.pad * (a.K >> 1);
      ibytes = (t.r1 - t.r0) * (a.K >> 1);
    } else {
      ip = (const uint8_t*)a.a + t.r0 * lda * 2;
      ibytes = ((t.r1 - t.r0 - 1) * lda + len) * 2;
    }
    istep = 64;
    constexpr bool MX = P::MX || Q4;
    const int64_t ldw = MX ? a.K : a.ldw;
    ldb = Q4 ? a.K >> 2 : ldw;
    const int64_t first = OP == LIN_FORWARD ? (t.group * a.N + t.j0) * ldw : t.group * a.N * ldw + t.j0;
    const int64_t count = OP == LIN_FORWARD ? (a.N - t.j0) * ldw : a.N * ldw - t.j0;
    constexpr bool BYTES = I8 || JK == KR8;
    jp = (const uint8_t*)a.w + (MX ? first >> 1 : BYTES ? first : first * 2);
    jbytes = MX ? count >> 1 : BYTES ? count : count * 2;
    jstep = OP == LIN_FORWARD ? (P::MX ? 16 : BYTES ? 0 : 64) : CS * (MX ? ldw >> 1 : I8 ? ldw : ldw * 2);
  }
  // stages [kb, ke) of nk: this workgroup's part where the contraction is split
  const int nk = (int)((len + CS - 1) / CS);
  const int splits = OP == LIN_WEIGHT_GRAD ? gridDim.z : gridDim.y, split = OP == LIN_WEIGHT_GRAD ? blockIdx.z : blockIdx.y;
  const int per = ((nk + splits - 1) / splits + 3) & ~3, kb = split * per, ke = kb + per < nk ? kb + per : nk;
  v4f32 acc[FI][FJ] = {};
  constexpr bool SHIFT = JK == KS8 && HALF;
  const int shift = SHIFT && t.group < a.experts ? __builtin_amdgcn_readfirstlane(a.shift[t.group]) : 0;

  if (kb < ke) {
    uint32_t io[P::IL], jo[P::JL];
    mm_offsets<IK, BM, P::IL, P::NW>(io, wave, lane, lda);
    if constexpr (!REG) mm_offsets<JK, BN, P::JL, P::NW>(jo, wave, lane, ldb);
    const int nb = (int)(a.K >> 5);
    const uint8_t* sp = P::MX ? a.scale + t.group * a.scale_stride : nullptr;
    // KC4: the scales of four stages, one word per fragment column
    uint32_t so[JK == KC4 ? FJ : 1], sv[JK == KC4 ? FJ : 1], sn[JK == KC4 ? FJ : 1];
    const int64_t stile = a.swizzled ? (t.j0 >> 7) * ((nb + 3) >> 2) * 512 : t.j0 * nb;
    const uint32_t sleft = a.scale_stride - stile > LIN_SPAN ? (uint32_t)LIN_SPAN : (uint32_t)(a.scale_stride - stile);
    const uint32_t slast = sleft < 4 ? LIN_OUT : sleft - 4;  // the last whole word, if there is one
    if constexpr (JK == KC4) {
#pragma unroll
      for (int f = 0; f < FJ; ++f) {
        int n = wj * (FJ * 16) + f * 16 + (lane & 15);
        if (t.j0 + n >= a.N) n = (int)(a.N - 1 - t.j0);
        so[f] = a.swizzled ? (uint32_t)((n >> 7) * ((nb + 3) >> 2) * 512 + (n & 31) * 16 + ((n & 127) >> 5) * 4) : (uint32_t)(n * nb);
      }
    }
    auto load_scales = [&](int st) {  // of stages st .. st + 3: always FJ loads
      if constexpr (JK == KC4) {
        const __amdgpu_buffer_rsrc_t rs = lin_rsrc(sp + stile, sleft);
#pragma unroll
        for (int f = 0; f < FJ; ++f) {
          uint32_t o = so[f] + (a.swizzled ? st * 128 : st);
          if (o > slast) o = slast;  // (the last word of all: next_scales shifts)
          sn[f] = __builtin_amdgcn_raw_buffer_load_b32(rs, (int)o, 0, 0);
        }
      }
    };
    // Fewer than 4 bytes in all: rows of at most 3 blocks, so these are all stages'.
    // A word would end past the resource, and reads past the tensor or as zeros.
    auto load_bytes = [&]() {
      if constexpr (JK == KC4) {
        const __amdgpu_buffer_rsrc_t rs = lin_rsrc(sp + stile, sleft);
#pragma unroll
        for (int f = 0; f < FJ; ++f) {
          sn[f] = 0;
#pragma unroll
          for (int b = 0; b < 3; ++b) sn[f] |= (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(rs, (int)so[f] + b, 0, 0) << (8 * b);
        }
      }
    };
    auto next_scales = [&](int st) {  // zeros past the row's last block
      if constexpr (JK == KC4) {
        const int have = nb - st;
        const uint32_t mask = have >= 4 ? 0xffffffffu : (have <= 0 ? 0u : (1u << (8 * have)) - 1);
#pragma unroll
        for (int f = 0; f < FJ; ++f) {
          sv[f] = sn[f] & mask;
          if (have < 4) {
            const uint32_t o = so[f] + (a.swizzled ? st * 128 : st);
            const uint32_t by = o > slast ? o - slast : 0;
            sv[f] = by < 4 ? (sn[f] >> (8 * by)) & mask : 0u;
          }
        }
      }
    };
    // Q4: the packed scales of one 64-slot group of this tile, nk pieces of 256
    // bytes, are this wave's to load
    const uint8_t* scp = nullptr;
    int64_t scleft = 0;
    if constexpr (Q4) {
      const int64_t gj = (a.N + 63) >> 6, ig = (t.pad >> 6) + wave, jg = (t.j0 >> 6) + wave - BM / 64;
      if (wave < BM / 64) {
        scp = a.xs + ig * nk * 256;
        scleft = ig < a.padded ? (int64_t)nk * 256 : 0;
      } else if (wave < BM / 64 + BN / 64) {
        scp = a.wsc + (t.group * gj + jg) * nk * 256;
        scleft = jg < gj ? (int64_t)nk * 256 : 0;
      }
    }
    const __amdgpu_buffer_rsrc_t rsc = lin_rsrc(scp, scleft);
    // Contraction contiguous: one resource for the tile (its offsets stay below
    // 2^31), the offset runs along, and from this value of st * CS on the lane's
    // chunk is past the end (of the row or of this workgroup's part) and reads
    // zeros, not the next row.  Strided: the resource runs along; rows past
    // the end are past its end.  Every stage has the same number of loads, the
    // ones past the last too, which is what the waits below count.
    const int end = ke * CS < len ? ke * CS : (int)len;
    const int last = end - ((lane & 3) ^ mm_key(lane >> 2)) * (CS / 4);
    const int lastj = end - ((lane & 3) ^ ((lane >> 4) & 3)) * CS;  // KC4: a chunk is a stage
    const uint8_t *ir = ip + kb * istep, *jr = jp + kb * jstep;
    int64_t il = ibytes - kb * istep, jl = jbytes - kb * jstep;
    auto left32 = [&](int64_t left, bool none) {  // (scalar instructions only)
      const int hi = (int)(left >> 32);
      const uint32_t lo = (uint32_t)left < (uint32_t)LIN_SPAN ? (uint32_t)left : (uint32_t)LIN_SPAN;
      const uint32_t n = hi > 0 ? (uint32_t)LIN_SPAN : (hi < 0 ? 0u : lo);
      return none ? 0u : n;
    };
    const uint32_t in = left32(il, false), jn = left32(jl, false);
    // KS4: this thread decodes 16 codes of contraction row kr.  (Its loads are
    // issued for every stage, inside the weight or not: the waits count them.)
    // KS8 does the same; KC8: 16 codes of column kr, a row's last 16 from there on: x
    // holds its elements in that order (k_lin8_tail), zeros where they were had before.
    // KR8: twice 16 codes in the same way (k_lin8_prep).
    constexpr bool ALONG = JK == KC8 || JK == KR8;
    const int kr = ALONG ? tid >> 1 : tid / (BN / 16), kc = ALONG ? tid & 1 : tid % (BN / 16);
    lm_u32x2 code[JK == KS4 ? 2 : 1];
    lm_u32x4 code8[JK == KR8 ? 4 : REG && JK != KS4 ? 2 : 1];
    uint32_t code_s[2];
    const bool cin = ALONG ? t.j0 + kr < a.N : t.j0 + kc * 16 < a.K;
    const uint32_t co = !cin ? LIN_OUT : JK == KS4 ? (uint32_t)(kr * (a.K >> 1) + kc * 8) : (uint32_t)(kr * a.ldw + (ALONG ? 0 : kc * 16));
    const int klast = (int)a.ldw - 16;
    const uint32_t cb = (uint32_t)((t.j0 + kc * 16) >> 5);  // block of the row
    const uint32_t cso = a.swizzled ? (cb >> 2) * 512 + (kr & 31) * 16 + (cb & 3) : (uint32_t)(kr * nb) + cb;
    auto load_codes = [&](int st, int set) {
      if constexpr (JK == KR8) {
        const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)jr, 0, left32(jl, st >= ke), 0x00027000);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int c = st * (2 * CS) + kc * 32 + n * 16;
          code8[2 * set + n] = __builtin_bit_cast(lm_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, (int)(co + (c < klast ? c : klast)), 0, 0));
        }
      }
      if constexpr (JK == KC8 || JK == KS8) {
        const bool none = st >= ke;
        const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)jr, 0, left32(jl, none), 0x00027000);
        jr += jstep;
        jl -= jstep;
        uint32_t o = co;
        if constexpr (JK == KC8) {
          const int c = st * CS + kc * 16;
          o += c < klast ? c : klast;
        }
        code8[set] = __builtin_bit_cast(lm_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, (int)o, 0, 0));
      }
      if constexpr (JK == KS8) {  // (rows past N: zeros, as their codes are)
        const int sz = a.scale16 ? 2 : 4;
        const int64_t sleft8 = st >= ke ? 0 : (a.N - (int64_t)st * CS) * sz;
        const __amdgpu_buffer_rsrc_t rs = lin_rsrc(a.scale + (t.group * a.N + (int64_t)st * CS) * sz, sleft8);
        if (a.scale16) code_s[set] = (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, kr * 2, 0, 0) << 16;
        else code_s[set] = __builtin_amdgcn_raw_buffer_load_b32(rs, kr * 4, 0, 0);
      }
      if constexpr (JK == KS4) {
        const int64_t sbase = a.swizzled ? (int64_t)(st >> 2) * ((nb + 3) >> 2) * 512 + (st & 3) * 4 : (int64_t)st * CS * nb;
        const bool none = st >= ke;
        const uint32_t left = left32(jl, none);
        const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)jr, 0, left, 0x00027000);
        jr += jstep;
        jl -= jstep;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(sp + sbase), 0, left32(a.scale_stride - sbase, none), 0x00027000);
        code[set] = __builtin_bit_cast(lm_u32x2, __builtin_amdgcn_raw_buffer_load_b64(rc, (int)co, 0, 0));
        // (a scale only where there are codes: past row N swizzled scales have padding, which may hold a NaN)
        code_s[set] = __builtin_amdgcn_raw_buffer_load_b8(rs, (int)(co < left ? cso : LIN_OUT), 0, 0);
      }
    };
    auto store_codes = [&](lds_u8* tj, int set) {
      if constexpr (JK == KR8) {
#pragma unroll
        for (int n = 0; n < 2; ++n) *(lds_u32x4*)(tj + kr * 64 + (((kc * 2 + n) ^ mm_key(kr)) << 4)) = code8[2 * set + n];
      }
      if constexpr (JK == KC8 || JK == KS8) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float s = JK != KS8 ? 1.0f : SHIFT ? __builtin_ldexpf(u2f(code_s[set]), shift) : u2f(code_s[set]);
          const lm_u32x4 v = lin_decode8i<HALF, JK == KS8>(code8[set][2 * c], code8[set][2 * c + 1], s);
          if constexpr (JK == KC8) *(lds_u32x4*)(tj + kr * 64 + (((kc * 2 + c) ^ mm_key(kr)) << 4)) = v;
          else *(lds_u32x4*)(tj + kr * (BN * 2) + (((kc * 2 + c) ^ mm_row_key<BN>(kr)) << 4)) = v;
        }
      }
      if constexpr (JK == KS4) {
        const float s = lin_e8m0(code_s[set], 0);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *(lds_u32x4*)(tj + kr * (BN * 2) + (((kc * 2 + c) ^ mm_row_key<BN>(kr)) << 4)) = lin_decode8<HALF>(code[set][c], s);
      }
    };
    // (called for every stage, in order; KC4: half says which half of the codes, tj where they go)
    auto load = [&](int st, int jst, int half, lds_u8* ti, lds_u8* tj, lds_u8* ts) {
      const bool none = st >= ke, out = st * CS >= last;
      if constexpr (JK == KC4) {  // half of the codes of stages jst .. jst + 3
        if (half >= 0) {
          lin_dma(__builtin_amdgcn_make_buffer_rsrc((void*)jr, 0, jn, 0x00027000), tj + (half * P::NW + wave) * 1024,
                  jst * CS >= lastj ? LIN_OUT : jo[half]);
          jo[half] += 64;
        }
      }
      const __amdgpu_buffer_rsrc_t ri = __builtin_amdgcn_make_buffer_rsrc((void*)ir, 0, IK == KC16 ? in : left32(il, none), 0x00027000);
#pragma unroll
      for (int n = 0; n < P::IL; ++n) {
        lin_dma(ri, ti + (n * P::NW + wave) * 1024, IK == KC16 && out ? LIN_OUT : io[n]);
        if constexpr (IK == KC16) io[n] += 64;
      }
      if constexpr (IK != KC16) {
        ir += istep;
        il -= istep;
      }
      if constexpr (JK == KC16 || JK == KS16) {
        const __amdgpu_buffer_rsrc_t rj = __builtin_amdgcn_make_buffer_rsrc((void*)jr, 0, JK == KS16 ? left32(jl, none) : jn, 0x00027000);
#pragma unroll
        for (int n = 0; n < P::JL; ++n) {
          lin_dma(rj, tj + (n * P::NW + wave) * 1024, JK == KC16 && out ? LIN_OUT : jo[n]);
          if constexpr (JK == KC16) jo[n] += 64;
        }
        if constexpr (JK != KC16) {
          jr += jstep;
          jl -= jstep;
        }
      }
      if constexpr (Q4) {
        if (lane < 16) lin_dma(rsc, ts + wave * 256, st * 256 + lane * 16);
      }
    };
    const uint32_t ati = mm_at<IK, BM>(wi * (FI * 16), lane), atj = mm_at<P::LK, BN>(wj * (FJ * 16), lane);
    lm_u32x4 fi[FI], fj[FJ];
    constexpr int IW = (FI + 3) / 4, JW = (FJ + 3) / 4;  // words of scales
    uint32_t isc[IW], jsc[JW], jc[JK == KC4 ? FJ : 1];
    auto read = [&](int b, const lds_u8* ti, const lds_u8* tj, const lds_u8* ts) {
      const uint32_t ai = mm_hide(ati), aj = mm_hide(atj);
#pragma unroll
      for (int f = 0; f < FJ; ++f) {
        if constexpr (JK == KC4) jc[f] = *(const lds_u32*)(tj + (aj ^ ((b & 3) << 4)) + f * 1024);
        else fj[f] = mm_frag<P::LK, BN>(tj, aj, f);
      }
#pragma unroll
      for (int f = 0; f < FI; ++f) fi[f] = mm_frag<IK, BM>(ti, ai, f);
      if constexpr (Q4) {
        const uint32_t as = mm_hide(lane * 4);
#pragma unroll
        for (int f = 0; f < IW; ++f) isc[f] = *(const lds_u32*)(ts + as + (wi * FI / 4 + f) * 256) >> (FI < 4 ? 8 * (wi * FI & 3) : 0);
#pragma unroll
        for (int f = 0; f < JW; ++f) jsc[f] = *(const lds_u32*)(ts + as + (BM / 64 + wj * FJ / 4 + f) * 256) >> (FJ < 4 ? 8 * (wj * FJ & 3) : 0);
      }
    };
    auto decode = [&](int b) {
      if constexpr (JK == KC4) {
#pragma unroll
        for (int f = 0; f < FJ; ++f) fj[f] = lin_decode8<HALF>(jc[f], lin_e8m0(sv[f], b & 3));
      }
    };
    auto multiply = [&]() {
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) {
          if constexpr (Q4) acc[x][y] = lin_mfma4(fj[y], fi[x], acc[x][y], jsc[y >> 2], isc[x >> 2], y & 3, x & 3);
          else if constexpr (Q8) acc[x][y] = lin_mfma8(fj[y], fi[x], acc[x][y]);
          else acc[x][y] = lin_mfma<HALF>(fj[y], fi[x], acc[x][y]);
        }
      // (the products have no side effects: nothing else keeps them from moving
      // past the barriers, the fragments of several stages with them)
#pragma unroll
      for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) asm volatile("" : "+v"(acc[x][y]));
      __builtin_amdgcn_s_setprio(0);
    };
    lds_u8* const ti[4] = {(lds_u8*)si0, (lds_u8*)si1, (lds_u8*)si2, (lds_u8*)si3};
    lds_u8* const tj[4] = {(lds_u8*)sj0, (lds_u8*)sj1, (lds_u8*)sj2, (lds_u8*)sj3};
    lds_u8* const ts[4] = {(lds_u8*)ss0, (lds_u8*)ss1, (lds_u8*)ss2, (lds_u8*)ss3};
    // loads of a stage per wave
    constexpr int L = P::IL + (JK == KC4 ? 0 : P::JL) + (Q4 ? 1 : 0);

    if constexpr (SHORT) {
      static_assert(W == W_DENSE && !PP, "short contractions: dense weights");
      load(0, 0, -1, ti[0], tj[0], ts[0]);
      if (nk > 1) load(1, 0, -1, ti[1], tj[1], ts[1]);
      lin_wait<0>();
      lin_barrier();
      read(0, ti[0], tj[0], ts[0]);
      multiply();
      if (nk > 1) {
        read(1, ti[1], tj[1], ts[1]);
        multiply();
      }
    } else {
      if (JK == KC4 && sleft < 4) load_bytes();
      else load_scales(kb);
      // KC4: the first four stages' codes; the loop asks for the next four in the
      // first two of every four stages
#pragma unroll
      for (int b = 0; b < 3; ++b) load(kb + b, kb, b < 2 ? b : -1, ti[b], JK == KC4 ? tj[0] : tj[b], ts[b]);
      if constexpr (REG) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          load_codes(kb + b, 0);
          store_codes(tj[b], 0);
        }
        load_codes(kb + 2, 0);
      }
      lin_wait<REG ? 0 : 2 * L>();  // stage kb is in LDS
      lin_barrier();
      if (PP && wave >= 4) lin_barrier();  // the second half runs one barrier behind
      auto four = [&](int st, auto half) {  // stages st .. st + 3; KC4: their codes are in buffer `half`
        constexpr int H = decltype(half)::value;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int n = (b + 3) & 3;  // the buffer of stage st + b + 3
          if (b == 0) next_scales(st);
          read(b, ti[b], JK == KC4 ? tj[H] : tj[b], ts[b]);
          __builtin_amdgcn_sched_barrier(0);
          // (while the reads are on their way)  Buffer n was read for stage
          // st + b - 1, and all waves are past that.
          if (b == 0) load_scales(st + 4);
          load_codes(st + b + 3, (b + 1) & 1);
          load(st + b + 3, st + 4, b < 2 ? b : -1, ti[n], JK == KC4 ? tj[1 - H] : tj[n], ts[n]);
          decode(b);
          // Stage st + b + 1 is in LDS, and this one in registers: what may be left
          // are the loads of stages st + b + 2 and st + b + 3, with KC4 the scales and
          // codes that were asked for since.
          if constexpr (JK == KC4) {
            if (b == 0) lin_wait<2 * L + FJ + 1>();
            else if (b == 1) lin_wait<2 * L + FJ + 2>();
            else if (b == 2) lin_wait<2 * L + 1>();
            else lin_wait<2 * L>();
          } else {
            lin_wait<2 * L>();
          }
          lin_barrier();
          multiply();
          store_codes(tj[(b + 2) & 3], b & 1);
          if constexpr (PP) lin_barrier();
        }
      };
      for (int st = kb; st < ke; st += JK == KC4 ? 8 : 4) {
        four(st, std::integral_constant<int, 0>{});
        if constexpr (JK == KC4) {
          if (st + 4 < ke) four(st + 4, std::integral_constant<int, 1>{});
        }
      }
      if constexpr (PP) {
        if (wave < 4) lin_barrier();
      }
      lin_wait<0>();  // no load may reach LDS after the workgroup
    }
  }

  if constexpr (SHIFT) {
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
      for (int y = 0; y < FJ; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][y][e] = __builtin_ldexpf(acc[x][y][e], -shift);
  }
  const int64_t rows0 = OP == LIN_WEIGHT_GRAD ? t.group * a.N : 0;  // of the output above this group's
  if (a.part) {  // a part of the sums: k_lin_join adds them up
    float* part = a.part + (split * (OP == LIN_WEIGHT_GRAD ? a.experts * a.N : a.T) + rows0) * jend;
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      const int64_t i = t.r0 + wi * (FI * 16) + x * 16 + (lane & 15);
#pragma unroll
      for (int y = 0; y < FJ; ++y) {
        const int64_t j = t.j0 + wj * (FJ * 16) + y * 16 + 4 * g;
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
  auto column = [&](int y) { return t.j0 + wj * (FJ * 16) + (y + (g & 1)) * 16 + 8 * (g >> 1); };
  float bias[FJ / 2][8] = {};
  if (OP == LIN_FORWARD && a.bias && t.group < a.experts) {
#pragma unroll
    for (int y = 0; y < FJ; y += 2) {
      const int64_t j = column(y);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        bias[y / 2][e] = val_dt<DT>(((const LM_GLOBAL uint16_t*)a.bias)[j + e < jend ? j + e : jend - 1]);
    }
  }
  // INT8 weights: the columns' scales
  float cs[I8 || Q8 ? FJ / 2 : 1][8];
  if constexpr ((I8 || Q8) && OP == LIN_FORWARD) {
#pragma unroll
    for (int y = 0; y < FJ; y += 2) {
      const int64_t j = column(y);
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[y / 2][e] = t.group < a.experts ? lin_scale8(a, t.group * a.N + (j + e < jend ? j + e : jend - 1)) : 0.0f;
    }
  }
  // A row's columns one store after the other: the halves of a 128-byte line reach
  // the L2 together, which otherwise writes many of them to memory by themselves
  // (dense weight gradient, 134 MB: 165 -> 137 MB written, 2% fewer cycles).  KS4 and KS8
  // have no register left for this order and take a column's rows.
#pragma unroll
  for (int n = 0; n < FI * FJ / 2; ++n) {
    constexpr bool DOWN = JK == KS4 || JK == KS8;
    const int x = DOWN ? n % FI : n / (FJ / 2), y = 2 * (DOWN ? n / FI : n % (FJ / 2));
    const int64_t i = t.r0 + wi * (FI * 16) + x * 16 + (lane & 15), j = column(y);
    // lane groups 0, 2 keep fragment y and get columns 4 .. 7 (12 .. 15) of it
    // from groups 1, 3, which get columns 0 .. 3 (8 .. 11) of fragment y + 1
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const auto r = __builtin_amdgcn_permlane16_swap(f2u(acc[x][y][e]), f2u(acc[x][y + 1][e]), false, false);
      v[e] = u2f(r[0]);
      v[4 + e] = u2f(r[1]);
    }
    if constexpr ((I8 || Q8) && OP == LIN_FORWARD) {
      const float rs = Q8 ? a.row_scale[i < t.r1 && t.group < a.experts ? i : 0] : 1.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = Q8 ? (float)(int)f2u(v[e]) * cs[y / 2][e] * rs : v[e] * cs[y / 2][e];
        if (t.group >= a.experts) v[e] = 0.0f;  // (rows of no group, whatever row 0 holds)
      }
    }
    lm_u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float lo = v[2 * e] + bias[y / 2][2 * e], hi = v[2 * e + 1] + bias[y / 2][2 * e + 1];
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

// The sum of the parts of a split contraction, in their order, rounded.  Rows of no
// group have no bias (`ends` is read only where there is one).  Bound by
// memory: two parts of [2048, 4096], 84 MB moved, 14 us (6 TB/s, much of it from the
// last-level cache).
template <int DT>
__global__ __launch_bounds__(256) void k_lin_join(LinArgs a, int splits, int64_t n, int64_t J) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  int64_t biased = n;  // of the sums, those before this one
  if (a.bias && a.ends) {
    int64_t b, e;
    lin_group(a, a.experts - 1, b, e);
    biased = e * J;
  }
  if (i >= n) return;
  float s[4] = {};
  for (int k = 0; k < splits; ++k) {
    const LM_GLOBAL float* p = (const LM_GLOBAL float*)a.part + k * n + i;
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
      if (a.bias && i + e < biased) s[e] += val_dt<DT>(((const LM_GLOBAL uint16_t*)a.bias)[(i + e) % J]);
      ((LM_GLOBAL uint16_t*)a.out)[i + e] = bits_dt<DT>(s[e]);
    }
}

// The same for INT8 weights, whose scales come after the sum: a wave has 256 columns
// of a row, so its group is the wave's.  Q8: the parts are whole numbers, and so is
// their sum.
template <int DT, bool Q8>
__global__ __launch_bounds__(256) void k_lin_join8(LinArgs a, int splits, uint32_t chunks) {
  const int64_t item = (int64_t)blockIdx.x * 4 + wave_index(), t = item / chunks;
  if (t >= a.T) return;
  const int64_t j0 = (item - t * chunks) * 256 + (threadIdx.x & 63) * 4;
  int group = 0;
  int64_t place;
  if (a.ends) lin_row(a, (int)t, group = a.experts, place);
  if (j0 >= a.N) return;
  const bool some = group < a.experts, whole = j0 + 4 <= a.N;
  float v[4] = {};
  if (some) {
    const LM_GLOBAL uint32_t* p = (const LM_GLOBAL uint32_t*)a.part + t * a.N + j0;
    const int64_t n = a.T * a.N;
    uint32_t sum[4] = {};
    auto add = [&](int e, uint32_t x) {
      if constexpr (Q8) sum[e] += x;
      else v[e] += u2f(x);
    };
    if (whole) {
      for (int k0 = 0; k0 < splits; k0 += 4) {  // (four parts on their way at once, zeros where there are fewer)
        lm_u32x4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = k0 + k < splits ? *(const LM_GLOBAL lm_u32x4_any*)(p + (k0 + k) * n) : lm_u32x4{};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) add(e, x[k][e]);
      }
    } else {
      for (int k = 0; k < splits; ++k)
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (j0 + e < a.N) add(e, p[k * n + e]);
    }
    const float rs = Q8 ? a.row_scale[t] : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t j = j0 + e < a.N ? j0 + e : a.N - 1;
      if constexpr (Q8) v[e] = (float)(int)sum[e];
      v[e] *= lin_scale8(a, group * a.N + j);
      if constexpr (Q8) v[e] *= rs;
      if (a.bias) v[e] += val_dt<DT>(((const LM_GLOBAL uint16_t*)a.bias)[j]);
    }
  }
  LM_GLOBAL uint16_t* const to = (LM_GLOBAL uint16_t*)a.out + t * a.N + j0;
  if (whole) {
    *(LM_GLOBAL lm_u32x2_any*)to = lm_u32x2{(uint32_t)bits_dt<DT>(v[0]) | (uint32_t)bits_dt<DT>(v[1]) << 16,
                                            (uint32_t)bits_dt<DT>(v[2]) | (uint32_t)bits_dt<DT>(v[3]) << 16};
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (j0 + e < a.N) to[e] = bits_dt<DT>(v[e]);
  }
}

// Rows of any stride and alignment, copied to a stride of whole 16-byte pieces
// and filled up with zeros.  Bound by memory: 8192 rows of 4096 at a stride of 4097
// add 21 us to a product (134 MB moved, 6.4 TB/s).
static __global__ __launch_bounds__(256) void k_lin_align(const uint16_t* src, int64_t lds, int64_t rows, int64_t cols, uint16_t* dst,
                                                   int64_t ldd) {
  const int64_t pieces = ldd >> 3, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * pieces) return;
  const int64_t r = i / pieces, c = (i - r * pieces) * 8;
  store_b128_guarded((LM_GLOBAL lm_u32x4*)(dst + r * ldd + c), lin_chunk(src + r * lds + c, cols - c));
}
