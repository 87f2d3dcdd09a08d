// lm_linear_host.h -- how a product of many rows is run: its plan, its tiles, its launches.
#pragma once
#include <algorithm>

#include "lm_linear_mm.h"

static int64_t round8(int64_t x) { return (x + 7) & ~(int64_t)7; }
// whether a launch can have so many workgroups: it has fewer than 2^32 threads
static bool lin_holds(int64_t groups, int threads) { return groups < ((int64_t)1 << 32) / threads; }

struct LinPlan {
  bool few;                       // k_lin_few, else k_lin_mm
  bool brief;                     // k_lin_mm<SHORT>
  int tile, splits;               // of k_lin_mm
  bool rounds;                    // 256 x 256 tiles in whole rounds, the rest in smaller ones
  bool copy_a, copy_b, copy_w;    // rows realigned in the workspace first
  int64_t lda, ldb, ldw, len;
  int64_t padded;                 // 4-bit inputs: 64-row pieces
  size_t a, b, w, part, xq, xs, wsc, total;
};


// Tile and splits of k_lin_mm: the least of a model of its time.  A CU works on
// its tiles in turn; LinCost has the microseconds per stage, measured at 300 to
// 4096 rows of [4096, 4096], [14336, 4096] and [4096, 14336] and of 4 to 32 groups:
// 256 x 256 tiles alone, where less than half of the CUs have one, 128 x 128 two at
// a time and one, 64 x 128 three, two and one.  A stage of 4-bit inputs, four times
// as deep, takes 1.65 times as long as a dense one.  Per tile there are 8, 2.5 / 2
// and 2 / 1.5 / 1 us besides (the store of a 256 x 256 tile is not covered by
// another workgroup's work).  A split contraction writes and reads its sums in fp32
// (4.5 TB/s) and has one launch more; its parts have 8 stages and more.  Groups end
// in a part of a tile, 0.4 of one on average, and one in ten has no rows.
// Whole rounds and the rest apart (lin_rounds): the rest in 128 x 128 tiles after a
// second launch, 5 us, which groups with fewer than 48 stages do not wait for.
// Measured in graphs, us at 256 x 256 / 128 x 128 / 64 x 128: MXFP4 [14336, 4096] at 300
// rows 62 / 66 / 55, [4096, 4096] at 2048 rows 76 / 77 / 82 (input gradient 78 / 77 /
// 103), 4 groups [4096, 4096] at 1024 rows 63 / 74 / 61, 32 groups [2816, 2048] at 2048
// rows 84 / 56 / 44, at 8192 104 / 126 / 126; dense, 8 groups [4096, 2048] at 4096 rows
// in rounds 79, whole 92 / 99 / 121.  The worst of 48: dense, 32 groups [2816, 2048] at
// 2048 rows, input gradient, 90 where 256 x 256 takes 72.
struct LinCost {
  double full, alone, pair, one, three, two, single;
};
static void lin_tiling(LinPlan& p, int op, int64_t I, int64_t J, int64_t len, int64_t E, bool mx, bool quant) {
  static const LinCost dense{0.70, 0.50, 0.55, 0.28, 0.58, 0.40, 0.21}, forward{0.72, 0.64, 0.60, 0.38, 0.48, 0.36, 0.26},
      input_grad{0.72, 0.69, 0.60, 0.39, 0.60, 0.42, 0.32};
  const LinCost& k = !mx || quant ? dense : op == LIN_FORWARD ? forward : input_grad;
  const int64_t nk = (len + (quant ? 127 : 31)) / (quant ? 128 : 32);
  const double stage = quant ? 1.65 : 1.0;
  const bool wgrad = op == LIN_WEIGHT_GRAD;
  auto pairs = [&](int64_t n, double stages) {  // n 128 x 128 tiles on a CU
    return ((double)(n / 2) * k.pair + (double)(n % 2) * k.one) * stages + (double)(n / 2) * 2.5 + (double)(n % 2) * 2.0;
  };
  double best = 1e30;
  for (int tile = 256; tile >= 64; tile /= 2) {
    const int64_t bn = tile == 256 ? 256 : 128, gj = (J + bn - 1) / bn, groups = E < I ? E : I;
    int64_t gi = (I + tile - 1) / tile;
    if (wgrad) gi *= E;
    else if (E > 1) gi = std::max((groups * 9 + 9) / 10, (I * 10 + groups * tile * 4 + tile * 10 - 1) / (tile * 10));
    const int64_t tiles = gi * gj;
    int64_t most = tiles < 256 ? nk / 8 : 1;
    if (most > 16) most = 16;
    for (int64_t s = 1; s == 1 || s <= most; ++s) {
      const int64_t per = s == 1 ? nk : ((nk + s - 1) / s + 3) & ~(int64_t)3, n = (tiles * s + 255) / 256;  // tiles a CU
      const double stages = stage * (double)per;
      double t;
      bool rounds = false;
      if (tile == 256) {
        t = (double)n * (k.full * stages + 8.0);
        if (tiles * s <= 128) t = k.alone * stages + 8.0;
        const int64_t rest = tiles % 256;
        if (s == 1 && !wgrad && tiles >= 256 && (E > 1 ? (double)nk * stage >= 48.0 && rest <= 128 : rest > 0 && rest <= 64)) {
          const double apart = (double)(tiles / 256) * (k.full * stages + 8.0) + 5.0 + pairs((4 * rest + 255) / 256, stages);
          rounds = apart < t;
          if (rounds) t = apart;
        }
      } else if (tile == 128) {
        t = pairs(n, stages);
      } else {
        const double c64[3] = {0.0, k.single, k.two}, f64[3] = {0.0, 1.0, 1.5};
        t = ((double)(n / 3) * k.three + c64[n % 3]) * stages + (double)(n / 3) * 2.0 + f64[n % 3];
      }
      if (s > 1) t += 4.0 + (double)(s * I * (wgrad ? E : 1) * J) * 8.0 / 4.5e6;
      if (t < best) {
        best = t;
        p.tile = tile;
        p.splits = (int)s;
        p.rounds = rounds;
      }
    }
  }
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int DT, int OP, int W, int BM, int BN, int WM, int WN, bool SHORT = false>
static int launch_mm(const LinArgs& a, const LinPlan& p, hipStream_t st) {
  TimedLaunch timed("linear", st);
  const int64_t J = OP == LIN_FORWARD ? a.N : a.K, gj = (J + BN - 1) / BN;
  const int64_t gi = OP == LIN_WEIGHT_GRAD ? (a.N + BM - 1) / BM : lin_tiles<BM>(a.T, a.experts, a.ends != nullptr);
  if (!lin_holds(gi * gj, WM * WN * 64)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
  // (the rest of whole rounds: at most 128 tiles, four workgroups each)
  const int64_t n0 = BM == 128 && a.rounds ? 512 : gi * gj;
  const dim3 grid((unsigned)n0, OP == LIN_WEIGHT_GRAD ? a.experts : p.splits, OP == LIN_WEIGHT_GRAD ? p.splits : 1);
  hipLaunchKernelGGL((k_lin_mm<DT, OP, W, BM, BN, WM, WN, SHORT>), grid, dim3(WM * WN * 64), 0, st, a);
  LAUNCH_CHECK();
  if constexpr (OP == LIN_FORWARD && (W == W_Q8 || W == W_R8 || W == W_I8)) {
    if (p.splits > 1) {
      const int64_t chunks = (J + 255) / 256, blocks = (a.T * chunks + 3) / 4;
      if (!lin_holds(blocks, 256)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
      hipLaunchKernelGGL((k_lin_join8<DT, W != W_I8>), dim3((unsigned)blocks), dim3(256), 0, st, a, p.splits, (uint32_t)chunks);
      LAUNCH_CHECK();
    }
    return LM_OK;
  }
  if (p.splits > 1) {
    const int64_t n = (OP == LIN_WEIGHT_GRAD ? a.experts * a.N : a.T) * J, blocks = (n + 1023) / 1024;
    if (!lin_holds(blocks, 256)) return fail(LM_EUNSUPPORTED, "product too large for one launch");
    hipLaunchKernelGGL((k_lin_join<DT>), dim3((unsigned)blocks), dim3(256), 0, st, a, p.splits, n, J);
    LAUNCH_CHECK();
  }
  return LM_OK;
}
template <int DT, int OP, int W>
static int run_mm_dt(const LinArgs& a, const LinPlan& p, hipStream_t st) {
  if (p.tile == 256) {
    LinArgs b = a;
    b.rounds = p.rounds;
    const int rc = launch_mm<DT, OP, W, 256, 256, 2, 4>(b, p, st);
    return rc || !p.rounds ? rc : launch_mm<DT, OP, W, 128, 128, 2, 2>(b, p, st);
  }
  if constexpr (W == W_DENSE && OP != LIN_WEIGHT_GRAD) {
    if (p.brief) return launch_mm<DT, OP, W, 64, 128, 1, 4, true>(a, p, st);
  }
  if (p.tile == 64) return launch_mm<DT, OP, W, 64, 128, 1, 4>(a, p, st);
  return launch_mm<DT, OP, W, 128, 128, 2, 2>(a, p, st);
}
template <int OP, int W>
static int run_mm(const LinArgs& a, const LinPlan& p, int dtype, hipStream_t st) {
  return dtype == LM_F16 ? run_mm_dt<F16, OP, W>(a, p, st) : run_mm_dt<BF16, OP, W>(a, p, st);
}

