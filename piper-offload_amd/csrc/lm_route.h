// lm_route.h -- what the routing kernels share.
#pragma once
#include "lm_linear.h"

// Up to this many tokens k_route_place adds up the counts by itself: every workgroup
// reads those of all.  The reading grows with the square of the tokens, so above it two
// launches share the sums.  Whole calls, itself / shared: 8192 tokens, 64 experts 11.8 /
// 15.0 us; 16384, 256 experts 28.1 / 30.6; 32768, 64 experts 22.5 / 26.4, 256 experts 48.3 /
// 48.5.  (It grows with the experts too, which the bound leaves out: 1024 experts 41.7 / 38.2 at
// 4096 tokens, 174 / 160 at 32768.)
constexpr int64_t ROUTE_NEAR = 32768;

struct RouteArgs {
  const void* logits;  // [T, ld]
  int64_t ld;
  const float* bias;  // [E] or null
  int64_t T;
  int E, k;
  int sigmoid, renormalize;
  float scale;
  int groups, top_groups, group_best;
  int per, lanes;      // experts of a group; lanes that look at one (a power of two)
  uint32_t per_mul;    // e / per = e * per_mul >> 20 for e < 1024
  float* weight;       // [T, k]
  int32_t* expert;     // [T, k]
  int32_t* position;   // [T, k]
  int32_t* ends;       // [E]
  int block, blocks;   // tokens of a workgroup, workgroups
  int pitch;           // E in whole words of bytes (and of a wave's scores)
  uint8_t* counts;     // [blocks, pitch]: choices of a workgroup per expert, at most its tokens
  uint32_t* none;      // [blocks]: those without an expert
  uint32_t* starts;    // [blocks + 1, E + 1], more than ROUTE_NEAR tokens: those of the workgroups before; the last row has all
  FastDiv entries;     // choices of a workgroup
};

// ---- reductions over a wave (all lanes active), results in scalar registers ----
template <int CTRL, int ROWS>
DEV uint32_t route_dpp(uint32_t x) {  // 0 where no lane is read
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
DEV uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
DEV uint32_t route_max(uint32_t x) {
  x = umax(x, route_dpp<0x111, 0xf>(x));
  x = umax(x, route_dpp<0x112, 0xf>(x));
  x = umax(x, route_dpp<0x114, 0xf>(x));
  x = umax(x, route_dpp<0x118, 0xf>(x));
  x = umax(x, route_dpp<0x142, 0xa>(x));
  x = umax(x, route_dpp<0x143, 0xc>(x));
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
DEV float route_sum(float x) {
  x += u2f(route_dpp<0x111, 0xf>(f2u(x)));
  x += u2f(route_dpp<0x112, 0xf>(f2u(x)));
  x += u2f(route_dpp<0x114, 0xf>(f2u(x)));
  x += u2f(route_dpp<0x118, 0xf>(f2u(x)));
  x += u2f(route_dpp<0x142, 0xa>(f2u(x)));
  x += u2f(route_dpp<0x143, 0xc>(f2u(x)));
  return u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(x), 63));
}

// Numbers as whole numbers of the same order: both zeros alike, a NaN above all,
// nothing at 0 (which stands for no number at all).
DEV uint32_t route_key(float x) {
  const uint32_t u = f2u(x + 0.0f), k = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
  return x != x ? 0xffffffffu : k;
}
DEV float route_value(uint32_t k) {
  return u2f(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
DEV float route_fmax(float x) {  // NaN are passed over
  return route_value(route_max(x == x ? route_key(x) : 0u));
}
