// lm_route.hip -- routing to experts, and rows to their experts and back.
//
//   p = softmax or sigmoid of a token's logits;  c = p + bias
//   groups of consecutive experts: a group's value is the sum of its group_best best
//   c; the top_groups best groups stay
//   the k best c of what is left are chosen, the best first;  w = scale p (/ sum of the chosen p)
//   position: the choices sorted by expert, in the order of the tokens; ends: the
//   number of choices of the experts up to each
//
// An expert with logit (or bias) -inf is closed.  Choices that no expert is left
// for are -1 with weight 0 and come last.
//
// A token is a wave's: lane l has the experts l, l + 64, ... in registers, a maximum
// over the wave is six DPP steps, and the choice is that maximum taken k times.  Bound
// by instructions: 16384 tokens, 256 experts in 8 groups, 8 of them chosen 34 us, 680
// vector and as many scalar instructions a token, the vector unit issuing 70% of the
// time (its bytes alone: 4 us).  8192 tokens, 64 experts, 4 chosen: 8 us; 8 tokens: 4.
#include "lm_impl.h"
#include "lm_route.h"

template <int DT>
DEV float route_load(const void* p, int64_t i) {
  if constexpr (DT == F32) return ((const LM_GLOBAL float*)p)[i];
  else return val_dt<DT>(((const LM_GLOBAL uint16_t*)p)[i]);
}

// e^x.  Rough: v_exp_f32 of x log2(e), off by 2^-22 of it and x 2^-23 more.
template <typename F, bool ROUGH>
DEV F route_exp(F x) {
  if constexpr (sizeof(F) == 8) return exp(x);
  else if constexpr (ROUGH) return __builtin_amdgcn_exp2f(x * 1.44269504f);
  else return expf(x);
}

// The scores of a token: lane l has experts l, l + 64, ...; those there are not have logit -inf.
template <typename F, bool ROUGH, int P>
DEV void route_scores(const float (&v)[P], bool sigmoid, F (&s)[P]) {
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const F d = F(1) + route_exp<F, ROUGH>(-(F)v[i]);
      if constexpr (ROUGH) s[i] = __builtin_amdgcn_rcpf(d);
      else s[i] = F(1) / d;
    }
    return;
  }
  float top = v[0];
#pragma unroll
  for (int i = 1; i < P; ++i) top = __builtin_fmaxf(top, v[i]);
  top = route_fmax(top);
  F sum = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    s[i] = v[i] == -INFINITY ? F(0) : route_exp<F, ROUGH>((F)v[i] - (F)top);
    sum += s[i];
  }
  if constexpr (sizeof(F) == 8) {
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
  } else {
    sum = route_sum(sum);
  }
  const F inv = F(1) / sum;
#pragma unroll
  for (int i = 0; i < P; ++i) s[i] *= inv;
}

DEV uint64_t route_key64(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0), k = u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
  return x != x ? ~0ull : k;
}
template <int CTRL, int ROWS>
DEV uint64_t route_max64_step(uint64_t x) {
  const uint64_t o = (uint64_t)route_dpp<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | route_dpp<CTRL, ROWS>((uint32_t)x);
  return o > x ? o : x;
}
DEV uint64_t route_max64(uint64_t x) {
  x = route_max64_step<0x111, 0xf>(x);
  x = route_max64_step<0x112, 0xf>(x);
  x = route_max64_step<0x114, 0xf>(x);
  x = route_max64_step<0x118, 0xf>(x);
  x = route_max64_step<0x142, 0xa>(x);
  x = route_max64_step<0x143, 0xc>(x);
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// The choice in 64 bits.  Lane j returns expert j, or -1.
template <int P>
DEV int route_choose64(const float (&v)[P], const float (&b)[P], bool even, int E, int k, int sigmoid, int groups, int per, int top_groups,
                       int group_best) {
  const int lane = threadIdx.x & 63;
  double s[P];
  uint64_t key[P];
  route_scores<double, false, P>(v, sigmoid, s);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    s[i] += (double)b[i];
    key[i] = v[i] == -INFINITY || s[i] == -INFINITY ? 0 : route_key64(s[i]);
  }
  if (top_groups < groups) {
    auto number = [](uint64_t k) {
      return k == ~0ull ? (double)NAN : __longlong_as_double((long long)(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
    };
    uint64_t value = 0;  // lane g: of group g
    for (int g = 0; g < groups; ++g) {  // its best, and its second: the best once more if two have it
      uint64_t best = 0, second = 0;
#pragma unroll
      for (int i = 0; i < P; ++i)
        if ((lane + 64 * i) / per == g && key[i] > best) best = key[i];
      best = route_max64(best);
      if (best == 0) continue;
      if (group_best == 2) {
        int same = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const bool in = (lane + 64 * i) / per == g;
          same += __builtin_popcountll(__ballot(in && key[i] == best));
          if (in && key[i] < best && key[i] > second) second = key[i];
        }
        second = route_max64(second);
        if (same > 1) second = best;
      }
      if (lane == g) value = route_key64(number(best) + (second != 0 ? number(second) : 0.0));
    }
    uint64_t kept = 0;
    for (int n = 0; n < top_groups; ++n) {
      const uint64_t m = route_max64(value);
      if (m == 0) break;
      const int g = __builtin_ctzll(__ballot(value == m));
      kept |= 1ull << g;
      if (lane == g) value = 0;
    }
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (lane + 64 * i < E && !(kept >> ((lane + 64 * i) / per) & 1)) key[i] = 0;
  }
  if (even) {
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (key[i] != 0) key[i] = route_key64((double)v[i]);
  }
  int mine = -1;
  for (int j = 0; j < k; ++j) {
    uint64_t m = key[0];
#pragma unroll
    for (int i = 1; i < P; ++i) m = key[i] > m ? key[i] : m;
    m = route_max64(m);
    if (m == 0) break;
    int e = -1;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint64_t hit = __ballot(key[i] == m);
      if (e < 0 && hit) e = 64 * i + __builtin_ctzll(hit);
    }
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (lane + 64 * i == e) key[i] = 0;
    if (lane == j) mine = e;
  }
  return mine;
}

// Two numbers of 32 bits whose order, as numbers of 64, they leave open.  A sigmoid
// is off by 2^-22 (its exponential's error counts a quarter at most, the sum, the
// reciprocal and the bias come to it), the scores of a softmax, which add up to 1,
// by 2^-20 all together; with its bias each is rounded once more.
DEV bool route_close(uint32_t larger, uint32_t smaller) {
  const float x = route_value(larger), d = x - route_value(smaller);
  return !(d > 0x1p-18f * __builtin_fmaxf(1.0f, __builtin_fabsf(x)));
}

// The k largest of key (0: none there), the largest first, ties by index.  Lane j
// returns index j, or -1.  MORE: and those after them, up to the first that is not
// close to the one before; n of them, lane j has the key too; n = 65 if 64 do not end.
template <int P, bool MORE>
DEV int route_best(uint32_t (&key)[P], int k, uint32_t& has, int& n) {
  int mine = -1;
  uint32_t before = 0;
  has = 0;
  for (n = 0; MORE || n < k; ++n) {
    uint32_t m = key[0];
#pragma unroll
    for (int i = 1; i < P; ++i) m = umax(m, key[i]);
    m = route_max(m);
    if (m == 0) break;
    if constexpr (MORE) {
      if (n >= k && !route_close(before, m)) break;
      if (n == 64) {
        n = 65;
        break;
      }
      before = m;
    }
    // (the lowest i that has it, and its lowest lane)
    uint64_t hit = __ballot(key[P - 1] == m);
    int at = P - 1;
#pragma unroll
    for (int i = P - 2; i >= 0; --i) {
      const uint64_t h = __ballot(key[i] == m);
      at = h ? i : at;
      hit = h ? h : hit;
    }
    const int l = __builtin_ctzll(hit);
    const uint64_t one = 1ull << l, me = 1ull << n;
#pragma unroll
    for (int i = 0; i < P; ++i) key[i] = __builtin_amdgcn_inverse_ballot_w64(at == i ? one : 0ull) ? 0u : key[i];
    mine = __builtin_amdgcn_inverse_ballot_w64(me) ? 64 * at + l : mine;
    if constexpr (MORE) has = __builtin_amdgcn_inverse_ballot_w64(me) ? m : has;
  }
  return mine;
}

// The first n experts in the order of 64 bits: lane j has one, and gets the one of place j.
template <int DT, int P>
DEV int route_settle(const RouteArgs& a, int64_t t, const float (&v)[P], int mine, int n) {
  const int lane = threadIdx.x & 63;
  const bool on = lane < n;
  const double x = on ? (double)route_load<DT>(a.logits, t * a.ld + mine) : 0.0;
  double c;
  if (a.sigmoid) {
    c = 1.0 / (1.0 + exp(-x));
  } else {
    float top = v[0];
    double sum = 0.0;
#pragma unroll
    for (int i = 1; i < P; ++i) top = __builtin_fmaxf(top, v[i]);
    top = route_fmax(top);
#pragma unroll
    for (int i = 0; i < P; ++i) sum += v[i] == -INFINITY ? 0.0 : exp((double)v[i] - (double)top);
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
    c = exp(x - (double)top) * (1.0 / sum);
  }
  if (a.bias && on) c += (double)a.bias[mine];
  const uint64_t key = route_key64(c);
  int place = 0;
  for (int i = 0; i < n; ++i) {
    const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)key, i);
    const int e = __builtin_amdgcn_readlane(mine, i);
    place += o > key || (o == key && e < mine);
  }
  return __builtin_amdgcn_ds_permute((on ? place : lane) * 4, mine);
}

// best and second best of a group, joined with those of the lanes that CTRL reads
template <int CTRL>
DEV void route_two(float& one, float& two) {
  const float o1 = u2f(route_dpp<CTRL, 0xf>(f2u(one))), o2 = u2f(route_dpp<CTRL, 0xf>(f2u(two)));
  two = __builtin_fmaxf(__builtin_fmaxf(two, o2), __builtin_fminf(one, o1));
  one = __builtin_fmaxf(one, o1);
}

// The choice.  Without a bias it follows the logits themselves; with one it is made
// in 32 bits, and where numbers that decide are close (`open`), in 64: among the chosen
// and those next to them, or, where groups are close, all of it.  That is what LATE
// does, and does it apart from the rest: with its registers the kernel runs 5 waves a
// SIMD instead of 8, and one token in 300 needs it.  (A bias that is the same for all is
// one too: far logits are the same number beside it, and the lowest index has them.  Its
// choices are close where logits are equal: 8192 tokens, 64 experts, bf16 logits 19.9 us
// with a bias of zeros, 16.2 with another, 11.6 without.)
template <int DT, int P, bool LATE>
DEV int route_choose(const RouteArgs& a, int64_t t, const float (&v)[P], const float (&b)[P], float* lds, bool& open) {
  const int lane = threadIdx.x & 63;
  const bool even = !a.bias;  // the logits' order
  const bool in_groups = a.top_groups < a.groups, sums = in_groups && a.group_best == 2;
  float c[P];
  if (!even || sums) {
    float s[P];
    route_scores<float, true, P>(v, a.sigmoid, s);
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = v[i] == -INFINITY ? -INFINITY : s[i] + b[i];
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = v[i];
  }
  uint32_t key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) key[i] = c[i] == -INFINITY ? 0u : route_key(even ? v[i] : c[i]);
  open = false;
  if (in_groups) {
    // a.lanes lanes look at a group, each at a part of its members; its two best are joined among them
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (lane + 64 * i < a.E) lds[lane + 64 * i] = c[i] == c[i] ? c[i] : INFINITY;
    __builtin_amdgcn_wave_barrier();
    const int g = lane / a.lanes, part = lane & (a.lanes - 1);
    float one = -INFINITY, two = -INFINITY;
    auto take = [&](float y) {
      two = __builtin_fmaxf(two, __builtin_fminf(one, y));
      one = __builtin_fmaxf(one, y);
    };
    if (g < a.groups) {
      if (a.per % 4 == 0) {
        for (int m = part * 4; m < a.per; m += a.lanes * 4) {
          const v4f32 y = *(const v4f32*)(lds + g * a.per + m);
#pragma unroll
          for (int i = 0; i < 4; ++i) take(y[i]);
        }
      } else {
        for (int m = part; m < a.per; m += a.lanes) take(lds[g * a.per + m]);
      }
    }
    __builtin_amdgcn_wave_barrier();
    if (a.lanes > 1) route_two<0xB1>(one, two);   // lane xor 1
    if (a.lanes > 2) route_two<0x4E>(one, two);   // lane xor 2
    if (a.lanes > 4) route_two<0x141>(one, two);  // 7 - lane, of 8 lanes
    if (a.lanes > 8) route_two<0x140>(one, two);  // 15 - lane, of 16
    for (int m = 16; m < a.lanes; m <<= 1) {
      const float o1 = __shfl_xor(one, m), o2 = __shfl_xor(two, m);
      two = __builtin_fmaxf(__builtin_fmaxf(two, o2), __builtin_fminf(one, o1));
      one = __builtin_fmaxf(one, o1);
    }
    const float sum = sums && two > -INFINITY ? one + two : one;
    uint32_t value = part == 0 && one > -INFINITY ? route_key(sum) : 0u;
    uint64_t kept = 0;
    uint32_t last = 0;
    for (int n = 0; n < a.top_groups; ++n) {
      last = route_max(value);
      if (last == 0) break;
      const uint64_t l = __ballot(value == last), first = l & (0 - l);
      kept |= first;
      value = __builtin_amdgcn_inverse_ballot_w64(first) ? 0u : value;
    }
    if ((!even || sums) && last != 0) {
      // A value is off by its addends' errors, whatever they cancel to: at most 2^-20 and a
      // rounding of 2^-24 of each addend and of the sum, below 2^-19 of their size.  The order
      // is left open if a kept group may be below one that is not.
      const float size = sums && two > -INFINITY ? __builtin_fabsf(one) + __builtin_fabsf(two) : __builtin_fabsf(one);
      const float off = 0x1p-19f * __builtin_fmaxf(1.0f, size);
      const uint32_t low = route_max(__builtin_amdgcn_inverse_ballot_w64(kept) ? route_key(off - sum) : 0u);  // (minus the least)
      const uint32_t high = route_max(value != 0 ? route_key(off + sum) : 0u);
      open = high != 0 && !(-route_value(low) > route_value(high));
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int of = (int)((uint32_t)(lane + 64 * i) * a.per_mul >> 20) * a.lanes;
      if (!(kept >> (of & 63) & 1)) key[i] = 0;
    }
  }
  uint32_t has;
  int n, mine = -1;
  if (!open && even) return route_best<P, false>(key, a.k, has, n);
  bool close = false;
  if (!open) {
    mine = route_best<P, true>(key, a.k, has, n);
    const uint32_t before = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)has, 0x138, 0xf, 0xf, false);  // of the lane below
    open = n > 64;
    close = __ballot(lane > 0 && lane < n && route_close(before, has)) != 0;
  }
  if constexpr (LATE) {
    if (open) mine = route_choose64<P>(v, b, even, a.E, a.k, a.sigmoid, a.groups, a.per, a.top_groups, a.group_best);
    else if (close) mine = route_settle<DT, P>(a, t, v, mine, n);
  }
  open = open || close;
  return lane < a.k ? mine : -1;
}

// One token: its choice, weights, and in ent its choice once more (E: none).  False,
// and nothing done, where the choice is left to LATE.
template <int DT, int P, bool LATE>
DEV bool route_token(const RouteArgs& a, int64_t t, const float (&b)[P], float* row, uint16_t* ent) {
  const int lane = threadIdx.x & 63;
  float v[P];
#pragma unroll
  for (int i = 0; i < P; ++i) v[i] = lane + 64 * i < a.E ? route_load<DT>(a.logits, t * a.ld + lane + 64 * i) : -INFINITY;
  bool open;
  const int mine = route_choose<DT, P, LATE>(a, t, v, b, row, open);
  if (!LATE && open) return false;
  // the chosen experts' logits: e^x of softmax, e^min(x, 0) / (1 + e^-|x|) of sigmoid, so that none overflows
  const bool on = mine >= 0;
  const float x = on ? route_load<DT>(a.logits, t * a.ld + mine) : 0.0f;
  const float e = a.sigmoid ? (x < 0.0f ? x : 0.0f) : x, q = a.sigmoid ? 1.0f / (1.0f + expf(-__builtin_fabsf(x))) : 1.0f;
  float w;
  if (a.renormalize) {
    const float top = route_fmax(on ? e : -INFINITY), r = on ? expf(e - top) * q : 0.0f;
    w = a.scale * (r / route_sum(r));
  } else if (a.sigmoid) {
    w = a.scale * (expf(e) * q);
  } else {
    float top = v[0], z = 0.0f;
#pragma unroll
    for (int i = 1; i < P; ++i) top = __builtin_fmaxf(top, v[i]);
    top = route_fmax(top);
#pragma unroll
    for (int i = 0; i < P; ++i) z += v[i] == -INFINITY ? 0.0f : expf(v[i] - top);
    w = a.scale * (expf(x - top) / route_sum(z));
  }
  bool bad = false;
#pragma unroll
  for (int i = 0; i < P; ++i) bad = bad || v[i] != v[i] || (!a.sigmoid && v[i] == INFINITY);
  if (__ballot(bad)) w = NAN;
  if (lane < a.k) {
    a.weight[t * a.k + lane] = on ? w : 0.0f;
    a.expert[t * a.k + lane] = mine;
    ent[lane] = (uint16_t)(on ? mine : a.E);
  }
  return true;
}
// The lane's biases.
template <int P>
DEV void route_bias(const RouteArgs& a, float (&b)[P]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < P; ++i) b[i] = a.bias && lane + 64 * i < a.E ? a.bias[lane + 64 * i] : 0.0f;
}
// A call, so that its registers are not the loop's.
template <int DT, int P>
__device__ __attribute__((noinline)) void route_late(const RouteArgs* a, int64_t t, float* row, uint16_t* ent) {
  float b[P];
  route_bias<P>(*a, b);
  route_token<DT, P, true>(*a, t, b, row, ent);
}

// A workgroup has a.block tokens, a wave one of them at a time.  Ranks of its choices
// among those of the same expert go to a.position, the numbers of its choices to
// a.counts and a.none: k_route_place makes places of them.  One workgroup alone has
// everything itself.
template <int P>
constexpr int ROUTE_THREADS = P <= 4 ? 1024 : 512;  // (registers)
template <int DT, int P>
__global__ __launch_bounds__(ROUTE_THREADS<P>, P <= 4 ? 8 : P <= 8 ? 4 : 2) void k_route(RouteArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index();
  constexpr int threads = ROUTE_THREADS<P>, waves = threads / 64;
  // this wave's scores, if there are groups; counts of the experts; this workgroup's choices and their ranks
  float* const row = (float*)lds + wave * a.pitch;
  uint32_t* const count = lds + (a.top_groups < a.groups ? waves * a.pitch : 0);
  uint16_t* const ent = (uint16_t*)(count + a.E + 1);
  uint16_t* const rank = ent + a.block * a.k;
  const int64_t t0 = (int64_t)blockIdx.x * a.block;
  const int tokens = (int)(a.T - t0 < a.block ? a.T - t0 : a.block), n = tokens * a.k;
  for (int i = tid; i <= a.E; i += threads) count[i] = 0;
  float b[P];
  route_bias<P>(a, b);
  uint32_t left = 0;  // of this wave's tokens, at most 8
  for (int i = 0, tl = wave; tl < tokens; ++i, tl += waves)
    if (!route_token<DT, P, false>(a, t0 + tl, b, row, ent + tl * a.k)) left |= 1u << i;
  const RouteArgs* const args = (const RouteArgs*)__builtin_amdgcn_kernarg_segment_ptr();  // (the kernel's one argument)
  for (; left; left &= left - 1) {
    const int tl = wave + __builtin_ctz(left) * waves;
    route_late<DT, P>(args, t0 + tl, row, ent + tl * a.k);
  }
  __syncthreads();
  // ranks among the choices of one expert, 64 choices a wave, one wave after the other
  const int bits = 32 - __builtin_clz(a.E), chunks = (n + 63) >> 6;
  for (int c0 = 0; c0 < chunks; c0 += waves) {
    const int i = (c0 + wave) * 64 + lane;
    const bool in = i < n;
    const uint32_t e = in ? ent[i] : 0u;
    uint64_t same = __ballot(in);
    for (int bit = 0; bit < bits; ++bit) {
      const bool one = e >> bit & 1;
      const uint64_t with = __ballot(one);
      same &= one ? with : ~with;
    }
    for (int w = 0; w < waves && c0 + w < chunks; ++w) {
      if (w == wave && in) {
        const uint32_t before = count[e], to = before + __builtin_popcountll(same & ((1ull << lane) - 1));
        if (a.blocks > 1) a.position[t0 * a.k + i] = (int32_t)to;
        else rank[i] = (uint16_t)to;
        __builtin_amdgcn_wave_barrier();
        if (same >> lane == 1) count[e] = before + __builtin_popcountll(same);
      }
      __syncthreads();
    }
  }
  if (a.blocks > 1) {  // (an expert has at most one choice of a token)
    for (int i = tid; i < a.pitch; i += threads) a.counts[(int64_t)blockIdx.x * a.pitch + i] = i < a.E ? (uint8_t)count[i] : (uint8_t)0;
    if (tid == 0) a.none[blockIdx.x] = count[a.E];
    return;
  }
  if (wave == 0) {
    uint32_t before = 0;
    for (int c = 0; c <= a.E; c += 64) {
      const int e = c + lane;
      const uint32_t x = e <= a.E ? count[e] : 0, sum = (uint32_t)lin_scan_add((int)x);
      if (e <= a.E) count[e] = before + sum - x;
      if (e < a.E) a.ends[e] = (int32_t)(before + sum);
      before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += threads) a.position[i] = (int32_t)(count[ent[i]] + rank[i]);
}

// Many workgroups: the choices of those before each, per expert (and without one).
// 16 experts a workgroup, 64 threads for each, which take a run of the workgroups,
// 16 at a time in registers.
__global__ __launch_bounds__(1024) void k_route_scan(RouteArgs a) {
  __shared__ uint32_t part[16][65];
  const int c = threadIdx.x & 15, seg = threadIdx.x >> 4, e = blockIdx.x * 16 + c, cols = a.E + 1, lane = threadIdx.x & 63;
  const int each = (a.blocks + 63) / 64, b0 = seg * each, b1 = b0 + each < a.blocks ? b0 + each : a.blocks;
  uint32_t x[16], sum = 0;
  auto load = [&](int b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool in = b + i < b1;
      x[i] = in && e < a.E ? ((const LM_GLOBAL uint8_t*)a.counts)[(int64_t)(b + i) * a.pitch + e]
             : in && e == a.E ? ((const LM_GLOBAL uint32_t*)a.none)[b + i] : 0u;
    }
  };
  for (int b = b0; b < b1; b += 16) {
    load(b);
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += x[i];
  }
  part[c][seg] = sum;
  __syncthreads();
  // (a wave scans an expert's 64 sums)
  {
    const int w = threadIdx.x >> 6;
    const uint32_t y = part[w][lane], z = (uint32_t)lin_scan_add((int)y);
    part[w][lane] = z - y;
    if (lane == 63 && blockIdx.x * 16 + w < cols) ((LM_GLOBAL uint32_t*)a.starts)[(int64_t)a.blocks * cols + blockIdx.x * 16 + w] = z;
  }
  __syncthreads();
  uint32_t before = part[c][seg];
  for (int b = b0; b < b1; b += 16) {
    if (each > 16) load(b);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (e < cols && b + i < b1) {
        ((LM_GLOBAL uint32_t*)a.starts)[(int64_t)(b + i) * cols + e] = before;
        before += x[i];
      }
  }
}

// exclusive sums over the experts, by one wave; their ends
DEV void route_first(const uint32_t* total, uint32_t* first, int E, int32_t* ends) {
  const int lane = threadIdx.x & 63;
  uint32_t before = 0;
  for (int c = 0; c <= E; c += 64) {
    const int e = c + lane;
    const uint32_t x = e < E ? total[e] : 0, sum = (uint32_t)lin_scan_add((int)x);
    if (e <= E) first[e] = before + sum - x;
    if (e < E && ends) ends[e] = (int32_t)(before + sum);
    before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
}

__global__ __launch_bounds__(256) void k_route_place_far(RouteArgs a, int64_t n) {
  extern __shared__ uint32_t first[];  // choices of the experts before each
  const int cols = a.E + 1;
  if (threadIdx.x < 64) route_first(a.starts + (int64_t)a.blocks * cols, first, a.E, blockIdx.x == 0 ? a.ends : nullptr);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = (int64_t)blockIdx.x * 1024 + j * 256 + threadIdx.x;
    if (i < n) {
      const int32_t x = a.expert[i], e = x < 0 ? a.E : x;
      const uint32_t b = div_by(a.entries, (uint32_t)i);
      a.position[i] = (int32_t)(first[e] + a.starts[(int64_t)b * cols + e] + (uint32_t)a.position[i]);
    }
  }
}

// Places of the choices of four workgroups of k_route.  Every workgroup adds up all
// the counts (a byte each: 128 KB for 16384 tokens and 256 experts, from the L2)
// instead of waiting for a launch that does it once.  Bound by the latency of its
// loads, so what does not depend on the sums is asked for first.
__global__ __launch_bounds__(1024) void k_route_place(RouteArgs a) {
  __shared__ uint32_t total[1024], first[1028], start[4][1028];
  __shared__ uint32_t none;
  const int tid = threadIdx.x, b0 = blockIdx.x * 4, blocks = a.blocks - b0 < 4 ? a.blocks - b0 : 4;
  const int64_t i0 = (int64_t)b0 * a.block * a.k, all = a.T * a.k - i0;
  const int n = (int)(all < 4 * a.block * a.k ? all : 4 * a.block * a.k);
  const LM_GLOBAL uint8_t* const counts = (const LM_GLOBAL uint8_t*)a.counts;
  const LM_GLOBAL int32_t* const expert = (const LM_GLOBAL int32_t*)a.expert + i0;
  LM_GLOBAL int32_t* const position = (LM_GLOBAL int32_t*)a.position + i0;
  int32_t x0 = 0, p0 = 0;
  if (tid < n) {
    x0 = expert[tid];
    p0 = position[tid];
  }
  uint32_t own[4], without[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    own[i] = tid < a.E && i < blocks ? counts[(int64_t)(b0 + i) * a.pitch + tid] : 0u;
    without[i] = tid == 0 && i < blocks ? a.none[b0 + i] : 0u;
  }
  for (int i = tid; i < b0; i += 1024) mine += a.none[i];
  total[tid] = start[0][tid] = 0;
  if (tid == 0) none = 0;
  __syncthreads();
  if (mine) atomicAdd(&none, mine);
  const int words = a.pitch >> 2, shift = words <= 1 ? 0 : 32 - __builtin_clz(words - 1), w = tid & ((1 << shift) - 1), step = 1024 >> shift;
  if (w < words) {
    uint32_t t0 = 0, t1 = 0, s0 = 0, s1 = 0;  // of two experts each, in 16 bits: at most ROUTE_NEAR tokens
    const LM_GLOBAL uint32_t* const at = (const LM_GLOBAL uint32_t*)a.counts + w;
    for (int r0 = tid >> shift; r0 < a.blocks; r0 += step * 16) {
      uint32_t x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = r0 + i * step < a.blocks ? at[(int64_t)(r0 + i * step) * words] : 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t even = x[i] & 0x00ff00ffu, odd = x[i] >> 8 & 0x00ff00ffu;
        const bool in = r0 + i * step < b0;
        t0 += even;
        t1 += odd;
        s0 += in ? even : 0u;
        s1 += in ? odd : 0u;
      }
    }
    const uint32_t t[4] = {t0 & 0xffffu, t1 & 0xffffu, t0 >> 16, t1 >> 16}, s[4] = {s0 & 0xffffu, s1 & 0xffffu, s0 >> 16, s1 >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t[i]) atomicAdd(&total[4 * w + i], t[i]);
      if (s[i]) atomicAdd(&start[0][4 * w + i], s[i]);
    }
  }
  __syncthreads();
  if (tid < 64) route_first(total, first, a.E, blockIdx.x == 0 ? a.ends : nullptr);
  __syncthreads();
  if (tid < a.E) {
    uint32_t x = first[tid] + start[0][tid];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      start[i][tid] = x;
      x += own[i];
    }
  }
  if (tid == 0) {
    uint32_t x = first[a.E] + none;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      start[i][a.E] = x;
      x += without[i];
    }
  }
  __syncthreads();
  auto place = [&](int i, int32_t x, int32_t p) {
    position[i] = (int32_t)start[div_by(a.entries, (uint32_t)i)][x < 0 ? a.E : x] + p;
  };
  if (tid < n) place(tid, x0, p0);
  for (int i = tid + 1024; i < n; i += 1024) place(i, expert[i], position[i]);
}

// The gradient to the logits, a wave a token: 8192 tokens, 64 experts 4.8 us, most of it
// a launch's ends.  g = d loss / d w, for the chosen experts j:
//   renormalised   w_j (g_j - sum_i g_i w_i / scale), for sigmoid times 1 - p_j
//   sigmoid        w_j g_j (1 - p_j)
//   softmax        w_j g_j - p_e sum_i g_i w_i, the second term for every expert e
template <int DT, int P>
__global__ __launch_bounds__(256) void k_route_grad(RouteArgs a, const float* dweight, void* out) {
  const int lane = threadIdx.x & 63;
  for (int64_t t = (int64_t)blockIdx.x * 4 + wave_index(); t < a.T; t += (int64_t)gridDim.x * 4) {
    int mine = lane < a.k ? a.expert[t * a.k + lane] : -1;
    const bool on = mine >= 0 && mine < a.E;
    const float g = on ? dweight[t * a.k + lane] : 0.0f;
    const float x = on ? route_load<DT>(a.logits, t * a.ld + mine) : 0.0f;
    const float e = a.sigmoid ? (x < 0.0f ? x : 0.0f) : x, z = expf(-__builtin_fabsf(x));
    const float q = a.sigmoid ? 1.0f / (1.0f + z) : 1.0f;
    const float rest = a.sigmoid ? (x < 0.0f ? 1.0f : z) * q : 1.0f;  // 1 - p of sigmoid
    float d[P] = {}, mine_d;
    if (a.renormalize) {
      const float top = route_fmax(on ? e : -INFINITY), r = on ? expf(e - top) * q : 0.0f, p = r / route_sum(r);
      const float mean = route_sum(on ? g * p : 0.0f);
      mine_d = a.scale * p * (g - mean) * rest;
    } else if (a.sigmoid) {
      mine_d = a.scale * (expf(e) * q) * g * rest;
    } else {
      float v[P], s[P];
#pragma unroll
      for (int i = 0; i < P; ++i) v[i] = lane + 64 * i < a.E ? route_load<DT>(a.logits, t * a.ld + lane + 64 * i) : -INFINITY;
      route_scores<float, false, P>(v, false, s);
      float p = 0.0f;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float o = __shfl(s[i], mine & 63);
        if (mine >> 6 == i) p = o;
      }
      mine_d = a.scale * p * g;
      const float sum = route_sum(on ? mine_d : 0.0f);
#pragma unroll
      for (int i = 0; i < P; ++i) d[i] = v[i] == -INFINITY ? 0.0f : -s[i] * sum;
    }
    for (uint64_t left = __ballot(on); left; left &= left - 1) {
      const int j = __builtin_ctzll(left), to = __builtin_amdgcn_readlane(mine, j);
      const float add = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(mine_d), j));
#pragma unroll
      for (int i = 0; i < P; ++i) d[i] += lane + 64 * i == to ? add : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int64_t at = t * a.E + lane + 64 * i;
      if (lane + 64 * i < a.E) {
        if constexpr (DT == F32) ((float*)out)[at] = d[i];
        else ((uint16_t*)out)[at] = bits_dt<DT>(d[i]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// rows to their experts, and back as weighted sums
// ---------------------------------------------------------------------------
struct RowsArgs {
  const void* x;  // rows of tokens [T, ld]
  int64_t ld;
  const void* h;  // rows of choices [T k, ldh]
  int64_t ldh;
  const float* weight;      // [T, k]
  const int32_t* position;  // [T, k]
  const int32_t* ends;      // [E]
  void* out;
  float* dweight;
  int64_t T, N;
  int E, k;
};

// choices from this place on have no expert
DEV int rows_end(const RowsArgs& a) {
  const int end = a.ends[a.E - 1];
  const int64_t n = a.T * a.k;
  return end < 0 ? 0 : (end > n ? (int)n : end);
}
// NT: past the caches
template <bool NT>
DEV void rows_store(uint16_t* p, lm_u32x4 w, int64_t left) {
  if (left >= 8) {
    if constexpr (NT) __builtin_nontemporal_store(w, (LM_GLOBAL lm_u32x4_any*)p);
    else *(LM_GLOBAL lm_u32x4_any*)p = w;
    asm volatile("s_nop 1" ::"v"(w) : "memory");  // (store_b128_guarded)
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < left) ((LM_GLOBAL uint16_t*)p)[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
  }
}

// 8 values of each of M rows, `left` of which exist; all of them before the first is used.
//
// Rows of choices go past the caches, both ways: there are top_k of them for every
// row of a token, and each is read or written once (8192 x 2048, four choices, by
// themselves: rows out 34 -> 26 us, back 33 -> 28, gradients 58 -> 48).  Rows of tokens do
// not: with both past the caches rows out take 31 us, gradients 53.  Bound by memory: called
// in turn with others 26 us out (6.4 TB/s), 29 to 30 back (5.7), 53 to 54 the gradients (5.6),
// where a copy reaches 5.1 to 6.1.
template <bool NT, int M>
DEV void rows_load(lm_u32x4 (&w)[M], const uint16_t* const (&p)[M], int64_t left) {
  if (left >= 8) {
#pragma unroll
    for (int n = 0; n < M; ++n) w[n] = NT ? __builtin_nontemporal_load((const LM_GLOBAL lm_u32x4_any*)p[n]) : *(const LM_GLOBAL lm_u32x4_any*)p[n];
  } else {
#pragma unroll
    for (int n = 0; n < M; ++n) w[n] = lin_chunk(p[n], left);
  }
}

// Where a wave works: WPT waves (1, or all 4 of the workgroup) have a token, 512
// columns each and the next ones after that; blockIdx.y shares the columns out.
template <int WPT>
struct RowsAt {
  int64_t t, next, c0, step;
  DEV RowsAt() {
    t = WPT == 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave_index();
    next = (int64_t)gridDim.x * (WPT == 4 ? 1 : 4);
    c0 = ((int64_t)blockIdx.y * WPT + (WPT == 4 ? wave_index() : 0)) * 512 + (threadIdx.x & 63) * 8;
    step = (int64_t)gridDim.y * WPT * 512;
  }
};
// the places of choices j0 .. j0 + 3 of a token; -1: not one of those below `end`
DEV void rows_places(const RowsArgs& a, int64_t t, int j0, int end, int (&p)[4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    p[n] = j0 + n < a.k ? a.position[t * a.k + j0 + n] : -1;
    if (p[n] >= end) p[n] = -1;
  }
}

template <int WPT>
__global__ __launch_bounds__(256) void k_rows_out(RowsArgs a) {
  RowsAt<WPT> at;
  const int end = rows_end(a), all = (int)(a.T * a.k);
  for (; at.t < a.T; at.t += at.next)
    for (int64_t c = at.c0; c < a.N; c += at.step) {
      lm_u32x4 w[1];
      const uint16_t* const p[1] = {(const uint16_t*)a.x + at.t * a.ld + c};
      rows_load<false>(w, p, a.N - c);
      for (int j = 0; j < a.k; ++j) {
        const int to = a.position[at.t * a.k + j];
        if (to < 0 || to >= all) continue;
        rows_store<true>((uint16_t*)a.out + to * a.N + c, to < end ? w[0] : lm_u32x4{}, a.N - c);
      }
    }
}

template <int DT, bool WEIGHTS, int WPT>
__global__ __launch_bounds__(256) void k_rows_back(RowsArgs a) {
  RowsAt<WPT> at;
  const int end = rows_end(a);
  for (; at.t < a.T; at.t += at.next)
    for (int64_t c = at.c0; c < a.N; c += at.step) {
      float s[8] = {};
      for (int j0 = 0; j0 < a.k; j0 += 4) {
        int p[4];
        rows_places(a, at.t, j0, end, p);
        lm_u32x4 w[4];
        const uint16_t* from[4];  // (row 0 instead of none: it is there)
        float by[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          from[n] = (const uint16_t*)a.h + (p[n] < 0 ? 0 : p[n]) * a.ldh + c;
          by[n] = WEIGHTS && p[n] >= 0 ? a.weight[at.t * a.k + j0 + n] : 1.0f;
        }
        rows_load<true>(w, from, a.N - c);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          if (p[n] < 0) continue;
#pragma unroll
          for (int i = 0; i < 8; ++i) s[i] = __builtin_fmaf(by[n], val_dt<DT>(i & 1 ? w[n][i >> 1] >> 16 : w[n][i >> 1] & 0xffffu), s[i]);
        }
      }
      lm_u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (uint32_t)bits_dt<DT>(s[2 * i]) | (uint32_t)bits_dt<DT>(s[2 * i + 1]) << 16;
      rows_store<false>((uint16_t*)a.out + at.t * a.N + c, w, a.N - c);
    }
}

// Gradients of the weighted sums, for four choices of a token at a time.
template <int DT, int WPT>
__global__ __launch_bounds__(256) void k_rows_back_grad(RowsArgs a) {
  __shared__ float red[4][4];
  RowsAt<WPT> at;
  const int end = rows_end(a), all = (int)(a.T * a.k), lane = threadIdx.x & 63;
  for (; at.t < a.T; at.t += at.next)  // (with WPT 4 the same for all waves)
    for (int j0 = 0; j0 < a.k; j0 += 4) {
      int p[4], to[4];
      rows_places(a, at.t, j0, all, to);
      rows_places(a, at.t, j0, end, p);
      float by[4], sum[4] = {};
#pragma unroll
      for (int n = 0; n < 4; ++n) by[n] = p[n] < 0 ? 0.0f : a.weight[at.t * a.k + j0 + n];
      for (int64_t c = at.c0; c < a.N; c += at.step) {
        lm_u32x4 w[4], dy[1];
        const uint16_t* from[4];
        const uint16_t* const x[1] = {(const uint16_t*)a.x + at.t * a.ld + c};
#pragma unroll
        for (int n = 0; n < 4; ++n) from[n] = (const uint16_t*)a.h + (p[n] < 0 ? 0 : p[n]) * a.ldh + c;
        rows_load<false>(dy, x, a.N - c);
        rows_load<true>(w, from, a.N - c);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          lm_u32x4 dh = {};
          if (p[n] >= 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float lo = val_dt<DT>(dy[0][i] & 0xffffu), hi = val_dt<DT>(dy[0][i] >> 16);
              sum[n] = __builtin_fmaf(lo, val_dt<DT>(w[n][i] & 0xffffu), sum[n]);
              sum[n] = __builtin_fmaf(hi, val_dt<DT>(w[n][i] >> 16), sum[n]);
              dh[i] = (uint32_t)bits_dt<DT>(by[n] * lo) | (uint32_t)bits_dt<DT>(by[n] * hi) << 16;
            }
          }
          if (to[n] >= 0) rows_store<true>((uint16_t*)a.out + to[n] * a.N + c, dh, a.N - c);
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) sum[n] = route_sum(sum[n]);
      if constexpr (WPT == 4) {
        __syncthreads();  // (the sums before these are read)
        if (lane == 0) {
#pragma unroll
          for (int n = 0; n < 4; ++n) red[n][wave_index()] = sum[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < 4; ++n) sum[n] = red[n][0] + red[n][1] + red[n][2] + red[n][3];
      }
      if (threadIdx.x == 0 || (WPT == 1 && lane == 0)) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (j0 + n < a.k) a.dweight[at.t * a.k + j0 + n] = p[n] < 0 ? 0.0f : sum[n];
      }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int64_t ROWS_GRID = 1 << 22;  // workgroups that take a token after the other (a launch has fewer than 2^32 threads)
constexpr int64_t ROUTE_TOKENS = (1 << 28) - 64;  // (k_route: 64 a workgroup of 1024 threads then)

static int check_route(const lm_route* r) {
  if (!r) return fail(LM_EINVAL, "routing needs its description");
  if (r->dtype != LM_F32 && r->dtype != LM_BF16 && r->dtype != LM_F16) return fail(LM_EUNSUPPORTED, "routing takes fp32, bf16 and fp16 logits");
  if (r->T < 0 || r->experts < 1 || r->experts > LM_LINEAR_MAX_EXPERTS)
    return fail(LM_EINVAL, "routing takes 1 to %d experts, got %d", LM_LINEAR_MAX_EXPERTS, r->experts);
  if (r->score != LM_ROUTE_SOFTMAX && r->score != LM_ROUTE_SIGMOID) return fail(LM_EINVAL, "unknown score");
  if (r->groups < 1 || r->groups > LM_ROUTE_MAX_GROUPS || r->experts % r->groups != 0)
    return fail(LM_EINVAL, "experts must divide into 1 to %d groups, got %d in %d", LM_ROUTE_MAX_GROUPS, r->experts, r->groups);
  if (r->top_groups < 1 || r->top_groups > r->groups) return fail(LM_EINVAL, "top_groups must be 1 to the number of groups");
  if (r->group_best < 1 || r->group_best > 2 || r->group_best > r->experts / r->groups)
    return fail(LM_EINVAL, "group_best must be 1 or 2 and at most the experts of a group");
  if (r->top_k < 1 || r->top_k > LM_ROUTE_MAX_BEST || r->top_k > r->top_groups * (r->experts / r->groups))
    return fail(LM_EINVAL, "top_k must be 1 to %d and at most the experts of the kept groups", LM_ROUTE_MAX_BEST);
  if (r->T > ROUTE_TOKENS || r->T * r->top_k > 0x7fffffff) return fail(LM_EUNSUPPORTED, "more than 2^28 - 64 tokens or 2^31 - 1 choices");
  if (r->T > 0 && !r->logits) return fail(LM_EINVAL, "logits must be non-null");
  if (r->ld < r->experts) return fail(LM_EINVAL, "row stride below the row length");
  return LM_OK;
}

// Waves of a workgroup of k_route (ROUTE_THREADS)
static int route_waves(int64_t experts) { return experts <= 256 ? 16 : 8; }
// Tokens of a workgroup: all of them while they are few, so that one launch does; one
// a wave up to 4096 tokens, then two (8192 tokens, 64 experts: as fast as one), and more
// where k_route_place would add up the counts of more than 1024 workgroups.
static int route_block(int64_t T, int64_t experts) {
  if (T <= 32) return (int)T;
  const int waves = route_waves(experts);
  if (T <= 4096) return waves;
  int block = 2 * waves;
  while (block < 64 && T > (int64_t)block * 1024) block *= 2;
  return block;
}
static int64_t route_pitch(int64_t experts) { return (experts + 3) & ~(int64_t)3; }

struct RouteSpace {
  size_t none, starts, total;
};
static RouteSpace route_space(int64_t T, int64_t experts) {
  const int64_t block = route_block(T, experts), blocks = (T + block - 1) / block;
  RouteSpace s{};
  if (blocks <= 1) return s;
  s.none = align256((size_t)(blocks * route_pitch(experts)));
  s.starts = s.none + align256((size_t)blocks * 4);
  s.total = s.starts + (T > ROUTE_NEAR ? align256((size_t)(blocks + 1) * (size_t)(experts + 1) * 4) : 0);
  return s;
}

static RouteArgs route_args(const lm_route* r) {
  RouteArgs a{};
  a.logits = r->logits;
  a.ld = r->ld;
  a.bias = r->bias;
  a.T = r->T;
  a.E = r->experts;
  a.k = r->top_k;
  a.sigmoid = r->score == LM_ROUTE_SIGMOID;
  a.renormalize = r->renormalize != 0;
  a.scale = r->scale;
  a.groups = r->groups;
  a.top_groups = r->top_groups;
  a.group_best = r->group_best;
  a.per = r->experts / r->groups;
  a.lanes = 64;
  while (a.lanes * a.groups > 64) a.lanes >>= 1;
  a.per_mul = ((1u << 20) + a.per - 1) / a.per;
  a.block = a.T > 0 ? route_block(a.T, a.E) : 1;
  a.blocks = (int)((a.T + a.block - 1) / a.block);
  a.pitch = (int)route_pitch(a.E);
  a.entries = fast_div((uint32_t)(a.block * a.k));
  return a;
}

#define ROUTE_BY_WIDTH(KERNEL, DT, ...)                                                   \
  do {                                                                                    \
    if (a.E <= 64) hipLaunchKernelGGL((KERNEL<DT, 1>), __VA_ARGS__);                      \
    else if (a.E <= 128) hipLaunchKernelGGL((KERNEL<DT, 2>), __VA_ARGS__);                \
    else if (a.E <= 256) hipLaunchKernelGGL((KERNEL<DT, 4>), __VA_ARGS__);                \
    else if (a.E <= 512) hipLaunchKernelGGL((KERNEL<DT, 8>), __VA_ARGS__);                \
    else hipLaunchKernelGGL((KERNEL<DT, 16>), __VA_ARGS__);                               \
  } while (0)
#define ROUTE_BY_TYPE(KERNEL, ...)                                                        \
  do {                                                                                    \
    if (r->dtype == LM_F32) ROUTE_BY_WIDTH(KERNEL, F32, __VA_ARGS__);                     \
    else if (r->dtype == LM_F16) ROUTE_BY_WIDTH(KERNEL, F16, __VA_ARGS__);                \
    else ROUTE_BY_WIDTH(KERNEL, BF16, __VA_ARGS__);                                       \
  } while (0)

extern "C" size_t lm_route_workspace_size(int64_t T, int32_t experts) {
  if (T <= 0 || T > ROUTE_TOKENS || experts < 1 || experts > LM_LINEAR_MAX_EXPERTS) return 0;
  return route_space(T, experts).total;
}

extern "C" int lm_route_topk(const lm_route* r, float* weight, int32_t* expert, int32_t* position, int32_t* ends,
                             void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_route(r))) return rc;
  if (!ends || (r->T > 0 && (!weight || !expert || !position))) return fail(LM_EINVAL, "output pointers must be non-null");
  RouteArgs a = route_args(r);
  a.weight = weight;
  a.expert = expert;
  a.position = position;
  a.ends = ends;
  if (a.blocks > 1) {
    const size_t need = lm_route_workspace_size(a.T, a.E);
    if (!workspace || workspace_bytes < need)
      return fail(LM_EWORKSPACE, "workspace too small: %zu < %zu bytes", workspace ? workspace_bytes : 0, need);
    if (((uintptr_t)workspace & 255) != 0) return fail(LM_EINVAL, "workspace must be 256-byte aligned");
    const RouteSpace s = route_space(a.T, a.E);
    a.counts = (uint8_t*)workspace;
    a.none = (uint32_t*)((uint8_t*)workspace + s.none);
    a.starts = (uint32_t*)((uint8_t*)workspace + s.starts);
  }
  hipStream_t st = (hipStream_t)stream;
  TimedLaunch timed("route", st);
  const int threads = 64 * route_waves(a.E);
  const size_t lds = (a.top_groups < a.groups ? (size_t)threads / 64 * a.pitch * 4 : 0) + (size_t)(a.E + 1) * 4 + (size_t)a.block * a.k * 4;
  ROUTE_BY_TYPE(k_route, dim3((unsigned)(a.blocks > 0 ? a.blocks : 1)), dim3(threads), lds, st, a);
  LAUNCH_CHECK();
  if (a.blocks <= 1) return LM_OK;
  if (a.T <= ROUTE_NEAR) {
    hipLaunchKernelGGL(k_route_place, dim3((unsigned)((a.blocks + 3) / 4)), dim3(1024), 0, st, a);
    LAUNCH_CHECK();
    return LM_OK;
  }
  hipLaunchKernelGGL(k_route_scan, dim3((unsigned)((a.E + 16) / 16)), dim3(1024), 0, st, a);
  LAUNCH_CHECK();
  const int64_t n = a.T * a.k;
  hipLaunchKernelGGL(k_route_place_far, dim3((unsigned)((n + 1023) / 1024)), dim3(256), (size_t)(a.E + 1) * 4, st, a, n);
  LAUNCH_CHECK();
  return LM_OK;
}

extern "C" int lm_route_topk_grad(const lm_route* r, const float* dweight, const int32_t* expert, void* dlogits, void* stream) {
  int rc;
  if ((rc = check_route(r))) return rc;
  if (r->T == 0) return LM_OK;
  if (!dweight || !expert || !dlogits) return fail(LM_EINVAL, "pointers must be non-null");
  RouteArgs a = route_args(r);
  a.expert = (int32_t*)expert;
  hipStream_t st = (hipStream_t)stream;
  TimedLaunch timed("route", st);
  const int64_t n = (a.T + 3) / 4;
  ROUTE_BY_TYPE(k_route_grad, dim3((unsigned)(n < ROWS_GRID ? n : ROWS_GRID)), dim3(256), 0, st, a, dweight, dlogits);
  LAUNCH_CHECK();
  return LM_OK;
}

static int check_rows(const lm_rows* r) {
  if (!r) return fail(LM_EINVAL, "rows need their description");
  if (r->dtype != LM_BF16 && r->dtype != LM_F16) return fail(LM_EUNSUPPORTED, "rows are bf16 or fp16");
  if (r->T < 0 || r->N < 1 || r->top_k < 1 || r->experts < 1 || r->experts > LM_LINEAR_MAX_EXPERTS)
    return fail(LM_EINVAL, "empty rows, no choices or no experts");
  if (r->T * r->top_k > 0x7fffffff || r->N > 0x7fffffff) return fail(LM_EUNSUPPORTED, "more than 2^31 - 1 rows or columns");
  if (r->T > 0 && (!r->position || !r->ends)) return fail(LM_EINVAL, "positions and ends must be non-null");
  return LM_OK;
}
static RowsArgs rows_args(const lm_rows* r) {
  RowsArgs a{};
  a.position = r->position;
  a.ends = r->ends;
  a.T = r->T;
  a.N = r->N;
  a.E = r->experts;
  a.k = r->top_k;
  return a;
}
// Rows of up to 1024 columns are a wave's, longer ones a workgroup's; while there are
// few tokens the columns are shared out too (not where they are added up).
static bool rows_short(const RowsArgs& a) { return a.N <= 1024; }
static dim3 rows_grid(const RowsArgs& a, bool whole) {
  const int64_t x = rows_short(a) ? (a.T + 3) / 4 : a.T, parts = (a.N + 2047) / 2048;
  return dim3((unsigned)(x < ROWS_GRID ? x : ROWS_GRID), (unsigned)(whole || rows_short(a) || x >= 2048 ? 1 : parts < 64 ? parts : 64));
}

extern "C" int lm_dispatch_rows(const lm_rows* r, const void* x, int64_t ldx, void* out, void* stream) {
  int rc;
  if ((rc = check_rows(r))) return rc;
  if (r->T == 0) return LM_OK;
  if (!x || !out) return fail(LM_EINVAL, "row pointers must be non-null");
  if (ldx < r->N) return fail(LM_EINVAL, "row stride below the row length");
  RowsArgs a = rows_args(r);
  a.x = x;
  a.ld = ldx;
  a.out = out;
  TimedLaunch timed("rows_experts", (hipStream_t)stream);
  if (rows_short(a)) hipLaunchKernelGGL(k_rows_out<1>, rows_grid(a, false), dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(k_rows_out<4>, rows_grid(a, false), dim3(256), 0, (hipStream_t)stream, a);
  LAUNCH_CHECK();
  return LM_OK;
}

template <int DT, bool WEIGHTS>
static void launch_rows_back(const RowsArgs& a, hipStream_t st) {
  if (rows_short(a)) hipLaunchKernelGGL((k_rows_back<DT, WEIGHTS, 1>), rows_grid(a, false), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_rows_back<DT, WEIGHTS, 4>), rows_grid(a, false), dim3(256), 0, st, a);
}
static int rows_back(const lm_rows* r, const void* h, int64_t ldh, const float* weight, void* out, void* stream) {
  int rc;
  if ((rc = check_rows(r))) return rc;
  if (r->T == 0) return LM_OK;
  if (!h || !out) return fail(LM_EINVAL, "row pointers must be non-null");
  if (ldh < r->N) return fail(LM_EINVAL, "row stride below the row length");
  RowsArgs a = rows_args(r);
  a.h = h;
  a.ldh = ldh;
  a.weight = weight;
  a.out = out;
  hipStream_t st = (hipStream_t)stream;
  TimedLaunch timed("rows_experts", st);
  if (weight) {
    if (r->dtype == LM_F16) launch_rows_back<F16, true>(a, st);
    else launch_rows_back<BF16, true>(a, st);
  } else {
    if (r->dtype == LM_F16) launch_rows_back<F16, false>(a, st);
    else launch_rows_back<BF16, false>(a, st);
  }
  LAUNCH_CHECK();
  return LM_OK;
}

extern "C" int lm_dispatch_rows_grad(const lm_rows* r, const void* dy, int64_t lddy, void* dx, void* stream) {
  return rows_back(r, dy, lddy, nullptr, dx, stream);
}
extern "C" int lm_combine_rows(const lm_rows* r, const void* h, int64_t ldh, const float* weight, void* out, void* stream) {
  if (r && r->T > 0 && !weight) return fail(LM_EINVAL, "weights must be non-null");
  return rows_back(r, h, ldh, weight, out, stream);
}
template <int DT>
static void launch_rows_back_grad(const RowsArgs& a, hipStream_t st) {
  if (rows_short(a)) hipLaunchKernelGGL((k_rows_back_grad<DT, 1>), rows_grid(a, true), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_rows_back_grad<DT, 4>), rows_grid(a, true), dim3(256), 0, st, a);
}
extern "C" int lm_combine_rows_grad(const lm_rows* r, const void* dy, int64_t lddy, const void* h, int64_t ldh,
                                    const float* weight, void* dh, float* dweight, void* stream) {
  int rc;
  if ((rc = check_rows(r))) return rc;
  if (r->T == 0) return LM_OK;
  if (!dy || !h || !weight || !dh || !dweight) return fail(LM_EINVAL, "pointers must be non-null");
  if (lddy < r->N || ldh < r->N) return fail(LM_EINVAL, "row stride below the row length");
  RowsArgs a = rows_args(r);
  a.x = dy;
  a.ld = lddy;
  a.h = h;
  a.ldh = ldh;
  a.weight = weight;
  a.out = dh;
  a.dweight = dweight;
  hipStream_t st = (hipStream_t)stream;
  TimedLaunch timed("rows_experts", st);
  if (r->dtype == LM_F16) launch_rows_back_grad<F16>(a, st);
  else launch_rows_back_grad<BF16>(a, st);
  LAUNCH_CHECK();
  return LM_OK;
}
