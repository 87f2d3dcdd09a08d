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
#include "lm_impl.h"
#include "lm_route.h"

template <int DT>
DEV float route_load(const void* p, int64_t i) {
  if constexpr (DT == F32) return ((const LM_GLOBAL float*)p)[i];
  else return val_dt<DT>(((const LM_GLOBAL uint16_t*)p)[i]);
}

// The scores of a token: lane l has experts l, l + 64, ...; those there are not have logit -inf.
template <typename F, int P>
DEV void route_scores(const float (&v)[P], bool sigmoid, F (&s)[P]) {
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < P; ++i) s[i] = F(1) / (F(1) + (sizeof(F) == 8 ? (F)exp(-(double)v[i]) : (F)expf(-v[i])));
    return;
  }
  float top = v[0];
#pragma unroll
  for (int i = 1; i < P; ++i) top = __builtin_fmaxf(top, v[i]);
  top = route_fmax(top);
  F sum = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const F d = (F)v[i] - (F)top;
    s[i] = v[i] == -INFINITY ? F(0) : (sizeof(F) == 8 ? (F)exp((double)d) : (F)expf((float)d));
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

// The choice in 64 bits, for tokens where 32 leave it open.  Lane j returns expert
// j, or -1.  (Logits from `at` on are read again: the caller's registers stay free.)
template <int DT, int P>
__device__ __attribute__((noinline)) int route_choose64(const void* logits, int64_t at, const float* bias, int E, int k, int sigmoid,
                                                       int groups, int per, int top_groups, int group_best) {
  const int lane = threadIdx.x & 63;
  float v[P];
  double s[P];
  uint64_t key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) v[i] = lane + 64 * i < E ? route_load<DT>(logits, at + lane + 64 * i) : -INFINITY;
  route_scores<double, P>(v, sigmoid, s);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (bias && lane + 64 * i < E) s[i] += (double)bias[lane + 64 * i];
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

// Two numbers of 32 bits whose order, as numbers of 64, they leave open: scores are
// off by at most 2^-20 (exponentials of relative 2^-21, sums of them), a sum of two
// and two biases by twice that and its own rounding.
DEV bool route_close(uint32_t larger, uint32_t smaller) {
  const float x = route_value(larger), d = x - route_value(smaller);
  return !(d > 0x1p-18f * __builtin_fmaxf(1.0f, __builtin_fabsf(x)));
}

// The k largest of key (0: none there), the largest first, ties by index.  Lane j
// returns index j, or -1.  CHECK: open says whether two neighbours are close.
template <int P, bool CHECK>
DEV int route_best(uint32_t (&key)[P], int k, bool& open) {
  const int lane = threadIdx.x & 63;
  int mine = -1;
  uint32_t before = 0;
  for (int j = 0; j < k + (CHECK ? 1 : 0); ++j) {
    uint32_t m = key[0];
#pragma unroll
    for (int i = 1; i < P; ++i) m = umax(m, key[i]);
    m = route_max(m);
    if (m == 0) break;
    if constexpr (CHECK) {
      if (j > 0 && route_close(before, m)) open = true;
      if (j == k) break;
      before = m;
    }
    // (the lowest i that has it, and its lowest lane)
    uint64_t hit = 0;
    int at = 0;
#pragma unroll
    for (int i = P - 1; i >= 0; --i) {
      const uint64_t h = __ballot(key[i] == m);
      at = h ? i : at;
      hit = h ? h : hit;
    }
    const int l = __builtin_ctzll(hit);
#pragma unroll
    for (int i = 0; i < P; ++i) key[i] = at == i && lane == l ? 0u : key[i];
    mine = lane == j ? 64 * at + l : mine;
  }
  return mine;
}

// The choice.  Without a bias it follows the logits themselves; with one it is made
// in 32 bits, and again in 64 where two numbers that decide are close.
template <int DT, int P>
DEV int route_choose(const RouteArgs& a, int64_t t, const float (&v)[P], const float (&b)[P], bool even, float* lds) {
  const int lane = threadIdx.x & 63;
  const bool in_groups = a.top_groups < a.groups, sums = in_groups && a.group_best == 2;
  float c[P];
  if (!even || sums) {
    float s[P];
    route_scores<float, P>(v, a.sigmoid, s);
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = v[i] == -INFINITY ? -INFINITY : s[i] + b[i];
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = v[i];
  }
  uint32_t key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) key[i] = c[i] == -INFINITY ? 0u : route_key(even ? v[i] : c[i]);
  bool open = false;
  if (in_groups) {
    // a.lanes lanes look at a group, each at every a.lanes-th member; its two best are joined among them
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (lane + 64 * i < a.E) lds[lane + 64 * i] = c[i] == c[i] ? c[i] : INFINITY;
    __builtin_amdgcn_wave_barrier();
    const int g = lane / a.lanes, part = lane % a.lanes;
    float one = -INFINITY, two = -INFINITY;
    if (g < a.groups)
      for (int m = part; m < a.per; m += a.lanes) {
        const float y = lds[g * a.per + m];
        two = __builtin_fmaxf(two, __builtin_fminf(one, y));
        one = __builtin_fmaxf(one, y);
      }
    __builtin_amdgcn_wave_barrier();
    for (int m = 1; m < a.lanes; m <<= 1) {
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
      const int l = __builtin_ctzll(__ballot(value == last));
      kept |= 1ull << l;
      value = lane == l ? 0u : value;
    }
    if ((!even || sums) && last != 0) {
      const uint32_t next = route_max(value);
      open = next != 0 && route_close(last, next);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int of = (int)((uint32_t)(lane + 64 * i) * a.per_mul >> 20) * a.lanes;
      if (!(kept >> (of & 63) & 1)) key[i] = 0;
    }
  }
  int mine = -1;
  if (!open) mine = even ? route_best<P, false>(key, a.k, open) : route_best<P, true>(key, a.k, open);
  if (open) mine = route_choose64<DT, P>(a.logits, t * a.ld, a.bias, a.E, a.k, a.sigmoid, a.groups, a.per, a.top_groups, a.group_best);
  return mine;
}

template <int DT, int P>
__global__ __launch_bounds__(512) void k_route(RouteArgs a) {
  extern __shared__ uint32_t lds[];
  // counts of the experts, then this workgroup's choices and their ranks
  uint32_t* const count = lds;
  uint16_t* const ent = (uint16_t*)(lds + a.E + 1);
  float* const row = (float*)(lds + a.E + 1 + a.block * a.k) + (threadIdx.x >> 6) * a.E;  // this wave's scores, if there are groups
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(), waves = blockDim.x >> 6;
  const int64_t t0 = (int64_t)blockIdx.x * a.block;
  const int tokens = (int)(a.T - t0 < a.block ? a.T - t0 : a.block), n = tokens * a.k;
  for (int i = tid; i <= a.E; i += blockDim.x) count[i] = 0;
  float b[P];
#pragma unroll
  for (int i = 0; i < P; ++i) b[i] = a.bias && lane + 64 * i < a.E ? a.bias[lane + 64 * i] : 0.0f;
  // a bias that is the same for all decides nothing
  bool even = true;
  if (a.bias) {
    const float b0 = u2f((uint32_t)__builtin_amdgcn_readfirstlane((int)f2u(b[0])));
#pragma unroll
    for (int i = 0; i < P; ++i) even = even && (lane + 64 * i >= a.E || b[i] == b0);
    even = __ballot(even) == ~0ull && __builtin_fabsf(b0) < INFINITY;
  }
  for (int tl = wave; tl < tokens; tl += waves) {
    const int64_t t = t0 + tl;
    float v[P];
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = lane + 64 * i < a.E ? route_load<DT>(a.logits, t * a.ld + lane + 64 * i) : -INFINITY;
    const int mine = route_choose<DT, P>(a, t, v, b, even, row);
    // the chosen experts' logits: e^x of softmax, e^min(x, 0) / (1 + e^-|x|) of sigmoid, so that none overflows
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float o = __shfl(v[i], mine & 63);
      if (mine >> 6 == i) x = o;
    }
    const bool on = mine >= 0;
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
      ent[tl * a.k + lane] = (uint16_t)(on ? mine : a.E);
    }
  }
  __syncthreads();
  // ranks among the choices of one expert, 64 choices at a time, in order
  uint16_t* const rank = ent + a.block * a.k;
  if (wave == 0) {
    for (int i0 = 0; i0 < n; i0 += 64) {
      const bool in = i0 + lane < n;
      const uint32_t e = in ? ent[i0 + lane] : 0u;
      uint64_t same = __ballot(in);
      for (int bit = 0; bit < 11; ++bit) {
        const bool one = e >> bit & 1;
        const uint64_t with = __ballot(one);
        same &= one ? with : ~with;
      }
      if (in) {
        const uint32_t before = count[e];
        rank[i0 + lane] = (uint16_t)(before + __builtin_popcountll(same & ((1ull << lane) - 1)));
        __builtin_amdgcn_wave_barrier();
        if (same >> lane == 1) count[e] = before + __builtin_popcountll(same);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  __syncthreads();
  if (a.blocks > 1) {
    for (int i = tid; i <= a.E; i += blockDim.x) a.counts[(int64_t)blockIdx.x * (a.E + 1) + i] = count[i];
    for (int i = tid; i < n; i += blockDim.x) a.position[t0 * a.k + i] = rank[i];
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
  for (int i = tid; i < n; i += blockDim.x) a.position[i] = (int32_t)(count[ent[i]] + rank[i]);
}

// The choices of the workgroups before each one, per expert: 16 experts a
// workgroup, 64 threads for each, which take a run of the workgroups, 16 at a time
// in registers.
__global__ __launch_bounds__(1024) void k_route_scan(RouteArgs a) {
  __shared__ uint32_t part[16][65];
  const int c = threadIdx.x & 15, seg = threadIdx.x >> 4, e = blockIdx.x * 16 + c, cols = a.E + 1, lane = threadIdx.x & 63;
  const int each = (a.blocks + 63) / 64, b0 = seg * each, b1 = b0 + each < a.blocks ? b0 + each : a.blocks;
  LM_GLOBAL uint32_t* const at = (LM_GLOBAL uint32_t*)a.counts + e;
  uint32_t x[16], sum = 0;
  auto load = [&](int b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = e < cols && b + i < b1 ? at[(int64_t)(b + i) * cols] : 0u;
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
    if (lane == 63 && blockIdx.x * 16 + w < cols) ((LM_GLOBAL uint32_t*)a.counts)[(int64_t)a.blocks * cols + blockIdx.x * 16 + w] = z;
  }
  __syncthreads();
  uint32_t before = part[c][seg];
  for (int b = b0; b < b1; b += 16) {
    if (each > 16) load(b);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (e < cols && b + i < b1) {
        at[(int64_t)(b + i) * cols] = before;
        before += x[i];
      }
  }
}

__global__ __launch_bounds__(256) void k_route_place(RouteArgs a, int64_t n) {
  extern __shared__ uint32_t first[];  // choices of the experts before each
  const int lane = threadIdx.x & 63, cols = a.E + 1;
  const uint32_t* total = a.counts + (int64_t)a.blocks * cols;
  if (threadIdx.x < 64) {
    uint32_t before = 0;
    for (int c = 0; c < cols; c += 64) {
      const int e = c + lane;
      const uint32_t x = e < cols ? total[e] : 0, sum = (uint32_t)lin_scan_add((int)x);
      if (e < cols) first[e] = before + sum - x;
      if (e < a.E && blockIdx.x == 0) a.ends[e] = (int32_t)(before + sum);
      before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = (int64_t)blockIdx.x * 1024 + j * 256 + threadIdx.x;
    if (i < n) {
      const int32_t x = a.expert[i], e = x < 0 ? a.E : x;
      const uint32_t b = div_by(a.entries, (uint32_t)i);
      a.position[i] = (int32_t)(first[e] + a.counts[(int64_t)b * cols + e] + (uint32_t)a.position[i]);
    }
  }
}

// The gradient to the logits.  g = d loss / d w, for the chosen experts j:
//   renormalised   w_j (g_j - sum_i g_i w_i / scale), for sigmoid times 1 - p_j
//   sigmoid        w_j g_j (1 - p_j)
//   softmax        w_j g_j - p_e sum_i g_i w_i, the second term for every expert e
template <int DT, int P>
__global__ __launch_bounds__(256) void k_route_grad(RouteArgs a, const float* dweight, void* out) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave_index();
  if (t >= a.T) return;
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
    route_scores<float, P>(v, false, s);
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
    for (int i = 0; i < P; ++i)
      if (lane + 64 * i == to) d[i] += add;
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
DEV void rows_store(uint16_t* p, lm_u32x4 w, int64_t left) {
  if (left >= 8) {
    *(LM_GLOBAL lm_u32x4_any*)p = w;
    asm volatile("s_nop 1" ::"v"(w) : "memory");  // (store_b128_guarded)
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < left) ((LM_GLOBAL uint16_t*)p)[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
  }
}

// A wave has 512 columns of a token.
__global__ __launch_bounds__(256) void k_rows_out(RowsArgs a, uint32_t chunks) {
  const int64_t item = (int64_t)blockIdx.x * 4 + wave_index(), t = item / chunks;
  if (t >= a.T) return;
  const int64_t c = (item - t * chunks) * 512 + (threadIdx.x & 63) * 8, left = a.N - c;
  const lm_u32x4 w = lin_chunk((const uint16_t*)a.x + t * a.ld + c, left);
  const int end = rows_end(a);
  for (int j = 0; j < a.k; ++j) {
    const int p = a.position[t * a.k + j];
    if (p < 0 || p >= a.T * a.k) continue;
    rows_store((uint16_t*)a.out + p * a.N + c, p < end ? w : lm_u32x4{}, left);
  }
}

template <int DT, bool WEIGHTS>
__global__ __launch_bounds__(256) void k_rows_back(RowsArgs a, uint32_t chunks) {
  const int64_t item = (int64_t)blockIdx.x * 4 + wave_index(), t = item / chunks;
  if (t >= a.T) return;
  const int64_t c = (item - t * chunks) * 512 + (threadIdx.x & 63) * 8, left = a.N - c;
  const int end = rows_end(a);
  float s[8] = {};
  for (int j0 = 0; j0 < a.k; j0 += 4) {  // four rows on their way at once
    lm_u32x4 w[4];
    float by[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int j = j0 + n < a.k ? j0 + n : a.k - 1, p = a.position[t * a.k + j];
      const bool on = j0 + n < a.k && p >= 0 && p < end;
      by[n] = !on ? 0.0f : WEIGHTS ? a.weight[t * a.k + j] : 1.0f;
      w[n] = lm_u32x4{};
      if (on) w[n] = lin_chunk((const uint16_t*)a.h + p * a.ldh + c, left);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = __builtin_fmaf(by[n], val_dt<DT>(i & 1 ? w[n][i >> 1] >> 16 : w[n][i >> 1] & 0xffffu), s[i]);
  }
  lm_u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)bits_dt<DT>(s[2 * i]) | (uint32_t)bits_dt<DT>(s[2 * i + 1]) << 16;
  rows_store((uint16_t*)a.out + t * a.N + c, w, left);
}

// Gradients of the weighted sums: a workgroup has a token.
template <int DT>
__global__ __launch_bounds__(256) void k_rows_back_grad(RowsArgs a) {
  __shared__ float red[4];
  const int64_t t = blockIdx.x;
  const int end = rows_end(a);
  for (int j = 0; j < a.k; ++j) {
    const int p = a.position[t * a.k + j];
    const bool in = p >= 0 && p < a.T * a.k, on = in && p < end;
    const float by = a.weight[t * a.k + j];
    float sum = 0.0f;
    for (int64_t c = threadIdx.x * 8; in && c < a.N; c += 2048) {
      lm_u32x4 w = {};
      if (on) {
        const lm_u32x4 dy = lin_chunk((const uint16_t*)a.x + t * a.ld + c, a.N - c);
        const lm_u32x4 h = lin_chunk((const uint16_t*)a.h + p * a.ldh + c, a.N - c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float lo = val_dt<DT>(dy[i] & 0xffffu), hi = val_dt<DT>(dy[i] >> 16);
          sum = __builtin_fmaf(lo, val_dt<DT>(h[i] & 0xffffu), sum);
          sum = __builtin_fmaf(hi, val_dt<DT>(h[i] >> 16), sum);
          w[i] = (uint32_t)bits_dt<DT>(by * lo) | (uint32_t)bits_dt<DT>(by * hi) << 16;
        }
      }
      rows_store((uint16_t*)a.out + p * a.N + c, w, a.N - c);
    }
    sum = route_sum(sum);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.dweight[t * a.k + j] = on ? red[0] + red[1] + red[2] + red[3] : 0.0f;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
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
  if (r->T * r->top_k > 0x7fffffff) return fail(LM_EUNSUPPORTED, "more than 2^31 - 1 choices");
  if (r->T > 0 && !r->logits) return fail(LM_EINVAL, "logits must be non-null");
  if (r->ld < r->experts) return fail(LM_EINVAL, "row stride below the row length");
  return LM_OK;
}

// Tokens of a workgroup: all of them while they are few, so that one launch does.
static int route_block(int64_t T) {
  if (T <= 32) return (int)T;
  int block = 16;
  while (block < 64 && (T + block - 1) / block > 1024) block *= 2;
  return block;
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
  a.block = a.T > 0 ? route_block(a.T) : 1;
  a.blocks = (int)((a.T + a.block - 1) / a.block);
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
  if (T <= 0 || T > 0x7fffffff || experts < 1 || experts > LM_LINEAR_MAX_EXPERTS) return 0;
  const int64_t block = route_block(T), blocks = (T + block - 1) / block;
  return blocks > 1 ? align256((size_t)(blocks + 1) * (size_t)(experts + 1) * 4) : 0;
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
    a.counts = (uint32_t*)workspace;
  }
  hipStream_t st = (hipStream_t)stream;
  TimedLaunch timed("route", st);
  const int threads = 512;
  const size_t lds = (size_t)(a.E + 1) * 4 + (size_t)a.block * a.k * 4 + (a.top_groups < a.groups ? (size_t)threads / 64 * a.E * 4 : 0);
  ROUTE_BY_TYPE(k_route, dim3((unsigned)(a.blocks > 0 ? a.blocks : 1)), dim3(threads), lds, st, a);
  LAUNCH_CHECK();
  if (a.blocks > 1) {
    hipLaunchKernelGGL(k_route_scan, dim3((unsigned)((a.E + 16) / 16)), dim3(1024), 0, st, a);
    LAUNCH_CHECK();
    const int64_t n = a.T * a.k;
    hipLaunchKernelGGL(k_route_place, dim3((unsigned)((n + 1023) / 1024)), dim3(256), (size_t)(a.E + 1) * 4, st, a, n);
    LAUNCH_CHECK();
  }
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
  ROUTE_BY_TYPE(k_route_grad, dim3((unsigned)n), dim3(256), 0, st, a, dweight, dlogits);
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
static int rows_grid(const RowsArgs& a, uint32_t& chunks, dim3& grid) {
  chunks = (uint32_t)((a.N + 511) / 512);
  const int64_t n = (a.T * (int64_t)chunks + 3) / 4;
  if (n > 0x7fffffff) return fail(LM_EUNSUPPORTED, "rows too large for one launch");
  grid = dim3((unsigned)n);
  return LM_OK;
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
  uint32_t chunks;
  dim3 grid;
  if ((rc = rows_grid(a, chunks, grid))) return rc;
  TimedLaunch timed("rows_experts", (hipStream_t)stream);
  hipLaunchKernelGGL(k_rows_out, grid, dim3(256), 0, (hipStream_t)stream, a, chunks);
  LAUNCH_CHECK();
  return LM_OK;
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
  uint32_t chunks;
  dim3 grid;
  if ((rc = rows_grid(a, chunks, grid))) return rc;
  hipStream_t st = (hipStream_t)stream;
  TimedLaunch timed("rows_experts", st);
  if (weight) {
    if (r->dtype == LM_F16) hipLaunchKernelGGL((k_rows_back<F16, true>), grid, dim3(256), 0, st, a, chunks);
    else hipLaunchKernelGGL((k_rows_back<BF16, true>), grid, dim3(256), 0, st, a, chunks);
  } else {
    if (r->dtype == LM_F16) hipLaunchKernelGGL((k_rows_back<F16, false>), grid, dim3(256), 0, st, a, chunks);
    else hipLaunchKernelGGL((k_rows_back<BF16, false>), grid, dim3(256), 0, st, a, chunks);
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
  if (r->dtype == LM_F16) hipLaunchKernelGGL((k_rows_back_grad<F16>), dim3((unsigned)a.T), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_rows_back_grad<BF16>), dim3((unsigned)a.T), dim3(256), 0, st, a);
  LAUNCH_CHECK();
  return LM_OK;
}
