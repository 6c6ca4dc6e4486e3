// Log probabilities of given symbols under distributions given class by class, with entropy, the most likely
// alternatives, and the gradient (include/dvc_hip.h).
//
// Mathematics.  One pass over the logits l_v of a site with the running maximum m:
//   S = sum e^(l_v - m),  T = sum e^(l_v - m) (l_v - m)   (both rescaled when m grows)
//   log p_v = (l_v - m) - log S,   H = log S - T / S
// S >= 1 and T <= 0, so both terms of H are >= 0 and nothing cancels.  m and log S are kept apart for the backward pass:
// their sum would round away what distinguishes probabilities once |m| is large.
//   dL/dl_v = g_lp (1[v = s] - p_v) - g_H p_v (log p_v + H)
// Classes at minus infinity add nothing (0 * -inf is kept out by a floor on l_v - m in T); a NaN or +inf makes the whole
// site NaN.  Everything is held in fp32 whatever the logits' type; a lane's sums over very many classes go on in 64 bits.
#include "dvc_common.h"

namespace {

struct Logits { const void* p; long long bs, cs; int groups, classes; };

template <int DT> struct Elem;
template <> struct Elem<DVC_F32> {
  typedef float type;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct Elem<DVC_BF16> {
  typedef unsigned short type;
  static __device__ __forceinline__ float up(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
  static __device__ __forceinline__ unsigned short down(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
};
template <> struct Elem<DVC_F16> {
  typedef _Float16 type;
  static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 down(float v) { return (_Float16)v; }
};

// below this e^x is zero in fp32: a floor that keeps 0 * (-inf) out of the entropy sums
constexpr float kFloor = -200.f;
#define NEG_INF (-__builtin_inff())

// the running statistics of one site (or of a part of its classes)
struct Stat {
  float m, s, t;
  __device__ __forceinline__ void clear() { m = NEG_INF; s = 0.f; t = 0.f; }
  // join with another part: either may be empty (m = -inf, s = 0)
  __device__ __forceinline__ void join(float m2, float s2, float t2) {
    const float mm = fmaxf(m, m2);
    const float a = m == mm ? 1.f : __expf(m - mm), b = m2 == mm ? 1.f : __expf(m2 - mm);
    t = a * (t + s * fmaxf(m == mm ? 0.f : m - mm, kFloor)) + b * (t2 + s2 * fmaxf(m2 == mm ? 0.f : m2 - mm, kFloor));
    s = a * s + b * s2;
    m = mm;
  }
  __device__ __forceinline__ void add(float x) {
    if (x > m) {
      const float a = __expf(m - x);
      t = a * (t + s * fmaxf(m - x, kFloor));
      s = a * s;
      m = x;
    }
    const float d = m == NEG_INF ? x : x - m;   // (all classes so far at -inf: e = exp(-inf) = 0)
    const float e = __expf(d);
    s += e;
    t += e * fmaxf(d, kFloor);
  }
};

// The sums of more classes than fp32 adds up one by one without losing bits (a sum that is large against its terms rounds
// equal ones the same way each time: 131072 classes of logits -3..3 in one lane had a log S off by 1e-3): every kChain classes
// a lane's sums move to 64 bits, its maximum stays.
constexpr int kChain = 256;
struct WideStat {
  float m;
  double s, t;
  __device__ __forceinline__ void clear() { m = NEG_INF; s = 0.; t = 0.; }
  __device__ __forceinline__ void take(Stat* st) {
    if (m != st->m) {                     // (the lane's maximum only grows)
      const float a = __expf(m - st->m);
      t = (double)a * (t + s * (double)fmaxf(m - st->m, kFloor));
      s = (double)a * s;
      m = st->m;
    }
    s += (double)st->s;
    t += (double)st->t;
    st->s = 0.f;
    st->t = 0.f;
  }
  __device__ __forceinline__ void give(Stat* st) {      // all of it, in fp32 again
    take(st);
    st->s = (float)s;
    st->t = (float)t;
  }
};

__device__ __forceinline__ void finish(const Stat& st, float* log_s, float* entropy) {
  const bool empty = st.m == NEG_INF && st.s == 0.f;   // (s is NaN when a class was)
  *log_s = empty ? 0.f : __logf(st.s);
  *entropy = empty ? 0.f : *log_s - st.t / st.s;
}

// log p of a logit
__device__ __forceinline__ float log_p(float x, float m, float log_s) {
  return (x - (m == NEG_INF ? 0.f : m)) - log_s;
}

// log of the probability of the given symbol (bounds are checked here: nothing outside the row is read)
template <int DT>
__device__ __forceinline__ float given(const typename Elem<DT>::type* row, long long cs, int classes, int sym, float m, float log_s) {
  if (sym < 0) return 0.f;
  if (sym >= classes) return __uint_as_float(0x7fc00000u);
  return log_p(Elem<DT>::up(row[sym * cs]), m, log_s);
}

__device__ __forceinline__ float given_log_p(int sym, int classes, float x, float m, float log_s) {
  return sym < 0 ? 0.f : sym >= classes ? __uint_as_float(0x7fc00000u) : log_p(x, m, log_s);
}

// order of the alternatives: larger logit first, NaN above all, then the lower class.  +0 and -0 are equal.
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// ---------------------------------------------------------------- wave helpers
__device__ __forceinline__ unsigned wave_max(unsigned v) {    // uniform result
  unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);
  v = v > o ? v : o;
  o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);
  v = v > o ? v : o;
  o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true);   // row_half_mirror
  v = v > o ? v : o;
  o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true);   // row_mirror: all 16 lanes of a row agree
  v = v > o ? v : o;
  const unsigned a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16);
  const unsigned c = __builtin_amdgcn_readlane((int)v, 32), d = __builtin_amdgcn_readlane((int)v, 48);
  const unsigned ab = a > b ? a : b, cd = c > d ? c : d;
  return ab > cd ? ab : cd;
}

// Lanes 0..15 hold a value each (others: anything): the `nth` largest of the sixteen, uniform.  A value has at least `nth`
// not smaller than itself exactly if it is at most the nth largest.
template <int R>
__device__ __forceinline__ int not_below(unsigned v) {
  const unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x120 + R, 0xF, 0xF, true);      // row_ror R
  if constexpr (R > 1) return (o >= v ? 1 : 0) + not_below<R - 1>(v);
  else return o >= v ? 1 : 0;
}
__device__ __forceinline__ unsigned nth_of_16(unsigned v, int nth, int lane) {
  const int ge = 1 + not_below<15>(v);
  return wave_max(lane < 16 && ge >= nth ? v : 0);
}
// the same over lanes 0..31: a row's own sixteen and the other row's
template <int R>
__device__ __forceinline__ int other_not_below(unsigned o, unsigned v) {
  const unsigned r = (unsigned)__builtin_amdgcn_mov_dpp((int)o, 0x120 + R, 0xF, 0xF, true);
  if constexpr (R > 1) return (r >= v ? 1 : 0) + other_not_below<R - 1>(o, v);
  else return r >= v ? 1 : 0;
}
__device__ __forceinline__ unsigned nth_of_32(unsigned v, int nth, int lane) {
  const unsigned o = (unsigned)__shfl_xor((int)v, 16, 64);
  const int ge = 1 + not_below<15>(v) + (o >= v ? 1 : 0) + other_not_below<15>(o, v);
  return wave_max(lane < 32 && ge >= nth ? v : 0);
}

template <int CTRL> __device__ __forceinline__ unsigned max_with(unsigned v) {
  const unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
  return v > o ? v : o;
}
// a bound for the `top` best of a wave whose lanes hold the maxima of pairs: over the pairs, or over pairs of them
__device__ __forceinline__ unsigned group_bound(unsigned pair, int top, int lane) {
  if (top > 8) return nth_of_32((unsigned)__shfl((int)pair, 2 * (lane & 31), 64), top, lane);
  return nth_of_16((unsigned)__shfl((int)max_with<0x4E>(pair), 4 * (lane & 15), 64), top, lane);
}
template <int CTRL> __device__ __forceinline__ float lane_of(float v) {
  return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float read_lane(float v, int l) { return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), l)); }
__device__ __forceinline__ float wave_maxf(float v) {         // uniform results; the same swaps as in wave_max
  v = fmaxf(v, lane_of<0xB1>(v));
  v = fmaxf(v, lane_of<0x4E>(v));
  v = fmaxf(v, lane_of<0x141>(v));
  v = fmaxf(v, lane_of<0x140>(v));
  return fmaxf(fmaxf(read_lane(v, 0), read_lane(v, 16)), fmaxf(read_lane(v, 32), read_lane(v, 48)));
}
__device__ __forceinline__ float wave_sumf(float v) {
  v += lane_of<0xB1>(v);
  v += lane_of<0x4E>(v);
  v += lane_of<0x141>(v);
  v += lane_of<0x140>(v);
  return (read_lane(v, 0) + read_lane(v, 16)) + (read_lane(v, 32) + read_lane(v, 48));
}

// the 64 lanes' statistics in one: the maximum first, so that each lane is rescaled once (262144 rows of 1000 bf16: 143 us;
// joined in pairs, with six shuffles of three values and twelve exponentials, 177)
__device__ __forceinline__ void wave_join(Stat* st) {
  const float mm = wave_maxf(st->m);
  const float a = st->m == mm ? 1.f : __expf(st->m - mm), d = st->m == mm ? 0.f : fmaxf(st->m - mm, kFloor);
  st->t = wave_sumf(a * (st->t + st->s * d));
  st->s = wave_sumf(a * st->s);
  st->m = mm;
}

// A wave's list of the best classes so far: lane j < top holds the j-th (key, class), best first.  An empty place has
// key 0, below every number's.
struct WaveList {
  unsigned key;
  int cls;
  unsigned last_key;     // uniform: the list's last place
  int last_cls;
  __device__ __forceinline__ void clear() { key = 0; cls = 0x7fffffff; last_key = 0; last_cls = 0x7fffffff; }
  __device__ __forceinline__ bool beaten_by(unsigned k, int c) const { return k > last_key || (k == last_key && c < last_cls); }
  // take a uniform candidate that beats the last place
  __device__ __forceinline__ void insert(unsigned k, int c, int lane, int top) {
    const bool before = lane < top && (key > k || (key == k && cls < c));
    const int pos = __popcll(__ballot(before));
    const unsigned pk = (unsigned)__builtin_amdgcn_mov_dpp((int)key, 0x111, 0xF, 0xF, true);    // row_shr 1: top <= 16, one row
    const int pc = __builtin_amdgcn_mov_dpp(cls, 0x111, 0xF, 0xF, true);
    if (lane > pos) { key = pk; cls = pc; }
    if (lane == pos) { key = k; cls = c; }
    last_key = (unsigned)__builtin_amdgcn_readlane((int)key, top - 1);
    last_cls = __builtin_amdgcn_readlane(cls, top - 1);
  }
  // candidates of all lanes at once (k = 0: none)
  __device__ __forceinline__ void offer(unsigned k, int c, int lane, int top) {
    unsigned long long who = __ballot(k != 0 && beaten_by(k, c));
    while (who) {
      const int l = __ffsll((long long)who) - 1;
      insert((unsigned)__builtin_amdgcn_readlane((int)k, l), __builtin_amdgcn_readlane(c, l), lane, top);
      who &= who - 1;
      who &= __ballot(k != 0 && beaten_by(k, c));
    }
  }
};

// What reaches the bound, in any order (LDS).  More than 64 -- many equal classes -- overflow: the list takes over.
struct Pool {
  unsigned key[64];
  int cls[64];
  int count;
  __device__ __forceinline__ void push(unsigned k, int c) {
    const int at = atomicAdd(&count, 1);
    if (at < 64) { key[at] = k; cls[at] = c; }
  }
};
// A lane's (key, class) of `count` in lanes 0 .. count - 1: how many of the others come before it.  All are different, so the
// places are, too, whatever order they were pushed in.
__device__ __forceinline__ int place_of(unsigned k, int c, int count) {
  int r = 0;
  for (int i = 0; i < count; ++i) {
    const unsigned ki = (unsigned)__builtin_amdgcn_readlane((int)k, i);
    const int ci = __builtin_amdgcn_readlane(c, i);
    r += ki > k || (ki == k && ci < c) ? 1 : 0;
  }
  return r;
}

__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

// ---------------------------------------------------------------- rows: the classes of a site are adjacent
// One wave or one workgroup of four per row, 16-byte loads with the row's unaligned ends taken one by one.  Bound by HBM
// for many rows; where there are few, a row is cut over several workgroups (one workgroup reads a row of 131072 at the
// latency of its own loads: 25 us) and a second kernel joins the parts.
//
// The alternatives cost no second pass: a lane's running maximum is the largest of its own classes.  The lanes form
// sixteen groups (32 above 8 alternatives: the least of 16 maxima is a poor bound, 262144 rows of 1000 bf16 with 16
// alternatives 585 us, 336 with 32); the `top`-th largest of the groups' maxima (top <= 16) is a lower bound for the top-th best class, and only lanes whose maximum reaches it can hold one (of random classes about 16 ln 2 reach the
// bound for top 8).  The classes of those few lanes are gone over again (in cache; shared out over the wave: 4096 rows of
// 32768 bf16 with 8 alternatives 62 us, 82 with each lane on its own), and what reaches the bound goes into a small pool, whose members are then
// placed by counting (inserting them one by one into a sorted list, which remains for pools that overflow, was half the
// time of a short row).
template <int DT> struct Vec {
  typedef typename Elem<DT>::type T;
  static constexpr int N = 16 / sizeof(T);
  union { uint4 q; T e[N]; };
};

struct RowPart {      // how a row's classes are dealt out: head one by one, body in vectors, tail one by one
  int head, body, tail0;
};
template <int DT>
__device__ __forceinline__ RowPart row_part(const typename Elem<DT>::type* row, int classes) {
  constexpr int N = Vec<DT>::N;
  RowPart r;
  r.head = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(typename Elem<DT>::type);
  r.head = r.head < classes ? r.head : classes;
  r.body = (classes - r.head) / N;
  r.tail0 = r.head + r.body * N;
  return r;
}

// one vector's worth of classes into a lane's statistics
template <int N>
__device__ __forceinline__ void add_many(Stat* st, const float* x) {
  float vm = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) vm = fmaxf(vm, x[i]);
  if (vm > st->m) {
    const float a = __expf(st->m - vm);
    st->t = a * (st->t + st->s * fmaxf(st->m - vm, kFloor));
    st->s = a * st->s;
    st->m = vm;
  }
  const float m = st->m == NEG_INF ? 0.f : st->m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = x[i] - m, e = __expf(d);
    st->s += e;
    st->t += e * fmaxf(d, kFloor);
  }
}

// what a cut row's parts leave for the join: [site][part] statistics and lists
struct Parts {
  float* stat;        // 3 floats each
  unsigned* key;      // `top` each
  int* cls;
};

template <int DT, int NT>
__global__ __launch_bounds__(256) void symbol_rows_kernel(Logits l, const int* symbols, int top, float* log_prob, float* entropy,
                                                          float* stats, float* top_lp, int* top_sym, int sites, int nparts,
                                                          Parts parts) {
  typedef typename Elem<DT>::type T;
  constexpr int N = Vec<DT>::N, WAVES = NT / 64, ROWS = 256 / NT;
  static_assert(NT == 64 || NT == 256, "a wave or a workgroup per row (part)");
  __shared__ float part[WAVES > 1 ? WAVES * 3 : 1];
  __shared__ unsigned keys[WAVES > 1 ? WAVES * DVC_MAX_TOP : 1];
  __shared__ int classes_of[WAVES > 1 ? WAVES * DVC_MAX_TOP : 1];
  __shared__ Pool pools[ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  Pool* const pool = &pools[ROWS > 1 ? wave : 0];
  const int tid = ROWS > 1 ? lane : (int)threadIdx.x;
  const int unit = __builtin_amdgcn_readfirstlane((int)blockIdx.x * ROWS + (ROWS > 1 ? wave : 0));
  const int site = NT == 64 ? unit : unit / nparts, piece = NT == 64 ? 0 : unit - site * nparts;
  if (site >= sites) return;            // (whole waves, and only where a row is a wave: no barrier below is missed)
  const int n = site / l.groups, g = site - n * l.groups;
  const T* const row = static_cast<const T*>(l.p) + (long long)n * l.bs + (long long)g * l.classes;
  RowPart rp = row_part<DT>(row, l.classes);
  const int all_vecs = rp.body, b0 = (int)((long long)all_vecs * piece / nparts), b1 = (int)((long long)all_vecs * (piece + 1) / nparts);
  const uint4* const body = reinterpret_cast<const uint4*>(row + rp.head) + b0;
  const int body_v = rp.head + b0 * N;  // this part's first class
  rp.body = b1 - b0;

  if (tid == 0) pool->count = 0;
  float given_x = 0.f;                  // (requested before the row is read: at the end it would be a wait of its own)
  int sym = -1;
  if (nparts == 1) {
    sym = symbols[site];
    if (sym >= 0 && sym < l.classes) given_x = Elem<DT>::up(row[sym]);
  }

  Stat st;
  st.clear();
  // ends: at most N - 1 classes on either side
  const int ends = piece == 0 ? rp.head + l.classes - rp.tail0 : 0;
  const int end_v = tid < rp.head ? tid : rp.tail0 + tid - rp.head;
  const bool has_end = tid < ends;
  const float end_x = has_end ? Elem<DT>::up(row[end_v]) : NEG_INF;
  if (has_end) st.add(end_x);
  constexpr int U = 4;                  // vectors in flight per lane
  constexpr int STRETCH = kChain / N * NT;      // vectors over which a lane adds up kChain classes
  WideStat wide;
  wide.clear();
  for (int j = tid; j < rp.body; j += U * NT) {
    Vec<DT> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u * NT < rp.body) q[u].q = body[j + u * NT];
    if (WAVES > 1 && j >= STRETCH && (j - tid) % STRETCH == 0) wide.take(&st);      // (a row of one wave is shorter)
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u * NT < rp.body) {
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = Elem<DT>::up(q[u].e[i]);
        add_many<N>(&st, x);
      }
  }
  if (WAVES > 1 && rp.body > STRETCH) wide.give(&st);

  // what the lane's best class is worth; a lane that met a NaN or +inf looks again (its maximum ignores NaN)
  unsigned best = 0;
  if (top > 0) {
    if (has_end || tid < rp.body) best = order_key(st.m);
    if (st.s != st.s) {
      if (has_end) best = order_key(end_x);
      for (int v = tid; v < rp.body; v += NT) {
        Vec<DT> q;
        q.q = body[v];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const unsigned k = order_key(Elem<DT>::up(q.e[i]));
          best = k > best ? k : best;
        }
      }
    }
  }

  Stat all = st;
  wave_join(&all);
  if constexpr (WAVES > 1) {
    if (lane == 0) { part[wave * 3] = all.m; part[wave * 3 + 1] = all.s; part[wave * 3 + 2] = all.t; }
  }
  // the groups' maxima: four (two) lanes each where the row is a wave, sixteen (eight) where it is a workgroup
  unsigned bound = 0;
  const bool many = top > 8;
  if (top > 0) {
    unsigned k = max_with<0xB1>(best);
    if constexpr (WAVES > 1) {
      k = max_with<0x141>(max_with<0x4E>(k));
      if (many) {
        if ((lane & 7) == 0) keys[wave * 8 + (lane >> 3)] = k;
      } else {
        k = max_with<0x140>(k);
        if ((lane & 15) == 0) keys[wave * 4 + (lane >> 4)] = k;
      }
    } else {
      bound = group_bound(k, top, lane);
    }
  }
  if constexpr (WAVES > 1) {
    __syncthreads();
    all.clear();
    for (int w = 0; w < WAVES; ++w) all.join(part[w * 3], part[w * 3 + 1], part[w * 3 + 2]);
    if (top > 0) bound = many ? nth_of_32(keys[lane & 31], top, lane) : nth_of_16(keys[lane & 15], top, lane);
  }
  float log_s, h;
  finish(all, &log_s, &h);

  if (top > 0) {
    const bool in = best >= bound && best != 0;      // (fewer groups than `top` with a class: bound 0, all look)
    const unsigned end_k = in && has_end ? order_key(end_x) : 0;
    // goes over the vectors of the lanes whose best reaches the bound -- a handful, so the wave shares them out, a vector per
    // lane -- and hands on what reaches `least` as well; uniform over the wave
    const unsigned long long who = __ballot(in);
    const int n_in = __popcll(who), ahead = (int)__builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0u));
    const int ids = __builtin_amdgcn_ds_permute(4 * (in ? ahead : n_in + lane - ahead), lane);      // lane j: the j-th of them
    const int wave0 = tid - lane, each = rp.body > wave0 ? (rp.body - wave0 + NT - 1) / NT : 0, pairs = n_in * each;
    auto look = [&](auto&& least, auto&& take) __attribute__((always_inline)) {
      for (int p0 = 0; p0 < pairs; p0 += 64) {
        const int p = p0 + lane < pairs ? p0 + lane : pairs - 1, j = p / each;
        const int v = wave0 + __builtin_amdgcn_ds_bpermute(4 * j, ids) + (p - j * each) * NT;
        const bool have = p0 + lane < pairs && v < rp.body;
        Vec<DT> q;
        if (have) q.q = body[v];
        float vm = NEG_INF;
        bool nan = false;
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          x[i] = have ? Elem<DT>::up(q.e[i]) : 0.f;
          vm = fmaxf(vm, x[i]);
          nan |= x[i] != x[i];
        }
        const unsigned km = nan ? 0xffffffffu : order_key(vm);
        if (!__ballot(have && km >= bound && km >= least())) continue;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const unsigned k = order_key(x[i]);
          take(have && k >= bound ? k : 0, body_v + v * N + i);
        }
      }
    };
    if (end_k != 0 && end_k >= bound) pool->push(end_k, end_v);
    look([] { return 0u; }, [&](unsigned k, int c) { if (k != 0) pool->push(k, c); });
    if constexpr (WAVES > 1) __syncthreads();
    else __threadfence_block();
    const int count = __builtin_amdgcn_readfirstlane(pool->count);
    unsigned key = 0;
    int cls = 0, place = top;
    if (count <= 64) {
      if (ROWS > 1 || wave == 0) {
        if (lane < count) { key = pool->key[lane]; cls = pool->cls[lane]; }
        place = place_of(key, cls, count);
        place = lane < count ? place : top;
      }
    } else {
      WaveList list;
      list.clear();
      list.offer(end_k >= bound ? end_k : 0, end_v, lane, top);
      look([&] { return list.last_key; }, [&](unsigned k, int c) { list.offer(k, c, lane, top); });
      if constexpr (WAVES > 1) {
        if (lane < top) {                 // (the groups' maxima in `keys` were read before the barrier above)
          keys[wave * DVC_MAX_TOP + lane] = list.key;
          classes_of[wave * DVC_MAX_TOP + lane] = list.cls;
        }
        __syncthreads();
        if (wave == 0) {                  // place 0..15 is this wave's own list
          const bool have = lane >= DVC_MAX_TOP && lane % DVC_MAX_TOP < top;
          static_assert(WAVES * DVC_MAX_TOP == 64, "the waves' lists are a lane each");
          list.offer(have ? keys[lane] : 0, have ? classes_of[lane] : 0, lane, top);
        }
      }
      key = list.key;
      cls = list.cls;
      place = (ROWS > 1 || wave == 0) && lane < top ? lane : top;
    }
    if (place < top) {
      const long long at = (long long)unit * top + place;       // (a whole row's unit is its site)
      if (nparts > 1) {
        parts.key[at] = key;
        parts.cls[at] = cls;
      } else {
        top_lp[at] = log_p(key_value(key), all.m, log_s);
        top_sym[at] = cls;
      }
    }
  }
  if (nparts > 1) {
    if (threadIdx.x == 0) {
      parts.stat[(long long)unit * 3] = all.m;
      parts.stat[(long long)unit * 3 + 1] = all.s;
      parts.stat[(long long)unit * 3 + 2] = all.t;
    }
  } else if (tid == 0) {
    log_prob[site] = given_log_p(sym, l.classes, given_x, all.m, log_s);
    entropy[site] = h;
    stats[site] = all.m;
    stats[(long long)sites + site] = log_s;
  }
}

// The parts of a cut row (at most 64: a lane each) joined, a wave per row.
constexpr int kMaxParts = 64;

template <int DT>
__global__ __launch_bounds__(64) void symbol_rows_join_kernel(Logits l, const int* symbols, int top, float* log_prob, float* entropy,
                                                              float* stats, float* top_lp, int* top_sym, int sites, int nparts,
                                                              Parts parts) {
  typedef typename Elem<DT>::type T;
  __shared__ Pool pool;
  const int lane = threadIdx.x, site = blockIdx.x;
  const bool have = lane < nparts;
  const long long at = (long long)site * nparts + (have ? lane : 0);
  const int n = site / l.groups, g = site - n * l.groups;
  const T* const row = static_cast<const T*>(l.p) + (long long)n * l.bs + (long long)g * l.classes;
  const int sym = symbols[site];
  Stat st;
  st.clear();
  if (have) { st.m = parts.stat[at * 3]; st.s = parts.stat[at * 3 + 1]; st.t = parts.stat[at * 3 + 2]; }
  unsigned key[DVC_MAX_TOP];        // (all requested before the first is used)
  int cls[DVC_MAX_TOP];
#pragma unroll
  for (int j = 0; j < DVC_MAX_TOP; ++j) {
    key[j] = have && j < top ? parts.key[at * top + j] : 0;
    cls[j] = have && j < top ? parts.cls[at * top + j] : 0;
  }
  const float given_x = sym >= 0 && sym < l.classes ? Elem<DT>::up(row[sym]) : 0.f;
  if (lane == 0) pool.count = 0;
  wave_join(&st);
  float log_s, h;
  finish(st, &log_s, &h);
  if (top > 0) {
    // four (two) parts' first places a group: the same bound as over a row's lanes
    const unsigned bound = group_bound(max_with<0xB1>(key[0]), top, lane);
    __threadfence_block();
#pragma unroll
    for (int j = 0; j < DVC_MAX_TOP; ++j)
      if (key[j] != 0 && key[j] >= bound) pool.push(key[j], cls[j]);
    __threadfence_block();
    const int count = __builtin_amdgcn_readfirstlane(pool.count);
    unsigned my_key = 0;
    int my_cls = 0, place = top;
    if (count <= 64) {
      if (lane < count) { my_key = pool.key[lane]; my_cls = pool.cls[lane]; }
      place = place_of(my_key, my_cls, count);
      place = lane < count ? place : top;
    } else {
      WaveList list;
      list.clear();
#pragma unroll
      for (int j = 0; j < DVC_MAX_TOP; ++j) list.offer(key[j], cls[j], lane, top);
      my_key = list.key;
      my_cls = list.cls;
      place = lane;
    }
    if (place < top) {
      top_lp[(long long)site * top + place] = log_p(key_value(my_key), st.m, log_s);
      top_sym[(long long)site * top + place] = my_cls;
    }
  }
  if (lane == 0) {
    log_prob[site] = given_log_p(sym, l.classes, given_x, st.m, log_s);
    entropy[site] = h;
    stats[site] = st.m;
    stats[(long long)sites + site] = log_s;
  }
}

// ---------------------------------------------------------------- planes: the classes of a site are planes apart
// A lane per site, so a wave reads 64 adjacent pixels of one class at a time.  With few sites the classes are cut into SL
// ranges, one per wave of the workgroup, joined through LDS.  The alternatives are a short sorted list per thread.
template <int TOP>
struct ThreadList {
  unsigned key[TOP > 0 ? TOP : 1];
  int cls[TOP > 0 ? TOP : 1];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < TOP; ++j) { key[j] = 0; cls[j] = 0x7fffffff; }
  }
  // candidates come in rising class order: an equal key goes behind
  __device__ __forceinline__ void insert(unsigned k, int c) {
#pragma unroll
    for (int j = TOP - 1; j >= 1; --j) {
      const bool above = k > key[j - 1], here = k > key[j];
      cls[j] = above ? cls[j - 1] : here ? c : cls[j];
      key[j] = above ? key[j - 1] : here ? k : key[j];
    }
    if (k > key[0]) { key[0] = k; cls[0] = c; }
  }
};

// The same for 16-bit logits of at most 65536 classes: key and class share a word (higher class, smaller word), all words
// differ, and taking one is a minimum and a maximum per place -- no compares to carry, no order of arrival (bf16 planes 32 x 4 x 64
// classes x 64 x 64: 32 us with 4 alternatives, 60 with 16, the list above 42 and 98; a single alternative is cheaper above).
constexpr int kPackedClasses = 65536;
template <int DT> __device__ __forceinline__ unsigned order_key16(typename Elem<DT>::type v) {
  const unsigned b = __builtin_bit_cast(unsigned short, v);
  constexpr unsigned INF = DT == DVC_BF16 ? 0x7f80u : 0x7c00u;
  const unsigned k = (b & 0x8000u) ? ~b & 0xffffu : b | 0x8000u;
  return (b & 0x7fffu) > INF ? 0xffffu : b == 0x8000u ? 0x8000u : k;
}
template <int DT> __device__ __forceinline__ float key16_value(unsigned k) {
  return Elem<DT>::up(__builtin_bit_cast(typename Elem<DT>::type, (unsigned short)((k & 0x8000u) ? k ^ 0x8000u : ~k)));
}
template <int TOP>
struct PackedList {
  unsigned word[TOP > 0 ? TOP : 1];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < TOP; ++j) word[j] = 0;
  }
  __device__ __forceinline__ void insert(unsigned w) {
#pragma unroll
    for (int j = 0; j < TOP; ++j) {
      const unsigned up = w > word[j] ? w : word[j];
      w = w > word[j] ? word[j] : w;
      word[j] = up;
    }
  }
  static __device__ __forceinline__ unsigned pack(unsigned key, int c) { return key << 16 | (0xffffu - (unsigned)c); }
  __device__ __forceinline__ int cls(int j) const { return (int)(0xffffu - (word[j] & 0xffffu)); }
};

template <int DT, int TOP, int SL, bool PACK>
__global__ __launch_bounds__(SL == 16 ? 1024 : 256) void symbol_planes_kernel(Logits l, const int* symbols, int top, float* log_prob,
                                                                              float* entropy, float* stats, float* top_lp,
                                                                              int* top_sym, long long sites, unsigned hw) {
  typedef typename Elem<DT>::type T;
  constexpr int SITES = SL == 1 ? 256 : 64;
  __shared__ float part[SL > 1 ? SL * 3 * 64 : 1];
  __shared__ unsigned keys[SL > 1 && TOP > 0 ? SL * TOP * 64 : 1];
  __shared__ int classes_of[SL > 1 && TOP > 0 && !PACK ? SL * TOP * 64 : 1];
  const int slot = threadIdx.x % SITES;
  const int slice = SL == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)(threadIdx.x / SITES));
  const long long i = (long long)blockIdx.x * SITES + slot;
  const bool live = i < sites;
  const long long ic = live ? i : sites - 1;             // idle lanes repeat the last site
  const long long ng = ic / hw;
  const unsigned p = (unsigned)(ic - ng * hw);
  const int n = (int)(ng / l.groups), g = (int)(ng - (long long)n * l.groups);
  const T* const row = static_cast<const T*>(l.p) + (long long)n * l.bs + (long long)g * l.classes * l.cs + p;
  const int per = (l.classes + SL - 1) / SL;
  const int v0 = slice * per, v1 = v0 + per < l.classes ? v0 + per : l.classes;

  Stat st;
  st.clear();
  ThreadList<PACK ? 0 : TOP> list;
  PackedList<PACK ? TOP : 0> packed;
  list.clear();
  packed.clear();
  float last = NEG_INF;
  auto take = [&](T raw, float x, int v) {
    if constexpr (TOP > 0 && PACK) {
      packed.insert(packed.pack(order_key16<DT>(raw), v));
    } else if constexpr (TOP > 0) {
      if (v - v0 < TOP || !(x <= last)) {      // (a NaN, or behind one, compares false: the keys decide)
        list.insert(order_key(x), v);
        last = list.key[TOP - 1] != 0 ? key_value(list.key[TOP - 1]) : NEG_INF;
      }
    }
  };
  constexpr int U = 8;
  WideStat wide;
  wide.clear();
  int v = v0;
  for (; v + U <= v1; v += U) {
    T raw[U];
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = row[(long long)(v + u) * l.cs];
      x[u] = Elem<DT>::up(raw[u]);
    }
    if (v > v0 && (v - v0) % kChain == 0) wide.take(&st);
    add_many<U>(&st, x);
#pragma unroll
    for (int u = 0; u < U; ++u) take(raw[u], x[u], v + u);
  }
  for (; v < v1; ++v) {
    const T raw = row[(long long)v * l.cs];
    const float x = Elem<DT>::up(raw);
    add_many<1>(&st, &x);
    take(raw, x, v);
  }
  if (v1 - v0 > kChain) wide.give(&st);

  if constexpr (SL > 1) {
    part[(slice * 3 + 0) * 64 + slot] = st.m;
    part[(slice * 3 + 1) * 64 + slot] = st.s;
    part[(slice * 3 + 2) * 64 + slot] = st.t;
    if constexpr (TOP > 0)
#pragma unroll
      for (int j = 0; j < TOP; ++j) {
        if constexpr (PACK) {
          keys[(slice * TOP + j) * 64 + slot] = packed.word[j];
        } else {
          keys[(slice * TOP + j) * 64 + slot] = list.key[j];
          classes_of[(slice * TOP + j) * 64 + slot] = list.cls[j];
        }
      }
    __syncthreads();
    if (slice != 0) return;
    for (int s = 1; s < SL; ++s) {
      st.join(part[(s * 3 + 0) * 64 + slot], part[(s * 3 + 1) * 64 + slot], part[(s * 3 + 2) * 64 + slot]);
      if constexpr (TOP > 0)
        for (int j = 0; j < TOP; ++j) {
          const unsigned k = keys[(s * TOP + j) * 64 + slot];
          if constexpr (PACK) packed.insert(k);
          else if (k > list.key[TOP - 1]) list.insert(k, classes_of[(s * TOP + j) * 64 + slot]);
        }
    }
  }
  if (!live) return;
  float log_s, h;
  finish(st, &log_s, &h);
  log_prob[i] = given<DT>(row, l.cs, l.classes, symbols[i], st.m, log_s);
  entropy[i] = h;
  stats[i] = st.m;
  stats[sites + i] = log_s;
  if constexpr (TOP > 0)
#pragma unroll
    for (int j = 0; j < TOP; ++j)
      if (j < top) {
        const long long at = (ng * top + j) * hw + p;
        if constexpr (PACK) {
          top_lp[at] = log_p(key16_value<DT>(packed.word[j] >> 16), st.m, log_s);
          top_sym[at] = packed.cls(j);
        } else {
          top_lp[at] = log_p(key_value(list.key[j]), st.m, log_s);
          top_sym[at] = list.cls[j];
        }
      }
}

// ---------------------------------------------------------------- many short rows
// A wave of its own is far too much for a row of a few classes.  Here a wave takes 64 / L rows at once: their logits go
// through LDS (read as one run of 16-byte vectors where rows follow each other), then L lanes share a row, `per` adjacent
// classes each.  `per` is odd, so the lanes' addresses lane * per + k fall on different banks.  Rows are evenly spaced,
// `pitch` elements apart.
constexpr int kShortClasses = 256;        // longest row of this form
constexpr int kShortPer = 32;             // classes of a lane

struct ShortRows {
  const void* p;
  long long pitch;
  int classes, lanes, per;
  unsigned inv;                           // ceil(2^32 / classes): i / classes = umulhi(i, inv) for i < 2^16 (classes >= 2)
  __device__ __forceinline__ unsigned row_of(unsigned i) const { return classes == 1 ? i : __umulhi(i, inv); }
};

template <int DT, int TOP>
__global__ __launch_bounds__(64) void symbol_short_rows_kernel(ShortRows l, const int* symbols, int top, float* log_prob, float* entropy,
                                                               float* stats, float* top_lp, int* top_sym, int sites) {
  typedef typename Elem<DT>::type T;
  constexpr int N = Vec<DT>::N;
  constexpr bool PACK = DT != DVC_F32 && TOP > 1;    // (at most kShortClasses classes)
  extern __shared__ float tile[];         // 64 * per
  const int lane = threadIdx.x, rows = 64 / l.lanes, site0 = (int)blockIdx.x * rows;
  const int count = sites - site0 < rows ? sites - site0 : rows;
  const T* const base = static_cast<const T*>(l.p) + (long long)site0 * l.pitch;
  const int row_floats = l.lanes * l.per, total = count * l.classes;
  auto put1 = [&](int i) {
    const int r = (int)l.row_of((unsigned)i), c = i - r * l.classes;
    tile[r * row_floats + c] = Elem<DT>::up(base[(long long)r * l.pitch + c]);
  };
  if (l.pitch == l.classes) {
    const RowPart rp = row_part<DT>(base, total);
    if (lane < rp.head + total - rp.tail0) put1(lane < rp.head ? lane : rp.tail0 + lane - rp.head);
    const uint4* const body = reinterpret_cast<const uint4*>(base + rp.head);
    constexpr int U = 4;                  // vectors in flight per lane
    for (int j = lane; j < rp.body; j += U * 64) {
      Vec<DT> q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j + u * 64 < rp.body) q[u].q = body[j + u * 64];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j + u * 64 < rp.body) {
          const int i = rp.head + (j + u * 64) * N;
          const int r = (int)l.row_of((unsigned)i);
          int c = i - r * l.classes;
          float* at = tile + r * row_floats + c;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            *at = Elem<DT>::up(q[u].e[e]);
            ++at;
            if (++c == l.classes) { c = 0; at += row_floats - l.classes; }
          }
        }
    }
  } else {
    for (int i = lane; i < total; i += 64) put1(i);
  }
  const int r = lane / l.lanes, part = lane - r * l.lanes;
  const bool live = r < count;
  const int sym = live && part == 0 ? symbols[site0 + r] : -1;
  __syncthreads();

  Stat st;
  st.clear();
  ThreadList<PACK ? 0 : TOP> list;
  PackedList<PACK ? TOP : 0> packed;
  list.clear();
  packed.clear();
  if (live) {
    const float* const x = tile + lane * l.per;
    const int v0 = part * l.per, mine = l.classes - v0 < l.per ? l.classes - v0 : l.per;
    auto take = [&](float f, int k) {
      if constexpr (TOP > 0 && PACK) {
        packed.insert(packed.pack(order_key16<DT>(Elem<DT>::down(f)), v0 + k));      // (exact: it was of that type)
      } else if constexpr (TOP > 0) {
        const unsigned key = order_key(f);
        if (key > list.key[TOP - 1]) list.insert(key, v0 + k);
      }
    };
    constexpr int U = 8;
    int k = 0;
    for (; k + U <= mine; k += U) {
      float f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) f[u] = x[k + u];
      add_many<U>(&st, f);
#pragma unroll
      for (int u = 0; u < U; ++u) take(f[u], k + u);
    }
    for (; k < mine; ++k) {
      const float f = x[k];
      add_many<1>(&st, &f);
      take(f, k);
    }
  }
  // a row's first lane collects: the lane o further on holds higher classes, so equal keys go behind
  for (int o = 1; o < l.lanes; o <<= 1) {
    st.join(__shfl_down(st.m, o, 64), __shfl_down(st.s, o, 64), __shfl_down(st.t, o, 64));
    if constexpr (TOP > 0 && PACK) {
      unsigned word[TOP];
#pragma unroll
      for (int j = 0; j < TOP; ++j) word[j] = (unsigned)__shfl_down((int)packed.word[j], o, 64);
#pragma unroll
      for (int j = 0; j < TOP; ++j) packed.insert(word[j]);
    } else if constexpr (TOP > 0) {
      unsigned key[TOP];
      int cls[TOP];
#pragma unroll
      for (int j = 0; j < TOP; ++j) { key[j] = (unsigned)__shfl_down((int)list.key[j], o, 64); cls[j] = __shfl_down(list.cls[j], o, 64); }
#pragma unroll
      for (int j = 0; j < TOP; ++j)
        if (key[j] > list.key[TOP - 1]) list.insert(key[j], cls[j]);
    }
  }
  if (!live || part != 0) return;
  float log_s, h;
  finish(st, &log_s, &h);
  const int site = site0 + r;
  const float given_x = sym >= 0 && sym < l.classes ? tile[r * row_floats + sym] : 0.f;
  log_prob[site] = given_log_p(sym, l.classes, given_x, st.m, log_s);
  entropy[site] = h;
  stats[site] = st.m;
  stats[(long long)sites + site] = log_s;
  if constexpr (TOP > 0)
#pragma unroll
    for (int j = 0; j < TOP; ++j)
      if (j < top) {
        const long long at = (long long)site * top + j;
        if constexpr (PACK) {
          top_lp[at] = log_p(key16_value<DT>(packed.word[j] >> 16), st.m, log_s);
          top_sym[at] = packed.cls(j);
        } else {
          top_lp[at] = log_p(key_value(list.key[j]), st.m, log_s);
          top_sym[at] = list.cls[j];
        }
      }
}

// ---------------------------------------------------------------- gradient: one read, one write
struct SiteGrad {
  float m, log_s, h, a, b;
  int sym;
  __device__ __forceinline__ void load(int classes, const int* symbols, const float* stats, const float* entropy, const float* g_lp,
                                       const float* g_h, long long i, long long sites) {
    sym = symbols[i];
    m = stats[i];
    m = m == NEG_INF ? 0.f : m;
    log_s = stats[sites + i];
    h = entropy[i];
    a = g_lp != nullptr && sym >= 0 ? (sym < classes ? g_lp[i] : __uint_as_float(0x7fc00000u)) : 0.f;
    b = g_h != nullptr ? g_h[i] : 0.f;
  }
  __device__ __forceinline__ float of(float x, int v) const {
    const float lp = (x - m) - log_s, pv = __expf(lp);
    const float d = -pv * (a + b * (fmaxf(lp, kFloor) + h));
    return v == sym ? d + a : d;
  }
};

// Rows of up to kFlatClasses: a wave takes `rows` (at most 64) of them, their statistics wait in LDS, and the lanes go over
// the rows' logits as one run (2097152 x 37 fp32 125 us, 2455 with a workgroup per row; 262144 x 1000 bf16 204 / 393).
constexpr int kFlatClasses = 1024;

template <int DT>
__global__ __launch_bounds__(64) void symbol_short_rows_backward_kernel(ShortRows l, const int* symbols, const float* stats,
                                                                        const float* entropy, const float* g_lp, const float* g_h,
                                                                        typename Elem<DT>::type* grad, int sites, int rows) {
  typedef typename Elem<DT>::type T;
  constexpr int N = Vec<DT>::N;
  __shared__ SiteGrad of_row[64];
  const int lane = threadIdx.x, site0 = (int)blockIdx.x * rows;
  const int count = sites - site0 < rows ? sites - site0 : rows;
  const T* const base = static_cast<const T*>(l.p) + (long long)site0 * l.pitch;
  T* const out = grad + (long long)site0 * l.classes;
  const int total = count * l.classes;
  if (lane < count) of_row[lane].load(l.classes, symbols, stats, entropy, g_lp, g_h, site0 + lane, sites);
  __syncthreads();
  auto one = [&](int i) {
    const int r = (int)l.row_of((unsigned)i), c = i - r * l.classes;
    out[i] = Elem<DT>::down(of_row[r].of(Elem<DT>::up(base[(long long)r * l.pitch + c]), c));
  };
  if (l.pitch == l.classes && ((reinterpret_cast<uintptr_t>(base) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0) {
    const RowPart rp = row_part<DT>(base, total);
    if (lane < rp.head + total - rp.tail0) one(lane < rp.head ? lane : rp.tail0 + lane - rp.head);
    const uint4* const body = reinterpret_cast<const uint4*>(base + rp.head);
    uint4* const to = reinterpret_cast<uint4*>(out + rp.head);
    constexpr int U = 4;                  // vectors in flight per lane
    for (int j = lane; j < rp.body; j += U * 64) {
      Vec<DT> q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j + u * 64 < rp.body) q[u].q = body[j + u * 64];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j + u * 64 < rp.body) {
          const int i = rp.head + (j + u * 64) * N;
          int r = (int)l.row_of((unsigned)i), c = i - r * l.classes;
          SiteGrad sg = of_row[r];
#pragma unroll
          for (int e = 0; e < N; ++e) {
            q[u].e[e] = Elem<DT>::down(sg.of(Elem<DT>::up(q[u].e[e]), c));
            if (e < N - 1 && ++c == l.classes) { c = 0; sg = of_row[++r]; }
          }
          to[j + u * 64] = q[u].q;
        }
    }
  } else {
    for (int i = lane; i < total; i += 64) one(i);
  }
}

constexpr int kRowVecs = 4;      // vectors per thread of the row form

template <int DT>
__global__ __launch_bounds__(256) void symbol_rows_backward_kernel(Logits l, const int* symbols, const float* stats, const float* entropy,
                                                                   const float* g_lp, const float* g_h,
                                                                   typename Elem<DT>::type* grad, int sites, int chunks) {
  typedef typename Elem<DT>::type T;
  constexpr int N = Vec<DT>::N;
  const int site = (int)(blockIdx.x / (unsigned)chunks), chunk = (int)(blockIdx.x - (unsigned)site * chunks);
  const int n = site / l.groups, g = site - n * l.groups;
  const T* const row = static_cast<const T*>(l.p) + (long long)n * l.bs + (long long)g * l.classes;
  T* const out = grad + (long long)site * l.classes;
  SiteGrad sg;
  sg.load(l.classes, symbols, stats, entropy, g_lp, g_h, site, sites);
  RowPart rp = row_part<DT>(row, l.classes);
  const bool together = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;   // one vector grid for both
  const int j0 = chunk * 256 * kRowVecs + threadIdx.x;
  if (chunk == 0) {
    const int ends = rp.head + l.classes - rp.tail0;
    if ((int)threadIdx.x < ends) {
      const int v = (int)threadIdx.x < rp.head ? (int)threadIdx.x : rp.tail0 + (int)threadIdx.x - rp.head;
      out[v] = Elem<DT>::down(sg.of(Elem<DT>::up(row[v]), v));
    }
  }
  const uint4* const body = reinterpret_cast<const uint4*>(row + rp.head);
  Vec<DT> q[kRowVecs];
#pragma unroll
  for (int u = 0; u < kRowVecs; ++u)
    if (j0 + u * 256 < rp.body) q[u].q = body[j0 + u * 256];
#pragma unroll
  for (int u = 0; u < kRowVecs; ++u) {
    const int j = j0 + u * 256;
    if (j < rp.body) {
      const int v = rp.head + j * N;
#pragma unroll
      for (int i = 0; i < N; ++i) q[u].e[i] = Elem<DT>::down(sg.of(Elem<DT>::up(q[u].e[i]), v + i));
      if (together) {
        reinterpret_cast<uint4*>(out + rp.head)[j] = q[u].q;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) out[v + i] = q[u].e[i];
      }
    }
  }
}

constexpr int kPlaneClasses = 16;      // classes per thread of the plane form

template <int DT>
__global__ __launch_bounds__(256) void symbol_planes_backward_kernel(Logits l, const int* symbols, const float* stats,
                                                                     const float* entropy, const float* g_lp, const float* g_h,
                                                                     typename Elem<DT>::type* grad, long long sites, unsigned hw,
                                                                     unsigned chunks) {
  typedef typename Elem<DT>::type T;
  const unsigned blk = blockIdx.x / chunks, chunk = blockIdx.x - blk * chunks;
  const long long i = (long long)blk * 256 + threadIdx.x;
  if (i >= sites) return;
  const long long ng = i / hw;
  const unsigned p = (unsigned)(i - ng * hw);
  const int n = (int)(ng / l.groups), g = (int)(ng - (long long)n * l.groups);
  const T* const row = static_cast<const T*>(l.p) + (long long)n * l.bs + (long long)g * l.classes * l.cs + p;
  T* const out = grad + ng * l.classes * hw + p;
  SiteGrad sg;
  sg.load(l.classes, symbols, stats, entropy, g_lp, g_h, i, sites);
  const int v0 = (int)chunk * kPlaneClasses;
  T q[kPlaneClasses];
#pragma unroll
  for (int u = 0; u < kPlaneClasses; ++u)
    if (v0 + u < l.classes) q[u] = row[(long long)(v0 + u) * l.cs];
#pragma unroll
  for (int u = 0; u < kPlaneClasses; ++u)
    if (v0 + u < l.classes) out[(long long)(v0 + u) * hw] = Elem<DT>::down(sg.of(Elem<DT>::up(q[u]), v0 + u));
}

int check_logits(const DvcLogits* l, int batch, int h, int w, const char* who) {
  DVC_REQUIRE(l != nullptr && l->ptr != nullptr, "%s: null logits", who);
  DVC_REQUIRE(l->groups >= 1 && l->classes >= 1, "%s: bad groups / classes (%d, %d)", who, l->groups, l->classes);
  DVC_REQUIRE(l->dtype == DVC_F32 || l->dtype == DVC_BF16 || l->dtype == DVC_F16, "%s: type %d unknown", who, l->dtype);
  DVC_REQUIRE(batch >= 1 && h >= 1 && w >= 1, "%s: bad dims", who);
  DVC_REQUIRE((long long)h * w < (1LL << 28), "%s: plane too large", who);
  DVC_REQUIRE((long long)batch * l->groups < (1LL << 31) - 64, "%s: too many groups", who);
  DVC_REQUIRE(l->class_stride >= (int64_t)h * w, "%s: class stride < H*W", who);
  return DVC_OK;
}
inline Logits mk(const DvcLogits* l) { return Logits{l->ptr, l->batch_stride, l->class_stride, l->groups, l->classes}; }

// (a launch has below 2^32 threads)
inline bool fits(long long blocks, int threads) { return blocks * threads < (1ll << 32); }

// The classes of a site are adjacent: one pixel per plane and unit class stride (groups follow each other).
inline bool is_rows(const DvcLogits* l, int h, int w) {
  return h == 1 && w == 1 && (l->class_stride == 1 || (l->classes == 1 && l->groups == 1));
}

// Rows one pitch apart, whatever their group: what the short forms take.
inline bool evenly_spaced(const DvcLogits* l, int batch) {
  return l->groups == 1 || batch == 1 || l->batch_stride == (int64_t)l->groups * l->classes;
}
inline ShortRows short_rows(const DvcLogits* l, int batch) {
  ShortRows r{l->ptr, l->groups == 1 && batch > 1 ? l->batch_stride : l->classes, l->classes, 1, 0,
              l->classes == 1 ? 0u : (unsigned)(((1ull << 32) + l->classes - 1) / l->classes)};
  while (r.lanes * kShortPer < r.classes) r.lanes *= 2;
  r.per = (r.classes + r.lanes - 1) / r.lanes | 1;
  return r;
}

// Into how many parts a row is cut: while the rows alone give fewer than 512 workgroups (two per CU), as long as a part
// keeps two 16-byte vectors per thread (one row of 131072 bf16: 25 us whole, 9 us in 32 parts and a join).
inline int row_parts(const DvcLogits* l, int batch, int h, int w) {
  const long long sites = (long long)batch * l->groups;
  if (!is_rows(l, h, w) || l->classes <= 1024 || sites >= 512) return 1;
  const long long vecs = (long long)l->classes * (l->dtype == DVC_F32 ? 4 : 2) / 16, want = (512 + sites - 1) / sites;
  const long long most = vecs / 512 < kMaxParts ? vecs / 512 : kMaxParts;
  return (int)(want < most ? want : most < 1 ? 1 : most);
}

template <int DT>
int launch_forward(const DvcLogits* l, const int32_t* symbols, int top, float* log_prob, float* entropy, float* stats, float* top_lp,
                   int32_t* top_sym, float* scratch, int batch, int h, int w, hipStream_t st) {
  const unsigned hw = (unsigned)((long long)h * w);
  const long long sites = (long long)batch * l->groups * hw;
  if (is_rows(l, h, w)) {
    // Many short rows share waves (below 8192 rows both forms are the call's own latency)
    if (l->classes <= kShortClasses && sites >= 8192 && evenly_spaced(l, batch)) {
      const ShortRows r = short_rows(l, batch);
      const int rows = 64 / r.lanes;
      const dim3 grid((unsigned)((sites + rows - 1) / rows));
      DVC_REQUIRE(fits((sites + rows - 1) / rows, 64), "dvc_symbol_log_probs: too many sites");
#define SHORT(TOP) hipLaunchKernelGGL((symbol_short_rows_kernel<DT, TOP>), grid, dim3(64), 64 * r.per * sizeof(float), st, r, symbols, top, \
                                      log_prob, entropy, stats, top_lp, top_sym, (int)sites)
      if (top == 0) SHORT(0);
      else if (top == 1) SHORT(1);
      else if (top <= 4) SHORT(4);
      else if (top <= 8) SHORT(8);
      else SHORT(16);
#undef SHORT
      return dvc::check_launch("symbol_short_rows_kernel");
    }
    // a wave per row while a row is at most a few vectors per lane
    if (l->classes <= 1024) {
      DVC_REQUIRE(fits((sites + 3) / 4, 256), "dvc_symbol_log_probs: too many sites");
      hipLaunchKernelGGL((symbol_rows_kernel<DT, 64>), dim3((unsigned)((sites + 3) / 4)), dim3(256), 0, st, mk(l), symbols, top, log_prob,
                         entropy, stats, top_lp, top_sym, (int)sites, 1, Parts{});
      return dvc::check_launch("symbol_rows_kernel");
    }
    const int nparts = row_parts(l, batch, h, w);
    const long long units = sites * nparts;
    DVC_REQUIRE(fits(units, 256), "dvc_symbol_log_probs: too many sites");
    Parts parts{};
    if (nparts > 1) {
      DVC_REQUIRE(scratch != nullptr, "dvc_symbol_log_probs: null scratch");
      parts = Parts{scratch, reinterpret_cast<unsigned*>(scratch + units * 3), reinterpret_cast<int*>(scratch + units * (3 + top))};
    }
    hipLaunchKernelGGL((symbol_rows_kernel<DT, 256>), dim3((unsigned)units), dim3(256), 0, st, mk(l), symbols, top, log_prob, entropy,
                       stats, top_lp, top_sym, (int)sites, nparts, parts);
    if (int rc = dvc::check_launch("symbol_rows_kernel")) return rc;
    if (nparts == 1) return DVC_OK;
    hipLaunchKernelGGL(symbol_rows_join_kernel<DT>, dim3((unsigned)sites), dim3(64), 0, st, mk(l), symbols, top, log_prob, entropy, stats,
                       top_lp, top_sym, (int)sites, nparts, parts);
    return dvc::check_launch("symbol_rows_join_kernel");
  }
  const long long waves = (sites + 63) / 64;
  DVC_REQUIRE(fits((sites + 255) / 256, 256), "dvc_symbol_log_probs: too many sites");
#define PLANES(TOP, SL, PACK)                                                                                                          \
  hipLaunchKernelGGL((symbol_planes_kernel<DT, TOP, SL, PACK>), dim3((unsigned)((sites + (SL == 1 ? 255 : 63)) / (SL == 1 ? 256 : 64))), \
                     dim3(SL == 1 ? 256 : 64 * SL), 0, st, mk(l), symbols, top, log_prob, entropy, stats, top_lp, top_sym, sites, hw)
  // Cut the classes while the sites alone give fewer than eight waves per CU and a range keeps eight classes; the joining
  // lists of 16 ranges fit LDS up to 4 alternatives
#define SLICES_OF(TOP, PACK)                                                                     \
  do {                                                                                           \
    if (TOP <= 4 && waves < 512 && l->classes >= 128) PLANES(TOP, (TOP <= 4 ? 16 : 4), PACK);    \
    else if (waves < 2048 && l->classes >= 32) PLANES(TOP, 4, PACK);                             \
    else PLANES(TOP, 1, PACK);                                                                   \
  } while (0)
#define SLICES(TOP)                                                                              \
  do {                                                                                           \
    if (TOP > 1 && DT != DVC_F32 && l->classes <= kPackedClasses) SLICES_OF(TOP, (TOP > 1 && DT != DVC_F32)); \
    else SLICES_OF(TOP, false);                                                                  \
  } while (0)
  if (top == 0) SLICES(0);
  else if (top == 1) SLICES(1);
  else if (top <= 4) SLICES(4);
  else if (top <= 8) SLICES(8);
  else SLICES(16);
#undef SLICES
#undef SLICES_OF
#undef PLANES
  return dvc::check_launch("symbol_planes_kernel");
}

template <int DT>
int launch_backward(const DvcLogits* l, const int32_t* symbols, const float* stats, const float* entropy, const float* g_lp,
                    const float* g_h, void* grad, int batch, int h, int w, hipStream_t st, const char* who) {
  typedef typename Elem<DT>::type T;
  const unsigned hw = (unsigned)((long long)h * w);
  const long long sites = (long long)batch * l->groups * hw;
  if (is_rows(l, h, w) && l->classes <= kFlatClasses && evenly_spaced(l, batch)) {
    // up to 4096 logits a wave, fewer while that gives below 2048 waves
    int rows = 64;
    while (rows > 1 && ((long long)rows * l->classes > 4096 || sites < 2048ll * rows)) rows /= 2;
    DVC_REQUIRE(fits((sites + rows - 1) / rows, 64), "%s: too many sites", who);
    hipLaunchKernelGGL(symbol_short_rows_backward_kernel<DT>, dim3((unsigned)((sites + rows - 1) / rows)), dim3(64), 0, st,
                       short_rows(l, batch), symbols, stats, entropy, g_lp, g_h, static_cast<T*>(grad), (int)sites, rows);
    return dvc::check_launch("symbol_short_rows_backward_kernel");
  }
  if (is_rows(l, h, w)) {
    const int per = 256 * kRowVecs * Vec<DT>::N;
    const long long chunks = (l->classes + per - 1) / per;
    DVC_REQUIRE(fits(sites * chunks, 256), "%s: too many sites", who);
    hipLaunchKernelGGL(symbol_rows_backward_kernel<DT>, dim3((unsigned)(sites * chunks)), dim3(256), 0, st, mk(l), symbols, stats, entropy,
                       g_lp, g_h, static_cast<T*>(grad), (int)sites, (int)chunks);
    return dvc::check_launch("symbol_rows_backward_kernel");
  }
  const long long chunks = (l->classes + kPlaneClasses - 1) / kPlaneClasses, blocks = (sites + 255) / 256;
  DVC_REQUIRE(fits(blocks * chunks, 256), "%s: too many sites", who);
  hipLaunchKernelGGL(symbol_planes_backward_kernel<DT>, dim3((unsigned)(blocks * chunks)), dim3(256), 0, st, mk(l), symbols, stats, entropy,
                     g_lp, g_h, static_cast<T*>(grad), sites, hw, (unsigned)chunks);
  return dvc::check_launch("symbol_planes_backward_kernel");
}

}  // namespace

extern "C" int64_t dvc_symbol_log_probs_scratch_floats(const DvcLogits* logits, int32_t top, int32_t batch, int32_t h, int32_t w) {
  if (int rc = check_logits(logits, batch, h, w, "dvc_symbol_log_probs_scratch_floats")) return rc;
  DVC_REQUIRE(top >= 0 && top <= DVC_MAX_TOP, "dvc_symbol_log_probs_scratch_floats: top=%d (0..%d)", top, DVC_MAX_TOP);
  const int nparts = row_parts(logits, batch, h, w);
  return nparts == 1 ? 0 : (int64_t)batch * logits->groups * nparts * (3 + 2 * top);
}

extern "C" int dvc_symbol_log_probs(const DvcLogits* logits, const int32_t* symbols, int32_t top, float* log_prob, float* entropy,
                                    float* stats, float* top_log_prob, int32_t* top_symbol, float* scratch, int32_t batch,
                                    int32_t h, int32_t w, void* stream) {
  if (int rc = check_logits(logits, batch, h, w, "dvc_symbol_log_probs")) return rc;
  DVC_REQUIRE(symbols != nullptr && log_prob != nullptr && entropy != nullptr && stats != nullptr, "dvc_symbol_log_probs: null pointer");
  DVC_REQUIRE(top >= 0 && top <= DVC_MAX_TOP && top <= logits->classes, "dvc_symbol_log_probs: top=%d (0..%d, at most the %d classes)",
              top, DVC_MAX_TOP, logits->classes);
  DVC_REQUIRE(top == 0 || (top_log_prob != nullptr && top_symbol != nullptr), "dvc_symbol_log_probs: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
#define GO(DT) launch_forward<DT>(logits, symbols, top, log_prob, entropy, stats, top_log_prob, top_symbol, scratch, batch, h, w, st)
  return logits->dtype == DVC_F32 ? GO(DVC_F32) : logits->dtype == DVC_BF16 ? GO(DVC_BF16) : GO(DVC_F16);
#undef GO
}

extern "C" int dvc_symbol_log_probs_backward(const DvcLogits* logits, const int32_t* symbols, const float* stats, const float* entropy,
                                             const float* grad_log_prob, const float* grad_entropy, void* grad_logits, int32_t batch,
                                             int32_t h, int32_t w, void* stream) {
  const char* const who = "dvc_symbol_log_probs_backward";
  if (int rc = check_logits(logits, batch, h, w, who)) return rc;
  DVC_REQUIRE(symbols != nullptr && stats != nullptr && entropy != nullptr && grad_logits != nullptr, "%s: null pointer", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define GO(DT) launch_backward<DT>(logits, symbols, stats, entropy, grad_log_prob, grad_entropy, grad_logits, batch, h, w, st, who)
  return logits->dtype == DVC_F32 ? GO(DVC_F32) : logits->dtype == DVC_BF16 ? GO(DVC_BF16) : GO(DVC_F16);
#undef GO
}
