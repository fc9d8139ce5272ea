// Beam search on the paged cache, gfx950: the n best continuations of a
// request's beams (beam_part_kernel, beam_join_kernel) and the cache following
// them (beam_reorder_kernel).
//
// Selection. total(k, v) = score_k + logit_kv - log sum_v exp(logit_kv) over the
// K beams of a request and the vocabulary; the n largest, the lower beam and then
// the lower token first among equals. Inside a beam the order of the totals is
// that of the logits, so the vocabulary is read once: a wavefront takes a part of
// a row and leaves its maximum, its sum of exponentials and its n best tokens; one
// workgroup per request joins the parts. A part is one step of the wavefront, whose
// values stay in LDS, or several, of which only each lane's maximum stays and the
// few values that the selection needs are read again from memory.
//
// The sums and totals are 64-bit: which of two beams' tokens comes first hangs on
// their difference, and 32 bits of a sum over a vocabulary of 1e5 leave 1e-6 of a
// total undecided, which a search over a thousand candidates a step does meet. (The
// exponentials are good to 6e-11, so totals nearer than about 1e-10 may change places.)
//
// n best of a wavefront's values: the n-th largest of the 64 lanes' own maxima
// bounds the n-th largest value from below. nth_largest finds it two bits a round,
// with three ballots, and ends as soon as exactly n lanes reach the bound; where no
// more than n lanes hold anything, everything is taken. Mostly a few more than n
// values then reach the bound, all in those lanes; they are listed in LDS and ranked
// by counting. Where equal values let more than 64 reach it, the best is taken n
// times: the largest of the lanes' best keys (the value in an order-preserving code
// above the complement of the token, so that no two are equal), after which the lane
// that had it gets its next one, all lanes reading one unit of its values each.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "pdk_common.h"

namespace {

using pdk::v8;

constexpr int kMaxBeams = 16;
constexpr int kMaxOut = 32;
constexpr int kWaves = 4;                 // of a part workgroup, each a part of its own
constexpr int kMaxLists = 8;              // parts of a row per lane of the join
constexpr int kMaxVocab = 1 << 20;
constexpr int kBusyWaves = 4096;          // four for each SIMD
constexpr int kMaxSteps = 16;             // of a part
constexpr uint32_t kLeastCode = 0x00800000u;   // of the lowest finite value

typedef unsigned long long Key;

// Order-preserving 32-bit code of x, -0 equal to 0, 0 for -inf and below any
// other code: a token at -inf is none.
__device__ __forceinline__ uint32_t code_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x == -INFINITY ? 0u : (u >> 31 ? ~u : u | 0x80000000u);
}

__device__ __forceinline__ float value_of(uint32_t code) {
  return __uint_as_float(code >> 31 ? code & 0x7fffffffu : ~code);
}

__device__ __forceinline__ Key key_of(float x, uint32_t token) {
  const uint32_t c = code_of(x);
  return c ? ((Key)c << 32) | (0xffffffffu - token) : 0ull;
}

constexpr double kLog2e = 1.4426950408889634074;

// e^x for |x| <= 700: 2^k p(f), x log2(e) = k + f, |f| <= 1/2, p the polynomial
// of degree 7 that meets 2^f at the 8 Chebyshev nodes (off by less than 6e-11 of
// it). k is left in the low bits of a sum with 3 * 2^51 and added to the exponent.
__device__ __forceinline__ double exp_of(double x) {
  constexpr double kRound = 6755399441055744.0;
  const double t = fma(x, kLog2e, kRound);
  const double f = fma(x, kLog2e, kRound - t);
  double p = 1.5303701161442145e-05;
  p = fma(p, f, 0.00015469729221575116);
  p = fma(p, f, 0.0013333478471058548);
  p = fma(p, f, 0.009618025613268967);
  p = fma(p, f, 0.055504109063307244);
  p = fma(p, f, 0.24022651213498578);
  p = fma(p, f, 0.6931471805568296);
  p = fma(p, f, 0.9999999999595621);
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}

// ln x for 1/2 <= x <= 2^64: a 32-bit logarithm and one Newton step in 64 bits,
// which leaves the square of its error and exp_of's.
__device__ __forceinline__ double log_of(double x) {
  const double y = (double)__logf((float)x);
  const double e = x * exp_of(-y) - 1.0;
  return y + (e - 0.5 * e * e);
}

// x reduced over the wavefront by f, the same in every lane: halves and quarters
// exchanged by the lane swaps, rows of 16 lanes by rotations (no LDS round trip, a
// tenth of the time of six __shfl_xor). f is symmetric, so all lanes end with the
// same bits.
template <typename T, class F>
__device__ __forceinline__ T wave_all(T x, F f) {
  constexpr int W = sizeof(T) / 4;
  union U {
    T v;
    uint32_t w[W];
  };
  U a{x}, b;
  auto swap = [&](auto op) __attribute__((always_inline)) {
    U c;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const auto r = op(a.w[i]);
      b.w[i] = r[0];
      c.w[i] = r[1];
    }
    a.v = f(b.v, c.v);
  };
  swap([](uint32_t v) { return __builtin_amdgcn_permlane32_swap(v, v, false, false); });
  swap([](uint32_t v) { return __builtin_amdgcn_permlane16_swap(v, v, false, false); });
  auto turn = [&](auto ctrl) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      b.w[i] = __builtin_amdgcn_update_dpp(0, a.w[i], decltype(ctrl)::value, 0xf, 0xf, true);
    a.v = f(a.v, b.v);
  };
  turn(std::integral_constant<int, 0x128>{});            // row_ror:8, 4, 2, 1
  turn(std::integral_constant<int, 0x124>{});
  turn(std::integral_constant<int, 0x122>{});
  turn(std::integral_constant<int, 0x121>{});
  return a.v;
}

__device__ __forceinline__ double wave_sum(double x) {
  return wave_all(x, [](double a, double b) { return a + b; });
}

// The n-th largest of the wavefront's 64 values (0 if no more than n are not 0),
// or a lower bound that no more of them reach: two bits at a time from the top,
// the largest bound that n lanes reach.
template <typename U>
__device__ __forceinline__ U nth_largest(U mine, int n) {
  if (__popcll(__ballot(mine != 0)) <= n) return 0;
  U bound = 0;
#pragma unroll 1
  for (int bit = 8 * sizeof(U) - 2; bit >= 0; bit -= 2) {
    const U t1 = bound | ((U)1 << bit), t2 = bound | ((U)2 << bit), t3 = bound | ((U)3 << bit);
    const int c1 = __popcll(__ballot(mine >= t1)), c2 = __popcll(__ballot(mine >= t2));
    const int c3 = __popcll(__ballot(mine >= t3));
    const U next = c3 >= n ? t3 : c2 >= n ? t2 : c1 >= n ? t1 : bound;
    const int c = c3 >= n ? c3 : c2 >= n ? c2 : c1;
    bound = next;
    if (c == n) break;
  }
  return bound;
}

// Bits of `who` below the lane's own.
__device__ __forceinline__ int below(uint64_t who) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
}

// What the wavefront's lanes wrote to LDS is there for all of them.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ Key lane_key(Key k, int lane) {
  return ((Key)__builtin_amdgcn_readlane((uint32_t)(k >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((uint32_t)k, lane);
}

// The largest n of list[0..c) in order to best[0..n), zeros behind them.
__device__ __forceinline__ void rank(const Key* list, int c, Key* best, int n) {
  const int lane = threadIdx.x & 63;
  if (c <= 64) {
    const Key mine = lane < c ? list[lane] : 0;
    int r = 0;
    for (int j = 0; j < c; ++j) r += lane_key(mine, j) > mine;
    if (lane < c && r < n) best[r] = mine;
    if (lane >= c && lane < n) best[lane] = 0;
    return;
  }
  for (int i = lane; i < c; i += 64) {
    const Key mine = list[i];
    int r = 0;
    for (int j = 0; j < c; ++j) r += list[j] > mine;
    if (r < n) best[r] = mine;
  }
}

// What a part leaves: its maximum and its sum of e^(x - maximum) (NaN where the
// part holds a NaN or +inf).
struct Part {
  double top, sum;
};

// 16 bytes of a row, the values in their own type.
struct Unit {
  uint32_t w[4];
};

// f(value) of a unit's values in turn.
template <typename T, class F>
__device__ __forceinline__ void each_value(const Unit& u, F f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      f(2 * i, __uint_as_float(u.w[i] << 16));
      f(2 * i + 1, __uint_as_float(u.w[i] & 0xffff0000u));
    } else {
      f(i, __uint_as_float(u.w[i]));
    }
  }
}

// The unit whose first value is the row's value e: it starts at unit_at(e), and the
// values in front of e, which the unit before it holds, are -inf, all of them where
// e is V or more. Rows of odd lengths start anywhere: the 16-byte loads take any
// address, and a row's parts and sums do not depend on where it lies (equal rows
// have equal totals).
template <typename T>
__device__ __forceinline__ int unit_at(int e, int V) {
  return min(e, max(V - (int)(16 / sizeof(T)), 0));
}

template <typename T>
__device__ __forceinline__ void drop_front(Unit& u, int n) {
  constexpr uint32_t kNone = sizeof(T) == 2 ? 0xff80u : 0xff800000u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      if (2 * i < n) u.w[i] = (u.w[i] & 0xffff0000u) | kNone;
      if (2 * i + 1 < n) u.w[i] = (u.w[i] & 0xffffu) | (kNone << 16);
    } else {
      if (i < n) u.w[i] = kNone;
    }
  }
}

// A row of fewer values than a unit: those in front of value e dropped as above.
template <typename T>
__device__ __forceinline__ Unit short_row(const T* p, int V) {
  T x[16 / sizeof(T)];
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) {
    if constexpr (sizeof(T) == 2) x[i] = i < V ? p[i] : 0xff80;
    else x[i] = i < V ? p[i] : -INFINITY;
  }
  Unit u;
  __builtin_memcpy(&u, x, 16);
  return u;
}

// grid: x = kWaves parts, y = row. T is uint16_t (bf16) or float. A part is `steps`
// times 64 lanes' kVals values, the next step's on their way while one's are summed;
// bound by the 64-bit operations of that (14 for a value, of some 20 instructions in
// all). Of the steps only each lane's maximum is kept: the selection reads the few
// lanes' values it needs again, from LDS if there is one step only, else from memory.
// kShort: V is less than a unit.
template <typename T, int kVals, bool kMany, bool kShort = false>
__global__ __launch_bounds__(64 * kWaves) void beam_part_kernel(const T* logits, int64_t ld, int V,
                                                                int n, int n_parts, int steps,
                                                                const int32_t* last_tokens,
                                                                int eos, Part* parts, Key* keys) {
  constexpr int kEl = 16 / sizeof(T), kUnits = kVals / kEl, kStep = 64 * kVals;
  static_assert(!kMany || kMaxSteps * kUnits <= 64, "one unit of a lane's for every lane");
  __shared__ Unit held[kWaves][kMany ? 1 : kUnits * 64];         // [unit][lane]
  __shared__ float most[kWaves][kMany ? kMaxSteps * 64 : 1];     // [step][lane]
  __shared__ Key lists[kWaves][64];
  __shared__ uint16_t places[kWaves][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = blockIdx.y, part = blockIdx.x * kWaves + wave;
  if (part >= n_parts) return;
  if (last_tokens && last_tokens[row] == eos) return;   // an ended beam's logits count for nothing
  const T* p = logits + (int64_t)row * ld;
  const int first = part * (kMany ? steps : 1) * kStep;  // of the part's values
  if (kMany) steps = min(steps, (V - first + kStep - 1) / kStep);
  else steps = 1;
  auto value_at = [&](int step, int unit, int of) {
    return first + step * kStep + (unit * 64 + of) * kEl;
  };
  auto load = [&](int e) __attribute__((always_inline)) {
    Unit u;
    if constexpr (kShort) u = short_row(p, V);
    else __builtin_memcpy(&u, p + unit_at<T>(e, V), 16);
    return u;
  };
  auto load_step = [&](Unit* u, int step) __attribute__((always_inline)) {
    if (!kShort && first + (step + 1) * kStep <= V) {
      const T* q = p + first + step * kStep;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) __builtin_memcpy(&u[i], q + (i * 64 + lane) * kEl, 16);
      return;
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int e = value_at(step, i, lane);
      u[i] = load(e);
      drop_front<T>(u[i], e - unit_at<T>(e, V));
    }
  };
  // sum is that of e^(x - ref), ref the first step's maximum: 64 bits hold what lies
  // up to 600 above it, and only beyond that it is taken anew.
  auto larger = [](float a, float b) { return __builtin_elementwise_maximum(a, b); };
  float ref = -INFINITY, best = -INFINITY;               // of the part; of the lane
  double sum = 0.0;                                      // the lane's
  auto use = [&](const Unit* u, int step) __attribute__((always_inline)) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      if (!kMany) held[wave][i * 64 + lane] = u[i];
      each_value<T>(u[i], [&](int, float x) { m = __builtin_elementwise_maximum(m, x); });
    }
    if (kMany) most[wave][step * 64 + lane] = m;
    best = __builtin_elementwise_maximum(best, m);
    if (__ballot(m > ref + 600.f)) {
      const float top = wave_all(m, larger);
      if (!(top < INFINITY)) {                           // the part counts for nothing (below)
        ref = 0.f;
      } else {
        if (kMany) sum *= exp_of(fmax((double)ref - (double)top, -690.0));
        ref = top;
      }
    }
    if (ref == -INFINITY) return;                        // nothing above -inf yet
    // Clamped in 32 bits, near enough to ref to be exact there.
    if (fabsf(ref) <= 4096.f) {
      const double r = ref;
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        each_value<T>(u[i], [&](int, float x) {
          sum += exp_of((double)__builtin_amdgcn_fmed3f(x, ref - 690.f, ref + 690.f) - r);
        });
    } else {
#pragma unroll 1
      for (int i = 0; i < kUnits; ++i) {
        const int e = value_at(step, i, lane), skip = kMany ? e - unit_at<T>(e, V) : 0;
        each_value<T>(kMany ? load(e) : held[wave][i * 64 + lane], [&](int j, float x) {
          sum += j < skip ? 0.0 : exp_of((double)__builtin_amdgcn_fmed3f(x - ref, -690.f, 690.f));
        });
      }
    }
  };
  {
    Unit u[kUnits];
    load_step(u, 0);
    if constexpr (kMany) {
      Unit v[kUnits];
#pragma unroll 1
      for (int step = 0; step < steps; step += 2) {
        if (step + 1 < steps) load_step(v, step + 1);
        use(u, step);
        if (step + 1 >= steps) break;
        if (step + 2 < steps) load_step(u, step + 2);
        use(v, step + 1);
      }
    } else {
      use(u, 0);
    }
  }
  sum = wave_sum(sum);
  const float top = wave_all(best, larger);
  if (kMany) sum *= exp_of(fmax((double)ref - (double)top, -690.0));
  if (!(top < INFINITY)) sum = NAN;
  const int64_t at = (int64_t)row * n_parts + part;
  if (lane == 0) parts[at] = Part{(double)top, sum};

  // The values that reach the bound, of the lanes' steps whose maximum does; all but
  // -inf where there are few enough.
  auto unit_of = [&](int step, int unit, int of) {
    return kMany ? load(value_at(step, unit, of)) : held[wave][unit * 64 + of];
  };
  Key* list = lists[wave];
  uint16_t* place = places[wave];
  const uint32_t code = code_of(best), bound = max(nth_largest(code, n), kLeastCode);
  const float least = value_of(bound);
  int c = 0, m = 0;
  for (int s = 0; s < steps; ++s) {
    const bool in = (kMany ? code_of(most[wave][s * 64 + lane]) : code) >= bound;
    const uint64_t who = __ballot(in);
    const int to = m + below(who);
    if (in && to < 64) place[to] = (uint16_t)(s * 64 + lane);
    m += __popcll(who);
  }
  wave_sync();
  if (m > 64) c = 65;
#pragma unroll 1
  for (int t0 = 0; t0 < m * kUnits && c <= 64; t0 += 64) {
    const int t = min(t0 + lane, m * kUnits - 1), unit = t % kUnits, at = place[t / kUnits];
    const int e = value_at(at >> 6, unit, at & 63), start = unit_at<T>(e, V);
    each_value<T>(unit_of(at >> 6, unit, at & 63), [&](int i, float x) {
      const bool in = t0 + lane < m * kUnits && x >= least && (!kMany || start + i >= e);
      const uint64_t which = __ballot(in);
      const int to = c + below(which);
      if (in && to < 64) list[to] = key_of(x, start + i);
      c += __popcll(which);
    });
  }
  if (c > 64) {                                          // many equal values: one by one
    auto best_of = [&](Key& k1, int step, int unit, int of, Key last) __attribute__((always_inline)) {
      const int e = value_at(step, unit, of), start = unit_at<T>(e, V);
      each_value<T>(unit_of(step, unit, of), [&](int i, float x) {
        const Key k = key_of(x, start + i);
        k1 = k > k1 && k < last && (!kMany || start + i >= e) ? k : k1;
      });
    };
    auto larger_key = [](Key a, Key b) { return a > b ? a : b; };
    Key mine = 0;                                        // the lane's best that is not taken yet
#pragma unroll 1
    for (int i = 0; i < steps * kUnits; ++i) best_of(mine, i / kUnits, i % kUnits, lane, ~0ull);
#pragma unroll 1
    for (c = 0; c < n; ++c) {
      const Key taken = wave_all(mine, larger_key);
      if (!taken) break;
      list[c] = taken;
      // All lanes look for the next of the lane that had it.
      const int of = __builtin_ctzll(__ballot(mine == taken));
      Key next = 0;
      if (lane < steps * kUnits) best_of(next, lane / kUnits, lane % kUnits, of, taken);
      next = wave_all(next, larger_key);
      if (lane == of) mine = next;
    }
  }
  wave_sync();
  rank(list, c, keys + at * n, n);
}

// One workgroup per request, one wavefront per beam: the beam's log sum, its n
// best tokens of all parts and their totals; then every candidate counts those
// that come before it. Each workgroup runs this code once, so what it takes is
// mostly the instructions' first fetch: one call of each helper, no unrolling.
__global__ __launch_bounds__(64 * kMaxBeams) void beam_join_kernel(
    const Part* parts, const Key* keys, int n_parts, int n, const float* scores, int K,
    const int32_t* last_tokens, int eos, int32_t* tokens, int32_t* parents, float* out_scores) {
  constexpr int kList = 512;                             // keys of a beam held at a time
  __shared__ Key list[kMaxBeams][kList];
  __shared__ Key best[kMaxBeams][kMaxOut];
  __shared__ uint16_t lists[kMaxBeams][kMaxOut * kMaxLists];
  __shared__ double totals[kMaxBeams * kMaxOut];         // [beam][n]
  const int r = blockIdx.x, lane = threadIdx.x & 63;
  const int k = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = r * K + k;
  // Heads of the parts' lists; only lists whose head reaches the n-th largest of the
  // lanes' own best heads hold any of the n best: those of at most n lanes. Where
  // there are fewer than 64 lists, the other lanes' keys are the next of them. Of up
  // to 128 parts all is asked for at once, an ended beam's (never written) too.
  const Key* kp = keys + (int64_t)row * n_parts * n;
  const Part* pp = parts + (int64_t)row * n_parts;
  const int next = n_parts < 64 ? lane / n_parts : 0;
  const bool in0 = next < n, in1 = lane + 64 < n_parts;
  const Key key0 = kp[in0 ? (lane - next * n_parts) * n + next : 0];
  const Key key1 = kp[in1 ? (lane + 64) * n : 0];
  const Part part0 = pp[min(lane, n_parts - 1)], part1 = pp[in1 ? lane + 64 : 0];
  const bool ended = last_tokens && last_tokens[row] == eos;
  const float score = scores[row];
  const bool alive = score > -INFINITY && score < INFINITY;
  double total = lane == 0 && alive ? (double)score : -INFINITY;   // of an ended beam
  int32_t token = eos;
  if (!ended) {
    const Key head0 = in0 ? key0 : 0, head1 = in1 ? key1 : 0;
    Key mine = head0 > head1 ? head0 : head1;
    double top = fmax(part0.top, in1 ? part1.top : -INFINITY), sum = 0.0;
#pragma unroll 1
    for (int s = lane + 128; s < n_parts; s += 64) {
      const Key head = kp[s * n];
      mine = head > mine ? head : mine;
      top = fmax(top, pp[s].top);
    }
    top = wave_all(top, [](double a, double b) { return fmax(a, b); });
#pragma unroll 1
    for (int s = lane, i = 0; s < n_parts; s += 64, ++i) {
      const Part q = i == 0 ? part0 : i == 1 ? part1 : pp[s];
      // NaN in q.sum stays; a part without a finite value adds nothing.
      sum += q.sum != 0.0 ? q.sum * exp_of(fmax(q.top - top, -690.0)) : 0.0;
    }
    const double log_sum = log_of(wave_sum(sum));        // beside the maximum: it may be any size
    // By the codes first; the tokens count only where equal codes leave too many.
    const uint32_t code = nth_largest((uint32_t)(mine >> 32), n);
    Key least = code ? (Key)code << 32 : 1;
    if (__popcll(__ballot(mine >= least)) > n) {         // equal codes: of those, the first tokens
      const uint32_t c = (uint32_t)(mine >> 32);
      const int more = n - __popcll(__ballot(c > code));
      least |= nth_largest(c == code ? (uint32_t)mine : 0u, more);
    }
    int m = 0;                                           // lists that reach it
#pragma unroll 1
    for (int s = lane, i = 0; s - lane < n_parts; s += 64, ++i) {
      const Key head = i == 0 ? head0 : i == 1 ? head1 : kp[min(s, n_parts - 1) * n];
      const bool in = s < n_parts && head >= least;
      const uint64_t who = __ballot(in);
      if (in) lists[k][m + below(who)] = (uint16_t)s;
      m += __popcll(who);
    }
    wave_sync();
    int c = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < m * n; i0 += 256) {            // four loads of a lane in flight
      Key q[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int i = i0 + 64 * x + lane, which = i / n;
        q[x] = i < m * n ? kp[(int)lists[k][which] * n + (i - which * n)] : 0;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const bool in = q[x] >= least;
        const uint64_t who = __ballot(in);
        if (in) list[k][c + below(who)] = q[x];
        c += __popcll(who);
      }
      if (c <= kList - 256 && i0 + 256 < m * n) continue;
      wave_sync();                                       // the n best so far
      rank(list[k], c, best[k], n);
      wave_sync();
      if (lane < n) list[k][lane] = best[k][lane];
      c = n;
    }
    const Key b = m && lane < n ? best[k][lane] : 0;
    // (log_sum of a row without a finite value, or with NaN or +inf, is NaN.)
    const bool ok = b && alive && log_sum >= 0.0 - 1e-6;
    token = (int32_t)(0xffffffffu - (uint32_t)b);
    total = ok ? (double)score + (((double)value_of((uint32_t)(b >> 32)) - top) - log_sum) : -INFINITY;
  }
  if (lane < n) totals[k * n + lane] = total;
  __syncthreads();
  // Candidate lane % w of the beam counts every 64 / w-th of all that there are.
  const int w = n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32, i = lane & (w - 1);
  const double mine = i < n ? totals[k * n + i] : -INFINITY;
  int at = 0, found = 0;
  for (int j0 = lane / w; j0 < K * n; j0 += 4 * (64 / w)) {
    double u[4];                                         // four reads in flight
#pragma unroll
    for (int x = 0; x < 4; ++x) u[x] = totals[min(j0 + x * (64 / w), K * n - 1)];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int j = j0 + x * (64 / w);
      const bool in = j < K * n;
      at += in & ((u[x] > mine) | ((u[x] == mine) & (j < k * n + i)));
      found += in & (u[x] > -INFINITY);
    }
  }
  for (int o = w; o < 64; o <<= 1) {
    at += __shfl_xor(at, o);
    found += __shfl_xor(found, o);
  }
  if (lane < n && total > -INFINITY && at < n) {
    tokens[(int64_t)r * n + at] = token;
    parents[(int64_t)r * n + at] = k;
    out_scores[(int64_t)r * n + at] = (float)total;
  }
  if (k == 0 && lane < n && lane >= found) {             // fewer candidates than asked for
    tokens[(int64_t)r * n + lane] = -1;
    parents[(int64_t)r * n + lane] = -1;
    out_scores[(int64_t)r * n + lane] = -INFINITY;
  }
}

// Reordering. Beam k of request r goes on from beam p = parents[r][k]: its table
// takes p's entries of the filled blocks (shared from now on, never written
// again), and its own block at the partly filled place the contents of p's there.
// A lane carries one 16-byte place of that block for all beams of the request
// (or one table column): it has read every beam's before it writes any, so beams
// may swap, and no two lanes touch one address: no staging, no second launch.
// Bound by the bytes of the blocks that move.
// What steers a workgroup (the count of tokens, the parents, the blocks' ids) is
// read as scalars; the launch writes none of it (of the tables only entries below
// the one that is read).
// Consecutive workgroups move the blocks of one layer.
// grid: x = chunk, y = r, z = 2 * layer + (0 for K, 1 for V) or, last, the tables.
// kK: at least K.
template <int kK>
__global__ __launch_bounds__(256) void beam_reorder_kernel(const int32_t* parents,
                                                           const int32_t* ctx_lens, int K,
                                                           int32_t* tables, int max_blocks,
                                                           uint16_t* ck, uint16_t* cv,
                                                           int64_t layer_stride, int num_blocks,
                                                           int block_units) {
  typedef const __attribute__((address_space(4))) int32_t* scalars;
  const int r = blockIdx.y;
  const int held = ((scalars)ctx_lens)[(int64_t)r * K];  // the same for a request's beams
  int32_t* rows = tables + (int64_t)r * K * max_blocks;
  int from[kK];                                          // the beam that beam k goes on from
#pragma unroll
  for (int k = 0; k < kK; ++k) {
    const int p = ((scalars)parents)[(int64_t)r * K + min(k, K - 1)];
    from[k] = k < K && p >= 0 && p < K ? p : k;          // no parent: the beam stays itself
  }
  if (held <= 0) return;
  const int full = held / PDK_BLOCK_SIZE;
  if (blockIdx.z == gridDim.z - 1) {
    const int cols = min(full, max_blocks);
    for (int j = blockIdx.x * 256 + threadIdx.x; j < cols; j += gridDim.x * 256) {
      int32_t id[kK];
#pragma unroll
      for (int k = 0; k < kK; ++k)
        if (from[k] != k) id[k] = rows[(int64_t)from[k] * max_blocks + j];
#pragma unroll
      for (int k = 0; k < kK; ++k)
        if (from[k] != k) rows[(int64_t)k * max_blocks + j] = id[k];
    }
    return;
  }
  const int u = blockIdx.x * 256 + threadIdx.x;
  if (held % PDK_BLOCK_SIZE == 0 || full >= max_blocks) return;
  int place[kK];                                         // beam k's partly filled block
#pragma unroll
  for (int k = 0; k < kK; ++k)
    place[k] = ((scalars)rows)[(int64_t)min(k, K - 1) * max_blocks + full];
  uint16_t* base = (blockIdx.z & 1 ? cv : ck) + (int64_t)(blockIdx.z >> 1) * layer_stride +
                   (int64_t)u * 8;
  const int64_t block = (int64_t)block_units * 8;
  v8 x[kK];
  bool moves[kK];
#pragma unroll
  for (int k = 0; k < kK; ++k) {
    int src = place[0];
#pragma unroll
    for (int p = 1; p < kK; ++p) src = from[k] == p ? place[p] : src;
    moves[k] = from[k] != k && src >= 0 && src < num_blocks && place[k] >= 0 &&
               place[k] < num_blocks;
    if (moves[k] && u < block_units) x[k] = pdk::ld16(base + src * block);
  }
#pragma unroll
  for (int k = 0; k < kK; ++k)
    if (moves[k] && u < block_units) pdk::st16(base + place[k] * block, x[k]);
}

// How rows are cut into parts (times of both launches, 128256 values a row, in us).
// Up to four wavefronts for each SIMD a part is one step: 16 values a lane, or 32
// where that still gives every SIMD two wavefronts (4 rows 13.5 and 14.9, 64 rows
// 16.8 and 15.2, 16.7 as two steps of 16). Beyond, steps of 16, as many as leave
// four wavefronts for each SIMD, all of them resident (256 fp32 rows: 38.7, steps of
// 32 40.8, one step of 32 a part 43.9).
struct Cut {
  int vals, steps, n_parts;
};

Cut cut_of(int rows, int V) {
  Cut c;
  const int64_t waves = (int64_t)rows * ((V + 2047) / 2048);
  c.vals = waves <= kBusyWaves && (waves >= 2048 || V > kMaxVocab / 2) ? 32 : 16;
  c.steps = 1;
  if (waves > kBusyWaves) {
    const int64_t w16 = (int64_t)rows * ((V + 1023) / 1024);
    c.steps = (int)std::min<int64_t>((w16 + kBusyWaves - 1) / kBusyWaves, kMaxSteps);
  }
  const int part = 64 * c.vals * c.steps;
  c.n_parts = (V + part - 1) / part;
  return c;
}

int check_select(int R, int K, int V, int n) {
  PDK_REQUIRE(R >= 1 && R <= 65535 / kMaxBeams, "R must be in [1, %d] (got %d)", 65535 / kMaxBeams, R);
  if (K < 1 || K > kMaxBeams || n < 1 || n > kMaxOut) {
    pdk::set_error("beam search takes 1 to %d beams and 1 to %d results (got %d, %d)", kMaxBeams,
                   kMaxOut, K, n);
    return PDK_ENOTSUP;
  }
  PDK_REQUIRE(V >= 1, "V must be >= 1 (got %d)", V);
  if (V > kMaxVocab) {
    pdk::set_error("a vocabulary of %d is above the supported %d", V, kMaxVocab);
    return PDK_ENOTSUP;
  }
  return PDK_OK;
}

}  // namespace

extern "C" int64_t pdk_beam_select_workspace_bytes(int R, int K, int V, int n) {
  pdk::clear_error();
  if (check_select(R, K, V, n)) return 0;
  return (int64_t)R * K * cut_of(R * K, V).n_parts * (sizeof(Part) + n * sizeof(Key));
}

extern "C" int pdk_beam_select(const void* logits, int elem_bytes, int64_t ld, int R, int K, int V,
                               const float* scores, const int32_t* last_tokens, int eos, int n,
                               void* workspace, int64_t workspace_bytes, int32_t* tokens,
                               int32_t* parents, float* out_scores, uintptr_t stream) {
  pdk::clear_error();
  if (int rc = check_select(R, K, V, n)) return rc;
  PDK_REQUIRE(logits && scores && tokens && parents && out_scores, "null pointer argument");
  PDK_REQUIRE(elem_bytes == 2 || elem_bytes == 4, "logits are bf16 (2) or fp32 (4), got %d",
              elem_bytes);
  PDK_REQUIRE(reinterpret_cast<uintptr_t>(logits) % elem_bytes == 0, "logits are not aligned");
  PDK_REQUIRE(ld >= V, "rows of %d logits do not fit a stride of %lld", V, (long long)ld);
  const int64_t need = pdk_beam_select_workspace_bytes(R, K, V, n);
  PDK_REQUIRE(workspace && workspace_bytes >= need && pdk::aligned16(workspace),
              "workspace of %lld bytes needed (got %lld)", (long long)need,
              (long long)workspace_bytes);
  const int rows = R * K;
  // A request's workgroup reads its beams' scores and last tokens before it writes, and
  // others' not at all: an output may lie place for place where they do.
  using pdk::Range;
  using pdk::overlap;
  const int64_t outs = (int64_t)R * n * 4;
  const Range in[2] = {{scores, (int64_t)rows * 4}, {last_tokens, (int64_t)rows * 4}};
  const Range out[3] = {{tokens, outs}, {parents, outs}, {out_scores, outs}};
  const Range ws{workspace, need};
  PDK_REQUIRE(!overlap(ws, Range{logits, ((int64_t)(rows - 1) * ld + V) * elem_bytes}),
              "the workspace must not overlap the logits");
  for (const Range& i : in) PDK_REQUIRE(!overlap(ws, i), "the workspace must not overlap an input");
  for (int o = 0; o < 3; ++o) {
    PDK_REQUIRE(!overlap(ws, out[o]), "the workspace must not overlap an output");
    for (int p = 0; p < o; ++p) PDK_REQUIRE(!overlap(out[o], out[p]), "outputs must not overlap");
    for (const Range& i : in)
      PDK_REQUIRE(!overlap(out[o], i) || (n == K && out[o].p == i.p),
                  "an output may overlap scores or last_tokens only in their places, with n = K");
  }
  const Cut cut = cut_of(rows, V);
  const int n_parts = cut.n_parts;
  Part* parts = static_cast<Part*>(workspace);
  Key* keys = reinterpret_cast<Key*>(parts + (int64_t)rows * n_parts);
  const dim3 grid((n_parts + kWaves - 1) / kWaves, rows), block(64 * kWaves);
  hipStream_t st = pdk::as_stream(stream);
  auto launch = [&](auto kern, auto x) {
    hipLaunchKernelGGL(kern, grid, block, 0, st, x, ld, V, n, n_parts, cut.steps, last_tokens,
                       eos, parts, keys);
  };
  const uint16_t* x16 = static_cast<const uint16_t*>(logits);
  const float* x32 = static_cast<const float*>(logits);
  if (elem_bytes == 2) {
    if (V < 8) launch(beam_part_kernel<uint16_t, 16, false, true>, x16);
    else if (cut.steps > 1) launch(beam_part_kernel<uint16_t, 16, true>, x16);
    else if (cut.vals == 32) launch(beam_part_kernel<uint16_t, 32, false>, x16);
    else launch(beam_part_kernel<uint16_t, 16, false>, x16);
  } else {
    if (V < 4) launch(beam_part_kernel<float, 16, false, true>, x32);
    else if (cut.steps > 1) launch(beam_part_kernel<float, 16, true>, x32);
    else if (cut.vals == 32) launch(beam_part_kernel<float, 32, false>, x32);
    else launch(beam_part_kernel<float, 16, false>, x32);
  }
  if (int rc = pdk::check_launch("beam_part_kernel")) return rc;
  hipLaunchKernelGGL(beam_join_kernel, dim3(R), dim3(64 * K), 0, st, parts, keys, n_parts, n,
                     scores, K, last_tokens, eos, tokens, parents, out_scores);
  return pdk::check_launch("beam_join_kernel");
}

extern "C" int pdk_beam_reorder(const int32_t* parents, const int32_t* ctx_lens, int R, int K,
                                int32_t* tables, int max_blocks, uint16_t* cache_k,
                                uint16_t* cache_v, int64_t cache_layer_stride, int n_layers,
                                int num_blocks, int n_kv_heads, int head_dim, uintptr_t stream) {
  pdk::clear_error();
  if (K < 1 || K > kMaxBeams) {
    pdk::set_error("beam search takes 1 to %d beams (got %d)", kMaxBeams, K);
    return PDK_ENOTSUP;
  }
  PDK_REQUIRE(R >= 1 && R <= 65535, "R must be in [1, 65535] (got %d)", R);
  PDK_REQUIRE(parents && ctx_lens && tables && cache_k && cache_v, "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(cache_k) && pdk::aligned16(cache_v), "caches must be 16-byte aligned");
  PDK_REQUIRE(n_layers >= 1 && n_layers <= 32767 && num_blocks >= 1 && max_blocks >= 1,
              "n_layers, num_blocks or max_blocks out of range");
  PDK_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 65535 && head_dim >= 1 && head_dim <= 4096,
              "n_kv_heads or head_dim out of range");
  const int64_t block = (int64_t)n_kv_heads * PDK_BLOCK_SIZE * head_dim;
  PDK_REQUIRE(cache_layer_stride % 8 == 0 &&
                  (n_layers == 1 || cache_layer_stride >= (int64_t)num_blocks * block),
              "the layer stride must be a multiple of 8 and hold num_blocks blocks");
  const int units = (int)(block / 8);
  const auto kern = K <= 4 ? beam_reorder_kernel<4> : K <= 8 ? beam_reorder_kernel<8>
                                                             : beam_reorder_kernel<16>;
  hipLaunchKernelGGL(kern, dim3((units + 255) / 256, R, 2 * n_layers + 1), dim3(256),
                     0, pdk::as_stream(stream), parents, ctx_lens, K, tables, max_blocks, cache_k,
                     cache_v, cache_layer_stride, num_blocks, units);
  return pdk::check_launch("beam_reorder_kernel");
}
