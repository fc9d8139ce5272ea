// Beam search on the paged cache, gfx950: the n best continuations of a
// request's beams (beam_part_kernel, beam_join_kernel) and the cache following
// them (beam_reorder_kernel).
//
// Selection. total(k, v) = score_k + logit_kv - log sum_v exp(logit_kv) over the
// K beams of a request and the vocabulary; the n largest, the lower beam and then
// the lower token first among equals. Inside a beam the order of the totals is
// that of the logits, so the vocabulary is read once: a wavefront takes a part of
// a row into registers and leaves its maximum, its sum of exponentials and its n
// best tokens; one workgroup per request joins the parts.
//
// The sums and totals are 64-bit: which of two beams' tokens comes first hangs on
// their difference, and 32 bits of a sum over a vocabulary of 1e5 leave 1e-6 of a
// total undecided, which a search over a thousand candidates a step does meet.
//
// n best of a wavefront's values: the n-th largest of the 64 lanes' own maxima
// bounds the n-th largest value from below, bit by bit with one ballot each until
// exactly n lanes reach it (some 10 to 15 bits). Mostly a few more than n values
// then reach the bound; they are compacted into LDS and ranked by counting. Where
// equal values let more than 64 reach it, the bound is taken again over unique
// 64-bit keys (the value in an order-preserving code above the complement of the
// token): only n lanes reach that one, so at most n times a lane's values do,
// whatever the logits are.
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

// 2^y for y <= 0: 2^k p(f), y = k + f, |f| <= 1/2, p the polynomial of degree 7
// that meets 2^f at the 8 Chebyshev nodes (off by less than 6e-11 of it). Down to
// y = -1000; the callers clamp.
__device__ __forceinline__ double exp2_neg(double y) {
  const double k = rint(y), f = y - k;
  double p = 1.5303701161442145e-05;
  p = fma(p, f, 0.00015469729221575116);
  p = fma(p, f, 0.0013333478471058548);
  p = fma(p, f, 0.009618025613268967);
  p = fma(p, f, 0.055504109063307244);
  p = fma(p, f, 0.24022651213498578);
  p = fma(p, f, 0.6931471805568296);
  p = fma(p, f, 0.9999999999595621);
  return __builtin_amdgcn_ldexp(p, (int)k);
}

// ln x for x >= 1/2: a 32-bit logarithm and one Newton step in 64 bits, which
// leaves the square of its error and exp2_neg's.
__device__ __forceinline__ double log_of(double x) {
  const double y = (double)__logf((float)x);
  const double e = x * exp2_neg(-y * 1.4426950408889634074) - 1.0;
  return y + (e - 0.5 * e * e);
}

constexpr double kLog2e = 1.4426950408889634074;

__device__ __forceinline__ double exp_neg(double x) { return exp2_neg(fmax(x, -690.0) * kLog2e); }

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

// x[i], i a lane's own: halved bit by bit with masks (a choice between registers
// would be made through memory).
template <int kN>
__device__ __forceinline__ float pick(const float (&x)[kN], int i) {
  uint32_t y[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j) y[j] = __float_as_uint(x[j]);
#pragma unroll
  for (int w = kN / 2, bit = 0; w; w >>= 1, ++bit) {
    const uint32_t odd = 0u - ((i >> bit) & 1u);
#pragma unroll
    for (int j = 0; j < w; ++j) y[j] = (y[2 * j + 1] & odd) | (y[2 * j] & ~odd);
  }
  return __uint_as_float(y[0]);
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

// Values e .. e + kEl - 1 of the row, those from V on as -inf. Rows of odd lengths
// start anywhere: the 16-byte loads take any address, and a row's parts and sums
// do not depend on where it lies (equal rows have equal totals).
template <typename T>
__device__ __forceinline__ void load_vals(const T* row, int e, int V, float* x) {
  constexpr int kEl = 16 / sizeof(T);
  if (e + kEl <= V) {
    uint32_t w[4];
    __builtin_memcpy(w, row + e, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        x[2 * i] = pdk::bf16_to_f32(w[i] & 0xffffu);
        x[2 * i + 1] = pdk::bf16_to_f32(w[i] >> 16);
      } else {
        x[i] = __uint_as_float(w[i]);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kEl; ++i) {
    x[i] = -INFINITY;
    if (e + i < V) {
      if constexpr (sizeof(T) == 2) x[i] = pdk::bf16_to_f32(row[e + i]);
      else x[i] = row[e + i];
    }
  }
}

// grid: x = kWaves parts, y = row. T is uint16_t (bf16) or float; a lane holds
// kVals values.
template <typename T, int kVals>
__global__ __launch_bounds__(64 * kWaves) void beam_part_kernel(const T* logits, int64_t ld, int V,
                                                                int n, int n_parts,
                                                                const int32_t* last_tokens,
                                                                int eos, Part* parts, Key* keys) {
  constexpr int kEl = 16 / sizeof(T), kGroups = kVals / kEl;
  __shared__ Key lists[kWaves][kMaxOut * kVals];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = blockIdx.y, part = blockIdx.x * kWaves + wave;
  if (part >= n_parts) return;
  if (last_tokens && last_tokens[row] == eos) return;   // an ended beam's logits count for nothing
  const T* p = logits + (int64_t)row * ld;
  float x[kVals];
  const int e0 = part * (64 * kVals) + lane * kEl;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) load_vals(p, e0 + i * 64 * kEl, V, x + i * kEl);
  float mine = x[0];
#pragma unroll
  for (int i = 1; i < kVals; ++i) mine = __builtin_elementwise_maximum(mine, x[i]);
  const float top = wave_all(mine, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
  double sum = 0.0;
  if (top < INFINITY && top > -INFINITY) {
#pragma unroll
    for (int i = 0; i < kVals; ++i) sum += exp_neg((double)x[i] - (double)top);
    sum = wave_sum(sum);
  } else if (!(top == -INFINITY)) {
    sum = NAN;
  }
  const int64_t at = (int64_t)row * n_parts + part;
  if (lane == 0) parts[at] = Part{(double)top, sum};

  // The values that reach the bound; all but -inf where there are few enough.
  Key* list = lists[wave];
  const uint32_t bound = nth_largest(code_of(mine), n);
  const float least = bound ? value_of(bound) : -3.402823466e38f;
  auto token = [&](int i) { return (uint32_t)(e0 + i / kEl * (64 * kEl) + i % kEl); };
  uint32_t mask = 0;                                     // bit i: value i reaches the bound
#pragma unroll
  for (int i = 0; i < kVals; ++i) mask |= x[i] >= least ? 1u << i : 0u;
  int c = 0;
  for (uint64_t who; (who = __ballot(mask != 0)) && c <= 64;) {   // a value of every such lane
    const int i = __builtin_ctz(mask | 0x80000000u);
    const float v = pick(x, i);
    const int to = c + __popcll(who & ((1ull << lane) - 1));
    if (mask && to < 64) list[to] = key_of(v, token(i));
    mask &= mask - 1;
    c += __popcll(who);
  }
  if (c > 64) {                                          // equal values
    Key best = 0;
#pragma unroll 1
    for (int i = 0; i < kVals; ++i) {
      Key k = 0;
#pragma unroll
      for (int j = 0; j < kVals; ++j)
        if (j == i) k = key_of(x[j], token(j));
      best = k > best ? k : best;
    }
    const Key b = nth_largest(best, n);
    c = 0;
#pragma unroll
    for (int i = 0; i < kVals; ++i) {
      const Key k = key_of(x[i], token(i));
      const bool in = k >= (b ? b : 1);
      const uint64_t who = __ballot(in);
      if (in) list[c + __popcll(who & ((1ull << lane) - 1))] = k;
      c += __popcll(who);
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
  const bool ended = last_tokens && last_tokens[row] == eos;
  const float score = scores[row];
  const bool alive = score > -INFINITY && score < INFINITY;
  double total = lane == 0 && alive ? (double)score : -INFINITY;   // of an ended beam
  int32_t token = eos;
  if (!ended) {
    // Heads of the parts' lists; only lists whose head reaches the n-th largest of
    // the lanes' own best heads hold any of the n best: those of at most n lanes.
    const Key* kp = keys + (int64_t)row * n_parts * n;
    const Part* pp = parts + (int64_t)row * n_parts;
    Key mine = 0;
    double top = -INFINITY, sum = 0.0;
#pragma unroll 1
    for (int s = lane; s < n_parts; s += 64) {
      const Key head = kp[s * n];
      mine = head > mine ? head : mine;
      top = fmax(top, pp[s].top);
    }
    top = wave_all(top, [](double a, double b) { return fmax(a, b); });
#pragma unroll 1
    for (int s = lane; s < n_parts; s += 64) {
      const Part q = pp[s];
      // NaN in q.sum stays; a part without a finite value adds nothing.
      sum += q.sum != 0.0 ? q.sum * exp_neg(q.top - top) : 0.0;
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
    for (int s = lane; s - lane < n_parts; s += 64) {
      const bool in = s < n_parts && kp[s * n] >= least;
      const uint64_t who = __ballot(in);
      if (in) lists[k][m + __popcll(who & ((1ull << lane) - 1))] = (uint16_t)s;
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
        if (in) list[k][c + __popcll(who & ((1ull << lane) - 1))] = q[x];
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

// Values of a lane: 32, or 16 where rows are too few for 32 to give every SIMD two
// wavefronts (128256 bf16 or fp32 values a row, in us with 16 and with 32: 4 rows
// 13.5 and 14.9, 64 rows 16.8 and 15.8, 256 fp32 rows 49.6 and 44.6).
int lane_vals(int rows, int V) {
  const bool many = (int64_t)rows * ((V + 2047) / 2048) >= 2048;
  return many || V > kMaxVocab / 2 ? 32 : 16;
}

int parts_of(int rows, int V) {
  const int part = 64 * lane_vals(rows, V);
  return (V + part - 1) / part;
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
  return (int64_t)R * K * parts_of(R * K, V) * (sizeof(Part) + n * sizeof(Key));
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
  const int rows = R * K, n_parts = parts_of(rows, V), vals = lane_vals(rows, V);
  Part* parts = static_cast<Part*>(workspace);
  Key* keys = reinterpret_cast<Key*>(parts + (int64_t)rows * n_parts);
  const dim3 grid((n_parts + kWaves - 1) / kWaves, rows), block(64 * kWaves);
  hipStream_t st = pdk::as_stream(stream);
  auto launch = [&](auto kern, auto x) {
    hipLaunchKernelGGL(kern, grid, block, 0, st, x, ld, V, n, n_parts, last_tokens, eos, parts, keys);
  };
  const uint16_t* x16 = static_cast<const uint16_t*>(logits);
  const float* x32 = static_cast<const float*>(logits);
  if (elem_bytes == 2) {
    if (vals == 32) launch(beam_part_kernel<uint16_t, 32>, x16);
    else launch(beam_part_kernel<uint16_t, 16>, x16);
  } else {
    if (vals == 32) launch(beam_part_kernel<float, 32>, x32);
    else launch(beam_part_kernel<float, 16>, x32);
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
