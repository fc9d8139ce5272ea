// Beam search on the paged cache, gfx950: the n best continuations of a
// request's beams (beam_part_kernel, beam_join_kernel) and the cache following
// them (beam_reorder_kernel).
//
// Selection. total(k, v) = score_k + logit_kv - log sum_v exp(logit_kv) over the
// K beams of a request and the vocabulary; the n largest, the lower beam and then
// the lower token first among equals. Inside a beam the order of the totals is
// that of the logits, so the vocabulary is read once: a workgroup takes a part of
// a row, and leaves its maximum, its sum of exponentials and its n best tokens;
// one workgroup per request joins the parts.
//
// The sums and totals are 64-bit: which of two beams' tokens comes first hangs on
// their difference, and 32 bits of a sum over a vocabulary of 1e5 leave 1e-6 of a
// total undecided, which a search over a thousand candidates a step does meet.
// exp is a degree-9 polynomial (below 1e-11), a dozen full-rate operations.
//
// n best of 64 lanes' values: values are made unique integer keys (the value in
// an order-preserving code above the complement of the token). The n-th largest
// of the lanes' own maxima bounds the n-th largest key from below, and only n
// lanes hold keys above that bound, so at most n times a lane's values are
// compacted into LDS and ranked there by counting, whatever the logits are.
#include <math.h>

#include <algorithm>

#include "pdk_common.h"

namespace {

using pdk::v8;

constexpr int kMaxBeams = 16;
constexpr int kMaxOut = 32;
constexpr int kWaves = 4;                 // of a part's workgroup
constexpr int kLaneVals = 16;             // values a lane holds
constexpr int kPartVals = 64 * kWaves * kLaneVals;   // 4096 values of a row per workgroup
constexpr int kMaxLists = 4;              // parts' lists a lane of the join looks at
constexpr int kMaxParts = 64 * kMaxLists;

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

// e^x for x <= 0 (0 below -700): 2^k p(f), x = (k + f) ln 2, |f| <= 1/2, p the
// Taylor polynomial of 2^f to degree 9, off by (ln 2 / 2)^10 / 10! = 7e-12.
__device__ __forceinline__ double exp_neg(double x) {
  const double y = fmax(x, -700.0) * 1.4426950408889634074;
  const double k = rint(y);
  const double f = (y - k) * 0.69314718055994530942;
  double p = 1.0 / 362880.0;
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return x < -700.0 ? 0.0 : ldexp(p, (int)k);
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// The n-th largest of the wavefront's 64 keys (0 if fewer than n are not 0):
// bit by bit from the top, the largest bound that n lanes reach.
__device__ __forceinline__ Key nth_largest(Key mine, int n) {
  Key bound = 0;
#pragma unroll 1
  for (int bit = 63; bit >= 0; --bit) {
    const Key t = bound | (1ull << bit);
    const int c = __popcll(__ballot(mine >= t));
    if (c >= n) bound = t;
    if (c == n) break;
  }
  return bound;
}

// The keys >= bound of the wavefront's lanes, compacted into list; how many.
template <int kN>
__device__ __forceinline__ int compact(const Key (&keys)[kN], Key bound, Key* list) {
  int at = 0;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const bool in = keys[i] >= bound;
    const uint64_t who = __ballot(in);
    if (in) list[at + __popcll(who & ((1ull << (threadIdx.x & 63)) - 1))] = keys[i];
    at += __popcll(who);
  }
  return at;
}

// What the wavefront's lanes wrote to LDS is there for all of them.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The largest n of list[0..c) in order to best[0..n), zeros behind them.
__device__ __forceinline__ void rank(const Key* list, int c, Key* best, int n) {
  const int lane = threadIdx.x & 63;
  if (lane < n) best[lane] = 0;
  wave_sync();
  for (int i = lane; i < c; i += 64) {
    const Key mine = list[i];
    int r = 0;
    for (int j = 0; j < c; ++j) r += list[j] > mine;
    if (r < n) best[r] = mine;
  }
  wave_sync();
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
__device__ __forceinline__ void load_vals(const T* row, int64_t e, int64_t V, float* x) {
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

// grid: x = part, y = row. T is uint16_t (bf16) or float.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void beam_part_kernel(const T* logits, int64_t ld, int V,
                                                                int n, const int32_t* last_tokens,
                                                                int eos, Part* parts, Key* keys) {
  constexpr int kEl = 16 / sizeof(T), kGroups = kLaneVals / kEl;
  __shared__ Key list[kWaves][64 * kLaneVals / 2];   // n * kLaneVals <= 512 per wavefront
  __shared__ Key best[kWaves][kMaxOut];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  const int row = blockIdx.y, part = blockIdx.x, n_parts = gridDim.x;
  if (last_tokens && last_tokens[row] == eos) return;   // an ended beam's logits count for nothing
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const T* p = logits + (int64_t)row * ld;
  float x[kLaneVals];
  int64_t e[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    e[i] = (int64_t)part * kPartVals + ((wave * kGroups + i) * 64 + lane) * kEl;
    load_vals(p, e[i], V, x + i * kEl);
  }
  float top = x[0];
#pragma unroll
  for (int i = 1; i < kLaneVals; ++i) top = __builtin_elementwise_maximum(top, x[i]);
#pragma unroll
  for (int o = 32; o; o >>= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, o));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = __builtin_elementwise_maximum(top, tops[w]);
  double sum = 0.0;
  if (top < INFINITY && top > -INFINITY) {
#pragma unroll
    for (int i = 0; i < kLaneVals; ++i) sum += exp_neg((double)x[i] - (double)top);
    sum = wave_sum(sum);
  } else if (!(top == -INFINITY)) {
    sum = NAN;
  }
  if (lane == 0) sums[wave] = sum;

  Key k[kLaneVals], mine = 0;
#pragma unroll
  for (int i = 0; i < kLaneVals; ++i) {
    k[i] = key_of(x[i], (uint32_t)(e[i / kEl] + i % kEl));
    mine = k[i] > mine ? k[i] : mine;
  }
  const Key bound = nth_largest(mine, n);
  const int c = compact(k, bound ? bound : 1, list[wave]);
  __syncthreads();
  rank(list[wave], c, best[wave], n);
  __syncthreads();
  // The wavefronts' ordered lists become one.
  const int64_t at = (int64_t)row * n_parts + part;
  if ((int)threadIdx.x < kWaves * n) {
    const int w = threadIdx.x / n, i = threadIdx.x - w * n;
    const Key m = best[w][i];
    int r = i;
    for (int o = 0; o < kWaves; ++o)
      if (o != w)
        for (int j = 0; j < n; ++j) r += best[o][j] > m || (m == 0 && best[o][j] == 0 && o < w);
    if (r < n) keys[at * n + r] = m;
  }
  if (threadIdx.x == 0) {
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += sums[w];
    parts[at] = Part{(double)top, s};
  }
}

// One workgroup per request, one wavefront per beam: the beam's log sum, its n
// best tokens of all parts and their totals; then every candidate counts those of
// the other beams that come before it.
__global__ __launch_bounds__(64 * kMaxBeams) void beam_join_kernel(
    const Part* parts, const Key* keys, int n_parts, int n, const float* scores, int K,
    const int32_t* last_tokens, int eos, int32_t* tokens, int32_t* parents, float* out_scores) {
  __shared__ Key list[kMaxBeams][kMaxOut * 8];
  __shared__ Key best[kMaxBeams][kMaxOut];
  __shared__ double totals[kMaxBeams][kMaxOut];
  __shared__ int32_t token[kMaxBeams][kMaxOut];
  __shared__ int found;
  const int r = blockIdx.x, k = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int row = r * K + k;
  const bool ended = last_tokens && last_tokens[row] == eos;
  const float score = scores[row];
  const bool alive = score > -INFINITY && score < INFINITY;
  if (threadIdx.x == 0) found = 0;
  if (!ended) {
    // Heads of the parts' lists; only lists whose head reaches the n-th largest
    // head hold any of the n best.
    Key head[kMaxLists], mine = 0;
    double top = -INFINITY, sum = 0.0;
#pragma unroll
    for (int i = 0; i < kMaxLists; ++i) {
      const int s = lane + 64 * i;
      head[i] = 0;
      if (s < n_parts) {
        head[i] = keys[((int64_t)row * n_parts + s) * n];
        const Part q = parts[(int64_t)row * n_parts + s];
        // NaN in q.sum stays; a part without a finite value adds nothing.
        if (q.sum != 0.0) {
          const double m = fmax(top, q.top);
          sum = sum * exp_neg(top - m) + q.sum * exp_neg(q.top - m);
          top = m;
        }
      }
      mine = head[i] > mine ? head[i] : mine;
    }
    double all = top;
#pragma unroll
    for (int o = 32; o; o >>= 1) all = fmax(all, __shfl_xor(all, o));
    sum = wave_sum(top > -INFINITY || sum != sum ? sum * exp_neg(top - all) : 0.0);
    const double lse = all + log(sum);
    const Key bound = nth_largest(mine, n);
    int c = 0;
#pragma unroll
    for (int i = 0; i < kMaxLists; ++i) {
      // Lists that reach the bound, one after the other: their keys from the bound on.
      const Key least = bound ? bound : 1;
      for (uint64_t who = __ballot(head[i] >= least); who; who &= who - 1) {
        const int s = __ffsll((long long)who) - 1 + 64 * i;
        const Key q = lane < n ? keys[((int64_t)row * n_parts + s) * n + lane] : 0;
        const uint64_t in = __ballot(q >= least);
        const int m = __popcll(in);
        if (c + m > kMaxOut * 8) {
          // More than the list holds: keep the n best so far.
          rank(list[k], c, best[k], n);
          if (lane < n) list[k][lane] = best[k][lane];
          wave_sync();
          c = min(c, n);
        }
        if (q >= least) list[k][c + lane] = q;          // the list is ordered: a prefix of lanes
        c += m;
      }
    }
    rank(list[k], c, best[k], n);
    if (lane < n) {
      const Key b = best[k][lane];
      const bool ok = b && alive && lse > -INFINITY && lse < INFINITY;
      token[k][lane] = (int32_t)(0xffffffffu - (uint32_t)b);
      totals[k][lane] = ok ? (double)score + ((double)value_of((uint32_t)(b >> 32)) - lse) : -INFINITY;
    }
  } else if (lane < n) {
    token[k][lane] = eos;
    totals[k][lane] = lane == 0 && alive ? (double)score : -INFINITY;
  }
  __syncthreads();
  if (lane < n) {
    const double t = totals[k][lane];
    if (t > -INFINITY) {
      int at = lane;
      for (int o = 0; o < K; ++o) {
        if (o == k) continue;
        int lo = 0, hi = n;                              // the first of beam o behind this one
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          const double u = totals[o][mid];
          if (u > t || (u == t && o < k)) lo = mid + 1;
          else hi = mid;
        }
        at += lo;
      }
      atomicAdd(&found, 1);
      if (at < n) {
        tokens[(int64_t)r * n + at] = token[k][lane];
        parents[(int64_t)r * n + at] = k;
        out_scores[(int64_t)r * n + at] = (float)t;
      }
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < n && (int)threadIdx.x >= found) {   // fewer candidates than asked for
    tokens[(int64_t)r * n + threadIdx.x] = -1;
    parents[(int64_t)r * n + threadIdx.x] = -1;
    out_scores[(int64_t)r * n + threadIdx.x] = -INFINITY;
  }
}

// Reordering. Beam k of request r goes on from beam p = parents[r][k]: its table
// takes p's entries of the filled blocks (shared from now on, never written
// again), and its own block at the partly filled place the contents of p's there.
// A lane carries one 16-byte place of that block for all beams of the request
// (or one table column): it has read every beam's before it writes any, so beams
// may swap, and no two lanes touch one address: no staging, no second launch.
// Bound by the bytes of the blocks that move.
// grid: x = chunk, y = 2 * layer + (0 for K, 1 for V) or, last, the tables, z = r.
__global__ __launch_bounds__(256) void beam_reorder_kernel(const int32_t* parents,
                                                           const int32_t* ctx_lens, int K,
                                                           int32_t* tables, int max_blocks,
                                                           uint16_t* ck, uint16_t* cv,
                                                           int64_t layer_stride, int num_blocks,
                                                           int block_units) {
  const int r = blockIdx.z;
  const int held = ctx_lens[r * K];                      // the same for a request's beams
  if (held <= 0) return;
  const int full = held / PDK_BLOCK_SIZE;
  int32_t* rows = tables + (int64_t)r * K * max_blocks;
  auto parent = [&](int k) {
    const int p = k < K ? parents[r * K + k] : -1;
    return p >= 0 && p < K ? p : k;                      // no parent: the beam stays itself
  };
  if (blockIdx.y == gridDim.y - 1) {
    const int cols = min(full, max_blocks);
    for (int j = blockIdx.x * 256 + threadIdx.x; j < cols; j += gridDim.x * 256) {
      int32_t id[kMaxBeams];
#pragma unroll
      for (int k = 0; k < kMaxBeams; ++k)
        if (k < K) id[k] = rows[(int64_t)parent(k) * max_blocks + j];
#pragma unroll
      for (int k = 0; k < kMaxBeams; ++k)
        if (k < K && parent(k) != k) rows[(int64_t)k * max_blocks + j] = id[k];
    }
    return;
  }
  const int u = blockIdx.x * 256 + threadIdx.x;
  if (held % PDK_BLOCK_SIZE == 0 || full >= max_blocks || u >= block_units) return;
  uint16_t* base = (blockIdx.y & 1 ? cv : ck) + (int64_t)(blockIdx.y >> 1) * layer_stride;
  const int64_t block = (int64_t)block_units * 8;
  auto place = [&](int k) {                              // beam k's partly filled block, or -1
    const int id = rows[(int64_t)k * max_blocks + full];
    return id >= 0 && id < num_blocks ? id : -1;
  };
  v8 x[kMaxBeams];
#pragma unroll
  for (int k = 0; k < kMaxBeams; ++k) {
    const int p = parent(k);
    if (k < K && p != k) {
      const int s = place(p);
      if (s >= 0) x[k] = pdk::ld16(base + s * block + (int64_t)u * 8);
    }
  }
#pragma unroll
  for (int k = 0; k < kMaxBeams; ++k) {
    const int p = parent(k);
    if (k < K && p != k) {
      const int s = place(p), d = place(k);
      if (s >= 0 && d >= 0) pdk::st16(base + d * block + (int64_t)u * 8, x[k]);
    }
  }
}

int parts_of(int V) { return (V + kPartVals - 1) / kPartVals; }

int check_select(int R, int K, int V, int n) {
  PDK_REQUIRE(R >= 1 && R <= 65535 / kMaxBeams, "R must be in [1, %d] (got %d)", 65535 / kMaxBeams, R);
  if (K < 1 || K > kMaxBeams || n < 1 || n > kMaxOut) {
    pdk::set_error("beam search takes 1 to %d beams and 1 to %d results (got %d, %d)", kMaxBeams,
                   kMaxOut, K, n);
    return PDK_ENOTSUP;
  }
  PDK_REQUIRE(V >= 1, "V must be >= 1 (got %d)", V);
  if (V > kMaxParts * kPartVals) {
    pdk::set_error("a vocabulary of %d is above the supported %d", V, kMaxParts * kPartVals);
    return PDK_ENOTSUP;
  }
  return PDK_OK;
}

}  // namespace

extern "C" int64_t pdk_beam_select_workspace_bytes(int R, int K, int V, int n) {
  pdk::clear_error();
  if (check_select(R, K, V, n)) return 0;
  return (int64_t)R * K * parts_of(V) * (sizeof(Part) + n * sizeof(Key));
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
  const int rows = R * K, n_parts = parts_of(V);
  Part* parts = static_cast<Part*>(workspace);
  Key* keys = reinterpret_cast<Key*>(parts + (int64_t)rows * n_parts);
  const dim3 grid(n_parts, rows), block(64 * kWaves);
  hipStream_t st = pdk::as_stream(stream);
  if (elem_bytes == 2)
    hipLaunchKernelGGL(beam_part_kernel<uint16_t>, grid, block, 0, st,
                       static_cast<const uint16_t*>(logits), ld, V, n, last_tokens, eos, parts, keys);
  else
    hipLaunchKernelGGL(beam_part_kernel<float>, grid, block, 0, st,
                       static_cast<const float*>(logits), ld, V, n, last_tokens, eos, parts, keys);
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
  hipLaunchKernelGGL(beam_reorder_kernel, dim3((units + 255) / 256, 2 * n_layers + 1, R), dim3(256),
                     0, pdk::as_stream(stream), parents, ctx_lens, K, tables, max_blocks, cache_k,
                     cache_v, cache_layer_stride, num_blocks, units);
  return pdk::check_launch("beam_reorder_kernel");
}
