// What a step over several requests' next tokens (pieces of prompts, a draft's
// tokens, single ones) does to the paged cache, gfx950: the map of the tokens
// (chunk_map_kernel) and their keys and values (rope_write_kernel).
//
// Map. Request r holds past_r tokens and gets new_r: with held = ceil(past / 16)
// blocks, need = ceil((past + new) / 16) - held and first_r = the sum of need over
// the requests before it, entry held + i of its table becomes free[first_r + i].
// Every workgroup adds up all requests' lengths itself (a few loads a thread), so
// one launch does it all; a token finds its request by bisection in LDS and reads
// its block from the free list where its entry is new, so no workgroup waits for
// another's entries. Bound by one launch and a chain of two loads: 3.5 us for 64 requests'
// single tokens and for 48 pieces of prompts in a launch of 16384.
//
// Write. Token i's q and k heads turn by the angle positions[i] * inv_freq: the
// product in 64 bits, in turns, so that far positions keep their angle (in 32 bits
// position 10^6 is off by up to 0.03). A workgroup computes the 64 angles of 16 tokens
// once and takes some of the heads: a lane turns the dims d .. d + 7 and d + 64 .. d + 71 of
// a head (two 16-byte loads and stores); lanes go through q in whole rows, through k so that
// 16 tokens' places in a block are stored together. V lies dim by dim in the cache: where
// eight tokens fill one half of a block, a lane transposes their 8 dims and stores 16
// bytes for each; any other token is stored value by value. Bound by memory where there
// are many tokens (8192 with 32 + 16 heads, eager over several sets of tensors: 41.8 us, 4.8 TB/s
// of the bytes that must move; HBM sees 2 % more), by one launch and a chain of three loads
// where there are few (16: 3.5 us).
#include <math.h>

#include <algorithm>

#include "pdk_common.h"

namespace {

using pdk::v8;

constexpr int kMaxRequests = 4096;
constexpr int kThreads = 256;
constexpr int kD = 128;
constexpr int kTok = 16;                  // tokens of a write workgroup

__device__ __forceinline__ int clamp_to(int x, int lo, int hi) { return min(max(x, lo), hi); }

__global__ __launch_bounds__(kThreads) void chunk_map_kernel(
    const int32_t* past, const int32_t* added, int R, int32_t* tables, int W, const int32_t* free_ids,
    int n_free, int N, int32_t* starts, int32_t* ctx, int32_t* positions, int32_t* slots,
    int32_t* taken) {
  // Per request the sums before it: tokens in the launch, blocks taken.
  __shared__ int32_t s_tok[kMaxRequests + 1], s_blk[kMaxRequests + 1];
  __shared__ int32_t w_tok[kThreads / 64], w_blk[kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, cap = W * 16;
  const int per = (R + kThreads - 1) / kThreads, r0 = min(tid * per, R), r1 = min(r0 + per, R);
  auto length = [&](int r, int& p, int& n) {
    p = clamp_to(past[r], 0, cap);
    n = clamp_to(added[r], 0, cap - p);
  };
  auto blocks = [](int t) { return (t + 15) >> 4; };
  int tok = 0, blk = 0;
  for (int r = r0; r < r1; ++r) {
    int p, n;
    length(r, p, n);
    tok += n;
    blk += blocks(p + n) - blocks(p);
  }
  int tok_to = tok, blk_to = blk;         // inclusive sums over the wavefront
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(tok_to, o), b = __shfl_up(blk_to, o);
    if (lane >= o) {
      tok_to += a;
      blk_to += b;
    }
  }
  if (lane == 63) {
    w_tok[wave] = tok_to;
    w_blk[wave] = blk_to;
  }
  __syncthreads();
  tok = tok_to - tok;
  blk = blk_to - blk;
  for (int w = 0; w < wave; ++w) {
    tok += w_tok[w];
    blk += w_blk[w];
  }
  for (int r = r0; r < r1; ++r) {
    int p, n;
    length(r, p, n);
    s_tok[r] = tok;
    s_blk[r] = blk;
    tok += n;
    blk += blocks(p + n) - blocks(p);
    if (r == R - 1) {
      s_tok[R] = tok;
      s_blk[R] = blk;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int r = tid; r <= R; r += kThreads) {
      starts[r] = s_tok[r];
      if (r < R) ctx[r] = clamp_to(past[r], 0, cap) + s_tok[r + 1] - s_tok[r];
    }
    if (tid == 0) *taken = s_blk[R];
  }
  auto fresh = [&](int at) { return at < n_free ? free_ids[at] : -1; };
  // The request of item j of those that sums [R + 1] counts.
  auto request_of = [&](const int32_t* sums, int j) {
    int lo = 0, hi = R;                   // sums[lo] <= j < sums[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid] <= j) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  for (int k = blockIdx.x * kThreads + tid; k < s_blk[R]; k += gridDim.x * kThreads) {
    const int r = request_of(s_blk, k), held = blocks(clamp_to(past[r], 0, cap));
    tables[(int64_t)r * W + held + k - s_blk[r]] = fresh(k);
  }
  const int j = blockIdx.x * kThreads + tid;
  if (j >= N) return;
  int pos = -1, slot = -1;
  if (j < s_tok[R]) {
    const int lo = request_of(s_tok, j);
    const int p = clamp_to(past[lo], 0, cap), held = blocks(p);
    pos = p + j - s_tok[lo];
    const int e = pos >> 4;
    const int id = e < held ? tables[(int64_t)lo * W + e] : fresh(s_blk[lo] + e - held);
    if (id >= 0 && id < (1 << 27)) slot = id * 16 + (pos & 15);
  }
  positions[j] = pos;
  slots[j] = slot;
}

struct Turn {
  float c, s;
};

// A head's dims d .. d + 7 and d + 64 .. d + 71 turned by the angles z[d ..].
__device__ __forceinline__ void turn_head(const Turn* z, const v8& a, const v8& b, v8& x, v8& y) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float r[2][2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      pdk::rope_pair(pdk::bf16_to_f32(e ? a.w[w] >> 16 : a.w[w] & 0xffffu),
                     pdk::bf16_to_f32(e ? b.w[w] >> 16 : b.w[w] & 0xffffu), z[2 * w + e].c,
                     z[2 * w + e].s, r[0][e], r[1][e]);
    x.w[w] = pdk::pack_bf16x2_rne(r[0][0], r[0][1]);
    y.w[w] = pdk::pack_bf16x2_rne(r[1][0], r[1][1]);
  }
}

// grid: x = 16 tokens, y = a share of their units. First the units of q: 256 of the tokens'
// (token, head, 8 dims) in order, so that a unit reads and writes whole rows; then those
// of k: two heads of the 16 tokens, whose 16 bytes at a dim lie together in the cache; then
// those of v: 16 / kLanes heads, kLanes lanes for 8 dims of one.
template <int kLanes, bool kStream>
__global__ __launch_bounds__(kThreads) void rope_write_kernel(
    const uint16_t* qkv, int64_t ld, const float* inv_freq, const int32_t* positions,
    const int32_t* slots, int N, int NH, int NKV, uint16_t* q_out, uint16_t* cache_k,
    uint16_t* cache_v, int64_t n_slots) {
  __shared__ Turn turn[kTok][kD / 2 + 1];
  __shared__ int32_t slot_of[kTok + 14];  // of tokens j0 - 7 .. j0 + kTok + 6
  const int tid = threadIdx.x, j0 = blockIdx.x * kTok;
  if (tid < kTok + 14) {
    const int j = j0 - 7 + tid;
    const int s = j >= 0 && j < N ? slots[j] : -1;
    slot_of[tid] = s < n_slots ? s : -1;
  }
  const int units_q = (kTok * NH * 8 + kThreads - 1) / kThreads, units_k = (NKV + 1) / 2;
  const int units = units_q + units_k + (NKV * kLanes + 15) / 16, u0 = blockIdx.y;
  const int d = (tid & 7) * 8;            // q and k: the lane's dims
  struct Place {
    int t, head;                          // token of the 16, head of qkv's
    bool real;
  };
  auto place = [&](int u) {
    if (u < units_q) {
      const int i = u * (kThreads / 8) + (tid >> 3), t = i / NH;
      return Place{min(t, kTok - 1), i - t * NH, t < kTok && j0 + t < N};
    }
    const int t = (tid >> 3) & 15, h = 2 * (u - units_q) + (tid >> 7);
    return Place{t, NH + min(h, NKV - 1), h < NKV && j0 + t < N};
  };
  v8 a, b;
  auto load = [&](int u) __attribute__((always_inline)) {
    const Place p = place(u);
    const uint16_t* from = qkv + (int64_t)min(j0 + p.t, N - 1) * ld + (int64_t)p.head * kD + d;
    a = pdk::ld16_as<kStream>(from);
    b = pdk::ld16_as<kStream>(from + 64);
  };
  // The first unit's values are under way while the angles are computed: those of its own
  // tokens where the workgroup has one unit, else of all.
  if (u0 < units_q + units_k) {
    load(u0);
    const bool one = u0 + (int)gridDim.y >= units_q + units_k && u0 < units_q;
    const int t_lo = one ? u0 * (kThreads / 8) / NH : 0;
    const int t_hi = one ? min((u0 * (kThreads / 8) + kThreads / 8 - 1) / NH, kTok - 1) : kTok - 1;
    for (int t = t_lo + (tid >> 6); t <= t_hi; t += kThreads / 64) {
      const int i = tid & 63, pos = max(positions[min(j0 + t, N - 1)], 0);
      const double turns = (double)pos * ((double)inv_freq[i] * 0.15915494309189535);
      float s, c;
      sincosf((float)((turns - rint(turns)) * 6.283185307179586), &s, &c);
      turn[t][i] = Turn{c, s};
    }
  }
  __syncthreads();
  int u = u0;
  for (; u < units_q + units_k; u += gridDim.y) {
    const Place p = place(u);
    v8 x, y;
    turn_head(&turn[p.t][d], a, b, x, y);
    if (u + (int)gridDim.y < units_q + units_k) load(u + gridDim.y);
    if (!p.real) continue;
    if (u < units_q) {
      uint16_t* to = q_out + ((int64_t)(j0 + p.t) * NH + p.head) * kD + d;
      pdk::st16_as<kStream>(to, x);
      pdk::st16_as<kStream>(to + 64, y);
    } else {
      const int s = slot_of[p.t + 7];
      if (s < 0) continue;
      uint16_t* to = cache_k + ((int64_t)(s >> 4) * NKV + p.head - NH) * (16 * kD);
      pdk::st16(to + pdk::k_unit(s & 15, d, kD) * 8, x);
      pdk::st16(to + pdk::k_unit(s & 15, d + 64, kD) * 8, y);
    }
  }
  if (u >= units) return;
  // V: which of the 16 tokens lead eight that fill a half of a block (at most two), and
  // which are in no such eight; the others' lead does them, here or in the tile before.
  uint64_t leads, lone;
  {
    const int t = tid & 15, s = slot_of[t + 7], lead = t + 7 - (s & 7);
    bool whole = s >= 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) whole &= slot_of[lead + i] == (s & ~7) + i;
    const bool mine = (tid & 63) < kTok;
    leads = __ballot(mine && whole && (s & 7) == 0);
    lone = __ballot(mine && s >= 0 && !whole);
  }
  const int n_leads = __popcll(leads);
  const int lead_at[2] = {__builtin_ctzll(leads | 1ull << kTok), 63 - __builtin_clzll(leads | 1)};
  for (; u < units; u += gridDim.y) {
    const int sub = tid % kLanes, dv = (tid / kLanes % 16) * 8;
    const int h = (u - units_q - units_k) * (16 / kLanes) + tid / (16 * kLanes);
    if (h >= NKV) continue;
    const uint16_t* const column = qkv + (int64_t)j0 * ld + (int64_t)(NH + NKV + h) * kD + dv;
    auto target = [&](int s) { return cache_v + (((int64_t)(s >> 4) * NKV + h) * kD + dv) * 16 + (s & 15); };
    if (sub < n_leads) {
      const int t = sub ? lead_at[1] : lead_at[0];
      v8 in[8], out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) in[i] = pdk::ld16(column + (t + i) * ld);
      pdk::transpose8x8(in, out);
      uint16_t* to = target(slot_of[t + 7]);
#pragma unroll
      for (int i = 0; i < 8; ++i) pdk::st16(to + 16 * i, out[i]);
    }
    // The lone tokens, every kLanes-th by each of the lanes of 8 dims: all loads first.
    if (lone) {
      v8 x[kTok / kLanes];
      int at[kTok / kLanes];
      uint64_t left = lone;
#pragma unroll
      for (int i = 0; i < kTok / kLanes; ++i) {
        at[i] = -1;
#pragma unroll
        for (int e = 0; e < kLanes; ++e) {
          const int t = left ? __builtin_ctzll(left) : -1;
          left &= left - 1;
          at[i] = sub == e ? t : at[i];
        }
        x[i] = pdk::ld16(column + max(at[i], 0) * ld);
      }
#pragma unroll
      for (int i = 0; i < kTok / kLanes; ++i) {
        if (at[i] < 0) break;
        uint16_t* to = target(slot_of[at[i] + 7]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          to[32 * w] = (uint16_t)x[i].w[w];
          to[32 * w + 16] = (uint16_t)(x[i].w[w] >> 16);
        }
      }
    }
  }
}

}  // namespace

extern "C" int pdk_chunk_map(const int32_t* past, const int32_t* added, int R, int32_t* tables,
                             int max_blocks, const int32_t* free_ids, int n_free, int max_tokens,
                             int32_t* starts, int32_t* ctx_lens, int32_t* positions, int32_t* slots,
                             int32_t* taken, uintptr_t stream) {
  pdk::clear_error();
  PDK_REQUIRE(R >= 1 && R <= kMaxRequests, "R must be in [1, %d] (got %d)", kMaxRequests, R);
  PDK_REQUIRE(max_blocks >= 1 && (int64_t)R * max_blocks < (1ll << 27),
              "tables of %d x %d blocks hold none or 2^31 tokens or more", R, max_blocks);
  PDK_REQUIRE(n_free >= 0 && max_tokens >= 0 && max_tokens < (1 << 30),
              "n_free or max_tokens out of range");
  PDK_REQUIRE(past && added && tables && starts && ctx_lens && taken && (n_free == 0 || free_ids) &&
                  (max_tokens == 0 || (positions && slots)),
              "null pointer argument");
  const int64_t tokens = max_tokens * 4ll;
  const pdk::Range out[6] = {{tables, (int64_t)R * max_blocks * 4}, {starts, (R + 1) * 4ll},
                             {ctx_lens, R * 4ll}, {positions, tokens}, {slots, tokens}, {taken, 4}};
  const pdk::Range in[3] = {{past, R * 4ll}, {added, R * 4ll}, {free_ids, n_free * 4ll}};
  for (int o = 0; o < 6; ++o) {
    for (int p = 0; p < o; ++p)
      PDK_REQUIRE(!pdk::overlap(out[o], out[p]), "the tables and the outputs must not overlap");
    for (const pdk::Range& i : in)
      PDK_REQUIRE(!pdk::overlap(out[o], i),
                  "the tables and the outputs must not overlap what the call reads");
  }
  const int grid = std::max((max_tokens + kThreads - 1) / kThreads, 1);
  hipLaunchKernelGGL(chunk_map_kernel, dim3(grid), dim3(kThreads), 0, pdk::as_stream(stream), past,
                     added, R, tables, max_blocks, free_ids, n_free, max_tokens, starts, ctx_lens,
                     positions, slots, taken);
  return pdk::check_launch("chunk_map_kernel");
}

extern "C" int pdk_rope_cache_write(const uint16_t* qkv, int64_t ld, const float* inv_freq,
                                    const int32_t* positions, const int32_t* slots, int N,
                                    int n_q_heads, int n_kv_heads, int head_dim, uint16_t* q_out,
                                    uint16_t* cache_k, uint16_t* cache_v, int num_blocks,
                                    uintptr_t stream) {
  pdk::clear_error();
  if (head_dim != kD) {
    pdk::set_error("the chunk kernels implement head_dim %d only (got %d)", kD, head_dim);
    return PDK_ENOTSUP;
  }
  PDK_REQUIRE(N >= 0 && N <= (1 << 20), "N must be in [0, 2^20] (got %d)", N);
  PDK_REQUIRE(n_q_heads >= 1 && n_kv_heads >= 1 && n_q_heads <= 65535 && n_kv_heads <= 65535,
              "head counts out of range");
  PDK_REQUIRE(ld >= (int64_t)(n_q_heads + 2 * n_kv_heads) * kD && ld % 8 == 0 && ld < (1ll << 31),
              "ld must be a multiple of 8 and hold the heads");
  PDK_REQUIRE(num_blocks >= 1 && num_blocks <= (1 << 27), "num_blocks out of range");
  if (N == 0) return PDK_OK;
  PDK_REQUIRE(qkv && inv_freq && positions && slots && q_out && cache_k && cache_v,
              "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(qkv) && pdk::aligned16(q_out) && pdk::aligned16(cache_k) &&
                  pdk::aligned16(cache_v),
              "tensors must be 16-byte aligned");
  const int64_t width = (int64_t)(n_q_heads + 2 * n_kv_heads) * kD;
  const int64_t cache = (int64_t)num_blocks * n_kv_heads * 16 * kD;
  const pdk::Range out[3] = {
      {q_out, (int64_t)N * n_q_heads * kD * 2}, {cache_k, cache * 2}, {cache_v, cache * 2}};
  const pdk::Range in[4] = {{qkv, ((N - 1) * ld + width) * 2},
                            {inv_freq, kD / 2 * 4},
                            {positions, N * 4ll},
                            {slots, N * 4ll}};
  for (int o = 0; o < 3; ++o) {
    for (int p = 0; p < o; ++p) PDK_REQUIRE(!pdk::overlap(out[o], out[p]), "q_out and the caches must not overlap");
    for (const pdk::Range& i : in)
      PDK_REQUIRE(!pdk::overlap(out[o], i), "q_out and the caches must not overlap what the call reads");
  }
  const int tiles = (N + kTok - 1) / kTok;
  // Units apart until there are four workgroups for every CU, and in four parts at least (8192
  // tokens, one set of tensors again and again: 39.8 us, in two 41.8). Up to 1024 tokens a token that lies alone in V's block, as
  // single tokens do, has a lane of its own for 8 dims, stored value by value; beyond, a
  // lane has 8 of them (48 heads, a lane each and a lane for 8: 3.5 and 6.7 us for 16 tokens,
  // 8.5 and 9.8 for 1024, 12.4 and 12.7 for 2048).
  const bool few = tiles <= 64;
  const int units = (kTok * n_q_heads * 8 + kThreads - 1) / kThreads + (n_kv_heads + 1) / 2 +
                    (n_kv_heads * (few ? 16 : 2) + 15) / 16;
  const int shares = std::min(units, std::max(4, (1024 + tiles - 1) / tiles));
  // q and k of more than the eight L2s pass them by, read and written (8192 tokens with 48 heads
  // over three sets of tensors in turn: 42.3 us, q's stores alone 46.7, none 50.3; with the product
  // before and the attention behind 283, 285, 289; 5000 tokens 187, 188, 185).
  const auto kern = few ? rope_write_kernel<16, false>
                    : (int64_t)N * n_q_heads * kD * 2 > (32 << 20) ? rope_write_kernel<2, true>
                                                                   : rope_write_kernel<2, false>;
  hipLaunchKernelGGL(kern, dim3(tiles, shares), dim3(kThreads), 0, pdk::as_stream(stream), qkv, ld,
                     inv_freq, positions, slots, N, n_q_heads, n_kv_heads, q_out, cache_k, cache_v,
                     (int64_t)num_blocks * 16);
  return pdk::check_launch("rope_write_kernel");
}
