// Causal GQA attention of one prompt under a sliding window with sinks, gfx950,
// head_dim 128: the query at position p sees the tokens t <= p with t > p -
// window or t < sinks.
//
// A unit is 32 queries of one query head. S^T = K Q^T with
// v_mfma_f32_32x32x16_bf16, so a lane holds one query (column j = lane & 31) and
// 16 of a tile's 32 scores; O^T += V^T P^T takes them as its B operand with no
// exchange between lanes, because row r of the S^T tile is token pi(r), pi
// swapping bits 2 and 3: accumulators 8 ks .. 8 ks + 7 are then tokens 16 ks + 8
// (lane >> 5) + 0..7. Maximum, sum and rescale are per lane, one lane swap each.
// Scores, maxima, sums and O are fp32; a weight is rounded to bf16 once, for the
// product with V (half a step, 2^-8 of each weight, adds a share of 2^-8 / sqrt(3)
// rms to the output's own rounding of that size, and takes 8 MFMA per tile where
// an exact split into three bf16 parts takes 24, as pdk_prefill_attn does: 4000 tokens
// whole 137 us here and 246 there).
//
// K and V come as rows. A tile is 32 tokens, staged row by row into LDS by
// global_load_lds (16 lanes a row of 256 bytes, no registers, two tiles ahead),
// 16-byte chunk u of token t at place u ^ (t & 15) for K and u ^ 4 (t & 3) for V:
// each is the permutation that gives its reads all banks (K: 16 tokens at one
// chunk; V: 4 tokens at 4 chunks; no conflicts counted). V's operand is dims by
// tokens: the transposing LDS read gives a lane four tokens of its dim. One
// barrier per tile: it waits for the oldest tile's loads (the younger ones counted
// off) and for the reads of the tile whose buffer is filled next.
//
// A token that a query does not see has the weight 0 whatever its score; but 0
// times a V of NaN or infinity is NaN. Where an output comes out NaN and a tile that
// hides tokens from the unit's queries holds such a V, it is done over token by
// token (without_hidden), so what stands in a hidden place reaches no query.
//
// Bound by the wavefronts' issue: per tile and wavefront 16 MFMA (512 cycles) and
// some 100 vector instructions, of which 16 exp2; counted over a prompt of 8000
// with a window of 1024 the matrix cores are busy 40 % of the time and the vector
// units 45 to 50 %, half of it together, at 2.0 to 2.1 GHz. Three workgroups per CU (164
// registers, 48 KiB) hide the rest best; where there are no more workgroups than CUs
// a second team of wavefronts shares the walk (the entry point has the rule). In us,
// 32 query and 8 KV heads, (tokens, window): (8000, 1024) 150, (4000, whole) 140,
// (8000, 128) 46, (470, 128) 10.6.
// Tried and slower there: two workgroups per CU with the scores of the next tile
// computed beside the weights of this one (176, 161, 51, 10.6), two tiles at a
// time (178, 163, 52, 11.2), two units per wavefront (180, 213, 63, 22.6), tiles
// laid out by a launch of their own (166, -, -, 15).
#include <math.h>

#include <algorithm>

#include "pdk_common.h"

namespace {

using pdk::v8;

typedef __bf16 bf16x8_t __attribute__((__vector_size__(16)));
typedef float f32x16 __attribute__((__vector_size__(64)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) uint16_t lds_u16;
typedef const __attribute__((address_space(1))) void global_void;

constexpr int kD = 128;
constexpr int kTile = 32;                 // tokens per K/V tile and queries per unit
constexpr int kTileElems = kTile * kD;    // 8 KiB of K, 8 KiB of V
constexpr int kWaves = 4;
constexpr int kRing = 3;                  // tiles in LDS: 48 KiB, three workgroups per CU
constexpr int kCUs = 256;
constexpr int kLoads = 4;                 // of a wavefront per tile, 1 KiB each

__device__ __forceinline__ f32x16 mfma32(const v8& a, const v8& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ int pi(int x) { return (x & 0x13) | ((x & 4) << 1) | ((x & 8) >> 1); }

// All but the youngest N of this wavefront's loads have arrived and its LDS
// reads are done; then the workgroup's barrier.
template <int N>
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// O^T's operands of a tile, va[n][h] of dims 32 (n0 + n) .. and tokens 16h .., by
// transposing reads at at0, at1 (n = 0, 1) and 4, 16 and 20 rows on. The builtin
// would make the compiler wait for every tile in flight, which it cannot tell
// from the one read here; the wait for these reads is part of the statement.
__device__ __forceinline__ void read_v(uint32_t at0, uint32_t at1, v8 (&va)[2][2]) {
  uint2 x[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:1024\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:4096\n\t"
      "ds_read_b64_tr_b16 %3, %8 offset:5120\n\t"
      "ds_read_b64_tr_b16 %4, %9\n\t"
      "ds_read_b64_tr_b16 %5, %9 offset:1024\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:4096\n\t"
      "ds_read_b64_tr_b16 %7, %9 offset:5120\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]),
        "=&v"(x[6]), "=&v"(x[7])
      : "v"(at0), "v"(at1)
      : "memory");
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      va[n][h] = v8{{x[4 * n + 2 * h].x, x[4 * n + 2 * h].y, x[4 * n + 2 * h + 1].x,
                     x[4 * n + 2 * h + 1].y}};
}

struct Rows {
  const uint16_t* p;
  int64_t ld;
};

// Whether some query of the unit does not see some token of tile t0.
__device__ __forceinline__ bool hides(int t0, int p0, int window, int sinks) {
  return t0 + kTile - 1 > p0 || (t0 + window < p0 + kTile && t0 + kTile > sinks);
}

// Whether tile t0's V (rows past T: row T - 1) holds a NaN or an infinity.
__device__ bool not_finite(const Rows& v, int T, int kvh, int t0, int lane) {
  const uint16_t* p = v.p + (int64_t)min(t0 + (lane >> 1), T - 1) * v.ld + kvh * kD + (lane & 1) * 64;
  uint32_t found = 0;
#pragma unroll 1
  for (int x = 0; x < 8; ++x) {
    const v8 a = pdk::ld16(p + 8 * x);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      found |= (a.w[w] & 0x7f80u) == 0x7f80u || (a.w[w] & 0x7f800000u) == 0x7f800000u;
  }
  return __any(found);
}

// The outputs that are NaN done over, token by token without the hidden ones; m is
// the maximum that the others' weights have been taken with. It ends as soon as
// each of them is NaN by a token that is seen.
__device__ void without_hidden(const Rows& q, const Rows& k, const Rows& v, int T, int head, int kvh,
                               int qt, int lane, float c, int window, int sinks, float m, float l,
                               f32x16 (&o)[4]) {
  const int j = lane & 31, hh = lane >> 5, p = min(qt * kTile + j, T - 1);
  const int last = min(qt * kTile + kTile, T) - 1, first = max(qt * kTile - window + 1, 0);
  const uint16_t* qp = q.p + (int64_t)p * q.ld + head * kD + 8 * hh;
  const float mc = m == -INFINITY ? 0.f : m * c;
  uint32_t open[2] = {0, 0};               // a bit for each of the lane's outputs to be done over
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (l == l && o[n][i] != o[n][i]) {
        open[n >> 1] |= 1u << (16 * (n & 1) + i);
        o[n][i] = 0.f;
      }
#pragma unroll 1
  for (int t = 0; t <= last; t = t + 1 < first && t + 1 >= sinks ? first : t + 1) {
    const uint16_t* kp = k.p + (int64_t)t * k.ld + kvh * kD + 8 * hh;
    float s = 0.f;
#pragma unroll 1
    for (int x = 0; x < 8; ++x) {
      const v8 a = pdk::ld16(qp + 16 * x), b = pdk::ld16(kp + 16 * x);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        s += pdk::bf16_to_f32(a.w[w] & 0xffffu) * pdk::bf16_to_f32(b.w[w] & 0xffffu);
        s += pdk::bf16_to_f32(a.w[w] >> 16) * pdk::bf16_to_f32(b.w[w] >> 16);
      }
    }
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(s), false,
                                                    false);
    const bool seen = t <= p && (t > p - window || t < sinks);
    const float w = __builtin_amdgcn_exp2f((__uint_as_float(x[0]) + __uint_as_float(x[1])) * c - mc);
    const uint16_t* vp = v.p + (int64_t)t * v.ld + kvh * kD + 4 * hh;
    bool left = false;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint2 u = *reinterpret_cast<const uint2*>(vp + 32 * n + 8 * g);
        const uint32_t h[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * g + e;
          if (open[n >> 1] >> (16 * (n & 1) + i) & 1) {
            if (seen) o[n][i] += w * pdk::bf16_to_f32(h[e]);
            left |= o[n][i] == o[n][i];
          }
        }
      }
    if (!__any(left)) break;
  }
}

// One wavefront: one unit. A workgroup takes kWaves consecutive units of one KV
// head, heads of the group fastest (for G = 4 one query tile's heads), which read
// the same tiles; the KV head is the fastest index of the grid, so that 8 of them
// spread over the 8 XCDs. The last query tiles go first: without a window they
// have the most to walk.
// kTeams 2: a second team of kWaves walks every other tile with buffers of its own,
// and hands its sums to the first at the end.
template <int kTeams>
__global__ __launch_bounds__(64 * kWaves * kTeams, kTeams == 1 ? 3 : 2) void prefill_window_kernel(
    Rows q, Rows k, Rows v, int T, int NH, int NKV, float c, int window, int sinks,
    uint16_t* out) {
  __shared__ __align__(1024) uint16_t smem[kTeams][2 * kRing * kTileElems];   // K tiles, V tiles
  const int team = kTeams == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & (kWaves - 1);
  const int lane = threadIdx.x & 63;
  uint16_t* const sm = smem[team];
  const int j = lane & 31, hh = lane >> 5;
  const int G = NH / NKV, units = (T + kTile - 1) / kTile * G;
  const int kvh = blockIdx.x % NKV;
  const int wg = (units + kWaves - 1) / kWaves - 1 - (int)(blockIdx.x / NKV);
  const int u_first = wg * kWaves, u_last = min(u_first + kWaves, units) - 1;
  // The tiles that the workgroup walks: number i is i below `lead` (the sinks'),
  // i + skip from there on (those from its first query's window to its last query).
  const int w_tile = max(u_first / G * kTile - window + 1, 0) / kTile;
  const int lead = min((sinks + kTile - 1) / kTile, w_tile), skip = w_tile - lead;
  const int n_all = u_last / G + 1 - skip;
  const int n_walk = kTeams == 1 ? n_all : (n_all + 1 - team) / 2;   // the team's, from its `team`th on
  const int u = min(u_first + wave, units - 1);                  // a spare one repeats the last
  const int qt = u / G, head = kvh * G + (u - qt * G);
  auto tile_at = [&](int i) {
    const int x = kTeams * i + team;
    return x >= lead ? x + skip : x;
  };

  // Staging: load l of a wavefront covers tokens 8 wave + 4 l + lane / 16. A whole
  // tile's offsets from its first row are the same for every tile.
  const int tok = 8 * wave + (lane >> 4);
  uint32_t k_off[2], v_off[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int t = tok + 4 * x;
    k_off[x] = (t * (uint32_t)k.ld + ((lane & 15) ^ (t & 15)) * 8) * 2;
    v_off[x] = (t * (uint32_t)v.ld + ((lane & 15) ^ ((t & 3) << 2)) * 8) * 2;
  }
  auto fetch = [&](uint16_t* __restrict__ to, int i) __attribute__((always_inline)) {
    const int t0 = tile_at(i) * kTile;
    const char* tk = reinterpret_cast<const char*>(k.p + (int64_t)t0 * k.ld + kvh * kD);
    const char* tv = reinterpret_cast<const char*>(v.p + (int64_t)t0 * v.ld + kvh * kD);
    uint32_t ko[2] = {k_off[0], k_off[1]}, vo[2] = {v_off[0], v_off[1]};
    if (t0 + kTile > T) {                  // rows past T, hidden from every query, read row T - 1
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t past = max(t0 + tok + 4 * x - (T - 1), 0);
        ko[x] -= past * (uint32_t)k.ld * 2;
        vo[x] -= past * (uint32_t)v.ld * 2;
      }
    }
    uint16_t* at = to + 8 * wave * kD;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      __builtin_amdgcn_global_load_lds((global_void*)(tk + ko[x]), (lds_void*)(at + 4 * x * kD), 16,
                                       0, 0);
      __builtin_amdgcn_global_load_lds((global_void*)(tv + vo[x]),
                                       (lds_void*)(at + (kRing * kTileElems + 4 * x * kD)), 16, 0, 0);
    }
  };
  v8 qv[8];
  {
    const uint16_t* p = q.p + (int64_t)min(qt * kTile + j, T - 1) * q.ld + head * kD + 8 * hh;
#pragma unroll
    for (int s = 0; s < 8; ++s) qv[s] = pdk::ld16(p + 16 * s);
  }
#pragma unroll
  for (int x = 0; x < kRing - 1; ++x)
    if (x < n_walk) fetch(sm + x * kTileElems, x);
  // Where this lane's operands lie in a tile (elements): K chunk 2x + hh of token
  // pi(j), so chunk x is this place with bits 4 to 6 flipped by x; of V, in its
  // group of 16 lanes, tokens 8 hh + (lane & 15) / 4 (and 4, 16, 20 on) at dims 32n
  // + 16 (j / 16) + 4 (lane & 3).
  const int k_at = pi(j) * kD + ((hh ^ pi(j)) & 15) * 8;
  const int vr = (lane & 15) >> 2;
  const int v_at = (8 * hh + vr) * kD + ((2 * (j >> 4) + ((lane & 3) >> 1)) ^ (vr << 2)) * 8 +
                   (lane & 1) * 4;
  uint32_t v_addr[4];
#pragma unroll
  for (int n = 0; n < 4; ++n)
    v_addr[n] = (uint32_t)(uintptr_t)(lds_u16*)(sm + kRing * kTileElems + (v_at ^ (n << 5)));

  f32x16 o[4], s;
  v8 p[2];
  float m = -INFINITY, l = 0.f;           // m: raw-score maximum in use; l: this lane's tokens
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;

  auto load_k = [&](const uint16_t* __restrict__ st, v8 (&kr)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 8; ++x) kr[x] = pdk::ld16(st + (k_at ^ (x << 4)));
  };
  auto scores = [&](const v8 (&kr)[8]) __attribute__((always_inline)) {
    f32x16 r;
#pragma unroll
    for (int x = 0; x < 16; ++x) r[x] = 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) r = mfma32(kr[x], qv[x], r);
    return r;
  };
  auto step = [&](int i, const uint16_t* __restrict__ at_k, uint16_t* __restrict__ to,
                  uint32_t at_v) __attribute__((always_inline)) {
    if (i + 1 < n_walk) tile_barrier<kLoads>();
    else tile_barrier<0>();
    if (i + 2 < n_walk) fetch(to, i + 2);
    v8 kr[8];
    load_k(at_k, kr);
    s = scores(kr);
    v8 va[2][2];
    read_v(v_addr[0] + at_v, v_addr[1] + at_v, va);              // during the products
    const int t0 = tile_at(i) * kTile, p0 = qt * kTile;
    // Tokens after some query (and so those past T), or that have left some
    // query's window.
    if (hides(t0, p0, window, sinks)) {
      const int ago = p0 + j - t0 - 8 * hh;                      // of the lane's first token
      const int sink = sinks - t0 - 8 * hh;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int e = 16 * (x >> 3) + (x & 7);
        s[x] = (e > ago) | ((ago - e >= window) & (e >= sink)) ? -INFINITY : s[x];
      }
    }
    float mx = s[0];
#pragma unroll
    for (int x = 1; x < 16; ++x) mx = vmax(mx, s[x]);
    {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx),
                                                      false, false);
      mx = vmax(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    // The maximum in use follows the running one only when it falls more than
    // 2^8 behind: a common factor costs neither P nor the sums any precision,
    // and O is rescaled a few times per query instead of at almost every tile.
    if (__any((mx - m) * c > 8.f)) {
      const float m_new = vmax(m, mx);
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * c);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[n][x] *= alpha;
    }
    const float mc = m == -INFINITY ? 0.f : m * c;               // no token so far: weights are 0
    float part[2] = {0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 16; x += 2) {
      const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], c, -mc));
      const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x + 1], c, -mc));
      part[0] += a;
      part[1] += b;
      p[x >> 3].w[(x & 7) >> 1] = pdk::pack_bf16x2_rne(a, b);
    }
    l += part[0] + part[1];
#pragma unroll
    for (int n0 = 0; n0 < 4; n0 += 2) {                          // O += V^T P^T
      if (n0) read_v(v_addr[n0] + at_v, v_addr[n0 + 1] + at_v, va);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < 2; ++n) o[n0 + n] = mfma32(va[n][h], p[h], o[n0 + n]);
    }
  };
  for (int i = 0, r = 0; i < n_walk; ++i) {
    const int r2 = r == 0 ? kRing - 1 : r - 1;                   // of tile i + 2: that of tile i - 1
    step(i, sm + r * kTileElems, sm + r2 * kTileElems, r * kTileElems * 2);
    r = r + 1 == kRing ? 0 : r + 1;
  }
  if constexpr (kTeams == 2) {
    // The barriers match: the second team has as many tiles, or one less.
    if (n_walk < (n_all + 1) / 2) tile_barrier<0>();
    tile_barrier<0>();                                           // nobody reads tiles any more
    float4* const mem = reinterpret_cast<float4*>(smem) + wave * (17 * 64) + lane;
    if (team == 1) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int x = 0; x < 16; x += 4)
          mem[(4 * n + x / 4) * 64] = make_float4(o[n][x], o[n][x + 1], o[n][x + 2], o[n][x + 3]);
      mem[16 * 64] = make_float4(m, l, 0.f, 0.f);
    }
    tile_barrier<0>();
    if (team == 1) return;
    const float4 ml = mem[16 * 64];
    const float m_new = vmax(m, ml.x);
    const float a0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * c);
    const float a1 = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - m_new) * c);
    m = m_new;
    l = l * a0 + ml.y * a1;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int x = 0; x < 16; x += 4) {
        const float4 y = mem[(4 * n + x / 4) * 64];
        o[n][x] = o[n][x] * a0 + y.x * a1;
        o[n][x + 1] = o[n][x + 1] * a0 + y.y * a1;
        o[n][x + 2] = o[n][x + 2] * a0 + y.z * a1;
        o[n][x + 3] = o[n][x + 3] * a0 + y.w * a1;
      }
  }

  float bad = 0.f;                        // NaN once an output is not finite
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) bad += o[n][i] * 0.f;
  if (__builtin_expect(__any(bad != bad), 0)) {
    bool hidden = false;
#pragma unroll 1
    for (int i = 0; i < n_all && !hidden; ++i) {
      const int t0 = (i >= lead ? i + skip : i) * kTile;
      if (hides(t0, qt * kTile, window, sinks)) hidden = not_finite(v, T, kvh, t0, lane);
    }
    int ln = lane;                        // q's addresses anew: kept, they would be spilled
    asm("" : "+v"(ln));
    if (hidden) without_hidden(q, k, v, T, head, kvh, qt, ln, c, window, sinks, m, l, o);
  }

  // Lane (hh, j) holds dims 32n + 8g + 4hh + 0..3 of query j (g = 0..3); a lane
  // swap of groups g, g + 1 gives each half 8 consecutive dims: 16-byte stores.
  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false,
                                                    false);
    const float inv = 1.f / (__uint_as_float(x[0]) + __uint_as_float(x[1]));   // its own token: > 0
    const int t = qt * kTile + j;
    const bool mine = t < T && u_first + wave < units;
    uint16_t* op = out + ((int64_t)min(t, T - 1) * NH + head) * kD + 8 * hh;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        uint32_t w[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            w[i][e] = pdk::pack_bf16x2_rne(o[n][4 * (g + i) + 2 * e] * inv,
                                           o[n][4 * (g + i) + 2 * e + 1] * inv);
        const auto b0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto b1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        const v8 res{{b0[0], b1[0], b0[1], b1[1]}};
        if (mine) pdk::st16(op + 32 * n + 8 * g, res);
      }
  }
}

}  // namespace

extern "C" int pdk_prefill_attn_window(const uint16_t* q, int64_t q_tok_stride, const uint16_t* k,
                                       int64_t k_tok_stride, const uint16_t* v,
                                       int64_t v_tok_stride, int T, int n_q_heads, int n_kv_heads,
                                       int head_dim, float scale, int window, int sinks,
                                       uint16_t* out, uintptr_t stream) {
  pdk::clear_error();
  if (head_dim != kD) {
    pdk::set_error("the prefill kernels implement head_dim %d only (got %d)", kD, head_dim);
    return PDK_ENOTSUP;
  }
  PDK_REQUIRE(T >= 1 && T <= (1 << 20), "T must be in [1, 2^20] (got %d)", T);
  PDK_REQUIRE(n_kv_heads >= 1 && n_q_heads >= n_kv_heads && n_q_heads % n_kv_heads == 0 &&
                  n_q_heads <= 65535,
              "n_q_heads=%d must be a multiple of n_kv_heads=%d", n_q_heads, n_kv_heads);
  PDK_REQUIRE(window >= 1 && sinks >= 0, "window must be >= 1 and sinks >= 0 (got %d, %d)", window,
              sinks);
  PDK_REQUIRE(q && k && v && out, "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(q) && pdk::aligned16(k) && pdk::aligned16(v) && pdk::aligned16(out),
              "tensors must be 16-byte aligned");
  PDK_REQUIRE(q_tok_stride >= (int64_t)n_q_heads * kD && q_tok_stride % 8 == 0 &&
                  k_tok_stride >= (int64_t)n_kv_heads * kD && k_tok_stride % 8 == 0 &&
                  v_tok_stride >= (int64_t)n_kv_heads * kD && v_tok_stride % 8 == 0,
              "token strides must be multiples of 8 and hold heads * D elements");
  PDK_REQUIRE(k_tok_stride < (1 << 24) && v_tok_stride < (1 << 24),
              "k and v token strides must be below 2^24");
  PDK_REQUIRE(scale > 0.f && scale < INFINITY, "scale must be positive and finite (got %g)",
              (double)scale);
  // Beyond T neither hides anything.
  window = std::min(window, T);
  sinks = std::min(sinks, T);
  const int64_t units = (int64_t)((T + kTile - 1) / kTile) * (n_q_heads / n_kv_heads);
  const int64_t blocks = (units + kWaves - 1) / kWaves * n_kv_heads;
  PDK_REQUIRE(units < (1ll << 30) && blocks < (1ll << 31), "launch too large");
  // A second team where a workgroup has a CU to itself and more than 8 tiles to walk:
  // it halves that chain (0.7 us a tile) for 1.5 us of handing over. us with one team
  // and with two, 32 query and 8 KV heads, (tokens, window): (1000, whole) 29.9 and 25.2,
  // (1000, 512) 20.4 and 18.2, (470, whole) 16.4 and 14.4, (256, whole) 11.0 and 11.0,
  // (470, 128) 10.7 and 11.0, (100, 64) 7.5 and 8.6.
  const int walk = std::min((T + kTile - 1) / kTile,
                            (window + kTile - 2) / kTile + 1 + (sinks + kTile - 1) / kTile);
  const bool two = blocks <= kCUs && walk > 8;
  hipLaunchKernelGGL(two ? prefill_window_kernel<2> : prefill_window_kernel<1>,
                     dim3((unsigned)blocks), dim3(64 * kWaves * (two ? 2 : 1)), 0,
                     pdk::as_stream(stream), Rows{q, q_tok_stride}, Rows{k, k_tok_stride},
                     Rows{v, v_tok_stride}, T, n_q_heads, n_kv_heads, scale * 1.4426950408889634f,
                     window, sinks, out);
  return pdk::check_launch("prefill_window_kernel");
}
