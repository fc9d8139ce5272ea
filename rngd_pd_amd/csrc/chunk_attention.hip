// Causal GQA attention of several requests' new tokens over the paged cache, gfx950,
// head_dim 128: new token i of request r stands at position p = ctx_r - n_r + i and sees
// the cached tokens t <= p (its own among them), under a window t > p - window or t <
// sinks. Tokens of blocks that the table does not name are seen by nobody; a token
// that sees nothing gets zeros.
//
// A unit is 32 rows: the query heads that share a KV head, token after token (row =
// token * G + head of the group), so that a few tokens' heads fill it and read each key
// and value once. S^T = K Q^T with v_mfma_f32_32x32x16_bf16: a lane holds one row
// (column j = lane & 31) and 16 of a tile's 32 scores. Row r of the S^T tile is token
// pi(r), pi swapping bits 2 and 3: accumulators 8 ks .. 8 ks + 7 are then tokens 16 ks +
// 8 (lane >> 5) + 0..7, which are the B operand of O^T += V^T P^T with no exchange
// between lanes, and the cache's own order is that of both A operands: 8 tokens of a
// K block at one group of 8 dims are 128 consecutive bytes, V's rows of 16 tokens 32.
// Maximum, sum and rescale are per lane, one lane swap each. Scores, maxima, sums and O
// are fp32; a weight is rounded to bf16 once, for the product with V (half a step,
// 2^-8 of each weight: a share of 2^-8 / sqrt(3) rms beside the output's own rounding).
//
// Requests of one unit (n G <= 32: single tokens, drafts) are bound by HBM: a
// workgroup's four wavefronts walk every fourth tile of a split with operands straight
// from memory in registers, the next tile's under way, and add up in LDS. Longer ones
// are bound by the wavefronts' issue: a workgroup takes 128 rows, its four wavefronts
// share tiles staged into LDS by global_load_lds two ahead, one barrier per tile. Both
// split the context over workgroups where those are few; a second launch joins the
// splits in a fixed order.
//
// A token that a row does not see has the weight 0 whatever its score; 0 times a V of
// NaN or infinity would be NaN, so a tile that hides tokens and holds such a V is
// multiplied without those values, and what they come to where they are seen is added
// at the end (clean, add_cleaned).
#include <math.h>

#include <algorithm>

#include "lds_copy.h"

namespace {

using pdk::v8;

typedef __bf16 bf16x8_t __attribute__((__vector_size__(16)));
typedef float f32x16 __attribute__((__vector_size__(64)));

constexpr int kD = 128;
constexpr int kBlockElems = 16 * kD;      // of K or V in a block, per head
constexpr int kTile = 32;                 // tokens: two blocks
constexpr int kTileElems = 2 * kBlockElems;
constexpr int kWaves = 4;
constexpr int kRows = 32 * kWaves;        // of a workgroup of a long request
constexpr int kRing = 3;                  // tiles in LDS
constexpr int kLoads = 4;                 // of a wavefront per tile, 1 KiB each
constexpr int kMaxRequests = 65535;
constexpr int kMaxSplits = 64;
constexpr int kRecord = 64 * 66;          // floats of a unit's sums: O 64 lanes x 64, (m, l)

struct Args {
  const uint16_t* q;
  int64_t q_ld;
  const uint16_t *k, *v;
  int num_blocks;
  const int32_t* tables;
  int W;
  const int32_t *starts, *ctx;
  int N, R, NH, NKV;
  float c;                                // scale * log2(e)
  int window, sinks;
  float* ws;
  uint16_t* out;
  // Rows up to which a request is one unit's (32, or 0 where all are taken as longer
  // ones); tiles of a split and splits at most, of the former and the latter; workgroups of
  // the longer ones' rows at most.
  int few_rows, few_per, few_splits, big_per, big_splits, big_tiles;
};

__device__ __forceinline__ f32x16 mfma32(const v8& a, const v8& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ float swap_add(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A request's new tokens as far as the tensors hold them.
struct Request {
  int start, n, past;
};

__device__ __forceinline__ Request request(const Args& a, int r) {
  const int s = a.starts[r], e = a.starts[r + 1];
  Request q;
  q.start = min(max(s, 0), a.N);
  q.n = max(min(e, a.N) - q.start, 0);
  q.past = min(max(a.ctx[r], 0), 1 << 30) - q.n;
  return q;
}

// The tiles that rows of the positions p0 .. p1 walk: number i is i below `lead` (the
// sinks'), i + skip from there on (from p0's window to p1).
struct Walk {
  int lead, skip, n;
  __device__ __forceinline__ int tile(int i) const { return i >= lead ? i + skip : i; }
};

__device__ __forceinline__ Walk walk(const Args& a, int p0, int p1) {
  Walk w;
  const int end = p1 < 0 ? 0 : min(p1, a.W * 16 - 1) / kTile + 1;
  const int first = min(max(p0 - a.window + 1, 0) / kTile, end);
  w.lead = min((a.sinks + kTile - 1) / kTile, first);
  w.skip = first - w.lead;
  w.n = end - w.skip;
  return w;
}

// The splits that a walk of n tiles has.
__device__ __forceinline__ int splits_of(int n, int per, int most) {
  return min(max((n + per - 1) / per, 1), most);
}

// Ids of block b of 64 tiles, one tile a lane; which of the tiles' blocks are there.
struct BlockIds {
  int id;
  uint64_t ok[2];
};

__device__ __forceinline__ int block_id(const Args& a, int r, int e) {
  const int id = a.tables[(int64_t)r * a.W + min(e, a.W - 1)];
  return e < a.W && id >= 0 && id < a.num_blocks ? id : -1;
}

__device__ __forceinline__ BlockIds load_ids(const Args& a, int r, int tile, int b) {
  const int id[2] = {block_id(a, r, 2 * tile), block_id(a, r, 2 * tile + 1)};
  return BlockIds{max(b ? id[1] : id[0], 0), {__ballot(id[0] >= 0), __ballot(id[1] >= 0)}};
}

// One lane's row of a unit.
struct Row {
  int token, head, p;                     // row of q, query head, position
  bool mine;                              // a row of its own, not a repeated last one
};

__device__ __forceinline__ Row row_at(const Args& a, const Request& q, int kvh, int row) {
  const int G = a.NH / a.NKV, last = q.n * G - 1;
  Row r;
  r.mine = row <= last;
  const int x = min(row, last), i = x / G;
  r.token = q.start + i;
  r.head = kvh * G + (x - i * G);
  r.p = q.past + i;
  return r;
}

__device__ __forceinline__ void load_q(const Args& a, const Row& r, int hh, v8 (&qv)[8]) {
  const uint16_t* p = a.q + (int64_t)r.token * a.q_ld + r.head * kD + 8 * hh;
#pragma unroll
  for (int x = 0; x < 8; ++x) qv[x] = pdk::ld16(p + 16 * x);
}

// The sums of a lane: its row's maximum in use, its tokens' weights, its row's O^T.
struct Sums {
  float m, l;
  f32x16 o[4];
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[n][x] = 0.f;
  }
};

__device__ __forceinline__ f32x16 scores(const v8 (&kr)[8], const v8 (&qv)[8]) {
  f32x16 s;
#pragma unroll
  for (int x = 0; x < 16; ++x) s[x] = 0.f;
#pragma unroll
  for (int x = 0; x < 8; ++x) s = mfma32(kr[x], qv[x], s);
  return s;
}

// A lane's place in a tile, for masks: how long ago the lane's first token is, how far
// the sinks reach from it; whether the tile's two blocks are there.
struct Place {
  int ago, sink, window;
  bool ok[2];
  __device__ __forceinline__ bool hidden(int x) const {
    const int e = 16 * (x >> 3) + (x & 7);
    return (e > ago) | ((ago - e >= window) & (e >= sink)) | !ok[x >> 3];
  }
};

__device__ __forceinline__ Place place(const Args& a, int t0, int p, int hh, bool ok0, bool ok1) {
  return Place{p - t0 - 8 * hh, a.sinks - t0 - 8 * hh, a.window, {ok0, ok1}};
}

// Whether some row of the positions p0 .. p1 does not see some token of tile t0.
__device__ __forceinline__ bool hides(const Args& a, int t0, int p0, int p1, bool ok) {
  return t0 + kTile - 1 > p0 || (t0 + a.window <= p1 && t0 + kTile > a.sinks) || !ok;
}

// Scores to weights, the sums' maximum following.
__device__ __forceinline__ void weigh(const f32x16& s, float c, Sums& a, v8 (&p)[2]) {
  float mx = s[0];
#pragma unroll
  for (int x = 1; x < 16; ++x) mx = vmax(mx, s[x]);
  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false,
                                                    false);
    mx = vmax(__uint_as_float(x[0]), __uint_as_float(x[1]));
  }
  // The maximum in use follows the running one only when it falls more than 2^8
  // behind: a common factor costs neither weights nor sums any precision, and O is
  // rescaled a few times per row instead of at almost every tile.
  if (__any((mx - a.m) * c > 8.f)) {
    const float m_new = vmax(a.m, mx);
    const float alpha = a.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((a.m - m_new) * c);
    a.m = m_new;
    a.l *= alpha;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int x = 0; x < 16; ++x) a.o[n][x] *= alpha;
  }
  const float mc = a.m == -INFINITY ? 0.f : a.m * c;             // no token so far: weights are 0
  float part[2] = {0.f, 0.f};
#pragma unroll
  for (int x = 0; x < 16; x += 2) {
    const float u = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], c, -mc));
    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x + 1], c, -mc));
    part[0] += u;
    part[1] += w;
    p[x >> 3].w[(x & 7) >> 1] = pdk::pack_bf16x2_rne(u, w);
  }
  a.l += part[0] + part[1];
}

// The values of a that are not finite replaced by 0; whether there are any.
__device__ __forceinline__ bool clean(v8& a) {
  bool odd = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const bool lo = (a.w[w] & 0x7f80u) == 0x7f80u, hi = (a.w[w] & 0x7f800000u) == 0x7f800000u;
    odd |= lo | hi;
    a.w[w] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
  }
  return odd;
}

// What clean() took from the tiles `first` to `end` of a walk that hide something:
// infinities and NaN of the tokens that a row sees, added to its O. Marks of them (1 for
// infinity, 64 for -infinity, 4096 for NaN) times 1 for each token that is seen: the
// digits say what to add.
__device__ __forceinline__ void add_cleaned(const Args& a, const Walk& w, int first, int end, int r,
                                            int kvh, int p, int p0, int p1, int lane, f32x16 (&o)[4]) {
  const int j = lane & 31, hh = lane >> 5;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    uint32_t plus = 0, minus = 0, none = 0;          // a bit for each of the lane's 16 outputs
#pragma unroll 1
    for (int i = first; i < end; ++i) {
      const int t0 = w.tile(i) * kTile;
      int id[2];
      Place at = place(a, t0, p, hh, true, true);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        id[b] = block_id(a, r, t0 / 16 + b);
        at.ok[b] = id[b] >= 0;
      }
      if (!hides(a, t0, p0, p1, at.ok[0] && at.ok[1])) continue;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (!at.ok[b]) continue;
        const v8 v = pdk::ld16(a.v + ((int64_t)id[b] * a.NKV + kvh) * kBlockElems + (32 * n + j) * 16 + hh * 8);
        v8 mark, seen;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t m = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t u = v.w[x] >> (16 * e) & 0xffffu;
            const uint32_t code = u == 0x7f80u ? 0x3f80u : u == 0xff80u ? 0x4280u : 0x4580u;
            m |= ((u & 0x7f80u) == 0x7f80u ? code : 0u) << (16 * e);
          }
          mark.w[x] = m;
          seen.w[x] = (at.hidden(8 * b + 2 * x) ? 0u : 0x3f80u) |
                      (at.hidden(8 * b + 2 * x + 1) ? 0u : 0x3f800000u);
        }
        f32x16 found;
#pragma unroll
        for (int x = 0; x < 16; ++x) found[x] = 0.f;
        found = mfma32(mark, seen, found);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const uint32_t u = (uint32_t)found[x];
          plus |= (u & 63 ? 1u : 0u) << x;
          minus |= (u & 0xfc0 ? 1u : 0u) << x;
          none |= (u >> 12 ? 1u : 0u) << x;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      float add = plus >> x & 1 ? INFINITY : 0.f;
      add = minus >> x & 1 ? add - INFINITY : add;
      o[n][x] += none >> x & 1 ? __builtin_nanf("") : add;
    }
  }
}

// A unit's 32 dims 32n .. as bf16: the lane holds dims 8g + 4hh + 0..3 of its row (g =
// 0..3); a lane swap of groups g, g + 1 gives each half 8 consecutive dims.
__device__ __forceinline__ void store_dims(const Args& a, const Row& r, int n, int hh, float inv,
                                           const float (&o)[16]) {
  uint16_t* op = a.out + ((int64_t)r.token * a.NH + r.head) * kD + 32 * n + 8 * hh;
#pragma unroll
  for (int g = 0; g < 4; g += 2) {
    uint32_t w[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        w[i][e] = pdk::pack_bf16x2_rne(o[4 * (g + i) + 2 * e] * inv, o[4 * (g + i) + 2 * e + 1] * inv);
    const auto b0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
    const auto b1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
    const v8 res{{b0[0], b1[0], b0[1], b1[1]}};
    if (r.mine) pdk::st16(op + 8 * g, res);
  }
}

__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// A split's sums of a unit: float4s [16][64 lanes], then (m, l) per lane, both halves'
// weights in l.
__device__ __forceinline__ float* record(const Args& a, int64_t unit, int splits, int z) {
  return a.ws + (unit * splits + z) * kRecord;
}

__device__ __forceinline__ int64_t big_base(const Args& a) {
  return a.few_splits > 1 ? (int64_t)a.R * a.NKV * a.few_splits * kRecord : 0;
}

__device__ __forceinline__ void keep_dims(float* rec, int n, int lane, const float (&o)[16]) {
  float4* p = reinterpret_cast<float4*>(rec) + 4 * n * 64 + lane;
#pragma unroll
  for (int x = 0; x < 16; x += 4) p[x / 4 * 64] = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
}

__device__ __forceinline__ void keep_sums(float* rec, int lane, float m, float l) {
  reinterpret_cast<float2*>(rec + 64 * 64)[lane] = make_float2(m, l);
}

// ---- requests of one unit -----------------------------------------------------
struct FewShared {
  float4 o[kWaves][16][64];
  float2 ml[kWaves][64];
};

__device__ __forceinline__ void few_unit(const Args& a, FewShared& sm, int r, int kvh, int z) {
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.NH / a.NKV;
  const Request q = request(a, r);
  if (q.n == 0 || q.n > 32 || q.n * G > a.few_rows) return;
  const int p0 = q.past, p1 = q.past + q.n - 1;
  const Walk w = walk(a, p0, p1);
  const int splits = splits_of(w.n, a.few_per, a.few_splits);
  if (z >= splits) return;
  const int first = z * a.few_per, end = z + 1 == splits ? w.n : first + a.few_per;
  const Row row = row_at(a, q, kvh, j);
  Sums sum;
  sum.clear();
  const int n_own = (end - first - wave + kWaves - 1) / kWaves;
  bool odd = false;
  if (n_own > 0) {
    v8 qv[8], kr[8], va[2][4];
    load_q(a, row, hh, qv);
    auto tile_of = [&](int i) { return w.tile(first + wave + kWaves * min(i, n_own - 1)); };
    BlockIds ids[2];                      // of both blocks
    auto next_ids = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < 2; ++b) ids[b] = load_ids(a, r, tile_of(i + lane), b);
    };
    next_ids(0);
    // Where a lane's operands lie in a tile (elements): K's token pi(j) at dims 16 x + 8 hh
    // is 256 x bytes on; V's dims 32 n + j, tokens 8 hh .. of block ks.
    const int k_at = ((j >> 3) & 1) * 1024 + hh * 64 + (j & 7) * 8;
    const int v_at = j * 16 + hh * 8;
    auto block = [&](int i, int b) {
      const int id = __builtin_amdgcn_readlane(ids[b].id, i & 63);
      return ((int64_t)id * a.NKV + kvh) * kBlockElems;
    };
    auto load_k = [&](int i) __attribute__((always_inline)) {
      const int64_t b0 = block(i, 0), b1 = block(i, 1);
      const uint16_t* p = a.k + (j & 16 ? b1 : b0) + k_at;
#pragma unroll
      for (int x = 0; x < 8; ++x) kr[x] = pdk::ld16(p + 128 * x);
    };
    auto load_v = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint16_t* p = a.v + block(i, b) + v_at;
#pragma unroll
        for (int n = 0; n < 4; ++n) va[b][n] = pdk::ld16(p + 512 * n);
      }
    };
    load_k(0);
    load_v(0);
    auto step = [&](int i, bool more) __attribute__((always_inline)) {
      const bool ok0 = ids[0].ok[0] >> (i & 63) & 1, ok1 = ids[0].ok[1] >> (i & 63) & 1;
      const int t0 = tile_of(i) * kTile;
      if (more && (i & 63) == 63) next_ids(i + 1);
      f32x16 s = scores(kr, qv);
      if (more) load_k(i + 1);
      const Place at = place(a, t0, row.p, hh, ok0, ok1);
      const bool edge = hides(a, t0, p0, p1, ok0 && ok1);
      if (edge) {
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = at.hidden(x) ? -INFINITY : s[x];
      }
      v8 p[2];
      weigh(s, a.c, sum, p);
      if (edge) {
        bool found = false;
#pragma unroll
        for (int x = 0; x < 8; ++x) found |= clean(va[x >> 2][x & 3]);
        odd |= __any(found);
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) sum.o[x & 3] = mfma32(va[x >> 2][x & 3], p[x >> 2], sum.o[x & 3]);
      if (more) load_v(i + 1);
    };
#pragma unroll 1
    for (int i = 0; i + 1 < n_own; ++i) step(i, true);
    step(n_own - 1, false);
  }
  // The wavefront's own tiles alone are its sums', any of which may be added to.
  if (__builtin_expect(odd, 0))
    for (int i = first + wave; i < end; i += kWaves)
      add_cleaned(a, w, i, i + 1, r, kvh, row.p, p0, p1, lane, sum.o);
  // Wavefront n adds up dims 32 n .. of the four.
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int x = 0; x < 16; x += 4)
      sm.o[wave][4 * n + x / 4][lane] = make_float4(sum.o[n][x], sum.o[n][x + 1], sum.o[n][x + 2],
                                                    sum.o[n][x + 3]);
  sm.ml[wave][lane] = make_float2(sum.m, swap_add(sum.l));
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
  for (int u = 0; u < kWaves; ++u) m = vmax(m, sm.ml[u][lane].x);
#pragma unroll
  for (int x = 0; x < 16; ++x) o[x] = 0.f;
#pragma unroll
  for (int u = 0; u < kWaves; ++u) {
    const float2 ml = sm.ml[u][lane];
    const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - m) * a.c);
    l += ml.y * f;
#pragma unroll
    for (int x = 0; x < 16; x += 4) {
      const float4 y = sm.o[u][4 * wave + x / 4][lane];
      o[x] += y.x * f;
      o[x + 1] += y.y * f;
      o[x + 2] += y.z * f;
      o[x + 3] += y.w * f;
    }
  }
  if (splits == 1) {
    store_dims(a, row, wave, hh, inverse(l), o);
    return;
  }
  float* rec = record(a, (int64_t)r * a.NKV + kvh, a.few_splits, z);
  keep_dims(rec, wave, lane, o);
  if (wave == 0) keep_sums(rec, lane, m, l);
}

// ---- longer requests ----------------------------------------------------------
// The request of the tile-th 128 rows of longer requests, and which of its own it is
// (the last ones first: they walk the most). False past the last.
__device__ __forceinline__ bool find_rows(const Args& a, int tile, int& r, int& row0) {
  const int lane = threadIdx.x & 63, G = a.NH / a.NKV;
  int before = 0;
  for (int base = 0; base < a.R; base += 64) {
    int mine = 0;
    if (base + lane < a.R) {
      const Request q = request(a, base + lane);
      if (q.n * G > a.few_rows) mine = (q.n * G + kRows - 1) / kRows;
    }
    int to = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(to, o);
      if (lane >= o) to += x;
    }
    const uint64_t hit = __ballot(before + to > tile);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      r = __builtin_amdgcn_readfirstlane(base + l);
      row0 = __builtin_amdgcn_readfirstlane((before + __shfl(to, l) - 1 - tile) * kRows);
      return true;
    }
    before += __shfl(to, 63);
  }
  return false;
}

__device__ __forceinline__ void big_unit(const Args& a, uint16_t* sm, int tile, int kvh, int z) {
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.NH / a.NKV;
  int r, row0;
  if (!find_rows(a, tile, r, row0)) return;
  const Request q = request(a, r);
  const int row1 = min(row0 + kRows, q.n * G) - 1;
  const Walk w = walk(a, q.past + row0 / G, q.past + row1 / G);
  const int splits = splits_of(w.n, a.big_per, a.big_splits);
  if (z >= splits) return;
  const int first = z * a.big_per, n_walk = (z + 1 == splits ? w.n : first + a.big_per) - first;
  v8 qv[8];
  int p;                                  // the lane's position
  {
    const Row row = row_at(a, q, kvh, row0 + 32 * wave + j);
    load_q(a, row, hh, qv);
    p = row.p;
  }
  // The unit's own rows; a spare unit repeats the last row.
  const int p0 = q.past + min(row0 + 32 * wave, q.n * G - 1) / G;
  const int p1 = q.past + min(row0 + 32 * wave + 31, q.n * G - 1) / G;
  auto tile_of = [&](int i) { return w.tile(first + min(i, n_walk - 1)); };

  // Staging: a wavefront brings half h = wave & 1 of block b = wave >> 1, of K and of V, 1
  // KiB at a time, lane l's 16 bytes to place l. K's half is the tokens of one t; those of t = 1
  // lie 128 bytes the other way, V's dims 8 .. 15 of each 16 with their halves
  // swapped: 16 lanes then read all banks, with no conflicts.
  const int b = wave >> 1, h = wave & 1;
  const uint32_t k_src = h * 2048 + (lane ^ (h << 3)) * 16;
  const uint32_t v_src = h * 2048 + (lane ^ ((lane >> 4) & 1)) * 16;
  BlockIds ids = load_ids(a, r, tile_of(lane), b);
  uint32_t ok_next = 0;                   // two bits for each tile under way, the oldest lowest
  const uint32_t lds = pdk::lds_address(sm) + (b * kBlockElems + h * 1024) * 2;
  auto fetch = [&](int slot, int i) __attribute__((always_inline)) {
    if (i && (i & 63) == 0) ids = load_ids(a, r, tile_of(i + lane), b);
    const int64_t from = ((int64_t)__builtin_amdgcn_readlane(ids.id, i & 63) * a.NKV + kvh) * kBlockElems;
    const uint32_t to = lds + slot * kTileElems * 2;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      pdk::copy16(a.k + from + 512 * x, k_src, to + 1024 * x);
      pdk::copy16(a.v + from + 512 * x, v_src, to + (kRing * kTileElems * 2 + 1024 * x));
    }
    return (uint32_t)((ids.ok[0] >> (i & 63) & 1) | (ids.ok[1] >> (i & 63) & 1) << 1);
  };
#pragma unroll
  for (int x = 0; x < kRing - 1; ++x)
    if (x < n_walk) ok_next |= fetch(x, x) << (2 * x);
#pragma unroll
  for (int x = 0; x < 8; ++x) pdk::settle(qv[x]);
  // Where this lane's operands lie in a staged tile (elements): K's at dims 16 x + 8 hh 128 x
  // on, V's dims 32 n + j of block ks 2048 ks + 512 n on.
  const int kt = (j >> 3) & 1;
  const int k_at = (j >> 4) * kBlockElems + kt * 1024 + (hh ^ kt) * 64 + (j & 7) * 8;
  const int v_at = kRing * kTileElems + j * 16 + (hh ^ kt) * 8;
  Sums sum;
  sum.clear();
  bool odd = false;
  auto load_k = [&](const uint16_t* st, v8 (&kr)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 8; ++x) kr[x] = pdk::ld16(st + k_at + 128 * x);
  };
  auto load_v = [&](const uint16_t* st, int b, v8 (&va)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < 4; ++n) va[n] = pdk::ld16(st + v_at + b * kBlockElems + n * 512);
  };
  auto step = [&](int i, const uint16_t* st, int next) __attribute__((always_inline)) {
    if (i + 1 < n_walk) pdk::copies_done<kLoads>();
    else pdk::copies_done<0>();
    const bool ok0 = ok_next & 1, ok1 = ok_next & 2;
    ok_next >>= 2;
    if (i + 2 < n_walk) ok_next |= fetch(next, i + 2) << 2;
    v8 kr[8], va[2][4];
    load_k(st, kr);
    f32x16 s = scores(kr, qv);
    __builtin_amdgcn_sched_barrier(0);                           // V into K's registers
    load_v(st, 0, va[0]);
    const int t0 = tile_of(i) * kTile;
    const Place at = place(a, t0, p, hh, ok0, ok1);
    const bool edge = hides(a, t0, p0, p1, ok0 && ok1);
    if (edge) {
#pragma unroll
      for (int x = 0; x < 16; ++x) s[x] = at.hidden(x) ? -INFINITY : s[x];
    }
    v8 wt[2];
    weigh(s, a.c, sum, wt);
    load_v(st, 1, va[1]);
    if (edge) {
      bool found = false;
#pragma unroll
      for (int x = 0; x < 8; ++x) found |= clean(va[x >> 2][x & 3]);
      odd |= __any(found);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) sum.o[x & 3] = mfma32(va[x >> 2][x & 3], wt[x >> 2], sum.o[x & 3]);
  };
  for (int i = 0, at = 0; i < n_walk; ++i) {
    const int next = at == 0 ? kRing - 1 : at - 1;               // of tile i + 2: that of tile i - 1
    step(i, sm + at * kTileElems, next);
    at = at + 1 == kRing ? 0 : at + 1;
  }
  int ln = lane;                          // the row anew: kept, it would be spilled
  asm("" : "+v"(ln));
  const Row row = row_at(a, q, kvh, row0 + 32 * wave + (ln & 31));
  if (__builtin_expect(odd, 0))
    add_cleaned(a, w, first, first + n_walk, r, kvh, row.p, p0, p1, ln, sum.o);
  const float l = swap_add(sum.l), inv = inverse(l);
  float* rec = record(a, ((int64_t)tile * a.NKV + kvh) * kWaves + wave, a.big_splits, z) + big_base(a);
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    float o[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) o[x] = sum.o[n][x];
    if (splits == 1) store_dims(a, row, n, ln >> 5, inv, o);
    else keep_dims(rec, n, ln, o);
  }
  if (splits > 1) keep_sums(rec, ln, sum.m, l);
}

__global__ __launch_bounds__(256, 2) void chunk_few_kernel(Args a) {
  __shared__ FewShared sm;
  const int rest = blockIdx.x / a.NKV;
  few_unit(a, sm, rest % a.R, blockIdx.x % a.NKV, rest / a.R);
}

__global__ __launch_bounds__(256, 3) void chunk_big_kernel(Args a) {
  __shared__ __align__(1024) uint16_t sm[2 * kRing * kTileElems];
  const int rest = blockIdx.x / a.NKV;
  big_unit(a, sm, rest % a.big_tiles, blockIdx.x % a.NKV, rest / a.big_tiles);
}

// One workgroup per unit whose context was split: wavefront n adds up dims 32 n .. of
// the splits, in order.
__global__ __launch_bounds__(256) void chunk_join_kernel(Args a, int few_units) {
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.NH / a.NKV;
  int r, row0 = 0, kvh, splits;
  const float* rec;
  Request q;
  if ((int)blockIdx.x < few_units) {
    r = blockIdx.x / a.NKV;
    kvh = blockIdx.x - r * a.NKV;
    q = request(a, r);
    if (q.n == 0 || q.n > 32 || q.n * G > a.few_rows) return;
    splits = splits_of(walk(a, q.past, q.past + q.n - 1).n, a.few_per, a.few_splits);
    rec = record(a, blockIdx.x, a.few_splits, 0);
  } else {
    const int unit = blockIdx.x - few_units, rest = unit / kWaves;
    kvh = rest % a.NKV;
    if (!find_rows(a, rest / a.NKV, r, row0)) return;
    q = request(a, r);
    const int row1 = min(row0 + kRows, q.n * G) - 1;
    splits = splits_of(walk(a, q.past + row0 / G, q.past + row1 / G).n, a.big_per, a.big_splits);
    rec = record(a, unit, a.big_splits, 0) + big_base(a);
    row0 += 32 * (unit - rest * kWaves);
    if (row0 > row1) return;
  }
  if (splits == 1) return;
  const Row row = row_at(a, q, kvh, row0 + j);
  auto sums = [&](int z) { return reinterpret_cast<const float2*>(rec + (int64_t)z * kRecord + 64 * 64)[lane]; };
  float m = -INFINITY, l = 0.f, o[16];
  for (int z = 0; z < splits; ++z) m = vmax(m, sums(z).x);
#pragma unroll
  for (int x = 0; x < 16; ++x) o[x] = 0.f;
  for (int z = 0; z < splits; ++z) {
    const float2 ml = sums(z);
    const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - m) * a.c);
    l += ml.y * f;
    const float4* p = reinterpret_cast<const float4*>(rec + (int64_t)z * kRecord) + 4 * wave * 64 + lane;
#pragma unroll
    for (int x = 0; x < 16; x += 4) {
      const float4 y = p[x / 4 * 64];
      o[x] += y.x * f;
      o[x + 1] += y.y * f;
      o[x + 2] += y.z * f;
      o[x + 3] += y.w * f;
    }
  }
  store_dims(a, row, wave, hh, inverse(l), o);
}

// How a call is split up.
struct Plan {
  bool few, big;
  int few_per, few_splits, big_per, big_splits, big_tiles;
  int64_t bytes;
};

Plan plan_for(int N, int R, int max_new, int64_t max_ctx, int NH, int NKV, int window, int sinks) {
  Plan p{};
  const int G = NH / NKV;
  p.few = max_new >= 1;
  p.big = (int64_t)max_new * G > 32;
  if (p.big && R == 1) p.few = false;
  auto tiles = [&](int64_t span) {        // walked at most by rows over `span` positions
    const int64_t all = (max_ctx + kTile - 1) / kTile;
    return (int)std::max<int64_t>(
        1, std::min<int64_t>(all, (window + span + kTile - 2) / kTile + 1 + (sinks + kTile - 1) / kTile));
  };
  auto split = [](int n, int64_t groups, int64_t wanted, int least, int& per, int& splits) {
    const int64_t want = std::min<int64_t>(kMaxSplits, std::max<int64_t>(1, wanted / std::max<int64_t>(groups, 1)));
    per = std::max<int>(least, (int)((n + want - 1) / want));
    splits = std::max(1, (n + per - 1) / per);
  };
  split(tiles(32 / G), (int64_t)R * NKV, 1024, 8, p.few_per, p.few_splits);
  const int64_t rows = (int64_t)N * G;
  p.big_tiles = (int)(rows / kRows + std::min<int64_t>(R, rows / 33 + 1));
  split(tiles(kRows / G + 1), (int64_t)std::max<int64_t>(1, rows / kRows) * NKV, 768, 8, p.big_per,
        p.big_splits);
  if (!p.few) p.few_splits = 1;
  if (!p.big) p.big_splits = 1;
  const int64_t units = (p.few_splits > 1 ? (int64_t)R * NKV * p.few_splits : 0) +
                        (p.big_splits > 1 ? (int64_t)p.big_tiles * NKV * kWaves * p.big_splits : 0);
  p.bytes = units * kRecord * 4;
  return p;
}

int check_sizes(int N, int R, int max_new, int max_ctx, int max_blocks, int n_q_heads, int n_kv_heads,
                int head_dim, int window, int sinks) {
  if (head_dim != kD) {
    pdk::set_error("the chunk kernels implement head_dim %d only (got %d)", kD, head_dim);
    return PDK_ENOTSUP;
  }
  PDK_REQUIRE(N >= 0 && N <= (1 << 20), "N must be in [0, 2^20] (got %d)", N);
  PDK_REQUIRE(R >= 1 && R <= kMaxRequests, "R must be in [1, %d] (got %d)", kMaxRequests, R);
  PDK_REQUIRE(n_kv_heads >= 1 && n_q_heads >= n_kv_heads && n_q_heads % n_kv_heads == 0 &&
                  n_q_heads / n_kv_heads <= 16 && n_q_heads <= 65535,
              "n_q_heads=%d must be 1 to 16 times n_kv_heads=%d", n_q_heads, n_kv_heads);
  PDK_REQUIRE(max_blocks >= 1 && max_blocks <= 65535, "max_blocks must be in [1, 65535] (got %d)",
              max_blocks);
  PDK_REQUIRE(max_ctx >= 1 && max_ctx <= 16 * max_blocks, "max_ctx=%d outside [1, %d]", max_ctx,
              16 * max_blocks);
  PDK_REQUIRE(max_new >= 0, "max_new must be >= 0 (got %d)", max_new);
  PDK_REQUIRE(window >= 0 && sinks >= 0 && (window || !sinks),
              "window and sinks must be >= 0, sinks with a window (got %d, %d)", window, sinks);
  return PDK_OK;
}

}  // namespace

extern "C" int64_t pdk_chunk_attn_workspace_bytes(int N, int R, int max_new, int max_ctx,
                                                  int n_q_heads, int n_kv_heads, int window,
                                                  int sinks) {
  pdk::clear_error();
  if (check_sizes(N, R, max_new, max_ctx, 65535, n_q_heads, n_kv_heads, kD, window, sinks)) return -1;
  max_new = std::min(max_new, N);
  return plan_for(N, R, max_new, max_ctx, n_q_heads, n_kv_heads, window ? window : 1 << 30,
                  std::min(sinks, 1 << 20)).bytes;
}

extern "C" int pdk_chunk_attn(const uint16_t* q, int64_t q_tok_stride, const uint16_t* cache_k,
                              const uint16_t* cache_v, int num_blocks, const int32_t* block_tables,
                              int max_blocks, const int32_t* starts, const int32_t* ctx_lens, int N,
                              int R, int max_new, int max_ctx, int n_q_heads, int n_kv_heads,
                              int head_dim, float scale, int window, int sinks, void* workspace,
                              size_t workspace_bytes, uint16_t* out, uintptr_t stream) {
  pdk::clear_error();
  if (int rc = check_sizes(N, R, max_new, max_ctx, max_blocks, n_q_heads, n_kv_heads, head_dim, window,
                           sinks))
    return rc;
  PDK_REQUIRE(num_blocks >= 1, "num_blocks must be >= 1");
  PDK_REQUIRE(scale > 0.f && scale < INFINITY, "scale must be positive and finite (got %g)",
              (double)scale);
  PDK_REQUIRE(q_tok_stride >= (int64_t)n_q_heads * kD && q_tok_stride % 8 == 0,
              "the token stride of q must be a multiple of 8 and hold the heads");
  max_new = std::min(max_new, N);
  if (max_new == 0) return PDK_OK;
  PDK_REQUIRE(q && cache_k && cache_v && block_tables && starts && ctx_lens && out,
              "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(q) && pdk::aligned16(cache_k) && pdk::aligned16(cache_v) &&
                  pdk::aligned16(out),
              "tensors must be 16-byte aligned");
  window = window ? std::min(window, 1 << 30) : 1 << 30;
  sinks = std::min(sinks, 1 << 20);
  const Plan p = plan_for(N, R, max_new, max_ctx, n_q_heads, n_kv_heads, window, sinks);
  PDK_REQUIRE(p.bytes == 0 || (workspace && pdk::aligned16(workspace)),
              "a workspace, 16-byte aligned, is needed");
  if (p.bytes > 0 && workspace_bytes < (size_t)p.bytes) {
    pdk::set_error("workspace of %zu bytes, %lld needed", workspace_bytes, (long long)p.bytes);
    return PDK_ENOMEM;
  }
  const int64_t few_blocks = (int64_t)R * n_kv_heads * p.few_splits;
  const int64_t big_blocks = (int64_t)p.big_tiles * n_kv_heads * p.big_splits;
  const int64_t big_units = p.big && p.big_splits > 1 ? (int64_t)p.big_tiles * n_kv_heads * kWaves : 0;
  const int64_t few_units = p.few && p.few_splits > 1 ? (int64_t)R * n_kv_heads : 0;
  PDK_REQUIRE(few_blocks < (1ll << 31) && big_blocks < (1ll << 31) && big_units + few_units < (1ll << 31),
              "launch too large");
  const Args a{q, q_tok_stride, cache_k, cache_v, num_blocks, block_tables, max_blocks, starts,
               ctx_lens, N, R, n_q_heads, n_kv_heads, scale * 1.4426950408889634f, window, sinks,
               static_cast<float*>(workspace), out, p.few ? 32 : 0, p.few_per, p.few_splits, p.big_per,
               p.big_splits, p.big_tiles};
  const hipStream_t st = pdk::as_stream(stream);
  if (p.big) {
    hipLaunchKernelGGL(chunk_big_kernel, dim3((unsigned)big_blocks), dim3(256), 0, st, a);
    if (int rc = pdk::check_launch("chunk_big_kernel")) return rc;
  }
  if (p.few) {
    hipLaunchKernelGGL(chunk_few_kernel, dim3((unsigned)few_blocks), dim3(256), 0, st, a);
    if (int rc = pdk::check_launch("chunk_few_kernel")) return rc;
  }
  if (few_units + big_units) {
    hipLaunchKernelGGL(chunk_join_kernel, dim3((unsigned)(few_units + big_units)), dim3(256), 0, st, a,
                       (int)few_units);
    if (int rc = pdk::check_launch("chunk_join_kernel")) return rc;
  }
  return PDK_OK;
}
