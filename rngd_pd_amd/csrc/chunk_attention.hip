// Causal GQA attention of several requests' new tokens over the paged cache, gfx950,
// head_dim 128: new token i of request r stands at position p = ctx_r - n_r + i and sees
// the cached tokens t <= p (its own among them), under a window t > p - window or t <
// sinks. Tokens of blocks that the table does not name are seen by nobody; a token
// that sees nothing gets zeros.
//
// Rows are the query heads that share a KV head, token after token (row = token * G + head
// of the group), so that a few tokens' heads fill a tile and read each key and value
// once. S^T = K Q^T, so that a lane holds one row: maximum, sum and rescale are per lane,
// with an exchange or two. The tokens of a tile are taken in an order that makes the
// accumulators of S^T, as they lie, the B operand of O^T += V^T P^T, and the cache's own
// order is that of both A operands: 8 tokens of a K block at one group of 8 dims are 128
// consecutive bytes, V's rows of 16 tokens 32. Scores, maxima, sums and O are fp32; a
// weight is rounded to bf16 once, for the product with V (half a step, 2^-8 of each weight: a
// share of 2^-8 / sqrt(3) rms beside the output's own rounding).
//
// Requests of few rows (16, or 32 where no request has more: single tokens, drafts) are
// bound by HBM: v_mfma_f32_16x16x32_bf16 on 32 tokens by 16 rows, a workgroup's four
// wavefronts take every fourth tile of a split with operands straight from memory in
// registers, the next tile's under way, and add up in LDS. 32 to 64 single tokens on
// thousands: 5.5 to 5.9 TB/s, 32 drafts of 5 6.4 TB/s; 8 drafts are 22 us, of which 12 are the
// bytes, the rest two starts and the join.
//
// Longer ones are bound by the wavefronts' issue (matrix and vector instructions; a loop
// without the exponentials is 6 % faster, one without copies 11, one without the product with
// V 21): a workgroup takes 128 rows, its four wavefronts (v_mfma_f32_32x32x16_bf16, 32
// rows each) share tiles of 32 tokens staged into LDS two ahead by copies that pass no
// register, one barrier per tile, three workgroups on a CU. 4096 tokens on 28000: 1750 to
// 1850 us, 1090 to 1150 TFLOP/s, where library products of 8192^3 have 1290 to 1555.
// With two wavefronts per SIMD and the next scores under the weights it was 2026 to 2107.
//
// Contexts are split over workgroups where those are few; a second launch joins the splits
// in a fixed order. One request's split is shared by three teams of four wavefronts in a
// workgroup, which add up in LDS (256 tokens on 3500: 34.8 us, by workgroups alone 40.6). Both
// kinds of request together take one launch.
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
typedef float f32x4 __attribute__((__vector_size__(16)));

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
constexpr int kLeastSplit = 8;            // tiles of a split at least
constexpr int kCUs = 256;
constexpr int kMostRecords = 4096;        // of four units each, of longer requests: 277 MB
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
  // Rows up to which a request has few (16 or 32, or 0 where all are taken as longer
  // ones), tiles of a split and splits at most of those; of the longer ones, workgroups
  // that run at once and splits of what they leave over.
  int few_rows, few_per, few_splits, big_slots, big_splits;
  int big_over;                           // workgroups' rows left over that there are records for
  int64_t big_base;                       // floats of the workspace before the longer ones' records
};

__device__ __forceinline__ f32x16 mfma32(const v8& a, const v8& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16(const v8& a, const v8& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ float swap_add(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A request's new tokens as far as q has rows for them: n of them from row `start` on, the
// first at position `past`. The others count for the positions all the same: token i of the
// whole request stands at ctx - (e - s) + i, cut off or not.
struct Request {
  int start, n, past;
};

__device__ __forceinline__ Request request(const Args& a, int r) {
  Request q;
  q.start = min(max(a.starts[r], 0), a.N);
  const int e = min(max(a.starts[r + 1], q.start), 1 << 30);
  q.n = min(e, a.N) - q.start;
  q.past = min(max(a.ctx[r], 0), 1 << 30) - (e - q.start);
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
  const int id = a.tables[(int64_t)r * a.W + min(max(e, 0), a.W - 1)];
  return e >= 0 && e < a.W && id >= 0 && id < a.num_blocks ? id : -1;
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

// A lane holds row j = lane & 31 and 16 of a tile's 32 scores. Row r of S^T's tile is token
// pi(r), pi swapping bits 2 and 3: accumulators 8 ks .. 8 ks + 7 are then tokens 16 ks + 8
// (lane >> 5) + 0..7.
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

__device__ __forceinline__ uint32_t mark_of(uint32_t u) {
  return (u & 0x7f80u) != 0x7f80u ? 0u : u == 0x7f80u ? 0x3f80u : u == 0xff80u ? 0x4280u : 0x4580u;
}

// What a mark's count comes to: infinities and NaN to add.
__device__ __forceinline__ float found_value(float found) {
  const uint32_t u = (uint32_t)found;
  float add = u & 63 ? INFINITY : 0.f;
  add = u & 0xfc0 ? add - INFINITY : add;
  return u >> 12 ? __builtin_nanf("") : add;
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
          mark.w[x] = mark_of(v.w[x] & 0xffffu) | mark_of(v.w[x] >> 16) << 16;
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
__device__ __forceinline__ void keep_dims(float* rec, int n, int lane, bool mine, const float (&o)[16]) {
  if (!mine) return;                      // few rows: little to store and to join
  float4* p = reinterpret_cast<float4*>(rec) + 4 * n * 64 + lane;
#pragma unroll
  for (int x = 0; x < 16; x += 4) p[x / 4 * 64] = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
}

__device__ __forceinline__ void keep_sums(float* rec, int lane, float m, float l) {
  reinterpret_cast<float2*>(rec + 64 * 64)[lane] = make_float2(m, l);
}

// ---- requests of few rows -----------------------------------------------------
// Up to kSets x 16 rows; a lane's row of a set is i = lane & 15, and of 32 tokens it holds
// 8 kg .. 8 kg + 7, kg = lane >> 4: S^T's tile u (v_mfma_f32_16x16x32_bf16) has token 8
// (r / 4) + 4 u + r % 4 in row r, so that its accumulators are 4 kg + 0..3 of both tiles,
// which are the B operand of O^T.
template <int kSets>
struct FewSums {
  float m[kSets], l[kSets];
  f32x4 o[kSets][8];                      // dims 16 n + 4 kg + 0..3
};

template <int kSets>
struct FewShared {
  f32x4 o[kWaves][kSets * 8][64];
  float2 ml[kWaves][kSets][64];
};

template <int kSets>
constexpr int kFewRecord = kSets * (8 * 64 * 4 + 64 * 2);        // floats

// The largest, or the sum, over the four lanes that have a row.
__device__ __forceinline__ float row_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float row_sum(float x) {
  x = swap_add(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// add_cleaned for one tile and these rows.
template <int kSets>
__device__ __forceinline__ void few_cleaned(const Args& a, int t0, int r, int kvh, const int (&p)[kSets],
                                            int p0, int p1, int lane, f32x4 (&o)[kSets][8]) {
  const int i = lane & 15, kg = lane >> 4;
  const int id[2] = {block_id(a, r, t0 / 16), block_id(a, r, t0 / 16 + 1)};
  if (!hides(a, t0, p0, p1, id[0] >= 0 && id[1] >= 0)) return;
  const int mine = kg >> 1 ? id[1] : id[0];
  const uint16_t* v = a.v + ((int64_t)max(mine, 0) * a.NKV + kvh) * kBlockElems + i * 16 + (kg & 1) * 8;
  v8 seen[kSets];
#pragma unroll
  for (int c = 0; c < kSets; ++c)
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int t = t0 + 8 * kg + x;
      const bool hid = t > p[c] || (p[c] - t >= a.window && t >= a.sinks) || mine < 0;
      const uint32_t one = hid ? 0u : 0x3f80u;
      seen[c].w[x >> 1] = x & 1 ? seen[c].w[x >> 1] | one << 16 : one;
    }
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const v8 x = pdk::ld16(v + 256 * n);
    v8 mark;
#pragma unroll
    for (int w = 0; w < 4; ++w) mark.w[w] = mine < 0 ? 0u : mark_of(x.w[w] & 0xffffu) | mark_of(x.w[w] >> 16) << 16;
#pragma unroll
    for (int c = 0; c < kSets; ++c) {
      const f32x4 found = mfma16(mark, seen[c], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int e = 0; e < 4; ++e) o[c][n][e] += found_value(found[e]);
    }
  }
}

__device__ __forceinline__ void store_four(const Args& a, const Row& r, int dim, float inv, const f32x4& o) {
  if (r.mine)
    *reinterpret_cast<uint2*>(a.out + ((int64_t)r.token * a.NH + r.head) * kD + dim) =
        make_uint2(pdk::pack_bf16x2_rne(o[0] * inv, o[1] * inv), pdk::pack_bf16x2_rne(o[2] * inv, o[3] * inv));
}

// The four wavefronts' sums of set c added up, dims 32 wave .. by each wavefront.
template <int kSlots, int kSets, class F>
__device__ __forceinline__ void few_out(const Args& a, const f32x4 (&so)[kWaves][kSlots][64],
                                        const float2 (&sml)[kWaves][kSets][64], int c, int wave,
                                        int lane, F use) {
  float m = -INFINITY, l = 0.f;
  f32x4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
  for (int u = 0; u < kWaves; ++u) m = vmax(m, sml[u][c][lane].x);
#pragma unroll
  for (int u = 0; u < kWaves; ++u) {
    const float2 ml = sml[u][c][lane];
    const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - m) * a.c);
    l += ml.y * f;
#pragma unroll
    for (int n = 0; n < 2; ++n) o[n] += so[u][8 * c + 2 * wave + n][lane] * f;
  }
  use(m, l, o);
}

template <int kSets>
__device__ __forceinline__ void few_unit(const Args& a, FewShared<kSets>& sm, int r, int kvh, int z) {
  const int lane = threadIdx.x & 63, i = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.NH / a.NKV;
  const Request q = request(a, r);
  if (q.n == 0 || q.n > a.few_rows || q.n * G > a.few_rows) return;
  const int p0 = q.past, p1 = q.past + q.n - 1;
  const Walk w = walk(a, p0, p1);
  const int splits = splits_of(w.n, a.few_per, a.few_splits);
  if (z >= splits) return;
  const int first = z * a.few_per, end = z + 1 == splits ? w.n : first + a.few_per;
  int p[kSets];
  FewSums<kSets> sum;
#pragma unroll
  for (int c = 0; c < kSets; ++c) {
    sum.m[c] = -INFINITY;
    sum.l[c] = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) sum.o[c][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int n_own = (end - first - wave + kWaves - 1) / kWaves;
  bool odd = false;
  if (n_own > 0) {
    auto tile_of = [&](int x) { return w.tile(first + wave + kWaves * min(x, n_own - 1)); };
    BlockIds ids[2]{};                    // of both blocks
    uint64_t ok_was[2] = {0, 0};          // of the 64 tiles before
    auto next_ids = [&](int x) __attribute__((always_inline)) {
      ok_was[0] = ids[0].ok[0];
      ok_was[1] = ids[0].ok[1];
#pragma unroll
      for (int b = 0; b < 2; ++b) ids[b] = load_ids(a, r, tile_of(x + lane), b);
    };
    next_ids(0);
    int ids_from = 0;
    auto ok_of = [&](int x, int b) { return (x < ids_from ? ok_was[b] : ids[0].ok[b]) >> (x & 63) & 1; };
    v8 qv[kSets][4];
#pragma unroll
    for (int c = 0; c < kSets; ++c) {
      const Row row = row_at(a, q, kvh, 16 * c + i);
      const uint16_t* from = a.q + (int64_t)row.token * a.q_ld + row.head * kD + 8 * kg;
      p[c] = row.p;
#pragma unroll
      for (int x = 0; x < 4; ++x) qv[c][x] = pdk::ld16(from + 32 * x);
    }
    // Where a lane's operands lie in a tile (elements): K's tokens of tile u at dims 32 x + 8 kg
    // are 1024 u + 256 x on, in the block of token 8 (i / 4); V's dims 16 n + i 256 n on, in
    // the block of token 8 kg.
    const int k_at = kg * 64 + (i & 7) * 8, v_at = i * 16 + (kg & 1) * 8;
    auto block = [&](int x, int b) {
      const int id = __builtin_amdgcn_readlane(ids[b].id, x & 63);
      return ((int64_t)id * a.NKV + kvh) * kBlockElems;
    };
    // Tile x's loads, or past the last as many of one 16-byte piece each: no load is under a
    // branch that would make the compiler wait for all of them.
    v8 k[2][4], v[8];
    auto load_k = [&](int x) __attribute__((always_inline)) {
      const int64_t b0 = block(x, 0), b1 = block(x, 1);
      const uint16_t* from = a.k + (x >= n_own ? 0 : (i & 8 ? b1 : b0) + k_at);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < 4; ++d) k[u][d] = pdk::ld16(from + 1024 * u + 256 * d);
    };
    auto load_v = [&](int x) __attribute__((always_inline)) {
      const int64_t b0 = block(x, 0), b1 = block(x, 1);
      const uint16_t* from = a.v + (x >= n_own ? 0 : (kg & 2 ? b1 : b0) + v_at);
#pragma unroll
      for (int n = 0; n < 8; ++n) v[n] = pdk::ld16_stream(from + 256 * n);
    };
    load_k(0);
    load_v(0);
    // A tile's registers take the next one's K after the scores, its V after the products.
#pragma unroll 1
    for (int x = 0; x < n_own; ++x) {
      if ((x & 63) == 63) next_ids(ids_from = x + 1);
      const bool ok0 = ok_of(x, 0), ok1 = ok_of(x, 1);
      const int t0 = tile_of(x) * kTile;
      f32x4 s[kSets][2];
#pragma unroll
      for (int c = 0; c < kSets; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[c][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int d = 0; d < 4; ++d) s[c][u] = mfma16(k[u][d], qv[c][d], s[c][u]);
        }
      load_k(x + 1);
      const bool edge = hides(a, t0, p0, p1, ok0 && ok1);
      if (edge) {
        const bool ok = kg & 2 ? ok1 : ok0;
#pragma unroll
        for (int c = 0; c < kSets; ++c) {
          const int ago = p[c] - t0 - 8 * kg, sink = a.sinks - t0 - 8 * kg;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int at = 4 * u + e;
              const bool hid = (at > ago) | ((ago - at >= a.window) & (at >= sink)) | !ok;
              s[c][u][e] = hid ? -INFINITY : s[c][u][e];
            }
        }
      }
      v8 wt[kSets];
#pragma unroll
      for (int c = 0; c < kSets; ++c) {
        float mx = s[c][0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = vmax(mx, s[c][e >> 2][e & 3]);
        mx = row_max(mx);
        // The maximum in use follows only when it falls more than 2^8 behind, as in weigh.
        if (__any((mx - sum.m[c]) * a.c > 8.f)) {
          const float m_new = vmax(sum.m[c], mx);
          const float f = sum.m[c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((sum.m[c] - m_new) * a.c);
          sum.m[c] = m_new;
          sum.l[c] *= f;
#pragma unroll
          for (int n = 0; n < 8; ++n) sum.o[c][n] *= f;
        }
        const float mc = sum.m[c] == -INFINITY ? 0.f : sum.m[c] * a.c;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float u = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][e >> 2][e & 3], a.c, -mc));
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][e >> 2][(e & 3) + 1], a.c, -mc));
          sum.l[c] += u + y;
          wt[c].w[e >> 1] = pdk::pack_bf16x2_rne(u, y);
        }
      }
      if (edge) {
        bool found = false;
#pragma unroll
        for (int n = 0; n < 8; ++n) found |= clean(v[n]);
        odd |= __any(found);
      }
#pragma unroll
      for (int c = 0; c < kSets; ++c)
#pragma unroll
        for (int n = 0; n < 8; ++n) sum.o[c][n] = mfma16(v[n], wt[c], sum.o[c][n]);
      load_v(x + 1);
    }
  }
  // The wavefront's own tiles alone are its sums', any of which may be added to.
  if (__builtin_expect(odd, 0))
    for (int x = first + wave; x < end; x += kWaves)
      few_cleaned<kSets>(a, w.tile(x) * kTile, r, kvh, p, p0, p1, lane, sum.o);
  // Wavefront n adds up dims 32 n .. of the four.
#pragma unroll
  for (int c = 0; c < kSets; ++c) {
#pragma unroll
    for (int n = 0; n < 8; ++n) sm.o[wave][8 * c + n][lane] = sum.o[c][n];
    sm.ml[wave][c][lane] = make_float2(sum.m[c], row_sum(sum.l[c]));
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < kSets; ++c) {
    const Row row = row_at(a, q, kvh, 16 * c + i);
    few_out(a, sm.o, sm.ml, c, wave, lane, [&](float m, float l, const f32x4 (&o)[2]) {
      if (splits == 1) {
        const float inv = inverse(l);
#pragma unroll
        for (int n = 0; n < 2; ++n) store_four(a, row, 16 * (2 * wave + n) + 4 * kg, inv, o[n]);
      } else if (row.mine) {              // few rows: little to store and to join
        float* rec = a.ws + (((int64_t)r * a.NKV + kvh) * a.few_splits + z) * kFewRecord<kSets>;
#pragma unroll
        for (int n = 0; n < 2; ++n) reinterpret_cast<f32x4*>(rec)[(8 * c + 2 * wave + n) * 64 + lane] = o[n];
        if (wave == 0) reinterpret_cast<float2*>(rec + kSets * 2048)[c * 64 + lane] = make_float2(m, l);
      }
    });
  }
}

// A split request's sums: wavefront w adds up splits w, w + 4, ..., four of them in one
// round of loads, then the four's are added in LDS.
template <int kSets>
__device__ __forceinline__ void few_join(const Args& a, FewShared<1>& sm, int r, int kvh) {
  const int lane = threadIdx.x & 63, i = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.NH / a.NKV;
  const Request q = request(a, r);
  if (q.n == 0 || q.n > a.few_rows || q.n * G > a.few_rows) return;
  const int splits = splits_of(walk(a, q.past, q.past + q.n - 1).n, a.few_per, a.few_splits);
  if (splits == 1) return;
  const float* rec = a.ws + ((int64_t)r * a.NKV + kvh) * a.few_splits * kFewRecord<kSets>;
#pragma unroll
  for (int c = 0; c < kSets; ++c) {
    const Row row = row_at(a, q, kvh, 16 * c + i);
    float m = -INFINITY, l = 0.f;
    f32x4 o[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (row.mine)
      for (int z0 = wave; z0 < splits; z0 += 16) {
        float2 ml[4];
        f32x4 y[4][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float* at = rec + (int64_t)min(z0 + 4 * k, splits - 1) * kFewRecord<kSets>;
          ml[k] = reinterpret_cast<const float2*>(at + kSets * 2048)[c * 64 + lane];
          if (z0 + 4 * k >= splits) ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
          for (int n = 0; n < 8; ++n) y[k][n] = reinterpret_cast<const f32x4*>(at)[(8 * c + n) * 64 + lane];
        }
        const float m_new = vmax(m, vmax(vmax(ml[0].x, ml[1].x), vmax(ml[2].x, ml[3].x)));
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * a.c);
        m = m_new;
        l *= f;
#pragma unroll
        for (int n = 0; n < 8; ++n) o[n] *= f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (z0 + 4 * k >= splits) break;
          const float g = ml[k].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[k].x - m) * a.c);
          l += ml[k].y * g;
#pragma unroll
          for (int n = 0; n < 8; ++n) o[n] += y[k][n] * g;
        }
      }
    if (c) __syncthreads();
#pragma unroll
    for (int n = 0; n < 8; ++n) sm.o[wave][n][lane] = o[n];
    sm.ml[wave][0][lane] = make_float2(m, l);
    __syncthreads();
    few_out(a, sm.o, sm.ml, 0, wave, lane, [&](float, float l, const f32x4 (&o)[2]) {
      const float inv = inverse(l);
#pragma unroll
      for (int n = 0; n < 2; ++n) store_four(a, row, 16 * (2 * wave + n) + 4 * kg, inv, o[n]);
    });
  }
}

// ---- longer requests ----------------------------------------------------------
// How many workgroups' rows (128 each) 64 requests from `base` on have, up to lane's.
__device__ __forceinline__ int rows_up_to(const Args& a, int base, int lane) {
  const int G = a.NH / a.NKV;
  int n = 0;
  if (base + lane < a.R) {
    const Request q = request(a, base + lane);
    if (q.n * G > a.few_rows) n = (q.n * G + kRows - 1) / kRows;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(n, o);
    if (lane >= o) n += x;
  }
  return n;
}

// A longer request's workgroup: 128 rows from row0 on of request r, split z of them.
// Whole rounds of big_slots workgroups walk their contexts whole; the workgroups' rows
// that are left over, fewer than would fill the card, are split (none are where they are
// more than the host could count on: one request with far fewer tokens than q has rows).
struct Big {
  int r, row0;
  int left;                               // number among those left over, or -1
  int z;
};

// Of the rest-th workgroup of a KV head, or (kLeft) the first split of the rest-th of its
// rows that are left over; false past the last.
template <bool kLeft>
__device__ __forceinline__ bool find_big(const Args& a, int rest, Big& w) {
  const int lane = threadIdx.x & 63;
  int all = 0, to = 0;
  if (a.R == 1) {
    all = (request(a, 0).n * (a.NH / a.NKV) + kRows - 1) / kRows;
  } else {
    for (int base = 0; base < a.R; base += 64) {
      to = rows_up_to(a, base, lane);
      all += __shfl(to, 63);
    }
    all = __builtin_amdgcn_readfirstlane(all);
  }
  int whole = (int)((int64_t)all * a.NKV / a.big_slots * a.big_slots / a.NKV);
  if (all - whole > a.big_over) whole = all;                     // more than there are records for
  const int left = all - whole;
  if (kLeft) {
    if (rest >= left) return false;
    rest += whole;
  }
  int tile = rest;
  w.left = -1;
  w.z = 0;
  if (rest >= whole) {
    if (left == 0) return false;
    w.z = (rest - whole) / left;
    w.left = rest - whole - w.z * left;
    tile = whole + w.left;
    if (w.z >= a.big_splits) return false;
  }
  if (a.R == 1) {
    w.r = 0;
    w.row0 = (all - 1 - tile) * kRows;    // the last rows first: they walk the most
    return tile < all;
  }
  int before = 0;
  for (int base = 0; base < a.R; base += 64) {
    if (a.R > 64) to = rows_up_to(a, base, lane);
    const uint64_t hit = __ballot(before + to > tile);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      w.r = __builtin_amdgcn_readfirstlane(base + l);
      w.row0 = __builtin_amdgcn_readfirstlane((before + __shfl(to, l) - 1 - tile) * kRows);
      return true;
    }
    before += __shfl(to, 63);
  }
  return false;
}

// The tiles of a split of a walk of n, of a longer request left over.
__device__ __forceinline__ int big_per(const Args& a, int n) {
  return max((n + a.big_splits - 1) / a.big_splits, kLeastSplit);
}

// kTeams times four wavefronts share the tiles of a split, each four with a ring of
// their own.
template <int kTeams>
__device__ __forceinline__ void big_unit(const Args& a, uint16_t* shared, int rest, int kvh) {
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int number = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = number % kWaves, team = number / kWaves;
  uint16_t* const sm = shared + team * 2 * kRing * kTileElems;
  const int G = a.NH / a.NKV;
  Big wg;
  if (!find_big<false>(a, rest, wg)) return;
  const int r = wg.r, row0 = wg.row0;
  const Request q = request(a, r);
  const int row1 = min(row0 + kRows, q.n * G) - 1;
  const Walk w = walk(a, q.past + row0 / G, q.past + row1 / G);
  const int per = wg.left < 0 ? w.n : big_per(a, w.n);
  const int splits = wg.left < 0 ? 1 : splits_of(w.n, per, a.big_splits);
  if (wg.z >= splits) return;
  // The team's tiles of the split's, at most n_most.
  const int n_split = (wg.z + 1 == splits ? w.n : (wg.z + 1) * per) - wg.z * per;
  const int n_most = (n_split + kTeams - 1) / kTeams;
  const int first = wg.z * per + team * n_most, n_walk = min(n_most, n_split - team * n_most);
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
    v8 kr[8], va[2][4];
    load_k(st, kr);
    // Scores before weights before the products with V, of the wavefronts that share a SIMD
    // (4096 tokens on 28000 1891 us without, 1800 so; 6000 from the first on 305 and 282, 4000
    // 147 and 153).
    __builtin_amdgcn_s_setprio(2);
    f32x16 s = scores(kr, qv);
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);                           // V into K's registers
    if (i + 2 < n_walk) ok_next |= fetch(next, i + 2) << 2;
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
    __builtin_amdgcn_s_setprio(0);
    if (edge) {
      bool found = false;
#pragma unroll
      for (int x = 0; x < 8; ++x) found |= clean(va[x >> 2][x & 3]);
      odd |= __any(found);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) sum.o[x & 3] = mfma32(va[x >> 2][x & 3], wt[x >> 2], sum.o[x & 3]);
  };
  for (int i = 0, at = 0; i < n_most; ++i) {
    const int next = at == 0 ? kRing - 1 : at - 1;               // of tile i + 2: that of tile i - 1
    if (kTeams == 1 || i < n_walk) step(i, sm + at * kTileElems, next);
    else pdk::copies_done<0>();                                  // the others' barrier
    at = at + 1 == kRing ? 0 : at + 1;
  }
  int ln = lane;                          // the row anew: kept, it would be spilled
  asm("" : "+v"(ln));
  if (__builtin_expect(odd, 0)) {
    const Row row = row_at(a, q, kvh, row0 + 32 * wave + (ln & 31));
    add_cleaned(a, w, first, first + n_walk, r, kvh, row.p, p0, p1, ln, sum.o);
  }
  float4* const so = reinterpret_cast<float4*>(shared);
  float share[kTeams];
  if constexpr (kTeams > 1) {
    // The other teams' sums by LDS, where the tiles were, the m and l of a lane last.
    float2* const sml = reinterpret_cast<float2*>(shared) + (kTeams - 1) * kWaves * 64 * 32;
    __syncthreads();
    if (team > 0) {
      const int to = (team - 1) * kWaves + wave;
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int x = 0; x < 16; x += 4)
          so[(to * 16 + 4 * n + x / 4) * 64 + ln] =
              make_float4(sum.o[n][x], sum.o[n][x + 1], sum.o[n][x + 2], sum.o[n][x + 3]);
      sml[to * 64 + ln] = make_float2(sum.m, sum.l);
    }
    __syncthreads();
    if (team > 0) return;
    float m = sum.m;
    float2 ml[kTeams - 1];
#pragma unroll
    for (int t = 0; t < kTeams - 1; ++t) {
      ml[t] = sml[(t * kWaves + wave) * 64 + ln];
      m = vmax(m, ml[t].x);
    }
    share[0] = sum.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((sum.m - m) * a.c);
    sum.m = m;
    sum.l *= share[0];
#pragma unroll
    for (int t = 0; t < kTeams - 1; ++t) {
      share[t + 1] = ml[t].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[t].x - m) * a.c);
      sum.l += ml[t].y * share[t + 1];
    }
  }
  asm("" : "+v"(ln));
  const Row row = row_at(a, q, kvh, row0 + 32 * wave + (ln & 31));
  const float l = swap_add(sum.l), inv = inverse(l);
  float* rec = a.ws + a.big_base + ((((int64_t)wg.left * a.NKV + kvh) * kWaves + wave) * a.big_splits + wg.z) * kRecord;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    float o[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) o[x] = kTeams == 1 ? sum.o[n][x] : sum.o[n][x] * share[0];
#pragma unroll
    for (int t = 1; t < kTeams; ++t)
#pragma unroll
      for (int x = 0; x < 16; x += 4) {
        const float4 y = so[(((t - 1) * kWaves + wave) * 16 + 4 * n + x / 4) * 64 + ln];
        o[x] += y.x * share[t];
        o[x + 1] += y.y * share[t];
        o[x + 2] += y.z * share[t];
        o[x + 3] += y.w * share[t];
      }
    if (splits == 1) store_dims(a, row, n, ln >> 5, inv, o);
    else keep_dims(rec, n, ln, row.mine, o);
  }
  if (splits > 1) keep_sums(rec, ln, sum.m, l);
}

template <int kSets>
__global__ __launch_bounds__(256, kSets == 1 ? 3 : 2) void chunk_few_kernel(Args a) {
  __shared__ FewShared<kSets> sm;
  const int rest = blockIdx.x / a.NKV;
  few_unit<kSets>(a, sm, rest % a.R, blockIdx.x % a.NKV, rest / a.R);
}

template <int kTeams>
__global__ __launch_bounds__(256 * kTeams, 3) void chunk_big_kernel(Args a) {
  __shared__ __align__(1024) uint16_t sm[kTeams * 2 * kRing * kTileElems];
  big_unit<kTeams>(a, sm, blockIdx.x / a.NKV, blockIdx.x % a.NKV);
}

// Requests of both kinds: a workgroup for each CU of the one kind, then of the other, as
// long as both last, so that those that wait for memory and those that multiply share
// the CUs (2000 new tokens beside 31 single ones: 213 us; with 128 in turn 7 % more). Few
// rows first, their walks are the longest (224 us the other way round).
__global__ __launch_bounds__(256, 3) void chunk_both_kernel(Args a, int few, int big) {
  constexpr int kTiles = 2 * kRing * kTileElems * sizeof(uint16_t);
  __shared__ __align__(1024) char sm[std::max(kTiles, (int)sizeof(FewShared<1>))];
  const int g = blockIdx.x / kCUs, turns = min((few + kCUs - 1) / kCUs, (big + kCUs - 1) / kCUs);
  const bool is_big = g < 2 * turns ? g & 1 : big > few;
  const int u = (g < 2 * turns ? g >> 1 : g - turns) * kCUs + blockIdx.x % kCUs;
  if (u >= (is_big ? big : few)) return;
  const int rest = u / a.NKV, kvh = u - rest * a.NKV;
  if (is_big) big_unit<1>(a, reinterpret_cast<uint16_t*>(sm), rest, kvh);
  else few_unit<1>(a, *reinterpret_cast<FewShared<1>*>(sm), rest % a.R, kvh, rest / a.R);
}

// One workgroup per unit whose context was split: wavefront n adds up dims 32 n .. of
// the splits, in order.
template <int kSets>
__global__ __launch_bounds__(256) void chunk_join_kernel(Args a, int few_units) {
  if ((int)blockIdx.x < few_units) {
    __shared__ FewShared<1> sm;
    const int r = blockIdx.x / a.NKV;
    few_join<kSets>(a, sm, r, blockIdx.x - r * a.NKV);
    return;
  }
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.NH / a.NKV;
  const int unit = blockIdx.x - few_units, at = unit / kWaves, left = at / a.NKV, kvh = at - left * a.NKV;
  const float* rec = a.ws + a.big_base + (int64_t)unit * a.big_splits * kRecord;
  // Four splits' loads at a time, the last one again past the end. One request's first four
  // wait for nothing that says how many there are; of several requests fewer rows may be
  // left over than there are records for.
  float2 ml[4];
  float4 y[4][4];
  auto load = [&](int z) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* from = rec + (int64_t)min(z + i, a.big_splits - 1) * kRecord;
      ml[i] = reinterpret_cast<const float2*>(from + 64 * 64)[lane];
#pragma unroll
      for (int x = 0; x < 4; ++x) y[i][x] = reinterpret_cast<const float4*>(from)[(4 * wave + x) * 64 + lane];
    }
  };
  if (a.R == 1) load(0);
  Big wg;
  if (!find_big<true>(a, left, wg)) return;
  const Request q = request(a, wg.r);
  const int row1 = min(wg.row0 + kRows, q.n * G) - 1, row0 = wg.row0 + 32 * (unit - at * kWaves);
  const Walk w = walk(a, q.past + wg.row0 / G, q.past + row1 / G);
  const int splits = splits_of(w.n, big_per(a, w.n), a.big_splits);
  if (row0 > row1) return;
  if (splits == 1) return;
  const Row row = row_at(a, q, kvh, row0 + j);
  if (!row.mine) return;                  // both lanes of a row alike
  float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
  for (int x = 0; x < 16; ++x) o[x] = 0.f;
  for (int z = 0; z < splits; z += 4) {
    if (z || a.R > 1) load(z);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (z + i >= splits) ml[i].x = -INFINITY;
    const float m_new = vmax(m, vmax(vmax(ml[0].x, ml[1].x), vmax(ml[2].x, ml[3].x)));
    const float g = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * a.c);
    m = m_new;
    l *= g;
#pragma unroll
    for (int x = 0; x < 16; ++x) o[x] *= g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (z + i >= splits) break;
      const float f = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[i].x - m) * a.c);
      l += ml[i].y * f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        o[4 * x] += y[i][x].x * f;
        o[4 * x + 1] += y[i][x].y * f;
        o[4 * x + 2] += y[i][x].z * f;
        o[4 * x + 3] += y[i][x].w * f;
      }
    }
  }
  store_dims(a, row, wave, hh, inverse(l), o);
}

// How a call is split up.
struct Plan {
  bool big, teams;
  int few_rows;                           // 0 where no request is taken as one of few rows
  int few_per, few_splits, big_slots, big_splits, big_over;
  int64_t few_blocks, big_blocks;         // workgroups
  int64_t few_units, big_units;           // units that may be split
  int64_t few_floats;                     // of the former's records
  int64_t bytes;
};

// How long n equal workgroups per CU take, three at once, in the time that one of three
// takes: one alone has 0.78 of the three's rate (4096 tokens after 28000: 588 us of 256
// beside 1374 of 768), two 0.93.
double rounds(int64_t n) {
  return (double)(n / 3 * 3) + (n % 3 == 0 ? 0. : n % 3 == 1 ? 1 / 0.78 : 2 / 0.93);
}

Plan plan_for(int N, int R, int max_new, int64_t max_ctx, int NH, int NKV, int window, int sinks) {
  Plan p{};
  const int G = NH / NKV;
  p.big = (int64_t)max_new * G > 32;
  p.few_rows = p.big ? (R == 1 ? 0 : 16) : max_new * G > 16 ? 32 : 16;
  auto tiles = [&](int64_t span) {        // walked at most by rows over `span` positions
    const int64_t all = (max_ctx + kTile - 1) / kTile;
    return (int)std::max<int64_t>(
        1, std::min<int64_t>(all, (window + span + kTile - 2) / kTile + 1 + (sinks + kTile - 1) / kTile));
  };
  p.few_splits = p.big_splits = 1;
  p.few_per = 1 << 30;
  p.big_slots = 3 * kCUs;
  if (p.few_rows) {
    const int n = tiles(p.few_rows / G);
    const int64_t groups = (int64_t)R * NKV;
    const int64_t want = std::min<int64_t>(kMaxSplits, std::max<int64_t>(1, (p.few_rows == 32 ? 1 : 3) * kCUs / groups));
    p.few_per = std::max<int>(kLeastSplit, (int)((n + want - 1) / want));
    p.few_splits = (n + p.few_per - 1) / p.few_per;
    p.few_blocks = groups * p.few_splits;
    if (p.few_splits > 1) p.few_units = groups;
  }
  if (p.big) {
    const int64_t rows = (int64_t)N * G, n = tiles(kRows / G + 1);
    const int64_t all = (rows + kRows - 1) / kRows;              // if they were one request's
    const int64_t most = R == 1 ? all : rows / kRows + std::min<int64_t>(R, rows / (p.few_rows + 1) + 1);
    const int64_t left = std::max<int64_t>(1, all * NKV % p.big_slots);
    // Left over at most: known of one request, of several up to a whole round.
    const int64_t over = R == 1 ? all - all * NKV / p.big_slots * p.big_slots / NKV
                                : std::min<int64_t>(most, p.big_slots / NKV + 1);
    // The split that ends soonest of the workgroups left over; each costs as much again as
    // ten tiles for its start, for handing over its sums (136 KB) and for the join. At most
    // kMostRecords of them; beside those of few rows, 768 of 9 KB, the workspace is 284 MB at most.
    double best = 1e30;
    for (int s = 1; s <= kMaxSplits && (s == 1 || (n / s >= kLeastSplit && s * over * NKV <= kMostRecords)); ++s) {
      const double t = rounds((left * s + kCUs - 1) / kCUs) * ((double)n / s + (s > 1 ? 10 : 0));
      // One request with less than a round of them: three teams a workgroup, one on a CU.
      // Their common barrier costs some 5 %, a start and the teams' sums as much as 6 tiles.
      const double teams = (left * s + kCUs - 1) / kCUs * ((double)n / s + (s > 1 ? 16 : 6)) * 1.05;
      if (t < best) {
        best = t;
        p.big_splits = s;
        p.teams = false;
      }
      if (R == 1 && all * NKV < p.big_slots && teams < best) {
        best = teams;
        p.big_splits = s;
        p.teams = true;
      }
    }
    if (p.teams) p.big_slots = 1 << 30;
    p.big_over = (int)over;
    p.big_blocks = (most + (p.big_splits - 1) * over) * NKV;
    if (p.big_splits > 1) p.big_units = over * NKV * kWaves;
  }
  p.few_floats = p.few_units * p.few_splits * (p.few_rows == 32 ? kFewRecord<2> : kFewRecord<1>);
  p.bytes = (p.few_floats + p.big_units * p.big_splits * kRecord) * 4;
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
  PDK_REQUIRE(p.few_blocks < (1ll << 30) && p.big_blocks < (1ll << 30) &&
                  p.big_units + p.few_units < (1ll << 31),
              "launch too large");
  const Args a{q, q_tok_stride, cache_k, cache_v, num_blocks, block_tables, max_blocks, starts,
               ctx_lens, N, R, n_q_heads, n_kv_heads, scale * 1.4426950408889634f, window, sinks,
               static_cast<float*>(workspace), out, p.few_rows, p.few_per, p.few_splits, p.big_slots,
               p.big_splits, p.big_over, p.few_floats};
  const hipStream_t st = pdk::as_stream(stream);
  const bool two = p.few_rows == 32;
  if (p.big && p.few_rows) {
    const unsigned turns = (unsigned)((p.few_blocks + kCUs - 1) / kCUs + (p.big_blocks + kCUs - 1) / kCUs);
    hipLaunchKernelGGL(chunk_both_kernel, dim3(kCUs * turns), dim3(256), 0, st, a, (int)p.few_blocks,
                       (int)p.big_blocks);
  } else if (p.big) {
    hipLaunchKernelGGL(p.teams ? chunk_big_kernel<3> : chunk_big_kernel<1>, dim3((unsigned)p.big_blocks),
                       dim3(p.teams ? 768 : 256), 0, st, a);
  } else {
    hipLaunchKernelGGL(two ? chunk_few_kernel<2> : chunk_few_kernel<1>, dim3((unsigned)p.few_blocks),
                       dim3(256), 0, st, a);
  }
  if (int rc = pdk::check_launch("chunk attention")) return rc;
  if (p.few_units + p.big_units) {
    hipLaunchKernelGGL(two ? chunk_join_kernel<2> : chunk_join_kernel<1>,
                       dim3((unsigned)(p.few_units + p.big_units)), dim3(256), 0, st, a, (int)p.few_units);
    if (int rc = pdk::check_launch("chunk_join_kernel")) return rc;
  }
  return PDK_OK;
}
