// y [T][N] bf16 = x . w^T of 8-bit (e4m3) rows x [T][K] with a scale for each 128 columns
// of a row and weights w [N][K] with a scale for each block of 128 x 128, gfx950:
//   y[t][n] = sum over groups g of xs[t][g] ws[n / 128][g] * (x[t] . w[n] over g's columns)
//
// A group is two v_mfma_f32_32x32x64_f8f6f4 (one v_mfma_f32_16x16x128 where there are few
// rows) into zero; then the group's sum is added with its scale, one fused multiply-add an
// element, in fp32. The instruction aligns the products of 8 consecutive columns to the
// largest of them and cuts what lies 13 binary places below it, then adds in fp32
// (measured: beside 2^13 a product of 1 is kept, beside 2^14 it is not; columns from the
// next 8 on are). That is some 2e-4 rms of a result where the values' own 8 bits
// are 3e-2 and the output's rounding 1e-3; the 16-bit instructions would be exact at half
// the rate. The weights are the A operand, so that a lane's column is one token and the
// scale one value per lane; a wavefront's weights lie in one block of 128, so ws is one
// value. Both operands take the columns of a group in the same order (16-byte chunks),
// whichever the instruction gives them.
//
// Tiles: rows of 128 bytes are staged by copies straight into LDS (no registers), 16-byte
// chunk c of row r at place c ^ (r / 2 & 7): 16 lanes at one chunk of 16 rows then read all
// banks. The next groups' tiles are under way while one is multiplied, one barrier per
// group; their copies are issued a few at a time between the products (all at once they
// hold up the LDS reads behind them: 8192 x 28672 x 4096 961 us, spread 899), the scales
// come the same way (as vector loads of each wavefront 899, so 861). A tile's scaled addition
// runs under the next tile's products (one after the other 1003, so 961).
//
// Bound by the matrix cores' power at the largest sizes: 870 to 900 us, 2140 to 2210
// TFLOP/s, where the loop without any copy takes 737 and the library's product with one
// scale for all 769. Smaller ones are bound by a group's chain (barrier, LDS read, two
// products, addition), 0.54 to 1.5 us by tile, so that the tile and the split of K are chosen
// by the time that these chains take (Shape, below). Up to 16 rows by the weights' bytes.
#include <math.h>

#include <algorithm>

#include "lds_copy.h"

namespace {

using pdk::v8;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kGroup = 128;

struct Args {
  const uint8_t* x;
  int64_t x_ld;
  const float* xs;
  int64_t xs_t, xs_g;                     // strides of xs over tokens and groups
  const uint8_t* w;
  const float* ws;
  int T, N, K;
  uint16_t* y;
  int splits, per;                        // of the groups over workgroups, groups of a split
  float* part;                            // their sums, where there are several
};

__device__ __forceinline__ i32x8 join(const uint4& a, const uint4& b) {
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// A lane's 32 tokens x 32 weights tile as bf16: it holds weights 8 q + 4 hh + 0..3 of token
// `row`; a lane swap of q, q + 1 gives each half 8 consecutive ones.
__device__ __forceinline__ void store_tile(const Args& a, const f32x16& v, int row, int col, int hh) {
#pragma unroll
  for (int q = 0; q < 4; q += 2) {
    uint32_t w[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        w[i][e] = pdk::pack_bf16x2_rne(v[4 * (q + i) + 2 * e], v[4 * (q + i) + 2 * e + 1]);
    const auto b0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
    const auto b1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
    const int c = col + 8 * (q + hh);
    if (row < a.T && c < a.N) pdk::st16(a.y + (int64_t)row * a.N + c, v8{{b0[0], b1[0], b0[1], b1[1]}});
  }
}

// kTT x kWT tiles of 32 tokens x 32 weights per wavefront, kWavesT x kWavesW wavefronts. An
// item is a split of a tile; a workgroup takes the items blockIdx.x, blockIdx.x +
// gridDim.x, ...: the next one's first groups are under way while the last ones of this
// are multiplied and stored.
template <int kTT, int kWT, int kWavesT, int kWavesW, int kPerSimd, int kRing>
__global__ __launch_bounds__(64 * kWavesT * kWavesW, kPerSimd) void fp8_tile_kernel(Args a, int items) {
  static_assert(kWavesT * kWavesW > kWavesT * kTT / 2 && kWavesT * kTT % 2 == 0, "wavefronts for all scales");
  constexpr int kBT = 32 * kTT * kWavesT, kBW = 32 * kWT * kWavesW, kNW = kWavesT * kWavesW;
  constexpr int kLoadsX = kBT / 8 / kNW, kLoadsW = kBW / 8 / kNW;   // of a wavefront, 8 rows each
  constexpr int kLoads = kLoadsX + kLoadsW, kPairs = kTT * kWT;
  constexpr int kSpread = kPairs > 1 ? kPairs / 2 : 1;   // half tiles that copies are issued under
  __shared__ __align__(1024) uint8_t sm[kRing][(kBT + kBW) * kGroup];
  // A group's scales of the tokens; of the weights' blocks of 128 from the first on.
  __shared__ __align__(256) float sm_s[kRing][kBT + 64];
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wt = wave % kWavesT, ww = wave / kWavesT;
  const int t_tiles = (a.T + kBT - 1) / kBT;
  const int groups = a.K / kGroup;
  // Staging: load l of a wavefront takes rows 8 (l kNW + wave) .. of x's tile, then of w's.
  uint32_t x_off[kLoadsX], w_off[kLoadsW];
  const uint8_t *xp, *wp;
  uint32_t s_off;                         // of the scales a wavefront brings, if it does
  const float *xsp, *wsp;
  int t0, n0;
  auto aim = [&](int item) __attribute__((always_inline)) {
    const int tile = item / a.splits;
    int lane = threadIdx.x & 63;          // anew for each tile: kept, it would be spilled
    asm("" : "+v"(lane));
    const int j = lane & 31;
    t0 = tile % t_tiles * kBT;
    n0 = tile / t_tiles * kBW;
    xp = a.x + t0 * a.x_ld;
    wp = a.w + (int64_t)n0 * a.K;
#pragma unroll
    for (int l = 0; l < kLoadsX; ++l) {
      const int r = 8 * (l * kNW + wave) + (lane >> 3);
      x_off[l] = (uint32_t)(min(r, a.T - 1 - t0) * a.x_ld) + ((lane & 7) ^ (r >> 1 & 7)) * 16;
    }
#pragma unroll
    for (int l = 0; l < kLoadsW; ++l) {
      const int r = 8 * (l * kNW + wave) + (lane >> 3);
      w_off[l] = (uint32_t)(min(r, a.N - 1 - n0) * a.K) + ((lane & 7) ^ (r >> 1 & 7)) * 16;
    }
    // Scales: wavefronts 0 .. bring 64 tokens' each, the next one the weights' blocks' (as do
    // those behind it, so that all have as many copies under way).
    xsp = a.xs + t0 * a.xs_t;
    wsp = a.ws + (int64_t)(n0 / kGroup) * groups;
    s_off = wave < kBT / 64 ? min(64 * wave + lane, a.T - 1 - t0) * (int)a.xs_t * 4
                            : min(lane, (a.N - 1) / kGroup - n0 / kGroup) * groups * 4;
  };
  const uint32_t lds = pdk::lds_address(sm) + wave * 1024;
  const uint32_t lds_s = pdk::lds_address(sm_s);
  // Piece `at` of the loads of group g (x's tile, then w's), and the group's scales.
  auto fetch = [&](int slot, int g, int at) __attribute__((always_inline)) {
    const uint32_t to = lds + slot * sizeof(sm[0]) + at * kNW * 1024;
    if (at < kLoadsX) pdk::copy16(xp + g * kGroup, x_off[at < kLoadsX ? at : 0], to);
    else pdk::copy16(wp + g * kGroup, w_off[at < kLoadsX ? 0 : at - kLoadsX], to);
  };
  auto fetch_scales = [&](int slot, int g) __attribute__((always_inline)) {
    const uint32_t to = lds_s + slot * sizeof(sm_s[0]) + min(wave, kBT / 64) * 256;
    pdk::copy4(wave < kBT / 64 ? xsp + g * a.xs_g : wsp + g, s_off, to);
  };
  // Chunk c of row r: c ^ (r / 2 & 7); rows of a lane differ by 32, so its place does not.
  uint32_t place[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int k = 0; k < 2; ++k) place[h][k] = j * kGroup + ((4 * h + 2 * k + hh) ^ (j >> 1 & 7)) * 16;
  auto operand = [&](const uint8_t* rows, int h) __attribute__((always_inline)) {
    return join(*reinterpret_cast<const uint4*>(rows + place[h][0]),
                *reinterpret_cast<const uint4*>(rows + place[h][1]));
  };
  // Group `next` of item `ahead` is the last one fetched; kRing - 1 are under way. Behind the
  // last item its groups are fetched again.
  auto first_of = [&](int item) { return item % a.splits * a.per; };
  int slot = 0, ahead = blockIdx.x, next = first_of(ahead);
  auto advance = [&]() __attribute__((always_inline)) {
    if (++next < min(first_of(ahead) + a.per, groups)) return;
    if (ahead + (int)gridDim.x < items) {
      ahead += gridDim.x;
      aim(ahead);
    }
    next = first_of(ahead);
  };
  aim(ahead);
#pragma unroll
  for (int r = 0; r < kRing - 1; ++r) {
    if (r) advance();
#pragma unroll
    for (int l = 0; l < kLoads; ++l) fetch(r, next, l);
    fetch_scales(r, next);
  }
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int tile = item / a.splits, t0_now = tile % t_tiles * kBT, n0_now = tile / t_tiles * kBW;
    const int steps = min(a.per, groups - first_of(item));
    f32x16 acc[kTT][kWT];
#pragma unroll
    for (int t = 0; t < kTT; ++t)
#pragma unroll
      for (int n = 0; n < kWT; ++n)
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[t][n][x] = 0.f;
    auto multiply = [&]() __attribute__((always_inline)) {
      const int to = slot == 0 ? kRing - 1 : slot - 1;          // that of the group before
      const uint8_t* const sx = sm[slot] + 32 * wt * kTT * kGroup;
      const uint8_t* const sw = sm[slot] + (kBT + 32 * ww * kWT) * kGroup;
      fetch_scales(to, next);
      float s[kTT];
      {
        const float w_scale = sm_s[slot][kBT + 32 * ww * kWT / kGroup];
#pragma unroll
        for (int t = 0; t < kTT; ++t) s[t] = sm_s[slot][32 * (wt * kTT + t) + j] * w_scale;
      }
      i32x8 wv[kWT][2], xv[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) xv[h] = operand(sx, h);
#pragma unroll
      for (int n = 0; n < kWT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) wv[n][h] = operand(sw + 32 * n * kGroup, h);
      // A tile's products, and meanwhile the scaled addition of the one before.
      f32x16 part[2];
      auto add = [&](int i, int from, int to) __attribute__((always_inline)) {
#pragma unroll
        for (int x = from; x < to; ++x)
          acc[i / kWT][i % kWT][x] = __builtin_fmaf(part[i & 1][x], s[i / kWT], acc[i / kWT][i % kWT][x]);
      };
#pragma unroll
      for (int i = 0; i < kTT * kWT; ++i) {
        const int t = i / kWT, n = i % kWT;
        f32x16 z;
#pragma unroll
        for (int x = 0; x < 16; ++x) z[x] = 0.f;
        // Half a group's products, and under them half of the addition of the tile before;
        // a half of the next tokens is read as soon as this one has been taken.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          part[i & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[n][h], xv[h], h ? part[i & 1] : z, 0, 0,
                                                                        0, 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          if (n == kWT - 1 && t + 1 < kTT) xv[h] = operand(sx + 32 * (t + 1) * kGroup, h);
          if (i) add(i - 1, 8 * h, 8 * h + 8);
          // The next group's copies, a few at a time.
#pragma unroll
          for (int l = 0; l < kLoads; ++l)
            if (l * kSpread / kLoads == 2 * i + h) fetch(to, next, l);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      add(kTT * kWT - 1, 0, 16);
      slot = slot + 1 == kRing ? 0 : slot + 1;
    };
    for (int g = 0; g < steps; ++g) {
      pdk::copies_done<(kRing - 2) * (kLoads + 1)>();
      advance();
      multiply();
    }
    if (a.splits == 1) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        store_tile(a, acc[i / kWT][i % kWT], t0_now + 32 * (wt * kTT + i / kWT) + j,
                   n0_now + 32 * (ww * kWT + i % kWT), hh);
    } else {
      // As the registers have them: [item][wavefront][tile][4][lane] float4s.
      float4* const to = reinterpret_cast<float4*>(a.part) +
                         (((int64_t)item * kNW + wave) * kPairs) * 256 + lane;
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const f32x16& v = acc[i / kWT][i % kWT];
          to[(4 * i + x) * 64] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
        }
    }
  }
  pdk::copies_done<0>();                  // none may arrive in another workgroup's LDS
}

// The splits' sums of a tile added in order, a wavefront for each 32 x 32.
template <int kTT, int kWT, int kWavesT, int kWavesW>
__global__ __launch_bounds__(256) void fp8_join_kernel(Args a, int tiles32) {
  constexpr int kPairs = kTT * kWT, kNW = kWavesT * kWavesW;
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int u = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (u >= tiles32) return;
  const int i = u % kPairs, wave = u / kPairs % kNW, tile = u / (kPairs * kNW);
  const int t_tiles = (a.T + 32 * kTT * kWavesT - 1) / (32 * kTT * kWavesT);
  const int row0 = (tile % t_tiles * kWavesT + wave % kWavesT) * 32 * kTT + i / kWT * 32;
  const int col0 = (tile / t_tiles * kWavesW + wave / kWavesT) * 32 * kWT + i % kWT * 32;
  if (row0 >= a.T || col0 >= a.N) return;
  const float4* from = reinterpret_cast<const float4*>(a.part) +
                       (((int64_t)tile * a.splits * kNW + wave) * kPairs + i) * 256 + lane;
  const int64_t stride = (int64_t)kNW * kPairs * 256;
  f32x16 sum;
#pragma unroll
  for (int x = 0; x < 16; ++x) sum[x] = 0.f;
  for (int z0 = 0; z0 < a.splits; z0 += 4) {         // four splits' loads at a time
    float4 y[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int x = 0; x < 4; ++x) y[k][x] = from[min(z0 + k, a.splits - 1) * stride + x * 64];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (z0 + k >= a.splits) break;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        sum[4 * x] += y[k][x].x;
        sum[4 * x + 1] += y[k][x].y;
        sum[4 * x + 2] += y[k][x].z;
        sum[4 * x + 3] += y[k][x].w;
      }
    }
  }
  store_tile(a, sum, row0 + j, col0, hh);
}

// Up to 16 rows: bound by the weights' bytes. A workgroup has 16 kRT weights, its wavefronts
// every kNW-th group each, operands straight from memory (v_mfma_f32_16x16x128_f8f6f4: a
// lane has chunks kg and kg + 4 of row i); their sums are added in LDS.
template <int kRT, int kNW>
__global__ __launch_bounds__(64 * kNW) void fp8_few_kernel(Args a) {
  __shared__ f32x4 sm[kNW][kRT][64];
  const int lane = threadIdx.x & 63, i = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16 * kRT, groups = a.K / kGroup;
  const int64_t row = min(i, a.T - 1);
  const uint8_t* const xp = a.x + row * a.x_ld + kg * 16;
  const float* const xsp = a.xs + row * a.xs_t;
  const float* const wsp = a.ws + (int64_t)(n0 / kGroup) * groups;   // 16 kRT divides 128
  const uint8_t* wp[kRT];
  f32x4 acc[kRT];
#pragma unroll
  for (int r = 0; r < kRT; ++r) {
    wp[r] = a.w + (int64_t)min(n0 + 16 * r + i, a.N - 1) * a.K + kg * 16;
    acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  struct Operands {
    uint4 w[kRT][2], x[2];
    float xs, ws;
  };
  // Every workgroup begins at another group: rows lie a power of two apart, and at the same
  // columns they all ask the same channels of the memory (28672 x 4096 26.0 us, so 23.2; 4096
  // x 14336 14.6 and 14.9).
  const int first = (int)(blockIdx.x * (kNW + 1) % groups);
  auto load = [&](int g) __attribute__((always_inline)) {
    Operands o;
    g += first;
    if (g >= groups) g -= groups;
    const int64_t at = (int64_t)g * kGroup;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r = 0; r < kRT; ++r) o.w[r][h] = *reinterpret_cast<const uint4*>(wp[r] + at + 64 * h);
      o.x[h] = *reinterpret_cast<const uint4*>(xp + at + 64 * h);
    }
    o.xs = xsp[g * a.xs_g];
    o.ws = wsp[g];
    return o;
  };
  if (wave < groups) {
    // The next group's operands are under way as soon as this one's have been taken; more
    // of them gained nothing (28672 x 4096, 16 rows, before the starts at other groups: 26.9 us,
    // two 29.1, three 31.9).
    Operands o = load(wave);
    for (int g = wave; g < groups; g += kNW) {
      const i32x8 x = join(o.x[0], o.x[1]);
      const float s = o.xs * o.ws;
#pragma unroll
      for (int r = 0; r < kRT; ++r) {
        const f32x4 part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            join(o.w[r][0], o.w[r][1]), x, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] = __builtin_fmaf(part[e], s, acc[r][e]);
      }
      o = load(min(g + kNW, groups - 1));
    }
  }
#pragma unroll
  for (int r = 0; r < kRT; ++r) sm[wave][r][lane] = acc[r];
  __syncthreads();
  // Lane (i, kg): token i, weights 4 kg .. + 3 of each tile.
  for (int r = wave; r < kRT; r += kNW) {
    f32x4 sum = sm[0][r][lane];
#pragma unroll
    for (int w = 1; w < kNW; ++w) sum += sm[w][r][lane];
    const int col = n0 + 16 * r + 4 * kg;
    if (i < a.T && col < a.N)
      *reinterpret_cast<uint2*>(a.y + (int64_t)i * a.N + col) =
          make_uint2(pdk::pack_bf16x2_rne(sum[0], sum[1]), pdk::pack_bf16x2_rne(sum[2], sum[3]));
  }
}

// A tile of tokens x weights: workgroups at once on the card; us that a group takes where each
// has a CU to itself, and where all run.
struct Shape {
  int t, w, at_once;
  double alone, full;
};

constexpr Shape kShapes[] = {
    {256, 256, 256, 1.6, 1.98},
    {128, 256, 256, 0.98, 1.16},
    {128, 128, 256, 0.62, 0.72},
    {64, 128, 512, 0.54, 0.84},
};

// Items of a product whose K is split: the splits' sums take at most 2048 tiles of 256 KB, 512 MiB.
constexpr int kMostItems = 2048;

struct Plan {
  int shape, splits, per;                 // groups of a split
  int64_t bytes;                          // of the splits' sums
};

// The shape and split that end soonest: rounds of workgroups, each its groups and 2 us for
// its start and its store; where K is split another launch (3 us) and the splits' sums
// written and read, 4.5 TB/s. Chosen and another, us, operands from memory: 64 x 4096 x 14336
// (rows, weights, columns) 64 x 128 split in 8 20.0, unsplit 63.5; 470 x 4096 x 14336 128 x 256 in 4
// 46 to 51, 64 x 128 unsplit 68; 470 x 28672 x 4096 256 x 256 69, 128 x 256 83; 1000 x 4096 x 4096
// 128 x 128 25.7, 256 x 256 49; 2000 x 4096 x 14336 256 x 256 in 2 126, 128 x 256 132.
Plan plan_for(int T, int K, int N) {
  const int groups = K / kGroup;
  Plan best{};
  double least = 1e30;
  for (int i = 0; i < (int)(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
    const Shape& s = kShapes[i];
    const int64_t tiles = (int64_t)((T + s.t - 1) / s.t) * ((N + s.w - 1) / s.w);
    for (int splits = 1; splits <= 16 && splits <= groups; ++splits) {
      const int per = (groups + splits - 1) / splits;
      if (per * (splits - 1) >= groups) continue;              // the last one would be empty
      const int64_t items = tiles * splits, bytes = splits > 1 ? items * s.t * s.w * 4 : 0;
      if (splits > 1 && items > kMostItems) break;
      const double rounds = (double)((items + s.at_once - 1) / s.at_once);
      const double us = rounds * (per * (items <= 256 ? s.alone : s.full) + 2.0) +
                        (splits > 1 ? 3.0 + 2.0 * bytes / 4.5e6 : 0.0);
      if (us < least) {
        least = us;
        best = Plan{i, splits, per, bytes};
      }
    }
  }
  return best;
}

template <int kTT, int kWT, int kWavesT, int kWavesW, int kPerSimd, int kRing>
void launch_tiles(const Args& a, const Shape& s, hipStream_t st) {
  constexpr int kBT = 32 * kTT * kWavesT, kBW = 32 * kWT * kWavesW, kNW = kWavesT * kWavesW;
  const int tiles = (a.T + kBT - 1) / kBT * ((a.N + kBW - 1) / kBW), items = tiles * a.splits;
  hipLaunchKernelGGL((fp8_tile_kernel<kTT, kWT, kWavesT, kWavesW, kPerSimd, kRing>),
                     dim3(std::min(items, s.at_once)), dim3(64 * kNW), 0, st, a, items);
  if (a.splits > 1) {
    const int n = tiles * kNW * kTT * kWT;
    hipLaunchKernelGGL((fp8_join_kernel<kTT, kWT, kWavesT, kWavesW>), dim3((n + 3) / 4), dim3(256), 0,
                       st, a, n);
  }
}

template <int kRT, int kNW>
void launch_few(const Args& a, hipStream_t st) {
  hipLaunchKernelGGL((fp8_few_kernel<kRT, kNW>), dim3((a.N + 16 * kRT - 1) / (16 * kRT)), dim3(64 * kNW),
                     0, st, a);
}

constexpr int kFewRows = 16;

int check_sizes(int T, int K, int N) {
  PDK_REQUIRE(T >= 0 && T <= (1 << 20), "T must be in [0, 2^20] (got %d)", T);
  PDK_REQUIRE(K >= kGroup && K % kGroup == 0 && K <= (1 << 20),
              "K must be a multiple of %d in [%d, 2^20] (got %d)", kGroup, kGroup, K);
  PDK_REQUIRE(N >= 8 && N % 8 == 0 && N <= (1 << 20), "N must be a multiple of 8 in [8, 2^20] (got %d)", N);
  return PDK_OK;
}

}  // namespace

extern "C" int64_t pdk_linear_fp8_workspace_bytes(int T, int K, int N) {
  pdk::clear_error();
  if (check_sizes(T, K, N)) return -1;
  return T <= kFewRows ? 0 : plan_for(T, K, N).bytes;
}

extern "C" int pdk_linear_fp8(const uint8_t* x, int64_t x_ld, const float* x_scales, int64_t xs_tok_stride,
                              int64_t xs_group_stride, const uint8_t* w, const float* w_scales, int T,
                              int K, int N, void* workspace, size_t workspace_bytes, uint16_t* y,
                              uintptr_t stream) {
  pdk::clear_error();
  if (int rc = check_sizes(T, K, N)) return rc;
  PDK_REQUIRE(x_ld >= K && x_ld % 16 == 0 && x_ld < (1 << 24),
              "x_ld must be a multiple of 16 below 2^24 that holds a row");
  PDK_REQUIRE(xs_tok_stride >= 1 && xs_tok_stride < (1 << 21) && xs_group_stride >= 1,
              "scale strides must be >= 1, between tokens below 2^21");
  if (T == 0) return PDK_OK;
  PDK_REQUIRE(x && x_scales && w && w_scales && y, "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(x) && pdk::aligned16(w) && pdk::aligned16(y),
              "tensors must be 16-byte aligned");
  Args a{x, x_ld, x_scales, xs_tok_stride, xs_group_stride, w, w_scales, T, N, K, y, 1, K / kGroup, nullptr};
  const hipStream_t st = pdk::as_stream(stream);
  if (T <= kFewRows) {
    // Weights of a workgroup: as many as leave every CU one. us with 16, 32 and 64, 16 rows, operands
    // from memory: 28672 x 4096 32.7, 26.5, 23.3; 16384 x 4096 19.7, 14.8, 16.4; 6144 x 4096 10.5, 7.7,
    // 12.7; 4096 x 4096 6.0, 7.6, 12.6; 4096 x 14336 18.2, 21.6, 45.9. Not always the best: 18432 x 4096
    // 23.8, 19.8, 21.9; 57344 x 8192 116, 87, 90.
    if (N > 64 * 256) launch_few<4, 4>(a, st);
    else if (N > 16 * 256) launch_few<2, 8>(a, st);
    else launch_few<1, 8>(a, st);
    return pdk::check_launch("fp8_few_kernel");
  }
  const Plan p = plan_for(T, K, N);
  PDK_REQUIRE(p.bytes == 0 || (workspace && pdk::aligned16(workspace)),
              "a workspace, 16-byte aligned, is needed");
  if (p.bytes > 0 && workspace_bytes < (size_t)p.bytes) {
    pdk::set_error("workspace of %zu bytes, %lld needed", workspace_bytes, (long long)p.bytes);
    return PDK_ENOMEM;
  }
  a.splits = p.splits;
  a.per = p.per;
  a.part = static_cast<float*>(workspace);
  const Shape& s = kShapes[p.shape];
  switch (p.shape) {
    case 0: launch_tiles<4, 2, 2, 4, 2, 2>(a, s, st); break;
    case 1: launch_tiles<2, 2, 2, 4, 2, 3>(a, s, st); break;
    case 2: launch_tiles<2, 1, 2, 4, 2, 4>(a, s, st); break;
    default: launch_tiles<1, 2, 2, 2, 2, 3>(a, s, st); break;
  }
  return pdk::check_launch("fp8_tile_kernel");
}
