// y [T][N] bf16 = x . w^T of 8-bit (e4m3) rows x [T][K] with a scale for each 128 columns
// of a row and weights w [N][K] with a scale for each block of 128 x 128, gfx950:
//   y[t][n] = sum over groups g of xs[t][g] ws[n / 128][g] * (x[t] . w[n] over g's columns)
//
// A group is two v_mfma_f32_32x32x64_f8f6f4 (one v_mfma_f32_16x16x128 where there are few
// rows) into zero, the products and their sums in fp32; then the group's sum is added
// with its scale, one fused multiply-add an element. The weights are the A operand, so
// that a lane's column is one token and the scale one value per lane; a wavefront's
// weights lie in one block of 128, so ws is a scalar. Both operands take the columns of
// a group in the same order (16-byte chunks), whichever the instruction gives them.
//
// Tiles: rows of 128 bytes are staged by global_load_lds (no registers), 16-byte chunk c of
// row r at place c ^ (r / 2 & 7): 16 lanes at one chunk of 16 rows then read all banks. The
// next group's tile is under way while one is multiplied; one barrier per group.
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
};

__device__ __forceinline__ i32x8 join(const uint4& a, const uint4& b) {
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// kTT x kWT tiles of 32 tokens x 32 weights per wavefront, kWavesT x kWavesW wavefronts.
template <int kTT, int kWT, int kWavesT, int kWavesW, int kPerSimd>
__global__ __launch_bounds__(64 * kWavesT * kWavesW, kPerSimd) void fp8_tile_kernel(Args a) {
  constexpr int kBT = 32 * kTT * kWavesT, kBW = 32 * kWT * kWavesW, kNW = kWavesT * kWavesW;
  constexpr int kLoadsX = kBT / 8 / kNW, kLoadsW = kBW / 8 / kNW;   // of a wavefront, 8 rows each
  __shared__ __align__(1024) uint8_t sm[2][(kBT + kBW) * kGroup];
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wt = wave % kWavesT, ww = wave / kWavesT;
  const int t_tiles = (a.T + kBT - 1) / kBT;
  const int t0 = (blockIdx.x % t_tiles) * kBT, n0 = (blockIdx.x / t_tiles) * kBW;
  const int groups = a.K / kGroup;
  // Staging: load l of a wavefront takes rows 8 (l kNW + wave) .. of x's tile, then of w's.
  uint32_t x_off[kLoadsX], w_off[kLoadsW];
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
  const uint8_t *const xp = a.x + t0 * a.x_ld, *const wp = a.w + (int64_t)n0 * a.K;
  const uint32_t lds = pdk::lds_address(sm) + wave * 1024;
  auto fetch = [&](int slot, int g) __attribute__((always_inline)) {
    const uint32_t to = lds + slot * sizeof(sm[0]);
#pragma unroll
    for (int l = 0; l < kLoadsX; ++l) pdk::copy16(xp + g * kGroup, x_off[l], to + l * kNW * 1024);
#pragma unroll
    for (int l = 0; l < kLoadsW; ++l)
      pdk::copy16(wp + g * kGroup, w_off[l], to + kBT * kGroup + l * kNW * 1024);
  };
  // Scales: a lane's tokens', the wavefront's weights'.
  const float* xsp[kTT];
#pragma unroll
  for (int t = 0; t < kTT; ++t)
    xsp[t] = a.xs + (int64_t)min(t0 + 32 * (wt * kTT + t) + j, a.T - 1) * a.xs_t;
  const float* wsp = a.ws + (int64_t)(min(n0 + 32 * kWT * ww, a.N - 1) / kGroup) * groups;
  float xs[kTT], w_scale = wsp[0];
#pragma unroll
  for (int t = 0; t < kTT; ++t) xs[t] = xsp[t][0];
  fetch(0, 0);
  f32x16 acc[kTT][kWT];
#pragma unroll
  for (int t = 0; t < kTT; ++t)
#pragma unroll
    for (int n = 0; n < kWT; ++n)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[t][n][x] = 0.f;
  // Chunk c of row r: c ^ (r / 2 & 7); rows of a lane differ by 32, so its place does not.
  const int key = j >> 1 & 7;
  const int x_at = (32 * wt * kTT + j) * kGroup, w_at = (kBT + 32 * ww * kWT + j) * kGroup;
  auto step = [&](int g, const uint8_t* st) __attribute__((always_inline)) {
    pdk::copies_done<0>();
    float s[kTT];
#pragma unroll
    for (int t = 0; t < kTT; ++t) {
      s[t] = xs[t] * w_scale;
      asm volatile("" : "+v"(s[t]));      // before the next copies, for which it would wait
    }
    if (g + 1 < groups) {
      fetch(g & 1 ^ 1, g + 1);
#pragma unroll
      for (int t = 0; t < kTT; ++t) xs[t] = xsp[t][(int64_t)(g + 1) * a.xs_g];
      w_scale = wsp[g + 1];
    }
    auto operand = [&](int at, int half) {
      const uint4 u = *reinterpret_cast<const uint4*>(st + at + ((4 * half + hh) ^ key) * 16);
      const uint4 v = *reinterpret_cast<const uint4*>(st + at + ((4 * half + 2 + hh) ^ key) * 16);
      return join(u, v);
    };
    i32x8 wv[kWT][2];
#pragma unroll
    for (int n = 0; n < kWT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) wv[n][h] = operand(w_at + 32 * n * kGroup, h);
#pragma unroll
    for (int t = 0; t < kTT; ++t) {
      const i32x8 x0 = operand(x_at + 32 * t * kGroup, 0), x1 = operand(x_at + 32 * t * kGroup, 1);
#pragma unroll
      for (int n = 0; n < kWT; ++n) {
        f32x16 part;
#pragma unroll
        for (int x = 0; x < 16; ++x) part[x] = 0.f;
        part = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[n][0], x0, part, 0, 0, 0, 0, 0, 0);
        part = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[n][1], x1, part, 0, 0, 0, 0, 0, 0);
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[t][n][x] = __builtin_fmaf(part[x], s[t], acc[t][n][x]);
      }
    }
  };
  for (int g = 0; g < groups; ++g) step(g, sm[g & 1]);
  // A lane holds weights 8 q + 4 hh + 0..3 of its token; a lane swap of q, q + 1 gives each
  // half 8 consecutive ones.
#pragma unroll
  for (int t = 0; t < kTT; ++t) {
    const int row = t0 + 32 * (wt * kTT + t) + j;
#pragma unroll
    for (int n = 0; n < kWT; ++n)
#pragma unroll
      for (int q = 0; q < 4; q += 2) {
        uint32_t w[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            w[i][e] = pdk::pack_bf16x2_rne(acc[t][n][4 * (q + i) + 2 * e], acc[t][n][4 * (q + i) + 2 * e + 1]);
        const auto b0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto b1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        const int col = n0 + 32 * (ww * kWT + n) + 8 * (q + hh);
        if (row < a.T && col < a.N)
          pdk::st16(a.y + (int64_t)row * a.N + col, v8{{b0[0], b1[0], b0[1], b1[1]}});
      }
  }
}

// Few rows: a workgroup has 16 kRT weights for all tokens (16 kTT of them), its wavefronts
// every kNW-th group each, operands straight from memory; their sums are added in LDS.
template <int kRT, int kTT, int kNW>
__global__ __launch_bounds__(64 * kNW) void fp8_few_kernel(Args a) {
  __shared__ f32x4 sm[kNW][kRT * kTT][64];
  const int lane = threadIdx.x & 63, i = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16 * kRT, t0 = blockIdx.y * 16 * kTT, groups = a.K / kGroup;
  const uint8_t *wp[kRT], *xp[kTT];
  const float* xsp[kTT];
#pragma unroll
  for (int r = 0; r < kRT; ++r) wp[r] = a.w + (int64_t)min(n0 + 16 * r + i, a.N - 1) * a.K + kg * 16;
#pragma unroll
  for (int t = 0; t < kTT; ++t) {
    const int64_t row = min(t0 + 16 * t + i, a.T - 1);
    xp[t] = a.x + row * a.x_ld + kg * 16;
    xsp[t] = a.xs + row * a.xs_t;
  }
  const float* wsp = a.ws + (int64_t)(n0 / kGroup) * groups;   // 16 kRT divides 128
  f32x4 acc[kRT][kTT];
#pragma unroll
  for (int r = 0; r < kRT; ++r)
#pragma unroll
    for (int t = 0; t < kTT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Operands {
    uint4 w[kRT][2], x[kTT][2];
    float xs[kTT], ws;
  };
  auto load = [&](int g) __attribute__((always_inline)) {
    Operands o;
    const int64_t at = (int64_t)g * kGroup;
#pragma unroll
    for (int r = 0; r < kRT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) o.w[r][h] = *reinterpret_cast<const uint4*>(wp[r] + at + 64 * h);
#pragma unroll
    for (int t = 0; t < kTT; ++t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) o.x[t][h] = *reinterpret_cast<const uint4*>(xp[t] + at + 64 * h);
      o.xs[t] = xsp[t][g * a.xs_g];
    }
    o.ws = wsp[g];
    return o;
  };
  auto multiply = [&](const Operands& o) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kTT; ++t) {
      const i32x8 x = join(o.x[t][0], o.x[t][1]);
      const float s = o.xs[t] * o.ws;
#pragma unroll
      for (int r = 0; r < kRT; ++r) {
        const f32x4 part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            join(o.w[r][0], o.w[r][1]), x, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][t][e] = __builtin_fmaf(part[e], s, acc[r][t][e]);
      }
    }
  };
  if (wave < groups) {
    // Two groups' operands are under way beside the one that is multiplied.
    Operands now = load(wave);
    for (int g = wave; g < groups; g += kNW) {
      const Operands next = load(min(g + kNW, groups - 1));
      multiply(now);
      now = next;
    }
  }
#pragma unroll
  for (int r = 0; r < kRT; ++r)
#pragma unroll
    for (int t = 0; t < kTT; ++t) sm[wave][r * kTT + t][lane] = acc[r][t];
  __syncthreads();
  // Lane (i, kg): token i, weights 4 kg .. + 3 of each tile.
  for (int u = wave; u < kRT * kTT; u += kNW) {
    f32x4 sum = sm[0][u][lane];
#pragma unroll
    for (int w = 1; w < kNW; ++w) sum += sm[w][u][lane];
    const int row = t0 + 16 * (u % kTT) + i, col = n0 + 16 * (u / kTT) + 4 * kg;
    if (row < a.T && col < a.N)
      *reinterpret_cast<uint2*>(a.y + (int64_t)row * a.N + col) =
          make_uint2(pdk::pack_bf16x2_rne(sum[0], sum[1]), pdk::pack_bf16x2_rne(sum[2], sum[3]));
  }
}

template <int kTT, int kWT, int kWavesT, int kWavesW, int kPerSimd>
void launch_tiles(const Args& a, hipStream_t st) {
  constexpr int kBT = 32 * kTT * kWavesT, kBW = 32 * kWT * kWavesW;
  const int blocks = (a.T + kBT - 1) / kBT * ((a.N + kBW - 1) / kBW);
  hipLaunchKernelGGL((fp8_tile_kernel<kTT, kWT, kWavesT, kWavesW, kPerSimd>), dim3(blocks),
                     dim3(64 * kWavesT * kWavesW), 0, st, a);
}

}  // namespace

extern "C" int pdk_linear_fp8(const uint8_t* x, int64_t x_ld, const float* x_scales, int64_t xs_tok_stride,
                              int64_t xs_group_stride, const uint8_t* w, const float* w_scales, int T,
                              int K, int N, uint16_t* y, uintptr_t stream) {
  pdk::clear_error();
  PDK_REQUIRE(T >= 0 && T <= (1 << 20), "T must be in [0, 2^20] (got %d)", T);
  PDK_REQUIRE(K >= kGroup && K % kGroup == 0 && K <= (1 << 20),
              "K must be a multiple of %d in [%d, 2^20] (got %d)", kGroup, kGroup, K);
  PDK_REQUIRE(N >= 8 && N % 8 == 0 && N <= (1 << 20), "N must be a multiple of 8 in [8, 2^20] (got %d)", N);
  PDK_REQUIRE(x_ld >= K && x_ld % 16 == 0 && x_ld < (1 << 24), "x_ld must be a multiple of 16 below 2^24 that holds a row");
  PDK_REQUIRE(xs_tok_stride >= 1 && xs_group_stride >= 1, "scale strides must be >= 1");
  if (T == 0) return PDK_OK;
  PDK_REQUIRE(x && x_scales && w && w_scales && y, "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(x) && pdk::aligned16(w) && pdk::aligned16(y),
              "tensors must be 16-byte aligned");
  const Args a{x, x_ld, x_scales, xs_tok_stride, xs_group_stride, w, w_scales, T, N, K, y};
  const hipStream_t st = pdk::as_stream(stream);
  if (T <= 16) {
    hipLaunchKernelGGL((fp8_few_kernel<4, 1, 4>), dim3((N + 63) / 64), dim3(256), 0, st, a);
  } else if ((int64_t)((T + 255) / 256) * ((N + 255) / 256) >= 256) {
    launch_tiles<4, 2, 2, 4, 2>(a, st);
  } else if ((int64_t)((T + 127) / 128) * ((N + 127) / 128) >= 256) {
    launch_tiles<2, 2, 2, 2, 2>(a, st);
  } else {
    launch_tiles<1, 1, 2, 2, 2>(a, st);
  }
  return pdk::check_launch("fp8 product");
}
