// RMSNorm with the residual's addition and an output in 8 bits, and rows (of bf16,
// or SwiGLU's of gate|up) brought to 8 bits, gfx950: with x + add rounded to bf16
// and kept,
//   y = (x + add) * rsqrt(mean((x + add)^2) + eps) * w
// and, for each 128 columns of a row, scale = max(|y|, 2^-100) / 448 and the e4m3
// values of y / scale: the largest of a group becomes 448, the largest e4m3 value.
// fp32 between; y itself is never rounded to bf16.
//
// A row is held in registers between its sum of squares and its output, one
// 16-byte load per 8 columns; 16 lanes hold a group and find its largest value by
// four exchanges. A NaN makes its group's scale NaN, an infinity makes it
// infinite. Bound by HBM: 7 bytes a column with the addition (8192 x 4096: 40.7 us,
// 5.8 TB/s; 16 rows 3.2 us), 3 without (23.4 us, 4.3 TB/s).
#include <math.h>

#include "pdk_common.h"

namespace {

using pdk::v8;

constexpr int kMaxH = 8192;
constexpr float kTop = 448.f, kLeast = 0x1p-100f;

__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ void unpack(const v8& a, float (&f)[8]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[2 * w] = pdk::bf16_to_f32(a.w[w] & 0xffffu);
    f[2 * w + 1] = __uint_as_float(a.w[w] & 0xffff0000u);
  }
}

// A lane's 8 values of a group that lies over 16 lanes: stored in 8 bits, the
// scale by the first lane. All 16 lanes must be active.
__device__ __forceinline__ void store_group(const float (&y)[8], uint8_t* to, float* scale) {
  float top = __builtin_fabsf(y[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) top = vmax(top, __builtin_fabsf(y[e]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) top = vmax(top, __shfl_xor(top, o));
  const float s = vmax(top, kLeast) / kTop, r = 1.f / s;
  // y / s rounded once: the product with 1 / s and what it leaves of y. Quotients of bf16
  // values often lie right between two of 8 bits, where the product alone (rounded twice)
  // goes to the wrong one. An infinite scale leaves nothing: 0 for what is finite.
  const float left = s == INFINITY ? 0.f : s;
  float z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = y[e] * r;
    z[e] = __builtin_fmaf(__builtin_fmaf(-q, left, y[e]), r, q);
  }
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(z[4], z[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(z[6], z[7], hi, true);
  *reinterpret_cast<int2*>(to) = make_int2(lo, hi);
  if ((threadIdx.x & 15) == 0) *scale = s;
}

// One workgroup per row; a thread has the chunks of 8 columns tid, tid + 256, ...
// kNorm 0: the row itself in 8 bits, 1: its norm, 2: the norm of its sum with add.
template <int kNorm, int kChunks>
__global__ __launch_bounds__(256) void norm_fp8_kernel(const uint16_t* x, const uint16_t* add,
                                                       const uint16_t* w, float eps, int H, int64_t ld,
                                                       uint16_t* sum, uint8_t* out, float* scales,
                                                       int64_t scale_ld) {
  __shared__ float part[4];
  const int64_t row = blockIdx.x;
  const int n8 = H >> 3, tid = threadIdx.x;
  // What the sum takes the place of is not read again: a stream leaves the caches to what is
  // written (8192 x 4096: 39.6 us, without and with add behind the loop 46.9).
  constexpr bool kSum = kNorm == 2;
  v8 keep[kChunks], more[kChunks], gain[kChunks];
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int c = tid + 256 * j;
    keep[j] = c < n8 ? pdk::ld16_as<kSum>(x + row * ld + 8 * c) : pdk::zero8();
    if (kSum) more[j] = c < n8 ? pdk::ld16_stream(add + row * H + 8 * c) : pdk::zero8();
    if (kNorm) gain[j] = c < n8 ? pdk::ld16(w + 8 * c) : pdk::zero8();
  }
  float r = 1.f;
  if (kNorm) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int c = tid + 256 * j;
      float f[8];
      unpack(keep[j], f);
      if (kSum && c < n8) {
        float g[8];
        unpack(more[j], g);
#pragma unroll
        for (int k = 0; k < 4; ++k) keep[j].w[k] = pdk::pack_bf16x2_rne(f[2 * k] + g[2 * k], f[2 * k + 1] + g[2 * k + 1]);
        pdk::st16(sum + row * H + 8 * c, keep[j]);
        unpack(keep[j], f);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(f[e], f[e], ss);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) ss += __shfl_xor(ss, o);
    if ((tid & 63) == 0) part[tid >> 6] = ss;
    __syncthreads();
    r = rsqrtf((part[0] + part[1] + part[2] + part[3]) / (float)H + eps);
  }
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int c = tid + 256 * j;
    if (c >= n8) continue;                // H % 128 == 0: 16 lanes together
    float y[8], g[8];
    unpack(keep[j], y);
    if (kNorm) {
      unpack(gain[j], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = y[e] * r * g[e];
    }
    store_group(y, out + row * H + 8 * c, scales + (int64_t)(c >> 4) * scale_ld + row);
  }
}

template <int kNorm>
int launch(const uint16_t* x, const uint16_t* add, const uint16_t* w, float eps, int T, int H,
           int64_t ld, uint16_t* sum, uint8_t* out, float* scales, int64_t scale_ld, uintptr_t stream) {
  const auto kern = H <= 2048 ? norm_fp8_kernel<kNorm, 1>
                    : H <= 4096 ? norm_fp8_kernel<kNorm, 2> : norm_fp8_kernel<kNorm, 4>;
  hipLaunchKernelGGL(kern, dim3(T), dim3(256), 0, pdk::as_stream(stream), x, add, w, eps, H, ld, sum,
                     out, scales, scale_ld);
  return pdk::check_launch("norm_fp8_kernel");
}

}  // namespace

extern "C" int pdk_rmsnorm_fp8(const uint16_t* x, const uint16_t* add, const uint16_t* weight, int T,
                               int H, float eps, uint16_t* sum_out, uint8_t* out, float* scales,
                               int64_t scale_ld, uintptr_t stream) {
  pdk::clear_error();
  PDK_REQUIRE(T >= 0 && T <= (1 << 24), "T must be in [0, 2^24] (got %d)", T);
  PDK_REQUIRE(H >= 128 && H % 128 == 0 && H <= kMaxH, "H must be a multiple of 128 in [128, %d] (got %d)",
              kMaxH, H);
  PDK_REQUIRE(eps >= 0.f, "eps must be >= 0");
  PDK_REQUIRE(scale_ld >= T, "scale_ld must be at least T");
  if (T == 0) return PDK_OK;
  PDK_REQUIRE(x && weight && out && scales && (!add || sum_out), "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(x) && pdk::aligned16(add) && pdk::aligned16(weight) &&
                  pdk::aligned16(sum_out) && pdk::aligned16(out),
              "tensors must be 16-byte aligned");
  return add ? launch<2>(x, add, weight, eps, T, H, H, sum_out, out, scales, scale_ld, stream)
             : launch<1>(x, nullptr, weight, eps, T, H, H, nullptr, out, scales, scale_ld, stream);
}

namespace {

// Rows of K columns in 8 bits, 8 columns a thread. kGated: of silu(g) * u, a row of x
// being g's K columns and then u's. 8192 x 4096 plain 21.8 us, 8192 x 14336 gated 121.5 (4.7 and 4.8
// TB/s; 16 rows 2.0 and 2.4): beside the bytes the row's division in 64 bits and, gated, a division
// for each value.
template <bool kGated>
__global__ __launch_bounds__(256) void quantize_fp8_kernel(const uint16_t* x, int64_t ld, int T, int K,
                                                           uint8_t* out, float* scales,
                                                           int64_t scale_ld) {
  const int n8 = K >> 3;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / n8;
  const int c = (int)(id - row * n8);
  if (row >= T) return;                   // K % 128 == 0: 16 lanes together
  float y[8];
  unpack(pdk::ld16(x + row * ld + 8 * c), y);
  if (kGated) {
    float u[8];
    unpack(pdk::ld16(x + row * ld + K + 8 * c), u);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = y[e] / (1.f + __expf(-y[e])) * u[e];
  }
  store_group(y, out + row * K + 8 * c, scales + (int64_t)(c >> 4) * scale_ld + row);
}

template <bool kGated>
int quantize(const uint16_t* x, int64_t ld, int T, int K, uint8_t* out, float* scales,
             int64_t scale_ld, uintptr_t stream) {
  pdk::clear_error();
  PDK_REQUIRE(T >= 0 && T <= (1 << 24), "T must be in [0, 2^24] (got %d)", T);
  PDK_REQUIRE(K >= 128 && K % 128 == 0 && K <= (1 << 20),
              "the columns must be a multiple of 128 in [128, 2^20] (got %d)", K);
  PDK_REQUIRE(ld >= (kGated ? 2ll : 1ll) * K && ld % 8 == 0, "ld must be a multiple of 8 and hold a row");
  PDK_REQUIRE(scale_ld >= T, "scale_ld must be at least T");
  const int64_t blocks = ((int64_t)T * (K / 8) + 255) / 256;
  PDK_REQUIRE(blocks < (1ll << 31), "launch too large");
  if (T == 0) return PDK_OK;
  PDK_REQUIRE(x && out && scales, "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(x) && pdk::aligned16(out), "tensors must be 16-byte aligned");
  hipLaunchKernelGGL(quantize_fp8_kernel<kGated>, dim3((unsigned)blocks), dim3(256), 0,
                     pdk::as_stream(stream), x, ld, T, K, out, scales, scale_ld);
  return pdk::check_launch("quantize_fp8_kernel");
}

}  // namespace

extern "C" int pdk_quantize_fp8(const uint16_t* x, int64_t ld, int T, int K, uint8_t* out,
                                float* scales, int64_t scale_ld, uintptr_t stream) {
  return quantize<false>(x, ld, T, K, out, scales, scale_ld, stream);
}

extern "C" int pdk_swiglu_fp8(const uint16_t* gate_up, int64_t ld, int T, int M, uint8_t* out,
                              float* scales, int64_t scale_ld, uintptr_t stream) {
  return quantize<true>(gate_up, ld, T, M, out, scales, scale_ld, stream);
}
