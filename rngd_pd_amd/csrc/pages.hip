// Whole blocks of the paged KV cache copied inside it, gfx950: what sharing a
// prompt between requests (its last, partly filled block), compacting the cache
// and beam search's reordering move.
//
// One launch copies every pair's K and V block in all layers. The pairs lie in
// host memory (block tables are the host's) and travel as kernel arguments, so a
// call needs no device array, no copy to the device and no synchronisation, and
// a captured graph holds them.
//
// Bound by HBM: each byte is read and written once. Consecutive workgroups copy
// pairs of one layer (a region of tens of MB, whose address translations stay at
// hand) rather than layers of one pair, one 16-byte vector per lane, without
// keeping the lines: 512 pairs of 32 layers (2.1 GB moved) 431 -> 379 us, 5.7 TB/s;
// with four vectors per lane 396, kept in the caches 409. Up to 16 pairs (a fork,
// whose blocks are read again in the next step) stay in the caches: 3 pairs 3.2 us
// on the GPU.
#include <algorithm>
#include <new>
#include <vector>

#include "pdk_common.h"

namespace {

constexpr int kPairs = 448;               // per launch: 3.5 KiB of the 4 KiB of arguments
constexpr int kFew = 16;                  // and of a launch of few

// The launch's arguments are copied by the host at every call: few pairs travel
// in a small struct (3 pairs, an eager call 9.4 -> 7 us).
template <int kN>
struct Pairs {
  int32_t src[kN], dst[kN];
};

// grid: x = chunk of a block, y = pair, z = 2 * layer + (0 for K, 1 for V).
template <int kN, int kUnits, bool kStream>
__global__ __launch_bounds__(256) void copy_blocks_kernel(uint16_t* ck, uint16_t* cv,
                                                          int64_t layer_stride, int block_units,
                                                          Pairs<kN> p) {
  uint16_t* base = (blockIdx.z & 1 ? cv : ck) + (int64_t)(blockIdx.z >> 1) * layer_stride;
  const int64_t block = (int64_t)block_units * 8;
  const uint16_t* from = base + p.src[blockIdx.y] * block;
  uint16_t* to = base + p.dst[blockIdx.y] * block;
  const int u0 = blockIdx.x * (256 * kUnits) + threadIdx.x;
  pdk::v8 r[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i)
    if (u0 + 256 * i < block_units) r[i] = pdk::ld16_as<kStream>(from + (int64_t)(u0 + 256 * i) * 8);
#pragma unroll
  for (int i = 0; i < kUnits; ++i)
    if (u0 + 256 * i < block_units) pdk::st16_as<kStream>(to + (int64_t)(u0 + 256 * i) * 8, r[i]);
}

// PDK_OK if the pairs' ids are blocks of the cache, no block is written twice
// and none is both read and written, so that the copies' order does not matter.
int check_pairs(const int32_t* src, const int32_t* dst, int n, int num_blocks) {
  std::vector<uint64_t> written(((int64_t)num_blocks + 63) / 64, 0);
  auto bit = [](int32_t id) { return 1ull << (id & 63); };
  for (int i = 0; i < n; ++i) {
    PDK_REQUIRE(src[i] >= 0 && src[i] < num_blocks && dst[i] >= 0 && dst[i] < num_blocks,
                "pair %d: block %d -> %d outside [0, %d)", i, src[i], dst[i], num_blocks);
    PDK_REQUIRE(!(written[dst[i] >> 6] & bit(dst[i])), "block %d is the destination of two pairs",
                dst[i]);
    written[dst[i] >> 6] |= bit(dst[i]);
  }
  for (int i = 0; i < n; ++i)
    PDK_REQUIRE(!(written[src[i] >> 6] & bit(src[i])), "block %d is both a source and a destination",
                src[i]);
  return PDK_OK;
}

template <int kN, int kUnits, bool kStream>
int launch(uint16_t* cache_k, uint16_t* cache_v, int64_t layer_stride, int n_layers, int units,
           const int32_t* src, const int32_t* dst, int n, hipStream_t st) {
  Pairs<kN> p{};
  std::copy(src, src + n, p.src);
  std::copy(dst, dst + n, p.dst);
  constexpr int kChunk = 256 * kUnits;      // 16-byte units of one workgroup
  const auto kern = copy_blocks_kernel<kN, kUnits, kStream>;
  hipLaunchKernelGGL(kern, dim3((units + kChunk - 1) / kChunk, n, 2 * n_layers), dim3(256),
                     0, st, cache_k, cache_v, layer_stride, units, p);
  return pdk::check_launch("copy_blocks_kernel");
}

}  // namespace

extern "C" int pdk_copy_blocks(uint16_t* cache_k, uint16_t* cache_v, int64_t cache_layer_stride,
                               int n_layers, int num_blocks, int n_kv_heads, int head_dim,
                               const int32_t* src, const int32_t* dst, int n, uintptr_t stream) {
  pdk::clear_error();
  PDK_REQUIRE(n >= 0, "n must be >= 0 (got %d)", n);
  PDK_REQUIRE(cache_k && cache_v && (n == 0 || (src && dst)), "null pointer argument");
  PDK_REQUIRE(pdk::aligned16(cache_k) && pdk::aligned16(cache_v), "caches must be 16-byte aligned");
  PDK_REQUIRE(n_layers >= 1 && n_layers <= 32767 && num_blocks >= 1,
              "n_layers or num_blocks out of range");
  PDK_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 65535 && head_dim >= 1 && head_dim <= 4096,
              "n_kv_heads or head_dim out of range");
  const int64_t block = (int64_t)n_kv_heads * PDK_BLOCK_SIZE * head_dim;
  PDK_REQUIRE(cache_layer_stride % 8 == 0 &&
                  (n_layers == 1 || cache_layer_stride >= (int64_t)num_blocks * block),
              "the layer stride must be a multiple of 8 and hold num_blocks blocks");
  try {
    if (int rc = check_pairs(src, dst, n, num_blocks)) return rc;
  } catch (const std::bad_alloc&) {
    pdk::set_error("no host memory to check %d blocks", num_blocks);
    return PDK_ENOMEM;
  }
  const int units = (int)(block / 8);
  for (int at = 0; at < n; at += kPairs) {
    const int m = std::min(n - at, kPairs);
    const auto go = m <= kFew ? launch<kFew, 2, false> : launch<kPairs, 1, true>;
    if (int rc = go(cache_k, cache_v, cache_layer_stride, n_layers, units, src + at, dst + at, m,
                    pdk::as_stream(stream)))
      return rc;
  }
  return PDK_OK;
}
