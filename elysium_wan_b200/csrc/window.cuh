// What the forward and backward of window attention share.
#pragma once

#include "common.cuh"

namespace ewb {

constexpr float kLog2eWa = 1.4426950408889634f;
constexpr uint32_t kWaChunk = 16384;  // 128 rows x 64 columns of bf16, 128-byte swizzle

__device__ __forceinline__ float ex2_wa(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bits c < n of a 32-bit word.
__device__ __forceinline__ uint32_t bits_below(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// The key tiles (128 keys) that the rows [q0, q1] can see: [0, ns) and [w0, e].
// The host bounds window and sinks by the sequence length, so that sums of
// them and positions stay inside 32 bits.
struct TileList {
  int ns, w0, e;
  __device__ __forceinline__ TileList(int q0, int q1, int window, int sinks) {
    w0 = max(0, q0 - window + 1) >> 7;
    e = q1 >> 7;
    ns = min((sinks + 127) >> 7, w0);
  }
  __device__ __forceinline__ int count() const { return ns + e - w0 + 1; }
  __device__ __forceinline__ int tile(int k) const { return k < ns ? k : w0 + (k - ns); }
};

// 64-column chunks of a head and the 16-wide k-steps of chunk c.
template <int HD>
struct HeadChunks {
  static constexpr int kCount = (HD + 63) / 64;
  __device__ static constexpr int steps(int c) { return (HD - 64 * c >= 64 ? 64 : HD - 64 * c) / 16; }
};

}  // namespace ewb
