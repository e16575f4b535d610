// Backward of attention in a sliding window with sinks (see
// window_attention.cu for the mask), on the 5th-generation tensor cores.
//
//   P = 2^(x log2 e - lse2);  D = rowsum(dO o);  dV = P^T dO;  dP = dO V^T;
//   dS = P (dP - D);  dQ = dS K / sqrt(hd);  dK = dS^T Q / sqrt(hd)
//
// Two passes, so that every output has one owner and one order of summation
// (no atomics; a kv head's gradient sums its query heads in head order): one
// over key tiles for dK and dV, one over query tiles for dQ. S and dP are so
// formed twice: 7 products for 5.
//
// A first kernel writes D and the statistic into rows padded to 128, with lse2 =
// +inf past the sequence's length: P is then 0 there without a test.
//
// A sinks' key tile is seen by every later query, so its work is split along the
// queries into parts of a common tile's length. Each part leaves fp32 sums,
// which a last kernel adds in order.
#include "common.cuh"
#include "gemm.h"
#include "kernels.h"
#include "window.cuh"

#include <algorithm>

namespace ewb {
namespace {

constexpr int kWbThreads = 320;  // producer, MMA issuer, two warpgroups of softmax warps

// ---------------------------------------------------------------- D and lse2
// One half warp per (row, head): 16 bytes of o and dO a lane.
__global__ void __launch_bounds__(256)
    window_dot_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ dout,
                      int64_t ldo, const float* __restrict__ lse2, const int* __restrict__ lengths,
                      float* __restrict__ Lp, float* __restrict__ Dp, int S, int Sp, int H, int HD,
                      int64_t units) {
  const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 16 + half;  // (b, s, h), h fastest
  if (u >= units) return;
  const int h = static_cast<int>(u % H);
  const int64_t bs = u / H;
  const int s = static_cast<int>(bs % Sp);
  const int64_t b = bs / Sp;
  const int n = lengths != nullptr ? min(max(lengths[b], 0), S) : S;
  float d = 0.f;
  if (s < n && 8 * l < HD) {
    const int64_t row = b * S + s;
    const uint4 x = *reinterpret_cast<const uint4*>(o + (row * H + h) * HD + 8 * l);
    const uint4 y = *reinterpret_cast<const uint4*>(dout + row * ldo + static_cast<int64_t>(h) * HD + 8 * l);
    float f[8], g[8];
    unpack8_fmt(x, kFmtBf16, 1.0f, f);
    unpack8_fmt(y, kFmtBf16, 1.0f, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) d = fmaf(f[e], g[e], d);
  }
#pragma unroll
  for (int k = 8; k > 0; k >>= 1) d += __shfl_xor_sync(0xffffffffu, d, k);
  if (l == 0) {
    const int64_t at = (b * H + h) * Sp + s;
    Dp[at] = d;
    Lp[at] = s < n ? lse2[(b * H + h) * S + s] : INFINITY;
  }
}

// ---------------------------------------------------------------- dK, dV
// A CTA owns 128 keys of one (batch, kv head) and walks (query head of the
// group, block of 64 queries): S^T = K Q^T and dP^T = V dO^T into one of two
// TMEM buffers, P^T and dS^T (bf16) into shared memory, then dV += P^T dO and
// dK += dS^T Q in TMEM. S^T / dP^T of the next pair start before the
// gradients of this one. TMEM: S^T x2 | dP^T x2 (64 columns each) | dV | dK.
constexpr uint32_t kKvOffK = 0, kKvOffV = 32768, kKvOffQ = 65536, kKvOffDO = 98304;
constexpr uint32_t kKvOffL = 131072, kKvOffD = 131584, kKvOffP = 132096 + 1024, kKvOffS = kKvOffP + 32768;
constexpr uint32_t kKvOffBar = kKvOffS + 32768;
constexpr int kKvSmem = kKvOffBar + 256 + 1024;
static_assert(kKvOffP % 1024 == 0 && kKvOffS % 1024 == 0, "swizzled tiles start on 1024 bytes");

struct KvPlan {
  int window, sinks;  // bounded by S
  int sink_tiles;     // key tiles with a sink
  int parts;          // parts of a sinks' tile
  int span;           // query blocks of a part
};

template <int HD>
__global__ void __launch_bounds__(kWbThreads, 1)
    window_dkdv_kernel(const __grid_constant__ CUtensorMap map_kv,
                       const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_do, const float* __restrict__ Lp,
                       const float* __restrict__ Dp, const int* __restrict__ lengths,
                       __nv_bfloat16* __restrict__ dqkv, float* __restrict__ part_ws, int S, int Sp,
                       int H, int Hkv, KvPlan plan, float scale_log2, float scale, int* status) {
  using C = HeadChunks<HD>;
  constexpr uint32_t kTile = C::kCount * kWaChunk;  // 128 rows
  constexpr uint32_t kBlk = C::kCount * 8192;       // 64 rows
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kKvOffBar);
  uint64_t* kvfull = bars;
  uint64_t* qfull = bars + 1;  // [2]
  uint64_t* done = bars + 3;   // [2]  gradient MMAs of a pair finished (stage and P/dS free)
  uint64_t* sfull = bars + 5;  // [2]
  uint64_t* sfree = bars + 7;  // [2]
  uint64_t* pfull = bars + 9;  // [2]
  uint64_t* fin = bars + 11;
  uint64_t* drain = bars + 12;
  uint64_t* landed = bars + 13;  // a query block that the producer clears
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);

  const int hk = blockIdx.x, bz = blockIdx.z;
  const int u = blockIdx.y, su = plan.sink_tiles * plan.parts;
  const int kt = u < su ? u / plan.parts : u - su + plan.sink_tiles;  // earliest keys first
  const int part = u < su ? u % plan.parts : 0;
  const bool split = u < su && plan.parts > 1;
  const int n = lengths != nullptr ? min(max(lengths[bz], 0), S) : S;
  const int k0 = kt * 128, rep = H / Hkv;
  // query blocks that see a key of this tile, this part's share of them
  int i0 = 2 * kt, i1 = 0;
  if (k0 < n) {
    const int last = k0 < plan.sinks ? n : min(n, k0 + 127 + plan.window);
    i1 = (last + 63) / 64;
    if (split) {
      i0 += part * plan.span;
      i1 = min(i1, i0 + plan.span);
    }
  }
  const int nqs = max(0, i1 - i0);
  const int steps = rep * nqs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    mbar_init(kvfull, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&qfull[i], 1);
      mbar_init(&done[i], 1);
      mbar_init(&sfull[i], 1);
      mbar_init(&sfree[i], 8);
      mbar_init(&pfull[i], 8);
    }
    mbar_init(fin, 1);
    mbar_init(drain, 1);
    mbar_init(landed, 1);
    fence_mbar_init();
    tma_prefetch_desc(&map_kv);
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_do);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    const int clear = (n < S && (n & 63)) ? n >> 6 : -1;  // the block that holds row n
    bool ok = true;
    int issued = 0, cleared = 0;
    if (lane == 0 && steps > 0) {
      mbar_arrive_expect_tx(kvfull, 2 * kTile);
      for (int c = 0; c < C::kCount; ++c) {
        tma_load_3d(smem + kKvOffK + c * kWaChunk, &map_kv, kvfull, (H + hk) * HD + c * 64, k0, bz, status);
        tma_load_3d(smem + kKvOffV + c * kWaChunk, &map_kv, kvfull, (H + Hkv + hk) * HD + c * 64, k0, bz,
                    status);
      }
    }
    for (int t = 0; t < steps && ok; ++t) {
      const int sb = t & 1;
      const int h = hk * rep + t / nqs, i = i0 + t % nqs;
      uint8_t* sq = smem + kKvOffQ + sb * 16384;
      uint8_t* so = smem + kKvOffDO + sb * 16384;
      uint64_t* bar = i == clear ? landed : &qfull[sb];
      if (lane == 0) {
        ok = mbar_wait(&done[sb], ((t >> 1) & 1) ^ 1, status, kStatusTimeoutSmemEmpty);
        if (ok) {
          mbar_arrive_expect_tx(bar, 2 * kBlk + 512);
          for (int c = 0; c < C::kCount; ++c) {
            tma_load_3d(sq + c * 8192, &map_q, bar, h * HD + c * 64, i * 64, bz, status);
            tma_load_3d(so + c * 8192, &map_do, bar, h * HD + c * 64, i * 64, bz, status);
          }
          const int64_t li = (static_cast<int64_t>(bz) * H + h) * Sp + i * 64;
          bulk_load(smem + kKvOffL + sb * 256, Lp + li, 256, bar);
          bulk_load(smem + kKvOffD + sb * 256, Dp + li, 256, bar);
          issued = t + 1;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (ok && i == clear) {
        if (!mbar_wait(landed, cleared & 1, status, kStatusTimeoutSmemFull)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        ++cleared;
        const int r0 = n & 63, w = (64 - r0) * 8;
        for (int k = lane; k < 2 * w * C::kCount; k += 32) {
          const int c = k / w;
          uint8_t* base = (c & 1) ? so : sq;
          *reinterpret_cast<uint4*>(base + (c >> 1) * 8192 + r0 * 128 + (k - c * w) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&qfull[sb]);
      }
    }
    if (lane == 0 && steps > 0) {
      mbar_wait(kvfull, 0, nullptr, kStatusTimeoutDrain);
      // a cleared block has landed before it was handed over
      for (int t = issued - 1; t >= 0 && t >= issued - 2; --t)
        if (i0 + t % nqs != clear) mbar_wait(&qfull[t & 1], (t >> 1) & 1, nullptr, kStatusTimeoutDrain);
        else if (!ok) mbar_wait(landed, (cleared + 1) & 1, nullptr, kStatusTimeoutDrain);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t IS = idesc_bf16_f32(128, 64, false, false);
      constexpr uint32_t IG = idesc_bf16_f32(128, HD, false, true);
      const uint32_t k_addr = smem_u32(smem + kKvOffK), v_addr = smem_u32(smem + kKvOffV);
      bool ok = steps > 0 && mbar_wait(kvfull, 0, status, kStatusTimeoutSmemFull);
      auto grads = [&](int t) -> bool {
        const int sb = t & 1;
        if (!mbar_wait(&pfull[sb], (t >> 1) & 1, status, kStatusTimeoutTmemFull)) return false;
        tc_fence_after();
        const uint32_t p_addr = smem_u32(smem + kKvOffP + sb * 16384);
        const uint32_t s_addr = smem_u32(smem + kKvOffS + sb * 16384);
        const uint32_t q_addr = smem_u32(smem + kKvOffQ + sb * 16384);
        const uint32_t o_addr = smem_u32(smem + kKvOffDO + sb * 16384);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          umma_f16(tmem + 256, sdesc_sw128(p_addr + kk * 32, 16, 1024),
                   sdesc_sw128(o_addr + kk * 2048, 8192, 1024), IG, (t > 0 || kk > 0) ? 1u : 0u);
          umma_f16(tmem + 384, sdesc_sw128(s_addr + kk * 32, 16, 1024),
                   sdesc_sw128(q_addr + kk * 2048, 8192, 1024), IG, (t > 0 || kk > 0) ? 1u : 0u);
        }
        umma_commit(&done[sb]);
        return true;
      };
      for (int t = 0; t < steps && ok; ++t) {
        const int sb = t & 1;
        const uint32_t ph = (t >> 1) & 1;
        if (!mbar_wait(&qfull[sb], ph, status, kStatusTimeoutSmemFull) ||
            !mbar_wait(&sfree[sb], ph ^ 1, status, kStatusTimeoutTmemEmpty)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t q_addr = smem_u32(smem + kKvOffQ + sb * 16384);
        const uint32_t o_addr = smem_u32(smem + kKvOffDO + sb * 16384);
#pragma unroll
        for (int c = 0; c < C::kCount; ++c)
#pragma unroll
          for (int kk = 0; kk < C::steps(c); ++kk) {
            const uint32_t acc = (c > 0 || kk > 0) ? 1u : 0u;
            umma_f16(tmem + sb * 64, sdesc_sw128(k_addr + c * kWaChunk + kk * 32, 16, 1024),
                     sdesc_sw128(q_addr + c * 8192 + kk * 32, 16, 1024), IS, acc);
            umma_f16(tmem + 128 + sb * 64, sdesc_sw128(v_addr + c * kWaChunk + kk * 32, 16, 1024),
                     sdesc_sw128(o_addr + c * 8192 + kk * 32, 16, 1024), IS, acc);
          }
        umma_commit(&sfull[sb]);
        if (t > 0 && !grads(t - 1)) {
          ok = false;
          break;
        }
      }
      if (ok && grads(steps - 1)) umma_commit(fin);
      umma_commit(drain);
      mbar_wait(drain, 0, nullptr, kStatusTimeoutDrain);
    }
  } else {
    const int wq = warp & 3;
    const int g = (warp - 2) >> 2;  // this warpgroup's half of the 64 query columns
    const int q0 = g * 32;
    const int r = wq * 32 + lane;  // key row within the tile = TMEM lane
    const int kpos = k0 + r;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    bool ok = true;
    for (int t = 0; t < steps; ++t) {
      const int sb = t & 1;
      const uint32_t ph = (t >> 1) & 1;
      const int i = i0 + t % nqs;
      if (!mbar_wait(&sfull[sb], ph, status, kStatusTimeoutTmemFull) ||
          !mbar_wait(&qfull[sb], ph, status, kStatusTimeoutSmemFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sv[32], pv[32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_ld16(tmem + sb * 64 + q0 + lanes + c * 16, sv + c * 16);
        tmem_ld16(tmem + 128 + sb * 64 + q0 + lanes + c * 16, pv + c * 16);
      }
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sfree[sb]);
      // P^T / dS^T buffer sb was read by the gradients of pair t - 2.
      if (!mbar_wait(&done[sb], ph ^ 1, status, kStatusTimeoutSmemEmpty)) {
        ok = false;
        break;
      }
      // queries of this half that see key kpos: from kpos on, below kpos + window
      uint32_t vis = 0xffffffffu;
      const bool whole = i * 64 >= k0 + 127 && k0 + 128 <= n &&
                         (i * 64 + 63 - k0 < plan.window || k0 + 128 <= plan.sinks);
      if (!whole) {
        const int c0 = i * 64 + q0;
        vis = kpos < n ? ~bits_below(kpos - c0) : 0u;
        if (kpos >= plan.sinks) vis &= bits_below(kpos + plan.window - c0);
      }
      const float* Ls = reinterpret_cast<const float*>(smem + kKvOffL + sb * 256) + q0;
      const float* Ds = reinterpret_cast<const float*>(smem + kKvOffD + sb * 256) + q0;
      uint8_t* prow = smem + kKvOffP + sb * 16384 + r * 128;
      uint8_t* srow = smem + kKvOffS + sb * 16384 + r * 128;
#pragma unroll
      for (int u4 = 0; u4 < 4; ++u4) {
        const int u8 = g * 4 + u4;  // 16-byte unit of the 64-query row
        uint32_t pk[4], dk[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float pp[2], dd[2];
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const int q = u4 * 8 + 2 * e + z;  // within this half
            const bool see = (vis >> q) & 1u;
            const float p = ex2_wa(__uint_as_float(sv[q]) * scale_log2 - Ls[q]);
            pp[z] = see ? p : 0.f;
            dd[z] = see ? p * (__uint_as_float(pv[q]) - Ds[q]) : 0.f;
          }
          pk[e] = pack_bf16x2(pp[0], pp[1]);
          dk[e] = pack_bf16x2(dd[0], dd[1]);
        }
        const uint32_t off = static_cast<uint32_t>((u8 ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(prow + off) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        *reinterpret_cast<uint4*>(srow + off) = make_uint4(dk[0], dk[1], dk[2], dk[3]);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[sb]);
    }
    if (ok && steps > 0) ok = mbar_wait(fin, 0, status, kStatusTimeoutTmemFull);
    if (ok) {  // warpgroup 0 writes dV, warpgroup 1 dK
      tc_fence_after();
      const int ldq = (H + 2 * Hkv) * HD;
      __nv_bfloat16* out = dqkv + (static_cast<size_t>(bz) * S + kpos) * ldq + (g ? H + hk : H + Hkv + hk) * HD;
      float* sum = part_ws;
      if (split)
        sum += ((((static_cast<size_t>(bz) * Hkv + hk) * plan.sink_tiles + kt) * plan.parts + part) * 128 + r) *
                   (2 * HD) + g * HD;
      const float mul = g ? scale : 1.0f;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t v[16];
        if (steps > 0) {
          tmem_ld16(tmem + 256 + g * 128 + lanes + c * 16, v);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = 0u;
        }
        if (split) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(sum + c * 16 + e * 4) = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
        } else if (kpos < S) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(v[8 * e]) * mul, __uint_as_float(v[8 * e + 1]) * mul);
            w.y = pack_bf16x2(__uint_as_float(v[8 * e + 2]) * mul, __uint_as_float(v[8 * e + 3]) * mul);
            w.z = pack_bf16x2(__uint_as_float(v[8 * e + 4]) * mul, __uint_as_float(v[8 * e + 5]) * mul);
            w.w = pack_bf16x2(__uint_as_float(v[8 * e + 6]) * mul, __uint_as_float(v[8 * e + 7]) * mul);
            *reinterpret_cast<uint4*>(out + c * 16 + e * 8) = w;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dK, dV of the sinks' tiles: the parts' sums, added in order. One thread per
// four columns of a row ([dV | dK], 2 HD wide).
__global__ void __launch_bounds__(256)
    window_sinks_kernel(const float* __restrict__ ws, __nv_bfloat16* __restrict__ dqkv, int S, int H,
                        int Hkv, int HD, int sink_tiles, int parts, float scale, int64_t units) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= units) return;
  const int per = 2 * HD / 4;
  const int c = static_cast<int>(t % per) * 4;
  int64_t rest = t / per;
  const int r = static_cast<int>(rest % 128);
  rest /= 128;  // (b, hk, kt)
  const int kt = static_cast<int>(rest % sink_tiles);
  const int64_t bh = rest / sink_tiles;
  const int hk = static_cast<int>(bh % Hkv);
  const int64_t b = bh / Hkv;
  const int kpos = kt * 128 + r;
  if (kpos >= S) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = 0; p < parts; ++p) {
    const float4 v = *reinterpret_cast<const float4*>(ws + ((rest * parts + p) * 128 + r) * (2 * HD) + c);
    a.x += v.x;
    a.y += v.y;
    a.z += v.z;
    a.w += v.w;
  }
  const bool key = c >= HD;
  const float mul = key ? scale : 1.0f;
  __nv_bfloat16* out = dqkv + (b * S + kpos) * static_cast<int64_t>(H + 2 * Hkv) * HD +
                       (key ? (H + hk) * HD + c - HD : (H + Hkv + hk) * HD + c);
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(a.x * mul, a.y * mul), pack_bf16x2(a.z * mul, a.w * mul));
}

// ---------------------------------------------------------------- dQ
// A CTA owns 128 query rows of one (batch, head) and walks the key tiles they
// see: S = Q K^T and dP = dO V^T into TMEM, dS (bf16) into shared memory, then
// dQ += dS K in TMEM, issued after S / dP of the next tile. The K tile serves
// as both a K-major (S) and an MN-major (dQ) operand. TMEM: S | dP | dQ.
constexpr uint32_t kDqOffQ = 0, kDqOffDO = 32768, kDqOffK = 65536, kDqOffV = 131072;
constexpr uint32_t kDqOffS = 196608, kDqOffBar = 229376;
constexpr int kDqSmem = 229376 + 256 + 1024;

template <int HD>
__global__ void __launch_bounds__(kWbThreads, 1)
    window_dq_kernel(const __grid_constant__ CUtensorMap map_qkv,
                     const __grid_constant__ CUtensorMap map_do, const float* __restrict__ Lp,
                     const float* __restrict__ Dp, const int* __restrict__ lengths,
                     __nv_bfloat16* __restrict__ dqkv, int S, int Sp, int H, int Hkv, int window,
                     int sinks, float scale_log2, float scale, int* status) {
  using C = HeadChunks<HD>;
  constexpr uint32_t kTile = C::kCount * kWaChunk;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kDqOffBar);
  uint64_t* qfull = bars;
  uint64_t* kfull = bars + 1;   // [2]
  uint64_t* kempty = bars + 3;  // [2]
  uint64_t* sfull = bars + 5;
  uint64_t* sfree = bars + 6;   // S read into registers
  uint64_t* pfull = bars + 7;
  uint64_t* dsfree = bars + 8;  // dQ MMA of the previous tile finished
  uint64_t* drain = bars + 9;
  uint64_t* dpfree = bars + 10;  // dP read
  uint64_t* landed = bars + 11;  // the K tile that the producer clears
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 12);

  const int h = blockIdx.x, bz = blockIdx.z;
  const int hk = h / (H / Hkv);
  const int q0 = (gridDim.y - 1 - blockIdx.y) * 128;  // the latest rows first: most tiles
  const int n = lengths != nullptr ? min(max(lengths[bz], 0), S) : S;
  const TileList list(q0, min(q0 + 127, max(n, 1) - 1), window, sinks);
  const int tiles = q0 < n ? list.count() : 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    mbar_init(qfull, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&kempty[i], 1);
    }
    mbar_init(sfull, 1);
    mbar_init(sfree, 8);
    mbar_init(dpfree, 8);
    mbar_init(pfull, 8);
    mbar_init(dsfree, 1);
    mbar_init(drain, 1);
    mbar_init(landed, 1);
    fence_mbar_init();
    tma_prefetch_desc(&map_qkv);
    tma_prefetch_desc(&map_do);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    const int clear = (n < S && (n & 127)) ? n >> 7 : -1;
    bool ok = true;
    int issued = 0;
    if (lane == 0 && tiles > 0) {
      mbar_arrive_expect_tx(qfull, 2 * kTile);
      for (int c = 0; c < C::kCount; ++c) {
        tma_load_3d(smem + kDqOffQ + c * kWaChunk, &map_qkv, qfull, h * HD + c * 64, q0, bz, status);
        tma_load_3d(smem + kDqOffDO + c * kWaChunk, &map_do, qfull, h * HD + c * 64, q0, bz, status);
      }
    }
    for (int k = 0; k < tiles && ok; ++k) {
      const int sb = k & 1, j = list.tile(k);
      uint8_t* sk = smem + kDqOffK + sb * 32768;
      uint64_t* bar = j == clear ? landed : &kfull[sb];
      if (lane == 0) {
        ok = mbar_wait(&kempty[sb], ((k >> 1) & 1) ^ 1, status, kStatusTimeoutSmemEmpty);
        if (ok) {
          mbar_arrive_expect_tx(bar, 2 * kTile);
          for (int c = 0; c < C::kCount; ++c) {
            tma_load_3d(sk + c * kWaChunk, &map_qkv, bar, (H + hk) * HD + c * 64, j * 128, bz, status);
            tma_load_3d(smem + kDqOffV + sb * 32768 + c * kWaChunk, &map_qkv, bar,
                        (H + Hkv + hk) * HD + c * 64, j * 128, bz, status);
          }
          issued = k + 1;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (ok && j == clear) {
        if (!mbar_wait(landed, 0, status, kStatusTimeoutSmemFull)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        const int r0 = n & 127, w = (128 - r0) * 8;
        for (int i = lane; i < w * C::kCount; i += 32) {
          const int c = i / w;
          *reinterpret_cast<uint4*>(sk + c * kWaChunk + r0 * 128 + (i - c * w) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kfull[sb]);
      }
    }
    if (lane == 0 && tiles > 0) {
      mbar_wait(qfull, 0, nullptr, kStatusTimeoutDrain);
      for (int k = issued - 1; k >= 0 && k >= issued - 2; --k) {
        if (list.tile(k) == clear) mbar_wait(landed, 0, nullptr, kStatusTimeoutDrain);
        else mbar_wait(&kfull[k & 1], (k >> 1) & 1, nullptr, kStatusTimeoutDrain);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t IS = idesc_bf16_f32(128, 128, false, false);
      constexpr uint32_t IQ = idesc_bf16_f32(128, HD, false, true);
      const uint32_t q_addr = smem_u32(smem + kDqOffQ), o_addr = smem_u32(smem + kDqOffDO);
      const uint32_t ds_addr = smem_u32(smem + kDqOffS);
      bool ok = tiles > 0 && mbar_wait(qfull, 0, status, kStatusTimeoutSmemFull);
      auto dq = [&](int i) -> bool {
        const int sb = i & 1;
        if (!mbar_wait(pfull, i & 1, status, kStatusTimeoutTmemFull)) return false;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(smem + kDqOffK + sb * 32768);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_f16(tmem + 256, sdesc_sw128(ds_addr + (kk >> 2) * kWaChunk + (kk & 3) * 32, 16, 1024),
                   sdesc_sw128(k_addr + kk * 2048, kWaChunk, 1024), IQ, (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&kempty[sb]);
        umma_commit(dsfree);
        return true;
      };
      for (int k = 0; k < tiles && ok; ++k) {
        const int sb = k & 1;
        const uint32_t fr = (k & 1) ^ 1;
        if (!mbar_wait(&kfull[sb], (k >> 1) & 1, status, kStatusTimeoutSmemFull) ||
            !mbar_wait(sfree, fr, status, kStatusTimeoutTmemEmpty)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t k_addr = smem_u32(smem + kDqOffK + sb * 32768);
        const uint32_t v_addr = smem_u32(smem + kDqOffV + sb * 32768);
#pragma unroll
        for (int c = 0; c < C::kCount; ++c)
#pragma unroll
          for (int kk = 0; kk < C::steps(c); ++kk)
            umma_f16(tmem, sdesc_sw128(q_addr + c * kWaChunk + kk * 32, 16, 1024),
                     sdesc_sw128(k_addr + c * kWaChunk + kk * 32, 16, 1024), IS,
                     (c > 0 || kk > 0) ? 1u : 0u);
        if (!mbar_wait(dpfree, fr, status, kStatusTimeoutTmemEmpty)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < C::kCount; ++c)
#pragma unroll
          for (int kk = 0; kk < C::steps(c); ++kk)
            umma_f16(tmem + 128, sdesc_sw128(o_addr + c * kWaChunk + kk * 32, 16, 1024),
                     sdesc_sw128(v_addr + c * kWaChunk + kk * 32, 16, 1024), IS,
                     (c > 0 || kk > 0) ? 1u : 0u);
        umma_commit(sfull);
        if (k > 0 && !dq(k - 1)) {
          ok = false;
          break;
        }
      }
      if (ok) dq(tiles - 1);
      umma_commit(drain);
      mbar_wait(drain, 0, nullptr, kStatusTimeoutDrain);
    }
  } else {
    const int wq = warp & 3;
    const int g = (warp - 2) >> 2;  // this warpgroup's half of the 128 key columns
    const int c0 = g * 64;
    const int r = wq * 32 + lane;
    const int row = q0 + r;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    const int64_t li = (static_cast<int64_t>(bz) * H + h) * Sp + row;
    const float lr = Lp[li], dr = Dp[li];  // padded rows: +inf, 0
    bool ok = true;
    for (int k = 0; k < tiles; ++k) {
      if (!mbar_wait(sfull, k & 1, status, kStatusTimeoutTmemFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sv[64];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld16(tmem + lanes + c0 + c * 16, sv + c * 16);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sfree);
      const int k0 = list.tile(k) * 128;
      uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
      const bool whole = k0 + 127 <= q0 && q0 + 128 <= n &&
                         (q0 + 127 - k0 < window || k0 + 128 <= sinks);
      if (!whole) {
        const int hi = (row < n ? row : -1) - k0 + 1, lo = row - k0 - window + 1, sk = sinks - k0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int at = c0 + 32 * c;
          vis[c] = bits_below(hi - at) & (~bits_below(lo - at) | bits_below(sk - at));
        }
      }
#pragma unroll
      for (int e = 0; e < 64; ++e) {
        const float p = ex2_wa(__uint_as_float(sv[e]) * scale_log2 - lr);
        sv[e] = __float_as_uint((vis[e >> 5] >> (e & 31)) & 1u ? p : 0.f);
      }
      // dS buffer: the dQ MMA of the previous tile must be done reading it.
      if (k > 0 && !mbar_wait(dsfree, (k - 1) & 1, status, kStatusTimeoutSmemEmpty)) {
        ok = false;
        break;
      }
      uint8_t* srow = smem + kDqOffS + g * kWaChunk + r * 128;  // this half's 64-key chunk
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t dp[32];
        tmem_ld32(tmem + 128 + lanes + c0 + c * 32, dp);
        tmem_wait_ld();
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4) {
          uint32_t pk[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float d[2];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int at = t4 * 8 + 2 * e + z;
              const float p = __uint_as_float(sv[c * 32 + at]);
              // dP of a key past the length may be NaN; its weight is 0
              d[z] = (vis[c] >> at) & 1u ? p * (__uint_as_float(dp[at]) - dr) : 0.f;
            }
            pk[e] = pack_bf16x2(d[0], d[1]);
          }
          const int unit = c * 4 + t4;
          *reinterpret_cast<uint4*>(srow + ((unit ^ (r & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dpfree);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull);
    }
    if (ok && tiles > 0) ok = mbar_wait(dsfree, (tiles - 1) & 1, status, kStatusTimeoutTmemFull);
    if (ok) {
      tc_fence_after();
      __nv_bfloat16* out = dqkv + (static_cast<size_t>(bz) * S + row) * ((H + 2 * Hkv) * HD) + h * HD;
      // warpgroup g: the g-th half of the head's 16-column groups
      constexpr int kGroups = HD / 16, kHalf = (kGroups + 1) / 2;
#pragma unroll
      for (int k = 0; k < kHalf; ++k) {
        const int c = g * kHalf + k;
        if (c >= kGroups) break;
        uint32_t v[16];
        if (tiles > 0) {
          tmem_ld16(tmem + 256 + lanes + c * 16, v);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = 0u;
        }
        if (row < S) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(v[8 * e]) * scale, __uint_as_float(v[8 * e + 1]) * scale);
            w.y = pack_bf16x2(__uint_as_float(v[8 * e + 2]) * scale, __uint_as_float(v[8 * e + 3]) * scale);
            w.z = pack_bf16x2(__uint_as_float(v[8 * e + 4]) * scale, __uint_as_float(v[8 * e + 5]) * scale);
            w.w = pack_bf16x2(__uint_as_float(v[8 * e + 6]) * scale, __uint_as_float(v[8 * e + 7]) * scale);
            *reinterpret_cast<uint4*>(out + c * 16 + e * 8) = w;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

int padded(int S) { return (S + 127) / 128 * 128; }

KvPlan make_plan(const WindowAttnArgs& f) {
  KvPlan p{};
  p.window = std::min(f.window, f.S);
  p.sinks = std::min(f.sinks, f.S);
  p.sink_tiles = (p.sinks + 127) / 128;
  p.span = (127 + p.window + 63) / 64;  // the query blocks that a common tile meets
  const int blocks = (f.S + 63) / 64;
  p.parts = p.sink_tiles > 0 ? std::max(1, (blocks + p.span - 1) / p.span) : 1;
  return p;
}

template <int HD>
int launch_bwd(const WindowAttnBwdArgs& a, cudaStream_t stream) {
  const WindowAttnArgs& f = a.f;
  const int Sp = padded(f.S);
  const KvPlan plan = make_plan(f);
  const uint64_t width = static_cast<uint64_t>(f.H + 2 * f.Hkv) * HD, owidth = static_cast<uint64_t>(f.H) * HD;
  CUtensorMap m128, m64, do64, do128;
  if (!tma_map_bf16_3d(&m128, f.qkv, width, f.S, f.B, f.ldq, 64, 128) ||
      !tma_map_bf16_3d(&m64, f.qkv, width, f.S, f.B, f.ldq, 64, 64) ||
      !tma_map_bf16_3d(&do64, a.dout, owidth, f.S, f.B, a.ldo, 64, 64) ||
      !tma_map_bf16_3d(&do128, a.dout, owidth, f.S, f.B, a.ldo, 64, 128))
    return 1;
  static bool attr = false;
  if (!attr) {
    if (cudaFuncSetAttribute(window_dkdv_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kKvSmem) !=
            cudaSuccess ||
        cudaFuncSetAttribute(window_dq_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kDqSmem) !=
            cudaSuccess)
      return 2;
    attr = true;
  }
  const int64_t cells = static_cast<int64_t>(f.B) * f.H * Sp;
  float* Lp = a.ws;
  float* Dp = Lp + cells;
  float* parts = Dp + cells;
  window_dot_kernel<<<static_cast<unsigned>((cells + 15) / 16), 256, 0, stream>>>(
      f.o, a.dout, a.ldo, f.lse, f.lengths, Lp, Dp, f.S, Sp, f.H, HD, cells);
  const float sl2 = f.scale * kLog2eWa;
  const int units = plan.sink_tiles * plan.parts + Sp / 128 - plan.sink_tiles;
  window_dkdv_kernel<HD><<<dim3(f.Hkv, units, f.B), kWbThreads, kKvSmem, stream>>>(
      m128, m64, do64, Lp, Dp, f.lengths, a.dqkv, parts, f.S, Sp, f.H, f.Hkv, plan, sl2, f.scale, f.status);
  if (plan.parts > 1) {
    const int64_t t = static_cast<int64_t>(f.B) * f.Hkv * plan.sink_tiles * 128 * (2 * HD / 4);
    window_sinks_kernel<<<static_cast<unsigned>((t + 255) / 256), 256, 0, stream>>>(
        parts, a.dqkv, f.S, f.H, f.Hkv, HD, plan.sink_tiles, plan.parts, f.scale, t);
  }
  window_dq_kernel<HD><<<dim3(f.H, Sp / 128, f.B), kWbThreads, kDqSmem, stream>>>(
      m128, do128, Lp, Dp, f.lengths, a.dqkv, f.S, Sp, f.H, f.Hkv, plan.window, plan.sinks, sl2, f.scale,
      f.status);
  return cudaGetLastError() == cudaSuccess ? 0 : 2;
}

}  // namespace

int64_t window_attention_bwd_ws(const WindowAttnArgs& f) {
  const KvPlan p = make_plan(f);
  int64_t n = 2 * static_cast<int64_t>(f.B) * f.H * padded(f.S);
  if (p.parts > 1) n += static_cast<int64_t>(f.B) * f.Hkv * p.sink_tiles * p.parts * 128 * 2 * f.hd;
  return n;
}

int window_attention_bwd_launches(const WindowAttnArgs& f) { return make_plan(f).parts > 1 ? 4 : 3; }

int window_attention_bwd(const WindowAttnBwdArgs& a, cudaStream_t stream) {
  const WindowAttnArgs& f = a.f;
  if (f.B < 0 || f.S < 0 || f.H < 1 || f.Hkv < 1 || f.H % f.Hkv || f.window < 1 || f.sinks < 0) return 1;
  if (f.B > 65535 || f.S > 65535 * 64) return 1;  // the grid's y and z
  if (f.B == 0 || f.S == 0) return 0;
  switch (f.hd) {
    case 64: return launch_bwd<64>(a, stream);
    case 80: return launch_bwd<80>(a, stream);
    case 96: return launch_bwd<96>(a, stream);
    case 128: return launch_bwd<128>(a, stream);
    default: return 1;
  }
}

}  // namespace ewb
