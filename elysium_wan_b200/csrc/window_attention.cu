// Attention in a sliding window with sinks, forward, on the 5th-generation
// tensor cores: query i sees key j <= i when i - j < window or j < sinks, both
// below the sequence's length.
//
//   x = q k / sqrt(hd);  p = e^(x - m);  o = sum p v / sum p;  lse2 = log2 sum e^x
//
// One CTA owns 256 query rows of one (batch, head) as two subtiles of 128 and
// walks the key tiles of 128 that either can see: the sinks' tiles, then the
// window's. Each K and V tile is loaded once for both subtiles, which halves the
// traffic from the L2 (at 128 rows a CTA it would bound the kernel: 64 KB for
// 1024 cycles of tensor work on each SM). Ten warps:
//   warp 0     TMA producer: Q once, then K and V tiles into their rings;
//   warp 1     MMA issuer (one thread): for each tile k and subtile t,
//              O_t += P_t V_{k-1}, then S_t = Q_t K_k^T over the same TMEM columns
//              (MMAs of one thread run in order, so S_t may overwrite P_t);
//   warps 2-5, 6-9  softmax of subtile 0 and 1, one query row a thread: while
//              one subtile is in the tensor cores the other one is here.
// P never leaves TMEM: the softmax thread reads its row of S, and writes the
// row's bf16 weights over the first half of the same columns, from where the
// second product reads them as its A operand. The running maximum moves only
// when it grows by more than 2^8 (weights and sums share it, so o is unchanged),
// and then the same thread rescales its row of O: S_t is complete only after
// every earlier product of this CTA, so O_t rests meanwhile.
// TMEM: S_0 | S_1 | O_0 | O_1 = 512 columns. Shared memory: Q 2 tiles, K 2, V 3.
//
// Rows past a sequence's end: boxes of the 3D tensor map read zeros past S; the
// V tile that holds the end of a shorter sequence is cleared from there on by
// the producer, so that 0 x NaN cannot reach a sum. Every wait is bounded.
#include "common.cuh"
#include "gemm.h"
#include "kernels.h"
#include "window.cuh"

#include <algorithm>

namespace ewb {
namespace {

constexpr int kWaKStages = 2, kWaVStages = 3;
constexpr int kWaThreads = 320;
constexpr float kWaRescale = 8.0f;

template <int HD>
struct WaLayout {
  static constexpr int kChunks = HeadChunks<HD>::kCount;
  static constexpr uint32_t kTile = kChunks * kWaChunk;
  static constexpr uint32_t kQ = 0, kK = 2 * kTile, kV = kK + kWaKStages * kTile;
  static constexpr uint32_t kBar = kV + kWaVStages * kTile;
  static constexpr int kSmem = static_cast<int>(kBar) + 256 + 1024;
};

template <int HD>
__global__ void __launch_bounds__(kWaThreads, 1)
    window_fwd_kernel(const __grid_constant__ CUtensorMap map, __nv_bfloat16* __restrict__ o,
                      float* __restrict__ lse2, const int* __restrict__ lengths, int S, int H,
                      int Hkv, int window, int sinks, float scale_log2, int* status) {
  using L = WaLayout<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* qfull = bars;                       // [2]
  uint64_t* kfull = qfull + 2;                  // [kWaKStages]
  uint64_t* kempty = kfull + kWaKStages;
  uint64_t* vfull = kempty + kWaKStages;        // [kWaVStages]
  uint64_t* vempty = vfull + kWaVStages;
  uint64_t* sfull = vempty + kWaVStages;        // [2]
  uint64_t* pfull = sfull + 2;                  // [2]
  uint64_t* ofull = pfull + 2;                  // [2]
  uint64_t* landed = ofull + 2;                 // the V tile that the producer clears
  uint64_t* drain = landed + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int h = blockIdx.x, b = blockIdx.z;
  const int q0 = (gridDim.y - 1 - blockIdx.y) * 256;  // the latest rows first: most tiles
  const int hk = h / (H / Hkv);
  const int n = lengths != nullptr ? min(max(lengths[b], 0), S) : S;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // subtile t: rows q0 + 128 t ..; none of them below the length: no work
  const int live = n <= q0 ? 0 : n <= q0 + 128 ? 1 : 2;
  const TileList all(q0, min(q0 + 255, max(n, 1) - 1), window, sinks);
  const TileList sub0(q0, min(q0 + 127, max(n, 1) - 1), window, sinks);
  const TileList sub1(q0 + 128, min(q0 + 255, max(n, 1) - 1), window, sinks);
  const int tiles = live > 0 ? all.count() : 0;
  // does subtile t see tile j?
  auto sees = [&](int t, int j) -> bool {
    if (t >= live) return false;
    const TileList& s = t ? sub1 : sub0;
    return (j < s.ns || j >= s.w0) && j <= s.e;
  };

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&qfull[i], 1);
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
      mbar_init(&ofull[i], 1);
    }
    for (int i = 0; i < kWaKStages; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&kempty[i], 1);
    }
    for (int i = 0; i < kWaVStages; ++i) {
      mbar_init(&vfull[i], 1);
      mbar_init(&vempty[i], 1);
    }
    mbar_init(landed, 1);
    mbar_init(drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&map);
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
    // The V tile that holds row n of a sequence shorter than S is cleared
    // from that row on before it is handed over.
    const int clear = (n < S && (n & 127)) ? n >> 7 : -1;
    const int kcol = (H + hk) * HD, vcol = (H + Hkv + hk) * HD;
    bool ok = true;
    int kdone = 0, vdone = 0;  // tiles whose loads were issued
    if (lane == 0) {
      for (int t = 0; t < live; ++t) {
        mbar_arrive_expect_tx(&qfull[t], L::kTile);
        for (int c = 0; c < L::kChunks; ++c)
          tma_load_3d(smem + L::kQ + t * L::kTile + c * kWaChunk, &map, &qfull[t], h * HD + c * 64,
                      q0 + t * 128, b, status);
      }
    }
    for (int k = 0; k < tiles && ok; ++k) {
      const int j = all.tile(k);
      const int ks = k % kWaKStages, vs = k % kWaVStages;
      uint8_t* sv = smem + L::kV + vs * L::kTile;
      uint64_t* vbar = j == clear ? landed : &vfull[vs];
      if (lane == 0) {
        ok = mbar_wait(&kempty[ks], ((k / kWaKStages) & 1) ^ 1, status, kStatusTimeoutSmemEmpty);
        if (ok) {
          mbar_arrive_expect_tx(&kfull[ks], L::kTile);
          for (int c = 0; c < L::kChunks; ++c)
            tma_load_3d(smem + L::kK + ks * L::kTile + c * kWaChunk, &map, &kfull[ks], kcol + c * 64,
                        j * 128, b, status);
          kdone = k + 1;
          ok = mbar_wait(&vempty[vs], ((k / kWaVStages) & 1) ^ 1, status, kStatusTimeoutSmemEmpty);
        }
        if (ok) {
          mbar_arrive_expect_tx(vbar, L::kTile);
          for (int c = 0; c < L::kChunks; ++c)
            tma_load_3d(sv + c * kWaChunk, &map, vbar, vcol + c * 64, j * 128, b, status);
          vdone = k + 1;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (ok && j == clear) {
        if (!mbar_wait(landed, 0, status, kStatusTimeoutSmemFull)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        const int r0 = n & 127;
        for (int i = lane; i < (128 - r0) * 8 * L::kChunks; i += 32) {
          const int c = i / ((128 - r0) * 8), w = i - c * (128 - r0) * 8;
          *reinterpret_cast<uint4*>(sv + c * kWaChunk + r0 * 128 + w * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&vfull[vs]);
      }
    }
    // Loads already issued must land before this CTA's memory goes away.
    if (lane == 0) {
      for (int t = 0; t < live; ++t) mbar_wait(&qfull[t], 0, nullptr, kStatusTimeoutDrain);
      for (int k = kdone - 1; k >= 0 && k >= kdone - kWaKStages; --k)
        mbar_wait(&kfull[k % kWaKStages], (k / kWaKStages) & 1, nullptr, kStatusTimeoutDrain);
      for (int k = vdone - 1; k >= 0 && k >= vdone - kWaVStages; --k) {
        if (all.tile(k) == clear) mbar_wait(landed, 0, nullptr, kStatusTimeoutDrain);
        else mbar_wait(&vfull[k % kWaVStages], (k / kWaVStages) & 1, nullptr, kStatusTimeoutDrain);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t IS = idesc_bf16_f32(128, 128, false, false);
      constexpr uint32_t IP = idesc_bf16_f32(128, HD, false, true);
      const uint32_t q_addr = smem_u32(smem + L::kQ);
      bool ok = true;
      int done[2] = {0, 0};  // products P V issued
      for (int t = 0; t < live; ++t) ok = ok && mbar_wait(&qfull[t], 0, status, kStatusTimeoutSmemFull);
      for (int k = 0; k <= tiles && ok; ++k) {
        if (tiles == 0) break;
        const int j = all.tile(k), jp = k > 0 ? all.tile(k - 1) : 0;
        const int ks = k % kWaKStages, vs = (k + kWaVStages - 1) % kWaVStages;
        if (k < tiles)
          ok = mbar_wait(&kfull[ks], (k / kWaKStages) & 1, status, kStatusTimeoutSmemFull);
        if (ok && k > 0)
          ok = mbar_wait(&vfull[vs], ((k - 1) / kWaVStages) & 1, status, kStatusTimeoutSmemFull);
        if (!ok) break;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(smem + L::kK + ks * L::kTile);
        const uint32_t v_addr = smem_u32(smem + L::kV + vs * L::kTile);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (k > 0 && sees(t, jp)) {
            if (!mbar_wait(&pfull[t], done[t] & 1, status, kStatusTimeoutTmemFull)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8,
                          sdesc_sw128(v_addr + kk * 2048, kWaChunk, 1024), IP,
                          (done[t] > 0 || kk > 0) ? 1u : 0u);
            ++done[t];
            if (jp == (t ? sub1.e : sub0.e)) umma_commit(&ofull[t]);
          }
          if (k < tiles && sees(t, j)) {
#pragma unroll
            for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
              for (int kk = 0; kk < HeadChunks<HD>::steps(c); ++kk)
                umma_f16(tmem + t * 128,
                         sdesc_sw128(q_addr + t * L::kTile + c * kWaChunk + kk * 32, 16, 1024),
                         sdesc_sw128(k_addr + c * kWaChunk + kk * 32, 16, 1024), IS,
                         (c > 0 || kk > 0) ? 1u : 0u);
            umma_commit(&sfull[t]);
          }
        }
        if (!ok) break;
        if (k < tiles) umma_commit(&kempty[ks]);
        if (k > 0) umma_commit(&vempty[vs]);
      }
      umma_commit(drain);
      mbar_wait(drain, 0, nullptr, kStatusTimeoutDrain);
    }
  } else {
    const int t = (warp - 2) >> 2;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;  // row of the subtile = TMEM lane
    const int row = q0 + t * 128 + r;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t s_t = tmem + t * 128 + lanes, o_t = tmem + 256 + t * 128 + lanes;
    const TileList& sub = t ? sub1 : sub0;
    const int mine = t < live ? sub.count() : 0;
    const int first = q0 + t * 128;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
      if (!mbar_wait(&sfull[t], i & 1, status, kStatusTimeoutTmemFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int k0 = sub.tile(i) * 128;
      uint32_t v[128];
#pragma unroll
      for (int c = 0; c < 8; ++c) tmem_ld16(s_t + c * 16, v + c * 16);
      tmem_wait_ld();
      // whole tile visible to every row below the length?
      const bool whole = k0 + 127 <= first && k0 + 128 <= n &&
                         (first + 127 - k0 < window || k0 + 128 <= sinks);
      if (!whole) {
        const int hi = min(row, n - 1) - k0 + 1;       // visible below this column,
        const int lo = row - k0 - window + 1;          // and from this one
        const int sk = sinks - k0;                     // or below this one
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t vis = bits_below(hi - 32 * c) &
                               (~bits_below(lo - 32 * c) | bits_below(sk - 32 * c));
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((vis >> e) & 1u)) v[32 * c + e] = 0xff800000u;  // -inf
        }
      }
      float mx = __uint_as_float(v[0]);
#pragma unroll
      for (int e = 1; e < 128; ++e) mx = fmaxf(mx, __uint_as_float(v[e]));
      mx *= scale_log2;
      float mnew = m;
      if (__any_sync(0xffffffffu, mx > m + kWaRescale)) mnew = fmaxf(m, mx);
      const float alpha = m == -INFINITY ? 0.f : ex2_wa(m - mnew);
      const float sub_m = mnew == -INFINITY ? 0.f : mnew;  // nothing visible yet: weights 0
      float rs = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = ex2_wa(fmaf(__uint_as_float(v[32 * c + 2 * e]), scale_log2, -sub_m));
          const float p1 = ex2_wa(fmaf(__uint_as_float(v[32 * c + 2 * e + 1]), scale_log2, -sub_m));
          rs += p0 + p1;
          pk[e] = pack_bf16x2(p0, p1);
        }
        tmem_st16(s_t + c * 16, pk);
      }
      l = l * alpha + rs;
      if (i > 0 && __any_sync(0xffffffffu, mnew != m)) {
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
          uint32_t ov[16];
          tmem_ld16(o_t + c * 16, ov);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
          tmem_st16(o_t + c * 16, ov);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[t]);
      m = mnew;
    }
    if (mine > 0 && ok) ok = mbar_wait(&ofull[t], 0, status, kStatusTimeoutTmemFull);
    if (ok) {
      tc_fence_after();
      const bool in = row < n;  // a row at or past the length: 0, -inf
      const float inv = in ? 1.0f / l : 0.f;
      __nv_bfloat16* orow = o + ((static_cast<size_t>(b) * S + row) * H + h) * HD;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t v[16];
        if (mine > 0) {
          tmem_ld16(o_t + c * 16, v);
          tmem_wait_ld();
        }
        if (row < S) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (in) {
              w.x = pack_bf16x2(__uint_as_float(v[8 * u]) * inv, __uint_as_float(v[8 * u + 1]) * inv);
              w.y = pack_bf16x2(__uint_as_float(v[8 * u + 2]) * inv, __uint_as_float(v[8 * u + 3]) * inv);
              w.z = pack_bf16x2(__uint_as_float(v[8 * u + 4]) * inv, __uint_as_float(v[8 * u + 5]) * inv);
              w.w = pack_bf16x2(__uint_as_float(v[8 * u + 6]) * inv, __uint_as_float(v[8 * u + 7]) * inv);
            }
            *reinterpret_cast<uint4*>(orow + c * 16 + u * 8) = w;
          }
        }
      }
      if (row < S)
        lse2[(static_cast<size_t>(b) * H + h) * S + row] = in ? m + log2f(l) : -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
int launch_fwd(const WindowAttnArgs& a, cudaStream_t stream) {
  using L = WaLayout<HD>;
  CUtensorMap map;
  const uint64_t width = static_cast<uint64_t>(a.H + 2 * a.Hkv) * HD;
  if (!tma_map_bf16_3d(&map, a.qkv, width, a.S, a.B, a.ldq, 64, 128)) return 1;
  static bool attr = false;
  if (!attr) {
    if (cudaFuncSetAttribute(window_fwd_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             L::kSmem) != cudaSuccess)
      return 2;
    attr = true;
  }
  const dim3 grid(a.H, (a.S + 255) / 256, a.B);
  window_fwd_kernel<HD><<<grid, kWaThreads, L::kSmem, stream>>>(
      map, a.o, a.lse, a.lengths, a.S, a.H, a.Hkv, std::min(a.window, a.S), std::min(a.sinks, a.S),
      a.scale * kLog2eWa, a.status);
  return cudaGetLastError() == cudaSuccess ? 0 : 2;
}

}  // namespace

int window_attention_fwd(const WindowAttnArgs& a, cudaStream_t stream) {
  if (a.B < 0 || a.S < 0 || a.H < 1 || a.Hkv < 1 || a.H % a.Hkv || a.window < 1 || a.sinks < 0) return 1;
  if (a.B > 65535 || a.S > 65535 * 128) return 1;  // the grid's y and z
  if (a.B == 0 || a.S == 0) return 0;
  switch (a.hd) {
    case 64: return launch_fwd<64>(a, stream);
    case 80: return launch_fwd<80>(a, stream);
    case 96: return launch_fwd<96>(a, stream);
    case 128: return launch_fwd<128>(a, stream);
    default: return 1;
  }
}

}  // namespace ewb
