// Log probabilities of given tokens, entropy and top alternatives of logit
// rows, and the gradient of a weighted sum of the first two.
//
//   lse = log sum_v e^x_v      logp = x_t - lse      H = -sum_v p_v log p_v
//   d/dx_v (gl logp + ge H) = gl ([v = t] - p_v) - ge p_v (log p_v + H)
//
// Forward: one pass over the row. Each thread keeps a running maximum m and,
// with u = (x - m) log2 e, s = sum 2^u and w = sum 2^u u, rescaled when m moves;
// then lse = m + ln s and H = (log2 s - w / s) ln 2. Both terms of H are
// non-negative, so nothing cancels. x - m is taken first, here and in log p =
// (x - m) - ln s, so that logits as low as the type goes neither overflow nor
// drown the rest.
//
// Alternatives (up to 32) without a second pass: each thread also keeps where
// its maximum stood, four neighbouring threads form a quad, and the K-th
// largest of the quads' maxima bounds the K-th largest logit from below, since
// K different logits reach it. Only the K quads whose maximum reaches that
// bound can hold an alternative, so only their share of the row (about K / 128) is read again, out of the
// L2. A logit and its index make one 64-bit key (greater logit first, then the
// lower index), so keys are distinct and ranks are counts: no order of arrival
// shows in the result.
//
// A cluster of 1, 2, 4 or 8 CTAs shares a row when there are few rows and joins
// through distributed shared memory.
//
// Rows may start anywhere (an odd vocabulary): vectors are aligned in memory
// and the two at the ends of the row are read element by element.
#include "common.cuh"
#include "kernels.h"

#include <algorithm>

namespace ewb {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpQuads = kLpThreads / 4;
constexpr int kLpTopMax = 32;
constexpr int kLpCand = 1024;
constexpr int kLpMaxCluster = 8;
constexpr float kLog2eLp = 1.4426950408889634f;
constexpr float kLn2Lp = 0.6931471805599453f;
// 2^u is 0 in fp32 from here down; keeps 0 * -inf out of the sums
constexpr float kFloorLp = -200.0f;

__device__ __forceinline__ float ex2_lp(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums of a set of logits: m = max x, s = sum 2^u, w = sum 2^u u, u = (x - m) log2 e.
struct Sums {
  float m, s, w;
};

__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) {  // no finite logit so far; a NaN stays one
    return Sums{m, a.s + b.s, a.w + b.w};
  }
  const float da = fmaxf((a.m - m) * kLog2eLp, kFloorLp), db = fmaxf((b.m - m) * kLog2eLp, kFloorLp);
  const float fa = ex2_lp(da), fb = ex2_lp(db);
  return Sums{m, a.s * fa + b.s * fb, fa * (a.w + a.s * da) + fb * (b.w + b.s * db)};
}

// Distinct keys, the better first: the greater logit, then the lower index.
__device__ __forceinline__ unsigned long long make_key(float x, int idx) {
  uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as 0
  u ^= (u >> 31) ? 0xffffffffu : 0x80000000u;
  return (static_cast<unsigned long long>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(idx));
}
__device__ __forceinline__ int key_index(unsigned long long k) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  uint32_t u = static_cast<uint32_t>(k >> 32);
  u ^= (u >> 31) ? 0x80000000u : 0xffffffffu;
  return __uint_as_float(u);
}

// A row in 16-byte vectors of kVE logits; vector i holds [i kVE - mis, + kVE).
template <typename T>
struct Row {
  static constexpr int kVE = 16 / sizeof(T);
  const T* x;  // first logit
  int mis;     // logits between the aligned address and the first one
  int V;

  __device__ __forceinline__ Row(const T* p, int v) : x(p), V(v) {
    mis = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  }
  __device__ __forceinline__ int vectors() const { return (V + mis + kVE - 1) / kVE; }
  __device__ __forceinline__ int first(int i) const { return i * kVE - mis; }
  // outside the row: -inf, which adds nothing
  __device__ __forceinline__ void load(int i, float* f) const {
    const int j = first(i);
    if (j >= 0 && j + kVE <= V) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(x + j));
      if constexpr (sizeof(T) == 4) {
        f[0] = __uint_as_float(w.x);
        f[1] = __uint_as_float(w.y);
        f[2] = __uint_as_float(w.z);
        f[3] = __uint_as_float(w.w);
      } else {
        unpack8_fmt(w, kFmtBf16, 1.0f, f);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVE; ++e) {
        f[e] = -INFINITY;
        if (j + e >= 0 && j + e < V) f[e] = static_cast<float>(x[j + e]);
      }
    }
  }
};

__device__ __forceinline__ float peer_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ int peer_s32(uint32_t a) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long peer_u64(uint32_t a) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

// Rank by counting: the keys of list[0..n) with rank < k go to out[rank].
__device__ __forceinline__ void rank_keys(const unsigned long long* list, int n, int k,
                                          unsigned long long* out) {
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const unsigned long long mine = list[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += list[j] > mine ? 1 : 0;
    if (r < k) out[r] = mine;
  }
}

struct LpShared {
  float m[kLpWarps], s[kLpWarps], w[kLpWarps];
  Sums row;                              // this CTA's sums, read by the cluster
  unsigned long long quad[kLpQuads];     // the quads' maxima
  unsigned long long thr;                // lower bound of this CTA's K-th key
  unsigned long long cand[kLpCand];
  unsigned long long top[kLpTopMax];     // this CTA's best keys, read by the cluster
  unsigned long long join[kLpTopMax * kLpMaxCluster];
  unsigned long long best;
  int ncand, ntop;
};

template <typename T, bool kTop>
__global__ void __launch_bounds__(kLpThreads)
    token_logprobs_kernel(const T* __restrict__ logits, int64_t ld, int V,
                          const int64_t* __restrict__ targets, int top, int cluster,
                          float* __restrict__ logp, float* __restrict__ entropy,
                          float* __restrict__ lse, float* __restrict__ top_logp,
                          int64_t* __restrict__ top_ids, int* status) {
  __shared__ LpShared sh;
  constexpr int kVE = Row<T>::kVE;
  constexpr int kUnroll = 4;
  const int64_t r = blockIdx.x / cluster;
  const int part = blockIdx.x % cluster;
  const Row<T> row(logits + r * ld, V);
  const int nv = row.vectors();
  const int per = (nv + cluster - 1) / cluster;
  const int v0 = part * per, v1 = min(nv, v0 + per);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  int64_t target = -1;
  float xt = 0.f;
  if (part == 0 && tid == 0 && targets != nullptr) {
    target = targets[r];
    if (target >= 0 && target < V) xt = static_cast<float>(row.x[target]);
  }

  Sums a{-INFINITY, 0.f, 0.f};
  int bi = max(0, row.first(v0 + tid));  // where this thread's largest logit stands first
  const bool any = v0 + tid < v1;
  for (int i = v0 + tid; i < v1; i += kLpThreads * kUnroll) {
    float f[kUnroll][kVE];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int iu = i + u * kLpThreads;
      if (iu < v1) {
        row.load(iu, f[u]);
      } else {
#pragma unroll
        for (int e = 0; e < kVE; ++e) f[u][e] = -INFINITY;
      }
    }
    float cx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < kVE; ++e) cx = fmaxf(cx, f[u][e]);
    if constexpr (kTop) {
      if (cx > a.m) {
#pragma unroll
        for (int u = kUnroll - 1; u >= 0; --u)
#pragma unroll
          for (int e = kVE - 1; e >= 0; --e)
            if (f[u][e] == cx) bi = row.first(i + u * kLpThreads) + e;
      }
    }
    if (cx > a.m) {
      const float df = fmaxf((a.m - cx) * kLog2eLp, kFloorLp);
      const float fa = ex2_lp(df);
      a.w = fa * (a.w + a.s * df);
      a.s *= fa;
      a.m = cx;
    }
    const float mm = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < kVE; ++e) {
        float d = (f[u][e] - mm) * kLog2eLp;
        d = d < kFloorLp ? kFloorLp : d;  // keeps a NaN
        const float p = ex2_lp(d);
        a.s += p;
        a.w = fmaf(p, d, a.w);
      }
  }
  unsigned long long k = 0ull;
  if constexpr (kTop) k = any ? make_key(a.m, bi) : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
           __shfl_xor_sync(0xffffffffu, a.w, o)};
    // the lower lane's sums first, so both lanes add in the same order
    a = (lane & o) ? join(b, a) : join(a, b);
  }
  if (lane == 0) {
    sh.m[warp] = a.m;
    sh.s[warp] = a.s;
    sh.w[warp] = a.w;
  }
  if constexpr (kTop) {
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      const unsigned long long q = __shfl_xor_sync(0xffffffffu, k, o);
      k = q > k ? q : k;
    }
    if ((lane & 3) == 0) sh.quad[tid >> 2] = k;
    if (tid == 0) {
      sh.thr = 1ull;  // fewer than K quads have logits: every logit counts
      sh.ncand = 0;
    }
  }
  __syncthreads();
  if (tid == 0) {
    Sums t{sh.m[0], sh.s[0], sh.w[0]};
    for (int k = 1; k < kLpWarps; ++k) t = join(t, Sums{sh.m[k], sh.s[k], sh.w[k]});
    sh.row = t;
  }
  if constexpr (kTop) {
    if (tid < kLpQuads) {
      const unsigned long long mine = sh.quad[tid];
      int rank = 0;
#pragma unroll 16
      for (int j = 0; j < kLpQuads; ++j) rank += sh.quad[j] > mine ? 1 : 0;
      if (rank == top - 1 && mine != 0ull) sh.thr = mine;
    }
    __syncthreads();
    const unsigned long long thr = sh.thr;
    for (int qw = 0; qw < 8; ++qw) {  // the warp's eight quads, all lanes on one
      const int q = warp * 8 + qw;
      const unsigned long long qmax = sh.quad[q];
      if (qmax < thr || qmax == 0ull) continue;
      // lane l: thread q * 4 + l % 4 of rounds l / 4, l / 4 + 8, ...
      for (int i = v0 + q * 4 + (lane & 3) + (lane >> 2) * kLpThreads; i < v1; i += 8 * kLpThreads) {
        float f[kVE];
        row.load(i, f);
        const int j = row.first(i);
#pragma unroll
        for (int e = 0; e < kVE; ++e) {
          if (j + e < 0 || j + e >= V) continue;
          const unsigned long long k = make_key(f[e], j + e);
          if (k >= thr) {
            const int at = atomicAdd(&sh.ncand, 1);
            if (at < kLpCand) sh.cand[at] = k;
          }
        }
      }
    }
    __syncthreads();
    const int n = sh.ncand;
    if (n <= kLpCand) {
      rank_keys(sh.cand, n, top, sh.top);
      if (tid == 0) sh.ntop = min(n, top);
    } else {
      // Many logits of few threads at the top (a row of steps): one pass over
      // this CTA's share of the row for each alternative, best first.
      unsigned long long prev = ~0ull;
      for (int t = 0; t < top; ++t) {
        if (tid == 0) sh.best = 0ull;
        __syncthreads();
        unsigned long long k = 0ull;
        for (int i = v0 + tid; i < v1; i += kLpThreads) {
          float f[kVE];
          row.load(i, f);
          const int j = row.first(i);
#pragma unroll
          for (int e = 0; e < kVE; ++e) {
            if (j + e < 0 || j + e >= V) continue;
            const unsigned long long c = make_key(f[e], j + e);
            if (c < prev && c > k) k = c;
          }
        }
        atomicMax(&sh.best, k);
        __syncthreads();
        prev = sh.best;
        if (tid == 0) sh.top[t] = prev;
        __syncthreads();
      }
      if (tid == 0) sh.ntop = top;
    }
  }
  // ---- join the row's CTAs
  Sums tot;
  if (cluster > 1) {
    cluster_sync_all();
    if (part == 0 && tid == 0) {
      tot = sh.row;
      for (int k = 1; k < cluster; ++k) {
        const uint32_t p = peer_smem(smem_u32(&sh.row), k);
        tot = join(tot, Sums{peer_f32(p), peer_f32(p + 4), peer_f32(p + 8)});
      }
      sh.row = tot;
    }
    if constexpr (kTop) {
      if (part == 0 && tid < cluster * kLpTopMax) {
        const int k = tid / kLpTopMax, e = tid % kLpTopMax;
        const int have = peer_s32(peer_smem(smem_u32(&sh.ntop), k));
        sh.join[tid] = e < have ? peer_u64(peer_smem(smem_u32(&sh.top[e]), k)) : 0ull;
      }
    }
    cluster_sync_all();  // nobody leaves while its shared memory is read
    if (part != 0) return;
    if constexpr (kTop) {
      const int n = cluster * kLpTopMax;
      if (tid < n && sh.join[tid] != 0ull) {
        const unsigned long long mine = sh.join[tid];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sh.join[j] > mine ? 1 : 0;
        if (rank < top) sh.top[rank] = mine;
      }
    }
  }
  __syncthreads();
  tot = sh.row;
  // A NaN or +inf among the logits leaves NaN in s. No finite logit: lse -inf.
  const bool empty = tot.m == -INFINITY && !(tot.s != tot.s);
  const float l2 = log2f(tot.s);
  const float lns = l2 * kLn2Lp;
  const float z = empty ? -INFINITY : tot.m + lns;
  if (tid == 0) {
    lse[r] = z;
    entropy[r] = empty ? 0.f : (l2 - tot.w / tot.s) * kLn2Lp;
    if (logp != nullptr) {
      float v = 0.f;  // a negative target: no token given
      if (target >= V) {
        record_check(status, kStatusBadArgument, kSiteCeTarget, r, target);
        v = __int_as_float(0x7fc00000);
      } else if (target >= 0) {
        v = empty ? -INFINITY : (xt - tot.m) - lns;
      }
      logp[r] = v;
    }
  }
  if constexpr (kTop) {
    if (tid < top) {
      const bool nan = z != z;
      const unsigned long long k = sh.top[tid];
      top_logp[r * top + tid] = nan ? z : empty ? -INFINITY : (key_value(k) - tot.m) - lns;
      top_ids[r * top + tid] = nan ? -1 : key_index(k);
    }
  }
}

// ---------------------------------------------------------------- gradient
// d = p (A + B u) + gl [v = t] with u = log2 p, A = -(gl + ge H), B = -ge ln 2.
// Bound by memory: the logits read and the gradient written once. Rows that
// are 16-byte aligned on both sides go in vectors of eight; others (an odd
// vocabulary) one element per lane, whose loads and stores still coalesce.
constexpr int kLgThreads = 256;

// x - lse first: it is exact to half a unit of the (small) difference.
__device__ __forceinline__ float lp_grad(float x, float lse, float A, float B) {
  float u = (x - lse) * kLog2eLp;
  u = u < kFloorLp ? kFloorLp : u;
  return ex2_lp(u) * fmaf(B, u, A);
}

template <typename T, typename TG, bool kVec>
__global__ void __launch_bounds__(kLgThreads)
    token_logprobs_bwd_kernel(const T* __restrict__ logits, int64_t ld, int V,
                              const int64_t* __restrict__ targets, const float* __restrict__ lse,
                              const float* __restrict__ entropy, const float* __restrict__ g_logp,
                              const float* __restrict__ g_entropy, TG* __restrict__ grad,
                              int64_t ldg, int cols, int64_t rows) {
  constexpr int kPer = kVec ? 8 : 16;  // elements a thread handles per step
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const T* x = logits + r * ld;
    TG* g = grad + r * ldg;
    // no finite logit: every p is 0, as an lse of +inf makes it
    const float z = lse[r] == -INFINITY ? INFINITY : lse[r];
    const int64_t t = targets != nullptr ? targets[r] : -1;
    const bool given = t >= 0 && t < V;
    const float gl = given && g_logp != nullptr ? g_logp[r] : 0.f;
    const float ge = g_entropy != nullptr ? g_entropy[r] : 0.f;
    const float A = -(gl + ge * entropy[r]), B = -ge * kLn2Lp;
    const int step = gridDim.x * kLgThreads * kPer;
    for (int j0 = blockIdx.x * kLgThreads * kPer; j0 < cols; j0 += step) {
      if constexpr (kVec) {
        const int j = j0 + threadIdx.x * 8;
        if (j >= cols) continue;
        float f[8];
        if (j + 8 <= V) {
          if constexpr (sizeof(T) == 4) {
            const uint4 w = __ldcs(reinterpret_cast<const uint4*>(x + j));
            const uint4 q = __ldcs(reinterpret_cast<const uint4*>(x + j) + 1);
            const uint32_t u[8] = {w.x, w.y, w.z, w.w, q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(u[e]);
          } else {
            unpack8_fmt(__ldcs(reinterpret_cast<const uint4*>(x + j)), kFmtBf16, 1.0f, f);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = j + e < V ? static_cast<float>(x[j + e]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v = lp_grad(f[e], z, A, B);
          if (given && j + e == t) v += gl;
          f[e] = j + e < V ? v : 0.f;
        }
        if constexpr (sizeof(TG) == 4) {
          float4* o = reinterpret_cast<float4*>(g + j);
          o[0] = make_float4(f[0], f[1], f[2], f[3]);
          o[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
          *reinterpret_cast<uint4*>(g + j) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                        pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
        }
      } else {
        float f[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int j = j0 + e * kLgThreads + threadIdx.x;
          f[e] = j < V ? static_cast<float>(x[j]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int j = j0 + e * kLgThreads + threadIdx.x;
          float v = lp_grad(f[e], z, A, B);
          if (given && j == t) v += gl;
          if (j >= V) v = 0.f;
          if (j < cols) {
            if constexpr (sizeof(TG) == 4) g[j] = v;
            else g[j] = __float2bfloat16_rn(v);
          }
        }
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, bool kTop>
int launch_fwd(const LogprobsArgs& a, int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows * cluster));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, kTop>, static_cast<const T*>(a.logits),
                            a.ld, a.V, a.targets, a.top, cluster, a.logp, a.entropy, a.lse,
                            a.top_logp, a.top_ids, a.status) == cudaSuccess
             ? 0
             : 2;
}

template <typename T, typename TG>
int launch_bwd(const LogprobsBwdArgs& a, cudaStream_t stream) {
  const T* x = static_cast<const T*>(a.logits);
  TG* g = static_cast<TG*>(a.grad);
  constexpr int64_t kVT = 16 / sizeof(T), kVG = 16 / sizeof(TG);
  const bool vec = aligned16(x) && aligned16(g) && a.ld % kVT == 0 && a.ldg % kVG == 0 && a.cols % 8 == 0;
  const int span = kLgThreads * (vec ? 8 : 16);
  const int64_t bx = (a.cols + span - 1) / span;
  const int64_t by = std::min<int64_t>(a.rows, 65535);
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by));
  if (vec)
    token_logprobs_bwd_kernel<T, TG, true><<<grid, kLgThreads, 0, stream>>>(
        x, a.ld, a.V, a.targets, a.lse, a.entropy, a.g_logp, a.g_entropy, g, a.ldg, a.cols, a.rows);
  else
    token_logprobs_bwd_kernel<T, TG, false><<<grid, kLgThreads, 0, stream>>>(
        x, a.ld, a.V, a.targets, a.lse, a.entropy, a.g_logp, a.g_entropy, g, a.ldg, a.cols, a.rows);
  return cudaGetLastError() == cudaSuccess ? 0 : 2;
}

}  // namespace

int token_logprobs(const LogprobsArgs& a, cudaStream_t stream) {
  if (a.rows < 0 || a.V < 1 || a.top < 0 || a.top > kLpTopMax || a.top > a.V) return 1;
  if (a.rows == 0) return 0;
  const bool bf16 = a.type == kElemBf16;
  if (!bf16 && a.type != kElemF32) return 1;
  // CTAs a row: while the rows leave SMs idle and a CTA's share stays above one
  // round of its threads' vectors.
  int cluster = 1;
  const int64_t vectors = static_cast<int64_t>(a.V) * (bf16 ? 2 : 4) / 16;
  while (cluster < kLpMaxCluster && a.rows * cluster * 2 <= 2 * 148 && vectors / (cluster * 2) >= kLpThreads)
    cluster *= 2;
  if (a.rows * cluster > 0x7fffffffll) return 1;
  if (bf16)
    return a.top > 0 ? launch_fwd<__nv_bfloat16, true>(a, cluster, stream)
                     : launch_fwd<__nv_bfloat16, false>(a, cluster, stream);
  return a.top > 0 ? launch_fwd<float, true>(a, cluster, stream)
                   : launch_fwd<float, false>(a, cluster, stream);
}

int token_logprobs_bwd(const LogprobsBwdArgs& a, cudaStream_t stream) {
  if (a.rows < 0 || a.V < 1 || a.cols < a.V || a.cols > 0x7fff0000) return 1;
  if (a.rows == 0) return 0;
  const bool bf16 = a.type == kElemBf16, gbf16 = a.grad_type == kElemBf16;
  if ((!bf16 && a.type != kElemF32) || (!gbf16 && a.grad_type != kElemF32)) return 1;
  if (bf16)
    return gbf16 ? launch_bwd<__nv_bfloat16, __nv_bfloat16>(a, stream)
                 : launch_bwd<__nv_bfloat16, float>(a, stream);
  return gbf16 ? launch_bwd<float, __nv_bfloat16>(a, stream) : launch_bwd<float, float>(a, stream);
}

}  // namespace ewb
