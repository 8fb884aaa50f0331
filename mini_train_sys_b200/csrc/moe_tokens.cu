// A whole mixture-of-experts layer for a few tokens in two kernels.
//
//   p = softmax(x Wr^T);  the K largest (ties to the lower expert), optionally divided by their sum
//   y = sum_k w_k Wd[e_k] (silu(Wg[e_k] x) * (Wu[e_k] x))
//
// What bounds it: reading the weights of every expert that has a token, 6 H I bytes each, once.  A weight matrix is the row
// operand (16 rows) of m16n8k16 and the tokens of its expert are the columns (8 at a time), so one pass over the weights serves
// up to 64 tokens; a lane takes 16 bytes of a weight row per load, straight from global memory into fragments.
//   1  every CTA routes all tokens for itself (T * E * H products: less than another launch would cost), then takes
//      (expert, 16 columns of the hidden layer) items; its warps share the contraction over H.  The hidden value is multiplied by the
//      route's weight, so that the second kernel's accumulators are sums over the experts already.
//   2  a CTA takes 16 output rows and a share of all (expert, contraction) steps; the CTAs of a cluster add their shares
//      through distributed shared memory, in order.
//
// Rounding: logits, softmax, sums and the hidden values are fp32; a hidden value enters the second product as the sum of two bf16
// values (2^-16), so y is rounded to bf16 once.
#include "decode.cuh"
#include "ops.cuh"
#include "mma_sync.cuh"

#include <cooperative_groups.h>
#include <math_constants.h>

namespace mts {

namespace {

namespace cg = cooperative_groups;

constexpr int kExperts = 64;
constexpr int kTopK = 8;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRoutes = kMoeTokensMax * kTopK;

struct Params {
  const __nv_bfloat16* x;
  long long ldx;
  const void* router;
  int router_bf16;
  const __nv_bfloat16* gate_up;
  const __nv_bfloat16* down;
  __nv_bfloat16* y;
  __nv_bfloat16* hidden;       // [2][T * K][I]: high and low part
  int* routes;
  int T, E, K, H, I, normalize;
};

// Routes by expert: `order` holds the routes of expert e, ascending, at [first[e], first[e + 1]); `active` the experts with one.
struct Routing {
  int expert[kRoutes];
  int order[kRoutes];
  int first[kExperts + 1];
  int active[kExperts];
  int num_active;
};

__device__ __forceinline__ float2 bf2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }

// first / order / active from expert[]: one warp an expert, so the order is that of the routes whatever the timing.
__device__ __forceinline__ void sort_routes(Routing& r, int routes, int E) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = warp; e < E; e += kWarps) {
    int n = 0;
    for (int i = lane; i < routes; i += 32) n += r.expert[i] == e;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) r.first[e + 1] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int at = 0, live = 0;
    r.first[0] = 0;
    for (int e = 0; e < E; ++e) {
      const int n = r.first[e + 1];
      if (n > 0) r.active[live++] = e;
      at += n;
      r.first[e + 1] = at;
    }
    r.num_active = live;
  }
  __syncthreads();
  for (int e = warp; e < E; e += kWarps) {
    int at = r.first[e];
    for (int i0 = 0; i0 < routes; i0 += 32) {
      const bool mine = i0 + lane < routes && r.expert[i0 + lane] == e;
      const unsigned votes = __ballot_sync(0xffffffffu, mine);
      if (mine) r.order[at + __popc(votes & ((1u << lane) - 1))] = i0 + lane;
      at += __popc(votes);
    }
  }
  __syncthreads();
}

// logits[t][e] in fp32: a warp takes one expert and four tokens at a time, every (token, expert) sum in the same order.
__device__ __forceinline__ void router_logits(const Params& p, float* logits) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int quads = (p.T + 3) / 4;
  for (int job = warp; job < p.E * quads; job += kWarps) {
    const int e = job % p.E, t0 = (job / p.E) * 4;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int d = lane * 8; d < p.H; d += 256) {
      float w[8];
      if (p.router_bf16) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.router) + (long long)e * p.H + d));
        const float2 a = bf2(q.x), b = bf2(q.y), c = bf2(q.z), f = bf2(q.w);
        w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y; w[4] = c.x; w[5] = c.y; w[6] = f.x; w[7] = f.y;
      } else {
        const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.router) + (long long)e * p.H + d);
        const float4 a = __ldg(src), b = __ldg(src + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = min(t0 + j, p.T - 1);
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(p.x + t * p.ldx + d));
        const float2 a = bf2(q.x), b = bf2(q.y), c = bf2(q.z), f = bf2(q.w);
        acc[j] = fmaf(a.x, w[0], acc[j]); acc[j] = fmaf(a.y, w[1], acc[j]);
        acc[j] = fmaf(b.x, w[2], acc[j]); acc[j] = fmaf(b.y, w[3], acc[j]);
        acc[j] = fmaf(c.x, w[4], acc[j]); acc[j] = fmaf(c.y, w[5], acc[j]);
        acc[j] = fmaf(f.x, w[6], acc[j]); acc[j] = fmaf(f.y, w[7], acc[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], off);
      if (lane == 0 && t0 + j < p.T) logits[(t0 + j) * p.E + e] = acc[j];
    }
  }
}

// One warp a token: K rounds of arg-max over the logits (two experts a lane), then the softmax of the chosen ones.
__device__ __forceinline__ void choose_experts(const Params& p, const float* logits, Routing& r, float* weight) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int t = warp; t < p.T; t += kWarps) {
    float v[2];
    unsigned key[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int e = lane + 32 * j;
      v[j] = e < p.E ? logits[t * p.E + e] : -CUDART_INF_F;
      const unsigned u = __float_as_uint(v[j]);
      key[j] = e < p.E ? ((u & 0x80000000u) ? ~u : (u | 0x80000000u)) : 0u;        // unsigned order = float order
      if (e < p.E && key[j] == 0u) key[j] = 1u;                                     // a negative NaN still beats "taken"
    }
    float mx = fmaxf(v[0], v[1]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    float sum = (lane < p.E ? expf(v[0] - mx) : 0.f) + (lane + 32 < p.E ? expf(v[1] - mx) : 0.f);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    float chosen = 0.f;                                    // lane k: the weight of choice k
    int which = 0;
    for (int k = 0; k < p.K; ++k) {
      const unsigned best = __reduce_max_sync(0xffffffffu, max(key[0], key[1]));
      const unsigned low = __ballot_sync(0xffffffffu, key[0] == best), high = __ballot_sync(0xffffffffu, key[1] == best);
      const int e = low != 0u ? __ffs(low) - 1 : 32 + __ffs(high) - 1;
      const float l = __shfl_sync(0xffffffffu, e < 32 ? v[0] : v[1], e & 31);
      if (lane == (e & 31)) key[e >> 5] = 0u;
      if (lane == k) { chosen = expf(l - mx) / sum; which = e; }
    }
    if (p.normalize) {
      float total = lane < p.K ? chosen : 0.f;
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
      chosen = chosen / fmaxf(total, 1.1920929e-07f);
    }
    if (lane < p.K) { r.expert[t * p.K + lane] = which; weight[t * p.K + lane] = chosen; }
  }
}

// ---- kernel 1: routing, gate and up projection, SwiGLU ----
template <int NT>
__global__ void __launch_bounds__(kThreads)
moe_up_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Routing r;
  __shared__ float weight[kRoutes];
  constexpr int COLS = 8 * NT, PITCH = COLS + 1;
  float* red = reinterpret_cast<float*>(smem);             // [warps][2][16][PITCH]
  float* logits = red;                                     // [T][E], before the first item needs `red`
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int routes = p.T * p.K;
  router_logits(p, logits);
  __syncthreads();
  choose_experts(p, logits, r, weight);
  __syncthreads();
  sort_routes(r, routes, p.E);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < routes; i += kThreads) p.routes[i] = r.expert[i];

  const int tiles = (p.I + 15) / 16, steps = (p.H + 31) / 32;
  for (int item = blockIdx.x; item < r.num_active * tiles; item += gridDim.x) {
    const int e = r.active[item / tiles], i0 = (item % tiles) * 16;
    const int n0 = r.first[e], n = r.first[e + 1] - n0, nts = (n + 7) / 8;
    const __nv_bfloat16* wrow[4];                          // gate rows g, g + 8 and up rows g, g + 8
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = min(i0 + g + 8 * u, p.I - 1);
      wrow[u] = p.gate_up + ((long long)e * 2 * p.I + row) * p.H + c * 8;
      wrow[2 + u] = wrow[u] + (long long)p.I * p.H;
    }
    const __nv_bfloat16* xrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) xrow[j] = p.x + (long long)(r.order[n0 + min(j * 8 + g, n - 1)] / p.K) * p.ldx + c * 8;
    float acc[2][NT][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
    constexpr int UNROLL = 4;
    for (int s0 = warp; s0 < steps; s0 += kWarps * UNROLL) {
      uint4 a[UNROLL][4];
#pragma unroll
      for (int q = 0; q < UNROLL; ++q) {
        const int s = s0 + q * kWarps;
        const bool ok = s * 32 + c * 8 < p.H;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          a[q][i] = ok ? __ldg(reinterpret_cast<const uint4*>(wrow[i] + s * 32)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int q = 0; q < UNROLL; ++q) {
        const int s = s0 + q * kWarps;
        const bool ok = s * 32 + c * 8 < p.H;
        if (s >= steps) break;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j >= nts) break;
          const uint4 b = ok ? __ldg(reinterpret_cast<const uint4*>(xrow[j] + s * 32)) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            mma_bf16(acc[m][j], a[q][2 * m].x, a[q][2 * m + 1].x, a[q][2 * m].y, a[q][2 * m + 1].y, b.x, b.y);
            mma_bf16(acc[m][j], a[q][2 * m].z, a[q][2 * m + 1].z, a[q][2 * m].w, a[q][2 * m + 1].w, b.z, b.w);
          }
        }
      }
    }
    __syncthreads();                                       // the previous item's readers (or the routing's) are done with `red`
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j < nts) red[((warp * 2 + m) * 16 + g + 8 * (i >> 1)) * PITCH + j * 8 + 2 * c + (i & 1)] = acc[m][j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * n; i += kThreads) {
      const int row = i & 15, col = i >> 4;
      if (i0 + row >= p.I) continue;
      float gate = 0.f, up = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        gate += red[((w * 2 + 0) * 16 + row) * PITCH + col];
        up += red[((w * 2 + 1) * 16 + row) * PITCH + col];
      }
      const int route = r.order[n0 + col];
      const float h = gate / (1.f + expf(-gate)) * up * weight[route];
      const __nv_bfloat16 high = __float2bfloat16_rn(h);
      __nv_bfloat16* dst = p.hidden + (long long)route * p.I + i0 + row;
      dst[0] = high;
      dst[(long long)routes * p.I] = __float2bfloat16_rn(h - __bfloat162float(high));
    }
  }
}

// ---- kernel 2: down projection, summed over the experts of each token ----
template <int NT>
__global__ void __launch_bounds__(kThreads)
moe_down_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Routing r;
  float* sums = reinterpret_cast<float*>(smem);            // [warps][T][16]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int routes = p.T * p.K;
  cg::cluster_group cluster = cg::this_cluster();
  const int shares = int(cluster.num_blocks()), share = int(cluster.block_rank());
  for (int i = threadIdx.x; i < routes; i += kThreads) r.expert[i] = p.routes[i];
  for (int i = threadIdx.x; i < kWarps * p.T * 16; i += kThreads) sums[i] = 0.f;
  __syncthreads();
  sort_routes(r, routes, p.E);

  const int row0 = (blockIdx.x / shares) * 16;
  const int steps = (p.I + 31) / 32;
  const long long total = (long long)r.num_active * steps;
  const int workers = shares * kWarps, me = share * kWarps + warp;
  long long at = total * me / workers;
  const long long end = total * (me + 1) / workers;
  float* mine = sums + warp * p.T * 16;
  while (at < end) {
    const int ai = int(at / steps), e = r.active[ai];
    const int s_begin = int(at % steps), s_end = int(min((long long)steps, s_begin + (end - at)));
    at += s_end - s_begin;
    const int n0 = r.first[e], n = r.first[e + 1] - n0, nts = (n + 7) / 8;
    const __nv_bfloat16* wrow[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) wrow[u] = p.down + ((long long)e * p.H + min(row0 + g + 8 * u, p.H - 1)) * p.I + c * 8;
    const __nv_bfloat16* hrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) hrow[j] = p.hidden + (long long)r.order[n0 + min(j * 8 + g, n - 1)] * p.I + c * 8;
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    constexpr int UNROLL = 8;
    for (int s0 = s_begin; s0 < s_end; s0 += UNROLL) {
      uint4 a[UNROLL][2];
#pragma unroll
      for (int q = 0; q < UNROLL; ++q) {
        const bool ok = s0 + q < s_end && (s0 + q) * 32 + c * 8 < p.I;
#pragma unroll
        for (int u = 0; u < 2; ++u) a[q][u] = ok ? __ldg(reinterpret_cast<const uint4*>(wrow[u] + (s0 + q) * 32)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int q = 0; q < UNROLL; ++q) {
        if (s0 + q >= s_end) break;
        const bool ok = (s0 + q) * 32 + c * 8 < p.I;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j >= nts) break;
          const __nv_bfloat16* src = hrow[j] + (s0 + q) * 32;
          const uint4 bh = ok ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
          const uint4 bl = ok ? *reinterpret_cast<const uint4*>(src + (long long)routes * p.I) : make_uint4(0, 0, 0, 0);
          mma_bf16(acc[j], a[q][0].x, a[q][1].x, a[q][0].y, a[q][1].y, bh.x, bh.y);
          mma_bf16(acc[j], a[q][0].z, a[q][1].z, a[q][0].w, a[q][1].w, bh.z, bh.w);
          mma_bf16(acc[j], a[q][0].x, a[q][1].x, a[q][0].y, a[q][1].y, bl.x, bl.y);
          mma_bf16(acc[j], a[q][0].z, a[q][1].z, a[q][0].w, a[q][1].w, bl.z, bl.w);
        }
      }
    }
    // an expert has a token at most once, so the lanes of a warp write different sums
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = j * 8 + 2 * c + (i & 1);
        if (col < n) mine[(r.order[n0 + col] / p.K) * 16 + g + 8 * (i >> 1)] += acc[j][i];
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * 16; i += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += sums[w * p.T * 16 + i];
    sums[i] = v;                                           // slot i of warp 0: read by this thread only
  }
  cluster.sync();
  for (int i = share * kThreads + threadIdx.x; i < p.T * 16; i += shares * kThreads) {
    const int t = i >> 4, row = row0 + (i & 15);
    float v = 0.f;
    for (int s = 0; s < shares; ++s) v += cluster.map_shared_rank(sums, s)[i];
    if (row < p.H) p.y[(long long)t * p.H + row] = __float2bfloat16_rn(v);
  }
  cluster.sync();                                          // nobody leaves while its sums may still be read
}

template <int NT>
cudaError_t launch_typed(const Params& p, cudaStream_t stream) {
  const size_t red = size_t(kWarps) * 2 * 16 * (8 * NT + 1) * 4, logits = size_t(p.T) * p.E * 4;
  const size_t up_smem = red > logits ? red : logits, down_smem = size_t(kWarps) * p.T * 16 * 4;
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev]) {
    const int most = int(size_t(kWarps) * 2 * 16 * (8 * NT + 1) * 4 > size_t(8 * NT) * kExperts * 4 ? size_t(kWarps) * 2 * 16 * (8 * NT + 1) * 4
                                                                                                    : size_t(8 * NT) * kExperts * 4);
    err = cudaFuncSetAttribute(moe_up_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (err != cudaSuccess) return err;
    ready[dev] = true;
  }
  const int sms = device_sm_count();
  const long long experts = (long long)p.T * p.K < p.E ? (long long)p.T * p.K : p.E;
  const long long items = experts * ((p.I + 15) / 16), cap = 2LL * sms;
  moe_up_kernel<NT><<<unsigned(items < cap ? items : cap), kThreads, up_smem, stream>>>(p);
  ++g_launch_count;
  if ((err = cudaGetLastError()) != cudaSuccess) return err;

  const int row_tiles = (p.H + 15) / 16;
  int shares = 1;
  while (shares < 8 && row_tiles * shares < 2 * sms) shares *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(row_tiles * shares));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = down_smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(shares);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, moe_down_kernel<NT>, p);
  ++g_launch_count;
  return err;
}

}  // namespace

cudaError_t launch_moe_tokens(const MoeTokensArgs& a) {
  Params p;
  p.x = static_cast<const __nv_bfloat16*>(a.x); p.ldx = a.ldx;
  p.router = a.router; p.router_bf16 = a.router_bf16;
  p.gate_up = static_cast<const __nv_bfloat16*>(a.gate_up); p.down = static_cast<const __nv_bfloat16*>(a.down);
  p.y = static_cast<__nv_bfloat16*>(a.y); p.hidden = static_cast<__nv_bfloat16*>(a.hidden); p.routes = a.routes;
  p.T = a.T; p.E = a.E; p.K = a.K; p.H = a.H; p.I = a.I; p.normalize = a.normalize;
  if (a.T < 1 || a.T > kMoeTokensMax || a.E < 1 || a.E > kExperts || a.K < 1 || a.K > kTopK || a.K > a.E || a.H % 8 != 0 || a.I % 8 != 0)
    return cudaErrorInvalidValue;
  if (a.T <= 8) return launch_typed<1>(p, a.stream);
  if (a.T <= 16) return launch_typed<2>(p, a.stream);
  if (a.T <= 32) return launch_typed<4>(p, a.stream);
  return launch_typed<8>(p, a.stream);
}

}  // namespace mts
