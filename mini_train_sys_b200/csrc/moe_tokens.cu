// A whole mixture-of-experts layer for a few tokens in two kernels.
//
//   p = softmax(x Wr^T);  the K largest (ties to the lower expert), optionally divided by their sum
//   y = sum_k w_k Wd[e_k] (silu(Wg[e_k] x) * (Wu[e_k] x))
//
// What bounds it: reading the weights of every expert that has a token, 6 H I bytes each, once.  Weight rows are the row operand of
// m16n8k16 and the tokens of their expert the columns (8 at a time), so one pass over the weights serves up to 64 tokens.  Every warp
// streams its own weight tiles through a ring in shared memory, 4 KB a TMA copy and 16 or 20 KB in flight a warp, across the ends of
// items: 128 to 160 KB in flight an SM, and no barrier between warps inside a stream.
//   1  every CTA (or cluster, where the router is large) routes all tokens for itself; then a warp takes (expert, 8 columns of the
//      hidden layer) items: 8 gate rows and 8 up rows are one tile, so a lane ends up with both factors of its hidden values and
//      applies SwiGLU in registers.  The hidden value is multiplied by the route's weight, so that the sums of the second
//      kernel are over the experts already.
//   2  the (32 output rows, expert, 64 columns) units of the down projections are one list, cut into equal parts for the CTAs; what
//      a CTA has of a row tile is added in shared memory, and where a tile was cut its last CTA adds the parts, in order.
//
// Rounding: logits, softmax, sums and the hidden values are fp32 (the router's fp32 weight enters the tensor cores as the sum of three
// bf16 values, 24 bits); a hidden value enters the second product as the sum of two (2^-16), so y is rounded to bf16 once.
#include "decode.cuh"
#include "ops.cuh"
#include "mma_sync.cuh"
#include "ptx_sm100.cuh"

#include <cooperative_groups.h>
#include <cudaTypedefs.h>
#include <math_constants.h>

#include <mutex>

namespace mts {

namespace {

namespace cg = cooperative_groups;

constexpr int kExperts = 64;
constexpr int kTopK = 8;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRoutes = kMoeTokensMax * kTopK;
constexpr int kTile = 4096;              // bytes of a copy: 16 rows x 128 columns (gate and up), 32 x 64 (down)
constexpr int kUpCols = 128, kUpRows = 8, kDownCols = 64, kDownRows = 32;
constexpr int kStagesMax = 5;
constexpr int kSumPitch = kDownRows + 1;
// Five stages of ring a warp, four where the sums of more than 32 tokens need the room.
__host__ __device__ constexpr int ring_stages(int T) { return T > 32 ? 4 : 5; }
__host__ __device__ constexpr int ring_bytes(int T) { return kWarps * ring_stages(T) * kTile; }

// Routes by expert: `order` holds the routes of expert e, ascending, at [first[e], first[e + 1]); `active` the experts with one.
struct Routing {
  int expert[kRoutes];
  int order[kRoutes];
  int first[kExperts + 1];
  int active[kExperts];
  int num_active;
};

struct Params {
  const __nv_bfloat16* x;
  long long ldx;
  const void* router;
  int router_bf16;
  __nv_bfloat16* y;
  __nv_bfloat16* hidden;       // [2][T * K][I]: high and low part
  Routing* routing;            // written by the first kernel for the second
  unsigned* arrived;           // [row tiles] parts of a row tile that are there; zeroed by the first kernel
  float* part;                 // [2 * CTAs][T][32]
  int* status;
  int T, E, K, H, I, normalize;
};

__device__ __forceinline__ int cut(int N, int i, int n) { return int((long long)N * i / n); }
__device__ __forceinline__ int owner(int N, int u, int n) { return int(((long long)(u + 1) * n - 1) / N); }

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

// The ring of one warp.  Lane 0 starts copies; a stage is free once every lane has taken its fragments.
struct Ring {
  uint8_t* base;
  uint64_t* bars;
  int* status;
  int stages, lane;
  int put = 0, get = 0;        // stage of the next copy, of the next tile
  uint32_t parity = 0;
  bool lost = false;           // a copy did not come in time: the rest is not waited for, the host sees the status

  __device__ __forceinline__ void init() {
    if (lane == 0) {
      for (int s = 0; s < stages; ++s) mbar_init(&bars[s], 1);
      mbar_fence_init();
    }
    __syncwarp();
  }
  __device__ __forceinline__ void copy(const CUtensorMap* map, int x, int y, int z) {
    if (lane == 0) {
      mbar_expect_tx(&bars[put], kTile);
      tma_load_3d(base + put * kTile, map, &bars[put], x, y, z);
    }
    if (++put == stages) put = 0;
  }
  __device__ __forceinline__ const uint8_t* wait() {
    if (!lost && !mbar_test(&bars[get], parity)) {
      const uint64_t t0 = global_timer_ns();
      while (!mbar_test(&bars[get], parity))
        if (global_timer_ns() - t0 > kWaitDeadlineNs) {
          lost = true;
          if (lane == 0) atomicMax(status, int(STATUS_WAIT_TIMEOUT));
          break;
        }
    }
    return base + get * kTile;
  }
  __device__ __forceinline__ void taken() {
    __syncwarp();
    if (++get == stages) { get = 0; parity ^= 1; }
  }
  __device__ __forceinline__ void finish() {
    if (!lost) return;         // copies may still be on their way: give them time before the memory changes hands
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000000ull) __nanosleep(1000);
  }
};

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

// One warp a token: K rounds of arg-max over the logits (two experts a lane), then the softmax of the chosen ones.
// The tokens of this CTA are rank, rank + ranks, ...
__device__ __forceinline__ void choose_experts(const Params& p, const float* logits, Routing& r, float* weight, int rank, int ranks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int t = rank + ranks * warp; t < p.T; t += ranks * kWarps) {
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

// Three bf16 values whose sum is v to 24 bits.
__device__ __forceinline__ void split3(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
  h = pack_bf162(a, b);
  const float a1 = a - __uint_as_float(h << 16), b1 = b - __uint_as_float(h & 0xFFFF0000u);
  m = pack_bf162(a1, b1);
  l = pack_bf162(a1 - __uint_as_float(m << 16), b1 - __uint_as_float(m & 0xFFFF0000u));
}

// Partial logits part[warp][e][t] of this CTA's share of the contraction: 32 columns a warp and step, experts in tiles of 16 as rows.
template <int MT, int NT, int UNROLL>
__device__ __forceinline__ void router_products(const Params& p, float* part, int worker, int workers) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int E16 = (p.E + 15) & ~15, T8 = (p.T + 7) & ~7;
  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
#pragma unroll UNROLL
  for (int q = worker; q * 32 < p.H; q += workers) {
    const int k = q * 32 + c * 8;
    const bool in = k < p.H;
    uint4 b[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      b[j] = make_uint4(0, 0, 0, 0);
      if (in && j * 8 < p.T) b[j] = __ldg(reinterpret_cast<const uint4*>(p.x + min(j * 8 + g, p.T - 1) * p.ldx + k));
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m * 16 >= p.E) break;
      uint32_t hi[2][4], mid[2][4], low[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const long long at = (long long)min(m * 16 + g + 8 * u, p.E - 1) * p.H + k;
        if (p.router_bf16) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (in) w = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.router) + at));
          hi[u][0] = w.x; hi[u][1] = w.y; hi[u][2] = w.z; hi[u][3] = w.w;
        } else {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f), w = v;
          if (in) {
            v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.router) + at));
            w = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.router) + at) + 1);
          }
          split3(v.x, v.y, hi[u][0], mid[u][0], low[u][0]);
          split3(v.z, v.w, hi[u][1], mid[u][1], low[u][1]);
          split3(w.x, w.y, hi[u][2], mid[u][2], low[u][2]);
          split3(w.z, w.w, hi[u][3], mid[u][3], low[u][3]);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (j * 8 >= p.T) break;
        if (!p.router_bf16) {          // the small parts first
          mma_bf16(acc[m][j], low[0][0], low[1][0], low[0][1], low[1][1], b[j].x, b[j].y);
          mma_bf16(acc[m][j], low[0][2], low[1][2], low[0][3], low[1][3], b[j].z, b[j].w);
          mma_bf16(acc[m][j], mid[0][0], mid[1][0], mid[0][1], mid[1][1], b[j].x, b[j].y);
          mma_bf16(acc[m][j], mid[0][2], mid[1][2], mid[0][3], mid[1][3], b[j].z, b[j].w);
        }
        mma_bf16(acc[m][j], hi[0][0], hi[1][0], hi[0][1], hi[1][1], b[j].x, b[j].y);
        mma_bf16(acc[m][j], hi[0][2], hi[1][2], hi[0][3], hi[1][3], b[j].z, b[j].w);
      }
    }
  }
  float* mine = part + (threadIdx.x >> 5) * (E16 * T8);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (m * 16 < p.E && j * 8 < p.T) mine[(m * 16 + g + 8 * (i >> 1)) * T8 + j * 8 + 2 * c + (i & 1)] = acc[m][j][i];
}

// ---- kernel 1: routing, gate and up projection, SwiGLU ----
template <bool CLUSTER>
__global__ void __launch_bounds__(kThreads)
moe_up_kernel(const __grid_constant__ CUtensorMap weights, const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Routing r;
  __shared__ float weight[kRoutes];
  __shared__ uint64_t bars[kWarps][kStagesMax];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int routes = p.T * p.K;
  float* part = reinterpret_cast<float*>(smem);            // partial logits, before the rings are used
  float* logits = reinterpret_cast<float*>(smem + ring_bytes(p.T));                       // [T][E]
  const int E16 = (p.E + 15) & ~15, T8 = (p.T + 7) & ~7;
  int rank = 0, ranks = 1;
  if constexpr (CLUSTER) {
    rank = int(cg::this_cluster().block_rank());
    ranks = int(cg::this_cluster().num_blocks());
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) tma_prefetch_desc(&weights);
  if (p.E <= 16 && p.T <= 8) router_products<1, 1, 4>(p, part, rank * kWarps + warp, ranks * kWarps);
  else router_products<4, 8, 1>(p, part, rank * kWarps + warp, ranks * kWarps);
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * p.E; i += kThreads) {
    const int t = i / p.E, e = i % p.E;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += part[w * (E16 * T8) + e * T8 + t];
    logits[i] = v;
  }
  if constexpr (CLUSTER) {
    // every CTA adds the shares of its tokens, chooses for them and tells the others
    cg::cluster_group cluster = cg::this_cluster();
    float* full = part;
    cluster.sync();
    for (int i = threadIdx.x; i < p.T * p.E; i += kThreads) {
      if (i / p.E % ranks != rank) continue;
      float v = 0.f;
      for (int k = 0; k < ranks; ++k) v += cluster.map_shared_rank(logits, k)[i];
      full[i] = v;
    }
    __syncthreads();
    choose_experts(p, full, r, weight, rank, ranks);
    __syncthreads();
    for (int i = threadIdx.x; i < routes; i += kThreads)
      if (i / p.K % ranks == rank)
        for (int k = 0; k < ranks; ++k)
          if (k != rank) {
            cluster.map_shared_rank(r.expert, k)[i] = r.expert[i];
            cluster.map_shared_rank(weight, k)[i] = weight[i];
          }
    cluster.sync();
  } else {
    __syncthreads();
    choose_experts(p, logits, r, weight, 0, 1);
    __syncthreads();
  }
  sort_routes(r, routes, p.E);
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < routes; i += kThreads) p.routing->order[i] = r.order[i];
    for (int i = threadIdx.x; i <= p.E; i += kThreads) p.routing->first[i] = r.first[i];
    for (int i = threadIdx.x; i < r.num_active; i += kThreads) p.routing->active[i] = r.active[i];
    if (threadIdx.x == 0) p.routing->num_active = r.num_active;
    for (int i = threadIdx.x; i < (p.H + kDownRows - 1) / kDownRows; i += kThreads) p.arrived[i] = 0u;
  }

  const int tiles = (p.I + kUpRows - 1) / kUpRows, steps = (p.H + kUpCols - 1) / kUpCols;
  const int N = r.num_active * tiles;
  const int c0 = cut(N, blockIdx.x, gridDim.x), c1 = cut(N, blockIdx.x + 1, gridDim.x);
  const int i0 = c0 + cut(c1 - c0, warp, kWarps), i1 = c0 + cut(c1 - c0, warp + 1, kWarps);
  if (i0 == i1) return;
  Ring ring;
  ring.stages = ring_stages(p.T);
  ring.base = smem + warp * ring.stages * kTile;
  ring.bars = bars[warp];
  ring.status = p.status;
  ring.lane = lane;
  ring.init();
  int ahead = i0, ahead_step = 0;
  auto next_copy = [&]() {
    if (ahead == i1) return;
    ring.copy(&weights, ahead_step * kUpCols, ahead % tiles * kUpRows, 2 * r.active[ahead / tiles]);
    if (++ahead_step == steps) { ahead_step = 0; ++ahead; }
  };
  fence_proxy_async_smem();              // the ring's memory held partial logits
  __syncwarp();
  for (int s = 0; s < ring.stages; ++s) next_copy();

  for (int item = i0; item < i1; ++item) {
    const int e = r.active[item / tiles], row = item % tiles * kUpRows + g;
    const int n0 = r.first[e], n = r.first[e + 1] - n0, nts = (n + 7) / 8;
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    for (int step = 0; step < steps; ++step) {
      const int k = step * kUpCols + c * 8;
      uint4 b[4];
      auto load_x = [&](int j) {
        const __nv_bfloat16* src = p.x + (long long)(r.order[n0 + min(j * 8 + g, n - 1)] / p.K) * p.ldx + k;
#pragma unroll
        for (int s = 0; s < 4; ++s) b[s] = k + 32 * s < p.H ? __ldg(reinterpret_cast<const uint4*>(src + 32 * s)) : make_uint4(0, 0, 0, 0);
      };
      load_x(0);
      const uint8_t* tile = ring.wait() + g * (kUpCols * 2) + c * 16;
      uint4 a[4][2];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) a[s][u] = *reinterpret_cast<const uint4*>(tile + u * (kUpRows * kUpCols * 2) + s * 64);
      ring.taken();
      next_copy();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j >= nts) break;
        if (j > 0) load_x(j);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          mma_bf16(acc[j], a[s][0].x, a[s][1].x, a[s][0].y, a[s][1].y, b[s].x, b[s].y);
          mma_bf16(acc[j], a[s][0].z, a[s][1].z, a[s][0].w, a[s][1].w, b[s].z, b[s].w);
        }
      }
    }
    if (row >= p.I) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = j * 8 + 2 * c + i;
        if (col >= n) continue;
        const int route = r.order[n0 + col];
        const float gate = acc[j][i], up = acc[j][i + 2];
        const float h = gate / (1.f + expf(-gate)) * up * weight[route];
        const __nv_bfloat16 high = __float2bfloat16_rn(h);
        __nv_bfloat16* dst = p.hidden + (long long)route * p.I + row;
        dst[0] = high;
        dst[(long long)routes * p.I] = __float2bfloat16_rn(h - __bfloat162float(high));
      }
  }
  ring.finish();
}

// ---- kernel 2: down projection, summed over the experts of each token ----
__global__ void __launch_bounds__(kThreads)
moe_down_kernel(const __grid_constant__ CUtensorMap weights, const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Routing r;
  __shared__ uint64_t bars[kWarps][kStagesMax];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int routes = p.T * p.K, sum_size = p.T * kSumPitch;
  float* sums = reinterpret_cast<float*>(smem + ring_bytes(p.T));                         // [warps][T][pitch]
  for (int i = threadIdx.x; i < kWarps * sum_size; i += kThreads) sums[i] = 0.f;
  if (threadIdx.x == 0) tma_prefetch_desc(&weights);
  Ring ring;
  ring.stages = ring_stages(p.T);
  ring.base = smem + warp * ring.stages * kTile;
  ring.bars = bars[warp];
  ring.status = p.status;
  ring.lane = lane;
  ring.init();
  asm volatile("griddepcontrol.wait;" ::: "memory");       // what follows reads what the first kernel wrote
  for (int i = threadIdx.x; i < routes; i += kThreads) r.order[i] = __ldcg(&p.routing->order[i]);
  for (int i = threadIdx.x; i <= p.E; i += kThreads) r.first[i] = __ldcg(&p.routing->first[i]);
  const int live = __ldcg(&p.routing->num_active);
  for (int i = threadIdx.x; i < live; i += kThreads) r.active[i] = __ldcg(&p.routing->active[i]);
  __syncthreads();

  const int steps = (p.I + kDownCols - 1) / kDownCols, tiles = (p.H + kDownRows - 1) / kDownRows;
  const int per_tile = live * steps, N = tiles * per_tile, parts = min(int(gridDim.x), N);
  if (int(blockIdx.x) >= parts) return;
  const int c0 = cut(N, blockIdx.x, parts), c1 = cut(N, blockIdx.x + 1, parts);
  // The units of this warp: its share of what the CTA has of each row tile, one after the other.
  struct Stream {
    int tile, u, end;
  };
  auto enter = [&](Stream& s) {          // the first row tile from s.tile on that has units for this warp
    for (; s.tile * per_tile < c1; ++s.tile) {
      const int s0 = max(c0, s.tile * per_tile), s1 = min(c1, (s.tile + 1) * per_tile);
      s.u = s0 + cut(s1 - s0, warp, kWarps);
      s.end = s0 + cut(s1 - s0, warp + 1, kWarps);
      if (s.u < s.end) return;
    }
    s.u = s.end = 0;
  };
  Stream ahead{c0 / per_tile, 0, 0};
  enter(ahead);
  auto next_copy = [&]() {
    if (ahead.u == ahead.end) return;
    const int rest = ahead.u - ahead.tile * per_tile;
    ring.copy(&weights, rest % steps * kDownCols, ahead.tile * kDownRows, r.active[rest / steps]);
    if (++ahead.u == ahead.end) { ++ahead.tile; enter(ahead); }
  };
  for (int s = 0; s < ring.stages; ++s) next_copy();

  float* mine = sums + warp * sum_size;
  for (int tile = c0 / per_tile; tile * per_tile < c1; ++tile) {
    const int s0 = max(c0, tile * per_tile), s1 = min(c1, (tile + 1) * per_tile);
    int u = s0 + cut(s1 - s0, warp, kWarps);
    const int end = s0 + cut(s1 - s0, warp + 1, kWarps);
    while (u < end) {
      const int rest = u - tile * per_tile, ai = rest / steps, e = r.active[ai];
      const int step0 = rest % steps, step1 = min(steps, step0 + end - u);
      u += step1 - step0;
      const int n0 = r.first[e], n = r.first[e + 1] - n0, nts = (n + 7) / 8;
      float acc[2][8][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
      for (int step = step0; step < step1; ++step) {
        const int k = step * kDownCols + c * 8;
        uint4 b[2][2];
        auto load_h = [&](int j) {
          const __nv_bfloat16* src = p.hidden + (long long)r.order[n0 + min(j * 8 + g, n - 1)] * p.I + k;
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int v = 0; v < 2; ++v)
              b[s][v] = k + 32 * s < p.I ? *reinterpret_cast<const uint4*>(src + (long long)v * routes * p.I + 32 * s) : make_uint4(0, 0, 0, 0);
        };
        load_h(0);
        const uint8_t* at = ring.wait() + g * (kDownCols * 2) + c * 16;
        uint4 a[2][2][2];                // [row tile of 16][32 columns][rows g, g + 8]
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int v = 0; v < 2; ++v) a[m][s][v] = *reinterpret_cast<const uint4*>(at + (16 * m + 8 * v) * (kDownCols * 2) + s * 64);
        ring.taken();
        next_copy();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= nts) break;
          if (j > 0) load_h(j);
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int v = 1; v >= 0; --v)
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                mma_bf16(acc[m][j], a[m][s][0].x, a[m][s][1].x, a[m][s][0].y, a[m][s][1].y, b[s][v].x, b[s][v].y);
                mma_bf16(acc[m][j], a[m][s][0].z, a[m][s][1].z, a[m][s][0].w, a[m][s][1].w, b[s][v].z, b[s][v].w);
              }
        }
      }
      // an expert has a token at most once, so the lanes of a warp write different sums
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j >= nts) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = j * 8 + 2 * c + i;
          if (col >= n) continue;
          float* dst = mine + r.order[n0 + col] / p.K * kSumPitch + g;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            dst[16 * m] += acc[m][j][i];
            dst[16 * m + 8] += acc[m][j][i + 2];
          }
        }
      }
    }
    // ---- what the CTA has of this row tile ----
    __syncthreads();
    const bool whole = s0 == tile * per_tile && s1 == (tile + 1) * per_tile;
    float* own = p.part + (2 * (long long)blockIdx.x + (s0 == tile * per_tile ? 1 : 0)) * p.T * kDownRows;
    for (int i = threadIdx.x; i < p.T * kDownRows; i += kThreads) {
      const int t = i / kDownRows, row = i % kDownRows;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        float* s = sums + w * sum_size + t * kSumPitch + row;
        v += *s;
        *s = 0.f;
      }
      if (!whole) own[i] = v;
      else if (tile * kDownRows + row < p.H) p.y[(long long)t * p.H + tile * kDownRows + row] = __float2bfloat16_rn(v);
    }
    if (!whole) {
      const int f = owner(N, tile * per_tile, parts), l = owner(N, (tile + 1) * per_tile - 1, parts);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        last = atomicAdd(&p.arrived[tile], 1u) == unsigned(l - f);
        __threadfence();
      }
      __syncthreads();
      if (last)
        for (int i = threadIdx.x; i < p.T * kDownRows; i += kThreads) {
          const int t = i / kDownRows, row = tile * kDownRows + i % kDownRows;
          float v = 0.f;
#pragma unroll 8
          for (int k = f; k <= l; ++k)
            v += __ldcg(p.part + (2 * (long long)k + (cut(N, k, parts) <= tile * per_tile ? 1 : 0)) * p.T * kDownRows + i);
          if (row < p.H) p.y[(long long)t * p.H + row] = __float2bfloat16_rn(v);
        }
    }
    __syncthreads();                     // the sums are zero again, `last` is read
  }
  ring.finish();
}

// ---- host side ----
// [planes, rows, cols] bf16, cut into boxes of box_planes x box_rows x box_cols; what lies outside reads zero.
bool encode_weights(CUtensorMap* map, const void* base, long long cols, long long rows, long long planes, int box_cols, int box_rows, int box_planes) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(planes)};
  const cuuint64_t strides[2] = {cuuint64_t(cols) * 2, cuuint64_t(cols) * cuuint64_t(rows) * 2};
  const cuuint32_t box[3] = {cuuint32_t(box_cols), cuuint32_t(box_rows), cuuint32_t(box_planes)};
  const cuuint32_t elem[3] = {1u, 1u, 1u};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kCluster = 4;

size_t up_shared(int T, int E) { return size_t(ring_bytes(T)) + size_t(T) * E * 4; }
size_t down_shared(int T) { return size_t(ring_bytes(T)) + size_t(kWarps) * T * kSumPitch * 4; }

// What a launch needs to know of a device, found once.
struct DeviceFacts {
  std::once_flag once;
  cudaError_t error = cudaSuccess;
  int sms = 0, clustered = 0;            // CTAs of the first kernel that are resident at once in clusters
};
DeviceFacts& facts(int dev) {
  static DeviceFacts all[64];
  DeviceFacts& f = all[dev];
  std::call_once(f.once, [&f] {
    const int up = int(up_shared(kMoeTokensMax, kExperts) > up_shared(32, kExperts) ? up_shared(kMoeTokensMax, kExperts) : up_shared(32, kExperts));
    const int down = int(down_shared(kMoeTokensMax) > down_shared(32) ? down_shared(kMoeTokensMax) : down_shared(32));
    f.sms = device_sm_count();
    if ((f.error = cudaFuncSetAttribute(moe_up_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, up)) != cudaSuccess) return;
    if ((f.error = cudaFuncSetAttribute(moe_up_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, up)) != cudaSuccess) return;
    if ((f.error = cudaFuncSetAttribute(moe_down_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, down)) != cudaSuccess) return;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(f.sms / kCluster * kCluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = size_t(up);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if ((f.error = cudaOccupancyMaxActiveClusters(&clusters, moe_up_kernel<true>, &cfg)) != cudaSuccess) return;
    f.clustered = clusters * kCluster < f.sms ? clusters * kCluster : f.sms / kCluster * kCluster;
    if (f.clustered < kCluster) f.error = cudaErrorInvalidConfiguration;
  });
  return f;
}

struct Workspace {                       // byte offsets of its parts
  size_t hidden, part, arrived, total;
};
Workspace workspace_of(int T, int K, int H, int I) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Workspace w;
  w.hidden = up(sizeof(Routing));
  w.part = w.hidden + up(size_t(2) * T * K * I * 2);
  w.arrived = w.part + up(size_t(2) * device_sm_count() * T * kDownRows * 4);
  w.total = w.arrived + up(size_t((H + kDownRows - 1) / kDownRows) * 4);
  return w;
}

}  // namespace

size_t moe_tokens_workspace_bytes(int T, int K, int H, int I) { return workspace_of(T, K, H, I).total; }

cudaError_t launch_moe_tokens(const MoeTokensArgs& a) {
  if (a.T < 1 || a.T > kMoeTokensMax || a.E < 1 || a.E > kExperts || a.K < 1 || a.K > kTopK || a.K > a.E || a.H % 8 != 0 || a.I % 8 != 0)
    return cudaErrorInvalidValue;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  static thread_local int bound = -1;    // the tensor-map encoder needs the device's context on this thread
  if (bound != dev) {
    if ((err = cudaSetDevice(dev)) != cudaSuccess) return err;
    bound = dev;
  }
  DeviceFacts& f = facts(dev);
  if (f.error != cudaSuccess) return f.error;
  const Workspace w = workspace_of(a.T, a.K, a.H, a.I);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  Params p;
  p.x = static_cast<const __nv_bfloat16*>(a.x); p.ldx = a.ldx;
  p.router = a.router; p.router_bf16 = a.router_bf16;
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.routing = reinterpret_cast<Routing*>(ws);
  p.hidden = reinterpret_cast<__nv_bfloat16*>(ws + w.hidden);
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.arrived = reinterpret_cast<unsigned*>(ws + w.arrived);
  p.status = a.status;
  p.T = a.T; p.E = a.E; p.K = a.K; p.H = a.H; p.I = a.I; p.normalize = a.normalize;
  CUtensorMap up, down;
  if (!encode_weights(&up, a.gate_up, a.H, a.I, 2LL * a.E, kUpCols, kUpRows, 2) ||
      !encode_weights(&down, a.down, a.I, a.H, a.E, kDownCols, kDownRows, 1))
    return cudaErrorInvalidValue;

  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(kThreads);
  cfg.stream = a.stream;
  cfg.attrs = attr;
  // What a CTA reads to route by itself (x and the router's weight, from L2); above 256 KB four CTAs share it.
  const long long routing = (long long)a.E * a.H * (a.router_bf16 ? 2 : 4) + (long long)a.T * a.H * 2;
  cfg.dynamicSmemBytes = up_shared(a.T, a.E);
  ++g_launch_count;
  if (routing > 256 * 1024) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(unsigned(f.clustered));
    err = cudaLaunchKernelEx(&cfg, moe_up_kernel<true>, up, p);
  } else {
    cfg.gridDim = dim3(unsigned(f.sms));
    err = cudaLaunchKernelEx(&cfg, moe_up_kernel<false>, up, p);
  }
  if (err != cudaSuccess) return err;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(unsigned(f.sms));
  cfg.dynamicSmemBytes = down_shared(a.T);
  ++g_launch_count;
  return cudaLaunchKernelEx(&cfg, moe_down_kernel, down, p);
}

}  // namespace mts
