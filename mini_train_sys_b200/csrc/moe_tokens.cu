// A whole mixture-of-experts layer for a few tokens in two kernels (three where the router is large).
//
//   p = softmax(x Wr^T);  the K largest (ties to the lower expert), optionally divided by their sum
//   y = sum_k w_k Wd[e_k] (silu(Wg[e_k] x) * (Wu[e_k] x))
//
// What bounds it: reading the weights of every expert that has a token, 6 H I bytes each, once.  Weight rows are the row operand of
// m16n8k16 and the tokens of their expert the columns (8 at a time), so one pass over an expert's weights serves up to 32 of its
// tokens, and an expert with more is streamed again for every 32.  Every warp streams its own weight tiles
// through a ring in shared memory, 8 KB a TMA copy and 16 or 24 KB in flight a warp, across the ends of items: 128 to 192 KB in
// flight an SM, and no barrier between warps inside a stream.
//   0  Routing reads x and the router's weight.  Up to 48 KB of them every CTA of the first kernel reads for itself (a launch costs
//      more); above that one cluster of eight CTAs routes in a kernel of its own.
//   1  A warp takes (entry, 8 columns of the hidden layer) items, an entry being an expert and its tokens: 8 gate rows and 8 up rows
//      are one tile, so a lane ends up with both factors of its hidden values and applies SwiGLU in registers.  The hidden value
//      is multiplied by the route's weight, so that the sums of the second kernel are over the experts already.
//   2  The (32 output rows, expert, 128 columns) units of the down projections are one list, cut into equal parts for the CTAs; what
//      a CTA has of a row tile is added in shared memory, and where a tile was cut its last CTA adds the parts, in order.
//
// Measured on the GPU (replayed graph, caches flushed): one token, 2 of 8 experts of 768 x 1,024, 12.1 us (9.4 MB of weights: two launches'
// latency); 64 tokens of the same 30.5 us (38 MB); 17 tokens, 8 of 64 experts of 2,048 x 1,024, 133 us (58 of them asked for, 0.73 GB,
// 5.5 TB/s, the routing kernel's 11 us included); 8 tokens, 2 of 8 experts of 4,096 x 14,336, 386 us where they ask for seven (2.47 GB,
// 6.4 TB/s), some 440 where for all eight.
//
// Rounding: logits, softmax, sums and the hidden values are fp32 (the router's fp32 weight enters the tensor cores as the sum of three
// bf16 values, 24 bits); a hidden value enters the second product as the sum of two (2^-16), so y is rounded to bf16 once.
#include "decode.cuh"
#include "launch.cuh"
#include "ops.cuh"
#include "mma_sync.cuh"
#include "parts.cuh"
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
constexpr int kTile = 8192;              // bytes of a copy: 16 rows x 256 columns (8 gate, 8 up rows), 32 x 128 (down)
constexpr int kUpCols = 256, kUpRows = 8, kDownCols = 128, kDownRows = 32;
constexpr int kColumns = 32;             // tokens of an entry: four products of eight
constexpr int kEntries = kExperts + kRoutes / kColumns;
constexpr int kSumPitch = kDownRows + 4;  // floats; keeps four rows of a token on 16 bytes
// Stages of a warp's ring in the first kernel, and in the second, whose sums need room too.
constexpr int kUpStages = 3;
__host__ __device__ constexpr int down_stages(int T) { return T <= 16 ? 3 : 2; }

// The routes sorted by expert, and the entries that the weights are streamed for: an expert with at most kColumns of its tokens (one
// with more has several and is read as often).
struct Routing {
  int expert[kRoutes];         // of a route, as chosen
  int order[kRoutes];          // routes by expert, ascending
  int token[kRoutes];          // of the routes in order
  int first[kExperts];         // place of an expert's first route
  int entry_expert[kEntries], entry_begin[kEntries], entry_tokens[kEntries];
  int entries;
  float weight[kRoutes];       // of a route
};
constexpr int kChunks = kRoutes / 32;

struct Params {
  const __nv_bfloat16* x;
  long long ldx;
  const void* router;
  int router_bf16;
  const __nv_bfloat16* gate_up;
  const __nv_bfloat16* down;
  int prefetch_up, prefetch_down;        // bring weights to L2 ahead of their use
  __nv_bfloat16* y;
  __nv_bfloat16* hidden;       // [2][T * K][I]: high and low part
  int* routing;                // published: number of entries, the entries, order and token of every route, weights (1 + kEntries + 2 T K words)
  unsigned* arrived;           // [row tiles] parts of a row tile that are there; zeroed by the first kernel
  float* part;                 // [2 * CTAs][T][32]
  int* status;
  int T, E, K, H, I, normalize;
  int tile_ctas;               // CTAs of a row tile in the second kernel; 0 where all CTAs share the list of units
  int up_warps, down_warps;    // warps of a CTA that stream: no more than can have work, so that small problems leave shared memory free
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

// Asks for `bytes` at p to come to L2; p and bytes are multiples of 16.
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  if (bytes > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
// The share of part i of n of a matrix of `bytes`.
__device__ __forceinline__ void prefetch_share(const void* p, long long bytes, int i, int n) {
  const long long share = (bytes / n / 16 + 1) * 16, begin = share * i;
  if (begin < bytes) prefetch_l2(static_cast<const uint8_t*>(p) + begin, uint32_t(min(share, bytes - begin)));
}

// The ring of one warp.  Lane 0 starts copies; a stage is free once every lane has taken its fragments.
struct Ring {
  uint8_t* base;
  uint64_t* bars;
  int* status;
  int stages, lane;
  int put = 0, get = 0;        // stage of the next copy, of the next tile
  uint32_t parity = 0;
  // A copy did not come in time: the rest is neither asked for, since a barrier counts bytes to 2^20 only, nor waited for, and DecodeSession
  // looks at the status.
  bool lost = false;

  __device__ __forceinline__ void init() {
    if (lane == 0) {
      for (int s = 0; s < stages; ++s) mbar_init(&bars[s], 1);
      mbar_fence_init();
    }
    __syncwarp();
  }
  __device__ __forceinline__ void copy(const CUtensorMap* map, int x, int y, int z) {
    if (lane == 0 && !lost) {
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

// Order, tokens and entries from expert[].  A route's place is the number of routes before it that go to its expert: those of its chunk
// of 32 by a vote, those of the chunks before by a running sum, so that it does not depend on timing.
__device__ __forceinline__ void sort_routes(Routing& r, int (*counts)[kExperts], int routes, int K) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (routes <= 32) {                    // one warp, by comparison
    if (warp == 0) {
      const int e = lane < routes ? r.expert[lane] : kExperts;
      const unsigned same = __match_any_sync(0xffffffffu, e), below = (1u << lane) - 1;
      const unsigned leaders = __ballot_sync(0xffffffffu, lane < routes && (same & below) == 0u);
      int to = __popc(same & below), entry = 0;
#pragma unroll 1
      for (int j = 0; j < routes; ++j) {
        const int other = __shfl_sync(0xffffffffu, e, j);
        to += other < e;
        entry += other < e && ((leaders >> j) & 1u);
      }
      if (lane < routes) { r.order[to] = lane; r.token[to] = lane / K; }
      if ((leaders >> lane) & 1u) { r.entry_expert[entry] = e; r.entry_begin[entry] = to; r.entry_tokens[entry] = __popc(same); }
      if (lane == 0) r.entries = __popc(leaders);
    }
    __syncthreads();
    return;
  }
  for (int i = threadIdx.x; i < kChunks * kExperts; i += kThreads) counts[i / kExperts][i % kExperts] = 0;
  __syncthreads();
  constexpr int MINE = kChunks / kWarps;
  int expert[MINE], rank[MINE];
#pragma unroll
  for (int q = 0; q < MINE; ++q) {
    const int chunk = warp + q * kWarps, i = chunk * 32 + lane;
    expert[q] = -1;
    rank[q] = 0;
    if (chunk * 32 >= routes) continue;
    if (i < routes) expert[q] = r.expert[i];
    const unsigned same = __match_any_sync(0xffffffffu, expert[q]);
    rank[q] = __popc(same & ((1u << lane) - 1));
    if (expert[q] >= 0 && rank[q] == 0) counts[chunk][expert[q]] = __popc(same);
  }
  __syncthreads();
  if (warp == 0) {
    int n[2], before = 0, entries_before = 0;              // experts 2 lane, 2 lane + 1
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      n[j] = 0;
      for (int chunk = 0; chunk * 32 < routes; ++chunk) {
        const int here = counts[chunk][2 * lane + j];
        counts[chunk][2 * lane + j] = n[j];
        n[j] += here;
      }
    }
    int sum = n[0] + n[1], parts = (n[0] + kColumns - 1) / kColumns + (n[1] + kColumns - 1) / kColumns;
    before = sum;
    entries_before = parts;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, off), v = __shfl_up_sync(0xffffffffu, entries_before, off);
      if (lane >= off) { before += u; entries_before += v; }
    }
    if (lane == 31) r.entries = entries_before;
    before -= sum;
    entries_before -= parts;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      r.first[2 * lane + j] = before;
      for (int i = 0; i < n[j]; i += kColumns, ++entries_before) {
        r.entry_expert[entries_before] = 2 * lane + j;
        r.entry_begin[entries_before] = before + i;
        r.entry_tokens[entries_before] = min(n[j] - i, kColumns);
      }
      before += n[j];
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < MINE; ++q) {
    if (expert[q] < 0) continue;
    const int chunk = warp + q * kWarps, i = chunk * 32 + lane, to = r.first[expert[q]] + counts[chunk][expert[q]] + rank[q];
    r.order[to] = i;
    r.token[to] = i / K;
  }
  __syncthreads();
}

// One warp a token: K rounds of arg-max over the logits (two experts a lane), the first of which is the softmax's maximum.
// A logit is the sum of `parts` values, the first at [e * se + t * st].  The tokens of this CTA are rank, rank + ranks, ...
__device__ __forceinline__ void choose_experts(const Params& p, const float* logits, int parts, int pitch, int se, int st, Routing& r, int rank,
                                               int ranks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
  for (int t = rank + ranks * warp; t < p.T; t += ranks * kWarps) {
    float v0 = 0.f, v1 = 0.f;
#pragma unroll 8
    for (int w = 0; w < parts; ++w) {
      const float* at = logits + w * pitch + t * st;
      if (lane < p.E) v0 += at[lane * se];
      if (lane + 32 < p.E) v1 += at[(lane + 32) * se];
    }
    if (lane >= p.E) v0 = -CUDART_INF_F;
    if (lane + 32 >= p.E) v1 = -CUDART_INF_F;
    auto key_of = [](float v) {                            // unsigned order = float order; 0 is "taken", which a negative NaN still beats
      const unsigned u = __float_as_uint(v);
      return max((u & 0x80000000u) ? ~u : (u | 0x80000000u), 1u);
    };
    unsigned k0 = lane < p.E ? key_of(v0) : 0u, k1 = lane + 32 < p.E ? key_of(v1) : 0u;
    float chosen = 0.f, top = 0.f, sum = 1.f;              // lane k: the weight of choice k
    int which = 0;
#pragma unroll 1
    for (int k = 0; k < p.K; ++k) {
      const unsigned best = __reduce_max_sync(0xffffffffu, max(k0, k1));
      const unsigned low = __ballot_sync(0xffffffffu, k0 == best), high = __ballot_sync(0xffffffffu, k1 == best);
      const int e = low != 0u ? __ffs(low) - 1 : 31 + __ffs(high);
      const float l = __shfl_sync(0xffffffffu, e < 32 ? v0 : v1, e & 31);
      if (k == 0) {
        top = l;
        sum = (lane < p.E ? expf(v0 - top) : 0.f) + (lane + 32 < p.E ? expf(v1 - top) : 0.f);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      }
      if (lane == e) k0 = 0u;
      if (lane + 32 == e) k1 = 0u;
      if (lane == k) { chosen = expf(l - top) / sum; which = e; }
    }
    if (p.normalize) {
      float total = lane < p.K ? chosen : 0.f;
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
      chosen = chosen / fmaxf(total, 1.1920929e-07f);
    }
    if (lane < p.K) { r.expert[t * p.K + lane] = which; r.weight[t * p.K + lane] = chosen; }
  }
}

// Three bf16 values whose sum is v to 24 bits.
__device__ __forceinline__ void split3(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
  h = pack_bf162(a, b);
  const float a1 = a - __uint_as_float(h << 16), b1 = b - __uint_as_float(h & 0xFFFF0000u);
  m = pack_bf162(a1, b1);
  l = pack_bf162(a1 - __uint_as_float(m << 16), b1 - __uint_as_float(m & 0xFFFF0000u));
}

// Partial logits part[warp][e][t] of this CTA's share of the contraction: steps of 16 experts (rows) by 32 columns, eight tokens a
// product.  One loop over (expert tile, columns) whose loads run a step ahead: the code is run once or twice a launch, so
// what it costs is its latency and its own size in the instruction cache.
__device__ __forceinline__ void router_products(const Params& p, float* part, int worker, int workers) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int E16 = (p.E + 15) & ~15, T8 = (p.T + 7) & ~7;
  float* mine = part + (threadIdx.x >> 5) * (E16 * T8);
  float acc[8][4];
  float4 w[2][2];
  uint4 b[8];
  auto load = [&](int m, int q) {
    const int k = q * 32 + c * 8;
    const bool in = m < E16 && k < p.H;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const long long at = (long long)min(m + g + 8 * u, p.E - 1) * p.H + k;
      w[u][0] = w[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in && p.router_bf16) {
        w[u][0] = *reinterpret_cast<const float4*>(static_cast<const __nv_bfloat16*>(p.router) + at);      // eight bf16 values
      } else if (in) {
        w[u][0] = *reinterpret_cast<const float4*>(static_cast<const float*>(p.router) + at);
        w[u][1] = reinterpret_cast<const float4*>(static_cast<const float*>(p.router) + at)[1];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j * 8 >= p.T) break;
      b[j] = in ? *reinterpret_cast<const uint4*>(p.x + min(j * 8 + g, p.T - 1) * p.ldx + k) : make_uint4(0, 0, 0, 0);
    }
  };
  int m = 0, q = worker;
  load(m, q);
#pragma unroll 1
  while (m < E16) {
    if (q == worker) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    }
    uint32_t part3[3][2][4];           // high, middle, low
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float v[8] = {w[u][0].x, w[u][0].y, w[u][0].z, w[u][0].w, w[u][1].x, w[u][1].y, w[u][1].z, w[u][1].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (p.router_bf16) {
          part3[0][u][i] = __float_as_uint(v[i]);
          part3[1][u][i] = part3[2][u][i] = 0u;
        } else {
          split3(v[2 * i], v[2 * i + 1], part3[0][u][i], part3[1][u][i], part3[2][u][i]);
        }
      }
    }
    uint4 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = b[j];
    const int m_now = m;
    q += workers;
    const bool last = q * 32 >= p.H;
    if (last) { q = worker; m += 16; }
    load(m, q);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j * 8 >= p.T) break;
#pragma unroll
      for (int i = 2; i >= 0; --i) {   // the small parts first
        mma_bf16(acc[j], part3[i][0][0], part3[i][1][0], part3[i][0][1], part3[i][1][1], x[j].x, x[j].y);
        mma_bf16(acc[j], part3[i][0][2], part3[i][1][2], part3[i][0][3], part3[i][1][3], x[j].z, x[j].w);
      }
      if (last) {
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[(m_now + g + 8 * (i >> 1)) * T8 + j * 8 + 2 * c + (i & 1)] = acc[j][i];
      }
    }
  }
}

// The logits [t][e] of up to four tokens: a warp an expert, the loads of 1024 columns in flight, every sum in the same order.
constexpr int kFewTokens = 4;
__device__ __forceinline__ void router_few(const Params& p, float* logits) {
  const int lane = threadIdx.x & 31;
  constexpr int AHEAD = 4;
#pragma unroll 1
  for (int e = threadIdx.x >> 5; e < p.E; e += kWarps) {
    float acc[kFewTokens] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int d0 = lane * 8; d0 < p.H; d0 += 256 * AHEAD) {
      float4 w[AHEAD][2];
      uint4 x[AHEAD][kFewTokens];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int d = d0 + 256 * i;
        w[i][0] = w[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (d < p.H) {
          const long long at = (long long)e * p.H + d;
          if (p.router_bf16) {
            w[i][0] = *reinterpret_cast<const float4*>(static_cast<const __nv_bfloat16*>(p.router) + at);          // eight bf16 values
          } else {
            w[i][0] = *reinterpret_cast<const float4*>(static_cast<const float*>(p.router) + at);
            w[i][1] = reinterpret_cast<const float4*>(static_cast<const float*>(p.router) + at)[1];
          }
        }
#pragma unroll
        for (int t = 0; t < kFewTokens; ++t) {
          x[i][t] = make_uint4(0, 0, 0, 0);
          if (d < p.H && t < p.T) x[i][t] = *reinterpret_cast<const uint4*>(p.x + t * p.ldx + d);
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        float v[8] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w, w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
        if (p.router_bf16) {
#pragma unroll
          for (int j = 3; j >= 0; --j) {
            const uint32_t pair = __float_as_uint(v[j]);
            v[2 * j + 1] = __uint_as_float(pair & 0xFFFF0000u);
            v[2 * j] = __uint_as_float(pair << 16);
          }
        }
#pragma unroll
        for (int t = 0; t < kFewTokens; ++t) {
          if (t >= p.T) break;
          const uint32_t q[4] = {x[i][t].x, x[i][t].y, x[i][t].z, x[i][t].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[t] = fmaf(__uint_as_float(q[j] << 16), v[2 * j], acc[t]);
            acc[t] = fmaf(__uint_as_float(q[j] & 0xFFFF0000u), v[2 * j + 1], acc[t]);
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kFewTokens; ++t) {
      if (t >= p.T) break;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], off);
      if (lane == 0) logits[t * p.E + e] = acc[t];
    }
  }
}

// What the CTA's warps have of the logits, added.
__device__ __forceinline__ void add_logits(const Params& p, const float* part, float* logits) {
  const int E16 = (p.E + 15) & ~15, T8 = (p.T + 7) & ~7;
#pragma unroll 1
  for (int i = threadIdx.x; i < p.T * p.E; i += kThreads) {
    const int t = i / p.E, e = i % p.E;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += part[w * (E16 * T8) + e * T8 + t];
    logits[i] = v;
  }
}

__device__ __forceinline__ void publish(const Params& p, const Routing& r) {
  const int routes = p.T * p.K;
  if (threadIdx.x == 0) p.routing[0] = r.entries;
  if (threadIdx.x < kEntries) p.routing[1 + threadIdx.x] = r.entry_expert[threadIdx.x] | (r.entry_tokens[threadIdx.x] << 8) | (r.entry_begin[threadIdx.x] << 16);
#pragma unroll 1
  for (int i = threadIdx.x; i < routes; i += kThreads) {
    p.routing[1 + kEntries + i] = r.order[i] | (r.token[i] << 16);
    p.routing[1 + kEntries + routes + i] = __float_as_int(r.weight[i]);
  }
#pragma unroll 1
  for (int i = threadIdx.x; i < (p.H + kDownRows - 1) / kDownRows; i += kThreads) p.arrived[i] = 0u;
}

template <bool WEIGHTS>
__device__ __forceinline__ void read_routing(const Params& p, Routing& r) {
  const int routes = p.T * p.K, words = 1 + kEntries + (WEIGHTS ? 2 : 1) * routes;
  constexpr int MOST = (1 + kEntries + (WEIGHTS ? 2 : 1) * kRoutes + kThreads - 1) / kThreads;
  int v[MOST];                           // all loads before the first use
#pragma unroll
  for (int i = 0; i < MOST; ++i) v[i] = threadIdx.x + i * kThreads < words ? __ldcg(p.routing + threadIdx.x + i * kThreads) : 0;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int at = threadIdx.x + i * kThreads, route = at - 1 - kEntries;
    if (at >= words) break;
    if (at == 0) {
      r.entries = v[i];
    } else if (at <= kEntries) {
      r.entry_expert[at - 1] = v[i] & 0xFF;
      r.entry_tokens[at - 1] = (v[i] >> 8) & 0xFF;
      r.entry_begin[at - 1] = (v[i] >> 16) & 0xFFFF;
    } else if (route < routes) {
      r.order[route] = v[i] & 0xFFFF;
      r.token[route] = v[i] >> 16;
    } else {
      r.weight[route - routes] = __int_as_float(v[i]);
    }
  }
  __syncthreads();
}

// ---- kernel 0, where the router is large: one cluster; its CTAs share the contraction, then the tokens ----
constexpr int kRouteCluster = 8;
__global__ void __launch_bounds__(kThreads)
moe_route_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Routing r;
  __shared__ int counts[kChunks][kExperts];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = int(cluster.block_rank()), warp = threadIdx.x >> 5;
  float* logits = reinterpret_cast<float*>(smem);          // [T][E] of this CTA's columns
  float* full = logits + p.T * p.E;
  float* part = full + p.T * p.E;
  let_next_start();
  wait_for_previous();
  router_products(p, part, rank * kWarps + warp, kRouteCluster * kWarps);
  __syncthreads();
  add_logits(p, part, logits);
  cluster.sync();
  for (int i = threadIdx.x; i < p.T * p.E; i += kThreads) {
    if (i / p.E % kRouteCluster != rank) continue;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kRouteCluster; ++k) v += cluster.map_shared_rank(logits, k)[i];
    full[i] = v;
  }
  __syncthreads();
  choose_experts(p, full, 1, 0, 1, p.E, r, rank, kRouteCluster);
  __syncthreads();
  if (rank != 0) {
    for (int i = threadIdx.x; i < p.T * p.K; i += kThreads)
      if (i / p.K % kRouteCluster == rank) {
        cluster.map_shared_rank(r.expert, 0)[i] = r.expert[i];
        cluster.map_shared_rank(r.weight, 0)[i] = r.weight[i];
      }
  }
  cluster.sync();
  if (rank != 0) return;
  sort_routes(r, counts, p.T * p.K, p.K);
  publish(p, r);
}

// ---- kernel 1: gate and up projection, SwiGLU; ROUTED: kernel 0 has routed ----
template <bool ROUTED>
__global__ void __launch_bounds__(kThreads)
moe_up_kernel(const __grid_constant__ CUtensorMap weights, const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Routing r;
  __shared__ uint64_t bars[kWarps][kUpStages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int routes = p.T * p.K;
  let_next_start();
  Ring ring;
  ring.stages = kUpStages;
  ring.base = smem + warp * kUpStages * kTile;
  ring.bars = bars[warp];
  ring.status = p.status;
  ring.lane = lane;
  ring.init();
  if (threadIdx.x == 0) tma_prefetch_desc(&weights);
  // While the routing kernel runs: bring what nearly all experts will be asked for to L2.
  if (ROUTED && p.prefetch_up && threadIdx.x < p.E)
    prefetch_share(p.gate_up + (long long)threadIdx.x * 2 * p.I * p.H, 4LL * p.I * p.H, blockIdx.x, gridDim.x);
  wait_for_previous();
  if constexpr (ROUTED) {
    read_routing<true>(p, r);
  } else {
    __shared__ int counts[kChunks][kExperts];
    float* part = reinterpret_cast<float*>(smem);          // partial logits, before the rings are used
    const int E16 = (p.E + 15) & ~15, T8 = (p.T + 7) & ~7;
    if (p.T <= kFewTokens) {
      router_few(p, part);
      __syncthreads();
      choose_experts(p, part, 1, 0, 1, p.E, r, 0, 1);
    } else {
      router_products(p, part, warp, kWarps);
      __syncthreads();
      choose_experts(p, part, kWarps, E16 * T8, T8, 1, r, 0, 1);
    }
    __syncthreads();
    sort_routes(r, counts, routes, p.K);
    fence_proxy_async_smem();            // the rings' memory held the logits
    __syncwarp();
  }

  const int tiles = (p.I + kUpRows - 1) / kUpRows, steps = (p.H + kUpCols - 1) / kUpCols;
  const int N = r.entries * tiles;
  // Items in turn over all warps of the machine, the CTAs first: every SM reads from all over the weights.  With one stretch of them
  // for each CTA the slowest SM took a quarter longer than the mean (58 experts of 2,048 x 1,024: 146 against 134 us for the layer;
  // 8 of 4,096 x 14,336: 420 against 383).
  const int stride = int(gridDim.x) * p.up_warps, i0 = warp < p.up_warps ? warp * int(gridDim.x) + int(blockIdx.x) : N;
  const int count = i0 < N ? (N - 1 - i0) / stride + 1 : 0, by_expert = stride / tiles, by_tile = stride % tiles;
  auto advance = [&](int& expert, int& tile) {
    expert += by_expert;
    tile += by_tile;
    if (tile >= tiles) { tile -= tiles; ++expert; }
  };
  int left = count * steps, ahead_step = 0, ahead_expert = i0 / tiles, ahead_tile = i0 % tiles;
  int expert = ahead_expert, tile_at = ahead_tile;
  auto next_copy = [&]() {
    if (left == 0) return;
    --left;
    ring.copy(&weights, ahead_step * kUpCols, ahead_tile * kUpRows, 2 * r.entry_expert[ahead_expert]);
    if (++ahead_step == steps) {
      ahead_step = 0;
      advance(ahead_expert, ahead_tile);
    }
  };
#pragma unroll 1
  for (int s = 0; s < ring.stages; ++s) next_copy();
  if constexpr (!ROUTED) {
    if (blockIdx.x == 0) publish(p, r);
  }
  if (p.prefetch_down && threadIdx.x < r.entries)          // what the second kernel will read
    prefetch_share(p.down + (long long)r.entry_expert[threadIdx.x] * p.H * p.I, 2LL * p.H * p.I, blockIdx.x, gridDim.x);

  // The columns of up to 16 tokens of a unit are loaded before its tile is waited for, those of more in place.
  struct Columns {
    uint4 v[kUpCols / 32];
  };
  auto load = [&](Columns& b, const __nv_bfloat16* row, int step) {
    const __nv_bfloat16* src = row + step * kUpCols;
    if ((step + 1) * kUpCols <= p.H) {
#pragma unroll
      for (int s = 0; s < kUpCols / 32; ++s) b.v[s] = *reinterpret_cast<const uint4*>(src + 32 * s);
    } else {
#pragma unroll
      for (int s = 0; s < kUpCols / 32; ++s) {
        b.v[s] = make_uint4(0, 0, 0, 0);
        if (step * kUpCols + 32 * s + c * 8 < p.H) b.v[s] = *reinterpret_cast<const uint4*>(src + 32 * s);
      }
    }
  };
#pragma unroll 1
  for (int items = count; items > 0; --items) {
    const int row = tile_at * kUpRows + g, n0 = r.entry_begin[expert], n = r.entry_tokens[expert];
    advance(expert, tile_at);
    const __nv_bfloat16* rows[kColumns / 8];
#pragma unroll
    for (int j = 0; j < kColumns / 8; ++j) rows[j] = p.x + (long long)r.token[n0 + min(j * 8 + g, n - 1)] * p.ldx + c * 8;
    float acc[kColumns / 8][4], acc_odd[4];                // the first product in two chains
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc_odd[i] = 0.f;
#pragma unroll
      for (int j = 0; j < kColumns / 8; ++j) acc[j][i] = 0.f;
    }
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      Columns b0, b1;
      load(b0, rows[0], step);
      if (n > 8) load(b1, rows[1], step);
      const uint8_t* tile = ring.wait() + g * (kUpCols * 2) + c * 16;
      uint4 a[kUpCols / 32][2];
#pragma unroll
      for (int s = 0; s < kUpCols / 32; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) a[s][u] = *reinterpret_cast<const uint4*>(tile + u * (kUpRows * kUpCols * 2) + s * 64);
      ring.taken();
      next_copy();
#pragma unroll
      for (int s = 0; s < kUpCols / 32; ++s) {
        mma_bf16(acc[0], a[s][0].x, a[s][1].x, a[s][0].y, a[s][1].y, b0.v[s].x, b0.v[s].y);
        mma_bf16(acc_odd, a[s][0].z, a[s][1].z, a[s][0].w, a[s][1].w, b0.v[s].z, b0.v[s].w);
      }
      auto multiply = [&](int j, const Columns& b) {
#pragma unroll
        for (int s = 0; s < kUpCols / 32; ++s) {
          mma_bf16(acc[j], a[s][0].x, a[s][1].x, a[s][0].y, a[s][1].y, b.v[s].x, b.v[s].y);
          mma_bf16(acc[j], a[s][0].z, a[s][1].z, a[s][0].w, a[s][1].w, b.v[s].z, b.v[s].w);
        }
      };
      if (n > 8) {                       // each set of columns is loaded while the one before is multiplied
        if (n > 16) load(b0, rows[2], step);
        multiply(1, b1);
        if (n > 16) {
          if (n > 24) load(b1, rows[3], step);
          multiply(2, b0);
          if (n > 24) multiply(3, b1);
        }
      }
    }
    // ---- the hidden values of the item ----
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[0][i] += acc_odd[i];
#pragma unroll
    for (int j = 0; j < kColumns / 8; ++j) {
      if (j * 8 >= n) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = j * 8 + 2 * c + i;
        if (col >= n || row >= p.I) continue;
        const int route = r.order[n0 + col];
        const float gate = acc[j][i], up = acc[j][i + 2];
        const float h = gate / (1.f + expf(-gate)) * up * r.weight[route];
        const __nv_bfloat16 high = __float2bfloat16_rn(h);
        __nv_bfloat16* dst = p.hidden + (long long)route * p.I + row;
        dst[0] = high;
        dst[(long long)routes * p.I] = __float2bfloat16_rn(h - __bfloat162float(high));
      }
    }
  }
  ring.finish();
}

// ---- kernel 2: down projection, summed over the experts of each token ----
__global__ void __launch_bounds__(kThreads)
moe_down_kernel(const __grid_constant__ CUtensorMap weights, const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Routing r;
  __shared__ uint64_t bars[kWarps][3];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int routes = p.T * p.K, sum_size = p.T * kSumPitch;
  float* sums = reinterpret_cast<float*>(smem + p.down_warps * down_stages(p.T) * kTile); // [warps][T][pitch]
#pragma unroll 4
  for (int i = threadIdx.x * 4; i < p.down_warps * sum_size; i += kThreads * 4) *reinterpret_cast<float4*>(sums + i) = make_float4(0.f, 0.f, 0.f, 0.f);
  if (threadIdx.x == 0) tma_prefetch_desc(&weights);
  Ring ring;
  ring.stages = down_stages(p.T);
  ring.base = smem + warp * ring.stages * kTile;
  ring.bars = bars[warp];
  ring.status = p.status;
  ring.lane = lane;
  ring.init();
  let_next_start();
  wait_for_previous();
  read_routing<false>(p, r);
  const int live = r.entries;

  const int steps = (p.I + kDownCols - 1) / kDownCols, tiles = (p.H + kDownRows - 1) / kDownRows;
  const int per_tile = live * steps, N = tiles * per_tile;
  // Small problems: a row tile is the work of as many CTAs as there are for each, so that every CTA has one piece to hand over.
  const int group = min(p.tile_ctas, per_tile), ctas = group > 0 ? group : min(int(gridDim.x), N);
  const Parts parts(group > 0 ? per_tile : N, ctas);
  int c0, c1, first_tile;
  if (group > 0) {
    first_tile = int(blockIdx.x / unsigned(p.tile_ctas));
    const int at = int(blockIdx.x) - first_tile * p.tile_ctas;
    if (first_tile >= tiles || at >= group) return;
    c0 = first_tile * per_tile + parts.begin(at);
    c1 = first_tile * per_tile + parts.begin(at + 1);
  } else {
    if (int(blockIdx.x) >= ctas) return;
    c0 = parts.begin(blockIdx.x);
    c1 = parts.begin(blockIdx.x + 1);
    first_tile = int(unsigned(c0) / unsigned(per_tile));
  }
  // The units of this warp: its share of what the CTA has of each row tile, one after the other.
  struct Stream {
    int tile, u, end, expert, step;
  };
  auto enter = [&](Stream& s) {          // the first row tile from s.tile on that has units for this warp
    for (; s.tile * per_tile < c1; ++s.tile) {
      const int s0 = max(c0, s.tile * per_tile), s1 = min(c1, (s.tile + 1) * per_tile);
      const Parts shares(s1 - s0, p.down_warps);
      s.u = s0 + shares.begin(min(warp, p.down_warps));
      s.end = s0 + shares.begin(min(warp + 1, p.down_warps));
      if (s.u == s.end) continue;
      s.expert = int(unsigned(s.u - s.tile * per_tile) / unsigned(steps));
      s.step = s.u - s.tile * per_tile - s.expert * steps;
      return;
    }
    s.u = s.end = 0;
  };
  Stream ahead{first_tile, 0, 0, 0, 0};
  enter(ahead);
  Stream now = ahead;                    // where the products are
  auto next_copy = [&]() {
    if (ahead.u == ahead.end) return;
    ring.copy(&weights, ahead.step * kDownCols, ahead.tile * kDownRows, r.entry_expert[ahead.expert]);
    if (++ahead.step == steps) { ahead.step = 0; ++ahead.expert; }
    if (++ahead.u == ahead.end) { ++ahead.tile; enter(ahead); }
  };
#pragma unroll 1
  for (int s = 0; s < ring.stages; ++s) next_copy();

  // Hidden values of a unit, as the columns in the first kernel: [32 columns][high, low]
  struct Columns {
    uint4 v[kDownCols / 32][2];
  };
  const long long low = (long long)routes * p.I;           // from a high part to its low part
  auto load = [&](Columns& b, const __nv_bfloat16* row, int step) {
    const __nv_bfloat16 *src = row + step * kDownCols, *src_low = src + low;
    if ((step + 1) * kDownCols <= p.I) {
#pragma unroll
      for (int s = 0; s < kDownCols / 32; ++s) {
        b.v[s][0] = *reinterpret_cast<const uint4*>(src + 32 * s);
        b.v[s][1] = *reinterpret_cast<const uint4*>(src_low + 32 * s);
      }
    } else {
#pragma unroll
      for (int s = 0; s < kDownCols / 32; ++s) {
        b.v[s][0] = b.v[s][1] = make_uint4(0, 0, 0, 0);
        if (step * kDownCols + 32 * s + c * 8 < p.I) {
          b.v[s][0] = *reinterpret_cast<const uint4*>(src + 32 * s);
          b.v[s][1] = *reinterpret_cast<const uint4*>(src_low + 32 * s);
        }
      }
    }
  };
  float* mine = sums + warp * sum_size;
#pragma unroll 1
  for (int tile = first_tile; tile * per_tile < c1; ++tile) {
    const int s0 = max(c0, tile * per_tile), s1 = min(c1, (tile + 1) * per_tile);
    int units = now.tile == tile ? now.end - now.u : 0, at_entry = now.expert, step = now.step;
    if (now.tile == tile) {
      ++now.tile;
      enter(now);
    }
#pragma unroll 1
    for (; units > 0; ++at_entry) {      // one entry of this row tile
      const int n0 = r.entry_begin[at_entry], n = r.entry_tokens[at_entry];
      const __nv_bfloat16* rows[kColumns / 8];
#pragma unroll
      for (int j = 0; j < kColumns / 8; ++j) rows[j] = p.hidden + (long long)r.order[n0 + min(j * 8 + g, n - 1)] * p.I + c * 8;
      float acc[2][kColumns / 8][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < kColumns / 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
#pragma unroll 1
      for (; units > 0 && step < steps; ++step, --units) {
        Columns b0, b1;
        load(b0, rows[0], step);
        if (n > 8) load(b1, rows[1], step);
        const uint8_t* at = ring.wait() + g * (kDownCols * 2) + c * 16;
        uint4 a[2][kDownCols / 32][2];   // [row tile of 16][32 columns][rows g, g + 8]
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int s = 0; s < kDownCols / 32; ++s)
#pragma unroll
            for (int v = 0; v < 2; ++v) a[m][s][v] = *reinterpret_cast<const uint4*>(at + (16 * m + 8 * v) * (kDownCols * 2) + s * 64);
        ring.taken();
        next_copy();
        auto multiply = [&](int j, const Columns& x) {
#pragma unroll
          for (int s = 0; s < kDownCols / 32; ++s)
#pragma unroll
            for (int v = 1; v >= 0; --v)
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                mma_bf16(acc[m][j], a[m][s][0].x, a[m][s][1].x, a[m][s][0].y, a[m][s][1].y, x.v[s][v].x, x.v[s][v].y);
                mma_bf16(acc[m][j], a[m][s][0].z, a[m][s][1].z, a[m][s][0].w, a[m][s][1].w, x.v[s][v].z, x.v[s][v].w);
              }
        };
        multiply(0, b0);
        if (n > 8) {
          if (n > 16) load(b0, rows[2], step);
          multiply(1, b1);
          if (n > 16) {
            if (n > 24) load(b1, rows[3], step);
            multiply(2, b0);
            if (n > 24) multiply(3, b1);
          }
        }
      }
      step = 0;
      // an entry has a token at most once, so the lanes of a warp write different sums
#pragma unroll
      for (int j = 0; j < kColumns / 8; ++j) {
        if (j * 8 >= n) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = j * 8 + 2 * c + i;
          if (col >= n) continue;
          float* dst = mine + r.token[n0 + col] * kSumPitch + g;
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
    // four rows of a token a thread
    auto store = [&](int i, const float (&v)[4]) {
      const int t = i / kDownRows, row = tile * kDownRows + i % kDownRows;
      if (row < p.H) *reinterpret_cast<uint2*>(p.y + (long long)t * p.H + row) = make_uint2(pack_bf162(v[0], v[1]), pack_bf162(v[2], v[3]));
    };
#pragma unroll 1
    for (int i = threadIdx.x * 4; i < p.T * kDownRows; i += kThreads * 4) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      float* at = sums + i / kDownRows * kSumPitch + i % kDownRows;
#pragma unroll
      for (int w = 0; w < kWarps; ++w, at += sum_size) {
        if (w >= p.down_warps) break;
        const float4 q = *reinterpret_cast<const float4*>(at);
        *reinterpret_cast<float4*>(at) = make_float4(0.f, 0.f, 0.f, 0.f);
        v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
      }
      if (whole) store(i, v);
      else *reinterpret_cast<float4*>(own + i) = make_float4(v[0], v[1], v[2], v[3]);
    }
    if (!whole) {
      const int f = group > 0 ? tile * p.tile_ctas : parts.owner(tile * per_tile);
      const int l = group > 0 ? f + group - 1 : parts.owner((tile + 1) * per_tile - 1);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        last = atomicAdd(&p.arrived[tile], 1u) == unsigned(l - f);
        __threadfence();
      }
      __syncthreads();
      if (last) {
        // the row tile begins in CTA f, whose second part it is; the others begin with it
        const float* from = p.part + (2 * (long long)f + 1) * p.T * kDownRows;
        const float* rest = p.part + 2 * (long long)(f + 1) * p.T * kDownRows;
#pragma unroll 1
        for (int i = threadIdx.x * 4; i < p.T * kDownRows; i += kThreads * 4) {
          const float4 q = __ldcg(reinterpret_cast<const float4*>(from + i));
          float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll 1
          for (int k0 = 0; k0 < l - f; k0 += 8) {
            float4 o[8];                 // eight parts in flight
#pragma unroll
            for (int k = 0; k < 8; ++k)
              o[k] = k0 + k < l - f ? __ldcg(reinterpret_cast<const float4*>(rest + 2 * (long long)(k0 + k) * p.T * kDownRows + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k) { v[0] += o[k].x; v[1] += o[k].y; v[2] += o[k].z; v[3] += o[k].w; }
          }
          store(i, v);
        }
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

// Bytes of x and the router's weight up to which every CTA of the first kernel routes by itself.  Measured in place against in a kernel of
// its own: 8 experts of 768, one token (26 KB) 12.2 against 14.2 us for the layer, 8 (36 KB) 16.6 and 16.9, 12 (42 KB) 18.4 and 17.6, 16
// (48 KB) 19.2 and 18.3, 24 (60 KB) 21.5 and 19.2; one token of 16 experts of 1,024 (66 KB) 13.5 and 14.4, of 32 (130 KB) 15.2 and 14.9.
constexpr long long kRouteInPlace = 48 * 1024;
constexpr long long kPrefetchBytes = 48ll << 20;
// Units of a CTA up to which the second kernel gives a row tile to CTAs of its own.  Measured with and without, the layer: 8 experts of 768 x
// 1,024, one token (2.6 units) 12.0 and 14.9 us, 64 tokens (16 units) 30.4 and 33.4; of 768 x 2,048 (31) 41.9 and 43.8; of 2,048 x 2,048 (62)
// 48.8 and 51.2; of 2,048 x 8,192 (221) 140.0 and 141.2: what it saves is a few microseconds at any size, a small part above the border.
constexpr long long kSmallUnits = 32;

size_t part_bytes(int T, int E) { return size_t(kWarps) * ((E + 15) / 16 * 16) * ((T + 7) / 8 * 8) * 4; }
size_t route_shared(int T, int E) { return part_bytes(T, E) + size_t(2) * T * E * 4; }
size_t up_shared(int T, int E, int warps, bool routed) {
  const size_t ring = size_t(warps) * kUpStages * kTile, part = routed ? 0 : part_bytes(T, E);
  return ring > part ? ring : part;
}
size_t down_shared(int T, int warps) { return size_t(warps) * (down_stages(T) * kTile + T * kSumPitch * 4); }

// The kernels' shared memory, allowed once a device.
cudaError_t prepare(int dev) {
  static std::once_flag once[64];
  static cudaError_t result[64];
  std::call_once(once[dev], [dev] {
    auto allow = [](auto kernel, size_t bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)); };
    const size_t few = down_shared(16, kWarps), many = down_shared(kMoeTokensMax, kWarps), down = few > many ? few : many;
    cudaError_t e = allow(moe_route_kernel, route_shared(kMoeTokensMax, kExperts));
    if (e == cudaSuccess) e = allow(moe_up_kernel<false>, up_shared(kMoeTokensMax, kExperts, kWarps, false));
    if (e == cudaSuccess) e = allow(moe_up_kernel<true>, up_shared(kMoeTokensMax, kExperts, kWarps, true));
    if (e == cudaSuccess) e = allow(moe_down_kernel, down);
    result[dev] = e;
  });
  return result[dev];
}

struct Workspace {                       // byte offsets of its parts
  size_t hidden, part, arrived, total;
};
Workspace workspace_of(int T, int K, int H, int I) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Workspace w;
  w.hidden = up(size_t(1 + kEntries + 2 * T * K) * 4);
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
  if ((err = prepare(dev)) != cudaSuccess) return err;
  const int sms = device_sm_count();
  // upper bounds of the items and units, hence of the warps that can have some
  const long long entries = ((long long)a.T * a.K < a.E ? a.T * a.K : a.E) + a.T * a.K / kColumns;
  const long long items = entries * ((a.I + kUpRows - 1) / kUpRows);
  const long long units = entries * ((a.H + kDownRows - 1) / kDownRows) * ((a.I + kDownCols - 1) / kDownCols);
  auto warps_for = [sms](long long n) { return n >= (long long)sms * kWarps ? kWarps : int((n + sms - 1) / sms); };
  const Workspace w = workspace_of(a.T, a.K, a.H, a.I);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  Params p;
  p.x = static_cast<const __nv_bfloat16*>(a.x); p.ldx = a.ldx;
  p.router = a.router; p.router_bf16 = a.router_bf16;
  p.gate_up = static_cast<const __nv_bfloat16*>(a.gate_up);
  p.down = static_cast<const __nv_bfloat16*>(a.down);
  // Half of L2 at most, and gate and up only where the routing can be guessed: four routes an expert and more.
  const long long matrix = 2LL * a.H * a.I;
  p.prefetch_up = 2 * matrix * a.E <= kPrefetchBytes && (long long)a.T * a.K >= 4LL * a.E;
  p.prefetch_down = matrix * entries <= kPrefetchBytes;
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.routing = reinterpret_cast<int*>(ws);
  p.hidden = reinterpret_cast<__nv_bfloat16*>(ws + w.hidden);
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.arrived = reinterpret_cast<unsigned*>(ws + w.arrived);
  p.status = a.status;
  p.T = a.T; p.E = a.E; p.K = a.K; p.H = a.H; p.I = a.I; p.normalize = a.normalize;
  const int row_tiles = (a.H + kDownRows - 1) / kDownRows;
  p.tile_ctas = row_tiles <= sms / 2 && units <= kSmallUnits * sms ? sms / row_tiles : 0;
  p.up_warps = warps_for(items);
  p.down_warps = p.tile_ctas > 0 ? warps_for((units + row_tiles * p.tile_ctas - 1) / (row_tiles * p.tile_ctas) * sms) : warps_for(units);
  CUtensorMap up, down;
  if (!encode_weights(&up, a.gate_up, a.H, a.I, 2LL * a.E, kUpCols, kUpRows, 2) ||
      !encode_weights(&down, a.down, a.I, a.H, a.E, kDownCols, kDownRows, 1))
    return cudaErrorInvalidValue;

  const bool routed = (long long)a.E * a.H * (a.router_bf16 ? 2 : 4) + (long long)a.T * a.H * 2 > kRouteInPlace;
  if (routed) {
    ++g_launch_count;
    err = launch_chained(moe_route_kernel, dim3(kRouteCluster), kThreads, route_shared(a.T, a.E), kRouteCluster, a.stream, p);
    if (err != cudaSuccess) return err;
  }
  ++g_launch_count;
  err = launch_chained(routed ? moe_up_kernel<true> : moe_up_kernel<false>, dim3(unsigned(sms)), kThreads, up_shared(a.T, a.E, p.up_warps, routed), 0,
                       a.stream, up, p);
  if (err != cudaSuccess) return err;
  ++g_launch_count;
  return launch_chained(moe_down_kernel, dim3(unsigned(sms)), kThreads, down_shared(a.T, p.down_warps), 0, a.stream, down, p);
}

}  // namespace mts
