// Attention of a few new tokens over the 8-bit key / value cache (layout: decode.cuh).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(D) - max),  j <= position of the query
//
// One pass over the cache with a running maximum and sum.  Keys and values are read once per tile of query rows (the heads that
// share a K/V head, times the new tokens of the step).  Every warp has a ring of blocks of its own in shared memory, which bulk
// copies fill (one for the keys of a block with its scales, one for its values; two each at D = 128), so the warps run without barriers
// and each keeps 8 to 16 KB of the cache in flight.  A lane's 16 adjacent bytes are its K or V fragment of several steps (the V rows are
// stored in that order); 4 bytes become two fp16 pairs in four instructions; both products run on m16n8k16 with the tokens (K) or
// the head's dims (V) as rows and eight query rows as columns.  The (sequence, head, row tile, block) units of
// the whole batch are one list, cut into equal parts for the warps that fit on the machine: sequences of unlike lengths, and a
// single long one, keep every SM busy, and a warp streams across the ends of sequences.  A second kernel joins the parts of
// the (sequence, head, row tile) items that were cut.
// What bounds it: reading the codes, 2 D bytes per token and K/V head.  Measured on the GPU (replayed graph, caches flushed), one new
// token: 64 ragged sequences of up to 2,048 tokens, 12 heads of 64, 24.7 us (95 MB, 3.8 TB/s); one of 131,071 tokens, 16 heads
// on 4 of 64, 21.1 us (67 MB, 3.2 TB/s); eight ragged ones of up to 32,768 (146,699 tokens in all), 32 heads on 8 of 128, 56.4 us (301 MB,
// 5.3 TB/s).  The first two are short streams behind a launch and the counting of units, and before the join.
//
// Rounding: codes are exact in fp16.  A query row is scaled by the power of two that brings its largest value to [1, 2): bf16 queries
// keep their eight bits in fp16 down to 2^-17 of that value, and lose up to 2^-25 of it below.  Probabilities are rounded to fp16
// (2^-11 of each, at a scale of 2^14 so that the smallest kept one is 2^-38 of the largest); the sum of probabilities, the maximum and
// the output accumulators are fp32.  In the unfinished block, whose values are bf16, a probability is the sum of two bf16 values.
#include "decode.cuh"
#include "launch.cuh"
#include "ops.cuh"
#include "mma_sync.cuh"
#include "parts.cuh"
#include "ptx_sm100.cuh"

#include <cooperative_groups.h>
#include <math_constants.h>

namespace mts {

namespace {

namespace cg = cooperative_groups;

constexpr int BLK = kCacheBlock;
constexpr int kWarps = 4;
// Resident CTAs an SM: what fits in registers (four with eight query rows) and, at D = 128, in shared memory as long as the counts of
// units leave room (resident_ctas).
__host__ __device__ constexpr int ctas_per_sm(int D, int nq) { return nq > 1 ? 2 : D == 128 ? 3 : 4; }
constexpr int kBatchMax = 2048;          // sequences: their units are counted in shared memory
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kProbShift = 14.f;       // probabilities are held times 2^14
constexpr uint32_t kOnes = 0x3C003C00u;  // a pair of fp16 ones

struct Params {
  const uint8_t* records;
  const void* tail;
  const int* start;
  const int* count;
  int B, Hkv, blocks, Hq, T, group, row_tiles;
  const void* q;
  long long sb, sh, st;
  void* o;
  float* part;                           // [2 * warps][rows of a tile][D + 2]: parts of items that were cut
  int ctas;
  float sm_log2;                         // log2(e) / sqrt(D)
  int* status;
};

// Tokens of sequence b: before the step, and of it.
__device__ __forceinline__ int2 span_of(const Params& p, int b) {
  const int capacity = p.blocks * BLK;
  const int start = min(max(p.start[b], 0), capacity);
  return make_int2(start, min(min(max(p.count[b], 0), p.T), capacity - start));
}
// Units of a (head, row tile) of it: the finished blocks, and the unfinished one in halves of 32 tokens, which are as many bytes.
__device__ __forceinline__ int units_of(int2 span) {
  const int total = span.x + span.y, rest = total % BLK;
  return span.y > 0 ? total / BLK + (rest > 0) + (rest > BLK / 2) : 0;
}

// prefix[b] = units of the sequences before b; every thread of the CTA takes part.
template <int THREADS>
__device__ __forceinline__ void count_units(const Params& p, int* prefix, int* scratch) {
  const int heads = p.Hkv * p.row_tiles, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) prefix[0] = 0;
  int carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    int v = b < p.B ? units_of(span_of(p, b)) * heads : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, off);
      if (lane >= off) v += u;
    }
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += scratch[w];
      carry += scratch[w];
    }
    if (b < p.B) prefix[b + 1] = before + v;
    __syncthreads();
  }
}

// A stage of a warp's ring: the head of a record (its scales), keys, values, and the query rows of an item that begins.  Keys and values
// come in pieces of 4 KB (2 KB at D = 32), each with a barrier of its own, so that a piece is asked for again as soon as it is read:
// at D = 128, where they are two pieces each, three are on their way while one is worked on (54.3 against 62.0 us with one piece
// each for eight ragged sequences of up to 32,768, 32 heads on 8).  Pieces of 2 KB at D = 64 cost more instructions than they hide.
__host__ __device__ constexpr int pieces(int D) { return D < 128 ? 1 : 2; }
__host__ __device__ constexpr int ring_stages(int D) { return D < 64 ? 2 : 1; }
__host__ __device__ constexpr int stage_bytes(int D, int NQ) { return record_bytes(D) + 8 * NQ * D * 2; }
__host__ __device__ constexpr int ring_bytes(int D, int NQ) { return kWarps * ring_stages(D) * stage_bytes(D, NQ); }
__host__ __device__ constexpr int exchange_bytes(int D, int NQ) { return kWarps * D * (8 * NQ + 1) * 4; }
__host__ __device__ constexpr int result_bytes(int D, int NQ) { return 8 * NQ * (D + 2) * 4; }
// The rings, and where they were: the exchange of the warps' outputs with the CTA's result behind it.  With the result behind the rings two CTAs
// of 128 dims fit an SM instead of three: 24 sequences of 500 tokens, 32 heads on 8, took 22.2 us and now 14.1; 50 of 500, 8 heads, 24.6 and
// 16.9; but 8 of 500, 32 heads, 13.7 and 15.8.
__host__ __device__ constexpr int shared_bytes(int D, int NQ) {
  const int joined = exchange_bytes(D, NQ) + result_bytes(D, NQ);
  return ring_bytes(D, NQ) > joined ? ring_bytes(D, NQ) : joined;
}
// Resident CTAs an SM with the counts of units of `counted` sequences behind that: an SM has 228 KB, 1 KB of it is taken for a CTA,
// and statistics and barriers are below 512 bytes for every eight rows.  (700 sequences of 1,000 tokens, 2 heads on 1 of 128: 60.7 us planned for
// two CTAs an SM, 72.5 for three, of which two fit; 1,000 of 1,000, 8 heads on 4: 269 and 253.)
__host__ inline int resident_ctas(int D, int nq, int counted) {
  const int room = (228 << 10) / (shared_bytes(D, nq) + (counted > 0 ? (counted + 1) * 4 : 0) + 512 * nq + 1024);
  return room < ctas_per_sm(D, nq) ? room : ctas_per_sm(D, nq);
}

// `bytes` (a multiple of 16, like both addresses) from global to shared memory; completion is counted on the barrier.
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// WORDS words (4 or 8 of them 16 bytes at a time) at p in shared memory.
template <int WORDS>
__device__ __forceinline__ void read_words(const uint8_t* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + i * 16);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}

template <typename T> struct Act;
template <> struct Act<__nv_bfloat16> {
  static constexpr bool kHalf = false;
  static constexpr uint32_t kOnes = 0x3F803F80u;
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t from_half2(uint32_t w) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pack_bf162(v.x, v.y);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};
template <> struct Act<__half> {
  static constexpr bool kHalf = true;
  static constexpr uint32_t kOnes = 0x3C003C00u;
  static __device__ __forceinline__ float lo(uint32_t w) { return __low2float(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __high2float(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ uint32_t from_half2(uint32_t w) { return w; }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};

// The values of a pair that are infinite or NaN, as a mask: the exponent is all ones, and one more carries into the sign's place.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t kExponent = Act<T>::kHalf ? 0x7C007C00u : 0x7F807F80u, kOne = Act<T>::kHalf ? 0x04000400u : 0x00800080u;
  return (((w & kExponent) + kOne) >> 15 & 0x00010001u) * 0xFFFFu;
}

// Running statistics and output of 8 * NQ query rows in one warp.  A lane holds the columns 2c and 2c + 1 of every tile of
// eight rows (the statistics are the same in the eight lanes that share c) and the dims g and g + 8 of every 16.
template <int D, int NQ>
struct State {
  float m[NQ][2], l[NQ][2], o[NQ][D / 16][4];              // l: the sum of the probabilities, complete in every lane
};

__device__ __forceinline__ float exp2_fast(float x) {     // 2^x to 2 ulp; 0 below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Scores of 16 M tokens, of which `f` times is the logit in the log2 domain (-inf where masked), to probabilities times 2^14;
// rescales the state.  s[m][n][i]: token 16 m + g + 8 (i >> 1), query 2c + (i & 1) of tile n.
template <int D, int NQ, int M>
__device__ __forceinline__ void update_max(State<D, NQ>& st, float (&s)[M][NQ][4], const float (&f)[NQ][2]) {
  bool moved = false;
  float alpha[NQ][2];
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float mx = fmaxf(s[0][n][j], s[0][n][j + 2]);
#pragma unroll
      for (int m = 1; m < M; ++m) mx = fmaxf(mx, fmaxf(s[m][n][j], s[m][n][j + 2]));
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      mx = fmaxf(mx * f[n][j], st.m[n][j]);
      const float base = mx == -CUDART_INF_F ? 0.f : mx;     // a row that has seen nothing yet
      alpha[n][j] = exp2_fast(st.m[n][j] - base);
      moved |= mx != st.m[n][j];
      st.m[n][j] = mx;
      const float shift = kProbShift - base;
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) s[m][n][j + 2 * i] = exp2_fast(fmaf(s[m][n][j + 2 * i], f[n][j], shift));
    }
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) st.l[n][j] *= alpha[n][j];
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[n][d][i] *= alpha[n][i & 1];
    }
  }
}

// True when the copies of a stage have come, false when they have not within the limit.
__device__ __forceinline__ bool wait_copy(uint64_t* bar, uint32_t parity) {
  if (mbar_test(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (!mbar_test(bar, parity))
    if (global_timer_ns() - t0 > kWaitDeadlineNs) return false;
  return true;
}

// Where a warp is in the list of units: number `at` of the `units` of row tile `tile` of head h of sequence b, whose first
// `closed` are finished blocks.
struct Cursor {
  int b, h, tile, at, units, closed;
  __device__ __forceinline__ void enter(const Params& p, int seq) {
    b = seq;
    const int2 s = span_of(p, b);
    units = units_of(s);
    closed = (s.x + s.y) / BLK;
  }
  __device__ __forceinline__ void seek(const Params& p, const int* prefix, int u) {
    int lo = 0, hi = p.B - 1;            // the last sequence whose units begin at or before u (one with none ends where it begins)
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (prefix[mid] <= u) lo = mid; else hi = mid - 1;
    }
    enter(p, lo);
    const int rest = u - prefix[lo];
    at = rest % units;
    tile = rest / units % p.row_tiles;
    h = rest / units / p.row_tiles;
  }
  __device__ __forceinline__ void next(const Params& p) {
    if (++at < units) return;
    at = 0;
    if (++tile < p.row_tiles) return;
    tile = 0;
    if (++h < p.Hkv) return;
    h = 0;
    units = 0;
    for (int seq = b + 1; seq < p.B && units == 0; ++seq) enter(p, seq);
  }
};

// CLUSTER: the CTAs of a cluster share one item, else the CTAs of the grid share the list of units.
template <typename T, int D, int NQ, bool CLUSTER>
__global__ void __launch_bounds__(kWarps * 32, ctas_per_sm(D, NQ))
cached_attention_kernel(const Params p) {
  constexpr int KW = D / 16;             // K words per lane and token = steps of 16 dims
  constexpr int DT = D / 16;             // tiles of 16 dims of the output
  constexpr int ROWS = 8 * NQ;
  constexpr int OP = ROWS + 1;           // pitch of the output exchange
  constexpr int STAGES = ring_stages(D);
  constexpr int STAGE = stage_bytes(D, NQ), KEYS = kCacheHead, VALUES = KEYS + BLK * D, QUERIES = VALUES + BLK * D;
  constexpr int KB = D / 4;              // bytes of a key that a lane owns
  extern __shared__ __align__(16) uint8_t smem[];          // rings (afterwards the exchange of the outputs and the result), prefix
  __shared__ float ml_sm[kWarps][ROWS][2];
  __shared__ int scratch[kWarps];
  constexpr int SPLIT = pieces(D), PIECE = BLK * D / SPLIT;
  __shared__ uint64_t bars[kWarps][STAGES][2 * SPLIT];     // the pieces of a stage: keys, then values
  int* prefix = reinterpret_cast<int*>(smem + shared_bytes(D, NQ));
  float* o_sm = reinterpret_cast<float*>(smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  if (CLUSTER) let_next_start();
  wait_for_previous();
  if (!CLUSTER) let_next_start();        // the joining kernel reads the lengths before it waits: whatever wrote them has ended by now
  Cursor cur;
  int c0, c1;                            // units of this CTA
  if constexpr (CLUSTER) {
    const int shares = int(cg::this_cluster().num_blocks()), item = blockIdx.x / shares, share = blockIdx.x % shares;
    cur.tile = item % p.row_tiles;
    cur.h = item / p.row_tiles % p.Hkv;
    cur.enter(p, item / p.row_tiles / p.Hkv);
    const Parts parts(cur.units, shares);
    c0 = parts.begin(share);
    c1 = parts.begin(share + 1);
    cur.at = c0;
  } else {
    count_units<kWarps * 32>(p, prefix, scratch);
    const Parts parts(prefix[p.B], p.ctas);
    c0 = parts.begin(blockIdx.x);
    c1 = parts.begin(blockIdx.x + 1);
    if (c0 == c1) return;
    cur.seek(p, prefix, c0);
  }
  const int u0 = c0 + part_begin<kWarps>(c1 - c0, warp), u1 = c0 + part_begin<kWarps>(c1 - c0, warp + 1);
  const int rows = p.group * p.T;

  State<D, NQ> st;
  auto reset = [&]() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) { st.m[n][j] = -CUDART_INF_F; st.l[n][j] = 0.f; }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[n][d][i] = 0.f;
    }
  };
  reset();
  // does the CTA stay within one item?  Then its four warps are joined here and count as one part.
  const int item_begin = c0 - cur.at, item_end = item_begin + cur.units;
  const bool one_item = CLUSTER || c1 <= item_end;
  if constexpr (CLUSTER) cur.at = u0;
  else if (u0 < u1 && u0 != c0) cur.seek(p, prefix, u0);

  if (u0 < u1) {
    uint8_t* ring = smem + warp * (STAGES * STAGE);
    // Lane 0 starts the copies of a stage; the lanes below 8 NQ add the query rows where an item begins.  Tokens of the unfinished block
    // that do not exist are copied with the rest and not used.
    if (lane == 0) {
#pragma unroll
      for (int t = 0; t < STAGES; ++t)
#pragma unroll
        for (int i = 0; i < 2 * SPLIT; ++i) mbar_init(&bars[warp][t][i], 1);
      mbar_fence_init();
    }
    __syncwarp();
    Cursor ahead = cur;
    int u_ahead = u0;
    const uint8_t* src;                  // of the unit ahead: its keys; its values are values_at bytes behind them
    bool finished;
    auto locate = [&]() {
      const long long bh = (long long)ahead.b * p.Hkv + ahead.h;
      finished = ahead.at < ahead.closed;
      src = finished ? p.records + (bh * p.blocks + ahead.at) * record_bytes(D) + kCacheHead
                     : static_cast<const uint8_t*>(p.tail) + (bh * 2 + (ahead.closed & 1)) * (4 * BLK * D) + (ahead.at - ahead.closed) * (BLK * D);
    };
    locate();
    // A copy did not come in time: the rest is neither asked for, since a barrier counts bytes to 2^20 only, nor waited for, and DecodeSession
    // looks at the status.
    bool lost = false;
    // piece i of the unit ahead; behind the last one the cursor moves on
    auto copy = [&](int stage, int i) {
      __syncwarp();                      // every lane has read what the copy overwrites
      if (u_ahead < u1) {
        uint8_t* dst = ring + stage * STAGE;
        uint64_t* bar = &bars[warp][stage][i];
        const bool begins = i == 0 && (u_ahead == u0 || ahead.at == 0);
        const int head = i == 0 && finished ? kCacheHead : 0;
        if (lane == 0 && !lost) {
          mbar_expect_tx(bar, PIECE + head + (begins ? ROWS * D * 2 : 0));
          bulk_copy(dst + KEYS + i * PIECE - head, src + (i >= SPLIT && !finished ? BLK * D : 0) + i * PIECE - head, PIECE + head, bar);
        }
        if (begins) {
          __syncwarp();                  // the bytes are expected before any arrive
          if (lane < ROWS && !lost) {
            const int r = ahead.tile * ROWS + lane;
            const int t = r < rows ? r / p.group : 0, head = ahead.h * p.group + (r < rows ? r % p.group : 0);
            bulk_copy(dst + QUERIES + lane * (D * 2), static_cast<const T*>(p.q) + ahead.b * p.sb + head * p.sh + t * p.st, D * 2, bar);
          }
        }
        if (i == 2 * SPLIT - 1) {
          ++u_ahead;
          if (u_ahead < u1) {
            ahead.next(p);
            locate();
          }
        }
      }
    };
    auto arrive = [&](int stage, int which, uint32_t parity) {
      if (!lost && !wait_copy(&bars[warp][stage][which], parity)) {
        lost = true;
        if (lane == 0) atomicMax(p.status, int(STATUS_WAIT_TIMEOUT));
      }
    };
#pragma unroll
    for (int t = 0; t < STAGES; ++t)
#pragma unroll
      for (int i = 0; i < 2 * SPLIT; ++i) copy(t, i);

    uint32_t qf[NQ][KW][2];              // fp16 query fragments, scaled: column g of every tile, dims 4 KW c ... of the head
    float qscale[NQ][2];                 // log2(e) / sqrt(D) times the power of two taken out, for the columns 2c, 2c + 1
    int limit[NQ][2];                    // last position that a column sees
    int start = 0, fresh = 0;
    int stage = 0;
    uint32_t parity = 0;
    for (int u = u0; u < u1; ++u) {
      const uint8_t* here = ring + stage * STAGE;
      arrive(stage, 0, parity);
      if (u == u0 || cur.at == 0) {
        const int2 span = span_of(p, cur.b);
        start = span.x; fresh = span.y;
        const int row0 = cur.tile * ROWS;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = row0 + n * 8 + 2 * c + j;
            limit[n][j] = r < fresh * p.group ? start + r / p.group : -1;
          }
          uint32_t w[2 * KW];
          read_words<2 * KW>(here + QUERIES + (n * 8 + g) * (D * 2) + c * (2 * KB), w);
          float amax = 0.f;
          if (!Act<T>::kHalf) {
#pragma unroll
            for (int i = 0; i < 2 * KW; ++i) amax = fmaxf(amax, fmaxf(fabsf(Act<T>::lo(w[i])), fabsf(Act<T>::hi(w[i]))));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          }
          // exponent of the largest value (fp16 queries stay as they are); kept within what 2^-e and 2^e can express
          int e = Act<T>::kHalf ? 0 : int(__float_as_uint(amax) >> 23) - 127;
          e = min(max(e, -120), 120);
          const float down = __uint_as_float(uint32_t(127 - e) << 23), up = __uint_as_float(uint32_t(127 + e) << 23);
#pragma unroll
          for (int i = 0; i < KW; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              qf[n][i][j] = Act<T>::kHalf ? w[2 * i + j] : pack_half2(Act<T>::lo(w[2 * i + j]) * down, Act<T>::hi(w[2 * i + j]) * down);
#pragma unroll
          for (int j = 0; j < 2; ++j) qscale[n][j] = p.sm_log2 * __shfl_sync(0xffffffffu, up, (2 * c + j) * 4);
        }
      }
      if (cur.at < cur.closed) {
        const int base = cur.at * BLK;
        const uint8_t* kst = here + KEYS + g * D + c * KB;
        const uint8_t* vst = here + VALUES + g * BLK + c * 16;
        const float2 sc = *reinterpret_cast<const float2*>(here);
        float s[4][NQ][4];
#pragma unroll
        for (int m0 = 0; m0 < 4; m0 += 2) {                  // two token tiles at a time: two chains of products
          if (SPLIT == 2 && m0 == 2) arrive(stage, 1, parity);
          uint32_t kr[2][2][KW];
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int v = 0; v < 2; ++v) read_words<KW>(kst + (16 * (m0 + m) + 8 * v) * D, kr[m][v]);
#pragma unroll
          for (int i = 0; i < KW; ++i)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              uint32_t a0, a1, a2, a3;
              codes_to_half(kr[m][0][i], a0, a2);
              codes_to_half(kr[m][1][i], a1, a3);
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                if (i == 0) mma_f16_first(s[m0 + m][n], a0, a1, a2, a3, qf[n][0][0], qf[n][0][1]);
                else mma_f16(s[m0 + m][n], a0, a1, a2, a3, qf[n][i][0], qf[n][i][1]);
              }
            }
          if (SPLIT == 2 || m0 == 2) copy(stage, m0 / 2 * (SPLIT - 1));
        }
        float f[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) f[n][j] = qscale[n][j] * sc.x;
        const bool masked = base + BLK > start;              // blocks of the step itself: rows see different lengths
        if (masked) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool seen = base + 16 * m + g + 8 * (i >> 1) <= limit[n][i & 1];
                s[m][n][i] = seen ? s[m][n][i] * f[n][i & 1] : -CUDART_INF_F;
              }
            f[n][0] = f[n][1] = 1.f;                         // a scale of 0 would make a NaN of -inf
          }
        }
        update_max<D, NQ, 4>(st, s, f);
        uint32_t pf[4][NQ][2];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            pf[m][n][0] = transpose8x8(pack_half2(s[m][n][0], s[m][n][1]));
            pf[m][n][1] = transpose8x8(pack_half2(s[m][n][2], s[m][n][3]));
          }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {                       // the sum of the rounded probabilities
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int m = 0; m < 4; ++m) mma_f16(sum, kOnes, kOnes, kOnes, kOnes, pf[m][n][0], pf[m][n][1]);
          st.l[n][0] += sum[0];
          st.l[n][1] += sum[1];
        }
        arrive(stage, SPLIT, parity);
#pragma unroll
        for (int d0 = 0; d0 < DT; d0 += 2) {
          if (SPLIT == 2 && d0 == DT / 2) arrive(stage, 3, parity);
          uint32_t vr[2][2][4];
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int v = 0; v < 2; ++v) read_words<4>(vst + (16 * (d0 + d) + 8 * v) * BLK, vr[d][v]);
          float acc[2][NQ][4];
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              uint32_t a0, a1, a2, a3;
              codes_to_half(vr[d][0][m], a0, a2);
              codes_to_half(vr[d][1][m], a1, a3);
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                if (m == 0) mma_f16_first(acc[d][n], a0, a1, a2, a3, pf[0][n][0], pf[0][n][1]);
                else mma_f16(acc[d][n], a0, a1, a2, a3, pf[m][n][0], pf[m][n][1]);
              }
            }
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i)  // a block that a row does not see at all must not reach it through its scale
                if (!masked || base <= limit[n][i & 1]) st.o[n][d0 + d][i] = fmaf(acc[d][n][i], sc.y, st.o[n][d0 + d][i]);
          if (SPLIT == 2 && d0 + 2 == DT / 2) copy(stage, 2);
        }
        copy(stage, 2 * SPLIT - 1);
      } else {                             // ---- half of the unfinished block, in the activation type ----
        const int base = cur.closed * BLK + (cur.at - cur.closed) * 32;
        const int valid = start + fresh - base;              // tokens that exist
        if (SPLIT == 2) arrive(stage, 1, parity);
        float s[2][NQ][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          uint32_t a[2][2 * KW];
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            read_words<2 * KW>(here + KEYS + (16 * m + 8 * v + g) * (D * 2) + c * (2 * KB), a[v]);
            const uint32_t keep = 16 * m + 8 * v + g < valid ? 0xFFFFFFFFu : 0u;
#pragma unroll
            for (int i = 0; i < 2 * KW; ++i) a[v][i] &= keep;
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[m][n][i] = 0.f;
#pragma unroll
            for (int i = 0; i < KW; ++i) {
              const uint32_t f[4] = {a[0][2 * i], a[1][2 * i], a[0][2 * i + 1], a[1][2 * i + 1]};
              Act<T>::mma(s[m][n], f, Act<T>::from_half2(qf[n][i][0]), Act<T>::from_half2(qf[n][i][1]));   // eight bits at most: exact
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool seen = base + 16 * m + g + 8 * (i >> 1) <= limit[n][i & 1];
              s[m][n][i] = seen ? s[m][n][i] * qscale[n][i & 1] : -CUDART_INF_F;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < SPLIT; ++i) copy(stage, i);
        float one[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) one[n][0] = one[n][1] = 1.f;
        update_max<D, NQ, 2>(st, s, one);
#pragma unroll
        for (int i = SPLIT; i < 2 * SPLIT; ++i) arrive(stage, i, parity);
        uint32_t ph[2][NQ][2], pl[2][NQ][2], keep[2][2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              const float x = s[m][n][2 * v], y = s[m][n][2 * v + 1];
              if (Act<T>::kHalf) {
                ph[m][n][v] = transpose8x8(pack_half2(x, y));
              } else {
                const uint32_t hi2 = pack_bf162(x, y);
                ph[m][n][v] = transpose8x8(hi2);
                pl[m][n][v] = transpose8x8(pack_bf162(x - Act<T>::lo(hi2), y - Act<T>::hi(hi2)));
              }
            }
          const int left = valid - 16 * m - 2 * c;           // tokens 16 m + 2c + {0, 1, 8, 9} of this lane that exist
          keep[m][0] = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u;
          keep[m][1] = left >= 10 ? 0xFFFFFFFFu : left == 9 ? 0xFFFFu : 0u;
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            constexpr uint32_t ones = Act<T>::kOnes;
            const uint32_t f[4] = {ones, ones, ones, ones};
            Act<T>::mma(sum, f, ph[m][n][0], ph[m][n][1]);
            if (!Act<T>::kHalf) Act<T>::mma(sum, f, pl[m][n][0], pl[m][n][1]);
          }
          st.l[n][0] += sum[0];
          st.l[n][1] += sum[1];
        }
        // A token that some rows do not see has the probability 0 there, which times an infinity or a NaN is a NaN.  Where the half may
        // hold such a token, values that are not finite are added to the rows that see them, and are zero in the product.
        if (fresh > 1 && base + 32 > start + 1) {
          uint8_t* mine = ring + stage * STAGE + VALUES + g * 64 + c * 16;
          uint32_t found = 0;
#pragma unroll 1
          for (int d = 0; d < D; d += 8) {
            uint32_t w[4];
            read_words<4>(mine + d * 64, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) found |= not_finite<T>(w[i] & keep[i >> 1][i & 1]);
          }
          if (__any_sync(0xffffffffu, found != 0)) {
#pragma unroll 1
            for (int token = 0; token < min(valid, 32); ++token) {
              const uint8_t* row = here + VALUES + g * 64 + tail_slot(0, 0, token) * 2;
#pragma unroll
              for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                  const uint32_t bits = *reinterpret_cast<const uint16_t*>(row + (16 * d + 8 * v) * 64);
                  const float value = Act<T>::lo(bits & not_finite<T>(bits));
#pragma unroll
                  for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                      if (base + token <= limit[n][j]) st.o[n][d][j + 2 * v] += value;
                }
            }
            __syncwarp();
#pragma unroll 1
            for (int d = 0; d < D; d += 8) {
              uint32_t w[4];
              read_words<4>(mine + d * 64, w);
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] &= ~not_finite<T>(w[i]);
              *reinterpret_cast<uint4*>(mine + d * 64) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_proxy_async_smem();      // before the next copy into this stage
            __syncwarp();
          }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          uint32_t w[2][4];
#pragma unroll
          for (int v = 0; v < 2; ++v) read_words<4>(here + VALUES + (16 * d + 8 * v + g) * 64 + c * 16, w[v]);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const uint32_t f[4] = {w[0][2 * m] & keep[m][0], w[1][2 * m] & keep[m][0], w[0][2 * m + 1] & keep[m][1], w[1][2 * m + 1] & keep[m][1]};
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              Act<T>::mma(st.o[n][d], f, ph[m][n][0], ph[m][n][1]);
              if (!Act<T>::kHalf) Act<T>::mma(st.o[n][d], f, pl[m][n][0], pl[m][n][1]);
            }
          }
        }
#pragma unroll
        for (int i = SPLIT; i < 2 * SPLIT; ++i) copy(stage, i);
      }
      if (++stage == STAGES) { stage = 0; parity ^= 1; }

      const bool ends = cur.at + 1 == cur.units;
      if (!one_item && (ends || u + 1 == u1)) {
        // ---- the warp is done with this item: its output if the item was not cut, else its part ----
        const bool whole = ends && u - cur.at >= u0;
        const int row0 = cur.tile * ROWS;
        float* dst = p.part + (2 * ((long long)blockIdx.x * kWarps + warp) + (u - cur.at >= u0 ? 1 : 0)) * (ROWS * (D + 2));
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float l = st.l[n][j];
            const int r = n * 8 + 2 * c + j, row = row0 + r;
            if (row >= fresh * p.group) continue;
            const int t = row / p.group, head = cur.h * p.group + row % p.group;
            T* out = static_cast<T*>(p.o) + (((long long)cur.b * p.T + t) * p.Hq + head) * D;
            float* part = dst + r * (D + 2);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int dim = 16 * d + g + 8 * i;
                if (whole) out[dim] = Act<T>::from(st.o[n][d][j + 2 * i] / l);
                else part[dim] = st.o[n][d][j + 2 * i];
              }
            if (!whole && g == 0) { part[D] = st.m[n][j]; part[D + 1] = l; }
          }
        reset();
      }
      if (u + 1 < u1) cur.next(p);
    }
    if (lost) {                          // copies may still be on their way: give them time before the memory changes hands
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 200000000ull) __nanosleep(1000);
    }
  }
  if (!one_item) return;

  // ---- join the warps ----
  __syncthreads();                       // the rings are read; their memory takes the outputs
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (g == 0) {
        ml_sm[warp][n * 8 + 2 * c + j][0] = st.m[n][j];
        ml_sm[warp][n * 8 + 2 * c + j][1] = st.l[n][j];
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o_sm[warp * (D * OP) + (16 * d + g + 8 * (i >> 1)) * OP + n * 8 + 2 * c + (i & 1)] = st.o[n][d][i];
  }
  __syncthreads();
  const int live = span_of(p, cur.b).y * p.group, row0 = cur.tile * ROWS;
  const bool whole = c0 == item_begin && c1 == item_end;
  float* result = reinterpret_cast<float*>(smem + exchange_bytes(D, NQ));                // [ROWS][D + 2] of this CTA
  for (int i = threadIdx.x; i < ROWS * D; i += kWarps * 32) {
    const int r = i / D, d = i % D, row = row0 + r;
    if (row >= live) break;
    float m = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml_sm[w][r][0]);
    const float base = m == -CUDART_INF_F ? 0.f : m;
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float a = exp2f(ml_sm[w][r][0] - base);
      l = fmaf(ml_sm[w][r][1], a, l);
      o = fmaf(o_sm[w * (D * OP) + d * OP + r], a, o);
    }
    if (CLUSTER) {
      float* dst = result + r * (D + 2);
      dst[d] = o;
      if (d == 0) { dst[D] = m; dst[D + 1] = l; }
    } else if (whole) {
      const int t = row / p.group, head = cur.h * p.group + row % p.group;
      static_cast<T*>(p.o)[(((long long)cur.b * p.T + t) * p.Hq + head) * D + d] = Act<T>::from(o / l);
    } else {
      float* dst = p.part + (2 * (long long)blockIdx.x * kWarps * ROWS + r) * (D + 2);
      dst[d] = o;
      if (d == 0) { dst[D] = m; dst[D + 1] = l; }
    }
  }
  if constexpr (CLUSTER) {
    cg::cluster_group cluster = cg::this_cluster();
    const int shares = int(cluster.num_blocks());
    cluster.sync();
    for (int i = int(cluster.block_rank()) * (kWarps * 32) + threadIdx.x; i < ROWS * D; i += shares * kWarps * 32) {
      const int r = i / D, d = i % D, row = row0 + r;
      if (row >= rows) break;
      const int t = row / p.group, head = cur.h * p.group + row % p.group;
      float l = 0.f, o = 0.f;
      if (row < live) {
        float m = -CUDART_INF_F;
        for (int k = 0; k < shares; ++k) m = fmaxf(m, cluster.map_shared_rank(result, k)[r * (D + 2) + D]);
        const float base = m == -CUDART_INF_F ? 0.f : m;
        for (int k = 0; k < shares; ++k) {
          const float* part = cluster.map_shared_rank(result, k) + r * (D + 2);
          const float a = exp2f(part[D] - base);
          l = fmaf(part[D + 1], a, l);
          o = fmaf(part[d], a, o);
        }
      }
      static_cast<T*>(p.o)[(((long long)cur.b * p.T + t) * p.Hq + head) * D + d] = Act<T>::from(row < live ? o / l : 0.f);
    }
    cluster.sync();                      // nobody leaves while its result may still be read
  }
}

// (This kernel does not let the next one start early: CTAs of another attention that fill the SMs would hold the room of those
// that have yet to join, 24.8 against 31.7 us for 64 ragged sequences.)
// The parts of an item [begin, end): its candidates are the warps of the first and of the last CTA, and one part of every CTA
// between (those lie within the item).
struct ItemParts {
  const Parts parts;
  int begin, end, i0, i1, between, candidates;
  __device__ __forceinline__ ItemParts(const Parts& all, int first, int units) : parts(all), begin(first), end(first + units) {
    i0 = parts.owner(begin);
    i1 = parts.owner(end - 1);
    between = max(i1 - i0 - 1, 0);
    candidates = kWarps + (i1 > i0 ? between + kWarps : 0);
  }
  // where candidate k is, -1 where it has nothing of the item; `whole`: it has all of it, and its owner has written the output
  __device__ __forceinline__ int at(int k, bool& whole) const {
    const int i = k < kWarps ? i0 : k < kWarps + between ? i0 + 1 + k - kWarps : i1;
    const int w = k < kWarps ? k : k < kWarps + between ? 0 : k - kWarps - between;
    const int c0 = parts.begin(i), c1 = parts.begin(i + 1);
    if (c0 >= begin && c1 <= end) {                        // within the item: its warps are one part
      whole |= c0 == begin && c1 == end;
      return w == 0 && c0 < c1 ? 2 * i * kWarps : -1;
    }
    const int x0 = c0 + part_begin<kWarps>(c1 - c0, w), x1 = c0 + part_begin<kWarps>(c1 - c0, w + 1);
    if (x0 >= end || x1 <= begin || x0 >= x1) return -1;
    whole |= x0 <= begin && x1 >= end;
    return 2 * (i * kWarps + w) + (x0 <= begin ? 1 : 0);
  }
};

// Joins the parts of one row, a CTA a row, and zeroes the rows of padding; rows of items that were not cut are there already.
// The weight of every part first, then the eight warps add the outputs of every eighth part, and the eight sums in order.
constexpr int kJoinThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
join_parts_kernel(const Params p, int rows_per_tile) {
  extern __shared__ __align__(16) uint8_t smem[];
  int* prefix = reinterpret_cast<int*>(smem);              // [B + 1]
  int* slot = prefix + p.B + 1;                            // [parts]
  float* weight = reinterpret_cast<float*>(slot + p.ctas + 2 * kWarps);
  __shared__ float red[kJoinThreads / 32], o_sm[kJoinThreads / 32][D];
  __shared__ int scratch[kJoinThreads / 32];
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.group * p.T;
  const int row = int(blockIdx.x % unsigned(rows));
  const int bh = int(blockIdx.x / unsigned(rows));
  const int h = bh % p.Hkv, b = bh / p.Hkv;
  const int t = row / p.group, head = h * p.group + row % p.group;
  T* out = static_cast<T*>(p.o) + (((long long)b * p.T + t) * p.Hq + head) * D;
  const int2 span = span_of(p, b);
  if (t >= span.y) {
    wait_for_previous();
    for (int d = threadIdx.x; d < D; d += kJoinThreads) out[d] = Act<T>::from(0.f);
    return;
  }
  count_units<kJoinThreads>(p, prefix, scratch);
  const Parts parts(prefix[p.B], p.ctas);
  const ItemParts item(parts, prefix[b] + (h * p.row_tiles + row / rows_per_tile) * units_of(span), units_of(span));
  const int candidates = item.candidates;
  wait_for_previous();                   // everything above read the lengths only, which were there when the kernel before this one began
  bool whole = false;
  float m = -CUDART_INF_F;
  const float* src = p.part + (long long)(row % rows_per_tile) * (D + 2);
  const long long pitch = (long long)rows_per_tile * (D + 2);
  for (int k = threadIdx.x; k < candidates; k += kJoinThreads) {
    const int at = item.at(k, whole);
    slot[k] = at;
    if (at >= 0) m = fmaxf(m, src[at * pitch + D]);
  }
  if (__syncthreads_or(whole)) return;                     // its owner has written the output
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) m = fmaxf(m, red[w]);
  const float base = m == -CUDART_INF_F ? 0.f : m;
  __syncthreads();
  float l = 0.f;
  for (int k = threadIdx.x; k < candidates; k += kJoinThreads) {
    float a = 0.f;
    if (slot[k] >= 0) {
      a = exp2f(src[slot[k] * pitch + D] - base);
      l = fmaf(src[slot[k] * pitch + D + 1], a, l);
    }
    weight[k] = a;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  if (lane == 0) red[warp] = l;
  __syncthreads();
  float o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = 0.f;
#pragma unroll 8
  for (int k = warp; k < candidates; k += kJoinThreads / 32) {
    const int at = slot[k];
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = fmaf(at >= 0 ? src[at * pitch + j * 32 + lane] : 0.f, weight[k], o[j]);
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) o_sm[warp][j * 32 + lane] = o[j];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kJoinThreads) {
    float sum = 0.f, total = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) { sum += o_sm[w][d]; total += red[w]; }
    out[d] = Act<T>::from(sum / total);
  }
}

// The same, a warp a row: the candidates are gone through 32 at a time with a running maximum and sum.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
join_rows_kernel(const Params p, int rows_per_tile, int total_rows) {
  extern __shared__ __align__(16) uint8_t smem[];
  int* prefix = reinterpret_cast<int*>(smem);              // [B + 1]
  __shared__ int scratch[kJoinThreads / 32];
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31, rows = p.group * p.T;
  count_units<kJoinThreads>(p, prefix, scratch);
  const int at_row = int(blockIdx.x) * (kJoinThreads / 32) + (threadIdx.x >> 5);
  wait_for_previous();                   // everything above read the lengths only, which were there when the kernel before this one began
  if (at_row >= total_rows) return;
  const int row = at_row % rows, bh = at_row / rows, h = bh % p.Hkv, b = bh / p.Hkv;
  const int t = row / p.group, head = h * p.group + row % p.group;
  T* out = static_cast<T*>(p.o) + (((long long)b * p.T + t) * p.Hq + head) * D;
  const int2 span = span_of(p, b);
  if (t >= span.y) {
#pragma unroll
    for (int j = 0; j < PER; ++j) out[j * 32 + lane] = Act<T>::from(0.f);
    return;
  }
  const ItemParts item(Parts(prefix[p.B], p.ctas), prefix[b] + (h * p.row_tiles + row / rows_per_tile) * units_of(span), units_of(span));
  const float* src = p.part + (long long)(row % rows_per_tile) * (D + 2);
  const long long pitch = (long long)rows_per_tile * (D + 2);
  float m = -CUDART_INF_F, l = 0.f, o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = 0.f;
  for (int k0 = 0; k0 < item.candidates; k0 += 32) {
    bool whole = false;
    const int at = k0 + lane < item.candidates ? item.at(k0 + lane, whole) : -1;
    if (__any_sync(0xffffffffu, whole)) return;
    const float part_m = at >= 0 ? src[at * pitch + D] : -CUDART_INF_F, part_l = at >= 0 ? src[at * pitch + D + 1] : 0.f;
    float most = fmaxf(part_m, m);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    const float base = most == -CUDART_INF_F ? 0.f : most, before = exp2f(m - base);
    const float weight = at >= 0 ? exp2f(part_m - base) : 0.f;
    m = most;
    l *= before;
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] *= before;
    float sum = part_l * weight;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    l += sum;
    unsigned left = __ballot_sync(0xffffffffu, at >= 0);   // the parts, in order, eight loads at a time
    while (left != 0) {
      float v[8][PER], a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int from = left != 0 ? __ffs(int(left)) - 1 : 0;
        a[i] = __shfl_sync(0xffffffffu, weight, from);
        const int slot = __shfl_sync(0xffffffffu, at, from);
#pragma unroll
        for (int j = 0; j < PER; ++j) v[i][j] = left != 0 ? src[slot * pitch + j * 32 + lane] : 0.f;
        if (left == 0) a[i] = 0.f;
        left &= left - 1;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < PER; ++j) o[j] = fmaf(v[i][j], a[i], o[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) out[j * 32 + lane] = Act<T>::from(o[j] / l);
}

struct Plan {
  int nq, row_tiles, ctas, cluster;      // cluster: 0 for the list of units
};

// Where a cluster of up to eight CTAs has at most two blocks a warp and there is room for all CTAs at once, an item is the work of one
// cluster, which joins its parts through distributed shared memory: one launch, no counting of units.  Such problems are bound by
// latency, so the smallest row tile that allows it is taken (17 rows over 2,000 tokens in tiles of 8: 0.4 us of 12.8 less than in one of 24).
// Otherwise rows are taken in tiles of up to 32 (16 at D = 128, where the accumulators of 32 would not fit in registers), so that the
// cache is read as few times as possible, by as many CTAs as are resident at once, or as there can be units for.
// The capacity decides, not the lengths, which only the device knows.
Plan plan_for(int B, int Hkv, int Hq, int T, int D, int blocks) {
  Plan pl;
  const int rows = Hq / Hkv * T, most = D == 128 ? 2 : 4;
  auto tiles = [&](int nq) { return (rows + 8 * nq - 1) / (8 * nq); };
  for (pl.nq = 1; pl.nq <= most; ++pl.nq) {
    pl.row_tiles = tiles(pl.nq);
    const long long slots = (long long)device_sm_count() * resident_ctas(D, pl.nq, 0), items = (long long)B * Hkv * pl.row_tiles;
    pl.cluster = 1;
    while (pl.cluster < 8 && pl.cluster * kWarps < blocks) pl.cluster *= 2;
    while (pl.cluster > 1 && items * pl.cluster > slots) pl.cluster /= 2;
    pl.ctas = int(items * pl.cluster < slots ? items * pl.cluster : slots);
    if (blocks <= 2 * kWarps * pl.cluster && items * pl.cluster <= slots) return pl;
    if (pl.row_tiles == 1) break;
  }
  pl.nq = (rows + 7) / 8 < most ? (rows + 7) / 8 : most;
  pl.row_tiles = tiles(pl.nq);
  pl.cluster = 0;
  const long long units = (long long)B * Hkv * pl.row_tiles * blocks, slots = (long long)device_sm_count() * resident_ctas(D, pl.nq, B);
  pl.ctas = int(units < slots ? units : slots);
  return pl;
}

// Allows a kernel its dynamic shared memory, once a device.
template <typename T, int D, int NQ, bool CLUSTER>
cudaError_t allow_shared() {
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (ready[dev]) return cudaSuccess;
  err = cudaFuncSetAttribute(cached_attention_kernel<T, D, NQ, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             shared_bytes(D, NQ) + (CLUSTER ? 0 : (kBatchMax + 1) * 4));
  if (err == cudaSuccess) ready[dev] = true;
  return err;
}

// CTAs of a plan's kernel that an SM holds at once, by the runtime.
template <typename T, int D, int NQ>
cudaError_t measured_residency(const Plan& pl, int B, int* ctas) {
  const cudaError_t err = pl.cluster > 0 ? allow_shared<T, D, NQ, true>() : allow_shared<T, D, NQ, false>();
  if (err != cudaSuccess) return err;
  const auto kernel = pl.cluster > 0 ? cached_attention_kernel<T, D, NQ, true> : cached_attention_kernel<T, D, NQ, false>;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(ctas, kernel, kWarps * 32, size_t(shared_bytes(D, NQ)) + (pl.cluster > 0 ? 0 : (B + 1) * 4));
}

template <typename T, int D, int NQ>
cudaError_t launch_typed(const Params& p, int cluster, cudaStream_t stream) {
  const int bytes = shared_bytes(D, NQ);
  cudaError_t err = cluster > 0 ? allow_shared<T, D, NQ, true>() : allow_shared<T, D, NQ, false>();
  if (err != cudaSuccess) return err;
  if (cluster > 0) {
    ++g_launch_count;
    return launch_chained(cached_attention_kernel<T, D, NQ, true>, dim3(unsigned(p.ctas)), kWarps * 32, size_t(bytes), cluster, stream, p);
  }
  const long long rows = (long long)p.B * p.Hkv * p.group * p.T;
  if (rows > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  ++g_launch_count;
  err = launch_chained(cached_attention_kernel<T, D, NQ, false>, dim3(unsigned(p.ctas)), kWarps * 32, size_t(bytes) + (p.B + 1) * 4, 0, stream, p);
  if (err != cudaSuccess) return err;
  ++g_launch_count;
  // A CTA a row is the shorter chain (64 sequences, 768 rows: 24.8 us, with a warp a row 27.6) as long as all are resident at once; 4,480
  // rows (14 sequences, 10 new tokens, 32 heads on 8 of 32) take 33.1 us in all with a CTA a row and 24.3 with a warp a row.
  if (rows > (2048 / kJoinThreads) * (long long)device_sm_count())
    return launch_chained(join_rows_kernel<T, D>, dim3(unsigned((rows + kJoinThreads / 32 - 1) / (kJoinThreads / 32))), kJoinThreads, size_t(p.B + 1) * 4, 0, stream,
                          p, 8 * NQ, int(rows));
  return launch_chained(join_parts_kernel<T, D>, dim3(unsigned(rows)), kJoinThreads, size_t(p.B + 1 + 2 * (p.ctas + 2 * kWarps)) * 4, 0, stream, p, 8 * NQ);
}

struct Launch {
  const Params& p;
  int cluster;
  cudaStream_t stream;
  template <typename T, int D, int NQ> cudaError_t run() const { return launch_typed<T, D, NQ>(p, cluster, stream); }
};
struct Residency {
  const Plan& plan;
  int B, *ctas;
  template <typename T, int D, int NQ> cudaError_t run() const { return measured_residency<T, D, NQ>(plan, B, ctas); }
};
// f.run of the kernel that serves a type, a head dimension and a row tile.
template <typename F>
cudaError_t for_kernel(bool fp16, int D, int nq, const F& f) {
  auto rows = [&](auto t, auto d) -> cudaError_t {
    constexpr int kD = decltype(d)::value;
    using T = decltype(t);
    if (nq == 1) return f.template run<T, kD, 1>();
    if (nq == 2) return f.template run<T, kD, 2>();
    if constexpr (kD != 128) return nq == 3 ? f.template run<T, kD, 3>() : f.template run<T, kD, 4>();
    return cudaErrorInvalidValue;
  };
  auto dims = [&](auto t) -> cudaError_t {
    if (D == 32) return rows(t, std::integral_constant<int, 32>());
    if (D == 64) return rows(t, std::integral_constant<int, 64>());
    if (D == 128) return rows(t, std::integral_constant<int, 128>());
    return cudaErrorInvalidValue;
  };
  return fp16 ? dims(__half()) : dims(__nv_bfloat16());
}

}  // namespace

bool cached_attention_fits(int B, int Hkv, int Hq, int T, int D, int blocks) {
  const Plan pl = plan_for(B, Hkv, Hq, T, D, blocks);
  return B <= kBatchMax && (long long)B * Hkv * pl.row_tiles * blocks <= (1ll << 30);
}

size_t cached_attention_workspace_floats(int B, int Hkv, int Hq, int T, int D, int blocks) {
  const Plan pl = plan_for(B, Hkv, Hq, T, D, blocks);
  return pl.cluster > 0 ? 0 : size_t(2) * pl.ctas * kWarps * (8 * pl.nq) * (D + 2);
}

cudaError_t launch_cached_attention(const CachedAttentionArgs& a) {
  const CacheView& c = a.cache;
  if (!cached_attention_fits(c.B, c.Hkv, a.Hq, a.T, c.D, c.blocks)) return cudaErrorInvalidValue;
  const Plan pl = plan_for(c.B, c.Hkv, a.Hq, a.T, c.D, c.blocks);
  if (pl.cluster == 0 && a.workspace == nullptr) return cudaErrorInvalidValue;
  Params p;
  p.records = c.records; p.tail = c.tail; p.start = c.start; p.count = c.count;
  p.B = c.B; p.Hkv = c.Hkv; p.blocks = c.blocks; p.Hq = a.Hq; p.T = a.T; p.group = a.Hq / c.Hkv;
  p.row_tiles = pl.row_tiles; p.ctas = pl.ctas;
  p.q = a.q.p; p.sb = a.q.sb; p.sh = a.q.sh; p.st = a.q.st;
  p.o = a.o; p.part = a.workspace; p.sm_log2 = a.scale * kLog2e; p.status = a.status;
  return for_kernel(c.fp16, c.D, pl.nq, Launch{p, pl.cluster, a.stream});
}

cudaError_t cached_attention_plan(int B, int Hkv, int Hq, int T, int D, int blocks, bool fp16, CachedAttentionPlan* out) {
  const Plan pl = plan_for(B, Hkv, Hq, T, D, blocks);
  out->rows = 8 * pl.nq;
  out->ctas = pl.ctas;
  out->cluster = pl.cluster;
  return for_kernel(fp16, D, pl.nq, Residency{pl, B, &out->resident});
}

}  // namespace mts
