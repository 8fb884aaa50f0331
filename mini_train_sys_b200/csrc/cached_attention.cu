// Attention of a few new tokens over the 8-bit key / value cache (layout: decode.cuh).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(D) - max),  j <= position of the query
//
// One pass over the cache with a running maximum and sum.  Keys and values are read once per tile of query rows (the heads that
// share a K/V head, times the new tokens of the step) and go from global memory straight into matrix fragments: a lane's 16
// bytes are the K or V fragment of several steps (the V rows are stored in that order), 4 bytes become two fp16 pairs in four
// instructions, and both products run on m16n8k16 with the tokens (K) or the head's dims (V) as rows and eight query rows as
// columns.  What bounds it: reading the codes, 2 D bytes per token and K/V head.
//
// Rounding: codes are exact in fp16.  A query row is scaled by the power of two that brings its largest value to [1, 2), so bf16
// queries keep their eight bits in fp16.  Probabilities are rounded to fp16 (2^-11 of each, at a scale of 2^14 so that the
// smallest kept one is 2^-38 of the largest); the sum of probabilities, the maximum and the output accumulators are fp32.  In
// the unfinished block, whose values are bf16, a probability is the sum of two bf16 values.
#include "decode.cuh"
#include "ops.cuh"
#include "mma_sync.cuh"

#include <math_constants.h>

namespace mts {

namespace {

constexpr int BLK = kCacheBlock;
constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kProbShift = 14.f;       // probabilities are held times 2^14

struct Params {
  const uint8_t* codes;
  const float* scale;
  const void* tail;
  const int* start;
  const int* count;
  int Hkv, blocks, Hq, T, group, row_tiles, splits;
  const void* q;
  long long sb, sh, st;
  void* o;
  float* part;                           // [item][split][rows][D + 2]
  float sm_log2;                         // log2(e) / sqrt(D)
};

template <typename T> struct Act;
template <> struct Act<__nv_bfloat16> {
  static constexpr bool kHalf = false;
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};
template <> struct Act<__half> {
  static constexpr bool kHalf = true;
  static __device__ __forceinline__ float lo(uint32_t w) { return __low2float(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __high2float(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};

// N bytes (8, 16 or 32) into N / 4 words; cache lines of the codes are read once, so they do not stay in L1.
template <int WORDS>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 2) {
    const uint2 v = __ldg(static_cast<const uint2*>(p));
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
      const uint4 v = __ldg(static_cast<const uint4*>(p) + i);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}

// Running statistics and output of 8 * NQ query rows in one warp.  A lane holds the columns 2c and 2c + 1 of every tile of
// eight rows (the statistics are the same in the eight lanes that share c) and the dims g and g + 8 of every 16.
template <int D, int NQ>
struct State {
  float m[NQ][2], l[NQ][2], o[NQ][D / 16][4];
};

// Scores of one block (log2 domain, -inf where masked) -> probabilities as fragments; rescales the state.
// s[m][n][i]: token 16 m + g + 8 (i >> 1), query 2c + (i & 1) of tile n.
template <int D, int NQ>
__device__ __forceinline__ void update_max(State<D, NQ>& st, float (&s)[4][NQ][4]) {
  bool moved = false;
  float alpha[NQ][2];
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float mx = -CUDART_INF_F;
#pragma unroll
      for (int m = 0; m < 4; ++m) mx = fmaxf(mx, fmaxf(s[m][n][j], s[m][n][j + 2]));
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      mx = fmaxf(mx, st.m[n][j]);
      const float base = mx == -CUDART_INF_F ? 0.f : mx;     // a row that has seen nothing yet
      alpha[n][j] = exp2f(st.m[n][j] - base);
      moved |= mx != st.m[n][j];
      st.m[n][j] = mx;
      const float shift = base - kProbShift;
      float sum = 0.f;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[m][n][j + 2 * i] = exp2f(s[m][n][j + 2 * i] - shift);
          sum += s[m][n][j + 2 * i];
        }
      st.l[n][j] = st.l[n][j] * alpha[n][j] + sum;           // per lane: summed over the eight g at the end
    }
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[n][d][i] *= alpha[n][i & 1];
  }
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(kWarps * 32)
cached_attention_kernel(const Params p) {
  constexpr int KW = D / 16;             // K words per lane and token = steps of 16 dims
  constexpr int DT = D / 16;             // tiles of 16 dims of the output
  constexpr int ROWS = 8 * NQ;
  constexpr int OP = ROWS + 1;           // pitch of the output exchange
  __shared__ float ml_sm[kWarps][ROWS][2];
  __shared__ float o_sm[kWarps][D * OP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, item = blockIdx.y + blockIdx.z * gridDim.y;
  const int tile = item % p.row_tiles, bh = item / p.row_tiles;
  const int h = bh % p.Hkv, b = bh / p.Hkv;
  const int rows = p.group * p.T, row0 = tile * ROWS;
  const int capacity = p.blocks * BLK;
  const int start = min(max(p.start[b], 0), capacity);
  const int total = min(start + min(max(p.count[b], 0), p.T), capacity);
  const int fresh = total - start;       // rows of tokens t >= fresh are padding
  const int t_last = min(min(row0 + ROWS, rows) - 1, fresh * p.group - 1) / p.group;
  const bool live = row0 < fresh * p.group;
  const int blocks = live ? (start + t_last) / BLK + 1 : 0;
  const int closed = total / BLK;
  const int lo = int((long long)blocks * split / p.splits), hi = int((long long)blocks * (split + 1) / p.splits);

  State<D, NQ> st;
  int limit[NQ][2];                      // last position that a column sees
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      st.m[n][j] = -CUDART_INF_F;
      st.l[n][j] = 0.f;
      const int r = row0 + n * 8 + 2 * c + j;
      limit[n][j] = r < fresh * p.group ? start + r / p.group : -1;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[n][d][i] = 0.f;
  }

  if (lo + warp < hi) {
    // ---- query fragments: column g of every tile, dims 4 KW c ... of the head ----
    uint32_t qf[NQ][KW][2];              // fp16, scaled
    float qscale[NQ][2];                 // log2(e) / sqrt(D) times the power of two taken out, for the columns 2c, 2c + 1
    const T* qrow[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = row0 + n * 8 + g;
      const bool ok = r < rows;
      const int t = ok ? r / p.group : 0, head = h * p.group + (ok ? r % p.group : 0);
      qrow[n] = static_cast<const T*>(p.q) + b * p.sb + head * p.sh + t * p.st + c * (4 * KW);
      uint32_t w[2 * KW];
      load_words<2 * KW>(qrow[n], w);
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

    const uint8_t* base = p.codes + (long long)bh * p.blocks * (2 * BLK * D);
    const float2* scales = reinterpret_cast<const float2*>(p.scale) + (long long)bh * p.blocks;
    const int hi8 = min(hi, closed);
    uint32_t kr[4][2][KW];
    float2 sc_next = make_float2(0.f, 0.f);
    auto load_k = [&](int blk) {
      const uint8_t* kp = base + (long long)blk * (2 * BLK * D) + g * D + c * (4 * KW);
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int u = 0; u < 2; ++u) load_words<KW>(kp + (16 * m + 8 * u) * D, kr[m][u]);
      sc_next = __ldg(scales + blk);
    };
    int blk = lo + warp;
    if (blk < hi8) load_k(blk);
    for (; blk < hi8; blk += kWarps) {
      const float2 sc = sc_next;
      uint32_t vr[DT][2][4];
      const uint8_t* vp = base + (long long)blk * (2 * BLK * D) + BLK * D + g * BLK + c * 16;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u) load_words<4>(vp + (16 * d + 8 * u) * BLK, vr[d][u]);
      float s[4][NQ][4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][n][i] = 0.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          uint32_t a0, a1, a2, a3;
          codes_to_half(kr[m][0][i], a0, a2);
          codes_to_half(kr[m][1][i], a1, a3);
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma_f16(s[m][n], a0, a1, a2, a3, qf[n][i][0], qf[n][i][1]);
        }
      }
      if (blk + kWarps < hi8) load_k(blk + kWarps);
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float f = qscale[n][j] * sc.x;
#pragma unroll
          for (int m = 0; m < 4; ++m) { s[m][n][j] *= f; s[m][n][j + 2] *= f; }
        }
      const bool masked = blk * BLK + BLK > start;           // blocks of the step itself: rows see different lengths
      if (masked) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (blk * BLK + 16 * m + g + 8 * (i >> 1) > limit[n][i & 1]) s[m][n][i] = -CUDART_INF_F;
      }
      update_max<D, NQ>(st, s);
      uint32_t pf[4][NQ][2];
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          pf[m][n][0] = transpose8x8(pack_half2(s[m][n][0], s[m][n][1]));
          pf[m][n][1] = transpose8x8(pack_half2(s[m][n][2], s[m][n][3]));
        }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        float acc[NQ][4];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          uint32_t a0, a1, a2, a3;
          codes_to_half(vr[d][0][m], a0, a2);
          codes_to_half(vr[d][1][m], a1, a3);
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma_f16(acc[n], a0, a1, a2, a3, pf[m][n][0], pf[m][n][1]);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)      // a block that a row does not see at all must not reach it through its scale
            if (!masked || blk * BLK <= limit[n][i & 1]) st.o[n][d][i] = fmaf(acc[n][i], sc.y, st.o[n][d][i]);
      }
    }

    // ---- the unfinished block, in the activation type ----
    if (blk == closed && blk < hi) {
      const T* tk = static_cast<const T*>(p.tail) + ((long long)bh * 2 + (blk & 1)) * (2 * BLK * D);
      const T* tv = tk + BLK * D;
      const int valid = total - blk * BLK;                   // what lies behind is not read
      uint32_t qa[NQ][2 * KW];
#pragma unroll
      for (int n = 0; n < NQ; ++n) load_words<2 * KW>(qrow[n], qa[n]);
      float s[4][NQ][4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        uint32_t a[2][2 * KW];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int tok = 16 * m + 8 * u + g;
          if (tok < valid) {
            load_words<2 * KW>(tk + tok * D + c * (4 * KW), a[u]);
          } else {
#pragma unroll
            for (int i = 0; i < 2 * KW; ++i) a[u][i] = 0;
          }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][n][i] = 0.f;
#pragma unroll
          for (int i = 0; i < KW; ++i) {
            const uint32_t f[4] = {a[0][2 * i], a[1][2 * i], a[0][2 * i + 1], a[1][2 * i + 1]};
            Act<T>::mma(s[m][n], f, qa[n][2 * i], qa[n][2 * i + 1]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool seen = blk * BLK + 16 * m + g + 8 * (i >> 1) <= limit[n][i & 1];
            s[m][n][i] = seen ? s[m][n][i] * p.sm_log2 : -CUDART_INF_F;
          }
        }
      }
      update_max<D, NQ>(st, s);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (16 * m >= valid) break;
        uint32_t ph[NQ][2], pl[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float x = s[m][n][2 * u], y = s[m][n][2 * u + 1];
            if (Act<T>::kHalf) {
              ph[n][u] = transpose8x8(pack_half2(x, y));
            } else {
              const uint32_t hi2 = pack_bf162(x, y);
              ph[n][u] = transpose8x8(hi2);
              pl[n][u] = transpose8x8(pack_bf162(x - Act<T>::lo(hi2), y - Act<T>::hi(hi2)));
            }
          }
        const int left = valid - 16 * m - 2 * c;             // tokens 16 m + 2c + {0, 1, 8, 9} of this lane that exist
        const uint32_t keep0 = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u;
        const uint32_t keep1 = left >= 10 ? 0xFFFFFFFFu : left == 9 ? 0xFFFFu : 0u;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          uint32_t f[4];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint2 w = *reinterpret_cast<const uint2*>(tv + (16 * d + 8 * u + g) * BLK + c * 16 + m * 4);
            f[u] = w.x & keep0;
            f[u + 2] = w.y & keep1;
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            Act<T>::mma(st.o[n][d], f, ph[n][0], ph[n][1]);
            if (!Act<T>::kHalf) Act<T>::mma(st.o[n][d], f, pl[n][0], pl[n][1]);
          }
        }
      }
    }
  }

  // ---- join the warps ----
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float l = st.l[n][j];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      if (g == 0) {
        ml_sm[warp][n * 8 + 2 * c + j][0] = st.m[n][j];
        ml_sm[warp][n * 8 + 2 * c + j][1] = l;
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o_sm[warp][(16 * d + g + 8 * (i >> 1)) * OP + n * 8 + 2 * c + (i & 1)] = st.o[n][d][i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * D; i += kWarps * 32) {
    const int r = i / D, d = i % D, row = row0 + r;
    if (row >= rows) break;
    float m = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml_sm[w][r][0]);
    const float base = m == -CUDART_INF_F ? 0.f : m;
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float a = exp2f(ml_sm[w][r][0] - base);
      l = fmaf(ml_sm[w][r][1], a, l);
      o = fmaf(o_sm[w][d * OP + r], a, o);
    }
    if (p.splits == 1) {
      const int t = row / p.group, head = h * p.group + row % p.group;
      static_cast<T*>(p.o)[(((long long)b * p.T + t) * p.Hq + head) * D + d] = Act<T>::from(t < fresh ? o / l : 0.f);
    } else {
      float* dst = p.part + (((long long)item * p.splits + split) * ROWS + r) * (D + 2);
      dst[d] = o;
      if (d == 0) { dst[D] = m; dst[D + 1] = l; }
    }
  }
}

// Joins the splits of one row: one warp a row, splits in order.
template <typename T, int D>
__global__ void __launch_bounds__(128)
join_splits_kernel(const Params p, int rows_per_tile, long long total_rows) {
  const long long gr = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (gr >= total_rows) return;
  const int lane = threadIdx.x & 31;
  const int rows = p.group * p.T;
  const int row = int(gr % rows);
  const long long bh = gr / rows;
  const int h = int(bh % p.Hkv), b = int(bh / p.Hkv);
  const long long item = bh * p.row_tiles + row / rows_per_tile;
  const float* src = p.part + (item * p.splits * rows_per_tile + row % rows_per_tile) * (D + 2);
  const long long pitch = (long long)rows_per_tile * (D + 2);
  const int capacity = p.blocks * BLK;
  const int start = min(max(p.start[b], 0), capacity);
  const int fresh = min(start + min(max(p.count[b], 0), p.T), capacity) - start;
  const int t = row / p.group, head = h * p.group + row % p.group;
  float m = -CUDART_INF_F;
  for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, src[s * pitch + D]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float base = m == -CUDART_INF_F ? 0.f : m;
  float l = 0.f, o[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) o[j] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float a = exp2f(src[s * pitch + D] - base);
    l = fmaf(src[s * pitch + D + 1], a, l);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) o[j] = fmaf(src[s * pitch + j * 32 + lane], a, o[j]);
  }
  T* dst = static_cast<T*>(p.o) + (((long long)b * p.T + t) * p.Hq + head) * D;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) dst[j * 32 + lane] = Act<T>::from(t < fresh ? o[j] / l : 0.f);
}

struct Plan {
  int nq, row_tiles, splits;
  long long items;
};

// Query rows in tiles of 8, 16 or 32 (16 at D = 128, where the accumulators of 32 would not fit in registers), and as many splits
// of the cache as fill the machine with four CTAs an SM, while each warp of a split still has a block of its own.
// The capacity decides, not the lengths, which only the device knows.
Plan plan_for(int B, int Hkv, int Hq, int T, int D, int blocks) {
  Plan pl;
  const int rows = Hq / Hkv * T, most = D == 128 ? 2 : 4;
  pl.nq = rows <= 8 ? 1 : rows <= 16 ? 2 : most;
  pl.row_tiles = (rows + 8 * pl.nq - 1) / (8 * pl.nq);
  pl.items = (long long)B * Hkv * pl.row_tiles;
  const long long want = ((long long)device_sm_count() * 4 + pl.items - 1) / pl.items;
  const long long fit = (blocks + kWarps - 1) / kWarps;
  const long long s = want < fit ? want : fit;
  pl.splits = int(s < 1 ? 1 : s);
  return pl;
}

template <typename T, int D, int NQ>
cudaError_t launch_typed(const Params& p, const Plan& pl, int B, cudaStream_t stream) {
  // the grid's y and z extents hold at most 65,535 each
  const long long y = pl.items < 32768 ? pl.items : 1;
  long long gy = y, gz = 1;
  if (pl.items >= 32768) {
    gy = (long long)p.Hkv * p.row_tiles;
    gz = B;
    if (gy > 65535 || gz > 65535) return cudaErrorInvalidConfiguration;
  }
  cached_attention_kernel<T, D, NQ><<<dim3(unsigned(p.splits), unsigned(gy), unsigned(gz)), kWarps * 32, 0, stream>>>(p);
  ++g_launch_count;
  if (p.splits > 1) {
    const long long rows = (long long)B * p.Hkv * p.group * p.T;
    join_splits_kernel<T, D><<<unsigned((rows + 3) / 4), 128, 0, stream>>>(p, 8 * NQ, rows);
    ++g_launch_count;
  }
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_dim(const Params& p, const Plan& pl, int B, cudaStream_t stream) {
  if (pl.nq == 1) return launch_typed<T, D, 1>(p, pl, B, stream);
  if (pl.nq == 2) return launch_typed<T, D, 2>(p, pl, B, stream);
  if constexpr (D != 128) return launch_typed<T, D, 4>(p, pl, B, stream);
  return cudaErrorInvalidValue;
}

}  // namespace

size_t cached_attention_workspace_floats(int B, int Hkv, int Hq, int T, int D, int blocks) {
  const Plan pl = plan_for(B, Hkv, Hq, T, D, blocks);
  return pl.splits == 1 ? 0 : size_t(pl.items) * pl.splits * (8 * pl.nq) * (D + 2);
}

cudaError_t launch_cached_attention(const CachedAttentionArgs& a) {
  const CacheView& c = a.cache;
  const Plan pl = plan_for(c.B, c.Hkv, a.Hq, a.T, c.D, c.blocks);
  if (pl.splits > 1 && a.workspace == nullptr) return cudaErrorInvalidValue;
  Params p;
  p.codes = c.codes; p.scale = c.scale; p.tail = c.tail; p.start = c.start; p.count = c.count;
  p.Hkv = c.Hkv; p.blocks = c.blocks; p.Hq = a.Hq; p.T = a.T; p.group = a.Hq / c.Hkv;
  p.row_tiles = pl.row_tiles; p.splits = pl.splits;
  p.q = a.q.p; p.sb = a.q.sb; p.sh = a.q.sh; p.st = a.q.st;
  p.o = a.o; p.part = a.workspace; p.sm_log2 = a.scale * kLog2e;
  if (c.D == 32) return c.fp16 ? launch_dim<__half, 32>(p, pl, c.B, a.stream) : launch_dim<__nv_bfloat16, 32>(p, pl, c.B, a.stream);
  if (c.D == 64) return c.fp16 ? launch_dim<__half, 64>(p, pl, c.B, a.stream) : launch_dim<__nv_bfloat16, 64>(p, pl, c.B, a.stream);
  if (c.D == 128) return c.fp16 ? launch_dim<__half, 128>(p, pl, c.B, a.stream) : launch_dim<__nv_bfloat16, 128>(p, pl, c.B, a.stream);
  return cudaErrorInvalidValue;
}

}  // namespace mts
