// Appending to the 8-bit key / value cache, and reading it back (layout: decode.cuh).
//
//   a = max |x| over the 64 x D values of a finished block,  scale = a / 127,  code = rint(127 x / a)  (half to even)
//
// What bounds them: appending reads the new tokens once and writes their codes, 3 bytes a value (and q, 4 bytes a value); reading
// back reads a byte a value and writes four.  So they are bound by memory for a prompt and by their launch for one token.
// Measured on the GPU (replayed graph, caches flushed), an append and a read-back of 12 heads of 64: one sequence of 448 tokens,
// one new, 5.2 us; 64 ragged sequences of up to 512 tokens, one new, 17.7 us (51 MB, 2.9 TB/s); 16 ragged prompts of up to
// 2,048 tokens 75.8 us (338 MB, 4.5 TB/s), of which the append, whose conversions keep the issue slots busy, takes half.
#include "decode.cuh"
#include "launch.cuh"
#include "ops.cuh"
#include "mma_sync.cuh"

#include <math_constants.h>

namespace mts {

namespace {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> union Vec8T { uint4 q; uint32_t w[4]; T v[8]; };

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf162(a, b); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return pack_half2(a, b); }

// Half-split rotation as the rotary kernel computes it: the products of 16-bit factors are exact in fp32, their sum is rounded there
// and then to T.
template <typename T>
__device__ __forceinline__ void rotate8(Vec8T<T>& lo, Vec8T<T>& hi, const T* c, const T* s) {
  Vec8T<T> cv, sv;
  cv.q = *reinterpret_cast<const uint4*>(c);
  sv.q = *reinterpret_cast<const uint4*>(s);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 a = unpack2<T>(lo.w[j]), b = unpack2<T>(hi.w[j]), cc = unpack2<T>(cv.w[j]), ss = unpack2<T>(sv.w[j]);
    lo.w[j] = pack2<T>(fmaf(a.x, cc.x, -__fmul_rn(b.x, ss.x)), fmaf(a.y, cc.y, -__fmul_rn(b.y, ss.y)));
    hi.w[j] = pack2<T>(fmaf(b.x, cc.x, __fmul_rn(a.x, ss.x)), fmaf(b.y, cc.y, __fmul_rn(a.y, ss.y)));
  }
}

// Codes of eight values of a block whose largest magnitude is amax: 127 x / amax to the nearest integer, a half to the even one.
// With whole mantissas, and in units of amax's last place, amax = A and x = X 2^-d; a half is 254 X = A 2^d (2n + 1).  127 is prime, so
// it divides 2n + 1 (then n is 63: x is half of amax, not a rare value) or A.  Where it does not divide A, the difference of the two sides
// is a whole number, an even one for d > 0, so everything else is at least 1 / (2 A) from a half for d = 0 and 2^-d / A for d > 0: more than
// 2^-12 and 2^-11 2^-d in fp16, and than these in bf16.  A product with 127 / amax, rounded and made two units in the last place too large,
// is off by at most 2.5 x 2^-23 of itself: 127 x 2.5 x 2^-23 = 3.8e-5 for d = 0 and, since X < 2 A, 7.6e-5 2^-d above, less than either
// distance.  It takes half of amax to just above 63.5, hence to 64, the even one.  Adding 1.5 * 2^23 leaves the integer in the low bits of the
// sum.  Blocks with other A (and with a subnormal or huge amax) take correctly rounded quotients, scaled by a power of two.
struct Quantizer {
  float amax, inv;
  bool quick;
};
template <typename T> __device__ __forceinline__ bool mantissa_is_plain(uint32_t bits);
template <> __device__ __forceinline__ bool mantissa_is_plain<__nv_bfloat16>(uint32_t bits) { return (bits & 0x7Fu) != 0x7Eu; }   // 254 = 2 * 127
template <> __device__ __forceinline__ bool mantissa_is_plain<__half>(uint32_t bits) { return bits >= 0x400u && ((bits & 0x3FFu) | 0x400u) % 127u != 0u; }

template <typename T>
__device__ __forceinline__ uint2 codes_of(const Vec8T<T>& x, const Quantizer& q) {
  constexpr float kMagic = 12582912.f;
  uint32_t bits[8];
  if (q.quick) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 v = unpack2<T>(x.w[j]);
      bits[2 * j] = __float_as_uint(fmaf(v.x, q.inv, kMagic));
      bits[2 * j + 1] = __float_as_uint(fmaf(v.y, q.inv, kMagic));
    }
  } else {
    const float scale = q.amax > 1.f ? 0x1p-60f : 0x1p60f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 v = unpack2<T>(x.w[j >> 1]);
      bits[j] = q.amax > 0.f ? uint32_t(int(rintf(__fdiv_rn(((j & 1) ? v.y : v.x) * scale * 127.f, q.amax * scale)))) : 0u;
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = __byte_perm(__byte_perm(bits[4 * i], bits[4 * i + 1], 0x0040), __byte_perm(bits[4 * i + 2], bits[4 * i + 3], 0x0040), 0x5410) ^ 0x80808080u;
  return make_uint2(w[0], w[1]);
}

// Largest magnitude of pairs of 16-bit values, as their bits: the order of the bits is the order of the values, and a NaN is above
// infinity.
__device__ __forceinline__ uint32_t larger(uint32_t most, uint32_t pair) { return __vmaxu2(most, pair & 0x7FFF7FFFu); }
__device__ __forceinline__ uint32_t larger(uint32_t most, const uint4& q) { return larger(larger(larger(larger(most, q.x), q.y), q.z), q.w); }
template <typename T> __device__ __forceinline__ float value_of(uint32_t bits);
template <> __device__ __forceinline__ float value_of<__nv_bfloat16>(uint32_t bits) { return __uint_as_float(bits << 16); }
template <> __device__ __forceinline__ float value_of<__half>(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }

constexpr int kAppendThreads = 256;
constexpr int kQPieces = 4;              // of 32 bytes of q, a thread

// One CTA per (block that the step touches, K/V head, sequence); the CTAs behind those rotate q.
// A thread owns eight dims of the lower half of a head and their partners in the upper half, for one token.
template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads, D == 128 ? 2 : 4)
kv_append_kernel(CacheView c, Strided q, int Hq, Strided k, Strided v, T* __restrict__ q_out, const T* cosv, const T* sinv,
                 int table_rows, int Tn, int kv_ctas, int q_ctas, int blocks_per_head) {
  constexpr int VEC = D / 16;                              // threads per token
  constexpr int ITER = (kCacheBlock * VEC + kAppendThreads - 1) / kAppendThreads;
  constexpr int BLK = kCacheBlock;
  const int tid = threadIdx.x;
  let_next_start();
  wait_for_previous();
  if (int(blockIdx.x) >= kv_ctas) {                        // ---- q: a CTA takes consecutive pieces of one sequence ----
    const unsigned per_token = unsigned(Hq) * VEC, pieces = unsigned(Tn) * per_token;    // at most 2^31, checked by the launcher
    const unsigned at = unsigned(blockIdx.x) - unsigned(kv_ctas), b = at / unsigned(q_ctas), base = at % unsigned(q_ctas) * (kQPieces * kAppendThreads) + tid;
    const int start = c.start[b], count = c.count[b];
    Vec8T<T> lo[kQPieces], hi[kQPieces];
    unsigned t[kQPieces], rest[kQPieces];
#pragma unroll
    for (int i = 0; i < kQPieces; ++i) {                   // all loads before the first store
      const unsigned piece = base + i * kAppendThreads;
      t[i] = piece / per_token;
      rest[i] = piece % per_token;
      lo[i].q = hi[i].q = make_uint4(0, 0, 0, 0);
      const int p = start + int(t[i]);
      if (piece < pieces && int(t[i]) < count && p >= 0 && p < c.blocks * BLK) {
        const T* src = static_cast<const T*>(q.p) + b * q.sb + rest[i] / VEC * q.sh + t[i] * q.st + rest[i] % VEC * 8;
        lo[i].q = *reinterpret_cast<const uint4*>(src);
        hi[i].q = *reinterpret_cast<const uint4*>(src + D / 2);
      }
    }
#pragma unroll
    for (int i = 0; i < kQPieces; ++i) {
      const int p = start + int(t[i]);
      if (base + i * kAppendThreads >= pieces) break;
      if (cosv != nullptr && int(t[i]) < count && p >= 0 && p < c.blocks * BLK) {
        const long long at = (long long)min(p, table_rows - 1) * D + rest[i] % VEC * 8;
        rotate8(lo[i], hi[i], cosv + at, sinv + at);
      }
      T* dst = q_out + (((long long)b * Tn + t[i]) * Hq + rest[i] / VEC) * D + rest[i] % VEC * 8;
      *reinterpret_cast<uint4*>(dst) = lo[i].q;
      *reinterpret_cast<uint4*>(dst + D / 2) = hi[i].q;
    }
    return;
  }

  __shared__ unsigned amax_sm[2][kAppendThreads / 32];
  constexpr int V_PITCH = BLK + 4;
  __shared__ __align__(16) uint8_t v_sm[D * V_PITCH];
  const int item = int(blockIdx.x) % blocks_per_head;
  const int bh = int(blockIdx.x) / blocks_per_head;
  const int h = bh % c.Hkv, b = bh / c.Hkv;
  const int limit = c.blocks * BLK;
  const int start = min(max(c.start[b], 0), limit);
  const int end = min(start + min(max(c.count[b], 0), Tn), limit);
  if (end <= start) return;
  const int first_block = start / BLK, last_block = (end - 1) / BLK;
  const int block = first_block + item;
  if (block > last_block) return;
  // The first block takes its older tokens from the tail, and a last, unfinished block may go to the same half of it: then this
  // CTA writes that block too, after it has read.
  const bool last_open = (end % BLK) != 0;
  const bool shared_half = last_open && last_block > first_block && ((last_block - first_block) & 1) == 0 && (start % BLK) != 0;
  if (shared_half && item > 0 && block == last_block) return;

  const T* kb = static_cast<const T*>(k.p) + b * k.sb + h * k.sh;
  const T* vb = static_cast<const T*>(v.p) + b * v.sb + h * v.sh;
  T* tail = static_cast<T*>(c.tail) + (long long)bh * 4 * BLK * D;
  for (int pass = 0; pass < (shared_half && item == 0 ? 2 : 1); ++pass) {
    const int blk = pass == 0 ? block : last_block;
    const int base = blk * BLK;
    T* tk = tail + (blk & 1) * 2 * BLK * D;
    T* tv = tk + BLK * D;
    const bool closes = end >= base + BLK;
    if (pass == 1) __syncthreads();
    Vec8T<T> klo[ITER], khi[ITER], vlo[ITER], vhi[ITER];
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int idx = it * kAppendThreads + tid;
      const int tok = idx / VEC, vec = idx % VEC;
      const int p = base + tok;
      klo[it].q = khi[it].q = vlo[it].q = vhi[it].q = make_uint4(0, 0, 0, 0);
      if (tok >= BLK) continue;
      if (p >= start && p < end) {
        const T* ks = kb + (p - start) * k.st + vec * 8;
        const T* vs = vb + (p - start) * v.st + vec * 8;
        klo[it].q = *reinterpret_cast<const uint4*>(ks);
        khi[it].q = *reinterpret_cast<const uint4*>(ks + D / 2);
        vlo[it].q = *reinterpret_cast<const uint4*>(vs);
        vhi[it].q = *reinterpret_cast<const uint4*>(vs + D / 2);
        if (cosv != nullptr) {
          const long long at = (long long)min(p, table_rows - 1) * D + vec * 8;
          rotate8(klo[it], khi[it], cosv + at, sinv + at);
        }
      } else if (closes && p < start) {
        klo[it].q = *reinterpret_cast<const uint4*>(tk + tok * D + vec * 8);
        khi[it].q = *reinterpret_cast<const uint4*>(tk + tok * D + D / 2 + vec * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          vlo[it].v[j] = tv[tail_slot(D, vec * 8 + j, tok)];
          vhi[it].v[j] = tv[tail_slot(D, D / 2 + vec * 8 + j, tok)];
        }
      }
    }
    if (!closes) {                                         // the block stays open: the new tokens go to the tail
#pragma unroll
      for (int it = 0; it < ITER; ++it) {
        const int idx = it * kAppendThreads + tid;
        const int tok = idx / VEC, vec = idx % VEC;
        const int p = base + tok;
        if (tok >= BLK || p < start || p >= end) continue;
        *reinterpret_cast<uint4*>(tk + tok * D + vec * 8) = klo[it].q;
        *reinterpret_cast<uint4*>(tk + tok * D + D / 2 + vec * 8) = khi[it].q;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          tv[tail_slot(D, vec * 8 + j, tok)] = vlo[it].v[j];
          tv[tail_slot(D, D / 2 + vec * 8 + j, tok)] = vhi[it].v[j];
        }
      }
      continue;
    }
    uint32_t ka = 0, va = 0;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      ka = larger(larger(ka, klo[it].q), khi[it].q);
      va = larger(larger(va, vlo[it].q), vhi[it].q);
    }
    ka = __reduce_max_sync(0xffffffffu, max(ka & 0xFFFFu, ka >> 16));
    va = __reduce_max_sync(0xffffffffu, max(va & 0xFFFFu, va >> 16));
    if ((tid & 31) == 0) { amax_sm[0][tid >> 5] = ka; amax_sm[1][tid >> 5] = va; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) { ka = max(ka, amax_sm[0][w]); va = max(va, amax_sm[1][w]); }
    auto quantizer = [](uint32_t bits) {
      Quantizer q;
      q.amax = value_of<T>(bits);
      q.quick = mantissa_is_plain<T>(bits) && q.amax > 1e-30f && q.amax < 1e30f;
      q.inv = __uint_as_float(__float_as_uint(__fdiv_rn(127.f, q.amax)) + 2u);
      if (!(q.amax < CUDART_INF_F)) q.amax = CUDART_NAN_F;                               // the whole block reads NaN
      return q;
    };
    const Quantizer kq = quantizer(ka), vq = quantizer(va);
    uint8_t* record = c.records + ((long long)bh * c.blocks + blk) * record_bytes(D);
    uint8_t* kc = record + kCacheHead;
    uint8_t* vc = kc + BLK * D;
    if (tid == 0) {
      float* sc = reinterpret_cast<float*>(record);
      sc[0] = __fdiv_rn(kq.amax, 127.f);
      sc[1] = __fdiv_rn(vq.amax, 127.f);
    }
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int idx = it * kAppendThreads + tid;
      const int tok = idx / VEC, vec = idx % VEC;
      if (tok >= BLK) continue;
      *reinterpret_cast<uint2*>(kc + tok * D + vec * 8) = codes_of(klo[it], kq);
      *reinterpret_cast<uint2*>(kc + tok * D + D / 2 + vec * 8) = codes_of(khi[it], kq);
      // Values are stored by dim, where the tokens of a pair are neighbours: each of the two threads takes four dims of both.
      const int slot = cache_slot(tok & ~1), odd = tok & 1;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint2 w = codes_of(half ? vhi[it] : vlo[it], vq);
        const uint32_t theirs = __shfl_xor_sync(0xffffffffu, odd ? w.x : w.y, VEC);
        const uint32_t even_token = odd ? theirs : w.x, odd_token = odd ? w.y : theirs;
        uint8_t* dst = v_sm + (half * (D / 2) + vec * 8 + odd * 4) * V_PITCH + slot;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint16_t*>(dst + j * V_PITCH) = uint16_t(((even_token >> (8 * j)) & 0xFFu) | (((odd_token >> (8 * j)) & 0xFFu) << 8));
      }
    }
    __syncthreads();
    for (int i = tid; i < D * BLK / 16; i += kAppendThreads) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(v_sm + i / 4 * V_PITCH + i % 4 * 16);
      reinterpret_cast<uint4*>(vc)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// One CTA of D threads per 64 positions of a (sequence, K/V head), which lie in two blocks at most.  A thread has four dims of the 16
// tokens whose values are adjacent in a row of V: it reads 16 bytes of four rows of V and four dims of each token's keys, so the
// values need not pass through shared memory to be written by token, all loads are in flight at once, and two lanes with
// neighbouring tokens use a whole sector of V between them.
template <int D>
struct ReadThread {
  static constexpr int VEC = D / 4, L = VEC < 16 ? VEC : 16;
  int a, dim;                            // the tokens 2 a + {0, 1, 8, 9} of every 16; first dim
  __device__ __forceinline__ ReadThread(int tid) : a(tid / L % 4), dim((tid % L + tid / (4 * L) * L) * 4) {}
  __device__ __forceinline__ int token(int x) const { return 2 * a + ((x >> 1) & 1) * 8 + (x & 1); }
};

// code - 128 from byte x of w: 2^23 + code is the float with code in its low bits
__device__ __forceinline__ float decode(uint32_t w, int x) { return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540 + x)) - 8388736.f; }

template <typename T, int D>
__global__ void __launch_bounds__(D)
kv_read_kernel(CacheView c, const int* first, int n, float* __restrict__ ko, float* __restrict__ vo, int chunks) {
  constexpr int BLK = kCacheBlock;
  let_next_start();
  wait_for_previous();
  const ReadThread<D> me(threadIdx.x);
  const int chunk = int(blockIdx.x) % chunks;
  const int bh = int(blockIdx.x) / chunks;
  const int b = bh / c.Hkv;
  const int total = min(min(max(c.start[b], 0), c.blocks * BLK) + max(c.count[b], 0), c.blocks * BLK), closed = total / BLK;
  const long long from = first[b], p0 = from + chunk * 64;
  const long long out0 = (long long)bh * n - from;         // row of position 0
#pragma unroll 1
  for (long long blk = p0 >> 6; blk <= (p0 + 63) >> 6; ++blk) {
    const long long base = blk * BLK;
    const int lo = int(max(p0 - base, 0ll)), hi = int(min(min(p0 + 64, from + n) - base, (long long)BLK));      // of the block's tokens
    const int live = blk < 0 ? 0 : int(min(max(total - base, 0ll), (long long)BLK));
    auto write = [&](int t, float4 k, float4 v) {
      if (t < lo || t >= hi) return;
      if (t >= live) k = v = make_float4(0.f, 0.f, 0.f, 0.f);
      const long long at = (out0 + base + t) * D + me.dim;
      *reinterpret_cast<float4*>(ko + at) = k;
      *reinterpret_cast<float4*>(vo + at) = v;
    };
    if (live == BLK) {
      const uint8_t* record = c.records + ((long long)bh * c.blocks + blk) * record_bytes(D);
      uint4 v[4];
      uint32_t k[BLK / 4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(record + kCacheHead + BLK * D + (me.dim + j) * BLK + me.a * 16);
#pragma unroll
      for (int i = 0; i < BLK / 4; ++i) k[i] = *reinterpret_cast<const uint32_t*>(record + kCacheHead + (i / 4 * 16 + me.token(i)) * D + me.dim);
      const float2 sc = *reinterpret_cast<const float2*>(record);
#pragma unroll
      for (int i = 0; i < BLK / 4; ++i) {
        const int x = i & 3;
        auto word = [&](const uint4& w) { return i < 4 ? w.x : i < 8 ? w.y : i < 12 ? w.z : w.w; };
        write(i / 4 * 16 + me.token(i), make_float4(decode(k[i], 0) * sc.x, decode(k[i], 1) * sc.x, decode(k[i], 2) * sc.x, decode(k[i], 3) * sc.x),
              make_float4(decode(word(v[0]), x) * sc.y, decode(word(v[1]), x) * sc.y, decode(word(v[2]), x) * sc.y, decode(word(v[3]), x) * sc.y));
      }
    } else if (live > 0) {
      const T* tail = static_cast<const T*>(c.tail) + ((long long)bh * 2 + (closed & 1)) * 2 * BLK * D;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        Vec8T<T> v[4];
        uint2 k[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j].q = *reinterpret_cast<const uint4*>(tail + BLK * D + (half * D + me.dim + j) * (BLK / 2) + me.a * 8);
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = *reinterpret_cast<const uint2*>(tail + (half * 32 + i / 4 * 16 + me.token(i)) * D + me.dim);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 k01 = unpack2<T>(k[i].x), k23 = unpack2<T>(k[i].y);
          write(half * 32 + i / 4 * 16 + me.token(i), make_float4(k01.x, k01.y, k23.x, k23.y),
                make_float4(to_f(v[0].v[i]), to_f(v[1].v[i]), to_f(v[2].v[i]), to_f(v[3].v[i])));
        }
      }
    } else {
#pragma unroll 4
      for (int i = 0; i < BLK / 4; ++i) write(i / 4 * 16 + me.token(i), make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
}

template <typename T, int D>
cudaError_t append_typed(const CacheView& c, const Strided& q, int Hq, const Strided& k, const Strided& v, void* q_out, const void* cosv,
                         const void* sinv, int table_rows, int Tn, cudaStream_t stream) {
  const int per_head = (Tn + kCacheBlock - 2) / kCacheBlock + 1;       // blocks that T tokens can touch
  const long long kv_ctas = (long long)c.B * c.Hkv * per_head;
  const long long pieces = q.p == nullptr ? 0 : (long long)Hq * Tn * (D / 16);
  const long long q_ctas = (pieces + kQPieces * kAppendThreads - 1) / (kQPieces * kAppendThreads);      // of a sequence
  if (kv_ctas + q_ctas * c.B > 0x7fffffffll || pieces > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  ++g_launch_count;
  return launch_chained(kv_append_kernel<T, D>, dim3(unsigned(kv_ctas + q_ctas * c.B)), kAppendThreads, 0, 0, stream, c, q, Hq, k, v, static_cast<T*>(q_out),
                        static_cast<const T*>(cosv), static_cast<const T*>(sinv), table_rows, Tn, int(kv_ctas), int(q_ctas), per_head);
}

template <typename T, int D>
cudaError_t read_typed(const CacheView& c, const int* first, int n, float* k, float* v, cudaStream_t stream) {
  const int chunks = (n + 63) / 64;
  const long long ctas = (long long)c.B * c.Hkv * chunks;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  ++g_launch_count;
  return launch_chained(kv_read_kernel<T, D>, dim3(unsigned(ctas)), D, 0, 0, stream, c, first, n, k, v, chunks);
}

}  // namespace

cudaError_t launch_kv_append(const CacheView& c, const Strided& q, int Hq, const Strided& k, const Strided& v, void* q_out, const void* cosv,
                             const void* sinv, int table_rows, int T, cudaStream_t stream) {
  if (c.D == 32) return c.fp16 ? append_typed<__half, 32>(c, q, Hq, k, v, q_out, cosv, sinv, table_rows, T, stream)
                               : append_typed<__nv_bfloat16, 32>(c, q, Hq, k, v, q_out, cosv, sinv, table_rows, T, stream);
  if (c.D == 64) return c.fp16 ? append_typed<__half, 64>(c, q, Hq, k, v, q_out, cosv, sinv, table_rows, T, stream)
                               : append_typed<__nv_bfloat16, 64>(c, q, Hq, k, v, q_out, cosv, sinv, table_rows, T, stream);
  if (c.D == 128) return c.fp16 ? append_typed<__half, 128>(c, q, Hq, k, v, q_out, cosv, sinv, table_rows, T, stream)
                                : append_typed<__nv_bfloat16, 128>(c, q, Hq, k, v, q_out, cosv, sinv, table_rows, T, stream);
  return cudaErrorInvalidValue;
}

cudaError_t launch_kv_read(const CacheView& c, const int* first, int n, float* k, float* v, cudaStream_t stream) {
  if (c.D == 32) return c.fp16 ? read_typed<__half, 32>(c, first, n, k, v, stream) : read_typed<__nv_bfloat16, 32>(c, first, n, k, v, stream);
  if (c.D == 64) return c.fp16 ? read_typed<__half, 64>(c, first, n, k, v, stream) : read_typed<__nv_bfloat16, 64>(c, first, n, k, v, stream);
  if (c.D == 128) return c.fp16 ? read_typed<__half, 128>(c, first, n, k, v, stream) : read_typed<__nv_bfloat16, 128>(c, first, n, k, v, stream);
  return cudaErrorInvalidValue;
}

}  // namespace mts
