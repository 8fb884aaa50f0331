// Appending to the 8-bit key / value cache, and reading it back (layout: decode.cuh).
//
//   a = max |x| over the 64 x D values of a finished block,  scale = a / 127,  code = rint(127 x / a)  (half to even)
//
// What bounds them: appending reads the new tokens once and writes their codes, 3 bytes a value (and q, 4 bytes a value); reading
// back reads a byte a value and writes four.  So they are bound by memory for a prompt and by their launch for one token.
// Measured on the GPU (replayed graph, caches flushed), an append and a read-back of 12 heads of 64: one sequence of 448 tokens,
// one new, 6.4 us; 64 ragged sequences of up to 512 tokens, one new, 18.4 us (50 MB moved, 2.7 TB/s); 16 ragged prompts of up to
// 2,048 tokens 80.7 us (338 MB, 4.2 TB/s), of which the append, whose conversions keep the issue slots busy, takes half.
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
// With whole mantissas, x = X 2^i and amax = A 2^j, a half is 254 X 2^(i-j) = A (2n + 1).  127 is prime, so it divides 2n + 1 (then n
// is 63: x is half of amax, not a rare value) or A.  Where it does not divide A, everything else is at least 1 / (2 A) >= 2^-12 from a
// half, and a product with 127 / amax, made two units in the last place too large, is right: it is off by 4e-5 at most, and takes
// half of amax to just above 63.5, hence to 64, the even one.  Adding 1.5 * 2^23 leaves the integer in the low bits of the sum.
// Blocks with other A (and with a subnormal or huge amax) take correctly rounded quotients, scaled by a power of two.
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
kv_append_kernel(CacheView c, Strided q, int Hq, Strided k, Strided v, T* __restrict__ q_out, const T* __restrict__ cosv,
                 const T* __restrict__ sinv, int table_rows, int Tn, int kv_ctas, int q_ctas, int blocks_per_head) {
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
      if (cosv != nullptr && int(t[i]) < count && p >= 0 && p < table_rows && p < c.blocks * BLK)
        rotate8(lo[i], hi[i], cosv + (long long)p * D + rest[i] % VEC * 8, sinv + (long long)p * D + rest[i] % VEC * 8);
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
        if (cosv != nullptr && p < table_rows)
          rotate8(klo[it], khi[it], cosv + (long long)p * D + vec * 8, sinv + (long long)p * D + vec * 8);
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

// One CTA per 64 positions of a (sequence, K/V head), which lie in two blocks at most.  The values of a block are stored by dim, so
// they pass through shared memory; then D / 4 consecutive threads write the dims of one token.
template <typename T, int D>
__global__ void __launch_bounds__(256)
kv_read_kernel(CacheView c, const int* __restrict__ first, int n, float* __restrict__ ko, float* __restrict__ vo, int chunks) {
  constexpr int BLK = kCacheBlock;
  constexpr int PITCH = BLK + 4;                           // bytes of a row of codes
  constexpr int HALF_PITCH = BLK / 2 + 2;                  // values of a row of half the unfinished block
  __shared__ __align__(16) uint8_t codes_sm[2][D * PITCH];
  __shared__ __align__(16) T tail_sm[2 * D * HALF_PITCH];
  let_next_start();
  wait_for_previous();
  const int chunk = int(blockIdx.x) % chunks;
  const int bh = int(blockIdx.x) / chunks;
  const int b = bh / c.Hkv;
  const int total = min(min(max(c.start[b], 0), c.blocks * BLK) + max(c.count[b], 0), c.blocks * BLK), closed = total / BLK;
  const long long p0 = (long long)first[b] + chunk * 64;
  const int lo = int(max(p0, 0ll) / BLK);                  // the two blocks
  const uint8_t* record0 = c.records + ((long long)bh * c.blocks + lo) * record_bytes(D);
  const T* tail = static_cast<const T*>(c.tail) + ((long long)bh * 2 + (closed & 1)) * 2 * BLK * D;
  const bool reaches = p0 + 64 > 0 && p0 < total;          // else only zeros are written
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (!reaches || lo + j > closed || (lo + j) * (long long)BLK >= total) continue;
    if (lo + j < closed) {
      const uint8_t* vc = record0 + j * record_bytes(D) + kCacheHead + BLK * D;
      for (int i = threadIdx.x; i < D * BLK / 16; i += 256) {
        const uint4 w = *reinterpret_cast<const uint4*>(vc + i * 16);
        uint32_t* dst = reinterpret_cast<uint32_t*>(&codes_sm[j][i / 4 * PITCH + i % 4 * 16]);
        dst[0] = w.x; dst[1] = w.y; dst[2] = w.z; dst[3] = w.w;
      }
    } else {
      for (int i = threadIdx.x; i < D * BLK / 8; i += 256) {
        const uint4 w = *reinterpret_cast<const uint4*>(tail + BLK * D + i * 8);
        uint32_t* dst = reinterpret_cast<uint32_t*>(&tail_sm[i / 4 * HALF_PITCH + i % 4 * 8]);
        dst[0] = w.x; dst[1] = w.y; dst[2] = w.z; dst[3] = w.w;
      }
    }
  }
  __syncthreads();
  constexpr int VEC = D / 4;
#pragma unroll 2
  for (int i = threadIdx.x; i < 64 * VEC; i += 256) {
    const int tok = i / VEC, d = i % VEC * 4, at_out = chunk * 64 + tok;
    if (at_out >= n) break;
    const long long p = p0 + tok;
    float kf[4], vf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) kf[j] = vf[j] = 0.f;
    if (p >= 0 && p < total) {
      const int blk = int(p / BLK), at = int(p % BLK);
      if (blk < closed) {
        const uint8_t* record = record0 + (blk - lo) * record_bytes(D);
        const float2 sc = *reinterpret_cast<const float2*>(record);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(record + kCacheHead + at * D + d);
        const uint8_t* vs = &codes_sm[blk - lo][d * PITCH + cache_slot(at)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kf[j] = float(int((w >> (8 * j)) & 0xFFu) - 128) * sc.x;
          vf[j] = float(int(vs[j * PITCH]) - 128) * sc.y;
        }
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(tail + at * D + d);
        const T* ks = reinterpret_cast<const T*>(&w);
        const T* vs = tail_sm + ((at >> 5) * D + d) * HALF_PITCH + tail_slot(0, 0, at & 31);
#pragma unroll
        for (int j = 0; j < 4; ++j) { kf[j] = to_f(ks[j]); vf[j] = to_f(vs[j * HALF_PITCH]); }
      }
    }
    const long long at_d = ((long long)bh * n + at_out) * D + d;
    *reinterpret_cast<float4*>(ko + at_d) = make_float4(kf[0], kf[1], kf[2], kf[3]);
    *reinterpret_cast<float4*>(vo + at_d) = make_float4(vf[0], vf[1], vf[2], vf[3]);
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
  return launch_chained(kv_read_kernel<T, D>, dim3(unsigned(ctas)), 256, 0, 0, stream, c, first, n, k, v, chunks);
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
