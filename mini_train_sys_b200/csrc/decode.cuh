// Launchers of the decoding-step kernels: the 8-bit key / value cache (append, read back, attention over it) and the
// mixture-of-experts layer for a few tokens.  Raw pointers and a stream, as in ops.cuh.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mts {

// ---- the cache of one layer -----------------------------------------------------------------------------------------
// Tokens of a (sequence, K/V head) are grouped in blocks of kCacheBlock.  A finished block is held in 8 bits, the unfinished
// one in the activation type, so that a value is rounded to 8 bits once, whatever calls brought the tokens.
//   records [B, Hkv, blocks, 16 + 2 * 64 * D] bytes: the fp32 scales of K and V (and 8 bytes of padding), then excess-128 codes, K as
//                    [token][dim], V as [dim][cache_slot(token)];  value = (code - 128) * scale
//   tail    [B, Hkv, 2, 2, 64 * D] activation type: block j is at index j & 1; K as [token][dim], V as tail_slot(dim, token)
// One copy of adjacent bytes brings the keys of a block with its scales, one its values; a half of the unfinished block (32 tokens in
// 16 bits) is as many bytes.  In a row of V the tokens that one lane of an m16n8k16 product needs are adjacent: four of every 16.
constexpr int kCacheBlock = 64;
constexpr int kCacheHead = 16;           // bytes before the codes of a record
__host__ __device__ constexpr int cache_slot(int token) {
  return ((token & 7) >> 1) * 16 + (token >> 4) * 4 + ((token >> 3) & 1) * 2 + (token & 1);
}
__host__ __device__ constexpr int tail_slot(int D, int dim, int token) {      // halves of 32 tokens one after the other
  return ((token >> 5) * D + dim) * 32 + ((token & 7) >> 1) * 8 + ((token >> 4) & 1) * 4 + ((token >> 3) & 1) * 2 + (token & 1);
}
__host__ __device__ constexpr int record_bytes(int D) { return kCacheHead + 2 * kCacheBlock * D; }

struct CacheView {
  uint8_t* records;
  void* tail;
  const int* start;      // [B] tokens before this step
  const int* count;      // [B] new tokens of this step
  int B, Hkv, blocks, D;
  bool fp16;             // activation type: fp16 or bf16
};

struct Strided {         // [B, heads, T, D] view with a unit inner stride
  const void* p;
  long long sb, sh, st;
};

// Appends token t < count[b] at position start[b] + t; keys and queries are rotated when `cosv` is given (tables [P, D], P > 0; a
// position behind their end, which only a replayed graph can reach, takes the last row).
// q_out: [B, Hq, T, D] over [B, T, Hq, D] storage; rows t >= count[b] are zeroed.  q.p may be null.
cudaError_t launch_kv_append(const CacheView& c, const Strided& q, int Hq, const Strided& k, const Strided& v, void* q_out, const void* cosv,
                             const void* sinv, int table_rows, int T, cudaStream_t stream);
// k / v [B, Hkv, n, D] fp32: positions first[b] + i; zeros outside [0, start + count).
cudaError_t launch_kv_read(const CacheView& c, const int* first, int n, float* k, float* v, cudaStream_t stream);

struct CachedAttentionArgs {
  CacheView cache;
  Strided q;             // [B, Hq, T, D]
  void* o;               // [B, T, Hq, D] storage
  int Hq, T;
  float scale;
  float* workspace;      // cached_attention_workspace_floats(...) floats; null when that is 0
  int* status;           // raised to STATUS_WAIT_TIMEOUT by a wait that gives up
  cudaStream_t stream;
};
bool cached_attention_fits(int B, int Hkv, int Hq, int T, int D, int blocks);
size_t cached_attention_workspace_floats(int B, int Hkv, int Hq, int T, int D, int blocks);
cudaError_t launch_cached_attention(const CachedAttentionArgs& a);
// How such a call is launched: rows of a tile, CTAs, CTAs of a cluster (0: one list of units for all), and the CTAs that an SM holds at once.
struct CachedAttentionPlan {
  int rows, ctas, cluster, resident;
};
cudaError_t cached_attention_plan(int B, int Hkv, int Hq, int T, int D, int blocks, bool fp16, CachedAttentionPlan* plan);

// ---- mixture of experts for a few tokens ----------------------------------------------------------------------------
constexpr int kMoeTokensMax = 64;
struct MoeTokensArgs {
  const void* x;         // [T, H] bf16, row stride ldx
  long long ldx;
  const void* router;    // [E, H] fp32 or bf16
  bool router_bf16;
  const void* gate_up;   // [E, 2 I, H] bf16
  const void* down;      // [E, H, I] bf16
  void* y;               // [T, H] bf16, contiguous
  void* workspace;       // moe_tokens_workspace_bytes(...), 256-byte aligned
  int* status;           // raised to STATUS_WAIT_TIMEOUT by a wait that gives up
  int T, E, K, H, I;
  bool normalize;
  cudaStream_t stream;
};
size_t moe_tokens_workspace_bytes(int T, int K, int H, int I);
cudaError_t launch_moe_tokens(const MoeTokensArgs& a);

}  // namespace mts
