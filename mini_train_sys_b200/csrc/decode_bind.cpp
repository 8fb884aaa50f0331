// Python bindings of the decoding-step kernels: everything that could become an access out of range is checked here.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "decode.cuh"

namespace {

using torch::Tensor;

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

void check_same_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the cache's device");
}

void check_ints(const Tensor& t, int64_t n, const Tensor& like, const char* name) {
  check_same_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() == n, name, " must be contiguous int32 with one entry per sequence");
}

// codes [B, Hkv, blocks, 2, 64 * D], scale [B, Hkv, blocks, 2], tail [B, Hkv, 2, 2, 64 * D]
mts::CacheView cache_view(const Tensor& codes, const Tensor& scale, const Tensor& tail, const Tensor& start, const Tensor& count) {
  TORCH_CHECK(codes.is_cuda() && codes.dim() == 5 && codes.scalar_type() == at::kByte && codes.is_contiguous() && aligned16(codes) &&
                  codes.size(3) == 2 && codes.size(4) % mts::kCacheBlock == 0, "cache codes must be contiguous uint8 [B, Hkv, blocks, 2, 64 * D]");
  const int64_t B = codes.size(0), H = codes.size(1), N = codes.size(2), D = codes.size(4) / mts::kCacheBlock;
  TORCH_CHECK(D == 32 || D == 64 || D == 128, "cache head dimension must be 32, 64 or 128");
  TORCH_CHECK(B > 0 && H > 0 && N > 0 && B <= 65535 && H <= 65535 && N <= (1 << 24), "unsupported cache extents");
  check_same_device(scale, codes, "cache scale");
  TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.is_contiguous() && scale.dim() == 4 && scale.size(0) == B && scale.size(1) == H &&
                  scale.size(2) == N && scale.size(3) == 2 && aligned16(scale), "cache scale must be contiguous fp32 [B, Hkv, blocks, 2]");
  check_same_device(tail, codes, "cache tail");
  TORCH_CHECK((tail.scalar_type() == at::kBFloat16 || tail.scalar_type() == at::kHalf) && tail.is_contiguous() && aligned16(tail) &&
                  tail.dim() == 5 && tail.size(0) == B && tail.size(1) == H && tail.size(2) == 2 && tail.size(3) == 2 &&
                  tail.size(4) == mts::kCacheBlock * D, "cache tail must be contiguous bf16 or fp16 [B, Hkv, 2, 2, 64 * D]");
  check_ints(start, B, codes, "start");
  check_ints(count, B, codes, "count");
  mts::CacheView c;
  c.codes = codes.data_ptr<uint8_t>(); c.scale = scale.data_ptr<float>(); c.tail = tail.data_ptr();
  c.start = start.data_ptr<int>(); c.count = count.data_ptr<int>();
  c.B = int(B); c.Hkv = int(H); c.blocks = int(N); c.D = int(D);
  c.fp16 = tail.scalar_type() == at::kHalf;
  return c;
}

mts::Strided rows_of(const Tensor& t, const Tensor& tail, int64_t B, int64_t H, int64_t T, int64_t D, const char* name) {
  check_same_device(t, tail, name);
  TORCH_CHECK(t.scalar_type() == tail.scalar_type(), name, " must have the cache's activation type");
  TORCH_CHECK(t.dim() == 4 && t.size(0) == B && t.size(1) == H && t.size(2) == T && t.size(3) == D, name, " must be [B, heads, T, D]");
  TORCH_CHECK(t.stride(3) == 1 && aligned16(t), name, " must have a contiguous, 16-byte aligned last dimension");
  for (int i = 0; i < 3; ++i)
    TORCH_CHECK(t.size(i) == 1 || t.stride(i) % 8 == 0, name, " rows must be 16-byte aligned");
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

c10::optional<Tensor> kv_append(Tensor codes, Tensor scale, Tensor tail, const Tensor& start, const Tensor& count, const Tensor& k, const Tensor& v,
                                const c10::optional<Tensor>& q, const c10::optional<Tensor>& cosv, const c10::optional<Tensor>& sinv) {
  const mts::CacheView c = cache_view(codes, scale, tail, start, count);
  TORCH_CHECK(k.dim() == 4 && k.size(2) > 0 && k.size(2) <= (1 << 30), "k must be [B, heads, T, D] with at least one token");
  const int64_t T = k.size(2);
  const mts::Strided kr = rows_of(k, tail, c.B, c.Hkv, T, c.D, "k"), vr = rows_of(v, tail, c.B, c.Hkv, T, c.D, "v");
  const bool rotate = cosv.has_value() && cosv->defined();
  TORCH_CHECK(rotate == (sinv.has_value() && sinv->defined()), "cos and sin come together");
  if (rotate)
    for (const Tensor* t : {&*cosv, &*sinv}) {
      check_same_device(*t, codes, "rotary table");
      TORCH_CHECK(t->scalar_type() == tail.scalar_type() && t->dim() == 2 && t->size(1) == c.D && t->size(0) == cosv->size(0) &&
                      t->size(0) <= (1 << 30) && t->is_contiguous() && aligned16(*t), "rotary tables must be contiguous [positions, D] in the activation type");
    }
  c10::cuda::CUDAGuard guard(codes.device());
  mts::Strided qr{nullptr, 0, 0, 0};
  Tensor out;
  int64_t Hq = 0;
  if (q.has_value() && q->defined()) {
    TORCH_CHECK(q->dim() == 4 && q->size(1) > 0 && q->size(1) <= 65535, "q must be [B, heads, T, D]");
    Hq = q->size(1);
    qr = rows_of(*q, tail, c.B, Hq, T, c.D, "q");
    out = torch::empty({c.B, T, Hq, c.D}, q->options()).transpose(1, 2);
  }
  const cudaError_t e = mts::launch_kv_append(c, qr, int(Hq), kr, vr, out.defined() ? out.data_ptr() : nullptr, rotate ? cosv->data_ptr() : nullptr,
                                              rotate ? sinv->data_ptr() : nullptr, rotate ? int(cosv->size(0)) : 0, int(T),
                                              at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(e == cudaSuccess, "kv_append failed: ", cudaGetErrorString(e));
  if (!out.defined()) return c10::nullopt;
  return out;
}

std::vector<Tensor> kv_read(const Tensor& codes, const Tensor& scale, const Tensor& tail, const Tensor& start, const Tensor& count,
                            const Tensor& first, int64_t n) {
  const mts::CacheView c = cache_view(codes, scale, tail, start, count);
  check_ints(first, c.B, codes, "first");
  TORCH_CHECK(n >= 0 && n <= (1 << 30), "the number of positions must not be negative");
  c10::cuda::CUDAGuard guard(codes.device());
  Tensor k = torch::empty({c.B, c.Hkv, n, c.D}, codes.options().dtype(torch::kFloat)), v = torch::empty_like(k);
  if (n > 0) {
    const cudaError_t e = mts::launch_kv_read(c, first.data_ptr<int>(), int(n), k.data_ptr<float>(), v.data_ptr<float>(),
                                              at::cuda::getCurrentCUDAStream().stream());
    TORCH_CHECK(e == cudaSuccess, "kv_read failed: ", cudaGetErrorString(e));
  }
  return {k, v};
}

Tensor cached_attention(const Tensor& codes, const Tensor& scale, const Tensor& tail, const Tensor& start, const Tensor& count, const Tensor& q,
                        double softmax_scale) {
  mts::CachedAttentionArgs a;
  a.cache = cache_view(codes, scale, tail, start, count);
  TORCH_CHECK(q.dim() == 4 && q.size(1) > 0 && q.size(1) % a.cache.Hkv == 0 && q.size(2) > 0, "q must be [B, heads, T, D] with a multiple of the cache's heads");
  TORCH_CHECK(q.size(1) / a.cache.Hkv * q.size(2) <= (1 << 24), "too many query rows");
  a.Hq = int(q.size(1)); a.T = int(q.size(2));
  a.q = rows_of(q, tail, a.cache.B, a.Hq, a.T, a.cache.D, "q");
  a.scale = float(softmax_scale);
  c10::cuda::CUDAGuard guard(codes.device());
  Tensor o = torch::empty({a.cache.B, a.T, a.Hq, a.cache.D}, q.options()).transpose(1, 2);
  a.o = o.data_ptr();
  const size_t floats = mts::cached_attention_workspace_floats(a.cache.B, a.cache.Hkv, a.Hq, a.T, a.cache.D, a.cache.blocks);
  Tensor ws;
  if (floats > 0) ws = torch::empty({int64_t(floats)}, codes.options().dtype(torch::kFloat));
  a.workspace = floats > 0 ? ws.data_ptr<float>() : nullptr;
  a.stream = at::cuda::getCurrentCUDAStream().stream();
  const cudaError_t e = mts::launch_cached_attention(a);
  TORCH_CHECK(e == cudaSuccess, "cached_attention failed: ", cudaGetErrorString(e));
  return o;
}

Tensor moe_tokens(const Tensor& x, const Tensor& router, const Tensor& gate_up, const Tensor& down, int64_t top_k, bool normalize) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() == 2 && x.stride(1) == 1 && aligned16(x) &&
                  (x.size(0) == 1 || x.stride(0) % 8 == 0), "x must be bf16 [T, H] with 16-byte aligned rows");
  const int64_t T = x.size(0), H = x.size(1), E = router.size(0);
  TORCH_CHECK(T <= mts::kMoeTokensMax && H > 0 && H % 8 == 0 && H <= (1 << 20), "moe_tokens takes up to 64 tokens and a hidden size that is a multiple of 8");
  check_same_device(router, x, "router weight");
  TORCH_CHECK(router.dim() == 2 && router.size(1) == H && router.is_contiguous() && aligned16(router) &&
                  (router.scalar_type() == at::kFloat || router.scalar_type() == at::kBFloat16), "router weight must be contiguous fp32 or bf16 [E, H]");
  TORCH_CHECK(E >= 1 && E <= 64 && top_k >= 1 && top_k <= 8 && top_k <= E, "moe_tokens takes up to 64 experts and top-8");
  for (const Tensor* w : {&gate_up, &down}) {
    check_same_device(*w, x, "expert weight");
    TORCH_CHECK(w->scalar_type() == at::kBFloat16 && w->is_contiguous() && aligned16(*w) && w->dim() == 3 && w->size(0) == E, "expert weights must be contiguous bf16 [E, ., .]");
  }
  const int64_t I = down.size(2);
  TORCH_CHECK(I > 0 && I % 8 == 0 && I <= (1 << 20) && down.size(1) == H && gate_up.size(1) == 2 * I && gate_up.size(2) == H,
              "expert weights must be [E, 2 I, H] and [E, H, I] with I a multiple of 8");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = torch::empty({T, H}, x.options());
  if (T == 0) return y;
  Tensor hidden = torch::empty({2, T * top_k, I}, x.options()), routes = torch::empty({T * top_k}, x.options().dtype(torch::kInt));
  mts::MoeTokensArgs a;
  a.x = x.data_ptr(); a.ldx = x.stride(0);
  a.router = router.data_ptr(); a.router_bf16 = router.scalar_type() == at::kBFloat16;
  a.gate_up = gate_up.data_ptr(); a.down = down.data_ptr(); a.y = y.data_ptr();
  a.hidden = hidden.data_ptr(); a.routes = routes.data_ptr<int>();
  a.T = int(T); a.E = int(E); a.K = int(top_k); a.H = int(H); a.I = int(I);
  a.normalize = normalize;
  a.stream = at::cuda::getCurrentCUDAStream().stream();
  const cudaError_t e = mts::launch_moe_tokens(a);
  TORCH_CHECK(e == cudaSuccess, "moe_tokens failed: ", cudaGetErrorString(e));
  return y;
}

}  // namespace

void bind_decode(pybind11::module_& m) {
  m.def("kv_append", &kv_append);
  m.def("kv_read", &kv_read);
  m.def("cached_attention", &cached_attention);
  m.def("moe_tokens", &moe_tokens);
}
