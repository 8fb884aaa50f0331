// Python bindings of the decoding-step kernels: everything that could become an access out of range is checked here.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "decode.cuh"

namespace {

using torch::Tensor;
namespace py = pybind11;

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

void check_same_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the cache's device");
}

void check_ints(const Tensor& t, int64_t n, const Tensor& like, const char* name) {
  check_same_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() == n, name, " must be contiguous int32 with one entry per sequence");
}

// One layer of a cache, checked once: records [B, Hkv, blocks, 16 + 128 D] bytes, tail [B, Hkv, 2, 2, 64 D], lengths and counts [B].
// The operators answer None for inputs that they do not cover; the caller then takes its plain path, which also words the errors.
struct KvLayer {
  Tensor records, tail, start, count;
  mts::CacheView c;
  int* status;

  KvLayer(Tensor records_, Tensor tail_, Tensor start_, Tensor count_, Tensor status_)
      : records(std::move(records_)), tail(std::move(tail_)), start(std::move(start_)), count(std::move(count_)), status_word_(std::move(status_)) {
    TORCH_CHECK(tail.is_cuda() && tail.dim() == 5 && tail.is_contiguous() && aligned16(tail) && tail.size(2) == 2 && tail.size(3) == 2 &&
                    (tail.scalar_type() == at::kBFloat16 || tail.scalar_type() == at::kHalf) && tail.size(4) % mts::kCacheBlock == 0,
                "cache tail must be contiguous bf16 or fp16 [B, Hkv, 2, 2, 64 * D]");
    const int64_t B = tail.size(0), H = tail.size(1), D = tail.size(4) / mts::kCacheBlock;
    TORCH_CHECK(D == 32 || D == 64 || D == 128, "cache head dimension must be 32, 64 or 128");
    check_same_device(records, tail, "cache records");
    TORCH_CHECK(records.scalar_type() == at::kByte && records.dim() == 4 && records.is_contiguous() && aligned16(records) && records.size(0) == B &&
                    records.size(1) == H && records.size(3) == mts::record_bytes(int(D)), "cache records must be contiguous uint8 [B, Hkv, blocks, 16 + 128 * D]");
    TORCH_CHECK(B > 0 && H > 0 && records.size(2) > 0 && B <= 65535 && H <= 65535 && records.size(2) <= (1 << 24), "unsupported cache extents");
    check_ints(start, B, tail, "lengths");
    check_ints(count, B, tail, "counts");
    check_ints(status_word_, 4, tail, "status");
    c.records = records.data_ptr<uint8_t>(); c.tail = tail.data_ptr();
    c.start = start.data_ptr<int>(); c.count = count.data_ptr<int>();
    c.B = int(B); c.Hkv = int(H); c.blocks = int(records.size(2)); c.D = int(D);
    c.fp16 = tail.scalar_type() == at::kHalf;
    status = status_word_.data_ptr<int>();
  }

  // [B, heads, T, D] rows of the cache's type that can be read 16 bytes at a time, without a gradient to be kept
  bool covers(const Tensor& t, int64_t heads, int64_t T) const {
    if (t.dim() != 4 || t.scalar_type() != tail.scalar_type() || t.device() != tail.device()) return false;
    if (t.size(0) != c.B || t.size(1) != heads || t.size(2) != T || t.size(3) != c.D || t.stride(3) != 1 || !aligned16(t)) return false;
    for (int i = 0; i < 3; ++i)
      if (t.size(i) != 1 && t.stride(i) % 8 != 0) return false;
    return !(t.requires_grad() && at::GradMode::is_enabled());
  }

  // `padded`: tokens of the open step (0: none is open); `reach`: positions that the rotary tables have to hold.  True, or the rotated q.
  py::object append(const Tensor& k, const Tensor& v, const c10::optional<Tensor>& q, const c10::optional<Tensor>& cosv,
                    const c10::optional<Tensor>& sinv, int64_t padded, int64_t reach) const {
    if (padded <= 0 || padded > (1 << 30) || !covers(k, c.Hkv, padded) || !covers(v, c.Hkv, padded)) return py::none();
    const bool rotate = cosv.has_value();
    if (rotate != sinv.has_value()) return py::none();
    if (rotate)
      for (const Tensor* t : {&*cosv, &*sinv})
        if (t->device() != tail.device() || t->scalar_type() != tail.scalar_type() || t->dim() != 2 || t->size(1) != c.D || t->size(0) != cosv->size(0) ||
            t->size(0) < reach || t->size(0) > (1 << 30) || !t->is_contiguous() || !aligned16(*t))
          return py::none();
    int64_t Hq = 0;
    if (q.has_value()) {
      if (q->dim() != 4) return py::none();
      Hq = q->size(1);
      if (Hq <= 0 || Hq > 65535 || Hq % c.Hkv != 0 || !covers(*q, Hq, padded)) return py::none();
    }
    c10::cuda::CUDAGuard guard(tail.device());
    mts::Strided qr{nullptr, 0, 0, 0};
    Tensor out;
    if (q.has_value()) {
      qr = rows_of(*q);
      out = at::empty({c.B, padded, Hq, c.D}, q->options()).transpose(1, 2);
    }
    const cudaError_t e = mts::launch_kv_append(c, qr, int(Hq), rows_of(k), rows_of(v), out.defined() ? out.data_ptr() : nullptr,
                                                rotate ? cosv->data_ptr() : nullptr, rotate ? sinv->data_ptr() : nullptr,
                                                rotate ? int(cosv->size(0)) : 0, int(padded), at::cuda::getCurrentCUDAStream().stream());
    TORCH_CHECK(e == cudaSuccess, "kv_append failed: ", cudaGetErrorString(e));
    if (!out.defined()) return py::bool_(true);
    return py::cast(out);
  }

  py::object read(const Tensor& first, int64_t n) const {
    if (n < 0 || n > (1 << 30) || first.device() != tail.device() || first.scalar_type() != at::kInt || first.dim() != 1 || first.size(0) != c.B ||
        !first.is_contiguous())
      return py::none();
    c10::cuda::CUDAGuard guard(tail.device());
    Tensor k = at::empty({c.B, c.Hkv, n, c.D}, tail.options().dtype(at::kFloat)), v = at::empty_like(k);
    if (n > 0) {
      const cudaError_t e = mts::launch_kv_read(c, first.data_ptr<int>(), int(n), k.data_ptr<float>(), v.data_ptr<float>(),
                                                at::cuda::getCurrentCUDAStream().stream());
      TORCH_CHECK(e == cudaSuccess, "kv_read failed: ", cudaGetErrorString(e));
    }
    return py::make_tuple(k, v);
  }

  py::object attend(const Tensor& q, int64_t padded, double softmax_scale) const {
    if (padded <= 0 || q.dim() != 4) return py::none();
    const int64_t Hq = q.size(1);
    if (Hq <= 0 || Hq % c.Hkv != 0 || Hq / c.Hkv * padded > (1 << 24) || !covers(q, Hq, padded)) return py::none();
    if (!mts::cached_attention_fits(c.B, c.Hkv, int(Hq), int(padded), c.D, c.blocks)) return py::none();
    c10::cuda::CUDAGuard guard(tail.device());
    mts::CachedAttentionArgs a;
    a.cache = c;
    a.Hq = int(Hq); a.T = int(padded);
    a.q = rows_of(q);
    a.scale = float(softmax_scale);
    Tensor o = at::empty({c.B, a.T, Hq, c.D}, q.options()).transpose(1, 2);
    a.o = o.data_ptr();
    const size_t floats = mts::cached_attention_workspace_floats(c.B, c.Hkv, a.Hq, a.T, c.D, c.blocks);
    Tensor ws;
    if (floats > 0) ws = at::empty({int64_t(floats)}, tail.options().dtype(at::kFloat));
    a.workspace = floats > 0 ? ws.data_ptr<float>() : nullptr;
    a.status = status;
    a.stream = at::cuda::getCurrentCUDAStream().stream();
    const cudaError_t e = mts::launch_cached_attention(a);
    TORCH_CHECK(e == cudaSuccess, "cached_attention failed: ", cudaGetErrorString(e));
    return py::cast(o);
  }

 private:
  Tensor status_word_;
  static mts::Strided rows_of(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }
};

// (rows of a tile, CTAs, CTAs of a cluster or 0, CTAs that an SM holds at once) of a call with these extents on the current device
py::tuple cached_attention_plan(int64_t B, int64_t Hkv, int64_t Hq, int64_t T, int64_t D, int64_t blocks, bool fp16) {
  TORCH_CHECK(B > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && T > 0 && blocks > 0 && (D == 32 || D == 64 || D == 128), "unsupported extents");
  TORCH_CHECK(B <= 65535 && Hkv <= 65535 && blocks <= (1 << 24) && T <= (1 << 24) && Hq / Hkv * T <= (1 << 24) &&
                  mts::cached_attention_fits(int(B), int(Hkv), int(Hq), int(T), int(D), int(blocks)), "unsupported extents");
  mts::CachedAttentionPlan plan{};
  const cudaError_t e = mts::cached_attention_plan(int(B), int(Hkv), int(Hq), int(T), int(D), int(blocks), fp16, &plan);
  TORCH_CHECK(e == cudaSuccess, "cached_attention_plan failed: ", cudaGetErrorString(e));
  return py::make_tuple(plan.rows, plan.ctas, plan.cluster, plan.resident);
}

// What the kernels cover of a layer with experts of width I, its weights aside.
bool moe_tokens_fits(const Tensor& x, const Tensor& router, int64_t I, int64_t top_k) {
  if (!x.is_cuda() || x.scalar_type() != at::kBFloat16 || x.dim() != 2 || router.dim() != 2) return false;
  const int64_t T = x.size(0), H = x.size(1), E = router.size(0);
  if (T > mts::kMoeTokensMax || H <= 0 || H % 8 != 0 || H > (1 << 20) || x.stride(1) != 1 || !aligned16(x) || (T > 1 && x.stride(0) % 8 != 0)) return false;
  if (E < 1 || E > 64 || top_k < 1 || top_k > 8 || top_k > E || I <= 0 || I % 8 != 0 || I > (1 << 20)) return false;
  return router.size(1) == H && (router.scalar_type() == at::kFloat || router.scalar_type() == at::kBFloat16) && router.device() == x.device() &&
         router.is_contiguous() && aligned16(router);
}

// None for inputs that the kernels do not cover.
py::object moe_tokens(const Tensor& x, const Tensor& router, const Tensor& gate_up, const Tensor& down, int64_t top_k, bool normalize,
                      const Tensor& status) {
  if (gate_up.dim() != 3 || down.dim() != 3 || !moe_tokens_fits(x, router, down.size(2), top_k)) return py::none();
  const int64_t T = x.size(0), H = x.size(1), E = router.size(0), I = down.size(2);
  if (gate_up.size(0) != E || gate_up.size(1) != 2 * I || gate_up.size(2) != H || down.size(0) != E || down.size(1) != H) return py::none();
  if (gate_up.scalar_type() != at::kBFloat16 || down.scalar_type() != at::kBFloat16) return py::none();
  for (const Tensor* w : {&gate_up, &down})
    if (w->device() != x.device() || !w->is_contiguous() || !aligned16(*w)) return py::none();
  if (at::GradMode::is_enabled() && (x.requires_grad() || router.requires_grad() || gate_up.requires_grad() || down.requires_grad())) return py::none();
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty({T, H}, x.options());
  if (T == 0) return py::cast(y);
  check_ints(status, 4, x, "status");
  Tensor ws = at::empty({int64_t(mts::moe_tokens_workspace_bytes(int(T), int(top_k), int(H), int(I)))}, x.options().dtype(at::kByte));
  mts::MoeTokensArgs a;
  a.x = x.data_ptr(); a.ldx = x.stride(0);
  a.router = router.data_ptr(); a.router_bf16 = router.scalar_type() == at::kBFloat16;
  a.gate_up = gate_up.data_ptr(); a.down = down.data_ptr(); a.y = y.data_ptr();
  a.workspace = ws.data_ptr(); a.status = status.data_ptr<int>();
  a.T = int(T); a.E = int(E); a.K = int(top_k); a.H = int(H); a.I = int(I);
  a.normalize = normalize;
  a.stream = at::cuda::getCurrentCUDAStream().stream();
  const cudaError_t e = mts::launch_moe_tokens(a);
  TORCH_CHECK(e == cudaSuccess, "moe_tokens failed: ", cudaGetErrorString(e));
  return py::cast(y);
}

}  // namespace

void bind_decode(pybind11::module_& m) {
  py::class_<KvLayer>(m, "KvLayer")
      .def(py::init<Tensor, Tensor, Tensor, Tensor, Tensor>())
      .def("append", &KvLayer::append)
      .def("read", &KvLayer::read)
      .def("attend", &KvLayer::attend);
  m.def("cached_attention_plan", &cached_attention_plan);
  m.def("moe_tokens", &moe_tokens);
  m.def("moe_tokens_fits", &moe_tokens_fits);
}
