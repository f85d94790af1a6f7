// Python binding of the serving operators (include/popcorn_serve.h): checks of
// tensors, allocation of outputs and workspaces and the current stream, in
// front of the C entry points of libpopcorn.so. popcorn_b200/__init__.py holds
// the documented functions and calls these with positional arguments. It
// exists for its speed: the same checks through ctypes and tensor attributes
// take 10 to 14 us a call, several times the kernels of a small decode step.
//
// With a stream given the whole call is as inside torch.cuda.stream(...): what
// it allocates belongs to that stream.
//
// Argument errors raise ValueError; the entry point's status is returned. A call
// without work ends here once its arguments are checked: tensors without elements
// have null pointers, which the entry points refuse.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>

#include "popcorn_serve.h"

namespace {

using Tensor = at::Tensor;
using Optional = std::optional<Tensor>;

std::string form(at::ScalarType type, at::IntArrayRef shape, const at::Device& device) {
    std::string s = std::string(at::toString(type)) + " [";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + "] on " + device.str();
}

[[noreturn]] void refuse(const char* where, const char* name, const std::string& wanted, const Tensor* got) {
    std::string s = std::string(where) + ": " + name + ": " + wanted;
    if (got != nullptr) s += " wanted, got " + form(got->scalar_type(), got->sizes(), got->device());
    throw std::invalid_argument(s);  // ValueError
}

struct Call {
    const char* where;
    at::Device device;

    bool placed(const Tensor& t, at::ScalarType type, std::initializer_list<int64_t> shape) const {
        return t.scalar_type() == type && t.sizes() == at::IntArrayRef(shape) && t.device() == device;
    }
    void* contiguous(const Tensor& t, at::ScalarType type, std::initializer_list<int64_t> shape,
                     const char* name) const {
        if (!placed(t, type, shape) || !t.is_contiguous()) refuse(where, name, "contiguous " + form(type, shape, device), &t);
        return t.data_ptr();
    }
    const int32_t* whole(const Tensor& t, std::initializer_list<int64_t> shape, const char* name) const {
        return static_cast<const int32_t*>(contiguous(t, at::kInt, shape, name));
    }
    // [tokens, heads, dim], the last dimension contiguous.
    void* rows(const Tensor& t, at::ScalarType type, std::initializer_list<int64_t> shape, const char* name) const {
        if (!placed(t, type, shape)) refuse(where, name, form(type, shape, device), &t);
        if (t.stride(2) != 1) refuse(where, name, "the last dimension must be contiguous", nullptr);
        return t.data_ptr();
    }
    popcornType_t type(at::ScalarType t) const {
        switch (t) {
            case at::kFloat: return POPCORN_TYPE_F32;
            case at::kHalf: return POPCORN_TYPE_F16;
            case at::kBFloat16: return POPCORN_TYPE_BF16;
            default: refuse(where, "dtype", "float32, float16 or bfloat16 wanted", nullptr);
        }
    }
};

// The stream of a call: the current one, or the caller's, which is then the
// current one until the call returns. Outputs and workspaces come from the
// allocator's blocks of the stream that the kernels run on: a block of another
// stream may still be in use by that stream's earlier work, and the workspace,
// released on return, would go to that stream's next tensor while the kernels
// run. Outputs are recorded on the stream that was current before, where the
// caller goes on with them: a block released there is not written again before
// that stream's work on it has ended.
class OnStream {
  public:
    OnStream(const Call& c, const std::optional<int64_t>& given)
        : before_(c10::cuda::getCurrentCUDAStream(c.device.index())), handle_(before_.stream()) {
        if (!given) return;
        handle_ = reinterpret_cast<cudaStream_t>(*given);
        if (handle_ == before_.stream()) return;
        const bool legacy = handle_ == nullptr || handle_ == cudaStreamLegacy;
        guard_.emplace(legacy ? c10::cuda::getDefaultCUDAStream(c.device.index())
                              : c10::cuda::getStreamFromExternal(handle_, c.device.index()));
    }
    cudaStream_t handle() const { return handle_; }
    Tensor output(at::IntArrayRef shape, const at::TensorOptions& options) const {
        Tensor t = at::empty(shape, options);
        if (guard_) t.record_stream(before_.unwrap());
        return t;
    }

  private:
    c10::cuda::CUDAStream before_;
    cudaStream_t handle_;
    std::optional<c10::cuda::CUDAStreamGuard> guard_;
};

Call on_cache(const char* where, int64_t device) {
    return {where, at::Device(at::kCUDA, static_cast<at::DeviceIndex>(device))};
}

const popcornKvCache_t& cache_at(int64_t ref) { return *reinterpret_cast<const popcornKvCache_t*>(ref); }

void three(const Call& c, const Tensor& t, const char* name) {
    if (t.dim() != 3) refuse(c.where, name, "[tokens, heads, dim]", &t);
}

// Sequences of a block table and their runs of tokens.
struct Batch {
    int64_t seqs, width;
    const int32_t *table, *first;
};
Batch batch(const Call& c, const Tensor& table, const Optional& first, int64_t tokens) {
    if (table.dim() != 2) refuse(c.where, "table", "[seqs, pages]", &table);
    const int64_t seqs = table.size(0), width = table.size(1);
    Batch b = {seqs, width, c.whole(table, {seqs, width}, "table"), nullptr};
    if (first) b.first = c.whole(*first, {seqs + 1}, "first");
    else if (tokens != seqs) refuse(c.where, "first", "more or fewer tokens than sequences need `first`", nullptr);
    return b;
}

Tensor bytes_on(at::Device device, int64_t n) { return at::empty({n}, at::TensorOptions().dtype(at::kChar).device(device)); }

py::tuple kv_append(int64_t ref, int64_t device, const Tensor& k, const Tensor& v, const Tensor& table,
                    const Tensor& start, const Optional& first, const Optional& q, const Optional& cos,
                    const Optional& sin, bool interleaved, Optional q_out, std::optional<int64_t> stream) {
    const Call c = on_cache("kv_append", device);
    const c10::cuda::CUDAGuard guard(c.device);
    const OnStream on(c, stream);
    const popcornKvCache_t& cache = cache_at(ref);
    three(c, k, "k");
    const int64_t tokens = k.size(0);
    const at::ScalarType kind = k.scalar_type();
    const popcornType_t type = c.type(kind);
    const void* kp = c.rows(k, kind, {tokens, cache.heads, cache.dim}, "k");
    const void* vp = c.rows(v, kind, {tokens, cache.heads, cache.dim}, "v");
    const Batch b = batch(c, table, first, tokens);
    const int32_t* sp = c.whole(start, {b.seqs}, "start");
    const void* qp = nullptr;
    void* op = nullptr;
    int64_t q_heads = 0, qt = 0, qh = 0;
    if (q) {
        three(c, *q, "q");
        q_heads = q->size(1);
        qp = c.rows(*q, kind, {tokens, q_heads, cache.dim}, "q");
        qt = q->stride(0), qh = q->stride(1);
        if (!q_out) q_out = on.output({tokens, q_heads, cache.dim}, q->options());
        op = c.contiguous(*q_out, kind, {tokens, q_heads, cache.dim}, "q_out");
    } else if (q_out) {
        refuse(c.where, "q_out", "q_out needs q", nullptr);
    }
    const float *cp = nullptr, *np = nullptr;
    int64_t positions = 0, half = 0;
    if (cos.has_value() != sin.has_value()) refuse(c.where, "cos", "cos and sin come together", nullptr);
    if (cos) {
        if (cos->dim() != 2) refuse(c.where, "cos", "[positions, rot_dim / 2]", &*cos);
        positions = cos->size(0), half = cos->size(1);
        cp = static_cast<const float*>(c.contiguous(*cos, at::kFloat, {positions, half}, "cos"));
        np = static_cast<const float*>(c.contiguous(*sin, at::kFloat, {positions, half}, "sin"));
    }
    if (tokens == 0 || b.seqs == 0) return py::make_tuple(static_cast<int>(POPCORN_SUCCESS), q_out);
    const int status = popcornKvAppend(&cache, kp, k.stride(0), k.stride(1), vp, v.stride(0), v.stride(1), type, b.table,
                                       b.width, b.first, sp, b.seqs, tokens, op, qp, qt, qh, q_heads, cp, np, positions,
                                       2 * half, interleaved, on.handle());
    return py::make_tuple(status, q_out);
}

py::tuple kv_read(int64_t ref, int64_t device, const Tensor& pages, int type, Optional k_out, Optional v_out,
                  std::optional<int64_t> stream) {
    const Call c = on_cache("kv_read", device);
    const c10::cuda::CUDAGuard guard(c.device);
    const OnStream on(c, stream);
    const popcornKvCache_t& cache = cache_at(ref);
    if (pages.dim() != 1) refuse(c.where, "pages", "[n]", &pages);
    const int64_t n = pages.size(0);
    const at::ScalarType kind = type == POPCORN_TYPE_F32 ? at::kFloat : type == POPCORN_TYPE_F16 ? at::kHalf : at::kBFloat16;
    const int32_t* list = c.whole(pages, {n}, "pages");
    const auto options = at::TensorOptions().dtype(kind).device(c.device);
    if (!k_out) k_out = on.output({n, cache.heads, cache.page_size, cache.dim}, options);
    if (!v_out) v_out = on.output({n, cache.heads, cache.page_size, cache.dim}, options);
    void* kp = c.contiguous(*k_out, kind, {n, cache.heads, cache.page_size, cache.dim}, "k_out");
    void* vp = c.contiguous(*v_out, kind, {n, cache.heads, cache.page_size, cache.dim}, "v_out");
    if (n == 0) return py::make_tuple(static_cast<int>(POPCORN_SUCCESS), k_out, v_out);
    const int status = popcornKvRead(kp, vp, static_cast<popcornType_t>(type), &cache, list, n, on.handle());
    return py::make_tuple(status, k_out, v_out);
}

py::tuple kv_attention(int64_t ref, int64_t device, const Tensor& q, const Tensor& table, const Tensor& length,
                       const Optional& first, std::optional<int64_t> max_tokens, bool causal, int64_t window,
                       std::optional<double> scale, Optional out, const Optional& lse, std::optional<int64_t> stream) {
    const Call c = on_cache("kv_attention", device);
    const c10::cuda::CUDAGuard guard(c.device);
    const OnStream on(c, stream);
    const popcornKvCache_t& cache = cache_at(ref);
    three(c, q, "q");
    const int64_t tokens = q.size(0), q_heads = q.size(1);
    const at::ScalarType kind = q.scalar_type();
    const popcornType_t type = c.type(kind);
    const void* qp = c.rows(q, kind, {tokens, q_heads, cache.dim}, "q");
    if (q_heads % cache.heads != 0) refuse(c.where, "q", "a multiple of the cache's heads", &q);
    const Batch b = batch(c, table, first, tokens);
    const int32_t* lp = c.whole(length, {b.seqs}, "length");
    if (!out) out = on.output({tokens, q_heads, cache.dim}, q.options());
    void* op = c.contiguous(*out, kind, {tokens, q_heads, cache.dim}, "out");
    float* ep = lse ? static_cast<float*>(c.contiguous(*lse, at::kFloat, {tokens, q_heads}, "lse")) : nullptr;
    if (tokens == 0 || b.seqs == 0) return py::make_tuple(static_cast<int>(POPCORN_SUCCESS), out);
    const int64_t most = max_tokens ? *max_tokens : b.first == nullptr ? 1 : tokens;
    const int64_t need = popcornKvAttentionWorkspace(&cache, type, b.seqs, tokens, most, q_heads);
    Tensor ws;
    if (need > 0) ws = bytes_on(c.device, need);
    const float by = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(cache.dim)));
    const int status = popcornKvAttention(op, ep, qp, q.stride(0), q.stride(1), type, &cache, b.table, b.width, b.first,
                                          lp, b.seqs, tokens, most, q_heads, causal, window, by,
                                          need > 0 ? ws.data_ptr() : nullptr, need, on.handle());
    return py::make_tuple(status, out);
}

py::tuple moe(const Tensor& x, const Tensor& router, const Tensor& q_gate, const Tensor& s_gate, const Tensor& q_up,
              const Tensor& s_up, const Tensor& q_down, const Tensor& s_down, int64_t top_k, bool renormalize,
              Optional out, bool routing, std::optional<int64_t> stream) {
    const Call c = {"moe", x.device()};
    if (!x.is_cuda() || x.dim() != 2) refuse(c.where, "x", "a CUDA tensor [M, K]", &x);
    const c10::cuda::CUDAGuard guard(c.device);
    const OnStream on(c, stream);
    if (s_gate.dim() != 2) refuse(c.where, "s_gate", "[E, F]", &s_gate);
    const int64_t M = x.size(0), K = x.size(1), E = s_gate.size(0), F = s_gate.size(1);
    const auto floats = [&](const Tensor& t, std::initializer_list<int64_t> shape, const char* name) {
        return static_cast<float*>(c.contiguous(t, at::kFloat, shape, name));
    };
    const auto codes = [&](const Tensor& t, std::initializer_list<int64_t> shape, const char* name) {
        return static_cast<const int8_t*>(c.contiguous(t, at::kChar, shape, name));
    };
    const float *xp = floats(x, {M, K}, "x"), *rp = floats(router, {E, K}, "router");
    const int8_t* gp = codes(q_gate, {E, F, K}, "q_gate");
    const float* gs = floats(s_gate, {E, F}, "s_gate");
    const int8_t* up = codes(q_up, {E, F, K}, "q_up");
    const float* us = floats(s_up, {E, F}, "s_up");
    const int8_t* dp = codes(q_down, {E, K, F}, "q_down");
    const float* ds = floats(s_down, {E, K}, "s_down");
    if (!out) out = on.output({M, K}, x.options());
    float* op = floats(*out, {M, K}, "out");
    Optional experts, weights;
    if (routing) {
        if (top_k < 0) refuse(c.where, "top_k", "a positive number wanted", nullptr);
        experts = on.output({M, top_k}, x.options().dtype(at::kInt));
        weights = on.output({M, top_k}, x.options());
    }
    if (M == 0) return py::make_tuple(static_cast<int>(POPCORN_SUCCESS), out, experts, weights);
    const int64_t need = popcornMoeWorkspace(M, K, F, E, top_k);
    Tensor ws;
    if (need > 0) ws = bytes_on(c.device, need);
    const int status = popcornMoe_i8f32(op, routing ? experts->data_ptr<int32_t>() : nullptr,
                                        routing ? weights->data_ptr<float>() : nullptr, xp, rp, gp, gs, up, us, dp, ds,
                                        M, K, F, E, top_k, renormalize, need > 0 ? ws.data_ptr() : nullptr, need,
                                        on.handle());
    return py::make_tuple(status, out, experts, weights);
}

}  // namespace

PYBIND11_MODULE(_serve, m) {
    m.def("kv_append", &kv_append);
    m.def("kv_read", &kv_read);
    m.def("kv_attention", &kv_attention);
    m.def("moe", &moe);
}
