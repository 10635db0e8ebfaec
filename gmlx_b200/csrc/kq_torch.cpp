// kq_torch.cpp -- native fast path of the decode-time kq ops for torch tensors
// (the projections and the operators of the serving step around them).
//
// kq.quantized_matmul / kq.quantized_glu are called once per projection per
// token; going through Python argument handling and ctypes costs ~15-20 us a
// call on the host, more than a decode GEMV takes on the GPU, so an eager
// decode loop would be host-bound.  This extension does the same work -- shape
// and layout checks, output allocation, the per-(device, stream) workspace,
// the libkq_cuda C-ABI call on torch's current stream -- in one native call.
//
// It only takes the common well-formed case (2-D wire weights with whole
// 256-weight groups, bf16/f16 activations whose rows are 16-byte aligned);
// for anything else, or when the C call reports an error, it returns None and
// the Python op runs its full path, which raises the reference's exception
// types.  The C entry points come in as addresses of the already-loaded
// libkq_cuda.so (set_entry_points), so this module has no link-time
// dependency on it.  The workspace registry here is the one the Python layer
// uses too (workspace()), so kq.workspace_error() sees every call's error word.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cstdint>
#include <map>
#include <mutex>
#include <tuple>
#include <vector>

#include "../../include/kq_cuda.h"

namespace {

using MatmulFn = int (*)(int, const void *, int, int64_t, int64_t, int64_t, const void *, int64_t, int64_t, void *,
                         int, int64_t, void *, size_t, void *);
using GluFn = int (*)(int, const void *, int, int64_t, int64_t, int64_t, const void *, const void *, int64_t, int64_t,
                      int, void *, int, int64_t, void *, size_t, void *);
using WsFn = size_t (*)(int, int64_t, int64_t, int64_t);

MatmulFn g_matmul = nullptr;
GluFn g_glu = nullptr;
WsFn g_matmul_ws = nullptr, g_glu_ws = nullptr;

std::mutex g_mu;
struct Workspace {
    at::Tensor now;
    bool captured = false;         // a graph was captured with `now`
    std::vector<at::Tensor> kept;  // workspaces outgrown since that graphs write to, or that a capture outgrew
};
std::map<std::pair<int, int64_t>, Workspace> g_ws;                     // (device, stream) -> workspace
std::map<std::tuple<int, int, int64_t, int64_t, int64_t>, size_t> g_ws_bytes;  // (op, codec, m, n, k) -> bytes

int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1;
}

void set_entry_points(int64_t matmul, int64_t glu, int64_t matmul_ws, int64_t glu_ws) {
    g_matmul = reinterpret_cast<MatmulFn>(matmul);
    g_glu = reinterpret_cast<GluFn>(glu);
    g_matmul_ws = reinterpret_cast<WsFn>(matmul_ws);
    g_glu_ws = reinterpret_cast<WsFn>(glu_ws);
}

bool capturing(cudaStream_t s) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &cap) == cudaSuccess) return cap != cudaStreamCaptureStatusNone;
    (void)cudaGetLastError();  // the default stream beside a capture: the call itself will say so
    return false;
}

// A new workspace.  Made in a capture it is allocated and zeroed outside of it, or every
// replay would zero it again.
at::Tensor zeroed(int device, int64_t sz, bool in_capture) {
    const auto opt = at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device);
    if (!in_capture) return at::zeros({sz}, opt);
    c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    c10::cuda::CUDAStream side = c10::cuda::getStreamFromPool(false, (c10::DeviceIndex)device);
    for (int i = 0; i < 64 && capturing(side.stream()); i++) side = c10::cuda::getStreamFromPool(false, (c10::DeviceIndex)device);
    c10::cuda::CUDAStreamGuard guard(side);
    at::Tensor t = at::zeros({sz}, opt);
    side.synchronize();
    return t;
}

// The zero-filled workspace of (device, stream), grown to at least nbytes
// (at least 1 MiB); the library leaves every workspace zero after each call but
// for the error word in front, which goes along when it grows.  A workspace that
// a graph was captured with stays for the graph's replays.
at::Tensor workspace(int64_t device, int64_t stream, int64_t nbytes) {
    std::lock_guard<std::mutex> lk(g_mu);
    auto key = std::make_pair((int)device, stream);
    Workspace &w = g_ws[key];
    if (!w.now.defined() || w.now.numel() < nbytes) {
        const int64_t sz = nbytes > (1 << 20) ? nbytes : (1 << 20);
        const bool in_capture = capturing(reinterpret_cast<cudaStream_t>(stream));
        at::Tensor t = zeroed((int)device, sz, in_capture);
        if (w.now.defined()) {
            if (!in_capture) t.narrow(0, 0, 4).copy_(w.now.narrow(0, 0, 4), true);
            if (in_capture || w.captured) w.kept.push_back(w.now);
        }
        w.now = t, w.captured = in_capture;
    } else if (!w.captured)
        w.captured = capturing(reinterpret_cast<cudaStream_t>(stream));
    return w.now;
}

// The existing workspace of (device, stream), or an undefined tensor.
at::Tensor workspace_peek(int64_t device, int64_t stream) {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_ws.find(std::make_pair((int)device, stream));
    return it == g_ws.end() ? at::Tensor() : it->second.now;
}

// All workspaces of (device, stream) that a call or a graph may still write to.
std::vector<at::Tensor> workspaces(int64_t device, int64_t stream) {
    std::lock_guard<std::mutex> lk(g_mu);
    std::vector<at::Tensor> all;
    auto it = g_ws.find(std::make_pair((int)device, stream));
    if (it == g_ws.end()) return all;
    if (it->second.now.defined()) all.push_back(it->second.now);
    all.insert(all.end(), it->second.kept.begin(), it->second.kept.end());
    return all;
}

size_t ws_bytes(int op, int codec, int64_t m, int64_t n, int64_t k) {
    const auto key = std::make_tuple(op, codec, m, n, k);
    {
        std::lock_guard<std::mutex> lk(g_mu);
        auto it = g_ws_bytes.find(key);
        if (it != g_ws_bytes.end()) return it->second;
    }
    const size_t v = op == 0 ? g_matmul_ws(codec, m, n, k) : g_glu_ws(codec, m, n, k);
    std::lock_guard<std::mutex> lk(g_mu);
    g_ws_bytes[key] = v;
    return v;
}

// The checks both ops share; false sends the call down the Python path.
bool common(const at::Tensor &x, const at::Tensor &w, int64_t bpb, int64_t &k, int64_t &wstride) {
    if (!x.is_cuda() || !w.is_cuda() || w.scalar_type() != at::kByte || w.dim() != 2 || x.dim() < 1) return false;
    if (dtype_code(x.scalar_type()) < 1 || w.stride(1) != 1 || bpb <= 0) return false;
    const int64_t rb = w.size(1);
    if (rb % bpb) return false;
    k = rb / bpb * 256;
    if (x.size(-1) != k || w.size(0) < 1) return false;
    wstride = w.size(0) > 1 ? w.stride(0) : rb;
    return true;
}

bool act_rows(const at::Tensor &x, int64_t k, at::Tensor &x2) {
    x2 = x.reshape({-1, k});
    if (x2.stride(1) != 1 || x2.stride(0) % 8 || (reinterpret_cast<uintptr_t>(x2.data_ptr()) & 15)) x2 = x2.contiguous();
    return true;
}

at::Tensor shaped(const at::Tensor &y, const at::Tensor &x, int64_t n) {
    auto sizes = x.sizes().vec();
    sizes.back() = n;
    return y.view(sizes);
}

// kq.quantized_matmul(x, w, None, codec) for 2-D wire weights; out_code < 0:
// the activation dtype.  None: take the Python path.
py::object quantized_matmul(const at::Tensor &x, const at::Tensor &w, int64_t codec, int64_t bpb, int64_t out_code) {
    int64_t k, wstride;
    if (!g_matmul || !common(x, w, bpb, k, wstride)) return py::none();
    at::Tensor x2;
    act_rows(x, k, x2);
    const int64_t m = x2.size(0), n = w.size(0);
    const at::ScalarType od = out_code == 0 ? at::kFloat : out_code == 1 ? at::kHalf : out_code == 2 ? at::kBFloat16
                                                                                                  : x.scalar_type();
    at::Tensor y = at::empty({m, n}, x.options().dtype(od));
    if (m) {
        const int dev = x.get_device();
        cudaStream_t st = at::cuda::getCurrentCUDAStream(dev).stream();
        at::Tensor ws = workspace(dev, reinterpret_cast<int64_t>(st), (int64_t)ws_bytes(0, (int)codec, m, n, k));
        const int rc = g_matmul((int)codec, x2.data_ptr(), dtype_code(x2.scalar_type()), m, k, x2.stride(0),
                                w.data_ptr(), n, wstride, y.data_ptr(), dtype_code(od), n, ws.data_ptr(),
                                (size_t)ws.numel(), st);
        if (rc) return py::none();
    }
    return py::cast(shaped(y, x, n));
}

// kq.quantized_glu(x, gate_w, up_w, codec, act) for 2-D wire weights of one shape.
py::object quantized_glu(const at::Tensor &x, const at::Tensor &wg, const at::Tensor &wu, int64_t codec, int64_t bpb,
                         int64_t act, int64_t out_code) {
    int64_t k, wstride, k2, wstride2;
    if (!g_glu || !common(x, wg, bpb, k, wstride) || !common(x, wu, bpb, k2, wstride2)) return py::none();
    if (wg.sizes() != wu.sizes() || wstride != wstride2) return py::none();
    at::Tensor x2;
    act_rows(x, k, x2);
    const int64_t m = x2.size(0), n = wg.size(0);
    const at::ScalarType od = out_code == 0 ? at::kFloat : out_code == 1 ? at::kHalf : out_code == 2 ? at::kBFloat16
                                                                                                  : x.scalar_type();
    at::Tensor y = at::empty({m, n}, x.options().dtype(od));
    if (m) {
        const int dev = x.get_device();
        cudaStream_t st = at::cuda::getCurrentCUDAStream(dev).stream();
        at::Tensor ws = workspace(dev, reinterpret_cast<int64_t>(st), (int64_t)ws_bytes(1, (int)codec, m, n, k));
        const int rc = g_glu((int)codec, x2.data_ptr(), dtype_code(x2.scalar_type()), m, k, x2.stride(0), wg.data_ptr(),
                             wu.data_ptr(), n, wstride, (int)act, y.data_ptr(), dtype_code(od), n, ws.data_ptr(),
                             (size_t)ws.numel(), st);
        if (rc) return py::none();
    }
    return py::cast(shaped(y, x, n));
}

// ---- the serving step ------------------------------------------------------
// As above: each takes the well-formed call and returns None for the rest.

decltype(&kq_paged_plan) g_plan = nullptr;
decltype(&kq_rope_kv_write) g_rope = nullptr;
decltype(&kq_paged_attention) g_attn = nullptr;
decltype(&kq_paged_attention_workspace_size) g_attn_ws = nullptr;
decltype(&kq_moe_route) g_route = nullptr;

void set_serve_entry_points(int64_t plan, int64_t rope, int64_t attn, int64_t attn_ws, int64_t route) {
    g_plan = reinterpret_cast<decltype(g_plan)>(plan);
    g_rope = reinterpret_cast<decltype(g_rope)>(rope);
    g_attn = reinterpret_cast<decltype(g_attn)>(attn);
    g_attn_ws = reinterpret_cast<decltype(g_attn_ws)>(attn_ws);
    g_route = reinterpret_cast<decltype(g_route)>(route);
}

bool vec(const at::Tensor &t, int64_t n, at::ScalarType type, int dev) {
    return t.is_cuda() && t.get_device() == dev && t.dim() == 1 && (n < 0 || t.size(0) == n) && t.scalar_type() == type &&
           t.is_contiguous();
}

int64_t st(const at::Tensor &t, int i) { return t.size(i) == 1 ? 0 : t.stride(i); }
bool dense(const at::Tensor &t, int i) { return t.size(i) <= 1 || t.stride(i) == 1; }

bool table_ok(const at::Tensor &t, int64_t b, int dev) {
    return t.is_cuda() && t.get_device() == dev && t.dim() == 2 && t.size(0) == b && t.scalar_type() == at::kInt &&
           dense(t, 1);
}
int64_t table_stride(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

bool cache_of(const at::Tensor &k, const at::Tensor &v, kq_paged_cache &c) {
    if (!k.is_cuda() || !v.is_cuda() || v.get_device() != k.get_device() || k.dim() != 4 || v.dim() != 4 ||
        k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || k.numel() == 0)
        return false;
    const int code = dtype_code(k.scalar_type());
    if (code < 1) return false;
    for (int i = 0; i < 4; i++)
        if (st(k, i) != st(v, i)) return false;
    if (!dense(k, 3)) return false;
    c = kq_paged_cache{k.data_ptr(), v.data_ptr(), code, k.size(0), k.size(1), k.size(2), k.size(3), st(k, 0), st(k, 1), st(k, 2)};
    return true;
}

bool heads_ok(const at::Tensor &t, const kq_paged_cache &c, int dev) {
    return t.is_cuda() && t.get_device() == dev && t.dim() == 3 && t.size(2) == c.dim && dtype_code(t.scalar_type()) == c.dtype &&
           dense(t, 2) && st(t, 0) % 8 == 0 && st(t, 1) % 8 == 0 && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15);
}

// Tensors that share one allocation: a caching-allocator round trip costs the host as
// much as the rest of such a call, and these outputs live and die together.
struct Block {
    at::Tensor all;
    int64_t at = 0;
    Block(const at::Tensor &like, int64_t bytes) : all(at::empty({bytes}, like.options().dtype(at::kByte))) {}
    static int64_t room(int64_t n, int64_t size) { return (n * size + 15) / 16 * 16; }
    at::Tensor take(at::IntArrayRef sizes, at::ScalarType type) {
        int64_t n = 1;
        for (auto v : sizes) n *= v;
        const int64_t size = (int64_t)c10::elementSize(type);
        auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
        t.unsafeGetTensorImpl()->set_storage_offset(at / size);
        at += room(n, size);
        return t;
    }
};

at::Tensor stream_workspace(int dev, cudaStream_t s, size_t bytes) { return workspace(dev, reinterpret_cast<int64_t>(s), (int64_t)bytes); }

py::object paged_plan(const at::Tensor &ctx, const at::Tensor &qlen, const at::Tensor &table, const at::Tensor &free_pages,
                      int64_t page, int64_t tokens) {
    if (!g_plan || !ctx.is_cuda() || tokens < 0) return py::none();
    const int dev = ctx.get_device();
    if (!vec(ctx, -1, at::kInt, dev)) return py::none();
    const int64_t b = ctx.size(0);
    if (!vec(qlen, b, at::kInt, dev) || !vec(free_pages, -1, at::kInt, dev) || !table_ok(table, b, dev)) return py::none();
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    Block m(ctx, Block::room(b + 1, 4) + Block::room(b, 4) + Block::room(tokens, 8) + Block::room(tokens, 4) + 16);
    at::Tensor cu = m.take({b + 1}, at::kInt), seq = m.take({b}, at::kInt), slots = m.take({tokens}, at::kLong),
               pos = m.take({tokens}, at::kInt), used = m.take({1}, at::kInt);
    cudaStream_t s = at::cuda::getCurrentCUDAStream(dev).stream();
    at::Tensor ws = stream_workspace(dev, s, 256);
    const int rc = g_plan(ctx.data_ptr<int>(), qlen.data_ptr<int>(), b, table.data_ptr<int>(), table_stride(table), table.size(1),
                          free_pages.data_ptr<int>(), free_pages.size(0), page, tokens, cu.data_ptr<int>(), seq.data_ptr<int>(),
                          slots.data_ptr<int64_t>(), pos.data_ptr<int>(), used.data_ptr<int>(), ws.data_ptr(), (size_t)ws.numel(), s);
    if (rc) return py::none();
    return py::make_tuple(cu, seq, slots, pos, used);
}

py::object rope_kv_write(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &cos, const at::Tensor &sin,
                         const at::Tensor &pos, const at::Tensor &kc, const at::Tensor &vc, const at::Tensor &slots, bool interleaved) {
    kq_paged_cache c;
    if (!g_rope || !cache_of(kc, vc, c)) return py::none();
    const int dev = kc.get_device();
    if (!heads_ok(q, c, dev) || !heads_ok(k, c, dev) || !heads_ok(v, c, dev)) return py::none();
    const int64_t t = q.size(0), h = q.size(1);
    if (k.size(0) != t || v.size(0) != t || k.size(1) != c.kv_heads || v.size(1) != c.kv_heads) return py::none();
    if (!cos.is_cuda() || cos.get_device() != dev || cos.dim() != 2 || cos.scalar_type() != at::kFloat || !cos.is_contiguous() ||
        !sin.is_cuda() || sin.get_device() != dev || sin.sizes() != cos.sizes() || sin.scalar_type() != at::kFloat || !sin.is_contiguous())
        return py::none();
    if (!vec(pos, t, at::kInt, dev) || !vec(slots, t, at::kLong, dev)) return py::none();
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    at::Tensor out = at::empty({t, h, c.dim}, q.options());
    cudaStream_t s = at::cuda::getCurrentCUDAStream(dev).stream();
    at::Tensor ws = stream_workspace(dev, s, 256);
    const int rc = g_rope(&c, q.data_ptr(), st(q, 0), st(q, 1), k.data_ptr(), st(k, 0), st(k, 1), v.data_ptr(), st(v, 0), st(v, 1), t,
                          h, cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0), (int)(2 * cos.size(1)), interleaved,
                          pos.data_ptr<int>(), slots.data_ptr<int64_t>(), out.data_ptr(), ws.data_ptr(), (size_t)ws.numel(), s);
    if (rc) return py::none();
    return py::cast(out);
}

py::object paged_attention(const at::Tensor &q, const at::Tensor &kc, const at::Tensor &vc, const at::Tensor &table, const at::Tensor &seq,
                           const at::Tensor &cu, int64_t max_query_len, double scale, int64_t window, double softcap, bool causal,
                           bool return_lse) {
    kq_paged_cache c;
    if (!g_attn || !cache_of(kc, vc, c)) return py::none();
    const int dev = kc.get_device();
    if (!heads_ok(q, c, dev) || !vec(seq, -1, at::kInt, dev)) return py::none();
    const int64_t t = q.size(0), h = q.size(1), b = seq.size(0);
    if (!vec(cu, b + 1, at::kInt, dev) || !table_ok(table, b, dev)) return py::none();
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    at::Tensor out = at::empty({t, h, c.dim}, q.options()), lse;
    if (return_lse) lse = at::empty({t, h}, q.options().dtype(at::kFloat));
    cudaStream_t s = at::cuda::getCurrentCUDAStream(dev).stream();
    at::Tensor ws = stream_workspace(dev, s, g_attn_ws(c.dim));
    const int rc = g_attn(&c, q.data_ptr(), st(q, 0), st(q, 1), t, h, table.data_ptr<int>(), table_stride(table), table.size(1),
                          seq.data_ptr<int>(), cu.data_ptr<int>(), b, max_query_len, (float)scale, causal, window, (float)softcap,
                          out.data_ptr(), return_lse ? lse.data_ptr<float>() : nullptr, ws.data_ptr(), (size_t)ws.numel(), s);
    if (rc) return py::none();
    return return_lse ? py::object(py::make_tuple(out, lse)) : py::object(py::cast(out));
}

py::object moe_route(const at::Tensor &logits, int64_t k, int64_t scoring, const c10::optional<at::Tensor> &bias, int64_t n_groups,
                     int64_t topk_groups, bool norm, double scale) {
    if (!g_route || !logits.is_cuda() || logits.dim() != 2 || k < 1) return py::none();
    const int code = dtype_code(logits.scalar_type()), dev = logits.get_device();
    const int64_t t = logits.size(0), e = logits.size(1);
    if (code < 0 || !dense(logits, 1) || (bias && !vec(*bias, e, at::kFloat, dev))) return py::none();
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    Block m(logits, 2 * Block::room(t * k, 4));
    at::Tensor idx = m.take({t, k}, at::kInt), w = m.take({t, k}, at::kFloat);
    cudaStream_t s = at::cuda::getCurrentCUDAStream(dev).stream();
    const int rc = g_route(logits.data_ptr(), code, t, e, st(logits, 0), (int)k, (int)scoring, bias ? bias->data_ptr<float>() : nullptr,
                           (int)n_groups, (int)topk_groups, norm, (float)scale, idx.data_ptr<int>(), w.data_ptr<float>(), s);
    if (rc) return py::none();
    return py::make_tuple(idx, w);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("set_entry_points", &set_entry_points);
    m.def("workspace", &workspace);
    m.def("workspace_peek", &workspace_peek);
    m.def("workspaces", &workspaces);
    m.def("quantized_matmul", &quantized_matmul);
    m.def("quantized_glu", &quantized_glu);
    m.def("set_serve_entry_points", &set_serve_entry_points);
    m.def("paged_plan", &paged_plan);
    m.def("rope_kv_write", &rope_kv_write);
    m.def("paged_attention", &paged_attention);
    m.def("moe_route", &moe_route);
}
