// The host sides of linear and latent attention: the checks of a call's tensors, its workspace, and the call of the C ABI, in native
// code as for fwd (a step of single tokens runs for a few microseconds on the GPU).
#include "fkda_host_args.h"

using namespace fkda_host;

namespace {

void check_tensor(const at::Tensor& t, const char* name, at::ScalarType type, const char* type_name, const c10::Device& dev) {
    check_named(t.is_cuda(), name, " must be on CUDA");
    check_named(t.device() == dev, name, " must be on the same device as q");
    if (t.scalar_type() != type) throw Refused(std::string(name) + " must be " + type_name);
}
// bf16, of this shape, with a contiguous last dimension
void check_bf16(const at::Tensor& t, const char* name, const c10::Device& dev, std::initializer_list<int64_t> shape, const char* shape_name) {
    check_tensor(t, name, at::kBFloat16, "bfloat16", dev);
    if (!shape_is(t, shape)) throw Refused(std::string(name) + " must be " + shape_name);
    check_named(t.numel() == 0 || t.stride(t.dim() - 1) == 1, name, " must be contiguous in its last dimension");
}
const int64_t* cu_arg(PyObject* o, const char* name, const c10::Device& dev, int64_t B, int64_t* N) {
    const at::Tensor* cu = optional_tensor_arg(o, name);
    if (cu == nullptr) return nullptr;
    check_named(B == 1, "B must be 1 when ", (std::string(name) + " is provided").c_str());
    check_tensor(*cu, name, at::kLong, "int64", dev);
    check_named(cu->dim() == 1, name, " must be 1D");
    check_named(cu->numel() >= 2, name, " must have at least 2 elements");
    check_named(cu->is_contiguous(), name, " must be contiguous");
    *N = cu->numel() - 1;
    return static_cast<const int64_t*>(cu->data_ptr());
}
float* lse_arg(PyObject* o, const c10::Device& dev, std::initializer_list<int64_t> shape, const char* shape_name) {
    const at::Tensor* lse = optional_tensor_arg(o, "lse");
    if (lse == nullptr) return nullptr;
    check_tensor(*lse, "lse", at::kFloat, "float32", dev);
    if (!shape_is(*lse, shape)) throw Refused(std::string("lse must be ") + shape_name);
    check(lse->is_contiguous(), "lse must be contiguous");
    return static_cast<float*>(lse->data_ptr());
}
void strides(const at::Tensor& t, int64_t* to, int n) {
    for (int i = 0; i < n; ++i) to[i] = t.stride(i);
}

// Switches to the tensors' device if it is not the current one; the stream is that device's current one.
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    cudaStream_t stream;
    explicit On(const c10::Device& dev) {
        if (c10::cuda::current_device() != dev.index()) guard.set_index(dev.index());
        stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    }
};
// The caller's workspace, or one of the caching allocator that goes back to it, in stream order, with this object.
struct Workspace {
    c10::DataPtr own;
    void* ptr = nullptr;
    size_t bytes = 0;
    Workspace(PyObject* o, size_t need, const c10::Device& dev) {
        const at::Tensor* ws = optional_tensor_arg(o, "workspace");
        if (ws != nullptr) {
            check(ws->is_cuda() && ws->device() == dev && ws->is_contiguous() && ws->scalar_type() == at::kByte && (size_t)ws->numel() >= need,
                  "workspace must be a contiguous CUDA uint8 tensor of sufficient size");
            ptr = ws->data_ptr();
            bytes = (size_t)ws->numel();
        } else if (need > 0) {
            own = c10::cuda::CUDACachingAllocator::get()->allocate(need);
            ptr = own.get();
            bytes = need;
        }
    }
};
template <typename Call>
void enqueue(const char* name, const Call& call) {
    int rc;
    Py_BEGIN_ALLOW_THREADS   // (a launch may wait for room in the stream's queue; the caller holds the tensors)
    rc = call();
    Py_END_ALLOW_THREADS
    if (rc != 0) throw Refused(std::string(name) + " failed: " + fkda_status_string(rc) + " (status " + std::to_string(rc) + ")");
}

// linear_attention_fwd(q, k, v, g, scale, out, initial_state, final_state, cu_seqlens, workspace)
void linear(PyObject* const* a) {
    const at::Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &v = tensor_arg(a[2], "v"), &g = tensor_arg(a[3], "g"), &out = tensor_arg(a[5], "out");
    const c10::Device dev = q.device();
    check(q.is_cuda(), "q must be on CUDA");
    check(q.dim() == 4 && v.dim() == 4, "q and v must be [B, T, H, 128]");
    const int64_t B = q.size(0), T = q.size(1), H = v.size(2), Hk = q.size(2);
    check(H >= 1 && Hk >= 1 && H % Hk == 0, "the heads of q must divide those of v");
    check_bf16(q, "q", dev, {B, T, Hk, FKDA_HEAD_DIM}, "[B, T, Hk, 128]");
    check_bf16(k, "k", dev, {B, T, Hk, FKDA_HEAD_DIM}, "[B, T, Hk, 128]");
    check_bf16(v, "v", dev, {B, T, H, FKDA_HEAD_DIM}, "[B, T, H, 128]");
    check_bf16(out, "out", dev, {B, T, H, FKDA_HEAD_DIM}, "[B, T, H, 128]");
    check_tensor(g, "g", at::kFloat, "float32", dev);
    check(shape_is(g, {B, T, H}) || shape_is(g, {H}), "g must be [B, T, H] or [H]");
    check(B >= 1, "B must be at least 1");
    fkda_linear_params p{};
    p.N = B;
    p.cu_seqlens = cu_arg(a[8], "cu_seqlens", dev, B, &p.N);
    const at::Tensor* states[2] = {optional_tensor_arg(a[6], "initial_state"), optional_tensor_arg(a[7], "final_state")};
    static const char* const names[2] = {"initial_state", "final_state"};
    bool fp32 = false;
    for (int i = 0; i < 2; ++i) {
        if (states[i] == nullptr) continue;
        const at::Tensor& s = *states[i];
        check_named(s.is_cuda() && s.is_contiguous(), names[i], " must be contiguous CUDA tensor");
        check_named(s.scalar_type() == at::kBFloat16 || s.scalar_type() == at::kFloat, names[i], " must be bfloat16 or float32");
        check_named(shape_is(s, {p.N, H, FKDA_HEAD_DIM, FKDA_HEAD_DIM}), names[i], " must be [N, H, D, D]");
        check_named(s.device() == dev, names[i], " must be on the same device as q");
        fp32 |= s.scalar_type() == at::kFloat;
    }
    if (states[0] != nullptr && states[1] != nullptr)
        check(states[0]->scalar_type() == states[1]->scalar_type(), "initial_state and final_state must have the same dtype");
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.out = out.data_ptr();
    p.g = static_cast<const float*>(g.data_ptr());
    p.initial_state = states[0] != nullptr ? states[0]->data_ptr() : nullptr;
    p.final_state = states[1] != nullptr ? states[1]->data_ptr() : nullptr;
    p.B = B; p.T = T; p.H = H; p.Hk = Hk;
    strides(q, p.q_stride, 3);
    strides(k, p.k_stride, 3);
    strides(v, p.v_stride, 3);
    strides(out, p.out_stride, 3);
    if (g.dim() == 3) strides(g, p.g_stride, 3);
    else p.g_stride[2] = g.stride(0);
    p.scale = (float)number_arg(a[4]);
    p.state_dtype = fp32 ? FKDA_STATE_FP32 : FKDA_STATE_BF16;
    On on(dev);
    Workspace ws(a[9], fkda_linear_workspace_bytes(&p), dev);
    p.workspace = ws.ptr;
    p.workspace_bytes = ws.bytes;
    enqueue("fkda_linear_attention_fwd", [&] { return fkda_linear_attention_fwd(&p, on.stream); });
}

// latent_attention_fwd(q, k, k_rope, v, scale, out, lse, cu_seqlens, cu_seqlens_k, causal)
void latent(PyObject* const* a) {
    const at::Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &r = tensor_arg(a[2], "k_rope"), &v = tensor_arg(a[3], "v"), &out = tensor_arg(a[5], "out");
    const c10::Device dev = q.device();
    check(q.is_cuda(), "q must be on CUDA");
    check(q.dim() == 4, "q must be [B, T, H, 192]");
    check(k.dim() == 4, "k must be [B, Tk, H, 128]");
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), Tk = k.size(1);
    check(B >= 1 && H >= 1, "B and H must be at least 1");
    check_bf16(q, "q", dev, {B, T, H, 192}, "[B, T, H, 192]");
    check_bf16(k, "k", dev, {B, Tk, H, 128}, "[B, Tk, H, 128]");
    check_bf16(r, "k_rope", dev, {B, Tk, 64}, "[B, Tk, 64]");
    check_bf16(v, "v", dev, {B, Tk, H, 128}, "[B, Tk, H, 128]");
    check_bf16(out, "out", dev, {B, T, H, 128}, "[B, T, H, 128]");
    fkda_latent_params p{};
    p.lse = lse_arg(a[6], dev, {B, T, H}, "[B, T, H]");
    p.N = B;
    int64_t n_k = B;
    p.cu_seqlens = cu_arg(a[7], "cu_seqlens", dev, B, &p.N);
    p.cu_seqlens_k = cu_arg(a[8], "cu_seqlens_k", dev, B, &n_k);
    if (p.cu_seqlens != nullptr && p.cu_seqlens_k == nullptr) {   // keys packed as the queries
        check(T == Tk, "k must have as many tokens as q where cu_seqlens_k is not given");
        p.cu_seqlens_k = p.cu_seqlens;
        n_k = p.N;
    }
    check((p.cu_seqlens != nullptr) == (p.cu_seqlens_k != nullptr), "cu_seqlens_k needs cu_seqlens");
    check(p.N == n_k, "cu_seqlens and cu_seqlens_k must have the same length");
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.k_rope = r.data_ptr(); p.v = v.data_ptr(); p.out = out.data_ptr();
    p.B = B; p.T = T; p.Tk = Tk; p.H = H;
    strides(q, p.q_stride, 3);
    strides(k, p.k_stride, 3);
    strides(v, p.v_stride, 3);
    strides(out, p.out_stride, 3);
    strides(r, p.k_rope_stride, 2);
    p.scale = (float)number_arg(a[4]);
    const int causal = PyObject_IsTrue(a[9]);
    if (causal < 0) throw std::bad_cast();
    p.causal = causal;
    On on(dev);
    enqueue("fkda_latent_attention_fwd", [&] { return fkda_latent_attention_fwd(&p, on.stream); });
}

// latent_attention_decode(q, cache, block_table, cache_lens, scale, out, lse, workspace)
void decode(PyObject* const* a) {
    const at::Tensor &q = tensor_arg(a[0], "q"), &cache = tensor_arg(a[1], "cache"), &table = tensor_arg(a[2], "block_table"), &lens = tensor_arg(a[3], "cache_lens"),
                     &out = tensor_arg(a[5], "out");
    const c10::Device dev = q.device();
    check(q.is_cuda(), "q must be on CUDA");
    check(q.dim() == 4, "q must be [B, Tq, H, 576]");
    check(cache.dim() == 3, "cache must be [pages, page_size, 576]");
    check(table.dim() == 2, "block_table must be [B, max_pages]");
    const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2);
    check(H >= 1, "H must be at least 1");
    check_bf16(q, "q", dev, {B, Tq, H, 576}, "[B, Tq, H, 576]");
    check_bf16(cache, "cache", dev, {cache.size(0), cache.size(1), 576}, "[pages, page_size, 576]");
    check_bf16(out, "out", dev, {B, Tq, H, 512}, "[B, Tq, H, 512]");
    check_tensor(table, "block_table", at::kInt, "int32", dev);
    check(table.size(0) == B && (table.size(1) <= 1 || table.stride(1) == 1), "block_table must be [B, max_pages], contiguous in its last dimension");
    check_tensor(lens, "cache_lens", at::kInt, "int32", dev);
    check(shape_is(lens, {B}) && lens.is_contiguous(), "cache_lens must be [B] and contiguous");
    check(cache.size(1) >= 16 && cache.size(1) % 16 == 0, "page_size must be a multiple of 16");
    // rows = new token x head have one stride
    auto row_stride = [&](const at::Tensor& t, const char* name) {
        if (Tq > 1 && H > 1) check_named(t.stride(1) == H * t.stride(2), name, " must have its new tokens H heads apart");
        return H > 1 ? t.stride(2) : t.stride(1);
    };
    fkda_latent_decode_params p{};
    p.lse = lse_arg(a[6], dev, {B, Tq, H}, "[B, Tq, H]");
    p.q = q.data_ptr(); p.cache = cache.data_ptr(); p.out = out.data_ptr();
    p.block_table = static_cast<const int32_t*>(table.data_ptr());
    p.cache_lens = static_cast<const int32_t*>(lens.data_ptr());
    p.B = B; p.Tq = Tq; p.H = H;
    p.pages = cache.size(0); p.page_size = cache.size(1); p.max_pages = table.size(1);
    p.q_stride[0] = q.stride(0);
    p.q_stride[1] = row_stride(q, "q");
    p.out_stride[0] = out.stride(0);
    p.out_stride[1] = row_stride(out, "out");
    strides(cache, p.cache_stride, 2);
    p.block_table_stride = table.stride(0);
    p.scale = (float)number_arg(a[4]);
    On on(dev);
    Workspace ws(a[7], fkda_latent_decode_workspace_bytes(&p), dev);
    p.workspace = ws.ptr;
    p.workspace_bytes = ws.bytes;
    enqueue("fkda_latent_attention_decode", [&] { return fkda_latent_attention_decode(&p, on.stream); });
}

}  // namespace

PyObject* host_linear_attention_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) { return refusing("linear_attention_fwd", 10, n, [&] { linear(args); }); }
PyObject* host_latent_attention_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) { return refusing("latent_attention_fwd", 10, n, [&] { latent(args); }); }
PyObject* host_latent_attention_decode(PyObject*, PyObject* const* args, Py_ssize_t n) { return refusing("latent_attention_decode", 8, n, [&] { decode(args); }); }
