// Operator registration of pathsig_b200 with the PyTorch dispatcher (libpathsig_b200_torch.so).
//
// Counterpart of the reference's src/pathsig/bindings.cpp:7-64 (schemas, pt2_compliant_tag) and of the
// TORCH_LIBRARY_IMPL(pathsig, CUDA, ...) blocks of its launchers (src/pathsig/forward/sig_launch.cu:345-348,
// src/pathsig/backward/sig_backward_launch.cu:468-471): the same four schemas, registered for the CUDA key
// only, in the namespace `pathsig_b200` (so that a build of the reference can be loaded in the same
// process), plus the operators the reference does not have (projected log-signature, Chen product, decayed linear
// attention, norm around a block).
// Every implementation validates like the reference launchers (src/pathsig/forward/sig_launch.cu:84-121,
// src/pathsig/backward/sig_backward_launch.cu:94-155), allocates its outputs with the caching allocator
// and hands raw pointers plus the current stream to the C ABI of include/pathsig_b200.h.  torch is used
// for memory, streams and dispatch only; fake (meta) implementations and autograd formulas are registered
// from Python (pathsig_b200/ops.py), but for the autograd formulas of the sequence operators, which are below.
#include <ATen/ATen.h>
#include <ATen/Context.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>
#include <nvtx3/nvToolsExt.h>

#include <atomic>
#include <cmath>
#include <list>
#include <mutex>
#include <optional>
#include <tuple>
#include <type_traits>
#include <vector>

#include "../../include/pathsig_b200.h"

namespace {

std::atomic<int> g_algo{PSIG_ALGO_AUTO};

// NVTX range around an operator call (host side: validation, allocation, enqueue), so that a timeline
// shows which operator a kernel belongs to.  Costs nothing measurable without a tool attached.
struct Range {
    explicit Range(const char *name) { nvtxRangePushA(name); }
    ~Range() { nvtxRangePop(); }
    Range(const Range &) = delete;
    Range &operator=(const Range &) = delete;
};

void check(int64_t status, const char *what)
{
    TORCH_CHECK(status >= 0, "pathsig_b200::", what, ": ", psig_status_string((int)status), " (status ", status, ")");
}

int dtype_id(const at::Tensor &t)
{
    if (t.scalar_type() == at::kFloat) return PSIG_F32;
    if (t.scalar_type() == at::kDouble) return PSIG_F64;
    TORCH_CHECK(false, "path must be float32 or float64");
}

void *stream_of(const at::Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

const void *ptr(const at::Tensor &t) { return t.numel() > 0 ? t.data_ptr() : nullptr; }

// Every tensor operand must live on the device the kernels are launched on.  The dispatcher checks this
// for operators with structured kernels only; a pointer into another GPU's memory would fault there.
void same_device(const at::Tensor &anchor, const at::Tensor &t, const char *name)
{
    TORCH_CHECK(t.device() == anchor.device(), name, " must be on the same device as the path/signature (", name,
                " is on ", t.device(), ", expected ", anchor.device(), ")");
}

void check_words(const at::Tensor &words)
{
    TORCH_CHECK(words.is_cuda(), "encoded_words must be CUDA");
    TORCH_CHECK(words.scalar_type() == at::kLong, "encoded_words must be int64");
    TORCH_CHECK(words.is_contiguous(), "encoded_words must be contiguous");
    TORCH_CHECK(words.dim() == 1, "encoded_words must be 1D");
}

// Host copies of word-code tensors.  The prefix-closure kernels are generated from the word set, so the
// library wants the codes in host memory; reading them back on every call would synchronise, so the copy
// is made once per (storage, version) and kept while the device tensor is alive.  An entry holds a
// reference to its device tensor, which keeps the address from being reused by another tensor.
struct HostWords {
    const void *data;
    int64_t version;
    int64_t numel;
    int device;
    at::Tensor on_device, on_host;
};
std::mutex g_words_mutex;
std::list<HostWords> g_words;  // most recently used first
constexpr size_t kHostWordsLimit = 64;

at::Tensor host_words(const at::Tensor &words)
{
    std::lock_guard<std::mutex> lock(g_words_mutex);
    for (auto it = g_words.begin(); it != g_words.end(); ++it) {
        if (it->data == words.data_ptr() && it->version == words._version() && it->numel == words.numel() &&
            it->device == words.get_device()) {
            g_words.splice(g_words.begin(), g_words, it);
            return g_words.front().on_host;
        }
    }
    // no device read inside a graph capture; the library then uses another kernel family
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return at::Tensor();
    HostWords e{words.data_ptr(), words._version(), words.numel(), (int)words.get_device(), words,
                words.detach().to(at::kCPU).contiguous()};
    g_words.push_front(e);
    while (g_words.size() > kHostWordsLimit) g_words.pop_back();
    return g_words.front().on_host;
}

int64_t ipow(int64_t b, int64_t e) { int64_t r = 1; for (int64_t i = 0; i < e; ++i) r *= b; return r; }

int64_t row_width(int64_t d, int64_t depth, bool alt, at::IntArrayRef level_sizes)
{
    int64_t w = 0;
    for (int64_t k = 1; k <= depth; ++k) w += alt ? level_sizes[k] : ipow(d, k);
    return w;
}

// Validated PsigSigDesc; `keep` receives tensors that must stay alive during the call.
PsigSigDesc sig_desc(const at::Tensor &path, int64_t depth, bool alt, const at::Tensor &encoded_words,
                     at::IntArrayRef level_sizes, bool use_windows, const at::Tensor &windows, std::vector<at::Tensor> &keep)
{
    TORCH_CHECK(path.is_cuda(), "path must be CUDA");
    TORCH_CHECK(path.dim() == 3, "path must be [B,T,d]");
    TORCH_CHECK(depth >= 1 && depth <= PSIG_MAX_DEPTH, "depth must be in [1,12]");
    TORCH_CHECK(path.size(1) >= 2, "path must have at least 2 time steps");
    PsigSigDesc desc{};
    desc.dtype = dtype_id(path);
    desc.d = (int32_t)path.size(2);
    desc.depth = (int32_t)depth;
    desc.B = path.size(0);
    desc.L = path.size(1);
    desc.projected = alt ? 1 : 0;
    desc.algo = g_algo.load();
    // torch.use_deterministic_algorithms(True): ask for the fixed-order backward where the library has one
    if (at::globalContext().deterministicAlgorithms()) desc.flags |= PSIG_FLAG_DETERMINISTIC;
    if (alt) {
        check_words(encoded_words);
        same_device(path, encoded_words, "encoded_words");
        TORCH_CHECK((int64_t)level_sizes.size() >= depth + 1, "level_sizes must cover at least depth + 1 entries");
        int64_t need = 0;
        for (int64_t k = 1; k <= depth; ++k) {
            desc.level_sizes[k] = level_sizes[k];
            if (level_sizes[k] != ipow(desc.d, k)) need += level_sizes[k];
        }
        TORCH_CHECK(encoded_words.numel() >= need, "encoded_words holds fewer codes than level_sizes requires");
        if (encoded_words.numel() > 0) {
            desc.words = encoded_words.data_ptr<int64_t>();
            at::Tensor host = host_words(encoded_words);
            if (host.defined()) {
                desc.words_host = host.data_ptr<int64_t>();
                keep.push_back(host);
            }
        }
    }
    if (use_windows) {
        TORCH_CHECK(windows.is_cuda(), "windows must be CUDA");
        TORCH_CHECK(windows.dim() == 2 && windows.size(1) == 2, "windows must be [W,2]");
        TORCH_CHECK(windows.scalar_type() == at::kInt || windows.scalar_type() == at::kLong, "windows must be int32");
        same_device(path, windows, "windows");
        at::Tensor win = windows.to(at::kInt).contiguous();
        keep.push_back(win);
        desc.W = win.size(0);
        desc.windows = win.numel() > 0 ? win.data_ptr<int32_t>() : nullptr;
    }
    return desc;
}

at::Tensor compute_signature(const at::Tensor &path_in, int64_t depth, bool alt, const at::Tensor &encoded_words,
                             at::IntArrayRef level_sizes, bool use_windows, const at::Tensor &windows)
{
    Range range("pathsig_b200::compute_signature");
    TORCH_CHECK(path_in.is_cuda(), "path must be CUDA");
    c10::cuda::CUDAGuard guard(path_in.device());
    at::Tensor path = path_in.contiguous();
    std::vector<at::Tensor> keep;
    PsigSigDesc desc = sig_desc(path, depth, alt, encoded_words, level_sizes, use_windows, windows, keep);
    const int64_t D = row_width(desc.d, desc.depth, alt, level_sizes);
    at::Tensor out = use_windows ? at::empty({desc.B, desc.W, D}, path.options()) : at::empty({desc.B, D}, path.options());
    if (out.numel() == 0) return out;  // no paths, no windows or no requested words: nothing to launch
    check(psig_sig_forward(&desc, path.data_ptr(), out.data_ptr(), stream_of(path)), "compute_signature");
    return out;
}

at::Tensor signature_backward(const at::Tensor &path_in, const at::Tensor &signature_in, const at::Tensor &grad_in,
                              int64_t depth, bool alt, const at::Tensor &encoded_words, at::IntArrayRef level_sizes,
                              bool use_windows, const at::Tensor &windows)
{
    Range range("pathsig_b200::signature_backward");
    TORCH_CHECK(path_in.is_cuda(), "path must be CUDA");
    TORCH_CHECK(signature_in.is_cuda(), "signature must be CUDA");
    TORCH_CHECK(grad_in.is_cuda(), "grad_signature must be CUDA");
    TORCH_CHECK(signature_in.scalar_type() == path_in.scalar_type(), "signature must have same dtype as path");
    TORCH_CHECK(grad_in.scalar_type() == path_in.scalar_type(), "grad_signature must have same dtype as path");
    TORCH_CHECK(signature_in.sizes() == grad_in.sizes(), "grad_signature must match signature shape");
    same_device(path_in, signature_in, "signature");
    same_device(path_in, grad_in, "grad_signature");
    c10::cuda::CUDAGuard guard(path_in.device());
    at::Tensor path = path_in.contiguous(), sig = signature_in.contiguous(), grad = grad_in.contiguous();
    std::vector<at::Tensor> keep;
    PsigSigDesc desc = sig_desc(path, depth, alt, encoded_words, level_sizes, use_windows, windows, keep);
    const int64_t D = row_width(desc.d, desc.depth, alt, level_sizes);
    const bool shape_ok = use_windows ? (sig.dim() == 3 && sig.size(0) == desc.B && sig.size(1) == desc.W && sig.size(2) == D)
                                      : (sig.dim() == 2 && sig.size(0) == desc.B && sig.size(1) == D);
    if (!shape_ok) {
        TORCH_CHECK(!(use_windows && sig.dim() == 3 && sig.size(1) != desc.W), "windows.size(0) must match signature num_windows");
        TORCH_CHECK(false, "signature must be [B,S] or [B,W,S]");
    }
    if (sig.numel() == 0) return at::zeros_like(path);  // an empty signature carries no gradient
    at::Tensor grad_path = at::empty_like(path);
    const int64_t ws_bytes = psig_sig_backward_workspace(&desc);
    check(ws_bytes, "signature_backward");
    at::Tensor ws = at::empty({std::max<int64_t>(ws_bytes, 1)}, path.options().dtype(at::kByte));
    check(psig_sig_backward(&desc, path.data_ptr(), sig.data_ptr(), grad.data_ptr(), grad_path.data_ptr(), ws.data_ptr(),
                            ws_bytes, stream_of(path)),
          "signature_backward");
    return grad_path;
}

PsigLogDesc log_desc(const at::Tensor &signature, int64_t depth, int64_t d, bool alt, const at::Tensor &encoded_words,
                     at::IntArrayRef level_sizes)
{
    TORCH_CHECK(depth >= 1 && depth <= PSIG_MAX_DEPTH, "depth must be in [1,12]");
    TORCH_CHECK(d >= 1, "d must be >= 1");
    TORCH_CHECK(signature.dim() == 2 || signature.dim() == 3, "signature must be [B,S] or [B,W,S]");
    PsigLogDesc desc{};
    desc.dtype = dtype_id(signature);
    desc.d = (int32_t)d;
    desc.depth = (int32_t)depth;
    desc.algo = g_algo.load();
    desc.rows = signature.size(-1) > 0 ? signature.numel() / signature.size(-1) : 0;
    desc.top_size = ipow(d, depth);
    if (alt) {
        check_words(encoded_words);
        same_device(signature, encoded_words, "encoded_words");
        TORCH_CHECK((int64_t)level_sizes.size() >= depth + 1, "level_sizes must have entries up to depth");
        desc.top_size = level_sizes[depth];
        if (desc.top_size != ipow(d, depth)) {
            TORCH_CHECK(encoded_words.numel() >= desc.top_size, "encoded_words holds fewer codes than level_sizes[depth]");
            desc.top_words = encoded_words.numel() > 0 ? encoded_words.data_ptr<int64_t>() : nullptr;
        }
    }
    return desc;
}

std::vector<int64_t> with_last(const at::Tensor &t, int64_t last)
{
    std::vector<int64_t> shape(t.sizes().begin(), t.sizes().end());
    shape.back() = last;
    return shape;
}

std::tuple<at::Tensor, at::Tensor> sig_to_logsig(const at::Tensor &signature_in, int64_t depth, int64_t d, bool alt,
                                                 const at::Tensor &encoded_words, at::IntArrayRef level_sizes)
{
    Range range("pathsig_b200::sig_to_logsig");
    TORCH_CHECK(signature_in.is_cuda(), "signature must be CUDA");
    c10::cuda::CUDAGuard guard(signature_in.device());
    at::Tensor sig = signature_in.contiguous();
    PsigLogDesc desc = log_desc(sig, depth, d, alt, encoded_words, level_sizes);
    const int64_t S = psig_logsig_size(&desc);
    check(S, "sig_to_logsig");
    TORCH_CHECK(S == sig.size(-1), "signature width ", sig.size(-1), " does not match the layout width ", S);
    at::Tensor logsig = at::empty_like(sig);
    const int64_t per_row = psig_logsig_cache_size(&desc);
    check(per_row, "sig_to_logsig");
    at::Tensor cache = at::empty(with_last(sig, per_row), sig.options());
    check(psig_logsig_forward(&desc, ptr(sig), const_cast<void *>(ptr(logsig)), const_cast<void *>(ptr(cache)), stream_of(sig)),
          "sig_to_logsig");
    return std::make_tuple(logsig, cache);
}

at::Tensor logsig_backward(const at::Tensor &signature_in, const at::Tensor &P_in, const at::Tensor &grad_in, int64_t depth,
                           bool alt, const at::Tensor &encoded_words, at::IntArrayRef level_sizes)
{
    Range range("pathsig_b200::logsig_backward");
    TORCH_CHECK(signature_in.is_cuda(), "sig must be CUDA");
    TORCH_CHECK(P_in.is_cuda(), "P must be CUDA");
    TORCH_CHECK(grad_in.is_cuda(), "grad_logsig must be CUDA");
    TORCH_CHECK(P_in.scalar_type() == signature_in.scalar_type(), "P must have same dtype as sig");
    TORCH_CHECK(grad_in.scalar_type() == signature_in.scalar_type(), "grad_logsig must have same dtype as sig");
    TORCH_CHECK(grad_in.sizes() == signature_in.sizes(), "grad_logsig must match sig shape");
    same_device(signature_in, P_in, "P");
    same_device(signature_in, grad_in, "grad_logsig");
    TORCH_CHECK((int64_t)level_sizes.size() > depth, "level_sizes must have entries up to depth");
    const int64_t d = level_sizes[1];  // the channel count travels in level_sizes[1], as in the reference
    TORCH_CHECK(d >= 1, "level_sizes[1] must be >= 1 (infers path_dim)");
    c10::cuda::CUDAGuard guard(signature_in.device());
    at::Tensor sig = signature_in.contiguous(), cache = P_in.contiguous(), grad = grad_in.contiguous();
    PsigLogDesc desc = log_desc(sig, depth, d, alt, encoded_words, level_sizes);
    // The cache tells which form of the kernels produced it: S*depth scalars per row belong to the form
    // that streams through global scratch, an empty one to the row-in-shared-memory form.
    bool lead_ok = cache.dim() == sig.dim();
    for (int64_t i = 0; lead_ok && i + 1 < sig.dim(); ++i) lead_ok = cache.size(i) == sig.size(i);
    TORCH_CHECK(lead_ok && (cache.size(-1) == 0 || cache.size(-1) == sig.size(-1) * depth),
                "P must be [B,(W),S*depth] (or [B,(W),0] as returned by sig_to_logsig)");
    desc.algo = cache.size(-1) > 0 ? PSIG_ALGO_GENERIC : PSIG_ALGO_AUTO;
    TORCH_CHECK(psig_logsig_cache_size(&desc) == cache.size(-1), "P does not belong to a sig_to_logsig call with these arguments");
    at::Tensor grad_sig = at::empty_like(sig);
    const int64_t ws_bytes = psig_logsig_backward_workspace(&desc);
    check(ws_bytes, "logsig_backward");
    at::Tensor ws = at::empty({std::max<int64_t>(ws_bytes, 1)}, sig.options().dtype(at::kByte));
    check(psig_logsig_backward(&desc, ptr(sig), ptr(cache), ptr(grad), const_cast<void *>(ptr(grad_sig)), ws.data_ptr(), ws_bytes,
                               stream_of(sig)),
          "logsig_backward");
    return grad_sig;
}

PsigLogDesc projected_log_desc(const at::Tensor &sig, int64_t depth, int64_t d, const at::Tensor &top_words,
                               at::IntArrayRef level_sizes, const at::Tensor &lower_columns)
{
    PsigLogDesc desc = log_desc(sig, depth, d, true, top_words, level_sizes);
    TORCH_CHECK(lower_columns.dim() == 1 && lower_columns.scalar_type() == at::kLong, "lower_columns must be a 1D int64 tensor");
    TORCH_CHECK(lower_columns.is_cuda() && lower_columns.is_contiguous(), "lower_columns must be a contiguous CUDA tensor");
    same_device(sig, lower_columns, "lower_columns");
    desc.n_lower_columns = lower_columns.numel();
    // an empty list still selects the projected layout: any non-null pointer marks it
    static const int64_t kNoColumns = 0;
    desc.lower_columns = lower_columns.numel() > 0 ? lower_columns.data_ptr<int64_t>() : &kNoColumns;
    return desc;
}

at::Tensor logsig_projected(const at::Tensor &signature_in, int64_t depth, int64_t d, const at::Tensor &top_words,
                            at::IntArrayRef level_sizes, const at::Tensor &lower_columns)
{
    Range range("pathsig_b200::logsig_projected");
    TORCH_CHECK(signature_in.is_cuda(), "signature must be CUDA");
    c10::cuda::CUDAGuard guard(signature_in.device());
    at::Tensor sig = signature_in.contiguous();
    PsigLogDesc desc = projected_log_desc(sig, depth, d, top_words, level_sizes, lower_columns);
    const int64_t S = psig_logsig_size(&desc);
    check(S, "logsig_projected");
    TORCH_CHECK(S == sig.size(-1), "signature width ", sig.size(-1), " does not match the layout width ", S);
    const int64_t width = psig_logsig_out_size(&desc);
    check(width, "logsig_projected");
    at::Tensor out = at::empty(with_last(sig, width), sig.options());
    if (out.numel() == 0) return out;
    check(psig_logsig_forward(&desc, ptr(sig), out.data_ptr(), nullptr, stream_of(sig)), "logsig_projected");
    return out;
}

at::Tensor logsig_projected_backward(const at::Tensor &signature_in, const at::Tensor &grad_in, int64_t depth, int64_t d,
                                     const at::Tensor &top_words, at::IntArrayRef level_sizes, const at::Tensor &lower_columns)
{
    Range range("pathsig_b200::logsig_projected_backward");
    TORCH_CHECK(signature_in.is_cuda() && grad_in.is_cuda(), "signature and grad_out must be CUDA");
    TORCH_CHECK(grad_in.scalar_type() == signature_in.scalar_type(), "grad_out must have same dtype as signature");
    same_device(signature_in, grad_in, "grad_out");
    c10::cuda::CUDAGuard guard(signature_in.device());
    at::Tensor sig = signature_in.contiguous(), grad = grad_in.contiguous();
    PsigLogDesc desc = projected_log_desc(sig, depth, d, top_words, level_sizes, lower_columns);
    const int64_t width = psig_logsig_out_size(&desc);
    check(width, "logsig_projected_backward");
    TORCH_CHECK(grad.sizes().vec() == with_last(sig, width), "grad_out must be [B,(W),n_lower_columns + top_size]");
    at::Tensor grad_sig = at::empty_like(sig);
    if (grad_sig.numel() == 0) return grad_sig;
    check(psig_logsig_backward(&desc, ptr(sig), nullptr, ptr(grad), grad_sig.data_ptr(), nullptr, 0, stream_of(sig)),
          "logsig_projected_backward");
    return grad_sig;
}

PsigChenDesc chen_desc(const at::Tensor &a, const at::Tensor &b, int64_t depth, int64_t d)
{
    TORCH_CHECK(a.is_cuda() && b.is_cuda(), "signatures must be CUDA");
    TORCH_CHECK(depth >= 1 && depth <= PSIG_MAX_DEPTH, "depth must be in [1,12]");
    TORCH_CHECK(d >= 1, "d must be >= 1");
    TORCH_CHECK(a.scalar_type() == b.scalar_type(), "signatures must have the same dtype");
    same_device(a, b, "sig_b");
    TORCH_CHECK(a.sizes() == b.sizes() && a.dim() >= 1, "signatures must have the same shape (..., D)");
    const int64_t D = row_width(d, depth, false, {});
    TORCH_CHECK(a.size(-1) == D, "signature width ", a.size(-1), " is not the dense width ", D, " for d=", d, ", depth=", depth);
    PsigChenDesc desc{};
    desc.dtype = dtype_id(a);
    desc.d = (int32_t)d;
    desc.depth = (int32_t)depth;
    desc.rows = a.numel() / D;
    return desc;
}

at::Tensor chen_product(const at::Tensor &sig_a, const at::Tensor &sig_b, int64_t depth, int64_t d)
{
    Range range("pathsig_b200::chen_product");
    PsigChenDesc desc = chen_desc(sig_a, sig_b, depth, d);
    c10::cuda::CUDAGuard guard(sig_a.device());
    at::Tensor a = sig_a.contiguous(), b = sig_b.contiguous(), out = at::empty_like(a);
    if (out.numel() == 0) return out;
    check(psig_chen_forward(&desc, a.data_ptr(), b.data_ptr(), out.data_ptr(), stream_of(a)), "chen_product");
    return out;
}

std::tuple<at::Tensor, at::Tensor> chen_product_backward(const at::Tensor &sig_a, const at::Tensor &sig_b,
                                                         const at::Tensor &grad_out, int64_t depth, int64_t d)
{
    Range range("pathsig_b200::chen_product_backward");
    PsigChenDesc desc = chen_desc(sig_a, sig_b, depth, d);
    TORCH_CHECK(grad_out.is_cuda(), "grad_out must be CUDA");
    TORCH_CHECK(grad_out.scalar_type() == sig_a.scalar_type() && grad_out.sizes() == sig_a.sizes(),
                "grad_out must match the signatures in dtype and shape");
    same_device(sig_a, grad_out, "grad_out");
    c10::cuda::CUDAGuard guard(sig_a.device());
    at::Tensor a = sig_a.contiguous(), b = sig_b.contiguous(), g = grad_out.contiguous();
    at::Tensor ga = at::empty_like(a), gb = at::empty_like(a);
    if (ga.numel() == 0) return std::make_tuple(ga, gb);
    check(psig_chen_backward(&desc, a.data_ptr(), b.data_ptr(), g.data_ptr(), ga.data_ptr(), gb.data_ptr(), stream_of(a)),
          "chen_product_backward");
    return std::make_tuple(ga, gb);
}

// ---- decayed linear attention and the norm around a block (no counterpart in the reference) ----

// A wait inside a kernel that ran out leaves wrong results behind and a mark in a word of host memory; the next call of a
// sequence operator raises for it, once.  (The word is written by the devices: one page-locked integer for the process.)
void refuse_after_failure()
{
    static volatile int32_t *const flag = []() -> volatile int32_t * {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;   // the first call may stand in a capture
        if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
        void *host = nullptr, *device = nullptr;
        if (cudaHostAlloc(&host, sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess ||
            cudaHostGetDevicePointer(&device, host, 0) != cudaSuccess) {
            cudaGetLastError();
            host = nullptr;
        }
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (host == nullptr) return nullptr;
        *static_cast<volatile int32_t *>(host) = 0;
        psig_set_sequence_failure_flag(static_cast<int32_t *>(device));
        return static_cast<volatile int32_t *>(host);
    }();
    if (flag == nullptr || *flag == 0) return;
    *flag = 0;
    TORCH_CHECK(false, "a wait inside an earlier linear_attention or gated_residual_norm kernel ran out: results since then are not "
                       "valid (psig_sequence_wait_timeouts counts such waits)");
}

int sequence_dtype(const at::Tensor &t, const char *name)
{
    switch (t.scalar_type()) {
        case at::kFloat: return PSIG_F32;
        case at::kDouble: return PSIG_F64;
        case at::kBFloat16: return PSIG_BF16;
        case at::kHalf: return PSIG_F16;
        default: TORCH_CHECK(false, name, " must be float32, float64, bfloat16 or float16");
    }
}

// Type of states, decays and parameters next to operands of this type.
at::ScalarType sum_type(const at::Tensor &t) { return t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

void check_operand(const at::Tensor &anchor, const at::Tensor &t, const char *name, at::ScalarType type)
{
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == anchor.device(), name, " must be on the same device as q or x (", name, " is on ",
                t.device(), ", expected ", anchor.device(), ")");
    TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
}

// The kernels read operands through their strides; only the last dimension has to be dense.  Rows of whole 16-byte pieces are
// copied where they do not start on 16-byte boundaries (an odd offset, a broadcast dimension): that costs less than what the
// tensor-core kernels, which want this, save.
at::Tensor readable(const at::Tensor &t)
{
    if (t.size(-1) > 1 && t.stride(-1) != 1) return t.contiguous();
    const int64_t unit = 16 / t.element_size();
    if (t.size(-1) % unit != 0 || t.size(-1) > 128) return t;
    bool fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) fits = fits && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % unit == 0));
    return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

void set_strides(int64_t *to, const at::Tensor &t, bool has_time)
{
    to[0] = t.stride(0);
    to[1] = has_time ? t.stride(1) : 0;
    to[2] = t.stride(has_time ? 2 : 1);
}

// q (B, [L,] H, dk), k (B, [L,] Hkv, dk), v (B, [L,] Hkv, dv), log_decay (H) or (B, [L,] H)
PsigAttnDesc attn_desc(at::Tensor &q, at::Tensor &k, at::Tensor &v, at::Tensor &log_decay, double scale, bool has_time)
{
    const int64_t dims = has_time ? 4 : 3;
    const char *shape = has_time ? "(B, L, H, D)" : "(B, H, D)";
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    PsigAttnDesc desc{};
    desc.dtype = sequence_dtype(q, "q");
    check_operand(q, k, "k", q.scalar_type());
    check_operand(q, v, "v", q.scalar_type());
    check_operand(q, log_decay, "log_decay", sum_type(q));
    TORCH_CHECK(q.dim() == dims && k.dim() == dims && v.dim() == dims, "q, k and v must have shape ", shape);
    for (int64_t i = 0; i + 2 < dims; ++i)
        TORCH_CHECK(k.size(i) == q.size(i) && v.size(i) == q.size(i), "q, k and v must agree in all but heads and head size");
    TORCH_CHECK(k.size(-1) == q.size(-1), "k must have the head size of q");
    TORCH_CHECK(k.size(-2) == v.size(-2), "k and v must have the same number of heads");
    TORCH_CHECK(q.size(-2) >= 1 && k.size(-2) >= 1 && q.size(-2) % k.size(-2) == 0, "the number of heads of q (", q.size(-2),
                ") must be a multiple of that of k and v (", k.size(-2), ")");
    TORCH_CHECK(q.size(-1) >= 1 && q.size(-1) <= 256 && v.size(-1) >= 1 && v.size(-1) <= 256, "head sizes must be in [1,256]");
    TORCH_CHECK(q.size(-2) <= 65535, "there may be at most 65535 heads");   // before they are narrowed
    TORCH_CHECK(std::isfinite(scale), "scale must be finite");
    desc.B = q.size(0);
    desc.L = has_time ? q.size(1) : 1;
    desc.H = (int32_t)q.size(-2);
    desc.Hkv = (int32_t)k.size(-2);
    desc.dk = (int32_t)q.size(-1);
    desc.dv = (int32_t)v.size(-1);
    desc.scale = scale;
    desc.algo = g_algo.load() == PSIG_ALGO_GENERIC ? PSIG_ALGO_GENERIC : PSIG_ALGO_AUTO;
    q = readable(q), k = readable(k), v = readable(v);
    set_strides(desc.q_strides, q, has_time);
    set_strides(desc.k_strides, k, has_time);
    set_strides(desc.v_strides, v, has_time);
    log_decay = log_decay.contiguous();
    if (log_decay.dim() == 1) {
        TORCH_CHECK(log_decay.size(0) == desc.H, "log_decay must have one entry per head of q");
        desc.decay_strides[2] = 1;
    } else {
        TORCH_CHECK(log_decay.dim() == dims - 1 && log_decay.size(0) == desc.B && (!has_time || log_decay.size(1) == desc.L) &&
                    log_decay.size(-1) == desc.H, "log_decay must have shape (H) or ", has_time ? "(B, L, H)" : "(B, H)");
        desc.decay_strides[0] = desc.L * desc.H;
        desc.decay_strides[1] = has_time ? desc.H : 0;
        desc.decay_strides[2] = 1;
    }
    return desc;
}

void check_state(const PsigAttnDesc &desc, const at::Tensor &q, const at::Tensor &t, const char *name)
{
    check_operand(q, t, name, sum_type(q));
    TORCH_CHECK(t.dim() == 4 && t.size(0) == desc.B && t.size(1) == desc.H && t.size(2) == desc.dk && t.size(3) == desc.dv, name,
                " must have shape (B, H, Dk, Dv)");
}

at::Tensor sequence_lengths(const PsigAttnDesc &desc, const at::Tensor &q, const std::optional<at::Tensor> &lengths)
{
    if (!lengths.has_value()) return at::Tensor();
    TORCH_CHECK(lengths->is_cuda() && lengths->device() == q.device(), "lengths must be on the same device as q");
    TORCH_CHECK(lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong, "lengths must be int32 or int64");
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == desc.B, "lengths must have shape (B)");
    // clamped before the narrowing, so that no 64-bit value wraps into the valid range
    return (lengths->scalar_type() == at::kLong ? lengths->clamp(0, desc.L).to(at::kInt) : *lengths).contiguous();
}

std::tuple<at::Tensor, at::Tensor> linear_attention(const at::Tensor &q_in, const at::Tensor &k_in, const at::Tensor &v_in,
                                                    const at::Tensor &log_decay_in, const std::optional<at::Tensor> &initial_state,
                                                    const std::optional<at::Tensor> &lengths_in, double scale, bool return_state)
{
    Range range("pathsig_b200::linear_attention");
    TORCH_CHECK(q_in.is_cuda(), "q must be a CUDA tensor");
    c10::cuda::CUDAGuard guard(q_in.device());
    refuse_after_failure();
    at::Tensor q = q_in, k = k_in, v = v_in, decay = log_decay_in;
    PsigAttnDesc desc = attn_desc(q, k, v, decay, scale, true);
    at::Tensor init;
    if (initial_state.has_value()) {
        check_state(desc, q, *initial_state, "initial_state");
        init = initial_state->contiguous();
    }
    at::Tensor lengths = sequence_lengths(desc, q, lengths_in);
    desc.lengths = lengths.defined() && lengths.numel() > 0 ? lengths.data_ptr<int32_t>() : nullptr;
    at::Tensor out = at::empty({desc.B, desc.L, desc.H, desc.dv}, q.options());
    at::Tensor final = return_state ? at::empty({desc.B, desc.H, desc.dk, desc.dv}, decay.options())
                                    : at::empty({0}, decay.options());
    if (desc.B == 0) return std::make_tuple(out, final);
    if (desc.L == 0) {
        if (return_state) init.defined() ? final.copy_(init) : final.zero_();
        return std::make_tuple(out, final);
    }
    const int64_t ws_bytes = psig_attn_forward_workspace(&desc);
    check(ws_bytes, "linear_attention");
    at::Tensor ws = at::empty({ws_bytes}, q.options().dtype(at::kByte));
    check(psig_attn_forward(&desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), init.defined() ? init.data_ptr() : nullptr,
                            out.data_ptr(), return_state ? final.data_ptr() : nullptr, ws_bytes > 0 ? ws.data_ptr() : nullptr,
                            ws_bytes, stream_of(q)),
          "linear_attention");
    return std::make_tuple(out, final);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> linear_attention_backward(
    const at::Tensor &q_in, const at::Tensor &k_in, const at::Tensor &v_in, const at::Tensor &log_decay_in,
    const std::optional<at::Tensor> &initial_state, const std::optional<at::Tensor> &lengths_in,
    const std::optional<at::Tensor> &grad_out, const std::optional<at::Tensor> &grad_state, double scale, bool decay_grad)
{
    Range range("pathsig_b200::linear_attention_backward");
    TORCH_CHECK(q_in.is_cuda(), "q must be a CUDA tensor");
    c10::cuda::CUDAGuard guard(q_in.device());
    refuse_after_failure();
    at::Tensor q = q_in, k = k_in, v = v_in, decay = log_decay_in;
    PsigAttnDesc desc = attn_desc(q, k, v, decay, scale, true);
    at::Tensor init, go, gs;
    if (initial_state.has_value()) {
        check_state(desc, q, *initial_state, "initial_state");
        init = initial_state->contiguous();
    }
    if (grad_out.has_value()) {
        check_operand(q, *grad_out, "grad_out", q.scalar_type());
        TORCH_CHECK(grad_out->dim() == 4 && grad_out->size(0) == desc.B && grad_out->size(1) == desc.L &&
                    grad_out->size(2) == desc.H && grad_out->size(3) == desc.dv, "grad_out must have the shape of the output");
        go = readable(grad_out->contiguous());
    } else {
        go = at::zeros({desc.B, desc.L, desc.H, desc.dv}, q.options());
    }
    if (grad_state.has_value()) {
        check_state(desc, q, *grad_state, "grad_state");
        gs = grad_state->contiguous();
    }
    at::Tensor lengths = sequence_lengths(desc, q, lengths_in);
    desc.lengths = lengths.defined() && lengths.numel() > 0 ? lengths.data_ptr<int32_t>() : nullptr;
    at::Tensor gq = at::empty(q.sizes(), q.options()), gk = at::empty(k.sizes(), q.options()), gv = at::empty(v.sizes(), q.options());
    at::Tensor gd = decay_grad ? at::empty(decay.sizes(), decay.options()) : at::empty({0}, decay.options());
    at::Tensor gi = init.defined() ? at::empty(init.sizes(), init.options()) : at::empty({0}, decay.options());
    if (desc.B == 0 || desc.L == 0) {
        gd.zero_();
        if (init.defined()) gs.defined() ? gi.copy_(gs) : gi.zero_();
        return std::make_tuple(gq, gk, gv, gd, gi);
    }
    const int64_t ws_bytes = psig_attn_backward_workspace(&desc);
    check(ws_bytes, "linear_attention_backward");
    at::Tensor ws = at::empty({ws_bytes}, q.options().dtype(at::kByte));
    check(psig_attn_backward(&desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), init.defined() ? init.data_ptr() : nullptr,
                             go.data_ptr(), gs.defined() ? gs.data_ptr() : nullptr, gq.data_ptr(), gk.data_ptr(), gv.data_ptr(),
                             decay_grad ? gd.data_ptr() : nullptr, init.defined() ? gi.data_ptr() : nullptr,
                             ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes, stream_of(q)),
          "linear_attention_backward");
    return std::make_tuple(gq, gk, gv, gd, gi);
}

at::Tensor linear_attention_step(const at::Tensor &q_in, const at::Tensor &k_in, const at::Tensor &v_in,
                                 const at::Tensor &log_decay_in, at::Tensor &state, double scale)
{
    Range range("pathsig_b200::linear_attention_step");
    TORCH_CHECK(q_in.is_cuda(), "q must be a CUDA tensor");
    c10::cuda::CUDAGuard guard(q_in.device());
    refuse_after_failure();
    at::Tensor q = q_in, k = k_in, v = v_in, decay = log_decay_in;
    PsigAttnDesc desc = attn_desc(q, k, v, decay, scale, false);
    check_state(desc, q, state, "state");
    TORCH_CHECK(state.is_contiguous(), "state must be contiguous: it is updated in place");
    for (const at::Tensor *t : {&q_in, &k_in, &v_in, &log_decay_in})
        TORCH_CHECK(!t->is_alias_of(state), "state must not share memory with the other operands: it is updated in place");
    at::Tensor out = at::empty({desc.B, desc.H, desc.dv}, q.options());
    if (desc.B == 0) return out;
    check(psig_attn_step(&desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), state.data_ptr(), out.data_ptr(),
                         stream_of(q)),
          "linear_attention_step");
    return out;
}

// Operands of the norm, checked and contiguous; undefined where they are left out.
struct NormOperands {
    PsigNormDesc desc{};
    at::Tensor x, weight, gate, residual, scale, next;
};

const void *data_or_null(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

NormOperands norm_operands(const at::Tensor &x, const std::optional<at::Tensor> &weight, const std::optional<at::Tensor> &gate,
                           const std::optional<at::Tensor> &residual, const std::optional<at::Tensor> &residual_scale,
                           const std::optional<at::Tensor> &next_weight, int64_t activation, double eps)
{
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "x must have shape (..., D) with D >= 1");
    TORCH_CHECK(activation == 0 || activation == 1, "activation must be 0 (silu) or 1 (sigmoid)");
    TORCH_CHECK(std::isfinite(eps) && eps >= 0, "eps must be finite and not negative");
    NormOperands n;
    n.desc.dtype = sequence_dtype(x, "x");
    n.desc.activation = (int32_t)activation;
    n.desc.D = x.size(-1);
    n.desc.rows = x.numel() / x.size(-1);
    n.desc.eps = eps;
    n.x = x.contiguous();
    auto rows = [&](const std::optional<at::Tensor> &t, const char *name, at::Tensor *to) {
        if (!t.has_value()) return;
        check_operand(x, *t, name, x.scalar_type());
        TORCH_CHECK(t->sizes() == x.sizes(), name, " must have the shape of x");
        *to = t->contiguous();
    };
    auto vector = [&](const std::optional<at::Tensor> &t, const char *name, at::Tensor *to) {
        if (!t.has_value()) return;
        check_operand(x, *t, name, sum_type(x));
        TORCH_CHECK(t->dim() == 1 && t->size(0) == n.desc.D, name, " must have shape (D)");
        *to = t->contiguous();
    };
    rows(gate, "gate", &n.gate);
    rows(residual, "residual", &n.residual);
    vector(weight, "weight", &n.weight);
    vector(residual_scale, "residual_scale", &n.scale);
    vector(next_weight, "next_weight", &n.next);
    return n;
}

std::tuple<at::Tensor, at::Tensor> gated_residual_norm(const at::Tensor &x, const std::optional<at::Tensor> &weight,
                                                       const std::optional<at::Tensor> &gate, const std::optional<at::Tensor> &residual,
                                                       const std::optional<at::Tensor> &residual_scale,
                                                       const std::optional<at::Tensor> &next_weight, int64_t activation, double eps)
{
    Range range("pathsig_b200::gated_residual_norm");
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    c10::cuda::CUDAGuard guard(x.device());
    refuse_after_failure();
    NormOperands o = norm_operands(x, weight, gate, residual, residual_scale, next_weight, activation, eps);
    at::Tensor h = at::empty(x.sizes(), x.options());
    at::Tensor n = o.next.defined() ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options());
    if (o.desc.rows == 0) return std::make_tuple(h, n);
    check(psig_norm_forward(&o.desc, o.x.data_ptr(), data_or_null(o.weight), data_or_null(o.gate), data_or_null(o.residual),
                            data_or_null(o.scale), data_or_null(o.next), h.data_ptr(), o.next.defined() ? n.data_ptr() : nullptr,
                            stream_of(x)),
          "gated_residual_norm");
    return std::make_tuple(h, n);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> gated_residual_norm_backward(
    const at::Tensor &x, const std::optional<at::Tensor> &weight, const std::optional<at::Tensor> &gate,
    const std::optional<at::Tensor> &residual, const std::optional<at::Tensor> &residual_scale,
    const std::optional<at::Tensor> &next_weight, const std::optional<at::Tensor> &grad_h_in,
    const std::optional<at::Tensor> &grad_n_in, int64_t activation, double eps)
{
    Range range("pathsig_b200::gated_residual_norm_backward");
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    c10::cuda::CUDAGuard guard(x.device());
    refuse_after_failure();
    NormOperands o = norm_operands(x, weight, gate, residual, residual_scale, next_weight, activation, eps);
    at::Tensor grad_h, grad_n;
    for (auto [t, name, to] : {std::make_tuple(&grad_h_in, "grad_h", &grad_h), std::make_tuple(&grad_n_in, "grad_n", &grad_n)}) {
        if (!t->has_value()) continue;
        check_operand(x, **t, name, x.scalar_type());
        TORCH_CHECK((*t)->sizes() == x.sizes(), name, " must have the shape of x");
        *to = (*t)->contiguous();
    }
    if (o.next.defined() && !grad_n.defined()) grad_n = at::zeros(x.sizes(), x.options());
    auto like = [&](const at::Tensor &t) { return t.defined() ? at::empty(t.sizes(), t.options()) : at::empty({0}, x.options()); };
    at::Tensor gx = at::empty(x.sizes(), x.options()), gw = like(o.weight), gg = like(o.gate), gr = like(o.residual),
               gs = like(o.scale), gn = like(o.next);
    if (o.desc.rows == 0) {
        for (at::Tensor *t : {&gw, &gs, &gn}) t->zero_();
        return std::make_tuple(gx, gw, gg, gr, gs, gn);
    }
    const int64_t ws_bytes = psig_norm_backward_workspace(&o.desc);
    check(ws_bytes, "gated_residual_norm_backward");
    at::Tensor ws = at::empty({ws_bytes}, x.options().dtype(at::kByte));
    auto to = [](const at::Tensor &operand, at::Tensor &grad) { return operand.defined() ? grad.data_ptr() : nullptr; };
    check(psig_norm_backward(&o.desc, o.x.data_ptr(), data_or_null(o.weight), data_or_null(o.gate), data_or_null(o.residual),
                             data_or_null(o.scale), data_or_null(o.next), data_or_null(grad_h), data_or_null(grad_n), gx.data_ptr(),
                             to(o.weight, gw), to(o.gate, gg), to(o.residual, gr), to(o.scale, gs), to(o.next, gn), ws.data_ptr(),
                             ws_bytes, stream_of(x)),
          "gated_residual_norm_backward");
    return std::make_tuple(gx, gw, gg, gr, gs, gn);
}

// ---- autograd of the sequence operators ----
//
// In C++ because their small calls (one row, one window) are bound by the host: the formulas registered from Python
// cost 150-250 us for a forward and backward pass (8 us here is a whole step of a kept state).

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using OptionalTensor = std::optional<at::Tensor>;

OptionalTensor given(const Variable &t) { return t.defined() ? OptionalTensor(t) : std::nullopt; }
Variable plain(const OptionalTensor &t) { return t.has_value() ? *t : Variable(); }
bool tracked(const OptionalTensor &t) { return t.has_value() && t->defined() && t->requires_grad(); }

// Forward-mode tangents are refused: an operand that has one may not require a gradient, and would pass by the functions below.
template <typename... Operands>
void refuse_tangents(const char *name, const Operands &...operands)
{
    auto has = [](const at::Tensor &t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); };
    auto any = [&](const auto &t) {
        if constexpr (std::is_same_v<std::decay_t<decltype(t)>, OptionalTensor>) return t.has_value() && has(*t);
        else return has(t);
    };
    TORCH_CHECK(!(any(operands) || ...), name, " has no forward-mode derivative: an operand has a tangent");
}

template <typename Fn>
c10::TypedOperatorHandle<Fn> handle(const char *name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();
}

std::tuple<at::Tensor, at::Tensor> attention_below(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                                                   const at::Tensor &decay, const OptionalTensor &init,
                                                   const OptionalTensor &lengths, double scale, bool return_state)
{
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(linear_attention)>("pathsig_b200::linear_attention");
    return op.call(q, k, v, decay, init, lengths, scale, return_state);
}

// The gradients' own gradients are refused (torch would warn and leave them out).
using AttentionGrads = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

AttentionGrads attention_backward_below(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &decay,
                                        const OptionalTensor &init, const OptionalTensor &lengths, const OptionalTensor &go,
                                        const OptionalTensor &gs, double scale, bool decay_grad)
{
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(linear_attention_backward)>("pathsig_b200::linear_attention_backward");
    return op.call(q, k, v, decay, init, lengths, go, gs, scale, decay_grad);
}

struct AttentionGradsFunction : torch::autograd::Function<AttentionGradsFunction> {
    static variable_list forward(AutogradContext *, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                                 const at::Tensor &decay, const OptionalTensor &init, const OptionalTensor &lengths,
                                 const OptionalTensor &go, const OptionalTensor &gs, double scale, bool decay_grad)
    {
        auto [gq, gk, gv, gd, gi] = attention_backward_below(q, k, v, decay, init, lengths, go, gs, scale, decay_grad);
        return {gq, gk, gv, gd, gi};
    }
    static variable_list backward(AutogradContext *, variable_list)
    {
        TORCH_CHECK(false, "linear_attention is differentiable once: its gradients have no gradient");
    }
};

AttentionGrads linear_attention_backward_autograd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                                                  const at::Tensor &decay, const OptionalTensor &init,
                                                  const OptionalTensor &lengths, const OptionalTensor &go,
                                                  const OptionalTensor &gs, double scale, bool decay_grad)
{
    refuse_tangents("linear_attention_backward", q, k, v, decay, init, go, gs);
    if (!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad() || decay.requires_grad() ||
                                         tracked(init) || tracked(go) || tracked(gs)))
        return attention_backward_below(q, k, v, decay, init, lengths, go, gs, scale, decay_grad);
    variable_list g = AttentionGradsFunction::apply(q, k, v, decay, init, lengths, go, gs, scale, decay_grad);
    return std::make_tuple(g[0], g[1], g[2], g[3], g[4]);
}

struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                                 const at::Tensor &decay, const OptionalTensor &init, const OptionalTensor &lengths, double scale,
                                 bool return_state)
    {
        auto [out, state] = attention_below(q, k, v, decay, init, lengths, scale, return_state);
        ctx->save_for_backward({q, k, v, decay, plain(init), plain(lengths)});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["state"] = return_state;
        ctx->saved_data["decay"] = decay.requires_grad();
        ctx->set_materialize_grads(false);
        return {out, state};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        variable_list none(8);
        if (!ctx->saved_data["state"].toBool()) grads[1] = Variable();
        if (!grads[0].defined() && !grads[1].defined()) return none;
        const variable_list s = ctx->get_saved_variables();
        static const auto op = handle<decltype(linear_attention_backward)>("pathsig_b200::linear_attention_backward");
        const bool decay_grad = ctx->saved_data["decay"].toBool();
        auto [gq, gk, gv, gd, gi] = op.call(s[0], s[1], s[2], s[3], given(s[4]), given(s[5]), given(grads[0]), given(grads[1]),
                                            ctx->saved_data["scale"].toDouble(), decay_grad);
        none[0] = gq, none[1] = gk, none[2] = gv;
        if (decay_grad) none[3] = gd;
        if (s[4].defined()) none[4] = gi;
        return none;
    }
};

std::tuple<at::Tensor, at::Tensor> linear_attention_autograd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                                                             const at::Tensor &decay, const OptionalTensor &init,
                                                             const OptionalTensor &lengths, double scale, bool return_state)
{
    refuse_tangents("linear_attention", q, k, v, decay, init);
    if (!at::GradMode::is_enabled() ||
        !(q.requires_grad() || k.requires_grad() || v.requires_grad() || decay.requires_grad() || tracked(init)))
        return attention_below(q, k, v, decay, init, lengths, scale, return_state);
    variable_list got = AttentionFunction::apply(q, k, v, decay, init, lengths, scale, return_state);
    return std::make_tuple(got[0], got[1]);
}

// The step changes its state in place: the state's version says so to graphs that have saved it, which then refuse to run
// (the schema alone does not).  Tensors made in inference mode have no version.
at::Tensor linear_attention_step_in_place(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &decay,
                                          at::Tensor &state, double scale)
{
    refuse_tangents("linear_attention_step", q, k, v, decay, state);
    at::Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op = handle<decltype(linear_attention_step)>("pathsig_b200::linear_attention_step");
        out = op.call(q, k, v, decay, state, scale);
    }
    if (!state.is_inference()) torch::autograd::increment_version(state);
    return out;
}

std::tuple<at::Tensor, at::Tensor> norm_below(const at::Tensor &x, const OptionalTensor &weight, const OptionalTensor &gate,
                                              const OptionalTensor &residual, const OptionalTensor &residual_scale,
                                              const OptionalTensor &next_weight, int64_t activation, double eps)
{
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(gated_residual_norm)>("pathsig_b200::gated_residual_norm");
    return op.call(x, weight, gate, residual, residual_scale, next_weight, activation, eps);
}

using NormGrads = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

NormGrads norm_backward_below(const at::Tensor &x, const OptionalTensor &weight, const OptionalTensor &gate,
                              const OptionalTensor &residual, const OptionalTensor &residual_scale,
                              const OptionalTensor &next_weight, const OptionalTensor &grad_h, const OptionalTensor &grad_n,
                              int64_t activation, double eps)
{
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(gated_residual_norm_backward)>("pathsig_b200::gated_residual_norm_backward");
    return op.call(x, weight, gate, residual, residual_scale, next_weight, grad_h, grad_n, activation, eps);
}

struct NormGradsFunction : torch::autograd::Function<NormGradsFunction> {
    static variable_list forward(AutogradContext *, const at::Tensor &x, const OptionalTensor &weight, const OptionalTensor &gate,
                                 const OptionalTensor &residual, const OptionalTensor &residual_scale,
                                 const OptionalTensor &next_weight, const OptionalTensor &grad_h, const OptionalTensor &grad_n,
                                 int64_t activation, double eps)
    {
        auto [gx, gw, gg, gr, gs, gn] =
            norm_backward_below(x, weight, gate, residual, residual_scale, next_weight, grad_h, grad_n, activation, eps);
        return {gx, gw, gg, gr, gs, gn};
    }
    static variable_list backward(AutogradContext *, variable_list)
    {
        TORCH_CHECK(false, "gated_residual_norm is differentiable once: its gradients have no gradient");
    }
};

NormGrads gated_residual_norm_backward_autograd(const at::Tensor &x, const OptionalTensor &weight, const OptionalTensor &gate,
                                                const OptionalTensor &residual, const OptionalTensor &residual_scale,
                                                const OptionalTensor &next_weight, const OptionalTensor &grad_h,
                                                const OptionalTensor &grad_n, int64_t activation, double eps)
{
    refuse_tangents("gated_residual_norm_backward", x, weight, gate, residual, residual_scale, next_weight, grad_h, grad_n);
    if (!at::GradMode::is_enabled() || !(x.requires_grad() || tracked(weight) || tracked(gate) || tracked(residual) ||
                                         tracked(residual_scale) || tracked(next_weight) || tracked(grad_h) || tracked(grad_n)))
        return norm_backward_below(x, weight, gate, residual, residual_scale, next_weight, grad_h, grad_n, activation, eps);
    variable_list g =
        NormGradsFunction::apply(x, weight, gate, residual, residual_scale, next_weight, grad_h, grad_n, activation, eps);
    return std::make_tuple(g[0], g[1], g[2], g[3], g[4], g[5]);
}

struct NormFunction : torch::autograd::Function<NormFunction> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const OptionalTensor &weight, const OptionalTensor &gate,
                                 const OptionalTensor &residual, const OptionalTensor &residual_scale,
                                 const OptionalTensor &next_weight, int64_t activation, double eps)
    {
        auto [h, n] = norm_below(x, weight, gate, residual, residual_scale, next_weight, activation, eps);
        ctx->save_for_backward({x, plain(weight), plain(gate), plain(residual), plain(residual_scale), plain(next_weight)});
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        return {h, n};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        variable_list none(8);
        const variable_list s = ctx->get_saved_variables();
        if (!s[5].defined()) grads[1] = Variable();
        if (!grads[0].defined() && !grads[1].defined()) return none;
        static const auto op = handle<decltype(gated_residual_norm_backward)>("pathsig_b200::gated_residual_norm_backward");
        auto [gx, gw, gg, gr, gs, gn] =
            op.call(s[0], given(s[1]), given(s[2]), given(s[3]), given(s[4]), given(s[5]), given(grads[0]), given(grads[1]),
                    ctx->saved_data["activation"].toInt(), ctx->saved_data["eps"].toDouble());
        const at::Tensor *got[6] = {&gx, &gw, &gg, &gr, &gs, &gn};
        for (int i = 0; i < 6; ++i)
            if (s[i].defined()) none[i] = *got[i];
        return none;
    }
};

std::tuple<at::Tensor, at::Tensor> gated_residual_norm_autograd(const at::Tensor &x, const OptionalTensor &weight,
                                                                const OptionalTensor &gate, const OptionalTensor &residual,
                                                                const OptionalTensor &residual_scale, const OptionalTensor &next_weight,
                                                                int64_t activation, double eps)
{
    refuse_tangents("gated_residual_norm", x, weight, gate, residual, residual_scale, next_weight);
    if (!at::GradMode::is_enabled() || !(x.requires_grad() || tracked(weight) || tracked(gate) || tracked(residual) ||
                                         tracked(residual_scale) || tracked(next_weight)))
        return norm_below(x, weight, gate, residual, residual_scale, next_weight, activation, eps);
    variable_list got = NormFunction::apply(x, weight, gate, residual, residual_scale, next_weight, activation, eps);
    return std::make_tuple(got[0], got[1]);
}

}  // namespace

// Kernel family used by the signature operators (PsigAlgo); tests flip it to compare families.
extern "C" void psig_torch_set_algorithm(int algo) { g_algo.store(algo); }
extern "C" int psig_torch_get_algorithm(void) { return g_algo.load(); }

TORCH_LIBRARY(pathsig_b200, m)
{
    const auto tag = at::Tag::pt2_compliant_tag;
    m.set_python_module("pathsig_b200.ops");  // where the fake implementations and autograd formulas live
    m.def("compute_signature(Tensor path_in, int depth, bool alternative_projection, Tensor encoded_words, "
          "int[] level_sizes, bool use_windows, Tensor windows) -> Tensor", {tag});
    m.def("signature_backward(Tensor path_in, Tensor signature_in, Tensor grad_signature_in, int depth, "
          "bool alternative_projection, Tensor encoded_words, int[] level_sizes, bool use_windows, Tensor windows) -> Tensor", {tag});
    m.def("sig_to_logsig(Tensor signature_in, int depth, int d, bool alternative_projection, Tensor encoded_words, "
          "int[] level_sizes) -> (Tensor, Tensor)", {tag});
    m.def("logsig_backward(Tensor signature_in, Tensor P_in, Tensor grad_logsig_in, int depth, "
          "bool alternative_projection, Tensor encoded_words, int[] level_sizes) -> Tensor", {tag});
    m.def("logsig_projected(Tensor signature_in, int depth, int d, Tensor top_words, int[] level_sizes, "
          "Tensor lower_columns) -> Tensor", {tag});
    m.def("logsig_projected_backward(Tensor signature_in, Tensor grad_out, int depth, int d, Tensor top_words, "
          "int[] level_sizes, Tensor lower_columns) -> Tensor", {tag});
    m.def("chen_product(Tensor sig_a, Tensor sig_b, int depth, int d) -> Tensor", {tag});
    m.def("chen_product_backward(Tensor sig_a, Tensor sig_b, Tensor grad_out, int depth, int d) -> (Tensor, Tensor)", {tag});
    m.def("linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? initial_state, Tensor? lengths, "
          "float scale, bool return_state) -> (Tensor, Tensor)", {tag});
    m.def("linear_attention_backward(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? initial_state, Tensor? lengths, "
          "Tensor? grad_out, Tensor? grad_state, float scale, bool decay_grad) -> (Tensor, Tensor, Tensor, Tensor, Tensor)", {tag});
    m.def("linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, float scale) -> Tensor", {tag});
    m.def("gated_residual_norm(Tensor x, Tensor? weight, Tensor? gate, Tensor? residual, Tensor? residual_scale, "
          "Tensor? next_weight, int activation, float eps) -> (Tensor, Tensor)", {tag});
    m.def("gated_residual_norm_backward(Tensor x, Tensor? weight, Tensor? gate, Tensor? residual, Tensor? residual_scale, "
          "Tensor? next_weight, Tensor? grad_h, Tensor? grad_n, int activation, float eps) "
          "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)", {tag});
}

TORCH_LIBRARY_IMPL(pathsig_b200, CUDA, m)
{
    m.impl("compute_signature", &compute_signature);
    m.impl("signature_backward", &signature_backward);
    m.impl("sig_to_logsig", &sig_to_logsig);
    m.impl("logsig_backward", &logsig_backward);
    m.impl("logsig_projected", &logsig_projected);
    m.impl("logsig_projected_backward", &logsig_projected_backward);
    m.impl("chen_product", &chen_product);
    m.impl("chen_product_backward", &chen_product_backward);
    m.impl("linear_attention", &linear_attention);
    m.impl("linear_attention_backward", &linear_attention_backward);
    m.impl("linear_attention_step", &linear_attention_step);
    m.impl("gated_residual_norm", &gated_residual_norm);
    m.impl("gated_residual_norm_backward", &gated_residual_norm_backward);
}

TORCH_LIBRARY_IMPL(pathsig_b200, ADInplaceOrView, m)
{
    m.impl("linear_attention_step", &linear_attention_step_in_place);
}

TORCH_LIBRARY_IMPL(pathsig_b200, Autograd, m)
{
    m.impl("linear_attention", &linear_attention_autograd);
    m.impl("linear_attention_backward", &linear_attention_backward_autograd);
    m.impl("gated_residual_norm", &gated_residual_norm_autograd);
    m.impl("gated_residual_norm_backward", &gated_residual_norm_backward_autograd);
}
