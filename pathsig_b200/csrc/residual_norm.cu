// Norm around a block, fused with the block's gate, the residual sum and the norm before the next block.
//     z = x r w,  r = (mean(x^2) + eps)^(-1/2);   u = z act(gate);   h = residual + c u;
//     n = h r2 w2,  r2 = (mean(h^2) + eps)^(-1/2)
// Backward, per row, with the total gradient of h first:
//     dh += r2 (w2 dn) - h r2^3 mean(w2 dn h)            dw2 += dn h r2
//     dresidual = dh,  dc += dh u,  dgate = dh c z act'(gate),  dz = dh c act(gate),  dw += dz x r
//     dx = r (w dz) - x r^3 mean(w dz x)
// h is recomputed from the operands (the residual is read where a saved h would have been), so that nothing of
// the forward pass is kept and h is not rounded in between.  Sums are in 32 bits (64 for float64).
#include "sequence.cuh"

namespace psig {
namespace {

constexpr int kNormThreads = 256;

struct NormArgs {
    const void *x, *gate, *residual, *grad_h, *grad_n;
    const void *weight, *scale, *next_weight;
    void *h, *n;
    void *grad_x, *grad_gate, *grad_residual;
    void *partial;   // (blocks, 3, D) sums for weight, scale, next_weight
    long long rows, D;
    double eps;
    int activation;
};

template <typename A>
__device__ __forceinline__ A block_sum(A v, A *shared)
{
    for (int s = 16; s >= 1; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    A sum = A(0);
    for (int i = 0; i < kNormThreads / 32; ++i) sum += shared[i];
    return sum;
}

// act(g) and its derivative
template <typename A>
__device__ __forceinline__ A gate_value(A g, int activation, A *slope)
{
    const A s = A(1) / (A(1) + exp_acc(-g));
    *slope = activation == 0 ? s * (A(1) + g * (A(1) - s)) : s * (A(1) - s);
    return activation == 0 ? g * s : s;
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_forward_rows(const NormArgs a)
{
    using A = typename Acc<T>::type;
    __shared__ A shared[kNormThreads / 32];
    const A *w = static_cast<const A *>(a.weight), *c = static_cast<const A *>(a.scale);
    const A *w2 = static_cast<const A *>(a.next_weight);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.D;
        const T *gate = a.gate ? static_cast<const T *>(a.gate) + row * a.D : nullptr;
        const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.D : nullptr;
        T *h = static_cast<T *>(a.h) + row * a.D;
        A sum = A(0);
        for (long long i = threadIdx.x; i < a.D; i += kNormThreads) { const A v = to_acc<A>(x[i]); sum += v * v; }
        const A r = A(1) / sqrt(block_sum(sum, shared) / A(a.D) + A(a.eps));
        auto value = [&](long long i) {
            A v = to_acc<A>(x[i]) * r, slope;
            if (w) v *= w[i];
            if (gate) v *= gate_value(to_acc<A>(gate[i]), a.activation, &slope);
            if (c) v *= c[i];
            return res ? to_acc<A>(res[i]) + v : v;
        };
        sum = A(0);
        for (long long i = threadIdx.x; i < a.D; i += kNormThreads) {
            const A v = value(i);
            sum += v * v;
            h[i] = from_acc<T>(v);
        }
        if (w2 == nullptr) continue;
        const A r2 = A(1) / sqrt(block_sum(sum, shared) / A(a.D) + A(a.eps));
        for (long long i = threadIdx.x; i < a.D; i += kNormThreads)
            static_cast<T *>(a.n)[row * a.D + i] = from_acc<T>(value(i) * r2 * w2[i]);
    }
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_backward_rows(const NormArgs a)
{
    using A = typename Acc<T>::type;
    __shared__ A shared[kNormThreads / 32];
    const A *w = static_cast<const A *>(a.weight), *c = static_cast<const A *>(a.scale);
    const A *w2 = static_cast<const A *>(a.next_weight);
    A *part = static_cast<A *>(a.partial) + (long long)blockIdx.x * 3 * a.D;
    for (long long i = threadIdx.x; i < 3 * a.D; i += kNormThreads) part[i] = A(0);
    __syncthreads();
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.D;
        const T *gate = a.gate ? static_cast<const T *>(a.gate) + row * a.D : nullptr;
        const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.D : nullptr;
        const T *gh = a.grad_h ? static_cast<const T *>(a.grad_h) + row * a.D : nullptr;
        const T *gn = w2 ? static_cast<const T *>(a.grad_n) + row * a.D : nullptr;
        A sum = A(0);
        for (long long i = threadIdx.x; i < a.D; i += kNormThreads) { const A v = to_acc<A>(x[i]); sum += v * v; }
        const A r = A(1) / sqrt(block_sum(sum, shared) / A(a.D) + A(a.eps));
        A r2 = A(0), m2 = A(0);
        auto value = [&](long long i) {
            A v = to_acc<A>(x[i]) * r, slope;
            if (w) v *= w[i];
            if (gate) v *= gate_value(to_acc<A>(gate[i]), a.activation, &slope);
            if (c) v *= c[i];
            return res ? to_acc<A>(res[i]) + v : v;
        };
        if (w2) {
            A hh = A(0), nh = A(0);
            for (long long i = threadIdx.x; i < a.D; i += kNormThreads) {
                const A v = value(i);
                hh += v * v;
                nh += w2[i] * to_acc<A>(gn[i]) * v;
            }
            r2 = A(1) / sqrt(block_sum(hh, shared) / A(a.D) + A(a.eps));
            m2 = block_sum(nh, shared) / A(a.D) * r2 * r2 * r2;
        }
        auto total = [&](long long i) {   // gradient of h
            A v = gh ? to_acc<A>(gh[i]) : A(0);
            if (w2) v += w2[i] * to_acc<A>(gn[i]) * r2 - value(i) * m2;
            return v;
        };
        sum = A(0);
        for (long long i = threadIdx.x; i < a.D; i += kNormThreads) {
            const A dh = total(i), xv = to_acc<A>(x[i]), ci = c ? c[i] : A(1), wi = w ? w[i] : A(1);
            A slope = A(0), act = A(1);
            if (gate) act = gate_value(to_acc<A>(gate[i]), a.activation, &slope);
            const A z = xv * r * wi, dz = dh * ci * act;
            if (w2) part[2 * a.D + i] += to_acc<A>(gn[i]) * value(i) * r2;
            part[a.D + i] += dh * z * act;
            part[i] += dz * xv * r;
            if (a.grad_residual) static_cast<T *>(a.grad_residual)[row * a.D + i] = from_acc<T>(dh);
            if (a.grad_gate) static_cast<T *>(a.grad_gate)[row * a.D + i] = from_acc<T>(dh * ci * z * slope);
            sum += wi * dz * xv;
        }
        const A m = block_sum(sum, shared) / A(a.D) * r * r * r;
        if (a.grad_x)
            for (long long i = threadIdx.x; i < a.D; i += kNormThreads) {
                const A dh = total(i), ci = c ? c[i] : A(1), wi = w ? w[i] : A(1);
                A slope, act = A(1);
                if (gate) act = gate_value(to_acc<A>(gate[i]), a.activation, &slope);
                static_cast<T *>(a.grad_x)[row * a.D + i] = from_acc<T>(r * wi * dh * ci * act - to_acc<A>(x[i]) * m);
            }
    }
}

// Sums of the blocks' partial rows, in a fixed order.
template <typename A>
__global__ void norm_sum_partials(const A *__restrict__ partial, int blocks, long long D, A *__restrict__ out_w,
                                  A *__restrict__ out_c, A *__restrict__ out_w2)
{
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= 3 * D) return;
    A *out = i < D ? out_w : i < 2 * D ? out_c : out_w2;
    if (out == nullptr) return;
    A sum = A(0);
    for (int b = 0; b < blocks; ++b) sum += partial[(long long)b * 3 * D + i];
    out[i % D] = sum;
}

int check_norm(const PsigNormDesc *d)
{
    if (d == nullptr) return PSIG_ERR_NULL;
    if (d->dtype < PSIG_F32 || d->dtype > PSIG_F16) return PSIG_ERR_DTYPE;
    if (d->rows < 0 || d->D < 1 || d->activation < 0 || d->activation > 1) return PSIG_ERR_SHAPE;
    return PSIG_OK;
}

int backward_blocks(const PsigNormDesc &d) { return (int)(d.rows < 148 * 4 ? d.rows : 148 * 4); }

}  // namespace
}  // namespace psig

using namespace psig;

extern "C" int psig_norm_forward(const PsigNormDesc *desc, const void *x, const void *weight, const void *gate,
                                 const void *residual, const void *residual_scale, const void *next_weight, void *h,
                                 void *n, void *stream)
{
    const int rc = check_norm(desc);
    if (rc != PSIG_OK) return rc;
    if (desc->rows == 0) return PSIG_OK;
    if (x == nullptr || h == nullptr || (next_weight != nullptr && n == nullptr)) return PSIG_ERR_NULL;
    NormArgs a{};
    a.x = x, a.weight = weight, a.gate = gate, a.residual = residual, a.scale = residual_scale;
    a.next_weight = next_weight, a.h = h, a.n = n;
    a.rows = desc->rows, a.D = desc->D, a.eps = desc->eps, a.activation = desc->activation;
    const unsigned grid = (unsigned)(a.rows < 148 * 16 ? a.rows : 148 * 16);
    return with_dtype(desc->dtype, [&](auto t) {
        norm_forward_rows<decltype(t)><<<grid, kNormThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
        return check_launch();
    });
}

extern "C" int64_t psig_norm_backward_workspace(const PsigNormDesc *desc)
{
    const int rc = check_norm(desc);
    if (rc != PSIG_OK) return rc;
    return (int64_t)backward_blocks(*desc) * 3 * desc->D * (desc->dtype == PSIG_F64 ? 8 : 4);
}

extern "C" int psig_norm_backward(const PsigNormDesc *desc, const void *x, const void *weight, const void *gate,
                                  const void *residual, const void *residual_scale, const void *next_weight,
                                  const void *grad_h, const void *grad_n, void *grad_x, void *grad_weight,
                                  void *grad_gate, void *grad_residual, void *grad_residual_scale,
                                  void *grad_next_weight, void *workspace, int64_t workspace_bytes, void *stream)
{
    const int rc = check_norm(desc);
    if (rc != PSIG_OK) return rc;
    if (desc->rows == 0) return PSIG_OK;   // the caller zeroes the gradients of the vectors
    if (x == nullptr || (next_weight != nullptr && grad_n == nullptr)) return PSIG_ERR_NULL;
    if (workspace == nullptr || workspace_bytes < psig_norm_backward_workspace(desc)) return PSIG_ERR_WORKSPACE;
    NormArgs a{};
    a.x = x, a.weight = weight, a.gate = gate, a.residual = residual, a.scale = residual_scale;
    a.next_weight = next_weight, a.grad_h = grad_h, a.grad_n = grad_n;
    a.grad_x = grad_x, a.grad_gate = gate ? grad_gate : nullptr, a.grad_residual = residual ? grad_residual : nullptr;
    a.partial = workspace;
    a.rows = desc->rows, a.D = desc->D, a.eps = desc->eps, a.activation = desc->activation;
    const int blocks = backward_blocks(*desc);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        using A = typename Acc<T>::type;
        norm_backward_rows<T><<<blocks, kNormThreads, 0, s>>>(a);
        int status = check_launch();
        if (status != PSIG_OK) return status;
        norm_sum_partials<A><<<(unsigned)((3 * a.D + 255) / 256), 256, 0, s>>>(
            static_cast<const A *>(workspace), blocks, a.D, static_cast<A *>(grad_weight),
            static_cast<A *>(grad_residual_scale), static_cast<A *>(grad_next_weight));
        return check_launch();
    });
}
