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

// ---- rows held in registers (up to kNormWidest features) ----
//
// A team of 2^k threads takes a row, E values to an access and NV accesses to a thread, so that every operand is read
// once and the sums over a row are the only exchange: shuffles inside a warp, one barrier for teams of several warps.

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

template <typename T, int E>
struct Pack {
    using raw = typename Raw<(int)sizeof(T) * E>::type;
    union {
        raw bits;
        T v[E];
    };
    __device__ __forceinline__ Pack() : bits{} {}
    __device__ __forceinline__ void load(const void *p, long long at) { bits = *reinterpret_cast<const raw *>(static_cast<const T *>(p) + at); }
    __device__ __forceinline__ void store(void *p, long long at) const { *reinterpret_cast<raw *>(static_cast<T *>(p) + at) = bits; }
};

// E values of a parameter vector (type of sums); 1 where there is none.
template <typename A, int E>
__device__ __forceinline__ void load_vector(const void *p, long long at, A (&v)[E])
{
    if (p == nullptr) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = A(1);
        return;
    }
    constexpr int W = 16 / (int)sizeof(A) < E ? 16 / (int)sizeof(A) : E;   // vectors start on 16 bytes where E > 1
#pragma unroll
    for (int e = 0; e < E; e += W) {
        Pack<A, W> w;
        w.load(p, at + e);
#pragma unroll
        for (int i = 0; i < W; ++i) v[e + i] = w.v[i];
    }
}

constexpr int kTeamMax = 512;
constexpr int kNormWidest = kTeamMax * 16;

// Sums N values over the team.  `round` alternates between two sets of partial sums, so that one barrier is enough.
template <typename A, int N>
__device__ __forceinline__ void team_sum(A (&v)[N], int team_log2, A *shared, int round)
{
    const int inside = team_log2 < 5 ? team_log2 : 5;
    for (int s = 0; s < inside; ++s)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 1 << s);
    if (team_log2 <= 5) return;
    A *mine = shared + (round & 1) * 2 * (kTeamMax / 32);
    const int warp = threadIdx.x >> 5, warps = 1 << (team_log2 - 5);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) mine[warp * 2 + i] = v[i];
    __syncthreads();
    const int first = warp & ~(warps - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = A(0);
    for (int w = 0; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += mine[(first + w) * 2 + i];
}

__device__ __forceinline__ float inverse_root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return rsqrt(v); }

template <typename T, int E, int NV>
__global__ void __launch_bounds__(kTeamMax) norm_forward_team(const NormArgs a, int team_log2)
{
    using A = typename Acc<T>::type;
    __shared__ A shared[4 * (kTeamMax / 32)];
    const int team = threadIdx.x >> team_log2, j = threadIdx.x & ((1 << team_log2) - 1);
    const long long row = (long long)blockIdx.x * (blockDim.x >> team_log2) + team;
    const long long base = row * a.D;
    Pack<T, E> x[NV], g[NV], res[NV];
    bool live[NV];
    int col[NV];
    A sum[1] = {A(0)};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        col[v] = (j + (v << team_log2)) * E;
        live[v] = row < a.rows && col[v] < a.D;
        if (live[v]) {
            x[v].load(a.x, base + col[v]);
            if (a.gate) g[v].load(a.gate, base + col[v]);
            if (a.residual) res[v].load(a.residual, base + col[v]);
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) { const A t = to_acc<A>(x[v].v[e]); sum[0] += t * t; }
    team_sum(sum, team_log2, shared, 0);
    const A r = inverse_root(sum[0] / A(a.D) + A(a.eps));
    A h[NV * E];
    sum[0] = A(0);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if (!live[v]) continue;
        A w[E], c[E];
        load_vector<A, E>(a.weight, col[v], w);
        load_vector<A, E>(a.scale, col[v], c);
        Pack<T, E> out;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            A slope, t = to_acc<A>(x[v].v[e]) * r * w[e];
            if (a.gate) t *= gate_value(to_acc<A>(g[v].v[e]), a.activation, &slope);
            t *= c[e];
            if (a.residual) t += to_acc<A>(res[v].v[e]);
            h[v * E + e] = t;
            sum[0] += t * t;
            out.v[e] = from_acc<T>(t);
        }
        out.store(a.h, base + col[v]);
    }
    if (a.next_weight == nullptr) return;
    team_sum(sum, team_log2, shared, 1);
    const A r2 = inverse_root(sum[0] / A(a.D) + A(a.eps));
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if (!live[v]) continue;
        A w[E];
        load_vector<A, E>(a.next_weight, col[v], w);
        Pack<T, E> out;
#pragma unroll
        for (int e = 0; e < E; ++e) out.v[e] = from_acc<T>(h[v * E + e] * r2 * w[e]);
        out.store(a.n, base + col[v]);
    }
}

// Blocks walk the rows; a thread keeps the sums over rows for its own columns in registers.  NEXT: with the norm before
// the next block (three exchanges a row instead of one).
template <typename T, int E, int NV, bool NEXT>
__global__ void __launch_bounds__(kTeamMax) norm_backward_team(const NormArgs a, int team_log2)
{
    using A = typename Acc<T>::type;
    __shared__ A shared[4 * (kTeamMax / 32)];
    extern __shared__ __align__(16) unsigned char fold_raw[];
    A *fold = reinterpret_cast<A *>(fold_raw);
    const int team = threadIdx.x >> team_log2, j = threadIdx.x & ((1 << team_log2) - 1), teams = blockDim.x >> team_log2;
    A sum_w[NV * E], sum_c[NV * E], sum_n[NEXT ? NV * E : 1];
#pragma unroll
    for (int i = 0; i < NV * E; ++i) {
        sum_w[i] = sum_c[i] = A(0);
        if (NEXT) sum_n[i] = A(0);
    }
    const bool want_c = a.scale != nullptr, want_w = a.weight != nullptr;
    const A mean = A(1) / A(a.D);
    int round = 0;
    for (long long first = (long long)blockIdx.x * teams; first < a.rows; first += (long long)gridDim.x * teams) {
        const long long row = first + team, base = row * a.D;
        Pack<T, E> x[NV], g[NV], res[NV], gh[NV], gn[NV];
        bool live[NV];
        int col[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            col[v] = (j + (v << team_log2)) * E;
            live[v] = row < a.rows && col[v] < a.D;
            if (live[v]) {
                x[v].load(a.x, base + col[v]);
                if (a.gate) g[v].load(a.gate, base + col[v]);
                if (NEXT && a.residual) res[v].load(a.residual, base + col[v]);
                if (a.grad_h) gh[v].load(a.grad_h, base + col[v]);
                if (NEXT) gn[v].load(a.grad_n, base + col[v]);
            }
        }
        A r, r2 = A(0), m2 = A(0), m;
        A xx[2] = {A(0), A(0)};
        if (!NEXT) {   // the gradient of h is there: both sums in one exchange
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!live[v]) continue;
                A w[E], c[E];
                load_vector<A, E>(a.weight, col[v], w);
                load_vector<A, E>(a.scale, col[v], c);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    A act = A(1), slope, t = to_acc<A>(x[v].v[e]);
                    if (a.gate) act = gate_value(to_acc<A>(g[v].v[e]), a.activation, &slope);
                    xx[0] += t * t;
                    xx[1] += w[e] * (to_acc<A>(gh[v].v[e]) * c[e] * act) * t;
                }
            }
            team_sum(xx, team_log2, shared, round++);
            r = inverse_root(xx[0] * mean + A(a.eps));
            m = xx[1] * mean * r * r * r;
        } else {
            A sx[1] = {A(0)};
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < E; ++e) { const A t = to_acc<A>(x[v].v[e]); sx[0] += t * t; }
            team_sum(sx, team_log2, shared, round++);
            r = inverse_root(sx[0] * mean + A(a.eps));
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!live[v]) continue;
                A w[E], c[E], w2[E];
                load_vector<A, E>(a.weight, col[v], w);
                load_vector<A, E>(a.scale, col[v], c);
                load_vector<A, E>(a.next_weight, col[v], w2);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    A slope, t = to_acc<A>(x[v].v[e]) * r * w[e];
                    if (a.gate) t *= gate_value(to_acc<A>(g[v].v[e]), a.activation, &slope);
                    t *= c[e];
                    if (a.residual) t += to_acc<A>(res[v].v[e]);
                    xx[0] += t * t;
                    xx[1] += w2[e] * to_acc<A>(gn[v].v[e]) * t;
                }
            }
            team_sum(xx, team_log2, shared, round++);
            r2 = inverse_root(xx[0] * mean + A(a.eps));
            m2 = xx[1] * mean * r2 * r2 * r2;
            sx[0] = A(0);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!live[v]) continue;
                A w[E], c[E], w2[E];
                load_vector<A, E>(a.weight, col[v], w);
                load_vector<A, E>(a.scale, col[v], c);
                load_vector<A, E>(a.next_weight, col[v], w2);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const A t = to_acc<A>(x[v].v[e]);
                    A act = A(1), slope;
                    if (a.gate) act = gate_value(to_acc<A>(g[v].v[e]), a.activation, &slope);
                    A h = t * r * w[e] * act * c[e];
                    if (a.residual) h += to_acc<A>(res[v].v[e]);
                    const A dh = to_acc<A>(gh[v].v[e]) + w2[e] * to_acc<A>(gn[v].v[e]) * r2 - h * m2;
                    sx[0] += w[e] * dh * c[e] * act * t;
                }
            }
            team_sum(sx, team_log2, shared, round++);
            m = sx[0] * mean * r * r * r;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (!live[v]) continue;
            A w[E], c[E], w2[E];
            load_vector<A, E>(a.weight, col[v], w);
            load_vector<A, E>(a.scale, col[v], c);
            if (NEXT) load_vector<A, E>(a.next_weight, col[v], w2);
            Pack<T, E> out_x, out_g, out_r;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const A t = to_acc<A>(x[v].v[e]);
                A act = A(1), slope = A(0);
                if (a.gate) act = gate_value(to_acc<A>(g[v].v[e]), a.activation, &slope);
                const A z = t * r * w[e];
                A dh = to_acc<A>(gh[v].v[e]);
                if (NEXT) {
                    A h = z * act * c[e];
                    if (a.residual) h += to_acc<A>(res[v].v[e]);
                    const A dn = to_acc<A>(gn[v].v[e]);
                    dh += w2[e] * dn * r2 - h * m2;
                    sum_n[v * E + e] += dn * h * r2;
                }
                const A dz = dh * c[e] * act;
                sum_c[v * E + e] += dh * z * act;
                sum_w[v * E + e] += dz * t * r;
                out_r.v[e] = from_acc<T>(dh);
                out_g.v[e] = from_acc<T>(dh * c[e] * z * slope);
                out_x.v[e] = from_acc<T>(r * w[e] * dz - t * m);
            }
            if (a.grad_residual) out_r.store(a.grad_residual, base + col[v]);
            if (a.grad_gate) out_g.store(a.grad_gate, base + col[v]);
            if (a.grad_x) out_x.store(a.grad_x, base + col[v]);
        }
        }
    // the block's teams hold the same columns: fold them in order, one vector after the other
    A *part = static_cast<A *>(a.partial) + (long long)blockIdx.x * 3 * a.D;
#pragma unroll
    for (int which = 0; which < (NEXT ? 3 : 2); ++which) {
        if (which == 0 ? !want_w : which == 1 ? !want_c : false) continue;
        if (teams > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV * E; ++i)
                fold[i * blockDim.x + threadIdx.x] = which == 0 ? sum_w[i] : which == 1 ? sum_c[i] : sum_n[NEXT ? i : 0];
            __syncthreads();
        }
        if (team == 0)
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int c = (j + (v << team_log2)) * E + e, i = v * E + e;
                    if (c >= a.D) continue;
                    A s = which == 0 ? sum_w[i] : which == 1 ? sum_c[i] : sum_n[NEXT ? i : 0];
                    if (teams > 1)
                        for (int k = 1; k < teams; ++k) s += fold[i * blockDim.x + (k << team_log2) + j];
                    part[which * a.D + c] = s;
                }
    }
}

// Sums of the blocks' partial rows, in a fixed order: 32 columns to a block, its warps take every 8th partial row.
template <typename A>
__global__ void __launch_bounds__(256) norm_sum_partials(const A *__restrict__ partial, int blocks, long long D,
                                                         A *__restrict__ out_w, A *__restrict__ out_c, A *__restrict__ out_w2)
{
    __shared__ A shared[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * 32 + lane;
    A *out = blockIdx.y == 0 ? out_w : blockIdx.y == 1 ? out_c : out_w2;
    if (out == nullptr) return;
    A sum = A(0);
    if (col < D)
#pragma unroll 4
        for (int b = warp; b < blocks; b += 8) sum += partial[((long long)b * 3 + blockIdx.y) * D + col];
    shared[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && col < D) {
        for (int i = 1; i < 8; ++i) sum += shared[i][lane];
        out[col] = sum;
    }
}

int check_norm(const PsigNormDesc *d)
{
    if (d == nullptr) return PSIG_ERR_NULL;
    if (d->dtype < PSIG_F32 || d->dtype > PSIG_F16) return PSIG_ERR_DTYPE;
    if (d->rows < 0 || d->D < 1 || d->activation < 0 || d->activation > 1) return PSIG_ERR_SHAPE;
    return PSIG_OK;
}

// How a row is dealt to threads: 8 values to a thread while the team has at most kTeamMax threads then 16.
struct TeamPlan {
    int team_log2, values, threads;   // values per thread; threads per block
};

TeamPlan team_plan(long long D)
{
    TeamPlan p{0, 8, 256};
    while ((8LL << p.team_log2) < D && (1 << p.team_log2) < kTeamMax) ++p.team_log2;
    while ((long long)p.values << p.team_log2 < D) p.values *= 2;
    if (1 << p.team_log2 > p.threads) p.threads = 1 << p.team_log2;
    return p;
}

// Resident blocks are enough: each keeps its column sums over all its rows.
int backward_blocks(const PsigNormDesc &d)
{
    if (d.D > kNormWidest) return (int)(d.rows < 148 * 4 ? d.rows : 148 * 4);
    const TeamPlan p = team_plan(d.D);
    const long long teams = p.threads >> p.team_log2, need = (d.rows + teams - 1) / teams;
    const long long most = 148LL * (p.threads > 256 ? 2 : 4);
    return (int)(need < most ? need : most);
}

// Largest number of values that one access of every operand can hold (all rows start on such a boundary).
template <typename T>
int access_width(const NormArgs &a)
{
    const void *rows[] = {a.x, a.gate, a.residual, a.grad_h, a.grad_n, a.h, a.n, a.grad_x, a.grad_gate, a.grad_residual};
    const void *vectors[] = {a.weight, a.scale, a.next_weight};
    int width = 16 / (int)sizeof(T);
    for (; width > 1; width /= 2) {
        bool ok = a.D % width == 0;
        for (const void *p : rows) ok = ok && reinterpret_cast<uintptr_t>(p) % (width * sizeof(T)) == 0;
        for (const void *p : vectors) ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
        if (ok) break;
    }
    return width;
}

// Calls fn with (values per access, accesses per thread) as compile-time numbers.
template <typename T, typename Fn>
int with_shape(int width, int values, Fn fn)
{
    constexpr int full = sizeof(T) == 8 ? 1 : 16 / (int)sizeof(T);
    auto by_values = [&](auto w) {
        constexpr int E = decltype(w)::value;
        if (values == 8) return fn(w, std::integral_constant<int, 8 / E>{});
        return fn(w, std::integral_constant<int, 16 / E>{});
    };
    if (width >= full) return by_values(std::integral_constant<int, full>{});
    if constexpr (full == 8)
        if (width >= 2) return by_values(std::integral_constant<int, 2>{});
    return by_values(std::integral_constant<int, 1>{});
}

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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        if (a.D > kNormWidest) {
            const unsigned grid = (unsigned)(a.rows < 148 * 16 ? a.rows : 148 * 16);
            norm_forward_rows<T><<<grid, kNormThreads, 0, s>>>(a);
            return check_launch();
        }
        const TeamPlan p = team_plan(a.D);
        const long long teams = p.threads >> p.team_log2, blocks = (a.rows + teams - 1) / teams;
        if (blocks > 0x7fffffffLL) return (int)PSIG_ERR_TOO_LARGE;
        return with_shape<T>(access_width<T>(a), p.values, [&](auto e, auto nv) {
            norm_forward_team<T, decltype(e)::value, decltype(nv)::value><<<(unsigned)blocks, p.threads, 0, s>>>(a, p.team_log2);
            return check_launch();
        });
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
        int status;
        if (a.D > kNormWidest) {
            norm_backward_rows<T><<<blocks, kNormThreads, 0, s>>>(a);
            status = check_launch();
        } else {
            const TeamPlan p = team_plan(a.D);
            status = with_shape<T>(access_width<T>(a), p.values, [&](auto e, auto nv) {
                constexpr int E = decltype(e)::value, NV = decltype(nv)::value;
                const size_t fold = (p.threads >> p.team_log2) > 1 ? sizeof(A) * E * NV * p.threads : 0;
                if (a.next_weight) norm_backward_team<T, E, NV, true><<<blocks, p.threads, fold, s>>>(a, p.team_log2);
                else norm_backward_team<T, E, NV, false><<<blocks, p.threads, fold, s>>>(a, p.team_log2);
                return check_launch();
            });
        }
        if (status != PSIG_OK || (!grad_weight && !grad_residual_scale && !grad_next_weight)) return status;
        norm_sum_partials<A><<<dim3((unsigned)((a.D + 31) / 32), 3), 256, 0, s>>>(
            static_cast<const A *>(workspace), blocks, a.D, static_cast<A *>(grad_weight),
            static_cast<A *>(grad_residual_scale), static_cast<A *>(grad_next_weight));
        return check_launch();
    });
}
