// Decayed linear attention over the time axis: entry points, the kernels that serve every size and type, the
// decay gradient, and the single time step.  Formulas: include/pathsig_b200.h; the sweep that the forward
// pass and the three gradients share: sequence.cuh.
//
// Gradients.  With A_t = scale q_t go_t^T + exp(g_{t+1}) A_{t+1} (A behind the last step: grad_state),
//     grad_q_t = scale S_t go_t,   grad_k_t = A_t v_t,   grad_v_t = A_t^T k_t,   grad_g_t = <A_t, exp(g_t) S_{t-1}>.
// The first three are sweeps.  The last is the sum over all pairs s < t <= u of what the pair (s, u) adds to the
// result; with x_t = q_t . grad_q_t (pairs that end at t) and y_s = k_s . grad_k_s (pairs that begin at s),
//     grad_g_t = B_e + sum_{t <= i < e} (x_i - y_i),     B_e = <exp(g_e) A_e, S_{e-1}> (pairs across e)
// for any e > t.  e is the end of t's segment of kSegment steps: B_e comes from the two states themselves, so that
// the difference of the two sums never runs over more than a segment, however long the sequence is.
#include "sequence.cuh"

#include <atomic>

namespace psig {
namespace {

constexpr int kSweepThreads = 256;
constexpr int kSweepSteps = 16;   // time steps staged at once
constexpr int kSweepCols = 32;    // columns of the state per block

__device__ __forceinline__ long long length_of(const int *lengths, long long b, long long L)
{
    if (lengths == nullptr) return L;
    const long long n = lengths[b];
    return n < 0 ? 0 : n > L ? L : n;
}

// The simplest sweep: one block per (sequence, head, 32 columns of the state), the state in registers (lane =
// column, warp w holds rows w, w + 8, ...), one time step after another; each warp's share of the step's output
// row goes to shared memory and is summed once per 16 steps.  Serves every type, size and alignment.
template <typename T, int RPT>
__global__ void __launch_bounds__(kSweepThreads) attn_sweep_rows(const Sweep a)
{
    using A = typename Acc<T>::type;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    A *r_s = reinterpret_cast<A *>(smem_raw);                // [steps][d1]
    A *k_s = r_s + kSweepSteps * a.d1;                       // [steps][d1]
    A *v_s = k_s + kSweepSteps * a.d1;                       // [steps][32]
    A *part = v_s + kSweepSteps * kSweepCols;                // [8][steps][32]
    A *w_s = part + 8 * kSweepSteps * kSweepCols;            // [steps]
    __shared__ A dot_s[8];

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long bh = blockIdx.x;
    const long long b = bh / a.H;
    const int h = (int)(bh % a.H);
    const int col0 = blockIdx.y * kSweepCols, col = col0 + lane;
    const bool live = col < a.d2;
    const long long n = length_of(a.lengths, b, a.L);
    const T *r = static_cast<const T *>(a.r.data) + b * a.r.stride[0] + (h / a.r.share) * a.r.stride[2];
    const T *k = static_cast<const T *>(a.k.data) + b * a.k.stride[0] + (h / a.k.share) * a.k.stride[2];
    const T *v = static_cast<const T *>(a.v.data) + b * a.v.stride[0] + (h / a.v.share) * a.v.stride[2];
    const A *g = static_cast<const A *>(a.decay) + b * a.decay_stride[0] + h * a.decay_stride[2];
    const long long state0 = bh * a.d1 * a.d2;

    A S[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int row = warp + 8 * i;
        S[i] = A(0);
        if (a.init != nullptr && live && row < a.d1)
            S[i] = static_cast<const A *>(a.init)[state0 + (a.init_transposed ? (long long)col * a.d1 + row
                                                                              : (long long)row * a.d2 + col)];
    }

    const long long stages = (n + kSweepSteps - 1) / kSweepSteps;
    const long long segments = (a.L + kSegment - 1) / kSegment;
    for (long long st = 0; st < stages; ++st) {
        const long long t0 = (a.reverse ? stages - 1 - st : st) * kSweepSteps;
        const long long t1 = t0 + kSweepSteps < n ? t0 + kSweepSteps : n;
        const int m = (int)(t1 - t0);
        for (int e = threadIdx.x; e < m * a.d1; e += kSweepThreads) {
            const int j = e / a.d1, d = e % a.d1;
            const long long t = a.reverse ? t1 - 1 - j : t0 + j;
            r_s[e] = to_acc<A>(r[t * a.r.stride[1] + d]);
            k_s[e] = to_acc<A>(k[t * a.k.stride[1] + d]);
        }
        for (int e = threadIdx.x; e < m * kSweepCols; e += kSweepThreads) {
            const int j = e / kSweepCols, c = col0 + e % kSweepCols;
            const long long t = a.reverse ? t1 - 1 - j : t0 + j;
            v_s[e] = c < a.d2 ? to_acc<A>(v[t * a.v.stride[1] + c]) * A(a.kv_scale) : A(0);
        }
        if (threadIdx.x < m) {
            const long long t = a.reverse ? t1 - threadIdx.x : t0 + threadIdx.x;   // reverse: the step behind
            w_s[threadIdx.x] = t < n ? exp_acc(g[t * a.decay_stride[1]]) : A(1);
        }
        __syncthreads();
        const bool boundary = t1 == n || t1 % kSegment == 0;
        const long long segment = (t1 - 1) / kSegment;
        A first = w_s[0];
        if (a.reverse && a.anchor_dots != nullptr && boundary) {
            // the state just behind t1, decayed over t1, against the stored state of the steps before t1
            const A *anchor = static_cast<const A *>(a.anchors) + (bh * segments + segment) * a.d1 * a.d2;
            A dot = A(0);
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
                const int row = warp + 8 * i;
                S[i] *= first;
                if (live && row < a.d1) dot += S[i] * anchor[(long long)row * a.d2 + col];
            }
            first = A(1);
            for (int s = 16; s >= 1; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
            if (lane == 0) dot_s[warp] = dot;
            __syncthreads();
            if (threadIdx.x == 0) {
                A sum = A(0);
                for (int i = 0; i < 8; ++i) sum += dot_s[i];
                static_cast<A *>(a.anchor_dots)[(bh * segments + segment) * gridDim.y + blockIdx.y] = sum;
            }
        }
        for (int j = 0; j < m; ++j) {
            const A w = j == 0 ? first : w_s[j], vj = v_s[j * kSweepCols + lane];
            A acc = A(0);
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
                const int row = warp + 8 * i;
                if (row < a.d1) {
                    S[i] = fma(k_s[j * a.d1 + row], vj, S[i] * w);
                    acc = fma(r_s[j * a.d1 + row], S[i], acc);
                }
            }
            part[(warp * kSweepSteps + j) * kSweepCols + lane] = acc;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < m * kSweepCols; e += kSweepThreads) {
            const int j = e / kSweepCols, c = col0 + e % kSweepCols;
            if (c >= a.d2) continue;
            A sum = A(0);
            for (int i = 0; i < 8; ++i) sum += part[(i * kSweepSteps + j) * kSweepCols + e % kSweepCols];
            sum *= A(a.out_scale);
            const long long t = a.reverse ? t1 - 1 - j : t0 + j;
            const long long at = ((b * a.L + t) * a.H + h) * a.d2 + c;
            if (a.out_acc) static_cast<A *>(a.out)[at] = sum;
            else static_cast<T *>(a.out)[at] = from_acc<T>(sum);
        }
        if (!a.reverse && a.anchors != nullptr && boundary) {
            A *anchor = static_cast<A *>(a.anchors) + (bh * segments + segment) * a.d1 * a.d2;
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
                const int row = warp + 8 * i;
                if (live && row < a.d1) anchor[(long long)row * a.d2 + col] = S[i];
            }
        }
        __syncthreads();
    }
    for (long long e = threadIdx.x; e < (a.L - n) * kSweepCols; e += kSweepThreads) {
        const long long t = n + e / kSweepCols;
        const int c = col0 + (int)(e % kSweepCols);
        const long long at = ((b * a.L + t) * a.H + h) * a.d2 + c;
        if (c >= a.d2) continue;
        if (a.out_acc) static_cast<A *>(a.out)[at] = A(0);
        else static_cast<T *>(a.out)[at] = from_acc<T>(A(0));
    }
    if (a.final != nullptr) {
        const A w = a.reverse && n > 0 ? exp_acc(g[0]) : A(1);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int row = warp + 8 * i;
            if (live && row < a.d1)
                static_cast<A *>(a.final)[state0 + (a.final_transposed ? (long long)col * a.d1 + row
                                                                       : (long long)row * a.d2 + col)] = S[i] * w;
        }
    }
}

inline int column_tiles(int d2) { return (d2 + kSweepCols - 1) / kSweepCols; }

template <typename T>
int sweep_rows(const Sweep &a, cudaStream_t stream)
{
    using A = typename Acc<T>::type;
    const dim3 grid((unsigned)(a.B * a.H), (unsigned)column_tiles(a.d2));
    const size_t smem = sizeof(A) * (size_t)(2 * kSweepSteps * a.d1 + 9 * kSweepSteps * kSweepCols + kSweepSteps);
    auto launch = [&](auto kernel) {
        if (!prepare_kernel(kernel, smem, false)) return (int)PSIG_ERR_CUDA;
        kernel<<<grid, kSweepThreads, smem, stream>>>(a);
        return check_launch();
    };
    if (a.d1 <= 64) return launch(attn_sweep_rows<T, 8>);
    if (a.d1 <= 128) return launch(attn_sweep_rows<T, 16>);
    return launch(attn_sweep_rows<T, 32>);
}

// Sums of the query heads that share a key/value head, rounded once: (B*L, H, d) -> (B*L, Hkv, d).
template <typename T>
__global__ void attn_sum_heads(const typename Acc<T>::type *__restrict__ acc, T *__restrict__ out, long long total,
                               int share, int d)
{
    using A = typename Acc<T>::type;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (long long)gridDim.x * blockDim.x) {
        const long long head = i / d;
        const A *p = acc + head * share * d + i % d;
        A sum = p[0];
        for (int s = 1; s < share; ++s) sum += p[(long long)s * d];
        out[i] = from_acc<T>(sum);
    }
}

// x_t - y_t per (b, t, h), a warp each: q . grad_q - k . grad_k from the unrounded gradients.
template <typename T>
__global__ void attn_pair_difference(const SweepOperand q, const SweepOperand k,
                                     const typename Acc<T>::type *__restrict__ gq,
                                     const typename Acc<T>::type *__restrict__ gk, double *__restrict__ out,
                                     long long rows, long long L, int H, int d)
{
    using A = typename Acc<T>::type;
    const int lane = threadIdx.x & 31;
    const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
    for (long long row = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); row < rows; row += warps) {
        const int h = (int)(row % H);
        const long long bt = row / H, b = bt / L, t = bt % L;
        const T *qr = static_cast<const T *>(q.data) + b * q.stride[0] + t * q.stride[1] + (h / q.share) * q.stride[2];
        const T *kr = static_cast<const T *>(k.data) + b * k.stride[0] + t * k.stride[1] + (h / k.share) * k.stride[2];
        A sum = A(0);
        for (int i = lane; i < d; i += 32) {
            const A x = gq[row * d + i], y = gk[row * d + i];
            // rows behind the last step hold zeros; what stands in q and k there is not looked at
            if (x != A(0)) sum += to_acc<A>(qr[i]) * x;
            if (y != A(0)) sum -= to_acc<A>(kr[i]) * y;
        }
        for (int s = 16; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        if (lane == 0) out[row] = (double)sum;
    }
}

// grad_g over one segment per block: B_e plus the sums of x - y from the segment's end, in 64 bits.  Writes
// (B, L, H), or the segment's total for a decay per head.  A step whose decay underflows to 0 has gradient 0.
struct PairSums {      // x - y of a step: the sum over `plus` arrays minus the sum over `minus` arrays, `step` apart
    const void *plus, *minus;
    int n_plus, n_minus;
    long long step;
};
template <typename A, typename P>
__global__ void attn_decay_grad(const PairSums pairs, const A *__restrict__ dots, int tiles,
                                const A *__restrict__ decay, long long s0, long long s1, long long s2,
                                const int *__restrict__ lengths, long long L, int H, A *__restrict__ out,
                                double *__restrict__ totals)
{
    __shared__ double carry_s[kSegment / 32], total_s[kSegment / 32];
    const long long segments = gridDim.x;
    const long long segment = blockIdx.x;
    const int h = blockIdx.y % H;
    const long long b = blockIdx.y / H, bh = blockIdx.y;
    const long long n = length_of(lengths, b, L);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long end = (segment + 1) * kSegment < n ? (segment + 1) * kSegment : n;
    // thread i takes step end - 1 - i, so that sums from the end are running sums over the threads
    const long long t = end - 1 - threadIdx.x;
    const bool live = t >= segment * kSegment && end > segment * kSegment;
    double sum = 0.0;
    if (live) {
        const P *x = static_cast<const P *>(pairs.plus) + (b * L + t) * H + h;
        const P *y = static_cast<const P *>(pairs.minus) + (b * L + t) * H + h;
        for (int i = 0; i < pairs.n_plus; ++i) sum += (double)x[i * pairs.step];
        for (int i = 0; i < pairs.n_minus; ++i) sum -= (double)y[i * pairs.step];
    }
    for (int s = 1; s < 32; s <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, sum, s);
        if (lane >= s) sum += up;
    }
    if (lane == 31) carry_s[warp] = sum;
    __syncthreads();
    for (int i = 0; i < warp; ++i) sum += carry_s[i];
    if (live)
        for (int i = 0; i < tiles; ++i) sum += (double)dots[(bh * segments + segment) * tiles + i];
    if (live && exp_acc(decay[b * s0 + t * s1 + h * s2]) == A(0)) sum = 0.0;
    if (out != nullptr) {
        if (live) out[(b * L + t) * H + h] = (A)sum;
        const long long z = segment * kSegment + threadIdx.x;
        if (z >= n && z < L) out[(b * L + z) * H + h] = A(0);
    }
    if (totals != nullptr) {
        double all = live ? sum : 0.0;
        for (int s = 16; s >= 1; s >>= 1) all += __shfl_xor_sync(0xffffffffu, all, s);
        if (lane == 0) total_s[warp] = all;
        __syncthreads();
        if (threadIdx.x == 0) {
            double v = 0.0;
            for (int i = 0; i < blockDim.x >> 5; ++i) v += total_s[i];
            totals[bh * segments + segment] = v;
        }
    }
}

// One block per head: the segments' totals over all sequences, in a fixed order.
template <typename A>
__global__ void attn_decay_total(const double *__restrict__ totals, long long B, int H, long long segments,
                                 A *__restrict__ out)
{
    __shared__ double part_s[8];
    const int h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double sum = 0.0;
    for (long long i = threadIdx.x; i < B * segments; i += blockDim.x)
        sum += totals[(i / segments * H + h) * segments + i % segments];
    for (int s = 16; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (lane == 0) part_s[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double v = 0.0;
        for (int i = 0; i < 8; ++i) v += part_s[i];
        out[h] = (A)v;
    }
}

// One time step: a block takes 32 columns of one state, reads each entry once, writes it back decayed and with the
// new product, and sums its columns of the output row.
template <typename T>
__global__ void __launch_bounds__(256) attn_step_rows(const SweepOperand q, const SweepOperand k, const SweepOperand v,
                                                      const typename Acc<T>::type *__restrict__ decay, long long s0,
                                                      long long s2, typename Acc<T>::type *__restrict__ state,
                                                      T *__restrict__ out, int H, int dk, int dv, double scale)
{
    using A = typename Acc<T>::type;
    __shared__ A part[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long bh = blockIdx.x, b = bh / H;
    const int h = (int)(bh % H), col = blockIdx.y * 32 + lane;
    const T *qr = static_cast<const T *>(q.data) + b * q.stride[0] + (h / q.share) * q.stride[2];
    const T *kr = static_cast<const T *>(k.data) + b * k.stride[0] + (h / k.share) * k.stride[2];
    const T *vr = static_cast<const T *>(v.data) + b * v.stride[0] + (h / v.share) * v.stride[2];
    const A w = exp_acc(decay[b * s0 + h * s2]);
    A acc = A(0);
    if (col < dv) {
        const A vj = to_acc<A>(vr[col]);
        A *s = state + bh * dk * dv + col;
        for (int row = warp; row < dk; row += 8) {
            const A next = fma(to_acc<A>(kr[row]), vj, s[(long long)row * dv] * w);
            s[(long long)row * dv] = next;
            acc = fma(to_acc<A>(qr[row]), next, acc);
        }
    }
    part[warp][lane] = acc;
    __syncthreads();
    if (warp == 0 && col < dv) {
        A sum = A(0);
        for (int i = 0; i < 8; ++i) sum += part[i][lane];
        out[bh * dv + col] = from_acc<T>(sum * A(scale));
    }
}

// The same for states of 32 bits whose rows are whole 16-byte pieces: COLS columns to a block, four to a thread, several
// rows of the state in flight per thread.  Bound by memory, the state once in and once out: 256 streams of 16 heads of 128 x 128
// (537 MB) take 104 us (79 % of the copy rate) with 128 columns to a block, 200 us with one column to a thread.  32 columns give the few
// blocks of a few streams more parts.
template <typename T, int COLS>
__global__ void __launch_bounds__(256) attn_step_vector(const SweepOperand q, const SweepOperand k, const SweepOperand v,
                                                        const float *__restrict__ decay, long long s0, long long s2,
                                                        float *__restrict__ state, T *__restrict__ out, int H, int dk, int dv,
                                                        float scale)
{
    constexpr int LANES = COLS / 4, GROUPS = 256 / LANES, FLIGHT = 8;
    __shared__ float q_s[256], k_s[256];
    __shared__ float4 part[GROUPS][LANES];
    const int x = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const long long bh = blockIdx.x, b = bh / H;
    const int h = (int)(bh % H), col = blockIdx.y * COLS + x * 4;
    const bool live = col < dv;
    float4 *s = reinterpret_cast<float4 *>(state + bh * dk * dv + col);
    const long long step = (long long)GROUPS * dv / 4;
    s += (long long)group * dv / 4;
    float4 held[FLIGHT];
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i)
        if (live && group + i * GROUPS < dk) held[i] = s[i * step];
    if (threadIdx.x < dk) {
        q_s[threadIdx.x] = to_acc<float>((static_cast<const T *>(q.data) + b * q.stride[0] + (h / q.share) * q.stride[2])[threadIdx.x]) * scale;
        k_s[threadIdx.x] = to_acc<float>((static_cast<const T *>(k.data) + b * k.stride[0] + (h / k.share) * k.stride[2])[threadIdx.x]);
    }
    const T *vr = static_cast<const T *>(v.data) + b * v.stride[0] + (h / v.share) * v.stride[2] + col;
    const float w = expf(decay[b * s0 + h * s2]);
    float4 vj = {0.f, 0.f, 0.f, 0.f}, acc = vj;
    if (live) vj = make_float4(to_acc<float>(vr[0]), to_acc<float>(vr[1]), to_acc<float>(vr[2]), to_acc<float>(vr[3]));
    __syncthreads();
    for (int row0 = group; row0 < dk; row0 += FLIGHT * GROUPS, s += FLIGHT * step) {
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) {
            const int row = row0 + i * GROUPS;
            if (!live || row >= dk) continue;
            const float kr = k_s[row], qr = q_s[row];
            float4 t = held[i];
            t.x = fmaf(kr, vj.x, t.x * w), t.y = fmaf(kr, vj.y, t.y * w), t.z = fmaf(kr, vj.z, t.z * w), t.w = fmaf(kr, vj.w, t.w * w);
            s[i * step] = t;
            acc.x = fmaf(qr, t.x, acc.x), acc.y = fmaf(qr, t.y, acc.y), acc.z = fmaf(qr, t.z, acc.z), acc.w = fmaf(qr, t.w, acc.w);
            if (row + FLIGHT * GROUPS < dk) held[i] = s[(i + FLIGHT) * step];
        }
    }
    part[group][x] = acc;
    __syncthreads();
    if (group == 0 && live) {
        for (int i = 1; i < GROUPS; ++i) {
            const float4 p = part[i][x];
            acc.x += p.x, acc.y += p.y, acc.z += p.z, acc.w += p.w;
        }
        T *o = out + bh * dv + col;
        o[0] = from_acc<T>(acc.x), o[1] = from_acc<T>(acc.y), o[2] = from_acc<T>(acc.z), o[3] = from_acc<T>(acc.w);
    }
}

// ------------------------------------------------------------------------------------------ host side

int check_attn(const PsigAttnDesc *d)
{
    if (d == nullptr) return PSIG_ERR_NULL;
    if (d->dtype < PSIG_F32 || d->dtype > PSIG_F16) return PSIG_ERR_DTYPE;
    if (d->B < 0 || d->L < 0 || d->dk < 1 || d->dv < 1 || d->H < 1 || d->Hkv < 1 || d->H % d->Hkv != 0)
        return PSIG_ERR_SHAPE;
    if (d->dk > 256 || d->dv > 256) return PSIG_ERR_TOO_LARGE;
    if (d->H > 65535 || d->B > 0x7fffffffLL / d->H) return PSIG_ERR_TOO_LARGE;   // a block's index, a grid's second dimension
    return PSIG_OK;
}

SweepOperand operand(const void *data, const int64_t *strides, int share)
{
    return SweepOperand{data, {strides[0], strides[1], strides[2]}, share};
}

Sweep sweep_of(const PsigAttnDesc &d, const void *decay)
{
    Sweep s{};
    s.decay = decay;
    for (int i = 0; i < 3; ++i) s.decay_stride[i] = d.decay_strides[i];
    s.lengths = d.lengths;
    s.B = d.B;
    s.L = d.L;
    s.H = d.H;
    s.out_scale = 1.0;
    s.kv_scale = 1.0;
    s.splits = 1;
    s.failure = failure_flag();
    return s;
}

std::atomic<int *> g_failure_flag{nullptr};

bool per_head(const PsigAttnDesc &d) { return d.decay_strides[0] == 0 && d.decay_strides[1] == 0; }

// The operands of the sweeps of a call, and whether the tensor-core form serves them.
struct Call {
    const PsigAttnDesc &d;
    const void *decay;
    SweepOperand q, k, v, go;
    int share;

    Call(const PsigAttnDesc &desc, const void *q_, const void *k_, const void *v_, const void *decay_, const void *go_)
        : d(desc), decay(decay_), share(desc.H / desc.Hkv)
    {
        const int64_t go_strides[3] = {d.L * d.H * d.dv, (int64_t)d.H * d.dv, d.dv};
        q = operand(q_, d.q_strides, 1);
        k = operand(k_, d.k_strides, share);
        v = operand(v_, d.v_strides, share);
        go = operand(go_, go_strides, 1);
    }
    Sweep forward() const
    {
        Sweep s = sweep_of(d, decay);
        s.r = q, s.k = k, s.v = v;
        s.d1 = d.dk, s.d2 = d.dv;
        s.out_scale = d.scale;
        return s;
    }
    Sweep grad_q() const
    {
        Sweep s = sweep_of(d, decay);
        s.r = go, s.k = v, s.v = k;
        s.d1 = d.dv, s.d2 = d.dk;
        s.out_scale = d.scale;
        s.init_transposed = true;
        return s;
    }
    Sweep grad_k() const
    {
        Sweep s = sweep_of(d, decay);
        s.r = v, s.k = go, s.v = q;
        s.d1 = d.dv, s.d2 = d.dk;
        s.reverse = true;
        s.kv_scale = d.scale;
        s.init_transposed = true;
        return s;
    }
    Sweep grad_v() const
    {
        Sweep s = sweep_of(d, decay);
        s.r = k, s.k = q, s.v = go;
        s.d1 = d.dk, s.d2 = d.dv;
        s.reverse = true;
        s.kv_scale = d.scale;
        return s;
    }
    // By sizes and strides; with null pointers for the operands this is what the workspace queries go by.
    // A tile is computed whole, 128 steps, however few are there; the row kernel's time grows with the steps and with the heads'
    // sizes.  Tiles / rows, us, bfloat16: 1024 heads of 128 forward 53 / 45 at 2 steps, 53 / 57 at 4, backward 197 / 185 and 197 / 228;
    // 720 heads of 64 forward 19 / 15 at 4 steps, 19 / 21 at 8, backward 76 / 65 and 76 / 85; 4096 heads of 32 forward 94 / 47 at 8
    // steps, 94 / 105 at 24, backward 363 / 188 and 363 / 400.  So 800 / (dk + dv) steps, at most 16; 16 where a state is carried
    // from call to call (1024 heads of 128: 206 / 174 at 16 steps, 207 / 245 at 24) and in the other types: 720 heads of 64, float16
    // forward 41 / 32 at 16 steps, 41 / 45 at 24, backward 150 / 125 and 152 / 171, float32 forward 54 / 31 and 54 / 45.  (Heads of 32
    // and less would gain from a higher limit there: 4096 of them, 24 steps, float16 218 / 105, float32 290 / 105.)
    bool tiles(bool carries, const void *o1 = nullptr, const void *o2 = nullptr, const void *o3 = nullptr) const
    {
        if (d.L <= 16 && (d.dtype != PSIG_BF16 || carries || d.L * (d.dk + d.dv) <= 800)) return false;
        for (const void *o : {o1, o2, o3})
            if (reinterpret_cast<uintptr_t>(o) % 16 != 0) return false;
        return d.algo != PSIG_ALGO_GENERIC && attn_tiles_supported(forward(), d.dtype) && attn_tiles_supported(grad_q(), d.dtype);
    }
};

// Scratch for the parts of long sequences in a sweep over heads of d1 and d2 (bytes, a multiple of 256; 0: one part).
long long split_bytes(const PsigAttnDesc &d, int d1, int d2)
{
    if (d.dtype == PSIG_F64 || d.dk > 128 || d.dv > 128) return 0;
    const int splits = split_plan(d.B, d.L, d.H, d2);
    return splits == 1 ? 0 : (4 * d.B * d.H * splits * (split_state_size(d1, d2) + 1) + 255) / 256 * 256;
}
void set_splits(Sweep &s, void *scratch)
{
    s.splits = split_plan(s.B, s.L, s.H, s.d2);
    s.split_states = static_cast<float *>(scratch);
    s.split_decays = s.split_states + s.B * s.H * s.splits * split_state_size(s.d1, s.d2);
}

// Scratch of the backward pass, in the order it is laid out (256-byte aligned pieces).  The tensor-core sweeps write
// gradients to their place, but for heads that share a key/value head; the others keep them unrounded first.
struct BackwardScratch {
    long long gq, gk, gv, pairs, anchors, dots, totals, parts, bytes;
};

int anchor_parts(const PsigAttnDesc &d)
{
    const int rows = column_tiles(d.dk), tiles = kTileDots * tile_columns(d.dk);
    return rows > tiles ? rows : tiles;
}

BackwardScratch backward_scratch(const PsigAttnDesc &d, bool tiles)
{
    const long long acc = d.dtype == PSIG_F64 ? 8 : 4, rows = d.B * d.L * d.H, bh = d.B * d.H, seg = segments_of(d.L);
    BackwardScratch s{};
    long long at = 0;
    auto take = [&](long long bytes) {
        const long long here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const bool shared = d.H != d.Hkv;
    s.gq = take(tiles ? 0 : acc * rows * d.dk);
    s.gk = take(tiles && !shared ? 0 : acc * rows * d.dk);
    s.gv = take(tiles && !shared ? 0 : acc * rows * d.dv);
    // the tiles' two sets of float arrays, one array or two per column tile
    s.pairs = take((tiles ? 2 * 4 * attn_tile_dots(d.dtype) * tile_columns(d.dk) : 8) * rows);
    // the tensor-core sweeps store whole tiles of 64 by 64
    s.anchors = take(acc * bh * seg * ((d.dk + 63) / 64 * 64) * ((d.dv + 63) / 64 * 64));
    s.dots = take(acc * bh * seg * anchor_parts(d));
    s.totals = take(8 * bh * seg);
    const long long one = split_bytes(d, d.dv, d.dk), two = split_bytes(d, d.dk, d.dv);
    s.parts = take(one > two ? one : two);
    s.bytes = at;
    return s;
}

template <typename T>
int run_forward(const Call &c, const void *init, void *out, void *final, void *ws, cudaStream_t stream)
{
    Sweep s = c.forward();
    s.init = init;
    s.final = final;
    s.out = out;
    if (!c.tiles(init != nullptr && final != nullptr, out)) return sweep_rows<T>(s, stream);
    set_splits(s, ws);
    return attn_sweep_on_tiles(s, false, c.d.dtype, stream);
}

unsigned blocks_for(long long items, int per_block)
{
    const long long n = (items + per_block - 1) / per_block;
    return (unsigned)(n < 1 ? 1 : n > 148 * 32 ? 148 * 32 : n);
}

template <typename T, typename P>
int decay_gradient(const Call &c, PairSums pairs, const typename Acc<T>::type *dots, int parts, void *grad_decay,
                   double *totals, cudaStream_t stream)
{
    using A = typename Acc<T>::type;
    const PsigAttnDesc &d = c.d;
    const long long segments = segments_of(d.L);
    const bool total = per_head(d);
    int rc;
    // the grid's second dimension is limited to 65535
    const long long per_launch = 65535 / d.H > 0 ? 65535 / d.H : 1;
    const int threads = d.L < kSegment ? (int)(d.L + 31) / 32 * 32 : kSegment;   // a thread per step of a segment
    for (long long b0 = 0; b0 < d.B; b0 += per_launch) {
        const long long nb = d.B - b0 < per_launch ? d.B - b0 : per_launch;
        PairSums p = pairs;
        p.plus = static_cast<const P *>(pairs.plus) + b0 * d.L * d.H;
        p.minus = static_cast<const P *>(pairs.minus) + b0 * d.L * d.H;
        attn_decay_grad<A, P><<<dim3((unsigned)segments, (unsigned)(nb * d.H)), threads, 0, stream>>>(
            p, dots + b0 * d.H * segments * parts, parts,
            static_cast<const A *>(c.decay) + b0 * d.decay_strides[0], d.decay_strides[0], d.decay_strides[1],
            d.decay_strides[2], d.lengths == nullptr ? nullptr : d.lengths + b0, d.L, d.H,
            total ? nullptr : static_cast<A *>(grad_decay) + b0 * d.L * d.H, total ? totals + b0 * d.H * segments : nullptr);
        if ((rc = check_launch()) != PSIG_OK) return rc;
    }
    if (total) {
        attn_decay_total<A><<<(unsigned)d.H, 256, 0, stream>>>(totals, d.B, d.H, segments, static_cast<A *>(grad_decay));
        if ((rc = check_launch()) != PSIG_OK) return rc;
    }
    return PSIG_OK;
}

template <typename T>
int sum_heads(const void *acc, void *out, long long rows, int share, int d, cudaStream_t stream)
{
    using A = typename Acc<T>::type;
    attn_sum_heads<T><<<blocks_for(rows * d, 256), 256, 0, stream>>>(static_cast<const A *>(acc), static_cast<T *>(out),
                                                                     rows * d, share, d);
    return check_launch();
}

// Three sweeps on the tensor cores.  Gradients go straight to their place, in 32 bits to scratch where heads share
// a key/value head.  With a decay gradient the sweeps of grad_q and grad_k are the exact ones.
template <typename T>
int run_backward_tiles(const Call &c, const void *init, const void *gs, void *grad_q, void *grad_k, void *grad_v,
                       void *grad_decay, void *grad_init, char *ws, cudaStream_t stream)
{
    const PsigAttnDesc &d = c.d;
    const BackwardScratch at = backward_scratch(d, true);
    const long long rows = d.B * d.L * d.H, kv_rows = d.B * d.L * d.Hkv;
    const int tiles = tile_columns(d.dk);
    const bool shared = c.share > 1;
    float *x = reinterpret_cast<float *>(ws + at.pairs), *y = x + attn_tile_dots(d.dtype) * tiles * rows;
    int rc;
    Sweep s = c.grad_q();
    s.init = init;
    s.out = grad_q;
    if (grad_decay != nullptr) s.anchors = ws + at.anchors, s.keep_last = gs != nullptr, s.dot = c.q, s.dots = x;
    set_splits(s, ws + at.parts);
    if ((rc = attn_sweep_on_tiles(s, grad_decay != nullptr, d.dtype, stream)) != PSIG_OK) return rc;
    s = c.grad_k();
    s.init = gs;
    s.out = shared ? ws + at.gk : grad_k, s.out_acc = shared;
    if (grad_decay != nullptr) s.anchors = ws + at.anchors, s.anchor_dots = ws + at.dots, s.dot = c.k, s.dots = y;
    set_splits(s, ws + at.parts);
    if ((rc = attn_sweep_on_tiles(s, grad_decay != nullptr, d.dtype, stream)) != PSIG_OK) return rc;
    s = c.grad_v();
    s.init = gs;
    s.final = grad_init;
    s.out = shared ? ws + at.gv : grad_v, s.out_acc = shared;
    set_splits(s, ws + at.parts);
    if ((rc = attn_sweep_on_tiles(s, false, d.dtype, stream)) != PSIG_OK) return rc;
    if (shared) {
        if ((rc = sum_heads<T>(ws + at.gk, grad_k, kv_rows, c.share, d.dk, stream)) != PSIG_OK) return rc;
        if ((rc = sum_heads<T>(ws + at.gv, grad_v, kv_rows, c.share, d.dv, stream)) != PSIG_OK) return rc;
    }
    if (grad_decay == nullptr) return PSIG_OK;
    const int arrays = attn_tile_dots(d.dtype) * tiles;
    const PairSums pairs{x, y, arrays, arrays, rows};
    return decay_gradient<T, float>(c, pairs, reinterpret_cast<const typename Acc<T>::type *>(ws + at.dots), kTileDots * tiles,
                                    grad_decay, reinterpret_cast<double *>(ws + at.totals), stream);
}

template <typename T>
int run_backward(const Call &c, const void *init, const void *gs, void *grad_q, void *grad_k, void *grad_v,
                 void *grad_decay, void *grad_init, char *ws, long long ws_bytes, cudaStream_t stream)
{
    using A = typename Acc<T>::type;
    const bool tiles = c.tiles(false, grad_q, grad_k, grad_v);
    const long long need = backward_scratch(c.d, tiles).bytes;
    if (need > 0 && (ws == nullptr || ws_bytes < need)) return PSIG_ERR_WORKSPACE;
    if (tiles)
        return run_backward_tiles<T>(c, init, gs, grad_q, grad_k, grad_v, grad_decay, grad_init, ws, stream);
    const PsigAttnDesc &d = c.d;
    const BackwardScratch at = backward_scratch(d, false);
    const long long rows = d.B * d.L * d.H, kv_rows = d.B * d.L * d.Hkv;
    A *gq = reinterpret_cast<A *>(ws + at.gq), *gk = reinterpret_cast<A *>(ws + at.gk);
    double *pairs = reinterpret_cast<double *>(ws + at.pairs);
    int rc;
    Sweep s = c.grad_q();
    s.init = init;
    s.out = gq, s.out_acc = true;
    s.anchors = ws + at.anchors;
    if ((rc = sweep_rows<T>(s, stream)) != PSIG_OK) return rc;
    s = c.grad_k();
    s.init = gs;
    s.out = gk, s.out_acc = true;
    s.anchors = ws + at.anchors, s.anchor_dots = ws + at.dots;
    if ((rc = sweep_rows<T>(s, stream)) != PSIG_OK) return rc;
    s = c.grad_v();
    s.init = gs;
    s.final = grad_init;
    s.out = ws + at.gv, s.out_acc = true;
    if ((rc = sweep_rows<T>(s, stream)) != PSIG_OK) return rc;
    if ((rc = sum_heads<T>(gq, grad_q, rows, 1, d.dk, stream)) != PSIG_OK) return rc;
    if ((rc = sum_heads<T>(gk, grad_k, kv_rows, c.share, d.dk, stream)) != PSIG_OK) return rc;
    if ((rc = sum_heads<T>(ws + at.gv, grad_v, kv_rows, c.share, d.dv, stream)) != PSIG_OK) return rc;
    if (grad_decay == nullptr) return PSIG_OK;
    attn_pair_difference<T><<<blocks_for(rows, 8), 256, 0, stream>>>(c.q, c.k, gq, gk, pairs, rows, d.L, d.H, d.dk);
    if ((rc = check_launch()) != PSIG_OK) return rc;
    return decay_gradient<T, double>(c, PairSums{pairs, pairs, 1, 0, 0}, reinterpret_cast<const A *>(ws + at.dots),
                                     column_tiles(d.dk), grad_decay, reinterpret_cast<double *>(ws + at.totals), stream);
}

}  // namespace

int *failure_flag() { return g_failure_flag.load(std::memory_order_acquire); }

}  // namespace psig

using namespace psig;

extern "C" int64_t psig_attn_forward_workspace(const PsigAttnDesc *desc)
{
    const int rc = check_attn(desc);
    return rc != PSIG_OK ? rc : split_bytes(*desc, desc->dk, desc->dv);
}

extern "C" int64_t psig_attn_backward_workspace(const PsigAttnDesc *desc)
{
    const int rc = check_attn(desc);
    return rc != PSIG_OK ? rc : backward_scratch(*desc, Call(*desc, nullptr, nullptr, nullptr, nullptr, nullptr).tiles(false)).bytes;
}

extern "C" int psig_attn_forward(const PsigAttnDesc *desc, const void *q, const void *k, const void *v,
                                 const void *log_decay, const void *initial_state, void *out, void *final_state,
                                 void *workspace, int64_t workspace_bytes, void *stream)
{
    const int rc = check_attn(desc);
    if (rc != PSIG_OK) return rc;
    if (desc->B == 0) return PSIG_OK;
    if (desc->L > 0 && (!q || !k || !v || !log_decay || !out)) return PSIG_ERR_NULL;
    if (desc->L == 0 && final_state == nullptr) return PSIG_OK;
    const int64_t need = split_bytes(*desc, desc->dk, desc->dv);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return PSIG_ERR_WORKSPACE;
    return with_dtype(desc->dtype, [&](auto t) {
        return run_forward<decltype(t)>(Call(*desc, q, k, v, log_decay, nullptr), initial_state, out, final_state,
                                        workspace, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int psig_attn_backward(const PsigAttnDesc *desc, const void *q, const void *k, const void *v,
                                  const void *log_decay, const void *initial_state, const void *grad_out,
                                  const void *grad_state, void *grad_q, void *grad_k, void *grad_v,
                                  void *grad_log_decay, void *grad_initial_state, void *workspace,
                                  int64_t workspace_bytes, void *stream)
{
    const int rc = check_attn(desc);
    if (rc != PSIG_OK) return rc;
    if (desc->B == 0 || desc->L == 0) return PSIG_OK;   // nothing depends on the operands
    if (!q || !k || !v || !log_decay || !grad_out || !grad_q || !grad_k || !grad_v) return PSIG_ERR_NULL;
    return with_dtype(desc->dtype, [&](auto t) {
        return run_backward<decltype(t)>(Call(*desc, q, k, v, log_decay, grad_out), initial_state, grad_state, grad_q, grad_k,
                                         grad_v, grad_log_decay, grad_initial_state, static_cast<char *>(workspace),
                                         workspace_bytes, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int64_t psig_sequence_wait_timeouts(void) { return attn_tile_timeouts() + attn_split_timeouts() + norm_timeouts(); }

extern "C" int psig_set_sequence_failure_flag(int32_t *flag)
{
    g_failure_flag.store(flag, std::memory_order_release);
    return PSIG_OK;
}

extern "C" int psig_attn_step(const PsigAttnDesc *desc, const void *q, const void *k, const void *v,
                              const void *log_decay, void *state, void *out, void *stream)
{
    const int rc = check_attn(desc);
    if (rc != PSIG_OK) return rc;
    if (desc->B == 0) return PSIG_OK;
    if (!q || !k || !v || !log_decay || !state || !out) return PSIG_ERR_NULL;
    const int share = desc->H / desc->Hkv;
    const dim3 grid((unsigned)(desc->B * desc->H), (unsigned)column_tiles(desc->dv));
    return with_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        using A = typename Acc<T>::type;
        if constexpr (sizeof(A) == 4)
            if (desc->dv % 4 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0) {
                const long long blocks = desc->B * desc->H * ((desc->dv + 127) / 128);
                auto launch = [&](auto kernel, int cols) {
                    kernel<<<dim3((unsigned)(desc->B * desc->H), (unsigned)((desc->dv + cols - 1) / cols)), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                        operand(q, desc->q_strides, 1), operand(k, desc->k_strides, share), operand(v, desc->v_strides, share),
                        static_cast<const float *>(log_decay), desc->decay_strides[0], desc->decay_strides[2], static_cast<float *>(state),
                        static_cast<T *>(out), desc->H, desc->dk, desc->dv, (float)desc->scale);
                    return check_launch();
                };
                // wide blocks once they fill the SMs several times
                return blocks >= 148 * 4 && desc->dv > 32 ? launch(attn_step_vector<T, 128>, 128) : launch(attn_step_vector<T, 32>, 32);
            }
        attn_step_rows<T><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
            operand(q, desc->q_strides, 1), operand(k, desc->k_strides, share), operand(v, desc->v_strides, share),
            static_cast<const A *>(log_decay), desc->decay_strides[0], desc->decay_strides[2], static_cast<A *>(state),
            static_cast<T *>(out), desc->H, desc->dk, desc->dv, desc->scale);
        return check_launch();
    });
}
