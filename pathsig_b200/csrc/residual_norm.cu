// Norm around a block, fused with the block's gate, the residual sum and the norm before the next block.
//     z = x r w,  r = (mean(x^2) + eps)^(-1/2);   u = z act(gate);   h = residual + c u;
//     n = h r2 w2,  r2 = (mean(h^2) + eps)^(-1/2)
// Backward, per row, with the total gradient of h first:
//     dh += r2 (w2 dn) - h r2^3 mean(w2 dn h)            dw2 += dn h r2
//     dresidual = dh,  dc += dh u,  dgate = dh c z act'(gate),  dz = dh c act(gate),  dw += dz x r
//     dx = r (w dz) - x r^3 mean(w dz x)
// h is recomputed from the operands (the residual is read where a saved h would have been), so that nothing of
// the forward pass is kept and h is not rounded in between.  Sums are in 32 bits (64 for float64).
//
// What bounds it: memory, each operand once.  A row is held in registers by a team of threads (part of a warp for short rows,
// a whole block else), 8 or 16 values to a thread, in accesses of 16 bytes where the rows allow it; sums over the row
// are the only exchange, by shuffles and, between warps, one barrier each.  Rows too wide for that are walked in
// pieces and read again, mostly from L2.
#include "sequence.cuh"

#include <atomic>

namespace psig {
namespace {

constexpr int kTeamMax = 512;                  // threads of a block that holds one row
constexpr int kNormWidest = kTeamMax * 16;     // widest row held in registers
constexpr int kShortThreads = 256;             // block size for rows of at most one warp
constexpr int kWideThreads = 512;              // block size for rows that are walked

struct NormArgs {
    const void *x, *gate, *residual, *grad_h, *grad_n;
    const void *weight, *scale, *next_weight;
    void *h, *n;
    void *grad_x, *grad_gate, *grad_residual;
    void *partial;   // (blocks, 3, D) sums for weight, scale, next_weight
    long long rows, D;
    double mean, eps;      // 1 / D
    float mean_f, eps_f;   // the same: converting costs a thread as much as some values of its row
    int activation;
    int *failure;          // see failure_flag
};

template <typename A> __device__ __forceinline__ A scalar(double wide, float narrow)
{
    if constexpr (sizeof(A) == 8) return wide;
    else return narrow;
}

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

// E neighbouring values as one access.
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

// The E values of an access in the type of sums, and back (16-bit types two at a time).
template <typename T, int E>
__device__ __forceinline__ void widen(const Pack<T, E> &p, typename Acc<T>::type (&x)[E])
{
    if constexpr (std::is_same<T, __nv_bfloat16>::value && E > 1) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(&p.bits);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            x[e] = __uint_as_float(w[e / 2] << 16);
            x[e + 1] = __uint_as_float(w[e / 2] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = to_acc<typename Acc<T>::type>(p.v[e]);
    }
}
template <typename T, int E>
__device__ __forceinline__ void narrow(const typename Acc<T>::type (&x)[E], Pack<T, E> &p)
{
    if constexpr (sizeof(T) == 2 && E > 1) {
        uint32_t *w = reinterpret_cast<uint32_t *>(&p.bits);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(x[e], x[e + 1]);
                w[e / 2] = *reinterpret_cast<const uint32_t *>(&two);
            } else {
                const __half2 two = __floats2half2_rn(x[e], x[e + 1]);
                w[e / 2] = *reinterpret_cast<const uint32_t *>(&two);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) p.v[e] = from_acc<T>(x[e]);
    }
}

// E values of a parameter vector (type of sums; 16-byte aligned where E > 1); 1 where there is none.
template <typename A, int E>
__device__ __forceinline__ void load_vector(const void *p, long long at, A (&v)[E])
{
    if (p == nullptr) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = A(1);
        return;
    }
    constexpr int W = 16 / (int)sizeof(A) < E ? 16 / (int)sizeof(A) : E;
#pragma unroll
    for (int e = 0; e < E; e += W) {
        Pack<A, W> w;
        w.load(p, at + e);
#pragma unroll
        for (int i = 0; i < W; ++i) v[e + i] = w.v[i];
    }
}

// 1 / (1 + exp(-g)), good to the type of sums for rows of that type (in 32 bits with the hardware's reciprocal, which is one
// place off at most; a division took 370 us for the forward pass of 15616 x 4680 with gate and residual, this 296, the
// form for 16 bits 281).  For 16-bit rows with the hardware's exponential too: the rounding of g / ln 2 is relative to |g|, so
// that it is up to |g| + 8 units of 2^-24 off, 2^-17 where the result is not below 2^-126, far below their half step.
template <typename T>
__device__ __forceinline__ typename Acc<T>::type sigmoid(typename Acc<T>::type g)
{
    using A = typename Acc<T>::type;
    if constexpr (sizeof(A) == 8) {
        return A(1) / (A(1) + exp_acc(-g));
    } else {
        float e, s;
        if constexpr (sizeof(T) == 2) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
        else e = expf(-g);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
        return s;
    }
}

template <typename T>
__device__ __forceinline__ typename Acc<T>::type gate_value(typename Acc<T>::type g, int activation)
{
    const auto s = sigmoid<T>(g);
    return activation == 0 ? g * s : s;
}
template <typename T>
__device__ __forceinline__ typename Acc<T>::type gate_slope(typename Acc<T>::type g, int activation)
{
    using A = typename Acc<T>::type;
    const A s = sigmoid<T>(g);
    return activation == 0 ? s * (A(1) + g * (A(1) - s)) : s * (A(1) - s);
}

__device__ __forceinline__ float inverse_root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return rsqrt(v); }

// Sums N values over the team: 2^team_log2 neighbouring lanes, or the whole block when team_log2 is 5.  Partial sums
// of the warps go to one of two sets in turn (`round`), so that one barrier is enough.
template <typename A, int N>
__device__ __forceinline__ void team_sum(A (&v)[N], int team_log2, A *shared, int round)
{
    for (int s = 0; s < team_log2; ++s)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 1 << s);
    if (team_log2 < 5) return;
    if (blockDim.x == 32) {
        __syncwarp();
        return;
    }
    A *mine = shared + (round & 1) * 2 * (kTeamMax / 32);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) mine[(threadIdx.x >> 5) * 2 + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = A(0);
    for (int w = 0; w < blockDim.x >> 5; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += mine[w * 2 + i];
}

// ---- rows held by a team ----
//
// RING: the rows of one block are streamed into shared memory ahead of their use (one thread, cp.async.bulk, an mbarrier
// for each of the stages), so that the memory system is busy while a row waits at its barriers; every pass
// reads its operands from there.  Needs rows that are whole 16-byte pieces.  Otherwise a thread loads its part of a row itself.
// Waits for a row are bounded.  When one runs out the block leaves its loop -- all threads at once: the flag is set before
// the row's first barrier, read behind it, and not set for the next row before another barrier -- writes nothing from that row
// on, and waits (bounded again) for the copies in flight before it gives its shared memory back.

__device__ __forceinline__ uint32_t norm_shared(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

constexpr int kNormOperands = 5;
// Polls of a row's wait; a test lowers it to make the wait run out.  The wait for the copies in flight keeps its own limit.
std::atomic<unsigned> g_row_polls{kWaitPolls};
__device__ unsigned long long g_norm_timeouts;

struct Ring {
    int stages;
    unsigned polls;                      // of the wait for a row
    int row_bytes;                       // of one operand
    int count;                           // operands per stage
    const void *data[kNormOperands];     // in the order of their slots
};

struct RingState {
    unsigned char *buffer;
    uint32_t bars;
    const Ring &ring;
    volatile int *failed;   // of the block
    __device__ __forceinline__ uint32_t bar(int stage) const { return bars + 8 * stage; }
    __device__ __forceinline__ void init() const
    {
        *failed = 0;
        for (int i = 0; i < ring.stages; ++i)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar(i)) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // one thread: row `row` into stage `stage`
    __device__ __forceinline__ void load(int stage, long long row) const
    {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar(stage)), "r"(ring.count * ring.row_bytes) : "memory");
        for (int i = 0; i < ring.count; ++i)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(norm_shared(buffer + (long long)(stage * ring.count + i) * ring.row_bytes)),
                           "l"(static_cast<const unsigned char *>(ring.data[i]) + row * ring.row_bytes), "r"(ring.row_bytes), "r"(bar(stage))
                         : "memory");
    }
    __device__ __forceinline__ bool arrived(int stage, uint32_t parity, unsigned polls) const
    {
        unsigned long long start = 0;
        for (unsigned i = 0; i < polls; ++i) {
            uint32_t ok;
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                         : "=r"(ok) : "r"(bar(stage)), "r"(parity) : "memory");
            if (ok) return true;
            if (wait_expired(i, start)) break;
        }
        return false;
    }
    __device__ __forceinline__ void wait(int stage, uint32_t parity) const
    {
        if (!arrived(stage, parity, ring.polls)) *failed = 1;
    }
    // one thread, behind a wait that ran out for row `row` in `stage`: the copies of that row and of the rows behind it, as many
    // as there are stages, have been started
    __device__ __forceinline__ void drain(int stage, uint32_t parity, long long row, long long step, long long rows, int *failure) const
    {
        atomicAdd(&g_norm_timeouts, 1ull);
        report_failure(failure);
        for (int i = 0; i < ring.stages && row + i * step < rows; ++i) {
            const int s = stage + i;
            arrived(s < ring.stages ? s : s - ring.stages, s < ring.stages ? parity : parity ^ 1, kWaitPolls);
        }
    }
};

template <typename T, int E, int NV, bool NEXT, bool RING>
__global__ void __launch_bounds__(kTeamMax) norm_forward_team(const NormArgs a, int team_log2, int threads, const Ring ring)
{
    using A = typename Acc<T>::type;
    __shared__ A shared[4 * (kTeamMax / 32)];
    extern __shared__ __align__(128) unsigned char dynamic[];
    const int teams = team_log2 < 5 ? blockDim.x >> team_log2 : 1;
    const int team = team_log2 < 5 ? threadIdx.x >> team_log2 : 0, j = team_log2 < 5 ? threadIdx.x & (threads - 1) : threadIdx.x;
    const A mean = scalar<A>(a.mean, a.mean_f), eps = scalar<A>(a.eps, a.eps_f);
    const long long step = (long long)gridDim.x * teams;
    const RingState rs{dynamic + 128, norm_shared(dynamic), ring, reinterpret_cast<int *>(dynamic + 64)};
    if (RING) {
        if (threadIdx.x == 0) {
            rs.init();
            for (int i = 0; i < ring.stages; ++i)
                if (blockIdx.x + i * step < a.rows) rs.load(i, blockIdx.x + i * step);
        }
        __syncthreads();
    }
    int round = 0, stage = 0;
    uint32_t phase = 0;
    for (long long first = (long long)blockIdx.x * teams; first < a.rows; first += step) {
        const long long row = first + team, base = row * a.D;
        const int D = row < a.rows ? (int)a.D : 0;
        Pack<T, E> x[NV], g[NV], res[NV];
        const unsigned char *here = rs.buffer + (long long)stage * ring.count * ring.row_bytes;
        if (RING) rs.wait(stage, phase);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = (j + v * threads) * E;
            if (col >= D) continue;
            if (RING) {
                x[v].load(here, col);
            } else {
                x[v].load(a.x, base + col);
                if (a.gate) g[v].load(a.gate, base + col);
                if (a.residual) res[v].load(a.residual, base + col);
            }
        }
        A sum[1] = {A(0)};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            A t[E];
            widen(x[v], t);
#pragma unroll
            for (int e = 0; e < E; ++e) sum[0] += t[e] * t[e];
        }
        team_sum(sum, team_log2, shared, round++);
        if (RING && *rs.failed) {
            if (threadIdx.x == 0) rs.drain(stage, phase, first, step, a.rows, a.failure);
            break;
        }
        const A r = inverse_root(sum[0] * mean + eps);
        A h[NEXT ? NV * E : 1];
        sum[0] = A(0);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = (j + v * threads) * E;
            if (col >= D) continue;
            if (RING) {
                if (a.gate) g[v].load(here + ring.row_bytes, col);
                if (a.residual) res[v].load(here + (a.gate ? 2 : 1) * ring.row_bytes, col);
            }
            A f[E];
            load_vector<A, E>(a.weight, col, f);
            if (a.scale) {
                A c[E];
                load_vector<A, E>(a.scale, col, c);
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] *= c[e];
            }
            A t[E];
            if (a.gate) {
                widen(g[v], t);
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] *= sigmoid<T>(t[e]);
                if (a.activation == 0)
#pragma unroll
                    for (int e = 0; e < E; ++e) f[e] *= t[e];
            }
            widen(x[v], t);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] *= t[e] * r;
            if (a.residual) {
                widen(res[v], t);
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] += t[e];
            }
            if (NEXT)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    h[NEXT ? v * E + e : 0] = f[e];
                    sum[0] += f[e] * f[e];
                }
            Pack<T, E> out;
            narrow(f, out);
            out.store(a.h, base + col);
        }
        if (NEXT || RING) team_sum(sum, team_log2, shared, round++);   // RING: also tells that the stage has been read
        if (RING) {
            if (threadIdx.x == 0 && first + ring.stages * step < a.rows) rs.load(stage, first + ring.stages * step);
            if (++stage == ring.stages) stage = 0, phase ^= 1;
        }
        if (!NEXT) continue;
        const A r2 = inverse_root(sum[0] * mean + eps);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = (j + v * threads) * E;
            if (col >= D) continue;
            A w[E];
            load_vector<A, E>(a.next_weight, col, w);
            Pack<T, E> out;
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] *= h[NEXT ? v * E + e : 0] * r2;
            narrow(w, out);
            out.store(a.n, base + col);
        }
    }
}

// Blocks walk the rows; a thread keeps the sums over rows for its own columns in registers: q = sum dh act x r, which
// is the gradient of weight but for the factor residual_scale of the column, and the other way round, and sum dn h r2.
// NEXT: with the norm before the next block (three exchanges a row instead of one).
// Registers: where float32 rows are streamed without the next norm, so many that an SM holds two blocks of 320 threads (15616 x 4680
// signatures 170 us, 220 with two registers more and one block); else what a block of 512 threads can have (a bound on the
// block's size instead made the compiler stop at 64 for eight values to a thread: 15616 x 1528 81 us, in this form 64).
template <typename T, int E, int NV, bool NEXT, bool RING>
__global__ void __maxnreg__(RING && !NEXT && NV * E == 16 && sizeof(T) == 4 ? 96 : 128) norm_backward_team(const NormArgs a, int team_log2, int threads, const Ring ring)
{
    using A = typename Acc<T>::type;
    __shared__ A shared[4 * (kTeamMax / 32)];
    extern __shared__ __align__(128) unsigned char dynamic[];
    const int teams = team_log2 < 5 ? blockDim.x >> team_log2 : 1;
    const int team = team_log2 < 5 ? threadIdx.x >> team_log2 : 0, j = team_log2 < 5 ? threadIdx.x & (threads - 1) : threadIdx.x;
    constexpr bool KEEP = NV * E == 8;       // column constants and the next row fit in registers
    constexpr bool PREFETCH = KEEP && !RING;
    const A mean = scalar<A>(a.mean, a.mean_f), eps = scalar<A>(a.eps, a.eps_f);
    const int D = (int)a.D;
    const long long step = (long long)gridDim.x * teams;
    A q[NV * E], qn[NEXT ? NV * E : 1], wc_kept[KEEP ? NV * E : 1], w2_kept[KEEP && NEXT ? NV * E : 1];
    auto product = [&](int col, A (&f)[E]) {   // weight times residual_scale
        load_vector<A, E>(a.weight, col, f);
        if (a.scale) {
            A c[E];
            load_vector<A, E>(a.scale, col, c);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] *= c[e];
        }
    };
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int col = (j + v * threads) * E;
        A f[E], w[E];
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = w[e] = A(0);
        if (KEEP && col < D) {
            product(col, f);
            if (NEXT) load_vector<A, E>(a.next_weight, col, w);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            q[v * E + e] = A(0);
            if (NEXT) qn[NEXT ? v * E + e : 0] = A(0);
            if (KEEP) wc_kept[KEEP ? v * E + e : 0] = f[e];
            if (KEEP && NEXT) w2_kept[KEEP && NEXT ? v * E + e : 0] = w[e];
        }
    }
    struct Operands { Pack<T, E> x, g, res, gh, gn; };
    Operands now[RING ? 1 : NV];
    auto fetch = [&](auto &o, long long row) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = (j + v * threads) * E;
            if (row < a.rows && col < D) {
                const long long at = row * a.D + col;
                o[v].x.load(a.x, at);
                if (a.gate) o[v].g.load(a.gate, at);
                if (NEXT && a.residual) o[v].res.load(a.residual, at);
                if (a.grad_h) o[v].gh.load(a.grad_h, at);
                if (NEXT) o[v].gn.load(a.grad_n, at);
            }
        }
    };
    const RingState rs{dynamic + 128, norm_shared(dynamic), ring, reinterpret_cast<int *>(dynamic + 64)};
    if (RING) {
        if (threadIdx.x == 0) {
            rs.init();
            for (int i = 0; i < ring.stages; ++i)
                if (blockIdx.x + i * step < a.rows) rs.load(i, blockIdx.x + i * step);
        }
        __syncthreads();
    } else if (PREFETCH) {
        fetch(now, (long long)blockIdx.x * teams + team);
    }
    int round = 0, stage = 0;
    uint32_t phase = 0;
    for (long long first = (long long)blockIdx.x * teams; first < a.rows; first += step) {
        const long long row = first + team, base = row * a.D;
        const bool live_row = row < a.rows;
        Operands next[PREFETCH ? NV : 1];
        const unsigned char *here = rs.buffer + (long long)stage * ring.count * ring.row_bytes;
        if (RING) rs.wait(stage, phase);
        else if constexpr (PREFETCH) fetch(next, row + step);
        else fetch(now, row);
        // operand number `slot` of the stage: x, then gate, residual, grad_h, grad_n as far as they are there
        int slot = 1;
        const unsigned char *at_g = here + (a.gate ? slot++ : 0) * ring.row_bytes, *at_res = here + (NEXT && a.residual ? slot++ : 0) * ring.row_bytes;
        const unsigned char *at_gh = here + (a.grad_h ? slot++ : 0) * ring.row_bytes, *at_gn = here + (NEXT ? slot++ : 0) * ring.row_bytes;
        auto get = [&](int v, const unsigned char *at, bool given, const Pack<T, E> &held) {
            Pack<T, E> p;
            if (!RING) return held;
            const int col = (j + v * threads) * E;
            if (given && col < D) p.load(at, col);
            return p;
        };
#define PSIG_OPERAND(v, at, given, name) get(v, at, given, now[RING ? 0 : v].name)
        A r, r2 = A(0), m2 = A(0), m;
        A dh[NV * E], f[NV * E], sig[NV * E];   // gradient of h; factor of x in u, without r; sigmoid of the gate
        A two[2] = {A(0), A(0)}, one[1] = {A(0)};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = (j + v * threads) * E;
            const Pack<T, E> x = PSIG_OPERAND(v, here, true, x), gh = PSIG_OPERAND(v, at_gh, a.grad_h != nullptr, gh);
            A fv[E];
#pragma unroll
            for (int e = 0; e < E; ++e) fv[e] = KEEP ? wc_kept[KEEP ? v * E + e : 0] : A(0);
            if (!KEEP && col < D) product(col, fv);
            A t[E], d[E];
            if (a.gate) {
                widen(PSIG_OPERAND(v, at_g, true, g), t);
#pragma unroll
                for (int e = 0; e < E; ++e) fv[e] *= sig[v * E + e] = sigmoid<T>(t[e]);
                if (a.activation == 0)
#pragma unroll
                    for (int e = 0; e < E; ++e) fv[e] *= t[e];
            }
            widen(x, t);
            widen(gh, d);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                f[v * E + e] = fv[e];
                dh[v * E + e] = d[e];
                two[0] += t[e] * t[e];
                if (!NEXT) two[1] += d[e] * fv[e] * t[e];
            }
        }
        if (!NEXT) {   // the gradient of h is there: both sums in one exchange
            team_sum(two, team_log2, shared, round++);
        } else {
            one[0] = two[0];
            team_sum(one, team_log2, shared, round++);
        }
        if (RING && *rs.failed) {
            if (threadIdx.x == 0) rs.drain(stage, phase, first, step, a.rows, a.failure);
            break;
        }
        if (!NEXT) {
            r = inverse_root(two[0] * mean + eps);
            m = two[1] * mean * r * r * r;
        } else {
            r = inverse_root(one[0] * mean + eps);
            two[0] = two[1] = A(0);
            A h[NV * E];
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int col = (j + v * threads) * E;
                const Pack<T, E> x = PSIG_OPERAND(v, here, true, x), gn = PSIG_OPERAND(v, at_gn, true, gn);
                const Pack<T, E> res = PSIG_OPERAND(v, at_res, a.residual != nullptr, res);
                A w2[E];
#pragma unroll
                for (int e = 0; e < E; ++e) w2[e] = KEEP ? w2_kept[KEEP && NEXT ? v * E + e : 0] : A(0);
                if (!KEEP && col < D) load_vector<A, E>(a.next_weight, col, w2);
                A t[E], u[E], d[E];
                widen(x, t);
                widen(res, u);
                widen(gn, d);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int i = v * E + e;
                    h[i] = t[e] * r * f[i] + u[e];
                    two[0] += h[i] * h[i];
                    two[1] += w2[e] * d[e] * h[i];
                }
            }
            team_sum(two, team_log2, shared, round++);
            r2 = inverse_root(two[0] * mean + eps);
            m2 = two[1] * mean * r2 * r2 * r2;
            one[0] = A(0);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int col = (j + v * threads) * E;
                const Pack<T, E> x = PSIG_OPERAND(v, here, true, x), gn = PSIG_OPERAND(v, at_gn, true, gn);
                A w2[E];
#pragma unroll
                for (int e = 0; e < E; ++e) w2[e] = KEEP ? w2_kept[KEEP && NEXT ? v * E + e : 0] : A(0);
                if (!KEEP && col < D) load_vector<A, E>(a.next_weight, col, w2);
                A t[E], d[E];
                widen(x, t);
                widen(gn, d);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int i = v * E + e;
                    const A dn = d[e] * r2;
                    dh[i] += w2[e] * dn - h[i] * m2;
                    // a team without a row holds zeros, whose root with eps = 0 is infinite
                    if (live_row) qn[NEXT ? i : 0] += dn * h[i];
                    one[0] += dh[i] * f[i] * t[e];
                }
            }
            team_sum(one, team_log2, shared, round++);
            m = one[0] * mean * r * r * r;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = (j + v * threads) * E;
            if (!live_row || col >= D) continue;
            A t[E], o[E];
            widen(PSIG_OPERAND(v, here, true, x), t);
            Pack<T, E> out;
            if (a.grad_residual) {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = dh[v * E + e];
                narrow(o, out);
                out.store(a.grad_residual, base + col);
            }
            if (a.grad_x) {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = r * f[v * E + e] * dh[v * E + e] - t[e] * m;
                narrow(o, out);
                out.store(a.grad_x, base + col);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) t[e] *= dh[v * E + e] * r;
            if (a.gate) {
                A g[E], fv[E];
                widen(PSIG_OPERAND(v, at_g, true, g), g);
#pragma unroll
                for (int e = 0; e < E; ++e) fv[e] = KEEP ? wc_kept[KEEP ? v * E + e : 0] : A(0);
                if (!KEEP) product(col, fv);
                if (a.activation == 0) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const A s1 = sig[v * E + e], act = g[e] * s1;
                        o[e] = t[e] * fv[e] * (s1 + act * (A(1) - s1));
                        q[v * E + e] += t[e] * act;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const A s1 = sig[v * E + e];
                        o[e] = t[e] * fv[e] * (s1 * (A(1) - s1));
                        q[v * E + e] += t[e] * s1;
                    }
                }
                narrow(o, out);
                if (a.grad_gate) out.store(a.grad_gate, base + col);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) q[v * E + e] += t[e];
            }
        }
#undef PSIG_OPERAND
        if (RING) {
            __syncthreads();   // the stage has been read
            if (threadIdx.x == 0 && first + ring.stages * step < a.rows) rs.load(stage, first + ring.stages * step);
            if (++stage == ring.stages) stage = 0, phase ^= 1;
        }
        if constexpr (PREFETCH)
#pragma unroll
            for (int v = 0; v < NV; ++v) now[v] = next[v];
    }
    // the block's teams hold the same columns: fold them in order
    A *fold = reinterpret_cast<A *>(dynamic);
    A *part = static_cast<A *>(a.partial) + (long long)blockIdx.x * 3 * a.D;
#pragma unroll
    for (int which = 0; which < (NEXT ? 2 : 1); ++which) {
        if (which == 0 && a.weight == nullptr && a.scale == nullptr) continue;
        if (teams > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV * E; ++i) fold[i * blockDim.x + threadIdx.x] = which == 0 ? q[i] : qn[NEXT ? i : 0];
            __syncthreads();
        }
        if (team != 0) continue;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = (j + v * threads) * E;
            if (col >= D) continue;
            A w[E], c[E];
            load_vector<A, E>(a.weight, col, w);
            load_vector<A, E>(a.scale, col, c);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = v * E + e;
                A s = which == 0 ? q[i] : qn[NEXT ? i : 0];
                for (int k = 1; k < teams; ++k) s += fold[i * blockDim.x + (k << team_log2) + j];
                if (which == 1) part[2 * a.D + col + e] = s;
                else if (a.weight) part[col + e] = s * c[e];
                if (which == 0 && a.scale) part[a.D + col + e] = s * w[e];
            }
        }
    }
}

// ---- rows wider than a block holds: walked in accesses of E values, read again for each sum ----

template <typename T, int E>
__device__ __forceinline__ void wide_values(const NormArgs &a, long long base, long long col,
                                            typename Acc<T>::type r, typename Acc<T>::type (&x)[E], typename Acc<T>::type (&f)[E],
                                            typename Acc<T>::type (&h)[E])
{
    using A = typename Acc<T>::type;
    Pack<T, E> p, g, res;
    p.load(a.x, base + col);
    if (a.gate) g.load(a.gate, base + col);
    if (a.residual) res.load(a.residual, base + col);
    load_vector<A, E>(a.weight, col, f);
    if (a.scale) {
        A c[E];
        load_vector<A, E>(a.scale, col, c);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] *= c[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (a.gate) f[e] *= gate_value<T>(to_acc<A>(g.v[e]), a.activation);
        x[e] = to_acc<A>(p.v[e]);
        h[e] = x[e] * r * f[e] + to_acc<A>(res.v[e]);
    }
}

template <typename T, int E>
__global__ void __launch_bounds__(kWideThreads) norm_forward_wide(const NormArgs a)
{
    using A = typename Acc<T>::type;
    __shared__ A shared[4 * (kTeamMax / 32)];
    const A mean = scalar<A>(a.mean, a.mean_f), eps = scalar<A>(a.eps, a.eps_f);
    int round = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long base = row * a.D;
        A sum[1] = {A(0)};
#pragma unroll 4
        for (long long col = threadIdx.x * E; col < a.D; col += kWideThreads * E) {
            Pack<T, E> p;
            p.load(a.x, base + col);
#pragma unroll
            for (int e = 0; e < E; ++e) { const A t = to_acc<A>(p.v[e]); sum[0] += t * t; }
        }
        team_sum(sum, 5, shared, round++);
        const A r = inverse_root(sum[0] * mean + eps);
        sum[0] = A(0);
        for (long long col = threadIdx.x * E; col < a.D; col += kWideThreads * E) {
            A x[E], f[E], h[E];
            wide_values<T, E>(a, base, col, r, x, f, h);
            Pack<T, E> out;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                out.v[e] = from_acc<T>(h[e]);
                sum[0] += h[e] * h[e];
            }
            out.store(a.h, base + col);
        }
        if (a.next_weight == nullptr) continue;
        team_sum(sum, 5, shared, round++);
        const A r2 = inverse_root(sum[0] * mean + eps);
        for (long long col = threadIdx.x * E; col < a.D; col += kWideThreads * E) {
            A x[E], f[E], h[E], w[E];
            wide_values<T, E>(a, base, col, r, x, f, h);
            load_vector<A, E>(a.next_weight, col, w);
            Pack<T, E> out;
#pragma unroll
            for (int e = 0; e < E; ++e) out.v[e] = from_acc<T>(h[e] * r2 * w[e]);
            out.store(a.n, base + col);
        }
    }
}

// The block's sums over its rows are kept in its part of the workspace, each entry by the thread that owns the column.
template <typename T, int E>
__global__ void __launch_bounds__(kWideThreads) norm_backward_wide(const NormArgs a)
{
    using A = typename Acc<T>::type;
    __shared__ A shared[4 * (kTeamMax / 32)];
    const A mean = scalar<A>(a.mean, a.mean_f), eps = scalar<A>(a.eps, a.eps_f);
    A *part = static_cast<A *>(a.partial) + (long long)blockIdx.x * 3 * a.D;
    int round = 0;
    bool fresh = true;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long base = row * a.D;
        A one[1] = {A(0)}, two[2] = {A(0), A(0)};
#pragma unroll 4
        for (long long col = threadIdx.x * E; col < a.D; col += kWideThreads * E) {
            Pack<T, E> p;
            p.load(a.x, base + col);
#pragma unroll
            for (int e = 0; e < E; ++e) { const A t = to_acc<A>(p.v[e]); one[0] += t * t; }
        }
        team_sum(one, 5, shared, round++);
        const A r = inverse_root(one[0] * mean + eps);
        A r2 = A(0), m2 = A(0);
        if (a.next_weight != nullptr) {
            for (long long col = threadIdx.x * E; col < a.D; col += kWideThreads * E) {
                A x[E], f[E], h[E], w2[E];
                Pack<T, E> gn;
                wide_values<T, E>(a, base, col, r, x, f, h);
                load_vector<A, E>(a.next_weight, col, w2);
                gn.load(a.grad_n, base + col);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    two[0] += h[e] * h[e];
                    two[1] += w2[e] * to_acc<A>(gn.v[e]) * h[e];
                }
            }
            team_sum(two, 5, shared, round++);
            r2 = inverse_root(two[0] * mean + eps);
            m2 = two[1] * mean * r2 * r2 * r2;
        }
        auto gradient = [&](long long col, const A (&h)[E], A (&dh)[E], A (&dn)[E]) {
            Pack<T, E> gh;
            if (a.grad_h) gh.load(a.grad_h, base + col);
#pragma unroll
            for (int e = 0; e < E; ++e) dh[e] = to_acc<A>(gh.v[e]), dn[e] = A(0);
            if (a.next_weight != nullptr) {
                A w2[E];
                Pack<T, E> gn;
                load_vector<A, E>(a.next_weight, col, w2);
                gn.load(a.grad_n, base + col);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    dn[e] = to_acc<A>(gn.v[e]);
                    dh[e] += w2[e] * dn[e] * r2 - h[e] * m2;
                }
            }
        };
        one[0] = A(0);
        for (long long col = threadIdx.x * E; col < a.D; col += kWideThreads * E) {
            A x[E], f[E], h[E], dh[E], dn[E];
            wide_values<T, E>(a, base, col, r, x, f, h);
            gradient(col, h, dh, dn);
#pragma unroll
            for (int e = 0; e < E; ++e) one[0] += dh[e] * f[e] * x[e];
        }
        team_sum(one, 5, shared, round++);
        const A m = one[0] * mean * r * r * r;
        for (long long col = threadIdx.x * E; col < a.D; col += kWideThreads * E) {
            A x[E], f[E], h[E], dh[E], dn[E], w[E], c[E];
            wide_values<T, E>(a, base, col, r, x, f, h);
            gradient(col, h, dh, dn);
            load_vector<A, E>(a.weight, col, w);
            load_vector<A, E>(a.scale, col, c);
            Pack<T, E> out_x, out_g, out_r, g;
            if (a.gate) g.load(a.gate, base + col);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                A act = A(1), slope = A(0);
                if (a.gate) {
                    act = gate_value<T>(to_acc<A>(g.v[e]), a.activation);
                    slope = gate_slope<T>(to_acc<A>(g.v[e]), a.activation);
                }
                const A t = dh[e] * act * x[e] * r;
                if (a.weight) part[col + e] = (fresh ? A(0) : part[col + e]) + t * c[e];
                if (a.scale) part[a.D + col + e] = (fresh ? A(0) : part[a.D + col + e]) + t * w[e];
                if (a.next_weight) part[2 * a.D + col + e] = (fresh ? A(0) : part[2 * a.D + col + e]) + dn[e] * h[e] * r2;
                out_r.v[e] = from_acc<T>(dh[e]);
                out_g.v[e] = from_acc<T>(dh[e] * c[e] * w[e] * x[e] * r * slope);
                out_x.v[e] = from_acc<T>(r * f[e] * dh[e] - x[e] * m);
            }
            if (a.grad_residual) out_r.store(a.grad_residual, base + col);
            if (a.grad_gate) out_g.store(a.grad_gate, base + col);
            if (a.grad_x) out_x.store(a.grad_x, base + col);
        }
        fresh = false;
    }
}

// Sums of the blocks' partial rows, in a fixed order: 32 columns to a block, its warps take the partial rows in turn, then the
// columns.  Few columns are few blocks, so the loads in flight count: 32 warps (17909 x 376 8.8 -> 4.8 us, 15616 x 1024 9.3 -> 5.2);
// where the columns fill the SMs 8 are quicker (12794 x 8192 9.8 us, 12.2 with 32).
template <typename A>
__global__ void __launch_bounds__(1024) norm_sum_partials(const A *__restrict__ partial, int blocks, long long D,
                                                         A *__restrict__ out_w, A *__restrict__ out_c, A *__restrict__ out_w2)
{
    __shared__ A shared[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const long long col = (long long)blockIdx.x * 32 + lane;
    A *out = blockIdx.y == 0 ? out_w : blockIdx.y == 1 ? out_c : out_w2;
    if (out == nullptr) return;
    A sum = A(0);
    if (col < D)
#pragma unroll 4
        for (int b = warp; b < blocks; b += warps) sum += partial[((long long)b * 3 + blockIdx.y) * D + col];
    shared[warp][lane] = sum;
    __syncthreads();
    for (int c = warp; c < 32; c += warps) {
        sum = lane < warps ? shared[lane][c] : A(0);
        for (int i = 16; i >= 1; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
        const long long own = (long long)blockIdx.x * 32 + c;
        if (lane == 0 && own < D) out[own] = sum;
    }
}

int check_norm(const PsigNormDesc *d)
{
    if (d == nullptr) return PSIG_ERR_NULL;
    if (d->dtype < PSIG_F32 || d->dtype > PSIG_F16) return PSIG_ERR_DTYPE;
    if (d->rows < 0 || d->D < 1 || d->activation < 0 || d->activation > 1) return PSIG_ERR_SHAPE;
    return PSIG_OK;
}

void set_sizes(NormArgs &a, const PsigNormDesc &d)
{
    a.rows = d.rows, a.D = d.D, a.activation = d.activation;
    a.mean = 1.0 / (double)d.D, a.eps = d.eps;
    a.mean_f = (float)a.mean, a.eps_f = (float)a.eps;
    a.failure = failure_flag();
}

// How a row is dealt to threads: 8 values to a thread, 16 where the row would need more than 256 threads.
struct TeamPlan {
    int team_log2, threads, block;   // log2 of the team inside a warp (5: the block is the team); threads per row; block size
    int values;                      // per thread
    int teams() const { return team_log2 < 5 ? block >> team_log2 : 1; }
};

TeamPlan team_plan(long long D)
{
    TeamPlan p{0, 1, kShortThreads, 8};
    if (D <= 128) {
        while ((8LL << p.team_log2) < D) ++p.team_log2;
        p.threads = 1 << p.team_log2;
        return p;
    }
    if (D > 256 * 8) p.values = 16;
    p.team_log2 = 5;
    p.threads = p.block = (int)((D + p.values - 1) / p.values + 31) / 32 * 32;
    return p;
}

// Blocks of the backward pass: about as many as are resident together (each keeps its column sums over all its rows).  Measured
// with 1 to 12 to an SM: 15616 x 1024 tokens 103 us with 4 (118 with 8), 15616 x 4680 signatures 169 us with 2 (284 with 3, where no
// ring of two stages fits), 262144 x 128 heads 81 us with 2 (91 with 4).
int backward_blocks(const PsigNormDesc &d)
{
    if (d.D > kNormWidest) return (int)(d.rows < 148 * 2 ? d.rows : 148 * 2);
    const TeamPlan p = team_plan(d.D);
    const long long need = (d.rows + p.teams() - 1) / p.teams(), per_sm = p.team_log2 == 5 && p.block <= 128 ? 4 : p.team_log2 == 5 && p.block <= 256 ? 3 : 2;
    return (int)(need < 148 * per_sm ? need : 148 * per_sm);
}

// Shared memory of a block's ring, with `per_sm` blocks on an SM: as many stages (2 to 4) as fit; none when rows are no whole
// 16-byte pieces, or too short for a block of their own.
template <typename T>
int plan_ring(const NormArgs &a, const TeamPlan &p, bool backward, bool next, int per_sm, Ring *ring)
{
    *ring = Ring{};
    const void *operands[] = {a.x, a.gate, backward && !next ? nullptr : a.residual, backward ? a.grad_h : nullptr,
                              backward && next ? a.grad_n : nullptr};
    for (const void *o : operands) {
        if (o == nullptr) continue;
        if (reinterpret_cast<uintptr_t>(o) % 16 != 0) return 0;
        ring->data[ring->count++] = o;
    }
    const long long bytes = a.D * (long long)sizeof(T);
    if (p.team_log2 < 5 || bytes % 16 != 0 || sizeof(T) == 8) return 0;
    ring->row_bytes = (int)bytes;
    ring->polls = g_row_polls.load(std::memory_order_relaxed);
    const long long room = 220 * 1024 / per_sm - 1024 - 128, stage = bytes * ring->count;
    ring->stages = (int)(room / stage < 4 ? room / stage : 4);
    return ring->stages < 2 ? 0 : 128 + (int)(stage * ring->stages);
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

// Calls fn with the values per access, or with them and the accesses per thread, as compile-time numbers.
template <typename T, typename Fn>
int with_width(int width, Fn fn)
{
    constexpr int full = sizeof(T) == 8 ? 1 : 16 / (int)sizeof(T);
    if (width >= full) return fn(std::integral_constant<int, full>{});
    if constexpr (full == 8)
        if (width >= 2) return fn(std::integral_constant<int, 2>{});
    return fn(std::integral_constant<int, 1>{});
}
template <typename T, typename Fn>
int with_shape(int width, int values, Fn fn)
{
    return with_width<T>(width, [&](auto e) {
        constexpr int E = decltype(e)::value;
        if (values == 8) return fn(e, std::integral_constant<int, 8 / E>{});
        return fn(e, std::integral_constant<int, 16 / E>{});
    });
}

}  // namespace

long long norm_timeouts()
{
    unsigned long long count = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&count, g_norm_timeouts, sizeof(count)) != cudaSuccess) return -1;
    if (count != 0) cudaMemcpyToSymbol(g_norm_timeouts, &zero, sizeof(zero));
    return (long long)count;
}

}  // namespace psig

using namespace psig;

extern "C" int psig_set_norm_wait_polls(int polls)
{
    g_row_polls.store(polls < 0 ? kWaitPolls : (unsigned)polls, std::memory_order_relaxed);
    return PSIG_OK;
}

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
    set_sizes(a, *desc);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        if (a.D > kNormWidest) {
            const unsigned grid = (unsigned)(a.rows < 148 * 4 ? a.rows : 148 * 4);
            return with_width<T>(access_width<T>(a), [&](auto e) {
                norm_forward_wide<T, decltype(e)::value><<<grid, kWideThreads, 0, s>>>(a);
                return check_launch();
            });
        }
        const TeamPlan p = team_plan(a.D);
        const long long blocks = (a.rows + p.teams() - 1) / p.teams();
        const unsigned grid = (unsigned)(blocks < 148 * 32 ? blocks : 148 * 32);
        // Wide rows: a ring of rows and 3 blocks to an SM (15616 x 4680 signatures 115 us, 143 with 2).  Shorter ones are faster without,
        // on many small blocks (15616 x 1024 tokens 43 us, with a ring 47 to 54).
        const int per_sm = 3;
        Ring ring;
        const int smem = p.block > 256 && a.rows >= 148LL * per_sm * 4 ? plan_ring<T>(a, p, false, a.next_weight != nullptr, per_sm, &ring) : 0;
        return with_shape<T>(access_width<T>(a), p.values, [&](auto e, auto nv) {
            constexpr int E = decltype(e)::value, NV = decltype(nv)::value;
            auto launch = [&](auto kernel, unsigned grid, int bytes) {
                if (!prepare_kernel(kernel, bytes, false)) return (int)PSIG_ERR_CUDA;
                kernel<<<grid, p.block, bytes, s>>>(a, p.team_log2, p.threads, ring);
                return check_launch();
            };
            if constexpr (E * sizeof(T) == 16)
                if (smem > 0)
                    return a.next_weight ? launch(norm_forward_team<T, E, NV, true, true>, 148 * per_sm, smem)
                                         : launch(norm_forward_team<T, E, NV, false, true>, 148 * per_sm, smem);
            return a.next_weight ? launch(norm_forward_team<T, E, NV, true, false>, grid, 0)
                                 : launch(norm_forward_team<T, E, NV, false, false>, grid, 0);
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
    set_sizes(a, *desc);
    const int blocks = backward_blocks(*desc);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        using A = typename Acc<T>::type;
        int status;
        if (a.D > kNormWidest) {
            status = with_width<T>(access_width<T>(a), [&](auto e) {
                norm_backward_wide<T, decltype(e)::value><<<blocks, kWideThreads, 0, s>>>(a);
                return check_launch();
            });
        } else {
            const TeamPlan p = team_plan(a.D);
            Ring ring;
            const int per_sm = (blocks + 147) / 148;
            const int smem = a.rows >= blocks * 4LL ? plan_ring<T>(a, p, true, a.next_weight != nullptr, per_sm, &ring) : 0;
            status = with_shape<T>(access_width<T>(a), p.values, [&](auto e, auto nv) {
                constexpr int E = decltype(e)::value, NV = decltype(nv)::value;
                auto launch = [&](auto kernel, int bytes) {
                    if (!prepare_kernel(kernel, bytes, false)) return (int)PSIG_ERR_CUDA;
                    kernel<<<blocks, p.block, bytes, s>>>(a, p.team_log2, p.threads, ring);
                    return check_launch();
                };
                if constexpr (E * sizeof(T) == 16)
                    if (smem > 0)
                        return a.next_weight ? launch(norm_backward_team<T, E, NV, true, true>, smem)
                                             : launch(norm_backward_team<T, E, NV, false, true>, smem);
                const int fold = p.teams() > 1 ? (int)sizeof(A) * E * NV * p.block : 0;
                return a.next_weight ? launch(norm_backward_team<T, E, NV, true, false>, fold)
                                     : launch(norm_backward_team<T, E, NV, false, false>, fold);
            });
        }
        if (status != PSIG_OK || (!grad_weight && !grad_residual_scale && !grad_next_weight)) return status;
        norm_sum_partials<A><<<dim3((unsigned)((a.D + 31) / 32), 3), a.D >= 32 * 128 ? 256 : 1024, 0, s>>>(
            static_cast<const A *>(workspace), blocks, a.D, static_cast<A *>(grad_weight),
            static_cast<A *>(grad_residual_scale), static_cast<A *>(grad_next_weight));
        return check_launch();
    });
}
