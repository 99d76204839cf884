// Decayed linear attention on the tensor cores (bfloat16 / float16 operands): one sweep over pieces of 128 time steps.
//
// With the decays summed inside a piece, a_t (towards the end of the sweep), r_t, k_s, v_s the rows of the sweep
// (sequence.cuh) and S the state (d1, 64 columns) at the piece's beginning,
//     out_t = out_scale ( sum_{s to t} exp(a_t - a_s) (r_t . k_s) kv_scale v_s + exp(a_t) r_t^T S )
//     S    <- exp(a_end) S + sum_s k_s ( exp(a_end - a_s) kv_scale v_s )^T
// that is four matrix products a piece: scores = R K^T, O2 = R S, I = K^T V', O1 = P V with P the weighted scores.
// All run as tcgen05.mma with M = 128 and fp32 accumulators in tensor memory; R, K, V come by TMA into 128-byte
// swizzled tiles, in which K and V serve both as they are and transposed (the descriptor's major bit).
//
// Rounding.  The products take 16-bit operands, exact for R, K and V.  P, S and V' are computed in 32 bits and
// enter as a sum of NP, NS and NV 16-bit terms (the value, what its rounding left, what that left): one term where
// only a 16-bit output depends on it, three (24 bits) where a 32-bit result does: the state itself, and the decay
// gradient.  The state lives in registers in 32 bits and is never rounded but for its copy as an operand.  Sums of
// decays are in 64 bits, so that a weight exp(a_t - a_s) does not lose the difference of two long sums.
//
// Warps: 8 compute (thread = time step or state row, two warps share 32 rows and split the columns), one that
// issues TMA and MMA from a single thread, one that sums the next piece's decays.  They meet at mbarriers; every
// wait is bounded (see attn_tile_timeouts).
#include "sequence.cuh"

#include <cuda.h>

namespace psig {
namespace {

constexpr int kPiece = 128;
constexpr int kCompute = 256;                 // compute threads
constexpr int kTileThreads = kCompute + 64;   // + issuing warp + decay warp
constexpr int kTileBytes = kPiece * 128;      // 128 rows of 64 16-bit values
constexpr unsigned kWaitPolls = 1u << 22;     // each poll blocks for a hardware-defined time at most

__device__ unsigned long long g_tile_timeouts;

struct DecayTables {       // of one piece; all exponents are of 2
    double a[kPiece];      // a_t
    float la[kPiece];      // a_s - (a at the low end of s's block of 32)
    float cf[kPiece];      // 2^-la
    float tail[kPiece];    // 2^(a_end - a_s)
    float head[kPiece];    // 2^a_t
    float keep;            // 2^a_end, what is left of the state
    float pad[3];
};

enum Barrier { kFullRK, kFullV0, kFullV1, kVReady, kScores, kInc, kP, kO1, kEpi, kFix, kDecFull0, kDecFull1, kDecFree0, kDecFree1, kBarriers };

template <int KP, int NP, int NS, int NV, int VS>
struct TileLayout {
    static constexpr int panels = KP / 64;
    static constexpr int r = 0;
    static constexpr int k = r + panels * kTileBytes;
    static constexpr int v = k + panels * kTileBytes;
    static constexpr int vw = v + VS * kTileBytes;          // V' terms
    static constexpr int s = vw + NV * kTileBytes;          // state terms, KP rows of 128 bytes
    static constexpr int decay = s + NS * KP * 128;
    static constexpr int bars = decay + 2 * (int)sizeof(DecayTables);
    static constexpr int tmem = bars + kBarriers * 8;
    static constexpr int bytes = tmem + 16;
    static constexpr int alloc = bytes + 1024;              // the tiles start on a 1024-byte boundary
    // tensor memory columns: scores (P's first term takes the columns its own thread has read), the further terms
    // of P, O2, I and O1
    static constexpr int c_p = 128;
    static constexpr int c_o2 = 128 + (NP - 1) * 64;
    static constexpr int c_o1 = c_o2 + 64;
    static constexpr int columns = c_o1 + 64 <= 256 ? 256 : 512;
};

__device__ __forceinline__ uint32_t shared_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Waits for the phase of this parity; false when the bound ran out here or in another thread of the block.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *failed)
{
    for (unsigned i = 0; i < kWaitPolls; ++i) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if (*failed) return false;
    }
    if (atomicExch(const_cast<int *>(failed), 1) == 0) atomicAdd(&g_tile_timeouts, 1ull);
    return false;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int head, int t, int b)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(head), "r"(t), "r"(b) : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle.  Rows of 128 bytes, eight rows (1024 bytes) to a swizzle
// atom; `lead` is the distance of neighbouring 64-element blocks where the row runs along M or N.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t lead)
{
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t instr_desc(int n, bool a_rows_along_m, bool b_rows_along_n)
{
    const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | ((a_rows_along_m ? 1u : 0u) << 15) | ((b_rows_along_n ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&x)[16])
{
    uint32_t *r = reinterpret_cast<uint32_t *>(x);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                   "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp_two(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two values as 16-bit pair (low half first), and back.
__device__ __forceinline__ uint32_t pack(float x, float y, __nv_bfloat16) { __nv_bfloat162 p = __floats2bfloat162_rn(x, y); return *reinterpret_cast<uint32_t *>(&p); }
__device__ __forceinline__ uint32_t pack(float x, float y, __half) { __half2 p = __floats2half2_rn(x, y); return *reinterpret_cast<uint32_t *>(&p); }
__device__ __forceinline__ float2 unpack(uint32_t v, __nv_bfloat16) { return float2{__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)}; }
__device__ __forceinline__ float2 unpack(uint32_t v, __half) { return __half22float2(*reinterpret_cast<__half2 *>(&v)); }

// The next 16-bit term of a pair; leaves what the rounding left.
template <typename T>
__device__ __forceinline__ uint32_t next_term(float &x, float &y, bool last)
{
    const uint32_t p = pack(x, y, T{});
    if (!last) {
        const float2 back = unpack(p, T{});
        x -= back.x;
        y -= back.y;
    }
    return p;
}

__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

template <typename T, int KP, int NP, int NS, int NV, int VS, bool REV, int MINB>
__global__ void __launch_bounds__(kTileThreads, MINB)
attn_sweep_tiles(const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const Sweep a)
{
    using Lay = TileLayout<KP, NP, NS, NV, VS>;
    constexpr int SC = KP == 128 ? 32 : 16;   // state columns per thread (with 64 rows, lanes 64.. hold them once more)
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024 - (shared_addr(smem_raw) & 1023)) & 1023);
    const uint32_t base = shared_addr(smem);
    DecayTables *tables = reinterpret_cast<DecayTables *>(smem + Lay::decay);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Lay::tmem);
    volatile int *failed = reinterpret_cast<volatile int *>(smem + Lay::tmem + 4);
    auto bar = [&](int i) { return base + Lay::bars + 8 * i; };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tiles = (a.d2 + 63) / 64;
    const int vt = blockIdx.x % tiles;
    const long long bh = blockIdx.x / tiles, b = bh / a.H;
    const int h = (int)(bh % a.H);
    long long n = a.L;
    if (a.lengths != nullptr) {
        n = a.lengths[b];
        n = n < 0 ? 0 : n > a.L ? a.L : n;
    }
    const int pieces = (int)((n + kPiece - 1) / kPiece);
    const long long segments = (a.L + kSegment - 1) / kSegment;

    if (tid == 0) {
        bar_init(bar(kFullRK), 1);
        bar_init(bar(kFullV0), 1);
        bar_init(bar(kFullV1), 1);
        bar_init(bar(kVReady), kCompute);
        bar_init(bar(kScores), 1);
        bar_init(bar(kInc), 1);
        bar_init(bar(kP), kCompute);
        bar_init(bar(kO1), 1);
        bar_init(bar(kEpi), kCompute);
        bar_init(bar(kFix), kCompute);
        bar_init(bar(kDecFull0), 1);
        bar_init(bar(kDecFull1), 1);
        bar_init(bar(kDecFree0), kCompute);
        bar_init(bar(kDecFree1), kCompute);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(tmem_slot)), "n"(Lay::columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }

    // the state: thread (row, columns c0 .. c0 + SC)
    const int quarter = warp & 3, half = (warp >> 2) & 1;
    const int srow = KP == 128 ? quarter * 32 + lane : (quarter & 1) * 32 + lane;
    const int sc0 = KP == 128 ? half * 32 : (quarter >> 1) * 32 + half * 16;
    float S[SC];
    const long long state0 = bh * a.d1 * a.d2;
    const int gcol0 = vt * 64 + sc0;   // column in the whole state
    if (warp < 8) {
#pragma unroll
        for (int j = 0; j < SC; ++j) {
            S[j] = 0.f;
            if (a.init != nullptr && srow < a.d1 && gcol0 + j < a.d2)
                S[j] = static_cast<const float *>(a.init)[state0 + (a.init_transposed ? (long long)(gcol0 + j) * a.d1 + srow
                                                                                      : (long long)srow * a.d2 + gcol0 + j)];
        }
    }
    auto store_state_terms = [&]() {   // S as the B operand of R S: rows = state rows, 64 columns to a row
#pragma unroll
        for (int c = 0; c < SC / 8; ++c) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = S[c * 8 + j];
#pragma unroll
            for (int term = 0; term < NS; ++term) {
                uint4 w;
                w.x = next_term<T>(x[0], x[1], term == NS - 1);
                w.y = next_term<T>(x[2], x[3], term == NS - 1);
                w.z = next_term<T>(x[4], x[5], term == NS - 1);
                w.w = next_term<T>(x[6], x[7], term == NS - 1);
                *reinterpret_cast<uint4 *>(smem + Lay::s + term * KP * 128 + swizzled(srow, sc0 / 8 + c)) = w;
            }
        }
    };
    if (warp < 8) {
        store_state_terms();
        fence_async();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 8) {
        // ------------------------------------------------------------------ TMA and MMA, one thread
        if (lane == 0 && pieces > 0) {
            const int rh = h / a.r.share, kh = h / a.k.share, vh = h / a.v.share;
            auto load_rk = [&](int piece) {
                const int t0 = (REV ? pieces - 1 - piece : piece) * kPiece;
                bar_expect(bar(kFullRK), 2 * Lay::panels * kTileBytes);
#pragma unroll
                for (int p = 0; p < Lay::panels; ++p) {
                    tma_load(base + Lay::r + p * kTileBytes, &map_r, bar(kFullRK), p * 64, rh, t0, (int)b);
                    tma_load(base + Lay::k + p * kTileBytes, &map_k, bar(kFullRK), p * 64, kh, t0, (int)b);
                }
            };
            auto load_v = [&](int piece) {
                const int t0 = (REV ? pieces - 1 - piece : piece) * kPiece;
                const uint32_t full = bar(kFullV0 + piece % VS);
                bar_expect(full, kTileBytes);
                tma_load(base + Lay::v + (piece % VS) * kTileBytes, &map_v, full, vt * 64, vh, t0, (int)b);
            };
            load_rk(0);
            load_v(0);
            if (VS == 2 && pieces > 1) load_v(1);
            int loaded_rk = 1, done_rk = 0;
            for (int i = 0; i < pieces; ++i) {
                const uint32_t ph = i & 1;
                const long long t0 = (long long)(REV ? pieces - 1 - i : i) * kPiece;
                if (!bar_wait(bar(kFullRK), ph, failed)) break;
                ++done_rk;
                if (a.lengths != nullptr && n - t0 < kPiece && !bar_wait(bar(kFix), 0, failed)) break;
                if (i > 0 && !bar_wait(bar(kO1), ph ^ 1, failed)) break;   // P of the piece before has been used
                fence_after();
                // scores = R K^T
#pragma unroll
                for (int j = 0; j < KP / 16; ++j) {
                    const uint32_t off = (j / 4) * kTileBytes + (j % 4) * 32;
                    mma_ss(tmem, tile_desc(base + Lay::r + off, 16), tile_desc(base + Lay::k + off, 16), instr_desc<T>(128, false, false), j > 0);
                }
                mma_commit(bar(kScores));
                if (i > 0 && !bar_wait(bar(kEpi), ph ^ 1, failed)) break;
                fence_after();
                // O2 = R S
#pragma unroll
                for (int term = 0; term < NS; ++term)
#pragma unroll
                    for (int j = 0; j < KP / 16; ++j)
                        mma_ss(tmem + Lay::c_o2, tile_desc(base + Lay::r + (j / 4) * kTileBytes + (j % 4) * 32, 16),
                               tile_desc(base + Lay::s + term * KP * 128 + j * 2048, kTileBytes), instr_desc<T>(64, false, true),
                               term > 0 || j > 0);
                if (!bar_wait(bar(kVReady), ph, failed)) break;
                fence_after();
                // I = K^T V'; with 64 state rows the second block of 64 is the first once more
#pragma unroll
                for (int term = 0; term < NV; ++term)
#pragma unroll
                    for (int j = 0; j < kPiece / 16; ++j)
                        mma_ss(tmem + Lay::c_o1, tile_desc(base + Lay::k + j * 2048, KP == 128 ? kTileBytes : 0),
                               tile_desc(base + Lay::vw + term * kTileBytes + j * 2048, kTileBytes), instr_desc<T>(64, true, true),
                               term > 0 || j > 0);
                mma_commit(bar(kInc));
                if (!bar_wait(bar(kInc), ph, failed)) break;
                if (i + 1 < pieces) {
                    load_rk(i + 1);
                    ++loaded_rk;
                }
                if (VS == 2 && i > 0 && i + 1 < pieces) load_v(i + 1);   // the buffer of piece i - 1, whose O1 has been read
                if (!bar_wait(bar(kP), ph, failed)) break;
                fence_after();
                // O1 = P V
#pragma unroll
                for (int term = 0; term < NP; ++term)
#pragma unroll
                    for (int j = 0; j < kPiece / 16; ++j) {
                        const int col = term == 0 ? (j / 4) * 64 + (j % 4) * 8 : Lay::c_p + (term - 1) * 64 + j * 8;
                        mma_ts(tmem + Lay::c_o1, tmem + col, tile_desc(base + Lay::v + (i % VS) * kTileBytes + j * 2048, kTileBytes),
                               instr_desc<T>(64, false, true), term > 0 || j > 0);
                    }
                mma_commit(bar(kO1));
                if (VS == 1 && i + 1 < pieces) {
                    if (!bar_wait(bar(kO1), ph, failed)) break;
                    load_v(i + 1);
                }
            }
            if (*failed) {
                // let what is in flight land before the block gives its memory back
                int none = 0;
                if (loaded_rk > done_rk) bar_wait(bar(kFullRK), (loaded_rk - 1) & 1, &none);
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        // ------------------------------------------------------------------ decays of each piece
        const float *g = static_cast<const float *>(a.decay) + b * a.decay_stride[0] + h * a.decay_stride[2];
        for (int i = 0; i < pieces; ++i) {
            const long long t0 = (long long)(REV ? pieces - 1 - i : i) * kPiece;
            const int m = (int)(n - t0 < kPiece ? n - t0 : kPiece);
            double c[4];
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = lane * 4 + j;
                float x = t < m ? g[(t0 + t) * a.decay_stride[1]] : 0.f;
                x = x < -100.f ? -100.f : x;   // exp(-100) is 0 in 32 bits already; keeps sums finite, lets a NaN through
                sum += (double)x * 1.4426950408889634;
                c[j] = sum;
            }
            double before = sum;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, before, s);
                if (lane >= s) before += up;
            }
            const double end = __shfl_sync(0xffffffffu, before, 31);
            before -= sum;
#pragma unroll
            for (int j = 0; j < 4; ++j) c[j] = REV ? end - (before + c[j]) : before + c[j];
            // the low end of each block of 32 steps: its last step, or, in reverse, its first
            const double low = __shfl_sync(0xffffffffu, REV ? c[0] : c[3], REV ? (lane & ~7) : (lane | 7));
            bool ok = i < 2 || bar_wait(bar(kDecFree0 + (i & 1)), ((i >> 1) & 1) ^ 1, failed);
            if (!__all_sync(0xffffffffu, ok)) break;
            DecayTables &d = tables[i & 1];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = lane * 4 + j;
                const float la = (float)(c[j] - low);
                d.a[t] = c[j];
                d.la[t] = la;
                d.cf[t] = exp2f(-la);
                d.tail[t] = exp2f((float)(end - c[j]));
                d.head[t] = exp2f((float)c[j]);
            }
            if (lane == 0) d.keep = exp2f((float)end);
            __syncwarp();
            if (lane == 0) bar_arrive(bar(kDecFull0 + (i & 1)));
        }
    } else {
        // ------------------------------------------------------------------ compute
        const int row = quarter * 32 + lane;                    // time step in the piece
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const float *anchors = static_cast<const float *>(a.anchors);
        T *out_t = static_cast<T *>(a.out);
        float *out_f = static_cast<float *>(a.out);
        const T *dot_row = static_cast<const T *>(a.dot.data);
        if (dot_row != nullptr) dot_row += b * a.dot.stride[0] + (h / a.dot.share) * a.dot.stride[2];
        const int ocol0 = vt * 64 + half * 32;                  // output columns of this thread
        for (int i = 0; i < pieces; ++i) {
            const uint32_t ph = i & 1;
            const long long t0 = (long long)(REV ? pieces - 1 - i : i) * kPiece;
            const int m = (int)(n - t0 < kPiece ? n - t0 : kPiece);
            const long long end = t0 + m;
            const bool boundary = end == n || end % kSegment == 0;
            if (REV && a.anchor_dots != nullptr && boundary) {
                // the state behind this piece against the stored state of the steps up to here
                const long long segment = (end - 1) / kSegment;
                const float *s0 = anchors + (bh * segments + segment) * a.d1 * a.d2;
                float dot = 0.f;
                if (srow < a.d1)
#pragma unroll
                    for (int j = 0; j < SC; ++j)
                        if (gcol0 + j < a.d2) dot += S[j] * s0[(long long)srow * a.d2 + gcol0 + j];
                for (int s = 16; s >= 1; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
                if (lane == 0) static_cast<float *>(a.anchor_dots)[((bh * segments + segment) * tiles + vt) * 8 + warp] = dot;
            }
            const DecayTables &d = tables[i & 1];
            bool ok = bar_wait(bar(kDecFull0 + (i & 1)), (i >> 1) & 1, failed);
            ok = ok && bar_wait(bar(kFullV0 + i % VS), (i / VS) & 1, failed);
            const bool fix = a.lengths != nullptr && m < kPiece;
            if (fix) ok = ok && bar_wait(bar(kFullRK), ph, failed);
            if (!__all_sync(0xffffffffu, ok)) break;
            unsigned char *v_tile = smem + Lay::v + (i % VS) * kTileBytes;
            if (fix && row >= m) {
                // rows behind the sequence's last step: whatever stands there must not reach a product
                const uint4 zero = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4 *>(v_tile + swizzled(row, half * 4 + c)) = zero;
#pragma unroll
                for (int p = 0; p < Lay::panels; ++p)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        *reinterpret_cast<uint4 *>(smem + Lay::k + p * kTileBytes + swizzled(row, half * 4 + c)) = zero;
            }
            if (fix) {
                fence_async();
                bar_arrive(bar(kFix));
            }
            {   // V' = tail weights times V
                const float w = d.tail[row];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t at = swizzled(row, half * 4 + c);
                    const uint4 p = *reinterpret_cast<const uint4 *>(v_tile + at);
                    float2 x[4] = {unpack(p.x, T{}), unpack(p.y, T{}), unpack(p.z, T{}), unpack(p.w, T{})};
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j].x *= w, x[j].y *= w;
#pragma unroll
                    for (int term = 0; term < NV; ++term) {
                        uint4 o;
                        o.x = next_term<T>(x[0].x, x[0].y, term == NV - 1);
                        o.y = next_term<T>(x[1].x, x[1].y, term == NV - 1);
                        o.z = next_term<T>(x[2].x, x[2].y, term == NV - 1);
                        o.w = next_term<T>(x[3].x, x[3].y, term == NV - 1);
                        *reinterpret_cast<uint4 *>(smem + Lay::vw + term * kTileBytes + at) = o;
                    }
                }
            }
            fence_async();
            bar_arrive(bar(kVReady));
            // P = scores, weighted
            ok = bar_wait(bar(kScores), ph, failed);
            if (!__all_sync(0xffffffffu, ok)) break;
            fence_after();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int s0 = half * 64 + q * 16;              // first column; 16 at a time
                const int block = half * 2 + q / 2;
                const uint32_t own = tmem + lanes + half * 64;  // this thread's columns of the scores
                uint32_t p0[16], p1[16], p2[16];
                float x[16];
                const bool beyond = REV ? block < quarter : block > quarter;
                if (!beyond) {
                    tmem_load16(own + q * 16, x);
                    tmem_loaded();
                    if (block == quarter) {
                        const float la = d.la[row];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int s = s0 + j;
                            const bool in = REV ? s >= row : s <= row;
                            x[j] = in ? x[j] * exp_two(la - d.la[s]) : 0.f;
                        }
                    } else {
                        const float f = exp_two((float)(d.a[row] - d.a[REV ? block * 32 : block * 32 + 31]));
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] *= f * d.cf[s0 + j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p0[j] = next_term<T>(x[2 * j], x[2 * j + 1], NP == 1);
                    if (NP > 1) p1[j] = next_term<T>(x[2 * j], x[2 * j + 1], NP == 2);
                    if (NP > 2) p2[j] = next_term<T>(x[2 * j], x[2 * j + 1], NP == 3);
                }
                auto store8 = [&](uint32_t addr, const uint32_t (&r)[16]) {
                    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
                };
                store8(own + q * 8, p0);
                if (NP > 1) store8(tmem + lanes + Lay::c_p + half * 32 + q * 8, p1);
                if (NP > 2) store8(tmem + lanes + Lay::c_p + 64 + half * 32 + q * 8, p2);
            }
            tmem_stored();
            // the state behind the piece, and its operand for the next one
            ok = bar_wait(bar(kInc), ph, failed);
            if (!__all_sync(0xffffffffu, ok)) break;
            fence_after();
            {
                const float keep = d.keep, kv_scale = (float)a.kv_scale;
#pragma unroll
                for (int c = 0; c < SC / 16; ++c) {
                    float x[16];
                    tmem_load16(tmem + lanes + Lay::c_o1 + sc0 + c * 16, x);
                    tmem_loaded();
#pragma unroll
                    for (int j = 0; j < 16; ++j) S[c * 16 + j] = fmaf(S[c * 16 + j], keep, x[j] * kv_scale);
                }
            }
            if (i + 1 < pieces) store_state_terms();
            fence_async();
            fence_before();
            bar_arrive(bar(kP));
            if (!REV && anchors != nullptr && boundary && srow < a.d1) {
                float *s0 = static_cast<float *>(a.anchors) + (bh * segments + (end - 1) / kSegment) * a.d1 * a.d2;
#pragma unroll
                for (int j = 0; j < SC; ++j)
                    if (gcol0 + j < a.d2) s0[(long long)srow * a.d2 + gcol0 + j] = S[j];
            }
            // out
            const float head = d.head[row];
            ok = bar_wait(bar(kO1), ph, failed);
            if (!__all_sync(0xffffffffu, ok)) break;
            fence_after();
            const long long t = t0 + row;
            float dot = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x[16], y[16];
                tmem_load16(tmem + lanes + Lay::c_o1 + half * 32 + c * 16, x);
                tmem_load16(tmem + lanes + Lay::c_o2 + half * 32 + c * 16, y);
                tmem_loaded();
                const float f1 = (float)(a.out_scale * a.kv_scale), f2 = (float)a.out_scale * head;
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = row < m ? fmaf(x[j], f1, y[j] * f2) : 0.f;
                if (t >= a.L) continue;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int col = ocol0 + c * 16 + e * 8;
                    if (col >= a.d2) continue;
                    const long long at = ((b * a.L + t) * a.H + h) * a.d2 + col;
                    if (a.out_acc) {
                        *reinterpret_cast<float4 *>(out_f + at) = make_float4(x[e * 8], x[e * 8 + 1], x[e * 8 + 2], x[e * 8 + 3]);
                        *reinterpret_cast<float4 *>(out_f + at + 4) = make_float4(x[e * 8 + 4], x[e * 8 + 5], x[e * 8 + 6], x[e * 8 + 7]);
                    } else {
                        uint4 o;
                        o.x = pack(x[e * 8], x[e * 8 + 1], T{});
                        o.y = pack(x[e * 8 + 2], x[e * 8 + 3], T{});
                        o.z = pack(x[e * 8 + 4], x[e * 8 + 5], T{});
                        o.w = pack(x[e * 8 + 6], x[e * 8 + 7], T{});
                        *reinterpret_cast<uint4 *>(out_t + at) = o;
                    }
                    if (dot_row != nullptr && row < m) {
                        const uint4 p = *reinterpret_cast<const uint4 *>(dot_row + t * a.dot.stride[1] + col);
                        const float2 w[4] = {unpack(p.x, T{}), unpack(p.y, T{}), unpack(p.z, T{}), unpack(p.w, T{})};
#pragma unroll
                        for (int j = 0; j < 4; ++j) dot += x[e * 8 + 2 * j] * w[j].x + x[e * 8 + 2 * j + 1] * w[j].y;
                    }
                }
            }
            fence_before();
            bar_arrive(bar(kEpi));
            bar_arrive(bar(kDecFree0 + (i & 1)));
            if (dot_row != nullptr && t < a.L) a.dots[((long long)(vt * 2 + half) * a.B * a.L + b * a.L + t) * a.H + h] = dot;
        }
        // rows behind the last piece, and the last state
        const long long first = (long long)pieces * kPiece;
        for (long long e = tid; e < (a.L - first) * 8; e += kCompute) {
            const long long t = first + e / 8;
            const int col = vt * 64 + (int)(e % 8) * 8;
            if (col >= a.d2) continue;
            const long long at = ((b * a.L + t) * a.H + h) * a.d2 + col;
            const uint4 zero = {0, 0, 0, 0};
            *reinterpret_cast<uint4 *>(a.out_acc ? (void *)(out_f + at) : (void *)(out_t + at)) = zero;
            if (a.out_acc) *reinterpret_cast<uint4 *>(out_f + at + 4) = zero;
        }
        if (dot_row != nullptr)
            for (long long e = tid; e < (a.L - first) * 2; e += kCompute)
                a.dots[((vt * 2 + e % 2) * a.B * a.L + b * a.L + first + e / 2) * a.H + h] = 0.f;
        if (a.final != nullptr && srow < a.d1)
#pragma unroll
            for (int j = 0; j < SC; ++j)
                if (gcol0 + j < a.d2)
                    static_cast<float *>(a.final)[state0 + (a.final_transposed ? (long long)(gcol0 + j) * a.d1 + srow
                                                                               : (long long)srow * a.d2 + gcol0 + j)] = S[j];
    }
    fence_before();
    __syncthreads();
    if (warp == 8) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Lay::columns));
    }
}

// ------------------------------------------------------------------------------------------ host side

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder()
{
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &st) != cudaSuccess ||
            st != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// (d, heads, L, B) of 16-bit values; a box is 64 values of one head at 128 time steps.
bool encode(CUtensorMap *map, const SweepOperand &o, const Sweep &a, int d, int dtype)
{
    const long long heads = a.H / o.share;
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)a.L, (cuuint64_t)a.B};
    // the stride of a dimension of one element is never used, but has to be a valid one
    auto bytes = [&](long long stride, long long size) { return (cuuint64_t)(size > 1 ? stride * 2 : (d * 2 + 15) / 16 * 16); };
    const cuuint64_t strides[3] = {bytes(o.stride[2], heads), bytes(o.stride[1], a.L), bytes(o.stride[0], a.B)};
    const cuuint32_t box[4] = {64, 1, kPiece, 1}, unit[4] = {1, 1, 1, 1};
    auto call = [&] {
        return encoder()(map, dtype == PSIG_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void *>(o.data), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    if (call() == CUDA_SUCCESS) return true;
    // a thread that has made no runtime call yet (autograd's) has no current context, which the driver call wants
    int device = 0;
    return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && call() == CUDA_SUCCESS;
}

template <typename T, int KP, int NP, int NS, int NV, int VS, bool REV, int MINB>
int launch_tiles(const Sweep &a, int dtype, cudaStream_t stream)
{
    using Lay = TileLayout<KP, NP, NS, NV, VS>;
    CUtensorMap r, k, v;
    if (encoder() == nullptr || !encode(&r, a.r, a, a.d1, dtype) || !encode(&k, a.k, a, a.d1, dtype) ||
        !encode(&v, a.v, a, a.d2, dtype))
        return PSIG_ERR_CUDA;
    auto kernel = attn_sweep_tiles<T, KP, NP, NS, NV, VS, REV, MINB>;
    if (!prepare_kernel(kernel, Lay::alloc, true)) return PSIG_ERR_CUDA;
    const long long blocks = a.B * a.H * ((a.d2 + 63) / 64);
    kernel<<<(unsigned)blocks, kTileThreads, Lay::alloc, stream>>>(r, k, v, a);
    return check_launch();
}

template <typename T, bool REV>
int select_tiles(const Sweep &a, bool exact, int dtype, cudaStream_t stream)
{
    if (exact)
        return a.d1 <= 64 ? launch_tiles<T, 64, 3, 3, 3, 2, REV, 1>(a, dtype, stream)
                          : launch_tiles<T, 128, 3, 3, 3, 2, REV, 1>(a, dtype, stream);
    return a.d1 <= 64 ? launch_tiles<T, 64, 1, 1, 3, 1, REV, 1>(a, dtype, stream)
                      : launch_tiles<T, 128, 1, 1, 3, 2, REV, 1>(a, dtype, stream);
}

bool operand_fits(const SweepOperand &o, const Sweep &a, int d)
{
    if (d % 8 != 0 || (reinterpret_cast<uintptr_t>(o.data) & 15) != 0) return false;
    const long long sizes[3] = {a.B, a.L, a.H / o.share};
    for (int i = 0; i < 3; ++i)
        if (sizes[i] > 1 && (o.stride[i] <= 0 || o.stride[i] % 8 != 0 || o.stride[i] >= (1LL << 38))) return false;
    return true;
}

}  // namespace

bool attn_tiles_supported(const Sweep &a, int dtype)
{
    return dtype == PSIG_BF16 && a.d1 <= 128 && a.d2 <= 128 && a.L < (1LL << 31) && a.B < (1LL << 31) &&
           a.B * a.H < (1LL << 30) && operand_fits(a.r, a, a.d1) && operand_fits(a.k, a, a.d1) && operand_fits(a.v, a, a.d2);
}

int attn_sweep_on_tiles(const Sweep &a, bool exact, int dtype, cudaStream_t stream)
{
    return a.reverse ? select_tiles<__nv_bfloat16, true>(a, exact, dtype, stream)
                     : select_tiles<__nv_bfloat16, false>(a, exact, dtype, stream);
}

long long attn_tile_timeouts()
{
    unsigned long long count = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&count, g_tile_timeouts, sizeof(count)) != cudaSuccess) return -1;
    if (count != 0) cudaMemcpyToSymbol(g_tile_timeouts, &zero, sizeof(zero));
    return (long long)count;
}

}  // namespace psig
