// Decayed linear attention on the tensor cores for float16 and float32 operands.
//
// The sweep of linear_attention_tiles.cu (same products, same tables), with every operand as a sum of bfloat16 terms:
// two hold a float16 value exactly (11 bits, and its whole range), three a float32 value (24 bits).  A product runs over the
// pairs of terms that matter, all into one fp32 accumulator: pairs (i, j) with i + j <= LEVEL, LEVEL 1 (16 bits: what a
// float16 result needs) or 2 (24 bits).  So float32 calls keep float32's precision at six bfloat16 products instead
// of fused multiply-adds, which have a thirtieth of the rate; and float16 scores, weights and states cannot overflow.
//
// Where the second operand's terms stand one behind the other in shared memory, the terms that belong with one term of the
// first are one product: P_x [V_0 V_1 ..], with the columns for x + y = 0, 1, 2 side by side in tensor memory (added up on
// the way out), reads P_x once.  A product of 64 columns is bound by reading its operands from shared memory.
//
// TMA brings the raw rows; eight warps turn them into terms in place (the raw tile of a float16 operand is as large as its
// first term, that of a float32 operand as its first two), clearing rows behind the sequence's end on the way, and hold
// the state; eight more weigh the scores and write the output, so that one piece's conversion overlaps with the piece
// before.  Rows of more than 64 values are taken in two halves, one after the other through the same buffers: the scores
// add up, and each half of the state is its own product.
//
// Measured, 8 x 2047 steps of 8 heads of 64 in float32: 20000 cycles a piece when eight warps did all stages (4200
// conversion, 11000 products, 3400 output) and each pair of terms was its own product; 15000 in this form (132 us in one part,
// 31 + 74 us in two; the bytes alone: 20 us).  Bound by the products: six of bfloat16 for one of float32.
#include "tiles.cuh"

namespace psig {
namespace {

enum Barrier { kRaw, kRawV, kReady, kReadyV, kScores, kInc, kIncRead, kP, kO1, kEpi, kDecFull0, kDecFull1, kDecFree0, kDecFree1, kSwap, kFinish, kBarriers };

using bf16 = __nv_bfloat16;

constexpr int kStateThreads = 256, kOutThreads = 256;
constexpr int kSplitThreads = kStateThreads + kOutThreads + 96;   // + products, copies, decays

template <int NI, int PANELS, int LEVEL>
struct SplitLayout {
    static constexpr int NP = LEVEL + 1, NS = LEVEL + 1, NV = 3;
    static constexpr int r = 0;
    static constexpr int k = r + NI * kTileBytes;
    static constexpr int v = k + NI * kTileBytes;
    static constexpr int vw = v + NI * kTileBytes;          // V' terms
    static constexpr int s = vw + NV * kTileBytes;          // state terms of one half, 64 rows of 128 bytes
    static constexpr int decay = s + NS * 64 * 128;
    static constexpr int bars = decay + 2 * (int)sizeof(DecayTables);
    static constexpr int tmem = bars + kBarriers * 8;
    static constexpr int alloc = tmem + 16;
    // tensor memory columns: scores (P's first term takes the columns its own thread has read), the further terms of P,
    // O2, and I, whose place O1 takes: both by the order x + y of their terms
    static constexpr int c_p = 128;
    static constexpr int c_o2 = 256;
    static constexpr int c_i = 320;
    static constexpr int orders = 3;
    static constexpr int columns = 512;
};

// The pairs (x, y) of nx by ny terms with x + y <= level, the smallest products (largest x + y) first: the accumulator drops
// what does not fit its 24 bits at every step, towards zero, so the steps that come while it is still small cost nothing
// (error of float32 outputs over a 128-step piece: 1.7e-7, with the large products first 1.8e-6).  As numbers of
// four bits, x in the lower two.
__host__ __device__ constexpr int pair_count(int nx, int ny, int level)
{
    int n = 0;
    for (int x = 0; x < nx; ++x)
        for (int y = 0; y < ny; ++y) n += x + y <= level;
    return n;
}
__host__ __device__ constexpr unsigned long long pair_list(int nx, int ny, int level)
{
    unsigned long long list = 0;
    int n = 0;
    for (int sum = level; sum >= 0; --sum)
        for (int x = 0; x < nx; ++x)
            if (sum - x >= 0 && sum - x < ny) list |= (unsigned long long)(x | (sum - x) << 2) << (4 * n++);
    return list;
}

// 32 neighbouring values of a row of a raw tile (columns 32 half .. ), and their terms into the tiles.
template <typename T>
__device__ __forceinline__ void read_raw(const unsigned char *tile, int row, int half, bool live, float (&x)[32])
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float4 p = *reinterpret_cast<const float4 *>(tile + half * kTileBytes + swizzled(row, c));
            x[4 * c] = p.x, x[4 * c + 1] = p.y, x[4 * c + 2] = p.z, x[4 * c + 3] = p.w;
        }
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint4 p = *reinterpret_cast<const uint4 *>(tile + swizzled(row, half * 4 + c));
            const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 two = unpack(w[j], T{});
                x[8 * c + 2 * j] = two.x, x[8 * c + 2 * j + 1] = two.y;
            }
        }
    }
    if (!live)
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = 0.f;
}
template <int TERMS>
__device__ __forceinline__ void write_terms(unsigned char *tile, int stride, int row, int chunk0, float (&x)[32])
{
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int term = 0; term < TERMS; ++term) {
            uint4 o;
            o.x = next_term<bf16>(x[8 * c], x[8 * c + 1], term == TERMS - 1);
            o.y = next_term<bf16>(x[8 * c + 2], x[8 * c + 3], term == TERMS - 1);
            o.z = next_term<bf16>(x[8 * c + 4], x[8 * c + 5], term == TERMS - 1);
            o.w = next_term<bf16>(x[8 * c + 6], x[8 * c + 7], term == TERMS - 1);
            *reinterpret_cast<uint4 *>(tile + term * stride + swizzled(row, chunk0 + c)) = o;
        }
}

template <typename T, int PANELS, int LEVEL, bool REV, bool STATE>
__global__ void __launch_bounds__(kSplitThreads, 1)
attn_sweep_split_terms(const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const Sweep a)
{
    constexpr int NI = sizeof(T) == 4 ? 3 : 2;
    using Lay = SplitLayout<NI, PANELS, LEVEL>;
    constexpr int RAW_BOXES = sizeof(T) == 4 ? 2 : 1;   // boxes of 128 bytes to a half row of 64 values
    extern __shared__ __align__(1024) unsigned char smem[];   // the swizzle atoms start on 1024-byte boundaries
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
    const int all = (int)((n + kPiece - 1) / kPiece);                 // pieces of the sequence
    const int part = blockIdx.y;
    const int first = (int)((long long)all * part / a.splits), pieces = (int)((long long)all * (part + 1) / a.splits) - first;
    const long long segments = (a.L + kSegment - 1) / kSegment;
    auto piece_start = [&](int i) { return (long long)(REV ? all - 1 - first - i : first + i) * kPiece; };

    if (tid == 0) {
        const int warps_state = kStateThreads / 32, warps_out = kOutThreads / 32;
        bar_init(bar(kRaw), 1);
        bar_init(bar(kRawV), 1);
        bar_init(bar(kReady), warps_state);
        bar_init(bar(kReadyV), warps_state);
        bar_init(bar(kScores), 1);
        bar_init(bar(kInc), 1);
        bar_init(bar(kIncRead), warps_state);
        bar_init(bar(kP), warps_out);
        bar_init(bar(kO1), 1);
        bar_init(bar(kEpi), warps_out);
        bar_init(bar(kSwap), warps_state);
        bar_init(bar(kFinish), 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(bar(kDecFull0 + i), 1);
            bar_init(bar(kDecFree0 + i), warps_state + (STATE ? 0 : warps_out));
        }
        failed[0] = failed[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(tmem_slot)), "n"(Lay::columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    constexpr uint32_t tmem = 0;   // all columns are ours, so they start at 0
    if (tid == 0 && (*tmem_slot != 0 || (base & 1023) != 0)) *failed = 1, atomicAdd(&g_tile_timeouts, 1ull);
    const int quarter = warp & 3, half = (warp >> 2) & 1;
    const int row = quarter * 32 + lane;                       // time step in the piece
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;

    if (warp < 8) {
        // ------------------------------------------------------------------ terms of R, K, V and V'; the state
        const int srow = (quarter & 1) * 32 + lane;                // row of a half of the state (they stand twice in the 128 lanes)
        const int sc0 = (quarter >> 1) * 32 + half * 16;           // first of 16 columns of the state
        const int gcol0 = vt * 64 + sc0;
        const long long state0 = bh * a.d1 * a.d2;
        float S[PANELS][16];
        auto all_state = [&](bool transposed, auto fn) {   // fn(value, its position), (d1, d2) or (d2, d1)
            const int step = transposed ? a.d1 : 1;
#pragma unroll
            for (int p = 0; p < PANELS; ++p) {
                const int r1 = p * 64 + srow;
                long long at = state0 + (transposed ? (long long)gcol0 * a.d1 + r1 : (long long)r1 * a.d2 + gcol0);
#pragma unroll
                for (int j = 0; j < 16; ++j, at += step)
                    if (r1 < a.d1 && gcol0 + j < a.d2) fn(S[p][j], at);
            }
        };
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
            for (int j = 0; j < 16; ++j) S[p][j] = 0.f;
        float *parts = a.split_states + ((bh * a.splits + part) * tiles + vt) * PANELS * 4096 + tid;   // this part's, in the threads' order
        if (part > 0 && !STATE) {
            parts -= (long long)tiles * PANELS * 4096;
#pragma unroll
            for (int p = 0; p < PANELS; ++p)
#pragma unroll
                for (int j = 0; j < 16; ++j) S[p][j] = parts[(p * 16 + j) * kStateThreads];
        } else if (part == 0 && a.init != nullptr)
            all_state(a.init_transposed, [&](float &v, long long at) { v = static_cast<const float *>(a.init)[at]; });
        const float kv_scale = (float)a.kv_scale;
        uint32_t swaps = 0;
        // float32: the terms of a row's one half overwrite the raw values of its other half, which another thread holds
        auto swap = [&]() {
            if constexpr (sizeof(T) != 4) return true;
            warp_arrive(bar(kSwap));
            return warp_wait(bar(kSwap), swaps++ & 1, failed);
        };
        auto convert = [&](int at, int m) {
            float x[32];
            read_raw<T>(smem + at, row, half, row < m, x);
            if (!swap()) return false;
            write_terms<NI>(smem + at, kTileBytes, row, half * 4, x);
            return true;
        };
        bool ok = true;
#pragma unroll 1
        for (int i = 0; i < pieces && ok; ++i) {
            const long long t0 = piece_start(i);
            const int m = (int)(n - t0 < kPiece ? n - t0 : kPiece);
            const long long end = t0 + m;
            const bool boundary = end == n || end % kSegment == 0;
            if (REV && !STATE && a.anchor_dots != nullptr && boundary) {
                const long long segment = (end - 1) / kSegment;
                const float *anchor = static_cast<const float *>(a.anchors) + ((bh * segments + segment) * tiles + vt) * PANELS * 4096 + tid;
                float dot = 0.f;
#pragma unroll
                for (int p = 0; p < PANELS; ++p)
#pragma unroll
                    for (int j = 0; j < 16; ++j) dot = fmaf(S[p][j], anchor[(p * 16 + j) * kStateThreads], dot);
                for (int s = 16; s >= 1; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
                if (lane == 0) static_cast<float *>(a.anchor_dots)[((bh * segments + segment) * tiles + vt) * 8 + warp] = dot;
            }
            const DecayTables &d = tables[i & 1];
            ok = warp_wait(bar(kDecFull0 + (i & 1)), (i >> 1) & 1, failed);
            if (!ok) break;
            const float keep = d.keep, w = d.tail[row];
            warp_arrive(bar(kDecFree0 + (i & 1)));
#pragma unroll
            for (int p = 0; p < PANELS; ++p) {
                const int idx = i * PANELS + p;
                // the products of the half before are done, so its tiles and the state's operand are free
                ok = warp_wait(bar(kRaw), idx & 1, failed);
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < (STATE ? 0 : 2); ++c) {   // the state's half as an operand
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = S[p][c * 8 + j];
#pragma unroll
                    for (int term = 0; term < Lay::NS; ++term) {
                        uint4 o;
                        o.x = next_term<bf16>(x[0], x[1], term == Lay::NS - 1);
                        o.y = next_term<bf16>(x[2], x[3], term == Lay::NS - 1);
                        o.z = next_term<bf16>(x[4], x[5], term == Lay::NS - 1);
                        o.w = next_term<bf16>(x[6], x[7], term == Lay::NS - 1);
                        *reinterpret_cast<uint4 *>(smem + Lay::s + term * 8192 + swizzled(srow, sc0 / 8 + c)) = o;
                    }
                }
#pragma unroll 1
                for (int tile = STATE ? 1 : 0; tile < 2 && ok; ++tile) ok = convert(tile == 0 ? Lay::r : Lay::k, m);
                if (!ok) break;
                fence_async();
                warp_arrive(bar(kReady));
                if (p == 0) {
                    ok = warp_wait(bar(kRawV), i & 1, failed);
                    if (!ok) break;
                    float x[32], y[32];
                    read_raw<T>(smem + Lay::v, row, half, row < m, x);
#pragma unroll
                    for (int j = 0; j < 32; ++j) y[j] = x[j] * w;
                    ok = swap();
                    if (!ok) break;
                    write_terms<Lay::NV>(smem + Lay::vw, kTileBytes, row, half * 4, y);
                    if (!STATE) write_terms<NI>(smem + Lay::v, kTileBytes, row, half * 4, x);
                    fence_async();
                    warp_arrive(bar(kReadyV));
                }
                ok = warp_wait(bar(kInc), idx & 1, failed);
                if (!ok) break;
                fence_after();
                float x[3][16];
#pragma unroll
                for (int o = 0; o < 3; ++o) tmem_load16(tmem + lanes + Lay::c_i + o * 64 + sc0, x[o]);
                tmem_loaded();
                fence_before();
                warp_arrive(bar(kIncRead));
#pragma unroll
                for (int j = 0; j < 16; ++j) S[p][j] = fmaf(S[p][j], keep, (x[0][j] + (x[1][j] + x[2][j])) * kv_scale);
            }
            if (!ok) break;
            if (!REV && !STATE && a.anchors != nullptr && boundary) {
                // in the threads' own order: the sweep that reads them has the same threads
                float *anchor = static_cast<float *>(a.anchors) + ((bh * segments + (end - 1) / kSegment) * tiles + vt) * PANELS * 4096 + tid;
#pragma unroll
                for (int p = 0; p < PANELS; ++p)
#pragma unroll
                    for (int j = 0; j < 16; ++j) anchor[(p * 16 + j) * kStateThreads] = S[p][j];
            }
        }
        if (STATE) {
#pragma unroll
            for (int p = 0; p < PANELS; ++p)
#pragma unroll
                for (int j = 0; j < 16; ++j) parts[(p * 16 + j) * kStateThreads] = S[p][j];
        } else if (a.final != nullptr && part == a.splits - 1)
            all_state(a.final_transposed, [&](float &v, long long at) { static_cast<float *>(a.final)[at] = v; });
    } else if (warp < 16) {
        // ------------------------------------------------------------------ P = scores, weighted; out
        const uint32_t own = tmem + lanes + half * 64;      // this thread's columns of the scores
        T *out_t = static_cast<T *>(a.out);
        float *out_f = static_cast<float *>(a.out);
        const T *dot_row = static_cast<const T *>(a.dot.data);
        if (dot_row != nullptr) dot_row += b * a.dot.stride[0] + (h / a.dot.share) * a.dot.stride[2];
        const int ocol0 = vt * 64 + half * 32;
        constexpr int G = 16 / (int)sizeof(T);              // values of an access of an output row
        const int tid_out = tid - kStateThreads;
#pragma unroll 1
        for (int i = 0; i < (STATE ? 0 : pieces); ++i) {
            const uint32_t ph = i & 1;
            const long long t0 = piece_start(i), t = t0 + row;
            const int m = (int)(n - t0 < kPiece ? n - t0 : kPiece);
            const DecayTables &d = tables[i & 1];
            if (!warp_wait(bar(kDecFull0 + (i & 1)), (i >> 1) & 1, failed)) break;
            const float la = d.la[row], lb = d.lb[row], head = d.head[row];
            float f[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) f[q] = exp_two((float)(d.a[row] - d.a[(half * 2 + q) * 32 + (REV ? 0 : 31)]));
            if (!warp_wait(bar(kScores), ph, failed)) break;
            fence_after();
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {   // 16 columns each
                const int block = half * 2 + q / 2, s0 = half * 64 + q * 16;
                float x[16];
                if (REV ? block >= quarter : block <= quarter) {
                    tmem_load16(own + q * 16, x);
                    const float4 *table = reinterpret_cast<const float4 *>((block == quarter ? d.la : d.cf) + s0);
                    float w[16];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 v = table[j];
                        w[4 * j] = v.x, w[4 * j + 1] = v.y, w[4 * j + 2] = v.z, w[4 * j + 3] = v.w;
                    }
                    if (block == quarter) {
                        const float4 *rest = reinterpret_cast<const float4 *>(d.lb + s0);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {   // a_t - a_s to 24 bits of its own size, not of the two's
                            const float4 v = rest[j];
                            w[4 * j] = (la - w[4 * j]) + (lb - v.x), w[4 * j + 1] = (la - w[4 * j + 1]) + (lb - v.y);
                            w[4 * j + 2] = (la - w[4 * j + 2]) + (lb - v.z), w[4 * j + 3] = (la - w[4 * j + 3]) + (lb - v.w);
                        }
                        const int j0 = row - s0;   // the step's own column
#pragma unroll
                        for (int j = 0; j < 16; ++j) w[j] = (REV ? j >= j0 : j <= j0) ? exp_two(w[j]) : 0.f;
                    } else {
                        const float fq = q < 2 ? f[0] : f[1];
#pragma unroll
                        for (int j = 0; j < 16; ++j) w[j] *= fq;
                    }
                    tmem_loaded();
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] *= w[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = 0.f;
                }
                uint32_t p0[8], p1[8], p2[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p0[j] = next_term<bf16>(x[2 * j], x[2 * j + 1], false);
                    p1[j] = next_term<bf16>(x[2 * j], x[2 * j + 1], Lay::NP == 2);
                    if (Lay::NP > 2) p2[j] = next_term<bf16>(x[2 * j], x[2 * j + 1], true);
                }
                tmem_store8(own + q * 8, p0);
                tmem_store8(tmem + lanes + Lay::c_p + half * 32 + q * 8, p1);
                if (Lay::NP > 2) tmem_store8(tmem + lanes + Lay::c_p + 64 + half * 32 + q * 8, p2);
            }
            tmem_stored();
            fence_before();
            warp_arrive(bar(kP));
            warp_arrive(bar(kDecFree0 + (i & 1)));
            if (!warp_wait(bar(kO1), ph, failed)) break;
            fence_after();
            float dot = 0.f;
            const float f1 = (float)(a.out_scale * a.kv_scale), f2 = (float)a.out_scale * head;
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                float x[16], y[16], z[16], o2[16];
                tmem_load16(tmem + lanes + Lay::c_i + half * 32 + c * 16, x);
                tmem_load16(tmem + lanes + Lay::c_i + 64 + half * 32 + c * 16, y);
                if (LEVEL > 1) tmem_load16(tmem + lanes + Lay::c_i + 128 + half * 32 + c * 16, z);
                tmem_load16(tmem + lanes + Lay::c_o2 + half * 32 + c * 16, o2);
                tmem_loaded();
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = row < m ? fmaf(x[j] + (LEVEL > 1 ? y[j] + z[j] : y[j]), f1, o2[j] * f2) : 0.f;
                if (t >= a.L) continue;
#pragma unroll
                for (int e = 0; e < 16; e += G) {
                    const int col = ocol0 + c * 16 + e;
                    if (col >= a.d2) continue;
                    const long long at = ((b * a.L + t) * a.H + h) * a.d2 + col;
                    if constexpr (sizeof(T) == 4) {
                        *reinterpret_cast<float4 *>(out_f + at) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                    } else if (a.out_acc) {
                        *reinterpret_cast<float4 *>(out_f + at) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                        *reinterpret_cast<float4 *>(out_f + at + 4) = make_float4(x[e + 4], x[e + 5], x[e + 6], x[e + 7]);
                    } else {
                        uint4 o;
                        o.x = pack(x[e], x[e + 1], T{});
                        o.y = pack(x[e + 2], x[e + 3], T{});
                        o.z = pack(x[e + 4], x[e + 5], T{});
                        o.w = pack(x[e + 6], x[e + 7], T{});
                        *reinterpret_cast<uint4 *>(out_t + at) = o;
                    }
                    if (dot_row != nullptr && row < m) {
                        const uint4 p = *reinterpret_cast<const uint4 *>(dot_row + t * a.dot.stride[1] + col);
                        const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if constexpr (sizeof(T) == 4) {
                                dot += x[e + j] * __uint_as_float(w[j]);
                            } else {
                                const float2 two = unpack(w[j], T{});
                                dot += x[e + 2 * j] * two.x + x[e + 2 * j + 1] * two.y;
                            }
                        }
                    }
                }
            }
            fence_before();
            warp_arrive(bar(kEpi));
            if (dot_row != nullptr && t < a.L) a.dots[((long long)(vt * 2 + half) * a.B * a.L + b * a.L + t) * a.H + h] = dot;
        }
        // rows behind the last piece
        const long long end = STATE || part < a.splits - 1 ? a.L : (long long)all * kPiece;
        for (long long e = tid_out; e < (a.L - end) * 16; e += kOutThreads) {
            const long long t = end + e / 16;
            const int col = vt * 64 + (int)(e % 16) * 4;
            if (col >= a.d2) continue;
            const long long at = ((b * a.L + t) * a.H + h) * a.d2 + col;
            if (sizeof(T) == 4 || a.out_acc) *reinterpret_cast<float4 *>(out_f + at) = make_float4(0.f, 0.f, 0.f, 0.f);
            else *reinterpret_cast<uint2 *>(out_t + at) = make_uint2(0u, 0u);
        }
        if (dot_row != nullptr)
            for (long long e = tid_out; e < (a.L - end) * 2; e += kOutThreads)
                a.dots[((vt * 2 + e % 2) * a.B * a.L + b * a.L + end + e / 2) * a.H + h] = 0.f;
    } else if (warp == 16) {
        // ------------------------------------------------------------------ products
        const uint32_t lead = lane == 0, base16 = base >> 4;
        bool ok = true;
#pragma unroll 1
        for (int i = 0; i < pieces && ok; ++i) {
            const uint32_t ph = i & 1;
#pragma unroll 1
            for (int p = 0; p < PANELS; ++p) {
                const int idx = i * PANELS + p;
                ok = warp_wait(bar(kReady), idx & 1, failed);
                if (!STATE && ok && p == 0 && i > 0) ok = warp_wait(bar(kO1), ph ^ 1, failed);   // P of the piece before has been used
                if (!ok) break;
                fence_after();
                // scores += R K^T
#pragma unroll 1
                for (int pair = 0; pair < (STATE ? 0 : pair_count(NI, NI, LEVEL)); ++pair) {
                    const int x = (int)(pair_list(NI, NI, LEVEL) >> (4 * pair)) & 3, y = (int)(pair_list(NI, NI, LEVEL) >> (4 * pair + 2)) & 3;
                    const uint32_t r16 = base16 + ((Lay::r + x * kTileBytes) >> 4), k16 = base16 + ((Lay::k + y * kTileBytes) >> 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_ss(tmem, tile_desc(r16 + j * 2, 16), tile_desc(k16 + j * 2, 16), instr_desc<bf16>(128, false, false),
                               p > 0 || pair > 0 || j > 0, lead);
                }
                if (p == PANELS - 1 && !STATE) mma_commit(bar(kScores), lead);
                if (!STATE && p == 0 && i > 0) ok = warp_wait(bar(kEpi), ph ^ 1, failed);        // O2 and O1 of the piece before have been read
                if (!ok) break;
                fence_after();
                // O2 += R S
#pragma unroll 1
                for (int pair = 0; pair < (STATE ? 0 : pair_count(NI, Lay::NS, LEVEL)); ++pair) {
                    const int x = (int)(pair_list(NI, Lay::NS, LEVEL) >> (4 * pair)) & 3, y = (int)(pair_list(NI, Lay::NS, LEVEL) >> (4 * pair + 2)) & 3;
                    const uint32_t r16 = base16 + ((Lay::r + x * kTileBytes) >> 4), s16 = base16 + ((Lay::s + y * 8192) >> 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_ss(tmem + Lay::c_o2, tile_desc(r16 + j * 2, 16), tile_desc(s16 + j * 128, kTileBytes), instr_desc<bf16>(64, false, true),
                               p > 0 || pair > 0 || j > 0, lead);
                }
                if (p == 0) ok = warp_wait(bar(kReadyV), ph, failed);
                if (STATE ? idx > 0 : p > 0) ok = ok && warp_wait(bar(kIncRead), (idx - 1) & 1, failed);
                if (!ok) break;
                fence_after();
                // I = K^T V', term x of K with the terms 0 .. 2 - x of V'; the state's 64 rows twice (the distance of the second
                // block is 0), so that all lanes hold some
#pragma unroll 1
                for (int j = 0; j < kPiece / 16; ++j) {
                    const uint32_t k16 = base16 + (Lay::k >> 4) + j * 128, w16 = base16 + (Lay::vw >> 4) + j * 128;
                    mma_ss(tmem + Lay::c_i, tile_desc(k16, 0), tile_desc(w16, kTileBytes), instr_desc<bf16>(192, true, true), j > 0, lead);
                    mma_ss(tmem + Lay::c_i + 64, tile_desc(k16 + (kTileBytes >> 4), 0), tile_desc(w16, kTileBytes), instr_desc<bf16>(128, true, true), true, lead);
                    if (NI > 2)
                        mma_ss(tmem + Lay::c_i + 128, tile_desc(k16 + (2 * kTileBytes >> 4), 0), tile_desc(w16, kTileBytes), instr_desc<bf16>(64, true, true), true, lead);
                }
                mma_commit(bar(kInc), lead);
            }
            if (!ok) break;
            if constexpr (STATE) continue;
            ok = warp_wait(bar(kP), ph, failed) && warp_wait(bar(kIncRead), (i * PANELS + PANELS - 1) & 1, failed);
            if (!ok) break;
            fence_after();
            // O1 = P V, term x of P with the terms 0 .. LEVEL - x of V (as many as there are)
#pragma unroll 1
            for (int j = 0; j < kPiece / 16; ++j) {
                const uint32_t v16 = base16 + (Lay::v >> 4) + j * 128, p0 = tmem + (j / 4) * 64 + (j % 4) * 8, p1 = tmem + Lay::c_p + j * 8;
                constexpr int first = LEVEL + 1 < NI ? LEVEL + 1 : NI;
                // orders that term 0 does not reach (float16 at LEVEL 2) start with term 1
                mma_ts(tmem + Lay::c_i, p0, tile_desc(v16, kTileBytes), instr_desc<bf16>(first * 64, false, true), j > 0, lead);
                if constexpr (LEVEL == 2 && NI == 2) {
                    mma_ts(tmem + Lay::c_i + 64, p1, tile_desc(v16, kTileBytes), instr_desc<bf16>(64, false, true), true, lead);
                    mma_ts(tmem + Lay::c_i + 128, p1, tile_desc(v16 + (kTileBytes >> 4), kTileBytes), instr_desc<bf16>(64, false, true), j > 0, lead);
                } else {
                    mma_ts(tmem + Lay::c_i + 64, p1, tile_desc(v16, kTileBytes), instr_desc<bf16>(LEVEL * 64, false, true), true, lead);
                }
                if constexpr (LEVEL == 2)
                    mma_ts(tmem + Lay::c_i + 128, p1 + 64, tile_desc(v16, kTileBytes), instr_desc<bf16>(64, false, true), true, lead);
            }
            mma_commit(bar(kO1), lead);
        }
    } else if (warp == 17) {
        // ------------------------------------------------------------------ copies
        if (pieces > 0) {
            const uint32_t lead = lane == 0;
            const int rh = h / a.r.share, kh = h / a.k.share, vh = h / a.v.share;
            constexpr int per_box = 128 / (int)sizeof(T);
            auto load_rk = [&](int idx) {
                if (!lead) return;
                const int t0 = (int)piece_start(idx / PANELS), x0 = idx % PANELS * 64;
                bar_expect(bar(kRaw), (STATE ? 1 : 2) * RAW_BOXES * kTileBytes);
#pragma unroll
                for (int p = 0; p < RAW_BOXES; ++p) {
                    if (!STATE) tma_load(base + Lay::r + p * kTileBytes, &map_r, bar(kRaw), x0 + p * per_box, rh, t0, (int)b);
                    tma_load(base + Lay::k + p * kTileBytes, &map_k, bar(kRaw), x0 + p * per_box, kh, t0, (int)b);
                }
            };
            auto load_v = [&](int piece) {
                if (!lead) return;
                bar_expect(bar(kRawV), RAW_BOXES * kTileBytes);
#pragma unroll
                for (int p = 0; p < RAW_BOXES; ++p)
                    tma_load(base + Lay::v + p * kTileBytes, &map_v, bar(kRawV), vt * 64 + p * per_box, vh, (int)piece_start(piece), (int)b);
            };
            load_rk(0);
            load_v(0);
            int loaded = 1, loaded_v = 1;
            bool ok = true;
#pragma unroll 1
            for (int idx = 0; idx + 1 < pieces * PANELS && ok; ++idx) {
                ok = warp_wait(bar(kInc), idx & 1, failed);        // the last product that reads this half of R and K
                if (!ok) break;
                load_rk(idx + 1);
                ++loaded;
                const int i = idx / PANELS;
                if (idx % PANELS != PANELS - 1) continue;
                if (!STATE) ok = warp_wait(bar(kO1), i & 1, failed);           // the last product that reads V
                if (!ok) break;
                load_v(i + 1);
                ++loaded_v;
            }
            // let what is in flight land before the block gives its memory back, whoever else fails from here on
            warp_wait(bar(kRaw), (loaded - 1) & 1, failed + 1);
            warp_wait(bar(kRawV), (loaded_v - 1) & 1, failed + 1);
        }
    } else {
        const float *g = static_cast<const float *>(a.decay) + b * a.decay_stride[0] + h * a.decay_stride[2];
        int count = 0;
        const double whole = sum_decays<REV>(g, a.decay_stride[1], n, first, pieces, count, tables, bar(kDecFull0), bar(kDecFree0), failed);
        if (STATE && vt == 0 && lane == 0) a.split_decays[bh * a.splits + part] = (float)whole;
    }
    fence_before();
    __syncthreads();
    if (warp == 16) {
        fence_after();
        if (*failed) {   // products in flight read shared and tensor memory
            if (lane == 0) report_failure(a.failure);
            mma_commit(bar(kFinish), lane == 0);
            warp_wait(bar(kFinish), 0, failed + 1);
        }
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Lay::columns));
    }
}

template <typename T, int PANELS, int LEVEL, bool REV>
int launch_split(const Sweep &a, int dtype, cudaStream_t stream)
{
    using Lay = SplitLayout<sizeof(T) == 4 ? 3 : 2, PANELS, LEVEL>;
    CUtensorMap r, k, v;
    if (encoder() == nullptr || !encode(&r, a.r, a, a.d1, dtype) || !encode(&k, a.k, a, a.d1, dtype) ||
        !encode(&v, a.v, a, a.d2, dtype))
        return PSIG_ERR_CUDA;
    const int tiles = tile_columns(a.d2);
    const unsigned blocks = (unsigned)(a.B * a.H * tiles);
    auto launch = [&](auto kernel, int parts) {
        if (!prepare_kernel(kernel, Lay::alloc, true)) return (int)PSIG_ERR_CUDA;
        kernel<<<dim3(blocks, parts), kSplitThreads, Lay::alloc, stream>>>(r, k, v, a);
        return check_launch();
    };
    if (a.splits > 1) {
        int rc = launch(attn_sweep_split_terms<T, PANELS, LEVEL, REV, true>, a.splits - 1);
        if (rc != PSIG_OK || (rc = chain_states(a, 4096LL * PANELS * tiles, stream)) != PSIG_OK) return rc;
    }
    return launch(attn_sweep_split_terms<T, PANELS, LEVEL, REV, false>, a.splits);
}

template <typename T, int LEVEL>
int select_split(const Sweep &a, int dtype, cudaStream_t stream)
{
    if (a.d1 <= 64)
        return a.reverse ? launch_split<T, 1, LEVEL, true>(a, dtype, stream) : launch_split<T, 1, LEVEL, false>(a, dtype, stream);
    return a.reverse ? launch_split<T, 2, LEVEL, true>(a, dtype, stream) : launch_split<T, 2, LEVEL, false>(a, dtype, stream);
}

}  // namespace

int attn_sweep_split(const Sweep &a, bool exact, int dtype, cudaStream_t stream)
{
    if (dtype == PSIG_F32) return select_split<float, 2>(a, dtype, stream);
    return exact ? select_split<__half, 2>(a, dtype, stream) : select_split<__half, 1>(a, dtype, stream);
}

long long attn_split_timeouts() { return take_timeouts(); }

}  // namespace psig
