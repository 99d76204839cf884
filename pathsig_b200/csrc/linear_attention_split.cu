// Decayed linear attention on the tensor cores for float16 and float32 operands.
//
// The sweep of linear_attention_tiles.cu (same products, same tables), with every operand as a sum of bfloat16 terms:
// two hold a float16 value exactly (11 bits, and its whole range), three a float32 value (24 bits).  A product runs over the
// pairs of terms that matter, all into one fp32 accumulator: pairs (i, j) with i + j <= LEVEL, LEVEL 1 (16 bits: what a
// float16 result needs) or 2 (24 bits).  So float32 calls keep float32's precision at six bfloat16 products instead
// of fused multiply-adds, which have a thirtieth of the rate; and float16 scores, weights and states cannot overflow.
//
// TMA brings the raw rows; the compute threads turn them into terms in place (the raw tile of a float16 operand is as
// large as its first term, that of a float32 operand as its first two), clearing rows behind the sequence's end on
// the way.  Rows of more than 64 values are taken in two halves, one after the other through the same buffers: the
// scores add up, and each half of the state is its own product.
#include "tiles.cuh"

namespace psig {
namespace {

enum Barrier { kRaw, kRawV, kReady, kScores, kInc, kP, kO1, kEpi, kDecFull0, kDecFull1, kDecFree0, kDecFree1, kSwap, kBarriers };

using bf16 = __nv_bfloat16;

constexpr int kCompute = 256;                 // compute threads
constexpr int kTileThreads = kCompute + 64;   // + issuing warp + decay warp

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
    static constexpr int c_p = 128;                          // further terms of P
    static constexpr int c_o2 = 128 + (NP - 1) * 64;
    static constexpr int c_i = c_o2 + 64;                    // one I per half; O1 takes the first's columns
    static constexpr int columns = c_i + PANELS * 64 <= 256 ? 256 : 512;
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

template <typename T, int PANELS, int LEVEL, bool REV>
__global__ void __launch_bounds__(kTileThreads, 1)
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
    const int pieces = (int)((n + kPiece - 1) / kPiece);
    const long long segments = (a.L + kSegment - 1) / kSegment;

    if (tid == 0) {
        bar_init(bar(kRaw), 1);
        bar_init(bar(kRawV), 1);
        bar_init(bar(kReady), kCompute / 32);
        bar_init(bar(kScores), 1);
        bar_init(bar(kInc), 1);
        bar_init(bar(kP), kCompute / 32);
        bar_init(bar(kO1), 1);
        bar_init(bar(kEpi), kCompute / 32);
        bar_init(bar(kDecFull0), 1);
        bar_init(bar(kDecFull1), 1);
        bar_init(bar(kDecFree0), kCompute / 32);
        bar_init(bar(kDecFree1), kCompute / 32);
        bar_init(bar(kSwap), kCompute / 32);
        *failed = 0;
        failed[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(tmem_slot)), "n"(Lay::columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 8) {
        // ------------------------------------------------------------------ TMA and MMA, one thread
        if (pieces > 0) {
            const uint32_t lead = lane == 0, base16 = base >> 4;
            const int rh = h / a.r.share, kh = h / a.k.share, vh = h / a.v.share;
            const int halves = pieces * PANELS;
            auto start = [&](int piece) { return (REV ? pieces - 1 - piece : piece) * kPiece; };
            constexpr int per_box = 128 / (int)sizeof(T);
            auto load_rk = [&](int idx) {
                if (!lead) return;
                const int t0 = start(idx / PANELS), x0 = idx % PANELS * 64;
                bar_expect(bar(kRaw), 2 * RAW_BOXES * kTileBytes);
#pragma unroll
                for (int p = 0; p < RAW_BOXES; ++p) {
                    tma_load(base + Lay::r + p * kTileBytes, &map_r, bar(kRaw), x0 + p * per_box, rh, t0, (int)b);
                    tma_load(base + Lay::k + p * kTileBytes, &map_k, bar(kRaw), x0 + p * per_box, kh, t0, (int)b);
                }
            };
            auto load_v = [&](int piece) {
                if (!lead) return;
                bar_expect(bar(kRawV), RAW_BOXES * kTileBytes);
#pragma unroll
                for (int p = 0; p < RAW_BOXES; ++p)
                    tma_load(base + Lay::v + p * kTileBytes, &map_v, bar(kRawV), vt * 64 + p * per_box, vh, start(piece), (int)b);
            };
            load_rk(0);
            load_v(0);
            int loaded = 1, loaded_v = 1;
            bool ok = true;
            for (int i = 0; i < pieces && ok; ++i) {
                const uint32_t ph = i & 1;
                for (int p = 0; p < PANELS && ok; ++p) {
                    const int idx = i * PANELS + p;
                    ok = warp_wait(bar(kReady), idx & 1, failed);
                    if (ok && p == 0 && i > 0) ok = warp_wait(bar(kO1), ph ^ 1, failed) && warp_wait(bar(kEpi), ph ^ 1, failed);
                    if (!ok) break;
                    fence_after();
                    bool add = p > 0;
#pragma unroll 1
                    for (int pair = 0; pair < pair_count(NI, NI, LEVEL); ++pair)
                        if (const int x = (int)(pair_list(NI, NI, LEVEL) >> (4 * pair)) & 3, y = (int)(pair_list(NI, NI, LEVEL) >> (4 * pair + 2)) & 3; true)
#pragma unroll
                            for (int j = 0; j < 4; ++j, add = true)
                                mma_ss(tmem, tile_desc(base16 + ((Lay::r + x * kTileBytes + j * 32) >> 4), 16),
                                       tile_desc(base16 + ((Lay::k + y * kTileBytes + j * 32) >> 4), 16), instr_desc<bf16>(128, false, false), add, lead);
                    if (p == PANELS - 1) mma_commit(bar(kScores), lead);
                    add = p > 0;
#pragma unroll 1
                    for (int pair = 0; pair < pair_count(NI, Lay::NS, LEVEL); ++pair)
                        if (const int x = (int)(pair_list(NI, Lay::NS, LEVEL) >> (4 * pair)) & 3, y = (int)(pair_list(NI, Lay::NS, LEVEL) >> (4 * pair + 2)) & 3; true)
#pragma unroll
                            for (int j = 0; j < 4; ++j, add = true)
                                mma_ss(tmem + Lay::c_o2, tile_desc(base16 + ((Lay::r + x * kTileBytes + j * 32) >> 4), 16),
                                       tile_desc(base16 + ((Lay::s + y * 8192 + j * 2048) >> 4), kTileBytes), instr_desc<bf16>(64, false, true), add, lead);
                    add = false;
                    // the state's 64 rows twice (the distance of the second block is 0), so that all lanes hold some
#pragma unroll 1
                    for (int pair = 0; pair < pair_count(NI, Lay::NV, 2); ++pair)
                        if (const int x = (int)(pair_list(NI, Lay::NV, 2) >> (4 * pair)) & 3, y = (int)(pair_list(NI, Lay::NV, 2) >> (4 * pair + 2)) & 3; true)
#pragma unroll
                            for (int j = 0; j < kPiece / 16; ++j, add = true)
                                mma_ss(tmem + Lay::c_i + p * 64, tile_desc(base16 + ((Lay::k + x * kTileBytes + j * 2048) >> 4), 0),
                                       tile_desc(base16 + ((Lay::vw + y * kTileBytes + j * 2048) >> 4), kTileBytes), instr_desc<bf16>(64, true, true), add, lead);
                    mma_commit(bar(kInc), lead);
                    ok = warp_wait(bar(kInc), idx & 1, failed);
                    if (ok && idx + 1 < halves) {
                        load_rk(idx + 1);
                        ++loaded;
                    }
                }
                ok = ok && warp_wait(bar(kP), ph, failed);
                if (!ok) break;
                fence_after();
                bool add = false;
#pragma unroll 1
                for (int pair = 0; pair < pair_count(Lay::NP, NI, LEVEL); ++pair)
                    if (const int x = (int)(pair_list(Lay::NP, NI, LEVEL) >> (4 * pair)) & 3, y = (int)(pair_list(Lay::NP, NI, LEVEL) >> (4 * pair + 2)) & 3; true)
#pragma unroll
                        for (int j = 0; j < kPiece / 16; ++j, add = true) {
                            const int col = x == 0 ? (j / 4) * 64 + (j % 4) * 8 : Lay::c_p + (x - 1) * 64 + j * 8;
                            mma_ts(tmem + Lay::c_i, tmem + col, tile_desc(base16 + ((Lay::v + y * kTileBytes + j * 2048) >> 4), kTileBytes),
                                   instr_desc<bf16>(64, false, true), add, lead);
                        }
                mma_commit(bar(kO1), lead);
                if (i + 1 < pieces) {
                    ok = warp_wait(bar(kO1), ph, failed);
                    if (!ok) break;
                    load_v(i + 1);
                    ++loaded_v;
                }
            }
            if (*failed) {
                // let what is in flight land before the block gives its memory back
                warp_wait(bar(kRaw), (loaded - 1) & 1, failed + 1);
                warp_wait(bar(kRawV), (loaded_v - 1) & 1, failed + 1);
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        const float *g = static_cast<const float *>(a.decay) + b * a.decay_stride[0] + h * a.decay_stride[2];
        sum_decays<REV>(g, a.decay_stride[1], n, pieces, tables, bar(kDecFull0), bar(kDecFree0), failed);
    } else {
        // ------------------------------------------------------------------ compute
        const int quarter = warp & 3, half = warp >> 2;
        const int row = quarter * 32 + lane;                       // time step in the piece
        const int srow = (quarter & 1) * 32 + lane;                // row of a half of the state
        const int sc0 = (quarter >> 1) * 32 + half * 16;           // first of 16 columns of the state
        const int gcol0 = vt * 64 + sc0;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const long long state0 = bh * a.d1 * a.d2;
        float S[PANELS][16];
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int r1 = p * 64 + srow;
                S[p][j] = 0.f;
                if (a.init != nullptr && r1 < a.d1 && gcol0 + j < a.d2)
                    S[p][j] = static_cast<const float *>(a.init)[state0 + (a.init_transposed ? (long long)(gcol0 + j) * a.d1 + r1
                                                                                             : (long long)r1 * a.d2 + gcol0 + j)];
            }
        auto all_state = [&](auto fn) {   // fn(value, position in a (d1, d2) state, transposed position)
#pragma unroll
            for (int p = 0; p < PANELS; ++p)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int r1 = p * 64 + srow;
                    if (r1 < a.d1 && gcol0 + j < a.d2) fn(S[p][j], (long long)r1 * a.d2 + gcol0 + j, (long long)(gcol0 + j) * a.d1 + r1);
                }
        };
        T *out_t = static_cast<T *>(a.out);
        float *out_f = static_cast<float *>(a.out);
        const T *dot_row = static_cast<const T *>(a.dot.data);
        if (dot_row != nullptr) dot_row += b * a.dot.stride[0] + (h / a.dot.share) * a.dot.stride[2];
        const int ocol0 = vt * 64 + half * 32;
        constexpr int G = 16 / (int)sizeof(T);   // values of an access of an output row
        const float kv_scale = (float)a.kv_scale;
        uint32_t swaps = 0;
        // float32: the terms of a row's one half overwrite the raw values of its other half, which another thread holds
        auto swap = [&]() {
            if constexpr (sizeof(T) != 4) return true;
            warp_arrive(bar(kSwap));
            return warp_wait(bar(kSwap), swaps++ & 1, failed);
        };
        bool ok = true;
        for (int i = 0; i < pieces; ++i) {
            const uint32_t ph = i & 1;
            const long long t0 = (long long)(REV ? pieces - 1 - i : i) * kPiece;
            const int m = (int)(n - t0 < kPiece ? n - t0 : kPiece);
            const long long end = t0 + m;
            const bool boundary = end == n || end % kSegment == 0;
            if (REV && a.anchor_dots != nullptr && boundary) {
                const long long segment = (end - 1) / kSegment;
                const float *anchor = static_cast<const float *>(a.anchors) + ((bh * segments + segment) * tiles + vt) * PANELS * 4096 + tid;
                float dot = 0.f;
#pragma unroll
                for (int p = 0; p < PANELS; ++p)
#pragma unroll
                    for (int j = 0; j < 16; ++j) dot = fmaf(S[p][j], anchor[(p * 16 + j) * kCompute], dot);
                for (int s = 16; s >= 1; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
                if (lane == 0) static_cast<float *>(a.anchor_dots)[((bh * segments + segment) * tiles + vt) * 8 + warp] = dot;
            }
            const DecayTables &d = tables[i & 1];
            ok = warp_wait(bar(kDecFull0 + (i & 1)), (i >> 1) & 1, failed);
#pragma unroll
            for (int p = 0; p < PANELS; ++p) {
                const int idx = i * PANELS + p;
                ok = ok && warp_wait(bar(kRaw), idx & 1, failed);   // all products of the half before are done, too
                if (p == 0) ok = ok && warp_wait(bar(kRawV), ph, failed);
                if (!ok) break;
                {   // the state's half as an operand
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float x[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = S[p][c * 8 + j];
#pragma unroll
                        for (int term = 0; term < Lay::NS; ++term) {
                            uint4 w;
                            w.x = next_term<bf16>(x[0], x[1], term == Lay::NS - 1);
                            w.y = next_term<bf16>(x[2], x[3], term == Lay::NS - 1);
                            w.z = next_term<bf16>(x[4], x[5], term == Lay::NS - 1);
                            w.w = next_term<bf16>(x[6], x[7], term == Lay::NS - 1);
                            *reinterpret_cast<uint4 *>(smem + Lay::s + term * 8192 + swizzled(srow, sc0 / 8 + c)) = w;
                        }
                    }
                }
                // R, K and, with the first half, V and V'.  One loop for all: the code has to stay in the instruction cache
#pragma unroll 1
                for (int tile = 0; tile < (p == 0 ? 3 : 2); ++tile) {
                    unsigned char *at = smem + tile * NI * kTileBytes;   // R, K, V stand one behind the other
                    float x[32];
                    read_raw<T>(at, row, half, row < m, x);
                    ok = swap();
                    if (!ok) break;
                    if (tile == 2) {
                        float y[32];
                        const float w = d.tail[row];
#pragma unroll
                        for (int j = 0; j < 32; ++j) y[j] = x[j] * w;
                        write_terms<Lay::NV>(smem + Lay::vw, kTileBytes, row, half * 4, y);
                    }
                    write_terms<NI>(at, kTileBytes, row, half * 4, x);
                }
                if (!ok) break;
                fence_async();
                warp_arrive(bar(kReady));
            }
            if (!ok) break;
            // P = scores, weighted
            ok = warp_wait(bar(kScores), ph, failed);
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int s0 = half * 64 + q * 16;
                const int block = half * 2 + q / 2;
                const uint32_t own = tmem + lanes + half * 64;
                uint32_t p0[8], p1[8], p2[8];
                float x[16];
                if (REV ? block >= quarter : block <= quarter) {
                    tmem_load16(own + q * 16, x);
                    tmem_loaded();
                    if (block == quarter) {
                        const float la = d.la[row];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int s = s0 + j;
                            x[j] = (REV ? s >= row : s <= row) ? x[j] * exp_two(la - d.la[s]) : 0.f;
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
                    p0[j] = next_term<bf16>(x[2 * j], x[2 * j + 1], false);
                    p1[j] = next_term<bf16>(x[2 * j], x[2 * j + 1], Lay::NP == 2);
                    if (Lay::NP > 2) p2[j] = next_term<bf16>(x[2 * j], x[2 * j + 1], true);
                }
                tmem_store8(own + q * 8, p0);
                tmem_store8(tmem + lanes + Lay::c_p + half * 32 + q * 8, p1);
                if (Lay::NP > 2) tmem_store8(tmem + lanes + Lay::c_p + 64 + half * 32 + q * 8, p2);
            }
            tmem_stored();
            // the state behind the piece
            ok = warp_wait(bar(kInc), (i * PANELS + PANELS - 1) & 1, failed);
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int p = 0; p < PANELS; ++p) {
                float x[16];
                tmem_load16(tmem + lanes + Lay::c_i + p * 64 + sc0, x);
                tmem_loaded();
#pragma unroll
                for (int j = 0; j < 16; ++j) S[p][j] = fmaf(S[p][j], d.keep, x[j] * kv_scale);
            }
            fence_before();
            warp_arrive(bar(kP));
            if (!REV && a.anchors != nullptr && boundary) {
                // in the threads' own order: the sweep that reads them has the same threads
                float *anchor = static_cast<float *>(a.anchors) + ((bh * segments + (end - 1) / kSegment) * tiles + vt) * PANELS * 4096 + tid;
#pragma unroll
                for (int p = 0; p < PANELS; ++p)
#pragma unroll
                    for (int j = 0; j < 16; ++j) anchor[(p * 16 + j) * kCompute] = S[p][j];
            }
            // out
            const float head = d.head[row];
            ok = warp_wait(bar(kO1), ph, failed);
            if (!ok) break;
            fence_after();
            const long long t = t0 + row;
            float dot = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x[16], y[16];
                tmem_load16(tmem + lanes + Lay::c_i + half * 32 + c * 16, x);
                tmem_load16(tmem + lanes + Lay::c_o2 + half * 32 + c * 16, y);
                tmem_loaded();
                const float f1 = (float)(a.out_scale * a.kv_scale), f2 = (float)a.out_scale * head;
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = row < m ? fmaf(x[j], f1, y[j] * f2) : 0.f;
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
            warp_arrive(bar(kDecFree0 + (i & 1)));
            if (dot_row != nullptr && t < a.L) a.dots[((long long)(vt * 2 + half) * a.B * a.L + b * a.L + t) * a.H + h] = dot;
        }
        // rows behind the last piece, and the last state
        const long long first = (long long)pieces * kPiece;
        for (long long e = tid; e < (a.L - first) * 16; e += kCompute) {
            const long long t = first + e / 16;
            const int col = vt * 64 + (int)(e % 16) * 4;
            if (col >= a.d2) continue;
            const long long at = ((b * a.L + t) * a.H + h) * a.d2 + col;
            if (sizeof(T) == 4 || a.out_acc) *reinterpret_cast<float4 *>(out_f + at) = make_float4(0.f, 0.f, 0.f, 0.f);
            else *reinterpret_cast<uint2 *>(out_t + at) = make_uint2(0u, 0u);
        }
        if (dot_row != nullptr)
            for (long long e = tid; e < (a.L - first) * 2; e += kCompute)
                a.dots[((vt * 2 + e % 2) * a.B * a.L + b * a.L + first + e / 2) * a.H + h] = 0.f;
        if (a.final != nullptr)
            all_state([&](float v, long long at, long long transposed) {
                static_cast<float *>(a.final)[state0 + (a.final_transposed ? transposed : at)] = v;
            });
    }
    fence_before();
    __syncthreads();
    if (warp == 8) {
        fence_after();
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
    auto kernel = attn_sweep_split_terms<T, PANELS, LEVEL, REV>;
    if (!prepare_kernel(kernel, Lay::alloc, true)) return PSIG_ERR_CUDA;
    const long long blocks = a.B * a.H * ((a.d2 + 63) / 64);
    kernel<<<(unsigned)blocks, kTileThreads, Lay::alloc, stream>>>(r, k, v, a);
    return check_launch();
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
