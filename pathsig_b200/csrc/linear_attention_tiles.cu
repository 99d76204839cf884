// Decayed linear attention on the tensor cores (bfloat16 operands): one sweep over pieces of 128 time steps.
//
// With the decays summed inside a piece, a_t (towards the end of the sweep), r_t, k_s, v_s the rows of the sweep
// (sequence.cuh) and S the state (d1, 64 columns) at the piece's beginning,
//     out_t = out_scale ( sum_{s to t} exp(a_t - a_s) kv_scale (r_t . k_s) v_s + exp(a_t) r_t^T S )
//     S    <- exp(a_end) S + sum_s k_s ( exp(a_end - a_s) kv_scale v_s )^T
// that is four matrix products a piece: scores = R K^T, O2 = R S, I = K^T V', O1 = P V with P the weighted scores.
// All run as tcgen05.mma with M = 128 and fp32 accumulators in tensor memory; R, K, V come by TMA into 128-byte
// swizzled tiles, in which K and V serve both as they are and transposed (the descriptor's major bit).
//
// Rounding.  The products take 16-bit operands, exact for R, K and V.  P, S and V' are computed in 32 bits and enter as sums of
// 16-bit terms (the value, what its rounding left, what that left): P as two, S as NS and V' as NV, two (15 or 16 bits) where
// only a 16-bit output depends on them, so that its one rounding is all that counts (error of the outputs 1.66e-3 of their size;
// 2.35e-3 with P and S as one term each), three (24 bits) where a 32-bit result does, the state itself or the decay gradient.
// Terms of S and of V' stand side by side in one product where tensor memory has room, so that R and K are read once; the rest of
// them, and P's second term, are products of their own, the small ones first into a common accumulator.  The state lives in
// registers in 32 bits and is never rounded but for its copy as an operand.  Sums of decays are in 64 bits, and an exponent
// a_t - a_s has 24 bits of its own size, so that a weight exp(a_t - a_s) does not lose the difference of two long sums.
//
// DOT: the sweep also gives x_t = out_t . y_t for the rows y of a third operand, to 32 bits (the decay gradient needs
// q . grad_q and k . grad_k).  The part of the piece's own pairs is sum_s exp(a_t - a_s) (r_t . k_s) (y_t . v_s), the
// weighted scores times a second product Y V^T, entry by entry before anything is rounded; the state's part is
// exp(a_t) (r_t^T S) . y_t.  (With the output row itself, P would have to enter as three terms.)
//
// Warps, so that a piece's stages overlap with the neighbouring pieces': 8 hold the state and weigh V (thread = state
// row, and = time step), 8 weigh the scores, 4 write the output, one each issues the products, starts the copies, and sums the next piece's decays.
// A thread reads the 32 lanes of tensor memory that its warp's number allows; two warps share 32 rows and split the
// columns.  They meet at mbarriers; every wait is bounded (psig_sequence_wait_timeouts).
//
// Measured, 8 sequences of 4096 steps of 16 heads of 128 (the bytes alone: 82 us forward), with one term of P and S: 382 us forward
// when the same 8 warps did all stages one after the other (of 7000 cycles a piece: 2150 scores to P, 1400 output, 1000 V', 1100
// issue), 197 us in this form; with two terms 240 us (263 with a product for each term of S and V' and rounded first terms), 372 us
// with DOT.  Tensor pipe 32 % busy: the products of 64 columns are limited by reading their operands from shared memory, and a
// piece's chain of scores, weights and products by latency.  Code size matters: with all loops unrolled the six roles miss the
// instruction cache (63 % hits, 290 us with one term).
#include "tiles.cuh"

namespace psig {
namespace {

constexpr int kStateThreads = 256, kScoreThreads = 256, kOutThreads = 128;
constexpr int kTileThreads = kStateThreads + kScoreThreads + kOutThreads + 96;

// A wait names the parity of a phase, so nobody may be two phases behind: what a place of V waits for (I or O1 of two pieces
// before) is counted by that place.
enum Barrier {
    kFullRK, kFullV0, kFullV1, kVReady, kScores, kInc0, kInc1, kP, kO2, kO1_0, kO1_1, kFix, kOutFull, kOutFree, kDot, kDotFree,
    kDecFull0, kDecFull1, kDecFree0, kDecFree1, kFinish, kBarriers
};

template <int KP, int NS, int NV, bool DOT>
struct TileLayout {
    static constexpr int panels = KP / 64;
    static constexpr int VS = DOT && KP == 128 ? 1 : 2;     // pieces of V in turn (else shared memory is full)
    static constexpr int r = 0;
    static constexpr int k = r + panels * kTileBytes;
    static constexpr int v = k + panels * kTileBytes;
    static constexpr int vw = v + VS * kTileBytes;          // V' terms
    static constexpr int s = vw + NV * kTileBytes;          // state terms, KP rows of 128 bytes
    static constexpr int out = s + NS * KP * 128;           // the output tile on its way out
    static constexpr int dot = out + kTileBytes;            // the third operand's tile
    static constexpr int decay = dot + (DOT ? kTileBytes : 0);
    static constexpr int sums = decay + 2 * (int)sizeof(DecayTables);   // [2 pieces][2 halves][128] sums of pairs
    static constexpr int bars = sums + (DOT ? 4 * kPiece * 4 : 0);
    static constexpr int tmem = bars + kBarriers * 8;
    static constexpr int alloc = tmem + 16;
    // tensor memory columns: scores (P's two terms for 16 steps take the columns that those steps' scores were read from), the
    // second scores, O2 and I with the terms of S and V' side by side as far as there is room, O1
    static constexpr int o2_blocks = NS > 1 ? 2 : 1, i_blocks = DOT ? 1 : NV;   // of 64 columns
    static constexpr int c_two = 128;
    static constexpr int c_o2 = DOT ? 256 : 128;
    static constexpr int c_i = c_o2 + 128;
    static constexpr int c_o1 = c_i + 64 * i_blocks;
    static constexpr int columns = 512;
    static_assert(c_o1 + 64 <= columns, "tensor memory");
};

template <typename T, int KP, int NS, int NV, bool DOT, bool REV, bool STATE>
__global__ void __launch_bounds__(kTileThreads, 1)
attn_sweep_tiles(const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
                 const __grid_constant__ CUtensorMap map_dot, const Sweep a)
{
    using Lay = TileLayout<KP, NS, NV, DOT>;
    constexpr int VS = Lay::VS;
    extern __shared__ __align__(1024) unsigned char smem[];   // the swizzle atoms start on 1024-byte boundaries
    const uint32_t base = shared_addr(smem);
    DecayTables *tables = reinterpret_cast<DecayTables *>(smem + Lay::decay);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Lay::tmem);
    volatile int *failed = reinterpret_cast<volatile int *>(smem + Lay::tmem + 4);
    auto bar = [&](int i) { return base + Lay::bars + 8 * i; };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tiles = (a.d2 + 63) / 64;
    const int part = blockIdx.y, items = (int)(a.B * a.H * tiles);
    const long long segments = (a.L + kSegment - 1) / kSegment;

    if (tid == 0) {
        bar_init(bar(kFullRK), 1);
        bar_init(bar(kFullV0), 1);
        bar_init(bar(kFullV1), 1);
        bar_init(bar(kVReady), kStateThreads / 32);
        bar_init(bar(kScores), 1);
        bar_init(bar(kInc0), 1);
        bar_init(bar(kInc1), 1);
        bar_init(bar(kP), kScoreThreads / 32);
        bar_init(bar(kO1_0), 1);
        bar_init(bar(kO1_1), 1);
        bar_init(bar(kO2), kOutThreads / 32);
        bar_init(bar(kFix), kStateThreads / 32);
        bar_init(bar(kOutFull), kOutThreads / 32);
        bar_init(bar(kOutFree), 1);
        bar_init(bar(kDot), 1);
        bar_init(bar(kFinish), 1);
        bar_init(bar(kDotFree), kOutThreads / 32);
        for (int i = 0; i < 2; ++i) {
            bar_init(bar(kDecFull0 + i), 1);
            bar_init(bar(kDecFree0 + i), (kStateThreads + (STATE ? 0 : kScoreThreads + kOutThreads)) / 32);
        }
        failed[0] = failed[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(tmem_slot)), "n"(Lay::columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    // All columns are ours, so they start at 0: as a constant it costs the issuing warp no register moves per product.
    constexpr uint32_t tmem = 0;
    if (tid == 0 && (*tmem_slot != 0 || (base & 1023) != 0)) *failed = 1, atomicAdd(&g_tile_timeouts, 1ull);
    float *sums = reinterpret_cast<float *>(smem + Lay::sums);
    const int quarter = warp & 3, half = (warp >> 2) & 1;
    const int row = quarter * 32 + lane;                 // time step in the piece, or lane of tensor memory
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;

    // Pieces that nothing stands before (O2 is 0), and whose state nobody asks for (no V', no I)
    auto no_past = [&](const Item &it, int i) { return !STATE && it.first + i == 0 && a.init == nullptr; };
    auto no_future = [&](const Item &it, int i) {
        return !STATE && it.first + i + 1 == it.all && a.final == nullptr && !(DOT && !REV && a.keep_last);
    };

    if (warp < 8) {
        // ------------------------------------------------------------------ the state, and V' = tail weights times V
        constexpr int SC = KP == 128 ? 32 : 16;   // state columns per thread (64 state rows stand twice in the 128 lanes)
        const int srow = KP == 128 ? row : (quarter & 1) * 32 + lane;
        const int sc0 = KP == 128 ? half * 32 : (quarter >> 1) * 32 + half * 16;
        float S[SC];
        auto store_terms = [&]() {   // S as the B operand of R S: rows = state rows, 64 columns to a row
#pragma unroll
            for (int c = 0; c < SC / 8; ++c) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = S[c * 8 + j];
#pragma unroll
                for (int term = 0; term < NS; ++term) {
                    uint4 w;
                    if (NS == 2 && term == 0) {
                        w.x = cut_term(x[0], x[1]), w.y = cut_term(x[2], x[3]), w.z = cut_term(x[4], x[5]), w.w = cut_term(x[6], x[7]);
                    } else {
                        w.x = next_term<T>(x[0], x[1], term == NS - 1);
                        w.y = next_term<T>(x[2], x[3], term == NS - 1);
                        w.z = next_term<T>(x[4], x[5], term == NS - 1);
                        w.w = next_term<T>(x[6], x[7], term == NS - 1);
                    }
                    *reinterpret_cast<uint4 *>(smem + Lay::s + term * KP * 128 + swizzled(srow, sc0 / 8 + c)) = w;
                }
            }
            fence_before();
        };
        const float kv_scale = (float)a.kv_scale;
        int g = 0;
        bool ok = true;
#pragma unroll 1
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            const Item it(a, item, tiles, part);
            const int gcol0 = it.vt * 64 + sc0;
            const long long state0 = it.bh * a.d1 * a.d2;
            auto all_state = [&](bool transposed, long long first, auto fn) {   // fn(value, its position), (d1, d2) or (d2, d1)
                if (srow >= a.d1) return;
                const int step = transposed ? a.d1 : 1;
                long long at = first + (transposed ? (long long)gcol0 * a.d1 + srow : (long long)srow * a.d2 + gcol0);
#pragma unroll
                for (int j = 0; j < SC; ++j, at += step)
                    if (gcol0 + j < a.d2) fn(S[j], at);
            };
#pragma unroll
            for (int j = 0; j < SC; ++j) S[j] = 0.f;
            float *parts = a.split_states + ((it.bh * a.splits + part) * tiles + it.vt) * KP * 64 + tid;   // this part's, in the threads' order
            if (part > 0 && !STATE) {
                parts -= (long long)tiles * KP * 64;
#pragma unroll
                for (int j = 0; j < SC; ++j) S[j] = parts[j * kStateThreads];
            } else if (part == 0 && a.init != nullptr)
                all_state(a.init_transposed, state0, [&](float &v, long long at) { v = static_cast<const float *>(a.init)[at]; });
            if (!STATE && (part > 0 || a.init != nullptr)) store_terms();   // nothing stands before the first piece else
#pragma unroll 1
            for (int i = 0; i < it.pieces; ++i, ++g) {
                const uint32_t ph = g & 1;
                const long long t0 = it.start<REV>(i);
                const int m = (int)(it.n - t0 < kPiece ? it.n - t0 : kPiece);
                const long long end = t0 + m;
                const bool boundary = end == it.n || end % kSegment == 0;
                const DecayTables &d = tables[g & 1];
                if (!(ok = warp_wait(bar(kDecFull0 + (g & 1)), (g >> 1) & 1, failed))) break;
                if (!(ok = warp_wait(bar(kFullV0 + g % VS), (g / VS) & 1, failed))) break;
                const bool fix = a.lengths != nullptr && m < kPiece;
                unsigned char *v_tile = smem + Lay::v + (g % VS) * kTileBytes;
                if (fix) {
                    if (!(ok = warp_wait(bar(kFullRK), ph, failed))) break;
                    if (row >= m) {
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
                    fence_async();
                    warp_arrive(bar(kFix));
                }
                const float w = d.tail[row], keep = d.keep;
                const bool last = no_future(it, i);
#pragma unroll 2
                for (int c = 0; c < (last ? 0 : 4); ++c) {   // not wholly unrolled, like the loop over the scores: the roles' code has to stay in the instruction cache
                    const uint32_t at = swizzled(row, half * 4 + c);
                    const uint4 in = *reinterpret_cast<const uint4 *>(v_tile + at);
                    float2 x[4] = {unpack(in.x, T{}), unpack(in.y, T{}), unpack(in.z, T{}), unpack(in.w, T{})};
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
                fence_async();
                warp_arrive(bar(kVReady));
                warp_arrive(bar(kDecFree0 + (g & 1)));
                if (REV && !STATE && a.anchor_dots != nullptr && boundary) {
                    // the state behind this piece against the stored state of the steps up to here
                    const long long segment = (end - 1) / kSegment;
                    const float *anchor = static_cast<const float *>(a.anchors) + ((it.bh * segments + segment) * tiles + it.vt) * KP * 64 + tid;
                    float dot = 0.f;
                    if (end != it.n || a.init != nullptr)   // behind the last step there is nothing else
#pragma unroll
                        for (int j = 0; j < SC; ++j) dot = fmaf(S[j], anchor[j * kStateThreads], dot);
                    for (int s = 16; s >= 1; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
                    if (lane == 0) static_cast<float *>(a.anchor_dots)[((it.bh * segments + segment) * tiles + it.vt) * 8 + warp] = dot;
                }
                if (!(ok = warp_wait(bar(kInc0 + (g & 1)), (g >> 1) & 1, failed))) break;
                if (last) continue;
                fence_after();
#pragma unroll
                for (int c = 0; c < SC; c += 16) {
                    float x[16];
                    tmem_load16(tmem + lanes + Lay::c_i + (Lay::i_blocks - 1) * 64 + sc0 + c, x);
                    tmem_loaded();
#pragma unroll
                    for (int b = Lay::i_blocks - 2; b >= 0; --b) {
                        float y[16];
                        tmem_load16(tmem + lanes + Lay::c_i + b * 64 + sc0 + c, y);
                        tmem_loaded();
#pragma unroll
                        for (int j = 0; j < 16; j += 2) add_two(x[j], x[j + 1], y[j], y[j + 1]);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) S[c + j] = fmaf(S[c + j], keep, x[j] * kv_scale);
                }
                if (STATE || i + 1 == it.pieces) fence_before();
                else store_terms();
                if (!REV && !STATE && a.anchors != nullptr && boundary) {
                    // in the threads' own order: the sweep that reads them has the same threads
                    float *anchor = static_cast<float *>(a.anchors) + ((it.bh * segments + (end - 1) / kSegment) * tiles + it.vt) * KP * 64 + tid;
#pragma unroll
                    for (int j = 0; j < SC; ++j) anchor[j * kStateThreads] = S[j];
                }
            }
            if (STATE) {
#pragma unroll
                for (int j = 0; j < SC; ++j) parts[j * kStateThreads] = S[j];
            } else if (a.final != nullptr && part == a.splits - 1)
                all_state(a.final_transposed, state0, [&](float &v, long long at) { static_cast<float *>(a.final)[at] = v; });
        }
    } else if (warp < 16) {
        // ------------------------------------------------------------------ P = scores, weighted
        const uint32_t own = tmem + lanes + half * 64;   // this thread's columns of the scores
        const float kv_scale = (float)a.kv_scale;
        int g = 0;
        bool ok = !STATE;
#pragma unroll 1
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            const Item it(a, item, tiles, part);
#pragma unroll 1
            for (int i = 0; i < it.pieces; ++i, ++g) {
                const DecayTables &d = tables[g & 1];
                if (!(ok = warp_wait(bar(kDecFull0 + (g & 1)), (g >> 1) & 1, failed))) break;
                const float la = d.la[row], lb = d.lb[row];
                float f[2];   // 2^(a_t - (a at the low end of the block)) for the two blocks of 32 columns
#pragma unroll
                for (int q = 0; q < 2; ++q) f[q] = kv_scale * exp_two((float)(d.a[row] - d.a[(half * 2 + q) * 32 + (REV ? 0 : 31)]));
                if (!(ok = warp_wait(bar(kScores), g & 1, failed))) break;
                fence_after();
                float sum = 0.f;
                // rows behind the last step are nobody's, and the product leaves out a second half of 64 columns without any
                const int m = (int)(it.n - it.start<REV>(i));
                const int chunks = quarter * 32 < m && half * 64 < m ? 4 : 0;
#pragma unroll 1
                for (int q = 0; q < chunks; ++q) {   // 16 columns each
                    const int block = half * 2 + q / 2, s0 = half * 64 + q * 16;
                    uint32_t p[8], left[8];   // P's two terms
                    if (REV ? block >= quarter : block <= quarter) {
                        float x[16], y[16];
                        tmem_load16(own + q * 16, x);
                        if (DOT) tmem_load16(own + Lay::c_two + q * 16, y);
                        const float4 *table = reinterpret_cast<const float4 *>((block == quarter ? d.la : d.cf) + s0);
                        float t[16];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float4 v = table[j];
                            t[4 * j] = v.x, t[4 * j + 1] = v.y, t[4 * j + 2] = v.z, t[4 * j + 3] = v.w;
                        }
                        if (block == quarter) {
                            const float4 *rest = reinterpret_cast<const float4 *>(d.lb + s0);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {   // a_t - a_s to 24 bits of its own size, not of the two's
                                const float4 v = rest[j];
                                t[4 * j] = (la - t[4 * j]) + (lb - v.x), t[4 * j + 1] = (la - t[4 * j + 1]) + (lb - v.y);
                                t[4 * j + 2] = (la - t[4 * j + 2]) + (lb - v.z), t[4 * j + 3] = (la - t[4 * j + 3]) + (lb - v.w);
                            }
                            const int j0 = row - s0;   // the step's own column
#pragma unroll
                            for (int j = 0; j < 16; ++j) t[j] = (REV ? j >= j0 : j <= j0) ? kv_scale * exp_two(t[j]) : 0.f;
                        } else {
                            const float fq = q < 2 ? f[0] : f[1];
#pragma unroll
                            for (int j = 0; j < 16; j += 2) mul_two(t[j], t[j + 1], fq, fq);
                        }
                        tmem_loaded();
                        // (a score that is not finite gives NaN against a weight of 0, too: in rows behind the end nobody reads it,
                        // in others the operands have to be finite)
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            mul_two(x[j], x[j + 1], t[j], t[j + 1]);
                            if (DOT) sum = fmaf(x[j + 1], y[j + 1], fmaf(x[j], y[j], sum));
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            p[j] = cut_term(x[2 * j], x[2 * j + 1]);
                            left[j] = next_term<T>(x[2 * j], x[2 * j + 1], true);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) p[j] = left[j] = 0;
                    }
                    tmem_store8(own + q * 16, p);
                    tmem_store8(own + q * 16 + 8, left);
                }
                if (DOT) sums[((g & 1) * 2 + half) * kPiece + row] = sum;
                tmem_stored();
                fence_before();
                warp_arrive(bar(kP));
                warp_arrive(bar(kDecFree0 + (g & 1)));
            }
        }
    } else if (warp < 20) {
        // ------------------------------------------------------------------ out
        T *out_t = static_cast<T *>(a.out);
        float *out_f = static_cast<float *>(a.out);
        const bool staged = !a.out_acc;
        const bool writer = tid == kStateThreads + kScoreThreads;   // starts the copies of the output tiles
        int g = 0;
        bool ok = true;
#pragma unroll 1
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            const Item it(a, item, tiles, part);
            const int col0 = it.vt * 64;
#pragma unroll 1
            for (int i = 0; i < (STATE ? 0 : it.pieces); ++i, ++g) {
                const long long t0 = it.start<REV>(i), t = t0 + row;
                const int m = (int)(it.n - t0 < kPiece ? it.n - t0 : kPiece);
                if (!(ok = warp_wait(bar(kDecFull0 + (g & 1)), (g >> 1) & 1, failed))) break;
                const float out_scale = (float)a.out_scale, head = tables[g & 1].head[row];
                warp_arrive(bar(kDecFree0 + (g & 1)));
                // the state's part first, into O1's columns: it is there before P, and O2's columns are free at once
                const bool past = !no_past(it, i);
                float dot = 0.f;
                if (DOT && !(ok = warp_wait(bar(kDot), g & 1, failed))) break;
                if (!(ok = warp_wait(bar(kInc0 + (g & 1)), (g >> 1) & 1, failed))) break;   // without a past too: no phase is left out
                fence_after();
                if (past) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {   // 16 columns each
                        float u[16];
                        tmem_load16(tmem + lanes + Lay::c_o2 + c * 16, u);
                        if constexpr (Lay::o2_blocks > 1) {
                            float w[16];
                            tmem_load16(tmem + lanes + Lay::c_o2 + 64 + c * 16, w);
                            tmem_loaded();
#pragma unroll
                            for (int j = 0; j < 16; j += 2) add_two(u[j], u[j + 1], w[j], w[j + 1]);
                        } else {
                            tmem_loaded();
                        }
#pragma unroll
                        for (int j = 0; j < 16; j += 2) mul_two(u[j], u[j + 1], head, head);
                        tmem_store16(tmem + lanes + Lay::c_o1 + c * 16, u);
                        if (DOT && row < m)
#pragma unroll
                            for (int e = 0; e < 16; e += 8) {
                                const uint4 p = *reinterpret_cast<const uint4 *>(smem + Lay::dot + swizzled(row, c * 2 + e / 8));
                                const float2 two[4] = {unpack(p.x, T{}), unpack(p.y, T{}), unpack(p.z, T{}), unpack(p.w, T{})};
#pragma unroll
                                for (int j = 0; j < 4; ++j) dot = fmaf(u[e + 2 * j], two[j].x, fmaf(u[e + 2 * j + 1], two[j].y, dot));
                            }
                    }
                    tmem_stored();
                    fence_before();
                }
                warp_arrive(bar(kO2));
                if (DOT) warp_arrive(bar(kDotFree));
                if (staged && g > 0 && !(ok = warp_wait(bar(kOutFree), (g - 1) & 1, failed))) break;
                if (!(ok = warp_wait(bar(kO1_0 + (g & 1)), (g >> 1) & 1, failed))) break;
                fence_after();
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float u[16];
                    tmem_load16(tmem + lanes + Lay::c_o1 + c * 16, u);
                    tmem_loaded();
#pragma unroll
                    for (int j = 0; j < 16; ++j) u[j] = row < m ? u[j] * out_scale : 0.f;
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        const int col = col0 + c * 16 + e;
                        if (staged) {
                            uint4 o;
                            o.x = pack(u[e], u[e + 1], T{});
                            o.y = pack(u[e + 2], u[e + 3], T{});
                            o.z = pack(u[e + 4], u[e + 5], T{});
                            o.w = pack(u[e + 6], u[e + 7], T{});
                            *reinterpret_cast<uint4 *>(smem + Lay::out + swizzled(row, c * 2 + e / 8)) = o;
                        } else if (t < a.L && col < a.d2) {
                            float *at = out_f + (((long long)it.b * a.L + t) * a.H + it.h) * a.d2 + col;
                            *reinterpret_cast<float4 *>(at) = make_float4(u[e], u[e + 1], u[e + 2], u[e + 3]);
                            *reinterpret_cast<float4 *>(at + 4) = make_float4(u[e + 4], u[e + 5], u[e + 6], u[e + 7]);
                        }
                    }
                }
                if (DOT && t < a.L) {
                    const float pairs = sums[((g & 1) * 2) * kPiece + row] + sums[((g & 1) * 2 + 1) * kPiece + row];
                    a.dots[((long long)it.vt * a.B * a.L + (long long)it.b * a.L + t) * a.H + it.h] = row < m ? (pairs + dot) * out_scale : 0.f;
                }
                fence_before();
                if (staged) {
                    fence_async();
                    warp_arrive(bar(kOutFull));
                    if (writer && bar_wait(bar(kOutFull), g & 1, failed)) {
                        // steps behind the tensor's end and columns behind its rows are not written
                        tma_store(base + Lay::out, &map_out, col0, it.h, (int)t0, (int)it.b);
                        tma_store_read();
                        bar_arrive(bar(kOutFree));
                    }
                    __syncwarp();
                }
            }
            if (!ok) break;
            // rows behind the last piece
            const long long end = STATE || part < a.splits - 1 ? a.L : (long long)it.all * kPiece;
            for (long long e = tid - (kStateThreads + kScoreThreads); e < (a.L - end) * 8; e += kOutThreads) {
                const long long t = end + e / 8;
                const int col = col0 + (int)(e % 8) * 8;
                if (col >= a.d2) continue;
                const long long at = (((long long)it.b * a.L + t) * a.H + it.h) * a.d2 + col;
                const uint4 zero = {0, 0, 0, 0};
                *reinterpret_cast<uint4 *>(a.out_acc ? (void *)(out_f + at) : (void *)(out_t + at)) = zero;
                if (a.out_acc) *reinterpret_cast<uint4 *>(out_f + at + 4) = zero;
            }
            if (DOT)
                for (long long t = end + tid - (kStateThreads + kScoreThreads); t < a.L; t += kOutThreads)
                    a.dots[((long long)it.vt * a.B * a.L + (long long)it.b * a.L + t) * a.H + it.h] = 0.f;
        }
        if (writer) tma_store_done();
    } else if (warp == 20) {
        // ------------------------------------------------------------------ TMA and MMA
        const uint32_t lead = lane == 0, base16 = base >> 4;
        // I = K^T V' (all terms of V' in one product where they have columns of their own: K is read once); with 64 state rows the
        // second block of 64 is the first once more
        auto state_product = [&](int g) {
#pragma unroll
            for (int term = NV - Lay::i_blocks; term >= 0; --term)
#pragma unroll
                for (int j = 0; j < kPiece / 16; ++j)
                    mma_ss(tmem + Lay::c_i, tile_desc(base16 + ((Lay::k + j * 2048) >> 4), KP == 128 ? kTileBytes : 0),
                           tile_desc(base16 + ((Lay::vw + term * kTileBytes + j * 2048) >> 4), kTileBytes),
                           instr_desc<T>(Lay::i_blocks * 64, true, true), term < NV - Lay::i_blocks || j > 0, lead);
            mma_commit(bar(kInc0 + (g & 1)), lead);
        };
        int g = 0, fixes = 0;
        bool ok = true;
#pragma unroll 1
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            const Item it(a, item, tiles, part);
#pragma unroll 1
            for (int i = 0; i < it.pieces; ++i, ++g) {
                const uint32_t ph = g & 1;
                if (!(ok = warp_wait(bar(kFullRK), ph, failed))) break;
                if (a.lengths != nullptr && it.n - it.start<REV>(i) < kPiece && !(ok = warp_wait(bar(kFix), fixes++ & 1, failed))) break;
                if constexpr (STATE) {   // I alone
                    if (!(ok = warp_wait(bar(kVReady), ph, failed))) break;
                    fence_after();
                    state_product(g);
                    continue;
                }
                if (g > 0 && !(ok = warp_wait(bar(kO1_0 + (ph ^ 1)), ((g - 1) >> 1) & 1, failed))) break;   // P of the piece before has been used
                if (DOT && !(ok = warp_wait(bar(kDot), ph, failed) && warp_wait(bar(kFullV0 + g % VS), (g / VS) & 1, failed))) break;
                fence_after();
                const uint32_t v16 = base16 + (Lay::v >> 4) + (VS == 2 ? ph * (kTileBytes >> 4) : 0);
                // scores = R K^T
#pragma unroll
                for (int j = 0; j < KP / 16; ++j) {
                    const uint32_t off = (j / 4) * kTileBytes + (j % 4) * 32;
                    mma_ss(tmem, tile_desc(base16 + ((Lay::r + off) >> 4), 16), tile_desc(base16 + ((Lay::k + off) >> 4), 16),
                           instr_desc<T>(128, false, false), j > 0, lead);
                }
                if (DOT)   // Y V^T
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_ss(tmem + Lay::c_two, tile_desc(base16 + ((Lay::dot + j * 32) >> 4), 16), tile_desc(v16 + j * 2, 16),
                               instr_desc<T>(128, false, false), j > 0, lead);
                mma_commit(bar(kScores), lead);
                // O2 = R S, when the state's operand is there (it was written before V').  Small terms go first into a common accumulator
                // here and below, or into one that holds small ones only: it drops what does not fit its 24 bits at every step, towards zero.
                if (!(ok = warp_wait(bar(kVReady), ph, failed))) break;
                fence_after();
                const bool past = !no_past(it, i), future = !no_future(it, i);
                if (past)
#pragma unroll
                for (int term = 0; term < NS; term += 2)   // the first two terms in one product, the third added to the second
#pragma unroll
                    for (int j = 0; j < KP / 16; ++j)
                        mma_ss(tmem + Lay::c_o2 + term / 2 * 64, tile_desc(base16 + ((Lay::r + (j / 4) * kTileBytes + (j % 4) * 32) >> 4), 16),
                               tile_desc(base16 + ((Lay::s + term * KP * 128 + j * 2048) >> 4), KP * 128),
                               instr_desc<T>(term == 0 ? Lay::o2_blocks * 64 : 64, false, true), term > 0 || j > 0, lead);
                if (future) state_product(g);
                else mma_commit(bar(kInc0 + (g & 1)), lead);
                // O1 += P V, on top of the state's part, which the output warps put there
                if (!(ok = warp_wait(bar(kP), ph, failed) && warp_wait(bar(kO2), ph, failed))) break;
                fence_after();
                auto half_product = [&](int j0, bool add) {   // of 64 steps; P's second term, then its first
#pragma unroll
                    for (int left = 8; left >= 0; left -= 8)
#pragma unroll
                        for (int j = j0; j < j0 + 4; ++j)
                            mma_ts(tmem + Lay::c_o1, tmem + j * 16 + left, tile_desc(v16 + (j * 2048 >> 4), kTileBytes),
                                   instr_desc<T>(64, false, true), add || left == 0 || j > j0, lead);
                };
                half_product(0, past);
                if (it.n - it.start<REV>(i) > kPiece / 2) half_product(4, true);
                mma_commit(bar(kO1_0 + (g & 1)), lead);
            }
        }
    } else if (warp == 21) {
        // ------------------------------------------------------------------ TMA
        if (lane == 0) {   // one thread; the piece's copies in the order in which their places become free
            int g = 0, stop = 0;
#pragma unroll 1
            for (int item = blockIdx.x; item < items && !stop; item += gridDim.x) {
                const Item it(a, item, tiles, part);
                const int rh = it.h / a.r.share, kh = it.h / a.k.share, vh = it.h / a.v.share, dh = DOT ? it.h / a.dot.share : 0;
#pragma unroll 1
                for (int i = 0; i < it.pieces; ++i, ++g) {
                    const int t0 = (int)it.start<REV>(i), b = (int)it.b;
                    auto load_v = [&]() {   // behind the last product that reads the V in its place
                        if (g >= VS && !bar_wait(bar((STATE ? kInc0 : kO1_0) + ((g - VS) & 1)), ((g - VS) >> 1) & 1, failed)) return false;
                        bar_expect(bar(kFullV0 + g % VS), kTileBytes);
                        tma_load(base + Lay::v + (g % VS) * kTileBytes, &map_v, bar(kFullV0 + g % VS), it.vt * 64, vh, t0, b);
                        return true;
                    };
                    if (VS == 2 && !load_v()) { stop = 1; break; }
                    if (DOT) {
                        if (g > 0 && !(bar_wait(bar(kScores), (g - 1) & 1, failed) && bar_wait(bar(kDotFree), (g - 1) & 1, failed))) { stop = 2; break; }
                        bar_expect(bar(kDot), kTileBytes);
                        tma_load(base + Lay::dot, &map_dot, bar(kDot), it.vt * 64, dh, t0, b);
                    }
                    if (g > 0 && !bar_wait(bar(kInc0 + ((g - 1) & 1)), ((g - 1) >> 1) & 1, failed)) { stop = 3; break; }   // the last product that reads R and K
                    bar_expect(bar(kFullRK), (STATE ? 1 : 2) * Lay::panels * kTileBytes);
#pragma unroll
                    for (int p = 0; p < Lay::panels; ++p) {
                        if (!STATE) tma_load(base + Lay::r + p * kTileBytes, &map_r, bar(kFullRK), p * 64, rh, t0, b);
                        tma_load(base + Lay::k + p * kTileBytes, &map_k, bar(kFullRK), p * 64, kh, t0, b);
                    }
                    if (VS == 1 && !load_v()) { stop = 4; break; }
                }
            }
            // let what is in flight land before the block gives its memory back, whoever else fails from here on: g whole pieces,
            // and what the last one got
            const int v = g + (stop > 1 && VS == 2), dots = g + (stop > 2), rk = g + (stop > 3);
            if (rk > 0) bar_wait(bar(kFullRK), (rk - 1) & 1, failed + 1);
            if (DOT && dots > 0) bar_wait(bar(kDot), (dots - 1) & 1, failed + 1);
            for (int i = v > VS ? v - VS : 0; i < v; ++i) bar_wait(bar(kFullV0 + i % VS), (i / VS) & 1, failed + 1);
        }
        __syncwarp();
    } else {
        int count = 0;
#pragma unroll 1
        for (int item = blockIdx.x; item < items && !*failed; item += gridDim.x) {
            const Item it(a, item, tiles, part);
            const float *g = static_cast<const float *>(a.decay) + (long long)it.b * a.decay_stride[0] + it.h * a.decay_stride[2];
            const double whole = sum_decays<REV>(g, a.decay_stride[1], it.n, it.first, it.pieces, count, tables, bar(kDecFull0), bar(kDecFree0), failed);
            if (STATE && it.vt == 0 && lane == 0) a.split_decays[it.bh * a.splits + part] = (float)whole;
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 20) {
        fence_after();
        if (*failed) {   // products in flight read shared and tensor memory
            if (lane == 0) report_failure(a.failure);
            mma_commit(bar(kFinish), lane == 0);
            warp_wait(bar(kFinish), 0, failed + 1);
        }
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Lay::columns));
    }
}

// ------------------------------------------------------------------------------------------ host side

template <typename T, int KP, int NS, int NV, bool DOT, bool REV>
int launch_tiles(const Sweep &a, int dtype, cudaStream_t stream)
{
    CUtensorMap r, k, v, out, dot;
    const SweepOperand o{a.out, {a.L * a.H * a.d2, (long long)a.H * a.d2, a.d2}, 1};
    if (encoder() == nullptr || !encode(&r, a.r, a, a.d1, dtype) || !encode(&k, a.k, a, a.d1, dtype) ||
        !encode(&v, a.v, a, a.d2, dtype) || !encode(&out, o, a, a.d2, dtype) ||
        !encode(&dot, a.dot.data ? a.dot : o, a, a.d2, dtype))
        return PSIG_ERR_CUDA;
    const int tiles = tile_columns(a.d2);
    // an SM holds one block: no more than that, each takes every so many items
    const long long items = a.B * a.H * tiles;
    const unsigned blocks = (unsigned)(items < 148 ? items : 148);
    if (a.splits > 1) {
        using Lay = TileLayout<KP, 1, 3, false>;
        auto kernel = attn_sweep_tiles<T, KP, 1, 3, false, REV, true>;
        if (!prepare_kernel(kernel, Lay::alloc, true)) return PSIG_ERR_CUDA;
        kernel<<<dim3(blocks, a.splits - 1), kTileThreads, Lay::alloc, stream>>>(r, k, v, out, dot, a);
        int rc = check_launch();
        if (rc != PSIG_OK || (rc = chain_states(a, (long long)KP * 64 * tiles, stream)) != PSIG_OK) return rc;
    }
    using Lay = TileLayout<KP, NS, NV, DOT>;
    auto kernel = attn_sweep_tiles<T, KP, NS, NV, DOT, REV, false>;
    if (!prepare_kernel(kernel, Lay::alloc, true)) return PSIG_ERR_CUDA;
    kernel<<<dim3(blocks, a.splits), kTileThreads, Lay::alloc, stream>>>(r, k, v, out, dot, a);
    return check_launch();
}

template <typename T, bool REV>
int select_tiles(const Sweep &a, int dtype, cudaStream_t stream)
{
    if (a.dot.data != nullptr)
        return a.d1 <= 64 ? launch_tiles<T, 64, 3, 3, true, REV>(a, dtype, stream) : launch_tiles<T, 128, 3, 3, true, REV>(a, dtype, stream);
    // two terms of V' (16 bits) are plenty for a state that nobody sees but through a 16-bit output
    if (a.final == nullptr)
        return a.d1 <= 64 ? launch_tiles<T, 64, 2, 2, false, REV>(a, dtype, stream) : launch_tiles<T, 128, 2, 2, false, REV>(a, dtype, stream);
    return a.d1 <= 64 ? launch_tiles<T, 64, 2, 3, false, REV>(a, dtype, stream) : launch_tiles<T, 128, 2, 3, false, REV>(a, dtype, stream);
}

}  // namespace

// Head sizes up to 128, in whole 16-byte pieces (TMA); as many items (two tiles a head) as an int counts in steps of a
// grid.  Both forms take the same sizes; a backward pass's three sweeps go the same way.
bool attn_tiles_supported(const Sweep &a, int dtype)
{
    const int size = dtype == PSIG_F32 ? 4 : 2;
    return dtype != PSIG_F64 && a.d1 <= 128 && a.d2 <= 128 && a.L < (1LL << 31) - kPiece && a.B < (1LL << 31) && a.B * a.H < (1LL << 30) - 148 &&
           operand_fits(a.r, a, a.d1, size) && operand_fits(a.k, a, a.d1, size) && operand_fits(a.v, a, a.d2, size);
}

int attn_sweep_on_tiles(const Sweep &a, bool exact, int dtype, cudaStream_t stream)
{
    if (dtype != PSIG_BF16) return attn_sweep_split(a, exact, dtype, stream);
    return a.reverse ? select_tiles<__nv_bfloat16, true>(a, dtype, stream) : select_tiles<__nv_bfloat16, false>(a, dtype, stream);
}

long long attn_tile_timeouts() { return take_timeouts(); }

}  // namespace psig
