// Decayed linear attention on the tensor cores (bfloat16 operands): one sweep over pieces of 128 time steps.
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
// wait is bounded (psig_sequence_wait_timeouts).
#include "tiles.cuh"

namespace psig {
namespace {

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
        failed[1] = 0;
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
            int loaded_rk = 1, done_rk = 0, loaded_v = 0;
            load_rk(0);
            load_v(0);
            if (VS == 2 && pieces > 1) load_v(1);
            loaded_v = VS == 2 && pieces > 1 ? 2 : 1;
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
                for (int term = NS - 1; term >= 0; --term)   // small terms first, as the accumulator truncates
#pragma unroll
                    for (int j = 0; j < KP / 16; ++j)
                        mma_ss(tmem + Lay::c_o2, tile_desc(base + Lay::r + (j / 4) * kTileBytes + (j % 4) * 32, 16),
                               tile_desc(base + Lay::s + term * KP * 128 + j * 2048, kTileBytes), instr_desc<T>(64, false, true),
                               term < NS - 1 || j > 0);
                if (!bar_wait(bar(kVReady), ph, failed)) break;
                fence_after();
                // I = K^T V'; with 64 state rows the second block of 64 is the first once more
#pragma unroll
                for (int term = NV - 1; term >= 0; --term)   // small terms first, as the accumulator truncates
#pragma unroll
                    for (int j = 0; j < kPiece / 16; ++j)
                        mma_ss(tmem + Lay::c_o1, tile_desc(base + Lay::k + j * 2048, KP == 128 ? kTileBytes : 0),
                               tile_desc(base + Lay::vw + term * kTileBytes + j * 2048, kTileBytes), instr_desc<T>(64, true, true),
                               term < NV - 1 || j > 0);
                mma_commit(bar(kInc));
                if (!bar_wait(bar(kInc), ph, failed)) break;
                if (i + 1 < pieces) {
                    load_rk(i + 1);
                    ++loaded_rk;
                }
                if (VS == 2 && i > 0 && i + 1 < pieces) load_v(i + 1), ++loaded_v;   // the buffer of piece i - 1, whose O1 has been read
                if (!bar_wait(bar(kP), ph, failed)) break;
                fence_after();
                // O1 = P V
#pragma unroll
                for (int term = NP - 1; term >= 0; --term)   // small terms first, as the accumulator truncates
#pragma unroll
                    for (int j = 0; j < kPiece / 16; ++j) {
                        const int col = term == 0 ? (j / 4) * 64 + (j % 4) * 8 : Lay::c_p + (term - 1) * 64 + j * 8;
                        mma_ts(tmem + Lay::c_o1, tmem + col, tile_desc(base + Lay::v + (i % VS) * kTileBytes + j * 2048, kTileBytes),
                               instr_desc<T>(64, false, true), term < NP - 1 || j > 0);
                    }
                mma_commit(bar(kO1));
                if (VS == 1 && i + 1 < pieces) {
                    if (!bar_wait(bar(kO1), ph, failed)) break;
                    load_v(i + 1);
                    ++loaded_v;
                }
            }
            if (*failed) {
                // let what is in flight land before the block gives its memory back
                if (loaded_rk > done_rk) bar_wait(bar(kFullRK), (loaded_rk - 1) & 1, failed + 1);
                for (int i = 0; i < VS && i < loaded_v; ++i)
                    bar_wait(bar(kFullV0 + (loaded_v - 1 - i) % VS), ((loaded_v - 1 - i) / VS) & 1, failed + 1);
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        const float *g = static_cast<const float *>(a.decay) + b * a.decay_stride[0] + h * a.decay_stride[2];
        sum_decays<REV>(g, a.decay_stride[1], n, pieces, tables, bar(kDecFull0), bar(kDecFree0), failed);
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
                uint32_t p0[8], p1[8], p2[8];
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
                tmem_store8(own + q * 8, p0);
                if (NP > 1) tmem_store8(tmem + lanes + Lay::c_p + half * 32 + q * 8, p1);
                if (NP > 2) tmem_store8(tmem + lanes + Lay::c_p + 64 + half * 32 + q * 8, p2);
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

}  // namespace

// Head sizes up to 128, in whole 16-byte pieces (TMA).  Both forms take the same sizes: a call's forward pass and its
// three gradients go the same way.
bool attn_tiles_supported(const Sweep &a, int dtype)
{
    const int size = dtype == PSIG_F32 ? 4 : 2;
    return dtype != PSIG_F64 && a.d1 <= 128 && a.d2 <= 128 && a.L < (1LL << 31) && a.B < (1LL << 31) && a.B * a.H < (1LL << 30) &&
           operand_fits(a.r, a, a.d1, size) && operand_fits(a.k, a, a.d1, size) && operand_fits(a.v, a, a.d2, size);
}

int attn_sweep_on_tiles(const Sweep &a, bool exact, int dtype, cudaStream_t stream)
{
    if (dtype != PSIG_BF16) return attn_sweep_split(a, exact, dtype, stream);
    return a.reverse ? select_tiles<__nv_bfloat16, true>(a, exact, dtype, stream)
                     : select_tiles<__nv_bfloat16, false>(a, exact, dtype, stream);
}

long long attn_tile_timeouts() { return take_timeouts(); }

}  // namespace psig
