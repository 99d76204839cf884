// Building blocks of the tensor-core sweeps (linear_attention_tiles.cu, linear_attention_split.cu): tensor memory,
// matrix instructions, TMA, bounded waits, and the decay tables of a piece (internal header).
#pragma once

#include "sequence.cuh"

#include <cuda.h>

#include <type_traits>

namespace psig {

namespace {

__device__ unsigned long long g_tile_timeouts;   // of the translation unit

// Read and clear.
[[maybe_unused]] long long take_timeouts()
{
    unsigned long long count = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&count, g_tile_timeouts, sizeof(count)) != cudaSuccess) return -1;
    if (count != 0) cudaMemcpyToSymbol(g_tile_timeouts, &zero, sizeof(zero));
    return (long long)count;
}

constexpr int kPiece = 128;
constexpr int kTileBytes = kPiece * 128;      // 128 rows of 64 16-bit values

struct DecayTables {       // of one piece; all exponents are of 2
    double a[kPiece];      // a_t
    float la[kPiece];      // a_s - (a at the low end of s's block of 32)
    float lb[kPiece];      // what rounding that to la left
    float cf[kPiece];      // 2^-la
    float tail[kPiece];    // 2^(a_end - a_s)
    float head[kPiece];    // 2^a_t
    float keep;            // 2^a_end, what is left of the state
    float pad[3];
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
__device__ __forceinline__ bool bar_passed(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Out of line: the code of all roles has to fit the instruction cache.
__device__ __noinline__ bool bar_wait_on(uint32_t bar, uint32_t parity, volatile int *failed)
{
    unsigned long long start = 0;
#pragma unroll 1
    for (unsigned i = 0; i < kWaitPolls; ++i) {
        if (bar_passed(bar, parity)) return true;
        if (*failed || wait_expired(i, start)) break;
    }
    if (*failed) return false;
    if (atomicExch(const_cast<int *>(failed), 1) == 0) atomicAdd(&g_tile_timeouts, 1ull);
    return false;
}
// Waits for the phase of this parity; false when the bound ran out here or in another thread of the block.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *failed)
{
    return bar_passed(bar, parity) || bar_wait_on(bar, parity, failed);
}
// For a whole warp: all lanes wait (one lane that polls for the others measured slower, 404 -> 652 us for a 16384-step history),
// one lane arrives for all lanes' work before it.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *failed)
{
    return __all_sync(0xffffffffu, bar_wait(bar, parity, failed));
}
__device__ __forceinline__ void warp_arrive(uint32_t bar)
{
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(bar);
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int head, int t, int b)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(head), "r"(t), "r"(b) : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle, from an address in units of 16 bytes.  Rows of 128 bytes, eight
// rows (1024 bytes) to a swizzle atom; `lead` (bytes) is the distance of neighbouring 64-element blocks where the row
// runs along M or N.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr16, uint32_t lead)
{
    return (uint64_t)(addr16 | (lead >> 4) << 16) | (uint64_t)((1024u >> 4) | 1u << 14 | 2u << 29) << 32;
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t instr_desc(int n, bool a_rows_along_m, bool b_rows_along_n)
{
    const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | ((a_rows_along_m ? 1u : 0u) << 15) | ((b_rows_along_n ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// Matrix instructions run in the one thread of the warp with `lead` set, but the warp stays together: the operands are then
// uniform, and issuing one takes a handful of cycles (from a branch of a single thread it took 55 to 65).
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add, uint32_t lead)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add, uint32_t lead)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t lead)
{
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&x)[16])
{
    uint32_t *r = reinterpret_cast<uint32_t *>(x);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_load8(uint32_t addr, float (&x)[8])
{
    uint32_t *r = reinterpret_cast<uint32_t *>(x);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr));
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const float (&x)[16])
{
    const uint32_t *r = reinterpret_cast<const uint32_t *>(x);
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

// Two additions, subtractions or products in one instruction.
__device__ __forceinline__ void add_two(float &x, float &y, float a, float b)
{
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ void mul_two(float &x, float &y, float a, float b)
{
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}

// The first of two bfloat16 terms of a pair, cut instead of rounded (one instruction for both); leaves the rest, which the second
// term rounds: together within 2^-15, where two rounded terms are within 2^-16.
__device__ __forceinline__ uint32_t cut_term(float &x, float &y)
{
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    add_two(x, y, -__uint_as_float(a & 0xFFFF0000u), -__uint_as_float(b & 0xFFFF0000u));
    return __byte_perm(a, b, 0x7632);
}
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

__device__ __forceinline__ void tma_store(uint32_t src, const CUtensorMap *map, int x, int head, int t, int b)
{
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                 ::"l"(map), "r"(src), "r"(x), "r"(head), "r"(t), "r"(b) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

// A block's work: one column tile of one head of one sequence, or a part of it.  Blocks take items one after the other; the
// pieces of all of them are counted through (`g` below), so that a piece's stages overlap across the items, too: with
// sequences of one piece (61 steps, 2048 of them) a block each, 82 us a sweep went to starting blocks up.
struct Item {
    int vt, h, b, all, first, pieces;   // column tile, head, sequence; pieces of the sequence; this part's first and number
    long long bh, n;                    // n: steps of the sequence
    __device__ __forceinline__ Item(const Sweep &a, int item, int tiles, int part)
    {
        // fewer than 2^31 items (attn_tiles_supported), one or two column tiles
        const unsigned head = tiles == 1 ? item : (unsigned)item >> 1;
        vt = tiles == 1 ? 0 : item & 1;
        b = (int)(head / (unsigned)a.H);
        h = (int)(head - (unsigned)b * a.H);
        bh = head;
        int steps = (int)a.L;
        if (a.lengths != nullptr) {
            const int len = a.lengths[b];
            steps = len < 0 ? 0 : len > steps ? steps : len;
        }
        n = steps;
        all = (steps + (kPiece - 1)) / kPiece;
        first = 0, pieces = all;
        if (a.splits > 1) {   // at most 64 parts of at most 2^24 pieces
            first = (int)((unsigned)all * part / (unsigned)a.splits);
            pieces = (int)((unsigned)all * (part + 1) / (unsigned)a.splits) - first;
        }
    }
    template <bool REV>
    __device__ __forceinline__ long long start(int i) const { return (long long)(REV ? all - 1 - first - i : first + i) * kPiece; }
};

// One warp: the decay tables of `pieces` of the sweep's pieces from number `first` on, one piece ahead of their use, in two
// buffers in turn (`count` counts the pieces over all items).  Returns the sum of all their decays (exponent of 2).
template <bool REV>
__device__ __forceinline__ double sum_decays(const float *g, long long stride, long long n, int first, int pieces, int &count, DecayTables *tables,
                                             uint32_t full0, uint32_t free0, volatile int *failed)
{
    const int all = (int)((n + kPiece - 1) / kPiece);
    double whole = 0.0;
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int i = 0; i < pieces; ++i, ++count) {
        const long long t0 = (long long)(REV ? all - 1 - first - i : first + i) * kPiece;
        const int m = (int)(n - t0 < kPiece ? n - t0 : kPiece);
        double c[4];
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t = lane * 4 + j;
            float x = t < m ? g[(t0 + t) * stride] : 0.f;
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
        whole += end;
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = REV ? end - (before + c[j]) : before + c[j];
        // the low end of each block of 32 steps: its last step, or, in reverse, its first
        const double low = __shfl_sync(0xffffffffu, REV ? c[0] : c[3], REV ? (lane & ~7) : (lane | 7));
        if (count >= 2 && !warp_wait(free0 + 8 * (count & 1), ((count >> 1) & 1) ^ 1, failed)) break;
        DecayTables &d = tables[count & 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t = lane * 4 + j;
            const float la = (float)(c[j] - low);
            d.a[t] = c[j];
            d.la[t] = la;
            d.lb[t] = (float)((c[j] - low) - (double)la);
            d.cf[t] = exp_two(-la);
            d.tail[t] = exp_two((float)(end - c[j]));
            d.head[t] = exp_two((float)c[j]);
        }
        if (lane == 0) d.keep = exp_two((float)end);
        warp_arrive(full0 + 8 * (count & 1));
    }
    return whole;
}

// Parts of a long sequence, each swept by a block of its own: a first launch computes every part's state (all but the last; the
// first from the initial state), these are chained, and the sweep starts each part from the state before it.
__global__ void __launch_bounds__(256) chain_split_states(float *__restrict__ states, const float *__restrict__ decays, int splits,
                                                          long long per_part, long long per_head)
{
    // states (heads, splits, per_part), decays (heads, splits); parts of one head are chained in order
    const long long head = blockIdx.x;
    const long long e = (long long)blockIdx.y * 256 + threadIdx.x;
    if (e >= per_part) return;
    float *s = states + head * splits * per_part + e;
    float before = s[0];
    for (int i = 1; i + 1 < splits; ++i) {
        before = fmaf(before, exp_two(decays[head * per_head + i]), s[i * per_part]);
        s[i * per_part] = before;
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encoder()
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

// (d, heads, L, B) of values of a type; a box is one row of 128 bytes of one head at 128 time steps.
inline bool encode(CUtensorMap *map, const SweepOperand &o, const Sweep &a, int d, int dtype)
{
    const int size = dtype == PSIG_F32 ? 4 : 2;
    const long long heads = a.H / o.share;
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)a.L, (cuuint64_t)a.B};
    // the stride of a dimension of one element is never used, but has to be a valid one
    auto bytes = [&](long long stride, long long n) { return (cuuint64_t)(n > 1 ? stride * size : (d * size + 15) / 16 * 16); };
    const cuuint64_t strides[3] = {bytes(o.stride[2], heads), bytes(o.stride[1], a.L), bytes(o.stride[0], a.B)};
    const cuuint32_t box[4] = {(cuuint32_t)(128 / size), 1, kPiece, 1}, unit[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = dtype == PSIG_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                     : dtype == PSIG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    auto call = [&] {
        return encoder()(map, type, 4, const_cast<void *>(o.data), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    if (call() == CUDA_SUCCESS) return true;
    // a thread that has made no runtime call yet (autograd's) has no current context, which the driver call wants
    int device = 0;
    return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && call() == CUDA_SUCCESS;
}

inline int chain_states(const Sweep &a, long long per_part, cudaStream_t stream)
{
    if (a.splits < 3) return PSIG_OK;
    chain_split_states<<<dim3((unsigned)(a.B * a.H), (unsigned)((per_part + 255) / 256)), 256, 0, stream>>>(
        a.split_states, a.split_decays, a.splits, per_part, a.splits);
    return check_launch();
}

bool operand_fits(const SweepOperand &o, const Sweep &a, int d, int size)
{
    const int unit = 16 / size;   // TMA wants 16-byte addresses, strides and rows
    if (d % unit != 0 || (reinterpret_cast<uintptr_t>(o.data) & 15) != 0) return false;
    const long long sizes[3] = {a.B, a.L, a.H / o.share};
    for (int i = 0; i < 3; ++i)
        if (sizes[i] > 1 && (o.stride[i] <= 0 || o.stride[i] % unit != 0 || o.stride[i] >= (1LL << 37))) return false;
    return true;
}

}  // namespace
}  // namespace psig
