// What the sequence operators (decayed linear attention, norm around a block) share: scalar types, the
// description of one sweep over the time axis, and the checks of the C entry points (internal header).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace psig {

// Type of sums, states and parameters next to a storage type: 32 bits, 64 for float64.
template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };

template <typename A> __device__ __forceinline__ A to_acc(float v) { return (A)v; }
template <typename A> __device__ __forceinline__ A to_acc(double v) { return (A)v; }
template <typename A> __device__ __forceinline__ A to_acc(__nv_bfloat16 v) { return (A)__bfloat162float(v); }
template <typename A> __device__ __forceinline__ A to_acc(__half v) { return (A)__half2float(v); }

template <typename T> __device__ __forceinline__ T from_acc(float v) { return (T)v; }
template <typename T> __device__ __forceinline__ T from_acc(double v) { return (T)v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_acc<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float exp_acc(float v) { return expf(v); }
__device__ __forceinline__ double exp_acc(double v) { return exp(v); }

// Limits of a wait for an mbarrier: this many polls (each of which may sleep for a time that the hardware sets), and about this
// many nanoseconds, looked at every 64 polls.
constexpr unsigned kWaitPolls = 1u << 22;
constexpr unsigned long long kWaitTime = 2000000000ull;
__device__ __forceinline__ bool wait_expired(unsigned poll, unsigned long long &start)
{
    if ((poll & 63) != 63) return false;
    unsigned long long now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (start == 0) start = now;
    return now - start > kWaitTime;
}

// Where the host sees that a wait ran out (psig_set_sequence_failure_flag), or NULL.
int *failure_flag();
__device__ __forceinline__ void report_failure(int *flag)
{
    if (flag == nullptr) return;
    *reinterpret_cast<volatile int *>(flag) = 1;
    __threadfence_system();
}

// Calls fn.template operator()<T>() with the storage type of a PsigDtype.
template <typename Fn>
int with_dtype(int dtype, Fn fn)
{
    switch (dtype) {
        case PSIG_F32: return fn(float{});
        case PSIG_F64: return fn(double{});
        case PSIG_BF16: return fn(__nv_bfloat16{});
        case PSIG_F16: return fn(__half{});
        default: return PSIG_ERR_DTYPE;
    }
}

// One sweep over the time axis, the shape that the forward pass and the three gradients share.  With weights
// w(t, s) = exp(sum of the decays of the steps from s to t), S held per (sequence, head) with shape (d1, d2):
//     out_t = out_scale * ( sum_{s before or at t} w(t, s) kv_scale (r_t . k_s) v_s + w(t, start) r_t^T init )
// "before" is earlier, or later when `reverse` is set.
//     forward:  r = q,  k = k,  v = v,  init = initial_state                  (d1, d2) = (dk, dv)
//     grad_q:   r = go, k = v,  v = k,  init = initial_state^T                (d1, d2) = (dv, dk)
//     grad_k:   r = v,  k = go, v = q,  init = grad_state^T, reverse          (d1, d2) = (dv, dk)
//     grad_v:   r = k,  k = q,  v = go, init = grad_state,   reverse          (d1, d2) = (dk, dv)
struct SweepOperand {
    const void *data;
    long long stride[3];  // elements, for (b, t, head)
    int share;            // sweep heads per operand head
};

constexpr int kSegment = 512;  // time steps between two kept states of the decay gradient

struct Sweep {
    SweepOperand r, k, v;
    const void *decay;
    long long decay_stride[3];
    const int *lengths;
    long long B, L;
    int H, d1, d2;
    bool reverse;
    double out_scale, kv_scale;
    const void *init;     // (B, H, d1, d2), or (B, H, d2, d1) when transposed; NULL: zeros
    bool init_transposed;
    void *final;          // same, or NULL
    bool final_transposed;
    void *out;            // (B, L, H, d2): storage type, or the type of sums when out_acc is set
    bool out_acc;
    // Decay gradient (see attn_decay_grad): the grad_q sweep stores the state at the end of every kSegment steps,
    // the grad_k sweep multiplies its own state into it and leaves one number per segment and column tile.
    void *anchors;        // (B, H, segments, d1, d2); the tensor-core forms keep them in an order of their own
    bool keep_last;       // whether the state behind the last step counts (there is a grad_state)
    void *anchor_dots;    // (B, H, segments, parts of the sum)
    // Tensor-core sweeps only: the unrounded output row times the row of a third operand, summed over each block's and
    // each warp's columns: (attn_tile_dots * column tiles of 64, B, L, H).
    SweepOperand dot;
    float *dots;
    // Tensor-core sweeps of few long sequences: parts of a sequence (see split_plan), and the scratch for their states
    // (B, H, splits, tiles of 64 by 64) and decays (B, H, splits).
    int splits;
    float *split_states, *split_decays;
    int *failure;         // see failure_flag
};

inline int tile_columns(int d2) { return (d2 + 63) / 64; }
inline long long split_state_size(int d1, int d2) { return 4096LL * tile_columns(d1) * tile_columns(d2); }

// Parts to cut each sequence into.  A block sweeps one column tile of one head, so few long sequences leave most of the 148 SMs
// idle.  The first launch over the parts costs about half a sweep, so two parts pay already (32-bit sequences 132 -> 105 us); a
// part is at least four pieces long.  (16 heads of 128, 16384 steps: 412 us in one part, 62 + 3 + 123 us in four.)
inline int split_plan(long long B, long long L, int H, int d2)
{
    const long long blocks = B * H * tile_columns(d2), pieces = (L + 127) / 128;
    if (blocks == 0 || blocks * 2 > 148) return 1;
    long long splits = 148 / blocks;
    if (splits > pieces / 4) splits = pieces / 4;
    if (splits > 64) splits = 64;
    return splits < 2 ? 1 : (int)splits;
}

inline long long segments_of(long long L) { return (L + kSegment - 1) / kSegment; }

// Tensor-core form of the sweep (linear_attention_tiles.cu).  `exact`: results are good to 32 bits, not only to the
// storage type.
bool attn_tiles_supported(const Sweep &a, int dtype);
int attn_sweep_on_tiles(const Sweep &a, bool exact, int dtype, cudaStream_t stream);
int attn_sweep_split(const Sweep &a, bool exact, int dtype, cudaStream_t stream);   // float16 and float32
long long attn_tile_timeouts();
long long attn_split_timeouts();
long long norm_timeouts();
inline int attn_tile_dots(int dtype) { return dtype == PSIG_BF16 ? 1 : 2; }   // at most 2
constexpr int kTileDots = 8;   // parts of an anchor's sum per column tile of 64

}  // namespace psig
