// Shared parts of the attention kernels: operands, packed sequences, which keys a query sees.
//
// Query i of a sequence with nq queries and nk keys stands at position p = i + nk - nq (the queries are the last nq positions).
// It sees key j when j <= p and either j > p - window or j < sinks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "rode_common.cuh"

namespace rode {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Sequences packed along the rows of an operand.  offsets == nullptr: one sequence of all rows.
struct Packed {
    const int *q_offsets;
    const int *k_offsets;
    int n_seq;
    int q_rows;
    int k_rows;
};

struct Window {
    int window;
    int sinks;
    int heads;
    int kv_heads;
    int dim;
    float scale;
};

// Forward and backward of packed sequences.  Strides in elements; the last dimension is contiguous; out, dq, dk and dv are
// contiguous [rows, heads, dim]; lse and delta are [heads, q_rows].
struct Prompt {
    Packed seqs;
    Window win;
    rode_heads_t q, k, v, dout;
    void *out;
    float *lse;
    void *dq, *dk, *dv;
    float *delta;
    // Chunks of the queries that see sinks only (key_gradient_tiles); far_slots == 0: none
    int far_chunk, far_slots;
    float *near_part, *far_part;
    bool clear;  // rows of no sequence become zero (else they are left as they were)
};

// One query per request against its cache and, if prefix > 0, against keys that all requests share.
struct Cached {
    int batch, capacity, prefix;
    Window win;
    rode_heads_t q, k, v, pk, pv;
    const int *lengths;
    void *out;
    // Partial results: [splits, batch, heads, dim] (normalised) and [splits, batch, heads] (base-2 logarithm of the sum)
    float *part_out;
    float *part_lse;
};

int simple_prompt(int dtype, const Prompt &p, cudaStream_t stream);
int simple_prompt_backward(int dtype, const Prompt &p, cudaStream_t stream);
int simple_shared(int dtype, const Cached &c, int first_split, int splits, cudaStream_t stream);
int simple_step(int dtype, const Cached &c, int first_split, int splits, cudaStream_t stream);

// On the tensor cores, where *_take_* says so.
bool tiles_take_prompt(int dtype, const Prompt &p);
bool tiles_take_shared(int dtype, const Cached &c);
int tiles_prompt(int dtype, const Prompt &p, cudaStream_t stream);
bool tiles_take_backward(int dtype, const Prompt &p);
struct FarPlan {
    int chunk, slots;
    size_t near_bytes, far_bytes;
};
FarPlan plan_far(int n_seq, bool packed, int q_rows, int kv_heads, int dim, int window, int sinks);
int tiles_backward(int dtype, const Prompt &p, cudaStream_t stream);
int tiles_shared(int dtype, const Cached &c, int first_split, int splits, cudaStream_t stream);
bool step_takes(int dtype, const Cached &c);
int step_on_tensor_cores(int dtype, const Cached &c, int first_split, int splits, cudaStream_t stream);
int tiles_waits_failed(int *failed);

int join_parts(int dtype, const Cached &c, int splits, cudaStream_t stream);

#ifdef __CUDACC__

// One tile of a sequence.  Boundaries of the sequences, extended by the rows in front of the first and behind the last one, are
// cut into tiles; sequence e's tiles start at slot boundary(e) / tile + e, so that a slot finds its sequence by bisection
// over the offsets and a grid of rows / tile + n_seq + 2 slots covers any lengths, which the host does not know.
struct Tile {
    int seq;    // -1: rows of no sequence
    int row0;   // first row of the sequence in the packed operand
    int rows;   // rows of the sequence
    int first;  // first row of the tile within the sequence; >= rows: nothing to do
};

__device__ __forceinline__ int boundary(const int *offsets, int n_seq, int total, int e) {
    if (e == 0) return 0;
    if (e == n_seq + 2) return total;
    return min(max(__ldg(offsets + e - 1), 0), total);
}

__device__ __forceinline__ Tile find_tile(const int *offsets, int n_seq, int total, int slot, int tile) {
    if (offsets == nullptr) return {0, 0, total, slot * tile};
    int lo = 0, hi = n_seq + 2;  // the answer is in [lo, hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (boundary(offsets, n_seq, total, mid) / tile + mid <= slot)
            lo = mid;
        else
            hi = mid;
    }
    const int begin = boundary(offsets, n_seq, total, lo);
    const int rows = max(boundary(offsets, n_seq, total, lo + 1) - begin, 0);
    const long long first = static_cast<long long>(slot - begin / tile - lo) * tile;
    return {lo == 0 || lo == n_seq + 1 ? -1 : lo - 1, begin, rows, static_cast<int>(min(first, static_cast<long long>(rows)))};
}

inline int tile_slots(const int *offsets, int n_seq, int total, int tile) {
    return offsets == nullptr ? (total + tile - 1) / tile : total / tile + n_seq + 2;
}

// Rows of sequence `seq` of the other operand: where they start, how many.
__device__ __forceinline__ int2 sequence_rows(const int *offsets, int total, int seq) {
    if (offsets == nullptr) return make_int2(0, total);
    const int begin = min(max(__ldg(offsets + seq), 0), total);
    return make_int2(begin, min(max(__ldg(offsets + seq + 1), begin), total) - begin);
}

// Key blocks of `block` keys that queries at positions [p0, p1) see: the blocks of the sinks in front of the window, then those
// of the window.  Block i of count() starts at key at(i).
struct KeyBlocks {
    int n_sink, first, n;
    __device__ __forceinline__ KeyBlocks(int p0, int p1, int window, int sinks, int block) {
        p1 = max(p1, 0);
        const int lo = window > p0 ? 0 : p0 - window + 1;
        n_sink = (min(sinks, lo) + block - 1) / block;
        first = max(lo / block, n_sink);
        n = n_sink + max((p1 + block - 1) / block - first, 0);
    }
    __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : first + i - n_sink; }
};

__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
    return j <= p && (p - j < window || j < sinks);
}

template <typename T>
__device__ __forceinline__ float to_float(T x) {
    return static_cast<float>(x);
}
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// Four elements at once (the operands' strides and the head dimension are multiples of four elements).
template <typename T>
__device__ __forceinline__ float4 load4(const T *p) {
    if constexpr (sizeof(T) == 4) {
        return __ldg(reinterpret_cast<const float4 *>(p));
    } else {
        const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
        const T *t = reinterpret_cast<const T *>(&x);
        return make_float4(to_float(t[0]), to_float(t[1]), to_float(t[2]), to_float(t[3]));
    }
}
template <typename T>
__device__ __forceinline__ void store4(T *p, float4 v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = v;
    } else {
        uint2 x;
        T *t = reinterpret_cast<T *>(&x);
        t[0] = from_float<T>(v.x);
        t[1] = from_float<T>(v.y);
        t[2] = from_float<T>(v.z);
        t[3] = from_float<T>(v.w);
        *reinterpret_cast<uint2 *>(p) = x;
    }
}

template <typename T>
__device__ __forceinline__ const T *row_of(const rode_heads_t &x, long long batch, long long row, int head) {
    return static_cast<const T *>(x.data) + batch * x.batch + row * x.row + head * x.head;
}

#endif  // __CUDACC__

// Lets a kernel have `bytes` of dynamic shared memory on the current device.
template <typename K>
int allow_shared(K *kernel, int bytes) {
    RODE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return RODE_OK;
}

}  // namespace rode
