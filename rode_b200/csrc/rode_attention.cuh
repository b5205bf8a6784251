// Shared parts of the attention kernels: operands, packed sequences, which keys a query sees.
//
// Query i of a sequence with nq queries and nk keys stands at position p = i + nk - nq (the queries are the last nq positions).
// It sees key j when j <= p and either j > p - window or j < sinks.
//
// Times beside the kernels are of the cases of perf/operators.py that they name, in us a pass or a kernel.
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
    void *rest;  // what rounding took from out, in the same type; may be null
    float *lse;
    void *dq, *dk, *dv;
    float *delta;
    // Chunks of the queries that see sinks only (key_gradient_tiles); far_slots == 0: none
    int far_chunk, far_slots;
    float *near_part, *far_part;
    float *head_part;  // fp32 sums of dK and dV by query head, [2, k_rows, heads, dim] (key_gradients); null: not apart
    bool clear;  // rows of no sequence become zero (else they are left as they were)
};

// One query per request against its cache and, if prefix > 0, against keys that all requests share.
//
// The work on the caches is a list of segments, (request, key head, chunk of the heads of its group), each with as many blocks of 16 keys as its request
// sees.  `whole`: one CTA per segment.  Else all blocks, segment by segment, are dealt out to `ctas` CTAs in equal shares, whatever the
// lengths are: a CTA works on the end of one segment, on whole ones, on the beginning of another.  What a CTA has of a segment that it shares with others is a
// piece: 2 * cta for the first segment of its share, 2 * cta + 1 for the last one.
constexpr int kTensorCoreChunk = 16, kSimpleChunk = 8;  // heads of a segment
struct Cached {
    int batch, capacity, prefix;
    Window win;
    rode_heads_t q, k, v, pk, pv;
    const int *lengths;
    void *out;
    int chunk;  // heads of a segment
    bool whole;
    int ctas;
    // Partial results, normalised, and the base-2 logarithms of their sums.  Prefix: [prefix_parts, batch, heads, dim] and without dim.  Own
    // keys, if there is a prefix to join them with: [batch, heads, dim] of segments that one CTA had.  Pieces: [2 ctas, chunk, dim].
    int prefix_parts;
    float *prefix_out, *prefix_lse, *own_out, *own_lse, *piece_out, *piece_lse;
};

int simple_prompt(int dtype, const Prompt &p, cudaStream_t stream);
int simple_prompt_backward(int dtype, const Prompt &p, cudaStream_t stream);
int simple_shared(int dtype, const Cached &c, cudaStream_t stream);
int simple_step(int dtype, const Cached &c, cudaStream_t stream);

// On the tensor cores, where *_take_* says so.
bool tiles_take_prompt(int dtype, const Prompt &p);
bool tiles_take_shared(int dtype, const Cached &c);
int tiles_prompt(int dtype, const Prompt &p, cudaStream_t stream);
bool tiles_take_backward(int dtype, const Prompt &p);
struct FarPlan {
    int chunk, slots;
    size_t near_bytes, far_bytes;
};
// Bytes of Prompt::head_part, 0 where the heads of a group need not be apart.
size_t simple_backward_bytes(int dtype, int n_seq, int k_rows, int heads, int kv_heads, int dim);
FarPlan plan_far(int n_seq, bool packed, int q_rows, int kv_heads, int dim, int window, int sinks);
int tiles_backward(int dtype, const Prompt &p, cudaStream_t stream);
int tiles_shared(int dtype, const Cached &c, cudaStream_t stream);
bool step_takes(int dtype, const Cached &c);
int step_on_tensor_cores(int dtype, const Cached &c, cudaStream_t stream);
int tiles_waits_failed(int *failed);

int join_parts(int dtype, const Cached &c, cudaStream_t stream);

#ifdef __CUDACC__

// Two numbers in one 64-bit register: one instruction for both.
struct Pair {
    unsigned long long x;
};
__device__ __forceinline__ Pair pair_of(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.x) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(Pair p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.x)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.x) : "l"(a.x), "l"(b.x), "l"(c.x));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.x) : "l"(a.x), "l"(b.x));
    return r;
}

__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.x) : "l"(a.x), "l"(b.x));
    return r;
}
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

// By whole warps: 32 offsets are looked at at once.
__device__ __forceinline__ Tile find_tile(const int *offsets, int n_seq, int total, int slot, int tile) {
    if (offsets == nullptr) return {0, 0, total, slot * tile};
    int lo = 0, hi = n_seq + 2;  // the answer is in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, e = lo + static_cast<int>(threadIdx.x % 32) * step;
        const bool below = e < hi && boundary(offsets, n_seq, total, e) / tile + e <= slot;
        // (offsets that are out of order may leave holes: the lanes up to the first one count)
        const unsigned votes = __ballot_sync(0xffffffffu, below) | 1u;
        const int n = votes == 0xffffffffu ? 32 : __ffs(~votes) - 1;
        lo += (n - 1) * step;
        hi = min(lo + step, hi);
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

// Keys that the query of request b sees: those of the sinks, [0, sinks), and of the window, [lo, n); blocks of 16 of each.
struct Seen {
    int n, lo, sinks, sink_blocks, blocks;
    __device__ __forceinline__ int first_of(int i) const { return i < sink_blocks ? i * 16 : lo + (i - sink_blocks) * 16; }
    __device__ __forceinline__ int end_of(int i) const { return i < sink_blocks ? sinks : n; }
};
__device__ __forceinline__ Seen seen_by(const Cached &c, int b) {
    Seen s;
    s.n = min(max(__ldg(c.lengths + b), 0), c.capacity);
    s.lo = max(s.n - c.win.window, 0);
    s.sinks = min(c.win.sinks, s.lo);
    s.sink_blocks = (s.sinks + 15) / 16;
    s.blocks = s.sink_blocks + (s.n - s.lo + 15) / 16;
    return s;
}
__device__ __forceinline__ int segments_per_request(const Cached &c) {
    const int group = c.win.heads / c.win.kv_heads;
    return c.win.kv_heads * ((group + c.chunk - 1) / c.chunk);
}
// Blocks of a CTA's share.
__device__ __forceinline__ long long share_of(const Cached &c, long long total) { return (total + c.ctas - 1) / c.ctas; }

// Where the share of CTA blockIdx.x begins and ends, in blocks of all segments, and the request that its first (or last) block is in, with that
// request's own first block.  By all 128 threads of a CTA: each adds up a run of requests.
struct Share {
    long long begin, end, first;
    int request;
};
__device__ __forceinline__ Share find_share(const Cached &c, bool last = false) {
    __shared__ long long sums[4];
    __shared__ Share found;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, per = segments_per_request(c);
    const int run = (c.batch + 127) / 128, b0 = min(static_cast<int>(threadIdx.x) * run, c.batch), b1 = min(b0 + run, c.batch);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += seen_by(c, b).blocks;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long before = upto - mine, total = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (u < warp) before += sums[u];
        total += sums[u];
    }
    total *= per;
    before *= per;
    const long long share = share_of(c, total), begin = min(share * blockIdx.x, total), end = min(begin + share, total);
    const long long at = last ? end - 1 : begin;
    if (begin < end && at >= before && at < before + mine * per) {
        int b = b0;
        for (; b < b1; ++b) {
            const long long blocks = static_cast<long long>(seen_by(c, b).blocks) * per;
            if (at < before + blocks) break;
            before += blocks;
        }
        found = {begin, end, before, b};
    }
    __syncthreads();
    return begin < end ? found : Share{0, 0, 0, 0};
}

// Requests that see nothing are in no share: their rows become zero (with a prefix, join_rows does without them).
template <typename T>
__device__ __forceinline__ void clear_unseen(const Cached &c) {
    if (c.whole || c.prefix_parts > 0) return;
    for (int b = blockIdx.x; b < c.batch; b += gridDim.x) {
        if (seen_by(c, b).blocks > 0) continue;
        T *out = static_cast<T *>(c.out) + static_cast<long long>(b) * c.win.heads * c.win.dim;
        for (int i = threadIdx.x * 4; i < c.win.heads * c.win.dim; i += 512) store4(out + i, make_float4(0.f, 0.f, 0.f, 0.f));
    }
}

template <typename T>
__device__ __forceinline__ const T *row_of(const rode_heads_t &x, long long batch, long long row, int head) {
    return static_cast<const T *>(x.data) + batch * x.batch + row * x.row + head * x.head;
}

// Where a CTA's result for a segment goes: to the output, to the rows that are joined with the prefix, or to a piece.
struct StepResult {
    float *lse;
    float *part;
    long long row;  // of the output
    __device__ __forceinline__ StepResult(const Cached &c, int b, int head0, bool all, bool first_of_share) {
        row = static_cast<long long>(b) * c.win.heads + head0;
        lse = nullptr;
        part = nullptr;
        if (!all) {
            const long long piece = (2ll * blockIdx.x + !first_of_share) * c.chunk;
            lse = c.piece_lse + piece;
            part = c.piece_out + piece * c.win.dim;
        } else if (c.prefix_parts > 0) {
            lse = c.own_lse + row;
            part = c.own_out + row * c.win.dim;
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(const Cached &c, int r, int d, float4 x) const {
        if (part != nullptr)
            store4(part + static_cast<long long>(r) * c.win.dim + d, x);
        else
            store4(static_cast<T *>(c.out) + (row + r) * c.win.dim + d, x);
    }
    __device__ __forceinline__ void store_lse(int r, float x) const {
        if (lse != nullptr) lse[r] = x;
    }
};

#endif  // __CUDACC__

// Lets a kernel have `bytes` of dynamic shared memory on the current device.
template <typename K>
int allow_shared(K *kernel, int bytes) {
    RODE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return RODE_OK;
}

// How a kernel of a call on a cache is launched: `chained`, it may start beside the one before it.
template <typename K, typename... A>
cudaError_t launch_part(K *kernel, dim3 grid, int threads, int shared, cudaStream_t stream, bool chained, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = chained ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace rode
