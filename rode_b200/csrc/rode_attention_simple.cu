// Attention on the window-and-sinks and shared-prefix patterns by fused multiply-adds in 32 bits: every type and every head
// dimension that is a multiple of 4 up to 256.  What 16-bit operands of common shapes run on is in rode_attention_tiles.cu
// and rode_attention_step.cu; single precision stays here, because a tensor core would round its operands to 11 bits.
//
// One pass over the keys with the running maximum m and sum l of the softmax: scores of a tile in base 2 (scale * log2 e
// folded into the queries' products), m' = max(m, max s), the accumulator times 2^(m - m'), plus 2^(s - m') V.
//
// A CTA of 256 threads works on 64 rows x 64 keys (32 x 32 at head dimensions above 128, where the operands' tiles would not fit
// the shared memory; at all of them, cases of fewer tiles than SMs gain 10 to 25 %, larger ones lose up to 16 %); a thread holds 4 x 4 scores and 4 rows x
// dim / 16 columns of the result, so that eight 16-byte loads from shared memory feed 64 FMAs (32 instructions, two at once).  Rows of shared memory are 4
// floats longer than the tile: eight threads that read one column of eight keys hit different banks.  Bound by the loads from shared memory (7600
// wavefronts per block of 64 x 64 x 80, forward) and, in small cases, by the SMs that get two tiles.
#include <algorithm>
#include <type_traits>

#include "rode_attention.cuh"

namespace rode {
namespace {

constexpr int kThreads = 256;

template <int kDim>
constexpr int tile_rows() {
    return kDim <= 128 ? 64 : 32;
}

// rows x kDim floats, columns beyond dim and rows beyond `have` zero.  The loads first, then the stores.
template <typename T, int kDim>
__device__ __forceinline__ void fetch_tile(float *dst, const T *src, long long stride, int have, int dim) {
    constexpr int kQuads = kDim / 4, kLoads = tile_rows<kDim>() * kQuads / kThreads;
    float4 x[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        const int i = threadIdx.x + u * kThreads, r = i / kQuads, c = i % kQuads * 4;
        x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < have && c < dim) x[u] = load4(src + r * stride + c);
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        const int i = threadIdx.x + u * kThreads, r = i / kQuads, c = i % kQuads * 4;
        *reinterpret_cast<float4 *>(dst + r * (kDim + 4) + c) = x[u];
    }
}

__device__ __forceinline__ void load_pairs(const float *p, Pair (&x)[2]) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(p);
    x[0].x = v.x;
    x[1].x = v.y;
}

// acc[i][j] = a[row i] . b[row j] for rows ty * R + i and tx + 16 * j
template <int kDim, int R>
__device__ __forceinline__ void dot_tile(const float *a, const float *b, int dim, float (&acc)[R][R]) {
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    Pair two[R][R];  // sums over even and odd head dimensions
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) two[i][j] = pair_of(0.f, 0.f);
#pragma unroll 2
    for (int d = 0; d < dim; d += 4) {
        Pair x[R][2], y[R][2];
#pragma unroll
        for (int i = 0; i < R; ++i) load_pairs(a + (ty * R + i) * (kDim + 4) + d, x[i]);
#pragma unroll
        for (int j = 0; j < R; ++j) load_pairs(b + (tx + 16 * j) * (kDim + 4) + d, y[j]);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < R; ++j) two[i][j] = fma2(x[i][1], y[j][1], fma2(x[i][0], y[j][0], two[i][j]));
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float even, odd;
            split(two[i][j], even, odd);
            acc[i][j] = even + odd;
        }
}

// acc[i][c] += sum over n of w[ty * R + i][n] * x[n][(tx + 16 * c) * 4 ..]; w has rows of kRows + 4 floats.
// The tile's sum by itself first: one addition to acc per tile, so that the error over many keys grows with the tiles, not with the keys (16,384
// values that all round one way: 2.4e-4 off in one sum, 8e-7 so; head dimensions up to 128 take as long, -2 to +4 %, 256 1 to 7 % longer).
template <int kDim, int R>
__device__ __forceinline__ void weigh_rows(const float *w, const float *x, float4 (&acc)[R][kDim / 64]) {
    constexpr int kRows = tile_rows<kDim>();
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    Pair sum[R][kDim / 64][2];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) sum[i][c][0] = sum[i][c][1] = pair_of(0.f, 0.f);
    for (int n = 0; n < kRows; n += 4) {
        float4 p[R];
#pragma unroll
        for (int i = 0; i < R; ++i) p[i] = *reinterpret_cast<const float4 *>(w + (ty * R + i) * (kRows + 4) + n);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < kDim / 64; ++c) {
                Pair y[2];
                load_pairs(x + (n + u) * (kDim + 4) + (tx + 16 * c) * 4, y);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float weight = reinterpret_cast<const float *>(&p[i])[u];
                    sum[i][c][0] = fma2(pair_of(weight, weight), y[0], sum[i][c][0]);
                    sum[i][c][1] = fma2(pair_of(weight, weight), y[1], sum[i][c][1]);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) {
            Pair *to = reinterpret_cast<Pair *>(&acc[i][c]);
            to[0] = add2(to[0], sum[i][c][0]);
            to[1] = add2(to[1], sum[i][c][1]);
        }
}

// Maximum and sum over the 16 threads that share a row.
__device__ __forceinline__ float row_max(float x) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// The running softmax of one tile's scores: s becomes the weights, which go to `weights` for weigh_rows.
// m + log2 l is -inf for a row that has seen no key (m = -inf, l = 0), and NaN for one whose scores are NaN (l is; m need not be).
template <int kDim, int R>
__device__ __forceinline__ void softmax_tile(float (&s)[R][R], float (&m)[R], float (&l)[R], float4 (&acc)[R][kDim / 64],
                                             float *weights) {
    constexpr int kRows = tile_rows<kDim>();
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float top = s[i][0];
#pragma unroll
        for (int j = 1; j < R; ++j) top = fmaxf(top, s[i][j]);
        const float next = fmaxf(m[i], row_max(top));
        const float base = next == -INFINITY ? 0.f : next;  // a row that has seen no key: all weights 0, not NaN
        const float keep = exp2f(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            s[i][j] = exp2f(s[i][j] - base);
            sum += s[i][j];
            weights[(ty * R + i) * (kRows + 4) + tx + 16 * j] = s[i][j];
        }
        l[i] = l[i] * keep + row_sum(sum);
        m[i] = next;
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) {
            acc[i][c].x *= keep;
            acc[i][c].y *= keep;
            acc[i][c].z *= keep;
            acc[i][c].w *= keep;
        }
    }
}

template <int kDim>
constexpr int forward_shared() {
    return 4 * (2 * tile_rows<kDim>() * (kDim + 4) + tile_rows<kDim>() * (tile_rows<kDim>() + 4));
}

// One tile of a sequence's queries, one head.
template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 2) prompt_rows(Prompt p) {
    constexpr int kRows = tile_rows<kDim>(), R = kRows / 16;
    extern __shared__ float4 shared4[];
    float *qs = reinterpret_cast<float *>(shared4), *ks = qs + kRows * (kDim + 4), *vs = ks, *ws = ks + kRows * (kDim + 4);
    const Window &w = p.win;
    const int head = blockIdx.y, kv = head / (w.heads / w.kv_heads);
    const Tile t = find_tile(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, blockIdx.x, kRows);
    if (t.first < 0 || t.first >= t.rows || (t.seq < 0 && !p.clear)) return;
    const int2 keys = t.seq < 0 ? make_int2(0, 0) : sequence_rows(p.seqs.k_offsets, p.seqs.k_rows, t.seq);
    const int have = min(kRows, t.rows - t.first);
    const long long row0 = static_cast<long long>(t.row0) + t.first;
    const int pos0 = t.first + keys.y - t.rows;  // position of the tile's first query
    fetch_tile<T, kDim>(qs, row_of<T>(p.q, 0, row0, head), p.q.row, have, w.dim);

    float m[R], l[R];
    float4 acc[R][kDim / 64];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const KeyBlocks blocks(pos0, pos0 + have, w.window, w.sinks, kRows);
    for (int b = 0; b < blocks.n; ++b) {
        const int k0 = blocks.at(b) * kRows, n = min(kRows, keys.y - k0);
        __syncthreads();
        fetch_tile<T, kDim>(ks, row_of<T>(p.k, 0, keys.x + k0, kv), p.k.row, n, w.dim);
        __syncthreads();
        float s[R][R];
        dot_tile<kDim, R>(qs, ks, w.dim, s);
        __syncthreads();
        fetch_tile<T, kDim>(vs, row_of<T>(p.v, 0, keys.x + k0, kv), p.v.row, n, w.dim);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < R; ++j)
                s[i][j] = sees(pos0 + ty * R + i, k0 + tx + 16 * j, w.window, w.sinks) ? s[i][j] * (w.scale * kLog2e) : -INFINITY;
        softmax_tile<kDim, R>(s, m, l, acc, ws);
        __syncthreads();
        weigh_rows<kDim, R>(ws, vs, acc);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = ty * R + i;
        if (r >= have) continue;
        const float inv = l[i] > 0.f || l[i] != l[i] ? 1.f / l[i] : 0.f;
        T *out = static_cast<T *>(p.out) + ((row0 + r) * w.heads + head) * w.dim;
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) {
            const int d = (tx + 16 * c) * 4;
            if (d >= w.dim) continue;
            const float4 x = make_float4(acc[i][c].x * inv, acc[i][c].y * inv, acc[i][c].z * inv, acc[i][c].w * inv);
            store4(out + d, x);
            if (p.rest != nullptr)
                store4(static_cast<T *>(p.rest) + ((row0 + r) * w.heads + head) * w.dim + d,
                       make_float4(x.x - to_float(from_float<T>(x.x)), x.y - to_float(from_float<T>(x.y)),
                                   x.z - to_float(from_float<T>(x.z)), x.w - to_float(from_float<T>(x.w))));
        }
        if (tx == 0 && p.lse != nullptr)
            p.lse[static_cast<long long>(head) * p.seqs.q_rows + row0 + r] = (m[i] + log2f(l[i])) * kLn2;
    }
}

// Queries of all requests that share a key head, row r = request r / group, head r % group of the group, against a part of the prefix.
template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 2) shared_rows(Cached c) {
    constexpr int kRows = tile_rows<kDim>(), R = kRows / 16;
    extern __shared__ float4 shared4[];
    float *qs = reinterpret_cast<float *>(shared4), *ks = qs + kRows * (kDim + 4), *vs = ks, *ws = ks + kRows * (kDim + 4);
    chain_begin();  // the requests' own keys are worked on beside the prefix
    const Window &w = c.win;
    const int kv = blockIdx.y, group = w.heads / w.kv_heads, split = blockIdx.z;
    const int row0 = blockIdx.x * kRows, have = min(kRows, c.batch * group - row0);
    for (int i = threadIdx.x; i < kRows * (kDim / 4); i += kThreads) {
        const int r = i / (kDim / 4), d = i % (kDim / 4) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < have && d < w.dim) x = load4(row_of<T>(c.q, (row0 + r) / group, 0, kv * group + (row0 + r) % group) + d);
        *reinterpret_cast<float4 *>(qs + r * (kDim + 4) + d) = x;
    }
    float m[R], l[R];
    float4 acc[R][kDim / 64];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < kDim / 64; ++d) acc[i][d] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int blocks = (c.prefix + kRows - 1) / kRows;
    const int b1 = static_cast<int>(static_cast<long long>(blocks) * (split + 1) / c.prefix_parts);
    for (int b = static_cast<int>(static_cast<long long>(blocks) * split / c.prefix_parts); b < b1; ++b) {
        const int k0 = b * kRows, n = min(kRows, c.prefix - k0);
        __syncthreads();
        fetch_tile<T, kDim>(ks, row_of<T>(c.pk, 0, k0, kv), c.pk.row, n, w.dim);
        __syncthreads();
        float s[R][R];
        dot_tile<kDim, R>(qs, ks, w.dim, s);
        __syncthreads();
        fetch_tile<T, kDim>(vs, row_of<T>(c.pv, 0, k0, kv), c.pv.row, n, w.dim);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < R; ++j) s[i][j] = tx + 16 * j < n ? s[i][j] * (w.scale * kLog2e) : -INFINITY;
        softmax_tile<kDim, R>(s, m, l, acc, ws);
        __syncthreads();
        weigh_rows<kDim, R>(ws, vs, acc);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = row0 + ty * R + i;
        if (ty * R + i >= have) continue;
        const float inv = l[i] > 0.f || l[i] != l[i] ? 1.f / l[i] : 0.f;
        const long long at = (static_cast<long long>(split) * c.batch + r / group) * w.heads + kv * group + r % group;
#pragma unroll
        for (int d4 = 0; d4 < kDim / 64; ++d4) {
            const int d = (tx + 16 * d4) * 4;
            if (d < w.dim)
                store4(c.prefix_out + at * w.dim + d,
                       make_float4(acc[i][d4].x * inv, acc[i][d4].y * inv, acc[i][d4].z * inv, acc[i][d4].w * inv));
        }
        if (tx == 0) c.prefix_lse[at] = m[i] + log2f(l[i]);
    }
}

template <int kDim>
constexpr int backward_shared() {
    return 4 * (4 * tile_rows<kDim>() * (kDim + 4) + 2 * tile_rows<kDim>() * (tile_rows<kDim>() + 4) + 2 * tile_rows<kDim>());
}

// Base-2 logarithm of a row's sum of weights, for the weights 2^(s - it).  -inf (all visible scores were -inf, if there were any) as 0, for the weights to
// be 0 then, not 2^(-inf + inf).
__device__ __forceinline__ float sum_log2(float lse) { return lse == -INFINITY ? 0.f : lse * kLog2e; }

// Weights P and score gradients dS = P (dP - delta) of a tile from s = q.k and dp = do.v.
template <int R>
__device__ __forceinline__ void score_gradients(float (&s)[R][R], float (&dp)[R][R], const float *lse2, const float *delta, int pos0,
                                                int have, int k0, const Window &w) {
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int r = ty * R + i;
            const bool on = r < have && sees(pos0 + r, k0 + tx + 16 * j, w.window, w.sinks);
            s[i][j] = on ? exp2f(s[i][j] * (w.scale * kLog2e) - lse2[r]) : 0.f;
            dp[i][j] = on ? s[i][j] * (dp[i][j] - delta[r]) : 0.f;
        }
}

// Gradient of one tile of queries, one head; also delta = do . o of its rows, for key_gradients.
template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads) query_gradients(Prompt p) {
    constexpr int kRows = tile_rows<kDim>(), R = kRows / 16, kTile = kRows * (kDim + 4);
    extern __shared__ float4 shared4[];
    float *qs = reinterpret_cast<float *>(shared4), *gs = qs + kTile, *ks = gs + kTile, *vs = ks + kTile, *ds = vs + kTile,
          *lse2 = ds + 2 * kRows * (kRows + 4), *delta = lse2 + kRows;
    const Window &w = p.win;
    const int head = blockIdx.y, kv = head / (w.heads / w.kv_heads);
    const Tile t = find_tile(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, blockIdx.x, kRows);
    if (t.first < 0 || t.first >= t.rows || (t.seq < 0 && !p.clear)) return;
    const int2 keys = t.seq < 0 ? make_int2(0, 0) : sequence_rows(p.seqs.k_offsets, p.seqs.k_rows, t.seq);
    const int have = min(kRows, t.rows - t.first);
    const long long row0 = static_cast<long long>(t.row0) + t.first;
    const int pos0 = t.first + keys.y - t.rows;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    fetch_tile<T, kDim>(qs, row_of<T>(p.q, 0, row0, head), p.q.row, have, w.dim);
    fetch_tile<T, kDim>(gs, row_of<T>(p.dout, 0, row0, head), p.dout.row, have, w.dim);
    __syncthreads();
    for (int r = ty; r < kRows; r += 16) {
        float sum = 0.f;
        if (r < have) {
            const T *o = static_cast<const T *>(p.out) + ((row0 + r) * w.heads + head) * w.dim;
            for (int d = tx * 4; d < w.dim; d += 64) {
                float4 x = load4(o + d);
                const float4 g = *reinterpret_cast<const float4 *>(gs + r * (kDim + 4) + d);
                if (p.rest != nullptr) vadd(x, load4(static_cast<const T *>(p.rest) + ((row0 + r) * w.heads + head) * w.dim + d));
                sum += x.x * g.x + x.y * g.y + x.z * g.z + x.w * g.w;
            }
        }
        sum = row_sum(sum);
        if (tx == 0) {
            const long long at = static_cast<long long>(head) * p.seqs.q_rows + row0 + r;
            delta[r] = sum;
            lse2[r] = r < have ? sum_log2(p.lse[at]) : 0.f;
            if (r < have) p.delta[at] = sum;
        }
    }
    float4 acc[R][kDim / 64];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    const KeyBlocks blocks(pos0, pos0 + have, w.window, w.sinks, kRows);
    for (int b = 0; b < blocks.n; ++b) {
        const int k0 = blocks.at(b) * kRows, n = min(kRows, keys.y - k0);
        __syncthreads();
        fetch_tile<T, kDim>(ks, row_of<T>(p.k, 0, keys.x + k0, kv), p.k.row, n, w.dim);
        fetch_tile<T, kDim>(vs, row_of<T>(p.v, 0, keys.x + k0, kv), p.v.row, n, w.dim);
        __syncthreads();
        float s[R][R], dp[R][R];
        dot_tile<kDim, R>(qs, ks, w.dim, s);
        dot_tile<kDim, R>(gs, vs, w.dim, dp);
        score_gradients<R>(s, dp, lse2, delta, pos0, have, k0, w);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < R; ++j) ds[(ty * R + i) * (kRows + 4) + tx + 16 * j] = dp[i][j];
        __syncthreads();
        weigh_rows<kDim, R>(ds, ks, acc);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = ty * R + i;
        if (r >= have) continue;
        T *out = static_cast<T *>(p.dq) + ((row0 + r) * w.heads + head) * w.dim;
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) {
            const int d = (tx + 16 * c) * 4;
            if (d < w.dim)
                store4(out + d, make_float4(acc[i][c].x * w.scale, acc[i][c].y * w.scale, acc[i][c].z * w.scale,
                                            acc[i][c].w * w.scale));
        }
    }
}

// Gradients of one tile of keys and values, one key head: the queries of all its heads, one after the other, so that the sum
// over a group has one order.  Or of one query head (p.head_part), where that leaves SMs without work; add_heads adds them up, in order too (1107
// rows of 16 heads on 2 key heads, forward and backward: 1380 us, 333 with the heads apart).
template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads) key_gradients(Prompt p) {
    constexpr int kRows = tile_rows<kDim>(), R = kRows / 16, kTile = kRows * (kDim + 4);
    extern __shared__ float4 shared4[];
    float *qs = reinterpret_cast<float *>(shared4), *gs = qs + kTile, *ks = gs + kTile, *vs = ks + kTile, *pt = vs + kTile,
          *dt = pt + kRows * (kRows + 4), *lse2 = dt + kRows * (kRows + 4), *delta = lse2 + kRows;
    const Window &w = p.win;
    const int group = w.heads / w.kv_heads;
    const bool apart = p.head_part != nullptr;
    const int kv = apart ? blockIdx.y / group : blockIdx.y, h0 = apart ? blockIdx.y : kv * group, h1 = apart ? h0 + 1 : h0 + group;
    const int *offsets = p.seqs.k_offsets;
    const Tile t = find_tile(offsets, p.seqs.n_seq, p.seqs.k_rows, blockIdx.x, kRows);
    if (t.first < 0 || t.first >= t.rows || (t.seq < 0 && !p.clear)) return;
    const int2 queries = t.seq < 0 ? make_int2(0, 0) : sequence_rows(p.seqs.q_offsets, p.seqs.q_rows, t.seq);
    const int have = min(kRows, t.rows - t.first);
    const long long row0 = static_cast<long long>(t.row0) + t.first;
    const int shift = t.rows - queries.y;  // position of the first query
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    fetch_tile<T, kDim>(ks, row_of<T>(p.k, 0, row0, kv), p.k.row, have, w.dim);
    fetch_tile<T, kDim>(vs, row_of<T>(p.v, 0, row0, kv), p.v.row, have, w.dim);
    float4 dk[R][kDim / 64], dv[R][kDim / 64];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) dk[i][c] = dv[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    // queries at positions from the tile's first key to the end of its last key's window (sinks: to the end)
    const int last = t.first < w.sinks || w.window >= t.rows - (t.first + have - 1) ? t.rows : t.first + have - 1 + w.window;
    const int i0 = max(t.first - shift, 0) / kRows * kRows, i1 = min(last - shift, queries.y);
    for (int h = h0; h < h1; ++h)
        for (int i = i0; i < i1; i += kRows) {
            const int n = min(kRows, queries.y - i);
            const long long q0 = static_cast<long long>(queries.x) + i;
            __syncthreads();
            fetch_tile<T, kDim>(qs, row_of<T>(p.q, 0, q0, h), p.q.row, n, w.dim);
            fetch_tile<T, kDim>(gs, row_of<T>(p.dout, 0, q0, h), p.dout.row, n, w.dim);
            if (threadIdx.x < kRows) {
                const long long at = static_cast<long long>(h) * p.seqs.q_rows + q0 + threadIdx.x;
                const bool in = static_cast<int>(threadIdx.x) < n;
                lse2[threadIdx.x] = in ? sum_log2(p.lse[at]) : 0.f;
                delta[threadIdx.x] = in ? p.delta[at] : 0.f;
            }
            __syncthreads();
            float s[R][R], dp[R][R];
            dot_tile<kDim, R>(qs, ks, w.dim, s);
            dot_tile<kDim, R>(gs, vs, w.dim, dp);
            score_gradients<R>(s, dp, lse2, delta, shift + i, n, t.first, w);
#pragma unroll
            for (int a = 0; a < R; ++a)
#pragma unroll
                for (int j = 0; j < R; ++j) {
                    pt[(tx + 16 * j) * (kRows + 4) + ty * R + a] = s[a][j];
                    dt[(tx + 16 * j) * (kRows + 4) + ty * R + a] = dp[a][j];
                }
            __syncthreads();
            weigh_rows<kDim, R>(pt, gs, dv);
            weigh_rows<kDim, R>(dt, qs, dk);
        }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = ty * R + i;
        if (r >= have) continue;
        const long long at = ((row0 + r) * w.kv_heads + kv) * w.dim, part = ((row0 + r) * w.heads + h0) * w.dim;
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) {
            const int d = (tx + 16 * c) * 4;
            if (d >= w.dim) continue;
            if (apart) {
                const long long half = static_cast<long long>(p.seqs.k_rows) * w.heads * w.dim;
                store4(p.head_part + part + d, dk[i][c]);
                store4(p.head_part + half + part + d, dv[i][c]);
                continue;
            }
            store4(static_cast<T *>(p.dk) + at + d,
                   make_float4(dk[i][c].x * w.scale, dk[i][c].y * w.scale, dk[i][c].z * w.scale, dk[i][c].w * w.scale));
            store4(static_cast<T *>(p.dv) + at + d, dv[i][c]);
        }
    }
}

// dK and dV from the parts of the query heads, a thread per four elements.  Rows of no sequence have no parts.
template <typename T>
__global__ void __launch_bounds__(256) add_heads(Prompt p) {
    const Window &w = p.win;
    const int group = w.heads / w.kv_heads, quads = w.dim / 4;
    const long long half = static_cast<long long>(p.seqs.k_rows) * w.heads * w.dim, i = blockIdx.x * 256ll + threadIdx.x;
    if (i >= static_cast<long long>(p.seqs.k_rows) * w.kv_heads * quads) return;
    const int d = static_cast<int>(i % quads) * 4, kv = static_cast<int>(i / quads % w.kv_heads);
    const long long row = i / quads / w.kv_heads;
    if (p.seqs.k_offsets != nullptr && !p.clear &&
        (row < boundary(p.seqs.k_offsets, p.seqs.n_seq, p.seqs.k_rows, 1) ||
         row >= boundary(p.seqs.k_offsets, p.seqs.n_seq, p.seqs.k_rows, p.seqs.n_seq + 1)))
        return;
    float4 dk = make_float4(0.f, 0.f, 0.f, 0.f), dv = dk;
    for (int h = kv * group; h < (kv + 1) * group; ++h) {
        const float *part = p.head_part + (row * w.heads + h) * w.dim + d;
        vadd(dk, *reinterpret_cast<const float4 *>(part));
        vadd(dv, *reinterpret_cast<const float4 *>(part + half));
    }
    const long long at = (row * w.kv_heads + kv) * w.dim + d;
    store4(static_cast<T *>(p.dk) + at, make_float4(dk.x * w.scale, dk.y * w.scale, dk.z * w.scale, dk.w * w.scale));
    store4(static_cast<T *>(p.dv) + at, dv);
}

// --- single tokens -------------------------------------------------------------------------------------------------------------

// Segments of eight heads: the queries of a request and a key head against a part of the keys that they see, 32 at a time.
constexpr int kStepThreads = 128, kStepKeys = 32, kStepQueries = kSimpleChunk;

template <typename T, int kDim>
__global__ void __launch_bounds__(kStepThreads) step_rows(Cached c) {
    constexpr int kQuads = kDim / 4, kGroups = kStepThreads / kQuads, kPer = kStepQueries / kGroups;
    extern __shared__ float4 shared4[];
    float *ks = reinterpret_cast<float *>(shared4), *vs = ks + kStepKeys * (kDim + 4), *qs = vs + kStepKeys * (kDim + 4),
          *ws = qs + kStepQueries * (kDim + 4), *keeps = ws + kStepQueries * kStepKeys, *sums = keeps + kStepQueries,
          *tops = sums + kStepQueries;
    chain_begin();
    const Window &w = c.win;
    const int group = w.heads / w.kv_heads, chunks = (group + kStepQueries - 1) / kStepQueries, per = w.kv_heads * chunks;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int d0 = tid % kQuads * 4, r0 = tid / kQuads * kPer;
    Share share = {0, 0, 0, 0};
    if (!c.whole) share = find_share(c);
    clear_unseen<T>(c);
    int b = c.whole ? blockIdx.x / per : share.request;
    Seen seen = seen_by(c, b);
    int y = c.whole ? blockIdx.x % per : 0;
    long long first = share.first;  // of segment (b, y)
    if (!c.whole && seen.blocks > 0) {
        y = static_cast<int>((share.begin - first) / seen.blocks);
        first += static_cast<long long>(y) * seen.blocks;
    }
    while (c.whole || first < share.end) {
        const int from = c.whole ? 0 : static_cast<int>(max(share.begin - first, 0ll));
        const int to = c.whole ? seen.blocks : static_cast<int>(min(share.end - first, static_cast<long long>(seen.blocks)));
        const int kv = y / chunks, g0 = y % chunks * kStepQueries, have = min(kStepQueries, group - g0), head0 = kv * group + g0;
        __syncthreads();
        for (int i = tid; i < kStepQueries * kQuads; i += kStepThreads) {
            const int r = i / kQuads, d = i % kQuads * 4;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < have && d < w.dim) x = load4(row_of<T>(c.q, b, 0, head0 + r) + d);
            *reinterpret_cast<float4 *>(qs + r * (kDim + 4) + d) = x;
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // of queries 2 * warp and 2 * warp + 1, in every lane
        float4 acc[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = from; i < to; i += 2) {  // two blocks of 16 keys
            __syncthreads();
            for (int x = tid; x < kStepKeys * kQuads; x += kStepThreads) {
                const int r = x / kQuads, d = x % kQuads * 4, block = i + r / 16;
                const int j = seen.first_of(block) + r % 16;
                float4 key = make_float4(0.f, 0.f, 0.f, 0.f), value = key;
                if (block < to && j < seen.end_of(block) && d < w.dim) {
                    key = load4(row_of<T>(c.k, b, j, kv) + d);
                    value = load4(row_of<T>(c.v, b, j, kv) + d);
                }
                *reinterpret_cast<float4 *>(ks + r * (kDim + 4) + d) = key;
                *reinterpret_cast<float4 *>(vs + r * (kDim + 4) + d) = value;
            }
            __syncthreads();
            {
                const int key = tid / 4, r = tid % 4 * 2;
                float s0 = 0.f, s1 = 0.f;
                for (int d = 0; d < w.dim; d += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(ks + key * (kDim + 4) + d);
                    const float4 p = *reinterpret_cast<const float4 *>(qs + r * (kDim + 4) + d);
                    const float4 z = *reinterpret_cast<const float4 *>(qs + (r + 1) * (kDim + 4) + d);
                    s0 = fmaf(x.x, p.x, fmaf(x.y, p.y, fmaf(x.z, p.z, fmaf(x.w, p.w, s0))));
                    s1 = fmaf(x.x, z.x, fmaf(x.y, z.y, fmaf(x.z, z.z, fmaf(x.w, z.w, s1))));
                }
                const int block = i + key / 16;
                const bool in = block < to && seen.first_of(block) + key % 16 < seen.end_of(block);
                ws[r * kStepKeys + key] = in ? s0 * (w.scale * kLog2e) : -INFINITY;
                ws[(r + 1) * kStepKeys + key] = in ? s1 * (w.scale * kLog2e) : -INFINITY;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = 2 * warp + u;
                const float s = ws[r * kStepKeys + lane];
                float top = s;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float next = fmaxf(m[u], top), base = next == -INFINITY ? 0.f : next;
                const float keep = exp2f(m[u] - base), e = exp2f(s - base);
                float sum = e;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                l[u] = l[u] * keep + sum;
                m[u] = next;
                ws[r * kStepKeys + lane] = e;
                if (lane == 0) keeps[r] = keep;
            }
            __syncthreads();
#pragma unroll
            for (int x = 0; x < kPer; ++x) {
                const float keep = keeps[r0 + x];
                acc[x].x *= keep;
                acc[x].y *= keep;
                acc[x].z *= keep;
                acc[x].w *= keep;
            }
            float4 sum[kPer];  // of these keys by themselves, as in weigh_rows
#pragma unroll
            for (int x = 0; x < kPer; ++x) sum[x] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int key = 0; key < kStepKeys; ++key) {
                const float4 value = *reinterpret_cast<const float4 *>(vs + key * (kDim + 4) + d0);
#pragma unroll
                for (int x = 0; x < kPer; ++x) vfma(sum[x], ws[(r0 + x) * kStepKeys + key], value);
            }
#pragma unroll
            for (int x = 0; x < kPer; ++x) vadd(acc[x], sum[x]);
        }
        if (lane == 0) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                sums[2 * warp + u] = l[u];
                tops[2 * warp + u] = m[u];
            }
        }
        __syncthreads();
        const StepResult result(c, b, head0, from == 0 && to == seen.blocks, first < share.begin || c.whole);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int r = r0 + i;
            if (r >= have || d0 >= w.dim) continue;
            const float inv = sums[r] > 0.f || sums[r] != sums[r] ? 1.f / sums[r] : 0.f;
            result.store<T>(c, r, d0, make_float4(acc[i].x * inv, acc[i].y * inv, acc[i].z * inv, acc[i].w * inv));
            if (d0 == 0) result.store_lse(r, tops[r] + log2f(sums[r]));
        }
        if (c.whole) break;
        first += seen.blocks;
        if (++y == per) {
            y = 0;
            do {
                if (first >= share.end || ++b >= c.batch) break;
                seen = seen_by(c, b);
            } while (seen.blocks == 0);
        }
    }
    if (blockIdx.x == 0) chain_wait();  // this grid is not complete before the prefix is
}

template <int kDim>
constexpr int step_shared() {
    return 4 * ((2 * kStepKeys + kStepQueries) * (kDim + 4) + kStepQueries * kStepKeys + 3 * kStepQueries);
}

// Result of one row from its parts, by all 128 threads: weights 2^(lse - max lse), the warps take the parts in turn.  lse_of(s) and part_of(s, d):
// part s's base-2 logarithm and its columns d .. d + 3.
template <typename T, typename Lse, typename Part>
__device__ __forceinline__ void join_parts_of_row(T *out, int dim, int parts, Lse &&lse_of, Part &&part_of) {
    __shared__ float4 joined[4][64];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    float top = -INFINITY, sum = 0.f;
    for (int s = lane; s < parts; s += 32) top = fmaxf(top, lse_of(s));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.f;
    for (int s = lane; s < parts; s += 32) sum += exp2f(lse_of(s) - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    for (int d = lane * 4; d < dim; d += 128) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = warp; s < parts; s += 4) {
            const float x = exp2f(lse_of(s) - top);
            const float4 part = part_of(s, d);
            // (a part without keys has no weight, whatever its rows hold)
            if (x != 0.f) vfma(acc, x * inv, part);
        }
        joined[warp][d / 4] = acc;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < dim / 4; d += 128) {
        float4 acc = joined[0][d];
#pragma unroll
        for (int u = 1; u < 4; ++u) vadd(acc, joined[u][d]);
        store4(out + d * 4, acc);
    }
    __syncthreads();
}

// Segments in pieces, without a prefix: CTA (x, r) has head r of the segment that begins in share x and goes on behind it.  (A CTA per row of
// the result, most of which have no pieces, took 13 us behind step_batch.)
template <typename T>
__global__ void __launch_bounds__(128) join_pieces(Cached c) {
    const int group = c.win.heads / c.win.kv_heads, chunks = (group + c.chunk - 1) / c.chunk;
    const Share share = find_share(c, true);
    const float *piece_lse = after_chain(c.piece_lse), *piece_out = after_chain(c.piece_out);
    if (share.begin >= share.end) return;
    const int blocks = seen_by(c, share.request).blocks;
    const int y = static_cast<int>((share.end - 1 - share.first) / blocks);
    const long long begin = share.first + static_cast<long long>(y) * blocks, end = begin + blocks, size = share.end - share.begin;
    if (begin < share.begin || end <= share.end) return;  // another share's, or whole (the last share ends with its segment)
    const int r = blockIdx.y, g = y % chunks * c.chunk + r;
    if (g >= group) return;
    const int parts = 1 + static_cast<int>((end - share.end + size - 1) / size);
    const auto place = [&](int s) { return (2ll * (blockIdx.x + s) + (s == 0)) * c.chunk + r; };
    const int dim = c.win.dim;
    join_parts_of_row(static_cast<T *>(c.out) + (static_cast<long long>(share.request) * c.win.heads + y / chunks * group + g) * dim, dim, parts,
                      [&](int s) { return __ldcg(piece_lse + place(s)); },
                      [&](int s, int d) { return __ldcg(reinterpret_cast<const float4 *>(piece_out + place(s) * dim + d)); });
}

// With a prefix: every row, from the prefix's parts and what its own keys gave, which is one row or some pieces.
template <typename T>
__global__ void __launch_bounds__(128) join_rows(Cached c) {
    __shared__ long long below[4], all[4];
    const long long rows = static_cast<long long>(c.batch) * c.win.heads, row = blockIdx.x;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, dim = c.win.dim;
    const int b = static_cast<int>(row / c.win.heads), head = static_cast<int>(row % c.win.heads), group = c.win.heads / c.win.kv_heads;
    const int in_group = head % group, per = segments_per_request(c), y = head / group * (per / c.win.kv_heads) + in_group / c.chunk;
    // the CTAs that had a part of this row's segment
    int c0 = 0, c1 = 0;
    bool none = false;
    if (!c.whole) {
        long long mine = 0, sum = 0;
        for (int i = threadIdx.x; i < c.batch; i += 128) {
            const int blocks = seen_by(c, i).blocks;
            sum += blocks;
            if (i < b) mine += blocks;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            mine += __shfl_xor_sync(0xffffffffu, mine, o);
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (lane == 0) {
            below[warp] = mine;
            all[warp] = sum;
        }
        __syncthreads();
        const int blocks = seen_by(c, b).blocks;
        const long long begin = (below[0] + below[1] + below[2] + below[3]) * per + static_cast<long long>(y) * blocks;
        const long long share = max(share_of(c, (all[0] + all[1] + all[2] + all[3]) * per), 1ll);
        none = blocks == 0;
        c0 = static_cast<int>(begin / share);
        c1 = none ? c0 : static_cast<int>((begin + blocks - 1) / share);
    }
    const bool pieces = c1 > c0;
    const int parts = c.prefix_parts + (none ? 0 : c1 - c0 + 1);
    // (through the result of the wait: what the grids before this one have written)
    const float *prefix_lse = after_chain(c.prefix_lse), *own_lse = after_chain(c.own_lse), *piece_lse = after_chain(c.piece_lse);
    const float *prefix_out = after_chain(c.prefix_out), *own_out = after_chain(c.own_out), *piece_out = after_chain(c.piece_out);
    const auto place = [&](int s) {  // of part s, in rows of its array
        if (s < c.prefix_parts) return s * rows + row;
        if (!pieces) return row;
        const int i = s - c.prefix_parts;
        return (2ll * (c0 + i) + (i == 0)) * c.chunk + in_group % c.chunk;
    };
    join_parts_of_row(static_cast<T *>(c.out) + row * dim, dim, parts,
                      [&](int s) { return __ldcg((s < c.prefix_parts ? prefix_lse : pieces ? piece_lse : own_lse) + place(s)); },
                      [&](int s, int d) {
                          const float *from = s < c.prefix_parts ? prefix_out : pieces ? piece_out : own_out;
                          return __ldcg(reinterpret_cast<const float4 *>(from + place(s) * dim + d));
                      });
}

template <typename F>
int by_type(int dtype, F &&f) {
    if (dtype == RODE_F32) return f(static_cast<float *>(nullptr));
    if (dtype == RODE_F16) return f(static_cast<__half *>(nullptr));
    return f(static_cast<__nv_bfloat16 *>(nullptr));
}
template <typename F>
int by_dim(int dim, F &&f) {
    if (dim <= 64) return f(std::integral_constant<int, 64>());
    if (dim <= 128) return f(std::integral_constant<int, 128>());
    return f(std::integral_constant<int, 256>());
}

}  // namespace

int simple_prompt(int dtype, const Prompt &p, cudaStream_t stream) {
    return by_type(dtype, [&](auto *type) {
        return by_dim(p.win.dim, [&](auto dim) {
            using T = std::remove_pointer_t<decltype(type)>;
            constexpr int kDim = decltype(dim)::value;
            auto *kernel = &prompt_rows<T, kDim>;
            if (const int e = allow_shared(kernel, forward_shared<kDim>())) return e;
            const int slots = tile_slots(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, tile_rows<kDim>());
            kernel<<<dim3(slots, p.win.heads), kThreads, forward_shared<kDim>(), stream>>>(p);
            RODE_CHECK_LAUNCH("prompt_rows");
            return static_cast<int>(RODE_OK);
        });
    });
}

int simple_prompt_backward(int dtype, const Prompt &p, cudaStream_t stream) {
    return by_type(dtype, [&](auto *type) {
        return by_dim(p.win.dim, [&](auto dim) {
            using T = std::remove_pointer_t<decltype(type)>;
            constexpr int kDim = decltype(dim)::value;
            auto *kernel = &query_gradients<T, kDim>;
            auto *kernel2 = &key_gradients<T, kDim>;
            if (const int e = allow_shared(kernel, backward_shared<kDim>())) return e;
            if (const int e = allow_shared(kernel2, backward_shared<kDim>())) return e;
            const int slots = tile_slots(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, tile_rows<kDim>());
            if (slots > 0) kernel<<<dim3(slots, p.win.heads), kThreads, backward_shared<kDim>(), stream>>>(p);
            RODE_CHECK_LAUNCH("query_gradients");
            const int k_slots = tile_slots(p.seqs.k_offsets, p.seqs.n_seq, p.seqs.k_rows, tile_rows<kDim>());
            if (p.dk == nullptr || k_slots == 0) return static_cast<int>(RODE_OK);
            kernel2<<<dim3(k_slots, p.head_part ? p.win.heads : p.win.kv_heads), kThreads, backward_shared<kDim>(), stream>>>(p);
            RODE_CHECK_LAUNCH("key_gradients");
            if (p.head_part != nullptr) {
                const long long threads = static_cast<long long>(p.seqs.k_rows) * p.win.kv_heads * (p.win.dim / 4);
                add_heads<T><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, stream>>>(p);
                RODE_CHECK_LAUNCH("add_heads");
            }
            return static_cast<int>(RODE_OK);
        });
    });
}

// Apart where the tiles of keys and key heads fill less than half of the SMs.
size_t simple_backward_bytes(int dtype, int n_seq, int k_rows, int heads, int kv_heads, int dim) {
    if (dtype != RODE_F32 || heads == kv_heads) return 0;
    const int rows = dim <= 128 ? tile_rows<128>() : tile_rows<256>();
    const long long tiles = (static_cast<long long>(k_rows) + rows - 1) / rows + n_seq;
    return tiles * kv_heads * 2 > sm_count() ? 0 : 2 * sizeof(float) * k_rows * heads * dim;
}

int simple_shared(int dtype, const Cached &c, cudaStream_t stream) {
    return by_type(dtype, [&](auto *type) {
        return by_dim(c.win.dim, [&](auto dim) {
            using T = std::remove_pointer_t<decltype(type)>;
            constexpr int kDim = decltype(dim)::value;
            auto *kernel = &shared_rows<T, kDim>;
            if (const int e = allow_shared(kernel, forward_shared<kDim>())) return e;
            const long long rows = static_cast<long long>(c.batch) * (c.win.heads / c.win.kv_heads);
            const int tiles = static_cast<int>((rows + tile_rows<kDim>() - 1) / tile_rows<kDim>());
            kernel<<<dim3(tiles, c.win.kv_heads, c.prefix_parts), kThreads, forward_shared<kDim>(), stream>>>(c);
            RODE_CHECK_LAUNCH("shared_rows");
            return static_cast<int>(RODE_OK);
        });
    });
}

int simple_step(int dtype, const Cached &c, cudaStream_t stream) {
    return by_type(dtype, [&](auto *type) {
        return by_dim(c.win.dim, [&](auto dim) {
            using T = std::remove_pointer_t<decltype(type)>;
            constexpr int kDim = decltype(dim)::value;
            auto *kernel = &step_rows<T, kDim>;
            if (const int e = allow_shared(kernel, step_shared<kDim>())) return e;
            RODE_CUDA_TRY(launch_part(kernel, dim3(c.ctas), kStepThreads, step_shared<kDim>(), stream, c.prefix_parts > 0, c));
            return static_cast<int>(RODE_OK);
        });
    });
}

int join_parts(int dtype, const Cached &c, cudaStream_t stream) {
    return by_type(dtype, [&](auto *type) {
        using T = std::remove_pointer_t<decltype(type)>;
        const long long rows = static_cast<long long>(c.batch) * c.win.heads;
        if (c.prefix_parts > 0)
            RODE_CUDA_TRY(launch_part(&join_rows<T>, dim3(static_cast<unsigned>(rows)), 128, 0, stream, true, c));
        else
            RODE_CUDA_TRY(launch_part(&join_pieces<T>, dim3(c.ctas, std::min(c.chunk, c.win.heads / c.win.kv_heads)), 128, 0, stream, true, c));
        return static_cast<int>(RODE_OK);
    });
}

}  // namespace rode
