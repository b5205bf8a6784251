// Single tokens against a cache, 16-bit operands whose rows are whole 16-byte units: bound by the reads of keys and values.
//
// Segments of 16 heads (Cached).  A CTA's four warps take blocks of 16 keys in turn, each with a
// running softmax of its own, joined at the end.  All heads of a group share what is read.  Products by mma.sync m16n8k16 (16 query rows are all
// there are: a tile of 128 rows would be empty in the main, and the products are a tenth of the time of the loads): S = Q K^T with the keys as
// columns, whose accumulator layout is the operand layout of P in O = P V.
//
// Keys and values go from memory straight into the registers of the product, 16 bytes per load, because the order of the summands
// and of the columns is free.  K: lane (c = lane % 4, key = lane / 4) loads head dimensions 32 j + 8 c .. + 7 of its key, which serve as the summands
// {2c, 2c + 1, 2c + 8, 2c + 9} of two products; Q is laid out the same.  V: lane (c, g = lane / 4) loads dimensions 64 j + 8 g .. + 7 of keys 2c, 2c + 1,
// 2c + 8, 2c + 9; the pairs of keys that a product wants in one register come from two byte permutations, and column g of product
// i is dimension 64 j + 8 g + i.  Eight rows of 64 bytes resp. four of 128 per load instruction, no shared memory, no barrier.
// The next block's K is loaded while the softmax runs, the next V behind P V: 4 to 8 KB per warp in flight.
#include <type_traits>

#include "rode_attention.cuh"
#include "rode_tensor_cores.cuh"

namespace rode {
namespace {

constexpr int kWarps = 4, kQueries = kTensorCoreChunk;

template <typename T>
__device__ __forceinline__ void small_product(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Read once: past the L1.
__device__ __forceinline__ uint4 load_once(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kWarps * 32, 2) step_tiles(const Cached c) {
    constexpr int kK = kDim / 32, kV = kDim / 64;
    __shared__ float4 joined[kWarps][kQueries * kDim / 4];
    __shared__ float tops[kWarps][kQueries], sums[kWarps][kQueries];
    chain_begin();
    const Window &w = c.win;
    const int group = w.heads / w.kv_heads, chunks = (group + kQueries - 1) / kQueries, per = w.kv_heads * chunks;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane % 4, row = lane / 4;
    const float s2 = w.scale * kLog2e;
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
        const int begin = c.whole ? 0 : static_cast<int>(max(share.begin - first, 0ll));
        const int end = c.whole ? seen.blocks : static_cast<int>(min(share.end - first, static_cast<long long>(seen.blocks)));
        const int kv = y / chunks, g0 = y % chunks * kQueries, have = min(kQueries, group - g0), head0 = kv * group + g0;

        uint4 q[kK][2];
#pragma unroll
        for (int j = 0; j < kK; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = row + 8 * u, d = 32 * j + 8 * quad;
                q[j][u] = make_uint4(0, 0, 0, 0);
                if (r < have && d < w.dim) q[j][u] = __ldg(reinterpret_cast<const uint4 *>(row_of<T>(c.q, b, 0, head0 + r) + d));
            }
        float o[kV * 8][4];
#pragma unroll
        for (int i = 0; i < kV * 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        const T *keys = row_of<T>(c.k, b, 0, kv) + 8 * quad, *values = row_of<T>(c.v, b, 0, kv) + 8 * row;

        uint4 k[2][kK], v[4][kV];
        // Rows behind the last visible one of their segment are read as that one (it is visible, so it holds what its owner wrote), with
        // weight 0.
        const auto load_keys = [&](int i) {
            const int k0 = seen.first_of(i), last = seen.end_of(i) - 1;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const T *p = keys + min(k0 + 8 * u + row, last) * c.k.row;
#pragma unroll
                for (int j = 0; j < kK; ++j) {
                    k[u][j] = make_uint4(0, 0, 0, 0);
                    if (32 * j + 8 * quad < w.dim) k[u][j] = load_once(p + 32 * j);
                }
            }
        };
        const auto load_values = [&](int i) {
            const int k0 = seen.first_of(i), last = seen.end_of(i) - 1;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const T *p = values + min(k0 + 2 * quad + u % 2 + u / 2 * 8, last) * c.v.row;
#pragma unroll
                for (int j = 0; j < kV; ++j) {
                    v[u][j] = make_uint4(0, 0, 0, 0);
                    if (64 * j + 8 * row < w.dim) v[u][j] = load_once(p + 64 * j);
                }
            }
        };
        int i = begin + warp;
        if (i < end) {
            load_keys(i);
            load_values(i);
        }
        for (; i < end; i += kWarps) {
            float s[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
#pragma unroll
                for (int j = 0; j < kK; ++j) {
                    small_product<T>(s[u], q[j][0].x, q[j][1].x, q[j][0].y, q[j][1].y, k[u][j].x, k[u][j].y);
                    small_product<T>(s[u], q[j][0].z, q[j][1].z, q[j][0].w, q[j][1].w, k[u][j].z, k[u][j].w);
                }
            }
            const bool more = i + kWarps < end;
            if (more) load_keys(i + kWarps);
            const int rest = seen.end_of(i) - seen.first_of(i);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[u][x] = 8 * u + 2 * quad + x % 2 < rest ? s[u][x] * s2 : -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // rows `row` and `row + 8`
                float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float next = fmaxf(m[h], top), base = next == -INFINITY ? 0.f : next;
                if (__any_sync(0xffffffffu, next > m[h])) {
                    const float keep = exp2f(m[h] - base);
                    l[h] *= keep;
#pragma unroll
                    for (int x = 0; x < kV * 8; ++x) {
                        o[x][2 * h] *= keep;
                        o[x][2 * h + 1] *= keep;
                    }
                }
                m[h] = next;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int x = 2 * h; x < 2 * h + 2; ++x) {
                        s[u][x] = exp2f(s[u][x] - base);
                        l[h] += s[u][x];  // of this lane's keys; joined at the end
                    }
            }
            const uint32_t p0 = pack2<T>(s[0][0], s[0][1]), p1 = pack2<T>(s[0][2], s[0][3]), p2 = pack2<T>(s[1][0], s[1][1]),
                           p3 = pack2<T>(s[1][2], s[1][3]);
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                const uint32_t *a = reinterpret_cast<const uint32_t *>(&v[0][j]), *e = reinterpret_cast<const uint32_t *>(&v[1][j]),
                               *f = reinterpret_cast<const uint32_t *>(&v[2][j]), *g = reinterpret_cast<const uint32_t *>(&v[3][j]);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    small_product<T>(o[8 * j + 2 * x], p0, p1, p2, p3, __byte_perm(a[x], e[x], 0x5410), __byte_perm(f[x], g[x], 0x5410));
                    small_product<T>(o[8 * j + 2 * x + 1], p0, p1, p2, p3, __byte_perm(a[x], e[x], 0x7632), __byte_perm(f[x], g[x], 0x7632));
                }
            }
            if (more) load_values(i + kWarps);
        }
        // Columns of product x of chunk j: lane quad holds columns 2 quad and 2 quad + 1, dimensions 64 j + 8 (2 quad) + x and 64 j + 8 (2 quad + 1) + x.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            const int r = row + 8 * h;
            if (quad == 0) {
                tops[warp][r] = m[h];
                sums[warp][r] = l[h];
            }
#pragma unroll
            for (int j = 0; j < kV; ++j)
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        joined[warp][(r * kDim + 64 * j + 8 * (2 * quad + y)) / 4 + x] =
                            make_float4(o[8 * j + 4 * x][2 * h + y], o[8 * j + 4 * x + 1][2 * h + y], o[8 * j + 4 * x + 2][2 * h + y],
                                        o[8 * j + 4 * x + 3][2 * h + y]);
        }
        __syncthreads();
        const StepResult result(c, b, head0, begin == 0 && end == seen.blocks, first < share.begin || c.whole);
        for (int x = threadIdx.x; x < have * (kDim / 4); x += kWarps * 32) {
            const int r = x / (kDim / 4), d = x % (kDim / 4) * 4;
            float top = tops[0][r];
#pragma unroll
            for (int u = 1; u < kWarps; ++u) top = fmaxf(top, tops[u][r]);
            const float base = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < kWarps; ++u) {
                const float keep = exp2f(tops[u][r] - base);
                sum = fmaf(sums[u][r], keep, sum);
                vfma(acc, keep, joined[u][x]);
            }
            const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
            acc.x *= inv;
            acc.y *= inv;
            acc.z *= inv;
            acc.w *= inv;
            if (d < w.dim) result.store<T>(c, r, d, acc);
            if (d == 0) result.store_lse(r, top + log2f(sum));
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
        __syncthreads();  // (the next segment's results go where this one's are read)
    }
    if (blockIdx.x == 0) chain_wait();  // this grid is not complete before the prefix is
}

bool whole_units(const rode_heads_t &x) { return aligned_to(x.data, 16) && x.batch % 8 == 0 && x.row % 8 == 0 && x.head % 8 == 0; }

}  // namespace

bool step_takes(int dtype, const Cached &c) {
    return dtype != RODE_F32 && c.win.dim % 8 == 0 && c.win.dim <= 128 && whole_units(c.q) && whole_units(c.k) &&
           whole_units(c.v);
}

int step_on_tensor_cores(int dtype, const Cached &c, cudaStream_t stream) {
    const auto run = [&](auto *kernel) {
        RODE_CUDA_TRY(launch_part(kernel, dim3(c.ctas), kWarps * 32, 0, stream, c.prefix_parts > 0, c));
        return static_cast<int>(RODE_OK);
    };
    if (dtype == RODE_F16) return c.win.dim <= 64 ? run(&step_tiles<__half, 64>) : run(&step_tiles<__half, 128>);
    return c.win.dim <= 64 ? run(&step_tiles<__nv_bfloat16, 64>) : run(&step_tiles<__nv_bfloat16, 128>);
}

}  // namespace rode
