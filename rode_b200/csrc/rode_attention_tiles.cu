// Attention of 16-bit operands on the tensor cores (tcgen05): prompts and shared prefixes, head dimensions that are multiples of 8
// up to 128, 16-byte aligned operands.
//
// Rows of a tile are (query, head of the group) pairs, the heads innermost: all heads that read one key head share its key and
// value tiles, and a tile spans few positions, so that few keys of its blocks are out of its window.  128 / group queries per
// tile, two tiles per CTA.
//
// Forward, per block of 128 keys and tile: S = Q K^T into tensor memory, each thread of a warpgroup takes one row of S into
// registers (maximum and sum need no exchange), writes the weights P back over S in 16 bits, O += P V with P read
// from tensor memory.  One warpgroup per tile, so that while one tile is in its softmax the tensor cores work on the other; one
// warp issues the products, one the copies.
// O stays in tensor memory.  The running maximum is taken over only when it grows by more than 8 (in base 2): weights may then be as large
// as 2^8, which costs no precision (the sum has the same factor), and the multiplication of O by 2^(old - new) is rare.
// P is rounded to the operands' type (the products take 16-bit operands); the sum is that of the unrounded weights.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "rode_attention.cuh"
#include "rode_tensor_cores.cuh"

namespace rode {

// Waits that were given up (never, unless a kernel has an error), per GPU.
__device__ int waits_failed;

namespace {

constexpr int kRows = 128;                  // rows and keys of a tile
constexpr int kPanel = kRows * 128;         // bytes of a panel of 64 columns
constexpr float kLazy = 8.f;

// The last part of a sequence's keys, queries, ...: rows from `have` on of a tile of `panels` panels become zero (they belong to
// another sequence, or to nobody, and 0 x NaN is NaN).  One warp.
__device__ __forceinline__ void clear_rows(uint32_t tile, int panels, int have) {
    const int lane = threadIdx.x % 32;
    for (int p = 0; p < panels; ++p)
        for (int i = have * 8 + lane; i < kRows * 8; i += 32)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + p * kPanel + i * 16), "r"(0) : "memory");
    fence_async_proxy();
    __syncwarp();
}

// The columns of a tile that a row sees: column j when j < to and (j >= from or j < sink).
struct Range {
    int from, to, sink;
};

__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }

// Columns that are not seen become `value`.  By words of 32 bits, whose tests cost two instructions per column; the empty statement keeps
// the compiler from running them, predicated off, for blocks that are seen whole too (1040 clocks of a block's 5000).
template <int n>
__device__ __forceinline__ void hide(uint32_t (&x)[n], const Range &r, uint32_t value) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int c = 0; c < n; c += 32) {
        const uint32_t seen = bits_below(r.to - c) & (~bits_below(r.from - c) | bits_below(r.sink - c));
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (!(seen >> j & 1)) x[c + j] = value;
    }
}

__device__ __forceinline__ Pair load_pair(uint32_t shared) {
    Pair r;
    asm volatile("ld.shared.b64 %0, [%1];" : "=l"(r.x) : "r"(shared));
    return r;
}

// 2^x by additions and products, for x < 128: x = n + f with f in [-1/2, 1/2], 2^f by the polynomial of degree 4 with the least relative
// error there (Remez' exchange, 2.7e-6 after rounding its coefficients, far below the rounding of the weights to 16 bits), times 2^n.  Adding 1.5 * 2^23 + 127
// rounds to an integer, whose bits shifted by 23 are those of 2^n alone, or of 0 for n = -127: so x below -126.5, -infinity too, gives 0.  NaN gives NaN, by
// the product (n added to p's exponent made NaN a finite number, and ended at 2^-125, which bf16 holds, without being faster).
__device__ __forceinline__ void exp2_by_fma(Pair x, float &a, float &b) {
    split(x, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
    x = pair_of(a, b);
    const Pair t = add2(x, pair_of(12583039.f, 12583039.f));
    const Pair f = fma2(add2(t, pair_of(-12583039.f, -12583039.f)), pair_of(-1.f, -1.f), x);
    Pair p = fma2(f, pair_of(0x1.3997d6p-7f, 0x1.3997d6p-7f), pair_of(0x1.ca1440p-5f, 0x1.ca1440p-5f));
    p = fma2(f, p, pair_of(0x1.ec06dap-3f, 0x1.ec06dap-3f));
    p = fma2(f, p, pair_of(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
    p = fma2(f, p, pair_of(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
    float na, nb;
    split(t, na, nb);
    split(mul2(p, pair_of(__uint_as_float(__float_as_uint(na) << 23), __uint_as_float(__float_as_uint(nb) << 23))), a, b);
}
__device__ __forceinline__ float exp2_fast(float x) {
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
    return x;
}

// Scores o .. o + 63 to weights 2^(s2 x + off), packed in pairs into registers o / 2 ..; their sum is added.  The exponential unit makes 16 of
// them per clock and SM, which would take as long as the products: kByFma of every 8 pairs go to the FMA units instead (not in blocks with
// hidden columns, whose weights are exactly 0).
template <typename T, int o, int kByFma>
__device__ __forceinline__ void weights_of(uint32_t (&s)[128], float s2, float off, Pair &sum) {
    const Pair factor = pair_of(s2, s2), shift = pair_of(off, off);
#pragma unroll
    for (int j = o; j < o + 64; j += 2) {
        const Pair x = fma2(pair_of(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), factor, shift);
        float a, b;
        if (j / 2 % 8 < kByFma) {
            exp2_by_fma(x, a, b);
        } else {
            split(x, a, b);
            a = exp2_fast(a);
            b = exp2_fast(b);
        }
        sum = add2(sum, pair_of(a, b));
        s[j / 2] = pack2<T>(a, b);
    }
}
constexpr int kByFma = 2;

// Gradients: weights 2^(s2 x + off), left in 32 bits, of columns o .. o + 31 of a thread's 64.  The two warpgroups of a tile are at it side by side,
// so more go to the FMA units.
constexpr int kByFmaInPairs = 3;
template <int o, int kByFma, typename Off>
__device__ __forceinline__ void weights_in_place(uint32_t (&s)[64], float s2, Off &&off) {
    const Pair factor = pair_of(s2, s2);
#pragma unroll
    for (int j = o; j < o + 32; j += 2) {
        const Pair x = fma2(pair_of(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), factor, off(j));
        float a, b;
        if (j / 2 % 8 < kByFma) {
            exp2_by_fma(x, a, b);
        } else {
            split(x, a, b);
            a = exp2_fast(a);
            b = exp2_fast(b);
        }
        s[j] = __float_as_uint(a);
        s[j + 1] = __float_as_uint(b);
    }
}
// P (dP - delta) of columns o .. o + 31, rounded, in registers o / 2 .. of s (whose P it takes).
template <typename T, int o, typename Minus>
__device__ __forceinline__ void gradients_in_place(uint32_t (&s)[64], const uint32_t (&d)[64], Minus &&minus) {
#pragma unroll
    for (int j = o; j < o + 32; j += 2) {
        const Pair x = mul2(pair_of(__uint_as_float(s[j]), __uint_as_float(s[j + 1])),
                            add2(pair_of(__uint_as_float(d[j]), __uint_as_float(d[j + 1])), minus(j)));
        float a, b;
        split(x, a, b);
        s[j / 2] = pack2<T>(a, b);
    }
}

// A piece of work: two tiles of rows of a key head, the blocks of keys that any of them sees.
struct Work {
    int kv, part;       // key head, part of the prefix
    long long row0;     // first query (of the packed operand, or first request)
    int n_queries;      // queries of this CTA that exist
    int pos0;           // position of the first one
    long long key0;     // first key of the sequence
    int keys;           // its keys
    int blocks, n_sink, first;
    __device__ __forceinline__ int key_of(int i) const { return (i < n_sink ? i : first + i - n_sink) * kRows; }
};

struct TileMaps {
    CUtensorMap q, k, v;
};

template <int kDim>
constexpr int forward_stages() {
    return kDim == 64 ? 4 : 2;
}
template <int kDim>
constexpr int forward_bytes() {
    return 1024 + kDim / 64 * kPanel * (2 + 2 * forward_stages<kDim>()) + 512;
}

// Two warpgroups of softmax, one whose first warp issues the products and whose second one issues the copies.  The registers of a
// launch (384 x 168) are dealt out anew: 2 x 128 x 216 + 128 x 72 is the same number.
constexpr int kTileThreads = 384;
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;"); }
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); }

// What rounding to `rounded` took from two numbers.
template <typename T>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t rounded) {
    const T *t = reinterpret_cast<const T *>(&rounded);
    return pack2<T>(a - to_float(t[0]), b - to_float(t[1]));
}

// kShared: rows are requests, keys a part of the prefix, results go to the parts; else prompts.
template <typename T, int kDim, bool kShared>
__global__ void __launch_bounds__(kTileThreads, 1)
    forward_tiles(const __grid_constant__ TileMaps maps, const Prompt p, const Cached c, int items) {
    constexpr int kPanels = kDim / 64, kStages = forward_stages<kDim>(), kTile = kPanels * kPanel;
    extern __shared__ char shared_raw[];
    const Window &w = kShared ? c.win : p.win;
    const int group = w.heads / w.kv_heads, per_tile = kRows / group;
    if constexpr (kShared) chain_begin();  // the requests' own keys are worked on beside the prefix

    Work wk;
    // Item i: row tiles innermost by key heads, so that heads of the same positions run side by side.  False: nothing there.
    const auto load_work = [&](int item) {
        wk.kv = item % w.kv_heads;
        const int slot = item / w.kv_heads;
        if constexpr (kShared) {
            wk.part = slot % c.prefix_parts;
            wk.row0 = static_cast<long long>(slot / c.prefix_parts) * 2 * per_tile;
            wk.n_queries = static_cast<int>(min(static_cast<long long>(2 * per_tile), c.batch - wk.row0));
            wk.pos0 = 0;
            wk.key0 = 0;
            wk.keys = c.prefix;
            const long long all = (c.prefix + kRows - 1) / kRows;
            wk.n_sink = 0;
            wk.first = static_cast<int>(all * wk.part / c.prefix_parts);
            wk.blocks = static_cast<int>(all * (wk.part + 1) / c.prefix_parts) - wk.first;
        } else {
            const Tile t = find_tile(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, slot, 2 * per_tile);
            if (t.first < 0 || t.first >= t.rows || (t.seq < 0 && !p.clear)) return false;
            const int2 keys = t.seq < 0 ? make_int2(0, 0) : sequence_rows(p.seqs.k_offsets, p.seqs.k_rows, t.seq);
            wk.row0 = static_cast<long long>(t.row0) + t.first;
            wk.n_queries = min(2 * per_tile, t.rows - t.first);
            wk.pos0 = t.first + keys.y - t.rows;
            wk.key0 = keys.x;
            wk.keys = keys.y;
            const KeyBlocks b(wk.pos0, wk.pos0 + wk.n_queries, w.window, w.sinks, kRows);
            wk.blocks = b.n;
            wk.n_sink = b.n_sink;
            wk.first = b.first;
        }
        return true;
    };
    // Queries of tile t, and whether it sees any key of the block from k0 on.
    const auto queries_of = [&](int t) { return min(per_tile, wk.n_queries - t * per_tile); };
    const auto sees_block = [&](int t, int k0) {
        const int n = queries_of(t);
        if (n <= 0) return false;
        if constexpr (kShared) return true;
        const int a = wk.pos0 + t * per_tile, b = a + n - 1;  // positions
        return k0 <= b && (k0 + kRows - 1 > a - w.window || k0 < w.sinks);
    };

    const uint32_t base = uniform((shared_address(shared_raw) + 1023) & ~1023u);
    const uint32_t qs = base, ks = qs + 2 * kTile, vs = ks + kStages * kTile, bars = vs + kStages * kTile;
    const uint32_t q_full = bars, v_raw = bars + 8, q_empty = bars + 96, s_full = bars + 16, o_done = bars + 32, p_full = bars + 48, turn = bars + 80, k_full = bars + 104,
                   k_empty = k_full + 8 * kStages, v_full = k_empty + 8 * kStages, v_empty = v_full + 8 * kStages,
                   tmem_at = v_empty + 8 * kStages;
    const int warp = uniform(threadIdx.x / 32), lane = threadIdx.x % 32;
    if (warp == 9 && lane < 3) prefetch_map(lane == 0 ? &maps.q : lane == 1 ? &maps.k : &maps.v);
    if (warp == 8) {
        tmem_alloc(tmem_at, 512);
        if (lane == 0) {
            barrier_init(q_full, 1);
            barrier_init(v_raw, 1);
            barrier_init(q_empty, 2);
            barrier_init(turn, 128);
            barrier_init(turn + 8, 128);
            for (int t = 0; t < 2; ++t) {
                barrier_init(s_full + 8 * t, 1);
                barrier_init(p_full + 16 * t, 128);
                barrier_init(p_full + 16 * t + 8, 128);
                barrier_init(o_done + 8 * t, 1);
            }
            for (int i = 0; i < kStages; ++i) {
                barrier_init(k_full + 8 * i, 1);
                barrier_init(k_empty + 8 * i, 2);
                barrier_init(v_full + 8 * i, 1);
                barrier_init(v_empty + 8 * i, 2);
            }
            barrier_init_done();
        }
        __syncwarp();
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));
    tmem = uniform(tmem);
    bool ok = true;  // (a wait that was given up ends the CTA's work; it took seconds, so that no copy is in flight any more)

    if (warp >= 8) give_registers();
    if (warp == 9) {
        // copies
        int raw = 0, loaded = 0, filled = 0;  // raw blocks, items, blocks so far
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            if (!load_work(item) || wk.blocks == 0) continue;
            ok = barrier_wait(q_empty, (loaded++ & 1) ^ 1);
            if (ok && lane == 0) {
                const int tiles = queries_of(1) > 0 ? 2 : 1;
                barrier_expect(q_full, tiles * kPanels * per_tile * group * 128);
                for (int t = 0; t < tiles; ++t)
                    for (int x = 0; x < kPanels; ++x)
                        copy_box(qs + t * kTile + x * kPanel, &maps.q, x * 64, wk.kv * group, static_cast<int>(wk.row0) + t * per_tile, q_full);
            }
            __syncwarp();
            for (int i = 0; i < wk.blocks && ok; ++i, ++filled) {
                const int st = filled % kStages, k0 = wk.key_of(i), have = wk.keys - k0;
                const uint32_t free = (filled / kStages & 1) ^ 1;
                const int y = static_cast<int>(wk.key0) + k0;
                ok = barrier_wait(k_empty + 8 * st, free);
                if (ok && lane == 0) {
                    barrier_expect(k_full + 8 * st, kTile);
                    for (int x = 0; x < kPanels; ++x) copy_box(ks + st * kTile + x * kPanel, &maps.k, x * 64, wk.kv, y, k_full + 8 * st);
                }
                ok = ok && barrier_wait(v_empty + 8 * st, free);
                if (!ok) break;
                const uint32_t bar = have < kRows ? v_raw : v_full + 8 * st;
                if (lane == 0) {
                    barrier_expect(bar, kTile);
                    for (int x = 0; x < kPanels; ++x) copy_box(vs + st * kTile + x * kPanel, &maps.v, x * 64, wk.kv, y, bar);
                }
                __syncwarp();
                if (have < kRows) {
                    ok = barrier_wait(v_raw, raw & 1);
                    ++raw;
                    clear_rows(vs + st * kTile, kPanels, have);
                    if (lane == 0) barrier_arrive(v_full + 8 * st);
                }
            }
        }
    } else if (warp == 8 || warp == 10) {
        // products, one warp per tile, so that a wait for one tile holds up nothing of the other
        const int t = warp == 8 ? 0 : 1;
        const uint32_t scores = product_descriptor<T>(kRows, false), values = product_descriptor<T>((w.dim + 15) / 16 * 16, true);
        const uint32_t one = elect_one();
        const int steps = (w.dim + 15) / 16;
        const uint32_t s_at = tmem + t * kRows, o_at = tmem + 256 + t * kDim;
        int loaded = 0, filled = 0, issued = 0;  // items, blocks, blocks of this tile so far
        const auto issue_scores = [&](int i) {   // of block i of the item, and its keys' stage is done with
            const int st = (filled + i) % kStages;
            ok = barrier_wait(k_full + 8 * st, (filled + i) / kStages & 1);
            if (!ok) return;
            if (sees_block(t, wk.key_of(i))) {
                tmem_fence_after();
                const uint64_t a = tile_descriptor(qs + t * kTile, 16), b = tile_descriptor(ks + st * kTile, 16);
#pragma unroll
                for (int s = 0; s < kDim / 16; ++s)
                    if (s < steps) {
                        const uint32_t at = (s / 4 * kPanel + s % 4 * 32) >> 4;
                        product(one, s_at, a + at, b + at, scores, s > 0);
                    }
                products_arrive(one, s_full + 8 * t);
                products_arrive(one, k_empty + 8 * st);
            } else if (one) {
                barrier_arrive(k_empty + 8 * st);
            }
            if (i + 1 == wk.blocks) products_arrive(one, q_empty);  // the next item's queries may come
            __syncwarp();
        };
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            if (!load_work(item) || wk.blocks == 0) continue;
            ok = barrier_wait(q_full, loaded++ & 1);
            if (ok) issue_scores(0);
            bool add = false;
            for (int i = 0; i < wk.blocks && ok; ++i) {
                const int st = (filled + i) % kStages;
                ok = barrier_wait(v_full + 8 * st, (filled + i) / kStages & 1);
                if (!ok) break;
                if (sees_block(t, wk.key_of(i))) {
                    const uint64_t b = tile_descriptor(vs + st * kTile, kPanel);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        ok = ok && barrier_wait(p_full + 16 * t + 8 * half, issued & 1);
                        tmem_fence_after();
                        if (ok)
#pragma unroll
                            for (int s = 4 * half; s < 4 * half + 4; ++s)
                                product_from_tmem(one, o_at, s_at + s * 8, b + s * 128, values, add || s > 0);
                    }
                    if (!ok) break;
                    add = true;
                    products_arrive(one, o_done + 8 * t);
                    products_arrive(one, v_empty + 8 * st);
                    // the next scores go where the weights were
                    ok = barrier_wait(o_done + 8 * t, issued & 1);
                    ++issued;
                } else if (one) {
                    barrier_arrive(v_empty + 8 * st);
                }
                __syncwarp();
                if (ok && i + 1 < wk.blocks) issue_scores(i + 1);
            }
            filled += wk.blocks;
        }
    } else if (warp < 8) {
        // softmax: one row per thread
        take_registers();
        const int t = warp / 4, r = threadIdx.x % 128;
        const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
        const uint32_t s_at = tmem + lanes + t * kRows, o_at = tmem + lanes + 256 + t * kDim;
        const int query = r / group;
        const float s2 = w.scale * kLog2e;
        int seen = 0, turn_of = 0;  // blocks of this tile, turns so far
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            if (!load_work(item)) continue;
            const int n = queries_of(t), head = wk.kv * group + r % group;
            const bool mine = query < n;
            const int a = wk.pos0 + t * per_tile, pos = a + query;
            float m = -INFINITY, l = 0.f;
            int done = 0;
            // The tiles' exponentials take turns: side by side they would take twice as long and then wait for the products side by side
            // (blocks of both tiles in 3250 clocks instead of 3800).
            const bool turns = queries_of(1) > 0;
            for (int i = 0; i < wk.blocks; ++i) {
                const int k0 = wk.key_of(i);
                if (!sees_block(t, k0)) {
                    if (turns) {
                        ok = barrier_wait(turn + 8 * t, (turn_of++ + t + 1) & 1);
                        if (!ok) break;
                        barrier_arrive(turn + 8 * (t ^ 1));
                    }
                    continue;
                }
                ok = barrier_wait(s_full + 8 * t, seen & 1);
                if (!ok) break;
                tmem_fence_after();
                uint32_t s[128];
                tmem_load32<0>(s_at, s);
                tmem_load32<32>(s_at + 32, s);
                tmem_load32<64>(s_at + 64, s);
                tmem_load32<96>(s_at + 96, s);
                tmem_wait_load32<0>(s);
                tmem_wait_load32<32>(s);
                tmem_wait_load32<64>(s);
                tmem_wait_load32<96>(s);
                bool whole;
                if constexpr (kShared)
                    whole = k0 + kRows <= wk.keys;
                else
                    whole = k0 + kRows - 1 <= a && (a + n - 1 - k0 < w.window || k0 + kRows <= w.sinks);
                if (!whole) {
                    if constexpr (kShared)
                        hide(s, {0, wk.keys - k0, 0}, 0xff800000u);  // -infinity
                    else
                        hide(s, {pos - w.window + 1 - k0, pos + 1 - k0, w.sinks - k0}, 0xff800000u);
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 128; j += 2)
                    top[j / 2 % 4] = fmaxf(top[j / 2 % 4], fmaxf(__uint_as_float(s[j]), __uint_as_float(s[j + 1])));
                const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                const bool grows = (high - m) * s2 > kLazy;
                if (__any_sync(0xffffffffu, grows)) {
                    const float next = grows ? high : m;
                    const float keep = grows ? exp2f((m - next) * s2) : 1.f;
                    m = next;
                    l *= keep;
                    if (done > 0) {
#pragma unroll
                        for (int x = 0; x < kDim; x += 32) {
                            uint32_t o[32];
                            tmem_load32<0>(o_at + x, o);
                            tmem_wait_load32<0>(o);
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                            tmem_store32<0>(o_at + x, o);
                        }
                    }
                }
                const float off = m == -INFINITY ? 0.f : -m * s2;
                if (turns) {
                    ok = barrier_wait(turn + 8 * t, (turn_of++ + t + 1) & 1);
                    if (!ok) break;
                }
                // the first half's products run during the second half's exponentials
                Pair sum = pair_of(0.f, 0.f);
                if (whole)
                    weights_of<T, 0, kByFma>(s, s2, off, sum);
                else
                    weights_of<T, 0, 0>(s, s2, off, sum);
                tmem_store32<0>(s_at, s);
                tmem_wait_store();
                tmem_fence_before();
                barrier_arrive(p_full + 16 * t);
                if (whole)
                    weights_of<T, 64, kByFma>(s, s2, off, sum);
                else
                    weights_of<T, 64, 0>(s, s2, off, sum);
                tmem_store32<32>(s_at + 32, s);
                tmem_wait_store();
                tmem_fence_before();
                barrier_arrive(p_full + 16 * t + 8);
                if (turns) barrier_arrive(turn + 8 * (t ^ 1));
                float even, odd;
                split(sum, even, odd);
                l += even + odd;
                ++done;
                ++seen;
            }
            if (ok && done > 0) {
                ok = barrier_wait(o_done + 8 * t, (seen - 1) & 1);
                tmem_fence_after();
            }
            const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
            const float lse2 = m * s2 + log2f(l);  // -inf for a row that has seen no key, NaN for one whose scores are
            if (kShared) {
                const long long at = (wk.part * static_cast<long long>(c.batch) + wk.row0 + t * per_tile + query) * w.heads + head;
                if (mine) c.prefix_lse[at] = lse2;
#pragma unroll
                for (int x = 0; x < kDim; x += 32) {
                    uint32_t o[32];
                    tmem_load32<0>(o_at + x, o);
                    tmem_wait_load32<0>(o);
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        if (mine && x + j < w.dim)
                            store4(c.prefix_out + at * w.dim + x + j,
                                   done > 0 ? make_float4(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv,
                                                          __uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv)
                                            : make_float4(0.f, 0.f, 0.f, 0.f));
                }
            } else {
                const long long row = wk.row0 + t * per_tile + query;
                if (mine && p.lse != nullptr)
                    p.lse[static_cast<long long>(head) * p.seqs.q_rows + row] = lse2 * kLn2;
                T *out = static_cast<T *>(p.out) + (row * w.heads + head) * w.dim;
#pragma unroll
                for (int x = 0; x < kDim; x += 32) {
                    uint32_t o[32];
                    tmem_load32<0>(o_at + x, o);
                    tmem_wait_load32<0>(o);
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        uint4 y = make_uint4(0, 0, 0, 0);
                        if (done > 0) {
                            y.x = pack2<T>(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv);
                            y.y = pack2<T>(__uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv);
                            y.z = pack2<T>(__uint_as_float(o[j + 4]) * inv, __uint_as_float(o[j + 5]) * inv);
                            y.w = pack2<T>(__uint_as_float(o[j + 6]) * inv, __uint_as_float(o[j + 7]) * inv);
                        }
                        if (mine && x + j < w.dim) *reinterpret_cast<uint4 *>(out + x + j) = y;
                        if (p.rest != nullptr) {
                            uint4 z = make_uint4(0, 0, 0, 0);
                            if (done > 0) {
                                z.x = rest2<T>(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv, y.x);
                                z.y = rest2<T>(__uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv, y.y);
                                z.z = rest2<T>(__uint_as_float(o[j + 4]) * inv, __uint_as_float(o[j + 5]) * inv, y.z);
                                z.w = rest2<T>(__uint_as_float(o[j + 6]) * inv, __uint_as_float(o[j + 7]) * inv, y.w);
                            }
                            if (mine && x + j < w.dim) *reinterpret_cast<uint4 *>(static_cast<T *>(p.rest) + (out - static_cast<T *>(p.out)) + x + j) = z;
                        }
                    }
                }
            }
        }
    }
    if (!ok) waits_failed = 1;
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == 8) tmem_free(tmem, 512);
}

// --- gradients ------------------------------------------------------------------------------------------------------------------
//
// dS = P (dP - delta) with P = 2^(scale log2e S - lse) and dP = dO V^T again from the operands, delta = dO . O per row.  Two kernels, so that
// every sum has one owner and one order: one CTA per tile of queries adds up dQ = dS K, one per tile of keys dV = P^T dO and dK = dS^T Q
// (7 products instead of the 5 that one kernel with atomic additions would need).  The first takes rows of queries as the rows of S, the
// second computes S^T and dP^T, so that in both the 16-bit factor that the threads compute (dS, P^T, dS^T) is the operand from tensor
// memory, over the columns it was computed from, and no tile is transposed.  P and dS are rounded to the operands' type for that.
// Two warpgroups share a tile, each 64 columns.

template <int kDim>
constexpr int backward_stages() {
    return kDim == 64 ? 4 : 2;
}
template <int kDim>
constexpr int backward_bytes() {
    return 1024 + kDim / 64 * kPanel * (2 + 2 * backward_stages<kDim>()) + backward_stages<kDim>() * 2 * kRows * 4 + 512;
}

struct GradientMaps {
    CUtensorMap q, dout, k, v;
};

// delta = do . o of all rows, a lane per 16 bytes, with what rounding took from o: in rows of few keys dP - delta cancels, and the rounding
// of o counted as much as that of the result (fp16, sequences of some tens of rows: dQ 0.00042 off instead of 0.0003; writing and reading it costs 70 us of
// train_long's 2396).  (By two spare warps of the kernel below it took as long as three blocks of keys, more than short windows
// have.)
template <typename T, int kDim>
__global__ void __launch_bounds__(256) row_deltas(const Prompt p) {
    constexpr int kLanes = kDim / 8;
    chain_begin();
    const int dim = p.win.dim, heads = p.win.heads, d = threadIdx.x % kLanes * 8;
    const long long rows = static_cast<long long>(p.seqs.q_rows) * heads, i = blockIdx.x * (256ll / kLanes) + threadIdx.x / kLanes;
    const long long row = i / heads;
    const int head = static_cast<int>(i % heads);
    float sum = 0.f;
    if (i < rows && d < dim) {
        const uint4 x = __ldg(reinterpret_cast<const uint4 *>(row_of<T>(p.dout, 0, row, head) + d));
        const uint4 y = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.out) + i * dim + d));
        uint4 z = make_uint4(0, 0, 0, 0);
        if (p.rest != nullptr) z = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.rest) + i * dim + d));
        const T *s = reinterpret_cast<const T *>(&x), *t = reinterpret_cast<const T *>(&y), *rest = reinterpret_cast<const T *>(&z);
#pragma unroll
        for (int u = 0; u < 8; ++u) sum = fmaf(to_float(s[u]), to_float(t[u]) + to_float(rest[u]), sum);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (i < rows && threadIdx.x % kLanes == 0) p.delta[head * static_cast<long long>(p.seqs.q_rows) + row] = sum;
}

// -lse in base 2 and -delta of the rows of a tile (row r = query r / group, head r % group) to shared memory, by one warp.
__device__ __forceinline__ void fetch_rows(const Prompt &p, const float *deltas, long long row0, int head0, int group, int n, uint32_t to) {
#pragma unroll
    for (int r = threadIdx.x % 32; r < kRows; r += 32) {
        float lse = 0.f, delta = 0.f;
        if (r / group < n) {
            const long long at = static_cast<long long>(head0 + r % group) * p.seqs.q_rows + row0 + r / group;
            lse = __ldg(p.lse + at);
            lse = lse == -INFINITY ? 0.f : -lse * kLog2e;
            delta = __ldcg(deltas + at);
        }
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + r * 4), "f"(lse) : "memory");
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + (kRows + r) * 4), "f"(-delta) : "memory");
    }
}

// Columns x .. x + 31 of an accumulator row, times factor, to 32 elements of a row of `dim`.
template <typename T>
__device__ __forceinline__ void store_columns(T *row, uint32_t at, int x, int dim, float factor, bool mine, bool any) {
    uint32_t o[32];
    tmem_load32<0>(at + x, o);
    tmem_wait_load32<0>(o);
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
        uint4 y = make_uint4(0, 0, 0, 0);
        if (any) {
            y.x = pack2<T>(__uint_as_float(o[j]) * factor, __uint_as_float(o[j + 1]) * factor);
            y.y = pack2<T>(__uint_as_float(o[j + 2]) * factor, __uint_as_float(o[j + 3]) * factor);
            y.z = pack2<T>(__uint_as_float(o[j + 4]) * factor, __uint_as_float(o[j + 5]) * factor);
            y.w = pack2<T>(__uint_as_float(o[j + 6]) * factor, __uint_as_float(o[j + 7]) * factor);
        }
        if (mine && x + j < dim) *reinterpret_cast<uint4 *>(row + x + j) = y;
    }
}

// dQ, a tile of rows at a time.  Tensor memory: S twice (dS over it), dP, dQ.  The products of block i + 1 that need no dS (S, then
// dP) run while the threads work on block i.  Persistent: the next tile's rows, sums and first products come while this tile's dQ is written (tiles of 18
// blocks of 2000 clocks took another 20000 each as CTAs of their own).
template <typename T, int kDim>
__global__ void __launch_bounds__(kTileThreads, 1)
    query_gradient_tiles(const __grid_constant__ GradientMaps maps, const Prompt p, int items) {
    constexpr int kPanels = kDim / 64, kStages = backward_stages<kDim>(), kTile = kPanels * kPanel;
    extern __shared__ char shared_raw[];
    const Window &w = p.win;
    const int group = w.heads / w.kv_heads, per_tile = kRows / group;
    struct {
        int kv, n, pos0, keys, key0;
        long long row0;
    } wk;
    KeyBlocks blocks(0, 0, 1, 0, kRows);
    // Item i: tiles by key heads, so that heads of the same positions run side by side.  False: nothing there.
    const auto load_work = [&](int item) {
        wk.kv = item % w.kv_heads;
        const Tile t = find_tile(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, item / w.kv_heads, per_tile);
        if (t.first < 0 || t.first >= t.rows || (t.seq < 0 && !p.clear)) return false;
        const int2 keys = t.seq < 0 ? make_int2(0, 0) : sequence_rows(p.seqs.k_offsets, p.seqs.k_rows, t.seq);
        wk.row0 = static_cast<long long>(t.row0) + t.first;
        wk.n = min(per_tile, t.rows - t.first);
        wk.pos0 = t.first + keys.y - t.rows;
        wk.key0 = keys.x;
        wk.keys = keys.y;
        blocks = KeyBlocks(wk.pos0, wk.pos0 + wk.n, w.window, w.sinks, kRows);
        return true;
    };

    const uint32_t base = uniform((shared_address(shared_raw) + 1023) & ~1023u);
    const uint32_t qs = base, gs = qs + kTile, ks = gs + kTile, vs = ks + kStages * kTile, rows_at = vs + kStages * kTile,
                   bars = rows_at + kStages * 2 * kRows * 4;
    const uint32_t q_full = bars, q_empty = bars + 8, k_raw = bars + 16, dp_full = bars + 24, dq_done = bars + 32, dq_free = bars + 40,
                   s_full = bars + 48, ds_full = bars + 64, rows_full = bars + 80, rows_empty = bars + 96, k_full = bars + 112,
                   k_empty = k_full + 8 * kStages, v_full = k_empty + 8 * kStages, v_empty = v_full + 8 * kStages,
                   tmem_at = v_empty + 8 * kStages;
    const int warp = uniform(threadIdx.x / 32), lane = threadIdx.x % 32;
    if (warp == 9 && lane < 4) prefetch_map(lane == 0 ? &maps.q : lane == 1 ? &maps.dout : lane == 2 ? &maps.k : &maps.v);
    if (warp == 8) {
        tmem_alloc(tmem_at, 512);
        if (lane == 0) {
            barrier_init(q_full, 1);
            barrier_init(q_empty, 1);
            barrier_init(k_raw, 1);
            barrier_init(dp_full, 1);
            barrier_init(dq_done, 1);
            barrier_init(dq_free, 256);
            for (int i = 0; i < 2; ++i) {
                barrier_init(s_full + 8 * i, 1);
                barrier_init(ds_full + 8 * i, 256);
                barrier_init(rows_full + 8 * i, 32);
                barrier_init(rows_empty + 8 * i, 256);
            }
            for (int i = 0; i < kStages; ++i) {
                barrier_init(k_full + 8 * i, 1);
                barrier_init(k_empty + 8 * i, 1);
                barrier_init(v_full + 8 * i, 1);
                barrier_init(v_empty + 8 * i, 1);
            }
            barrier_init_done();
        }
        __syncwarp();
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));
    tmem = uniform(tmem);
    const uint32_t dp_at = tmem + 256, dq_at = tmem + 384;
    bool ok = true;

    if (warp >= 8) give_registers();
    if (warp == 9) {
        int raw = 0, loaded = 0, filled = 0;  // raw blocks, items, blocks so far
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            if (!load_work(item) || blocks.n == 0) continue;
            ok = barrier_wait(q_empty, (loaded++ & 1) ^ 1);
            if (ok && lane == 0) {
                barrier_expect(q_full, 2 * kPanels * per_tile * group * 128);
                for (int x = 0; x < kPanels; ++x) {
                    copy_box(qs + x * kPanel, &maps.q, x * 64, wk.kv * group, static_cast<int>(wk.row0), q_full);
                    copy_box(gs + x * kPanel, &maps.dout, x * 64, wk.kv * group, static_cast<int>(wk.row0), q_full);
                }
            }
            __syncwarp();
            for (int i = 0; i < blocks.n && ok; ++i, ++filled) {
                const int st = filled % kStages, k0 = blocks.at(i) * kRows, have = wk.keys - k0, y = wk.key0 + k0;
                const uint32_t free = (filled / kStages & 1) ^ 1;
                ok = barrier_wait(k_empty + 8 * st, free);
                const uint32_t bar = have < kRows ? k_raw : k_full + 8 * st;
                if (ok && lane == 0) {
                    barrier_expect(bar, kTile);
                    for (int x = 0; x < kPanels; ++x) copy_box(ks + st * kTile + x * kPanel, &maps.k, x * 64, wk.kv, y, bar);
                }
                __syncwarp();
                if (ok && have < kRows) {
                    ok = barrier_wait(k_raw, raw++ & 1);
                    clear_rows(ks + st * kTile, kPanels, have);
                    if (lane == 0) barrier_arrive(k_full + 8 * st);
                }
                ok = ok && barrier_wait(v_empty + 8 * st, free);
                if (ok && lane == 0) {
                    barrier_expect(v_full + 8 * st, kTile);
                    for (int x = 0; x < kPanels; ++x) copy_box(vs + st * kTile + x * kPanel, &maps.v, x * 64, wk.kv, y, v_full + 8 * st);
                }
                __syncwarp();
            }
        }
    } else if (warp == 8) {
        const uint32_t scores = product_descriptor<T>(kRows, false), sums = product_descriptor<T>((w.dim + 15) / 16 * 16, true);
        const int steps = (w.dim + 15) / 16;
        const uint32_t one = elect_one();
        const auto issue = [&](uint32_t d, uint32_t a, uint32_t b, uint32_t bar) {
            const uint64_t x = tile_descriptor(a, 16), y = tile_descriptor(b, 16);
#pragma unroll
            for (int s = 0; s < kDim / 16; ++s)
                if (s < steps) {
                    const uint32_t at = (s / 4 * kPanel + s % 4 * 32) >> 4;
                    product(one, d, x + at, y + at, scores, s > 0);
                }
            products_arrive(one, bar);
        };
        int loaded = 0, g = 0;  // items and blocks so far
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            if (!load_work(item) || blocks.n == 0) continue;
            // the first block's S and dP: S goes where dS of the block before the last one was
            ok = barrier_wait(q_full, loaded & 1) && barrier_wait(k_full + 8 * (g % kStages), g / kStages & 1) &&
                 barrier_wait(v_full + 8 * (g % kStages), g / kStages & 1);
            if (!ok) break;
            tmem_fence_after();
            issue(tmem + (g & 1) * kRows, qs, ks + g % kStages * kTile, s_full + 8 * (g & 1));
            issue(dp_at, gs, vs + g % kStages * kTile, dp_full);
            products_arrive(one, v_empty + 8 * (g % kStages));
            if (blocks.n == 1) products_arrive(one, q_empty);
            for (int i = 0; i < blocks.n && ok; ++i, ++g) {
                const int st = g % kStages, next = (g + 1) % kStages, buf = g & 1;
                const uint32_t next_full = (g + 1) / kStages & 1;
                const bool more = i + 1 < blocks.n;
                ok = g == 0 || barrier_wait(dq_done, (g - 1) & 1);
                if (!ok) break;
                if (more) {
                    // S of the next block where dS of the last one was
                    ok = barrier_wait(k_full + 8 * next, next_full);
                    if (!ok) break;
                    tmem_fence_after();
                    issue(tmem + (buf ^ 1) * kRows, qs, ks + next * kTile, s_full + 8 * (buf ^ 1));
                }
                if (i == 0) {  // dQ of the item before is written
                    ok = barrier_wait(dq_free, (loaded & 1) ^ 1);
                    if (!ok) break;
                }
                const uint64_t keys_of_block = tile_descriptor(ks + st * kTile, kPanel);
#pragma unroll
                for (int piece = 0; piece < 2; ++piece) {  // 32 of each warpgroup's 64 columns
                    ok = ok && barrier_wait(ds_full + 8 * piece, g & 1);
                    tmem_fence_after();
                    if (ok)
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int s = u / 2 * 4 + piece * 2 + u % 2;
                            product_from_tmem(one, dq_at, tmem + buf * kRows + s / 4 * 64 + s % 4 * 8, keys_of_block + s * 128, sums,
                                              i > 0 || piece > 0 || u > 0);
                        }
                }
                if (!ok) break;
                products_arrive(one, dq_done);
                products_arrive(one, k_empty + 8 * st);
                if (more) {
                    ok = barrier_wait(v_full + 8 * next, next_full);
                    if (!ok) break;
                    issue(dp_at, gs, vs + next * kTile, dp_full);
                    products_arrive(one, v_empty + 8 * next);
                    if (i + 2 == blocks.n) products_arrive(one, q_empty);
                }
                __syncwarp();
            }
            ++loaded;
        }
    } else if (warp == 10) {
        const float *deltas = after_chain(p.delta);
        int i = 0;
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            if (!load_work(item) || blocks.n == 0) continue;
            ok = barrier_wait(rows_empty + 8 * (i & 1), (i / 2 & 1) ^ 1);
            if (!ok) break;
            fetch_rows(p, deltas, wk.row0, wk.kv * group, group, wk.n, rows_at + (i & 1) * 2 * kRows * 4);
            barrier_arrive(rows_full + 8 * (i & 1));
            ++i;
        }
    } else if (warp < 8) {
        take_registers();
        const int half = warp / 4, r = threadIdx.x % 128, query = r / group;
        const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
        const float s2 = w.scale * kLog2e;
        int started = 0, g = 0;  // items and blocks so far
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            if (!load_work(item)) continue;
            const int head = wk.kv * group + r % group, pos = wk.pos0 + query, n = wk.n;
            const bool mine = query < n;
            const uint32_t rows = rows_at + (started & 1) * 2 * kRows * 4;
            float off = 0.f, minus_delta = 0.f;
            if (blocks.n > 0) {
                ok = barrier_wait(rows_full + 8 * (started & 1), started / 2 & 1);
                if (!ok) break;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(off) : "r"(rows + 4 * r) : "memory");
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(minus_delta) : "r"(rows + 4 * (kRows + r)) : "memory");
                barrier_arrive(rows_empty + 8 * (started & 1));
                ++started;
            }
            for (int i = 0; i < blocks.n; ++i, ++g) {
                const int k0 = blocks.at(i) * kRows, buf = g & 1, c0 = k0 + half * 64;
                const uint32_t s_at = tmem + lanes + buf * kRows + half * 64;
                const bool whole = k0 + kRows - 1 <= wk.pos0 && (wk.pos0 + n - 1 - k0 < w.window || k0 + kRows <= w.sinks);
                const Range range = {pos - w.window + 1 - c0, pos + 1 - c0, w.sinks - c0};
                ok = barrier_wait(s_full + 8 * buf, g / 2 & 1);
                if (!ok) break;
                tmem_fence_after();
                uint32_t s[64], d[64];
                tmem_load32<0>(s_at, s);
                tmem_load32<32>(s_at + 32, s);
                tmem_wait_load32<0>(s);
                tmem_wait_load32<32>(s);
                if (!whole) hide(s, range, 0xff800000u);
                const auto weight_off = [&](int) { return pair_of(off, off); };
                if (whole) {
                    weights_in_place<0, kByFmaInPairs>(s, s2, weight_off);
                    weights_in_place<32, kByFmaInPairs>(s, s2, weight_off);
                } else {
                    weights_in_place<0, 0>(s, s2, weight_off);
                    weights_in_place<32, 0>(s, s2, weight_off);
                }
                // (dQ of the block before is complete by now; every phase of its barrier is waited for, so that the last one of the item
                // cannot be taken for an earlier one)
                ok = barrier_wait(dp_full, g & 1) && (i == 0 || barrier_wait(dq_done, (g - 1) & 1));
                if (!ok) break;
                tmem_fence_after();
                tmem_load32<0>(dp_at + lanes + half * 64, d);
                tmem_load32<32>(dp_at + lanes + half * 64 + 32, d);
                tmem_wait_load32<0>(d);
                tmem_wait_load32<32>(d);
                if (!whole) hide(d, range, 0u);
                const auto minus = [&](int) { return pair_of(minus_delta, minus_delta); };
                gradients_in_place<T, 0>(s, d, minus);
                tmem_store16<0>(s_at, s);
                tmem_wait_store();
                tmem_fence_before();
                barrier_arrive(ds_full);
                gradients_in_place<T, 32>(s, d, minus);
                tmem_store16<16>(s_at + 16, s);
                tmem_wait_store();
                tmem_fence_before();
                barrier_arrive(ds_full + 8);
            }
            if (ok && blocks.n > 0) {
                ok = barrier_wait(dq_done, (g - 1) & 1);
                tmem_fence_after();
            }
            T *out = static_cast<T *>(p.dq) + ((wk.row0 + query) * w.heads + head) * w.dim;
#pragma unroll
            for (int x = 0; x < kDim / 2; x += 32)
                store_columns(out, dq_at + lanes, half * (kDim / 2) + x, w.dim, w.scale, mine, blocks.n > 0);
            if (blocks.n > 0) {
                tmem_fence_before();
                barrier_arrive(dq_free);
            }
        }
    }
    if (!ok) waits_failed = 1;
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == 8) tmem_free(tmem, 512);
}

// Queries up to the end of the window of the last of `have` keys from key `first` on.
__device__ __forceinline__ int near_queries(int first, int have, int keys, int queries, int window) {
    const int last = window >= keys - (first + have - 1) ? keys : first + have - 1 + window;
    return min(max(last - (keys - queries), max(first - (keys - queries), 0)), queries);
}
// Whether the far queries of a sequence's first tile are worked on in chunks.
__device__ __forceinline__ bool far_chunks(const Prompt &p, int near, int queries) {
    return p.far_chunk > 0 && queries - near > p.far_chunk / 2;
}

// dK and dV of one tile of 128 keys: all rows of queries that see any of them, 128 at a time.  Tensor memory: S^T, dP^T (P^T and dS^T over it; twice
// where the head dimension leaves room), dV, dK.  S^T of the next tile of queries is made as soon as the threads have this one's in registers, so
// that they never wait for it; what they wait for is dP^T, which must wait for dV and dK of the tile before.
//
// The first tile of a sequence has the sinks, which all later queries see: as one CTA it took 4 times as long as the others on 8192 positions with a
// window of 2048, and the grid waited for it (train_long 1436 us, 923 without it).  So queries behind the window of the first tile's keys ("far" ones) are cut into chunks of
// p.far_chunk for CTAs of their own, which come first in the grid; these and the first tile leave their sums in 32 bits, and add_far_gradients adds
// them up in order.
template <typename T, int kDim>
__global__ void __launch_bounds__(kTileThreads, 1) key_gradient_tiles(const __grid_constant__ GradientMaps maps, const Prompt p) {
    constexpr int kPanels = kDim / 64, kStages = backward_stages<kDim>(), kTile = kPanels * kPanel;
    extern __shared__ char shared_raw[];
    const Window &w = p.win;
    const int group = w.heads / w.kv_heads, per_tile = kRows / group, kv = blockIdx.y;
    const int far = static_cast<int>(blockIdx.x) < p.far_slots ? static_cast<int>(blockIdx.x) : -1;
    Tile t;
    int2 queries;
    int chunk = 0;  // first query of a far chunk
    if (far >= 0) {
        const Tile u = find_tile(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, far, p.far_chunk);
        if (u.first < 0 || u.first >= u.rows || u.seq < 0) return;
        const int2 keys = sequence_rows(p.seqs.k_offsets, p.seqs.k_rows, u.seq);
        t = {u.seq, keys.x, keys.y, 0};
        queries = make_int2(u.row0, u.rows);
        chunk = u.first;
    } else {
        t = find_tile(p.seqs.k_offsets, p.seqs.n_seq, p.seqs.k_rows, blockIdx.x - p.far_slots, kRows);
        if (t.first < 0 || t.first >= t.rows || (t.seq < 0 && !p.clear)) return;
        queries = t.seq < 0 ? make_int2(0, 0) : sequence_rows(p.seqs.q_offsets, p.seqs.q_rows, t.seq);
    }
    const long long row0 = static_cast<long long>(t.row0) + t.first;
    const int have = min(kRows, t.rows - t.first), shift = t.rows - queries.y;
    const int near = near_queries(t.first, have, t.rows, queries.y, w.window);
    const bool split = far_chunks(p, near, queries.y) && t.first == 0;  // the far queries are others' work
    // queries from the tile's first key to the end of its last key's window (sinks: to the end)
    int i0 = max(t.first - shift, 0), i1 = t.first < w.sinks && !split ? queries.y : near;
    if (far >= 0) {
        i0 = max(near, chunk);
        i1 = min(queries.y, chunk + p.far_chunk);
        if (!split || i0 >= i1) return;
    }
    const int tiles = max(i1 - i0 + per_tile - 1, 0) / per_tile;
    // queries of tile i that exist
    const auto queries_of = [&](int i) { return min(per_tile, i1 - i0 - i * per_tile); };

    const uint32_t base = uniform((shared_address(shared_raw) + 1023) & ~1023u);
    const uint32_t ks = base, vs = ks + kTile, qs = vs + kTile, gs = qs + kStages * kTile, rows_at = gs + kStages * kTile,
                   bars = rows_at + kStages * 2 * kRows * 4;
    const uint32_t k_full = bars, raw = bars + 8, s_full = bars + 16, s_read = bars + 24, dp_full = bars + 32, ds_full = bars + 48,
                   done = bars + 80, all_done = bars + 88, q_full = bars + 96, q_empty = q_full + 8 * kStages, g_full = q_empty + 8 * kStages,
                   g_empty = g_full + 8 * kStages, rows_full = g_empty + 8 * kStages, tmem_at = rows_full + 8 * kStages;
    const int warp = uniform(threadIdx.x / 32), lane = threadIdx.x % 32;
    if (warp == 8) {
        tmem_alloc(tmem_at, 512);
        if (lane == 0) {
            barrier_init(k_full, 1);
            barrier_init(raw, 1);
            barrier_init(s_full, 1);
            barrier_init(s_read, 256);
            for (int i = 0; i < 2; ++i) {
                barrier_init(dp_full + 8 * i, 1);
                barrier_init(ds_full + 16 * i, 256);
                barrier_init(ds_full + 16 * i + 8, 256);
            }
            barrier_init(done, 1);
            barrier_init(all_done, 1);
            for (int i = 0; i < kStages; ++i) {
                barrier_init(q_full + 8 * i, 1);
                barrier_init(q_empty + 8 * i, 1);
                barrier_init(g_full + 8 * i, 1);
                barrier_init(g_empty + 8 * i, 1);
                barrier_init(rows_full + 8 * i, 32);
            }
            barrier_init_done();
        }
        __syncwarp();
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));
    tmem = uniform(tmem);
    constexpr int kBuffers = kDim == 64 ? 2 : 1;  // of dP (each with barriers of its own: the threads may be a tile ahead of the products)
    const uint32_t dp_at = tmem + 128, dv_at = tmem + 512 - 2 * kDim, dk_at = tmem + 512 - kDim;
    bool ok = true;

    if (warp >= 8) give_registers();
    if (warp == 9) {
        if (lane == 0 && tiles > 0) {
            barrier_expect(k_full, 2 * kTile);
            for (int x = 0; x < kPanels; ++x) {
                copy_box(ks + x * kPanel, &maps.k, x * 64, kv, static_cast<int>(row0), k_full);
                copy_box(vs + x * kPanel, &maps.v, x * 64, kv, static_cast<int>(row0), k_full);
            }
        }
        // rows that no copy writes, where the group does not divide 128
        const int full = per_tile * group;
        if (full < kRows)
            for (int i = 0; i < kStages; ++i) {
                clear_rows(qs + i * kTile, kPanels, full);
                clear_rows(gs + i * kTile, kPanels, full);
            }
        int cleared = 0;
        for (int i = 0; i < tiles && ok; ++i) {
            const int st = i % kStages, n = queries_of(i), y = queries.x + i0 + i * per_tile;
            const uint32_t free = (i / kStages & 1) ^ 1;
            for (int u = 0; u < 2 && ok; ++u) {  // queries, then gradients of the results
                const uint32_t tile = (u ? gs : qs) + st * kTile, done = (u ? g_full : q_full) + 8 * st, bar = n < per_tile ? raw : done;
                ok = barrier_wait((u ? g_empty : q_empty) + 8 * st, free);
                if (ok && lane == 0) {
                    barrier_expect(bar, kPanels * full * 128);
                    for (int x = 0; x < kPanels; ++x) copy_box(tile + x * kPanel, u ? &maps.dout : &maps.q, x * 64, kv * group, y, bar);
                }
                __syncwarp();
                if (ok && n < per_tile) {
                    ok = barrier_wait(raw, cleared++ & 1);
                    clear_rows(tile, kPanels, n * group);
                    if (lane == 0) barrier_arrive(done);
                }
            }
        }
    } else if (warp == 10) {
        // lse and delta of the tiles' rows
        for (int i = 0; i < tiles && ok; ++i) {
            const int st = i % kStages;
            // (free when the queries of the stage are: their last product comes behind ds_full)
            ok = barrier_wait(q_empty + 8 * st, (i / kStages & 1) ^ 1);
            if (!ok) break;
            fetch_rows(p, p.delta, static_cast<long long>(queries.x) + i0 + i * per_tile, kv * group, group, queries_of(i),
                       rows_at + st * 2 * kRows * 4);
            barrier_arrive(rows_full + 8 * st);
        }
    } else if (warp == 8) {
        const uint32_t scores = product_descriptor<T>(kRows, false), sums = product_descriptor<T>((w.dim + 15) / 16 * 16, true);
        const int steps = (w.dim + 15) / 16;
        const uint32_t one = elect_one();
        const auto issue = [&](uint32_t d, uint32_t a, uint32_t b, uint32_t bar) {
            const uint64_t x = tile_descriptor(a, 16), y = tile_descriptor(b, 16);
#pragma unroll
            for (int s = 0; s < kDim / 16; ++s)
                if (s < steps) {
                    const uint32_t at = (s / 4 * kPanel + s % 4 * 32) >> 4;
                    product(one, d, x + at, y + at, scores, s > 0);
                }
            products_arrive(one, bar);
        };
        if (tiles > 0) {
            ok = barrier_wait(k_full, 0) && barrier_wait(q_full, 0) && barrier_wait(g_full, 0);
            tmem_fence_after();
            if (ok) {
                issue(tmem, ks, qs, s_full);
                issue(dp_at, vs, gs, dp_full);
            }
        }
        for (int i = 0; i < tiles && ok; ++i) {
            const int st = i % kStages, next = (i + 1) % kStages;
            const uint32_t next_full = (i + 1) / kStages & 1, buf = dp_at + i % kBuffers * kRows;
            const bool more = i + 1 < tiles;
            if (more) {
                ok = barrier_wait(q_full + 8 * next, next_full) && barrier_wait(s_read, i & 1);
                if (!ok) break;
                tmem_fence_after();
                issue(tmem, ks, qs + next * kTile, s_full);
            }
            ok = i == 0 || kBuffers == 1 || barrier_wait(done, (i - 1) & 1);
            if (!ok) break;
            if (kBuffers == 2 && more) {
                ok = barrier_wait(g_full + 8 * next, next_full);
                if (!ok) break;
                issue(dp_at + (i + 1) % 2 * kRows, vs, gs + next * kTile, dp_full + (i + 1) % 2 * 8);
            }
            const uint64_t x = tile_descriptor(qs + st * kTile, kPanel), y = tile_descriptor(gs + st * kTile, kPanel);
#pragma unroll
            for (int piece = 0; piece < 2; ++piece) {  // 32 of each warpgroup's 64 columns
                ok = ok && barrier_wait(ds_full + i % kBuffers * 16 + 8 * piece, i / kBuffers & 1);
                tmem_fence_after();
                if (ok)
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const int s = u / 2 % 2 * 4 + piece * 2 + u % 2;
                        product_from_tmem(one, u < 4 ? dv_at : dk_at, buf + s / 4 * 64 + s % 4 * 8 + (u < 4 ? 32 : 0), (u < 4 ? y : x) + s * 128, sums,
                                          i > 0 || piece > 0 || u % 4 > 0);
                    }
            }
            if (!ok) break;
            products_arrive(one, done);
            if (!more) products_arrive(one, all_done);
            products_arrive(one, q_empty + 8 * st);
            products_arrive(one, g_empty + 8 * st);
            if (kBuffers == 1) {
                ok = barrier_wait(done, i & 1) && (!more || barrier_wait(g_full + 8 * next, next_full));
                if (!ok) break;
                if (more) issue(dp_at, vs, gs + next * kTile, dp_full);
            }
            __syncwarp();
        }
    } else if (warp < 8) {
        take_registers();
        const int half = warp / 4, r = threadIdx.x % 128, key = t.first + r;
        const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
        const uint32_t s_at = tmem + lanes + half * 64;
        const float s2 = w.scale * kLog2e;
        for (int i = 0; i < tiles; ++i) {
            const int st = i % kStages, q0 = i0 + i * per_tile, n = queries_of(i), pos0 = q0 + shift;
            // columns are (query, head): the queries that see this thread's key are a range of them
            const bool whole = n * group == kRows && pos0 >= t.first + have - 1 && (pos0 + n - 1 - t.first < w.window || t.first + have <= w.sinks);
            const int a = min(max(key - pos0, 0), n), b = key < w.sinks ? n : max(min(n, key - pos0 + w.window), 0);
            const Range range = {a * group - half * 64, b * group - half * 64, 0};
            const uint32_t d_at = dp_at + lanes + i % kBuffers * kRows + half * 64;
            const uint32_t off_at = rows_at + (st * 2 * kRows + half * 64) * 4, delta_at = off_at + kRows * 4;
            ok = barrier_wait(rows_full + 8 * st, i / kStages & 1) && barrier_wait(s_full, i & 1);
            if (!ok) break;
            tmem_fence_after();
            uint32_t s[64], d[64];
            tmem_load32<0>(s_at, s);
            tmem_load32<32>(s_at + 32, s);
            tmem_wait_load32<0>(s);
            tmem_wait_load32<32>(s);
            tmem_fence_before();
            barrier_arrive(s_read);
            const auto weight_off = [&](int j) { return load_pair(off_at + j * 4); };
            uint32_t packed[32];
            if (whole) {
                weights_in_place<0, kByFmaInPairs>(s, s2, weight_off);
                weights_in_place<32, kByFmaInPairs>(s, s2, weight_off);
            } else {
                weights_in_place<0, 0>(s, s2, weight_off);
                weights_in_place<32, 0>(s, s2, weight_off);
                hide(s, range, 0u);  // (the weights, not the scores: a query whose lse is NaN leaves the keys alone that it does not see)
            }
#pragma unroll
            for (int j = 0; j < 64; j += 2) packed[j / 2] = pack2<T>(__uint_as_float(s[j]), __uint_as_float(s[j + 1]));
            ok = barrier_wait(dp_full + i % kBuffers * 8, i / kBuffers & 1);
            if (!ok) break;
            tmem_fence_after();
            tmem_load32<0>(d_at, d);
            tmem_load32<32>(d_at + 32, d);
            tmem_wait_load32<0>(d);
            tmem_wait_load32<32>(d);
            if (!whole) hide(d, range, 0u);
            // over this thread's part of dP: 32 columns of dS, 32 of P
            const auto minus = [&](int j) { return load_pair(delta_at + j * 4); };
            tmem_store32<0>(d_at + 32, packed);
            gradients_in_place<T, 0>(s, d, minus);
            tmem_store16<0>(d_at, s);
            tmem_wait_store();
            tmem_fence_before();
            barrier_arrive(ds_full + i % kBuffers * 16);
            gradients_in_place<T, 32>(s, d, minus);
            tmem_store16<16>(d_at + 16, s);
            tmem_wait_store();
            tmem_fence_before();
            barrier_arrive(ds_full + i % kBuffers * 16 + 8);
        }
        if (ok && tiles > 0) {
            // (not `done`, which may still be two tiles behind the threads: a wait for its last phase would take an earlier one for it)
            ok = barrier_wait(all_done, 0);
            tmem_fence_after();
        }
        const uint32_t sum_at = (half == 0 ? dv_at : dk_at) + lanes;
        const float factor = half == 0 ? 1.f : w.scale;
        if (split) {
            float *part = far >= 0 ? p.far_part + (static_cast<long long>(far) * w.kv_heads + kv) * 2 * kRows * w.dim
                                   : p.near_part + (static_cast<long long>(t.seq) * w.kv_heads + kv) * 2 * kRows * w.dim;
            part += (half * kRows + r) * w.dim;
#pragma unroll
            for (int x = 0; x < kDim; x += 32) {
                uint32_t o[32];
                tmem_load32<0>(sum_at + x, o);
                tmem_wait_load32<0>(o);
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                    if (r < have && x + j < w.dim)
                        *reinterpret_cast<float4 *>(part + x + j) =
                            tiles > 0 ? make_float4(__uint_as_float(o[j]) * factor, __uint_as_float(o[j + 1]) * factor,
                                                    __uint_as_float(o[j + 2]) * factor, __uint_as_float(o[j + 3]) * factor)
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        } else {
            T *out = static_cast<T *>(half == 0 ? p.dv : p.dk) + ((row0 + r) * w.kv_heads + kv) * w.dim;
#pragma unroll
            for (int x = 0; x < kDim; x += 32) store_columns(out, sum_at, x, w.dim, factor, r < have, tiles > 0);
        }
    }
    if (!ok) waits_failed = 1;
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == 8) tmem_free(tmem, 512);
}

// dK and dV of the first tiles whose far queries were worked on in chunks: the tile's own part, then the chunks' in order.
template <typename T>
__global__ void __launch_bounds__(256) add_far_gradients(const Prompt p) {
    const Window &w = p.win;
    const int seq = blockIdx.x, kv = blockIdx.y, chunk = p.far_chunk;
    const int2 keys = sequence_rows(p.seqs.k_offsets, p.seqs.k_rows, seq), queries = sequence_rows(p.seqs.q_offsets, p.seqs.q_rows, seq);
    const int have = min(kRows, keys.y), near = near_queries(0, have, keys.y, queries.y, w.window);
    if (have == 0 || !far_chunks(p, near, queries.y)) return;
    const int slot = p.seqs.q_offsets == nullptr ? 0 : queries.x / chunk + seq + 1;
    const int first = near / chunk, n = (queries.y + chunk - 1) / chunk;
    const long long size = 2ll * kRows * w.dim, step = size * w.kv_heads;
    for (int i = (blockIdx.z * 256 + threadIdx.x) * 4; i < 2 * have * w.dim; i += gridDim.z * 256 * 4) {
        const int half = i / (have * w.dim), at = i % (have * w.dim);  // row * dim + column
        const long long from = static_cast<long long>(half) * kRows * w.dim + at;
        float4 sum = *reinterpret_cast<const float4 *>(p.near_part + (static_cast<long long>(seq) * w.kv_heads + kv) * size + from);
        for (int f = first; f < n; ++f)
            vadd(sum, *reinterpret_cast<const float4 *>(p.far_part + (slot + f) * step + kv * size + from));
        store4(static_cast<T *>(half == 0 ? p.dv : p.dk) + (static_cast<long long>(keys.x) + at / w.dim) * w.kv_heads * w.dim + kv * w.dim + at % w.dim,
               sum);
    }
}

// --- host -----------------------------------------------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            return static_cast<EncodeTiled>(nullptr);
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// (A call of the driver, for which the thread must have a context: it has one behind allow_shared, a call of the runtime.  Autograd's
// threads may come here without.)
// [rows][heads][dim] in boxes of 64 columns x box_heads x box_rows; outer is x.row or x.batch.
int encode(CUtensorMap *map, int dtype, const rode_heads_t &x, long long outer, int rows, int heads, int dim, int box_heads, int box_rows) {
    const EncodeTiled fn = encoder();
    if (fn == nullptr) return fail(RODE_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t line = static_cast<cuuint64_t>(dim) * 2;
    const cuuint64_t size[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
    // (the strides of dimensions of one element are never used)
    const cuuint64_t strides[2] = {heads > 1 ? static_cast<cuuint64_t>(x.head) * 2 : line, rows > 1 ? static_cast<cuuint64_t>(outer) * 2 : line};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)}, step[3] = {1, 1, 1};
    const CUresult e = fn(map, dtype == RODE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                          const_cast<void *>(x.data), size, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (e != CUDA_SUCCESS) return fail(RODE_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", static_cast<int>(e));
    return RODE_OK;
}

// Base and strides are whole 16-byte units, as a tensor copy wants them, and no dimension repeats.
bool copyable(const rode_heads_t &x, long long outer, int rows, int heads) {
    const auto fits = [](long long stride, int n) { return n <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 39)); };
    return aligned_to(x.data, 16) && fits(x.head, heads) && fits(outer, rows);
}

template <typename F>
int by_half(int dtype, int dim, F &&f) {
    const auto g = [&](auto *type) {
        return dim <= 64 ? f(type, std::integral_constant<int, 64>()) : f(type, std::integral_constant<int, 128>());
    };
    return dtype == RODE_F16 ? g(static_cast<__half *>(nullptr)) : g(static_cast<__nv_bfloat16 *>(nullptr));
}

}  // namespace

bool tiles_take(int dtype, const Window &w) {
    return dtype != RODE_F32 && w.dim % 8 == 0 && w.dim <= 128 && w.heads / w.kv_heads <= kRows && w.scale > 0.f;
}

bool tiles_take_prompt(int dtype, const Prompt &p) {
    return tiles_take(dtype, p.win) && p.seqs.k_rows > 0 && copyable(p.q, p.q.row, p.seqs.q_rows, p.win.heads) &&
           copyable(p.k, p.k.row, p.seqs.k_rows, p.win.kv_heads) && copyable(p.v, p.v.row, p.seqs.k_rows, p.win.kv_heads);
}

bool tiles_take_backward(int dtype, const Prompt &p) {
    return tiles_take_prompt(dtype, p) && p.seqs.q_rows > 0 && copyable(p.dout, p.dout.row, p.seqs.q_rows, p.win.heads);
}

bool tiles_take_shared(int dtype, const Cached &c) {
    return tiles_take(dtype, c.win) && copyable(c.q, c.q.batch, c.batch, c.win.heads) &&
           copyable(c.pk, c.pk.row, c.prefix, c.win.kv_heads) && copyable(c.pv, c.pv.row, c.prefix, c.win.kv_heads);
}

int tiles_prompt(int dtype, const Prompt &p, cudaStream_t stream) {
    const Window &w = p.win;
    const int group = w.heads / w.kv_heads, per_tile = kRows / group;
    TileMaps maps;
    return by_half(dtype, w.dim, [&](auto *type, auto dim) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int kDim = decltype(dim)::value;
        auto *kernel = &forward_tiles<T, kDim, false>;
        if (const int e = allow_shared(kernel, forward_bytes<kDim>())) return e;
        if (const int e = encode(&maps.q, dtype, p.q, p.q.row, p.seqs.q_rows, w.heads, w.dim, group, per_tile)) return e;
        if (const int e = encode(&maps.k, dtype, p.k, p.k.row, p.seqs.k_rows, w.kv_heads, w.dim, 1, kRows)) return e;
        if (const int e = encode(&maps.v, dtype, p.v, p.v.row, p.seqs.k_rows, w.kv_heads, w.dim, 1, kRows)) return e;
        const long long items = static_cast<long long>(tile_slots(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, 2 * per_tile)) * w.kv_heads;
        if (items > INT_MAX / 2) return fail(RODE_ERR_INVALID_ARGUMENT, "rode_window_attention: too many rows and heads");
        const int ctas = static_cast<int>(std::min<long long>(items, sm_count()));
        kernel<<<ctas, kTileThreads, forward_bytes<kDim>(), stream>>>(maps, p, Cached{}, static_cast<int>(items));
        RODE_CHECK_LAUNCH("forward_tiles");
        return static_cast<int>(RODE_OK);
    });
}

// Chunks of about a tile's own work, and only where the sequences are long on average: the first tile is then at least three times the work
// of the others.  (One long sequence among many short ones, and more sinks than a tile has keys, are left whole: the same results, but the grid waits for the
// tiles of the sinks.)
FarPlan plan_far(int n_seq, bool packed, int q_rows, int kv_heads, int dim, int window, int sinks) {
    FarPlan f = {0, 0, 0, 0};
    if (sinks <= 0 || sinks > kRows || n_seq <= 0 || window > (1 << 29)) return f;
    const int chunk = std::max(1024, window + kRows);
    if (q_rows / n_seq <= 2ll * chunk) return f;
    f.chunk = chunk;
    f.slots = packed ? q_rows / chunk + n_seq + 2 : (q_rows + chunk - 1) / chunk;
    const size_t tile = 2 * sizeof(float) * kRows * dim * kv_heads;
    f.near_bytes = tile * n_seq;
    f.far_bytes = tile * f.slots;
    return f;
}

int tiles_backward(int dtype, const Prompt &p, cudaStream_t stream) {
    const Window &w = p.win;
    const int group = w.heads / w.kv_heads, per_tile = kRows / group;
    GradientMaps maps;
    return by_half(dtype, w.dim, [&](auto *type, auto dim) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int kDim = decltype(dim)::value;
        auto *rows = &query_gradient_tiles<T, kDim>;
        auto *keys = &key_gradient_tiles<T, kDim>;
        if (const int e = allow_shared(rows, backward_bytes<kDim>())) return e;
        if (const int e = allow_shared(keys, backward_bytes<kDim>())) return e;
        if (const int e = encode(&maps.q, dtype, p.q, p.q.row, p.seqs.q_rows, w.heads, w.dim, group, per_tile)) return e;
        if (const int e = encode(&maps.dout, dtype, p.dout, p.dout.row, p.seqs.q_rows, w.heads, w.dim, group, per_tile)) return e;
        if (const int e = encode(&maps.k, dtype, p.k, p.k.row, p.seqs.k_rows, w.kv_heads, w.dim, 1, kRows)) return e;
        if (const int e = encode(&maps.v, dtype, p.v, p.v.row, p.seqs.k_rows, w.kv_heads, w.dim, 1, kRows)) return e;
        const long long items = static_cast<long long>(tile_slots(p.seqs.q_offsets, p.seqs.n_seq, p.seqs.q_rows, per_tile)) * w.kv_heads;
        if (items > INT_MAX / 2) return fail(RODE_ERR_INVALID_ARGUMENT, "rode_window_attention_backward: too many rows and heads");
        const long long all = static_cast<long long>(p.seqs.q_rows) * w.heads, per_cta = 256 / (kDim / 8);
        row_deltas<T, kDim><<<static_cast<unsigned>((all + per_cta - 1) / per_cta), 256, 0, stream>>>(p);
        RODE_CHECK_LAUNCH("row_deltas");
        RODE_CUDA_TRY(launch_part(rows, dim3(static_cast<unsigned>(std::min<long long>(items, sm_count()))), kTileThreads, backward_bytes<kDim>(),
                                  stream, true, maps, p, static_cast<int>(items)));
        if (p.dk == nullptr) return static_cast<int>(RODE_OK);
        const int k_slots = tile_slots(p.seqs.k_offsets, p.seqs.n_seq, p.seqs.k_rows, kRows);
        // (Not beside dQ's grid: a grid that starts early sees what the grids before its predecessor wrote only by waiting for that one.)
        keys<<<dim3(p.far_slots + k_slots, w.kv_heads), kTileThreads, backward_bytes<kDim>(), stream>>>(maps, p);
        RODE_CHECK_LAUNCH("key_gradient_tiles");
        if (p.far_slots > 0) {
            add_far_gradients<T><<<dim3(p.seqs.n_seq, w.kv_heads, 8), 256, 0, stream>>>(p);
            RODE_CHECK_LAUNCH("add_far_gradients");
        }
        return static_cast<int>(RODE_OK);
    });
}

int tiles_shared(int dtype, const Cached &c, cudaStream_t stream) {
    const Window &w = c.win;
    const int group = w.heads / w.kv_heads, per_tile = kRows / group;
    TileMaps maps;
    return by_half(dtype, w.dim, [&](auto *type, auto dim) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int kDim = decltype(dim)::value;
        auto *kernel = &forward_tiles<T, kDim, true>;
        if (const int e = allow_shared(kernel, forward_bytes<kDim>())) return e;
        if (const int e = encode(&maps.q, dtype, c.q, c.q.batch, c.batch, w.heads, w.dim, group, per_tile)) return e;
        if (const int e = encode(&maps.k, dtype, c.pk, c.pk.row, c.prefix, w.kv_heads, w.dim, 1, kRows)) return e;
        if (const int e = encode(&maps.v, dtype, c.pv, c.pv.row, c.prefix, w.kv_heads, w.dim, 1, kRows)) return e;
        const long long items = (static_cast<long long>(c.batch) + 2 * per_tile - 1) / (2 * per_tile) * w.kv_heads * c.prefix_parts;
        if (items > INT_MAX / 2) return fail(RODE_ERR_INVALID_ARGUMENT, "rode_shared_prefix_attention: too many requests and heads");
        const int ctas = static_cast<int>(std::min<long long>(items, sm_count()));
        kernel<<<ctas, kTileThreads, forward_bytes<kDim>(), stream>>>(maps, Prompt{}, c, static_cast<int>(items));
        RODE_CHECK_LAUNCH("forward_tiles");
        return static_cast<int>(RODE_OK);
    });
}

int tiles_waits_failed(int *failed) {
    RODE_CUDA_TRY(cudaDeviceSynchronize());  // (the copy alone does not wait for streams that do not block, as torch's do not)
    RODE_CUDA_TRY(cudaMemcpyFromSymbol(failed, waits_failed, sizeof(int)));
    return RODE_OK;
}

}  // namespace rode
