// q3cu_prompt.cuh -- attention of many rows on the tensor cores: the kernel of k_prompt.cu (over bf16 caches),
// k_prompt_q8.cu (over Q8_0 caches) and k_shared.cu (what groups of sequences share).
#pragma once

#include "q3cu_f16.cuh"
#include "q3cu_paged.cuh"
#include "q3cu_split.cuh"
#include "q3cu_tcgen05.cuh"
#include "q3cu_tma.h"

#include <type_traits>

namespace q3 {

constexpr int PT_ROWS = 128, PT_KEYS = 128;                  // rows of a tile, keys of a tile
enum PromptMode { PT_ITEMS, PT_CLUSTER, PT_SHARED };
constexpr int PT_WHOLE = 8;                                  // key tiles from which on an item may be shared
constexpr uint32_t PT_HALF = PT_ROWS * 128;                  // bytes of 128 rows x 64 elements
constexpr uint32_t PT_TILE = 2 * PT_HALF;                    // 32 KB
constexpr uint32_t PT_RAW = PT_KEYS * HD + PT_KEYS * 8;      // Q8_0: codes and scales of a tile of keys or values
// Of a bf16 cache or a Q8_0 one: threads, K / V buffers in flight, and stages of codes.
template <bool Q8> struct PromptShape {
    static constexpr int THREADS = Q8 ? 16 * 32 : 12 * 32, NS = Q8 ? 3 : 5, RAWS = Q8 ? 3 : 0;
    static constexpr size_t SMEM = size_t(2 + NS) * PT_TILE + RAWS * PT_RAW + 1024;
};
// Instruction descriptors: f32 accumulator, bf16 A and B, M = N = 128; B K-major (K) or MN-major (V).
constexpr uint32_t PT_IDESC = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 / 8) << 17) | (uint32_t(128 / 16) << 24);
constexpr uint32_t PT_IDESC_V = PT_IDESC | (1u << 16);
constexpr uint32_t PT_F16 = (1u << 7) | (1u << 10);          // the bits that say bf16 where f16 has none
constexpr int PT_BIAS = 7;                                   // Q8_0: probabilities are times 2^7 in f16, at most 2^15
constexpr int PT_DEEP = 120;                                 // Q8_0: O lowered by more may leave binary32
constexpr int PT_SLACK = 8;                                  // Q8_0: the most by which values' probabilities are lowered (2^-8)
constexpr float PT_LOG2 = ATT_SCALE * 1.44269504088896341f;  // scores to base-2 exponents
constexpr float PT_LAZY = 8.0f / PT_LOG2;                    // growth of the maximum (as a raw score) that rescales O

// 2^x of a pair without the special-function unit, which is as busy as the tensor cores when every exponential goes
// through it: x = n + f with n whole and |f| <= 1/2, a polynomial for 2^f, times 2^n.  The coefficients are the minimax
// fit of degree 3 to 2^f (relative error 7.5e-5, a fiftieth of the bf16 rounding that follows), found by Remez exchange.
// Below 2^-126.5 the result is 0 (n = -127 makes the exponent's bits 0), as a masked score of -inf has to give; a NaN
// stays one.
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void exp2_poly(float &x, float &y) {
    const f2 v = pk2(max_nan(x, -127.0f), max_nan(y, -127.0f)), magic = pk2(12582912.0f, 12582912.0f);   // 1.5 * 2^23
    const f2 t = add2(v, magic), f = sub2(v, sub2(t, magic));
    f2 p = pk2(0.0551716685295105f, 0.0551716685295105f);
    p = fma2(p, f, pk2(0.2426111251115799f, 0.2426111251115799f));
    p = fma2(p, f, pk2(0.6932609677314758f, 0.6932609677314758f));
    p = fma2(p, f, pk2(0.9999280571937561f, 0.9999280571937561f));
    float t0, t1;
    up2(t, t0, t1);                                          // n in the low bits
    up2(mul2(p, pk2(__uint_as_float((__float_as_uint(t0) << 23) + 0x3f800000u),
                    __uint_as_float((__float_as_uint(t1) << 23) + 0x3f800000u))), x, y);
}
constexpr uint64_t PT_AGAIN_NS = 1000000000;                 // the longest that a warp computes rows again: others wait for it
constexpr int PT_POLY = 8;                                   // one pair of exponentials in PT_POLY / 2 by polynomial (Q8_0:
                                                             // none, the conversion needs the same pipes)

// The item of a round, as warp 9 announces it (s < 0: no more), with the key tiles of each row tile.
struct PromptRound : PromptItem {
    int nt[2];
    __device__ __forceinline__ int from() const { return 0; }
};
// Of an item that `parts` CTAs share: nt counts this CTA's key tiles, the first of which is j0.  (One that has no part
// has no rows either.)
struct PromptShare : PromptItem {
    int nt[2], j0, parts;
    __device__ __forceinline__ int from() const { return j0; }
};
// Of what a group of sequences shares (PT_SHARED): `s` is the group's first sequence, a row is a sequence and sees all
// `len` keys, or is none of this item's where it holds fewer; `dst` is where its results go.
struct PromptPrefix : PromptItem {
    int nt[2], j0;
    int64_t dst;
    __device__ __forceinline__ int from() const { return j0; }
};
// Asks for the work of a CTA of this launch that has not started (it then never does); the answer arrives on `bar`
// (16 bytes).  After an answer of none, nothing more may be asked.
__device__ __forceinline__ void take_over_cta(ulonglong2 *answer, uint64_t *bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 :: "r"(smem_addr(answer)), "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ int64_t taken_cta(const ulonglong2 &answer) {     // its blockIdx.x, or -1
    uint32_t got, x = 0;
    asm volatile(
        "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\tmov.b128 h, {%2, %3};\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
        : "=r"(got), "=r"(x) : "l"(answer.x), "l"(answer.y));
    return got ? int64_t(x) : -1;
}

// A place in the ring, in the order of use: buffer and how often (parity) it was used before.
template <int NS> struct RingAt {
    int st = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next() {
        if (++st == NS) st = 0, ph ^= 1u;
    }
};

// ---- what groups of sequences share ---------------------------------------------------------------
// The items of a PT_SHARED launch, in the order group, kv head, block of `per_block` sequences; each is as many units as
// the shared positions have key tiles.  All units are cut into one run per CTA (PagedCut).  A run that covers all of an item
// leaves its rows' results at row (sequence, head); one that begins or ends inside leaves them in slot 2 run, or 2 run + 1 if
// the run began with another item, of the slots behind.
// The plan of a call, which its first launch makes (shared_plan_kernel): the groups that share something, with the units before
// them (of one kv head), and of each sequence the span and units of its own part (TailSeqs) and its group.
struct SharedEntry {
    int first, count, len;   // first sequence, sequences, positions
    int pad;
    int64_t units;
};
struct SharedPlan {
    int2 *spans;             // [n_seqs]
    int64_t *before;         // [n_seqs + 1]
    int *entry;              // [n_seqs]: the entry whose first sequence it is
    SharedEntry *entries;    // [shared_entries(n_seqs)]
    SharedEntry *of;         // [n_seqs]: the entry of a sequence (where its span begins behind 0)
    SharedEntry *all;        // count: the entries; units: of all
};
__host__ __device__ __forceinline__ int shared_entries(int n_seqs) { return n_seqs / 2 + 1; }
struct SharedOut {
    SharedPlan plan;
    float *rows;             // of SHARED_ROW floats: [n_seqs][n_heads], then [runs][2][slot_rows]
    int slot_rows;
};
struct SharedWalk {
    SharedEntry e;
    int index, head, block, tile, tiles, blocks;             // index of the entry, tiles of its positions, blocks of its sequences
    __device__ __forceinline__ void enter(const FastDiv &per_block) {
        tiles = (e.len + PT_KEYS - 1) / PT_KEYS;
        blocks = per_block(e.count - 1) + 1;
    }
};
// A run's units [u, u1) of all, and the place of u (one warp; every lane returns it).
__device__ __forceinline__ SharedWalk shared_run(const SharedPlan &plan, const PagedKV &c, const FastDiv &per_block, int n_seqs,
                                                 int run, int runs, int64_t &u, int64_t &u1) {
    const int lane = threadIdx.x & 31, room = shared_entries(n_seqs);
    const SharedEntry all = *plan.all;
    SharedEntry mine = plan.entries[min(lane, room - 1)];    // under way together
    SharedWalk w = {};
    const PagedCut cut(all.units * c.n_kv, runs);
    u = cut.begin(run);
    u1 = cut.begin(run + 1);
    if (u == u1) return w;
    for (int i0 = 0; i0 < all.count; i0 += 32) {
        if (i0) mine = plan.entries[min(i0 + lane, room - 1)];
        const unsigned hit = __ballot_sync(FULL, i0 + lane < all.count && mine.units * c.n_kv <= u);
        const int64_t end = i0 + 32 < all.count ? plan.entries[i0 + 32].units : all.units;
        if (u >= end * c.n_kv) continue;
        const int l = 31 - __clz(hit);                       // the last that begins at or before u
        w.index = i0 + l;
        w.e.first = __shfl_sync(FULL, mine.first, l);
        w.e.count = __shfl_sync(FULL, mine.count, l);
        w.e.len = __shfl_sync(FULL, mine.len, l);
        w.enter(per_block);
        const int64_t at = u - __shfl_sync(FULL, mine.units, l) * c.n_kv, item = quot(at, w.tiles);
        w.tile = int(at - item * w.tiles);
        w.head = int(quot(item, w.blocks));
        w.block = int(item - int64_t(w.head) * w.blocks);
        return w;
    }
    u = u1;
    return w;
}
// To the item behind.
__device__ __forceinline__ void shared_next(const SharedPlan &plan, const PagedKV &c, const FastDiv &per_block, SharedWalk &w) {
    w.tile = 0;
    if (++w.block < w.blocks) return;
    w.block = 0;
    if (++w.head < c.n_kv) return;
    w.head = 0;
    w.e = plan.entries[++w.index];
    w.enter(per_block);
}

struct NoOrder {             // in place of a PromptOrder
    __device__ __forceinline__ NoOrder(const PagedSeqs &, const PagedKV &, int, const FastDiv &, int, uint32_t *) {}
    __device__ __forceinline__ PromptItem find(int64_t) { return {}; }
};

// ---- Q8_0 tiles and their queries as f16 ------------------------------------------------------------
// What the rows of a converted tile were multiplied by: 2^(e - 7), and whether their scales differ by more than 2^24.
struct TileLift {
    int e;
    bool uneven;
};
// The lift of 128 rows by their scales, of which those before `rows` count (one warp; every lane returns it): by the power of
// two that brings the largest finite one to [2^14, 2^15).  Whether they are uneven is found if COMPARE.
template <bool COMPARE> __device__ __forceinline__ TileLift q8_lift(const uint8_t *raw, int rows) {
    const int lane = threadIdx.x & 31;
    uint32_t w[8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const uint4 v = *reinterpret_cast<const uint4 *>(raw + PT_KEYS * HD + 32 * lane + 16 * x);
        w[4 * x] = v.x, w[4 * x + 1] = v.y, w[4 * x + 2] = v.z, w[4 * x + 3] = v.w;
    }
    if (rows < PT_KEYS)
#pragma unroll
        for (int y = 0; y < 8; ++y)
            if (4 * lane + y / 2 >= rows) w[y] = 0;
    // Without its sign a binary32's bits order it, the exponent on top.  2^24 more, and no numbers wrap around to below all
    // others; one less, and zero does to above (where no numbers are already).
    uint32_t top = 0, low = 0xffffffffu;
#pragma unroll
    for (int y = 0; y < 8; ++y) {
        top = max(top, 2 * w[y] + (1u << 24));
        if (COMPARE) low = min(low, 2 * w[y] - 1);
    }
    top = __reduce_max_sync(FULL, top);
    if (COMPARE) low = __reduce_min_sync(FULL, low);
    const int top_e = max(int(top >> 24) - 1, 0), low_e = int((low + 1) >> 24);          // (low_e: 0 without any, as is top_e)
    return {min(141 - top_e, 126), low < 0xfeffffffu && top_e - low_e > 24};
}
// Whether a row that sees the first n keys of a sequence lost bits to others: behind them in the same tile lies a scale that
// is more than 2^24 times the largest it sees there, of keys or of values (one warp; every lane returns it).  Where it sees
// none but zeros there, nothing of the tile can be lost.
__device__ __forceinline__ bool larger_behind(const PagedKV &c, const PagedSeqs &b, int s, int head, int n, int len) {
    const int tile = n / PT_KEYS * PT_KEYS, t = tile + 4 * (threadIdx.x & 31), end = min(len, tile + PT_KEYS);
    uint32_t seen[2] = {0, 0}, hidden[2] = {0, 0};           // of K and V; magnitudes compare as their bits do
    const int page = t < end ? paged_page(b, c, s, t, nullptr) : -1;
    if (page >= 0) {
        const int64_t at = paged_scale_at(c, page, head, t); // four positions, which one page holds
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint4 *p = reinterpret_cast<const uint4 *>((x ? c.v_scale : c.k_scale) + at);
            const uint4 lo = p[0], hi = p[1];
            const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                const uint32_t bits = w[y] & 0x7fffffffu;
                if (t + y / 2 >= end || bits >= 0x7f800000u) continue;
                if (t + y / 2 < n) seen[x] = max(seen[x], bits);
                else hidden[x] = max(hidden[x], bits);
            }
        }
    }
    bool larger = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const uint32_t a = __reduce_max_sync(FULL, seen[x]), z = __reduce_max_sync(FULL, hidden[x]);
        larger |= a && (z >> 23) > (a >> 23) + 24;
    }
    return larger;
}
// 128 rows' codes (128-byte swizzle) and scales at `raw` become the 32 KB f16 operand tile at `to`, by four warps: a lane
// takes 16 codes of eight rows.  Rows from `rows` on are zeros.  The lifted scales are rounded to f16 (2^-11), code / 128 is
// exact, the product is rounded once more: 1.75 instructions an element.  A word's codes become the pairs (0, 2) and (1, 3), one
// logical operation each and a permutation for the second (in byte order each takes a permutation, and the signs one
// operation more): of four dimensions the middle two change places, in the queries (q_tile_f16) and the result (column) as
// well.
__device__ __forceinline__ void q8_tile(const uint8_t *raw, uint8_t *to, int rows, int e) {
    const int lane = threadIdx.x & 31, key0 = int(threadIdx.x >> 5 & 3) * 32 + (lane & 7);
    const float *scales = reinterpret_cast<const float *>(raw + PT_KEYS * HD);
    const float up = __uint_as_float(uint32_t(e + 127) << 23);
    // Not unrolled: the warps of an SM run several pieces of code at once, and the instructions they do not have at hand cost
    // more than the wait for these loads (253 against 244 us for the chunks of prompts; all codes loaded ahead 243 against 228 on
    // another GPU).
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        const int key = key0 + 8 * i;
        uint4 v[2];                                          // codes 16 ch .., ch = lane / 8 and 4 further
#pragma unroll
        for (int half = 0; half < 2; ++half)
            v[half] = *reinterpret_cast<const uint4 *>(raw + key * HD + ((((lane >> 3) + 4 * half) ^ (key0 & 7)) << 4));
        const float2 sc = *reinterpret_cast<const float2 *>(scales + 2 * key);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float s = key < rows ? (half ? sc.y : sc.x) * up : 0.0f;
            const uint32_t s2 = pack_f16(s, s);
            const uint32_t words[4] = {v[half].x, v[half].y, v[half].z, v[half].w};
            uint32_t w[8];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                w[2 * y] = mul_f16(codes_f16_128th(words[y]), s2);
                w[2 * y + 1] = mul_f16(codes_f16_128th(__byte_perm(words[y], 0, 0x4341)), s2);
            }
            uint8_t *row = to + half * PT_HALF + key * 128;  // 64 elements, chunks of 8
            const int c0 = 2 * (lane >> 3);
            *reinterpret_cast<uint4 *>(row + ((c0 ^ (key & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4 *>(row + (((c0 + 1) ^ (key & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
}
// Where dimension x of a head is in the result of a Q8_0 tile's product.
template <bool Q8> __host__ __device__ constexpr int column(int x) { return Q8 && ((x & 3) == 1 || (x & 3) == 2) ? x ^ 3 : x; }
// The bf16 queries of a row tile become f16 in their places, each row lifted so that its largest element lies in
// [2^14, 2^15); one thread a row, its 16-byte chunks in an order in which the lanes' lie in different banks.  Returns the
// inverse of the row's lift.
__device__ __forceinline__ float q_tile_f16(uint8_t *tile, int row) {
    uint8_t *at = tile + row * 128;
    auto chunk = [&](int x) { return reinterpret_cast<uint4 *>(at + (x >> 3) * PT_HALF + (((x ^ row) & 7) << 4)); };
    uint32_t top = 0;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        const uint4 v = *chunk(x);
        top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
    }
    top = max(top & 0xffffu, top >> 16) << 16;
    const float up = lift(top);
#pragma unroll
    for (int x0 = 0; x0 < 16; x0 += 4) {
        uint4 v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = *chunk(x0 + x);
        auto low = [&](uint32_t a, uint32_t b) { return pack_f16(bf16_to_f32(a & 0xffffu) * up, bf16_to_f32(b & 0xffffu) * up); };
        auto high = [&](uint32_t a, uint32_t b) {
            return pack_f16(__uint_as_float(a & 0xffff0000u) * up, __uint_as_float(b & 0xffff0000u) * up);
        };
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *chunk(x0 + x) = make_uint4(low(v[x].x, v[x].y), high(v[x].x, v[x].y), low(v[x].z, v[x].w), high(v[x].z, v[x].w));
    }
    return lift_back(top);
}

// PT_ITEMS: a CTA takes items one after the other; PT_CLUSTER: clusters of `ctas` CTAs, each with one item; PT_SHARED: a run
// of what groups of sequences share.  Q8: over a Q8_0 cache (tmks, tmvs: its scales).
template <PromptMode MODE, bool Q8>
__global__ void __launch_bounds__(PromptShape<Q8>::THREADS, 1)
prompt_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                 const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmks,
                 const __grid_constant__ CUtensorMap tmvs, const SharedOut sh, const PagedKV c, const PagedSeqs b, int rows,
                 const uint16_t *q, int64_t q_stride, int n_heads, int group, const FastDiv per_block,
                 const FastDiv by_group, int ctas, uint16_t *out, uint32_t *status) {
    constexpr bool SPLIT = MODE == PT_CLUSTER, SHARED = MODE == PT_SHARED;
    constexpr int PT_NS = PromptShape<Q8>::NS, PT_THREADS = PromptShape<Q8>::THREADS, RAWS = PromptShape<Q8>::RAWS;
    typedef RingAt<PT_NS> RingAt;
    typedef typename std::conditional<Q8, q8raw, bf16raw>::type Cached;
    typedef typename std::conditional<SPLIT, PromptShare, typename std::conditional<SHARED, PromptPrefix, PromptRound>::type>::type Round;
    extern __shared__ uint8_t pt_dyn[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pt_dyn) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = smem + 2 * PT_TILE, *raw = ring + PT_NS * PT_TILE;       // raw: Q8_0 codes and scales
    __shared__ __align__(8) uint64_t q_full, q_empty, full[PT_NS], empty[PT_NS], s_full[2], p_full[2][2], o_full[2],
        o_empty[2], item_full[2], item_empty[2], taken, tail_go, tail, drain, raw_full[Q8 ? RAWS : 1], raw_empty[Q8 ? RAWS : 1],
        q_ready, lifts[2];
    // Q8_0: the inverse lifts of the queries' rows (by item), and of the tiles in turn: keys' inverse, values' exponent
    __shared__ float q_back[Q8 ? 2 : 1][Q8 ? 2 * PT_ROWS : 1], k_back[2];
    __shared__ int v_lift[2];
    __shared__ bool rough[2];                                // scales of keys or values are uneven
    __shared__ Round item_sh[2];
    __shared__ ulonglong2 taken_sh;
    __shared__ uint32_t tmem_sh;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 1);
        mbar_init(&q_ready, 4);
        for (int i = 0; i < PT_NS; ++i) {
            mbar_init(&full[i], Q8 ? 4 : 1);                 // Q8_0: the warps that convert
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < RAWS; ++i) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], 4);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t][0], 4);
            mbar_init(&p_full[t][1], 4);
            mbar_init(&o_full[t], 1);
            mbar_init(&o_empty[t], 4);
            mbar_init(&item_full[t], 1);
            mbar_init(&lifts[t], 1);
            mbar_init(&item_empty[t], Q8 ? 13 : 10);         // warps 0-7, 8 and 10, or 12-15
        }
        mbar_init(&taken, 1);
        mbar_init(&tail_go, 1);
        mbar_init(&tail, 1);
        mbar_init(&drain, 1);
        mbar_init_fence();
    }
    if (warp == 8) tc_alloc512(&tmem_sh);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tmem_sh;
    griddep_wait();
    if constexpr (SHARED) griddep_launch_dependents();

    const int qt = PT_ROWS / group;                          // queries of a tile
    float2 stat = make_float2(-INFINITY, -1.0f);             // SPLIT: maximum and sum of this thread's row, -1: given up
    [[maybe_unused]] float part_back = 1.0f;                 // and what its O is to be multiplied by (Q8_0),
    [[maybe_unused]] int part_redo = 0;                      // and whether the part lost bits
    // the item of a round, copied from its announcement; false after the last, or if a wait gave up
    auto next_item = [&](int round, Round &it, bool whole_warp) -> bool {
        bool ok = mbar_wait(&item_full[round & 1], uint32_t(round >> 1) & 1u, !whole_warp || lane == 0 ? status : nullptr);
        if (whole_warp) ok = __all_sync(FULL, ok);
        if (!ok) return false;
        it = item_sh[round & 1];
        if (whole_warp) __syncwarp();
        if (!whole_warp || lane == 0) mbar_arrive(&item_empty[round & 1]);
        return it.s >= 0;
    };

    // Registers move to the softmax: 256 threads x 208 + 128 x 88 is the launch's 384 x 168, 256 x 184 + 256 x 72 its
    // 512 x 128.
    if (warp >= 8) {
        if constexpr (Q8) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 9) {
            // ---- items and copies ------------------------------------------------------------
            const int br = min(1 << c.page_shift, PT_KEYS), nb = PT_KEYS / br;  // rows of a box, boxes of a tile
            // lane = box: column half lane / nb, positions lane % nb
            // (Q8_0: codes, then scales)
            const int box = lane % nb, half = lane / nb;
            typename std::conditional<Q8, ::q3::RingAt<Q8 ? RAWS : 1>, RingAt>::type at;
            int entries = 0, qs = 0;                         // copies of tiles and of Q so far
            bool ok = true;
            // PT_SHARED: this CTA's run [u, u1), and the place of u
            int64_t u = 0, u1 = 0;
            [[maybe_unused]] SharedWalk walk = {};
            [[maybe_unused]] int fragment = 0;
            auto prefix_item = [&](Round &it) {              // the run's next item, or a part of one
                it.s = -1;
                it.nt[0] = it.nt[1] = 0;
                if constexpr (SHARED) {
                    if (u == u1) return;
                    const int tiles = int(min(int64_t(walk.tiles - walk.tile), u1 - u));
                    it.s = it.base = walk.e.first;
                    it.head = walk.head;
                    it.rows = walk.e.count;
                    it.first = walk.block * 2 * qt;
                    it.len = walk.e.len;
                    it.pos0 = 0;
                    it.j0 = walk.tile;
                    for (int t = 0; t < 2; ++t) it.nt[t] = it.first + t * qt < it.rows ? tiles : 0;
                    it.dst = tiles == walk.tiles ? -1 : (2 * int64_t(blockIdx.x) + (fragment > 0)) * sh.slot_rows;
                    ++fragment;
                    u += tiles;
                    if (u < u1) shared_next(sh.plan, c, per_block, walk);
                }
            };
            if constexpr (SHARED) {
                walk = shared_run(sh.plan, c, per_block, b.n_seqs, int(blockIdx.x), int(gridDim.x), u, u1);
            }
            typedef typename std::conditional<SHARED, NoOrder, PromptOrder>::type Order;
            Order order(b, c, rows, per_block, PT_KEYS, status);
            PromptItem item = order.find(SPLIT ? blockIdx.x / unsigned(ctas) : blockIdx.x);
            // The first item is this CTA's own; the others are those of CTAs that have not started.  One is taken over
            // when the copies for the item before are nearly all under way: no earlier, so that the CTA that is done
            // first gets the next item, and no later, since finding it takes some thousand cycles.
            auto take_over = [&](int round) -> PromptItem {
                PromptItem none;
                none.s = -1;
                if constexpr (SPLIT || SHARED) return none;
                if (lane == 0) {
                    fence_proxy_async_smem();
                    mbar_arrive_expect_tx(&taken, 16);
                    take_over_cta(&taken_sh, &taken);
                }
                ok = __all_sync(FULL, mbar_wait(&taken, uint32_t(round) & 1u, lane == 0 ? status : nullptr));
                if (!ok) return none;
                const int64_t index = taken_cta(taken_sh);
                __syncwarp();
                return index < 0 ? none : order.find(index);
            };
            for (int round = 0; ok; ++round) {
                Round it;
                if constexpr (SHARED) prefix_item(it);
                else static_cast<PromptItem &>(it) = item, it.nt[0] = it.nt[1] = 0;
                for (int t = 0; t < 2 && it.s >= 0 && !SHARED; ++t) {
                    const int first = it.first + t * qt, last = min(first + qt, it.rows) - 1;
                    if (last >= first) it.nt[t] = (it.seen(last) + PT_KEYS - 1) / PT_KEYS;
                }
                if constexpr (SPLIT) {
                    const int all = max(it.nt[0], it.nt[1]), rank = int(blockIdx.x % unsigned(ctas));
                    it.parts = it.s < 0 ? 1 : prompt_parts(ctas, all, PT_WHOLE);
                    const bool mine = rank < it.parts;
                    it.j0 = mine ? prompt_part(all, it.parts, rank) : 0;
                    const int end = mine ? prompt_part(all, it.parts, rank + 1) : 0;
                    for (int t = 0; t < 2; ++t) it.nt[t] = max(min(it.nt[t], end) - it.j0, 0);
                    if (!mine) it.rows = 0;
                }
                if (round >= 2)
                    ok = __all_sync(FULL, mbar_wait(&item_empty[round & 1], uint32_t((round >> 1) - 1) & 1u,
                                                    lane == 0 ? status : nullptr));
                if (!ok) break;
                if (lane == 0) {
                    item_sh[round & 1] = it;
                    mbar_arrive(&item_full[round & 1]);
                }
                __syncwarp();
                if (it.s < 0) break;
                const int nkv = max(it.nt[0], it.nt[1]);
                if (nkv == 0) {
                    item = take_over(round);
                    continue;
                }
                auto page_of = [&](int j) -> int {           // n_pages reads as zeros
                    const int t = (it.from() + j) * PT_KEYS + box * br;
                    if (half > 1 || t >= it.len) return c.n_pages;
                    const int p = paged_page(b, c, it.s, t, status);
                    return p < 0 ? c.n_pages : p;
                };
                int page = page_of(0);
                if (qs) ok = __all_sync(FULL, mbar_wait(&q_empty, uint32_t(qs - 1) & 1u, lane == 0 ? status : nullptr));
                if (!ok) break;
                ++qs;
                if (lane == 0) {
                    uint32_t bytes = 0;
                    for (int t = 0; t < 2; ++t)
                        if (it.nt[t]) bytes += 2u * qt * group * 128;
                    mbar_arrive_expect_tx(&q_full, bytes);
                    for (int t = 0; t < 2; ++t)
                        for (int h = 0; h < 2 && it.nt[t]; ++h)
                            tma_load_3d(smem + t * PT_TILE + h * PT_HALF, &tmq, 64 * h, it.head * group,
                                        it.base + it.first + t * qt, &q_full);
                }
                __syncwarp();
                for (int j = 0; j < nkv && ok; ++j) {
                    const int next = j + 1 < nkv ? page_of(j + 1) : 0;
                    const int slot = ((it.from() + j) * PT_KEYS + box * br) & ((1 << c.page_shift) - 1);
                    for (int kv = 0; kv < 2; ++kv) {
                        if (entries >= (Q8 ? RAWS : PT_NS))
                            ok = mbar_wait(Q8 ? &raw_empty[at.st] : &empty[at.st], at.ph ^ 1u, lane == 0 ? status : nullptr);
                        ok = __all_sync(FULL, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(Q8 ? &raw_full[at.st] : &full[at.st], Q8 ? PT_RAW : PT_TILE);
                        __syncwarp();
                        if constexpr (Q8) {
                            uint8_t *to = raw + at.st * PT_RAW;
                            if (half == 0) tma_load_4d(to + box * br * HD, kv ? &tmv : &tmk, 0, slot, it.head, page, &raw_full[at.st]);
                            if (half == 1)
                                tma_load_3d(to + PT_KEYS * HD + box * br * 8, kv ? &tmvs : &tmks, 2 * slot, it.head, page, &raw_full[at.st]);
                        } else if (half < 2)
                            tma_load_4d(ring + at.st * PT_TILE + half * PT_HALF + box * br * 128, kv ? &tmv : &tmk, 64 * half,
                                        slot, it.head, page, &full[at.st]);
                        at.next();
                        ++entries;
                    }
                    page = next;
                    if (j == max(0, nkv - 3) && ok) item = take_over(round);
                }
            }
            // no copy outlives the CTA (bounded)
            constexpr int HELD = Q8 ? RAWS : PT_NS;
            for (int d = entries > HELD ? entries - HELD : 0; d < entries; ++d)
                mbar_wait(Q8 ? &raw_full[d % HELD] : &full[d % HELD], uint32_t(d / HELD) & 1u, nullptr);
            if (qs) mbar_wait(&q_full, uint32_t(qs - 1) & 1u, nullptr);
        } else if (warp == 8) {
            // ---- products: one lane, which queues ahead while the tensor cores work -----------
            if (tc_elect()) {
                // operand descriptors of the first row tile and the first buffer; a 32 KB tile further is + 2048
                const uint64_t dq = tc_sdesc(smem_addr(smem)), dk = tc_sdesc(smem_addr(ring)),
                               dv = tc_sdesc_mn(smem_addr(ring), PT_HALF);
                auto scores = [&](int t, int buf) {          // S_t = Q_t K^T
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t off = (uint32_t(k / 4) * PT_HALF + uint32_t(k % 4) * 32) >> 4;
                        tc_mma_bf16_ss(tbase + t * 128, dq + t * (PT_TILE >> 4) + off, dk + buf * (PT_TILE >> 4) + off,
                                       Q8 ? PT_IDESC & ~PT_F16 : PT_IDESC, uint32_t(k > 0));
                    }
                    tc_commit(&s_full[t]);
                };
                auto values = [&](int t, int buf, int half, bool add) {      // O_t += P_t V over 64 keys
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc_mma_bf16_ts(tbase + 256 + t * 128, tbase + t * 128 + (4 * half + k) * 8,
                                       dv + buf * (PT_TILE >> 4) + (4 * half + k) * (2048 >> 4), Q8 ? PT_IDESC_V & ~PT_F16 : PT_IDESC_V,
                                       k > 0 ? 1u : uint32_t(add));
                };
                RingAt at;
                int qs = 0, tails = 0;
                uint32_t steps[2] = {0, 0}, outs[2] = {0, 0};                // key tiles and results of each row tile so far
                bool ok = true;
                Round it;
                for (int round = 0; ok && next_item(round, it, false); ++round) {
                    const int nkv = max(it.nt[0], it.nt[1]);
                    if (nkv == 0) continue;
                    if (!(ok = mbar_wait(Q8 ? &q_ready : &q_full, uint32_t(qs++) & 1u, status))) break;
                    if (!(ok = mbar_wait(&full[at.st], at.ph, status))) break;
                    tc_fence_after();
                    if (it.nt[0]) scores(0, at.st);
                    if (it.nt[1]) scores(1, at.st);
                    tc_commit(&empty[at.st]);
                    if (nkv == 1) tc_commit(&q_empty);
                    at.next();
                    for (int j = 0; j < nkv; ++j) {
                        const RingAt v = at;
                        at.next();                           // K(j + 1), or the next item's K(0)
                        if (!Q8 && j == max(0, nkv - 2) && it.len < (it.from() + nkv) * PT_KEYS) mbar_arrive(&tail_go);
                        if (!(ok = mbar_wait(&full[v.st], v.ph, status))) break;
                        if (!Q8 && j == nkv - 1 && it.len < (it.from() + nkv) * PT_KEYS)      // cleared behind the sequence's end
                            if (!(ok = mbar_wait(&tail, uint32_t(tails++) & 1u, status))) break;
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            if (j < it.nt[t]) {
                                if (j == 0 && outs[t] && !(ok = mbar_wait(&o_empty[t], (outs[t] - 1) & 1u, status))) break;
#pragma unroll
                                for (int half = 0; half < 2; ++half) {
                                    if (!ok) break;
                                    ok = mbar_wait(&p_full[t][half], steps[t] & 1u, status);
                                    tc_fence_after();
                                    if (ok) values(t, v.st, half, j > 0 || half > 0);
                                }
                                if (!ok) break;
                                if (t == int(j < it.nt[1])) tc_commit(&empty[v.st]);         // the last to use it
                                ++steps[t];
                                if (j + 1 == it.nt[t]) {
                                    tc_commit(&o_full[t]);
                                    ++outs[t];
                                }
                            }
                            if (j + 1 < it.nt[t]) {
                                if (!(ok = mbar_wait(&full[at.st], at.ph, status))) break;
                                tc_fence_after();
                                scores(t, at.st);
                            }
                        }
                        if (!ok) break;
                        if (j + 1 < nkv) {
                            tc_commit(&empty[at.st]);
                            if (j + 2 == nkv) tc_commit(&q_empty);            // the item's last scores
                            at.next();
                        }
                    }
                }
                // every product issued has completed before tensor memory is given back (bounded)
                tc_commit(&drain);
                mbar_wait(&drain, 0, nullptr);
            }
            __syncwarp();
        } else if (Q8 && warp >= 12) {
            // ---- codes to operands --------------------------------------------------------------
            Round it;
            ::q3::RingAt<Q8 ? RAWS : 1> from;
            RingAt to;
            int entries = 0, qs = 0;
            bool ok = true;
            for (int round = 0; ok && next_item(round, it, true); ++round) {
                const int nkv = max(it.nt[0], it.nt[1]);
                if (nkv) {
                    ok = __all_sync(FULL, mbar_wait(&q_full, uint32_t(qs) & 1u, lane == 0 ? status : nullptr));
                    if (!ok) break;
                    const int r = threadIdx.x & 127;
                    for (int t = 0; t < 2; ++t)
                        if (it.nt[t]) q_back[qs & 1][t * PT_ROWS + r] = q_tile_f16(smem + t * PT_TILE, r);
                    ++qs;
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_ready);
                }
                // Entry 2 n is the keys of the n-th key tile, 2 n + 1 its values.  Both lifts are found, and announced,
                // before the keys are converted, so that no softmax waits for them; but after the buffer of the values two
                // tiles before is free, when no softmax needs that tile's any more.
                TileLift lift[2];
                for (int x = 0; x < 2 * nkv; ++x) {
                    const int rows = it.len - (it.from() + x / 2) * PT_KEYS, n = entries >> 1;
                    if (x & 1) {
                        if (entries >= PT_NS) ok = mbar_wait(&empty[to.st], to.ph ^ 1u, lane == 0 ? status : nullptr);
                    } else {
                        ::q3::RingAt<Q8 ? RAWS : 1> values = from;
                        values.next();
                        ok = mbar_wait(&raw_full[from.st], from.ph, lane == 0 ? status : nullptr) &&
                             mbar_wait(&raw_full[values.st], values.ph, lane == 0 ? status : nullptr);
                        ok = __all_sync(FULL, ok);
                        if (!ok) break;
                        // (shared positions: every row sees the whole tile, so that uneven scales are of no account)
                        lift[0] = q8_lift<!SHARED>(raw + from.st * PT_RAW, rows);
                        lift[1] = q8_lift<!SHARED>(raw + values.st * PT_RAW, rows);
                        if (entries >= PT_NS) ok = mbar_wait(&empty[to.st], to.ph ^ 1u, lane == 0 ? status : nullptr);
                        if (threadIdx.x == 12 * 32) {        // every warp finds the same
                            k_back[n & 1] = __uint_as_float(uint32_t(134 - lift[0].e) << 23);
                            v_lift[n & 1] = lift[1].e;
                            rough[n & 1] = lift[0].uneven || lift[1].uneven;
                            mbar_arrive(&lifts[n & 1]);
                        }
                    }
                    ok = __all_sync(FULL, ok);
                    if (!ok) break;
                    q8_tile(raw + from.st * PT_RAW, ring + to.st * PT_TILE, rows, x & 1 ? lift[1].e : lift[0].e);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&full[to.st]);
                        mbar_arrive(&raw_empty[from.st]);
                    }
                    from.next();
                    to.next();
                    ++entries;
                }
            }
        } else if (!Q8 && warp == 10) {
            // ---- values behind a sequence's end: zeros -----------------------------------------
            Round it;
            int entries = 0, tails = 0;                      // of the ring, and cleared ends, in the items so far
            bool ok = true;
            for (int round = 0; ok && next_item(round, it, true); ++round) {
                const int nkv = max(it.nt[0], it.nt[1]);
                entries += 2 * nkv;
                if (it.len >= (it.from() + nkv) * PT_KEYS || nkv == 0) continue;
                // The last tile's values.  The products are at the tile before, so the buffer's earlier use is over and
                // the parity means this one.
                const int last = entries - 1, st = last % PT_NS;
                ok = __all_sync(FULL, mbar_wait(&tail_go, uint32_t(tails) & 1u, lane == 0 ? status : nullptr));
                if (!ok) break;
                ok = __all_sync(FULL, mbar_wait(&full[st], uint32_t(last / PT_NS) & 1u, lane == 0 ? status : nullptr));
                if (!ok) break;
                for (int x = (it.len - (it.from() + nkv - 1) * PT_KEYS) * 8 + lane; x < PT_KEYS * 8; x += 32)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        *reinterpret_cast<uint4 *>(ring + st * PT_TILE + h * PT_HALF + x * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&tail);
                ++tails;
            }
        }
    } else {
        if constexpr (Q8) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax -----------------------------------------------------------------
        const int t = warp >> 2, r = threadIdx.x & 127;      // row tile, row = tensor-memory lane
        const uint32_t lane_base = tbase + (uint32_t(32 * (warp & 3)) << 16);
        const uint32_t ts = lane_base + t * 128, to = lane_base + 256 + t * 128;
        const int r_query = t * qt + r / group, r_head = r % group;
        const bool r_used = r < qt * group;
        uint32_t steps = 0, outs = 0;                        // key tiles and results so far
        [[maybe_unused]] uint32_t qs = 0, tiles = 0;         // Q8_0: queries and key tiles of either row tile so far
        bool ok = true;
        Round it;
        for (int round = 0; ok && next_item(round, it, true); ++round) {
            const int nt = it.nt[t], i = it.first + r_query; // i: the sequence's row
            // (PT_SHARED: a sequence that holds fewer positions attends by itself, and one that another group claims too, where
            // offsets do not rise, behind the one that the plan found it in)
            bool live = r_used && i < it.rows;
            if constexpr (SHARED)
                if (live && sh.plan.spans[it.base + i].x > 0) {
                    const SharedEntry of = sh.plan.of[it.base + i];
                    live = of.first == it.base && of.count == it.rows && of.len == it.len;
                } else {
                    live = false;
                }
            const int limit = SHARED ? it.len : live ? it.seen(i) : 0;
            const int sure = SHARED ? it.len : it.seen(it.first + t * qt);   // keys that every row of the tile sees
            float m = -INFINITY, sum = 0.0f;
            // Q8_0: S is q . k times 1 / (row's and tile's inverse lifts), O is times 2^lift
            [[maybe_unused]] float row_back = 0.0f;
            [[maybe_unused]] int lifted = 0;
            [[maybe_unused]] int redo = 0;                   // 1: the tile that the row sees in part is uneven, 2: O went down too far
            const int nkv = max(it.nt[0], it.nt[1]);
            for (int j = 0; j < nt; ++j, ++steps) {
                ok = __all_sync(FULL, mbar_wait(&s_full[t], steps & 1u, lane == 0 ? status : nullptr));
                if (!ok) break;
                tc_fence_after();
                uint32_t u[128];
#pragma unroll
                for (int x = 0; x < 4; ++x) tc_ld32(ts + 32 * x, u + 32 * x);
#pragma unroll
                for (int x = 0; x < 4; ++x) tc_wait_ld32(u + 32 * x);
                if ((it.from() + j + 1) * PT_KEYS > sure) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) mask32(u + 32 * x, limit - (it.from() + j) * PT_KEYS - 32 * x);
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int x = 0; x < 128; x += 8)
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        mx[y] = fmaxf(fmaxf(mx[y], __uint_as_float(u[x + y])), __uint_as_float(u[x + y + 4]));
                float tile_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                float unit = PT_LOG2;                        // of S to exponents
                [[maybe_unused]] int e = 0, change = 0;      // the tile's lift; of the exponent of O's
                if constexpr (Q8) {
                    // (after the scores' wait: before it the barrier may be phases behind, where its parity means another tile)
                    const uint32_t n = tiles + j;
                    ok = __all_sync(FULL, mbar_wait(&lifts[n & 1], n >> 1 & 1u, lane == 0 ? status : nullptr));
                    if (!ok) break;
                    // (the queries were converted before this tile; q_ready may be a phase ahead by now)
                    if (j == 0) row_back = q_back[qs & 1][t * PT_ROWS + r];
                    const float back = fmaxf(row_back * k_back[n & 1], 0x1p-120f);
                    e = v_lift[n & 1];
                    const int tile = (it.from() + j) * PT_KEYS;
                    if (!SHARED && rough[n & 1] && limit > tile && limit < min(it.len, tile + PT_KEYS)) redo = max(redo, 1);
                    tile_max *= back;
                    unit *= back;
                    if (j == 0) lifted = e;
                    // larger values than before: O goes down; much smaller ones: up again; a tile that the row does not see
                    // changes nothing
                    if ((e < lifted || e > lifted + PT_SLACK) && (SHARED || limit > tile)) change = e - lifted;
                    if (!SHARED && change < -PT_DEEP) redo = 2;
                }
                const bool grow = tile_max > m + PT_LAZY || (m == -INFINITY && tile_max > m);
                if (__any_sync(FULL, grow || change != 0)) {
                    const float nm = grow ? tile_max : m;
                    float f = grow ? (m == -INFINITY ? 0.0f : ex2_approx_ftz((m - nm) * PT_LOG2)) : 1.0f;
                    m = nm;
                    sum *= f;
                    if constexpr (Q8) {
                        if (__any_sync(FULL, change > 0)) {      // (j > 0) no higher than binary32 allows
                            float top = 0.0f;
#pragma unroll 1
                            for (int x = 0; x < 8; ++x) {
                                uint32_t o[16];
                                tc_ld16(to + 16 * x, o);
                                tc_wait_ld16(o);
#pragma unroll
                                for (int y = 0; y < 16; ++y) top = fmaxf(top, fabsf(__uint_as_float(o[y])));
                            }
                            top *= f;
                            if (top > 0.0f && change > 0) change = max(min(change, min(227 - int(__float_as_uint(top) >> 23), 126)), 0);
                        }
                        lifted += change;
                        f *= change < -126 ? 0.0f : __uint_as_float(uint32_t(127 + min(change, 126)) << 23);
                    }
                    if (j > 0) {                                 // O of the tiles before (their product has completed)
#pragma unroll 1
                        for (int x = 0; x < 8; ++x) {
                            uint32_t o[16];
                            tc_ld16(to + 16 * x, o);
                            tc_wait_ld16(o);
#pragma unroll
                            for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                            tc_st16(to + 16 * x, o);
                        }
                    }
                }
                float off = m == -INFINITY ? 0.0f : -m * PT_LOG2;
                // smaller values than O is kept for: their probabilities go down
                [[maybe_unused]] const int shift = Q8 ? max(min(lifted - e, 0), -64) : 0;
                if constexpr (Q8) off += float(shift + PT_BIAS);
                const f2 off2 = pk2(off, off), scale2 = pk2(unit, unit);
                f2 part[2] = {pk2(0.0f, 0.0f), pk2(0.0f, 0.0f)};
#pragma unroll
                for (int x = 0; x < 4; ++x) {                    // 32 probabilities at a time; two halves are handed over
                    uint32_t w[16];
                    // Q8_0: the last 32 scores are read a second time rather than kept, where registers are short (prompts:
                    // 296 us without for the chunks of 243)
                    if constexpr (Q8 && !SHARED) {
                        if (x == 2) tc_ld32(ts + 96, u + 96);
                        if (x == 3) {
                            tc_wait_ld32(u + 96);
                            if ((it.from() + j + 1) * PT_KEYS > sure) mask32(u + 96, limit - (it.from() + j) * PT_KEYS - 96);
                        }
                    }
#pragma unroll
                    for (int y = 0; y < 32; y += 2) {
                        const f2 e = fma2(pk2(__uint_as_float(u[32 * x + y]), __uint_as_float(u[32 * x + y + 1])), scale2, off2);
                        float p0, p1;
                        up2(e, p0, p1);
                        if (y % PT_POLY == PT_POLY - 2 && !Q8) {
                            exp2_poly(p0, p1);
                        } else {
                            p0 = ex2_approx_ftz(p0);
                            p1 = ex2_approx_ftz(p1);
                        }
                        part[y / 2 & 1] = add2(part[y / 2 & 1], pk2(p0, p1));
                        w[y / 2] = Q8 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
                    }
                    tc_st16(ts + 16 * x, w);
                    if (x & 1) {
                        tc_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[t][x >> 1]);
                    }
                }
                float s0, s1;
                up2(add2(part[0], part[1]), s0, s1);
                if constexpr (Q8) sum = fmaf(s0 + s1, __uint_as_float(uint32_t(127 - PT_BIAS - shift) << 23), sum);
                else sum += s0 + s1;
            }
            // what O is to be multiplied by (values are 2^7 below their lift, probabilities 2^7 above)
            [[maybe_unused]] float o_back = 1.0f;
            if constexpr (Q8) {
                tiles += nkv;
                qs += nkv > 0;
                o_back = ldexpf(1.0f, -lifted);
            }
            // ---- the result ----------------------------------------------------------------
            if (nt > 0 && ok) {
                ok = __all_sync(FULL, mbar_wait(&o_full[t], outs++ & 1u, lane == 0 ? status : nullptr));
                tc_fence_after();
            }
            if constexpr (SPLIT) {
                if (ok) stat = make_float2(m, sum);
                if constexpr (Q8) part_back = o_back, part_redo = redo;
                if (it.parts > 1) continue;                  // joined below
            }
            if constexpr (SHARED) {
                if (ok && nt > 0) {
                    const int64_t row = it.dst < 0 ? int64_t(it.base + i) * n_heads + it.head * group + r_head
                                                   : int64_t(b.n_seqs) * n_heads + it.dst + r_query * group + r_head;
                    if (live) *reinterpret_cast<float2 *>(sh.rows + row * SHARED_ROW + HD) = make_float2(m, sum);
#pragma unroll 1
                    for (int x = 0; x < 4; ++x) {
                        uint32_t o[32];
                        tc_ld32(to + 32 * x, o);
                        tc_wait_ld32(o);
                        if (live)
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                U8 v;
#pragma unroll
                                for (int z = 0; z < 8; ++z) v.w[z] = Q8 ? __float_as_uint(__uint_as_float(o[column<Q8>(8 * y + z)]) * o_back) : o[8 * y + z];
                                st_v8(sh.rows + row * SHARED_ROW + 32 * x + 8 * y, v);
                            }
                    }
                    tc_fence_before();                       // the next item's products may overwrite O
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_empty[t]);
                }
                continue;
            }
            if (ok) {
                const float inv = limit > 0 ? (Q8 ? o_back / sum : 1.0f / sum) : 0.0f;
                const unsigned lives = __ballot_sync(FULL, live);
                // Four lanes exchange their rows' pieces, so that they store 64 bytes of a row together.  This lane
                // stores piece lane % 4 of rows (lane / 4) * 4 + k.
                uint16_t *dst[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = 32 * (warp & 3) + (lane & 28) + k, query = by_group(row);
                    dst[k] = out + (int64_t(it.base + it.first + t * qt + query) * n_heads + it.head * group + row - query * group) * HD +
                             8 * (lane & 3);
                }
                f2 zero = pk2(0.0f, 0.0f);                   // becomes NaN with a value that is no number (or infinite)
#pragma unroll 1
                for (int x = 0; x < 4; ++x) {                // 32 columns: four 16-byte pieces of bf16
                    uint32_t o[32], w[4][4];
                    if (nt > 0) {
                        tc_ld32(to + 32 * x, o);
                        tc_wait_ld32(o);
                    }
#pragma unroll
                    for (int z = 0; z < 32; z += 2) {
                        const f2 v = mul2(pk2(__uint_as_float(o[column<Q8>(z)]), __uint_as_float(o[column<Q8>(z + 1)])), pk2(inv, inv));
                        zero = fma2(v, pk2(0.0f, 0.0f), zero);
                        float a, d;
                        up2(v, a, d);
                        w[z / 8][z / 2 & 3] = limit > 0 ? pack_bf16(a, d) : 0u;
                    }
#pragma unroll
                    for (int s = 2; s > 0; s >>= 1)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (!(k & s))
#pragma unroll
                                for (int y = 0; y < 4; ++y) {
                                    const uint32_t got = __shfl_xor_sync(FULL, lane & s ? w[k][y] : w[k ^ s][y], s);
                                    if (lane & s) w[k][y] = got;
                                    else w[k ^ s][y] = got;
                                }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (lives >> ((lane & 28) + k) & 1u)
                            st_cs_v4(dst[k] + 32 * x, make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]));
                }
                float z0, z1;
                up2(zero, z0, z1);
                const bool nan = z0 + z1 != 0.0f;
                if (nt > 0) {                                // the next item's products may overwrite O
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_empty[t]);
                }
                // rows that came out as no numbers, and such as lost bits to positions that they do not see, once more from
                // the formula (over what is stored, which stays where time is up)
                unsigned again = __ballot_sync(FULL, live && limit > 0 && (nan || (Q8 && redo > 0)));
                SecondLook<Cached> second;
                const uint64_t began = again ? global_ns() : 0;
                while (again) {
                    if (global_ns() - began > PT_AGAIN_NS) {
                        if (lane == 0) flag_timeout(status);
                        break;
                    }
                    const int l = __ffs(again) - 1;
                    again &= again - 1;
                    __syncwarp();
                    const int il = __shfl_sync(FULL, i, l), n = __shfl_sync(FULL, limit, l);
                    const int h = it.head * group + __shfl_sync(FULL, r_head, l);
                    float4 x = load_quad(q + int64_t(it.base + il) * q_stride + int64_t(h) * HD + 4 * lane);
                    const int lost = Q8 ? __shfl_sync(FULL, redo, l) : 0;
                    bool want = lost == 2;
                    if (!want && __shfl_sync(FULL, int(nan), l)) {
                        second.look(t, c, b, it.s, it.head, it.seen(it.first + t * qt), min(it.len, it.nt[t] * PT_KEYS));
                        want = second.wanted(n, x);
                    }
                    if constexpr (Q8)
                        if (!want && lost) want = larger_behind(c, b, it.s, it.head, n, it.len);
                    if (!want) continue;
                    x = make_float4(x.x * ATT_SCALE, x.y * ATT_SCALE, x.z * ATT_SCALE, x.w * ATT_SCALE);
                    store_quad(out + (int64_t(it.base + il) * n_heads + h) * HD + 4 * lane,
                               attend_row<Cached, 4>(c, b, it.s, it.head, n, x, status));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if constexpr (SPLIT) {
        const Round it = item_sh[0];
        const int rank = int(blockIdx.x % unsigned(ctas));
        if (it.parts > 1 && rank < it.parts) {               // the same for all of the CTA
            float2 *stats = reinterpret_cast<float2 *>(smem);
            [[maybe_unused]] uint32_t *marks = reinterpret_cast<uint32_t *>(stats + 2 * PT_ROWS);
            if (warp < 8) {                                  // the rows' results, 128 KB in the ring's place
                stats[threadIdx.x] = stat;
                if constexpr (Q8) marks[threadIdx.x] = part_redo;
                const int t = warp >> 2;
                uint8_t *row = ring + threadIdx.x * (HD * 4);
#pragma unroll 1
                for (int x = 0; x < 4; ++x) {
                    uint32_t o[32];
                    if (it.nt[t]) {
                        tc_ld32(tbase + (uint32_t(32 * (warp & 3)) << 16) + 256 + t * 128 + 32 * x, o);
                        tc_wait_ld32(o);
                    } else {
#pragma unroll
                        for (int y = 0; y < 32; ++y) o[y] = 0u;
                    }
                    if constexpr (Q8)
#pragma unroll
                        for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * part_back);
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        *reinterpret_cast<uint4 *>(row + (((8 * x + y) ^ (lane & 7)) << 4)) =
                            make_uint4(o[4 * y], o[column<Q8>(4 * y + 1)], o[column<Q8>(4 * y + 2)], o[4 * y + 3]);
                }
                tc_fence_before();
            }
            cluster_sync();
            SecondLook<Cached> second;
            for (int r = prompt_part(2 * PT_ROWS, it.parts, rank) + warp; r < prompt_part(2 * PT_ROWS, it.parts, rank + 1);
                 r += PT_THREADS / 32) {
                const int in_tile = r & 127, query = by_group(in_tile), i = it.first + (r >> 7) * qt + query;
                const int head = it.head * group + in_tile - query * group;
                if (query >= qt || i >= it.rows) continue;
                const int limit = it.seen(i);
                bool ok;
                float4 v = join_parts(smem_addr(ring) + r * (HD * 4), smem_addr(stats + r), r, it.parts, PT_LOG2, ok);
                if (!ok) continue;
                if (limit <= 0) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const bool nan = __any_sync(FULL, !all_finite(v));
                uint32_t lost = 0;
                if constexpr (Q8) {
                    uint32_t mark = 0;
                    if (lane < it.parts)
                        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(mark) : "r"(peer_smem(smem_addr(marks + r), lane)) : "memory");
                    lost = __reduce_max_sync(FULL, mark);
                }
                if (limit > 0 && (nan || lost)) {
                    const float4 x = load_quad(q + int64_t(it.base + i) * q_stride + int64_t(head) * HD + 4 * lane);
                    bool want = lost == 2;
                    if (!want && nan) {
                        const int first = it.first + (r >> 7) * qt, seen = it.seen(min(first + qt, it.rows) - 1);
                        second.look(r >> 7, c, b, it.s, it.head, it.seen(first), min(it.len, (seen + PT_KEYS - 1) / PT_KEYS * PT_KEYS));
                        want = second.wanted(limit, x);
                    }
                    if constexpr (Q8)
                        if (!want && lost) want = larger_behind(c, b, it.s, it.head, limit, it.len);
                    if (want)
                        v = attend_row<Cached, 4>(c, b, it.s, it.head, limit,
                                                make_float4(x.x * ATT_SCALE, x.y * ATT_SCALE, x.z * ATT_SCALE, x.w * ATT_SCALE),
                                                status);
                }
                store_quad(out + (int64_t(it.base + i) * n_heads + head) * HD + 4 * lane, v);
            }
            cluster_sync();                                  // no CTA's shared memory goes while others read it
            tc_fence_after();
        }
    }
    if (warp == 8) tc_free512(tbase);
}

// The queries, [rows][n_heads][128] in bf16, in boxes of the rows and heads of a tile by 64 elements (k_prompt.cu).
bool encode_prompt_q_map(CUtensorMap *map, const void *q, int n_heads, int64_t rows, int64_t q_stride, int group);

}  // namespace q3
