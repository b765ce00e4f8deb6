// k_prompt.cu -- causal attention of packed prompt rows over the paged cache.
//
// A row at position p: o = sum_t softmax_t(q . k_t / sqrt(128)) v_t over the
// positions t <= p of its sequence, in one pass over the keys with the running
// maximum and sum of the softmax.
//
// bf16, on the tensor cores (prompt_tc_kernel).  A work item is a block of
// consecutive queries of one sequence under one kv head, with all the query
// heads that read it: row r of a 128-row tile is query r / g, head r % g of the
// group of g, so short chunks fill the tile and the keys are fetched once for
// the whole group.  An item has two such tiles, which share the keys and take
// turns: while one tile's scores go through the softmax, the tensor cores work
// on the other's.  A CTA per SM takes items one after the
// other, its warps each at their own pace, so that one item's first fetches and
// products run beside the last softmax and the stores of the item before:
//   warps 0-3, 4-7  the softmax of tile 0 and of tile 1: thread = row = tensor-
//            memory lane.  Reads the 128 scores of a key tile, folds the
//            maximum, writes the probabilities back as bf16 over the scores
//            (they are the next product's operand in tensor memory) and keeps
//            the sum in binary32.  O is rescaled only when the maximum has
//            grown by more than 2^8 since the last time; until then the old
//            maximum stays the reference, which changes no result (numerator
//            and sum share it) and keeps every value far inside binary32.
//   warp 8   issues the products: S = Q K^T from shared memory, O += P V with P
//            from tensor memory.
//   warp 9   finds the items, announces them in shared memory, and fetches Q and
//            the key and value tiles of 128 positions, page by page, by TMA into
//            a ring of five 32 KB buffers.
//   warp 10  clears the values behind a sequence's end (below).
// Items go from the longest to the shortest; a CTA that is done with one takes
// over that of a CTA that has not started.
//
// Bound by the tensor cores and what keeps them waiting: a step (128 keys, two
// row tiles) has 2,048 cycles of products and takes 2,990, the time from a tile's
// last probabilities to its next scores and through the softmax, which the other
// tile fills in part.  Over changing inputs a prompt of 16,384 (40/8 heads) takes
// 2.55 ms, 1,078 TFLOP/s, at 1.6 GHz under the power cap; 2,043 rows in chunks behind
// prefixes of up to 8,192 (32/8) 200 us, 880 TFLOP/s; 4,096 rows in six prompts (32/8)
// 54 us.  A replayed graph on one input: 2.15 to 2.3 ms, 175 and 50 us.
// Tensor memory (512 columns): S0, S1, O0, O1; P_t lies over the first half of S_t.
//
// With few items (prompt_tc_kernel<true>) a cluster of up to eight CTAs takes one, each a part of its key tiles, and joins
// the parts through shared memory (join_parts): 16 rows behind 8,000 positions (32/8 heads) 120 -> 28 us, 100 rows
// behind 8,000 138 -> 36 us, 30 behind 30,000 440 -> 62 us.  Up to 64 of 148 SMs work then (8 kv heads).
//
// Masks: keys at and beyond the row's limit become -inf before the maximum.
// Their probability is exactly 0, but 0 times a NaN or an infinity in V is not:
// the values behind the sequence's end (never written, anything may be there) are
// zeroed in shared memory, and a row that comes out with elements that are no
// numbers is computed again from the formula by one warp (attend_row), so that a
// value at a later position of the sequence never reaches an earlier row.  That is
// some hundred times slower than the tile, so it is done only where it may change
// the row (SecondLook): a prompt of 4,096 rows (32/8) takes 0.14 ms, 1.3 with a NaN
// that all rows see, and 24 with one in the last value, which spoils a tile.
//
// Every wait is bounded (2 s; the longest, for the next item, lasts as long as an
// item, some 10 ns a key); a wait that gives up sets Q3CU_DEV_TIMEOUT and the CTA
// drains its own copies and products, frees tensor memory and returns.  So that no
// other warp's wait gives up meanwhile, a warp computes rows again for a second at
// most; past that (32 rows of 170,000 keys) the rest stay NaN, with the same bit set.
#include "q3cu_paged.cuh"
#include "q3cu_tcgen05.cuh"
#include "q3cu_tma.h"

#include <atomic>
#include <type_traits>

namespace q3 {

constexpr int PT_ROWS = 128, PT_KEYS = 128;                  // rows of a tile, keys of a tile
constexpr int PT_THREADS = 12 * 32;
constexpr int PT_WHOLE = 8;                                  // key tiles from which on an item may be shared
constexpr int PT_NS = 5;                                     // K / V buffers in flight
constexpr uint32_t PT_HALF = PT_ROWS * 128;                  // bytes of 128 rows x 64 elements
constexpr uint32_t PT_TILE = 2 * PT_HALF;                    // 32 KB
constexpr size_t PT_SMEM = size_t(2 + PT_NS) * PT_TILE + 1024;
// Instruction descriptors: f32 accumulator, bf16 A and B, M = N = 128; B K-major (K) or MN-major (V).
constexpr uint32_t PT_IDESC = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 / 8) << 17) | (uint32_t(128 / 16) << 24);
constexpr uint32_t PT_IDESC_V = PT_IDESC | (1u << 16);
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
constexpr int PT_POLY = 8;                                   // one pair of exponentials in PT_POLY / 2 by polynomial

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
struct RingAt {
    int st = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next() {
        if (++st == PT_NS) st = 0, ph ^= 1u;
    }
};

// SPLIT: clusters of `ctas` CTAs, each with one item.
template <bool SPLIT>
__global__ void __launch_bounds__(PT_THREADS, 1)
prompt_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                 const __grid_constant__ CUtensorMap tmv, const PagedKV c, const PagedSeqs b, int rows,
                 const uint16_t *q, int64_t q_stride, int n_heads, int group, const FastDiv per_block,
                 const FastDiv by_group, int ctas, uint16_t *out, uint32_t *status) {
    typedef typename std::conditional<SPLIT, PromptShare, PromptRound>::type Round;
    extern __shared__ uint8_t pt_dyn[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pt_dyn) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = smem + 2 * PT_TILE;
    __shared__ __align__(8) uint64_t q_full, q_empty, full[PT_NS], empty[PT_NS], s_full[2], p_full[2][2], o_full[2],
        o_empty[2], item_full[2], item_empty[2], taken, tail_go, tail, drain;
    __shared__ Round item_sh[2];
    __shared__ ulonglong2 taken_sh;
    __shared__ uint32_t tmem_sh;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 1);
        for (int i = 0; i < PT_NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t][0], 4);
            mbar_init(&p_full[t][1], 4);
            mbar_init(&o_full[t], 1);
            mbar_init(&o_empty[t], 4);
            mbar_init(&item_full[t], 1);
            mbar_init(&item_empty[t], 10);                   // warps 0-7, 8 and 10
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

    const int qt = PT_ROWS / group;                          // queries of a tile
    float2 stat = make_float2(-INFINITY, -1.0f);             // SPLIT: maximum and sum of this thread's row, -1: given up
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

    // Registers move to the softmax: 256 threads x 208 + 128 x 88 is the launch's 384 x 168.
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 9) {
            // ---- items and copies ------------------------------------------------------------
            const int br = min(1 << c.page_shift, PT_KEYS), nb = PT_KEYS / br;  // rows of a box, boxes of a tile
            // lane = box: column half lane / nb, positions lane % nb
            const int box = lane % nb, half = lane / nb;
            RingAt at;
            int entries = 0, qs = 0;                         // copies of tiles and of Q so far
            bool ok = true;
            PromptOrder order(b, c, rows, per_block, PT_KEYS, status);
            PromptItem item = order.find(SPLIT ? blockIdx.x / unsigned(ctas) : blockIdx.x);
            // The first item is this CTA's own; the others are those of CTAs that have not started.  One is taken over
            // when the copies for the item before are nearly all under way: no earlier, so that the CTA that is done
            // first gets the next item, and no later, since finding it takes some thousand cycles.
            auto take_over = [&](int round) -> PromptItem {
                PromptItem none;
                none.s = -1;
                if constexpr (SPLIT) return none;
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
                static_cast<PromptItem &>(it) = item;
                it.nt[0] = it.nt[1] = 0;
                for (int t = 0; t < 2 && it.s >= 0; ++t) {
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
                        if (entries >= PT_NS) ok = mbar_wait(&empty[at.st], at.ph ^ 1u, lane == 0 ? status : nullptr);
                        ok = __all_sync(FULL, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&full[at.st], PT_TILE);
                        __syncwarp();
                        if (half < 2)
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
            for (int d = entries > PT_NS ? entries - PT_NS : 0; d < entries; ++d)
                mbar_wait(&full[d % PT_NS], uint32_t(d / PT_NS) & 1u, nullptr);
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
                                       PT_IDESC, uint32_t(k > 0));
                    }
                    tc_commit(&s_full[t]);
                };
                auto values = [&](int t, int buf, int half, bool add) {      // O_t += P_t V over 64 keys
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc_mma_bf16_ts(tbase + 256 + t * 128, tbase + t * 128 + (4 * half + k) * 8,
                                       dv + buf * (PT_TILE >> 4) + (4 * half + k) * (2048 >> 4), PT_IDESC_V,
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
                    if (!(ok = mbar_wait(&q_full, uint32_t(qs++) & 1u, status))) break;
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
                        if (j == max(0, nkv - 2) && it.len < (it.from() + nkv) * PT_KEYS) mbar_arrive(&tail_go);
                        if (!(ok = mbar_wait(&full[v.st], v.ph, status))) break;
                        if (j == nkv - 1 && it.len < (it.from() + nkv) * PT_KEYS)     // cleared behind the sequence's end
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
                        tc_commit(&empty[v.st]);
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
        } else if (warp == 10) {
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax -----------------------------------------------------------------
        const int t = warp >> 2, r = threadIdx.x & 127;      // row tile, row = tensor-memory lane
        const uint32_t lane_base = tbase + (uint32_t(32 * (warp & 3)) << 16);
        const uint32_t ts = lane_base + t * 128, to = lane_base + 256 + t * 128;
        const int r_query = t * qt + r / group, r_head = r % group;
        const bool r_used = r < qt * group;
        uint32_t steps = 0, outs = 0;                        // key tiles and results so far
        bool ok = true;
        Round it;
        for (int round = 0; ok && next_item(round, it, true); ++round) {
            const int nt = it.nt[t], i = it.first + r_query; // i: the sequence's row
            const bool live = r_used && i < it.rows;
            const int limit = live ? it.seen(i) : 0;
            const int sure = it.seen(it.first + t * qt);    // keys that every row of the tile sees
            float m = -INFINITY, sum = 0.0f;
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
                const float tile_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const bool grow = tile_max > m + PT_LAZY || (m == -INFINITY && tile_max > m);
                if (__any_sync(FULL, grow)) {
                    const float nm = grow ? tile_max : m;
                    const float f = grow ? (m == -INFINITY ? 0.0f : ex2_approx_ftz((m - nm) * PT_LOG2)) : 1.0f;
                    m = nm;
                    sum *= f;
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
                const float off = m == -INFINITY ? 0.0f : -m * PT_LOG2;
                const f2 off2 = pk2(off, off), scale2 = pk2(PT_LOG2, PT_LOG2);
                f2 part[2] = {pk2(0.0f, 0.0f), pk2(0.0f, 0.0f)};
#pragma unroll
                for (int x = 0; x < 4; ++x) {                    // 32 probabilities at a time; two halves are handed over
                    uint32_t w[16];
#pragma unroll
                    for (int y = 0; y < 32; y += 2) {
                        const f2 e = fma2(pk2(__uint_as_float(u[32 * x + y]), __uint_as_float(u[32 * x + y + 1])), scale2, off2);
                        float p0, p1;
                        up2(e, p0, p1);
                        if (y % PT_POLY == PT_POLY - 2) {
                            exp2_poly(p0, p1);
                        } else {
                            p0 = ex2_approx_ftz(p0);
                            p1 = ex2_approx_ftz(p1);
                        }
                        part[y / 2 & 1] = add2(part[y / 2 & 1], pk2(p0, p1));
                        w[y / 2] = pack_bf16(p0, p1);
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
                sum += s0 + s1;
            }
            // ---- the result ----------------------------------------------------------------
            if (nt > 0 && ok) {
                ok = __all_sync(FULL, mbar_wait(&o_full[t], outs++ & 1u, lane == 0 ? status : nullptr));
                tc_fence_after();
            }
            if constexpr (SPLIT) {
                if (ok) stat = make_float2(m, sum);
                if (it.parts > 1) continue;                  // joined below
            }
            if (ok) {
                const float inv = limit > 0 ? 1.0f / sum : 0.0f;
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
                        const f2 v = mul2(pk2(__uint_as_float(o[z]), __uint_as_float(o[z + 1])), pk2(inv, inv));
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
                // rows that came out as no numbers, once more from the formula
                unsigned again = __ballot_sync(FULL, live && limit > 0 && nan);
                SecondLook<bf16raw> second;
                const uint64_t began = again ? global_ns() : 0;
                while (again) {
                    if (global_ns() - began > PT_AGAIN_NS) {
                        if (lane == 0) flag_timeout(status);
                        break;
                    }
                    const int l = __ffs(again) - 1;
                    again &= again - 1;
                    __syncwarp();
                    second.look(t, c, b, it.s, it.head, it.seen(it.first + t * qt), min(it.len, it.nt[t] * PT_KEYS));
                    const int il = __shfl_sync(FULL, i, l), n = __shfl_sync(FULL, limit, l);
                    const int h = it.head * group + __shfl_sync(FULL, r_head, l);
                    float4 x = load_quad(q + int64_t(it.base + il) * q_stride + int64_t(h) * HD + 4 * lane);
                    if (!second.wanted(n, x)) continue;
                    x = make_float4(x.x * ATT_SCALE, x.y * ATT_SCALE, x.z * ATT_SCALE, x.w * ATT_SCALE);
                    store_quad(out + (int64_t(it.base + il) * n_heads + h) * HD + 4 * lane,
                               attend_row<bf16raw, 4>(c, b, it.s, it.head, n, x, status));
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
            if (warp < 8) {                                  // the rows' results, 128 KB in the ring's place
                stats[threadIdx.x] = stat;
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
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        *reinterpret_cast<uint4 *>(row + (((8 * x + y) ^ (lane & 7)) << 4)) =
                            make_uint4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
                }
                tc_fence_before();
            }
            cluster_sync();
            SecondLook<bf16raw> second;
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
                if (limit > 0 && __any_sync(FULL, !all_finite(v))) {
                    const int first = it.first + (r >> 7) * qt, seen = it.seen(min(first + qt, it.rows) - 1);
                    second.look(r >> 7, c, b, it.s, it.head, it.seen(first), min(it.len, (seen + PT_KEYS - 1) / PT_KEYS * PT_KEYS));
                    const float4 x = load_quad(q + int64_t(it.base + i) * q_stride + int64_t(head) * HD + 4 * lane);
                    if (second.wanted(limit, x))
                        v = attend_row<bf16raw, 4>(c, b, it.s, it.head, limit,
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

// The largest cluster of which the GPU holds as many at once as there are items (an SM holds one CTA, and a cluster lies
// within one group of SMs: 15 of 8, 33 of 4, 74 of 2 on a B200).
int prompt_cluster(const void *kernel, int slot, int threads, size_t smem, int64_t items, int64_t tiles) {
    static std::atomic<int> room[64][2][9];                  // clusters of a size that the device holds, plus 1; 0: not asked
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    for (int ctas = 8; ctas > 1; --ctas) {
        if (ctas > tiles / PROMPT_PART) continue;
        int n = room[dev][slot][ctas].load(std::memory_order_relaxed);
        if (n == 0) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(unsigned(ctas));
            cfg.blockDim = dim3(unsigned(threads));
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = unsigned(ctas);
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int held = 0;
            if (cudaOccupancyMaxActiveClusters(&held, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                held = 0;
            }
            room[dev][slot][ctas].store(n = held + 1, std::memory_order_relaxed);
        }
        if (items < n) return ctas;
    }
    return 1;
}

cudaError_t launch_attention_prompt(const PagedKV &c, const PagedSeqs &b, int64_t rows, const void *q, q3cu_dtype dt,
                                    int64_t q_stride, int n_heads, void *out, uint32_t *status, cudaStream_t stream,
                                    int sms) {
    if (dt == Q3CU_F32) return launch_prompt_f32(c, b, rows, q, q_stride, n_heads, out, status, stream);
    const int group = n_heads / c.n_kv, qt = PT_ROWS / group;
    CUtensorMap mq, mk, mv;
    const uint64_t dims[3] = {HD, uint64_t(n_heads), uint64_t(rows)};
    const uint64_t strides[2] = {HD * 2, uint64_t(q_stride) * 2};
    const uint32_t box[3] = {64, uint32_t(group), uint32_t(qt)};
    if (!encode_lines_map(&mq, q, Q3CU_BF16, 3, dims, strides, box) || !encode_pages_map(&mk, c.k, c, Q3CU_BF16, PT_KEYS) ||
        !encode_pages_map(&mv, c.v, c, Q3CU_BF16, PT_KEYS))
        return cudaErrorInvalidValue;
    // no more blocks of 2 * qt queries than this, however the rows are split into sequences
    const int64_t items = (rows / (2 * qt) + b.n_seqs) * c.n_kv;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(prompt_tc_kernel<true>), PT_SMEM, 43);
    if (e == cudaSuccess) e = ensure_smem_attr(reinterpret_cast<const void *>(prompt_tc_kernel<false>), PT_SMEM, 32);
    if (e != cudaSuccess) return e;
    const int ctas = prompt_cluster(reinterpret_cast<const void *>(prompt_tc_kernel<true>), 0, PT_THREADS, PT_SMEM, items,
                                    (int64_t(b.max_pages) << c.page_shift) / PT_KEYS);
    auto kernel = ctas > 1 ? prompt_tc_kernel<true> : prompt_tc_kernel<false>;
    return launch_clusters(kernel, ctas, dim3(unsigned(items * ctas)), dim3(PT_THREADS), PT_SMEM, stream, mq, mk, mv, c, b,
                           int(rows), static_cast<const uint16_t *>(q), q_stride, n_heads, group, FastDiv(2 * qt),
                           FastDiv(group), ctas, static_cast<uint16_t *>(out), status);
}

}  // namespace q3
