// q3cu_paged.cuh -- the paged key-value cache as the kernels see it: where a
// position's row lies, and which sequence a packed token row belongs to.
#pragma once

#include "q3cu_device.cuh"
#include "q3cu_internal.h"

namespace q3 {

constexpr int HD = PAGED_HD;

template <typename T> struct Elem;
template <> struct Elem<float> {
    typedef float type;
    static constexpr int BYTES = 4;
};
template <> struct Elem<bf16raw> {
    typedef uint16_t type;
    static constexpr int BYTES = 2;
};

struct q8raw {};                                             // Q8_0: codes here, their scales beside them
template <> struct Elem<q8raw> {
    typedef uint8_t type;
    static constexpr int BYTES = 1;
};

// (Host and device: the index arithmetic is also checked on the CPU.)
__host__ __device__ __forceinline__ void flag_bad_index(uint32_t *status) {
    if (!status) return;
#ifdef __CUDA_ARCH__
    atomicOr(status, Q3CU_DEV_BAD_INDEX);
#else
    *status |= Q3CU_DEV_BAD_INDEX;
#endif
}

__device__ __forceinline__ void flag_timeout(uint32_t *status) {
    if (status) atomicOr(status, Q3CU_DEV_TIMEOUT);
}

// Keys a sequence holds: kv_len, no more than its table row has pages for (a
// longer kv_len is flagged) and no fewer than none.
__host__ __device__ __forceinline__ int paged_len(const PagedSeqs &b, const PagedKV &c, int s, uint32_t *status) {
    const int64_t cap = int64_t(b.max_pages) << c.page_shift;
    const int n = b.kv_len[s];
    if (n > cap) {
        flag_bad_index(status);
        return int(cap);
    }
    return n < 0 ? 0 : n;
}

// Page of position t (t >= 0, below max_pages << page_shift) of sequence s; -1 and the status bit for an id
// outside the cache.
__host__ __device__ __forceinline__ int paged_page(const PagedSeqs &b, const PagedKV &c, int s, int t, uint32_t *status) {
    const int page = b.pages[int64_t(s) * b.max_pages + (t >> c.page_shift)];
    if (page >= 0 && page < c.n_pages) return page;
    flag_bad_index(status);
    return -1;
}

// Element offset of (page, kv head, slot): 64 bits, a cache is larger than 2^31 elements.
__host__ __device__ __forceinline__ int64_t paged_at(const PagedKV &c, int page, int head, int t) {
    const int slot = t & ((1 << c.page_shift) - 1);
    return int64_t(page) * c.page_stride + ((int64_t(head) << c.page_shift) + slot) * HD;
}

// Index of (page, kv head, slot)'s first scale (Q8_0).
__host__ __device__ __forceinline__ int64_t paged_scale_at(const PagedKV &c, int page, int head, int t) {
    const int slot = t & ((1 << c.page_shift) - 1);
    return int64_t(page) * c.scale_stride + ((int64_t(head) << c.page_shift) + slot) * 2;
}

// The sequence of packed row r: the last s with row_off[s] <= r, or -1 when r
// lies in no sequence (behind the last one, or offsets that do not rise).
__host__ __device__ __forceinline__ int paged_seq_of(const PagedSeqs &b, int64_t r) {
    int lo = 0, hi = b.n_seqs;                               // row_off[lo] <= r < row_off[hi], if any does
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.row_off[mid] <= r) lo = mid;
        else hi = mid;
    }
    return b.n_seqs > 0 && b.row_off[lo] <= r && r < b.row_off[lo + 1] ? lo : -1;
}

// The same by a whole warp: 33-way search, one round of loads for up to 31 sequences and two for up to 1,023.
__device__ __forceinline__ int paged_seq_of_warp(const PagedSeqs &b, int64_t r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = b.n_seqs;                               // as above
    int64_t at_lo = 0, at_hi = 0;
    bool have_lo = false, have_hi = false;
    while (hi - lo > 1 || !have_lo || !have_hi) {
        // probes lo, lo + step, ..., and hi in the last lane
        const int step = (hi - lo + 30) / 31, p = lane == 31 ? hi : min(lo + lane * step, hi);
        const int64_t x = b.row_off[p];
        const unsigned below = __ballot_sync(FULL, x <= r && p < hi) & 0x7fffffffu;
        const int l = below ? 31 - __clz(below) : 0;         // the last probe at or before r
        const int nl = __shfl_sync(FULL, p, l), nh = __shfl_sync(FULL, p, l + 1);
        at_lo = __shfl_sync(FULL, x, l);
        at_hi = __shfl_sync(FULL, x, l + 1);
        have_lo = have_hi = true;
        lo = nl;
        hi = nh;
    }
    return b.n_seqs > 0 && at_lo <= r && r < at_hi ? lo : -1;
}

// Position of packed row r of sequence s (as paged_seq_of finds it): negative for padding before position 0, and,
// flagged, beyond the table's pages.
__host__ __device__ __forceinline__ int paged_pos(const PagedSeqs &b, const PagedKV &c, int s, int64_t r,
                                                  uint32_t *status) {
    const int64_t p = int64_t(b.kv_len[s]) - b.row_off[s + 1] + r;
    if (p < 0) return -1;
    if (p < int64_t(b.max_pages) << c.page_shift) return int(p);
    flag_bad_index(status);
    return -1;
}

// Sequence and position of packed row r (as paged_seq_of_warp and paged_pos find them) by a whole warp: for up to 31
// sequences one round of loads in place of two.
__device__ __forceinline__ int paged_row_of_warp(const PagedSeqs &b, const PagedKV &c, int64_t r, int &pos, uint32_t *status) {
    const int lane = threadIdx.x & 31;
    int s;
    if (b.n_seqs < 32) {
        const int off = b.row_off[min(lane, b.n_seqs)], len = b.kv_len[min(lane, b.n_seqs - 1)];
        const unsigned below = __ballot_sync(FULL, off <= r && lane < b.n_seqs);
        s = below ? 31 - __clz(below) : 0;
        const int end = __shfl_sync(FULL, off, s + 1), n = __shfl_sync(FULL, len, s);
        if (!below || r >= end) return -1;
        const int64_t p = int64_t(n) - end + r;
        pos = p < 0 ? -1 : int(min(p, int64_t(INT32_MAX)));
        if (p >= int64_t(b.max_pages) << c.page_shift) {
            if (lane == 0) flag_bad_index(status);
            pos = -1;
        }
        return s;
    }
    s = paged_seq_of_warp(b, r);
    if (s >= 0) pos = paged_pos(b, c, s, r, lane == 0 ? status : nullptr);
    return s;
}

// Keys that packed row r of sequence s attends to: the positions up to its own, as far as the sequence holds them
// (`len` of paged_len).
__host__ __device__ __forceinline__ int paged_seen(const PagedSeqs &b, int s, int64_t r, int len) {
    const int64_t n = int64_t(b.kv_len[s]) - b.row_off[s + 1] + r + 1;
    return n < 0 ? 0 : n < len ? int(n) : len;
}

// Two floats rounded to bf16, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Four consecutive elements as floats, and a float4 stored as T.
__device__ __forceinline__ float4 load_quad(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load_quad(const uint16_t *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(bf16_to_f32(u.x & 0xffffu), bf16_to_f32(u.x >> 16), bf16_to_f32(u.y & 0xffffu),
                       bf16_to_f32(u.y >> 16));
}
__device__ __forceinline__ void store_quad(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store_quad(uint16_t *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// Four Q8_0 codes as floats: code + 128 as the low byte of 2^23 + it, less 2^23 + 128 (exact, and on the common pipes
// where a conversion is not).
__device__ __forceinline__ float4 q8_floats(uint32_t codes) {
    codes ^= 0x80808080u;
    auto one = [&](uint32_t pick) { return __uint_as_float(__byte_perm(codes, 0x4b000000u, pick)) - 8388736.0f; };
    return make_float4(one(0x7440), one(0x7441), one(0x7442), one(0x7443));
}

// Four elements of a key or value: `at` in the cache, of the row whose scales begin at index `scale` (Q8_0; lane as in
// attend_row).
template <typename TC>
__device__ __forceinline__ float4 cached_quad(const PagedKV &c, bool value, int64_t at, int64_t scale) {
    const typename Elem<TC>::type *p = static_cast<const typename Elem<TC>::type *>(value ? c.v : c.k) + at;
    if constexpr (Elem<TC>::BYTES == 1) {
        const float4 x = q8_floats(*reinterpret_cast<const uint32_t *>(p));
        const float s = (value ? c.v_scale : c.k_scale)[scale + ((threadIdx.x & 31) >> 4)];
        return make_float4(s * x.x, s * x.y, s * x.z, s * x.w);
    } else {
        return load_quad(p);
    }
}

// Whether none of them is infinite or NaN.
__device__ __forceinline__ bool all_finite(float4 v) {
    return fmaf(v.x, 0.0f, fmaf(v.y, 0.0f, fmaf(v.z, 0.0f, v.w * 0.0f))) == 0.0f;
}

// Attention of one query row and head by one warp, straight from the formula:
// lane l holds elements 4l .. 4l+3 of q (scaled by 1/sqrt(128)), of every key
// and value and of the result.  The running maximum and sum of the softmax, one pass over
// the keys 0 .. n-1 of sequence s, STEP at a time (a page holds them all): 0.18 us a key by fours, 0.15 by eights, whose
// registers cost every bf16 prompt 1 %.  A score of -inf (an infinite key) weighs nothing; a row that has no other is
// 0 / 0.  Returns zeros for n = 0.
template <typename TC, int STEP>
__device__ __forceinline__ float4 attend_row(const PagedKV &c, const PagedSeqs &b, int s, int head, int n, float4 q,
                                             uint32_t *status) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY, sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int t = 0; t < n; t += STEP) {
        const int page = paged_page(b, c, s, t, lane == 0 ? status : nullptr);
        const int64_t at = page >= 0 ? paged_at(c, page, head, t) + 4 * lane : 0;
        const int64_t scale = Elem<TC>::BYTES == 1 && page >= 0 ? paged_scale_at(c, page, head, t) : 0;
        float4 k[STEP], v[STEP];
#pragma unroll
        for (int u = 0; u < STEP; ++u) {
            k[u] = v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (page >= 0 && t + u < n) {
                k[u] = cached_quad<TC>(c, false, at + u * HD, scale + 2 * u);
                v[u] = cached_quad<TC>(c, true, at + u * HD, scale + 2 * u);
            }
        }
        float d[STEP], nm = m;
#pragma unroll
        for (int u = 0; u < STEP; ++u) {
            d[u] = fmaf(q.x, k[u].x, fmaf(q.y, k[u].y, fmaf(q.z, k[u].z, q.w * k[u].w)));
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) d[u] += __shfl_xor_sync(FULL, d[u], x);
            if (t + u >= n) d[u] = -INFINITY;
            nm = fmaxf(nm, d[u]);
        }
        const float f = m == nm ? 1.0f : expf(m - nm);
        m = nm;
        sum *= f;
        o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
        for (int u = 0; u < STEP; ++u) {
            const float p = d[u] == -INFINITY ? 0.0f : expf(d[u] - nm);    // also while nm is -inf
            sum += p;
            o = make_float4(fmaf(p, v[u].x, o.x), fmaf(p, v[u].y, o.y), fmaf(p, v[u].z, o.z), fmaf(p, v[u].w, o.w));
        }
        // nothing changes a row of NaN any more
        if (__all_sync(FULL, sum != sum || (o.x != o.x && o.y != o.y && o.z != o.z && o.w != o.w))) break;
    }
    if (n == 0) return o;
    const float r = 1.0f / sum;
    return make_float4(o.x * r, o.y * r, o.z * r, o.w * r);
}

// ---- rows that are computed again ----------------------------------------------------------------
// A tile of rows under one kv head shares the products of its key tiles, so 0 times a value that a row does not see may
// make that row NaN, and elements near the end of a type's range may overflow on the way.  Rows that come out as no
// numbers are computed again from the formula, unless that can only give NaN once more: a key or value that is NaN, where
// all else is ordinary, is not looked for again in every row that sees it.
// What one warp finds out about a tile of rows.
template <typename TC> struct SecondLook {
    int tile = -1;           // looked at; of it:
    int last;                // the last position that not all rows see whose value is no finite number, or -1
    bool huge;               // the keys or values hold infinities or elements from 2^100 on
    // The first row of tile `id` sees the keys 0 .. lo - 1, and its key tiles end at hi.
    __device__ __forceinline__ void look(int id, const PagedKV &c, const PagedSeqs &b, int s, int head, int lo, int hi) {
        if (tile == id) return;
        tile = id;
        last = -1;
        huge = false;
        typedef typename Elem<TC>::type E;
        const int lane = threadIdx.x & 31;
        for (int t = hi - 1; t >= lo && last < 0; t -= 4) {
            bool odd[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int page = t - u >= lo ? paged_page(b, c, s, t - u, nullptr) : -1;
                odd[u] = page >= 0 && !all_finite(load_quad(static_cast<const E *>(c.v) + paged_at(c, page, head, t - u) + 4 * lane));
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (__any_sync(FULL, odd[u]) && last < 0) last = t - u;
        }
        // the positions of a page lie one after the other: 16 bytes a lane
        constexpr int STEP = 16 / Elem<TC>::BYTES * 32;      // elements of a load by the warp
        for (int t = 0; t < hi && !huge; t += 16) {
            const int page = paged_page(b, c, s, t, nullptr);
            if (page < 0) continue;
            const int64_t at = paged_at(c, page, head, t) + lane * (16 / Elem<TC>::BYTES);
            const int n = min(16, hi - t) * HD / STEP;       // loads (a position is half of one, or one)
            for (int side = 0; side < 2; ++side) {
                const E *p = static_cast<const E *>(side ? c.v : c.k) + at;
                uint32_t top = 0;                            // the largest magnitude that is no NaN
#pragma unroll 4
                for (int u = 0; u < n; ++u) top = max(top, magnitude(p + u * STEP));
                if (n * STEP < min(16, hi - t) * HD && lane < 16) top = max(top, magnitude(p + n * STEP));
                huge |= top >= 0x71800000u;
            }
            huge = __any_sync(FULL, huge);
        }
    }
    // whether a row that sees `limit` keys is to be computed again (q: its query, a quad a lane)
    __device__ __forceinline__ bool wanted(int limit, float4 q) const {
        const float top = fmaxf(fmaxf(fabsf(q.x), fabsf(q.y)), fmaxf(fabsf(q.z), fabsf(q.w)));
        return huge || limit <= last || __any_sync(FULL, top >= 0x1p100f);
    }
    static __device__ __forceinline__ uint32_t no_nan(uint32_t bits) {
        bits &= 0x7fffffffu;
        return bits > 0x7f800000u ? 0u : bits;
    }
    // the largest magnitude, as binary32's bits, of 16 bytes of elements that are no NaN
    static __device__ __forceinline__ uint32_t magnitude(const typename Elem<TC>::type *p) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (Elem<TC>::BYTES == 4) top = max(top, no_nan(x[i]));
            else top = max(top, max(no_nan(x[i] << 16), no_nan(x[i] & 0xffff0000u)));
        }
        return top;
    }
};
// Over a Q8_0 cache only a scale can be no finite number, or large.
template <> struct SecondLook<q8raw> {
    int tile = -1, last;
    bool huge;
    __device__ __forceinline__ void look(int id, const PagedKV &c, const PagedSeqs &b, int s, int head, int lo, int hi) {
        if (tile == id) return;
        tile = id;
        last = -1;
        huge = false;
        const int lane = threadIdx.x & 31;
        // 16 positions, which one page holds: a lane looks at one scale of K and of V
        for (int t = 0; t < hi; t += 16) {
            const int page = paged_page(b, c, s, t, nullptr), at = t + (lane >> 1);
            if (page < 0) continue;
            float k = 0.0f, v = 0.0f;
            if (at < hi) {
                const int64_t i = paged_scale_at(c, page, head, t) + lane;
                k = fabsf(c.k_scale[i]);
                v = fabsf(c.v_scale[i]);
            }
            huge |= __any_sync(FULL, k >= 0x1p93f || v >= 0x1p93f);          // times 127: 2^100
            const unsigned odd = __ballot_sync(FULL, at >= lo && !(v < INFINITY));
            if (odd) last = t + ((31 - __clz(odd)) >> 1);
        }
    }
    __device__ __forceinline__ bool wanted(int limit, float4 q) const {
        const float top = fmaxf(fmaxf(fabsf(q.x), fabsf(q.y)), fmaxf(fabsf(q.z), fabsf(q.w)));
        return huge || limit <= last || __any_sync(FULL, top >= 0x1p100f);
    }
};

// ---- the work items of a prompt launch ------------------------------------------------------
// A sequence's rows fall into blocks of `per_block` queries; a block under one kv head is an item.  Its work is the
// number of key tiles that its last row sees.
struct PromptItem {
    int s, head;             // sequence (-1: none), kv head
    int first, rows, len;    // first query row within the sequence; the sequence's rows and keys
    int base, pos0;          // the sequence's first packed row and its position
    __host__ __device__ __forceinline__ int seen(int i) const {            // keys that the sequence's row i sees
        const int n = pos0 + i + 1;                          // at most the sequence's kv_len
        return n < 0 ? 0 : n < len ? n : len;
    }
};
// What a lane knows of its sequence.
struct PromptSeq {
    int base, pos0, rows, blocks, len;
    // blocks whose last row sees at least `keys` keys
    __host__ __device__ __forceinline__ int at_least(int keys, const FastDiv &per_block) const {
        if (keys > len) return 0;
        const int need = keys - pos0;                        // rows that it takes: at most all
        return keys <= 0 || need <= 0 ? blocks : blocks - per_block(need - 1);
    }
};
__host__ __device__ __forceinline__ PromptSeq prompt_seq(const PagedSeqs &b, const PagedKV &c, int total_rows,
                                                         const FastDiv &per_block, int s, uint32_t *status) {
    PromptSeq q = {0, 0, 0, 0, 0};
    if (s >= b.n_seqs) return q;
    int lo = b.row_off[s], hi = b.row_off[s + 1];
    if (hi > total_rows) hi = total_rows;
    if (lo < 0 || hi <= lo) return q;                        // no rows, or offsets that do not rise
    const int kv_len = b.kv_len[s];
    q.base = lo;
    q.rows = hi - lo;
    q.blocks = per_block(q.rows - 1) + 1;
    q.pos0 = (kv_len < 0 ? 0 : kv_len) - q.rows;
    q.len = paged_len(b, c, s, status);
    return q;
}
__device__ __forceinline__ int lanes_before(int x) {         // sum over the lanes below this one
    int y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(FULL, y, o);
        if ((threadIdx.x & 31) >= o) y += z;
    }
    return y - x;
}
// The order of a launch's items: kv heads innermost, blocks from the most key tiles to the fewest, so that no long item
// begins last.  Held by one warp, lane l with sequences l and l + 32; find() returns the same in every lane.  It takes any
// indices, rising ones quickest: a smaller one than before begins the search anew (the CTAs that are taken over come in no
// promised order).  A block's place is found by the number of tiles at which the count of larger blocks passes its index:
// the level of the item before or the next lower one mostly, bisection otherwise.
// Past PROMPT_SORTED sequences, which the lanes cannot hold, an index is a slot: the blocks of sequence s begin at slot
// row_off[s] / per_block + s, the last block first.  Each sequence has a slot for each of its blocks, as
// ceil(r / d) <= floor((o + r) / d) - floor(o / d) + 1, and there are as many slots as a launch has indices; some are
// empty (an item without rows).  So an index is found by a search of a few rounds, where a walk along the sequences made
// the launch quadratic in them: 52 ms for 20,000 f32 prompts of one row, now 3.1.
constexpr int PROMPT_SORTED = 64;
struct PromptOrder {
    PromptSeq q[2];
    const PagedSeqs &b;
    const PagedKV &c;
    const FastDiv &per_block;
    int total_rows, tile_keys;
    uint32_t *status;
    int latest;              // the latest index, of blocks
    int hi, above;           // blocks of at least hi tiles are `above`, no more than the latest index

    __device__ __forceinline__ PromptOrder(const PagedSeqs &b_, const PagedKV &c_, int total_rows_, const FastDiv &per_block_,
                                           int tile_keys_, uint32_t *status_)
        : b(b_), c(c_), per_block(per_block_), total_rows(total_rows_), tile_keys(tile_keys_), status(status_) {
        const int lane = threadIdx.x & 31;
        const bool sorted = b.n_seqs <= PROMPT_SORTED;
        q[0] = prompt_seq(b, c, total_rows, per_block, sorted ? lane : b.n_seqs, status);
        q[1] = PromptSeq{0, 0, 0, 0, 0};
        if (sorted && b.n_seqs > 32) q[1] = prompt_seq(b, c, total_rows, per_block, lane + 32, status);
        restart();
    }
    __device__ __forceinline__ void restart() {
        hi = (max(__reduce_max_sync(FULL, q[0].len), __reduce_max_sync(FULL, q[1].len)) + tile_keys - 1) / tile_keys + 1;
        latest = above = 0;
    }
    __device__ __forceinline__ int at_least(int x, int tiles) const {
        return q[x].at_least(tiles ? (tiles - 1) * tile_keys + 1 : 0, per_block);
    }
    __device__ __forceinline__ int count(int tiles) const {
        return int(__reduce_add_sync(FULL, at_least(0, tiles) + (b.n_seqs > 32 ? at_least(1, tiles) : 0)));
    }
    static __device__ __forceinline__ void take(PromptItem &it, const PromptSeq &from, int s, int l, int first) {
        it.s = s;
        it.rows = __shfl_sync(FULL, from.rows, l);
        it.len = __shfl_sync(FULL, from.len, l);
        it.base = __shfl_sync(FULL, from.base, l);
        it.pos0 = __shfl_sync(FULL, from.pos0, l);
        it.first = __shfl_sync(FULL, first, l);
    }
    // The last sequence whose slots begin at or before `slot`, and where.  33-way search: two rounds of loads for up to
    // 1,023 sequences.
    __device__ __forceinline__ int slot_seq(int slot, int &begin) const {
        const int lane = threadIdx.x & 31;
        int lo = 0, hi = b.n_seqs;
        begin = 0;
        do {
            const int step = (hi - lo + 30) / 31, p = lane == 31 ? hi : min(lo + lane * step, hi);
            const int x = per_block(max(0, min(b.row_off[p], total_rows))) + p;
            const unsigned below = __ballot_sync(FULL, x <= slot && p < hi) & 0x7fffffffu;
            const int l = below ? 31 - __clz(below) : 0;
            begin = __shfl_sync(FULL, x, l);
            lo = __shfl_sync(FULL, p, l);
            hi = __shfl_sync(FULL, p, l + 1);
        } while (hi - lo > 1);
        return lo;
    }
    __device__ __forceinline__ PromptItem find(int64_t index) {
        PromptItem it;
        it.s = -1;
        it.head = int(uint32_t(index) % uint32_t(c.n_kv));
        int left = int(uint32_t(index) / uint32_t(c.n_kv));
        const int lane = threadIdx.x & 31;
        if (b.n_seqs > PROMPT_SORTED) {
            int begin;
            it.s = slot_seq(left, begin);
            const PromptSeq p = prompt_seq(b, c, total_rows, per_block, it.s, lane == 0 ? status : nullptr);
            const int block = p.blocks - 1 - (left - begin);
            const bool there = block >= 0 && left >= begin;
            it.first = there ? block * per_block.d : 0;
            it.rows = there ? p.rows : 0;
            it.len = there ? p.len : 0;
            it.base = p.base;
            it.pos0 = p.pos0;
            return it;
        }
        if (left < latest) restart();
        latest = left;
        if (b.n_seqs == 1) {
            const int blocks = __shfl_sync(FULL, q[0].blocks, 0);
            if (left < blocks) take(it, q[0], 0, 0, (blocks - 1 - left) * per_block.d);
            return it;
        }
        // to the level with above <= left < count(hi - 1)
        int down = hi > 0 ? count(hi - 1) : 0;
        if (down <= left) {
            const int all = count(0);
            if (hi == 0 || left >= all) return it;           // there are no more
            int lo = 0, top = hi - 1;                        // count(lo) > left >= count(top)
            above = down;
            down = all;
            while (top - lo > 1) {
                const int mid = (lo + top) >> 1, n = count(mid);
                if (n > left) lo = mid, down = n;
                else top = mid, above = n;
            }
            hi = top;
        }
        left -= above;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int more = at_least(x, hi), equal = at_least(x, hi - 1) - more, before = lanes_before(equal);
            const unsigned hit = __ballot_sync(FULL, left >= before && left < before + equal);
            if (hit) {
                const int l = __ffs(hit) - 1;
                take(it, q[x], 32 * x + l, l, (q[x].blocks - more - 1 - (left - before)) * per_block.d);
                return it;
            }
            left -= __reduce_add_sync(FULL, equal);
        }
        return it;
    }
};

// ---- items that a cluster shares --------------------------------------------------------------
// When there are fewer items than SMs, a cluster of CTAs takes an item: part p of its key tiles goes to the CTA of rank
// p, and the parts' unnormalised results are joined through the cluster's shared memory, which costs about 4 us.  A part
// has at least PROMPT_PART tiles, and an item of fewer than `least` tiles stays whole (bf16, tiles of 128 keys of 1.3 us:
// 600 keys take 19 us whole and 23 in two parts, 1,000 keys 22 and, in four, 17; f32, tiles of 64 keys of 1.9 us: 500
// keys 27 whole and 20 in four).
constexpr int PROMPT_PART = 2;
__host__ __device__ __forceinline__ int prompt_parts(int ctas, int tiles, int least) {
    return tiles < least ? 1 : tiles / PROMPT_PART < ctas ? tiles / PROMPT_PART : ctas;
}
// First tile of part p (of `parts`: behind the last).
__host__ __device__ __forceinline__ int prompt_part(int tiles, int parts, int p) { return int(int64_t(tiles) * p / parts); }

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// A row of `parts` parts by one warp: its results lie, 16-byte chunk x of the 128 floats at x ^ (r % 8), at `row` of each
// CTA's shared memory, and (maximum, sum) at `stat`; a negative sum marks a part that was given up, which makes `ok`
// false.  Returns lane's chunk; `scale` makes scores base-2 exponents.
__device__ __forceinline__ float4 join_parts(uint32_t row, uint32_t stat, int r, int parts, float scale, bool &ok) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY, l = 0.0f;
    if (lane < parts)
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(m), "=f"(l) : "r"(peer_smem(stat, lane)) : "memory");
    ok = !__any_sync(FULL, l < 0.0f);
    float top = m;
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, x));
    const float w = m == -INFINITY ? 0.0f : ex2_approx_ftz((m - top) * scale);
    float sum = w * l;
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) sum += __shfl_xor_sync(FULL, sum, x);
    const float inv = 1.0f / __shfl_sync(FULL, sum, 0);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p = 0; p < parts; ++p) {
        const float f = __shfl_sync(FULL, w, p);
        float4 v;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                     : "r"(peer_smem(row + uint32_t((lane ^ (r & 7)) << 4), p)) : "memory");
        o = make_float4(fmaf(f, v.x, o.x), fmaf(f, v.y, o.y), fmaf(f, v.z, o.z), fmaf(f, v.w, o.w));
    }
    return make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// Scores from column n of 32 on become -inf.
__device__ __forceinline__ void mask32(uint32_t *v, int n) {
#pragma unroll
    for (int y = 0; y < 32; ++y)
        if (y >= n) v[y] = 0xff800000u;
}

constexpr float ATT_SCALE = 0.08838834764831845f;            // 1/sqrt(128)

}  // namespace q3
