// q3cu_split.cuh -- one-token attention cut into equal runs of tiles: the cut, the place of a tile in the batch, and the
// join of what the runs leave (k_paged.cu, k_paged_q8.cu and the sequences' own part of k_shared.cu).
#pragma once

#include "q3cu_paged.cuh"

namespace q3 {

constexpr float PD_LOG2 = ATT_SCALE * 1.44269504088896341f;  // scores to base-2 exponents
constexpr int PD_PART = HD + 2;                              // floats of a row's partial result: 128, maximum, sum

// a / b for 0 <= a, 0 < b: 32-bit division where it serves (a 64-bit one is a chain of some hundred instructions).
// (This and the cut below host and device: their arithmetic is also checked on the CPU.)
__host__ __device__ __forceinline__ int64_t quot(int64_t a, int b) {
    return a < (int64_t(1) << 32) ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

// How `total` tiles are cut into `runs` runs: the first `more` have each + 1 tiles, the others `each`.
struct PagedCut {
    int64_t total, each;
    int more;
    __host__ __device__ __forceinline__ PagedCut(int64_t t, int runs) : total(t), each(quot(t, runs)), more(int(t - each * runs)) {}
    __host__ __device__ __forceinline__ int64_t begin(int run) const { return each * run + (run < more ? run : more); }
    __host__ __device__ __forceinline__ int run_of(int64_t u) const {        // u < total
        const int64_t edge = (each + 1) * more;
        return u < edge ? int(each < INT32_MAX ? quot(u, int(each + 1)) : u / (each + 1))
                        : more + int(each < INT32_MAX ? quot(u - edge, int(each)) : (u - edge) / each);
    }
};
// Where the parts of an item lie that begins with unit `begin` and has its tiles in units a .. z - 1 (a < z): in the first slots
// of runs first .. first + n - 1, but the first of them in its run's second slot if the run began with another item (`late`).
struct PartsOf {
    int first, n;
    bool late;
    __host__ __device__ __forceinline__ PartsOf(const PagedCut &cut, int64_t begin, int64_t a, int64_t z)
        : first(cut.run_of(a)), n(cut.run_of(z - 1) - first + 1), late(begin > cut.begin(first)) {}
    __host__ __device__ __forceinline__ int64_t slot(int i) const { return 2 * int64_t(first + i) + (i == 0 && late); }
};

// Positions from .. len - 1 of a sequence that one-token attention goes through, one tile after the other.  The first tile
// begins at a multiple of TAIL_ALIGN, and may hold positions before `from`.  (At a multiple of its size, with boxes as large:
// 143 against 141 us for 150 sequences behind 12,001 Q8_0 positions; boxes of 16 rows cost more than they save.)
constexpr int TAIL_ALIGN = 32;                               // rows of a box, at most, where `from` is not 0
struct PagedSpan {
    int from, len;
    __host__ __device__ __forceinline__ int base() const { return from & -TAIL_ALIGN; }
    __host__ __device__ __forceinline__ int tiles(int tile) const { return len > from ? (len - base() + tile - 1) / tile : 0; }
    template <int TILE> __host__ __device__ __forceinline__ int tiles() const { return tiles(TILE); }
};
// The batch's whole sequences.
struct WholeSeqs : PagedSeqs {
    static constexpr bool TAILS = false;
    __device__ __forceinline__ PagedSpan span(const PagedKV &c, int s, uint32_t *status) const {
        return {0, paged_len(*this, c, s, status)};
    }
};

// What a group of sequences shares: sequences off[g] .. off[g+1] - 1 have their first len[g] positions in common, on the
// pages of the group's first.
struct PagedGroups {
    const int32_t *off, *len;
    int n;
    // Sequences of group g: none where the offsets do not rise within the batch.
    __host__ __device__ __forceinline__ int count(int g, int n_seqs) const {
        const int a = off[g], z = off[g + 1];
        return a >= 0 && z <= n_seqs && a < z ? z - a : 0;
    }
    // Positions that the group's first sequence holds and all have in common; one sequence alone shares nothing, and neither
    // do those whose first holds fewer (its slot may have been freed, and its page ids be another's).
    __host__ __device__ __forceinline__ int shared(int g, const PagedSeqs &b, const PagedKV &c, uint32_t *status) const {
        const int64_t cap = int64_t(b.max_pages) << c.page_shift;
        const int n = len[g];
        if (n <= 0 || count(g, b.n_seqs) < 2) return 0;
        if (n > cap) flag_bad_index(status);
        const int cut = int(n > cap ? cap : n);
        return paged_len(b, c, off[g], nullptr) < cut ? 0 : cut;
    }
    // The group of sequence s, or -1.
    __host__ __device__ __forceinline__ int of(int s, int n_seqs) const {
        int lo = 0, hi = n;                                  // off[lo] <= s < off[hi], if any does
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (off[mid] <= s) lo = mid;
            else hi = mid;
        }
        return n > 0 && count(lo, n_seqs) > 0 && off[lo] <= s && s < off[lo + 1] ? lo : -1;
    }
};
// The batch's sequences behind what they share, as a launch before this one planned them (SharedPlan).  A (sequence, head) of
// T tiles is TAIL_LEAD + T units of the cut: what it costs to begin and end one is worth about two tiles.
constexpr int TAIL_LEAD = 2;
constexpr int SHARED_ROW = 136;                              // floats of a row's part there: 128, maximum, sum (32-byte aligned)
struct TailSeqs : PagedSeqs {
    static constexpr bool TAILS = true;
    const int2 *spans;       // from, len
    const int64_t *before;   // [n_seqs + 1] units of the sequences before, of one kv head
    __device__ __forceinline__ PagedSpan span(const PagedKV &, int s, uint32_t *) const {
        const int2 x = spans[s];
        return {x.x, x.y};
    }
};

// Unit `at` of a sequence of `tiles` tiles: kv head, tile, and units before the tile.
__host__ __device__ __forceinline__ void tail_place(int64_t at, int tiles, int &head, int &tile, int &lead) {
    head = int(quot(at, TAIL_LEAD + tiles));
    const int unit = int(at - int64_t(head) * (TAIL_LEAD + tiles));
    tile = unit > TAIL_LEAD ? unit - TAIL_LEAD : 0;
    lead = unit < TAIL_LEAD ? TAIL_LEAD - unit : 0;
}

// A place in the batch's tiles: sequence, kv head, tile, and the sequence's span and tiles.
struct PagedWalk {
    int s, head, tile, from, len, tiles;
    int lead;                // tails: units before the tile
    template <int TILE, typename Seqs> __device__ __forceinline__ int pos(int at) const {    // of tile `at`'s first row
        return (Seqs::TAILS ? from & -TAIL_ALIGN : 0) + at * TILE;
    }
};

// Inclusive sum over the lanes; 32 sequences have at most 2^31 / 32 tiles each.
__device__ __forceinline__ uint32_t warp_prefix(uint32_t x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(FULL, x, o);
        if ((threadIdx.x & 31) >= o) x += y;
    }
    return x;
}
// The tiles of the whole batch, the run's [u0, u1) of them and the place of u0 (one warp; every lane returns it).
template <int TILE, typename Seqs>
__device__ __forceinline__ PagedWalk walk_run(const Seqs &b, const PagedKV &c, int run, int runs, PagedCut &cut,
                                              int64_t &u0, int64_t &u1, uint32_t *status) {
    PagedWalk w = {};
    const int lane = threadIdx.x & 31;
    if constexpr (Seqs::TAILS) {
        // up to 256 sequences are searched in one round of loads
        constexpr int ROUND = 8;
        cut = PagedCut(b.before[b.n_seqs] * c.n_kv, runs);
        u0 = cut.begin(run);
        u1 = cut.begin(run + 1);
        if (u0 == u1) return w;
        for (int s0 = 0; s0 < b.n_seqs; s0 += 32 * ROUND) {
            int64_t x[ROUND];                                // of sequences s0 + 32 r + lane
#pragma unroll
            for (int r = 0; r < ROUND; ++r) x[r] = b.before[min(s0 + 32 * r + lane, b.n_seqs)];
            const int64_t end = b.before[min(s0 + 32 * ROUND, b.n_seqs)];
            if (u0 >= end * c.n_kv) continue;
#pragma unroll
            for (int r = ROUND - 1; r >= 0; --r) {           // the last sequence that begins at or before u0
                const unsigned hit = __ballot_sync(FULL, s0 + 32 * r + lane < b.n_seqs && x[r] * c.n_kv <= u0);
                if (hit) {
                    const int l = 31 - __clz(hit);
                    w.s = s0 + 32 * r + l;
                    const PagedSpan mine = b.span(c, w.s, nullptr);
                    w.from = mine.from;
                    w.len = mine.len;
                    w.tiles = mine.tiles<TILE>();
                    tail_place(u0 - __shfl_sync(FULL, x[r], l) * c.n_kv, w.tiles, w.head, w.tile, w.lead);
                    return w;
                }
            }
        }
        return w;
    }
    int64_t total = 0;                                       // in tiles of one kv head
    uint32_t end = 0;
    PagedSpan len = {0, 0};
    for (int s0 = 0; s0 < b.n_seqs; s0 += 32) {              // 32 sequences at a time
        len = s0 + lane < b.n_seqs ? b.span(c, s0 + lane, status) : PagedSpan{0, 0};
        end = warp_prefix(uint32_t(len.template tiles<TILE>()));
        total += __shfl_sync(FULL, end, 31);
    }
    cut = PagedCut(total * c.n_kv, runs);
    u0 = cut.begin(run);
    u1 = cut.begin(run + 1);
    int64_t u = u0;
    for (int s0 = 0; s0 < b.n_seqs; s0 += 32) {
        if (b.n_seqs > 32) {                                 // otherwise the lanes still hold them
            len = s0 + lane < b.n_seqs ? b.span(c, s0 + lane, nullptr) : PagedSpan{0, 0};
            end = warp_prefix(uint32_t(len.template tiles<TILE>()));
        }
        const unsigned hit = __ballot_sync(FULL, u < int64_t(end) * c.n_kv);
        if (hit) {
            const int l = __ffs(hit) - 1;
            w.s = s0 + l;
            w.len = __shfl_sync(FULL, len.len, l);
            w.tiles = PagedSpan{0, w.len}.tiles<TILE>();
            const int64_t at = u - int64_t(__shfl_sync(FULL, end, l) - uint32_t(w.tiles)) * c.n_kv;
            w.head = int(quot(at, w.tiles));
            w.tile = int(at - int64_t(w.head) * w.tiles);
            return w;
        }
        u -= int64_t(__shfl_sync(FULL, end, 31)) * c.n_kv;
    }
    return w;
}
// `n` tiles further, which lie in the same (sequence, head) or begin the next one that has any (one warp: 32 sequences at
// a time, so that a million empty ones take 3 ms and not 100, while others wait).
template <int TILE, typename Seqs>
__device__ __forceinline__ void walk_on(const Seqs &b, const PagedKV &c, PagedWalk &w, int n) {
    w.tile += n;
    w.lead = 0;
    if (w.tile < w.tiles) return;
    w.tile = 0;
    if (Seqs::TAILS) w.lead = TAIL_LEAD;
    if (++w.head < c.n_kv) return;
    w.head = 0;
    for (++w.s; w.s < b.n_seqs; w.s += 32) {
        const int s = w.s + int(threadIdx.x & 31);
        const PagedSpan x = s < b.n_seqs ? b.span(c, s, nullptr) : PagedSpan{0, 0};
        const unsigned some = __ballot_sync(FULL, x.len > x.from);
        if (some) {
            const int l = __ffs(some) - 1;
            w.s += l;
            w.from = Seqs::TAILS ? __shfl_sync(FULL, x.from, l) : 0;
            w.len = __shfl_sync(FULL, x.len, l);
            w.tiles = PagedSpan{w.from, w.len}.tiles<TILE>();
            return;
        }
    }
}

// One pair of result elements (row, dims at, at + step) as the output's type.
__device__ __forceinline__ void put2(float *p, int step, float x, float y) { p[0] = x, p[step] = y; }
__device__ __forceinline__ void put2(uint16_t *p, int step, float x, float y) {
    if (step == 1) *reinterpret_cast<uint32_t *>(p) = pack_bf16(x, y);
    else p[0] = uint16_t(f32_to_bf16(x)), p[step] = uint16_t(f32_to_bf16(y));
}

// Joins what the runs left of one query head, one CTA per run and head of the group; the CTA of the second run of a
// (sequence, kv head) does it: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  The
// parts' maxima and sums are read side by side, one thread each; then two groups of 128 threads (thread = element) add
// half of the weighted parts each, eight loads under way at a time.  The order of every sum is fixed.
constexpr int PJ_GROUPS = 2, PJ_THREADS = PJ_GROUPS * HD, PJ_RUNS = 1024;
template <typename T, int TILE>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const PagedKV c, const WholeSeqs b, int n_heads, int group,
                                                                int runs, typename Elem<T>::type *out, const float *part) {
    __shared__ float weight[PJ_RUNS], red[2][PJ_THREADS / 32], sum[PJ_GROUPS][HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = threadIdx.x % HD, half_id = threadIdx.x / HD;
    // Before the wait: the lengths are older than the first kernel, which has begun (this one starts when all its CTAs
    // have passed their own wait).
    PagedCut cut(0, 1);
    int64_t u0, u1;
    const int second = int(blockIdx.x) + 1;
    const PagedWalk w = walk_run<TILE>(b, c, second, runs, cut, u0, u1, nullptr);
    const int64_t a = u0 - w.tile;                           // the (sequence, head)'s first tile
    const int first = second - 1;
    // it has tiles, does not begin with a new (sequence, head), and is the second of that one's runs
    const bool joins = u0 != u1 && w.tile != 0 && a >= cut.begin(first);
    // The first CTA waits whatever it finds: the next launch waits for this grid alone, which must not end before the first
    // kernel.  (Were all to wait: 1.6 us more for nine ragged sequences, since not all fit beside that kernel.)
    if (!joins && blockIdx.x + blockIdx.y > 0) return;
    griddep_wait();
    if (!joins) return;
    const int last = cut.run_of(a + w.tiles - 1), n = last - first + 1;
    // part i: in the first slot of run first + i, but the second of a run that began before this (sequence, head)
    const float *row = part + int(blockIdx.y) * PD_PART;
    const int64_t run_stride = int64_t(2) * group * PD_PART;
    const float *head = row + first * run_stride + (a != cut.begin(first) ? group * PD_PART : 0);
    auto at = [&](int i) { return i == 0 ? head : row + (first + i) * run_stride; };
    // the first parts of this thread's half are on their way together with the maxima and sums
    const int i0 = n * half_id / PJ_GROUPS, i1 = n * (half_id + 1) / PJ_GROUPS;
    float v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = i0 + x < i1 ? at(i0 + x)[d] : 0.0f;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < n; i += PJ_THREADS) {
        weight[i] = at(i)[HD];
        m = fmaxf(m, weight[i]);
    }
    m = warp_max(m);
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
    m = warp_max(red[0][lane % (PJ_THREADS / 32)]);
    float l = 0.0f;
    for (int i = threadIdx.x; i < n; i += PJ_THREADS) {
        const float f = weight[i] == m ? 1.0f : ex2_approx_ftz((weight[i] - m) * PD_LOG2);
        weight[i] = f;
        l = fmaf(at(i)[HD + 1], f, l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(FULL, l, o);
    if (lane == 0) red[1][warp] = l;
    __syncthreads();
    float o = 0.0f;
#pragma unroll
    for (int x = 0; x < 8; ++x)
        if (i0 + x < i1) o = fmaf(v[x], weight[i0 + x], o);
#pragma unroll 8
    for (int i = i0 + 8; i < i1; ++i) o = fmaf(at(i)[d], weight[i], o);
    sum[half_id][d] = o;
    __syncthreads();
    if (half_id) return;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < PJ_THREADS / 32; ++i) l += red[1][i];
    o = (sum[0][d] + sum[1][d]) / l;
    typename Elem<T>::type *dst = out + (int64_t(w.s) * n_heads + w.head * group + blockIdx.y) * HD + d;
    if constexpr (Elem<T>::BYTES == 4) *dst = o;
    else *dst = uint16_t(f32_to_bf16(o));
}

static inline int paged_runs(int sms) { return 2 * sms < PJ_RUNS ? 2 * sms : PJ_RUNS; }

template <typename T, int TILE>
static cudaError_t launch_paged_join(const PagedKV &c, const PagedSeqs &b, int n_heads, int runs, void *out, const float *part,
                                     cudaStream_t stream) {
    const int group = n_heads / c.n_kv;
    return launch_dependent(paged_join_kernel<T, TILE>, dim3(runs - 1, group), dim3(PJ_THREADS), 0, stream, c, WholeSeqs{b},
                            n_heads, group, runs, static_cast<typename Elem<T>::type *>(out), part);
}

// The sequences' own part of attention_shared: the first kernel of one-token attention, over tails.
cudaError_t launch_tails_bf16(const PagedKV &c, const TailSeqs &b, const void *q, int64_t q_stride, int n_heads, float *part,
                              float *tails, void *out, uint32_t *status, cudaStream_t stream, int runs);
cudaError_t launch_tails_q8(const PagedKV &c, const TailSeqs &b, const void *q, int64_t q_stride, int n_heads, float *part,
                            float *tails, void *out, uint32_t *status, cudaStream_t stream, int runs);
constexpr int PD_TAIL_BF16 = 64, PD_TAIL_Q8 = 128;           // positions of a tile

}  // namespace q3
