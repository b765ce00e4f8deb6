// k_paged.cu -- attention of one new token per sequence over the paged cache.
//
// Query head h of sequence s: o = sum_t softmax_t(q . k_t / sqrt(128)) v_t over
// its kv_len positions, in one pass with the running maximum and sum of the
// softmax.  Bound by memory: every key and value of the batch is read once, for
// all the query heads of its kv head together.
//
// The split.  Lengths are ragged and known to the device only, so the unit of
// work is a tile of positions of one (sequence, kv head): all tiles, in the
// order sequence, head, position, are cut into one equal run per CTA, two CTAs
// on each SM.  A run that covers all tiles of a (sequence, head) writes its
// result; one that begins or ends inside leaves maximum, sum and unnormalised
// result in the workspace (at most two per CTA), and a second kernel joins
// those.  One long sequence spreads over the whole GPU just as a full batch does.
//
// A CTA is one fetching warp and four computing warps around a ring of three
// 32 KB stages, filled page by page by TMA (128-byte swizzle).  A stage is K
// and V of 64 positions in bf16 or 32 in f32; each computing warp takes 16 of
// them (of every other stage in f32), with its own running maximum, sum and
// result, and the four are joined when the run leaves the (sequence, head).
//
// The products run on mma.sync with 16 positions as the rows and eight query
// heads as the columns, scores = K Q^T and result = V^T P^T, so that a group of
// eight heads or fewer leaves none of a product unused beyond its missing heads;
// the keys and values are read as they lie.  They lose nothing that an f32 result
// would show: an f32 query against a bf16 cache is three bf16 parts (the keys are
// exact), and so is a probability, two where the result is bf16; an f32 cache is
// multiplied as tf32 parts, high x high + high x low + low x high, whose remainder
// is 2^-22 of the product.  Sums are binary32.
//
// Positions at and beyond the length score -inf, and their values are masked to
// zero in registers: unused page space may hold anything.
//
// Measured: 64 sequences of up to 16,384 (32/8 heads, f32 queries, bf16 cache)
// 332 to 345 us, 6.1 to 6.4 TB/s; of up to 8,192 over an f32 cache (32/8) 341 us, 6.5
// TB/s, but 83 us, 3.4 TB/s, with 16 query heads to a kv head (instructions of two
// blocks of products to each key, and a join of 4,720 CTAs; bf16 51 us, 2.7 TB/s);
// one of 100,003 (bf16) 71 us, 5.8 TB/s, where the CTAs'
// equal shares end up to 12 us apart; one of 512 (16/8, f32) 8.5 us, all latency.
#include "q3cu_mma.cuh"
#include "q3cu_paged.cuh"
#include "q3cu_tma.h"

namespace q3 {

constexpr int PD_WARPS = 4, PD_THREADS = (PD_WARPS + 1) * 32;
constexpr int PD_NS = 3;                                     // stages
constexpr uint32_t PD_SIDE = 16384, PD_STAGE = 2 * PD_SIDE;  // K or V of a stage; both
constexpr int PD_SPARE = 12288;                              // queries (f32 cache, at most 8 KB), then the join of the warps
constexpr size_t PD_SMEM = size_t(PD_NS) * PD_STAGE + PD_SPARE + 1024;
constexpr float PD_LOG2 = ATT_SCALE * 1.44269504088896341f;  // scores to base-2 exponents
constexpr int PD_PART = HD + 2;                              // floats of a row's partial result: 128, maximum, sum

template <typename TC> __host__ __device__ constexpr int pd_tile() { return int(PD_SIDE) / (HD * Elem<TC>::BYTES); }   // positions of a stage

// a / b for 0 <= a, 0 < b: 32-bit division where it serves (a 64-bit one is a chain of some hundred instructions).
__device__ __forceinline__ int64_t quot(int64_t a, int b) {
    return a < (int64_t(1) << 32) ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

// How `total` tiles are cut into `runs` runs: the first `more` have each + 1 tiles, the others `each`.
struct PagedCut {
    int64_t total, each;
    int more;
    __device__ __forceinline__ PagedCut(int64_t t, int runs) : total(t), each(quot(t, runs)), more(int(t - each * runs)) {}
    __device__ __forceinline__ int64_t begin(int run) const { return each * run + min(run, more); }
    __device__ __forceinline__ int run_of(int64_t u) const {                 // u < total
        const int64_t edge = (each + 1) * more;
        return u < edge ? int(each < INT32_MAX ? quot(u, int(each + 1)) : u / (each + 1))
                        : more + int(each < INT32_MAX ? quot(u - edge, int(each)) : (u - edge) / each);
    }
};

// A place in the batch's tiles: sequence, kv head, tile, and the sequence's length and tiles.
struct PagedWalk {
    int s, head, tile, len, tiles;
};
template <typename TC>
__device__ __forceinline__ int tiles_of(int len) { return (len + pd_tile<TC>() - 1) / pd_tile<TC>(); }

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
template <typename TC>
__device__ __forceinline__ PagedWalk walk_run(const PagedSeqs &b, const PagedKV &c, int run, int runs, PagedCut &cut,
                                              int64_t &u0, int64_t &u1, uint32_t *status) {
    PagedWalk w = {};
    const int lane = threadIdx.x & 31;
    int64_t total = 0;                                       // in tiles of one kv head
    uint32_t end = 0;
    int len = 0;
    for (int s0 = 0; s0 < b.n_seqs; s0 += 32) {              // 32 sequences at a time
        len = s0 + lane < b.n_seqs ? paged_len(b, c, s0 + lane, status) : 0;
        end = warp_prefix(uint32_t(tiles_of<TC>(len)));
        total += __shfl_sync(FULL, end, 31);
    }
    cut = PagedCut(total * c.n_kv, runs);
    u0 = cut.begin(run);
    u1 = cut.begin(run + 1);
    int64_t u = u0;
    for (int s0 = 0; s0 < b.n_seqs; s0 += 32) {
        if (b.n_seqs > 32) {                                 // otherwise the lanes still hold them
            len = s0 + lane < b.n_seqs ? paged_len(b, c, s0 + lane, nullptr) : 0;
            end = warp_prefix(uint32_t(tiles_of<TC>(len)));
        }
        const unsigned hit = __ballot_sync(FULL, u < int64_t(end) * c.n_kv);
        if (hit) {
            const int l = __ffs(hit) - 1;
            w.s = s0 + l;
            w.len = __shfl_sync(FULL, len, l);
            w.tiles = tiles_of<TC>(w.len);
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
template <typename TC>
__device__ __forceinline__ void walk_on(const PagedSeqs &b, const PagedKV &c, PagedWalk &w, int n) {
    w.tile += n;
    if (w.tile < w.tiles) return;
    w.tile = 0;
    if (++w.head < c.n_kv) return;
    w.head = 0;
    for (++w.s; w.s < b.n_seqs; w.s += 32) {
        const int s = w.s + int(threadIdx.x & 31), len = s < b.n_seqs ? paged_len(b, c, s, nullptr) : 0;
        const unsigned some = __ballot_sync(FULL, len > 0);
        if (some) {
            const int l = __ffs(some) - 1;
            w.s += l;
            w.len = __shfl_sync(FULL, len, l);
            w.tiles = tiles_of<TC>(w.len);
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

// WIDE: more than 8 query heads to a kv head (two blocks of columns).
template <typename T, typename TC, bool WIDE>
__global__ void __launch_bounds__(PD_THREADS, 2)
paged_split_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const PagedKV c,
                   const PagedSeqs b, const typename Elem<T>::type *q, int64_t q_stride, int n_heads, int group,
                   typename Elem<T>::type *out, float *part, uint32_t *status) {
    constexpr bool CF32 = Elem<TC>::BYTES == 4;
    constexpr int TILE = pd_tile<TC>(), NH = WIDE ? 2 : 1;   // NH: blocks of eight heads
    extern __shared__ uint8_t pd_dyn[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pd_dyn) + 1023) & ~uintptr_t(1023));
    float *spare = reinterpret_cast<float *>(ring + PD_NS * PD_STAGE);
    __shared__ __align__(8) uint64_t full[PD_NS], empty[PD_NS];
    __shared__ float join_m[3][8 * NH], join_l[3][8 * NH];
    __shared__ volatile int dead;                            // a wait gave up
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PD_NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], PD_WARPS);
        }
        mbar_init_fence();
        dead = 0;
    }
    __syncthreads();
    griddep_wait();
    griddep_launch_dependents();

    PagedCut cut(0, 1);
    int64_t u0, u1;
    PagedWalk w = walk_run<TC>(b, c, int(blockIdx.x), int(gridDim.x), cut, u0, u1,
                               blockIdx.x == 0 && warp == 0 ? status : nullptr);
    for (int s = int(blockIdx.x); s < b.n_seqs; s += int(gridDim.x))       // sequences without positions: zeros
        if (b.kv_len[s] <= 0 || b.max_pages == 0)
            for (int i = threadIdx.x; i < n_heads * (HD / 4); i += PD_THREADS)
                store_quad(out + int64_t(s) * n_heads * HD + 4 * i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    if (u0 == u1) return;

    if (warp == PD_WARPS) {
        // ---- fetch: lane = box (K or V, column block, rows of one page) ------------------
        constexpr int TS = CF32 ? 5 : 6, CS = CF32 ? 2 : 1, CB = 1 << CS;     // log2 of TILE; column blocks of 128 B
        const int bs = min(c.page_shift, TS), br = 1 << bs, ns = TS - bs;     // rows of a box; log2 of boxes of a tile
        const int box = lane & ((1 << ns) - 1), col = (lane >> ns) & (CB - 1), side = lane >> (ns + CS);
        auto page_of = [&]() -> int {                        // n_pages reads as zeros
            const int t = w.tile * TILE + box * br;
            if (side > 1 || t >= w.len) return c.n_pages;
            const int p = paged_page(b, c, w.s, t, status);
            return p < 0 ? c.n_pages : p;
        };
        uint8_t *dst = ring + side * PD_SIDE + col * (PD_SIDE / CB) + box * br * 128;
        int page = page_of(), e = 0;
        bool ok = true;
        for (int64_t u = u0; u < u1; ++u, ++e) {
            const int head = w.head, slot = (w.tile * TILE + box * br) & ((1 << c.page_shift) - 1), now = page;
            if (u + 1 < u1) {
                walk_on<TC>(b, c, w, 1);
                page = page_of();                            // under way while this tile waits for its stage
            }
            const int st = e % PD_NS;
            if (e >= PD_NS) ok = mbar_wait(&empty[st], uint32_t(e / PD_NS - 1) & 1u, lane == 0 ? status : nullptr);
            if (!__all_sync(FULL, ok)) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[st], PD_STAGE);
            __syncwarp();
            if (side < 2)
                tma_load_4d(dst + st * PD_STAGE, side ? &tmv : &tmk, (CF32 ? 32 : 64) * col, slot, head, now, &full[st]);
        }
        // no copy outlives the CTA (bounded)
        for (int d = e > PD_NS ? e - PD_NS : 0; d < e; ++d) mbar_wait(&full[d % PD_NS], uint32_t(d / PD_NS) & 1u, nullptr);
        return;
    }

    // ---- the computing warps ---------------------------------------------------------
    const int g = lane >> 2, t4 = lane & 3;                  // products: row g (and g + 8), columns 2 t4 and + 1
    const uint32_t ring_a = smem_addr(ring);
    const int key0 = CF32 ? 16 * (warp & 1) : 16 * warp;     // this warp's 16 positions of a tile
    int e = 0;
    bool ok = true;
    for (int64_t u = u0; u < u1 && ok;) {
        const int run = int(min(int64_t(w.tiles - w.tile), u1 - u));       // tiles of this (sequence, head) here
        const typename Elem<T>::type *qs = q + w.s * q_stride + int64_t(w.head) * group * HD;
        constexpr bool PARTS3 = !CF32 && Elem<T>::BYTES == 4;                // f32 queries, bf16 cache
        uint32_t qf[CF32 || PARTS3 ? 1 : 8][NH][2];          // bf16 queries, bf16 cache: operands in registers
        if constexpr (CF32) {
            // the group's rows in shared memory, zeros below; 16-byte chunk x of row r at x ^ (r % 8) of its 128 bytes
            for (int i = threadIdx.x; i < 8 * NH * (HD / 4); i += PD_WARPS * 32) {
                const int row = i / (HD / 4), ch = i % (HD / 4);
                *reinterpret_cast<float4 *>(spare + row * HD + 4 * ((ch & 24) | ((ch ^ row) & 7))) =
                    row < group ? load_quad(qs + row * HD + 4 * ch) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            named_sync(1, PD_WARPS * 32);
        } else if constexpr (PARTS3) {
            // three bf16 parts of the rows, zeros below; chunk x of row r at x ^ (r % 8)
            for (int i = threadIdx.x; i < 8 * NH * (HD / 2); i += PD_WARPS * 32) {
                const int row = i / (HD / 2), col = 2 * (i % (HD / 2));
                const float2 v = row < group ? *reinterpret_cast<const float2 *>(qs + row * HD + col) : make_float2(0.0f, 0.0f);
                uint32_t part[3];
                split_bf16(v.x, v.y, part);
#pragma unroll
                for (int x = 0; x < 3; ++x)
                    reinterpret_cast<uint32_t *>(spare)[((x * 8 * NH + row) * HD + (col ^ ((row & 7) << 3))) / 2] = part[x];
            }
            named_sync(1, PD_WARPS * 32);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int n = 0; n < NH; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {            // dimensions 16 k + 2 t4 (+ 1), and 8 further
                        const int row = 8 * n + g;
                        qf[k][n][x] = row < group ? *reinterpret_cast<const uint32_t *>(qs + row * HD + 16 * k + 2 * t4 + 8 * x) : 0u;
                    }
        }
        // o[j][n]: dimensions (rows) of block j by heads 8 n + 2 t4, + 1.  In bf16 the rows g and g + 8 are dimensions
        // 16 j + g and 8 further; in f32 32 (j / 2) + 4 g + 2 (j % 2) and the next one.
        float o[8][NH][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int n = 0; n < NH; ++n) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;
        float m[NH][2], l[NH][2];                            // of heads 8 n + 2 t4, + 1; l over this lane's positions
#pragma unroll
        for (int n = 0; n < NH; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;

        for (int i = 0; i < run; ++i, ++e) {
            const int st = e % PD_NS;
            ok = __all_sync(FULL, mbar_wait(&full[st], uint32_t(e / PD_NS) & 1u, lane == 0 ? status : nullptr));
            if (!ok) break;
            if (CF32 && ((e ^ (warp >> 1)) & 1)) {           // an f32 tile is two warps' work, the next one the others'
                if (lane == 0) mbar_arrive(&empty[st]);
                continue;
            }
            const uint32_t ka = ring_a + st * PD_STAGE, va = ka + PD_SIDE;
            const int left = w.len - (w.tile + i) * TILE - key0;             // visible ones of this warp's 16
            float s[NH][4];                                  // positions g and g + 8 by heads 8 n + 2 t4, + 1
#pragma unroll
            for (int n = 0; n < NH; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            if constexpr (CF32) {
                // k index t4 is dimension 32 d + 8 t4 + 4 x + y, k index t4 + 4 is y + 1 (y = 0, 2): an order that query
                // and key share, so that both are read 16 bytes at a time without conflicts
                const uint32_t kr = ka + (key0 + g) * 128, qa = smem_addr(spare) + g * (HD * 4);
#pragma unroll 1
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t ch = uint32_t((2 * t4 + x) ^ g) << 4;
                        const float4 v0 = lds4(kr + d * (PD_SIDE / 4) + ch), v1 = lds4(kr + d * (PD_SIDE / 4) + 8 * 128 + ch);
                        uint32_t ah[2][4], al[2][4];
                        split_tf32(v0.x, ah[0][0], al[0][0]);
                        split_tf32(v1.x, ah[0][1], al[0][1]);
                        split_tf32(v0.y, ah[0][2], al[0][2]);
                        split_tf32(v1.y, ah[0][3], al[0][3]);
                        split_tf32(v0.z, ah[1][0], al[1][0]);
                        split_tf32(v1.z, ah[1][1], al[1][1]);
                        split_tf32(v0.w, ah[1][2], al[1][2]);
                        split_tf32(v1.w, ah[1][3], al[1][3]);
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
                            const float4 v = lds4(qa + n * 8 * (HD * 4) + 128 * d + ch);
                            uint32_t bh[4], bl[4];
                            split_tf32(v.x, bh[0], bl[0]);
                            split_tf32(v.y, bh[1], bl[1]);
                            split_tf32(v.z, bh[2], bl[2]);
                            split_tf32(v.w, bh[3], bl[3]);
                            float part[4] = {}, low[4] = {};
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                mma_tf32(low, al[y][0], al[y][1], al[y][2], al[y][3], bh[2 * y], bh[2 * y + 1]);
                                mma_tf32(part, ah[y][0], ah[y][1], ah[y][2], ah[y][3], bh[2 * y], bh[2 * y + 1]);
                                mma_tf32(low, ah[y][0], ah[y][1], ah[y][2], ah[y][3], bl[2 * y], bl[2 * y + 1]);
                            }
                            add_to(part, low);
                            add_to(s[n], part);
                        }
                    }
            } else {
                const int key = key0 + ((lane >> 3) & 1) * 8 + (lane & 7);
                auto keys = [&](int k, uint32_t (&a)[4]) {   // the 16 positions by dimensions 16 k ..
                    const int chunk = 2 * k + (lane >> 4);
                    ldsm4(ka + (chunk >> 3) * (PD_SIDE / 2) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4), a);
                };
                if constexpr (PARTS3) {
                    const uint32_t qa = smem_addr(spare) + (lane & 7) * (HD * 2);
#pragma unroll
                    for (int k = 0; k < 8; k += 2) {         // 32 dimensions
                        uint32_t a[2][4];
                        keys(k, a[0]);
                        keys(k + 1, a[1]);
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
                            float part[4] = {}, low[4] = {};
#pragma unroll
                            for (int x = 2; x >= 0; --x) {
                                uint32_t bq[4];              // chunks 2 k .. 2 k + 3 of heads 8 n ..
                                ldsm4(qa + (x * NH + n) * 8 * (HD * 2) + (((2 * k + (lane >> 3)) ^ (lane & 7)) << 4), bq);
                                mma_bf16(x ? low : part, a[0][0], a[0][1], a[0][2], a[0][3], bq[0], bq[1]);
                                mma_bf16(x ? low : part, a[1][0], a[1][1], a[1][2], a[1][3], bq[2], bq[3]);
                            }
                            add_to(part, low);
                            add_to(s[n], part);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint32_t a[4];
                        keys(k, a);
#pragma unroll
                        for (int n = 0; n < NH; ++n) mma_bf16(s[n], a[0], a[1], a[2], a[3], qf[k][n][0], qf[k][n][1]);
                    }
                }
            }
            // softmax over the 16 positions, which the lanes of one t4 share
            if (left < 16) {
#pragma unroll
                for (int n = 0; n < NH; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (g + 8 * (x >> 1) >= left) s[n][x] = -INFINITY;
            }
            float f[NH][2];
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NH; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float tm = fmaxf(s[n][h], s[n][2 + h]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) tm = fmaxf(tm, __shfl_xor_sync(FULL, tm, x));
                    f[n][h] = 1.0f;
                    if (tm > m[n][h]) {
                        f[n][h] = ex2_approx_ftz((m[n][h] - tm) * PD_LOG2);
                        m[n][h] = tm;
                        grow = true;
                    }
                    const float off = m[n][h] == -INFINITY ? 0.0f : -m[n][h] * PD_LOG2;
                    s[n][h] = ex2_approx_ftz(fmaf(s[n][h], PD_LOG2, off));
                    s[n][2 + h] = ex2_approx_ftz(fmaf(s[n][2 + h], PD_LOG2, off));
                    l[n][h] = fmaf(l[n][h], f[n][h], s[n][h] + s[n][2 + h]);
                }
            if (__any_sync(FULL, grow)) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int n = 0; n < NH; ++n)
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[j][n][x] *= f[n][x & 1];
            }
            // the weighted values
            if constexpr (CF32) {
                // In a block of eight positions k index t4 is position 2 t4, t4 + 4 the next one, and heads are columns:
                // the probabilities of lanes 8 t4 + g / 2 and 4 further, of head g % 2 there.
                uint32_t ph[2][NH][2], pl[2][NH][2];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int n = 0; n < NH; ++n)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int from = 8 * t4 + 4 * x + (g >> 1);
                            const float p0 = __shfl_sync(FULL, s[n][2 * kb], from), p1 = __shfl_sync(FULL, s[n][2 * kb + 1], from);
                            split_tf32(g & 1 ? p1 : p0, ph[kb][n][x], pl[kb][n][x]);
                        }
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    float part[2][NH][4] = {}, low[2][NH][4] = {};
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        const int k0 = key0 + 8 * kb + 2 * t4;
                        const uint32_t at = va + d * (PD_SIDE / 4) + k0 * 128;
                        const float4 v0 = lds4(at + ((g ^ (2 * t4)) << 4)), v1 = lds4(at + 128 + ((g ^ (2 * t4 + 1)) << 4));
                        const bool live0 = 8 * kb + 2 * t4 < left, live1 = 8 * kb + 2 * t4 + 1 < left;
                        const float x0[4] = {v0.x, v0.y, v0.z, v0.w}, x1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            uint32_t ah[4], al[4];
                            split_tf32(live0 ? x0[2 * y] : 0.0f, ah[0], al[0]);
                            split_tf32(live0 ? x0[2 * y + 1] : 0.0f, ah[1], al[1]);
                            split_tf32(live1 ? x1[2 * y] : 0.0f, ah[2], al[2]);
                            split_tf32(live1 ? x1[2 * y + 1] : 0.0f, ah[3], al[3]);
#pragma unroll
                            for (int n = 0; n < NH; ++n) {
                                mma_tf32(low[y][n], al[0], al[1], al[2], al[3], ph[kb][n][0], ph[kb][n][1]);
                                mma_tf32(part[y][n], ah[0], ah[1], ah[2], ah[3], ph[kb][n][0], ph[kb][n][1]);
                                mma_tf32(low[y][n], ah[0], ah[1], ah[2], ah[3], pl[kb][n][0], pl[kb][n][1]);
                            }
                        }
                    }
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
                            add_to(part[y][n], low[y][n]);
                            add_to(o[2 * d + y][n], part[y][n]);
                        }
                }
            } else {
                constexpr int PARTS = Elem<T>::BYTES == 4 ? 3 : 2;
                uint32_t p[PARTS][NH][2];                    // positions by heads: the scores' blocks, transposed
#pragma unroll
                for (int n = 0; n < NH; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        uint32_t part[PARTS];
                        split_bf16(s[n][2 * x], s[n][2 * x + 1], part);
#pragma unroll
                        for (int y = 0; y < PARTS; ++y) p[y][n][x] = transpose8x8(part[y]);
                    }
                // keep[x]: which of the positions 8 x + 2 t4, + 1 exist
                uint32_t keep[2];
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    keep[x] = (8 * x + 2 * t4 < left ? 0xffffu : 0u) | (8 * x + 2 * t4 + 1 < left ? 0xffff0000u : 0u);
                const int key = key0 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int chunk = 2 * j + ((lane >> 3) & 1);
                    uint32_t a[4];                           // dimensions 16 j + g, + 8 by positions 0-7, then by 8-15
                    ldsm4_t(va + (chunk >> 3) * (PD_SIDE / 2) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4), a);
#pragma unroll
                    for (int x = 0; x < 4; ++x) a[x] &= keep[x >> 1];
#pragma unroll
                    for (int n = 0; n < NH; ++n) {
                        float part[4] = {};
#pragma unroll
                        for (int y = PARTS - 1; y >= 0; --y) mma_bf16(part, a[0], a[1], a[2], a[3], p[y][n][0], p[y][n][1]);
                        add_to(o[j][n], part);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        if (!ok && lane == 0) dead = 1;
        // join the four warps into warp 0 through shared memory
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][h] += __shfl_xor_sync(FULL, l[n][h], x);
        constexpr int AT_ONCE = WIDE ? 1 : 3;                // warps whose results fit the spare memory
#pragma unroll
        for (int src = 1; src < PD_WARPS; src += AT_ONCE) {
            named_sync(1, PD_WARPS * 32);
            if (warp >= src && warp < src + AT_ONCE) {
                float *to = spare + (warp - src) * (8 * NH * 4 * 32) + lane;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int n = 0; n < NH; ++n)
#pragma unroll
                        for (int x = 0; x < 4; ++x) to[((j * NH + n) * 4 + x) * 32] = o[j][n][x];
                if (g == 0)
#pragma unroll
                    for (int n = 0; n < NH; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            join_m[warp - src][8 * n + 2 * t4 + h] = m[n][h], join_l[warp - src][8 * n + 2 * t4 + h] = l[n][h];
            }
            named_sync(1, PD_WARPS * 32);
            if (warp == 0) {
                float f0[NH][2], f1[AT_ONCE][NH][2];
#pragma unroll
                for (int n = 0; n < NH; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int head = 8 * n + 2 * t4 + h;
                        float nm = m[n][h];
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i) nm = fmaxf(nm, join_m[i][head]);
                        f0[n][h] = m[n][h] == nm ? 1.0f : ex2_approx_ftz((m[n][h] - nm) * PD_LOG2);
                        l[n][h] *= f0[n][h];
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i) {
                            const float om = join_m[i][head];
                            f1[i][n][h] = om == nm ? 1.0f : ex2_approx_ftz((om - nm) * PD_LOG2);
                            l[n][h] = fmaf(join_l[i][head], f1[i][n][h], l[n][h]);
                        }
                        m[n][h] = nm;
                    }
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int n = 0; n < NH; ++n)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            o[j][n][x] *= f0[n][x & 1];
#pragma unroll
                            for (int i = 0; i < AT_ONCE; ++i)
                                o[j][n][x] = fmaf(spare[(((i * 8 + j) * NH + n) * 4 + x) * 32 + lane], f1[i][n][x & 1], o[j][n][x]);
                        }
            }
        }
        ok = dead == 0;                                      // the same for every warp: the next barrier follows the read
        if (warp == 0 && ok) {
            const bool whole = run == w.tiles;
            const int at0 = CF32 ? 4 * g : g, step = CF32 ? 1 : 8;           // this lane's first element, and to its pair
            auto block = [](int j) { return CF32 ? 32 * (j >> 1) + 2 * (j & 1) : 16 * j; };
#pragma unroll
            for (int n = 0; n < NH; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = 8 * n + 2 * t4 + h;
                    if (row >= group) continue;
                    if (whole) {
                        const float r = 1.0f / l[n][h];
                        typename Elem<T>::type *dst = out + (int64_t(w.s) * n_heads + w.head * group + row) * HD + at0;
#pragma unroll
                        for (int j = 0; j < 8; ++j) put2(dst + block(j), step, o[j][n][h] * r, o[j][n][2 + h] * r);
                    } else {
                        float *pd = part + ((2 * int64_t(blockIdx.x) + (u != u0)) * group + row) * PD_PART;
#pragma unroll
                        for (int j = 0; j < 8; ++j) put2(pd + at0 + block(j), step, o[j][n][h], o[j][n][2 + h]);
                        if (g == 0) pd[HD] = m[n][h], pd[HD + 1] = l[n][h];
                    }
                }
        }
        u += run;
        if (u < u1) walk_on<TC>(b, c, w, run);
        named_sync(1, PD_WARPS * 32);
    }
}

// Joins what the runs left of one query head, one CTA per run and head of the group; the CTA of the second run of a
// (sequence, kv head) does it: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  The
// parts' maxima and sums are read side by side, one thread each; then two groups of 128 threads (thread = element) add
// half of the weighted parts each, eight loads under way at a time.  The order of every sum is fixed.
constexpr int PJ_GROUPS = 2, PJ_THREADS = PJ_GROUPS * HD, PJ_RUNS = 1024;
template <typename T, typename TC>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const PagedKV c, const PagedSeqs b, int n_heads, int group,
                                                                int runs, typename Elem<T>::type *out, const float *part) {
    __shared__ float weight[PJ_RUNS], red[2][PJ_THREADS / 32], sum[PJ_GROUPS][HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = threadIdx.x % HD, half_id = threadIdx.x / HD;
    // Before the wait: the lengths are older than the first kernel, which has begun (this one starts when all its CTAs
    // have passed their own wait).
    PagedCut cut(0, 1);
    int64_t u0, u1;
    const int second = int(blockIdx.x) + 1;
    const PagedWalk w = walk_run<TC>(b, c, second, runs, cut, u0, u1, nullptr);
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

static int paged_runs(int sms) { return 2 * sms < PJ_RUNS ? 2 * sms : PJ_RUNS; }

size_t attention_paged_workspace(int n_heads, int n_kv, int sms) {
    return size_t(paged_runs(sms)) * 2 * (n_heads / n_kv) * PD_PART * sizeof(float);
}

template <typename T, typename TC>
static cudaError_t launch_split(const PagedKV &c, const PagedSeqs &b, const void *q, int64_t q_stride, int n_heads,
                                void *work, void *out, uint32_t *status, cudaStream_t stream, int sms, int slot) {
    typedef typename Elem<T>::type E;
    CUtensorMap mk, mv;
    const q3cu_dtype dt = Elem<TC>::BYTES == 4 ? Q3CU_F32 : Q3CU_BF16;
    if (!encode_pages_map(&mk, c.k, c, dt, pd_tile<TC>()) || !encode_pages_map(&mv, c.v, c, dt, pd_tile<TC>())) return cudaErrorInvalidValue;
    const int group = n_heads / c.n_kv, runs = paged_runs(sms);
    auto *kernel = group > 8 ? paged_split_kernel<T, TC, true> : paged_split_kernel<T, TC, false>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(kernel), PD_SMEM, slot + (group > 8));
    if (e != cudaSuccess) return e;
    e = launch_dependent(kernel, dim3(runs), dim3(PD_THREADS), PD_SMEM, stream, mk, mv, c, b, static_cast<const E *>(q),
                         q_stride, n_heads, group, static_cast<E *>(out), static_cast<float *>(work), status);
    if (e != cudaSuccess) return e;
    return launch_dependent(paged_join_kernel<T, TC>, dim3(runs - 1, group), dim3(PJ_THREADS), 0, stream, c, b,
                            n_heads, group, runs, static_cast<E *>(out), static_cast<const float *>(work));
}

cudaError_t launch_attention_paged(const PagedKV &c, q3cu_dtype cache_dt, const PagedSeqs &b, const void *q,
                                   q3cu_dtype dt, int64_t q_stride, int n_heads, void *work, void *out,
                                   uint32_t *status, cudaStream_t stream, int sms) {
    if (dt == Q3CU_F32)
        return cache_dt == Q3CU_F32
                   ? launch_split<float, float>(c, b, q, q_stride, n_heads, work, out, status, stream, sms, 33)
                   : launch_split<float, bf16raw>(c, b, q, q_stride, n_heads, work, out, status, stream, sms, 35);
    return cache_dt == Q3CU_F32
               ? launch_split<bf16raw, float>(c, b, q, q_stride, n_heads, work, out, status, stream, sms, 37)
               : launch_split<bf16raw, bf16raw>(c, b, q, q_stride, n_heads, work, out, status, stream, sms, 39);
}

}  // namespace q3
