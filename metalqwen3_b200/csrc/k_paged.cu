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
// and V of 64 positions in bf16 or 32 in f32; each computing warp takes a
// quarter of them, with its own running maximum, sum and result, and the four
// are joined when the run leaves the (sequence, head).
//
// The products run on mma.sync with the group's query heads as the 16 rows of
// the tile: at one to sixteen query rows the tensor cores are mostly idle by
// either path, and the operands come straight from registers.  They lose nothing
// that an f32 result would show: an f32 query against a bf16 cache is three bf16
// parts (the keys are exact), and so is a probability, two where the result is
// bf16; an f32 cache is multiplied as tf32 parts, high x high + high x low +
// low x high, whose remainder is 2^-22 of the product.  Sums are binary32.
//
// Positions at and beyond the length score -inf, and their values are masked to
// zero in registers: unused page space may hold anything.
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
// `n` tiles further, which lie in the same (sequence, head) or begin the next one that has any.
template <typename TC>
__device__ __forceinline__ void walk_on(const PagedSeqs &b, const PagedKV &c, PagedWalk &w, int n) {
    w.tile += n;
    if (w.tile < w.tiles) return;
    w.tile = 0;
    if (++w.head < c.n_kv) return;
    w.head = 0;
    do {
        if (++w.s >= b.n_seqs) return;
        w.len = paged_len(b, c, w.s, nullptr);
    } while (w.len == 0);
    w.tiles = tiles_of<TC>(w.len);
}

// One pair of result elements (row, dims at, at + step) as the output's type.
__device__ __forceinline__ void put2(float *p, int step, float x, float y) { p[0] = x, p[step] = y; }
__device__ __forceinline__ void put2(uint16_t *p, int step, float x, float y) {
    if (step == 1) *reinterpret_cast<uint32_t *>(p) = pack_bf16(x, y);
    else p[0] = uint16_t(f32_to_bf16(x)), p[step] = uint16_t(f32_to_bf16(y));
}

// WIDE: more than 8 query heads to a kv head (rows 8-15 of the products are used).
template <typename T, typename TC, bool WIDE>
__global__ void __launch_bounds__(PD_THREADS, 2)
paged_split_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const PagedKV c,
                   const PagedSeqs b, const typename Elem<T>::type *q, int64_t q_stride, int n_heads, int group,
                   typename Elem<T>::type *out, float *part, uint32_t *status) {
    constexpr bool CF32 = Elem<TC>::BYTES == 4;
    constexpr int TILE = pd_tile<TC>(), KW = TILE / PD_WARPS, NH = WIDE ? 2 : 1;
    extern __shared__ uint8_t pd_dyn[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pd_dyn) + 1023) & ~uintptr_t(1023));
    float *spare = reinterpret_cast<float *>(ring + PD_NS * PD_STAGE);
    __shared__ __align__(8) uint64_t full[PD_NS], empty[PD_NS];
    __shared__ float join_m[3][2][8], join_l[3][2][8];
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
    const int g = lane >> 2, t4 = lane & 3;                  // row g (and g + 8) of the products, column pair t4
    const uint32_t ring_a = smem_addr(ring);
    int e = 0;
    bool ok = true;
    for (int64_t u = u0; u < u1 && ok;) {
        const int run = int(min(int64_t(w.tiles - w.tile), u1 - u));       // tiles of this (sequence, head) here
        const typename Elem<T>::type *qs = q + w.s * q_stride + int64_t(w.head) * group * HD;
        constexpr bool PARTS3 = !CF32 && Elem<T>::BYTES == 4;                // f32 queries, bf16 cache
        uint32_t qf[CF32 || PARTS3 ? 1 : 8][2 * NH];         // bf16 queries, bf16 cache: operands in registers
        if constexpr (CF32) {                                // the group's rows in shared memory, zeros below
            for (int i = threadIdx.x; i < 8 * NH * (HD / 4); i += PD_WARPS * 32)
                *reinterpret_cast<float4 *>(spare + 4 * i) =
                    i / (HD / 4) < group ? load_quad(qs + 4 * i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            named_sync(1, PD_WARPS * 32);
        } else if constexpr (PARTS3) {
            // three bf16 parts of the group's rows in shared memory, zeros below; 16-byte chunk x of row r at x ^ (r % 8)
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
                for (int x = 0; x < 2 * NH; ++x) {           // x: columns + 8 (bit 0), row + 8 (bit 1)
                    const int row = g + 8 * (x >> 1), at = row * HD + 16 * k + 2 * t4 + 8 * (x & 1);
                    qf[k][x] = row < group ? *reinterpret_cast<const uint32_t *>(qs + at) : 0u;
                }
        }
        float o[16][4];
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m[NH], l[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) m[h] = -INFINITY, l[h] = 0.0f;

        for (int i = 0; i < run; ++i, ++e) {
            const int st = e % PD_NS;
            ok = __all_sync(FULL, mbar_wait(&full[st], uint32_t(e / PD_NS) & 1u, lane == 0 ? status : nullptr));
            if (!ok) break;
            const uint32_t ka = ring_a + st * PD_STAGE, va = ka + PD_SIDE;
            const int left = w.len - (w.tile + i) * TILE - warp * KW;      // visible positions of this warp's KW
            // scores: rows g, g + 8; columns (positions) 8 n + 2 t4, + 1
            float s[KW / 8][4];
#pragma unroll
            for (int n = 0; n < KW / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            if constexpr (CF32) {
                // k index t4 is dimension 32 d + 8 t4 + x, k index t4 + 4 is + 1 of it (x = 0, 2, then 4, 6): a
                // permutation that query and key share, so both are read 16 bytes at a time without conflicts
                const uint32_t row = ka + (warp * KW + g) * 128, qa = smem_addr(spare) + g * (HD * 4);
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float4 kv = lds4(row + d * (PD_SIDE / 4) + (((2 * t4 + x) ^ g) << 4));
                        const float kf[4] = {kv.x, kv.y, kv.z, kv.w};
                        float qf[NH][4];
#pragma unroll
                        for (int h = 0; h < NH; ++h) {
                            const float4 v = lds4(qa + h * 8 * (HD * 4) + (32 * d + 8 * t4 + 4 * x) * 4);
                            qf[h][0] = v.x, qf[h][1] = v.y, qf[h][2] = v.z, qf[h][3] = v.w;
                        }
                        float part[4] = {}, low[4] = {};
#pragma unroll
                        for (int y = 0; y < 4; y += 2) {
                            uint32_t bh[2], bl[2], ah[4] = {0, 0, 0, 0}, al[4] = {0, 0, 0, 0};
                            split_tf32(kf[y], bh[0], bl[0]);
                            split_tf32(kf[y + 1], bh[1], bl[1]);
#pragma unroll
                            for (int h = 0; h < NH; ++h) {
                                split_tf32(qf[h][y], ah[h], al[h]);
                                split_tf32(qf[h][y + 1], ah[2 + h], al[2 + h]);
                            }
                            mma_tf32(low, al[0], al[1], al[2], al[3], bh[0], bh[1]);
                            mma_tf32(low, ah[0], ah[1], ah[2], ah[3], bl[0], bl[1]);
                            mma_tf32(part, ah[0], ah[1], ah[2], ah[3], bh[0], bh[1]);
                        }
                        add_to(part, low);
                        add_to(s[0], part);
                    }
            } else {
                const int key = warp * KW + (lane >> 4) * 8 + (lane & 7);
                auto keys = [&](int k, uint32_t (&r)[4]) {   // dimensions 16 k ..; positions 0-7 in r[0], r[1], 8-15 in r[2], r[3]
                    const int chunk = 2 * k + ((lane >> 3) & 1);
                    ldsm4(ka + (chunk >> 3) * (PD_SIDE / 2) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4), r);
                };
                if constexpr (PARTS3) {
                    // a lane's address in the parts: WIDE rows 0-15 of chunks 2 k, 2 k + 1, otherwise rows 0-7 of four chunks
                    const int row = WIDE ? lane & 15 : lane & 7, first = WIDE ? lane >> 4 : lane >> 3;
                    const uint32_t qa = smem_addr(spare) + row * (HD * 2);
#pragma unroll
                    for (int k = 0; k < 8; k += 2) {
                        uint32_t r[2][4], a[3][2][4];
                        keys(k, r[0]);
                        keys(k + 1, r[1]);
#pragma unroll
                        for (int x = 0; x < 3; ++x) {
                            const uint32_t pa = qa + x * 8 * NH * (HD * 2);
                            if constexpr (WIDE) {            // rows 0-7, 8-15 of chunk 2 k, then of 2 k + 1
                                ldsm4(pa + (((2 * k + first) ^ (row & 7)) << 4), a[x][0]);
                                ldsm4(pa + (((2 * k + 2 + first) ^ (row & 7)) << 4), a[x][1]);
                            } else {
                                uint32_t v[4];
                                ldsm4(pa + (((2 * k + first) ^ row) << 4), v);
#pragma unroll
                                for (int y = 0; y < 2; ++y)
                                    a[x][y][0] = v[2 * y], a[x][y][1] = 0u, a[x][y][2] = v[2 * y + 1], a[x][y][3] = 0u;
                            }
                        }
                        float part[2][4] = {}, low[2][4] = {};
#pragma unroll
                        for (int y = 0; y < 2; ++y)
#pragma unroll
                            for (int n = 0; n < 2; ++n) {
                                mma_bf16(low[n], a[2][y][0], a[2][y][1], a[2][y][2], a[2][y][3], r[y][2 * n], r[y][2 * n + 1]);
                                mma_bf16(low[n], a[1][y][0], a[1][y][1], a[1][y][2], a[1][y][3], r[y][2 * n], r[y][2 * n + 1]);
                                mma_bf16(part[n], a[0][y][0], a[0][y][1], a[0][y][2], a[0][y][3], r[y][2 * n], r[y][2 * n + 1]);
                            }
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            add_to(part[n], low[n]);
                            add_to(s[n], part[n]);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint32_t r[4];
                        keys(k, r);
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            mma_bf16(s[n], qf[k][0], WIDE ? qf[k][2 * NH - 2] : 0u, qf[k][1], WIDE ? qf[k][2 * NH - 1] : 0u,
                                     r[2 * n], r[2 * n + 1]);
                    }
                }
            }
            // softmax over this warp's positions
            if (left < KW) {
#pragma unroll
                for (int n = 0; n < KW / 8; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (8 * n + 2 * t4 + (x & 1) >= left) s[n][x] = -INFINITY;
            }
            float f[NH];
            bool grow = false;
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                float tm = -INFINITY;
#pragma unroll
                for (int n = 0; n < KW / 8; ++n) tm = fmaxf(tm, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
                tm = fmaxf(tm, __shfl_xor_sync(FULL, tm, 1));
                tm = fmaxf(tm, __shfl_xor_sync(FULL, tm, 2));
                f[h] = 1.0f;
                if (tm > m[h]) {
                    f[h] = ex2_approx_ftz((m[h] - tm) * PD_LOG2);
                    m[h] = tm;
                    grow = true;
                }
                const float off = m[h] == -INFINITY ? 0.0f : -m[h] * PD_LOG2;
                float add = 0.0f;
#pragma unroll
                for (int n = 0; n < KW / 8; ++n)
#pragma unroll
                    for (int x = 2 * h; x < 2 * h + 2; ++x) {
                        s[n][x] = ex2_approx_ftz(fmaf(s[n][x], PD_LOG2, off));
                        add += s[n][x];
                    }
                l[h] = fmaf(l[h], f[h], add);
            }
            if (__any_sync(FULL, grow)) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int x = 0; x < 2 * NH; ++x) o[j][x] *= f[x >> 1];
            }
            // the weighted values
            if constexpr (CF32) {
                // k index t4 is position 2 t4, t4 + 4 is 2 t4 + 1: the columns this thread's scores have;
                // column n of product (d, x) is dimension 32 d + 4 n + x
                uint32_t ph[4] = {0, 0, 0, 0}, pl[4] = {0, 0, 0, 0};
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    split_tf32(s[0][2 * h], ph[h], pl[h]);
                    split_tf32(s[0][2 * h + 1], ph[2 + h], pl[2 + h]);
                }
                const int k0 = warp * KW + 2 * t4;
                const bool live0 = 2 * t4 < left, live1 = 2 * t4 + 1 < left;
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t blk = va + d * (PD_SIDE / 4);
                    const float4 v0 = lds4(blk + k0 * 128 + ((g ^ (k0 & 7)) << 4));
                    const float4 v1 = lds4(blk + (k0 + 1) * 128 + ((g ^ ((k0 + 1) & 7)) << 4));
                    const float a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t bh[2], bl[2];
                        split_tf32(live0 ? a0[x] : 0.0f, bh[0], bl[0]);
                        split_tf32(live1 ? a1[x] : 0.0f, bh[1], bl[1]);
                        float part[4] = {};
                        mma_tf32(part, pl[0], pl[1], pl[2], pl[3], bh[0], bh[1]);
                        mma_tf32(part, ph[0], ph[1], ph[2], ph[3], bl[0], bl[1]);
                        mma_tf32(part, ph[0], ph[1], ph[2], ph[3], bh[0], bh[1]);
                        add_to(o[4 * d + x], part);
                    }
                }
            } else {
                constexpr int PARTS = Elem<T>::BYTES == 4 ? 3 : 2;
                uint32_t p[PARTS][4] = {};
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int h = 0; h < NH; ++h) {
                        uint32_t part[PARTS];
                        split_bf16(s[n][2 * h], s[n][2 * h + 1], part);
#pragma unroll
                        for (int x = 0; x < PARTS; ++x) p[x][2 * n + h] = part[x];
                    }
                // keep[n]: which of the positions 8 n + 2 t4, + 1 exist
                uint32_t keep[2];
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    keep[n] = (8 * n + 2 * t4 < left ? 0xffffu : 0u) | (8 * n + 2 * t4 + 1 < left ? 0xffff0000u : 0u);
                const int key = warp * KW + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const int chunk = 2 * d + (lane >> 4);
                    uint32_t r[4];
                    ldsm4_t(va + (chunk >> 3) * (PD_SIDE / 2) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4), r);
#pragma unroll
                    for (int x = 0; x < 4; ++x) r[x] &= keep[x & 1];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        float part[4] = {};
#pragma unroll
                        for (int x = PARTS - 1; x >= 0; --x)
                            mma_bf16(part, p[x][0], p[x][1], p[x][2], p[x][3], r[2 * n], r[2 * n + 1]);
                        add_to(o[2 * d + n], part);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        if (!ok && lane == 0) dead = 1;
        // join the four warps into warp 0 through shared memory
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            l[h] += __shfl_xor_sync(FULL, l[h], 1);
            l[h] += __shfl_xor_sync(FULL, l[h], 2);
        }
        constexpr int AT_ONCE = WIDE ? 1 : 3;                // warps whose results fit the spare memory
#pragma unroll
        for (int src = 1; src < PD_WARPS; src += AT_ONCE) {
            named_sync(1, PD_WARPS * 32);
            if (warp >= src && warp < src + AT_ONCE) {
                float *to = spare + (warp - src) * (16 * 2 * NH * 32);
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int x = 0; x < 2 * NH; ++x) to[(j * 2 * NH + x) * 32 + lane] = o[j][x];
#pragma unroll
                for (int h = 0; h < NH; ++h)
                    if (t4 == 0) join_m[warp - src][h][g] = m[h], join_l[warp - src][h][g] = l[h];
            }
            named_sync(1, PD_WARPS * 32);
            if (warp == 0) {
                float f0[NH], f1[AT_ONCE][NH];
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    float nm = m[h];
#pragma unroll
                    for (int i = 0; i < AT_ONCE; ++i) nm = fmaxf(nm, join_m[i][h][g]);
                    f0[h] = m[h] == nm ? 1.0f : ex2_approx_ftz((m[h] - nm) * PD_LOG2);
                    l[h] *= f0[h];
#pragma unroll
                    for (int i = 0; i < AT_ONCE; ++i) {
                        const float om = join_m[i][h][g];
                        f1[i][h] = om == nm ? 1.0f : ex2_approx_ftz((om - nm) * PD_LOG2);
                        l[h] = fmaf(join_l[i][h][g], f1[i][h], l[h]);
                    }
                    m[h] = nm;
                }
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int x = 0; x < 2 * NH; ++x) {
                        o[j][x] *= f0[x >> 1];
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i)
                            o[j][x] = fmaf(spare[((i * 16 + j) * 2 * NH + x) * 32 + lane], f1[i][x >> 1], o[j][x]);
                    }
            }
        }
        ok = dead == 0;                                      // the same for every warp: the next barrier follows the read
        if (warp == 0 && ok) {
            const bool whole = run == w.tiles;
            const int slot = 2 * int(blockIdx.x) + (u != u0);
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const int row = g + 8 * h;
                if (row >= group) continue;
                const float r = whole ? 1.0f / l[h] : 1.0f;
                typename Elem<T>::type *dst = out + (int64_t(w.s) * n_heads + w.head * group + row) * HD;
                float *pd = part + (int64_t(slot) * group + row) * PD_PART;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int at = CF32 ? 32 * (j >> 2) + 8 * t4 + (j & 3) : 8 * j + 2 * t4;
                    const float x = o[j][2 * h] * r, y = o[j][2 * h + 1] * r;
                    if (whole) put2(dst + at, CF32 ? 4 : 1, x, y);
                    else put2(pd + at, CF32 ? 4 : 1, x, y);
                }
                if (!whole && t4 == 0) pd[HD] = m[h], pd[HD + 1] = l[h];
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
    if (u0 == u1 || w.tile == 0) return;                     // no tiles, or it begins with a new (sequence, head)
    const int64_t a = u0 - w.tile;                           // the (sequence, head)'s first tile
    const int first = second - 1, last = cut.run_of(a + w.tiles - 1), n = last - first + 1;
    if (a < cut.begin(first)) return;                        // not the second of its runs
    griddep_wait();
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
