// k_paged_q8.cu -- attention of one new token per sequence over a Q8_0 paged cache.
//
// The operation, the split into equal runs of tiles and the join are those of
// k_paged.cu; a key is k_i = c_i s_(i / 64) with int8 codes c and one f32 scale to
// 64 elements, a value likewise.  Bound by memory: 136 bytes a position, kv head
// and side, where bf16 takes 256.  64 sequences of up to 16,384 positions (32/8 heads,
// bf16 queries): 176 to 194 us, up to 6.2 TB/s; one of 512 (16/8, f32 queries): 9 us,
// all latency.  f32 queries for 64 such sequences: 220 us where bf16 ones take 177.
//
// A CTA is one fetching warp and four computing warps around a ring of three 34 KB
// stages, filled page by page by TMA: 128 positions' codes of K and of V (128-byte
// swizzle) and their scales.  Each computing warp takes 32 of the positions.
//
// The products run on mma.sync with 16 positions as the rows (or 16 dimensions, for
// the values) and eight query heads as the columns, in f16, whose 11 bits hold a
// code exactly: a byte becomes 1024 + (code + 128) by a byte permutation and the
// code by one packed subtraction, 1.25 instructions an element, where going through
// bf16 (8 bits) or f32 takes twice that.  The scales never touch the elements:
//     score = s_0 (q_lo . c_lo) + s_1 (q_hi . c_hi)         two chains of products (s with q's inverse lift, see below)
//     o_lo += sum_t (p_t s_0t) c_t,lo                       the weights take them
// The other operands go to f16 as well, each times a power of two that brings the
// largest of them to [2^14, 2^15) (of a query row, and of a warp's 32 value scales),
// so that the smaller ones keep their bits down to 2^-28 of it and reach 2^-39:
// bf16 queries are exact, f32 queries two parts (2^-23); a weight is one part with
// a bf16 result (2^-11 each, an eighth of the result's own rounding) and two with an
// f32 one.  Sums are binary32.
//
// Which position is which row of a product is free as long as the scores, the mask
// and the values agree: row g of eight is position (g % 2) * 4 + g / 2, with which
// the lanes of a quarter warp read 16-byte pieces of the swizzled codes without
// conflicts.  Dimensions are permuted likewise, query and key alike.
//
// Positions at and beyond the length, and before a tail, score -inf and weigh
// exactly 0: unused page space may hold anything, scales that are NaN included.
#include "q3cu_f16.cuh"
#include "q3cu_mma.cuh"
#include "q3cu_paged.cuh"
#include "q3cu_split.cuh"
#include "q3cu_tma.h"

namespace q3 {

constexpr int PQ_WARPS = 4, PQ_THREADS = (PQ_WARPS + 1) * 32;
constexpr int PQ_NS = 3, PQ_TILE = 128;                      // stages, positions of one
constexpr uint32_t PQ_CODES = PQ_TILE * HD, PQ_SCALES = PQ_TILE * 8;        // bytes of one side
constexpr uint32_t PQ_STAGE = 2 * (PQ_CODES + PQ_SCALES);    // codes of K, of V, scales of K, of V
constexpr int PQ_SPARE = 8192;                               // f16 queries, then the join of the warps
constexpr size_t PQ_SMEM = size_t(PQ_NS) * PQ_STAGE + PQ_SPARE + 1024;
static_assert(PQ_TILE == PD_TAIL_Q8, "the tails' tiles");

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ int pq_row(int g) { return ((g & 1) << 2) | ((g & 7) >> 1); }   // the position of row g of eight

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 lds2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

template <typename T, bool WIDE, typename Seqs>
__global__ void __launch_bounds__(PQ_THREADS, 2)
paged_q8_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                const __grid_constant__ CUtensorMap tmks, const __grid_constant__ CUtensorMap tmvs, const PagedKV c,
                const Seqs b, const typename Elem<T>::type *q, int64_t q_stride, int n_heads, int group,
                typename Elem<T>::type *out, float *part, float *tails, uint32_t *status) {
    constexpr int NH = WIDE ? 2 : 1;                         // blocks of eight heads
    constexpr int PARTS = Elem<T>::BYTES == 4 ? 2 : 1;       // f16 parts of a query element, and of a weight
    constexpr bool QREG = PARTS * NH <= 2;                   // queries in registers
    extern __shared__ uint8_t pq_dyn[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pq_dyn) + 1023) & ~uintptr_t(1023));
    float *spare = reinterpret_cast<float *>(ring + PQ_NS * PQ_STAGE);
    __shared__ __align__(8) uint64_t full[PQ_NS], empty[PQ_NS];
    __shared__ float join_m[2][8 * NH], join_l[2][8 * NH], row_back[8 * NH];
    __shared__ volatile int dead;                            // a wait gave up
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PQ_NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], PQ_WARPS);
        }
        mbar_init_fence();
        dead = 0;
    }
    __syncthreads();
    // Tails do not wait for the launch before, whose results they do not need: when it let this one begin, the plan and all that
    // is older were complete.  The first CTA waits for it at its end, since the launch behind waits for this grid alone.
    if constexpr (Seqs::TAILS) __threadfence();              // nothing here is read from an older copy of a line
    else griddep_wait();
    griddep_launch_dependents();

    PagedCut cut(0, 1);
    int64_t u0, u1;
    PagedWalk w = walk_run<PQ_TILE>(b, c, int(blockIdx.x), int(gridDim.x), cut, u0, u1,
                                    blockIdx.x == 0 && warp == 0 ? status : nullptr);
    for (int s = int(blockIdx.x); s < b.n_seqs; s += int(gridDim.x))       // sequences without positions: zeros
        if (b.span(c, s, nullptr).len == 0)
            for (int i = threadIdx.x; i < n_heads * (HD / 4); i += PQ_THREADS)
                store_quad(out + int64_t(s) * n_heads * HD + 4 * i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    if (u0 == u1) {
        if (Seqs::TAILS && blockIdx.x == 0) griddep_wait();
        return;
    }

    if (warp == PQ_WARPS) {
        // ---- fetch: lane = box (codes of K or V, or their scales; rows of one page) --------
        static_assert(TAIL_ALIGN == 32, "5 below");
        const int bs = min(c.page_shift, Seqs::TAILS ? 5 : 7), br = 1 << bs, ns = 7 - bs;       // rows of a box; log2 of boxes of a tile
        const int box = lane & ((1 << ns) - 1), kind = lane >> ns;           // kind: K, V, scales of K, of V
        auto page_of = [&]() -> int {                        // n_pages reads as zeros
            const int t = w.template pos<PQ_TILE, Seqs>(w.tile) + box * br;
            if (kind > 3 || t >= w.len || (Seqs::TAILS && t + br <= w.from)) return c.n_pages;
            const int p = paged_page(b, c, w.s, t, status);
            return p < 0 ? c.n_pages : p;
        };
        uint8_t *dst = ring + (kind < 2 ? kind * PQ_CODES + box * br * HD : 2 * PQ_CODES + (kind & 1) * PQ_SCALES + box * br * 8);
        int page = page_of(), e = 0;
        bool ok = true;
        const uint64_t once = evict_first_policy();
        for (int64_t u = Seqs::TAILS ? u0 + w.lead : u0, next; u < u1; u = next, ++e) {
            next = u + 1;
            const int head = w.head, now = page;
            const int slot = (w.template pos<PQ_TILE, Seqs>(w.tile) + box * br) & ((1 << c.page_shift) - 1);
            if (next < u1) {
                walk_on<PQ_TILE>(b, c, w, 1);
                if (Seqs::TAILS) next += w.lead;
                page = page_of();                            // under way while this tile waits for its stage
            }
            const int st = e % PQ_NS;
            if (e >= PQ_NS) ok = mbar_wait(&empty[st], uint32_t(e / PQ_NS - 1) & 1u, lane == 0 ? status : nullptr);
            if (!__all_sync(FULL, ok)) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[st], PQ_STAGE);
            __syncwarp();
            // read once (and tails while the shared positions' results wait in L2)
            if (kind < 2) tma_load_4d_once(dst + st * PQ_STAGE, kind ? &tmv : &tmk, 0, slot, head, now, &full[st], once);
            else if (kind < 4) tma_load_3d_once(dst + st * PQ_STAGE, kind & 1 ? &tmvs : &tmks, 2 * slot, head, now, &full[st], once);
        }
        // no copy outlives the CTA (bounded)
        for (int d = e > PQ_NS ? e - PQ_NS : 0; d < e; ++d) mbar_wait(&full[d % PQ_NS], uint32_t(d / PQ_NS) & 1u, nullptr);
        if (Seqs::TAILS && blockIdx.x == 0) griddep_wait();
        return;
    }

    // ---- the computing warps ---------------------------------------------------------
    const int g = lane >> 2, t4 = lane & 3;                  // products: row g (and g + 8), columns 2 t4 and + 1
    const uint32_t ring_a = smem_addr(ring), spare_a = smem_addr(spare);
    const int key0 = 32 * warp, pg = pq_row(g);              // this warp's 32 positions of a tile; row g's among eight
    int e = 0;
    bool ok = true;
    for (int64_t u = u0; u < u1 && ok;) {
        const int lead = Seqs::TAILS ? w.lead : 0, units = int(min(int64_t(lead) + w.tiles - w.tile, u1 - u));
        const int run = units - lead;                        // tiles of this (sequence, head) here
        if (Seqs::TAILS && run <= 0) break;                  // it begins where the run ends
        const typename Elem<T>::type *qs = q + w.s * q_stride + int64_t(w.head) * group * HD;
        // the group's rows as f16 parts in shared memory, lifted, zeros below; 16-byte piece x of row r at x ^ (r % 2)
        for (int r = warp; r < 8 * NH; r += PQ_WARPS) {
            const float4 v = r < group ? load_quad(qs + r * HD + 4 * lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const uint32_t top = __reduce_max_sync(FULL, __float_as_uint(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)))));
            const float up = lift(top);
            uint32_t lo[PARTS], hi[PARTS];
            split_f16(v.x * up, v.y * up, lo);
            split_f16(v.z * up, v.w * up, hi);
#pragma unroll
            for (int x = 0; x < PARTS; ++x)
                *reinterpret_cast<uint2 *>(reinterpret_cast<uint8_t *>(spare) + (x * 8 * NH + r) * (HD * 2) +
                                           (((lane >> 1) ^ (r & 1)) << 4) + (lane & 1) * 8) = make_uint2(lo[x], hi[x]);
            if (lane == 0) row_back[r] = lift_back(top);
        }
        named_sync(1, PQ_WARPS * 32);
        // queries of heads 8 n + g, dimensions 64 h + 16 t4 ..: in product (h, y), k index 2 t4 (+ 1) is 4 y (+ 1) of
        // these and 8 further 4 y + 2 (+ 1)
        auto query = [&](int x, int n, int h, uint32_t (&r)[8]) {
            const uint32_t at = spare_a + (x * 8 * NH + 8 * n + g) * (HD * 2);
            const uint4 a = lds16(at + (((8 * h + 2 * t4) ^ (g & 1)) << 4)), d = lds16(at + (((8 * h + 2 * t4 + 1) ^ (g & 1)) << 4));
            r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w, r[4] = d.x, r[5] = d.y, r[6] = d.z, r[7] = d.w;
        };
        uint32_t qf[QREG ? PARTS : 1][QREG ? NH : 1][2][8];
        if constexpr (QREG) {
#pragma unroll
            for (int x = 0; x < PARTS; ++x)
#pragma unroll
                for (int n = 0; n < NH; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) query(x, n, h, qf[x][n][h]);
        }
        float back[NH][2];                                   // products times this are those with q, of heads 8 n + 2 t4, + 1
#pragma unroll
        for (int n = 0; n < NH; ++n) back[n][0] = row_back[8 * n + 2 * t4], back[n][1] = row_back[8 * n + 2 * t4 + 1];
        // o[j][n]: dimensions 16 j + 2 g and (+ 2) the next one by heads 8 n + 2 t4, + 1
        float o[8][NH][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int n = 0; n < NH; ++n) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;
        float m[NH][2], l[NH][2];                            // of heads 8 n + 2 t4, + 1; l over this lane's positions
#pragma unroll
        for (int n = 0; n < NH; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;

        for (int i = 0; i < run; ++i, ++e) {
            const int st = e % PQ_NS;
            ok = __all_sync(FULL, mbar_wait(&full[st], uint32_t(e / PQ_NS) & 1u, lane == 0 ? status : nullptr));
            if (!ok) break;
            const uint32_t ka = ring_a + st * PQ_STAGE, va = ka + PQ_CODES, ksa = ka + 2 * PQ_CODES, vsa = ksa + PQ_SCALES;
            const int key_pos = w.template pos<PQ_TILE, Seqs>(w.tile + i) + key0;
            const int left = w.len - key_pos, early = Seqs::TAILS ? w.from - key_pos : 0;   // the warp's positions early .. left - 1 count
            if (left <= 0 || (Seqs::TAILS && early >= 32)) {  // none does
                if (lane == 0) mbar_arrive(&empty[st]);
                continue;
            }
            // scores of positions 16 kb + pg and 8 further by heads 8 n + 2 t4, + 1
            float s[2][NH][4];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int r0 = key0 + 16 * kb + pg;
                const float2 sc0 = lds2(ksa + r0 * 8), sc1 = lds2(ksa + (r0 + 8) * 8);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t at = ka + r0 * HD + (((4 * h + t4) ^ pg) << 4);
                    const uint4 x0 = lds16(at), x1 = lds16(at + 8 * HD);
                    const uint32_t c0[4] = {x0.x, x0.y, x0.z, x0.w}, c1[4] = {x1.x, x1.y, x1.z, x1.w};
                    uint32_t a[4][4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const uint32_t f0 = c0[y] ^ 0x80808080u, f1 = c1[y] ^ 0x80808080u;
                        a[y][0] = codes_f16(f0, 0x4140);
                        a[y][1] = codes_f16(f1, 0x4140);
                        a[y][2] = codes_f16(f0, 0x4342);
                        a[y][3] = codes_f16(f1, 0x4342);
                    }
#pragma unroll
                    for (int n = 0; n < NH; ++n) {
                        float acc[4] = {};
#pragma unroll
                        for (int x = PARTS - 1; x >= 0; --x) {
                            uint32_t mem[8];
                            if constexpr (!QREG) query(x, n, h, mem);
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                mma_f16(acc, a[y][0], a[y][1], a[y][2], a[y][3], QREG ? qf[QREG ? x : 0][QREG ? n : 0][h][2 * y] : mem[2 * y],
                                        QREG ? qf[QREG ? x : 0][QREG ? n : 0][h][2 * y + 1] : mem[2 * y + 1]);
                        }
                        // scales times the query's inverse lift, a power of two: products alone of a lifted query and keys from
                        // 2^100 on would leave binary32, where scores do not
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float sc = x < 2 ? (h ? sc0.y : sc0.x) : (h ? sc1.y : sc1.x), f = sc * back[n][x & 1];
                            s[kb][n][x] = h == 0 ? f * acc[x] : fmaf(f, acc[x], s[kb][n][x]);
                        }
                    }
                }
            }
            const bool cut_off = left < 32 || (Seqs::TAILS && early > 0);
            auto counts = [&](int at) { return at < left && (!Seqs::TAILS || at >= early); };
            if (cut_off) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        if (!counts(16 * kb + 8 * x + pg))
#pragma unroll
                            for (int n = 0; n < NH; ++n) s[kb][n][2 * x] = s[kb][n][2 * x + 1] = -INFINITY;
            }
            // softmax over the 32 positions, which the lanes of one t4 share
            float f[NH][2];
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NH; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float tm = fmaxf(fmaxf(s[0][n][h], s[0][n][2 + h]), fmaxf(s[1][n][h], s[1][n][2 + h]));
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) tm = fmaxf(tm, __shfl_xor_sync(FULL, tm, x));
                    f[n][h] = 1.0f;
                    if (tm > m[n][h]) {
                        f[n][h] = ex2_approx_ftz((m[n][h] - tm) * PD_LOG2);
                        m[n][h] = tm;
                        grow = true;
                    }
                    const float off = m[n][h] == -INFINITY ? 0.0f : -m[n][h] * PD_LOG2;
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        s[kb][n][h] = ex2_approx_ftz(fmaf(s[kb][n][h], PD_LOG2, off));
                        s[kb][n][2 + h] = ex2_approx_ftz(fmaf(s[kb][n][2 + h], PD_LOG2, off));
                    }
                    l[n][h] = fmaf(l[n][h], f[n][h], (s[0][n][h] + s[0][n][2 + h]) + (s[1][n][h] + s[1][n][2 + h]));
                }
            if (__any_sync(FULL, grow)) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int n = 0; n < NH; ++n)
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[j][n][x] *= f[n][x & 1];
            }
            // the values' scales: this lane's position's, for the lift, and those of the rows
            const float2 mine = lds2(vsa + (key0 + lane) * 8);
            const bool has = counts(lane);
            uint32_t top[2];
            top[0] = __reduce_max_sync(FULL, has ? __float_as_uint(mine.x) & 0x7fffffffu : 0u);
            top[1] = __reduce_max_sync(FULL, has ? __float_as_uint(mine.y) & 0x7fffffffu : 0u);
            float2 vs[2][2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 2; ++x) vs[kb][x] = lds2(vsa + (key0 + 16 * kb + 8 * x + pg) * 8);
            // a lane's share of the rows ldmatrix reads: positions 8 (i / 8 % 2) + row i % 8, 16-byte chunk + i / 16
            const int vrow = key0 + ((lane >> 3) & 1) * 8 + pq_row(lane & 7);
#pragma unroll
            for (int h = 0; h < 2; ++h) {                    // the dimensions of one scale
                const float up = lift(top[h]), down = lift_back(top[h]);
                uint32_t p[2][PARTS][NH][2];                 // weights: positions by heads, transposed
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float v = h ? vs[kb][x].y : vs[kb][x].x;
                        v = cut_off && !counts(16 * kb + 8 * x + pg) ? 0.0f : v * up;
#pragma unroll
                        for (int n = 0; n < NH; ++n) {
                            uint32_t w16[PARTS];
                            split_f16(s[kb][n][2 * x] * v, s[kb][n][2 * x + 1] * v, w16);
#pragma unroll
                            for (int y = 0; y < PARTS; ++y) p[kb][y][n][x] = transpose8x8(w16[y]);
                        }
                    }
#pragma unroll
                for (int jj = 0; jj < 2; ++jj) {             // two blocks of 16 dimensions
                    float acc[2][NH][4] = {};
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        uint32_t r[4];
                        ldsm4_t(va + (vrow + 16 * kb) * HD + (((4 * h + 2 * jj + (lane >> 4)) ^ (vrow & 7)) << 4), r);
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            const uint32_t f0 = r[2 * z] ^ 0x80808080u, f1 = r[2 * z + 1] ^ 0x80808080u;
                            const uint32_t a0 = codes_f16(f0, 0x4240), a1 = codes_f16(f0, 0x4341), a2 = codes_f16(f1, 0x4240),
                                           a3 = codes_f16(f1, 0x4341);
#pragma unroll
                            for (int n = 0; n < NH; ++n)
#pragma unroll
                                for (int y = PARTS - 1; y >= 0; --y)
                                    mma_f16(acc[z][n], a0, a1, a2, a3, p[kb][y][n][0], p[kb][y][n][1]);
                        }
                    }
#pragma unroll
                    for (int z = 0; z < 2; ++z)
#pragma unroll
                        for (int n = 0; n < NH; ++n)
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                float &to = o[4 * h + 2 * jj + z][n][x];
                                to = fmaf(acc[z][n][x], down, to);
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
        constexpr int AT_ONCE = WIDE ? 1 : 2;                // warps whose results fit the spare memory
#pragma unroll
        for (int src = 1; src < PQ_WARPS; src += AT_ONCE) {
            named_sync(1, PQ_WARPS * 32);
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
            named_sync(1, PQ_WARPS * 32);
            if (warp == 0) {
#pragma unroll
                for (int a = 0; a < AT_ONCE && src + a < PQ_WARPS; ++a) {
                    float f0[NH][2], f1[NH][2];
#pragma unroll
                    for (int n = 0; n < NH; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int head = 8 * n + 2 * t4 + h;
                            const float om = join_m[a][head], nm = fmaxf(m[n][h], om);
                            f0[n][h] = m[n][h] == nm ? 1.0f : ex2_approx_ftz((m[n][h] - nm) * PD_LOG2);
                            f1[n][h] = om == nm ? 1.0f : ex2_approx_ftz((om - nm) * PD_LOG2);
                            l[n][h] = fmaf(join_l[a][head], f1[n][h], l[n][h] * f0[n][h]);
                            m[n][h] = nm;
                        }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int n = 0; n < NH; ++n)
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                o[j][n][x] = fmaf(spare[(((a * 8 + j) * NH + n) * 4 + x) * 32 + lane], f1[n][x & 1], o[j][n][x] * f0[n][x & 1]);
                }
            }
        }
        ok = dead == 0;                                      // the same for every warp: the next barrier follows the read
        if (warp == 0 && ok) {
            const bool whole = run == w.tiles;
            constexpr int ROW = Seqs::TAILS ? SHARED_ROW : PD_PART;
#pragma unroll
            for (int n = 0; n < NH; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = 8 * n + 2 * t4 + h;
                    if (row >= group) continue;
                    if (whole && (!Seqs::TAILS || w.from == 0)) {
                        const float r = 1.0f / l[n][h];
                        typename Elem<T>::type *dst = out + (int64_t(w.s) * n_heads + w.head * group + row) * HD + 2 * g;
#pragma unroll
                        for (int j = 0; j < 8; ++j) put2(dst + 16 * j, 1, o[j][n][h] * r, o[j][n][2 + h] * r);
                    } else {
                        float *pd = Seqs::TAILS && whole
                                        ? tails + (int64_t(w.s) * n_heads + w.head * group + row) * ROW
                                        : part + ((2 * int64_t(blockIdx.x) + (u != u0)) * group + row) * ROW;
#pragma unroll
                        for (int j = 0; j < 8; ++j) put2(pd + 2 * g + 16 * j, 1, o[j][n][h], o[j][n][2 + h]);
                        if (g == 0) pd[HD] = m[n][h], pd[HD + 1] = l[n][h];
                    }
                }
        }
        u += units;
        if (u < u1) walk_on<PQ_TILE>(b, c, w, run);
        named_sync(1, PQ_WARPS * 32);
    }
}

template <typename T, typename Seqs>
static cudaError_t launch_q8(const PagedKV &c, const Seqs &b, const void *q, int64_t q_stride, int n_heads, float *part,
                             float *tails, void *out, uint32_t *status, cudaStream_t stream, int runs, int slot) {
    typedef typename Elem<T>::type E;
    CUtensorMap mk, mv, mks, mvs;
    const int box = Seqs::TAILS ? TAIL_ALIGN : PQ_TILE;
    if (!encode_pages_map(&mk, c.k, c, Q3CU_Q8_0, box) || !encode_pages_map(&mv, c.v, c, Q3CU_Q8_0, box) ||
        !encode_scales_map(&mks, c.k_scale, c, box) || !encode_scales_map(&mvs, c.v_scale, c, box))
        return cudaErrorInvalidValue;
    const int group = n_heads / c.n_kv;
    auto *kernel = group > 8 ? paged_q8_kernel<T, true, Seqs> : paged_q8_kernel<T, false, Seqs>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(kernel), PQ_SMEM, slot + (group > 8));
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, dim3(runs), dim3(PQ_THREADS), PQ_SMEM, stream, mk, mv, mks, mvs, c, b,
                            static_cast<const E *>(q), q_stride, n_heads, group, static_cast<E *>(out), part, tails, status);
}

cudaError_t launch_paged_q8(const PagedKV &c, const PagedSeqs &b, const void *q, q3cu_dtype dt, int64_t q_stride,
                            int n_heads, void *work, void *out, uint32_t *status, cudaStream_t stream, int sms) {
    const int runs = paged_runs(sms);
    float *part = static_cast<float *>(work);
    const WholeSeqs whole{b};
    if (dt == Q3CU_F32) {
        cudaError_t e = launch_q8<float>(c, whole, q, q_stride, n_heads, part, nullptr, out, status, stream, runs, 50);
        return e != cudaSuccess ? e : launch_paged_join<float, PQ_TILE>(c, b, n_heads, runs, out, part, stream);
    }
    cudaError_t e = launch_q8<bf16raw>(c, whole, q, q_stride, n_heads, part, nullptr, out, status, stream, runs, 52);
    return e != cudaSuccess ? e : launch_paged_join<bf16raw, PQ_TILE>(c, b, n_heads, runs, out, part, stream);
}

cudaError_t launch_tails_q8(const PagedKV &c, const TailSeqs &b, const void *q, int64_t q_stride, int n_heads, float *part,
                            float *tails, void *out, uint32_t *status, cudaStream_t stream, int runs) {
    return launch_q8<bf16raw>(c, b, q, q_stride, n_heads, part, tails, out, status, stream, runs, 54);
}

}  // namespace q3
