// k_prompt_f32.cu -- causal attention of packed f32 prompt rows over an f32 paged cache.
//
// The operation of k_prompt.cu, with nothing rounded below binary32's sums: each
// f32 operand is taken as three bf16 parts (24 bits of mantissa, split_bf16), and
// a product as the six products of parts that count (what is dropped is 2^-25 of
// it), on tcgen05 with binary32 accumulators.  The tensor cores cut their sums
// where binary32 would round them, so the small products go first and each key
// tile's P V starts afresh: the result itself is kept in registers and summed by
// ordinary additions.
//
// A work item is 128 rows -- row r is query r / g, head r % g of a group of g
// query heads -- against one kv head, 64 keys at a time, one CTA per SM:
//   warps 0-3    thread = row = tensor-memory lane.  Splits the row's query into
//                tensor memory once.  For each key tile: the running maximum and
//                sum of the softmax, the probabilities as three parts over the
//                scores, then the tile before's P V into the row's 128 registers.
//   warp 4       issues the products, queries and probabilities (the A operands)
//                from tensor memory, keys and values from shared memory.  The
//                next tile's scores are issued before this tile's P V, so that
//                the softmax runs beside them.
//   warps 8-11   read the keys, page by page, split them and store the parts as
//                the swizzled operand tiles, two stages; warps 12-15 the values.
// Tensor memory (512 columns): the query's parts 0-191, two slots of 96 for scores
// and the probabilities' parts over them, the tile's P V 384-511.
//
// With fewer items than SMs a cluster of up to eight CTAs takes an item, each a part of its key tiles, and joins the
// parts through shared memory (join_parts): 16 rows behind 8,000 positions (32/8 heads) 260 -> 51 us, 30 behind 30,000
// 1,140 -> 147 us.
//
// Bound by the instructions that split, exponentiate and add, beside a tensor pipe that is busy 72 % of the cycles
// when the prompt is long: 4,096 rows (32/8 heads) take 584 us in a replayed graph on one input and 665 over changing
// inputs (1.2 PFLOP/s of bf16 parts, at 1.6 GHz under the power cap), 2,000 rows in three prompts (16/8) 54 and 56 us,
// of which the longest prompt's last block is 42.
// Measured and left out: two threads to a row (they and the splitting warps then spill registers: 80 us for the three
// prompts), the next tile's loads ahead of this tile's split (57 us: the splitting warps then keep the rows' warps
// waiting for issue slots), parts by truncation in place of rounding (57 us, and a larger error).
//
// Masks and rows that come out as NaN are treated as in k_prompt.cu (SecondLook in q3cu_paged.cuh); keys and values
// behind the sequence's end are stored as zeros.  (An infinity splits into infinity and NaN, so its rows go the way of
// NaN rows and are computed from the formula.  An element below 2^-109 keeps fewer bits: its last part would be below
// bf16's least normal number, 2^-126.)
#include "q3cu_mma.cuh"
#include "q3cu_paged.cuh"
#include "q3cu_tcgen05.cuh"
#include "q3cu_tma.h"

namespace q3 {

constexpr int PF_ROWS = 128, PF_KEYS = 64, PF_THREADS = 16 * 32, PF_NS = 2;
constexpr int PF_WHOLE = 4;                                  // key tiles from which on an item may be shared
constexpr uint32_t PF_HALF = PF_KEYS * 128;                  // bytes of 64 keys x 64 elements of a part
constexpr uint32_t PF_PART = 2 * PF_HALF, PF_TILE = 3 * PF_PART;
constexpr size_t PF_SMEM = size_t(PF_NS) * 2 * PF_TILE + 1024;
constexpr uint32_t PF_SLOT = 192, PF_OUT = 384;              // tensor-memory columns: first slot, P V
// Instruction descriptors (f32 accumulator, bf16 A and B, M = 128): scores, N = 64 keys, and P V, N = 128, B MN-major.
constexpr uint32_t PF_IDESC_BASE = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 / 16) << 24);
constexpr uint32_t PF_IDESC = PF_IDESC_BASE | (uint32_t(PF_KEYS / 8) << 17);
constexpr uint32_t PF_IDESC_V = PF_IDESC_BASE | (uint32_t(HD / 8) << 17) | (1u << 16);
constexpr float PF_LOG2 = ATT_SCALE * 1.44269504088896341f;
// The products of parts from the smallest, the parts' numbers as hexadecimal digits from the right: low x high,
// high x low, mid x mid, mid x high, high x mid, high x high.
constexpr uint32_t PF_A = 0x001102, PF_B = 0x010120;
__host__ __device__ constexpr uint32_t pf_part(uint32_t parts, int x) { return parts >> (4 * x) & 15u; }
// Column of a slot where a part of 32 probabilities lies: those of keys 32 .. 63 (half 1) are stored first, over columns
// whose scores have been read (32 ..) or that have none (64 ..).
__host__ __device__ constexpr uint32_t pf_col(int half, uint32_t part) { return half ? 64 + part * 16 - part / 2 * 48 : part * 16; }

// 16 floats as three bf16 parts each, packed in pairs, to columns at[0 .. 2] of this thread's tensor-memory lane.
__device__ __forceinline__ void store_parts16(const float (&x)[16], uint32_t at0, uint32_t at1, uint32_t at2) {
    uint32_t w[3][8];
#pragma unroll
    for (int y = 0; y < 8; ++y) {
        uint32_t p[3];
        split_bf16<3>(x[2 * y], x[2 * y + 1], p);
        w[0][y] = p[0];
        w[1][y] = p[1];
        w[2][y] = p[2];
    }
    tc_st8(at0, w[0]);
    tc_st8(at1, w[1]);
    tc_st8(at2, w[2]);
}

// Eight consecutive floats, 32 bytes aligned, in one load.
__device__ __forceinline__ void load_eight(const float *p, float4 (&v)[2]) {
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0].x), "=f"(v[0].y), "=f"(v[0].z), "=f"(v[0].w), "=f"(v[1].x), "=f"(v[1].y), "=f"(v[1].z),
                   "=f"(v[1].w)
                 : "l"(p) : "memory");
}

// Row r of an item once more from the formula, where that may give numbers; false where not.
template <int STEP>
__device__ __forceinline__ bool look_again(SecondLook<float> &second, const PagedKV &c, const PagedSeqs &b,
                                           const PromptItem &it, int group, int r, const float *q, int64_t q_stride,
                                           uint32_t *status, float4 &v) {
    const int lane = threadIdx.x & 31, query = r / group, i = it.first + query, limit = it.seen(i);
    const int last = it.seen(min(it.first + PF_ROWS / group, it.rows) - 1);
    second.look(0, c, b, it.s, it.head, it.seen(it.first), min(it.len, (last + PF_KEYS - 1) / PF_KEYS * PF_KEYS));
    const float4 x = load_quad(q + int64_t(it.base + i) * q_stride + int64_t(it.head * group + r - query * group) * HD + 4 * lane);
    if (!second.wanted(limit, x)) return false;
    v = attend_row<float, STEP>(c, b, it.s, it.head, limit,
                          make_float4(x.x * ATT_SCALE, x.y * ATT_SCALE, x.z * ATT_SCALE, x.w * ATT_SCALE), status);
    return true;
}

template <bool SPLIT>
__global__ void __launch_bounds__(PF_THREADS, 1)
prompt_f32_kernel(const PagedKV c, const PagedSeqs b, int rows, const float *q, int64_t q_stride, int n_heads, int group,
                  const FastDiv per_block, int ctas, float *out, uint32_t *status) {
    extern __shared__ uint8_t pf_dyn[];
    uint8_t *tiles = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pf_dyn) + 1023) & ~uintptr_t(1023));
    // tiles of keys (side 0) and values (side 1), two stages each
    __shared__ __align__(8) uint64_t full[2][PF_NS], empty[2][PF_NS], q_full, s_full[2], p_full, o_full, drain;
    __shared__ PromptItem item_sh;
    __shared__ float2 stat_sh[SPLIT ? PF_ROWS : 1];          // maximum and sum of a shared item's rows
    __shared__ uint32_t tmem_sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PF_NS; ++i) {
            for (int side = 0; side < 2; ++side) {
                mbar_init(&full[side][i], 4);
                mbar_init(&empty[side][i], 1);
            }
            mbar_init(&s_full[i], 1);
        }
        mbar_init(&q_full, 4);
        mbar_init(&p_full, 4);
        mbar_init(&o_full, 1);
        mbar_init(&drain, 1);
        mbar_init_fence();
    }
    if (warp == 4) tc_alloc512(&tmem_sh);
    griddep_wait();
    if (warp == 8) {
        const PromptItem found = PromptOrder(b, c, rows, per_block, PF_KEYS, status).find(SPLIT ? blockIdx.x / unsigned(ctas) : blockIdx.x);
        if (lane == 0) item_sh = found;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tmem_sh;
    const PromptItem it = item_sh;
    const int block_queries = it.s < 0 ? 0 : min(per_block.d, it.rows - it.first);
    const int tiles_all = it.s < 0 ? 0 : (it.seen(it.first + block_queries - 1) + PF_KEYS - 1) / PF_KEYS;
    // this CTA's part of the item's key tiles: nkv from j0 on
    const int rank = SPLIT ? int(blockIdx.x % unsigned(ctas)) : 0, parts = SPLIT ? prompt_parts(ctas, tiles_all, PF_WHOLE) : 1;
    const bool mine = rank < parts;
    const int j0 = SPLIT && mine ? prompt_part(tiles_all, parts, rank) : 0;
    const int nkv = !SPLIT ? tiles_all : mine ? prompt_part(tiles_all, parts, rank + 1) - j0 : 0;
    const int queries = mine ? block_queries : 0;

    // Registers move to the rows: 128 threads x 224 + 384 x 96 is the launch's 512 x 128.
    if (warp >= 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (warp >= 8) {
            // ---- keys (warps 8-11) or values: 16 of a tile's rows per warp, in one page --------
            const int side = (warp - 8) >> 2, first = 16 * (warp & 3);
            const float *src = static_cast<const float *>(side ? c.v : c.k);
            const bool wide = reinterpret_cast<uintptr_t>(src) % 32 == 0;    // (a page's stride is a multiple of 32 bytes)
            const int chunk = lane & 15, row = lane >> 4;    // elements 8 chunk .. + 7 of rows row, row + 2, ...
            uint8_t *dst = tiles + side * PF_NS * PF_TILE + (chunk >> 3) * PF_HALF;
            // a page id is loaded one tile ahead
            auto id_of = [&](int j) -> int {
                const int t = (j0 + j) * PF_KEYS + first;
                return t < it.len ? b.pages[int64_t(it.s) * b.max_pages + (t >> c.page_shift)] : -1;
            };
            int next = nkv ? id_of(0) : -1;
            for (int j = 0; j < nkv; ++j) {
                const int st = j & 1, t = (j0 + j) * PF_KEYS + first, id = next;
                if (j + 1 < nkv) next = id_of(j + 1);
                const bool good = id >= 0 && id < c.n_pages;
                if (!good && t < it.len && lane == 0) flag_bad_index(status);
                const int n = good ? it.len - t : 0;         // rows from n on read as zeros
                const float *at = src + (good ? paged_at(c, id, it.head, t) : 0) + row * HD + 8 * chunk;
                float4 x[8][2];
                if (n >= 16 && wide) {
#pragma unroll
                    for (int u = 0; u < 8; ++u) load_eight(at + 2 * u * HD, x[u]);
                } else {
#pragma unroll
                    for (int u = 0; u < 8; ++u)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            x[u][h] = 2 * u + row < n ? load_quad(at + 2 * u * HD + 4 * h) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
                if (j >= PF_NS &&
                    !__all_sync(FULL, mbar_wait(&empty[side][st], uint32_t((j >> 1) - 1) & 1u, lane == 0 ? status : nullptr)))
                    break;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int r = first + row + 2 * u;
                    uint32_t w[4][3];
                    split_bf16<3>(x[u][0].x, x[u][0].y, w[0]);
                    split_bf16<3>(x[u][0].z, x[u][0].w, w[1]);
                    split_bf16<3>(x[u][1].x, x[u][1].y, w[2]);
                    split_bf16<3>(x[u][1].z, x[u][1].w, w[3]);
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        *reinterpret_cast<uint4 *>(dst + st * PF_TILE + p * PF_PART + r * 128 + (((chunk ^ r) & 7) << 4)) =
                            make_uint4(w[0][p], w[1][p], w[2][p], w[3][p]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[side][st]);
            }
        } else if (warp == 4) {
            // ---- products -----------------------------------------------------------------
            if (nkv && tc_elect()) {
                const uint64_t dk = tc_sdesc(smem_addr(tiles)), dv = tc_sdesc_mn(smem_addr(tiles + PF_NS * PF_TILE), PF_HALF);
                auto scores = [&](int st) {                  // S = Q K^T
#pragma unroll
                    for (int x = 0; x < 6; ++x)
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            tc_mma_bf16_ts(tbase + PF_SLOT + 96 * st, tbase + 64 * pf_part(PF_A, x) + 8 * k,
                                           dk + ((st * PF_TILE + pf_part(PF_B, x) * PF_PART + (k / 4) * PF_HALF + (k % 4) * 32) >> 4),
                                           PF_IDESC, uint32_t(x + k > 0));
                    tc_commit(&s_full[st]);
                    tc_commit(&empty[0][st]);
                };
                auto values = [&](int st) {                  // P V of one tile
#pragma unroll
                    for (int x = 0; x < 6; ++x)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc_mma_bf16_ts(tbase + PF_OUT, tbase + PF_SLOT + 96 * st + pf_col(k / 2, pf_part(PF_A, x)) + 8 * (k % 2),
                                           dv + ((st * PF_TILE + pf_part(PF_B, x) * PF_PART + k * 2048) >> 4), PF_IDESC_V,
                                           uint32_t(x + k > 0));
                    tc_commit(&o_full);
                    tc_commit(&empty[1][st]);
                };
                bool ok = mbar_wait(&q_full, 0, status) && mbar_wait(&full[0][0], 0, status);
                if (ok) {
                    tc_fence_after();
                    scores(0);
                }
                for (int j = 0; ok && j < nkv; ++j) {
                    if (j + 1 < nkv) {
                        // over the probabilities of tile j - 1, whose products are before these in the pipe
                        if (!(ok = mbar_wait(&full[0][(j + 1) & 1], uint32_t((j + 1) >> 1) & 1u, status))) break;
                        tc_fence_after();
                        scores((j + 1) & 1);
                    }
                    ok = mbar_wait(&full[1][j & 1], uint32_t(j >> 1) & 1u, status) &&
                         mbar_wait(&p_full, uint32_t(j) & 1u, status);
                    if (!ok) break;
                    tc_fence_after();
                    values(j & 1);
                }
                // every product issued has completed before tensor memory is given back (bounded)
                tc_commit(&drain);
                mbar_wait(&drain, 0, nullptr);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---- rows ---------------------------------------------------------------------
        const int r = threadIdx.x, r_query = r / group, i = it.first + r_query;
        const int head = it.head * group + r - r_query * group;
        const bool live = r_query < queries;
        const int limit = live ? it.seen(i) : 0;
        const int sure = queries ? it.seen(it.first) : 0;    // keys that every row sees
        const uint32_t lane_base = tbase + (uint32_t(32 * warp) << 16);
        bool ok = true;
        if (nkv) {
            const float *row = q + int64_t(it.base + i) * q_stride + int64_t(head) * HD;
#pragma unroll
            for (int z = 0; z < 2; ++z) {                    // 64 elements' loads at a time
                float4 f[16];
#pragma unroll
                for (int y = 0; y < 16; ++y)
                    f[y] = live ? load_quad(row + 64 * z + 4 * y) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    float v[16];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        v[4 * y] = f[4 * x + y].x;
                        v[4 * y + 1] = f[4 * x + y].y;
                        v[4 * y + 2] = f[4 * x + y].z;
                        v[4 * y + 3] = f[4 * x + y].w;
                    }
                    const uint32_t at = lane_base + 32 * z + 8 * x;
                    store_parts16(v, at, at + 64, at + 128);
                }
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
        }
        float o[HD];
#pragma unroll
        for (int x = 0; x < HD; ++x) o[x] = 0.0f;
        float m = -INFINITY, sum = 0.0f, f_before = 0.0f;
        // adds the P V of the latest tile, whose maximum was `f` times further up than what o holds
        auto add_tile = [&](float f) {
#pragma unroll
            for (int x = 0; x < HD / 32; ++x) {
                uint32_t u[32];
                tc_ld32(lane_base + PF_OUT + 32 * x, u);
                tc_wait_ld32(u);
#pragma unroll
                for (int y = 0; y < 32; ++y) o[32 * x + y] = fmaf(o[32 * x + y], f, __uint_as_float(u[y]));
            }
        };
        for (int j = 0; j < nkv; ++j) {
            ok = __all_sync(FULL, mbar_wait(&s_full[j & 1], uint32_t(j >> 1) & 1u, lane == 0 ? status : nullptr));
            if (!ok) break;
            tc_fence_after();
            const uint32_t slot = lane_base + PF_SLOT + 96 * (j & 1);
            const int left = limit - (j0 + j) * PF_KEYS;            // columns of this tile that the row sees
            const bool mask = (j0 + j + 1) * PF_KEYS > sure;
            float tile_max = -INFINITY;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t u[32];
                tc_ld32(slot + 32 * x, u);
                tc_wait_ld32(u);
                if (mask) mask32(u, left - 32 * x);
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int y = 0; y < 32; ++y) mx[y & 3] = fmaxf(mx[y & 3], __uint_as_float(u[y]));
                tile_max = fmaxf(tile_max, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
            }
            float f = 1.0f;
            if (tile_max > m) {
                f = ex2_approx_ftz((m - tile_max) * PF_LOG2);
                m = tile_max;
            }
            const float off = m == -INFINITY ? 0.0f : -m * PF_LOG2;
            float add[2] = {0.0f, 0.0f};
#pragma unroll
            for (int x = 1; x >= 0; --x) {
                uint32_t u[32];
                tc_ld32(slot + 32 * x, u);
                tc_wait_ld32(u);
                if (mask) mask32(u, left - 32 * x);
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    float p[16];
#pragma unroll
                    for (int y = 0; y < 16; ++y) {
                        p[y] = ex2_approx_ftz(fmaf(__uint_as_float(u[16 * z + y]), PF_LOG2, off));
                        add[y & 1] += p[y];
                    }
                    store_parts16(p, slot + pf_col(x, 0) + 8 * z, slot + pf_col(x, 1) + 8 * z, slot + pf_col(x, 2) + 8 * z);
                }
            }
            sum = fmaf(sum, f, add[0] + add[1]);
            if (j > 0) {
                ok = __all_sync(FULL, mbar_wait(&o_full, uint32_t(j - 1) & 1u, lane == 0 ? status : nullptr));
                if (!ok) break;
                tc_fence_after();
                add_tile(f_before);
            }
            f_before = f;
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full);
        }
        if (nkv && ok) {
            ok = __all_sync(FULL, mbar_wait(&o_full, uint32_t(nkv - 1) & 1u, lane == 0 ? status : nullptr));
            if (ok) {
                tc_fence_after();
                add_tile(f_before);
            }
        }
        if (ok) {
            const float inv = SPLIT && parts > 1 ? 1.0f : limit > 0 ? 1.0f / sum : 0.0f;
            bool nan = false;
            // through shared memory (its tiles are done with), so that a warp stores a row at a time: chunk x of the
            // warp's row l at x ^ (l % 8)
            uint8_t *stage = tiles + warp * 32 * (HD * 4);
#pragma unroll
            for (int x = 0; x < HD / 4; ++x) {
                float v[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    v[y] = limit > 0 ? o[4 * x + y] * inv : 0.0f;
                    nan |= v[y] != v[y];
                }
                *reinterpret_cast<float4 *>(stage + lane * (HD * 4) + ((x ^ (lane & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
            }
            __syncwarp();
            const unsigned lives = __ballot_sync(FULL, live && !(SPLIT && parts > 1));
            for (int l = 0; l < 32; ++l) {
                const int at = __shfl_sync(FULL, i * n_heads + head, l);     // below rows * n_heads
                if (lives >> l & 1u)
                    store_quad(out + (int64_t(it.base) * n_heads + at) * HD + 4 * lane,
                               *reinterpret_cast<const float4 *>(stage + l * (HD * 4) + ((lane ^ (l & 7)) << 4)));
            }
            __syncwarp();
            // rows that came out as NaN, once more from the formula; the item is read anew, so that it takes no registers until
            // then (1.2 us of the three prompts' 54)
            unsigned again = __ballot_sync(FULL, live && limit > 0 && nan && !(SPLIT && parts > 1));
            if (again) {
                const PromptItem *same = &item_sh;
                asm volatile("" : "+l"(same) :: "memory");
                SecondLook<float> second;
                __syncwarp();
                for (; again; again &= again - 1) {
                    const int row = 32 * warp + __ffs(again) - 1, query = row / group;
                    float4 v;
                    if (look_again<8>(second, c, b, *same, group, row, q, q_stride, status, v))
                        store_quad(out + (int64_t(same->base + same->first + query) * n_heads + same->head * group + row - query * group) * HD +
                                       4 * lane, v);
                }
            }
        }
        if constexpr (SPLIT) stat_sh[r] = make_float2(m, ok ? sum : -1.0f);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 4) tc_free512(tbase);
    if constexpr (SPLIT) {
        if (parts == 1 || !mine) return;                     // the same for all of a part's threads
        cluster_sync();
        SecondLook<float> second;
        for (int r = prompt_part(PF_ROWS, parts, rank) + warp; r < prompt_part(PF_ROWS, parts, rank + 1); r += PF_THREADS / 32) {
            const int query = r / group, i = it.first + query, head = it.head * group + r - query * group;
            if (query >= queries) break;
            const int limit = it.seen(i);
            bool ok;
            float4 v = join_parts(smem_addr(tiles) + r * (HD * 4), smem_addr(&stat_sh[r]), r, parts, PF_LOG2, ok);
            if (!ok) continue;
            if (limit <= 0) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (__any_sync(FULL, v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w))
                look_again<4>(second, c, b, it, group, r, q, q_stride, status, v);
            store_quad(out + (int64_t(it.base + i) * n_heads + head) * HD + 4 * lane, v);
        }
        cluster_sync();                                      // no CTA's shared memory goes while others read it
    }
}

cudaError_t launch_prompt_f32(const PagedKV &c, const PagedSeqs &b, int64_t rows, const void *q, int64_t q_stride,
                              int n_heads, void *out, uint32_t *status, cudaStream_t stream) {
    const int group = n_heads / c.n_kv, qt = PF_ROWS / group;
    // no more items than this, however the rows are split into sequences
    const int64_t items = (rows / qt + b.n_seqs) * c.n_kv;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(prompt_f32_kernel<true>), PF_SMEM, 42);
    if (e == cudaSuccess) e = ensure_smem_attr(reinterpret_cast<const void *>(prompt_f32_kernel<false>), PF_SMEM, 41);
    if (e != cudaSuccess) return e;
    const int ctas = prompt_cluster(reinterpret_cast<const void *>(prompt_f32_kernel<true>), 1, PF_THREADS, PF_SMEM, items,
                                    (int64_t(b.max_pages) << c.page_shift) / PF_KEYS);
    auto kernel = ctas > 1 ? prompt_f32_kernel<true> : prompt_f32_kernel<false>;
    return launch_clusters(kernel, ctas, dim3(unsigned(items * ctas)), dim3(PF_THREADS), PF_SMEM, stream, c, b, int(rows),
                           static_cast<const float *>(q), q_stride, n_heads, group, FastDiv(qt), ctas,
                           static_cast<float *>(out), status);
}

}  // namespace q3
