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
// on the other's.  One CTA per item, twelve warps (two of them idle):
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
//   warp 9   fetches Q and then the key and value tiles of 128 positions, page by page, by TMA
//            into a ring of five 32 KB buffers.
// Tensor memory (512 columns): S0, S1, O0, O1; P_t lies over the first half of S_t.
//
// Masks: keys at and beyond the row's limit become -inf before the maximum.
// Their probability is exactly 0, but 0 times a NaN or an infinity in V is not:
// the values behind the sequence's end (never written, anything may be there) are
// zeroed in shared memory, and a row whose result is NaN is computed again from
// the formula by one warp (attend_row), so that a value at a later position of
// the sequence never reaches an earlier row.
//
// Every wait is bounded; a wait that gives up sets Q3CU_DEV_TIMEOUT and the CTA
// drains its own copies and products, frees tensor memory and returns.
#include "q3cu_paged.cuh"
#include "q3cu_tcgen05.cuh"
#include "q3cu_tma.h"

namespace q3 {

constexpr int PT_ROWS = 128, PT_KEYS = 128;                  // rows of a tile, keys of a tile
constexpr int PT_THREADS = 12 * 32;
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
// through it: x = n + f with n whole and |f| <= 1/2, a polynomial for 2^f, n added to the exponent.  The coefficients
// are the minimax fit of degree 3 to 2^f (relative error 7.5e-5, a fiftieth of the bf16 rounding that follows), found
// by Remez exchange.  Below 2^-126 the result is 2^-126.
__device__ __forceinline__ void exp2_poly(float &x, float &y) {
    const f2 v = pk2(fmaxf(x, -126.0f), fmaxf(y, -126.0f)), magic = pk2(12582912.0f, 12582912.0f);   // 1.5 * 2^23
    const f2 t = add2(v, magic), f = sub2(v, sub2(t, magic));
    f2 p = pk2(0.0551716685295105f, 0.0551716685295105f);
    p = fma2(p, f, pk2(0.2426111251115799f, 0.2426111251115799f));
    p = fma2(p, f, pk2(0.6932609677314758f, 0.6932609677314758f));
    p = fma2(p, f, pk2(0.9999280571937561f, 0.9999280571937561f));
    float t0, t1, p0, p1;
    up2(t, t0, t1);
    up2(p, p0, p1);
    x = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
    y = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}
#ifndef PT_POLY
#define PT_POLY 8                                            // one pair of exponentials in PT_POLY / 2 by polynomial
#endif

// Scores from column n of 32 on become -inf.
__device__ __forceinline__ void mask32(uint32_t *v, int n) {
#pragma unroll
    for (int y = 0; y < 32; ++y)
        if (y >= n) v[y] = 0xff800000u;
}

__global__ void __launch_bounds__(PT_THREADS, 1)
prompt_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                 const __grid_constant__ CUtensorMap tmv, const PagedKV c, const PagedSeqs b, int64_t rows,
                 const uint16_t *q, int64_t q_stride, int n_heads, int group, uint16_t *out, uint32_t *status) {
    extern __shared__ uint8_t pt_dyn[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pt_dyn) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = smem + 2 * PT_TILE;
    __shared__ __align__(8) uint64_t q_full, full[PT_NS], empty[PT_NS], s_full[2], p_full[2][2], o_full[2], drain;
    __shared__ uint32_t tmem_sh;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        for (int i = 0; i < PT_NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t][0], 4);
            mbar_init(&p_full[t][1], 4);
            mbar_init(&o_full[t], 1);
        }
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
    const PromptItem it = prompt_item(b, c, rows, 2 * qt, blockIdx.x);
    const bool item = it.s >= 0;
    // position of the sequence's row i is pos0 + i; keys that row sees: min(len, pos + 1)
    const int len = item ? paged_len(b, c, it.s, threadIdx.x == 0 ? status : nullptr) : 0;
    const int64_t pos0 = item ? int64_t(b.kv_len[it.s]) - it.rows : 0;
    auto seen = [&](int i) -> int {
        const int64_t n = pos0 + i + 1;
        return n < 0 ? 0 : n < len ? int(n) : len;
    };
    int nt[2];                                               // key tiles of each row tile
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = it.first + t * qt, last = min(first + qt, it.rows) - 1;
        nt[t] = item && last >= first ? (seen(last) + PT_KEYS - 1) / PT_KEYS : 0;
    }
    const int nkv = max(nt[0], nt[1]);

    // Registers move to the softmax: 256 threads x 208 + 128 x 88 is the launch's 384 x 168.
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 9) {
            // ---- fetch -------------------------------------------------------------------
            const int br = min(1 << c.page_shift, PT_KEYS), nb = PT_KEYS / br;      // rows of a box, boxes of a tile
            if (nkv > 0) {
                if (lane == 0) {
                    uint32_t bytes = 0;
                    for (int t = 0; t < 2; ++t)
                        if (nt[t]) bytes += 2u * qt * group * 128;
                    mbar_arrive_expect_tx(&q_full, bytes);
                    for (int t = 0; t < 2; ++t)
                        for (int h = 0; h < 2 && nt[t]; ++h)
                            tma_load_3d(smem + t * PT_TILE + h * PT_HALF, &tmq, 64 * h, it.head * group,
                                        int(it.base) + it.first + t * qt, &q_full);
                }
                __syncwarp();
                int e = 0;
                bool ok = true;
                // lane = box: column half lane / nb, positions lane % nb
                const int box = lane % nb, half = lane / nb;
                auto page_of = [&](int j) -> int {               // n_pages reads as zeros
                    const int t = j * PT_KEYS + box * br;
                    if (half > 1 || t >= len) return c.n_pages;
                    const int p = paged_page(b, c, it.s, t, status);
                    return p < 0 ? c.n_pages : p;
                };
                int page = page_of(0);
                for (int j = 0; j < nkv && ok; ++j) {
                    const int next = j + 1 < nkv ? page_of(j + 1) : 0;
                    const int slot = (j * PT_KEYS + box * br) & ((1 << c.page_shift) - 1);
                    for (int kv = 0; kv < 2 && ok; ++kv, ++e) {
                        const int st = e % PT_NS;
                        if (e >= PT_NS)
                            ok = mbar_wait(&empty[st], uint32_t(e / PT_NS - 1) & 1u, lane == 0 ? status : nullptr);
                        ok = __all_sync(FULL, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&full[st], PT_TILE);
                        __syncwarp();
                        if (half < 2)
                            tma_load_4d(ring + st * PT_TILE + half * PT_HALF + box * br * 128, kv ? &tmv : &tmk, 64 * half, slot,
                                        it.head, page, &full[st]);
                    }
                    page = next;
                }
                // no copy outlives the CTA (bounded)
                for (int d = e > PT_NS ? e - PT_NS : 0; d < e; ++d) mbar_wait(&full[d % PT_NS], uint32_t(d / PT_NS) & 1u, nullptr);
                mbar_wait(&q_full, 0, nullptr);
            }
        } else if (warp == 8) {
            // ---- products ----------------------------------------------------------------
            if (nkv > 0) {
                bool ok = mbar_wait(&q_full, 0, lane == 0 ? status : nullptr);
                // operand descriptors of the first row tile and the first buffer; a 32 KB tile further is + 2048
                const uint64_t dq = tc_sdesc(smem_addr(smem)), dk = tc_sdesc(smem_addr(ring)),
                               dv = tc_sdesc_mn(smem_addr(ring), PT_HALF);
                auto wait = [&](uint64_t *bar, uint32_t parity) {
                    if (ok) ok = mbar_wait(bar, parity, lane == 0 ? status : nullptr);
                    ok = __all_sync(FULL, ok);
                    tc_fence_after();
                };
                auto scores = [&](int t, int buf) {          // S_t = Q_t K^T
                    if (tc_elect()) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const uint32_t off = (uint32_t(k / 4) * PT_HALF + uint32_t(k % 4) * 32) >> 4;
                            tc_mma_bf16_ss(tbase + t * 128, dq + t * (PT_TILE >> 4) + off, dk + buf * (PT_TILE >> 4) + off,
                                           PT_IDESC, uint32_t(k > 0));
                        }
                        tc_commit(&s_full[t]);
                    }
                    __syncwarp();
                };
                wait(&full[0], 0);
                if (ok)
                    for (int t = 0; t < 2; ++t)
                        if (nt[t]) scores(t, 0);
                if (ok && tc_elect()) tc_commit(&empty[0]);
                __syncwarp();
                int bv = 1, bk = 2;                          // buffers of V(j) and K(j + 1), and how often each was filled before
                uint32_t pv = 0, pk = 0;
                for (int j = 0; j < nkv && ok; ++j) {
                    wait(&full[bv], pv & 1u);
                    if (!ok) break;
                    if (j == nkv - 1 && len < nkv * PT_KEYS) {        // values behind the sequence's end: zeros
                        for (int r = len - j * PT_KEYS + lane / 8; r < PT_KEYS; r += 4)
                            for (int h = 0; h < 2; ++h)
                                *reinterpret_cast<uint4 *>(ring + bv * PT_TILE + h * PT_HALF + r * 128 + (lane & 7) * 16) =
                                    make_uint4(0, 0, 0, 0);
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    for (int t = 0; t < 2 && ok; ++t) {
                        if (j < nt[t]) {
#pragma unroll
                            for (int half = 0; half < 2; ++half) {    // O_t += P_t V, 64 keys at a time
                                wait(&p_full[t][half], uint32_t(j) & 1u);
                                if (!ok) break;
                                if (tc_elect()) {
#pragma unroll
                                    for (int k = 4 * half; k < 4 * half + 4; ++k)
                                        tc_mma_bf16_ts(tbase + 256 + t * 128, tbase + t * 128 + k * 8,
                                                       dv + bv * (PT_TILE >> 4) + k * (2048 >> 4), PT_IDESC_V,
                                                       k > 0 ? 1u : uint32_t(j > 0));
                                    if (half && j + 1 == nt[t]) tc_commit(&o_full[t]);
                                }
                                __syncwarp();
                            }
                            if (!ok) break;
                        }
                        if (j + 1 < nt[t]) {
                            wait(&full[bk], pk & 1u);
                            if (!ok) break;
                            scores(t, bk);
                        }
                    }
                    if (ok && tc_elect()) {
                        tc_commit(&empty[bv]);
                        if (j + 1 < nkv) tc_commit(&empty[bk]);
                    }
                    __syncwarp();
                    if ((bv += 2) >= PT_NS) bv -= PT_NS, ++pv;
                    if ((bk += 2) >= PT_NS) bk -= PT_NS, ++pk;
                }
                // every product issued has completed before tensor memory is given back (bounded)
                if (tc_elect()) tc_commit(&drain);
                __syncwarp();
                mbar_wait(&drain, 0, nullptr);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax -----------------------------------------------------------------
        const int t = warp >> 2, r = threadIdx.x & 127;      // row tile, row = tensor-memory lane
        const uint32_t lane_base = tbase + (uint32_t(32 * (warp & 3)) << 16);
        const uint32_t ts = lane_base + t * 128, to = lane_base + 256 + t * 128;
        const int i = it.first + t * qt + r / group;         // the sequence's row
        const bool live = item && r < qt * group && i < it.rows;
        const int limit = live ? seen(i) : 0;
        const int sure = item ? seen(it.first + t * qt) : 0; // keys that every row of the tile sees
        float m = -INFINITY, sum = 0.0f;
        bool ok = true;
        for (int j = 0; j < nt[t] && ok; ++j) {
            ok = __all_sync(FULL, mbar_wait(&s_full[t], uint32_t(j) & 1u, lane == 0 ? status : nullptr));
            if (!ok) break;
            tc_fence_after();
            uint32_t u[128];
#pragma unroll
            for (int x = 0; x < 4; ++x) tc_ld32(ts + 32 * x, u + 32 * x);
#pragma unroll
            for (int x = 0; x < 4; ++x) tc_wait_ld32(u + 32 * x);
            if ((j + 1) * PT_KEYS > sure) {
#pragma unroll
                for (int x = 0; x < 4; ++x) mask32(u + 32 * x, limit - j * PT_KEYS - 32 * x);
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
        if (nt[t] > 0 && ok) {
            ok = __all_sync(FULL, mbar_wait(&o_full[t], 0, lane == 0 ? status : nullptr));
            tc_fence_after();
        }
        if (ok && item) {
            uint16_t *dst = out + ((it.base + i) * n_heads + it.head * group + r % group) * HD;
            const float inv = limit > 0 ? 1.0f / sum : 0.0f;
            bool nan = false;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t o[32];
                if (nt[t] > 0) {
                    tc_ld32(to + 32 * x, o);
                    tc_wait_ld32(o);
                }
#pragma unroll
                for (int y = 0; y < 32; y += 2) {
                    const float a = __uint_as_float(o[y]) * inv, d = __uint_as_float(o[y + 1]) * inv;
                    nan |= a != a || d != d;
                    o[y / 2] = limit > 0 ? pack_bf16(a, d) : 0u;
                }
                if (live) {
#pragma unroll
                    for (int y = 0; y < 16; y += 4)
                        st_cs_v4(dst + 32 * x + 2 * y, make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]));
                }
            }
            // rows that came out as NaN, once more from the formula
            unsigned again = __ballot_sync(FULL, live && limit > 0 && nan);
            while (again) {
                const int l = __ffs(again) - 1;
                again &= again - 1;
                __syncwarp();
                const int il = __shfl_sync(FULL, i, l), n = __shfl_sync(FULL, limit, l);
                const int h = it.head * group + __shfl_sync(FULL, r % group, l);
                float4 x = load_quad(q + (it.base + il) * q_stride + int64_t(h) * HD + 4 * lane);
                x = make_float4(x.x * ATT_SCALE, x.y * ATT_SCALE, x.z * ATT_SCALE, x.w * ATT_SCALE);
                store_quad(out + ((it.base + il) * n_heads + h) * HD + 4 * lane,
                           attend_row<bf16raw>(c, b, it.s, it.head, n, x, status));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tc_free512(tbase);
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
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(prompt_tc_kernel), PT_SMEM, 32);
    if (e != cudaSuccess) return e;
    // no more blocks of 2 * qt queries than this, however the rows are split into sequences
    const int64_t items = (rows / (2 * qt) + b.n_seqs) * c.n_kv;
    return launch_dependent(prompt_tc_kernel, dim3(unsigned(items)), dim3(PT_THREADS), PT_SMEM, stream, mq, mk, mv, c, b,
                            rows, static_cast<const uint16_t *>(q), q_stride, n_heads, group,
                            static_cast<uint16_t *>(out), status);
}

}  // namespace q3
