// k_prompt_f32.cu -- causal attention of packed f32 prompt rows over an f32 paged cache.
//
// The operation of k_prompt.cu, with nothing rounded below binary32's sums: a
// product of two f32 operands is taken as tf32 parts, high x high + high x low
// + low x high (the dropped low x low is 2^-22 of it), on mma.sync, in short
// chains that are added in binary32.  That is three tensor-core products for one, and still ahead of
// the FMA units.
//
// A work item is 64 rows -- row r is query r / g, head r % g of a group of g
// query heads -- against one kv head.  Four computing warps take 16 rows each
// over all keys, 32 at a time, with the running maximum and sum of the softmax;
// one warp fetches the key and value tiles page by page (TMA, 128-byte swizzle,
// two stages).  Two CTAs share an SM, so one's softmax runs beside the other's
// products.  The operands' index orders are chosen so that every shared-memory
// read is 16 bytes wide and free of bank conflicts (see the comments below).
// 2,000 rows in three prompts (16/8 heads): 166 us, 38 TFLOP/s of the operator,
// three times that of the tensor cores, whose mma.sync pipe is busy half the time.
// Masks and rows that come out as NaN are treated as in k_prompt.cu; values
// behind the sequence's end are masked in registers.
#include "q3cu_mma.cuh"
#include "q3cu_paged.cuh"
#include "q3cu_tma.h"

namespace q3 {

constexpr int PF_WARPS = 4, PF_THREADS = (PF_WARPS + 1) * 32, PF_ROWS = 16 * PF_WARPS, PF_KEYS = 32, PF_NS = 2;
constexpr uint32_t PF_SIDE = PF_KEYS * HD * 4, PF_STAGE = 2 * PF_SIDE;
constexpr size_t PF_SMEM = size_t(PF_NS) * PF_STAGE + size_t(PF_ROWS) * HD * 4 + 1024;
constexpr float PF_LOG2 = ATT_SCALE * 1.44269504088896341f;

__global__ void __launch_bounds__(PF_THREADS, 2)
prompt_f32_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const PagedKV c,
                  const PagedSeqs b, int rows, const float *q, int64_t q_stride, int n_heads, int group,
                  const FastDiv per_block, float *out, uint32_t *status) {
    extern __shared__ uint8_t pf_dyn[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pf_dyn) + 1023) & ~uintptr_t(1023));
    float *qs = reinterpret_cast<float *>(ring + PF_NS * PF_STAGE);
    __shared__ __align__(8) uint64_t full[PF_NS], empty[PF_NS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PF_NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], PF_WARPS);
        }
        mbar_init_fence();
    }
    griddep_wait();
    const int qt = per_block.d;                              // queries of an item
    const PromptItem it = PromptOrder(b, c, rows, per_block, PF_KEYS, warp == 0 ? status : nullptr).find(blockIdx.x);
    if (it.s < 0) return;
    const int len = it.len;
    auto seen = [&](int i) { return it.seen(i); };
    const int queries = min(qt, it.rows - it.first);
    const int nkv = (seen(it.first + queries - 1) + PF_KEYS - 1) / PF_KEYS;
    // the queries, 16-byte chunk x of row r at x ^ (r % 8) of its 128-byte block
    for (int x = threadIdx.x; x < PF_ROWS * (HD / 4); x += PF_THREADS) {
        const int r = x / (HD / 4), ch = x % (HD / 4);
        const bool live = r < queries * group;
        const float4 v = live ? load_quad(q + int64_t(it.base + it.first + r / group) * q_stride +
                                          int64_t(it.head * group + r % group) * HD + 4 * ch)
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        *reinterpret_cast<float4 *>(qs + r * HD + 4 * ((ch & 24) | ((ch ^ r) & 7))) = v;
    }
    __syncthreads();

    if (warp == PF_WARPS) {
        // ---- fetch: lane = box (K or V, 32 columns, rows of one page) --------------------
        const int br = min(1 << c.page_shift, PF_KEYS), nb = PF_KEYS / br;
        const int box = lane % nb, col = lane / nb % 4, side = lane / (4 * nb);
        auto page_of = [&](int j) -> int {                   // n_pages reads as zeros
            const int t = j * PF_KEYS + box * br;
            if (side > 1 || t >= len) return c.n_pages;
            const int p = paged_page(b, c, it.s, t, status);
            return p < 0 ? c.n_pages : p;
        };
        int page = nkv ? page_of(0) : 0, e = 0;
        bool ok = true;
        for (; e < nkv; ++e) {
            const int st = e % PF_NS, now = page, slot = (e * PF_KEYS + box * br) & ((1 << c.page_shift) - 1);
            if (e + 1 < nkv) page = page_of(e + 1);
            if (e >= PF_NS) ok = mbar_wait(&empty[st], uint32_t(e / PF_NS - 1) & 1u, lane == 0 ? status : nullptr);
            if (!__all_sync(FULL, ok)) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[st], PF_STAGE);
            __syncwarp();
            if (side < 2)
                tma_load_4d(ring + st * PF_STAGE + side * PF_SIDE + col * (PF_SIDE / 4) + box * br * 128,
                            side ? &tmv : &tmk, 32 * col, slot, it.head, now, &full[st]);
        }
        // no copy outlives the CTA (bounded)
        for (int d = e > PF_NS ? e - PF_NS : 0; d < e; ++d) mbar_wait(&full[d % PF_NS], uint32_t(d / PF_NS) & 1u, nullptr);
        return;
    }

    const int g = lane >> 2, t4 = lane & 3;                  // rows g, g + 8 of the warp's 16; column pair t4
    int limit[2], i_of[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = 16 * warp + g + 8 * h;
        i_of[h] = it.first + r / group;
        limit[h] = r < queries * group ? seen(i_of[h]) : 0;
    }
    const int sure = seen(it.first);                         // keys that every row sees
    float o[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const uint32_t qa = smem_addr(qs) + (16 * warp + g) * (HD * 4), ring_a = smem_addr(ring);
    bool ok = true;
    for (int j = 0; j < nkv; ++j) {
        const int st = j % PF_NS, base = j * PF_KEYS;
        ok = __all_sync(FULL, mbar_wait(&full[st], uint32_t(j / PF_NS) & 1u, lane == 0 ? status : nullptr));
        if (!ok) break;
        const uint32_t ka = ring_a + st * PF_STAGE, va = ka + PF_SIDE;
        float s[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
        // k index t4 is dimension 32 d + 8 t4 + 4 x + y, k index t4 + 4 is y + 1 (y = 0, 2): an order that query and
        // key share, so a lane reads 16 bytes of either, and the swizzle spreads eight rows over all banks
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t ch = uint32_t((2 * t4 + x) ^ g) << 4;
                uint32_t ah[2][4], al[2][4];                 // [y / 2]: rows g, g + 8 of k index t4, then of t4 + 4
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 v = lds4(qa + h * 8 * (HD * 4) + 128 * d + ch);
                    split_tf32(v.x, ah[0][h], al[0][h]);
                    split_tf32(v.y, ah[0][2 + h], al[0][2 + h]);
                    split_tf32(v.z, ah[1][h], al[1][h]);
                    split_tf32(v.w, ah[1][2 + h], al[1][2 + h]);
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float4 v = lds4(ka + d * (PF_SIDE / 4) + (8 * n + g) * 128 + ch);
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
        if (base + PF_KEYS > sure) {
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (base + 8 * n + 2 * t4 + (x & 1) >= limit[x >> 1]) s[n][x] = -INFINITY;
        }
        float f[2];
        bool grow = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float tm = -INFINITY;
#pragma unroll
            for (int n = 0; n < 4; ++n) tm = fmaxf(tm, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
            tm = fmaxf(tm, __shfl_xor_sync(FULL, tm, 1));
            tm = fmaxf(tm, __shfl_xor_sync(FULL, tm, 2));
            f[h] = 1.0f;
            if (tm > m[h]) {
                f[h] = ex2_approx_ftz((m[h] - tm) * PF_LOG2);
                m[h] = tm;
                grow = true;
            }
            const float off = m[h] == -INFINITY ? 0.0f : -m[h] * PF_LOG2;
            float add = 0.0f;
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int x = 2 * h; x < 2 * h + 2; ++x) {
                    s[n][x] = ex2_approx_ftz(fmaf(s[n][x], PF_LOG2, off));
                    add += s[n][x];
                }
            l[h] = fmaf(l[h], f[h], add);
        }
        if (__any_sync(FULL, grow)) {
#pragma unroll
            for (int x = 0; x < 16; ++x)
#pragma unroll
                for (int y = 0; y < 4; ++y) o[x][y] *= f[y >> 1];
        }
        // k index t4 is position 8 n + 2 t4, t4 + 4 the next one: the columns this thread's scores have; column i of
        // product (d, x) is dimension 32 d + 4 i + x
        const bool tail = base + PF_KEYS > len;
        uint32_t ph[4][4], pl[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                split_tf32(s[n][2 * h], ph[n][h], pl[n][h]);
                split_tf32(s[n][2 * h + 1], ph[n][2 + h], pl[n][2 + h]);
            }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            float part[4][4] = {}, low[4][4] = {};
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int k0 = 8 * n + 2 * t4;
                const uint32_t blk = va + d * (PF_SIDE / 4) + k0 * 128;
                float4 v0 = lds4(blk + ((g ^ (2 * t4)) << 4)), v1 = lds4(blk + 128 + ((g ^ (2 * t4 + 1)) << 4));
                if (tail) {
                    if (base + k0 >= len) v0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (base + k0 + 1 >= len) v1 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
                const float a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t bh[2], bl[2];
                    split_tf32(a0[x], bh[0], bl[0]);
                    split_tf32(a1[x], bh[1], bl[1]);
                    mma_tf32(low[x], pl[n][0], pl[n][1], pl[n][2], pl[n][3], bh[0], bh[1]);
                    mma_tf32(low[x], ph[n][0], ph[n][1], ph[n][2], ph[n][3], bl[0], bl[1]);
                    mma_tf32(part[x], ph[n][0], ph[n][1], ph[n][2], ph[n][3], bh[0], bh[1]);
                }
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) add_to(part[x], low[x]), add_to(o[4 * d + x], part[x]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
    }
    if (!ok) return;
    bool nan[2] = {false, false};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(FULL, l[h], 1);
        l[h] += __shfl_xor_sync(FULL, l[h], 2);
        const int r = 16 * warp + g + 8 * h;
        const float inv = limit[h] > 0 ? 1.0f / l[h] : 0.0f;
        float *dst = out + (int64_t(it.base + i_of[h]) * n_heads + it.head * group + r % group) * HD + 8 * t4;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float v[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    v[x] = limit[h] > 0 ? o[4 * d + x][2 * h + y] * inv : 0.0f;
                    nan[h] |= v[x] != v[x];
                }
                if (r < queries * group) store_quad(dst + 32 * d + 4 * y, make_float4(v[0], v[1], v[2], v[3]));
            }
    }
    // rows that came out as NaN, once more from the formula
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        unsigned again = __ballot_sync(FULL, nan[h] && limit[h] > 0);
        while (again) {
            const int first = (__ffs(again) - 1) & ~3;       // the row's four lanes
            again &= ~(15u << first);
            __syncwarp();
            const int i = __shfl_sync(FULL, i_of[h], first), n = __shfl_sync(FULL, limit[h], first);
            const int head = it.head * group + (16 * warp + first / 4 + 8 * h) % group;
            float4 x = load_quad(q + int64_t(it.base + i) * q_stride + int64_t(head) * HD + 4 * lane);
            x = make_float4(x.x * ATT_SCALE, x.y * ATT_SCALE, x.z * ATT_SCALE, x.w * ATT_SCALE);
            store_quad(out + (int64_t(it.base + i) * n_heads + head) * HD + 4 * lane,
                       attend_row<float>(c, b, it.s, it.head, n, x, status));
        }
    }
}

cudaError_t launch_prompt_f32(const PagedKV &c, const PagedSeqs &b, int64_t rows, const void *q, int64_t q_stride,
                              int n_heads, void *out, uint32_t *status, cudaStream_t stream) {
    const int group = n_heads / c.n_kv, qt = PF_ROWS / group;
    CUtensorMap mk, mv;
    if (!encode_pages_map(&mk, c.k, c, Q3CU_F32, PF_KEYS) || !encode_pages_map(&mv, c.v, c, Q3CU_F32, PF_KEYS))
        return cudaErrorInvalidValue;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(prompt_f32_kernel), PF_SMEM, 41);
    if (e != cudaSuccess) return e;
    // no more items than this, however the rows are split into sequences
    const int64_t items = (rows / qt + b.n_seqs) * c.n_kv;
    return launch_dependent(prompt_f32_kernel, dim3(unsigned(items)), dim3(PF_THREADS), PF_SMEM, stream, mk, mv, c, b,
                            int(rows), static_cast<const float *>(q), q_stride, n_heads, group, FastDiv(qt),
                            static_cast<float *>(out), status);
}

}  // namespace q3
