// k_append.cu -- packed token rows into the paged key-value cache, with the
// QK-RMSNorm and the rotation of query and key on the way.
//
// Per token row at position p, per query and key head x of 128 (the operation of
// src/cpu/qwen3_original.c:361-393, batched; without norm weights only the
// rotation):
//     y_i = w_i * (x_i / sqrtf(mean(x^2) + eps))
//     o_j      = y_j cos(a_j) - y_{j+64} sin(a_j)
//     o_{j+64} = y_j sin(a_j) + y_{j+64} cos(a_j),   a_j = p * theta^(-j/64), j < 64
// The key heads go to their page slots in the cache's type, the value heads are
// converted and stored beside them, the query heads go to q_out.
//
// The angle is formed in binary64 as turns, p * (theta^(-j/64) / 2 pi) less its
// nearest whole number, so it is as exact at position 100,000 as at 0 (a
// binary32 product is off by up to 0.004 rad there); the remainder is carried
// as a pair of floats into sincospif and a first-order correction.  Sums are
// binary32; the one rounding to fewer bits is the store.
//
// Bound by memory: every element is read once and written once.  A warp takes
// one row, or with few rows a part of its heads, in batches of APPEND_HEADS
// heads of one kind: lane l holds elements 2l, 2l+1, 64+2l, 65+2l of each head,
// so both halves of a rotated pair are in one lane, a half row is one contiguous
// access, and the two angles of a lane, found once, serve all its heads.  The
// row is on its way to L2 while the warp finds its sequence, position and page.
// 4,096 rows (32/8 heads): f32 to bf16 30.4 us, 5.0 TB/s, bf16 to bf16 24.1 us, 4.2
// TB/s, f32 to f32 38.5 us, 5.2 TB/s; one row: 3.3 us.
#include "q3cu_paged.cuh"

namespace q3 {

__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" :: "l"(p)); }

constexpr int APPEND_HEADS = 4, APPEND_WARPS = 8;

// Coherent loads: q_out may be q itself (a lane reads its elements before it stores them).
__device__ __forceinline__ float2 load_pair(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 load_pair(const uint16_t *p) {
    const uint32_t u = *reinterpret_cast<const uint32_t *>(p);
    return make_float2(bf16_to_f32(u & 0xffffu), bf16_to_f32(u >> 16));
}
// v as elements at, at + 1 of base.
template <bool BF16>
__device__ __forceinline__ void store_pair(void *base, int64_t at, float2 v) {
    if constexpr (BF16) *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(base) + at) = pack_bf16(v.x, v.y);
    else *reinterpret_cast<float2 *>(static_cast<float *>(base) + at) = v;
}

// Up to APPEND_HEADS heads from x (this lane's elements of the first), `step` elements apart where they go; turned by
// w if ROTATE, and normalised before if `norm` (the norm's weights are in w).
struct Turn { float2 c[2], s[2]; };                          // weight * cosine, weight * sine of both halves
template <typename E, bool BF16, bool ROTATE>
__device__ __forceinline__ void append_heads(const E *x, int n, bool norm, float eps, const Turn &w, void *to, int64_t at,
                                             int64_t step) {
    float2 l[APPEND_HEADS], h[APPEND_HEADS];
#pragma unroll
    for (int i = 0; i < APPEND_HEADS; ++i) {
        l[i] = h[i] = make_float2(0.0f, 0.0f);
        if (i < n) {
            l[i] = load_pair(x + i * HD);
            h[i] = load_pair(x + i * HD + 64);
        }
    }
    if constexpr (ROTATE) {
        float g[APPEND_HEADS] = {1.0f, 1.0f, 1.0f, 1.0f};
        if (norm) {
#pragma unroll
            for (int i = 0; i < APPEND_HEADS; ++i)
                g[i] = fmaf(l[i].x, l[i].x, fmaf(l[i].y, l[i].y, fmaf(h[i].x, h[i].x, h[i].y * h[i].y)));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int i = 0; i < APPEND_HEADS; ++i) g[i] += __shfl_xor_sync(FULL, g[i], o);
#pragma unroll
            for (int i = 0; i < APPEND_HEADS; ++i) g[i] = rsqrtf(fmaf(g[i], 1.0f / HD, eps));
        }
#pragma unroll
        for (int i = 0; i < APPEND_HEADS; ++i) {
            const float2 y = make_float2(g[i] * l[i].x, g[i] * l[i].y), z = make_float2(g[i] * h[i].x, g[i] * h[i].y);
            l[i] = make_float2(fmaf(y.x, w.c[0].x, -(z.x * w.s[1].x)), fmaf(y.y, w.c[0].y, -(z.y * w.s[1].y)));
            h[i] = make_float2(fmaf(y.x, w.s[0].x, z.x * w.c[1].x), fmaf(y.y, w.s[0].y, z.y * w.c[1].y));
        }
    }
#pragma unroll
    for (int i = 0; i < APPEND_HEADS; ++i)
        if (i < n) {
            store_pair<BF16>(to, at + i * step, l[i]);
            store_pair<BF16>(to, at + i * step + 64, h[i]);
        }
}

template <typename T, bool QB, bool CB>
__global__ void __launch_bounds__(APPEND_WARPS * 32, 4)
kv_append_kernel(const PagedKV c, const PagedSeqs b, int rows, const typename Elem<T>::type *q,
                 const typename Elem<T>::type *k, const typename Elem<T>::type *v, int64_t q_stride,
                 int64_t kv_stride, int n_heads, const float *__restrict__ q_norm, const float *__restrict__ k_norm,
                 const __grid_constant__ TurnFreq freq, float eps, void *q_out, uint32_t *status) {
    typedef typename Elem<T>::type E;
    __shared__ double turn[64];
    if (threadIdx.x < 64) turn[threadIdx.x] = freq.v[threadIdx.x];
    __syncthreads();
    griddep_wait();
    const int lane = threadIdx.x & 31, r = int(blockIdx.x) * APPEND_WARPS + int(threadIdx.x >> 5);
    if (r >= rows) return;
    // the row's batches: of query heads, of key heads, of value heads; this warp's are first .. last - 1
    const int qn = (n_heads + APPEND_HEADS - 1) / APPEND_HEADS, kn = (c.n_kv + APPEND_HEADS - 1) / APPEND_HEADS;
    const int first = int(int64_t(qn + 2 * kn) * blockIdx.y / gridDim.y);
    const int last = int(int64_t(qn + 2 * kn) * (blockIdx.y + 1) / gridDim.y);
    const E *qr = q + r * q_stride, *kr = k + r * kv_stride, *vr = v + r * kv_stride;
    constexpr int LINES = APPEND_HEADS * HD * int(sizeof(E)) / 128;        // 128-byte lines of a batch
    for (int i = lane + LINES * first; i < LINES * last; i += 32) {
        const int x = i / LINES, heads = x < qn ? n_heads : c.n_kv, at = x < qn ? x : x < qn + kn ? x - qn : x - qn - kn;
        const int e = at * APPEND_HEADS * HD + i % LINES * (128 / int(sizeof(E)));
        if (e < heads * HD) prefetch_l2((x < qn ? qr : x < qn + kn ? kr : vr) + e);
    }

    const int s = paged_seq_of_warp(b, r);
    if (s < 0) return;                                       // a row behind the last sequence
    const int pos = paged_pos(b, c, s, r, lane == 0 ? status : nullptr);
    if (pos < 0) return;                                     // padding, or beyond the table
    const int page = last > qn ? paged_page(b, c, s, pos, lane == 0 ? status : nullptr) : -1;
    float cs[2], sn[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const double t = double(pos) * turn[2 * lane + e];
        const double half = 2.0 * (t - rint(t));             // half turns in [-1, 1]
        const float h = float(half), rest = 3.14159265f * float(half - double(h));
        float s0, c0;
        sincospif(h, &s0, &c0);
        sn[e] = fmaf(c0, rest, s0);
        cs[e] = fmaf(-s0, rest, c0);
    }
    auto weighted = [&](const float *n) {
        Turn w;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const float2 f = n ? __ldg(reinterpret_cast<const float2 *>(n) + 32 * y + lane) : make_float2(1.0f, 1.0f);
            w.c[y] = make_float2(f.x * cs[0], f.y * cs[1]);
            w.s[y] = make_float2(f.x * sn[0], f.y * sn[1]);
        }
        return w;
    };
    Turn w = weighted(q_norm);
    for (int x = first; x < min(last, qn); ++x) {
        const int u = x * APPEND_HEADS;
        append_heads<E, QB, true>(qr + u * HD + 2 * lane, n_heads - u, q_norm, eps, w, q_out,
                                  (int64_t(r) * n_heads + u) * HD + 2 * lane, HD);
    }
    if (page < 0) return;                                    // no keys or values here, or a bad page (flagged): none stored
    const int64_t at = paged_at(c, page, 0, pos) + 2 * lane, step = HD << c.page_shift;
    w = weighted(k_norm);
    for (int x = max(first, qn); x < min(last, qn + kn); ++x) {
        const int u = (x - qn) * APPEND_HEADS;
        append_heads<E, CB, true>(kr + u * HD + 2 * lane, c.n_kv - u, k_norm, eps, w, c.k, at + u * step, step);
    }
    for (int x = max(first, qn + kn); x < last; ++x) {
        const int u = (x - qn - kn) * APPEND_HEADS;
        append_heads<E, CB, false>(vr + u * HD + 2 * lane, c.n_kv - u, false, eps, w, c.v, at + u * step, step);
    }
}

cudaError_t launch_kv_append(const PagedKV &c, q3cu_dtype cache_dt, const PagedSeqs &b, int64_t rows, const void *q,
                             const void *k, const void *v, q3cu_dtype dt, int64_t q_stride, int64_t kv_stride,
                             int n_heads, const float *q_norm, const float *k_norm, const TurnFreq &freq, float eps,
                             void *q_out, q3cu_dtype q_dt, uint32_t *status, cudaStream_t stream, int sms) {
    // A row is split over warps only while the rows alone are fewer than 32 warps per SM.
    const int64_t all = (n_heads + APPEND_HEADS - 1) / APPEND_HEADS + (c.n_kv + APPEND_HEADS - 1) / APPEND_HEADS * 2;
    const int64_t batches = all < 65535 ? all : 65535;       // a grid's height
    const int64_t parts = rows >= 32 * sms ? 1 : (32 * int64_t(sms) + rows - 1) / rows;
    const dim3 grid(unsigned((rows + APPEND_WARPS - 1) / APPEND_WARPS), unsigned(parts < batches ? parts : batches));
    auto go = [&](auto kernel, auto *typed) {
        typedef decltype(typed) P;
        return launch_dependent(kernel, grid, dim3(APPEND_WARPS * 32), 0, stream, c, b, int(rows), static_cast<P>(q),
                                static_cast<P>(k), static_cast<P>(v), q_stride, kv_stride, n_heads, q_norm, k_norm, freq,
                                eps, q_out, status);
    };
    const int kind = 2 * (q_dt == Q3CU_BF16) + (cache_dt == Q3CU_BF16);
    if (dt == Q3CU_F32) {
        const float *t = nullptr;
        return kind == 0   ? go(kv_append_kernel<float, false, false>, t)
               : kind == 1 ? go(kv_append_kernel<float, false, true>, t)
               : kind == 2 ? go(kv_append_kernel<float, true, false>, t)
                           : go(kv_append_kernel<float, true, true>, t);
    }
    const uint16_t *t = nullptr;
    return kind == 0   ? go(kv_append_kernel<bf16raw, false, false>, t)
           : kind == 1 ? go(kv_append_kernel<bf16raw, false, true>, t)
           : kind == 2 ? go(kv_append_kernel<bf16raw, true, false>, t)
                       : go(kv_append_kernel<bf16raw, true, true>, t);
}

}  // namespace q3
