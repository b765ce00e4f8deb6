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
// APPEND_UNITS heads of one row: lane l holds elements 2l, 2l+1, 64+2l, 65+2l
// of each, so both halves of a rotated pair are in one lane, a half row is one
// contiguous access, and the two angles of a lane serve all its heads.
#include "q3cu_paged.cuh"

namespace q3 {

constexpr int APPEND_UNITS = 4, APPEND_WARPS = 8;

// Coherent loads: q_out may be q itself (a lane reads its elements before it stores them).
__device__ __forceinline__ float2 load_pair(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 load_pair(const uint16_t *p) {
    const uint32_t u = *reinterpret_cast<const uint32_t *>(p);
    return make_float2(bf16_to_f32(u & 0xffffu), bf16_to_f32(u >> 16));
}
__device__ __forceinline__ void store_pair(void *base, int64_t at, bool bf16, float2 v) {
    if (bf16)
        *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(base) + at) = f32_to_bf16(v.x) | (f32_to_bf16(v.y) << 16);
    else
        *reinterpret_cast<float2 *>(static_cast<float *>(base) + at) = v;
}

template <typename T>
__global__ void __launch_bounds__(APPEND_WARPS * 32)
kv_append_kernel(const PagedKV c, const PagedSeqs b, int64_t rows, const typename Elem<T>::type *q,
                 const typename Elem<T>::type *k, const typename Elem<T>::type *v, int64_t q_stride,
                 int64_t kv_stride, int n_heads, const float *__restrict__ q_norm, const float *__restrict__ k_norm,
                 const __grid_constant__ TurnFreq freq, float eps, void *q_out, int q_bf16, int cache_bf16,
                 int groups, uint32_t *status) {
    __shared__ double turn[64];
    if (threadIdx.x < 64) turn[threadIdx.x] = freq.v[threadIdx.x];
    __syncthreads();
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t w = int64_t(blockIdx.x) * APPEND_WARPS + (threadIdx.x >> 5);
    const int64_t r = w / groups;
    const int u0 = int(w % groups) * APPEND_UNITS, units = n_heads + 2 * c.n_kv;
    if (r >= rows) return;
    float2 lo[APPEND_UNITS], hi[APPEND_UNITS];
#pragma unroll
    for (int i = 0; i < APPEND_UNITS; ++i) {
        const int u = u0 + i;
        lo[i] = hi[i] = make_float2(0.0f, 0.0f);
        if (u >= units) continue;
        const typename Elem<T>::type *x = u < n_heads             ? q + r * q_stride + int64_t(u) * HD
                                          : u < n_heads + c.n_kv  ? k + r * kv_stride + int64_t(u - n_heads) * HD
                                                                  : v + r * kv_stride + int64_t(u - n_heads - c.n_kv) * HD;
        lo[i] = load_pair(x + 2 * lane);
        hi[i] = load_pair(x + 64 + 2 * lane);
    }
    // the place, while the loads above are under way
    const int s = paged_seq_of_warp(b, r);
    if (s < 0) return;                                       // a row behind the last sequence
    const int pos = paged_pos(b, c, s, r, lane == 0 ? status : nullptr);
    if (pos < 0) return;                                     // padding, or beyond the table
    int page = -1;
    if (u0 + APPEND_UNITS > n_heads) page = paged_page(b, c, s, pos, lane == 0 ? status : nullptr);
    float cs[2], sn[2];
    if (u0 < n_heads + c.n_kv) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const double t = double(pos) * turn[2 * lane + e];
            const double half = 2.0 * (t - rint(t));         // half turns in [-1, 1]
            const float h = float(half), rest = 3.14159265f * float(half - double(h));
            float s0, c0;
            sincospif(h, &s0, &c0);
            sn[e] = fmaf(c0, rest, s0);
            cs[e] = fmaf(-s0, rest, c0);
        }
    }
    float ss[APPEND_UNITS];
#pragma unroll
    for (int i = 0; i < APPEND_UNITS; ++i)
        ss[i] = fmaf(lo[i].x, lo[i].x, fmaf(lo[i].y, lo[i].y, fmaf(hi[i].x, hi[i].x, hi[i].y * hi[i].y)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < APPEND_UNITS; ++i) ss[i] += __shfl_xor_sync(FULL, ss[i], o);
#pragma unroll
    for (int i = 0; i < APPEND_UNITS; ++i) {
        const int u = u0 + i;
        if (u >= units) break;
        float2 a = lo[i], d = hi[i];
        if (u < n_heads + c.n_kv) {
            const float *wn = u < n_heads ? q_norm : k_norm;
            if (wn) {
                const float g = 1.0f / sqrtf(ss[i] * (1.0f / HD) + eps);
                const float2 w0 = __ldg(reinterpret_cast<const float2 *>(wn) + lane);
                const float2 w1 = __ldg(reinterpret_cast<const float2 *>(wn) + 32 + lane);
                a = make_float2(w0.x * (g * a.x), w0.y * (g * a.y));
                d = make_float2(w1.x * (g * d.x), w1.y * (g * d.y));
            }
            const float2 y = a, z = d;
            a = make_float2(fmaf(y.x, cs[0], -(z.x * sn[0])), fmaf(y.y, cs[1], -(z.y * sn[1])));
            d = make_float2(fmaf(y.x, sn[0], z.x * cs[0]), fmaf(y.y, sn[1], z.y * cs[1]));
        }
        void *base;
        int64_t at;
        bool bf16;
        if (u < n_heads) {
            base = q_out;
            at = (r * n_heads + u) * HD;
            bf16 = q_bf16 != 0;
        } else {
            if (page < 0) continue;                          // flagged above; nothing is stored
            const bool key = u < n_heads + c.n_kv;
            base = key ? c.k : c.v;
            at = paged_at(c, page, u - n_heads - (key ? 0 : c.n_kv), pos);
            bf16 = cache_bf16 != 0;
        }
        store_pair(base, at + 2 * lane, bf16, a);
        store_pair(base, at + 64 + 2 * lane, bf16, d);
    }
}

cudaError_t launch_kv_append(const PagedKV &c, q3cu_dtype cache_dt, const PagedSeqs &b, int64_t rows, const void *q,
                             const void *k, const void *v, q3cu_dtype dt, int64_t q_stride, int64_t kv_stride,
                             int n_heads, const float *q_norm, const float *k_norm, const TurnFreq &freq, float eps,
                             void *q_out, q3cu_dtype q_dt, uint32_t *status, cudaStream_t stream) {
    const int groups = (n_heads + 2 * c.n_kv + APPEND_UNITS - 1) / APPEND_UNITS;
    const int64_t blocks = (rows * groups + APPEND_WARPS - 1) / APPEND_WARPS;
    if (blocks == 0) return cudaSuccess;
    const dim3 grid = dim3(unsigned(blocks)), block = dim3(APPEND_WARPS * 32);
    const int qb = q_dt == Q3CU_BF16, cb = cache_dt == Q3CU_BF16;
    if (dt == Q3CU_F32)
        return launch_dependent(kv_append_kernel<float>, grid, block, 0, stream, c, b, rows,
                                static_cast<const float *>(q), static_cast<const float *>(k),
                                static_cast<const float *>(v), q_stride, kv_stride, n_heads, q_norm, k_norm, freq, eps,
                                q_out, qb, cb, groups, status);
    return launch_dependent(kv_append_kernel<bf16raw>, grid, block, 0, stream, c, b, rows,
                            static_cast<const uint16_t *>(q), static_cast<const uint16_t *>(k),
                            static_cast<const uint16_t *>(v), q_stride, kv_stride, n_heads, q_norm, k_norm, freq, eps,
                            q_out, qb, cb, groups, status);
}

}  // namespace q3
