// k_paged.cu -- attention of one new token per sequence over the paged cache.
#include "q3cu_paged.cuh"

namespace q3 {

template <typename T, typename TC>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedKV c, const PagedSeqs b,
                                                         const typename Elem<T>::type *q, int64_t q_stride,
                                                         int n_heads, typename Elem<T>::type *out, uint32_t *status) {
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int64_t s = w / n_heads;
    const int h = int(w % n_heads);
    if (s >= b.n_seqs) return;
    const int n = paged_len(b, c, int(s), lane == 0 ? status : nullptr);
    float4 x = load_quad(q + s * q_stride + int64_t(h) * HD + 4 * lane);
    x = make_float4(x.x * ATT_SCALE, x.y * ATT_SCALE, x.z * ATT_SCALE, x.w * ATT_SCALE);
    store_quad(out + w * HD + 4 * lane, attend_row<TC>(c, b, int(s), h / (n_heads / c.n_kv), n, x, status));
}

size_t attention_paged_workspace(int n_heads, int n_kv, int sms) { return 16; }

cudaError_t launch_attention_paged(const PagedKV &c, q3cu_dtype cache_dt, const PagedSeqs &b, const void *q,
                                   q3cu_dtype dt, int64_t q_stride, int n_heads, void *work, void *out,
                                   uint32_t *status, cudaStream_t stream, int sms) {
    const dim3 grid(unsigned((int64_t(b.n_seqs) * n_heads + 3) / 4)), block(128);
    auto go = [&](auto kernel, auto *typed) {
        typedef decltype(typed) P;
        return launch_dependent(kernel, grid, block, 0, stream, c, b, static_cast<P>(const_cast<void *>(q)), q_stride,
                                n_heads, static_cast<P>(out), status);
    };
    if (dt == Q3CU_F32)
        return cache_dt == Q3CU_F32 ? go(paged_rows_kernel<float, float>, (float *)nullptr)
                                    : go(paged_rows_kernel<float, bf16raw>, (float *)nullptr);
    return cache_dt == Q3CU_F32 ? go(paged_rows_kernel<bf16raw, float>, (uint16_t *)nullptr)
                                : go(paged_rows_kernel<bf16raw, bf16raw>, (uint16_t *)nullptr);
}

}  // namespace q3
