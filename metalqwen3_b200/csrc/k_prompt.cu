// k_prompt.cu -- causal attention of packed prompt rows over the paged cache.
#include "q3cu_paged.cuh"

namespace q3 {

template <typename T>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const PagedKV c, const PagedSeqs b, int64_t rows,
                                                          const typename Elem<T>::type *q, int64_t q_stride,
                                                          int n_heads, typename Elem<T>::type *out,
                                                          uint32_t *status) {
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int64_t r = w / n_heads;
    const int h = int(w % n_heads);
    if (r >= rows) return;
    const int s = paged_seq_of(b, r);
    if (s < 0) return;
    const int n = paged_seen(b, s, r, paged_len(b, c, s, lane == 0 ? status : nullptr));
    float4 x = load_quad(q + r * q_stride + int64_t(h) * HD + 4 * lane);
    x = make_float4(x.x * ATT_SCALE, x.y * ATT_SCALE, x.z * ATT_SCALE, x.w * ATT_SCALE);
    store_quad(out + w * HD + 4 * lane, attend_row<T>(c, b, s, h / (n_heads / c.n_kv), n, x, status));
}

cudaError_t launch_attention_prompt(const PagedKV &c, const PagedSeqs &b, int64_t rows, const void *q, q3cu_dtype dt,
                                    int64_t q_stride, int n_heads, void *out, uint32_t *status, cudaStream_t stream,
                                    int sms) {
    const dim3 grid(unsigned((rows * n_heads + 3) / 4)), block(128);
    if (dt == Q3CU_F32)
        return launch_dependent(prompt_rows_kernel<float>, grid, block, 0, stream, c, b, rows,
                                static_cast<const float *>(q), q_stride, n_heads, static_cast<float *>(out), status);
    return launch_dependent(prompt_rows_kernel<bf16raw>, grid, block, 0, stream, c, b, rows,
                            static_cast<const uint16_t *>(q), q_stride, n_heads, static_cast<uint16_t *>(out), status);
}

}  // namespace q3
