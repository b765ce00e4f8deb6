// k_shared.cu -- attention of one new token per sequence where groups of consecutive sequences share their first
// positions: those are attended to once for the whole group.
//
// Query head h of sequence s: o = sum_t softmax_t(q . k_t / sqrt(128)) v_t over its kv_len positions, the first len[g] of
// which lie on the pages of the group's first sequence.  Three launches, joined by the softmax's maxima and sums:
//
//   shared positions  the tensor-core kernel of k_prompt.cu (q3cu_prompt.cuh, PT_SHARED) with sequences in the place of
//                     prompt rows: row r of a tile is sequence r / g, head r % g of the g query heads of a kv head, and
//                     all rows see the same keys.  The units are key tiles (128 positions) of (group, kv head, block of
//                     two row tiles), cut into one equal run per SM.
//   own positions     the first kernel of one-token attention (k_paged.cu, k_paged_q8.cu), over positions len[g] and up.
//   join              shared_join_kernel: a warp per (sequence, head) adds the parts,
//                     o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
//
// What the keys cost: read once per block of 256 / g sequences and kv head, from L2 after the first, where one-token
// attention reads them for every sequence.  The probabilities of the shared positions are rounded to bf16, as in prompts.
#include "q3cu_prompt.cuh"

namespace q3 {

constexpr int SJ_WARPS = 4, SJ_PARTS = 8;                    // parts of a row under way at a time

// One CTA per (sequence, kv head), one warp per query head of the group at a time.
template <int TILE>
__global__ void __launch_bounds__(SJ_WARPS * 32)
shared_join_kernel(const SharedOut sh, const PagedKV c, const TailSeqs b, const FastDiv per_block, int n_heads, int group,
                   int shared_runs, int tail_runs, const float *part, const float *tails, uint16_t *out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int s = int(blockIdx.x / unsigned(c.n_kv)), kv = int(blockIdx.x % unsigned(c.n_kv));
    // Before the wait: the plan is older than the launch before this one, which has begun.  Runs are kept within what the
    // workspace holds, whatever the plan says.
    const PagedSpan mine = b.span(c, s, nullptr);
    const int64_t tails_before = b.before[s], tails_all = b.before[b.n_seqs], shared_all = sh.group[b.n_seqs].units;
    const SharedGroup of = sh.group[s];
    const int tiles = mine.tiles<TILE>();
    int tail_first = 0, tail_n = 0, shared_first = 0, shared_n = 0, slot = 0;
    bool tail_late = false, shared_late = false;             // part 0 is the second of its run
    if (tiles > 0) {
        const PagedCut cut(tails_all * c.n_kv, tail_runs);
        const int64_t a = tails_before * c.n_kv + int64_t(kv) * (TAIL_LEAD + tiles);
        tail_first = cut.run_of(a + TAIL_LEAD);
        tail_n = cut.run_of(a + TAIL_LEAD + tiles - 1) - tail_first + 1;
        tail_late = a > cut.begin(tail_first);
    }
    if (mine.from > 0) {
        const PagedCut cut(shared_all * c.n_kv, shared_runs);
        const int keys = (mine.from + PT_KEYS - 1) / PT_KEYS, at = s - of.first, block = per_block(at);
        const int64_t a = of.units * c.n_kv + (int64_t(kv) * (per_block(of.count - 1) + 1) + block) * keys;
        shared_first = min(max(cut.run_of(a), 0), shared_runs - 1);
        shared_n = min(max(cut.run_of(a + keys - 1), shared_first), shared_runs - 1) - shared_first + 1;
        shared_late = a > cut.begin(shared_first);
        slot = (at - block * per_block.d) * group;
    }
    griddep_wait();
    const int n = shared_n + tail_n;
    if (shared_n == 0 && tail_n <= 1) return;                // no positions, or all of them written by the launch before
    for (int h = warp; h < group; h += SJ_WARPS) {
        const int64_t row = int64_t(s) * n_heads + kv * group + h;
        auto at = [&](int i) -> const float * {              // part i: 128 elements, maximum, sum
            if (i < shared_n)
                return sh.rows + SHARED_ROW * (shared_n == 1 ? row
                                                             : int64_t(b.n_seqs) * n_heads +
                                                                   (2 * int64_t(shared_first + i) + (i == 0 && shared_late)) * sh.slot_rows + slot + h);
            i -= shared_n;
            return tail_n == 1 ? tails + row * SHARED_ROW
                               : part + ((2 * int64_t(tail_first + i) + (i == 0 && tail_late)) * group + h) * SHARED_ROW;
        };
        float m = -INFINITY;
        for (int i = lane; i < n; i += 32) m = fmaxf(m, at(i)[HD]);
        m = warp_max(m);
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i0 = 0; i0 < n; i0 += 32) {
            const float *mine_at = at(min(i0 + lane, n - 1));
            float w = 0.0f;
            if (i0 + lane < n) {
                const float2 x = *reinterpret_cast<const float2 *>(mine_at + HD);
                w = x.x == m ? 1.0f : ex2_approx_ftz((x.x - m) * PD_LOG2);
                l = fmaf(x.y, w, l);
            }
            const int end = min(32, n - i0);
            for (int i = 0; i < end; i += SJ_PARTS) {
                float4 v[SJ_PARTS];
#pragma unroll
                for (int k = 0; k < SJ_PARTS; ++k) {
                    const float *p = reinterpret_cast<const float *>(__shfl_sync(FULL, reinterpret_cast<uint64_t>(mine_at), min(i + k, 31)));
                    v[k] = i + k < end ? *reinterpret_cast<const float4 *>(p + 4 * lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
#pragma unroll
                for (int k = 0; k < SJ_PARTS; ++k) {
                    const float f = __shfl_sync(FULL, w, min(i + k, 31));
                    if (i + k < end)
                        o = make_float4(fmaf(f, v[k].x, o.x), fmaf(f, v[k].y, o.y), fmaf(f, v[k].z, o.z), fmaf(f, v[k].w, o.w));
                }
            }
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(FULL, l, x);
        const float r = 1.0f / l;
        store_quad(out + row * HD + 4 * lane, make_float4(o.x * r, o.y * r, o.z * r, o.w * r));
    }
}

// The workspace: rows of the shared positions, of whole tails, of parts of tails, then the plan.
struct SharedWork {
    size_t tails, part, spans, before, group, bytes;
    int slot_rows;
};
static SharedWork shared_work(int n_seqs, int n_heads, int n_kv, int sms) {
    auto round = [](size_t x) { return (x + 255) / 256 * 256; };
    const int group = n_heads / n_kv, block = 2 * (PT_ROWS / group);
    const size_t row = SHARED_ROW * sizeof(float), rows = size_t(n_seqs) * n_heads;
    SharedWork w;
    w.slot_rows = (n_seqs < block ? n_seqs : block) * group;
    w.tails = round((rows + size_t(2) * sms * w.slot_rows) * row);
    w.part = w.tails + round(rows * row);
    w.spans = w.part + round(size_t(paged_runs(sms)) * 2 * group * row);
    w.before = w.spans + round(size_t(n_seqs) * sizeof(int2));
    w.group = w.before + round((size_t(n_seqs) + 1) * sizeof(int64_t));
    w.bytes = w.group + round((size_t(n_seqs) + 1) * sizeof(SharedGroup));
    return w;
}
size_t attention_shared_workspace(int n_seqs, int n_heads, int n_kv, int sms) {
    return shared_work(n_seqs, n_heads, n_kv, sms).bytes;
}

template <bool Q8>
static cudaError_t launch_prefixes(const SharedOut &sh, const PagedKV &c, const PagedSeqs &b, const void *q, int64_t q_stride,
                                   int n_heads, uint32_t *status, cudaStream_t stream, int sms) {
    typedef PromptShape<Q8> Shape;
    const int group = n_heads / c.n_kv, qt = PT_ROWS / group;
    const q3cu_dtype dt = Q8 ? Q3CU_Q8_0 : Q3CU_BF16;
    CUtensorMap mq, mk, mv, mks, mvs;
    if (!encode_prompt_q_map(&mq, q, n_heads, b.n_seqs, q_stride, group) || !encode_pages_map(&mk, c.k, c, dt, PT_KEYS) ||
        !encode_pages_map(&mv, c.v, c, dt, PT_KEYS))
        return cudaErrorInvalidValue;
    mks = mk, mvs = mv;
    if (Q8 && (!encode_scales_map(&mks, c.k_scale, c, PT_KEYS) || !encode_scales_map(&mvs, c.v_scale, c, PT_KEYS)))
        return cudaErrorInvalidValue;
    auto *kernel = prompt_tc_kernel<PT_SHARED, Q8>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(kernel), Shape::SMEM, 58 + Q8);
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, dim3(sms), dim3(Shape::THREADS), Shape::SMEM, stream, mq, mk, mv, mks, mvs, sh, c, b,
                            b.n_seqs, static_cast<const uint16_t *>(q), q_stride, n_heads, group, FastDiv(2 * qt),
                            FastDiv(group), 1, static_cast<uint16_t *>(nullptr), status);
}

cudaError_t launch_attention_shared(const PagedKV &c, q3cu_dtype cache_dt, const PagedSeqs &b, const int32_t *off,
                                    const int32_t *len, int n_groups, const void *q, int64_t q_stride, int n_heads,
                                    void *work, void *out, uint32_t *status, cudaStream_t stream, int sms) {
    const int group = n_heads / c.n_kv, runs = paged_runs(sms);
    const SharedWork w = shared_work(b.n_seqs, n_heads, c.n_kv, sms);
    uint8_t *base = static_cast<uint8_t *>(work);
    float *tails = reinterpret_cast<float *>(base + w.tails), *part = reinterpret_cast<float *>(base + w.part);
    if (n_groups == 0)                                       // (its parts fit where those of the tails would lie)
        return launch_attention_paged(c, cache_dt, b, q, Q3CU_BF16, q_stride, n_heads, part, out, status, stream, sms);
    const SharedOut sh{PagedGroups{off, len, n_groups},
                       reinterpret_cast<float *>(base),
                       w.slot_rows,
                       reinterpret_cast<int2 *>(base + w.spans),
                       reinterpret_cast<int64_t *>(base + w.before),
                       reinterpret_cast<SharedGroup *>(base + w.group),
                       cache_dt == Q3CU_Q8_0 ? PD_TAIL_Q8 : PD_TAIL_BF16};
    TailSeqs seqs;
    static_cast<PagedSeqs &>(seqs) = b;
    seqs.spans = sh.spans;
    seqs.before = sh.before;
    const bool q8 = cache_dt == Q3CU_Q8_0;
    cudaError_t e = q8 ? launch_prefixes<true>(sh, c, b, q, q_stride, n_heads, status, stream, sms)
                       : launch_prefixes<false>(sh, c, b, q, q_stride, n_heads, status, stream, sms);
    if (e != cudaSuccess) return e;
    e = (q8 ? launch_tails_q8 : launch_tails_bf16)(c, seqs, q, q_stride, n_heads, part, tails, out, status, stream, runs);
    if (e != cudaSuccess) return e;
    auto *join = q8 ? shared_join_kernel<PD_TAIL_Q8> : shared_join_kernel<PD_TAIL_BF16>;
    return launch_dependent(join, dim3(unsigned(b.n_seqs) * unsigned(c.n_kv)), dim3(SJ_WARPS * 32), 0, stream, sh, c, seqs,
                            FastDiv(2 * (PT_ROWS / group)), n_heads, group, sms, runs, part, tails, static_cast<uint16_t *>(out));
}

}  // namespace q3
