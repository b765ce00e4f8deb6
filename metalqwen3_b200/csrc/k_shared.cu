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

constexpr int SJ_WARPS = 4;
// What the join of (sequence s, kv head) reads, found by one warp.
struct JoinPlan {
    int shared_first, shared_n;      // runs that have a part of the shared positions
    int tail_first, tail_n;
    int slot;                        // this sequence's first row in a slot of the shared results
    bool skip, shared_late, tail_late;       // part 0 is the second of its run
};

template <int TILE>
__global__ void __launch_bounds__(SJ_WARPS * 32)
shared_join_kernel(const SharedOut sh, const PagedKV c, const TailSeqs b, const FastDiv per_block, int n_heads, int group,
                   int shared_runs, int tail_runs, const float *part, const float *tails, uint16_t *out) {
    __shared__ JoinPlan plan_sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int s = int(blockIdx.x / unsigned(c.n_kv)), kv = int(blockIdx.x % unsigned(c.n_kv));
    // before the wait: lengths and tables are older than the launches before this one
    if (warp == 0) {
        JoinPlan p = {};
        const PagedSpan mine = b.span(c, s, nullptr);
        int64_t total = 0, before = 0;                       // tiles of the tails, of one kv head
        for (int s0 = 0; s0 < b.n_seqs; s0 += 32) {
            const int n = s0 + lane < b.n_seqs ? b.span(c, s0 + lane, nullptr).tiles<TILE>() : 0;
            const uint32_t end = warp_prefix(uint32_t(n));
            if (s >= s0 && s < s0 + 32) before = total + __shfl_sync(FULL, end - uint32_t(n), s - s0);
            total += __shfl_sync(FULL, end, 31);
        }
        const int tiles = mine.tiles<TILE>();
        if (tiles > 0) {
            const PagedCut cut(total * c.n_kv, tail_runs);
            const int64_t a = before * c.n_kv + int64_t(kv) * tiles;
            p.tail_first = cut.run_of(a);
            p.tail_n = cut.run_of(a + tiles - 1) - p.tail_first + 1;
            p.tail_late = a != cut.begin(p.tail_first);
        }
        if (mine.from > 0) {
            const int g = b.groups.of(s, b.n_seqs), at = s - b.groups.off[g];
            int64_t first;
            const PagedCut cut(shared_units(sh, b, c, per_block, g, first, nullptr) * c.n_kv, shared_runs);
            const int keys = (mine.from + PT_KEYS - 1) / PT_KEYS, block = per_block(at);
            const int blocks = per_block(b.groups.count(g, b.n_seqs) - 1) + 1;
            const int64_t a = first * c.n_kv + (int64_t(kv) * blocks + block) * keys;
            p.shared_first = cut.run_of(a);
            p.shared_n = cut.run_of(a + keys - 1) - p.shared_first + 1;
            p.shared_late = a != cut.begin(p.shared_first);
            p.slot = (at - block * per_block.d) * group;
        }
        // nothing to do: no positions, or all of them written by the kernel before
        p.skip = p.shared_n == 0 && p.tail_n <= 1;
        if (lane == 0) plan_sh = p;
    }
    __syncthreads();
    griddep_wait();
    const JoinPlan p = plan_sh;
    if (p.skip) return;
    const int64_t rows = int64_t(b.n_seqs) * n_heads;
    const int n = p.shared_n + p.tail_n;
    for (int h = warp; h < group; h += SJ_WARPS) {
        const int64_t row = int64_t(s) * n_heads + kv * group + h;
        auto shared_row = [&](int i) {                       // part i < shared_n
            return p.shared_n == 1 ? row
                                   : rows + (2 * int64_t(p.shared_first + i) + (i == 0 && p.shared_late)) * sh.slot_rows + p.slot + h;
        };
        auto tail_part = [&](int i) -> const float * {       // part i < tail_n
            return p.tail_n == 1 ? tails + row * PD_PART
                                 : part + ((2 * int64_t(p.tail_first + i) + (i == 0 && p.tail_late)) * group + h) * PD_PART;
        };
        auto stat = [&](int i) -> float2 {
            if (i < p.shared_n) return sh.stat[shared_row(i)];
            const float *t = tail_part(i - p.shared_n);
            return make_float2(t[HD], t[HD + 1]);
        };
        float m = -INFINITY;
        for (int i = lane; i < n; i += 32) m = fmaxf(m, stat(i).x);
        m = warp_max(m);
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i0 = 0; i0 < n; i0 += 32) {
            float w = 0.0f;
            if (i0 + lane < n) {
                const float2 x = stat(i0 + lane);
                w = x.x == m ? 1.0f : ex2_approx_ftz((x.x - m) * PD_LOG2);
                l = fmaf(x.y, w, l);
            }
            const int end = min(32, n - i0);
#pragma unroll 4
            for (int i = 0; i < end; ++i) {
                const float f = __shfl_sync(FULL, w, i);
                float4 v;
                if (i0 + i < p.shared_n) {
                    v = *reinterpret_cast<const float4 *>(sh.o + shared_row(i0 + i) * HD + 4 * lane);
                } else {
                    const float2 *t = reinterpret_cast<const float2 *>(tail_part(i0 + i - p.shared_n) + 4 * lane);
                    const float2 a = t[0], d = t[1];
                    v = make_float4(a.x, a.y, d.x, d.y);
                }
                o = make_float4(fmaf(f, v.x, o.x), fmaf(f, v.y, o.y), fmaf(f, v.z, o.z), fmaf(f, v.w, o.w));
            }
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(FULL, l, x);
        const float r = 1.0f / l;
        store_quad(out + row * HD + 4 * lane, make_float4(o.x * r, o.y * r, o.z * r, o.w * r));
    }
}

// The workspace: results of the shared positions and their maxima and sums, whole tails, parts of tails.
struct SharedWork {
    size_t stat, tails, part, bytes;
    int slot_rows;
};
static SharedWork shared_work(int n_seqs, int n_heads, int n_kv, int sms) {
    auto round = [](size_t x) { return (x + 255) / 256 * 256; };
    const int group = n_heads / n_kv, block = 2 * (PT_ROWS / group);
    SharedWork w;
    w.slot_rows = (n_seqs < block ? n_seqs : block) * group;
    const size_t rows = size_t(n_seqs) * n_heads, all = rows + size_t(2) * sms * w.slot_rows;
    w.stat = round(all * HD * sizeof(float));
    w.tails = w.stat + round(all * sizeof(float2));
    w.part = w.tails + round(rows * PD_PART * sizeof(float));
    w.bytes = w.part + size_t(paged_runs(sms)) * 2 * group * PD_PART * sizeof(float);
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
    const PagedGroups groups{off, len, n_groups};
    const SharedOut sh{groups, reinterpret_cast<float *>(base), reinterpret_cast<float2 *>(base + w.stat), w.slot_rows};
    TailSeqs seqs;
    static_cast<PagedSeqs &>(seqs) = b;
    seqs.groups = groups;
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
