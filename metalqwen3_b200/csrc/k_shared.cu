// k_shared.cu -- attention of one new token per sequence where groups of consecutive sequences share their first
// positions: those are attended to once for the whole group.
//
// Query head h of sequence s: o = sum_t softmax_t(q . k_t / sqrt(128)) v_t over its kv_len positions, the first len[g] of
// which lie on the pages of the group's first sequence.  Four launches, joined by the softmax's maxima and sums:
//
//   plan              one CTA: which groups share something, and how the work of the others is cut.  Lengths and groups are
//                     read here and by no launch behind, so that all go by the same ones, whatever the arrays hold.
//   shared positions  the tensor-core kernel of k_prompt.cu (q3cu_prompt.cuh, PT_SHARED) with sequences in the place of
//                     prompt rows: row r of a tile is sequence r / g, head r % g of the g query heads of a kv head, and
//                     all rows see the same keys.  The units are key tiles (128 positions) of (group, kv head, block of
//                     two row tiles), cut into one equal run per SM.
//   own positions     the first kernel of one-token attention (k_paged.cu, k_paged_q8.cu), over positions len[g] and up.
//                     It does not wait for the launch before: its CTAs take the SMs as those finish.
//   join              shared_join_kernel: a warp per (sequence, head) adds the parts,
//                     o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
//
// What the keys cost: read once per block of 256 / g sequences and kv head, from L2 after the first, where one-token
// attention reads them for every sequence.  The probabilities of the shared positions are rounded to bf16, as in prompts
// (over Q8_0 to f16, k_prompt_q8.cu).
//
// Measured: 64 sequences behind 16,384 bf16 positions, 512 of their own (32/8 heads) 56 to 60 us, 150 in three groups behind
// 12,001 Q8_0 ones, up to 1,024 of their own (40/8) 133 to 136 us, five behind 700 (16/8) 16 to 17 us.  Bound by the steps of the
// tensor-core kernel (some 3,600 cycles a key tile for 2,048 of products, over Q8_0 4,200, or 3,800 where a group is one row
// tile), then by the bytes of the own positions (69 and 178 MB in 20 and 49 us), then by latency: set-up some 10 us, the join
// 8.  With the plan made beside the products of the second launch, each CTA searching the groups for itself and the tails
// waiting, 57 to 60, 156 to 160 and 19 us; with the plan in a first launch that all others waited for, 81 us for the 64.
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
    __threadfence();                                         // before the wait: the plan was complete when the launch before began
    const PagedSpan mine = b.span(c, s, nullptr);
    const int64_t tails_before = b.before[s], tails_all = b.before[b.n_seqs], shared_all = sh.plan.all->units;
    const SharedEntry of = sh.plan.of[s];
    const int tiles = mine.tiles<TILE>();
    int tail_n = 0, shared_n = 0, slot = 0;
    PartsOf tail_parts(PagedCut(1, 1), 0, 0, 1), shared_parts = tail_parts;
    if (tiles > 0) {
        const PagedCut cut(tails_all * c.n_kv, tail_runs);
        const int64_t a = tails_before * c.n_kv + int64_t(kv) * (TAIL_LEAD + tiles);
        tail_parts = PartsOf(cut, a, a + TAIL_LEAD, a + TAIL_LEAD + tiles);
        tail_n = tail_parts.n;
    }
    if (mine.from > 0) {
        const PagedCut cut(shared_all * c.n_kv, shared_runs);
        const int keys = (mine.from + PT_KEYS - 1) / PT_KEYS, at = s - of.first, block = per_block(at);
        const int64_t a = of.units * c.n_kv + (int64_t(kv) * (per_block(of.count - 1) + 1) + block) * keys;
        shared_parts = PartsOf(cut, a, a, a + keys);
        shared_n = shared_parts.n;
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
                                                             : int64_t(b.n_seqs) * n_heads + shared_parts.slot(i) * sh.slot_rows + slot + h);
            i -= shared_n;
            return tail_n == 1 ? tails + row * SHARED_ROW
                               : part + (tail_parts.slot(i) * group + h) * SHARED_ROW;
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

// ---- the plan ------------------------------------------------------------------------------------
constexpr int SP_THREADS = 1024;
// Inclusive sums over the CTA of two numbers of each thread; `all_x`, `all_y`: of all.
__device__ __forceinline__ void block_prefix(int64_t &x, int &y, int64_t &all_x, int &all_y) {
    __shared__ int64_t sum_x[32];
    __shared__ int sum_y[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto prefix = [&](int64_t &u, int &v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t pu = __shfl_up_sync(FULL, u, o);
            const int pv = __shfl_up_sync(FULL, v, o);
            if (lane >= o) u += pu, v += pv;
        }
    };
    prefix(x, y);
    __syncthreads();                                         // the sums of a call before are read
    if (lane == 31) sum_x[warp] = x, sum_y[warp] = y;
    __syncthreads();
    int64_t u = sum_x[lane];
    int v = sum_y[lane];
    prefix(u, v);
    all_x = __shfl_sync(FULL, u, 31);
    all_y = __shfl_sync(FULL, v, 31);
    u = __shfl_sync(FULL, u, max(warp - 1, 0));
    v = __shfl_sync(FULL, v, max(warp - 1, 0));
    if (warp) x += u, y += v;
}

// One CTA.  Offsets that do not rise may make groups overlap, or more groups than there is room for: then those that come
// too late, and sequences that find no entry of their own group, share nothing.
__global__ void __launch_bounds__(SP_THREADS)
shared_plan_kernel(const PagedGroups groups, const SharedPlan plan, const PagedKV c, const PagedSeqs b, const FastDiv per_block,
                   int tail_tile, uint32_t *status) {
    __shared__ int off_sh[SP_THREADS + 1];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = int(threadIdx.x), room = shared_entries(b.n_seqs);
    const bool held = groups.n <= SP_THREADS;                // the offsets fit shared memory
    const int my_len = tid < b.n_seqs ? paged_len(b, c, tid, status) : 0;    // on its way meanwhile
    int64_t units = 0;
    int n = 0;
    for (int g0 = 0; g0 < groups.n; g0 += SP_THREADS) {
        const int g = g0 + tid, shared = g < groups.n ? groups.shared(g, b, c, status) : 0;
        if (held && g < groups.n) off_sh[g] = groups.off[g];
        if (held && tid == 0) off_sh[groups.n] = groups.off[groups.n];
        const int count = shared ? groups.count(g, b.n_seqs) : 0;
        int64_t mine = shared ? int64_t((shared + PT_KEYS - 1) / PT_KEYS) * (per_block(count - 1) + 1) : 0, x = mine, all_x;
        int one = shared > 0, y = one, all_y;
        block_prefix(x, y, all_x, all_y);
        const int index = n + y - one;
        if (n + all_y > room) {                              // (the same for all threads)
            if (index >= room) mine = 0, one = 0;
            x = mine, y = one;
            block_prefix(x, y, all_x, all_y);
        }
        if (one) {
            const int first = groups.off[g];
            plan.entries[index] = {first, count, shared, 0, units + x - mine};
            plan.entry[first] = index;
        }
        units += all_x;
        n += all_y;
    }
    if (tid == 0) *plan.all = {0, n, 0, 0, units};
    __syncthreads();
    int64_t sum = 0;
    for (int s0 = 0; s0 < b.n_seqs; s0 += SP_THREADS) {
        const int s = s0 + tid;
        int64_t x = 0, all_x;
        int y = 0, all_y;
        if (s < b.n_seqs) {
            const int len = s0 ? paged_len(b, c, s, status) : my_len;
            int from = 0;
            const PagedGroups near{held ? off_sh : groups.off, groups.len, groups.n};
            const int g = n ? near.of(s, b.n_seqs) : -1;
            if (g >= 0) {
                const int first = near.off[g], count = near.count(g, b.n_seqs), index = count > 1 ? plan.entry[first] : -1;
                if (index >= 0 && index < n) {
                    const SharedEntry e = plan.entries[index];
                    if (e.first == first && e.count == count && len >= e.len) {      // one that holds fewer attends by itself
                        from = e.len;
                        plan.of[s] = e;
                    }
                }
            }
            plan.spans[s] = make_int2(from, len);
            if (len > from) x = TAIL_LEAD + PagedSpan{from, len}.tiles(tail_tile);
        }
        const int64_t mine = x;
        block_prefix(x, y, all_x, all_y);
        if (s < b.n_seqs) plan.before[s] = sum + x - mine;
        sum += all_x;
    }
    if (tid == 0) plan.before[b.n_seqs] = sum;
}

// The workspace: rows of the shared positions, of whole tails, of parts of tails, then the plan.
struct SharedWork {
    size_t tails, part, spans, before, entry, entries, of, bytes;
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
    w.entry = w.before + round((size_t(n_seqs) + 1) * sizeof(int64_t));
    w.entries = w.entry + round(size_t(n_seqs) * sizeof(int));
    w.of = w.entries + round((size_t(shared_entries(n_seqs)) + 1) * sizeof(SharedEntry));       // and one for all
    w.bytes = w.of + round(size_t(n_seqs) * sizeof(SharedEntry));
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
    SharedEntry *entries = reinterpret_cast<SharedEntry *>(base + w.entries);
    const SharedPlan plan{reinterpret_cast<int2 *>(base + w.spans), reinterpret_cast<int64_t *>(base + w.before),
                          reinterpret_cast<int *>(base + w.entry), entries, reinterpret_cast<SharedEntry *>(base + w.of),
                          entries + shared_entries(b.n_seqs)};
    const SharedOut sh{plan, reinterpret_cast<float *>(base), w.slot_rows};
    TailSeqs seqs;
    static_cast<PagedSeqs &>(seqs) = b;
    seqs.spans = plan.spans;
    seqs.before = plan.before;
    const bool q8 = cache_dt == Q3CU_Q8_0;
    const FastDiv per_block(2 * (PT_ROWS / group));
    cudaError_t e = launch_dependent(shared_plan_kernel, dim3(1), dim3(SP_THREADS), 0, stream, PagedGroups{off, len, n_groups},
                                     plan, c, b, per_block, q8 ? PD_TAIL_Q8 : PD_TAIL_BF16, status);
    if (e != cudaSuccess) return e;
    e = q8 ? launch_prefixes<true>(sh, c, b, q, q_stride, n_heads, status, stream, sms)
           : launch_prefixes<false>(sh, c, b, q, q_stride, n_heads, status, stream, sms);
    if (e != cudaSuccess) return e;
    e = (q8 ? launch_tails_q8 : launch_tails_bf16)(c, seqs, q, q_stride, n_heads, part, tails, out, status, stream, runs);
    if (e != cudaSuccess) return e;
    auto *join = q8 ? shared_join_kernel<PD_TAIL_Q8> : shared_join_kernel<PD_TAIL_BF16>;
    return launch_dependent(join, dim3(unsigned(b.n_seqs) * unsigned(c.n_kv)), dim3(SJ_WARPS * 32), 0, stream, sh, c, seqs,
                            per_block, n_heads, group, sms, runs, part, tails, static_cast<uint16_t *>(out));
}

}  // namespace q3
