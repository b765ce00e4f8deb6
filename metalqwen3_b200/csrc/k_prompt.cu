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
// on the other's.  A CTA per SM takes items one after the
// other, its warps each at their own pace, so that one item's first fetches and
// products run beside the last softmax and the stores of the item before:
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
//   warp 9   finds the items, announces them in shared memory, and fetches Q and
//            the key and value tiles of 128 positions, page by page, by TMA into
//            a ring of five 32 KB buffers.
//   warp 10  clears the values behind a sequence's end (below).
// Items go from the longest to the shortest; a CTA that is done with one takes
// over that of a CTA that has not started.
//
// Bound by the tensor cores and what keeps them waiting: a step (128 keys, two
// row tiles) has 2,048 cycles of products and takes 2,990, the time from a tile's
// last probabilities to its next scores and through the softmax, which the other
// tile fills in part.  Over changing inputs a prompt of 16,384 (40/8 heads) takes
// 2.55 ms, 1,078 TFLOP/s, at 1.6 GHz under the power cap; 2,043 rows in chunks behind
// prefixes of up to 8,192 (32/8) 200 us, 880 TFLOP/s; 4,096 rows in six prompts (32/8)
// 54 us.  A replayed graph on one input: 2.15 to 2.3 ms, 175 and 50 us.
// Tensor memory (512 columns): S0, S1, O0, O1; P_t lies over the first half of S_t.
//
// With few items (prompt_tc_kernel<true>) a cluster of up to eight CTAs takes one, each a part of its key tiles, and joins
// the parts through shared memory (join_parts): 16 rows behind 8,000 positions (32/8 heads) 120 -> 28 us, 100 rows
// behind 8,000 138 -> 36 us, 30 behind 30,000 440 -> 62 us.  Up to 64 of 148 SMs work then (8 kv heads).
//
// Masks: keys at and beyond the row's limit become -inf before the maximum.
// Their probability is exactly 0, but 0 times a NaN or an infinity in V is not:
// the values behind the sequence's end (never written, anything may be there) are
// zeroed in shared memory, and a row that comes out with elements that are no
// numbers is computed again from the formula by one warp (attend_row), so that a
// value at a later position of the sequence never reaches an earlier row.  That is
// some hundred times slower than the tile, so it is done only where it may change
// the row (SecondLook): a prompt of 4,096 rows (32/8) takes 0.14 ms, 1.3 with a NaN
// that all rows see, and 24 with one in the last value, which spoils a tile.
//
// Every wait is bounded (2 s; the longest, for the next item, lasts as long as an
// item, some 10 ns a key); a wait that gives up sets Q3CU_DEV_TIMEOUT and the CTA
// drains its own copies and products, frees tensor memory and returns.  So that no
// other warp's wait gives up meanwhile, a warp computes rows again for a second at
// most; past that (32 rows of 170,000 keys) the rest stay NaN, with the same bit set.
#include "q3cu_prompt.cuh"

#include <atomic>

namespace q3 {

bool encode_prompt_q_map(CUtensorMap *map, const void *q, int n_heads, int64_t rows, int64_t q_stride, int group) {
    const uint64_t dims[3] = {HD, uint64_t(n_heads), uint64_t(rows)};
    const uint64_t strides[2] = {HD * 2, uint64_t(q_stride) * 2};
    const uint32_t box[3] = {64, uint32_t(group), uint32_t(PT_ROWS / group)};
    return encode_lines_map(map, q, Q3CU_BF16, 3, dims, strides, box);
}

// The largest cluster of which the GPU holds as many at once as there are items (an SM holds one CTA, and a cluster lies
// within one group of SMs: 15 of 8, 33 of 4, 74 of 2 on a B200).
int prompt_cluster(const void *kernel, int slot, int threads, size_t smem, int64_t items, int64_t tiles) {
    static std::atomic<int> room[64][3][9];                  // clusters of a size that the device holds, plus 1; 0: not asked
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    for (int ctas = 8; ctas > 1; --ctas) {
        if (ctas > tiles / PROMPT_PART) continue;
        int n = room[dev][slot][ctas].load(std::memory_order_relaxed);
        if (n == 0) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(unsigned(ctas));
            cfg.blockDim = dim3(unsigned(threads));
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = unsigned(ctas);
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int held = 0;
            if (cudaOccupancyMaxActiveClusters(&held, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                held = 0;
            }
            room[dev][slot][ctas].store(n = held + 1, std::memory_order_relaxed);
        }
        if (items < n) return ctas;
    }
    return 1;
}

cudaError_t launch_attention_prompt(const PagedKV &c, q3cu_dtype cache_dt, const PagedSeqs &b, int64_t rows, const void *q, q3cu_dtype dt,
                                    int64_t q_stride, int n_heads, void *out, uint32_t *status, cudaStream_t stream,
                                    int sms) {
    if (cache_dt == Q3CU_Q8_0) return launch_prompt_q8(c, b, rows, q, q_stride, n_heads, out, status, stream);
    if (dt == Q3CU_F32) return launch_prompt_f32(c, b, rows, q, q_stride, n_heads, out, status, stream);
    const int group = n_heads / c.n_kv, qt = PT_ROWS / group;
    CUtensorMap mq, mk, mv;
    if (!encode_prompt_q_map(&mq, q, n_heads, rows, q_stride, group) || !encode_pages_map(&mk, c.k, c, Q3CU_BF16, PT_KEYS) ||
        !encode_pages_map(&mv, c.v, c, Q3CU_BF16, PT_KEYS))
        return cudaErrorInvalidValue;
    // no more blocks of 2 * qt queries than this, however the rows are split into sequences
    const int64_t items = (rows / (2 * qt) + b.n_seqs) * c.n_kv;
    typedef PromptShape<false> Shape;
    auto *whole = prompt_tc_kernel<PT_ITEMS, false>, *cluster = prompt_tc_kernel<PT_CLUSTER, false>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(cluster), Shape::SMEM, 43);
    if (e == cudaSuccess) e = ensure_smem_attr(reinterpret_cast<const void *>(whole), Shape::SMEM, 32);
    if (e != cudaSuccess) return e;
    const int ctas = prompt_cluster(reinterpret_cast<const void *>(cluster), 0, Shape::THREADS, Shape::SMEM, items,
                                    (int64_t(b.max_pages) << c.page_shift) / PT_KEYS);
    return launch_clusters(ctas > 1 ? cluster : whole, ctas, dim3(unsigned(items * ctas)), dim3(Shape::THREADS), Shape::SMEM,
                           stream, mq, mk, mv, mk, mv, SharedOut{}, c, b,
                           int(rows), static_cast<const uint16_t *>(q), q_stride, n_heads, group, FastDiv(2 * qt),
                           FastDiv(group), ctas, static_cast<uint16_t *>(out), status);
}

}  // namespace q3
