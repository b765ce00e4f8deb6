// k_prompt_q8.cu -- causal attention of packed prompt rows over a Q8_0 paged cache: the kernel of k_prompt.cu (its header
// has the mathematics, the work items and the warps) with four more warps, which make the operands.
//
// TMA brings a key or value tile's codes and scales, 17 KB, to one of three stages; warps 12-15 turn each into the 32 KB
// operand tile that the tensor cores read, zeros behind the sequence's end (so no warp clears values here).  Three such
// tiles are in flight where a bf16 cache has five; the codes ahead of them make up for it.
//
// The operands are f16: a code times its scale has more than bf16's 8 bits, and rounding keys and values to bf16 doubled the
// error of the result (0.0039 of it against 0.0019 now, of which the result's own rounding is 0.0017).  f16 has 11 bits but little
// range, so everything is lifted by powers of two:
//   keys, values  by tile: the largest scale to [2^14, 2^15), codes as code / 128.  An element is rounded by 2^-10 of itself
//                 (its scale and the product, 2^-11 each) and by no less than 2^-39 of the tile's largest.
//   queries       by row, by the same warps when an item begins; exact, but for 2^-39 of the row's largest.
//   probabilities times 2^7, by 2^-11 of themselves and no less than 2^-32; up to 2^8 lower, so 2^-24, as the next lines say.
// The inverse lifts of query and keys go into the factor that makes scores exponents.  O is kept, row by row, times the lift
// of the tiles that it sees: a tile of larger values takes O down with it (in binary32, on the path that rescales O for a larger
// maximum), a tile of values up to 2^8 smaller has its probabilities lowered, and one of still smaller ones takes O up, as far
// as binary32 goes: what does not fit then is 2^-100 of the row's result.  (Kept times the smallest lift so far, a row lost
// values 2^33 smaller than any before them, though those had no weight.)  A tile that the row does not see leaves O as it is.
// (Where O would go down by more than 2^120 at once, which binary32 may not hold, the row is computed again from the formula.)
// Where the scales of one tile differ by more than 2^24, rows that see only a part of the tile look at the scales again: one that
// has a scale more than 2^24 times the largest it sees behind it in the tile is computed again from the formula, so that a
// later position takes no bits from an earlier row (larger_behind; some 0.2 us a key, a look alone a microsecond).
//
// Bound as k_prompt.cu is, by the chain from scores to probabilities to products, with the conversion beside it: a key tile
// takes 4,200 to 4,400 cycles (3,000 over a bf16 cache) for 2,048 of products and as many of exponentials.  The conversion beside it
// makes the softmax slower, though its 1.75 instructions an element are not the cost (none of them: the same time): the two
// share each quarter's queue for shared memory and special functions, and its store of instructions, for which a smaller
// loop is quicker than one that is unrolled (q8_tile).  2,043 rows in four chunks behind up to 8,192 positions (32/8 heads)
// 229 to 245 us from one GPU to the next, 720 to 770 TFLOP/s; 4,096 rows in six prompts 96 to 98 us; 16 rows behind 8,000 34 us.
// Measured and left out (us for the chunks, against 241 or what it was at the time): scores read twice in two halves, for
// smaller code and fewer registers (244 for 229), a quarter of the exponentials by
// polynomial (275, an eighth 258), eight warps converting (410 for 240: registers), items of 32 rows less with a ring of four
// (320 for 252), lifts by a warp of their own (267 for 247; with the scales in a ring of theirs, far ahead, 281), lifts without
// the comparison where it can be told beforehand (253: what runs earlier is in the softmax's way), codes read before the wait
// for their place (253 for 247), waits that suspend longer or poll less (280, 246).
#include "q3cu_prompt.cuh"

namespace q3 {

cudaError_t launch_prompt_q8(const PagedKV &c, const PagedSeqs &b, int64_t rows, const void *q, int64_t q_stride, int n_heads,
                             void *out, uint32_t *status, cudaStream_t stream) {
    const int group = n_heads / c.n_kv, qt = PT_ROWS / group;
    CUtensorMap mq, mk, mv, mks, mvs;
    if (!encode_prompt_q_map(&mq, q, n_heads, rows, q_stride, group) || !encode_pages_map(&mk, c.k, c, Q3CU_Q8_0, PT_KEYS) ||
        !encode_pages_map(&mv, c.v, c, Q3CU_Q8_0, PT_KEYS) || !encode_scales_map(&mks, c.k_scale, c, PT_KEYS) ||
        !encode_scales_map(&mvs, c.v_scale, c, PT_KEYS))
        return cudaErrorInvalidValue;
    typedef PromptShape<true> Shape;
    const int64_t items = (rows / (2 * qt) + b.n_seqs) * c.n_kv;             // as in k_prompt.cu
    auto *whole = prompt_tc_kernel<PT_ITEMS, true>, *cluster = prompt_tc_kernel<PT_CLUSTER, true>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(cluster), Shape::SMEM, 56);
    if (e == cudaSuccess) e = ensure_smem_attr(reinterpret_cast<const void *>(whole), Shape::SMEM, 57);
    if (e != cudaSuccess) return e;
    const int ctas = prompt_cluster(reinterpret_cast<const void *>(cluster), 2, Shape::THREADS, Shape::SMEM, items,
                                    (int64_t(b.max_pages) << c.page_shift) / PT_KEYS);
    return launch_clusters(ctas > 1 ? cluster : whole, ctas, dim3(unsigned(items * ctas)), dim3(Shape::THREADS), Shape::SMEM,
                           stream, mq, mk, mv, mks, mvs, SharedOut{}, c, b, int(rows), static_cast<const uint16_t *>(q),
                           q_stride, n_heads, group, FastDiv(2 * qt), FastDiv(group), ctas, static_cast<uint16_t *>(out), status);
}

}  // namespace q3
