// Host checks of the paged cache at its largest sizes, no GPU: the longest table that the entry points take, and the
// arithmetic of the kernels at the lengths that it allows.  Includes the API's source for a context without a device.
#include <algorithm>
#include <climits>
#include <cstdlib>

#include "q3cu_api.cu"
#include "q3cu_paged.cuh"

#define EXPECT(x)                                                   \
    do {                                                            \
        if (!(x)) {                                                 \
            std::printf("line %d: %s (%s)\n", __LINE__, #x, g_err); \
            std::exit(1);                                           \
        }                                                           \
    } while (0)

// Sizes are compared in 64 bits: what a 32-bit sum makes of them must be the same.
static int round_up(int len, int tile) {
    const int64_t want = (int64_t(len) + tile - 1) / tile;
    EXPECT(int64_t(len) + tile - 1 <= INT_MAX && want * tile <= INT_MAX);
    return int(want);
}

int main() {
    q3cu_ctx ctx;
    ctx.alive = true;
    ctx.sms = 148;
    alignas(16) static char m[4096];
    static int32_t ints[64];
    for (int page : {16, 32, 64, 128, 256}) {
        const q3cu_kv_cache cache{m, m, int64_t(2) * page * 128, 4, 2, page, 128, Q3CU_BF16};
        const int most = (INT_MAX - 511) / page;
        for (int pages : {most, most + 1}) {
            // no sequences: nothing is launched where the descriptors are taken
            const q3cu_kv_batch batch{ints, ints, ints, 0, pages};
            const q3cu_status want = pages == most ? Q3CU_OK : Q3CU_ERR_INVALID;
            EXPECT(q3cu_attention_paged(&ctx, &cache, &batch, m, Q3CU_BF16, 512, 4, m, 1 << 30, m + 16, nullptr) == want);
            EXPECT(q3cu_attention_prompt(&ctx, &cache, &batch, 1, m, Q3CU_BF16, 512, 4, m + 16, nullptr) == want);
            EXPECT(q3cu_kv_append(&ctx, &cache, &batch, 1, m, m, m, Q3CU_F32, 512, 256, 4, nullptr, nullptr, 1e6f, 1e-6f, m,
                                  Q3CU_F32, nullptr) == want);
        }
        int shift = 4;
        while ((1 << shift) < page) ++shift;
        const q3::PagedKV c{nullptr, nullptr, int64_t(1) << 20, 4, 2, shift};
        const int longest = most * page;
        for (int32_t len : {longest, longest - 1, longest + 1, INT_MAX}) {
            const int32_t off[2] = {0, 300};
            const q3::PagedSeqs b{off, &len, nullptr, 1, most};
            uint32_t status = 0;
            const q3::PromptSeq s = q3::prompt_seq(b, c, 300, q3::FastDiv(64), 0, &status);
            EXPECT(s.len == std::min(len, longest) && (status != 0) == (len > longest));
            const q3::PromptItem item{0, 0, 256, s.rows, s.len, s.base, s.pos0};
            for (int i : {0, 255, 299}) EXPECT(item.seen(i) == int(std::min<int64_t>(s.len, int64_t(len) - 300 + i + 1)));
            for (int tile : {32, 64, 128}) {
                const int tiles = round_up(s.len, tile);
                EXPECT(s.at_least((tiles - 1) * tile + 1, q3::FastDiv(64)) >= 1 && s.at_least(1, q3::FastDiv(64)) == 5);
            }
        }
    }
    std::printf("ok\n");
    return 0;
}
