// Host checks of the paged-cache operators, no GPU: the index arithmetic the kernels share (every table entry and
// cache row it reaches stays inside its array, whatever the lengths, offsets and page ids say) and the entry points'
// refusals (each returns before its first CUDA call).  Includes the API's source for a context without a device.
#include <algorithm>
#include <climits>
#include <cstdlib>
#include <vector>

#include "q3cu_api.cu"
#include "q3cu_paged.cuh"

#define EXPECT(x)                                                   \
    do {                                                            \
        if (!(x)) {                                                 \
            std::printf("line %d: %s (%s)\n", __LINE__, #x, g_err); \
            std::exit(1);                                           \
        }                                                           \
    } while (0)

static uint32_t seed = 12345;
static uint32_t rnd() { return seed = seed * 1664525u + 1013904223u, seed >> 8; }
static int32_t wild() {
    const int32_t pick[] = {0, 1, -1, 7, 15, 16, 17, 100, INT_MAX, INT_MIN, INT_MAX - 3, 1 << 30};
    return rnd() % 2 ? int32_t(rnd() % 300) : pick[rnd() % 12];
}

static void indices() {
    for (int trial = 0; trial < 20000; ++trial) {
        const int n_seqs = rnd() % 6, max_pages = rnd() % 5, shift = 4 + rnd() % 3, n_kv = 1 + rnd() % 3, n_pages = 1 + rnd() % 4;
        const int64_t stride = (int64_t(n_kv) << shift) * 128 + 8 * (rnd() % 3);
        std::vector<int32_t> off(n_seqs + 1), len(n_seqs), table(size_t(n_seqs) * max_pages);
        for (auto &x : off) x = wild();
        for (auto &x : len) x = wild();
        for (auto &x : table) x = wild();
        const q3::PagedKV c{nullptr, nullptr, stride, n_pages, n_kv, shift};
        const q3::PagedSeqs b{off.data(), len.data(), table.data(), n_seqs, max_pages};
        const int64_t r = rnd() % 400;
        const int s = q3::paged_seq_of(b, r);
        EXPECT(s >= -1 && s < n_seqs);
        if (s < 0) continue;
        EXPECT(off[s] <= r && r < off[s + 1]);
        uint32_t status = 0;
        const int keys = q3::paged_len(b, c, s, &status);
        EXPECT(keys >= 0 && keys <= max_pages << shift);
        EXPECT((status != 0) == (len[s] > (max_pages << shift)));
        const int seen = q3::paged_seen(b, s, r, keys);
        EXPECT(seen >= 0 && seen <= keys);
        const int pos = q3::paged_pos(b, c, s, r, &status);
        EXPECT(pos < max_pages << shift);
        for (int t : {pos, seen - 1, 0}) {
            if (t < 0 || t >= max_pages << shift) continue;
            status = 0;
            const int page = q3::paged_page(b, c, s, t, &status);
            const int id = table[size_t(s) * max_pages + (t >> shift)];
            EXPECT(page == (id >= 0 && id < n_pages ? id : -1) && (status != 0) == (page < 0));
            if (page < 0) continue;
            for (int h = 0; h < n_kv; ++h) {
                const int64_t at = q3::paged_at(c, page, h, t);
                EXPECT(at >= 0 && at + 128 <= (n_pages - 1) * stride + (int64_t(n_kv) << shift) * 128);
            }
        }
    }
    const q3::PagedKV big{nullptr, nullptr, int64_t(1) << 36, INT_MAX, 8, 8};
    EXPECT(q3::paged_at(big, INT_MAX - 1, 7, 255) == (int64_t(1) << 36) * (INT_MAX - 1) + (7 * 256 + 255) * 128);
}

// The blocks of prompt rows: divisions by multiplication, and the count of blocks that see a number of keys.
static void blocks() {
    for (int d = 1; d <= 256; ++d) {
        const q3::FastDiv div(d);
        for (int i = 0; i < 2000; ++i) {
            const int q = int(rnd() * 128u % (INT_MAX / d)), n = q * d;
            for (int x : {i, n, n + d - 1, n - 1, INT_MAX - i}) EXPECT(x < 0 || div(x) == x / d);
        }
    }
    for (int trial = 0; trial < 20000; ++trial) {
        const int32_t off[2] = {int32_t(rnd() % 50) - 3, int32_t(rnd() % 700) - 3}, pages = 0;
        const int32_t len = rnd() % 8 ? int32_t(rnd() % 900) : wild();
        const q3::PagedKV c{nullptr, nullptr, 0, 1, 1, 4};
        const q3::PagedSeqs b{off, &len, &pages, 1, int(rnd() % 60)};
        const int total = rnd() % 600;
        const q3::FastDiv per(1 + rnd() % 64);
        const q3::PromptSeq q = q3::prompt_seq(b, c, total, per, 0, nullptr);
        if (off[0] < 0 || off[1] <= off[0] || total <= off[0]) {
            EXPECT(q.blocks == 0 && q.rows == 0);
            continue;
        }
        const int rows = std::min(off[1], total) - off[0];
        EXPECT(q.rows == rows && q.base == off[0] && q.blocks == (rows + per.d - 1) / per.d);
        EXPECT(q.len >= 0 && q.len <= 16 * b.max_pages && (len < 0 || q.pos0 == len - rows));
        const q3::PromptItem item{0, 0, 0, q.rows, q.len, q.base, q.pos0};
        for (int i = 0; i < rows; ++i) {
            const int64_t pos = int64_t(len < 0 ? 0 : len) - rows + i;
            EXPECT(item.seen(i) == int(std::max<int64_t>(0, std::min<int64_t>(q.len, pos + 1))));
        }
        for (int keys : {0, 1, 16, 17, 128, 129, q.len, q.len + 1, 700}) {
            int n = 0;
            for (int i = 0; i < q.blocks; ++i) n += item.seen(std::min((i + 1) * per.d, rows) - 1) >= keys;
            EXPECT(q.at_least(keys, per) == n);
        }
    }
}

static void refusals() {
    q3cu_ctx ctx;
    ctx.alive = true;
    ctx.sms = 148;
    alignas(16) static char m[4096];
    static int32_t ints[64];
    const q3cu_kv_cache good{m, m, 2 * 16 * 128, 4, 2, 16, 128, Q3CU_BF16};
    const q3cu_kv_batch batch{ints, ints, ints, 1, 2};
    auto append = [&](const q3cu_kv_cache *c, const q3cu_kv_batch *b, int64_t rows, const void *q, const void *k,
                      int64_t qs, int64_t ks, int heads, float theta, void *out, int odt) {
        return q3cu_kv_append(&ctx, c, b, rows, q, k, m, Q3CU_F32, qs, ks, heads, nullptr, nullptr, theta, 1e-6f, out,
                              q3cu_dtype(odt), nullptr);
    };
    auto paged = [&](const q3cu_kv_cache *c, const q3cu_kv_batch *b, int heads, size_t work, void *out) {
        return q3cu_attention_paged(&ctx, c, b, m, Q3CU_BF16, heads * 128, heads, m, work, out, nullptr);
    };
    auto prompt = [&](const q3cu_kv_cache *c, const q3cu_kv_batch *b, int64_t rows, int dt, int heads) {
        return q3cu_attention_prompt(&ctx, c, b, rows, m, q3cu_dtype(dt), heads * 128, heads, m + 16, nullptr);
    };
    const size_t plenty = size_t(1) << 40;
    auto each = [&](const q3cu_kv_cache *c, const q3cu_kv_batch *b, q3cu_status st) {
        EXPECT(append(c, b, 1, m, m, 512, 256, 4, 1e6f, m, Q3CU_F32) == st);
        EXPECT(paged(c, b, 4, plenty, m + 16) == st);
        EXPECT(prompt(c, b, 1, Q3CU_BF16, 4) == st);
    };
    each(nullptr, &batch, Q3CU_ERR_INVALID);
    each(&good, nullptr, Q3CU_ERR_INVALID);
    auto cache_with = [&](auto change, q3cu_status st) {
        q3cu_kv_cache c = good;
        change(c);
        each(&c, &batch, st);
    };
    cache_with([](auto &c) { c.k = nullptr; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.v = m + 8; }, Q3CU_ERR_ALIGN);
    cache_with([](auto &c) { c.page_size = 8; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.page_size = 48; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.page_size = 512; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.page_size = 0; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.page_size = INT_MIN; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.head_dim = 64; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.n_kv = 0; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.n_kv = INT_MAX; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.n_pages = 0; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.dtype = 2; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.page_stride = 4095; }, Q3CU_ERR_INVALID);
    cache_with([](auto &c) { c.page_stride = 4097; }, Q3CU_ERR_ALIGN);
    cache_with([](auto &c) { c.page_stride = int64_t(1) << 40; }, Q3CU_ERR_INVALID);
    auto batch_with = [&](auto change, q3cu_status st) {
        q3cu_kv_batch b = batch;
        change(b);
        each(&good, &b, st);
    };
    batch_with([](auto &b) { b.n_seqs = -1; }, Q3CU_ERR_INVALID);
    batch_with([](auto &b) { b.max_pages = -1; }, Q3CU_ERR_INVALID);
    batch_with([](auto &b) { b.max_pages = 1 << 27; }, Q3CU_ERR_INVALID);
    batch_with([](auto &b) { b.kv_len = nullptr; }, Q3CU_ERR_INVALID);
    batch_with([](auto &b) { b.pages = nullptr; }, Q3CU_ERR_INVALID);
    batch_with([](auto &b) { b.pages = reinterpret_cast<int32_t *>(m + 2); }, Q3CU_ERR_ALIGN);
    batch_with([](auto &b) { b.n_seqs = 0; }, Q3CU_OK);

    q3cu_kv_batch no_rows = batch;
    no_rows.row_off = nullptr;
    EXPECT(append(&good, &no_rows, 1, m, m, 512, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);
    EXPECT(prompt(&good, &no_rows, 1, Q3CU_BF16, 4) == Q3CU_ERR_INVALID);
    EXPECT(append(&good, &batch, 0, nullptr, nullptr, 0, 0, 0, 1e6f, nullptr, Q3CU_F32) == Q3CU_OK);
    EXPECT(append(&good, &batch, -1, m, m, 512, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);
    EXPECT(append(&good, &batch, INT_MAX, m, m, 512, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);
    EXPECT(append(&good, &batch, 1, nullptr, m, 512, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);
    EXPECT(append(&good, &batch, 1, m, nullptr, 512, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);
    EXPECT(append(&good, &batch, 1, m + 16, m, 511, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);
    EXPECT(append(&good, &batch, 1, m + 16, m, 513, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_ALIGN);
    EXPECT(append(&good, &batch, 1, m + 16, m, 512, 255, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);
    EXPECT(append(&good, &batch, 1, m + 4, m, 512, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_ALIGN);
    EXPECT(append(&good, &batch, 1, m, m, 516, 256, 4, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);    // in place, not dense
    EXPECT(append(&good, &batch, 1, m, m, 512, 256, 4, 1e6f, m, Q3CU_BF16) == Q3CU_ERR_INVALID);   // in place, other type
    EXPECT(append(&good, &batch, 1, m, m, 512, 256, 4, 1e6f, m, 7) == Q3CU_ERR_INVALID);
    for (float theta : {0.0f, -1.0f, NAN, INFINITY})
        EXPECT(append(&good, &batch, 1, m, m, 512, 256, 4, theta, m, Q3CU_F32) == Q3CU_ERR_INVALID);
    for (int heads : {3, 34, -2}) {
        EXPECT(append(&good, &batch, 1, m, m, 512, 256, heads, 1e6f, m, Q3CU_F32) == Q3CU_ERR_INVALID);
        EXPECT(paged(&good, &batch, heads, plenty, m + 16) == Q3CU_ERR_INVALID);
        EXPECT(prompt(&good, &batch, 1, Q3CU_BF16, heads) == Q3CU_ERR_INVALID);
    }
    EXPECT(paged(&good, &batch, 0, plenty, m + 16) == Q3CU_ERR_INVALID);
    EXPECT(paged(&good, &batch, 4, plenty, nullptr) == Q3CU_ERR_INVALID);
    EXPECT(paged(&good, &batch, 4, plenty, m) == Q3CU_ERR_INVALID);                                // out is q
    EXPECT(paged(&good, &batch, 4, plenty, m + 8) == Q3CU_ERR_ALIGN);
    size_t need = 0;
    EXPECT(q3cu_attention_paged_workspace(&ctx, 4, 2, &need) == Q3CU_OK && need > 0);
    EXPECT(paged(&good, &batch, 4, need - 1, m + 16) == Q3CU_ERR_INVALID);
    EXPECT(q3cu_attention_paged_workspace(&ctx, 5, 2, &need) == Q3CU_ERR_INVALID);
    EXPECT(q3cu_attention_paged_workspace(&ctx, 4, 2, nullptr) == Q3CU_ERR_INVALID);
    EXPECT(prompt(&good, &batch, 1, Q3CU_F32, 4) == Q3CU_ERR_INVALID);
    EXPECT(prompt(&good, &batch, -1, Q3CU_BF16, 4) == Q3CU_ERR_INVALID);
    EXPECT(prompt(&good, &batch, INT_MAX, Q3CU_BF16, 4) == Q3CU_ERR_INVALID);
    EXPECT(prompt(&good, &batch, 0, Q3CU_BF16, 4) == Q3CU_OK);
    EXPECT(q3cu_kv_append(nullptr, &good, &batch, 1, m, m, m, Q3CU_F32, 512, 256, 4, nullptr, nullptr, 1e6f, 1e-6f, m,
                          Q3CU_F32, nullptr) == Q3CU_ERR_NOT_INIT);
    EXPECT(q3cu_attention_paged(nullptr, &good, &batch, m, Q3CU_BF16, 512, 4, m, 16, m, nullptr) == Q3CU_ERR_NOT_INIT);
    EXPECT(q3cu_attention_prompt(nullptr, &good, &batch, 1, m, Q3CU_BF16, 512, 4, m, nullptr) == Q3CU_ERR_NOT_INIT);
    EXPECT(q3cu_attention_paged_workspace(nullptr, 4, 2, &need) == Q3CU_ERR_NOT_INIT);
}

// The parts of a shared item cover its key tiles once, in order, none of fewer tiles than a part may have.
static void parts() {
    for (int ctas = 1; ctas <= 8; ++ctas)
        for (int tiles : {0, 1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 63, 64, 1000, 1 << 24, INT_MAX / 64})
            for (int least : {4, 8}) {
                const int n = q3::prompt_parts(ctas, tiles, least);
                EXPECT(n >= 1 && n <= ctas && (tiles >= least || n == 1));
                EXPECT(q3::prompt_part(tiles, n, 0) == 0 && q3::prompt_part(tiles, n, n) == tiles);
                for (int p = 0; p < n && n > 1; ++p)
                    EXPECT(q3::prompt_part(tiles, n, p + 1) - q3::prompt_part(tiles, n, p) >= q3::PROMPT_PART);
            }
}

int main() {
    indices();
    blocks();
    parts();
    refusals();
    std::printf("ok\n");
    return 0;
}
