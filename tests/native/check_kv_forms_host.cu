// Host checks of the paged cache's further forms, no GPU: rotations' frequencies, the groups of sequences that share a
// prefix (whatever their arrays say), the places of a Q8_0 cache's scales, and the entry points' refusals (each returns
// before its first CUDA call).  Includes the API's source for a context without a device.
#include <algorithm>
#include <climits>
#include <cstdlib>
#include <vector>

#include "q3cu_api.cu"
#include "q3cu_paged.cuh"
#include "q3cu_split.cuh"

#define EXPECT(x)                                                   \
    do {                                                            \
        if (!(x)) {                                                 \
            std::printf("line %d: %s (%s)\n", __LINE__, #x, g_err); \
            std::exit(1);                                           \
        }                                                           \
    } while (0)

static uint32_t seed = 4321;
static uint32_t rnd() { return seed = seed * 1664525u + 1013904223u, seed >> 8; }
static int32_t wild() {
    const int32_t pick[] = {0, 1, -1, 7, 15, 16, 17, 100, INT_MAX, INT_MIN, INT_MAX - 3, 1 << 30};
    return rnd() % 2 ? int32_t(rnd() % 12) : pick[rnd() % 12];
}

static void groups() {
    for (int trial = 0; trial < 200000; ++trial) {
        const int n_seqs = 1 + rnd() % 8, n = rnd() % 5, shift = 4 + rnd() % 5, max_pages = rnd() % 4;
        std::vector<int32_t> off(n + 1), len(n), kv_len(n_seqs), table(size_t(n_seqs) * max_pages);
        if (trial % 2)
            for (auto &x : off) x = wild();
        else {                                               // as they should be
            for (auto &x : off) x = rnd() % (n_seqs + 1);
            std::sort(off.begin(), off.end());
        }
        for (auto &x : len) x = wild();
        const q3::PagedKV c{nullptr, nullptr, 1 << 20, 3, 1, shift};
        const q3::PagedSeqs b{nullptr, kv_len.data(), table.data(), n_seqs, max_pages};
        const q3::PagedGroups g{off.data(), len.data(), n};
        const int64_t cap = int64_t(max_pages) << shift;
        for (int i = 0; i < n; ++i) {
            uint32_t status = 0;
            const int count = g.count(i, n_seqs), shared = g.shared(i, b, c, &status);
            EXPECT(count >= 0 && count <= n_seqs && (count == 0 || (off[i] >= 0 && off[i] + count <= n_seqs)));
            EXPECT(shared >= 0 && shared <= cap && (shared == 0 || count > 1));
            EXPECT((status != 0) == (count > 1 && len[i] > cap));
        }
        for (int s = 0; s < n_seqs; ++s) {
            const int of = g.of(s, n_seqs);
            EXPECT(of >= -1 && of < n);
            if (of >= 0) EXPECT(off[of] <= s && s < off[of + 1] && off[of] >= 0 && off[of + 1] <= n_seqs);
            int want = -1;
            for (int i = 0; i < n; ++i)
                if (off[i] <= s && s < off[i + 1]) want = i;
            if (trial % 2 == 0) EXPECT(of == want);
        }
    }
}

static void scales() {
    for (int trial = 0; trial < 20000; ++trial) {
        const int shift = 4 + rnd() % 5, n_kv = 1 + rnd() % 9, n_pages = 1 + rnd() % 5;
        const int64_t dense = (int64_t(n_kv) << shift) * 2, stride = dense + 4 * (rnd() % 3);
        const q3::PagedKV c{nullptr, nullptr, 1 << 20, n_pages, n_kv, shift, nullptr, nullptr, stride};
        const int page = rnd() % n_pages, head = rnd() % n_kv, t = rnd() % 100000;
        const int64_t at = q3::paged_scale_at(c, page, head, t);
        EXPECT(at >= page * stride && at + 2 <= page * stride + dense && at % 2 == 0);
    }
    const q3::PagedKV far{nullptr, nullptr, 1, INT_MAX, 1, 4, nullptr, nullptr, int64_t(1) << 30};
    EXPECT(q3::paged_scale_at(far, 1 << 20, 0, 3) == (int64_t(1) << 50) + 6);
}

static bool near(double a, double b) { return std::fabs(a - b) <= 1e-14 * std::fabs(b) + 1e-300; }

static void frequencies() {
    q3cu_ctx ctx;
    const double turn = 2.0 * 3.14159265358979323846;
    q3cu_rope r{1e6f, 128, Q3CU_ROPE_HALVES, Q3CU_ROPE_UNSCALED, 0, 0, 0, 0, 0, nullptr};
    for (int dim : {4, 52, 64, 128})
        for (float theta : {1e4f, 1e6f}) {
            r.dim = dim, r.theta = theta, r.scaling = Q3CU_ROPE_UNSCALED;
            const q3::TurnFreq plain = rope_freq_for(&ctx, r);
            for (int j = 0; j < 64; ++j)
                EXPECT(j < dim / 2 ? near(plain.v[j] * turn, std::exp(-2.0 * j / dim * std::log(double(theta)))) : plain.v[j] == 0.0);
            r.scaling = Q3CU_ROPE_LINEAR, r.factor = 4.0f;
            const q3::TurnFreq linear = rope_freq_for(&ctx, r);
            for (int j = 0; j < dim / 2; ++j) EXPECT(near(linear.v[j], plain.v[j] / 4));
            // YaRN: turns over the trained length decide
            r.scaling = Q3CU_ROPE_YARN, r.factor = 8.0f, r.original = 4096.0f, r.beta_fast = 32.0f, r.beta_slow = 1.0f;
            const q3::TurnFreq yarn = rope_freq_for(&ctx, r);
            const double fast = dim * std::log(4096.0 / (32.0 * turn)) / (2.0 * std::log(double(theta)));
            const double slow = dim * std::log(4096.0 / turn) / (2.0 * std::log(double(theta)));
            const double lo = std::max(std::floor(fast), 0.0), hi = std::min(std::ceil(slow), dim - 1.0);
            for (int j = 0; j < dim / 2; ++j) {
                if (j <= lo) EXPECT(near(yarn.v[j], plain.v[j]));
                if (j >= hi) EXPECT(near(yarn.v[j], plain.v[j] / 8));
                EXPECT(yarn.v[j] <= plain.v[j] * (1 + 1e-12) && yarn.v[j] >= plain.v[j] / 8 * (1 - 1e-12));
                const double share = (j - lo) / std::max(hi - lo, 0.001);
                if (share > 0 && share < 1) EXPECT(near(yarn.v[j], plain.v[j] * (1 - share) + plain.v[j] / 8 * share));
            }
            EXPECT(std::fabs(rope_form(r).gain - (0.1 * std::log(8.0) + 1.0)) < 1e-6);
        }
    // the same description again, another one between, given frequencies whose values change in place
    double f[2] = {0.5, 0.25};
    q3cu_rope given{1e6f, 4, Q3CU_ROPE_PAIRS, Q3CU_ROPE_UNSCALED, 0, 0, 0, 0, 2.0f, f};
    EXPECT(near(rope_freq_for(&ctx, given).v[1] * turn, 0.25) && rope_form(given).gain == 2.0f && rope_form(given).pairs);
    f[1] = 3.0;
    EXPECT(near(rope_freq_for(&ctx, given).v[1] * turn, 3.0));
    r.dim = 4, r.theta = 1e6f, r.scaling = Q3CU_ROPE_UNSCALED;
    EXPECT(near(rope_freq_for(&ctx, r).v[1] * turn, 1e-3) && near(rope_freq_for(&ctx, r).v[1] * turn, 1e-3));
}

static void refusals() {
    q3cu_ctx ctx;
    ctx.alive = true;
    ctx.sms = 148;
    alignas(32) static char m[8192];
    static int32_t ints[64];
    float *fs = reinterpret_cast<float *>(m);
    const q3cu_kv_cache_q8 good{{m, m, 2 * 16 * 128, 4, 2, 16, 128, Q3CU_Q8_0}, fs, fs, 2 * 16 * 2};
    const q3cu_kv_cache wide{m, m, 2 * 16 * 128, 4, 2, 16, 128, Q3CU_F32}, half{m, m, 2 * 16 * 128, 4, 2, 16, 128, Q3CU_BF16};
    const q3cu_kv_batch batch{ints, ints, ints, 1, 2};
    const q3cu_kv_prefix prefix{ints, ints, 1};
    const q3cu_rope rope{1e6f, 128, Q3CU_ROPE_HALVES, Q3CU_ROPE_UNSCALED, 0, 0, 0, 0, 0, nullptr};
    const size_t plenty = size_t(1) << 40;
    auto append = [&](const q3cu_kv_cache *c, const q3cu_rope *r, int64_t rows) {
        return q3cu_kv_append_rope(&ctx, c, &batch, rows, m, m, m, Q3CU_F32, 512, 256, 4, nullptr, nullptr, r, 1e-6f, m + 16,
                                   Q3CU_F32, nullptr);
    };
    auto read = [&](const q3cu_kv_cache *c, int64_t rows, void *k, void *v, int dt, int64_t stride) {
        return q3cu_kv_read(&ctx, c, &batch, rows, k, v, q3cu_dtype(dt), stride, nullptr);
    };
    auto paged = [&](const q3cu_kv_cache *c, size_t work) {
        return q3cu_attention_paged(&ctx, c, &batch, m, Q3CU_F32, 512, 4, m, work, m + 16, nullptr);
    };
    auto prompt = [&](const q3cu_kv_cache *c, int dt, int64_t rows) {
        return q3cu_attention_prompt(&ctx, c, &batch, rows, m, q3cu_dtype(dt), 512, 4, m + 16, nullptr);
    };
    auto shared = [&](const q3cu_kv_cache *c, const q3cu_kv_prefix *p, int dt, int heads, void *work, size_t bytes, void *out) {
        return q3cu_attention_shared(&ctx, c, &batch, p, m, q3cu_dtype(dt), heads * 128, heads, work, bytes, out, nullptr);
    };
    auto with = [&](auto change, q3cu_status st) {           // a Q8_0 cache that is refused everywhere
        q3cu_kv_cache_q8 c = good;
        change(c);
        EXPECT(append(&c.codes, &rope, 1) == st);
        EXPECT(read(&c.codes, 1, m, m + 4096, Q3CU_F32, 256) == st);
        EXPECT(paged(&c.codes, plenty) == st);
        EXPECT(prompt(&c.codes, Q3CU_BF16, 1) == st);
        EXPECT(shared(&c.codes, &prefix, Q3CU_BF16, 4, m, plenty, m + 16) == st);
    };
    with([](auto &c) { c.k_scale = nullptr; }, Q3CU_ERR_INVALID);
    with([](auto &c) { c.v_scale = nullptr; }, Q3CU_ERR_INVALID);
    with([](auto &c) { c.v_scale += 1; }, Q3CU_ERR_ALIGN);
    with([](auto &c) { c.scale_stride = 63; }, Q3CU_ERR_INVALID);
    with([](auto &c) { c.scale_stride = 66; }, Q3CU_ERR_ALIGN);
    with([](auto &c) { c.scale_stride = int64_t(1) << 40; }, Q3CU_ERR_INVALID);
    with([](auto &c) { c.codes.page_stride += 8; }, Q3CU_ERR_ALIGN);
    with([](auto &c) { c.codes.k = nullptr; }, Q3CU_ERR_INVALID);
    with([](auto &c) { c.codes.page_size = 24; }, Q3CU_ERR_INVALID);

    auto rope_with = [&](auto change) {
        q3cu_rope r = rope;
        change(r);
        return append(&good.codes, &r, 1) == Q3CU_ERR_INVALID;
    };
    EXPECT(append(&good.codes, nullptr, 1) == Q3CU_ERR_INVALID && append(&good.codes, &rope, 0) == Q3CU_OK);
    for (int dim : {0, 2, -4, 6, 130, 132}) EXPECT(rope_with([&](auto &r) { r.dim = dim; }));
    EXPECT(rope_with([](auto &r) { r.layout = 2; }) && rope_with([](auto &r) { r.scaling = 3; }));
    for (float x : {0.0f, -1.0f, NAN, INFINITY}) EXPECT(rope_with([&](auto &r) { r.theta = x; }));
    for (float x : {0.5f, -4.0f, NAN, INFINITY}) EXPECT(rope_with([&](auto &r) { r.scaling = Q3CU_ROPE_LINEAR, r.factor = x; }));
    for (float x : {-1.0f, NAN, INFINITY}) EXPECT(rope_with([&](auto &r) { r.gain = x; }));
    auto yarn = [](auto &r) { r.scaling = Q3CU_ROPE_YARN, r.factor = 4, r.original = 4096, r.beta_fast = 32, r.beta_slow = 1; };
    EXPECT(rope_with([&](auto &r) { yarn(r), r.original = 0; }) && rope_with([&](auto &r) { yarn(r), r.beta_slow = 32; }));
    EXPECT(rope_with([&](auto &r) { yarn(r), r.theta = 1; }) && rope_with([&](auto &r) { yarn(r), r.beta_fast = NAN; }));
    static double bad[64];
    bad[63] = NAN;
    EXPECT(rope_with([&](auto &r) { r.freq = bad; }));

    EXPECT(read(&good.codes, 0, nullptr, nullptr, Q3CU_F32, 0) == Q3CU_OK);
    EXPECT(read(&good.codes, -1, m, m + 4096, Q3CU_F32, 256) == Q3CU_ERR_INVALID);
    EXPECT(read(&good.codes, INT_MAX, m, m + 4096, Q3CU_F32, 256) == Q3CU_ERR_INVALID);
    EXPECT(read(&good.codes, 1, m, m, Q3CU_F32, 256) == Q3CU_ERR_INVALID);
    EXPECT(read(&good.codes, 1, nullptr, m, Q3CU_F32, 256) == Q3CU_ERR_INVALID);
    EXPECT(read(&good.codes, 1, m, m + 4096, Q3CU_F32, 255) == Q3CU_ERR_INVALID);
    EXPECT(read(&good.codes, 1, m, m + 4096, Q3CU_BF16, 260) == Q3CU_ERR_ALIGN);
    EXPECT(read(&good.codes, 1, m + 8, m + 4096, Q3CU_F32, 256) == Q3CU_ERR_ALIGN);
    EXPECT(read(&good.codes, 1, m, m + 4096, Q3CU_Q8_0, 256) == Q3CU_ERR_INVALID);

    EXPECT(prompt(&good.codes, Q3CU_F32, 1) == Q3CU_ERR_INVALID && prompt(&good.codes, Q3CU_BF16, 0) == Q3CU_OK);
    EXPECT(q3cu_quantize_q8(&ctx, m, Q3CU_Q8_0, 1, 64, reinterpret_cast<int8_t *>(m), fs, nullptr) == Q3CU_ERR_INVALID);

    size_t need = 0;
    EXPECT(q3cu_attention_shared_workspace(&ctx, 1, 4, 2, &need) == Q3CU_OK && need > 0);
    EXPECT(shared(&good.codes, &prefix, Q3CU_BF16, 4, m, need - 1, m + 16) == Q3CU_ERR_INVALID);
    EXPECT(shared(&good.codes, &prefix, Q3CU_BF16, 4, nullptr, need, m + 16) == Q3CU_ERR_INVALID);
    EXPECT(shared(&good.codes, &prefix, Q3CU_BF16, 4, m + 16, plenty, m + 16) == Q3CU_ERR_ALIGN);
    EXPECT(shared(&good.codes, &prefix, Q3CU_BF16, 4, m, plenty, m) == Q3CU_ERR_INVALID);            // out is q
    EXPECT(shared(&good.codes, &prefix, Q3CU_F32, 4, m, plenty, m + 16) == Q3CU_ERR_INVALID);
    EXPECT(shared(&wide, &prefix, Q3CU_BF16, 4, m, plenty, m + 16) == Q3CU_ERR_INVALID);
    EXPECT(shared(&half, nullptr, Q3CU_BF16, 4, m, plenty, m + 16) == Q3CU_ERR_INVALID);
    for (int heads : {0, 3, 34, -2}) EXPECT(shared(&half, &prefix, Q3CU_BF16, heads, m, plenty, m + 16) == Q3CU_ERR_INVALID);
    auto prefix_with = [&](auto change) {
        q3cu_kv_prefix p = prefix;
        change(p);
        return shared(&half, &p, Q3CU_BF16, 4, m, plenty, m + 16);
    };
    EXPECT(prefix_with([](auto &p) { p.seq_off = nullptr; }) == Q3CU_ERR_INVALID);
    EXPECT(prefix_with([](auto &p) { p.len = nullptr; }) == Q3CU_ERR_INVALID);
    EXPECT(prefix_with([](auto &p) { p.n_groups = -1; }) == Q3CU_ERR_INVALID);
    EXPECT(prefix_with([](auto &p) { p.n_groups = INT_MAX; }) == Q3CU_ERR_INVALID);
    EXPECT(prefix_with([](auto &p) { p.len = reinterpret_cast<int32_t *>(m + 2); }) == Q3CU_ERR_ALIGN);
    EXPECT(q3cu_attention_shared_workspace(&ctx, -1, 4, 2, &need) == Q3CU_ERR_INVALID);
    EXPECT(q3cu_attention_shared_workspace(&ctx, 1, 5, 2, &need) == Q3CU_ERR_INVALID);
    EXPECT(q3cu_attention_shared_workspace(&ctx, 1, 4, 2, nullptr) == Q3CU_ERR_INVALID);
    // a larger batch never needs less, and 64 bits hold the largest
    size_t before = 0;
    for (int n : {0, 1, 2, 63, 64, 65, 1000, 1 << 24}) {
        EXPECT(q3cu_attention_shared_workspace(&ctx, n, 64, 8, &need) == Q3CU_OK && need >= before);
        before = need;
    }
    EXPECT(before > (size_t(1) << 39));
    EXPECT(q3cu_kv_read(nullptr, &wide, &batch, 1, m, m, Q3CU_F32, 256, nullptr) == Q3CU_ERR_NOT_INIT);
    EXPECT(q3cu_attention_shared(nullptr, &half, &batch, &prefix, m, Q3CU_BF16, 512, 4, m, 1, m, nullptr) == Q3CU_ERR_NOT_INIT);
    EXPECT(q3cu_attention_shared_workspace(nullptr, 1, 4, 2, &need) == Q3CU_ERR_NOT_INIT);
    EXPECT(q3cu_kv_append_rope(nullptr, &wide, &batch, 1, m, m, m, Q3CU_F32, 512, 256, 4, nullptr, nullptr, &rope, 1e-6f, m,
                               Q3CU_F32, nullptr) == Q3CU_ERR_NOT_INIT);
}

int main() {
    groups();
    scales();
    frequencies();
    refusals();
    std::printf("ok\n");
    return 0;
}
