// Host checks of how attention_shared cuts its work, no GPU: every tile of every item belongs to one run, what a run leaves of an
// item lies where the join looks for it and nothing else does, and all of it inside the workspace.  The runs are walked here
// as the kernels walk them (q3cu_split.cuh, q3cu_prompt.cuh), with their arithmetic.  Includes the source of the join.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <tuple>
#include <vector>

#include "k_shared.cu"

#define EXPECT(x)                                           \
    do {                                                    \
        if (!(x)) {                                         \
            std::printf("line %d: %s\n", __LINE__, #x);     \
            std::exit(1);                                   \
        }                                                   \
    } while (0)

static uint32_t seed = 2468;
static uint32_t rnd() { return seed = seed * 1664525u + 1013904223u, seed >> 8; }

static void cuts() {
    for (int trial = 0; trial < 20000; ++trial) {
        const int64_t total = trial % 3 == 0 ? rnd() % 2000 : trial % 3 == 1 ? int64_t(rnd()) * rnd() : int64_t(rnd()) << 20;
        const int runs = 1 + rnd() % 400;
        const q3::PagedCut cut(total, runs);
        EXPECT(cut.begin(0) == 0 && cut.begin(runs) == total);
        for (int i = 0; i < 8 && total; ++i) {
            const int64_t u = (int64_t(rnd()) << 24 | rnd()) % total;
            const int run = cut.run_of(u);
            EXPECT(run >= 0 && run < runs && cut.begin(run) <= u && u < cut.begin(run + 1));
        }
    }
}

typedef std::tuple<int, int> Item;                          // sequence and kv head, or item of shared positions

// The sequences' own positions (paged_split_kernel, paged_q8_kernel over TailSeqs).
static void tails() {
    for (int trial = 0; trial < 2000; ++trial) {
        const int n_seqs = 1 + rnd() % 12, n_kv = 1 + rnd() % 4, runs = 1 + rnd() % (trial % 2 ? 12 : 300), tile = rnd() % 2 ? 64 : 128;
        std::vector<q3::PagedSpan> span(n_seqs);
        std::vector<int64_t> before(n_seqs + 1);
        for (int s = 0; s < n_seqs; ++s) {
            const int from = rnd() % 3 ? rnd() % 1000 : 0, more = rnd() % 4 ? rnd() % (trial % 5 ? 300 : 5000) : 0;
            span[s] = {from, from + more};
            const int n = span[s].tiles(tile);
            EXPECT((n > 0) == (more > 0) && (n == 0 || (span[s].base() <= from && span[s].base() + n * tile >= span[s].len &&
                                                       span[s].base() + (n - 1) * tile < span[s].len)));
            before[s + 1] = before[s] + (n ? q3::TAIL_LEAD + n : 0);
        }
        const q3::PagedCut cut(before[n_seqs] * n_kv, runs);
        std::map<Item, std::set<int>> seen;                  // tiles of an item
        std::map<int64_t, Item> slots;
        std::set<Item> whole;
        for (int run = 0; run < runs; ++run) {
            const int64_t u0 = cut.begin(run), u1 = cut.begin(run + 1);
            if (u0 == u1) continue;
            int s = n_seqs - 1, head, at, lead;
            while (before[s] * n_kv > u0 || before[s + 1] == before[s]) --s;
            q3::tail_place(u0 - before[s] * n_kv, span[s].tiles(tile), head, at, lead);
            EXPECT(head < n_kv && at < span[s].tiles(tile) && lead <= q3::TAIL_LEAD);
            for (int64_t u = u0; u < u1;) {
                const int tiles = span[s].tiles(tile);
                const int units = int(std::min(int64_t(lead) + tiles - at, u1 - u)), n = units - lead;
                if (n <= 0) break;
                for (int i = 0; i < n; ++i) EXPECT(seen[Item(s, head)].insert(at + i).second);
                if (n == tiles) EXPECT(whole.insert(Item(s, head)).second);
                else EXPECT(slots.emplace(2 * int64_t(run) + (u != u0), Item(s, head)).second);
                u += units;
                if (u < u1) {                                // walk_on
                    EXPECT(at + n == tiles);
                    at = 0, lead = q3::TAIL_LEAD;
                    if (++head == n_kv) {
                        head = 0;
                        do EXPECT(++s < n_seqs); while (span[s].tiles(tile) == 0);
                    }
                }
            }
        }
        size_t found = 0;
        for (int s = 0; s < n_seqs; ++s)
            for (int head = 0; head < n_kv; ++head) {
                const int tiles = span[s].tiles(tile);
                EXPECT(int(seen[Item(s, head)].size()) == tiles);
                if (!tiles) continue;
                const int64_t a = before[s] * n_kv + int64_t(head) * (q3::TAIL_LEAD + tiles);
                const q3::PartsOf p(cut, a, a + q3::TAIL_LEAD, a + q3::TAIL_LEAD + tiles);
                EXPECT((p.n == 1) == (whole.count(Item(s, head)) == 1));
                for (int i = 0; p.n > 1 && i < p.n; ++i, ++found) {
                    EXPECT(slots.count(p.slot(i)) && slots[p.slot(i)] == Item(s, head));
                    EXPECT(p.slot(i) < 2 * int64_t(runs));
                }
            }
        EXPECT(found == slots.size());
    }
}

// What groups share (prompt_tc_kernel<PT_SHARED>): items in the order group, kv head, block of sequences.
static void prefixes() {
    for (int trial = 0; trial < 1500; ++trial) {
        const int n_kv = 1 + rnd() % 4, group = 1 + rnd() % 16, sms = 1 + rnd() % (trial % 2 ? 10 : 160);
        const q3::FastDiv per_block(2 * (q3::PT_ROWS / group));
        std::vector<q3::SharedEntry> entries(1 + rnd() % 5);
        int n_seqs = 0;
        int64_t units = 0;
        for (auto &e : entries) {
            e = {n_seqs, 2 + int(rnd() % (trial % 3 ? 20 : 400)), 1 + int(rnd() % (trial % 5 ? 600 : 20000)), 0, units};
            units += int64_t((e.len + q3::PT_KEYS - 1) / q3::PT_KEYS) * (per_block(e.count - 1) + 1);
            n_seqs += e.count;
        }
        const q3::SharedWork w = q3::shared_work(n_seqs, n_kv * group, n_kv, sms);
        const size_t row = q3::SHARED_ROW * sizeof(float);
        EXPECT((size_t(n_seqs) * n_kv * group + size_t(2) * sms * w.slot_rows) * row <= w.tails);
        EXPECT(w.tails + size_t(n_seqs) * n_kv * group * row <= w.part);
        EXPECT(w.part + size_t(q3::paged_runs(sms)) * 2 * group * row <= w.spans && w.spans < w.before && w.before < w.entry &&
               w.entry < w.entries && w.entries < w.of && w.of + n_seqs * sizeof(q3::SharedEntry) <= w.bytes);
        const q3::PagedCut cut(units * n_kv, sms);
        typedef std::tuple<int, int, int> Part;              // entry, kv head, block
        std::map<Part, std::set<int>> seen;
        std::map<int64_t, Part> slots;
        std::set<Part> whole;
        for (int run = 0; run < sms; ++run) {
            int64_t u = cut.begin(run);
            const int64_t u1 = cut.begin(run + 1);
            if (u == u1) continue;
            int g = int(entries.size()) - 1;
            while (entries[g].units * n_kv > u) --g;         // shared_run
            int keys = (entries[g].len + q3::PT_KEYS - 1) / q3::PT_KEYS, blocks = per_block(entries[g].count - 1) + 1;
            const int64_t at = u - entries[g].units * n_kv, item = q3::quot(at, keys);
            int tile = int(at - item * keys), head = int(q3::quot(item, blocks)), block = int(item - int64_t(head) * blocks);
            for (int fragment = 0; u < u1; ++fragment) {     // the kernel's items
                EXPECT(head < n_kv && block < blocks && tile < keys);
                const int n = int(std::min(int64_t(keys - tile), u1 - u));
                for (int i = 0; i < n; ++i) EXPECT(seen[Part(g, head, block)].insert(tile + i).second);
                if (n == keys) EXPECT(whole.insert(Part(g, head, block)).second);
                else EXPECT(slots.emplace(2 * int64_t(run) + (fragment > 0), Part(g, head, block)).second);
                u += n;
                tile = 0;                                    // shared_next
                if (u < u1 && ++block == blocks) {
                    block = 0;
                    if (++head == n_kv) {
                        head = 0;
                        EXPECT(++g < int(entries.size()));
                        keys = (entries[g].len + q3::PT_KEYS - 1) / q3::PT_KEYS, blocks = per_block(entries[g].count - 1) + 1;
                    }
                }
            }
        }
        std::set<int64_t> found;
        for (int g = 0; g < int(entries.size()); ++g) {
            const q3::SharedEntry &e = entries[g];
            const int keys = (e.len + q3::PT_KEYS - 1) / q3::PT_KEYS, blocks = per_block(e.count - 1) + 1;
            for (int head = 0; head < n_kv; ++head)
                for (int at = 0; at < e.count; ++at) {       // shared_join_kernel
                    const int block = per_block(at), slot = (at - block * per_block.d) * group;
                    const int64_t a = e.units * n_kv + (int64_t(head) * blocks + block) * keys;
                    const q3::PartsOf p(cut, a, a, a + keys);
                    EXPECT(slot + group <= w.slot_rows && int(seen[Part(g, head, block)].size()) == keys);
                    EXPECT((p.n == 1) == (whole.count(Part(g, head, block)) == 1));
                    for (int i = 0; p.n > 1 && i < p.n; ++i) {
                        EXPECT(slots.count(p.slot(i)) && slots[p.slot(i)] == Part(g, head, block) && p.slot(i) < 2 * int64_t(sms));
                        found.insert(p.slot(i));
                    }
                }
        }
        EXPECT(found.size() == slots.size());
    }
}

int main() {
    cuts();
    tails();
    prefixes();
    std::printf("ok\n");
    return 0;
}
