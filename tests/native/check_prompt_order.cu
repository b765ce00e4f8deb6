// The items of a prompt launch, found in any order: one warp asks PromptOrder for every index of a launch once, rising and
// shuffled, and the host compares what has rows with its own list of (sequence, block, kv head).
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "q3cu_paged.cuh"

struct Found { int s, head, first; };

__global__ void ask(q3::PagedKV c, q3::PagedSeqs b, int rows, q3::FastDiv per_block, int tile_keys, const int *index, int n,
                    Found *out) {
    q3::PromptOrder order(b, c, rows, per_block, tile_keys, nullptr);
    for (int i = 0; i < n; ++i) {
        const q3::PromptItem it = order.find(index[i]);
        if (threadIdx.x == 0) out[i] = it.s < 0 || it.rows == 0 ? Found{-1, 0, 0} : Found{it.s, it.head, it.first};
    }
}

static uint32_t seed = 2024;
static uint32_t rnd() { return seed = seed * 1664525u + 1013904223u, seed >> 8; }

template <typename T> static T *upload(const std::vector<T> &v) {
    T *p = nullptr;
    if (cudaMalloc(&p, std::max<size_t>(1, v.size()) * sizeof(T)) != cudaSuccess ||
        cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice) != cudaSuccess)
        std::printf("no device memory\n"), std::exit(2);
    return p;
}

int main() {
    for (int n_seqs : {1, 2, 7, 31, 33, 64, 65, 130, 1000, 2500})
        for (int trial = 0; trial < 6; ++trial) {
            const int n_kv = 1 + int(rnd() % 8), block = 1 + int(rnd() % 64), tile_keys = trial % 2 ? 64 : 128;
            std::vector<int> off(n_seqs + 1, 0), len(n_seqs);
            for (int s = 0; s < n_seqs; ++s) {
                off[s + 1] = off[s] + (rnd() % 5 ? int(rnd() % 150) : 0);
                len[s] = off[s + 1] - off[s] + (rnd() % 2 ? int(rnd() % 3000) : 0);
            }
            std::vector<Found> want;                         // in any order
            for (int s = 0; s < n_seqs; ++s)
                for (int first = 0; first < off[s + 1] - off[s]; first += block)
                    for (int h = 0; h < n_kv; ++h) want.push_back({s, h, first});
            const int items = int(want.size()), asked = (off[n_seqs] / block + n_seqs) * n_kv;
            std::vector<int> rising(asked), mixed;
            for (int i = 0; i < asked; ++i) rising[i] = i;
            mixed = rising;
            for (int i = asked - 1; i > 0; --i) std::swap(mixed[i], mixed[rnd() % (i + 1)]);
            const q3::PagedKV c{nullptr, nullptr, 0, 1, n_kv, 4};
            const q3::PagedSeqs b{upload(off), upload(len), nullptr, n_seqs, 1000};
            std::vector<Found> got[2];
            for (int x = 0; x < 2; ++x) {
                const std::vector<int> &index = x ? mixed : rising;
                Found *d_out = upload(std::vector<Found>(asked));
                int *d_index = upload(index);
                ask<<<1, 32>>>(c, b, off[n_seqs], q3::FastDiv(block), tile_keys, d_index, asked, d_out);
                std::vector<Found> out(asked);
                if (cudaMemcpy(out.data(), d_out, asked * sizeof(Found), cudaMemcpyDeviceToHost) != cudaSuccess)
                    return std::printf("kernel failed\n"), 2;
                got[x].resize(asked);
                for (int i = 0; i < asked; ++i) got[x][index[i]] = out[i];
                cudaFree(d_out), cudaFree(d_index);
            }
            cudaFree(const_cast<int *>(b.row_off)), cudaFree(const_cast<int *>(b.kv_len));
            auto less = [](const Found &p, const Found &q) {
                return p.s != q.s ? p.s < q.s : p.first != q.first ? p.first < q.first : p.head < q.head;
            };
            for (int x = 0; x < 2; ++x) {
                got[x].erase(std::remove_if(got[x].begin(), got[x].end(), [](const Found &f) { return f.s < 0; }), got[x].end());
                if (int(got[x].size()) != items)
                    return std::printf("%d sequences, %s: %d items of %d\n", n_seqs, x ? "shuffled" : "rising",
                                       int(got[x].size()), items), 1;
                std::sort(got[x].begin(), got[x].end(), less);
                std::sort(want.begin(), want.end(), less);
                for (int i = 0; i < items; ++i)
                    if (less(got[x][i], want[i]) || less(want[i], got[x][i]))
                        return std::printf("%d sequences, %s: item %d of %d is missing\n", n_seqs, x ? "shuffled" : "rising", i,
                                           items), 1;
            }
        }
    std::printf("ok\n");
    return 0;
}
