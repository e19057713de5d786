// The C++ host mirror's block tables and paged 4-bit cache (include/peregrine_hip.hpp, namespace paged), two requests through two
// steps: attention against double-precision attention over the values that the cache says it holds, over all blocks and over chosen ones.
#include <cmath>
#include <cstdio>

#include "peregrine_hip.hpp"

using namespace peregrine;

static int failures = 0;
#define EXPECT(cond, ...)                                     \
    do {                                                      \
        if (!(cond)) {                                        \
            ++failures;                                       \
            std::printf("FAIL %s:%d: ", __FILE__, __LINE__); \
            std::printf(__VA_ARGS__);                         \
            std::printf("\n");                                \
        }                                                     \
    } while (0)

static float lcg(uint32_t &st) { return (float)((st = st * 1664525u + 1013904223u) >> 8) * (2.0f / 16777216.0f) - 1.0f; }

// Largest difference from attention in double precision over the cache's own values, blocks chosen by `in` (all where empty).
static double off(const paged::PagedKV4Cache &cache, const paged::BlockTables &t, size_t bs, const std::vector<float> &q, size_t heads, const std::vector<int32_t> &start,
                  const std::vector<float> &got, const std::vector<int32_t> &in, size_t top, float scale) {
    const size_t hd = cache.head_dim, group = heads / cache.num_kv_heads;
    double worst = 0;
    for (size_t b = 0; b < t.seq_lens.size(); ++b) {
        std::vector<int32_t> slots;
        for (int i = 0; i < t.seq_lens[b]; ++i) slots.push_back(t.table[b * t.max_blocks() + i / bs] * (int)bs + i % (int)bs);
        auto [k, v] = cache.read(slots);
        for (int r = start[b]; r < start[b + 1]; ++r)
            for (size_t h = 0; h < heads; ++h) {
                const int pos = t.seq_lens[b] - (start[b + 1] - r);
                const size_t kh = h / group;
                std::vector<double> o(hd, 0.0), s(pos + 1);
                double m = -INFINITY, l = 0;
                for (int i = 0; i <= pos; ++i) {
                    bool seen = in.empty();
                    for (size_t j = 0; j < top && !seen; ++j) seen = in[(r * cache.num_kv_heads + kh) * top + j] == i / (int)bs;
                    s[i] = seen ? 0.0 : -INFINITY;
                    for (size_t d = 0; d < hd && seen; ++d) s[i] += (double)q[(r * heads + h) * hd + d] * k[(i * cache.num_kv_heads + kh) * hd + d] * scale;
                    m = std::fmax(m, s[i]);
                }
                for (int i = 0; i <= pos; ++i) {
                    const double p = std::exp(s[i] - m);
                    l += p;
                    for (size_t d = 0; d < hd; ++d) o[d] += p * v[(i * cache.num_kv_heads + kh) * hd + d];
                }
                for (size_t d = 0; d < hd; ++d) worst = std::fmax(worst, std::fabs(o[d] / l - got[(r * heads + h) * hd + d]));
            }
    }
    return worst;
}

static void run(const GpuContext &gpu) {
    const size_t bs = 16, hk = 2, heads = 4, hd = 64, top = 3;
    const float scale = 0.125f;
    paged::BlockTables t(gpu, 2, 20, bs, 8);
    paged::PagedKV4Cache cache(gpu, 20, bs, hk, hd);
    uint32_t st = 7;
    for (const std::vector<int32_t> &add : {std::vector<int32_t>{100, 37}, std::vector<int32_t>{1, 3}}) {
        auto step = t.extend(add);
        EXPECT(step.granted[0] == 1 && step.granted[1] == 1, "not granted");
        const size_t n = step.slots.size();
        std::vector<float> k(n * hk * hd), v(k.size()), q(n * heads * hd);
        for (auto *a : {&k, &v, &q})
            for (auto &x : *a) x = lcg(st);
        cache.append(k, v, step.slots);
        cache.summarise(step.query_start, t.seq_lens, t.table);
        // Values within 1, scores within 0.125 * 64 = 8: fixed point takes 5e-7 of a score and two f32 roundings 2e-6, which moves
        // weights by 5e-6 at most; 22 bits of p d 5e-7, sums of up to 101 weights and of as many products 101 * 2^-24 = 6e-6 each.
        auto out = cache.attention(q, heads, step.query_start, t.seq_lens, t.table, scale, paged::AttentionMask::Causal(0), 0.0f);
        EXPECT(off(cache, t, bs, q, heads, step.query_start, out, {}, 0, scale) < 2e-5, "attention off by %.3g", off(cache, t, bs, q, heads, step.query_start, out, {}, 0, scale));
        auto in = cache.select(q, heads, step.query_start, t.seq_lens, t.table, top, 1, 1);
        auto part = cache.attention_selected(q, heads, step.query_start, t.seq_lens, t.table, in, top, scale, 0.0f);
        EXPECT(off(cache, t, bs, q, heads, step.query_start, part, in, top, scale) < 2e-5, "selected attention off by %.3g",
               off(cache, t, bs, q, heads, step.query_start, part, in, top, scale));
    }
    EXPECT(t.free_count == 20 - 7 - 3, "%d blocks are free", t.free_count);
    t.release({1, 0});
    EXPECT(t.free_count == 17 && t.seq_lens[0] == 0 && t.seq_lens[1] == 40, "after the release");
    bool refused = false;
    try {
        cache.append(std::vector<float>(5), std::vector<float>(5), {0});
    } catch (const Panic &e) {
        refused = e.status == PG_EINVAL;
    }
    EXPECT(refused, "a short slice was taken");
    refused = false;
    try {
        cache.attention(std::vector<float>(heads * hd), heads, {0, 0, 1}, t.seq_lens, t.table, scale, paged::AttentionMask::Causal(3), 0.0f);
    } catch (const Panic &e) {
        refused = e.status == PG_EINVAL;
    }
    EXPECT(refused, "a mask's offset was taken");
}

int main() {
    try {
        GpuContext gpu(0);
        run(gpu);
    } catch (const std::exception &e) {
        std::printf("FAIL: uncaught %s\n", e.what());
        return 2;
    }
    std::printf(failures ? "FAILED: %d check(s)\n" : "OK: all checks passed\n", failures);
    return failures ? 1 : 0;
}
