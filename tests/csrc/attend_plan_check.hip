// Checks how attention calls over the paged cache are cut (si_attend_plan.h), host code alone, over
// seeded descriptors up to the longest tables and the most rows that a call may have:
//   * a part is a whole number of steps, no longer than the keys rounded up to one, so that the
//     kernels' 32-bit positions hold its end wherever it begins;
//   * no sequence that fits the table has more parts than there are places for;
//   * the keys are shared out evenly (few_per 0) only among at most 64 sequences, the ones that a
//     wave can hold, and then in at most as many shares a sequence as a join can take;
//   * the workspace's regions hold every place and do not overlap.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <random>

#include "si_attend_plan.h"

namespace {

unsigned long long cases, bad;

void expect(bool ok, const char* what, const si_paged_attention_desc& d)
{
    if (ok) return;
    if (++bad <= 10)
        std::printf("# %s: tokens %u seqs %u heads %u/%u dim %u pages %u x %u starts %d\n", what, d.tokens, d.seqs,
                    d.q_heads, d.kv_heads, d.head_dim, d.table_pages, d.page_tokens, d.q_starts != nullptr);
}

void check(const si_paged_attention_desc& d)
{
    using namespace si;
    ++cases;
    const Plan p = attend_plan(d);
    if (!p.fits) return;
    const uint64_t keys = uint64_t(d.table_pages) * d.page_tokens, pairs = uint64_t(d.seqs) * d.kv_heads;
    uint64_t at = 0;
    const auto region = [&](uint64_t from, uint64_t bytes) {
        expect(from >= at && from + bytes <= p.bytes, "workspace", d);
        at = from + bytes;
    };
    if (p.few && p.few_per) {
        const uint64_t per = uint64_t(p.few_per) * kFewKeys, parts = (keys + per - 1) / per;
        expect(per % kFewStep == 0 && per <= (keys + kFewStep - 1) / kFewStep * kFewStep, "few-row part", d);
        expect(pairs * parts <= p.few_groups && parts <= kMaxSplit, "few-row parts", d);
        if (parts > 1) {
            region(p.few_o, uint64_t(p.few_groups) * kFewRows * d.head_dim * 4);
            region(p.few_ml, uint64_t(p.few_groups) * kFewRows * 8);
            region(p.few_parts, pairs * 8);
        }
    } else if (p.few) {
        expect(d.seqs <= 64, "even shares", d);
        const uint64_t units = (keys + kFewKeys - 1) / kFewKeys;
        expect(p.few_groups >= 1 && p.few_least >= 1, "even shares' number", d);
        // a sequence's units, from anywhere in a share on
        expect((units + p.few_least - 2) / p.few_least + 1 <= kMaxSplit, "even shares of a sequence", d);
        if (units > kFewWhole) {
            region(p.few_o, 2ull * p.few_groups * kFewRows * d.head_dim * 4);
            region(p.few_ml, 2ull * p.few_groups * kFewRows * 8);
            region(p.few_parts, pairs * 8);
        }
    }
    if (p.tile) {
        expect(p.tile_per >= kTileKeys && p.tile_per % kTileKeys == 0 &&
                   p.tile_per <= (keys + kTileKeys - 1) / kTileKeys * kTileKeys,
               "tile part", d);
        if (p.tile_per) expect((keys + p.tile_per - 1) / p.tile_per <= p.tile_split, "tile parts", d);
        expect(p.tile_split <= kMaxSplit, "tile parts' number", d);
        if (p.tile_split > 1) {
            const uint64_t n = uint64_t(p.tile_split) * d.tokens * d.q_heads;
            region(p.tile_o, n * d.head_dim * 4);
            region(p.tile_ml, n * 8);
        }
    }
}

}  // namespace

int main()
{
    std::mt19937_64 g(7);
    const auto log2 = [&](int most) { return uint32_t((1ull << (g() % (most + 1))) + (g() % 3 ? 0 : g() % 7)); };
    static const int64_t starts = 0;
    for (int i = 0; i < 2000000; ++i) {
        si_paged_attention_desc d{};
        d.page_tokens = 8u << g() % 13;
        const uint32_t widest = (1u << 30) / d.page_tokens;
        d.table_pages = g() % 4 ? log2(30) : widest;
        if (d.table_pages > widest) d.table_pages = widest;
        d.kv_heads = log2(12);
        d.q_heads = d.kv_heads * log2(8);
        d.head_dim = 8 * (1 + g() % 32);
        d.seqs = log2(25);
        d.tokens = log2(25);
        d.q_starts = g() % 3 ? &starts : nullptr;
        if (!d.q_starts) d.tokens = d.seqs;
        if (uint64_t(d.tokens) * d.q_heads >= 1ull << 26 || d.seqs >= 1u << 26) continue;
        check(d);
    }
    std::printf("cases %llu bad %llu\n", cases, bad);
    return bad != 0;
}
