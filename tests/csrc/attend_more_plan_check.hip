// Checks how attention calls with sinks and shared prefixes are cut (si_attend_plan.h), host code alone,
// over seeded descriptors up to the longest tables and the most rows that a call may have:
//   * without either a call is cut as it is without them;
//   * no sequence has more parts of its own keys than there are places for, wherever its window and its
//     prefix lie, and no prefix more than share_split;
//   * a row's parts of both fit one join;
//   * the workspace's regions hold every place and do not overlap.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstring>
#include <random>

#include "si_attend_plan.h"

namespace {

unsigned long long cases, bad;

void expect(bool ok, const char* what, const si_paged_attention_desc& d, const si_paged_attention_more& m)
{
    if (ok) return;
    if (++bad <= 10)
        std::printf("# %s: tokens %u seqs %u heads %u/%u dim %u pages %u x %u starts %d window %u sinks %u groups %u\n", what,
                    d.tokens, d.seqs, d.q_heads, d.kv_heads, d.head_dim, d.table_pages, d.page_tokens,
                    d.q_starts != nullptr, d.window, m.sinks, m.groups);
}

// The keys that are left of a sequence of `len` with n new tokens and its group's first `from`, in steps.
uint64_t left(const si_paged_attention_desc& d, uint32_t sinks, uint64_t len, uint64_t n, uint64_t from, uint64_t step)
{
    const int64_t window = d.window < si::kMostLength ? d.window : 0;
    int64_t lo = window ? int64_t(len) - int64_t(n) - window + 1 : 0;
    lo = lo > int64_t(from) ? lo : int64_t(from);
    lo = (lo < int64_t(len) ? lo : int64_t(len)) / int64_t(step) * int64_t(step);
    int64_t head = 0;
    const int64_t head_lo = int64_t(from / step * step);
    if (window && sinks > from) {
        const int64_t end = int64_t((sinks + step - 1) / step * step);
        head = (end < lo ? end : lo) - head_lo;
        head = head > 0 ? head : 0;
    }
    return uint64_t(head) + (int64_t(len) > lo ? uint64_t(int64_t(len) - lo) : 0);
}

void check(const si_paged_attention_desc& d, const si_paged_attention_more& m, std::mt19937_64& g)
{
    using namespace si;
    ++cases;
    const Plan p = attend_plan(d, &m);
    if (!d.window || d.window >= kMostLength) expect(p.sinks == 0, "sinks without a window", d, m);
    if (!p.sinks && !m.groups) {
        const Plan q = attend_plan(d);
        expect(p.bytes == q.bytes && p.few_groups == q.few_groups && p.few_per == q.few_per && p.tile_per == q.tile_per &&
                   p.tile_split == q.tile_split && p.tiles == q.tiles && p.fits == q.fits && p.share_groups == 0,
               "plain", d, m);
    }
    if (!p.fits) return;
    const uint64_t keys = uint64_t(d.table_pages) * d.page_tokens, pairs = uint64_t(d.seqs) * d.kv_heads;
    uint64_t at = 0, most = 0;
    const auto region = [&](uint64_t from, uint64_t bytes) {
        expect(from >= at && from + bytes <= p.bytes, "workspace", d, m);
        at = from + bytes;
    };
    if (p.few) {
        const bool places = p.few_ml != 0;
        if (places) {
            const uint64_t n = p.few_per ? p.few_groups : 2ull * p.few_groups;
            region(p.few_o, n * kFewRows * d.head_dim * 4);
            region(p.few_ml, n * kFewRows * 8);
            if (!p.sinks && !m.groups) region(p.few_parts, pairs * 8);
        }
        for (int i = 0; i < 6; ++i) {
            const uint64_t len = i < 2 ? keys : g() % (keys + 1), group = d.q_heads / d.kv_heads;
            const uint64_t n = 1 + (d.q_starts ? g() % (kFewRows / group ? kFewRows / group : 1) : 0);
            const uint64_t from = m.groups && i % 2 ? g() % (keys + 1) : 0;
            const uint64_t unit = p.sinks || m.groups ? kFewStep : kFewKeys;
            const uint64_t units = (left(d, p.sinks, len, n, from, kFewKeys) + unit - 1) / unit;
            uint64_t parts = 1;
            if (p.few_per) {
                parts = (units + p.few_per - 1) / p.few_per;
                expect(parts * pairs <= p.few_groups || parts <= 1, "few-row parts", d, m);
            } else {
                expect(d.seqs <= (m.groups ? kShareSeqs : 64), "even shares", d, m);
                // from anywhere in a share on; shares are of `least` units or more
                const bool more = p.sinks || m.groups;
                const uint64_t least = more ? (units + p.few_least - 2) / (p.few_least - 1) : p.few_least;
                if (units > (more ? 1 : kFewWhole)) parts = (units + least - 2) / least + 1;
            }
            expect(parts <= 1 || places, "few-row places", d, m);
            most = most > parts ? most : parts;
        }
    }
    if (p.tile) {
        expect(p.tile_per >= kTileKeys && p.tile_per % kTileKeys == 0, "tile part", d, m);
        for (int i = 0; i < 6; ++i) {
            const uint64_t len = i < 2 ? keys : g() % (keys + 1), n = 1 + (i % 3 ? g() % d.tokens : d.tokens - 1);
            const uint64_t from = m.groups && i % 2 ? g() % (keys + 1) : 0;
            const uint64_t parts = (left(d, p.sinks, len, n, from, kTileKeys) + p.tile_per - 1) / p.tile_per;
            expect(parts <= p.tile_split || parts <= 1, "tile parts", d, m);
            most = most > parts ? most : parts;
        }
    }
    if (p.tile_split > 1 || m.groups) {
        const uint64_t n = uint64_t(p.tile_split) * d.tokens * d.q_heads;
        region(p.tile_o, n * d.head_dim * 4);
        region(p.tile_ml, n * 8);
    }
    if (m.groups) {
        const uint64_t n = uint64_t(p.share_split) * d.tokens * d.q_heads;
        region(p.share_o, n * d.head_dim * 4);
        region(p.share_ml, n * 8);
        expect(p.share_split >= 1 && p.share_split <= kMaxSplit / 4 * 3, "prefix parts' number", d, m);
        expect(p.share_groups > 0 && p.share_groups % 8 == 0, "prefix tiles", d, m);
        for (uint64_t len : {uint64_t(1), keys, 1 + g() % keys}) {
            const uint64_t per = share_part(uint32_t(len), p.share_split, g() % (1 + uint64_t(d.tokens) * d.q_heads));
            expect(per % kTileKeys == 0 && per >= kTileKeys && (len + per - 1) / per <= p.share_split, "prefix part", d, m);
        }
        most += p.share_split;
    }
    if (p.few_joins) region(p.few_joins, pairs * 16);
    expect(p.few_joins || !p.few || p.bytes == 0 || !(p.sinks || m.groups), "joins", d, m);
    if (p.sinks || m.groups) {
        // workgroups for every tile that lengths can make: n sequences, or groups, of rows that add up
        const uint64_t group = d.q_heads / d.kv_heads, tokens = d.tokens;
        for (int i = 0; i < 4; ++i) {
            // sequences of n tokens each, and the tokens that are left to one more
            const uint64_t n = i ? 1 + g() % (i == 1 ? 2 * kTileRows / group + 1 : tokens) : kFewRows / group + 1;
            uint64_t seqs = tokens / n < d.seqs ? tokens / n : d.seqs, rest = seqs < d.seqs ? tokens - seqs * n : 0;
            const auto tiles = [&](uint64_t t) { return t * group > p.few_rows ? (t * group + kTileRows - 1) / kTileRows : 0; };
            if (!d.q_starts) seqs = tokens, rest = 0;
            const uint64_t there = seqs * tiles(d.q_starts ? n : 1) + tiles(rest);
            if (p.tile) expect(there * d.kv_heads * p.tile_split <= p.tile_groups, "tiles", d, m);
            else expect(there == 0, "tiles without a kernel", d, m);
            // groups of at least two sequences, of n tokens each
            if (m.groups) {
                const uint64_t most_groups = m.groups < d.seqs / 2 ? m.groups : d.seqs / 2;
                const uint64_t k = tokens / n < most_groups ? tokens / n : most_groups;
                const uint64_t t = k * ((n * group + kTileRows - 1) / kTileRows);
                expect(t * d.kv_heads * p.share_split <= p.share_groups, "prefix tiles", d, m);
            }
        }
    }
    expect(most <= kMaxSplit, "parts of a row", d, m);
}

}  // namespace

int main()
{
    std::mt19937_64 g(11);
    const auto log2 = [&](int most) { return uint32_t((1ull << (g() % (most + 1))) + (g() % 3 ? 0 : g() % 7)); };
    static const int64_t starts = 0;
    for (int i = 0; i < 1000000; ++i) {
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
        d.window = g() % 4 ? log2(31) : 0;
        si_paged_attention_more m{};
        m.sinks = g() % 3 ? log2(29) : 0;
        m.groups = g() % 2 ? log2(25) : 0;
        check(d, m, g);
    }
    std::printf("cases %llu bad %llu\n", cases, bad);
    return bad != 0;
}
