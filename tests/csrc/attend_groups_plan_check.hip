// Checks that naming groups does not leave a long sequence to fewer workgroups (si_attend_plan.h), host code alone,
// over seeded descriptors: where the parts of few-row sequences have one length, it is no longer beside groups than
// without them, but for the sixteen parts that a row's own keys may have there.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <random>

#include "si_attend_plan.h"

int main()
{
    using namespace si;
    std::mt19937_64 g(12);
    const auto log2 = [&](int most) { return uint32_t((1ull << (g() % (most + 1))) + (g() % 3 ? 0 : g() % 7)); };
    static const int64_t starts = 0;
    unsigned long long cases = 0, bad = 0;
    for (int i = 0; i < 300000; ++i) {
        si_paged_attention_desc d{};
        d.page_tokens = 8u << g() % 13;
        d.table_pages = log2(16);
        if (uint64_t(d.table_pages) * d.page_tokens > 1ull << 30) continue;
        d.kv_heads = log2(6);
        d.q_heads = d.kv_heads * log2(4);
        d.head_dim = 8 * (1 + g() % 32);
        d.seqs = i % 2 ? 257 + uint32_t(g() % 6000) : log2(14);
        d.q_starts = g() % 2 ? &starts : nullptr;
        d.tokens = d.q_starts ? d.seqs + uint32_t(g() % 999) : d.seqs;
        if (uint64_t(d.tokens) * d.q_heads >= 1ull << 26) continue;
        si_paged_attention_more m{};
        m.groups = log2(6);
        const Plan p = attend_plan(d, &m), q = attend_plan(d);
        if (!p.few || !p.fits) continue;
        ++cases;
        if (!p.few_per || !q.few_per) continue;
        const uint64_t keys = uint64_t(d.table_pages) * d.page_tokens;
        const uint64_t part = uint64_t(p.few_per) * kFewStep, without = uint64_t(q.few_per) * kFewKeys;
        const uint64_t least = ((keys + 15) / 16 + kFewStep - 1) / kFewStep * kFewStep;
        if (part > (without > least ? without : least) && ++bad <= 10)
            std::printf("# part %llu keys, without groups %llu: seqs %u heads %u/%u keys %llu\n",
                        static_cast<unsigned long long>(part), static_cast<unsigned long long>(without), d.seqs, d.q_heads,
                        d.kv_heads, static_cast<unsigned long long>(keys));
    }
    std::printf("cases %llu bad %llu\n", cases, bad);
    return bad != 0;
}
