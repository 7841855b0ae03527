// How an attention call over the paged cache is cut and launched: host code
// alone, so that it can be checked without a GPU.
#pragma once

#include <stdint.h>

#include <numeric>

#include "secure_infer_gpu.h"

namespace si {

// The tile kernel's keys per step, and its rows: 32 a wave, whose scores of a step, numerators and
// queries fill the registers that two waves a SIMD leave each other at head dim 128.  (64 rows a
// wave, one wave a SIMD: 2,984 us where 32 rows take 2,430: the accumulators
// move between the two halves of the registers.  8 waves on rings of 2 to 4
// buffers: 2,385 and 2,400.)
constexpr uint32_t kTileKeys = 64;
constexpr uint32_t kTileWaves = 4;
constexpr uint32_t kTileRows = 32 * kTileWaves;
// The few-row kernel's keys per wave and step; a workgroup's step.
constexpr uint32_t kFewKeys = 32;
constexpr uint32_t kFewWaves = 4;
constexpr uint32_t kFewStep = kFewKeys * kFewWaves;
// Most rows of a sequence in the few-row kernel, one to a column of its matrix
// instructions.  (Two columns blocks, for 32 rows: 32 sequences of 4 tokens x 8
// heads over 4,096 keys 96 us, in tiles 64; 4 such sequences 22.5 and 22.8.)
constexpr uint32_t kFewRows = 16;
constexpr uint32_t kMaxSplit = 64;
// Workgroups that parts of a fixed length are made for, at the longest lengths the tables
// allow.  Few-row parts, 64 ragged sequences to 8,192 keys of 4 heads: 4,096 62.2 us, 2,048
// 64.4, 8,192 64.5.
constexpr uint64_t kFewTarget = 4096;
// Tiles are cut where there are fewer than kTileFew, into parts of at least kTileSplitMin keys.
// Target and least 768 and 512, against 1,280 and 256, and 2,048 and 512: a chunk of 128 tokens over 8,192
// keys, 32/8 heads, 43.7 us, 56, 55; 512 tokens over 32,768, 8/1 heads, 127, 131, 140.
// 2,048 tokens over 8,192 keys, 32/8 heads (more than kTileFew): uncut 317, in 2 parts 393.
constexpr uint64_t kTileTarget = 768;
constexpr uint64_t kTileFew = 384;
constexpr uint64_t kTileSplitMin = 512;
// Longest length that counts as it is: more than a table holds (2^30) by more than a call's
// rows, so that a position, a window and their difference from a key fit 32 bits.
constexpr uint32_t kMostLength = 3u << 29;
// Sequences of at most this many units a KV head are left to the workgroup of
// their first unit.
constexpr uint32_t kFewWhole = kFewStep / kFewKeys;

// How a call is launched.  The device's lengths are not known here: the table's
// width bounds them, and a sequence is cut into fewer parts on the device where
// it is shorter.
struct Plan {
    uint32_t few_rows = 0, few_groups = 0, few_least = 0, few_per = 0, tile_per = 0, tile_split = 1, tiles = 0;
    bool few = false, tile = false, fits = true;
    uint64_t few_o = 0, few_ml = 0, few_parts = 0, tile_o = 0, tile_ml = 0, bytes = 0;
};

// Keys of a part, so that `groups` sequences of `keys` keys make about `target`
// workgroups, and the parts of the longest sequence.  A part is no longer than all the keys
// (at most 2^30), whatever the number of groups: the kernels' positions have 32 bits.
inline uint32_t part_keys(uint64_t groups, uint64_t keys, uint64_t least, uint64_t step, uint64_t target, uint32_t* parts)
{
    uint64_t per = groups * keys / target;
    const uint64_t fewest = (keys + kMaxSplit - 1) / kMaxSplit;
    per = per > least ? per : least;
    per = per > fewest ? per : fewest;
    per = per < keys ? per : keys;
    per = (per + step - 1) / step * step;
    *parts = uint32_t((keys + per - 1) / per);
    return uint32_t(per);
}

inline Plan attend_plan(const si_paged_attention_desc& d)
{
    Plan p;
    const uint64_t group = d.q_heads / d.kv_heads, keys = uint64_t(d.table_pages) * d.page_tokens;
    const uint64_t rows = d.tokens * group;
    // One token each: one kernel.  Any mix of lengths: both, unless no
    // sequence can be long or the only one is.
    p.few = group <= kFewRows && (!d.q_starts || d.seqs > 1 || rows <= kFewRows);
    if (p.few) p.few_rows = kFewRows;
    p.tile = d.q_starts ? rows > p.few_rows : !p.few;
    const uint64_t pairs = uint64_t(d.seqs) * d.kv_heads;
    uint64_t few_groups = 0, places = 0;
    if (p.few) {
        const uint64_t units = (keys + kFewKeys - 1) / kFewKeys, fewest = (units + kMaxSplit - 2) / (kMaxSplit - 1);
        // workgroups that run at a time: 3 a CU for heads up to 64 (2 beside tiles), 2 up to 128, 1
        // (768 or 1,536 for heads of 128: 64 sequences of 8,192 keys 229 and 209 us, 512 197)
        const uint64_t at_once = d.head_dim <= 64 && !p.tile ? 768 : d.head_dim <= 128 ? 512 : 256;
        p.few_least = uint32_t(fewest > kFewWhole ? fewest : kFewWhole);
        if (d.seqs <= 64 && pairs <= at_once) {
            const uint64_t most = (pairs * units + p.few_least - 1) / p.few_least;
            few_groups = most < at_once ? most : at_once;
            places = units > kFewWhole ? 2 * few_groups : 0;
        } else {
            uint32_t parts;
            p.few_per = part_keys(pairs, keys, kFewStep, kFewStep, kFewTarget, &parts) / kFewKeys;
            few_groups = pairs * parts;
            places = parts > 1 ? few_groups : 0;
        }
    }
    if (p.tile) {
        const uint64_t tile_rows = kTileRows;
        p.tiles = uint32_t(d.q_starts ? rows / tile_rows + d.seqs
                                      : uint64_t(d.seqs) * ((group + tile_rows - 1) / tile_rows));
        // Cut only where the tiles alone leave CUs idle; sequences of the
        // few-row kernel have none.
        const uint64_t groups = (rows / tile_rows + (p.few ? 1 : d.seqs)) * d.kv_heads;
        p.tile_per = part_keys(groups, keys, groups < kTileFew ? kTileSplitMin : keys, kTileKeys, kTileTarget,
                               &p.tile_split);
        if (p.tile_split > 1) {
            // whole columns for every XCD (see the kernel's order)
            const uint32_t even = 8 / uint32_t(std::gcd(8u, d.kv_heads));
            p.tile_split = (p.tile_split + even - 1) / even * even;
        }
    }
    // (threads of a launch dimension fit 32 bits)
    const uint64_t most = (1ull << 32) / 256 - 1;
    const uint64_t tile_groups = uint64_t(p.tiles) * d.kv_heads * p.tile_split;
    p.few_groups = uint32_t(few_groups);
    p.fits = few_groups + tile_groups <= most && uint64_t(d.tokens) * d.q_heads / 4 < most;
    const auto take = [&](uint64_t n) {
        const uint64_t at = p.bytes;
        p.bytes += (n + 255) / 256 * 256;
        return at;
    };
    if (places) {
        const uint64_t n = places * kFewRows;
        p.few_o = take(n * d.head_dim * 4);
        p.few_ml = take(n * 8);
        p.few_parts = take(pairs * 8);
    }
    if (p.tile_split > 1) {
        const uint64_t n = uint64_t(p.tile_split) * d.tokens * d.q_heads;
        p.tile_o = take(n * d.head_dim * 4);
        p.tile_ml = take(n * 8);
    }
    return p;
}

}  // namespace si
