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

// Prefixes that groups of sequences share: workgroups their tiles are cut for, and the least keys of a part.
// A part's numerators (rows x dim floats, written and read again) weigh against its K and V (keys x dim x
// 4 bytes): four keys a row, of a tile's 128.  64 next tokens x 7 heads behind 8,192 keys: least 512 33.3 us, 256
// 38.5; 8 x 4 heads behind 6,144: 25.5 and 18.6.
constexpr uint64_t kShareTarget = 512;
constexpr uint32_t kShareMin = 256;
constexpr uint32_t kShareMost = 4 * kTileRows;

// Sequences of groups whose own keys are shared out evenly, 64 looked at at a time: short ones are not among them
// beyond 64, so that what is left may be few, and long (137 next tokens x 32/8 heads, one of them in a group of its
// own with 7,605 keys: 208 us in one part, 90 shared out).  More than these get parts of one length, as without groups.
// Next tokens behind 2,048 keys, with up to 100 own ones, and with one of 30,000 among up to 256, shared out and
// not: 300 x 32/8 heads 49 and 66 us, 132 and 415; 2,000 252 and 296, 471 and 811; 2,000 x 8/1 92 and 91, 179 and
// 300; but 4,000 x 8/1, whose every workgroup looks at all of them, 106 and 80, 281 and 622.
constexpr uint32_t kShareSeqs = 2048;

// Keys of a prefix for each row (of a KV head, on average) of the sequences that share it, from which on they do.
constexpr uint64_t kShareKeys = 16;

// Keys of a part of a prefix that is cut into at most `split` parts, of a group of `rows` rows a KV head.
constexpr uint32_t share_part(uint32_t keys, uint32_t split, uint64_t rows)
{
    const uint32_t even = ((keys + split - 1) / split + kTileKeys - 1) / kTileKeys * kTileKeys;
    const uint64_t four = (4 * rows + kTileKeys - 1) / kTileKeys * kTileKeys;
    const uint32_t least = four < kShareMin ? kShareMin : four < kShareMost ? uint32_t(four) : kShareMost;
    return even > least ? even : least;
}

// How a call is launched.  The device's lengths are not known here: the table's
// width bounds them, and a sequence is cut into fewer parts on the device where
// it is shorter.
struct Plan {
    uint32_t few_rows = 0, few_groups = 0, few_least = 0, few_per = 0, tile_per = 0, tile_split = 1, tiles = 0;
    bool few = false, tile = false, fits = true;
    uint64_t few_o = 0, few_ml = 0, few_parts = 0, tile_o = 0, tile_ml = 0, bytes = 0;
    uint32_t sinks = 0, share_groups = 0, share_split = 1, tile_groups = 0, alone_groups = 0;
    uint64_t share_o = 0, share_ml = 0, few_joins = 0;
};

// Keys of a part, so that `groups` sequences of `keys` keys make about `target`
// workgroups, and the parts of the longest sequence.  A part is no longer than all the keys
// (at most 2^30), whatever the number of groups: the kernels' positions have 32 bits.
inline uint32_t part_keys(uint64_t groups, uint64_t keys, uint64_t least, uint64_t step, uint64_t target, uint32_t* parts,
                          uint64_t most = kMaxSplit)
{
    uint64_t per = groups * keys / target;
    const uint64_t fewest = (keys + most - 1) / most;
    per = per > least ? per : least;
    per = per > fewest ? per : fewest;
    per = per < keys ? per : keys;
    per = (per + step - 1) / step * step;
    *parts = uint32_t((keys + per - 1) / per);
    return uint32_t(per);
}

inline Plan attend_plan(const si_paged_attention_desc& d, const si_paged_attention_more* more = nullptr)
{
    Plan p;
    const uint64_t group = d.q_heads / d.kv_heads, keys = uint64_t(d.table_pages) * d.page_tokens;
    const uint64_t rows = d.tokens * group;
    const uint64_t window = d.window < kMostLength ? d.window : 0;
    if (more && !(window && more->sinks) && !more->groups) more = nullptr;
    p.sinks = more && window ? more->sinks : 0;
    const uint32_t groups = more ? more->groups : 0;
    // A row's parts of its prefix and of its own keys are joined together; the prefix is the longer, mostly.  (21 tokens
    // of two prefixes to 20,908 keys, 8/2 heads: 48 and 16 parts 25.8 us, 32 and 32 32.5.)
    const uint64_t most_share = kMaxSplit / 4 * 3, most_parts = groups ? kMaxSplit - most_share : kMaxSplit;
    // Beside sinks a call is cut for the keys that its windows leave: a sequence's n new tokens see at most
    // window + n - 1 keys, in whole steps, and the sinks.  (Without sinks by the table alone, as ever.)
    const auto kept = [&](uint64_t n) {
        const uint64_t left = window + n + p.sinks + 3 * kTileKeys;
        return p.sinks && left < keys ? left : keys;
    };
    // One token each: one kernel.  Any mix of lengths: both, unless no
    // sequence can be long or the only one is.
    p.few = group <= kFewRows && (!d.q_starts || d.seqs > 1 || rows <= kFewRows);
    if (p.few) p.few_rows = kFewRows;
    p.tile = d.q_starts ? rows > p.few_rows : !p.few;
    const uint64_t pairs = uint64_t(d.seqs) * d.kv_heads;
    uint64_t few_groups = 0, places = 0;
    if (p.few) {
        const uint64_t keys = kept(kFewRows), unit = more ? kFewStep : kFewKeys, whole = more ? 1 : kFewWhole;
        const uint64_t units = (keys + unit - 1) / unit, fewest = (units + most_parts - 2) / (most_parts - 1);
        // workgroups that run at a time: 3 a CU for heads up to 64 (2 beside tiles), 2 up to 128, 1
        // (768 or 1,536 for heads of 128: 64 sequences of 8,192 keys 229 and 209 us, 512 197)
        const uint64_t at_once = d.head_dim <= 64 && (more || !p.tile) ? 768 : d.head_dim <= 128 ? 512 : 256;
        p.few_least = uint32_t(more ? most_parts : fewest > whole ? fewest : whole);
        if (d.seqs <= 64 ? pairs <= at_once || groups : groups && d.seqs <= kShareSeqs) {
            // (kMore: the device finds the least units of a share from the lengths)
            const uint64_t least = more ? 1 : p.few_least, most = (pairs * units + least - 1) / least;
            few_groups = most < at_once ? most : at_once;
            places = units > whole ? 2 * few_groups : 0;
        } else {
            uint32_t parts;
            p.few_per = uint32_t(part_keys(pairs, keys, kFewStep, kFewStep, kFewTarget, &parts, most_parts) / unit);
            few_groups = pairs * parts;
            places = parts > 1 ? few_groups : 0;
        }
    }
    if (p.tile) {
        const uint64_t tile_rows = kTileRows, keys = kept(d.tokens);
        p.tiles = uint32_t(d.q_starts ? rows / tile_rows + d.seqs
                                      : uint64_t(d.seqs) * ((group + tile_rows - 1) / tile_rows));
        // Cut only where the tiles alone leave CUs idle; sequences of the
        // few-row kernel have none.
        const uint64_t groups = (rows / tile_rows + (p.few ? 1 : d.seqs)) * d.kv_heads;
        // (beside sinks and prefixes shorter parts where they all run at a time: 15 tokens of two sequences x 56/8
        // heads under a window of 3,063 24.6 us, parts of 512 31.0; but 128 tokens x 32/8 under 4,096, which would
        // then take two rounds, 39 and 35)
        const uint64_t shortest = more && groups * ((keys + kTileKeys * 4 - 1) / (kTileKeys * 4)) <= 512 ? kTileKeys * 4
                                                                                                        : kTileSplitMin;
        p.tile_per = part_keys(groups, keys, groups < kTileFew ? shortest : keys, kTileKeys, kTileTarget, &p.tile_split,
                               most_parts);
        if (p.tile_split > 1) {
            // whole columns for every XCD (see the kernel's order)
            const uint32_t even = 8 / uint32_t(std::gcd(8u, d.kv_heads));
            p.tile_split = (p.tile_split + even - 1) / even * even;
        }
    }
    // Workgroups: a place for each tile and column that the call's sizes allow.  Beside sinks and shared prefixes the
    // device counts the tiles there are: all rows' full ones and one more of each sequence that is long enough, or
    // of each group of two or more.  (A multiple of the XCDs.)
    uint64_t tile_groups = uint64_t(p.tiles) * d.kv_heads * p.tile_split, share_groups = 0;
    const auto least = [](uint64_t x, uint64_t y) { return x < y ? x : y; };
    if (more && p.tile && d.q_starts)
        tile_groups = (rows / kTileRows + least(d.seqs, rows / (p.few_rows + 1))) * d.kv_heads * p.tile_split;
    if (more && p.tile) tile_groups = (tile_groups + 7) / 8 * 8;
    if (groups) {
        const uint64_t columns = (rows / kTileRows + 1) * d.kv_heads, split = (kShareTarget + columns - 1) / columns;
        p.share_split = uint32_t(split < most_share ? split : most_share);
        share_groups = (rows / kTileRows + least(groups, d.seqs / 2)) * d.kv_heads * p.share_split;
        share_groups = (share_groups + 8) / 8 * 8;
    }
    // Of many sequences the short ones go by a wave each (256 of 1 to 256 own keys x 8 KV heads behind 32,768: 336 us
    // without, 332).
    const uint64_t alone = groups && p.few && (d.seqs > 64 || p.few_per) ? (pairs + kFewWaves - 1) / kFewWaves : 0;
    // (threads of a launch dimension fit 32 bits)
    const uint64_t most = (1ull << 32) / 256 - 1;
    p.few_groups = uint32_t(few_groups);
    p.fits = share_groups + few_groups + tile_groups + alone <= most && uint64_t(d.tokens) * d.q_heads / 4 < most;
    p.tile_groups = uint32_t(tile_groups);
    p.share_groups = uint32_t(share_groups);
    p.alone_groups = uint32_t(alone);
    const auto take = [&](uint64_t n) {
        const uint64_t at = p.bytes;
        p.bytes += (n + 255) / 256 * 256;
        return at;
    };
    if (places) {
        const uint64_t n = places * kFewRows;
        p.few_o = take(n * d.head_dim * 4);
        p.few_ml = take(n * 8);
        if (!more) p.few_parts = take(pairs * 8);
    }
    if (p.tile_split > 1 || groups) {
        const uint64_t n = uint64_t(p.tile_split) * d.tokens * d.q_heads;
        p.tile_o = take(n * d.head_dim * 4);
        p.tile_ml = take(n * 8);
    }
    if (groups) {
        const uint64_t n = uint64_t(p.share_split) * d.tokens * d.q_heads;
        p.share_o = take(n * d.head_dim * 4);
        p.share_ml = take(n * 8);
    }
    if (more && p.few && p.bytes) p.few_joins = take(pairs * 16);
    return p;
}

}  // namespace si
