// Attention of new tokens over a paged KV cache:
//   out = sum_j w_j V_j / sum_j w_j,  w_j = exp(scale q.K_j - m),  m >= max_j scale q.K_j
// over the keys j a token sees, in one pass with a running m and sum, in float.
//
// Both kernels compute the transposed scores S^T = K Q^T with matrix
// instructions, so a query is a column: a lane holds one query's scores of
// several keys, the softmax statistics are per lane, and the weights already
// lie where the second product O^T = V^T P^T takes them (its contraction runs
// over keys, whose order within an instruction is free as long as V's rows
// come in the same order).  V^T comes out of LDS through transposing reads.
// The rows of one KV head are (token, query head) pairs of its group, so K and V
// are read once for all heads that share them.
//
// A sequence of at most 16 rows (a decoding step) is bound by the bytes of its K
// and V and runs in the few-row kernel; longer ones are bound by the matrix
// and vector instructions and run in tiles of 128 rows.  Keys are cut into parts where
// there are too few rows for the chip.  Beside a window and sinks the keys that are left are walked over
// without the gap between them (kMore); a prefix that a group of sequences shares is attended to in tiles of all
// the group's rows (kShare), beside each sequence's own keys.  Parts are joined by a second launch (the join by the
// workgroup that ends last was tried: its fences, which write back and drop
// whole L2s, cost one token 38 us, stores past the L2 16.9, the launch 8 + 4).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

#include "secure_infer_gpu.h"
#include "si_attend_plan.h"
#include "si_launch.h"

namespace si {

namespace {

struct AttendArgs {
    const uint16_t* q;
    uint64_t q_token, q_head;
    uint16_t* out;
    uint64_t out_token, out_head;
    float* lse;
    const uint8_t* cache_k;
    const uint8_t* cache_v;
    uint64_t slot_bytes;
    int64_t nslots;
    const int64_t* tables;
    uint64_t table_stride;
    const int64_t* kv_lens;
    const int64_t* q_starts;
    uint32_t pages, tokens, seqs, q_heads, kv_heads, group, dim, page_shift, causal, window;
    // A negative scale flips q's sign, one of 0 clears q (with a positive one here, so
    // that a masked score's -inf times it is still -inf).
    uint32_t q_keep, q_flip;
    float scale_log2;  // |scale| * log2(e): weights are powers of two
    // Sequences of at most few_rows rows (tokens * group) belong to the few-row
    // kernel, the others to the tile kernel.
    // (few_least: kMore, the parts that a sequence may have.)
    uint32_t few_rows, few_groups, few_least, few_per, tile_per, tile_split, tiles;
    // Parts of split sequences: numerators (dim floats a row) and (m, l).
    float* few_o;
    float2* few_ml;
    uint2* few_parts;  // of each sequence and KV head: place of its first part, number of parts
    float* tile_o;
    float2* tile_ml;
    // Sinks and shared prefixes (kMore and kShare).  Sequences that share one leave their own
    // keys' whole parts in tile_o's first part.
    uint32_t sinks;  // first keys seen in spite of the window (0 without one)
    uint32_t groups, share_groups, share_split;  // share_groups: workgroups for the prefixes' tiles
    const int64_t* group_starts;
    const int64_t* prefix_lens;
    float* share_o;
    float2* share_ml;
    uint4* few_joins;  // few_parts' place, and the parts of the prefix besides
    uint32_t tile_groups;  // workgroups for the tiles
    uint32_t alone_groups;  // workgroups whose waves take a short sequence's KV head each (0: none do)
};

// What a kernel's code knows of: a call without sinks and shared prefixes, one with them, and of the
// latter the pass of the groups' tokens over their prefixes.
enum Kind { kPlain = 0, kMore = 1, kShare = 2 };

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Rows up to which a whole workgroup joins one row's parts, all at once; above, groups of lanes
// join a row each, the parts one after another.  Only the first: 27 sequences of 2,105 tokens x 12
// heads 72 us in all, only the second 52; one token x 32 heads 20.0 and 20.3, 64 x 28 63.6
// and 64.3.
constexpr uint32_t kJoinRows = 2048;

// The last key of a query without one, behind every position.
constexpr int32_t kNoLast = 0x7ffffffe;

__device__ __forceinline__ bool held(int64_t e, int64_t nslots) { return e >= 0 && e < nslots; }

template <bool kBf16>
__device__ __forceinline__ float to_f32(uint16_t x)
{
    if constexpr (kBf16) return __uint_as_float(uint32_t(x) << 16);
    else return float(__builtin_bit_cast(_Float16, x));
}

template <bool kBf16>
__device__ __forceinline__ uint16_t from_f32(float x)
{
    if constexpr (kBf16) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
    else return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
}

template <bool kBf16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (kBf16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

template <bool kBf16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (kBf16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// Eight floats rounded to nearest even: the weights' one rounding, to the
// type the matrix instruction takes (relative 2^-8 / 2^-11 a weight; the sum
// they are divided by is that of the unrounded ones, in float).
template <bool kBf16>
__device__ __forceinline__ u32x4 pack8(f32x8 x)
{
    if constexpr (kBf16) return __builtin_bit_cast(u32x4, __builtin_convertvector(x, bf16x8));
    else return __builtin_bit_cast(u32x4, __builtin_convertvector(x, f16x8));
}

// LDS is addressed by byte offsets where instructions without a pointer form
// read or fill it.
typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ u32x4 read_lds(uint32_t at)
{
    return *reinterpret_cast<__attribute__((address_space(3))) const u32x4*>(at);
}

// 16 bytes a lane from memory to LDS (a wave's 1 KiB at `to`), without passing
// through registers.  Written as instructions because the compiler, which cannot tell the
// two buffers apart, would wait for them at the next read of LDS; a wait_loads() and a
// barrier stand before their data is read.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is named because it is written
__device__ __forceinline__ void to_lds(const uint8_t* p, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(p)
                 : "memory", "m0");
}
__device__ __forceinline__ void to_lds(const uint8_t* base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base)
                 : "memory", "m0");
}

#pragma clang diagnostic pop

// Everything this wave has asked memory for has arrived.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A number, a pointer that is the same in every lane, as one.
__device__ __forceinline__ uint32_t same(uint32_t x) { return uint32_t(__builtin_amdgcn_readfirstlane(int(x))); }
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p)
{
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const uint8_t*>(uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(x >> 32)))) << 32 |
                                            uint32_t(__builtin_amdgcn_readfirstlane(int(x))));
}

// Four rows of a 16-bit matrix in LDS, transposed: each 16 lanes read 4 rows x
// 16 columns (lane i: row i / 4, columns 4 (i % 4) ..) and lane i receives column
// i of the 4 rows.
__device__ __forceinline__ u32x2 read_tr(uint32_t at)
{
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at)));
}

// max / sum over lanes l, l ^ 32 and (kQuarters) l ^ 16: the lanes that hold
// the same query.
template <bool kQuarters, class F>
__device__ __forceinline__ float across(float x, F f)
{
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    if constexpr (kQuarters) {
        const uint32_t v = __float_as_uint(x);
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        x = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    return x;
}

__device__ __forceinline__ float fmax2(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float fadd2(float a, float b) { return a + b; }

// Bits 15 and 31 of the result mark infinities and NaN among eight values: an
// exponent of ones carries into the sign's place.
template <bool kBf16>
__device__ __forceinline__ uint32_t nonfinite_marks(u32x4 x)
{
    constexpr uint32_t e = kBf16 ? 0x7f807f80u : 0x7c007c00u, one = kBf16 ? 0x00800080u : 0x04000400u;
    return ((x[0] & e) + one) | ((x[1] & e) + one) | ((x[2] & e) + one) | ((x[3] & e) + one);
}

// One sequence's rows of q and positions.
struct Seq {
    uint32_t b;
    uint32_t q0, n_new;  // rows [q0, q0 + n_new) of q
    int32_t len;         // keys: its length, as far as the table goes
    int32_t base;        // position of its first new token (may be negative, or past len)
    int32_t from;        // keys below are its group's (kMore)
};

__device__ __forceinline__ uint32_t start_of(const AttendArgs& a, uint32_t b)
{
    const int64_t s = a.q_starts[b];
    return uint32_t(s < 0 ? 0 : s > int64_t(a.tokens) ? int64_t(a.tokens) : s);
}

// Rows of q from sequence b's first on.
__device__ __forceinline__ uint32_t rows_at(const AttendArgs& a, uint32_t b)
{
    return a.q_starts ? start_of(a, b) : b;
}

// Sequences [first, end) and the keys of the prefix they share, as far as the table goes: none for
// fewer than two sequences, or where they have many rows each for the prefix's keys, and are better off by
// themselves: what the parts cost grows with the rows, what is saved with the prefix.  32/8 heads of 128, behind
// 2,048 keys, together and alone: 32 sequences of 32 tokens 84 and 100 us, of 256 543 and 352; 128 of 64 545 and
// 385; behind 512, 32 of 64 86 and 61, 128 of 4 37 and 70; behind 8,192, 32 of 64 337 and 479.
struct Group {
    uint32_t first, end;
    int32_t prefix;
};



__device__ __forceinline__ Group group_at(const AttendArgs& a, uint32_t g)
{
    const int64_t lo = a.group_starts[g], hi = a.group_starts[g + 1], seqs = a.seqs;
    Group x;
    x.first = uint32_t(lo < 0 ? 0 : lo > seqs ? seqs : lo);
    x.end = uint32_t(hi < 0 ? 0 : hi > seqs ? seqs : hi);
    const int64_t most = int64_t(a.pages) << a.page_shift, n = a.prefix_lens[g];
    x.prefix = x.end < x.first + 2 || n < 0 ? 0 : int32_t(n > most ? most : n);
    const uint32_t row = rows_at(a, x.first), row_end = rows_at(a, x.end);
    const uint64_t rows = row_end > row ? uint64_t(row_end - row) * a.group : 0;
    if (uint64_t(x.prefix) * (x.end - x.first) < kShareKeys * rows) x.prefix = 0;
    return x;
}

// The group of sequence b: the last one that starts at or before it; without a prefix where there is none.
__device__ __forceinline__ Group group_of(const AttendArgs& a, uint32_t b)
{
    uint32_t at = 0;
    for (uint32_t n = a.groups; n;) {
        const uint32_t half = n / 2;
        const bool up = a.group_starts[at + half] <= int64_t(b);
        at = up ? at + half + 1 : at;
        n = up ? n - half - 1 : half;
    }
    Group g{0, 0, 0};
    if (at > 0) g = group_at(a, at - 1);
    if (b >= g.end) g.prefix = 0;
    return g;
}

// Parts of the prefix, of `from` keys, that sequence b shares.
__device__ __forceinline__ uint32_t share_parts(const AttendArgs& a, uint32_t b, int32_t from)
{
    if (from == 0) return 0;
    const Group g = group_of(a, b);
    const uint32_t row = rows_at(a, g.first), end = rows_at(a, g.end);
    const uint32_t per = share_part(uint32_t(from), a.share_split, end > row ? uint64_t(end - row) * a.group : 0);
    return (uint32_t(from) + per - 1) / per;
}

// Where a sequence of n tokens, s.n_new of them new, stands: these stand where the append puts them,
// also where the length outgrows the table.
__device__ __forceinline__ void place_seq(const AttendArgs& a, Seq& s, int64_t n)
{
    const int64_t most = int64_t(a.pages) << a.page_shift;
    s.len = int32_t(n < 0 ? 0 : n > most ? most : n);
    // (see source_of)
    if (a.window && s.len < s.from) s.from = 0;
    s.base = (n > most && n <= int64_t(kMostLength) ? int32_t(n) : s.len) - int32_t(s.n_new);
}

template <int kKind = kPlain>
__device__ __forceinline__ Seq seq_of(const AttendArgs& a, uint32_t b)
{
    Seq s;
    s.b = b;
    s.from = 0;
    if constexpr (kKind == kMore) s.from = group_of(a, b).prefix;
    s.q0 = b;
    s.n_new = 1;
    if (a.q_starts) {
        s.q0 = start_of(a, b);
        const uint32_t end = start_of(a, b + 1);
        s.n_new = end > s.q0 ? end - s.q0 : 0;
    }
    place_seq(a, s, a.kv_lens[b]);
    return s;
}

// Keys of a sequence at positions up to p.
__device__ __forceinline__ int32_t keys_up_to(const Seq& s, int32_t p)
{
    return p < 0 ? 0 : p < s.len ? p + 1 : s.len;
}

// How a sequence's keys are cut: parts of `per` keys from `lo` (a multiple of
// 64, behind every row's window).  All sequences' parts have one length, which
// keeps workgroups of ragged batches alike.  (Behind the last key: at most 63 keys, none seen.)
//
// With sinks, or a prefix that the group attends to, the keys that are left are counted without the
// gap: `head` keys from head_lo (the sinks), then those from lo on.  All three are multiples of `step`,
// so that a step's keys follow one another.
struct Cut {
    int32_t lo;
    uint32_t parts;
    int32_t head_lo, head;

    // The key in place x, and the first place with a key of at least k.
    __device__ __forceinline__ int32_t key(int32_t x) const { return x < head ? head_lo + x : lo + (x - head); }
    __device__ __forceinline__ int32_t place(int32_t k) const
    {
        return k <= head_lo ? 0 : k - head_lo < head ? k - head_lo : k <= lo ? head : k - lo + head;
    }
};

template <int kKind = kPlain>
__device__ __forceinline__ Cut cut_of(const AttendArgs& a, const Seq& s, uint32_t per, uint32_t step = kTileKeys)
{
    Cut c;
    c.lo = 0;
    c.head_lo = c.head = 0;
    if constexpr (kKind == kMore) {
        const int32_t whole = -int32_t(step);  // & whole: down to a multiple
        int32_t lo = a.window ? s.base - int32_t(a.window) + 1 : 0;
        lo = lo > s.from ? lo : s.from;
        c.lo = (lo < s.len ? lo : s.len) & whole;
        c.head_lo = s.from & whole;
        if (int32_t(a.sinks) > s.from) {
            const int32_t end = (int32_t(a.sinks) + int32_t(step) - 1) & whole;
            c.head = (end < c.lo ? end : c.lo) - c.head_lo;
            c.head = c.head > 0 ? c.head : 0;
        }
        const uint32_t span = uint32_t(c.head) + (s.len > c.lo ? uint32_t(s.len - c.lo) : 0);
        c.parts = (span + per - 1) / per;
        return c;
    }
    if (a.window && s.base - int32_t(a.window) + 1 > 0) c.lo = s.base - int32_t(a.window) + 1;
    c.lo = (c.lo < s.len ? c.lo : s.len) & ~63;
    const uint32_t span = s.len > c.lo ? uint32_t(s.len - c.lo) : 0;
    c.parts = (span + per - 1) / per;
    return c;
}

// Sums of x over the lanes up to and with this one.
__device__ __forceinline__ uint32_t sums_up_to(uint32_t x)
{
    const auto add = [&](uint32_t y) { x += y; };
    add(uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x111, 0xf, 0xf, false)));  // lane - 1, of 16
    add(uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x112, 0xf, 0xf, false)));
    add(uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x114, 0xf, 0xf, false)));
    add(uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x118, 0xf, 0xf, false)));
    add(uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x142, 0xa, 0xf, false)));  // the last lane of the 16 before
    add(uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x143, 0xc, 0xf, false)));  // lane 31, to the upper half
    return x;
}

__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b)
{
    return (a | b) >> 32 ? a / b : uint32_t(a) / uint32_t(b);
}

// The few-row kernel's units of keys: a wave's step, or a workgroup's beside sinks and shared prefixes, whose
// sequences are short: several in a workgroup follow one another, at about 4 us each.
template <int kKind>
constexpr uint32_t few_unit()
{
    return kKind == kPlain ? kFewKeys : kFewStep;
}

// Units of a KV head of a sequence for the few-row kernel.  (A
// sequence without keys has outputs all the same: one.)
template <int kKind>
__device__ __forceinline__ uint32_t few_units(const AttendArgs& a, const Seq& s)
{
    const uint32_t rows = s.n_new * a.group;
    if (rows == 0 || rows > a.few_rows) return 0;
    const uint32_t n = cut_of<kKind>(a, s, few_unit<kKind>(), kFewKeys).parts;
    if (kKind == kMore && a.alone_groups && n <= 1) return 0;  // a wave's alone
    return n ? n : 1;
}

// Up to 64 sequences, one a lane: their units one sequence after another, each KV
// head of it after the other.  Every workgroup takes `per` consecutive
// ones, wherever sequences begin and end.
struct Few {
    uint32_t units, with;  // of a KV head; their sum up to and with the lane's (at most 64 * 2^25)
    uint64_t total, per;
    Seq mine;
    // kMany: 64 sequences at a time, from s0 on; the units of those before.  (In the other kernels this
    // would spill 8 registers: 64 next tokens under a window 30.1 us, 33.0 with it.)
    uint32_t s0;
    uint64_t before;

    template <int kKind, bool kMany>
    __device__ __forceinline__ void load(const AttendArgs& a)
    {
        const uint32_t b = (threadIdx.x & 63u) + (kMany ? s0 : 0);
        units = 0;
        mine = Seq{b, 0, 0, 0, 0, 0};
        if (b < a.seqs) {
            mine = seq_of<kKind>(a, b);
            units = few_units<kKind>(a, mine);
        }
        with = sums_up_to(units);
    }
    // On to the sequences that unit `at` belongs to.
    __device__ __forceinline__ void reach(const AttendArgs& a, uint64_t at)
    {
        while (at - before >= upto(a, 63) && s0 + 64 < a.seqs) {
            before += upto(a, 63);
            s0 += 64;
            load<kMore, true>(a);
        }
    }
    template <int kKind, bool kMany>
    __device__ __forceinline__ void start(const AttendArgs& a)
    {
        s0 = 0;
        before = 0;
        load<kKind, kMany>(a);
        total = upto(a, 63);
        uint32_t longest = units;
        if (kMany && a.seqs > 64) {
            for (s0 = 64; s0 < a.seqs; s0 += 64) {
                load<kKind, kMany>(a);
                total += upto(a, 63);
                longest = units > longest ? units : longest;
            }
            s0 = 0;
            load<kKind, kMany>(a);
        }
        const uint64_t even = quotient(total + a.few_groups - 1, a.few_groups);
        uint32_t least = a.few_least;
        if constexpr (kKind == kMore) {
            // as many units a share as keep the longest sequence's parts to few_least
            uint32_t most = longest;
#pragma unroll
            for (int x = 32; x; x >>= 1) {
                const uint32_t y = uint32_t(__shfl_xor(int(most), x));
                most = y > most ? y : most;
            }
            least = (same(most) + a.few_least - 2) / (a.few_least - 1);
        }
        per = even > least ? even : least;
    }
    __device__ __forceinline__ uint64_t upto(const AttendArgs& a, int x) const  // x: the same in every lane
    {
        return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(with), x))) * a.kv_heads;
    }
};

// Rows of q before the first sequence and after the last: nothing to see.
template <bool kBf16>
__device__ void zero_unowned(const AttendArgs& a)
{
    const uint32_t first = start_of(a, 0), end = start_of(a, a.seqs);
    const uint32_t n = first + (end < a.tokens ? a.tokens - end : 0);
    for (uint32_t i = threadIdx.x; i < n * a.q_heads; i += blockDim.x) {
        const uint32_t x = i / a.q_heads, h = i - x * a.q_heads;
        const uint32_t t = x < first ? x : end + (x - first);
        for (uint32_t d = 0; d < a.dim; d += 8)
            *reinterpret_cast<u32x4*>(a.out + t * a.out_token + h * a.out_head + d) = u32x4{0, 0, 0, 0};
        if (a.lse) a.lse[uint64_t(t) * a.q_heads + h] = -INFINITY;
    }
}

// The pages of `kKeys` consecutive keys from k0 (lane j: key k0 + j % kKeys):
// fetch() reads the table, a step before resolve() needs it to say which keys
// may be read (held pages, lo <= key < hi) and where they are.
template <int kKeys>
struct Keys {
    int64_t entry;  // of the step fetched
    int32_t slot;
    uint64_t ok;    // bit j: key k0 + j

    // (No bound but the row's: the sequence's length may still be on its way.)
    __device__ __forceinline__ void fetch(const AttendArgs& a, const int64_t* table, int32_t k0)
    {
        const uint32_t page = (uint32_t(k0) + (threadIdx.x & (kKeys - 1))) >> a.page_shift;
        entry = table[page < a.pages ? page : a.pages - 1];
    }
    template <int kKind>
    __device__ __forceinline__ void resolve(const AttendArgs& a, int32_t k0, int32_t lo, int32_t hi, int32_t from)
    {
        const int32_t k = k0 + int32_t(threadIdx.x & (kKeys - 1));
        slot = int32_t(entry);
        if constexpr (kKind == kPlain)
            ok = __ballot(held(entry, a.nslots) && k >= lo && k < hi);
        else
            ok = __ballot(held(entry, a.nslots) && (k >= lo || k < int32_t(a.sinks)) && k >= from && k < hi);
        if constexpr (kKeys < 64) ok &= (1ull << kKeys) - 1ull;
    }
    // Byte offset of key k0 + j's row of KV head kvh in its cache (j: this
    // lane's choice; every lane calls it).
    __device__ __forceinline__ uint64_t row(const AttendArgs& a, int32_t k0, uint32_t j, uint32_t kvh) const
    {
        const uint32_t s = uint32_t(__shfl(slot, int(j)));
        return uint64_t(s) * a.slot_bytes +
               (uint64_t((uint32_t(k0) + j) & ((1u << a.page_shift) - 1u)) * a.kv_heads + kvh) * (a.dim * 2u);
    }
};

// The slots of 64 pages of a sequence, one a lane (-1: not held), from a
// multiple of 64 on, and of the 64 after them, read ahead.
struct Window {
    int32_t now;
    int64_t ahead;
    uint32_t base;

    __device__ __forceinline__ int64_t entry(const AttendArgs& a, const int64_t* table, uint32_t from, int32_t hi)
    {
        const uint32_t page = from + (threadIdx.x & 63u);
        return int64_t(page) << a.page_shift < hi ? table[page] : -1;
    }
    __device__ __forceinline__ void start(const AttendArgs& a, const int64_t* table, int32_t k0, int32_t hi)
    {
        base = (uint32_t(k0) >> a.page_shift) & ~63u;
        const int64_t e = entry(a, table, base, hi);
        now = held(e, a.nslots) ? int32_t(e) : -1;
        ahead = entry(a, table, base + 64, hi);
    }
    // Moves on to the page of key k (kPlain: by at most 64 pages).
    template <int kKind>
    __device__ __forceinline__ void reach(const AttendArgs& a, const int64_t* table, int32_t k, int32_t hi)
    {
        if ((uint32_t(k) >> a.page_shift) - base < 64) return;
        if constexpr (kKind != kPlain)
            if ((uint32_t(k) >> a.page_shift) - base >= 128) return start(a, table, k, hi);
        base += 64;
        now = held(ahead, a.nslots) ? int32_t(ahead) : -1;
        ahead = entry(a, table, base + 64, hi);
    }
    __device__ __forceinline__ int32_t slot(uint32_t page) const { return __builtin_amdgcn_readlane(now, int(page - base)); }
    __device__ __forceinline__ int32_t slot_of(uint32_t page) const { return __shfl(now, int(page - base) & 63); }
};

// Bits j of the keys k0 + j a query at position p sees among the `ok` ones.
__device__ __forceinline__ uint64_t seen_bits(const AttendArgs& a, uint64_t ok, int32_t k0, int32_t p)
{
    if (a.causal) {
        const int32_t last = p - k0;  // keys up to bit `last`
        ok &= last < 0 ? 0ull : last >= 63 ? ~0ull : (2ull << last) - 1ull;
    }
    if (a.window) {
        const int32_t first = p - int32_t(a.window) + 1 - k0;
        ok &= first <= 0 ? ~0ull : first > 63 ? 0ull : ~0ull << first;
    }
    return ok;
}

// Bits j of the keys k0 + j below `end`, at most 64.
__device__ __forceinline__ uint64_t bits_below(int32_t k0, int32_t end)
{
    const int32_t n = end - k0;
    return n <= 0 ? 0ull : n > 63 ? ~0ull : (1ull << n) - 1ull;
}

// The same beside sinks, for a query whose last key is `last` and whose window begins at `behind`.
__device__ __forceinline__ uint64_t seen_bits(const AttendArgs& a, uint64_t ok, int32_t k0, int32_t last, int32_t behind)
{
    return ok & bits_below(k0, last + 1) & (~bits_below(k0, behind) | bits_below(k0, int32_t(a.sinks)));
}

// Four dims of one row: the numerators divided by the weights' sum.  l = 0: no
// key had a weight.
template <bool kBf16>
__device__ __forceinline__ void store_out(const AttendArgs& a, uint32_t t, uint32_t h, uint32_t d, f32x4 acc, float l,
                                          float shift)
{
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    u32x2 v;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        v[i] = uint32_t(from_f32<kBf16>(acc[2 * i] * inv)) | uint32_t(from_f32<kBf16>(acc[2 * i + 1] * inv)) << 16;
    *reinterpret_cast<u32x2*>(a.out + t * a.out_token + h * a.out_head + d) = v;
    if (a.lse && d == 0)
        a.lse[uint64_t(t) * a.q_heads + h] = l == 0.0f ? -INFINITY : (shift + log2f(l)) * 0.69314718055994531f;
}

// One row by one wave, key by key: the keys in [from, to) that token t (at pos)
// sees, one a lane for the scores, the head's dims over the lanes for the sum
// over the values.  No key that is not seen takes part in anything: the way
// out where V holds an infinity or NaN among keys that not every row of a
// workgroup sees, which the matrix product would multiply by 0.
// (kMore and kShare: [from, to) are places of `cut`; `first` the first key of the rows' own, `last` the last.)
template <bool kBf16, int kKind>
__device__ void plain_row(const AttendArgs& a, const int64_t* table, uint32_t t, uint32_t h, uint32_t kvh, int32_t pos,
                          int32_t from, int32_t to, bool split, float* part_o, float2* part_ml, const Cut& cut,
                          int32_t first, int32_t last)
{
    const uint32_t lane = threadIdx.x & 63u;
    const int32_t behind = pos - int32_t(a.window) + 1;
    if constexpr (kKind == kPlain) {
        if (a.causal && to > pos + 1) to = pos + 1;
        if (a.window && from < behind) from = behind;
    }
    const uint16_t* q = a.q + t * a.q_token + h * a.q_head;
    const float c = a.q_keep == 0 ? 0.0f : a.q_flip ? -a.scale_log2 : a.scale_log2;
    float m = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int32_t j0 = from; j0 < to; j0 += 64) {
        int32_t j = j0 + int32_t(lane);
        bool in = j < to;
        if constexpr (kKind != kPlain) {
            j = cut.key(j);
            in = in && j >= first && j <= last && (!a.window || j >= behind || j < int32_t(a.sinks));
        }
        int64_t slot = -1;
        if (in) slot = table[j >> a.page_shift];
        const bool seen = held(slot, a.nslots);
        const uint64_t at = seen ? uint64_t(slot) * a.slot_bytes +
                                       (uint64_t(uint32_t(j) & ((1u << a.page_shift) - 1u)) * a.kv_heads + kvh) * a.dim * 2
                                 : 0;
        float s = -INFINITY;
        if (seen) {
            const uint16_t* k = reinterpret_cast<const uint16_t*>(a.cache_k + at);
            float dot = 0.0f;
            for (uint32_t d = 0; d < a.dim; ++d) dot = __builtin_fmaf(to_f32<kBf16>(q[d]), to_f32<kBf16>(k[d]), dot);
            s = dot * c;
        }
        float top = s;
#pragma unroll
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const uint64_t mask = __ballot(seen);
        if (!mask) continue;
        // (a maximum passes over NaN: where every score is, they still reach the sums)
        const float mn = fmaxf(m, top), safe = mn == -INFINITY ? 0.0f : mn;
        const float w = seen ? __builtin_amdgcn_exp2f(s - safe) : 0.0f;
        const float keep = __builtin_amdgcn_exp2f(m - safe);
        m = mn;
        float sum = w;
#pragma unroll
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
        l = __builtin_fmaf(l, keep, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= keep;
        for (int x = 0; x < 64; ++x) {
            if (!(mask >> x & 1)) continue;
            const float wx = __shfl(w, x);
            const uint16_t* v = reinterpret_cast<const uint16_t*>(a.cache_v + __shfl(at, x));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < a.dim) acc[i] = __builtin_fmaf(wx, to_f32<kBf16>(v[lane + 64 * i]), acc[i]);
        }
    }
    const float shift = m == -INFINITY ? 0.0f : m, inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t d = lane + 64 * i;
        if (d >= a.dim) continue;
        if (split) part_o[d] = acc[i];
        else a.out[t * a.out_token + h * a.out_head + d] = from_f32<kBf16>(acc[i] * inv);
    }
    if (lane != 0) return;
    if (split) *part_ml = float2{shift, l};
    else if (a.lse) a.lse[uint64_t(t) * a.q_heads + h] = l == 0.0f ? -INFINITY : (shift + log2f(l)) * 0.69314718055994531f;
}

// ---------------------------------------------------------------- few rows

// A workgroup's work is a run of 32-key units of a (sequence, KV head): each wave
// takes every fourth unit, K straight into the registers of S^T = K Q^T, V
// through the wave's own LDS.  Memory bounds it: the next unit's K and V are in
// flight while one is computed, with no barrier until the waves' results are
// joined at the end.
//
// Up to 64 sequences whose (sequence, KV head) pairs number at most the workgroups that run at
// a time (beside groups any number of pairs, and up to kShareSeqs sequences) are shared out evenly: each of those takes the same number of
// consecutive units of the whole batch, wherever sequences begin and end.  More pairs fill
// the chip by themselves and get parts of one length, a workgroup each.  64 sequences of 130
// to 8,192 keys, 28/4 heads of 128 (261 MB), inputs in the caches and not: shared evenly 55
// and 67 us, parts of one length 68 and 81; 64 of 8,192 keys (1.07 GB) 197 us, 5.5 TB/s, and 218;
// 32 sequences of heads of 256 68 and 118.  But 1,000 sequences of 20 to 300 keys
// 99 to 121 us and 59 (several short sequences one after another in a workgroup).
// K through LDS as well took 61.4 us where this way took 62.2, for twice the LDS.
template <int kDim>
constexpr int few_wave_bytes()
{
    const int v = int(kFewKeys) * (kDim + 16) * 2, o = 16 * (kDim + 4) * 4;
    return v > o ? v : o;
}
template <int kDim>
constexpr int few_lds_bytes()
{
    return int(kFewWaves) * (few_wave_bytes<kDim>() + 16 * 8 + 16);
}

// Where row r (token s.q0 + tok, query head h) of a sequence leaves its numerators and (m, l): in part
// `slot`, or, where it is the only one of a sequence that shares a prefix, in tile_o's first part.
template <int kKind>
__device__ __forceinline__ void few_place(const AttendArgs& a, const Seq& s, bool whole, uint32_t slot, uint32_t r,
                                          uint32_t tok, uint32_t h, float*& o, float2*& ml)
{
    uint64_t row = uint64_t(slot) * kFewRows + r;
    o = a.few_o;
    ml = a.few_ml;
    if constexpr (kKind == kMore) {
        if (whole) {
            row = uint64_t(s.q0 + tok) * a.q_heads + h;
            o = a.tile_o;
            ml = a.tile_ml;
        }
    }
    o += row * a.dim;
    ml += row;
}

// Units [first, first + n) of KV head kvh of a sequence whose keys are `cut`; not
// `whole`: into part `slot`.  kAlone: by this wave alone, which waits for no other.
template <bool kBf16, int kDim, int kKind, bool kAlone = false>
__device__ __forceinline__ void attend_few(const AttendArgs& a, uint8_t* lds, const Seq& s, uint32_t kvh, const Cut& cut,
                                           uint32_t first, uint32_t n, bool whole, uint32_t slot)
{
    constexpr int kSteps = kDim / 32;       // contraction steps of K Q^T
    constexpr int kOut = kDim / 16;         // 16-wide blocks of the output
    constexpr int kChunks = kDim / 8;       // 16-byte chunks of a row
    constexpr int kPitch = kDim + 16;       // LDS row of V: 32 bytes of padding spread the rows over the banks
    constexpr int kLoads = kChunks / 2;     // 16-byte loads a lane makes for 32 rows
    constexpr int kOPitch = kDim + 4;
    constexpr int kWaveBytes = few_wave_bytes<kDim>();
    float2(*const ml)[16] = reinterpret_cast<float2(*)[16]>(lds + kFewWaves * kWaveBytes);
    uint32_t* const odd = reinterpret_cast<uint32_t*>(lds + kFewWaves * (kWaveBytes + 16 * 8));
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t col = lane & 15u, quad = lane >> 4;
    const int64_t* table = a.tables + uint64_t(s.b) * a.table_stride;
    // (kMore: k0, next and hi are places of the cut)
    const auto key = [&](int32_t x) { return kKind == kPlain ? x : cut.key(x); };
    constexpr uint32_t kUnit = few_unit<kKind>();
    const int32_t k_first = (kKind == kPlain ? cut.lo : 0) + int32_t(first * kUnit);
    Keys<kFewKeys> keys;
    constexpr uint32_t kStep = kAlone ? kFewKeys : kFewStep;
    int32_t k0 = k_first + (kAlone ? 0 : int32_t(wave * kFewKeys));
    keys.fetch(a, table, key(k0));
    const uint32_t rows = s.n_new * a.group;
    const bool out = whole && (kKind == kPlain || s.from == 0);  // nothing to be joined

    // Positions: row r is token r / group; the last row's token sees most.
    const uint32_t tok = col / a.group, h = kvh * a.group + (col - tok * a.group);
    const int32_t pos = s.base + int32_t(tok);
    u32x4 q[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const uint32_t d = 32 * k + 8 * quad;
        u32x4 v{0, 0, 0, 0};
        if (col < rows && d < a.dim)
            v = *reinterpret_cast<const u32x4*>(a.q + (s.q0 + tok) * a.q_token + h * a.q_head + d);
        q[k] = (v & a.q_keep) ^ a.q_flip;
    }
    const int32_t p_last = s.base + int32_t(s.n_new) - 1;
    const int32_t hi_key = a.causal ? keys_up_to(s, p_last) : s.len;
    const int32_t hi0 = kKind == kPlain ? hi_key : cut.place(hi_key);
    const int32_t hi = hi0 < k_first + int32_t(n * kUnit) ? hi0 : k_first + int32_t(n * kUnit);
    // keys below lo are behind every row's window
    const int32_t lo = a.window ? s.base - int32_t(a.window) + 1 : 0;

    uint16_t* const vs = reinterpret_cast<uint16_t*>(lds + wave * kWaveBytes);
    const uint32_t vs_at = uint32_t(reinterpret_cast<uintptr_t>((lds_void*)lds)) + wave * kWaveBytes;
    float m = -INFINITY, l = 0.0f;
    f32x4 o[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i) o[i] = f32x4{0, 0, 0, 0};

    const int32_t last = a.causal ? pos : kNoLast;
    const int32_t behind = a.window ? pos - int32_t(a.window) + 1 : 0;

    uint32_t marks = 0;  // of V that not every row sees
    u32x4 kr[2][kSteps], vr[kLoads];
    const auto load_k = [&](int32_t k0) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const uint32_t j = 16 * y + col;
            const uint64_t off = keys.row(a, k0, j, kvh);
            const bool ok = keys.ok >> j & 1;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const uint32_t d = 32 * k + 8 * quad;
                kr[y][k] = u32x4{0, 0, 0, 0};
                if (ok && d < a.dim) kr[y][k] = *reinterpret_cast<const u32x4*>(a.cache_k + off + d * 2);
            }
        }
    };
    const auto load_v = [&](int32_t k0) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t c = 64 * i + lane, j = c / kChunks, d = (c % kChunks) * 8;
            const uint64_t off = keys.row(a, k0, j, kvh);
            vr[i] = u32x4{0, 0, 0, 0};
            if ((keys.ok >> j & 1) && d < a.dim) vr[i] = *reinterpret_cast<const u32x4*>(a.cache_v + off + d * 2);
        }
    };
    const int32_t hi_seen = kKind == kPlain ? hi : hi_key;
    if (k0 < hi) {
        keys.template resolve<kKind>(a, key(k0), lo, hi_seen, s.from);
        keys.fetch(a, table, key(k0 + int32_t(kStep)));
        load_k(key(k0));
        load_v(key(k0));
    }
    for (; k0 < hi; k0 += int32_t(kStep)) {
        const uint64_t ok = keys.ok;
        const int32_t next = k0 + int32_t(kStep);
        if (next < hi) {
            keys.template resolve<kKind>(a, key(next), lo, hi_seen, s.from);
            keys.fetch(a, table, key(next + int32_t(kStep)));
        }
        f32x4 st[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            st[y] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) st[y] = mfma16<kBf16>(kr[y][k], q[k], st[y]);
        }
        if (next < hi) load_k(key(next));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t c = 64 * i + lane;
            *reinterpret_cast<u32x4*>(vs + (c / kChunks) * kPitch + (c % kChunks) * 8) = vr[i];
        }
        // Keys that some rows see and others do not: an infinity or NaN in their
        // V would meet a weight of 0.
        const bool partial =
            s.n_new > 1 && ((a.causal && key(k0) + int32_t(kFewKeys) - 1 > s.base) ||
                            (a.window && key(k0) <= p_last - int32_t(a.window)));
        if (partial) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) marks |= nonfinite_marks<kBf16>(vr[i]);
        }
        if (next < hi) load_v(key(next));

        uint64_t seen = ok;
        if (partial) seen = kKind == kPlain ? seen_bits(a, ok, k0, pos) : seen_bits(a, ok, key(k0), last, behind);
        const uint32_t mine = uint32_t(seen) >> (4 * quad);
        float top = -INFINITY;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!(mine >> (16 * y + i) & 1)) st[y][i] = -INFINITY;
                top = fmaxf(top, st[y][i]);
            }
        top = across<true>(top, fmax2);
        const float mn = fmaxf(m, top);
        const float safe = mn == -INFINITY ? 0.0f : mn;
        const float keep = __builtin_amdgcn_exp2f((m - safe) * a.scale_log2);
        const float shift = safe * a.scale_log2;
        m = mn;
        f32x8 w;
        float sum = 0.0f;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[4 * y + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[y][i], a.scale_log2, -shift));
                sum += w[4 * y + i];
            }
        l = __builtin_fmaf(l, keep, sum);
        const u32x4 pw = pack8<kBf16>(w);
#pragma unroll
        for (int i = 0; i < kOut; ++i) o[i] *= keep;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            // keys 4 quad + 0..3 and 16 + 4 quad + 0..3 of 16 columns
            const uint32_t v = vs_at + 2 * ((4 * quad + (col >> 2)) * kPitch + 16 * i + 4 * (col & 3u));
            const u32x2 v0 = read_tr(v), v1 = read_tr(v + 32 * kPitch);
            o[i] = mfma16<kBf16>(u32x4{v0[0], v0[1], v1[0], v1[1]}, pw, o[i]);
        }
        __builtin_amdgcn_wave_barrier();
    }

    bool any_odd = false;
    if (s.n_new > 1) {
        const uint64_t any = __ballot((marks & 0x80008000u) != 0);
        if constexpr (kAlone) {
            any_odd = any != 0;
        } else {
            if (lane == 0) odd[wave] = any != 0;
            __syncthreads();
            any_odd = odd[0] | odd[1] | odd[2] | odd[3];
        }
    }
    if (any_odd) {
        for (uint32_t x = kAlone ? 0 : wave; x < rows; x += kAlone ? 1 : kFewWaves) {
            const uint32_t xt = x / a.group, xh = kvh * a.group + (x - xt * a.group);
            const int32_t xp = s.base + int32_t(xt);
            float* o_at;
            float2* ml_at;
            few_place<kKind>(a, s, whole, slot, x, xt, xh, o_at, ml_at);
            plain_row<kBf16, kKind>(a, table, s.q0 + xt, xh, kvh, xp, k_first, hi, !out, o_at, ml_at, cut, s.from,
                                    a.causal ? xp : kNoLast);
        }
        return;
    }
    // Join the waves.
    const auto all_there = [] {
        if constexpr (kAlone) __builtin_amdgcn_wave_barrier();
        else __syncthreads();
    };
    all_there();
    l = across<true>(l, fadd2);
    if (quad == 0) ml[wave][col] = float2{m, l};
    float* const ow = reinterpret_cast<float*>(lds + wave * kWaveBytes);
#pragma unroll
    for (int i = 0; i < kOut; ++i) *reinterpret_cast<f32x4*>(ow + col * kOPitch + 16 * i + 4 * quad) = o[i];
    all_there();
    const uint32_t quads = a.dim / 4;
    const int w_first = kAlone ? int(same(wave)) : 0, w_end = kAlone ? w_first + 1 : int(kFewWaves);
    for (uint32_t e = kAlone ? lane : threadIdx.x; e < rows * quads; e += kAlone ? 64 : 64 * kFewWaves) {
        const uint32_t r = e / quads, d = (e - r * quads) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = w_first; w < w_end; ++w) top = fmaxf(top, ml[w][r].x);
        const float safe = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        f32x4 acc{0, 0, 0, 0};
#pragma unroll
        for (int w = w_first; w < w_end; ++w) {
            const float2 v = ml[w][r];
            const float f = __builtin_amdgcn_exp2f((v.x - safe) * a.scale_log2);
            sum = __builtin_fmaf(v.y, f, sum);
            acc += *reinterpret_cast<const f32x4*>(lds + w * kWaveBytes + (r * kOPitch + d) * 4) * f;
        }
        const uint32_t rt = r / a.group, rh = kvh * a.group + (r - rt * a.group);
        if (!out) {
            float* o_at;
            float2* ml_at;
            few_place<kKind>(a, s, whole, slot, r, rt, rh, o_at, ml_at);
            *reinterpret_cast<f32x4*>(o_at + d) = acc;
            if (d == 0) *ml_at = float2{safe * a.scale_log2, sum};
        } else {
            store_out<kBf16>(a, s.q0 + rt, rh, d, acc, sum, safe * a.scale_log2);
        }
    }
}

// Workgroup `group`'s work (see above).  With few_per it is a part of few_per units of one
// sequence and KV head, in place `group`; without, consecutive units of all of them:
// where a part begins in an earlier workgroup it is in this one's place
// 2 group, where it goes on in the next in place 2 group + 1.
template <bool kBf16, int kDim, int kKind, bool kMany = false>
__device__ __forceinline__ void attend_few_units(const AttendArgs& a, uint8_t* lds, uint32_t group)
{
    const uint32_t few_per = a.few_per;
    if (a.q_starts && group == 0) zero_unowned<kBf16>(a);
    Few w;
    uint64_t at = 0, to = 1, per = few_per;
    if (!per) {
        w.template start<kKind, kMany>(a);
        per = w.per;
        at = group * per;
        to = at + per < w.total ? at + per : w.total;
    }
    for (bool again = false; at < to; again = true) {
        uint32_t b, kvh, first, n = 0, units = 0, place = group;
        if (few_per) {
            const uint32_t pairs = a.seqs * a.kv_heads, part = group / pairs, pair = group - part * pairs;
            b = pair / a.kv_heads;
            kvh = pair - b * a.kv_heads;
            first = part * few_per;
            at = to;
        } else {
            uint64_t here = at;
            if constexpr (kMany) {
                w.reach(a, at);
                here -= w.before;
            }
            b = uint32_t(__ffsll(static_cast<unsigned long long>(__ballot(uint64_t(w.with) * a.kv_heads > here))) - 1);
            units = uint32_t(__builtin_amdgcn_readlane(int(w.units), int(b)));
            const uint64_t in = here + uint64_t(units) * a.kv_heads - w.upto(a, int(b));
            kvh = uint32_t(quotient(in, units));
            first = uint32_t(in - uint64_t(kvh) * units);
            n = units - first;
            const bool alone = units <= (kKind == kPlain ? kFewWhole : 1);
            if (!alone && n > to - at) n = uint32_t(to - at);
            at += n;
            if (alone && first > 0) continue;
            place = 2 * group + (first == 0);
        }
        Seq s;
        if (kKind == kMore && !few_per) {
            const auto of_b = [&](uint32_t x) { return uint32_t(__builtin_amdgcn_readlane(int(x), int(b))); };
            s = Seq{kMany ? w.s0 + b : b, of_b(w.mine.q0), of_b(w.mine.n_new), int32_t(of_b(uint32_t(w.mine.len))),
                    int32_t(of_b(uint32_t(w.mine.base))), int32_t(of_b(uint32_t(w.mine.from)))};
            b = s.b;
        } else {
            s = seq_of<kKind>(a, b);
        }
        if (few_per) {
            units = few_units<kKind>(a, s);
            if (first >= units) return;
            n = units - first < few_per ? units - first : few_per;
        }
        if (kKind == kPlain && first == 0 && a.few_parts && threadIdx.x == 0)
            a.few_parts[b * a.kv_heads + kvh] = uint2{place, 1 + uint32_t(quotient(units - n + per - 1, per))};
        if (again) __syncthreads();  // the last ones' results in LDS have been read
        attend_few<kBf16, kDim, kKind>(a, lds, s, kvh, cut_of<kKind>(a, s, few_unit<kKind>(), kFewKeys), first, n, n == units, place);
        // (at the end: the join's kernel alone reads it)
        if (kKind == kMore && first == 0 && a.few_joins && threadIdx.x == 0)
            a.few_joins[b * a.kv_heads + kvh] =
                uint4{place, 1 + uint32_t(quotient(units - n + per - 1, per)), share_parts(a, b, s.from), 0};
    }
}

// Many sequences of groups: those whose own keys are at most one step of a workgroup's, a wave for each KV head of
// them, where a workgroup would wait for as long.
template <bool kBf16, int kDim>
__device__ __forceinline__ void attend_alone(const AttendArgs& a, uint8_t* lds, uint32_t group)
{
    const uint32_t pair = same(group * kFewWaves + (threadIdx.x >> 6));
    if (pair >= a.seqs * a.kv_heads) return;
    const uint32_t b = pair / a.kv_heads, kvh = pair - b * a.kv_heads;
    const Seq s = seq_of<kMore>(a, b);
    const uint32_t rows = s.n_new * a.group;
    if (rows == 0 || rows > a.few_rows) return;
    const Cut cut = cut_of<kMore>(a, s, kFewStep, kFewKeys);
    if (cut.parts > 1) return;
    attend_few<kBf16, kDim, kMore, true>(a, lds, s, kvh, cut, 0, 1, true, 0);
    if ((threadIdx.x & 63u) == 0) a.few_joins[pair] = uint4{0, 1, share_parts(a, b, s.from), 0};
}

// ---------------------------------------------------------------- tiles of rows

// One workgroup per (128 rows of a sequence and KV head, part of the keys):
// each of the 4 waves holds 32 rows, all of them share the K and V of 64 keys
// at a time, which go from memory straight to one of two LDS buffers while the
// other is used (one barrier a step).  Rows of LDS are 16-byte chunks in an order
// permuted by the row (a power of two of them), so that the rows of a read
// fall on different banks.
//
// 2,048 tokens over 32,768 keys, 64/8 heads of 128, bf16 (2.13 TFLOP): 2,040 to 2,220 us, about 1,000
// TFLOP/s; a large library matrix product reaches 1,271 on this card.  The vector instructions
// of the softmax bound it beside the matrix ones: of a step's 64 keys x 32 rows a wave spends 32 matrix
// instructions (17.2 ns each) and some 64 exponentials and 200 other vector
// instructions a lane, of which the two waves of a SIMD hide a part.  Rescaling
// numerators only past 2^8, V's order in LDS, unpredicated whole pages and matrix instructions
// first took it from 2,430 to 2,168, loads straight to LDS to 2,040.  Computing the next step's scores
// beside this one's weights gained nothing (2,341 and 2,316 then).
// The sequence of the group that token t is of (every lane its own).
__device__ __forceinline__ Seq owner_of(const AttendArgs& a, const Group& g, uint32_t t)
{
    uint32_t b = t;
    if (a.q_starts) {
        // the last one of [first, end) that starts at or before t
        uint32_t at = g.first;
        for (uint32_t n = g.end - g.first; n;) {
            const uint32_t half = n / 2;
            const bool up = start_of(a, at + half) <= t;
            at = up ? at + half + 1 : at;
            n = up ? n - half - 1 : half;
        }
        b = at > g.first ? at - 1 : g.first;
    }
    return seq_of(a, b);
}

// The sequence of the group whose row the prefix is read from: the first that is as long as the prefix, or else the
// longest, which holds every key of the prefix that any of them sees (the others may have ended).  Beside a window
// a row may have given up the pages that none of its tokens sees any more: of those as long as the prefix the one whose
// new tokens stand first, whose window holds what the others' do of the prefix.  The ones that have ended inside
// it may see keys that no such row still has, and attend to them by themselves.  The same in every wave.
__device__ __forceinline__ uint32_t source_of(const AttendArgs& a, const Group& g)
{
    uint32_t row = g.first;
    int32_t best = -1;
    for (uint32_t s0 = g.first; s0 < g.end && (a.window || best < g.prefix); s0 += 64) {
        const uint32_t s = s0 + (threadIdx.x & 63u);
        int32_t good = -1;
        if (s < g.end) {
            if (a.window) {
                const Seq x = seq_of(a, s);
                good = x.len < g.prefix ? -1 : int32_t(kMostLength) - x.base;
            } else {
                const int64_t n = a.kv_lens[s];
                good = int32_t(n < 0 ? 0 : n > g.prefix ? g.prefix : n);
            }
        }
        int32_t most = good;
#pragma unroll
        for (int x = 32; x; x >>= 1) {
            const int32_t y = __shfl_xor(most, x);
            most = y > most ? y : most;
        }
        most = int32_t(same(uint32_t(most)));
        if (most > best) {
            best = most;
            row = s0 + uint32_t(__ffsll(static_cast<unsigned long long>(__ballot(good == most)))) - 1;
        }
    }
    return same(row);
}

// The least x of the wave, and of the workgroup's waves (which all call it before anything lies in LDS).
__device__ __forceinline__ int32_t least_of(int32_t x)
{
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const int32_t y = __shfl_xor(x, d);
        x = y < x ? y : x;
    }
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int32_t tile_least(uint8_t* lds, uint32_t wave, int32_t x)
{
    int32_t* const each = reinterpret_cast<int32_t*>(lds);
    if ((threadIdx.x & 63u) == 0) each[wave] = x;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kTileWaves; ++w) {
        const int32_t y = each[w];
        x = y < x ? y : x;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(x);
}

template <int kDim>
constexpr int tile_chunks()  // 16-byte chunks of an LDS row
{
    return kDim <= 64 ? 8 : kDim <= 128 ? 16 : 32;
}
// K lies in groups of the rows that one instruction of a wave fills (1 KiB),
// with a gap after each.
template <int kDim>
constexpr int k_group_bytes()
{
    return 1024 + (tile_chunks<kDim>() == 32 ? 32 : 64);
}
template <int kDim>
constexpr int k_bytes()
{
    return int(kTileKeys) * tile_chunks<kDim>() / 64 * k_group_bytes<kDim>();
}
template <int kDim>
constexpr int tile_lds_bytes()  // two buffers of K and V
{
    return 2 * (k_bytes<kDim>() + int(kTileKeys) * tile_chunks<kDim>() * 16);
}
// kShare: and each row's last key and window's first, which would cost the registers that the loop lacks.
template <int kDim>
constexpr int share_lds_bytes()
{
    return tile_lds_bytes<kDim>() + int(kTileRows) * 8;
}

// kShare: the same over (128 rows of all the tokens of a group of sequences, part of the prefix they share);
// the rows differ in what they see of it.  Rows from r0 on of sequence s (kShare: all the tokens of group g, and
// its prefix).
template <bool kBf16, int kDim, int kKind>
__device__ __forceinline__ void tile_rows(const AttendArgs& a, uint8_t* lds, uint32_t kvh, uint32_t part, const Seq& s,
                                          uint32_t r0, const Group& g)
{
    constexpr int kChunks = tile_chunks<kDim>();
    constexpr int kPitch = kChunks * 8;  // elements of a row
    constexpr int kThreads = 64 * int(kTileWaves);
    constexpr int kLoads = int(kTileKeys) * kChunks / kThreads;
    constexpr int kRowStep = kThreads / kChunks;
    constexpr int kSteps = kDim / 16;
    constexpr int kOut = kDim / 32;
    constexpr uint32_t kBufBytes = tile_lds_bytes<kDim>() / 2, kKBytes = k_bytes<kDim>();  // of a buffer: K, then V
    constexpr uint32_t kGroup = k_group_bytes<kDim>(), kGroupRows = 64 / kChunks;
    const uint32_t lds_at = uint32_t(reinterpret_cast<uintptr_t>((lds_void*)lds));
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t col = lane & 31u, half = lane >> 5;
    const uint32_t rows = s.n_new * a.group;
    if ((kKind != kShare && rows <= a.few_rows) || r0 >= rows) return;
    const uint32_t per = kKind == kShare ? share_part(uint32_t(s.len), a.share_split, rows) : a.tile_per;
    Cut cut;
    if constexpr (kKind == kShare) {
        cut.lo = cut.head_lo = cut.head = 0;
        cut.parts = (uint32_t(s.len) + per - 1) / per;
    } else {
        cut = cut_of<kKind>(a, s, per);
    }
    if (part > 0 && part >= cut.parts) return;
    const int64_t* table = a.tables + uint64_t(s.b) * a.table_stride;

    const uint32_t r_last = (r0 + kTileRows < rows ? r0 + kTileRows : rows) - 1;
    const int32_t p_first = s.base + int32_t(r0 / a.group), p_last = s.base + int32_t(r_last / a.group);
    // of this wave's rows (rows past the last repeat it)
    const uint32_t w_first = r0 + wave * 32 < rows ? r0 + wave * 32 : r_last;
    const uint32_t w_last = w_first + 31 < r_last ? w_first + 31 : r_last;
    int32_t pw_first = s.base + int32_t(w_first / a.group), pw_last = s.base + int32_t(w_last / a.group);
    const uint32_t r = r0 + wave * 32 + col;
    const uint32_t tok = r / a.group;
    uint32_t h = kvh * a.group + (r - tok * a.group);
    const int32_t pos = s.base + int32_t(tok);
    // The last key that a row sees, and its window's first.
    const auto last_of = [&](int32_t p, int32_t len) { return a.causal ? (p < len ? p : len - 1) : len - 1; };
    const auto behind_of = [&](int32_t p) {
        return a.window && p >= int32_t(a.window) ? p - int32_t(a.window) + 1 : 0;
    };
    // (kShare: whether the sequence attends to the prefix here, see source_of)
    const auto shares = [&](const Seq& x) { return !a.window || x.len >= g.prefix; };
    int2* const limits = reinterpret_cast<int2*>(lds + tile_lds_bytes<kDim>());
    int32_t least_last = 0, most_behind = 0, least_behind = 0;  // of the wave's rows, the last of the tile's
    const auto find_limits = [&] {
        int2 x{kNoLast, 0};
        if (r < rows) {
            const Seq mine = owner_of(a, g, s.q0 + tok);
            const int32_t p = mine.base + int32_t(s.q0 + tok - mine.q0);
            x = int2{shares(mine) ? last_of(p, mine.len) : -1, behind_of(p)};
        }
        if (half == 0) limits[wave * 32 + col] = x;
        least_last = least_of(x.x);
        if (a.window) {
            most_behind = -least_of(-x.y);
            least_behind = tile_least(lds, wave, least_of(r < rows && x.x >= 0 ? x.y : kNoLast));
        }
    };
    // (kShare: the first keys' place does not wait for the rows' sequences, but where a window moves it)
    if (kKind == kShare && a.window) find_limits();
    u32x4 q[kSteps];
    const auto load_q = [&] {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const uint32_t d = 16 * k + 8 * half;
            u32x4 v{0, 0, 0, 0};
            if (r < rows && d < a.dim)
                v = *reinterpret_cast<const u32x4*>(a.q + (s.q0 + tok) * a.q_token + h * a.q_head + d);
            q[k] = (v & a.q_keep) ^ a.q_flip;
        }
    };
    if constexpr (kKind == kPlain) load_q();  // (else behind the first keys, which do not wait for it)
    // The tile's keys: from k0 (behind every row's window below lo) to hi.  kMore and kShare: k0, k_first and
    // k_end are places of the cut, from k_skip on those below k_lo are behind every window.
    const int32_t hi_all = a.causal && kKind != kShare ? keys_up_to(s, p_last) : s.len;
    int32_t hi = hi_all, lo, k_skip = 0, k_lo = 0;
    const int32_t k_first = (kKind == kPlain ? cut.lo : 0) + int32_t(part * per);
    int32_t k0 = k_first, k_end;
    if constexpr (kKind == kPlain) {
        if (hi - k0 > int32_t(per)) hi = k0 + int32_t(per);
        lo = a.window ? p_first - int32_t(a.window) + 1 : 0;
        if (a.window && lo > k0) k0 = lo & ~int32_t(kTileKeys - 1);
        k_end = hi;
    } else {
        // what some rows of the wave, and all rows of the tile, do not see
        lo = kKind == kShare ? least_behind : behind_of(p_first);
        k_skip = cut.place((int32_t(a.sinks) + int32_t(kTileKeys) - 1) & ~int32_t(kTileKeys - 1));
        k_lo = lo > cut.lo ? cut.head + ((lo - cut.lo) & ~int32_t(kTileKeys - 1)) : 0;
        k_end = cut.place(hi);
        if (k_end - k0 > int32_t(per)) k_end = k0 + int32_t(per);
        if (k0 >= k_skip && k0 < k_lo) k0 = k_lo;
    }
    const auto key = [&](int32_t x) { return kKind == kPlain ? x : cut.key(x); };
    const auto step_from = [&](int32_t x) {
        x += int32_t(kTileKeys);
        if (kKind != kPlain && x >= k_skip && x < k_lo) x = k_lo;
        return x;
    };

    const bool out = kKind != kShare && cut.parts <= 1 && s.from == 0;  // nothing to be joined
    float* const part_o = kKind == kShare ? a.share_o : a.tile_o;
    float2* const part_ml = kKind == kShare ? a.share_ml : a.tile_ml;
    f32x16 o[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    uint32_t marks = 0;  // of V that not every row sees

    // Chunk orders in LDS.  K is read a chunk of 32 rows at a time: x of a row
    // permutes its lowest chunks so that the rows of a group, and the gaps so
    // that the groups, fall on different banks; chunks 2k and 2k + 1 are read at
    // one of two addresses plus a constant.  V is read four chunks of 4 rows at
    // a time: the row's number permutes fours of chunks.  A thread fills the same
    // place of every kRowStep-th row, which all have one order.
    const auto k_order = [](uint32_t row) {
        return kGroupRows == 8 ? (row >> 1) & 3u : row & (kGroupRows - 1);
    };
    const auto v_order = [](uint32_t row) { return (row << 2) & (kChunks - 1) & 12u; };
    const auto k_place = [](uint32_t row, uint32_t c) {
        return row / kGroupRows * kGroup + row % kGroupRows * (kChunks * 16) + c * 16;
    };
    const uint32_t place = threadIdx.x % kChunks, row0 = threadIdx.x / kChunks;
    const uint32_t kv_row = a.kv_heads * a.dim * 2u;
    const bool in_page = (1u << a.page_shift) >= kTileKeys;
    // Steps of one page whose rows are read by 32-bit offsets from its first: below 2^32
    // for rows below 2^26 bytes.
    const bool by_offset = in_page && a.dim == kPitch && kv_row < (1u << 26);
    Window pages;
    // The keys of [kb, kb + 64) that may be read: on held pages, in [lo, hi).
    const auto readable = [&](int32_t kb) {
        uint64_t ok = ~0ull;
        if constexpr (kKind == kPlain) {
            if (kb < lo) ok <<= lo - kb;
        } else {
            ok &= ~bits_below(kb, s.from);
            if (kb < lo) ok &= ~bits_below(kb, lo) | bits_below(kb, int32_t(a.sinks));
        }
        if (hi - kb < 64) ok &= ~0ull >> (64 - (hi - kb));
        if (in_page) return pages.slot(uint32_t(kb) >> a.page_shift) >= 0 ? ok : 0ull;
        return ok & __ballot(pages.slot_of(uint32_t(kb + int32_t(lane)) >> a.page_shift) >= 0);
    };
    // K and V of keys [kb, kb + 64) into one buffer; the keys that may be read.
    // Whole steps go from memory to LDS; a step with keys that may not be read
    // comes through registers, which hold zeros for those.
    const uint32_t k_chunk = place ^ k_order(row0), v_chunk = place ^ v_order(row0);
    const auto fill = [&](int buf, int32_t kx) -> uint64_t {
        if (kx >= k_end) return 0;
        const int32_t kb = key(kx);
        pages.template reach<kKind>(a, table, kb, hi);
        const uint64_t ok = readable(kb);
        const uint32_t k_to = __builtin_amdgcn_readfirstlane(lds_at + buf * kBufBytes + wave * kGroup);
        const uint32_t v_to = __builtin_amdgcn_readfirstlane(lds_at + buf * kBufBytes + kKBytes + wave * 1024);
        const uint32_t in = uint32_t(kb) & ((1u << a.page_shift) - 1u);
        if (ok == ~0ull && by_offset) {
            const uint64_t page = uint64_t(uint32_t(pages.slot(uint32_t(kb) >> a.page_shift))) * a.slot_bytes +
                                  uint64_t(in) * kv_row + kvh * a.dim * 2u;
            const uint8_t* const kp = uniform(a.cache_k + page);
            const uint8_t* const vp = uniform(a.cache_v + page);
            const uint32_t row = row0 * kv_row;
            if constexpr (kKind != kPlain) {
                // (the rows' distance in the uniform base: one offset a lane and not one a load)
                const uint32_t k_at = row + k_chunk * 16, v_at = row + v_chunk * 16;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) to_lds(kp + uint64_t(i * kRowStep * kv_row), k_at, k_to + i * 4 * kGroup);
#pragma unroll
                for (int i = 0; i < kLoads; ++i) to_lds(vp + uint64_t(i * kRowStep * kv_row), v_at, v_to + i * 4096);
                return ok;
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) to_lds(kp, i * kRowStep * kv_row + row + k_chunk * 16, k_to + i * 4 * kGroup);
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                to_lds(vp, i * kRowStep * kv_row + row + v_chunk * 16, v_to + i * 4096);
            return ok;
        }
        const bool k_in = k_chunk * 8 < a.dim, v_in = v_chunk * 8 < a.dim;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t j = row0 + i * kRowStep, key = uint32_t(kb) + j;
            const uint64_t at = uint64_t(uint32_t(pages.slot_of(key >> a.page_shift))) * a.slot_bytes +
                                uint64_t(key & ((1u << a.page_shift) - 1u)) * kv_row + kvh * a.dim * 2u;
            const uint8_t* const kp = a.cache_k + at + k_chunk * 16;
            const uint8_t* const vp = a.cache_v + at + v_chunk * 16;
            if (ok == ~0ull) {
                if (k_in) to_lds(kp, k_to + i * 4 * kGroup);
                if (v_in) to_lds(vp, v_to + i * 4096);
            } else {
                const bool mine = ok >> j & 1;
                u32x4 k{0, 0, 0, 0}, v{0, 0, 0, 0};
                if (mine && k_in) k = *reinterpret_cast<const u32x4*>(kp);
                if (mine && v_in) v = *reinterpret_cast<const u32x4*>(vp);
                uint8_t* const b2 = lds + buf * kBufBytes;
                *reinterpret_cast<u32x4*>(b2 + k_place(j, place)) = k;
                *reinterpret_cast<u32x4*>(b2 + kKBytes + (j * kChunks + place) * 16) = v;
            }
        }
        return ok;
    };

    // The chunks past the head dim stay zero.
    if (a.dim < kPitch) {
        for (uint32_t x = threadIdx.x; x < kTileKeys * kChunks; x += kThreads) {
            const uint32_t j = x / kChunks, c = x % kChunks;
            for (int b2 = 0; b2 < 2; ++b2) {
                uint8_t* const b3 = lds + b2 * kBufBytes;
                if ((c ^ k_order(j)) * 8 >= a.dim) *reinterpret_cast<u32x4*>(b3 + k_place(j, c)) = u32x4{0, 0, 0, 0};
                if ((c ^ v_order(j)) * 8 >= a.dim) *reinterpret_cast<u32x4*>(b3 + kKBytes + x * 16) = u32x4{0, 0, 0, 0};
            }
        }
        __syncthreads();
    }
    // Where this lane reads: row col of K at chunk `half` of each pair, even and
    // odd k; the 4 rows of V at each 32 columns.
    uint32_t k_read[2], v_read[kOut];
#pragma unroll
    for (int x = 0; x < 2; ++x) k_read[x] = lds_at + k_place(col, (2 * x + half) ^ k_order(col));
    const uint32_t v_row = 4 * half + ((lane & 15u) >> 2);
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
        const uint32_t d = 32 * i + (lane & 16u) + 4 * (lane & 3u);
        v_read[i] = lds_at + kKBytes + v_row * (kChunks * 16) + (((d / 8) ^ v_order(v_row)) * 8 + d % 8) * 2;
    }
    pages.start(a, table, key(k0), hi);
    uint64_t ok_next = fill(0, k0);
    if constexpr (kKind != kPlain) load_q();
    if constexpr (kKind == kShare) {
        if (!a.window) find_limits();
        pw_first = least_last;
        pw_last = most_behind + int32_t(a.window) - 1;
    }
    int buf = 0;
    for (; k0 < k_end; k0 = step_from(k0)) {
        // This step's K and V are there, and every wave is done with the other
        // buffer: the next step's go into it.
        wait_loads();
        __syncthreads();
        const uint64_t ok = ok_next;
        ok_next = fill(1 - buf, step_from(k0));
        const uint32_t in_buf = buf * kBufBytes;
        const uint32_t k_even = k_read[0] + in_buf, k_odd = k_read[1] + in_buf;
        // The matrix instructions go first where two workgroups' waves meet on
        // a SIMD, so that one's weights are formed during the other's products.
        __builtin_amdgcn_s_setprio(1);
        f32x16 st[2];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) st[y][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const u32x4 kf = read_lds((k % 2 ? k_odd : k_even) + k / 2 * 64 + y * (32 / kGroupRows * kGroup));
                st[y] = mfma32<kBf16>(kf, q[k], st[y]);
            }
        __builtin_amdgcn_s_setprio(0);
        // Keys that some of the wave's rows see and others do not.
        const bool partial = ((kKind == kShare || a.causal) && key(k0) + int32_t(kTileKeys) - 1 > pw_first) ||
                             (a.window && key(k0) <= pw_last - int32_t(a.window));
        uint64_t seen = ok;
        if (partial || ok != ~0ull) {
            if (partial) {
                if constexpr (kKind == kPlain) {
                    seen = seen_bits(a, ok, k0, pos);
                } else if constexpr (kKind == kMore) {
                    seen = seen_bits(a, ok, key(k0), a.causal ? pos : kNoLast, behind_of(pos));
                } else {
                    const int2 x = limits[wave * 32 + col];
                    seen = seen_bits(a, ok, key(k0), x.x, x.y);
                }
            }
            const uint64_t mine = seen >> (4 * half);
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(mine >> (32 * y + 8 * (e / 4) + e % 4) & 1)) st[y][e] = -INFINITY;
        }
        float top = st[0][0];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, st[y][e]);
        top = across<false>(top, fmax2);
        // m follows the maximum only where a weight would pass 2^8 (float sums
        // and rounded weights keep their relative error), so that the
        // numerators are seldom rescaled.
        if (__ballot((top - m) * a.scale_log2 > 8.0f)) {
            const float mn = fmaxf(m, top);
            const float keep = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
            l *= keep;
#pragma unroll
            for (int i = 0; i < kOut; ++i) o[i] *= keep;
            m = mn;
        }
        const float shift = m == -INFINITY ? 0.0f : m * a.scale_log2;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                st[y][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[y][e], a.scale_log2, -shift));
                sum[e % 4] += st[y][e];
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        const auto v_frag = [&](int y, int i) {
            const uint32_t at = v_read[i] + in_buf + y * 16 * (kChunks * 16);
            const u32x2 v0 = read_tr(at), v1 = read_tr(at + 8 * (kChunks * 16));
            return u32x4{v0[0], v0[1], v1[0], v1[1]};
        };
        const auto weights = [&](int y) {
            f32x8 w;
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = st[y / 2][8 * (y % 2) + e];
            return pack8<kBf16>(w);
        };
        __builtin_amdgcn_s_setprio(1);
        if (!partial) {
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const u32x4 pw = weights(y);
#pragma unroll
                for (int i = 0; i < kOut; ++i) o[i] = mfma32<kBf16>(v_frag(y, i), pw, o[i]);
            }
        } else {
            // Not every row sees these keys: an infinity or NaN in their V would
            // meet a weight of 0.
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const u32x4 pw = weights(y);
#pragma unroll
                for (int i = 0; i < kOut; ++i) {
                    const u32x4 v = v_frag(y, i);
                    marks |= nonfinite_marks<kBf16>(v);
                    o[i] = mfma32<kBf16>(v, pw, o[i]);
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        buf = 1 - buf;
    }

    if (__ballot((marks & 0x80008000u) != 0)) {
        for (uint32_t x = r0 + wave * 32; x < r0 + wave * 32 + 32 && x < rows; ++x) {
            const uint32_t xt = x / a.group, xh = kvh * a.group + (x - xt * a.group);
            const uint64_t row = (uint64_t(part) * a.tokens + s.q0 + xt) * a.q_heads + xh;
            int32_t xp = s.base + int32_t(xt), x_last = a.causal ? xp : kNoLast;
            if constexpr (kKind == kShare) {
                const Seq mine = owner_of(a, g, s.q0 + xt);
                xp = mine.base + int32_t(s.q0 + xt - mine.q0);
                x_last = shares(mine) ? last_of(xp, mine.len) : -1;
            }
            plain_row<kBf16, kKind>(a, table, s.q0 + xt, xh, kvh, xp, k_first, k_end, !out, part_o + row * a.dim,
                                    part_ml + row, cut, s.from, x_last);
        }
        return;
    }
    l = across<false>(l, fadd2);
    // (kShare: worked out again, for the loop's registers)
    uint32_t thread = threadIdx.x;
    if constexpr (kKind == kShare) asm volatile("" : "+v"(thread));
    const uint32_t r_out = kKind == kShare ? r0 + (thread >> 6) * 32 + (thread & 31u) : r;
    if (r_out >= rows) return;
    const uint32_t tok_out = kKind == kShare ? r_out / a.group : tok;
    const uint32_t t = s.q0 + tok_out;
    if constexpr (kKind == kShare) h = kvh * a.group + (r_out - tok_out * a.group);
    const float shift = m == -INFINITY ? 0.0f : m * a.scale_log2;
    if (!out) {
        const uint64_t row = (uint64_t(part) * a.tokens + t) * a.q_heads + h;
        if (half == 0) part_ml[row] = float2{shift, l};
        // (numerators without a weight are not read)
        if (kKind != kPlain && l == 0.0f) return;
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const uint32_t d = 32 * i + 2 * e + 4 * half;
                if (d < a.dim)
                    *reinterpret_cast<f32x4*>(part_o + row * a.dim + d) =
                        f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
            }
    } else {
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const uint32_t d = 32 * i + 2 * e + 4 * half;
                if (d < a.dim)
                    store_out<kBf16>(a, t, h, d, f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]}, l, shift);
            }
    }
}

// Which (column, tile) workgroup `group` of `groups` takes.  A column is one KV head's part of the keys, over all
// tiles.  Workgroup i runs on XCD i % 8: whole columns go to one XCD, whose L2 then holds their
// K and V, dealt out back and forth, as the parts that only long sequences
// have come last; where the columns do not fill the XCDs evenly, each XCD
// takes an eighth of the list.
__device__ __forceinline__ void deal_tile(uint32_t group, uint32_t groups, uint32_t tiles, uint32_t& column, uint32_t& tile)
{
    const uint32_t xcd = group % 8, nth = group / 8;
    const uint32_t columns = groups / tiles;
    if (columns % 8 == 0) {
        const uint32_t deal = nth / tiles;
        column = 8 * deal + (deal % 2 ? 7 - xcd : xcd);
        tile = nth % tiles;
    } else {
        const uint32_t x8 = groups / 8, r8 = groups % 8;
        const uint32_t w = xcd * x8 + (xcd < r8 ? xcd : r8) + nth;
        column = w / tiles;
        tile = w % tiles;
    }
    tile = tiles - 1 - tile;  // the last tiles see most keys: first
}

template <bool kBf16, int kDim>
__device__ __forceinline__ void attend_tile(const AttendArgs& a, uint8_t* lds, uint32_t group, uint32_t groups)
{
    const uint32_t lane = threadIdx.x & 63u;
    if (a.q_starts && a.few_rows == 0 && group == 0) zero_unowned<kBf16>(a);
    uint32_t column, tile;
    deal_tile(group, groups, a.tiles, column, tile);
    const uint32_t kvh = column % a.kv_heads, part = column / a.kv_heads;

    // Sequence b's tiles start at floor(q_starts[b] * group / rows) + b, which
    // leaves it at least the tiles it needs.
    uint32_t b = tile;
    uint32_t first_tile = tile;
    if (a.q_starts) {
        uint32_t at_or_before = 0;
        for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
            const uint32_t s = s0 + lane;
            const uint32_t f = s < a.seqs ? uint32_t(uint64_t(start_of(a, s)) * a.group / kTileRows) + s : 0;
            const uint64_t le = __ballot(s < a.seqs && f <= tile);
            at_or_before += __popcll(le);
            if (le) first_tile = __builtin_amdgcn_readfirstlane(__shfl(f, 63 - __clzll(le)));
        }
        if (at_or_before == 0) return;
        b = at_or_before - 1;
    } else {
        b = tile / ((a.group + kTileRows - 1) / kTileRows);
        first_tile = b * ((a.group + kTileRows - 1) / kTileRows);
    }
    tile_rows<kBf16, kDim, kPlain>(a, lds, kvh, part, seq_of(a, b), (tile - first_tile) * kTileRows, Group{b, b + 1, 0});
}

// kMore and kShare: the tiles that there are, counted, one to a workgroup; the workgroups behind them leave.
template <bool kBf16, int kDim, int kKind>
__device__ __forceinline__ void attend_tiles(const AttendArgs& a, uint8_t* lds, uint32_t group)
{
    const uint32_t lane = threadIdx.x & 63u;
    if (kKind == kMore && a.q_starts && a.few_rows == 0 && group == 0) zero_unowned<kBf16>(a);
    const uint32_t n = kKind == kShare ? a.groups : a.seqs;
    // of the lane's sequence or group of 64: its tiles, their sum up to and with it
    Group mine{0, 0, 0};
    uint32_t tiles = 0, with = 0, from = 0, end = 0;
    int64_t length = 0;
    const auto count = [&](uint32_t s0) {
        const uint32_t s = s0 + lane;
        uint32_t least = 0;
        from = end = 0;
        if (s < n) {
            if constexpr (kKind == kShare) {
                mine = group_at(a, s);
                if (mine.prefix > 0) {
                    from = rows_at(a, mine.first);
                    end = rows_at(a, mine.end);
                }
            } else {
                from = rows_at(a, s);
                end = rows_at(a, s + 1);
                length = a.kv_lens[s];
                least = a.few_rows;
            }
        }
        const uint32_t rows = end > from ? (end - from) * a.group : 0;
        tiles = rows > least ? (rows + kTileRows - 1) / kTileRows : 0;
        with = sums_up_to(tiles);
        return uint32_t(__builtin_amdgcn_readlane(int(with), 63));
    };
    uint32_t total = count(0);
    for (uint32_t s0 = 64; s0 < n; s0 += 64) total += count(s0);
    // (tiles of a call fit 32 bits with their columns: the host's count of them does)
    const uint32_t groups = total * a.kv_heads * (kKind == kShare ? a.share_split : a.tile_split);
    if (group >= groups) return;
    uint32_t column, tile;
    deal_tile(group, groups, total, column, tile);
    uint32_t sum = 0, s0 = 0;
    uint64_t past = 0;
    for (; s0 < n; s0 += 64) {
        const uint32_t here = n > 64 ? count(s0) : total;
        past = __ballot(sum + with > tile);
        if (past) break;
        sum += here;
    }
    if (!past) return;  // (there is one, unless the starts are written meanwhile)
    const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
    const uint32_t before = sum + uint32_t(__builtin_amdgcn_readlane(int(with - tiles), at));
    // (the lane's own, without another look at memory)
    const auto of_at = [&](uint32_t x) { return uint32_t(__builtin_amdgcn_readlane(int(x), at)); };
    Group g{0, 0, 0};
    Seq seq;
    seq.q0 = of_at(from);
    seq.n_new = of_at(end) > seq.q0 ? of_at(end) - seq.q0 : 0;
    if constexpr (kKind == kShare) {
        g = Group{of_at(mine.first), of_at(mine.end), int32_t(of_at(uint32_t(mine.prefix)))};
        seq.b = source_of(a, g);
        seq.len = g.prefix;
        seq.base = seq.from = 0;
    } else {
        seq.b = s0 + uint32_t(at);
        seq.from = a.groups ? group_of(a, seq.b).prefix : 0;
        place_seq(a, seq, int64_t(uint64_t(of_at(uint32_t(uint64_t(length) >> 32))) << 32 | of_at(uint32_t(length))));
    }
    tile_rows<kBf16, kDim, kKind>(a, lds, column % a.kv_heads, column / a.kv_heads, seq, (tile - before) * kTileRows, g);
}

// ---------------------------------------------------------------- kernels

// (Three waves a SIMD for heads up to 64: tiles over 32,768 keys 365 us, two 442; for heads of 128 the
// few-row kernel spills: 125 us where two take 54.)
template <bool kBf16, int kDim, int kKind>
__global__ __launch_bounds__(256, kDim > 128 ? 1 : kDim > 64 ? 2 : 3) void attend_few_kernel(AttendArgs a)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[few_lds_bytes<kDim>()];
    attend_few_units<kBf16, kDim, kKind>(a, lds, blockIdx.x);
}

template <bool kBf16, int kDim, int kKind>
__global__ __launch_bounds__(256, kDim > 128 ? 1 : kDim > 64 ? 2 : 3) void attend_tile_kernel(AttendArgs a)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[tile_lds_bytes<kDim>()];
    if constexpr (kKind == kPlain) attend_tile<kBf16, kDim>(a, lds, blockIdx.x, gridDim.x);
    else attend_tiles<kBf16, kDim, kKind>(a, lds, blockIdx.x);
}

// Both kinds of sequences in one launch: the tiles' workgroups first, which take
// longest, and the few-row ones beside and after them.
template <int kDim>
constexpr int mixed_lds_bytes()
{
    return tile_lds_bytes<kDim>() > few_lds_bytes<kDim>() ? tile_lds_bytes<kDim>() : few_lds_bytes<kDim>();
}

template <bool kBf16, int kDim, int kKind>
__global__ __launch_bounds__(256, kDim > 128 ? 1 : kDim <= 64 && kKind == kMore ? 3 : 2) void attend_mixed_kernel(AttendArgs a)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[mixed_lds_bytes<kDim>()];
    const uint32_t tiles = kKind == kPlain ? a.tiles * a.kv_heads * a.tile_split : a.tile_groups;
    if (blockIdx.x < tiles) {
        if constexpr (kKind == kPlain) attend_tile<kBf16, kDim>(a, lds, blockIdx.x, tiles);
        else attend_tiles<kBf16, kDim, kKind>(a, lds, blockIdx.x);
    } else {
        attend_few_units<kBf16, kDim, kKind>(a, lds, blockIdx.x - tiles);
    }
}

// The groups' prefixes first, then each sequence's own keys.  (Three waves a SIMD for heads up to 64, here and in
// kMore's mixed kernel: 45 sequences of 4 tokens, 12/4 heads, behind seven prefixes 27.2 us, two 31.5.)
//
// Own tiles, of which there may be none, come last.  kMany: short sequences by a wave each; a kernel
// of its own, as more code makes the others slower to start (20.4 us where this takes 18.2, eight samples).
template <bool kBf16, int kDim, bool kMany>
__global__ __launch_bounds__(256, kDim > 128 ? 1 : kDim <= 64 ? 3 : 2) void attend_shared_kernel(AttendArgs a)
{
    constexpr int kBytes = share_lds_bytes<kDim>() > few_lds_bytes<kDim>() ? share_lds_bytes<kDim>() : few_lds_bytes<kDim>();
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBytes];
    uint32_t group = blockIdx.x;
    if (group < a.share_groups) return attend_tiles<kBf16, kDim, kShare>(a, lds, group);
    group -= a.share_groups;
    if constexpr (kMany) {
        if (group < a.alone_groups) return attend_alone<kBf16, kDim>(a, lds, group);
        group -= a.alone_groups;
    }
    if (group < a.few_groups) return attend_few_units<kBf16, kDim, kMore, kMany>(a, lds, group);
    attend_tiles<kBf16, kDim, kMore>(a, lds, group - a.few_groups);
}

// ---------------------------------------------------------------- parts joined

// Where a row's parts are, and how many: of its prefix (kMore: the first `share` ones), then of
// its sequence's own keys.
struct Parts {
    const float2* ml;
    const float* o;
    uint64_t step;  // rows from one part to the next
    uint32_t back;  // rows that the parts after the first lie before that
    uint32_t parts;
    uint32_t share;
    uint64_t row0;  // of the prefix's first part

    __device__ __forceinline__ uint64_t row(uint32_t n) const { return n * step - (n == 0 ? 0 : back); }
    template <int kKind>
    __device__ __forceinline__ float2 sums(const AttendArgs& a, uint32_t n) const
    {
        if (kKind == kMore && n < share) return a.share_ml[row0 + n * uint64_t(a.tokens) * a.q_heads];
        return ml[row(n - share)];
    }
    template <int kKind>
    __device__ __forceinline__ f32x4 four(const AttendArgs& a, uint32_t n, uint32_t d) const
    {
        if (kKind == kMore && n < share)
            return *reinterpret_cast<const f32x4*>(a.share_o + (row0 + n * uint64_t(a.tokens) * a.q_heads) * a.dim + d);
        return *reinterpret_cast<const f32x4*>(o + row(n - share) * a.dim + d);
    }
};

// The parts of a few-row sequence's row: `place` and `parts` as its first workgroup left them.
__device__ __forceinline__ void few_rows_of(const AttendArgs& a, Parts& p, uint32_t place, uint32_t parts, uint32_t r)
{
    const uint64_t row = uint64_t(place) * kFewRows + r;
    p.parts = parts;
    // a place a workgroup apart: first ones with few_per; else see attend_few_units
    p.step = a.few_per ? uint64_t(a.seqs) * a.kv_heads * kFewRows : 2 * kFewRows;
    p.back = a.few_per ? 0 : kFewRows;
    p.ml = a.few_ml + row;
    p.o = a.few_o + row * a.dim;
}

__device__ __forceinline__ void tile_rows_of(const AttendArgs& a, Parts& p, uint32_t parts, uint32_t t, uint32_t h)
{
    const uint64_t row = uint64_t(t) * a.q_heads + h;
    p.parts = parts;
    p.step = uint64_t(a.tokens) * a.q_heads;
    p.ml = a.tile_ml + row;
    p.o = a.tile_o + row * a.dim;
}

template <int kKind>
__device__ __forceinline__ Parts parts_of(const AttendArgs& a, uint32_t b, uint32_t t, uint32_t h)
{
    Parts p{nullptr, nullptr, 0, 0, 0, 0, 0};
    const uint32_t kvh = h / a.group;
    if constexpr (kKind == kPlain) {
        // (nothing the few-row kernel wrote where the sequence is not its)
        const uint2 few_parts = a.few_parts ? a.few_parts[uint64_t(b) * a.kv_heads + kvh] : uint2{0, 0};
        const Seq s = seq_of(a, b);
        if (t < s.q0 || t >= s.q0 + s.n_new) return p;
        if (s.n_new * a.group <= a.few_rows) few_rows_of(a, p, few_parts.x, few_parts.y, (t - s.q0) * a.group + (h - kvh * a.group));
        else tile_rows_of(a, p, cut_of(a, s, a.tile_per).parts, t, h);
        return p;
    }
    // A few-row sequence's parts are in few_joins: nothing else is waited for.
    const uint4 joins = a.few_joins ? a.few_joins[uint64_t(b) * a.kv_heads + kvh] : uint4{0, 0, 0, 0};
    const uint32_t q0 = rows_at(a, b), end = rows_at(a, b + 1);
    if (t < q0 || t >= end) return p;
    if ((end - q0) * a.group <= a.few_rows) {
        if (joins.y > 1) few_rows_of(a, p, joins.x, joins.y, (t - q0) * a.group + (h - kvh * a.group));
        else tile_rows_of(a, p, 1, t, h);
        p.share = joins.z;
    } else {
        const Seq s = seq_of<kKind>(a, b);
        const uint32_t parts = cut_of<kKind>(a, s, a.tile_per).parts;
        tile_rows_of(a, p, parts ? parts : 1, t, h);
        p.share = share_parts(a, b, s.from);
    }
    p.row0 = uint64_t(t) * a.q_heads + h;
    p.parts += p.share;
    return p;
}

// The last sequence that starts at or before row t (0 where there is none).
__device__ __forceinline__ uint32_t seq_at(const AttendArgs& a, uint32_t t)
{
    if (!a.q_starts) return t;
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t n = 0;
    for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64)
        n += __popcll(__ballot(s0 + lane < a.seqs && start_of(a, s0 + lane) <= t));
    return n ? n - 1 : 0;
}

// Lanes that hold one row, 4 dims a lane.
template <int kDim>
constexpr uint32_t row_lanes()
{
    return kDim <= 64 ? 16 : kDim <= 128 ? 32 : 64;
}

// Many rows: row_lanes lanes per (token, query head), the parts one after
// another.
template <bool kBf16, int kDim, int kKind>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a)
{
    constexpr uint32_t kLanes = row_lanes<kDim>(), kRows = 64 / kLanes, kHeld = kMaxSplit / kLanes, kAhead = 4;
    const uint32_t lane = threadIdx.x & 63u, sub = lane % kLanes, d = sub * 4;
    const uint32_t first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kRows, rows = a.tokens * a.q_heads;
    if (first >= rows) return;
    const uint32_t th = first + lane / kLanes;
    const uint32_t t = th / a.q_heads, h = th - t * a.q_heads;
    // (rows of a wave may belong to several sequences)
    uint32_t b = seq_at(a, first / a.q_heads);
    if (a.q_starts) {
        while (b + 1 < a.seqs && start_of(a, b + 1) <= t) ++b;
    } else {
        b = t < a.seqs ? t : a.seqs - 1;
    }
    Parts p{nullptr, nullptr, 0, 0, 0, 0, 0};
    if (th < rows) p = parts_of<kKind>(a, b, t, h);
    const uint32_t parts = p.parts > 1 ? p.parts : 0;
    if (__ballot(parts != 0) == 0) return;
    float2 v[kHeld];
    float top = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) {
        v[i] = float2{0.0f, 0.0f};
        if (i * kLanes + sub < parts) v[i] = p.template sums<kKind>(a, i * kLanes + sub);
        if (v[i].y != 0.0f) top = fmaxf(top, v[i].x);
    }
#pragma unroll
    for (uint32_t x = kLanes / 2; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, int(x)));
    if (top == -INFINITY) top = 0.0f;
    float f[kHeld], sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) {
        f[i] = v[i].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(v[i].x - top);
        sum = __builtin_fmaf(v[i].y, f[i], sum);
    }
#pragma unroll
    for (uint32_t x = kLanes / 2; x; x >>= 1) sum += __shfl_xor(sum, int(x));
    f32x4 acc{0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) {
        for (uint32_t p0 = 0; p0 < kLanes; p0 += kAhead) {
            if (__ballot(i * kLanes + p0 < parts) == 0) break;
            f32x4 part[kAhead];
#pragma unroll
            for (uint32_t x = 0; x < kAhead; ++x) {
                const uint32_t n = i * kLanes + p0 + x;
                part[x] = f32x4{0, 0, 0, 0};
                bool weighs = n < parts;
                if constexpr (kKind == kMore) {
                    const float fx = __shfl(f[i], int((lane & ~(kLanes - 1)) + p0 + x));
                    weighs = weighs && fx != 0.0f;
                }
                if (weighs && d < a.dim) part[x] = p.template four<kKind>(a, n, d);
            }
#pragma unroll
            for (uint32_t x = 0; x < kAhead; ++x) {
                const float fx = __shfl(f[i], int((lane & ~(kLanes - 1)) + p0 + x));
                if (fx != 0.0f) acc += part[x] * fx;
            }
        }
    }
    if (parts && d < a.dim) store_out<kBf16>(a, t, h, d, acc, sum, top);
}

// Few rows: a workgroup per (token, query head), its groups of row_lanes lanes
// taking every so-many-th part each, summed in their order at the end.
template <bool kBf16, int kDim, int kKind>
__global__ __launch_bounds__(256, 6) void attend_join_row_kernel(AttendArgs a)
{
    constexpr uint32_t kLanes = row_lanes<kDim>(), kStride = 256 / kLanes, kMost = kMaxSplit / kStride;
    __shared__ f32x4 sums[4][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t t = blockIdx.x / a.q_heads, h = blockIdx.x - t * a.q_heads;
    const uint32_t b = seq_at(a, t);
    const Parts p = parts_of<kKind>(a, b, t, h);
    if (p.parts <= 1) return;
    float2 v{0.0f, 0.0f};
    if (lane < p.parts) v = p.template sums<kKind>(a, lane);
    const uint32_t which = threadIdx.x / kLanes, d = lane % kLanes * 4;
    f32x4 part[kMost];
#pragma unroll
    for (uint32_t i = 0; i < kMost; ++i) {
        part[i] = f32x4{0, 0, 0, 0};
        const uint32_t n = which + i * kStride;
        if (n < p.parts && d < a.dim) part[i] = p.template four<kKind>(a, n, d);
    }
    float top = v.y == 0.0f ? -INFINITY : v.x;
#pragma unroll
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    if (top == -INFINITY) top = 0.0f;
    const float f = v.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(v.x - top);
    float sum = v.y * f;
#pragma unroll
    for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
    f32x4 acc{0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < kMost; ++i) {
        const float fx = __shfl(f, int(which + i * kStride));
        if (fx != 0.0f) acc += part[i] * fx;
    }
#pragma unroll
    for (uint32_t x = kLanes; x < 64; x <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], int(x));
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave != 0) return;
    acc = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    if (lane < kLanes && d < a.dim) store_out<kBf16>(a, t, h, d, acc, sum, top);
}

bool aligned(const void* p, uint64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

bool attend_ok(const si_paged_attention_desc& d)
{
    if (!d.q || !d.out || !d.cache_k || !d.cache_v || !d.tables || !d.kv_lens) return false;
    if (!d.tokens || !d.seqs || !d.q_heads || !d.kv_heads || d.q_heads % d.kv_heads || !d.table_pages) return false;
    if (!d.q_starts && d.tokens != d.seqs) return false;
    if (uint64_t(d.tokens) * d.q_heads >= (1ull << 26) || d.seqs >= (1u << 26)) return false;
    if (!d.head_dim || d.head_dim % 8 || d.head_dim > 256 || d.dtype > SI_DTYPE_FP16) return false;
    if (d.page_tokens < 8 || d.page_tokens > 32768 || (d.page_tokens & (d.page_tokens - 1))) return false;
    if (uint64_t(d.table_pages) * d.page_tokens > (1ull << 30)) return false;
    if (!d.nslots || d.nslots >= (1ull << 31)) return false;
    const uint64_t row = 2ull * d.kv_heads * d.head_dim;
    if (row >= (1ull << 30) || d.slot_bytes % 16 || d.slot_bytes < row * d.page_tokens) return false;
    if ((d.q_token_stride | d.q_head_stride | d.out_token_stride | d.out_head_stride) % 8) return false;
    if (!std::isfinite(d.scale)) return false;
    for (const void* p : {d.q, static_cast<const void*>(d.out), d.cache_k, d.cache_v})
        if (!aligned(p, 16)) return false;
    return true;
}

template <bool kBf16, int kDim, int kKind>
hipError_t attend_launch(hipStream_t stream, const AttendArgs& a, const Plan& p)
{
    const dim3 block(256);
    const uint32_t tiles = p.tile_groups;
    hipError_t e;
    if (p.share_groups) {
        const dim3 grid(p.share_groups + p.alone_groups + p.few_groups + tiles);
        e = p.alone_groups ? launch(attend_shared_kernel<kBf16, kDim, true>, grid, block, stream, a)
                      : launch(attend_shared_kernel<kBf16, kDim, false>, grid, block, stream, a);
    } else if (p.few && p.tile) {
        e = launch(attend_mixed_kernel<kBf16, kDim, kKind>, dim3(tiles + p.few_groups), block, stream, a);
    } else if (p.few) {
        e = launch(attend_few_kernel<kBf16, kDim, kKind>, dim3(p.few_groups), block, stream, a);
    } else {
        e = launch(attend_tile_kernel<kBf16, kDim, kKind>, dim3(tiles), block, stream, a);
    }
    if (e == hipSuccess && p.bytes) {
        const uint32_t rows = a.tokens * a.q_heads, each = 256 / row_lanes<kDim>();
        e = rows <= kJoinRows
                ? launch(attend_join_row_kernel<kBf16, kDim, kKind>, dim3(rows), block, stream, a)
                : launch(attend_join_kernel<kBf16, kDim, kKind>, dim3((rows + each - 1) / each), block, stream, a);
    }
    return e;
}

template <bool kBf16, int kKind>
hipError_t attend_by_dim(hipStream_t stream, const AttendArgs& a, const Plan& p)
{
    if (a.dim <= 64) return attend_launch<kBf16, 64, kKind>(stream, a, p);
    if (a.dim <= 96) return attend_launch<kBf16, 96, kKind>(stream, a, p);
    if (a.dim <= 128) return attend_launch<kBf16, 128, kKind>(stream, a, p);
    return attend_launch<kBf16, 256, kKind>(stream, a, p);
}

bool more_ok(const si_paged_attention_more* m)
{
    if (!m) return true;
    return m->sinks <= (1u << 30) && m->groups < (1u << 26) && (!m->groups || (m->group_starts && m->prefix_lens));
}

}  // namespace

}  // namespace si

extern "C" {

uint64_t secure_infer_gpu_paged_attention_more_workspace(const si_paged_attention_desc* d,
                                                         const si_paged_attention_more* more)
{
    if (!d || !si::attend_ok(*d) || !si::more_ok(more)) return UINT64_MAX;
    const si::Plan p = si::attend_plan(*d, more);
    return p.fits ? p.bytes : UINT64_MAX;
}

uint64_t secure_infer_gpu_paged_attention_workspace(const si_paged_attention_desc* d)
{
    return secure_infer_gpu_paged_attention_more_workspace(d, nullptr);
}

int secure_infer_gpu_paged_attention(hipStream_t stream, const si_paged_attention_desc* d)
{
    return secure_infer_gpu_paged_attention_more(stream, d, nullptr);
}

int secure_infer_gpu_paged_attention_more(hipStream_t stream, const si_paged_attention_desc* d,
                                          const si_paged_attention_more* more)
{
    using namespace si;
    if (!d || !attend_ok(*d) || !more_ok(more)) return -1;
    const Plan p = attend_plan(*d, more);
    if (!p.fits) return -1;
    if (p.bytes && (!d->workspace || d->workspace_bytes < p.bytes || !aligned(d->workspace, 16))) return -1;
    AttendArgs a{};
    a.q = static_cast<const uint16_t*>(d->q);
    a.q_token = d->q_token_stride;
    a.q_head = d->q_head_stride;
    a.out = static_cast<uint16_t*>(d->out);
    a.out_token = d->out_token_stride;
    a.out_head = d->out_head_stride;
    a.lse = d->lse;
    a.cache_k = static_cast<const uint8_t*>(d->cache_k);
    a.cache_v = static_cast<const uint8_t*>(d->cache_v);
    a.slot_bytes = d->slot_bytes;
    a.nslots = int64_t(d->nslots);
    a.tables = d->tables;
    a.table_stride = d->table_stride;
    a.kv_lens = d->kv_lens;
    a.q_starts = d->q_starts;
    a.pages = d->table_pages;
    a.tokens = d->tokens;
    a.seqs = d->seqs;
    a.q_heads = d->q_heads;
    a.kv_heads = d->kv_heads;
    a.dim = d->head_dim;
    a.page_shift = uint32_t(__builtin_ctz(d->page_tokens));
    a.causal = d->causal;
    a.window = d->window < kMostLength ? d->window : 0;  // no position is further
    a.group = d->q_heads / d->kv_heads;
    a.scale_log2 = std::fabs(d->scale) * 1.44269504088896341f;
    a.q_keep = a.scale_log2 > 0.0f ? ~0u : 0u;
    a.q_flip = d->scale < 0.0f ? 0x80008000u : 0u;
    if (!a.q_keep) a.scale_log2 = 1.0f;
    a.few_rows = p.few_rows;
    a.few_groups = p.few_groups;
    a.few_per = p.few_per;
    a.few_least = p.few_least;
    a.tile_per = p.tile_per;
    a.tile_split = p.tile_split;
    a.tiles = p.tiles;
    uint8_t* const ws = static_cast<uint8_t*>(d->workspace);
    a.few_o = reinterpret_cast<float*>(ws + p.few_o);
    a.few_ml = reinterpret_cast<float2*>(ws + p.few_ml);
    a.few_parts = p.few_parts ? reinterpret_cast<uint2*>(ws + p.few_parts) : nullptr;
    a.tile_o = reinterpret_cast<float*>(ws + p.tile_o);
    a.tile_ml = reinterpret_cast<float2*>(ws + p.tile_ml);
    const bool bf16 = d->dtype == SI_DTYPE_BF16;
    hipError_t e;
    if (!p.sinks && !p.share_groups) {
        e = bf16 ? attend_by_dim<true, kPlain>(stream, a, p) : attend_by_dim<false, kPlain>(stream, a, p);
    } else {
        a.sinks = p.sinks;
        if (p.share_groups) {
            a.groups = more->groups;
            a.group_starts = more->group_starts;
            a.prefix_lens = more->prefix_lens;
        }
        a.share_groups = p.share_groups;
        a.share_split = p.share_split;
        a.share_o = reinterpret_cast<float*>(ws + p.share_o);
        a.share_ml = reinterpret_cast<float2*>(ws + p.share_ml);
        a.few_joins = p.few_joins ? reinterpret_cast<uint4*>(ws + p.few_joins) : nullptr;
        a.tile_groups = p.tile_groups;
        a.alone_groups = p.alone_groups;
        e = bf16 ? attend_by_dim<true, kMore>(stream, a, p) : attend_by_dim<false, kMore>(stream, a, p);
    }
    return e == hipSuccess ? 0 : -1;
}

}  // extern "C"
