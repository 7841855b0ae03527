// Page management of the paged KV cache: new tokens' rows into their pages,
// and forking, freeing, compacting and reserving pages.
//
// A page call is two launches.  The plan kernel is one workgroup: it reads
// the reference counts and the rows concerned, ranks the free slots with a
// block scan and writes the new counts and lengths, the pages to copy or clear
// and the per-row decisions into the workspace; nothing in it depends on the
// order of atomics.  The data kernel rewrites the tables and copies or clears
// the listed pages in every tensor.  One workgroup plans because the counts are few (some
// thousand slots) and every decision needs the ranks of all: 3 to 10 us; the
// pages' bytes bound the rest, and below some 30 MB the launches and
// the host's checks of the call do.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "secure_infer_gpu.h"
#include "si_launch.h"

namespace si {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kMaxCaches = 256;  // tensors per data launch (kernel argument space)
constexpr int32_t kNone = 0x7fffffff;

enum PageOp { OP_FORK, OP_FREE, OP_COMPACT, OP_RESERVE };

// Workspace of a page call, int32 words: [pages listed][pad to 16]
// [(source, target) of each listed page; source -1: clear the target]
// [slot words: free slots ascending / holds given up / where a slot moved]
// [row words: the pair that makes the row / freed / first free slot taken]
// [pair words: parent's whole pages, page copied and then its copy, length] (fork)
struct PagesWs {
    int32_t* count;
    int32_t* moves;
    int32_t* slot;
    int32_t* row;
    int32_t* pair;
};

struct PagesArgs {
    PagesWs ws;
    const int64_t* tables;
    const int64_t* kv_lens;
    const int32_t* refs;
    int64_t* tables_out;
    int64_t* kv_lens_out;
    int32_t* refs_out;
    const int64_t* list;
    uint32_t* fail_count;
    int64_t nslots;
    uint32_t rows, pages, n, page_shift, scrub;
};

struct Caches {
    uint8_t* base[kMaxCaches];
};

__device__ __forceinline__ bool held(int64_t e, int64_t nslots) { return e >= 0 && e < nslots; }

// Exclusive prefix sum of v over the workgroup, and its total (shared memory:
// one word per wave).  Every thread of the workgroup calls it.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* part, uint32_t& total)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    if (lane == 63) part[wave] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
        const uint32_t p = part[w];
        before += w < wave ? p : 0u;
        all += p;
    }
    total = all;
    __syncthreads();
    return before + s - v;
}

// The free slots in ascending order into list[0, min(free, most)); their
// number, as far as it was counted (at least min(free, most)).
__device__ uint32_t list_free(const int32_t* refs, int64_t nslots, uint32_t most, int32_t* list, uint32_t* part)
{
    uint32_t found = 0;
    for (int64_t s0 = 0; s0 < nslots && found < most; s0 += kPlanThreads) {
        const int64_t s = s0 + threadIdx.x;
        const bool free = s < nslots && refs[s] <= 0;
        uint32_t total;
        const uint32_t r = found + block_scan(free, part, total);
        if (free && r < most) list[r] = int32_t(s);
        found += total;
    }
    return found;
}

__device__ __forceinline__ void fail(const PagesArgs& a, uint32_t n)
{
    if (n && a.fail_count) atomicAdd(a.fail_count, n);
}

// Tokens of row b that its table can hold.
__device__ __forceinline__ uint32_t row_len(const PagesArgs& a, int64_t b)
{
    const int64_t most = int64_t(a.pages) << a.page_shift;
    const int64_t n = a.kv_lens[b];
    return uint32_t(n < 0 ? 0 : n > most ? most : n);
}

__device__ void copy_refs(const PagesArgs& a)
{
    if (a.refs_out == a.refs) return;
    for (int64_t s = threadIdx.x; s < a.nslots; s += kPlanThreads) a.refs_out[s] = a.refs[s];
}

__device__ void plan_fork(const PagesArgs& a, uint32_t* part)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t nfree = list_free(a.refs, a.nslots, a.n, a.ws.slot, part);
    for (uint32_t b = threadIdx.x; b < a.rows; b += kPlanThreads) a.ws.row[b] = kNone;
    __syncthreads();
    // The first pair that names a child makes it.
    for (uint32_t i = threadIdx.x; i < a.n; i += kPlanThreads) {
        const int64_t p = a.list[2 * i], c = a.list[2 * i + 1];
        if (p >= 0 && p < a.rows && c >= 0 && c < a.rows) atomicMin(&a.ws.row[c], int32_t(i));
    }
    __syncthreads();
    // One wave per pair: is the child an empty row; the parent's length.
    // pair[3i]: the parent's whole pages (-1: not served), pair[3i + 1]: the
    // slot of its partly filled page (-1: none), pair[3i + 2]: its length.
    for (uint32_t i = wave; i < a.n; i += kPlanThreads / 64) {
        const int64_t p = a.list[2 * i], c = a.list[2 * i + 1];
        int32_t whole = -1, part_slot = -1, len = 0;
        if (p >= 0 && p < a.rows && c >= 0 && c < a.rows && a.ws.row[c] == int32_t(i) && a.kv_lens[c] == 0) {
            bool any = false;
            for (uint32_t j = lane; j < a.pages; j += 64) any |= held(a.tables[c * a.pages + j], a.nslots);
            if (__ballot(any) == 0) {
                len = int32_t(row_len(a, p));
                whole = len >> a.page_shift;
                if (len & ((1 << a.page_shift) - 1)) {
                    const int64_t e = a.tables[p * a.pages + whole];
                    if (held(e, a.nslots)) part_slot = int32_t(e);
                }
            }
        }
        if (lane == 0) {
            a.ws.pair[3 * i] = whole;
            a.ws.pair[3 * i + 1] = part_slot;
            a.ws.pair[3 * i + 2] = len;
        }
    }
    // From here on the outputs are written, which may be the inputs.
    __syncthreads();
    copy_refs(a);
    // Free slots to the pairs that copy a page, in the list's order.
    uint32_t taken = 0;
    for (uint32_t i0 = 0; i0 < a.n; i0 += kPlanThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const bool copies = i < a.n && a.ws.pair[3 * i] >= 0 && a.ws.pair[3 * i + 1] >= 0;
        uint32_t total;
        const uint32_t r = taken + block_scan(copies, part, total);
        if (copies) {
            if (r < nfree) {
                a.ws.moves[2 * r] = a.ws.pair[3 * i + 1];
                a.ws.moves[2 * r + 1] = a.ws.slot[r];
                a.ws.pair[3 * i + 1] = a.ws.slot[r];
                a.refs_out[a.ws.slot[r]] = 1;
            } else {
                a.ws.pair[3 * i] = -1;
            }
        }
        taken += total;
    }
    __syncthreads();
    if (threadIdx.x == 0) *a.ws.count = int32_t(taken < nfree ? taken : nfree);
    uint32_t bad = 0;
    for (uint32_t i = wave; i < a.n; i += kPlanThreads / 64) {
        const int32_t whole = a.ws.pair[3 * i];
        if (whole < 0) {
            bad += lane == 0;
            continue;
        }
        const int64_t p = a.list[2 * i];
        for (uint32_t j = lane; j < uint32_t(whole); j += 64) {
            const int64_t e = a.tables[p * a.pages + j];
            if (held(e, a.nslots)) atomicAdd(&a.refs_out[e], 1);
        }
    }
    fail(a, bad);
    for (uint32_t b = threadIdx.x; b < a.rows; b += kPlanThreads) {
        const int32_t i = a.ws.row[b];
        if (i != kNone && a.ws.pair[3 * i] >= 0) a.kv_lens_out[b] = a.ws.pair[3 * i + 2];
        else if (a.kv_lens_out != a.kv_lens) a.kv_lens_out[b] = a.kv_lens[b];
    }
}

__device__ void plan_free(const PagesArgs& a, uint32_t* shared)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (int64_t s = threadIdx.x; s < a.nslots; s += kPlanThreads) a.ws.slot[s] = 0;
    for (uint32_t b = threadIdx.x; b < a.rows; b += kPlanThreads) a.ws.row[b] = 0;
    if (threadIdx.x == 0) *shared = 0;
    __syncthreads();
    uint32_t bad = 0;
    for (uint32_t i = threadIdx.x; i < a.n; i += kPlanThreads) {
        const int64_t b = a.list[i];
        if (b >= 0 && b < a.rows) a.ws.row[b] = 1;
        else ++bad;
    }
    __syncthreads();
    for (uint32_t b = wave; b < a.rows; b += kPlanThreads / 64) {
        if (!a.ws.row[b]) continue;
        for (uint32_t j = lane; j < a.pages; j += 64) {
            const int64_t e = a.tables[uint64_t(b) * a.pages + j];
            if (held(e, a.nslots)) atomicAdd(&a.ws.slot[e], 1);
        }
    }
    __syncthreads();
    for (int64_t s = threadIdx.x; s < a.nslots; s += kPlanThreads) {
        const int32_t had = a.refs[s], gone = a.ws.slot[s];
        const int32_t hold = had > 0 ? had : 0;
        if (gone > hold) bad += uint32_t(gone - hold);
        const int32_t left = gone ? (hold > gone ? hold - gone : 0) : had;
        a.refs_out[s] = left;
        if (gone && hold && left == 0 && a.scrub) {
            const uint32_t k = atomicAdd(shared, 1u);
            a.ws.moves[2 * k] = -1;
            a.ws.moves[2 * k + 1] = int32_t(s);
        }
    }
    for (uint32_t b = threadIdx.x; b < a.rows; b += kPlanThreads) {
        if (a.ws.row[b]) a.kv_lens_out[b] = 0;
        else if (a.kv_lens_out != a.kv_lens) a.kv_lens_out[b] = a.kv_lens[b];
    }
    fail(a, bad);
    __syncthreads();
    if (threadIdx.x == 0) *a.ws.count = int32_t(*shared);
}

__device__ void plan_compact(const PagesArgs& a, uint32_t* part)
{
    uint32_t live = 0;
    for (int64_t s = threadIdx.x; s < a.nslots; s += kPlanThreads) live += a.refs[s] > 0;
    uint32_t nlive;
    block_scan(live, part, nlive);
    uint32_t holes = 0, movers = 0;
    for (int64_t s0 = 0; s0 < a.nslots; s0 += kPlanThreads) {
        const int64_t s = s0 + threadIdx.x;
        const bool in = s < a.nslots, used = in && a.refs[s] > 0;
        const bool hole = in && !used && s < nlive, mover = used && s >= nlive;
        uint32_t total;
        const uint32_t h = holes + block_scan(hole, part, total);
        holes += total;
        const uint32_t m = movers + block_scan(mover, part, total);
        movers += total;
        if (hole) a.ws.moves[2 * h + 1] = int32_t(s);
        if (mover) a.ws.moves[2 * m] = int32_t(s);
        if (in) a.ws.slot[s] = int32_t(s);
    }
    copy_refs(a);
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < movers; k += kPlanThreads) {
        const int32_t from = a.ws.moves[2 * k], to = a.ws.moves[2 * k + 1];
        a.ws.slot[from] = to;
        a.refs_out[to] = a.refs_out[from];
        a.refs_out[from] = 0;
    }
    if (threadIdx.x == 0) *a.ws.count = int32_t(movers);
}

__device__ void plan_reserve(const PagesArgs& a, uint32_t* part)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const int64_t most = int64_t(a.pages) << a.page_shift;
    // Pages each row lacks (-1: it outgrows its table).
    for (uint32_t b = wave; b < a.rows; b += kPlanThreads / 64) {
        const int64_t add = a.list[b];
        const int64_t had = a.kv_lens[b];
        const int64_t n = add > most || had > most ? most + 1 : had + (add > 0 ? add : 0);
        int32_t need = 0;
        if (n > most) need = -1;
        else if (n > 0) {
            const uint32_t pages = uint32_t((n + (1ll << a.page_shift) - 1) >> a.page_shift);
            for (uint32_t j = lane; j < pages; j += 64) need += !held(a.tables[uint64_t(b) * a.pages + j], a.nslots);
#pragma unroll
            for (int d = 32; d; d >>= 1) need += __shfl_xor(need, d);
        }
        if (lane == 0) a.ws.row[b] = need;
    }
    const uint32_t nfree = list_free(a.refs, a.nslots, uint32_t(a.nslots), a.ws.slot, part);
    __syncthreads();
    copy_refs(a);
    uint32_t taken = 0, bad = 0;
    for (uint32_t b0 = 0; b0 < a.rows; b0 += kPlanThreads) {
        const uint32_t b = b0 + threadIdx.x;
        const int32_t need = b < a.rows ? a.ws.row[b] : 0;
        uint32_t total;
        // Saturating: a row needs at most `pages` < 2^31 / page_tokens slots.
        uint32_t first = block_scan(need > 0 ? uint32_t(need) : 0u, part, total);
        first = first > 0xffffffffu - taken ? 0xffffffffu : first + taken;
        taken = total > 0xffffffffu - taken ? 0xffffffffu : total + taken;
        if (b < a.rows) {
            const bool served = need >= 0 && first <= nfree && uint32_t(need) <= nfree - first;
            bad += !served;
            a.ws.row[b] = served && need > 0 ? int32_t(first) : -1;
            const int64_t add = a.list[b];
            const int64_t had = a.kv_lens[b], room = had > 0 ? INT64_MAX - had : INT64_MAX;
            a.kv_lens_out[b] = had + (add < 0 ? 0 : add > room ? room : add);
        }
    }
    fail(a, bad);
    if (threadIdx.x == 0) *a.ws.count = 0;
}

template <int kOp>
__global__ __launch_bounds__(kPlanThreads) void pages_plan_kernel(PagesArgs a)
{
    __shared__ uint32_t part[kPlanThreads / 64];
    if constexpr (kOp == OP_FORK) plan_fork(a, part);
    if constexpr (kOp == OP_FREE) plan_free(a, part);
    if constexpr (kOp == OP_COMPACT) plan_compact(a, part);
    if constexpr (kOp == OP_RESERVE) plan_reserve(a, part);
}

// Row b of the tables, by one wave.
template <int kOp>
__device__ __forceinline__ void write_row(const PagesArgs& a, uint32_t b)
{
    const uint32_t lane = threadIdx.x & 63u;
    const int64_t* in = a.tables + uint64_t(b) * a.pages;
    int64_t* out = a.tables_out + uint64_t(b) * a.pages;
    if constexpr (kOp == OP_FORK) {
        const int32_t i = a.ws.row[b];
        const int32_t whole = i == kNone ? -1 : a.ws.pair[3 * i];
        if (whole >= 0) {
            const int64_t* from = a.tables + uint64_t(a.list[2 * i]) * a.pages;
            const int32_t slot = a.ws.pair[3 * i + 1];
            for (uint32_t j = lane; j < a.pages; j += 64)
                out[j] = j < uint32_t(whole) ? from[j] : j == uint32_t(whole) ? int64_t(slot) : int64_t(-1);
            return;
        }
    } else if constexpr (kOp == OP_FREE) {
        if (a.ws.row[b]) {
            for (uint32_t j = lane; j < a.pages; j += 64) out[j] = -1;
            return;
        }
    } else if constexpr (kOp == OP_COMPACT) {
        for (uint32_t j = lane; j < a.pages; j += 64) {
            const int64_t e = in[j];
            out[j] = held(e, a.nslots) ? int64_t(a.ws.slot[e]) : e;
        }
        return;
    } else {
        int32_t next = a.ws.row[b];
        if (next >= 0) {
            const int64_t n = a.kv_lens_out[b];
            const uint32_t pages = uint32_t((n + (1ll << a.page_shift) - 1) >> a.page_shift);
            for (uint32_t j0 = 0; j0 < a.pages; j0 += 64) {
                const uint32_t j = j0 + lane;
                int64_t e = j < a.pages ? in[j] : 0;
                const bool lacks = j < pages && !held(e, a.nslots);
                const uint64_t m = __ballot(lacks);
                if (lacks) {
                    e = a.ws.slot[next + __popcll(m & ((1ull << lane) - 1ull))];
                    a.refs_out[e] = 1;
                }
                next += __popcll(m);
                if (j < a.pages) out[j] = e;
            }
            return;
        }
    }
    if (out != in)
        for (uint32_t j = lane; j < a.pages; j += 64) out[j] = in[j];
}

// Workgroups walk the tables' rows (one wave each), then the units (listed
// page, tensor, chunk of kChunk bytes): the grid is fixed, as only the device knows
// the number of pages.  The bytes of the pages bound it.  A thread asks for its two 16 bytes
// of a chunk before it stores them, past the caches, which will not be asked
// for whole pages again soon.  60 pages of 56 tensors (441 MB each way) moved: 161 us, 5.5
// TB/s; 32 of them copied 77 us.  With ordinary stores 176 and 79; stored as
// each load arrives 175 and 81; chunks of 4 KiB 176 and 91, of 16 KiB 180 and 97;
// 1,024 workgroups 179 and 94, 4,096 of them 176 and 84 (both with ordinary stores).
constexpr uint32_t kChunk = 8192;
constexpr uint32_t kDataGroups = 2048;

template <int kOp>
__global__ __launch_bounds__(256) void pages_data_kernel(PagesArgs a, Caches caches, uint32_t ncaches,
                                                         uint64_t slot_bytes, uint64_t page_bytes, uint32_t rows)
{
    const uint32_t wave = threadIdx.x >> 6;
    for (uint32_t b = blockIdx.x * 4 + wave; b < rows; b += gridDim.x * 4) write_row<kOp>(a, b);
    if constexpr (kOp == OP_RESERVE) return;
    const uint32_t chunks = uint32_t((page_bytes + kChunk - 1) / kChunk);
    const uint64_t units = uint64_t(uint32_t(*a.ws.count)) * ncaches * chunks;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t chunk = uint32_t(u % chunks);
        const uint64_t pc = u / chunks;
        const uint32_t c = uint32_t(pc % ncaches), k = uint32_t(pc / ncaches);
        const int32_t from = a.ws.moves[2 * k], to = a.ws.moves[2 * k + 1];
        const uint64_t o = uint64_t(chunk) * kChunk;
        const uint32_t n = uint32_t((page_bytes - o < kChunk ? page_bytes - o : kChunk) / 16);
        u32x4* dst = reinterpret_cast<u32x4*>(caches.base[c] + uint64_t(to) * slot_bytes + o);
        u32x4* src = reinterpret_cast<u32x4*>(caches.base[c] + uint64_t(from < 0 ? to : from) * slot_bytes + o);
        if (from < 0) {
            // (176 MB cleared: 24.9 us, 7.1 TB/s; past the caches 34.9)
            for (uint32_t x = threadIdx.x; x < n; x += 256) dst[x] = u32x4{0, 0, 0, 0};
        } else {
            u32x4 r[kChunk / 4096];
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 4096; ++i)
                if (threadIdx.x + 256 * i < n) r[i] = src[threadIdx.x + 256 * i];
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 4096; ++i) {
                const uint32_t x = threadIdx.x + 256 * i;
                if (x >= n) break;
                __builtin_nontemporal_store(r[i], dst + x);
                if (kOp == OP_COMPACT && a.scrub) __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, src + x);
            }
        }
    }
}

// ---------------------------------------------------------------- append

struct AppendArgs {
    const uint16_t* k;
    const uint16_t* v;
    uint64_t k_token, k_head, v_token, v_head;
    uint8_t* cache_k;
    uint8_t* cache_v;
    uint64_t slot_bytes;
    int64_t nslots;
    const int64_t* tables;
    uint64_t table_stride;
    const int64_t* kv_lens;
    const int64_t* q_starts;
    uint32_t pages, tokens, seqs, heads, dim8, page_shift;
    uint32_t* fail_count;
};

// One wave per token: it finds the token's sequence by counting the starts at
// or before it, 64 at a time, then copies the token's K and V rows, 16 bytes a
// lane, four loads in flight.  The bytes bound it: 14,668 tokens of 8 x 128 heads, bf16,
// out of a fused projection (120 MB read and written) 25.5 us, 4.7 TB/s, 19.8 where
// the caches still hold them.  One load at a time 30.8 and 19.9, two 29.6; with ordinary
// stores 29.2 and 19.8; loads past the caches too 25.0 and 23.0.  64 tokens of 64 sequences:
// 3.6 us, the latency of finding the place and a copy.
constexpr uint32_t kAppendAhead = 4;

__global__ __launch_bounds__(256) void append_kernel(AppendArgs a)
{
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.tokens) return;
    uint32_t b = t;
    int64_t back = 1;  // tokens from here to the sequence's end
    if (a.q_starts) {
        uint32_t at_or_before = 0;
        for (uint32_t s0 = 0; s0 <= a.seqs; s0 += 64) {
            const bool le = s0 + lane <= a.seqs && a.q_starts[s0 + lane] <= int64_t(t);
            at_or_before += __popcll(__ballot(le));
        }
        if (at_or_before == 0 || at_or_before > a.seqs) {
            if (lane == 0 && a.fail_count) atomicAdd(a.fail_count, 1u);
            return;
        }
        b = at_or_before - 1;
        const int64_t end = a.q_starts[b + 1];
        back = (end < a.tokens ? end : a.tokens) - t;
    }
    const int64_t p = a.kv_lens[b] - back;
    const int64_t page = p >> a.page_shift;
    int64_t slot = -1;
    if (p >= 0 && page < a.pages) slot = a.tables[b * a.table_stride + uint64_t(page)];
    if (!held(slot, a.nslots)) {
        if (lane == 0 && a.fail_count) atomicAdd(a.fail_count, 1u);
        return;
    }
    const uint32_t row = a.heads * a.dim8;  // 16-byte chunks
    const uint64_t o = uint64_t(slot) * a.slot_bytes +
                       uint64_t(p & ((1ll << a.page_shift) - 1)) * row * 16;
    for (uint32_t x0 = lane; x0 < 2 * row; x0 += 64 * kAppendAhead) {
        u32x4 r[kAppendAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAppendAhead; ++i) {
            const uint32_t x = x0 + 64 * i;
            if (x >= 2 * row) break;
            const bool is_v = x >= row;
            const uint32_t y = is_v ? x - row : x;
            const uint32_t h = y / a.dim8, d = (y - h * a.dim8) * 8;
            r[i] = *reinterpret_cast<const u32x4*>(is_v ? a.v + t * a.v_token + h * a.v_head + d
                                                        : a.k + t * a.k_token + h * a.k_head + d);
        }
#pragma unroll
        for (uint32_t i = 0; i < kAppendAhead; ++i) {
            const uint32_t x = x0 + 64 * i;
            if (x >= 2 * row) break;
            __builtin_nontemporal_store(r[i], reinterpret_cast<u32x4*>(x < row ? a.cache_k + o + uint64_t(x) * 16
                                                                               : a.cache_v + o + uint64_t(x - row) * 16));
        }
    }
}

// ---------------------------------------------------------------- host side

bool aligned(const void* p, uint64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

bool power_of_two(uint32_t x) { return x && (x & (x - 1)) == 0; }

uint32_t log2_of(uint32_t x) { return uint32_t(__builtin_ctz(x)); }

uint64_t list_words(const si_pages_desc& d)
{
    // Pages listed at most: one per pair (fork), or one per slot (free, compact).
    const uint64_t pairs = 2ull * d.n, slots = 2 * d.nslots;
    return pairs > slots ? pairs : slots;
}

uint64_t pages_bytes(const si_pages_desc& d)
{
    return 4 * (16 + list_words(d) + d.nslots + d.rows + 3ull * d.n);
}

bool pages_ok(const si_pages_desc& d, PageOp op)
{
    if (!d.tables || !d.refs || !d.tables_out || !d.refs_out || !d.workspace) return false;
    if (d.nslots == 0 || d.nslots >= (1ull << 31) || d.rows == 0 || d.rows >= (1u << 31) || d.table_pages == 0)
        return false;
    if (!power_of_two(d.page_tokens) || (uint64_t(d.table_pages) << log2_of(d.page_tokens)) > (1ull << 30)) return false;
    if (op != OP_COMPACT && (!d.kv_lens || !d.kv_lens_out)) return false;
    if (op == OP_RESERVE ? !d.list : op != OP_COMPACT && d.n && !d.list) return false;
    if (d.n >= (1u << 29)) return false;
    if (op != OP_RESERVE) {
        if (d.ncaches && !d.caches) return false;
        if (d.ncaches && (d.page_bytes == 0 || d.page_bytes % 16 || d.slot_bytes % 16 || d.slot_bytes < d.page_bytes ||
                          d.page_bytes >= (1ull << 31)))
            return false;
        for (uint32_t c = 0; c < d.ncaches; ++c)
            if (!d.caches[c] || !aligned(d.caches[c], 16)) return false;
    }
    return aligned(d.workspace, 16) && d.workspace_bytes >= pages_bytes(d);
}

template <int kOp>
int run_pages(hipStream_t stream, const si_pages_desc* d)
{
    if (!d || !pages_ok(*d, PageOp(kOp))) return -1;
    PagesArgs a{};
    int32_t* w = static_cast<int32_t*>(d->workspace);
    a.ws.count = w;
    a.ws.moves = w + 16;
    a.ws.slot = a.ws.moves + list_words(*d);
    a.ws.row = a.ws.slot + d->nslots;
    a.ws.pair = a.ws.row + d->rows;
    a.tables = d->tables;
    a.kv_lens = d->kv_lens;
    a.refs = d->refs;
    a.tables_out = d->tables_out;
    a.kv_lens_out = d->kv_lens_out;
    a.refs_out = d->refs_out;
    a.list = d->list;
    a.fail_count = d->fail_count;
    a.nslots = int64_t(d->nslots);
    a.rows = d->rows;
    a.pages = d->table_pages;
    a.n = d->n;
    a.page_shift = log2_of(d->page_tokens);
    a.scrub = d->scrub;
    if (launch(pages_plan_kernel<kOp>, dim3(1), dim3(kPlanThreads), stream, a) != hipSuccess) return -1;
    const uint32_t ncaches = kOp == OP_RESERVE ? 0 : d->ncaches;
    uint32_t c0 = 0;
    do {
        Caches c{};
        const uint32_t nc = ncaches - c0 < kMaxCaches ? ncaches - c0 : kMaxCaches;
        for (uint32_t i = 0; i < nc; ++i) c.base[i] = static_cast<uint8_t*>(d->caches[c0 + i]);
        const uint32_t rows = c0 ? 0 : d->rows;
        if (launch(pages_data_kernel<kOp>, dim3(kDataGroups), dim3(256), stream, a, c, nc, d->slot_bytes, d->page_bytes,
                   rows) != hipSuccess)
            return -1;
        c0 += nc;
    } while (c0 < ncaches);
    return 0;
}

}  // namespace

}  // namespace si

extern "C" {

uint64_t secure_infer_gpu_pages_workspace(const si_pages_desc* d) { return d ? si::pages_bytes(*d) : 0; }

int secure_infer_gpu_pages_fork(hipStream_t stream, const si_pages_desc* d)
{
    return si::run_pages<si::OP_FORK>(stream, d);
}

int secure_infer_gpu_pages_free(hipStream_t stream, const si_pages_desc* d)
{
    return si::run_pages<si::OP_FREE>(stream, d);
}

int secure_infer_gpu_pages_compact(hipStream_t stream, const si_pages_desc* d)
{
    return si::run_pages<si::OP_COMPACT>(stream, d);
}

int secure_infer_gpu_pages_reserve(hipStream_t stream, const si_pages_desc* d)
{
    return si::run_pages<si::OP_RESERVE>(stream, d);
}

int secure_infer_gpu_paged_append(hipStream_t stream, const si_paged_append_desc* d)
{
    using namespace si;
    if (!d || !d->k || !d->v || !d->cache_k || !d->cache_v || !d->tables || !d->kv_lens) return -1;
    if (!d->tokens || d->tokens >= (1u << 26) || !d->seqs || !d->kv_heads || !d->head_dim || d->head_dim % 8 || !d->nslots ||
        d->nslots >= (1ull << 31) || !d->table_pages)
        return -1;
    if (!d->q_starts && d->tokens != d->seqs) return -1;
    if (!power_of_two(d->page_tokens) || d->page_tokens < 8 || d->page_tokens > 32768) return -1;
    const uint64_t row = 2ull * d->kv_heads * d->head_dim;
    if (row >= (1ull << 30) || d->slot_bytes % 16 || d->slot_bytes < row * d->page_tokens) return -1;
    if ((d->k_token_stride | d->k_head_stride | d->v_token_stride | d->v_head_stride) % 8) return -1;
    for (const void* p : {d->k, d->v, static_cast<const void*>(d->cache_k), static_cast<const void*>(d->cache_v)})
        if (!aligned(p, 16)) return -1;
    AppendArgs a{};
    a.k = static_cast<const uint16_t*>(d->k);
    a.v = static_cast<const uint16_t*>(d->v);
    a.k_token = d->k_token_stride;
    a.k_head = d->k_head_stride;
    a.v_token = d->v_token_stride;
    a.v_head = d->v_head_stride;
    a.cache_k = static_cast<uint8_t*>(d->cache_k);
    a.cache_v = static_cast<uint8_t*>(d->cache_v);
    a.slot_bytes = d->slot_bytes;
    a.nslots = int64_t(d->nslots);
    a.tables = d->tables;
    a.table_stride = d->table_stride;
    a.kv_lens = d->kv_lens;
    a.q_starts = d->q_starts;
    a.pages = d->table_pages;
    a.tokens = d->tokens;
    a.seqs = d->seqs;
    a.heads = d->kv_heads;
    a.dim8 = d->head_dim / 8;
    a.page_shift = log2_of(d->page_tokens);
    a.fail_count = d->fail_count;
    return launch(append_kernel, dim3((d->tokens + 3) / 4), dim3(256), stream, a) == hipSuccess ? 0 : -1;
}

}  // extern "C"
