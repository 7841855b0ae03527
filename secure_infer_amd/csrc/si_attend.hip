// Attention of new tokens over a paged KV cache.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

#include "secure_infer_gpu.h"
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
    uint32_t pages, tokens, seqs, q_heads, kv_heads, dim, page_shift, causal, window;
    float scale_log2;  // scale * log2(e): weights are powers of two
};

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

// One wave per (token, query head): 64 keys at a time, one key a lane for the
// scores, the head's dims over the lanes for the sum over the values.
template <bool kBf16>
__global__ __launch_bounds__(64) void attend_plain_kernel(AttendArgs a)
{
    __shared__ float qs[256];
    const uint32_t lane = threadIdx.x;
    const uint32_t t = blockIdx.x / a.q_heads, h = blockIdx.x - t * a.q_heads;
    const uint32_t kvh = h / (a.q_heads / a.kv_heads);
    uint32_t b = t;
    int64_t back = 1;  // tokens from here to the sequence's end
    bool owned = true;
    if (a.q_starts) {
        uint32_t at_or_before = 0;
        for (uint32_t s0 = 0; s0 <= a.seqs; s0 += 64) {
            const bool le = s0 + lane <= a.seqs && a.q_starts[s0 + lane] <= int64_t(t);
            at_or_before += __popcll(__ballot(le));
        }
        owned = at_or_before != 0 && at_or_before <= a.seqs;
        if (owned) {
            b = at_or_before - 1;
            const int64_t end = a.q_starts[b + 1];
            back = (end < a.tokens ? end : a.tokens) - t;
        }
    }
    const int64_t most = int64_t(a.pages) << a.page_shift;
    int64_t n = owned ? a.kv_lens[b] : 0;
    n = n < 0 ? 0 : n > most ? most : n;
    const int64_t p = n - back;
    const int64_t hi = a.causal ? p + 1 : n;
    int64_t lo = a.window && p - int64_t(a.window) + 1 > 0 ? p - int64_t(a.window) + 1 : 0;
    for (uint32_t d = lane; d < a.dim; d += 64)
        qs[d] = to_f32<kBf16>(a.q[t * a.q_token + h * a.q_head + d]) * a.scale_log2;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[4] = {0, 0, 0, 0};
    for (int64_t j0 = lo; j0 < hi; j0 += 64) {
        const int64_t j = j0 + lane;
        int64_t slot = -1;
        if (j < hi) slot = a.tables[b * a.table_stride + uint64_t(j >> a.page_shift)];
        const bool seen = held(slot, a.nslots);
        const uint64_t o = seen ? uint64_t(slot) * a.slot_bytes +
                                      (uint64_t(j & ((1ll << a.page_shift) - 1)) * a.kv_heads + kvh) * a.dim * 2
                                : 0;
        float s = -INFINITY;
        if (seen) {
            const uint16_t* k = reinterpret_cast<const uint16_t*>(a.cache_k + o);
            s = 0.0f;
            for (uint32_t d = 0; d < a.dim; ++d) s = __builtin_fmaf(qs[d], to_f32<kBf16>(k[d]), s);
        }
        float top = s;
#pragma unroll
        for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        const float mn = fmaxf(m, top);
        if (mn == -INFINITY) continue;
        const float w = seen ? exp2f(s - mn) : 0.0f;
        const float keep = exp2f(m - mn);
        m = mn;
        float sum = w;
#pragma unroll
        for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
        l = __builtin_fmaf(l, keep, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= keep;
        const uint64_t mask = __ballot(seen);
        for (int kk = 0; kk < 64; ++kk) {
            if (!(mask >> kk & 1)) continue;
            const float wk = __shfl(w, kk);
            const uint16_t* v = reinterpret_cast<const uint16_t*>(a.cache_v + __shfl(o, kk));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < a.dim) acc[i] = __builtin_fmaf(wk, to_f32<kBf16>(v[lane + 64 * i]), acc[i]);
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.dim)
            a.out[t * a.out_token + h * a.out_head + lane + 64 * i] = from_f32<kBf16>(acc[i] * inv);
    if (a.lse && lane == 0)
        a.lse[uint64_t(t) * a.q_heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

bool aligned(const void* p, uint64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

bool attend_ok(const si_paged_attention_desc& d)
{
    if (!d.q || !d.out || !d.cache_k || !d.cache_v || !d.tables || !d.kv_lens) return false;
    if (!d.tokens || !d.seqs || !d.q_heads || !d.kv_heads || d.q_heads % d.kv_heads || !d.table_pages) return false;
    if (!d.q_starts && d.tokens != d.seqs) return false;
    if (uint64_t(d.tokens) * d.q_heads >= (1ull << 31) || d.seqs >= (1u << 31)) return false;
    if (!d.head_dim || d.head_dim % 8 || d.head_dim > 256 || d.dtype > SI_DTYPE_FP16) return false;
    if (d.page_tokens < 8 || d.page_tokens > 32768 || (d.page_tokens & (d.page_tokens - 1))) return false;
    if (uint64_t(d.table_pages) * d.page_tokens >= (1ull << 31)) return false;
    if (!d.nslots || d.nslots >= (1ull << 31)) return false;
    const uint64_t row = 2ull * d.kv_heads * d.head_dim;
    if (row >= (1ull << 30) || d.slot_bytes % 16 || d.slot_bytes < row * d.page_tokens) return false;
    if ((d.q_token_stride | d.q_head_stride | d.out_token_stride | d.out_head_stride) % 8) return false;
    if (!std::isfinite(d.scale)) return false;
    for (const void* p : {d.q, static_cast<const void*>(d.out), d.cache_k, d.cache_v})
        if (!aligned(p, 16)) return false;
    return true;
}

uint64_t attend_workspace(const si_paged_attention_desc&) { return 0; }

}  // namespace

}  // namespace si

extern "C" {

uint64_t secure_infer_gpu_paged_attention_workspace(const si_paged_attention_desc* d)
{
    return d && si::attend_ok(*d) ? si::attend_workspace(*d) : UINT64_MAX;
}

int secure_infer_gpu_paged_attention(hipStream_t stream, const si_paged_attention_desc* d)
{
    using namespace si;
    if (!d || !attend_ok(*d)) return -1;
    const uint64_t need = attend_workspace(*d);
    if (need && (!d->workspace || d->workspace_bytes < need || !aligned(d->workspace, 16))) return -1;
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
    a.window = d->window;
    a.scale_log2 = d->scale * 1.44269504088896341f;
    const dim3 grid(d->tokens * d->q_heads);
    const hipError_t e = d->dtype == SI_DTYPE_BF16 ? launch(attend_plain_kernel<true>, grid, dim3(64), stream, a)
                                                   : launch(attend_plain_kernel<false>, grid, dim3(64), stream, a);
    return e == hipSuccess ? 0 : -1;
}

}  // extern "C"
