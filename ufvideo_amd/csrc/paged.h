// What the kernels of the paged KV cache share (paged_cache.hip: rotary positions, append, page management; paged_attn.hip: attention).
//
// The cache of one layer is pages [n_pages][page][ldkv] of bf16: a page holds `page` token rows (a power of two >= 16), a row is
// [Hkv * hd k | Hkv * hd v] as in the contiguous cache -- a contiguous cache buffer IS a run of consecutive pages.  A batch is S slots; slot s
// owns row s of block_table (int32 page ids in token order) and kv_len[s] cached tokens; the new tokens of a step are packed rows, slot s
// having rows cu_q[s] .. cu_q[s + 1) -- its LAST tokens: row r is token kv_len[s] - (cu_q[s + 1] - cu_q[s]) + r - cu_q[s] of the sequence.
// Page ids are bounds-checked by every kernel: a key whose page id is outside [0, n_pages) does not exist.
#pragma once
#include "common.h"

struct PagedTable {
    const int* table;       // [S, ld]
    int64_t ld;
    int width;              // page slots of a row
    const int* cu_q;        // [S + 1]
    const int* kv_len;      // [S]
    int S, n_pages, sh;     // sh = log2(page)
};

// cached tokens of slot s, never past what its table row can name
__host__ __device__ __forceinline__ int paged_len(const PagedTable& t, int s) {
    const int64_t cap = (int64_t)t.width << t.sh;
    const int n = t.kv_len[s];
    return n < 0 ? 0 : (n > cap ? (int)cap : n);
}

// the cache row of token j >= 0 of slot s (j below paged_len), or -1 where its page id lies outside the pool
__host__ __device__ __forceinline__ int64_t paged_row(const PagedTable& t, int s, int j) {
    const int page = t.table[(int64_t)s * t.ld + (j >> t.sh)];
    return (unsigned)page < (unsigned)t.n_pages ? ((int64_t)page << t.sh) + (j & ((1 << t.sh) - 1)) : -1;
}

// the slot of packed row n: the number of slots whose rows end at or before n (empty slots are passed over); S when n lies behind the last one.
// One load per 64 slots: every lane compares one entry of cu_q, the wave counts.  n must be wave-uniform.
__device__ __forceinline__ int paged_slot_of_row(const int* __restrict__ cu_q, int S, int n) {
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int s0 = 0; s0 < S; s0 += 64) {
        const bool before = s0 + lane < S && cu_q[s0 + lane + 1] <= n;
        const int c = __popcll(__ballot(before));
        b += c;
        if (c < 64) break;
    }
    return b;
}

static inline int paged_log2(int page) {
    for (int s = 4; s < 16; ++s)
        if (page == 1 << s) return s;
    return -1;              // not a power of two from 16 on
}

#define UFV_REQUIRE_PAGED(name, pages, n_pages, page, ldkv, table, ld_table, max_pages, cu_q, kv_len, S)                                              \
    UFV_REQUIRE((pages) && (table) && (cu_q) && (kv_len) && (n_pages) > 0 && (max_pages) > 0 && (S) > 0 && (ld_table) >= (max_pages),                 \
                name ": bad arguments (%d pages, %d slots, table %d of pitch %lld)", n_pages, S, max_pages, (long long)(ld_table));                   \
    UFV_REQUIRE((S) <= 1 << 29, name ": more than 2^29 slots (%d)", S);                                                                               \
    UFV_REQUIRE(paged_log2(page) > 0, name ": the page size must be a power of two from 16 to 32768 (%d)", page);                                     \
    UFV_REQUIRE((uintptr_t)(pages) % 16 == 0 && (ldkv) % 8 == 0, name ": cache rows must be 16-byte aligned (pitch %lld)", (long long)(ldkv));        \
    UFV_REQUIRE(((int64_t)(max_pages) << paged_log2(page)) <= 0x7fffffff - 65536, name ": a table row names more than 2^31 tokens (%d pages of %d)", max_pages, page)
