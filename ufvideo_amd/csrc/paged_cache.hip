// Paged KV cache (see paged.h for its layout): rotary positions with several axes, the rotated append of new tokens, and page management --
// all of it on the device, so that a decode step that reserves pages, appends and attends can be recorded into a HIP graph.
#include "paged.h"

#define ST(s) reinterpret_cast<hipStream_t>(s)

namespace {

// ---------------------------------------------------------------------------------------------------------------------------------
// cos | sin of p[a(i)][n] * inv_freq[i]: rotary positions with several axes.  Frequency pair i turns with the position on ITS axis (time, height, width:
// a(i) comes from the host, two bits per pair).  The angle is formed and reduced to a turn in 64 bits -- at position 10^6 a 32-bit product is off by up to
// 0.03 rad, 64 bits leave 10^-10 -- and the functions of the reduced angle are 32-bit (1-2 ulp).  A thread a pair: 2399 rows of 64 pairs 3.2 us (launch and latency), 16383 rows 6.1 us.
// ---------------------------------------------------------------------------------------------------------------------------------
struct AxisMap { uint32_t w[8]; };      // pair i: bits 2 (i & 15) of word i >> 4; by value: no device copy of the map exists

__global__ __launch_bounds__(256) void rope_axes_table_k(const float* __restrict__ inv_freq, const int64_t* __restrict__ pos, int64_t ld_pos, AxisMap map, int N, int half,
                                                         float* __restrict__ tab) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)N * half) return;
    const int i = id % half;
    const int64_t n = id / half;
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) w = (i >> 4) == k ? map.w[k] : w;
    const int a = (w >> (2 * (i & 15))) & 3;
    const double turns = (double)pos[a * ld_pos + n] * (double)inv_freq[i] * 0.15915494309189533577;
    const float t = (float)(2.0 * (turns - rint(turns)));            // the angle in units of pi, in [-1, 1]
    float s, c;
    sincospif(t, &s, &c);
    float* row = tab + n * (2 * half);
    row[i] = c;
    row[half + i] = s;
}

// one (x1, x2) chunk of 8 pairs; sg = -1 turns back (the transposed rotation: the backward pass)
__device__ __forceinline__ void rope_chunk8(const bf16x8 a, const bf16x8 b, const float* __restrict__ tr, int half, float sg, bf16x8& y1, bf16x8& y2) {
    const f32x4 c0 = *reinterpret_cast<const f32x4*>(tr), c1 = *reinterpret_cast<const f32x4*>(tr + 4);
    const f32x4 s0 = *reinterpret_cast<const f32x4*>(tr + half), s1 = *reinterpret_cast<const f32x4*>(tr + half + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float c = j < 4 ? c0[j & 3] : c1[j & 3], sn = sg * (j < 4 ? s0[j & 3] : s1[j & 3]);
        float r1, r2;
        rope_pair((float)a[j], (float)b[j], c, sn, r1, r2);
        y1[j] = (bf16)r1;
        y2[j] = (bf16)r2;
    }
}

// y = rotated x, rows of nheads heads.  Thread = (row, head, chunk of 8 pairs): two 16-byte loads and stores, the table row from the caches for all heads but one.  Bound by HBM: 16383 rows of
// 32 heads of 128 41 us = 6.8 TB/s, 2399 rows 6.9 us.
__global__ __launch_bounds__(256) void rope_rows_table_k(const bf16* x, int64_t ldx, bf16* y, int64_t ldy, int N, int nheads, int hd, const float* __restrict__ tab, float sg) {
    const int half = hd >> 1, cpr = half >> 3;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)N * nheads * cpr) return;
    const int ch = id % cpr, h = (id / cpr) % nheads;
    const int64_t n = id / ((int64_t)cpr * nheads);
    const bf16* p = x + n * ldx + h * hd + ch * 8;
    bf16x8 y1, y2;
    rope_chunk8(*reinterpret_cast<const bf16x8*>(p), *reinterpret_cast<const bf16x8*>(p + half), tab + n * hd + ch * 8, half, sg, y1, y2);
    bf16* d = y + n * ldy + h * hd + ch * 8;
    *reinterpret_cast<bf16x8*>(d) = y1;
    *reinterpret_cast<bf16x8*>(d + half) = y2;
}

// the same one pair per thread, for head dims or rows that 16-byte chunks do not fit
__global__ __launch_bounds__(256) void rope_rows_table_scalar_k(const bf16* x, int64_t ldx, bf16* y, int64_t ldy, int N, int nheads, int hd, const float* __restrict__ tab, float sg) {
    const int half = hd >> 1;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)N * nheads * half) return;
    const int i = id % half, h = (id / half) % nheads;
    const int64_t n = id / ((int64_t)half * nheads);
    const bf16* p = x + n * ldx + h * hd + i;
    float r1, r2;
    rope_pair((float)p[0], (float)p[half], tab[n * hd + i], sg * tab[n * hd + half + i], r1, r2);
    bf16* d = y + n * ldy + h * hd + i;
    d[0] = (bf16)r1;
    d[half] = (bf16)r2;
}

// q_out = rotated q, cache row = [rotated k | v] of every packed row.  Block = one row: its slot, position and page are block-uniform; thread = (head, chunk of 8 pairs).  Bound by HBM: 6449 rows
// of 28 + 2 x 4 heads of 128 20.6 us = 5.9 TB/s; one row 2.4 us.
__global__ void rope_kv_paged_k(const bf16* qkv, int64_t ldqkv, bf16* q_out, int64_t ldq, int Hq, int Hkv, int hd, const float* __restrict__ tab, bf16* __restrict__ pages,
                                int64_t ldkv, PagedTable t) {
    const int n = blockIdx.x;
    const int s = paged_slot_of_row(t.cu_q, t.S, n);
    if (s >= t.S) return;                                            // behind the last slot's rows: left as they are
    const int q0 = t.cu_q[s], q1 = t.cu_q[s + 1];
    if (n < q0 || n >= q1) return;
    const int pos = paged_len(t, s) - (q1 - q0) + (n - q0);          // < 0: more rows than cached tokens, this one has no place in the cache
    const int64_t at = pos >= 0 ? paged_row(t, s, pos) : -1;
    bf16* crow = pages + at * ldkv;
    const int half = hd >> 1, cpr = half >> 3, items = (Hq + 2 * Hkv) * cpr;
    const bf16* row = qkv + (int64_t)n * ldqkv;
    const float* tr = tab + (int64_t)n * hd;
    for (int id = threadIdx.x; id < items; id += blockDim.x) {
        const int ch = id % cpr, h = id / cpr;
        const bf16* p = row + h * hd + ch * 8;
        bf16x8 a = *reinterpret_cast<const bf16x8*>(p), b = *reinterpret_cast<const bf16x8*>(p + half), y1 = a, y2 = b;
        if (h < Hq + Hkv) rope_chunk8(a, b, tr + ch * 8, half, 1.f, y1, y2);
        bf16* d = (h < Hq ? q_out + (int64_t)n * ldq + h * hd : crow + (h - Hq) * hd) + ch * 8;
        if (h < Hq || at >= 0) {
            *reinterpret_cast<bf16x8*>(d) = y1;
            *reinterpret_cast<bf16x8*>(d + half) = y2;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Page management.  State: block_table [S, ld] (-1 = no page), kv_len [S], refs [n_pages] (how many table entries name a page; 0 = free).
// Slot s holds the first ceil(kv_len[s] / page) entries of its row.  Requests are dense vectors over the slots, so no slot can be named twice.
// ---------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int pages_held(int len, int sh, int width) {
    const int n = len > 0 ? (int)(((int64_t)len + (1 << sh) - 1) >> sh) : 0;
    return n < width ? n : width;
}

// exclusive prefix sum of one int per thread over a block of NT threads, and the block's total; `red` = NT / 64 + 1 ints of LDS
template <int NT>
__device__ __forceinline__ int block_scan(int v, int* red, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) red[w] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        const int r = red[i];
        before += i < w ? r : 0;
        all += r;
    }
    total = all;
    return before + x - v;
}

// slot s becomes another owner of every page of slot parent[s] (no page is copied; latency: 24 slots 3 us).  A slot that holds tokens is no child, a slot that is named a child is no parent:
// no block reads what another one writes, whatever the vector says.
__global__ __launch_bounds__(256) void kv_pages_fork_k(int* table, int64_t ld, int width, int* kv_len, int* refs, int n_pages, const int* __restrict__ parent, int S, int sh) {
    const int s = blockIdx.x, p = parent[s];
    if (p < 0 || p >= S || p == s || parent[p] >= 0) return;
    const int mine = kv_len[s], len = kv_len[p];
    __syncthreads();
    if (mine != 0) return;
    const int n = pages_held(len, sh, width);
    for (int j = threadIdx.x; j < n; j += 256) {
        const int id = table[(int64_t)p * ld + j];
        table[(int64_t)s * ld + j] = id;
        if ((unsigned)id < (unsigned)n_pages) atomicAdd(refs + id, 1);      // integers: the order of the adds does not show
    }
    if (threadIdx.x == 0) kv_len[s] = len;
}

__global__ __launch_bounds__(256) void kv_pages_free_k(int* table, int64_t ld, int width, int* kv_len, int* refs, int n_pages, const int* __restrict__ mask, int sh) {
    const int s = blockIdx.x;
    if (mask[s] == 0) return;
    const int n = pages_held(kv_len[s], sh, width);
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += 256) {
        const int id = table[(int64_t)s * ld + j];
        table[(int64_t)s * ld + j] = -1;
        if ((unsigned)id < (unsigned)n_pages) atomicSub(refs + id, 1);
    }
    if (threadIdx.x == 0) kv_len[s] = 0;
}

// Room for n_new[s] further tokens of every slot, one block of 1024 threads (a chain of scans and dependent loads, latency: 24 slots on 93 pages 7.8 us):
//  A  what every slot needs: new pages at its end, and a page of its own in place of a partly filled last page that it shares (copy on write); prefix sum over the slots
//  B  the lowest free page ids, as many as are needed (the scan of refs stops there)
//  C  slot s takes pages [off, off + need) of that list, one wave per slot; a slot whose share reaches past the free pages, or past its table row, gets nothing
//     (its later pages are not offered to the slots behind it; a slot that needs no page is served)
//  D  cu_q = prefix sum of the granted tokens
// ws: free list [n_pages] | off [S] | need [S] | shared [S]
__global__ __launch_bounds__(1024) void kv_pages_extend_k(int* table, int64_t ld, int width, int* kv_len, int* refs, int n_pages, const int* __restrict__ n_new, int S, int sh,
                                                          int* granted, int* cu_q, int* pairs, int* ws) {
    __shared__ int red[17];
    int* list = ws;
    int* off = ws + n_pages;
    int* need = off + S;
    int* shared = need + S;
    const int tid = threadIdx.x, page = 1 << sh;
    int64_t want_all = 0;
    for (int s0 = 0; s0 < S; s0 += 1024) {
        const int s = s0 + tid;
        int nd = 0, sd = 0;
        if (s < S) {
            const int n = max(n_new[s], 0), len = max(kv_len[s], 0);
            const int64_t have = ((int64_t)len + page - 1) >> sh, want = ((int64_t)len + n + page - 1) >> sh;
            if (n > 0 && want <= width) {
                if (len & (page - 1)) {
                    const int last = table[(int64_t)s * ld + have - 1];
                    sd = (unsigned)last < (unsigned)n_pages && refs[last] > 1;
                }
                nd = (int)(want - have) + sd;
            } else {
                sd = -1;                                              // nothing asked, or no room in the row
            }
        }
        int total;
        const int before = block_scan<1024>(nd, red, total);
        if (s < S) { off[s] = (int)min(want_all + before, (int64_t)0x7fffffff - width); need[s] = nd; shared[s] = sd; }
        want_all += total;
    }
    const int want = (int)min(want_all, (int64_t)n_pages);
    int found = 0;
    for (int i0 = 0; i0 < n_pages && found < want; i0 += 4096) {
        const int i = i0 + tid * 4;
        int f[4], c = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) { f[k] = i + k < n_pages && refs[i + k] == 0; c += f[k]; }
        int total;
        int at = found + block_scan<1024>(c, red, total);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (f[k]) list[at++] = i + k;
        found += total;
    }
    __syncthreads();                                                  // list, off, need, shared are written; refs has been read
    for (int s = tid >> 6; s < S; s += 16) {
        const int sd = shared[s], nd = need[s], o = off[s], len = max(kv_len[s], 0), n = max(n_new[s], 0);
        const bool ok = sd >= 0 && (nd == 0 || (int64_t)o + nd <= found);
        const int start = pages_held(len, sh, width) - (sd > 0), last = ok && sd > 0 ? table[(int64_t)s * ld + start] : -1;
        const int first = ok && sd > 0 ? list[o] : -1;
        if (ok)                                                       // (`last` is read before lane 0 replaces it: one wave, in order)
            for (int j = tid & 63; j < nd; j += 64) {
                const int id = list[o + j];
                table[(int64_t)s * ld + start + j] = id;
                refs[id] = 1;
            }
        if ((tid & 63) == 0) {
            if (last >= 0) atomicSub(refs + last, 1);
            pairs[3 * s] = last; pairs[3 * s + 1] = first; pairs[3 * s + 2] = last >= 0 ? (len & (page - 1)) : 0;
            granted[s] = ok ? n : 0;
            if (ok) kv_len[s] = len + n;
        }
    }
    __syncthreads();
    int base = 0;
    for (int s0 = 0; s0 < S; s0 += 1024) {
        const int s = s0 + tid;
        int total;
        const int before = block_scan<1024>(s < S ? granted[s] : 0, red, total);
        if (s < S) cu_q[s] = base + before;
        base += total;
    }
    if (tid == 0) cu_q[S] = base;
}

// Which pages move when the K live ones are to be pages 0 .. K - 1: the i-th free page below K takes the i-th live page from K on.  That is the least number of moves, and
// no page is both read and written, so all of them can be copied at once.  ws: dst [n_pages] | src [n_pages] | remap [n_pages]
__global__ __launch_bounds__(1024) void kv_pages_plan_k(int* refs, int n_pages, int* counts, int* ws) {
    __shared__ int red[17];
    int *dst = ws, *src = ws + n_pages, *remap = src + n_pages;
    const int tid = threadIdx.x;
    int live = 0;
    for (int i0 = 0; i0 < n_pages; i0 += 1024) {
        const int i = i0 + tid;
        int total;
        block_scan<1024>(i < n_pages && refs[i] > 0, red, total);
        live += total;
    }
    int holes = 0, movers = 0;
    for (int i0 = 0; i0 < n_pages; i0 += 1024) {
        const int i = i0 + tid;
        const bool l = i < n_pages && refs[i] > 0, hole = i < live && !l, mover = i >= live && l;
        int th, tm;
        const int a = block_scan<1024>(hole, red, th), b = block_scan<1024>(mover, red, tm);
        if (hole) dst[holes + a] = i;
        if (mover) src[movers + b] = i;
        if (i < n_pages) remap[i] = i;
        holes += th;
        movers += tm;
    }
    __syncthreads();
    for (int r = tid; r < movers; r += 1024) {                        // holes == movers: pages below K are K in all
        remap[src[r]] = dst[r];
        refs[dst[r]] = refs[src[r]];
        refs[src[r]] = 0;
    }
    if (tid == 0) { counts[0] = live; counts[1] = movers; }
}

// 16 KB of one page: 256 threads x 4 x 16 bytes, all four loads before the first store (copies of 82 MB in 15 us = 5.4 TB/s, moves of 228 MB in 37 = 6.1: bound by HBM)
__device__ __forceinline__ void copy_piece(const char* __restrict__ src, char* __restrict__ dst, int64_t bytes, int64_t at) {
    typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
    u32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t b = at + (int64_t)(k * 256 + threadIdx.x) * 16;
        if (b < bytes) v[k] = *reinterpret_cast<const u32x4*>(src + b);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t b = at + (int64_t)(k * 256 + threadIdx.x) * 16;
        if (b < bytes) *reinterpret_cast<u32x4*>(dst + b) = v[k];
    }
}

// rows 0 .. rows - 1 of page src -> page dst, every layer; pairs [n][3] = (src, dst, rows), src or dst outside the pool: nothing
__global__ __launch_bounds__(256) void kv_pages_copy_k(char* pool, int64_t layer_bytes, int64_t page_bytes, int n_pages, int page, const int* __restrict__ pairs) {
    const int* p = pairs + 3 * blockIdx.z;
    const int src = p[0], dst = p[1], rows = min(p[2], page);
    if ((unsigned)src >= (unsigned)n_pages || (unsigned)dst >= (unsigned)n_pages || src == dst || rows <= 0) return;
    const int64_t bytes = page_bytes / page * rows, at = (int64_t)blockIdx.x * 16384;
    if (at >= bytes) return;
    char* base = pool + blockIdx.y * layer_bytes;
    copy_piece(base + src * page_bytes, base + dst * page_bytes, bytes, at);
}

// the moves of kv_pages_plan_k (their number is known on the device only): a fixed grid walks over (move, layer, 16 KB piece).  The first blocks rewrite the table rows before that: a launch
// of its own for them cost 2.6 us.
__global__ __launch_bounds__(256) void kv_pages_move_k(char* pool, int layers, int64_t layer_bytes, int64_t page_bytes, int n_pages, const int* __restrict__ counts, const int* __restrict__ ws,
                                                       int* table, int64_t ld, int width, const int* __restrict__ kv_len, int S, int sh) {
    for (int s = blockIdx.x; s < S; s += gridDim.x) {
        const int n = pages_held(kv_len[s], sh, width);
        for (int j = threadIdx.x; j < n; j += 256) {
            const int id = table[(int64_t)s * ld + j];
            if ((unsigned)id < (unsigned)n_pages) table[(int64_t)s * ld + j] = ws[2 * (int64_t)n_pages + id];
        }
    }
    const int pieces = (int)((page_bytes + 16383) / 16384);
    const int64_t total = (int64_t)counts[1] * layers * pieces;
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const int piece = w % pieces, layer = (w / pieces) % layers, r = w / ((int64_t)pieces * layers);
        char* base = pool + layer * layer_bytes;
        copy_piece(base + ws[n_pages + r] * page_bytes, base + ws[r] * page_bytes, page_bytes, (int64_t)piece * 16384);
    }
}

}  // namespace

extern "C" int ufv_rope_axes_table(const float* inv_freq, const int64_t* positions, int64_t ld_pos, int n_axes, const uint8_t* axis_of, int N, int hd, float* table, void* stream) {
    UFV_REQUIRE(inv_freq && positions && axis_of && table && N > 0, "ufv_rope_axes_table: bad arguments");
    UFV_REQUIRE(hd > 0 && hd % 2 == 0 && hd <= 256, "ufv_rope_axes_table: head_dim must be even and at most 256 (%d)", hd);
    UFV_REQUIRE(n_axes >= 1 && n_axes <= 4 && (n_axes == 1 || ld_pos >= N || ld_pos == 0), "ufv_rope_axes_table: 1 to 4 axes, rows of at least N positions or one row for all (%d axes, pitch %lld)", n_axes, (long long)ld_pos);
    AxisMap m = {};
    for (int i = 0; i < hd / 2; ++i) {
        UFV_REQUIRE(axis_of[i] < n_axes, "ufv_rope_axes_table: pair %d names axis %d of %d", i, axis_of[i], n_axes);
        m.w[i >> 4] |= (uint32_t)axis_of[i] << (2 * (i & 15));
    }
    const int64_t total = (int64_t)N * (hd / 2);
    hipLaunchKernelGGL(rope_axes_table_k, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, ST(stream), inv_freq, positions, ld_pos, m, N, hd / 2, table);
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

extern "C" int ufv_rope_rows_table(const void* x, int64_t ldx, void* y, int64_t ldy, int N, int nheads, int hd, const float* table, int backward, void* stream) {
    UFV_REQUIRE(x && y && table && N > 0 && nheads > 0 && hd > 0 && hd % 2 == 0, "ufv_rope_rows_table: bad arguments (N=%d heads=%d hd=%d)", N, nheads, hd);
    UFV_REQUIRE(N == 1 || (ldx >= (int64_t)nheads * hd && ldy >= (int64_t)nheads * hd), "ufv_rope_rows_table: row pitch below %d heads of %d", nheads, hd);
    UFV_REQUIRE((int64_t)nheads * hd < 0x7fffffff, "ufv_rope_rows_table: rows of more than 2^31 columns (%d heads of %d)", nheads, hd);
    const float sg = backward ? -1.f : 1.f;
    const bool vec = hd % 16 == 0 && ldx % 8 == 0 && ldy % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)y % 16 == 0 && (uintptr_t)table % 16 == 0;
    const int64_t total = (int64_t)N * nheads * (vec ? hd / 16 : hd / 2);
    UFV_REQUIRE((total + 255) / 256 < 0x7fffffff, "ufv_rope_rows_table: too many rows (%d)", N);
    const dim3 grid((unsigned)((total + 255) / 256));
    if (vec) hipLaunchKernelGGL(rope_rows_table_k, grid, dim3(256), 0, ST(stream), (const bf16*)x, ldx, (bf16*)y, ldy, N, nheads, hd, table, sg);
    else hipLaunchKernelGGL(rope_rows_table_scalar_k, grid, dim3(256), 0, ST(stream), (const bf16*)x, ldx, (bf16*)y, ldy, N, nheads, hd, table, sg);
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

extern "C" int ufv_rope_kv_paged(const void* qkv, int64_t ldqkv, void* q_out, int64_t ldq, int N, int Hq, int Hkv, int hd, const float* table, void* pages, int n_pages, int page,
                                 int64_t ldkv, const int32_t* block_table, int64_t ld_table, int max_pages, const int32_t* cu_q, const int32_t* kv_len, int S, void* stream) {
    UFV_REQUIRE_PAGED("ufv_rope_kv_paged", pages, n_pages, page, ldkv, block_table, ld_table, max_pages, cu_q, kv_len, S);
    UFV_REQUIRE(qkv && q_out && table && N > 0 && Hq > 0 && Hkv > 0 && hd > 0 && hd % 16 == 0, "ufv_rope_kv_paged: bad arguments or head_dim no multiple of 16 (N=%d heads %d/%d hd=%d)", N, Hq, Hkv, hd);
    UFV_REQUIRE((uintptr_t)qkv % 16 == 0 && (uintptr_t)q_out % 16 == 0 && (uintptr_t)table % 16 == 0 && ldqkv % 8 == 0 && ldq % 8 == 0,
                "ufv_rope_kv_paged: rows must be 16-byte aligned (pitches %lld, %lld)", (long long)ldqkv, (long long)ldq);
    UFV_REQUIRE(ldkv >= 2 * (int64_t)Hkv * hd && (N == 1 || (ldqkv >= (int64_t)(Hq + 2 * Hkv) * hd && ldq >= (int64_t)Hq * hd)), "ufv_rope_kv_paged: a row pitch is too small");
    UFV_REQUIRE(((int64_t)Hq + 2 * (int64_t)Hkv) * hd < 0x7fffffff, "ufv_rope_kv_paged: rows of more than 2^31 columns (heads %d/%d of %d)", Hq, Hkv, hd);
    PagedTable t{block_table, ld_table, max_pages, cu_q, kv_len, S, n_pages, paged_log2(page)};
    const int items = (Hq + 2 * Hkv) * (hd / 16), threads = items < 512 ? (items + 63) / 64 * 64 : 512;
    hipLaunchKernelGGL(rope_kv_paged_k, dim3(N), dim3(threads), 0, ST(stream), (const bf16*)qkv, ldqkv, (bf16*)q_out, ldq, Hq, Hkv, hd, table, (bf16*)pages, ldkv, t);
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

// (2^30 pages, 2^29 slots: the loops over them and three entries a slot stay within 31 bits)
#define UFV_REQUIRE_TABLE(name)                                                                                                                   \
    UFV_REQUIRE(block_table && kv_len && refs && max_pages > 0 && S > 0 && n_pages > 0 && ld_table >= max_pages,                                 \
                name ": bad arguments (%d slots, %d pages, table %d of pitch %lld)", S, n_pages, max_pages, (long long)ld_table);                 \
    UFV_REQUIRE(n_pages <= 1 << 30 && S <= 1 << 29, name ": more than 2^30 pages or 2^29 slots (%d, %d)", n_pages, S);                            \
    UFV_REQUIRE(paged_log2(page) > 0, name ": the page size must be a power of two from 16 to 32768 (%d)", page);                                 \
    UFV_REQUIRE(((int64_t)max_pages << paged_log2(page)) <= 0x7fffffff - 65536, name ": a table row names more than 2^31 tokens (%d pages of %d)", max_pages, page)

extern "C" int ufv_kv_pages_fork(int32_t* block_table, int64_t ld_table, int max_pages, int32_t* kv_len, int S, int32_t* refs, int n_pages, int page, const int32_t* parent, void* stream) {
    UFV_REQUIRE_TABLE("ufv_kv_pages_fork");
    UFV_REQUIRE(parent, "ufv_kv_pages_fork: bad arguments");
    hipLaunchKernelGGL(kv_pages_fork_k, dim3(S), dim3(256), 0, ST(stream), block_table, ld_table, max_pages, kv_len, refs, n_pages, parent, S, paged_log2(page));
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

extern "C" int ufv_kv_pages_free(int32_t* block_table, int64_t ld_table, int max_pages, int32_t* kv_len, int S, int32_t* refs, int n_pages, int page, const int32_t* mask, void* stream) {
    UFV_REQUIRE_TABLE("ufv_kv_pages_free");
    UFV_REQUIRE(mask, "ufv_kv_pages_free: bad arguments");
    hipLaunchKernelGGL(kv_pages_free_k, dim3(S), dim3(256), 0, ST(stream), block_table, ld_table, max_pages, kv_len, refs, n_pages, mask, paged_log2(page));
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

extern "C" int64_t ufv_kv_pages_extend_ws_bytes(int S, int n_pages) { return 4 * (3 * (int64_t)S + n_pages); }

extern "C" int ufv_kv_pages_extend(int32_t* block_table, int64_t ld_table, int max_pages, int32_t* kv_len, int S, int32_t* refs, int n_pages, int page, const int32_t* n_new, int32_t* granted,
                                   int32_t* cu_q, int32_t* pairs, void* ws, int64_t ws_bytes, void* stream) {
    UFV_REQUIRE_TABLE("ufv_kv_pages_extend");
    UFV_REQUIRE(max_pages <= 1 << 20, "ufv_kv_pages_extend: a table row of more than 2^20 pages (%d)", max_pages);      // the sums over 1024 slots stay within 31 bits
    UFV_REQUIRE(n_new && granted && cu_q && pairs && ws && ws_bytes >= ufv_kv_pages_extend_ws_bytes(S, n_pages), "ufv_kv_pages_extend: bad arguments or a workspace of fewer than %lld bytes",
                (long long)ufv_kv_pages_extend_ws_bytes(S, n_pages));
    hipLaunchKernelGGL(kv_pages_extend_k, dim3(1), dim3(1024), 0, ST(stream), block_table, ld_table, max_pages, kv_len, refs, n_pages, n_new, S, paged_log2(page), granted, cu_q, pairs, (int*)ws);
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

#define UFV_REQUIRE_POOL(name)                                                                                                                             \
    UFV_REQUIRE(pool && layers > 0 && layers <= 65535 && n_pages > 0 && row_bytes > 0 && row_bytes % 16 == 0 && (uintptr_t)pool % 16 == 0 && layer_bytes % 16 == 0 && \
                (layers == 1 || layer_bytes >= (int64_t)n_pages * page * row_bytes), name ": bad arguments (%d layers of %d pages, rows of %lld bytes, 16-byte aligned)", layers, n_pages, \
                (long long)row_bytes);                                                                                                                      \
    UFV_REQUIRE(paged_log2(page) > 0, name ": the page size must be a power of two from 16 to 32768 (%d)", page)

extern "C" int ufv_kv_pages_copy(void* pool, int layers, int64_t layer_bytes, int n_pages, int page, int64_t row_bytes, const int32_t* pairs, int n, void* stream) {
    UFV_REQUIRE_POOL("ufv_kv_pages_copy");
    UFV_REQUIRE(pairs && n > 0 && n <= 65535, "ufv_kv_pages_copy: 1 to 65535 pairs (%d)", n);
    const int64_t pb = page * row_bytes;
    hipLaunchKernelGGL(kv_pages_copy_k, dim3((unsigned)((pb + 16383) / 16384), layers, n), dim3(256), 0, ST(stream), (char*)pool, layer_bytes, pb, n_pages, page, pairs);
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

extern "C" int64_t ufv_kv_pages_compact_ws_bytes(int n_pages) { return 12 * (int64_t)n_pages; }

extern "C" int ufv_kv_pages_compact(void* pool, int layers, int64_t layer_bytes, int64_t row_bytes, int32_t* block_table, int64_t ld_table, int max_pages, const int32_t* kv_len, int S,
                                    int32_t* refs, int n_pages, int page, int32_t* counts, void* ws, int64_t ws_bytes, void* stream) {
    UFV_REQUIRE_TABLE("ufv_kv_pages_compact");
    UFV_REQUIRE_POOL("ufv_kv_pages_compact");
    UFV_REQUIRE(counts && ws && ws_bytes >= ufv_kv_pages_compact_ws_bytes(n_pages), "ufv_kv_pages_compact: bad arguments or a workspace of fewer than %lld bytes",
                (long long)ufv_kv_pages_compact_ws_bytes(n_pages));
    const int sh = paged_log2(page);
    hipLaunchKernelGGL(kv_pages_plan_k, dim3(1), dim3(1024), 0, ST(stream), refs, n_pages, counts, (int*)ws);
    hipLaunchKernelGGL(kv_pages_move_k, dim3(2048), dim3(256), 0, ST(stream), (char*)pool, layers, layer_bytes, page * row_bytes, n_pages, counts, (const int*)ws,
                       block_table, ld_table, max_pages, kv_len, S, sh);
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}
