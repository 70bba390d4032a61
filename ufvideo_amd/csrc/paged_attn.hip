// Attention of a chunk of new tokens over a paged KV cache (see paged.h for the layout).
//   o[r, h] = sum_j softmax_j(q[r, h] . k[j, g] * scale) v[j, g],  g = h / (Hq / Hkv),  over the keys j < kv_len[s] (causal: j <= the row's own position);
// a row that sees no key gets zeros.  Keys that do not exist -- behind kv_len, in a page outside the pool -- are never read.
//
// One wave per (row, q head): 64 keys a step, one key per lane for the scores, then lanes over the dims for the weighted sum.
#include "paged.h"

namespace {

__global__ __launch_bounds__(64) void attn_paged_k(const bf16* __restrict__ q, int64_t ldq, bf16* __restrict__ o, int64_t ldo, int Hq, int Hkv, int hd, const bf16* __restrict__ pages,
                                                   int64_t ldkv, PagedTable t, float scale, int causal) {
    __shared__ float qs[256], ps[64];
    __shared__ int64_t rows[64];
    const int n = blockIdx.x, h = blockIdx.y, g = h / (Hq / Hkv), lane = threadIdx.x;
    const int s = paged_slot_of_row(t.cu_q, t.S, n);
    if (s >= t.S) return;
    const int q0 = t.cu_q[s], q1 = t.cu_q[s + 1];
    if (n < q0 || n >= q1) return;
    const int len = paged_len(t, s), pos = len - (q1 - q0) + (n - q0);
    const int nk = causal ? min(len, pos + 1) : len;
    for (int d = lane; d < hd; d += 64) qs[d] = (float)q[(int64_t)n * ldq + h * hd + d] * scale;
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < nk; j0 += 64) {
        const int j = j0 + lane;
        int64_t row = -1;
        float sc = -INFINITY;
        if (j < nk) row = paged_row(t, s, j);
        if (row >= 0) {
            const bf16* k = pages + row * ldkv + g * hd;
            sc = 0.f;
            for (int c = 0; c < hd; c += 8) {
                const bf16x8 kv = *reinterpret_cast<const bf16x8*>(k + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) sc += qs[c + e] * (float)kv[e];
            }
        }
        const float mn = fmaxf(m, wave_max(sc));
        const float alpha = m == -INFINITY ? 0.f : __expf(m - mn);
        const float p = row >= 0 ? __expf(sc - mn) : 0.f;
        m = mn;
        l = l * alpha + wave_sum(p);
        ps[lane] = p;
        rows[lane] = row;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= alpha;
        for (int jj = 0; jj < 64; ++jj) {
            if (rows[jj] < 0) continue;
            const bf16* v = pages + rows[jj] * ldkv + (Hkv + g) * hd;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < hd) acc[i] += ps[jj] * (float)v[lane + 64 * i];
        }
        __syncthreads();
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < hd) o[(int64_t)n * ldo + h * hd + lane + 64 * i] = (bf16)(acc[i] * inv);
}

}  // namespace

extern "C" int64_t ufv_attention_paged_ws_bytes(int N, int S, int Hq, int Hkv, int hd, int max_keys) { return 0; }

extern "C" int ufv_attention_paged(const void* q, int64_t ldq, void* o, int64_t ldo, int N, int Hq, int Hkv, int hd, const void* pages, int n_pages, int page, int64_t ldkv,
                                   const int32_t* block_table, int64_t ld_table, int max_pages, const int32_t* cu_q, const int32_t* kv_len, int S, float scale, int causal, void* ws,
                                   int64_t ws_bytes, void* stream) {
    UFV_REQUIRE_PAGED("ufv_attention_paged", pages, n_pages, page, ldkv, block_table, ld_table, max_pages, cu_q, kv_len, S);
    UFV_REQUIRE(q && o && N > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "ufv_attention_paged: bad arguments (N=%d, %d q heads on %d kv heads)", N, Hq, Hkv);
    UFV_REQUIRE(hd >= 8 && hd <= 256 && hd % 8 == 0, "ufv_attention_paged: head_dim must be a multiple of 8 up to 256 (%d)", hd);
    UFV_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)o % 16 == 0 && ldq % 8 == 0 && ldo % 8 == 0, "ufv_attention_paged: rows must be 16-byte aligned (pitches %lld, %lld)", (long long)ldq,
                (long long)ldo);
    UFV_REQUIRE(ldkv >= 2 * (int64_t)Hkv * hd && (N == 1 || (ldq >= (int64_t)Hq * hd && ldo >= (int64_t)Hq * hd)), "ufv_attention_paged: a row pitch is too small");
    PagedTable t{block_table, ld_table, max_pages, cu_q, kv_len, S, n_pages, paged_log2(page)};
    hipLaunchKernelGGL(attn_paged_k, dim3(N, Hq), dim3(64), 0, reinterpret_cast<hipStream_t>(stream), (const bf16*)q, ldq, (bf16*)o, ldo, Hq, Hkv, hd, (const bf16*)pages, ldkv, t, scale, causal);
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}
