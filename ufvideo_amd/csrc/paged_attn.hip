// Attention of a chunk of new tokens over a paged KV cache (see paged.h for the layout).
//   o[r, h] = sum_j softmax_j(q[r, h] . k[j, g] * scale) v[j, g],  g = h / G,  G = Hq / Hkv,  over the keys j < kv_len[s] (causal: j <= the row's own position);
// a row that sees no key gets zeros.  Keys that do not exist -- behind kv_len, in a page outside the pool -- are staged as zeros and their scores are -inf.
//
// The unit of work is a TILE of rows of one slot and one kv head, a row being a (token, q head of the group) pair: row r of a slot is token r / G, head g * G + r % G.  All G heads
// that share a kv head sit in one tile, so that every key is fetched once for the group and a single token already fills G of the 32 columns of a matrix instruction.
//
// Both kernels compute S^T = K Q^T with v_mfma_f32_32x32x16_bf16 (a lane owns one row of the tile: its column of S^T), keep the running maximum and sum of the softmax in
// 32 bits (log2 domain), and use the exponentiated tile, rounded to bf16, directly as the B operand of O^T += V^T P^T.  The rounding of P is the one step below 32 bits between
// the inputs and the output: the matrix instruction takes bf16 operands; the row sum is taken of the unrounded values.  V^T fragments come from row-major V rows in LDS by the transposing read.
//   attn_paged_tile_k   the waves of a block share 64-key tiles and split the ROWS: chunks of many rows, bound by the matrix unit
//   attn_paged_keys_k   the waves of a block share up to 32 rows and split the KEYS: a few new tokens over a long cache, bound by the bytes of the cache
// Either may be split further over the keys by blocks (few tiles on 256 CUs); the parts leave (max, sum, un-normalised O) in 32 bits in the workspace and attn_paged_join_k adds them in order.
#include "paged.h"

namespace {

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

struct PagedAttn {
    const bf16 *q, *pages;
    bf16* o;
    int64_t ldq, ldo, ldkv;
    PagedTable t;
    int N, Hq, Hkv, G, hd, causal;
    float sl2;              // scale * log2(e)
    int nsplit, tiles;      // key parts (upper bound), row tiles (upper bound)
    float* part;            // [nsplit][N * Hq][hd] un-normalised O, then [nsplit][N * Hq][2] max | sum; nullptr: nsplit == 1
};

// what a block works on: all of it wave-uniform
struct PagedTile {
    int s, q0, n, len;      // slot, its first packed row, its rows, its cached tokens
    int row0, rows;         // the tile's first (token, head) row, all such rows of the slot
    int g;                  // kv head
};

// Row tiles are numbered over the batch without the host knowing the lengths: slot s may use the numbers from floor(cu_q[s] * G / R) + s on; the next slot's first number is
// never less than what slot s needs (ceil(n G / R)).  Numbers without rows leave at once.
template <int R>
__device__ __forceinline__ bool paged_tile(const PagedAttn& a, int tile, PagedTile& w) {
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int s0 = 0; s0 < a.t.S; s0 += 64) {
        const int s = s0 + lane;
        const bool mine = s < a.t.S && (int)((int64_t)a.t.cu_q[s] * a.G / R) + s <= tile;
        const int c = __popcll(__ballot(mine));
        b += c;
        if (c < 64) break;
    }
    if (b == 0) return false;
    w.s = __builtin_amdgcn_readfirstlane(b - 1);
    w.q0 = a.t.cu_q[w.s];
    w.n = a.t.cu_q[w.s + 1] - w.q0;
    if (w.q0 < 0 || w.n <= 0 || w.q0 + w.n > a.N) return false;
    w.rows = w.n * a.G;
    w.row0 = (tile - ((int)((int64_t)w.q0 * a.G / R) + w.s)) * R;
    w.len = paged_len(a.t, w.s);
    return w.row0 < w.rows;
}

// keys that row r of a slot sees: tokens 0 .. paged_seen - 1
__device__ __forceinline__ int paged_seen(const PagedAttn& a, int len, int n, int tok) { return a.causal ? max(len - n + tok + 1, 0) : len; }

// the key parts of a slot of `len` tokens: every part holds the same number of UNIT-key steps, at least two of them
template <int UNIT>
__device__ __forceinline__ int paged_part(int len, int nsplit) {
    const int steps = (len + UNIT - 1) / UNIT, parts = max(min(nsplit, steps / 2), 1);
    return (steps + parts - 1) / parts;
}

__device__ __forceinline__ bf16x8 pack8(const float* p) {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2 v = __builtin_convertvector((f32x2){p[2 * i], p[2 * i + 1]}, bf16x2);
        r[2 * i] = v[0];
        r[2 * i + 1] = v[1];
    }
    return r;
}

template <int HDP>
struct PCfg {
    static constexpr int KS = HDP / 16, DT = HDP / 32;
    static constexpr int CPR = HDP <= 32 ? 4 : (HDP <= 64 ? 8 : (HDP <= 128 ? 16 : 32));     // lanes that fetch one cache row, 16 bytes each (a power of two; HDP 96: four idle)
    static constexpr int RPW = 64 / CPR;                                                     // rows of one wave load: at most 16, so all of one page
    static constexpr int PK = HDP * 2 + 16;                                                  // K row pitch: an odd number of 16-byte slots, conflict-free b128 reads
    static constexpr int PV = HDP == 32 ? 64 : (HDP <= 96 ? 192 : (HDP == 128 ? 320 : 576)); // V row pitch: 64 or 192 mod 256, conflict-free transposing reads
};

// One 32-key half tile in LDS against QG groups of 32 rows: S^T, running softmax, O^T.
// hide: key j of the half (0 .. 31) counts for the lane's row iff j < vis (and, in 16-key groups, iff its bit of `pages` is set)
template <int HDP, int QG>
struct PState {
    f32x16 o[QG][HDP / 32];
    float m[QG], l[QG];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int q = 0; q < QG; ++q) {
            m[q] = -INFINITY;
            l[q] = 0.f;
#pragma unroll
            for (int i = 0; i < HDP / 32; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[q][i][r] = 0.f;
        }
    }
};

template <int HDP, int QG, int NH>
__device__ __forceinline__ void paged_step(const char* kb, const char* vb, const bf16x8 (&qf)[QG][HDP / 16], PState<HDP, QG>& st, float sl2, bool hide, const int (&vis)[QG], unsigned groups) {
    using C = PCfg<HDP>;
    const int lane = threadIdx.x & 63, h = lane >> 5, l31 = lane & 31;
    const int k_off = l31 * C::PK + h * 16;
    const int v_off = (4 * h + ((lane & 15) >> 2)) * C::PV + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
    f32x16 s[QG][NH];
#pragma unroll
    for (int q = 0; q < QG; ++q)
#pragma unroll
        for (int hh = 0; hh < NH; ++hh)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[q][hh][r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks)
#pragma unroll
        for (int hh = 0; hh < NH; ++hh) {
            const bf16x8 kf = *reinterpret_cast<const bf16x8*>(kb + hh * 32 * C::PK + k_off + ks * 32);
#pragma unroll
            for (int q = 0; q < QG; ++q) s[q][hh] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[q][ks], s[q][hh], 0, 0, 0);
        }
    if (hide) {
#pragma unroll
        for (int q = 0; q < QG; ++q)
#pragma unroll
            for (int hh = 0; hh < NH; ++hh)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = hh * 32 + (r & 3) + 8 * (r >> 2) + 4 * h;
                    s[q][hh][r] = j < vis[q] && ((groups >> (2 * hh + (r >> 3))) & 1) ? s[q][hh][r] : -INFINITY;
                }
    }
    bf16x8 pf[QG][2 * NH];
#pragma unroll
    for (int q = 0; q < QG; ++q) {
        float tmax = s[q][0][0];
#pragma unroll
        for (int hh = 0; hh < NH; ++hh)
#pragma unroll
            for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s[q][hh][r]);
        tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64)) * sl2;
        // the rescale of O waits until the maximum has grown by 2^6: until then the exponentials stay below 2^6 and nothing is lost
        if (__any(tmax > st.m[q] + 6.0f)) {
            const float mnew = fmaxf(st.m[q], tmax);
            const float alpha = mnew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m[q] - mnew);
            st.l[q] *= alpha;
#pragma unroll
            for (int i = 0; i < C::DT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) st.o[q][i][r] *= alpha;
            st.m[q] = mnew;
        }
        const float msub = st.m[q] == -INFINITY ? 0.f : st.m[q];
        float sum = 0.f;
#pragma unroll
        for (int hh = 0; hh < NH; ++hh) {
            float p[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[q][hh][r], sl2, -msub));
                sum += p[r];
            }
            pf[q][2 * hh] = pack8(p);
            pf[q][2 * hh + 1] = pack8(p + 8);
        }
        st.l[q] += sum;
    }
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
        for (int c = 0; c < 2 * NH; ++c) {
            const char* vp = vb + 16 * c * C::PV + v_off + dt * 64;
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((bf16x4 __attribute__((address_space(3)))*)(vp));
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((bf16x4 __attribute__((address_space(3)))*)(vp + 8 * C::PV));
            const bf16x8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int q = 0; q < QG; ++q) st.o[q][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[q][c], st.o[q][dt], 0, 0, 0);
        }
}

// A key that a row does not see must not reach it even when its V row holds Inf or NaN (0 * Inf in the matrix product): among the new tokens of a causal chunk -- the only keys
// that some rows see and others do not -- such elements are staged as zeros, and if there was one, they are added after the walk to the rows that see them (keys j0 .. j1 - 1;
// p > 0 times Inf or NaN is Inf or NaN).
template <int HDP, int QG>
__device__ __forceinline__ void paged_add_bad(const PagedAttn& a, const PagedTile& w, int j0, int j1, PState<HDP, QG>& st, const int (&seen)[QG]) {
    const int h = (threadIdx.x & 63) >> 5;
    for (int j = j0; j < j1; ++j) {
        const int64_t at = paged_row(a.t, w.s, j);
        if (at < 0) continue;
        const bf16* v = a.pages + at * a.ldkv + (a.Hkv + w.g) * a.hd;
#pragma unroll
        for (int dt = 0; dt < HDP / 32; ++dt)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int d = dt * 32 + 8 * g4 + 4 * h;                                // hd is a multiple of 8: four dims exist or none
                asm volatile("" ::: "memory");                                         // four elements at a time: this path is rare and must not cost the main loop registers
                if (d < a.hd) {
                    const bf16x4 x = *reinterpret_cast<const bf16x4*>(v + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int q = 0; q < QG; ++q)
                            if (!(fabsf((float)x[e]) < INFINITY) && j < seen[q]) st.o[q][dt][4 * g4 + e] += (float)x[e];
                }
            }
    }
}

// zero the non-finite elements of a chunk of V; true if there was one
__device__ __forceinline__ bool paged_clean(u32x4& v) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool lo = (v[i] & 0x7f80u) == 0x7f80u, hi = (v[i] & 0x7f800000u) == 0x7f800000u;
        v[i] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
        any |= lo | hi;
    }
    return any;
}

// The lane's rows of the tile as B operands (lane: row l31 of the group, dims 16 ks + 8 h ..), and what they see.  Rows behind the tile's last take the last one's q; they are not stored.
template <int HDP, int QG>
__device__ __forceinline__ void paged_load_q(const PagedAttn& a, const PagedTile& w, int row0, bf16x8 (&qf)[QG][HDP / 16], int (&seen)[QG]) {
    const int lane = threadIdx.x & 63, h = lane >> 5, l31 = lane & 31;
#pragma unroll
    for (int q = 0; q < QG; ++q) {
        const int r = min(row0 + 32 * q + l31, w.rows - 1), tok = r / a.G, hq = w.g * a.G + (r - tok * a.G);
        const bf16* p = a.q + (int64_t)(w.q0 + tok) * a.ldq + hq * a.hd + h * 8;
        seen[q] = paged_seen(a, w.len, w.n, tok);
#pragma unroll
        for (int ks = 0; ks < HDP / 16; ++ks) {
            qf[q][ks] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (ks * 16 + h * 8 < a.hd) qf[q][ks] = *reinterpret_cast<const bf16x8*>(p + ks * 16);
        }
    }
}

// Staging of NG groups of 16 keys by NWS waves, cache -> registers -> LDS.  A wave load covers RPW <= 16 rows that start at a multiple of RPW, and a page holds whole groups of 16
// tokens: the page is the same for the whole load, its id a scalar, and the lane's part of the address does not change.  Lanes whose chunk lies behind hd (padded head dims) fetch
// chunk 0: their K meets zeros in Q, their V columns are not stored.
template <int HDP, int NG, int NWS>
struct PStage {
    using C = PCfg<HDP>;
    static constexpr int PASS = NWS * C::RPW, RPT = 16 * NG / PASS;
    static_assert(RPT >= 1 && RPT * PASS == 16 * NG, "whole passes");
    u32x4 k[RPT], v[RPT];
    int id[NG];             // page ids of the next step's groups, -1 behind the last token

    __device__ __forceinline__ void ids(const PagedAttn& a, const PagedTile& w, int step) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int64_t j = ((int64_t)step * NG + i) * 16;
            id[i] = j < w.len ? a.t.table[(int64_t)w.s * a.t.ld + (int)(j >> a.t.sh)] : -1;
        }
    }
    __device__ __forceinline__ unsigned valid(const PagedAttn& a) const {
        unsigned ok = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) ok |= (unsigned)id[i] < (unsigned)a.t.n_pages ? 1u << i : 0u;
        return ok;
    }
    // lane_off: element offset of the lane's row and chunk inside a load; wave: the wave's place among the NWS
    __device__ __forceinline__ void fetch(const PagedAttn& a, const PagedTile& w, int step, unsigned ok, int64_t lane_off, int srow, int wave) {
        const bool all = ok == (1u << NG) - 1 && ((int64_t)step + 1) * NG * 16 <= w.len;
        const bf16* base = a.pages + w.g * a.hd;
        const int64_t vo = (int64_t)a.Hkv * a.hd;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int row = i * PASS + wave * C::RPW, j = step * NG * 16 + row;
            int page = id[(i * PASS) >> 4];
            if (PASS > 16)
#pragma unroll
                for (int x = 1; x < PASS / 16; ++x) page = (wave * C::RPW) >> 4 == x ? id[((i * PASS) >> 4) + x] : page;
            const bf16* p = base + (((int64_t)page << a.t.sh) + (j & ((1 << a.t.sh) - 1))) * a.ldkv + lane_off;
            if (all) {
                k[i] = *reinterpret_cast<const u32x4*>(p);
                v[i] = *reinterpret_cast<const u32x4*>(p + vo);
            } else {
                k[i] = u32x4{0, 0, 0, 0};
                v[i] = u32x4{0, 0, 0, 0};
                if ((unsigned)page < (unsigned)a.t.n_pages && j + srow < w.len) {
                    k[i] = *reinterpret_cast<const u32x4*>(p);
                    v[i] = *reinterpret_cast<const u32x4*>(p + vo);
                }
            }
        }
    }
    __device__ __forceinline__ bool clean() {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < RPT; ++i) bad |= paged_clean(v[i]);
        return bad;
    }
    __device__ __forceinline__ void park(char* kb, char* vb, int srow, int sch, int wave) const {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int row = i * PASS + wave * C::RPW + srow;
            if (C::CPR * 8 == HDP || sch * 8 < HDP) {
                *reinterpret_cast<u32x4*>(kb + row * C::PK + sch * 16) = k[i];
                *reinterpret_cast<u32x4*>(vb + row * C::PV + sch * 16) = v[i];
            }
        }
    }
};

// ---------------------------------------------------------------------------------------------------------------------------------
// rows split over the waves
// ---------------------------------------------------------------------------------------------------------------------------------
template <int HDP, int QG, int NW>
__global__ __launch_bounds__(NW * 64, QG == 2 || HDP > 128 ? 1 : 2) void attn_paged_tile_k(PagedAttn a) {
    using C = PCfg<HDP>;
    constexpr int R = 32 * QG * NW, STAGE = 64 * (C::PK + C::PV);
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ int dirty;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    PagedTile w;
    int part;
    {
        // ids that differ by 8 run on one XCD: give every XCD a contiguous run of (kv head, part, tile) so that the tiles of one kv head share an L2; last rows (most keys) first
        const int total = a.tiles * a.Hkv * a.nsplit, per = (total + 7) >> 3, id = blockIdx.x, i = (id & 7) * per + (id >> 3);
        if ((id >> 3) >= per || i >= total) return;
        const int tile = a.tiles - 1 - i % a.tiles, rest = i / a.tiles;
        part = rest % a.nsplit;
        w.g = rest / a.nsplit;
        if (!paged_tile<R>(a, tile, w)) return;
    }
    const int per = paged_part<64>(w.len, a.nsplit);                                  // 64-key steps of a part
    const int last_tok = (min(w.row0 + R, w.rows) - 1) / a.G;
    const int kmax = paged_seen(a, w.len, w.n, last_tok);                              // keys that some row of the tile sees
    const int t0 = part * per, t1 = min(t0 + per, (kmax + 63) >> 6);
    const bool whole = per * 64 >= w.len;                                              // one part: the block writes the result itself
    if (t0 >= t1 && !(whole && part == 0)) return;
    const int row0 = w.row0 + wave * 32 * QG;
    bf16x8 qf[QG][C::KS];
    int seen[QG];
    paged_load_q<HDP, QG>(a, w, row0, qf, seen);
    const int seen_min = paged_seen(a, w.len, w.n, min(row0, w.rows - 1) / a.G);
    const int diag = a.causal && w.n > 1 ? w.len - w.n : 0x7fffffff;                   // keys from here on are seen by some rows only

    const int srow = lane / C::CPR, sch = lane % C::CPR;
    const int64_t lane_off = srow * a.ldkv + (sch * 8 < a.hd ? sch * 8 : 0);
    if (tid == 0) dirty = 0;
    PStage<HDP, 4, NW> sg;
    PState<HDP, QG> st;
    st.clear();
    unsigned groups = 0, next = 0;
    if (t0 < t1) {
        sg.ids(a, w, t0);
        next = sg.valid(a);
        sg.fetch(a, w, t0, next, lane_off, srow, wave);
        sg.ids(a, w, t0 + 1);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        char* kb = smem + ((t - t0) & 1) * STAGE;
        if ((int64_t)(t + 1) * 64 > diag && __any(sg.clean()) && lane == 0) dirty = 1;
        sg.park(kb, kb + 64 * C::PK, srow, sch, wave);
        groups = next;
        if (t + 1 < t1) {
            next = sg.valid(a);
            sg.fetch(a, w, t + 1, next, lane_off, srow, wave);
            sg.ids(a, w, t + 2);
        }
        __syncthreads();                                                                // one barrier a step: the buffer written now was last read two steps ago
        int vis[QG];
#pragma unroll
        for (int q = 0; q < QG; ++q) vis[q] = min(seen[q], w.len) - (t << 6);
        paged_step<HDP, QG, 2>(kb, kb + 64 * C::PK, qf, st, a.sl2, (t << 6) + 64 > min(seen_min, w.len) || groups != 15u, vis, groups);
    }
    if (diag < w.len) {
        __syncthreads();
        if (dirty) paged_add_bad<HDP, QG>(a, w, max(diag, t0 << 6), min(t1 << 6, w.len), st, seen);
    }
    const int h = lane >> 5, l31 = lane & 31;
#pragma unroll
    for (int q = 0; q < QG; ++q) {
        const float l = st.l[q] + __shfl_xor(st.l[q], 32, 64);
        const int r = row0 + 32 * q + l31;
        if (r >= w.rows) continue;
        const int tok = r / a.G, hq = w.g * a.G + (r - tok * a.G);
        if (whole) {
            const float inv = l > 0.f ? 1.f / l : l;                                   // l = 0: no key; NaN stays NaN
            bf16* op = a.o + (int64_t)(w.q0 + tok) * a.ldo + hq * a.hd;
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int d = dt * 32 + g4 * 8 + h * 4;
                    if (d < a.hd) {
                        const bf16x4 ov = {(bf16)(st.o[q][dt][g4 * 4] * inv), (bf16)(st.o[q][dt][g4 * 4 + 1] * inv), (bf16)(st.o[q][dt][g4 * 4 + 2] * inv), (bf16)(st.o[q][dt][g4 * 4 + 3] * inv)};
                        *reinterpret_cast<bf16x4*>(op + d) = ov;
                    }
                }
        } else {
            const int64_t rid = (int64_t)part * a.N * a.Hq + (int64_t)(w.q0 + tok) * a.Hq + hq;
            float* op = a.part + rid * a.hd;
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int d = dt * 32 + g4 * 8 + h * 4;
                    if (d < a.hd) *reinterpret_cast<f32x4*>(op + d) = f32x4{st.o[q][dt][g4 * 4], st.o[q][dt][g4 * 4 + 1], st.o[q][dt][g4 * 4 + 2], st.o[q][dt][g4 * 4 + 3]};
                }
            if (h == 0) {
                float* ml = a.part + (int64_t)a.nsplit * a.N * a.Hq * a.hd + 2 * rid;
                ml[0] = st.m[q];
                ml[1] = l;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// keys split over the waves: no barrier until the waves' parts are joined
// ---------------------------------------------------------------------------------------------------------------------------------
template <int HDP, int NW>
__global__ __launch_bounds__(NW * 64, 1) void attn_paged_keys_k(PagedAttn a) {
    using C = PCfg<HDP>;
    constexpr int STAGE = 32 * (C::PK + C::PV);
    static_assert(STAGE >= 32 * HDP * 4, "a wave's O fits its staging area");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float wm[NW][32], wl[NW][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, l31 = lane & 31;
    PagedTile w;
    const int part = blockIdx.y;
    w.g = blockIdx.z;
    if (!paged_tile<32>(a, blockIdx.x, w)) return;
    const int per = paged_part<32 * NW>(w.len, a.nsplit) * NW;                         // 32-key steps of a part
    const int kmax = paged_seen(a, w.len, w.n, (min(w.row0 + 32, w.rows) - 1) / a.G);
    const int t0 = part * per, t1 = min(t0 + per, (kmax + 31) >> 5);
    const bool whole = per * 32 >= w.len;
    if (t0 >= t1 && !(whole && part == 0)) return;
    char* kb = smem + wave * STAGE;
    char* vb = kb + 32 * C::PK;
    const int srow = lane / C::CPR, sch = lane % C::CPR;
    const int diag = a.causal && w.n > 1 ? w.len - w.n : 0x7fffffff;
    const int64_t lane_off = srow * a.ldkv + (sch * 8 < a.hd ? sch * 8 : 0);
    PStage<HDP, 2, 1> sg;
    unsigned next = 0;
    if (t0 + wave < t1) {
        sg.ids(a, w, t0 + wave);
        next = sg.valid(a);
        sg.fetch(a, w, t0 + wave, next, lane_off, srow, 0);
        sg.ids(a, w, t0 + wave + NW);
    }
    PState<HDP, 1> st;
    st.clear();
    bf16x8 qf[1][C::KS];
    int seen[1];
    paged_load_q<HDP, 1>(a, w, w.row0, qf, seen);
    const int seen_min = paged_seen(a, w.len, w.n, w.row0 / a.G);
    bool dirty = false;
    for (int t = t0 + wave; t < t1; t += NW) {
        if ((int64_t)(t + 1) * 32 > diag) dirty |= __any(sg.clean());
        sg.park(kb, vb, srow, sch, 0);
        const unsigned groups = next;
        if (t + NW < t1) {
            next = sg.valid(a);
            sg.fetch(a, w, t + NW, next, lane_off, srow, 0);
            sg.ids(a, w, t + 2 * NW);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");                          // the staged rows are read by other lanes of this wave
        __builtin_amdgcn_wave_barrier();
        int vis[1] = {min(seen[0], w.len) - (t << 5)};
        paged_step<HDP, 1, 1>(kb, vb, qf, st, a.sl2, (t << 5) + 32 > min(seen_min, w.len) || groups != 3u, vis, groups);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    if (dirty)
        for (int t = t0 + wave; t < t1; t += NW) paged_add_bad<HDP, 1>(a, w, max(diag, t << 5), min((t + 1) << 5, w.len), st, seen);
    // ---- join the waves: (m, l) and O [row][HDP] of every wave through LDS, then every thread sums columns of the rows that exist
    const float l = st.l[0] + __shfl_xor(st.l[0], 32, 64);
    if (h == 0) { wm[wave][l31] = st.m[0]; wl[wave][l31] = l; }
    float* ob = reinterpret_cast<float*>(kb);
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
            *reinterpret_cast<f32x4*>(ob + l31 * HDP + dt * 32 + g4 * 8 + h * 4) = f32x4{st.o[0][dt][g4 * 4], st.o[0][dt][g4 * 4 + 1], st.o[0][dt][g4 * 4 + 2], st.o[0][dt][g4 * 4 + 3]};
    __syncthreads();
    const int rows = min(w.rows - w.row0, 32), cols = a.hd >> 2;
    for (int i = tid; i < rows * cols; i += NW * 64) {
        const int r = i / cols, d = (i - r * cols) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NW; ++k) m = fmaxf(m, wm[k][r]);
        float sum = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const float f = wm[k][r] == -INFINITY ? (wl[k][r] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(wm[k][r] - m);      // (nothing but NaN has no maximum: the NaN stays)
            sum += f * wl[k][r];
            o += f * *reinterpret_cast<const f32x4*>(smem + k * STAGE + (r * HDP + d) * 4);
        }
        const int tok = (w.row0 + r) / a.G, hq = w.g * a.G + (w.row0 + r - tok * a.G);
        if (whole) {
            const float inv = sum > 0.f ? 1.f / sum : sum;
            *reinterpret_cast<bf16x4*>(a.o + (int64_t)(w.q0 + tok) * a.ldo + hq * a.hd + d) = bf16x4{(bf16)(o[0] * inv), (bf16)(o[1] * inv), (bf16)(o[2] * inv), (bf16)(o[3] * inv)};
        } else {
            const int64_t rid = (int64_t)part * a.N * a.Hq + (int64_t)(w.q0 + tok) * a.Hq + hq;
            *reinterpret_cast<f32x4*>(a.part + rid * a.hd + d) = o;
            if (d == 0) {
                float* ml = a.part + (int64_t)a.nsplit * a.N * a.Hq * a.hd + 2 * rid;
                ml[0] = m;
                ml[1] = sum;
            }
        }
    }
}

// The parts of one (row, q head), in a fixed order.  WPR waves work on it: lanes over quads of dims and over parts (64 / ql parts at once in a wave), so that even 64 parts are two rounds
// of loads; the partial sums meet in LDS.  WPR = 4 from 9 parts on, else one wave, four of them to a block.
template <int UNIT, int WPR>
__global__ __launch_bounds__(256) void attn_paged_join_k(PagedAttn a, int ql) {
    __shared__ float red[4][64 * 4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t id = WPR == 4 ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (id >= (int64_t)a.N * a.Hq) return;
    const int n = __builtin_amdgcn_readfirstlane((int)(id / a.Hq)), hq = __builtin_amdgcn_readfirstlane((int)(id % a.Hq));
    const int s = paged_slot_of_row(a.t.cu_q, a.t.S, n);
    if (s >= a.t.S) return;
    const int q0 = a.t.cu_q[s], q1 = a.t.cu_q[s + 1];
    if (n < q0 || n >= q1 || q0 < 0 || q1 > a.N) return;
    const int len = paged_len(a.t, s), keys = paged_part<UNIT>(len, a.nsplit) * UNIT;
    if (keys >= len) return;                                                           // one part: written already
    const int parts = (min(paged_seen(a, len, q1 - q0, n - q0), len) + keys - 1) / keys;      // <= 64
    const int64_t stride = (int64_t)a.N * a.Hq, rid = (int64_t)n * a.Hq + hq;
    float mp = -INFINITY, lp = 0.f;
    if (lane < parts) {
        const f32x2 v = *reinterpret_cast<const f32x2*>(a.part + a.nsplit * stride * a.hd + 2 * (lane * stride + rid));
        mp = v[0];
        lp = v[1];
    }
    const float m = wave_max(mp);
    const float f = mp == -INFINITY ? (lp == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mp - m);      // (a part of nothing but NaN has no maximum: its NaN stays)
    const float sum = wave_sum(f * lp), inv = sum > 0.f ? 1.f / sum : sum;
    const int quad = lane & (ql - 1), sub = lane / ql, np = 64 / ql;                   // ql: lanes per part, the power of two from hd / 4 on
    const bool mine = quad * 4 < a.hd;
    const float* x = a.part + rid * a.hd + quad * 4;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = (WPR == 4 ? wave * np : 0); p0 < parts; p0 += 4 * WPR * np) {
        f32x4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = p0 + k * WPR * np + sub;
            v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (mine && p < parts) v[k] = *reinterpret_cast<const f32x4*>(x + p * stride * a.hd);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = p0 + k * WPR * np + sub;
            const float fp = __shfl(f, p < parts ? p : 0, 64);
            if (p < parts) o += fp * v[k];
        }
    }
    for (int d = ql; d < 64; d <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], d, 64);
    if (WPR == 4) {
        *reinterpret_cast<f32x4*>(&red[wave][lane * 4]) = o;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int k = 1; k < 4; ++k) o += *reinterpret_cast<const f32x4*>(&red[k][lane * 4]);
    }
    if (sub == 0 && mine) *reinterpret_cast<bf16x4*>(a.o + (int64_t)n * a.ldo + hq * a.hd + quad * 4) = bf16x4{(bf16)(o[0] * inv), (bf16)(o[1] * inv), (bf16)(o[2] * inv), (bf16)(o[3] * inv)};
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
struct Plan {
    bool keys;              // keys split over the waves (else rows)
    int rows, unit, tiles, nsplit;
};

// N, S: packed rows and slots; the lengths are on the device, the choice is made from the sizes alone.  A slot has N / S rows on average.
Plan make_plan(int N, int S, int Hq, int Hkv, int hd, int max_keys) {
    const int G = Hq / Hkv;
    const int64_t rows = (int64_t)N * G;
    Plan p;
    p.keys = rows <= 32 * (int64_t)S;
    const int nw = hd > 128 ? 4 : 8;
    p.rows = p.keys ? 32 : 128;
    p.unit = p.keys ? 32 * nw : 64;
    p.tiles = (int)(rows / p.rows) + S;
    const int64_t full = rows / p.rows > S ? rows / p.rows : (N < S ? N : S);          // tiles that hold rows, about
    const int64_t blocks = full * Hkv, want = p.keys ? 256 : 512;
    const int64_t steps = ((int64_t)max_keys + p.unit - 1) / p.unit;
    int64_t ns = blocks >= want ? 1 : (want + blocks - 1) / blocks;
    if (ns > steps / 2) ns = steps / 2;
    if (ns > 64) ns = 64;
    p.nsplit = ns < 1 ? 1 : (int)ns;
    return p;
}

template <int UNIT>
void join(const PagedAttn& a, hipStream_t st) {
    int ql = 2;
    while (ql * 4 < a.hd) ql <<= 1;
    const int64_t rows = (int64_t)a.N * a.Hq;
    if (a.nsplit > 8) hipLaunchKernelGGL((attn_paged_join_k<UNIT, 4>), dim3((unsigned)rows), dim3(256), 0, st, a, ql);
    else hipLaunchKernelGGL((attn_paged_join_k<UNIT, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, ql);
}

template <int HDP, int QG>
void launch_tile(const PagedAttn& a, const Plan& p, hipStream_t st) {
    using C = PCfg<HDP>;
    constexpr int smem = 2 * 64 * (C::PK + C::PV);
    UFV_ONCE_PER_DEVICE((void)hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_paged_tile_k<HDP, QG, 4>), hipFuncAttributeMaxDynamicSharedMemorySize, smem););
    const int64_t total = (int64_t)p.tiles * a.Hkv * p.nsplit;
    hipLaunchKernelGGL((attn_paged_tile_k<HDP, QG, 4>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(256), smem, st, a);
    if (p.nsplit > 1) join<64>(a, st);
}

template <int HDP>
int launch(const PagedAttn& a, const Plan& p, hipStream_t st) {
    using C = PCfg<HDP>;
    constexpr int NW = HDP > 128 ? 4 : 8;
    if (p.keys) {
        constexpr int smem = NW * 32 * (C::PK + C::PV);
        UFV_ONCE_PER_DEVICE((void)hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_paged_keys_k<HDP, NW>), hipFuncAttributeMaxDynamicSharedMemorySize, smem););
        hipLaunchKernelGGL((attn_paged_keys_k<HDP, NW>), dim3(p.tiles, p.nsplit, a.Hkv), dim3(NW * 64), smem, st, a);
        if (p.nsplit > 1) join<32 * NW>(a, st);
    } else {
        launch_tile<HDP, 1>(a, p, st);
    }
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

}  // namespace

extern "C" int64_t ufv_attention_paged_ws_bytes(int N, int S, int Hq, int Hkv, int hd, int max_keys) {
    if (N <= 0 || S <= 0 || Hkv <= 0 || Hq < Hkv || hd <= 0) return 0;
    const Plan p = make_plan(N, S, Hq, Hkv, hd, max_keys);
    return p.nsplit > 1 ? 4 * (int64_t)p.nsplit * N * Hq * (hd + 2) : 0;
}

extern "C" int ufv_attention_paged(const void* q, int64_t ldq, void* o, int64_t ldo, int N, int Hq, int Hkv, int hd, const void* pages, int n_pages, int page, int64_t ldkv,
                                   const int32_t* block_table, int64_t ld_table, int max_pages, const int32_t* cu_q, const int32_t* kv_len, int S, float scale, int causal, void* ws,
                                   int64_t ws_bytes, void* stream) {
    UFV_REQUIRE_PAGED("ufv_attention_paged", pages, n_pages, page, ldkv, block_table, ld_table, max_pages, cu_q, kv_len, S);
    UFV_REQUIRE(q && o && N > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "ufv_attention_paged: bad arguments (N=%d, %d q heads on %d kv heads)", N, Hq, Hkv);
    UFV_REQUIRE(hd >= 8 && hd <= 256 && hd % 8 == 0, "ufv_attention_paged: head_dim must be a multiple of 8 up to 256 (%d)", hd);
    UFV_REQUIRE(scale > 0.f && scale < INFINITY, "ufv_attention_paged: the scale must be positive and finite (%g)", (double)scale);
    UFV_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)o % 16 == 0 && ldq % 8 == 0 && ldo % 8 == 0, "ufv_attention_paged: rows must be 16-byte aligned (pitches %lld, %lld)", (long long)ldq,
                (long long)ldo);
    UFV_REQUIRE(ldkv >= 2 * (int64_t)Hkv * hd && (N == 1 || (ldq >= (int64_t)Hq * hd && ldo >= (int64_t)Hq * hd)), "ufv_attention_paged: a row pitch is too small");
    UFV_REQUIRE((int64_t)N * Hq < 0x7fffffff && S < 1 << 24, "ufv_attention_paged: too many rows or slots (N=%d S=%d)", N, S);
    const Plan p = make_plan(N, S, Hq, Hkv, hd, max_pages << paged_log2(page));
    UFV_REQUIRE((int64_t)p.tiles * Hkv * p.nsplit < 0x7fffffff - 8 && Hkv < 65536, "ufv_attention_paged: too many row tiles (N=%d S=%d)", N, S);
    UFV_REQUIRE(p.nsplit == 1 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= ufv_attention_paged_ws_bytes(N, S, Hq, Hkv, hd, max_pages << paged_log2(page))),
                "ufv_attention_paged: a workspace of %lld bytes is needed (%lld given)", (long long)ufv_attention_paged_ws_bytes(N, S, Hq, Hkv, hd, max_pages << paged_log2(page)), (long long)ws_bytes);
    PagedAttn a;
    a.q = (const bf16*)q; a.pages = (const bf16*)pages; a.o = (bf16*)o;
    a.ldq = ldq; a.ldo = ldo; a.ldkv = ldkv;
    a.t = PagedTable{block_table, ld_table, max_pages, cu_q, kv_len, S, n_pages, paged_log2(page)};
    a.N = N; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.hd = hd; a.causal = causal != 0;
    a.sl2 = scale * 1.4426950408889634f;
    a.nsplit = p.nsplit; a.tiles = p.tiles; a.part = (float*)ws;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (hd <= 32) return launch<32>(a, p, st);
    if (hd <= 64) return launch<64>(a, p, st);
    if (hd <= 96) return launch<96>(a, p, st);
    if (hd <= 128) return launch<128>(a, p, st);
    return launch<256>(a, p, st);
}
