// Attention of a chunk of new tokens over a paged KV cache (see paged.h for the layout).
//   o[r, h] = sum_j softmax_j(q[r, h] . k[j, g] * scale) v[j, g],  g = h / G,  G = Hq / Hkv,  over the keys j < kv_len[s] (causal: j <= the row's own position);
// a row that sees no key gets zeros, one that sees keys of score -inf only NaN.  Keys that do not exist -- behind kv_len, in a page outside the pool -- are staged as zeros and their scores are -inf.
//
// The unit of work is a TILE of rows of one slot and one kv head, a row being a (token, q head of the group) pair: row r of a slot is token r / G, head g * G + r % G.  All G heads
// that share a kv head sit in one tile, so that every key is fetched once for the group and a single token already fills G of the 32 columns of a matrix instruction.
//
// Both kernels compute S^T = K Q^T with v_mfma_f32_32x32x16_bf16 (a lane owns one row of the tile: its column of S^T), keep the running maximum and sum of the softmax in
// 32 bits (log2 domain), and use the exponentiated tile, rounded to bf16, directly as the B operand of O^T += V^T P^T.  The rounding of P is the one step below 32 bits between
// the inputs and the output: the matrix instruction takes bf16 operands; the row sum is taken of the unrounded values.  V^T fragments come from row-major V rows in LDS by the transposing read.
//   attn_paged_tile_k   the waves of a block share 64-key tiles and split the ROWS: chunks of many rows, bound by the matrix unit.  28 / 4 heads of 128: 2399 tokens over 20011 in 690 us
//                       (0.94 PF/s with its join; 650 .. 725 from run to run), 8192 causal tokens 575 us, 16 questions of 12 .. 82 tokens behind 2304 shared ones 49 us and 9 for the join
//                       (0.44 PF/s: 14 steps a block of 2.2 us, 11 of starts and ends, 6 until the longest block is done)
//   attn_paged_keys_k   the waves of a block share up to 32 rows and split the KEYS: a few new tokens over a long cache, bound by the bytes of the cache.  48 slots of 792 .. 6045 tokens
//                       73 us and 5 for the join (4.4 TB/s; a large read reaches 6.1), one of 31999 17 us and 6 (2.8 TB/s: 4 us until the first keys are asked for)
// The work is cut over the keys for the 256 CUs; the parts leave (max, sum, un-normalised O) in 32 bits in the workspace and attn_paged_join_k adds them in order.
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
    int tiles;              // row tiles (upper bound)
    int target, sh;         // keys kernel: parts of a head that are aimed at (0: no item is cut), log2 of the keys of its step
    int cuts, parts;        // what the workspace holds: PCut [cuts], then the parts (paged_part)
    float* ws;
};

// What the join has to know of an item that several blocks worked on (parts = 0: nothing to do).  A part is un-normalised O as the lanes of the tile kernel hold it --
// [32 rows][HDP / 8][64 lanes][4], so that every store is whole lines -- then R pairs (max, sum).
struct PCut { int first, parts;               // its first part (tile kernel: that part's worker); the number of its parts
              int q0, row0, rows, g;          // as in PagedTile
              int used, pad; };               // (of the first: how many records are valid)
__device__ __forceinline__ PCut* paged_cut(const PagedAttn& a) { return reinterpret_cast<PCut*>(a.ws); }
template <int HDP>
__device__ __forceinline__ int part_at(int row, int quad) { return (((row >> 5) * (HDP / 8) + (quad >> 1)) * 64 + (quad & 1) * 32 + (row & 31)) * 4; }
template <int HDP, int R>
__device__ __forceinline__ float* paged_part(const PagedAttn& a, int i) { return a.ws + (int64_t)a.cuts * (sizeof(PCut) / 4) + (int64_t)i * (R * (HDP + 2)); }

// what a block works on: all of it wave-uniform
struct PagedTile {
    int s, q0, n, len;      // slot, its first packed row, its rows, its cached tokens
    int row0, rows;         // the tile's first (token, head) row, all such rows of the slot
    int g;                  // kv head
};

// Row tiles of R rows are numbered over the batch without the host knowing the lengths: slot s may use the numbers from floor(cu_q[s] * G / R) + s on; the next slot's first number is never
// less than what slot s needs (ceil(n G / R)).  Numbers without rows have no work.
template <int R>
__device__ __forceinline__ int paged_number(int G, int s, int cu) { return (int)((int64_t)cu * G / R) + s; }

// keys that row r of a slot sees: tokens 0 .. paged_seen - 1
__device__ __forceinline__ int paged_seen(const PagedAttn& a, int len, int n, int tok) { return a.causal ? max(len - n + tok + 1, 0) : len; }

// inclusive prefix sums over the wave, by lane shifts within rows of 16 and the row ends passed on
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T lane_shift(T x) {
    if constexpr (sizeof(T) == 8) {
        const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
        return (T)((uint64_t)hi << 32 | lo);
    } else {
        return (T)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
    }
}
template <class T>
__device__ __forceinline__ T lane_scan(T x) {
    x += lane_shift<0x111, 0xf>(x);                       // row_shr 1, 2, 4, 8
    x += lane_shift<0x112, 0xf>(x);
    x += lane_shift<0x114, 0xf>(x);
    x += lane_shift<0x118, 0xf>(x);
    x += lane_shift<0x142, 0xa>(x);                       // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
    return x + lane_shift<0x143, 0xc>(x);
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

// K and V rows in LDS: P bytes a row, chunk c (16 bytes) of row r at slot c ^ f(r) -- without padding, so that a row can come straight from memory, and free of bank conflicts: eight rows'
// same chunk (a K fragment) and four rows' neighbouring chunk pairs (a transposing V read) fall on different banks.  The matrix instructions' addresses are one per lane, XORed with constants.
template <int HDP>
struct PCfg {
    static constexpr int KS = HDP / 16, DT = HDP / 32;
    static constexpr int CPR = HDP <= 32 ? 4 : (HDP <= 64 ? 8 : (HDP <= 128 ? 16 : 32));     // chunks of a row, lanes that fetch it (a power of two; HDP 96: four more than it has)
    static constexpr int RPW = 64 / CPR;                                                     // rows of one wave load: at most 16, so all of one page
    static constexpr int P = CPR * 16;
    __device__ static __forceinline__ int f(int r) { return CPR >= 16 ? 2 * (r & 7) : (CPR == 8 ? r & 7 : (r >> 2) & 3); }
    // lane (l31, h): K row l31 chunk 2 ks + h at kaddr ^ (ks << 5); 32 rows on: + 32 P
    __device__ static __forceinline__ int kaddr(int lane) { return (lane & 31) * P + 16 * ((lane >> 5) ^ f(lane & 31)); }
    // lane's part of the transposing reads of keys 4 h .. 4 h + 3 (the second: 8 keys on), dims 32 dt ..: vaddr ^ (dt << 6), second: (vaddr ^ VX) + 8 P; 16 keys on: + 16 P
    static constexpr int VX = CPR == 4 ? 32 : 0;
    __device__ static __forceinline__ int vaddr(int lane) {
        const int r = 4 * (lane >> 5) + ((lane & 15) >> 2), u = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        return r * P + 16 * (u ^ f(r)) + 8 * (lane & 1);
    }
};

// what a lane keeps of its row: its part of O^T, the running maximum (log2 domain), its half of the running sum
template <int HDP>
struct PState {
    f32x16 o[HDP / 32];
    float m, l;
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    }
};

// NH half tiles of 32 keys in LDS (K rows at kb, V rows at vb) against 32 rows: S^T, running softmax, O^T.  hide: key j of the step counts for the lane's row iff j < vis and, in groups of 16
// keys, iff its bit of `groups` is set.
// at_qk(i, n, next) runs behind the i-th of the n products of S^T: the loads of a later step (memory -> LDS at `next`) go there, a few at a time -- issued in one go they hold the wave
// (the memory pipe takes one 1 KB load in 16 cycles), behind the products they cost little.  kb, vb, next do not overlap (__restrict__ lets the compiler
// keep the loads in flight across the reads: who issues them waits for them before the barrier that publishes them).
// A step of 64 keys at head_dim 128 is 1024 cycles of the matrix unit, two waves a SIMD: 2048.  16384 tokens over 8192 keys (28 / 4 heads) run at 1.02 PF/s, 4400 cycles a step; without the LDS reads they
// would take 7 % less, without the exponentials 8 %, without the loads 7 %, without all three 23 % -- no one of them bounds it, and then the clock falls: the products alone reach 1.26 PF/s, a
// large library product 1.41.  Tried and slower: the exponentials between the products of the next step's S^T (8 %; the maximum between those of O^T), 64 rows a wave (30 %), waves in two groups
// half a step apart (4 %).
template <int HDP, int NH, class FQ>
__device__ __forceinline__ void paged_step(const char* __restrict__ kb, const char* __restrict__ vb, char* __restrict__ next, const bf16x8 (&qf)[HDP / 16], PState<HDP>& st, float sl2, bool hide, int vis,
                                           unsigned groups, FQ&& at_qk) {
    using C = PCfg<HDP>;
    const int lane = threadIdx.x & 63, h = lane >> 5;
    int k_off = C::kaddr(lane), v_off = C::vaddr(lane);
    if (NH == 1) asm volatile("" : "+v"(k_off), "+v"(v_off));      // opaque: the keys kernel holds a step of K and V in registers and has none left for the fragments' addresses
    // Left to itself the compiler puts every LDS read right in front of the matrix instruction that needs it and waits out the LDS latency 32 times a step.  The order below is pinned
    // (sched_barrier): AHEAD fragments are in flight at any time, the V reads start before the exponentials, and the second half's exponentials go between the first half's products.
    constexpr int AHEAD = 4, NR = C::KS * NH, PRE = AHEAD < NR ? AHEAD : NR;
    f32x16 s[NH];
#pragma unroll
    for (int hh = 0; hh < NH; ++hh)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[hh][r] = 0.f;
    // NH = 2: a wave among its products goes before one among its exponentials (two of different blocks on a SIMD: 8 x 1000 causal tokens 126 -> 121 us, 16 questions 59 -> 56)
    {
        bf16x8 kf[PRE];
        auto read = [&](int i) { return *reinterpret_cast<const bf16x8*>(kb + (k_off ^ ((i / NH) << 5)) + (i % NH) * 32 * C::P); };
#pragma unroll
        for (int i = 0; i < PRE; ++i) kf[i] = read(i);
        __builtin_amdgcn_sched_barrier(0);
        if (NH == 2) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            s[i % NH] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i % PRE], qf[i / NH], s[i % NH], 0, 0, 0);
            if (i + PRE < NR) kf[i % PRE] = read(i + PRE);
            at_qk(i, NR, next);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (NH == 2) __builtin_amdgcn_s_setprio(0);
    if (hide) {
        const int lim = vis - 4 * h;
#pragma unroll
        for (int hh = 0; hh < NH; ++hh)
#pragma unroll
            for (int r = 0; r < 16; ++r)                              // key hh * 32 + (r & 3) + 8 (r >> 2) + 4 h
                s[hh][r] = hh * 32 + (r & 3) + 8 * (r >> 2) < lim && ((groups >> (2 * hh + (r >> 3))) & 1) ? s[hh][r] : -INFINITY;
    }
    float tmax = s[0][0];
#pragma unroll
    for (int hh = 0; hh < NH; ++hh)
#pragma unroll
        for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s[hh][r]);
    tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64)) * sl2;
    // the rescale of O waits until the maximum has grown by 2^6: until then the exponentials stay below 2^6.  No bits are lost, but range is: O before the division is up to 64 sum |v| (a sum of
    // weights up to 1 would be up to sum |v|) and has to stay below 2^128
    if (__any(tmax > st.m + 6.0f)) {
        const float mnew = fmaxf(st.m, tmax);
        const float alpha = mnew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m - mnew);
        st.l *= alpha;
#pragma unroll
        for (int i = 0; i < C::DT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[i][r] *= alpha;
        st.m = mnew;
    }
    const float msub = st.m == -INFINITY ? 0.f : st.m;
    constexpr int NM = 2 * C::DT, NV = NM * NH, PREV = AHEAD < NV ? AHEAD : NV, EPM = (16 + NM - 1) / NM;      // products of a half, of the step; elements per product
    bf16x4 vf[PREV][2];
    auto readv = [&](int i, int u) {                       // product i: keys 16 (i / DT) .., dims 32 (i % DT) ..
        const char* vp = vb + ((v_off ^ ((i % C::DT) << 6)) ^ (u ? C::VX : 0)) + (16 * (i / C::DT) + 8 * u) * C::P;
        return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((bf16x4 __attribute__((address_space(3)))*)(vp));
    };
#pragma unroll
    for (int i = 0; i < PREV; ++i) { vf[i][0] = readv(i, 0); vf[i][1] = readv(i, 1); }
    __builtin_amdgcn_sched_barrier(0);
    float sum = 0.f;
    auto exps = [&](int hh, int r0, int r1) {
#pragma unroll
        for (int r = r0; r < r1; ++r) {
            s[hh][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[hh][r], sl2, -msub));
            sum = hh == 0 && r == 0 ? s[hh][r] : sum + s[hh][r];
        }
    };
    exps(0, 0, 16);
    bf16x8 pf[2];
    if (NH == 2) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i % NM == 0) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float p[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) p[r] = s[i / NM][8 * c + r];
                pf[c] = pack8(p);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        const bf16x8 v = __builtin_shufflevector(vf[i % PREV][0], vf[i % PREV][1], 0, 1, 2, 3, 4, 5, 6, 7);
        st.o[i % C::DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, pf[(i % NM) / C::DT], st.o[i % C::DT], 0, 0, 0);
        if (i + PREV < NV) { vf[i % PREV][0] = readv(i + PREV, 0); vf[i % PREV][1] = readv(i + PREV, 1); }
        if (NH == 2 && i < NM) exps(1, EPM * i < 16 ? EPM * i : 16, EPM * (i + 1) < 16 ? EPM * (i + 1) : 16);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (NH == 2) __builtin_amdgcn_s_setprio(0);
    st.l += sum;
}

// zero the non-finite elements of a chunk; true if there was one
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

// A key that a row does not see must not reach it even when its V row holds Inf or NaN (0 * Inf in the matrix product): among the new tokens of a causal chunk -- the only keys
// that some rows see and others do not -- such elements are staged as zeros, and if there was one, they are added after the walk to the rows that see them (keys j0 .. j1 - 1;
// p > 0 times Inf or NaN is Inf or NaN; a K row with such an element has no finite score, so p is 0 or NaN and the product NaN).  Whole steps are cleaned, so the range begins at the first
// key of the step that holds the first new token, not at that token.
template <int HDP>
__device__ __forceinline__ void paged_add_bad(const PagedAttn& a, const PagedTile& w, int j0, int j1, PState<HDP>& st, int seen) {
    int h = (threadIdx.x & 63) >> 5;
    asm volatile("" : "+v"(h));                           // opaque: nothing of this path is kept in registers outside it
    for (int j = j0; j < j1; ++j) {
        const int64_t at = paged_row(a.t, w.s, j);
        if (at < 0) continue;
        const bf16 *k = a.pages + at * a.ldkv + w.g * a.hd, *v = k + a.Hkv * a.hd;
        const int lane = threadIdx.x & 63;
        u32x4 kc = {0, 0, 0, 0};
        if (lane * 8 < a.hd) kc = *reinterpret_cast<const u32x4*>(k + lane * 8);
        const bool nan = __any(paged_clean(kc));
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
                        if (!(fabsf((float)x[e]) < INFINITY) && j < seen) st.o[dt][4 * g4 + e] += nan ? __builtin_nanf("") : (float)x[e];
                }
            }
    }
}

// A row without a finite score has the maximum -inf and no weight at all.  Its sum is 0 where it sees no key (the row is zeros), and this where it sees keys, all of score -inf: 0 times the
// inverse, which is past 2^128, is the NaN of a row that has no softmax.  To a sum with a weight in it (at least about 1) this adds nothing.
constexpr float NO_WEIGHT = 0x1p-149f;
// behind a walk over the keys j0 .. j1 - 1
template <int HDP>
__device__ __forceinline__ void paged_no_weight(const PagedAttn& a, const PagedTile& w, int j0, int j1, PState<HDP>& st, int seen) {
    if (!__any(st.m == -INFINITY)) return;
    const int end = min(j1, w.len);
    while (j0 < end && paged_row(a.t, w.s, j0) < 0) j0 += 16;                          // the first key that exists
    if (st.m == -INFINITY && st.l == 0.f && j0 < min(seen, end)) st.l = NO_WEIGHT;
}

// The lane's rows of the tile as B operands (lane: row l31 of the group, dims 16 ks + 8 h ..), and what they see.  Rows behind the tile's last take the last one's q; they are not stored.
template <int HDP>
__device__ __forceinline__ int paged_load_q(const PagedAttn& a, const PagedTile& w, int row0, bf16x8 (&qf)[HDP / 16]) {
    const int lane = threadIdx.x & 63;
    int h = lane >> 5;
    asm volatile("" : "+v"(h));                           // opaque: the bounds of the chunks must not be kept in registers over the walk
    const int r = min(row0 + (lane & 31), w.rows - 1), tok = r / a.G, hq = w.g * a.G + (r - tok * a.G);
    const bf16* p = a.q + (int64_t)(w.q0 + tok) * a.ldq + hq * a.hd + h * 8;
#pragma unroll
    for (int ks = 0; ks < HDP / 16; ++ks) {
        qf[ks] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (ks * 16 + h * 8 < a.hd) qf[ks] = *reinterpret_cast<const bf16x8*>(p + ks * 16);
    }
    return paged_seen(a, w.len, w.n, tok);
}

// A lane's place in a load of rows (see PFetch): chunk sch of row srow.  Lanes whose chunk lies behind hd (padded head dims) ask for a place behind every range and get zeros: Q is 0 there, but
// so must K be (0 * Inf is NaN: a finite row with one score of -inf would become NaN).  A range has fewer than 2^29 bytes: 16 rows, ldkv below 2^24.
__device__ __forceinline__ unsigned paged_lane_offset(const PagedAttn& a, int srow, int sch) {
    return sch * 8 < a.hd ? (unsigned)(srow * (int)a.ldkv + sch * 8) * 2 : 0x7ffffff0u;
}

// Fetching NG groups of 16 keys (a step) by NWS waves.  A wave load covers RPW <= 16 rows that start at a multiple of RPW, and a page holds whole groups of 16 tokens: the page is the same
// for the whole load and its address a scalar; the lane's part of the address does not change.  It is a buffer load whose base is the load's first row and whose range ends behind the last row
// that is a key: what lies outside -- tokens behind the last one, a page outside the pool -- comes back as zeros and is not read.  Page ids: one vector load
// holds those of 64 groups, one a lane.
template <int HDP, int NG, int NWS>
struct PFetch {
    using C = PCfg<HDP>;
    static constexpr int PASS = NWS * C::RPW, RPT = 16 * NG / PASS, NL = 2 * RPT;       // rows of a pass, passes, loads of a wave (K, then V)
    static constexpr int SPC = 64 / NG;                                                 // steps whose ids one load holds
    static_assert(RPT >= 1 && RPT * PASS == 16 * NG, "whole passes");
    int id[NG];             // page ids of a step, -1 where there is no key or no such page

    // lane i: the id of group 64 c + i (tokens and groups stay below 2^31; past the table's last entry: that one)
    __device__ __forceinline__ static int chunk(const PagedAttn& a, const PagedTile& w, int c) {
        const int i = min((int)(((unsigned)c * 64u + (threadIdx.x & 63)) << 4 >> a.t.sh), a.t.width - 1);
        return *reinterpret_cast<const int*>(reinterpret_cast<const char*>(a.t.table + (int64_t)w.s * a.t.ld) + (unsigned)i * 4u);
    }
    // the ids of `step` out of its chunk; bit i: group i has keys.  From step `end` on there is nothing: no ids, nothing is read
    __device__ __forceinline__ unsigned take(const PagedAttn& a, const PagedTile& w, int ids, int step, int end) {
        unsigned ok = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            id[i] = __builtin_amdgcn_readlane(ids, (step % SPC) * NG + i);
            const bool there = step < end && (step * NG + i) * 16 < w.len && (unsigned)id[i] < (unsigned)a.t.n_pages;
            id[i] = there ? id[i] : -1;
            ok |= there ? 1u << i : 0u;
        }
        return ok;
    }
    // load l (l < RPT: K, else V) of the step whose ids were taken: its base, and the bytes of its range; wave: the wave's place among the NWS
    __device__ __forceinline__ bf16* rows(const PagedAttn& a, const PagedTile& w, int step, int l, int wave, int& bytes) const {
        const int i = l % RPT, j = step * NG * 16 + i * PASS + wave * C::RPW;
        int page = id[(i * PASS) >> 4];
        if (PASS > 16)
#pragma unroll
            for (int x = 1; x < PASS / 16; ++x) page = (wave * C::RPW) >> 4 == x ? id[((i * PASS) >> 4) + x] : page;
        const int keys = max(min((page < 0 ? 0 : w.len) - j, C::RPW), 0), ld = (int)a.ldkv;
        bytes = max(keys * ld - (ld - a.hd), 0) * 2;                                    // up to the end of the last key's chunks of this head
        return const_cast<bf16*>(a.pages) + (((int64_t)max(page, 0) << a.t.sh) + (j & ((1 << a.t.sh) - 1))) * a.ldkv + (l < RPT ? w.g : a.Hkv + w.g) * a.hd;
    }
};

// ---------------------------------------------------------------------------------------------------------------------------------
// rows split over the waves.  The work of a launch is the 64-key steps of all (kv head, row tile) items in order, every item with ITEM_COST steps more for its start and end; every worker (block) takes an equal, contiguous share of them, so that no CU waits for another whatever the lengths are: 528 equal items on 512 block slots would take two
// rounds, the second nearly empty.  A worker walks from where its share begins inside one item to where it ends inside another; an item that lies in one share is stored at once, of the
// others every worker leaves a part to the join.  The start of an item (its q rows, its first keys) is fetched before the stores of the one before it, whose time hides it.
// ---------------------------------------------------------------------------------------------------------------------------------
// ITEM_COST 2 | 3 | 4: 2399 causal tokens (28 / 4 heads of 128) 99 | 92 | 89 us, 16 questions of 9 .. 83 tokens 58 | 58 | 59
constexpr int ITEM_COST = 3;
constexpr int MIN_SHARE = 4;               // steps: the shortest item.  6 | 4: 40 causal tokens 18.5 | 13.0 us, 600 32 | 29, 2399 94 | 93
constexpr int NEAR = 4;                    // steps: a boundary that cuts less than this off an item moves to the item's end: fewer parts, no share longer by more than 1/8

// Block-uniform values into vector registers and back: the state of the share is not used over an item's steps, which need the scalar registers (held there it was spilled, and the reloads stood
// between the products).
template <class... T>
__device__ __forceinline__ void to_vector(T&... x) {
    auto one = [](auto& v) { asm volatile("" : "+v"(v)); };
    (one(x), ...);
}
template <class... T>
__device__ __forceinline__ void to_scalar(T&... x) {
    auto one = [](auto& v) {
        if constexpr (sizeof(v) == 8) v = (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v));
        else v = __builtin_amdgcn_readfirstlane(v);
    };
    (one(x), ...);
}

// a / b of numbers that nearly always fit 32 bits (a 64-bit division takes 1000 cycles)
__device__ __forceinline__ int64_t paged_div(int64_t a, int64_t b) { return ((a | b) >> 32) == 0 ? (int64_t)((unsigned)a / (unsigned)b) : a / b; }

struct PWalkLds {
    static constexpr int MAX = 512;        // slots whose cu_q and kv_len have a copy here
    int cu[MAX + 1], len[MAX];
    int64_t scan[8 + 2];                   // wave sums | the first item: slot and tile, its first step
};

template <int R, int NT>
struct PWalk {
    int64_t per_head, share, pos, end;     // steps of a kv head's items, of a share; the walk's place and end
    int64_t base;                          // steps of the head's items before `tile`
    int worker, g, tile, slot;

    __device__ static __forceinline__ int number(int G, int s, int cu) { return paged_number<R>(G, s, cu); }
    __device__ static __forceinline__ int cu(const PagedAttn& a, const PWalkLds& m, int s) { return a.t.S <= PWalkLds::MAX ? m.cu[s] : a.t.cu_q[s]; }

    // tile t of slot s, which is moved on to the one whose numbers t is among: its rows, its key steps (0: a number without rows; a tile that sees no key takes one, fully masked).
    // UNI: t and s are the same in all lanes
    template <bool UNI>
    __device__ static __forceinline__ int look(const PagedAttn& a, const PWalkLds& m, int t, int& s, PagedTile& w) {
        auto uni = [](int x) { return UNI ? __builtin_amdgcn_readfirstlane(x) : x; };
        int c0 = uni(cu(a, m, s)), c1 = uni(cu(a, m, s + 1));
        while (s + 1 < a.t.S && number(a.G, s + 1, c1) <= t) {
            ++s;
            c0 = c1;
            c1 = uni(cu(a, m, s + 1));
        }
        w.s = s;
        w.q0 = c0;
        w.n = c1 - c0;
        w.row0 = (t - number(a.G, s, c0)) * R;
        if (w.row0 < 0 || w.q0 < 0 || w.n <= 0 || w.q0 + w.n > a.N) return 0;
        w.rows = w.n * a.G;
        if (w.row0 >= w.rows) return 0;
        w.len = uni(a.t.S <= PWalkLds::MAX ? m.len[s] : paged_len(a.t, s));
        const int seen = min(paged_seen(a, w.len, w.n, (min(w.row0 + R, w.rows) - 1) / a.G), w.len);
        return max((seen + 63) >> 6, 1);
    }

    // Every block counts the steps of one kv head's tiles (thread: a run of them) and finds where its share begins; false: there is none.
    __device__ __forceinline__ bool start(const PagedAttn& a, PWalkLds& m) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        if (a.t.S <= PWalkLds::MAX) {
            for (int i = tid; i <= a.t.S; i += NT) m.cu[i] = a.t.cu_q[i];
            for (int i = tid; i < a.t.S; i += NT) m.len[i] = paged_len(a.t, i);
        }
        if (tid == 0) m.scan[8] = m.scan[9] = 0;
        __syncthreads();
        const int run = (a.tiles + NT - 1) / NT, t0 = min(tid * run, a.tiles), t1 = min(t0 + run, a.tiles);
        int s = 0;
        for (int lo = 0, hi = a.t.S; lo < hi;) {           // the last slot whose numbers start at or before t0
            const int mid = (lo + hi) >> 1;
            if (number(a.G, mid, cu(a, m, mid)) <= t0) { s = mid; lo = mid + 1; } else hi = mid;
        }
        PagedTile w;
        auto steps = [&](int t, int& s) { const int c = look<false>(a, m, t, s, w); return c ? c + ITEM_COST : 0; };
        int64_t mine = 0;
        int s1 = s;
        for (int t = t0; t < t1; ++t) mine += steps(t, s1);
        const int64_t x = lane_scan(mine);
        if (lane == 63) m.scan[wave] = x;
        __syncthreads();
        int64_t before = x - mine;
        per_head = 0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
            before += i < wave ? m.scan[i] : 0;
            per_head += m.scan[i];
        }
        to_scalar(per_head);
        const int64_t total = per_head * a.Hkv;
        int64_t workers = total / MIN_SHARE;
        workers = workers < 1 ? 1 : (workers > gridDim.x ? gridDim.x : workers);
        share = max(paged_div(total + workers - 1, workers), (int64_t)1);
        workers = paged_div(total + share - 1, share);
        // ids that differ by 8 run on one XCD: every XCD gets a contiguous run of shares, whose items share a kv head's keys in its L2
        const int per = (int)((workers + 7) >> 3), id = blockIdx.x;
        worker = (id & 7) * per + (id >> 3);
        if (id == 0 && tid == 0) paged_cut(a)->used = (int)workers;
        if ((id >> 3) >= per || worker >= workers) return false;
        pos = worker * share;
        end = min(pos + share, total);
        g = (int)paged_div(pos, per_head);
        const int64_t off = pos - g * per_head;
        if (off >= before && off < before + mine) {
            int64_t at = before;
            for (int t = t0; t < t1; ++t) {
                const int c = steps(t, s);
                if (off < at + c) { m.scan[8] = ((int64_t)s << 32) | t; m.scan[9] = at; break; }
                at += c;
            }
        }
        __syncthreads();
        tile = (int)m.scan[8];
        slot = (int)(m.scan[8] >> 32);
        base = m.scan[9];
        if (tid == 0) paged_cut(a)[worker].parts = 0;
        return true;
    }

    // the next item of the share, its steps t0 .. t1 - 1, cut: it lies in several shares; false: there is none
    __device__ __forceinline__ bool next(const PagedAttn& a, const PWalkLds& m, PagedTile& w, int& t0, int& t1, bool& cut) {
        to_scalar(per_head, share, pos, end, base, worker, g, tile, slot);
        bool more = false;
        while (!more && pos < end && g < a.Hkv) {
            const int cost = look<true>(a, m, tile, slot, w);
            w.g = g;
            if (cost) {
                const int64_t first = g * per_head + base + ITEM_COST;                      // the unit of the item's first step
                const int near = (int)min(max(share >> 3, (int64_t)1), (int64_t)NEAR);
                auto clip = [&](int64_t unit) {                                        // a share's end in steps of the item
                    const int64_t x = unit - first;
                    return x >= cost ? cost : (x < near ? 0 : (cost - x < near ? cost : (int)x));
                };
                t0 = clip(worker * share);
                t1 = clip(end);
                cut = t0 != 0 || t1 != cost;
                more = t0 < t1;
                if (more && t0 > 0 && t1 == cost && threadIdx.x == 0) {           // at most one item a share: its record
                    const int w0 = (int)paged_div(first + near - 1, share);            // the first whose share reaches a step of the item
                    PCut* c = paged_cut(a) + worker;
                    c->first = w0;
                    c->parts = worker - w0 + 1;
                    c->q0 = w.q0;
                    c->row0 = w.row0;
                    c->rows = w.rows;
                    c->g = g;
                }
                pos = first + cost;
                base += cost + ITEM_COST;
            }
            if (++tile >= a.tiles || base >= per_head) { tile = slot = 0; base = 0; ++g; }
        }
        to_vector(per_head, share, pos, end, base, tile, slot);
        return more;
    }
    __device__ __forceinline__ int me() const { return __builtin_amdgcn_readfirstlane(worker); }
};

template <int HDP, int NW, int NS>
__global__ __launch_bounds__(NW * 64, HDP > 128 ? 1 : HDP > 32 ? 2 : 4) void attn_paged_tile_k(PagedAttn a) {
    using C = PCfg<HDP>;
    constexpr int R = 32 * NW, HALF = 64 * C::P, STAGE = 2 * HALF;                         // a step's K rows, its K and V rows
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ int dirty;
    __shared__ PWalkLds shared;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, l31 = lane & 31;
    if (tid == 0) dirty = 0;
    PWalk<R, NW * 64> walk;
    if (!walk.start(a, shared)) return;
    const int srow = lane / C::CPR, sch = (lane % C::CPR) ^ C::f(wave * C::RPW + srow);  // the lane's row in a load, the chunk that belongs into its place
    const unsigned lane_off = paged_lane_offset(a, srow, sch);

    using F = PFetch<HDP, 4, NW>;
    constexpr int NL = F::NL, D = NS - 1;                                              // steps ahead
    F fe;
    PState<HDP> st;
    bf16x8 qf[C::KS];
    PagedTile w = {}, old = {};                                                        // the item, the one before
    int t0 = 0, t1 = 0, seen = 0, seen_min = 0, diag = 0;
    bool cut = false;                                                                  // the item lies in several shares
    int ids = 0, ids2 = 0;                                                             // of the step to be fetched next and its neighbours, of the chunk behind it
    unsigned groups[NS];                                                               // which groups of 16 keys of the steps under way exist
    auto dma = [&](int t, int l, char* buf) {
        int bytes;
        bf16* base = fe.rows(a, w, t, l, wave, bytes);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(base, 0, bytes, 0x20000), LDS_PTR(buf + (l < NL / 2 ? 0 : HALF) + ((l % (NL / 2)) * F::PASS + wave * C::RPW) * C::P), 16, lane_off, 0, 0, 0);
    };
    for (bool have = false;; have = true) {
        // ---- the next item of the share and its first loads
        const int old_t0 = t0;
        const bool old_cut = cut;
        old = w;
        const bool more = walk.next(a, shared, w, t0, t1, cut);
        if (more) {
            seen = paged_load_q<HDP>(a, w, w.row0 + wave * 32, qf);
            ids = F::chunk(a, w, t0 / F::SPC);
            ids2 = F::chunk(a, w, t0 / F::SPC + 1);
            seen_min = min(paged_seen(a, w.len, w.n, min(w.row0 + wave * 32, w.rows - 1) / a.G), w.len);
            diag = a.causal && w.n > 1 ? w.len - w.n : 0x7fffffff;                     // keys from here on are seen by some rows only
#pragma unroll
            for (int d = 0; d < D; ++d) {
                if (d > 0 && (t0 + d) % F::SPC == 0) { ids = ids2; ids2 = F::chunk(a, w, (t0 + d) / F::SPC + 1); }
                groups[d] = fe.take(a, w, ids, t0 + d, t1);
#pragma unroll
                for (int l = 0; l < NL; ++l) dma(t0 + d, l, smem + d * STAGE);
            }
        }
        // ---- O of the item before
        if (have) {
            int he = h;                                                                 // opaque: what follows from it (dims, bounds, addresses) must not be kept in registers over the walk
            asm volatile("" : "+v"(he));
            const float l = st.l + __shfl_xor(st.l, 32, 64);
            const int r = old.row0 + wave * 32 + l31;
            if (!old_cut) {
                const int tok = min(r, old.rows - 1) / a.G, hq = old.g * a.G + (r - tok * a.G);
                const float inv = l > 0.f ? 1.f / l : l;                               // l = 0: no key; NaN stays NaN
                bf16* op = a.o + (int64_t)(old.q0 + tok) * a.ldo + hq * a.hd;
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        const int d = dt * 32 + g4 * 8 + he * 4;
                        if (r < old.rows && d < a.hd)
                            *reinterpret_cast<bf16x4*>(op + d) = bf16x4{(bf16)(st.o[dt][g4 * 4] * inv), (bf16)(st.o[dt][g4 * 4 + 1] * inv), (bf16)(st.o[dt][g4 * 4 + 2] * inv), (bf16)(st.o[dt][g4 * 4 + 3] * inv)};
                    }
            } else {
                float* part = paged_part<HDP, R>(a, 2 * walk.me() + (old_t0 > 0 ? 0 : 1))         /* a share's first item, its last */;
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4)
                        *reinterpret_cast<f32x4*>(part + ((wave * (HDP / 8) + dt * 4 + g4) * 64 + lane) * 4) = f32x4{st.o[dt][g4 * 4], st.o[dt][g4 * 4 + 1], st.o[dt][g4 * 4 + 2], st.o[dt][g4 * 4 + 3]};
                if (he == 0) *reinterpret_cast<f32x2*>(part + R * HDP + 2 * (wave * 32 + l31)) = f32x2{st.m, l};
            }
        }
        if (!more) return;
        // ---- the walk
        st.clear();
        bool bad = false;
        // waits until this wave's loads of step t have arrived; those of the D - 1 steps behind it may still be under way (they come in order, and behind the last step of the item the loads
        // read nothing, but count); then takes care of elements that must not meet a zero of P.  The barrier behind it publishes the step.
        auto arrived = [&](int t, char* buf) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * NL < 63 ? (D - 1) * NL : 63) : "memory");
            if (t * 64 + 64 > diag) {
#pragma unroll
                for (int i = 0; i < NL / 2; ++i) {
                    u32x4* p = reinterpret_cast<u32x4*>(buf + HALF + (i * F::PASS + wave * C::RPW) * C::P + lane * 16);
                    u32x4 v = *p;
                    if (paged_clean(v)) {
                        bad = true;
                        *p = v;
                    }
                }
            }
        };
        arrived(t0, smem);
        __syncthreads();
        int cur = 0;                                                                    // the step's buffer in the ring
        for (int t = t0; t < t1; ++t) {
            const char* kb = smem + cur * STAGE;
            char* kn = smem + (cur == 0 ? NS - 1 : cur - 1) * STAGE;                     // of step t - 1, which every wave has left: step t + D goes there
            cur = cur == NS - 1 ? 0 : cur + 1;
            const unsigned keys = groups[0];
#pragma unroll
            for (int d = 0; d + 1 < D; ++d) groups[d] = groups[d + 1];
            if ((t + D) % F::SPC == 0) { ids = ids2; ids2 = F::chunk(a, w, (t + D) / F::SPC + 1); }
            groups[D - 1] = fe.take(a, w, ids, t + D, t1);
            paged_step<HDP, 2>(kb, kb + HALF, kn, qf, st, a.sl2, (t << 6) + 64 > seen_min || keys != 15u, min(seen, w.len) - (t << 6), keys, [&](int i, int n, char* next) {
#pragma unroll
                for (int l = i * NL / n; l < (i + 1) * NL / n; ++l) dma(t + D, l, next);
            });
            if (t + 1 < t1) arrived(t + 1, smem + cur * STAGE);
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                        // nothing is under way when the next item fills the ring
            __syncthreads();
        }
        paged_no_weight<HDP>(a, w, t0 << 6, t1 << 6, st, seen);
        if ((int64_t)t1 * 64 > diag) {
            if (bad) dirty = 1;
            __syncthreads();
            if (dirty) {
                paged_add_bad<HDP>(a, w, max(max(diag, 0) & ~63, t0 << 6), min(t1 << 6, w.len), st, seen);
                __syncthreads();
                if (tid == 0) dirty = 0;                                                // (the next item sets it behind barriers of its own)
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// keys split over the waves: no barrier until the waves' parts are joined.  A block works on one part of an item (kv head, 32 rows of a slot); the parts are made equally long over the whole
// batch, whatever the lengths are: `target` of them for a head, plus one for each item.  Blocks are dispatched as others end, which levels what is left.  (Equal shares as in the tile kernel
// were tried: 138 against 131 us for 128 slots, 99 against 87 for one of 200000 tokens: the memory system is busy when the second block of a CU starts up, and the start is shorter.)
// ---------------------------------------------------------------------------------------------------------------------------------
// TARGET 448 | 512 | 768 | 1024 (28 / 4 heads of 128): 48 slots of 714 .. 5825 tokens 58 | 65 | 61 | 59 us, 16 of about 2200 22 | 22 | 25 | 26, one of 200000 91 | 89 | 94 | 98, one of 20000
// with 31 of 500 23 | 23 | 27 | 28: two blocks run on a CU, and rounding up adds about half a part for each item.
constexpr int TARGET = 448;
constexpr int STEP_SH = 7;                 // log2 of the keys of a step: 4 waves x 32.  The shortest part is one step: one slot of 1000 tokens 10.2 us, 11.7 with two

// What unit u of a head is: its tile, its keys [k0, k1) in steps, part of parts.  Every block finds it for itself: it sums the steps of the batch for the length of a part, then the slots'
// units.  ALONE, up to 64 slots: every wave for itself, a slot a lane, no barrier (0.5 us less); else a slot a thread, 256 at a time (700 slots of 200 .. 1999 tokens 323 us, 353 with every wave
// for itself; 200 of 50 .. 798 42 | 46).  (Longest parts first, by classes of length: no gain.)
struct PUnitLds {
    unsigned sum[4];
    int scan[4][2];
    int cu, n, len, s, parts, per, r, first;
};
template <int NW, bool ALONE>
__device__ __forceinline__ bool paged_unit(const PagedAttn& a, PUnitLds& m, int u, PagedTile& w, int& part, int& parts, int& per, int& first) {
    static_assert(NW == 4, "the LDS holds the sums of four waves");
    constexpr int SPAN = ALONE ? 64 : NW * 64;                                         // slots of a round
    const int tid = threadIdx.x, lane = tid & 63, wave = ALONE ? 0 : tid >> 6, me = ALONE ? lane : tid;
    int c0, n, len, tiles, steps;
    auto load = [&](int s0) {
        const int s = min(s0 + me, a.t.S - 1), c1 = a.t.cu_q[s + 1];
        c0 = a.t.cu_q[s];
        len = paged_len(a.t, s);
        n = c1 - c0;
        const bool there = s0 + me < a.t.S && c0 >= 0 && n > 0 && c1 <= a.N;
        tiles = there ? (n * a.G + 31) >> 5 : 0;
        steps = (int)(((unsigned)len + (1u << a.sh) - 1) >> a.sh);
    };
    unsigned all = 0;
    for (int s0 = 0; s0 < a.t.S; s0 += SPAN) {
        load(s0);
        all += (unsigned)tiles * (unsigned)steps;                                      // (below 2^31 over the batch: see `sh`)
    }
    all = lane_scan(all);
    if constexpr (ALONE) {
        all = __builtin_amdgcn_readlane(all, 63);
    } else {
        if (lane == 63) m.sum[wave] = all;
        if (tid == 0) m.parts = 0;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) all += m.sum[i];
    }
    const int length = a.target ? max((int)((all + a.target - 1) / a.target), 1) : 1 << 30;
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    int before = 0, cut = 0, r;                                                        // units, units of cut items of the slots before
    for (int s0 = 0; s0 < a.t.S; s0 += SPAN) {
        if (!ALONE && a.t.S > SPAN) load(s0);
        const int most = max((steps + length - 1) / length, 1), p = max((steps + most - 1) / most, 1), k = max((steps + p - 1) / p, 1), mine = tiles * k, mc = k > 1 ? mine : 0;
        const int x = lane_scan(mine), xc = lane_scan(mc);
        if constexpr (ALONE) {
            const int c = __popcll(__ballot(x <= u));                                  // the first lane whose units go past u
            if (c == 64) return false;
            auto of = [&](int v) { return __builtin_amdgcn_readlane(v, c); };
            parts = of(k);
            per = of(p);
            w.s = c;
            w.q0 = of(c0);
            w.n = of(n);
            w.len = of(len);
            r = u - of(x - mine);
            first = of(xc - mc);
            if (r < 0) return false;
        } else {
            if (lane == 63) { m.scan[wave][0] = x; m.scan[wave][1] = xc; }
            __syncthreads();
            int b = before + x - mine, bc = cut + xc - mc;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                b += i < wave ? m.scan[i][0] : 0;
                bc += i < wave ? m.scan[i][1] : 0;
                before += m.scan[i][0];
                cut += m.scan[i][1];
            }
            if (u >= b && u < b + mine) {
                m.cu = c0;
                m.n = n;
                m.len = len;
                m.s = s0 + tid;
                m.parts = k;
                m.per = p;
                m.r = u - b;
                m.first = bc;
            }
            __syncthreads();
            if (u < before) break;
        }
    }
    if constexpr (!ALONE) {
        parts = uni(m.parts);
        if (parts == 0) return false;
        per = uni(m.per);
        w.s = uni(m.s);
        w.q0 = uni(m.cu);
        w.n = uni(m.n);
        w.len = uni(m.len);
        r = uni(m.r);
        first = uni(m.first);
    }
    w.rows = w.n * a.G;
    w.row0 = r / parts * 32;
    part = r % parts;
    first += r - part;
    return w.row0 < w.rows && (parts == 1 || (first >= 0 && (int64_t)(first + parts) * a.Hkv <= a.parts));      // (cu_q that does not ascend: nothing outside the arrays is touched)
}

template <int HDP, int NW, bool ALONE>
__global__ __launch_bounds__(NW * 64, HDP > 128 ? 1 : 2) void attn_paged_keys_k(PagedAttn a) {
    using C = PCfg<HDP>;
    constexpr int HALF = 32 * C::P, STAGE = 2 * HALF;
    static_assert(STAGE >= 32 * HDP * 4, "a wave's O fits its staging area");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float wm[NW][32], wl[NW][32];
    __shared__ PUnitLds unit;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, l31 = lane & 31, id = blockIdx.x;
    PagedTile w = {};
    int part = 0, parts = 0, per = 0, first = 0;
    w.g = id % a.Hkv;
    const bool work = paged_unit<NW, ALONE>(a, unit, id / a.Hkv, w, part, parts, per, first);
    if (!work) return;
    if (a.target && tid == 0 && part == 0) {                                           // the item's record is at its number
        PCut* c = paged_cut(a) + (int64_t)(paged_number<32>(a.G, w.s, w.q0) + (w.row0 >> 5)) * a.Hkv + w.g;
        c->first = first * a.Hkv + w.g;
        c->parts = parts;
        c->q0 = w.q0;
        c->row0 = w.row0;
        c->rows = w.rows;
        c->g = w.g;
    }
    const int kmax = min(paged_seen(a, w.len, w.n, (min(w.row0 + 32, w.rows) - 1) / a.G), w.len), k0 = part * per << a.sh;
    const int t0 = k0 >> 5, t1 = min((kmax + 31) >> 5, part + 1 == parts ? 0x7fffffff : (k0 + (per << a.sh)) >> 5);       // 32-key steps
    char* kb = smem + wave * STAGE;
    char* vb = kb + HALF;
    const int srow = lane / C::CPR, sch = lane % C::CPR;
    const unsigned lane_off = paged_lane_offset(a, srow, sch);
    const int diag = a.causal && w.n > 1 ? w.len - w.n : 0x7fffffff;
    using F = PFetch<HDP, 2, 1>;
    F fe;
    u32x4 kr[F::RPT], vr[F::RPT];
    unsigned next = 0;
    int chunk = -1, ids = 0;
    auto fetch = [&](int t) {
        if (t / F::SPC != chunk) { chunk = t / F::SPC; ids = F::chunk(a, w, chunk); }
        next = fe.take(a, w, ids, t, t1);
#pragma unroll
        for (int i = 0; i < F::RPT; ++i) {
            int nk, nv;
            bf16 *k = fe.rows(a, w, t, i, 0, nk), *v = fe.rows(a, w, t, F::RPT + i, 0, nv);
            kr[i] = __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc(k, 0, nk, 0x20000), lane_off, 0, 0);
            vr[i] = __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc(v, 0, nv, 0x20000), lane_off, 0, 0);
        }
    };
    if (t0 + wave < t1) fetch(t0 + wave);
    PState<HDP> st;
    st.clear();
    bf16x8 qf[C::KS];
    const int seen = paged_load_q<HDP>(a, w, w.row0, qf);
    const int seen_min = min(paged_seen(a, w.len, w.n, w.row0 / a.G), w.len);
    bool dirty = false;
    for (int t = t0 + wave; t < t1; t += NW) {
        if (t * 32 + 32 > diag) {
            bool b = false;
#pragma unroll
            for (int i = 0; i < F::RPT; ++i) b |= paged_clean(vr[i]);
            dirty |= __any(b);
        }
#pragma unroll
        for (int i = 0; i < F::RPT; ++i) {
            const int r = i * C::RPW + srow, at = r * C::P + 16 * (sch ^ C::f(r));
            *reinterpret_cast<u32x4*>(kb + at) = kr[i];
            *reinterpret_cast<u32x4*>(vb + at) = vr[i];
        }
        const unsigned groups = next;
        if (t + NW < t1) fetch(t + NW);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");                          // the staged rows are read by other lanes of this wave
        __builtin_amdgcn_wave_barrier();
        paged_step<HDP, 1>(kb, vb, nullptr, qf, st, a.sl2, (t << 5) + 32 > seen_min || groups != 3u, min(seen, w.len) - (t << 5), groups, [](int, int, char*) {});
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    if (dirty)
        for (int t = t0 + wave; t < t1; t += NW) paged_add_bad<HDP>(a, w, max(max(diag, 0) & ~31, t << 5), min((t + 1) << 5, w.len), st, seen);
    paged_no_weight<HDP>(a, w, t0 << 5, t1 << 5, st, seen);
    // ---- join the waves: (m, l) and O [row][HDP] of every wave through LDS, then every thread sums quads of the rows that exist
    const float l = st.l + __shfl_xor(st.l, 32, 64);
    if (h == 0) { wm[wave][l31] = st.m; wl[wave][l31] = l; }
    float* ob = reinterpret_cast<float*>(kb);
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
            *reinterpret_cast<f32x4*>(ob + l31 * HDP + (((dt * 8 + g4 * 2 + h) ^ (l31 & 7)) << 2)) = f32x4{st.o[dt][g4 * 4], st.o[dt][g4 * 4 + 1], st.o[dt][g4 * 4 + 2], st.o[dt][g4 * 4 + 3]};
    __syncthreads();
    const int rows = min(w.rows - w.row0, 32), cols = a.hd >> 2;
    for (int i = tid; i < rows * cols; i += NW * 64) {
        const int r = i / cols, quad = i - r * cols;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NW; ++k) m = fmaxf(m, wm[k][r]);
        float sum = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const float f = wm[k][r] == -INFINITY ? (wl[k][r] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(wm[k][r] - m);      // (nothing but NaN has no maximum: the NaN stays)
            sum += f * wl[k][r];
            o += f * *reinterpret_cast<const f32x4*>(smem + k * STAGE + (r * HDP + ((quad ^ (r & 7)) << 2)) * 4);
        }
        if (parts == 1) {
            const int tok = (w.row0 + r) / a.G, hq = w.g * a.G + (w.row0 + r - tok * a.G);
            const float inv = sum > 0.f ? 1.f / sum : sum;
            *reinterpret_cast<bf16x4*>(a.o + (int64_t)(w.q0 + tok) * a.ldo + hq * a.hd + quad * 4) = bf16x4{(bf16)(o[0] * inv), (bf16)(o[1] * inv), (bf16)(o[2] * inv), (bf16)(o[3] * inv)};
        } else {
            float* dst = paged_part<HDP, 32>(a, (first + part) * a.Hkv + w.g);
            *reinterpret_cast<f32x4*>(dst + part_at<HDP>(r, quad)) = o;
            if (quad == 0) *reinterpret_cast<f32x2*>(dst + 32 * HDP + 2 * r) = f32x2{m, sum};
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Does tile number t of 32 rows exist, that is, was its record written?  (a slot a lane, above 64 slots a slot a thread; the answer of one counts)
__device__ __forceinline__ bool paged_tile_exists(const PagedAttn& a, int t) {
    const bool alone = a.t.S <= 64;
    bool is = false;
    for (int s = alone ? threadIdx.x & 63 : threadIdx.x; s < a.t.S; s += 256) {
        const int c0 = a.t.cu_q[s], c1 = a.t.cu_q[s + 1], row0 = (t - paged_number<32>(a.G, s, c0)) * 32;
        is |= c0 >= 0 && c1 > c0 && c1 <= a.N && row0 >= 0 && row0 < (c1 - c0) * a.G;
    }
    return alone ? __any(is) : __syncthreads_or(is);
}

// The join of cut items.  blockIdx.x: the item's record.  A thread adds one quad of dims of one row over the parts, in their order, with weights 2^(m_p - m); eight lanes
// read 128 bytes of a part as the lanes of the tile kernel left them.  PG = 4 (few rows, many parts: the keys kernel): each wave takes a quarter of the parts, they meet in LDS.
// ---------------------------------------------------------------------------------------------------------------------------------
template <int HDP, int R, int PG>
__global__ __launch_bounds__(256) void attn_paged_join_k(PagedAttn a) {
    constexpr int T = 256 / PG, U = PG > 1 ? 8 : 4;                                    // threads over (row, quad); parts in flight
    __shared__ float red[PG > 1 ? PG - 1 : 1][6][64];
    const PCut c = paged_cut(a)[blockIdx.x];
    if (PG > 1 ? !paged_tile_exists(a, blockIdx.x / a.Hkv) : (int)blockIdx.x >= paged_cut(a)->used) return;
    const int step = PG > 1 ? a.Hkv : 1;                                                // keys kernel: the parts of a head; tile kernel: the workers, two parts each
    if (c.parts < 2 || c.first < 0 || c.first + (int64_t)(c.parts - 1) * step >= (PG > 1 ? a.parts : a.cuts)) return;
    if (c.q0 < 0 || c.row0 < 0 || c.rows > (int64_t)(a.N - c.q0) * a.G || (unsigned)c.g >= (unsigned)a.Hkv) return;   // (a record that nobody wrote: cu_q that does not ascend)
    const int pg = PG > 1 ? threadIdx.x / T : 0, per = (c.parts + PG - 1) / PG, pb = min(pg * per, c.parts), pe = min(pb + per, c.parts);
    for (int i0 = blockIdx.y * T; i0 < R * (HDP / 4); i0 += gridDim.y * T) {
        const int i = i0 + threadIdx.x % T, quad = (i >> 3) % (HDP / 4), row = (i >> 3) / (HDP / 4) * 8 + (i & 7), r = c.row0 + row;
        if (c.row0 + (i0 >> 3) / (HDP / 4) * 8 >= c.rows) return;                      // (the same for all threads)
        const bool mine = r < c.rows && quad * 4 < a.hd;
        const int at = part_at<HDP>(row, quad), at_ml = R * HDP + 2 * row;
        // one pass with a running maximum, U parts in flight
        float m = -INFINITY, sum = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        auto add = [&](float mp, float lp, const f32x4& op, float mn) {
            const float f = mp == -INFINITY ? (lp == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mp - mn);               // (a part of nothing but NaN has no maximum: its NaN stays)
            sum += f * lp;
            o += f * op;
        };
        auto raise = [&](float mn) {
            const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            sum *= f;
            o *= f;
            m = mn;
        };
        for (int p0 = mine ? pb : pe; p0 < pe; p0 += U) {
            f32x4 v[U];
            f32x2 ml[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int p = p0 + k;
                v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
                ml[k] = f32x2{-INFINITY, 0.f};
                if (p < pe) {
                    const float* part = paged_part<HDP, R>(a, PG > 1 ? c.first + p * step : 2 * (c.first + p) + (p == 0 ? 1 : 0));
                    v[k] = *reinterpret_cast<const f32x4*>(part + at);
                    ml[k] = *reinterpret_cast<const f32x2*>(part + at_ml);
                }
            }
            float mn = m;
#pragma unroll
            for (int k = 0; k < U; ++k) mn = fmaxf(mn, ml[k][0]);
            raise(mn);
#pragma unroll
            for (int k = 0; k < U; ++k) add(ml[k][0], ml[k][1], v[k], m);
        }
        if constexpr (PG > 1) {
            const int lane = threadIdx.x % T;
            __syncthreads();
            if (pg > 0) {
                red[pg - 1][0][lane] = m;
                red[pg - 1][1][lane] = sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) red[pg - 1][2 + e][lane] = o[e];
            }
            __syncthreads();
            if (pg > 0) continue;
#pragma unroll
            for (int k = 0; k < PG - 1; ++k) {
                const float mk = red[k][0][lane];
                raise(fmaxf(m, mk));
                add(mk, red[k][1][lane], f32x4{red[k][2][lane], red[k][3][lane], red[k][4][lane], red[k][5][lane]}, m);
            }
        }
        if (!mine) continue;
        const float inv = sum > 0.f ? 1.f / sum : sum;
        const int tok = r / a.G, hq = c.g * a.G + (r - tok * a.G);
        *reinterpret_cast<bf16x4*>(a.o + (int64_t)(c.q0 + tok) * a.ldo + hq * a.hd + quad * 4) = bf16x4{(bf16)(o[0] * inv), (bf16)(o[1] * inv), (bf16)(o[2] * inv), (bf16)(o[3] * inv)};
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
struct Plan {
    bool keys;              // keys split over the waves (else rows)
    int rows, tiles;        // of a tile; upper bound of their number
    int blocks;             // of the kernel
    int target, sh, cuts, parts;               // as in PagedAttn
    int64_t ws;             // bytes
};

// N, S: packed rows and slots; the lengths are on the device, the choice is made from the sizes alone: N / S rows a slot, as if all of them were as busy (the figures below are of such batches).  A
// batch of one long chunk in a table of idle slots is right, but may run through tiles of 32 rows that each fetch the chunk's whole cache.
Plan make_plan(int N, int S, int Hq, int Hkv, int hd, int max_keys) {
    const int G = Hq / Hkv, hdp = hd > 128 ? 256 : (hd + 31) / 32 * 32, used = S < N ? S : N;
    const int64_t rows = (int64_t)N * G;
    Plan p = {};
    p.keys = rows <= 32 * (int64_t)S;
    // Tiles of 256 rows (eight waves, one block a CU, a ring of four steps) fetch a key once for 256 rows, those of 128 (two to four blocks a CU, a ring of two) waste fewer rows and
    // steps on short slots and sequences.  28 / 4 heads of 128, 128 | 256: 2399 tokens over 20011 757 | 679 us, 8192 causal 675 | 606, 8 x 512 over 4096 289 | 261, 16 x 150 over 2048
    // 117 | 120, 4 x 100 over 2048 38 | 39, 8 x 600 causal 69 | 76, 300 causal 22 | 27; 14 / 2 heads of 64: 8192 tokens 412 | 443, 4 x 300 22 | 33.  Above 128 the registers of 256 rows do
    // not fit.
    p.rows = p.keys ? 32 : (hd > 64 && hd <= 128 && rows >= 2048 * (int64_t)used && max_keys >= 2048 ? 256 : 128);
    p.tiles = (int)(rows / p.rows) + S;
    if (p.keys) {
        p.target = max_keys > 4 << STEP_SH ? (TARGET + Hkv - 1) / Hkv : 0;                // (333 tokens in one block 10.3 us, in three and joined 10.2)
        p.blocks = (p.target + p.tiles) * Hkv;
        for (p.sh = STEP_SH; (int64_t)p.tiles * ((max_keys >> p.sh) + 1) > 0x7fffffff;) ++p.sh;
        p.cuts = p.target ? p.tiles * Hkv : 0;
        p.parts = 2 * p.target * Hkv;          // an item that is cut is longer than a part: its parts are at most twice its length in parts
    } else {
        // what fits the CUs at once: four blocks of four waves up to head_dim 32 (16 heads, 8192 causal tokens: 195 us, 210 with three), three up to 64, two up to 128, one above; one block of
        // eight
        const int slots = hd > 128 || p.rows == 256 ? 256 : (hd <= 32 ? 1024 : hd <= 64 ? 768 : 512);
        const int64_t steps = (rows / p.rows + used) * Hkv * (((int64_t)max_keys + 63) / 64 + ITEM_COST);
        p.blocks = steps / MIN_SHARE >= slots ? slots : (int)((steps / MIN_SHARE + 8) / 8 * 8);
        p.cuts = p.blocks;
        p.parts = 2 * p.blocks;
    }
    p.ws = (int64_t)p.cuts * (int64_t)sizeof(PCut) + (int64_t)p.parts * 4 * p.rows * (hdp + 2);
    return p;
}

template <int HDP, int NW, int NS>
void launch_tile(const PagedAttn& a, int blocks, hipStream_t st) {
    constexpr int smem = NS * 128 * PCfg<HDP>::P;
    UFV_ONCE_PER_DEVICE((void)hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_paged_tile_k<HDP, NW, NS>), hipFuncAttributeMaxDynamicSharedMemorySize, smem););
    hipLaunchKernelGGL((attn_paged_tile_k<HDP, NW, NS>), dim3(blocks), dim3(NW * 64), smem, st, a);
    hipLaunchKernelGGL((attn_paged_join_k<HDP, 32 * NW, 1>), dim3(blocks, 32 * NW * (HDP / 4) / 256), dim3(256), 0, st, a);
}

template <int HDP, bool ALONE>
void launch_keys(const PagedAttn& a, int blocks, hipStream_t st) {
    constexpr int NW = 4, smem = NW * 64 * PCfg<HDP>::P;
    UFV_ONCE_PER_DEVICE((void)hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_paged_keys_k<HDP, NW, ALONE>), hipFuncAttributeMaxDynamicSharedMemorySize, smem););
    hipLaunchKernelGGL((attn_paged_keys_k<HDP, NW, ALONE>), dim3(blocks), dim3(NW * 64), smem, st, a);
}

template <int HDP>
int launch(const PagedAttn& a, const Plan& p, hipStream_t st) {
    if (p.keys) {
        if (a.t.S <= 64) launch_keys<HDP, true>(a, p.blocks, st);
        else launch_keys<HDP, false>(a, p.blocks, st);
        if (p.target) hipLaunchKernelGGL((attn_paged_join_k<HDP, 32, 4>), dim3(a.tiles * a.Hkv, HDP / 32), dim3(256), 0, st, a);
    } else if (p.rows == 256) {
        if constexpr (HDP > 64 && HDP <= 128) launch_tile<HDP, 8, 4>(a, p.blocks, st);
    } else {
        launch_tile<HDP, 4, 2>(a, p.blocks, st);
    }
    UFV_CHECK_LAUNCH();
    return UFV_OK;
}

}  // namespace

extern "C" int64_t ufv_attention_paged_ws_bytes(int N, int S, int Hq, int Hkv, int hd, int max_keys) {
    if (N <= 0 || S <= 0 || Hkv <= 0 || Hq < Hkv || hd <= 0) return 0;
    return make_plan(N, S, Hq, Hkv, hd, max_keys).ws;
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
    UFV_REQUIRE(ldkv >= 2 * (int64_t)Hkv * hd && ldkv < 1 << 24 && (N == 1 || (ldq >= (int64_t)Hq * hd && ldo >= (int64_t)Hq * hd)), "ufv_attention_paged: a row pitch is out of range");
    // (token, head) rows and those of a last tile's width behind them, columns of a row: 31 bits
    UFV_REQUIRE((int64_t)N * Hq <= 0x7fffffff - 65536 && (int64_t)Hq * hd < 0x7fffffff && S <= 65536, "ufv_attention_paged: too many rows, columns or slots (N=%d, %d heads of %d, S=%d)", N, Hq, hd, S);
    const Plan p = make_plan(N, S, Hq, Hkv, hd, max_pages << paged_log2(page));
    UFV_REQUIRE(((int64_t)p.tiles + 2 * p.target) * Hkv < 0x7fffffff && Hkv < 65536, "ufv_attention_paged: too many row tiles (N=%d S=%d)", N, S);
    UFV_REQUIRE(p.ws == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= p.ws), "ufv_attention_paged: a 16-byte aligned workspace of %lld bytes is needed (%lld given)", (long long)p.ws,
                (long long)ws_bytes);
    PagedAttn a;
    a.q = (const bf16*)q; a.pages = (const bf16*)pages; a.o = (bf16*)o;
    a.ldq = ldq; a.ldo = ldo; a.ldkv = ldkv;
    a.t = PagedTable{block_table, ld_table, max_pages, cu_q, kv_len, S, n_pages, paged_log2(page)};
    a.N = N; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.hd = hd; a.causal = causal != 0;
    a.sl2 = scale * 1.4426950408889634f;
    a.tiles = p.tiles; a.target = p.target; a.sh = p.sh; a.cuts = p.cuts; a.parts = p.parts; a.ws = (float*)ws;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (hd <= 32) return launch<32>(a, p, st);
    if (hd <= 64) return launch<64>(a, p, st);
    if (hd <= 96) return launch<96>(a, p, st);
    if (hd <= 128) return launch<128>(a, p, st);
    return launch<256>(a, p, st);
}
