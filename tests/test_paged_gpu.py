"""GPU: the paged-cache operators against their 64-bit oracle (tests/paged_ref.py).  Floating-point results are compared element by element with the bound that the oracle
derives for each element (half steps of the types that a value is rounded to); integers and copied rows have to be equal."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from paged_ref import Batch, PageModel, attend, cdiv, rotate, EPS32  # noqa: E402
from ufvideo_amd import ops, _lib  # noqa: E402

DEV = "cuda"
BF = torch.bfloat16


def within(got, want, slack, what=""):
    d = (got.double() - want).abs()
    bad = ~(d <= slack)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} elements off, worst {float(d.nan_to_num(1e9).max()):.3e}, at {bad.nonzero()[0].tolist()}"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rnd(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV)


# ---- rotary positions with several axes ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("N,hd,sections,inter,pos0", [(1, 128, (16, 24, 24), False, 0), (7, 128, (24, 20, 20), True, 999_983), (130, 64, (8, 12, 12), False, 40_000), (33, 10, (1, 2, 2), False, 5),
                                                      (5, 2, (1,), False, 77), (65, 256, (32, 32, 32, 32), True, -123_456), (257, 96, (48,), False, 2_000_000)])
def test_rope_axes_table(N, hd, sections, inter, pos0):
    A = len(sections)
    g = torch.Generator().manual_seed(N + hd)
    pos = torch.randint(0, 5000, (A, N), generator=g) + pos0
    wide = torch.zeros(A, N + 3, dtype=torch.int64, device=DEV)
    wide[:, :N] = pos.to(DEV)                                       # a row pitch of its own
    inv = (1.0 / (1e6 ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd)))
    amap = ops.rope_axis_map(sections, inter)
    tab = ops.rope_axes_table(inv.to(DEV), wide[:, :N], amap).cpu()
    ang = pos[torch.tensor(amap)].t().double() * inv.double()
    # the reduced angle in units of pi is rounded once (<= 1), the functions to 2 half steps
    assert (tab.double() - torch.cat([ang.cos(), ang.sin()], 1)).abs().max() <= (math.pi + 2) * EPS32


def test_rope_axes_table_equal_axes_agree_with_the_one_axis_table():
    hd, N = 128, 300
    inv = (1.0 / (1e4 ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd))).to(DEV)
    pos = (torch.arange(N, device=DEV) + 11).expand(3, N).contiguous()
    a, b = ops.rope_axes_table(inv, pos, ops.rope_axis_map((16, 24, 24))), ops.rope_table(inv, 11, N, hd)
    # rope_table rounds the angle (<= 311) to 32 bits
    assert (a - b).abs().max() <= 311 * EPS32 + 8 * EPS32


@pytest.mark.parametrize("N,heads,hd,col0,pad,inplace", [(1, 1, 2, 0, 0, True), (3, 4, 128, 0, 0, False), (65, 32, 128, 0, 512, True), (17, 3, 64, 64, 8, False), (9, 5, 10, 3, 1, True),
                                                         (9, 5, 10, 3, 1, False), (129, 2, 96, 8, 0, True), (31, 1, 256, 0, 3, True), (2399, 32, 128, 0, 512, False)])
@pytest.mark.parametrize("backward", [False, True])
def test_rope_rows_table(N, heads, hd, col0, pad, inplace, backward):
    x = rnd(N, col0 + heads * hd + pad, seed=N).to(BF)
    tab = rnd(N, hd, seed=2)
    keep = x.clone()
    want, slack = rotate(x[:, col0:col0 + heads * hd].reshape(N, heads, hd), tab, backward)
    out = None if inplace else torch.full((N, heads * hd + 5), 7.0, device=DEV, dtype=BF)
    y = ops.rope_rows_table(x, tab, col0, heads, hd, out=out, backward=backward)
    got = y[:, col0:col0 + heads * hd] if inplace else y[:, :heads * hd]
    within(got.reshape(N, heads, hd), want, slack)
    if inplace:
        assert y is x and torch.equal(x[:, :col0], keep[:, :col0]) and torch.equal(x[:, col0 + heads * hd:], keep[:, col0 + heads * hd:])
    else:
        assert torch.equal(x, keep) and (out[:, heads * hd:] == 7.0).all()


def test_rope_rows_table_gradient_against_differences():
    """d <w, R x> / d x_i by differences of the forward kernel (steps of 1, exact in bf16) is what the backward kernel gives for w"""
    N, hd = 4, 16
    x = torch.randint(-3, 4, (N, hd), generator=torch.Generator().manual_seed(1)).to(DEV, BF)
    ang = rnd(N, hd // 2, seed=3) * 2
    tab = torch.cat([ang.cos(), ang.sin()], 1).contiguous()
    w = torch.randint(-2, 3, (N, hd), generator=torch.Generator().manual_seed(2)).to(DEV, BF)
    out = lambda v: ops.rope_rows_table(v, tab, 0, 1, hd, out=torch.empty_like(v)).double()
    base = out(x)
    grad = ops.rope_rows_table(w, tab, 0, 1, hd, out=torch.empty_like(w), backward=True).double()
    for i in range(hd):
        e = x.clone()
        e[:, i] += 1
        d = ((out(e) - base) * w.double()).sum(1)
        # two changed outputs, each the difference of two bf16 values below 8 in magnitude (half steps of 2^-6), weighted by |w| <= 2; grad itself is below 8
        assert (d - grad[:, i]).abs().max() <= 2 * 2 * 2 * 2.0 ** -6 + 2.0 ** -6, i


# ---- append ----------------------------------------------------------------------------------------------------------------------
APPENDS = [dict(q=[1], kv=[1], Hq=4, Hkv=2, hd=64, page=16), dict(q=[3, 0, 17, 1], kv=[20, 5, 17, 64], Hq=28, Hkv=4, hd=128, page=64), dict(q=[2, 5], kv=[1, 3], Hq=2, Hkv=1, hd=32, page=16),
           dict(q=[1] * 70, kv=[(i * 37) % 90 + 1 for i in range(70)], Hq=4, Hkv=4, hd=16, page=32), dict(q=[200, 0, 0, 331], kv=[200, 0, 7, 1000], Hq=16, Hkv=16, hd=96, page=128)]


@pytest.mark.parametrize("c", APPENDS, ids=lambda c: f"{len(c['q'])}slots_hd{c['hd']}_page{c['page']}")
@pytest.mark.parametrize("inplace", [False, True])
def test_rope_kv_paged(c, inplace):
    Hq, Hkv, hd = c["Hq"], c["Hkv"], c["hd"]
    holes = [(s, 0, b) for s, b in ((0, -1), (1, 2 ** 31 - 1)) if len(c["q"]) > 2 and c["kv"][s] > 0 and s == 1]
    b = Batch(c["q"], c["kv"], Hkv, hd, c["page"], seed=4, device=DEV, holes=holes, spare_rows=3, extra_width=1, pad=8)
    qkv = rnd(b.N, (Hq + 2 * Hkv) * hd + 8, seed=9).to(BF)
    tab = rnd(b.N, hd, seed=5)
    pages, keep = b.pages.clone(), qkv.clone()
    q_out = None if inplace else torch.full((b.N, Hq * hd + 8), 3.0, device=DEV, dtype=BF)
    q = ops.rope_kv_paged(qkv, tab, Hq, Hkv, hd, pages, b.table, b.cu_q, b.kv_len, q_out=q_out)
    n = b.cu[-1]
    heads = keep[:, :(Hq + Hkv) * hd].reshape(b.N, Hq + Hkv, hd)
    want, slack = rotate(heads, tab)
    within(q[:n, :Hq * hd].reshape(n, Hq, hd), want[:n, :Hq], slack[:n, :Hq], "q")
    touched = torch.zeros(b.P, b.page, dtype=torch.bool, device=DEV)
    for s in range(len(c["q"])):
        for r in range(b.cu[s], b.cu[s + 1]):
            pos = c["kv"][s] - c["q"][s] + r - b.cu[s]
            at = b.row(s, pos) if pos >= 0 else None
            if at is None:
                continue
            touched[at] = True
            within(pages[at][:Hkv * hd].reshape(Hkv, hd), want[r, Hq:], slack[r, Hq:], f"k of row {r}")
            assert torch.equal(pages[at][Hkv * hd:2 * Hkv * hd], keep[r, (Hq + Hkv) * hd:(Hq + 2 * Hkv) * hd])
            assert torch.equal(pages[at][2 * Hkv * hd:], b.pages[at][2 * Hkv * hd:])
    assert torch.equal(pages[~touched], b.pages[~touched])
    if inplace:
        assert torch.equal(qkv[:, Hq * hd:], keep[:, Hq * hd:]) and torch.equal(qkv[n:], keep[n:])
    else:
        assert torch.equal(qkv, keep) and (q_out[n:] == 3.0).all() and (q_out[:, Hq * hd:] == 3.0).all()


# ---- attention ------------------------------------------------------------------------------------------------------------------
HEADS = [(28, 4, 128), (14, 2, 64), (4, 4, 16), (8, 1, 96), (12, 2, 128), (3, 3, 40), (32, 8, 128), (2, 1, 8), (40, 1, 64), (5, 5, 256), (6, 2, 192)]
LENS = [([1], [1]), ([1], [63]), ([1], [64]), ([1], [65]), ([1], [1000]), ([1, 1, 1, 1], [17, 4097, 300, 1]), ([5], [5]), ([64], [64]), ([130], [131]), ([33, 1, 0, 70], [400, 129, 50, 70]),
        ([257, 31], [700, 31]), ([0, 0, 3], [9, 0, 3])]


def run_case(q_lens, kv_lens, Hq, Hkv, hd, page, causal=True, seed=0, holes=(), scale=None, kscale=1.0, pad=0, qpad=0):
    b = Batch(q_lens, kv_lens, Hkv, hd, page, seed=seed, device=DEV, holes=holes, spare_rows=2, extra_width=2, pad=pad, scale=kscale)
    q = rnd(b.N, Hq * hd + qpad, seed=seed + 1).to(BF)
    out = torch.full((b.N, Hq * hd + qpad), 5.0, device=DEV, dtype=BF)
    ops.attention_paged(q, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd, scale=scale, causal=causal, out=out)
    want, slack = attend(b, q, Hq, scale=scale, causal=causal, out=out)
    within(out[:, :Hq * hd], want, slack, f"q {q_lens} kv {kv_lens} heads {Hq}/{Hkv} hd {hd} page {page}")
    assert (out[b.cu[-1]:] == 5.0).all() and (out[:, Hq * hd:] == 5.0).all()
    return b, q, out


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
@pytest.mark.parametrize("lens", LENS, ids=lambda l: "q" + "_".join(map(str, l[0])) + "_kv" + "_".join(map(str, l[1])))
def test_attention_paged(Hq, Hkv, hd, lens):
    run_case(*lens, Hq, Hkv, hd, 64, seed=hd)


@pytest.mark.parametrize("page", [16, 32, 128, 256, 1024])
@pytest.mark.parametrize("Hq,Hkv,hd", [(28, 4, 128), (14, 2, 64), (4, 2, 32)])
def test_attention_paged_page_sizes(page, Hq, Hkv, hd):
    run_case([1, 40, 7], [page + 1, 3 * page + 5, page], Hq, Hkv, hd, page, seed=page) if page >= 40 else run_case([1, 9, 7], [page + 1, 3 * page + 5, page], Hq, Hkv, hd, page, seed=page)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q,kv", [([4, 40], [2, 13]), ([100], [60]), ([3, 2], [0, 0]), ([300], [1])])
def test_attention_paged_rows_that_see_nothing_are_zero(q, kv, causal):
    """more rows than cached tokens: the first rows have no position (causal) and an empty cache leaves every row empty"""
    for Hq, Hkv, hd in ((28, 4, 128), (4, 2, 64)):
        run_case(q, kv, Hq, Hkv, hd, 16, causal=causal)


def test_attention_paged_not_causal_and_scale():
    run_case([1, 70, 20], [100, 333, 20], 28, 4, 128, 32, causal=False)
    run_case([200], [900], 8, 2, 64, 64, causal=False, scale=0.03)
    run_case([9], [70], 8, 2, 128, 64, scale=0.5)


def test_attention_paged_strong_scores():
    """scores of hundreds: the running maximum moves often and one key takes nearly everything"""
    run_case([1, 64], [700, 777], 28, 4, 128, 64, kscale=12.0)
    run_case([150], [150], 14, 2, 64, 16, kscale=20.0)


def test_attention_paged_row_pitches():
    run_case([1, 50], [300, 310], 12, 2, 128, 64, pad=64, qpad=24)


@pytest.mark.parametrize("q,kv", [([1], [500]), ([90], [500]), ([400], [500])])
def test_attention_paged_skips_pages_outside_the_pool(q, kv):
    """-1, ids past the pool and the extreme ints name no page: their keys are absent, wherever they are; a slot with no page at all gives zeros"""
    run_case(q, kv, 28, 4, 128, 32, holes=[(0, 0, -1), (0, 3, 10 ** 6), (0, 4, 2 ** 31 - 1), (0, 9, -2 ** 31)])
    run_case(q, kv, 14, 2, 64, 16, holes=[(0, j, -1) for j in range(0, 32, 2)])
    run_case(q + q, kv + kv, 4, 2, 64, 128, holes=[(1, j, -1) for j in range(4)])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), -3.38e38])
@pytest.mark.parametrize("Hq,Hkv,hd", [(28, 4, 128), (4, 2, 64)])
def test_attention_paged_masked_places_may_hold_anything(bad, Hq, Hkv, hd):
    """rows of a page behind kv_len, free pages, and new tokens that a causal row does not see"""
    for q, kv in (([1], [70]), ([20], [90]), ([150, 3], [200, 17])):
        b = Batch(q, kv, Hkv, hd, 64, seed=3, device=DEV)
        used = torch.zeros(b.P, 64, dtype=torch.bool, device=DEV)
        for s in range(len(q)):
            for j in range(kv[s]):
                used[b.row(s, j)] = True
        b.pages[~used] = bad
        for s in range(len(q)):                      # the last new token of every slot with more than one: seen by its own row only
            if q[s] > 1:
                b.pages[b.row(s, kv[s] - 1)] = bad
        x = rnd(b.N, Hq * hd, seed=8).to(BF)
        out = ops.attention_paged(x, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd)
        rows = [r for s in range(len(q)) for r in range(b.cu[s], b.cu[s + 1] - (q[s] > 1))]
        assert torch.isfinite(out[rows]).all()
        want, slack = attend(b, x, Hq)
        within(out[rows], want[rows], slack[rows], f"{bad} q {q}")


def test_attention_paged_nan_in_a_seen_key_reaches_its_rows():
    b = Batch([3], [50], 2, 64, 16, device=DEV)
    b.pages[b.row(0, 20)] = float("nan")
    out = ops.attention_paged(rnd(3, 256).to(BF), b.pages, b.table, b.cu_q, b.kv_len, 4, 2, 64)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("q,kv", [([1], [9000]), ([1] * 5, [9000, 1, 64, 8191, 2500]), ([24], [9000]), ([300], [4000])])
def test_attention_paged_long(q, kv):
    run_case(q, kv, 28, 4, 128, 64, seed=2)


def test_attention_paged_many_slots():
    n = 150
    run_case([1 if i % 7 else 0 for i in range(n)], [(i * 53) % 400 + 1 for i in range(n)], 14, 2, 64, 16, seed=6)


def test_attention_paged_far_rows():
    """cache rows past 2^31 elements"""
    P, page, Hkv, hd = 16500, 64, 8, 128
    pages = torch.zeros(P, page, 2 * Hkv * hd, device=DEV, dtype=BF)        # 4.3 GB, 2.16e9 elements
    b = Batch([1, 3], [130, 64], Hkv, hd, page, device=DEV)
    far = [P - 1 - i for i in range(b.P)]
    for i, p in enumerate(far):
        pages[p] = b.pages[i]
    table = i32([[far[x] if x >= 0 else -1 for x in row] for row in b.table_list])
    qkv = rnd(4, (16 + 2 * Hkv) * hd).to(BF)
    tab = rnd(4, hd)
    near, q1 = b.pages.clone(), torch.empty(4, 16 * hd, device=DEV, dtype=BF)
    q2 = torch.empty_like(q1)
    ops.rope_kv_paged(qkv, tab, 16, Hkv, hd, near, b.table, b.cu_q, b.kv_len, q_out=q1)
    ops.rope_kv_paged(qkv, tab, 16, Hkv, hd, pages, table, b.cu_q, b.kv_len, q_out=q2)
    assert torch.equal(q1, q2) and all(torch.equal(pages[p], near[i]) for i, p in enumerate(far))
    a1 = ops.attention_paged(q1, near, b.table, b.cu_q, b.kv_len, 16, Hkv, hd)
    a2 = ops.attention_paged(q2, pages, table, b.cu_q, b.kv_len, 16, Hkv, hd)
    assert torch.equal(a1, a2) and a1.abs().max() > 0


def test_attention_paged_repeats_bit_for_bit():
    b = Batch([1, 1, 60], [5000, 800, 2000], 4, 128, 64, device=DEV)
    q = rnd(b.N, 28 * 128).to(BF)
    first = ops.attention_paged(q, b.pages, b.table, b.cu_q, b.kv_len, 28, 4, 128)
    for _ in range(5):
        assert torch.equal(first, ops.attention_paged(q, b.pages, b.table, b.cu_q, b.kv_len, 28, 4, 128))


def test_attention_paged_agrees_with_the_contiguous_cache():
    """a contiguous cache is a run of consecutive pages: the same prompt through ufv_attention"""
    Hq, Hkv, hd, S = 28, 4, 128, 512
    kv = rnd(S, 2 * Hkv * hd).to(BF)
    q = rnd(S, Hq * hd, seed=1).to(BF)
    want = ops.attention(q, kv, kv[:, Hkv * hd:], 1, Hq, Hkv, S, S, hd, (0, q.stride(0)), (0, kv.stride(0)), (0, kv.stride(0)), causal=True)
    got = ops.attention_paged(q, kv.view(S // 64, 64, -1), i32([list(range(S // 64))]), i32([0, S]), i32([S]), Hq, Hkv, hd)
    # two kernels that each round p and o to bf16 once: twice the distance of one to the exact result
    b = Batch([S], [S], Hkv, hd, 64, device=DEV)
    b.pages, b.table_list, b.P = kv.view(S // 64, 64, -1), [list(range(S // 64))], S // 64
    exact, slack = attend(b, q, Hq)
    within(got, exact, slack)
    within(got, want.double(), 2 * slack)


# ---- pages ------------------------------------------------------------------------------------------------------------------------
def books(m):
    return i32(m.table), i32(m.lens), i32(m.refs)


def same(m, table, lens, refs):
    assert table.tolist() == m.table and lens.tolist() == m.lens and refs.tolist() == m.refs


@pytest.mark.parametrize("S,W,P,page,seed", [(1, 1, 1, 16, 0), (3, 4, 7, 16, 1), (8, 12, 40, 64, 2), (33, 9, 150, 16, 3), (70, 40, 2000, 128, 4), (1100, 6, 5000, 16, 5), (5, 300, 1200, 32, 6)])
def test_page_management_against_the_model(S, W, P, page, seed):
    rng = random.Random(seed)
    m = PageModel(S, W, P, page)
    table, lens, refs = books(m)
    L, width = 2, 16
    pool = torch.randint(0, 1000, (L, P, page, width), generator=torch.Generator().manual_seed(seed)).to(DEV, BF)
    for step in range(40):
        k = rng.choice("eefexc") if step else "e"
        if k == "f":
            v = [rng.randint(-2, S) if rng.random() < 0.5 else -1 for _ in range(S)]
            m.fork(v)
            ops.kv_pages_fork(table, lens, refs, i32(v), page)
        elif k == "x":
            v = [int(rng.random() < 0.3) for _ in range(S)]
            m.free(v)
            ops.kv_pages_free(table, lens, refs, i32(v), page)
        elif k == "e":
            v = [rng.choice([0, 0, 1, 3, page, page + 1, rng.randint(0, W * page), -5, 2 ** 31 - 1]) for _ in range(S)]
            granted, cu, pairs = ops.kv_pages_extend(table, lens, refs, i32(v), page)
            g, c, p = m.extend(v)
            assert granted.tolist() == g and cu.tolist() == c and pairs.tolist() == p
            want = pool.clone()
            for src, dst, n in p:
                if src >= 0:
                    want[:, dst, :n] = want[:, src, :n]
            ops.kv_pages_copy(pool, pairs)
            assert torch.equal(pool, want)
        else:
            moves = m.compact()
            want = pool.clone()
            for src, dst in moves:
                want[:, dst] = pool[:, src]
            counts = ops.kv_pages_compact(pool, table, lens, refs)
            assert counts.tolist() == [sum(1 for r in m.refs if r > 0), len(moves)] and torch.equal(pool, want)
        same(m, table, lens, refs)
    m.check()


def test_pages_copy_rows_and_ids():
    L, P, page, width = 3, 9, 32, 1024 + 8
    pool = rnd(L, P, page, width).to(BF)
    want = pool.clone()
    pairs = [(0, 1, 32), (2, 3, 5), (4, 5, 0), (-1, 6, 9), (6, P, 9), (2 ** 31 - 1, 6, 1), (6, -2 ** 31, 1), (8, 8, 4), (0, 7, 99), (2, 4, -3)]
    for s, d, n in ((0, 1, 32), (2, 3, 5), (0, 7, 32)):
        want[:, d, :n] = pool[:, s, :n]
    ops.kv_pages_copy(pool, i32(pairs))
    assert torch.equal(pool, want)
    view = rnd(2 * L, P, page, width).to(BF)[::2]                     # layers at a pitch of two
    keep = view.clone()
    ops.kv_pages_copy(view, i32([(3, 4, 7)]))
    keep[:, 4, :7] = keep[:, 3, :7]
    assert torch.equal(view, keep)


def test_pages_survive_a_table_with_bad_ids():
    table, lens, refs = i32([[7, -9], [3, 1], [-1, -1]]), i32([40, 33, 0]), i32([0, 1, 0, 1])
    ops.kv_pages_fork(table, lens, refs, i32([-1, -1, 0]), 32)
    assert table.tolist() == [[7, -9], [3, 1], [7, -9]] and lens.tolist() == [40, 33, 40] and refs.tolist() == [0, 1, 0, 1]
    g, cu, pairs = ops.kv_pages_extend(table, lens, refs, i32([1, 1, 0]), 32)
    assert g.tolist() == [1, 1, 0] and pairs.tolist() == [[-1, -1, 0]] * 3 and refs.tolist() == [0, 1, 0, 1]
    pool = rnd(1, 4, 32, 8).to(BF)
    assert ops.kv_pages_compact(pool, table, lens, refs).tolist() == [2, 1]
    assert table.tolist() == [[7, -9], [0, 1], [7, -9]] and refs.tolist() == [1, 1, 0, 0]
    ops.kv_pages_free(table, lens, refs, i32([1, 1, 1]), 32)
    assert table.tolist() == [[-1, -1]] * 3 and refs.tolist() == [0] * 4 and lens.tolist() == [0] * 3


def test_paged_ops_refuse_wrong_tensors():
    b = Batch([2], [20], 2, 64, 16, device=DEV)
    q = rnd(2, 256).to(BF)
    ok = (q, b.pages, b.table, b.cu_q, b.kv_len, 4, 2, 64)
    ops.attention_paged(*ok)
    for i, t in ((0, q.float()), (0, q.t()), (0, q[:, :200]), (0, q.cpu()), (1, b.pages.float()), (1, b.pages[::2]), (1, b.pages[:, :, :192]), (1, b.pages[:, :12]), (2, b.table.long()),
                 (2, b.table.cpu()), (2, b.table.repeat(2, 1)), (3, b.cu_q[:1]), (3, b.cu_q.float()), (4, b.kv_len.long()), (5, 3), (7, 60)):
        with pytest.raises(_lib.UfvError):
            ops.attention_paged(*ok[:i], t, *ok[i + 1:])
    with pytest.raises(_lib.UfvError):
        ops.attention_paged(*ok, out=torch.empty(3, 256, device=DEV, dtype=BF))
    tab = rnd(2, 64)
    for args in ((q, tab[:1], 0, 4, 64), (q, tab.to(BF), 0, 4, 64), (q, tab, 1, 4, 64), (q, tab, -1, 1, 64), (q, tab, 0, 4, 63)):
        with pytest.raises(_lib.UfvError):
            ops.rope_rows_table(*args)
    pos, inv = torch.zeros(3, 5, dtype=torch.int64, device=DEV), rnd(32)
    for args in ((inv, pos.int(), [0] * 32), (inv, pos, [0] * 31), (inv, pos, [3] * 32), (inv, pos, [-1] * 32), (inv, pos.cpu(), [0] * 32), (inv, pos.repeat(2, 1), [0] * 32)):
        with pytest.raises(_lib.UfvError):
            ops.rope_axes_table(*args)
    for v in (b.kv_len.long(), b.kv_len.repeat(2)):
        with pytest.raises(_lib.UfvError):
            ops.kv_pages_free(b.table, b.kv_len, i32([0] * b.P), v, 16)
    with pytest.raises(_lib.UfvError):
        ops.kv_pages_compact(b.pages[None], b.table, b.kv_len, i32([0] * (b.P + 1)))
    with pytest.raises(_lib.UfvError):
        ops.kv_pages_copy(b.pages[None].transpose(1, 2), i32([(0, 1, 1)]))


def test_paged_calls_without_rows():
    b = Batch([0], [20], 2, 64, 16, device=DEV)
    empty = torch.empty(0, 256, device=DEV, dtype=BF)
    assert ops.attention_paged(empty, b.pages, b.table, b.cu_q, b.kv_len, 4, 2, 64).shape == (0, 256)
    assert ops.rope_axes_table(rnd(32), torch.zeros(2, 0, dtype=torch.int64, device=DEV), [0] * 32).shape == (0, 64)
    ops.rope_rows_table(empty, torch.empty(0, 64, device=DEV), 0, 4, 64)
    ops.kv_pages_copy(b.pages[None], torch.empty(0, 3, dtype=torch.int32, device=DEV))


# ---- together ---------------------------------------------------------------------------------------------------------------------
class Layer:
    """one layer's q / k / v of every token ever appended, as the oracle's contiguous history"""

    def __init__(self, S, Hkv, hd):
        self.k = [torch.zeros(0, Hkv, hd, dtype=torch.float64, device=DEV) for _ in range(S)]
        self.v = [torch.zeros(0, Hkv, hd, dtype=torch.float64, device=DEV) for _ in range(S)]


def test_one_prompt_many_questions():
    """a prompt is appended, forked, its children take questions as one packed chunk batch, decode together, some finish, the cache is compacted, decoding goes on:
    attention equals that over each conversation's own contiguous history at every step and in every layer"""
    L, S, Hq, Hkv, hd, page, P = 2, 6, 28, 4, 128, 16, 64
    W = 24
    table, lens, refs = torch.full((S, W), -1, dtype=torch.int32, device=DEV), i32([0] * S), i32([0] * P)
    pool = torch.full((L, P, page, 2 * Hkv * hd), float("nan"), device=DEV, dtype=BF)
    hist = [Layer(S, Hkv, hd) for _ in range(L)]
    inv = (1.0 / (1e6 ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd))).to(DEV)
    amap = ops.rope_axis_map((16, 24, 24))
    state = {"seed": 0, "pos": [0] * S}

    def step(n_new):
        granted, cu, pairs = ops.kv_pages_extend(table, lens, refs, i32(n_new), page)
        ops.kv_pages_copy(pool, pairs)
        assert granted.tolist() == n_new
        N = sum(n_new)
        pos = torch.cat([torch.arange(n) + state["pos"][s] for s, n in enumerate(n_new)])
        pos = torch.stack([pos, pos // 3, pos % 7]).to(DEV)
        tab = ops.rope_axes_table(inv, pos, amap)
        c = cu.tolist()
        for li in range(L):
            state["seed"] += 1
            qkv = rnd(N, (Hq + 2 * Hkv) * hd, seed=state["seed"]).to(BF)
            rot, _ = rotate(qkv[:, :(Hq + Hkv) * hd].reshape(N, Hq + Hkv, hd), tab)
            rot = rot.to(BF).double()
            q = ops.rope_kv_paged(qkv, tab, Hq, Hkv, hd, pool[li], table, cu, lens)
            o = ops.attention_paged(q, pool[li], table, cu, lens, Hq, Hkv, hd)
            v = qkv[:, (Hq + Hkv) * hd:].reshape(N, Hkv, hd).double()
            h = hist[li]
            for s in range(S):
                if not n_new[s]:
                    continue
                a, e = c[s], c[s + 1]
                h.k[s], h.v[s] = torch.cat([h.k[s], rot[a:e, Hq:]]), torch.cat([h.v[s], v[a:e]])
                n, kv = e - a, h.k[s].shape[0]
                seen = torch.arange(kv, device=DEV)[None] <= torch.arange(kv - n, kv, device=DEV)[:, None]
                K, V = (x.repeat_interleave(Hq // Hkv, 1).permute(1, 0, 2).contiguous() for x in (h.k[s], h.v[s]))
                sc = (rot[a:e, :Hq].permute(1, 0, 2) @ K.transpose(1, 2).contiguous() * hd ** -0.5).masked_fill(~seen, float("-inf"))
                p = torch.softmax(sc, -1)
                want, A = (p @ V).permute(1, 0, 2), (p @ V.abs()).permute(1, 0, 2)
                # q and k carry two bf16 steps of their own here (the kernel's fp32 rotation may round the other way): a score moves by up to 2 half steps of sum |q k| <= 2^-7 * |q||k| * scale
                es = 2.0 ** -7 * rot[a:e, :Hq].norm(dim=-1).amax() * h.k[s].norm(dim=-1).amax() * hd ** -0.5 * 2.0 ** -6      # few elements differ: 1 in 64 is far more than are seen
                within(o[a:e].reshape(n, Hq, hd), want, 2.0 ** -8 * want.abs() + A * (2.0 ** -8 + 2 * es + 1e-4), f"layer {li} slot {s}")
        for s in range(S):
            state["pos"][s] += n_new[s]

    step([150, 0, 0, 0, 0, 40])                                    # the prompts of two conversations, one batch
    parent = [-1, 0, 0, 0, 5, -1]
    ops.kv_pages_fork(table, lens, refs, i32(parent), page)
    for s, p in enumerate(parent):
        if p >= 0:
            state["pos"][s] = state["pos"][p]
            for h in hist:
                h.k[s], h.v[s] = h.k[p], h.v[p]
    assert refs[:10].tolist() == [4] * 10
    step([0, 9, 31, 16, 3, 0])                                     # the questions
    for _ in range(3):
        step([1, 1, 1, 1, 1, 1])
    ops.kv_pages_free(table, lens, refs, i32([0, 1, 0, 1, 0, 0]), page)
    for s in (1, 3):
        state["pos"][s] = 0
        for h in hist:
            h.k[s], h.v[s] = h.k[s][:0], h.v[s][:0]
    live, moved = ops.kv_pages_compact(pool, table, lens, refs).tolist()
    assert moved > 0 and (refs[:live] > 0).all() and not refs[live:].any()
    step([1, 0, 1, 0, 1, 1])
    step([0, 20, 1, 0, 2, 1])                                      # a freed slot starts anew


def decode_step(st):
    """reserve, copy on write, rotate + append, attend: one token of every slot, nothing of it decided on the host"""
    granted, cu, pairs = ops.kv_pages_extend(st["table"], st["lens"], st["refs"], st["one"], 16)
    ops.kv_pages_copy(st["pool"], pairs)
    tab = ops.rope_axes_table(st["inv"], st["pos"], st["amap"])
    q = ops.rope_kv_paged(st["qkv"], tab, 8, 2, 64, st["pool"][0], st["table"], cu, st["lens"], q_out=st["q"])
    ops.attention_paged(q, st["pool"][0], st["table"], cu, st["lens"], 8, 2, 64, out=st["o"])
    st["pos"].add_(1)


def fresh_state(kv=(700, 31, 47)):
    S = len(kv)
    st = dict(table=torch.full((S + 1, 60), -1, dtype=torch.int32, device=DEV), lens=i32([0] * (S + 1)), refs=i32([0] * 150), one=i32([1] * (S + 1)),
              pool=rnd(1, 150, 16, 256, seed=7).to(BF), inv=rnd(32, seed=1).abs(), pos=torch.arange(S + 1, device=DEV).repeat(3, 1), amap=ops.rope_axis_map((8, 12, 12)),
              qkv=rnd(S + 1, 768, seed=2).to(BF), q=torch.zeros(S + 1, 512, device=DEV, dtype=BF), o=torch.zeros(S + 1, 512, device=DEV, dtype=BF))
    ops.kv_pages_extend(st["table"], st["lens"], st["refs"], i32(list(kv) + [0]), 16)
    ops.kv_pages_fork(st["table"], st["lens"], st["refs"], i32([-1] * S + [1]), 16)           # the last slot shares slot 1's pages
    return st


def test_decode_steps_captured_into_graphs():
    """two graphs of a whole decode step, replayed in turn with eager work between: every replay equals the eager step on a second state"""
    a, b, c = fresh_state(), fresh_state((1, 300, 16)), fresh_state()
    d = fresh_state((1, 300, 16))
    for st in (a, b, c, d):
        decode_step(st)                                                                        # warm-up, eager on all four
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        decode_step(a)
    with torch.cuda.graph(gb):
        decode_step(b)
    for i in range(20):
        ga.replay()
        gb.replay()
        decode_step(c)
        decode_step(d)
        if i % 4 == 0:
            torch.cuda.synchronize()
        for x, y in ((a, c), (b, d)):
            for k in ("table", "lens", "refs", "pool", "q", "o"):
                assert torch.equal(x[k], y[k]), (i, k)
    assert a["lens"].tolist() == [721, 52, 68, 52]


def test_paged_ops_on_another_stream():
    a, b = fresh_state(), fresh_state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            decode_step(a)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        decode_step(b)
    assert torch.equal(a["o"], b["o"]) and torch.equal(a["pool"], b["pool"])


def test_two_calls_at_once():
    """the same cache attended to from two streams at the same time: workspaces are not shared"""
    b = Batch([1, 40, 1], [6000, 900, 3000], 4, 128, 64, device=DEV)
    q1, q2 = rnd(b.N, 28 * 128, seed=1).to(BF), rnd(b.N, 28 * 128, seed=2).to(BF)
    w1, w2 = (ops.attention_paged(q, b.pages, b.table, b.cu_q, b.kv_len, 28, 4, 128) for q in (q1, q2))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, q in ((s1, q1), (s2, q2)):
            with torch.cuda.stream(s):
                got.append(ops.attention_paged(q, b.pages, b.table, b.cu_q, b.kv_len, 28, 4, 128))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, (w1, w2)[i % 2])


@pytest.mark.parametrize("q,kv,Hq,Hkv,hd", [(190, 190, 16, 16, 8), (3, 61, 16, 16, 8), (70, 120, 8, 4, 64)])
def test_attention_paged_many_short_items(q, kv, Hq, Hkv, hd):
    """items of one to four steps, so many that the ends of the blocks' shares fall close behind, into and close before short items"""
    n = 300
    run_case([max(q - (i * 7) % 5, 1) for i in range(n)], [kv + (i * 11) % 70 for i in range(n)], Hq, Hkv, hd, 16, seed=q)


@pytest.mark.parametrize("q,kv,Hq,Hkv,hd", [(300, 2400, 8, 1, 96), (280, 2100, 16, 2, 104), (2100, 2100, 3, 3, 72), (300, 2111, 28, 4, 128), (700, 2050, 12, 4, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_paged_wide_tiles(q, kv, Hq, Hkv, hd, causal):
    """slots of 2048 rows and more over 2048 keys and more"""
    run_case([q], [kv], Hq, Hkv, hd, 64, causal=causal, seed=q)


@pytest.mark.parametrize("q", [1, 40])
def test_attention_paged_hundreds_of_slots(q):
    """more slots than fit the copy of their lengths on chip; every ninth has no new token"""
    n = 700
    run_case([0 if i % 9 == 4 else q for i in range(n)], [q + (i * 37) % 150 for i in range(n)], 4, 4, 16, 16, seed=q)


@pytest.mark.parametrize("q,kv,Hq,Hkv,hd,lo,hi", [(1, 9000, 28, 4, 128, 1000, 3000), (1, 9000, 4, 4, 64, 8000, 9000), (300, 4000, 28, 4, 128, 0, 2000), (100, 6000, 4, 2, 64, 2000, 5000)])
def test_attention_paged_stretch_of_nan_reaches_every_row(q, kv, Hq, Hkv, hd, lo, hi):
    """K rows of NaN, more of them than a block's keys: a part with no number in it leaves NaN, not nothing"""
    b = Batch([q, 1], [kv, 50], Hkv, hd, 64, device=DEV)
    for j in range(lo, hi):
        b.pages[b.row(0, j)] = float("nan")
    out = ops.attention_paged(rnd(q + 1, Hq * hd).to(BF), b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd)
    assert torch.isnan(out[:q]).all() and torch.isfinite(out[q:]).all()


def test_attention_paged_nan_in_a_new_key_stays_with_the_rows_that_see_it():
    for q, kv, at in ((300, 4000, 3900), (20, 3000, 2990)):
        b = Batch([q], [kv], 4, 128, 64, device=DEV)
        b.pages[b.row(0, at)] = float("nan")
        out = ops.attention_paged(rnd(q, 28 * 128).to(BF), b.pages, b.table, b.cu_q, b.kv_len, 28, 4, 128)
        first = at - (kv - q)
        assert torch.isfinite(out[:first]).all() and torch.isnan(out[first:]).all()


def test_attention_paged_new_workspace_contents_do_not_show():
    """the workspace is not cleared between calls: whatever it holds, results are the same bit for bit"""
    for q, kv, Hq, Hkv, hd in (([1, 1, 0, 1], [9000, 40, 7, 700], 28, 4, 128), ([300, 5], [4000, 900], 28, 4, 128), ([70, 64], [300, 1000], 14, 2, 64)):
        b = Batch(q, kv, Hkv, hd, 64, device=DEV)
        x, outs = rnd(b.N, Hq * hd).to(BF), []
        n = ops._attention_paged_ws(b.N, len(q), Hq, Hkv, hd, b.table.shape[1] * 64)
        for fill in (0, 1, 255, 127):
            w = torch.full((max(n, 16),), fill, device=DEV, dtype=torch.uint8)
            out = torch.zeros(b.N, Hq * hd, device=DEV, dtype=BF)
            _lib.call("ufv_attention_paged", x.data_ptr(), Hq * hd, out.data_ptr(), Hq * hd, b.N, Hq, Hkv, hd, b.pages.data_ptr(), b.P, 64, 2 * Hkv * hd, b.table.data_ptr(), b.table.shape[1],
                      b.table.shape[1], b.cu_q.data_ptr(), b.kv_len.data_ptr(), len(q), hd ** -0.5, 1, w.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            outs.append(out)
        assert all(torch.equal(outs[0], o) for o in outs) and outs[0].abs().max() > 0


@pytest.mark.parametrize("Hq,Hkv,hd", [(28, 4, 128), (4, 2, 64)])
def test_attention_paged_captured_with_changing_lengths(Hq, Hkv, hd):
    """one graph per number of rows, replayed while cu_q, kv_len and the table change on the device: every replay equals the eager call, rows behind cu_q[S] stay"""
    page, S, cap = 64, 3, 5000
    for N, steps in ((400, ([300, 5, 95], [10, 200, 190], [1, 1, 1], [0, 400, 0], [0, 0, 0], [133, 133, 134])), (3, ([1, 1, 1], [0, 3, 0], [0, 0, 0], [2, 0, 1]))):
        b = Batch([N, 0, 0], [cap] * 3, Hkv, hd, page, seed=N, device=DEV)
        table, cu_q, kv_len = b.table.clone(), b.cu_q.clone(), b.kv_len.clone()
        q, out = rnd(N, Hq * hd).to(BF), torch.zeros(N, Hq * hd, device=DEV, dtype=BF)
        run = lambda o: ops.attention_paged(q, b.pages, table, cu_q, kv_len, Hq, Hkv, hd, out=o)
        run(out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(out)
        for i, n in enumerate(steps * 2):
            cu_q.copy_(i32([0, n[0], n[0] + n[1], sum(n)]))
            kv_len.copy_(i32([(977 * (i + s) + n[s]) % (cap - N) + n[s] for s in range(S)]))
            table.copy_(b.table.roll(i, 0))
            out.fill_(7.0)
            eager = torch.full_like(out, 7.0)
            g.replay()
            run(eager)
            if i % 3 == 0:
                torch.cuda.synchronize()
            assert torch.equal(out, eager) and (out[sum(n):] == 7.0).all() and not (sum(n) and (out[:sum(n)] == 7.0).all()), (N, i)


def test_compaction_captured_into_a_graph():
    S, page, L, P, width = 5, 16, 2, 60, 64
    states = []
    for _ in range(2):
        states.append(dict(pool=rnd(L, P, page, width, seed=3).to(BF), table=torch.full((S, 12), -1, dtype=torch.int32, device=DEV), lens=i32([0] * S), refs=i32([0] * P),
                           grow=i32([33, 17, 60, 5, 40]), drop=i32([0, 1, 0, 0, 1])))

    def turn(st):
        granted, cu_q, pairs = ops.kv_pages_extend(st["table"], st["lens"], st["refs"], st["grow"], page)
        ops.kv_pages_copy(st["pool"], pairs)
        ops.kv_pages_free(st["table"], st["lens"], st["refs"], st["drop"], page)
        st["counts"] = ops.kv_pages_compact(st["pool"], st["table"], st["lens"], st["refs"])

    for st in states:
        turn(st)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        turn(states[0])
    captured = states[0]["counts"]
    for i in range(8):
        for st in states:
            st["drop"].copy_(i32([(i + s) % 3 == 0 for s in range(S)]))
        g.replay()
        turn(states[1])
        if i % 3 == 0:
            torch.cuda.synchronize()
        for k in ("table", "lens", "refs", "pool"):
            assert torch.equal(states[0][k], states[1][k]), (i, k)
        assert torch.equal(captured, states[1]["counts"])
        live = int(captured[0])
        assert (states[0]["refs"][:live] > 0).all() and not states[0]["refs"][live:].any()


def test_rope_axes_table_refuses_axes_that_do_not_exist():
    inv, pos = torch.ones(32, device=DEV), torch.zeros(3, 4, dtype=torch.int64, device=DEV)
    for bad in (32, [0] * 31, [0] * 33, [-1] + [0] * 31, [3] + [0] * 31, [300] + [0] * 31, ["x"] * 32, None):
        with pytest.raises(_lib.UfvError):
            ops.rope_axes_table(inv, pos, bad)


def test_operators_on_parts_of_larger_tables_and_pools():
    """rows and columns of a larger table, slots of longer vectors, layers and columns of larger tensors: what lies beside them stays"""
    S, W, page, Hkv, Hq, hd, L = 3, 9, 16, 2, 4, 64, 2
    P, width = 40, 2 * Hkv * hd
    big_table = torch.full((S + 3, W + 4), 99, dtype=torch.int32, device=DEV)
    big_len, big_refs = i32([77] * (S + 2)), i32([0] * P)
    big_pool = rnd(L + 2, P, page, width, seed=1).to(BF)
    table, lens, pool = big_table[1:S + 1, 2:W + 2], big_len[1:S + 1], big_pool[1:L + 1]
    table.fill_(-1)
    lens.zero_()
    alone = dict(table=table.clone(), lens=lens.clone(), refs=big_refs.clone(), pool=pool.clone())
    qkv = rnd(60, (Hq + 2 * Hkv) * hd + 8, seed=2).to(BF)
    tab = rnd(60, hd, seed=3)
    outs = []
    for st in (dict(table=table, lens=lens, refs=big_refs, pool=pool), alone):
        x = qkv.clone()
        got = []
        for turn, (grow, parent, drop) in enumerate((([20, 0, 31], [-1, 0, -1], [0, 0, 0]), ([5, 7, 1], [-1, -1, -1], [0, 0, 1]), ([30, 2, 9], [-1, -1, -1], [1, 0, 0]))):
            granted, cu_q, pairs = ops.kv_pages_extend(st["table"], st["lens"], st["refs"], i32(grow), page)
            ops.kv_pages_copy(st["pool"], pairs)
            n = sum(grow)
            rows = x[:n].clone()
            for l in range(L):
                q = ops.rope_kv_paged(rows.clone(), tab[:n], Hq, Hkv, hd, st["pool"][l], st["table"], cu_q, st["lens"])
                got.append(ops.attention_paged(q, st["pool"][l], st["table"], cu_q, st["lens"], Hq, Hkv, hd))
            ops.kv_pages_fork(st["table"], st["lens"], st["refs"], i32(parent), page)
            ops.kv_pages_free(st["table"], st["lens"], st["refs"], i32(drop), page)
            got.append(ops.kv_pages_compact(st["pool"], st["table"], st["lens"], st["refs"]))
        outs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert torch.equal(table, alone["table"]) and torch.equal(lens, alone["lens"]) and torch.equal(big_refs, alone["refs"]) and torch.equal(pool, alone["pool"])
    inside = torch.zeros_like(big_table, dtype=torch.bool)
    inside[1:S + 1, 2:W + 2] = True
    assert (big_table[~inside] == 99).all() and big_len[0] == 77 and big_len[S + 1] == 77
    fresh = rnd(L + 2, P, page, width, seed=1).to(BF)
    assert torch.equal(big_pool[0], fresh[0]) and torch.equal(big_pool[-1], fresh[-1])


def test_operators_without_rows():
    S, page, Hkv, Hq, hd = 2, 16, 1, 2, 32
    pages = rnd(4, page, 2 * Hkv * hd).to(BF)
    table, cu_q, kv_len = i32([[0, 1], [2, 3]]), i32([0, 0, 0]), i32([5, 0])
    keep = pages.clone()
    q = ops.rope_kv_paged(torch.empty(0, (Hq + 2 * Hkv) * hd, device=DEV, dtype=BF), torch.empty(0, hd, device=DEV), Hq, Hkv, hd, pages, table, cu_q, kv_len)
    assert q.shape == (0, Hq * hd) and ops.attention_paged(q, pages, table, cu_q, kv_len, Hq, Hkv, hd).shape == (0, Hq * hd)
    assert ops.rope_axes_table(torch.ones(16, device=DEV), torch.zeros(2, 0, dtype=torch.int64, device=DEV), [0] * 16).shape == (0, 32)
    x = torch.full((7, Hq * hd), 2.0, device=DEV, dtype=BF)                    # rows, but of no slot
    out = torch.full_like(x, 3.0)
    ops.attention_paged(x, pages, table, cu_q, kv_len, Hq, Hkv, hd, out=out)
    assert (out == 3.0).all() and torch.equal(pages, keep)
