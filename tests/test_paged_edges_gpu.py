"""GPU: what the paged-cache operators make of infinities and NaN that a row does see, and of views whose strides say nothing (an axis of one entry, one set of positions for all axes).
Finite results are compared with the 64-bit oracle's bound element by element, the others have to be the same kind of value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from paged_ref import Batch, attend  # noqa: E402
from ufvideo_amd import _lib, ops  # noqa: E402

DEV = "cuda"
BF = torch.bfloat16
INF, NAN = float("inf"), float("nan")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def same_kind(got, want, slack, what=""):
    """+inf, -inf and NaN in the same places, the rest within slack"""
    got = got.double()
    for name, f in (("nan", torch.isnan), ("+inf", torch.isposinf), ("-inf", torch.isneginf)):
        d = f(got) != f(want)
        assert not d.any(), f"{what}: {name} differs in {int(d.sum())} places, first {d.nonzero()[0].tolist()}: {got[d][0]} for {want[d][0]}"
    ok = torch.isfinite(want)
    bad = ok & ~((got - want).abs() <= slack)
    assert not bad.any(), f"{what}: {int(bad.sum())} elements off, at {bad.nonzero()[0].tolist()}"


# ---- V alone ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("Hq,Hkv,hd", [(4, 2, 128), (4, 2, 64), (2, 1, 32), (3, 1, 72), (2, 1, 192)])
@pytest.mark.parametrize("q,kv", [(1, 50), (3, 50), (20, 90), (5, 700), (40, 40), (150, 1517), (300, 300), (20, 13)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_paged_bad_elements_of_v_reach_the_rows_that_see_them(Hq, Hkv, hd, q, kv, causal):
    """one V row at a time holds +inf, -inf and NaN, K is finite: before the new tokens (in the step of the first of them and in earlier ones), at the first, among them, at the last"""
    b = Batch([q, 1], [kv, 40], Hkv, hd, 16, seed=hd, device=DEV)
    x = rnd(b.N, Hq * hd, seed=q).to(BF)
    clean, first, v0 = b.pages.clone(), max(kv - q, 0), (2 * Hkv - 1) * hd        # V of the last kv head
    for at in sorted({0, first // 64 * 64, first // 32 * 32, max(first - 1, 0), first, min(first + 1, kv - 1), (first + kv) // 2, kv - 1}):
        b.pages.copy_(clean)
        for d, bad in ((0, INF), (5, -INF), (hd - 1, NAN)):
            b.pages[b.row(0, at)][v0 + d] = bad
        if at > 0:                                                                # both signs in one column: NaN where a row sees both
            b.pages[b.row(0, at - 1)][v0 + 3], b.pages[b.row(0, at)][v0 + 3] = INF, -INF
        got = ops.attention_paged(x, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd, causal=causal)
        want, slack = attend(b, x, Hq, causal=causal)
        assert not torch.isfinite(want).all()
        same_kind(got, want, slack, f"V row {at} of {kv}, {q} new")


@pytest.mark.parametrize("q,kv,Hq,Hkv,hd", [(24, 9000, 28, 4, 128), (300, 4000, 7, 1, 128), (700, 2050, 3, 1, 128), (2100, 2100, 1, 1, 72)])
def test_attention_paged_bad_elements_of_v_in_cut_items(q, kv, Hq, Hkv, hd):
    """the same where several blocks work on the item, and in the middle of a whole prompt of several tiles"""
    b = Batch([q], [kv], Hkv, hd, 64, seed=1, device=DEV)
    x = rnd(q, Hq * hd, seed=2).to(BF)
    want0, slack0 = attend(b, x, Hq)
    first, v0 = kv - q, (2 * Hkv - 1) * hd
    for at in sorted({10, first // 64 * 64, max(first - 1, 0), first, first + 1, (first + kv) // 2, kv - 1}):
        kept = b.pages[b.row(0, at)].clone()
        for d, bad in ((1, INF), (6, -INF), (hd - 1, NAN)):
            b.pages[b.row(0, at)][v0 + d] = bad
        got = ops.attention_paged(x, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd)
        b.pages[b.row(0, at)] = kept
        want = want0.view(q, Hkv, Hq // Hkv, hd).clone()                          # every weight of a seen key is above 0: its column is the bad value
        for d, bad in ((1, INF), (6, -INF), (hd - 1, NAN)):
            want[max(at - first, 0):, -1, :, d] = bad
        same_kind(got, want.view(q, -1), slack0, f"V row {at} of {kv}, {q} new")


# ---- scores of -inf ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [8, 16, 40, 64, 72, 80, 104, 128, 192, 256])
@pytest.mark.parametrize("q,kv", [(1, 70), (3, 200), (150, 300), (2100, 2100)])
def test_attention_paged_a_key_of_weight_nothing_leaves_its_row_finite(hd, q, kv):
    """K elements of -inf: rows whose q has the sign that makes the score -inf go on without the key, the others become NaN -- at every head_dim, full register width or not"""
    Hq, Hkv, page = 2, 1, 64
    junk = torch.full((4, page, 2 * Hkv * hd), NAN, device=DEV, dtype=BF)            # what ran before leaves NaN in the chip's memories
    junk_rows = max(q * Hq // 2, 1)
    ops.attention_paged(torch.ones(junk_rows, Hq * hd, device=DEV, dtype=BF), junk, i32([[0, 1, 2, 3]]), i32([0, junk_rows]), i32([200]), Hq, Hkv, hd)
    b = Batch([q], [kv], Hkv, hd, page, seed=hd, device=DEV)
    x = rnd(q, Hq * hd, seed=3).to(BF)
    for j, d in ((1, 0), (kv // 2, 7), (kv - 1, hd - 1)):
        b.pages[b.row(0, j)][d] = -INF
    xh = x.view(q, Hq, hd)[:(q + 1) // 2]
    xh[:, :, [0, 7, hd - 1]] = xh[:, :, [0, 7, hd - 1]].abs() + 0.125
    got = ops.attention_paged(x, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd)
    want, slack = attend(b, x, Hq)
    alone = torch.isnan(want.view(q, Hq, hd)).all(-1, keepdim=True).expand(q, Hq, hd).reshape(q, -1)
    assert (q <= 2 or not alone.all()) and torch.equal(alone, torch.isnan(want))
    same_kind(got, want, slack, f"hd {hd}, {q} new of {kv}")


def defined(b, q, Hq, causal):
    """the definition, a row at a time in 64 bits: softmax over the scores of the keys that the row sees; zeros where there is none"""
    hd, G = b.hd, Hq // b.Hkv
    o = torch.zeros(q.shape[0], Hq, hd, dtype=torch.float64)
    pages, x = b.pages.cpu().double(), q.cpu().double().view(q.shape[0], Hq, hd)
    for s, (n, kv) in enumerate(zip(b.q_lens, b.kv_lens)):
        for r in range(n):
            keys = [b.row(s, j) for j in range(min(kv, kv - n + r + 1) if causal else kv)]
            keys = [k for k in keys if k is not None]
            if not keys:
                continue
            rows = pages[torch.tensor([k[0] for k in keys]), torch.tensor([k[1] for k in keys])]
            for h in range(Hq):
                g = h // G
                p = torch.softmax((rows[:, g * hd:(g + 1) * hd] * x[b.cu[s] + r, h]).sum(1) * hd ** -0.5, 0)
                o[b.cu[s] + r, h] = (p[:, None] * rows[:, (b.Hkv + g) * hd:(b.Hkv + g + 1) * hd]).sum(0)
    return o.view(q.shape[0], -1).to(q.device)


@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hkv,hd", [([1, 1], [70, 20], 4, 2, 64), ([1, 1], [9000, 700], 4, 2, 128), ([5, 3], [9, 2], 4, 2, 72), ([40, 1], [60, 33], 4, 2, 128),
                                                      ([40], [13], 4, 2, 64), ([70, 9], [2100, 9], 2, 1, 128), ([1] * 70, [30] * 70, 2, 2, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_paged_rows_of_nothing_but_scores_of_minus_infinity(q_lens, kv_lens, Hq, Hkv, hd, causal):
    """a row all of whose keys score -inf has no softmax (NaN); a row that sees no key is 0; one that sees a finite score besides is finite"""
    b = Batch(q_lens, kv_lens, Hkv, hd, 16, seed=hd, device=DEV, extra_width=1)
    x = rnd(b.N, Hq * hd, seed=4).to(BF)
    x.view(b.N, Hq, hd)[:, :, 0] = x.view(b.N, Hq, hd)[:, :, 0].abs() + 0.125
    for some in (False, True):
        kv0 = kv_lens[0]
        for j in range(kv0 - 1 if some else kv0):                                   # all keys of the first slot, then all but its last
            b.pages[b.row(0, j)][:Hkv * hd:hd] = -INF
        if some:
            b.pages[b.row(0, kv0 - 1)][:Hkv * hd:hd] = 0.5
        got = ops.attention_paged(x, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd, causal=causal)
        want = defined(b, x, Hq, causal)
        q0 = q_lens[0]
        hidden = max(q0 - kv0, 0) if causal else 0                                  # rows without a position
        assert torch.isnan(want[hidden:q0]).any() == (not some or (causal and q0 > hidden + 1))
        _, slack = attend(b, x, Hq, causal=causal)
        same_kind(got, want, slack, f"some={some}")


def test_attention_paged_slots_whose_pages_are_all_outside_the_pool_stay_zero():
    for q, kv in ((1, 70), (1, 9000), (200, 300), (200, 4000)):
        b = Batch([q], [kv], 2, 64, 64, device=DEV, holes=[(0, j, -1) for j in range(-(-kv // 64))])
        b.pages.fill_(-INF)
        out = ops.attention_paged(rnd(q, 4 * 64).to(BF), b.pages, b.table, b.cu_q, b.kv_len, 4, 2, 64)
        assert (out == 0).all()


# ---- strides that say nothing -----------------------------------------------------------------------------------------------------
def test_rope_axes_table_of_one_set_of_positions_for_all_axes():
    """text: the same positions on every axis, expanded, not copied"""
    inv = (1.0 / (1e6 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))).to(DEV)
    for n in (1, 2, 300):
        p = torch.arange(n, device=DEV) + 7
        for axes in (1, 2, 3, 4):
            amap = [i % axes for i in range(64)]
            assert torch.equal(ops.rope_axes_table(inv, p.expand(axes, n), amap), ops.rope_axes_table(inv, p.expand(axes, n).contiguous(), amap))


def test_paged_views_of_one_entry():
    """a single page out of larger ones, a table of one column, a single row of an odd pitch, a single slot, a single layer: the stride along an axis of one entry says nothing"""
    Hq, Hkv, hd, page = 4, 2, 64, 16
    big = rnd(3, 64, 2 * Hkv * hd, seed=1).to(BF)
    one, same = big[1:2, :page], big[1:2, :page].contiguous()
    assert one.stride(0) != page * one.stride(1)
    column, dense = i32([[7, 0, 9]] * 2).t().contiguous().t()[:, 1:2], i32([[0], [0]])
    assert column.stride() == (1, 2)
    lens, cu = i32([9, 4]), i32([0, 1, 1])
    wide = rnd(1, (Hq + 2 * Hkv) * hd + 3, seed=2).to(BF)
    row = wide.as_strided((1, (Hq + 2 * Hkv) * hd), (wide.shape[1], 1))
    assert row.stride(0) % 8
    tab = rnd(1, hd, seed=3)
    b = same.clone()
    pool = big.clone()
    view = pool[1:2, :page]
    q1 = ops.rope_kv_paged(row, tab, Hq, Hkv, hd, view, column, cu, lens, q_out=torch.empty(1, Hq * hd + 1, device=DEV, dtype=BF))[:, :Hq * hd]
    q2 = ops.rope_kv_paged(row.clone(memory_format=torch.contiguous_format), tab, Hq, Hkv, hd, b, dense, cu, lens)
    assert torch.equal(q1, q2) and torch.equal(view, b) and torch.equal(pool[1, page:], big[1, page:]) and torch.equal(pool[::2], big[::2])
    o1 = ops.attention_paged(q1, view, column, cu, lens, Hq, Hkv, hd)
    assert torch.equal(o1, ops.attention_paged(q2.contiguous(), b, dense, cu, lens, Hq, Hkv, hd)) and o1.abs().max() > 0
    assert torch.equal(ops.rope_rows_table(row, tab, 3, 2, hd, out=torch.empty(1, 2 * hd + 5, device=DEV, dtype=BF))[:, :2 * hd],
                       ops.rope_rows_table(row[:, 3:].contiguous(), tab, 0, 2, hd, out=torch.empty(1, 2 * hd, device=DEV, dtype=BF)))
    layers = rnd(4, 5, 64, 24, seed=5).to(BF)
    few = layers[1:3, 2:3, :page]                                                     # one page a layer, out of larger ones
    assert few.stride(1) != page * 24
    keep = layers.clone()
    ops.kv_pages_copy(few, i32([(0, 0, 3), (-1, 0, 2)]))
    tables, held, refs = i32([[-1, -1], [0, -1]]), i32([0, 5]), i32([1])
    assert ops.kv_pages_compact(few, tables, held, refs).tolist() == [1, 0] and torch.equal(layers, keep)
    granted, cu_q, pairs = ops.kv_pages_extend(column, i32([1, 0]), i32([2]), i32([0, 1]), page)
    assert granted.tolist() == [0, 0]


def test_paged_ops_refuse_heads_that_do_not_exist():
    """no heads, no head_dim, negative ones: an error of the operators' own, whatever is computed from them on the way"""
    b = Batch([2], [20], 2, 64, 16, device=DEV)
    q, tab = rnd(2, 512).to(BF), rnd(2, 64)
    for Hq, Hkv, hd in ((4, 2, 0), (4, 2, -8), (0, 2, 64), (-4, 2, 64), (4, 0, 64), (4, -2, 64), (2, 4, 64)):
        with pytest.raises(_lib.UfvError):
            ops.attention_paged(q, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd)
        with pytest.raises(_lib.UfvError):
            ops.attention_paged(q, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd, out=torch.empty_like(q))
        with pytest.raises(_lib.UfvError):
            ops.rope_kv_paged(q, tab if hd == 64 else rnd(2, max(hd, 0)), Hq, Hkv, hd, b.pages, b.table, b.cu_q, b.kv_len)
    for heads, hd in ((0, 64), (-1, 64), (2, 0), (2, -4)):
        with pytest.raises(_lib.UfvError):
            ops.rope_rows_table(q, rnd(2, max(hd, 0)), 0, heads, hd)


@pytest.mark.parametrize("Hq,Hkv,hd", [(4, 2, 128), (4, 2, 72), (2, 1, 256)])
@pytest.mark.parametrize("q,kv", [(3, 50), (40, 300), (150, 1517), (300, 300)])
def test_attention_paged_an_infinite_v_of_weight_nothing_is_nan(Hq, Hkv, hd, q, kv):
    """a key whose score is -inf and whose V holds infinities: 0 times them is NaN in their columns, before the new tokens and among them; the other columns go on without the key"""
    b = Batch([q], [kv], Hkv, hd, 16, seed=hd, device=DEV)
    x = rnd(b.N, Hq * hd, seed=q).to(BF)
    x.view(q, Hq, hd)[:, :, 2] = x.view(q, Hq, hd)[:, :, 2].abs() + 0.125
    clean, first = b.pages.clone(), kv - q
    for at in sorted({first // 64 * 64, max(first - 1, 1), first + 1, kv - 1}):
        if at == 0:                                                               # the only key of the first row: that row has no softmax
            continue
        b.pages.copy_(clean)
        b.pages[b.row(0, at)][(Hkv - 1) * hd + 2] = -INF
        b.pages[b.row(0, at)][(2 * Hkv - 1) * hd + 4], b.pages[b.row(0, at)][2 * Hkv * hd - 1] = INF, -INF
        got = ops.attention_paged(x, b.pages, b.table, b.cu_q, b.kv_len, Hq, Hkv, hd)
        want, slack = attend(b, x, Hq)
        assert torch.isnan(want).any(0).sum() == 2 * (Hq // Hkv)
        same_kind(got, want, slack, f"key {at} of {kv}, {q} new")
