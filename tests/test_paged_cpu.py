"""CPU: refusals of the paged-cache entry points, the bounds of a page lookup, and the oracle's page bookkeeping (tests/paged_ref.py) against its own invariants."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from conftest import ROOT
from paged_ref import PageModel
from ufvideo_amd import _lib, ops


def _buf(n=1 << 14):
    b = (ctypes.c_char * (n + 64))()
    a = ctypes.addressof(b)
    return b, a + (-a) % 64


def _refused(name, good, **bad):
    """the call with one argument changed is refused on the host, before anything is launched (the arguments are host addresses: a launch would be noticed)"""
    args = dict(good)
    for k in bad:
        assert k in args, k
    args.update(bad)
    rc = getattr(_lib.load(), name)(*args.values())
    assert rc == -1, (name, bad, rc)
    assert name in _lib.load().ufv_last_error().decode()


def test_paged_entry_points_refuse_bad_arguments():
    keep, p = _buf()
    att = dict(q=p, ldq=256, o=p, ldo=256, N=4, Hq=4, Hkv=2, hd=64, pages=p, n_pages=8, page=16, ldkv=256, table=p, ld_table=4, max_pages=4, cu_q=p, kv_len=p, S=3, scale=0.1, causal=1,
               ws=p, ws_bytes=1 << 40, stream=0)
    for bad in (dict(q=0), dict(o=0), dict(pages=0), dict(table=0), dict(cu_q=0), dict(kv_len=0), dict(N=0), dict(N=-1), dict(S=0), dict(n_pages=0), dict(max_pages=0), dict(Hq=0), dict(Hq=3),
                dict(Hkv=0), dict(hd=0), dict(hd=4), dict(hd=60), dict(hd=264), dict(page=0), dict(page=8), dict(page=48), dict(page=1 << 16), dict(q=p + 2), dict(o=p + 8), dict(pages=p + 4),
                dict(ldq=255), dict(ldo=252), dict(ldkv=260), dict(ldkv=248), dict(ldq=248), dict(ldo=128), dict(ld_table=3), dict(max_pages=1 << 28, ld_table=1 << 28)):
        _refused("ufv_attention_paged", att, **bad)
    app = dict(qkv=p, ldqkv=512, q_out=p, ldq=256, N=4, Hq=4, Hkv=2, hd=64, tab=p, pages=p, n_pages=8, page=16, ldkv=256, table=p, ld_table=4, max_pages=4, cu_q=p, kv_len=p, S=3, stream=0)
    for bad in (dict(qkv=0), dict(q_out=0), dict(tab=0), dict(pages=0), dict(N=0), dict(hd=24), dict(Hkv=0), dict(page=12), dict(ldqkv=504), dict(ldqkv=508), dict(ldq=248), dict(ldkv=248),
                dict(qkv=p + 8), dict(q_out=p + 2), dict(tab=p + 4)):
        _refused("ufv_rope_kv_paged", app, **bad)
    axes = (ctypes.c_uint8 * 32)(*([0] * 16 + [1] * 8 + [2] * 8))
    tab = dict(inv=p, pos=p, ld=4, n_axes=3, axis_of=ctypes.addressof(axes), N=4, hd=64, table=p, stream=0)
    for bad in (dict(inv=0), dict(pos=0), dict(axis_of=0), dict(table=0), dict(N=0), dict(hd=63), dict(hd=258), dict(n_axes=0), dict(n_axes=5), dict(n_axes=2), dict(ld=3)):
        _refused("ufv_rope_axes_table", tab, **bad)
    rows = dict(x=p, ldx=256, y=p, ldy=256, N=4, nheads=4, hd=64, table=p, backward=0, stream=0)
    for bad in (dict(x=0), dict(y=0), dict(table=0), dict(N=0), dict(nheads=0), dict(hd=0), dict(hd=33), dict(ldx=255), dict(ldy=255)):
        _refused("ufv_rope_rows_table", rows, **bad)
    man = dict(table=p, ld=4, max_pages=4, kv_len=p, S=3, refs=p, n_pages=8, page=16)
    for name, more in (("ufv_kv_pages_fork", dict(v=p)), ("ufv_kv_pages_free", dict(v=p)), ("ufv_kv_pages_extend", dict(v=p, granted=p, cu_q=p, pairs=p, ws=p, ws_bytes=1 << 20))):
        good = dict(man, **more, stream=0)
        for bad in (dict(table=0), dict(kv_len=0), dict(refs=0), dict(v=0), dict(S=0), dict(n_pages=0), dict(max_pages=0), dict(ld=3), dict(page=0), dict(page=24)):
            _refused(name, good, **bad)
    ext = dict(man, v=p, granted=p, cu_q=p, pairs=p, ws=p, ws_bytes=1 << 20, stream=0)
    need = _lib.load().ufv_kv_pages_extend_ws_bytes(3, 8)
    for bad in (dict(ws=0), dict(ws_bytes=need - 1), dict(granted=0), dict(cu_q=0), dict(pairs=0), dict(max_pages=(1 << 20) + 1, ld=1 << 21)):
        _refused("ufv_kv_pages_extend", ext, **bad)
    cp = dict(pool=p, layers=2, layer_bytes=8 * 16 * 64, n_pages=8, page=16, row_bytes=64, pairs=p, n=2, stream=0)
    for bad in (dict(pool=0), dict(pool=p + 8), dict(layers=0), dict(layer_bytes=8 * 16 * 64 - 16), dict(layer_bytes=8 * 16 * 64 + 8), dict(n_pages=0), dict(page=20), dict(row_bytes=24),
                dict(row_bytes=0), dict(pairs=0), dict(n=0), dict(n=1 << 16)):
        _refused("ufv_kv_pages_copy", cp, **bad)
    co = dict(pool=p, layers=2, layer_bytes=8 * 16 * 64, row_bytes=64, **man, counts=p, ws=p, ws_bytes=1 << 20, stream=0)
    for bad in (dict(pool=0), dict(counts=0), dict(ws=0), dict(ws_bytes=_lib.load().ufv_kv_pages_compact_ws_bytes(8) - 1), dict(refs=0), dict(row_bytes=8), dict(page=17)):
        _refused("ufv_kv_pages_compact", co, **bad)


def test_attention_paged_refuses_what_its_kernels_do_not_hold_for():
    keep, p = _buf()
    att = dict(q=p, ldq=3584, o=p, ldo=3584, N=3, Hq=28, Hkv=4, hd=128, pages=p, n_pages=4, page=64, ldkv=1024, table=p, ld_table=2, max_pages=2, cu=p, kl=p, S=2, scale=0.1, causal=1, ws=p,
               ws_bytes=1 << 40, stream=0)
    for bad in (dict(scale=0.0), dict(scale=-0.1), dict(scale=float("inf")), dict(scale=float("nan")), dict(ldkv=1 << 24), dict(hd=264), dict(S=1 << 24), dict(N=1 << 27)):
        _refused("ufv_attention_paged", att, **bad)
    lib = _lib.load()
    for N, S, max_pages in ((2, 2, 64), (300, 2, 64), (4000, 2, 64)):
        need = lib.ufv_attention_paged_ws_bytes(N, S, 28, 4, 128, max_pages * 64)
        assert need > 0
        for bad in (dict(ws_bytes=need - 1), dict(ws=0), dict(ws=p + 8)):
            _refused("ufv_attention_paged", dict(att, N=N, S=S, max_pages=max_pages, ld_table=max_pages), **bad)


def test_attention_paged_workspace_does_not_grow_with_the_cache():
    """parts are a number of the card, not of the lengths or the slots; what grows with the slots is one record for each item"""
    ws = _lib.load().ufv_attention_paged_ws_bytes
    assert ws(1, 1, 28, 4, 128, 512) == 0
    one = ws(1, 1, 28, 4, 128, 1 << 20)
    assert one == ws(1, 1, 28, 4, 128, 1 << 24) and ws(5000, 5000, 28, 4, 128, 1 << 20) < 2 * one
    assert ws(16383, 1, 28, 4, 128, 1 << 24) == ws(16383, 1, 28, 4, 128, 1 << 20)


def test_paged_ops_refuse_tensors_off_the_gpu_and_wrong_shapes():
    bf, i32 = torch.bfloat16, torch.int32
    pages = torch.zeros(4, 16, 128, dtype=bf)
    tb, cu, kl, refs = torch.zeros(2, 3, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(4, dtype=i32)
    q = torch.zeros(5, 64, dtype=bf)
    with pytest.raises(_lib.UfvError):
        ops.attention_paged(q, pages, tb, cu, kl, 1, 1, 64)
    with pytest.raises(_lib.UfvError):
        ops.rope_kv_paged(torch.zeros(5, 192, dtype=bf), torch.zeros(5, 64), 1, 1, 64, pages, tb, cu, kl)
    with pytest.raises(_lib.UfvError):
        ops.rope_axes_table(torch.zeros(32), torch.zeros(3, 5, dtype=torch.int64), [0] * 32)
    with pytest.raises(_lib.UfvError):
        ops.rope_rows_table(q, torch.zeros(5, 64), 0, 1, 64)
    for call in (lambda: ops.kv_pages_fork(tb, kl, refs, kl, 16), lambda: ops.kv_pages_extend(tb, kl, refs, kl, 16), lambda: ops.kv_pages_free(tb, kl, refs, kl, 16),
                 lambda: ops.kv_pages_copy(pages[None], torch.zeros(1, 3, dtype=i32)), lambda: ops.kv_pages_compact(pages[None], tb, kl, refs)):
        with pytest.raises(_lib.UfvError):
            call()


def test_rope_axis_map():
    assert ops.rope_axis_map((2, 3, 1)) == [0, 0, 1, 1, 1, 2]
    m = ops.rope_axis_map((24, 20, 20), interleaved=True)
    assert len(m) == 64 and [m.count(a) for a in range(3)] == [24, 20, 20] and m[:6] == [0, 1, 2, 0, 1, 2] and m[60:] == [0] * 4


def test_page_lookup_stays_inside_the_pool(tmp_path):
    """paged_row / paged_len on the host: page ids and lengths outside their ranges name no row (the kernels read only rows that these functions name)"""
    src = tmp_path / "lookup.cpp"
    src.write_text('''
#include "ufvideo_amd/csrc/paged.h"
#include <cstdio>
void ufv_set_error(const char*, ...) {}
int main() {
    const int ids[8] = {2, -1, 5, 0, 4, 2147483647, -2147483647 - 1, 3};
    const int lens[6] = {0, -7, 33, 64, 65, 2147483647};
    PagedTable t{ids, 4, 4, nullptr, lens, 2, 5, 4};
    const int want_len[6] = {0, 0, 33, 64, 64, 64};
    for (int s = 0; s < 6; ++s) if (paged_len(t, s) != want_len[s]) { printf("len %d: %d\\n", s, paged_len(t, s)); return 1; }
    for (int s = 0; s < 2; ++s)
        for (int j = 0; j < 64; ++j) {
            const int id = ids[s * 4 + j / 16];
            const long long want = id >= 0 && id < 5 ? id * 16LL + j % 16 : -1;
            if (paged_row(t, s, j) != want) { printf("row %d %d: %lld\\n", s, j, (long long)paged_row(t, s, j)); return 1; }
        }
    const int far[1] = {200000000};                               // row 200000000 * 16 + 5: past 31 bits
    PagedTable u{far, 1, 1, nullptr, lens, 1, 200000001, 4};
    if (paged_row(u, 0, 5) != 3200000005LL) return 1;
    return paged_log2(16) == 4 && paged_log2(32768) == 15 && paged_log2(8) < 0 && paged_log2(24) < 0 && paged_log2(0) < 0 && paged_log2(65536) < 0 ? 0 : 1;
}
''')
    exe = tmp_path / "lookup"
    subprocess.run(["/opt/rocm/bin/hipcc", "--cuda-host-only", "-x", "hip", "-std=c++17", "-O1", "-I", ROOT, str(src), "-o", str(exe)], check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("seed", range(6))
def test_page_model_keeps_its_books(seed):
    rng = random.Random(seed)
    m = PageModel(rng.randint(1, 9), rng.randint(2, 9), rng.randint(4, 60), 16)
    for _ in range(60):
        k = rng.choice("ffeeeexc")
        if k == "f":
            m.fork([rng.randint(-1, m.S) for _ in range(m.S)])
        elif k == "e":
            before = list(m.lens)
            granted, cu, pairs = m.extend([rng.choice([0, 0, 1, 5, 16, 40, 400, -3]) for _ in range(m.S)])
            assert [a + b for a, b in zip(before, granted)] == m.lens and cu[-1] == sum(granted)
        elif k == "x":
            m.free([rng.random() < 0.3 for _ in range(m.S)])
        else:
            live = sum(1 for r in m.refs if r > 0)
            moves = m.compact()
            assert all(r > 0 for r in m.refs[:live]) and not any(m.refs[live:])
            assert not {a for a, _ in moves} & {b for _, b in moves}
        m.check()


def test_operator_workloads_agree_with_their_definitions():
    """perf/operators.py: the plain form of every kind of case against its 64-bit form, at small sizes on the CPU"""
    import importlib.util
    spec = importlib.util.spec_from_file_location("operator_workloads", os.path.join(ROOT, "perf", "operators.py"))
    O = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(O)
    O.DEV = "cpu"
    cap = dict(N=150, kv_lo=200, kv_hi=200, q_lo=12, q_hi=12, prompt=130, n_hi=70, n_lo=20, layers=2, shared=64, width=32)
    for c in O.listed():
        c = {k: (min(v, cap[k]) if k in cap else v) for k, v in c.items()}
        st = O.prepare(c, 5)
        got, want = O.run(st), O.exact(c, 5)
        for x, y in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            if x.dtype == torch.int32:
                assert torch.equal(x, y), c["name"]
            elif x.dtype == torch.bfloat16:          # one rounding of a 32-bit result
                assert ((x.double() - y).abs() <= 2.0 ** -8 * y.abs() + 2e-4).all(), c["name"]
            else:
                assert (x.double() - y).abs().max() < 1e-6, c["name"]
