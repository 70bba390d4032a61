"""CPU: sizes at which an index of the paged-cache kernels would leave 31 bits are refused on the host."""
from test_paged_cpu import _buf, _refused

BIG = 1 << 40


def test_page_management_refuses_more_pages_or_slots_than_its_loops_count():
    """the loops over the pages step by 4096, those over the slots by 1024, and three entries are written a slot"""
    keep, p = _buf()
    man = dict(table=p, ld=4, max_pages=4, kv_len=p, S=3, refs=p, n_pages=8, page=16)
    calls = {"ufv_kv_pages_fork": dict(man, v=p, stream=0), "ufv_kv_pages_free": dict(man, v=p, stream=0),
             "ufv_kv_pages_extend": dict(man, v=p, granted=p, cu_q=p, pairs=p, ws=p, ws_bytes=BIG, stream=0),
             "ufv_kv_pages_compact": dict(pool=p, layers=1, layer_bytes=0, row_bytes=16, **man, counts=p, ws=p, ws_bytes=BIG, stream=0)}
    for name, good in calls.items():
        for bad in (dict(n_pages=(1 << 31) - 4096), dict(n_pages=(1 << 31) - 1), dict(n_pages=(1 << 30) + 1), dict(S=(1 << 31) - 1), dict(S=(1 << 29) + 1)):
            _refused(name, good, **bad)


def test_rows_that_pass_31_bits_are_refused():
    keep, p = _buf()
    att = dict(q=p, ldq=BIG, o=p, ldo=BIG, N=1, Hq=4, Hkv=1, hd=256, pages=p, n_pages=4, page=64, ldkv=512, table=p, ld_table=2, max_pages=2, cu=p, kl=p, S=1, scale=0.1, causal=1, ws=p,
               ws_bytes=BIG, stream=0)
    for bad in (dict(Hq=1 << 23), dict(Hq=(1 << 31) - (1 << 16)), dict(N=(1 << 29) - 1)):             # q columns; (token, head) rows with those of the last tile
        _refused("ufv_attention_paged", att, **bad)
    app = dict(qkv=p, ldqkv=BIG, q_out=p, ldq=BIG, N=1, Hq=4, Hkv=2, hd=64, tab=p, pages=p, n_pages=8, page=16, ldkv=256, table=p, ld_table=4, max_pages=4, cu_q=p, kv_len=p, S=3, stream=0)
    for bad in (dict(Hq=1 << 25), dict(Hq=(1 << 25) - 4), dict(S=(1 << 29) + 1)):
        _refused("ufv_rope_kv_paged", app, **bad)
    rows = dict(x=p, ldx=BIG, y=p, ldy=BIG, N=1, nheads=1 << 25, hd=64, table=p, backward=0, stream=0)
    _refused("ufv_rope_rows_table", rows)
    _refused("ufv_rope_rows_table", rows, nheads=(1 << 30), hd=2)
