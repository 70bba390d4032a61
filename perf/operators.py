"""Workloads of the paged-cache operators: rotary positions with several axes, the rotated append of new tokens to a
paged KV cache, attention of a chunk of new tokens over such a cache, and the cache's page management (fork, extend,
free, compact, copy).

Every case is one pass through one operator as a program that answers several questions about one video makes it: the
prompt's pages are shared by all questions, new tokens are appended and attended to in one packed batch, and finished
answers give their pages back.  `run` computes a pass from elementary torch operations, or, where `own` is true, through
`ufvideo_amd.ops`; `exact` computes the same outputs in 64 bits from the definitions.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ---- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    heads7 = dict(Hq=28, Hkv=4, hd=128)                     # the decoder's own head layout
    return [
        # rotary positions (time, height, width) of a whole 32-frame prompt, q and k heads of the fused qkv rows, one layer
        dict(name="rope_prompt", kind="rope", N=2399, sections="16,24,24", interleaved=False, backward=False, pos0=0, **heads7),
        # the gradient of the same rotation over a long packed training batch, positions far out, axes interleaved
        dict(name="rope_grad_long", kind="rope", N=16383, sections="24,20,20", interleaved=True, backward=True, pos0=500000, **heads7),
        # one new token of one conversation: latency
        dict(name="append_one", kind="append", S=1, q_lo=1, q_hi=1, kv_lo=2400, kv_hi=2400, page=64, **heads7),
        # chunks of new tokens of eight conversations, ragged
        dict(name="append_chunks", kind="append", S=8, q_lo=130, q_hi=1900, kv_lo=2000, kv_hi=5000, page=64, **heads7),
        # one new token against a long cache: the decode step of a long video
        dict(name="attend_one_long", kind="attend", S=1, q_lo=1, q_hi=1, kv_lo=31999, kv_hi=31999, shared=0, page=64, **heads7),
        # the smallest call: the first answer tokens of a short prompt
        dict(name="attend_one_short", kind="attend", S=1, q_lo=1, q_hi=1, kv_lo=333, kv_hi=333, shared=0, page=64, **heads7),
        # a decode step of many conversations of different lengths
        dict(name="attend_batch", kind="attend", S=48, q_lo=1, q_hi=1, kv_lo=700, kv_hi=6100, shared=0, page=64, **heads7),
        # sixteen questions (their ids as one packed chunk batch) over the pages of one shared video prompt
        dict(name="attend_questions", kind="attend", S=16, q_lo=9, q_hi=83, kv_lo=2321, kv_hi=2395, shared=2304, page=64, **heads7),
        # a long chunk over a long cache: the second video of a conversation
        dict(name="attend_chunk_long", kind="attend", S=1, q_lo=2399, q_hi=2399, kv_lo=20011, kv_hi=20011, shared=0, page=64, **heads7),
        # whole prompts of a smaller decoder (head_dim 64, small pages), ragged, nothing cached before
        dict(name="attend_prompts_hd64", kind="attend", S=5, q_lo=190, q_hi=1700, kv_lo=190, kv_hi=1700, shared=0, page=16, Hq=14, Hkv=2, hd=64),
        # one prompt forked for its questions: shared pages, the copied last page of every child, room for the new tokens
        dict(name="pages_fork", kind="fork", S=24, prompt=2399, n_lo=9, n_hi=83, page=64, width=1024, layers=28),
        # requests come, half of them finish, the cache is compacted: whole pages of every layer move
        dict(name="pages_compact", kind="compact", S=16, prompt=1100, n_lo=120, n_hi=760, page=64, width=1024, layers=28),
    ]


def _spread(i, n, lo, hi):
    """length of entry i of n in [lo, hi], scattered, the same for every seed (`work` knows the sizes from the case alone)"""
    if n == 1 or lo == hi:
        return hi
    return lo + ((i * 7919 + 331) % 997) * (hi - lo) // 996


def _q_lens(c):
    return [_spread(i, c["S"], c["q_lo"], c["q_hi"]) for i in range(c["S"])]


def _kv_lens(c):
    q = _q_lens(c)
    return [max(_spread(i, c["S"], c["kv_lo"], c["kv_hi"]), q[i], c.get("shared", 0) + q[i]) for i in range(c["S"])]


def _n_new(c):
    return [0] + [_spread(i, c["S"], c["n_lo"], c["n_hi"]) for i in range(1, c["S"])]


def _cd(a, b):
    return -(-a // b)


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _third(hd):
    a = hd // 2 // 3
    return f"{hd // 2 - 2 * a},{a},{a}"


def draw(rng):
    """one more case of the listed ones' ranges, never larger than the largest of its kind"""
    top = {}
    for c in listed():
        w = work(c)
        t = top.setdefault(c["kind"], [0, 0])
        top[c["kind"]] = [max(t[0], w["bytes"]), max(t[1], w["flops"])]
    while True:
        kind = rng.choice(["rope", "append", "attend", "attend", "attend", "fork", "compact"])
        Hq, Hkv, hd = rng.choice([(28, 4, 128), (14, 2, 64), (16, 2, 128), (12, 2, 128), (8, 8, 64), (32, 8, 128), (16, 16, 96)])
        page = rng.choice([16, 32, 64, 128])
        if kind == "rope":
            c = dict(kind=kind, N=_log_int(rng, 1, 16383), Hq=Hq, Hkv=Hkv, hd=hd, sections=_third(hd), interleaved=rng.random() < 0.5,
                     backward=rng.random() < 0.5, pos0=_log_int(rng, 1, 1000000))
        elif kind in ("append", "attend"):
            S = _log_int(rng, 1, 64)
            q_hi = 1 if rng.random() < 0.4 else _log_int(rng, 2, 2399)
            kv_hi = _log_int(rng, q_hi, 32000)
            c = dict(kind=kind, S=S, q_lo=_log_int(rng, 1, q_hi), q_hi=q_hi, kv_lo=_log_int(rng, max(1, kv_hi // 8), kv_hi), kv_hi=kv_hi, page=page,
                     Hq=Hq, Hkv=Hkv, hd=hd)
            if kind == "attend":
                c["shared"] = page * (kv_hi // (2 * page)) if S > 1 and rng.random() < 0.3 else 0
        else:
            n_hi = _log_int(rng, 2, 760)
            c = dict(kind=kind, S=_log_int(rng, 2, 24), prompt=_log_int(rng, 17, 2399), n_lo=_log_int(rng, 1, n_hi), n_hi=n_hi, page=page,
                     width=rng.choice([256, 512, 1024, 2048]), layers=rng.choice([2, 12, 24, 28]))
        w = work(c)
        if w["bytes"] <= top[kind][0] and w["flops"] <= max(top[kind][1], 1):
            return c


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(c):
    k = c["kind"]
    if k == "rope":
        hs = (c["Hq"] + c["Hkv"]) * c["hd"]
        return {"bytes": c["N"] * (3 * 8 + c["hd"] * 4 + 2 * hs * 2), "flops": c["N"] * hs * 3}
    if k == "append":
        n = sum(_q_lens(c))
        return {"bytes": n * (2 * (c["Hq"] + 2 * c["Hkv"]) * c["hd"] * 2 + c["hd"] * 4), "flops": n * (c["Hq"] + c["Hkv"]) * c["hd"] * 3}
    if k == "attend":
        q, kv, sh = _q_lens(c), _kv_lens(c), c["shared"]
        keys = sh + sum(n - sh for n in kv)
        pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(q, kv))
        return {"bytes": keys * 2 * c["Hkv"] * c["hd"] * 2 + 2 * sum(q) * c["Hq"] * c["hd"] * 2, "flops": 4 * pairs * c["Hq"] * c["hd"]}
    row = c["layers"] * c["width"] * 2
    if k == "fork":
        rows = (c["S"] - 1) * (c["prompt"] % c["page"])
        return {"bytes": 2 * rows * row + 4 * (c["S"] * _table_width(c) + _pool_pages(c)), "flops": 0}
    live, moved = _compact_counts(c)
    return {"bytes": 2 * moved * c["page"] * row + 4 * (c["S"] * _table_width(c) + _pool_pages(c)), "flops": 0}


def _table_width(c):
    return _cd(c["prompt"] + c["n_hi"], c["page"]) + 2


def _pool_pages(c):
    if c["kind"] == "fork":
        return _cd(c["prompt"], c["page"]) + sum(_cd(n, c["page"]) + 1 for n in _n_new(c)) + 3
    return _cd(c["prompt"], c["page"]) + sum(_cd(n, c["page"]) for n in _n_new(c)) + 3


def _compact_counts(c):
    """(live pages, moved pages) after every second request has given its pages back"""
    p, at, live = c["page"], _cd(c["prompt"], c["page"]), list(range(_cd(c["prompt"], c["page"])))
    for i, n in enumerate(_n_new(c)):
        if i % 2 == 1:
            live += list(range(at, at + _cd(n, p)))
        at += _cd(n, p)
    return len(live), sum(1 for x in live if x >= len(live))


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _axis_map(sections, interleaved, half):
    s = [int(x) for x in sections.split(",")]
    if not interleaved:
        return [a for a, n in enumerate(s) for _ in range(n)]
    return [i % len(s) if i < len(s) * s[i % len(s)] else 0 for i in range(half)]


def _positions(N, pos0):
    """(time, height, width) of a text / video / text row sequence: a text row has its index on all three axes, a visual row its frame
    and its place in a 12 x 12 grid, and the text after a video goes on from the largest index used"""
    text, grid = 43, 12
    out, at, n = [], pos0, 0
    while n < N:
        t = np.arange(at, at + text)
        out.append(np.stack([t, t, t]))
        at, n = at + text, n + text
        frames = 16
        f, h, w = np.meshgrid(np.arange(frames), np.arange(grid), np.arange(grid), indexing="ij")
        out.append(np.stack([f.ravel(), h.ravel(), w.ravel()]) + at)
        at, n = at + max(frames, grid), n + frames * grid * grid
    return torch.from_numpy(np.concatenate(out, 1)[:, :N].astype(np.int64)).to(DEV)


def _inv_freq(hd, base=1e6):
    return (1.0 / (base ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd))).to(DEV)


def _gain(hd, g):
    """projections have a few strong channels"""
    v = torch.ones(hd, device=DEV)
    v[torch.randperm(hd, generator=g, device=DEV)[: hd // 16]] = 2.5
    return v


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    k = c["kind"]
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    bf = torch.bfloat16
    if k == "rope":
        H, hd, N = c["Hq"] + c["Hkv"], c["hd"], c["N"]
        x = (rnd(N, c["Hq"] + 2 * c["Hkv"], hd) * _gain(hd, g)).to(bf).view(N, -1)
        st = dict(x=x, positions=_positions(N, c["pos0"] + seed % 97), inv_freq=_inv_freq(hd), out=torch.zeros(N, H * hd, device=DEV, dtype=bf),
                  axis_of=_axis_map(c["sections"], c["interleaved"], hd // 2))
    elif k in ("append", "attend"):
        Hq, Hkv, hd, p, S = c["Hq"], c["Hkv"], c["hd"], c["page"], c["S"]
        ql, kl, sh = _q_lens(c), _kv_lens(c), c.get("shared", 0) // p
        need = [_cd(n, p) for n in kl]
        total = sh + sum(n - sh for n in need)
        P = total + total // 8 + 1
        perm = torch.randperm(P, generator=g, device=DEV).tolist()
        table, at = [[-1] * (max(need) + 1) for _ in range(S)], sh
        for s in range(S):
            for j in range(need[s]):
                table[s][j] = perm[j] if j < sh else perm[at + j - sh]
            at += need[s] - sh
        pages = rnd(P, p, 2 * Hkv, hd)
        pages[:, :, :Hkv] *= _gain(hd, g) * 0.7
        st = dict(pages=pages.to(bf).view(P, p, 2 * Hkv * hd), table=_i32(table), kv_len=_i32(kl), q_lens=ql, kv_lens=kl,
                  cu_q=_i32([0] + np.cumsum(ql).tolist()))
        del pages
        N = sum(ql)
        if k == "append":
            st["qkv"] = (rnd(N, Hq + 2 * Hkv, hd) * _gain(hd, g)).to(bf).view(N, -1)
            ang = rnd(N, hd // 2) * 100.0
            st["rot"] = torch.cat([torch.cos(ang), torch.sin(ang)], 1)
            st["q_out"] = torch.zeros(N, Hq * hd, device=DEV, dtype=bf)
        else:
            st["q"] = (rnd(N, Hq, hd) * _gain(hd, g)).to(bf).view(N, -1)
            st["out"] = torch.zeros(N, Hq * hd, device=DEV, dtype=bf)
    else:
        S, p, P, have = c["S"], c["page"], _pool_pages(c), _cd(c["prompt"], c["page"])
        table = [[-1] * _table_width(c) for _ in range(S)]
        table[0][:have] = list(range(have))
        n_new = _n_new(c)
        r = (seed % 5) if k == "fork" else 0                      # other inputs: another question takes another slot
        n_new = [0] + n_new[1 + r % (S - 1):] + n_new[1:1 + r % (S - 1)]
        st = dict(pool=rnd(c["layers"], P, p, c["width"]).to(bf), table=_i32(table), kv_len=_i32([c["prompt"]] + [0] * (S - 1)),
                  refs=_i32([1] * have + [0] * (P - have)), n_new=_i32(n_new), parent=_i32([-1] + [0] * (S - 1)),
                  others=_i32([0] + [1] * (S - 1)), half=_i32([1 if i and i % 2 == 0 else 0 for i in range(S)]))
    st["case"] = c
    return st


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    return (_run_own if own else _run_plain)(c["kind"], c, st)


def _run_own(k, c, st):
    from ufvideo_amd import ops
    if k == "rope":
        tab = ops.rope_axes_table(st["inv_freq"], st["positions"], st["axis_of"])
        ops.rope_rows_table(st["x"], tab, 0, c["Hq"] + c["Hkv"], c["hd"], out=st["out"], backward=c["backward"])
        return tab, st["out"]
    if k == "append":
        ops.rope_kv_paged(st["qkv"], st["rot"], c["Hq"], c["Hkv"], c["hd"], st["pages"], st["table"], st["cu_q"], st["kv_len"], q_out=st["q_out"])
        return st["q_out"], st["pages"]
    if k == "attend":
        return ops.attention_paged(st["q"], st["pages"], st["table"], st["cu_q"], st["kv_len"], c["Hq"], c["Hkv"], c["hd"], out=st["out"])
    pool, table, kv_len, refs = st["pool"], st["table"], st["kv_len"], st["refs"]
    ops.kv_pages_free(table, kv_len, refs, st["others"], c["page"])               # the answers of the pass before are finished
    if k == "fork":
        ops.kv_pages_fork(table, kv_len, refs, st["parent"], c["page"])
        granted, cu_q, pairs = ops.kv_pages_extend(table, kv_len, refs, st["n_new"], c["page"])
        ops.kv_pages_copy(pool, pairs)
        return table, kv_len, refs, granted, cu_q, pairs, pool
    ops.kv_pages_extend(table, kv_len, refs, st["n_new"], c["page"])
    ops.kv_pages_free(table, kv_len, refs, st["half"], c["page"])
    counts = ops.kv_pages_compact(pool, table, kv_len, refs)
    return table, kv_len, refs, counts, pool


def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h], x[..., h:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)


def _run_plain(k, c, st):
    if k == "rope":
        hd, H, N = c["hd"], c["Hq"] + c["Hkv"], c["N"]
        pos = st["positions"][torch.tensor(st["axis_of"], device=DEV)].double()              # [hd/2, N]; 64 bits: a far position's angle has no 32-bit value
        ang = pos.t() * st["inv_freq"].double()
        tab = torch.cat([torch.cos(ang), torch.sin(ang)], 1).float()
        cos, sin = tab[:, None, :hd // 2], tab[:, None, hd // 2:]
        y = _rotate(st["x"][:, :H * hd].view(N, H, hd).float(), cos, -sin if c["backward"] else sin)
        st["out"].copy_(y.view(N, H * hd))
        return tab, st["out"]
    if k == "append":
        Hq, Hkv, hd, p = c["Hq"], c["Hkv"], c["hd"], c["page"]
        cu, kl = st["cu_q"].long(), st["kv_len"].long()
        N = st["qkv"].shape[0]
        r = torch.arange(N, device=DEV)
        b = torch.searchsorted(cu[1:], r, right=True)
        pos = kl[b] - (cu[b + 1] - cu[b]) + r - cu[b]
        slot = st["table"].long()[b, pos // p] * p + pos % p
        x = st["qkv"].view(N, Hq + 2 * Hkv, hd).float()
        y = _rotate(x[:, :Hq + Hkv], st["rot"][:, None, :hd // 2], st["rot"][:, None, hd // 2:]).to(torch.bfloat16)
        st["q_out"].copy_(y[:, :Hq].reshape(N, -1))
        st["pages"].view(-1, 2 * Hkv * hd)[slot] = torch.cat([y[:, Hq:].reshape(N, -1), st["qkv"][:, (Hq + Hkv) * hd:]], 1)
        return st["q_out"], st["pages"]
    if k == "attend":
        Hq, Hkv, hd, p = c["Hq"], c["Hkv"], c["hd"], c["page"]
        G, at = Hq // Hkv, 0
        for s, (n, kv) in enumerate(zip(st["q_lens"], st["kv_lens"])):
            rows = st["pages"][st["table"][s, :_cd(kv, p)].long()].view(-1, 2 * Hkv, hd)[:kv].float()
            K, V = rows[:, :Hkv].permute(1, 2, 0).contiguous(), rows[:, Hkv:].permute(1, 0, 2).contiguous()
            step = max(1, (1 << 29) // (kv * Hq))
            for i0 in range(0, n, step):
                i1 = min(n, i0 + step)
                q = st["q"][at + i0:at + i1].view(i1 - i0, Hkv, G, hd).float().permute(1, 0, 2, 3).reshape(Hkv, -1, hd)
                sc = (q @ K) * hd ** -0.5
                if kv - n + i0 + 1 < kv:
                    seen = torch.arange(kv, device=DEV) <= torch.arange(kv - n + i0, kv - n + i1, device=DEV)[:, None]
                    sc = torch.where(seen.repeat_interleave(G, 0), sc, float("-inf"))
                e = torch.exp(sc - sc.amax(-1, keepdim=True))
                o = (e @ V) / e.sum(-1, keepdim=True)
                st["out"][at + i0:at + i1] = o.view(Hkv, i1 - i0, G, hd).permute(1, 0, 2, 3).reshape(i1 - i0, -1).to(torch.bfloat16)
                del sc, e, o
            at += n
        return st["out"]
    _plain_free(c, st, st["others"])
    if k == "fork":
        _plain_fork(c, st, st["parent"])
        granted, cu_q, pairs = _plain_extend(c, st, st["n_new"])
        rows = torch.arange(c["page"], device=DEV)
        src, dst, n = pairs[pairs[:, 0] >= 0].long().unbind(1)
        take = (rows < n[:, None]).view(1, -1, c["page"], 1)
        st["pool"][:, dst] = torch.where(take, st["pool"][:, src], st["pool"][:, dst])
        return st["table"], st["kv_len"], st["refs"], granted, cu_q, pairs, st["pool"]
    _plain_extend(c, st, st["n_new"])
    _plain_free(c, st, st["half"])
    live = st["refs"] > 0
    ids = torch.arange(live.numel(), device=DEV)
    K = live.sum()
    dst, src = ids[~live & (ids < K)], ids[live & (ids >= K)]
    new = ids.clone()
    new[src] = dst
    st["pool"][:, dst] = st["pool"][:, src]
    st["refs"][dst] = st["refs"][src]
    st["refs"][src] = 0
    st["table"].copy_(torch.where(st["table"] >= 0, new[st["table"].clamp(min=0).long()].int(), st["table"]))
    counts = torch.stack([K, torch.full_like(K, dst.numel())]).int()
    return st["table"], st["kv_len"], st["refs"], counts, st["pool"]


def _held(c, st):
    """which table entries hold a page"""
    W = st["table"].shape[1]
    return torch.arange(W, device=DEV) < ((st["kv_len"] + c["page"] - 1) // c["page"])[:, None]


def _plain_free(c, st, mask):
    gone = _held(c, st) & (mask != 0)[:, None]
    P = st["refs"].numel()
    n = torch.zeros(P + 1, dtype=torch.int32, device=DEV)
    n.scatter_add_(0, torch.where(gone, st["table"], P).long().view(-1), torch.ones(gone.numel(), dtype=torch.int32, device=DEV))
    st["refs"] -= n[:P]
    st["table"].masked_fill_(gone, -1)
    st["kv_len"].masked_fill_(mask != 0, 0)


def _plain_fork(c, st, parent):
    p = parent.clamp(min=0).long()
    ok = (parent >= 0) & (st["kv_len"] == 0) & (parent[p] < 0)
    st["kv_len"].copy_(torch.where(ok, st["kv_len"][p], st["kv_len"]))
    new = _held(c, st) & ok[:, None]
    st["table"].copy_(torch.where(new, st["table"][p], st["table"]))
    P = st["refs"].numel()
    n = torch.zeros(P + 1, dtype=torch.int32, device=DEV)
    n.scatter_add_(0, torch.where(new, st["table"], P).long().view(-1), torch.ones(new.numel(), dtype=torch.int32, device=DEV))
    st["refs"] += n[:P]


def _plain_extend(c, st, n_new):
    p, table, kv_len, refs = c["page"], st["table"], st["kv_len"], st["refs"]
    W, P = table.shape[1], refs.numel()
    n = n_new.clamp(min=0)
    have, want = (kv_len + p - 1) // p, (kv_len + n + p - 1) // p
    last = torch.gather(table, 1, (have - 1).clamp(min=0).long()[:, None])[:, 0]
    shared = (n > 0) & (kv_len % p != 0) & (refs[last.clamp(min=0).long()] > 1)
    fits = want <= W
    need = torch.where((n > 0) & fits, want - have + shared.int(), 0)
    end = torch.cumsum(need, 0)
    free = torch.argsort((refs != 0).int(), stable=True).int()                  # the free pages' ids come first, ascending
    ok = fits & (n > 0) & ((need == 0) | (end <= (refs == 0).sum()))
    start = have - shared.int()
    j = torch.arange(W, device=DEV) - start[:, None]
    new = (j >= 0) & (j < need[:, None]) & ok[:, None]
    page = free[(j + (end - need)[:, None]).clamp(0, P - 1).long()]
    copied = ok & shared
    gone = torch.zeros(P + 1, dtype=torch.int32, device=DEV)
    gone.scatter_add_(0, torch.where(copied, last, P).long(), torch.ones_like(last))
    got = torch.zeros(P + 1, dtype=torch.int32, device=DEV)
    got.scatter_(0, torch.where(new, page, P).long().view(-1), 1)
    table.copy_(torch.where(new, page, table))
    refs += got[:P] - gone[:P]
    dst = torch.gather(table, 1, start.clamp(0, W - 1).long()[:, None])[:, 0]
    pairs = torch.stack([torch.where(copied, last, -1), torch.where(copied, dst, -1), torch.where(copied, kv_len % p, 0)], 1)
    granted = torch.where(ok, n, 0)
    kv_len += granted
    cu_q = torch.cat([torch.zeros_like(granted[:1]), torch.cumsum(granted, 0).int()])
    return granted, cu_q, pairs


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------
def exact(case, seed):
    c, st = case, prepare(case, seed)
    k = c["kind"]
    if k == "rope":
        hd, N, H = c["hd"], c["N"], c["Hq"] + c["Hkv"]
        ang = torch.empty(N, hd // 2, dtype=torch.float64, device=DEV)
        for i, a in enumerate(st["axis_of"]):
            ang[:, i] = st["positions"][a].double() * float(st["inv_freq"][i])
        z = torch.polar(torch.ones_like(ang), -ang if c["backward"] else ang)[:, None]
        x = st["x"][:, :H * hd].double().view(N, H, 2, hd // 2)
        y = torch.complex(x[:, :, 0], x[:, :, 1]) * z                     # a rotation of (x_i, x_{i + hd/2}) is a complex product
        return torch.cat([torch.cos(ang), torch.sin(ang)], 1), torch.cat([y.real, y.imag], -1).view(N, H * hd)
    if k == "append":
        Hq, Hkv, hd, p = c["Hq"], c["Hkv"], c["hd"], c["page"]
        pages, table = st["pages"].double(), st["table"].tolist()
        z = torch.complex(st["rot"][:, :hd // 2].double(), st["rot"][:, hd // 2:].double())[:, None]
        x = st["qkv"].double().view(-1, Hq + 2 * Hkv, 2, hd // 2)
        y = torch.complex(x[:, :Hq + Hkv, 0], x[:, :Hq + Hkv, 1]) * z
        y = torch.cat([y.real, y.imag], -1)
        rows = torch.cat([y[:, Hq:], x[:, Hq + Hkv:].reshape(-1, Hkv, hd)], 1).view(-1, 2 * Hkv * hd)
        at = 0
        for s, (n, kv) in enumerate(zip(st["q_lens"], st["kv_lens"])):
            for pos in range(kv - n, kv):
                pages[table[s][pos // p], pos % p] = rows[at]
                at += 1
        return y[:, :Hq].reshape(-1, Hq * hd), pages
    if k == "attend":
        Hq, Hkv, hd, p = c["Hq"], c["Hkv"], c["hd"], c["page"]
        out, at = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV), 0
        for s, (n, kv) in enumerate(zip(st["q_lens"], st["kv_lens"])):
            rows = torch.cat([st["pages"][j] for j in st["table"][s, :_cd(kv, p)].tolist()])[:kv]
            for h in range(Hq):
                g = h // (Hq // Hkv)
                key, val = rows[:, g * hd:(g + 1) * hd].double(), rows[:, (Hkv + g) * hd:(Hkv + g + 1) * hd].double()
                for i0 in range(0, n, 1024):
                    i1 = min(n, i0 + 1024)
                    sc = st["q"][at + i0:at + i1, h * hd:(h + 1) * hd].double() @ key.t() / math.sqrt(hd)
                    late = torch.arange(kv, device=DEV)[None] > (kv - n + torch.arange(i0, i1, device=DEV))[:, None]
                    sc.masked_fill_(late, float("-inf"))
                    out[at + i0:at + i1, h * hd:(h + 1) * hd] = torch.exp(sc - torch.logsumexp(sc, 1, keepdim=True)) @ val
            at += n
        return out
    # page management: one request after another on the host
    S, p = c["S"], c["page"]
    table, lens, refs, n_new = st["table"].tolist(), st["kv_len"].tolist(), st["refs"].tolist(), st["n_new"].tolist()
    pool = st["pool"].double()
    granted, cu, pairs = [], [0], []
    if k == "fork":
        for s in range(1, S):
            table[s], lens[s] = list(table[0]), lens[0]
            for j in range(_cd(lens[0], p)):
                refs[table[0][j]] += 1
    was = list(refs)
    free = [i for i, r in enumerate(refs) if r == 0]
    for s in range(S):
        n, pair = n_new[s], [-1, -1, 0]
        if n:
            j = _cd(lens[s], p)
            if lens[s] % p and was[table[s][j - 1]] > 1:
                src, dst = table[s][j - 1], free.pop(0)
                pair = [src, dst, lens[s] % p]
                pool[:, dst, :pair[2]] = pool[:, src, :pair[2]]
                table[s][j - 1] = dst
                refs[src] -= 1
                refs[dst] += 1
            while j < _cd(lens[s] + n, p):
                table[s][j] = free.pop(0)
                refs[table[s][j]] += 1
                j += 1
            lens[s] += n
        granted.append(n)
        cu.append(cu[-1] + n)
        pairs.append(pair)
    if k == "fork":
        return _i32(table), _i32(lens), _i32(refs), _i32(granted), _i32(cu), _i32(pairs), pool
    for s in range(2, S, 2):
        for j in range(_cd(lens[s], p)):
            refs[table[s][j]] -= 1
            table[s][j] = -1
        lens[s] = 0
    live = sum(1 for r in refs if r)
    moved = 0
    for dst in range(live):
        if refs[dst] == 0:
            src = next(i for i in range(live, len(refs)) if refs[i])
            pool[:, dst] = pool[:, src]
            refs[dst], refs[src] = refs[src], 0
            table = [[dst if x == src else x for x in row] for row in table]
            moved += 1
    return _i32(table), _i32(lens), _i32(refs), _i32([live, moved]), pool
