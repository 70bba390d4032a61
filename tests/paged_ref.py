"""64-bit oracle of the paged-cache operators, used by tests/test_paged_cpu.py and tests/test_paged_gpu.py: plain loops over slots and rows."""
import torch

HALF_BF16 = 2.0 ** -8          # half a step of bf16, relative to the value
EPS32 = 2.0 ** -24             # half a step of fp32


def cdiv(a, b):
    return -(-a // b)


class Batch:
    """S slots with kv_lens[s] cached tokens, the last q_lens[s] of them new, on pages in random order.  holes: table entries without a valid page id."""

    def __init__(self, q_lens, kv_lens, Hkv, hd, page, seed=0, device="cpu", holes=(), spare_rows=0, extra_width=0, pad=0, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens, self.Hkv, self.hd, self.page = list(q_lens), list(kv_lens), Hkv, hd, page
        S = len(self.q_lens)
        need = [cdiv(n, page) for n in self.kv_lens]
        self.P = sum(need) + 3
        perm = torch.randperm(self.P, generator=g).tolist()
        W = max(need + [1]) + extra_width
        self.table_list, at = [[-1] * W for _ in range(S)], 0
        for s in range(S):
            for j in range(need[s]):
                self.table_list[s][j] = perm[at]
                at += 1
        for s, j, bad in holes:
            self.table_list[s][j] = bad
        self.N = sum(self.q_lens) + spare_rows
        cu = [0]
        for n in self.q_lens:
            cu.append(cu[-1] + n)
        self.cu = cu
        rows = torch.randn(self.P, page, 2 * Hkv * hd + pad, generator=g)
        rows[:, :, :Hkv * hd] *= scale
        self.pages = rows.to(torch.bfloat16).to(device)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
        self.table, self.cu_q, self.kv_len = i32(self.table_list), i32(cu), i32(self.kv_lens)
        self.gen = g

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen).to(torch.bfloat16).to(self.pages.device)

    def row(self, s, j):
        """(page, row in page) of token j of slot s, None where there is no page"""
        p = self.table_list[s][j // self.page]
        return (p, j % self.page) if 0 <= p < self.P else None


def attend(b, q, Hq, scale=None, causal=True, out=None):
    """-> (o, slack): o fp64 [N, Hq*hd] (rows behind the last slot: those of `out`), slack fp64: how far a kernel that forms scores and sums in fp32 and rounds
    the probabilities and the result to bf16 may be off, element by element:
      half a bf16 step of the result;
      A = sum_j p_j |v_j| times: half a bf16 step (every p_j rounded once), twice the largest error of a score (fp32 sum of hd products: hd half steps of sum |q_d k_d|),
      and a half step of fp32 for each of the n keys summed and for the exponentials (16 in all for the two, the log2 form's constant and the division)."""
    hd, Hkv = b.hd, b.Hkv
    scale = hd ** -0.5 if scale is None else scale
    dev = q.device
    o = torch.zeros(q.shape[0], Hq * hd, dtype=torch.float64, device=dev)
    if out is not None:
        o.copy_(out[:, :Hq * hd].double())
    slack = torch.zeros_like(o)
    for s, (n, kv) in enumerate(zip(b.q_lens, b.kv_lens)):
        if n == 0:
            continue
        o[b.cu[s]:b.cu[s + 1]] = 0
        where = [b.row(s, j) for j in range(kv)]
        keys = [j for j in range(kv) if where[j] is not None]
        if not keys:
            continue
        pg = torch.tensor([where[j][0] for j in keys], device=dev)
        rw = torch.tensor([where[j][1] for j in keys], device=dev)
        data = b.pages[pg, rw, :2 * Hkv * hd].double()
        kpos = torch.tensor(keys, device=dev)
        qpos = torch.arange(kv - n, kv, device=dev)
        seen = (kpos[None] <= qpos[:, None]) if causal else torch.ones(n, len(keys), dtype=torch.bool, device=dev)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            K, V = data[:, g * hd:(g + 1) * hd], data[:, (Hkv + g) * hd:(Hkv + g + 1) * hd]
            Q = q[b.cu[s]:b.cu[s + 1], h * hd:(h + 1) * hd].double()
            sc = (Q @ K.t() * scale).masked_fill(~seen, float("-inf"))
            m = sc.amax(1, keepdim=True)
            e = torch.where(seen, torch.exp(sc - torch.where(torch.isinf(m) & (m < 0), 0.0, m)), 0.0)
            l = e.sum(1, keepdim=True)
            p = torch.where(l > 0, e / l, 0.0) if not torch.isnan(l).any() else e / l
            r = torch.zeros(n, hd, dtype=torch.float64, device=dev)
            A = torch.zeros_like(r)
            if torch.isfinite(V).all():
                r, A = p @ V, p @ V.abs()
            else:                                          # a row takes nothing, not even NaN, from a key that it does not see
                for i in range(n):
                    r[i] = (p[i, seen[i], None] * V[seen[i]]).sum(0)
                    A[i] = (p[i, seen[i], None] * V[seen[i]].abs()).sum(0)
            es = hd * EPS32 * scale * (Q.abs() @ K.abs().t()).masked_fill(~seen, 0).nan_to_num(0, 0, 0).amax(1, keepdim=True)
            o[b.cu[s]:b.cu[s + 1], h * hd:(h + 1) * hd] = r
            slack[b.cu[s]:b.cu[s + 1], h * hd:(h + 1) * hd] = HALF_BF16 * r.abs() + A * (HALF_BF16 + 2 * es + (len(keys) + 16) * EPS32)
    return o, slack


def rotate(x, table, backward=False):
    """x [N, H, hd], table fp32 [N, hd] -> (y fp64, slack): three fp32 operations, one rounding to bf16"""
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h].double(), x[..., h:].double()
    c, s = table[:, None, :h].double(), table[:, None, h:].double()
    if backward:
        s = -s
    y = torch.cat([x1 * c - x2 * s, x1 * s + x2 * c], -1)
    mag = torch.cat([(x1 * c).abs() + (x2 * s).abs(), (x1 * s).abs() + (x2 * c).abs()], -1)
    return y, HALF_BF16 * y.abs() + 3 * EPS32 * mag


class PageModel:
    """one request after another, on lists"""

    def __init__(self, S, W, P, page):
        self.S, self.W, self.P, self.page = S, W, P, page
        self.table, self.lens, self.refs = [[-1] * W for _ in range(S)], [0] * S, [0] * P

    def held(self, s):
        return cdiv(self.lens[s], self.page)

    def fork(self, parent):
        was = list(self.lens)
        for s, p in enumerate(parent):
            if 0 <= p < self.S and p != s and parent[p] < 0 and was[s] == 0:
                self.lens[s] = was[p]
                for j in range(self.held(p)):
                    self.table[s][j] = self.table[p][j]
                    self.refs[self.table[p][j]] += 1

    def free(self, mask):
        for s, m in enumerate(mask):
            if m:
                for j in range(self.held(s)):
                    self.refs[self.table[s][j]] -= 1
                    self.table[s][j] = -1
                self.lens[s] = 0

    def extend(self, n_new):
        was, free = list(self.refs), [i for i, r in enumerate(self.refs) if r == 0]
        granted, cu, pairs, taken = [], [0], [], 0
        for s, n in enumerate(n_new):
            n, got, pair = max(n, 0), 0, [-1, -1, 0]
            want = cdiv(self.lens[s] + n, self.page)
            if n and want <= self.W:
                last = self.table[s][self.held(s) - 1] if self.lens[s] % self.page else -1
                copy = last >= 0 and was[last] > 1
                need = want - self.held(s) + copy
                mine = free[taken:taken + need]
                taken += need                                      # later slots do not get what an earlier one was refused
                if len(mine) == need:
                    j = self.held(s)
                    if copy:
                        j -= 1
                        pair = [last, mine[0], self.lens[s] % self.page]
                        self.refs[last] -= 1
                    for id_ in mine:
                        self.table[s][j] = id_
                        self.refs[id_] = 1
                        j += 1
                    self.lens[s] += n
                    got = n
            granted.append(got)
            cu.append(cu[-1] + got)
            pairs.append(pair)
        return granted, cu, pairs

    def compact(self):
        """-> [(src, dst)]"""
        K = sum(1 for r in self.refs if r > 0)
        holes = [i for i in range(K) if self.refs[i] == 0]
        movers = [i for i in range(K, self.P) if self.refs[i] > 0]
        new = dict(zip(movers, holes))
        for src, dst in new.items():
            self.refs[dst], self.refs[src] = self.refs[src], 0
        self.table = [[new.get(x, x) if j < self.held(s) else x for j, x in enumerate(row)] for s, row in enumerate(self.table)]
        return list(new.items())

    def check(self):
        count = [0] * self.P
        for s in range(self.S):
            for j in range(self.W):
                if j < self.held(s):
                    count[self.table[s][j]] += 1
                else:
                    assert self.table[s][j] == -1
        assert count == self.refs
