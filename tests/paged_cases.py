"""Paged batches for the tests, and their operators in 64 bits."""
import math

import torch

BF16 = torch.bfloat16


class Batch:
    """Sequences of past + q positions in pages scattered over a pool. Slots that
    no position holds are NaN, as are table entries past a sequence's pages no
    page at all; rows behind the last sequence (pad) belong to none."""

    def __init__(self, dev, q, past, nh, nkv, hd, page, cache, seed, pad=0, lead=0, extra=3, wide=0, apart=0, stray=0):
        g = torch.Generator(device="cpu")
        g.manual_seed(seed)
        self.dev, self.nh, self.nkv, self.hd, self.page, self.cache = dev, nh, nkv, hd, page, cache
        self.q, self.n = list(q), [a + b for a, b in zip(q, past)]
        self.B, self.T = len(q), sum(q) + pad + lead
        per = max(1, max(-(-x // page) for x in self.n))
        need = [-(-x // page) for x in self.n]
        self.npages = sum(need) + extra
        order = torch.randperm(self.npages, generator=g).tolist()
        table = torch.full((self.B, per + wide), -1, dtype=torch.int32)
        self.pages, at = [], 0
        for b, m in enumerate(need):
            ids = order[at:at + m]
            at += m
            table[b, :m] = torch.tensor(ids, dtype=torch.int32)
            self.pages.append(ids)
        self.table = table.to(dev)[:, :per]
        starts = [lead]
        for x in q:
            starts.append(starts[-1] + x)
        self.starts = starts
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=dev)
        self.kv_len = torch.tensor(self.n, dtype=torch.int32, device=dev)
        shape = (self.npages, page + apart, nkv, hd)
        self.k_all = torch.full(shape, float("nan"), dtype=cache, device=dev)
        self.v_all = torch.full(shape, float("nan"), dtype=cache, device=dev)
        self.k, self.v = self.k_all[:, :page], self.v_all[:, :page]
        self.keys = [torch.randn((x, nkv, hd), generator=g).to(dev).to(cache) for x in self.n]
        self.vals = [(3 * torch.randn((x, nkv, hd), generator=g)).to(dev).to(cache) for x in self.n]
        self.width = (nh + 2 * nkv) * hd + nh
        self.rows = (2 * torch.randn((self.T, self.width + stray), generator=g)).to(BF16).to(dev)
        self.store()

    def store(self):
        """The keys and values into their slots."""
        for b in range(self.B):
            for i, pg in enumerate(self.pages[b]):
                part = slice(i * self.page, min((i + 1) * self.page, self.n[b]))
                m = part.stop - part.start
                self.k[pg, :m], self.v[pg, :m] = self.keys[b][part], self.vals[b][part]

    def view(self, pq, q_start=True):
        return pq.PagedKV(self.k, self.v, self.table, self.kv_len, self.q_start if q_start else None)

    @property
    def gate(self):
        return self.rows[:, self.width - self.nh:self.width]


def attend64(q, p, keys, vals, scale, win, sinks, gate=None, have=None):
    """Rows q [c][nh][hd] at positions p [c] over one sequence's keys [n][nkv][hd],
    in 64 bits: (out [c][nh][hd], the tolerance's parts). have [n]: keys whose page exists."""
    c, nh, hd = q.shape
    n, nkv = keys.shape[0], keys.shape[1]
    G = nh // nkv
    out = torch.zeros((c, nh, hd), dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    slack = torch.zeros((c, nh, 1), dtype=torch.float64, device=q.device)
    if n == 0:
        return out, size, slack
    j = torch.arange(n, device=q.device)
    see = j[None] <= p[:, None]
    if win:
        see &= (j[None] > p[:, None] - win) | (j < sinks)[None]
    if have is not None:
        see &= have[None]
    some = see.any(1)
    for h in range(nh):
        k, v = keys[:, h // G].double(), vals[:, h // G].double()
        qh = q[:, h].double()
        s = (scale * (qh @ k.t())).masked_fill(~see, -math.inf)
        s[~some] = 0.0
        w = torch.softmax(s, 1) * some[:, None]
        g = torch.sigmoid(gate[:, h].double())[:, None] if gate is not None else 1.0
        # a key that a row does not see is not in its sum, whatever its value is
        odd = ~torch.isfinite(v)
        o = w @ v.masked_fill(odd, 0.0)
        for at in torch.nonzero(odd.any(1)).flatten().tolist():
            part = w[:, at:at + 1] * v[at][None]
            o = o + torch.where(see[:, at:at + 1] & odd[at][None], part, torch.zeros_like(part))
        out[:, h] = o * g
        size[:, h] = w @ v.abs().masked_fill(odd, 0.0) * g
        big = (qh.abs() @ k.abs().nan_to_num(0.0).t()).masked_fill(~see, 0.0).amax(1, keepdim=True) * abs(scale)
        slack[:, h] = big * (hd + 8) * 2.0 ** -24 * 2
    return out, size, slack


def tolerance(out, size, slack, n, cache):
    """How far an output may be off: one bf16 rounding (half a step of its value);
    the weights' rounding to the cache's type (half a step each, of the summed
    sizes); fp32 scores (hd + 8 roundings of the products' summed sizes, in the
    exponent, twice: a weight and the sum it is divided by); fp32 sums of n keys
    in chains of at most an eighth of them; e^x, division and sigmoid, 16 steps."""
    half = torch.finfo(cache).eps / 2
    f32 = 2.0 ** -24
    return (torch.finfo(BF16).eps / 2) * out.abs() + size * (half + slack + (n / 8 + 64 + 16) * f32) + 1e-37


def want(bt, scale, win, sinks, rows=None, gate=True, q_start=True, have=None):
    """Every row of the batch: (out [T][nh][hd], tolerance), NaN where a row is no sequence's."""
    nh, hd = bt.nh, bt.hd
    rows = bt.rows if rows is None else rows
    T = rows.shape[0]
    out = torch.full((T, nh, hd), float("nan"), dtype=torch.float64, device=rows.device)
    tol = torch.zeros_like(out)
    for b in range(bt.B):
        r = slice(bt.starts[b], bt.starts[b + 1]) if q_start else slice(b, b + 1)
        c = r.stop - r.start
        if not c:
            continue
        p = bt.n[b] - c + torch.arange(c, device=rows.device)
        g = rows[r, bt.width - nh:bt.width] if gate else None
        o, size, slack = attend64(rows[r, :nh * hd].reshape(c, nh, hd), p, bt.keys[b], bt.vals[b], scale, win, sinks, g,
                                  have[b] if have is not None else None)
        out[r], tol[r] = o, tolerance(o, size, slack, bt.n[b], bt.cache)
    return out, tol


def check(got, out, tol):
    """got [T][nh * hd] bf16 against out within tol; NaN for NaN."""
    got = got.double().view(out.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    inf = torch.isinf(out)
    assert torch.equal(got[inf], out[inf])
    d = (got - out).abs()
    bad = (d > tol) & torch.isfinite(out)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first {torch.nonzero(bad)[0].tolist()}: " \
                          f"{float(got[bad][0])} for {float(out[bad][0])}, tolerance {float(tol[bad][0]):.3g}"
