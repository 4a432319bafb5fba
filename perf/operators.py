"""The paged-cache operators as cases that can be timed: the q/k head norm,
rotation and cache write of a ragged batch ("prep"), attention of one new token
a sequence ("decode") and of prompt rows ("prefill") over the pages.

Sequence b holds `past_b + q_b` positions, of which the last q_b are the rows of
this call; its pages lie anywhere in a pool [pages][page][kv heads][head_dim].
Rows are those of the attention layer's input projection, [q | k | v | gate].
Head shapes are those of the two backbones the library is configured for (32 q /
8 kv heads of 64, 16 / 4 of 128, windows of 256) and other groups it takes.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-5
BF16 = torch.bfloat16
CACHE = {"f16": torch.float16, "bf16": torch.bfloat16}


def _pq():
    """The library's Python package (where `own` is true)."""
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "pulsar-asm_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import pulsar_amd
    return pulsar_amd


def _case(name, op, B, hd, cache, page, q=1, q_lo=1, past=0, past_lo=0, nh=None, nkv=None, rot=None, win=0, sinks=0):
    d = dict(op=op, B=B, nh=nh or (32 if hd == 64 else 16), nkv=nkv or (8 if hd == 64 else 4), hd=hd,
             rot=rot or (32 if hd == 64 else 64), cache=cache, page=page, q=q, q_lo=q_lo, past=past, past_lo=past_lo,
             win=win, sinks=sinks)
    return dict(name=name, **d) if name else d


def listed():
    return [
        # one request's next token: the launch and its latency count
        _case("prep_token", "prep", 1, 64, "f16", 16, past=299, past_lo=299),
        # a decode step of many requests
        _case("prep_batch", "prep", 128, 128, "bf16", 32, past=1500, past_lo=100),
        # a step of prompts of many lengths, some behind a past
        _case("prep_prompts", "prep", 8, 64, "f16", 64, q=4096, q_lo=77, past=1500),
        # one request's next token, a few hundred keys: latency
        _case("decode_short", "decode", 1, 64, "f16", 16, past=299, past_lo=299),
        # one request far into a long document: the work has to be split over the keys
        _case("decode_long", "decode", 1, 128, "bf16", 64, past=131071, past_lo=131071),
        # a decode step of many requests of many lengths
        _case("decode_batch", "decode", 64, 64, "f16", 32, past=8191, past_lo=100),
        # the same in a sliding-window layer whose first tokens stay visible
        _case("decode_window", "decode", 256, 128, "bf16", 16, past=16383, past_lo=1, win=256, sinks=4, rot=128),
        # the end of a prompt in a sliding-window layer: a short ragged chunk
        _case("prefill_short", "prefill", 1, 128, "bf16", 16, q=203, q_lo=203, past=300, past_lo=300, win=256, sinks=4),
        # prompts of many lengths in one step, among them single tokens
        _case("prefill_prompts", "prefill", 8, 64, "f16", 64, q=2048, q_lo=1, past=512),
        # a chunk of a prompt far behind its start: few rows, many keys
        _case("prefill_far", "prefill", 1, 128, "bf16", 64, q=512, q_lo=512, past=32000, past_lo=32000),
        # a whole long prompt in a sliding-window layer with sinks
        _case("prefill_window", "prefill", 1, 128, "bf16", 64, q=16384, q_lo=16384, win=256, sinks=4, rot=128),
        # a whole long prompt, every key: the largest
        _case("prefill_long", "prefill", 1, 128, "bf16", 64, q=16384, q_lo=16384),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 64), (32, 8, 64), (16, 4, 128), (16, 4, 128), (8, 8, 64), (16, 2, 64), (8, 1, 128), (16, 8, 128)]


def draw(rng):
    op = rng.choice(["prep", "decode", "prefill"])
    nh, nkv, hd = rng.choice(HEADS)
    kw = dict(nh=nh, nkv=nkv, rot=rng.choice([hd // 2, hd]), page=rng.choice([16, 32, 64, 128, 256]))
    cache = rng.choice(["f16", "bf16"])
    if op == "prep":
        B = _log(rng, 1, 256)
        q = rng.choice([1, _log(rng, 2, max(2, 16384 // B))])
        past = rng.choice([0, _log(rng, 1, 8192)])
        return _case(None, op, B, hd, cache, q=q, q_lo=1, past=past, past_lo=past // 3, **kw)
    win, sinks = rng.choice([(0, 0), (0, 0), (256, 4), (_log(rng, 16, 4096), rng.choice([0, 1, 4, 33]))])
    kw.update(win=win, sinks=sinks)
    if op == "decode":
        B = _log(rng, 1, 256)
        past = _log(rng, 16, min(131071, 300000 // B))
        return _case(None, op, B, hd, cache, past=past, past_lo=rng.choice([past, past // 9]), **kw)
    B = rng.choice([1, _log(rng, 1, 16)])
    q = _log(rng, 2, 8192 // B)
    past = rng.choice([0, _log(rng, 1, 16384 // B)])
    return _case(None, op, B, hd, cache, q=q, q_lo=rng.choice([q, 1]), past=past, past_lo=rng.choice([past, 0]), **kw)


def _spread(B, lo, hi, step):
    """B whole numbers spread over lo .. hi; the first is hi."""
    return [hi - int((hi - lo + 1) * ((b * step) % 1.0)) for b in range(B)]


def _lengths(c):
    q = _spread(c["B"], c["q_lo"], c["q"], 0.6180339887498949)
    past = _spread(c["B"], c["past_lo"], c["past"], 0.7548776662466927)
    return q, past


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    B, nh, nkv, hd, page = c["B"], c["nh"], c["nkv"], c["hd"], c["page"]
    q, past = _lengths(c)
    n = [a + b for a, b in zip(q, past)]
    T, most = sum(q), max(n)
    per = -(-most // page)
    need = sum(-(-x // page) for x in n)
    npages = need + 8                                   # the pool has pages that no sequence holds
    order = torch.randperm(npages, device=DEV, generator=g).to(torch.int32)
    have = torch.tensor([-(-x // page) for x in n], device=DEV)
    first = torch.cumsum(have, 0) - have
    at = torch.arange(per, device=DEV)
    table = torch.where(at[None] < have[:, None], order[(first[:, None] + at[None]).clamp(max=npages - 1)], 0)
    starts = [0]
    for x in q:
        starts.append(starts[-1] + x)
    qn = torch.tensor(q, device=DEV)
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), qn, output_size=T)
    start = torch.tensor(starts, device=DEV, dtype=torch.int32)
    dt = CACHE[c["cache"]]
    # a pool that is read holds keys and values, one that is only written is as it was allocated
    pool = torch.zeros if c["op"] == "prep" else lambda *a, **kw: torch.randn(*a, generator=g, **kw)
    s = dict(case=c, T=T, most=most, table=table.to(torch.int32).contiguous(), start=start,
             n=torch.tensor(n, device=DEV, dtype=torch.int32), seq=seq,
             nth=torch.arange(T, device=DEV) - start[:-1].long()[seq],
             k=pool((npages, page, nkv, hd), device=DEV).to(dt),
             v=pool((npages, page, nkv, hd), device=DEV).to(dt))
    width = (nh + 2 * nkv) * hd + nh                    # [q | k | v | gate]
    if c["op"] == "prep":
        # as the projection leaves them: neither centred nor of one size from head to head
        size = torch.exp(torch.randn((1, width), device=DEV, generator=g))
        s["rows"] = (torch.randn((T, width), device=DEV, generator=g) * size).to(BF16)
        s["q_norm"] = 1 + 0.1 * torch.randn(hd, device=DEV, generator=g)
        s["k_norm"] = 1 + 0.1 * torch.randn(hd, device=DEV, generator=g)
        # [position][rot / 2][cos, sin]: the angles in 64 bits, as the positions go far
        half = c["rot"] // 2
        inv = 1e6 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
        ang = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * inv
        s["cs"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        s["q_out"] = torch.empty((T, nh * hd), device=DEV, dtype=BF16)
    else:
        # normed queries meet normed keys: scores of a few units after the scale
        s["rows"] = torch.randn((T, width), device=DEV, generator=g).to(BF16)
        s["rows"][:, :nh * hd] *= 2
        s["out"] = torch.empty((T, nh * hd), device=DEV, dtype=BF16)
    return s


# ------------------------------------------------------------- plain forms
def _slots(s, j):
    """The pool rows of positions j of every sequence: [B][len(j)]."""
    page = s["case"]["page"]
    return s["table"].long()[:, j // page] * page + j % page


def _prep(s):
    c = s["case"]
    nh, nkv, hd, half = c["nh"], c["nkv"], c["hd"], c["rot"] // 2
    pos = s["n"].long()[s["seq"]] - (s["start"][1:] - s["start"][:-1]).long()[s["seq"]] + s["nth"]
    x = s["rows"][:, :(nh + 2 * nkv) * hd].float().view(s["T"], nh + 2 * nkv, hd)
    qk, v = x[:, :nh + nkv], x[:, nh + nkv:]
    y = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    y = torch.cat([y[:, :nh] * s["q_norm"], y[:, nh:] * s["k_norm"]], 1)
    co, si = s["cs"][pos][:, None, :, 0], s["cs"][pos][:, None, :, 1]
    a, b = y[..., :half], y[..., hd // 2:hd // 2 + half]
    y = torch.cat([a * co - b * si, y[..., half:hd // 2], b * co + a * si, y[..., hd // 2 + half:]], -1)
    at = s["table"].long()[s["seq"], pos // c["page"]] * c["page"] + pos % c["page"]
    s["k"].view(-1, nkv, hd)[at] = y[:, nh:].to(s["k"].dtype)
    s["v"].view(-1, nkv, hd)[at] = v.to(s["v"].dtype)
    return dict(q=y[:, :nh].reshape(s["T"], nh * hd).to(BF16), k=s["k"], v=s["v"])


def _attend(s):
    c = s["case"]
    B, nh, nkv, hd, Q, L = c["B"], c["nh"], c["nkv"], c["hd"], c["q"], s["most"]
    G = nh // nkv
    start, count, n = s["start"][:-1].long(), (s["start"][1:] - s["start"][:-1]).long(), s["n"].long()
    i, j = torch.arange(Q, device=DEV), torch.arange(L, device=DEV)
    pos = (n - count)[:, None] + i                                                     # [B][Q]
    q = s["rows"][(start[:, None] + i).clamp(max=s["T"] - 1), :nh * hd].float()
    q = q.view(B, Q, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, Q * G, hd)
    at = _slots(s, j)
    k = s["k"].view(-1, nkv, hd)[at].float().permute(0, 2, 3, 1)                       # [B][nkv][hd][L]
    v = s["v"].view(-1, nkv, hd)[at].float().masked_fill_((j >= n[:, None])[..., None, None], 0.0).permute(0, 2, 1, 3)
    sc = torch.matmul(q, k.contiguous()).view(B, nkv, Q, G, L)
    hide = j > pos[..., None]
    if c["win"]:
        hide = hide | ((j <= pos[..., None] - c["win"]) & (j >= c["sinks"]))
    sc.mul_(hd ** -0.5).masked_fill_(hide[:, None, :, None, :], -math.inf)
    sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(sc.view(B, nkv, Q * G, L), v.contiguous()).view(B, nkv, Q, G, hd) / sc.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, Q, nh, hd)[s["seq"], s["nth"]]
    gate = s["rows"][:, -nh:].float()
    return (o / (1 + torch.exp(-gate))[..., None]).view(s["T"], nh * hd).to(BF16)


def _view(s):
    """The batch's view of the pools, as a program keeps it from step to step."""
    if "kv" not in s:
        s["kv"] = _pq().PagedKV(s["k"], s["v"], s["table"], s["n"], s["start"] if s["case"]["op"] != "decode" else None)
    return s["kv"]


def run(state):
    s, c = state, state["case"]
    if not own:
        return _prep(s) if c["op"] == "prep" else _attend(s)
    pq, kv = _pq(), _view(s)
    if c["op"] == "prep":
        pq.paged_qk_prep(kv, s["rows"], s["q_norm"], s["k_norm"], s["cs"], c["nh"], c["rot"], eps=EPS, out=s["q_out"])
        return dict(q=s["q_out"], k=s["k"], v=s["v"])
    call = pq.paged_attn_decode if c["op"] == "decode" else pq.paged_attn_prefill
    return call(kv, s["rows"], c["nh"], c["hd"] ** -0.5, gate=s["rows"][:, -c["nh"]:], win=c["win"], sinks=c["sinks"],
                max_kv=s["most"], out=s["out"])


# ------------------------------------------------------------------- floors
def _pairs(c):
    """Visible (row, key) pairs of one head, and keys that some row of their sequence sees."""
    win, sinks = c["win"] or 1 << 40, c["sinks"]
    seqs = list(zip(*_lengths(c)))
    # a row at p sees the keys of its window, lo .. p, and the sinks before them
    pairs = sum(p + 1 - max(0, p + 1 - win) + min(sinks, max(0, p + 1 - win)) for q, past in seqs
                for p in range(past, past + q))
    keys = sum(q + past - max(0, past + 1 - win) + min(sinks, max(0, past + 1 - win)) for q, past in seqs)
    return pairs, keys


def work(case):
    c = case
    T = sum(_lengths(c)[0])
    row = 2 * c["nh"] * c["hd"]
    kv = 2 * 2 * c["nkv"] * c["hd"]
    if c["op"] == "prep":
        # each row read and written once, a row of cosines and sines for each position
        heads = c["nh"] + c["nkv"]
        at = set(p for q, past in zip(*_lengths(c)) for p in range(past, past + q))
        return dict(bytes=T * 2 * (row + kv) + len(at) * 4 * c["rot"], flops=T * heads * (4 * c["hd"] + 3 * c["rot"]))
    pairs, keys = _pairs(c)
    return dict(bytes=T * (2 * row + 2 * c["nh"]) + keys * kv, flops=4 * c["hd"] * c["nh"] * pairs)


# ------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    G = nh // nkv
    rows = s["rows"].double()
    table, starts, lens = s["table"].tolist(), s["start"].tolist(), s["n"].tolist()
    kp, vp = s["k"].double(), s["v"].double()
    if c["op"] == "prep":
        out = torch.zeros((s["T"], nh * hd), device=DEV, dtype=torch.float64)
        half = c["rot"] // 2
        for b in range(c["B"]):
            r = torch.arange(starts[b], starts[b + 1], device=DEV)
            p = lens[b] - len(r) + torch.arange(len(r), device=DEV)
            pg, sl = s["table"][b].long()[p // page], p % page
            cos, sin = s["cs"].double()[p, :, 0], s["cs"].double()[p, :, 1]
            for h in range(nh + nkv):
                x = rows[r, h * hd:(h + 1) * hd]
                w = (s["q_norm"] if h < nh else s["k_norm"]).double()
                y = w * x * (x.pow(2).sum(1, keepdim=True) / hd + EPS).rsqrt()
                lo, hi = y[:, :half].clone(), y[:, hd // 2:hd // 2 + half].clone()
                y[:, :half] = lo * cos - hi * sin
                y[:, hd // 2:hd // 2 + half] = hi * cos + lo * sin
                if h < nh:
                    out[r, h * hd:(h + 1) * hd] = y
                else:
                    kp[pg, sl, h - nh] = y
            vp[pg, sl] = rows[r, (nh + nkv) * hd:(nh + 2 * nkv) * hd].view(-1, nkv, hd)
        return dict(q=out, k=kp, v=vp)
    out = torch.zeros((s["T"], nh * hd), device=DEV, dtype=torch.float64)
    for b in range(c["B"]):
        n, r0, r1 = lens[b], starts[b], starts[b + 1]
        ids = torch.tensor(table[b][:-(-n // page)], device=DEV)
        keys, vals = kp[ids].reshape(-1, nkv, hd)[:n], vp[ids].reshape(-1, nkv, hd)[:n]
        for a in range(r0, r1, 4096):                    # 4096 rows at a time, their scores in 64 bits
            e = min(a + 4096, r1)
            p = torch.arange(n - (r1 - a), n - (r1 - e), device=DEV)[:, None]
            j = torch.arange(n, device=DEV)[None]
            see = j <= p
            if c["win"]:
                see &= (p - j < c["win"]) | (j < c["sinks"])
            for h in range(nh):
                z = rows[a:e, h * hd:(h + 1) * hd] @ keys[:, h // G].t() / math.sqrt(hd)
                w = torch.softmax(z.masked_fill(~see, -math.inf), 1)
                gate = torch.sigmoid(rows[a:e, -nh + h])[:, None]
                out[a:e, h * hd:(h + 1) * hd] = (w @ vals[:, h // G]) * gate
    return out
