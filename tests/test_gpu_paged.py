"""GPU tests of the paged cache: the q/k norm + RoPE + cache write of a ragged
batch and the two attentions over the pages, against 64-bit statements."""
import math

import pytest
import torch

import paged_cases as pc

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
EPS = 1e-5


# ------------------------------------------------------------- norm, RoPE, cache
def _rope(dev, rows, rot, g):
    ang = torch.rand((rows, rot // 2), generator=g) * 6.28
    return torch.stack([ang.cos(), ang.sin()], -1).to(dev).contiguous()


def _prep64(bt, rows, qn, kn, cs, rot, b, have_rope):
    """Sequence b's rows: (q, k, v) in 64 bits, the rotation's operands' size, positions, which rows take part."""
    nh, nkv, hd = bt.nh, bt.nkv, bt.hd
    r = slice(bt.starts[b], bt.starts[b + 1])
    c = r.stop - r.start
    x = rows[r, :(nh + 2 * nkv) * hd].double().view(c, nh + 2 * nkv, hd)
    p = bt.n[b] - c + torch.arange(c, device=rows.device)
    on = (p >= 0) & (p < have_rope)
    qk = x[:, :nh + nkv]
    y = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    y = torch.cat([y[:, :nh] * qn.double(), y[:, nh:] * kn.double()], 1)
    half = rot // 2
    co, si = (cs.double()[p.clamp(0, have_rope - 1)][:, None, :, i] for i in (0, 1))
    z, size = y.clone(), y.abs()
    a, bb = y[..., :half], y[..., hd // 2:hd // 2 + half]
    z[..., :half], z[..., hd // 2:hd // 2 + half] = a * co - bb * si, bb * co + a * si
    size[..., :half] = size[..., hd // 2:hd // 2 + half] = a.abs() + bb.abs()
    return z[:, :nh], z[:, nh:], x[:, nh + nkv:], size[:, :nh], size[:, nh:], p, on


def _near(got, want, size, dtype, what):
    """One rounding to the type (half a step; fp16 below its normal range: half of
    2^-24), and fp32 up to it: hd / 2 + 16 roundings at most of the operands' size."""
    tol = torch.finfo(dtype).eps / 2 * want.abs() + size * (80 * 2.0 ** -24) + (2.0 ** -25 if dtype == F16 else 1e-38)
    d = (got.double() - want).abs()
    assert (d <= tol).all(), f"{what}: {float((d - tol).max())} over at {torch.nonzero(d > tol)[0].tolist()}"


@pytest.mark.parametrize("nh,nkv,hd,rot,cache,page,q,past,kw", [
    (32, 8, 64, 32, F16, 16, [1], [0], {}),
    (32, 8, 64, 32, F16, 16, [1, 0, 17, 5], [299, 3, 40, 0], dict(pad=3, lead=2)),
    (16, 4, 128, 64, BF16, 32, [33, 1, 64], [0, 77, 31], dict(stray=3)),
    (16, 4, 128, 128, F16, 8, [9, 2], [7, 100], dict(apart=8, wide=2)),
    (8, 8, 64, 64, BF16, 64, [130], [5], {}),
    (8, 1, 128, 0, BF16, 16, [3, 3], [0, 0], {}),
    (3, 1, 64, 22, F16, 16, [4, 1], [2, 9], {}),
    (32, 8, 64, 32, F16, 256, [1] * 70, list(range(70)), {}),
    (16, 16, 128, 64, BF16, 16, [300, 211], [0, 1], dict(pad=1))])
@pytest.mark.parametrize("inplace", [False, True])
def test_prep(pq, dev, nh, nkv, hd, rot, cache, page, q, past, kw, inplace):
    print(f"prep {nh}/{nkv}x{hd} rot={rot} {cache} page={page} q={q[:4]} {kw} {inplace}", flush=True)
    bt = pc.Batch(dev, q, past, nh, nkv, hd, page, cache, seed=sum(q) + hd, **kw)
    g = torch.Generator()
    g.manual_seed(1)
    limit = max(bt.n) - (1 if max(bt.n) > 2 else 0)      # the last position has no row in the table: left out
    cs = _rope(dev, limit, rot, g)
    qn, kn = (1 + 0.2 * torch.randn(hd, generator=g)).to(dev), (1 + 0.2 * torch.randn(hd, generator=g)).to(dev)
    k0, v0, rows = bt.k_all.clone(), bt.v_all.clone(), bt.rows.clone()
    out = bt.rows if inplace else torch.full((bt.T, nh * hd + 5), 7.0, dtype=BF16, device=dev)
    before = out.clone()
    pq.paged_qk_prep(bt.view(pq), bt.rows, qn, kn, cs, nh, rot, eps=EPS, out=out)
    for b in range(bt.B):
        qq, kk, vv, qs, ks, p, on = _prep64(bt, rows, qn, kn, cs, rot, b, limit)
        r = torch.arange(bt.starts[b], bt.starts[b + 1], device=dev)
        _near(out[r[on], :nh * hd].view(-1, nh, hd), qq[on], qs[on], BF16, "q")
        before[r[on], :nh * hd] = out[r[on], :nh * hd]
        for i in torch.nonzero(on).flatten().tolist():
            pg, s = bt.pages[b][int(p[i]) // page], int(p[i]) % page
            _near(bt.k[pg, s], kk[i], ks[i], cache, "k")
            _near(bt.v[pg, s], vv[i], torch.zeros_like(vv[i]), cache, "v")
            k0[pg, s], v0[pg, s] = bt.k[pg, s], bt.v[pg, s]
    # nothing else was written: not other slots, rows or columns
    assert torch.equal(bt.k_all.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(bt.v_all.view(torch.int16), v0.view(torch.int16))
    assert torch.equal(out.view(torch.int16), before.view(torch.int16))


def test_prep_bad_pages_and_lengths(pq, dev):
    """Pages outside the pool, lengths past the table and below the rows: such positions are not written."""
    bt = pc.Batch(dev, [4, 4, 4], [30, 0, 10], 32, 8, 64, 16, F16, seed=3)
    cs = torch.zeros((64, 16, 2), device=dev)
    cs[..., 0] = 1
    one = torch.ones(64, device=dev)
    table = bt.table.clone()
    table[0, 2], table[2, 0] = bt.npages, -5
    bt.table = table
    bt.kv_len[1] = 2                                     # its first two rows lie at -2, -1
    kv = bt.view(pq)
    k0 = bt.k_all.clone()
    out = torch.full((bt.T, 2048), 7.0, dtype=BF16, device=dev)
    pq.paged_qk_prep(kv, bt.rows, one, one, cs, 32, 32, out=out)
    changed = (bt.k_all.view(torch.int16) != k0.view(torch.int16)).flatten(1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {bt.pages[0][1], bt.pages[1][0], bt.pages[2][0]} and bt.pages[1][0] in changed
    assert (out[4:6] == 7).all() and not (out[6:8] == 7).any() and not (out[8:] == 7).any()
    k0 = bt.k_all.clone()
    bt.kv_len.fill_(60000)                               # past every page of the table, and past the RoPE table
    pq.paged_qk_prep(kv, bt.rows, one, one, torch.zeros((60000, 16, 2), device=dev), 32, 32, out=out)
    assert torch.equal(bt.k_all.view(torch.int16), k0.view(torch.int16))


# ---------------------------------------------------------------- one new token
DECODE = [
    # nh, nkv, hd, cache, page, past (a list: one row behind each), win, sinks, kw
    (32, 8, 64, F16, 16, [0], 0, 0, {}),
    (32, 8, 64, F16, 16, [299, 0, 15, 16, 17, 31, 32, 1000], 0, 0, {}),
    (16, 4, 128, BF16, 64, [2000, 1, 63, 64, 511, 512, 513], 0, 0, dict(wide=3, apart=16)),
    (16, 4, 128, F16, 8, [700, 7, 8, 9], 0, 0, {}),
    (8, 8, 64, BF16, 32, [100, 333], 0, 0, dict(stray=1)),
    (16, 8, 64, F16, 128, [1027], 0, 0, {}),
    (6, 2, 128, BF16, 16, [90, 260], 0, 0, {}),
    (10, 2, 64, F16, 16, [90, 260], 0, 0, {}),
    (8, 1, 128, F16, 256, [5000, 3], 0, 0, {}),
    (16, 1, 64, BF16, 32, [1500, 31], 0, 0, {}),
    (13, 1, 128, BF16, 16, [200], 0, 0, {}),
    (32, 8, 64, F16, 16, [3000, 10, 255, 256, 257, 259, 260, 300], 256, 4, {}),
    (16, 4, 128, BF16, 32, [4000, 100, 33, 40], 1, 33, {}),
    (16, 4, 128, BF16, 16, [5000, 1, 129], 100, 0, {}),
    (16, 4, 128, F16, 64, [700, 20], 31, 1000, {}),
    (16, 4, 128, BF16, 64, [40000], 0, 0, {}),
    (32, 8, 64, F16, 16, [20000, 1, 600], 8192, 65, {}),
]


@pytest.mark.parametrize("nh,nkv,hd,cache,page,past,win,sinks,kw", DECODE)
def test_decode(pq, dev, nh, nkv, hd, cache, page, past, win, sinks, kw):
    print(f"decode {nh}/{nkv}x{hd} {cache} page={page} past={past[:4]} win={win} sinks={sinks} {kw}", flush=True)
    bt = pc.Batch(dev, [1] * len(past), past, nh, nkv, hd, page, cache, seed=past[0] + win, **kw)
    scale = 1 / math.sqrt(hd)
    out, tol = pc.want(bt, scale, win, sinks)
    kv = bt.view(pq, q_start=False)
    got = pq.paged_attn_decode(kv, bt.rows, nh, scale, gate=bt.gate, win=win, sinks=sinks, max_kv=max(bt.n))
    pc.check(got, out, tol)
    # no gate; a hint that is far off; both outputs at once, into strided rows: the Q8_0 form is that of out
    out, tol = pc.want(bt, scale, win, sinks, gate=False)
    wide = torch.full((bt.B, nh * hd + 3), 5.0, dtype=BF16, device=dev)
    qx, dx = torch.empty((bt.B, nh * hd), dtype=torch.int8, device=dev), torch.empty((bt.B, nh * hd // 32), device=dev)
    for hint in (1, None):
        pq.paged_attn_decode(kv, bt.rows, nh, scale, win=win, sinks=sinks, max_kv=hint, out=wide, qx=qx, dx=dx)
        got = wide[:, :nh * hd].contiguous()
        pc.check(got, out, tol)
        assert (wide[:, nh * hd:] == 5).all()
        rx, rd = pq.q8_quant(got)
        assert torch.equal(qx, rx) and torch.equal(dx, rd)


def test_decode_empty_rows_and_bad_pages(pq, dev):
    """Lengths of zero and below, pages that do not exist, a window that lies on such pages, lengths past the table."""
    for hd, cache, nh, nkv in ((64, F16, 32, 8), (128, BF16, 16, 4)):
        bt = pc.Batch(dev, [1] * 6, [99, 40, 700, 0, 63, 500], nh, nkv, hd, 16, cache, seed=5)
        table, have = bt.table.clone(), [torch.ones(n, dtype=torch.bool, device=dev) for n in bt.n]
        for b, i, bad in ((0, 2, -1), (1, 0, bt.npages), (2, 20, -7), (2, 43, 1 << 30), (5, 0, -1), (5, 31, -1)):
            table[b, i] = bad
            have[b][i * 16:(i + 1) * 16] = False
        bt.table = table
        bt.n[3] = 0
        bt.keys[3], bt.vals[3] = bt.keys[3][:0], bt.vals[3][:0]
        have[3] = have[3][:0]
        bt.kv_len[3] = 0
        for win, sinks in ((0, 0), (20, 4), (4, 3), (300, 40)):
            want, tol = pc.want(bt, 0.1, win, sinks, q_start=False, have=have)
            kv = bt.view(pq, q_start=False)
            got = pq.paged_attn_decode(kv, bt.rows, nh, 0.1, gate=bt.gate, win=win, sinks=sinks)
            pc.check(got, want, tol)
            assert (got[3] == 0).all()
            if win == 4:
                assert (got[5] == 0).all()               # the window and the sinks are on pages that do not exist
        bt.kv_len[3] = -3
        assert (pq.paged_attn_decode(bt.view(pq, q_start=False), bt.rows, nh, 0.1)[3] == 0).all()
        # 60 positions past the table's end: the keys that the table holds are seen
        bt = pc.Batch(dev, [1], [112], nh, nkv, hd, 16, cache, seed=6)
        full, tol = pc.want(bt, 0.1, 0, 0)
        kv = bt.view(pq, q_start=False)
        bt.kv_len[0] = bt.n[0] + 60
        k112 = bt.k.clone()
        lastpg = bt.pages[0][-1]
        bt.k[lastpg] = 0
        bt.v[lastpg] = 0
        bt.k[lastpg, :1], bt.v[lastpg, :1] = k112[lastpg, :1], 0
        n = kv.capacity
        keys = torch.stack([bt.k[bt.pages[0][j // 16], j % 16] for j in range(n)])
        vals = torch.stack([bt.v[bt.pages[0][j // 16], j % 16] for j in range(n)])
        o, size, slack = pc.attend64(bt.rows[:, :nh * hd].view(1, nh, hd), torch.tensor([n + 50], device=dev), keys, vals,
                                     0.1, 0, 0)
        pc.check(pq.paged_attn_decode(kv, bt.rows, nh, 0.1), o, pc.tolerance(o, size, slack, n, cache))


@pytest.mark.parametrize("cache", [F16, BF16])
def test_decode_values_at_the_edges(pq, dev, cache):
    """Scores that fill the type's range, keys and values that are infinite or NaN where the row sees them and
    where it does not, queries larger than fp16 holds and smaller than its normal range."""
    nh, nkv, hd = 16, 4, 128
    bt = pc.Batch(dev, [1] * 5, [200, 300, 130, 64, 500], nh, nkv, hd, 16, cache, seed=9)
    bt.rows[0, :nh * hd] *= 2.0 ** 18                    # far over 65504
    bt.keys[0] *= 2.0 ** -18 if cache == BF16 else 2.0 ** -10
    bt.rows[1, :nh * hd] *= 2.0 ** -30
    bt.keys[2][:] = bt.keys[2][:1]                       # every score the same
    bt.vals[3][5, 1, 7] = float("inf")                   # seen
    bt.vals[3][9, 2, 3] = float("nan")
    bt.keys[4][:100] = float("nan")                      # outside the window
    bt.vals[4][:100] = float("inf")
    bt.store()
    scale = 2.0 ** -8 if cache == F16 else 0.1
    want, tol = pc.want(bt, scale, 256, 0)
    got = pq.paged_attn_decode(bt.view(pq, q_start=False), bt.rows, nh, scale, gate=bt.gate, win=256)
    pc.check(got, want, tol)
    assert not torch.isnan(got[4]).any()


def test_decode_offsets_past_32_bits(pq, dev):
    """A pool of more than 2^31 elements, its pages in use at both ends."""
    nh, nkv, hd, page = 16, 4, 128, 64
    npages = (1 << 31) // (page * nkv * hd) + 40
    bt = pc.Batch(dev, [1, 1], [500, 130], nh, nkv, hd, page, BF16, seed=11)
    big_k = torch.zeros((npages, page, nkv, hd), dtype=BF16, device=dev)
    big_v = torch.zeros_like(big_k)
    table = bt.table.clone()
    for b in range(2):
        for i, pg in enumerate(bt.pages[b]):
            new = npages - 1 - pg if i % 2 else pg
            big_k[new], big_v[new] = bt.k[pg], bt.v[pg]
            table[b, i] = new
    want, tol = pc.want(bt, 0.09, 0, 0)
    kv = pq.PagedKV(big_k, big_v, table, bt.kv_len, bt.q_start)
    pc.check(pq.paged_attn_decode(kv, bt.rows, nh, 0.09, gate=bt.gate), want, tol)
    pc.check(pq.paged_attn_prefill(kv, bt.rows, nh, 0.09, gate=bt.gate), want, tol)
    cs = torch.zeros((600, 32, 2), device=dev)
    cs[..., 0] = 1
    one = torch.ones(hd, device=dev)
    pq.paged_qk_prep(kv, bt.rows, one, one, cs, nh, 64)
    v = bt.rows[0, (nh + nkv) * hd:(nh + 2 * nkv) * hd].view(nkv, hd)
    assert torch.equal(big_v[int(table[0, 500 // page]), 500 % page], v)


def test_decode_many_sequences(pq, dev):
    """More sequences than the split's threads, lengths from none to long, both ways of laying the call out."""
    past = [(37 * i) % 190 for i in range(300)]
    past[123], past[299] = 1700, 2500
    for nh, nkv, hd, cache in ((8, 8, 64, F16), (4, 1, 128, BF16)):
        bt = pc.Batch(dev, [1] * 300, past, nh, nkv, hd, 16, cache, seed=13)
        for win, sinks in ((0, 0), (64, 2)):
            want, tol = pc.want(bt, 0.1, win, sinks)
            for hint in (64, None):
                print(f"decode 300 {nh}/{nkv}x{hd} win={win} hint={hint}", flush=True)
                pc.check(pq.paged_attn_decode(bt.view(pq, False), bt.rows, nh, 0.1, gate=bt.gate, win=win, sinks=sinks,
                                              max_kv=hint), want, tol)


# ------------------------------------------------------------------ prompt rows
PREFILL = [
    (32, 8, 64, F16, 16, [1], [0], 0, 0, {}),
    (32, 8, 64, F16, 16, [33, 0, 1, 130, 64], [0, 5, 99, 17, 0], 0, 0, dict(pad=4, lead=3)),
    (16, 4, 128, BF16, 64, [203], [300], 256, 4, {}),
    (16, 4, 128, BF16, 64, [513, 2], [0, 700], 0, 0, dict(wide=2, apart=8)),
    (16, 4, 128, F16, 8, [100, 31], [1, 64], 0, 0, dict(stray=3)),
    (8, 8, 64, BF16, 32, [257], [0], 0, 0, {}),
    (8, 8, 64, F16, 32, [300, 1, 5], [700, 1, 0], 40, 0, {}),
    (16, 8, 128, BF16, 128, [129, 128, 127], [0, 1, 2], 0, 0, {}),
    (6, 2, 128, F16, 16, [77, 90], [13, 0], 0, 0, {}),
    (10, 2, 64, BF16, 16, [77, 90], [13, 0], 19, 3, {}),
    (8, 1, 128, BF16, 256, [70], [500], 0, 0, {}),
    (16, 1, 64, F16, 16, [40, 9], [0, 1200], 128, 7, {}),
    (13, 1, 64, F16, 16, [65], [3], 0, 0, {}),
    (32, 8, 64, F16, 16, [700], [0], 1, 0, {}),
    (16, 4, 128, BF16, 16, [600], [100], 64, 100, {}),
    (16, 4, 128, BF16, 64, [40], [9000], 0, 0, {}),
    (32, 8, 64, F16, 32, [5, 3], [6000, 20], 1024, 33, {}),
    (16, 4, 128, F16, 64, [1] * 40 + [90], list(range(0, 1200, 30)) + [0], 0, 0, {}),
]


@pytest.mark.parametrize("nh,nkv,hd,cache,page,q,past,win,sinks,kw", PREFILL)
def test_prefill(pq, dev, nh, nkv, hd, cache, page, q, past, win, sinks, kw):
    print(f"prefill {nh}/{nkv}x{hd} {cache} page={page} q={q[:4]} past={past[:4]} win={win} sinks={sinks} {kw}", flush=True)
    bt = pc.Batch(dev, q, past, nh, nkv, hd, page, cache, seed=q[0] + past[0] + win, **kw)
    scale = 1 / math.sqrt(hd)
    want, tol = pc.want(bt, scale, win, sinks)
    mine = ~torch.isnan(want).any(-1).any(-1)
    kv = bt.view(pq)
    out = torch.full((bt.T, nh * hd + 1), 5.0, dtype=BF16, device=dev)
    qx = torch.full((bt.T, nh * hd), 99, dtype=torch.int8, device=dev)
    dx = torch.full((bt.T, nh * hd // 32), 99.0, device=dev)
    for hint in (max(bt.n), 1, None):
        pq.paged_attn_prefill(kv, bt.rows, nh, scale, gate=bt.gate, win=win, sinks=sinks, max_kv=hint, out=out, qx=qx, dx=dx)
        got = out[:, :nh * hd].contiguous()
        pc.check(got[mine], want[mine], tol[mine])
        assert (out[:, nh * hd:] == 5).all() and (out[~mine] == 5).all()
        assert (qx[~mine] == 99).all() and (dx[~mine] == 99).all()
        rx, rd = pq.q8_quant(got)
        assert torch.equal(qx[mine], rx[mine]) and torch.equal(dx[mine], rd[mine])
    want, tol = pc.want(bt, scale, win, sinks, gate=False)
    got = pq.paged_attn_prefill(kv, bt.rows, nh, scale, win=win, sinks=sinks)
    pc.check(got[mine], want[mine], tol[mine])


@pytest.mark.parametrize("cache,nh,nkv,hd", [(F16, 32, 8, 64), (BF16, 16, 4, 128), (F16, 8, 8, 128), (BF16, 16, 1, 64)])
def test_prefill_values_that_some_rows_see(pq, dev, cache, nh, nkv, hd):
    """Infinite and NaN values and keys at positions that the chunk's later rows see and its earlier ones do not,
    and that have left the window of the last ones."""
    bt = pc.Batch(dev, [150, 90], [70, 0], nh, nkv, hd, 16, cache, seed=21)
    bt.vals[0][100, 0, 3] = float("inf")
    bt.vals[0][101, 0, hd - 1] = float("nan")
    bt.keys[0][140, nkv - 1, 5] = float("nan")
    bt.vals[0][140, nkv - 1] = float("nan")
    bt.vals[1][40, 0, 0] = -float("inf")
    bt.keys[1][70] = float("nan")
    bt.vals[0][2, 0, 9] = float("inf")                   # among the sinks
    bt.store()
    for win, sinks in ((0, 0), (30, 0), (30, 2), (16, 3)):
        want, tol = pc.want(bt, 0.125, win, sinks)
        got = pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, 0.125, gate=bt.gate, win=win, sinks=sinks)
        pc.check(got, want, tol)


def test_prefill_empty_rows_and_bad_pages(pq, dev):
    nh, nkv, hd = 16, 4, 128
    bt = pc.Batch(dev, [20, 40, 33], [100, 0, 64], nh, nkv, hd, 16, BF16, seed=31)
    whole = bt.table
    table, have = bt.table.clone(), [torch.ones(n, dtype=torch.bool, device=dev) for n in bt.n]
    for b, i, bad in ((0, 3, -1), (1, 0, bt.npages), (2, 5, -9)):
        table[b, i] = bad
        have[b][i * 16:(i + 1) * 16] = False
    bt.table = table
    for win, sinks in ((0, 0), (8, 0), (8, 2)):
        want, tol = pc.want(bt, 0.09, win, sinks, have=have)
        got = pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, 0.09, gate=bt.gate, win=win, sinks=sinks)
        pc.check(got, want, tol)
        if not win:
            assert (got[20:36] == 0).all()               # rows whose every key is on the missing page
    # fewer positions than rows: the first rows lie before the sequence and see nothing
    bt.table = whole
    bt.kv_len[1] = 25
    got = pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, 0.09)
    assert (got[20:35] == 0).all() and torch.isfinite(got[35:60]).all() and (got[35:60] != 0).any()
    # the widest window and as many sinks are no window
    for kw in (dict(win=1 << 30), dict(win=1 << 30, sinks=2 ** 31 - 1), dict(sinks=2 ** 31 - 1)):
        assert torch.equal(pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, 0.09, **kw), got)


def test_prefill_many_sequences_and_one_row_each(pq, dev):
    """More sequences than a wave's lanes; and without q_start: a row a sequence, as the decode call."""
    nh, nkv, hd = 8, 2, 64
    q, past = [(7 * i) % 23 for i in range(150)], [(31 * i) % 170 for i in range(150)]
    bt = pc.Batch(dev, q, past, nh, nkv, hd, 16, F16, seed=32)
    want, tol = pc.want(bt, 0.1, 0, 0)
    pc.check(pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, 0.1, gate=bt.gate), want, tol)
    bt = pc.Batch(dev, [1] * 150, past, nh, nkv, hd, 16, F16, seed=33)
    want, tol = pc.want(bt, -0.1, 90, 3)
    for hint in (20, 4000):
        pc.check(pq.paged_attn_prefill(bt.view(pq, False), bt.rows, nh, -0.1, gate=bt.gate, win=90, sinks=3, max_kv=hint),
                 want, tol)
        pc.check(pq.paged_attn_decode(bt.view(pq, False), bt.rows, nh, -0.1, gate=bt.gate, win=90, sinks=3, max_kv=hint),
                 want, tol)


@pytest.mark.parametrize("cache,hd", [(F16, 64), (BF16, 128)])
def test_scale_of_zero(pq, dev, cache, hd):
    """Every visible key has one weight."""
    bt = pc.Batch(dev, [70, 1], [30, 200], 8, 2, hd, 16, cache, seed=34)
    want, tol = pc.want(bt, 0.0, 40, 2)
    pc.check(pq.paged_attn_prefill(bt.view(pq), bt.rows, 8, 0.0, gate=bt.gate, win=40, sinks=2), want, tol)
    one = pq.PagedKV(bt.k, bt.v, bt.table[1:], bt.kv_len[1:])
    pc.check(pq.paged_attn_decode(one, bt.rows[70:], 8, 0.0, gate=bt.gate[70:], win=40, sinks=2), want[70:], tol[70:])


def test_row_starts_that_do_not_ascend(pq, dev):
    """Such a sequence has no rows: the others' are right, and nothing else is written."""
    nh, nkv, hd = 8, 2, 64
    bt = pc.Batch(dev, [40, 30, 20], [10, 50, 0], nh, nkv, hd, 16, F16, seed=35)
    want, tol = pc.want(bt, 0.1, 0, 0)
    kv = bt.view(pq)
    for starts in ([0, 40, 10, 20], [90, 60, 30, 0], [-5, 40, 70, 200], [0, 1 << 30, 5, 90]):
        print(starts, flush=True)
        bt.q_start.copy_(torch.tensor(starts))
        out = torch.full((bt.T + 8, nh * hd), 5.0, dtype=BF16, device=dev)
        pq.paged_attn_prefill(kv, bt.rows, nh, 0.1, gate=bt.gate, out=out[4:-4])
        pq.paged_qk_prep(kv, bt.rows, torch.ones(hd, device=dev), torch.ones(hd, device=dev),
                         torch.ones((100, 16, 2), device=dev), nh, 32)
        assert (out[:4] == 5).all() and (out[-4:] == 5).all()
    torch.cuda.synchronize()
    bt.q_start.copy_(torch.tensor(bt.starts))
    bt.store()
    pc.check(pq.paged_attn_prefill(kv, bt.rows, nh, 0.1, gate=bt.gate), want, tol)


# --------------------------------------------------------------------- together
def test_beside_the_contiguous_attention(pq, dev):
    """One sequence whose pages are one cache: the paged calls and pq_attn_decode see the same keys."""
    nh, nkv, hd, n = 32, 8, 64, 777
    bt = pc.Batch(dev, [40], [n - 40], nh, nkv, hd, 1024, F16, seed=41)
    pg = bt.pages[0][0]
    kc, vc = bt.k[pg], bt.v[pg]
    want = torch.empty((40, nh * hd), dtype=BF16, device=dev)
    pq.attn_decode(bt.rows, bt.rows.stride(0), kc, vc, n - 40, nh, nkv, hd, 40, 0.125, out=want, out_stride=nh * hd, win=100)
    got = pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, 0.125, win=100)
    ref, tol = pc.want(bt, 0.125, 100, 0, gate=False)
    pc.check(got, ref, tol)
    pc.check(want, ref, tol)
    one = pq.PagedKV(bt.k, bt.v, bt.table, bt.kv_len)
    got = pq.paged_attn_decode(one, bt.rows[39:], nh, 0.125, win=100)
    pc.check(got, ref[39:], tol[39:])


@pytest.mark.parametrize("cache,nh,nkv,hd,rot,win,sinks", [(F16, 32, 8, 64, 32, 0, 0), (BF16, 16, 4, 128, 128, 48, 4)])
def test_prompts_then_tokens(pq, dev, cache, nh, nkv, hd, rot, win, sinks):
    """Two chunks of prompts, then decode steps, as a server runs them: each writes the pages (paged_qk_prep) that
    its attention reads, whose Q8_0 output goes into a GEMM; against 64 bits from the cache's own contents."""
    page, scale = 16, 1 / math.sqrt(hd)
    plan = [[37, 90, 1], [20, 1, 64], [1, 1, 1], [1, 1, 1], [1, 1, 1]]
    total = [sum(x) for x in zip(*plan)]
    bt = pc.Batch(dev, [0, 0, 0], total, nh, nkv, hd, page, cache, seed=51)
    bt.k_all.fill_(float("nan"))
    bt.v_all.fill_(float("nan"))
    g = torch.Generator()
    g.manual_seed(52)
    cs = _rope(dev, max(total), rot, g)
    qn, kn = torch.ones(hd, device=dev) * 1.5, torch.ones(hd, device=dev)
    codes = torch.randint(-127, 128, (128, nh * hd), generator=g, dtype=torch.int8).to(dev)
    w = pq.Q8Weight(codes, (torch.rand((128, nh * hd // 32), generator=g) * 1e-3).half().to(dev))
    kv = bt.view(pq)
    done = [0, 0, 0]
    for step, q in enumerate(plan):
        print(f"step {step}", flush=True)
        done = [a + b for a, b in zip(done, q)]
        bt.starts = [0, q[0], q[0] + q[1], sum(q)]
        bt.kv_len.copy_(torch.tensor(done))
        bt.q_start.copy_(torch.tensor(bt.starts))
        rows = torch.randn((sum(q), bt.width), generator=g).to(BF16).to(dev)
        pq.paged_qk_prep(kv, rows, qn, kn, cs, nh, rot, out=rows)
        qx = torch.empty((sum(q), nh * hd), dtype=torch.int8, device=dev)
        dx = torch.empty((sum(q), nh * hd // 32), device=dev)
        out = torch.empty((sum(q), nh * hd), dtype=BF16, device=dev)
        call = pq.paged_attn_decode if max(q) == 1 else pq.paged_attn_prefill
        gate = rows[:, bt.width - nh:]
        call(kv, rows, nh, scale, gate=gate, win=win, sinks=sinks, max_kv=max(done), out=out, qx=qx, dx=dx)
        y = pq.q8_gemm(w, qx, dx)
        for b in range(3):
            slots = [(bt.pages[b][j // page], j % page) for j in range(done[b])]
            bt.keys[b] = torch.stack([bt.k[a, s] for a, s in slots])
            bt.vals[b] = torch.stack([bt.v[a, s] for a, s in slots])
            assert torch.isfinite(bt.keys[b]).all() and torch.isfinite(bt.vals[b]).all()
        bt.n = list(done)
        want, tol = pc.want(bt, scale, win, sinks, rows=rows)
        pc.check(out, want, tol)
        rx, rd = pq.q8_quant(out)
        assert torch.equal(y, pq.q8_gemm(w, rx, rd))


def test_captured_step_replays_for_other_lengths(pq, dev):
    """Prep, decode and prefill captured once; replayed with other lengths, pages and rows, eager work of the same
    calls between the replays; each replay gives the eager call's bits. Two graphs share one workspace."""
    nh, nkv, hd, page = 16, 4, 128, 16
    L = pq.lib()
    sets = []
    for seed, past in ((61, [900, 5, 300]), (62, [100, 640, 77]), (63, [33, 1000, 0])):
        sets.append(pc.Batch(dev, [1, 1, 1], past, nh, nkv, hd, page, BF16, seed=seed, extra=140 - sum(-(-(x + 1) // page) for x in past)))
    cs = _rope(dev, 1024, 128, torch.Generator())
    one = torch.ones(hd, device=dev)
    k, v = sets[0].k.clone(), sets[0].v.clone()
    table = torch.zeros((3, 64), dtype=torch.int32, device=dev)
    n, start, rows = sets[0].kv_len.clone(), sets[0].q_start.clone(), sets[0].rows.clone()
    kv = pq.PagedKV(k, v, table, n, start)
    need = max(L.pq_paged_decode_workspace_bytes(3, nh, nkv, hd, 1024, 0, 0),
               L.pq_paged_prefill_workspace_bytes(3, 3, nh, nkv, hd, 1024, 64, 4), 16)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    qo = torch.empty((3, nh * hd), dtype=BF16, device=dev)
    o1, o2 = torch.empty_like(qo), torch.empty_like(qo)

    def one_step():
        pq.paged_qk_prep(kv, rows, one, one, cs, nh, 128, out=qo)
        pq.paged_attn_decode(kv, qo, nh, 0.088, max_kv=1024, out=o1, ws=ws)

    def two_step():
        pq.paged_attn_prefill(kv, qo, nh, 0.088, win=64, sinks=4, max_kv=1024, out=o2, ws=ws)

    def fill(bt):
        k.copy_(bt.k), v.copy_(bt.v), n.copy_(bt.kv_len), rows.copy_(bt.rows)
        table.fill_(-1)
        table[:, :bt.table.shape[1]] = bt.table

    fill(sets[0])
    one_step(), two_step()
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        one_step()
    with torch.cuda.graph(gb):
        two_step()
    for i in (1, 2, 0, 1):
        fill(sets[i])
        one_step(), two_step()
        want = [t.clone() for t in (qo, o1, o2, k, v)]
        torch.cuda.synchronize()
        fill(sets[i])
        qo.zero_(), o1.zero_(), o2.zero_(), ws.fill_(255)
        ga.replay(), gb.replay()
        torch.cuda.synchronize()
        for a, b in zip((qo, o1, o2, k, v), want):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), i


def test_other_streams(pq, dev):
    """Calls on two streams at once, each with its own output: the bits of the same calls in turn."""
    a = pc.Batch(dev, [1] * 4, [700, 30, 2000, 64], 32, 8, 64, 16, F16, seed=71)
    b = pc.Batch(dev, [100, 60], [40, 0], 16, 4, 128, 32, BF16, seed=72)
    wa = pq.paged_attn_decode(a.view(pq, False), a.rows, 32, 0.125, gate=a.gate)
    wb = pq.paged_attn_prefill(b.view(pq), b.rows, 16, 0.09, gate=b.gate)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    sa.wait_stream(torch.cuda.current_stream()), sb.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(sa):
            ga = pq.paged_attn_decode(a.view(pq, False), a.rows, 32, 0.125, gate=a.gate)
        with torch.cuda.stream(sb):
            gb = pq.paged_attn_prefill(b.view(pq), b.rows, 16, 0.09, gate=b.gate)
    torch.cuda.synchronize()
    assert torch.equal(ga, wa) and torch.equal(gb, wb)


def test_same_call_same_bits(pq, dev):
    a = pc.Batch(dev, [1] * 3, [5000, 300, 64], 16, 4, 128, 16, BF16, seed=81)
    b = pc.Batch(dev, [200, 3], [900, 2500], 16, 4, 128, 64, BF16, seed=82)
    wa = pq.paged_attn_decode(a.view(pq, False), a.rows, 16, 0.09, gate=a.gate)
    wb = pq.paged_attn_prefill(b.view(pq), b.rows, 16, 0.09, gate=b.gate)
    for _ in range(3):
        assert torch.equal(pq.paged_attn_decode(a.view(pq, False), a.rows, 16, 0.09, gate=a.gate), wa)
        assert torch.equal(pq.paged_attn_prefill(b.view(pq), b.rows, 16, 0.09, gate=b.gate), wb)


@pytest.mark.parametrize("cache,nh,nkv,hd", [(F16, 8, 2, 64), (BF16, 4, 1, 128)])
def test_lengths_and_sinks_near_the_largest_int(pq, dev, cache, nh, nkv, hd):
    """Lengths near 2^31, far past the table, with as many sinks: the keys of the table that the sinks reach are seen,
    those of a window that lies past it are not."""
    top = 2 ** 31 - 1
    bt = pc.Batch(dev, [1, 1], [319, 63], nh, nkv, hd, 16, cache, seed=91)
    for n in (top, top - 40, -top - 1):
        bt.kv_len.fill_(n)
        for win, sinks in ((1, top), (30, top), (1, 50), (30, 0), (0, 0), (1 << 30, top)):
            print(n, win, sinks, flush=True)
            table = bt.table.clone()
            table[1, 4:] = -1
            kv = pq.PagedKV(bt.k, bt.v, table, bt.kv_len)
            for call in (pq.paged_attn_decode, pq.paged_attn_prefill):
                for hint in (1, top):
                    got = call(kv, bt.rows, nh, 0.1, win=win, sinks=sinks, max_kv=hint)
                    for b in range(2):
                        p = torch.tensor([n - 1], device=dev)
                        o, size, slack = pc.attend64(bt.rows[b:b + 1, :nh * hd].view(1, nh, hd), p, bt.keys[b], bt.vals[b],
                                                     0.1, win, sinks)
                        pc.check(got[b:b + 1], o, pc.tolerance(o, size, slack, bt.n[b], cache))


@pytest.mark.parametrize("cache,nh,nkv,hd", [(F16, 8, 2, 64), (BF16, 3, 1, 128)])
def test_rows_that_belong_to_a_sequence(pq, dev, cache, nh, nkv, hd):
    """Row r is sequence b's where q_start[b] <= r < q_start[b + 1], whether the starts run past the call's rows at
    either end or stop to ascend (then b's before that): the cache write and the attention, in one piece and in
    splits, agree on them, give the rows of a sequence their output and leave the others as they were."""
    T, lens = 90, [2040, 530, 40]
    bt = pc.Batch(dev, [40, 30, 20], [a - b for a, b in zip(lens, (40, 30, 20))], nh, nkv, hd, 16, cache, seed=36)
    one, cs = torch.ones(hd, device=dev), torch.ones((2100, 16, 2), device=dev)
    L = pq.lib()
    sizes = {hint: L.pq_paged_prefill_workspace_bytes(3, T, nh, nkv, hd, hint, 0, 0) for hint in (1, 2040)}
    assert sizes[1] == 0 and sizes[2040] > 0             # in one piece, in splits
    for starts in ([0, 40, 70, 90], [0, 40, 70, 95], [0, 40, 70, 2 ** 31 - 1], [-5, 40, 70, 200], [-2 ** 31, 40, 90, 90],
                   [0, 40, 10, 20], [0, 40, 0, 0], [3, 40, 40, 90], [90, 60, 30, 0], [0, 1 << 30, 5, 90], [95, 96, 97, 98],
                   [0, 0, 0, 89]):
        print(starts, flush=True)
        bt.q_start.copy_(torch.tensor(starts))
        mine = torch.zeros(T, dtype=torch.bool, device=dev)
        there = torch.zeros(T, dtype=torch.bool, device=dev)
        want = torch.zeros((T, nh, hd), dtype=torch.float64, device=dev)
        tol = torch.zeros_like(want)
        for b in range(3):
            if starts[b] > starts[b + 1]:
                break
            r = torch.arange(max(starts[b], 0), max(min(starts[b + 1], T), max(starts[b], 0)), device=dev)
            p = lens[b] - starts[b + 1] + r
            if not len(r):
                continue
            rows = bt.rows[r]
            o, size, slack = pc.attend64(rows[:, :nh * hd].view(-1, nh, hd), p, bt.keys[b], bt.vals[b], 0.1, 0, 0,
                                         rows[:, bt.width - nh:bt.width])
            want[r], tol[r], mine[r] = o, pc.tolerance(o, size, slack, lens[b], cache), True
            there[r] = p >= 0
        for hint in (1, 2040):
            out = torch.full((T + 8, nh * hd), 5.0, dtype=BF16, device=dev)
            ws = torch.full((max(sizes[hint], 16) // 4,), 1e30, device=dev)
            pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, 0.1, gate=bt.gate, max_kv=hint, out=out[4:-4], ws=ws)
            got = out[4:-4]
            assert (out[:4] == 5).all() and (out[-4:] == 5).all()
            assert (got[~mine] == 5).all(), (hint, "a row of no sequence was written")
            pc.check(got[mine], want[mine], tol[mine])
        # the cache write takes the same rows, those whose position there is
        k, v = bt.k_all.clone(), bt.v_all.clone()
        q = torch.full((T, nh * hd), 5.0, dtype=BF16, device=dev)
        pq.paged_qk_prep(bt.view(pq), bt.rows, one, one, cs, nh, 32, out=q)
        assert torch.equal((q != 5).any(1), there)
        bt.k_all.copy_(k), bt.v_all.copy_(v)


@pytest.mark.parametrize("cache,hd", [(F16, 64), (F16, 128), (BF16, 64), (BF16, 128)])
def test_scales_beside_small_and_large_queries(pq, dev, cache, hd):
    """A scale of 0, or so small that it vanishes beside the queries', leaves every visible key one weight, whatever
    the queries are: the values' mean, beside keys that are hidden."""
    nh, nkv = 8, 2
    bt = pc.Batch(dev, [70, 1], [30, 200], nh, nkv, hd, 16, cache, seed=37)
    rows = bt.rows.clone()
    big = 2.0 ** 60 if cache == BF16 else 2.0 ** 100
    keys = [k.clone() for k in bt.keys]
    for scale, size, kscale in ((0.0, 1.0, 1.0), (0.0, 2.0 ** -30, 1.0), (0.0, 2.0 ** -132, 1.0), (2.0 ** -20, 2.0 ** -132, 1.0),
                                (2.0 ** -140, 2.0 ** -10, 1.0), (0.0, big, 2.0 ** 60 if cache == BF16 else 1.0),
                                (-(2.0 ** -149), 2.0 ** -20, 1.0), (0.125, 0.0, 1.0)):
        print(scale, size, flush=True)
        bt.rows.copy_(rows)
        bt.rows[:, :nh * hd] *= size
        bt.keys = [k * kscale for k in keys]
        bt.store()
        for win, sinks in ((0, 0), (40, 2)):
            want, tol = pc.want(bt, 0.0, win, sinks)
            assert (tol < 0.1).all() or size == big
            one = pq.PagedKV(bt.k, bt.v, bt.table[1:], bt.kv_len[1:])
            tol = torch.minimum(tol, torch.full_like(tol, 0.1))
            for hint in (1, 4000):
                kw = dict(win=win, sinks=sinks, max_kv=hint)
                pc.check(pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, scale, gate=bt.gate, **kw), want, tol)
                pc.check(pq.paged_attn_decode(one, bt.rows[70:], nh, scale, gate=bt.gate[70:], **kw), want[70:], tol[70:])


@pytest.mark.parametrize("cache,hd", [(F16, 64), (F16, 128), (BF16, 64), (BF16, 128)])
def test_scales_that_outgrow_fp32(pq, dev, cache, hd):
    """A scale whose product with the queries' size is past fp32 leaves a score of 0 what it is: keys of zero have one
    weight each, also where a whole tile is seen and where a part of one is."""
    nh, nkv = 8, 2
    bt = pc.Batch(dev, [70, 1], [130, 300], nh, nkv, hd, 16, cache, seed=38)
    bt.keys = [k * 0.0 for k in bt.keys]
    bt.store()
    rows = torch.sign(bt.rows[:, :nh * hd].clone())
    one = pq.PagedKV(bt.k, bt.v, bt.table[1:], bt.kv_len[1:])
    for scale, size in ((2.0, 2.0 ** 127), (-4.0, 2.0 ** 127), (2.0 ** 120, 2.0 ** 20), (3e38, 1.0)):
        bt.rows[:, :nh * hd] = rows * size
        for win, sinks in ((0, 0), (40, 2)):
            want, tol = pc.want(bt, 0.0, win, sinks)
            for hint in (1, 4000):
                kw = dict(win=win, sinks=sinks, max_kv=hint)
                pc.check(pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, scale, gate=bt.gate, **kw), want, tol)
                pc.check(pq.paged_attn_decode(one, bt.rows[70:], nh, scale, gate=bt.gate[70:], **kw), want[70:], tol[70:])


@pytest.mark.parametrize("cache,nh,nkv,hd", [(F16, 8, 2, 64), (F16, 4, 1, 128), (BF16, 8, 2, 64), (BF16, 4, 1, 128)])
def test_mean_of_equal_values(pq, dev, cache, nh, nkv, hd):
    """Where every visible value is one number, so is the output, to the bit: the weights' sum is that of the weights
    that meet the values, as they are rounded, and fp32 sums of 700 of them are off by far less than half a step."""
    bt = pc.Batch(dev, [150, 3, 40], [550, 40, 0], nh, nkv, hd, 16, cache, seed=39)
    g = torch.Generator()
    g.manual_seed(40)
    for b in range(3):
        row = (1 + torch.rand((1, nkv, hd), generator=g)).to(dev).to(BF16).to(cache)
        bt.vals[b] = row.expand(bt.n[b], nkv, hd).clone()
    bt.store()
    for scale in (0.03, 0.125, 1.0):
        for win, sinks in ((0, 0), (100, 3)):
            for hint in (1, 700):
                got = pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, scale, win=win, sinks=sinks, max_kv=hint)
                for b in range(3):
                    want = bt.vals[b][0].to(BF16).repeat_interleave(nh // nkv, 0).view(-1)
                    rows = got[bt.starts[b]:bt.starts[b + 1]]
                    assert (rows == want).all(), f"{int((rows != want).sum())} of {rows.numel()} at {scale} {win} {hint}"
                last = torch.tensor([bt.starts[b + 1] - 1 for b in range(3)], device=dev)
                one = pq.paged_attn_decode(bt.view(pq, False), bt.rows[last], nh, scale, win=win, sinks=sinks, max_kv=hint)
                assert torch.equal(one, got[last])


# ------------------------------------------------- the forms that large calls take
def _rows_of(bt):
    """Every row's sequence and position."""
    seq = [b for b in range(bt.B) for _ in range(bt.q[b])]
    pos = [bt.n[b] - bt.q[b] + i for b in range(bt.B) for i in range(bt.q[b])]
    return seq, pos


@pytest.mark.parametrize("nh,nkv,cache,q,past,win,sinks", [
    (16, 16, F16, [2500, 1, 777, 601], [0, 1300, 5, 64], 0, 0),
    (16, 4, BF16, [2101, 0, 1301, 700], [500, 7, 0, 1100], 0, 0),
    (16, 4, F16, [2101, 3, 1301, 700], [500, 7, 0, 1100], 1024, 5),
    (16, 16, BF16, [2500, 1, 777, 601], [0, 1300, 5, 64], 1000, 24)])
def test_prefill_of_256_row_tiles(pq, dev, nh, nkv, cache, q, past, win, sinks):
    """The kernel of 8 waves: head_dim 128, row tiles of 256 for each kv head that fill 256 CUs, 1024 keys or more
    and no shorter window. Some rows see infinite and NaN values, some have left them behind."""
    hd, page = 128, 32
    bt = pc.Batch(dev, q, past, nh, nkv, hd, page, cache, seed=101, pad=3)
    assert -(-bt.T * (nh // nkv) // 256) * nkv >= 256 and max(bt.n) >= 1024 and (win == 0 or win + sinks >= 1024)
    bt.vals[0][1500, 0, 3] = float("inf")
    bt.vals[0][1777, nkv - 1, 100] = float("nan")
    bt.vals[2][40, 1, 64] = -float("inf")
    bt.vals[2][2, 0, 9] = float("inf")
    bt.keys[3][200, 2] = float("nan")
    bt.vals[3][200, 2] = float("nan")
    bt.store()
    want, tol = pc.want(bt, hd ** -0.5, win, sinks)
    mine = ~torch.isnan(want).all(-1).all(-1)
    out = torch.full((bt.T, nh * hd), 5.0, dtype=BF16, device=dev)
    qx = torch.full((bt.T, nh * hd), 99, dtype=torch.int8, device=dev)
    dx = torch.full((bt.T, nh * hd // 32), 99.0, device=dev)
    pq.paged_attn_prefill(bt.view(pq), bt.rows, nh, hd ** -0.5, gate=bt.gate, win=win, sinks=sinks, max_kv=max(bt.n), out=out,
                          qx=qx, dx=dx)
    pc.check(out[mine], want[mine], tol[mine])
    assert mine[:sum(q)].all() and not mine[sum(q):].any()
    assert (out[sum(q):] == 5).all() and (qx[sum(q):] == 99).all() and (dx[sum(q):] == 99).all()
    rx, rd = pq.q8_quant(out)
    fine = torch.isfinite(out).view(bt.T, -1, 32).all(-1) & mine[:, None]
    assert torch.equal(dx[fine], rd[fine]) and torch.equal(qx.view(bt.T, -1, 32)[fine], rx.view(bt.T, -1, 32)[fine])


@pytest.mark.parametrize("nh,nkv,hd,rot,cache,q,past", [
    (32, 8, 64, 32, F16, [1900, 1, 0, 899], [0, 77, 5, 300]), (32, 8, 64, 64, BF16, [2800], [3]),
    (16, 4, 128, 64, BF16, [1900, 1, 0, 899], [0, 77, 5, 300]), (16, 4, 128, 128, F16, [2800], [3]),
    (24, 2, 64, 32, F16, [4200], [0])])
def test_prep_of_many_rows(pq, dev, nh, nkv, hd, rot, cache, q, past):
    """More than 8192 turns of 64 / (hd / 16) heads: one wave takes a row's heads, turn after turn (the last one short
    where the heads do not fill it)."""
    page = 64
    turn = 64 // (hd // 16)
    bt = pc.Batch(dev, q, past, nh, nkv, hd, page, cache, seed=102, pad=2)
    assert bt.T * -(-(nh + 2 * nkv) // turn) > 8192 and nh + 2 * nkv > turn
    g = torch.Generator()
    g.manual_seed(2)
    limit = max(bt.n)
    cs = _rope(dev, limit, rot, g)
    qn, kn = (1 + 0.2 * torch.randn(hd, generator=g)).to(dev), (1 + 0.2 * torch.randn(hd, generator=g)).to(dev)
    k0, v0 = bt.k_all.clone(), bt.v_all.clone()
    out = torch.full((bt.T, nh * hd), 7.0, dtype=BF16, device=dev)
    pq.paged_qk_prep(bt.view(pq), bt.rows, qn, kn, cs, nh, rot, eps=EPS, out=out)
    seq, pos = _rows_of(bt)
    pages = torch.tensor([bt.pages[b][p // page] for b, p in zip(seq, pos)], device=dev)
    slots = torch.tensor([p % page for p in pos], device=dev)
    k, v = bt.k[pages, slots], bt.v[pages, slots]
    for b in range(bt.B):
        qq, kk, vv, qs, ks, p, on = _prep64(bt, bt.rows, qn, kn, cs, rot, b, limit)
        r = slice(bt.starts[b], bt.starts[b + 1])
        _near(out[r].view(-1, nh, hd), qq, qs, BF16, "q") if bt.q[b] else None
        _near(k[r], kk, ks, cache, "k") if bt.q[b] else None
        _near(v[r], vv, torch.zeros_like(vv), cache, "v") if bt.q[b] else None
    k0[pages, slots], v0[pages, slots] = k, v
    assert torch.equal(bt.k_all.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(bt.v_all.view(torch.int16), v0.view(torch.int16))
    assert (out[sum(q):] == 7).all()


@pytest.mark.parametrize("nh,nkv,hd,cache", [(32, 8, 64, F16), (32, 8, 64, BF16), (16, 4, 128, F16), (16, 4, 128, BF16)])
def test_decode_past_the_caches(pq, dev, nh, nkv, hd, cache):
    """A call that is said to read 256 MiB or more of keys and values reads them past the caches."""
    past = [3000, 1, 700, 40]
    bt = pc.Batch(dev, [1] * 4, past, nh, nkv, hd, 16, cache, seed=103)
    hint = 1 << 18
    assert 4 * nkv * (hint // 32) * 32 * 4 * hd >= 256 << 20
    for win, sinks in ((0, 0), (1 << 18, 3), (1 << 17, 70)):
        want, tol = pc.want(bt, 0.1, win, sinks)
        got = pq.paged_attn_decode(bt.view(pq, False), bt.rows, nh, 0.1, gate=bt.gate, win=win, sinks=sinks, max_kv=hint)
        pc.check(got, want, tol)


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_weights_of_16_bits(pq, dev, hd):
    """A bf16 pool's weights go into the value product as two bf16, 16 bits of them in all: where the values cancel, the
    output is what the weights' roundings leave, half a step of the second bf16, 2^-16 of a weight at most."""
    lens = [2, 3, 5, 9, 33, 64, 65, 200] * 4
    nh = nkv = 4
    bt = pc.Batch(dev, [1] * len(lens), [n - 1 for n in lens], nh, nkv, hd, 16, BF16, seed=104)
    bt.rows[:, :nh * hd] *= 0.25
    scale = 0.125
    for b, n in enumerate(lens):
        q = bt.rows[b, :nh * hd].double().view(nh, hd)
        s = scale * torch.einsum("hd,nhd->hn", q, bt.keys[b].double())
        w = torch.softmax(s, 1)                          # [nh][n]
        v = bt.vals[b].double()
        top = w.argmax(1)
        for h in range(nh):                              # the key of the largest weight takes the others' sum back
            rest = w[h] @ v[:, h] - w[h, top[h]] * v[top[h], h]
            bt.vals[b][top[h], h] = (-rest / w[h, top[h]]).to(BF16)
    bt.store()
    want, tol = torch.zeros((len(lens), nh, hd), dtype=torch.float64, device=dev), None
    tol = torch.zeros_like(want)
    for b, n in enumerate(lens):
        o, size, slack = pc.attend64(bt.rows[b:b + 1, :nh * hd].view(1, nh, hd), torch.tensor([n - 1], device=dev), bt.keys[b],
                                     bt.vals[b], scale, 0, 0)
        want[b], tol[b] = o[0], (2.0 ** -8 * o.abs() + size * (2.0 ** -16 + slack + (n / 8 + 80) * 2.0 ** -24))[0]
        assert (tol[b] < 2.0 ** -12 * size[0]).float().mean() > 0.9       # far below one bf16's 2^-8
    for hint in (1, 1 << 16):
        pc.check(pq.paged_attn_decode(bt.view(pq, False), bt.rows, nh, scale, max_kv=hint), want, tol)
