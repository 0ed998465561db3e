"""The 4-bit cache's operators on the GPU against the 64-bit definition (oracle/kv4_ref.py).

store and load are decided exactly, so their results are compared bit for bit; attention within the bound that
kv4_ref.attention derives for each output from the roundings the kernels make."""
import ctypes as C

import pytest
import torch

from oracle import kv4_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
I32 = torch.int32


@pytest.fixture(scope="module")
def kv4(a8):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    a8.load()
    a8._lib.call("a8_clear_error")
    return a8


def no_error(a8):
    torch.cuda.synchronize()
    assert a8.device_error()[0] == 0, a8.device_error()


def bounds_error(a8):
    torch.cuda.synchronize()
    code = a8.device_error()[0]
    a8._lib.call("a8_clear_error")
    return code == 4


def i32(xs):
    return torch.tensor(xs, dtype=I32, device="cuda")


def rnd(seed, *shape, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF)


def tables(hd, n, seed=0):
    ph = torch.outer(torch.arange(n).float(), 1.0 / (1e4 ** (torch.arange(0, hd, 2).float() / hd)))
    return tuple(torch.cat([f, f], -1).to(BF).contiguous() for f in (ph.cos(), ph.sin()))


def same(a, b):
    """Equal bits up to the sign of zero and the payload of NaN."""
    a, b = a.float().cpu(), b.float().cpu()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def garbage(c):
    """Every byte 0xFF: NaN scales and the code +7 wherever nothing has been stored."""
    c.buf.fill_(255)
    return c


# ------------------------------------------------------------------------------------------------- store and load
@pytest.mark.parametrize("hd,nq,nkv", [(64, 14, 2), (128, 8, 8), (64, 0, 1), (128, 6, 1), (64, 7, 7), (128, 0, 3)])
@pytest.mark.parametrize("rows", [1, 3, 65])
def test_store_then_load(kv4, hd, nq, nkv, rows):
    S, CR = 70, 5
    c = garbage(kv4.KV4Cache(CR, nkv, hd, S, layers=3))
    ld = (nq + 2 * nkv) * hd + 24                                # rows with a gap behind them
    x = rnd(rows + hd, rows, ld)
    g = torch.Generator().manual_seed(rows)
    at = torch.randperm(S * CR, generator=g)[:rows]              # distinct (row, position) pairs
    pos, slot = (at % S).to(I32), (at // S).to(I32)
    cos, sin = tables(hd, S)
    q = c.store(x.cuda(), pos.cuda(), slot.cuda(), layer=1, nq=nq, cos=cos.cuda(), sin=sin.cuda())
    k, v = c.load(pos.cuda(), slot.cuda(), layer=1)
    no_error(kv4)
    h = x[:, :(nq + 2 * nkv) * hd].view(rows, nq + 2 * nkv, hd)
    qk = R.rotate(h[:, :nq + nkv], cos[pos.long()], sin[pos.long()])
    if nq:
        assert same(q, qk[:, :nq].reshape(rows, -1))
    else:
        assert q is None
    assert same(k, R.values(qk[:, nq:]).to(BF)) and same(v, R.values(h[:, nq + nkv:]).to(BF))
    # nothing else changed: every other position of the layer, and the other layers, still read as they did
    every = torch.arange(S * CR)
    other = every[~torch.isin(every, at)]
    k, v = c.load((other % S).to(I32).cuda(), (other // S).to(I32).cuda(), layer=1)
    assert bool(k.isnan().all()) and bool(v.isnan().all())
    n = c.nbytes // 3
    assert bool((c.buf[:n] == 255).all()) and bool((c.buf[2 * n:] == 255).all())
    no_error(kv4)


@pytest.mark.parametrize("hd", [64, 128])
def test_store_without_rotation_extremes(kv4, hd):
    """Groups of zeros, of one tiny value, of subnormals, of the largest values, with an infinity or a NaN; codes on
    every border."""
    nkv = 2
    x = rnd(5, 40, 2 * nkv * hd, scale=2.0)
    x[0] = 0
    x[1] = 0
    x[1, 3] = 2.0 ** -133
    x[2] *= 2.0 ** -130
    x[3] = 3.38e38 * torch.sign(x[3].float()).to(BF)
    x[4, 7], x[4, hd], x[5, 40] = float("inf"), float("-inf"), float("nan")
    x[6] = -0.0
    s = torch.tensor(0.140625)                                   # a bf16 scale: 7 s is the group's maximum
    x[7] = ((torch.arange(2 * nkv * hd) % 14 - 6.5) * s).to(BF)
    x[7, ::32] = (7 * s).to(BF)
    c = kv4.KV4Cache(1, nkv, hd, 40)
    pos, slot = torch.arange(40, dtype=I32), torch.zeros(40, dtype=I32)
    c.store(x.cuda(), pos.cuda(), slot.cuda())
    k, v = c.load(pos.cuda(), slot.cuda())
    no_error(kv4)
    h = x.view(40, 2, nkv, hd)
    assert same(k, R.values(h[:, 0]).to(BF)) and same(v, R.values(h[:, 1]).to(BF))
    assert int(k.isnan().sum() + v.isnan().sum()) == 3 * 32


def test_store_ring_padding_in_place_and_default_rows(kv4):
    hd, nq, nkv, ring, S = 64, 4, 2, 24, 40
    rows = 9
    c = garbage(kv4.KV4Cache(rows, nkv, hd, S))
    cos, sin = tables(hd, 200)
    pos = torch.tensor([0, 23, 24, 199, -1, 48, -7, 100, 25], dtype=I32)
    x = rnd(8, rows, (nq + 2 * nkv) * hd)
    buf = x.cuda()
    out = c.store(buf, pos.cuda(), nq=nq, cos=cos.cuda(), sin=sin.cuda(), ring=ring, q=buf)
    assert out.data_ptr() == buf.data_ptr()
    live = pos >= 0
    at = torch.where(live, pos % ring, 0).to(I32)
    k, v = c.load(at.cuda())
    no_error(kv4)
    h = x.view(rows, nq + 2 * nkv, hd)
    qk = R.rotate(h[:, :nq + nkv], cos[pos.clamp(min=0).long()], sin[pos.clamp(min=0).long()])
    assert same(k[live], R.values(qk[:, nq:]).to(BF)[live]) and same(v[live], R.values(h[:, nq + nkv:]).to(BF)[live])
    assert bool(k[~live].isnan().all())
    want = x.clone()
    want[live, :nq * hd] = qk[:, :nq].reshape(rows, -1).to(BF)[live]
    assert same(buf, want)                                       # padding rows and the k / v columns are as they were


def test_load_leaves_padding_and_strides(kv4):
    hd, nkv = 128, 3
    c = kv4.KV4Cache(2, nkv, hd, 33)
    x = rnd(9, 33, 2 * nkv * hd)
    pos = torch.arange(33, dtype=I32).cuda()
    c.store(x.cuda(), pos, torch.ones(33, dtype=I32, device="cuda"))
    big = torch.full((6, nkv * hd + 40), 3.0, dtype=BF, device="cuda")
    k = big[:, :nkv * hd].unflatten(1, (nkv, hd))
    want = R.values(x.view(33, 2, nkv, hd)).to(BF)
    at = i32([5, 32, -1, 5, 0])
    _, v = c.load(at, i32([1] * 5), k=k)
    no_error(kv4)
    for r, a in ((0, 5), (1, 32), (3, 5), (4, 0)):
        assert same(k[r], want[a, 0]) and same(v[r], want[a, 1])
    assert bool((k[2] == 3).all()) and bool((k[5] == 3).all()) and bool((big[:, nkv * hd:] == 3).all())


def test_out_of_range_rows_are_recorded_not_written(kv4):
    hd, nkv, S = 64, 1, 20
    c = garbage(kv4.KV4Cache(3, nkv, hd, S))
    x = rnd(10, 1, 2 * nkv * hd).cuda()
    cos, sin = (t.cuda() for t in tables(hd, 10))
    for pos, slot, kw in ((S, 0, {}), (0, 3, {}), (0, -1, {}), (12, 0, dict(cos=cos, sin=sin))):
        c.store(x, i32([pos]), i32([slot]), **kw)
        assert bounds_error(kv4), (pos, slot)
        assert bool((c.buf == 255).all())
    for pos, slot in ((S, 0), (0, 3), (0, -1)):
        k = torch.full((1, nkv, hd), 3.0, dtype=BF, device="cuda")
        c.load(i32([pos]), i32([slot]), k=k)
        assert bounds_error(kv4) and bool((k == 3).all())
    no_error(kv4)


# ------------------------------------------------------------------------------------------------- decode attention
def filled(kv4, seed, fill, CR, nkv, hd, S, layers=1, layer=0, kscale=1.0):
    """A cache full of garbage with rows [0, n) of the cache rows in fill {row: n} stored; and those K / V, float64."""
    c = garbage(kv4.KV4Cache(CR, nkv, hd, S, layers=layers))
    kv = {}
    for row, n in fill.items():
        if n <= 0:
            continue
        x = rnd(seed * 1000 + row, n, 2 * nkv * hd)
        x[:, :nkv * hd] *= kscale
        c.store(x.cuda(), torch.arange(n, dtype=I32).cuda(), torch.full((n,), row, dtype=I32).cuda(), layer=layer)
        kv[row] = R.values(x.view(n, 2, nkv, hd))
    return c, kv


def check_rows(got, q, kv, spans, nq, nkv, hd, scale=None):
    """got bf16 [rows, nq hd]; spans: (row, count, cache row, first position) -- row + i attends [0, first + i]."""
    scale = scale or hd ** -0.5
    got, q = got.float().cpu().double().view(-1, nq, hd), q.cpu().double().view(-1, nq, hd)
    grp = nq // nkv
    for r, n, crow, first in spans:
        if first < 0:
            assert bool((got[r:r + n] == 0).all())
            continue
        k, v = kv[crow][:first + n, 0], kv[crow][:first + n, 1]
        for h in range(nq):
            o, tol = R.attention(q[r:r + n, h], k[:, h // grp], v[:, h // grp], first, scale)
            d = (got[r:r + n, h] - o).abs()
            assert bool((d <= tol).all()), (r, h, float(d.max()), float(tol[d > tol].max()))


HEADS = [(14, 2, 64), (8, 8, 128), (32, 8, 128), (6, 1, 128), (7, 7, 64), (16, 1, 64), (9, 1, 64), (11, 1, 128),
         (16, 1, 128), (4, 4, 64)]


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_attention_ragged(kv4, nq, nkv, hd):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 100, 0, 129, 3]
    rows, S = len(lens), 150
    rowmap = torch.randperm(rows + 2, generator=torch.Generator().manual_seed(nq)).tolist()[:rows]
    c, kv = filled(kv4, nq + hd, dict(zip(rowmap, lens)), rows + 2, nkv, hd, S, layers=2, layer=1)
    q = rnd(nq, rows, nq * hd, scale=1.5)
    spans = [(r, 1, rowmap[r], n - 1) for r, n in enumerate(lens)]
    out = c.attention(q.cuda(), i32(lens), i32(rowmap), layer=1)
    no_error(kv4)
    check_rows(out, q, kv, spans, nq, nkv, hd)
    # rows with gaps, another scale, every length cut at max_len
    big = torch.full((rows, nq * hd + 16), 5.0, dtype=BF, device="cuda")
    qs = torch.zeros(rows, nq * hd + 8, dtype=BF, device="cuda")
    qs[:, :nq * hd] = q.cuda()
    c.attention(qs[:, :nq * hd], i32(lens), i32(rowmap), layer=1, max_len=64, scale=0.3, out=big[:, :nq * hd])
    no_error(kv4)
    assert bool((big[:, nq * hd:] == 5).all())
    check_rows(big[:, :nq * hd].contiguous(), q, kv, [(r, 1, m, min(f, 63)) for r, _, m, f in spans], nq, nkv, hd, 0.3)


@pytest.mark.parametrize("nq,nkv,hd,lens", [(14, 2, 64, [733]), (32, 8, 128, [5003, 1, 2600]), (6, 1, 128, [4999]),
                                            (16, 1, 64, [3001, 40]), (8, 8, 128, [128] * 5), (1, 1, 64, [1]),
                                            (14, 2, 64, [2047, 1999, 3, 0, 512] * 8)])
def test_attention_lengths(kv4, nq, nkv, hd, lens):
    rows = len(lens)
    c, kv = filled(kv4, 7, dict(enumerate(lens)), rows, nkv, hd, max(lens) + 9)
    q = rnd(21, rows, nq * hd, scale=1.5)
    out = c.attention(q.cuda(), i32(lens))
    again = c.attention(q.cuda(), i32(lens), max_len=max(lens))
    no_error(kv4)
    check_rows(out, q, kv, [(r, 1, r, n - 1) for r, n in enumerate(lens)], nq, nkv, hd)
    check_rows(again, q, kv, [(r, 1, r, n - 1) for r, n in enumerate(lens)], nq, nkv, hd)
    assert torch.equal(out, c.attention(q.cuda(), i32(lens)))    # equal calls, equal bits


def test_attention_many_short_rows(kv4):
    rows, nq, nkv, hd = 1000, 14, 2, 64
    lens = torch.randint(0, 40, (rows,), generator=torch.Generator().manual_seed(2)).tolist()
    c, kv = filled(kv4, 3, {r: 40 for r in range(7)}, 7, nkv, hd, 40)
    q = rnd(22, rows, nq * hd)
    rowmap = [r % 7 for r in range(rows)]
    out = c.attention(q.cuda(), i32(lens), i32(rowmap))
    no_error(kv4)
    check_rows(out, q, kv, [(r, 1, rowmap[r], n - 1) for r, n in enumerate(lens)], nq, nkv, hd)


def test_attention_peaked_and_growing_logits(kv4):
    """Logits far apart, the maximum first, last, and rising with every key: the running maximum moves at each step."""
    nq, nkv, hd, n = 4, 2, 64, 400
    c = garbage(kv4.KV4Cache(3, nkv, hd, n))
    q = rnd(31, 3, nq * hd, scale=2.0)
    kv = {}
    for row, ramp in enumerate((torch.linspace(0, 8, n), torch.linspace(8, 0, n), torch.linspace(-40, 40, n))):
        x = rnd(40 + row, n, 2, nkv, hd)
        for h in range(nkv):
            x[:, 0, h] = (q[row].view(nq, hd)[h * 2].float() * ramp[:, None]).to(BF)
        c.store(x.view(n, -1).cuda(), torch.arange(n, dtype=I32).cuda(), torch.full((n,), row, dtype=I32).cuda())
        kv[row] = R.values(x)
    out = c.attention(q.cuda(), i32([n] * 3))
    no_error(kv4)
    check_rows(out, q, kv, [(r, 1, r, n - 1) for r in range(3)], nq, nkv, hd)


def test_attention_wide_value_scales(kv4):
    """Values of very different size within a row: from 2^-100 to 2^100 by position."""
    nq, nkv, hd, n = 7, 1, 128, 90
    c = garbage(kv4.KV4Cache(1, nkv, hd, n))
    x = rnd(50, n, 2, nkv, hd)
    x[:, 1] *= (2.0 ** torch.linspace(-100, 100, n)).to(BF)[:, None, None]
    c.store(x.view(n, -1).cuda(), torch.arange(n, dtype=I32).cuda(), torch.zeros(n, dtype=I32).cuda())
    q = rnd(51, 1, nq * hd)
    for m in (1, 30, 90):
        check_rows(c.attention(q.cuda(), i32([m])), q, {0: R.values(x)}, [(0, 1, 0, m - 1)], nq, nkv, hd)
    no_error(kv4)


def test_attention_nan_is_its_row_and_head_only(kv4):
    nq, nkv, hd = 4, 2, 64
    c = kv4.KV4Cache(3, nkv, hd, 50)
    for row in range(3):
        x = rnd(60 + row, 50, 2, nkv, hd)
        if row == 1:
            x[20, 1, 1, 5] = float("nan")                        # a value of kv head 1: dims 0..31 of its query heads
        c.store(x.view(50, -1).cuda(), torch.arange(50, dtype=I32).cuda(), torch.full((50,), row, dtype=I32).cuda())
    q = rnd(61, 3, nq * hd).cuda()
    out = c.attention(q, i32([50, 50, 50])).view(3, nq, 2, 32)
    cut = c.attention(q, i32([50, 20, 50])).view(3, nq, 2, 32)   # the NaN lies behind the length
    no_error(kv4)
    nan = out.isnan().all(-1).cpu()
    assert int(nan.sum()) == 2 and bool(nan[1, 2:, 0].all()) and int(out.isnan().sum()) == 64
    assert not bool(cut.isnan().any())


def test_attention_bad_cache_row(kv4):
    nq, nkv, hd = 14, 2, 64
    c, kv = filled(kv4, 4, {0: 30, 1: 30}, 2, nkv, hd, 30)
    q = rnd(62, 4, nq * hd)
    out = c.attention(q.cuda(), i32([30, 30, 30, 30]), i32([0, 2, 1, -1]))
    assert bounds_error(kv4)
    check_rows(out, q, kv, [(0, 1, 0, 29), (1, 1, 0, -1), (2, 1, 1, 29), (3, 1, 0, -1)], nq, nkv, hd)


def test_attention_two_streams_and_graphs(kv4):
    """Calls that overlap on two streams, and two captured graphs replayed at once, do not disturb each other; a
    replay reads lens and cache as they are then."""
    nq, nkv, hd, S = 14, 2, 64, 3000
    c, kv = filled(kv4, 5, {0: S, 1: S}, 2, nkv, hd, S)
    qs = [rnd(70 + i, 2, nq * hd) for i in range(2)]
    dq = [q.cuda() for q in qs]
    lens = [i32([3000, 17]), i32([1200, 2999])]
    want = [c.attention(dq[i], lens[i]) for i in range(2)]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(st[i]):
                outs[i].append(c.attention(dq[i], lens[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    graphs, gout = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gout.append(c.attention(dq[i], lens[i]))
        graphs.append(g)
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(st[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(gout[i], want[i])
    lens[0].copy_(i32([5, 64]))
    graphs[0].replay()
    no_error(kv4)
    check_rows(gout[0], qs[0], kv, [(0, 1, 0, 4), (1, 1, 1, 63)], nq, nkv, hd)


def test_attention_past_32_bit_offsets(kv4):
    """A cache of 4.8 GB: the last row's records lie past 2^32 bytes."""
    nq, nkv, hd, S, CR = 8, 8, 128, 131072, 32
    c = kv4.KV4Cache(CR, nkv, hd, S)
    assert c.nbytes > 1 << 32
    x = rnd(80, 50, 2, nkv, hd)
    pos = torch.arange(S - 50, S, dtype=I32).cuda()
    c.store(x.view(50, -1).cuda(), pos, torch.full((50,), CR - 1, dtype=I32).cuda())
    k, v = c.load(pos, torch.full((50,), CR - 1, dtype=I32).cuda())
    assert same(k, R.values(x[:, 0]).to(BF)) and same(v, R.values(x[:, 1]).to(BF))
    # keys before them are zeros of an empty cache: scale 0, logit 0, value 0
    q = rnd(81, 1, nq * hd, scale=3.0)
    out = c.attention(q.cuda(), i32([S]), i32([CR - 1]))
    no_error(kv4)
    full = torch.zeros(S, 2, nkv, hd, dtype=torch.float64)
    full[S - 50:] = R.values(x)
    check_rows(out, q, {CR - 1: full}, [(0, 1, CR - 1, S - 1)], nq, nkv, hd)


# ------------------------------------------------------------------------------------------------- prompt attention
def packed(kv4, seed, parts, nq, nkv, hd, S, CR, kscale=1.0):
    """parts: (slot, first position, count) of each request -> cache, kv, q, blocks, spans."""
    from audio8_b200.engine import FastEngine
    c, kv = filled(kv4, seed, {s: a + n for s, a, n in parts}, CR, nkv, hd, S, kscale=kscale)
    rows = sum(n for _, _, n in parts)
    q = rnd(seed + 500, rows, nq * hd, scale=1.5)
    pos = [p for _, a, n in parts for p in range(a, a + n)]
    slot = [s for s, _, n in parts for _ in range(n)]
    spans, r = [], 0
    for s, a, n in parts:
        spans.append((r, n, s, a))
        r += n
    return c, kv, q, torch.from_numpy(FastEngine.query_blocks(pos, slot)), spans


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_prefill_ragged(kv4, nq, nkv, hd):
    parts = [(4, 0, 1), (0, 0, 64), (2, 17, 65), (1, 63, 3), (5, 128, 130), (3, 0, 200)]
    c, kv, q, blocks, spans = packed(kv4, nq, parts, nq, nkv, hd, 300, 6)
    out = c.prefill_attention(q.cuda(), blocks.cuda())
    no_error(kv4)
    check_rows(out, q, kv, spans, nq, nkv, hd)


@pytest.mark.parametrize("nq,nkv,hd,parts", [(14, 2, 64, [(0, 0, 1500)]), (4, 1, 128, [(0, 0, 1111)]),
                                             (8, 8, 128, [(0, 700, 70), (1, 1300, 1)]), (14, 2, 64, [(0, 0, 1)]),
                                             (14, 2, 64, [(1, 317, 211), (0, 317, 33), (2, 317, 90)])])
def test_prefill_lengths(kv4, nq, nkv, hd, parts):
    c, kv, q, blocks, spans = packed(kv4, 11, parts, nq, nkv, hd, max(a + n for _, a, n in parts), 3)
    out = c.prefill_attention(q.cuda(), blocks.cuda())
    no_error(kv4)
    check_rows(out, q, kv, spans, nq, nkv, hd)
    assert torch.equal(out, c.prefill_attention(q.cuda(), blocks.cuda()))


def test_prefill_peaked(kv4):
    """Keys along the query with a rising and a falling factor: the running maximum moves in every tile."""
    nq, nkv, hd, n = 2, 1, 64, 333
    c = garbage(kv4.KV4Cache(2, nkv, hd, n))
    base = rnd(90, hd, scale=2.0)
    q = (base.float()[None, None] * (1 + 0.2 * rnd(91, 2 * n, nq, 1).float())).to(BF).reshape(2 * n, nq * hd)
    kv = {}
    for row, ramp in enumerate((torch.linspace(-20, 20, n), torch.linspace(30, 0, n))):
        x = rnd(92 + row, n, 2, nkv, hd)
        x[:, 0, 0] = (base.float() * ramp[:, None] / 4).to(BF)
        c.store(x.view(n, -1).cuda(), torch.arange(n, dtype=I32).cuda(), torch.full((n,), row, dtype=I32).cuda())
        kv[row] = R.values(x)
    from audio8_b200.engine import FastEngine
    blocks = FastEngine.query_blocks(list(range(n)) * 2, [0] * n + [1] * n)
    out = c.prefill_attention(q.cuda(), torch.from_numpy(blocks).cuda())
    no_error(kv4)
    check_rows(out, q, kv, [(0, n, 0, 0), (n, n, 1, 0)], nq, nkv, hd)


def test_prefill_blocks_skipped_uncovered_and_bad(kv4):
    """Empty blocks are skipped, rows no block covers stay, blocks in any order and of any size up to 64 are taken, and
    a block out of range writes nothing and is recorded."""
    nq, nkv, hd, S = 14, 2, 64, 140
    c, kv = filled(kv4, 6, {0: S, 1: S}, 2, nkv, hd, S)
    q = rnd(95, 120, nq * hd)
    out = torch.full((120, nq * hd), 9.0, dtype=BF, device="cuda")
    good = [(70, 50, 1, 90), (0, 0, 0, 0), (3, 7, 0, 5), (64, 1, 0, 139), (20, -1, 0, 0)]
    c.prefill_attention(q.cuda(), i32(good), out=out)
    no_error(kv4)
    spans = [(r, n, s, a) for r, n, s, a in good if n > 0]
    check_rows(out, q, kv, spans, nq, nkv, hd)
    kept = torch.ones(120, dtype=torch.bool)
    for r, n, _, _ in spans:
        kept[r:r + n] = False
    assert bool((out[kept.cuda()] == 9).all())
    bad = [(0, 65, 0, 0), (100, 21, 0, 0), (-1, 2, 0, 0), (0, 4, 2, 0), (0, 4, -1, 0), (0, 4, 0, -1), (0, 4, 0, 137),
           (2147483647, 2, 0, 0), (0, 2, 0, 2147483647)]
    for b in bad:
        out.fill_(9.0)
        c.prefill_attention(q.cuda(), i32([b]), out=out)
        assert bounds_error(kv4), b
        assert bool((out == 9).all()), b


# ------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("nq,nkv,hd", [(14, 2, 64), (8, 8, 128)])
def test_a_layer_prompt_then_decode(kv4, nq, nkv, hd):
    """As an engine's layer runs: the qkv GEMM with its bias, store, prompt attention; then decode steps, captured into
    a graph, each storing one token a row and attending what is there."""
    L = kv4._lib
    dim, S, NQ = 256, 120, nq * hd
    N = (nq + 2 * nkv) * hd
    w, bias = rnd(1, N, dim, scale=dim ** -0.5), rnd(2, N, scale=0.1)
    W, Bi = w.cuda(), bias.cuda()
    cos, sin = tables(hd, S)
    Cs, Sn = cos.cuda(), sin.cuda()
    parts = [(2, 0, 37), (0, 0, 5)]
    c = garbage(kv4.KV4Cache(3, nkv, hd, S))
    from audio8_b200.engine import FastEngine

    def gemm(x, y):
        e = L.A8Epilogue(kind=L.EPI_BF16, bias=L.ptr(Bi))
        L.call("a8_gemm", L.ptr(x), dim, L.ptr(W), N, dim, x.shape[0], L.ptr(y), N, C.byref(e), 0, L.stream_handle())

    pos = [p for _, a, n in parts for p in range(a, a + n)]
    slot = [s for s, _, n in parts for _ in range(n)]
    x = rnd(3, 42, dim).cuda()
    y = torch.empty(42, N, dtype=BF, device="cuda")
    gemm(x, y)
    raw = y.cpu()                                                # the kernels' own input: the GEMM is tested elsewhere
    q = c.store(y, i32(pos), i32(slot), nq=nq, cos=Cs, sin=Sn)
    out = c.prefill_attention(q, torch.from_numpy(FastEngine.query_blocks(pos, slot)).cuda())
    no_error(kv4)
    hist = {s: [] for s, _, _ in parts}

    def remember(raw, pos, slot):
        """float64 queries; keys and values appended to their rows."""
        p, h = torch.tensor(pos), raw.view(len(pos), nq + 2 * nkv, hd)
        qk = R.rotate(h[:, :nq + nkv], cos[p], sin[p])
        for i, s in enumerate(slot):
            hist[s].append(R.values(torch.stack([qk[i, nq:].to(BF), h[i, nq + nkv:]])))
        return qk[:, :nq].reshape(len(pos), NQ)

    qo = remember(raw, pos, slot)
    kv = {s: torch.stack(v) for s, v in hist.items()}
    check_rows(out, qo, kv, [(0, 37, 2, 0), (37, 5, 0, 0)], nq, nkv, hd)
    # decode: two rows; the graph holds the GEMM, the store and the attention, and advances the positions itself
    dpos, dslot = i32([37, 5]), i32([2, 0])
    xin, yd = torch.zeros(2, dim, dtype=BF, device="cuda"), torch.zeros(2, N, dtype=BF, device="cuda")
    gemm(xin, yd)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gemm(xin, yd)
        qd = c.store(yd, dpos, dslot, nq=nq, cos=Cs, sin=Sn)
        dpos.add_(1)
        od = c.attention(qd, dpos, dslot)
    for step in range(12):
        xin.copy_(rnd(100 + step, 2, dim))
        g.replay()
        no_error(kv4)
        at = [37 + step, 5 + step]
        qo = remember(yd.cpu(), at, [2, 0])
        kv = {s: torch.stack(v) for s, v in hist.items()}
        assert same(qd, qo)
        check_rows(od, qo, kv, [(0, 1, 2, at[0]), (1, 1, 0, at[1])], nq, nkv, hd)


# ------------------------------------------------------------------------------------------------- many shapes
def gpu_reference(q, kv, row_keys, nq, nkv, hd):
    """check_rows' reference and bound on the GPU in 64 bits, one query row at a time: row_keys (cache row, keys) each."""
    out = torch.zeros(len(row_keys), nq, hd, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    qd = q.double().view(-1, nkv, nq // nkv, hd)
    for r, (row, n) in enumerate(row_keys):
        if n <= 0:
            continue
        k, v = kv[row][:n, 0].transpose(0, 1), kv[row][:n, 1].transpose(0, 1)          # [nkv, n, hd]
        z = qd[r] @ k.transpose(1, 2) * hd ** -0.5
        w = torch.softmax(z, -1)
        o, pv = w @ v, w @ v.abs()
        logit = (R.logit_error(qd[r], k) * hd ** -0.5).amax(-1, keepdim=True)
        out[r] = o.reshape(nq, hd)
        tol[r] = (2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -10 + 2 * logit) * pv + 1e-30).reshape(nq, hd)
    return out, tol


def random_case(seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda xs: xs[int(torch.randint(0, len(xs), (1,), generator=g))]
    nq, nkv, hd = pick([(14, 2, 64), (8, 8, 128), (12, 3, 128), (16, 1, 64), (10, 1, 128), (3, 3, 64), (5, 1, 64)])
    rows = pick([1, 2, 5, 40, 300, 700, 1537])
    top = pick([1, 33, 64, 200, 900, 2500]) if rows < 300 else pick([1, 40, 130])
    kind = pick(["even", "any", "one long", "mostly empty"])
    lens = torch.randint(0, top + 1, (rows,), generator=g)
    if kind == "even":
        lens[:] = top
    elif kind == "one long":
        lens = lens.clamp(max=3)
        lens[rows // 2] = top
    elif kind == "mostly empty":
        lens[torch.rand(rows, generator=g) < 0.9] = 0
    return nq, nkv, hd, rows, top, lens.tolist(), g


@pytest.mark.parametrize("seed", range(36))
def test_attention_random_shapes(kv4, seed):
    nq, nkv, hd, rows, top, lens, g = random_case(seed)
    CR = min(rows, 11)
    c, kv = filled(kv4, seed, {r: top for r in range(CR)}, CR, nkv, hd, top + seed % 40)
    kv = {r: x.cuda() for r, x in kv.items()}
    q = rnd(seed + 7000, rows, nq * hd, scale=1.5).cuda()
    rowmap = torch.randint(0, CR, (rows,), generator=g).tolist()
    got = c.attention(q, i32(lens), i32(rowmap), max_len=top).double().view(rows, nq, hd)
    no_error(kv4)
    want, tol = gpu_reference(q, kv, list(zip(rowmap, lens)), nq, nkv, hd)
    d = (got - want).abs()
    assert bool((d <= tol).all()), (nq, nkv, hd, rows, top, float((d - tol).max()))


@pytest.mark.parametrize("seed", range(24))
def test_prefill_random_shapes(kv4, seed):
    from audio8_b200.engine import FastEngine
    nq, nkv, hd, rows, top, lens, g = random_case(seed + 100)
    parts, slot = [], 0
    for n in [x for x in lens if x > 0][:9]:
        parts.append((slot, int(torch.randint(0, 300, (1,), generator=g)), n))
        slot += 1
    if not parts:
        parts = [(0, 5, 70)]
    S = max(a + n for _, a, n in parts)
    c, kv = filled(kv4, seed, {s: a + n for s, a, n in parts}, len(parts), nkv, hd, S)
    kv = {r: x.cuda() for r, x in kv.items()}
    pos = [p for _, a, n in parts for p in range(a, a + n)]
    sl = [s for s, _, n in parts for _ in range(n)]
    q = rnd(seed + 9000, len(pos), nq * hd, scale=1.5).cuda()
    blocks = FastEngine.query_blocks(pos, sl)
    blocks = torch.from_numpy(blocks)[torch.randperm(len(blocks), generator=g)].contiguous().cuda()
    got = c.prefill_attention(q, blocks).double().view(len(pos), nq, hd)
    no_error(kv4)
    take = torch.randperm(len(pos), generator=g)[:150].tolist()
    want, tol = gpu_reference(q[take], kv, [(sl[r], pos[r] + 1) for r in take], nq, nkv, hd)
    d = (got[take] - want).abs()
    assert bool((d <= tol).all()), (nq, nkv, hd, parts, float((d - tol).max()))
    # in place
    same_place = q.clone()
    assert c.prefill_attention(same_place, blocks, out=same_place).data_ptr() == same_place.data_ptr()
    assert torch.equal(same_place.double().view(len(pos), nq, hd), got)


def test_prefill_nan_reaches_its_own_rows_only(kv4):
    """A NaN among the values at position 70 makes the 32 dims of its group NaN for rows from 70 on, one among the keys at
    position 90 whole rows from 90 on; earlier rows of the same tiles are untouched."""
    nq, nkv, hd, n = 4, 2, 128, 130
    x = rnd(123, n, 2, nkv, hd)
    q = rnd(124, n, nq * hd).cuda()
    pos = torch.arange(n, dtype=I32).cuda()
    from audio8_b200.engine import FastEngine
    blocks = torch.from_numpy(FastEngine.query_blocks(list(range(n)), [0] * n)).cuda()

    def run(y):
        c = garbage(kv4.KV4Cache(1, nkv, hd, n))
        c.store(y.reshape(n, -1).cuda(), pos, torch.zeros(n, dtype=I32).cuda())
        return c.prefill_attention(q, blocks).view(n, nq, 4, 32).cpu()
    clean = run(x)
    y = x.clone()
    y[70, 1, 1, 40] = float("nan")
    y[90, 0, 0, 3] = float("nan")
    got = run(y)
    no_error(kv4)
    nan = torch.zeros(n, nq, 4, 32, dtype=torch.bool)
    nan[70:, 2:, 1] = True                               # kv head 1: query heads 2, 3; dims 32..63
    nan[90:, :2] = True                                  # kv head 0
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], clean[~nan])


def test_prefill_wide_scales(kv4):
    """Keys and values from 2^-90 to 2^20 and values rising by tiles (the exponent that V is divided by grows)."""
    from audio8_b200.engine import FastEngine
    nq, nkv, hd, n = 2, 1, 64, 300
    x = rnd(130, n, 2, nkv, hd)
    x[:, 1] *= (2.0 ** torch.linspace(-90, 20, n)).to(BF)[:, None, None]
    x[:, 0] *= (2.0 ** torch.linspace(-60, 0, n)).to(BF)[:, None, None]
    c = garbage(kv4.KV4Cache(1, nkv, hd, n))
    c.store(x.reshape(n, -1).cuda(), torch.arange(n, dtype=I32).cuda(), torch.zeros(n, dtype=I32).cuda())
    q = rnd(131, n, nq * hd, scale=2.0)
    out = c.prefill_attention(q.cuda(), torch.from_numpy(FastEngine.query_blocks(list(range(n)), [0] * n)).cuda())
    no_error(kv4)
    got, qd, kv = out.cpu().double().view(n, nq, hd), q.double().view(n, nq, hd), R.values(x)
    for h in range(nq):
        o, tol = R.attention(qd[:, h], kv[:, 0, 0], kv[:, 1, 0], 0, hd ** -0.5)
        # (the exponents fp16 operands are divided by come from whole tiles: the bound of kv4_ref.prompt_slack)
        tol = tol + R.prompt_slack(qd[:, h], kv[:, 0, 0], kv[:, 1, 0], 0, hd ** -0.5)
        d = (got[:, h] - o).abs()
        assert bool((d <= tol).all()), (h, float((d - tol).max()))


def test_attention_in_place(kv4):
    for nq, nkv, hd, lens in ((14, 2, 64, [5000, 3, 0, 70]), (8, 8, 128, [128] * 40), (16, 1, 64, [9000])):
        c, _ = filled(kv4, 9, {0: max(lens)}, 1, nkv, hd, max(lens))
        q = rnd(150, len(lens), nq * hd).cuda()
        rowmap = torch.zeros(len(lens), dtype=I32, device="cuda")
        want = c.attention(q, i32(lens), rowmap)
        place = q.clone()
        c.attention(place, i32(lens), rowmap, out=place)
        no_error(kv4)
        assert torch.equal(place, want)


def test_prompt_attention_between_gemms(kv4):
    """Many CTAs of the prompt attention between GEMMs that hold tensor memory, over and over in one stream and captured:
    each result is the first one's."""
    from audio8_b200.engine import FastEngine
    L = kv4._lib
    nq, nkv, hd, n, dim = 14, 2, 64, 1900, 256
    c, _ = filled(kv4, 8, {0: n}, 1, nkv, hd, n)
    q = rnd(140, n, nq * hd).cuda()
    blocks = torch.from_numpy(FastEngine.query_blocks(list(range(n)), [0] * n)).cuda()
    w = rnd(141, dim, nq * hd, scale=0.03).cuda()
    y = torch.empty(n, dim, dtype=BF, device="cuda")
    o = torch.empty_like(q)

    def chain():
        for _ in range(4):
            c.prefill_attention(q, blocks, out=o)
            e = L.A8Epilogue(kind=L.EPI_BF16)
            L.call("a8_gemm", L.ptr(o), nq * hd, L.ptr(w), dim, nq * hd, n, L.ptr(y), dim, C.byref(e), 0,
                   L.stream_handle())
    chain()
    no_error(kv4)
    first_o, first_y = o.clone(), y.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chain()
    for _ in range(10):
        o.zero_()
        y.zero_()
        g.replay()
    no_error(kv4)
    assert torch.equal(o, first_o) and torch.equal(y, first_y)


@pytest.mark.parametrize("nq,nkv,hd", [(8, 8, 128), (14, 2, 64), (16, 1, 64), (10, 1, 128)])
@pytest.mark.parametrize("kind", ["windows", "at the border", "long among short", "one row"])
def test_attention_units_of_few_steps(kv4, nq, nkv, hd, kind):
    """Units (a row's kv head) of a few steps of 32 keys are kept whole in a warp, longer ones are cut: both, mixed, and at
    the border between them."""
    rows = {"windows": 192, "at the border": 100, "long among short": 150, "one row": 1}[kind]
    g = torch.Generator().manual_seed(rows + nq)
    lens = torch.randint(1, 129, (rows,), generator=g)
    if kind == "at the border":
        lens = torch.tensor([255, 256, 257, 288, 289, 32, 33, 1, 0, 224])[torch.randint(0, 10, (rows,), generator=g)]
    elif kind == "long among short":
        lens[torch.randint(0, rows, (4,), generator=g)] = 1111
        lens[-1] = 700
    lens = lens.tolist()
    top, CR = max(lens), 7
    c, kv = filled(kv4, 31 + nq, {r: top for r in range(CR)}, CR, nkv, hd, top + 3)
    kv = {r: x.cuda() for r, x in kv.items()}
    q = rnd(9000 + rows, rows, nq * hd, scale=1.5).cuda()
    rowmap = torch.randint(0, CR, (rows,), generator=g).tolist()
    got = c.attention(q, i32(lens), i32(rowmap), max_len=top).double().view(rows, nq, hd)
    no_error(kv4)
    want, tol = gpu_reference(q, kv, list(zip(rowmap, lens)), nq, nkv, hd)
    d = (got - want).abs()
    assert bool((d <= tol).all()), float((d - tol).max())


def test_attention_with_a_workspace_of_the_callers(kv4):
    """The caller's workspace serves smaller calls too, comes back ready for the next, and is refused when it is too small
    or not what workspace() gives."""
    nq, nkv, hd, lens = 14, 2, 64, [1900, 0, 700, 1]
    c, kv = filled(kv4, 12, dict(enumerate(lens)), 4, nkv, hd, 2000)
    q = rnd(150, 4, nq * hd, scale=1.5)
    ws = c.workspace(nq, 4, 2000)
    want = c.attention(q.cuda(), i32(lens))
    for n in (4, 2, 4):
        got = c.attention(q[:n].cuda(), i32(lens[:n]), ws=ws, max_len=2000)
        no_error(kv4)
        assert torch.equal(got, c.attention(q[:n].cuda(), i32(lens[:n]))) and not bool(ws[1].any())
    assert torch.equal(got, want)
    check_rows(got, q, kv, [(r, 1, r, n - 1) for r, n in enumerate(lens)], nq, nkv, hd)
    for bad in ((ws[0][:8], ws[1]), (ws[0], ws[1][:7]), (ws[0].double(), ws[1]), (ws[0], ws[1].long()),
                (ws[0].cpu(), ws[1]), (ws[0][::2], ws[1])):
        with pytest.raises(kv4.A8Error):
            c.attention(q.cuda(), i32(lens), ws=bad)
    assert torch.equal(want, c.attention(q.cuda(), i32(lens)))
