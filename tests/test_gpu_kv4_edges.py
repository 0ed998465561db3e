"""Calls of the 4-bit cache's operators that its other tests do not make, on the GPU: degenerate and tiny queries and keys,
against the 64-bit definition (oracle/kv4_ref.py) under its derived bounds."""
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


def rnd(seed, *shape, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF)


def one_row(a8, x, hd):
    """A cache of one row that holds x [n, 2, nkv, hd] at positions 0 .. n - 1."""
    n, _, nkv, _ = x.shape
    c = a8.KV4Cache(1, nkv, hd, n)
    c.store(x.reshape(n, -1).cuda(), torch.arange(n, dtype=I32).cuda(), torch.zeros(n, dtype=I32).cuda())
    return c


def prompt(a8, c, q, n, **kw):
    blocks = torch.from_numpy(a8.FastEngine.query_blocks(list(range(n)), [0] * n)).cuda()
    out = c.prefill_attention(q.cuda(), blocks, **kw)
    no_error(a8)
    return out.cpu().double()


def check_prompt(a8, x, q, hd, scale=None):
    """All n causal rows of q [n, nq hd] over x against the definition."""
    n, nkv, nq = x.shape[0], x.shape[2], q.shape[1] // hd
    got = prompt(a8, one_row(a8, x, hd), q, n, scale=scale or 0.0).view(n, nq, hd)
    kv, qd, scale = R.values(x), q.double().view(n, nq, hd), scale or hd ** -0.5
    for h in range(nq):
        k, v = kv[:, 0, h * nkv // nq], kv[:, 1, h * nkv // nq]
        o, tol = R.attention(qd[:, h], k, v, 0, scale)
        tol = tol + R.prompt_slack(qd[:, h], k, v, 0, scale)
        d = (got[:, h] - o).abs()
        assert bool((d <= tol).all()), (h, float((d - tol).max()), int(got.isnan().sum()))


# ------------------------------------------------------------------------------------------------- logits that vanish
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("qs,ks", [(0.0, 0.0), (0.0, 1.0), (0.0, 2.0 ** -30), (2.0 ** -30, 0.0), (2.0 ** -75, 2.0 ** -75),
                                   (1.0, 0.0), (2.0 ** -120, 2.0 ** -120)])
def test_prompt_of_vanishing_logits_is_the_mean(kv4, hd, qs, ks):
    """Queries and keys of nothing, or so small that their product underflows: every weight is the same, a row is the mean of
    its values (over an empty cache, zero)."""
    n, nq, nkv = 150, 4, 2
    x = rnd(1, n, 2, nkv, hd)
    x[:, 0] = (x[:, 0].float() * ks).to(BF)
    check_prompt(kv4, x, (rnd(2, n, nq * hd).float() * qs).to(BF), hd)


def test_prompt_of_an_empty_cache_is_zero(kv4):
    nq, nkv, hd, n = 14, 2, 64, 100
    c = kv4.KV4Cache(1, nkv, hd, n)
    assert bool((prompt(kv4, c, torch.zeros(n, nq * hd, dtype=BF), n) == 0).all())


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_with_some_vanishing_rows_and_tiles(kv4, hd):
    """Zero queries between others, a whole tile of zero keys between others."""
    n, nq, nkv = 200, 4, 2
    x, q = rnd(3, n, 2, nkv, hd), rnd(4, n, nq * hd)
    x[64:128, 0] = 0
    q[::3] = 0
    q[100:140, :hd] = 0
    check_prompt(kv4, x, q, hd)


@pytest.mark.parametrize("scale", [1e-9, 1e-37])
def test_prompt_of_a_tiny_scale(kv4, scale):
    n, hd = 150, 64
    x, q = rnd(5, n, 2, 2, hd), rnd(6, n, 4 * hd)
    x[:64, 0] = (x[:64, 0].float() * 2.0 ** -60).to(BF)
    q[::2] = 0
    check_prompt(kv4, x, q, hd, scale)


@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 64), (4, 2, 128), (10, 1, 64)])
@pytest.mark.parametrize("scale", [1e-8, 1e-9, 1e-30, 1e-37])
def test_decode_of_a_tiny_scale(kv4, nq, nkv, hd, scale):
    """Rows of zero, tiny and ordinary queries under a scale that leaves nothing of a logit: the mean of the values."""
    n, rows = 77, 6
    x, q = rnd(7, n, 2, nkv, hd), rnd(8, rows, nq * hd)
    q[::2] = 0
    q[1] = (q[1].float() * 2.0 ** -100).to(BF)
    lens = [n, n, 33, 70, 1, 40]
    c = one_row(kv4, x, hd)
    got = c.attention(q.cuda(), torch.tensor(lens, dtype=I32, device="cuda"), torch.zeros(rows, dtype=I32, device="cuda"),
                      scale=scale)
    no_error(kv4)
    got, kv, qd = got.cpu().double().view(rows, nq, hd), R.values(x), q.double().view(rows, nq, hd)
    for r, m in enumerate(lens):
        for h in range(nq):
            k, v = kv[:m, 0, h * nkv // nq], kv[:m, 1, h * nkv // nq]
            o, tol = R.attention(qd[r:r + 1, h], k, v, m - 1, scale)
            d = (got[r:r + 1, h] - o).abs()
            assert bool((d <= tol).all()), (r, h, float((d - tol).max()))


# ------------------------------------------------------------------------------------------------- after a timeout
def test_clear_error_restores_the_tickets(kv4):
    """Tickets left partly taken, as by a kernel that gave up a wait: clear_error() brings a cache's and an engine's back."""
    nq, nkv, hd, n = 14, 2, 64, 3000
    x = rnd(9, n, 2, nkv, hd)
    c = one_row(kv4, x, hd)
    q = rnd(10, 3, nq * hd).cuda()
    lens, row = torch.tensor([n, 17, 2900], dtype=I32, device="cuda"), torch.zeros(3, dtype=I32, device="cuda")
    want = c.attention(q, lens, row)
    no_error(kv4)
    assert c._ws
    for *_, tensors in (have[3] for have in c._ws.values()):
        assert not bool(tensors[1].any())                    # a call leaves them zero
        tensors[1].fill_(1)
        tensors[0].fill_(float("nan"))
    from audio8_b200.engine import Scratch
    sc = Scratch(8, 64, 128, 64, 2, 64, 200, torch.device("cuda", 0), c)
    sc.attn_counters.fill_(1)
    kv4.clear_error()
    assert not bool(sc.attn_counters.any())
    for _ in range(2):
        assert torch.equal(c.attention(q, lens, row), want)
    no_error(kv4)


# ------------------------------------------------------------------------------------------------- one row
def test_a_single_row_of_any_row_stride(kv4):
    """The row stride of a single row is never used: rows cut from wider or oddly strided tensors are taken as they are, in
    place too, and nothing beside them is touched."""
    nq, nkv, hd = 6, 2, 64
    W, Q = (nq + 2 * nkv) * hd, nq * hd
    x = rnd(20, 1, W)
    i0, i1 = torch.zeros(1, dtype=I32, device="cuda"), torch.ones(1, dtype=I32, device="cuda")
    c = kv4.KV4Cache(1, nkv, hd, 20)
    want = c.store(x.cuda(), i0, i0, nq=nq)
    wk, wv = c.load(i0, i0)
    wo = c.attention(want, i1)
    blocks = torch.tensor([[0, 1, 0, 0]], dtype=I32, device="cuda")
    wp = c.prefill_attention(want, blocks)
    no_error(kv4)
    for width, stride in ((W + 4, W + 4), (W, W + 3), (W, 1), (W, W)):
        c = kv4.KV4Cache(1, nkv, hd, 20)
        base = torch.full((2 * W + 64,), 5.0, dtype=BF, device="cuda")
        qkv = torch.as_strided(base, (1, width), (stride, 1))
        qkv[:, :W] = x.cuda()
        q = c.store(qkv, i0, i0, nq=nq)
        kv = torch.full((2 * W + 64,), 5.0, dtype=BF, device="cuda")
        k = torch.as_strided(kv, (1, nkv, hd), (stride, hd, 1))
        gk, gv = c.load(i0, i0, k=k)
        big = torch.full((2 * W + 64,), 5.0, dtype=BF, device="cuda")
        out = torch.as_strided(big, (1, Q), (stride, 1))
        qrow = torch.as_strided(base.clone(), (1, Q), (stride, 1))
        qrow.copy_(q)
        o = c.attention(qrow, i1, out=out).clone()
        p = c.prefill_attention(qrow, blocks, out=out)
        no_error(kv4)
        assert torch.equal(q, want) and torch.equal(gk, wk) and torch.equal(gv, wv)
        assert torch.equal(o, wo) and torch.equal(p, wp)
        assert bool((big[Q:] == 5).all()) and bool((kv[nkv * hd:] == 5).all()) and bool((base[W:] == 5).all())
        # in place
        assert c.store(qkv, i0, i0, nq=nq, q=qkv[:, :Q]).data_ptr() == base.data_ptr()
        no_error(kv4)
        assert torch.equal(base[:Q], want[0]) and torch.equal(base[Q:W], x[0, Q:].cuda()) and bool((base[W:] == 5).all())


# ------------------------------------------------------------------------------------------------- the bytes
def codes_and_scales(c, n):
    """Codes and scales of positions [0, n) of cache row 0, layer 0, read off the buffer by the layout in csrc/kv4.cu's head
    comment: float64 [n, 2, nkv, hd] and [n, 2, nkv, hd / 32]."""
    hd, nkv = c.hd, c.nkv
    G = hd // 32
    buf = c.buf.cpu().view(-1, 18 * hd)[:nkv * -(-c.cache_len // 16)].view(nkv, -1, 18 * hd)
    slot = {64: [0, 1], 128: [0, 2, 1, 3]}[hd]                   # of group g
    code, scale = torch.zeros(n, 2, nkv, hd), torch.zeros(n, 2, nkv, G)
    for p in range(n):
        rec, j = buf[:, p // 16], p % 16
        i, t = [(i, t) for i in range(4) for t in range(4) if j == 4 * i + (t ^ 3 if i % 2 else t)][0]
        sw = 4 * (j >> 1 & 1) if hd == 128 else 0
        for g in range(G):
            for d in range(32):
                word = j * (hd // 2) + ((d // 8) * G + slot[g]) * 4 + (d % 8) // 2
                half = 8 * hd + j * (hd // 2) + (((d // 4) ^ sw) * G + slot[g]) * 2 + (d % 4) // 2
                for kv, byte in enumerate((word, half)):
                    code[p, kv, :, 32 * g + d] = ((rec[:, byte].int() >> (4 * (d % 2))) & 15).float() - 8
            for kv in range(2):
                at = (16 + kv) * hd + ((4 * t + i) * G + slot[g]) * 2
                scale[p, kv, :, g] = rec[:, at:at + 2].contiguous().view(BF)[:, 0].float()
    return code.double(), scale.double()


@pytest.mark.parametrize("hd", [64, 128])
def test_bytes_are_the_documented_layout(kv4, hd):
    n, nkv = 37, 2
    x = rnd(30, n, 2, nkv, hd)
    x[3, 0, 1, 32:64] = 0
    x[5, 1, 0, :32] *= 2.0 ** -110
    x[7, 0, 0, 40] = float("nan")
    c = one_row(kv4, x, hd)
    no_error(kv4)
    code, scale = codes_and_scales(c, n)
    want, s = R.quantise(x)
    assert torch.equal(code, want.flatten(-2))
    assert torch.equal(scale.isnan(), s.isnan()) and torch.equal(scale.nan_to_num(), s.nan_to_num())


@pytest.mark.parametrize("e", [0, 119, -92, -93, -94, -97, -101, -120])
def test_quantiser_decides_every_quotient(kv4, e):
    """Every 8-bit significand of a group's largest (times 2^e, e to either side of where the scale's range is shifted, and the
    largest and smallest there are) against every bf16 number within 2^-6 of it, both signs: codes as 64 bits give them."""
    hd, rows = 128, 512
    mags = torch.arange(128, 256).double()
    rest = torch.cat([mags * 2.0 ** -k for k in range(7)])           # against a largest of 128 .. 255
    rest = torch.cat([rest, -rest])
    groups = []
    for m in mags.tolist():
        r = rest[rest.abs() <= m]
        r = torch.cat([r, torch.zeros(-len(r) % 31, dtype=torch.float64)]).view(-1, 31)
        top = torch.full((len(r), 1), m, dtype=torch.float64)
        top[::2] *= -1
        groups.append(torch.cat([r[:, :13], top, r[:, 13:]], 1))
    x = torch.cat(groups) * 2.0 ** (e - 7 if e < 119 else e)         # (the largest: 255 x 2^119, the next to infinity's 2^127)
    x = torch.cat([x, torch.zeros(-len(x) % 8, 32, dtype=torch.float64)]).view(-1, 2, 1, hd)
    x = x.float().to(BF)
    for part in x.split(rows):
        c = one_row(kv4, part, hd)
        k, v = c.load(torch.arange(len(part), dtype=I32, device="cuda"), torch.zeros(len(part), dtype=I32, device="cuda"))
        no_error(kv4)
        want = R.values(part)
        for got, w in ((k, want[:, 0]), (v, want[:, 1])):
            assert torch.equal(got.cpu().double(), w.to(BF).double())


# ------------------------------------------------------------------------------------------------- keys behind a row
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", [0, 1])
def test_prompt_and_a_large_key_behind_a_row(kv4, hd, which):
    """A key or value far above the others, late in a 64-key tile: rows before it, which do not attend it, keep every bit, the
    others are within their bound."""
    n, nq, nkv, at = 128, 4, 2, 60
    x, q = rnd(31, n, 2, nkv, hd), rnd(32, n, nq * hd)
    clean = prompt(kv4, one_row(kv4, x, hd), q, n)
    for up in (10, 18, 22):
        y = x.clone()
        y[at, which] = (y[at, which].float() * 2.0 ** up).to(BF)
        got = prompt(kv4, one_row(kv4, y, hd), q, n)
        assert torch.equal(got[:at], clean[:at])
        check_prompt(kv4, y, q, hd)


@pytest.mark.parametrize("hd", [64, 128])
def test_logits_of_a_million(kv4, hd):
    """Logits up to about 2^20: finite, and one key takes the row."""
    n, nq, nkv = 100, 4, 2
    x, q = rnd(33, n, 2, nkv, hd), rnd(34, n, nq * hd)
    x[:, 0] = (x[:, 0].float() * 2.0 ** 9).to(BF)
    q = (q.float() * 2.0 ** 9).to(BF)
    c = one_row(kv4, x, hd)
    got = prompt(kv4, c, q, n)
    lens = torch.arange(1, n + 1, dtype=I32, device="cuda")
    dec = c.attention(q.cuda(), lens, torch.zeros(n, dtype=I32, device="cuda")).cpu().double()
    no_error(kv4)
    kv, qd = R.values(x), q.double().view(n, nq, hd)
    for h in range(nq):
        z = (qd[:, h] @ kv[:, 0, h * nkv // nq].T * hd ** -0.5)
        z = z.masked_fill(torch.arange(n)[None] > torch.arange(n)[:, None], float("-inf"))
        top = z.topk(min(2, n), -1).values
        sure = (top[:, 0] - top[:, 1]) > 2.0 ** -10 * top[:, 0].abs() + 40     # (far above any rounding of a logit)
        best = kv[:, 1, h * nkv // nq][z.argmax(-1)]
        for o in (got, dec):
            o = o.view(n, nq, hd)[:, h]
            assert bool(o.isfinite().all())
            assert bool(((o - best).abs() <= 2.0 ** -7 * best.abs())[sure].all()) and int(sure.sum()) > n // 2


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("pos0", [0, 37])
def test_prompt_rows_do_not_depend_on_keys_behind_them(kv4, hd, which, pos0):
    """However large a key or value is that a row does not attend, the row keeps every bit: within a tile, in a block over two
    tiles, among zeros, with an infinity."""
    n, nq, nkv, at = 64, 4, 2, pos0 + 43
    S = pos0 + n
    x, q = rnd(35, S, 2, nkv, hd), rnd(36, n, nq * hd)
    blocks = torch.tensor([[0, n, 0, pos0]], dtype=I32, device="cuda")

    def run(y):
        out = one_row(kv4, y, hd).prefill_attention(q.cuda(), blocks)
        no_error(kv4)
        return out.cpu()[:at - pos0]
    for thin in (False, True):
        x = x.clone()
        if thin:                                          # (the tile's own exponent is then the large key's alone)
            x[at // 64 * 64:at] = 0
            x[at + 1:] = 0
        clean = run(x)
        assert bool(clean.isfinite().all())
        for up in (10, 16, 18, 22, 40, 60, 100, 120, float("inf")):
            y = x.clone()
            y[at, which] = (y[at, which].float().clamp(-2, 2) * 2.0 ** up).to(BF)
            assert torch.equal(run(y), clean), up


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_with_keys_and_values_of_every_size(kv4, hd):
    """Scales over 2^40 within a tile, in any order."""
    n, nq, nkv = 200, 4, 2
    g = torch.Generator().manual_seed(37)
    x, q = rnd(38, n, 2, nkv, hd), rnd(39, n, nq * hd)
    x[:, 0] *= (2.0 ** torch.randint(-40, 3, (n,), generator=g).float()).to(BF)[:, None, None]
    x[:, 1] *= (2.0 ** torch.randint(-20, 21, (n,), generator=g).float()).to(BF)[:, None, None]
    check_prompt(kv4, x, q, hd)
