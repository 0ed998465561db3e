"""The 4-bit cache on the CPU: its size rule, the argument checks of its entry points (nothing is launched), the oracle's
own properties, and the layout the kernels write, checked against the header comment of csrc/kv4.cu."""
import ctypes as C
import os
import re

import pytest
import torch

from conftest import REPO
from oracle import kv4_ref as R

ARG, ALIGN, SIZE, OK = 1, 3, 4, 0


@pytest.fixture(scope="module")
def L(a8):
    a8.load()
    return a8._lib


def desc(L, buf=256, layers=2, cache_rows=3, nkv=2, hd=64, cache_len=100):
    return L.A8KV4(buf, layers, cache_rows, nkv, hd, cache_len)


@pytest.mark.parametrize("shape", [(1, 1, 1, 64, 1), (2, 3, 2, 64, 100), (24, 1537, 2, 64, 2048), (1, 3, 8, 128, 131072),
                                   (80, 256, 8, 128, 131072)])
def test_bytes(L, shape):
    layers, rows, nkv, hd, n = shape
    want = layers * rows * nkv * -(-n // 16) * 18 * hd
    assert L.load().a8_kv4_bytes(C.byref(L.A8KV4(None, *shape))) == want
    assert want == layers * rows * nkv * -(-n // 16) * 16 * 2 * (hd // 2 + hd // 32 * 2)     # codes and scales, K and V


@pytest.mark.parametrize("shape", [(0, 1, 1, 64, 1), (1, 0, 1, 64, 1), (1, 1, 0, 64, 1), (1, 1, 1, 96, 1),
                                   (1, 1, 1, 64, 0), (1, 1, 1, 64, -5), (1, 1, 1, 64, (1 << 30) + 1),
                                   (1 << 30, 1 << 30, 4, 64, 1 << 20)])
def test_bytes_refused(L, shape):
    assert L.load().a8_kv4_bytes(C.byref(L.A8KV4(None, *shape))) == -1


def test_struct_matches_header(L, tmp_path):
    import shutil
    import subprocess
    body = re.search(r"typedef struct A8KV4 \{(.*?)\} A8KV4;", open(os.path.join(REPO, "include", "audio8_b200.h")).read(),
                     flags=re.S).group(1)
    names = [f.strip(" *") for d in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";") if d.strip()
             for f in re.sub(r"^\s*(void|int)\s*", "", d.strip()).split(",")]
    assert names == [f[0] for f in L.A8KV4._fields_]
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "audio8_b200.h"\nint main(void){printf("%zu %zu",'
                   'sizeof(A8KV4), offsetof(A8KV4, cache_len));return 0;}')
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == [C.sizeof(L.A8KV4), L.A8KV4.cache_len.offset]


def p(n=256):
    return C.c_void_p(n)


def test_store_refusals(L):
    lib, N = L.load(), None

    def store(d=None, layer=0, qkv=p(), ld=18 * 64, nq=14, cos=p(), sin=p(), npos=100, pos=p(), slot=N, rows=4, ring=0,
              q=p(), ldq=14 * 64):
        return lib.a8_kv4_store(C.byref(d if d is not None else desc(L)), layer, qkv, ld, nq, cos, sin, npos, pos, slot,
                                rows, ring, q, ldq, N)
    assert lib.a8_kv4_store(N, 0, p(), 18 * 64, 14, N, N, 0, p(), N, 4, 0, p(), 14 * 64, N) == ARG
    for kw in (dict(d=desc(L, buf=None)), dict(d=desc(L, hd=80)), dict(d=desc(L, cache_len=0)), dict(layer=2),
               dict(layer=-1), dict(qkv=N), dict(pos=N), dict(rows=0), dict(rows=-3), dict(nq=-1), dict(q=N),
               dict(cos=N), dict(sin=N), dict(npos=0), dict(ld=18 * 64 - 8), dict(ldq=14 * 64 - 8), dict(ring=-1),
               dict(ring=101)):
        assert store(**kw) == ARG, kw
    for kw in (dict(d=desc(L, buf=264)), dict(qkv=p(258)), dict(ld=18 * 64 + 4), dict(q=p(264)), dict(ldq=14 * 64 + 4),
               dict(cos=p(264)), dict(sin=p(264))):
        assert store(**kw) == ALIGN, kw
    assert store(d=desc(L, layers=1 << 30, cache_rows=1 << 20, cache_len=1 << 20)) == SIZE
    assert store(rows=(1 << 31) - 1, nq=1 << 20, ld=(1 << 31) - 8, ldq=(1 << 31) - 8) == SIZE


def test_load_refusals(L):
    lib, N = L.load(), None

    def load(d=None, layer=0, pos=p(), slot=N, rows=4, k=p(), ldk=128, v=p(), ldv=128):
        return lib.a8_kv4_load(C.byref(d if d is not None else desc(L)), layer, pos, slot, rows, k, ldk, v, ldv, N)
    for kw in (dict(d=desc(L, buf=None)), dict(layer=2), dict(pos=N), dict(rows=0), dict(k=N, v=N), dict(ldk=120),
               dict(ldv=120)):
        assert load(**kw) == ARG, kw
    for kw in (dict(k=p(258)), dict(v=p(264)), dict(ldk=132), dict(ldv=132)):
        assert load(**kw) == ALIGN, kw


def test_attention_refusals(L):
    lib, N = L.load(), None

    def attn(d=None, layer=0, q=p(), qs=896, nq=14, lens=p(), rowmap=N, rows=4, max_len=100, scale=0.0, out=p(), os_=896,
             ws=p(), nws=1 << 40, cnt=p(), ncnt=1 << 30):
        return lib.a8_kv4_attention(C.byref(d if d is not None else desc(L)), layer, q, qs, nq, lens, rowmap, rows,
                                    max_len, scale, out, os_, ws, nws, cnt, ncnt, N)
    for kw in (dict(d=desc(L, buf=None)), dict(d=desc(L, hd=32)), dict(layer=2), dict(q=N), dict(lens=N), dict(out=N),
               dict(rows=0), dict(nq=0), dict(nq=15), dict(nq=34, qs=34 * 64, os_=34 * 64), dict(max_len=0),
               dict(max_len=101), dict(qs=888), dict(os_=888), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attn(**kw) == ARG, kw
    for kw in (dict(q=p(258)), dict(out=p(264)), dict(qs=900), dict(os_=900), dict(d=desc(L, buf=260))):
        assert attn(**kw) == ALIGN, kw
    n, t = C.c_longlong(), C.c_int()
    assert lib.a8_kv4_attention_workspace(C.byref(desc(L)), 14, 4, 100, C.byref(n), C.byref(t)) == OK
    assert n.value >= 0 and t.value >= 0
    if n.value > 0:
        assert attn(nws=n.value - 1) == SIZE and attn(ws=N) == SIZE
    if t.value > 0:
        assert attn(ncnt=t.value - 1) == SIZE and attn(cnt=N) == SIZE
    for bad in ((15, 4, 100), (0, 4, 100), (14, 0, 100), (14, 4, 0), (14, 4, 101), (34, 4, 100)):
        assert lib.a8_kv4_attention_workspace(C.byref(desc(L)), *bad, C.byref(n), C.byref(t)) == ARG, bad


def test_prefill_attention_refusals(L):
    lib, N = L.load(), None

    def pf(d=None, layer=0, q=p(), qs=896, nq=14, blocks=p(), nb=1, rows=4, scale=0.0, out=p(), os_=896):
        return lib.a8_kv4_prefill_attention(C.byref(d if d is not None else desc(L)), layer, q, qs, nq, blocks, nb, rows,
                                            scale, out, os_, N)
    for kw in (dict(d=desc(L, buf=None)), dict(layer=2), dict(q=N), dict(blocks=N), dict(nb=0), dict(out=N), dict(rows=0),
               dict(nq=15), dict(nq=34, qs=34 * 64, os_=34 * 64), dict(qs=888), dict(os_=888),
               dict(scale=float("nan"))):
        assert pf(**kw) == ARG, kw
    for kw in (dict(q=p(258)), dict(out=p(264)), dict(qs=900), dict(os_=900)):
        assert pf(**kw) == ALIGN, kw


def test_python_refuses_cpu_and_shapes(a8):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(a8.A8Error):
        a8.KV4Cache(1, 1, 96, 16, dev="cpu")             # hd
    c = a8.KV4Cache(2, 2, 64, 40, dev="cpu")             # memory only: the checks below run before any launch
    assert c.nbytes == 2 * 2 * 3 * 18 * 64
    x = torch.zeros(3, 18 * 64, dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    for f in (lambda: c.store(x.float(), i, nq=14), lambda: c.store(x[:, :64], i, nq=14),
              lambda: c.store(x.t(), i, nq=14), lambda: c.store(x[:2], i, nq=14),
              lambda: c.store(x, i.long(), nq=14), lambda: c.store(x, i, torch.zeros(2, dtype=torch.int32), nq=14),
              lambda: c.store(x, i, nq=14, cos=torch.zeros(4, 64, dtype=torch.bfloat16)),
              lambda: c.store(x, i, nq=14, sin=torch.zeros(4, 64, dtype=torch.bfloat16)),
              lambda: c.load(i, k=torch.zeros(3, 2, 128, dtype=torch.bfloat16)),
              lambda: c.attention(x[:, :100], i), lambda: c.attention(x[:, :896].contiguous(), i[:2]),
              lambda: c.prefill_attention(x[:, :896].contiguous(), torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(a8.A8Error):
            f()


# ------------------------------------------------------------------------------------------------- the oracle itself
def test_quantise_decides_exactly():
    """rint(x / s) in fp32 and in 64 bits agree for every bf16 x against scales that put x near the borders."""
    x = torch.arange(0x3F80, 0x4100, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)       # [1, 8)
    s = torch.arange(0x3E80, 0x3F90, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    q32 = torch.round(x.float()[:, None] / s.float()[None, :])
    q64 = torch.round(x.double()[:, None] / s.double()[None, :])
    assert torch.equal(q32.double(), q64)


def test_quantise_error_and_extremes():
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(50, 128, generator=g) * 10.0 ** (torch.rand(50, 1, generator=g) * 60 - 30)).to(R.BF)
    c, s = R.quantise(x)
    assert c.abs().max() == 7
    # half a step (s) away at most, and the scale's own rounding moves the largest by 7 2^-9 s more
    err = (x.double().unflatten(-1, (-1, 32)) - c * s[..., None]).abs()
    assert bool((err <= (0.5 + 7 * 2.0 ** -8) * s[..., None]).all())
    z = torch.zeros(1, 64, dtype=R.BF)
    assert torch.equal(R.values(z), z.double())
    z[0, 3] = float("inf")
    assert R.values(z).isnan().tolist() == [[True] * 32 + [False] * 32]


def test_record_layout_is_a_permutation():
    """Every byte of a record belongs to one (K / V, position, dim pair) or one scale; read off the kernel source's own
    index functions, restated here."""
    for hd in (64, 128):
        G = hd // 32
        slot = lambda g: (g % (G // 2)) * 2 + g // (G // 2)
        vsw = lambda j: ((j >> 1) & 1) * 4 if G == 4 else 0
        seen = set()
        for j in range(16):
            i = j >> 2
            t = (j & 3) ^ (3 if i & 1 else 0)
            for g in range(G):
                for t8 in range(4):
                    b = j * (hd // 2) + (t8 * G + slot(g)) * 4
                    seen |= set(range(b, b + 4))
                for q in range(8):
                    b = 8 * hd + j * (hd // 2) + ((q ^ vsw(j)) * G + slot(g)) * 2
                    seen |= set(range(b, b + 2))
                for base in (16 * hd, 17 * hd):
                    b = base + ((t * 4 + i) * G + slot(g)) * 2
                    seen |= set(range(b, b + 2))
        assert len(seen) == 18 * hd and max(seen) == 18 * hd - 1


def test_overlapping_outputs_refused(L):
    lib, N = L.load(), None
    d = C.byref(desc(L))
    # store: q may be qkv itself only with its stride
    assert lib.a8_kv4_store(d, 0, p(), 18 * 64 + 64, 14, N, N, 0, p(4096), N, 4, 0, p(), 14 * 64, N) == ARG
    # attention: in place only with the same stride
    assert lib.a8_kv4_attention(d, 0, p(), 896, 14, p(4096), N, 4, 100, 0.0, p(), 960, p(8192), 1 << 40, p(8192), 1 << 30,
                                N) == ARG
    assert lib.a8_kv4_prefill_attention(d, 0, p(), 896, 14, p(4096), 1, 4, 0.0, p(), 960, N) == ARG
