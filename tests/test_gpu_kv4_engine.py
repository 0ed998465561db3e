"""The slow stack and the engine on a 4-bit key/value cache: a8_stack_forward is, bit for bit, the sequence of the public
calls it is made of; admission (graphs, the voices' cached prefixes) and ticks run on it as they do on a bf16 cache."""
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from oracle.standin import StubTokenizer

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def dev(a8):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    a8.load()
    a8._lib.call("a8_clear_error")
    return torch.device("cuda", 0)


def stacks(a8, model, dev, **kw):
    from audio8_b200.engine import PackedStack, Scratch
    c = model.config
    st = PackedStack(model.layers, model.norm, c.n_head, c.n_local_heads, c.head_dim, c.norm_eps, c.rope_base,
                     cache_rows=4, cache_len=250, max_pos=256, dev=dev, kv_bits=4, **kw)
    sc = Scratch(256, c.dim, c.n_head * c.head_dim, c.intermediate_size, c.n_local_heads, c.head_dim, 250, dev, st.kv4)
    return st, sc


def by_calls(a8, st, sc, x, pos, slot, lens, blocks):
    """a8_stack_forward's calls one by one: (final-normed rows)."""
    L, kv4 = a8._lib, st.kv4
    n, D, s = x.shape[0], st.dim, L.stream_handle()
    N = (st.nq + 2 * st.nkv) * st.hd
    new = lambda w: torch.empty(n, w, dtype=BF, device=x.device)
    h, a, m = new(D), new(D), new(st.inter)
    norm = lambda src, res, w: L.call("a8_rmsnorm", L.ptr(src), D, L.ptr(res), D, L.ptr(w), L.ptr(h), D, n, D, st.eps, s)

    def gemm(src, w, out, **kw):
        e = L.A8Epilogue(**kw)
        L.call("a8_gemm", L.ptr(src), src.shape[1], L.ptr(w), w.shape[0], w.shape[1], n, L.ptr(out), out.shape[1],
               C.byref(e), 0, s)
    norm(x, None, st.ln1[0])
    for l in range(st.layers):
        qkv = new(N)
        if l == 0:
            gemm(h, st.wqkv[l], qkv, kind=L.EPI_BF16, bias=L.ptr(st.bqkv[l]))
        else:
            gemm(x, st.wqkv[l], qkv, kind=L.EPI_BF16, bias=L.ptr(st.bqkv[l]), norm_w=L.ptr(st.ln1[l]),
                 ssq_in=L.ptr(sc.ssq), ssq_ld=sc.rows, eps=st.eps)
        q = kv4.store(qkv, pos, slot, layer=l, nq=st.nq, cos=st.cos, sin=st.sin)
        o = kv4.prefill_attention(q, blocks, layer=l) if blocks is not None else \
            kv4.attention(q, lens, slot, layer=l, max_len=250)
        gemm(o, st.wo[l], a, kind=L.EPI_BF16)
        norm(a, x, st.ln2[l])
        gemm(h, st.w13[l], m, kind=L.EPI_SILU)
        gemm(m, st.w2[l], x, kind=L.EPI_RESID, res=L.ptr(x), ldres=D, ssq_out=L.ptr(sc.ssq), ssq_ld=sc.rows)
    norm(x, None, st.norm)
    return h


def test_stack_forward_is_its_calls(a8, dev, tiny_model):
    from audio8_b200.engine import FastEngine
    L = a8._lib
    st, sc = stacks(a8, tiny_model, dev)
    other, sc2 = stacks(a8, tiny_model, dev)
    assert st.kc is None and st.kv4.nbytes == 2 * 4 * 2 * 16 * 18 * 64
    g = torch.Generator().manual_seed(1)
    ns, slots = [70, 20, 133], [1, 3, 0]
    pos = torch.cat([torch.arange(n, dtype=I32) for n in ns])
    slot = torch.cat([torch.full((n,), s, dtype=I32) for n, s in zip(ns, slots)])
    blk = torch.from_numpy(FastEngine.query_blocks(pos.numpy(), slot.numpy())).to(dev)
    P, S = pos.to(dev), slot.to(dev)
    x = (torch.randn(sum(ns), st.dim, generator=g) * 0.1).to(BF)

    def run(X, P, S, rows, lens, blocks):
        r = L.A8StackRun(x=L.ptr(X), ldx=st.dim, rows=rows, pos=L.ptr(P), slot=L.ptr(S), lens=L.ptr(lens), lens_max=0,
                         rowmap=L.ptr(S), max_len=0, scratch=sc.desc, blocks=L.ptr(blocks),
                         nblocks=0 if blocks is None else blocks.shape[0])
        L.call("a8_stack_forward", C.byref(st.desc), C.byref(r), L.stream_handle())
        return sc.h[:rows]
    X, Y = x.to(dev), x.to(dev)
    got = run(X, P, S, len(pos), None, blk).clone()
    want = by_calls(a8, other, sc2, Y, P, S, None, blk)
    torch.cuda.synchronize()
    assert a8.device_error()[0] == 0
    assert torch.equal(got, want) and torch.equal(X, Y) and torch.equal(st.kv4.buf, other.kv4.buf)
    # decode rows on what that left, keys counted from the positions (lens NULL) and given
    for t in range(3):
        dp = torch.tensor([70 + t, 20 + t, 133 + t], dtype=I32, device=dev)
        ds = torch.tensor(slots, dtype=I32, device=dev)
        dl = (dp + 1).contiguous()
        x = (torch.randn(3, st.dim, generator=g) * 0.1).to(BF)
        X, Y = x.to(dev), x.to(dev)
        got = run(X, dp, ds, 3, dl if t == 1 else None, None).clone()
        want = by_calls(a8, other, sc2, Y, dp, ds, dl, None)
        torch.cuda.synchronize()
        assert a8.device_error()[0] == 0
        assert torch.equal(got, want) and torch.equal(st.kv4.buf, other.kv4.buf), t


def test_stack_refusals(a8, dev, tiny_model):
    """An MLP too narrow for the q, k and v rows; query blocks with a ring."""
    L = a8._lib
    st, sc = stacks(a8, tiny_model, dev)
    d = L.A8StackDesc.from_buffer_copy(st.desc)
    d.inter = 1088                                       # below the 1,152 columns of q, k and v
    x = torch.zeros(1, st.dim, dtype=BF, device=dev)
    p = torch.zeros(1, dtype=I32, device=dev)
    r = L.A8StackRun(x=L.ptr(x), ldx=st.dim, rows=1, pos=L.ptr(p), slot=None, lens=None, lens_max=0, rowmap=None,
                     max_len=0, scratch=sc.desc, blocks=None, nblocks=0)
    assert L.load().a8_stack_forward(C.byref(d), C.byref(r), L.stream_handle()) == 4        # A8_ERR_SIZE
    d = L.A8StackDesc.from_buffer_copy(st.desc)
    d.ring = 64
    b = torch.zeros(1, 4, dtype=I32, device=dev)
    r.blocks, r.nblocks = L.ptr(b), 1
    assert L.load().a8_stack_forward(C.byref(d), C.byref(r), L.stream_handle()) == 1        # A8_ERR_ARG
    torch.cuda.synchronize()


def requests(seed, n, keys=2):
    g = torch.Generator().manual_seed(seed)
    voice = lambda i: SimpleNamespace(ref_code=torch.randint(0, 4096, (20 + 7 * i, 10), generator=g),
                                      ref_text="12 34 56 78")
    voices = [voice(i) for i in range(keys)]
    return [dict(text=" ".join(str(int(x)) for x in torch.randint(100, 900, (4 + 3 * i,), generator=g)),
                 item=voices[i % keys], key=f"v{i % keys}") for i in range(n)]


@pytest.fixture()
def four_bits(monkeypatch):
    monkeypatch.setenv("TTS_KV_BITS", "4")


def rows_of(eng, slot, n):
    """Every layer's keys and values of a cache row's first n positions."""
    pos = torch.arange(n, dtype=I32, device=eng.dev)
    s = torch.full((n,), slot, dtype=I32, device=eng.dev)
    return [t for l in range(eng.slow.layers) for t in eng.slow.kv4.load(pos, s, layer=l)]


def test_engine_admits_and_ticks_on_four_bits(a8, dev, tiny_model, four_bits):
    """Graphs and eager launches leave the same state; a slot's prefix is the voice's; a second admission of the same
    request (its prefix from the kept blob) writes the same cache; ticks advance every row."""
    gp = dict(do_sample=True, temperature=0.8, top_k=50, top_p=0.95)
    mk = lambda: a8.FastEngine(tiny_model, StubTokenizer(), gp, max_slots=4, max_seq=300, buckets=[4],
                               seq_from_env=False, seed=21)
    eager, graphed = mk(), mk()
    assert eager.slow.kv4 is not None and eager.slow.kc is None and eager.fast.kv4 is None
    graphed.capture(log=lambda *a: None)
    reqs = requests(4, 4)
    for eng in (eager, graphed):
        lens = eng.admit([0, 1, 2, 3], reqs)
        assert all(n > 0 for n in lens)
    torch.cuda.synchronize()
    assert a8.device_error()[0] == 0
    for name in ("tok", "hid", "cpos", "prev", "nstep", "frame_prev"):
        assert torch.equal(getattr(eager, name), getattr(graphed, name)), name
    for s in range(4):
        for x, y in zip(rows_of(eager, s, lens[s]), rows_of(graphed, s, lens[s])):
            assert torch.equal(x, y) and bool(torch.isfinite(x.float()).all())
    # rows 0 and 2 have one voice: the same prefix, position for position
    Lp = eager._pkv["v0"].Lp
    for x, y in zip(rows_of(eager, 0, Lp), rows_of(eager, 2, Lp)):
        assert torch.equal(x, y)
    before = rows_of(eager, 1, lens[1])
    eager.admit([3], [reqs[1]])
    for x, y in zip(rows_of(eager, 3, lens[1]), before):
        assert torch.equal(x, y)
    # ticks
    eager.admit([3], [reqs[3]])
    eager.tick_ctr.copy_(graphed.tick_ctr)
    for name in ("tok", "hid", "prev", "nstep", "frame_prev"):
        getattr(eager, name).copy_(getattr(graphed, name))
    for t in range(4):
        eager.tick(4)
        graphed.replay(4)
        torch.cuda.synchronize()
        assert a8.device_error()[0] == 0
        assert torch.equal(eager.tok[:4], graphed.tok[:4]) and torch.equal(eager.hid[:4], graphed.hid[:4]), t
        assert torch.equal(eager.audio, graphed.audio), t
        assert eager.cpos[:4].tolist() == [n + t + 1 for n in lens]


def test_engine_refuses_other_widths(a8, dev, tiny_model, monkeypatch):
    monkeypatch.setenv("TTS_KV_BITS", "8")
    with pytest.raises(a8.A8Error):
        a8.FastEngine(tiny_model, StubTokenizer(), dict(), max_slots=2, max_seq=128, buckets=[2], seq_from_env=False)
