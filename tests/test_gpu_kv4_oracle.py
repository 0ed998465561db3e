"""An engine on a 4-bit cache against the CPU oracle engine whose slow stack keeps what the 4-bit cache keeps: admission behind
cached voice prefixes, a continuation, and ticks.

How far they may differ. The engine's keys and values are the oracle's up to a step of bf16 here and there (2^-8 of the value, up to
7 scales: 0.03 of a code's step), so about 3 % of those elements land on the next code, a step (a scale) away. Taking a fifth of
all elements to differ by a step of bf16, 0.6 % of the codes differ by one, a noise of sqrt(0.006) = 0.08 scales against the
quantisation's own 0.29. What the quantisation as a whole does to the last hidden rows of this stand-in is about 0.11 of their
largest; the flips' share is 0.03, and twice that is allowed.

Later layers' keys and values start from hidden rows that differ by that: by e of themselves they move e x rms, a group's rms being
about 7 / 2.2 = 3.2 scales (its largest of 32 normal ones is 2.2 rms), and a shift of d scales changes a share d of the codes, on
average over a normal shift 0.8 of its rms: 0.8 x 3.2 e, 8 % of them at e = 0.03 and 16 % at the 0.06 allowed."""
import pytest
import torch

from oracle import kv4_ref
from oracle import ref_cpu as R
from oracle.standin import StubTokenizer
from test_gpu_engine import _requests, rel

pytestmark = pytest.mark.gpu
S = 512


@pytest.fixture(scope="module")
def dev(a8):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    a8.load()
    a8._lib.call("a8_clear_error")
    return torch.device("cuda", 0)


@pytest.fixture()
def four_bit_oracle(monkeypatch):
    """The oracle's slow stack (its cache is S long) keeps code * scale of what it stores."""
    store = R.bias_rope_store

    def quantised(qkv, bias, cos, sin, pos, slot, kc, vc, *a, **kw):
        q = store(qkv, bias, cos, sin, pos, slot, kc, vc, *a, **kw)
        if kc.shape[2] == S:
            for c in (kc, vc):
                x = c[slot.long(), :, pos.long()]
                c[slot.long(), :, pos.long()] = kv4_ref.values(x.to(torch.bfloat16)).float()
        return q
    monkeypatch.setattr(R, "bias_rope_store", quantised)


def same_cache(eng, ora, row, n):
    """Keys and values of a row's first n positions: nearly all the oracle's, the others one code away."""
    pos = torch.arange(n, dtype=torch.int32, device=eng.dev)
    for l in range(eng.slow.layers):
        got = eng.slow.kv4.load(pos, torch.full_like(pos, row), layer=l)
        for g, c in zip(got, (ora.slow.kc, ora.slow.vc)):
            g, w = g.float().cpu(), c[l, row, :, :n].transpose(0, 1)
            step = w.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2) / 7
            d = (g - w).abs()
            assert float((d > 0.5 * step).float().mean()) < (0.03 if l == 0 else 0.16), (l, row)
            if l == 0:
                assert bool((d <= 1.1 * step + 1e-6).all()), row


def test_engine_matches_an_oracle_with_a_four_bit_cache(a8, dev, tiny_model, four_bit_oracle):
    gp = dict(do_sample=False, temperature=0.8, top_k=50, top_p=0.95, max_new_tokens=64)
    eng = a8.FastEngine(tiny_model, StubTokenizer(), gp, max_slots=3, max_seq=S, buckets=[1, 2, 3], seq_from_env=False,
                        seed=31, kv_bits=4)
    ora = R.OracleEngine(tiny_model, StubTokenizer(), gp, max_slots=3, max_seq=S, seed=31, with_voc=False)
    first = _requests(4)
    g = torch.Generator().manual_seed(8)
    cont = [dict(first[0], ctx_text="12 34 56", ctx_codes=torch.randint(0, 4096, (6, eng.ncg), generator=g)),
            dict(first[1], ctx_text="78 90")]
    for reqs in (first[:2], cont):                       # plain, then over the same rows with context
        lens = eng.admit([0, 1], reqs)
        assert lens == ora.admit([0, 1], reqs)
        torch.cuda.synchronize()
        assert a8.device_error()[0] == 0
        assert torch.equal(eng.cpos[:2].cpu(), ora.cpos[:2])
        for s in range(2):
            same_cache(eng, ora, s, lens[s])
        assert rel(eng.hid[:2], ora.hid[:2]) < 0.06
    # decode: the engine's own codes through the oracle's slow step, at the engine's positions
    for t in range(3):
        pos, tok = eng.cpos[:2].cpu().clone(), eng.tok[:2].cpu().clone()
        eng.tick(2)
        torch.cuda.synchronize()
        assert a8.device_error()[0] == 0
        h = ora.slow.forward(ora.embed(tok, eng.codes[:2].cpu()), pos, torch.arange(2, dtype=torch.int32), pos + 1,
                             rowmap=False)
        assert rel(eng.hid[:2], h) < 0.06, t
        for s in range(2):
            same_cache(eng, ora, s, int(pos[s]) + 1)
