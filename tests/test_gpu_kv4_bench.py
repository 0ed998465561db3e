"""The benchmark and the smoke run with TTS_KV_BITS=4 set."""
import sys

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(a8):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    a8.load()
    a8._lib.call("a8_clear_error")
    return torch.device("cuda", 0)


def test_smoke_runs_with_four_bits_set(a8, dev, monkeypatch):
    monkeypatch.setenv("TTS_KV_BITS", "4")
    sys.path.insert(0, REPO)
    import __graft_entry__ as G
    from oracle import ref_cpu as R
    G._smoke_tick(a8, R, dev, torch.Generator().manual_seed(7))


@pytest.mark.parametrize("bits", [16, 4])
def test_bench_fills_either_cache(a8, dev, tiny_model, bits):
    """Every position of the rows asked for is random, the next row is untouched; the config names a cache that is not bf16."""
    sys.path.insert(0, REPO)
    import bench
    from audio8_b200.engine import PackedStack
    c = tiny_model.config
    st = PackedStack(tiny_model.layers, tiny_model.norm, c.n_head, c.n_local_heads, c.head_dim, c.norm_eps, c.rope_base,
                     cache_rows=3, cache_len=50, max_pos=64, dev=dev, kv_bits=bits)
    bench.fill_slow(st, torch.Generator(device=dev).manual_seed(3), 2)
    torch.cuda.synchronize()
    assert a8.device_error()[0] == 0
    pos = torch.arange(50, dtype=torch.int32, device=dev)
    for l in range(st.layers):
        for row in range(3):
            if bits == 4:
                kv = st.kv4.load(pos, torch.full_like(pos, row), layer=l)
            else:
                kv = (st.kc[l, row].transpose(0, 1), st.vc[l, row].transpose(0, 1))
            for t in kv:
                std = t.float().std(-1)
                assert bool((std > 0.5).all() if row < 2 else (std == 0).all())
    assert bench.with_cache({"model": "m"}, st) == ({"model": "m"} if bits == 16 else {
        "model": "m", "kv_cache": "slow AR in 4 bits (4.5 with scales, 9 / 32 of a bf16 cache)"})
