"""The 4-bit cache's entry points on the CPU: calls at the edges of what their arguments allow. Nothing is launched."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from conftest import REPO

ARG, CUDA, ALIGN, SIZE, OK = 1, 2, 3, 4, 0


@pytest.fixture(scope="module")
def L(a8):
    a8.load()
    return a8._lib


# A8StackDesc as callers of a bf16 cache have it compiled in
STACK = """typedef struct { int layers, dim, nq, nkv, hd, inter; float eps; const void *wqkv, *bqkv, *wo, *w13, *w2, *ln1, *ln2,
*norm, *cos, *sin; void *kc, *vc; int cache_rows, cache_len, ring; } Stack;"""


def test_stack_struct_is_the_bf16_cache_s(L, tmp_path):
    """A 4-bit cache is told by vc NULL, not by a field behind the struct that a caller compiled before it does not have."""
    import shutil
    assert [f[0] for f in L.A8StackDesc._fields_][-3:] == ["cache_rows", "cache_len", "ring"]
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "audio8_b200.h"\n' + STACK + "\nint main(void)"
                   '{printf("%d %d %zu", sizeof(Stack) == sizeof(A8StackDesc), offsetof(Stack, ring) == '
                   'offsetof(A8StackDesc, ring), sizeof(A8StackDesc));return 0;}')
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert out == ["1", "1", str(C.sizeof(L.A8StackDesc))]


def test_stack_refuses_before_it_launches(L):
    """No cache at all; with a 4-bit one, an MLP too narrow for the q, k and v rows, and query blocks with a ring."""
    p = C.c_void_p(256)

    def run(nblocks=0, **kw):
        d = dict(layers=1, dim=896, nq=14, nkv=2, hd=64, inter=4864, eps=1e-6, kc=p, vc=None, cache_rows=1, cache_len=64,
                 ring=0)
        d.update(kw)
        r = L.A8StackRun(x=p, ldx=896, rows=1, pos=p, blocks=p if nblocks else None, nblocks=nblocks)
        before = L.load().a8_launch_count()
        rc = L.load().a8_stack_forward(C.byref(L.A8StackDesc(**d)), C.byref(r), None)
        assert L.load().a8_launch_count() == before
        return rc
    assert run(kc=None) == ARG and run(kc=None, vc=p) == ARG
    assert run(inter=1088) == SIZE
    assert run(ring=32, nblocks=1) == ARG


def test_prompt_kernel_s_registers(tmp_path):
    """The registers that the prompt kernel is compiled to cover what its warpgroups take (one that asks for more than the
    block has waits for good), and the rule by which the host refuses to launch it otherwise."""
    import re
    import shutil
    if shutil.which("nvcc") is None:
        pytest.skip("no CUDA compiler")
    src = tmp_path / "t.cu"
    src.write_text("""#include <stdio.h>
#include "common.cuh"
namespace a8 {
static long long g_launches;
__device__ __forceinline__ uint32_t sw128(int row, int c) { return row * 128 + ((c ^ (row & 7)) << 4); }
}
#include "kv4.cu"
#include "kv4_prefill.cu"
int main() { for (int r : {64, 80, 88, 96, 102}) printf("%d ", a8::kv4p_registers_cover(r)); }
""")
    r = subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-diag-suppress", "177",
                        "-Xptxas", "-v", "-I", os.path.join(REPO, "include"), "-I",
                        os.path.join(REPO, "audio8-turbo-engine_b200", "csrc"), str(src), "-o", str(tmp_path / "t")],
                       capture_output=True, text=True, check=True)
    used = re.findall(r"Compiling entry function '(\w*k_kv4_prefill\w*)'.*?Used (\d+) registers", r.stderr, flags=re.S)
    assert len(used) == 2 and all(int(n) == 96 for _, n in used), used
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()
    assert out == ["0", "0", "0", "1", "1"]


def test_clear_error_reaches_every_cache(a8, L, monkeypatch):
    """The package's clear_error clears the record, and the counters of what is alive (here without a device)."""
    c, gone = (a8.KV4Cache(1, 1, 64, 16, dev="cpu") for _ in range(2))
    c._ws["stream"] = gone._ws["stream"] = "tickets"
    del gone
    calls = []
    monkeypatch.setattr(L, "call", lambda name, *a: calls.append(name))
    monkeypatch.setattr(L, "counters", [o for o in L.counters if o is c])       # (others may need a device)
    a8.clear_error()
    assert calls == ["a8_clear_error"] and c._ws == {}


def test_imports_on_a_torch_without_cuda():
    """The engine and the cache import, and a cache on the CPU can be made, where torch has no CUDA bindings."""
    code = ("import torch\n"
            "for n in ('_cuda_getDevice', '_cuda_getCurrentRawStream', '_cuda_isCurrentStreamCapturing'):\n"
            "    delattr(torch._C, n)\n"
            "import __graft_entry__ as g\n"
            "a8 = g.load_package()\n"
            "a8.FastEngine, a8.KV4Cache(1, 1, 64, 16, dev='cpu')\n")
    r = subprocess.run([os.sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-800:]


def test_a_capture_on_the_cache_s_device_is_noticed(a8, monkeypatch):
    """With another device current, whether the call is captured is the cache's device's matter: a captured call gets a
    workspace of its own, an eager one the stream's."""
    c = a8.KV4Cache(2, 2, 64, 64, dev="cpu")
    c.dev = torch.device("cuda", 1)
    current, capturing, made = [0], {0: False, 1: True}, []

    class Device:
        def __init__(self, dev):
            self.dev = torch.device(dev).index if not isinstance(dev, int) else dev

        def __enter__(self):
            self.was, current[0] = current[0], self.dev

        def __exit__(self, *a):
            current[0] = self.was

    def workspace(nq, rows, max_len):
        made.append(current[0])
        return torch.zeros(4), torch.zeros(4, dtype=torch.int32)
    monkeypatch.setattr(torch.cuda, "device", Device)
    c.workspace = workspace
    c._current_device = lambda: current[0]
    c._current_stream = lambda dev: 7
    c._capturing = lambda: capturing[current[0]]
    a, b = c._workspace(14, 2, 64), c._workspace(14, 2, 64)
    assert a[0] != b[0] and not c._ws                    # captured: each its own, nothing kept
    capturing.update({0: True, 1: False})                # another device's capture is not this call's
    assert c._workspace(14, 2, 64)[0] == c._workspace(14, 2, 64)[0] and set(c._ws) == {7}
    assert made == [1, 1, 1]                             # where the call will run


def test_numbers_that_a_c_int_would_wrap_are_refused(a8):
    """2^32 + n is not n: layers, rings, bounds, shapes and row strides are refused, not cut to 32 bits."""
    W = 1 << 32
    for shape in ((W + 2, 2, 64, 40), (2, W + 2, 64, 40), (2, 2, W + 64, 40), (2, 2, 64, W + 40), (2, 2, 64, -W + 40)):
        with pytest.raises(a8.A8Error, match="unsupported shape"):
            a8.KV4Cache(*shape, dev="cpu")
    with pytest.raises(a8.A8Error, match="unsupported shape"):
        a8.KV4Cache(2, 2, 64, 40, dev="cpu", layers=W + 1)
    c = a8.KV4Cache(2, 2, 64, 40, dev="cpu", layers=3)
    c._workspace = lambda *a: (0, 0, 0, 0, None)
    bf, i32 = torch.bfloat16, torch.int32
    x, i, q = torch.zeros(3, 18 * 64, dtype=bf), torch.zeros(3, dtype=i32), torch.zeros(3, 896, dtype=bf)
    b = torch.zeros(1, 4, dtype=i32)
    for layer in (-1, 3, W, W + 1, -W):
        for f in (lambda: c.store(x, i, nq=14, layer=layer), lambda: c.load(i, layer=layer),
                  lambda: c.attention(q, i, layer=layer), lambda: c.prefill_attention(q, b, layer=layer)):
            with pytest.raises(a8.A8Error, match="layer"):
                f()
    for ring in (-1, 41, W, W + 8):
        with pytest.raises(a8.A8Error, match="ring"):
            c.store(x, i, nq=14, ring=ring)
    for n in (-1, 41, W + 40):
        with pytest.raises(a8.A8Error, match="max_len"):
            c.attention(q, i, max_len=n)
        with pytest.raises(a8.A8Error):
            c.workspace(14, 3, n)
    for nq, rows in ((W + 14, 3), (14, W + 3), (14, 0)):
        with pytest.raises(a8.A8Error):
            c.workspace(nq, rows, 40)
    for scale in (1e-39, 1e-60):                         # (0 in a C float: the default)
        for f in (lambda: c.attention(q, i, scale=scale), lambda: c.prefill_attention(q, b, scale=scale)):
            with pytest.raises(a8.A8Error, match="scale"):
                f()


def test_strides_past_32_bits_are_refused(a8):
    c = a8.KV4Cache(2, 2, 64, 40, dev="cpu")
    i = torch.zeros(2, dtype=torch.int32)
    # (two rows 2^32 + 1,152 elements apart, on a meta tensor: only its shape and strides are looked at)
    far = torch.empty_strided((2, 18 * 64), ((1 << 32) + 18 * 64, 1), dtype=torch.bfloat16, device="meta")
    kv = torch.empty_strided((2, 2, 64), ((1 << 32) + 128, 64, 1), dtype=torch.bfloat16, device="meta")
    c.dev = far.device
    i = i.to("meta")
    for f in (lambda: c.store(far, i, nq=14), lambda: c.attention(far[:, :896], i),
              lambda: c.prefill_attention(far[:, :896], torch.zeros(1, 4, dtype=torch.int32, device="meta")),
              lambda: c.load(i, k=kv), lambda: c.load(i, v=kv)):
        with pytest.raises(a8.A8Error, match="stride"):
            f()


def test_rotation_tables_without_rows_are_refused(a8):
    """cos and sin of no rows have no address, which the C call takes for no rotation at all."""
    c = a8.KV4Cache(2, 2, 64, 40, dev="cpu")
    x, t = torch.zeros(3, 18 * 64, dtype=torch.bfloat16), torch.zeros(0, 64, dtype=torch.bfloat16)
    with pytest.raises(a8.A8Error, match="cos, sin"):
        c.store(x, torch.zeros(3, dtype=torch.int32), nq=14, cos=t, sin=t)


def test_attention_steps_stay_within_32_bits(L):
    """The steps of 32 keys of all rows are counted in 32 bits, a CTA's share rounded up among them: calls that could pass
    them are refused, the next smaller ones are not."""
    lib, N, p = L.load(), None, C.c_void_p(256)

    def attn(rows, steps):
        d = L.A8KV4(256, 1, 1, 1, 64, steps * 32)
        return lib.a8_kv4_attention(C.byref(d), 0, p, 64, 1, p, N, rows, steps * 32, 0.0, p, 64, p, 1 << 40, p, 1 << 30, N)
    top = (1 << 31) - 1
    for rows, steps in ((104643, 20522), (1 << 11, 1 << 20)):        # 2^31 - 2 and 2^31
        assert top - 24 < rows * steps and attn(rows, steps) == SIZE, (rows, steps)
    if not torch.cuda.is_available():
        assert attn((1 << 11) - 1, 1 << 20) == CUDA                   # (no device here: the launch itself fails)
