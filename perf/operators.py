"""The operators on a key/value cache held in 4 bits, as measured: cases, their plain form and their definition in 64
bits.

The cache keeps, for every (row, kv head, position), hd 4-bit codes and one bf16 scale per 32 of them:
s = bf16(max|x| / 7), code = rint(x / s) in [-7, 7], the value is code * s. Four operators work on it: `store` (rotate
the query and key heads of packed rows, quantise their keys and values into the cache; measured together with the
read-back of what it wrote), `load` (read positions back as bf16), `attn` (one query token a row over its cached keys)
and `prefill` (packed causal prompt rows over the cache).
"""
import importlib
import math
import sys

import torch

own = False

GROUP = 32
BF = torch.bfloat16


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step's rows of the slow stack at 192 streams: each at its own position of its own cache row
        dict(name="store_tick", op="store", rows=192, nq=14, nkv=2, hd=64, cache_rows=193, cache_len=2048, seqs=192),
        # one admission chunk: 2,048 packed prompt rows of nine requests
        dict(name="store_admit", op="store", rows=2048, nq=14, nkv=2, hd=64, cache_rows=193, cache_len=2048, seqs=9),
        # one long document, wide heads, an odd count of rows
        dict(name="store_long", op="store", rows=16381, nq=32, nkv=8, hd=128, cache_rows=2, cache_len=16384, seqs=1),
        # a voice prefix of 317 positions read back
        dict(name="load_prefix", op="load", rows=317, nkv=2, hd=64, cache_rows=193, cache_len=2048, seqs=1),
        # a long document's cache read back (moved to a bf16 cache, or checked)
        dict(name="load_long", op="load", rows=65533, nkv=8, hd=128, cache_rows=3, cache_len=65536, seqs=2),
        # one stream's decode step: latency
        dict(name="attn_one", op="attn", rows=1, nq=14, nkv=2, hd=64, cache_rows=5, cache_len=2048, lo=733, hi=733),
        # 192 streams of every age
        dict(name="attn_tick", op="attn", rows=192, nq=14, nkv=2, hd=64, cache_rows=193, cache_len=2048, lo=1,
             hi=2047),
        # a loaded server: 1,408 streams, most of them mid-utterance
        dict(name="attn_serving", op="attn", rows=1408, nq=14, nkv=2, hd=64, cache_rows=1409, cache_len=2048, lo=97,
             hi=911),
        # the codec transformer's ring of 128 positions, one query head a kv head
        dict(name="attn_window", op="attn", rows=192, nq=8, nkv=8, hd=128, cache_rows=192, cache_len=128, lo=1,
             hi=128),
        # three long documents of unequal lengths: the work has to be split over a long axis
        dict(name="attn_long", op="attn", rows=3, nq=32, nkv=8, hd=128, cache_rows=3, cache_len=131072, lo=40009,
             hi=131071),
        # an admission chunk of ragged requests, each behind its voice's cached prefix
        dict(name="prefill_admit", op="prefill", rows=2048, nq=14, nkv=2, hd=64, cache_rows=10, cache_len=2048,
             seqs=9, prefix=317),
        # one long prompt
        dict(name="prefill_long", op="prefill", rows=8189, nq=32, nkv=8, hd=128, cache_rows=2, cache_len=8192, seqs=1,
             prefix=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges: rows, lengths, head counts and widths spread over them, odd ones among them."""
    op = rng.choice(["store", "load", "attn", "attn", "prefill", "prefill"])
    nq, nkv, hd = rng.choice([(14, 2, 64), (8, 8, 128), (32, 8, 128), (16, 4, 64), (6, 1, 128), (7, 7, 64)])
    if op == "store":
        rows = _log(rng, 1, 12000)
        seqs = min(rows, _log(rng, 1, 256))
        longest = rows - (seqs - 1) if seqs > 1 else rows
        return dict(op=op, rows=rows, nq=nq, nkv=nkv, hd=hd, cache_rows=seqs + rng.randint(0, 3),
                    cache_len=max(longest + rng.randint(0, 77), 40), seqs=seqs)
    if op == "load":
        rows = _log(rng, 1, 40000)
        seqs = min(rows, _log(rng, 1, 9))
        longest = rows - (seqs - 1) if seqs > 1 else rows
        return dict(op=op, rows=rows, nkv=nkv, hd=hd, cache_rows=seqs + rng.randint(0, 3),
                    cache_len=max(longest + rng.randint(0, 77), 40), seqs=seqs)
    if op == "attn":
        hi = _log(rng, 1, 100000)
        lo = rng.randint(1, hi)
        rows = max(1, min(1400, _log(rng, 1, max(2, 400000 // (hi * nkv)))))
        return dict(op=op, rows=rows, nq=nq, nkv=nkv, hd=hd, cache_rows=rows + rng.randint(0, 3),
                    cache_len=hi + rng.randint(0, 77), lo=lo, hi=hi)
    rows = _log(rng, 1, 5000)
    seqs = min(rows, _log(rng, 1, 12))
    prefix = rng.choice([0, _log(rng, 1, 900)])
    longest = rows - (seqs - 1) if seqs > 1 else rows
    return dict(op=op, rows=rows, nq=nq, nkv=nkv, hd=hd, cache_rows=seqs + rng.randint(0, 3),
                cache_len=prefix + longest + rng.randint(0, 77), seqs=seqs, prefix=prefix)


def _rng_ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g).tolist()


def _host_plan(case, seed):
    """What the host knows of a case: sequence lengths, cache rows, positions (from the seed alone)."""
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    op, rows = case["op"], case["rows"]
    if op == "attn":
        lens = _rng_ints(g, case["lo"], case["hi"], rows)
        lens[-1] = case["hi"]
        return dict(lens=lens, rowmap=torch.randperm(case["cache_rows"], generator=g)[:rows].tolist())
    seqs = case["seqs"]
    if seqs == rows:
        ns = [1] * rows
    else:                                    # ragged parts, none empty
        w = torch.rand(seqs, generator=g) + 0.25
        ns = [max(1, int(x)) for x in (w / w.sum() * (rows - seqs)).tolist()]
        ns[-1] += rows - sum(ns)
        if ns[-1] < 1:
            ns = [1] * (seqs - 1) + [rows - seqs + 1]
    slots = torch.randperm(case["cache_rows"], generator=g)[:seqs].tolist()
    assert max(ns) + case.get("prefix", 0) <= case["cache_len"]
    room = [case["cache_len"] - n for n in ns]
    if op == "prefill":
        starts = [case["prefix"]] * seqs
    elif seqs == rows:
        starts = [_rng_ints(g, 0, r, 1)[0] for r in room]
    else:
        starts = [min(r, 3) for r in room]
    return dict(ns=ns, slots=slots, starts=starts)


def _cuda_gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _kv_rows(g, rows, nkv, hd):
    """Keys with a few strong channels (as rotary keys have) and values, bf16 [rows, nkv, hd]."""
    k = torch.randn(rows, nkv, hd, device="cuda", generator=g)
    k *= 0.5 + 2.5 * (torch.rand(nkv, hd, device="cuda", generator=g) > 0.94)
    v = torch.randn(rows, nkv, hd, device="cuda", generator=g) * 0.6
    return k.to(BF), v.to(BF)


def _inputs(case, seed):
    """Host plan + device tensors of a case, the same for every form."""
    plan = _host_plan(case, seed)
    op, rows, nkv, hd = case["op"], case["rows"], case["nkv"], case["hd"]
    g = _cuda_gen(seed, 1)
    d = dict(plan=plan)
    i32 = lambda xs: torch.tensor(xs, dtype=torch.int32).cuda()
    if op != "attn":
        d["pos"] = i32([p for a, n in zip(plan["starts"], plan["ns"]) for p in range(a, a + n)])
        d["slot"] = i32([s for s, n in zip(plan["slots"], plan["ns"]) for _ in range(n)])
    if op == "store":
        nq = case["nq"]
        q = torch.randn(rows, nq, hd, device="cuda", generator=g).to(BF)
        k, v = _kv_rows(g, rows, nkv, hd)
        d["qkv"] = torch.cat([q.reshape(rows, -1), k.reshape(rows, -1), v.reshape(rows, -1)], 1).contiguous()
        npos = case["cache_len"]
        fr = 1.0 / (1e6 ** (torch.arange(0, hd, 2, device="cuda").float() / hd))
        ph = torch.outer(torch.arange(npos, device="cuda").float(), fr)
        d["cos"] = torch.cat([ph.cos(), ph.cos()], -1).to(BF).contiguous()
        d["sin"] = torch.cat([ph.sin(), ph.sin()], -1).to(BF).contiguous()
        return d
    if op == "attn":
        d["lens"], d["rowmap"] = i32(plan["lens"]), i32(plan["rowmap"])
    # the cache's content: rows (slot, pos) as packed keys and values
    if op == "attn":
        fill = [(s, 0, n) for s, n in zip(plan["rowmap"], plan["lens"])]
    elif op == "load":
        fill = [(s, a, n) for s, a, n in zip(plan["slots"], plan["starts"], plan["ns"])]
    else:
        fill = [(s, 0, a + n) for s, a, n in zip(plan["slots"], plan["starts"], plan["ns"])]
    d["fill"] = fill
    d["k"], d["v"] = _kv_rows(g, sum(n for _, _, n in fill), nkv, hd)
    if op != "load":
        d["q"] = (torch.randn(rows, case["nq"], hd, device="cuda", generator=g) * 1.5).to(BF).reshape(rows, -1)
    return d


def _fill_index(fill):
    """(slot, pos) int64 of the packed content rows."""
    n = torch.tensor([f[2] for f in fill])
    slot = torch.repeat_interleave(torch.tensor([f[0] for f in fill]), n)
    first = torch.repeat_interleave(torch.cumsum(n, 0) - n - torch.tensor([f[1] for f in fill]), n)
    return slot.cuda(), (torch.arange(int(n.sum())) - first).cuda()


# ------------------------------------------------------------------------------------------------- the plain form
def _quantise(x):
    """bf16 [..., hd] -> codes int8 [..., hd], scales bf16 [..., hd / 32]."""
    xg = x.float().unflatten(-1, (-1, GROUP))
    s = (xg.abs().amax(-1) / 7.0).to(BF)
    sf = s.float().unsqueeze(-1)
    c = torch.where(sf > 0, torch.round(xg / sf), torch.zeros_like(xg)).clamp(-7, 7)
    return c.to(torch.int8).flatten(-2), s


def _values(c, s):
    return (c.float().unflatten(-1, (-1, GROUP)) * s.float().unsqueeze(-1)).flatten(-2)


def _rotate(x, cos, sin):
    """rotate_half of bf16 heads [rows, heads, hd] by table rows [rows, hd]: fp32 products and sum, one rounding."""
    h = x.shape[-1] // 2
    a, b = x[..., :h].float(), x[..., h:].float()
    c, s = cos[:, None, :h].float(), sin[:, None, :h].float()
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(BF)


def _plain_store(st):
    case, rows, nkv, hd, nq = st["case"], st["case"]["rows"], st["case"]["nkv"], st["case"]["hd"], st["case"]["nq"]
    p, sl = st["pos"].long(), st["slot"].long()
    x = st["qkv"].view(rows, nq + 2 * nkv, hd)
    qk = _rotate(x[:, :nq + nkv], st["cos"][p], st["sin"][p])
    for name, t in (("k", qk[:, nq:]), ("v", x[:, nq + nkv:])):
        c, s = _quantise(t)
        st[name + "c"][sl, :, p] = c
        st[name + "s"][sl, :, p] = s
    return qk[:, :nq].reshape(rows, nq * hd), *_plain_load(st)


def _plain_load(st):
    p, sl = st["pos"].long(), st["slot"].long()
    return tuple(_values(st[n + "c"][sl, :, p], st[n + "s"][sl, :, p]).to(BF) for n in "kv")


def _plain_softmax_pv(q, k, v, ok, scale):
    """q [..., m, hd], k / v [..., n, hd] fp32, ok [..., m, n]: masked softmax(q k^T scale) v."""
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~ok, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (p @ v) / p.sum(-1, keepdim=True)


def _plain_attn(st):
    case = st["case"]
    rows, nq, nkv, hd = case["rows"], case["nq"], case["nkv"], case["hd"]
    lens_h = st["plan"]["lens"]
    out = torch.empty(rows, nq * hd, dtype=BF, device="cuda")
    a = 0
    while a < rows:
        e, top = a, 0
        while e < rows and (e == a or (e - a + 1) * max(top, lens_h[e]) * nkv * hd <= 1 << 26):
            top = max(top, lens_h[e])
            e += 1
        m = st["rowmap"][a:e].long()
        k = _values(st["kc"][m, :, :top], st["ks"][m, :, :top])
        v = _values(st["vc"][m, :, :top], st["vs"][m, :, :top])
        ok = torch.arange(top, device="cuda") < st["lens"][a:e, None, None, None]
        q = st["q"][a:e].float().view(e - a, nkv, nq // nkv, hd)
        # masked positions hold whatever the cache held: keep their values out of the products
        keep = ok.view(e - a, 1, top, 1)
        o = _plain_softmax_pv(q, torch.where(keep, k, 0), torch.where(keep, v, 0), ok, hd ** -0.5)
        out[a:e] = o.reshape(e - a, nq * hd).to(BF)
        a = e
    return out


def _plain_prefill(st):
    case, plan = st["case"], st["plan"]
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    out = torch.empty(case["rows"], nq * hd, dtype=BF, device="cuda")
    r0 = 0
    for s, a, n in zip(plan["slots"], plan["starts"], plan["ns"]):
        q = st["q"][r0:r0 + n].float().view(n, nkv, nq // nkv, hd)
        o = torch.empty(n, nkv, nq // nkv, hd, device="cuda")
        ok = torch.arange(a + n, device="cuda") <= torch.arange(a, a + n, device="cuda")[:, None]
        for h in range(nkv):
            k = _values(st["kc"][s, h, :a + n], st["ks"][s, h, :a + n])
            v = _values(st["vc"][s, h, :a + n], st["vs"][s, h, :a + n])
            o[:, h] = _plain_softmax_pv(q[:, h].transpose(0, 1), k, v, ok, hd ** -0.5).transpose(0, 1)
        out[r0:r0 + n] = o.view(n, nq * hd).to(BF)
        r0 += n
    return out


# --------------------------------------------------------------------------------------------- prepare, run, work
def _package():
    if "audio8_b200" not in sys.modules:
        importlib.import_module("__graft_entry__").load_package()
    return sys.modules["audio8_b200"]


def prepare(case, seed):
    d = _inputs(case, seed)
    st = dict(case=case, plan=d["plan"])
    for n in ("pos", "slot", "qkv", "cos", "sin", "lens", "rowmap", "q"):
        if n in d:
            st[n] = d[n]
    op, nkv, hd, R, S = case["op"], case["nkv"], case["hd"], case["cache_rows"], case["cache_len"]
    if own:
        kv4 = importlib.import_module(_package().__name__ + ".kv4")
        st["cache"] = kv4.KV4Cache(R, nkv, hd, S)
        if op == "prefill":
            eng = importlib.import_module(_package().__name__ + ".engine")
            blocks = eng.FastEngine.query_blocks(d["pos"].cpu().numpy(), d["slot"].cpu().numpy())
            st["blocks"] = torch.from_numpy(blocks).cuda()
        if op != "store":
            slot, pos = _fill_index(d["fill"])
            n = len(pos)
            kv = torch.cat([d["k"].view(n, -1), d["v"].view(n, -1)], 1)
            st["cache"].store(kv, pos.int(), slot.int())
        return st
    for n in "kv":
        st[n + "c"] = torch.zeros(R, nkv, S, hd, dtype=torch.int8, device="cuda")
        st[n + "s"] = torch.zeros(R, nkv, S, hd // GROUP, dtype=BF, device="cuda")
    if op != "store":
        slot, pos = _fill_index(d["fill"])
        for n in "kv":
            c, s = _quantise(d[n])
            st[n + "c"][slot, :, pos] = c
            st[n + "s"][slot, :, pos] = s
    return st


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        cache = st["cache"]
        if op == "store":
            q = cache.store(st["qkv"], st["pos"], st["slot"], nq=case["nq"], cos=st["cos"], sin=st["sin"])
            k, v = cache.load(st["pos"], st["slot"])
            return q, k, v
        if op == "load":
            return cache.load(st["pos"], st["slot"])
        if op == "attn":
            return cache.attention(st["q"], st["lens"], st["rowmap"], max_len=case["hi"])
        return cache.prefill_attention(st["q"], st["blocks"])
    return dict(store=_plain_store, load=_plain_load, attn=_plain_attn, prefill=_plain_prefill)[op](st)


def work(case):
    """Bytes and operations the path cannot do without: every input and cached element it needs read once, every
    output written once (4.5 bits a cached element)."""
    op, rows, nkv, hd = case["op"], case["rows"], case["nkv"], case["hd"]
    key = nkv * hd * 2 * (0.5 + 2.0 / GROUP)              # a position's keys and values in the cache
    if op == "load":
        return dict(bytes=rows * (key + nkv * hd * 4 + 8), flops=rows * nkv * hd * 2)
    if op == "store":
        nq = case["nq"]
        return dict(bytes=rows * ((nq + 2 * nkv) * hd * 2 + nq * hd * 2 + hd * 2 + 8 + key + key + nkv * hd * 4),
                    flops=rows * (3 * (nq + nkv) + 8 * nkv) * hd)
    plan = _host_plan(case, 1)
    nq = case["nq"]
    if op == "attn":
        keys = sum(plan["lens"])
        pairs = keys
    else:
        keys = sum(a + n for a, n in zip(plan["starts"], plan["ns"]))
        pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(plan["starts"], plan["ns"]))
    return dict(bytes=keys * key + rows * nq * hd * 4, flops=pairs * nq * hd * 4)


# ------------------------------------------------------------------------------------------ the definition, 64 bits
def _exact_values(x):
    """What the cache holds of bf16 x, in 64 bits: the scale rounds max|x| / 7 to bf16, the code x / scale to the
    nearest whole number (ties to even)."""
    n, h, hd = x.shape
    xd = x.double().reshape(n, h, hd // GROUP, GROUP)
    top = xd.abs().max(dim=3, keepdim=True).values
    s = (top / 7).to(BF).double()
    c = torch.zeros_like(xd)
    live = (s > 0).expand_as(xd)
    c[live] = (xd / s.clamp(min=1e-300))[live].round().clamp(-7, 7)
    return (c * s).reshape(n, h, hd)


def _exact_attention(q, k, v, first, scale):
    """q [m, hd], k / v [n, hd] in 64 bits; row i attends keys [0, first + i]."""
    m, n = q.shape[0], k.shape[0]
    z = torch.einsum("id,jd->ij", q, k).mul_(scale)
    if first + 1 < n:
        i, j = torch.arange(m, device=q.device), torch.arange(n, device=q.device)
        z.masked_fill_(j[None, :] > first + i[:, None], -math.inf)
    w = torch.softmax(z, dim=1)
    return w @ v


def exact(case, seed):
    d = _inputs(case, seed)
    plan, op, rows, nkv, hd = d["plan"], case["op"], case["rows"], case["nkv"], case["hd"]
    if op == "store":
        nq = case["nq"]
        x = d["qkv"].reshape(rows, nq + 2 * nkv, hd)
        at = d["pos"].long()
        co, si = d["cos"].double()[at][:, None, :], d["sin"].double()[at][:, None, :]
        y = x[:, :nq + nkv].double()
        turned = torch.cat([-y[..., hd // 2:], y[..., :hd // 2]], dim=-1)
        r = y * co + turned * si
        # the cache holds the quantised bf16 key: the rotation's fp32 sum rounded to bf16
        k = r[:, nq:].float().to(BF)
        return r[:, :nq].reshape(rows, -1), _exact_values(k), _exact_values(x[:, nq + nkv:])
    k, v = _exact_values(d["k"]), _exact_values(d["v"])
    if op == "load":
        return k, v
    grp = case["nq"] // nkv
    q = d["q"].double().reshape(rows, case["nq"], hd)
    out = torch.empty(rows, case["nq"], hd, dtype=torch.float64, device="cuda")
    r0 = c0 = 0
    spans = [(n - 1, 1) for n in plan["lens"]] if op == "attn" else list(zip(plan["starts"], plan["ns"]))
    for a, n in spans:
        for h in range(case["nq"]):
            out[r0:r0 + n, h] = _exact_attention(q[r0:r0 + n, h], k[c0:c0 + a + n, h // grp],
                                                 v[c0:c0 + a + n, h // grp], a, hd ** -0.5)
        r0 += n
        c0 += a + n
    return out.reshape(rows, -1)
