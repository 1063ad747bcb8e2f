"""The operators of a growing session, as cases to be timed.

A session keeps what it has seen in a paged K/V cache and takes a few more tokens at a time.  Each decoder layer
then runs 4-bit projections over those tokens (`w4_linear`), rotates the queries and keys and appends keys and
values to the cache (`kv_append`), and attends over the 8-bit cache (`cache_attention`).

Where `own` is false the operators are computed in elementary torch operations, in 32 bits, rounded once.
"""
import importlib
import math
import random

import torch

own = False

PAGE = 64
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
E4M3_MAX = 448.0
E_MIN = -64
THETA = 1e6


def _lib():
    return importlib.import_module("qwen3-aligner-wgpu_b200")._lib


# ---------------------------------------------------------------- cases

def listed():
    """16 query / 8 K/V heads of 128 is this repository's decoder, 14 heads of 64 its audio tower."""
    return [
        # one live session takes one more token: latency
        dict(name="append-1x1", op="append", dtype="f16", seqs=1, q_max=1, ctx=420, nq=16, nkv=8, hd=128, bits=8,
             axes=1, norm=True, mix=1),
        # a server's step: one token for each of 64 sessions of uneven length
        dict(name="append-64x1", op="append", dtype="bf16", seqs=64, q_max=1, ctx=8000, nq=16, nkv=8, hd=128, bits=8,
             axes=3, norm=True, mix=2),
        # corrected words and new prompts of uneven lengths, positions in time, height and width
        dict(name="append-24-ragged", op="append", dtype="f16", seqs=24, q_max=751, ctx=3000, nq=14, nkv=2, hd=64,
             bits=8, axes=3, norm=False, mix=3),
        # long prompts into the 16-bit cache that the prefill attention reads
        dict(name="append-4x8192", op="append", dtype="bf16", seqs=4, q_max=8192, ctx=0, nq=16, nkv=8, hd=128,
             bits=16, axes=1, norm=True, mix=4),
        # one session, one token, a short cache: latency
        dict(name="attend-1x1", op="attend", dtype="f16", seqs=1, q_max=1, ctx=421, nq=16, nkv=8, hd=128,
             causal=True, mix=5),
        # a server's step over 64 uneven caches
        dict(name="attend-64x1", op="attend", dtype="bf16", seqs=64, q_max=1, ctx=8192, nq=16, nkv=8, hd=128,
             causal=True, mix=6),
        # a few very long sessions: the long axis has to be split
        dict(name="attend-2x1-long", op="attend", dtype="f16", seqs=2, q_max=1, ctx=131001, nq=28, nkv=4, hd=128,
             causal=True, mix=7),
        # a few new words for each of 16 sessions
        dict(name="attend-16x12", op="attend", dtype="f16", seqs=16, q_max=12, ctx=5000, nq=16, nkv=8, hd=128,
             causal=True, mix=8),
        # a long transcript scored against long cached prefixes
        dict(name="attend-4x1024", op="attend", dtype="bf16", seqs=4, q_max=1024, ctx=8192, nq=16, nkv=8, hd=128,
             causal=True, mix=9),
        # the decoder's fused QKV projection for one token
        dict(name="w4-qkv-1", op="w4", dtype="f16", m=1, n=4096, k=1024, group=128, zeros=False, bias=False),
        # a wide square layer for a handful of sessions, odd row count, zero points and a bias
        dict(name="w4-square-5", op="w4", dtype="bf16", m=5, n=8191, k=8192, group=64, zeros=True, bias=True),
        # the vocabulary of this repository's decoder for 16 tokens
        dict(name="w4-vocab-16", op="w4", dtype="f16", m=16, n=151936, k=1024, group=128, zeros=False, bias=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "w4"])
    dtype = rng.choice(["f16", "bf16"])
    nq, nkv = rng.choice([(16, 8), (8, 8), (14, 2), (12, 4), (28, 4), (16, 1), (5, 5)])
    hd = rng.choice([64, 128])
    if op == "append":
        seqs = _log(rng, 1, 200)
        return dict(op=op, dtype=dtype, seqs=seqs, q_max=_log(rng, 1, 32768 // seqs), ctx=_log(rng, 1, 8000) - 1,
                    nq=nq, nkv=nkv, hd=hd, bits=rng.choice([8, 8, 16]), axes=rng.choice([1, 2, 3]),
                    norm=rng.random() < 0.5, mix=rng.randrange(1 << 20))
    if op == "attend":
        seqs = _log(rng, 1, 96)
        ctx = _log(rng, 1, min(131000, 600000 // seqs))
        q_max = _log(rng, 1, max(1, min(1024, ctx, (1 << 25) // (seqs * ctx))))
        return dict(op=op, dtype=dtype, seqs=seqs, q_max=q_max, ctx=ctx, nq=nq, nkv=nkv, hd=hd,
                    causal=rng.random() < 0.8, mix=rng.randrange(1 << 20))
    group = rng.choice([32, 64, 128])
    k = group * _log(rng, 1, 8192 // group)
    return dict(op=op, dtype=dtype, m=_log(rng, 1, 24), n=_log(rng, 16, min(151936, 140000000 // k)), k=k, group=group,
                zeros=rng.random() < 0.5, bias=rng.random() < 0.5)


def lengths(case):
    """New tokens and cached tokens (the new ones among them) of every sequence."""
    r = random.Random(case["mix"])
    n = [case["q_max"]] + [r.randint(max(1, case["q_max"] // 4), case["q_max"]) for _ in range(case["seqs"] - 1)]
    if case["op"] == "append":
        total = [case["ctx"] + n[0]] + [r.randint(case["ctx"] // 8, case["ctx"]) + x for x in n[1:]]
    else:
        total = [max(case["ctx"], n[0])] + [max(x, r.randint(max(1, case["ctx"] // 8), case["ctx"])) for x in n[1:]]
    return n, total


# ---------------------------------------------------------------- inputs

def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _codes(g, *shape):
    """e4m3 codes of values that fill the range as a scaled cache does."""
    x = torch.empty(*shape, device=DEV, dtype=torch.float8_e4m3fn)
    for part, to in zip(x.view(-1, shape[-1]).split(1 << 20), x.view(-1, shape[-1]).view(torch.uint8).split(1 << 20)):
        y = (torch.randn(part.shape, device=DEV, generator=g) * 64).clamp_(-E4M3_MAX, E4M3_MAX)
        to.copy_(y.to(torch.float8_e4m3fn).view(torch.uint8))
    return x


def _scales(g, *shape):
    return torch.exp2(torch.randint(-8, -4, shape, device=DEV, generator=g).float())


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]
    if case["op"] == "w4":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        s = dict(case=case, x=_randn(g, m, k).to(dt),
                 wq=torch.randint(0, 256, (n, k // 2), device=DEV, generator=g, dtype=torch.uint8),
                 scales=((torch.rand(n, k // group, device=DEV, generator=g) + 0.5) * 0.2 / math.sqrt(k)).to(dt),
                 out=torch.empty(m, n, device=DEV, dtype=dt), zeros=None, bias=None)
        if case["zeros"]:
            s["zeros"] = torch.randint(5, 11, (n, k // group), device=DEV, generator=g, dtype=torch.uint8)
        if case["bias"]:
            s["bias"] = _randn(g, n)
        return s
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    n, total = lengths(case)
    pages_per = [-(-t // PAGE) for t in total]
    pages = sum(pages_per) + 3
    order = torch.randperm(pages, device=DEV, generator=g, dtype=torch.int64).to(torch.int32)
    at = torch.tensor([0] + pages_per, device=DEV).cumsum(0)
    col = torch.arange(max(pages_per), device=DEV)
    inside = col[None, :] < (at[1:] - at[:-1])[:, None]
    tab = torch.where(inside, order[(at[:-1, None] + col[None, :]).clamp(max=pages - 1)], order[0])
    starts = [0]
    for x in n:
        starts.append(starts[-1] + x)
    T = starts[-1]
    s = dict(case=case, block_tab=tab.contiguous(), max_q=max(n), max_kv=max(total), max_pages=max(pages_per),
             q_start=torch.tensor(starts, device=DEV, dtype=torch.int32),
             kv_len=torch.tensor(total, device=DEV, dtype=torch.int32))
    if case["op"] == "attend":
        s.update(q=(_randn(g, T, nq * hd) * 1.3).to(dt), kpool=_codes(g, pages, nkv, PAGE, hd),
                 vpool=_codes(g, pages, nkv, PAGE, hd), kscale=_scales(g, pages, nkv), vscale=_scales(g, pages, nkv),
                 out=torch.empty(T, nq * hd, device=DEV, dtype=dt),
                 lse=torch.empty(T, nq, device=DEV, dtype=torch.float32))
        return s
    half = hd // 2
    width = (nq + 2 * nkv) * hd
    spread = torch.exp(_randn(g, 1, width) * 0.4)
    qkv = (_randn(g, T, width) * spread).to(dt)
    rows = 8192 + max(total)
    ang = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] / THETA ** (
        2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / hd)[None, :]
    s.update(q=qkv[:, : nq * hd], k=qkv[:, nq * hd: (nq + nkv) * hd], v=qkv[:, (nq + nkv) * hd:],
             q_out=torch.empty(T, nq * hd, device=DEV, dtype=dt), cos=ang.cos().float(), sin=ang.sin().float(),
             pos=None, axis_of=None, qn=None, kn=None, kscale=None, vscale=None)
    if case["axes"] > 1:
        # frames of a picture: every axis counts on its own
        s["pos"] = torch.randint(0, rows, (case["axes"], T), device=DEV, generator=g, dtype=torch.int32)
        s["axis_of"] = (torch.arange(half, device=DEV) % case["axes"]).to(torch.int32)
    if case["norm"]:
        s["qn"], s["kn"] = 1 + 0.2 * _randn(g, hd), 1 + 0.2 * _randn(g, hd)
    if case["bits"] == 8:
        s.update(kpool=_codes(g, pages, nkv, PAGE, hd), vpool=_codes(g, pages, nkv, PAGE, hd),
                 kscale=_scales(g, pages, nkv), vscale=_scales(g, pages, nkv))
    else:
        s.update(kpool=_randn(g, pages, nkv, PAGE, hd).to(dt), vpool=_randn(g, pages, nkv, PAGE, hd).to(dt))
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if op == "append":
        if own:
            _lib().kv_append(s["q"], s["k"], s["v"], s["q_out"], s["q_start"], s["kv_len"], s["block_tab"],
                             s["kpool"], s["vpool"], kscale=s["kscale"], vscale=s["vscale"], cos=s["cos"],
                             sin=s["sin"], pos=s["pos"], axis_of=s["axis_of"], qn=s["qn"], kn=s["kn"], eps=1e-6,
                             max_q=s["max_q"], validate=False)
        else:
            _append(s)
        return [s["q_out"], s["kpool"], s["vpool"], s["kscale"], s["vscale"]]
    if op == "attend":
        if own:
            _lib().cache_attention(s["q"], s["q_start"], s["kv_len"], s["block_tab"], s["kpool"], s["vpool"],
                                   s["kscale"], s["vscale"], s["out"], lse=s["lse"], causal=s["case"]["causal"],
                                   max_q=s["max_q"], max_kv=s["max_kv"], validate=False)
            return [s["out"], s["lse"]]
        return _attend(s)
    if own:
        _lib().w4_linear(s["x"], s["wq"], s["scales"], s["out"], zeros=s["zeros"], bias=s["bias"])
        return s["out"]
    return _w4(s)


def _places(s):
    """Sequence, cache index and page of every new token."""
    T = s["q"].shape[0]
    t = torch.arange(T, device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(s["q_start"][1:], t, right=True)
    c = (s["kv_len"] - s["q_start"][1:])[seq] + t
    return seq, c, s["block_tab"][seq, (c // PAGE).long()].long(), (c % PAGE).long()


def _rotated(x, hd, gain, cos, sin):
    x = x.reshape(x.shape[0], -1, hd).float()
    if gain is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(s):
    hd = s["case"]["hd"]
    seq, c, page, slot = _places(s)
    if s["pos"] is None:
        cos, sin = s["cos"][c.long()][:, None], s["sin"][c.long()][:, None]
    else:
        row = s["pos"][s["axis_of"].long()].t().long()
        cos, sin = s["cos"].gather(0, row)[:, None], s["sin"].gather(0, row)[:, None]
    s["q_out"].copy_(_rotated(s["q"], hd, s["qn"], cos, sin).flatten(1))
    k = _rotated(s["k"], hd, s["kn"], cos, sin)
    v = s["v"].reshape(k.shape).float()
    _store(s["kpool"], s["kscale"], k, page, slot, s)
    _store(s["vpool"], s["vscale"], v, page, slot, s)


def _store(pool, scale, x, page, slot, s):
    if scale is None:
        pool[page, :, slot] = x.to(pool.dtype)
        return
    size = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)
    most = torch.zeros_like(scale).index_reduce_(0, page, size, "amax")
    m, e = torch.frexp(most)  # most = m 2^e, 0.5 <= m < 1, and 448 = 0.875 2^9
    e = torch.where(most > 0, e - 9 + (m > 0.875).int(), E_MIN).clamp(min=E_MIN)
    wanted = torch.exp2(e.float())
    first = s["block_tab"].gather(1, ((s["kv_len"] - s["q_start"].diff()) // PAGE).long()[:, None])[:, 0].long()
    filled = ((s["kv_len"] - s["q_start"].diff()) % PAGE).long()
    old = scale[first]
    now = torch.where((filled > 0)[:, None], torch.maximum(old, wanted[first]), wanted[first])
    scale[page] = wanted[page]
    scale[first] = now
    raw = pool.view(torch.uint8)
    codes = raw[first]
    kept = (codes.view(pool.dtype).float() * (old / now)[:, :, None, None]).to(pool.dtype).view(torch.uint8)
    before = torch.arange(PAGE, device=DEV)[None, :] < filled[:, None]
    raw[first] = torch.where(before[:, None, :, None], kept, codes)
    y = x / scale[page][:, :, None]
    raw[page, :, slot] = torch.where(torch.isfinite(x), y.clamp(-E4M3_MAX, E4M3_MAX), math.nan).to(pool.dtype).view(torch.uint8)


def _attend(s):
    case = s["case"]
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    S, P = s["block_tab"].shape
    tab = s["block_tab"].long()

    def whole(pool, scale):
        x = pool.view(torch.uint8)[tab].view(pool.dtype).float() * scale[tab][..., None, None]
        return x.transpose(1, 2).reshape(S, nkv, P * PAGE, hd)

    k, v = whole(s["kpool"], s["kscale"]), whole(s["vpool"], s["vscale"])
    T = s["q"].shape[0]
    i = torch.arange(s["max_q"], device=DEV)
    row = (s["q_start"][:-1, None] + i).clamp(max=T - 1).long()
    n = s["q_start"].diff()
    q = s["q"][row].float().view(S, s["max_q"], nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4)
    sc = (q.reshape(S, nkv, -1, hd) @ k.transpose(-1, -2)).view(S, nkv, nq // nkv, s["max_q"], P * PAGE)
    sc = sc / math.sqrt(hd)
    seen = (s["kv_len"] - n)[:, None] + i + 1 if case["causal"] else s["kv_len"][:, None].expand(-1, s["max_q"])
    hidden = torch.arange(P * PAGE, device=DEV)[None, None] >= seen[..., None]
    sc = sc.masked_fill_(hidden[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top.isfinite(), top, 0))
    den = p.sum(-1, keepdim=True)
    o = (p.view(S, nkv, -1, P * PAGE) @ v).view(S, nkv, nq // nkv, s["max_q"], hd)
    o = torch.where(den > 0, o / den, 0).permute(0, 3, 1, 2, 4).reshape(S, s["max_q"], nq * hd)
    lse = (top + den.log())[..., 0].permute(0, 3, 1, 2).reshape(S, s["max_q"], nq)
    real = i[None] < n[:, None]
    return [o[real].to(s["q"].dtype), lse[real]]


def _w4(s):
    n, k = s["scales"].shape[0], s["x"].shape[1]
    group = s["case"]["group"]
    codes = torch.stack([s["wq"] & 15, s["wq"] >> 4], -1).view(n, k // group, group).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    w = ((codes - zero) * s["scales"].float()[..., None]).view(n, k)
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "w4":
        m, n, k, g = case["m"], case["n"], case["k"], case["group"]
        by = n * k / 2 + n * (k // g) * (3 if case["zeros"] else 2) + 2 * m * k + 2 * m * n + (4 * n if case["bias"] else 0)
        return {"bytes": by, "flops": 2.0 * m * n * k}
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    n, total = lengths(case)
    T = sum(n)
    if case["op"] == "append":
        # q, k, v in; q out; k and v into the cache; a cos and a sin row a token (one position each)
        by = T * ((nq + 2 * nkv) * hd * 2 + nq * hd * 2 + 2 * nkv * hd * case["bits"] // 8 + hd * 4)
        return {"bytes": by, "flops": float(T * (3 * (nq + nkv) * hd + (4 * (nq + nkv) * hd if case["norm"] else 0)))}
    seen = sum(x * t - (x * (x - 1) // 2 if case["causal"] else 0) for x, t in zip(n, total))
    by = sum(total) * nkv * hd * 2 + sum(-(-t // PAGE) for t in total) * nkv * 8 + T * nq * hd * 4 + T * nq * 4
    return {"bytes": by, "flops": 4.0 * seen * nq * hd}


# ---------------------------------------------------------------- in 64 bits, sequence by sequence

def exact(case, seed):
    """Values before they are rounded to the outputs' types (8-bit codes among them)."""
    s = prepare(case, seed)
    if case["op"] == "w4":
        n, k, g = case["n"], case["k"], case["group"]
        y = torch.empty(case["m"], n, device=DEV, dtype=torch.float64)
        for at in range(0, n, 8192):
            b = s["wq"][at: at + 8192].to(torch.int64)
            w = torch.empty(b.shape[0], k, device=DEV, dtype=torch.float64)
            w[:, 0::2], w[:, 1::2] = (b % 16).double(), (b // 16).double()
            z = s["zeros"][at: at + 8192].double() if case["zeros"] else torch.full_like(s["scales"][at: at + 8192], 8).double()
            w = (w - z.repeat_interleave(g, 1)) * s["scales"][at: at + 8192].double().repeat_interleave(g, 1)
            y[:, at: at + 8192] = s["x"].double() @ w.t()
        return y + s["bias"].double() if case["bias"] else y
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    n, total = lengths(case)
    if case["op"] == "attend":
        out, lse, at = [], [], 0
        for i, (m, L) in enumerate(zip(n, total)):
            pages = s["block_tab"][i, : -(-L // PAGE)].tolist()
            kk = (torch.stack([s["kpool"][p].to(torch.float64) for p in pages]) * s["kscale"][pages].double()[..., None, None]).transpose(0, 1).reshape(nkv, -1, hd)[:, :L]
            vv = (torch.stack([s["vpool"][p].to(torch.float64) for p in pages]) * s["vscale"][pages].double()[..., None, None]).transpose(0, 1).reshape(nkv, -1, hd)[:, :L]
            o = torch.empty(m, nq, hd, device=DEV, dtype=torch.float64)
            e = torch.empty(m, nq, device=DEV, dtype=torch.float64)
            for h in range(nq):
                w = s["q"][at: at + m, h * hd: (h + 1) * hd].double() @ kk[h // (nq // nkv)].t() * hd ** -0.5
                if case["causal"]:
                    w += torch.full_like(w, -math.inf).triu(L - m + 1)
                e[:, h] = torch.logsumexp(w, 1)
                o[:, h] = torch.softmax(w, 1) @ vv[h // (nq // nkv)]
            out.append(o.flatten(1))
            lse.append(e)
            at += m
        return [torch.cat(out), torch.cat(lse)]
    half = hd // 2
    ch = torch.complex(s["cos"].double(), s["sin"].double())
    at, q_out = 0, torch.empty(sum(n), nq * hd, device=DEV, dtype=torch.float64)
    kp, vp = s["kpool"].to(torch.float64), s["vpool"].to(torch.float64)
    ks, vs = (None, None) if case["bits"] == 16 else (s["kscale"].double(), s["vscale"].double())
    for i, (m, L) in enumerate(zip(n, total)):
        c = torch.arange(L - m, L, device=DEV)
        ax = torch.zeros(half, device=DEV, dtype=torch.int64) if s["axis_of"] is None else s["axis_of"].long()
        pos = c[:, None].expand(m, half) if s["pos"] is None else torch.stack([s["pos"][a, at: at + m] for a in ax.tolist()], 1).long()
        turn = ch[pos, torch.arange(half, device=DEV)[None]][:, None]

        def heads(x, gain):
            x = x[at: at + m].double().view(m, -1, hd)
            if gain is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * gain.double()
            y = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            return torch.cat([y.real, y.imag], -1)

        q_out[at: at + m] = heads(s["q"], s["qn"]).flatten(1)
        new = (heads(s["k"], s["kn"]), s["v"][at: at + m].double().view(m, nkv, hd))
        for pool, scale, x in ((kp, ks, new[0]), (vp, vs, new[1])):
            for j in range((L - m) // PAGE, (L - 1) // PAGE + 1):
                lo, hi = max(0, j * PAGE - (L - m)), min(m, (j + 1) * PAGE - (L - m))
                a, p = lo + L - m - j * PAGE, int(s["block_tab"][i, j])
                y = x[lo:hi].transpose(0, 1)
                if scale is not None:
                    most = y.abs().amax((1, 2))
                    want = torch.exp2(torch.floor(torch.log2(most / 448)).clamp(min=-64) - 1)
                    for _ in range(3):  # the least power of two that reaches: a logarithm may be one off
                        want = torch.where(most > 448 * want, 2 * want, want)
                    want = want.clamp(min=2.0 ** -64)
                    if a:
                        old, want = scale[p].clone(), torch.maximum(scale[p], want)
                        pool[p, :, :a] *= (old / want)[:, None, None]
                    scale[p] = want
                    y = y / want[:, None, None]
                pool[p, :, a: a + hi - lo] = y
        at += m
    return [q_out, kp, vp, ks, vs]
