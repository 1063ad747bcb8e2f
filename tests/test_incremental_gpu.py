"""The session decoder against a plain one in 64 bits.

The plain decoder has no pages and no kernels: dense masks over whole
sequences.  It rounds where the decoder's format rounds (16-bit activations,
4-bit weights, e4m3 keys and values with a power-of-two scale for 64 tokens and
a head), so what is left is the order of sums and values that fall on the other
side of a rounding: at most 2 u of each of the ten 16-bit tensors of a layer, in
norm, and each may pass through the three products behind it with a gain of two
(RMSNorm divides by the norm; the softmax's scores have norm products of
unit-variance heads).  An e4m3 value flips where it lies within 2 u of a
midpoint, a fraction of about 2 u / 2^-4, and then moves by 2^-3: below u
sqrt(2^5 / u) 2^-3 in norm, which the same allowance covers.  With u = 2^-11 and
two layers: 2 * 10 * 2 * 2 * 2^-11 = 0.04 of the norm.
"""
import dataclasses

import pytest

from conftest import cuda_ok, pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_cuda():
    if not cuda_ok():
        pytest.skip("no CUDA device")


def _cfg(**kw):
    base = dict(num_layers=2, hidden_size=512, intermediate_size=768, num_heads=8, num_kv_heads=4,
                head_dim=128, vocab_size=500, num_labels=300, max_seq=512)
    base.update(kw)
    return dataclasses.replace(pkg().synth.ModelConfig(), **base)


def _weights(cfg, seed=5):
    import torch
    g = torch.Generator().manual_seed(seed)
    w = {}
    for name, shape, kind in pkg().synth.weight_specs(cfg):
        if "language_model" in name or name.startswith("score"):
            t = torch.randn(*shape, generator=g) * 0.04 if kind == "normal" else torch.rand(*shape, generator=g) + 0.5
            w[name] = t.to(torch.bfloat16)
    return w


def _dense(lin):
    import torch
    codes = torch.stack([lin.wq & 15, lin.wq >> 4], -1).flatten(1)
    N, groups = lin.scales.shape
    c = codes.reshape(N, groups, -1).double() - lin.zeros.double()[..., None]
    return (c * lin.scales.double()[..., None]).reshape(N, -1)


def _cached(x):
    """[T, heads, hd] through the 8-bit cache."""
    import torch
    out = torch.empty_like(x)
    for a in range(0, x.shape[0], 64):
        p = x[a: a + 64]
        most = p.abs().amax((0, 2))
        s = torch.exp2(torch.ceil(torch.log2(most / 448)).clamp(min=-64))[None, :, None]
        out[a: a + 64] = (p / s).float().to(torch.float8_e4m3fn).double() * s
    return out


def _plain(dec, ids):
    """Hidden states of one whole sequence."""
    import torch
    cfg, dt = dec.cfg, dec.dtype
    nq, nkv, hd, half = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.head_dim // 2

    def r(t):
        return t.to(dt).double()

    def norm(t, gain):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * gain.double()

    T = len(ids)
    x = dec.embed[torch.tensor(ids, device=dec.device)].double()
    cos, sin = dec.cos[:T].double()[:, None], dec.sin[:T].double()[:, None]

    def turn(t, gain):
        t = norm(t, gain)
        a, b = t[..., :half], t[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    for L in dec.layers:
        qkv = r(r(norm(x, L["norm1"])) @ _dense(L["qkv"]).T)
        q, k, v = (t.reshape(T, -1, hd) for t in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
        q = r(turn(q, L["qn"]))
        k, v = _cached(turn(k, L["kn"])), _cached(v)
        k, v = (t.repeat_interleave(nq // nkv, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * hd ** -0.5
        s.masked_fill_(torch.ones(T, T, dtype=torch.bool, device=s.device).triu(1), -float("inf"))
        o = r(torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(T, -1))
        x = x + r(o @ _dense(L["o"]).T)
        gate, up = r(r(norm(x, L["norm2"])) @ _dense(L["gate_up"]).T).chunk(2, 1)
        x = x + r(r(gate * torch.sigmoid(gate) * up) @ _dense(L["down"]).T)
    return norm(x, dec.norm)


def _decoder(cfg, **kw):
    import torch
    return pkg().incremental.SessionDecoder(cfg, _weights(cfg), pages=kw.pop("pages", 24),
                                            dtype=torch.float16, **kw)


def _tokens(n, seed, cfg):
    import torch
    return torch.randint(0, cfg.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("kw", [{}, dict(num_heads=14, num_kv_heads=2, head_dim=64, hidden_size=896)])
def test_sessions_that_grow_follow_the_plain_decoder(kw):
    """Each session's pages are filled at once, so its page scales are those of
    whole pages: 64 and 128 tokens first, then what stays within a page."""
    cfg = _cfg(**kw)
    dec = _decoder(cfg)
    a, b, c = dec.open(), dec.open(), dec.open()
    ids = {a: _tokens(128 + 5, 1, cfg), b: _tokens(64 + 40, 2, cfg), c: _tokens(1, 3, cfg)}
    got = {s: [] for s in ids}
    for step in ({a: 128, b: 64}, {a: 5, c: 1, b: 40}):
        at = {s: sum(len(t) for t in got[s]) for s in step}
        h = dec.step({s: ids[s][at[s]: at[s] + n] for s, n in step.items()})
        for s, part in zip(step, h.split(list(step.values()))):
            got[s].append(part)
    dec.check()
    import torch
    for s in ids:
        want, have = _plain(dec, ids[s]), torch.cat(got[s]).double()
        assert have.shape == want.shape
        assert float((have - want).norm()) <= 0.04 * float(want.norm())
        labels = dec.labels(torch.cat(got[s]))
        exact = torch.cat(got[s]).double() @ _dense(dec.head).T
        assert labels.shape == (len(ids[s]), cfg.num_labels)
        assert float((labels.double() - exact).norm()) <= 2.0 ** -10 * float(exact.norm())


def test_a_session_does_not_depend_on_its_company():
    import torch
    cfg = _cfg()
    alone, mixed = _decoder(cfg), _decoder(cfg)
    a, other, b = alone.open(), mixed.open(), mixed.open()
    ids, noise = _tokens(70, 7, cfg), _tokens(200, 8, cfg)
    first = alone.step({a: ids[:69]})
    both = mixed.step({other: noise[:69], b: ids[:69]})
    assert torch.equal(first, both[69:])
    last = alone.step({a: ids[69:]})
    both = mixed.step({b: ids[69:], other: [noise[69]]})
    assert torch.equal(last, both[:1])
    mixed.close(other)
    again = mixed.open()
    assert torch.equal(mixed.step({again: ids[:69]}), first)  # in the pages that `other` left
    alone.check(), mixed.check()


def test_refusals_leave_the_sessions_as_they_were():
    cfg = _cfg()
    dec = _decoder(cfg, pages=2)
    a = dec.open()
    dec.step({a: _tokens(64, 1, cfg)})
    for bad, err in (([cfg.vocab_size], ValueError), ([-1], ValueError), ([0] * 65, MemoryError),
                     ([0] * 449, ValueError)):
        with pytest.raises(err):
            dec.step({a: bad})
    assert dec.table.length(a) == 64
    assert dec.step({a: []}).shape == (0, cfg.hidden_size) and dec.step({}).shape == (0, cfg.hidden_size)
    dec.step({a: [1]})
    dec.check()


def test_operators_in_a_graph():
    """A graph replays while the same operators run outside of it: the
    attention's workspace is the graph's own."""
    import torch
    L = pkg()
    g = torch.Generator(device="cuda").manual_seed(1)
    pages, nkv, nq, hd, n, length = 80, 2, 4, 64, 2, 2500
    f16 = torch.float16
    pool = [torch.randn(pages, nkv, 64, hd, generator=g, device="cuda").to(torch.float8_e4m3fn) for _ in "kv"]
    scales = [torch.ones(pages, nkv, device="cuda") for _ in "kv"]
    tab = torch.arange(pages, dtype=torch.int32, device="cuda").view(n, -1).contiguous()
    qs = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    kl = torch.full((n,), length, dtype=torch.int32, device="cuda")
    x = torch.randn(n, 256, generator=g, device="cuda", dtype=f16)
    wq = torch.randint(0, 256, ((nq + 2 * nkv) * hd, 128), generator=g, device="cuda", dtype=torch.uint8)
    ws = torch.full((wq.shape[0], 2), 0.01, dtype=f16, device="cuda")

    def run():
        qkv = torch.empty(n, wq.shape[0], dtype=f16, device="cuda")
        L.w4_linear(x, wq, ws, qkv)
        q, k, v = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
        L.kv_append(q, k, v, q, qs, kl, tab, *pool, kscale=scales[0], vscale=scales[1], max_q=1, validate=False)
        out = torch.empty(n, nq * hd, dtype=f16, device="cuda")
        L.cache_attention(q, qs, kl, tab, *pool, *scales, out, max_q=1, max_kv=length, validate=False)
        return out

    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        out.zero_()
        graph.replay()
        other = run()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(other, want)
