"""The operators of growing sessions against plain implementations in 64 bits.

`kv_append` (rotation with one to four position axes, optional RMSNorm, append
to the paged cache in 16 or 8 bits), `cache_attention` (over the 8-bit cache)
and `w4_linear` (4-bit weights).  The cases sit where such kernels go wrong:
lengths of 0 and 1, a page's first and last slot, lengths around page ends,
ragged sequences, rows that see nothing, NaN past a sequence's end, head groups
of 1 to 16, packed and unaligned rows, pools past 2^31 bytes.

Tolerances.  u is the unit roundoff of the 16-bit type, 2^-11 for f16 and 2^-8
for bf16.
 - rotated values: f32 arithmetic (an RMSNorm of at most 128 squares and two
   products, under 2^-18 of the head's largest value) and one rounding;
 - e4m3 codes: half a unit in the last place, 2^-4 relative and 2^-10 absolute
   (the smallest code is 2^-9), plus the f32 part;
 - attention: probabilities held in 16 bits (2^-11 each, doubled for the f32
   exponentials and sums): 2^-10 sum_c p_c |v_c|, and one rounding; lse: f32
   sums of 64 or 128 products, under 2^-17 of sum |q_d k_d| scale;
 - 4-bit products: f32 sums, at most 2^-14 sum |x w| for K <= 16384 (a tensor
   core truncates below 2^-22 of a step's largest term, 8 steps a group, then
   at most 512 rounded additions), and one rounding.
"""
import math

import pytest

from conftest import cuda_ok, pkg

pytestmark = pytest.mark.gpu
PAGE = 64


@pytest.fixture(autouse=True)
def _needs_cuda():
    if not cuda_ok():
        pytest.skip("no CUDA device")


def _dt(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def _u(name):
    return {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]


def _maps(seqs, g, spare=3):
    """(n, len) pairs -> q_start, kv_len, block_tab (pages shuffled), pages."""
    import torch
    per = [-(-L // PAGE) for _, L in seqs]
    pages = sum(per) + spare
    perm = torch.randperm(pages, generator=g).tolist()
    tab = torch.full((len(seqs), max(per + [1])), -7, dtype=torch.int32)  # unused entries are no pages
    at = 0
    for s, m in enumerate(per):
        tab[s, :m] = torch.tensor(perm[at: at + m], dtype=torch.int32)
        at += m
    qs = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).to(torch.int32)
    return qs, torch.tensor([L for _, L in seqs], dtype=torch.int32), tab, pages


def _codes(shape, g, spread=60.0):
    import torch
    return (torch.randn(*shape, generator=g) * spread).clamp(-448, 448).to(torch.float8_e4m3fn)


def _pow2(shape, g, lo=-9, hi=-4):
    import torch
    return torch.exp2(torch.randint(lo, hi, shape, generator=g).float())


# ---------------------------------------------------------------- kv_append

APPEND_SEQS = [
    [(1, 1)],
    [(1, 64), (1, 65), (0, 70), (1, 63), (3, 66), (64, 64), (0, 0)],
    [(130, 130), (64, 191), (2, 129), (65, 128), (1, 500), (63, 126)],
    [(300, 307), (1, 2)],
]


def _append_case(seqs, dtype, hd, nq, nkv, bits, norm, axes, seed, offset=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    dt = _dt(dtype)
    qs, kl, tab, pages = _maps(seqs, g)
    T, rows = int(qs[-1]), 700
    packed = torch.empty(T, offset + (nq + 2 * nkv) * hd + offset, dtype=dt)
    x = packed[:, offset: offset + (nq + 2 * nkv) * hd]
    x.copy_(torch.randn(T, x.shape[1], generator=g) * torch.exp(torch.randn(1, x.shape[1], generator=g) * 0.5))
    ang = torch.rand(rows, hd // 2, generator=g, dtype=torch.float64) * 6.28
    c = dict(seqs=seqs, hd=hd, nq=nq, nkv=nkv, dtype=dtype, bits=bits, packed=packed, offset=offset,
             q_start=qs, kv_len=kl, tab=tab, pages=pages, cos=ang.cos().float(), sin=ang.sin().float(),
             pos=None, axis_of=None, qn=None, kn=None, kscale=None, vscale=None)
    if axes:
        c["pos"] = torch.randint(0, rows, (axes, T), generator=g, dtype=torch.int32)
        c["axis_of"] = torch.randint(0, axes, (hd // 2,), generator=g, dtype=torch.int32)
    if norm:
        c["qn"], c["kn"] = torch.rand(hd, generator=g) + 0.5, torch.rand(hd, generator=g) + 0.5
    shape = (pages, nkv, PAGE, hd)
    if bits == 8:
        c.update(kpool=_codes(shape, g), vpool=_codes(shape, g), kscale=_pow2((pages, nkv), g),
                 vscale=_pow2((pages, nkv), g))
    else:
        c.update(kpool=torch.randn(*shape, generator=g).to(dt), vpool=torch.randn(*shape, generator=g).to(dt))
    return c


def _split(c, packed):
    w, o = c["hd"], c["offset"]
    a, b, e = o + c["nq"] * w, o + (c["nq"] + c["nkv"]) * w, o + (c["nq"] + 2 * c["nkv"]) * w
    return packed[:, o:a], packed[:, a:b], packed[:, b:e]


def _append_run(c, in_place=False, stream=None, times=1):
    import torch
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    q, k, v = _split(c, d["packed"])
    q_out = q if in_place else torch.full((q.shape[0], q.shape[1]), float("nan"), dtype=q.dtype, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for _ in range(times):
        pkg()._lib.kv_append(q, k, v, q_out, d["q_start"], d["kv_len"], d["tab"], d["kpool"], d["vpool"],
                             max_q=max(n for n, _ in c["seqs"]), kscale=d["kscale"], vscale=d["vscale"],
                             cos=d["cos"], sin=d["sin"], pos=d["pos"], axis_of=d["axis_of"], qn=d["qn"],
                             kn=d["kn"], eps=1e-6, status=st, stream=stream)
    torch.cuda.synchronize()
    assert int(st.item()) == 0
    return {k: None if x is None else x.cpu() for k, x in dict(
        q=q_out, kpool=d["kpool"], vpool=d["vpool"], kscale=d["kscale"], vscale=d["vscale"]).items()}


def _turned(c, x, gain):
    """[T, heads * hd] in f64: normalised, rotated [T, heads, hd]."""
    import torch
    hd = c["hd"]
    x = x.double().reshape(x.shape[0], -1, hd)
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gain.double()
    at = torch.cat([torch.arange(L - n, L) for n, L in c["seqs"]])[:, None].expand(-1, hd // 2)
    if c["pos"] is not None:
        at = c["pos"].long()[c["axis_of"].long()].t()
    cs, sn = (c[k].double().gather(0, at)[:, None] for k in ("cos", "sin"))
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)




def _want_scale(most):
    """Least power of two >= 2^-64 with most <= 448 times it, by search."""
    import torch
    e = torch.full_like(most, -64)
    for k in range(-64, 121):
        e = torch.where(most > 448 * 2.0 ** k, float(k + 1), e)
    return torch.exp2(e)


def _check_append(c, got):
    import torch
    u, hd = _u(c["dtype"]), c["hd"]
    q, k, v = _split(c, c["packed"])
    q, k, v = _turned(c, q, c["qn"]), _turned(c, k, c["kn"]), v.double().reshape(v.shape[0], -1, hd)
    big = q.abs().amax(-1, keepdim=True)
    err = (got["q"].double().reshape(q.shape) - q).abs()
    assert bool((err <= u * q.abs() + 2.0 ** -18 * big + 2.0 ** -25).all()), err.max()
    t0 = 0
    seen = torch.zeros(c["pages"], PAGE, dtype=torch.bool)
    for s, (n, L) in enumerate(c["seqs"]):
        for j in range((L - n) // PAGE, -(-L // PAGE)) if n else []:
            lo, hi = max(L - n, j * PAGE), min(L, (j + 1) * PAGE)
            p, a, rows = int(c["tab"][s, j]), lo - j * PAGE, slice(t0 + lo - (L - n), t0 + hi - (L - n))
            seen[p, : a + hi - lo] = True
            for pool, scale, x in (("kpool", "kscale", k[rows]), ("vpool", "vscale", v[rows])):
                x = x.transpose(0, 1)
                new, old = got[pool][p].double(), c[pool][p].double()
                part = new[:, a: a + hi - lo]
                f32 = 2.0 ** -18 * x.abs().nan_to_num(0, 0, 0).amax(-1, keepdim=True)
                if c["bits"] == 16:
                    assert bool(((part - x).abs() <= u * x.abs() + f32 + 2.0 ** -25).all())
                    assert torch.equal(new[:, :a], old[:, :a])
                    continue
                fine = torch.where(x.isfinite(), x.abs(), 0).amax((1, 2))
                want = _want_scale(fine)
                was = c[scale][p].double()
                if a:
                    want = torch.maximum(want, was)
                assert torch.equal(got[scale][p].double(), want)
                y = x / want[:, None, None]
                ok = (part - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 + f32 / want[:, None, None]
                assert bool((ok | (part.isnan() & ~x.isfinite())).all())
                moved = (c[pool][p].float() * (was / want).float()[:, None, None]).to(torch.float8_e4m3fn)
                if a:
                    assert torch.equal(new[:, :a], moved.double()[:, :a])
        t0 += n
    rest = ~seen[:, None, :, None]
    for pool in ("kpool", "vpool"):
        assert torch.equal(torch.where(rest, got[pool].double(), 0), torch.where(rest, c[pool].double(), 0))


@pytest.mark.parametrize("seqs", APPEND_SEQS, ids=range(len(APPEND_SEQS)))
@pytest.mark.parametrize("dtype,hd,nq,nkv,bits,norm,axes", [
    ("f16", 128, 16, 8, 8, True, 0), ("bf16", 128, 16, 8, 16, True, 3), ("bf16", 64, 14, 2, 8, False, 2),
    ("f16", 64, 5, 5, 16, False, 1), ("f16", 128, 16, 1, 8, False, 4), ("bf16", 128, 28, 4, 8, True, 3)])
def test_append(seqs, dtype, hd, nq, nkv, bits, norm, axes):
    c = _append_case(seqs, dtype, hd, nq, nkv, bits, norm, axes, seed=hd + nq + len(seqs))
    _check_append(c, _append_run(c))


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("offset", [1, 4, 8])
def test_append_from_unaligned_rows_in_place_and_twice(offset, bits):
    """Rows that cannot be read 16 bytes at a time; q rotated where it stands."""
    import torch
    c = _append_case(APPEND_SEQS[2], "f16", 128, 4, 2, bits, True, 2, seed=offset, offset=offset)
    _check_append(c, _append_run(c, in_place=True))
    once, twice = _append_run(c), _append_run(c, times=2)  # the same tokens again: the same cache
    for k in ("q", "kpool", "vpool"):
        assert torch.equal(once[k].double(), twice[k].double())
    if bits == 8:
        assert torch.equal(once["kscale"], twice["kscale"]) and torch.equal(once["vscale"], twice["vscale"])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_append_of_extreme_values(dtype):
    """Zeros, subnormals, the largest finite values, infinities and NaN."""
    import torch
    c = _append_case([(20, 20), (40, 90), (1, 1), (30, 33)], dtype, 64, 2, 2, 8, False, 0, seed=5)
    c["cos"], c["sin"] = torch.ones_like(c["cos"]), torch.zeros_like(c["sin"])
    x = c["packed"]
    top = torch.finfo(_dt(dtype)).max
    x[0:20] = 0
    x[20:40, 128:192] = top
    x[30, 130], x[31, 140], x[32, 300] = math.inf, -math.inf, math.nan
    x[60] = torch.finfo(_dt(dtype)).tiny
    x[61:, 128:] *= 1e-3 if dtype == "f16" else 1e-30
    _check_append(c, _append_run(c))


def test_append_on_a_stream_of_its_own():
    import torch
    c = _append_case(APPEND_SEQS[1], "bf16", 128, 16, 8, 8, True, 3, seed=9)
    s = torch.cuda.Stream()
    _check_append(c, _append_run(c, stream=s.cuda_stream))


def test_append_reports_bad_maps_and_keeps_out():
    """Checked on the device when the host does not: nothing is written for them."""
    import torch
    L = pkg()._lib
    c = _append_case([(5, 70), (2, 3), (4, 4)], "f16", 64, 4, 2, 8, False, 1, seed=3)
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    q, k, v = _split(c, d["packed"])

    def run(max_q=5, **change):
        e = {**d, **{n: x.cuda() for n, x in change.items()}}
        kp, st = e["kpool"].clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
        L.kv_append(q, k, v, torch.empty_like(q), e["q_start"], e["kv_len"], e["tab"], kp, e["vpool"].clone(),
                    max_q=max_q, kscale=e["kscale"].clone(), vscale=e["vscale"].clone(), cos=e["cos"], sin=e["sin"],
                    pos=e["pos"], status=st, validate=False)
        return int(st.item()), (kp.view(torch.uint8) != e["kpool"].view(torch.uint8)).any(-1).any(-1).any(-1).cpu()

    status, changed = run()
    pages = {int(c["tab"][0, 1]), int(c["tab"][1, 0]), int(c["tab"][2, 0])}
    assert status == 0 and set(changed.nonzero().flatten().tolist()) <= pages | {int(c["tab"][0, 0])}
    for page in (-1, c["pages"], 1 << 30):
        tab = c["tab"].clone()
        tab[1, 0] = page
        status, changed = run(tab=tab)
        assert status == 2 and not changed[int(c["tab"][1, 0])] and changed[int(c["tab"][2, 0])]
    for kl in (1 << 20, -1, 1):  # past the table, negative, fewer than the new tokens
        kv = c["kv_len"].clone()
        kv[1] = kl
        status, changed = run(kv_len=kv)
        assert status == 2 and not changed[int(c["tab"][1, 0])]
    assert run(max_q=4)[0] == 2
    pos = c["pos"].clone()
    pos[0, 3] = c["cos"].shape[0]
    assert run(pos=pos)[0] == 2


# ---------------------------------------------------------------- cache_attention

def _attn_case(seqs, dtype, hd, nq, nkv, seed, ldq_extra=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    qs, kl, tab, pages = _maps(seqs, g)
    T = int(qs[-1])
    buf = (torch.randn(T, nq * hd + ldq_extra, generator=g) * 1.5).to(_dt(dtype))
    c = dict(seqs=seqs, dtype=dtype, hd=hd, nq=nq, nkv=nkv, buf=buf, q_start=qs, kv_len=kl, tab=tab, pages=pages,
             kpool=_codes((pages, nkv, PAGE, hd), g), vpool=_codes((pages, nkv, PAGE, hd), g),
             kscale=_pow2((pages, nkv), g, -8, -4), vscale=_pow2((pages, nkv), g, -12, 3))
    used = torch.zeros(pages, PAGE, dtype=torch.bool)
    for s, (_, L) in enumerate(seqs):
        for j in range(-(-L // PAGE)):
            used[int(tab[s, j]), : max(0, min(PAGE, L - j * PAGE))] = True
    for pool in ("kpool", "vpool"):  # NaN wherever no token lies
        c[pool].view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7F)
    return c


def _attn_run(c, causal=True, scale=None, stream=None, max_kv=None):
    import torch
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    w = c["nq"] * c["hd"]
    q = d["buf"][:, -w:] if c["buf"].shape[1] > w else d["buf"]
    out = torch.full(d["buf"].shape, float("nan"), dtype=q.dtype, device="cuda")[:, -w:]
    lse = torch.full((q.shape[0], c["nq"]), float("nan"), device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    pkg()._lib.cache_attention(q, d["q_start"], d["kv_len"], d["tab"], d["kpool"], d["vpool"], d["kscale"],
                               d["vscale"], out, lse=lse, causal=causal, scale=scale, status=st, stream=stream,
                               max_q=max(n for n, _ in c["seqs"]), max_kv=max_kv or max(L for _, L in c["seqs"]))
    torch.cuda.synchronize()
    assert int(st.item()) == 0
    return q.cpu(), out.cpu(), lse.cpu()


def _check_attn(c, got, causal=True, scale=None, device="cpu"):
    import torch
    q, out, lse = (x.to(device) for x in got)
    hd, nq, nkv, u = c["hd"], c["nq"], c["nkv"], _u(c["dtype"])
    scale = hd ** -0.5 if scale is None else scale
    t0 = 0
    for s, (n, L) in enumerate(c["seqs"]):
        ids = c["tab"][s, : -(-L // PAGE)].long()
        k = (c["kpool"][ids].double() * c["kscale"][ids].double()[..., None, None]).transpose(0, 1).reshape(nkv, -1, hd)[:, :L].to(device)
        v = (c["vpool"][ids].double() * c["vscale"][ids].double()[..., None, None]).transpose(0, 1).reshape(nkv, -1, hd)[:, :L].to(device)
        x = q[t0: t0 + n].double().view(n, nkv, nq // nkv, hd).permute(1, 2, 0, 3).reshape(nkv, -1, hd)
        sc = (x @ k.transpose(1, 2) * scale).view(nkv, nq // nkv, n, L)
        size = (x.abs() @ k.abs().transpose(1, 2) * abs(scale)).view(nkv, nq // nkv, n, L)
        if causal:
            hidden = torch.arange(L, device=device)[None] >= (L - n + torch.arange(n, device=device) + 1)[:, None]
            sc, size = sc.masked_fill(hidden, -math.inf), size.masked_fill(hidden, 0)
        if L:
            ref_l = torch.logsumexp(sc, -1)
            p = torch.softmax(sc, -1).nan_to_num(0)
            big = size.amax(-1)
        else:
            ref_l, p, big = (torch.full((nkv, nq // nkv, n), -math.inf, device=device, dtype=torch.float64), sc,
                             torch.zeros(nkv, nq // nkv, n, device=device, dtype=torch.float64))
        ref = (p.reshape(nkv, nq // nkv * n, L) @ v).view(nkv, nq // nkv, n, hd)
        tol = (p.reshape(nkv, nq // nkv * n, L) @ v.abs()).view(ref.shape)
        # an error of e in a score moves its probability by a factor 1 + e
        tol = u * ref.abs() + (2.0 ** -10 + 2.0 ** -16 * big[..., None]) * tol + 2.0 ** -25
        o = out[t0: t0 + n].double().view(n, nkv, nq // nkv, hd).permute(1, 2, 0, 3)
        assert bool(((o - ref).abs() <= tol).all()), ((o - ref).abs() / tol).max()
        e = lse[t0: t0 + n].double().view(n, nkv, nq // nkv).permute(1, 2, 0)
        assert torch.equal(e.isinf(), ref_l.isinf())
        diff = torch.where(ref_l.isinf(), 0, e - ref_l).abs()
        assert bool((diff <= 2.0 ** -17 * (1 + big)).all()), diff.max()
        t0 += n


ATTN_SEQS = [
    [(1, 1)],
    [(1, 63), (1, 64), (0, 64), (1, 65), (1, 1000), (1, 2), (1, 129)],
    [(3, 3), (0, 0), (2, 0), (9, 4), (17, 700), (8, 128), (70, 200)],  # rows that see nothing
    [(130, 130), (64, 191), (2, 4097)],
]
HEADS = [("f16", 128, 16, 8), ("bf16", 128, 28, 4), ("f16", 64, 14, 2), ("bf16", 64, 5, 5), ("f16", 128, 16, 1),
         ("bf16", 128, 3, 1), ("bf16", 64, 16, 8)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("seqs", ATTN_SEQS, ids=range(len(ATTN_SEQS)))
@pytest.mark.parametrize("dtype,hd,nq,nkv", HEADS)
def test_attention(dtype, hd, nq, nkv, seqs, causal):
    c = _attn_case(seqs, dtype, hd, nq, nkv, seed=hd + nq + nkv)
    _check_attn(c, _attn_run(c, causal), causal)


@pytest.mark.parametrize("extra", [1, 4, 8])
@pytest.mark.parametrize("seqs", [[(1, 200), (1, 77)], [(40, 300), (33, 33)]])
def test_attention_on_strided_rows(extra, seqs):
    c = _attn_case(seqs, "bf16", 128, 16, 8, seed=extra, ldq_extra=extra)
    _check_attn(c, _attn_run(c))


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0])
@pytest.mark.parametrize("seqs", [[(2, 150), (1, 64)], [(90, 260)]])
def test_attention_scales(scale, seqs):
    c = _attn_case(seqs, "f16", 64, 4, 2, seed=17)
    _check_attn(c, _attn_run(c, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [1, 48])
def test_attention_over_uneven_scales(dtype, n):
    """Pages whose scales lie far apart, queries whose components do."""
    import torch
    c = _attn_case([(n, 700), (n, 130)], dtype, 128, 16, 8, seed=23)
    g = torch.Generator().manual_seed(1)
    c["vscale"] = _pow2(tuple(c["vscale"].shape), g, -60, 4)
    c["kscale"] = _pow2(tuple(c["kscale"].shape), g, -30, -4)
    c["buf"] *= torch.exp2(torch.randint(-12, 2, c["buf"].shape[-1:], generator=g).float()).to(c["buf"].dtype)
    _check_attn(c, _attn_run(c))


@pytest.mark.parametrize("n,max_kv", [(1, None), (1, 64), (4, None), (1, 1 << 20)])
def test_attention_over_a_long_cache(n, max_kv):
    """The long axis split; max_kv only sizes the launch."""
    import torch
    L = pkg()._lib
    c = _attn_case([(n, 40000), (n, 777)], "bf16", 128, 16, 8, seed=29)
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    out, lse = torch.empty_like(d["buf"]), torch.empty(2 * n, 16, device="cuda")
    L.cache_attention(d["buf"], d["q_start"], d["kv_len"], d["tab"], d["kpool"], d["vpool"], d["kscale"], d["vscale"],
                      out, lse=lse, max_q=n, max_kv=max_kv or 40000, validate=False)
    again = torch.empty_like(out)
    L.cache_attention(d["buf"], d["q_start"], d["kv_len"], d["tab"], d["kpool"], d["vpool"], d["kscale"], d["vscale"],
                      again, max_q=n, max_kv=max_kv or 40000, validate=False)
    assert torch.equal(out, again)  # the joined parts are summed in one order
    _check_attn(c, (d["buf"].cpu(), out.cpu(), lse.cpu()))


def test_attention_past_32_bit_offsets():
    """Pools of more than 2^31 bytes, the sequences' pages at their end."""
    import torch
    c = _attn_case([(1, 300), (20, 130)], "f16", 128, 16, 8, seed=31)
    move = (1 << 31) // (8 * PAGE * 128) + 5
    big = {}
    for pool in ("kpool", "vpool"):
        x = torch.empty(move + c["pages"], 8, PAGE, 128, dtype=torch.uint8, device="cuda")
        x[move:] = c[pool].view(torch.uint8).cuda()
        big[pool] = x.view(torch.float8_e4m3fn)
        x = torch.ones(move + c["pages"], 8, device="cuda")
        name = pool[0] + "scale"
        x[move:] = c[name].cuda()
        big[name] = x
    q, out = c["buf"].cuda(), torch.empty_like(c["buf"], device="cuda")
    lse = torch.empty(21, 16, device="cuda")
    pkg()._lib.cache_attention(q, c["q_start"].cuda(), c["kv_len"].cuda(), (c["tab"] + move).cuda(), big["kpool"],
                               big["vpool"], big["kscale"], big["vscale"], out, lse=lse, max_q=20, max_kv=300,
                               validate=False)
    _check_attn(c, (q.cpu(), out.cpu(), lse.cpu()))


def test_attention_keeps_nan_to_the_rows_that_see_it():
    import torch
    c = _attn_case([(3, 100), (3, 100)], "f16", 128, 16, 8, seed=37)
    c["vpool"].view(torch.uint8)[int(c["tab"][0, 1]), 2, 99 - 64] = 0x7F  # the last token, K/V head 2
    _, out, lse = _attn_run(c)
    bad = out.view(6, 16, 128).isnan()
    want = torch.zeros(6, 16, 1, dtype=torch.bool)
    want[2, 4:6] = True
    assert torch.equal(bad, want.expand_as(bad)) and bool(lse.isfinite().all())
    q = _attn_case([(3, 100), (3, 100)], "f16", 128, 16, 8, seed=37)
    q["buf"][4, 7 * 128 + 3] = math.nan
    _, out, lse = _attn_run(q)
    bad = out.view(6, 16, 128).isnan()
    want[:] = False
    want[4, 7] = True
    assert torch.equal(bad, want.expand_as(bad)) and torch.equal(lse.isnan(), want[..., 0])


def test_attention_reports_bad_maps():
    import torch
    L = pkg()._lib
    c = _attn_case([(2, 200), (1, 70)], "f16", 64, 4, 2, seed=41)
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}

    def run(max_q=2, **change):
        e = {**d, **{n: x.cuda() for n, x in change.items()}}
        out, st = torch.full_like(d["buf"], 7), torch.zeros(1, dtype=torch.int32, device="cuda")
        L.cache_attention(d["buf"], e["q_start"], e["kv_len"], e["tab"], d["kpool"], d["vpool"], d["kscale"],
                          d["vscale"], out, max_q=max_q, max_kv=256, status=st, validate=False)
        return int(st.item()), out.cpu()

    good = run()
    assert good[0] == 0
    for kl in (-1, 1 << 20):
        kv = c["kv_len"].clone()
        kv[0] = kl
        status, out = run(kv_len=kv)
        assert status == 2 and bool((out[:2] == 7).all()) and torch.equal(out[2], good[1][2])
    for page in (-1, c["pages"]):  # left out: what remains is attended to
        tab = c["tab"].clone()
        tab[0, 1] = page
        status, out = run(tab=tab)
        assert status == 2 and bool(out.isfinite().all()) and torch.equal(out[2], good[1][2])
    assert run(max_q=1)[0] == 2


# ---------------------------------------------------------------- w4_linear

def _w4_case(m, n, k, group, dtype, zeros, bias, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    dt = _dt(dtype)
    return dict(x=torch.randn(m, k, generator=g).to(dt),
                wq=torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8),
                scales=(torch.randn(n, k // group, generator=g) * 0.05).to(dt),
                zeros=torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None,
                bias=torch.randn(n, generator=g) if bias else None, group=group, dtype=dtype)


def _check_w4(c, out):
    import torch
    k, g = c["x"].shape[1], c["group"]
    w = torch.empty(c["wq"].shape[0], k, dtype=torch.float64)
    w[:, 0::2], w[:, 1::2] = (c["wq"] & 15).double(), (c["wq"] >> 4).double()
    z = 8.0 if c["zeros"] is None else c["zeros"].double().repeat_interleave(g, 1)
    w = (w - z) * c["scales"].double().repeat_interleave(g, 1)
    ref, size = c["x"].double() @ w.t(), c["x"].double().abs() @ w.abs().t()
    if c["bias"] is not None:
        ref, size = ref + c["bias"].double(), size + c["bias"].double().abs()
    tol = _u(c["dtype"]) * ref.abs() + 2.0 ** -14 * size + 2.0 ** -25
    err = (out.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), (err / tol).max()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 33, 70])
@pytest.mark.parametrize("n,k,group,zeros,bias", [
    (1, 32, 32, False, False), (17, 96, 32, True, True), (255, 1024, 128, False, False),
    (130, 832, 64, True, False), (4096, 1024, 128, False, True), (70, 16384, 128, True, True)])
def test_w4(dtype, m, n, k, group, zeros, bias):
    import torch
    c = _w4_case(m, n, k, group, dtype, zeros, bias, seed=m + n + k)
    d = {a: (b.cuda() if isinstance(b, torch.Tensor) else b) for a, b in c.items()}
    out = torch.full((m, n), float("nan"), dtype=c["x"].dtype, device="cuda")
    pkg()._lib.w4_linear(d["x"], d["wq"], d["scales"], out, zeros=d["zeros"], bias=d["bias"])
    _check_w4(c, out)


@pytest.mark.parametrize("pad_x,pad_w,pad_o", [(1, 1, 1), (8, 16, 8), (3, 0, 0), (0, 5, 0), (2, 8, 1)])
def test_w4_on_strided_rows(pad_x, pad_w, pad_o):
    import torch
    c = _w4_case(5, 100, 320, 64, "f16", True, True, seed=pad_w)
    x = torch.zeros(5, 320 + pad_x, dtype=torch.float16, device="cuda")[:, pad_x:]
    w = torch.zeros(100, 160 + pad_w, dtype=torch.uint8, device="cuda")[:, pad_w:]
    o = torch.full((5, 100 + pad_o), 3.0, dtype=torch.float16, device="cuda")
    x.copy_(c["x"]), w.copy_(c["wq"])
    pkg()._lib.w4_linear(x, w, c["scales"].cuda(), o[:, pad_o:], zeros=c["zeros"].cuda(), bias=c["bias"].cuda())
    _check_w4(c, o[:, pad_o:])
    assert bool((o[:, :pad_o] == 3).all())


def test_w4_keeps_nan_to_its_row_and_repeats():
    import torch
    c = _w4_case(11, 300, 512, 128, "bf16", False, False, seed=2)
    c["x"][4, 77] = math.nan
    d = {a: (b.cuda() if isinstance(b, torch.Tensor) else b) for a, b in c.items()}
    out = [torch.empty(11, 300, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for o in out:
        pkg()._lib.w4_linear(d["x"], d["wq"], d["scales"], o)
    bad = out[0].isnan().cpu()
    assert bool(bad[4].all()) and int(bad.sum()) == 300
    assert torch.equal(out[0].nan_to_num(0), out[1].nan_to_num(0))
