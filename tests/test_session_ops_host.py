"""What the session operators refuse, without a GPU: malformed tensors raise
ValueError before any launch, and the C entry points answer bad arguments with a
status code."""
import ctypes

import pytest

from conftest import pkg

PAGE = 64


def _cache(bits=8, pages=6, nkv=2, hd=64, T=5):
    import torch
    dt = torch.float16
    pool = (lambda: torch.zeros(pages, nkv, PAGE, hd, dtype=torch.uint8).view(torch.float8_e4m3fn)) if bits == 8 else (
        lambda: torch.zeros(pages, nkv, PAGE, hd, dtype=dt))
    c = dict(q=torch.zeros(T, 4 * hd, dtype=dt), k=torch.zeros(T, nkv * hd, dtype=dt),
             v=torch.zeros(T, nkv * hd, dtype=dt), q_out=torch.zeros(T, 4 * hd, dtype=dt),
             q_start=torch.tensor([0, 3, 5], dtype=torch.int32), kv_len=torch.tensor([70, 2], dtype=torch.int32),
             block_tab=torch.tensor([[1, 2], [3, 0]], dtype=torch.int32), kpool=pool(), vpool=pool(), max_q=3,
             kscale=None, vscale=None, cos=torch.ones(90, hd // 2), sin=torch.zeros(90, hd // 2))
    if bits == 8:
        c.update(kscale=torch.ones(pages, nkv), vscale=torch.ones(pages, nkv))
    return c


def _append(c, **change):
    pkg()._lib.kv_append(**{**c, **change})


def _attend(c, **change):
    a = {k: c[k] for k in ("q", "q_start", "kv_len", "block_tab", "kpool", "vpool", "kscale", "vscale", "max_q")}
    pkg()._lib.cache_attention(**{**a, "out": c["q_out"], "max_kv": 70, **change})


def test_a_sound_call_gets_as_far_as_the_device():
    for bits in (8, 16):
        with pytest.raises(ValueError, match="CUDA"):
            _append(_cache(bits))
    with pytest.raises(ValueError, match="CUDA"):
        _attend(_cache())


@pytest.mark.parametrize("what", range(26))
def test_append_refuses(what):
    import torch
    c = _cache()
    i32, f16 = torch.int32, torch.float16
    change = [
        dict(q=c["q"].float()), dict(q=c["q"][:, :-1]), dict(q=torch.zeros(5, 192, dtype=f16)), dict(q=c["q"][:4]),
        dict(k=c["k"].bfloat16()), dict(v=c["v"][:, ::2]), dict(q_out=torch.zeros(1, 256, dtype=f16).expand(5, 256)),
        dict(q_start=c["q_start"].long()), dict(q_start=c["q_start"][:2]), dict(kv_len=c["kv_len"].float()),
        dict(block_tab=c["block_tab"].t()), dict(kpool=c["kpool"][:, :, :32]), dict(kpool=c["kpool"].float()),
        dict(kscale=None), dict(vscale=torch.ones(6, 3)), dict(cos=None), dict(cos=torch.ones(90, 31)),
        dict(pos=torch.zeros(5, dtype=torch.int64)), dict(pos=torch.zeros(2, 5, dtype=i32)),
        dict(pos=torch.zeros(5, 5, dtype=i32), axis_of=torch.zeros(32, dtype=i32)), dict(qn=torch.ones(64)),
        # found by `validate`
        dict(max_q=2), dict(kv_len=torch.tensor([70, 1], dtype=i32)), dict(kv_len=torch.tensor([129, 2], dtype=i32)),
        dict(block_tab=torch.tensor([[1, 6], [3, 0]], dtype=i32)),
        dict(block_tab=torch.tensor([[1, 3], [3, 0]], dtype=i32)),  # both append to page 3
    ][what]
    with pytest.raises(ValueError) as e:
        _append(c, **change)
    assert "CUDA" not in str(e.value)


def test_append_refuses_positions_outside_the_tables():
    import torch
    c = _cache()
    with pytest.raises(ValueError, match="tables"):
        _append(c, pos=torch.full((5,), 90, dtype=torch.int32))
    with pytest.raises(ValueError, match="tables"):
        _append(c, cos=c["cos"][:69], sin=c["sin"][:69])
    with pytest.raises(ValueError, match="axis_of"):
        _append(c, pos=torch.zeros(2, 5, dtype=torch.int32), axis_of=torch.full((32,), 2, dtype=torch.int32))


@pytest.mark.parametrize("what", range(9))
def test_attention_refuses(what):
    import torch
    c = _cache()
    change = [
        dict(kpool=_cache(16)["kpool"], vpool=_cache(16)["vpool"]), dict(out=c["q_out"].bfloat16()),
        dict(out=c["q_out"][:, :192]), dict(lse=torch.zeros(5, 3)), dict(kscale=c["kscale"].half()), dict(max_q=-1),
        dict(max_kv=-1), dict(max_kv=69), dict(q_start=torch.tensor([0, 4, 3], dtype=torch.int32)),
    ][what]
    with pytest.raises(ValueError) as e:
        _attend(c, **change)
    assert "CUDA" not in str(e.value)


def test_w4_refuses():
    import torch
    f16, u8 = torch.float16, torch.uint8
    x, w, s, o = (torch.zeros(3, 256, dtype=f16), torch.zeros(10, 128, dtype=u8), torch.zeros(10, 2, dtype=f16),
                  torch.zeros(3, 10, dtype=f16))
    f = pkg()._lib.w4_linear
    with pytest.raises(ValueError, match="CUDA"):
        f(x, w, s, o)
    for a in [(x.float(), w, s, o), (x[:, :254], w, s, o), (x, w.to(torch.int8), s, o), (x, w[:9], s, o),
              (x, w, s.bfloat16(), o), (x, w, torch.zeros(10, 1, dtype=f16), o), (x, w, torch.zeros(10, 3, dtype=f16), o),
              (x, w, s, o[:, :9]), (x, w, s, o[:2]), (x[0], w, s, o)]:
        with pytest.raises(ValueError) as e:
            f(*a)
        assert "CUDA" not in str(e.value)
    for k in (dict(zeros=torch.zeros(10, 3, dtype=u8)), dict(zeros=s), dict(bias=torch.zeros(9)), dict(bias=s[:, 0])):
        with pytest.raises(ValueError) as e:
            f(x, w, s, o, **k)
        assert "CUDA" not in str(e.value)


def test_c_entry_points_answer_bad_arguments():
    """Refused before any CUDA call: the addresses here are never touched."""
    lib = pkg()._lib
    L, p = lib.lib(), 1 << 20

    def append(q=p, T=4, nq=4, nkv=2, hd=64, ldq=256, n=1, max_q=4, max_pages=2, kpool=p, pages=3, ks=p, vs=p, cos=p,
               sin=p, rows=9, pos=0, axes=1, axis_of=0, qn=0, kn=0):
        return L.qa_k_kv_append(q, ldq, p, 128, p, 128, p, 256, T, nq, nkv, hd, p, p, n, max_q, p, max_pages, kpool, p,
                                pages, ks, vs, cos, sin, rows, pos, 4, axes, axis_of, qn, kn, 1e-6, 0, 0, 0)

    for bad in (dict(q=0), dict(nq=3), dict(nkv=0), dict(max_pages=0), dict(pages=0), dict(kpool=0), dict(kpool=p + 8),
                dict(ks=0), dict(vs=0), dict(cos=0), dict(sin=0), dict(rows=0), dict(axes=0), dict(axes=5),
                dict(axes=3, pos=p), dict(qn=p), dict(T=-1), dict(T=1 << 31), dict(cos=p + 4), dict(n=-1)):
        assert append(**bad) == lib.QA_ERR_ARG, bad
    assert append(hd=96) == lib.QA_ERR_SHAPE and append(ldq=255) == lib.QA_ERR_SHAPE
    assert append(T=0) == lib.QA_OK and append(n=0) == lib.QA_OK

    def attend(q=p, T=4, nq=4, nkv=2, hd=64, ldo=256, n=1, ks=p, scale=0.1, out=p, vpool=p, max_kv=9, ws=0, ws_bytes=0):
        return L.qa_k_cache_attention(q, 256, T, nq, nkv, hd, p, p, n, 4, max_kv, p, 2, p, vpool, 3, ks, p, scale, 1, out,
                                      ldo, 0, ws, ws_bytes, 0, 0, 0)

    for bad in (dict(q=0), dict(out=0), dict(ks=0), dict(vpool=0), dict(vpool=p + 1), dict(max_kv=-1), dict(ws=p + 8), dict(ws_bytes=-1), dict(nq=5),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(T=-1)):
        assert attend(**bad) == lib.QA_ERR_ARG, bad
    assert attend(hd=256) == lib.QA_ERR_SHAPE and attend(ldo=100) == lib.QA_ERR_SHAPE
    assert attend(T=0) == lib.QA_OK and attend(n=0) == lib.QA_OK

    def w4(x=p, ldx=256, m=2, k=256, w=p, ldw=128, n=8, group=128, s=p, out=p, ldo=8):
        return L.qa_k_w4_linear(x, ldx, m, k, w, ldw, n, group, s, 0, 0, out, ldo, 0, 0)

    for bad in (dict(x=0), dict(w=0), dict(s=0), dict(out=0), dict(m=-1), dict(n=-1)):
        assert w4(**bad) == lib.QA_ERR_ARG, bad
    for bad in (dict(group=100), dict(k=200), dict(ldx=255), dict(ldw=127), dict(ldo=7), dict(k=0)):
        assert w4(**bad) == lib.QA_ERR_SHAPE, bad
    assert w4(m=0) == lib.QA_OK and w4(n=0) == lib.QA_OK
    assert ctypes.sizeof(ctypes.c_longlong) == 8
