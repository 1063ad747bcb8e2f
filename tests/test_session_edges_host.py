"""Host side of the session operators, without a GPU: where a call
launches, whose memory it works in, how much of it, what a step
that fails leaves behind, and 4-bit codes of tiny weights.

The tensors here lie in host memory and say that they are on a device; the
library's entry points are replaced by ones that record the call."""
import contextlib

import pytest
import torch

from conftest import pkg

PAGE = 64


class _OnDevice(torch.Tensor):
    """A host tensor that calls itself one of device 1."""

    def get_device(self):
        return 1


class _Gpu:
    """What the wrappers ask of CUDA, with device `current` current; `calls` holds
    (operator, current device, arguments) of each launch."""

    def __init__(self, monkeypatch, current):
        self.current, self.calls = current, []
        lib = pkg()._lib

        class Stream:
            cuda_stream = 4321

        @contextlib.contextmanager
        def device(d):
            was, self.current = self.current, d
            try:
                yield
            finally:
                self.current = was

        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: Stream)
        monkeypatch.setattr(torch.cuda, "device", device)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        monkeypatch.setattr(torch.cuda, "synchronize", lambda d=None: None)

        def entry(name, n):
            def call(packed, *rest):
                import struct
                self.calls.append((name, self.current, struct.unpack(f"{n}q", packed)))
                return 0
            return call

        monkeypatch.setattr(lib, "_fn_kv_append", lambda: entry("append", 35))
        monkeypatch.setattr(lib, "_fn_w4_linear", lambda: entry("w4", 15))
        size = lib.lib().qa_k_cache_attention_workspace
        monkeypatch.setattr(lib, "_fn_cache_attention", lambda: (entry("attend", 27), size))


def _there(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnDevice)


def _codes(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn).as_subclass(_OnDevice)


def _maps(n, pages, length):
    qs = torch.arange(n + 1, dtype=torch.int32).as_subclass(_OnDevice)
    kl = torch.full((n,), length, dtype=torch.int32).as_subclass(_OnDevice)
    tab = torch.arange(n * pages, dtype=torch.int32).view(n, pages).as_subclass(_OnDevice)
    return qs, kl, tab


def _append(n=2, pages=2, nkv=2, nq=4, hd=64, **kw):
    qs, kl, tab = _maps(n, pages, 70)
    kw = {**dict(max_q=1), **kw}
    pkg()._lib.kv_append(_there(n, nq * hd), _there(n, nkv * hd), _there(n, nkv * hd), _there(n, nq * hd), qs, kl, tab,
                         _codes(n * pages, nkv, PAGE, hd), _codes(n * pages, nkv, PAGE, hd),
                         kscale=_there(n * pages, nkv, dtype=torch.float32),
                         vscale=_there(n * pages, nkv, dtype=torch.float32), **kw)


def _attend(n=2, pages=2, nkv=2, nq=4, hd=64, **kw):
    qs, kl, tab = _maps(n, pages, 70)
    kw = {**dict(max_q=1, max_kv=70), **kw}
    pkg()._lib.cache_attention(_there(n, nq * hd), qs, kl, tab, _codes(n * pages, nkv, PAGE, hd),
                               _codes(n * pages, nkv, PAGE, hd), _there(n * pages, nkv, dtype=torch.float32),
                               _there(n * pages, nkv, dtype=torch.float32), _there(n, nq * hd), **kw)


def _w4(**kw):
    pkg()._lib.w4_linear(_there(3, 256), _there(10, 128, dtype=torch.uint8), _there(10, 2), _there(3, 10), **kw)


def test_the_attentions_workspace_belongs_to_the_launch_stream(monkeypatch):
    """Taken with the launch's stream current (a capture of that stream is seen, and
    memory given back is reused behind the call), and given back after the call."""
    import weakref
    gpu, on, taken = _Gpu(monkeypatch, 1), [4321], []

    @contextlib.contextmanager
    def stream(s):
        on.append(s)
        try:
            yield
        finally:
            on.pop()

    plain = torch.empty

    def empty(*shape, **kw):
        buf = plain(*shape, **kw)
        if kw.get("dtype") is torch.uint8:
            taken.append((on[-1], weakref.ref(buf)))
        return buf

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: handle)
    monkeypatch.setattr(torch, "empty", empty)
    for handle in (None, 77, 77):
        _attend(pages=40, max_kv=2500, stream=handle, validate=False)
    assert [s for s, _ in taken] == [4321, 77, 77] == [c[2][-1] for c in gpu.calls]
    assert all(buf() is None for _, buf in taken)
    assert all(c[2][22] and c[2][23] > 0 for c in gpu.calls)  # and it was passed on


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("op", [_append, _attend, _w4])
def test_a_call_launches_on_its_tensors_device(monkeypatch, op, current):
    gpu = _Gpu(monkeypatch, current)
    op()
    assert [c[1] for c in gpu.calls] == [1] and gpu.current == current
    assert gpu.calls[0][2][-1] == 4321  # the stream that was asked for there


@pytest.mark.parametrize("op", [_append, _attend])
def test_a_status_that_cannot_take_the_bits_is_refused(monkeypatch, op):
    gpu = _Gpu(monkeypatch, 1)
    for dtype, size in ((torch.int32, 0), (torch.uint8, 1), (torch.int16, 2), (torch.float32, 1), (torch.int64, 1)):
        with pytest.raises(ValueError, match="status"):
            op(status=_there(size, dtype=dtype))
    assert not gpu.calls
    op(status=_there(1, dtype=torch.int32))
    assert len(gpu.calls) == 1


def test_loose_bounds_are_cut_to_what_can_be(monkeypatch):
    """No sequence has more new tokens than there are rows, nor more cached ones than
    its pages hold: a caller that knows no better may give any bound."""
    gpu = _Gpu(monkeypatch, 1)
    for big in (3, 1 << 20, (1 << 31) - 1, 1 << 31, (1 << 32) + 1, 1 << 62):
        gpu.calls.clear()
        _append(n=2, max_q=big), _attend(n=2, pages=2, max_q=big, max_kv=64 * big)
        assert [gpu.calls[0][2][15], gpu.calls[1][2][9], gpu.calls[1][2][10]] == [2, 2, 128]
    gpu.calls.clear()
    _append(n=2, max_q=1), _attend(n=2, pages=2, max_q=1, max_kv=70)
    assert [gpu.calls[0][2][15], gpu.calls[1][2][9], gpu.calls[1][2][10]] == [1, 1, 70]


# ---------------------------------------------------------------- the session decoder

def _decoder(pages=4, **kw):
    import dataclasses
    cfg = dataclasses.replace(pkg().synth.ModelConfig(), **{**dict(
        num_layers=1, hidden_size=128, intermediate_size=128, num_heads=2, num_kv_heads=1, head_dim=64,
        vocab_size=50, num_labels=10, max_seq=256), **kw})
    g = torch.Generator().manual_seed(2)
    w = {name: (torch.randn(*shape, generator=g) * 0.04).to(torch.bfloat16)
         for name, shape, _ in pkg().synth.weight_specs(cfg)
         if "language_model" in name or name.startswith("score")}
    return pkg().incremental.SessionDecoder(cfg, w, pages=pages, device="cpu")


def _table(dec):
    t = dec.table
    return {s: (t.length(s), list(t.pages(s))) for s in t._len}, sorted(t._free)


@pytest.mark.parametrize("fails", ["w4_linear", "kv_append", "cache_attention", "device"])
def test_a_step_that_fails_leaves_the_sessions_as_they_were(monkeypatch, fails):
    """Whatever fails after the tokens were taken (memory, for one): the sessions do
    not count tokens that their caches do not hold, and the step can be repeated."""
    dec, lib = _decoder(pages=5), pkg()._lib

    def quiet(*a, **k):
        return None

    def loud(*a, **k):
        raise RuntimeError("no memory")

    for name in ("w4_linear", "kv_append", "cache_attention"):
        monkeypatch.setattr(lib, name, quiet)
    a, b = dec.open(), dec.open()
    dec.step({a: [1] * 60, b: [2]})
    before = _table(dec)
    with monkeypatch.context() as m:
        if fails == "device":
            m.setattr(torch.Tensor, "to", loud)
        else:
            m.setattr(lib, fails, loud)
        with pytest.raises(RuntimeError, match="no memory"):
            dec.step({a: [1] * 70, b: [], dec.open(): [3]})
    dec.close(max(dec.table._len))
    assert _table(dec) == before
    assert dec.step({a: [1] * 70, b: [4]}).shape == (71, 128)
    assert dec.table.length(a) == 130 and len(dec.table.pages(a)) == 3


def test_a_step_with_what_is_no_token_leaves_the_sessions_as_they_were():
    dec = _decoder()
    a = dec.open()
    for bad in (["x"], [None], [1, 2.5j]):
        with pytest.raises((TypeError, ValueError)):
            dec.step({a: bad})
    with pytest.raises(KeyError):
        dec.step({a: [1], a + 1: [1]})
    assert dec.table.length(a) == 0 and len(dec.table._free) == 4


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tiny_weights_keep_their_steps(dtype):
    """Half a step and half a step of the zero point; the step rounded to 16 bits moves
    the range's end by 15 u, or is up to 2^-24 longer where float16 has no more bits."""
    g = torch.Generator().manual_seed(6)
    w = torch.randn(14, 128, generator=g) * 10.0 ** -torch.arange(1, 8).repeat(2)[:, None]
    w[7:] = w[7:].abs()
    wq, scales, zeros = pkg().incremental.quantise4(w, 64, dtype)
    codes = torch.stack([wq & 15, wq >> 4], -1).reshape(14, 2, 64).double()
    back = scales.double()[..., None] * (codes - zeros.double()[..., None])
    w = w.double().reshape(14, 2, 64)
    step = (w.amax(-1).clamp(min=0) - w.amin(-1).clamp(max=0)) / 15
    u = 2.0 ** -11 if dtype is torch.float16 else 2.0 ** -8
    bound = step * (1 + 15 * 2 * u) + (2.0 ** -24 if dtype is torch.float16 else 0)
    assert ((back - w).abs() <= bound[..., None]).all()


def test_the_attentions_workspace_is_what_its_parts_need():
    """Many rows: 16 parts of 256 rows of a sequence and head at most, whatever their
    number, and as much for each sequence; nothing for arguments that are none."""
    size = pkg()._lib.lib().qa_k_cache_attention_workspace
    most = 16 * 4 * (256 * 128 + 2 * 256)
    for max_q in (128, 512, 1024, 8192, 100000):
        assert size(16, 8, 128, 1, max_q, 8192) <= 8 * most
        assert size(16, 8, 128, 8, max_q, 8192) == 8 * size(16, 8, 128, 1, max_q, 8192)
    assert size(16, 8, 128, 1, 1024, 700) <= 8 * most // 8
    for bad in ((0, 0, 128, 1, 64, 64), (16, 8, -2, 1, 64, 64), (16, 8, 128, 0, 64, 64), (16, 8, 128, 1, -5, 64)):
        assert size(*bad) == 0
    assert 0 < size(16, 8, 128, 1 << 30, (1 << 31) - 1, (1 << 31) - 1) <= 1 << 30
