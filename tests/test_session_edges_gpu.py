"""Edges of the operators of growing sessions, against the same plain
implementations in 64 bits and with the same bounds as test_session_ops_gpu.py:
zero points over the whole byte, scales below the normal range, any number of
rows, launches that fail; axes that are not there, any heads and tokens of a
CTA, calls without tables; bounds that say nothing, captures of a stream that is
not the current one, workspaces of any size, a sequence's company, many rows in
many chunks, many sequences, wide groups of heads, NaN codes that only some rows
see."""
import pytest

from conftest import cuda_ok, pkg
from test_session_ops_gpu import (PAGE, _append_case, _append_run, _attn_case, _attn_run, _check_append, _check_attn,
                                  _check_w4, _split, _w4_case)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_cuda():
    if not cuda_ok():
        pytest.skip("no CUDA device")


# ---------------------------------------------------------------- w4_linear

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,pad", [(1, 0), (13, 0), (5, 1)])
def test_w4_zero_points_are_any_byte(dtype, group, m, pad):
    """A zero point is a byte; codes only reach 15.  Each value meets every code,
    on rows that are read 16 bytes at a time and (pad) on rows that are not.
    A group's f32 sum holds terms of up to 255 |x|, inside the bound's sum."""
    import torch
    n, k = 512, 16 * group
    c = _w4_case(m, n, k, group, dtype, True, False, seed=group + m)
    edge = torch.tensor([0, 15, 16, 63, 64, 65, 127, 128, 129, 191, 192, 240, 241, 254, 255, 8], dtype=torch.uint8)
    c["zeros"][:16] = edge[(torch.arange(16)[:, None] + torch.arange(16)[None]) % 16]
    c["zeros"][16:] = torch.arange((n - 16) * 16).view(-1, 16) % 256
    x = torch.zeros(m, k + pad, dtype=c["x"].dtype, device="cuda")[:, pad:]
    x.copy_(c["x"])
    out = torch.full((m, n), float("nan"), dtype=c["x"].dtype, device="cuda")
    pkg()._lib.w4_linear(x, c["wq"].cuda(), c["scales"].cuda(), out, zeros=c["zeros"].cuda())
    _check_w4(c, out)

@pytest.mark.parametrize("pad", [0, 1])
def test_w4_scales_below_the_normal_range(pad):
    """What quantise4 gives for tiny weights in f16: steps of 2^-24 and up."""
    import torch
    m, n, k = 5, 200, 1024
    c = _w4_case(m, n, k, 64, "f16", True, True, seed=61)
    c["scales"] = (torch.randint(1, 1024, c["scales"].shape, generator=torch.Generator().manual_seed(62)) * 2.0 ** -24).half()
    c["x"] = c["x"] * 512
    x = torch.zeros(m, k + pad, dtype=torch.float16, device="cuda")[:, pad:]
    x.copy_(c["x"])
    out = torch.empty(m, n, dtype=torch.float16, device="cuda")
    pkg()._lib.w4_linear(x, c["wq"].cuda(), c["scales"].cuda(), out, zeros=c["zeros"].cuda(), bias=c["bias"].cuda())
    _check_w4(c, out)


def test_w4_takes_any_number_of_rows():
    """More rows than a grid has blocks for; compared where the pieces meet and at the
    ends."""
    import torch
    at = 65535 * 16
    m = at + 3
    c = _w4_case(40, 6, 32, 32, "bf16", True, True, seed=67)
    x = torch.zeros(m, 32, dtype=torch.bfloat16, device="cuda")
    rows = list(range(16)) + list(range(at - 16, at + 3))
    c["x"] = c["x"][: len(rows)]
    x[torch.tensor(rows, device="cuda")] = c["x"].cuda()
    out = torch.full((m, 6), float("nan"), dtype=torch.bfloat16, device="cuda")
    pkg()._lib.w4_linear(x, c["wq"].cuda(), c["scales"].cuda(), out, zeros=c["zeros"].cuda(), bias=c["bias"].cuda())
    _check_w4(c, out[torch.tensor(rows, device="cuda")])
    assert bool((out[16: at - 16] == c["bias"].cuda().bfloat16()).all())


def test_a_launch_that_fails_is_not_told_to_the_next_caller():
    """A stream whose capture has been invalidated takes no launch.  The call says so,
    and the runtime's record of errors is as clean as before."""
    import ctypes
    import torch
    rt = ctypes.CDLL("libcudart.so.12")
    c = _w4_case(2, 64, 128, 128, "f16", False, False, seed=83)
    x, wq, scales, out = c["x"].cuda(), c["wq"].cuda(), c["scales"].cuda(), torch.empty(2, 64, device="cuda").half()
    s = torch.cuda.Stream()
    pkg()._lib.w4_linear(x, wq, scales, out, stream=s.cuda_stream)
    torch.cuda.synchronize()
    stream, graph = ctypes.c_void_p(s.cuda_stream), ctypes.c_void_p()
    assert rt.cudaStreamBeginCapture(stream, 2) == 0
    try:
        assert rt.cudaStreamSynchronize(stream) != 0  # not while it captures
        rt.cudaGetLastError()
        with pytest.raises(pkg().QaError):
            pkg()._lib.w4_linear(x, wq, scales, out, stream=s.cuda_stream)
        left = rt.cudaPeekAtLastError()
    finally:
        rt.cudaStreamEndCapture(stream, ctypes.byref(graph))
        rt.cudaGetLastError()
    assert left == 0
    pkg()._lib.w4_linear(x, wq, scales, out, stream=s.cuda_stream)
    torch.cuda.synchronize()
    _check_w4(c, out)


# ---------------------------------------------------------------- kv_append

@pytest.mark.parametrize("bits", [8, 16])
def test_append_reports_an_axis_that_is_not_there(bits):
    """Without `validate`, an axis outside [0, axes) sets the status and counts as
    the first axis; the other frequencies are not affected."""
    import torch
    c = _append_case([(5, 70), (3, 3)], "f16", 64, 4, 2, bits, False, 3, seed=11)
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    q, k, v = _split(c, d["packed"])

    def run(axis_of):
        st, q_out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty_like(q)
        scales = {n: None if d[n] is None else d[n].clone() for n in ("kscale", "vscale")}
        pkg()._lib.kv_append(q, k, v, q_out, d["q_start"], d["kv_len"], d["tab"], d["kpool"].clone(),
                             d["vpool"].clone(), max_q=5, cos=d["cos"], sin=d["sin"], pos=d["pos"],
                             axis_of=axis_of.cuda(), status=st, validate=False, **scales)
        return int(st.item()), q_out

    assert run(c["axis_of"])[0] == 0
    for bad in (3, 4, 7, -1, 1 << 30, -(1 << 31)):
        axis, as_first = c["axis_of"].clone(), c["axis_of"].clone()
        axis[17], as_first[17] = bad, 0
        status, q_out = run(axis)
        assert status == 2, bad
        assert torch.equal(q_out, run(as_first)[1]), bad


@pytest.mark.parametrize("hd,bits", [(128, 8), (128, 16), (64, 8), (64, 16)])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 10, 14, 22, 46])
@pytest.mark.parametrize("n", [1, 2, 8, 16, 33, 64])
def test_append_of_any_group_and_number_of_tokens(hd, bits, group, n):
    """The heads of a CTA and its tokens make its shared memory: each size launches.
    (48 KB with the kernel's own variables is where a launch has to ask for more.)"""
    c = _append_case([(n, n + 70), (1, 1)], "f16", hd, group, 1, bits, False, 0, seed=group)
    _check_append(c, _append_run(c))


def _append_c(c, max_q, n_axes=1, axis_of=0):
    """Through the C entry, without tables or positions: what a caller may leave out."""
    import torch
    L = pkg()._lib
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    q, k, v = _split(c, d["packed"])
    q_out, st = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = L.lib().qa_k_kv_append(
        q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), q_out.data_ptr(),
        q_out.stride(0), q.shape[0], c["nq"], c["nkv"], c["hd"], d["q_start"].data_ptr(), d["kv_len"].data_ptr(),
        len(c["seqs"]), max_q, d["tab"].data_ptr(), d["tab"].shape[1], d["kpool"].data_ptr(), d["vpool"].data_ptr(),
        c["pages"], d["kscale"].data_ptr(), d["vscale"].data_ptr(), 0, 0, 0, 0, 0, n_axes, axis_of, 0, 0, 1e-6,
        1 if c["dtype"] == "bf16" else 0, st.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    c = dict(c, cos=torch.ones_like(c["cos"]), sin=torch.zeros_like(c["sin"]))  # what no rotation amounts to
    return rc, int(st.item()), c, {n: x.cpu() for n, x in dict(q=q_out, kpool=d["kpool"], vpool=d["vpool"],
                                                               kscale=d["kscale"], vscale=d["vscale"]).items()}


def test_append_without_tables_reads_no_axes():
    c = _append_case([(70, 75), (1, 9)], "bf16", 128, 4, 2, 8, False, 0, seed=13)
    rc, status, c, got = _append_c(c, 70, n_axes=3)
    assert rc == 0 and status == 0
    _check_append(c, got)


@pytest.mark.parametrize("max_q", [71, 1 << 20, (1 << 31) - 1])
def test_append_with_a_bound_that_says_nothing(max_q):
    c = _append_case([(70, 75), (1, 9)], "f16", 64, 4, 2, 8, False, 0, seed=13)
    rc, status, c, got = _append_c(c, max_q)
    assert rc == 0 and status == 0
    _check_append(c, got)


# ---------------------------------------------------------------- cache_attention

def test_attention_captured_on_a_stream_that_is_not_the_current_one():
    import torch
    c = _attn_case([(1, 5000), (1, 3100)], "f16", 128, 16, 8, seed=43)
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    out, lse = torch.empty_like(d["buf"]), torch.empty(2, 16, device="cuda")

    def run(stream):
        pkg()._lib.cache_attention(d["buf"], d["q_start"], d["kv_len"], d["tab"], d["kpool"], d["vpool"], d["kscale"],
                                   d["vscale"], out, lse=lse, max_q=1, max_kv=5000, stream=stream, validate=False)

    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    run(s.cuda_stream)
    torch.cuda.synchronize()
    want = out.clone()
    with torch.cuda.stream(s):
        graph.capture_begin()
    run(s.cuda_stream)
    with torch.cuda.stream(s):
        graph.capture_end()
    for _ in range(2):
        out.zero_(), lse.zero_()
        graph.replay()
        run(s.cuda_stream)  # does not work in the graph's memory
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    _check_attn(c, (c["buf"], out.cpu(), lse.cpu()))


def _attend_c(c, max_q, max_kv, workspace=None, causal=1):
    """Through the C entry, in a workspace of the caller's (none: a null pointer)."""
    import torch
    L = pkg()._lib
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    q, out = d["buf"], torch.full_like(d["buf"], float("nan"))
    lse = torch.full((q.shape[0], c["nq"]), float("nan"), device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = 0 if workspace is None else workspace.data_ptr()
    rc = L.lib().qa_k_cache_attention(
        q.data_ptr(), q.stride(0), q.shape[0], c["nq"], c["nkv"], c["hd"], d["q_start"].data_ptr(),
        d["kv_len"].data_ptr(), len(c["seqs"]), max_q, max_kv, d["tab"].data_ptr(), d["tab"].shape[1],
        d["kpool"].data_ptr(), d["vpool"].data_ptr(), c["pages"], d["kscale"].data_ptr(), d["vscale"].data_ptr(),
        c["hd"] ** -0.5, causal, out.data_ptr(), out.stride(0), lse.data_ptr(), ws,
        0 if workspace is None else workspace.numel(), 1 if c["dtype"] == "bf16" else 0, st.data_ptr(),
        torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0 and int(st.item()) == 0
    return c["buf"], out.cpu(), lse.cpu()


@pytest.mark.parametrize("seqs", [[(1, 200), (1, 2100)], [(40, 300), (1, 1500)]])
@pytest.mark.parametrize("bound", [1 << 20, (1 << 31) - 1])
def test_attention_with_bounds_that_say_nothing(seqs, bound):
    c = _attn_case(seqs, "bf16", 64, 14, 2, seed=47)
    _check_attn(c, _attend_c(c, bound, bound))


def _workspace(c, n_seqs, max_q, max_kv):
    import torch
    size = pkg()._lib.lib().qa_k_cache_attention_workspace(c["nq"], c["nkv"], c["hd"], n_seqs, max_q, max_kv)
    return torch.empty(size, dtype=torch.uint8, device="cuda")


def _only(c, s):
    """Sequence s of a case by itself."""
    a, b = int(c["q_start"][s]), int(c["q_start"][s + 1])
    return dict(c, seqs=[c["seqs"][s]], buf=c["buf"][a:b].contiguous(), q_start=c["q_start"][s: s + 2] - a,
                kv_len=c["kv_len"][s: s + 1], tab=c["tab"][s: s + 1].contiguous())


COMPANY = [
    [(1, 5000), (1, 20), (1, 3000), (0, 100)],
    [(12, 5000), (3, 2100), (12, 1025)],
    [(300, 2500), (129, 1500), (1, 3000), (40, 2000)],
    # eight sessions, the last of them beside one that brings far more tokens
    [(1024, 8192)] + [(16, 1200)] * 6 + [(16, 8192)],
]


@pytest.mark.parametrize("dtype,hd,nq,nkv", [("f16", 128, 16, 8), ("bf16", 64, 14, 2)])
@pytest.mark.parametrize("seqs", COMPANY, ids=range(len(COMPANY)))
def test_attention_of_a_sequence_does_not_depend_on_the_others(seqs, dtype, hd, nq, nkv):
    """The same bits alone and at any place of a batch of one max_q."""
    import torch
    c = _attn_case(seqs, dtype, hd, nq, nkv, seed=53)
    max_q, max_kv = max(n for n, _ in seqs), max(L for _, L in seqs)
    _, out, lse = _attend_c(c, max_q, max_kv, _workspace(c, len(seqs), max_q, max_kv))
    for s in range(len(seqs)):
        a, b = int(c["q_start"][s]), int(c["q_start"][s + 1])
        if a == b:
            continue
        # max_q counts as the rows that there are: rows of nobody keep it
        one = _only(c, s)
        one["buf"] = torch.cat([one["buf"], one["buf"].new_zeros(max_q - (b - a), nq * hd)])
        _, o, e = _attend_c(one, max_q, max_kv, _workspace(c, 1, max_q, max_kv))
        assert torch.equal(o[: b - a], out[a:b]) and torch.equal(e[: b - a], lse[a:b])


@pytest.mark.parametrize("dtype,hd,nq,nkv", [("f16", 128, 16, 8), ("bf16", 64, 14, 2)])
@pytest.mark.parametrize("seqs", COMPANY[:3], ids=range(3))
def test_attention_in_a_workspace_of_any_size(seqs, dtype, hd, nq, nkv):
    """None, and some of what is asked for: sequences without a place are not split."""
    import torch
    c = _attn_case(seqs, dtype, hd, nq, nkv, seed=59)
    max_q, max_kv = max(n for n, _ in seqs), max(L for _, L in seqs)
    whole = _workspace(c, len(seqs), max_q, max_kv)
    want = _attend_c(c, max_q, max_kv, whole)
    _check_attn(c, want)
    _check_attn(c, _attend_c(c, max_q, max_kv))
    one = whole.numel() // len(seqs)
    for bytes_ in (16, one - 16, one, one + 16, whole.numel() - 16):
        room = torch.full((whole.numel(),), 0x7F, dtype=torch.uint8, device="cuda")
        got = _attend_c(c, max_q, max_kv, room[:bytes_])
        assert bool((room[bytes_:] == 0x7F).all())
        _check_attn(c, got)
        if bytes_ >= one:
            n = int(c["q_start"][1])
            assert torch.equal(got[1][:n], want[1][:n]) and torch.equal(got[2][:n], want[2][:n])


MANY = [
    [(300, 2500), (129, 1500), (1, 3000)],  # units of two and of one tile of rows, one to three chunks
    [(700, 1400), (64, 1100), (256, 256)],  # every token hidden from some rows, in two chunks
    [(1100, 1100), (5, 9000)],              # many units of one chunk beside one of many
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("seqs", MANY, ids=range(len(MANY)))
@pytest.mark.parametrize("dtype,hd,nq,nkv", [("f16", 128, 16, 8), ("bf16", 128, 14, 2), ("f16", 64, 14, 2),
                                             ("bf16", 64, 16, 8), ("bf16", 128, 5, 5)])
def test_attention_of_many_rows_in_many_chunks(dtype, hd, nq, nkv, seqs, causal):
    c = _attn_case(seqs, dtype, hd, nq, nkv, seed=71)
    _check_attn(c, _attn_run(c, causal), causal, device="cuda")


def _spoil(c, pool, at):
    """NaN codes at (sequence, token, head, dims); returns the case with zeros there."""
    import torch
    clean = dict(c, **{pool: c[pool].clone()})
    for s, token, head, dims in at:
        page = int(c["tab"][s, token // PAGE])
        for x, code in ((c, 0x7F), (clean, 0)):
            x[pool].view(torch.uint8)[page, head, token % PAGE, dims] = code
    return clean


SPOILED = [
    ([(70, 200), (33, 300)], [131, 180, 199]),           # one unit a head, its streams' key tiles
    ([(300, 2500), (40, 2500)], [2250, 2330, 2460, 2499]),  # units of two tiles of rows and of one, the last chunk
    ([(700, 1400), (20, 1400)], [705, 900, 1050, 1399]),  # in the first chunk and in the second
    ([(3, 100), (2, 3000)], [98, 99]),                     # few rows
    ([(8, 3000), (12, 2000)], [2993, 2998, 2999]),         # few rows, the last chunk
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("seqs,tokens", SPOILED, ids=range(len(SPOILED)))
@pytest.mark.parametrize("dtype,hd,nq,nkv", [("f16", 128, 4, 2), ("bf16", 64, 6, 3)])
def test_attention_keeps_nan_values_to_the_rows_and_dims_that_see_them(dtype, hd, nq, nkv, seqs, tokens, causal):
    """NaN codes of V of the first sequence: its last rows see them, the others not."""
    import torch
    c = _attn_case(seqs, dtype, hd, nq, nkv, seed=73)
    n, L = seqs[0]
    at = [(0, t, i % nkv, [3 * i, hd // 2 + i, hd - 1 - i]) for i, t in enumerate(tokens)]
    clean = _attn_run(_spoil(c, "vpool", at), causal)
    _, out, lse = _attn_run(c, causal)
    want = torch.zeros(out.shape[0], nkv, nq // nkv, hd, dtype=torch.bool)
    for _, t, head, dims in at:
        want[max(0, t - (L - n)) if causal else 0: n, head][..., dims] = True
    want = want.view(out.shape[0], -1)
    assert torch.equal(out.isnan(), want)
    assert torch.equal(out.masked_fill(want, 0), clean[1].masked_fill(want, 0)) and torch.equal(lse, clean[2])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("seqs,tokens", SPOILED, ids=range(len(SPOILED)))
def test_attention_keeps_nan_keys_to_the_rows_that_see_them(seqs, tokens, causal):
    import torch
    nq, nkv, hd = 4, 2, 128
    c = _attn_case(seqs, "f16", hd, nq, nkv, seed=79)
    n, L = seqs[0]
    t = tokens[-2]
    clean = _attn_run(_spoil(c, "kpool", [(0, t, 1, [5])]), causal)
    _, out, lse = _attn_run(c, causal)
    want = torch.zeros(out.shape[0], nkv, nq // nkv, dtype=torch.bool)
    want[max(0, t - (L - n)) if causal else 0: n, 1] = True
    want = want.view(-1, nq)
    assert torch.equal(lse.isnan(), want)
    bad = want[..., None].expand(-1, -1, hd).reshape(out.shape)
    assert torch.equal(out.isnan(), bad)
    assert torch.equal(out[~bad], clean[1][~bad]) and torch.equal(lse[~want], clean[2][~want])


def _crowd(count, most, length, seed):
    """Many sequences, some without new tokens, some without any."""
    import random
    r = random.Random(seed)
    seqs = [(r.choice([0, 1, 1, most, r.randint(1, most)]), r.choice([0, 1, 64, r.randint(1, length)])) for _ in range(count)]
    return [(min(n, max(L, 1)), max(L, min(n, 1))) for n, L in seqs]


@pytest.mark.parametrize("most,length", [(1, 300), (1, 2600), (70, 500)])
@pytest.mark.parametrize("count", [129, 449, 1500])
def test_attention_of_many_sequences(count, most, length):
    """More of them than a CTA has threads to look for its share with."""
    seqs = _crowd(count, most, length, seed=count)
    c = _attn_case(seqs, "f16", 64, 4, 2, seed=89)
    _check_attn(c, _attn_run(c))


def test_append_of_many_sequences():
    seqs = _crowd(1500, 70, 500, seed=97)
    c = _append_case([(min(n, L), L) for n, L in seqs], "bf16", 64, 4, 2, 8, True, 0, seed=97)
    _check_append(c, _append_run(c))


@pytest.mark.parametrize("seqs", [[(1, 300), (1, 1)], [(3, 2000), (2, 64)]])
@pytest.mark.parametrize("nq", [24, 25, 300, 520])
def test_attention_of_wide_groups(nq, seqs):
    """A single token's heads of one K/V head fill a tile of rows, or several."""
    c = _attn_case(seqs, "bf16", 64, nq, 1, seed=101)
    _check_attn(c, _attn_run(c))
