"""Host logic of growing sessions: 4-bit codes and the page table."""
import pytest
import torch

from conftest import pkg


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantised_weights_are_within_a_step(group, dtype):
    g = torch.Generator().manual_seed(3)
    w = torch.randn(24, 256, generator=g) * 0.02
    w[3] = 0          # nothing to scale by
    w[4] = w[4].abs()  # no negative side
    w[5] += 1          # a range away from zero
    wq, scales, zeros = pkg().incremental.quantise4(w, group, dtype)
    assert wq.shape == (24, 128) and scales.dtype is dtype and int(zeros.max()) <= 15
    codes = torch.stack([wq & 15, wq >> 4], -1).reshape(24, -1, group).double()
    s = scales.double()[..., None]
    back = s * (codes - zeros.double()[..., None])
    # half a step, and half a step of the rounded zero point or the rounded scale's 15 steps
    u = 2.0 ** -11 if dtype is torch.float16 else 2.0 ** -8
    err = (back - w.double().reshape(24, -1, group)).abs()
    assert (err <= s * (1 + 15 * 2 * u) + 1e-12).all()
    assert (back.reshape(24, -1)[3] == 0).all()


def test_groups_that_do_not_divide_are_refused():
    for shape, group in (((4, 96), 64), ((4, 128), 16)):
        with pytest.raises(ValueError):
            pkg().incremental.quantise4(torch.zeros(shape), group)


def test_page_table_hands_out_each_page_once_and_takes_them_back():
    t = pkg().incremental.PageTable(6)
    a, b = t.open(), t.open()
    t.extend({a: 64, b: 1})
    t.extend({a: 1, b: 0})
    assert (t.length(a), t.length(b)) == (65, 1)
    assert len(t.pages(a)) == 2 and len(t.pages(b)) == 1
    assert len(set(t.pages(a) + t.pages(b))) == 3
    before = (list(t.pages(a)), list(t.pages(b)))
    with pytest.raises(MemoryError):
        t.extend({a: 64, b: 200})
    assert (t.pages(a), t.pages(b)) == before and t.length(a) == 65
    t.close(a)
    t.extend({b: 64 * 6 - 1})
    assert sorted(t.pages(b)) == list(range(6))
    t.close(b)
    c = t.open()
    assert c not in (a, b) and t.length(c) == 0
