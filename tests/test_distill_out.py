"""Where ``distill_loss_and_grad`` may write its gradient: rows apart from one another,
and from the logits' or the same."""

import itertools

import pytest
import torch

from test_distill import make


def overlap(x, y=None):
    """By every element's address."""
    def elements(z):
        at = torch.zeros((), dtype=torch.int64)
        for n, st in zip(z.shape, z.stride()):
            at = at[..., None] + torch.arange(n) * st
        return (at * z.element_size() + z.data_ptr()).flatten().tolist()

    mine = elements(x)
    return len(set(mine)) < len(mine) if y is None else bool(set(mine) & set(elements(y)))


def refused(out, logits):
    from autoindexer_b200.distill import check_out

    try:
        check_out(out, logits)
    except ValueError:
        return True
    return False


def test_rows_of_any_strides():
    base, logits = torch.zeros(400), torch.zeros(3, 4, 5)
    seen = set()
    for shape in ((3, 4, 5), (2, 2, 5), (1, 3, 4), (6, 5), (1, 5)):
        for st in itertools.product((0, 1, 4, 5, 6, 10, 11, 15, 20, 25), repeat=len(shape) - 1):
            x = base.as_strided(shape, (*st, 1))
            assert refused(x, torch.zeros(shape)) == overlap(x), (shape, st)
            seen.add(overlap(x))
    assert seen == {True, False} and not refused(logits, logits)


def test_the_logits_and_other_places():
    base = torch.zeros(2000)
    seen = set()
    logits = base.as_strided((3, 4, 5), (40, 10, 1), 700)
    for st in ((40, 10), (10, 30), (20, 5), (120, 10), (40, 11)):
        for at in range(560, 840):
            x = base.as_strided((3, 4, 5), (*st, 1), at)
            same = at == 700 and st == (40, 10)
            want = overlap(x) or (overlap(x, logits) and not same)
            assert refused(x, logits) == want, (st, at)
            seen.add((st, want))
    assert len(seen) >= 9
    one = base.as_strided((1, 4, 5), (7, 10, 1), 3)
    assert not refused(one, base.as_strided((1, 4, 5), (900, 10, 1), 3))  # (a stride of one row says nothing)


@pytest.mark.gpu
def test_refusals_and_neighbours(cuda_device):
    from autoindexer_b200 import distill_loss_and_grad

    x, ids, t, w, tau = (y.to(cuda_device) for y in make((3, 4), 100, 5, torch.float32, 2))
    want = distill_loss_and_grad(x, ids, t, w, tau)
    base = torch.zeros(3, 4, 2, 100, device=cuda_device)
    base[:, :, 0] = x
    logits, beside = base[:, :, 0], base[:, :, 1]  # (rows between the logits' rows)
    got = distill_loss_and_grad(logits, ids, t, w, tau, out=beside)
    assert torch.equal(got[0], want[0]) and torch.equal(beside, want[1]) and torch.equal(logits, x)
    flat = base.view(-1)
    for bad in (flat.as_strided((3, 4, 100), (400, 99, 1)), flat.as_strided((3, 4, 100), (800, 0, 1)),
                flat.as_strided((3, 4, 100), (800, 200, 1), 1), flat.as_strided((3, 4, 100), (800, 200, 1), 60)):
        before = base.clone()
        with pytest.raises(ValueError, match="share memory|overlaps"):
            distill_loss_and_grad(logits, ids, t, w, tau, out=bad)
        assert torch.equal(base, before)
    got = distill_loss_and_grad(logits, ids, t, w, tau, out=logits)
    assert torch.equal(logits, want[1]) and torch.equal(base[:, :, 1], want[1])
