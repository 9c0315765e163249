"""-m gpu: more rows than one launch takes (2^21 workgroups): top_logits and distillation on both sides of the border between launches."""
import numpy as np
import pytest
import torch

import rows_oracle
from test_rows_gpu import DEV, gpu, numbers  # noqa: F401  (gpu: the fixture that skips without one)

pytestmark = pytest.mark.gpu
LAUNCH = 1 << 21
ROWS = LAUNCH + 3


@pytest.fixture(scope="module")
def short():
    g = torch.Generator(device=DEV)
    g.manual_seed(0)
    return torch.randn(ROWS, 8, generator=g, device=DEV)


def test_top_logits(hip, short):
    values, index = torch.full((ROWS, 3), 77.0, device=DEV), torch.full((ROWS, 3), 77, dtype=torch.int32, device=DEV)
    stats = torch.full((ROWS, 2), 77.0, device=DEV)
    hip.top_logits(short, values, index, stats)
    want = torch.sort(short, dim=1, descending=True, stable=True)
    assert torch.equal(values, want.values[:, :3]) and torch.equal(index.long(), want.indices[:, :3])
    exact = torch.logsumexp(short.double(), 1) - short.double().amax(1)
    assert torch.equal(stats[:, 0], short.amax(1)) and float((stats[:, 1].double() - exact).abs().max()) <= 1e-5


@pytest.mark.parametrize("alone", [False, True])
def test_distill(hip, short, alone):
    """The step, one launch a row; and the gradient alone, which goes through the workspace."""
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    index = torch.randint(-1, 8, (ROWS, 4), generator=g, device=DEV, dtype=torch.int32)
    teacher = torch.randn(ROWS, 4, generator=g, device=DEV)
    weight = torch.rand(ROWS, generator=g, device=DEV)
    loss, stats, grad = torch.full((ROWS,), 77.0, device=DEV), torch.full((ROWS, 2), 77.0, device=DEV), torch.full((ROWS, 8), 77.0, device=DEV)
    hip.distill(short, index, teacher, loss, stats, weight=weight, grad=None if alone else grad)
    if alone:
        hip.distill_grad(short, index, teacher, stats, grad, weight=weight)
    z = short.double()
    entry = index >= 0
    t = torch.where(entry, teacher.double(), -float("inf"))
    q = torch.where(entry.any(1, keepdim=True), torch.softmax(t, 1), 0.0)
    log_p = torch.log_softmax(z, 1)
    terms = torch.where(q > 0, q * (torch.log(q) - log_p.gather(1, index.clamp(min=0).long())), 0.0)
    sizes = torch.where(q > 0, q * (torch.log(q).abs() + log_p.gather(1, index.clamp(min=0).long()).abs() + 1), 0.0)
    assert bool(((loss.double() - terms.sum(1)).abs() <= 2e-5 * sizes.sum(1)).all())
    listed = torch.zeros_like(z).scatter_add_(1, index.clamp(min=0).long(), q)
    p = log_p.exp() * q.sum(1, keepdim=True)
    w = weight.double()[:, None]
    # test_rows_gpu.py's tolerance of a gradient: 2e-5 of its terms, and half a step
    assert bool(((grad.double() - w * (p - listed)).abs() <= 2e-5 * w * (p + listed) + 2.0 ** -24 * (w * (p - listed)).abs() + 2.0 ** -126).all())


def test_top_logits_of_rows_in_slices(hip):
    """Rows of two slices: a launch takes 2^20 of them; 34 GB of logits, of which the rows around the border are looked at."""
    n, launch = 16400, 1 << 20
    rows = launch + 2
    logits = torch.empty(rows, n, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    logits[:2048].normal_(generator=g)
    for first in range(2048, rows, 2048):
        logits[first:first + 2048] = logits[:min(2048, rows - first)]
    looked = [0, 1, launch - 2, launch - 1, launch, launch + 1]
    for i, row in enumerate(looked):
        logits[row].normal_(mean=float(i - 2), generator=g)
    values, index = torch.empty(rows, 5, device=DEV), torch.empty(rows, 5, dtype=torch.int32, device=DEV)
    stats = torch.empty(rows, 2, device=DEV)
    hip.top_logits(logits, values, index, stats)
    want_values, want_index, want_stats = rows_oracle.top(numbers(logits[looked]), 5, 1.0)
    np.testing.assert_array_equal(index[looked].cpu().numpy(), want_index)
    np.testing.assert_array_equal(numbers(values[looked]), want_values)
    np.testing.assert_allclose(numbers(stats[looked]), want_stats, rtol=0, atol=1e-5)
    same = torch.arange(2048 + 5, rows - 2, 2048, device=DEV)  # copies of row 5, all along
    assert bool((index[same] == index[5]).all()) and bool((values[same] == values[5]).all()) and bool((stats[same] == stats[5]).all())
