"""-m gpu: the top of bf16 rows whose logits are mostly or all negative, as trained scores and log-probabilities are: the answers, and that they cost what those
of rows around zero cost.  Tolerances as in test_rows_gpu.py."""
import numpy as np
import pytest
import torch

from test_rows_gpu import DEV, check_top, gpu, strided  # noqa: F401  (gpu: the fixture that skips without one)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [9, 700, 5000, 16384, 40000])
def test_rows_below_zero(hip, kind, n):
    """All negative; negative but for a few, fewer than k, around k; masked in part; -0 the largest; one value, of many ties; NaN among them."""
    rng = np.random.default_rng(n)
    z = rng.standard_normal((9, n)) - 10.0
    z[1, rng.permutation(n)[:3]] = 2.0
    z[2, rng.permutation(n)[:min(n, 70)]] = np.linspace(1, 3, min(n, 70))
    z[3, rng.random(n) < 0.5] = -np.inf
    z[4, rng.random(n) < 0.9] = -np.inf
    z[5, ::3] = -0.0
    z[6] = -7.0
    z[7] = -np.arange(n) / 256.0 - 1
    z[8, rng.random(n) < 0.3] = 0.0
    for k in sorted({1, min(n, 64), min(n, 250)}):
        for lead in (0, 1):
            check_top(hip, strided(z, kind, lead, 3)[1], k, 1.0)


def time_of(call, repeats=15):
    for _ in range(3):
        call()
    times = []
    for _ in range(repeats):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    return sorted(times)[repeats // 2]


def test_the_sign_of_a_row_costs_nothing(hip):
    """256 x 400 000 bf16, k = 64, by the device's clock: rows around zero against rows of log-probabilities, negative scores and masked
    negative scores.  The work is the same; half as much again is allowed for the clock and for how many elements reach the bound.  (The exact
    way, which rows take whose elements all pass, costs several times as much.)"""
    rows, n, k = 256, 400000, 64
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    values, index = torch.empty(rows, k, device=DEV), torch.empty(rows, k, dtype=torch.int32, device=DEV)
    stats = torch.empty(rows, 2, device=DEV)
    noise = torch.randn(rows, n, generator=g, device=DEV)

    def cost(z):
        return time_of(lambda: hip.top_logits(z, values, index, stats))

    around = cost((2 * noise).bfloat16())
    negative = {"N(-10, 2)": 2 * noise - 10, "N(-3.5, 1.6)": 1.6 * noise - 3.5, "log-probabilities": torch.log_softmax(noise, 1)}
    negative["half of N(-10, 2) masked"] = torch.where(torch.rand(rows, n, generator=g, device=DEV) < 0.5, 2 * noise - 10, -float("inf"))
    costs = {name: cost(z.bfloat16()) for name, z in negative.items()}
    assert all(c <= 1.5 * around for c in costs.values()), (around, costs)
