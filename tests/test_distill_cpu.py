"""What GraphSolver.distill begins with, on the CPU: the tables of a solver that was only built, and the default learning rate."""
import numpy as np
import pytest
import torch

from graphvite_amd import scorer


@pytest.mark.parametrize("dim", [32, 128, 512])
def test_a_built_solver_s_tables_begin_alive(dim):
    vertex, context = scorer.start_tables(2000, dim, 7)
    assert vertex.shape == context.shape == (2000, dim) and vertex.dtype == context.dtype == torch.float32
    assert not torch.equal(vertex, context)
    again = scorer.start_tables(2000, dim, 7)
    assert torch.equal(again[0], vertex) and torch.equal(again[1], context)
    assert not torch.equal(scorer.start_tables(2000, dim, 8)[0], vertex)
    logits = (vertex @ context.t()).double()
    # 1/4 in expectation; over 4000 rows of dim >= 32 numbers its estimate is within 2 % many times over (the second moments' own error: 1 / sqrt(64000))
    assert abs(float(logits.std()) - 0.25) < 0.005


@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0])
@pytest.mark.parametrize("rows,n,k,batch", [(1, 5, 2, 1), (40, 300, 7, 16), (1000, 100, 20, 256)])
def test_the_default_rate_is_its_formula_s(rows, n, k, batch, temperature):
    rng = np.random.default_rng(n + k)
    z = rng.standard_normal((rows, n)) * 2 + 3 * (np.arange(n) == 1)  # candidate 1 is on most lists
    index = np.argsort(-z, 1)[:, :k]
    values = np.take_along_axis(z, index, 1)
    m = z.max(1)
    stats = np.stack([m, np.log(np.exp((z - m[:, None]) / temperature).sum(1))], 1)
    q = np.exp((values - stats[:, :1]) / temperature - stats[:, 1:])
    shares = np.zeros(n)
    np.add.at(shares, index, q)
    want = temperature ** 2 / (2 * q.sum() / rows * max(1.0, batch * shares.max() / q.sum()))
    as_float = lambda a: torch.from_numpy(a.astype(np.float32))  # noqa: E731
    rate = scorer.default_rate(torch.from_numpy(index.astype(np.int32)), as_float(values), as_float(stats), temperature, batch, n)
    # inputs and the exponential in 32 bits (arguments up to 40 in size: 40 * 3 * 2^-24), shares in steps of 2^-30 of at least 1 / n
    assert abs(rate - want) <= 1e-5 * want
    if batch == 256:
        assert batch * shares.max() / q.sum() > 1  # the batch's part of the rule is at work here


def test_no_nodes_no_trouble():
    assert scorer.default_rate(torch.zeros(0, 3, dtype=torch.int32), torch.zeros(0, 3), torch.zeros(0, 2), 1.0, 0, 10) > 0


class _Solver(object):
    """As much of a built solver as distill looks at before it touches a GPU."""
    graph, num_vertex, seed, num_worker, num_local_worker = object(), 5, 0, 1, 1

    def _no_session(self, what):
        pass


@pytest.mark.parametrize("bad", [dict(lr=-0.1), dict(lr=float("nan")), dict(num_epoch=-1), dict(batch_size=-2)])
def test_distill_refuses(bad):
    teacher = scorer.LinkScorer.__new__(scorer.LinkScorer)
    teacher.graph = _Solver.graph
    with pytest.raises(ValueError, match="must not be negative"):
        scorer.distill(_Solver(), teacher, k=2, **bad)
