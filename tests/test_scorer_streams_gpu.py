"""-m gpu: a LinkScorer made on one stream and asked on another, either of them late."""
import numpy as np
import pytest
import torch

from graphvite_amd import scorer as scorer_module
from graphvite_amd.kernels import HipKernels
from test_scorer_gpu import edges, solver_with  # noqa: F401  (edges: the fixture)

pytestmark = pytest.mark.gpu
LATE = 40000000  # cycles: some 20 ms


@pytest.fixture(scope="module")
def solver(edges):  # noqa: F811
    return solver_with(512, edges, 8)[1]


@pytest.mark.parametrize("ask", ["logits", "top"])
def test_a_table_that_is_late_is_waited_for(solver, monkeypatch, ask):
    """The table is quantised long after the other stream could have begun to ask."""
    heads = np.arange(40)
    want = solver.scorer().logits(heads)
    quantize = HipKernels.quantize_blocks

    def late(self, *args):
        torch.cuda._sleep(LATE)
        return quantize(self, *args)
    monkeypatch.setattr(HipKernels, "quantize_blocks", late)
    made, asked = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(made):
        scorer = solver.scorer()
    with torch.cuda.stream(asked):
        if ask == "logits":
            got = scorer.logits(heads)
            asked.synchronize()
            assert torch.equal(got, want)
        else:
            values = scorer.top(heads, 5)[1]
            np.testing.assert_array_equal(values, torch.topk(want, 5).values.cpu().numpy())


@pytest.mark.parametrize("ask", ["logits", "top_on_device"])
def test_a_scorer_dropped_while_it_answers(solver, monkeypatch, ask):
    """The other stream asks and is late, the scorer is dropped, and the stream it was made on takes memory of the same sizes and writes to it."""
    heads = np.arange(300)
    whole = solver.scorer()
    want = whole.logits(heads) if ask == "logits" else whole.top_on_device(torch.arange(300, device=whole.device), 9)[0]
    torch.cuda.synchronize()
    node_rows = scorer_module.node_rows

    def late(*args):
        rows = node_rows(*args)
        torch.cuda._sleep(LATE)
        return rows
    made, asked = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(made):
        scorer = solver.scorer()
        shapes = [(t.shape, t.dtype) for t in (scorer.vertex, scorer.table.values, scorer.table.exponents)]
    monkeypatch.setattr(scorer_module, "node_rows", late)
    with torch.cuda.stream(asked):
        if ask == "logits":
            got = scorer.logits(heads)
        else:
            got = scorer.top_on_device(late(heads, scorer.num_vertex, scorer.device), 9)[0]
    del scorer
    with torch.cuda.stream(made):
        taken = [torch.full(shape, 3, dtype=dtype, device="cuda:0") for shape, dtype in shapes for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(taken) == 9
