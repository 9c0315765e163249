"""-m gpu: GraphApplication.neighbor_prediction with a scorer that the program keeps, and what its answers in 8 bits are worth."""
import logging

import numpy as np
import pytest
import torch

import graphvite_amd as gv
from graphvite_amd import scorer as scorer_module
from graphvite_amd import synthetic

pytestmark = pytest.mark.gpu


def application(edges):
    app = gv.application.GraphApplication(dim=32, cpu_per_gpu=3)
    app.load(edge_list=edges)
    app.build(batch_size=1000, episode_size=10)
    return app


@pytest.fixture(scope="module")
def app():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    gv.init_logging(logging.ERROR)
    app = application(synthetic.community_edges(1500, 9000, num_community=10, seed=3))
    app.train(model="LINE", num_epoch=200, augmentation_step=2, log_frequency=1 << 30)
    return app


def test_a_scorer_that_is_kept_answers_every_call(app, monkeypatch):
    names = [app.graph.id2name[i] for i in (4, 9, 0)]
    want = app.neighbor_prediction(H=names, k=7)
    kept = app.solver.scorer()
    made = []
    monkeypatch.setattr(scorer_module.LinkScorer, "__init__", lambda self, *args: made.append(args))
    for _ in range(3):
        assert app.neighbor_prediction(H=names, k=7, scorer=kept) == want
    assert app.evaluate("neighbor prediction", H=names, k=7, scorer=kept) == want
    assert not made


def test_a_scorer_of_another_graph_is_refused(app):
    other = application(synthetic.community_edges(300, 2000, num_community=10, seed=4))
    with pytest.raises(ValueError, match="another graph"):
        app.neighbor_prediction(H=[app.graph.id2name[0]], scorer=other.solver.scorer())


@pytest.mark.parametrize("k", [1, 10, 64])
def test_the_best_by_8_bits_against_the_best(app, k):
    """Every answer's exact score reaches the exact k-th best but for what 8 bits may hide: a score is off by at most b = sum (|v| / 16 + v0) |c| + ... of
    its own two rows (each value by 2^-4 of itself, or 2^-10 of its block's scale, which is below 2^-7 of the block's largest); an
    answer that stands in the place of a better node lies below it by no more than the two nodes' b together."""
    s = app.solver
    v, c = s.vertex_embeddings.astype(np.float64), s.context_embeddings.astype(np.float64)
    exact = v @ c.T
    off = lambda x: np.abs(x) / 16 + np.abs(x).max(1, keepdims=True) / 2 ** 17  # noqa: E731
    bound = off(v) @ np.abs(c).T + np.abs(v) @ off(c).T + off(v) @ off(c).T + 2e-5 * (np.abs(v) @ np.abs(c).T)
    heads = np.arange(len(v))
    found = s.scorer().top(heads, k)[0]
    order = np.argsort(-exact, 1, kind="stable")[:, :k]
    kth = np.take_along_axis(exact, order, 1)[:, -1]
    hidden = np.take_along_axis(bound, order, 1).max(1)
    got = np.take_along_axis(exact, found, 1)
    assert (got >= kth[:, None] - hidden[:, None] - np.take_along_axis(bound, found, 1)).all()
    share = np.mean([len(set(a) & set(b)) for a, b in zip(found.tolist(), order.tolist())]) / k
    print("of the exact best %d, %.3f found" % (k, share))
