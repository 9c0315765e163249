"""-m gpu: GraphSolver.scorer / distill and GraphApplication.neighbor_prediction: the whole-row operators behind the solver."""
import logging

import numpy as np
import pytest
import torch

import graphvite_amd as gv
import rows_oracle
from graphvite_amd import synthetic

pytestmark = pytest.mark.gpu


def solver_with(dim, edges, seed, scale=0.4):
    gv.init_logging(logging.ERROR)
    g = gv.graph.Graph()
    g.load(edges)
    s = gv.solver.GraphSolver(dim, num_sampler_per_worker=2, seed=seed)
    s.build(g, batch_size=1000, episode_size=10)
    rng = np.random.default_rng(seed)
    s.vertex_embeddings[:] = scale * rng.standard_normal((g.num_vertex, dim))
    s.context_embeddings[:] = scale * rng.standard_normal((g.num_vertex, dim))
    return g, s


@pytest.fixture(scope="module")
def edges():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return synthetic.community_edges(1500, 9000, num_community=10, seed=3)


@pytest.mark.parametrize("dim", [32, 96, 512])
def test_scorer_answers_from_the_8_bit_table(edges, dim):
    g, s = solver_with(dim, edges, 5)
    scorer = s.scorer()
    heads = np.array([3, 0, g.num_vertex - 1, 3, 77])
    q, t = rows_oracle.quantise(s.vertex_embeddings[heads])[0], rows_oracle.quantise(s.context_embeddings)[0]
    exact, magnitude = q @ t.T, np.abs(q) @ np.abs(t).T
    logits = scorer.logits(heads)
    assert (np.abs(logits.cpu().double().numpy() - exact) <= 2 * dim * 2.0 ** -24 * magnitude + 2.0 ** -24 * np.abs(exact)).all()
    index, values, stats = scorer.top(heads, k=20, temperature=2.0)
    want_values, want_index, want_stats = rows_oracle.top(logits.cpu().double().numpy(), 20, 2.0)
    np.testing.assert_array_equal(index, want_index)
    np.testing.assert_array_equal(values, want_values.astype(np.float32))
    np.testing.assert_allclose(stats, want_stats, rtol=0, atol=1e-5)
    # near the logits of predict: each side is off by at most 2^-4 of every value (2^-10 of the block's scale, below 2^-9 of its largest, for the least)
    pairs = np.stack([np.repeat(heads, 20), index.ravel()], 1)
    v, c = np.abs(s.vertex_embeddings[pairs[:, 0]]).astype(np.float64), np.abs(s.context_embeddings[pairs[:, 1]]).astype(np.float64)
    v_off, c_off = v / 16 + v.max(1, keepdims=True) / 2 ** 17, c / 16 + c.max(1, keepdims=True) / 2 ** 17
    bound = (v_off * c + v * c_off + v_off * c_off).sum(1)
    assert (np.abs(s.predict(pairs) - values.ravel()) <= bound * 1.001).all()
    # what the scorer holds is of its making
    s.context_embeddings[:] = 0
    assert torch.equal(scorer.logits(heads), logits)
    assert scorer.logits(np.zeros(0, np.int64)).shape == (0, g.num_vertex)
    assert scorer.top(np.zeros(0, np.int64), 3)[0].shape == (0, 3)


def test_scorer_made_on_one_stream_answers_on_another(edges):
    g, s = solver_with(512, edges, 8)
    heads = np.arange(40)
    want = s.scorer().top(heads, 30)
    made, asked = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(made):
            scorer = s.scorer()
        with torch.cuda.stream(asked):
            got = scorer.top(heads, 30)
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a, b)


def test_scorer_refuses(edges):
    g, s = solver_with(32, edges, 1)
    scorer = s.scorer()
    for bad in ([-1], [g.num_vertex], [[1]], [0.5]):
        with pytest.raises(ValueError):
            scorer.logits(np.array(bad))
    for k in (0, 257, g.num_vertex + 1):
        with pytest.raises(ValueError, match="k must be"):
            scorer.top(np.array([1]), k=k)
    with pytest.raises(ValueError, match="k must be"):
        s.distill(scorer, k=257)
    with pytest.raises(TypeError, match="LinkScorer"):
        s.distill(s)
    with pytest.raises(ValueError, match="twice"):
        s.distill(scorer, heads=np.array([1, 2, 1]))
    other = solver_with(32, edges[:500], 2)[1]
    with pytest.raises(ValueError, match="nodes"):
        other.distill(scorer)
    session = s.session(model="LINE", num_epoch=1, augmentation_step=1)
    with pytest.raises(ValueError, match="session is open"):
        s.scorer()
    with pytest.raises(ValueError, match="session is open"):
        s.distill(scorer)
    session.close()
    s.scorer()
    with pytest.raises(RuntimeError, match="built"):
        gv.solver.GraphSolver(32).scorer()


def test_one_update_of_distill_is_the_formula_s(edges):
    """One batch of all nodes: both tables move by -lr times the gradient that the 64-bit oracle gives for the lists the teacher gave.
    Tolerance: logits in float32 sums of 32 products (32 * 2^-24 of their magnitude, below 1e-4 absolute for logits below 30) move
    probabilities by 1e-4 relative, the kernel adds 2e-5: 2e-4 of the sum of the gradient's terms."""
    g, teacher = solver_with(128, edges, 7)
    s = solver_with(32, edges, 8)[1]
    n, lr = g.num_vertex, 0.05
    scorer = teacher.scorer()
    index, values, stats = scorer.top(np.arange(n), k=16, temperature=1.5)
    v, c = s.vertex_embeddings.astype(np.float64), s.context_embeddings.astype(np.float64)
    loss, _, grad, terms, _ = rows_oracle.distill(v @ c.T, index, values, 1.5, stats)
    losses = s.distill(scorer, num_epoch=1, batch_size=n, k=16, temperature=1.5, lr=lr)
    assert abs(losses[0] - loss.mean()) <= 1e-4 * (1 + np.abs(loss).mean())
    for got, before, change, scale in ((s.vertex_embeddings, v, grad @ c, terms @ np.abs(c)), (s.context_embeddings, c, grad.T @ v, terms.T @ np.abs(v))):
        assert (np.abs(got - (before - lr * change)) <= 2e-4 * lr * scale + 2.0 ** -23 * np.abs(before)).all()


def test_distill_runs_in_batches_and_over_some_nodes(edges):
    g, teacher = solver_with(64, edges, 7)
    s = solver_with(32, edges, 8)[1]
    untouched = s.vertex_embeddings[1000:].copy()
    losses = s.distill(teacher.scorer(), heads=np.arange(1000), num_epoch=3, batch_size=128, k=8, lr=0.02)
    assert len(losses) == 3 and np.isfinite(losses).all()
    assert (s.vertex_embeddings[1000:] == untouched).all() and np.isfinite(s.context_embeddings).all()
    again = solver_with(32, edges, 8)[1]
    assert again.distill(teacher.scorer(), heads=np.arange(1000), num_epoch=0) == []
    pairs = np.array([[1, 2], [5, 7]])
    np.testing.assert_allclose(s.predict(pairs), (s.vertex_embeddings[pairs[:, 0]] * s.context_embeddings[pairs[:, 1]]).sum(1), rtol=1e-4, atol=1e-5)


def test_neighbor_prediction(edges, tmp_path):
    gv.init_logging(logging.ERROR)
    app = gv.application.GraphApplication(dim=32, cpu_per_gpu=3)
    app.load(edge_list=edges)
    app.build(batch_size=1000, episode_size=10)
    rng = np.random.default_rng(0)
    app.solver.vertex_embeddings[:] = rng.standard_normal(app.solver.vertex_embeddings.shape)
    app.solver.context_embeddings[:] = rng.standard_normal(app.solver.vertex_embeddings.shape)
    names = [app.graph.id2name[i] for i in (4, 9, 0)]
    found = app.evaluate("neighbor prediction", H=names, k=7)
    index, scores, _ = app.solver.scorer().top(np.array([4, 9, 0]), 7)
    assert [[name for name, _ in row] for row in found] == [[app.graph.id2name[int(t)] for t in row] for row in index]
    assert [[score for _, score in row] for row in found] == scores.tolist()
    (tmp_path / "nodes.txt").write_text("# nodes\n" + "\n".join(names) + "\n")
    assert app.neighbor_prediction(file_name=str(tmp_path / "nodes.txt"), k=7) == found
    with pytest.raises(ValueError, match="Can't find"):
        app.neighbor_prediction(H=["nobody"])
    with pytest.raises(ValueError):
        app.neighbor_prediction()
