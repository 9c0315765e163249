"""-m gpu: GraphSolver.distill as it is called by default: it teaches a student that was only built, and what it is given never gets worse
than it was found."""
import logging

import numpy as np
import pytest
import torch

import graphvite_amd as gv
from graphvite_amd import synthetic

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def teacher():
    """A trained solver of 128 dimensions over 1500 nodes in ten communities."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    gv.init_logging(logging.ERROR)
    g = gv.graph.Graph()
    g.load(synthetic.community_edges(1500, 9000, num_community=10, seed=3))
    s = gv.solver.GraphSolver(128, num_sampler_per_worker=4, seed=1)
    s.build(g, batch_size=1000, episode_size=10)
    s.train(model="LINE", num_epoch=300, augmentation_step=2, log_frequency=1 << 30)
    return s


def student_of(teacher, dim=32, seed=2):
    s = gv.solver.GraphSolver(dim, num_sampler_per_worker=2, seed=seed)
    s.build(teacher.graph, batch_size=1000, episode_size=10)
    return s


def shared_best(a, b, k=10):
    heads = np.arange(a.num_vertex)
    one, two = a.scorer().top(heads, k)[0], b.scorer().top(heads, k)[0]
    return float(np.mean([len(set(x) & set(y)) for x, y in zip(one.tolist(), two.tolist())])) / k


def test_a_student_that_was_only_built_learns(teacher):
    s = student_of(teacher)
    assert not s.vertex_embeddings.any() and not s.context_embeddings.any()
    assert s.distill(teacher.scorer(), num_epoch=0) == [] and not s.vertex_embeddings.any()
    losses = s.distill(teacher.scorer())
    print("losses", losses)
    assert len(losses) == 10 and all(b < a for a, b in zip(losses, losses[1:]))
    assert s.vertex_embeddings.any(1).all() and s.context_embeddings.any(1).all()
    assert np.isfinite(s.vertex_embeddings).all() and np.isfinite(s.context_embeddings).all()
    # ten of 1500 by chance: 0.007 shared
    first = shared_best(teacher, s)
    print("shared best after 10 epochs", first)
    assert first > 0.05
    more = s.distill(teacher.scorer(), num_epoch=20)  # goes on from its tables
    print("losses", more, "shared best after 30", shared_best(teacher, s))
    assert more[0] < losses[-1] and more[-1] < more[0] and shared_best(teacher, s) > first


def test_a_trained_student_goes_on_from_its_tables(teacher):
    s = student_of(teacher, 64, 3)
    s.train(model="LINE", num_epoch=20, augmentation_step=1, log_frequency=1 << 30)
    before = s.vertex_embeddings.copy()
    losses = s.distill(teacher.scorer(), num_epoch=3, lr=1e-6)
    assert len(losses) == 3 and 0 < np.abs(s.vertex_embeddings - before).max() < 1e-2


@pytest.mark.parametrize("k", [10, 64])
def test_a_trained_student_learns_at_the_default_rate(teacher, k):
    s = student_of(teacher, 64, 3)
    s.train(model="LINE", num_epoch=200, augmentation_step=2, log_frequency=1 << 30)
    losses = s.distill(teacher.scorer(), k=k)
    print("losses", losses)
    assert np.isfinite(losses).all() and losses[-1] < losses[0]


def test_the_same_seed_the_same_student(teacher):
    scorer = teacher.scorer()
    a, b = student_of(teacher), student_of(teacher)
    assert a.distill(scorer, num_epoch=2, heads=np.arange(700)) == b.distill(scorer, num_epoch=2, heads=np.arange(700))
    assert (a.vertex_embeddings == b.vertex_embeddings).all() and (a.context_embeddings == b.context_embeddings).all()


@pytest.mark.parametrize("num_epoch", [1, 5])
def test_a_rate_that_diverges_leaves_the_embeddings(teacher, num_epoch):
    s = student_of(teacher)
    s.distill(teacher.scorer(), num_epoch=1)
    before = s.vertex_embeddings.copy(), s.context_embeddings.copy()
    with pytest.raises(RuntimeError, match="diverged"):
        s.distill(teacher.scorer(), num_epoch=num_epoch, lr=1e20)
    assert (s.vertex_embeddings == before[0]).all() and (s.context_embeddings == before[1]).all()
