"""synthetic.py draws many numbers at a time and over threads; what it makes is what the plain loops make, number for number."""
import numpy as np
import pytest

from graphvite_amd import graph, synthetic


def plain_split(edges, portions, seed):
    """One draw after the other, as the reference's Dataset.link_prediction_split does."""
    rs = np.random.RandomState(seed)
    cum = np.cumsum(portions, dtype=np.float32) / np.sum(portions)
    which = np.searchsorted(cum, rs.rand(len(edges)))
    nodes = np.unique(edges)
    keys = set((edges[:, 0].astype(np.int64) << 32 | edges[:, 1].astype(np.int64)).tolist())
    splits = []
    for i in range(1, len(portions)):
        true = edges[which == i]
        H, T = [], []
        while len(H) < len(true):
            u = int(nodes[int(rs.rand() * len(nodes))])
            v = int(nodes[int(rs.rand() * len(nodes))])
            if u != v and (u << 32 | v) not in keys and (v << 32 | u) not in keys:
                H.append(u)
                T.append(v)
        splits.append((np.concatenate([true[:, 0], np.asarray(H, edges.dtype)]), np.concatenate([true[:, 1], np.asarray(T, edges.dtype)]),
                       np.concatenate([np.ones(len(true), np.int64), np.zeros(len(H), np.int64)])))
    return edges[which == 0], splits


@pytest.mark.parametrize("n,e,portions,dtype", [(20, 150, (1, 1, 1), np.uint32), (300, 3000, (100, 3, 3), np.uint32), (40, 500, (1, 2), np.int64),
                                                (5000, 200000, (10, 1, 2, 1), np.uint32), (50, 3, (100, 1, 1), np.uint32)])
def test_link_prediction_split(n, e, portions, dtype):
    edges = synthetic.power_law_edges(n, e, seed=n).astype(dtype)
    for seed in (1024, 5):
        (train, splits), (want_train, want_splits) = synthetic.link_prediction_split(edges, portions, seed), plain_split(edges, portions, seed)
        assert (train == want_train).all() and len(splits) == len(want_splits)
        for got, want in zip(splits, want_splits):
            for a, b in zip(got, want):
                assert a.dtype == b.dtype and a.shape == b.shape and (a == b).all()


@pytest.mark.parametrize("n,e", [(100, 1000), (70000, 300000)])
def test_power_law_edges(n, e):
    """The second one is large enough to be dealt over threads."""
    rng = np.random.default_rng(9)
    w = np.arange(1, n + 1, dtype=np.float64) ** (-1.0 / 1.3)
    cdf = np.cumsum(w)
    cdf /= cdf[-1]
    label = rng.permutation(n).astype(np.uint32)
    want = np.zeros((0, 2), np.uint32)
    while len(want) < e:
        m = e - len(want)
        u, v = (np.searchsorted(cdf, rng.random(m), side="right") for _ in range(2))
        keep = u != v
        want = np.concatenate([want, np.stack([label[np.minimum(x[keep], n - 1)] for x in (u, v)], 1)])
    assert (synthetic.power_law_edges(n, e, seed=9) == want).all()


@pytest.mark.parametrize("side", ["left", "right"])
def test_search_over_threads(side):
    rng = np.random.default_rng(1)
    ascending = np.sort(rng.integers(0, 1000, 5000))
    for size in (0, 1, 65536, 300001):
        values = rng.integers(-5, 1005, size)
        assert (synthetic._search(ascending, values, side) == np.searchsorted(ascending, values, side=side)).all()


def test_names_in_their_order():
    """Names longer than any buffer among them."""
    g = graph.Graph()
    names = ["a", "b" * 63, "c" * 64, "d" * 65, "e" * 1000, "é", "f"]
    g.load(edge_list=list(zip(names, names[1:])))
    assert list(g.id2name) == [g.id2name[i] for i in range(g.num_vertex)] and sorted(g.id2name) == sorted(names)
    assert list(g.name2id) == list(g.id2name) and g.id2name.index("f") == g.name2id["f"]
