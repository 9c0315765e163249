"""Answers of a trained model for whole rows of candidates, and learning from them.

`GraphSolver.predict` gives the logits <vertex[h], context[t]> of given pairs.  A `LinkScorer` — made by `GraphSolver.scorer()` — gives a
node's logits against EVERY node, or the best of them, from a context table held on the GPU in 8 bits
(`HipKernels.quantize_blocks`): a quarter of the memory, and of the time where reading the table is what an answer costs.
`distill` (as `GraphSolver.distill`) trains a solver's embeddings — of a smaller dimension, say — to answer as a scorer does.
"""
import math

import numpy as np
import torch

from .kernels import HipKernels

_CHUNK = 1 << 28  # logits of a batch: a float32 GiB


def node_rows(heads, num_vertex, device):
    """Node ids as an index tensor on `device`, checked on the host."""
    heads = np.asarray(heads)
    if heads.ndim != 1 or heads.dtype.kind not in "iu":
        raise ValueError("Expect a one-dimensional array of node ids, but %s of shape %s is found" % (heads.dtype, heads.shape))
    if len(heads) and (int(heads.min()) < 0 or int(heads.max()) >= num_vertex):
        raise ValueError("node index out of range")
    return torch.from_numpy(heads.astype(np.int64)).to(device)


class LinkScorer(object):
    """
    LinkScorer(solver, device=None)
    The embeddings of a built solver as they are now, ready to answer: vertex rows in float32, the context table in 8 bits with a
    power-of-two scale per 128 columns, both on one GPU.  Later changes of the solver's embeddings do not show; make another.

    Parameters:
        solver (GraphSolver): built (and trained, or loaded) solver, no session open
        device (int, optional): GPU id, default is the solver's first

    Logits are off from `GraphSolver.predict` by the rounding to 8 bits on both sides: up to 2^-4 of each value.
    """

    def __init__(self, solver, device=None):
        if solver.graph is None:
            raise RuntimeError("The model must be built on a graph first")
        solver._no_session("scorer")
        if not torch.cuda.is_available():
            raise RuntimeError("a scorer answers on a GPU; graphvite_amd has no CPU path for it")
        self.device = torch.device("cuda", solver.device if device is None else int(device))
        self.graph, self.dim, self.num_vertex = solver.graph, solver.dim, solver.num_vertex
        self.kernels = HipKernels()
        self.vertex = torch.from_numpy(solver.vertex_embeddings).to(self.device)
        self.table = self.kernels.quantize_blocks(torch.from_numpy(solver.context_embeddings).to(self.device))
        self._made_on = torch.cuda.current_stream(self.device)
        self._made_on.synchronize()  # whichever stream asks first finds the table whole

    def _ask(self):
        """The embeddings' memory belongs to the stream they were made on: where another one asks, it is not handed on before that one has
        passed the question, also if the scorer is dropped meanwhile."""
        stream = torch.cuda.current_stream(self.device)
        if stream != self._made_on:
            for t in (self.vertex, self.table.values, self.table.exponents):
                t.record_stream(stream)

    def logits(self, heads, dtype=torch.float32):
        """
        logits(heads, dtype=torch.float32)
        Logits of nodes against all nodes.

        Parameters:
            heads (ndarray): node ids
            dtype (torch.dtype): float32, bfloat16 or float16

        Returns:
            Tensor: [len(heads), num_vertex] on the scorer's GPU, ordered on its current stream
        """
        with torch.cuda.device(self.device):
            rows = node_rows(heads, self.num_vertex, self.device)
            self._ask()
            out = torch.empty((len(rows), self.num_vertex), dtype=dtype, device=self.device)
            return self.kernels.block_logits(self.vertex[rows], self.table, out)

    def top_on_device(self, rows, k, temperature=1.0):
        """(logits float32 [n, k], index int32 [n, k], stats float32 [n, 2]) of an index tensor on the scorer's GPU; HipKernels.top_logits."""
        n, device = len(rows), self.device
        self._ask()
        values = torch.empty((n, k), dtype=torch.float32, device=device)
        index = torch.empty((n, k), dtype=torch.int32, device=device)
        stats = torch.empty((n, 2), dtype=torch.float32, device=device)
        batch = max(1, min(n, _CHUNK // self.num_vertex))
        logits = torch.empty((batch, self.num_vertex), dtype=torch.float32, device=device)
        for first in range(0, n, batch):
            part = rows[first:first + batch]
            z = logits[:len(part)]
            self.kernels.block_logits(self.vertex[part], self.table, z)
            self.kernels.top_logits(z, values[first:first + batch], index[first:first + batch], stats[first:first + batch], temperature)
        return values, index, stats

    def top(self, heads, k=10, temperature=1.0):
        """
        top(heads, k=10, temperature=1.0)
        The k nodes with the largest logits for each node, the largest first, of equal ones the lowest id.

        Parameters:
            heads (ndarray): node ids
            k (int): up to 256, and no more than there are nodes
            temperature (float): of the statistics

        Returns:
            (ndarray, ndarray, ndarray): ids int64 [n, k]; logits float32 [n, k]; float32 [n, 2] = max m and
            log sum exp((logit - m) / temperature) of each whole row
        """
        if not 1 <= int(k) <= min(256, self.num_vertex):
            raise ValueError("k must be 1 to %d, not %s" % (min(256, self.num_vertex), k))
        with torch.cuda.device(self.device):
            values, index, stats = self.top_on_device(node_rows(heads, self.num_vertex, self.device), int(k), float(temperature))
            return index.cpu().numpy().astype(np.int64), values.cpu().numpy(), stats.cpu().numpy()


def start_tables(num_vertex, dim, seed):
    """Where a solver that was only built begins: both tables uniform, the logits' standard deviation 1/4.  (Training's own start, a context
    of zeros, has next to no gradient here: 1500 nodes, 10 epochs at the default rate: 1.170 -> 1.146, against 1.185 -> 0.013 from here.)"""
    generator = torch.Generator()
    generator.manual_seed(seed)
    bound = 0.5 * dim ** -0.25 * 3 ** 0.5
    return tuple((2 * torch.rand((num_vertex, dim), generator=generator) - 1) * bound for _ in range(2))


def default_rate(index, values, stats, temperature, batch, num_vertex):
    """The learning rate of distill by default: T^2 / (2 Q max(1, H)) of a teacher's lists (top_logits).

    A row's gradient by its logits is (Q p - q) / T: its size goes by the mean share Q of the teacher's probability that a list holds.  The
    steps of a context row add up over a batch: H = batch times the largest share of all lists' probability that one candidate has is
    how many heads' worth of it the most listed one is given at once.  With two trained teachers (1500 nodes in communities, 6000 with hubs;
    k 10 and 64, T 1/2 to 2, student dimensions 32 and 128) twice this rate diverged within 10 epochs in one of ten settings, four times in five;
    this one in none, nor in 60 epochs with k 8 to 256."""
    q = torch.exp((values - stats[:, :1]) / temperature - stats[:, 1:])
    # the sums in whole numbers, 2^-30 each: the same whatever order they are added in
    shares = torch.zeros(num_vertex, dtype=torch.int64, device=q.device)
    shares.index_add_(0, index.reshape(-1).long(), (q.double() * 2 ** 30).round().long().reshape(-1))
    total = max(float(shares.sum()), 1.0)
    hub = batch * float(shares.max()) / total
    return temperature ** 2 / (2 * total / 2 ** 30 / max(len(q), 1) * max(1.0, hub))


def distill(solver, teacher, heads=None, num_epoch=10, batch_size=0, k=64, temperature=1.0, lr=0.0, seed=None):
    """GraphSolver.distill."""
    if solver.graph is None:
        raise RuntimeError("The model must be built on a graph first")
    solver._no_session("distill")
    if not isinstance(teacher, LinkScorer):
        raise TypeError("teacher must be a LinkScorer (GraphSolver.scorer() of the solver to learn from)")
    if solver.num_local_worker < solver.num_worker:  # every rank's tables are alike after train(), and would not be after this
        raise ValueError("distill trains the tables of one process, and this solver's are shared by a job of %d; use a solver made outside of the job "
                         "(its embeddings may be set to these)" % solver.num_worker)
    if teacher.graph is not solver.graph and list(teacher.graph.id2name) != list(solver.graph.id2name):
        raise ValueError("the teacher's nodes are not this solver's nodes")
    n = solver.num_vertex
    if not 1 <= int(k) <= min(256, n):
        raise ValueError("k must be 1 to %d, not %s" % (min(256, n), k))
    if int(num_epoch) < 0 or int(batch_size) < 0 or not lr >= 0:
        raise ValueError("num_epoch, batch_size and lr must not be negative")
    device, kernels = teacher.device, teacher.kernels
    batch = int(batch_size) or max(1, min(256, _CHUNK // n))
    seed = solver.seed if seed is None else int(seed)
    generator = torch.Generator()
    generator.manual_seed(seed)
    vertex, context = torch.from_numpy(solver.vertex_embeddings), torch.from_numpy(solver.context_embeddings)
    if int(num_epoch) and not (vertex.any() or context.any()):  # built and never trained: at zero every gradient is zero, too
        vertex, context = start_tables(n, solver.dim, seed)
    with torch.cuda.device(device):
        rows = node_rows(np.arange(n) if heads is None else heads, n, device)
        if len(torch.unique(rows)) != len(rows):
            raise ValueError("a node is named twice")  # its row would be written twice in a batch
        values, index, teacher_stats = teacher.top_on_device(rows, int(k), float(temperature))
        rate = float(lr) or default_rate(index, values, teacher_stats, float(temperature), min(batch, len(rows)), n)
        vertex, context = vertex.to(device), context.to(device)
        losses = []
        for epoch in range(int(num_epoch)):
            total = torch.zeros((), dtype=torch.float64, device=device)
            for part in torch.randperm(len(rows), generator=generator).to(device).split(batch):
                ids = rows[part]
                v = vertex[ids]
                logits = v @ context.t()
                loss = torch.empty(len(ids), device=device)
                stats = torch.empty((len(ids), 2), device=device)
                kernels.distill(logits, index[part], values[part], loss, stats, teacher_stats[part], float(temperature), grad=logits)
                change = logits @ context  # before the context moves: both sides from what the batch began with
                context.addmm_(logits.t(), v, alpha=-rate)
                vertex[ids] = v - rate * change
                total += loss.sum(dtype=torch.float64)
            losses.append(float(total) / max(len(rows), 1))
            last = epoch + 1 == int(num_epoch)  # what its last steps made of the tables shows in no loss
            if not math.isfinite(losses[-1]) or last and not (torch.isfinite(vertex).all() and torch.isfinite(context).all()):
                raise RuntimeError("distill diverged in epoch %d at a learning rate of %g; the embeddings are as they were" % (epoch, rate))
        solver.vertex_embeddings[:] = vertex.cpu().numpy()
        solver.context_embeddings[:] = context.cpu().numpy()
    return losses
