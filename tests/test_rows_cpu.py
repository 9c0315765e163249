"""Whole rows of candidates (8-bit block tables, their logits, top logits, distillation) without a GPU: what the C entry points and
the Python face refuse before anything is launched, the workspace sizes, and the 64-bit oracle of the GPU tests against torch."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import rows_oracle
from graphvite_amd import _lib, scorer
from graphvite_amd.kernels import BlockTable, HipKernels

P = C.c_void_p(1 << 20)  # never followed: every call below is refused (or has nothing to do) before a launch


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def refused(lib, rc, text, code=-1):
    message = lib.gvk_last_error().decode()
    assert rc == code and text in message, (rc, message)


def test_block_entry_points_refuse(lib):
    quantize = lambda dtype=0, rows=P, n=4, dim=40, stride=40, values=P, vstride=48, exponents=P: lib.gvk_block_quantize(  # noqa: E731
        None, dtype, rows, n, dim, stride, values, vstride, exponents)
    refused(lib, quantize(dtype=3), "type")
    refused(lib, quantize(n=-1), "rows")
    refused(lib, quantize(n=1 << 31), "rows")
    refused(lib, quantize(dim=0), "dim", -2)
    refused(lib, quantize(dim=4097, stride=4097, vstride=4112), "dim", -2)
    refused(lib, quantize(stride=39), "stride")
    refused(lib, quantize(rows=None), "null")
    refused(lib, quantize(values=None), "null")
    refused(lib, quantize(exponents=None), "null")
    refused(lib, quantize(vstride=32), "stride")
    refused(lib, quantize(vstride=56), "multiples of 16")
    refused(lib, quantize(values=C.c_void_p((1 << 20) + 8)), "multiples of 16")
    assert quantize(n=0, rows=None, values=None) == 0
    dequantize = lambda dtype=0, n=4, dim=40, stride=40, vstride=48, rows=P: lib.gvk_block_dequantize(  # noqa: E731
        None, P, vstride, P, n, dim, dtype, rows, stride)
    refused(lib, dequantize(dtype=-1), "type")
    refused(lib, dequantize(stride=3), "stride")
    refused(lib, dequantize(rows=None), "null")
    refused(lib, dequantize(vstride=40), "stride")
    assert dequantize(n=0) == 0

    def logits(qtype=0, query=P, m=2, qstride=40, values=P, vstride=48, exponents=P, n=9, dim=40, ztype=0, z=P, zstride=9, space=None, nbytes=0):
        return lib.gvk_block_logits(None, qtype, query, m, qstride, values, vstride, exponents, n, dim, ztype, z, zstride, space, nbytes)
    refused(lib, logits(qtype=7), "type")
    refused(lib, logits(ztype=7), "type")
    refused(lib, logits(dim=0), "dim", -2)
    refused(lib, logits(m=(1 << 20) + 1, space=P, nbytes=1 << 40), "queries")
    refused(lib, logits(m=-1), "rows")
    refused(lib, logits(n=-1), "rows")
    refused(lib, logits(qstride=39), "stride")
    refused(lib, logits(zstride=8), "stride")
    refused(lib, logits(query=None), "null")
    refused(lib, logits(z=None), "null")
    refused(lib, logits(values=None), "null")
    many = dict(m=17, dim=200, qstride=200, vstride=208)
    refused(lib, logits(**many), "workspace")
    refused(lib, logits(space=P, nbytes=16383, **many), "workspace of 16384")
    refused(lib, logits(space=C.c_void_p((1 << 20) + 4), nbytes=16384, **many), "workspace")
    assert logits(m=0) == 0 and logits(n=0, zstride=0) == 0
    assert lib.gvk_block_logits_workspace(16, 512) == 0 and lib.gvk_block_logits_workspace(16, 513) == 5 * 4096
    assert lib.gvk_block_logits_workspace(1000, 96) == 63 * 4096


def test_top_logits_refuses(lib):
    def top(dtype=0, z=P, m=2, n=9, stride=9, k=3, temperature=1.0, values=P, index=P, space=None, nbytes=0):
        return lib.gvk_top_logits(None, dtype, z, m, n, stride, k, temperature, values, index, None, space, nbytes)
    refused(lib, top(dtype=9), "type")
    refused(lib, top(m=-1), "rows")
    refused(lib, top(n=1 << 31, stride=1 << 31), "rows")
    refused(lib, top(stride=8), "stride")
    refused(lib, top(z=None), "null")
    refused(lib, top(z=C.c_void_p((1 << 20) + 2)), "aligned")
    refused(lib, top(k=0), "top 0")
    refused(lib, top(k=10), "top 10 of 9")
    refused(lib, top(n=1000, stride=1000, k=257), "top 257")
    refused(lib, top(values=None), "null")
    refused(lib, top(index=None), "null")
    for bad in (0.0, -1.0, math.inf, math.nan, 1e-42):
        refused(lib, top(temperature=bad), "temperature")
    refused(lib, top(n=99991, stride=99991), "workspace")
    assert top(m=0) == 0
    need = lib.gvk_top_logits_workspace(1, 1024, 1000000, 64)
    assert need == 1024 * 62 * (128 * 8 + 8 + 4)
    refused(lib, top(dtype=1, m=1024, n=1000000, stride=1000000, k=64, space=P, nbytes=need - 1), "workspace")
    assert lib.gvk_top_logits_workspace(0, 7, 10312, 10) == 0 and lib.gvk_top_logits_workspace(0, 7, 10312, 257) == 0


def test_distill_refuses(lib):
    def distill(dtype=0, z=P, m=2, n=9, stride=9, k=3, index=P, teacher=P, temperature=1.0, loss=P, stats=P, grad=None, gstride=0, space=None, nbytes=0):
        return lib.gvk_distill(None, dtype, z, m, n, stride, k, index, teacher, None, temperature, None, loss, stats, grad, gstride, space, nbytes)
    apart = C.c_void_p(1 << 30)
    refused(lib, distill(dtype=3), "type")
    refused(lib, distill(n=0, stride=0), "without logits")
    refused(lib, distill(m=-2), "rows")
    refused(lib, distill(stride=8), "stride")
    refused(lib, distill(k=0), "1 to 1024")
    refused(lib, distill(k=1025), "1 to 1024")
    for name in ("z", "index", "teacher", "loss", "stats"):
        refused(lib, distill(**{name: None}), "null")
    refused(lib, distill(temperature=0.0), "temperature")
    refused(lib, distill(grad=apart, gstride=8), "stride")
    refused(lib, distill(grad=C.c_void_p((1 << 30) + 1), gstride=9), "aligned")
    refused(lib, distill(grad=C.c_void_p((1 << 20) + 16), gstride=9), "overlaps")
    refused(lib, distill(grad=P, gstride=10), "overlaps")
    refused(lib, distill(n=20000, stride=20000), "workspace")
    refused(lib, distill(n=20000, stride=20000, space=P, nbytes=lib.gvk_distill_workspace(0, 2, 20000, 3) - 1), "workspace")
    assert distill(m=0) == 0
    assert lib.gvk_distill_workspace(0, 2, 16000, 3) == 0 and lib.gvk_distill_workspace(0, 2, 20000, 3) == 2 * (16 + 3 * 8 + 3 * 8)

    def grad(z=P, m=2, n=9, stride=9, k=3, index=P, teacher=P, temperature=1.0, stats=P, g=apart, gstride=9, space=P, nbytes=1 << 20):
        return lib.gvk_distill_grad(None, 0, z, m, n, stride, k, index, teacher, None, temperature, None, stats, g, gstride, space, nbytes)
    need = lib.gvk_distill_grad_workspace(0, 2, 9, 3)
    assert need == 2 * (16 + 8 + 3 * 8)
    refused(lib, grad(space=None), "workspace")
    refused(lib, grad(nbytes=need - 1), "workspace")
    for name in ("z", "index", "teacher", "stats", "g"):
        refused(lib, grad(**{name: None}), "null")
    refused(lib, grad(temperature=-1.0), "temperature")
    refused(lib, grad(gstride=8), "stride")
    refused(lib, grad(g=C.c_void_p((1 << 20) + 4)), "overlaps")
    assert grad(m=0) == 0


def test_python_face_refuses_tensors_off_the_gpu():
    K = HipKernels()
    z = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="GPU memory"):
        K.quantize_blocks(z)
    with pytest.raises(ValueError, match="GPU memory"):
        BlockTable(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 8)
    with pytest.raises(ValueError, match="dim"):
        BlockTable(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 0)
    with pytest.raises(ValueError, match="BlockTable"):
        K.block_logits(z, z, z)
    with pytest.raises(ValueError, match="GPU memory"):
        K.top_logits(z, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="two-dimensional"):
        K.top_logits(z[0], torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="dtype"):
        K.top_logits(z.double(), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="contiguous"):
        K.quantize_blocks(torch.zeros(8, 3).t())
    with pytest.raises(ValueError, match="GPU memory"):
        K.distill(z, torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2), torch.zeros(3), torch.zeros(3, 2))


def test_the_oracle_against_torch():
    """The oracle's quantiser against torch's own e4m3 conversion, its loss and gradient against torch's softmax and differences."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((7, 300)) * np.exp(rng.standard_normal((7, 300)))
    x[2, :128] = 0
    x[3, 5] = np.inf
    got, exponents = rows_oracle.quantise(x.astype(np.float32))
    for b in range(3):
        part = torch.from_numpy(x.astype(np.float32)[:, 128 * b:128 * b + 128])
        scale = torch.exp2(torch.from_numpy(exponents[:, b].astype(np.float32)) - 127)[:, None]
        want = ((part / scale).to(torch.float8_e4m3fn).float() * scale).numpy()
        ok = exponents[:, b] != 255
        assert (got[ok, 128 * b:128 * b + 128] == want[ok]).all()
        largest = np.abs(x[ok, 128 * b:128 * b + 128]).max(1)
        s = np.exp2(exponents[ok, b].astype(np.float64) - 127)
        assert (largest <= 448 * s).all() and ((largest > 224 * s) | (largest == 0)).all()
    assert exponents[3, 0] == 255 and np.isnan(got[3, :128]).all()

    z, t = rng.standard_normal((4, 30)) * 3, rng.standard_normal((4, 5))
    index = np.stack([rng.permutation(30)[:5] for _ in range(4)])
    loss, stats, grad, _, _ = rows_oracle.distill(z, index, t, 2.0, weight=[1.0, 2.0, 0.5, 0.0])
    zt = torch.from_numpy(z).requires_grad_()
    log_p, q = torch.log_softmax(zt / 2, 1), torch.softmax(torch.from_numpy(t) / 2, 1)
    want = (q * (q.log() - log_p.gather(1, torch.from_numpy(index)))).sum(1)
    (want * torch.tensor([1.0, 2.0, 0.5, 0.0])).sum().backward()
    assert np.allclose(loss, want.detach().numpy(), rtol=1e-12) and np.allclose(grad, zt.grad.numpy(), rtol=1e-10, atol=1e-14)
    for j in range(30):  # differences, h = 1e-5: h^2 / 6 of a third derivative below 1, plus 1e-16 / h
        up, down = z.copy(), z.copy()
        up[1, j] += 1e-5
        down[1, j] -= 1e-5
        slope = (rows_oracle.distill(up, index, t, 2.0)[0][1] - rows_oracle.distill(down, index, t, 2.0)[0][1]) / 2e-5
        assert abs(2.0 * slope - grad[1, j]) < 1e-9


class _Built(object):
    """What a scorer asks of a solver before it touches a GPU."""
    graph, device, num_vertex, seed = object(), 0, 5, 0

    def __init__(self, session=False):
        self.session = session

    def _no_session(self, what):
        if self.session:
            raise ValueError("%s: a training session is open" % what)


def test_scorer_and_distill_refuse_before_any_gpu():
    unbuilt = _Built()
    unbuilt.graph = None
    for call in (lambda s: scorer.LinkScorer(s), lambda s: scorer.distill(s, None)):
        with pytest.raises(RuntimeError, match="must be built"):
            call(unbuilt)
        with pytest.raises(ValueError, match="session is open"):
            call(_Built(session=True))
    with pytest.raises(TypeError, match="LinkScorer"):
        scorer.distill(_Built(), _Built())
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no CPU path"):
            scorer.LinkScorer(_Built())


@pytest.mark.parametrize("bad", [[[1]], [0.5], [-1], [5], "1"])
def test_node_rows_refuses(bad):
    with pytest.raises(ValueError):
        scorer.node_rows(bad, 5, "cpu")


def test_node_rows():
    assert scorer.node_rows(np.array([4, 0, 4], np.uint32), 5, "cpu").tolist() == [4, 0, 4]
    assert scorer.node_rows(np.zeros(0, np.int64), 5, "cpu").shape == (0,)
