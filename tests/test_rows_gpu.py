"""-m gpu: whole rows of candidates (include/gvk.h: gvk_block_quantize / _dequantize / _logits, gvk_top_logits, gvk_distill,
gvk_distill_grad) against the 64-bit oracle of rows_oracle.py.

Tolerances, u = 2^-24:
  logits   products of two e4m3 numbers are floats; a sum of K of them in any order, each addition off by at most 2 u of the running sum of
           magnitudes, is off by 2 K u * sum |q x|; then one rounding to the output type
  stats    a term exp((z - m) / T): its exponent takes three roundings (3 u |x|), the exponential 4 u; a softmax's mean |x| is at most
           log n <= 16; a thread adds up to 64 terms, the joins 20 more: the logarithm of the sum is off by (48 + 4 + 84) u plus
           its own rounding, below 1e-5 in all
  loss     terms q (log q - log p), each factor off by less than 1e-5 relative (or absolutely in the logarithms): 2e-5 times
           sum q (|log q| + |log p| + 1)
  grad     w / T (Q p - q): p and q off by less than 2e-5 relative for |z - m| / T up to 80 (3 u 80 + the sum's 1e-5), then one rounding
           to the output type (half a step: eps / 2 relative, or half of the least step)."""
import numpy as np
import pytest
import torch

import rows_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LEAST = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -24}  # below it a type's steps are absolute (fp32 and bf16: flushed)


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def rounding(kind, exact):
    return torch.finfo(TYPES[kind]).eps / 2 * np.abs(exact) + LEAST[kind]


def strided(x, kind, lead=0, extra=0):
    """x [rows, n] on the device, its rows `extra` elements apart and the first one `lead` elements into the storage; the gaps hold 77."""
    rows, n = x.shape
    base = torch.full((lead + rows * (n + extra),), 77.0, dtype=TYPES[kind], device=DEV)
    view = base.as_strided((rows, n), (n + extra, 1), lead)
    view.copy_(torch.as_tensor(x, dtype=torch.float64).to(TYPES[kind]))
    return base, view


def gaps_intact(base, view):
    mask = torch.ones_like(base, dtype=torch.bool)
    mask.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(False)
    return bool((base[mask] == 77.0).all())


def same_place(view):
    """A copy whose rows begin where those of `view` do within 16 bytes."""
    base = torch.empty(view.storage_offset() + view.shape[0] * view.stride(0), dtype=view.dtype, device=DEV)
    copy = base.as_strided(view.shape, view.stride(), view.storage_offset())
    copy.copy_(view)
    return copy


def numbers(view):
    return view.detach().cpu().double().numpy()


def table_numbers(hip, table):
    x = torch.empty(table.rows, table.dim, device=DEV)
    return numbers(hip.dequantize_blocks(table, x))


# ---- 8-bit tables ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,dim,lead,extra", [(1, 1, 0, 0), (5, 15, 0, 0), (3, 32, 0, 0), (33, 127, 1, 2), (64, 128, 0, 0), (7, 129, 3, 0),
                                                 (1000, 96, 0, 32), (17, 512, 0, 0), (3, 1000, 1, 1), (2, 4096, 0, 0)])
def test_quantise_is_the_oracle_s(hip, kind, rows, dim, lead, extra):
    rng = np.random.default_rng(rows * dim)
    x = rng.standard_normal((rows, dim)) * np.exp(2 * rng.standard_normal((rows, 1)))
    x[rng.random((rows, dim)) < 0.1] = 0
    base, view = strided(x, kind, lead, extra)
    table = hip.quantize_blocks(view)
    want, exponents = rows_oracle.quantise(numbers(view))
    assert (table.exponents.cpu().numpy() == exponents).all()
    assert (table_numbers(hip, table) == want).all()
    assert int(table.values[:, dim:].max()) == 0 if table.values.shape[1] > dim else True
    # the values back in each type, rounded once
    for out in TYPES:
        back_base, back = strided(np.zeros((rows, dim)), out, lead, extra)
        hip.dequantize_blocks(table, back)
        expected = torch.from_numpy(want).to(TYPES[out])  # every value is a float, so one rounding
        assert torch.equal(back.cpu(), expected) and gaps_intact(back_base, back)
    again = hip.quantize_blocks(view)
    assert torch.equal(again.values, table.values) and torch.equal(again.exponents, table.exponents)


def test_quantise_edges(hip):
    """Blocks at the border of a scale, ties, the least steps, tiny blocks, zeros of both signs, NaN and infinities."""
    x = np.zeros((10, 200), np.float32)
    x[0, :5] = [448, 17, 19, 1 / 512, 3 / 1024]           # exponent 0: 17 and 19 lie between two steps of 2
    x[1, :2] = [448.0000305, 1]                          # just above: the next power
    x[2, :3] = [np.float32(1e-40), -np.float32(2e-41), 0]  # below every exponent
    x[3, 150] = np.inf                                   # the second block only
    x[4, 3] = np.nan
    x[5, 3] = -np.inf
    x[6] = -0.0
    x[7, :2] = [3.4e38, -3.4e38]
    x[8, :4] = [1.75, 1.75 * 2 ** -9, 2.0 ** -18, 2.0 ** -19]
    x[9, :2] = [2.0 ** -126, 2.0 ** -130]
    table = hip.quantize_blocks(torch.from_numpy(x).to(DEV))
    want, exponents = rows_oracle.quantise(x)
    assert (table.exponents.cpu().numpy() == exponents).all()
    with np.errstate(over="ignore"):  # 3.4e38 is nearest to 2^128 among the block's values, and that rounds to infinity in float32
        np.testing.assert_array_equal(table_numbers(hip, table), want.astype(np.float32))


@pytest.mark.parametrize("query_kind,kind", [("f32", "f32"), ("bf16", "f16"), ("f16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("m,n,dim", [(1, 1, 1), (1, 63, 32), (1, 5000, 128), (3, 257, 100), (16, 1000, 512), (16, 300, 513), (17, 64, 128),
                                     (33, 1023, 96), (65, 2049, 200), (128, 256, 256), (129, 5001, 64), (300, 777, 130), (1, 1000, 1000),
                                     (40, 130, 4096)])
def test_logits_against_the_oracle(hip, query_kind, kind, m, n, dim):
    rng = np.random.default_rng(m + n + dim)
    x = rng.standard_normal((n, dim)) * (0.1 + rng.random((n, 1)) ** 3)
    table = hip.quantize_blocks(strided(x, "f32")[1])
    lead, extra = (0, 0) if n % 2 else (3, 5)
    _, query = strided(rng.standard_normal((m, dim)), query_kind, lead, extra)
    base, logits = strided(np.zeros((m, n)), kind, lead, extra)
    hip.block_logits(query, table, logits)
    q, t = rows_oracle.quantise(numbers(query))[0], table_numbers(hip, table)
    exact, magnitude = q @ t.T, np.abs(q) @ np.abs(t).T
    error = np.abs(numbers(logits) - exact)
    assert (error <= 2 * dim * 2.0 ** -24 * magnitude * 1.01 + rounding(kind, exact)).all(), error.max()
    assert gaps_intact(base, logits)
    again = torch.empty_like(logits)
    hip.block_logits(query, table, again)
    assert torch.equal(again, logits)


@pytest.mark.parametrize("n", [1, 64, 65, 192, 193, 255, 257, 320, 321, 448, 449])
def test_strips_that_end_before_their_waves(hip, n):
    """Tables whose last strip of 256 candidates leaves whole waves without any."""
    rng = np.random.default_rng(n)
    _, rows = strided(rng.standard_normal((n, 260)), "f32")
    _, query = strided(rng.standard_normal((21, 260)), "bf16")
    table = hip.quantize_blocks(rows)
    out_base, out = strided(np.zeros((21, n)), "f32", 1, 2)
    hip.block_logits(query, table, out)
    q, x = rows_oracle.quantise(numbers(query))[0], table_numbers(hip, table)  # the product rounds its queries to 8 bits too
    bound = 2 * 260 * 2.0 ** -24 * (np.abs(q) @ np.abs(x).T)
    exact = q @ x.T
    assert (np.abs(numbers(out) - exact) <= bound + rounding("f32", exact)).all()
    assert gaps_intact(out_base, out)


def test_few_and_many_queries_agree(hip):
    """The two kernels add in the same order: a query's logits do not depend on how many ask with it."""
    rng = np.random.default_rng(0)
    table = hip.quantize_blocks(strided(rng.standard_normal((3001, 256)), "f32")[1])
    query = strided(rng.standard_normal((200, 256)), "f32")[1]
    whole = torch.empty(200, 3001, device=DEV)
    hip.block_logits(query, table, whole)
    for first, count in ((0, 1), (7, 16), (50, 17), (100, 40), (120, 80)):
        part = torch.empty(count, 3001, device=DEV)
        hip.block_logits(query[first:first + count], table, part)
        assert torch.equal(part, whole[first:first + count])


def test_logits_of_marked_blocks_and_padding(hip):
    """A row with a NaN answers NaN and no other row does; a table whose rows are wider than their columns; a float8 view of the bytes."""
    from graphvite_amd.kernels import BlockTable
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 40)).astype(np.float32)
    x[7, 3] = np.nan
    query = torch.from_numpy(rng.standard_normal((20, 40)).astype(np.float32)).to(DEV)
    query[4, 0] = np.inf
    wide = BlockTable(torch.full((50, 80), 0x7f, dtype=torch.uint8, device=DEV), torch.empty(50, 1, dtype=torch.uint8, device=DEV), 40)
    hip.quantize_blocks(torch.from_numpy(x).to(DEV), wide)
    assert bool((wide.values[:, 48:] == 0x7f).all())  # behind the padded columns nothing is written, nor read
    logits = torch.empty(20, 50, device=DEV)
    hip.block_logits(query, wide, logits)
    nan = torch.isnan(logits).cpu().numpy()
    want = np.zeros((20, 50), bool)
    want[:, 7] = want[4] = True
    assert (nan == want).all()
    other = torch.empty_like(logits)
    hip.block_logits(query, BlockTable(wide.values.view(torch.float8_e4m3fn), wide.exponents, 40), other)
    assert torch.equal(other[:4], logits[:4]) or bool((torch.nan_to_num(other[:4]) == torch.nan_to_num(logits[:4])).all())
    empty = torch.empty(0, 50, device=DEV)
    hip.block_logits(query[:0], wide, empty)


def test_block_calls_refuse_what_does_not_fit(hip):
    from graphvite_amd.kernels import BlockTable
    table = hip.quantize_blocks(torch.zeros(8, 40, device=DEV))
    with pytest.raises(ValueError, match="columns"):
        hip.block_logits(torch.zeros(2, 41, device=DEV), table, torch.zeros(2, 8, device=DEV))
    with pytest.raises(ValueError, match="shape"):
        hip.block_logits(torch.zeros(2, 40, device=DEV), table, torch.zeros(2, 9, device=DEV))
    with pytest.raises(ValueError, match="dtype"):
        hip.block_logits(torch.zeros(2, 40, device=DEV).double(), table, torch.zeros(2, 8, device=DEV))
    with pytest.raises(ValueError, match="expected cuda"):
        hip.block_logits(torch.zeros(2, 40), table, torch.zeros(2, 8, device=DEV))
    with pytest.raises(ValueError, match="BlockTable of the rows' shape"):
        hip.quantize_blocks(torch.zeros(9, 40, device=DEV), table)
    with pytest.raises(ValueError, match="multiples of 16"):
        BlockTable(torch.zeros(8, 40, dtype=torch.uint8, device=DEV), table.exponents, 40)
    with pytest.raises(ValueError, match="shape"):
        BlockTable(table.values, torch.zeros(8, 2, dtype=torch.uint8, device=DEV), 40)
    with pytest.raises(ValueError, match="overlap"):
        hip.block_logits(torch.zeros(2, 40, device=DEV), table, torch.zeros(9, device=DEV).as_strided((2, 8), (1, 1)))


# ---- the top of a row ----------------------------------------------------------------------------------------------------------

def check_top(hip, view, k, temperature):
    rows = view.shape[0]
    values, index = torch.empty(rows, k, device=DEV), torch.empty(rows, k, dtype=torch.int32, device=DEV)
    stats = torch.empty(rows, 2, device=DEV)
    hip.top_logits(view, values, index, stats, temperature=temperature)
    want_values, want_index, want_stats = rows_oracle.top(numbers(view), k, temperature)
    np.testing.assert_array_equal(index.cpu().numpy(), want_index)
    np.testing.assert_array_equal(numbers(values), want_values)
    np.testing.assert_array_equal(numbers(stats)[:, 0], want_stats[:, 0])
    np.testing.assert_allclose(numbers(stats)[:, 1], want_stats[:, 1], rtol=0, atol=1e-5)
    again_values, again_index = torch.empty_like(values), torch.empty_like(index)
    hip.top_logits(view, again_values, again_index, temperature=temperature)  # without stats
    assert torch.equal(again_index, index)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,n,k,lead,extra", [(1, 1, 1, 0, 0), (3, 7, 7, 1, 0), (2, 255, 255, 0, 1), (4, 256, 256, 0, 0), (5, 1000, 256, 3, 0),
                                                 (3, 4096, 10, 0, 0), (2, 4097, 64, 1, 1), (7, 10312, 10, 0, 0), (2, 16384, 100, 0, 0),
                                                 (2, 16385, 256, 5, 0), (1, 99991, 1, 0, 0), (9, 99991, 100, 0, 0), (100, 99991, 33, 0, 0),
                                                 (2, 300007, 256, 1, 2)])
def test_top_logits_against_the_oracle(hip, kind, rows, n, k, lead, extra):
    rng = np.random.default_rng(rows + n + k)
    z = 2 * rng.standard_normal((rows, n))
    z[rng.random((rows, n)) < 0.01] = -np.inf
    base, view = strided(z, kind, lead, extra)
    check_top(hip, view, k, [1.0, 0.5, 4.0][k % 3])
    assert gaps_intact(base, view)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [100, 5000, 20000, 100003])
def test_top_logits_of_rows_that_defeat_the_bound(hip, kind, n):
    """All equal, all masked, sorted either way, few distinct values, zeros of both signs, the type's least value, one spike among masks,
    all the large ones in one thread's chunks."""
    rng = np.random.default_rng(n)
    low = float(torch.finfo(TYPES[kind]).min)
    z = np.zeros((11, n))
    z[1] = -np.inf
    z[2] = np.arange(n) / 64.0
    z[3] = -np.arange(n) / 64.0
    z[4] = rng.integers(0, 3, n)
    z[5] = np.where(rng.random(n) < 0.5, 0.0, -0.0)
    z[6] = low
    z[7] = -np.inf
    z[7, n // 2] = 5
    z[8] = rng.standard_normal(n)
    z[8, :60] = 100
    z[9] = low
    z[9, ::7] = -np.inf
    z[10] = rng.standard_normal(n) + 300.0
    for k in (1, 37, 64) if n == 100 else (1, 37, 256):
        check_top(hip, strided(z, kind)[1], k, 1.0)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [4088, 4097, 8185, 8193, 12281, 12289, 16377, 16385])
def test_top_logits_at_the_sizes_between_builds(hip, kind, n):
    """Rows that just fit a build and rows that just do not, beginning on sixteen bytes and elsewhere; the last elements among the largest."""
    z = np.random.default_rng(n).standard_normal((3, n))
    z[:, -3:] += 5
    z[0, :9] += 5
    for lead, extra in ((0, 8 - n % 8), (1, 0)):
        for k in (5, 64, 200):
            check_top(hip, strided(z, kind, lead, extra)[1], k, 1.0)


def test_top_logits_shows_nan_and_infinity(hip):
    for n in (50, 30000):
        z = np.random.default_rng(n).standard_normal((4, n))
        z[0, 11] = np.nan
        z[1, 20], z[1, 7] = -np.nan, np.nan
        z[2, 3] = np.inf
        z[3, 3], z[3, 40], z[3, 41] = np.inf, np.nan, np.inf
        view = strided(z, "f32")[1]
        values, index, stats = torch.empty(4, 5, device=DEV), torch.empty(4, 5, dtype=torch.int32, device=DEV), torch.empty(4, 2, device=DEV)
        hip.top_logits(view, values, index, stats)
        want_values, want_index, _ = rows_oracle.top(numbers(view), 5, 1.0)
        np.testing.assert_array_equal(index.cpu().numpy(), want_index)
        np.testing.assert_array_equal(numbers(values), want_values)
        assert np.isnan(numbers(stats)[:, 1]).all()
        assert np.isinf(numbers(stats)[2:, 0]).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [40, 3000, 70000])
def test_top_logits_with_nan_beside_the_largest(hip, kind, n):
    """A NaN of either sign next to the row's largest logit: the NaN comes first, the largest after it, and m is the largest all the same."""
    z = np.random.default_rng(n).standard_normal((4, n)) - 10.0
    for r, (nan, large) in enumerate([(np.nan, 3.0), (-np.nan, 3.0), (np.nan, -2.0), (-np.nan, -2.0)]):
        z[r, n // 2], z[r, n // 2 + 1] = nan, large
    view = strided(z, kind)[1]
    values, index, stats = torch.empty(4, 3, device=DEV), torch.empty(4, 3, dtype=torch.int32, device=DEV), torch.empty(4, 2, device=DEV)
    hip.top_logits(view, values, index, stats)
    want_values, want_index, want_stats = rows_oracle.top(numbers(view), 3, 1.0)
    np.testing.assert_array_equal(index.cpu().numpy(), want_index)
    np.testing.assert_array_equal(numbers(values), want_values)
    np.testing.assert_array_equal(numbers(stats)[:, 0], want_stats[:, 0])
    assert np.isnan(numbers(stats)[:, 1]).all()


def test_calls_from_two_threads_on_two_streams(hip):
    """Two host threads, a stream each, the same calls over inputs of their own, interleaved as they come: every answer is what one thread gets."""
    import threading

    def inputs(seed):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        return torch.randn(40, 200, generator=g, device=DEV), torch.randn(30011, 200, generator=g, device=DEV)

    def answers(query, rows):
        table = hip.quantize_blocks(rows)
        logits = torch.empty(40, 30011, device=DEV)
        hip.block_logits(query, table, logits)
        values, index = torch.empty(40, 50, device=DEV), torch.empty(40, 50, dtype=torch.int32, device=DEV)
        stats, loss, grad = torch.empty(40, 2, device=DEV), torch.empty(40, device=DEV), torch.empty_like(logits)
        hip.top_logits(logits, values, index, stats)
        hip.distill(logits, index, values + 1, loss, stats, grad=grad)
        return logits, values, index, loss, grad

    given = [inputs(1), inputs(2)]
    want = [answers(*x) for x in given]
    torch.cuda.synchronize()
    wrong = []

    def work(which):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(15):
                    got = answers(*given[which])
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[which])):
                        wrong.append(which)
        except Exception as e:  # shown by the main thread
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(which,)) for which in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_rows_behind_the_32_bit_line(hip):
    """Row starts beyond 2^32 elements: 5 rows 2^30 apart."""
    stride, n = 1 << 30, 3000
    base = torch.empty(4 * stride + n, dtype=torch.bfloat16, device=DEV)
    z = np.random.default_rng(0).standard_normal((5, n))
    view = base.as_strided((5, n), (stride, 1))
    view.copy_(torch.from_numpy(z).to(torch.bfloat16))
    check_top(hip, view, 20, 1.0)
    table = hip.quantize_blocks(view)
    assert (table_numbers(hip, table) == rows_oracle.quantise(numbers(view))[0]).all()
    index = torch.from_numpy(np.random.default_rng(1).integers(0, n, (5, 9)).astype(np.int32)).to(DEV)
    teacher = torch.randn(5, 9, device=DEV)
    loss, stats = torch.empty(5, device=DEV), torch.empty(5, 2, device=DEV)
    near, near_stats = torch.empty(5, device=DEV), torch.empty(5, 2, device=DEV)
    small = view.clone()
    small_grad = torch.empty_like(small)
    hip.distill(small, index, teacher, near, near_stats, grad=small_grad)
    hip.distill(view, index, teacher, loss, stats, grad=view)
    assert torch.equal(loss, near) and torch.equal(view, small_grad)
    query = torch.randn(5, 64, device=DEV)
    small_table = hip.quantize_blocks(torch.randn(n, 64, device=DEV))
    plain = torch.empty(5, n, dtype=torch.bfloat16, device=DEV)
    hip.block_logits(query, small_table, plain)
    hip.block_logits(query, small_table, view)
    assert torch.equal(plain, view)


def test_top_logits_refuses(hip):
    z = torch.zeros(3, 8, device=DEV)
    with pytest.raises(ValueError, match="top 9 of 8"):
        hip.top_logits(z, torch.zeros(3, 9, device=DEV), torch.zeros(3, 9, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="shape"):
        hip.top_logits(z, torch.zeros(3, 2, device=DEV), torch.zeros(3, 3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="dtype"):
        hip.top_logits(z, torch.zeros(3, 2, device=DEV), torch.zeros(3, 2, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="temperature"):
        hip.top_logits(z, torch.zeros(3, 2, device=DEV), torch.zeros(3, 2, dtype=torch.int32, device=DEV), temperature=0.0)


# ---- distillation --------------------------------------------------------------------------------------------------------------

def make_lists(rng, rows, n, k, repeats):
    index = np.stack([rng.integers(0, n, k) if repeats or k > n else rng.permutation(n)[:k] for _ in range(rows)]).astype(np.int32)
    teacher = (3 * rng.standard_normal((rows, k))).astype(np.float32)
    index[rng.random((rows, k)) < 0.1] = -1
    teacher[rng.random((rows, k)) < 0.05] = -np.inf
    if rows > 2:
        index[1] = -1        # no entries
        teacher[2] = -np.inf  # none either
    return index, teacher


def check_distill(hip, view, index, teacher, temperature, teacher_stats=None, weight=None, grad_lead=0, grad_extra=0):
    kind = {v: k for k, v in TYPES.items()}[view.dtype]
    z = numbers(view)
    rows, n = z.shape
    want_loss, want_stats, want_grad, grad_scale, loss_scale = rows_oracle.distill(z, index, teacher, temperature, teacher_stats, weight)
    put = lambda a, t: None if a is None else torch.as_tensor(np.asarray(a), dtype=t).to(DEV)  # noqa: E731
    lists = put(index, torch.int32), put(teacher, torch.float32)
    given = dict(teacher_stats=put(teacher_stats, torch.float32), temperature=temperature, weight=put(weight, torch.float32))

    def compare(loss, stats, grad):
        if loss is not None:
            np.testing.assert_array_equal(numbers(stats)[:, 0], want_stats[:, 0])
            np.testing.assert_allclose(numbers(stats)[:, 1], want_stats[:, 1], rtol=0, atol=1e-5)
            got = numbers(loss)
            # a loss within the tolerance of the largest float may round to infinity: (1 + 2e-5) * 3.40282e38 is above it
            border = want_loss > (1 - 2e-5) * np.finfo(np.float32).max
            assert (got[border] > 3.4e38).all()
            got, want_loss_, loss_scale_ = got[~border], want_loss[~border], loss_scale[~border]
            finite = np.isfinite(want_loss_)
            np.testing.assert_array_equal(got[~finite], want_loss_[~finite])
            assert (np.abs(got[finite] - want_loss_[finite]) <= 2e-5 * loss_scale_[finite]).all(), (got, want_loss_)
        if grad is not None:
            got = numbers(grad)
            assert (np.isnan(got) == np.isnan(want_grad)).all()
            error = np.where(np.isnan(want_grad), 0, np.abs(got - want_grad))
            bound = np.where(np.isnan(want_grad), 0, 2e-5 * grad_scale + rounding(kind, want_grad) + 2e-5 * rounding(kind, grad_scale))
            assert (error <= bound).all(), (error.max(), np.argwhere(error > bound)[:5])

    empty = lambda *shape: torch.full(shape, 77.0, device=DEV)  # noqa: E731
    loss, stats = empty(rows), empty(rows, 2)
    hip.distill(view, *lists, loss, stats, **given)
    compare(loss, stats, None)
    base, grad = strided(np.zeros((rows, n)), kind, grad_lead, grad_extra)
    loss2, stats2 = empty(rows), empty(rows, 2)
    hip.distill(view, *lists, loss2, stats2, grad=grad, **given)
    compare(loss2, stats2, grad)
    assert gaps_intact(base, grad)
    alone = torch.full_like(view, 77.0)
    hip.distill_grad(view, *lists, stats2, alone, **given)
    compare(None, None, alone)
    over = same_place(view)  # a sum's order goes by where in 16 bytes a row begins
    loss3, stats3 = empty(rows), empty(rows, 2)
    hip.distill(over, *lists, loss3, stats3, grad=over, **given)  # over the logits
    assert torch.equal(torch.nan_to_num(over), torch.nan_to_num(grad)) and torch.equal(torch.nan_to_num(loss3), torch.nan_to_num(loss2))
    over = same_place(view)
    hip.distill_grad(over, *lists, stats2, over, **given)
    assert torch.equal(torch.nan_to_num(over), torch.nan_to_num(alone))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,n,k,lead,extra", [(1, 1, 1, 0, 0), (3, 2, 5, 1, 0), (5, 63, 7, 0, 0), (4, 1000, 10, 3, 5), (3, 2041, 100, 0, 0),
                                                 (3, 2049, 3, 1, 0), (3, 8192, 64, 0, 0), (4, 10312, 10, 0, 0), (3, 16380, 1024, 0, 4),
                                                 (3, 16384, 32, 0, 0), (3, 16391, 300, 7, 0), (3, 40000, 128, 0, 1), (2, 99991, 100, 0, 0)])
def test_distill_against_the_oracle(hip, kind, rows, n, k, lead, extra):
    rng = np.random.default_rng(rows + n + k)
    z = 2 * rng.standard_normal((rows, n))
    masked = rng.random((rows, n)) < 0.02
    index, teacher = make_lists(rng, rows, n, k, repeats=k % 2 == 0)
    for r in range(rows):
        masked[r, index[r][index[r] >= 0]] = False
    z[masked] = -np.inf
    whole = rng.random() < 0.5
    with np.errstate(all="ignore"):
        top = np.where(np.isfinite(teacher), teacher, -1e9).max(1)
        top = np.where(top < -1e8, 0, top)
        teacher_stats = np.stack([top, np.log(np.exp((np.where(np.isfinite(teacher), teacher, -1e9) - top[:, None]) / 2.0).sum(1) / 0.7 + 1e-3)], 1).astype(np.float32)
    weight = rng.random(rows).astype(np.float32)
    view = strided(z, kind, lead, extra)[1]
    check_distill(hip, view, index, teacher, 1.0)
    check_distill(hip, view, index, teacher, 2.0, teacher_stats=teacher_stats, weight=weight, grad_lead=1, grad_extra=3)
    check_distill(hip, view, index, teacher, 0.5, weight=-weight if whole else None, grad_lead=lead, grad_extra=extra)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2041, 2049, 4089, 4097, 6137, 6145, 8185, 8193, 12281, 12289, 16377, 16385])
def test_distill_at_the_sizes_between_builds(hip, kind, n):
    """As above, with entries on the row's first and last candidates, and one of them twice."""
    rng = np.random.default_rng(n)
    z = rng.standard_normal((3, n))
    index = np.stack([rng.permutation(n)[:40] for _ in range(3)]).astype(np.int32)
    index[:, :3] = (0, n - 1, n // 2)
    index[1, 7] = index[1, 30] = n - 1
    for lead, extra in ((0, 8 - n % 8), (1, 0)):
        check_distill(hip, strided(z, kind, lead, extra)[1], index, (rng.standard_normal((3, 40)) * 2).astype(np.float32), 1.5, grad_lead=lead)


@pytest.mark.parametrize("n", [200, 3000, 33000])
def test_distill_edges(hip, n):
    """Rows all masked, the type's lowest value as a mask, a listed candidate masked, an index outside the row on either side, one candidate
    listed by every entry, NaN and infinity among the logits, weights zero and negative."""
    rng = np.random.default_rng(n)
    z = rng.standard_normal((10, n))
    index = np.stack([rng.permutation(n)[:6] for _ in range(10)]).astype(np.int32)
    teacher = rng.standard_normal((10, 6)).astype(np.float32)
    z[0] = -np.inf
    z[1, 10:] = np.finfo(np.float32).min
    z[2] = np.finfo(np.float32).min
    z[3, index[3, 0]] = -np.inf
    index[4, 2] = n
    index[5, 5] = -2
    index[6] = n - 1
    index[7, 0] = 2 ** 31 - 1
    z[8] -= 500
    z[9] += 500
    weight = np.array([1, 2, 0, 1, 1, 0, -3, 1, 1, 1], np.float32)
    check_distill(hip, strided(z, "f32")[1], index, teacher, 1.0, weight=weight)
    # a teacher list whose other entries underflow: q = 0 there, and 0 log 0 = 0 also where that candidate is masked
    sharp = np.full((10, 6), -2000.0, np.float32)
    sharp[:, 1] = 0
    check_distill(hip, strided(z, "f32")[1], index, sharp, 1.0)
    # NaN and plus infinity in a row show in its answer; without entries the row answers 0
    bad = rng.standard_normal((3, n))
    bad[0, 5], bad[1, 6], bad[2, 7] = np.nan, np.inf, np.nan
    lists = torch.tensor([[1, 2], [1, 2], [-1, -1]], dtype=torch.int32, device=DEV), torch.zeros(3, 2, device=DEV)
    view = strided(bad, "f32")[1]
    loss, stats, grad = torch.empty(3, device=DEV), torch.empty(3, 2, device=DEV), torch.empty(3, n, device=DEV)
    hip.distill(view, *lists, loss, stats, grad=grad)
    assert torch.isnan(loss).tolist() == [True, True, False] and loss[2] == 0
    assert bool(torch.isnan(grad[:2]).all()) and bool((grad[2] == 0).all())
    hip.distill_grad(view, *lists, stats, grad)
    assert bool(torch.isnan(grad[:2]).all()) and bool((grad[2] == 0).all())


def test_distill_refuses(hip):
    z, index, teacher = torch.zeros(3, 8, device=DEV), torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.zeros(3, 2, device=DEV)
    loss, stats = torch.zeros(3, device=DEV), torch.zeros(3, 2, device=DEV)
    with pytest.raises(ValueError, match="shape"):
        hip.distill(z, index, teacher[:, :1].contiguous(), loss, stats)
    with pytest.raises(ValueError, match="dtype"):
        hip.distill(z, index.long(), teacher, loss, stats)
    with pytest.raises(ValueError, match="dtype"):
        hip.distill(z, index, teacher, loss, stats, grad=torch.zeros(3, 8, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="shape"):
        hip.distill(z, index, teacher, loss, stats, weight=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError, match="overlaps"):
        both = torch.zeros(40, device=DEV)
        hip.distill(both[:24].view(3, 8), index, teacher, loss, stats, grad=both[8:32].view(3, 8))
    with pytest.raises(ValueError, match="temperature"):
        hip.distill(z, index, teacher, loss, stats, temperature=float("nan"))
    with pytest.raises(ValueError, match="expected cuda"):
        hip.distill(z, index, teacher.cpu(), loss, stats)


# ---- together -------------------------------------------------------------------------------------------------------------------

def run_together(hip, teacher_query, teacher_table, student_logits, k, temperature):
    """A teacher answers from its 8-bit table, its top logits are kept, a student's logits learn from them."""
    rows, n = student_logits.shape
    logits = torch.empty(rows, n, dtype=torch.bfloat16, device=DEV)
    hip.block_logits(teacher_query, teacher_table, logits)
    values, index, teacher_stats = torch.empty(rows, k, device=DEV), torch.empty(rows, k, dtype=torch.int32, device=DEV), torch.empty(rows, 2, device=DEV)
    hip.top_logits(logits, values, index, teacher_stats, temperature=temperature)
    loss, stats, grad = torch.empty(rows, device=DEV), torch.empty(rows, 2, device=DEV), torch.empty_like(student_logits)
    hip.distill(student_logits, index, values, loss, stats, teacher_stats=teacher_stats, temperature=temperature, grad=grad)
    return logits, values, index, teacher_stats, loss, grad


@pytest.mark.parametrize("rows,n", [(3, 2000), (70, 30011)])
def test_a_teacher_s_answers_train_a_student(hip, rows, n):
    """The operators in a row, each output against the oracle on the inputs it had."""
    rng = np.random.default_rng(n)
    table = hip.quantize_blocks(strided(rng.standard_normal((n, 96)), "f32")[1])
    query = strided(rng.standard_normal((rows, 96)) * 0.5, "f32")[1]
    student = strided(2 * rng.standard_normal((rows, n)), "f32")[1]
    logits, values, index, teacher_stats, loss, grad = run_together(hip, query, table, student, 32, 2.0)
    want_values, want_index, want_stats = rows_oracle.top(numbers(logits), 32, 2.0)
    np.testing.assert_array_equal(index.cpu().numpy(), want_index)
    np.testing.assert_allclose(numbers(teacher_stats), want_stats, rtol=0, atol=1e-5)
    want_loss, _, want_grad, grad_scale, loss_scale = rows_oracle.distill(numbers(student), index.cpu().numpy(), numbers(values), 2.0, numbers(teacher_stats))
    assert (np.abs(numbers(loss) - want_loss) <= 2e-5 * loss_scale).all()
    assert (np.abs(numbers(grad) - want_grad) <= 2e-5 * grad_scale + rounding("f32", want_grad)).all()
    # the gradient against differences of the loss itself (64-bit oracle; h = 1e-4, third derivatives below 1)
    for j in [int(want_index[0, 0]), int(want_index[0, 5]), 0]:
        z = numbers(student)[:1]
        up, down = z.copy(), z.copy()
        up[0, j] += 1e-4
        down[0, j] -= 1e-4
        one = lambda x: rows_oracle.distill(x, index.cpu().numpy()[:1], numbers(values)[:1], 2.0, numbers(teacher_stats)[:1])[0][0]  # noqa: E731
        assert abs((one(up) - one(down)) / 2e-4 - numbers(grad)[0, j]) < 1e-7


def test_other_streams_and_graphs(hip):
    """The run on a side stream gives the same bits; captured, it does so in every replay with eager work of the same kind in between, also
    where two captured graphs take turns, and new inputs in the captured tensors give new answers."""
    rng = np.random.default_rng(9)
    n = 20011
    table = hip.quantize_blocks(strided(rng.standard_normal((n, 128)), "f32")[1])
    query, student = strided(rng.standard_normal((40, 128)), "f32")[1], strided(rng.standard_normal((40, n)), "f32")[1]
    query2, student2 = strided(rng.standard_normal((40, 128)), "f32")[1], strided(rng.standard_normal((40, n)), "f32")[1]
    eager = run_together(hip, query, table, student, 16, 1.0)
    eager2 = run_together(hip, query2, table, student2, 16, 1.0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = run_together(hip, query, table, student, 16, 1.0)
    side.synchronize()
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graphs, outputs = [], []
    for q, s in ((query, student), (query2, student2)):
        q, s = q.clone(), s.clone()
        with torch.cuda.stream(side):
            run_together(hip, q, table, s, 16, 1.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append((q, s, run_together(hip, q, table, s, 16, 1.0)))
        graphs.append(graph)
    for turn in range(4):
        for graph in graphs:
            graph.replay()
        run_together(hip, query2, table, student2, 16, 1.0)  # eager work between replays
        torch.cuda.synchronize()
        for got, want in zip([o for _, _, o in outputs], (eager, eager2)):
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    q, s, out = outputs[0]
    q.copy_(query2)
    s.copy_(student2)
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(out, eager2):
        assert torch.equal(a, b)
