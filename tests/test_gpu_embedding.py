"""Table operators on the GPU against the definition in 64 bits.

Tolerances count roundings. A lookup makes one product with a factor rounded to
32 bits (2 x 2^-24) and one conversion (half a step of the type). A row's
gradient adds m terms in 32 bits in some order: at most m roundings of partial
sums, each at most 2^-24 of the sum of the terms' sizes, then the factor as
above and one conversion.
"""

import math

import numpy as np
import pytest
import torch

import draws

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
SEED, OFFSET = 0xFEDCBA9876543210, 2 ** 35 + 7
U = 2.0 ** -24


def _step(dtype):
    """Half a step of the type relative to a value, and below its normal range."""
    return (0.0, 0.0) if dtype == torch.float32 else (torch.finfo(dtype).eps / 2, 2.0 ** -25)


def _tokens(kind, n, rows, rng):
    if kind == "uniform":
        return rng.integers(0, rows, n)
    if kind == "skewed":  # a few rows far more used than the rest
        return np.minimum((np.exp(rng.random(n) * math.log(rows + 1)) - 1).astype(np.int64), rows - 1)
    if kind == "same":
        return np.full(n, rows // 2)
    if kind == "sorted":
        return np.sort(rng.integers(0, rows, n))
    assert kind == "distinct"
    return rng.permutation(max(n, rows))[:n] % rows


def _case(n, rows, width, dtype, cuda, *, kind="uniform", bits=64, padding=False, seed=0):
    rng = np.random.default_rng(seed)
    index = _tokens(kind, n, rows, rng)
    if padding:
        index = np.where(rng.random(n) < 0.2, -1, index)
    index = torch.from_numpy(index.astype(np.int64)).to(torch.int64 if bits == 64 else torch.int32)
    table = torch.from_numpy(rng.standard_normal((rows, width))).to(dtype)
    grad = torch.from_numpy(rng.standard_normal((n, width))).to(dtype)
    return table.to(cuda), index.to(cuda), grad.to(cuda)


def _check_lookup(got, table, index, scale, p, dtype, offset=OFFSET):
    t, i = table.double().cpu().numpy(), index.cpu().numpy().reshape(-1)
    want = np.where((i >= 0)[:, None], t[np.maximum(i, 0)], 0.0) * scale
    if p > 0:
        want = want * draws.weight(want.shape, p, SEED, offset)
    half, tiny = _step(dtype)
    got = got.double().cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= np.abs(want) * (half + 2.01 * U) + tiny).all()


def _check_gradient(got, grad, index, rows, scale, p, dtype, offset=OFFSET):
    g, i = grad.double().cpu().numpy(), index.cpu().numpy().reshape(-1)
    g = g.reshape(len(i), -1) * scale
    if p > 0:
        g = g * draws.weight(g.shape, p, SEED, offset)
    want, size = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1]))
    real = i >= 0
    np.add.at(want, i[real], g[real])
    np.add.at(size, i[real], np.abs(g[real]))
    terms = np.bincount(i[real], minlength=rows)[:, None]
    half, tiny = _step(dtype)
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert not got[terms[:, 0] == 0].any()
    limit = size * (terms + 2.01) * U + np.abs(want) * half + tiny * (terms > 0)
    assert (np.abs(got - want) <= limit).all(), np.max(np.abs(got - want) - limit)


SIZES = [(1, 1, 1), (1, 5, 2048), (2, 1, 3), (7, 3, 45), (31, 100, 48), (32, 2, 16), (33, 1000, 77),
         (257, 9, 130), (1000, 64, 300), (4097, 5003, 33), (3000, 1, 8), (20_011, 700, 48)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width", SIZES)
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_lookup(cuda, dtype, n, rows, width, p):
    import embedding

    for bits, padding, scale in ((64, False, 1.0), (32, True, -2.7)):
        table, index, _ = _case(n, rows, width, dtype, cuda, bits=bits, padding=padding)
        got = embedding.lookup(table, index, scale=scale, padding_index=-1 if padding else None,
                               p=p, seed=SEED, offset=OFFSET)
        assert got.dtype == dtype and got.shape == (n, width)
        _check_lookup(got, table, index, scale, p, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width", SIZES)
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_gradient(cuda, dtype, n, rows, width, p):
    import embedding

    for kind, bits, padding, scale in (("uniform", 64, False, 1.0), ("skewed", 32, True, 0.3),
                                       ("same", 64, True, 1.0)):
        _, index, grad = _case(n, rows, width, dtype, cuda, kind=kind, bits=bits, padding=padding)
        got = embedding.lookup_gradient(grad, index, rows, scale=scale, p=p, seed=SEED,
                                        padding_index=-1 if padding else None, offset=OFFSET)
        assert got.dtype == dtype
        _check_gradient(got, grad, index, rows, scale, p, dtype)


@pytest.mark.parametrize("kind", ["uniform", "skewed", "same", "sorted", "distinct"])
@pytest.mark.parametrize("n,rows", [(1, 1), (100, 1000), (4096, 255), (4097, 256), (8191, 1023),
                                    (8193, 1024), (50_000, 70_000), (16_385, 70_000), (32_768, 5), (32_769, 600),
                                    (65_537, 31), (303_104, 4096), (303_105, 2047),
                                    (606_209, 511),
                                    (65_537, 3_000_000)])
def test_order(cuda, kind, n, rows):
    """The stable order, tokens without a row last."""
    import embedding

    for bits, padding in ((64, False), (32, True)):
        _, index, _ = _case(n, rows, 1, torch.float32, cuda, kind=kind, bits=bits, padding=padding)
        order = embedding.token_order(index, rows, padding_index=-1 if padding else None)
        i = index.cpu().numpy().astype(np.int64)
        i = np.where(i < 0, rows, i)
        place = np.argsort(i, kind="stable")
        assert np.array_equal(order.pairs.cpu().numpy(), np.stack([i[place], place], axis=1))


@pytest.mark.parametrize("kind", ["skewed", "same", "distinct"])
@pytest.mark.parametrize("n,rows,width", [(100_003, 4096, 48), (65_000, 60_000, 20),
                                          (300_000, 17, 5), (9000, 3, 513)])
def test_long_and_wide_sums(cuda, kind, n, rows, width):
    """Rows whose tokens lie in very many chunks; given and made orders agree
    bit for bit, and so do two runs."""
    import embedding

    _, index, grad = _case(n, rows, width, torch.float32, cuda, kind=kind)
    got = embedding.lookup_gradient(grad, index, rows)
    _check_gradient(got, grad, index, rows, 1.0, 0.0, torch.float32)
    order = embedding.token_order(index, rows)
    assert torch.equal(got, embedding.lookup_gradient(grad, None, rows, order=order))
    assert torch.equal(got, embedding.lookup_gradient(grad, index, rows))


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(cuda, dtype):
    """Strided and unaligned tables and gradients, indices of any shape, expanded
    and transposed gradients."""
    import embedding

    n, rows = 300, 50
    for width, gap, skip in ((48, 16, 0), (48, 5, 0), (48, 8, 1), (9, 3, 2), (64, 0, 0), (2, 6, 2)):
        table, index, grad = _case(n, rows, width + gap, dtype, cuda)
        table, grad = table[:, skip:skip + width], grad[:, skip:skip + width]
        got = embedding.lookup(table, index.view(3, 4, 25), p=0.2, seed=SEED, offset=OFFSET)
        assert got.shape == (3, 4, 25, width) and got.is_contiguous()
        _check_lookup(got, table, index, 1.0, 0.2, dtype)
        got = embedding.lookup_gradient(grad, index.view(20, 15), rows, p=0.2, seed=SEED,
                                        offset=OFFSET)
        _check_gradient(got, grad, index, rows, 1.0, 0.2, dtype)
    wide = torch.stack([index, index], dim=1)[:, 0]  # strided indices
    assert torch.equal(embedding.lookup(table, wide), embedding.lookup(table, index))
    for g in (grad[:1].expand(n, 2), grad.t().contiguous().t(), grad[0, :1].expand(n, 2),
              grad.reshape(20, 15, 2).transpose(0, 1)):
        i = index if g.dim() == 2 else index.view(20, 15).t()
        _check_gradient(embedding.lookup_gradient(g, i, rows), g.reshape(n, 2), i, rows, 1.0,
                        0.0, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_do(cuda, dtype):
    import embedding

    none = torch.empty(0, dtype=torch.int64, device=cuda)
    table = torch.ones(4, 3, dtype=dtype, device=cuda)
    assert embedding.lookup(table, none).shape == (0, 3)
    got = embedding.lookup_gradient(torch.empty(0, 3, dtype=dtype, device=cuda), none, 4)
    assert got.shape == (4, 3) and not got.any()
    assert embedding.token_order(none, 4).pairs.shape == (0, 2)
    only_padding = torch.full((70,), 9, device=cuda)
    assert not embedding.lookup(table, only_padding, padding_index=9).any()
    g = torch.full((70, 3), float("nan"), dtype=dtype, device=cuda)
    assert not embedding.lookup_gradient(g, only_padding, 4, padding_index=9).any()
    one = torch.zeros(5, dtype=torch.int32, device=cuda)
    assert embedding.lookup(torch.ones(4, 0, dtype=dtype, device=cuda), one).shape == (5, 0)
    assert embedding.lookup_gradient(torch.ones(5, 0, dtype=dtype, device=cuda), one, 4).shape == (4, 0)
    # A padding index inside the table: its row is neither read nor given anything.
    index = torch.tensor([0, 1, 2, 1], device=cuda)
    table = torch.arange(12, device=cuda).view(4, 3).to(dtype) + 1
    assert embedding.lookup(table, index, padding_index=1)[[1, 3]].eq(0).all()
    assert embedding.lookup_gradient(torch.ones(4, 3, dtype=dtype, device=cuda), index, 4,
                                     padding_index=1).tolist() == [[1] * 3, [0] * 3, [1] * 3, [0] * 3]
    # Everything dropped.
    assert not embedding.lookup(table, index, p=1.0).any()
    assert not embedding.lookup_gradient(torch.ones(4, 3, dtype=dtype, device=cuda), index, 4,
                                         p=1).any()


def test_indices_outside_the_table(cuda):
    """They read nothing, give nothing and set the fault word."""
    import _native as native
    import embedding

    native.fault_status()
    table = torch.ones(4, 8, device=cuda)
    for bits in (torch.int64, torch.int32):
        bad = torch.tensor([0, 4, -1, 2 ** 31 - 1, -2 ** 31, 3], device=cuda).to(bits)
        got = embedding.lookup(table, bad)
        assert got.sum(1).tolist() == [8, 0, 0, 0, 0, 8]
        assert native.fault_status() == 256 and native.fault_status() == 0
        got = embedding.lookup_gradient(torch.ones(6, 8, device=cuda), bad, 4)
        assert got.sum(1).tolist() == [8, 0, 0, 8]
        assert native.fault_status() == 256
    far = torch.tensor([2 ** 32, 2 ** 62, -2 ** 63, 1], device=cuda)
    assert embedding.lookup(table, far).sum(1).tolist() == [0, 0, 0, 8]
    assert native.fault_status() == 256
    assert embedding.lookup(table, far, padding_index=2 ** 32)[3].tolist() == [1] * 8
    assert native.fault_status() == 256
    embedding.lookup(table, torch.tensor([-7, 1], device=cuda), padding_index=-7)
    assert native.fault_status() == 0


def test_infinities_and_nan_stay_where_they_are(cuda):
    import embedding

    index = torch.tensor([0, 1, 1, 2, 0], device=cuda)
    grad = torch.ones(5, 4, device=cuda)
    grad[1, 0], grad[2, 1], grad[3, 2] = float("inf"), float("nan"), -float("inf")
    got = embedding.lookup_gradient(grad, index, 4)
    assert got[0].tolist() == [2] * 4 and got[3].tolist() == [0] * 4
    assert got[1, 0] == float("inf") and torch.isnan(got[1, 1]) and got[1, 2:].tolist() == [2, 2]
    assert got[2, 2] == -float("inf") and got[2, [0, 1, 3]].tolist() == [1] * 3
    # Dropped, they are gone.
    grad = torch.full((64, 16), float("nan"), device=cuda)
    kept = draws.keep(np.arange(1024), 0.5, 3, 4).reshape(64, 16)
    got = embedding.lookup_gradient(grad, torch.arange(64, device=cuda), 64, p=0.5, seed=3, offset=4)
    assert np.array_equal(torch.isnan(got).cpu().numpy(), kept) and not got.nan_to_num().any()


@pytest.mark.parametrize("n", [200, 5000])
def test_an_order_that_no_sort_made_stays_in_bounds(cuda, n):
    """A TokenOrder is an ordinary tensor: whatever it holds, nothing outside the
    gradient and the table is touched (what comes out is then anything)."""
    import embedding

    rows, width = 40, 48
    _, index, grad = _case(n, rows, width, torch.float32, cuda)
    room = torch.full((rows + 200, width), 7.0, device=cuda)  # the table lies inside
    state = [room[100:100 + rows], *(_adam_state(rows, width, cuda)[1:])]
    rng = np.random.default_rng(0)
    for pairs in (rng.integers(-2 ** 31, 2 ** 31, (n, 2)), rng.integers(0, 100, (n, 2)),
                  np.stack([rng.integers(0, 60, n), rng.integers(0, 2 * n, n)], axis=1)):
        order = embedding.TokenOrder(torch.from_numpy(pairs.astype(np.int32)).to(cuda), rows)
        embedding.lookup_gradient(grad, None, rows, order=order)
        embedding.consume_torch_adam(*state, grad, None, rate=0.1, bias1=0.5, bias2_sqrt=0.5,
                                     order=order)
        torch.cuda.synchronize()
        assert (room[:100] == 7).all() and (room[100 + rows:] == 7).all()


def test_far_rows(cuda):
    """Element offsets past 2^32 in the table and in its gradient."""
    import embedding

    rows, width = 66_000, 65_600
    table = torch.zeros(rows, width, dtype=torch.float16, device=cuda)
    table[rows - 1] = 3.0
    table[65_536] = 2.0
    index = torch.tensor([rows - 1, 0, 65_536], device=cuda)
    assert embedding.lookup(table, index)[:, [0, width - 1]].tolist() == [[3, 3], [0, 0], [2, 2]]
    del table
    grad = torch.arange(1, 4, device=cuda).to(torch.float16).view(3, 1).expand(3, width)
    got = embedding.lookup_gradient(grad, index, rows)
    assert got[index][:, [0, 1, width - 1]].tolist() == [[1] * 3, [2] * 3, [3] * 3]
    assert [int(got[r].any()) for r in (1, 65_535, 65_537, rows - 2)] == [0] * 4


def test_far_tokens(cuda):
    """Output elements past 2^32, aligned and odd rows: the lookup's zeros are the
    generator's, and the gradient counts what the lookup kept."""
    import embedding

    n = 66_000
    for width in (65_600, 65_601):
        table = torch.ones(2, width, dtype=torch.float16, device=cuda)
        index = torch.arange(n, device=cuda) % 2
        y = embedding.lookup(table, index, p=0.5, seed=SEED, offset=OFFSET)
        for token in (0, 65_500, n - 1):
            kept = draws.keep(token * width + np.arange(500), 0.5, SEED, OFFSET)
            assert np.array_equal(y[token, :500].cpu().numpy() > 0, kept)
        columns = [0, 1, 30_000, width - 1]
        want = torch.stack([(y[r::2][:, columns] > 0).sum(0) for r in (0, 1)])
        del y
        grad = torch.ones(1, width, device=cuda).expand(n, width)
        got = embedding.lookup_gradient(grad, index, 2, scale=0.5, p=0.5, seed=SEED, offset=OFFSET)
        assert torch.equal(got[:, columns], want.float())


# ---------------------------------------------------------------------------
# Adam.

def _adam_state(rows, width, cuda, seed=5):
    g = torch.Generator(device="cpu").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return [t.to(cuda) for t in (r(rows, width) * 0.05, r(rows, width) * 1e-3,
                                 torch.rand(rows, width, generator=g) * 3e-6 + 1e-6)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width,p", [(1, 3, 5, 0.0), (500, 70, 48, 0.0), (500, 2000, 45, 0.4),
                                            (5000, 3, 130, 0.2), (0, 4, 6, 0.0)])
def test_consume_against_64_bits(cuda, dtype, n, rows, width, p):
    import embedding

    step, rate = 20, 0.0025
    b1, b2 = 1 - 0.9 ** step, math.sqrt(1 - 0.999 ** step)
    _, index, grad = _case(n, rows, width, dtype, cuda, kind="skewed", padding=n > 1)
    grad = grad * 1e-3
    state = _adam_state(rows, width, cuda)
    t, m, v = [x.double().cpu().numpy() for x in state]
    embedding.consume_torch_adam(*state, grad, index, rate=rate, bias1=b1, bias2_sqrt=b2,
                                 scale=0.7, padding_index=-1, p=p, seed=SEED, offset=OFFSET)
    g, i = grad.double().cpu().numpy() * 0.7, index.cpu().numpy()
    if p > 0:
        g = g * draws.weight(g.shape, p, SEED, OFFSET)
    total, size = np.zeros((rows, width)), np.zeros((rows, width))
    np.add.at(total, i[i >= 0], g[i >= 0])
    np.add.at(size, i[i >= 0], np.abs(g[i >= 0]))
    off = size * (np.bincount(i[i >= 0], minlength=rows)[:, None] + 2.01) * U  # of the gradient
    m1, v1 = 0.9 * m + 0.1 * total, 0.999 * v + 0.001 * total ** 2
    move = rate / b1 / (np.sqrt(v1) / b2 + 1e-15)
    # Moments: the gradient's error through the formula, one rounding each.
    off_m = 0.1 * off + 1.01 * U * np.abs(m1)
    off_v = 0.001 * (2 * np.abs(total) + off) * off + 1.01 * U * v1
    # The step: those, and at most eight roundings of its own (rate / bias1 and
    # the bias correction to float, root, ratio, product, quotient).
    off_t = move * (off_m + (np.abs(m1) + off_m) * (off_v / v1 + 8 * U)) + 1.01 * U * np.abs(t)
    for got, want, limit in zip(state, (t - move * m1, m1, v1), (off_t, off_m, off_v)):
        assert (np.abs(got.double().cpu().numpy() - want) <= limit).all()


def _fused_adam(p, m, v, g, rate, b1, b2):
    """The framework's torch-fused Adam, operation by operation: moments in double
    rounded to float, step size rate / bias1 in float, eps added in double."""
    f, d = np.float32, np.float64
    g = g.astype(d)
    m = (d(0.9) * m.astype(d) + (d(1) - d(0.9)) * g).astype(f)
    v = (d(0.999) * v.astype(d) + ((d(1) - d(0.999)) * g) * g).astype(f)
    denom = ((np.sqrt(v) / f(b2)).astype(d) + d(1e-15)).astype(f)
    return p - (f(rate / d(f(b1))) * m) / denom, m, v


@pytest.mark.parametrize("n,rows,width", [(900, 50, 48), (70, 300, 7), (20_000, 11, 64)])
def test_consume_is_the_frameworks_adam(cuda, n, rows, width):
    """Three steps agree bit for bit with the restated Adam on the gradient that
    lookup_gradient writes."""
    import embedding

    table = _adam_state(rows, width, cuda)[0]
    first, second = torch.zeros_like(table), torch.zeros_like(table)
    want = [t.cpu().numpy() for t in (table, first, second)]
    for step in (1, 2, 3):
        _, index, grad = _case(n, rows, width, torch.float32, cuda, kind="skewed", seed=step)
        g = embedding.lookup_gradient(grad, index, rows, scale=0.3)
        b1 = float(np.float32(1 - 0.9 ** step))
        b2 = float(np.float32(math.sqrt(1 - 0.999 ** step)))
        want = _fused_adam(*want, g.cpu().numpy(), 0.0025, b1, b2)
        embedding.consume_torch_adam(table, first, second, grad, index, rate=0.0025, bias1=b1,
                                     bias2_sqrt=b2, scale=0.3)
        for got, value in zip((table, first, second), want):
            assert np.array_equal(got.cpu().numpy(), value)


# ---------------------------------------------------------------------------
# Autograd, graphs, streams, refusals.

@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(cuda, dtype):
    import embedding

    table, index, grad = _case(700, 90, 48, dtype, cuda, kind="skewed")
    table.requires_grad_(True)
    order = embedding.token_order(index, 90)
    for given in (None, order):
        y = embedding.lookup(table, index, scale=1.5, p=0.2, seed=SEED, offset=OFFSET, order=given)
        (got,) = torch.autograd.grad(y, table, grad)
        _check_gradient(got, grad, index, 90, 1.5, 0.2, dtype)
    (got,) = torch.autograd.grad(embedding.lookup(table, index).sum(), table)
    _check_gradient(got, torch.ones_like(grad), index, 90, 1.0, 0.0, dtype)
    y = embedding.lookup(table, index)
    with pytest.raises(RuntimeError, match="first-order"):
        torch.autograd.grad(y.sum(), table, create_graph=True)
    index.add_(0)  # written after the forward pass
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_gradient_against_differences(cuda):
    """The lookup is linear, so a difference quotient of small integers and
    powers of two is the derivative exactly."""
    import embedding

    index = torch.tensor([0, 2, 2, 1, 2], device=cuda)
    weight = torch.arange(1, 21, device=cuda).float().view(5, 4)
    table = torch.ones(4, 4, device=cuda, requires_grad=True)
    value = lambda t: (embedding.lookup(t, index, scale=2.0, p=0.5, seed=1, offset=2) * weight).sum()
    (got,) = torch.autograd.grad(value(table), table)
    with torch.no_grad():
        for k in range(4):
            for d in range(4):
                moved = table.detach().clone()
                moved[k, d] += 0.5
                assert (value(moved) - value(table)).item() / 0.5 == got[k, d].item()


def test_fused_dropout_is_the_dropout(cuda):
    """Lookup with p is dropout of the lookup (factors whose product is exact)."""
    import dropout
    import embedding

    table, index, _ = _case(999, 50, 77, torch.float32, cuda)
    got = embedding.lookup(table, index, scale=2.0, p=0.5, seed=SEED, offset=OFFSET)
    want = dropout.dropout(embedding.lookup(table, index, scale=2.0), 0.5, SEED, OFFSET)
    assert torch.equal(got, want)


def test_training_step_under_a_graph(cuda):
    """Lookup, dropout and backward captured twice; replays follow new indices and
    a new offset."""
    import embedding

    rows, width, n = 60, 48, 5000
    table, index, grad = _case(n, rows, width, torch.float32, cuda, kind="skewed")
    table.requires_grad_(True)
    offset = torch.zeros(1, dtype=torch.int64, device=cuda)

    def step():
        y = embedding.lookup(table, index, p=0.25, seed=SEED, offset=offset)
        return y.detach(), torch.autograd.grad(y, table, grad)[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        a = step()
    with torch.cuda.graph(second):
        b = step()
    for seed in (1, 2):
        index.copy_(_case(n, rows, width, torch.float32, cuda, kind="skewed", seed=seed)[1])
        offset.fill_(seed * 2 ** 33)
        first.replay()
        second.replay()
        for y, g in (a, b):
            _check_lookup(y, table.detach(), index, 1.0, 0.25, torch.float32, seed * 2 ** 33)
            _check_gradient(g, grad, index, rows, 1.0, 0.25, torch.float32, seed * 2 ** 33)


def test_two_streams_at_once(cuda):
    import embedding

    cases = [_case(20_000, 500, 48, torch.float32, cuda, kind="skewed", seed=s) for s in (0, 1)]
    want = [embedding.lookup_gradient(g, i, 500) for _, i, g in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for stream, (_, i, g) in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(embedding.lookup_gradient(g, i, 500))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_refusals(cuda):
    import embedding

    table, index, grad = _case(10, 4, 6, torch.float32, cuda)
    state = _adam_state(4, 6, cuda)
    order = embedding.token_order(index, 4)
    adam = dict(rate=0.1, bias1=0.5, bias2_sqrt=0.5)
    calls = [
        lambda: embedding.lookup(table.double(), index),
        lambda: embedding.lookup(table.view(2, 2, 6), index),
        lambda: embedding.lookup(table, index.float()),
        lambda: embedding.lookup(table, index.cpu()),
        lambda: embedding.lookup(table, index, scale=float("inf")),
        lambda: embedding.lookup(table, index, p=-1.0),
        lambda: embedding.lookup(table, index, padding_index=1.5),
        lambda: embedding.lookup_gradient(grad, index[:9], 4),
        lambda: embedding.lookup_gradient(grad, index, -1),
        lambda: embedding.lookup_gradient(grad, None, 5, order=order),
        lambda: embedding.lookup_gradient(grad[:9], None, 4, order=order),
        lambda: embedding.lookup_gradient(grad, None, 4, order=order._replace(
            pairs=order.pairs.long())),
        lambda: embedding.lookup_gradient(grad, None, 4, order=order._replace(
            pairs=order.pairs.t().contiguous().t())),
        lambda: embedding.lookup_gradient(grad, None, 4, order=order.pairs),
        lambda: embedding.lookup_gradient(grad.double(), index, 4),
        lambda: embedding.lookup_gradient(grad, index, 4, seed=-1),
        lambda: embedding.consume_torch_adam(*state, grad[:, :5], index, **adam),
        lambda: embedding.consume_torch_adam(state[0], state[1], state[1], grad, index, **adam),
        lambda: embedding.consume_torch_adam(*state[:2], state[2].half(), grad, index, **adam),
        lambda: embedding.consume_torch_adam(*state, grad, index, **{**adam, "bias1": 0.0}),
        lambda: embedding.consume_torch_adam(*state, grad, index, **{**adam, "rate": float("nan")}),
        lambda: embedding.lookup(table.requires_grad_(True), index[:5], order=order),
    ]
    before = [t.clone() for t in state]
    for call in calls:
        with pytest.raises(RuntimeError):
            call()
    assert all(torch.equal(a, b) for a, b in zip(state, before))


def test_lookup_feeds_the_renderer(cuda):
    """Codebook colours as they would be used: lookup, render, backward through
    the renderer, Adam on the codebook; the same numbers as the step with the
    gathered coefficients as leaves."""
    import embedding
    from data_parallel import orbit_camera
    from rasterizer import GaussianRasterizationSettings, GaussianRasterizer

    n, codes = 3000, 40
    rng = np.random.default_rng(3)
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32)).to(cuda)
    means = f(rng.uniform(-1, 1, (n, 3)))
    scales, rotations = f(np.full((n, 3), 0.03)), f(rng.standard_normal((n, 4)))
    rotations = rotations / rotations.norm(dim=1, keepdim=True)
    opacity = f(rng.uniform(0.2, 0.9, (n, 1)))
    camera = orbit_camera(1, 8, width=160, height=120, device=cuda)
    settings = GaussianRasterizationSettings(
        120, 160, camera.tan_x, camera.tan_y, torch.zeros(3, device=cuda), 1.0, camera.view,
        camera.proj, 3, camera.campos, False, False)
    index = torch.from_numpy(rng.integers(0, codes, n)).to(cuda)
    codebook = f(rng.normal(0.0, 0.2, (codes, 48))).requires_grad_(True)
    leaf = codebook.detach()[index].view(n, 16, 3).requires_grad_(True)
    weight = f(rng.standard_normal((3, 120, 160)))

    def image(sh):
        return GaussianRasterizer(settings)(means, torch.zeros_like(means), opacity, shs=sh,
                                            scales=scales, rotations=rotations)[0]

    got = image(embedding.lookup(codebook, index).view(n, 16, 3))
    want = image(leaf)
    assert torch.equal(got, want) and got.abs().sum() > 0
    (g,) = torch.autograd.grad((got * weight).sum(), codebook)
    (h,) = torch.autograd.grad((want * weight).sum(), leaf)
    # The renderer's atomics add in any order: the per-Gaussian adjoints of two
    # runs agree to about n roundings of their size, far below this limit.
    size = torch.zeros_like(g).index_add_(0, index, h.view(n, 48).abs())
    total = torch.zeros_like(g).index_add_(0, index, h.view(n, 48))
    assert (g - total).abs().le(1e-4 * size + 1e-12).all() and g.abs().sum() > 0
    first, second = torch.zeros_like(g), torch.zeros_like(g)
    before = codebook.detach().clone()
    with torch.no_grad():
        embedding.consume_torch_adam(codebook, first, second, h.view(n, 48), index, rate=0.0025,
                                     bias1=0.1, bias2_sqrt=math.sqrt(0.001))
    assert (codebook.detach() - before).abs().max() <= 0.0026 and (first != 0).any()


@pytest.mark.parametrize("dtype,n,rows,width", [(torch.float16, 300, 40_000, 1024),
                                                (torch.float32, 20_000, 131_072, 160),
                                                (torch.bfloat16, 3, 9_000_001, 8)])
def test_large_table_of_which_few_rows_are_named(cuda, dtype, n, rows, width):
    """64 MiB of gradient and more, most rows without a token: an uninitialised
    output is zero everywhere else."""
    import embedding

    _, index, grad = _case(n, 1000, width, dtype, cuda, kind="uniform", padding=True)
    index = torch.where(index >= 0, index * (rows // 1000), index)
    torch.full((rows, width), float("nan"), dtype=dtype, device=cuda)  # what the memory held
    got = embedding.lookup_gradient(grad, index, rows, padding_index=-1)
    named = index[index >= 0].unique()
    few = torch.full((rows,), -1, device=cuda)
    few[named] = torch.arange(len(named), device=cuda)
    _check_gradient(got[named], grad, torch.where(index >= 0, few[index.clamp(min=0)], -1),
                    len(named), 1.0, 0.0, dtype)
    got[named] = 0
    assert not got.any() and not torch.isnan(got).any()


def test_one_token_without_a_dimension(cuda):
    """An index of shape [] gives one row; its gradient is a vector."""
    import embedding

    table = torch.randn(5, 8, device=cuda, requires_grad=True)
    y = embedding.lookup(table, torch.tensor(3, device=cuda), scale=2.0)
    assert y.shape == (8,) and torch.equal(y, 2 * table[3])
    (g,) = torch.autograd.grad(y, table, torch.arange(8.0, device=cuda))
    assert g[3].tolist() == [2.0 * k for k in range(8)] and g.abs().sum() == g[3].sum()


def test_consume_under_two_graphs(cuda):
    """Adam steps captured twice, replayed in turn with new gradients, indices and
    offsets: the same bits as eager calls."""
    import embedding

    n, rows, width = 3000, 70, 48
    offset = torch.zeros(1, dtype=torch.int64, device=cuda)
    _, index, grad = _case(n, rows, width, torch.bfloat16, cuda, kind="skewed")
    how = dict(rate=0.01, bias1=0.5, bias2_sqrt=0.5, p=0.3, seed=SEED, offset=offset)
    captured, eager = _adam_state(rows, width, cuda), _adam_state(rows, width, cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        embedding.consume_torch_adam(*_adam_state(rows, width, cuda), grad, index, **how)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            embedding.consume_torch_adam(*captured, grad, index, **how)
    for step in range(4):
        _, i, g = _case(n, rows, width, torch.bfloat16, cuda, kind="skewed", seed=step)
        index.copy_(i)
        grad.copy_(g)
        offset.fill_(step + 2 ** 40)
        graphs[step % 2].replay()
        embedding.consume_torch_adam(*eager, grad, index, **how)
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_two_host_threads(cuda):
    import threading

    import embedding

    cases = [_case(9000, 300, 45, torch.float32, cuda, kind="skewed", seed=s) for s in range(4)]
    want = [embedding.lookup_gradient(g, i, 300, p=0.1, seed=1) for _, i, g in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = embedding.lookup_gradient(cases[k][2], cases[k][1], 300, p=0.1, seed=1)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[k]):
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width", [(1000, 30, 1001), (5000, 7, 11), (65_537, 4000, 5),
                                          (70_000, 3, 3), (9000, 800, 514)])
def test_odd_rows_through_the_dropout(cuda, dtype, n, rows, width):
    import embedding

    table, index, grad = _case(n, rows, width, dtype, cuda, kind="skewed", bits=32, padding=True)
    how = dict(scale=0.7, padding_index=-1, p=0.35, seed=SEED, offset=OFFSET)
    _check_lookup(embedding.lookup(table, index, **how), table, index, 0.7, 0.35, dtype)
    _check_gradient(embedding.lookup_gradient(grad, index, rows, **how), grad, index, rows, 0.7,
                    0.35, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width", [(1, 1, 1), (2, 3, 4), (63, 9, 48), (64, 200, 45),
                                          (65, 1, 7), (128, 1365, 48), (128, 1366, 48),
                                          (129, 1365, 48), (255, 2, 130), (256, 682, 48),
                                          (256, 683, 48), (257, 682, 48), (3, 1, 65_536),
                                          (3, 1, 65_537)])
@pytest.mark.parametrize("p", [0.0, 0.4])
def test_around_the_border_of_few_tokens(cuda, dtype, n, rows, width, p):
    """Both sides of 256 tokens, 2^16 elements and their product of 2^23; a given
    order gives the same bits as the call's own."""
    import embedding

    for kind, padding in (("same", False), ("skewed", True), ("distinct", False)):
        _, index, grad = _case(n, rows, width, dtype, cuda, kind=kind, bits=32, padding=padding)
        how = dict(scale=-0.6, p=p, seed=SEED, offset=OFFSET)
        got = embedding.lookup_gradient(grad, index, rows, padding_index=-1, **how)
        _check_gradient(got, grad, index, rows, -0.6, p, dtype)
        order = embedding.token_order(index, rows, padding_index=-1)
        assert torch.equal(got, embedding.lookup_gradient(grad, None, rows, order=order, **how))


def test_forked_streams_under_a_graph(cuda):
    """A capture that forks to a second stream and joins right before a call: the
    call's kernels then wait for two predecessors."""
    import dropout
    import embedding

    n, rows, width = 5000, 300, 48
    table, index, grad = _case(n, rows, width, torch.float32, cuda, kind="skewed")
    state = _adam_state(rows, width, cuda)

    def work(side):
        main = torch.cuda.current_stream()
        order = embedding.token_order(index, rows)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            d = dropout.apply(grad, 0.4, 1, 2)
        a = embedding.lookup(table, index)
        main.wait_stream(side)
        g = embedding.lookup_gradient(d, None, rows, order=order)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b = dropout.apply(a, 0.2, 3, 4)
        h = embedding.lookup_gradient(a, index, rows)
        main.wait_stream(side)
        embedding.consume_torch_adam(*state, b, None, order=order, rate=0.01, bias1=0.5,
                                     bias2_sqrt=0.5)
        return g, h, b

    side = torch.cuda.Stream()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        work(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(side)
    for seed in (1, 2):
        t, i, g = _case(n, rows, width, torch.float32, cuda, kind="skewed", seed=seed)
        table.copy_(t)
        index.copy_(i)
        grad.copy_(g)
        before = [x.clone() for x in state]
        graph.replay()
        torch.cuda.synchronize()
        after = [x.clone() for x in state]
        d = dropout.apply(grad, 0.4, 1, 2)
        a = embedding.lookup(table, index)
        b = dropout.apply(a, 0.2, 3, 4)
        assert torch.equal(got[0], embedding.lookup_gradient(d, index, rows))
        assert torch.equal(got[1], embedding.lookup_gradient(a, index, rows))
        assert torch.equal(got[2], b)
        embedding.consume_torch_adam(*before, b, index, rate=0.01, bias1=0.5, bias2_sqrt=0.5)
        assert all(torch.equal(x, y) for x, y in zip(before, after))


def test_threads_sort_by_digits_of_different_widths(cuda):
    """Host threads whose tables need narrow and wide digits of the same sort
    kernels (16000 tokens: one cluster; 70000: many blocks). Every call of every
    thread has to succeed, with the bits of a call alone."""
    import threading

    import embedding

    sizes = [(16_000, 5), (16_000, 131_072), (70_000, 3), (70_000, 131_072)]
    rounds, width = 120, 8
    cases = [_case(n, rows, width, torch.float32, cuda, seed=k) for k, (n, rows) in enumerate(sizes)]

    def call(k, which):
        (_, rows), (_, index, grad) = sizes[k], cases[k]
        if which == 0:
            return [embedding.token_order(index, rows).pairs]
        if which == 1:
            return [embedding.lookup_gradient(grad, index, rows)]
        state = [t.clone() for t in states[k]]
        embedding.consume_torch_adam(*state, grad, index, rate=0.1, bias1=0.5, bias2_sqrt=0.5)
        return state

    states = [_adam_state(rows, width, cuda, seed=k) for k, (_, rows) in enumerate(sizes)]
    want = [[call(k, which) for which in range(3)] for k in range(len(sizes))]
    torch.cuda.synchronize()
    done, wrong, errors = [0] * len(sizes), [], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(rounds):
                    got = call(k, i % 3)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k][i % 3])):
                        wrong.append((k, i))
                    done[k] += 1
        except Exception as e:  # a thread's exception does not fail a test by itself
            errors.append((k, done[k], repr(e)))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong and done == [rounds] * len(sizes)


@pytest.mark.parametrize("n", [16_000, 70_000])
def test_digits_of_different_widths_in_one_graph(cuda, n):
    """A graph that holds the same sort kernel with wide and then with narrow
    digits, instantiated after both."""
    import embedding

    _, wide, _ = _case(n, 131_072, 1, torch.float32, cuda, seed=1)
    _, narrow, _ = _case(n, 3, 1, torch.float32, cuda, seed=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [embedding.token_order(wide, 131_072), embedding.token_order(narrow, 3)]
    for seed in (3, 4):
        wide.copy_(_case(n, 131_072, 1, torch.float32, cuda, seed=seed)[1])
        narrow.copy_(_case(n, 3, 1, torch.float32, cuda, seed=seed)[1])
        graph.replay()
        for index, order in zip((wide, narrow), got):
            i = index.cpu().numpy()
            place = np.argsort(i, kind="stable")
            assert np.array_equal(order.pairs.cpu().numpy(), np.stack([i[place], place], axis=1))


@pytest.mark.parametrize("offset_on_device", [False, True])
def test_forward_mode_derivatives(cuda, offset_on_device):
    """The lookup is linear in the table: a tangent goes through the same lookup,
    in the forward pass and in the gradient's own derivative."""
    import embedding
    from torch.autograd import forward_ad

    table, index, _ = _case(300, 40, 48, torch.float32, cuda, kind="skewed")
    tangent = torch.randn(40, 48, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    offset = torch.full((1,), OFFSET, device=cuda) if offset_on_device else OFFSET
    how = dict(scale=0.5, p=0.25, seed=SEED, offset=offset)
    want, moved = embedding.lookup(table, index, **how), embedding.lookup(tangent, index, **how)
    for grad_needed in (False, True):
        leaf = table.clone().requires_grad_(grad_needed)
        with forward_ad.dual_level():
            y = embedding.lookup(forward_ad.make_dual(leaf, tangent), index, **how)
            value, slope = forward_ad.unpack_dual(y)
            assert torch.equal(value, want) and torch.equal(slope, moved)
            if grad_needed:
                (g,) = torch.autograd.grad((y * y).sum(), leaf)
                g, dg = forward_ad.unpack_dual(g)
                assert torch.equal(g, embedding.lookup_gradient(2 * want, index, 40, **how))
                assert torch.equal(dg, embedding.lookup_gradient(2 * moved, index, 40, **how))
            plain = embedding.lookup(table, index, **how)
            assert torch.equal(plain, want) and forward_ad.unpack_dual(plain).tangent is None


def _sums(terms, index, rows):
    """Sums of terms by row in 64 bits; exact for whole numbers."""
    return torch.zeros(rows, terms.shape[1], dtype=torch.float64, device=terms.device).index_add_(
        0, index, terms)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width,gap", [(300_000, 17, 5, 0), (100_003, 4096, 48, 0),
                                              (65_000, 3, 20, 1), (9000, 3, 513, 0),
                                              (40_000, 700, 64, 8), (20_011, 5, 1, 0)])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_sums_of_whole_numbers_are_exact(cuda, dtype, n, rows, width, gap, p):
    """Whole numbers up to 4 times the factor of 2 or 1: every sum of them and of
    any part is a whole number below 2^24, so 32 bits hold it in any order. One
    token lost, repeated or given to another row shows, however long the row:
    rows in many groups and blocks, aligned, strided and odd, through the
    dropout, to the gradient and to Adam (whose first moment, from zero, is the
    gradient times 1 - 0.9 rounded once)."""
    import embedding

    whole = torch.randint(-4, 5, (n, width + gap), device=cuda,
                          generator=torch.Generator(device=cuda).manual_seed(n)).to(dtype)
    grad = whole[:, :width]
    terms = grad.double()
    if p > 0:
        terms = terms * torch.from_numpy(draws.weight(grad.shape, p, SEED, OFFSET)).to(cuda)
    for kind in ("skewed", "same", "uniform"):
        index = torch.from_numpy(_tokens(kind, n, rows, np.random.default_rng(n))).to(cuda)
        want = _sums(terms, index, rows)
        got = embedding.lookup_gradient(grad, index, rows, p=p, seed=SEED, offset=OFFSET)
        assert torch.equal(got, want.to(dtype))
        table, first, second = (torch.zeros(rows, width, device=cuda) for _ in range(3))
        embedding.consume_torch_adam(table, first, second, grad, index, rate=0.1, bias1=0.5,
                                     bias2_sqrt=0.5, p=p, seed=SEED, offset=OFFSET)
        assert torch.equal(first, ((1.0 - 0.9) * want).float())


@pytest.mark.parametrize("width", [1, 5, 8])
def test_a_row_of_a_million_terms(cuda, width):
    """The error of a long sum of positive terms. A block adds 3584 terms at most
    in 32 bits: t a group (t x groups = 3584 at most), the groups' sums eight at
    a time, their sums in a row; blocks meet in 64 bits. A rounding is off by at
    most 2^-24 of the sum it rounds, so with terms below one the squares of a
    block's errors add up to (2^-24)^2 times at most 3584 t^2 + groups (8 t)^2 +
    groups / 8 x 3584^2, below 29000^2 for 8 to 256 groups. Roundings of terms
    that know nothing of each other are as good as independent: six times the
    root of the squares' sum over all blocks is passed with a probability of
    2 exp(-18) (Hoeffding). The result's own rounding comes on top."""
    import embedding

    n = 1_100_000
    grad = torch.rand(n, width, device=cuda,
                      generator=torch.Generator(device=cuda).manual_seed(width)) / 2 + 0.5
    got = embedding.lookup_gradient(grad, torch.zeros(n, dtype=torch.int32, device=cuda), 1)
    want = grad.double().sum(0, keepdim=True)
    blocks = -(-n // 3584)
    assert ((got - want).abs() <= 6 * math.sqrt(blocks) * 29_000 * U + want * U).all()


def test_bad_indices_are_seen_behind_work_on_another_stream(cuda):
    """Reading the fault word waits for the device, also for streams that do not
    wait for the legacy one; all three types and every operator report there."""
    import _native as native
    import embedding

    native.fault_status()
    side = torch.cuda.Stream()
    bad = torch.full((300,), 9, device=cuda)
    for dtype in TYPES:
        table = torch.ones(4, 8, dtype=dtype, device=cuda)
        grad = torch.ones(300, 8, dtype=dtype, device=cuda)
        state = _adam_state(4, 8, cuda)
        for call in (lambda: embedding.lookup(table, bad),
                     lambda: embedding.lookup_gradient(grad, bad, 4),
                     lambda: embedding.lookup_gradient(grad[:20], bad[:20], 4),
                     lambda: embedding.token_order(bad, 4),
                     lambda: embedding.consume_torch_adam(*state, grad, bad, rate=0.1, bias1=0.5,
                                                          bias2_sqrt=0.5)):
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                torch.cuda._sleep(20_000_000)  # about 10 ms
                call()
            assert native.fault_status() == 256 and native.fault_status() == 0


def test_first_call_of_a_process_under_capture(cuda):
    """A process whose first call of the library is captured into a graph."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
import _native as native
import embedding
table = torch.arange(32.0, device="cuda").view(8, 4)
index = torch.tensor([3, 9, 7], device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = embedding.lookup(table, index)
    g = embedding.lookup_gradient(y, index, 8)
graph.replay()
torch.cuda.synchronize()
assert y.tolist() == [table[3].tolist(), [0.0] * 4, table[7].tolist()]
assert g[3].tolist() == table[3].tolist() and g[7].tolist() == table[7].tolist()
assert native.fault_status() == 256
"""
    package = Path(__file__).resolve().parents[1] / "clad-3dgs_b200"
    run = subprocess.run([sys.executable, "-c", code, str(package)], capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


def test_reading_the_fault_word_clears_it_or_leaves_it(cuda):
    """One word for all operators: without `clear` its bits stay for the next
    reader, and the status says what it holds."""
    import ctypes

    import _native as native
    import embedding

    native.fault_status()
    word = ctypes.c_uint(7)
    status = lambda clear: native.library().clad3dgs_fault_status(clear, ctypes.byref(word))
    assert status(0) == native.OK and word.value == 0
    table, bad = torch.ones(4, 8, dtype=torch.float16, device=cuda), torch.full((3,), 4, device=cuda)
    embedding.lookup(table, bad)
    embedding.lookup_gradient(table[:3], bad, 4)
    for clear in (0, 0, 1):
        assert status(clear) == native.DEVICE_FAULT and word.value == 256
        assert b"index" in native.library().clad3dgs_last_error()
    assert status(1) == native.OK and word.value == 0


def test_what_only_the_library_could_refuse_is_a_runtime_error(cuda):
    """Factors and bias corrections that do not fit 32 bits, and tables and
    indices that are none."""
    import embedding

    table, index, grad = _case(10, 4, 6, torch.float32, cuda)
    state = _adam_state(4, 6, cuda)
    adam = dict(rate=0.1, bias1=0.5, bias2_sqrt=0.5)
    before = [t.clone() for t in state]
    leaf = torch.ones((), device=cuda, requires_grad=True)
    for call in (lambda: embedding.lookup(table, index, scale=1e38, p=0.999),
                 lambda: embedding.lookup(table, index, scale=1e39),
                 lambda: embedding.lookup_gradient(grad, index, 4, scale=-1e38, p=0.999),
                 lambda: embedding.consume_torch_adam(*state, grad, index, **adam, scale=1e38,
                                                      p=0.999),
                 lambda: embedding.consume_torch_adam(*state, grad, index, **{**adam, "bias1": 1e-50}),
                 lambda: embedding.consume_torch_adam(*state, grad, index,
                                                      **{**adam, "bias2_sqrt": 1e-50}),
                 lambda: embedding.lookup_gradient(grad, None, 4),
                 lambda: embedding.lookup(table, [0, 1]),
                 lambda: embedding.lookup(table.clone().requires_grad_(True), [0, 1]),
                 lambda: embedding.lookup(table.clone().requires_grad_(True), None,
                                          order=embedding.token_order(index, 4)),
                 lambda: embedding.lookup(leaf, index),
                 lambda: embedding.lookup(leaf.detach(), index),
                 lambda: embedding.lookup(leaf, index, order=embedding.token_order(index, 4))):
        with pytest.raises(RuntimeError):
            call()
    assert all(torch.equal(a, b) for a, b in zip(state, before))
    # A factor near the largest number is none of them.
    assert torch.isfinite(embedding.lookup(torch.full((4, 6), 0.5, device=cuda), index,
                                           scale=1e38, p=0.5)).all()


@pytest.mark.parametrize("n,rows", [(3000, 300_000), (40_000, 300_000), (40_000, 2000)])
def test_sorts_back_to_back(cuda, n, rows):
    """Passes and calls that overwrite the same memory one after the other, all in
    flight at once: every call sees its own passes' counts and pairs, and every
    update the sums of its own step."""
    import embedding

    g = torch.Generator(device=cuda).manual_seed(n)
    indices = [torch.randint(0, rows, (n,), device=cuda, generator=g) for _ in range(60)]
    grads = [torch.randint(-4, 5, (n, 4), device=cuda, generator=g).float() for _ in indices]
    torch.cuda.synchronize()
    first = torch.zeros(rows, 4, device=cuda)
    state = torch.zeros_like(first), first, torch.zeros_like(first)
    orders, firsts = [], []
    for index, grad in zip(indices, grads):
        orders.append(embedding.token_order(index, rows).pairs)
        first.zero_()
        embedding.consume_torch_adam(*state, grad, index, rate=0.1, bias1=0.5, bias2_sqrt=0.5)
        firsts.append(first[:2000].clone())
    for index, grad, order, moment in zip(indices, grads, orders, firsts):
        row, place = torch.sort(index, stable=True)
        assert torch.equal(order.long(), torch.stack([row, place], dim=1))
        want = _sums(grad.double(), index, rows)[:2000]
        assert torch.equal(moment, ((1.0 - 0.9) * want).float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_rows_wider_than_the_gpu_has_places(cuda, dtype, p):
    """More slices of columns than blocks that run at once: whole numbers, exact."""
    import embedding

    n, rows = 130, 3
    for width in (300_000, 300_001):
        grad = torch.randint(-4, 5, (n, width), device=cuda,
                             generator=torch.Generator(device=cuda).manual_seed(n)).to(dtype)
        index = torch.randint(0, rows, (n,), device=cuda,
                              generator=torch.Generator(device=cuda).manual_seed(1))
        got = embedding.lookup_gradient(grad, index, rows, p=p, seed=SEED, offset=OFFSET)
        terms = grad.double()
        if p > 0:
            ones = embedding.lookup(torch.ones(1, width, device=cuda), torch.zeros_like(index), p=p,
                                    seed=SEED, offset=OFFSET)
            kept = draws.keep(129 * width + np.arange(width - 1000, width), p, SEED, OFFSET)
            assert np.array_equal(ones[129, -1000:].cpu().numpy(), kept / (1 - p))
            terms = terms * ones
        assert torch.equal(got, _sums(terms, index, rows).to(dtype))


@pytest.mark.parametrize("n,borders", [(300, (65_536,)), (2000, (98_304,)),
                                       (8000, (294_912,)), (70_000, (1_179_648,))])
def test_slots_cleared_by_the_sort_or_before_it(cuda, n, borders):
    """Adam's slots on both sides of where a launch of their own clears them, over
    memory that is not zero: rows without tokens get no gradient."""
    import embedding

    for rows in [r + more for r in borders for more in (0, 1)]:
        index = torch.randint(0, rows, (n,), device=cuda,
                              generator=torch.Generator(device=cuda).manual_seed(rows))
        grad = torch.randint(1, 5, (n, 4), device=cuda,
                             generator=torch.Generator(device=cuda).manual_seed(n)).float()
        table, first, second = (torch.zeros(rows, 4, device=cuda) for _ in range(3))
        torch.full((rows * 8 + n * 64,), 1.0, device=cuda)  # what the workspace held
        embedding.consume_torch_adam(table, first, second, grad, index, rate=0.1, bias1=0.5,
                                     bias2_sqrt=0.5)
        assert torch.equal(first, ((1.0 - 0.9) * _sums(grad.double(), index, rows)).float())


def test_an_order_written_before_the_backward_is_refused(cuda):
    """As an index written after the forward pass is; an order of inference mode
    has no version and is taken as it is."""
    import embedding

    table, index, grad = _case(700, 90, 48, torch.float32, cuda)
    table.requires_grad_(True)
    want = embedding.lookup_gradient(grad, index, 90)
    with torch.inference_mode():
        order = embedding.token_order(index, 90)
    (got,) = torch.autograd.grad(embedding.lookup(table, index, order=order), table, grad)
    assert torch.equal(got, want)
    order = embedding.token_order(index, 90)
    y = embedding.lookup(table, index, order=order)
    order.pairs.copy_(embedding.token_order(index.flip(0).contiguous(), 90).pairs)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, table, grad)
