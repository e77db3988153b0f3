"""Dropout on the GPU against the definition in 64 bits: decisions exactly,
values within the roundings that one product and one conversion make."""

import numpy as np
import pytest
import torch

import draws

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
SEED = 0x1234567_89ABCDEF


def _input(shape, dtype, cuda, seed=0):
    rng = np.random.default_rng(seed)
    return torch.from_numpy(rng.standard_normal(shape)).to(dtype).to(cuda)


def _close(got, x, weight, dtype):
    """The factor 1/(1-p) and the product are rounded to 32 bits (2 x 2^-24 in
    all), then the result to its type (half a step; 2^-25 below fp16's normal
    range)."""
    want = x.double().cpu().numpy() * weight
    limit = np.abs(want) * (2.01 * 2.0 ** -24)
    if dtype != torch.float32:
        limit += np.abs(want) * torch.finfo(dtype).eps / 2 + 2.0 ** -25
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert np.array_equal(got == 0, want == 0)
    assert (np.abs(got - want) <= limit).all(), np.abs(got - want).max()


SHAPES = [(1,), (3,), (4, 1), (5, 3), (1, 2048), (257, 33), (2, 3, 7), (64, 128), (1000, 48),
          (3, 8191), (4097, 17), (100_003,)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("rows", [False, True])
def test_values_and_decisions(cuda, dtype, shape, rows):
    import dropout

    x = _input(shape, dtype, cuda)
    for p, offset in ((0.1, 5), (0.75, 2 ** 40 + 3)):
        y = dropout.dropout(x, p, SEED, offset, rows=rows)
        assert y.dtype == dtype and y.shape == x.shape
        _close(y, x, draws.weight(x.shape, p, SEED, offset, rows), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [False, True])
def test_layouts_draw_alike(cuda, dtype, rows):
    """Strided, unaligned, expanded and transposed inputs give what their packed
    copies give."""
    import dropout

    base = _input((40, 70), dtype, cuda)
    flat = _input((4001,), dtype, cuda)
    for x in (base[:, :64], base[:, 3:], base.t(), base[:, ::2], flat[1:], flat[3:1027],
              base[:1].expand(9, 70), base.view(4, 10, 70)[:, :, 1:9], base[5], base[3, 4]):
        y = dropout.dropout(x, 0.4, 99, 7, rows=rows)
        assert y.is_contiguous()
        assert torch.equal(y, dropout.dropout(x.contiguous().clone(), 0.4, 99, 7, rows=rows))
        _close(y, x, draws.weight(x.shape if x.dim() else (1,), 0.4, 99, 7, rows)
               .reshape(x.shape), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_edges_of_p(cuda, dtype):
    import dropout

    x = _input((123, 45), dtype, cuda)
    assert torch.equal(dropout.dropout(x, 0.0, 1, 2), x)
    x[0, 0], x[1, 1], x[2, 2] = float("inf"), float("nan"), -float("inf")
    for rows in (False, True):
        assert not dropout.dropout(x, 1.0, 1, 2, rows=rows).any()
    kept = torch.from_numpy(draws.keep(np.arange(x.numel()), 0.5, 1, 2).reshape(x.shape)).to(cuda)
    y = dropout.dropout(x, 0.5, 1, 2)
    assert torch.equal(y == 0, ~kept | (x == 0))  # dropped infinities and NaN give zero
    assert torch.equal(torch.isnan(y), torch.isnan(x) & kept)
    for empty in ((0,), (0, 5), (5, 0)):
        assert dropout.dropout(torch.empty(empty, dtype=dtype, device=cuda), 0.5, 1).shape == empty


def test_far_elements_and_large_numbers(cuda):
    """Element numbers and offsets past 32 bits: a row stride of zero makes a
    small array stand for one whose elements pass 2^32."""
    import dropout

    width = 2 ** 20
    x = torch.ones(1, width, dtype=torch.float16, device=cuda).expand(4100, width)
    y = dropout.dropout(x, 0.5, 2 ** 63 + 11, 2 ** 64 - 1)
    for row in (0, 1, 4095, 4096, 4099):
        kept = draws.keep(row * width + np.arange(1000), 0.5, 2 ** 63 + 11, 2 ** 64 - 1)
        assert np.array_equal(y[row, :1000].cpu().numpy() > 0, kept), row
    # The packed result once more, in place under another offset.
    before = y[4099, :1000].clone()
    dropout.apply(y, 0.5, 5, 6, out=y)
    kept = draws.keep(4099 * width + np.arange(1000), 0.5, 5, 6)
    assert np.array_equal(y[4099, :1000].cpu().numpy(), before.cpu().numpy() * kept * 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [False, True])
def test_gradient_is_the_same_map(cuda, dtype, rows):
    import dropout

    x = _input((301, 19), dtype, cuda).requires_grad_(True)
    g = _input((301, 19), dtype, cuda, seed=1)
    y = dropout.dropout(x, 0.3, 5, 6, rows=rows)
    (dx,) = torch.autograd.grad(y, x, g)
    _close(dx, g, draws.weight(g.shape, 0.3, 5, 6, rows), dtype)
    # A broadcast gradient (strides of zero) and a strided one.
    (dx,) = torch.autograd.grad(dropout.dropout(x, 0.3, 5, 6, rows=rows).sum(), x)
    _close(dx, torch.ones_like(x).detach(), draws.weight(g.shape, 0.3, 5, 6, rows), dtype)


def test_gradient_against_differences(cuda):
    """The map is linear in x, so a difference quotient is the derivative up to
    its roundings: with x and the step powers of two both are exact."""
    import dropout

    x = torch.ones(64, device=cuda, requires_grad=True)
    y = dropout.dropout(x, 0.5, 3, 4)
    (dx,) = torch.autograd.grad(y.sum(), x)
    for i in range(64):
        moved = torch.ones(64, device=cuda)
        moved[i] += 0.5
        quotient = (dropout.dropout(moved, 0.5, 3, 4) - y.detach()).sum() / 0.5
        assert quotient.item() == dx[i].item()


def test_second_derivative_runs(cuda):
    import dropout

    x = torch.ones(32, device=cuda, requires_grad=True)
    y = dropout.dropout(x * x, 0.5, 3, 4)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    (ddx,) = torch.autograd.grad(dx.sum(), x)
    kept = draws.weight((32,), 0.5, 3, 4)
    assert np.allclose(ddx.cpu().numpy(), 2 * kept)


def test_in_place_and_into(cuda):
    import dropout

    x = _input((77, 13), torch.float32, cuda)
    want = dropout.apply(x, 0.2, 1, 1)
    out = torch.full_like(x, 9.0)
    assert dropout.apply(x, 0.2, 1, 1, out=out) is out
    assert torch.equal(out, want)
    dropout.apply(x, 0.2, 1, 1, out=x)
    assert torch.equal(x, want)


def test_refusals(cuda):
    import dropout

    x = torch.ones(8, 8, device=cuda)
    for call in (lambda: dropout.dropout(x.double(), 0.5, 1),
                 lambda: dropout.dropout(x, 2.0, 1),
                 lambda: dropout.dropout(x, 0.5, 1, torch.zeros(1, dtype=torch.int64)),
                 lambda: dropout.apply(x, 0.5, 1, out=x.t()),
                 lambda: dropout.apply(x, 0.5, 1, out=torch.empty(8, 7, device=cuda)),
                 lambda: dropout.apply(x.view(-1)[:32], 0.5, 1, out=x.view(-1)[16:48]),
                 lambda: dropout.apply(x.half(), 0.5, 1, out=x)):
        with pytest.raises(RuntimeError):
            call()
    assert torch.equal(x, torch.ones(8, 8, device=cuda))


def test_offset_on_the_device_under_a_graph(cuda):
    """A captured forward and backward draw anew at each replay."""
    import dropout

    x = _input((50, 21), torch.float32, cuda).requires_grad_(True)
    g = _input((50, 21), torch.float32, cuda, seed=1)
    offset = torch.zeros(1, dtype=torch.int64, device=cuda)

    def step():
        y = dropout.dropout(x, 0.5, 8, offset)
        (dx,) = torch.autograd.grad(y, x, g)
        return y.detach(), dx

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    for number in (0, 1, 2 ** 33 + 5):
        offset.fill_(number)
        graph.replay()
        weight = draws.weight(x.shape, 0.5, 8, number)
        _close(y, x.detach(), weight, torch.float32)
        _close(dx, g, weight, torch.float32)


def test_offset_changed_before_the_backward_is_refused(cuda):
    import dropout

    x = torch.ones(16, device=cuda, requires_grad=True)
    offset = torch.zeros(1, dtype=torch.int64, device=cuda)
    y = dropout.dropout(x, 0.5, 8, offset)
    offset.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_other_stream(cuda):
    import dropout

    x = _input((1000, 100), torch.float32, cuda)
    want = dropout.dropout(x, 0.5, 8, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dropout.dropout(x, 0.5, 8, 9)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("offset_on_device", [False, True])
@pytest.mark.parametrize("rows", [False, True])
def test_forward_mode_derivatives(cuda, rows, offset_on_device):
    """The map is linear: a tangent goes through the same draw, in the forward
    pass and in the gradient's own derivative."""
    import dropout
    from torch.autograd import forward_ad

    x, tangent = _input((60, 33), torch.float32, cuda), _input((60, 33), torch.float32, cuda, seed=1)
    offset = torch.full((1,), 7, device=cuda) if offset_on_device else 7
    drop = lambda v: dropout.dropout(v, 0.5, 3, offset, rows=rows)
    want, moved = drop(x), drop(tangent)
    for grad_needed in (False, True):
        leaf = x.clone().requires_grad_(grad_needed)
        with forward_ad.dual_level():
            y = drop(forward_ad.make_dual(leaf, tangent))
            value, slope = forward_ad.unpack_dual(y)
            assert torch.equal(value, want) and torch.equal(slope, moved)
            if grad_needed:
                (g,) = torch.autograd.grad((y * y).sum(), leaf)
                g, dg = forward_ad.unpack_dual(g)
                assert torch.equal(g, drop(2 * want)) and torch.equal(dg, drop(2 * moved))
            assert forward_ad.unpack_dual(drop(x)).tangent is None


def test_writing_into_a_saved_tensor_is_seen_by_autograd(cuda):
    """`out` is written in place: a backward pass that needs its old values is
    refused, as after torch's own operations in place."""
    import dropout

    for place in (lambda x: dropout.apply(x, 0.5, 1, 2, out=x),
                  lambda x: dropout.apply(torch.ones_like(x), 0.5, 1, 2, out=x)):
        w = torch.ones(16, device=cuda, requires_grad=True)
        x = torch.full((16,), 3.0, device=cuda)
        y = (w * x).sum()
        place(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_writing_into_an_inference_tensor(cuda):
    import dropout

    x = _input((9, 5), torch.float32, cuda)
    with torch.inference_mode():
        out = torch.empty(9, 5, device=cuda)
        assert torch.equal(dropout.apply(x, 0.5, 1, 2, out=out), dropout.apply(x, 0.5, 1, 2))
        dropout.apply(x, 0.5, 1, 2, out=x)
        assert torch.equal(x, out)
