"""Table operators on the CPU: refusals of the Python and C entries (before any
launch) and the workspace sizes."""

import pytest
import torch


def test_entries_refuse_cpu_tensors():
    import embedding

    table, index = torch.ones(4, 3), torch.zeros(5, dtype=torch.int64)
    for call in (lambda: embedding.lookup(table, index),
                 lambda: embedding.token_order(index, 4),
                 lambda: embedding.lookup_gradient(torch.ones(5, 3), index, 4),
                 lambda: embedding.consume_torch_adam(table, table.clone(), table.clone(),
                                                      torch.ones(5, 3), index, rate=0.1,
                                                      bias1=0.5, bias2_sqrt=0.5)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


ORDER = dict(n=200_000, rows=4, index=256, index_bits=64, has_padding=0, padding=0, order=512,
             workspace=1024, workspace_bytes=1 << 20, stream=0)
LOOKUP = dict(type=0, n=10, rows=4, width=8, table=256, table_stride=8, index=512, index_bits=64,
              has_padding=0, padding=0, scale=1.0, p=0.0, seed=0, offset=0, offset_device=None,
              out=1024, stream=0)
GRADIENT = dict(type=0, n=1000, rows=4, width=8, grad=256, grad_stride=8, index=None, index_bits=0,
                has_padding=0, padding=0, order=512, scale=1.0, p=0.0, seed=0, offset=0,
                offset_device=None, out=1024, workspace=2048, workspace_bytes=1 << 20, stream=0)
NAN, INF = float("nan"), float("inf")


def _adam():
    import _native as native

    a = {k: v for k, v in GRADIENT.items() if k not in ("out", "workspace", "workspace_bytes",
                                                        "stream")}
    a.update(table=4096, first=8192, second=16384, rate=0.1, config=native.TorchAdamConfig(0.5, 0.5),
             workspace=2048, workspace_bytes=1 << 20, stream=0)
    return a


SHARED = [dict(n=-1), dict(rows=-1), dict(n=2 ** 31), dict(rows=2 ** 31)]
SIZED = SHARED + [dict(width=-1), dict(type=3), dict(type=-1), dict(scale=INF), dict(scale=NAN), dict(scale=1e39), dict(scale=1e38, p=0.999),
                  dict(p=-0.5), dict(p=1.5), dict(p=NAN), dict(n=2 ** 30, width=2 ** 40)]
SUMS = SIZED + [dict(grad=None), dict(order=None), dict(workspace=None), dict(workspace_bytes=8),
                dict(grad_stride=-1), dict(workspace=2064), dict(order=516),
                dict(order=None, index=256, index_bits=16),
                dict(order=None, index=256, index_bits=64, workspace_bytes=300)]


@pytest.mark.parametrize("entry,change", (
    [("token_order", c) for c in SHARED + [dict(index=None), dict(order=None), dict(workspace=None),
                                           dict(workspace_bytes=8), dict(index_bits=16),
                                           dict(workspace=1040), dict(order=516)]]
    + [("embedding_lookup", c) for c in SIZED + [dict(table=None), dict(index=None), dict(out=None),
                                                 dict(index_bits=0), dict(table_stride=-1)]]
    + [("embedding_gradient", c) for c in SUMS + [dict(out=None)]]
    + [("embedding_consume_torch_adam", c) for c in SUMS + [
        dict(table=None), dict(first=None), dict(second=None), dict(rate=NAN), dict(rate=-1.0)]]))
def test_c_entries_refuse_bad_arguments(entry, change):
    """Refused on the host: these run without a GPU, so nothing is launched."""
    import _native as native

    base = {"token_order": ORDER, "embedding_lookup": LOOKUP, "embedding_gradient": GRADIENT}
    a = dict(base.get(entry) or _adam())
    assert set(change) <= set(a)
    a.update(change)
    lib = native.library()
    assert getattr(lib, "clad3dgs_" + entry)(*a.values()) == native.INVALID_ARGUMENT
    assert lib.clad3dgs_last_error()


@pytest.mark.parametrize("bias1,bias2", [(0.0, 0.5), (0.5, 0.0), (1.5, 0.5), (0.5, NAN)])
def test_c_entry_refuses_bad_bias_corrections(bias1, bias2):
    import _native as native

    a = _adam()
    a["config"] = native.TorchAdamConfig(bias1, bias2)
    assert (native.library().clad3dgs_embedding_consume_torch_adam(*a.values())
            == native.INVALID_ARGUMENT)


def test_nothing_to_do_needs_no_arrays():
    import _native as native

    lib = native.library()
    assert lib.clad3dgs_token_order(*{**ORDER, "n": 0, "index": None, "order": None,
                                      "workspace": None}.values()) == native.OK
    for change in (dict(n=0), dict(width=0)):
        assert lib.clad3dgs_embedding_lookup(*{**LOOKUP, **change, "table": None, "index": None,
                                               "out": None}.values()) == native.OK
    for change in (dict(rows=0), dict(width=0)):
        assert lib.clad3dgs_embedding_gradient(*{**GRADIENT, **change, "grad": None, "out": None,
                                                 "workspace": None}.values()) == native.OK


def test_workspaces():
    import _native as native

    lib = native.library()
    assert lib.clad3dgs_token_order_workspace(0, 5) == 0
    assert lib.clad3dgs_token_order_workspace(2 ** 31, 5) == 0
    assert lib.clad3dgs_embedding_workspace(0, 5, 5, 0, 1) == 0
    assert lib.clad3dgs_embedding_workspace(5, -1, 5, 0, 1) == 0
    assert lib.clad3dgs_embedding_workspace(2 ** 31, 5, 5, 1, 1) == 0
    sizes = [lib.clad3dgs_token_order_workspace(n, 4096) for n in (1, 10_000, 70_000, 1_000_000)]
    assert sizes == sorted(sizes) and sizes[2] > 0  # few tokens need none
    assert (lib.clad3dgs_embedding_workspace(70_000, 5, 5, 0, 0)
            >= lib.clad3dgs_embedding_workspace(70_000, 5, 5, 0, 1) + 8 * 70_000)
    few, many = (lib.clad3dgs_embedding_workspace(n, 4096, 48, 0, 1) for n in (1000, 1_000_000))
    assert 0 < few < many
    assert lib.clad3dgs_embedding_workspace(1000, 4096, 48, 1, 1) >= few + 4 * 4096 + 1000 * 48 * 4
    # Few tokens and a small table need none; a large table does.
    sizes = [lib.clad3dgs_embedding_workspace(n, rows, 48, 1, 0) > 0
             for n, rows in ((128, 1365), (128, 1366), (256, 682), (256, 683), (257, 1))]
    assert sizes == [False, True, False, True, True]


@pytest.mark.parametrize("scale,p,fits", [
    (1.0, 0.0, True), (-2, 0.5, True), (1e38, 0.5, True), (1e38, 1, True), (1e38, 1.0, True),
    (0.0, 1.0 - 1e-15, True), (1e38, 0.999, False), (-1e38, 0.999, False), (1e39, 0.0, False),
    (10 ** 400, 0.0, False), (INF, 0.0, False), (NAN, 0.0, False), (NAN, 1.0, False),
    ("1", 0.0, False), (None, 0.0, False)])
def test_scales_are_checked(scale, p, fits):
    import embedding

    if fits:
        embedding._check_scale(scale, p)
    else:
        with pytest.raises(RuntimeError, match="scale"):
            embedding._check_scale(scale, p)


def test_an_index_has_to_be_a_tensor():
    import embedding

    for index in (None, [0, 1]):
        with pytest.raises(RuntimeError, match="index"):
            embedding.token_order(index, 4)
