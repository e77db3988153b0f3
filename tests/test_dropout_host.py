"""Dropout on the CPU: the tests' generator against published vectors, the
refusals of the Python entries and of the C entry (before any launch)."""

import numpy as np
import pytest
import torch

import draws


@pytest.mark.parametrize("counter,key,words", [
    # Known answers published with the generator.
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_gives_the_published_words(counter, key, words):
    got = draws.philox([np.array([c]) for c in counter], key)
    assert tuple(int(w[0]) for w in got) == words


def test_share_of_dropped_elements():
    # 2^16 independent draws: standard deviation of the share is below 0.002.
    for p in (0.1, 0.5, 0.9):
        kept = draws.keep(np.arange(1 << 16), p, 7, 3)
        assert abs(kept.mean() - (1 - p)) < 0.01


def test_entries_refuse_cpu_tensors():
    import dropout

    with pytest.raises(RuntimeError, match="CUDA"):
        dropout.dropout(torch.ones(4), 0.5, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        dropout.apply(torch.ones(4, requires_grad=True), 0.5, 1)


@pytest.mark.parametrize("p,seed,offset,message", [
    (-0.1, 1, 0, "p must"), (1.5, 1, 0, "p must"), (float("nan"), 1, 0, "p must"),
    ("a", 1, 0, "p must"), (0.5, -1, 0, "seed"), (0.5, 2 ** 64, 0, "seed"), (0.5, 1.0, 0, "seed"),
    (0.5, 1, -1, "offset"), (0.5, 1, 2 ** 64, "offset"), (0.5, 1, 0.5, "offset"),
    (0.5, 1, torch.zeros(2, dtype=torch.int64), "one int64"),
    (0.5, 1, torch.zeros(1, dtype=torch.int32), "one int64"),
])
def test_draw_numbers_are_checked(p, seed, offset, message):
    import dropout

    with pytest.raises(RuntimeError, match=message):
        dropout.check_draw(p, seed, offset, torch.device("cpu"))


def test_rows_of_layouts():
    import dropout

    x = torch.zeros(6, 8)
    assert dropout.row_layout(x)[1:] == (6, 8, 8)
    assert dropout.row_layout(x.view(2, 3, 8))[1:] == (6, 8, 8)
    assert dropout.row_layout(x[:, :5])[1:] == (6, 5, 8)
    assert dropout.row_layout(x.t())[1:] == (8, 6, 6)  # packed
    assert dropout.row_layout(torch.zeros(()))[1:] == (1, 1, 1)
    assert dropout.row_layout(torch.zeros(0, 8))[1] == 0
    assert dropout.row_layout(x[:1].expand(4, 8))[1:] == (4, 8, 0)


def _call(lib, **change):
    a = dict(type=0, rows=4, width=4, x=64, x_stride=4, y=1 << 20, y_stride=4, p=0.5, seed=1,
             offset=0, offset_device=None, by_row=0, stream=0)
    a.update(change)
    return lib.clad3dgs_dropout(*a.values())


@pytest.mark.parametrize("change", [
    dict(type=3), dict(type=-1), dict(rows=-1), dict(width=-1), dict(p=2.0), dict(p=float("nan")),
    dict(x=None), dict(y=None), dict(x_stride=-4), dict(y_stride=3), dict(rows=2 ** 62),
])
def test_c_entry_refuses_bad_arguments(change):
    """Refused on the host: these run without a GPU, so nothing is launched."""
    import _native as native

    lib = native.library()
    assert _call(lib, **change) == native.INVALID_ARGUMENT
    assert lib.clad3dgs_last_error().startswith(b"dropout")
    assert _call(lib, rows=0, x=None, y=None) == native.OK
