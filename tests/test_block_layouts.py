"""How the operators around a block read a tensor as rows with one distance between them, without a GPU: whatever the strides, row r of what they read is row r of
the tensor."""

import itertools

import pytest
import torch


def _read(t):
    """The rows that a kernel would read, by address in the tensor's own memory, and whether they are a copy's."""
    from viola_amd import _lib
    count, pitch, copied = _lib.host().row_layout(t)
    if copied:
        return None, count, pitch
    storage = torch.as_strided(t, (t.untyped_storage().size() // t.element_size() - t.storage_offset(),), (1,), t.storage_offset())
    assert (count - 1) * pitch + t.shape[-1] <= storage.numel(), "reads beyond the tensor's memory"
    return torch.as_strided(t, (count, t.shape[-1]), (pitch, 1), t.storage_offset()), count, pitch


def _holds(t):
    rows, count, pitch = _read(t)
    assert count == t.numel() // t.shape[-1]
    if rows is None:
        assert pitch == t.shape[-1]                                          # a copy is contiguous
    else:
        assert torch.equal(rows, t.reshape(-1, t.shape[-1]))
    return rows is not None


def test_broadcast_dimensions_are_copied():
    """A dimension of stride 0 inside another one: rows repeat, so they have no common distance."""
    row = torch.arange(4 * 256.0).view(4, 1, 256)
    assert not _holds(row.expand(4, 9, 256))
    assert not _holds(torch.arange(256.0).expand(4, 9, 256))
    assert not _holds(torch.arange(9 * 256.0).view(1, 9, 256).expand(4, 9, 256))
    assert not _holds(torch.arange(4 * 8.0).view(4, 1, 1, 8).expand(4, 3, 5, 8))
    assert not _holds(torch.arange(4 * 3 * 8.0).view(4, 3, 1, 8).expand(4, 3, 5, 8))
    assert not _holds(torch.arange(5.0).view(5, 1).expand(5, 8))
    assert not _holds(torch.arange(5.0).view(5, 1, 1).expand(5, 3, 1))
    y = torch.zeros(4, 9, 256, requires_grad=True)                           # the gradient of a sum over tokens
    (y * 1.0).register_hook(lambda g: None)
    seen = []
    z = y * 1.0
    z.register_hook(lambda g: seen.append(g))
    (z.sum(1) * torch.arange(4 * 256.0).view(4, 256)).sum().backward()
    assert seen[0].stride() == (256, 0, 1) and not _holds(seen[0])


def test_rows_of_one_distance_are_read_where_they_are():
    wide = torch.arange(4 * 9 * 40.0).view(4, 9, 40)
    for t in (wide, wide[..., 8:24], wide[..., 3:20], wide[:, :1], wide[1:2], wide[:1, :1], wide[0], wide[0, 0], wide[::2, :1, :7], wide[:, 4, 1:9], wide[:, :, :1]):
        assert _holds(t), (t.shape, t.stride())
    for t in (wide.transpose(0, 1), wide.transpose(1, 2), wide[:, :5], wide[:, ::2], wide[..., ::2], torch.as_strided(wide, (30, 16), (8, 1))):
        assert not _holds(t), (t.shape, t.stride())


@pytest.mark.parametrize("sizes", [(1,), (7,), (3, 5), (1, 5), (2, 3, 4), (2, 1, 4), (1, 3, 1), (2, 3, 2, 5)])
def test_any_strides(sizes):
    """Every combination of a few strides, overlapping ones among them."""
    memory = torch.arange(4000.0)
    for strides in itertools.product((0, 1, 2, 4, 5, 8, 20, 60), repeat=len(sizes)):
        _holds(torch.as_strided(memory, sizes, strides, 3))


def test_no_rows():
    from viola_amd import _lib
    for t in (torch.zeros(0, 8), torch.zeros(2, 0, 8), torch.zeros(4, 8)[2:2]):
        assert _lib.host().row_layout(t)[0] == 0
