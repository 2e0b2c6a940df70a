"""How the sequence operators read views in place: the batch stride and row stride they hand to the kernels have to
lead to the view's own entries, within its storage.  The decision depends on shapes and strides alone, so it is
taken here for CPU tensors that call themselves CUDA ones."""
import math

import pytest
import torch

from pysiglib_b200.sequence_inputs import batched_rows

L, C = 3, 2


class OnDevice(torch.Tensor):
    """A CPU tensor on the path of the CUDA ones."""
    is_cuda = True


def count(*shape):
    return torch.arange(math.prod(shape), dtype=torch.float64).view(*shape)


VIEWS = {
    "a unit axis between a slice and the batch": lambda: count(4, 5, L, C)[:, None, :3],
    "a slice behind a unit axis": lambda: count(3, 1, 10, L, C)[:, :, :5],
    "one entry of a slice behind a unit axis": lambda: count(3, 1, 10, L, C)[:, :, :1],
    "an expanded batch behind a unit axis": lambda: count(1, 1, 5, L, C).expand(3, 7, 5, L, C)[:, :1],
    "an expanded batch": lambda: count(1, 5, L, C).expand(3, 5, L, C),
    "all entries the same": lambda: count(1, 1, L, C).expand(3, 5, L, C),
    "a unit axis in front": lambda: count(4, 5, L, C)[None, :, 1:4],
    "a unit axis behind": lambda: count(4, 5, L, C)[:, ::2, None],
    "unit axes all around": lambda: count(4, 6, L, C)[None, :, None, :, None],
    "unit axes alone": lambda: count(2, 1, 1, 1, L, C)[1:],
    "a unit axis unflattened from a slice's": lambda: count(3, 8, L, C).unflatten(0, (3, 1))[:, :, :4],
    "axes that join up": lambda: count(2, 3, 4, L, C),
    "axes that join up with a step": lambda: count(2, 3, 8, L, C)[:, :, ::2],
    "axes in another order": lambda: count(2, 3, 4, L, C).permute(2, 0, 1, 3, 4),
    "rows apart": lambda: count(2, 1, 3, 2 * L, C)[..., ::2, :],
    "channels apart": lambda: count(2, 1, 3, L, 2 * C)[..., ::2],
    "no entries": lambda: count(2, 3, 4, L, C)[:, :0],
}


@pytest.mark.parametrize("name", VIEWS)
def test_strides_lead_to_the_views_entries(name):
    view = VIEWS[name]()
    array, batch_stride, row_stride = batched_rows(view.as_subclass(OnDevice))
    batch = math.prod(view.shape[:-2])
    read = torch.as_strided(array.as_subclass(torch.Tensor), (batch, L, C), (batch_stride, row_stride, 1))
    assert torch.equal(read, view.reshape(batch, L, C))


@pytest.mark.parametrize("name,in_place", [("a unit axis unflattened from a slice's", False), ("a slice behind a unit axis", False),
                                           ("axes that join up", True), ("axes that join up with a step", True),
                                           ("unit axes all around", True),
                                           ("a unit axis behind", False),  # 5 L C from entry to entry, 3 times 2 L C inside
                                           ("rows apart", True),
                                           ("all entries the same", True)])
def test_what_is_read_in_place(name, in_place):
    view = VIEWS[name]()
    assert (batched_rows(view.as_subclass(OnDevice))[0].data_ptr() == view.data_ptr()) == in_place
