"""Calls of the decoding operators (mmf_amd/decoding.py) that the documentation allows: layouts of the cache's planes, indices outside their tables."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32


def D():
    from mmf_amd import decoding
    return decoding


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


@pytest.fixture(autouse=True)
def no_index_error():
    from mmf_amd import _native as nat
    nat.take_index_error()
    yield
    assert not nat.take_index_error()


# ---------------------------------------------------------------------------------------------
# planes: leading dimensions of the cache, some of size 1
# ---------------------------------------------------------------------------------------------
LEADING = [(), (1,), (4,), (4, 1), (1, 4), (4, 1, 2), (1, 1), (2, 1, 1), (1, 3, 1, 2)]


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 5)])
@pytest.mark.parametrize("lead", LEADING)
def test_copies_reach_every_plane(lead, dtype, dim):
    cache = torch.randn(*lead, 6, 2, 16, dim, device=DEV).to(dtype)
    copies = [[0, 3, 7], [5, 1, 16], [-1, -1, -1], [4, 4, 9]]
    want = cache.clone()
    for s, d, n in copies[:2]:
        want[..., d, :, :n, :] = cache[..., s, :, :n, :]
    D().copy_pages(i32(copies), cache)
    assert torch.equal(cache, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead", LEADING)
def test_reorder_copies_in_every_plane(lead, dtype):
    cache = torch.randn(*lead, 6, 2, 16, 64, device=DEV).to(dtype)
    want = cache.clone()
    want[..., 2, :, :5, :] = cache[..., 3, :, :5, :]            # both children of beam 1: the second takes beam 0's page
    want[..., 4, :, :5, :] = cache[..., 3, :, :5, :]            # and the third beam 2's
    got = D().reorder_pages(torch.tensor([[1, 1, 1]], device=DEV), i32([21]), i32([[0, 2], [1, 3], [5, 4]]), cache)
    assert got.tolist() == [[1, 3], [1, 2], [1, 4]] and torch.equal(cache, want)


def test_planes_of_a_slice_of_the_layers():
    """One leading dimension may have any stride: keys only, of a pool that holds keys and values."""
    cache = torch.randn(3, 2, 6, 2, 16, 64, device=DEV)
    want = cache.clone()
    want[:, 0, 3, :, :7] = cache[:, 0, 0, :, :7]
    D().copy_pages(i32([[0, 3, 7]]), cache[:, 0])
    assert torch.equal(cache, want)
