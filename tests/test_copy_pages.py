"""Copies of the first positions of pages, in every stage of a pool."""
import pytest
import torch

from beglin_b200.csrc import ops

DEV = "cuda:0"

# shape of a page in front of its positions and features, the features, the type, positions of a page, positions to copy
CASES = [((2, 2), 128, torch.bfloat16, 64, 45), ((2, 3), 80, torch.float32, 16, 1), ((2, 1), 20, torch.bfloat16, 4, 3), ((), 576, torch.bfloat16, 64, 64),
         ((2, 5), 3, torch.bfloat16, 5, 3), ((), 7, torch.float32, 1, 1), ((2, 2), 64, torch.float32, 64, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [[(3, 1)], [(2, 0), (2, 9), (5, 4), (2, 7), (5, 1)], [(0, i) for i in range(1, 300)]], ids=["one", "two sources", "many"])
@pytest.mark.parametrize("outer,features,dtype,rows,n", CASES)
def test_copied_pages(outer, features, dtype, rows, n, pairs):
    pages = max(max(p) for p in pairs) + 2
    pool = torch.randn((3, pages, *outer, rows, features), generator=torch.Generator().manual_seed(n)).to(dtype).to(DEV)
    want = pool.clone()
    for s, d in pairs:
        want[:, d, ..., :n, :] = pool[:, s, ..., :n, :]
    ops.copy_pages(pool, [s for s, _ in pairs], [d for _, d in pairs], n)
    assert torch.equal(pool, want)


@pytest.mark.gpu
def test_copied_pages_of_a_part_of_wider_pages():
    """Keys and values of different sizes lie one behind the other in a page: each part is a pool of its own."""
    flat = torch.randn((2, 6, 3 * 8 * (24 + 10)), device=DEV)
    want = flat.clone()
    keys = flat.as_strided((2, 6, 3, 8, 24), (flat.stride(0), flat.stride(1), 8 * 24, 24, 1))
    values = flat.as_strided((2, 6, 3, 8, 10), (flat.stride(0), flat.stride(1), 80, 10, 1), 3 * 8 * 24)
    for part, w in ((keys, 24), (values, 10)):
        ops.copy_pages(part, [1, 1], [4, 0], 5)
    k, v = want[:, :, :3 * 8 * 24].view(2, 6, 3, 8, 24).clone(), want[:, :, 3 * 8 * 24:].view(2, 6, 3, 8, 10).clone()
    for t in (k, v):
        t[:, 4, :, :5] = t[:, 1, :, :5]
        t[:, 0, :, :5] = t[:, 1, :, :5]
    assert torch.equal(flat, torch.cat([k.flatten(2), v.flatten(2)], dim=2))


def test_copied_pages_refusals():
    pool = torch.zeros(2, 5, 2, 8, 16)

    def refused(match, src, dst, n, pool=pool):
        with pytest.raises(ops.KernelError, match=match):
            ops.copy_pages(pool, src, dst, n)

    refused("CUDA device only", [0], [1], 3)
    refused("expected", [0], [1], 3, pool=torch.zeros(5, 8, 16))
    refused("side by side", [0], [1], 3, pool=torch.zeros(2, 5, 2, 16, 8).transpose(3, 4))
    refused("overlap", [0], [1], 3, pool=torch.zeros(2, 1, 2, 8, 16).expand(2, 5, 2, 8, 16))
    refused("positions", [0], [1], 9)
    refused("positions", [0], [1], -1)
    refused("to read", [0, 1], [2], 3)
    refused("outside", [0], [5], 3)
    refused("outside", [-1], [2], 3)
    refused("written twice", [0, 1], [2, 2], 3)
    refused("read and written", [0, 1], [1, 2], 3)
