"""Calls of the paged-cache ops at the edge of what they take: work that is more
than one launch can count, tables whose rows lie on each other."""
import pytest
import torch

import zentorch  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.zentorch


@pytest.fixture(autouse=True)
def _announce(request):
    print(f"\n[case] {request.node.name}", flush=True)


def test_copy_pages_of_many_pairs():
    """More pairs than a launch has workgroups for (2^24 of 256 threads)."""
    n = (1 << 24) + 3
    caches = [torch.randn(9, 2, 8, device=DEV) for _ in range(3)]
    want = [c.clone() for c in caches]
    copies = torch.full((n, 2), -1, dtype=torch.int32, device=DEV)
    for k, (src, dst) in ((0, (0, 1)), (n // 2, (2, 3)), (1 << 24, (4, 5)), (n - 1, (6, 7))):
        copies[k] = torch.tensor([src, dst])
        for w in want:
            w[dst] = w[src]
    ops.zentorch_cache_copy_pages(caches, copies)
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_rotary_of_many_elements():
    """More units than a launch has threads for (2^32), rows off 16 bytes."""
    T, H, D = (1 << 20) + 5, 32, 130
    assert T * H * (D - 1) > 1 << 32
    x = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
    row = torch.randn(H, D, device=DEV).bfloat16()
    x[:] = row
    pos = torch.zeros(T, dtype=torch.int64, device=DEV)
    pos[-1], pos[T // 2] = 1, 1
    table = torch.tensor([[1.0, 0.0], [0.0, 1.0]], device=DEV)  # no turn, a quarter
    y = ops.zentorch_rotary_embedding(x, pos, table)
    turned = row.clone()
    turned[:, 0], turned[:, 1] = -row[:, 1], row[:, 0]
    for t in (0, 1, T // 2 - 1, T // 2 + 1, T - 2):
        assert torch.equal(y[t], row), t
    for t in (T // 2, T - 1):
        assert torch.equal(y[t], turned), t
    y[T // 2], y[T - 1] = row, row
    assert (y.view(torch.int16) == row.view(torch.int16)).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_table_of_overlapping_rows(interleaved):
    """One row expanded to every position, and rows that begin inside the one
    before, as any other table."""
    x = torch.randn(6, 3, 16, device=DEV)
    pos = torch.arange(6, device=DEV)
    one = torch.randn(1, 8, device=DEV)
    flat = torch.randn(40, device=DEV)
    for table in (one.expand(9, 8), flat.as_strided((9, 8), (3, 1)), torch.randn(9, 16, device=DEV)[:, ::2],
                  torch.randn(8, 9, device=DEV).t()):
        got = ops.zentorch_rotary_embedding(x, pos, table, interleaved=interleaved)
        assert torch.equal(got, ops.zentorch_rotary_embedding(x, pos, table.contiguous(), interleaved=interleaved))
