"""The paged-cache ops under torch.compile: the ops that write the caches in
place, one of them in a list, keep their order and their effect."""
import pytest
import torch
import torch._dynamo

import zentorch  # noqa: F401
from test_kv_cache_gpu import BF, DEV, i32, pages_of, table_of

pytestmark = pytest.mark.gpu
ops = torch.ops.zentorch


@pytest.fixture(autouse=True)
def _announce(request):
    print(f"\n[case] {request.node.name}", flush=True)
    torch._dynamo.reset()
    yield
    torch._dynamo.reset()


S, H, KV, D, PAGE, WIDTH = 5, 8, 2, 64, 16, 8


def step(x, caches, table, ctx, refs, par, cu, cos_sin):
    """A decode step of two layers with the pages' upkeep before it."""
    table, ctx, refs, copies = ops.zentorch_cache_fork(table, ctx, refs, par, PAGE)
    ops.zentorch_cache_copy_pages(caches, copies)
    table, refs, copies = ops.zentorch_cache_compact(table, refs)
    ops.zentorch_cache_copy_pages(caches, copies)
    table, ctx, refs, pos, slots = ops.zentorch_cache_extend(table, ctx, refs, cu, PAGE, S)
    for cache in caches:
        k_cache, v_cache = cache[:, 0], cache[:, 1]
        q, k, v = (s.view(S, -1, D) for s in x.split([H * D, KV * D, KV * D], 1))
        q = ops.zentorch_rotary_cache_append(q, k, v, pos, cos_sin, slots, k_cache, v_cache)
        a = ops.zentorch_paged_attention(q, k_cache, v_cache, table, cu, ctx, 1).flatten(1)
        x = torch.cat([a, x[:, :2 * KV * D] + a[:, :2 * KV * D]], 1)
    return x, table, ctx, refs


@pytest.mark.parametrize("backend", ["eager", "aot_eager", "zentorch"])
def test_step(backend):
    torch.manual_seed(0)
    lens = [30, 16, 1, 50, 7]
    rows, refs = pages_of(lens, PAGE, 12, WIDTH, 3)
    caches = [torch.randn(len(refs), 2, KV, PAGE, D, device=DEV).to(BF) for _ in "ab"]
    args = (i32(rows), i32(lens), i32(refs), i32([0, 0, 2, 3, 3]), i32(list(range(S + 1))), table_of(200, D))
    x = torch.randn(S, (H + 2 * KV) * D, device=DEV).to(BF)
    mine = [c.clone() for c in caches]
    want = step(x, caches, *args)
    fast = torch.compile(step, backend=backend, fullgraph=True)
    with torch.no_grad():
        got = fast(x, mine, *args)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(mine, caches))
    # once more on what the first call left, through the compiled code's cache
    want = step(x, caches, *want[1:], *args[3:])
    with torch.no_grad():
        got = fast(x, mine, *got[1:], *args[3:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(mine, caches))
