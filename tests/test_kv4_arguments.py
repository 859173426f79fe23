"""Arguments of the 4-bit paged cache's calls whose results would depend on the order of threads, and what calls promise beyond one pool."""

import pytest
import torch

import mega_kernel_qwen36 as mk
from oracle import kv4_oracle as oracle
from test_kv4_cache import Server, _cu, _lists


@pytest.mark.gpu
def test_read_refuses_outputs_that_lie_over_one_another(cuda_device):
    s = Server(cuda_device, torch.bfloat16, 128, 2, 16, [20, 3])
    s.fill()
    make = lambda *shape: torch.full(shape, 7, dtype=torch.bfloat16, device=cuda_device)
    one, rows = make(2, 3, 2, 128), make(1, 3, 2, 128).expand(2, 3, 2, 128)
    both = make(2 * 2 * 3 * 2 * 128)
    n = one.numel()
    for out in ((one, one), (rows, one), (one, rows), (make(2, 1, 2, 128).expand(2, 3, 2, 128), one),
                (both[:n].view(2, 3, 2, 128), both[128 : n + 128].view(2, 3, 2, 128)),
                (one, s.cache.pool.view(-1).view(torch.bfloat16)[:n].view(2, 3, 2, 128))):
        with pytest.raises(RuntimeError, match="memory"):
            mk.kv4_read(s.cache, s.gpu, 3, out=out)
    ragged = make(1, 2, 128).expand(6, 2, 128)
    with pytest.raises(RuntimeError, match="memory"):
        mk.kv4_read(s.cache, s.gpu, 6, cu_tokens=_cu([3, 3], cuda_device), out=(ragged, make(6, 2, 128)))
    assert (one == 7).all() and (both == 7).all()
    s.same_pool()
    want = mk.kv4_read(s.cache, s.gpu, 3)
    halves = both.view(2, 2, 3, 2, 128)
    got = mk.kv4_read(s.cache, s.gpu, 3, out=(halves[0], halves[1]))  # side by side in one allocation
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    wide = make(2, 3, 2, 2, 128)  # token by token, keys beside values
    got = mk.kv4_read(s.cache, s.gpu, 3, out=(wide[:, :, 0], wide[:, :, 1]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_layers_share_a_table_and_have_a_pool_each(cuda_device):
    """Each layer's call takes the table as it was before the step and gives the same new one, with that layer's pages copied and moved."""
    servers = [Server(cuda_device, torch.bfloat16, 64, heads, 32, [70, 0, 40, 0], seed=3) for heads in (1, 2, 1)]
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    table = servers[0].gpu
    for i, s in enumerate(servers):
        s.fill(seed=i)
        assert _lists(s.gpu) == _lists(table)
    state = _lists(table)
    *state, status = oracle.fork(*state, [0], [1])
    table, wrong = mk.kv_pages_fork(table, on([0]), on([1]))
    assert wrong.item() == status == 0
    after = [71, 74, 3, 33]
    for name in ("resize", "compact"):
        results = []
        for i, s in enumerate(servers):
            last = i == len(servers) - 1
            if name == "resize":
                *new_state, status = oracle.resize(s.pool, *state, after)
                new, got = mk.kv_pages_resize(s.cache, table, on(after), inplace=last)
            else:
                *new_state, status = oracle.compact(s.pool, *state)
                new, got = mk.kv_pages_compact(s.cache, table, inplace=last)
            assert got.item() == status and _lists(new) == tuple(new_state)
            s.same_pool()
            results.append(new)
        assert new is table  # the last layer's call may change the table where it lies
        state = new_state
