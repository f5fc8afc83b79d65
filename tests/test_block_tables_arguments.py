"""What BlockTables takes for a row's number or token count: whole numbers of any type, host or
device, and nothing that would have to be cut or wrapped to become one."""
import types

import pytest
import torch

DEV = "cuda:0"
BAD = [[0, 1.5, 2], [0, 0.0, 2], [0, None, 2], [0, "1", 2], [0, 1], [0, 1, 2, 0], [0, 1, 2 ** 32], [0, -2, 1], 1.0, None, "012",
       [0, 1, 3], [0, [1], 2], torch.tensor([0.9, 1, 2]), torch.tensor([0, 1, 2], dtype=torch.complex64),
       torch.tensor([0, 1, 2 ** 32 - 1], dtype=torch.uint32), torch.tensor([0, 1, 2 ** 64 - 1], dtype=torch.uint64)]
GOOD = [[0, 1, 2], (0, 1, 2), range(3), [False, True, 2], torch.arange(3), torch.arange(3, dtype=torch.uint8), torch.arange(3)[:, None],
        torch.tensor([0, 1, 2], dtype=torch.uint32), torch.tensor([0, 1, 2], dtype=torch.uint64), [torch.tensor(0), 1, 2]]


@pytest.mark.parametrize("i", range(len(BAD) + len(GOOD)))
def test_host_values(i):
    from heterokv import BlockTables, HeteroKVError
    rows = types.SimpleNamespace(num_sequences=3, device=torch.device("cpu"))
    x = (BAD + GOOD)[i]
    if i >= len(BAD):
        assert BlockTables._rows(rows, x, "rows", -1, 2).tolist() == [0, 1, 2]
    else:
        with pytest.raises(HeteroKVError):
            BlockTables._rows(rows, x, "rows", -1, 2)


def test_host_arrays():
    numpy = pytest.importorskip("numpy")
    from heterokv import BlockTables, HeteroKVError
    rows = types.SimpleNamespace(num_sequences=3, device=torch.device("cpu"))
    assert BlockTables._rows(rows, numpy.arange(3, dtype=numpy.uint16), "rows", -1, 2).tolist() == [0, 1, 2]
    with pytest.raises(HeteroKVError):
        BlockTables._rows(rows, numpy.array([0.0, 1.0, 2.0]), "rows", -1, 2)


@pytest.mark.gpu
def test_calls_and_device_values():
    import heterokv
    from heterokv import HeteroKVError, ops
    t = heterokv.BlockTables(ops.Int4Pool(50, 1, DEV), 3, 200)
    t.extend([20, 40, 5])
    before = t.state.clone()
    for bad in BAD:
        for call in (t.select, t.extend):
            if call == t.extend and bad in ([0, 1, 3],):
                continue     # a good count of tokens
            with pytest.raises(HeteroKVError):
                call(bad)
    for dtype in (torch.uint32, torch.uint64, torch.int64):
        for x in ([0, 1, 2 ** 32 - 1], [0, 1, 2 ** 31], [0, 1, 2 ** 64 - 1], [0, 1, 2 ** 63], [0, 1, 2 ** 32 + 1]):
            if max(x) > torch.iinfo(dtype).max:
                continue
            for call in (t.select, t.extend):
                call(torch.tensor(x, dtype=dtype).to(DEV))
                with pytest.raises(HeteroKVError):
                    t.check_errors()
    for bad in (torch.zeros(3, device=DEV), torch.zeros(2, dtype=torch.uint32, device=DEV)):
        with pytest.raises(HeteroKVError):
            t.select(bad)
    torch.cuda.synchronize()
    assert torch.equal(t.state, before)
    for dtype in (torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64, torch.uint64):
        t.select(torch.tensor([0, 1, 2], dtype=dtype).to(DEV))
        wide = torch.tensor([[0, 9], [1, 9], [2, 9]], dtype=dtype).to(DEV)[:, 0]
        t.select(wide)
        t.check_errors()
        assert torch.equal(t.state, before)


@pytest.mark.gpu
def test_tables_of_other_pools_are_not_taken_back():
    import heterokv
    from heterokv import HeteroKVError, ops
    pools = [ops.Int4Pool(20, 1, DEV) for _ in range(2)]
    t = heterokv.BlockTables(pools, 3, 64)
    t.extend([20, 5, 0])
    before = t.state.clone()
    for other in ([ops.Int4Pool(20, 1, DEV) for _ in range(2)], pools[:1], pools[::-1], [pools[0], pools[0]]):
        with pytest.raises(HeteroKVError, match="pools"):
            t.copy_(heterokv.BlockTables(other, 3, 64))
    assert torch.equal(t.state, before)
    saved = heterokv.BlockTables(pools, 3, 64).copy_(t)
    t.select([1, 1, 1])
    assert torch.equal(t.copy_(saved).state, before)


@pytest.mark.gpu
def test_rows_of_very_many_columns():
    """A row may be as long as 2^26 blocks of table, of which it can hold as many as the pool has:
    1024 threads for every 16 of its columns would be 2^32, more than a launch can have."""
    import heterokv
    from heterokv import HeteroKVError, ops
    pool = ops.Int4Pool(70, 1, DEV)
    t = heterokv.BlockTables(pool, 1, 2 ** 30)
    assert t.extend(16 * 69 + 3).tolist() == [0] and t.table[0, :70].tolist() == list(range(70))
    t.select([0])
    t.check_errors()
    assert t.lens.tolist() == [16 * 69 + 3] and t.refs.tolist() == [1] * 70
    t.select([-1])
    t.check_errors()
    assert t.lens.tolist() == [0] and t.refs.tolist() == [0] * 70 and bool((t.table == -1).all())
    assert t.free.tolist() == [-1, -1, 63]
    t.extend(100)
    t.compact()
    t.check_errors()
    assert t.table[0, :8].tolist() == list(range(7)) + [-1]
    with pytest.raises(HeteroKVError, match="too many"):
        heterokv.BlockTables(pool, 1, 2 ** 30 + 1)
