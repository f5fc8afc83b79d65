"""Block tables of sequences that share INT4 records, kept and changed on the GPU.

The rows of a BlockTables are the sequences of a batch; a row names the 16-token block records
that hold its tokens, in one pool or in the pools of all layers (one id, the same record of
every pool).  Rows that came from one another share their full records, counted by `refs`, so
n samples or beams of a prompt hold it once, and ops.shared_prefix_attention reads it once:

    tables = BlockTables(pools, num_sequences=16, max_tokens=40960)
    start = tables.extend([n] + [0] * 15)             # blocks for a prompt in row 0
    ops.pack_tokens(pool, k, v, start[:1], tables.table[:1])         # in every layer's pool
    tables.select([0] * 16)                            # 16 samples of it
    start = tables.extend(1)                           # blocks for a token each
    ops.pack_tokens(pool, k1, v1, start, tables.table)
    out = ops.shared_prefix_attention(q, n // 16, pool=pool, block_table=tables.table,
                                      int4_lens=tables.lens, int4_max_len=n + 1)
    tables.select([0, 3, 3, -1] + ...)                 # keep, drop, copy, finish rows
    tables.compact()                                   # live records to the front of the pools

Everything runs on the GPU without a host synchronization and can be captured in a HIP graph
(with device tensors for arguments).  A call that does not fit changes nothing; why is in the
error word, which check_errors() reads.
"""
import ctypes
import operator

import torch

from . import _lib
from . import ops
from ._lib import BLOCK_TOKENS, HEAD_DIM, HeteroKVError, check, load, stream_ptr

_WIDE = (torch.uint32, torch.int64, torch.uint64)


class BlockTables:
    """Device state: `table` int32 [S, columns] (entries past a row's blocks are -1), `lens`
    int32 [S] (tokens), `refs` int32 [N] (rows that hold a block) and `free` int32 [N / 32] (bit
    i % 32 of word i / 32: no row holds block i), views of the one int32 buffer `state`.  The
    pools' records are this object's to hand out and to move (others may hold saved copies of it).
    Calls on one object are ordered on one stream, as on any state."""

    def __init__(self, pools, num_sequences, max_tokens, err=None):
        """pools: the Int4Pool(s) that the ids name, of one size; num_sequences: rows (at most
        1024); max_tokens: the longest a row can get; err: an ErrorWord (default: an own one)."""
        self.pools = [pools] if isinstance(pools, ops.Int4Pool) else list(pools)
        if not self.pools:
            raise HeteroKVError(-1, "BlockTables: no pool")
        p = self.pools[0]
        ops._require_gpu(*(q.data for q in self.pools))
        for q in self.pools:
            if (q.num_blocks, q.num_kv_heads, q.device) != (p.num_blocks, p.num_kv_heads, p.device):
                raise HeteroKVError(-1, "BlockTables: pools of different sizes, heads or devices")
            if q.data.data_ptr() % 16 or not q.data.is_contiguous() or q.data.numel() < p.num_blocks * p.record_bytes:
                raise HeteroKVError(-1, "BlockTables: a pool's records must be contiguous and 16-byte aligned")
        if not 1 <= num_sequences <= _lib.MAX_SEQUENCES:
            raise HeteroKVError(-1, "BlockTables: %d sequences outside [1, %d]" % (num_sequences, _lib.MAX_SEQUENCES))
        if max_tokens < 1 or p.num_blocks < 1:
            raise HeteroKVError(-1, "BlockTables: max_tokens %d, %d blocks" % (max_tokens, p.num_blocks))
        self.device = p.device
        self.num_sequences, self.num_blocks = int(num_sequences), p.num_blocks
        self.columns = (int(max_tokens) + BLOCK_TOKENS - 1) // BLOCK_TOKENS
        if (self.num_sequences * self.columns >= 2 ** 31 or self.columns > _lib.MAX_TABLE_COLUMNS or
                p.num_blocks > _lib.MAX_TABLE_BLOCKS):
            raise HeteroKVError(-1, "BlockTables: %d rows of %d blocks out of %d are too many" %
                                (self.num_sequences, self.columns, p.num_blocks))
        words = (p.num_blocks + 31) // 32
        sizes = [self.num_sequences * self.columns, self.num_sequences, p.num_blocks, words]
        starts = [0]
        for n in sizes:
            starts.append((starts[-1] + n + 3) // 4 * 4)
        self.state = torch.zeros(starts[-1], dtype=torch.int32, device=self.device)
        table, self.lens, self.refs, self.free = (self.state[s:s + n] for s, n in zip(starts, sizes))
        self.table = table.view(self.num_sequences, self.columns)
        self.err = err if err is not None else ops.ErrorWord(self.device)
        self._records = [q.data for q in self.pools]   # held: their addresses are the kernels'
        self._addresses = [r.data_ptr() for r in self._records]
        self._pool_ptrs = torch.tensor(self._addresses, dtype=torch.int64).to(self.device)
        self._lib = load()
        nbytes = self._lib.hkv_blocks_workspace_bytes(self.num_sequences, self.num_blocks)
        self._ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self._args = _lib.BlockTablesArgs(
            table=self.table.data_ptr(), lens=self.lens.data_ptr(), refs=self.refs.data_ptr(),
            free_bits=self.free.data_ptr(), pools=self._pool_ptrs.data_ptr(), num_blocks=self.num_blocks,
            num_sequences=self.num_sequences, table_stride=self.columns, num_pools=len(self.pools),
            num_kv_heads=p.num_kv_heads, head_dim=HEAD_DIM, err_flag=self.err.ptr(), workspace=self._ws.data_ptr(),
            workspace_bytes=nbytes)
        self._ref = ctypes.byref(self._args)
        self._free_all()

    def clear(self):
        """No sequence holds a block."""
        self.state.zero_()
        self._free_all()

    def _free_all(self):
        """Of a state of zeros."""
        self.table.fill_(-1)
        self.free.fill_(-1)
        if self.num_blocks % 32:
            self.free[-1:].fill_((1 << (self.num_blocks % 32)) - 1)

    def copy_(self, other):
        """Take the tables, lengths and counts of `other` (of the same pools and sizes), to go back to
        them: the records that rows of `other` held have to be as they were."""
        if (other.num_sequences, other.columns, other.num_blocks) != (self.num_sequences, self.columns, self.num_blocks):
            raise HeteroKVError(-1, "BlockTables.copy_: other sizes")
        if other._addresses != self._addresses:
            raise HeteroKVError(-1, "BlockTables.copy_: tables of other pools")
        self.state.copy_(other.state)
        return self

    def _rows(self, x, what, least, most):
        """One int32 per row on the device; host values are checked here, device ones by the kernel."""
        if isinstance(x, torch.Tensor) and (x.is_floating_point() or x.is_complex()):
            raise HeteroKVError(-1, "%s: integers expected, one for each of %d rows" % (what, self.num_sequences))
        if isinstance(x, torch.Tensor) and x.device.type != "cpu":
            if x.numel() != self.num_sequences:
                raise HeteroKVError(-1, "%s: %d values for %d rows" % (what, x.numel(), self.num_sequences))
            if x.device != self.device:
                raise HeteroKVError(-1, "%s: a tensor on %s, the tables are on %s" % (what, x.device, self.device))
            if x.dtype in _WIDE:   # what 32 bits do not hold stays out of range
                if x.dtype == torch.uint64:
                    x = x.view(torch.int64)
                    x = torch.where(x < 0, 2 ** 31 - 1, x)
                x = x.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)
            return x if x.dtype == torch.int32 and x.is_contiguous() else x.reshape(-1).to(torch.int32).contiguous()
        try:
            x = [operator.index(v) for v in (x.reshape(-1).tolist() if isinstance(x, torch.Tensor) else x)]
        except TypeError:
            raise HeteroKVError(-1, "%s: integers expected, one for each of %d rows" % (what, self.num_sequences))
        if len(x) != self.num_sequences or any(v < least or v > most for v in x):
            raise HeteroKVError(-1, "%s: %d values in [%d, %d] expected, one for each row" %
                                (what, self.num_sequences, least, most))
        return ops.h2d(torch.tensor(x, dtype=torch.int32), self.device)

    def _launch(self, name, *args):
        if torch.cuda.current_device() != self.device.index:   # a default stream is that of the current device
            with torch.cuda.device(self.device):
                return self._launch(name, *args)
        check(getattr(self._lib, name)(self._ref, *args, stream_ptr(self.device)), name)

    def extend(self, tokens):
        """Make the rows `tokens` longer (an int for every row, or one value for each) and give
        them the blocks for it, the lowest free ids first, to the rows in order.  Returns the
        lengths before (int32 [S]), where ops.pack_tokens is to start."""
        rows, each = None, 0
        if not isinstance(tokens, torch.Tensor) and hasattr(tokens, "__index__"):
            tokens = operator.index(tokens)
            if not 0 <= tokens <= self.columns * BLOCK_TOKENS:
                raise HeteroKVError(-1, "BlockTables.extend: %d tokens" % tokens)
            each = tokens
        else:
            rows = self._rows(tokens, "BlockTables.extend", 0, self.columns * BLOCK_TOKENS)
        starts = torch.empty_like(self.lens)
        self._launch("hkv_blocks_extend", rows.data_ptr() if rows is not None else None, each, starts.data_ptr())
        return starts

    def select(self, source):
        """Row i becomes what row source[i] was (-1: empty), for all rows at once: a fork, a beam
        step, the end of a sequence.  Rows of one source share its full blocks; its partial last
        one stays with the first of them, the others get copies, in every pool.  Blocks that no row
        holds any more become free."""
        rows = self._rows(source, "BlockTables.select", -1, self.num_sequences - 1)
        self._launch("hkv_blocks_select", rows.data_ptr())

    def compact(self):
        """Move records, in every pool, so that the n held blocks have the ids 0 .. n - 1; of
        them, those that have such an id keep it."""
        self._launch("hkv_blocks_compact")

    def check_errors(self):
        """Raise HeteroKVError if a call since the last check changed nothing (synchronizes)."""
        self.err.check()
