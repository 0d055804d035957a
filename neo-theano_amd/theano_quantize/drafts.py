"""Drafted tokens and the pages of sequences that fork, grow and end.

The reference has neither; both stand behind ``KVCache.attention``'s drafted trees:

    o = cache.attention(q, new, tree=tree)                       # ... up to the target's probabilities
    path, kept, token = verify_drafts(tokens, target, new, accept, final, draft=draft, parents=parents)
    lengths = cache.keep(new, path, kept)                        # in each layer's cache

    pool = PagePool.allocate(pages=512, page=64)
    table, source, target = pool.fork(table, lengths, parents)   # samples of a prompt, beams
    cache.copy_pages(source, target)                             # in each layer's cache
    pool.grow(table, lengths + 1, lengths)
    ended |= pool.lacking(table, lengths + 1) > 0                # no page was left for them
    pool.free(table, ended)
"""
from __future__ import annotations

import torch

from . import _abi
from ._tensor import stream
from .cache import _TYPES, _current_device, _dense, _device, _Fixed, _indices
from .errors import InvalidArgument


def _probabilities(t, name, rows, like=None):
    if _device(t, name).dtype not in _TYPES or t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1 or \
            (like is not None and (t.dtype != like.dtype or t.shape != like.shape)):
        raise InvalidArgument(f"{name}: expected float32, bfloat16 or float16 [{rows}, vocab]"
                              f"{'' if like is None else ' as the target is'}, got {t.dtype} {tuple(t.shape)}")
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def verify_drafts(tokens, target, new, accept, final, draft=None, parents=None):
    """Which drafted tokens stay, and the token that follows, so that what comes out is distributed as
    the target's own samples (speculative sampling; trees try their siblings in order).

    new: the KVBatch of the call; the first row of a sequence is its root (already sampled), the others
    are drafted.  tokens: int64 [rows].  target: probabilities [rows, vocab] (f32, bf16 or f16) of the
    token after each row.  draft: likewise, those that a row's children were drawn from, each by itself (siblings
    drawn without replacement are not distributed so), or None where they were not drawn (a draft model's likeliest).  parents: int32 [rows], the row (counted within the sequence)
    that each drafted row follows, before it; None for a chain.  accept: float32 [rows] and final: float32
    [batch], uniform in [0, 1).

    Returns (path, kept, token): int32 [batch, new.tokens] the accepted rows, root first, -1 behind them;
    int32 [batch] how many; int64 [batch] the token to go on with (-1: a sequence without rows)."""
    n, batch, dev = new.rows, new.batch, _current_device()
    _dense(tokens, torch.int64, 1, dev) or _indices(tokens, torch.int64, 1, "verify_drafts: tokens")
    _dense(accept, torch.float32, 1, dev) or _indices(accept, torch.float32, 1, "verify_drafts: accept")
    _dense(final, torch.float32, 1, dev) or _indices(final, torch.float32, 1, "verify_drafts: final")
    if new.device_index != dev:
        raise InvalidArgument("verify_drafts: the batch and the current device differ")
    if tokens.shape[0] != n or accept.shape[0] != n or final.shape[0] != batch:
        raise InvalidArgument(f"verify_drafts: {tokens.shape[0]} tokens and {accept.shape[0]} numbers for {n} rows, "
                              f"{final.shape[0]} for {batch} sequences")
    target = _probabilities(target, "verify_drafts: target", n)
    dp, ds, pp = None, 0, None
    if draft is not None:
        draft = _probabilities(draft, "verify_drafts: draft", n, target)
        dp, ds = draft.data_ptr(), draft.stride(0)
    if parents is not None:
        _dense(parents, torch.int32, 1, dev) or _indices(parents, torch.int32, 1, "verify_drafts: parents")
        if parents.shape[0] != n:
            raise InvalidArgument(f"verify_drafts: {parents.shape[0]} parents for {n} rows")
        pp = parents.data_ptr()
    vocab = target.shape[1]
    path = new.lengths.new_empty((batch, new.tokens))
    kept = new.lengths.new_empty(batch)
    token = tokens.new_empty(batch)
    nb = _abi.entry("tq_verify_drafts_workspace_bytes")(new._desc, vocab)
    ws = final.new_empty(nb // 4) if nb > 0 else None
    _abi.call("tq_verify_drafts", new._desc, tokens.data_ptr(), target.data_ptr(), target.stride(0), dp, ds,
              _TYPES[target.dtype], vocab, pp, accept.data_ptr(), final.data_ptr(), None if ws is None else ws.data_ptr(), nb, path.data_ptr(),
              kept.data_ptr(), token.data_ptr(), stream())
    return path, kept, token


class PagePool(_Fixed):
    """Which pages of a cache (or of all layers' caches) are held, on the device.

    holders: int32 [pages], how many table entries name each page (0: free); page: its tokens.  Tables
    are int32 [batch, n] as in KVBatch, -1 where a sequence has no page, its pages first.  Nothing is
    read on the host: where pages run out entries stay -1, rows of such places are not written and
    seen by nobody, and `lacking` tells.  A page comes with what its last sequence left on it, so that the tokens of
    a missing page are lost: the sequence ends, or goes on without them, and then `grow` is told which
    of its tokens are stored, or it puts a page of somebody else's tokens in their place.  Calls on one pool belong on one stream."""

    def __init__(self, holders, page):
        _indices(holders, torch.int32, 1, "PagePool: holders")
        if holders.shape[0] < 1 or holders.data_ptr() % 16 or not 1 <= int(page) <= 65536:
            raise InvalidArgument(f"PagePool: expected 16-byte aligned holders of pages of 1 to 65536 tokens, got {holders.shape[0]} of {page}")
        self.__dict__.update(holders=holders, page=int(page), pages=holders.shape[0], device_index=holders.get_device(),
                             _desc=_abi.page_pool_desc(holders.data_ptr(), holders.shape[0], int(page)))

    @staticmethod
    def allocate(pages, page):
        """A pool of free pages on the current device."""
        return PagePool(torch.zeros(pages, dtype=torch.int32, device=torch.device("cuda", torch.cuda.current_device())), page)

    def _table(self, table, name):
        dev = self.device_index
        _dense(table, torch.int32, 2, dev) or _indices(table, torch.int32, 2, name)
        if dev != _current_device():
            raise InvalidArgument(f"{name}: the pool and the current device differ")
        return table.data_ptr(), table.stride(0), table.shape[1]

    def _lengths(self, lengths, table, name):
        _dense(lengths, torch.int32, 1, self.device_index) or _indices(lengths, torch.int32, 1, name)
        if lengths.shape[0] != table.shape[0]:
            raise InvalidArgument(f"{name}: {lengths.shape[0]} lengths for {table.shape[0]} sequences")
        return lengths.data_ptr()

    def grow(self, table, lengths, stored=None):
        """Gives each sequence pages for `lengths` (int32 [batch]) tokens, behind those it has, in `table` itself: the
        lowest free ones, sequence by sequence.  stored (int32 [batch]): how many of its tokens caches have been
        written for; entries of theirs that have no page stay so, for their tokens are lost.  None: no token behind its
        last page has been written yet."""
        where = self._table(table, "PagePool.grow: table")
        want = self._lengths(lengths, table, "PagePool.grow: lengths")
        if stored is None:
            _abi.call("tq_pages_grow", self._desc, *where, want, table.shape[0], stream())
        else:
            _abi.call("tq_pages_grow_stored", self._desc, *where, want, self._lengths(stored, table, "PagePool.grow: stored"), table.shape[0],
                      stream())

    def lacking(self, table, lengths):
        """How many pages of its `lengths` (int32 [batch]) tokens each sequence does not have, int32 [batch]: those that `grow` or
        `fork` found none for (past the table's end, too)."""
        where = self._table(table, "PagePool.lacking: table")
        want, out = self._lengths(lengths, table, "PagePool.lacking: lengths"), torch.empty_like(lengths)
        _abi.call("tq_pages_lacking", self._desc, *where, want, table.shape[0], out.data_ptr(), stream())
        return out

    def fork(self, table, lengths, parents):
        """(children, source, target): the table of copies of the sequences `parents` (int32 [n]) of `lengths` tokens.
        Whole pages are shared; a page that a sequence has begun is copied by
        ``KVCache.copy_pages(source, target)``, in each layer.  Where no page is left for the copy the child has none there and its tokens on it are
        lost (`lacking` of its lengths tells, and `grow` is told that they were stored).  The parents stay until they are freed."""
        where = self._table(table, "PagePool.fork: table")
        dev = self.device_index
        _dense(lengths, torch.int32, 1, dev) or _indices(lengths, torch.int32, 1, "PagePool.fork: lengths")
        _dense(parents, torch.int32, 1, dev) or _indices(parents, torch.int32, 1, "PagePool.fork: parents")
        if lengths.shape[0] != table.shape[0]:
            raise InvalidArgument(f"PagePool.fork: {lengths.shape[0]} lengths for {table.shape[0]} sequences")
        n = parents.shape[0]
        children = table.new_empty((n, table.shape[1]))
        source, target = torch.empty_like(parents), torch.empty_like(parents)
        _abi.call("tq_pages_fork", self._desc, *where, lengths.data_ptr(), table.shape[0], parents.data_ptr(), n,
                  children.data_ptr(), source.data_ptr(), target.data_ptr(), stream())
        return children, source, target

    def free(self, table, sequences=None):
        """The sequences (bool [batch]; None: all) give their pages back; their entries become -1."""
        where = self._table(table, "PagePool.free: table")
        if sequences is not None:
            _indices(sequences, torch.bool, 1, "PagePool.free: sequences")
            if sequences.shape[0] != table.shape[0]:
                raise InvalidArgument(f"PagePool.free: {sequences.shape[0]} truth values for {table.shape[0]} sequences")
        _abi.call("tq_pages_free", self._desc, *where, table.shape[0], None if sequences is None else sequences.data_ptr(),
                  stream())
