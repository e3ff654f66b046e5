"""A cache of pages for serving: its rows, pages and sequences, and the attention of drafted tokens over it.

The cache is two tensors ``k_cache`` and ``v_cache`` of shape (pages, Hk, slots, E): fp16 or bf16, any storage with unit last stride and
rows of aligned 16-byte pieces ((pages, slots, Hk, E) storage seen through ``.transpose(1, 2)`` is as good), E a multiple of 8 up to 256,
the slots of a page a power of two from 16 up.  A sequence is a row of ``page_table`` (int32 (sequences, columns), -1 where there
is no page) and an entry of ``lengths`` (int32): slot n lies in the page of column n // slots, at n % slots.

A step of speculative decoding, with nothing that waits for the device:

    append(key, value, k_cache, v_cache, page_table, lengths)                            # drafted rows behind each sequence
    out = tree_attention(query, k_cache, v_cache, page_table, lengths, parents, max_length)
    lengths = keep_path(k_cache, v_cache, page_table, lengths, path, counts)             # what the caller accepted moves together

Which pages belong to whom is the caller's: page_table, and ``uses``, the number of table entries that name a page (a page without
one is free).  fork and free keep both up to date.  Indices are read on the device and none is trusted: a page outside the
cache, a sequence outside the table, a slot outside a row of the table, a negative length stand for nothing, which is not read and not
written.  All functions run on torch's current stream and can be captured into a HIP graph.  None has a gradient: where autograd
would record one (NotImplementedError), call them under torch.no_grad().  Shapes, types, strides and devices
are checked on the host: ValueError, or RuntimeError with the library's hipError_t.
"""
import math

import torch

from . import _host

_host.load()      # registers the ops

__all__ = ['tree_attention', 'append', 'copy_pages', 'fork', 'keep_path', 'free']

_ops = torch.ops.aotriton_amd


@torch.library.register_fake('aotriton_amd::tree_attention')
def _(query, k_cache, v_cache, page_table, lengths, parents, max_length, window, sinks, sm_scale):
    out = torch.empty((query.shape[0], query.shape[1], query.shape[2], v_cache.shape[3]), device=query.device, dtype=query.dtype)
    return out, torch.empty(out.shape[:3], device=query.device, dtype=torch.float32)


@torch.library.register_fake('aotriton_amd::cache_keep_path')
def _(k_cache, v_cache, page_table, lengths, path, counts):
    return torch.empty_like(lengths)


for _name in ('cache_append', 'cache_copy_pages', 'cache_fork', 'cache_free'):
    torch.library.register_fake('aotriton_amd::' + _name)(lambda *args: None)


def tree_attention(query, k_cache, v_cache, page_table, lengths, parents=None, max_length=None, window=0, sinks=0, scale=None,
                   return_lse=False):
    """Attention of up to 64 drafted tokens per sequence over its cache; with one token, decoding.

    query is (sequences, Hq, tokens, E), Hq a multiple of Hk.  The tokens' own K and V lie in the cache already, token t in slot
    length + t (append).  ``parents`` (int32 (sequences, tokens)): the earlier token that each follows, -1 for those that follow the
    cache; any other value (-2 pads a small tree) says that the token is not there, nor what hangs on it.  Without parents
    every token follows the one before it.  A token sees the filled slots, its ancestors and itself; with a ``window`` > 0
    of these only the last ``window`` by position, itself included, and positions below ``sinks``.  A drafted token's position is
    length + its number of ancestors.  A token that is not there yields zeros (and a logsumexp of +inf); slots that no token
    sees may hold anything, inf and NaN included.

    ``max_length`` bounds the lengths (None: what the page table holds).  It only decides how finely the keys are split over the chip: it
    is a number on the host, so that nothing waits for the device.  Returns (sequences, Hq, tokens, Ev), with return_lse the
    (sequences, Hq, tokens) fp32 logsumexp as well.  No gradient.
    """
    sm_scale = 1.0 / math.sqrt(query.shape[-1]) if scale is None else float(scale)
    if max_length is None:
        max_length = page_table.shape[1] * k_cache.shape[2]
    out, lse = _ops.tree_attention(query, k_cache, v_cache, page_table, lengths, parents, max_length, window, sinks, sm_scale)
    return (out, lse) if return_lse else out


def append(key, value, k_cache, v_cache, page_table, lengths, counts=None):
    """Writes rows t < counts[s] (None: all) of key and value (sequences, Hk, tokens, E) into slots lengths[s] + t.  Lengths stay as
    they are.  The pages have to be there: rows whose slot has none are dropped."""
    _ops.cache_append(key, value, k_cache, v_cache, page_table, lengths, counts)


def copy_pages(k_cache, v_cache, source, target):
    """Makes page target[i] a copy of page source[i] (int32 vectors).  No target may be named twice or be a source of the same call."""
    _ops.cache_copy_pages(k_cache, v_cache, source, target)


def fork(k_cache, v_cache, page_table, lengths, uses, source, target, spare):
    """Makes sequence target[i] a fork of sequence source[i] (int32 vectors): it shares the full pages and gets a copy of the
    last, partial one in page spare[i], which has to be free (and is not looked at where the last page is full or is not there).
    page_table, lengths and uses are updated; what the target's row named before is overwritten, not freed; a source that is not
    there has no fork.  No target may be named twice or be a source of the same call."""
    _ops.cache_fork(k_cache, v_cache, page_table, lengths, uses, source, target, spare)


def keep_path(k_cache, v_cache, page_table, lengths, path, counts):
    """Moves the accepted drafted tokens together: row lengths[s] + path[s][i] to slot lengths[s] + i for i < counts[s], the path ascending
    (int32 (sequences, steps); a count above steps is steps).  Returns the new lengths, lengths + counts, as a new tensor."""
    return _ops.cache_keep_path(k_cache, v_cache, page_table, lengths, path, counts)


def free(page_table, uses, sequences, first, last):
    """Takes columns first[i] <= c < last[i] out of the rows sequences[i] of the table (int32 vectors): they become -1 and the uses of the
    pages that stood there go down by one.  A finished sequence gives up all its columns, one with a window those
    between the sinks and the window."""
    _ops.cache_free(page_table, uses, sequences, first, last)
