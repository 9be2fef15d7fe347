"""Rows of the tables of states that steps name by their `slots` (CUDA, `csrc/ttt_tables.cu`): convolution windows, scan states, the TTT operators'
weights of each sequence.

    copy_rows((windows, states), source, target)      # fork a sequence, or let rows change places
    clear_rows((windows, states), rows)               # a new sequence's empty states
    place = compact_rows((windows, states), used)     # the used rows in front of the tables

Tables [S, ...] are contiguous, of any types, all of a call (up to 16) with the same number of rows; they change in place, in one launch.  Calls are
stream-ordered and do not synchronise, so that the rows may be worked out on the GPU, in tensors that are none of the tables.  A backward that has kept rows
of a table from before such a call refuses, as after any change in place.  A bad argument raises ValueError.
"""
import torch

from . import ssm


def _tables(tables):
    if isinstance(tables, torch.Tensor):
        return (tables,)
    if not isinstance(tables, (tuple, list)):
        raise ValueError(f"tables must be a tensor or a list of tensors, got {type(tables).__name__}")
    return tuple(tables)


def copy_rows(tables, source, target):
    """table[target[i]] = table[source[i]] for each pair, all rows read before one is written: rows may change places.  `source`, `target`: int32 [n], n at
    most 4096.  A pair with an index that is no row does nothing; of several pairs with the same target the last one counts."""
    ssm._host().copy_rows(_tables(tables), source, target)


def clear_rows(tables, rows):
    """Zeros in the rows `rows`, int32 [n], n at most 4096; an index that is no row does nothing."""
    ssm._host().clear_rows(_tables(tables), rows)


def compact_rows(tables, used):
    """Moves the rows in use, `used` bool [S] (S at most 8192), in front of all others: with n of them, the k-th used row from row n on takes the place of the k-th
    free row in front of it, and no other row moves.  What was there is left behind.  Returns int32 [S]: where each used row is now, -1
    for the others."""
    return ssm._host().compact_rows(_tables(tables), used)
