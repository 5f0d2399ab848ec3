"""Calls of the attention, dropout and embedding operators that would give a wrong result without a word."""

import pytest
import torch

from nanofed_amd.core.exceptions import DeviceError
from nanofed_amd.ops import attention as A
from nanofed_amd.ops import dropout as D
from nanofed_amd.ops import embedding as E
from tests.unit.test_gpt2_dropout_cpu import _engine


def test_tensors_that_autograd_would_follow_are_refused():
    q, x = torch.zeros(1, 4, 2, 8), torch.zeros(4, 8)
    lse, tok = torch.zeros(1, 2, 4), torch.zeros(4, dtype=torch.int64)
    leaf = torch.zeros(1, 4, 2, 8, requires_grad=True)
    row = torch.zeros(4, 8, requires_grad=True)
    calls = [
        lambda: A.attention_fwd(leaf, q, q), lambda: A.attention_fwd(q, leaf, q), lambda: A.attention_fwd(q, q, leaf * 2),
        lambda: A.attention_bwd(q, q, q, q, lse, leaf, q.clone(), q.clone(), q.clone()),
        lambda: A.attention_bwd(leaf, q, q, q, lse, q, q.clone(), q.clone(), q.clone()),
        lambda: D.dropout_fwd(row, 0.5, seed=1), lambda: D.dropout_fwd(x, 0.5, seed=1, residual=row),
        lambda: D.dropout_bwd(row, 0.5, seed=1),
        lambda: E.embedding_fwd(tok, row), lambda: E.embedding_fwd(tok, x, positions=row),
        lambda: E.embedding_bwd(tok, row, x.clone()),
    ]
    for call in calls:
        with pytest.raises(DeviceError, match="autograd does not record"):
            call()
        with torch.no_grad():
            call()


def test_a_dropout_that_would_drop_nothing_is_refused():
    q, x, tok = torch.zeros(1, 4, 2, 8), torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for p in (0.0019, 1e-9):
        with pytest.raises(DeviceError, match="would drop nothing"):
            A.attention_fwd(q, q, q, dropout=p)
    for call in (lambda p: D.dropout_fwd(x, p, seed=1), lambda p: E.embedding_fwd(tok, x, dropout=p),
                 lambda p: E.embedding_bwd(tok, x, x.clone(), dropout=p)):
        with pytest.raises(DeviceError, match="would drop nothing"):
            call(7e-6)
        call(8e-6)
        call(0.0)
    A.attention_fwd(q, q, q, dropout=0.002)
    with pytest.raises(DeviceError, match="would drop nothing"):
        _engine(dict(dropout=0.001))
    _engine(dict(resid_dropout=0.001))


def test_masks_that_would_repeat_are_refused():
    """The sequence and head are 32 bits of the mask's counter."""
    q = torch.zeros(2, 4, 4, 8)
    how = dict(dropout=0.5, seed=1)
    A.attention_fwd(q, q, q, first_batch=(1 << 30) - 2, **how)
    for first in ((1 << 30) - 1, 1 << 30, (1 << 32) - 1):
        with pytest.raises(DeviceError, match="first_batch"):
            A.attention_fwd(q, q, q, first_batch=first, **how)


def test_tokens_of_a_table_without_rows_are_refused_both_ways():
    """(the gradient left that of the positions as it was)"""
    tok, none, pos = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(0, 4), torch.full((3, 4), 7.0)
    with pytest.raises(DeviceError, match="no rows"):
        E.embedding_fwd(tok, none)
    with pytest.raises(DeviceError, match="no rows"):
        E.embedding_bwd(tok, torch.ones(2, 3, 4), none, dpositions=pos)
    E.embedding_bwd(tok[:0], torch.ones(0, 3, 4), none, dpositions=pos)
    assert bool((pos == 0).all())
