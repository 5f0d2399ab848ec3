"""Calls of the attention, dropout and embedding operators that would give a wrong result without a word."""

import pytest
import torch

from nanofed_amd.core.exceptions import DeviceError
from nanofed_amd.ops import attention as A
from nanofed_amd.ops import dropout as D
from nanofed_amd.ops import embedding as E


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
