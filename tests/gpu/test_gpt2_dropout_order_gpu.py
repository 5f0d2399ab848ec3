"""The captured GPT-2 step with embedding dropout takes the token order that the host made with the batch."""

import pytest
import torch

from nanofed_amd.engine import gpt2_native
from tests.gpu.test_gpt2_dropout_gpu import _engine

pytestmark = pytest.mark.gpu


def test_captured_steps_do_not_sort_the_tokens_again(monkeypatch):
    given, made = [], gpt2_native.embed_ops.embedding_bwd

    def recorded(tokens, *args, order=None, **how):
        given.append(order)
        return made(tokens, *args, order=order, **how)

    monkeypatch.setattr(gpt2_native.embed_ops, "embedding_bwd", recorded)
    ends = []
    for capture in (True, False):
        given.clear()
        eng = _engine(num_clients=3, samples_per_client=16, learning_rate=0.1, graph_capture=capture)
        losses = [eng.run_round().agg_metrics["loss"] for _ in range(2)]
        torch.cuda.synchronize()
        assert given and all((order is not None) == capture for order in given)
        ends.append((losses, eng.global_arena.data.clone()))
    assert ends[0][0] == ends[1][0] and torch.equal(ends[0][1], ends[1][1])
