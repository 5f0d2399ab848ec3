"""The native GPT-2 step with dropout on the GPU: gradients against autograd with the same masks,
client after client against grouped, captured against eager."""

import pytest
import torch

from nanofed_amd.engine import EngineConfig, FederatedEngine
from nanofed_amd.engine.gpt2_native import GPT2NativeTrainer
from nanofed_amd.parallel import Communicator
from tests import gpt2_dropout_reference as reference

pytestmark = pytest.mark.gpu
KW = dict(vocab_size=1013, n_positions=128, n_embd=192, n_layer=3, n_head=3)
DROP = dict(dropout=0.2, embd_dropout=0.1, resid_dropout=0.1)


def _engine(kw=None, **over):
    cfg = dict(model="gpt2_125m", dataset="synthetic_tokens", num_clients=2, samples_per_client=8,
               batch_size=4, local_epochs=1, seq_len=128, learning_rate=0.05, eval_samples=4,
               backend="native", model_kwargs={**KW, **(DROP if kw is None else kw)})
    cfg.update(over)
    torch.cuda.set_device(0)
    return FederatedEngine(EngineConfig(**cfg), comm=Communicator(device=torch.device("cuda", 0)))


@pytest.mark.parametrize("kw,seq", [(dict(dropout=0.2), 128), (dict(embd_dropout=0.2), 128), (dict(resid_dropout=0.2), 128),
                                    (DROP, 101), (dict(DROP, n_head=6), 64), (dict(n_head=2), 77), (dict(), 50)])
def test_gradients_match_autograd_with_the_same_masks(kw, seq):
    eng = _engine(kw, seq_len=seq)
    tr = eng.trainer
    assert isinstance(tr, GPT2NativeTrainer)
    eng.pool.broadcast_from(eng.global_arena.data)
    toks = eng.shards.inputs[:4]
    for k, step in ((0, 0), (1, 5)):
        loss, grads = tr.loss_and_grads(k, toks, step)
        want, named = reference.loss_and_grads(eng, tr.m, toks, step, k)
        assert abs(loss - want) < 1e-2 * abs(want)
        for name, g in grads.items():
            err = float((g.float() - named[name]).norm() / (named[name].norm() + 1e-8))
            assert err < 6e-2, (name, err)


def test_grouped_steps_train_the_same_model_as_client_after_client(monkeypatch):
    """The same masks whichever clients share a launch (another order of the GEMMs' sums only)."""
    from nanofed_amd.engine import gpt2_native

    outs = []
    for group in (0, 8, 2):
        monkeypatch.setattr(gpt2_native, "GROUP", group)
        eng = _engine(num_clients=3, samples_per_client=8, learning_rate=0.1)
        assert eng.trainer.group == min(group, 3)
        reps = [eng.run_round() for _ in range(2)]
        torch.cuda.synchronize()
        outs.append((eng.global_arena.data.clone(), [r.agg_metrics["loss"] for r in reps]))
    init = _engine(num_clients=3, samples_per_client=8).global_arena.data
    for data, losses in outs[1:]:
        assert losses == pytest.approx(outs[0][1], rel=2e-3)
        a, b = outs[0][0] - init, data - init
        assert float(torch.dot(a, b) / (a.norm() * b.norm())) > 0.995


def test_captured_steps_equal_the_eager_ones_bit_for_bit(monkeypatch):
    """The masks of a replayed graph follow the step number in device memory: three rounds of four
    steps, in one group and in chunks of 2 + 1 clients."""
    from nanofed_amd.engine import gpt2_native

    for group in (8, 2):
        monkeypatch.setattr(gpt2_native, "GROUP", group)
        outs = []
        for capture in (False, True):
            eng = _engine(num_clients=3, samples_per_client=16, learning_rate=0.1, graph_capture=capture)
            reps = [eng.run_round() for _ in range(3)]
            torch.cuda.synchronize()
            assert len(eng.trainer._step_graphs) == ((1 if group == 8 else 2) if capture else 0)
            outs.append((eng.global_arena.data.clone(), [r.agg_metrics["loss"] for r in reps]))
        assert outs[0][1] == outs[1][1]
        assert torch.equal(outs[0][0], outs[1][0])


def test_evaluation_draws_no_masks_and_auto_stays_with_torch():
    a, b = _engine(), _engine({})
    assert a.evaluate() == b.evaluate()
    assert _engine(backend="auto").backend == "torch"
    assert _engine({}, backend="auto").backend == "native"
