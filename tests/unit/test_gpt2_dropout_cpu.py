"""The native GPT-2 trainer with dropout (PyTorch paths of the operations) against autograd with
the same masks."""

import pytest
import torch

from nanofed_amd.core.exceptions import DeviceError
from nanofed_amd.engine import EngineConfig, FederatedEngine
from nanofed_amd.engine.gpt2_native import GPT2NativeTrainer
from nanofed_amd.models import GPT2Config, GPT2LM
from nanofed_amd.ops.dropout import site_seed
from nanofed_amd.parallel import Communicator
from tests import gpt2_dropout_reference as reference

KW = dict(vocab_size=211, n_positions=40, n_embd=128, n_layer=2, n_head=2)
DROP = dict(dropout=0.2, embd_dropout=0.1, resid_dropout=0.3)


def _engine(kw=None, **over):
    cfg = dict(model="gpt2_125m", dataset="synthetic_tokens", num_clients=2, samples_per_client=4,
               batch_size=2, local_epochs=1, seq_len=33, learning_rate=0.05, eval_samples=2,
               backend="native", model_kwargs={**KW, **(DROP if kw is None else kw)})
    cfg.update(over)
    return FederatedEngine(EngineConfig(**cfg), comm=Communicator())


@pytest.mark.parametrize("kw", [dict(dropout=0.2), dict(embd_dropout=0.2), dict(resid_dropout=0.2), DROP,
                                dict(DROP, n_head=4), dict(n_head=8)])
def test_loss_and_gradients_match_autograd_with_the_same_masks(kw):
    eng = _engine(kw)
    assert isinstance(eng.trainer, GPT2NativeTrainer)
    eng.pool.broadcast_from(eng.global_arena.data)
    toks = eng.shards.inputs[:2]
    for k, step in ((0, 0), (1, 7)):
        loss, grads = eng.trainer.loss_and_grads(k, toks, step)
        want, named = reference.loss_and_grads(eng, eng.trainer.m, toks, step, k)
        assert abs(loss - want) < 2e-2 * abs(want)
        for name, g in grads.items():
            err = float((g.float() - named[name]).norm() / (named[name].norm() + 1e-8))
            assert err < 5e-2, (name, err)


def test_steps_and_clients_draw_different_masks_and_evaluation_none():
    eng, plain = _engine(), _engine({})
    eng.pool.broadcast_from(eng.global_arena.data)
    toks = eng.shards.inputs[:2]
    losses = {(k, n): eng.trainer.loss_and_grads(k, toks, n)[0] for k in (0, 1) for n in (0, 1)}
    assert len(set(losses.values())) == 4
    assert eng.trainer.loss_and_grads(0, toks, 1)[0] == losses[0, 1]
    assert eng.evaluate() == plain.evaluate()
    a, b = eng.run_round(), plain.run_round()
    assert a.status == b.status == "COMPLETED" and a.agg_metrics["loss"] != b.agg_metrics["loss"]


def test_rounds_are_a_function_of_the_seed():
    runs = []
    for seed in (0, 0, 1):
        eng = _engine(seed=seed)
        runs.append([eng.run_round().agg_metrics["loss"] for _ in range(2)])
    assert runs[0] == runs[1] != runs[2]


def test_torch_model_drops_in_training_only():
    torch.manual_seed(0)
    model = GPT2LM(GPT2Config(**KW, **DROP))
    toks = torch.randint(0, 211, (2, 20))
    assert not torch.equal(model(toks), model(toks))
    model.eval()
    assert torch.equal(model(toks), model(toks))


def test_refusals():
    for kw in (dict(dropout=1.0), dict(embd_dropout=-0.5), dict(resid_dropout=1.5)):
        with pytest.raises(DeviceError, match="in \\[0, 1\\)"):
            _engine(kw)
    with pytest.raises(DeviceError, match="head dimension"):
        _engine(dict(n_embd=120, n_head=10))


def test_site_seeds_differ_by_run_layer_and_kind():
    seeds = {site_seed(s, kind, l) for s in (0, 1) for kind in ("attn", "proj") for l in (0, 1)}
    assert len(seeds) == 8 and all(0 <= s < 1 << 64 for s in seeds)


def test_a_short_batch_draws_the_first_masks_of_its_clients_own_range():
    """Client 1 with one sequence drops what it drops in the first sequence of a full batch."""
    eng = _engine(dict(embd_dropout=0.5, n_layer=1))
    eng.pool.broadcast_from(eng.global_arena.data)
    toks = eng.shards.inputs[:2]
    tr, kept = eng.trainer, []
    for n in (2, 1):
        tr.loss_and_grads(1, toks[:n], 3)
        kept.append(tr._buffers(n, toks.shape[1] - 1).x[0].clone())
    assert torch.equal(kept[0][: len(kept[1])], kept[1]) and (kept[1] == 0).any()


def test_step_numbers_do_not_depend_on_the_shards_of_the_rank():
    a, b = _engine(local_epochs=2), _engine(local_epochs=2, samples_per_client=10)
    at = [(r, e, s) for r in range(40) for e in range(2) for s in range(50)]
    numbers = [a.trainer._step_number(*x) for x in at]
    assert numbers == [b.trainer._step_number(*x) for x in at]
    assert len(set(numbers)) == len(at)
