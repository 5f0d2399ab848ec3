"""GPT-2's loss in float32 PyTorch with given dropout masks, differentiable: what the native
trainer's step with dropout is compared with."""

import math

import torch
import torch.nn.functional as F

from nanofed_amd.ops.dropout import site_seed
from tests import transformer_oracles as oracle


def loss(params, cfg, tokens, *, seed, step, client, mask_device="cpu"):
    """Mean next-token loss of ``tokens`` ``[B, T + 1]``; ``params``: name -> leaf tensor."""
    inp, tgt = tokens[:, :-1], tokens[:, 1:]
    B, T = inp.shape
    C, H = cfg.n_embd, cfg.n_head

    def rows(x, p, *site):
        if not p:
            return x
        f = oracle.row_factor(x.numel(), p, site_seed(seed, *site), step, client * x.numel())
        return x * f.view(x.shape).to(x)

    x = params["wte.weight"][inp] + params["wpe.weight"][:T]
    x = rows(x, cfg.embd_dropout, "embd")
    seen = torch.ones(T, T, dtype=torch.bool, device=x.device).tril()
    for l in range(cfg.n_layer):
        def get(name):
            return params[f"h.{l}.{name}"]

        h = F.layer_norm(x, (C,), get("ln_1.weight"), get("ln_1.bias"))
        q, k, v = F.linear(h, get("attn.c_attn.weight"), get("attn.c_attn.bias")).view(B, T, 3, H, C // H).unbind(2)
        s = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(-1, -2).contiguous()) / math.sqrt(C // H)
        w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
        if cfg.dropout:
            w = w * oracle.pair_factor(B, H, T, T, cfg.dropout, site_seed(seed, "attn", l), step, client * B).to(w)
        y = (w @ v.transpose(1, 2)).transpose(1, 2).reshape(B, T, C)
        x = x + rows(F.linear(y, get("attn.c_proj.weight"), get("attn.c_proj.bias")), cfg.resid_dropout, "attn_proj", l)
        h = F.layer_norm(x, (C,), get("ln_2.weight"), get("ln_2.bias"))
        h = F.gelu(F.linear(h, get("c_fc.weight"), get("c_fc.bias")), approximate="tanh")
        x = x + rows(F.linear(h, get("c_proj.weight"), get("c_proj.bias")), cfg.resid_dropout, "proj", l)
    x = F.layer_norm(x, (C,), params["ln_f.weight"], params["ln_f.bias"])
    logits = F.linear(x, params["wte.weight"])
    return F.cross_entropy(logits.reshape(-1, logits.shape[-1]), tgt.reshape(-1))


def loss_and_grads(engine, cfg, tokens, step, k=0):
    """The same for client k of an engine whose weights the trainer rounds to bf16."""
    state = {n: v.to(torch.bfloat16).float().to(tokens.device) for n, v in engine.global_state_dict().items()}
    params = {n: v.clone().requires_grad_(True) for n, v in state.items()}
    out = loss(params, cfg, tokens, seed=engine.cfg.seed, step=step, client=engine.shards.client_ids[k])
    out.backward()
    return float(out.detach()), {n: p.grad for n, p in params.items()}
