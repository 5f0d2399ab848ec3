"""The operators of a transformer's training step with dropout, as cases that can be timed and
checked: attention with dropped probabilities (forward, backward, single tokens against a long
cache), dropout of rows with a residual, and the embedding lookup with its gradient.

``run(state)`` makes one pass through an operator: with ``own`` false in its plain form
(elementary torch operations in 32 bits, rounded once at the end), with ``own`` true through the
framework's kernels.  ``exact(case, seed)`` gives the same outputs from the definitions in 64 bits.

Masks.  No mask is stored: whether a value is dropped is a function of (seed, step, place).  The
generator is Philox4x32 with 7 rounds, the key is the seed, the counter is

* rows (dropout, embedding): element e of the flattened output takes the 16-bit half ``e & 1`` of
  word ``(e >> 1) & 3`` of the block with counter ``(e >> 3, 0, step)`` (64, 32, 32 bits).  It is
  kept where the half is at least ``round(65536 p)``;
* attention: the probability of query i and key j of head h of sequence b takes byte ``j & 3`` of
  word ``i & 3`` of the block with counter ``(j >> 2, i >> 2, b * heads + h, step)``.  It is kept
  where the byte is at least ``round(256 p)``.

What is kept is scaled by the inverse of the share that the threshold keeps.
"""

import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# -- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # GPT-2 small, 8 clients stacked at 4 sequences each: the attention of one layer of a
        # federated training step with attention dropout
        _attn("attn_train_gpt2", 32, 1024, 1024, 12, 12, 64, "bf16", "train", 0.1, packed=True),
        # fine-tuning on right-padded sequences of different lengths, heads that share keys and
        # values, a wider head; one sequence of the batch is empty
        _attn("attn_train_ragged", 6, 777, 777, 16, 4, 128, "fp16", "train", 0.2, ragged=True),
        # a local step on short sequences: latency
        _attn("attn_train_small", 2, 33, 33, 2, 2, 64, "bf16", "train", 0.1, packed=True),
        # held-out evaluation on long sequences: forward only, nothing dropped
        _attn("attn_eval_long", 2, 4096, 4096, 12, 12, 64, "bf16", "fwd", 0.0, packed=True),
        # one new token for each sequence against caches of different lengths
        _attn("attn_token_long", 4, 1, 8191, 32, 8, 128, "bf16", "fwd", 0.0, ragged=True),
        # residual dropout behind a projection of that training step
        _drop("dropout_residual_gpt2", 32768, 768, "bf16", "fwd", 0.1, residual=True),
        # forward and gradient of an odd-sized activation in full precision
        _drop("dropout_odd_fp32", 1237, 1001, "fp32", "train", 0.5),
        # a few rows: latency
        _drop("dropout_rows", 5, 200, "fp16", "train", 0.25, strided=True),
        # GPT-2 small: token and position embedding with dropout and its gradient, tokens as
        # text has them (a few very frequent ones)
        _embed("embed_train_gpt2", 32, 1024, 50257, 768, "bf16", "train", 0.1, zipf=1.0, positions=True),
        # a full-precision table, scaled rows, padding, one client's batch
        _embed("embed_train_fp32", 4, 1000, 32000, 513, "fp32", "train", 0.0, scale=True, padding=True),
        # one step of a short batch: latency
        _embed("embed_train_small", 2, 33, 211, 128, "fp16", "train", 0.1, zipf=1.0, positions=True),
        # the lookup of one token for each of a few sequences
        _embed("embed_tokens", 8, 1, 50257, 768, "bf16", "fwd", 0.0, scale=True),
    ]


def _attn(name, B, Tq, Tk, H, Hk, D, dtype, way, p, ragged=False, packed=False, causal=True):
    return {"name": name, "op": "attention", "B": B, "Tq": Tq, "Tk": Tk, "H": H, "Hk": Hk, "D": D,
            "dtype": dtype, "way": way, "p": p, "ragged": ragged, "packed": packed, "causal": causal}


def _drop(name, R, C, dtype, way, p, residual=False, strided=False):
    return {"name": name, "op": "dropout", "R": R, "C": C, "dtype": dtype, "way": way, "p": p,
            "residual": residual, "strided": strided}


def _embed(name, B, T, V, C, dtype, way, p, zipf=0.0, positions=False, scale=False, padding=False):
    return {"name": name, "op": "embedding", "B": B, "T": T, "V": V, "C": C, "dtype": dtype,
            "way": way, "p": p, "zipf": zipf, "positions": positions, "scale": scale,
            "padding": padding}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "token", "dropout", "embedding"])
    p = rng.choice([0.0, 0.1, rng.uniform(0.01, 0.6)])
    if kind == "attention":
        T = _log(rng, 1, 4096)
        Hk = rng.choice([1, 2, 4, 6, 12])
        H = Hk * rng.choice([1, 1, 2, 4])
        D = rng.choice([32, 64, 64, 80, 128])
        room = 32 * 12 * 1024 * 1024 * 64 // (H * max(T, 64) ** 2 * D)
        B = _log(rng, 1, max(1, min(32, room)))
        ragged = rng.random() < 0.4
        case = _attn("", B, T, T, H, Hk, D, rng.choice(["bf16", "bf16", "fp16"]),
                     rng.choice(["train", "train", "fwd"]), p, ragged=ragged,
                     packed=H == Hk and rng.random() < 0.7, causal=rng.random() < 0.8)
    elif kind == "token":
        Hk = rng.choice([1, 4, 8, 12])
        case = _attn("", _log(rng, 1, 32), rng.choice([1, 1, 2, 5]), _log(rng, 8, 16384),
                     Hk * rng.choice([1, 1, 4, 8]), Hk, rng.choice([64, 128]),
                     rng.choice(["bf16", "fp16"]), "fwd", 0.0, ragged=rng.random() < 0.7)
    elif kind == "dropout":
        C = _log(rng, 1, 4096)
        R = _log(rng, 1, max(1, min(32768, 32768 * 768 // C)))
        residual = rng.random() < 0.5
        case = _drop("", R, C, rng.choice(["bf16", "fp16", "fp32"]),
                     "fwd" if residual else rng.choice(["fwd", "train"]), p or 0.1,
                     residual=residual, strided=rng.random() < 0.3)
    else:
        T = _log(rng, 1, 1024)
        case = _embed("", _log(rng, 1, 32), T, _log(rng, 100, 50257), _log(rng, 8, 768),
                      rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                      rng.choice(["train", "train", "fwd"]), p, zipf=rng.choice([0.0, 1.0, 1.3]),
                      positions=rng.random() < 0.6, scale=rng.random() < 0.4,
                      padding=rng.random() < 0.3)
    del case["name"]
    return case


def _spread(B, T):
    """Lengths of the B sequences of a ragged batch, from none (one of five or more) to all of T."""
    return [0 if B >= 5 and b == 0 else max(1, T * (b + 1) // B) for b in range(B)]


def work(case):
    size = torch.empty(0, dtype=_TYPES[case["dtype"]]).element_size()
    if case["op"] == "attention":
        H, Hk, D, Tq, Tk = case["H"], case["Hk"], case["D"], case["Tq"], case["Tk"]
        keys = _spread(case["B"], Tk) if case["ragged"] else [Tk] * case["B"]
        rows = [min(n, Tq) for n in keys] if case["ragged"] else [Tq] * case["B"]
        pairs = sum(r * n - (r * (r - 1) // 2 if case["causal"] else 0) for r, n in zip(rows, keys))
        once = size * D * (2 * H * sum(rows) + 2 * Hk * sum(keys)) + 4 * H * sum(rows)
        if case["way"] == "fwd":
            return {"bytes": once, "flops": 4 * D * H * pairs}
        # the gradient reads dout and the values above once more and writes dq, dk, dv
        return {"bytes": once + size * D * (2 * H * sum(rows) + 2 * Hk * sum(keys)),
                "flops": 14 * D * H * pairs}
    n = (case["R"] if case["op"] == "dropout" else case["B"] * case["T"]) * case["C"]
    if case["op"] == "dropout":
        passes = 2 + case["residual"] + 2 * (case["way"] == "train")
        return {"bytes": passes * n * size, "flops": passes * n}
    # a looked-up row is read once for each different token at most; the gradient of the whole
    # table is written
    rows = min(case["B"] * case["T"], case["V"])
    there = (rows + case["T"] * case["positions"]) * case["C"] * size
    here = n * size + 8 * case["B"] * case["T"]
    back = here + (case["V"] + case["T"] * case["positions"]) * case["C"] * size
    return {"bytes": there + here + (back if case["way"] == "train" else 0), "flops": 2 * n}


# -- inputs -----------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(t)

    s = {"case": dict(case), "seed": (seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), "step": seed % 1009}
    if case["op"] == "attention":
        B, Tq, Tk, H, Hk, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hk", "D"))
        if case["packed"]:  # one matrix of a projection, queries | keys | values
            qkv, dqkv = normal(B, Tq, 3, H, D), torch.empty(B, Tq, 3, H, D, dtype=t, device=dev)
            s["q"], s["k"], s["v"] = qkv.unbind(2)
            s["dq"], s["dk"], s["dv"] = dqkv.unbind(2)
        else:
            s["q"], s["k"], s["v"] = normal(B, Tq, H, D), normal(B, Tk, Hk, D), normal(B, Tk, Hk, D)
            s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[n]) for n in "qkv")
        s["dout"] = normal(B, Tq, H, D)
        s["out"] = torch.empty(B, Tq, H, D, dtype=t, device=dev)
        s["lse"] = torch.empty(B, H, Tq, device=dev)
        s["q_lengths"] = s["k_lengths"] = None
        if case["ragged"]:
            order = torch.randperm(B, generator=g, device=dev)
            keys = torch.tensor(_spread(B, Tk), dtype=torch.int32, device=dev)[order].contiguous()
            s["k_lengths"], s["q_lengths"] = keys, keys.clamp(max=Tq)
    elif case["op"] == "dropout":
        wide = case["C"] + (8 if case["strided"] else 0)
        s["x"] = normal(case["R"], wide)[:, : case["C"]]
        s["residual"] = normal(case["R"], case["C"]) if case["residual"] else None
        s["dout"] = normal(case["R"], case["C"])
        s["out"], s["dx"] = torch.empty_like(s["dout"]), torch.empty_like(s["dout"])
    else:
        B, T, V, C = (case[k] for k in ("B", "T", "V", "C"))
        s["table"] = normal(V, C, scale=0.02)
        s["positions"] = normal(T, C, scale=0.01) if case["positions"] else None
        # ranks with a share proportional to rank ** -zipf, by the inverse of their distribution
        # (element by element: a running sum of the shares rounds differently from run to run)
        u, z = torch.rand(B * T, generator=g, device=dev, dtype=torch.float64), 1.0 - case["zipf"]
        rank = (u * math.log(V)).exp() if z == 0 else (1 + u * (V**z - 1)) ** (1 / z)
        pick = (rank.long() - 1).clamp(0, V - 1)
        s["tokens"] = torch.randperm(V, generator=g, device=dev)[pick].view(B, T)
        s["padding"] = None
        if case["padding"]:  # sequences end in padding
            s["padding"] = V - 1
            for b, n in enumerate(_spread(B, T)):
                s["tokens"][b, max(n, 1):] = V - 1
        s["scale"] = math.sqrt(C) if case["scale"] else 1.0
        s["dout"] = normal(B, T, C)
        s["out"] = torch.empty(B, T, C, dtype=t, device=dev)
        s["dtable"] = torch.empty(V, C, dtype=t, device=dev)
        s["dpositions"] = torch.empty(T, C, dtype=t, device=dev) if case["positions"] else None
    return s


# -- one pass ---------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "dropout": _own_dropout, "embedding": _own_embedding}[op](state)
    return {"attention": _plain_attention, "dropout": _plain_dropout, "embedding": _plain_embedding}[op](state)


def _own_attention(s):
    from nanofed_amd.ops import attention

    c = s["case"]
    how = dict(causal=c["causal"], q_lengths=s["q_lengths"], k_lengths=s["k_lengths"],
               dropout=c["p"], seed=s["seed"], step=s["step"])
    attention.attention_fwd(s["q"], s["k"], s["v"], s["out"], s["lse"], **how)
    if c["way"] == "fwd":
        return {"out": s["out"], "lse": s["lse"]}
    attention.attention_bwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["dq"], s["dk"],
                            s["dv"], **how)
    return {"out": s["out"], "lse": s["lse"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}


def _own_dropout(s):
    from nanofed_amd.ops import dropout

    c = s["case"]
    how = dict(seed=s["seed"], step=s["step"])
    got = {"out": dropout.dropout_fwd(s["x"], c["p"], residual=s["residual"], out=s["out"], **how)}
    if c["way"] == "train":
        got["dx"] = dropout.dropout_bwd(s["dout"], c["p"], out=s["dx"], **how)
    return got


def _own_embedding(s):
    from nanofed_amd.ops import embedding

    c = s["case"]
    how = dict(scale=s["scale"], dropout=c["p"], seed=s["seed"], step=s["step"])
    got = {"out": embedding.embedding_fwd(s["tokens"], s["table"], s["out"], positions=s["positions"], **how)}
    if c["way"] == "train":
        embedding.embedding_bwd(s["tokens"], s["dout"], s["dtable"], dpositions=s["dpositions"],
                                padding_idx=s["padding"], **how)
        got["dtable"] = s["dtable"]
        if s["dpositions"] is not None:
            got["dpositions"] = s["dpositions"]
    return got


# -- the plain form ---------------------------------------------------------------------------
def _round(c, key):
    """One round of the generator: 32-bit values in 64-bit integers (products wrap)."""
    low = 0xFFFFFFFF
    a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
    return ((b >> 32) & low ^ c[1] ^ key[0], b & low, (a >> 32) & low ^ c[3] ^ key[1], a & low), (
        key[0] + 0x9E3779B9 & low, key[1] + 0xBB67AE85 & low)


def _words(c, seed):
    """The four words of the blocks with counters ``c``, after seven rounds."""
    key = (seed & 0xFFFFFFFF, seed >> 32)
    for _ in range(7):
        c, key = _round(c, key)
    return torch.stack(torch.broadcast_tensors(*c), -1)


def _kept_rows(n, p, s, device):
    """For each of n flattened elements whether it is kept, and what kept ones are scaled by."""
    limit = round(65536 * p)
    block = torch.arange((n + 7) // 8, device=device)
    w = _words((block & 0xFFFFFFFF, block >> 32, torch.zeros_like(block), torch.full_like(block, s["step"])), s["seed"])
    halves = torch.stack([w & 0xFFFF, w >> 16], -1).reshape(-1)[:n]
    return halves >= limit, 65536 / (65536 - limit)


def _kept_pairs(s, B, H, Tq, Tk, p, device):
    """The same for each probability, ``[B, H, Tq, Tk]``."""
    limit = round(256 * p)
    keys = torch.arange((Tk + 3) // 4, device=device)
    rows = torch.arange((Tq + 3) // 4, device=device).view(-1, 1)
    heads = torch.arange(B * H, device=device).view(-1, 1, 1)
    w = _words((keys, rows, heads, torch.full_like(keys, s["step"])), s["seed"])  # [BH, rows, keys, 4]
    w = w.transpose(2, 3).unsqueeze(-1) >> torch.tensor([0, 8, 16, 24], device=device)
    kept = (w & 0xFF) >= limit                                                     # [.., word, keys, byte]
    return kept.reshape(B, H, rows.numel() * 4, keys.numel() * 4)[:, :, :Tq, :Tk], 256 / (256 - limit)


def _plain_attention(s):
    c, dtype = s["case"], s["q"].dtype
    B, Tq, Tk, H, Hk, D = (c[k] for k in ("B", "Tq", "Tk", "H", "Hk", "D"))
    dev = s["q"].device
    q = s["q"].float().transpose(1, 2)
    k, v = (x.float().transpose(1, 2).repeat_interleave(H // Hk, 1) for x in (s["k"], s["v"]))
    none = torch.full((B,), Tk, device=dev)
    keys = (s["k_lengths"] if s["k_lengths"] is not None else none).view(B, 1, 1, 1)
    rows = (s["q_lengths"] if s["q_lengths"] is not None else none * 0 + Tq).view(B, 1, 1, 1)
    i, j = torch.arange(Tq, device=dev).view(1, 1, Tq, 1), torch.arange(Tk, device=dev)
    seen = (i < rows) & (j < keys)
    if c["causal"]:
        seen = seen & (j <= i + keys - rows)
    scale = D ** -0.5
    scores = (torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale).masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    prob = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = prob.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    prob = prob / total.masked_fill(total == 0, 1.0)
    del scores
    kept, up = _kept_pairs(s, B, H, Tq, Tk, c["p"], dev) if c["p"] > 0 else (None, 1.0)
    dropped = prob if kept is None else torch.where(kept, prob * up, 0.0)
    out = torch.matmul(dropped, v)
    got = {"out": out.transpose(1, 2).to(dtype), "lse": lse}
    if c["way"] == "fwd":
        return got
    dout = s["dout"].float().transpose(1, 2)
    dv = torch.matmul(dropped.transpose(-1, -2), dout)
    del dropped
    dprob = torch.matmul(dout, v.transpose(-1, -2).contiguous())
    if kept is not None:
        dprob = torch.where(kept, dprob * up, 0.0)
    dscores = prob * (dprob - (dout * out).sum(-1, keepdim=True)) * scale
    del dprob, prob
    dq = torch.matmul(dscores, k)
    dk = torch.matmul(dscores.transpose(-1, -2), q)
    dk, dv = (x.view(B, Hk, H // Hk, Tk, D).sum(2) for x in (dk, dv))  # heads that share keys
    return got | {n: x.transpose(1, 2).to(dtype) for n, x in (("dq", dq), ("dk", dk), ("dv", dv))}


def _plain_dropout(s):
    c, x = s["case"], s["x"]
    kept, up = _kept_rows(x.numel(), c["p"], s, x.device)
    kept = kept.view(x.shape)
    y = torch.where(kept, x.float() * up, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    got = {"out": y.to(x.dtype)}
    if c["way"] == "train":
        got["dx"] = torch.where(kept, s["dout"].float() * up, 0.0).to(x.dtype)
    return got


def _plain_embedding(s):
    c, tokens, dtype = s["case"], s["tokens"], s["table"].dtype
    x = s["table"][tokens].float() * s["scale"]
    if s["positions"] is not None:
        x = x + s["positions"].float()
    kept, up = None, 1.0
    if c["p"] > 0:
        kept, up = _kept_rows(x.numel(), c["p"], s, x.device)
        kept = kept.view(x.shape)
        x = torch.where(kept, x * up, 0.0)
    got = {"out": x.to(dtype)}
    if c["way"] == "fwd":
        return got
    d = s["dout"].float()
    if kept is not None:
        d = torch.where(kept, d * up, 0.0)
    if s["positions"] is not None:
        got["dpositions"] = d.sum(0).to(dtype)
    if s["padding"] is not None:
        d = torch.where((tokens == s["padding"]).unsqueeze(-1), 0.0, d)
    # frequent tokens make long sums: in 64 bits
    dtable = torch.zeros(s["table"].shape, dtype=torch.float64, device=d.device)
    dtable.index_add_(0, tokens.reshape(-1), d.reshape(-1, c["C"]).double())
    got["dtable"] = (dtable * s["scale"]).to(dtype)
    return got


# -- the definition in 64 bits ----------------------------------------------------------------
def _philox(counter, seed):
    """Words ``[..., 4]`` of the blocks whose four counter words are the arrays ``counter``."""
    x, y, z, w = (np.asarray(a, dtype=np.uint64) for a in counter)
    k, l, cut, half = seed % 2**32, seed // 2**32, np.uint64(2**32 - 1), np.uint64(32)
    for _ in range(7):
        p, q = x * np.uint64(0xD2511F53), z * np.uint64(0xCD9E8D57)
        x, y, z, w = (q >> half) ^ y ^ np.uint64(k), q & cut, (p >> half) ^ w ^ np.uint64(l), p & cut
        k, l = (k + 0x9E3779B9) % 2**32, (l + 0xBB67AE85) % 2**32
    return np.stack(np.broadcast_arrays(x, y, z, w), -1).astype("<u4")


def _factor_rows(n, p, s):
    """What each flattened element is multiplied by, in 64 bits."""
    e = np.arange(-(-n // 8), dtype=np.uint64)
    u = _philox((e % np.uint64(2**32), e // np.uint64(2**32), 0 * e, 0 * e + np.uint64(s["step"])), s["seed"])
    u = np.ascontiguousarray(u).view("<u2").reshape(-1)[:n]
    cut = round(p * 65536)
    return torch.from_numpy(u >= cut).cuda().double() * (65536 / (65536 - cut))


def _factor_pairs(s, b, H, Tq, Tk, p):
    """What each probability of sequence b is multiplied by, ``[H, Tq, Tk]``."""
    h, i, j = np.meshgrid(np.arange(b * H, (b + 1) * H), np.arange(-(-Tq // 4)), np.arange(-(-Tk // 4)), indexing="ij")
    u = np.ascontiguousarray(_philox((j, i, h, 0 * h + s["step"]), s["seed"])).view("u1")
    u = torch.from_numpy(u.reshape(H, i.shape[1], j.shape[2], 4, 4)).cuda()
    u = u.permute(0, 1, 3, 2, 4).reshape(H, i.shape[1] * 4, -1)[:, :Tq, :Tk]
    cut = round(p * 256)
    return (u >= cut).double() * (256 / (256 - cut))


def exact(case, seed):
    s = prepare(case, seed)
    train = case["way"] == "train"
    if case["op"] == "attention":
        return _exact_attention(case, s, train)
    if case["op"] == "dropout":
        f = _factor_rows(s["x"].numel(), case["p"], s).view(s["x"].shape)
        out = s["x"].double() * f + (s["residual"].double() if case["residual"] else 0)
        return {"out": out, "dx": s["dout"].double() * f} if train else {"out": out}
    leaf = s["table"].double().requires_grad_(train)
    pos = s["positions"].double().requires_grad_(train) if case["positions"] else None
    x = torch.nn.functional.embedding(s["tokens"], leaf, padding_idx=s["padding"]) * s["scale"]
    x = x if pos is None else x + pos
    if case["p"] > 0:
        x = x * _factor_rows(x.numel(), case["p"], s).view(x.shape)
    got = {"out": x.detach()}
    if train:
        x.backward(s["dout"].double())
        got["dtable"] = leaf.grad
        if pos is not None:
            got["dpositions"] = pos.grad
    return got


def _exact_attention(case, s, train):
    B, Tq, Tk, H, Hk, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hk", "D"))
    if B * H * Tq * Tk > 5e8:
        return None
    names = ["out", "lse"] + (["dq", "dk", "dv"] if train else [])
    got = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in names}
    got["lse"].fill_(-math.inf)
    for b in range(B):
        n = int(s["k_lengths"][b]) if case["ragged"] else Tk
        m = int(s["q_lengths"][b]) if case["ragged"] else Tq
        if not n or not m:
            continue
        q, k, v = (s[x][b, :r].double().requires_grad_(train) for x, r in (("q", m), ("k", n), ("v", n)))
        group = (m, Hk, H // Hk, D)
        a = torch.einsum("ihgd,jhd->hgij", q.reshape(group), k).reshape(H, m, n) / math.sqrt(D)
        if case["causal"]:  # the last query sees every key
            a = a + torch.full((m, n), -math.inf, dtype=torch.float64, device="cuda").triu(1 + n - m)
        w = torch.softmax(a, -1)
        if case["p"] > 0:
            w = w * _factor_pairs(s, b, H, Tq, Tk, case["p"])[:, :m, :n]
        o = torch.einsum("hgij,jhd->ihgd", w.reshape(Hk, H // Hk, m, n), v).reshape(m, H, D)
        got["out"][b, :m], got["lse"][b, :, :m] = o.detach(), torch.logsumexp(a, -1).detach()
        if train:
            o.backward(s["dout"][b, :m].double())
            got["dq"][b, :m], got["dk"][b, :n], got["dv"][b, :n] = q.grad, k.grad, v.grad
    return got
