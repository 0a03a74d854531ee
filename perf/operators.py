"""Timed cases of the 8-bit integer Linear and of token scores, in plain torch and through the package.

* ``linear`` -- a quantized Linear whose activations are quantized too: every row of
  ``x`` gets a scale and int8 codes, the codes meet the weight's int8 codes in an
  integer product, and the sums take the row's scale, the channel's scale and the
  bias: ``y = (sum_k q_x q_w) s_x s_w + b``;
* ``score``  -- log probabilities of given tokens under rows of logits, the entropy of
  each row and its most probable alternatives;
* ``grad``   -- the same scores with the gradient that they send to the logits, as one
  training step asks for it.

Widths and the vocabulary are GPT-2's (768, 1024, 1280, 1600; 50257) or generic.
``run`` computes the plain form, or with ``own`` the package's calls; ``exact`` is
the definition in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

WIDTHS = (768, 1024, 1280, 1600)
VOCAB = 50257
#: the four Linears of a block as (inputs, outputs) in units of the width
LINEARS = ((1, 3), (1, 1), (1, 4), (4, 1))
#: the most work a drawn case may ask for: the largest listed ones
MAX_PRODUCT = 8192 * 6400 * 1600
MAX_LOGITS = 4096 * VOCAB
IGNORED = -100
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _package():
    root = str(Path(__file__).resolve().parents[1] / "gpt2-harness_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gpt2_harness_amd

    return gpt2_harness_amd


def listed() -> list[dict]:
    return [
        # the smallest call: one decode row through GPT-2 small's c_attn
        {"name": "linear-1", "op": "linear", "rows": 1, "k": 768, "n": 2304, "bias": True, "dtype": "fp32"},
        # a small serving batch through GPT-2-XL's widest Linear
        {"name": "linear-16", "op": "linear", "rows": 16, "k": 1600, "n": 6400, "bias": True, "dtype": "bf16"},
        # a short prompt through a matrix of odd sizes, no bias
        {"name": "linear-77-odd", "op": "linear", "rows": 77, "k": 1001, "n": 777, "bias": False, "dtype": "fp32"},
        # one long prompt of odd length, GPT-2 medium's c_fc
        {"name": "linear-1001", "op": "linear", "rows": 1001, "k": 1024, "n": 4096, "bias": True, "dtype": "fp32"},
        # 32 prompts of 128 tokens, GPT-2-XL's c_attn
        {"name": "linear-4096", "op": "linear", "rows": 4096, "k": 1600, "n": 4800, "bias": True, "dtype": "bf16"},
        # the largest batch: 64 prompts of 128 tokens, GPT-2-XL's long product
        {"name": "linear-8192", "op": "linear", "rows": 8192, "k": 6400, "n": 1600, "bias": True, "dtype": "fp32"},
        # generation: the next token's row, the five best alternatives beside it
        {"name": "score-1", "op": "score", "rows": 1, "vocab": VOCAB, "top": 5, "dtype": "fp32"},
        # one step of a serving batch, twenty alternatives a sequence, a wider vocabulary
        {"name": "score-64-wide", "op": "score", "rows": 64, "vocab": 131071, "top": 20, "dtype": "bf16"},
        # the perplexity evaluation: four windows of 1024 tokens
        {"name": "score-4096", "op": "score", "rows": 4096, "vocab": VOCAB, "top": 5, "dtype": "fp32"},
        # a distilled model's small vocabulary, many short rows, no alternatives
        {"name": "score-5000-small", "op": "score", "rows": 5000, "vocab": 1003, "top": 0, "dtype": "bf16"},
        # a fine-tuning step on one short sequence
        {"name": "grad-96", "op": "grad", "rows": 96, "vocab": VOCAB, "top": 0, "dtype": "fp32"},
        # a fine-tuning step over a batch of padded sequences
        {"name": "grad-4096", "op": "grad", "rows": 4096, "vocab": VOCAB, "top": 0, "dtype": "bf16"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng) -> dict:
    op = rng.choice(("linear", "linear", "score", "grad"))
    dtype = rng.choice(("fp32", "bf16"))
    if op == "linear":
        if rng.random() < 0.6:  # one of GPT-2's matrices
            (ki, ni), width = rng.choice(LINEARS), rng.choice(WIDTHS)
            k, n = ki * width, ni * width
        else:  # any matrix
            k, n = _log_int(rng, 17, 6400), _log_int(rng, 1, 6400)
        return {"op": op, "rows": _log_int(rng, 1, min(8192, MAX_PRODUCT // (k * n))), "k": k, "n": n,
                "bias": rng.random() < 0.7, "dtype": dtype}
    vocab = VOCAB if rng.random() < 0.5 else _log_int(rng, 33, 160000)
    return {"op": op, "rows": _log_int(rng, 1, min(8192, MAX_LOGITS // vocab)), "vocab": vocab,
            "top": rng.choice((0, 1, 5, 20)) if op == "score" else 0, "dtype": dtype}


# ------------------------------------------------------------------ inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=gen, device="cuda")


def _coded_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """int8 codes (as fp32 values) and scales of each row of ``x``: the largest
    magnitude is 127, a scale is never below the smallest normal number. (127 as a
    tensor: torch divides by a Python number as a product with its reciprocal.)"""
    x = x.float()
    scale = (x.abs().amax(dim=1, keepdim=True) / x.new_full((), 127.0)).clamp(min=1.17549435e-38)
    return torch.round(x / scale).clamp(-128.0, 127.0), scale


def _linear_inputs(case: dict, seed: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """LayerNorm-like rows (one column in 256 eight times larger, as a trained
    model has them) and a weight of GPT-2's initial distribution as codes."""
    gen, m, k, n = _gen(seed), case["rows"], case["k"], case["n"]
    x = _normal(gen, m, k)
    x[:, torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 256)]] *= 8.0
    codes, scale = _coded_rows(_normal(gen, n, k) * 0.02)
    bias = _normal(gen, n) * 0.1 if case["bias"] else None
    return x.to(DTYPES[case["dtype"]]), codes.to(torch.int8), scale.reshape(-1), bias


def _score_inputs(case: dict, seed: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of logits from flat to nearly certain, and the token that each row
    is asked for: its likeliest one in two rows of three, else any token."""
    gen, m, v = _gen(seed), case["rows"], case["vocab"]
    spread = 1.0 + 2.0 * torch.rand(m, 1, generator=gen, device="cuda")
    logits = _normal(gen, m, v) * spread - 5.0
    best = torch.randint(0, v, (m, 1), generator=gen, device="cuda")
    logits.scatter_add_(1, best, 5.0 + 12.0 * torch.rand(m, 1, generator=gen, device="cuda"))
    other = torch.randint(0, v, (m,), generator=gen, device="cuda")
    tokens = torch.where(torch.rand(m, generator=gen, device="cuda") < 2 / 3, best[:, 0], other)
    if case["op"] == "grad":  # padding at the ends of a batch's sequences
        tokens = torch.where(torch.rand(m, generator=gen, device="cuda") < 0.1, IGNORED, tokens)
    return logits.to(DTYPES[case["dtype"]]), tokens


def _score_grads(case: dict, seed: int) -> tuple[torch.Tensor, torch.Tensor]:
    """What a loss sends back: a weight for each token's log probability (an
    advantage, a mean's share) and one for each row's entropy (a bonus)."""
    gen, m = _gen(seed + 1_000_003), case["rows"]
    return _normal(gen, m) / m, _normal(gen, m) * (0.01 / m)


def prepare(case: dict, seed: int) -> dict:
    state = {"op": case["op"]}
    if case["op"] == "linear":
        x, codes, scale, bias = _linear_inputs(case, seed)
        state["x"] = x
        if own:
            state["linear"] = _package().QuantLinear(codes, scale, bias, case["k"], case["n"], 8, "per_channel", "w8a8")
        else:
            state.update(codes=codes, scale=scale, bias=bias)
        return state
    state["logits"], state["tokens"] = _score_inputs(case, seed)
    state["top"] = case["top"]
    if own:
        state["token_logprobs"] = _package().token_logprobs
    if case["op"] == "grad":
        state["grads"] = _score_grads(case, seed)
        if own:
            state["logits"].requires_grad_()
    return state


# --------------------------------------------------------------- plain forms
def _plain_linear(state: dict) -> torch.Tensor:
    x = state["x"]
    q, s = _coded_rows(x)
    y = (q @ state["codes"].float().t()) * s * state["scale"]
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(x.dtype)


def _plain_scores(logits: torch.Tensor, tokens: torch.Tensor, top: int):
    z = logits.float()
    z = z - z.amax(dim=1, keepdim=True)
    e = z.exp()
    total = e.sum(dim=1, keepdim=True)
    logp = z - total.log()
    p = e / total
    entropy = -(p * logp).sum(dim=1)
    seen = tokens != IGNORED
    chosen = logp.gather(1, torch.where(seen, tokens, 0).unsqueeze(1)).squeeze(1)
    chosen = torch.where(seen, chosen, 0.0)
    ids, values = [], []
    if top:
        place = torch.arange(z.shape[1], device=z.device)
        left = logits.float().clone()
        for _ in range(min(top, z.shape[1])):  # the largest that is left, the lowest index of equal logits
            best = left.amax(dim=1, keepdim=True)
            at = torch.where(left == best, place, z.shape[1]).amin(dim=1, keepdim=True)
            left.scatter_(1, at, float("-inf"))
            ids.append(at)
            values.append(logp.gather(1, at))
    return chosen, entropy, logp, p, ids, values


def _plain_score(state: dict):
    chosen, entropy, _, _, ids, values = _plain_scores(state["logits"], state["tokens"], state["top"])
    if not ids:
        return chosen, entropy
    return chosen, entropy, torch.cat(ids, dim=1), torch.cat(values, dim=1)


def _plain_grad(state: dict):
    logits, tokens = state["logits"], state["tokens"]
    chosen, entropy, logp, p, _, _ = _plain_scores(logits, tokens, 0)
    seen = tokens != IGNORED
    g_chosen, g_entropy = (g.unsqueeze(1) for g in state["grads"])
    g_chosen = torch.where(seen.unsqueeze(1), g_chosen, 0.0)
    hot = torch.arange(p.shape[1], device=p.device) == tokens.unsqueeze(1)
    grad = g_chosen * (hot.float() - p) - g_entropy * p * (logp + entropy.unsqueeze(1))
    return chosen, entropy, grad.to(logits.dtype)


def run(state: dict):
    if not own:
        return {"linear": _plain_linear, "score": _plain_score, "grad": _plain_grad}[state["op"]](state)
    if state["op"] == "linear":
        return state["linear"](state["x"])
    scores = state["token_logprobs"](state["logits"], state["tokens"], top=state["top"])
    if state["op"] == "grad":
        (grad,) = torch.autograd.grad((scores.logprob, scores.entropy), state["logits"], state["grads"])
        return scores.logprob.detach(), scores.entropy.detach(), grad
    if not state["top"]:
        return scores.logprob, scores.entropy
    return scores.logprob, scores.entropy, scores.top_ids, scores.top_logprobs


# ------------------------------------------------------------------- 64 bits
def _exact_linear(case: dict, seed: int) -> torch.Tensor:
    x, codes, scale, bias = _linear_inputs(case, seed)
    x = x.double()
    # a scale and a code's quotient are fp32 numbers by definition: 64-bit
    # quotients of fp32 numbers, rounded to fp32, are the rounded quotients
    s = (x.abs().max(dim=1).values / x.new_full((), 127.0)).float().clamp_min(torch.finfo(torch.float32).tiny).double()
    q = (x / s[:, None]).float().double().round().clamp(-128, 127)
    y = torch.matmul(q, codes.double().t()) * torch.outer(s, scale.double())
    return y if bias is None else y + bias.double()


def _exact_scores(case: dict, seed: int):
    logits, tokens = _score_inputs(case, seed)
    wants_grad = case["op"] == "grad"
    z = logits.double().requires_grad_(wants_grad)
    logp = torch.log_softmax(z, dim=1)
    entropy = -(logp.exp() * logp).sum(dim=1)
    seen = tokens != IGNORED
    chosen = logp[torch.arange(len(tokens), device=z.device), tokens.clamp_min(0)] * seen
    if wants_grad:
        g_chosen, g_entropy = _score_grads(case, seed)
        ((chosen * g_chosen.double()).sum() + (entropy * g_entropy.double()).sum()).backward()
        return chosen.detach(), entropy.detach(), z.grad
    if not case["top"]:
        return chosen, entropy
    values, ids = logits.double().sort(dim=1, descending=True, stable=True)
    k = min(case["top"], case["vocab"])
    ids = ids[:, :k].contiguous()
    return chosen, entropy, ids, logp.gather(1, ids)


def exact(case: dict, seed: int):
    return _exact_linear(case, seed) if case["op"] == "linear" else _exact_scores(case, seed)


# ---------------------------------------------------------------------- work
def work(case: dict) -> dict:
    size = {"fp32": 4, "bf16": 2}[case["dtype"]]
    m = case["rows"]
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        return {"bytes": m * k * size + n * k + n * (8 if case["bias"] else 4) + m * n * size, "flops": 2 * m * n * k}
    v = case["vocab"]
    if case["op"] == "score":
        return {"bytes": m * v * size + m * (16 + 12 * min(case["top"], v)), "flops": 6 * m * v}
    return {"bytes": 2 * m * v * size + m * 24, "flops": 12 * m * v}
