"""Token scores (``token_logprobs``) and their gradient against 64 bits.

Bounds, with u = 2^-24 (half a step of fp32) and A = sum_j e_j |z_j| / sum_j e_j:
z = x - m is rounded once, and a term e = exp(z) follows it by |z| u, takes at most
|z| u more in exp's argument and 2 u in exp itself; a sum of V terms in at least 256
strands adds (V / 256 + 16) u. So the sum d of the terms has a relative error of at
most D = (2 A + 2 + V / 256 + 16) u, and
  log p: |z| u + D d / (1 + d) + 4 u log1p(d) + u |log p|;
  H:     D d / (1 + d) + 4 u log1p(d) for its first part, and for the second, a
         quotient of two sums of the same kind whose terms e z weigh |z| once
         more, (2 B + (3 + V / 256 + 16) A) u + D A with B = sum_j e_j z_j^2 / sum_j e_j.
Logits are fp32 or bf16 numbers, exact in either.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

import gpt2_harness_amd as g
from gpt2_harness_amd import _lib
from gpt2_harness_amd.scoring import MAX_TOP

pytestmark = pytest.mark.gpu

FP32, BF16 = torch.float32, torch.bfloat16
U = 2.0**-24


def _logits(rows, v, seed, dtype=FP32, boost=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=gen) * (1.0 + 2.0 * torch.rand(rows, 1, generator=gen)) - 5.0
    if boost:  # from flat rows to nearly certain ones
        x[torch.arange(rows), torch.randint(0, v, (rows,), generator=gen)] += 20.0 * torch.rand(rows, generator=gen)
    tokens = torch.randint(0, v, (rows,), generator=gen)
    best = x.argmax(dim=1)
    return x.to(dtype), torch.where(torch.arange(rows) % 2 == 0, best, tokens)


def _reference(x, tokens):
    """log p of every token, entropy, d, and the bounds' ingredients, in 64 bits."""
    z = x.double() - x.double().amax(dim=1, keepdim=True)
    e = z.exp()
    s = e.sum(dim=1)
    zf = torch.where(e > 0, z, 0.0)
    # without the row's maximum: exact where 1 + d would lose it
    rest = e.clone()
    rest[torch.arange(len(x)), x.double().argmax(dim=1)] = 0.0
    d = rest.sum(dim=1)
    logp = z - torch.log1p(d)[:, None]
    entropy = torch.log1p(d) - (e * zf).sum(dim=1) / s
    A = (e * zf.abs()).sum(dim=1) / s
    B = (e * zf * zf).sum(dim=1) / s
    return z, logp, entropy, d, A, B


def _bounds(x, z, logp, d, A, B):
    n = x.shape[1] / 256 + 16
    S = (2 * A + (2 + n) * d / (1 + d)) * U
    L = torch.log1p(d)
    base = S + 4 * U * L
    zf = torch.where(torch.isfinite(z), z, 0.0)
    lp = zf.abs() * U + base[:, None] + U * torch.where(torch.isfinite(logp), logp, 0.0).abs() + 1e-44
    h = base + (2 * B + (3 + n) * A) * U + S * A + 2 * U * (L + A) + 1e-44
    return lp, h


def _check(out, x, tokens, top, ignore=-100):
    """``out`` (TokenScores of 2-D ``x`` on the CPU) against 64 bits."""
    z, logp, entropy, d, A, B = _reference(x, tokens)
    blp, bh = _bounds(x, z, logp, d, A, B)
    seen = tokens != ignore
    at = torch.where(seen, tokens, 0)[:, None]
    want = torch.where(seen, logp.gather(1, at)[:, 0], 0.0)
    got = out.logprob.double().cpu().reshape(-1)
    same = got == want  # -inf among them
    ok = bool((same | ((got - want).abs() <= blp.gather(1, at)[:, 0])).all())
    assert ok, "log probability"
    ok = bool(((out.entropy.double().cpu().reshape(-1) - entropy).abs() <= bh).all())
    assert ok, "entropy"
    if not top:
        assert out.top_ids is None and out.top_logprobs is None
        return
    _, ids = (x.double() + 0.0).sort(dim=1, descending=True, stable=True)
    assert torch.equal(out.top_ids.cpu().reshape(len(x), top), ids[:, :top]), "alternatives"
    got = out.top_logprobs.double().cpu().reshape(len(x), top)
    want = logp.gather(1, ids[:, :top])
    ok = bool(((got == want) | ((got - want).abs() <= blp.gather(1, ids[:, :top]))).all())
    assert ok, "their log probabilities"


SIZES = [(1, 1), (2, 2), (3, 7), (1, 33), (4, 63), (5, 64), (2, 65), (3, 255), (70, 257), (9, 1003), (300, 1000),
         (2, 4099), (7, 8192), (600, 2049), (1, 50257), (33, 50257), (3, 65537), (2, 131071), (1, 262147)]


@pytest.mark.parametrize("rows,v", SIZES)
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("top", [0, 1, 5, MAX_TOP])
def test_scores_against_64_bits(dev, rows, v, dtype, top):
    top = min(top, v)
    x, tokens = _logits(rows, v, rows + v, dtype)
    _check(g.token_logprobs(x.to(dev), tokens.to(dev), top=top), x, tokens, top)


@pytest.mark.parametrize("rows,v", [(3, 50257), (600, 1003), (5, 131072), (2, 262147)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_sure_rows_keep_their_digits(dev, rows, v, dtype):
    """log p of a token that the model is sure of, far below 2^-24, to full precision."""
    x, _ = _logits(rows, v, 3, dtype, boost=False)
    best = torch.arange(rows) * 37 % v
    x[torch.arange(rows), best] = 40.0
    out = g.token_logprobs(x.to(dev), best.to(dev), top=2)
    _check(out, x, best, 2)
    assert torch.all(out.logprob < 0) and torch.all(out.logprob > -1e-7)


@pytest.mark.parametrize("v", [5, 64, 1003, 9000, 70001, 150001])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_masked_logits(dev, v, dtype):
    """-inf and the type's lowest number where a mask left nothing; rows with one
    token left; ties; signed zeros."""
    lowest = torch.finfo(dtype).min
    x, tokens = _logits(8, v, 4, FP32)
    x[0, 1:] = float("-inf")              # one token left
    x[1, ::2] = float("-inf")
    x[2, 1:] = lowest
    x[3, ::3] = lowest
    x[4] = 0.25                           # every token the same
    x[5] = 0.0
    x[5, 1::2] = -0.0                     # equal to 0
    x[6, : v // 2] = float("-inf")        # a masked half, then ties
    x[6, v // 2 :] = -7.0
    x[7] = lowest
    x = x.to(dtype)
    tokens[0], tokens[1], tokens[2] = 0, 0, 1
    top = min(v, 20)
    out = g.token_logprobs(x.to(dev), tokens.to(dev), top=top)
    _check(out, x, tokens, top)
    assert out.logprob[0] == 0 and out.entropy[0] == 0 and out.logprob[1] == float("-inf")
    assert out.top_ids[4].tolist() == list(range(top)) and out.top_ids[5].tolist() == list(range(top))


@pytest.mark.parametrize("v", [4, 300, 20011, 150001])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_rows_without_a_distribution(dev, v, dtype):
    """NaN, +inf or nothing above -inf: NaN scores, as torch's log_softmax; NaN
    stands above everything among the alternatives; the other rows are not touched."""
    x, tokens = _logits(6, v, 5, FP32)
    x[0, 2] = float("nan")
    x[1, 1] = float("inf")
    x[2] = float("-inf")
    x[3, 3] = -float("nan")
    x = x.to(dtype)
    out = g.token_logprobs(x.to(dev), tokens.to(dev), top=2)
    assert torch.isnan(out.logprob[:4]).all() and torch.isnan(out.entropy[:4]).all()
    assert torch.isnan(out.top_logprobs[:4]).all()
    assert torch.isnan(F.log_softmax(x[:4].float(), dim=1)).any(dim=1).all()
    assert out.top_ids[0, 0] == 2 and out.top_ids[1, 0] == 1 and out.top_ids[3, 0] == 3
    assert out.top_ids[2].tolist() == [0, 1]
    rest = g.TokenScores(*(t[4:] for t in out))
    _check(rest, x[4:], tokens[4:], 2)


def test_ignored_and_foreign_tokens(dev):
    x, tokens = _logits(6, 777, 6)
    tokens[1], tokens[2], tokens[3], tokens[4] = -100, 777, -1, 1 << 40
    out = g.token_logprobs(x.to(dev), tokens.to(dev))
    assert out.logprob[1] == 0 and torch.isnan(out.logprob[2:5]).all()
    ok = [0, 1, 5]
    _check(g.TokenScores(out.logprob[ok], out.entropy[ok], None, None), x[ok], tokens[ok], 0)
    assert torch.isfinite(out.entropy).all()
    other = g.token_logprobs(x.to(dev), torch.full((6,), 5, device=dev), ignore_index=5)
    assert torch.all(other.logprob == 0)
    for t in (torch.int32, torch.int16, torch.uint8):
        small = torch.arange(6, dtype=t, device=dev)
        assert torch.equal(g.token_logprobs(x.to(dev), small).logprob,
                           g.token_logprobs(x.to(dev), small.long()).logprob)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_strides_and_alignment(dev, dtype):
    """Slices of a batch's logits in place, rows that start at any element, rows at
    stride 0, a vocabulary that is not consecutive, more leading dimensions."""
    gen = torch.Generator().manual_seed(7)
    big = (torch.randn(3, 5, 1003, generator=gen) * 3).to(dtype).to(dev)
    flat = big.view(-1)
    views = [big[:, :-1], big[:, 1:], big[1], big[:, 2], big[::2, ::2, 1:], big[..., 3:900], big[:1].expand(4, -1, -1),
             big.transpose(0, 1), big.permute(0, 2, 1)[..., :4], big[0, 0], big.view(3, 5, 17, 59),
             flat[1 : 1 + 12 * 1001].view(12, 1001), flat[7 : 7 + 4 * 3000].view(4, 3000)]
    for view in views:
        x = view.cpu().reshape(-1, view.shape[-1])
        tokens = torch.randint(0, x.shape[1], (len(x),), generator=gen)
        top = min(4, x.shape[1])
        out = g.token_logprobs(view, tokens.view(view.shape[:-1]).to(dev), top=top)
        assert out.logprob.shape == view.shape[:-1] and out.top_ids.shape == (*view.shape[:-1], top)
        _check(out, x, tokens, top)


def test_rows_past_32_bit_offsets(dev):
    """A batch's logits of more than 2^32 bytes and a stride that passes 2^31 elements."""
    v, sr = 1003, (1 << 31) // 2 + 1001
    buf = torch.empty(2 * sr + v, dtype=BF16, device=dev)
    x, tokens = _logits(3, v, 8, BF16)
    view = buf.as_strided((3, v), (sr, 1))
    view.copy_(x.to(dev))
    out = g.token_logprobs(view, tokens.to(dev), top=3)
    _check(out, x, tokens, 3)


def test_no_rows(dev):
    out = g.token_logprobs(torch.empty(0, 9, device=dev), torch.empty(0, dtype=torch.int64, device=dev), top=2)
    assert out.logprob.shape == (0,) and out.top_ids.shape == (0, 2)
    out = g.token_logprobs(torch.empty(2, 0, 9, device=dev), torch.empty(2, 0, dtype=torch.int64, device=dev))
    assert out.entropy.shape == (2, 0)


def test_results_do_not_depend_on_the_other_rows(dev):
    """A row alone, in a batch, and again: the same bits on the same path, the same
    alternatives on every path."""
    x, tokens = _logits(900, 4099, 9)
    x, tokens = x.to(dev), tokens.to(dev)
    a, b = g.token_logprobs(x, tokens, top=8), g.token_logprobs(x, tokens, top=8)
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    for n in (1, 3, 40, 300):
        c = g.token_logprobs(x[:n], tokens[:n], top=8)
        assert torch.equal(c.top_ids, a.top_ids[:n])
        assert (c.logprob - a.logprob[:n]).abs().max() < 1e-5


# ------------------------------------------------------------------ gradient
def _grad_reference(x, tokens, gl, gh, gt, top, ignore=-100):
    z = x.double().requires_grad_()
    logp = torch.log_softmax(z, dim=1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * torch.where(p > 0, logp, 0.0), 0.0)
    entropy = -plogp.sum(dim=1)
    seen = tokens != ignore
    total = (torch.where(seen, logp.gather(1, torch.where(seen, tokens, 0)[:, None])[:, 0], 0.0) * gl.double()).sum()
    total = total + (entropy * gh.double()).sum()
    if top:
        _, ids = (x.double() + 0.0).sort(dim=1, descending=True, stable=True)
        total = total + (logp.gather(1, ids[:, :top]) * gt.double()).sum()
    (grad,) = torch.autograd.grad(total, z)
    return grad, p.detach(), logp.detach()


def _check_grad(grad, x, tokens, gl, gh, gt, top):
    want, p, logp = _grad_reference(x, tokens, gl, gh, gt, top)
    z, _, entropy, d, A, B = _reference(x, tokens)
    _, bh = _bounds(x, z, logp, d, A, B)
    n = x.shape[1] / 256 + 16
    D = ((2 * A + 2 + n) * U)[:, None]
    zf = torch.where(p > 0, z, 0.0).abs()
    lf = torch.where(p > 0, logp, 0.0).abs()
    # p follows z twice, exp, the sum and the quotient; the bracket is a handful of
    # roundings of its parts and H's own error
    ep = 2 * zf * U + 4 * U + D
    seen = (tokens != -100).double()
    g1 = (gl.double().abs() * seen)[:, None]
    g2 = gh.double().abs()[:, None]
    g3 = gt.double().abs().sum(dim=1)[:, None] if top else torch.zeros_like(g1)
    size = g1 + g3 + g2 * (lf + entropy[:, None] + zf + torch.log1p(d)[:, None])
    bound = p * (size * (ep + (8 + top) * U) + g2 * bh[:, None]) + want.abs() * 4 * U
    # a hot element: (1 - p) of its weight, whose 1 - p follows p's error
    hot = torch.zeros_like(want)
    hot.scatter_(1, torch.where(tokens == -100, 0, tokens)[:, None], g1)
    if top:
        _, ids = (x.double() + 0.0).sort(dim=1, descending=True, stable=True)
        hot.scatter_add_(1, ids[:, :top], gt.double().abs())
    bound = bound + hot * (p * ep + 4 * U) + 1e-42
    if x.dtype == BF16:
        bound = bound + (want.abs() + bound) * 2.0**-8
    err = (grad.double().cpu() - want).abs()
    ok = bool((err <= bound).all())
    assert ok, f"gradient off by {(err / bound).max():.3g} bounds"


@pytest.mark.parametrize("rows,v", [(1, 1), (2, 2), (3, 7), (5, 64), (9, 65), (70, 257), (33, 1003), (300, 1000),
                                    (2, 4099), (40, 8192), (1, 50257), (17, 50257), (3, 65537), (2, 131071)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("top", [0, 3])
def test_gradient_against_64_bits(dev, rows, v, dtype, top):
    top = min(top, v)
    x, tokens = _logits(rows, v, rows * 3 + v, dtype)
    tokens[rows // 2 + 1 :: 5] = -100
    gen = torch.Generator().manual_seed(10)
    gl, gh, gt = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen), torch.randn(rows, max(top, 1),
                                                                                                generator=gen)
    leaf = x.to(dev).requires_grad_()
    s = g.token_logprobs(leaf, tokens.to(dev), top=top)
    outs, grads = [s.logprob, s.entropy], [gl.to(dev), gh.to(dev)]
    if top:
        assert not s.top_ids.requires_grad
        outs, grads = outs + [s.top_logprobs], grads + [gt.to(dev)]
    (grad,) = torch.autograd.grad(outs, leaf, grads)
    assert grad.dtype == dtype and grad.shape == leaf.shape
    _check_grad(grad, x, tokens, gl, gh, gt, top)


def test_gradient_of_each_part_alone(dev):
    x, tokens = _logits(6, 500, 11)
    zero, one = torch.zeros(6), torch.ones(6)
    leaf = x.to(dev).requires_grad_()
    for part in ("logprob", "entropy", "top_logprobs"):
        s = g.token_logprobs(leaf, tokens.to(dev), top=2)
        (grad,) = torch.autograd.grad(getattr(s, part).sum(), leaf)
        gl, gh = (one if part == "logprob" else zero), (one if part == "entropy" else zero)
        gt = torch.ones(6, 2) if part == "top_logprobs" else torch.zeros(6, 2)
        _check_grad(grad, x, tokens, gl, gh, gt, 2)
    s = g.token_logprobs(leaf, tokens.to(dev))
    s.logprob.sum().backward()
    s = g.token_logprobs(leaf, tokens.to(dev))
    s.logprob.sum().backward()  # accumulates
    _check_grad(leaf.grad / 2, x, tokens, one, zero, None, 0)


def test_gradient_against_differences(dev):
    """Central differences of the scores themselves: with step t the quotient is off
    by at most t^2 / 6 times a third derivative (below 8 for a weight of 1 on log p
    and H of a few tokens) and by the scores' own roundings over t."""
    x, tokens = _logits(2, 9, 12, boost=False)
    x = x / 2
    step = 2.0**-7
    leaf = x.to(dev).requires_grad_()
    s = g.token_logprobs(leaf, tokens.to(dev), top=3)
    (grad,) = torch.autograd.grad((s.logprob.sum() + 0.5 * s.entropy.sum() + 0.25 * s.top_logprobs.sum()), leaf)

    def value(z):
        t = g.token_logprobs(z.to(dev), tokens.to(dev), top=3)
        return (t.logprob.double() + 0.5 * t.entropy.double() + 0.25 * t.top_logprobs.double().sum(dim=1)).cpu()

    for j in range(9):
        up, down = x.clone(), x.clone()
        up[:, j] += step
        down[:, j] -= step
        width = (up[:, j].double() - down[:, j].double())
        diff = (value(up) - value(down)) / width
        assert torch.all((diff - grad[:, j].double().cpu()).abs() <= step**2 * 8 / 6 + 1e-4)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_gradient_of_masked_rows(dev, dtype):
    """-inf logits get gradient 0; a token whose logit is -inf still gets its own weight."""
    x, tokens = _logits(5, 300, 13, FP32)
    x[0, 1:] = float("-inf")
    x[1, ::2] = float("-inf")
    x[2, 5:] = torch.finfo(dtype).min
    x[3] = float("-inf")
    x = x.to(dtype)
    tokens[0], tokens[1], tokens[2] = 0, 1, 1
    gl, gh = torch.ones(5), torch.full((5,), 0.5)
    leaf = x.to(dev).requires_grad_()
    s = g.token_logprobs(leaf, tokens.to(dev))
    (grad,) = torch.autograd.grad((s.logprob, s.entropy), leaf, (gl.to(dev), gh.to(dev)))
    assert torch.isnan(grad[3]).all()
    keep = [0, 1, 2, 4]
    want, _, _ = _grad_reference(x[keep], tokens[keep], gl[keep], torch.zeros(4), None, 0)
    assert torch.all(grad[0] == 0) and torch.all(grad[1, ::2] == 0)
    (plain,) = torch.autograd.grad(g.token_logprobs(leaf, tokens.to(dev)).logprob.sum(), leaf)
    _check_grad(plain[keep], x[keep], tokens[keep], gl[keep], torch.zeros(4), None, 0)
    bad = tokens.clone()
    bad[4] = 300
    (grad,) = torch.autograd.grad(g.token_logprobs(leaf, bad.to(dev)).logprob.sum(), leaf)
    assert torch.isnan(grad[4]).all() and torch.isfinite(grad[[0, 1, 2]]).all()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_gradient_through_strided_logits(dev, dtype):
    gen = torch.Generator().manual_seed(14)
    x = (torch.randn(3, 6, 403, generator=gen) * 2).to(dtype)
    ids = torch.randint(0, 403, (3, 6), generator=gen)
    leaf = x.to(dev).requires_grad_()
    s = g.token_logprobs(leaf[:, :-1], ids[:, 1:].to(dev))
    (grad,) = torch.autograd.grad(-s.logprob.sum(), leaf)
    assert torch.all(grad[:, -1] == 0)
    one = -torch.ones(15)
    _check_grad(grad[:, :-1].reshape(15, 403), x[:, :-1].reshape(15, 403), ids[:, 1:].reshape(-1), one,
                torch.zeros(15), None, 0)


def test_gradient_replayed_from_a_graph(dev):
    """Forward and backward captured together, replayed with new logits between
    eager passes; two graphs at once."""
    cases = [_logits(r, 1003, 15 + r) for r in (2, 40)]
    graphs = []
    for x, tokens in cases:
        static, tok = x.to(dev).requires_grad_(), tokens.to(dev)
        gl = torch.ones(len(x), device=dev)

        def step(static=static, tok=tok, gl=gl):
            s = g.token_logprobs(static, tok, top=2)
            (grad,) = torch.autograd.grad((s.logprob, s.entropy), static, (gl, gl))
            return s.logprob.detach(), s.top_ids, grad

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, static, out, step))
    for turn in range(3):
        for graph, static, out, step in graphs:
            with torch.no_grad():
                static.copy_(_logits(static.shape[0], 1003, 100 + turn)[0])
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("rows,v", [(3, 150001), (40, 20011)])
def test_scores_replayed_from_graphs(dev, rows, v):
    """Two captured calls (rows in segments with a workspace; whole rows) replayed in
    turn with new logits, eager calls between, on another stream than the capture's."""
    graphs = []
    for seed in (19, 20):
        x, tokens = _logits(rows, v, seed)
        x, tokens = x.to(dev), tokens.to(dev)
        g.token_logprobs(x, tokens, top=5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = g.token_logprobs(x, tokens, top=5)
        graphs.append((graph, x, tokens, out))
    side = torch.cuda.Stream()
    for turn in range(3):
        for i, (graph, x, tokens, out) in enumerate(graphs):
            x.copy_(_logits(rows, v, 200 + 2 * turn + i)[0])
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            want = g.token_logprobs(x, tokens, top=5)  # beside the replay
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_changed_logits_are_refused_in_the_backward(dev):
    x, tokens = _logits(3, 50, 16)
    base = x.to(dev).requires_grad_()
    y = base * 1.0
    s = g.token_logprobs(y, tokens.to(dev))
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.logprob.sum().backward()


# ---------------------------------------------------------------- model paths
def _tiny(dev, seed=0):
    torch.manual_seed(seed)
    cfg = g.GPTConfig(vocab_size=211, n_positions=64, n_layer=2, n_head=2, n_embd=128)
    return g.GPT(cfg).to(dev).eval()


def test_scores_of_a_model_are_its_loss(dev):
    model = _tiny(dev)
    idx = torch.arange(40, device=dev).view(2, 20) * 5
    targets = idx.roll(-1, 1).clone()
    targets[0, 15:] = -100
    s = g.score_tokens(model, idx, targets, top=3)
    loss = model(idx, targets)["loss"]
    n = (targets != -100).sum()
    assert abs((-s.logprob.sum() / n - loss).item()) < 1e-5
    nxt = g.score_tokens(model, idx)
    assert nxt.logprob.shape == (2, 19) and nxt.top_ids is None
    assert torch.equal(nxt.logprob[1], s.logprob[1, :-1])
    assert torch.equal(s.top_ids[..., 0], model(idx)["logits"].argmax(dim=-1))
    with pytest.raises(ValueError, match="do not match"):
        g.score_tokens(model, idx, targets[:1])


def test_a_training_step_through_the_scores(dev):
    """The gradients that a loss on the scores gives the weights are those of the
    same loss in torch ops."""
    model = _tiny(dev, 1).train()
    idx = torch.arange(40, device=dev).view(2, 20) * 5
    y = idx.roll(-1, 1)

    def grads(loss):
        return torch.autograd.grad(loss, list(model.parameters()))

    s = g.token_logprobs(model(idx)["logits"], y)
    got = grads(-s.logprob.mean() - 0.01 * s.entropy.mean())
    logp = torch.log_softmax(model(idx)["logits"], dim=-1)
    plain = -logp.gather(-1, y[..., None]).mean() + 0.01 * (logp.exp() * logp).sum(-1).mean()
    for a, b in zip(got, grads(plain)):
        assert (a - b).abs().max() <= 1e-5 * b.abs().max() + 1e-8


@pytest.mark.parametrize("use_cache", [True, False])
def test_generate_returns_scores(dev, use_cache):
    model = _tiny(dev, 2)
    prompt = torch.arange(10, device=dev).view(2, 5) * 11
    ids, s = g.generate(model, prompt, 7, scores=4, use_cache=use_cache)
    assert torch.equal(ids, g.generate(model, prompt, 7, use_cache=use_cache))
    assert s.logprob.shape == (2, 7) and s.top_ids.shape == (2, 7, 4)
    assert torch.equal(s.top_ids[..., 0], ids[:, 5:])  # greedy
    assert torch.equal(s.top_logprobs[..., 0], s.logprob)
    whole = g.score_tokens(model, ids)
    assert (whole.logprob[:, 4:] - s.logprob).abs().max() < 1e-4
    same, none = g.generate(model, prompt, 0, scores=0)
    assert torch.equal(same, prompt) and none.logprob.shape == (2, 0) and none.top_ids is None


def test_perplexity_with_token_scores(dev):
    model = _tiny(dev, 3)
    data = g.SyntheticTokenStream(211, 900, 32)
    a = g.perplexity_with_error_bars(model, data, n_chunks=3, batches_per_chunk=2, batch_size=2)
    b = g.perplexity_with_error_bars(model, data, n_chunks=3, batches_per_chunk=2, batch_size=2, token_scores=True)
    assert set(b) - set(a) == {"entropy_mean", "top1_accuracy"}
    assert abs(a["loss_mean"] - b["loss_mean"]) < 1e-5 and a["n_chunks"] == b["n_chunks"]
    assert 0 < b["entropy_mean"] <= math.log(211)


def test_refusals(dev):
    x, t = torch.zeros(3, 8, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for bad, error, text in [
        (lambda: g.token_logprobs(x.double(), t), TypeError, "float32 or bfloat16"),
        (lambda: g.token_logprobs(x, t.float()), TypeError, "integers"),
        (lambda: g.token_logprobs(x, t.bool()), TypeError, "integers"),
        (lambda: g.token_logprobs(x, t[:2]), ValueError, "do not match"),
        (lambda: g.token_logprobs(x, t, top=9), ValueError, "top must be"),
        (lambda: g.token_logprobs(x, t, top=-1), ValueError, "top must be"),
        (lambda: g.token_logprobs(torch.zeros(3, 100, device=dev), t, top=65), ValueError, "top must be"),
        (lambda: g.token_logprobs(x[:, :0], t), ValueError, "no vocabulary"),
        (lambda: g.token_logprobs(x.cpu(), t), RuntimeError, "ROCm GPU"),
        (lambda: g.token_logprobs(x, t.cpu()), RuntimeError, "ROCm GPU"),
    ]:
        with pytest.raises(error, match=text):
            bad()
    L = _lib.lib()
    v = 131071  # a long row, cut into segments: too little workspace is refused before any launch
    nb = L.tiq_token_logprobs_workspace(_lib.F32, 1, v, 5)
    assert nb > 0 and L.tiq_token_logprobs_workspace(_lib.F32, 1, 50257, 5) == 0
    y = torch.zeros(1, v, device=dev)
    out = torch.full((8,), 3.0, device=dev)
    ids = torch.zeros(8, dtype=torch.int64, device=dev)
    for ws, n in ((None, nb), (out, nb - 1), (None, 0)):
        rc = L.tiq_token_logprobs(y.data_ptr(), _lib.F32, 1, 1, 0, v, v, t.data_ptr(), -100, 5, out.data_ptr(),
                                  out.data_ptr(), None, ids.data_ptr(), out.data_ptr(), _lib.ptr(ws), n,
                                  _lib.stream_of(y))
        assert rc == _lib.EWORKSPACE and torch.all(out == 3.0)


def test_second_derivatives_are_refused(dev):
    x, tokens = _logits(3, 50, 17)
    leaf = x.to(dev).requires_grad_()
    s = g.token_logprobs(leaf, tokens.to(dev))
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(s.logprob.sum(), leaf, create_graph=True)


def _check_top_on_gpu(x, out, top):
    """Alternatives of GPU logits against a stable sort in 64 bits."""
    values, ids = (x.double() + 0.0).sort(dim=1, descending=True, stable=True)
    assert torch.equal(out.top_ids, ids[:, :top])
    want = torch.log_softmax(x.double(), dim=1).gather(1, ids[:, :top])
    got = out.top_logprobs.double()
    ok = bool(((got == want) | ((got - want).abs() <= 1e-5 * (1 + want.abs()))).all())
    assert ok


def test_tangents_are_refused(dev):
    from torch.autograd import forward_ad
    x, tokens = _logits(2, 20, 18)
    x, tokens = x.to(dev), tokens.to(dev)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            g.token_logprobs(dual, tokens)
        assert torch.isfinite(g.token_logprobs(x, tokens).logprob).all()


@pytest.mark.parametrize("rows,v,threads", [(130, 20000, 512), (3, 20000, 512), (100, 200000, 256), (3, 200000, 256),
                                            (130, 2400, 256), (20, 1000, 64)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_large_logits_in_few_places(dev, rows, v, threads, dtype):
    """Rows whose large logits all fall to a few threads, ties by the thousand, rows with
    fewer tokens left than alternatives wanted: every way the selection can go."""
    vec = 16 // (4 if dtype is FP32 else 2)
    gen = torch.Generator(device=dev).manual_seed(18)
    x = torch.randn(rows, v, generator=gen, device=dev)
    place = torch.arange(v, device=dev)
    few = (place // vec) % threads < 8 * threads // 64
    x[0::5] += 50.0 * few
    x[1::5] = 1.5                                     # all equal
    x[2::5, 20:] = float("-inf")                      # as many left as wanted, or fewer
    x[2::10, 7:] = float("-inf")
    x[3::5] = torch.where(place % 3 == 0, 2.0, x[3::5])  # thousands of ties below a few larger ones
    x[3::5, 777] = 9.0
    x = x.to(dtype)
    for top in (4, 20, MAX_TOP):
        _check_top_on_gpu(x, g.token_logprobs(x, torch.zeros(rows, dtype=torch.int64, device=dev), top=top), top)


@pytest.mark.parametrize("rows,v", [(2, 40), (3, 1003), (2, 9001), (1030, 9001), (2, 150001)])
def test_signalling_nans(dev, rows, v):
    """NaN bits of every kind give NaN scores and the top place, and touch no other row."""
    for dtype, bits in ((FP32, (0x7F800001, -0x3FFFFF, 0x7FC00000)), (BF16, (0x7F81, -0x7F, 0x7FC0))):
        x, tokens = _logits(min(rows, 8), v, 19, dtype)
        x = x.repeat(-(-rows // len(x)), 1)[:rows].to(dev)
        tokens = tokens.repeat(-(-rows // len(tokens)))[:rows].to(dev)
        clean = g.token_logprobs(x, tokens, top=3)
        for b in bits:
            y = x.clone()
            y.view(torch.int32 if dtype is FP32 else torch.int16)[0, v - 2] = b
            out = g.token_logprobs(y, tokens, top=3)
            assert torch.isnan(out.logprob[0]) and torch.isnan(out.entropy[0]) and torch.isnan(out.top_logprobs[0]).all()
            assert out.top_ids[0, 0] == v - 2
            for a, c in zip(out, clean):
                assert torch.equal(a[1:], c[1:])


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_more_rows_than_one_launch_takes(dev, dtype):
    rows, v = (1 << 22) + 37, 9
    gen = torch.Generator(device=dev).manual_seed(20)
    x = torch.randn(rows, v, generator=gen, device=dev).to(dtype).requires_grad_()
    tokens = torch.randint(0, v, (rows,), generator=gen, device=dev)
    s = g.token_logprobs(x, tokens, top=2)
    logp = torch.log_softmax(x.detach().double(), dim=1)
    assert (s.logprob - logp.gather(1, tokens[:, None])[:, 0]).abs().max() < 2e-6
    assert (s.entropy + (logp.exp() * logp).sum(dim=1)).abs().max() < 2e-6
    assert torch.equal(s.top_ids[:, 0], x.detach().float().argmax(dim=1)) or dtype is BF16
    (grad,) = torch.autograd.grad(s.logprob.sum(), x)
    want = F.one_hot(tokens, v) - logp.exp()
    assert (grad.double() - want).abs().max() < (2e-6 if dtype is FP32 else 2.0**-8)
