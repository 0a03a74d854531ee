"""The Linear on int8 activations and int8 weights (``w8a8``) and the per-token
quantization before it.

Codes and scales are the CPU oracle's bit for bit. A product is compared with
the same codes in 64 bits: the kernel's sum is an exact integer, which is rounded
to fp32 once, times the row's scale (one rounding), times the channel's scale plus
the bias (one fused rounding), and once more for a bf16 output: half a step each.
"""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

import gpt2_harness_amd as g
from gpt2_harness_amd import _lib
from gpt2_harness_amd.model import gelu_tanh
from oracle import model as OM
from oracle import quant as OQ

pytestmark = pytest.mark.gpu

FP32, BF16 = torch.float32, torch.bfloat16


def _rows(m, k, seed, dtype=FP32):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen)
    x[:, :: max(2, min(k, 97))] *= 8.0
    return x.to(dtype)


def _weight(n, k, seed, bias=True):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, (n, k), generator=gen, dtype=torch.int64).to(torch.int8)
    s = torch.rand(n, generator=gen) * 1e-3 + 1e-5
    return q, s, (torch.randn(n, generator=gen) * 0.1 if bias else None)


def _linear(q, s, b, dev):
    n, k = q.shape
    return g.QuantLinear(q.to(dev), s.to(dev), None if b is None else b.to(dev), k, n, 8, "per_channel", "w8a8")


def _oracle_codes(x):
    q, s = OQ.quantize_tensor(x.float().numpy(), 8)
    return torch.from_numpy(np.array(q)), torch.from_numpy(np.array(s)).reshape(-1)


def _check(y, x, q, s, b):
    """``y`` against the codes' product in 64 bits, within the roundings above."""
    qx, sx = _oracle_codes(x)
    core = (qx.double() @ q.double().t()) * sx.double()[:, None] * s.double()
    want = core if b is None else core + b.double()
    u = 2.0**-24
    bound = core.abs() * (2 * u) * (1 + 4 * u) + want.abs() * u * 1.001 + 1e-44
    if y.dtype == BF16:
        bound = bound + (want.abs() + bound) * 2.0**-8
    err = (y.double().cpu() - want).abs()
    ok = bool((err <= bound).all())
    assert ok, f"error {(err - bound).max():.3g} beyond the bound"


# ------------------------------------------------------------ quantize_tokens
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (7, 64), (2, 63), (33, 1001), (5, 1600), (2, 6400), (1, 20000),
                                   (2, 3, 130)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_tokens_equal_the_oracle(dev, shape, dtype):
    x = _rows(int(np.prod(shape[:-1])), shape[-1], 1, dtype).reshape(shape)
    q, s = g.quantize_tokens(x.to(dev))
    qo, so = _oracle_codes(x.reshape(-1, shape[-1]))
    assert q.shape == x.shape and s.shape == (*shape[:-1], 1) and q.dtype == torch.int8
    assert torch.equal(q.cpu().reshape(qo.shape), qo)
    assert torch.equal(s.cpu().reshape(-1), so)
    if dtype is FP32 and len(shape) == 2:
        q2, s2 = g.quantize_tensor(x.to(dev), 8)
        assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("k", [7, 96, 1000])
def test_tokens_of_rows_that_are_not_ordinary(dev, dtype, k):
    x = _rows(8, k, 2)
    x[0] = 0.0                       # scale FLT_MIN, codes 0
    x[1] = 1e-41                     # below the normal numbers
    x[2, k // 2] = float("inf")
    x[3, 0] = float("nan")
    x[4] = -3.0                      # every element the largest
    x[5, -1] = 1e30
    x[6] = torch.arange(k) - (k - 1) / 2  # halves: ties to even
    x = x.to(dtype)
    q, s = g.quantize_tokens(x.to(dev))
    w = x.float().to(dev)
    q2, s2 = g.quantize_tensor(w, 8)
    assert torch.equal(q, q2)
    assert torch.equal(s.view(torch.int32)[torch.isfinite(s)], s2.view(torch.int32)[torch.isfinite(s2)])
    assert torch.equal(torch.isnan(s), torch.isnan(s2))


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_tokens_read_strided_and_shifted_rows_in_place(dev, dtype):
    big = _rows(9, 333, 3, dtype).to(dev)
    for view in (big[:, :100], big[1::2, 1:200], big.t(), big[:, 3:].unsqueeze(0), big[0]):
        q, s = g.quantize_tokens(view)
        qo, so = _oracle_codes(view.cpu().reshape(-1, view.shape[-1]))
        assert torch.equal(q.cpu().reshape(qo.shape), qo) and torch.equal(s.cpu().reshape(-1), so)


def test_tokens_of_nothing(dev):
    q, s = g.quantize_tokens(torch.empty(0, 5, device=dev))
    assert q.shape == (0, 5) and s.shape == (0, 1)


# ------------------------------------------------------------------- product
SHAPES = [(1, 1, 1), (1, 768, 2304), (2, 17, 5), (4, 1600, 100), (5, 64, 33), (16, 1600, 640), (17, 96, 1),
          (31, 64, 33), (32, 64, 32), (33, 65, 31), (64, 768, 96), (77, 1001, 777), (128, 640, 160), (130, 1600, 257),
          (257, 320, 511), (300, 4096, 200), (513, 129, 1025), (1001, 1024, 640)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_product_against_64_bits(dev, m, k, n, dtype):
    x = _rows(m, k, m + k, dtype)
    q, s, b = _weight(n, k, n + 3, bias=(m + n) % 3 != 0)
    y = _linear(q, s, b, dev)(x.to(dev))
    assert y.shape == (m, n) and y.dtype == dtype
    _check(y, x, q, s, b)


@pytest.mark.parametrize("m,k,n", [(2100, 256, 1100), (4096, 192, 768), (1500, 1600, 2400), (700, 6400, 1600),
                                   # 128 x 256 tiles: all whole; the last ones in halves, with ragged edges, in
                                   # uneven shares of the XCDs
                                   (4096, 96, 4096), (4096, 192, 4800), (4001, 130, 4701), (2500, 70, 3700)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_large_product_against_64_bits(dev, m, k, n, dtype):
    """The products of many rows, checked on the GPU in 64 bits."""
    x = _rows(m, k, 5, dtype).to(dev)
    q, s, b = _weight(n, k, 6)
    y = _linear(q, s, b, dev)(x).double()
    qx, sx = g.quantize_tokens(x)
    core = (qx.double() @ q.to(dev).double().t()) * sx.double() * s.to(dev).double()
    want = core + b.to(dev).double()
    u = 2.0**-24
    bound = core.abs() * (2 * u) * (1 + 4 * u) + want.abs() * u * 1.001
    if dtype == BF16:
        bound = bound + (want.abs() + bound) * 2.0**-8
    ok = bool(((y - want).abs() <= bound).all())
    assert ok


@pytest.mark.parametrize("m", [1, 3, 40, 200])
def test_the_longest_sum_fits(dev, m):
    """K = 131072 codes of the largest size: 131072 * 127 * 128 < 2^31."""
    k, n = 131072, 33
    x = torch.full((m, k), -1.0)
    q = torch.full((n, k), -128, dtype=torch.int8)
    q[1::2] = 127
    y = _linear(q, torch.ones(n), None, dev)(x.to(dev))
    _check(y, x, q, torch.ones(n), None)
    wide = _linear(torch.zeros(2, k + 1, dtype=torch.int8), torch.ones(2), None, dev)
    with pytest.raises(RuntimeError, match="unsupported"):
        wide(torch.zeros(1, k + 1, device=dev))


@pytest.mark.parametrize("m", [1, 20, 150])
def test_rows_with_infinities_are_nan_and_leave_the_others(dev, m):
    x = _rows(m + 3, 200, 7)
    q, s, b = _weight(70, 200, 8)
    lin = _linear(q, s, b, dev)
    x[1, 5], x[2, 100] = float("inf"), float("nan")
    y = lin(x.to(dev))
    assert torch.isnan(y[1:3]).all()
    keep = [i for i in range(m + 3) if i not in (1, 2)]
    _check(y[keep], x[keep], q, s, b)
    z = lin(torch.zeros(m, 200, device=dev))  # a row of zeros gives the bias
    assert torch.equal(z.cpu(), b.expand(m, -1))


@pytest.mark.parametrize("m,k,n", [(3, 100, 50), (70, 130, 45), (300, 640, 200)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_strided_input_and_output_through_the_library(dev, m, k, n, dtype):
    """Row strides on both sides; what lies beside and behind the output's rows stays."""
    big = _rows(m, k + 13, 9, dtype).to(dev)
    x = big[:, 5 : 5 + k]
    q, s, b = _weight(n, k, 10)
    lin = _linear(q, s, b, dev)
    out = torch.full((m + 2, n + 7), 5.0, dtype=dtype, device=dev)
    L = _lib.lib()
    nb = L.tiq_linear_w8a8_workspace(_lib.dtype_code(dtype), m, k, n)
    ws = torch.full((max(nb, 1),), 0x7F, dtype=torch.uint8, device=dev)
    rc = L.tiq_linear_w8a8(x.data_ptr(), _lib.dtype_code(dtype), m, k, x.stride(0), lin.codes.data_ptr(),
                           lin.scale.data_ptr(), lin.bias.data_ptr(), n, out[:, 3:].data_ptr(),
                           _lib.dtype_code(dtype), n + 7, ws.data_ptr(), nb, _lib.stream_of(x))
    assert rc == 0
    _check(out[:m, 3 : 3 + n], x.cpu(), q, s, b)
    rest = out.clone()
    rest[:m, 3 : 3 + n] = 5.0
    assert torch.all(rest == 5.0)
    assert torch.equal(lin(x), out[:m, 3 : 3 + n])  # the module, from the same strided view


def test_other_input_types_and_leading_dimensions(dev):
    q, s, b = _weight(40, 96, 11)
    lin = _linear(q, s, b, dev)
    x = _rows(6, 96, 12)
    y = lin(x.to(dev).view(2, 3, 96))
    assert y.shape == (2, 3, 40)
    _check(y.view(6, 40), x, q, s, b)
    _check(lin(x.half().to(dev)), x.half().float(), q, s, b)
    assert lin(torch.empty(0, 96, device=dev)).shape == (0, 40)
    assert torch.equal(lin.weight.cpu(), q.float() * s[:, None])


@pytest.mark.parametrize("m", [1, 8, 100, 600])
def test_captured_calls_and_other_streams(dev, m):
    """Two captured graphs, replayed in turn with eager calls between, each with
    new inputs; then a call on a side stream."""
    q, s, b = _weight(192, 320, 13)
    lin = _linear(q, s, b, dev)
    xs = [_rows(m, 320, 14 + i).to(dev) for i in range(4)]
    want = [lin(x) for x in xs]
    graphs = []
    for x in xs[:2]:
        static = x.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lin(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = lin(static)
        graphs.append((graph, static, y))
    for turn in range(4):
        for i, (graph, static, y) in enumerate(graphs):
            static.copy_(xs[(turn + i) % 4])
            graph.replay()
            assert torch.equal(lin(xs[turn]), want[turn])
            assert torch.equal(y, want[(turn + i) % 4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = lin(xs[3])
    side.synchronize()
    assert torch.equal(y, want[3])


# ------------------------------------------------- a prompt's rows, fused
FUSED = [(5, 64, 33), (16, 768, 96), (17, 100, 65), (77, 1001, 130), (130, 1600, 257), (400, 768, 768), (1030, 320, 1100),
         (1500, 1600, 2400), (600, 6400, 320), (2100, 256, 1100), (2500, 68, 3700)]


@pytest.mark.parametrize("m,k,n", FUSED)
def test_gelu_and_residual_are_the_separate_steps(dev, m, k, n):
    """Bit for bit: GELU as the rows are quantized, the residual beside the scales."""
    x = _rows(m, k, 30).to(dev)
    q, s, b = _weight(n, k, 31)
    lin = _linear(q, s, b, dev)
    gen = torch.Generator().manual_seed(32)
    res = torch.randn(m, n, generator=gen).to(dev)
    act = gelu_tanh(x)
    assert torch.equal(lin.forward_prefill(x, gelu=True), lin(act))
    assert torch.equal(lin.forward_prefill(x, residual=res), lin(x) + res)
    assert torch.equal(lin.forward_prefill(x, gelu=True, residual=res), lin(act) + res)
    assert torch.equal(lin.forward_prefill(x), lin(x))
    # the residual's place as the output's
    L = _lib.lib()
    nb = L.tiq_linear_w8a8_prefill_workspace(m, k, n)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    y = res.clone()
    rc = L.tiq_linear_w8a8_prefill(x.data_ptr(), m, k, k, lin.codes.data_ptr(), lin.scale.data_ptr(),
                                   lin.bias.data_ptr(), n, y.data_ptr(), n, None, None, 0.0, 0, y.data_ptr(), n,
                                   ws.data_ptr(), nb, _lib.stream_of(x))
    assert rc == 0 and torch.equal(y, lin(x) + res)


@pytest.mark.parametrize("m,k,n", FUSED)
@pytest.mark.parametrize("shift", [0.0, 3.0])
def test_layer_norm_before_the_product(dev, m, k, n, shift):
    """Against a LayerNorm in 64 bits and the codes' product. The fp32 LayerNorm is off by
    at most e = (|h| + |b|) 8 u + |w| (k + 40) u (|mean| + |x|) rstd, u = 2^-24: its sums of k
    terms, the subtraction, rsqrt and the affine step; so is a row's largest value, and
    the scale with it. A code is another than the exact one only where its quotient lies
    within that distance, over the scale, of a half, plus the quotient's own 3 u: each
    such code may move its outputs by sx sw |qw|, and the scale moves all by its part."""
    gen = torch.Generator().manual_seed(33)
    x = _rows(m, k, 34) + shift
    q, s, b = _weight(n, k, 35)
    lin = _linear(q, s, b, dev)
    ln = torch.nn.LayerNorm(k).to(dev)
    w, c = 1 + 0.1 * torch.randn(k, generator=gen), 0.1 * torch.randn(k, generator=gen)
    with torch.no_grad():
        ln.weight.copy_(w)
        ln.bias.copy_(c)
    with torch.no_grad():
        y = lin.forward_prefill(x.to(dev), ln=ln).double()
    u = 2.0**-24
    xd, wd, cd = x.to(dev).double(), w.to(dev).double(), c.to(dev).double()
    mu = xd.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(xd.var(1, unbiased=False, keepdim=True) + ln.eps)
    h = (xd - mu) * rstd * wd + cd
    e = (h.abs() + cd.abs()) * 8 * u + wd.abs() * (k + 40) * u * (mu.abs() + xd.abs()) * rstd
    top = h.abs().amax(1, keepdim=True)
    rel = e.amax(1, keepdim=True) / top + 2 * u  # of the scale
    sx = top / 127
    t = h / sx
    qx = torch.round(t)
    near = (((t - torch.floor(t)) - 0.5).abs() <= e / sx + t.abs() * (rel + 3 * u)).double()
    qw, sw = q.to(dev).double(), s.to(dev).double()
    core = (qx @ qw.t()) * sx * sw
    want = core + b.to(dev).double()
    bound = (near @ qw.abs().t()) * sx * sw + core.abs() * (rel + 2 * u) + want.abs() * 2 * u
    bad = ((y - want).abs() > bound * (1 + 1e-6) + 1e-30).sum().item()
    assert bad == 0, f"{bad} outputs beyond the bound"
    assert near.mean() < 0.05  # few codes are in doubt


def test_fused_rows_that_are_not_ordinary(dev):
    q, s, b = _weight(70, 96, 36)
    lin = _linear(q, s, b, dev)
    x = _rows(40, 96, 37)
    x[1, 5], x[2, 90], x[3], x[4] = float("inf"), float("nan"), 0.0, 5.0
    x = x.to(dev)
    ln = torch.nn.LayerNorm(96).to(dev).requires_grad_(False)
    y = lin.forward_prefill(x, ln=ln)
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[3:]).all()
    y = lin.forward_prefill(x, gelu=True)
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[5:]).all()
    assert torch.equal(y[3], b.to(dev))


def test_prompts_that_the_fused_call_leaves_alone(dev):
    """Four rows and fewer, long rows, a cache's slots: None, and the module's own steps."""
    q, s, b = _weight(8, 8256, 38)
    lin = _linear(q, s, b, dev)
    x = _rows(6, 8256, 39).to(dev)
    assert lin.forward_prefill(x, gelu=True) is None and lin.forward_gelu_in(x) is None
    assert not lin.writes_kv(600)
    q, s, b = _weight(64, 64, 40)
    lin = _linear(q, s, b, dev)
    assert lin.forward_prefill(_rows(4, 64, 41).to(dev), gelu=True) is None
    x = _rows(300, 64, 42).to(dev)
    assert lin.forward_prefill(x, kv=(x, x, 300)) is None
    assert lin.forward_prefill(x, residual=x[:1]) is None


# ---------------------------------------------------------------- model paths
def _tiny(dev, seed=0):
    torch.manual_seed(seed)
    cfg = g.GPTConfig(vocab_size=211, n_positions=64, n_layer=2, n_head=2, n_embd=128)
    return g.GPT(cfg).to(dev).eval()


def test_quantized_model_runs_every_linear_on_integers(dev):
    model = _tiny(dev)
    qm, stats = g.quantize_model(model, 8, act_bits=8)
    assert stats["act_bits"] == 8
    lins = [m for m in qm.modules() if isinstance(m, g.QuantLinear)]
    assert len(lins) == 8 and all(m.fmt == "w8a8" for m in lins)
    idx = torch.arange(34, device=dev).view(2, 17) * 5
    out = qm(idx)["logits"]
    # the same model with each Linear spelled out in torch
    ref = copy.deepcopy(model)
    for (name, mod) in list(ref.named_modules()):
        if name.endswith(g.TARGET_SUFFIXES):
            q, s = g.quantize_tensor(mod.weight.data, 8)

            class Plain(torch.nn.Module):
                def __init__(self, q, s, b):
                    super().__init__()
                    self.q, self.s, self.b = q, s, b

                def forward(self, x):
                    qx, sx = g.quantize_tokens(x)
                    y = (qx.double() @ self.q.double().t()) * sx.double() * self.s.double().view(-1)
                    return (y + self.b.double()).float()

            parent, _, leaf = name.rpartition(".")
            setattr(ref.get_submodule(parent), leaf, Plain(q, s, mod.bias.data))
    want = ref(idx)["logits"]
    # both compute the same codes but where a hidden value lies on the border of two
    # codes; one code is 1/127 of its row's largest, and these logits are of order 0.1
    assert (out - want).abs().max() < 2e-3
    assert (out - model(idx)["logits"]).abs().max() < 0.05  # near the unquantized model


@pytest.mark.parametrize("batch", [1, 6])
def test_generation_through_the_captured_decoder(dev, batch):
    qm, _ = g.quantize_model(_tiny(dev, 1), 8, act_bits=8)
    prompt = OM.benchmark_prompt(211, batch, 9).to(dev)
    dec = g.make_decoder(qm, batch, 32)
    assert isinstance(dec, g.GraphDecoder)
    with pytest.raises(ValueError, match="activations"):
        g.FusedDecoder(qm, batch, 32)
    out = dec.run(prompt, 12)
    assert out.shape == (batch, 21) and torch.equal(out[:, :9], prompt)
    assert torch.equal(dec.run(prompt, 12), out)
    eager = g.generate(qm, prompt, 12)
    assert (eager == out).float().mean() > 0.9  # equal but for codes on a border


@pytest.mark.parametrize("batch,length", [(1, 7), (2, 40), (5, 64)])
def test_fused_prompt_blocks_are_the_separate_modules(dev, batch, length):
    """A prompt through the blocks with everything inside the Linears, against the same
    model with a hook on every module, which runs them one by one."""
    qm, _ = g.quantize_model(_tiny(dev, 6), 8, act_bits=8)
    idx = (torch.arange(batch * length, device=dev) * 13 % 211).view(batch, length)
    with torch.no_grad():
        cache, plain_cache = g.KVCache.empty(2), g.KVCache.empty(2)
        fused = qm(idx, cache=cache)["logits"]
        hooks = [m.register_forward_hook(lambda *a: None) for m in qm.modules()]
        plain = qm(idx, cache=plain_cache)["logits"]
        for h in hooks:
            h.remove()
    assert not torch.equal(fused, torch.zeros_like(fused))
    assert (fused - plain).abs().max() < 2e-3  # equal but for codes on a border (1/127 of a row's largest)
    for a, b in zip(cache.keys + cache.values, plain_cache.keys + plain_cache.values):
        assert (a - b).abs().max() < 2e-2


def test_cached_steps_equal_the_whole_window(dev):
    """Prefill and single-token steps over a cache against one forward pass: a
    token's codes depend on its own row alone."""
    qm, _ = g.quantize_model(_tiny(dev, 2), 8, act_bits=8)
    idx = (torch.arange(24, device=dev) * 7 % 211).view(2, 12)
    whole = qm(idx)["logits"]
    cache = g.KVCache.empty(2)
    parts = [qm(idx[:, :5], cache=cache)["logits"]]
    for t in range(5, 12):
        parts.append(qm(idx[:, t : t + 1], cache=cache)["logits"])
    assert (torch.cat(parts, dim=1) - whole).abs().max() < 2e-3


def test_packed_checkpoint_round_trip(dev, tmp_path):
    model = _tiny(dev, 3)
    for bits in (8, 4, 3):
        qm, stats = g.quantize_model(model, bits, act_bits=8, save_to=tmp_path / f"m{bits}.pt")
        back = g.load_packed(_tiny(dev, 4), tmp_path / f"m{bits}.pt")
        for a, b in zip(qm.modules(), back.modules()):
            if isinstance(a, g.QuantLinear):
                assert b.fmt == "w8a8" and torch.equal(a.codes, b.codes) and torch.equal(a.scale, b.scale)
        idx = torch.arange(16, device=dev).view(1, 16)
        assert torch.equal(qm(idx)["logits"], back(idx)["logits"])
    again = copy.deepcopy(qm)
    again.load_state_dict(qm.state_dict())
    assert torch.equal(again(idx)["logits"], qm(idx)["logits"])


def test_experiment_takes_activation_schemes(dev):
    data = g.SyntheticTokenStream(211, 700, 32)
    table = g.run_quantization_table(_tiny(dev, 5), data, n_chunks=2, batches_per_chunk=1, batch_size=2, speed=False,
                                     schemes=(("int8", 8, "per_channel", False),
                                              ("int8, int8 activations", 8, "per_channel", False, 8)),
                                     token_scores=True)
    assert [r["label"] for r in table["rows"]] == ["int8", "int8, int8 activations"]
    assert table["rows"][1]["act_bits"] == 8 and "act_bits" not in table["rows"][0]
    for r in table["rows"]:
        assert abs(r["quality"]["loss_mean"] - table["baseline"]["loss_mean"]) < 0.05
        assert 0.0 < r["quality"]["entropy_mean"] < 5.5 and 0.0 <= r["quality"]["top1_accuracy"] <= 1.0


def test_refusals(dev):
    with pytest.raises(ValueError, match="8 bits only"):
        g.quantize_linear(torch.nn.Linear(8, 8).to(dev), 8, act_bits=4)
    with pytest.raises(ValueError, match="group_size"):
        g.quantize_model(_tiny(dev), 4, group_size=64, act_bits=8)
    with pytest.raises(ValueError, match="2-D int8"):
        g.QuantLinear(torch.zeros(4, 4, device=dev), torch.ones(4, device=dev), None, 4, 4, 8, "per_channel", "w8a8")
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        g.quantize_tokens(torch.zeros(2, 2, dtype=torch.float64, device=dev))
    q, s, b = _weight(8, 16, 1)
    with pytest.raises(ValueError, match="last dimension"):
        _linear(q, s, b, dev)(torch.zeros(2, 15, device=dev))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        _linear(q, s, b, dev)(torch.zeros(2, 16))


@pytest.mark.parametrize("m", [2, 40])
def test_a_module_cast_to_another_type_is_refused(dev, m):
    """The kernels read the scales and the bias as float32: a cast module would send
    them past the buffers' ends."""
    for bias in (torch.zeros(24, device=dev), None):
        lin = g.QuantLinear(torch.ones(24, 64, dtype=torch.int8, device=dev), torch.ones(24, device=dev), bias, 64, 24, 8,
                            "per_channel", "w8a8").to(torch.bfloat16)
        x = torch.ones(m, 64, device=dev)
        with pytest.raises(TypeError, match="float32"):
            lin(x)
        with pytest.raises(TypeError, match="float32"):
            lin(x.bfloat16())
        with pytest.raises(TypeError, match="float32"):
            lin.weight
        assert lin.forward_prefill(x) is None


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_more_rows_than_one_launch_takes(dev, dtype):
    m, k, n = (1 << 22) + 37, 12, 3
    gen = torch.Generator(device=dev).manual_seed(21)
    x = torch.randn(m, k, generator=gen, device=dev).to(dtype)
    qx, sx = g.quantize_tokens(x)
    q2, s2 = g.quantize_tensor(x.float(), 8)
    assert torch.equal(qx, q2) and torch.equal(sx, s2)
    q, s, b = _weight(n, k, 22)
    y = _linear(q, s, b, dev)(x).double()
    core = (qx.double() @ q.to(dev).double().t()) * sx.double() * s.to(dev).double()
    want = core + b.to(dev).double()
    bound = core.abs() * 2.0**-22 + want.abs() * 2.0**-23
    if dtype is BF16:
        bound = bound + (want.abs() + bound) * 2.0**-8
    ok = bool(((y - want).abs() <= bound).all())
    assert ok
