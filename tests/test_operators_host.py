"""Refusals of the int8-activation Linear and the token scores that need no GPU:
the C ABI's argument checks (nothing is launched on bad input) and the Python
errors raised before a device is touched."""

from __future__ import annotations

import pytest
import torch

import gpt2_harness_amd as g
from gpt2_harness_amd import _lib

EINVAL, EALIGN, EUNSUPPORTED, EWORKSPACE = -1, -3, -4, -5


def test_quantize_tokens_arguments():
    f = _lib.load().tiq_quantize_tokens
    assert f(None, 0, 0, 4, 4, None, 4, None, None) == 0
    assert f(None, 0, 4, 0, 4, None, 4, None, None) == 0
    assert f(None, 0, 4, 4, 4, None, 4, None, None) == EINVAL
    assert f(16, 2, 4, 4, 4, 16, 4, 16, None) == EINVAL       # no such type
    assert f(16, 0, -1, 4, 4, 16, 4, 16, None) == EINVAL
    assert f(16, 0, 4, 4, 3, 16, 4, 16, None) == EINVAL       # rows overlap
    assert f(16, 0, 4, 4, 4, 16, 3, 16, None) == EINVAL
    assert f(18, 0, 4, 4, 4, 16, 4, 16, None) == EALIGN
    assert f(17, 1, 4, 4, 4, 16, 4, 16, None) == EALIGN
    assert f(16, 0, 1 << 31, 4, 4, 16, 4, 16, None) == EUNSUPPORTED


def test_tiles_arguments():
    L = _lib.load()
    assert L.tiq_w8a8_tiles_bytes(0, 5) == 0 and L.tiq_w8a8_tiles_bytes(5, -1) == 0
    assert L.tiq_w8a8_tiles_bytes(1, 1) == 2048 and L.tiq_w8a8_tiles_bytes(33, 65) == 2 * 4 * 1024
    assert L.tiq_w8a8_tiles_bytes(4800, 1600) == 4800 * 1600
    for f, extra in ((L.tiq_w8a8_tile, (4,)), (L.tiq_w8a8_untile, ())):
        assert f(None, 0, 4, *extra, None, None) == 0
        assert f(None, 4, 4, *extra, None, None) == EINVAL
        assert f(16, -4, 4, *extra, 16, None) == EINVAL
    assert L.tiq_w8a8_tile(16, 4, 4, 3, 16, None) == EINVAL
    assert L.tiq_w8a8_tile(16, 4, 4, 4, 24, None) == EALIGN


def test_linear_w8a8_arguments():
    L = _lib.load()
    f = L.tiq_linear_w8a8
    need = L.tiq_linear_w8a8_workspace(0, 17, 64, 5)
    assert need >= 32 * 64 + 32 * 4 and L.tiq_linear_w8a8_workspace(0, 0, 64, 5) == 0
    assert L.tiq_linear_w8a8_workspace(2, 17, 64, 5) == 0
    # few rows the product quantizes itself: of 16 bytes at least, 32 KB of codes at most
    assert L.tiq_linear_w8a8_workspace(0, 8, 4096, 5) == 0 and L.tiq_linear_w8a8_workspace(0, 8, 4097, 5) > 0
    assert L.tiq_linear_w8a8_workspace(0, 16, 768, 5) == 0 and L.tiq_linear_w8a8_workspace(0, 16, 1600, 5) > 0
    assert L.tiq_linear_w8a8_workspace(0, 4, 64, 5) == 0 and L.tiq_linear_w8a8_workspace(0, 4, 3, 5) > 0
    assert L.tiq_linear_w8a8_workspace(1, 4, 8, 5) == 0 and L.tiq_linear_w8a8_workspace(1, 4, 7, 5) > 0
    ok = dict(x=16, xd=0, M=17, K=64, ldx=64, w=16, s=16, b=None, N=5, y=16, yd=0, ldy=5, ws=16, nb=need)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None)

    assert call(M=0) == 0 and call(N=0, ldy=0) == 0
    for bad in (dict(xd=2), dict(yd=-1), dict(M=-1), dict(K=0), dict(x=None), dict(w=None), dict(s=None), dict(y=None),
                dict(ldx=63), dict(ldy=4)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(x=18), dict(xd=1, x=17), dict(w=24), dict(y=18), dict(s=18), dict(b=18)):
        assert call(**bad) == EALIGN, bad
    for bad in (dict(ws=None), dict(nb=need - 1), dict(ws=24)):
        assert call(**bad) == EWORKSPACE, bad
    assert call(K=131073, ldx=131073, nb=1 << 40) == EUNSUPPORTED
    assert call(M=1 << 31, N=1 << 20, ldy=1 << 20, nb=1 << 60) == EUNSUPPORTED
    assert call(M=4, N=(1 << 25) + 1, ldy=1 << 26) == EUNSUPPORTED


def test_linear_w8a8_prefill_arguments():
    L = _lib.load()
    f = L.tiq_linear_w8a8_prefill
    need = L.tiq_linear_w8a8_prefill_workspace(3, 64, 5)
    assert need >= 32 * 64 + 32 * 4
    for size in ((0, 64, 5), (3, 3, 5), (3, 8193, 5), (3, 64, 0)):
        assert L.tiq_linear_w8a8_prefill_workspace(*size) == 0
    ok = dict(x=16, M=3, K=64, ldx=64, w=16, s=16, b=None, N=5, y=16, ldy=5, lw=None, lb=None, eps=1e-5, gelu=0, r=None,
              ldr=0, ws=16, nb=need)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None)

    assert call(M=0) == 0 and call(N=0) == 0
    for bad in (dict(M=-1), dict(K=0), dict(x=None), dict(w=None), dict(s=None), dict(y=None), dict(ldx=63), dict(ldy=4),
                dict(lw=16), dict(lb=16), dict(lw=16, lb=16, gelu=1), dict(r=16, ldr=4)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(x=18), dict(w=24), dict(y=18), dict(r=18, ldr=5), dict(lw=18, lb=16)):
        assert call(**bad) == EALIGN, bad
    for bad in (dict(ws=None), dict(nb=need - 1), dict(ws=24)):
        assert call(**bad) == EWORKSPACE, bad
    assert call(K=8256, ldx=8256, nb=1 << 40) == EUNSUPPORTED and call(K=3) == EUNSUPPORTED


def test_token_scores_arguments():
    L = _lib.load()
    ok = dict(x=16, d=0, batch=1, rows=2, sb=0, sr=9, v=9, t=16, ignore=-100, top=0, lp=16, h=16, st=None, ids=None,
              tlp=None, ws=16, nb=1 << 30)

    def call(**kw):
        return L.tiq_token_logprobs(*{**ok, **kw}.values(), None)

    assert call(rows=0) == 0 and call(batch=0) == 0
    for bad in (dict(d=2), dict(batch=-1), dict(rows=-1), dict(v=0), dict(top=-1), dict(top=10), dict(v=100, top=65),
                dict(x=None), dict(t=None), dict(lp=None), dict(h=None), dict(top=1), dict(top=1, ids=16)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(x=18), dict(d=1, x=17), dict(t=20)):
        assert call(**bad) == EALIGN, bad
    assert call(v=(1 << 30) + 1) == EUNSUPPORTED and call(batch=1 << 20, rows=1 << 20) == EUNSUPPORTED

    ok = dict(x=16, d=0, batch=1, rows=2, sb=0, sr=9, v=9, t=16, ignore=-100, st=16, h=16, gl=16, gh=None, top=0,
              ids=None, gt=None, grad=16)

    def back(**kw):
        return L.tiq_token_logprobs_grad(*{**ok, **kw}.values(), None)

    assert back(rows=0) == 0
    for bad in (dict(st=None), dict(h=None), dict(grad=None), dict(gt=16), dict(gt=16, top=2), dict(d=5)):
        assert back(**bad) == EINVAL, bad
    assert back(grad=18) == EALIGN


def test_python_errors_before_a_device():
    x, t = torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        g.token_logprobs(x, t)
    with pytest.raises(TypeError, match="torch.Tensor"):
        g.token_logprobs([[1.0]], t)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        g.quantize_tokens(x)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        g.QuantLinear(torch.zeros(4, 4, dtype=torch.int8), torch.ones(4), None, 4, 4, 8, "per_channel", "w8a8")
    with pytest.raises(ValueError, match="8 bits only"):
        g.quantize_linear(torch.nn.Linear(4, 4), 8, act_bits=7)
    with pytest.raises(ValueError, match="group_size"):
        g.quantize_linear(torch.nn.Linear(4, 4), 4, group_size=2, act_bits=8)
