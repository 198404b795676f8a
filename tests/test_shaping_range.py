"""Repetition and temperature at the ends of float32's range: their reciprocals have to be numbers too, so 2^-126 .. 2^126 is what the operators
take, all three alike."""
import ctypes
import os

import numpy as np
import pytest
import torch

import ps_vae_amd  # noqa: F401
from ps_vae_amd import hip, ops, optim  # noqa: F401
from oracle import shaping_ref

EINVAL = -1
P = 4096   # a non-null, 16-byte aligned stand-in for a device pointer: every call here returns from its checks
U = 2.0 ** -24
BELOW, LOW, HIGH, ABOVE = 2.0 ** -126 * (1 - 2.0 ** -23), 2.0 ** -126, 2.0 ** 126, 2.0 ** 126 * (1 + 2.0 ** -23)


def test_numbers_outside_are_refused():
    if not os.path.exists(hip.LIB_PATH):
        pytest.fail(f'{hip.LIB_PATH} not built (run __graft_entry__.build())')
    L = hip.lib()

    def fwd(B=4, **kw):
        s = hip.Shaping(B=B, T=1, V=302, dtype=hip.F32, logits=P, ld_b=302, repetition=1.0, temperature=1.0)
        for k, v in kw.items():
            setattr(s, k, v)
        # (an output of no rows' length: a description that passes is refused for that)
        return L.psvae_shape_logits_fwd(ctypes.byref(s), P, 301, None)
    for name in ('repetition', 'temperature'):
        for v in (2.0 ** -149, 1e-40, BELOW, ABOVE, 3e38):
            assert fwd(B=0, **{name: v}) == EINVAL, (name, v)
            assert b'2^-126' in L.psvae_last_error()
        for v in (LOW, 1e-30, 1e30, HIGH):
            assert fwd(B=0, **{name: v}) == 0, (name, v)


@pytest.mark.gpu
@pytest.mark.parametrize('V', [60, 5000])
def test_values_from_the_device(V):
    """Inside the range the values are the oracle's; outside all three operators say NaN."""
    if not torch.cuda.is_available():
        pytest.fail('GPU tests need a GPU')
    d = torch.device('cuda:0')
    ends = [BELOW, 1e-40, 2.0 ** -149, ABOVE, 3e38, LOW, HIGH, 1.0]
    bad = torch.tensor([True] * 5 + [False] * 3)
    values = torch.tensor(ends, device=d)
    g = torch.Generator().manual_seed(V)
    x = (torch.rand(8, V, generator=g) - 0.5).to(d)
    u = torch.full((8,), 0.5, device=d)
    for key, kw in (('temperature', {}), ('repetition', dict(history=torch.arange(V).repeat(8, 1).to(d)))):
        kw = dict(kw, **{key: values})
        y = ops.shape_logits(x, **kw)
        assert torch.equal(torch.isnan(y).all(1).cpu(), bad) and torch.equal(torch.isnan(y).any(1).cpu(), bad), key
        tok, lp = ops.shaped_draw(x, u, empty_token=-7, **kw)
        assert torch.equal((tok == -7).cpu(), bad) and torch.equal(torch.isnan(lp).cpu(), bad), key
        leaf = x.clone().requires_grad_(True)
        score = ops.shaped_log_prob(leaf, tok.clamp(min=0), **kw)
        assert torch.equal(torch.isnan(score.detach()).cpu(), bad), key
        for r in (5, 6, 7):
            past = range(V) if key == 'repetition' else []
            want, _, scale = shaping_ref.shaped_row(x[r].double().cpu().numpy(), past, **{key: ends[r]})
            # a quotient by a power of two is exact but where it falls below the smallest normal number, 2^-126: half a step there is 2^-150
            assert (np.abs(y[r].double().cpu().numpy() - want) <= 8 * U * scale + 2.0 ** -149).all(), (key, r)
