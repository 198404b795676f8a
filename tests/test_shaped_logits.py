"""Shaped logits and gradient lists without a GPU: the oracle against its own differences and a written-out example, the mask table's layout, and
what the C ABI and the Python entry points refuse (every call here returns from its checks: pointers are never followed)."""
import ctypes
import os

import numpy as np
import pytest
import torch

import ps_vae_amd  # noqa: F401
from ps_vae_amd import hip, ops, optim
from oracle import shaping_ref

EINVAL, ETOOLARGE, EWORKSPACE = -1, -2, -3
P = 4096   # a non-null, 16-byte aligned stand-in for a device pointer


@pytest.fixture(scope='module')
def L():
    if not os.path.exists(hip.LIB_PATH):
        pytest.fail(f'{hip.LIB_PATH} not built (run __graft_entry__.build())')
    return hip.lib()


def desc(**kw):
    s = hip.Shaping(B=4, T=1, V=302, dtype=hip.F32, logits=P, ld_b=302, repetition=1.0, temperature=1.0)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_oracle_on_a_written_out_row():
    l = np.array([2.0, -1.0, 0.5, 4.0])
    y, slope, _ = shaping_ref.shaped_row(l, [0, 1, 1, -1, 9], repetition=2.0, presence=0.25, frequency=0.5, bias=np.array([0., 0., 1., 0.]),
                                         allowed=np.array([True, True, True, False]), temperature=0.5)
    assert y.tolist() == [(1.0 - 0.5 - 0.25) * 2, (-2.0 - 1.0 - 0.25) * 2, 3.0, -np.inf]
    assert slope.tolist() == [1.0, 4.0, 2.0, 0.0]
    assert shaping_ref.draw_row(y, 0.0)[0] == 0 and shaping_ref.draw_row(y, 1.0 - 2 ** -24)[0] == 2
    assert shaping_ref.draw_row(np.full(3, -np.inf), 0.5, empty=7)[:2] == (7, -np.inf)


def test_oracle_gradient_against_differences():
    rng = np.random.default_rng(0)
    V = 23
    l, ids = rng.normal(size=V) * 2, rng.integers(0, V, 9)
    kw = dict(repetition=1.3, presence=0.2, frequency=0.1, bias=rng.normal(size=V), allowed=rng.random(V) < 0.8, temperature=0.7)
    tok = int(np.nonzero(kw['allowed'])[0][3])
    y, slope, _ = shaping_ref.shaped_row(l, ids, **kw)
    _, d, _ = shaping_ref.log_prob_row(y, slope, tok, 1.7)
    h = 1e-6
    for i in range(V):
        v = []
        for step in (h, -h):
            x = l.copy()
            x[i] += step
            yy, sl, _ = shaping_ref.shaped_row(x, ids, **kw)
            v.append(1.7 * shaping_ref.log_prob_row(yy, sl, tok)[0])
        # central differences: h^2 |f'''| / 6 + rounding of the two values / h
        assert abs((v[0] - v[1]) / (2 * h) - d[i]) < 1e-8


@pytest.mark.parametrize('V', [1, 31, 32, 33, 302])
def test_pack_allowed_layout(V):
    m = torch.rand(5, V, generator=torch.Generator().manual_seed(V)) < 0.5
    m[1], m[2] = True, False
    w = ops.pack_allowed(m)
    assert w.dtype == torch.int32 and tuple(w.shape) == (5, (V + 31) // 32)
    assert np.array_equal(shaping_ref.unpack(w.numpy(), V), m.numpy())
    with pytest.raises(ValueError):
        ops.pack_allowed(m.int())
    with pytest.raises(ValueError):
        ops.pack_allowed(m[0])


def test_rejected_descriptions(L):
    def fwd(s, out=P, ld=302):
        return L.psvae_shape_logits_fwd(ctypes.byref(s) if s is not None else None, out, ld, None)

    assert fwd(desc(B=0)) == 0                                        # nothing to do
    assert fwd(None) == EINVAL
    bad = [dict(B=-1), dict(T=0), dict(V=0), dict(dtype=3), dict(dtype=-1), dict(logits=None), dict(logits=P + 2), dict(repetition=0.0),
           dict(repetition=float('nan')), dict(repetition=float('inf')), dict(temperature=0.0), dict(temperature=-1.0),
           dict(presence=float('inf')), dict(frequency=float('nan')), dict(L=3), dict(history_len=P), dict(L=-1, history=P),
           dict(L=(1 << 24) + 1, history=P), dict(state=P), dict(allowed=P, ld_allowed=10, S=0), dict(allowed=P, ld_allowed=9, S=2, state=P),
           dict(allowed=P, ld_allowed=10, S=3)]
    for kw in bad:
        assert fwd(desc(**kw)) == EINVAL, kw
        assert L.psvae_last_error().startswith(b'psvae_shape_logits_fwd')
    assert fwd(desc(), out=None) == EINVAL and fwd(desc(), ld=301) == EINVAL and fwd(desc(), out=P + 2) == EINVAL
    assert fwd(desc(V=(1 << 30) + 1, ld_b=1 << 31), ld=1 << 31) == ETOOLARGE
    assert fwd(desc(B=1 << 20, T=1 << 12)) == ETOOLARGE               # 2^32 rows
    assert fwd(desc(B=1 << 20, V=1 << 22, ld_b=1 << 22), ld=1 << 22) == ETOOLARGE   # more workgroups than a launch holds

    bwd = lambda s, g=P, d=P, ld=302: L.psvae_shape_logits_bwd(ctypes.byref(s), g, 302, 0, d, ld, None)   # noqa: E731
    assert bwd(desc(B=0)) == 0 and bwd(desc(), g=None) == EINVAL and bwd(desc(), d=None) == EINVAL and bwd(desc(), ld=300) == EINVAL
    assert bwd(desc(), g=P + 1) == EINVAL


def test_rejected_log_prob_and_draw(L):
    wide = dict(V=20000, ld_b=20000)
    assert L.psvae_shaped_log_prob_workspace_bytes(ctypes.byref(desc())) == 0            # a row fits a wave
    need = L.psvae_shaped_log_prob_workspace_bytes(ctypes.byref(desc(**wide)))
    assert need > 0 and L.psvae_shaped_log_prob_workspace_bytes(None) == 0

    def lp(s, tok=P, out=P, stats=P, ws=P, n=1 << 30):
        return L.psvae_shaped_log_prob_fwd(ctypes.byref(s), tok, out, stats, ws, n, None)

    assert lp(desc(B=0)) == 0
    for kw in (dict(tok=None), dict(out=None), dict(stats=None), dict(stats=P + 4)):
        assert lp(desc(), **kw) == EINVAL, kw
    for kw in (dict(n=need - 1), dict(ws=None), dict(ws=P + 4)):
        assert lp(desc(**wide), **kw) == EWORKSPACE, kw

    def lpb(s, tok=P, stats=P, g=P, d=P, ld=302):
        return L.psvae_shaped_log_prob_bwd(ctypes.byref(s), tok, stats, g, d, ld, None)

    assert lpb(desc(B=0)) == 0
    for kw in (dict(tok=None), dict(stats=None), dict(g=None), dict(d=None), dict(ld=301), dict(d=P + 2), dict(stats=P + 4)):
        assert lpb(desc(), **kw) == EINVAL, kw

    need = L.psvae_shaped_draw_workspace_bytes(ctypes.byref(desc(**wide)))
    assert need > 0

    def draw(s, u=P, tok=P, out=P, ws=P, n=1 << 30):
        return L.psvae_shaped_draw(ctypes.byref(s), u, 1, -1, tok, out, ws, n, None)

    assert draw(desc(B=0)) == 0
    assert draw(desc(T=2)) == EINVAL
    for kw in (dict(u=None), dict(tok=None), dict(out=None)):
        assert draw(desc(), **kw) == EINVAL, kw
    for kw in (dict(n=need - 1), dict(ws=None), dict(ws=P + 8)):
        assert draw(desc(**wide), **kw) == EWORKSPACE, kw


def lists(ptrs, numel, types):
    n = len(ptrs)
    return ((ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numel), (ctypes.c_int32 * n)(*types))


def test_rejected_gradient_lists(L):
    def norm(ptrs, numel, types, out=P, ws=P, nbytes=1 << 30, n=None):
        a, b, c = lists(ptrs, numel, types)
        return L.psvae_grad_norm(len(ptrs) if n is None else n, a, b, c, out, ws, nbytes, None)

    big = 1 << 20
    for ptrs, numel, types in (([None], [3], [0]), ([P + 2], [3], [0]), ([P + 1], [3], [1]), ([P], [-1], [0]), ([P], [1 << 41], [0]), ([P], [3], [3])):
        assert norm(ptrs, numel, types) == EINVAL, (ptrs, numel, types)
    assert norm([P], [3], [0], out=None) == EINVAL and norm([P], [3], [0], n=-1) == EINVAL
    assert norm([P], [3], [0], ws=None) == EWORKSPACE and norm([P], [3], [0], nbytes=7) == EWORKSPACE and norm([P], [3], [0], ws=P + 8) == EWORKSPACE
    assert L.psvae_grad_norm_workspace_bytes(0) == 0 and L.psvae_grad_norm_workspace_bytes(2) == L.psvae_grad_norm_workspace_bytes(200) > 0

    def clip(ptrs, numel, types, outs, out_types, max_norm=1.0, out=P, ws=P):
        a, b, c = lists(ptrs, numel, types)
        d, _, e = lists(outs, numel, out_types)
        return L.psvae_clip_grads(len(ptrs), a, b, c, d, e, max_norm, out, ws, 1 << 30, None)

    assert clip([P], [3], [0], [None], [0]) == EINVAL and clip([P], [3], [0], [P], [7]) == EINVAL
    assert clip([P], [3], [0], [P], [0], max_norm=-1.0) == EINVAL and clip([P], [3], [0], [P], [0], max_norm=float('nan')) == EINVAL
    assert clip([P], [3], [0], [P], [0], out=None) == EINVAL and clip([P], [3], [0], [P], [0], ws=None) == EWORKSPACE
    # outputs that share memory: one tensor twice, a slice that reaches into the next, an output over another gradient, in place as another type
    for case in (([P, P], [8, 8], [0, 0], [P, P], [0, 0]),
                 ([big, 2 * big], [8, 8], [0, 0], [P, P + 28], [0, 0]),
                 ([big, 2 * big], [8, 8], [0, 0], [2 * big + 16, P], [0, 0]),
                 ([big], [8], [1], [big], [0]),
                 ([big, big + 4], [8, 1], [0, 0], [big, P], [0, 0])):
        assert clip(*case) == EINVAL, case
        assert b'overlaps' in L.psvae_last_error()


def test_python_entry_points_refuse():
    x = torch.zeros(2, 5)
    for call in (lambda: ops.shape_logits(x), lambda: ops.shaped_log_prob(x, torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.shaped_draw(x, torch.zeros(2)), lambda: optim.grad_norm([x]), lambda: optim.clip_grads([x], 1.0)):
        with pytest.raises(RuntimeError, match='GPU tensors'):
            call()
    with pytest.raises(ValueError, match='history'):
        ops.shape_logits(x, repetition=1.2)
    with pytest.raises(ValueError, match='gradient'):
        ops.shape_logits(x, bias=torch.zeros(5, requires_grad=True))
    with pytest.raises(RuntimeError):
        optim.grad_norm([])
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(x)], 1.0)) == 0.0   # no gradients: nothing to do
