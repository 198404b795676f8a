"""ops.shape_logits / shaped_log_prob / shaped_draw on the GPU against the float64 oracle, at the widths, strides, masks, histories and values where
each can go wrong.

Tolerances.  u = 2^-24 is half a step of float32, h(t) = finfo(t).eps / 2 half a step of the output type.  With S the oracle's `scale` (the
largest intermediate of a value, divided by the temperature):
  value      at most 8 rounded operations on intermediates of at most S:  D = 8 u S, then one rounding to the output type
  log-prob   value and logsumexp are off by D each; the sum of exponentials is a chain of fewer than 80 additions, each exponential off by
             (|y - m| + 3) 2u relative and weighted by itself (t e^-t <= 0.4): 90 u in all; the last operations round values of |y|, |m|, |log s|
  gradient   p is off by p (2 D + 90 u) + 8 u p, the difference and the products by 4 u; then the output type's rounding"""
import numpy as np
import pytest
import torch

from oracle import shaping_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def dev():
    if not torch.cuda.is_available():
        pytest.fail('GPU tests need a GPU')
    return torch.device('cuda:0')


def half_step(dtype, y):
    """Half a step of `dtype` at |y|, denormals included."""
    f = torch.finfo(dtype)
    return np.maximum(f.eps / 2 * np.abs(y), f.tiny * f.eps / 2)


def make(B, T, V, L, dtype, seed, *, penalties=True, bias=1, states=7, temperature=True, dims=None, nasty=True):
    """A call's tensors on the host.  dims 2: logits [B, V]; 3: [B, T, V]."""
    g = torch.Generator().manual_seed(seed)
    dims = (3 if T > 1 else 2) if dims is None else dims
    rows = (B,) if dims == 2 else (B, T)
    c = dict(logits=(torch.randn(*rows, V, generator=g) * 3).to(TYPES[dtype]))
    kw = {}
    if penalties:
        ids = (V * torch.rand(B, L, generator=g) ** 3).long().clamp(max=V - 1)
        if nasty and L > 3:     # ids that no vocabulary holds
            ids[:, 1], ids[0, 2], ids[-1, 0] = -1, V, 1 << 40
        kw['history'] = ids
        lens = torch.randint(0, L + 1, rows, generator=g)
        if nasty:
            lens.view(-1)[0], lens.view(-1)[-1] = 0, L + 5      # nothing seen; longer than the history: cut
            if lens.numel() > 2:
                lens.view(-1)[1] = -3
        kw['history_len'] = lens.int()
        kw['repetition'] = 1 + torch.rand(B, generator=g) / 2
        kw['presence'], kw['frequency'] = torch.rand(B, generator=g), torch.rand(B, generator=g) / 3
    if bias:
        kw['bias'] = torch.randn(V, generator=g) if bias == 1 else torch.randn(B, V, generator=g)
    if states:
        allowed = torch.rand(states, V, generator=g) < 0.6
        if states > 2:
            allowed[1] = False
            allowed[2] = False
            allowed[2, V - 1] = True          # one token left: the last
        from ps_vae_amd import ops
        kw['allowed'] = ops.pack_allowed(allowed)
        s = torch.randint(-1, states + (1 if nasty else 0), rows, generator=g)     # -1: all, `states`: none
        if states > 2:
            s.view(-1)[:4] = torch.tensor([1, 2, -1, states if nasty else 0])[:s.numel()]
        kw['state'] = s.int()
    if temperature:
        kw['temperature'] = 0.5 + torch.rand(B, generator=g)
    c['kw'] = kw
    c['tokens'] = torch.randint(0, V, rows, generator=g)
    if nasty and c['tokens'].numel() > 5:
        c['tokens'].view(-1)[4], c['tokens'].view(-1)[5] = -1, V
    c['uniforms'] = torch.rand(B, generator=g)
    c['g'] = torch.randn(*rows, generator=g)
    return c


def oracle_rows(c):
    """(y, slope, scale) [R, V] of a call."""
    x = c['logits']
    B, V = x.shape[0], x.shape[-1]
    T = x.shape[1] if x.dim() == 3 else 1
    kw = c['kw']
    flat = x.double().reshape(B * T, V).numpy()
    table = shaping_ref.unpack(kw['allowed'].numpy(), V) if 'allowed' in kw else None

    def of(name, b, r, neutral):
        v = kw.get(name)
        if v is None:
            return neutral
        return float(v) if not torch.is_tensor(v) else float(v.reshape(-1)[r if v.numel() == B * T and v.dim() == x.dim() - 1 else b])
    out = []
    for r in range(B * T):
        b = r // T
        ids = []
        if kw.get('history') is not None:
            n = int(of('history_len', b, r, kw['history'].shape[1]))
            ids = kw['history'][b, :max(0, n)].numpy()
        bias = kw.get('bias')
        if bias is not None:
            bias = (bias if bias.dim() == 1 else bias[b]).double().numpy()
        allowed = None
        if table is not None:
            s = int(of('state', b, r, 0 if len(table) == 1 else b))
            allowed = None if s < 0 else (table[s] if s < len(table) else np.zeros(V, bool))
        f32 = lambda v: float(np.float32(v))   # noqa: E731
        out.append(shaping_ref.shaped_row(flat[r], ids, f32(of('repetition', b, r, 1.0)), f32(of('presence', b, r, 0.0)),
                                          f32(of('frequency', b, r, 0.0)), bias, allowed, f32(of('temperature', b, r, 1.0))))
    return [np.stack(v) for v in zip(*out)]


def on(c, device):
    return {k: v.to(device) if torch.is_tensor(v) else v for k, v in c['kw'].items()}


def close(got, want, tol, what):
    got = got.detach().double().cpu().numpy().reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)]), what
    ok = np.isfinite(want)
    assert np.array_equal(ok, np.isfinite(got)), what
    over = np.abs(got[ok] - want[ok]) - np.broadcast_to(tol, want.shape)[ok]
    assert over.size == 0 or over.max() <= 0, (what, float(over.max()), float(np.abs(got[ok] - want[ok]).max()))


def expect(c):
    """Everything the oracle says of a call, with tolerances."""
    y, slope, scale = oracle_rows(c)
    D = 8 * U * scale
    rows, V = y.shape
    tok, g = c['tokens'].reshape(-1).numpy(), c['g'].reshape(-1).double().numpy()
    lp, lp_tol = np.zeros(rows), np.zeros(rows)
    d, d_tol = np.zeros((rows, V)), np.zeros((rows, V))
    for r in range(rows):
        lp[r], d[r], p = shaping_ref.log_prob_row(y[r], slope[r], int(tok[r]), g[r])
        live = np.isfinite(y[r])
        if not live.any():
            continue
        Dm, big = D[r][live].max(), np.abs(y[r][live]).max()
        lp_tol[r] = 2 * Dm + 90 * U + 4 * U * (big + np.log(V))
        d_tol[r] = abs(g[r]) * slope[r] * (p * (2 * Dm + 98 * U) + 4 * U)
    return dict(y=y, y_tol=D, slope=slope, lp=lp, lp_tol=lp_tol, d=d, d_tol=d_tol)


def check_all(c, device, want=None):
    from ps_vae_amd import ops
    w = expect(c) if want is None else want
    t = c['logits'].dtype
    kw = on(c, device)
    x = c['logits'].to(device).requires_grad_(True)
    print('shape', flush=True)
    y = ops.shape_logits(x, **kw)
    assert y.dtype == t and y.shape == x.shape
    close(y, w['y'], w['y_tol'] + half_step(t, w['y']), 'shape')
    gy = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(t)
    dx, = torch.autograd.grad(y, x, gy.to(device))
    want_dx = gy.double().numpy().reshape(w['y'].shape) * w['slope']
    close(dx, want_dx, 4 * U * np.abs(want_dx) + half_step(t, want_dx), 'shape backward')
    print('log_prob', flush=True)
    lp = ops.shaped_log_prob(x, c['tokens'].to(device), **kw)
    assert lp.dtype == torch.float32 and lp.shape == c['tokens'].shape
    close(lp, w['lp'], w['lp_tol'], 'log_prob')
    dx, = torch.autograd.grad(lp, x, c['g'].to(device))
    assert dx.dtype == t and dx.shape == x.shape
    close(dx, w['d'], w['d_tol'] + half_step(t, w['d']), 'log_prob backward')
    with torch.no_grad():
        assert torch.equal(ops.shaped_log_prob(x, c['tokens'].to(device), **kw).nan_to_num(), lp.detach().nan_to_num())
    if x.dim() == 2:
        print('draw', flush=True)
        check_draw(c, w['y'], kw, device)


def check_draw(c, y, kw, device, empty=-7):
    from ps_vae_amd import ops
    u = c['uniforms']
    tok, lp = ops.shaped_draw(c['logits'].to(device), u.to(device), empty_token=empty, **kw)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32
    for r in range(len(y)):
        t, l, gap = shaping_ref.draw_row(y[r], float(u[r]), empty)
        got = int(tok[r])
        # the two sides' 64-bit sums differ by far less than 1e-12 of the total; u at a boundary to that is either side's (u = 0 has none)
        assert got == t or gap < 1e-12, (r, got, t, gap)
        if got == t:
            assert float(lp[r]) == l or abs(float(lp[r]) - l) <= 2 * U * abs(l) + 1e-9, (r, float(lp[r]), l)


WIDTHS = [1, 2, 7, 31, 33, 64, 302, 511, 512, 513, 1023, 1024, 1025, 2047, 2049, 8191, 8193, 20011]


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('V', WIDTHS)
def test_widths(V, dtype):
    check_all(make(9, 1, V, 40, dtype, seed=V), dev())


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('B,T,V', [(3, 5, 302), (2, 9, 1500), (1, 4, 9001), (5, 1, 40), (7, 2, 1)])
def test_positions(B, T, V, dtype):
    check_all(make(B, T, V, 17, dtype, seed=B * T + V, bias=2, dims=3), dev())


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('R,V', [(600, 8300), (130, 33000)])
def test_many_rows_of_wide_vocabularies(R, V, dtype):
    """Enough rows for the large units (the few-row calls above take the small ones); a slice of the rows against the oracle, the rest
    against the same rows called alone."""
    from ps_vae_amd import ops
    d = dev()
    c = make(R, 1, V, 300, dtype, seed=R)
    kw = on(c, d)
    n = 6
    first = dict(logits=c['logits'][:n], tokens=c['tokens'][:n], uniforms=c['uniforms'][:n], g=c['g'][:n],
                 kw={k: (v[:n] if k not in ('bias', 'allowed') else v) for k, v in c['kw'].items()})
    w = expect(first)
    x = c['logits'].to(d).requires_grad_(True)
    t = x.dtype
    y = ops.shape_logits(x, **kw)
    close(y[:n], w['y'], w['y_tol'] + half_step(t, w['y']), 'shape')
    lp = ops.shaped_log_prob(x, c['tokens'].to(d), **kw)
    close(lp[:n], w['lp'], w['lp_tol'], 'log_prob')
    dx, = torch.autograd.grad(lp, x, c['g'].to(d))
    close(dx[:n], w['d'], w['d_tol'] + half_step(t, w['d']), 'log_prob backward')
    tok, dlp = ops.shaped_draw(x.detach(), c['uniforms'].to(d), **kw)
    few = slice(R - 5, R)
    kw1 = {k: (v[few].contiguous() if k not in ('bias', 'allowed') else v) for k, v in kw.items()}
    x1 = x.detach()[few].requires_grad_(True)
    assert torch.equal(ops.shape_logits(x1, **kw1), y[few])
    tok1, dlp1 = ops.shaped_draw(x1.detach(), c['uniforms'].to(d)[few], **kw1)
    assert torch.equal(tok1, tok[few]) and torch.allclose(dlp1, dlp[few], rtol=2 * U, atol=1e-9)   # another tiling: the same picks
    lp1 = ops.shaped_log_prob(x1, c['tokens'].to(d)[few], **kw1)
    fin = torch.isfinite(lp[few])
    assert torch.equal(fin, torch.isfinite(lp1)) and float((lp1 - lp[few]).detach()[fin].abs().max()) <= 180 * U + 16 * U * 20


@pytest.mark.parametrize('which', ['none', 'penalties', 'bias', 'states', 'one_state', 'state_per_sequence', 'temperature', 'numbers', 'no_len',
                                   'empty_history'])
def test_options_alone(which):
    off = dict(penalties=False, bias=0, states=0, temperature=False)
    kw = {'none': {}, 'penalties': dict(penalties=True), 'bias': dict(bias=2), 'states': dict(states=5), 'one_state': dict(states=1),
          'state_per_sequence': dict(states=6), 'temperature': dict(temperature=True), 'numbers': dict(penalties=True, temperature=True),
          'no_len': dict(penalties=True), 'empty_history': dict(penalties=True)}[which]
    for V in (77, 3001):
        c = make(6, 1, V, 0 if which == 'empty_history' else 12, 'f32', seed=V, nasty=False, **{**off, **kw})
        if which in ('one_state', 'state_per_sequence'):
            del c['kw']['state']
        if which == 'numbers':
            c['kw'].update(repetition=1.25, presence=0.5, frequency=0.125, temperature=0.75)
        if which == 'no_len':
            del c['kw']['history_len']
        check_all(c, dev())


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_strides_and_alignment(dtype):
    """Logits, bias, history and masks that are views: odd row strides, odd starts, transposed sequences, reversed order of dimensions."""
    from ps_vae_amd import ops
    d = dev()
    for V in (45, 1333):
        c = make(4, 3, V, 9, dtype, seed=V, bias=2, dims=3)
        w = expect(c)
        kw = on(c, d)
        t = TYPES[dtype]
        big = torch.full((3, 4, V + 11), float('nan'), dtype=t, device=d)
        x = big[:, :, 3:3 + V].transpose(0, 1)                   # [4, 3, V], position-major, rows V + 11 apart, start 3
        x.copy_(c['logits'])
        pad = torch.full((4, V + 5), float('nan'), device=d)
        pad[:, 1:1 + V] = kw['bias']
        kw['bias'] = pad[:, 1:1 + V]
        hist = torch.zeros(4, 20, dtype=torch.int64, device=d)
        hist[:, 2:11] = kw['history']
        kw['history'] = hist[:, 2:11]
        W = kw['allowed'].shape[1]
        words = torch.zeros(kw['allowed'].shape[0], W + 3, dtype=torch.int32, device=d)
        words[:, 1:1 + W] = kw['allowed']
        kw['allowed'] = words[:, 1:1 + W]
        y = ops.shape_logits(x, **kw)
        close(y, w['y'], w['y_tol'] + half_step(t, w['y']), 'shape')
        leaf = x.detach().requires_grad_(True)                   # (keeps the strides)
        assert leaf.stride() == x.stride()
        y = ops.shape_logits(leaf, **kw)
        gy = torch.randn(3, 4, V, generator=torch.Generator().manual_seed(2)).to(t)
        dx, = torch.autograd.grad(y, leaf, gy.to(d).transpose(0, 1))
        want = gy.transpose(0, 1).double().numpy().reshape(w['y'].shape) * w['slope']
        close(dx, want, 4 * U * np.abs(want) + half_step(t, want), 'shape backward')
        dx, = torch.autograd.grad(ops.shape_logits(leaf, **kw).float().nan_to_num(neginf=0.).sum(), leaf)
        close(dx, w['slope'], 4 * U * w['slope'] + half_step(t, w['slope']), 'shape backward, expanded gradient')
        lp = ops.shaped_log_prob(leaf, c['tokens'].to(d), **kw)
        close(lp, w['lp'], w['lp_tol'], 'log_prob')
        dx, = torch.autograd.grad(lp, leaf, c['g'].to(d).t().contiguous().t())
        close(dx, w['d'], w['d_tol'] + half_step(t, w['d']), 'log_prob backward')
        # a draw from one position of the same buffer, uniforms and masks in columns of larger arrays
        cd = dict(logits=c['logits'][:, 1], uniforms=c['uniforms'], kw={})
        yd, _, _ = oracle_rows(cd)
        cols = torch.zeros(4, 6, device=d)
        cols[:, 2] = c['uniforms'].to(d)
        tok, lp = ops.shaped_draw(x[:, 1], cols[:, 2])
        for r in range(4):
            t0, l0, gap = shaping_ref.draw_row(yd[r], float(c['uniforms'][r]))
            assert int(tok[r]) == t0 or gap < 1e-12


@pytest.mark.parametrize('V', [50, 2500])
def test_masked_places_may_hold_anything(V):
    """NaN, infinities and the type's lowest value where the mask forbids: never looked at, forward or backward."""
    from ps_vae_amd import ops
    d = dev()
    for dtype in ('f32', 'bf16'):
        c = make(8, 1, V, 10, dtype, seed=3 * V, nasty=False)
        clean = expect(c)
        allowed = np.isfinite(clean['y'])
        x = c['logits'].clone()
        junk = torch.tensor([float('nan'), float('inf'), float('-inf'), torch.finfo(x.dtype).min, torch.finfo(x.dtype).max]).to(x.dtype)
        where = torch.from_numpy(~allowed)
        x[where] = junk[torch.arange(int(where.sum())) % 5]
        c['logits'] = x
        for k in ('y', 'lp', 'd'):
            assert not np.isnan(clean[k]).any()
        check_all(c, d, want=clean)


def test_values_that_are_allowed_and_not_finite():
    from ps_vae_amd import ops
    d = dev()
    for V in (60, 5000):
        x = torch.randn(6, V, generator=torch.Generator().manual_seed(1))
        x[0, 3] = float('nan')
        x[1, 4] = float('inf')
        x[2, 5] = float('-inf')
        x[3] = float('-inf')
        x[4] = torch.finfo(torch.float32).min            # a row masked by hand with the lowest value: uniform over it
        x = x.to(d)
        u = torch.full((6,), 0.5, device=d)
        tok, lp = ops.shaped_draw(x, u, temperature=0.5, empty_token=-3)
        assert tok.tolist()[:2] == [-3, -3] and torch.isnan(lp[:2]).all()
        assert 0 <= int(tok[2]) < V and int(tok[2]) != 5 and torch.isfinite(lp[2])
        assert int(tok[3]) == -3 and float(lp[3]) == float('-inf')
        assert abs(int(tok[4]) - V // 2) <= 1 and abs(float(lp[4]) + np.log(V)) < 1e-5
        t = torch.zeros(6, dtype=torch.int64, device=d)
        leaf = x.clone().requires_grad_(True)
        lp = ops.shaped_log_prob(leaf, t)
        assert torch.isnan(lp[:2]).all() and torch.isfinite(lp[2]) and float(lp[3].detach()) == float('-inf')
        assert abs(float(lp[4].detach()) + np.log(V)) < 1e-5
        dx, = torch.autograd.grad(lp, leaf, torch.ones(6, device=d))
        assert torch.isnan(dx[0]).any() and float(dx[2, 5]) == 0.0 and not dx[3].any()
        assert torch.isfinite(dx[2]).all() and torch.isfinite(dx[4:]).all()
        # tensors cannot be checked before the launch: what they spoil is NaN
        bad = torch.tensor([1.0, 0.0, -1.0, float('nan'), 1.0, float('inf')], device=d)
        y = ops.shape_logits(x.nan_to_num(0., 0., 0.), temperature=bad)
        assert torch.isnan(y).all(1).tolist() == [False, True, True, True, False, True]
        hist = torch.zeros(6, 1, dtype=torch.int64, device=d)
        y = ops.shape_logits(x.nan_to_num(0., 0., 0.), history=hist, repetition=bad)
        assert torch.isnan(y[:, 0]).tolist() == [False, True, True, True, False, True] and torch.isfinite(y[:, 1:]).all()


def test_rows_of_the_lowest_value_stay_uniform():
    """A row that holds the type's lowest value everywhere, at temperatures that round: equal values stay equal."""
    from ps_vae_amd import ops
    d = dev()
    for dtype in TYPES.values():
        for V in (60, 1000, 5000):
            x = torch.full((3, V), torch.finfo(dtype).min, dtype=dtype, device=d)
            T = torch.tensor([1.5, 3.0, 7.0], device=d)
            tok, lp = ops.shaped_draw(x, torch.full((3,), 0.5, device=d), temperature=T)
            assert bool(((tok - V // 2).abs() <= 1).all()) and bool(((lp + np.log(V)).abs() < 1e-5).all())
            leaf = x.requires_grad_(True)
            lp = ops.shaped_log_prob(leaf, torch.zeros(3, dtype=torch.int64, device=d), temperature=T)
            # y - m is exactly 0: what is left is the rounding of -log V and of the sum
            assert bool(((lp.detach() + np.log(V)).abs() < 1e-5).all())
            dx, = torch.autograd.grad(lp, leaf, torch.ones(3, device=d))
            want = -1 / (V * T.cpu().double().numpy())
            assert (np.abs(dx[:, 1:].double().cpu().numpy() - want[:, None]) <= 1e-5 * -want[:, None] + half_step(dtype, want)[:, None]).all()


def test_edges_of_the_draw():
    """u at 0, just under 1, at 1 and NaN; a single positive entry; probabilities that vanish next to the largest."""
    from ps_vae_amd import ops
    d = dev()
    for V in (9, 700, 4000, 30000):
        x = torch.full((6, V), -5.0)
        x[:, 1] = float('-inf')
        x[5] = float('-inf')
        x[5, V - 2] = -1000.0
        u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, float('nan'), 0.25, 0.999])
        tok, lp = ops.shaped_draw(x.to(d), u.to(d))
        assert tok.tolist()[:4] == [0, V - 1, V - 1, V - 1] and int(tok[5]) == V - 2 and float(lp[5]) == 0.0
        t0, l0, _ = shaping_ref.draw_row(x[4].double().numpy(), 0.25)
        assert int(tok[4]) == t0 and abs(float(lp[4]) - l0) <= 2 * U * abs(l0) + 1e-9
        x = torch.full((2, V), -2000.0)
        x[:, 4] = 0.0                                        # exp(-2000) is 0 in 64 bits: only one token has a probability
        tok, lp = ops.shaped_draw(x.to(d), torch.tensor([0.0, 0.9999]).to(d))
        assert tok.tolist() == [4, 4] and lp.tolist() == [0.0, 0.0]


def test_draw_frequencies():
    """200000 draws of one distribution: every bin within 5 standard deviations (independent numbers from a fixed seed: a fixed outcome)."""
    from ps_vae_amd import ops
    d = dev()
    n, V = 200000, 12
    x = torch.randn(1, V, generator=torch.Generator().manual_seed(4))
    p = torch.softmax(x[0].double() / 0.8, 0)
    u = torch.rand(n, generator=torch.Generator().manual_seed(5))
    tok, _ = ops.shaped_draw(x.expand(n, V).to(d), u.to(d), temperature=0.8)
    f = torch.bincount(tok.cpu(), minlength=V).double() / n
    assert bool(((f - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all())


def test_long_history_and_many_repeats():
    """History of 70000 ids (more than 16 bits count), most of them one token."""
    d = dev()
    for V in (100, 9000):
        c = make(2, 1, V, 70000, 'f32', seed=V, nasty=False, states=0)
        c['kw']['history'][:, ::2] = 3
        c['kw']['history_len'] = torch.tensor([70000, 66001], dtype=torch.int32)
        c['kw']['frequency'] = torch.tensor([1e-4, 2e-4])
        check_all(c, d)


def test_gradient_against_differences():
    """The kernel's gradient against central differences of the oracle in 64 bits."""
    from ps_vae_amd import ops
    d = dev()
    V, h = 37, 1e-6
    c = make(3, 1, V, 11, 'f32', seed=8, nasty=False)
    c['tokens'] = torch.tensor([V - 1, V - 1, 4])
    x = c['logits'].to(d).requires_grad_(True)
    dx, = torch.autograd.grad(ops.shaped_log_prob(x, c['tokens'].to(d), **on(c, d)), x, c['g'].to(d))
    w = expect(c)
    base = c['logits'].double()

    def lps(x64):
        y, slope, _ = oracle_rows(dict(c, logits=x64))
        return np.array([shaping_ref.log_prob_row(y[r], slope[r], int(c['tokens'][r]))[0] for r in range(3)])
    for i in range(V):
        e = torch.zeros(3, V, dtype=torch.float64)
        e[:, i] = h
        diff = lps(base + e) - lps(base - e)
        ok = np.isfinite(diff)
        want = c['g'].double().numpy() * np.where(ok, diff, 0.) / (2 * h)
        got = dx[:, i].double().cpu().numpy()
        assert (np.abs(got - want)[ok] <= w['d_tol'][ok, i] + 1e-7).all(), (i, got, want)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_a_run_is_the_row(dtype):
    """Enough rows that a workgroup has a whole one: a lane adds up to V / 256 terms.  The sum's share of the tolerance is V / 256 + 12 additions and
    the exponentials' 10 u in place of the 90 u above (which covers 80 additions)."""
    from ps_vae_amd import ops
    d = dev()
    R, V, n = 1030, 30001, 5
    more = (V / 256 + 12 + 10) * U
    c = make(R, 1, V, 200, dtype, seed=5)
    kw = on(c, d)
    first = dict(logits=c['logits'][:n], tokens=c['tokens'][:n], uniforms=c['uniforms'][:n], g=c['g'][:n],
                 kw={k: (v[:n] if k not in ('bias', 'allowed') else v) for k, v in c['kw'].items()})
    w = expect(first)
    x = c['logits'].to(d).requires_grad_(True)
    lp = ops.shaped_log_prob(x, c['tokens'].to(d), **kw)
    close(lp[:n], w['lp'], w['lp_tol'] + more, 'log_prob')
    dx, = torch.autograd.grad(lp, x, c['g'].to(d))
    close(dx[:n], w['d'], w['d_tol'] + more * np.abs(c['g'][:n].numpy())[:, None] * w['slope'] + half_step(x.dtype, w['d']), 'log_prob backward')
    tok, _ = ops.shaped_draw(x.detach(), c['uniforms'].to(d), **kw)
    for r in range(n):
        t, _, gap = shaping_ref.draw_row(w['y'][r], float(c['uniforms'][r]))
        assert int(tok[r]) == t or gap < 1e-12


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('R,V,L', [(1000, 8195, 300), (970, 12290, 6000), (970, 6001, 6500)])
def test_lines_with_seen_elements(R, V, L, dtype):
    """Runs of many steps, each with elements of the history in most of its lines; histories longer than a run has room for."""
    from ps_vae_amd import ops
    d = dev()
    n = 6
    c = make(R, 1, V, L, dtype, seed=R + L, bias=2)
    c['tokens'][:n // 2] = c['kw']['history'][:n // 2, -1].clamp(0, V - 1)          # half of the tokens seen, or likely to be
    kw = on(c, d)
    first = dict(logits=c['logits'][:n], tokens=c['tokens'][:n], g=c['g'][:n], kw={k: (v[:n] if k != 'allowed' else v) for k, v in c['kw'].items()})
    w = expect(first)
    x = c['logits'].to(d).requires_grad_(True)
    y = ops.shape_logits(x, **kw)
    close(y[:n], w['y'], w['y_tol'] + half_step(x.dtype, w['y']), 'shape')
    gy = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(x.dtype)
    dx, = torch.autograd.grad(y, x, gy.to(d))
    want = gy[:n].double().numpy() * w['slope']
    close(dx[:n], want, 4 * U * np.abs(want) + half_step(x.dtype, want), 'shape backward')
    lp = ops.shaped_log_prob(x, c['tokens'].to(d), **kw)
    close(lp[:n], w['lp'], w['lp_tol'], 'log_prob')
    dx, = torch.autograd.grad(lp, x, c['g'].to(d))
    close(dx[:n], w['d'], w['d_tol'] + half_step(x.dtype, w['d']), 'log_prob backward')
    # the last row against a call of its own, whose runs are others
    r = R - 1
    one = c['logits'][r:].to(d).requires_grad_(True)
    alone = {k: (v[r:] if k != 'allowed' else v) for k, v in kw.items()}
    assert torch.equal(ops.shape_logits(one, **alone), y[r:])


def test_offsets_past_32_bits():
    """Logits of more than 2^31 elements: the last rows come out as they do alone."""
    from ps_vae_amd import ops
    d = dev()
    R, V = 70000, 32003
    x = torch.empty(R, V, dtype=torch.bfloat16, device=d)
    x[-3:] = (torch.randn(3, V, generator=torch.Generator().manual_seed(1)) * 3).bfloat16().to(d)
    x[:-3] = 0.
    hist = torch.randint(0, V, (R, 20), generator=torch.Generator().manual_seed(2)).to(d)
    tok = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(3)).to(d)
    u = torch.rand(R, generator=torch.Generator().manual_seed(4)).to(d)
    opt = dict(repetition=1.3, presence=0.1, temperature=0.7)
    leaf = x[-3:].clone().requires_grad_(True)
    y = ops.shape_logits(x, history=hist, **opt)
    assert torch.equal(y[-3:], ops.shape_logits(leaf.detach(), history=hist[-3:], **opt)) and bool((y[0] <= 0).all())
    del y
    t, l = ops.shaped_draw(x, u, history=hist, **opt)
    t1, l1 = ops.shaped_draw(leaf.detach(), u[-3:], history=hist[-3:], **opt)
    assert torch.equal(t[-3:], t1) and torch.allclose(l[-3:], l1, rtol=4 * U, atol=1e-9)
    x.requires_grad_(True)
    lp = ops.shaped_log_prob(x, tok, history=hist, **opt)
    dx, = torch.autograd.grad(lp, x, torch.ones_like(lp))
    lp1 = ops.shaped_log_prob(leaf, tok[-3:], history=hist[-3:], **opt)
    dx1, = torch.autograd.grad(lp1, leaf, torch.ones_like(lp1))
    # another tiling adds the row's terms in another order: both sums are off by 90 u at most, one bfloat16 step where that tips a rounding
    assert bool(((lp[-3:] - lp1).abs() <= 180 * U + 8 * U * lp1.abs()).all())
    assert bool(((dx[-3:].float() - dx1.float()).abs() <= 2 ** -7 * dx1.float().abs() + 1e-30).all())


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_draw_over_unequal_levels(dtype):
    """Stretches of 512 logits at levels far apart, nothing or the type's lowest value: what a wave weighs its elements against fits only some."""
    from ps_vae_amd import ops
    d = dev()
    R, V = 250, 32003
    t = {'f32': torch.float32, 'bf16': torch.bfloat16}[dtype]
    gen = torch.Generator().manual_seed(8)
    levels = torch.tensor([0., 0., -2000., -700., 900., 400., 2e6, float('-inf'), torch.finfo(t).min])
    few = torch.randint(2, len(levels) + 1, (R, 1), generator=gen)             # how many of the levels a row has
    at = (torch.rand(R, (V + 511) // 512, generator=gen) * few).long().clamp(max=len(levels) - 1)
    x = (torch.randn(R, V, generator=gen) + levels[at].repeat_interleave(512, 1)[:, :V]).clamp(min=torch.finfo(t).min).to(t)
    x[:, ::7] = torch.where(levels[at].repeat_interleave(512, 1)[:, :V][:, ::7] == float('-inf'), torch.tensor(float('-inf'), dtype=t), x[:, ::7])
    allowed = torch.ones(2, V, dtype=torch.bool)
    allowed[1, torch.randint(0, V, (V - 40,), generator=gen)] = False
    state = torch.randint(-1, 2, (R,), generator=gen).int()
    u = torch.rand(R, generator=gen)
    tok, lp = ops.shaped_draw(x.to(d), u.to(d), allowed=ops.pack_allowed(allowed).to(d), state=state.to(d))
    for r in range(0, R, 3):
        y = x[r].double().numpy()
        if int(state[r]) >= 0:
            y = np.where(allowed[int(state[r])].numpy(), y, -np.inf)
        want, want_lp, gap = shaping_ref.draw_row(y, float(u[r]))
        # the running sum of 32003 doubles may be off by V half steps, 1.8e-12
        assert int(tok[r]) == want or gap < 2e-12, r
        if int(tok[r]) == want:
            assert abs(float(lp[r]) - want_lp) <= U * abs(want_lp) + 2e-12, r


def test_improbable_tokens():
    """u = 0 takes the first token of positive probability, however small: its score is exact, also far below the smallest double's logarithm's
    neighbourhood."""
    from ps_vae_amd import ops
    d = dev()
    for V in (20, 900, 6000):
        x = torch.zeros(3, V)
        x[0, 0], x[1, 0], x[2, 0] = -500., -700., -740.     # 2^-721, 2^-1010, 2^-1068 of the rest (the last below the normal doubles)
        tok, lp = ops.shaped_draw(x.to(d), torch.zeros(3, device=d))
        assert tok.tolist() == [0, 0, 0]
        want = torch.tensor([-500., -700., -740.], dtype=torch.float64) - np.log(V - 1.)
        # the third weight has 6 bits left
        assert bool(((lp.double().cpu() - want).abs() <= torch.tensor([1e-4, 1e-4, 2e-2])).all()), (V, lp)


def test_through_the_c_abi():
    """psvae_shaping as ctypes fills it: the same values as through the operator."""
    import ctypes
    from ps_vae_amd import hip, ops
    d = dev()
    for dims in (2, 3):
        c = make(4, 1 if dims == 2 else 3, 77, 9, 'bf16', seed=2, bias=2, dims=dims, states=5)
        kw = on(c, d)
        x = c['logits'].to(d)
        T = 1 if dims == 2 else 3
        s = hip.Shaping(B=4, T=T, V=77, dtype=hip.BF16, logits=x.data_ptr(), ld_b=x.stride(0), ld_t=x.stride(1) if dims == 3 else 0,
                        history=kw['history'].data_ptr(), ld_history=9, L=9, history_len=kw['history_len'].data_ptr(), len_per_row=int(dims == 3),
                        repetition_rows=kw['repetition'].data_ptr(), presence_rows=kw['presence'].data_ptr(), frequency_rows=kw['frequency'].data_ptr(),
                        temperature_rows=kw['temperature'].data_ptr(), repetition=1., temperature=1., bias=kw['bias'].data_ptr(), ld_bias=77,
                        allowed=kw['allowed'].data_ptr(), ld_allowed=3, S=5, state=kw['state'].data_ptr(), state_per_row=int(dims == 3))
        out = torch.empty_like(x)
        assert hip.lib().psvae_shape_logits_fwd(ctypes.byref(s), hip.ptr(out), 77, hip._stream()) == 0
        assert torch.equal(out, ops.shape_logits(x, **kw))
        assert hip.lib().psvae_shape_logits_fwd(ctypes.byref(s), hip.ptr(x), 77, hip._stream()) == 0     # in place
        assert torch.equal(out, x)


def test_in_place_over_a_wide_row():
    import ctypes
    from ps_vae_amd import hip, ops
    d = dev()
    c = make(3, 1, 20011, 300, 'f32', seed=12, states=0)
    kw = on(c, d)
    x = c['logits'].to(d)
    want = ops.shape_logits(x, **kw)
    s = hip.Shaping(B=3, T=1, V=20011, dtype=hip.F32, logits=x.data_ptr(), ld_b=20011, history=kw['history'].data_ptr(), ld_history=300, L=300,
                    history_len=kw['history_len'].data_ptr(), repetition_rows=kw['repetition'].data_ptr(), presence_rows=kw['presence'].data_ptr(),
                    frequency_rows=kw['frequency'].data_ptr(), temperature_rows=kw['temperature'].data_ptr(), repetition=1., temperature=1.,
                    bias=kw['bias'].data_ptr())
    assert hip.lib().psvae_shape_logits_fwd(ctypes.byref(s), hip.ptr(x), 20011, hip._stream()) == 0
    assert torch.equal(x, want)


def test_history_of_extreme_ids():
    """Ids at the ends of 64 bits are outside the vocabulary like any others."""
    from ps_vae_amd import ops
    d = dev()
    lo, hi = -2 ** 63, 2 ** 63 - 1
    for V in (70, 3001, 40001):
        x = torch.randn(2, V, generator=torch.Generator().manual_seed(V)).to(d)
        bad = torch.tensor([[lo, 7, hi, lo + 1, -1, V, 2 ** 32 + 7, lo + 7], [hi] * 8], device=d)
        good = torch.tensor([[7], [-1]], device=d)
        assert torch.equal(ops.shape_logits(x, history=bad, frequency=0.5), ops.shape_logits(x, history=good, frequency=0.5))


def test_empty_calls():
    from ps_vae_amd import ops
    d = dev()
    for shape in ((0, 7), (0, 3, 7), (3, 0, 7)):
        x = torch.zeros(shape, device=d, requires_grad=True)
        assert ops.shape_logits(x).shape == shape
        lp = ops.shaped_log_prob(x, torch.zeros(shape[:-1], dtype=torch.int64, device=d))
        assert lp.shape == shape[:-1]
        dx, = torch.autograd.grad(lp.sum(), x)
        assert dx.shape == shape
    tok, lp = ops.shaped_draw(torch.zeros(0, 7, device=d), torch.zeros(0, device=d))
    assert tok.shape == lp.shape == (0,)


def test_refusals():
    from ps_vae_amd import ops
    d = dev()
    x = torch.zeros(4, 9, device=d)
    h = torch.zeros(4, 5, dtype=torch.int64, device=d)
    m = ops.pack_allowed(torch.ones(3, 9, dtype=torch.bool, device=d))
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=d)   # noqa: E731
    for kw in (dict(history=h.int()), dict(history=h[:3]), dict(history=h.t().contiguous().t()), dict(history=h, history_len=i32(3)),
               dict(history=h, history_len=i32(4, 2)), dict(history=h, history_len=i32(4).long()), dict(history_len=i32(4)),
               dict(bias=torch.zeros(8, device=d)), dict(bias=torch.zeros(3, 9, device=d)), dict(bias=torch.zeros(9, device=d).double()),
               dict(bias=torch.zeros(9)), dict(allowed=m), dict(allowed=m.long(), state=i32(4)), dict(allowed=m, state=i32(5)),
               dict(state=i32(4)), dict(allowed=m[:, :0], state=i32(4)), dict(temperature=torch.ones(3, device=d)), dict(temperature=0.0),
               dict(temperature=float('nan')), dict(history=h, repetition=-1.0), dict(history=h, presence=float('inf')),
               dict(temperature=torch.ones(4, 1, device=d))):
        with pytest.raises((RuntimeError, ValueError)):
            ops.shape_logits(x, **kw)
    for bad in (x.double(), x.int(), x[0], x.t(), torch.zeros(4, 0, device=d), x.cpu()):
        with pytest.raises(RuntimeError):
            ops.shape_logits(bad)
    with pytest.raises(RuntimeError):
        ops.shaped_log_prob(x, torch.zeros(4, dtype=torch.int32, device=d))
    with pytest.raises(RuntimeError):
        ops.shaped_log_prob(x, torch.zeros(3, dtype=torch.int64, device=d))
    with pytest.raises(RuntimeError):
        ops.shaped_draw(x, torch.zeros(3, device=d))
    with pytest.raises(RuntimeError):
        ops.shaped_draw(x, torch.zeros(4, device=d).double())
    with pytest.raises(RuntimeError):
        ops.shaped_draw(x[None], torch.zeros(1, device=d))
    # no second derivative: an error, not a constant
    leaf = x.clone().requires_grad_(True)
    for y in (ops.shape_logits(leaf * leaf), ops.shaped_log_prob(leaf * leaf, torch.zeros(4, dtype=torch.int64, device=d))):
        first, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match='differentiated again'):
            first.sum().backward()
    # a history written to after the forward pass is noticed by autograd, not silently recounted
    leaf = x.clone().requires_grad_(True)
    y = ops.shape_logits(leaf, history=h, repetition=1.5)
    h[0, 0] = 3
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_another_stream_and_captured_graph():
    """Two graphs captured from one pool of calls (a draw over a wide row, a log-prob with its gradient), replayed in turn with new inputs and
    eager work between, equal the eager results bit for bit."""
    from ps_vae_amd import ops
    d = dev()
    c = make(5, 1, 9001, 30, 'f32', seed=11, nasty=False)
    kw = on(c, d)
    x, u, tok = c['logits'].to(d), c['uniforms'].to(d), c['tokens'].to(d)

    def both(x):
        t, l = ops.shaped_draw(x, u, **kw)
        leaf = x.detach().requires_grad_(True)
        lp = ops.shaped_log_prob(leaf, tok, **kw)
        dx, = torch.autograd.grad(lp, leaf, torch.ones_like(lp))
        return t, l, lp.detach(), dx
    eager = [v.clone() for v in both(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both(x)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    graphs, outs = [], []
    static = [x.clone(), (x * 0.5).clone()]
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both(s))
        graphs.append(g)
    gen = torch.Generator(device=d).manual_seed(1)
    for _ in range(4):
        for s, g, o in zip(static, graphs, outs):
            s.copy_(torch.randn(s.shape, generator=gen, device=d) * 3)
            want = [v.clone() for v in both(s)]
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(want, o):
                assert torch.equal(a.nan_to_num(), b.nan_to_num())
