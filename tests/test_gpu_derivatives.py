"""The derivatives that the shaped logits and the gradient lists do not have: asking for one is an error, never a silent zero."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def dev():
    if not torch.cuda.is_available():
        pytest.fail('GPU tests need a GPU')
    return torch.device('cuda:0')


def inputs(B=4, V=302):
    g = torch.Generator().manual_seed(B * 1000 + V)
    d = dev()
    return dict(x=torch.randn(B, V, generator=g).to(d), tok=torch.randint(0, V, (B,), generator=g).to(d), u=torch.rand(B, generator=g).to(d),
                h=torch.randint(0, V, (B, 9), generator=g).to(d), bias=torch.randn(V, generator=g).to(d), rows=(0.5 + torch.rand(B, generator=g)).to(d))


def calls(c, **kw):
    from ps_vae_amd import ops
    return {'shape_logits': lambda x: ops.shape_logits(x, **kw), 'shaped_log_prob': lambda x: ops.shaped_log_prob(x, c['tok'], **kw),
            'shaped_draw': lambda x: ops.shaped_draw(x, c['u'], **kw)}


@pytest.mark.parametrize('needs_grad', [False, True])
@pytest.mark.parametrize('V', [302, 5000])
def test_forward_mode_of_the_logits_is_refused(V, needs_grad):
    """A dual tensor came back without its tangent: a derivative that reads as zero."""
    c = inputs(V=V)
    for name, call in calls(c).items():
        want = call(c['x'])
        with fwAD.dual_level():
            x = fwAD.make_dual(c['x'].clone().requires_grad_(needs_grad), torch.ones_like(c['x']))
            with pytest.raises(RuntimeError, match='forward'):
                call(x)
            got = call(fwAD.unpack_dual(x).primal.detach())         # the values alone are fine
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a, b), name


def test_forward_mode_of_the_other_operands_is_refused():
    c = inputs()
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))   # noqa: E731
        for kw in (dict(bias=dual(c['bias'])), dict(temperature=dual(c['rows'])), dict(history=c['h'], repetition=dual(c['rows'])),
                   dict(history=c['h'], presence=dual(c['rows'])), dict(history=c['h'], frequency=dual(c['rows']))):
            for name, call in calls(c, **kw).items():
                with pytest.raises(RuntimeError, match='forward'):
                    call(c['x'])


def test_forward_mode_over_the_backward_pass_is_refused():
    """A tangent that only the incoming gradient has."""
    from ps_vae_amd import ops
    c = inputs()
    for out in (lambda x: ops.shape_logits(x), lambda x: ops.shaped_log_prob(x, c['tok'])):
        x = c['x'].clone().requires_grad_(True)
        y = out(x)
        g = torch.ones_like(y)
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match='forward'):
                torch.autograd.grad(y, x, fwAD.make_dual(g, torch.ones_like(g)), retain_graph=True)
        dx, = torch.autograd.grad(y, x, g)
        assert bool(torch.isfinite(dx).all())


def test_forward_mode_of_gradient_lists_is_refused():
    from ps_vae_amd import optim
    g = torch.ones(8, device=dev())
    with fwAD.dual_level():
        x = fwAD.make_dual(g, torch.ones_like(g))
        with pytest.raises(RuntimeError, match='forward'):
            optim.grad_norm([torch.ones(3, device=dev()), x])
        with pytest.raises(RuntimeError, match='forward'):
            optim.clip_grads([x], 1.0)
        with pytest.raises(RuntimeError, match='forward'):
            optim.clip_grads([g], 1.0, out=[fwAD.make_dual(torch.zeros(8, device=dev()), g)])
    assert bool((g == 1).all())


@pytest.mark.parametrize('V', [302, 5000])
def test_drawn_log_probability_is_not_a_silent_constant(V):
    """The draw has no backward pass: going back through its log-probability says so (it was a constant: a policy gradient of zero)."""
    from ps_vae_amd import ops
    c = inputs(V=V)
    tok, lp = ops.shaped_draw(c['x'], c['u'])
    assert not lp.requires_grad
    x = c['x'].clone().requires_grad_(True)
    tok1, lp1 = ops.shaped_draw(x, c['u'])
    assert torch.equal(tok, tok1) and torch.equal(lp, lp1.detach()) and not tok1.requires_grad
    with pytest.raises(RuntimeError, match='shaped_log_prob'):
        (lp1.sum() + (x * x).sum()).backward()
    with torch.no_grad():
        assert not ops.shaped_draw(x, c['u'])[1].requires_grad
    score = ops.shaped_log_prob(x, tok)                              # what takes its place
    score.sum().backward()
    assert bool(x.grad.any())


def test_norm_of_gradients_with_a_graph_is_not_a_silent_constant():
    """A penalty on the norm contributed nothing."""
    from ps_vae_amd import optim
    d = dev()
    w = torch.arange(1., 6., device=d, requires_grad=True)
    g, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    want = optim.grad_norm([g.detach()])
    assert not want.requires_grad
    norm = optim.grad_norm([torch.ones(0, device=d), g])
    assert torch.equal(norm.detach(), want)
    with pytest.raises(RuntimeError, match='grad_norm'):
        (norm + w.sum()).backward()
    with torch.no_grad():
        assert torch.equal(optim.grad_norm([g]), want) and not optim.grad_norm([g]).requires_grad


def test_clipping_what_autograd_follows_is_refused():
    """Written through its pointer, a leaf would change under autograd, a graph's gradient would keep its old derivative."""
    from ps_vae_amd import optim
    d = dev()
    w = torch.arange(1., 6., device=d, requires_grad=True)
    g, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    before, plain = g.detach().clone(), torch.ones(5, device=d)
    for grads, out in (([g], None), ([w], None), ([plain], [w]), ([g], [plain]), ([plain, g], None)):
        with pytest.raises(RuntimeError, match='no_grad'):
            optim.clip_grads(grads, 1e-3, out=out)
    assert torch.equal(g.detach(), before) and bool((plain == 1).all()) and w.detach().tolist() == [1., 2., 3., 4., 5.]
    # under no_grad, and in clip_grad_norm_ as in torch's, a gradient with a graph is data
    p = torch.nn.Parameter(torch.zeros(5, device=d))
    p.grad = g
    norm = optim.clip_grad_norm_([p], 1e-3)
    assert not norm.requires_grad and abs(float(before.double().norm()) - float(norm)) <= 2 ** -23 * float(norm)
    assert abs(float(g.detach().double().norm()) - 1e-3) < 1e-8
    n = float(g.detach().double().norm())
    with torch.no_grad():
        optim.clip_grads([g], 1e-4)
    # n 1e-4 / (n + 1e-6) with n = 1e-3 is 1e-4 / 1.001, a thousandth below 1e-4; the factor and each product are rounded once (2 * 2^-24 relative)
    want = n * 1e-4 / (n + 1e-6)
    assert abs(float(g.detach().double().norm()) - want) <= 2.01 * 2 ** -24 * want


def test_data_operands_that_want_a_gradient():
    """Refused where a gradient is being recorded, whichever way the operator is called; data like any other where none is."""
    from ps_vae_amd import hip, ops
    c = inputs()
    raw = hip.ops()
    for at, t in ((2, c['rows']), (3, c['rows']), (4, c['rows']), (5, c['rows']), (7, c['bias'])):
        for x in (c['x'], c['x'].clone().requires_grad_(True)):
            # history, its lengths, repetition, presence, frequency, temperature, their numbers, bias, allowed, state
            args = [c['h'], None, None, None, None, None, [1., 0., 0., 1.], None, None, None]
            args[at] = t.clone().requires_grad_(True)
            for call in (lambda: raw.shape_logits(x, *args), lambda: raw.shaped_log_prob(c['tok'], x, *args),
                         lambda: raw.shaped_draw(c['u'], -1, x, *args)):
                with pytest.raises(RuntimeError, match='none of them gets a gradient'):
                    call()
                with torch.no_grad():
                    call()
    for key, t in (('bias', c['bias']), ('temperature', c['rows'])):
        learned, plain = calls(c, **{key: torch.nn.Parameter(t)}), calls(c, **{key: t})
        for name in plain:
            with pytest.raises(ValueError, match='gradient'):
                learned[name](c['x'])
            with torch.no_grad():
                got, want = learned[name](c['x']), plain[name](c['x'])
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert torch.equal(a, b), name
    with torch.no_grad():
        assert torch.equal(ops.shape_logits(c['x'], bias=torch.nn.Parameter(c['bias'])), ops.shape_logits(c['x'], bias=c['bias']))


def test_function_transforms_are_errors():
    """torch.func's derivatives wrap their tensors: neither comes back with a result that lacks one."""
    from ps_vae_amd import optim
    c = inputs()
    ones = torch.ones_like(c['x'])
    single = {name: (lambda x, call=call: call(x)[1] if isinstance(call(x), tuple) else call(x)) for name, call in calls(c).items()}
    single['grad_norm'] = lambda x: optim.grad_norm([x])
    for f in single.values():
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (c['x'],), (ones,))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda x, f=f: f(x).sum())(c['x'])
        assert bool(torch.isfinite(f(c['x'])).all())
