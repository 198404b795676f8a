"""optim.grad_norm / clip_grads / clip_grad_norm_ on the GPU against the float64 oracle.

Tolerances.  The squares and sums are 64-bit (relative error < n 2^-53), so the norm is off by its rounding to float32: u = 2^-24 relative.
A scaled value: the factor is rounded to float32 (u), the product too (u), then to the output's type (half a step)."""
import math

import numpy as np
import pytest
import torch

from oracle import shaping_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def dev():
    if not torch.cuda.is_available():
        pytest.fail('GPU tests need a GPU')
    return torch.device('cuda:0')


def half_step(dtype, y):
    f = torch.finfo(dtype)
    return np.maximum(f.eps / 2 * np.abs(y), f.tiny * f.eps / 2)


def check(grads, max_norm, out=None):
    from ps_vae_amd import optim
    host = [g.double().cpu().numpy() for g in grads]
    norm, scaled = shaping_ref.clip(host, max_norm)
    got = float(optim.grad_norm(grads))
    assert got == norm or abs(got - norm) <= 1.01 * U * norm, (got, norm)
    ret = optim.clip_grads(grads, max_norm, out=out)
    assert ret.dtype == F32 and ret.dim() == 0 and float(ret) == got
    for g, o, w in zip(host, out or grads, scaled):
        have = o.detach().double().cpu().numpy().reshape(w.shape)
        assert (np.abs(have - w) <= 2.01 * U * np.abs(w) + half_step(o.dtype, w)).all()
    return got


SIZES = {'one': [1], 'small': [1, 2, 3, 4, 5, 7, 8, 9, 0, 63, 64, 65], 'chunks': [4095, 4096, 4097, 8192, 12289], 'model': [300 * 300, 300, 302 * 200, 302, 1] * 6,
         'many': [17 * i % 301 for i in range(300)], 'exact': [5] * 140, 'over': [5] * 141, 'exact norm': [5] * 200, 'over norm': [5] * 201, 'three': [3] * 401, 'large': [3000001, 5, 2500000]}


@pytest.mark.parametrize('mode', ['in place', 'flat f32', 'flat bf16'])
@pytest.mark.parametrize('types', [(F32,), (BF16,), (F16,), (BF16, F32, F16)])
@pytest.mark.parametrize('sizes', list(SIZES))
def test_sizes_and_types(sizes, types, mode):
    d = dev()
    gen = torch.Generator(device=d).manual_seed(len(sizes))
    grads = [torch.randn(n, generator=gen, device=d).to(types[i % len(types)]) for i, n in enumerate(SIZES[sizes])]
    out = None
    if mode != 'in place':
        t = F32 if mode == 'flat f32' else BF16
        flat = torch.full((sum(SIZES[sizes]) + 1,), 7.0, dtype=t, device=d)
        at, out = 1, []                          # slices at odd starts, end to end
        for n in SIZES[sizes]:
            out.append(flat[at:at + n])
            at += n
    before = [g.clone() for g in grads]
    check(grads, 0.37 * math.sqrt(max(1, sum(SIZES[sizes]))), out)
    if out is not None:
        assert all(torch.equal(a, b) for a, b in zip(before, grads)) and float(flat[0]) == 7.0


def test_no_clipping_leaves_the_bits():
    from ps_vae_amd import optim
    d = dev()
    for t in (F32, BF16, F16):
        g = [torch.randn(n, device=d).to(t) for n in (5, 5000)]
        before = [x.clone() for x in g]
        optim.clip_grads(g, 1e6)
        assert all(torch.equal(a, b) for a, b in zip(before, g))
        out = [torch.zeros_like(x) for x in g]
        optim.clip_grads(g, float('inf'), out=out)
        assert all(torch.equal(a, b) for a, b in zip(before, out))


def test_range():
    """Values whose squares leave float32 on either side."""
    d = dev()
    for scale in (1e30, 1e19, 1e-30, 1e-38):
        check([torch.full((1000,), scale, device=d), torch.full((77,), -scale, device=d)], scale)
    check([torch.zeros(10, device=d)], 1.0)


def test_thousands_of_tensors():
    """More partial sums than the scaling's workgroups add up by themselves."""
    from ps_vae_amd import optim
    d = dev()
    flat = torch.randn(9000 * 5, generator=torch.Generator().manual_seed(0)).to(d)
    norm = float(flat.double().pow(2).sum().sqrt())
    want = flat.double() * (0.5 * norm / (norm + 1e-6))
    assert abs(float(optim.clip_grads(list(flat.split(5)), 0.5 * norm)) - norm) <= 2 * U * norm
    assert bool(((flat.double() - want).abs() <= 2 * U * want.abs()).all())        # the factor's rounding and the product's
    assert abs(float(optim.grad_norm(list(flat.split(5)))) - 0.5 * norm) <= 4 * U * norm


def test_more_than_32_bits_of_elements():
    from ps_vae_amd import optim
    d = dev()
    n = 2 ** 31 + 2 ** 20 + 3
    g = torch.zeros(n, dtype=torch.bfloat16, device=d)
    g[0], g[2 ** 31 + 5], g[-1] = 3., 4., 12.
    assert float(optim.grad_norm([g])) == 13.0
    assert float(optim.clip_grads([g], 1.3)) == 13.0
    want = torch.tensor([0.3, 0.4, 1.2]).bfloat16().tolist()
    assert [float(g[0]), float(g[2 ** 31 + 5]), float(g[-1])] == want and int(torch.count_nonzero(g)) == 3


def test_not_finite():
    from ps_vae_amd import optim
    d = dev()
    g = [torch.ones(5, device=d), torch.ones(3, device=d).bfloat16()]
    g[1][1] = float('nan')
    assert math.isnan(float(optim.clip_grads(g, 1.0))) and all(torch.isnan(x).all() for x in g)
    g = [torch.ones(5, device=d), torch.ones(3, device=d)]
    g[0][2] = float('inf')
    want = [x.clone() for x in g]
    ps = [torch.nn.Parameter(torch.zeros_like(x)) for x in want]
    for p, w in zip(ps, want):
        p.grad = w
    ref = torch.nn.utils.clip_grad_norm_(ps, 1.0, foreach=False)
    assert float(optim.clip_grads(g, 1.0)) == float(ref) == float('inf')
    for a, p in zip(g, ps):
        assert torch.equal(a.nan_to_num(nan=9.), p.grad.nan_to_num(nan=9.))
    z = [torch.ones(4, device=d)]
    optim.clip_grads(z, 0.0)
    assert not z[0].any()


def test_same_bits_every_time_and_layouts():
    from ps_vae_amd import optim
    d = dev()
    g = [torch.randn(100000, device=d), torch.randn(33, 41, device=d).t(), torch.randn(2, 3, 4, 5, device=d).to(memory_format=torch.channels_last)]
    norms = {float(optim.grad_norm(g)) for _ in range(5)}
    assert len(norms) == 1
    host = [x.clone() for x in g]
    want = check(g, 1.0)
    assert all(x.stride() == h.stride() for x, h in zip(g, host)) and want in norms


def test_clip_grad_norm_follows_torch():
    from ps_vae_amd import optim
    d = dev()
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(70, 200), torch.nn.ReLU(), torch.nn.Linear(200, 31)).to(d)
    x = torch.randn(64, 70, device=d)
    for max_norm in (0.05, 1e4):
        net.zero_grad()
        (net(x) ** 2).mean().backward()
        own = [p.grad.clone() for p in net.parameters()]
        n1 = torch.nn.utils.clip_grad_norm_(net.parameters(), max_norm)
        theirs = [p.grad.clone() for p in net.parameters()]
        for p, g in zip(net.parameters(), own):
            p.grad = g
        net[2].bias.grad = None if max_norm > 1 else net[2].bias.grad
        n2 = optim.clip_grad_norm_(net.parameters(), max_norm)
        if max_norm < 1:
            assert abs(float(n1) - float(n2)) <= 1e-5 * float(n1)
            for p, t in zip(net.parameters(), theirs):
                assert torch.allclose(p.grad, t, rtol=1e-5, atol=0)
    assert float(optim.clip_grad_norm_(net[0].weight, 1.0)) > 0
    net.zero_grad()
    assert float(optim.clip_grad_norm_(net.parameters(), 1.0)) == 0.0


def test_refusals():
    from ps_vae_amd import optim
    d = dev()
    g = torch.ones(8, device=d)
    for bad in ([g.double()], [g.int()], [g.expand(3, 8)], [g[::2]], [g, g.cpu()], []):
        with pytest.raises(RuntimeError):
            optim.grad_norm(bad)
        with pytest.raises(RuntimeError):
            optim.clip_grads(bad, 1.0)
    for grads, out in (([g], [g[:4]]), ([g], []), ([g, g], None), ([g], [g.bfloat16().view(torch.int16)]), ([g[:6]], [g[2:]]),
                       ([torch.randn(3, 5, device=d).t()], [torch.zeros(5, 3, device=d)])):
        with pytest.raises(RuntimeError):
            optim.clip_grads(grads, 1.0, out=out)
    with pytest.raises(RuntimeError):
        optim.clip_grads([g], -1.0)
    assert bool((g == 1).all())


def test_in_place_clipping_is_seen_by_autograd():
    from ps_vae_amd import optim
    d = dev()
    a = torch.randn(5, device=d)
    w = torch.randn(5, device=d, requires_grad=True)
    y = (w * a).sum()
    optim.clip_grads([a], 1e-3)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


def test_captured_graphs_and_streams():
    from ps_vae_amd import optim
    d = dev()
    gen = torch.Generator(device=d).manual_seed(3)
    lists = [[torch.randn(n, generator=gen, device=d).to(t) for n, t in ((5000, F32), (77, BF16), (130001, F32))] for _ in range(2)]
    outs = [[torch.zeros(g.numel(), device=d) for g in gs] for gs in lists]
    graphs, norms = [], []
    for gs, os in zip(lists, outs):
        optim.clip_grads(gs, 3.0, out=os)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(optim.clip_grads(gs, 3.0, out=os))
        graphs.append(graph)
    for _ in range(4):
        for gs, os, graph, norm in zip(lists, outs, graphs, norms):
            for g in gs:
                g.copy_(torch.randn(g.shape, generator=gen, device=d))
            want = [torch.zeros_like(o) for o in os]
            n = optim.clip_grads(gs, 3.0, out=want)
            graph.replay()
            torch.cuda.synchronize()
            assert float(norm) == float(n) and all(torch.equal(a, b) for a, b in zip(os, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n = optim.grad_norm(lists[0])
    torch.cuda.current_stream().wait_stream(side)
    assert float(n) == float(optim.grad_norm(lists[0]))
