"""The operators between the piece language model's logits and its next token, and the gradient clipping of the step that trains it: what each
is called with, its plain form in elementary torch operations, and its value in 64 bits.

Logits cases: row (b, t) of logits [B, T, V] (or [B, V]) is shaped by the first history_len[b, t] tokens of history[b] (repetition, presence and
frequency penalties), a bias, a temperature and the bit mask of a grammar's state, and is then returned (shape), scored at a token
(log_prob) or drawn from with a uniform number (draw).  Gradient cases: the 2-norm over a list of tensors (norm), and the list scaled to a
largest norm into the slices of flat buffers (clip)."""
import math

import numpy as np
import torch

own = False

# 302 = 300 pieces, '<pad>' and '<s>': the vocabulary of the piece language model; 50 = its largest number of pieces; 32 and 4096 its batch sizes
# and 10000 the molecules of a generation run.  The wider vocabularies are generic.
PIECES, MAX_POS = 302, 50
NAMES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}


def listed():
    return [
        # one step of the sampling loop at the training recipe's batch: latency
        dict(name='shape f32 32x302', op='shape', B=32, T=1, V=PIECES, L=MAX_POS, dtype='f32', penalties=True, bias=0, states=39, temperature=True, grad=False),
        # a batch of requests over a wide vocabulary, every option on, a bias row for each request
        dict(name='shape bf16 256x131072', op='shape', B=256, T=1, V=131072, L=2000, dtype='bf16', penalties=True, bias=2, states=64, temperature=True, grad=False),
        # teacher-forced rows of a fine-tuning batch, both directions
        dict(name='shape f32 512x50x302 grad', op='shape', B=512, T=MAX_POS, V=PIECES, L=MAX_POS, dtype='f32', penalties=True, bias=1, states=39, temperature=True, grad=True),
        # scoring sampled molecules for a policy gradient at batch 32
        dict(name='log_prob f32 32x50x302', op='log_prob', B=32, T=MAX_POS, V=PIECES, L=MAX_POS, dtype='f32', penalties=True, bias=1, states=39, temperature=True, grad=True),
        # the same over a wide vocabulary, half precision
        dict(name='log_prob bf16 8x500x32768', op='log_prob', B=8, T=500, V=32768, L=500, dtype='bf16', penalties=True, bias=1, states=16, temperature=True, grad=True),
        # one request: the smallest serving step over a wide vocabulary
        dict(name='draw bf16 1x32003', op='draw', B=1, T=1, V=32003, L=1500, dtype='bf16', penalties=True, bias=1, states=4, temperature=True, grad=False),
        # the generation run: 10000 molecules at once
        dict(name='draw f32 10000x302', op='draw', B=10000, T=1, V=PIECES, L=MAX_POS, dtype='f32', penalties=True, bias=1, states=39, temperature=True, grad=False),
        # many requests, wide vocabulary of an odd width, long histories
        dict(name='draw f16 250x100003', op='draw', B=250, T=1, V=100003, L=4000, dtype='f16', penalties=True, bias=1, states=64, temperature=True, grad=False),
        # the gradients of the whole model: 8 of each 9 tensors are small
        dict(name='norm f32 model', op='norm', tensors=63, elements=1891727, dtypes='f32', scale=0.05),
        # gradients of a large model in half precision with its norms in f32
        dict(name='norm bf16+f32 400M', op='norm', tensors=420, elements=400000000, dtypes='bf16+f32', scale=0.01),
        dict(name='clip f32 model', op='clip', tensors=63, elements=1891727, dtypes='f32', scale=0.05),
        dict(name='clip bf16+f32 300M', op='clip', tensors=291, elements=300000000, dtypes='bf16+f32', scale=0.01),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['shape', 'shape', 'log_prob', 'log_prob', 'draw', 'draw', 'norm', 'clip'])
    if op in ('norm', 'clip'):
        return dict(op=op, tensors=_log(rng, 1, 420), elements=_log(rng, 1000, 250000000), dtypes=rng.choice(['f32', 'bf16', 'bf16+f32', 'f16+f32']),
                    scale=rng.choice([1e-4, 0.01, 1.0]))
    V = _log(rng, 60, 140000)
    rows = _log(rng, 1, min(20000, 30000000 // V))
    T = 1 if op == 'draw' else min(rows, rng.choice([1, 1, MAX_POS, 200]))
    B = max(1, rows // T)
    return dict(op=op, B=B, T=T, V=V, L=_log(rng, 1, min(4000, 4000000 // B)) if T == 1 else T, dtype=rng.choice(['f32', 'bf16', 'f16']),
                penalties=rng.random() < 0.8, bias=rng.choice([0, 1, 2]), states=rng.choice([0, 1, 39]), temperature=rng.random() < 0.7,
                grad=op == 'log_prob' or (op == 'shape' and rng.random() < 0.4))


# ------------------------------------------------------------------------------------------------ inputs
def _sizes(case):
    """Sizes of the gradient tensors: a few large, many small, as in a model; the last takes what is left."""
    rng = np.random.default_rng(case['tensors'] * 1000003 + case['elements'])
    n = min(case['tensors'], case['elements'])
    w = np.exp(rng.normal(0., 2., n))
    sizes = np.maximum(1, np.floor(w / w.sum() * (case['elements'] - n)).astype(np.int64))
    sizes[-1] += max(0, case['elements'] - int(sizes.sum()))
    return [int(s) for s in sizes]


def _types(case, n):
    kinds = [NAMES[k] for k in case['dtypes'].split('+')]
    return [kinds[0] if len(kinds) == 1 or i % 3 else kinds[1] for i in range(n)]


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.rand(*shape, generator=gen, device=dev)                      # noqa: E731
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev)                    # noqa: E731
    randint = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=gen, device=dev)  # noqa: E731
    if case['op'] in ('norm', 'clip'):
        sizes = _sizes(case)
        types = _types(case, len(sizes))
        # each its own allocation, as autograd leaves them
        grads = [(randn(n) * case['scale']).to(t) for n, t in zip(sizes, types)]
        state = dict(case=case, grads=grads)
        if case['op'] == 'clip':
            # the flat f32 buffer that the all-reduce and the optimiser work on: a slice, 16-byte aligned, for each tensor
            offs = [0]
            for n in sizes:
                offs.append(offs[-1] + (n + 3) // 4 * 4)
            flat = torch.zeros(offs[-1], dtype=torch.float32, device=dev)
            state.update(flat=flat, slices=[flat[o:o + n] for o, n in zip(offs, sizes)],
                         max_norm=0.5 * case['scale'] * math.sqrt(sum(sizes)))
        return state
    B, T, V, L = case['B'], case['T'], case['V'], case['L']
    shape = (B, T, V) if T > 1 else (B, V)
    rows = shape[:-1]
    s = dict(case=case, logits=(randn(*shape) * 3.).to(NAMES[case['dtype']]))
    kw = dict(history=None, history_len=None, repetition=None, presence=None, frequency=None, bias=None, allowed=None, state=None, temperature=None)
    if case['penalties']:
        # tokens of the past are skewed to a few; with several rows a sequence, row t has seen the t tokens before it
        kw['history'] = (V * rand(B, L).pow(3)).long().clamp(max=V - 1)
        kw['history_len'] = torch.arange(T, device=dev, dtype=torch.int32).clamp(max=L).repeat(B, 1) if T > 1 else randint(0, L + 1, B).int()
        kw['repetition'], kw['presence'], kw['frequency'] = 1. + 0.5 * rand(B), rand(B), 0.3 * rand(B)
    if case['bias']:
        kw['bias'] = randn(V) if case['bias'] == 1 else randn(B, V)
    if case['states']:
        # states of a grammar: each allows its own share of the vocabulary, the last none; some rows are not bound (-1)
        S = case['states']
        share = torch.linspace(1., 0.02, S, device=dev)
        bits = rand(S, (V + 31) // 32, 32) < share[:, None, None]
        if S > 1:
            bits[-1] = False
        weights = torch.tensor([1 << i if i < 31 else -(1 << 31) for i in range(32)], device=dev)
        kw['allowed'] = (bits.long() * weights).sum(-1).int()
        kw['state'] = randint(-1, S, *rows).int()
    if case['temperature']:
        kw['temperature'] = 0.6 + 0.8 * rand(B)
    s['kw'] = kw
    if case['op'] == 'log_prob':
        s['tokens'] = randint(0, V, *rows)
        s['g'] = randn(*rows)
    if case['op'] == 'draw':
        s['uniforms'] = rand(B)
    if case['op'] == 'shape' and case['grad']:
        s['g'] = randn(*shape).to(s['logits'].dtype)
    if case['grad']:
        s['logits'].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _counts(history, history_len, B, T, V):
    """How often each id occurs in the part of its history that a row has seen: [B * T, V] int32."""
    L = history.shape[1]
    lens = history_len.reshape(B, T, 1).long()
    live = (torch.arange(L, device=history.device) < lens).reshape(B * T, L)
    ids = history[:, None, :].expand(B, T, L).reshape(B * T, L)
    return torch.zeros(B * T, V, dtype=torch.int32, device=history.device).scatter_add_(1, ids, live.int())


def _permitted(allowed, state, R, V):
    at = torch.arange(V, device=allowed.device)
    words = allowed[state.reshape(R).long().clamp(min=0)][:, at >> 5]
    return ((words >> (at & 31)) & 1).bool() | (state.reshape(R, 1) < 0)


def _shaped(s, x):
    """The shaped values of x [B * T, V], in x's type."""
    case, kw = s['case'], s['kw']
    B, T, V = case['B'], case['T'], case['V']
    per_row = lambda p: p.to(x.dtype).repeat_interleave(T)[:, None]  # noqa: E731
    if kw['history'] is not None:
        n = _counts(kw['history'], kw['history_len'], B, T, V)
        rep = per_row(kw['repetition'])
        x = torch.where(n > 0, torch.where(x > 0, x / rep, x * rep), x)
        x = x - per_row(kw['frequency']) * n - per_row(kw['presence']) * (n > 0)
    if kw['bias'] is not None:
        x = x + (kw['bias'] if kw['bias'].dim() == 1 else kw['bias'].repeat_interleave(T, 0))
    if kw['temperature'] is not None:
        x = x / per_row(kw['temperature'])
    if kw['allowed'] is not None:
        x = torch.where(_permitted(kw['allowed'], kw['state'], B * T, V), x, -math.inf)
    return x


def _plain(s):
    case, logits = s['case'], s['logits']
    B, T, V = case['B'], case['T'], case['V']
    if case['op'] == 'shape':
        y = _shaped(s, logits.reshape(B * T, V).float()).to(logits.dtype).reshape(logits.shape)
        return (y.detach(), *torch.autograd.grad(y, logits, s['g'])) if case['grad'] else y
    if case['op'] == 'draw':
        # 64 bits: whether a running sum exceeds u times the total decides which token comes out
        y = _shaped(s, logits.double())
        m = y.max(-1, keepdim=True).values
        some = m[:, 0] > -math.inf
        p = torch.where(some[:, None], (y - m).exp(), 0.)
        cdf = p.cumsum(-1)
        total = cdf[:, -1:]
        below = (cdf <= s['uniforms'][:, None].double() * total).sum(-1)
        last = (torch.arange(V, device=p.device) * (p > 0)).max(-1).values
        pick = torch.minimum(below, last)
        lp = (y.gather(1, pick[:, None]) - m - total.log())[:, 0]
        return torch.where(some, pick, -1), torch.where(some, lp, -math.inf).float()
    y = _shaped(s, logits.reshape(B * T, V).float())
    some = (y > -math.inf).any(-1, keepdim=True)
    y = torch.where(some, y, 0.)
    m = y.detach().max(-1, keepdim=True).values
    lse = m + (y - m).exp().sum(-1, keepdim=True).log()
    lp = torch.where(some, y.gather(1, s['tokens'].reshape(-1, 1)) - lse, -math.inf).reshape(s['tokens'].shape)
    return (lp.detach(), *torch.autograd.grad(lp, logits, s['g']))


def _plain_clip(s):
    # 64 bits: sums of up to half a thousand million squares
    norm = torch.stack([g.double().square().sum() for g in s['grads']]).sum().sqrt()
    if s['case']['op'] == 'norm':
        return norm.float()
    coef = (s['max_norm'] / (norm + 1e-6)).clamp(max=1.).float()
    for g, out in zip(s['grads'], s['slices']):
        out.copy_(g.float() * coef)
    return norm.float(), s['flat']


def run(state):
    case = state['case']
    if not own:
        return _plain_clip(state) if case['op'] in ('norm', 'clip') else _plain(state)
    import ps_vae_amd  # noqa: F401
    from ps_vae_amd import ops, optim
    if case['op'] == 'norm':
        return optim.grad_norm(state['grads'])
    if case['op'] == 'clip':
        return optim.clip_grads(state['grads'], state['max_norm'], out=state['slices']), state['flat']
    if case['op'] == 'draw':
        return ops.shaped_draw(state['logits'], state['uniforms'], **state['kw'])
    if case['op'] == 'log_prob':
        lp = ops.shaped_log_prob(state['logits'], state['tokens'], **state['kw'])
        return (lp.detach(), *torch.autograd.grad(lp, state['logits'], state['g']))
    y = ops.shape_logits(state['logits'], **state['kw'])
    return (y.detach(), *torch.autograd.grad(y, state['logits'], state['g'])) if case['grad'] else y


def work(case):
    if case['op'] in ('norm', 'clip'):
        sizes = _sizes(case)
        read = sum(n * t.itemsize for n, t in zip(sizes, _types(case, len(sizes))))
        n = sum(sizes)
        return dict(bytes=read + (4 * n if case['op'] == 'clip' else 4), flops=(3 if case['op'] == 'clip' else 2) * n)
    B, T, V = case['B'], case['T'], case['V']
    e, cells = SIZE[case['dtype']], B * T * V
    side = 8 * B * case['L'] + 16 * B * T if case['penalties'] else 0
    side += {0: 0, 1: 4 * V, 2: 4 * B * V}[case['bias']]
    side += case['states'] * ((V + 31) // 32) * 4 + 4 * B * T if case['states'] else 0
    if case['op'] == 'shape':
        # logits in, values out; backward: gradient in, gradient out
        return dict(bytes=cells * e * (4 if case['grad'] else 2) + side, flops=cells * (6 if case['grad'] else 4))
    if case['op'] == 'draw':
        return dict(bytes=cells * e + side + 16 * B, flops=cells * 12)
    return dict(bytes=cells * e * 2 + side + 16 * B * T, flops=cells * 14)  # logits in, their gradient out


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_rows(s):
    """(shaped values, their slope against the logits) as [B * T, V] in 64 bits, a row's counts from a histogram over (row, id)."""
    case, kw = s['case'], s['kw']
    B, T, V = case['B'], case['T'], case['V']
    R = B * T
    l = s['logits'].detach().double().reshape(R, V)
    slope = torch.ones_like(l)
    seq = torch.arange(R, device=l.device) // T
    if kw['history'] is not None:
        lens = kw['history_len'].reshape(R).long()
        row = torch.repeat_interleave(torch.arange(R, device=l.device), lens)
        first = lens.cumsum(0) - lens
        ids = kw['history'][seq[row], torch.arange(row.numel(), device=l.device) - first[row]]
        n = torch.bincount(row * V + ids, minlength=R * V).reshape(R, V).double()
        rep = kw['repetition'].double()[seq][:, None].expand(R, V)
        slope = torch.where(n == 0, slope, torch.where(l > 0, rep.reciprocal(), rep))
        l = l * slope - n * kw['frequency'].double()[seq][:, None] - n.clamp(max=1.) * kw['presence'].double()[seq][:, None]
    if kw['bias'] is not None:
        l = l + (kw['bias'].double()[None] if kw['bias'].dim() == 1 else kw['bias'].double()[seq])
    if kw['temperature'] is not None:
        inv = kw['temperature'].double().reciprocal()[seq][:, None]
        l, slope = l * inv, slope * inv
    if kw['allowed'] is not None:
        words = kw['allowed'].cpu().numpy().view(np.uint8)
        bits = torch.from_numpy(np.unpackbits(words, axis=1, bitorder='little')[:, :V]).to(l.device).bool()
        bits = torch.cat([bits, torch.ones_like(bits[:1])])  # index -1: not bound
        ok = bits[kw['state'].reshape(R).long()]
        l, slope = l.masked_fill(~ok, -math.inf), slope.masked_fill(~ok, 0.)
    return l, slope


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] in ('norm', 'clip'):
        squares = torch.zeros((), dtype=torch.float64, device='cuda')
        for g in s['grads']:
            d = g.double()
            squares += torch.dot(d, d)
        norm = squares.sqrt()
        if case['op'] == 'norm':
            return norm
        coef = min(1., s['max_norm'] / (float(norm) + 1e-6))
        flat = torch.zeros(s['flat'].numel(), dtype=torch.float64, device='cuda')
        at = 0
        for g in s['grads']:
            flat[at:at + g.numel()] = g.double() * coef
            at += (g.numel() + 3) // 4 * 4
        return norm, flat
    y, slope = _exact_rows(s)
    shape = s['logits'].shape
    if case['op'] == 'shape':
        return (y.reshape(shape), (slope * s['g'].double().reshape(y.shape)).reshape(shape)) if case['grad'] else y.reshape(shape)
    lse = torch.logsumexp(y, -1)
    none = lse == -math.inf
    if case['op'] == 'draw':
        p = torch.exp(y - lse.masked_fill(none, 0.)[:, None])
        cdf = torch.cumsum(p, -1)
        pick = torch.searchsorted(cdf, s['uniforms'].double()[:, None] * cdf[:, -1:], right=True)[:, 0]
        positive = p > 0
        last = case['V'] - 1 - positive.flip(-1).to(torch.int8).argmax(-1)
        pick = torch.where(pick < last, pick, last)
        lp = y.gather(-1, pick[:, None])[:, 0] - lse
        return pick.masked_fill(none, -1), lp.masked_fill(none, -math.inf)
    tok = s['tokens'].reshape(-1, 1)
    lp = (y.gather(-1, tok)[:, 0] - lse).masked_fill(none, -math.inf)
    d = -torch.exp(y - lse.masked_fill(none, 0.)[:, None])
    d.scatter_add_(-1, tok, torch.ones_like(tok, dtype=d.dtype))
    return lp.reshape(s['tokens'].shape), (d * slope * s['g'].double().reshape(-1, 1)).masked_fill(none[:, None], 0.).reshape(shape)
