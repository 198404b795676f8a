"""The piece sampling loop under penalties, a bias and the atom budget, followed draw by draw with the float64 oracle; and the draws it returns scored
by piece_log_prob: exactly the tokens that were drawn, for every reason that a molecule can stop for."""
import numpy as np
import pytest
import torch

from oracle import shaping_ref
from test_gpu_policy_step import U, dev, make_model

pytestmark = pytest.mark.gpu


def short(model, max_pos):
    """The model with room for max_pos pieces."""
    old = model.decoder.pos_embedding
    model.decoder.pos_embedding = torch.nn.Embedding(max_pos, old.embedding_dim).to(old.weight.device)
    return model.decoder


class Steps:
    """What every step of a loop saw and did: the logits before they were shaped, the state before, the picks."""
    def __init__(self, monkeypatch):
        from ps_vae_amd import hip, ops
        self.logits, self.active, self.atoms, self.picks = [], [], [], []
        shape, draw = ops.shape_logits, hip.piece_draw

        def shape_logits(logits, **kw):
            self.logits.append(logits.detach().clone())
            return shape(logits, **kw)

        def piece_draw(logits, temperature, uniforms_col, pad, end, first_step, counts, budget, max_pos, active, atoms, length, out_col, cur):
            self.active.append(active.clone()), self.atoms.append(atoms.clone())
            draw(logits, temperature, uniforms_col, pad, end, first_step, counts, budget, max_pos, active, atoms, length, out_col, cur)
            self.picks.append(out_col.clone())
        monkeypatch.setattr(ops, 'shape_logits', shape_logits)
        monkeypatch.setattr(hip, 'piece_draw', piece_draw)


def setup(B, seed, max_pos):
    model, tok = make_model()
    dec = short(model, max_pos)
    z = torch.randn(B, dec.latent_dim, generator=torch.Generator().manual_seed(seed)).to(dev())
    u = torch.rand(B, max_pos, generator=torch.Generator().manual_seed(seed + 1)).to(dev())
    return dec, tok, z, u


OPTIONS = {'repetition': dict(repetition=1.7), 'presence': dict(presence=0.9), 'frequency': dict(frequency=0.6), 'bias': dict(bias=True),
           'all': dict(repetition=1.4, presence=0.3, frequency=0.2, bias=True, fit_atoms=True)}


@pytest.mark.parametrize('which', list(OPTIONS))
def test_every_draw_is_the_one_that_the_distribution_asks_for(which, monkeypatch):
    """With S the largest intermediate of a value over the temperature, a shaped value is off by D = 8 u S and the loop's division by the temperature by u
    of the value (in D's 8); a probability by 2 D relative, its exponential and product by 100 u at most, the running sum's at most 16 additions (5 chunks of
    64, 6 levels, the carry) by 16 u, the threshold by u: a pick whose u lies farther than 2 D + 120 u from every boundary is the oracle's."""
    budget, temperature, B, max_pos = 24, 0.8, 60, 12
    dec, tok, z, u = setup(B, 21, max_pos)
    shaping = dict(OPTIONS[which])
    bias = np.zeros(tok.num_piece_type())
    if shaping.pop('bias', False):
        shaping['bias'] = torch.linspace(-0.5, 0.5, tok.num_piece_type(), device=dev())
        bias = shaping['bias'].double().cpu().numpy()
    steps = Steps(monkeypatch)
    dec.sample_pieces_batch(z, budget, temperature, uniforms=u, shaping=shaping)
    cnt, pad, end = np.asarray(tok.piece_atom_counts()), tok.pad_idx(), tok.end_idx()
    f32 = lambda v: float(np.float32(v))   # noqa: E731
    past = [[] for _ in range(B)]
    checked = turned = total = 0
    for t, picks in enumerate(steps.picks):
        rows, live, picks = steps.logits[t].double().cpu().numpy(), steps.active[t].tolist(), picks.tolist()
        for b in range(B):
            if not live[b]:
                assert picks[b] == pad
                continue
            allowed = np.ones(len(cnt), dtype=bool)
            if shaping.get('fit_atoms'):
                allowed = cnt + cnt[past[b]].sum() <= budget if past[b] else cnt <= budget
            allowed[end] = t > 0
            allowed[pad] = False
            args = (f32(shaping.get('repetition', 1.)), f32(shaping.get('presence', 0.)), f32(shaping.get('frequency', 0.)), bias, allowed, f32(temperature))
            y, _, scale = shaping_ref.shaped_row(rows[b], past[b], *args)
            want, _, gap = shaping_ref.draw_row(y, float(u[b, t]))
            total += 1
            if gap > 2 * 8 * U * scale.max() + 120 * U:
                assert picks[b] == want, (t, b)
                checked += 1
                free, _, _ = shaping_ref.shaped_row(rows[b], [], 1., 0., 0., None, allowed, f32(temperature))
                turned += shaping_ref.draw_row(free, float(u[b, t]))[0] != want
            past[b].append(picks[b])
    # most draws are far enough from a boundary, and some would have been others without the shaping
    assert checked > 0.9 * total and turned >= 3 and max(len(p) for p in past) > 4


def scored(dec, tok, z, draws, counts, temperature, shaping, budget, monkeypatch, atoms=None):
    """piece_log_prob of returned draws, each value compared with the oracle on the logits that the model gave; returns the log-probabilities."""
    from ps_vae_amd import ops
    seen = {}
    real = ops.shaped_log_prob
    monkeypatch.setattr(ops, 'shaped_log_prob', lambda logits, tokens, **kw: (seen.update(logits=logits, tokens=tokens, kw=kw), real(logits, tokens, **kw))[1])
    pieces = torch.cat([torch.full_like(draws[:, :1], tok.end_idx()), draws], 1)
    with torch.no_grad():
        lp = dec.piece_log_prob(z, pieces, temperature, shaping, max_atom_num=budget, piece_atom_counts=atoms)
    monkeypatch.setattr(ops, 'shaped_log_prob', real)
    cnt = np.asarray(tok.piece_atom_counts() if atoms is None else atoms)
    f32 = lambda v: float(np.float32(v))   # noqa: E731
    rows, got = seen['logits'].double().cpu().numpy(), lp.double().cpu().numpy()
    assert lp.shape == draws.shape
    for b in range(draws.shape[0]):
        seq = draws[b].tolist()
        for t in range(draws.shape[1]):
            if t >= int(counts[b]):
                assert seq[t] == tok.pad_idx() and got[b, t] == 0.0
                continue
            past = seq[:t]
            allowed = np.ones(len(cnt), dtype=bool)
            if (shaping or {}).get('fit_atoms'):
                allowed = cnt + (cnt[past].sum() if past else 0) <= budget
            allowed[tok.end_idx()] = t > 0
            allowed[tok.pad_idx()] = False
            if not allowed.any():                      # the loop has no choice but the end token
                assert seq[t] == tok.end_idx() and got[b, t] == 0.0
                continue
            assert allowed[seq[t]], (b, t)
            s = shaping or {}
            y, slope, scale = shaping_ref.shaped_row(rows[b, t], past, f32(s.get('repetition', 1.)), f32(s.get('presence', 0.)),
                                                     f32(s.get('frequency', 0.)), None, allowed, f32(temperature))
            want, _, _ = shaping_ref.log_prob_row(y, slope, seq[t])
            D = 8 * U * scale.max()
            assert abs(got[b, t] - want) <= 2 * D + 90 * U + 4 * U * (np.abs(y[np.isfinite(y)]).max() + np.log(302)), (b, t)
    return lp


@pytest.mark.parametrize('fit', [False, True])
def test_pieces_without_atoms(fit, monkeypatch):
    """Atom counts of zero (a caller that counts something else, or nothing): the end token is out of the question at the first draw only, in the loop
    and in the score alike."""
    max_pos, B = 12, 80
    dec, tok, z, u = setup(B, 41, max_pos)
    with torch.no_grad():
        dec.to_vocab.bias[tok.end_idx()] += 4.          # so that some molecules end early
    bias = torch.zeros(tok.num_piece_type(), device=dev())
    for cnt in ([0] * tok.num_piece_type(), [c if i % 2 else 0 for i, c in enumerate(tok.piece_atom_counts())]):
        free, n0 = dec.sample_pieces_batch(z, 500, 1.0, uniforms=u, piece_atom_counts=cnt)
        ids, n1 = dec.sample_pieces_batch(z, 500, 1.0, uniforms=u, piece_atom_counts=cnt, shaping=dict(bias=bias, fit_atoms=fit))
        assert torch.equal(free, ids) and torch.equal(n0, n1)           # everything fits: the same molecules
        pieces = torch.full((B, max_pos + 2), tok.pad_idx(), dtype=torch.int64, device=dev())
        pieces[:, 0] = tok.end_idx()
        pieces[:, 1:max_pos + 1] = ids
        pieces.scatter_(1, n1[:, None] + 1, tok.end_idx())
        pieces = pieces[n1 > 0]
        assert pieces.shape[0] > 10
        scored(dec, tok, z[n1 > 0], pieces[:, 1:], n1[n1 > 0] + 1, 1.0, dict(fit_atoms=fit), 500, monkeypatch, atoms=cnt)


@pytest.mark.parametrize('max_pos,budget,shaping', [(3, 200, None), (12, 9, None), (12, 9, dict(presence=0.4)), (4, 30, dict(fit_atoms=True, repetition=1.3)),
                                                    (12, 20, dict(fit_atoms=True)), (5, 0, dict(fit_atoms=True))])
def test_the_draws_are_what_is_scored(max_pos, budget, shaping, monkeypatch):
    B, temperature = 80, 0.9
    dec, tok, z, u = setup(B, 31, max_pos)
    ids, lengths = dec.sample_pieces_batch(z, budget, temperature, uniforms=u, shaping=shaping)
    steps = Steps(monkeypatch)
    again, n, draws, counts = dec.sample_pieces_batch(z, budget, temperature, uniforms=u, shaping=shaping, return_draws=True)
    monkeypatch.undo()
    assert torch.equal(ids, again) and torch.equal(lengths, n)
    assert draws.shape == (B, max_pos) and draws.dtype == torch.int64 and counts.dtype == torch.int64 and torch.equal((counts - 1).clamp(min=0), lengths)
    taken = torch.stack(steps.picks, 1)
    assert torch.equal(draws[:, :taken.shape[1]], taken)
    # every reason to stop that these sizes allow is there, and the last draw is the one that was made
    cnt = np.asarray(tok.piece_atom_counts())
    reasons = set()
    for b in range(B):
        seq = draws[b, :int(counts[b])].tolist()
        assert draws[b, int(counts[b]):].eq(tok.pad_idx()).all() and seq[:-1] == ids[b, :int(lengths[b])].tolist()
        reasons.add('end' if seq[-1] == tok.end_idx() else 'atoms' if cnt[seq].sum() > budget else 'positions')
    if budget == 200:
        assert 'positions' in reasons
    if budget == 9:
        assert 'atoms' in reasons
    if shaping and 'fit_atoms' in shaping:
        assert 'atoms' not in reasons
    if budget == 30:
        assert 'positions' in reasons                # a piece that fits is dropped at the last position all the same
    lp = scored(dec, tok, z, draws, counts, temperature, shaping, budget, monkeypatch)
    assert bool(torch.isfinite(lp).all())


def test_options_that_would_be_overridden_are_refused():
    from ps_vae_amd import ops
    dec, tok, z, u = setup(4, 51, 6)
    masks = ops.pack_allowed(torch.ones(1, tok.num_piece_type(), dtype=torch.bool, device=dev()))
    past = torch.zeros(4, 3, dtype=torch.int64, device=dev())
    for shaping in (dict(fit_atoms=True, allowed=masks), dict(presence=0.5, history=past),
                    dict(presence=0.5, history_len=torch.zeros(4, dtype=torch.int32, device=dev()))):
        with pytest.raises(ValueError):
            dec.sample_pieces_batch(z, 20, 1.0, uniforms=u, shaping=shaping)
    ids, _ = dec.sample_pieces_batch(z, 20, 1.0, uniforms=u, shaping=dict(allowed=masks))     # alone it says what it does
    assert torch.equal(ids, dec.sample_pieces_batch(z, 20, 1.0, uniforms=u)[0])
    with pytest.raises(ValueError, match='max_atom_num'):
        dec.piece_log_prob(z, past, shaping=dict(fit_atoms=True))
