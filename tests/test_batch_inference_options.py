"""The model's batch entry point hands its sampling options on (no GPU: the decoder's part is replaced)."""
import torch

import ps_vae_amd  # noqa: F401


def test_shaping_reaches_the_decoder(monkeypatch):
    from ps_vae_amd.pl_models import PSVAEModel
    from ps_vae_amd.utils.nn_utils import build_config, default_args
    from ps_vae_amd.utils.tokenizer import Tokenizer
    tok = Tokenizer()
    model = PSVAEModel(build_config(default_args(), tok), tok)
    seen = []
    monkeypatch.setattr(model.decoder, 'inference_batch', lambda *a, **kw: (seen.append((a, kw)), (['mol'], {}))[1])
    z = torch.zeros(1, model.decoder.latent_dim)
    assert model.inference_batch_z(z, 20, 0.5, 1.0) == ['mol']
    assert model.inference_batch_z([z[0]], 20, 0.5, 1.0, shaping=dict(fit_atoms=True)) == ['mol']
    assert [kw.get('shaping') for _, kw in seen] == [None, dict(fit_atoms=True)]
    assert all(a[1:] == (20, 0.5, 1.0) and torch.equal(a[0], z) for a, _ in seen)
