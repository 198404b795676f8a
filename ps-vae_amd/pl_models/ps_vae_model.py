"""PSVAEModel with the reference's interface (src/pl_models/ps_vae_model.py:18-193).

pytorch_lightning is not part of this stack, so the class derives from nn.Module and keeps
the hook methods a Lightning Trainer (or ps_vae_amd.train.fit) calls: training_step,
validation_step, test_step, configure_optimizers, plus global_step / log.

forward() takes either the reference's batch dict (any source) or a CollatedBatch whose
`.compact` layout is present; in the second case no index preparation happens on the way:
the kernels read the CSR / pair lists collation wrote."""
import os
import time

import torch
import torch.nn as nn

from .. import ops
from ..data.bpe_dataset import BPEMolDataset, get_dataloader
from ..modules.encoder import Encoder
from ..modules.predictor import Predictor
from ..modules.vae_piece_decoder import VAEPieceDecoder

PROPS = ['qed', 'sa', 'logp']   # src/evaluation/utils.py:122


class PSVAEModel(nn.Module):
    def __init__(self, config, tokenizer):
        super(PSVAEModel, self).__init__()
        self.config = config
        self.tokenizer = tokenizer
        self.chem_vocab = tokenizer.chem_vocab
        self.predictor = Predictor(**(config['predictor']))
        self.encoder = Encoder(**(config['encoder']))
        self.decoder = VAEPieceDecoder(**(config['vae_piece_decoder']))
        self.pred_loss = nn.MSELoss()
        self.total_time = 0
        self.global_step = 0
        self.logged = {}
        # compact path only; PSVAE_STREAMS=1 keeps everything on the current stream
        self.two_streams = os.environ.get('PSVAE_STREAMS', '2') != '1'
        self.two_streams_min_nodes = 32768   # atoms in the batch from which the fork pays (measured)
        # A step recorded in a HIP graph (graph_step.GraphedTrainStep) cannot take values that change
        # from step to step as Python numbers: the KL weight then comes from this device scalar
        self.beta_tensor = None
        # and the noise of the reparameterisation can be supplied in a fixed tensor [>= batch, latent_dim]
        # (None: drawn with torch.randn_like, as the reference does)
        self.eps_tensor = None

    @property
    def device(self):
        return next(self.parameters()).device

    def hyper_parameters(self):
        """What the reference's save_hyperparameters() keeps in a checkpoint
        (src/pl_models/ps_vae_model.py:21: config and tokenizer), as plain data: the config dict
        with the tokenizer object taken out and the vocabulary rows in id order."""
        config = {k: (dict(v) if isinstance(v, dict) else v) for k, v in self.config.items()}
        config['vae_piece_decoder'] = {k: v for k, v in config['vae_piece_decoder'].items() if k != 'tokenizer'}
        vocab_state = getattr(self.tokenizer, 'vocab_state', None)    # (a stand-in tokenizer may not offer it)
        return {'config': config, 'vocab': vocab_state() if vocab_state is not None else None}

    @classmethod
    def load_from_checkpoint(cls, path, map_location=None):
        """Rebuild tokenizer and model from a checkpoint ps_vae_amd.train wrote and load its weights
        (the reference's PSVAEModel.load_from_checkpoint, used at src/generate.py:97).  The file is
        read with weights_only=True: tensors and plain containers only."""
        from ..utils.tokenizer import Tokenizer
        payload = torch.load(path, map_location='cpu', weights_only=True)
        hp = payload.get('hyper_parameters')
        if hp is None or hp.get('vocab') is None:
            raise KeyError(f'{path} holds no hyper_parameters / vocabulary: build the model yourself and use '
                           'train.load_checkpoint')
        tokenizer = Tokenizer(pieces=hp['vocab'])
        config = {k: (dict(v) if isinstance(v, dict) else v) for k, v in hp['config'].items()}
        config['vae_piece_decoder']['tokenizer'] = tokenizer
        model = cls(config, tokenizer)
        model.load_state_dict(payload['state_dict'])
        model.global_step = int(payload.get('global_step', 0))
        return model.to(map_location) if map_location is not None else model

    def log(self, name, value, **kwargs):
        # detached, like Lightning's self.log: a logged loss must not keep the step's autograd graph
        # (and with it the parameters' gradient accumulators, which remember the stream they were
        # created under) alive into the next step
        self.logged[name] = value.detach() if torch.is_tensor(value) else value

    def forward(self, batch, return_accu=False, eps=None):
        compact = getattr(batch, 'compact', None)
        if eps is None and self.eps_tensor is not None:
            n = compact.num_graphs if compact is not None else batch['x'].shape[0]
            eps = self.eps_tensor[:n]
        if compact is not None:
            # ids + tables instead of the embedded rows [V, D]: both encoders take their first layer from them
            x = self.decoder.embedded_ids(compact.cx, compact.cxp, compact.cxpos)
            # The decoder's message passing over the in-piece bonds depends only on x: it runs on
            # a second stream beside the encoder (and so does its backward), so that one
            # chain's HBM-bound aggregations and tile write-outs fill the gaps of the other's
            # matrix products.
            # (small batches are bound by the host's launch rate, where a second stream only adds joins)
            fork = self.two_streams and compact.num_nodes >= self.two_streams_min_nodes
            node_embedding = self.decoder.embed_nodes_async(x, compact.csr_in) if fork else None
            graph_embedding = self.encoder.embed_graph_of_nodes(x, compact.csr, compact.segments)
            batch_size = compact.num_graphs
            z, res = self.decoder(x=x, x_pieces=None, x_pos=None, edge_index=compact.csr_in, edge_attr=None,
                                  pieces=batch.pieces, conds=graph_embedding, edge_select=compact.pairs,
                                  golden_edge=compact.golden, return_accu=return_accu, eps=eps,
                                  node_embedding=node_embedding)
            props = batch.props
        else:
            x, edge_index, edge_attr = batch['x'], batch['edge_index'], batch['edge_attr']
            x_pieces, x_pos = batch['x_pieces'], batch['x_pos']
            x = self.decoder.embed_atom(x, x_pieces, x_pos)
            batch_size, node_num, node_dim = x.shape
            graph_ids = torch.repeat_interleave(torch.arange(0, batch_size, device=x.device), node_num)
            _, all_x = self.encoder.embed_node(x.view(-1, node_dim), edge_index, edge_attr)
            graph_embedding = self.encoder.embed_graph(all_x, graph_ids, batch['atom_mask'].flatten())
            in_piece_edge_idx = batch['in_piece_edge_idx']
            if not torch.is_tensor(in_piece_edge_idx):
                in_piece_edge_idx = torch.tensor(in_piece_edge_idx, dtype=torch.long, device=x.device)
            z, res = self.decoder(x=x, x_pieces=x_pieces, x_pos=x_pos,
                                  edge_index=edge_index[:, in_piece_edge_idx],
                                  edge_attr=edge_attr[in_piece_edge_idx],
                                  pieces=batch['pieces'], conds=graph_embedding,
                                  edge_select=batch['edge_select'], golden_edge=batch['golden_edge'],
                                  return_accu=return_accu, eps=eps)
            props = batch['props']
        pred_prop = self.predictor(z)
        if pred_prop.is_cuda and type(self.pred_loss) is nn.MSELoss and self.pred_loss.reduction == 'mean':
            pred_loss = ops.mse_selected(pred_prop, props.reshape(batch_size, -1), self._selected_props(props.device))
        else:
            golden = props.reshape(batch_size, -1).index_select(1, self._selected_props(props.device)).float()
            pred_loss = self.pred_loss(pred_prop, golden)
        return pred_loss, res

    def _selected_props(self, device):
        # the column indices as a device tensor made once: indexing with the Python list would
        # copy it to the device on every step (and cannot be captured in a HIP graph)
        idx = getattr(self, '_prop_idx', None)
        if idx is None or idx.device != device:
            idx = self._prop_idx = torch.tensor(self.config['selected_properties'], dtype=torch.int64, device=device)
        return idx

    def cal_beta(self):
        step = self.global_step
        warmup = self.config['kl_warmup']
        if step < warmup:
            beta = 0
        else:
            step_beta, anneal_iter = self.config['step_beta'], self.config['kl_anneal_iter']
            beta = min(self.config['max_beta'], ((step - warmup) // anneal_iter + 1) * step_beta)
        beta += self.config['beta']
        return beta

    def weighted_loss(self, pred_loss, rec_loss, kl_loss):
        alpha = self.config['alpha']
        beta = self.cal_beta() if self.beta_tensor is None else self.beta_tensor
        if all(torch.is_tensor(v) and v.is_cuda and v.dim() == 0 for v in (pred_loss, rec_loss, kl_loss)):
            return ops.loss_mix(rec_loss, pred_loss, kl_loss, alpha, beta)      # one launch each way instead of five
        return alpha * rec_loss + (1 - alpha) * pred_loss + beta * kl_loss

    def training_step(self, batch, batch_idx):
        st = time.time()
        pred_loss, rec_losses = self.forward(batch)
        loss = self.weighted_loss(pred_loss, rec_losses[0], rec_losses[-1])
        self.log('predictor loss', pred_loss)
        self.log('reconstruct loss', rec_losses[0])
        self.log('piece loss', rec_losses[1])
        self.log('edge loss', rec_losses[2])
        self.log('kl loss', rec_losses[3])
        self.log('beta', self.cal_beta())
        self.total_time += time.time() - st
        self.log('total time', self.total_time)
        return loss

    def validation_step(self, batch, batch_idx):
        pred_loss, rec_losses = self.forward(batch, return_accu=True)
        rec_losses, accus = rec_losses
        loss = self.weighted_loss(pred_loss, rec_losses[0], rec_losses[-1])
        self.log('val_loss', loss)
        for i, name in enumerate(['piece accu', 'edge accu']):
            self.log(name, accus[i])
        return loss

    def validation_epoch_end(self, outputs):
        return

    def test_step(self, batch, batch_idx):
        pred_loss, rec_losses = self.forward(batch)
        loss = self.weighted_loss(pred_loss, rec_losses[0], rec_losses[-1])
        self.log('test_loss', loss)
        return loss

    def configure_optimizers(self):
        """src/pl_models/ps_vae_model.py:123-127.  On the GPU the optimiser is optim.FlatAdam:
        the same Adam arithmetic on one flat parameter buffer, with the gradient exchange and
        the Trainer's global-norm clipping folded into its step()."""
        if self.device.type == 'cuda':
            from ..optim import FlatAdam
            optimizer = FlatAdam(self.parameters(), lr=self.config['lr'])
        else:
            optimizer = torch.optim.Adam(self.parameters(), lr=self.config['lr'])
        scheduler = torch.optim.lr_scheduler.LambdaLR(optimizer, lr_lambda=lambda epoch: 1 / (epoch + 1))
        return [optimizer], [scheduler]

    # interface
    def sample_z(self, n, device=None):
        return torch.randn(n, self.decoder.latent_dim, device=self.device if device is None else device)

    def inference_single_z(self, z, max_atom_num, add_edge_th, temperature):
        return self.decoder.inference(z, max_atom_num, add_edge_th, temperature)

    def inference_batch_z(self, zs, max_atom_num, add_edge_th, temperature, constraint_mol=None, shaping=None):
        """The reference loops inference_single_z over the latents (:139-141, "not accelerating,
        just a loop"); here the whole batch goes through sampling, link prediction and greedy
        assembly at once.  Returns one atoms / bonds dict per latent (see
        VAEPieceDecoder.inference_batch); shaping: see VAEPieceDecoder.sample_pieces_batch."""
        if constraint_mol is not None:
            raise NotImplementedError('constrained generation (inference_constraint) is outside the accelerated path')
        zs = torch.stack(list(zs)) if not torch.is_tensor(zs) else zs
        mols, _ = self.decoder.inference_batch(zs, max_atom_num, add_edge_th, temperature, shaping=shaping)
        return mols

    def predict_props(self, z):
        props = self.predictor(z)
        if len(props.shape) == 1:
            padded_props = [torch.tensor(0, device=props.device) for _ in PROPS]
            for i, val in zip(self.config['selected_properties'], props):
                padded_props[i] = val
            return torch.stack(padded_props)
        padded_props = torch.zeros(props.shape[0], len(PROPS), device=props.device)
        padded_props[:, self.config['selected_properties']] = props
        return padded_props

    def get_z(self, batch, eps=None):
        compact = getattr(batch, 'compact', None)
        if compact is not None:
            x = self.decoder.embed_atom(compact.cx, compact.cxp, compact.cxpos)
            _, all_x = self.encoder.embed_node(x, compact.csr)
            graph_embedding = self.encoder.embed_graph(all_x, compact.segments)
        else:
            x = self.decoder.embed_atom(batch['x'], batch['x_pieces'], batch['x_pos'])
            batch_size, node_num, node_dim = x.shape
            graph_ids = torch.repeat_interleave(torch.arange(0, batch_size, device=x.device), node_num)
            _, all_x = self.encoder.embed_node(x.view(-1, node_dim), batch['edge_index'], batch['edge_attr'])
            graph_embedding = self.encoder.embed_graph(all_x, graph_ids, batch['atom_mask'].flatten())
        z_vecs, _ = self.decoder.rsample(graph_embedding, eps)
        return z_vecs

    def get_z_from_return_data(self, step1_res, eps=None):
        """The reference takes an rdkit Mol and runs process_step1 on it
        (src/pl_models/ps_vae_model.py:175-181); without RDKit the entry is the process_step1
        dict itself."""
        step2_res = BPEMolDataset.process_step2(step1_res, self.tokenizer)
        res = BPEMolDataset.process_step3([step2_res], self.tokenizer, device=self.device)
        return self.get_z(res, eps).squeeze()

    get_z_from_mol = get_z_from_return_data

    def return_data_to_mol(self, data):
        return data

    def get_dataloader(self, fname, **kwargs):
        return get_dataloader(fname, self.tokenizer, **kwargs)

    def get_from_batch(self, batch, key):
        if key == 'batch_size':
            return getattr(batch, 'batch_size', None) or batch['x'].shape[0]
        elif key == 'props':
            return batch['props']
