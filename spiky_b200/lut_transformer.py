"""LUT transformer built from the LUT layers of :mod:`spiky_b200.lut_layer`.

Same constructor arguments, attribute names and forward contract as the reference's
``spiky.lut.LUTTransformer`` (src/spiky/lut/LUTTransformer.py:69-271): a frozen token embedding, then
``num_layers`` blocks of [LUT attention over the whole context -> dropout -> (BatchNorm1d) -> residual,
LUT feed-forward on every token -> dropout -> (BatchNorm1d) -> residual], then a LUT unembedder to the
vocabulary.  ``forward(tokens[B, S]) -> logits[B, S, V]``.

Beyond the reference: ``norm`` ('rms' or 'layer') puts a norm of each token before every block and before the unembedder,
``norm_after`` one after every block, ``gated`` a learned gate row on every block's output, ``skip_scale`` and ``branch_scale`` scale the two
parts of every residual sum, and ``counter_dropout`` draws the dropout masks from (``dropout_seed``, a buffer that counts training
passes) instead of storing them (``dropout_replica``: whose masks, by default those of the process's rank).  Each block is then joined to
the stream, with the next block's norm, in one kernel (:mod:`spiky_b200.residual`).
"""
import torch
import torch.nn as nn

from .lut_layer import (Conv2DLUTLayer, GradientPolicy, GradientType, LUTLayer, LUTSharedContext,  # noqa: F401
                        SynapseMeta, _normalise_device)
from .residual import ResidualJoin, RowNorm, counter_dropout as _counter_dropout, dropout_state, drawn_seed, replica_site, take_dropout_state


class LUTTransformer(nn.Module):
    # (of models that were pickled before these options)
    norm, counter_dropout, _joined, dropout_replica = None, False, False, None

    def __init__(self, vocab_size, embedding_dim, context_size, positional_dim, num_layers, num_heads, n_detectors,
                 n_anchors_per_detector, n_anchors_per_detector_attention=None, no_ffn=False,
                 concatenation_product=True, sliced_product_mode=False, unified_pe=False, do_normalise_weights=False,
                 weights_gradient_policy=None, device=None, synapse_meta=SynapseMeta(), lut_shared_context=None,
                 seed=None, summation_dtype=torch.float32, _int_rescaler=0.001, _forward_group_size=32,
                 _backward_group_size=32, dropout=0.0, use_batch_norm=False, norm=None, norm_after=False, gated=False, skip_scale=1.0,
                 branch_scale=1.0, counter_dropout=False, dropout_seed=None, dropout_replica=None):
        super().__init__()
        if norm not in (None, "rms", "layer"):
            raise ValueError("norm is None, 'rms' or 'layer'")
        if norm_after and norm is None:
            raise ValueError("norm_after needs norm")
        shaped = norm is not None or gated or skip_scale != 1.0 or branch_scale != 1.0
        if use_batch_norm and shaped:
            raise ValueError("use_batch_norm goes without norm, gated, skip_scale and branch_scale")
        if dropout_seed is not None and not counter_dropout:
            raise ValueError("dropout_seed is the seed of counter_dropout")
        if dropout_replica is not None:
            if not counter_dropout:
                raise ValueError("dropout_replica goes with counter_dropout")
            replica_site(dropout_replica)   # (refuses)
        self.vocab_size = vocab_size
        self.embedding_dim = embedding_dim
        self.context_size = context_size
        self.positional_dim = positional_dim
        self.num_layers = num_layers
        self.num_heads = num_heads
        self.n_detectors = n_detectors
        self.n_anchors_per_detector = n_anchors_per_detector
        self.n_anchors_per_detector_attention = (n_anchors_per_detector_attention
                                                 if n_anchors_per_detector_attention is not None
                                                 else n_anchors_per_detector)
        self.concatenation_product = concatenation_product
        self.sliced_product_mode = sliced_product_mode
        self.weights_gradient_policy = weights_gradient_policy
        self.dropout = dropout
        self.use_batch_norm = use_batch_norm
        self.norm, self.norm_after, self.gated, self.counter_dropout = norm, norm_after, gated, counter_dropout
        self.dropout_replica = dropout_replica   # (None: the rank)
        self._joined = shaped or (counter_dropout and not use_batch_norm)
        self.unified_pe = unified_pe
        self.no_ffn = no_ffn
        self.device = torch.device("cpu") if device is None else _normalise_device(device)
        self.lut_shared_context = (LUTSharedContext().to_device(self.device) if lut_shared_context is None
                                   else lut_shared_context)
        self._debug_last_forward = None

        flat = isinstance(embedding_dim, int)
        n_emb = embedding_dim if flat else embedding_dim[0] * embedding_dim[1]
        self._n_embeddings = n_emb

        # frozen random token embedding in [-1, 1]
        self.token_embedder = nn.Embedding(vocab_size, n_emb, device=self.device)
        self.token_embedder.weight.requires_grad_(False)
        with torch.no_grad():
            if seed is not None:
                gen = torch.Generator(device="cpu").manual_seed(seed)
                table = 2 * torch.rand(self.token_embedder.weight.shape, generator=gen) - 1.0
                self.token_embedder.weight.copy_(table)
            else:
                nn.init.uniform_(self.token_embedder.weight, -1.0, 1.0)

        common = dict(synapse_meta=synapse_meta, do_normalise_weights=do_normalise_weights,
                      weights_gradient_policy=weights_gradient_policy, shared_context=self.lut_shared_context,
                      summation_dtype=summation_dtype, _int_rescaler=_int_rescaler, device=self.device,
                      _forward_group_size=_forward_group_size, _backward_group_size=_backward_group_size)

        def per_token_lut(n_outputs, layer_seed):
            # sequences are processed token by token through a reshape [B, S, E] -> [B * S, 1, E]
            return LUTLayer(n_inputs=n_emb, n_outputs=n_outputs, n_detectors=n_detectors,
                            n_anchors_per_detector=n_anchors_per_detector, sequence_length=1, random_seed=layer_seed,
                            **common)

        def attention_lut(layer_seed):
            seq = dict(sequence_length=context_size, concatenation_product=concatenation_product,
                       sliced_product_mode=sliced_product_mode, positional_dim=positional_dim, unified_pe=unified_pe,
                       n_anchors_per_detector=self.n_anchors_per_detector_attention, random_seed=layer_seed, **common)
            if flat:
                return LUTLayer(n_inputs=embedding_dim, n_outputs=embedding_dim, n_detectors=n_detectors * num_heads,
                                **seq)
            # 2-D embeddings (used by the reference's tests only): one receptive field covering the whole input
            return Conv2DLUTLayer(input_shape=embedding_dim, detectors_shape=(1, n_detectors * num_heads),
                                  output_kernel_shape=embedding_dim, receptive_field_shape=embedding_dim,
                                  receptive_field_stride_shape=embedding_dim, **seq)

        def join():
            return ResidualJoin(n_emb, branch_norm=norm if norm_after else None, next_norm=norm, gated=gated, skip_scale=skip_scale,
                                branch_scale=branch_scale, dropout=dropout if counter_dropout else 0.0, device=self.device)

        self._n_dropouts = num_layers * (1 if no_ffn else 2)
        if counter_dropout:
            if dropout_seed is None:
                dropout_seed = drawn_seed() if seed is None else seed
            self.register_buffer("dropout_state", dropout_state(dropout_seed, self.device))
        if norm is not None:
            self.first_norm = RowNorm(n_emb, norm, device=self.device)

        self.layers = nn.ModuleList()
        for li in range(num_layers):
            block = nn.ModuleDict()
            base = None if seed is None else seed + li * num_heads
            block["attention_lut"] = attention_lut(base)
            block["attention_dropout"] = nn.Dropout(dropout)
            block["attention_bn"] = nn.BatchNorm1d(n_emb, device=self.device) if use_batch_norm else None
            if not no_ffn:
                block["ffn"] = per_token_lut(n_emb, None if seed is None else base + num_heads)
                block["ffn_dropout"] = nn.Dropout(dropout)
                block["ffn_bn"] = nn.BatchNorm1d(n_emb, device=self.device) if use_batch_norm else None
            if self._joined:
                block["attention_join"] = join()
                if not no_ffn:
                    block["ffn_join"] = join()
            self.layers.append(block)
        self.unembedder = per_token_lut(vocab_size, seed)

    # ------------------------------------------------------------------ helpers
    def _lut_layers(self):
        for block in self.layers:
            yield block["attention_lut"]
            if not self.no_ffn:
                yield block["ffn"]
        yield self.unembedder

    def set_external_learning_rate_hook(self, lr_hook):
        for layer in self._lut_layers():
            layer.set_external_learning_rate_hook(lr_hook)

    def _reset_shared_context(self, new_context):
        for layer in self._lut_layers():
            layer._reset_shared_context(new_context)

    def to(self, *args, **kwargs):
        device = kwargs.get("device", None)
        if device is None and args and not isinstance(args[0], torch.dtype):
            device = args[0]
        # strings and ordinals name a device in both the positional and the keyword form
        if isinstance(device, (str, int)) and not isinstance(device, bool):
            try:
                device = torch.device(device)
            except (RuntimeError, ValueError):
                device = None
        super().to(*args, **kwargs)
        if isinstance(device, torch.device):
            dev = _normalise_device(device)
            self.device = dev
            self.lut_shared_context.to_device(dev)
            for layer in self._lut_layers():
                layer.to(device=dev)
        return self

    @staticmethod
    def _residual_branch(z, out, dropout, bn):
        out = dropout(out)
        if bn is not None:
            out = bn(out.reshape(-1, out.shape[-1])).reshape(out.shape)
        return z + out

    def _add(self, z, out, block, part, state, site):
        """The stream with a block's output, and what the next block reads of it."""
        if not self._joined:
            dropout = block[part + "_dropout"]
            if self.counter_dropout:
                def dropout(o, training=dropout.training):
                    return _counter_dropout(o, self.dropout, state, site) if training and self.dropout > 0.0 else o
            z = self._residual_branch(z, out, dropout, block[part + "_bn"])
            return z, z
        if not self.counter_dropout:
            out = block[part + "_dropout"](out)
        return block[part + "_join"](z, out, state, site)

    # ------------------------------------------------------------------ forward
    def _drops(self):
        """Whether a pass draws masks from the counter: where what has a block's dropout - the join, or torch's module without one - is in training
        mode, whatever the model's own mode is, as with torch's dropout."""
        if not self.counter_dropout or self.dropout == 0.0:
            return False
        which = "_join" if self._joined else "_dropout"
        return any(block[part + which].training for block in self.layers for part in (("attention",) if self.no_ffn else ("attention", "ffn")))

    def take_dropout_state(self):
        """The state of one training pass's counter dropouts, for ``forward``; None where nothing is dropped."""
        return take_dropout_state(self.dropout_state, self._n_dropouts) if self._drops() else None

    def forward(self, tokens, dropout_state=None):
        """tokens: int64 [B, context_size] -> logits fp32 [B, context_size, vocab_size].

        ``dropout_state``: what ``take_dropout_state`` returned, for a model that ``torch.utils.checkpoint`` runs again in the backward pass
        (``checkpoint(model, tokens, model.take_dropout_state())``); by default the call takes its own.
        """
        B, S, E = tokens.shape[0], self.context_size, self._n_embeddings
        record = self._debug_last_forward is not None
        if record:
            self._debug_last_forward = [tokens.to(dtype=torch.float32)]
        z = self.token_embedder(tokens)
        if record:
            self._debug_last_forward.append(z.detach().clone())
        flat = isinstance(self.embedding_dim, int)
        if dropout_state is not None and not self.counter_dropout:
            raise ValueError("dropout_state goes with counter_dropout")
        state = None   # of this pass's dropouts, each with a site of its own
        if self._drops():
            state = self.take_dropout_state() if dropout_state is None else dropout_state
        site = replica_site(self.dropout_replica) if state is not None else 0
        y = z if self.norm is None else self.first_norm(z)
        for block in self.layers:
            att_in = y if flat else y.reshape((B, S) + tuple(self.embedding_dim))
            att = block["attention_lut"](att_in.contiguous()).reshape(B, S, E)
            if record:
                self._debug_last_forward.append(att.detach().clone())
            z, y = self._add(z, att, block, "attention", state, site)
            site += 1
            if not self.no_ffn:
                ffn = block["ffn"](y.reshape(B * S, 1, E)).reshape(B, S, E)
                if record:
                    self._debug_last_forward.append(ffn.detach().clone())
                z, y = self._add(z, ffn, block, "ffn", state, site)
                site += 1
        return self.unembedder(y.reshape(B * S, 1, E)).reshape(B, S, self.vocab_size)

    def get_profile_statistics(self) -> str:
        """Kernel timings collected by the opt-in profiler of the CUDA library, one line per kernel family."""
        from . import _native

        lines = []
        for name, rec in _native.profiler_read().items():
            if rec["launches"]:
                avg = rec["ms"] / rec["timed"] if rec["timed"] else 0.0
                lines.append(f"lut::runtime::{name}: {rec['ms']:.4f} ms / {rec['launches']} = {avg:.4f} ms")
        return "\n".join(lines)
