"""Paged decoder-only transformer — drop-in for serving/paged_model.py.

Same module tree and parameter names as the reference (embedding, layers[i]
{attn_norm, attn, mlp_norm, mlp}, final_norm, lm_head), built in the same
order, so reference checkpoints load and random init under one seed draws
the same weights. `forward_batch` packs the step's metadata once and shares
it across layers instead of rebuilding it per layer.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import fused_ops
from .adapters import step_adapters
from .layers import ModelConfig, RMSNorm, SwiGLU, TokenEmbedding
from .paged_meta import pack_batch_meta
from .paged_mqa import MQA_Paged


class PagedBlock(nn.Module):
    def __init__(self, config, layer_idx, backend="pytorch"):
        super().__init__()
        self.layer_idx = layer_idx
        self.attn_norm = RMSNorm(config.d_model)
        self.attn = MQA_Paged(config, backend=backend)
        self.mlp_norm = RMSNorm(config.d_model)
        self.mlp = SwiGLU(config.d_model, config.hidden_size, config.bias)

    def forward(self, x, pool, block_table, start):
        x = x + self.attn.forward_paged(self.attn_norm(x), pool, self.layer_idx, block_table, start)
        return x + self.mlp(self.mlp_norm(x))

    def forward_meta(self, x, pool, meta):
        x = x + self.attn.forward_meta(self.attn_norm(x), pool, self.layer_idx, meta)
        return x + self.mlp(self.mlp_norm(x))


fused_ops.PLAIN_MODULES.add(PagedBlock)


class PagedTransformer(nn.Module):
    def __init__(self, config, backend="pytorch"):
        super().__init__()
        self.embedding = TokenEmbedding(config.vocab_size, config.d_model)
        self.layers = nn.ModuleList(
            [PagedBlock(config, i, backend) for i in range(config.num_layers)])
        self.final_norm = RMSNorm(config.d_model)
        self.lm_head = nn.Linear(config.d_model, config.vocab_size, bias=False)

    def forward(self, input_ids, pool, block_table, start):
        """Single sequence (reference: paged_model.py:42-47): logits of the
        last token, [1, 1, vocab]."""
        x = self.embedding(input_ids)
        for layer in self.layers:
            x = layer(x, pool, block_table, start)
        x = x[:, -1:, :]
        return self.lm_head(self.final_norm(x))

    @torch.no_grad()
    def forward_batch(self, batch, pool, adapters=None, adapter_ids=None):
        """Ragged batch step (reference: paged_model.py:50-67): logits of each
        sequence's last new token, [num_seqs, vocab]. adapters: an AdapterSet
        (serving.adapters), adapter_ids one index of it a sequence, -1 for none."""
        T = batch.input_ids.numel()
        meta = pack_batch_meta(batch.block_tables, batch.query_start_loc, batch.positions,
                               T, batch.input_ids.device, pool.block_size)
        step = None
        if adapter_ids is not None and any(i != -1 for i in adapter_ids):
            if adapters is None:
                raise ValueError("forward_batch: adapter_ids needs an AdapterSet")
            step = step_adapters(adapters, adapter_ids, batch.query_start_loc,
                                 batch.input_ids.device)
        return self.forward_step(batch.input_ids, pool, meta, step)

    @torch.no_grad()
    def forward_step(self, input_ids, pool, meta, adapters=None):
        """forward_batch with pre-packed metadata (PagedBatchMeta). With lengths
        from the device (build_batch_meta) input_ids has num_tokens rows, those
        behind the last token of any value, and a sequence without a token gets
        logits of zeros.

        On a ROCm device every norm runs in the prologue of the projection
        that consumes it and every residual add in the epilogue of the
        projection that produces it, so a layer is four projection kernels
        and one attention call: norm + qkv GEMM + RoPE, append + attention,
        out GEMM + add, norm + gate/up GEMM + SwiGLU gate, down GEMM + add.
        The arithmetic is that of PagedBlock.forward_meta: each sum is
        rounded to the model dtype before it is normalised or carried on.

        adapters: the rows' low-rank adapters (StepAdapters, on a ROCm device). The
        norms, RoPE and the gate then run beside the projections, which are those of a
        step without adapters: rows without an adapter keep their bits."""
        x = self.embedding(input_ids)
        if not x.is_cuda:
            if adapters is not None:
                raise RuntimeError("adapters require the model on a ROCm GPU device")
            for layer in self.layers:
                x = layer.forward_meta(x, pool, meta)
            last = meta.query_start_loc[1:].long() - 1
            return self.lm_head(self.final_norm(x.index_select(0, last)))
        if not meta.exact and x.shape[0] == 0:
            return x.new_zeros((meta.num_seqs, self.lm_head.out_features))
        x = x.contiguous()
        attr = fused_ops.module_attr
        for i, layer in enumerate(self.layers):
            attn, mlp = attr(layer, "attn"), attr(layer, "mlp")
            if adapters is None:
                attn.forward_meta_residual_(x, attr(layer, "attn_norm"), pool, layer.layer_idx,
                                            meta)
                mlp.forward_residual_(x, attr(layer, "mlp_norm"))
            else:
                weights = adapters.weights.layers[i]
                attn.forward_adapted_residual_(x, attr(layer, "attn_norm"), pool,
                                               layer.layer_idx, meta, weights, adapters.plan)
                mlp.forward_adapted_residual_(x, attr(layer, "mlp_norm"), weights, adapters.plan)
        if not meta.exact:
            return self._logits_of_last(x, meta.query_start_loc)
        if not meta.is_decode:
            x = x.index_select(0, meta.query_start_loc[1:].long() - 1)
        return self.lm_head(self.final_norm(x))

    def _logits_of_last(self, x, qsl):
        """Logits of each sequence's last row of x, zeros where it has none."""
        rows = x.index_select(0, (qsl[1:].long() - 1).clamp_(min=0))
        return self.lm_head(self.final_norm(rows)).masked_fill_(
            (qsl[1:] == qsl[:-1])[:, None], 0)

    @torch.no_grad()
    def forward_tree(self, input_ids, pool, tree, status=None):
        """The nodes of drafted trees in one pass on a ROCm device: input_ids [T]
        their tokens, tree a TreeMeta (serving.tree_decode). Returns the logits of
        every node [T, vocab] and the nodes' K and V rows of all layers, each
        [num_layers, T, Hkv, D] in the model's dtype, for KVPool.write_accepted;
        the pool is read only. `status` as in build_batch_meta: table entries outside
        the pool, which read as zeros, and runs that were skipped."""
        x = self.embedding(input_ids).contiguous()
        if not x.is_cuda:
            raise RuntimeError("forward_tree requires the model on a ROCm GPU device")
        shape = (len(self.layers), x.shape[0], pool.num_kv_heads, pool.head_dim)
        k_rows, v_rows = x.new_empty(shape), x.new_empty(shape)
        if x.shape[0] == 0:  # every sequence finished
            return x.new_empty((0, self.lm_head.out_features)), k_rows, v_rows
        attr = fused_ops.module_attr
        for i, layer in enumerate(self.layers):
            attr(layer, "attn").forward_tree_residual_(x, attr(layer, "attn_norm"), pool,
                                                       layer.layer_idx, tree, k_rows[i],
                                                       v_rows[i], status)
            attr(layer, "mlp").forward_residual_(x, attr(layer, "mlp_norm"))
        return self.lm_head(self.final_norm(x)), k_rows, v_rows


def load_paged_model(ckpt_path, device):
    """Checkpoint {model, model_config, ...} -> (PagedTransformer, ModelConfig)
    (reference: paged_model.py:70-80). Loaded with weights_only=True."""
    ckpt = torch.load(ckpt_path, map_location="cpu", weights_only=True)
    raw = ckpt.get("model_config")
    if raw is None:
        raise ValueError("checkpoint is missing model_config")
    values = dict(raw) if isinstance(raw, dict) else vars(raw)
    cfg = ModelConfig(**{k: v for k, v in values.items() if k in ModelConfig.__dataclass_fields__})
    attn_type = ckpt.get("train_config", {}).get("attn_type", "mqa")
    if attn_type != "mqa":
        raise ValueError(f"paged serving supports MQA checkpoints, got {attn_type!r}")
    model = PagedTransformer(cfg, backend="pytorch")
    sd = {k.replace("_orig_mod.", ""): v for k, v in ckpt["model"].items()}
    model.load_state_dict(sd)
    return model.to(device).eval(), cfg
