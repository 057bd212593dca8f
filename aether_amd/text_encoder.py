"""MI355X-native T5 encoder for the pipeline's `text_encoder` slot.

The reference fills the slot with transformers' `T5EncoderModel` (/root/reference/scripts/demo.py:206-232) and calls it for the prompt's embedding
(/root/reference/aether/pipelines/aetherv1_pipeline_cogvideox.py:290-297: the empty prompt, once; any prompt through `encode_prompt`).  Here every block is

    h, y = rms_norm(h + delta);  delta = relbias_attn(y Wqkvᵀ) Woᵀ
    h, y = rms_norm(h + delta);  delta = gated_ff(y; Wg, Wu) Wdᵀ

on the HIP kernels of libaether_hip.so: the residual stream h stays in fp32, everything between is bf16, one bias table serves all blocks.  Gradients
(prompt tuning through `inputs_embeds`, fine-tuning of any parameter) go through `aether_amd.functional`; forward-mode derivatives are refused.  There is no
PyTorch fallback.
"""
from __future__ import annotations

import json
import os
import warnings
from types import SimpleNamespace
from typing import Dict, Optional

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _lib, functional, ops

_CONFIG_DEFAULTS = dict(vocab_size=32128, d_model=4096, d_kv=64, num_heads=64, d_ff=10240, num_layers=24, relative_attention_num_buckets=32,
                        relative_attention_max_distance=128, layer_norm_epsilon=1e-6, feed_forward_proj="gated-gelu")
_ACT_OF = {"gated-gelu": "gelu_tanh", "gated-silu": "silu"}


class _Block(nn.Module):
    def __init__(self, c, device):
        super().__init__()
        inner = c.num_heads * c.d_kv

        def weight(*shape, dtype=torch.bfloat16):
            return nn.Parameter(torch.empty(*shape, dtype=dtype, device=device))

        self.norm1 = weight(c.d_model, dtype=torch.float32)
        self.qkv = weight(3 * inner, c.d_model)
        self.out = weight(c.d_model, inner)
        self.norm2 = weight(c.d_model, dtype=torch.float32)
        self.gate = weight(c.d_ff, c.d_model)
        self.up = weight(c.d_ff, c.d_model)
        self.down = weight(c.d_model, c.d_ff)


class AetherTextEncoder(nn.Module):
    """`AetherTextEncoder(config)(input_ids, attention_mask)[0]` -> bfloat16 [B, S, d_model], the call `encode_prompt` makes."""

    def __init__(self, config: Optional[Dict] = None, device="cuda"):
        super().__init__()
        given = dict(config or {})
        act = given.get("feed_forward_proj", "gated-gelu")
        if act not in _ACT_OF:
            raise ValueError(f"aether_amd: feed_forward_proj must be one of {list(_ACT_OF)}, got {act!r}")
        c = self.config = SimpleNamespace(**{**_CONFIG_DEFAULTS, **{k: v for k, v in given.items() if k in _CONFIG_DEFAULTS}})
        if c.d_kv != 64:
            raise ValueError("aether_amd: d_kv must be 64")
        if c.d_model % 64 or c.d_ff % 64 or c.d_model > 16384:
            raise ValueError("aether_amd: d_model (up to 16384) and d_ff must be multiples of 64")
        ops.relbias_borders(c.relative_attention_num_buckets, c.relative_attention_max_distance)
        _lib.load()
        self._act = _ACT_OF[c.feed_forward_proj]
        self.embedding = nn.Parameter(torch.empty(c.vocab_size, c.d_model, dtype=torch.bfloat16, device=device))
        self.bias_table = nn.Parameter(torch.empty(c.relative_attention_num_buckets, c.num_heads, dtype=torch.bfloat16, device=device))
        self.blocks = nn.ModuleList(_Block(c, device) for _ in range(c.num_layers))
        self.final_norm = nn.Parameter(torch.empty(c.d_model, dtype=torch.float32, device=device))
        self._e4m3 = None

    # ------------------------------------------------------------------------------------------
    @classmethod
    def from_pretrained(cls, path, subfolder: Optional[str] = "text_encoder", torch_dtype=torch.bfloat16, device="cuda", **_):
        """Loads a transformers-format folder: config.json + (sharded) model*.safetensors (the folder of demo.py:206-232)."""
        from safetensors.torch import load_file

        if torch_dtype not in (None, torch.bfloat16):
            raise ValueError(f"aether_amd: the text encoder runs in bfloat16, got {torch_dtype}")
        root = os.path.join(path, subfolder) if subfolder else path
        with open(os.path.join(root, "config.json")) as f:
            model = cls(json.load(f), device=device)
        index = os.path.join(root, "model.safetensors.index.json")
        if os.path.exists(index):
            with open(index) as f:
                files = sorted(set(json.load(f)["weight_map"].values()))
        else:
            files = ["model.safetensors"]
        sd = {}
        for fn in files:
            sd.update(load_file(os.path.join(root, fn)))
        return model.load_t5_state_dict(sd).requires_grad_(False)

    @torch.no_grad()
    def load_t5_state_dict(self, sd: Dict[str, torch.Tensor]):
        """Packs a state dict with T5EncoderModel's keys into this module's parameters."""
        self._drop_e4m3()                                       # (first: a dict that is refused halfway has changed some weights)

        def put(param, *keys):
            rows = 0
            for key in keys:
                t = sd[key]
                param[rows:rows + t.shape[0]].copy_(t)
                rows += t.shape[0]
            if rows != param.shape[0]:
                raise ValueError(f"aether_amd: {keys} have {rows} rows, {param.shape[0]} are wanted")

        put(self.embedding, "shared.weight" if "shared.weight" in sd else "encoder.embed_tokens.weight")
        put(self.bias_table, "encoder.block.0.layer.0.SelfAttention.relative_attention_bias.weight")
        for i, b in enumerate(self.blocks):
            att, ff = f"encoder.block.{i}.layer.0.", f"encoder.block.{i}.layer.1."
            put(b.norm1, att + "layer_norm.weight")
            put(b.qkv, *(att + f"SelfAttention.{n}.weight" for n in "qkv"))
            put(b.out, att + "SelfAttention.o.weight")
            put(b.norm2, ff + "layer_norm.weight")
            put(b.gate, ff + "DenseReluDense.wi_0.weight")
            put(b.up, ff + "DenseReluDense.wi_1.weight")
            put(b.down, ff + "DenseReluDense.wo.weight")
        put(self.final_norm, "encoder.final_layer_norm.weight")
        return self

    @torch.no_grad()
    def init_random_weights(self, seed: int = 0):
        """Seeded random weights of the trained model's scales (no checkpoint: smoke runs, benchmarks, tests)."""
        self._drop_e4m3()
        g = torch.Generator(device=self.embedding.device).manual_seed(seed)
        c = self.config
        inner = c.num_heads * c.d_kv

        def normal(p, std):
            p.copy_(torch.randn(p.shape, generator=g, device=p.device) * std)

        normal(self.embedding, 1.0)
        normal(self.bias_table, 1.0)
        for b in self.blocks:
            b.norm1.fill_(1.0)
            b.norm2.fill_(1.0)
            normal(b.qkv, c.d_model ** -0.5)
            b.qkv[:inner] *= c.d_kv ** -0.5
            normal(b.out, inner ** -0.5)
            normal(b.gate, c.d_model ** -0.5)
            normal(b.up, c.d_model ** -0.5)
            normal(b.down, c.d_ff ** -0.5)
        self.final_norm.fill_(1.0)
        return self

    # ------------------------------------------------------------------------------------------
    @torch.no_grad()
    def quantize_feed_forward(self):
        """Serve the feed-forward's two input projections (half of a block's weights) in e4m3: half their bytes, twice the matrix rate, for an error of
        e4m3's rounding (2^-4) on each factor.  The 16-bit weights stay as they are; call it again after changing them.  Moving the module
        (`to`, also to where it is) or loading weights ends this form, with a warning.  No gradients in it."""
        if self.config.d_model % 128:
            raise ValueError("aether_amd: d_model must be a multiple of 128 for 8-bit operands")
        self._e4m3 = [(*ops.quantize_rows_e4m3(b.gate.detach()), *ops.quantize_rows_e4m3(b.up.detach())) for b in self.blocks]
        return self

    # the 8-bit weights are laid out for where and what the weights were

    def _drop_e4m3(self):
        if self._e4m3 is not None:
            warnings.warn("the text encoder's weights were moved or loaded: its 8-bit feed-forward is gone, the 16-bit one serves; call quantize_feed_forward() again", stacklevel=3)
        self._e4m3 = None

    def _apply(self, fn, *args, **kwargs):
        self._drop_e4m3()
        return super()._apply(fn, *args, **kwargs)

    def load_state_dict(self, *args, **kwargs):
        """torch's own: this module's parameter names (checkpoints of T5EncoderModel go through `load_t5_state_dict`)."""
        return super().load_state_dict(*args, **kwargs)

    def _load_from_state_dict(self, *args, **kwargs):        # (a module around this one comes in here)
        self._drop_e4m3()
        return super()._load_from_state_dict(*args, **kwargs)

    # ------------------------------------------------------------------------------------------
    def _embed(self, input_ids, inputs_embeds):
        if (input_ids is None) == (inputs_embeds is None):
            raise ValueError("give either input_ids or inputs_embeds")
        c = self.config
        if inputs_embeds is not None:
            if inputs_embeds.dim() != 3 or inputs_embeds.shape[2] != c.d_model:
                raise ValueError(f"inputs_embeds must be [B, S, {c.d_model}], got {list(inputs_embeds.shape)}")
            return inputs_embeds.float()
        if input_ids.dim() != 2 or input_ids.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"input_ids must be int64 or int32 [B, S], got {input_ids.dtype} {list(input_ids.shape)}")
        if input_ids.numel() and not (input_ids.is_cuda and torch.cuda.is_current_stream_capturing()):
            lo, hi = torch.aminmax(input_ids)
            if int(lo) < 0 or int(hi) >= c.vocab_size:
                raise ValueError(f"input_ids must lie in [0, {c.vocab_size})")
        return nn.functional.embedding(input_ids.to(self.embedding.device), self.embedding).float()

    def forward(self, input_ids=None, attention_mask=None, inputs_embeds=None):
        """-> (last hidden state, bfloat16 [B, S, d_model],).  attention_mask: [B, S], nonzero where a token counts as a key; None: all of them do."""
        if not self.embedding.is_cuda:
            raise RuntimeError("aether_amd needs the text encoder on the device (no CPU fallback)")
        with torch.cuda.device(self.embedding.device):
            return self._forward(self._embed(input_ids, inputs_embeds), attention_mask)

    def _forward(self, h, attention_mask):
        c = self.config
        B, S, D = h.shape
        if attention_mask is not None:
            if tuple(attention_mask.shape) != (B, S):
                raise ValueError(f"attention_mask must be [{B}, {S}], got {list(attention_mask.shape)}")
            attention_mask = attention_mask.to(h.device) != 0
        if h.numel() == 0:
            return (h.to(torch.bfloat16),)
        if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (h, *self.parameters())):
            raise ValueError("the text encoder has no forward-mode derivatives (the kernels would drop the tangent)")
        grad = torch.is_grad_enabled() and (h.requires_grad or any(p.requires_grad for p in self.parameters()))
        if grad and self._e4m3 is not None:
            raise ValueError("the 8-bit feed-forward has no gradients: run under torch.no_grad(), or without quantize_feed_forward()")
        F = functional if grad else ops
        linear = functional.linear if grad else ops.gemm_bf16
        eps, heads = c.layer_norm_epsilon, c.num_heads
        h, delta = h.reshape(B * S, D), None
        for i, b in enumerate(self.blocks):
            y, h = F.rms_norm(h, b.norm1, eps, delta=delta)
            q, k, v = linear(y, b.qkv).view(B, S, 3, heads, 64).unbind(2)
            o = F.relbias_attn(q, k, v, self.bias_table, c.relative_attention_max_distance, key_mask=attention_mask)
            delta = linear(o.view(B * S, heads * 64), b.out)
            if self._e4m3 is None:
                y, h = F.rms_norm(h, b.norm2, eps, delta=delta)
                g = F.gated_ff(y, b.gate, b.up, self._act)
            else:
                y, scale, h = ops.rms_norm_e4m3(h, b.norm2, eps, delta=delta)
                g = ops.gated_ff_e4m3(y, scale, *self._e4m3[i], self._act)
            delta = linear(g, b.down)
        y, _ = F.rms_norm(h, self.final_norm, eps, delta=delta)
        return (y.view(B, S, D),)
