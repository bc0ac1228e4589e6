"""The caller of llsa_l2 in the reference, restated small: a pixel-space DiT with adaLN-zero blocks
(models/rope_dit_transformer_2d.py: block :295-337 and :581-711, model :827-828, :891-897,
:940-1049, attention call site :180-260) and one flow-matching training step
(trainers/dit_trainer.py:243-315, schedulers/flow_training_scheduler.py:540-565,
trainers/ddpm_trainer.py:97-103).  Plain torch modules around this package's operators: the
attention, the qk RMS norms, the RoPE rotation and the Z-order permutation run in the HIP kernels,
everything else (linear layers, layer norms, GELU, AdamW) is torch's; with fused_layers=True the layer
norms, the linear layers and the feed-forward blocks are this package's too (layer_norm, linear,
feed_forward: modulation, bias, activation, gate and residual in the same passes).  With num_experts every
block's feed-forward is a mixture of that many (route_tokens, expert_feed_forward), which the reference does
not have; quantize_for_sampling() keeps the blocks' projections and feed-forward weights in 8-bit integers
(linear_int8).

The reference builds its model from diffusers classes, which are neither part of its checkout nor
installed here; the layer shapes below follow the arguments it passes to them (biases on q/k/v and
on the output projection, `gelu-approximate` MLP of 4x width, layer norms without weights, eps 1e-5
in the block and 1e-6 in the adaLN norms, 256 sinusoidal timestep channels with cos first).  It is
a workload for timing the operator inside a training step, not a weight-compatible model.
"""
from __future__ import annotations

import math
import weakref
from typing import Optional, Sequence, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..kernel.hip.experts import expert_feed_forward, route_tokens
from ..kernel.hip.layer_norm import layer_norm
from ..kernel.hip.linear import feed_forward, linear
from ..kernel.hip.linear_int8 import linear_int8, quantize_rows
from ..kernel.hip.permute import permute_tokens
from ..kernel.hip.rms_norm import my_rms_norm_fn
from ..kernel.hip.rope import my_rope_fn
from ..kernel.torch_op.flash_sparse_attention_res_1 import llsa_l1
from ..kernel.torch_op.flash_sparse_attention_res_2 import llsa_l2, llsa_l3
from ..utils.rope_table import rope_table
from ..utils.zorder import zorder_perm


def timestep_channels(t: torch.Tensor, channels: int = 256, max_period: float = 10000.0) -> torch.Tensor:
    """Sinusoidal embedding of the timesteps as the model's `Timesteps(256, flip_sin_to_cos=True,
    downscale_freq_shift=1)` makes it (:267-268): frequencies max_period^(-i/(half-1)), cosines
    first."""
    half = channels // 2
    freqs = torch.exp(-math.log(max_period) * torch.arange(half, dtype=torch.float32, device=t.device) / (half - 1))
    ang = t.float()[:, None] * freqs[None]
    return torch.cat([ang.cos(), ang.sin()], dim=-1)


def of(layer: nn.Linear, dtype: torch.dtype):
    """(weight, bias) of a layer in the dtype of the activations, as autocast would cast them."""
    return layer.weight.to(dtype), None if layer.bias is None else layer.bias.to(dtype)


class MadeOf:
    """The weight that whole numbers were made of: its memory, and how often that has been written to.  A copy of this, or one out of a file, is of no weight."""

    def __init__(self, weight: Optional[torch.Tensor] = None):
        self.memory = None if weight is None else weakref.ref(weight.untyped_storage())
        self.state = None if weight is None else self.state_of(weight)

    @staticmethod
    def state_of(weight: torch.Tensor):
        return weight.data_ptr(), None if weight.is_inference() else weight._version

    def still(self, weight: torch.Tensor) -> bool:
        return self.memory is not None and self.memory() is weight.untyped_storage() and self.state == self.state_of(weight)

    def __reduce__(self):
        return MadeOf, ()


def in_8_bits(layer: nn.Linear) -> bool:
    return hasattr(layer, "weight_q")


def keep_in_8_bits(layer: nn.Linear, keep: bool = True):
    """The layer's weight as whole numbers with a scale for each channel out, beside the weight itself; project() then takes these.  Made once more they stay
    where they are, so that captured graphs follow."""
    if not keep:
        if in_8_bits(layer):
            del layer.weight_q, layer.weight_scale, layer.weight_made_of
        return None
    with torch.inference_mode(False), torch.no_grad():        # (buffers that may be written to in any mode)
        q, scale = quantize_rows(layer.weight.detach())
        if layer.weight.is_cuda and torch.cuda.is_current_stream_capturing():
            return q, scale                                   # (of that graph, whose replays make them)
        if in_8_bits(layer) and (layer.weight_q.shape, layer.weight_q.device, layer.weight_scale.dtype) == (q.shape, q.device, scale.dtype):
            layer.weight_q.copy_(q)
            layer.weight_scale.copy_(scale)
        else:
            layer.register_buffer("weight_q", q, persistent=False)
            layer.register_buffer("weight_scale", scale, persistent=False)
    layer.weight_made_of = MadeOf(layer.weight)
    return layer.weight_q, layer.weight_scale


def kept_in_8_bits(layer: nn.Linear):
    """The whole numbers and scales of the layer's present weight: made again if it is another, or has been written to, cast or moved since."""
    fresh = layer.weight_made_of.still(layer.weight) and layer.weight_scale.dtype == torch.float32 and layer.weight_q.device == layer.weight.device
    return (layer.weight_q, layer.weight_scale) if fresh else keep_in_8_bits(layer)


def project(layer: nn.Linear, x: torch.Tensor, rows=None, **epilogue) -> torch.Tensor:
    """The layer by this package's operators.  rows: x as quantize_rows gives it, for layers that share it."""
    if in_8_bits(layer):
        bias = None if layer.bias is None else layer.bias.to(x.dtype)
        return linear_int8(x if rows is None else rows, *kept_in_8_bits(layer), bias, dtype=x.dtype, **epilogue)
    return linear(x, *of(layer, x.dtype), **epilogue)


class TimestepEmbedding(nn.Module):
    def __init__(self, dim: int, fused_layers: bool = False):
        super().__init__()
        self.fused_layers = fused_layers
        self.linear_1 = nn.Linear(256, dim)
        self.linear_2 = nn.Linear(dim, dim)

    def forward(self, t: torch.Tensor, dtype: torch.dtype, activated: bool = False) -> torch.Tensor:
        """The embedding, or silu of it (activated), through which all that reads it here does."""
        x = timestep_channels(t).to(dtype)
        if self.fused_layers:
            h = linear(x, *of(self.linear_1, dtype), activation="silu")
            return linear(h, *of(self.linear_2, dtype), activation="silu" if activated else None)
        e = self.linear_2(F.silu(self.linear_1(x)))
        return F.silu(e) if activated else e


class AdaLayerNormZero(nn.Module):
    """:295-337: six modulation vectors from the timestep embedding; returns the modulated
    normalised tokens and the other four vectors."""

    def __init__(self, dim: int, fused_layers: bool = False):
        super().__init__()
        self.fused_layers = fused_layers
        self.emb = TimestepEmbedding(dim, fused_layers)
        self.linear = nn.Linear(dim, 6 * dim)
        self.norm = nn.LayerNorm(dim, elementwise_affine=False, eps=1e-6)

    def forward(self, x, t):
        cond = self.emb(t, x.dtype, activated=True)
        vectors = linear(cond, *of(self.linear, x.dtype)) if self.fused_layers else self.linear(cond)
        shift_msa, scale_msa, gate_msa, shift_mlp, scale_mlp, gate_mlp = vectors.chunk(6, dim=1)
        if self.fused_layers:
            return layer_norm(x, scale=scale_msa, shift=shift_msa, eps=self.norm.eps), gate_msa, shift_mlp, scale_mlp, gate_mlp
        return self.norm(x) * (1 + scale_msa[:, None]) + shift_msa[:, None], gate_msa, shift_mlp, scale_mlp, gate_mlp


class LlsaSelfAttention(nn.Module):
    """The attention module with RopeAttnProcessor (:180-260).  q, k, v stay in the (B, N, H, D)
    memory of their linear layers (the kernels read the transposed views in place), and the output
    comes back in that layout, so the output projection reads it without a copy.

    fused_prologue=True hands the RMS-norm weights and the RoPE table to the operator, which
    normalises and rotates inside its pooling pass; False composes my_rms_norm_fn, my_rope_fn and
    the operator as the reference does.  gate and residual (both optional): what the block does with the
    output, residual + gate * output, in the output projection's pass with fused_layers=True."""

    def __init__(self, dim: int, heads: int, head_dim: int, levels: int = 2, sparse_topk: Tuple[int, int] = (16, 16),
                 block_size: int = 16, qk_norm: bool = True, eps: float = 1e-5, fused_prologue: bool = True, fused_layers: bool = False):
        super().__init__()
        inner = heads * head_dim
        self.fused_layers = fused_layers
        self.heads, self.head_dim, self.levels = heads, head_dim, levels
        self.sparse_topk, self.block_size, self.eps, self.fused_prologue = tuple(sparse_topk), block_size, eps, fused_prologue
        self.to_q, self.to_k, self.to_v = nn.Linear(dim, inner), nn.Linear(dim, inner), nn.Linear(dim, inner)
        self.to_out = nn.Linear(inner, dim)
        if qk_norm:
            self.norm_q_weight = nn.Parameter(torch.ones(head_dim))
            self.norm_k_weight = nn.Parameter(torch.ones(head_dim))
        else:
            self.norm_q_weight = self.norm_k_weight = None

    def forward(self, x: torch.Tensor, freq: torch.Tensor, gate: Optional[torch.Tensor] = None,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        B, N, _ = x.shape
        split = lambda y: y.view(B, N, self.heads, self.head_dim).transpose(1, 2)
        rows = quantize_rows(x) if self.fused_layers and in_8_bits(self.to_q) else None
        q, k, v = (split(project(layer, x, rows) if self.fused_layers else layer(x)) for layer in (self.to_q, self.to_k, self.to_v))
        norm = None
        if self.norm_q_weight is not None:
            norm = (self.norm_q_weight.float(), self.norm_k_weight.float(), self.eps)
        rope = freq
        if not self.fused_prologue:
            if norm is not None:
                q, k = my_rms_norm_fn(q, norm[0], self.eps), my_rms_norm_fn(k, norm[1], self.eps)
            q, k = my_rope_fn(q, freq), my_rope_fn(k, freq)
            norm = rope = None
        tk = self.sparse_topk                                   # coarsest level first, fine blocks last
        if self.levels == 1:
            o = llsa_l1(q, k, v, tk[-1], self.block_size, rope=rope, qk_norm=norm)
        elif self.levels == 2:      # the reference passes (sparse_topk[1], sparse_topk[0]) as (topk1, topk2), :249-250
            o = llsa_l2(q, k, v, tk[-1], tk[-2], self.block_size, rope=rope, qk_norm=norm)
        else:                       # three levels: no counterpart in the reference
            o = llsa_l3(q, k, v, tk[-1], tk[-2], tk[-3], self.block_size, rope=rope, qk_norm=norm)
        o = o.transpose(1, 2).reshape(B, N, self.heads * self.head_dim)
        if self.fused_layers:
            return project(self.to_out, o, gate=gate, residual=residual)
        o = self.to_out(o)
        if gate is not None:
            o = gate.unsqueeze(1) * o
        return o if residual is None else o + residual


class Experts(nn.Module):
    """A feed-forward block for each of num_experts, of which every token takes experts_per_token."""

    def __init__(self, dim: int, hidden: int, num_experts: int, experts_per_token: int):
        super().__init__()
        self.experts_per_token = experts_per_token
        self.router = nn.Linear(dim, num_experts, bias=False)
        one = lambda n, k: nn.Parameter((torch.rand(num_experts, n, k) * 2 - 1) / math.sqrt(k))
        self.w_in, self.w_out = one(hidden, dim), one(dim, hidden)
        self.b_in, self.b_out = nn.Parameter(torch.zeros(num_experts, hidden)), nn.Parameter(torch.zeros(num_experts, dim))

    def forward(self, x, gate, residual):
        routing = route_tokens(linear(x, self.router.weight.to(x.dtype)), self.experts_per_token)
        w = [p.to(x.dtype) for p in (self.w_in, self.b_in, self.w_out, self.b_out)]
        return expert_feed_forward(x, routing, *w, activation="gelu_tanh", gate=gate, residual=residual)


class RopeTransformerBlock(nn.Module):
    """:581-711 with norm_type 'ada_norm_zero' and no cross attention."""

    def __init__(self, dim: int, heads: int, head_dim: int, fused_layers: bool = False, num_experts: int = 0, experts_per_token: int = 2, **attn):
        super().__init__()
        if num_experts and not fused_layers:
            raise ValueError("num_experts needs fused_layers=True")
        self.fused_layers = fused_layers
        self.norm1 = AdaLayerNormZero(dim, fused_layers)
        self.attn1 = LlsaSelfAttention(dim, heads, head_dim, fused_layers=fused_layers, **attn)
        self.norm3 = nn.LayerNorm(dim, eps=1e-5, elementwise_affine=False)
        if num_experts:
            self.experts = Experts(dim, 4 * dim, num_experts, experts_per_token)
        else:
            self.ff_in, self.ff_out = nn.Linear(dim, 4 * dim), nn.Linear(4 * dim, dim)
        self.num_experts = num_experts

    def forward(self, x, t, freq):
        h, gate_msa, shift_mlp, scale_mlp, gate_mlp = self.norm1(x, t)
        x = self.attn1(h, freq, gate_msa, x)
        if self.fused_layers:
            h = layer_norm(x, scale=scale_mlp, shift=shift_mlp, eps=self.norm3.eps)
            if self.num_experts:
                return self.experts(h, gate_mlp, x)
            if in_8_bits(self.ff_in):
                return project(self.ff_out, project(self.ff_in, h, activation="gelu_tanh"), gate=gate_mlp, residual=x)
            return feed_forward(h, *of(self.ff_in, h.dtype), *of(self.ff_out, h.dtype), activation="gelu_tanh", gate=gate_mlp, residual=x)
        h = self.norm3(x) * (1 + scale_mlp[:, None]) + shift_mlp[:, None]
        return gate_mlp.unsqueeze(1) * self.ff_out(F.gelu(self.ff_in(h), approximate="tanh")) + x


class PixelDiT(nn.Module):
    """RopeDiTTransformer2DModel (:735-1058) at patch size 1 with token_permutation.  The defaults
    are configs/models/model_rope_dit_S_128_rms_llsa_l2.json (that file's sparse_topk is 8; the
    benchmark configuration uses 16).  fused_layers: layer norms, linear layers and feed-forward blocks
    by this package's operators, whose activations are bf16 or fp16 (autocast, or a model in that
    dtype); the parameters are the same.  num_experts (with fused_layers): a mixture of that many feed-forward
    blocks in each, of which a token takes experts_per_token."""

    def __init__(self, num_attention_heads: int = 6, attention_head_dim: int = 64, num_layers: int = 12, in_channels: int = 3,
                 out_channels: int = 3, sample_size: int = 128, axes_dims_rope: Sequence[int] = (32, 32), levels: int = 2,
                 sparse_topk=16, qk_norm: bool = True, fused_prologue: bool = True, fused_layers: bool = False, num_experts: int = 0,
                 experts_per_token: int = 2):
        super().__init__()
        self.fused_layers = fused_layers
        dim = num_attention_heads * attention_head_dim
        if isinstance(sparse_topk, int):
            sparse_topk = (sparse_topk,) * max(levels, 2)
        self.sample_size, self.out_channels = sample_size, out_channels
        self.proj_in = nn.Conv2d(in_channels, dim, kernel_size=1)
        self.transformer_blocks = nn.ModuleList(
            RopeTransformerBlock(dim, num_attention_heads, attention_head_dim, levels=levels, sparse_topk=sparse_topk,
                                 qk_norm=qk_norm, fused_prologue=fused_prologue, fused_layers=fused_layers, num_experts=num_experts,
                                 experts_per_token=experts_per_token) for _ in range(num_layers))
        self.norm_out = nn.LayerNorm(dim, elementwise_affine=False, eps=1e-6)
        self.proj_out_1 = nn.Linear(dim, 2 * dim)
        self.proj_out_2 = nn.Linear(dim, out_channels)
        perm, inv = zorder_perm(sample_size)
        self.register_buffer("bwd_perm", perm.to(torch.int32), persistent=False)     # Z-order -> raster
        self.register_buffer("fwd_perm", inv.to(torch.int32), persistent=False)      # raster -> Z-order
        # the table is kept in Z-order and in bf16, as register_rope_emb builds it (:153-173)
        self.register_buffer("freq", rope_table(sample_size, tuple(axes_dims_rope), dtype=torch.bfloat16), persistent=False)

    def quantize_for_sampling(self, on: bool = True) -> "PixelDiT":
        """Keeps the blocks' projections and feed-forward weights (not an experts') as 8-bit integers, which the forward then multiplies with: sample under
        torch.no_grad(), as the model gives no gradients until quantize_for_sampling(False).  A forward makes the integers of a weight again that has been loaded, replaced, written
        to, cast or moved; call this again after writing through `weight.data`, which leaves no trace, and before replaying graphs captured earlier."""
        if not self.fused_layers:
            raise ValueError("quantize_for_sampling needs fused_layers=True")
        for block in self.transformer_blocks:
            a = block.attn1
            for layer in [a.to_q, a.to_k, a.to_v, a.to_out] + ([] if block.num_experts else [block.ff_in, block.ff_out]):
                keep_in_8_bits(layer, on)
        return self

    def forward(self, images: torch.Tensor, timestep: torch.Tensor) -> torch.Tensor:
        B, _, Hh, Ww = images.shape
        if Hh != self.sample_size or Ww != self.sample_size:
            raise ValueError(f"this model is built for {self.sample_size} x {self.sample_size} images")
        x = self.proj_in(images).reshape(B, -1, Hh * Ww).transpose(1, 2)                 # :942-945
        x = permute_tokens(x, self.fwd_perm, self.bwd_perm)                              # :963-965
        for block in self.transformer_blocks:
            x = block(x, timestep, self.freq)
        x = permute_tokens(x, self.bwd_perm, self.fwd_perm)                              # :1028-1030
        cond = self.transformer_blocks[0].norm1.emb(timestep, x.dtype, activated=True)                   # :1033-1034
        if self.fused_layers:
            shift, scale = linear(cond, *of(self.proj_out_1, cond.dtype)).chunk(2, dim=1)
            x = linear(layer_norm(x, scale=scale, shift=shift, eps=self.norm_out.eps), *of(self.proj_out_2, x.dtype))
        else:
            shift, scale = self.proj_out_1(cond).chunk(2, dim=1)
            x = self.proj_out_2(self.norm_out(x) * (1 + scale[:, None]) + shift[:, None])
        return x.reshape(B, Hh, Ww, self.out_channels).permute(0, 3, 1, 2)               # :1039-1049 at patch size 1


class FlowMatchingStep:
    """One optimisation step of the trainer with is_flow_matching and v-prediction
    (dit_trainer.py:243-315, 346-349): noisy = (1 - sigma) x + sigma noise with sigma = t / 1000,
    target = noise - x, mean squared error in fp32, gradient norm clipped to 1, AdamW with the
    trainer's defaults (ddpm_trainer.py:39-43, 97-103), the model under bf16 autocast."""

    def __init__(self, model: nn.Module, lr: float = 1e-4, betas=(0.9, 0.999), weight_decay: float = 1e-2, eps: float = 1e-8,
                 num_train_timesteps: int = 1000, clip: float = 1.0):
        self.model, self.T, self.clip = model, num_train_timesteps, clip
        self.optimizer = torch.optim.AdamW(model.parameters(), lr=lr, betas=betas, weight_decay=weight_decay, eps=eps)

    def loss(self, images, noise, timesteps):
        sigma = (timesteps.float() / self.T)[:, None, None, None]
        noisy = (1.0 - sigma) * images + sigma * noise
        with torch.autocast(device_type=images.device.type, dtype=torch.bfloat16):
            out = self.model(noisy, timesteps)
        return F.mse_loss(out.float(), (noise - images).float())

    def __call__(self, images, noise, timesteps) -> torch.Tensor:
        loss = self.loss(images, noise, timesteps)
        loss.backward()
        if self.clip:
            torch.nn.utils.clip_grad_norm_(self.model.parameters(), self.clip)
        self.optimizer.step()
        self.optimizer.zero_grad(set_to_none=True)
        return loss.detach()
