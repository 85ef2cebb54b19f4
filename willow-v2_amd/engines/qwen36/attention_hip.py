"""The full-attention layers of the engine on the HIP backend, as a mixin beside HipMoE (engines/base.py:328-367 is the
reference's Engine.attention): projections, per-head norms, rotary positions, the paged 8-bit cache and attention over it,
the output gate and the output projection.

    class Qwen35MoEEngineHip(HipAttention, HipMoE, Qwen35MoEEngine): ...

    engine.kv_cache = HBMKVCache(layers=10, pages=4096, kv_heads=2, head_dim=256)
    engine.rotary = Rotary(256, rotary_dim=64, theta=1e7, sections=(11, 11, 10))
    step = engine.kv_cache.step(seqs, counts)                       # once a forward pass
    x = x + engine.hip_attention(engine.rms_norm(x, ...), layer, cache_layer, step, positions)

Weights are read under the names of the reference's engine, <prefix>layers.N.self_attn.{q,k,v,o}_proj.weight (dense tensors or
GGMLWeight) and .{q,k}_norm.weight (zero-centered RMSNorm over a head, engines/base.py:27-31; left out where absent). A q_proj
of twice the heads' width holds each head's query and, behind it, its output gate: out = sigmoid(gate) * attention.
"""
import torch
import torch.nn.functional as F

from gguf.hip import rope


class Rotary:
    """The rotary frequencies of a model: rotary_dim values of each head turn, frequency j by theta^(-2 j / rotary_dim) a
    position (or by inv_freq[j], fp64, where a model rescales them), sections[i] frequencies by axis i of the positions
    (interleaved over the frequencies, as models of text and images have them; one section: plain positions)."""

    def __init__(self, head_dim: int, rotary_dim: int = None, theta: float = 1e7, sections=None, interleaved: bool = True,
                 inv_freq=None, scale: float = 1.0, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim % 2 or not 0 < rotary_dim <= head_dim:
            raise ValueError(f"rotary_dim must be even and at most head_dim {head_dim} (got {rotary_dim})")
        half = rotary_dim // 2
        self.sections = (half,) if sections is None else tuple(int(s) for s in sections)
        if sum(self.sections) != half:
            raise ValueError(f"sections {self.sections} must add up to rotary_dim / 2 = {half}")
        if inv_freq is None:
            inv_freq = theta ** (-torch.arange(half, dtype=torch.float64) / half)
        self.inv_freq = torch.as_tensor(inv_freq, dtype=torch.float64).to(device).contiguous()
        if self.inv_freq.shape != (half,):
            raise ValueError(f"inv_freq must have {half} entries")
        self.interleaved, self.scale = bool(interleaved), float(scale)

    def positions(self, position_ids: torch.Tensor) -> torch.Tensor:
        """int64 [axes, tokens] of position ids that may be [tokens] (every axis the same: text)."""
        p = position_ids.to(device=self.inv_freq.device, dtype=torch.int64)
        return p.expand(len(self.sections), -1).contiguous() if p.dim() == 1 else p.contiguous()

    def __call__(self, q, k, positions):
        return rope(q, k, positions, self.inv_freq, sections=self.sections, interleaved=self.interleaved, scale=self.scale)


def head_norm(x: torch.Tensor, weight, eps: float) -> torch.Tensor:
    """The zero-centered RMSNorm of the last dimension (engines/base.py:27-31) in fp32, rounded to x's dtype; x itself
    without a weight."""
    if weight is None:
        return x
    f = x.float()
    f = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps)
    return (f * (1 + weight.to(device=x.device, dtype=torch.float32))).to(x.dtype)


class HipAttention:
    """Mixin with the attention of one layer on an HBMKVCache (self.kv_cache) and Rotary (self.rotary)."""

    attention_eps = 1e-6

    def hip_attention(self, x: torch.Tensor, layer: int, cache_layer: int, step, positions: torch.Tensor,
                      causal: bool = True) -> torch.Tensor:
        """x [tokens, hidden], the step's rows in its sequences' order -> [tokens, hidden] in x's dtype. layer: the layer's
        number in the weights' names; cache_layer: in the cache (which holds the attention layers alone); positions int64
        [axes, tokens] (Rotary.positions). The step's keys and values are written into the cache, then attended."""
        cache, p = self.kv_cache, f"{self.prefix}layers.{layer}.self_attn"
        dim, kv_heads = cache.pages.head_dim, cache.pages.kv_heads
        flat = x.reshape(-1, x.shape[-1]).to(device=cache.device, dtype=torch.bfloat16)

        def project(name, heads=None):
            y = F.linear(flat, self.weights[f"{p}.{name}.weight"]).to(torch.bfloat16)
            if y.shape[1] % dim or (heads is not None and y.shape[1] != heads * dim):
                raise ValueError(f"{p}.{name}: {y.shape[1]} rows for heads of {dim}"
                                 f"{'' if heads is None else f', {heads} of them'}")
            return y

        wide = project("q_proj")
        heads = self.weights[f"{p}.o_proj.weight"].shape[1] // dim
        if wide.shape[1] == 2 * heads * dim:
            q, gate = wide.view(-1, heads, 2, dim).unbind(2)
        elif wide.shape[1] == heads * dim:
            q, gate = wide.view(-1, heads, dim), None
        else:
            raise ValueError(f"{p}.q_proj: {wide.shape[1]} rows for {heads} heads of {dim}")
        k, v = (project(n, kv_heads).view(-1, kv_heads, dim) for n in ("k_proj", "v_proj"))
        q = head_norm(q, self.weights.get(f"{p}.q_norm.weight"), self.attention_eps)
        k = head_norm(k, self.weights.get(f"{p}.k_norm.weight"), self.attention_eps)
        q, k = self.rotary(q, k, positions)
        cache.append(cache_layer, step, k, v)
        o = cache.attend(cache_layer, step, q, causal=causal)
        if gate is not None:
            o = (o.float() * torch.sigmoid(gate.float())).to(torch.bfloat16)
        y = F.linear(o.view(o.shape[0], -1), self.weights[f"{p}.o_proj.weight"])
        return y.to(device=x.device, dtype=x.dtype).view(*x.shape[:-1], y.shape[-1])
