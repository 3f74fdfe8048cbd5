"""Model-side callers: `Attention_rel`-shaped multi-head attention on the fused
op, and the transformer block around it (`Block_rel`-shaped, on the fused layer
norm and gated feed-forward block).

graphnet reaches the reference operator through `Block_rel.forward_flash`
(reference README.md:105-116): the module projects q, k and v with
`proj_q`, `proj_k`, `proj_v` (and optional `q_bias`, `v_bias`), splits the
heads, calls `flash_spacetime_attention`, merges the heads and applies its
output projection `proj` (the parameter names `attention_rel_oracle_inputs`
reads, reference.py:198-223). The reference's op then copies the split views
to contiguous `[B, H, L, D]` (forward.py:274) and the merge copies the output
back to `[B, L, H*D]`.

Here self-attention projects q, k and v with one GEMM (`proj_q`, `proj_k`,
`proj_v` stacked into one `[3*H*D, dim]` weight) whose `[B, L, 3*H*D]`
output, viewed as `[B, L, 3, H, D]`, is what `flash_spacetime_attention_qkv`
reads in place; its gradient comes back as one tensor of that layout, which
the same linear's backward consumes. The output is `[B, L, H, D]`, so
merging the heads is free. Nothing is transposed, split, stacked or copied
around the fused op in either direction. Cross-attention (a separate `kv`)
uses three linears whose split heads are token-major views, also read in
place.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor, nn
from torch.nn import functional as F

from .reference import merge_heads, split_heads


class SpacetimeAttention(nn.Module):
    """Multi-head self-attention with the spacetime pair bias.

    Parameters follow graphnet's `Attention_rel`: `proj_q`, `proj_k`,
    `proj_v` (no bias), `q_bias` / `v_bias` when `qkv_bias`, `proj` (output),
    `num_heads`. `rel_proj` is the pair-embedding projection `R = E W^T + b`
    of the operator (`weight [D, C]`, `bias [D]`, nn.Linear layout).
    `forward(x, feats, seqlens | key_padding_mask)` takes `x [B, L, dim]`,
    detector features `feats [B, L, F >= 4]` and the event lengths, and
    returns `[B, L, dim]`; with `cu_seqlens` it takes packed events, `x
    [T, dim]` and `feats [T, F]`, and returns `[T, dim]`. Packed tokens past
    `cu_seqlens[-1]` belong to no event: they attend to nothing and add
    nothing to the gradients (where the loss leaves them out, and their x is
    finite).
    """

    def __init__(self, dim: int, num_heads: int = 8, channels: int = 16, qkv_bias: bool = False,
                 head_dim: Optional[int] = None, use_attn_bias: bool = True,
                 use_activation_bias: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        fk = {"device": device, "dtype": dtype}
        self.num_heads = num_heads
        self.head_dim = head_dim if head_dim is not None else dim // num_heads
        inner = self.head_dim * num_heads
        self.proj_q = nn.Linear(dim, inner, bias=False, **fk)
        self.proj_k = nn.Linear(dim, inner, bias=False, **fk)
        self.proj_v = nn.Linear(dim, inner, bias=False, **fk)
        if qkv_bias:
            self.q_bias = nn.Parameter(torch.zeros(inner, **fk))
            self.v_bias = nn.Parameter(torch.zeros(inner, **fk))
        else:
            self.q_bias = None
            self.v_bias = None
        self.rel_proj = nn.Linear(channels, self.head_dim, **fk)
        self.proj = nn.Linear(inner, dim, **fk)
        self.use_attn_bias = use_attn_bias
        self.use_activation_bias = use_activation_bias

    def qkv_weight(self) -> Tuple[Tensor, Optional[Tensor]]:
        """The stacked `[3*H*D, dim]` projection weight and its bias (k has none)."""
        w = torch.cat((self.proj_q.weight, self.proj_k.weight, self.proj_v.weight))
        if self.q_bias is None:
            return w, None
        return w, torch.cat((self.q_bias, torch.zeros_like(self.q_bias), self.v_bias))

    def project_qkv(self, x: Tensor, kv: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
        """q, k, v `[B, H, L, D]` with the values of `attention_rel_oracle_inputs`.

        Self-attention: heads-first views of the one fused projection
        (`[B, L, 3, H, D]`); with a separate `kv`: token-major views of three
        linears.
        """
        b, length, _ = x.shape
        if kv is None:
            w, bias = self.qkv_weight()
            qkv = F.linear(x, w, bias).view(b, length, 3, self.num_heads, self.head_dim)
            return tuple(qkv[:, :, i].transpose(1, 2) for i in range(3))
        if kv.shape != x.shape:
            raise ValueError(f"kv must have the shape of x {tuple(x.shape)}, got {tuple(kv.shape)}")
        q = F.linear(x, self.proj_q.weight, self.q_bias)
        k = F.linear(kv, self.proj_k.weight)
        v = F.linear(kv, self.proj_v.weight, self.v_bias)
        return tuple(split_heads(t, self.num_heads) for t in (q, k, v))

    def forward(self, x: Tensor, feats: Tensor, seqlens: Optional[Tensor] = None,
                key_padding_mask: Optional[Tensor] = None, kv: Optional[Tensor] = None,
                cu_seqlens: Optional[Tensor] = None) -> Tensor:
        from .forward import attention_qkv_zero_tail, flash_spacetime_attention, flash_spacetime_attention_qkv

        flags = (self.use_attn_bias, self.use_activation_bias)
        if cu_seqlens is not None:
            if kv is not None or seqlens is not None or key_padding_mask is not None:
                raise ValueError("packed input takes cu_seqlens only (self-attention, no lengths or mask)")
            if x.dim() != 2:
                raise ValueError(f"packed x must be [T, dim], got {tuple(x.shape)}")
            w, bias = self.qkv_weight()
            qkv = F.linear(x, w, bias).view(x.shape[0], 3, self.num_heads, self.head_dim)
            out = attention_qkv_zero_tail(qkv, feats, self.rel_proj.weight, self.rel_proj.bias, cu_seqlens, *flags)
            return self.proj(out.flatten(-2))
        b, length, _ = x.shape
        if kv is None:
            w, bias = self.qkv_weight()
            qkv = F.linear(x, w, bias).view(b, length, 3, self.num_heads, self.head_dim)
            out = flash_spacetime_attention_qkv(qkv, feats, self.rel_proj.weight, self.rel_proj.bias, seqlens,
                                                None, *flags, key_padding_mask=key_padding_mask)
            return self.proj(out.flatten(-2))
        q, k, v = self.project_qkv(x, kv)
        out = flash_spacetime_attention(q, k, v, feats, self.rel_proj.weight, self.rel_proj.bias, seqlens,
                                        None, *flags, key_padding_mask=key_padding_mask)
        return self.proj(merge_heads(out))


class SpacetimeBlock(nn.Module):
    """Pre-norm transformer block: spacetime attention and a gated feed-forward.

        x = x + attn(norm1(x));  x = x + ffn(norm2(x))

    as graphnet's `Block_rel` runs around the reference's operator (reference
    README.md:105-116), its two-layer MLP replaced by the gated block. `norm1`,
    `norm2`, `attn` (`SpacetimeAttention`) carry Block_rel's names; `ffn_gate`,
    `ffn_up`, `ffn_down` are the feed-forward's linears. `hidden` defaults to 8/3
    dim, rounded up to a multiple of 64 (the parameters of an ungated block of 4
    dim).

    `norm="rms"` runs root-mean-square norms (`nn.RMSNorm` parameters) in layer norm's
    place. With `experts=E` (up to 512) the feed-forward is a mixture: `router` (a linear
    without a bias) gives each token its logits, the `top_k` (up to 16) largest choose its
    experts and their softmax weighs them, and `experts_gate`, `experts_up` `[E, hidden, dim]` and
    `experts_down` `[E, dim, hidden]` are the experts' weights, without biases (`ffn_bias` is
    the one feed-forward's). Padding goes to no expert. Nothing keeps the loads
    even but the router: a penalty for uneven ones is the training's to add, from
    `router(..)`'s logits.

    `forward(x, feats, seqlens | key_padding_mask)` takes padded events `x [B, L,
    dim]`, or with `cu_seqlens` packed ones `[T, dim]`, and returns the same
    shape; padding rows (packed: those past `cu_seqlens[-1]`) are neither
    normalised nor multiplied by the feed-forward, whatever they hold, and come
    back as zeros. A stack saves a pass over the rows per block by leaving the last sum
    to the next block's norm: `defer=True` returns `(x, branch)`, whose sum is the
    block's output, and `branch=` takes the one the block before deferred.
    """

    # Of blocks pickled before there were experts, which have no attributes for them.
    experts: Optional[int] = None
    top_k = 2

    def __init__(self, dim: int, num_heads: int = 8, channels: int = 16, hidden: Optional[int] = None,
                 qkv_bias: bool = False, head_dim: Optional[int] = None, activation: str = "silu",
                 ffn_bias: bool = True, eps: float = 1e-5, use_attn_bias: bool = True,
                 use_activation_bias: bool = True, device=None, dtype=None, norm: str = "layer",
                 experts: Optional[int] = None, top_k: int = 2) -> None:
        super().__init__()
        fk = {"device": device, "dtype": dtype}
        if norm not in ("layer", "rms"):
            raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
        if experts is not None and not 1 <= top_k <= experts:
            raise ValueError(f"top_k must be 1 .. {experts} experts, got {top_k}")
        if experts is not None and (experts > 512 or top_k > 16):  # flash_expert_route's most
            raise ValueError(f"at most 512 experts and 16 of them a token, got {experts}, {top_k}")
        if hidden is None:
            hidden = -(-8 * dim // (3 * 64)) * 64
        make_norm = nn.LayerNorm if norm == "layer" else nn.RMSNorm
        self.norm1 = make_norm(dim, eps=eps, **fk)
        self.attn = SpacetimeAttention(dim, num_heads, channels, qkv_bias, head_dim, use_attn_bias,
                                       use_activation_bias, **fk)
        self.norm2 = make_norm(dim, eps=eps, **fk)
        self.experts, self.top_k = experts, top_k
        if experts is None:
            self.ffn_gate = nn.Linear(dim, hidden, bias=ffn_bias, **fk)
            self.ffn_up = nn.Linear(dim, hidden, bias=ffn_bias, **fk)
            self.ffn_down = nn.Linear(hidden, dim, bias=ffn_bias, **fk)
        else:
            self.router = nn.Linear(dim, experts, bias=False, **fk)
            self.experts_gate = nn.Parameter(torch.empty(experts, hidden, dim, **fk))
            self.experts_up = nn.Parameter(torch.empty(experts, hidden, dim, **fk))
            self.experts_down = nn.Parameter(torch.empty(experts, dim, hidden, **fk))
            for w in (self.experts_gate, self.experts_up, self.experts_down):  # as nn.Linear's
                nn.init.uniform_(w, -w.shape[-1] ** -0.5, w.shape[-1] ** -0.5)
        self.activation = activation

    def forward(self, x: Tensor, feats: Tensor, seqlens: Optional[Tensor] = None,
                key_padding_mask: Optional[Tensor] = None, cu_seqlens: Optional[Tensor] = None,
                branch: Optional[Tensor] = None, defer: bool = False):
        from .forward import _is_front_packed, _valid_from_mask

        if cu_seqlens is not None and (seqlens is not None or key_padding_mask is not None):
            raise ValueError("packed input takes cu_seqlens only (no lengths or mask)")
        if cu_seqlens is not None and (cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1):
            raise ValueError(f"cu_seqlens must be [events + 1], got {tuple(cu_seqlens.shape)}")
        if x.dim() != (2 if cu_seqlens is not None else 3):
            raise ValueError(f"x must be [T, dim] with cu_seqlens, else [B, L, dim], got {tuple(x.shape)}")
        if key_padding_mask is None and seqlens is not None and seqlens.dim() == 2:
            key_padding_mask, seqlens = seqlens, None
        if key_padding_mask is not None:
            if seqlens is not None:
                raise ValueError("pass either seqlens or key_padding_mask, not both")
            valid = _valid_from_mask(key_padding_mask, x.shape[1])
            if not _is_front_packed(valid):
                return self._scattered(x, feats, valid, branch, defer)
            seqlens = valid.sum(1, dtype=torch.int32)
        if cu_seqlens is None and seqlens is None:
            raise ValueError("seqlens, key_padding_mask or cu_seqlens is required")
        return self._block(x, feats, seqlens, cu_seqlens, branch, defer)

    def _block(self, x, feats, seqlens, cu_seqlens, branch, defer):
        from .norm import autocast_dtype

        if cu_seqlens is not None:  # packed tokens past the last offset are padding
            seqlens = cu_seqlens[-1:]
        if branch is None:
            y = self._norm(self.norm1, x, None, seqlens)
        else:
            y, x = self._norm(self.norm1, branch, x, seqlens)
        a = self.attn(y, feats, seqlens if cu_seqlens is None else None, cu_seqlens=cu_seqlens)
        y, x = self._norm(self.norm2, a, x, seqlens)
        low = autocast_dtype()
        if low is not None:  # as autocast has a linear's rows; the norms stay in the stream's type
            y = y.to(low)
        f = self._feed_forward(y, seqlens) if self.experts is None else self._mixture(y, seqlens)
        return (x, f) if defer else x + f

    def _norm(self, n, x, residual, seqlens):
        from .norm import flash_layer_norm
        from .rms_norm import flash_rms_norm

        if isinstance(n, nn.RMSNorm) or not hasattr(n, "bias"):
            return flash_rms_norm(x, n.weight, n.eps, residual=residual, seqlens=seqlens)
        return flash_layer_norm(x, n.weight, n.bias, n.eps, residual=residual, seqlens=seqlens)

    def _feed_forward(self, y, seqlens):
        from .feed_forward import flash_gated_feed_forward

        return flash_gated_feed_forward(y, self.ffn_gate.weight, self.ffn_up.weight, self.ffn_down.weight,
                                        self.ffn_gate.bias, self.ffn_up.bias, self.ffn_down.bias, self.activation,
                                        seqlens=seqlens)

    def _mixture(self, y, seqlens):
        from .experts import (flash_expert_combine, flash_expert_dispatch, flash_expert_feed_forward, flash_expert_route,
                              flash_expert_sort)

        weights, chosen = flash_expert_route(self.router(y), self.top_k, seqlens=seqlens)
        order = flash_expert_sort(chosen, self.experts)
        rows = flash_expert_feed_forward(flash_expert_dispatch(y, order), order.offsets, self.experts_gate, self.experts_up,
                                         self.experts_down, self.activation)
        return flash_expert_combine(rows, weights, order)

    def _scattered(self, x, feats, valid, branch, defer):
        """Masks with holes: the valid tokens as packed events, put back afterwards."""
        cu = torch.zeros(x.shape[0] + 1, dtype=torch.int32, device=x.device)
        cu[1:] = torch.cumsum(valid.sum(1, dtype=torch.int32), 0, dtype=torch.int32)
        out = self._block(x[valid], feats[valid], None, cu, None if branch is None else branch[valid], defer)
        back = lambda t: t.new_zeros(*x.shape[:2], t.shape[-1]).index_put((valid,), t)  # noqa: E731
        return tuple(back(t) for t in out) if defer else back(out)
