"""Multi-head differential attention as nn.Modules: the threshold form, and the softmax form with rotary
positions, a norm of the heads' outputs and decoding over a 4-bit or a paged cache (DifferentialAttention).

The reference ships only the functional operator (snap-research/TDA
triton_threshold_attention.py, TTA:472-519); the layer of the paper it accompanies (README.md:10)
wraps it between projections and learns beta and lambda.  This module is that wrapper:

    x (B, N, E) --fused projection--> q1, q2, k1, k2, v (B, N, H, d each)
      --> differential_threshold_rela_triton(q1, q2, k1, k2, v, beta, lambda, p, normalize)
      --> (B, N, H*d) --output projection--> (B, N, E)

The five projected tensors are strided (B, H, N, d) views of one (B, N, 5, H, d) projection
output, and the attention output is written in (B, N, H, d) order: no transposing copies on
either side (the kernels honour all four strides).  beta and lambda are learnable scalars by
default; lambda is clamped to [0, 1] inside the operator, with the inclusive gate of
torch.clamp on its gradient (TTA:516).
"""
from __future__ import annotations

import torch
from torch import nn

from .api import differential_threshold_rela_triton, threshold_rela_triton
from .kv_cache import Int4KVCache
from .norm import layer_norm
from .paged_cache import PagedKVCache
from .rotary import rotary_axes
from .softmax import differential_attention


class ThresholdDifferentialAttention(nn.Module):
    """Causal multi-head threshold differential attention (two-branch, TDA) or, with
    differential=False, threshold rectified attention (one branch, TRA).

    Args:
        embed_dim: model width E of the input and output.
        num_heads: H.
        head_dim: d, 16, 32, 64, 128 or 256 (default E // H).
        relu_power: p of ReLU(.)^p.
        normalize: cosine scores (L2-normalised q and k rows).
        beta_init, lambda_init: initial threshold scale and branch weight.
        learn_beta, learn_lambda: register them as parameters (else as buffers).
        differential: two branches (TDA) or one (TRA).
        bias: biases on the projections.
    """

    def __init__(self, embed_dim: int, num_heads: int, head_dim: int | None = None, *,
                 relu_power: float = 2.0, normalize: bool = True, beta_init: float = 1.0,
                 lambda_init: float = 0.5, learn_beta: bool = True, learn_lambda: bool = True,
                 differential: bool = True, bias: bool = False, device=None, dtype=None):
        super().__init__()
        head_dim = head_dim if head_dim is not None else embed_dim // num_heads
        if head_dim not in (16, 32, 64, 128, 256):
            raise ValueError(f"head_dim must be 16, 32, 64, 128 or 256, got {head_dim}")
        self.embed_dim, self.num_heads, self.head_dim = embed_dim, num_heads, head_dim
        self.relu_power, self.normalize, self.differential = float(relu_power), bool(normalize), differential
        self.n_proj = 5 if differential else 3  # q1, q2, k1, k2, v  |  q, k, v
        fk = {"device": device, "dtype": dtype}
        self.in_proj = nn.Linear(embed_dim, self.n_proj * num_heads * head_dim, bias=bias, **fk)
        self.out_proj = nn.Linear(num_heads * head_dim, embed_dim, bias=bias, **fk)
        beta = torch.tensor(float(beta_init), dtype=torch.float32, device=device)
        lam = torch.tensor(float(lambda_init), dtype=torch.float32, device=device)
        if learn_beta:
            self.beta = nn.Parameter(beta)
        else:
            self.register_buffer("beta", beta)
        if differential:
            if learn_lambda:
                self.lambda_param = nn.Parameter(lam)
            else:
                self.register_buffer("lambda_param", lam)
        else:
            self.lambda_param = None

    def _projection(self, x: torch.Tensor) -> torch.Tensor:
        b, n, _ = x.shape
        return self.in_proj(x).view(b, n, self.n_proj, self.num_heads, self.head_dim)

    def project(self, x: torch.Tensor):
        """The (B, H, N, d) views of the projected q1, q2, k1, k2, v (q, k, v for TRA).  A caller may
        edit a view in place."""
        y = self._projection(x)
        return [y[:, :, i].transpose(1, 2) for i in range(self.n_proj)]

    _own_project = project

    def _parts(self, x: torch.Tensor):
        """project(x), whoever defines it.  The class's own views are seen by the operator alone here, so
        they come from one unbind: its backward stacks the parts' gradients in one pass, where
        indexing fills, copies into and adds up a whole projection's gradient per part (a training step
        at (2, 1024), 16 heads of 64: 15 kernels and 268 us of GPU time against 28 and 340).
        autograd forbids editing an unbind's results in place."""
        if getattr(self.project, "__func__", None) is not ThresholdDifferentialAttention._own_project:
            return self.project(x)
        return [part.transpose(1, 2) for part in self._projection(x).unbind(2)]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x: (batch, seq_len, embed_dim), causal over seq_len."""
        if x.dim() != 3 or x.shape[-1] != self.embed_dim:
            raise ValueError(f"x must have shape (batch, seq_len, {self.embed_dim}), got {tuple(x.shape)}")
        b, n, _ = x.shape
        parts = self._parts(x)
        if self.differential:
            q1, q2, k1, k2, v = parts
            o = differential_threshold_rela_triton(q1, q2, k1, k2, v, self.beta, self.lambda_param,
                                                   self.relu_power, self.normalize)
        else:
            q, k, v = parts
            o = threshold_rela_triton(q, k, v, self.beta, self.relu_power, self.normalize)
        # o is (B, H, N, d) in (B, N, H, d) memory order when the inputs are such views
        return self.out_proj(o.transpose(1, 2).reshape(b, n, self.num_heads * self.head_dim))

    def extra_repr(self) -> str:
        return (f"embed_dim={self.embed_dim}, num_heads={self.num_heads}, head_dim={self.head_dim}, "
                f"relu_power={self.relu_power}, normalize={self.normalize}, differential={self.differential}")


class DifferentialAttention(nn.Module):
    """Causal multi-head softmax differential attention with rotary positions, for training and for decoding
    over a 4-bit or a paged cache:

        x (B, N, E) --fused projection--> q1, q2 (B, N, H, d), k1, k2 (B, N, Hk, d), v (B, N, Hk, dv)
          --> rotary_axes on q1, q2, k1, k2 --> differential_attention, or Int4KVCache.append and attend
              (or PagedKVCache.append, which turns them on the way, and attend)
          --> with head_norm: layer_norm of each head's output, without the mean
          --> (B, N, H*dv) --output projection--> (B, N, E)

    The projected tensors are strided views of one projection output and every operator keeps the
    (B, N, H, d) order: no transposing copies.

    Args:
        embed_dim: model width E of the input and output.
        num_heads, kv_heads: H and Hk (default H), a divisor of H.
        head_dim, v_head_dim: (64, 64), (64, 128), (128, 128) or (128, 256) (default E // H, head_dim).
        rotary_sections: rotated pairs of each axis of the positions, at most head_dim / 2 together
            (default: one axis that turns all of them).
        rotary_base: pair p of P turns by rotary_base^(-p / P) a position.
        lambda_init: initial weight of the second branch, learned per head.
        bias: biases on the projections.
        head_norm: normalise each head's output by its root mean square (with norm_eps, above 0: a row that saw no key
            is zeros, and zero by zero is NaN) and weigh its values, alike in every head; the weights are learned and
            start at 1 - lambda_init, the scale of a difference of maps.
    """

    def __init__(self, embed_dim: int, num_heads: int, head_dim: int | None = None, *, kv_heads: int | None = None,
                 v_head_dim: int | None = None, rotary_sections=None, rotary_base: float = 10000.0,
                 lambda_init: float = 0.5, bias: bool = False, head_norm: bool = False, norm_eps: float = 1e-5, device=None,
                 dtype=None):
        super().__init__()
        head_dim = head_dim if head_dim is not None else embed_dim // num_heads
        v_head_dim = v_head_dim if v_head_dim is not None else head_dim
        kv_heads = kv_heads if kv_heads is not None else num_heads
        if (head_dim, v_head_dim) not in ((64, 64), (64, 128), (128, 128), (128, 256)):
            raise ValueError("(head_dim, v_head_dim) must be (64, 64), (64, 128), (128, 128) or (128, 256), "
                             f"got {(head_dim, v_head_dim)}")
        if kv_heads < 1 or num_heads < 1 or num_heads % kv_heads:
            raise ValueError(f"num_heads ({num_heads}) must be a multiple of kv_heads ({kv_heads})")
        sections = (head_dim // 2,) if rotary_sections is None else tuple(int(s) for s in rotary_sections)
        pairs = sum(sections)
        if not 1 <= len(sections) <= 4 or min(sections) < 0 or not 1 <= pairs <= head_dim // 2:
            raise ValueError(f"rotary_sections must be 1 to 4 counts, together 1 to {head_dim // 2}, got {sections}")
        self.embed_dim, self.num_heads, self.kv_heads = embed_dim, num_heads, kv_heads
        self.head_dim, self.v_head_dim, self.rotary_sections = head_dim, v_head_dim, sections
        self._heads = (num_heads, num_heads, kv_heads, kv_heads, kv_heads)
        self._widths = (head_dim,) * 4 + (v_head_dim,)
        fk = {"device": device, "dtype": dtype}
        self.in_proj = nn.Linear(embed_dim, sum(h * w for h, w in zip(self._heads, self._widths)), bias=bias, **fk)
        self.out_proj = nn.Linear(num_heads * v_head_dim, embed_dim, bias=bias, **fk)
        self.lambda_param = nn.Parameter(torch.full((num_heads,), float(lambda_init), dtype=torch.float32, device=device))
        self.norm_eps = float(norm_eps)
        self.register_parameter("norm_weight", nn.Parameter(torch.full((v_head_dim,), 1.0 - float(lambda_init), **fk)) if head_norm else None)
        # on the CPU whatever the default device is: the frequencies have no copy in a checkpoint to come from
        self._inv_freq = (float(rotary_base) ** (-torch.arange(pairs, dtype=torch.float64, device="cpu") / pairs)).float()
        self._place()

    def __setstate__(self, state):
        super().__setstate__(state)
        self._parameters.setdefault("norm_weight", None)  # a layer that was pickled before it had a norm
        self.__dict__.setdefault("norm_eps", 1e-5)

    def _place(self):
        """The pairs' frequencies, in 32 bits whatever type the module is cast to, beside the weights: a call must not
        copy them from the host, which would make it wait and keep it out of a graph."""
        device = self.in_proj.weight.device
        if device.type != "meta" and self._inv_freq.device != device:
            with torch.inference_mode(False):  # as a tensor that a training step may save
                self._inv_freq = self._inv_freq.to(device)

    def _apply(self, fn, *args, **kw):
        super()._apply(fn, *args, **kw)
        self._place()
        return self

    def _frequencies(self) -> torch.Tensor:
        self._place()  # weights that were assigned, not moved
        return self._inv_freq

    def new_cache(self, batch: int, capacity: int) -> Int4KVCache:
        """An empty cache for this layer's keys and values, on its device."""
        return Int4KVCache(batch, self.kv_heads, capacity, self.head_dim, self.v_head_dim,
                           device=self.in_proj.weight.device)

    def new_paged_cache(self, pages: int, page_size: int = 64, *, dtype=None) -> PagedKVCache:
        """Pages for this layer's keys and values, on its weights' device and of their type, or of dtype: that in which the
        projection comes out, where the layer runs under torch.autocast."""
        w = self.in_proj.weight
        return PagedKVCache(pages, self.kv_heads, page_size, self.head_dim, self.v_head_dim, dtype=dtype or w.dtype, device=w.device)

    def project(self, x: torch.Tensor):
        """The (B, H or Hk, N, d or dv) views of the projected q1, q2, k1, k2, v.  They come from one split,
        whose backward joins the parts' gradients in one pass; autograd forbids editing them in place."""
        b, n, _ = x.shape
        parts = self.in_proj(x).split([h * w for h, w in zip(self._heads, self._widths)], dim=-1)
        return [p.view(b, n, h, w).transpose(1, 2) for p, h, w in zip(parts, self._heads, self._widths)]

    def forward(self, x: torch.Tensor, positions: torch.Tensor | None = None, kv_lens: torch.Tensor | None = None,
                cache: Int4KVCache | PagedKVCache | None = None, *, table: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None, starts: torch.Tensor | None = None,
                counts: torch.Tensor | None = None) -> torch.Tensor:
        """x: (batch, seq_len, embed_dim), causal over seq_len; positions: int32 or int64, (axes, batch,
        seq_len), by default the same count on every axis.  kv_lens (batch,) hides the rows of a padded
        batch from then on.

        With a cache, x are the next seq_len positions of each sequence: their keys and values are appended
        and the attention runs over all that the cache holds, without gradients; positions count from
        the cache's lengths by default.  Rows past the cache's capacity are dropped, as append() drops them: a
        caller keeps count.  A prompt padded at its end is decoded on from after cache.lengths
        is set to the sequences' own lengths.

        A PagedKVCache needs table and lengths, and takes x in any of its three forms (with counts a padded batch, with
        starts a packed one, (1, rows, embed_dim)): see there.  lengths are what the sequences held before, and are
        the caller's to add to once every layer has run.  Rows of no sequence give the output projection's bias."""
        if x.dim() != 3 or x.shape[-1] != self.embed_dim:
            raise ValueError(f"x must have shape (batch, seq_len, {self.embed_dim}), got {tuple(x.shape)}")
        paged = isinstance(cache, PagedKVCache)
        if paged and (table is None or lengths is None):
            raise ValueError("a paged cache needs table and lengths")
        if not paged and any(t is not None for t in (table, lengths, starts, counts)):
            raise ValueError("table, lengths, starts and counts go with a paged cache")
        where = {"table": table, "lengths": lengths, "starts": starts, "counts": counts}
        if cache is not None:
            if kv_lens is not None:
                raise ValueError("kv_lens and cache exclude each other: a cache has its own lengths")
            if not paged and x.shape[0] != cache.batch:
                raise ValueError(f"the cache holds {cache.batch} sequences, x has {x.shape[0]}")
            if torch.is_grad_enabled():
                with torch.no_grad():
                    return self.forward(x, positions, None, cache, **(where if paged else {}))
        b, n, _ = x.shape
        q1, q2, k1, k2, v = self.project(x)
        if paged:
            q1, q2 = cache.append(k1, k2, v, q1=q1, q2=q2, **where, inv_freq=self._frequencies(), sections=self.rotary_sections,
                                  positions=positions)
            return self._output(cache.attend(q1, q2, self.lambda_param, **where))
        if positions is None:
            positions = torch.arange(n, device=x.device).expand(len(self.rotary_sections), b, n)
            if cache is not None:
                positions = positions + cache.lengths[:, None]
        q1, q2, k1, k2 = rotary_axes((q1, q2, k1, k2), positions, self._frequencies(), self.rotary_sections)
        if cache is None:
            return self._output(differential_attention(q1, q2, k1, k2, v, self.lambda_param, kv_lens=kv_lens))
        cache.append(k1, k2, v)
        return self._output(cache.attend(q1, q2, self.lambda_param))

    def _output(self, o: torch.Tensor) -> torch.Tensor:
        if self.norm_weight is not None:
            o = layer_norm(o, self.norm_weight, eps=self.norm_eps, center=False)
        return self.out_proj(o.transpose(1, 2).flatten(2))

    def extra_repr(self) -> str:
        return (f"embed_dim={self.embed_dim}, num_heads={self.num_heads}, kv_heads={self.kv_heads}, "
                f"head_dim={self.head_dim}, v_head_dim={self.v_head_dim}, rotary_sections={self.rotary_sections}"
                + ("" if self.norm_weight is None else f", head_norm=True, norm_eps={self.norm_eps}"))
