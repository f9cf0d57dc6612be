"""A dense attention layer over an 8-bit cache, behind ``semblo::attention``.

A model's full-attention layers need not all be sparse: this is the layer beside ``model.SembloAttention`` that reads
every key.  It is reached through the same operator (its name in the operator's table), takes the same tensors, and
keeps one request's keys and values in a ``QuantizedKVCache``:

  prefill   a call of more than one token starts a new request: its tokens attend to one another in bf16
            (``kv_outer.dense_causal_attention``), and are left in the cache
  extend    more tokens at once (a further turn, a prompt in slices, a guess to be checked), over the cache
  decode    one token, over the cache

With ``keep_blocks`` the layer also weighs the cache's blocks as it decodes, and when the cache has no room for a block
more cuts it to the ``keep_blocks`` most attended ones (the first ``sink_blocks`` and the last ``recent_blocks`` always
stay).  With ``rotary`` the layer rotates the queries and keys itself: the operator's q_pre and k_pre are then
all it reads, and q_post and k_post may be any tensors.

The layer counts its tokens on the host, so its calls cannot be captured in a HIP graph (they raise): a captured decode
calls the cache itself, ``layer.cache.append`` and ``layer.cache.attend``.
"""
from __future__ import annotations

import torch

from .attention_op import register_layer
from .config import SembloRuntimeConfig
from .kv_cache8 import BLOCK, QuantizedKVCache
from .kv_outer import dense_causal_attention, dense_launch_queries
from .rotary import RotaryEmbedding

WEIGHED_ROWS = 64       # a prompt's last rows, whose attention is its blocks' first weight


class DenseCacheAttention:
    """One dense layer's attention and its cache (one request at a time)."""

    def __init__(self, config: SembloRuntimeConfig, *, capacity: int, device, fmt: str = "e4m3",
                 layer_name: str | None = None, rotary: RotaryEmbedding | None = None, keep_blocks: int = 0,
                 sink_blocks: int = 1, recent_blocks: int = 16) -> None:
        self.runtime_config = config
        self.num_heads, self.num_kv_heads, self.head_dim = config.num_q_heads, config.num_kv_heads, config.head_dim
        self.scaling = config.scale
        if self.num_heads % self.num_kv_heads or self.num_heads // self.num_kv_heads not in (1, 2, 4, 8):
            raise ValueError("a dense layer takes 1, 2, 4 or 8 query heads to a KV head")
        if rotary is not None and rotary.head_dim != self.head_dim:
            raise ValueError(f"the rotary embedding is for heads of {rotary.head_dim}, the layer's are {self.head_dim}")
        self.cache = QuantizedKVCache(num_seqs=1, num_kv_heads=self.num_kv_heads, head_dim=self.head_dim,
                                      capacity=capacity, fmt=fmt, device=device)
        if keep_blocks and not (sink_blocks >= 0 and recent_blocks >= 1
                                and sink_blocks + recent_blocks <= keep_blocks < self.cache.num_blocks):
            raise ValueError(f"keep_blocks ({keep_blocks}) must hold sink_blocks + recent_blocks ({sink_blocks} + "
                             f"{recent_blocks}, one recent at least) and be below the cache's {self.cache.num_blocks}")
        self.rotary = rotary
        self.keep_blocks, self.sink_blocks, self.recent_blocks = int(keep_blocks), int(sink_blocks), int(recent_blocks)
        self.tokens = 0         # held by the cache, counted on the host
        self.layer_name = layer_name or f"semblo.dense.{config.layer_idx}"
        register_layer(self.layer_name, self)

    def _heads(self, x: torch.Tensor, heads: int, what: str) -> torch.Tensor:
        t = x.shape[0]
        if x.numel() != t * heads * self.head_dim:
            raise ValueError(f"{what} must hold {heads} heads of {self.head_dim} per token, got {list(x.shape)}")
        return x.view(t, heads, self.head_dim) if x.is_contiguous() else x.reshape(t, heads, self.head_dim)

    def reset(self) -> None:
        """Ends the request: the next call starts a new one (as a prompt of more than one token does by itself)."""
        self.cache.reset()
        self.tokens = 0

    @staticmethod
    def _not_captured() -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a dense layer counts its tokens on the host: capture its cache's append and attend instead")

    def _room(self, tokens: int) -> None:
        """Makes room for ``tokens`` more, by an eviction where the layer evicts."""
        if self.tokens + tokens <= self.cache.capacity:
            return
        blocks = -(-self.tokens // BLOCK)
        if self.keep_blocks and blocks > self.keep_blocks:
            self.cache.evict(self.keep_blocks, sink=self.sink_blocks, recent=self.recent_blocks)
            self.tokens -= (blocks - self.keep_blocks) * BLOCK
        if self.tokens + tokens > self.cache.capacity:
            raise RuntimeError(f"the dense layer's cache has room for {self.cache.capacity} tokens, not for "
                               f"{self.tokens} + {tokens}")

    def prefill(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, output: torch.Tensor) -> torch.Tensor:
        """A new request's prompt: rotated q [T, Hq, D], k and v [T, Hkv, D], into ``output`` [T, Hq * D]."""
        t = q.shape[0]
        if t > self.cache.capacity:
            raise RuntimeError(f"a prompt of {t} tokens passes the cache's room for {self.cache.capacity}")
        self._not_captured()
        self.reset()
        out = output.view(t, self.num_heads, self.head_dim)
        most = dense_launch_queries(self.num_kv_heads, self.num_heads // self.num_kv_heads)
        if k.stride() != v.stride():
            k, v = k.contiguous(), v.contiguous()
        for start in range(0, t, most):
            end = min(t, start + most)
            dense_causal_attention(q[start:end], k, v, sm_scale=self.scaling, chunk_start=start, out=out[start:end])
        self.cache.append(k, v)
        self.tokens = t
        if self.keep_blocks:
            self.cache.attend(q[-WEIGHED_ROWS:], sm_scale=self.scaling, accumulate=True)
        return output

    def extend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, output: torch.Tensor) -> torch.Tensor:
        """More tokens of the request (one, or several at once), over the cache: as ``prefill``."""
        t = q.shape[0]
        self._not_captured()
        self._room(t)
        self.cache.append(k, v)
        self.tokens += t
        out = output.view(t, self.num_heads, self.head_dim)
        self.cache.attend(q, sm_scale=self.scaling, accumulate=bool(self.keep_blocks), out=out)
        return output

    def attention_forward(self, positions, hidden_states, q_post, k_post, v_states, q_pre, k_pre, output) -> None:
        """The operator's body: more than one token starts a new request, one goes on with it."""
        t = output.shape[0]
        if v_states is None or (k_post if self.rotary is None else k_pre) is None:
            raise RuntimeError("a dense layer needs the tokens' keys and values")
        if self.rotary is None:
            q, k = self._heads(q_post, self.num_heads, "q_post"), self._heads(k_post, self.num_kv_heads, "k_post")
        else:
            q, k = self.rotary(positions, self._heads(q_pre, self.num_heads, "q_pre"),
                               self._heads(k_pre, self.num_kv_heads, "k_pre"))
        v = self._heads(v_states, self.num_kv_heads, "v_states")
        if t > 1 or self.tokens == 0:
            self.prefill(q, k, v, output)
        else:
            self.extend(q, k, v, output)
