"""Multi-head attention layer over the gfx950 kernels.

``EnhancedMultiHeadAttention`` keeps the constructor and ``forward`` of the
reference's module (``examples/basic_usage.py:48-255``): Q/K/V/output linear
projections with Xavier-uniform weights and zero biases, (B, S, E) or
(S, B, E) inputs, boolean ``attn_mask`` / ``key_padding_mask`` turned into an
additive ``-inf`` bias, ``is_causal``, dropout only in training mode, and an
``(output, attn_weights)`` return whose weights are not computed.

Differences, all deliberate:

* The masks become a bias that broadcasts over the dimensions they do not
  name ((1|B, 1, Sq|1, Sk)) instead of a materialised (B, H, Sq, Sk) tensor;
  the kernels read broadcast dimensions with stride 0.  A float ``attn_mask``
  is added as it is (the reference's ``masked_fill`` accepted booleans only).
* A query row whose keys are all masked gives zeros (the reference's softmax
  gave NaN there).
* ``enable_gradient_checkpointing`` is honoured: the layer's attention keeps
  only q, k, v and the LSE for the backward (the reference stored the flag).
* ``enable_performance_monitoring`` times each forward with HIP events on the
  current stream (the reference used its profiler module, which is out of
  scope); :meth:`get_performance_stats` reports count and mean milliseconds.
* ``enable_multi_gpu`` is accepted and ignored (one GPU).

Beyond the reference's layer, all off by default: rotary positions
(``rotary_dim``), a cap on the scores (``softcap``), a learned distance bias per
head (``distance_bias``) and sequences packed from documents
(``forward(documents=)``).
"""
from __future__ import annotations

import contextlib
import warnings
from typing import Any, Dict, Optional, Tuple

import torch
import torch.nn as nn

from .interface import flash_attention_performance_mode, flash_attention_v100
from .ops.attention import gradient_checkpointing_mode
from .ops.rotary import rotary_embedding_v100, rotary_table_v100
from .ops.scored import flash_attention_v100_scored


def mask_to_bias(attn_mask: Optional[torch.Tensor], key_padding_mask: Optional[torch.Tensor], batch: int,
                 seq_q: int, seq_k: int, dtype: torch.dtype, device) -> Optional[torch.Tensor]:
    """Additive bias of shape (1|B, 1, Sq|1, Sk) from the reference's masks
    (``examples/basic_usage.py:232-251``): a True entry of a boolean mask
    removes that key (-inf); a float ``attn_mask`` is added as it is.
    ``attn_mask`` is (Sq, Sk) or (B, Sq, Sk); ``key_padding_mask`` is (B, Sk)."""
    if attn_mask is None and key_padding_mask is None:
        return None
    bias = None
    if attn_mask is not None:
        if attn_mask.dim() not in (2, 3):
            raise ValueError(f"attn_mask must be 2-D (Sq, Sk) or 3-D (B, Sq, Sk), got shape {tuple(attn_mask.shape)}")
        am = attn_mask.to(device)
        if am.dtype == torch.bool:
            am = torch.zeros(am.shape, device=device, dtype=dtype).masked_fill(am, float("-inf"))
        else:
            am = am.to(dtype)
        bias = am.unsqueeze(0).unsqueeze(0) if am.dim() == 2 else am.unsqueeze(1)
        if bias.shape[-2:] != (seq_q, seq_k) or bias.shape[0] not in (1, batch):
            raise ValueError(f"attn_mask shape {tuple(attn_mask.shape)} does not match (B={batch}, Sq={seq_q}, "
                             f"Sk={seq_k})")
    if key_padding_mask is not None:
        if tuple(key_padding_mask.shape) != (batch, seq_k):
            raise ValueError(f"key_padding_mask must be (B={batch}, Sk={seq_k}), got {tuple(key_padding_mask.shape)}")
        kp = key_padding_mask.to(device)
        if kp.dtype == torch.bool:
            kp = torch.zeros(kp.shape, device=device, dtype=dtype).masked_fill(kp, float("-inf"))
        else:
            kp = kp.to(dtype)
        kp = kp.view(batch, 1, 1, seq_k)
        bias = kp if bias is None else bias + kp
    return bias


class EnhancedMultiHeadAttention(nn.Module):
    """Multi-head attention with the reference's module interface
    (``examples/basic_usage.py:48-255``) over :func:`flash_attention_v100`.

    ``rotary_dim`` > 0 rotates the first columns of each head of q and k by
    their positions (:func:`rotary_embedding_v100`), below ``max_positions``;
    ``rotary_scaling`` are more arguments of :func:`rotary_table_v100`.
    ``softcap`` > 0, ``distance_bias`` (float32 slopes, a parameter, 2^(-8 h / H)
    for head h = 1 .. H at first) and ``forward(documents=)`` go to
    :func:`flash_attention_v100_scored`, which has no dropout and no additive
    mask: with one of them, training with ``dropout`` and any ``attn_mask`` raise
    ``ValueError``, and ``key_padding_mask`` must be boolean."""

    def __init__(self,
                 embed_dim: int,
                 num_heads: int,
                 dropout: float = 0.0,
                 bias: bool = True,
                 batch_first: bool = True,
                 optimization_strategy: str = "balanced",
                 enable_multi_gpu: bool = True,
                 enable_gradient_checkpointing: bool = False,
                 enable_performance_monitoring: bool = False,
                 rotary_dim: int = 0,
                 rotary_base: float = 10000.0,
                 rotary_interleaved: bool = False,
                 rotary_scaling: Optional[Dict[str, Any]] = None,
                 max_positions: int = 8192,
                 softcap: float = 0.0,
                 distance_bias: bool = False):
        super().__init__()
        assert embed_dim % num_heads == 0, "embed_dim must be divisible by num_heads"
        if rotary_dim < 0 or rotary_dim % 2 or rotary_dim > embed_dim // num_heads:
            raise ValueError(f"rotary_dim must be even, 0..{embed_dim // num_heads}, got {rotary_dim}")
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.head_dim = embed_dim // num_heads
        self.dropout = dropout
        self.batch_first = batch_first
        self.optimization_strategy = optimization_strategy
        self.enable_multi_gpu = enable_multi_gpu
        self.enable_gradient_checkpointing = enable_gradient_checkpointing
        self.enable_performance_monitoring = enable_performance_monitoring
        self.q_proj = nn.Linear(embed_dim, embed_dim, bias=bias)
        self.k_proj = nn.Linear(embed_dim, embed_dim, bias=bias)
        self.v_proj = nn.Linear(embed_dim, embed_dim, bias=bias)
        self.out_proj = nn.Linear(embed_dim, embed_dim, bias=bias)
        self.rotary_dim, self.rotary_base, self.rotary_interleaved = rotary_dim, rotary_base, rotary_interleaved
        self.rotary_scaling, self.max_positions = dict(rotary_scaling or {}), max_positions
        self.softcap = softcap
        self.distance_slopes = nn.Parameter(torch.empty(num_heads)) if distance_bias else None
        self._tables = {}  # rotary table of each device and set of options
        self.forward_count = 0
        self._times_ms = []
        self._pending = []
        self.reset_parameters()

    def reset_parameters(self):
        """Xavier-uniform projection weights, zero biases (reference ``:112-123``)."""
        for lin in (self.q_proj, self.k_proj, self.v_proj, self.out_proj):
            nn.init.xavier_uniform_(lin.weight)
            if lin.bias is not None:
                nn.init.constant_(lin.bias, 0)
        if self.distance_slopes is not None:
            with torch.no_grad():
                h = torch.arange(1, self.num_heads + 1, dtype=torch.float64)
                self.distance_slopes.copy_(torch.exp2(-8.0 * h / self.num_heads))

    def __getstate__(self):
        # the tables are made again where they are needed
        state = dict(super().__getstate__() if hasattr(super(), "__getstate__") else self.__dict__)
        state["_tables"] = {}
        return state

    def __setstate__(self, state):
        # layers saved before these existed
        off = {"rotary_dim": 0, "softcap": 0.0, "max_positions": 8192, "_tables": {}}
        super().__setstate__({**off, **state})
        if "distance_slopes" not in self._parameters and "distance_slopes" not in self.__dict__:
            self.distance_slopes = None

    def _rotary_table(self, device: torch.device) -> torch.Tensor:
        # (a table of earlier options stays: a graph captured with it may be replayed)
        key = (device, self.max_positions, self.rotary_dim, self.rotary_base, tuple(sorted(self.rotary_scaling.items())))
        t = self._tables.get(key)
        if t is None:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call the layer once before it is captured: its rotary table is made on first use, and "
                                   "again after a change of its options")
            # kept for training too, also where the first call runs in inference mode
            with torch.inference_mode(False):
                t = rotary_table_v100(self.max_positions, self.rotary_dim, self.rotary_base, device=device,
                                      **self.rotary_scaling)
            # made on this stream, read on any: whole before another can see it
            torch.cuda.current_stream(device).synchronize()
            self._tables[key] = t
        return t

    def _scored(self, q, k, v, attn_mask, key_padding_mask, is_causal, documents):
        """Attention with the rules that :func:`flash_attention_v100` has not."""
        if self.training and self.dropout > 0.0:
            raise ValueError("softcap, distance_bias and documents have no attention dropout: use dropout=0.0")
        if attn_mask is not None:
            raise ValueError("softcap, distance_bias and documents take no attn_mask (is_causal, key_padding_mask and "
                             "documents are supported)")
        B, Sq, Sk = q.shape[0], q.shape[1], k.shape[1]
        key_documents = None
        if documents is not None and Sq != Sk:
            raise ValueError(f"documents need queries and keys of one sequence, got lengths {Sq} and {Sk}")
        if key_padding_mask is not None:
            if key_padding_mask.dtype != torch.bool or tuple(key_padding_mask.shape) != (B, Sk):
                raise ValueError(f"key_padding_mask must be boolean (B={B}, Sk={Sk}) with softcap, distance_bias or "
                                 "documents")
            pad = key_padding_mask.to(q.device)
            if documents is None:
                documents = torch.zeros((B, Sq), dtype=torch.int32, device=q.device)
                key_documents = torch.zeros((B, Sk), dtype=torch.int32, device=q.device).masked_fill(pad, -1)
            else:
                key_documents = documents.expand(B, Sk).masked_fill(pad, -1)
        slopes = None if self.distance_slopes is None else self.distance_slopes.float()
        return flash_attention_v100_scored(q, k, v, causal=is_causal, softcap=self.softcap, distance_slopes=slopes,
                                           documents=documents, key_documents=key_documents)

    def forward(self,
                query: torch.Tensor,
                key: Optional[torch.Tensor] = None,
                value: Optional[torch.Tensor] = None,
                key_padding_mask: Optional[torch.Tensor] = None,
                attn_mask: Optional[torch.Tensor] = None,
                need_weights: bool = False,
                average_attn_weights: bool = True,
                is_causal: bool = False,
                positions: Optional[torch.Tensor] = None,
                documents: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """(output, attn_weights); see the module docstring.  ``positions``: the
        tokens' rotary positions, (B, S) or (S,), 0 .. S - 1 by default;
        ``documents``: integer ids, (B, S) or (S,), negative for padding.  ``need_weights``
        warns and returns zeros of shape (B, H, Sq, Sk), as the reference does
        (``:194-199, 218-221``): the kernels never form the weights."""
        timing = self.enable_performance_monitoring and query.is_cuda
        if timing:
            self.forward_count += 1
            ev0, ev1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            ev0.record()
        if not self.batch_first:
            query = query.transpose(0, 1)
            key = key.transpose(0, 1) if key is not None else None
            value = value.transpose(0, 1) if value is not None else None
        if key is None:
            key = query
        if value is None:
            value = key
        B, Sq, E = query.shape
        Sk = key.shape[1]
        q = self.q_proj(query).view(B, Sq, self.num_heads, self.head_dim)
        k = self.k_proj(key).view(B, Sk, self.num_heads, self.head_dim)
        v = self.v_proj(value).view(B, value.shape[1], self.num_heads, self.head_dim)
        if self.rotary_dim:
            table = self._rotary_table(q.device)
            if positions is not None and Sq != Sk:
                raise ValueError(f"positions need queries and keys of one sequence, got lengths {Sq} and {Sk}")
            if max(Sq, Sk) > self.max_positions and positions is None:
                raise ValueError(f"{max(Sq, Sk)} tokens exceed max_positions={self.max_positions}")
            if Sq == Sk:
                q, k = rotary_embedding_v100(q, k, table, positions, interleaved=self.rotary_interleaved)
            else:
                q = rotary_embedding_v100(q, None, table, interleaved=self.rotary_interleaved)
                k = rotary_embedding_v100(k, None, table, interleaved=self.rotary_interleaved)
        elif positions is not None:
            raise ValueError("positions need rotary_dim > 0")
        scored = self.softcap > 0.0 or self.distance_slopes is not None or documents is not None
        bias = None if scored else mask_to_bias(attn_mask, key_padding_mask, B, Sq, Sk, q.dtype, q.device)
        if need_weights:
            warnings.warn("need_weights=True not supported with Flash Attention. "
                          "Attention weights will not be returned.", UserWarning)
        ckpt = gradient_checkpointing_mode() if self.enable_gradient_checkpointing else contextlib.nullcontext()
        with flash_attention_performance_mode(self.optimization_strategy), ckpt:
            if scored:
                out = self._scored(q, k, v, attn_mask, key_padding_mask, is_causal, documents)
            else:
                out = flash_attention_v100(q, k, v, causal=is_causal,
                                           dropout_p=self.dropout if self.training else 0.0,
                                           bias=bias, optimization_strategy=self.optimization_strategy,
                                           enable_multi_gpu=self.enable_multi_gpu,
                                           enable_profiling=self.enable_performance_monitoring,
                                           fallback_on_error=True)
        out = self.out_proj(out.reshape(B, Sq, E))
        if not self.batch_first:
            out = out.transpose(0, 1)
        weights = None
        if need_weights:
            weights = torch.zeros(B, self.num_heads, Sq, Sk, device=out.device, dtype=out.dtype)
        if timing:
            ev1.record()
            self._pending.append((ev0, ev1))
        return out, weights

    def get_performance_stats(self) -> Optional[Dict[str, Any]]:
        """Forward count and HIP-event times (ms) when monitoring is enabled."""
        if not self.enable_performance_monitoring:
            return None
        for ev0, ev1 in self._pending:
            ev1.synchronize()
            self._times_ms.append(ev0.elapsed_time(ev1))
        self._pending = []
        n = len(self._times_ms)
        return {"forward_count": self.forward_count,
                "mean_ms": sum(self._times_ms) / n if n else None,
                "total_ms": sum(self._times_ms)}
