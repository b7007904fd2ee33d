"""Attention over the active sites of a ``SparseConvTensor``: the operators
and the module built from them.  The reference has no counterpart; they stand
beside its sparse convolutions, whose reach is a kernel window.

* ``packed_attention``: softmax attention over packed sequences of different
  lengths, full or causal, query heads sharing key heads, forward and
  backward; few queries against long keys (one token of a stream against its
  cache) are split over the keys.
* ``qk_norm_rotary``: RMS norm of each query and key head and its rotary
  position, from one or several coordinates, in one pass.
* ``residual_dropout``: dropout onto the residual stream from a counter-based
  generator; the mask is drawn again in the backward, never stored.
* ``SparseSelfAttention``: a pre-norm attention block that uses all three.

Under ``torch.autocast`` the attention's operands are cast to the autocast
dtype and results come back in the dtype of the input, as in the sparse
convolutions.
"""
from __future__ import annotations

import torch
from torch import nn

from ..._lib import ops
from .modules import SparseModule
from .ops import _require_cuda
from .structure import SparseConvTensor

_handles = None


def _native():
    """The three operators, looked up once: a call is short enough for the look-up to show."""
    global _handles
    if _handles is None:
        o = ops()
        _handles = (o.packed_attention.default, o.qk_norm_rotary.default, o.residual_dropout.default)
    return _handles


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                     cu_seqlens_k: torch.Tensor | None = None, kv_lengths: torch.Tensor | None = None,
                     causal: bool = False, scale: float | None = None, return_lse: bool = False):
    """Attention of each sequence's queries to its keys.

    ``q`` [queries, heads, dim], ``k`` and ``v`` [keys, kv_heads, dim]: fp16 or
    bf16 CUDA tensors, ``dim`` a multiple of 8 up to 128, ``heads`` a multiple
    of ``kv_heads`` (query head h reads key head h // (heads // kv_heads)).
    Slices of a wider projection are read in place where their rows start on
    16 bytes.  ``cu_seqlens_q`` [sequences + 1] (int32 or int64, ascending)
    holds where each sequence starts and the last ends; ``cu_seqlens_k`` the
    same for the keys (default: the queries').  ``kv_lengths`` [sequences]
    says how many of each sequence's key rows hold keys (default: all), for
    caches with room to grow.

    ``causal``: query i sees key j where j <= i + keys - queries, so the last
    query sees every key.  ``scale`` defaults to dim ** -0.5.

    Returns out [queries, heads, dim] (and, with ``return_lse``, the fp32
    log of each query's sum of exponentials, [heads, queries]).  A query that
    sees no key and a row that no sequence holds get 0 (and -inf), and pass
    no gradient, whatever they and their gradients hold.  Rows of ``k`` and
    ``v`` outside every sequence and past ``kv_lengths`` may hold anything; a
    non-finite ``v`` inside a sequence may reach all queries of that sequence,
    and a non-finite value of a query that sees keys, of a key or of a gradient
    all gradients of the sequence, hidden or not.  Gradients are deterministic;
    the probabilities and their gradients are rounded to the inputs' type
    inside (in fp16 times powers of two that keep them out of the subnormal
    numbers), which leaves dq and dk relative errors of up to 0.0026 in bf16
    and 0.0003 in fp16 (0.0017 and 0.0002 with fp32 inside).  Second derivatives
    and forward mode are refused.
    """
    _require_cuda(q, k, v, cu_seqlens_q)
    if scale is None:
        scale = max(q.size(-1), 1) ** -0.5
    back = None
    if torch.is_autocast_enabled('cuda') and q.is_cuda:
        dt = torch.get_autocast_dtype('cuda')
        back = None if q.dtype == dt else q.dtype
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    out, lse = _native()[0](q, k, v, cu_seqlens_q, cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k, kv_lengths,
                             bool(causal), float(scale))
    if back is not None:
        out = out.to(back)
    return (out, lse) if return_lse else out


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections,
                   q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                   interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys with the norm of each head and its rotary position.

    ``q`` [tokens, heads, dim] and ``k`` [tokens, kv_heads, dim] (fp32, fp16 or
    bf16; ``dim`` a multiple of 8 up to 256) are computed in fp32 and rounded
    once.  A head with a weight [dim] becomes x * rsqrt(mean(x ** 2) + eps) *
    weight; without one it is not normed.  Then pair f of its values turns by
    positions[token, axis(f)] * inv_freq[f]: ``sections`` counts the pairs of
    each axis, in order (1 to 8 axes), and their sum, the length of
    ``inv_freq`` (fp32 or fp64), is half the rotated width R <= dim.  A pair is
    (i, i + R / 2), with R a multiple of 16, or with ``interleaved``
    (2 i, 2 i + 1); values past R are not turned.  ``positions`` [tokens, axes]
    is int32, int64 or fp32, of any strides; far positions lose no accuracy
    (sine and cosine are good to fp32 for fp32 tensors, to 2 ** -20 for the
    others).  Differentiable in ``q``, ``k`` and the weights.
    """
    _require_cuda(q, k, positions, inv_freq)
    if q_weight is not None and q_weight.dtype != torch.float32:
        q_weight = q_weight.float()
    if k_weight is not None and k_weight.dtype != torch.float32:
        k_weight = k_weight.float()
    return _native()[1](q, k, positions, inv_freq, sections, q_weight, k_weight, eps, bool(interleaved))


def residual_dropout(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: torch.Tensor) -> torch.Tensor:
    """residual + dropout(x, p); ``residual`` None: dropout alone.

    ``seed`` is an int64 CUDA tensor of two values (key, offset): value i of
    ``x`` (in its contiguous order) is kept where word i % 4 of Philox 4x32-10
    at counter (i // 4, offset) is at least floor(p * 2 ** 32), and then scaled
    by 1 / (1 - p).  The same seed gives the same mask, in the backward pass
    too, which reads nothing but the seed; a captured graph draws anew when the
    seed's values are changed between replays.  0 <= p <= 1.
    """
    _require_cuda(x, seed)
    return _native()[2](x, residual, p, seed)


def sample_offsets(indices: torch.Tensor, batch_size: int) -> torch.Tensor:
    """Where each sample's rows start, int32 [batch_size + 1], from site rows
    (b, ..) that are in ascending order of b.  No host synchronisation."""
    samples = torch.arange(batch_size + 1, dtype=indices.dtype, device=indices.device)
    return torch.searchsorted(indices[:, 0].contiguous(), samples, out_int32=True)


class SparseSelfAttention(SparseModule):
    """Every active site attends to the sites of its sample: layer norm,
    projection to ``heads`` queries and ``kv_heads`` keys and values of
    channels // heads, ``qk_norm_rotary`` at the sites' coordinates,
    ``packed_attention``, projection, ``residual_dropout`` onto the input.

    The tensor's rows may come in any order: of several samples they are
    gathered by sample first (in their order within it) and the result is put
    back, without a look at the host; ``grouped=True`` promises that they come
    sample by sample already, in ascending order, as from voxelisation and the
    strided convolutions, and saves that.  Features are fp16 or bf16, or
    any floating type under ``torch.autocast``; the width of a head is a
    multiple of 16 up to 128.  ``causal`` lets a site see only the rows of its
    sample up to its own.
    """

    def __init__(self, channels, heads, kv_heads=None, ndim=3, dropout=0.0, causal=False, rotary_base=10000.0,
                 qk_norm=True, bias=True, eps=1e-6, grouped=False):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if channels % heads or heads % kv_heads:
            raise ValueError('channels must be a multiple of heads, and heads of kv_heads')
        dim = channels // heads
        if dim % 16 or dim > 128:
            raise ValueError(f'a head must have a multiple of 16 up to 128 channels, got {dim}')
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f'dropout must be a probability, got {dropout}')
        self.heads, self.kv_heads, self.dim, self.ndim = heads, kv_heads, dim, ndim
        self.dropout, self.causal, self.eps, self.grouped = dropout, causal, eps, grouped
        pairs = dim // 2
        # near equal shares of the pairs; the first axes (the coarser ones) get the smaller
        self.sections = [pairs // ndim + (1 if a >= ndim - pairs % ndim else 0) for a in range(ndim)]
        # kept out of the buffers, which .half() would round
        self.inv_freq = torch.cat([rotary_base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
                                   for n in self.sections]).float()
        self.norm = nn.LayerNorm(channels)
        self.qkv = nn.Linear(channels, (heads + 2 * kv_heads) * dim, bias=bias)
        self.proj = nn.Linear(channels, channels, bias=bias)
        self.q_weight = nn.Parameter(torch.ones(dim)) if qk_norm else None
        self.k_weight = nn.Parameter(torch.ones(dim)) if qk_norm else None

    def _apply(self, fn, recurse=True):
        """Moves ``inv_freq`` along with the parameters, so that no call has to (a copy from the host cannot be
        captured into a graph)."""
        super()._apply(fn, recurse)
        if not self.norm.weight.is_meta:  # there its values would be lost
            self.inv_freq = self.inv_freq.to(self.norm.weight.device)
        return self

    def forward(self, input: SparseConvTensor) -> SparseConvTensor:
        assert isinstance(input, SparseConvTensor)
        feats, h, m = input.features, self.heads, self.kv_heads
        if self.inv_freq.device != feats.device:
            self.inv_freq = self.inv_freq.to(feats.device)
        rows, sites, back = feats, input.indices, None
        if input.batch_size > 1 and not self.grouped:
            order = torch.argsort(sites[:, 0], stable=True)
            back = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=order.device))
            rows, sites = feats.index_select(0, order), sites.index_select(0, order)
        qkv = self.qkv(self.norm(rows)).unflatten(1, (h + 2 * m, self.dim))
        q, k, v = qkv.split([h, m, m], 1)
        q, k = qk_norm_rotary(q, k, sites[:, 1:], self.inv_freq, self.sections, self.q_weight, self.k_weight,
                              self.eps)
        out = packed_attention(q, k, v, sample_offsets(sites, input.batch_size), causal=self.causal)
        out = self.proj(out.flatten(1)).to(feats.dtype)
        if back is not None:
            out = out.index_select(0, back)
        if self.training and self.dropout > 0:
            seed = torch.randint(-(1 << 63), (1 << 63) - 1, (2,), device=feats.device)
            out = residual_dropout(out, feats, self.dropout, seed)
        else:
            out = out + feats
        res = SparseConvTensor(out, input.indices, input.spatial_shape, input.batch_size)
        res.indice_dict = input.indice_dict
        res.grid = input.grid
        return res
