"""Compute-op dispatch: hand-written CDNA4 HIP kernels on GPU, torch on CPU.

Every model shard calls through this module. On a CUDA (ROCm) device the ops
MUST run on the in-tree HIP extension (``pipeedge_amd/ops/hip``); if the
extension is missing or an op is unimplemented, the call raises instead of
silently falling back to eager PyTorch. Set ``PIPEEDGE_AMD_FORCE_TORCH=1`` to
explicitly opt into the eager path on GPU (used for A/B comparisons only).

The reference framework has no kernels at all - its
hot path is eager HF modules; this module is where the MI355X build replaces
them.
"""
import math
import os
from typing import Optional

import torch
from torch import Tensor

from . import torch_ref

_hip = None          # the loaded extension module, or None
_hip_load_err = None  # exception from the load attempt, if any
_hip_tried = False


def _load_hip():
    global _hip, _hip_load_err, _hip_tried
    if _hip_tried:
        return _hip
    _hip_tried = True
    try:
        from . import hip_loader
        _hip = hip_loader.load()
    except Exception as exc:  # noqa: BLE001 - report it at use time
        _hip_load_err = exc
        _hip = None
    return _hip


def force_torch() -> bool:
    return os.environ.get("PIPEEDGE_AMD_FORCE_TORCH", "0") == "1"


def _use_hip(x: Tensor) -> bool:
    """HIP-kernel path iff tensor is on GPU and the eager escape is not set."""
    if not x.is_cuda or force_torch():
        return False
    if _load_hip() is None:
        raise RuntimeError(
            "pipeedge_amd HIP extension is required for GPU execution but "
            f"failed to load: {_hip_load_err!r}. Build it with "
            "`python setup.py build_ext --inplace` (or __graft_entry__.build()); "
            "set PIPEEDGE_AMD_FORCE_TORCH=1 only to explicitly run eager torch."
        )
    return True


def hip_available() -> bool:
    return _load_hip() is not None


def layernorm(x: Tensor, weight: Tensor, bias: Tensor, eps: float = 1e-6) -> Tensor:
    if _use_hip(x):
        return _hip.layernorm(x, weight, bias, eps)
    return torch_ref.layernorm(x, weight, bias, eps)


def add_layernorm(x: Tensor, residual: Tensor, weight: Tensor, bias: Tensor,
                  eps: float = 1e-6) -> Tensor:
    if _use_hip(x):
        return _hip.add_layernorm(x, residual, weight, bias, eps)
    return torch_ref.add_layernorm(x, residual, weight, bias, eps)


_ACT_CODE = {None: 0, "gelu": 1, "tanh": 2}


def linear(x: Tensor, weight_nk: Tensor, bias: Optional[Tensor] = None,
           act: Optional[str] = None, residual: Optional[Tensor] = None,
           want_stats: bool = False):
    """GEMM + fused epilogue. With ``want_stats`` (GPU path) also returns
    per-row partial (sum, sumsq) of the OUTPUT, f32 [rows, parts, 2] -
    written without atomics by each column block and summed by the next
    folded-LN GEMM (see ln_linear)."""
    if _use_hip(x):
        out, stats = _hip.linear(x, weight_nk, bias, _ACT_CODE[act],
                                 residual, 0, None, None, None, 1e-12,
                                 want_stats)
        return (out, stats) if want_stats else out
    out = torch_ref.linear(x, weight_nk, bias, act, residual)
    return (out, None) if want_stats else out


def ln_stats(x: Tensor) -> Tensor:
    """Per-row (sum, sumsq) over the last dim, f32 [rows, 1, 2]."""
    if _use_hip(x):
        return _hip.ln_stats(x.reshape(-1, x.shape[-1]))
    xf = x.reshape(-1, x.shape[-1]).float()
    return torch.stack((xf.sum(-1), (xf * xf).sum(-1)), dim=-1).unsqueeze(1)


def make_ln_fold(weight_nk: Tensor, ln_weight: Tensor, ln_bias: Tensor):
    """Precompute the folded-LN GEMM operands (GPU):
    W' = W * ln_w (per-K column), s[n] = sum_k W'[n,k], c[n] = W @ ln_b.

    Because LayerNorm is affine per row,
      LN(x) @ W^T = r*(x @ W'^T) - r*mu*s + c
    with per-row mean mu and inv-std r - so the GEMM runs on RAW x and the
    LN collapses into the epilogue (no standalone LN kernel, no extra
    activation pass)."""
    w_p = (weight_nk.float() * ln_weight.float()).to(weight_nk.dtype)         .contiguous()
    s = w_p.float().sum(dim=1).contiguous()
    c = (weight_nk.float() @ ln_bias.float()).contiguous()
    return (w_p, s, c)


def ln_linear(x: Tensor, ln_weight: Tensor, ln_bias: Tensor, eps: float,
              weight_nk: Tensor, bias: Optional[Tensor] = None,
              act: Optional[str] = None, residual: Optional[Tensor] = None,
              stats: Optional[Tensor] = None, fused=None) -> Tensor:
    """LayerNorm -> Linear; folded into ONE GEMM on GPU (see make_ln_fold).

    ``stats``: per-row (sum, sumsq) of x if already known (emitted by the
    producing GEMM); computed by a ln_stats kernel otherwise."""
    if _use_hip(x):
        assert fused is not None, "ln_linear GPU path needs make_ln_fold(...)"
        w_p, s, c = fused
        if stats is None:
            stats = _hip.ln_stats(x.reshape(-1, x.shape[-1]))
        out, _ = _hip.linear(x, w_p, bias, _ACT_CODE[act], residual, 0,
                             stats, s, c, eps, False)
        return out
    y = torch_ref.layernorm(x, ln_weight, ln_bias, eps)
    return torch_ref.linear(y, weight_nk, bias, act, residual)


def fused_ln_active(x: Tensor) -> bool:
    """Whether the folded-LN GEMM path is used for this tensor.

    Default OFF: end-to-end A/B on MI355X measured the folded path at net
    ~parity-to-slower vs the standalone LN kernels (the LN savings are offset
    by partial-stats traffic in the consumer epilogues); enable with
    PIPEEDGE_FOLDED_LN=1 to experiment."""
    return (x.is_cuda and not force_torch()
            and os.environ.get("PIPEEDGE_FOLDED_LN", "0") == "1")


def attention_core(q: Tensor, k: Tensor, v: Tensor, scale: Optional[float] = None,
                   attn_mask: Optional[Tensor] = None) -> Tensor:
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if _use_hip(q):
        return _hip.attention(q, k, v, scale, attn_mask)
    return torch_ref.attention_core(q, k, v, scale, attn_mask)


def qkv_attention(qkv: Tensor, num_heads: int, scale: Optional[float] = None,
                  attn_mask: Optional[Tensor] = None) -> Tensor:
    if scale is None:
        scale = 1.0 / math.sqrt(qkv.shape[-1] // 3 // num_heads)
    if _use_hip(qkv):
        return _hip.qkv_attention(qkv, num_heads, scale, attn_mask)
    return torch_ref.qkv_attention(qkv, num_heads, scale, attn_mask)


def patchify(pixels: Tensor, patch_size: int) -> Tensor:
    if _use_hip(pixels):
        return _hip.patchify(pixels, patch_size)
    return torch_ref.patchify(pixels, patch_size)


def embed_finish(x: Tensor, prefix: Tensor, pos: Tensor) -> Tensor:
    """Prepend prefix token rows (cls / cls+dist) and add position
    embeddings: out[b, s] = (prefix[s] if s < T else x[b, s-T]) + pos[s]."""
    if _use_hip(x):
        return _hip.embed_finish(x, prefix, pos)
    return torch_ref.embed_finish(x, prefix, pos)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0,
                       scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None,
                       low_turns: float = 1.0, high_turns: float = 32.0,
                       device=None) -> Tensor:
    """Angle per position of each of ``rotary_dim / 2`` column pairs, float64.

    Unscaled f_i = base^(-2i / rotary_dim). ``scaling`` stretches a model
    trained for ``original_length`` positions to ``factor`` times as many:

    - "linear": every f_i / factor;
    - "base": base * factor^(rotary_dim / (rotary_dim - 2)) for base, which
      keeps the first frequency and divides the last by ``factor``;
    - "ramp": pairs that turn at least ``high_turns`` times within
      ``original_length`` keep f_i, those below ``low_turns`` get
      f_i / factor, between them the two are mixed linearly in the turns.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_frequencies: rotary_dim must be even, "
                         f"got {rotary_dim}")
    if not (base > 0.0 and factor > 0.0):
        raise ValueError("rotary_frequencies: base and factor must be "
                         "positive")
    if scaling not in (None, "linear", "base", "ramp"):
        raise ValueError(f"rotary_frequencies: unknown scaling: {scaling}")
    if scaling == "base":
        base = base * factor ** (rotary_dim / max(rotary_dim - 2, 1))
    index = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    freqs = base ** (-index / rotary_dim)
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "ramp":
        if original_length is None or not high_turns > low_turns:
            raise ValueError("rotary_frequencies: ramp needs original_length "
                             "and high_turns > low_turns")
        turns = original_length * freqs / (2.0 * math.pi)
        keep = ((turns - low_turns) / (high_turns - low_turns)).clamp(0., 1.)
        freqs = freqs * keep + freqs / factor * (1.0 - keep)
    return freqs.to(device)


def rotary(q: Tensor, positions: Tensor, freqs: Tensor,
           k: Optional[Tensor] = None, *, interleaved: bool = False,
           offset: int = 0, inverse: bool = False, scale: float = 1.0):
    """Rotary positions of queries and, in the same launch, keys.

    ``q`` is [.., heads, dim] and ``k`` the same but for its heads, in
    bfloat16, float16 or float32 with any strides but 1 in the last
    dimension; ``positions`` holds one integer a token ([..], any value) and
    ``freqs`` the float64 vector of ``rotary_frequencies``. Columns
    ``offset .. offset + 2 * len(freqs)`` of each head are turned, with the
    pairs half that width apart or, ``interleaved``, next to each other; the
    rest is copied. ``scale`` multiplies the turned columns. ``inverse`` turns
    the other way, which is also the gradient. Returns new tensors: the turned
    ``q``, or ``(q, k)``."""
    run = _hip.rotary if _use_hip(q) else torch_ref.rotary
    out = run(q, positions, freqs, k, interleaved, offset, inverse, scale,
              False)
    return out[0] if k is None else out


def rotary_(q: Tensor, positions: Tensor, freqs: Tensor,
            k: Optional[Tensor] = None, *, interleaved: bool = False,
            offset: int = 0, inverse: bool = False, scale: float = 1.0):
    """``rotary`` in place, for views of a larger tensor: the first 2H of the
    3H heads of a packed qkv, the rotary columns of each head, rows of a
    cache. The turned columns of two heads, of ``q``, of ``k`` or of both, must
    not overlap. Five and more dimensions whose leading ones are not one in
    memory take a launch for each of the first. Returns its arguments."""
    run = _hip.rotary if _use_hip(q) else torch_ref.rotary
    out = run(q, positions, freqs, k, interleaved, offset, inverse, scale,
              True)
    return out[0] if k is None else out


def latent_attention(q: Tensor, kv: Tensor, k_rope: Tensor, *,
                     scale: Optional[float] = None, causal: bool = False,
                     lengths: Optional[Tensor] = None,
                     past: Optional[Tensor] = None) -> Tensor:
    """Attention over latent vectors in expanded form, for prompts.

    ``q`` [B, Sq, H, DN + DR] holds plain and rotated columns, ``kv``
    [B, Sk, H, 2 DN] the keys' plain columns and the values of each head (the
    latent vectors' up-projection, as ``linear`` writes it) and ``k_rope``
    [B, Sk, DR] the rotated key columns that all heads share; DN is 64 or 128,
    DR 32 or 64, all bfloat16 or float16 (any strides, tokens less than 2^24
    elements apart). Returns [B, Sq, H, DN];
    ``scale`` is 1 / sqrt(DN + DR) unless given.

    ``lengths`` (int32 [B]) are the valid keys of each padded sequence, ``past``
    (int32 [B]) the position of its first query, Sk - Sq if both are absent; a
    ``causal`` query sees no key behind its own position. Queries whose
    position is outside their sequence are padding and come back zero; keys
    and values behind a sequence may hold anything. A value inside it that is
    not finite may also reach queries that do not see it, whose zero weight it
    is multiplied with; keys reach only queries that see them."""
    if scale is None:
        scale = 1.0 / math.sqrt(max(q.shape[-1], 1))
    run = _hip.latent_attention if _use_hip(q) else torch_ref.latent_attention
    return run(q, kv, k_rope, scale, causal, lengths, past)


def latent_cache_attention(q: Tensor, cache: Tensor, block_table: Tensor,
                           lengths: Tensor, *, latent_dim: int,
                           scale: float) -> Tensor:
    """Attention over latent vectors in absorbed form, for single tokens.

    ``cache`` [pages, page size, R + DR] holds a latent vector and the rotated
    shared key columns of each token (R = ``latent_dim`` 256 or 512, DR 32 or
    64, bfloat16 or float16, rows contiguous and at multiples of 16 bytes, any
    page size), ``block_table`` (int32 [B, P]) the pages of each sequence and
    ``lengths`` (int32 [B]) its tokens, the ``Sq`` newest of which are the
    queries. ``q`` [B, Sq, H, R + DR] are their heads with the key projection
    absorbed, [q_nope W_uk | q_rope]; ``scale`` is that of the expanded form.
    Returns [B, Sq, H, R], the weighted latent vectors, to which the value
    projection is applied afterwards. Query i sees tokens up to its own
    position, lengths - Sq + i; one before the start comes back zero, as does
    an empty sequence. Table entries behind a sequence are not read. A length
    that the table cannot hold, or a page number that the cache (of one page
    at least) does not have, makes that sequence's outputs NaN. A latent value
    that is not finite may also reach the call's earlier queries, whose zero
    weight it is multiplied with, but no other sequence. All heads and queries of a sequence
    share one pass over its tokens; a few queries at a time are what it is
    made for."""
    run = _hip.latent_cache_attention if _use_hip(q) \
        else torch_ref.latent_cache_attention
    return run(q, cache, block_table, lengths, latent_dim, scale)


def adapter_linear(x: Tensor, weight_nk: Tensor, down: Tensor, up: Tensor,
                   ids: Tensor, bias: Optional[Tensor] = None,
                   act: Optional[str] = None,
                   residual: Optional[Tensor] = None,
                   scales: Optional[Tensor] = None) -> Tensor:
    """``linear`` beside low-rank adapters of many requests, for a batch whose
    items belong to different tenants of one set of weights:

      y = act(x W^T + bias + scales[i] (x down[i]^T) up[i]^T) + residual

    ``down`` [n, r, K] and ``up`` [n, N, r] stack the adapters (r <= 256);
    ``ids`` (int32) gives each item of the batch ([B]) or each row
    (x.shape[:-1]) its adapter, and any value outside 0 .. n-1, such as -1,
    none. ``scales`` (float32 [n]) defaults to ones. bfloat16 on the GPU. A
    row is touched by no adapter but its own, whatever the others hold."""
    if act not in _ACT_CODE:
        raise ValueError(f"unknown activation: {act}")
    if _use_hip(x):
        return _hip.adapter_linear(x, weight_nk, down, up, ids, bias,
                                   _ACT_CODE[act], residual, scales)
    return torch_ref.adapter_linear(x, weight_nk, down, up, ids, bias, act,
                                    residual, scales)
