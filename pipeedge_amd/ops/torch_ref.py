"""Plain-PyTorch reference implementations of the framework's compute ops.

These are the numerics ground truth for the HIP/CDNA4 kernels in
``pipeedge_amd/ops/hip`` (GPU tests compare the kernels against this module
run in fp32) and the execution path on CPU, where the reference framework ran
its shards eagerly through HF modules (reference vit.py:55-70, bert.py:41-52).

Weight layout convention (MI355X-native): all linear weights are stored
``[N, K]`` (out-features x in-features, the torch.nn.Linear layout). This is
the MFMA-optimal operand layout on gfx950: both GEMM operands are then
k-contiguous per row, so A- and B-fragments alike stage through LDS with
16-B `global_load_lds` pieces and read back as single `ds_read_b128`s
(cdna_hip_programming.md section 5).
"""
import math
from typing import Dict, List, Optional, Tuple

import torch
from torch import Tensor


def layernorm(x: Tensor, weight: Tensor, bias: Tensor, eps: float = 1e-6) -> Tensor:
    """LayerNorm over the last dim."""
    return torch.nn.functional.layer_norm(x, (x.shape[-1],), weight, bias, eps)


def add_layernorm(x: Tensor, residual: Tensor, weight: Tensor, bias: Tensor,
                  eps: float = 1e-6) -> Tensor:
    """Fused (x + residual) -> LayerNorm (BERT post-LN pattern)."""
    return layernorm(x + residual, weight, bias, eps)


def linear(x: Tensor, weight_nk: Tensor, bias: Optional[Tensor] = None,
           act: Optional[str] = None, residual: Optional[Tensor] = None) -> Tensor:
    """GEMM with optionally fused bias + activation + residual add.

    ``weight_nk`` is ``[N, K]``; ``y = act(x @ w.T + b) + residual``.
    """
    y = x.matmul(weight_nk.t())
    if bias is not None:
        y = y + bias
    if act == "gelu":
        y = torch.nn.functional.gelu(y)
    elif act == "tanh":
        y = torch.tanh(y)
    elif act is not None:
        raise ValueError(f"unknown activation: {act}")
    if residual is not None:
        y = y + residual
    return y


def attention_core(q: Tensor, k: Tensor, v: Tensor, scale: Optional[float] = None,
                   attn_mask: Optional[Tensor] = None) -> Tensor:
    """softmax(q @ k^T * scale + mask) @ v over ``[B, H, S, D]`` inputs."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    scores = torch.matmul(q, k.transpose(-1, -2)) * scale
    if attn_mask is not None:
        scores = scores + attn_mask
    probs = torch.softmax(scores, dim=-1)
    return torch.matmul(probs, v)


def qkv_attention(qkv: Tensor, num_heads: int, scale: Optional[float] = None,
                  attn_mask: Optional[Tensor] = None) -> Tensor:
    """Multi-head attention over a packed ``[B, S, 3*D]`` QKV projection.

    Columns of the last dim are ``[q | k | v]``. Returns the merged-head
    context ``[B, S, D]``. This is the layout the fused HIP attention kernel
    consumes directly (no permute kernels on GPU).
    """
    b, s, three_d = qkv.shape
    d = three_d // 3
    dh = d // num_heads
    q, k, v = qkv.split(d, dim=-1)

    def _heads(t):
        return t.reshape(b, s, num_heads, dh).permute(0, 2, 1, 3)

    if attn_mask is not None and attn_mask.dim() == 2:
        # [B, S] per-kpos additive mask (the HIP kernel's contract):
        # broadcast over heads and query rows
        attn_mask = attn_mask.reshape(b, 1, 1, s)
    ctx = attention_core(_heads(q), _heads(k), _heads(v), scale, attn_mask)
    return ctx.permute(0, 2, 1, 3).reshape(b, s, d)


def embed_finish(x: Tensor, prefix: Tensor, pos: Tensor) -> Tensor:
    """out[b, s] = (prefix[s] if s < T else x[b, s-T]) + pos[s]."""
    b = x.shape[0]
    pre = prefix.unsqueeze(0).expand(b, -1, -1).to(x.dtype)
    return torch.cat((pre, x), dim=1) + pos.to(x.dtype)


def patchify(pixels: Tensor, patch_size: int) -> Tensor:
    """[B, C, H, W] -> [B, num_patches, C*P*P] for non-overlapping P x P patches.

    The inner layout per patch is (C, Ph, Pw), matching a Conv2d(P, stride=P)
    kernel flattened as [C*P*P, D].
    """
    b, c, h, w = pixels.shape
    p = patch_size
    x = pixels.reshape(b, c, h // p, p, w // p, p)
    x = x.permute(0, 2, 4, 1, 3, 5)  # B, H/p, W/p, C, p, p
    return x.reshape(b, (h // p) * (w // p), c * p * p)


def _check_inference(op: str, *tensors: Optional[Tensor]):
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{op}: inference only, an input requires a gradient")


def _reaches(steps: List[Tuple[int, int, int]], target: int, reach: int,
             nonzero: bool, tries: List[int]) -> bool:
    """Whether ``target`` less a sum of number x stride, with each number in
    its limits, can lie within ``reach`` of zero; ``nonzero``: with a number
    other than zero. ``steps`` by falling stride; more than ``tries`` is yes."""
    tries[0] -= 1
    if tries[0] < 0:
        return True
    if not steps:
        return not nonzero and abs(target) <= reach
    (stride, low, high), rest = steps[0], steps[1:]
    rest_low = sum(lo * s for s, lo, _ in rest) - reach
    rest_high = sum(hi * s for s, _, hi in rest) + reach
    first = max(low, -((rest_high - target) // stride))
    last = min(high, (target - rest_low) // stride)
    return any(_reaches(rest, target - n * stride, reach,
                        nonzero and n == 0, tries)
               for n in range(first, last + 1))


def _overlaps_itself(x: Tensor, width: int) -> bool:
    """Whether two heads of ``x`` share any of ``width`` adjacent columns."""
    dims = [(st, n) for st, n in zip(x.stride()[:-1], x.shape[:-1]) if n != 1]
    if any(n == 0 for _, n in dims):
        return False
    if any(st == 0 for st, _ in dims):
        return True
    steps = sorted(((st, 1 - n, n - 1) for st, n in dims), reverse=True)
    return _reaches(steps, 0, width - 1, True, [1 << 14])


def _overlap(q: Tensor, k: Tensor, width: int) -> bool:
    """The same for a head of ``q`` and one of ``k``."""
    size = q.element_size()
    limits: Dict[int, List[int]] = {}
    for x, at, sign in ((q, 1, 1), (k, 0, -1)):
        if 0 in x.shape[:-1]:
            return False
        for st, n in zip(x.stride()[:-1], x.shape[:-1]):
            if n > 1:
                limits.setdefault(st * size, [0, 0])[at] += sign * (n - 1)
    steps = sorted(((st, lo, hi) for st, (lo, hi) in limits.items()),
                   reverse=True)
    return _reaches(steps, k.data_ptr() - q.data_ptr(), width * size - 1,
                    False, [1 << 14])


def check_rotary(q: Tensor, positions: Tensor, freqs: Tensor,
                 k: Optional[Tensor], offset: int, in_place: bool):
    """The argument checks of the rotary kernel, for the CPU path."""
    if q.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError("rotary: q must be bfloat16, float16 or float32")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("rotary: positions must be int32 or int64")
    if freqs.dtype != torch.float64 or freqs.dim() != 1:
        raise TypeError("rotary: freqs must be a float64 vector")
    if k is not None and k.dtype != q.dtype:
        raise TypeError("rotary: q and k must have one type")
    if any(t is not None and t.device != q.device
           for t in (positions, freqs, k)):
        raise ValueError("rotary: tensors on different devices")
    _check_inference("rotary", q, k, freqs)
    for name, x in (("q", q), ("k", k)):
        if x is None:
            continue
        if x.dim() < 2:
            raise ValueError(f"rotary: {name} must be [.., heads, dim]")
        if x.shape[-1] > 1 and x.stride(-1) != 1:
            raise ValueError(f"rotary: {name} must be contiguous in its "
                             "last dimension")
    pairs, dim = freqs.numel(), q.shape[-1]
    if pairs < 1 or offset < 0 or offset + 2 * pairs > dim:
        raise ValueError(f"rotary: columns {offset} to {offset + 2 * pairs} "
                         f"do not fit a head of {dim}")
    if pairs > 1024:
        raise ValueError("rotary: more than 2048 rotated columns")
    if positions.shape != q.shape[:-2]:
        raise ValueError("rotary: positions must be one a token, shape "
                         f"{list(q.shape[:-2])}, got {list(positions.shape)}")
    if k is not None:
        if k.dim() != q.dim() or k.shape[-1] != dim \
                or k.shape[:-2] != q.shape[:-2]:
            raise ValueError("rotary: k must match q except in its heads")
    if in_place:
        if any(t is not None and _overlaps_itself(t, 2 * pairs)
               for t in (q, k)):
            raise ValueError("rotary_: a tensor overlaps itself")
        if k is not None and _overlap(q, k, 2 * pairs):
            raise ValueError("rotary_: q and k overlap")


def rotary(q: Tensor, positions: Tensor, freqs: Tensor,
           k: Optional[Tensor] = None, interleaved: bool = False,
           offset: int = 0, inverse: bool = False, scale: float = 1.0,
           in_place: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """Turn column pairs by ``position * freqs`` (angles in 64 bits)."""
    check_rotary(q, positions, freqs, k, offset, in_place)
    angle = positions.to(torch.float64).unsqueeze(-1) * freqs
    if inverse:
        angle = -angle
    cos = (torch.cos(angle) * scale).float().unsqueeze(-2)
    sin = (torch.sin(angle) * scale).float().unsqueeze(-2)
    width = 2 * freqs.numel()

    def _turn(x):
        part = x[..., offset:offset + width].float()
        a, b = (part[..., 0::2], part[..., 1::2]) if interleaved \
            else part.chunk(2, dim=-1)
        turned = (a * cos - b * sin, b * cos + a * sin)
        turned = torch.stack(turned, dim=-1).flatten(-2) if interleaved \
            else torch.cat(turned, dim=-1)
        out = x if in_place else x.clone(
            memory_format=torch.contiguous_format)
        out[..., offset:offset + width] = turned.to(x.dtype)
        return out

    return _turn(q), None if k is None else _turn(k)


def _softmax_seen(scores: Tensor, seen: Tensor) -> Tensor:
    """Softmax over the seen scores; a row that sees nothing gets zeros."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - top.masked_fill(top == float("-inf"), 0.0))
    total = weight.sum(-1, keepdim=True)
    return weight / total.masked_fill(total == 0.0, 1.0)


def _check_scale(op: str, scale: float):
    """A scale that 32 bits hold in powers of two, as the kernels take it."""
    limits = torch.finfo(torch.float32)
    if not limits.tiny <= scale * math.log2(math.e) <= limits.max:
        raise ValueError(f"{op}: scale must be positive and in the range of "
                         "32 bits")


def check_latent_attention(q: Tensor, kv: Tensor, k_rope: Tensor,
                           scale: float, lengths: Optional[Tensor],
                           past: Optional[Tensor]):
    """The argument checks of the latent attention kernel (CPU path)."""
    op = "latent_attention"
    if not (q.dtype == kv.dtype == k_rope.dtype):
        raise TypeError(f"{op}: q, kv and k_rope must have one type")
    if any(t is not None and t.device != q.device
           for t in (kv, k_rope, lengths, past)):
        raise ValueError(f"{op}: tensors on different devices")
    _check_inference(op, q, kv, k_rope)
    if q.dim() != 4 or kv.dim() != 4 or k_rope.dim() != 3:
        raise ValueError(f"{op}: q and kv must be [B, S, H, D], "
                         "k_rope [B, S, D]")
    b, sq, h, _ = q.shape
    sk, nope = kv.shape[1], q.shape[3] - k_rope.shape[2]
    if nope not in (64, 128) or k_rope.shape[2] not in (32, 64) \
            or kv.shape[3] != 2 * nope:
        raise ValueError(
            f"{op}: head parts must be 64 or 128 plain and 32 or 64 rotary "
            "columns with as many values as plain ones, got q "
            f"{q.shape[3]}, kv {kv.shape[3]}, k_rope {k_rope.shape[2]}")
    if kv.shape[:3] != (b, sk, h) or k_rope.shape[:2] != (b, sk):
        raise ValueError(f"{op}: q {list(q.shape)}, kv {list(kv.shape)} and "
                         f"k_rope {list(k_rope.shape)} do not match")
    _check_scale(op, scale)
    for t in (lengths, past):
        if t is None:
            continue
        if t.dtype != torch.int32:
            raise TypeError(f"{op}: lengths and past must be int32")
        if t.shape != (b,):
            raise ValueError(f"{op}: lengths and past must be one a sequence")
    if lengths is not None and past is None and sq != sk:
        raise ValueError(f"{op}: lengths with fewer or more queries than "
                         "keys need past")


def latent_attention(q: Tensor, kv: Tensor, k_rope: Tensor, scale: float,
                     causal: bool = False, lengths: Optional[Tensor] = None,
                     past: Optional[Tensor] = None) -> Tensor:
    """Attention with keys ``[kv[.., :DN] | k_rope]`` and values
    ``kv[.., DN:]``; the rotary key part is shared by all heads."""
    check_latent_attention(q, kv, k_rope, scale, lengths, past)
    b, sq, h, _ = q.shape
    sk, nope = kv.shape[1], q.shape[3] - k_rope.shape[2]
    if sk == 0:
        return q.new_zeros(b, sq, h, nope)
    length = torch.full((b, 1), sk, dtype=torch.int64, device=q.device) \
        if lengths is None else lengths.long().clamp(0, sk).reshape(b, 1)
    first = torch.full_like(length, sk - sq) if past is None \
        else past.long().reshape(b, 1)
    at = first + torch.arange(sq, device=q.device)
    key = torch.arange(sk, device=q.device)
    seen = ((at >= 0) & (at < length)).unsqueeze(-1) \
        & (key < length).unsqueeze(1)
    if causal:
        seen = seen & (key <= at.unsqueeze(-1))
    # what lies behind a sequence never reaches its sums
    inside = (key < length).reshape(b, 1, sk, 1)
    heads = kv.float().transpose(1, 2).masked_fill(~inside, 0.0)
    rope = k_rope.float().unsqueeze(1).masked_fill(~inside, 0.0)
    full = torch.cat((heads[..., :nope], rope.expand(-1, h, -1, -1)), dim=-1)
    scores = torch.matmul(q.float().transpose(1, 2),
                          full.transpose(-1, -2)) * scale
    weight = _softmax_seen(scores, seen.unsqueeze(1))
    out = torch.matmul(weight, heads[..., nope:].contiguous())
    # also where zero weights met values that are not finite
    out = out.masked_fill(~seen.any(-1).reshape(b, 1, sq, 1), 0.0)
    return out.transpose(1, 2).contiguous().to(q.dtype)


def check_latent_cache_attention(q: Tensor, cache: Tensor,
                                 block_table: Tensor, lengths: Tensor,
                                 latent_dim: int, scale: float):
    """The argument checks of the latent cache kernel (CPU path)."""
    op = "latent_cache_attention"
    if q.dtype != cache.dtype:
        raise TypeError(f"{op}: q and cache must have one type")
    if block_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError(f"{op}: block_table and lengths must be int32")
    if any(t.device != q.device for t in (cache, block_table, lengths)):
        raise ValueError(f"{op}: tensors on different devices")
    _check_inference(op, q, cache)
    if q.dim() != 4 or cache.dim() != 3 or q.shape[3] != cache.shape[2]:
        raise ValueError(f"{op}: q must be [B, Sq, H, D] and cache [pages, "
                         f"page size, D], got {list(q.shape)} and "
                         f"{list(cache.shape)}")
    b, rope = q.shape[0], q.shape[3] - latent_dim
    if latent_dim not in (256, 512) or rope not in (32, 64):
        raise ValueError(f"{op}: rows must be 256 or 512 latent and 32 or 64 "
                         f"rotary columns, got {latent_dim} and {rope}")
    if block_table.dim() != 2 or block_table.shape[0] != b \
            or lengths.shape != (b,):
        raise ValueError(f"{op}: block_table must be [B, P] and lengths [B]")
    _check_scale(op, scale)


def latent_cache_attention(q: Tensor, cache: Tensor, block_table: Tensor,
                           lengths: Tensor, latent_dim: int,
                           scale: float) -> Tensor:
    """Every head of the last ``Sq`` tokens attends to the cached rows, whose
    first ``latent_dim`` columns are also the values."""
    check_latent_cache_attention(q, cache, block_table, lengths, latent_dim,
                                 scale)
    b, sq, h, width = q.shape
    page = cache.shape[1]
    out = q.new_zeros(b, sq, h, latent_dim)
    for i in range(b):
        n = int(lengths[i])
        if n <= 0 or out.numel() == 0:
            continue
        place = torch.arange(n, device=q.device)
        if page == 0 or n > page * block_table.shape[1]:
            out[i] = float("nan")
            continue
        pages = block_table[i].long()[place // page]
        if ((pages < 0) | (pages >= cache.shape[0])).any():
            out[i] = float("nan")
            continue
        tokens = cache[pages, place % page].float()
        scores = torch.matmul(q[i].float().contiguous(), tokens.t()) * scale
        at = n - sq + torch.arange(sq, device=q.device)
        seen = place <= at.reshape(sq, 1, 1)
        weight = _softmax_seen(scores, seen.expand(sq, h, n))
        out[i] = torch.matmul(weight, tokens[:, :latent_dim]).to(q.dtype)
        # also where zero weights met values that are not finite
        out[i, at < 0] = 0.0
    return out


def check_adapter_linear(x: Tensor, weight: Tensor, down: Tensor, up: Tensor,
                         ids: Tensor, bias: Optional[Tensor],
                         residual: Optional[Tensor],
                         scales: Optional[Tensor]):
    """The argument checks of the adapter projection (CPU path)."""
    op = "adapter_linear"
    if any(t is not None and t.dtype != x.dtype
           for t in (weight, down, up, bias, residual)):
        raise TypeError(f"{op}: x, weight, down, up, bias and residual must "
                        "have one type")
    if ids.dtype != torch.int32:
        raise TypeError(f"{op}: ids must be int32")
    if scales is not None and scales.dtype != torch.float32:
        raise TypeError(f"{op}: scales must be float32")
    tensors = (weight, down, up, ids, bias, residual, scales)
    if any(t is not None and t.device != x.device for t in tensors):
        raise ValueError(f"{op}: tensors on different devices")
    _check_inference(op, x, *tensors)
    if x.dim() < 1 or weight.dim() != 2 or down.dim() != 3 or up.dim() != 3:
        raise ValueError(f"{op}: x must be [.., K], weight [N, K], "
                         "down [n, r, K] and up [n, N, r]")
    n, r, k = down.shape
    if x.shape[-1] != k or weight.shape[1] != k \
            or up.shape != (n, weight.shape[0], r):
        raise ValueError(f"{op}: x {list(x.shape)}, weight "
                         f"{list(weight.shape)}, down {list(down.shape)} and "
                         f"up {list(up.shape)} do not match")
    if k == 0:
        raise ValueError(f"{op}: no inner columns, or too many rows")
    if r > 256:
        raise ValueError(f"{op}: rank above 256")
    if ids.shape != x.shape[:-1] and not (
            x.dim() >= 2 and ids.shape == x.shape[:1]):
        raise ValueError(f"{op}: ids must be one a row or one an item of the "
                         f"batch, got {list(ids.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"{op}: bias must be [N]")
    if residual is not None \
            and residual.shape != x.shape[:-1] + weight.shape[:1]:
        raise ValueError(f"{op}: residual must have the output's shape")
    if scales is not None and scales.shape != (n,):
        raise ValueError(f"{op}: scales must be [n]")


def adapter_linear(x: Tensor, weight: Tensor, down: Tensor, up: Tensor,
                   ids: Tensor, bias: Optional[Tensor] = None,
                   act: Optional[str] = None,
                   residual: Optional[Tensor] = None,
                   scales: Optional[Tensor] = None) -> Tensor:
    """``linear`` plus ``scales[i] * (x @ down[i].T) @ up[i].T`` before the
    activation, with i the row's id; ids outside the stack have no adapter."""
    check_adapter_linear(x, weight, down, up, ids, bias, residual, scales)
    rows = x.float().reshape(-1, x.shape[-1])
    per = rows.shape[0] // max(ids.numel(), 1)
    row_ids = ids.reshape(-1).repeat_interleave(per)
    y = rows @ weight.float().t()
    for i in row_ids.unique().tolist():
        if not 0 <= i < down.shape[0]:
            continue
        mine = row_ids == i
        inner = rows[mine] @ down[i].float().t()
        if scales is not None:
            inner = inner * scales[i]
        y[mine] += inner @ up[i].float().t()
    if bias is not None:
        y = y + bias.float()
    if act == "gelu":
        # through erfc, which keeps its digits where 1 + erf cancels
        y = y * (0.5 * torch.special.erfc(y * -math.sqrt(0.5)))
    elif act == "tanh":
        y = torch.tanh(y)
    elif act is not None:
        raise ValueError(f"unknown activation: {act}")
    y = y.reshape(*x.shape[:-1], weight.shape[0])
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)
