"""Latent attention against its definition in 64 bits: expanded form over
padded prompts and absorbed form over a paged cache. Every case runs on the
CPU path; with a GPU the same cases run on the HIP kernels."""
import math

import pytest
import torch

from pipeedge_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float16]


def attend(q, keys, values, scale, upto):
    """One head in 64 bits; query i sees the first upto[i] keys. Also returns
    the same sum over absolute values, which the tolerance needs."""
    q, keys, values = q.double(), keys.double(), values.double()
    s = q @ keys.t() * scale
    hidden = torch.arange(keys.shape[0]) >= upto.unsqueeze(-1)
    s = s.masked_fill(hidden, -math.inf)
    p = torch.softmax(s, -1)
    p[upto == 0] = 0.0
    # a score's fp32 sum is off by at most n steps of the absolute products
    # (exact in fp32), which turns its weight by that much
    size = (q.abs() @ keys.abs().t() * scale).masked_fill(hidden, 0.0)
    drift = size.amax(-1) * q.shape[-1] * 2.0 ** -24
    return p @ values, p @ values.abs(), drift


def check(out, ref, size, drift, dtype):
    """Weights are rounded to the type once, half a step of eps each, and so
    is the result. Everything else is in fp32: the scores (drift, for both a
    weight and the sum), the exponential and scaling (2^-19 together), the
    sums over the tokens (2^-18)."""
    half = torch.finfo(dtype).eps / 2
    out = out.double().cpu()
    bound = ref.abs() * half + size * (
        half + 2.0 * drift.unsqueeze(-1) + 2.0 ** -17) + 1e-7
    assert torch.isfinite(out).all()
    assert ((out - ref).abs() <= bound).all(), \
        ((out - ref).abs() / bound).max()


def expanded_exact(q, kv, k_rope, scale, causal, lengths, past):
    b, sq, h, _ = q.shape
    sk, rope = kv.shape[1], k_rope.shape[2]
    nope = q.shape[3] - rope
    q, kv, k_rope = q.cpu(), kv.cpu(), k_rope.cpu()
    ref = torch.zeros(b, sq, h, nope, dtype=torch.float64)
    size, drift = torch.zeros_like(ref), torch.zeros(b, sq, h).double()
    for i in range(b):
        n = sk if lengths is None else int(lengths[i])
        first = sk - sq if past is None else int(past[i])
        at = first + torch.arange(sq)
        upto = (at + 1).clamp(max=n) if causal else torch.full((sq,), n)
        upto = torch.where((at < 0) | (at >= n), 0, upto)
        if n == 0:
            continue
        for j in range(h):
            keys = torch.cat((kv[i, :n, j, :nope], k_rope[i, :n]), -1)
            ref[i, :, j], size[i, :, j], drift[i, :, j] = attend(
                q[i, :, j], keys, kv[i, :n, j, nope:], scale, upto)
    return ref, size, drift


def make_expanded(b, sq, sk, h, nope, rope, dtype, device, seed=0):
    torch.manual_seed(seed + sq + sk)
    q = torch.randn(b, sq, h, nope + rope).to(dtype).to(device)
    kv = torch.randn(b, sk, h, 2 * nope).to(dtype).to(device)
    k_rope = torch.randn(b, sk, rope).to(dtype).to(device)
    return q, kv, k_rope


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,sq,sk,h,nope,rope", [
    (1, 1, 1, 1, 64, 32),
    (2, 37, 37, 4, 64, 32),
    (1, 64, 64, 2, 128, 32),
    (3, 129, 129, 3, 64, 64),
    (1, 200, 200, 2, 128, 64),
    (2, 1, 300, 2, 128, 64),         # one query, many keys
    (1, 70, 331, 2, 64, 64),         # the last queries of a prompt
    (1, 90, 33, 2, 128, 64),         # more queries than keys
])
def test_expanded_matches_exact(device, dtype, causal, b, sq, sk, h, nope,
                                rope):
    q, kv, k_rope = make_expanded(b, sq, sk, h, nope, rope, dtype, device)
    out = ops.latent_attention(q, kv, k_rope, causal=causal)
    assert out.shape == (b, sq, h, nope) and out.dtype == dtype
    check(out, *expanded_exact(q, kv, k_rope, (nope + rope) ** -0.5, causal,
                               None, None), dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sq,sk,lengths,past", [
    (150, 150, [150, 1, 0, 64, 65, 128], None),
    (150, 150, [150, 2, 0, 63, 127, 129], [0, 0, 0, 0, 0, 0]),
    (40, 260, [260, 41, 40, 100, 10, 0], [220, 1, 0, 60, 0, 0]),
    (40, 260, [260, 260, 260, 5, 50, 3], [0, 100, -7, 5, 49, -50]),
])
def test_expanded_padding(device, causal, sq, sk, lengths, past):
    """Rows outside their sequence are zero; the padding holds NaN and
    infinities, which reach nothing."""
    dtype = torch.bfloat16
    q, kv, k_rope = make_expanded(6, sq, sk, 2, 64, 64, dtype, device)
    n = torch.tensor(lengths, dtype=torch.int32)
    p = None if past is None else torch.tensor(past, dtype=torch.int32)
    ref = expanded_exact(q, kv, k_rope, 0.2, causal, n, p)
    for i, length in enumerate(lengths):
        kv[i, length:] = float("nan")
        k_rope[i, length:] = float("inf")
    out = ops.latent_attention(
        q, kv, k_rope, scale=0.2, causal=causal, lengths=n.to(device),
        past=None if p is None else p.to(device))
    check(out, *ref, dtype)


@pytest.mark.parametrize("device", DEVICES)
def test_expanded_strides(device):
    """Views: heads first, part of wider rows, misaligned storage."""
    dtype = torch.float16
    q, kv, k_rope = make_expanded(2, 70, 70, 3, 64, 32, dtype, device)
    want = ops.latent_attention(q, kv, k_rope, causal=True)
    q2 = q.transpose(1, 2).contiguous().transpose(1, 2)
    kv2 = torch.zeros(2, 70, 3, 131, dtype=dtype, device=device)[..., 3:]
    kv2.copy_(kv)
    r2 = torch.zeros(2, 70, 64, dtype=dtype, device=device)[..., 8:40]
    r2.copy_(k_rope)
    r3 = torch.zeros(2, 70, 32, 2, dtype=dtype, device=device)[..., 0]
    r3.copy_(k_rope)
    for args in ((q2, kv, k_rope), (q, kv2, k_rope), (q, kv, r2),
                 (q2, kv2, r3)):
        assert torch.equal(ops.latent_attention(*args, causal=True), want)
    one = ops.latent_attention(q[:1].expand(2, -1, -1, -1), kv[:1].expand(
        2, -1, -1, -1), k_rope[:1].expand(2, -1, -1), causal=True)
    assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_expanded_peaked_scores(device, dtype):
    """Scores that rise along the keys move the running reference in every
    tile; one far above the others leaves them no weight."""
    q, kv, k_rope = make_expanded(1, 64, 400, 1, 64, 32, dtype, device)
    q[..., 0] = 4.0
    kv[0, :, 0, 0] = torch.linspace(-30, 30, 400, device=device)
    kv[0, 137, 0, 0] = 60.0
    out = ops.latent_attention(q, kv, k_rope, scale=0.5)
    check(out, *expanded_exact(q, kv, k_rope, 0.5, False, None, None), dtype)


@pytest.mark.parametrize("device", DEVICES)
def test_expanded_many_small_weights(device):
    """A thousand weights that together count, each below fp16's normal
    range next to the largest."""
    dtype = torch.float16
    q, kv, k_rope = make_expanded(1, 3, 1025, 1, 64, 32, dtype, device)
    q.zero_()
    q[..., 0] = 1.0
    kv[..., 0] = 0.0
    kv[0, 700, 0, 0] = 12.0         # e^12 times the weight of each other
    kv[..., 64:] = kv[..., 64:].abs() * 8.0
    kv[0, 700, 0, 64:] = 0.0
    out = ops.latent_attention(q, kv, k_rope, scale=1.0)
    check(out, *expanded_exact(q, kv, k_rope, 1.0, False, None, None), dtype)


@pytest.mark.parametrize("device", DEVICES)
def test_expanded_empty(device):
    q, kv, k_rope = make_expanded(2, 3, 0, 2, 64, 32, torch.float16, device)
    assert torch.equal(ops.latent_attention(q, kv, k_rope),
                       torch.zeros(2, 3, 2, 64, dtype=q.dtype, device=device))
    for shape in ((0, 3, 2), (2, 0, 2), (2, 3, 0)):
        b, s, h = shape
        q, kv, k_rope = make_expanded(b, s, s, h, 64, 32, torch.float16,
                                      device)
        assert ops.latent_attention(q, kv, k_rope).shape == (b, s, h, 64)


@pytest.mark.parametrize("device", DEVICES)
def test_expanded_refusals(device):
    q, kv, k_rope = make_expanded(2, 5, 5, 2, 64, 32, torch.bfloat16, device)
    n = torch.full((2,), 5, dtype=torch.int32, device=device)
    bad = [
        ((q.half(), kv, k_rope), {}), ((q, kv[:1], k_rope), {}),
        ((q, kv, k_rope[:, :4]), {}), ((q, kv[:, :, :1], k_rope), {}),
        ((q[..., :80], kv, k_rope), {}), ((q, kv[..., :96], k_rope), {}),
        ((q[0], kv, k_rope), {}), ((q, kv, k_rope[..., :16]), {}),
        ((q, kv, k_rope), dict(scale=0.0)),
        ((q, kv, k_rope), dict(scale=float("nan"))),
        ((q, kv, k_rope), dict(lengths=n.long())),
        ((q, kv, k_rope), dict(lengths=n[:1])),
        ((q, kv, k_rope), dict(past=n.unsqueeze(0))),
        ((q[:, :3], kv, k_rope), dict(lengths=n)),
        ((q.clone().requires_grad_(), kv, k_rope), {}),
    ]
    for args, kw in bad:
        with pytest.raises((TypeError, ValueError)):
            ops.latent_attention(*args, **kw)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.latent_attention(q, kv.cpu(), k_rope)
        with pytest.raises(TypeError):
            ops.latent_attention(q.float(), kv.float(), k_rope.float())


@pytest.mark.gpu
def test_expanded_graph():
    q, kv, k_rope = make_expanded(2, 90, 90, 4, 128, 64, torch.bfloat16,
                                  "cuda")
    n = torch.tensor([90, 33], dtype=torch.int32, device="cuda")
    ops.latent_attention(q, kv, k_rope, causal=True, lengths=n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.latent_attention(q, kv, k_rope, causal=True, lengths=n)
    for i in range(3):
        kv.copy_(torch.randn_like(kv))
        n[1] = 20 * i + 7
        graph.replay()
        torch.cuda.synchronize()
        want = ops.latent_attention(q, kv, k_rope, causal=True, lengths=n)
        assert torch.equal(out, want)
