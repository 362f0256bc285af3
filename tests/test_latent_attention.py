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
    worst = ((out - ref).abs() / bound).max().item()
    assert worst <= 1.0             # also not if it is NaN


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
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sq,sk,h,nope,rope,lengths,past", [
    (1, 512, 1, 64, 32, None, None),
    (1, 1500, 3, 128, 64, [1500, 1, 0, 65, 1499], [1499, 0, 0, 64, 0]),
    (5, 2049, 2, 64, 64, [2049, 4, 600, 0, 1030], [2044, 0, 595, 0, -3]),
    (40, 1100, 2, 128, 32, [1100, 30, 70, 1025, 512], [1060, 0, 60, 990, 0]),
    (300, 1061, 1, 128, 64, [1061, 299, 64, 700, 3], [761, 0, 0, 400, 0]),
])
def test_expanded_long_keys(device, dtype, causal, sq, sk, h, nope, rope,
                            lengths, past):
    """Few queries of many keys, whose range is shared out: sequences that
    end before most of the shares begin, rows that see a part of one, shares
    of one tile and of none."""
    b = 1 if lengths is None else len(lengths)
    q, kv, k_rope = make_expanded(b, sq, sk, h, nope, rope, dtype, device)
    n = p = None
    if lengths is not None:
        n = torch.tensor(lengths, dtype=torch.int32)
        p = torch.tensor(past, dtype=torch.int32)
        for i, end in enumerate(lengths):
            kv[i, end:] = math.nan
            k_rope[i, end:] = math.inf
    out = ops.latent_attention(
        q, kv, k_rope, causal=causal,
        lengths=None if n is None else n.to(device),
        past=None if p is None else p.to(device))
    check(out, *expanded_exact(q, kv, k_rope, (nope + rope) ** -0.5, causal,
                               n, p), dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sq,sk,length,past", [
    (150, 150, 100, 0),              # padding in a tile with live queries
    (40, 40, 30, -9),                # queries before the start
    (3, 1500, 1400, 1398),           # the keys in parts
])
def test_expanded_padding_stays_zero(device, causal, sq, sk, length, past):
    """Queries outside their sequence are zero also where values inside it
    are not finite."""
    q, kv, k_rope = make_expanded(2, sq, sk, 2, 64, 32, torch.bfloat16,
                                  device)
    kv[1, 5, 1, 70] = math.inf
    kv[1, length - 1, 0, 80] = math.nan
    n = torch.full((2,), length, dtype=torch.int32, device=device)
    p = torch.full((2,), past, dtype=torch.int32, device=device)
    out = ops.latent_attention(q, kv, k_rope, causal=causal, lengths=n,
                               past=p)
    at = past + torch.arange(sq, device=device)
    outside = (at < 0) | (at >= length)
    assert outside.any() and not out[:, outside].any()
    assert out[0].isfinite().all() and out[0, ~outside].any(-1).all()
    last = int((~outside).nonzero().max())
    assert not out[1, last, 1, 6].isfinite() and out[1, last, 0, 16].isnan()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("b,sq,sk,h,parts", [
    (3, 1100, 1100, 11, 1),          # 297 blocks of 128 queries
    (5, 1027, 1027, 13, 1),          # 585
    (2, 300, 300, 113, 1),           # 678
    (3, 200, 2600, 11, 5),           # 66, the keys in 5 parts each
])
def test_expanded_causal_order_of_many_blocks(device, b, sq, sk, h, parts):
    """Causal blocks are put in another order where an XCD has more than 32:
    each of them has to be there once."""
    blocks = b * h * -(-sq // 128)
    assert parts == max(1, min(512 // blocks, -(-sk // 64) // 8))
    assert blocks * parts > 256 and blocks * parts % 8 != 0
    q, kv, k_rope = make_expanded(b, sq, sk, h, 64, 32, torch.bfloat16,
                                  device)
    out = ops.latent_attention(q, kv, k_rope, causal=True)
    check(out, *expanded_exact(q, kv, k_rope, 96 ** -0.5, True, None, None),
          torch.bfloat16)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("part,column", [("plain", 3), ("rope", 30)])
def test_expanded_hidden_keys_not_finite(device, part, column):
    """A key that is not finite reaches only the queries that see it. Others
    keep their result but not its bits: 32 rows move the reference of their
    softmax at the same time, and a weight 2^(score - reference) is rounded
    differently for another reference, within the same half step."""
    q, kv, k_rope = make_expanded(1, 200, 200, 2, 64, 32, torch.bfloat16,
                                  device)
    want = ops.latent_attention(q, kv, k_rope, causal=True)
    exact = expanded_exact(q, kv, k_rope, 96 ** -0.5, True, None, None)
    for value in (math.nan, math.inf):
        keys, rope = kv.clone(), k_rope.clone()
        (keys[0, 77, 1] if part == "plain" else rope[0, 77])[column] = value
        out = ops.latent_attention(q, keys, rope, causal=True)
        check(out[:, :77], *(x[:, :77] for x in exact), torch.bfloat16)
        assert torch.equal(out[:, :64], want[:, :64])
        if part == "plain":
            assert torch.equal(out[:, :, 0], want[:, :, 0])
        if math.isnan(value):
            assert out[:, 77:, 1].isnan().all()


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


@pytest.mark.gpu
@pytest.mark.parametrize("sq,sk", [(100, 100), (3, 1100)])
def test_expanded_far_sequences(sq, sk):
    """Sequences more than 2^32 bytes apart."""
    q, kv, k_rope = make_expanded(2, sq, sk, 2, 128, 64, torch.float16,
                                  "cuda")
    want = ops.latent_attention(q, kv, k_rope, causal=True)
    room = torch.empty(2 ** 31 + 2 * kv[0].numel(), dtype=torch.float16,
                       device="cuda")
    far = room.as_strided(kv.shape, (2 ** 31 + 8,) + kv.stride()[1:])
    far.copy_(kv)
    assert torch.equal(ops.latent_attention(q, far, k_rope, causal=True),
                       want)


@pytest.mark.gpu
def test_expanded_refuses_far_tokens():
    q, kv, k_rope = make_expanded(1, 2, 2, 1, 64, 32, torch.float16, "cuda")
    room = torch.zeros(2 ** 24 + 4096, dtype=torch.float16, device="cuda")
    for step, fits in ((2 ** 24 - 8, True), (2 ** 24, False)):
        far = room.as_strided(kv.shape, (step, step, 128, 1))
        far.copy_(kv)
        if fits:
            assert torch.equal(ops.latent_attention(q, far, k_rope),
                               ops.latent_attention(q, kv, k_rope))
        else:
            with pytest.raises(ValueError):
                ops.latent_attention(q, far, k_rope)


@pytest.mark.gpu
def test_expanded_refuses_more_rows_than_a_launch_takes():
    q, kv, k_rope = make_expanded(1, 1, 1, 1, 64, 32, torch.bfloat16, "cuda")
    b, h = 2 ** 10, 2 ** 14
    with pytest.raises(ValueError):
        ops.latent_attention(q.expand(b, 1, h, 96), kv.expand(b, 1, h, 128),
                             k_rope.expand(b, 1, 32))
    b -= 1
    out = ops.latent_attention(q.expand(b, 1, h, 96),
                               kv.expand(b, 1, h, 128),
                               k_rope.expand(b, 1, 32))
    assert torch.equal(out, kv[..., 64:].expand_as(out))


@pytest.mark.gpu
def test_expanded_token_distance_is_that_of_the_copy():
    """Values that have to be copied count with the copy's distance between
    tokens, and a single token has none."""
    heads = 2 ** 17
    q = torch.randn(1, 1, 1, 96, device="cuda").bfloat16()
    kv = torch.randn(1, 2, 1, 131, device="cuda").bfloat16()[..., 3:]
    k_rope = torch.randn(1, 2, 32, device="cuda").bfloat16()
    many = kv.expand(1, 2, heads, 128)
    with pytest.raises(ValueError):
        ops.latent_attention(q.expand(1, 1, heads, 96), many, k_rope)
    half = ops.latent_attention(q.expand(1, 1, heads // 2, 96),
                                many[:, :, :heads // 2], k_rope)
    one = ops.latent_attention(q, kv, k_rope)
    assert torch.equal(half, one.expand_as(half))
    want = ops.latent_attention(q, kv[:, :1], k_rope[:, :1])
    room = torch.zeros(1, 1, 2 ** 25, device="cuda", dtype=q.dtype)
    far = room.as_strided((1, 1, 1, 128), (2 ** 25, 2 ** 24, 128, 1))
    rope = room.as_strided((1, 1, 32), (2 ** 25, 2 ** 24, 1), 2 ** 23)
    far.copy_(kv[:, :1])
    rope.copy_(k_rope[:, :1])
    assert torch.equal(ops.latent_attention(q, far, rope), want)


@pytest.mark.gpu
def test_expanded_shared_range_graphs():
    """The partial sums are a graph's own: two graphs and eager calls on
    another stream, in turn and at once."""
    many = [make_expanded(3, 4, 1200, 4, 128, 64, torch.bfloat16, "cuda",
                          seed=i) for i in range(3)]
    want = [ops.latent_attention(*x, causal=True) for x in many]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in many[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.latent_attention(*x, causal=True))
    other = torch.cuda.Stream()
    for _ in range(4):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
            eager = ops.latent_attention(*many[2], causal=True)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0])
        assert torch.equal(outs[1], want[1])
        assert torch.equal(eager, want[2])


# ---------------------------------------------------------------- absorbed

def cache_exact(q, cache, table, lengths, latent, scale):
    b, sq, h, width = q.shape
    q, cache, table = q.cpu(), cache.cpu(), table.cpu().long()
    page = cache.shape[1]
    ref = torch.zeros(b, sq, h, latent, dtype=torch.float64)
    size, drift = torch.zeros_like(ref), torch.zeros(b, sq, h).double()
    for i in range(b):
        n = int(lengths[i])
        if n == 0:
            continue
        place = torch.arange(n)
        tokens = cache[table[i, place // page], place % page]
        upto = (n - sq + 1 + torch.arange(sq)).clamp(min=0)
        r, s, d = attend(q[i].reshape(sq * h, width), tokens,
                         tokens[:, :latent], scale,
                         upto.repeat_interleave(h))
        ref[i], size[i] = r.view(sq, h, latent), s.view(sq, h, latent)
        drift[i] = d.view(sq, h)
    return ref, size, drift


def make_cache(lengths, sq, h, latent, rope, page, dtype, device, seed=0,
               spare=2):
    """Pages in random order; unused table entries and the rows behind each
    sequence's last hold what must never be read or used."""
    torch.manual_seed(seed + sq + h)
    b, width = len(lengths), latent + rope
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    cache = torch.full((pages, page, width), float("nan"))
    order = torch.randperm(pages).tolist()
    table = torch.full((b, max(max(counts), 1) + 1), -12345,
                       dtype=torch.int32)
    at = 0
    for i, n in enumerate(lengths):
        for j in range(counts[i]):
            table[i, j] = order[at]
            rows = min(page, n - j * page)
            cache[order[at], :rows] = torch.randn(rows, width)
            at += 1
    q = torch.randn(b, sq, h, width)
    return (q.to(dtype).to(device), cache.to(dtype).to(device),
            table.to(device),
            torch.tensor(lengths, dtype=torch.int32, device=device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("latent,rope,page", [
    (512, 64, 64), (512, 32, 16), (256, 64, 8), (256, 32, 1),
    (512, 64, 24), (256, 64, 7), (512, 32, 3),
])
@pytest.mark.parametrize("sq,h,lengths", [
    (1, 1, [1]),
    (1, 16, [517, 1, 64, 0, 63, 65, 300]),
    (1, 20, [100, 33, 0, 257]),
    (3, 12, [2, 31, 190, 1, 0]),     # queries before the start
    (2, 64, [129, 400]),             # a full block of rows
    (3, 50, [77, 5]),                # two blocks of rows, the last ragged
])
def test_cache_matches_exact(device, dtype, latent, rope, page, sq, h,
                             lengths):
    q, cache, table, n = make_cache(lengths, sq, h, latent, rope, page, dtype,
                                    device)
    out = ops.latent_cache_attention(q, cache, table, n, latent_dim=latent,
                                     scale=0.07)
    assert out.shape == (len(lengths), sq, h, latent) and out.dtype == dtype
    check(out, *cache_exact(q, cache, table, lengths, latent, 0.07), dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("latent,rope,page", [
    (512, 64, 64), (512, 64, 7), (512, 32, 64), (512, 32, 1),
    (256, 64, 24), (256, 32, 16), (256, 32, 5),
])
@pytest.mark.parametrize("sq,h", [(1, 33), (3, 27), (2, 64)])
def test_cache_of_room_for_long_runs(device, dtype, latent, rope, page, sq,
                                     h):
    """More than 32 rows and tables that could hold long caches: two waves a
    row group, each with half of a tile's tokens, whatever the lengths."""
    lengths = [1500, 0, 700, 33, 1, 64]
    q, cache, table, n = make_cache(lengths, sq, h, latent, rope, page, dtype,
                                    device)
    groups = -(-sq * h // 64)
    # 16 tiles of 64 tokens for each of the runs that the chip takes
    room = 16 * (256 // groups) * 64
    wide = -(-room // (page * len(lengths))) + 1
    assert wide > table.shape[1]
    table = torch.nn.functional.pad(table, (0, wide - table.shape[1]),
                                    value=-12345)
    out = ops.latent_cache_attention(q, cache, table, n, latent_dim=latent,
                                     scale=0.07)
    check(out, *cache_exact(q, cache, table, lengths, latent, 0.07), dtype)


@pytest.mark.parametrize("device", DEVICES)
def test_cache_long_and_many(device):
    """Runs of tiles that cross sequences, and more sequences than a wave."""
    lengths = [(37 * i) % 200 for i in range(150)] + [5000, 0, 3]
    q, cache, table, n = make_cache(lengths, 1, 4, 256, 32, 16,
                                    torch.bfloat16, device)
    out = ops.latent_cache_attention(q, cache, table, n, latent_dim=256,
                                     scale=0.07)
    check(out, *cache_exact(q, cache, table, lengths, 256, 0.07),
          torch.bfloat16)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("h,page", [(16, 64), (32, 5), (70, 16)])
def test_cache_many_and_one_long(device, h, page):
    """Runs that hold many short sequences, end in a long one, are inside it
    and begin with its end."""
    lengths = [1 + i % 5 for i in range(90)] + [3001] + [i % 3
                                                         for i in range(80)]
    q, cache, table, n = make_cache(lengths, 1, h, 256, 64, page,
                                    torch.float16, device)
    out = ops.latent_cache_attention(q, cache, table, n, latent_dim=256,
                                     scale=0.06)
    check(out, *cache_exact(q, cache, table, lengths, 256, 0.06),
          torch.float16)


@pytest.mark.parametrize("device", DEVICES)
def test_cache_shared_pages(device):
    """Sequences with a common beginning share its pages, and a page may
    stand in a sequence twice."""
    lengths = [40, 33, 50]
    q, cache, table, n = make_cache(lengths, 2, 16, 256, 32, 16,
                                    torch.bfloat16, device)
    table[1, :2] = table[0, :2]
    table[2, 1] = table[2, 0]
    out = ops.latent_cache_attention(q, cache, table, n, latent_dim=256,
                                     scale=0.06)
    check(out, *cache_exact(q, cache, table, lengths, 256, 0.06),
          torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [64, 7])
def test_cache_far_pages(page):
    """Pages behind 2^32 bytes of a cache are those of a small one."""
    lengths = [3 * page, 2 * page + 1, 1, 0]
    q, cache, table, n = make_cache(lengths, 2, 16, 512, 64, page,
                                    torch.bfloat16, "cuda")
    want = ops.latent_cache_attention(q, cache, table, n, latent_dim=512,
                                      scale=0.05)
    first = 2 ** 32 // (page * 576 * 2) + 1
    large = torch.empty(first + cache.shape[0], page, 576,
                        dtype=torch.bfloat16, device="cuda")
    large[first:] = cache
    out = ops.latent_cache_attention(
        q, large, torch.where(table >= 0, table + first, table), n,
        latent_dim=512, scale=0.05)
    assert torch.equal(out, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_cache_peaked_scores(device, dtype):
    """Scores that rise along the cache move the reference in every tile."""
    lengths = [700, 900]
    q, cache, table, n = make_cache(lengths, 1, 16, 256, 32, 64, dtype,
                                    device)
    q[..., 0] = 4.0
    for i, length in enumerate(lengths):
        place = torch.arange(length, device=device)
        cache[table[i].long()[place // 64], place % 64, 0] = torch.linspace(
            -30, 30, length, device=device).to(dtype)
    out = ops.latent_cache_attention(q, cache, table, n, latent_dim=256,
                                     scale=0.5)
    check(out, *cache_exact(q, cache, table, lengths, 256, 0.5), dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("h,page", [(4, 16), (10, 7), (40, 64)])
def test_cache_before_the_start_stays_zero(device, h, page):
    """Queries before their sequence's start are zero also where what is
    cached is not finite, in whole sequences and in joined ones."""
    lengths = [2, 300, 5]
    q, cache, table, n = make_cache(lengths, 303, h, 256, 32, page,
                                    torch.bfloat16, device)
    for i in (0, 1):
        cache[table[i, 0].long(), 1, 7] = math.nan
    out = ops.latent_cache_attention(q, cache, table, n, latent_dim=256,
                                     scale=0.1)
    for i, length in enumerate(lengths):
        assert not out[i, :303 - length].any()
        assert out[i, 303 - length:].any(-1).all()
        assert out[i, -1, :, 7].isnan().all() == (i < 2)
    assert out[2].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("h", [8, 16, 40])
def test_cache_newest_row_not_finite(device, h):
    """What the newest row holds reaches its own query and, where it is a
    value, may reach earlier ones, but no other sequence; in the rotary
    columns, which are keys alone, it reaches no earlier query. (The rows of a
    wave move the reference of their softmax at the same time, so theirs may
    be rounded differently, within the same half step.)"""
    lengths = [70, 130, 5]
    q, cache, table, n = make_cache(lengths, 2, h, 256, 32, 16,
                                    torch.bfloat16, device)
    kw = dict(latent_dim=256, scale=0.1)
    want = ops.latent_cache_attention(q, cache, table, n, **kw)
    ref = [x[1, 0] for x in cache_exact(q, cache, table, lengths, 256, 0.1)]
    page, place = int(table[1, 129 // 16]), 129 % 16
    for column in (9, 260):
        for value in (math.nan, math.inf):
            bad = cache.clone()
            bad[page, place, column] = value
            out = ops.latent_cache_attention(q, bad, table, n, **kw)
            assert torch.equal(out[0], want[0])
            assert torch.equal(out[2], want[2])
            assert not out[1, 1].isfinite().all()
            other = torch.arange(256) != column
            check(out[1, 0].cpu()[:, other], ref[0][:, other],
                  ref[1][:, other], ref[2], torch.bfloat16)


@pytest.mark.parametrize("device", DEVICES)
def test_cache_strided(device):
    """A layer's slice of a larger cache, queries with heads first, a table
    that is part of a wider one."""
    lengths = [130, 64, 17]
    q, cache, table, n = make_cache(lengths, 2, 6, 256, 64, 16,
                                    torch.float16, device)
    want = ops.latent_cache_attention(q, cache, table, n, latent_dim=256,
                                      scale=0.1)
    layers = torch.zeros(cache.shape[0], 3, 16, 320, dtype=cache.dtype,
                         device=device)
    layers[:, 1] = cache
    by_token = torch.zeros(cache.shape[0], 16, 2, 336, dtype=cache.dtype,
                           device=device)
    by_token[:, :, 1, 16:] = cache
    q2 = q.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(3, table.shape[1] * 2, dtype=torch.int32,
                       device=device)
    wide[:, 1::2] = table
    for c in (layers[:, 1], by_token[:, :, 1, 16:]):
        for t in (table, wide[:, 1::2]):
            got = ops.latent_cache_attention(q2, c, t, n, latent_dim=256,
                                             scale=0.1)
            assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_cache_bad_pages_and_lengths(device):
    """They spoil their own sequence and no other. On the CPU first: the GPU
    run follows where the reference is clear."""
    lengths = [130, 64, 17, 40]
    args = (lengths, 1, 4, 256, 32, 16, torch.bfloat16, device)
    q, cache, table, n = make_cache(*args)
    good = ops.latent_cache_attention(q, cache, table, n, latent_dim=256,
                                      scale=0.1)
    assert torch.isfinite(good).all()
    for page in (-1, cache.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, 3] = page
        t[2, 0] = page
        out = ops.latent_cache_attention(q, cache, t, n, latent_dim=256,
                                         scale=0.1)
        assert torch.isnan(out[0]).all() and torch.isnan(out[2]).all()
        assert torch.equal(out[1], good[1]) and torch.equal(out[3], good[3])
    m = n.clone()
    m[1] = table.shape[1] * 16 + 1
    t = table.clone()
    t[1] = 0
    out = ops.latent_cache_attention(q, cache, t, m, latent_dim=256,
                                     scale=0.1)
    assert torch.isnan(out[1]).all()
    assert torch.equal(out[0], good[0]) and torch.equal(out[2:], good[2:])
    m[1] = -5
    out = ops.latent_cache_attention(q, cache, t, m, latent_dim=256,
                                     scale=0.1)
    assert not out[1].any() and torch.equal(out[0], good[0])


@pytest.mark.parametrize("device", DEVICES)
def test_cache_empty(device):
    q, cache, table, n = make_cache([5, 3], 1, 4, 256, 32, 16,
                                    torch.bfloat16, device)
    kw = dict(latent_dim=256, scale=0.1)
    for x in (q[:, :0], q[:, :, :0]):
        assert ops.latent_cache_attention(
            x, cache, table, n, **kw).shape == x.shape[:3] + (256,)
    assert ops.latent_cache_attention(q[:0], cache, table[:0], n[:0],
                                      **kw).shape == (0, 1, 4, 256)
    out = ops.latent_cache_attention(q, cache, table[:, :0], n * 0, **kw)
    assert not out.any()
    out = ops.latent_cache_attention(q, cache, table[:, :0], n, **kw)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("device", DEVICES)
def test_cache_refusals(device):
    q, cache, table, n = make_cache([5, 3], 1, 4, 256, 32, 16,
                                    torch.bfloat16, device)
    kw = dict(latent_dim=256, scale=0.1)
    bad = [
        ((q.half(), cache, table, n), kw), ((q[0], cache, table, n), kw),
        ((q, cache[0], table, n), kw), ((q[..., :280], cache, table, n), kw),
        ((q, cache, table.long(), n), kw), ((q, cache, table, n.long()), kw),
        ((q, cache, table[:1], n), kw), ((q, cache, table, n[:1]), kw),
        ((q, cache, table[0], n), kw),
        ((q, cache, table, n), dict(latent_dim=240, scale=0.1)),
        ((q, cache, table, n), dict(latent_dim=288, scale=0.1)),
        ((q, cache, table, n), dict(latent_dim=256, scale=-1.0)),
        ((q.clone().requires_grad_(), cache, table, n), kw),
    ]
    for args, k in bad:
        with pytest.raises((TypeError, ValueError)):
            ops.latent_cache_attention(*args, **k)
    if device == "cuda":
        odd = torch.zeros(3, 16, 292, dtype=q.dtype, device=device)[..., 4:]
        for c in (odd, cache.cpu(), cache[:0],
                  cache.transpose(1, 2).contiguous().transpose(1, 2)):
            with pytest.raises(ValueError):
                ops.latent_cache_attention(q, c, table, n, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("h", [4, 16, 40, 128])
def test_cache_graph_and_repeats(h):
    """Replays with other lengths and caches equal the eager call, and so do
    two graphs on two streams at once."""
    lengths = [900, 40, 333, 0]
    q, cache, table, n = make_cache(lengths, 1, h, 256, 64, 16,
                                    torch.bfloat16, "cuda")
    cache = torch.nan_to_num(cache)
    table = table.clamp(min=0)
    kw = dict(latent_dim=256, scale=0.1)
    ops.latent_cache_attention(q, cache, table, n, **kw)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.latent_cache_attention(q, cache, table, n, **kw))
        graphs.append(g)
    side = torch.cuda.Stream()
    for i in range(3):
        cache.copy_(torch.randn_like(cache))
        n.copy_(torch.tensor([900 - 300 * i, 1 + i, 320, 64 * i]))
        want = ops.latent_cache_attention(q, cache, table, n, **kw)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [1e-50, 1e-39, 2.5e38, 1e60, math.inf,
                                   math.nan, 0.0, -1.0])
def test_scales_outside_32_bits(device, scale):
    """Scales that are zero, subnormal or infinite in 32 bits, where they
    turned hidden scores into NaN; the next ones inside give what they give."""
    q, kv, k_rope = make_expanded(1, 3, 3, 2, 64, 32, torch.bfloat16, device)
    c, cache, table, n = make_cache([5], 2, 4, 256, 32, 16, torch.bfloat16,
                                    device)
    with pytest.raises(ValueError):
        ops.latent_attention(q, kv, k_rope, causal=True, scale=scale)
    with pytest.raises(ValueError):
        ops.latent_cache_attention(c, cache, table, n, latent_dim=256,
                                   scale=scale)
    # all weights alike, in rows that see one, two and three keys
    out = ops.latent_attention(q, kv, k_rope, causal=True, scale=1e-37)
    check(out, *expanded_exact(q, kv, k_rope, 1e-37, True, None, None),
          q.dtype)
    out = ops.latent_cache_attention(c, cache, table, n, latent_dim=256,
                                     scale=1e-37)
    check(out, *cache_exact(c, cache, table, [5], 256, 1e-37), q.dtype)
