"""Rotary positions against complex rotation in 64 bits: layouts, parts of a
head, strides, far positions, in-place views, refusals. Every case runs on
the CPU path; with a GPU the same cases run on the HIP kernel."""
import math
import random

import pytest
import torch

from pipeedge_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def exact(x, positions, freqs, interleaved, offset, inverse, scale):
    width = 2 * freqs.numel()
    x = x.double().cpu()
    angle = positions.double().cpu().unsqueeze(-1) * freqs.cpu()
    turn = torch.polar(torch.full_like(angle, scale),
                       -angle if inverse else angle).unsqueeze(-2)
    part = x[..., offset:offset + width]
    pair = part.unflatten(-1, (-1, 2)) if interleaved \
        else part.unflatten(-1, (2, -1)).transpose(-1, -2)
    out = torch.view_as_real(
        torch.complex(pair[..., 0], pair[..., 1]) * turn)
    out = out if interleaved else out.transpose(-1, -2)
    return torch.cat((x[..., :offset], out.flatten(-2),
                      x[..., offset + width:]), dim=-1)


def check(out, x, positions, freqs, interleaved, offset, inverse, scale):
    """A product pair in fp32 (4 roundings of cos, sin, two products and the
    sum, each eps32/2 of at most |a|+|b|, and the sine's own few units) and
    one rounding to the type of half a step of the result; halved steps of
    subnormal fp16 results are covered by its smallest step. An angle is off
    by at most four 64-bit roundings of the largest (frequencies are <= 1)."""
    ref = exact(x, positions, freqs, interleaved, offset, inverse, scale)
    size = x.double().cpu().abs().amax() * 2.0 * scale
    step = torch.finfo(x.dtype)
    far = positions.abs().max().item() * 4 * 2.0 ** -53
    bound = ref.abs() * step.eps / 2 + size * (16 * 2.0 ** -24 + far) \
        + step.tiny * step.eps
    assert out.dtype == x.dtype and out.shape == x.shape
    worst = ((out.double().cpu() - ref).abs() / bound).max().item()
    assert worst <= 1.0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,h,hk,dim,width,offset", [
    (1, 1, 1, 1, 2, 2, 0),           # the smallest call
    (8, 1, 16, 1, 64, 64, 0),        # a decoding step, one shared key
    (3, 37, 12, 12, 64, 64, 0),
    (2, 5, 5, 2, 80, 80, 0),
    (1, 130, 4, 4, 128, 64, 64),     # the last half of a head
    (1, 7, 3, 1, 96, 32, 16),        # columns on both sides
    (2, 9, 3, 2, 33, 10, 5),         # no alignment at all
    (1, 3, 130, 7, 24, 8, 8),
])
def test_rotary_matches_exact(device, dtype, interleaved, b, s, h, hk, dim,
                              width, offset):
    torch.manual_seed(b * 1000 + s)
    q = torch.randn(b, s, h, dim).to(dtype).to(device)
    k = torch.randn(b, s, hk, dim).to(dtype).to(device)
    pos = torch.randint(0, 100000, (b, s), device=device)
    freqs = ops.rotary_frequencies(width, device=device)
    for inverse, scale in ((False, 1.0), (True, 1.25)):
        args = (interleaved, offset, inverse, scale)
        kw = dict(interleaved=interleaved, offset=offset, inverse=inverse,
                  scale=scale)
        qo, ko = ops.rotary(q, pos, freqs, k, **kw)
        check(qo, q, pos, freqs, *args)
        check(ko, k, pos, freqs, *args)
        only = ops.rotary(q, pos.int(), freqs, **kw)
        assert torch.equal(only, qo)


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_far_positions(device):
    """The angle of a position past 2^31 keeps its low bits."""
    pos = torch.tensor([0, 1, -5, 2 ** 24 + 1, 2 ** 31 + 7, 2 ** 40 + 3],
                       device=device)
    q = torch.randn(6, 2, 64, device=device)
    freqs = ops.rotary_frequencies(64, device=device)
    out = ops.rotary(q, pos, freqs)
    check(out, q, pos, freqs, False, 0, False, 1.0)
    near = pos.cpu() < 2 ** 32
    check(out.cpu()[near], q.cpu()[near], pos.cpu()[near], freqs.cpu(),
          False, 0, False, 1.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strided_inputs(device, interleaved):
    """Heads before tokens, padded rows, misaligned storage, 3 and 5 dims."""
    torch.manual_seed(3)
    freqs = ops.rotary_frequencies(32, device=device)
    pos = torch.randint(0, 999, (2, 19), device=device)
    base = torch.randn(2, 6, 19, 80, device=device, dtype=torch.bfloat16)
    for q in (base.transpose(1, 2), base.transpose(1, 2)[..., 8:72],
              base.transpose(1, 2)[..., 3:67], base[:, ::2].transpose(1, 2)):
        out = ops.rotary(q, pos, freqs, interleaved=interleaved)
        assert out.is_contiguous()
        check(out, q, pos, freqs, interleaved, 0, False, 1.0)
    q = base.transpose(1, 2)
    whole = ops.rotary(q, pos, freqs, interleaved=interleaved)
    flat = ops.rotary(q.reshape(-1, 6, 80), pos.reshape(-1), freqs,
                      interleaved=interleaved)
    deep = ops.rotary(q.reshape(1, 2, 19, 6, 80), pos.unsqueeze(0), freqs,
                      interleaved=interleaved)
    token = ops.rotary(q[1, 4], pos[1, 4], freqs, interleaved=interleaved)
    assert torch.equal(flat.view_as(whole), whole)
    assert torch.equal(deep.view_as(whole), whole)
    assert torch.equal(token, whole[1, 4])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_in_place_packed_qkv(device, dtype):
    """The q and k heads of a packed projection, v left as it was."""
    torch.manual_seed(4)
    b, s, h, dh = 2, 21, 4, 64
    qkv = torch.randn(b, s, 3 * h * dh, device=device).to(dtype)
    before = qkv.clone()
    pos = torch.arange(s, device=device).expand(b, s)
    freqs = ops.rotary_frequencies(dh, device=device)
    heads = qkv.view(b, s, 3 * h, dh)[:, :, :2 * h]
    assert ops.rotary_(heads, pos, freqs) is not None
    want = ops.rotary(before.view(b, s, 3 * h, dh)[:, :, :2 * h], pos, freqs)
    assert torch.equal(heads, want)
    assert torch.equal(qkv[..., 2 * h * dh:], before[..., 2 * h * dh:])
    # part of a head, with a key that has its own strides
    x = torch.randn(b, s, h, 96, device=device).to(dtype)
    key = torch.randn(b, s, 40, device=device).to(dtype)
    x0, key0 = x.clone(), key.clone()
    freqs = ops.rotary_frequencies(32, device=device)
    ops.rotary_(x[..., 64:], pos, freqs, key[..., 8:].unsqueeze(2))
    wq, wk = ops.rotary(x0[..., 64:], pos, freqs, key0[..., 8:].unsqueeze(2))
    assert torch.equal(x[..., 64:], wq) and torch.equal(x[..., :64], x0[..., :64])
    assert torch.equal(key[..., 8:], wk.squeeze(2))
    assert torch.equal(key[..., :8], key0[..., :8])


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_inverse_is_gradient(device):
    """<rotary(x), g> = <x, inverse(g)>, and the gradient by differences."""
    torch.manual_seed(5)
    x = torch.randn(2, 3, 2, 16, device=device)
    g = torch.randn(2, 3, 2, 16, device=device)
    pos = torch.randint(0, 50, (2, 3), device=device)
    freqs = ops.rotary_frequencies(8, device=device)
    kw = dict(offset=4, scale=1.5)
    grad = ops.rotary(g, pos, freqs, inverse=True, **kw).double()
    for index in ((0, 0, 0, 5), (1, 2, 1, 9), (1, 0, 0, 0)):
        d = torch.zeros_like(x)
        d[index] = 0.5
        diff = (ops.rotary(x + d, pos, freqs, **kw).double()
                - ops.rotary(x - d, pos, freqs, **kw).double())
        # linear in x: each of four columns is off by a few fp32 steps of
        # values below 8
        assert abs((diff * g.double()).sum() - grad[index]) < 64 * 8 * 2.0 ** -24 * 4


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_nonfinite_stays_in_its_pair(device):
    x = torch.randn(1, 4, 2, 32, device=device, dtype=torch.bfloat16)
    x[0, 1, 0, 3] = float("nan")
    x[0, 2, 1, 30] = float("inf")
    pos = torch.arange(4, device=device).unsqueeze(0)
    freqs = ops.rotary_frequencies(16, device=device)
    out = ops.rotary(x, pos, freqs)
    bad = ~torch.isfinite(out)
    assert bad[0, 1, 0, 3] and bad[0, 1, 0, 11] and bad[0, 2, 1, 30]
    assert bad.sum() == 3


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_empty(device):
    freqs = ops.rotary_frequencies(8, device=device)
    q = torch.empty(2, 0, 4, 8, device=device)
    pos = torch.empty(2, 0, dtype=torch.int64, device=device)
    assert ops.rotary(q, pos, freqs).shape == q.shape
    q = torch.ones(2, 3, 0, 8, device=device)
    k = torch.ones(2, 3, 1, 8, device=device)
    pos = torch.zeros(2, 3, dtype=torch.int64, device=device)
    qo, ko = ops.rotary(q, pos, freqs, k)
    assert qo.shape == q.shape and torch.equal(ko, k)


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_refusals(device):
    q = torch.zeros(2, 3, 4, 16, device=device)
    pos = torch.zeros(2, 3, dtype=torch.int64, device=device)
    freqs = ops.rotary_frequencies(16, device=device)
    bad = [
        (q.double(), pos, freqs, {}), (q, pos.float(), freqs, {}),
        (q, pos, freqs.float(), {}), (q, pos, freqs, dict(offset=2)),
        (q, pos, freqs, dict(offset=-1)), (q, pos[:1], freqs, {}),
        (q, pos[0], freqs, {}), (q, pos, freqs[:0], {}),
        (q, pos, freqs, dict(k=q.half())),
        (q, pos, freqs, dict(k=q[:, :2])),
        (q, pos, freqs, dict(k=q[..., :8])),
        (q[..., 0], pos, freqs, {}),
        (q.transpose(-1, -2).contiguous().transpose(-1, -2), pos, freqs, {}),
        (q.clone().requires_grad_(), pos, freqs, {}),
    ]
    for x, p, f, kw in bad:
        for op in (ops.rotary, ops.rotary_):
            with pytest.raises((TypeError, ValueError)):
                op(x, p, f, **kw)
    with pytest.raises(ValueError):
        ops.rotary_(q, pos, freqs, q)
    with pytest.raises(ValueError):
        ops.rotary_(q[:, :1].expand(2, 3, 4, 16), pos, freqs)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.rotary(q, pos.cpu(), freqs)


def test_rotary_frequencies():
    f = ops.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert f[0] == 1.0
    assert math.isclose(f[31].item(), 10000.0 ** (-62 / 64))
    assert torch.equal(ops.rotary_frequencies(64, scaling="linear",
                                              factor=4.0), f / 4.0)
    g = ops.rotary_frequencies(64, scaling="base", factor=4.0)
    assert g[0] == 1.0 and math.isclose(g[31].item(), f[31].item() / 4.0)
    r = ops.rotary_frequencies(64, scaling="ramp", factor=4.0,
                               original_length=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(r[turns >= 32], f[turns >= 32])
    assert torch.allclose(r[turns <= 1], f[turns <= 1] / 4.0, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (r[mid] < f[mid]).all() and (r[mid] > f[mid] / 4).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0),
                dict(rotary_dim=8, scaling="cubic"),
                dict(rotary_dim=8, scaling="ramp"),
                dict(rotary_dim=8, factor=0.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)


@pytest.mark.gpu
def test_rotary_streams_and_graph():
    """Another stream, and a captured call replayed between eager work."""
    freqs = ops.rotary_frequencies(64, device="cuda")
    q = torch.randn(4, 50, 8, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.randn(4, 50, 2, 64, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(50, device="cuda").expand(4, 50).contiguous()
    want = ops.rotary(q, pos, freqs, k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rotary(q, pos, freqs, k)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary(q, pos, freqs, k)
    for i in range(3):
        q.copy_(torch.randn_like(q))
        pos.add_(100 * i)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.rotary(q, pos, freqs, k)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_in_place_is_seen_by_autograd(device):
    """A graph that saved a tensor refuses to go back once it was turned."""
    freqs = ops.rotary_frequencies(8, device=device)
    pos = torch.arange(6, device=device).reshape(2, 3)
    q = torch.randn(2, 3, 4, 8, device=device)
    k = torch.randn(2, 3, 1, 8, device=device)
    for kw in (dict(k=k), {}):
        for x in (q, k)[:1 + len(kw)]:
            w = torch.ones_like(x, requires_grad=True)
            loss = (w * x).sum()
            ops.rotary_(q, pos, freqs, **kw)
            with pytest.raises(RuntimeError):
                loss.backward()
    with torch.inference_mode():
        x = q.clone()
        ops.rotary_(x, pos, freqs)
    assert torch.equal(x, ops.rotary(q, pos, freqs))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("seed", range(12))
def test_rotary_in_place_overlap(device, seed):
    """In place, every layout whose turned columns are apart is turned, every
    other one is refused: random views of one storage, addresses counted."""
    rng = random.Random(seed)
    freqs = ops.rotary_frequencies(4, device=device)
    turned = 0
    for _ in range(40):
        b, s = rng.randint(1, 3), rng.randint(1, 4)
        base = torch.randn(2000, device=device)
        nested = rng.random() < 0.7
        views, places = [], []
        strides = None
        for heads in (rng.randint(1, 3), rng.randint(1, 3)):
            if strides is None or rng.random() < 0.4:
                strides = [rng.randint(0, 40) for _ in range(3)]
                if nested:
                    strides[2] = rng.randint(4, 9)
                    strides[1] = strides[2] * 3 + rng.randint(0, 30)
                    strides[0] = strides[1] * s + rng.randint(0, 20)
            start = rng.randint(0, 60)
            views.append(base.as_strided((b, s, heads, 6), strides + [1],
                                         start))
            # columns 1 to 4 of each head
            places.append([start + i * strides[0] + j * strides[1]
                           + h * strides[2] + c for i in range(b)
                           for j in range(s) for h in range(heads)
                           for c in range(1, 5)])
        pos = torch.randint(0, 99, (b, s), device=device)
        q, k = views
        own = [len(set(p)) < len(p) for p in places]
        both = bool(set(places[0]) & set(places[1]))
        for args, bad in (((q, pos, freqs), own[0]),
                          ((q, pos, freqs, k), any(own) or both)):
            before = base.clone()
            if bad:
                with pytest.raises(ValueError):
                    ops.rotary_(*args, offset=1)
                assert torch.equal(base, before)
                continue
            want = base.clone()
            for x in args[:1] + args[3:]:
                w = want.as_strided(x.shape, x.stride(), x.storage_offset())
                w[..., 1:5] = ops.rotary(x, pos, freqs, offset=1)[..., 1:5]
            ops.rotary_(*args, offset=1)
            assert torch.equal(base, want)
            turned += 1
    assert turned >= 5


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_in_place_keys_behind_queries(device):
    """Parts of one packed tensor, apart by heads, by columns and by tokens;
    and the same parts one head, one column, one token too long."""
    freqs = ops.rotary_frequencies(32, device=device)
    pos = torch.arange(14, device=device).reshape(2, 7)
    base = torch.randn(2, 9, 6, 96, device=device, dtype=torch.bfloat16)
    x = base[:, :7]
    for q, k in ((x[:, :, :4], x[:, :, 4:]), (x[:, :, ::2], x[:, :, 1::2]),
                 (x[..., :48], x[..., 48:]), (x[..., :40], x[..., 32:72]),
                 (base[:, :7, :3], base[:, 2:, 3:])):
        want = ops.rotary(q, pos, freqs, k)
        width = slice(0, 32)
        ops.rotary_(q, pos, freqs, k)
        assert torch.equal(q[..., width], want[0][..., width])
        assert torch.equal(k[..., width], want[1][..., width])
    for q, k in ((x[:, :, :4], x[:, :, 3:]), (x[..., :40], x[..., 31:71]),
                 (base[:, :7], base[:, 2:]), (x, x), (x, x[..., :96])):
        with pytest.raises(ValueError):
            ops.rotary_(q, pos, freqs, k)


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_in_place_empty(device):
    """No tokens, no query heads, no key heads: the others are turned."""
    freqs = ops.rotary_frequencies(8, device=device)
    for lead, heads in (((2, 0), (4, 1)), ((0, 3), (4, 1)), ((2, 3), (0, 1)),
                        ((2, 3), (1, 0)), ((2, 3), (0, 0))):
        q, k = (torch.randn(*lead, h, 8, device=device) for h in heads)
        pos = torch.ones(lead, dtype=torch.int64, device=device)
        want = ops.rotary(q, pos, freqs, k)
        got = ops.rotary_(q, pos, freqs, k)
        assert got[0] is q and got[1] is k
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_leading_dimensions(device):
    """Five and six dimensions whose leading ones are not one in memory."""
    freqs = ops.rotary_frequencies(16, device=device)
    x = torch.randn(3, 2, 5, 6, 16, device=device)
    y = torch.randn(2, 4, 3, 5, 6, 16, device=device)
    for x, pos in ((x.transpose(0, 1), torch.randint(0, 99, (2, 3, 5))),
                   (x[:, :1], torch.randint(0, 99, (3, 1, 5))),
                   (y.permute(2, 0, 1, 3, 4, 5),
                    torch.randint(0, 99, (3, 2, 4, 5))),
                   (y[:, :, :2, ::2], torch.randint(0, 99, (2, 4, 2, 3)))):
        pos = pos.to(device)
        for q, k in ((x[..., :4, :], x[..., 4:, :]),
                     (x[..., :4, :], x[..., 4:, :].contiguous()),
                     (x[..., :4, :].contiguous(), x[..., 4:, :])):
            want = ops.rotary(q.contiguous(), pos, freqs, k.contiguous())
            out = ops.rotary(q, pos, freqs, k)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert torch.equal(ops.rotary(q, pos, freqs), want[0])
            got = ops.rotary_(q, pos, freqs, k)
            assert got[0] is q and got[1] is k
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_refuses_gradients_of_frequencies(device):
    q = torch.randn(2, 3, 4, 16, device=device)
    pos = torch.arange(6, device=device).reshape(2, 3)
    freqs = ops.rotary_frequencies(16, device=device).requires_grad_()
    for op in (ops.rotary, ops.rotary_):
        with pytest.raises(ValueError):
            op(q, pos, freqs)
    with torch.no_grad():
        out = ops.rotary(q, pos, freqs)
    assert torch.equal(out, ops.rotary(q, pos, freqs.detach()))


@pytest.mark.gpu
def test_rotary_more_tokens_than_one_launch_has_blocks():
    """2^24 blocks of 256 threads are one more than a launch takes."""
    tokens, near = 2 ** 24 + 70, 2 ** 24
    freqs = ops.rotary_frequencies(2, device="cuda")
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32)
    q = torch.randn(1, 1, 770, device="cuda", dtype=torch.bfloat16)
    out = ops.rotary(q.expand(tokens, 1, 770), pos, freqs)
    for some in (slice(0, 70), slice(near - 70, tokens)):
        want = ops.rotary(q.expand(pos[some].numel(), 1, 770),
                          pos[some].clone(), freqs)
        assert torch.equal(out[some], want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,width,offset,h", [
    (2048, 2048, 0, 3), (2050, 2048, 1, 1), (1600, 1040, 560, 2)])
def test_rotary_wide_heads(device, interleaved, dim, width, offset, h):
    """Up to the 2048 columns that are turned at most."""
    torch.manual_seed(dim)
    q = torch.randn(2, 5, h, dim, device=device).bfloat16()
    pos = torch.randint(0, 9999, (2, 5), device=device)
    freqs = ops.rotary_frequencies(width, device=device)
    out = ops.rotary(q, pos, freqs, interleaved=interleaved, offset=offset)
    check(out, q, pos, freqs, interleaved, offset, False, 1.0)
    ops.rotary_(q, pos, freqs, interleaved=interleaved, offset=offset)
    assert torch.equal(q, out)
    with pytest.raises(ValueError):
        ops.rotary(torch.zeros(1, 1, 2050, device=device), pos[0, :1],
                   ops.rotary_frequencies(2050, device=device))
