"""The adapter projection against its definition in 64 bits. Every case runs
on the CPU path; with a GPU the same cases run on the HIP kernels."""
import pytest
import torch

from pipeedge_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make(shape, k, n, rank, count, device, seed=0):
    torch.manual_seed(seed + k + n + rank)
    x = torch.randn(*shape, k)
    w = torch.randn(n, k) * k ** -0.5
    down = torch.randn(count, rank, k) * k ** -0.5
    up = torch.randn(count, n, rank) * 0.3
    return [t.bfloat16().to(device) for t in (x, w, down, up)]


def check(out, x, w, down, up, ids, bias=None, act=None, residual=None,
          scales=None):
    """Row by row. fp32 sums over K (k steps of the absolute products, for
    the shared and the inner product), the inner values rounded to bf16 once
    (half a step), fp32 sums over the rank, an activation of slope at most
    1.13 that adds 2^-20, one rounding of the result."""
    half = 2.0 ** -8
    x, w, down, up, ids = (t.cpu() for t in (x, w, down, up, ids))
    k = x.shape[-1]
    rows = x.double().reshape(-1, k)
    per = rows.shape[0] // max(ids.numel(), 1)
    row_ids = ids.reshape(-1).repeat_interleave(per)
    y = rows @ w.double().t()
    bound = rows.abs() @ w.double().abs().t() * k * 2.0 ** -24
    for i in range(down.shape[0]):
        mine = row_ids == i
        a, b = down[i].double(), up[i].double()
        s = 1.0 if scales is None else float(scales[i])
        inner = rows[mine] @ a.t() * s
        slack = inner.abs() * half + (rows[mine].abs() @ a.abs().t()
                                      * abs(s) * (k + 2) * 2.0 ** -24)
        y[mine] += inner @ b.t()
        bound[mine] += slack @ b.abs().t() + (
            inner.abs() @ b.abs().t() * (b.shape[1] + 2) * 2.0 ** -24)
    if bias is not None:
        y = y + bias.cpu().double()
    bound = bound + y.abs() * 4 * 2.0 ** -24
    if act == "gelu":
        y = y * torch.special.ndtr(y)
    elif act == "tanh":
        y = torch.tanh(y)
    if act is not None:
        bound = bound * 1.13 + 2.0 ** -20
    if residual is not None:
        y = y + residual.cpu().double().reshape(y.shape)
    bound = bound + y.abs() * half + 1e-30
    assert out.dtype == torch.bfloat16
    err = (out.double().cpu().reshape(y.shape) - y).abs()
    worst = (err / bound).max().item()
    assert worst <= 1.0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape,k,n,rank,count", [
    ((1, 1), 64, 16, 8, 1),
    ((8, 1), 1024, 500, 16, 8),      # one row of each request
    ((70, 1), 256, 130, 16, 70),
    ((5, 13), 192, 257, 8, 3),       # requests that end inside a tile
    ((3, 197), 128, 96, 64, 2),
    ((4, 33), 72, 61, 3, 4),         # nothing a multiple of 8
    ((2, 9), 37, 23, 5, 2),
    ((2, 40), 320, 48, 100, 2),
    ((2, 20), 64, 40, 256, 2),
    ((9, 150), 2048, 70, 24, 3),     # the tiles of long rows
    ((11, 197), 64, 3200, 16, 3),    # of many wide rows
    ((8, 200), 128, 4100, 8, 3),
    ((17, 197), 2048, 3100, 8, 5),
])
def test_adapter_matches_exact(device, shape, k, n, rank, count):
    x, w, down, up = make(shape, k, n, rank, count, device)
    ids = torch.randperm(shape[0]).int() % (count + 1) - 1
    ids = ids.to(device)
    scales = (torch.rand(count) + 0.5).to(device)
    bias = torch.randn(n).bfloat16().to(device)
    res = torch.randn(*shape, n).bfloat16().to(device)
    args = (x, w, down, up, ids)
    out = ops.adapter_linear(*args)
    assert out.shape == shape + (n,)
    check(out, *args)
    for kw in (dict(bias=bias, scales=scales),
               dict(bias=bias, act="gelu", residual=res, scales=scales),
               dict(act="tanh")):
        check(ops.adapter_linear(*args, **kw), *args, **kw)
    # one id a row, the requests' rows mixed
    ids = (torch.arange(shape[0] * shape[1]) * 7 % (count + 2) - 1).int()
    ids = ids.reshape(shape).to(device)
    check(ops.adapter_linear(x, w, down, up, ids, bias, scales=scales),
          x, w, down, up, ids, bias=bias, scales=scales)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape,k,n,rank,count", [
    ((11, 197), 72, 3200, 12, 3),
    ((17, 197), 64, 3100, 3, 4),
    ((8, 200), 128, 4100, 70, 3),
    ((3, 100), 64, 300, 1, 5),
    ((2, 90), 136, 70, 255, 2),
    ((6, 400), 64, 90, 33, 4),       # inner values of each kernel
    ((3, 512), 72, 40, 12, 7),
])
def test_adapter_odd_ranks(device, shape, k, n, rank, count):
    x, w, down, up = make(shape, k, n, rank, count, device)
    ids = (torch.arange(shape[0]) % (count + 1) - 1).int().to(device)
    args = (x, w, down, up, ids)
    check(ops.adapter_linear(*args), *args)
    ids = (torch.arange(shape[0] * shape[1]) * 5 % (count + 2) - 1).int()
    args = (x, w, down, up, ids.reshape(shape).to(device))
    check(ops.adapter_linear(*args, act="gelu"), *args, act="gelu")


@pytest.mark.parametrize("device", DEVICES)
def test_adapter_ids_outside(device):
    """Rows without an adapter get the plain projection, bit for bit."""
    x, w, down, up = make((6, 21), 128, 192, 16, 2, device)
    bias = torch.randn(192).bfloat16().to(device)
    ids = torch.tensor([-1, 0, 2, 1, -2 ** 31, 2 ** 31 - 1],
                       dtype=torch.int32, device=device)
    out = ops.adapter_linear(x, w, down, up, ids, bias)
    check(out, x, w, down, up, ids, bias=bias)
    none = torch.full_like(ids, -1)
    plain = ops.adapter_linear(x, w, down, up, none, bias)
    for i in (0, 2, 4, 5):
        assert torch.equal(out[i], plain[i])
    for empty in (down[:0], up[:0]), (down[:, :0], up[..., :0]):
        assert torch.equal(ops.adapter_linear(x, w, *empty, ids, bias), plain)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(8, 1), (6, 21), (24, 5)])
def test_adapter_isolation(device, shape):
    """Another request's infinite or undefined adapter, scale or input
    reaches no row but its own."""
    x, w, down, up = make(shape, 128, 192, 16, 3, device)
    scales = torch.ones(3, device=device)
    ids = (torch.arange(shape[0]) % 4 - 1).int().to(device)
    want = ops.adapter_linear(x, w, down, up, ids, scales=scales)
    down[1, 3, 5] = float("inf")
    up[1, 100] = float("nan")
    up[1, 7, 2] = float("inf")
    scales[2] = float("nan")
    x[0, 0, 0] = float("inf")
    out = ops.adapter_linear(x, w, down, up, ids, scales=scales)
    for i in range(shape[0]):
        if int(ids[i]) in (-1, 0):
            keep = slice(1, None) if i == 0 else slice(None)
            assert torch.equal(out[i, keep], want[i, keep])
        else:
            assert not torch.isfinite(out[i]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape,rank", [
    ((4, 150), 16), ((7, 300), 64), ((5, 1000), 16), ((30, 20), 12),
])
def test_adapter_isolation_of_many_rows(device, shape, rank):
    """The same where tiles of the matrix unit hold rows of several
    requests."""
    x, w, down, up = make(shape, 72, 136, rank, 3, device)
    ids = (torch.arange(shape[0]) % 4 - 1).int().to(device)
    want = ops.adapter_linear(x, w, down, up, ids)
    down[1, 3, 5] = float("inf")
    up[1] = float("nan")
    x[2, 1, 0] = float("nan")
    out = ops.adapter_linear(x, w, down, up, ids)
    clean = torch.ones(shape[0], dtype=torch.bool)
    clean[2::4] = False             # requests of adapter 1
    assert torch.equal(out[clean], want[clean])
    assert out[2].isnan().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [4, 96])
def test_adapter_gelu_range(device, rows):
    """The activation alone over its range: an identity projection, whose
    sums are exact. Far out its value is exp(-x^2 / 2) times a slow factor;
    an exponent of up to 2^7 that is rounded to 2^-24 of itself moves it by
    2^-17, the rest by less than 2^-18. Then it is rounded once; results
    below the smallest normal number may be anything below it."""
    values = torch.cat((torch.linspace(-12, 12, 200),
                        torch.tensor([0.0, -0.0, 1e-3, -1e-3, 30.0, -30.0,
                                      3e38, -3e38])))
    w = values.bfloat16().reshape(-1, 1).to(device)
    x = torch.ones(rows, 1, device=device).bfloat16()
    down = torch.zeros(1, 8, 1, device=device).bfloat16()
    up = torch.zeros(1, w.shape[0], 8, device=device).bfloat16()
    ids = torch.zeros(rows, dtype=torch.int32, device=device)
    out = ops.adapter_linear(x, w, down, up, ids, act="gelu").double().cpu()
    v = w.double().cpu().reshape(-1)
    ref = v * 0.5 * torch.special.erfc(-v * 0.5 ** 0.5)
    bound = ref.abs() * (2.0 ** -8 + 2.0 ** -16) + 2.0 ** -126
    worst = ((out - ref).abs() / bound).max().item()
    assert worst <= 1.0


@pytest.mark.parametrize("device", DEVICES)
def test_adapter_strides(device):
    x, w, down, up = make((4, 10), 96, 80, 12, 3, device)
    ids = torch.tensor([2, 0, -1, 1], dtype=torch.int32, device=device)
    want = ops.adapter_linear(x, w, down, up, ids)

    def spread(t, at):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 7, dtype=t.dtype,
                           device=device)
        wide[..., at:at + t.shape[-1]] = t
        return wide[..., at:at + t.shape[-1]]
    got = ops.adapter_linear(spread(x, 3), spread(w, 1), spread(down, 5),
                             spread(up, 7), ids.repeat_interleave(2)[::2])
    assert torch.equal(got, want)
    got = ops.adapter_linear(x.transpose(0, 1).contiguous().transpose(0, 1),
                             w, down, up, ids)
    assert torch.equal(got, want)
    flat = ops.adapter_linear(x.reshape(-1, 96), w, down, up,
                              ids.repeat_interleave(10))
    assert torch.equal(flat.view_as(want), want)
    one = ops.adapter_linear(x[1, 2], w, down, up, ids[1])
    check(one, x[1, 2].unsqueeze(0), w, down, up, ids[1:2])


@pytest.mark.parametrize("device", DEVICES)
def test_adapter_empty(device):
    x, w, down, up = make((2, 3), 64, 32, 8, 2, device)
    ids = torch.zeros(2, dtype=torch.int32, device=device)
    assert ops.adapter_linear(x[:, :0], w, down, up, ids).shape == (2, 0, 32)
    assert ops.adapter_linear(x[:0], w, down, up, ids[:0]).shape == (0, 3, 32)
    assert ops.adapter_linear(x, w[:0], down, up[:, :0], ids).shape \
        == (2, 3, 0)


@pytest.mark.parametrize("device", DEVICES)
def test_adapter_refusals(device):
    x, w, down, up = make((2, 3), 64, 32, 8, 2, device)
    ids = torch.zeros(2, dtype=torch.int32, device=device)
    good = dict(x=x, weight_nk=w, down=down, up=up, ids=ids)
    big = torch.zeros(2, 257, 64, dtype=x.dtype, device=device)
    bad = [
        dict(x=x.half()), dict(weight_nk=w.float()), dict(ids=ids.long()),
        dict(ids=ids[:1]), dict(ids=ids.unsqueeze(1)), dict(x=x[..., :32]),
        dict(down=down[:1]), dict(up=up[:, :8]), dict(up=up[..., :4]),
        dict(weight_nk=w[0]), dict(down=big, up=big.transpose(1, 2)[:, :32]),
        dict(bias=w[0]), dict(bias=w[:, 0].float()), dict(residual=x),
        dict(scales=torch.ones(3, device=device)),
        dict(scales=torch.ones(2, device=device).half()),
        dict(act="relu"), dict(x=x.clone().requires_grad_()),
        dict(up=up.clone().requires_grad_()),
    ]
    ops.adapter_linear(**good)
    for change in bad:
        with pytest.raises((TypeError, ValueError)):
            ops.adapter_linear(**{**good, **change})
    with torch.no_grad():
        ops.adapter_linear(**{**good, "x": x.clone().requires_grad_()})
    if device == "cuda":
        for name in ("weight_nk", "ids"):
            with pytest.raises(ValueError):
                ops.adapter_linear(**{**good, name: good[name].cpu()})


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(8, 1), (8, 197)])
def test_adapter_graph(shape):
    x, w, down, up = make(shape, 256, 320, 16, 4, "cuda")
    ids = torch.zeros(shape[0], dtype=torch.int32, device="cuda")
    ops.adapter_linear(x, w, down, up, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.adapter_linear(x, w, down, up, ids)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        ids.copy_((torch.arange(shape[0]) + i) % 5 - 1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.adapter_linear(x, w, down, up, ids))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,rank", [((8, 1), 16), ((3, 100), 12),
                                        ((8, 197), 64)])
def test_adapter_streams(shape, rank):
    """Calls on two streams at once, whose inner values are their own."""
    sets = [make(shape, 512, 640, rank, 4, "cuda", seed=i) for i in range(2)]
    ids = (torch.arange(shape[0]) % 5 - 1).int().cuda()
    want = [ops.adapter_linear(*s, ids, act="gelu") for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                outs.append(ops.adapter_linear(*s, ids, act="gelu"))
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            assert torch.equal(out, ref)


@pytest.mark.gpu
def test_adapter_refuses_more_than_a_launch_takes():
    x, w, down, up = make((1,), 8, 8, 40, 1, "cuda")
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    for batch, length in ((2 ** 29, 1), (2 ** 22, 128), (2 ** 22, 65)):
        with pytest.raises(ValueError):
            ops.adapter_linear(x.expand(batch, length, 8), w, down, up,
                               ids.expand(batch))
    with pytest.raises(ValueError):
        ops.adapter_linear(x, w[:1].expand(2 ** 27, 8), down,
                           up[:, :1].expand(1, 2 ** 27, 40), ids)


def kernels_of(rows, n, rank, per):
    """The kernels that the rules on sizes choose: the product's tile as
    columns by rows, and the inner values'."""
    def blocks(wide, high):
        return -(-n // wide) * -(-rows // high)
    pad = 32 if rank <= 32 else -(-rank // 64) * 64
    tile = "step" if rows <= 64 else \
        (256, 256) if blocks(256, 256) >= 200 else \
        (256, 128) if blocks(256, 128) >= 160 else \
        (128, 128) if blocks(128, 128) >= 128 else (64, 64)
    if rows * max(pad, 64) <= 512 * 64:
        inner = "row"
    elif rows * pad >= 2048 * 64 * (2 if rank <= 32 else 1):
        inner = "lds32" if rank <= 32 else "lds64"
    else:
        inner = 16 if rank <= 16 else 32 if rank <= 32 else 64
    return tile, inner


VARIANTS = [
    # batch, rows of each, K, N, rank: tile, inner
    (19, 197, 72, 3500, 8, (256, 256), 16),
    (4, 1031, 200, 3333, 40, (256, 256), "lds64"),
    (42, 200, 136, 1801, 28, (256, 256), "lds32"),
    (12, 197, 136, 2300, 70, (256, 128), "lds64"),
    (9, 300, 68, 2050, 24, (256, 128), 32),
    (8, 197, 200, 2300, 8, (128, 128), 16),
    (7, 211, 72, 1537, 44, (128, 128), 64),
    (5, 257, 331, 2001, 3, (128, 128), 16),
    (8200, 1, 72, 270, 12, (128, 128), "lds32"),
    (41, 201, 67, 45, 32, (64, 64), "lds32"),
    (5, 100, 264, 310, 60, (64, 64), "row"),
    (3, 300, 100, 200, 90, (64, 64), 64),
    (3, 700, 40, 130, 200, (64, 64), "lds64"),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("batch,length,k,n,rank,tile,inner", VARIANTS)
def test_adapter_variants(device, batch, length, k, n, rank, tile, inner):
    """Every tile of the product with every odd end: rows, columns, K, rank;
    ids by item and mixed row by row."""
    assert kernels_of(batch * length, n, rank, length) == (tile, inner)
    count = 5
    x, w, down, up = make((batch, length), k, n, rank, count, device)
    bias = torch.randn(n).bfloat16().to(device)
    res = torch.randn(batch, length, n).bfloat16().to(device)
    scales = (torch.rand(count) + 0.5).to(device)
    ids = (torch.arange(batch) * 3 % (count + 1) - 1).int().to(device)
    args = (x, w, down, up, ids)
    check(ops.adapter_linear(*args), *args)
    kw = dict(bias=bias, act="gelu", residual=res, scales=scales)
    check(ops.adapter_linear(*args, **kw), *args, **kw)
    ids = (torch.arange(batch * length) * 7 % (count + 2) - 1).int()
    args = args[:4] + (ids.reshape(batch, length).to(device),)
    kw = dict(bias=bias, scales=scales)
    check(ops.adapter_linear(*args, **kw), *args, **kw)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("batch,length,k,n,rank,tile,inner", VARIANTS)
def test_adapter_variants_isolate(device, batch, length, k, n, rank, tile,
                                  inner):
    """Undefined values of one adapter, one scale and one row in each of
    them, ids by item and mixed row by row: every other row is as
    without them."""
    count = 4
    x, w, down, up = make((batch, length), k, n, rank, count, device)
    scales = torch.ones(count, device=device)
    by_item = (torch.arange(batch) % (count + 1) - 1).int()
    by_row = (torch.arange(batch * length) * 3 % (count + 1) - 1).int()
    for ids in (by_item, by_row.reshape(batch, length)):
        row_ids = ids.reshape(batch, -1).expand(batch, length)
        ids = ids.to(device)
        want = ops.adapter_linear(x, w, down, up, ids, scales=scales)
        x2, down2, up2, scales2 = (t.clone() for t in (x, down, up, scales))
        down2[1, rank - 1, k - 1] = float("inf")
        up2[1] = float("nan")
        scales2[2] = float("nan")
        x2[1, length // 2, k // 2] = float("nan")
        out = ops.adapter_linear(x2, w, down2, up2, ids, scales=scales2)
        clean = (row_ids != 1) & (row_ids != 2)
        bad = ~clean
        clean[1, length // 2] = False
        bad[1, length // 2] = True
        assert torch.equal(out[clean], want[clean])
        assert out[bad].isnan().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [16, 17, 32, 33, 64, 65, 129])
@pytest.mark.parametrize("k,n,rank", [(1, 1, 1), (9, 7, 2), (40, 8, 8)])
def test_adapter_smallest(device, rows, k, n, rank):
    """One column, one rank, one K, at the numbers of rows where the kernels
    change; items of more than one dimension."""
    x, w, down, up = make((rows, 1, 2), k, n, rank, 3, device)
    res = torch.randn(rows, 1, 2, n).bfloat16().to(device)
    ids = (torch.arange(rows) % 4 - 1).int().to(device)
    out = ops.adapter_linear(x, w, down, up, ids, act="tanh", residual=res)
    check(out, x, w, down, up, ids, act="tanh", residual=res)
    each = ids.reshape(rows, 1, 1).expand(rows, 1, 2)
    assert torch.equal(ops.adapter_linear(x, w, down, up, each, act="tanh",
                                          residual=res), out)
    half = ops.adapter_linear(x[:, :, 0], w, down, up, ids)
    check(half, x[:, :, 0], w, down, up, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 100, 3000])
@pytest.mark.parametrize("rank", [64, 60])
def test_adapter_far_stacks(rows, rank):
    """Adapters behind 2^32 bytes of their stacks."""
    k, n = 1032, 1096
    count = 2 ** 31 // (n * rank) + 40
    x, w, down, up = make((rows,), k, n, rank, 3, "cuda")
    ids = (torch.arange(rows) % 4 - 1).int().cuda()
    want = ops.adapter_linear(x, w, down, up, ids)
    far_down = torch.empty(count, rank, k, dtype=x.dtype, device="cuda")
    far_up = torch.empty(count, n, rank, dtype=x.dtype, device="cuda")
    far_down[-3:], far_up[-3:] = down, up
    assert far_up[-3].storage_offset() > 2 ** 31
    far = torch.where(ids >= 0, ids + (count - 3), ids)
    assert torch.equal(ops.adapter_linear(x, w, far_down, far_up, far), want)
