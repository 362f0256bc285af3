"""The operators together, as the attention half of a block uses them: each
tenant's adapters on the projections, rotary positions on the rotary columns
of the queries and on the shared key, then attention over the latent vectors -
expanded for the prompt, absorbed over a paged cache for its last tokens."""
import pytest
import torch

from pipeedge_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]

HIDDEN, HEADS, LATENT, NOPE, ROPE, PAGE = 192, 4, 256, 64, 32, 16


def make_block(device):
    torch.manual_seed(11)
    n, rank = 3, 8

    def weight(rows, cols, std=1.0):
        return (torch.randn(rows, cols) * std * cols ** -0.5).bfloat16() \
            .to(device)

    def adapters(rows, cols):
        return ((torch.randn(n, rank, cols) * cols ** -0.5).bfloat16()
                .to(device),
                (torch.randn(n, rows, rank) * 0.2).bfloat16().to(device))
    q_out, kv_out = HEADS * (NOPE + ROPE), LATENT + ROPE
    return dict(wq=weight(q_out, HIDDEN), wkv=weight(kv_out, HIDDEN),
                aq=adapters(q_out, HIDDEN), akv=adapters(kv_out, HIDDEN),
                up=weight(HEADS * 2 * NOPE, LATENT))


def project(block, x, positions, ids, freqs):
    """q [B, S, H, NOPE + ROPE] and cache rows [B, S, LATENT + ROPE]."""
    b, s, _ = x.shape
    q = ops.adapter_linear(x, block["wq"], *block["aq"], ids)
    rows = ops.adapter_linear(x, block["wkv"], *block["akv"], ids)
    q = q.view(b, s, HEADS, NOPE + ROPE)
    ops.rotary_(q[..., NOPE:], positions, freqs,
                rows[..., LATENT:].unsqueeze(2), interleaved=True)
    return q, rows


@pytest.mark.parametrize("device", DEVICES)
def test_block_expanded_and_absorbed(device):
    lengths, steps = [37, 5, 64, 18], 2
    b, s = len(lengths), max(lengths)
    block = make_block(device)
    freqs = ops.rotary_frequencies(ROPE, device=device)
    x = torch.randn(b, s, HIDDEN).bfloat16().to(device)
    ids = torch.tensor([0, 2, -1, 1], dtype=torch.int32, device=device)
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    positions = torch.arange(s, device=device).expand(b, s).contiguous()
    scale = (NOPE + ROPE) ** -0.5

    # the prompt in expanded form
    q, rows = project(block, x, positions, ids, freqs)
    kv = ops.linear(rows[..., :LATENT].contiguous(), block["up"])
    kv = kv.view(b, s, HEADS, 2 * NOPE)
    out = ops.latent_attention(q, kv, rows[..., LATENT:], causal=True,
                               lengths=n)

    # its last tokens in absorbed form, over the same rows in pages; the
    # tokens are projected by themselves, as a step does it
    table = torch.randperm(b * 4).int().view(b, 4).to(device)
    cache = torch.zeros(b * 4, PAGE, LATENT + ROPE, dtype=x.dtype,
                        device=device)
    cache.view(b * 4, -1)[table.long().view(-1)] = \
        rows.reshape(b * 4, -1).to(cache.dtype)
    last = (n.long().unsqueeze(1) - steps + torch.arange(
        steps, device=device))
    pick = last.unsqueeze(-1)
    q_step, rows_step = project(
        block, x.gather(1, pick.expand(-1, -1, HIDDEN)), last, ids, freqs)
    # an fp32 sum of the same terms in another order, rounded: one step apart
    same = rows.gather(1, pick.expand(-1, -1, LATENT + ROPE)).float()
    assert ((rows_step.float() - same).abs()
            <= same.abs() * 2.0 ** -7 + 2.0 ** -8).all()
    q_step = q.gather(1, pick.unsqueeze(-1).expand(
        -1, -1, HEADS, NOPE + ROPE))
    up = block["up"].double().view(HEADS, 2 * NOPE, LATENT)
    absorbed = torch.einsum("bshd,hdr->bshr", q_step[..., :NOPE].double(),
                            up[:, :NOPE])
    q_abs = torch.cat((absorbed.to(x.dtype), q_step[..., NOPE:]), dim=-1)
    latent = ops.latent_cache_attention(q_abs, cache, table, n,
                                        latent_dim=LATENT, scale=scale)
    got = torch.einsum("bshr,hdr->bshd", latent.double(), up[:, NOPE:])
    want = out.gather(1, pick.unsqueeze(-1).expand(
        -1, -1, HEADS, NOPE)).double()

    # The forms differ by independent bf16 roundings, each uniform in half a
    # step (2^-8 relative at most, so a variance of 2^-16 / 3 of its square):
    # the absorbed query and the expanded keys, which move the scores; the
    # weights of both forms and the expanded values; the latent sums; the
    # result. Their variances add up to sigma^2, and the root mean square
    # difference over thousands of values is at most that, which a factor of
    # two leaves room for.
    var = 2.0 ** -16 / 3
    for i, length in enumerate(lengths):
        c = rows[i, :length, :LATENT].double()
        keys = torch.einsum("tr,hdr->htd", c, up[:, :NOPE])
        values = torch.einsum("tr,hdr->htd", c, up[:, NOPE:])
        rope = rows[i, :length, LATENT:].double()
        for j in range(steps):
            seen = length - steps + j + 1
            qn, qr = q_step[i, j, :, :NOPE].double(), q_step[
                i, j, :, NOPE:].double()
            k, v = keys[:, :seen], values[:, :seen]
            score = (torch.einsum("hd,htd->ht", qn, k)
                     + qr @ rope[:seen].t()) * scale
            w = torch.softmax(score, -1)
            mean = torch.einsum("ht,htd->hd", w, v)
            moved = scale ** 2 * var * (
                torch.einsum("hr,tr->ht", absorbed[i, j] ** 2, c[:seen] ** 2)
                + torch.einsum("hd,htd->ht", qn ** 2, k ** 2))
            lat = torch.einsum("ht,tr->hr", w, c[:seen])
            sigma2 = torch.einsum("ht,htd->hd", w ** 2 * moved,
                                  (v - mean.unsqueeze(1)) ** 2)
            sigma2 += var * (
                3 * torch.einsum("ht,htd->hd", w ** 2, v ** 2) + mean ** 2
                + torch.einsum("hr,hdr->hd", lat ** 2, up[:, NOPE:] ** 2))
            diff = (got[i, j] - want[i, j]).pow(2).mean().sqrt()
            assert diff <= 2.0 * sigma2.mean().sqrt(), (i, j)
            assert diff < 0.02 * want[i, j].pow(2).mean().sqrt()
