"""Paged attention at the ends of what q, K and their products may be: large scores, small and large q."""
import pytest
import torch
from test_paged_gpu import attention, make_cache, put

from amd_c_b200 import kernels as K


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", [(torch.half, 3000.0), (torch.float, 3000.0), (torch.float, 60000.0)])
@pytest.mark.parametrize("heads,kv_heads,hd,lens", [(8, 1, 128, [3000, 1, 77, 500]), (8, 2, 64, [1500] * 5), (4, 4, 32, [20000]), (32, 8, 128, [40] * 70), (6, 2, 64, [5, 33, 9] * 60)])
def test_large_scores(cuda, dtype, size, heads, kv_heads, hd, lens):
    """Finite scores of 10^7 to 10^10, one position of each row a fifth ahead of the others: their weights are exactly 1 and 0, so the output is that
    position's V to the last bit, in one part or many, a warp's own units too."""
    gen = torch.Generator(device=cuda).manual_seed(hd + len(lens))
    kp, vp, table = make_cache(gen, lens, kv_heads, hd, 16, dtype)
    q, want = torch.empty(len(lens), heads, hd, device=cuda), torch.empty(len(lens), heads, hd, device=cuda)
    group = heads // kv_heads
    for s, n in enumerate(lens):
        way = (0.5 + 0.5 * torch.rand(kv_heads, hd, device=cuda, generator=gen)) * (torch.randint(0, 2, (kv_heads, hd), device=cuda, generator=gen) * 2 - 1)
        far = 0.2 + 0.6 * torch.rand(n, kv_heads, device=cuda, generator=gen)
        first = torch.randint(0, n, (kv_heads,), device=cuda, generator=gen)
        far[first, torch.arange(kv_heads, device=cuda)] = 1.0
        v = torch.randn(n, kv_heads, hd, device=cuda, generator=gen).to(dtype)
        put(kp, table, s, size * far[:, :, None] * way), put(vp, table, s, v)
        q[s] = size * (way.repeat_interleave(group, 0) * (0.6 + 0.4 * torch.rand(heads, 1, device=cuda, generator=gen)))
        want[s] = v[first, torch.arange(kv_heads, device=cuda)].float().repeat_interleave(group, 0)
    out, _ = K.attn_decode_paged(q.view(len(lens), -1), kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=cuda), heads, K.PagedScratch(heads, kv_heads, hd, cuda))
    assert torch.equal(out.view_as(want), want)


def filled(lens, heads, kv_heads, hd, dtype, k_of, seed=0):
    """q of 1.5 and a cache whose K rows are k_of(shape, generator) (nothing between what it gives and the pool is rounded but to the pool's type)."""
    gen = torch.Generator(device="cuda").manual_seed(seed + hd + len(lens))
    kp, vp, table = make_cache(gen, lens, kv_heads, hd, 16, dtype)
    for s, n in enumerate(lens):
        put(kp, table, s, k_of((n, kv_heads, hd), gen)), put(vp, table, s, torch.randn(n, kv_heads, hd, device="cuda", generator=gen))
    q = torch.randn(len(lens), heads * hd, device="cuda", generator=gen) * 1.5
    return q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def attend(q, kp, vp, table, n, heads):
    return K.attn_decode_paged(q, kp, vp, table, n, heads, K.PagedScratch(heads, kp.shape[1], kp.shape[3], "cuda"), quant=False)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.half, torch.float])
@pytest.mark.parametrize("heads,kv_heads,hd,lens", [(8, 1, 128, [3000, 1, 77, 500]), (12, 1, 64, [900, 20]), (4, 2, 32, [20000]), (32, 8, 128, [40] * 70)])
def test_powers_of_two_change_nothing(cuda, dtype, heads, kv_heads, hd, lens):
    """q times 2^x and K over 2^x have the same scores; K of 7 bits, so that 2^-17 to 2^14 of it are halves: the same bits come out.
    But where all of K is below 2^-14, f16's smallest normal: the tensor cores align products by their operands' exponents, which end there, and cut off
    what they would of products with |k| = 2^-14, of a sum up to 2^-23 in each of hd / 16 accumulations. A score is off by 2^-19 of those products' magnitudes, the
    other by 2^-19 of its own, a weighted mean of v by twice that times the largest |v| (as in check_attention)."""
    q, kp, vp, table, n = filled(lens, heads, kv_heads, hd, dtype, lambda shape, gen: torch.randint(-64, 65, shape, device="cuda", generator=gen) / 32.0)
    want = attend(q, kp, vp, table, n, heads)
    assert torch.isfinite(want).all()
    for x in (-14, -12, -5, 1, 10, 17):
        got = attend(q * 2.0 ** x, kp * 2.0 ** -x, vp, table, n, heads)
        if dtype == torch.half and 2.0 ** (1 - x) < 2.0 ** -14:
            _, own = attention(q, kp, vp, table, n, heads)
            size = q.view(len(lens), heads, hd).abs().sum(2).double() * (2.0 ** (x - 14) / hd ** 0.5)
            v = torch.stack([torch.cat([vp[int(table[s, c])] for c in range(-(-m // 16))], 1)[:, :m].abs().amax((1, 2)) for s, m in enumerate(lens)]).double()
            bound = own + ((size + 1) * v.repeat_interleave(heads // kv_heads, 1))[:, :, None]
            assert ((got - want).abs().view(len(lens), heads, hd) <= 2 * 2.0 ** -19 * bound).all(), x
        else:
            assert torch.equal(got, want), x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.half, torch.float])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_any_finite_q(cuda, dtype, hd):
    """Heads of one KV head with q of very different sizes. Far below what matters, or zeros: the mean of V, to sums in fp32 (at most 64 additions
    one after the other, each off by 2^-24 of a sum: 2^-18 of the largest |v|). Far above half's range, up to where products end being floats: the position whose K lies along
    q has all the weight."""
    heads, lens = 4, [600, 17]
    q, kp, vp, table, n = filled(lens, heads, 1, hd, dtype, lambda shape, gen: torch.randint(-64, 65, shape, device="cuda", generator=gen) / 32.0)
    way = torch.sign(q.view(2, heads, hd)[:, :1])
    q = way * torch.tensor([1e-35, 2.0 ** 100, 0.0, 2.0 ** 40], device="cuda")[:, None] * torch.rand(2, 1, hd, device="cuda").add(0.5)
    q[1, 1] *= 2.0 ** 16  # (128 products of it and 2 stay below 2^128)
    at = [511, 3]
    for s, p in enumerate(at):
        kp[int(table[s, p // 16]), 0, p % 16] = (2 * way[s, 0]).to(dtype)
    out = attend(q.view(2, -1), kp, vp, table, n, heads).view(2, heads, hd)
    for s, m in enumerate(lens):
        v = torch.cat([vp[int(table[s, c]), 0] for c in range(-(-m // 16))])[:m]
        for h in (0, 2):
            assert ((out[s, h].double() - v.double().mean(0)).abs() <= 2.0 ** -18 * v.abs().max()).all()
        for h in (1, 3):
            assert torch.equal(out[s, h], v[at[s]].float())


TIGHT = 2e-6


def error(out, want):
    """The error's norm against the output's: over all, and the worst of a head."""
    e = (out - want).double()
    return float(e.norm() / want.norm()), float((e.norm(dim=-1) / want.norm(dim=-1)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.half, torch.float])
@pytest.mark.parametrize("size,hd", [(1.5, 128), (1.5, 64), (1.5, 32), (0.01, 128), (1e-3, 128), (1e-4, 128), (1e-3, 32)])
def test_error_norm(cuda, dtype, size, hd):
    """Random q and K with scores of about 1.5. A weight's own error: a score's, sqrt(hd) products each off by up to 2^-22 of 1.5 / sqrt(hd) (q in two f16
    terms; with the float cache 2^-24 of the partial sums) and four accumulations that cut off up to 2^-23 of 1.5 each, together some 6e-7; the
    exponential's 2^-22; its own split's 2^-23. They are independent from position to position, as the outputs' terms are, so the output's relative
    error is about the weights': 1e-6 with the fp32 sums, TIGHT with room for half as much again and more. A head, of few terms, may have twice that."""
    q, kp, vp, table, n = filled([500, 3000, 129], 8, 2, hd, dtype, lambda shape, gen: torch.randn(shape, device="cuda", generator=gen) * min(1.5 / size, 9000.0))
    q = q / 1.5 * size
    want, _ = attention(q, kp, vp, table, n, 8)
    whole, head = error(attend(q, kp, vp, table, n, 8).view(3, 8, hd), want)
    assert whole <= TIGHT and head <= 2 * TIGHT, (whole, head)


@pytest.mark.parametrize("drop", ["q", "weights"])
def test_error_norm_sees_a_lost_low_term(drop):
    """The same inputs in 64 bits, but q or the weights in one f16 term: the check above must not pass them."""
    gen = torch.Generator().manual_seed(1)
    q, k, v = torch.randn(8, 128, generator=gen) * 1.5, torch.randn(8, 500, 128, generator=gen).half().double(), torch.randn(8, 500, 128, generator=gen).half().double()

    def out(q, round_weights):
        w = torch.softmax(torch.einsum("hd,hnd->hn", q, k) / 128 ** 0.5, 1)
        w = w / w.amax(1, keepdim=True)
        w = (w * 2.0 ** 15).half().double() if round_weights else w
        return torch.einsum("hn,hnd->hd", w / w.sum(1, keepdim=True), v)

    want = out(q.double(), False)
    whole, head = error(out((q.half() if drop == "q" else q).double(), drop == "weights"), want)
    assert whole > 10 * TIGHT and head > 10 * TIGHT
    assert max(error(out(q.double(), False), want)) == 0.0
