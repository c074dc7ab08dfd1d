"""Paged attention at the ends of what q, K and their products may be: large scores, small and large q."""
import pytest
import torch
from test_paged_gpu import make_cache, put

from amd_c_b200 import kernels as K

pytestmark = pytest.mark.gpu


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
