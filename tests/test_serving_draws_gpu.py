"""Tokens of a batched decode over pages against its 64-bit sequences, every one of them judged: where the device's token is another one, the
64-bit draw must have been so near to a border that the difference of the logits accounts for it."""
import numpy as np
import pytest
import torch
from test_sample_gpu import draw
from test_serving_gpu import HD, HEADS, KV_HEADS, LAYERS, N_CTX, PAGE, VOCAB, DIM, Host, model, tables

from amd_c_b200 import kernels as K
from amd_c_b200._lib import MAT_F32


def margin(x, u, temp, k, p, m):
    """How far, at least, a logit of x has to move (all of them by as much, either way) for another token to be drawn: half the gaps between
    neighbours in the order that the greedy choice, top_k and the end of top_p's run go by; where running sums of the weights pass p, half the weights' sum away, or u, the
    move that shifts the quotient F = before / all by the distance: each of the two parts by a factor of exp(2 d / temp) against the other at most, F
    by 2 d / temp F (1 - F), so d / (2 temp); where a weight is next to min_p, the move that takes it there."""
    n = len(x)
    order = np.argsort(-x, kind="stable")
    top = x[order]
    if not temp > 0:
        return (top[0] - top[1]) / 2
    near = np.inf
    kept = n
    if 0 < k < n:
        kept, near = k, (top[k - 1] - top[k]) / 2
    w = np.exp((top[:kept] - top[0]) / temp)
    if p < 1:
        before = (np.cumsum(w) - w) / w.sum()
        near = min(near, np.abs(before[1:] - p).min() * 2 * temp)
        w = w[: max(1, int((before < p).sum()))]
        if len(w) < kept:
            near = min(near, (top[len(w) - 1] - top[len(w)]) / 2)
    if m > 0:
        near = min(near, np.abs(np.log(w) - np.log(m)).min() * temp / 2)
        w = w[w >= m]
    by_index = np.argsort(order[: len(w)])
    run = np.cumsum(w[by_index])[:-1] / w.sum()
    return min(near, np.abs(run - u).min() * 2 * temp) if len(run) else near


@pytest.mark.parametrize("temp,k,p,m", [(0.9, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 12, 1.0, 0.02), (0.7, 0, 0.8, 0.05), (1.0, 0, 1.0, 0.0), (1.5, 40, 0.9, 0.0)])
def test_margin_bounds_what_moves_a_draw(temp, k, p, m):
    """In 64 bits: logits moved by less than the margin draw the same token; moved by some times as much they draw another one often."""
    rng = np.random.default_rng(int(100 * (temp + p)))
    same = other = 0
    for _ in range(300):
        x, u = rng.standard_normal(200) * 3, rng.random()
        own, d = draw(x.copy(), u, temp, k, p, m)[0], margin(x, u, temp, k, p, m)
        for sign in (rng.choice([-1.0, 1.0], 200), rng.uniform(-1, 1, 200)):
            assert draw(x + 0.999 * d * sign, u, temp, k, p, m)[0] == own
            same += 1
            other += draw(x + 40 * d * sign, u, temp, k, p, m)[0] != own
    assert same == 600 and other > 30


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.half, torch.float])
def test_every_token_of_a_batch(cuda, dtype):
    """Seven sequences of different settings and lengths, padding between them, 24 steps; a sequence is given the device's tokens, and so is its 64-bit one, so that every
    step is judged. The logits differ by `shift` (bounds as in test_serving_gpu); a token may differ only where the margin is within it."""
    rng = np.random.default_rng(8)
    m = model(rng)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    emb, head = K.Mat(MAT_F32, VOCAB, DIM, dev(m["embed"])), K.Mat(MAT_F32, VOCAB, DIM, dev(m["head"]))
    layers = [{n: K.Mat(MAT_F32, a.shape[0], a.shape[1], dev(a)) for n, a in layer.items()} for layer in m["layers"]]
    cos, sin = (dev(t) for t in tables())
    n, steps = 7, 24
    pool = torch.full((n * N_CTX // PAGE, LAYERS, 2, KV_HEADS, PAGE, HD), float("nan"), dtype=dtype, device=cuda)
    table = dev(rng.permutation(n * N_CTX // PAGE).astype(np.int32).reshape(n, -1))
    scratch, err = K.PagedScratch(HEADS, KV_HEADS, HD, cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    settings = [(0.9, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 12, 1.0, 0.02), (0.7, 0, 0.8, 0.05), (1.0, 0, 1.0, 0.0), (1.5, 40, 0.9, 0.0), (0.8, 0, 1.0, 0.1)]
    host, rows = [Host(m, dtype == torch.half) for _ in range(n)], [0, 1, -1, 2, 3, -1, 4, 5, 6]
    seq = torch.tensor(rows, dtype=torch.int32, device=cuda)
    pick = lambda i, dt: torch.tensor([settings[s][i] for s in rows], dtype=dt, device=cuda)  # noqa: E731
    temp, top_k, top_p, min_p = pick(0, torch.float), pick(1, torch.int32), pick(2, torch.float), pick(3, torch.float)
    tok = dev(rng.integers(0, VOCAB, len(rows)).astype(np.int32))
    agree = differ = 0
    for step in range(steps):
        u, pos = rng.random(len(rows), dtype=np.float32), torch.full((len(rows),), step, dtype=torch.int32, device=cuda)
        fed, x = tok.tolist(), K.embed(emb, tok)
        for i, layer in enumerate(layers):
            kp, vp = pool[:, i, 0], pool[:, i, 1]
            q = K.rope_kv_paged(K.gemv(layer["qkv"], x), kp, vp, table, cos, sin, pos, seq, HEADS, KV_HEADS, HD, False, err=err)
            a, _ = K.attn_decode_paged(q, kp, vp, table, pos + 1, HEADS, scratch, seq=seq, quant=False, err=err)
            x = K.gemv(layer["out"], a, res=x)
        logits = K.gemv(head, x)
        tok, _ = K.sample(logits, dev(u), temp, top_k, top_p, min_p)
        drawn, z = tok.tolist(), logits.cpu().numpy().astype(np.float64)
        assert all(0 <= t < VOCAB for t in drawn)
        for r, s in enumerate(rows):
            if s < 0:
                continue
            want = host[s].step(fed[r])
            shift = np.abs(z[r] - want).max()
            assert shift <= (2e-2 if dtype == torch.half else 1e-3), (step, s, shift)
            own = [np.float32(v) if i != 1 else v for i, v in enumerate(settings[s])]
            if drawn[r] == draw(want.copy(), u[r], *own)[0]:
                agree += 1
            else:
                differ += 1
                assert margin(want, float(u[r]), *map(float, own)) <= shift * (1 + 1e-6), (step, s)
    assert int(err) == 0 and agree + differ == n * steps and differ <= n * steps // 10
