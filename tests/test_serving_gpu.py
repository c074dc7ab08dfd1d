"""The operators of a batched decode step together, as a server runs them: embedding, q / k / v product, RoPE with the store into
pages, attention over the pages, output product, logits, draw; sequences that come and go, a page that two of them share."""
import numpy as np
import pytest
import torch
from test_sample_gpu import draw

from amd_c_b200 import kernels as K
from amd_c_b200._lib import MAT_F32

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, HD, PAGE, VOCAB, LAYERS, N_CTX = 8, 2, 32, 16, 503, 2, 96
DIM = HEADS * HD


def model(rng):
    mat = lambda rows, cols, s: (rng.standard_normal((rows, cols)) * s).astype(np.float32)  # noqa: E731
    layers = [dict(qkv=mat((HEADS + 2 * KV_HEADS) * HD, DIM, DIM ** -0.5 * 1.5), out=mat(DIM, DIM, DIM ** -0.5)) for _ in range(LAYERS)]
    return dict(embed=mat(VOCAB, DIM, 1.0), head=mat(VOCAB, DIM, DIM ** -0.5 * 3), layers=layers)


def tables():
    angle = np.arange(N_CTX)[:, None] * 1e4 ** (-np.arange(HD // 2) / (HD // 2))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


class Host:
    """One sequence in 64 bits; the cache rounds to half where the device's does."""

    def __init__(self, m, half):
        self.m, self.half, self.kv = m, half, [([], []) for _ in range(LAYERS)]
        self.cos, self.sin = (t.astype(np.float64) for t in tables())

    def step(self, tok):
        x = self.m["embed"][tok].astype(np.float64)
        store = (lambda a: a.astype(np.float16).astype(np.float64)) if self.half else (lambda a: a.astype(np.float32).astype(np.float64))
        for layer, (ks, vs) in zip(self.m["layers"], self.kv):
            y = (layer["qkv"].astype(np.float64) @ x).reshape(-1, HD)
            c, s = self.cos[len(ks)], self.sin[len(ks)]
            r = y.copy()
            r[:, 0::2], r[:, 1::2] = y[:, 0::2] * c - y[:, 1::2] * s, y[:, 0::2] * s + y[:, 1::2] * c
            ks.append(store(r[HEADS:HEADS + KV_HEADS])), vs.append(store(y[HEADS + KV_HEADS:]))
            k, v = np.stack(ks).repeat(HEADS // KV_HEADS, 1), np.stack(vs).repeat(HEADS // KV_HEADS, 1)
            z = np.einsum("hd,nhd->hn", r[:HEADS], k) / HD ** 0.5
            w = np.exp(z - z.max(1, keepdims=True))
            x = x + layer["out"].astype(np.float64) @ np.einsum("hn,nhd->hd", w / w.sum(1, keepdims=True), v).reshape(-1)
        return self.m["head"].astype(np.float64) @ x


@pytest.mark.parametrize("dtype", [torch.half, torch.float])
def test_batched_decode_with_pages(cuda, dtype):
    """Prompts in one packed pass, then steps of the batch; each token drawn on the device is the one that the 64-bit logits of its own sequence
    give, and the logits agree. Bound: the logits pass through two layers of fp32 products of 256 terms, each off by at most 256 x 2^-24 of
    its magnitudes (about 4, with sums of about 16 of them): well below 1e-3; half rows may round the other way where a key or value
    lies next to a border, 2^-11 of one of at least 10 positions' values: 2e-2. A draw nearer than 20 times the probabilities' shift to a border
    is no judge, and neither is what follows it in its sequence."""
    rng = np.random.default_rng(3)
    m = model(rng)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    mats = {"embed": K.Mat(MAT_F32, VOCAB, DIM, dev(m["embed"])), "head": K.Mat(MAT_F32, VOCAB, DIM, dev(m["head"]))}
    layers = [{n: K.Mat(MAT_F32, a.shape[0], a.shape[1], dev(a)) for n, a in layer.items()} for layer in m["layers"]]
    cos, sin = (dev(t) for t in tables())
    n_pages = 24
    pool = torch.full((n_pages, LAYERS, 2, KV_HEADS, PAGE, HD), float("nan"), dtype=dtype, device=cuda)
    free = list(rng.permutation(n_pages))
    scratch = K.PagedScratch(HEADS, KV_HEADS, HD, cuda)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (37, 1, 18)]
    prompts.append(prompts[0][:32] + rng.integers(0, VOCAB, 3).tolist())  # shares its first two pages with sequence 0
    table = torch.full((5, N_CTX // PAGE), -1, dtype=torch.int32, device=cuda)  # the last row pads the batch
    host, fed, err = [Host(m, dtype == torch.half) for _ in prompts], [[] for _ in prompts], torch.zeros(1, dtype=torch.int32, device=cuda)

    def forward(toks, seq, pos):
        """Rows of new tokens at positions of sequences (-1: padding); their logits."""
        for s, p in zip(seq, pos):
            if s >= 0 and int(table[s, p // PAGE]) < 0:
                table[s, p // PAGE] = int(free.pop())
        t = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
        x, sq, ps = K.embed(mats["embed"], t(toks)), t(seq), t(pos)
        for i, layer in enumerate(layers):
            kp, vp = pool[:, i, 0], pool[:, i, 1]
            q = K.rope_kv_paged(K.gemv(layer["qkv"], x), kp, vp, table, cos, sin, ps, sq, HEADS, KV_HEADS, HD, False, err=err)
            a, _ = K.attn_decode_paged(q, kp, vp, table, ps + 1, HEADS, scratch, seq=sq, quant=False, out=torch.zeros_like(q), err=err)
            x = K.gemv(layer["out"], a, res=x)
        return K.gemv(mats["head"], x)

    # prompts: all but the last token of each, packed; the last sequence's first 32 are in sequence 0's pages
    rows = [(tok, s, p) for s, prompt in enumerate(prompts[:3]) for p, tok in enumerate(prompt[:-1])]
    forward(*zip(*rows))
    table[3, :2] = table[0, :2]
    forward(*zip(*[(prompts[3][p], 3, p) for p in range(32, 34)]))
    for s, prompt in enumerate(prompts):
        for tok in prompt[:-1]:
            host[s].step(tok)
    last, pos, judged, live = [p[-1] for p in prompts], [len(p) - 1 for p in prompts], 0, [True] * 4
    temp, top_k, top_p, min_p = [0.9, 0.0, 1.2, 0.7], [0, 0, 12, 0], [0.95, 1.0, 1.0, 0.8], [0.0, 0.0, 0.02, 0.05]
    for step in range(14):
        batch = [s for s in range(4) if not (s == 1 and step < 3) and not (s == 2 and step > 9)]  # one comes later, one leaves
        u = rng.random(5, dtype=np.float32)
        pad = 5 - len(batch)
        logits = forward([last[s] for s in batch] + [0] * pad, batch + [-1] * pad, [pos[s] for s in batch] + [0] * pad)
        pick = lambda v, dt: torch.tensor([v[s] for s in batch] + [v[0]] * pad, dtype=dt, device=cuda)  # noqa: E731
        idx, prob = K.sample(logits, dev(u), pick(temp, torch.float), pick(top_k, torch.int32), pick(top_p, torch.float), pick(min_p, torch.float))
        idx, prob, logits = idx.tolist(), prob.tolist(), logits.cpu().numpy().astype(np.float64)
        for r, s in enumerate(batch):
            z = host[s].step(last[s])
            shift = np.abs(logits[r] - z).max()
            assert shift <= (2e-2 if dtype == torch.half else 1e-3), (step, s, shift)
            if live[s]:
                want, pr, _ = draw(z.copy(), u[r], np.float32(temp[s]), top_k[s], np.float32(top_p[s]), np.float32(min_p[s]))
                own = draw(logits[r].copy(), u[r], np.float32(temp[s]), top_k[s], np.float32(top_p[s]), np.float32(min_p[s]))[0]
                assert idx[r] == own  # the device's own logits, in 64 bits
                if idx[r] == want:
                    judged += 1
                    assert abs(prob[r] - pr) <= 20 * max(shift, 1e-6) * max(1.0, 1 / max(temp[s], 0.7))
                else:
                    live[s] = False  # (next to a border: see above)
            last[s], pos[s] = idx[r], pos[s] + 1
    assert int(err) == 0 and judged >= 30
