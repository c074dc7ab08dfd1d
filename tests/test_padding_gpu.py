"""What a batched step makes of rows that only pad the batch, of rows with nothing to draw and of memory that others have used: nothing that is
not the step's own is read or handed out."""
import numpy as np
import pytest
import torch

from amd_c_b200 import kernels as K
from amd_c_b200 import synth
from amd_c_b200._lib import MAT_F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [256, 96])
@pytest.mark.parametrize("kind", ["f32", "q4", "q8"])
def test_embed_tokens_that_are_no_rows(cuda, kind, cols):
    """A matrix that is the first half of a larger one: tokens behind its last row give zeros, not the rows that lie there; then the token of
    a row with nothing to draw."""
    rng = np.random.default_rng(cols)
    if kind == "f32":
        whole = K.Mat(MAT_F32, 40, cols, torch.from_numpy(rng.standard_normal((40, cols)).astype(np.float32)).to(cuda))
    else:
        ggml = {"q4": synth.GGML_Q4_0, "q8": synth.GGML_Q8_0}[kind]
        whole = K.Mat.from_gguf(ggml, torch.from_numpy(synth.make_gguf_bytes(ggml, rng, 40, cols)).to(cuda), 40, cols)
    half = K.Mat(whole.kind, 20, cols, whole.data)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    rows = K.embed(whole, t(range(40)))
    assert (rows != 0).any(1).all()
    got = K.embed(half, t([19, 20, 0, 39, 5, 21]))
    assert torch.equal(got[[0, 2, 4]], rows[[19, 0, 5]]) and (got[[1, 3, 5]] == 0).all()
    got = K.embed(half, t([-1, 7, -2, 0x7FFFFFFF, 40]))
    assert torch.equal(got[1], rows[7]) and (got[[0, 2, 3, 4]] == 0).all()


def test_tokens_drawn_from_nothing(cuda):
    """Rows of logits without a finite one: their token is -1 (looked at on the host before anything reads it), its embedding zeros."""
    logits = torch.randn(5, 300, device=cuda)
    logits[1], logits[3] = float("nan"), float("-inf")
    idx, prob = K.sample(logits, torch.rand(5, device=cuda), temp=torch.tensor([1.0, 1.0, 0.0, 0.0, 1.0], device=cuda))
    tokens = idx.tolist()
    assert tokens[1] == tokens[3] == -1 and all(0 <= tokens[r] < 300 for r in (0, 2, 4)) and prob.tolist()[1] == prob.tolist()[3] == 0.0
    w = torch.randn(300, 64, device=cuda)
    x = K.embed(K.Mat(MAT_F32, 300, 64, w), idx)
    assert (x[[1, 3]] == 0).all() and torch.equal(x[[0, 2, 4]], w[idx[[0, 2, 4]].long()])


def poison(*shapes):
    """Leaves NaN in the allocator's blocks of these sizes (float rows, or bytes): what a call gets for outputs that nobody writes."""
    held = [torch.full(s, float("nan"), device="cuda") if dtype is None else torch.full(s, 0xFF, dtype=dtype, device="cuda") for s, dtype in shapes]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("dtype", [torch.half, torch.float])
@pytest.mark.parametrize("rows,heads,kv_heads,hd,off", [(5, 8, 2, 64, 0), (700, 4, 4, 32, 0), (5, 28, 4, 128, 0), (9, 3, 1, 40, 1), (3, 0, 2, 64, 0)])
def test_padding_of_new_outputs_is_zeros(cuda, dtype, rows, heads, kv_heads, hd, off):
    """Where the wrappers make the outputs, the rows of padding (and q's of positions that do not exist) are zeros, in the Q8 copies too; the other
    rows have the bits that they have in an output of the caller's, whose padding keeps what was there."""
    gen = torch.Generator(device=cuda).manual_seed(rows + hd)
    width, seqs, page = (heads + 2 * kv_heads) * hd, 4, 16
    table = torch.arange(seqs * 4, dtype=torch.int32, device=cuda).view(seqs, 4)
    table[3, 1] = 999  # no page
    kp, vp = (torch.randn(16, kv_heads, page, hd, device=cuda, generator=gen).to(dtype) for _ in "kv")
    i = torch.arange(rows, device=cuda, dtype=torch.int32)
    seq = torch.where(i % 3 == 1, torch.where(i % 2 == 0, -1, seqs), i % seqs).int()
    pos = (i // seqs) % 64
    pos = torch.where(seq == 3, 16 + pos % 16, pos).int()
    angle = torch.rand(64, hd // 2, device=cuda, generator=gen)
    cos, sin = angle.cos(), angle.sin()
    qkv = torch.randn(rows, width + 1, device=cuda, generator=gen)[:, off:off + width]
    args = (kp, vp, table, cos, sin, pos, seq, heads, kv_heads, hd, True)
    given = torch.full((rows, heads * hd), 7.0, device=cuda)
    K.rope_kv_paged(qkv, *args, out=given)
    poison(((rows, heads * hd), None))
    q = K.rope_kv_paged(qkv, *args)
    nothing = (seq < 0) | (seq >= 3)
    assert (q[nothing] == 0).all() and (given[nothing] == 7).all() and torch.equal(q[~nothing], given[~nothing])
    if hd == 40 or heads == 0:
        return
    q = torch.randn(rows, heads * hd, device=cuda, generator=gen)
    args = (kp, vp, table, pos, heads, K.PagedScratch(heads, kv_heads, hd, cuda), seq)
    given = torch.full((rows, heads * hd), 7.0, device=cuda)
    copies = (rows, heads * hd // 32 * 40)
    poison((copies, torch.uint8))
    _, given_q8 = K.attn_decode_paged(q, *args, out=given)
    poison(((rows, heads * hd), None), (copies, torch.uint8))
    out, q8 = K.attn_decode_paged(q, *args)
    pad = (seq < 0) | (seq >= seqs)
    assert (out[pad] == 0).all() and (q8[pad] == 0).all() and (given[pad] == 7).all() and (given_q8[pad] == 0).all()
    assert torch.equal(out[~pad], given[~pad]) and torch.equal(q8, given_q8) and torch.equal(q8, K.quant_q8(out))


def test_padded_steps_fed_by_their_own_draws(cuda):
    """The documented step with the Q8 copies going into the output product, one graph replayed with the tokens of the last draw, on the device:
    rows of padding draw from logits that are numbers. Each step's tokens are looked at on the host before the next step reads them."""
    rng = np.random.default_rng(5)
    heads, kv_heads, hd, page, vocab, dim, rows = 8, 2, 32, 16, 320, 256, 6
    mat = lambda n, c: K.Mat.from_gguf(synth.GGML_Q4_0, torch.from_numpy(synth.make_gguf_bytes(synth.GGML_Q4_0, rng, n, c, 0.06)).to(cuda), n, c)  # noqa: E731
    emb, w_qkv, w_out, head = mat(vocab, dim), mat((heads + 2 * kv_heads) * hd, dim), mat(dim, heads * hd), mat(vocab, dim)
    kp, vp = (torch.zeros(8, kv_heads, page, hd, dtype=torch.half, device=cuda) for _ in "kv")
    table = torch.arange(8, dtype=torch.int32, device=cuda).view(4, 2)
    angle = torch.rand(32, hd // 2, device=cuda)
    cos, sin, ones = angle.cos(), angle.sin(), torch.ones(dim, device=cuda)
    tok, pos = torch.tensor([3, 0, 300, -1, 7, 320], dtype=torch.int32, device=cuda), torch.zeros(rows, dtype=torch.int32, device=cuda)
    lens, seq = torch.ones_like(pos), torch.tensor([0, -1, 1, 4, 2, -1], dtype=torch.int32, device=cuda)
    u, scratch = torch.rand(rows, device=cuda), K.PagedScratch(heads, kv_heads, hd, cuda)

    def step():
        x = K.embed(emb, tok)
        q = K.rope_kv_paged(K.gemv(w_qkv, K.rmsnorm(x, ones, 1e-5)[1]), kp, vp, table, cos, sin, pos, seq, heads, kv_heads, hd, False)
        _, copies = K.attn_decode_paged(q, kp, vp, table, lens, heads, scratch, seq=seq)
        logits = K.gemv(head, K.rmsnorm(K.gemv(w_out, copies, res=x), ones, 1e-5)[1])
        return q, copies, logits, K.sample(logits, u)[0]

    def look(q, copies, logits, idx):
        pad = (seq < 0) | (seq >= 4)
        assert (q[pad] == 0).all() and (copies[pad] == 0).all() and torch.isfinite(logits).all()
        tokens = idx.tolist()
        assert all(0 <= t < vocab for t in tokens)

    poison(((rows, heads * hd), None), ((rows, heads * hd // 32 * 40), torch.uint8))
    look(*step())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    for i in range(12):
        for t in results:
            t.fill_(float("nan") if t.is_floating_point() else 255 if t.dtype is torch.uint8 else -1)
        u.uniform_(), pos.fill_(i), lens.fill_(i + 1)
        graph.replay()
        look(*results)
        tok.copy_(results[3])


def test_a_new_scratch_on_another_stream(cuda):
    """A scratch made behind work that is still running is ready when a call on another stream uses it at once: the parts of a cut row are joined."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    kp, vp = (torch.randn(40, 2, 16, 64, device=cuda, generator=gen).half() for _ in "kv")
    table, lens = torch.randperm(40, device=cuda, generator=gen).int().view(1, 40), torch.tensor([640], dtype=torch.int32, device=cuda)
    q = torch.randn(1, 8 * 64, device=cuda, generator=gen)
    want, _ = K.attn_decode_paged(q, kp, vp, table, lens, 8, K.PagedScratch(8, 2, 64, cuda), quant=False)
    size, side, out = K.PagedScratch(8, 2, 64, cuda).data.numel(), torch.cuda.Stream(), torch.zeros_like(q)
    poison(((size,), torch.uint8))
    torch.cuda._sleep(400_000_000)  # some 0.2 s on this stream
    scratch = K.PagedScratch(8, 2, 64, cuda)
    with torch.cuda.stream(side):
        K.attn_decode_paged(q, kp, vp, table, lens, 8, scratch, quant=False, out=out)
    side.synchronize()
    assert torch.equal(out, want)
    torch.cuda.synchronize()


def test_a_scratch_made_in_a_graph(cuda):
    """A graph that makes its own scratch: every replay joins the parts of a cut row."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    kp, vp = (torch.randn(40, 2, 16, 64, device=cuda, generator=gen).half() for _ in "kv")
    table, lens = torch.randperm(40, device=cuda, generator=gen).int().view(1, 40), torch.tensor([640], dtype=torch.int32, device=cuda)
    q, out = torch.randn(1, 8 * 64, device=cuda, generator=gen), torch.zeros(1, 8 * 64, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.attn_decode_paged(q, kp, vp, table, lens, 8, K.PagedScratch(8, 2, 64, cuda), quant=False, out=out)
    for _ in range(3):
        q.normal_(generator=gen), out.zero_()
        graph.replay()
        assert torch.equal(out, K.attn_decode_paged(q, kp, vp, table, lens, 8, K.PagedScratch(8, 2, 64, cuda), quant=False)[0])
