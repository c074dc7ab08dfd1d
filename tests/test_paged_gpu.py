"""A batched decode step over a paged KV cache: RoPE with the store into the pages, and attention of one token per row, against the
formulas in 64 bits."""
import numpy as np
import pytest
import torch

from amd_c_b200 import kernels as K

pytestmark = pytest.mark.gpu
PAGES_WORD = 6  # the error word of a position or page that does not exist


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_cache(gen, lens, n_kv, hd, page, dtype, extra_cols=1, fill=None):
    """Pools whose pages are dealt out in random order, every row that no sequence holds NaN (or `fill`); positions are in the pages'
    order of the table."""
    used = [-(-n // page) for n in lens]
    total = sum(used) + 2
    order = torch.randperm(total, device="cuda", generator=gen).int()
    table = torch.full((len(lens), max(used + [1]) + extra_cols), 0x7FFFFFF0, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    kp, vp = (torch.full((total, n_kv, page, hd), float("nan") if fill is None else fill, dtype=dtype, device="cuda") for _ in "kv")
    return kp, vp, table


def put(pool, table, s, rows):
    """rows [n, n_kv, hd] as positions 0 .. n - 1 of sequence s."""
    n, page = rows.shape[0], pool.shape[2]
    for c in range(-(-n // page)):
        part = rows[c * page:(c + 1) * page]
        pool[int(table[s, c]), :, :part.shape[0]] = part.transpose(0, 1).to(pool.dtype)


def get(pool, table, s, n):
    page = pool.shape[2]
    return torch.cat([pool[int(table[s, c])] for c in range(-(-n // page))], 1)[:, :n].transpose(0, 1)


# ---------------------------------------------------------------- RoPE and the store
def rope_tables(n, hd):
    angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * 1e4 ** (-torch.arange(hd // 2, dtype=torch.float64, device="cuda") / (hd // 2))
    return angle.cos().float(), angle.sin().float()


def rotated(x, cos, sin, neox):
    """x [T, heads, hd] double; the rotation, and per element the sum of the two products' magnitudes."""
    hd = x.shape[2]
    i = torch.arange(hd // 2, device="cuda")
    lo, hi = (i, i + hd // 2) if neox else (2 * i, 2 * i + 1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    y, size = torch.empty_like(x), torch.empty_like(x)
    y[..., lo], size[..., lo] = x[..., lo] * c - x[..., hi] * s, (x[..., lo] * c).abs() + (x[..., hi] * s).abs()
    y[..., hi], size[..., hi] = x[..., lo] * s + x[..., hi] * c, (x[..., lo] * s).abs() + (x[..., hi] * c).abs()
    return y, size


@pytest.mark.parametrize("dtype", [torch.half, torch.float])
@pytest.mark.parametrize("nq,nkv,hd,page,neox,parts,off", [
    (32, 8, 128, 16, False, [(0, 1)], 0),
    (28, 4, 128, 16, True, [(i * 7 % 50, 1) for i in range(33)], 0),
    (8, 4, 32, 1, False, [(0, 5), (3, 1), (0, 17)], 0),
    (5, 1, 64, 5, True, [(4, 13), (0, 1), (9, 2)], 0),
    (3, 3, 40, 7, False, [(6, 9), (0, 8)], 0),
    (1, 1, 512, 16, True, [(15, 2)], 0),
    (2, 2, 8, 32, False, [(31, 3)], 0),
    (0, 4, 64, 16, True, [(0, 20)], 0),
    (32, 8, 128, 64, True, [(0, 700), (100, 333)], 0),
    (7, 1, 64, 16, False, [(2, 21), (0, 3)], 1),
    (4, 2, 128, 16, True, [(2, 21), (0, 3)], 3),
])
def test_rope_kv_paged(cuda, dtype, nq, nkv, hd, page, neox, parts, off):
    """Rotated q, and the pools' new rows, against the formula in 64 bits; every other row of the pools keeps its bits. Bound: two
    rounded products and a rounded sum are within 2 x 2^-24 of the products' magnitudes together; the store to half adds half a step, 2^-11
    of the value or 2^-25. `off`: qkv and the output start that many floats off their 16-byte alignment."""
    gen = generator(nq * 1000 + hd)
    T, width = sum(n for _, n in parts), (nq + 2 * nkv) * hd
    kp, vp, table = make_cache(gen, [a + n for a, n in parts], nkv, hd, page, dtype, fill=0.25)
    cos, sin = rope_tables(max(a + n for a, n in parts), hd)
    pos = torch.tensor([a + i for a, n in parts for i in range(n)], dtype=torch.int32, device=cuda)
    seq = torch.tensor([s for s, (_, n) in enumerate(parts) for _ in range(n)], dtype=torch.int32, device=cuda)
    qkv = torch.randn(T, width + 4, device=cuda, generator=gen)[:, off:off + width]
    before, kp0, vp0 = qkv.clone(), kp.clone(), vp.clone()
    out = torch.empty(T, nq * hd + 8, device=cuda)[:, off:off + nq * hd] if nq else None
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    q = K.rope_kv_paged(qkv, kp, vp, table, cos, sin, pos, seq, nq, nkv, hd, neox, out=out, err=err)
    assert int(err) == 0 and torch.equal(qkv, before)
    x = qkv.double().view(T, nq + 2 * nkv, hd) if qkv.is_contiguous() else qkv.contiguous().double().view(T, nq + 2 * nkv, hd)
    want, size = rotated(x, cos[pos.long()], sin[pos.long()], neox)
    assert ((q.double().view(T, nq, hd) - want[:, :nq]).abs() <= 2.001 * 2.0 ** -24 * size[:, :nq]).all()
    at, row = table[seq.long(), pos.long() // page].long(), pos.long() % page
    k, v = kp[at, :, row].double(), vp[at, :, row].double()
    half = (lambda y: 2.0 ** -11 * y.abs() + 2.0 ** -25) if dtype == torch.half else (lambda y: 0.0)
    y = want[:, nq:nq + nkv]
    assert ((k - y).abs() <= 2.01 * 2.0 ** -24 * size[:, nq:nq + nkv] + 1.001 * half(y)).all()
    assert torch.equal(v.to(dtype), x[:, nq + nkv:].to(dtype))
    kp0[at, :, row], vp0[at, :, row] = kp[at, :, row], vp[at, :, row]
    assert torch.equal(kp, kp0) and torch.equal(vp, vp0)


@pytest.mark.parametrize("neox,dtype", [(False, torch.half), (True, torch.float)])
def test_rope_kv_paged_has_the_bits_of_rope_kv(cuda, neox, dtype):
    gen = generator(3)
    nq, nkv, hd, T, page = 8, 2, 64, 45, 16
    qkv = torch.randn(T, (nq + 2 * nkv) * hd, device=cuda, generator=gen)
    cos, sin = rope_tables(T, hd)
    kp, vp, table = make_cache(gen, [T], nkv, hd, page, dtype)
    pos = torch.arange(T, dtype=torch.int32, device=cuda)
    q = K.rope_kv_paged(qkv, kp, vp, table, cos, sin, pos, torch.zeros_like(pos), nq, nkv, hd, neox)
    kc, vc = (torch.empty(nkv, T, hd, dtype=dtype, device=cuda) for _ in "kv")
    same = qkv.clone()
    K.rope_kv(same, kc, vc, cos, sin, torch.zeros(1, dtype=torch.int32, device=cuda), nq, nkv, hd, neox, T)
    assert torch.equal(q, same[:, :nq * hd])
    assert torch.equal(get(kp, table, 0, T).transpose(0, 1), kc) and torch.equal(get(vp, table, 0, T).transpose(0, 1), vc)
    in_place = K.rope_kv_paged(qkv, kp, vp, table, cos, sin, pos, torch.zeros_like(pos), nq, nkv, hd, neox, out=qkv[:, :nq * hd])
    assert torch.equal(in_place, q) and torch.equal(qkv[:, :nq * hd], q)


def test_rope_kv_paged_positions_that_do_not_exist(cuda):
    """Padding (-1), pages outside the pools, positions outside the table or the RoPE tables: nothing is stored, q's row is left as it
    was, and all but the padding are reported. The other tokens of the call are done."""
    gen = generator(4)
    nq, nkv, hd, page = 4, 2, 64, 16
    kp, vp, table = make_cache(gen, [40, 40], nkv, hd, page, torch.half, extra_cols=0, fill=1.0)
    table[1, 1] = -1
    cos, sin = rope_tables(30, hd)
    qkv = torch.randn(6, (nq + 2 * nkv) * hd, device=cuda, generator=gen)
    good = (0, 20)
    for bad, reported in [((-1, 0), 0), ((2, 0), 0), ((1, 17), 1), ((0, 48), 1), ((0, -5), 1), ((0, 30), 1)]:
        kp.fill_(1.0), vp.fill_(1.0)
        seq = torch.tensor([bad[0], good[0], bad[0]], dtype=torch.int32, device=cuda)
        pos = torch.tensor([bad[1], good[1], bad[1]], dtype=torch.int32, device=cuda)
        out, err = torch.full((3, nq * hd), 7.0, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
        K.rope_kv_paged(qkv[:3], kp, vp, table, cos, sin, pos, seq, nq, nkv, hd, True, out=out, err=err)
        assert int(err) == PAGES_WORD * reported, bad
        assert (out[0] == 7).all() and (out[2] == 7).all() and (out[1] != 7).any(), bad
        assert int((kp != 1).any(-1).sum()) == nkv and int((vp != 1).any(-1).sum()) == nkv, bad


# ---------------------------------------------------------------- attention
def attention(q, kp, vp, table, lens, n_head, seq=None):
    """In 64 bits, row by row; and per (row, head) the magnitudes that the bound goes by: the largest sum of |q k| / sqrt(hd) and |v|."""
    R, n_kv, hd = q.shape[0], kp.shape[1], kp.shape[3]
    out, bound = torch.zeros(R, n_head, hd, dtype=torch.float64, device="cuda"), torch.zeros(R, n_head, 1, dtype=torch.float64, device="cuda")
    for r in range(R):
        n, s = int(lens[r]), r if seq is None else int(seq[r])
        if n == 0:
            continue
        k, v = (get(p, table, s, n).double().repeat_interleave(n_head // n_kv, 1) for p in (kp, vp))
        x = torch.einsum("hd,nhd->hn", q[r].double().view(n_head, hd), k) / hd ** 0.5
        out[r] = torch.einsum("hn,nhd->hd", torch.softmax(x, 1), v)
        size = torch.einsum("hd,nhd->hn", q[r].double().abs().view(n_head, hd), k.abs()) / hd ** 0.5
        bound[r] = ((size.amax(1) + 1) * v.abs().amax((0, 2)))[:, None]
    return out, bound


def check_attention(out, oq, want, bound):
    """A score is off by what carries q in 22 bits and sums hd products in fp32: 2^-19 of the products' magnitudes covers both (2^-22, and
    hd / 16 accumulations that lose up to 2^-23 of a partial sum); a weight by as much, a weighted mean of v by twice that times the
    largest |v|; the fp32 sums over the positions and the exponentials' 2^-22 are in the added one."""
    R, n_head, hd = want.shape
    assert torch.isfinite(out).all()
    assert ((out.double().view(R, n_head, hd) - want).abs() <= 2 * 2.0 ** -19 * bound).all()
    if oq is not None:
        assert torch.equal(oq, K.quant_q8(out.contiguous()))


def case(seed, lens, n_head, n_kv, hd, page, dtype):
    gen = generator(seed)
    kp, vp, table = make_cache(gen, lens, n_kv, hd, page, dtype)
    for s, n in enumerate(lens):
        for pool in (kp, vp):
            put(pool, table, s, torch.randn(n, n_kv, hd, device="cuda", generator=gen))
    q = torch.randn(len(lens), n_head * hd, device="cuda", generator=gen) * 1.5
    return q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


LENS = [[1], [0, 5], [500], [15, 16, 17, 0, 1, 64, 63, 65, 128, 129], [3000], [700, 1, 0, 0, 2049, 33, 256, 257], [0, 0, 0]]


@pytest.mark.parametrize("dtype", [torch.half, torch.float])
@pytest.mark.parametrize("n_head,n_kv,hd,page", [(32, 8, 128, 16), (28, 4, 128, 32), (8, 8, 64, 16), (8, 4, 32, 48), (5, 1, 64, 128), (12, 1, 128, 16), (32, 2, 32, 64), (3, 3, 128, 16)])
@pytest.mark.parametrize("lens", LENS)
def test_attn_decode_paged(cuda, dtype, n_head, n_kv, hd, page, lens):
    """Lengths around the edges of chunks and pages, none at all, shares that cut a row into parts; 1 to 16 query heads per KV head. The
    pages' rows behind a sequence's last hold NaN, the table's columns behind its last a number that is no page."""
    q, kp, vp, table, n = case(sum(lens) + hd, lens, n_head, n_kv, hd, page, dtype)
    scratch, err = K.PagedScratch(n_head, n_kv, hd, cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    out, oq = K.attn_decode_paged(q, kp, vp, table, n, n_head, scratch, err=err)
    assert int(err) == 0
    check_attention(out, oq, *attention(q, kp, vp, table, n, n_head))
    again, _ = K.attn_decode_paged(q, kp, vp, table, n, n_head, scratch, quant=False)  # the scratch is left ready, the sums have an order
    assert torch.equal(again, out)


def test_attn_decode_paged_long(cuda):
    """One long sequence over all CTAs, and a batch of more rows than a CTA has threads."""
    for lens, heads in (([20011], (16, 2, 128)), ([33000], (4, 1, 64)), ([(i * 37) % 90 for i in range(700)], (8, 4, 64))):
        q, kp, vp, table, n = case(len(lens), lens, *heads, 16, torch.half)
        out, oq = K.attn_decode_paged(q, kp, vp, table, n, heads[0], K.PagedScratch(*heads, cuda))
        check_attention(out, oq, *attention(q, kp, vp, table, n, heads[0]))


@pytest.mark.parametrize("dtype", [torch.half, torch.float])
def test_attn_decode_paged_rows_of_one_sequence(cuda, dtype):
    """Rows that name their sequences: the tokens of a prompt one by one, a shared prefix, and padding, whose rows are left as they were."""
    q, kp, vp, table, _ = case(5, [90, 40, 90], 8, 2, 64, 16, dtype)
    table[2, :4] = table[0, :4]  # the first 64 positions are sequence 0's
    q = torch.randn(100, 8 * 64, device=cuda, generator=generator(6))
    seq = torch.tensor([0] * 90 + [2, 1, 1, -1, 2, 3, 0, 1, 2, -1], dtype=torch.int32, device=cuda)
    lens = torch.tensor(list(range(1, 91)) + [90, 40, 0, 70, 65, 9, 90, 39, 64, 0], dtype=torch.int32, device=cuda)
    out = torch.full((100, 8 * 64), 3.0, device=cuda)
    K.attn_decode_paged(q, kp, vp, table, lens, 8, K.PagedScratch(8, 2, 64, cuda), seq=seq, quant=False, out=out)
    real = (seq >= 0) & (seq < 3)
    assert (out[~real] == 3).all() and int((~real).sum()) == 3
    check_attention(out[real], None, *attention(q[real], kp, vp, table, lens[real], 8, seq[real]))


@pytest.mark.parametrize("dtype", [torch.half, torch.float])
def test_attn_decode_paged_pages_that_do_not_exist(cuda, dtype):
    """Positions on pages outside the pools, and lengths past the table, are left out and reported; a row with nothing else is zeros."""
    page, lens = 16, [100, 32, 64]
    q, kp, vp, table, n = case(7, lens, 4, 2, 64, page, dtype)
    kp2, vp2, whole = kp.clone(), vp.clone(), table.clone()
    table[0, 2], table[0, 6], table[1, 0], table[1, 1] = -1, kp.shape[0], 0x7FFFFFFF, -2
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, oq = K.attn_decode_paged(q, kp, vp, table, n, 4, K.PagedScratch(4, 2, 64, cuda), err=err)
    assert int(err) == PAGES_WORD and (out[1] == 0).all() and (oq[1] == 0).all()
    # sequence 0 without pages 2 and 6, closed up
    short = whole.clone()
    short[0, 2:5] = whole[0, 3:6]
    keep = torch.tensor([100 - 16 - 4, 0, 64], dtype=torch.int32, device=cuda)
    check_attention(out, oq, *attention(q, kp2, vp2, short, keep, 4))
    err.zero_()
    n[2] = 4 * page * 1000
    out, _ = K.attn_decode_paged(q[2:], kp, vp, whole[2:3, :4].contiguous(), n[2:], 4, K.PagedScratch(4, 2, 64, cuda), err=err)
    assert int(err) == PAGES_WORD
    check_attention(out, None, *attention(q[2:], kp, vp, whole[2:3], [64], 4))


@pytest.mark.parametrize("dtype", [torch.half, torch.float])
@pytest.mark.parametrize("hd,rows,page", [(32, 1, 16), (32, 30, 48), (64, 1, 32), (64, 30, 16), (128, 1, 16), (128, 30, 80)])
def test_attn_decode_paged_holes(cuda, dtype, hd, rows, page):
    """Every third page of a sequence is none, first, last and neighbouring ones among them; what is left is attended to, few and many rows."""
    lens = [900 + 37 * i % 700 for i in range(rows)]
    q, kp, vp, table, n = case(hd + rows, lens, 8, 2, hd, page, dtype)
    gen = torch.Generator().manual_seed(rows)
    hole = (torch.rand(table.shape, generator=gen) < 0.34).to(cuda)
    hole[0, 0] = hole[0, (lens[0] - 1) // page] = True
    holes = torch.where(hole, -1 - torch.randint(0, 9, table.shape, generator=gen).int().to(cuda), table)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, oq = K.attn_decode_paged(q, kp, vp, holes, n, 8, K.PagedScratch(8, 2, hd, cuda), err=err)
    assert int(err) == PAGES_WORD
    want, bound = torch.zeros(rows, 8, hd, dtype=torch.float64, device=cuda), torch.zeros(rows, 8, 1, dtype=torch.float64, device=cuda)
    for r, m in enumerate(lens):
        there = ~hole[r].repeat_interleave(page)[:m]
        k, v = (get(p, table, r, m)[there].double().repeat_interleave(4, 1) for p in (kp, vp))
        x = torch.einsum("hd,nhd->hn", q[r].double().view(8, hd), k) / hd ** 0.5
        want[r] = torch.einsum("hn,nhd->hd", torch.softmax(x, 1), v)
        size = torch.einsum("hd,nhd->hn", q[r].double().abs().view(8, hd), k.abs()) / hd ** 0.5
        bound[r] = ((size.amax(1) + 1) * v.abs().amax((0, 2)))[:, None]
    check_attention(out, oq, want, bound)


def test_attn_decode_paged_many_rows_most_of_them_empty(cuda):
    """More rows than the GPU has warps: rows of nothing are zeros wherever they lie, padding keeps what it had."""
    q, kp, vp, table, _ = case(12, [33, 70], 4, 2, 64, 16, torch.half)
    R = 5000
    gen = torch.Generator().manual_seed(0)
    seq, lens = torch.randint(-1, 2, (R,), generator=gen).int().to(cuda), torch.zeros(R, dtype=torch.int32, device=cuda)
    some = torch.randperm(R, generator=gen)[:300].to(cuda)
    lens[some] = torch.randint(1, 34, (300,), generator=gen).int().to(cuda)
    q = torch.randn(R, 4 * 64, device=cuda, generator=generator(13))
    out = torch.full_like(q, 5.0)
    _, oq = K.attn_decode_paged(q, kp, vp, table, lens, 4, K.PagedScratch(4, 2, 64, cuda), seq=seq, out=out)
    real, empty = seq >= 0, lens == 0
    assert (out[~real] == 5).all() and (out[real & empty] == 0).all() and (oq[real & empty] == 0).all()
    full = real & ~empty
    check_attention(out[full], oq[full], *attention(q[full], kp, vp, table, lens[full], 4, seq[full]))


@pytest.mark.parametrize("dtype", [torch.half, torch.float])
@pytest.mark.parametrize("n_head,n_kv,hd,page,extra", [(28, 4, 128, 16, 140), (40, 8, 128, 64, 1), (12, 1, 128, 48, 1), (16, 16, 64, 32, 1), (9, 1, 64, 16, 1), (8, 4, 32, 16, 1), (32, 2, 32, 80, 30)])
def test_attn_decode_paged_many_short_rows(cuda, dtype, n_head, n_kv, hd, page, extra):
    """More (row, KV head) pairs than the GPU has room for at once, of no to some chunks each; empty rows, padding, a missing page; narrow and wide tables."""
    lens = [(i * 37) % 210 for i in range(41)]
    gen = generator(hd + n_head)
    kp, vp, table = make_cache(gen, lens, n_kv, hd, page, dtype, extra_cols=extra)
    for s, n in enumerate(lens):
        for pool in (kp, vp):
            put(pool, table, s, torch.randn(n, n_kv, hd, device=cuda, generator=gen))
    R = 1300
    seq = (torch.arange(R, device=cuda, dtype=torch.int32) * 7) % 43 - 1  # -1 and 41 pad
    real = (seq >= 0) & (seq < 41)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda)[seq.long().clamp(0, 40)]
    n = (n - torch.arange(R, device=cuda, dtype=torch.int32) % 11).clamp(min=0)
    q = torch.randn(R, n_head * hd, device=cuda, generator=gen)
    out, scratch, err = torch.full_like(q, 4.0), K.PagedScratch(n_head, n_kv, hd, cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    _, oq = K.attn_decode_paged(q, kp, vp, table, n, n_head, scratch, seq=seq, out=out, err=err)
    assert int(err) == 0 and (out[~real] == 4).all()
    assert (out[real & (n == 0)] == 0).all() and (oq[real & (n == 0)] == 0).all()
    some = torch.nonzero(real)[:, 0]
    check_attention(out[some], oq[some], *attention(q[some], kp, vp, table, n[some], n_head, seq[some]))
    again, _ = K.attn_decode_paged(q, kp, vp, table, n, n_head, scratch, seq=seq, quant=False)
    assert torch.equal(again[real], out[real])
    table[5, 0] = -3  # sequence 5 has lost its first page
    lost, _ = K.attn_decode_paged(q, kp, vp, table, n, n_head, scratch, seq=seq, quant=False, err=err)
    assert int(err) == PAGES_WORD and torch.equal(lost[real & (seq != 5)], out[real & (seq != 5)])
    mine = torch.nonzero((seq == 5) & (n > page))[:, 0]
    if len(mine):
        table[5, :-1] = table[5, 1:].clone()
        check_attention(lost[mine], None, *attention(q[mine], kp, vp, table, n[mine] - page, n_head, seq[mine]))
    assert (lost[(seq == 5) & (n <= page)] == 0).all()


@pytest.mark.parametrize("own", [True, False])
def test_attn_decode_paged_wide_tables(cuda, own):
    """Tables of 2^24 positions, of which little is in use: 300 rows are more than one launch numbers; rows of their own sequences, and rows that
    name theirs."""
    lens = [(i * 13) % 41 for i in range(300 if own else 3)]
    gen = generator(14)
    kp, vp, table = make_cache(gen, lens, 8, 32, 1024, torch.half, extra_cols=(1 << 14) - 1)
    for s, n in enumerate(lens):
        for pool in (kp, vp):
            put(pool, table, s, torch.randn(n, 8, 32, device=cuda, generator=gen))
    q = torch.randn(300, 8 * 32, device=cuda, generator=gen)
    seq = None if own else (torch.arange(300, device=cuda, dtype=torch.int32) * 7) % 4 - 1
    n = torch.tensor(lens, dtype=torch.int32, device=cuda) if own else torch.tensor(lens, dtype=torch.int32, device=cuda)[seq.long().clamp(min=0)]
    before, out = K._lib.load().ie_b200_launch_count(), torch.full_like(q, 2.0)
    _, oq = K.attn_decode_paged(q, kp, vp, table, n, 8, K.PagedScratch(8, 8, 32, cuda), seq=seq, out=out)
    assert K._lib.load().ie_b200_launch_count() - before == 2
    real = torch.ones(300, dtype=torch.bool, device=cuda) if own else seq >= 0
    assert (out[~real] == 2).all()
    check_attention(out[real], oq[real], *attention(q[real], kp, vp, table, n[real], 8, None if own else seq[real]))


def test_attn_decode_paged_peaked(cuda):
    """Scores in the hundreds: a row's weight on very few positions, the largest anywhere among the parts."""
    for dtype in (torch.half, torch.float):
        q, kp, vp, table, n = case(15, [700, 3000, 40], 8, 2, 128, 16, dtype)
        out, oq = K.attn_decode_paged(q * 40, kp, vp, table, n, 8, K.PagedScratch(8, 2, 128, cuda))
        check_attention(out, oq, *attention(q * 40, kp, vp, table, n, 8))


def test_attn_decode_paged_strides(cuda):
    """Rows of q and of the output apart and off their 16-byte alignment; layers interleaved in one pool; a table that is a slice."""
    q, kp, vp, table, n = case(8, [77, 300], 6, 2, 64, 16, torch.half)
    pool = torch.full((kp.shape[0], 3, 2, *kp.shape[1:]), float("nan"), dtype=torch.half, device=cuda)
    pool[:, 1, 0], pool[:, 1, 1] = kp, vp
    wide = torch.empty(2, 6 * 64 * 3 + 2, device=cuda)
    wide[:, 2:2 + 6 * 64] = q
    table2 = torch.full((2, table.shape[1] + 5), -7, dtype=torch.int32, device=cuda)
    table2[:, :table.shape[1]] = table
    out = torch.full((2, 6 * 64 + 5), 9.0, device=cuda)
    K.attn_decode_paged(wide[:, 2:2 + 6 * 64], pool[:, 1, 0], pool[:, 1, 1], table2[:, :table.shape[1]], n, 6, K.PagedScratch(6, 2, 64, cuda), quant=False,
                        out=out[:, 3:3 + 6 * 64])
    assert (out[:, :3] == 9).all() and (out[:, -2:] == 9).all()
    check_attention(out[:, 3:3 + 6 * 64].contiguous(), None, *attention(q, kp, vp, table, n, 6))


def test_paged_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 bytes whose last pages are the ones in use: stores and reads land there."""
    nq, nkv, hd, page, T = 4, 2, 64, 16, 40
    n = (1 << 32) // (nkv * page * hd * 2) + 20
    kp, vp = (torch.empty(n, nkv, page, hd, dtype=torch.half, device=cuda) for _ in "kv")
    kp[:4], vp[:4] = 5.0, 5.0
    table = torch.tensor([[n - 1, n - 9, n - 3]], dtype=torch.int32, device=cuda)
    gen = generator(9)
    qkv = torch.randn(T, (nq + 2 * nkv) * hd, device=cuda, generator=gen)
    cos, sin = rope_tables(T, hd)
    pos = torch.arange(T, dtype=torch.int32, device=cuda)
    q = K.rope_kv_paged(qkv, kp, vp, table, cos, sin, pos, torch.zeros_like(pos), nq, nkv, hd, True)
    assert torch.equal(get(vp, table, 0, T), qkv.view(T, -1, hd)[:, nq + nkv:].half()) and (kp[:4] == 5).all() and (vp[:4] == 5).all()
    lens = torch.tensor([T], dtype=torch.int32, device=cuda)
    out, oq = K.attn_decode_paged(q[-1:], kp, vp, table, lens, nq, K.PagedScratch(nq, nkv, hd, cuda))
    check_attention(out, oq, *attention(q[-1:], kp, vp, table, lens, nq))


def test_paged_decode_steps_in_a_graph(cuda):
    """Append and attention of a decode step captured once and replayed on another stream with new tokens, positions and lengths; every
    step against the formula over the cache as it is then, and against the contiguous kernels for the first sequence."""
    n_head, n_kv, hd, page, steps, start = 8, 2, 64, 16, 20, [30, 0, 100]
    gen = generator(10)
    kp, vp, table = make_cache(gen, [n + steps for n in start], n_kv, hd, page, torch.half)
    for s, n in enumerate(start):
        for pool in (kp, vp):
            put(pool, table, s, torch.randn(n, n_kv, hd, device=cuda, generator=gen))
    cos, sin = rope_tables(200, hd)
    qkv = torch.empty(3, (n_head + 2 * n_kv) * hd, device=cuda)
    pos, lens = torch.zeros(3, dtype=torch.int32, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    q, out = torch.empty(3, n_head * hd, device=cuda), torch.empty(3, n_head * hd, device=cuda)
    scratch = K.PagedScratch(n_head, n_kv, hd, cuda)

    def step():
        K.rope_kv_paged(qkv, kp, vp, table, cos, sin, pos, None, n_head, n_kv, hd, False, out=q)
        K.attn_decode_paged(q, kp, vp, table, lens, n_head, scratch, quant=False, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step()
        for i in range(steps):
            qkv.normal_(generator=gen)
            pos.copy_(torch.tensor(start, dtype=torch.int32) + i)
            lens.copy_(pos + 1)
            graph.replay()
            check_attention(out, None, *attention(q, kp, vp, table, lens, n_head))
            if i % 7 == 0:
                kc, vc = (get(p, table, 0, start[0] + i + 1).transpose(0, 1).contiguous() for p in (kp, vp))
                n = kc.shape[1]
                one, _ = K.attn_decode(q[:1], kc, vc, pos[:1], n_head, n_kv, hd, n, K.AttnScratch(n_head, hd, n, 1, cuda), quant=False)
                assert (out[:1] - one).abs().max() <= 1e-5 * one.abs().max()
    torch.cuda.current_stream().wait_stream(side)


def test_paged_more_rows_than_a_grid_is_high(cuda):
    """70 000 tokens and rows in one call each: every one is done, and in its own place."""
    T, gen = 70000, generator(16)
    kp, vp, table = make_cache(gen, [T], 1, 32, 64, torch.float)
    cos, sin = rope_tables(T, 32)
    qkv = torch.randn(T, 96, device=cuda, generator=gen)
    pos = torch.randperm(T, device=cuda, generator=gen).int()
    q = K.rope_kv_paged(qkv, kp, vp, table, cos, sin, pos, torch.zeros_like(pos), 1, 1, 32, True)
    k, v = get(kp, table, 0, T)[:, 0], get(vp, table, 0, T)[:, 0]
    want, size = rotated(qkv.double().view(T, 3, 32), cos[pos.long()], sin[pos.long()], True)
    assert ((q.double() - want[:, 0]).abs() <= 2.001 * 2.0 ** -24 * size[:, 0]).all()
    assert ((k[pos.long()].double() - want[:, 1]).abs() <= 2.001 * 2.0 ** -24 * size[:, 1]).all() and torch.equal(v[pos.long()], qkv[:, 64:])
    lens = (pos % 4).int()
    out, oq = K.attn_decode_paged(q, kp, vp, table, lens, 1, K.PagedScratch(1, 1, 32, cuda), seq=torch.zeros_like(pos))
    x = (q.double() @ k[:3].double().T / 32 ** 0.5).masked_fill(torch.arange(3, device=cuda) >= lens[:, None], float("-inf"))
    w = torch.where(lens[:, None] > 0, torch.softmax(x, 1), 0.0)
    bound = ((q.double().abs() @ k[:3].double().abs().T / 32 ** 0.5).amax(1, keepdim=True) + 1) * v[:3].double().abs().max()
    check_attention(out, None, (w @ v[:3].double())[:, None], bound[:, None])
    assert torch.equal(oq, torch.cat([K.quant_q8(out[:T // 2]), K.quant_q8(out[T // 2:])]))  # (the quantiser takes 65 535 rows)


def test_paged_calls_at_once(cuda):
    """Two batches on two streams, each with its own scratch and pages, and a draw between them: the bits that they give one after the
    other; the same scratch in two graphs, replayed in turn."""
    sets = [case(20 + i, [900, 33, 2000, 0, 1], 8, 2, 64, 16, torch.half) for i in range(2)]
    scratch = [K.PagedScratch(8, 2, 64, cuda) for _ in sets]
    logits, u = torch.randn(5, 40000, device=cuda, generator=generator(22)), torch.rand(5, device=cuda)
    want = [K.attn_decode_paged(q, kp, vp, table, n, 8, scratch[0])[0] for q, kp, vp, table, n in sets]
    token = K.sample(logits, u)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[], [], []]
    for _ in range(20):
        for i, (q, kp, vp, table, n) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(K.attn_decode_paged(q, kp, vp, table, n, 8, scratch[i])[0])
        with torch.cuda.stream(streams[2]):
            got[2].append(K.sample(logits, u)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i]) and all(torch.equal(x, token) for x in got[2])
    graphs, outs = [torch.cuda.CUDAGraph() for _ in sets], [torch.zeros_like(w) for w in want]
    for (q, kp, vp, table, n), graph, out in zip(sets, graphs, outs):
        with torch.cuda.graph(graph):
            K.attn_decode_paged(q, kp, vp, table, n, 8, scratch[0], quant=False, out=out)
    for _ in range(10):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_paged_wrappers_refuse(cuda):
    q, kp, vp, table, n = case(11, [20], 4, 2, 64, 16, torch.half)
    sc = K.PagedScratch(4, 2, 64, cuda)
    for bad in (dict(q=q.half()), dict(q=q[:, :64]), dict(q=q.T), dict(vp=vp.float()), dict(vp=vp[1:]), dict(vp=vp.transpose(1, 2)), dict(table=table.long()), dict(table=table[0]),
                dict(lens=n.long()), dict(lens=n.cpu()), dict(lens=torch.cat([n, n])), dict(q=torch.cat([q, q]), lens=torch.cat([n, n])),
                dict(scratch=K.PagedScratch(8, 2, 64, cuda)), dict(out=torch.empty(2, 256, device=cuda)), dict(seq=n.cpu()), dict(err=n.long())):
        with pytest.raises((ValueError, AttributeError)):
            K.attn_decode_paged(**{**dict(q=q, kp=kp, vp=vp, table=table, lens=n, n_head=4, scratch=sc), **bad})
    cos, sin = rope_tables(40, 64)
    qkv = torch.zeros(1, 8 * 64, device=cuda)
    for bad in (dict(qkv=qkv[:, 1:]), dict(cos=cos[:, 1:]), dict(sin=sin[1:]), dict(pos=n.long()), dict(nkv=4, nq=0), dict(out=qkv), dict(seq=torch.cat([n, n]))):
        with pytest.raises((ValueError, AttributeError)):
            K.rope_kv_paged(**{**dict(qkv=qkv, kp=kp, vp=vp, table=table, cos=cos, sin=sin, pos=n, seq=None, nq=4, nkv=2, hd=64, neox=True), **bad})
    assert K.attn_decode_paged(q[:0], kp, vp, table, n[:0], 4, sc)[0].shape == (0, 256)
    assert K.rope_kv_paged(qkv[:0], kp, vp, table, cos, sin, n[:0], n[:0], 4, 2, 64, True).shape == (0, 256)
