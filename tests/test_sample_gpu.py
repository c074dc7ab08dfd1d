"""The draw of the next tokens against the definition in 64 bits, sorted and summed on the host."""
import numpy as np
import pytest
import torch

from amd_c_b200 import kernels as K

pytestmark = pytest.mark.gpu


def draw(x, u, temp=1.0, k=0, p=1.0, m=0.0, unit=0.0):
    """(index, probability, how near u or top_p came to a border, per weight of the sum and in units of the largest one) of one row, in
    64 bits."""
    x = x.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    if x.max() == -np.inf:
        return -1, 0.0, 1.0
    if not temp > 0:
        return int(x.argmax()), 1.0, 1.0
    n = len(x)
    order = np.argsort(-x, kind="stable")
    top = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(top == top[0], 1.0, np.exp((top - top[0]) / temp))
    w[np.isnan(w)] = 0.0  # (-inf at an infinite temperature)
    w[w < unit / 2] = 0.0
    near = 1.0
    if 0 < k < n:
        w[k:] = 0.0
    if p < 1:
        before = np.cumsum(w) - w
        keep = before < p * w.sum()
        keep[0] = True
        near = min(near, np.abs(before - p * w.sum())[w > 0].min() / (w > 0).sum()) if p > 0 else near
        w[~keep] = 0.0
    if m > 0:
        w[w < min(m, 1.0)] = 0.0
    by_index = np.zeros(n)
    by_index[order] = w
    run, u = np.cumsum(by_index), min(max(0.0 if np.isnan(u) else float(u), 0.0), 1.0)
    total = run[-1]
    at = int(np.argmax((run > u * total) & (by_index > 0))) if u < 1 else int(np.flatnonzero(by_index)[-1])
    return at, by_index[at] / total, min(near, np.abs(run[by_index > 0] - u * total).min() / (by_index > 0).sum())


def check(x, u, temp=None, k=None, p=None, m=None, exact=False, ends=()):
    """Every row against the definition. The kernel's weights are integers of 2^-F of the largest (F at least 43: 2^19 tokens), off by half
    a unit, 2^-44, and by the 2^-46.6 that the exponential's polynomial leaves out ((ln 2 / 1024)^4 / 24 of itself), so by less than 2^-43.7: a sum by that times the number of its weights, the sum that it is
    compared with too. A row whose u (or whose top_p) comes nearer than twice that to a border is no judge, and there is hardly one.
    The probability is the quotient of two such sums, rounded to 32 bits. exact: sums without any rounding, every row counts. ends: rows
    whose u is one of the two outer borders: the first or last token that has a weight in those integers."""
    T, n = x.shape
    to = lambda v, dt: None if v is None else torch.tensor(np.asarray(v, dt), device="cuda")  # noqa: E731
    idx, prob = K.sample(torch.from_numpy(x).cuda(), to(u, np.float32), to(temp, np.float32), to(k, np.int32), to(p, np.float32), to(m, np.float32))
    idx, prob = idx.cpu().numpy(), prob.cpu().numpy()
    skipped = 0
    for r in range(T):
        pick = lambda v, d: d if v is None else np.float32(v[r]) if d != 0 else v[r]  # noqa: E731
        want, pr, near = draw(x[r].copy(), np.float32(u[r]), pick(temp, 1.0), 0 if k is None else int(k[r]), pick(p, 1.0), np.float32(0.0 if m is None else m[r]))
        if r in ends:
            want = draw(x[r].copy(), np.float32(u[r]), pick(temp, 1.0), 0 if k is None else int(k[r]), pick(p, 1.0), np.float32(0.0 if m is None else m[r]),
                        2.0 ** -min(50, 62 - int(np.ceil(np.log2(n)))))[0]
            assert idx[r] == want, (r, idx[r], want)
            continue
        if not exact and near < 2 * 2.0 ** -43.7:
            skipped += 1
            continue
        assert idx[r] == want, (r, idx[r], want, near)
        assert abs(prob[r] - pr) <= pr * 2.0 ** -23 + n * 2.0 ** -43, (r, prob[r], pr)
    assert skipped <= max(1, T // 20)


def logits(rng, T, n, peaks=20):
    x = rng.standard_normal((T, n)).astype(np.float32) * 2.2
    for r in range(T):
        x[r, rng.integers(0, n, min(peaks, n))] += rng.random(min(peaks, n)).astype(np.float32) * 14
    return x


SIZES = [1, 2, 3, 5, 31, 100, 2047, 2049, 4096, 4097, 16384, 16387, 32003, 49153, 128256, 152064, 360448]


@pytest.mark.parametrize("n", SIZES)
def test_sample_settings(cuda, n):
    """Every combination of the filters on and off, odd sizes, one CTA per row up to a whole cluster of full slices."""
    rng = np.random.default_rng(n)
    combos = [(t, k, p, m) for t in (0.7,) for k in (0, 1, 7, 50) for p in (1.0, 0.9, 0.3) for m in (0.0, 0.03)]
    combos += [(1.3, 0, 0.99, 0.0), (0.2, 0, 0.95, 0.0), (1.0, 900, 0.97, 0.0), (2.5, 1024, 1.0, 0.001), (1.0, 1025, 1.0, 0.0), (1.0, 3000, 0.8, 0.0), (3.0, n - 1, 0.999, 0.0),
               (1.0, n, 1.0, 0.0), (1.0, n + 5, 0.5, 0.0), (1.0, -3, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (5.0, 0, 0.9, 0.0)]
    T = len(combos)
    t, k, p, m = zip(*combos)
    check(logits(rng, T, n), rng.random(T, dtype=np.float32), t, k, p, m)


def test_sample_without_settings(cuda):
    rng = np.random.default_rng(1)
    x = logits(rng, 9, 5000)
    check(x, rng.random(9, dtype=np.float32))
    check(x, rng.random(9, dtype=np.float32), k=[3] * 9)
    check(x, rng.random(9, dtype=np.float32), p=[0.6] * 9)


@pytest.mark.parametrize("T,n", [(75, 50001), (512, 3000), (515, 700)])
def test_sample_many_rows(cuda, T, n):
    """More rows than run at once, of all kinds in turn: the long ones are taken first, and every row has its own result."""
    rng = np.random.default_rng(T)
    i = np.arange(T)
    check(logits(rng, T, n), rng.random(T, dtype=np.float32), np.where(i % 7 == 3, 0.0, 0.5 + i % 5 * 0.3), np.where(i % 3 == 0, 5 + i % 40, 0) + np.where(i % 11 == 5, 600, 0),
          np.where(i % 2 == 0, 0.9, 1.0), np.where(i % 4 == 1, 0.02, 0.0))


@pytest.mark.parametrize("n", [10, 1000, 40000, 130000])
def test_sample_equal_logits(cuda, n):
    """Logits that are all equal, or of a few values: the runs end inside ties, which go by index; every sum of equal weights is exact."""
    rng = np.random.default_rng(n)
    u = rng.random(24, dtype=np.float32)
    x = np.full((24, n), -2.5, np.float32)
    check(x, u, k=[0, 1, 2, 5, 9, n // 2, n - 1, min(n, 1500)] * 3, p=[1.0] * 8 + [0.5] * 8 + [0.25] * 8, exact=True)
    few = rng.integers(0, 3, (24, n)).astype(np.float32) * 50  # the weights of the lower ones are below 2^-62: nothing
    check(few, u, k=[0, 1, 2, 5, 9, n // 4, n - 1, min(n, 1500)] * 3, p=[1.0] * 8 + [0.5] * 8 + [0.125] * 8, exact=True)
    some = rng.integers(0, 6, (24, n)).astype(np.float32)
    check(some, u, k=[0, 1, 3, 5, 9, n // 3, n - 2, min(n, 1500)] * 3, p=[1.0] * 8 + [0.7] * 8 + [0.33] * 8, m=[0.0] * 12 + [0.1] * 12)


def test_sample_neighbouring_floats(cuda):
    """Several hundred each of floats that differ in their last two bits: the border lies in the last split of the bits."""
    rng = np.random.default_rng(12)
    x = (np.float32(1.0) + rng.integers(0, 4, (12, 2800)).astype(np.float32) * np.float32(2.0 ** -23)).astype(np.float32)
    x[6:, ::3] -= np.float32(3.0)
    check(x, rng.random(12, dtype=np.float32), k=[513, 650, 800, 1300, 1500, 0] * 2, p=[1.0, 0.9, 1.0, 1.0, 0.7, 0.4] * 2)


def test_sample_masked_and_infinite(cuda):
    """Tokens masked by -inf, by the lowest float, by NaN; rows with nothing left; +inf."""
    rng = np.random.default_rng(5)
    n, T = 6001, 16
    inf, low, nan = np.float32(np.inf), np.finfo(np.float32).min, np.float32(np.nan)
    x = logits(rng, T, n)
    x[0], x[1], x[2] = -inf, nan, low
    x[3, :] = -inf
    x[3, 77] = -5.0
    x[4, :], x[4, [5, 5000]] = low, [1.0, 0.5]
    x[5, ::2], x[6, 1::2], x[7, 10:] = -inf, nan, low
    x[8, [3, 4, 5999]], x[9, 6000] = inf, inf
    x[10, :], x[10, [9, 8]] = nan, inf
    x[11, :], x[11, 0] = -inf, nan
    x[12] = np.where(np.arange(n) % 3 == 0, -np.float32(0.0), np.float32(0.0))  # both zeros are one value
    for k in (0, 1, 4, 1500):
        for p in (1.0, 0.9):
            check(x, rng.random(T, dtype=np.float32), [0.8] * T, [k] * T, [p] * T)
    idx, prob = K.sample(torch.from_numpy(x).cuda(), torch.zeros(T, device=cuda), torch.zeros(T, device=cuda))
    assert idx.tolist()[:4] == [-1, -1, 0, 77] and idx.tolist()[8:12] == [3, 6000, 8, -1] and prob.tolist()[:3] == [0.0, 0.0, 1.0]


def test_sample_extreme_settings(cuda):
    rng = np.random.default_rng(6)
    n, inf, nan = 9000, np.inf, np.nan
    t = [1e-38, 1e-45, 1e30, inf, -1.0, nan, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5]
    u = [0.3, 0.3, 0.3, 0.3, 0.3, 0.3, 0.0, 1.0, -2.0, nan, inf, 1 - 2.0 ** -24, 0.4, 0.4, 0.4, 0.4]
    p = [1.0] * 12 + [0.0, -1.0, nan, 2.0]
    m = [0.0] * 12 + [0.0, 0.0, 5.0, nan]
    for k in (0, 40):
        check(logits(rng, 16, n), np.float32(u), t, [k] * 16, p, m, ends=range(6, 11))


def test_sample_more_rows_than_a_grid_is_high(cuda):
    rng = np.random.default_rng(11)
    T, n = 70000, 6
    x, u = rng.standard_normal((T, n)).astype(np.float32), rng.random(T, dtype=np.float32)
    w = np.exp(x.astype(np.float64) - x.max(1, keepdims=True))
    run = np.cumsum(w, 1)
    goal = u.astype(np.float64)[:, None] * run[:, -1:]
    judge = np.abs(run - goal).min(1) > 2 * n * 2.0 ** -43.7
    idx, prob = K.sample(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda())
    want = (run > goal).argmax(1)
    assert judge.sum() >= T - 10 and (idx.cpu().numpy() == want)[judge].all()
    assert np.abs(prob.cpu().numpy() - (w / run[:, -1:])[np.arange(T), want])[judge].max() <= 2.0 ** -23


def test_sample_is_the_inverse_of_the_running_sum(cuda):
    """u over a fine even grid draws every token as often as its probability says, give or take one."""
    rng = np.random.default_rng(7)
    n, N = 61, 20000
    x = np.repeat(rng.standard_normal((1, n)).astype(np.float32) * 2, N, 0)
    u = ((np.arange(N) + 0.5) / N).astype(np.float32)
    idx, prob = K.sample(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda())
    w = np.exp(x[0].astype(np.float64) - x[0].max())
    w /= w.sum()
    count = np.bincount(idx.cpu().numpy(), minlength=n)
    assert (np.abs(count - w * N) <= 1 + 2.0 ** -24 * N).all() and (np.diff(idx.cpu().numpy()) >= 0).all()
    assert np.abs(prob.cpu().numpy() - w[idx.cpu().numpy()]).max() <= 2.0 ** -23


def test_sample_rows_apart(cuda):
    """Rows of any distance and off their alignment; results of one call do not depend on the others' rows."""
    rng = np.random.default_rng(8)
    for n, off, wide in ((1003, 1, 1010), (50001, 3, 50010), (128, 0, 131), (70000, 4, 70004)):
        x = torch.from_numpy(logits(rng, 6, wide)).cuda()
        part, u = x[:, off:off + n], torch.rand(6, device=cuda)
        k, p = torch.tensor([0, 20, 0, 2000, 1, 60], dtype=torch.int32, device=cuda), torch.tensor([0.9, 0.9, 1.0, 0.8, 1.0, 0.5], device=cuda)
        a = K.sample(part, u, None, k, p)
        b = K.sample(part.contiguous(), u, None, k, p)
        c = [K.sample(part[r:r + 1].clone(), u[r:r + 1], None, k[r:r + 1], p[r:r + 1]) for r in range(6)]
        for i in range(2):
            assert torch.equal(a[i], b[i]) and torch.equal(a[i], torch.cat([y[i] for y in c]))


def test_sample_agrees_with_argmax_and_topk(cuda):
    rng = np.random.default_rng(9)
    x = torch.from_numpy(logits(rng, 5, 128256)).cuda()
    x[:, 100] = x[:, 99000] = x.amax(1) + 1
    zero = torch.zeros(5, device=cuda)
    assert torch.equal(K.sample(x, zero, temp=zero)[0], K.argmax(x)[:, 0])
    val, idx = K.topk(x, 40)
    u = torch.rand(5, device=cuda)
    got, prob = K.sample(x, u, top_k=torch.full((5,), 40, dtype=torch.int32, device=cuda))
    w = torch.softmax(val.double(), 1)
    assert all(int(got[r]) in idx[r].tolist() for r in range(5))
    assert torch.allclose(prob.double(), (w * (idx == got[:, None])).sum(1), rtol=2e-7, atol=0)


def test_sample_in_a_graph(cuda):
    """Captured once, replayed on a side stream with other logits, numbers and settings."""
    rng = np.random.default_rng(10)
    T, n = 4, 20000
    x, u = torch.zeros(T, n, device=cuda), torch.zeros(T, device=cuda)
    temp, k, p = torch.ones(T, device=cuda), torch.zeros(T, dtype=torch.int32, device=cuda), torch.ones(T, device=cuda)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            idx, prob = K.sample(x, u, temp, k, p)
        for i in range(6):
            h = logits(rng, T, n)
            x.copy_(torch.from_numpy(h)), u.copy_(torch.rand(T)), k.fill_(i % 3 * 30), p.fill_(1 - i % 2 * 0.2)
            graph.replay()
            for r in range(T):
                want, pr, near = draw(h[r].copy(), float(u[r]), 1.0, i % 3 * 30, float(p[r]))
                assert near < 2 * 2.0 ** -43.7 or (int(idx[r]) == want and abs(float(prob[r]) - pr) <= pr * 2.0 ** -23 + n * 2.0 ** -43)
    torch.cuda.current_stream().wait_stream(side)


def test_sample_wrapper_refuses(cuda):
    x, u = torch.zeros(2, 100, device=cuda), torch.zeros(2, device=cuda)
    for bad in (dict(x=x.half()), dict(x=x[0]), dict(x=x.T), dict(x=x[:1].expand(2, 100)), dict(u=u[:1]), dict(u=u.double()), dict(u=u.cpu()), dict(temp=torch.ones(1, device=cuda)),
                dict(top_k=u), dict(top_p=torch.ones(2, 1, device=cuda)), dict(min_p=torch.ones(2))):
        with pytest.raises((ValueError, AttributeError)):
            K.sample(**{**dict(x=x, u=u), **bad})
    with pytest.raises(K._lib.IeB200Error, match="360449"):
        K.sample(torch.zeros(1, 360449, device=cuda), u[:1])
    assert K.sample(x[:0], u[:0])[0].shape == (0,)
