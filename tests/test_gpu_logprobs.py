"""Scores of tokens against the same in 64 bits: log probabilities, ranks, entropy and the most likely tokens, at the row
lengths, strides, masks and ties where a kernel that reads a row once, in pieces, can go wrong."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def S():
    from ferrum_b200 import surface
    return surface


def run(d, l, n, ids, k, stride=None):
    """`l`: a flat CUDA tensor of logits.  Outputs with a guard behind them."""
    rows = len(ids)
    new = lambda count, dtype, fill: torch.full((count + 4,), fill, dtype=dtype, device="cuda")
    lp, rk, en = new(rows, F32, 9.5), new(rows, torch.int32, -9), new(rows, F32, 9.5)
    tp, ti = new(rows * k, F32, 9.5), new(rows * k, torch.int32, -9)
    dev_ids = torch.from_numpy(np.asarray(ids, np.int64).astype(np.uint32).view(np.int32)).cuda()
    torch.cuda.synchronize()
    S().token_logprobs(d, l, n, rows, dev_ids, lp[:rows], rk[:rows], en[:rows], k,
                       tp[:rows * k] if k else None, ti[:rows * k] if k else None, stride)
    d.synchronize()
    for t, count in ((lp, rows), (rk, rows), (en, rows), (tp, rows * k), (ti, rows * k)):
        assert torch.all(t[count:] == (9.5 if t.dtype == F32 else -9))
    out = [t[:c].cpu().numpy() for t, c in ((lp, rows), (rk, rows), (en, rows), (tp, rows * k), (ti, rows * k))]
    return out[:3] + [o.reshape(rows, k) for o in out[3:]]


def check(l, ids, k, got):
    """`l`: [rows, n] float64 of exactly the logits that were passed; the same in 64 bits by torch, on the device for its speed."""
    lp, rk, en, tp, ti = got
    rows, n = l.shape
    x = torch.from_numpy(np.ascontiguousarray(l)).cuda()
    id_ = torch.from_numpy(np.asarray(ids, np.int64)).cuda()
    mx = x.max(dim=1).values  # NaN where a row holds one
    e = (x - mx[:, None]).exp()
    s = e.sum(dim=1)
    z = mx + s.log()
    p = e / s[:, None]
    entropy = -torch.where(p > 0, p * (x - z[:, None]), 0.0).sum(dim=1)
    z, entropy = z.where(mx.isfinite(), float("nan")), entropy.where(mx.isfinite(), float("nan"))
    inside = id_ < n
    given = x.gather(1, id_.where(inside, 0)[:, None])[:, 0].where(inside, float("nan"))
    want = given - z
    rank = (1 + (x > given[:, None]).sum(dim=1)).where(inside, 0)
    want, rank, entropy, z = (t.cpu().numpy() for t in (want, rank, entropy, z))
    if k:
        # NaN goes behind -infinity, which the order below cannot say: only rows without NaN are compared by it.
        clean = ~x.isnan().any(dim=1).cpu().numpy()
        order = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :k].cpu().numpy()
        top = x.gather(1, torch.from_numpy(ti.astype(np.int64)).cuda()).cpu().numpy()
    # Sums: a term exp(d) carries the roundings of d (|d| * 2^-24 twice), 2^-22 of the exponential, and the additions of a
    # thread's share (n / 256 at the most) and of a tree; far terms weigh nothing, so |d| is taken at 100.  The entropy's
    # second sum has one rounding more in terms of at most |d| times the first's.
    sums = (2 * 100 + 4 + n / 256 + 24) * 2.0 ** -24
    off = lambda v: np.abs(v) * 2.0 ** -23 + sums
    def near(a, b, off):
        with np.errstate(all="ignore"):
            return np.array_equal(np.isnan(a), np.isnan(b)) and np.all((a == b) | np.isnan(b) | (np.abs(a - b) <= off))
    assert near(lp, want, off(want)), (lp, want)
    span = np.log(n) + 1
    assert near(en, entropy, off(entropy) * (1 + span)), (en, entropy)
    assert np.array_equal(rk, rank), (rk, rank)
    if k:
        assert np.array_equal(ti[clean], order[clean])
        with np.errstate(all="ignore"):
            want = top - z[:, None]
        assert near(tp, want, off(want))


def logits(rng, rows, n):
    l = 2.5 * rng.standard_normal((rows, n))
    l[np.arange(rows), rng.integers(0, n, rows)] += 12
    return l


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 5, 18, 130, 700])
@pytest.mark.parametrize("n", [1, 2, 3, 7, 31, 33, 128, 1000, 4099, 32000, 50257, 151936])
def test_rows_of_every_length(device, n, rows, dtype):
    if n > 40000 and rows > 130:
        rows = 300
    rng = np.random.default_rng(n + rows)
    l = torch.from_numpy(logits(rng, rows, n)).to(dtype)
    ids = rng.integers(0, n, rows)
    ids[::2] = l.float().argmax(1).numpy()[::2]
    for k in {0, 1, min(n, 5), min(n, 32)}:
        check(l.double().numpy(), ids, k, run(device, l.cuda().view(-1), n, ids, k))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 9, 200])
@pytest.mark.parametrize("n", [20, 777, 33000])
def test_masked_rows(device, n, rows, dtype):
    """Masks of -infinity and of the type's lowest value, at random, all but one token, the first part, everything."""
    rng = np.random.default_rng(n + rows)
    low = torch.finfo(dtype).min
    for kind in range(6):
        l = torch.from_numpy(logits(rng, rows, n)).to(dtype)
        mask = torch.from_numpy(rng.random((rows, n)) < 0.5)
        keep = rng.integers(0, n, rows)
        if kind in (1, 4):
            mask[:] = True
            mask[np.arange(rows), keep] = False
        if kind == 2:
            mask[:] = False
            mask[:, :n - n // 8] = True
        if kind == 5:
            mask[:] = True
        l = l.masked_fill(mask, -float("inf") if kind in (0, 1, 2, 5) else low)
        ids = rng.integers(0, n, rows)
        ids[::2] = keep[::2]
        check(l.double().numpy(), ids, min(n, 32), run(device, l.cuda().view(-1), n, ids, min(n, 32)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 40])
def test_ties_and_orders(device, rows, dtype):
    """Equal logits (the two zeros among them), rising and falling rows, a few values in all: ties go to the lower id."""
    n = 20011
    rng = np.random.default_rng(rows)
    for row in (np.zeros(n), np.full(n, -3.25), np.where(rng.random(n) < 0.5, 0.0, -0.0), np.arange(n) / 1024.0, -np.arange(n) / 1024.0,
                rng.integers(0, 3, n), rng.integers(0, 40, n), np.full(n, -np.inf)):
        l = torch.from_numpy(np.tile(np.asarray(row, np.float64), (rows, 1))).to(dtype)
        ids = rng.integers(0, n, rows)
        check(l.double().numpy(), ids, 32, run(device, l.cuda().view(-1), n, ids, 32))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_offsets_and_peaks(device, dtype):
    """Rows shifted far from zero, one token that takes nearly everything, values that grow towards the end of the row."""
    n, rng = 9000, np.random.default_rng(1)
    rows = []
    for shift in (0, 1000, -1000, 3e4):
        rows.append(np.round(rng.standard_normal(n) * 4) + shift)
    peak = rng.standard_normal(n)
    peak[4567] = 60
    late = rng.standard_normal(n) - 200
    late[-5:] = 150
    l = torch.from_numpy(np.stack(rows + [peak, late, np.linspace(-300, 300, n)])).to(dtype)
    ids = np.array([0, 5, 8999, 17, 4567, 8996, 3])
    check(l.double().numpy(), ids, 32, run(device, l.cuda().view(-1), n, ids, 32))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_without_a_distribution(device, dtype):
    n, rng = 3000, np.random.default_rng(2)
    for n in (17, 3000, 40000):
        l = logits(rng, 8, n)
        l[1, n // 3] = np.nan
        l[3, 0] = np.inf
        l[4, n - 1] = np.inf
        l[4, n // 2] = np.nan
        l[6, :] = np.nan
        t = torch.from_numpy(l).to(dtype)
        ids = rng.integers(0, n, 8)
        got = run(device, t.cuda().view(-1), n, ids, 8)
        x = t.double().numpy()
        ordered = np.where(np.isnan(x), -1e300, np.where(np.isinf(x), 1e300, x))  # no -infinity here: NaN is below everything
        assert np.array_equal(got[4], np.argsort(-ordered, axis=1, kind="stable")[:, :8])
        for row in (1, 3, 4, 6):
            assert np.isnan(got[0][row]) and np.isnan(got[2][row]) and np.all(np.isnan(got[3][row]))
        with np.errstate(all="ignore"):
            assert np.array_equal(got[1], 1 + (x > x[np.arange(8), ids][:, None]).sum(1))
        good = [0, 2, 5, 7]
        check(x[good], ids[good], 8, [g[good] for g in got])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,stride,first", [(1000, 1024, 0), (1001, 1001, 1), (1001, 1003, 3), (997, 1003, 5), (33000, 33007, 7), (151936, 151943, 1)])
def test_padded_and_unaligned_rows(device, n, stride, first, dtype):
    """Rows apart, and a buffer that begins anywhere; what lies between the rows is NaN and infinity and is not read."""
    rng, rows = np.random.default_rng(n), 6
    l = torch.from_numpy(logits(rng, rows, n)).to(dtype)
    whole = torch.full((first + rows * stride + 64,), float("nan"), dtype=dtype)
    whole[::2] = float("inf")
    for r in range(rows):
        whole[first + r * stride:first + r * stride + n] = l[r]
    buf = whole.cuda()[first:first + (rows - 1) * stride + n]
    ids = rng.integers(0, n, rows)
    check(l.double().numpy(), ids, 16, run(device, buf, n, ids, 16, stride))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,n", [(1, 700001), (19, 1400003), (700, 50003)])
def test_rows_of_more_pieces_than_are_noted(device, rows, n, dtype):
    """A block notes 40 (20, 80) maxima a thread; longer rows share them, and a row of many that no cluster cuts is long early."""
    rng = np.random.default_rng(n)
    l = torch.randn(rows, n, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").mul_(2.5).to(dtype)
    l[rows // 2, -9:] += 9  # in the last, shorter piece
    ids = rng.integers(0, n, rows)
    got = run(device, l.view(-1), n, ids, 32)
    some = np.unique(np.r_[0, rows // 2, rows - 1, rng.integers(0, rows, 4)])
    check(l[torch.from_numpy(some).cuda()].double().cpu().numpy(), ids[some], 32, [g[some] for g in got])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [40, 5000, 60000])
def test_alternatives_where_few_tokens_are_numbers(device, n, dtype):
    """Rows of NaN but for a few tokens, fewer than are asked for: numbers in their order, then NaN by id."""
    rng, k = np.random.default_rng(n), 32
    for numbers in (0, 1, 5, 31, 33):
        l = np.full((3, n), np.nan)
        for r in range(3):
            l[r, rng.choice(n, numbers, replace=False)] = rng.standard_normal(numbers)
        t = torch.from_numpy(l).to(dtype)
        got = run(device, t.cuda().view(-1), n, [0, 1, n - 1], k)
        x = t.double().numpy()
        assert np.array_equal(got[4], np.argsort(np.where(np.isnan(x), np.inf, -x), axis=1, kind="stable")[:, :k])
        assert all(np.isnan(got[i]).all() for i in (0, 2, 3))
        with np.errstate(all="ignore"):
            assert np.array_equal(got[1], 1 + (x > x[[0, 1, 2], [0, 1, n - 1]][:, None]).sum(1))


@pytest.mark.parametrize("rows", [1, 60])
def test_more_best_tokens_than_are_kept(device, rows):
    """Hundreds to thousands of logits above every thread's typical one: in few pieces, in all pieces, equal or growing."""
    n, rng = 50000, np.random.default_rng(7)
    base = rng.standard_normal(n)
    cases = []
    for count in (300, 513, 4000):
        for kind in range(4):
            x = base.copy()
            at = np.arange(1000, 1000 + count) if kind % 2 else rng.choice(n, count, replace=False)
            x[at] = 10 if kind < 2 else 10 + np.arange(count) / 8.0
            cases.append(x)
    for x in cases:
        l = torch.from_numpy(np.tile(x, (rows, 1))).float()
        for k in (1, 17, 32):
            ids = rng.integers(0, n, rows)
            check(l.double().numpy(), ids, k, run(device, l.cuda().view(-1), n, ids, k))


def test_rows_whose_offsets_pass_32_bits(device):
    """Rows 2^31 values apart, the third beyond 2^32 of them, and a row that is itself longer than 2^30."""
    rng, n, stride = np.random.default_rng(3), 50000, (1 << 31) + 5
    whole = torch.empty(2 * stride + n, dtype=BF16, device="cuda")
    l = torch.from_numpy(logits(rng, 3, n)).to(BF16)
    for r in range(3):
        whole[r * stride:r * stride + n] = l[r].cuda()
    ids = rng.integers(0, n, 3)
    check(l.double().numpy(), ids, 20, run(device, whole, n, ids, 20, stride))
    n = (1 << 31) - 9
    row = whole[3:3 + n].fill_(-30)
    at = np.sort(rng.choice(n, 6, replace=False))
    values = torch.tensor([1.0, 2.0, 3.0, 0.5, 2.0, -1.0], dtype=BF16)
    row[torch.from_numpy(at).cuda()] = values.cuda()
    lp, rk, en, tp, ti = run(device, row, n, [at[3]], 6)
    assert ti[0].tolist() == at[[2, 1, 4, 0, 3, 5]].tolist() and rk[0] == 5
    z = np.log(np.exp(values.double().numpy()).sum() + (n - 6) * np.exp(-30.0))
    # The six terms as in `check`, (2 * 100 + 28) * 2^-24 = 1.4e-5 of their sum, 39.6; the far ones are 2e-4 together, 5e-6 of it
    # even if all of them were lost beside larger ones.
    assert abs(lp[0] - (0.5 - z)) <= 1e-5 * 2 + 2.0 ** -18


def test_padding_rows_and_unwanted_outputs(device):
    """Ids that name no token, the same id in every row, and each output alone with the same values."""
    s, rng, n = S(), np.random.default_rng(4), 5000
    l = torch.from_numpy(logits(rng, 6, n)).float()
    ids = np.array([7, 0xFFFFFFFF, 4999, 5000, 7, 7])
    got = run(device, l.cuda().view(-1), n, ids, 3)
    assert np.isnan(got[0][[1, 3]]).all() and not got[1][[1, 3]].any()
    check(l.double().numpy(), ids, 3, got)
    x, new = l.cuda(), lambda dtype, *shape: torch.zeros(shape, dtype=dtype, device="cuda")
    dev_ids = torch.from_numpy(ids.astype(np.uint32).view(np.int32)).cuda()
    lp, rk, en, tp, ti = new(F32, 6), new(torch.int32, 6), new(F32, 6), new(F32, 6, 3), new(torch.int32, 6, 3)
    torch.cuda.synchronize()
    s.token_logprobs(device, x, n, 6, dev_ids, lp, None, None)
    s.token_logprobs(device, x, n, 6, dev_ids, None, rk, None)
    s.token_logprobs(device, x, n, 6, None, None, None, en)
    s.token_logprobs(device, x, n, 6, None, None, None, None, 3, tp, ti)
    device.synchronize()
    for a, b in zip((lp, rk, en, tp, ti), got):
        assert np.array_equal(a.cpu().numpy(), b, equal_nan=a.dtype == F32)


def test_repeated_calls_give_the_same_bits(device):
    rng = np.random.default_rng(6)
    for rows, n in ((1, 151936), (17, 50001), (400, 3001)):
        l = torch.from_numpy(logits(rng, rows, n)).float().cuda().view(-1)
        ids = rng.integers(0, n, rows)
        first = run(device, l, n, ids, 32)
        for _ in range(3):
            assert all(np.array_equal(a, b) for a, b in zip(first, run(device, l, n, ids, 32)))


def test_captured_and_replayed(device):
    """Two captured graphs of the same logits on one handle, replayed in turn with new logits, give what direct calls give."""
    s, n, rows, k = S(), 32000, 5, 20
    rng = np.random.default_rng(12)
    l, ids = torch.zeros(rows, n, device="cuda"), torch.from_numpy(rng.integers(0, n, rows).astype(np.int32)).cuda()
    out = [[torch.zeros(shape, dtype=t, device="cuda") for shape, t in ((rows, F32), (rows, torch.int32), (rows, F32), ((rows, k), F32), ((rows, k), torch.int32))] for _ in range(3)]
    call = lambda o: s.token_logprobs(device, l, n, rows, ids, o[0], o[1], o[2], k, o[3], o[4])
    torch.cuda.synchronize()
    graphs = []
    for o in out[:2]:
        device.capture_begin()
        call(o)
        graphs.append(device.capture_end())
    for step in range(3):
        l.copy_(torch.from_numpy(logits(rng, rows, n)).float())
        torch.cuda.synchronize()
        for g in graphs:
            g.launch()
        call(out[2])
        device.synchronize()
        for o in out[:2]:
            assert all(torch.equal(a, b) for a, b in zip(o, out[2]))


def test_refused_calls(device):
    s, d = S(), device
    l, ids = torch.zeros(4, 100, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    lp, rk, en = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    tp, ti = torch.zeros(4, 33, device="cuda"), torch.zeros(4, 33, dtype=torch.int32, device="cuda")
    before = d.counters().dispatches
    for call, error in ((lambda: s.token_logprobs(d, l, 101, 4, ids, lp, rk, en), s.ShapeError), (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, rk, en, stride=99), s.ShapeError),
                        (lambda: s.token_logprobs(d, l, 100, 4, ids[:3], lp, rk, en), s.ShapeError), (lambda: s.token_logprobs(d, l, 100, 4, ids, lp[:3], rk, en), s.ShapeError),
                        (lambda: s.token_logprobs(d, l.half(), 100, 4, ids, lp, rk, en), s.Unsupported), (lambda: s.token_logprobs(d, l, 100, 4, ids.long(), lp, rk, en), s.Unsupported),
                        (lambda: s.token_logprobs(d, l, 100, 4, None, lp, None, en), s.ParameterError), (lambda: s.token_logprobs(d, l, 100, 4, ids, None, None, None), s.ParameterError),
                        (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, rk, en, 33, tp, ti), s.ParameterError),
                        (lambda: s.token_logprobs(d, l, 4, 4, ids, lp, rk, en, 5, tp.view(-1)[:20], ti.view(-1)[:20]), s.ParameterError),
                        (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, rk, en, 2, None, ti.view(-1)[:8]), s.RangeError),
                        (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, rk, lp), s.AliasError), (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, ids, en), s.AliasError),
                        (lambda: s.token_logprobs(d, l, 100, 4, ids, l.view(-1)[:4], rk, en), s.AliasError),
                        (lambda: s.token_logprobs(d, l.cpu(), 100, 4, ids, lp, rk, en), s.DeviceMismatch)):
        with pytest.raises(error):
            call()
    assert d.counters().dispatches == before, "a refused call enqueues nothing"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,n", [(2000, 1), (2000, 64), (300, 5000), (20, 60000), (3, 151936), (600, 33000)])
def test_one_token_with_all_of_the_probability(device, rows, n, dtype):
    """Where a grammar allows one token, or one is far above the others: no log probability above 0, no entropy below it."""
    rng = np.random.default_rng(n)
    for below in (-np.inf, torch.finfo(dtype).min, -300.0):
        l = np.full((rows, n), below)
        keep = rng.integers(0, n, rows)
        l[np.arange(rows), keep] = rng.uniform(-40, 40, rows)
        t = torch.from_numpy(l).to(dtype)
        ids = keep.copy()
        ids[::5] = rng.integers(0, n, len(ids[::5]))
        for k in (0, min(n, 3)):
            got = run(device, t.cuda().view(-1), n, ids, k)
            check(t.double().numpy(), ids, k, got)
            assert (got[0] <= 0).all() and (got[2] >= 0).all() and (got[3] <= 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 74, 75, 296, 400])
@pytest.mark.parametrize("n", [8191, 8192, 8193, 16384, 65536])
def test_lengths_at_which_rows_are_cut_otherwise(device, n, rows, dtype):
    """8192 logits are the fewest that two blocks share, and the longest rows of the smallest blocks; 65536 the longest bf16 ones.
    A block notes 8 (of 256 threads; of 512: 4, of 128: 16) maxima a thread."""
    rng = np.random.default_rng(n + rows)
    l = torch.from_numpy(logits(rng, rows, n)).to(dtype)
    ids = rng.integers(0, n, rows)
    for k in (0, 7, 32):
        check(l.double().numpy(), ids, k, run(device, l.cuda().view(-1), n, ids, k))
