"""Rows in 8 bits and their projections against the same in 64 bits.  The 8-bit values and the projections' sums are exact, so
they are compared bit for bit; a scale is one fp32 number rounded from 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-6
F32, BF16 = torch.float32, torch.bfloat16


def S():
    from ferrum_b200 import surface
    return surface


def gpu(a, dtype=F32):
    return torch.as_tensor(np.ascontiguousarray(a)).to(dtype).cuda()


def f64(t):
    return t.detach().cpu().double().numpy()


def rows_to_8_bits(v, factor):
    """The definition on 64-bit rows: whole numbers (ties to even) and scales."""
    a = np.abs(v).max(axis=1, keepdims=True)
    q = np.rint(v * 127 / np.where(a > 0, a, 1))
    # The quotient is rounded twice, which takes a tie to either side of it; half of the largest value is one, and the two
    # products of that comparison are one number rounded once: 127 (a / 2) = 63.5 a.
    half = 127 * np.abs(v) == 63.5 * a
    q[half & (a > 0)] = (64 * np.sign(v))[half & (a > 0)]
    return q, (a * factor / 127)[:, 0]


def values_of(op, x, r, w):
    """(v, factor, h) of the operators' definition in 64 bits from tensors as they are passed."""
    if op == "quantize":
        return f64(x), 1.0, None
    if op == "glu":
        g, u = f64(x), f64(r)
        with np.errstate(over="ignore"):
            return g / (1 + np.exp(-g)) * u, 1.0, None
    h = x if op == "rmsnorm" else (x.float().cpu() + r.float().cpu()).to(x.dtype)
    v = f64(h)
    return v * f64(w), 1 / np.sqrt((v * v).mean(axis=1, keepdims=True) + np.float64(np.float32(EPS))), h


def run_op(d, op, x, r, w, rows, h=None):
    n = x.numel() // rows
    q, s = torch.full((rows + 1, n), 99, dtype=torch.int8, device="cuda"), torch.full((rows + 4,), -7.0, device="cuda")
    qq, ss = q[:rows], s[:rows]
    torch.cuda.synchronize()
    if op == "quantize":
        S().quantize_i8(d, x, rows, qq, ss)
    elif op == "rmsnorm":
        S().rmsnorm_i8(d, x, w, EPS, rows, qq, ss)
    elif op == "add":
        S().add_rmsnorm_i8(d, x, r, w, EPS, rows, h, qq, ss)
    else:
        S().glu_i8(d, x, r, rows, qq, ss)
    d.synchronize()
    assert torch.all(q[rows:] == 99) and torch.all(s[rows:] == -7), "nothing behind the last row is written"
    return qq.cpu().numpy(), ss.cpu().numpy()


def check_rows(op, x, r, w, q, s):
    v, factor, _ = values_of(op, x, r, w)
    want_q, want_s = rows_to_8_bits(v, factor)
    assert np.array_equal(q, want_q), np.argwhere(q != want_q)[:5]
    # Half an fp32 step; scales below 2^-126 have steps of 2^-149.  The norms' squares are added by fours in 32 bits, which
    # takes three roundings of at most 2^-24 of a sum, and half of that reaches 1/rms.
    off = 2.0 ** -24 * (2.5 if op in ("rmsnorm", "add") else 1)
    assert np.all(np.abs(s - want_s) <= want_s * off * (1 + 1e-6) + 2.0 ** -149)


OPS = ["quantize", "rmsnorm", "add", "glu"]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 3, 310])
@pytest.mark.parametrize("n", [4, 12, 128, 132, 516, 1024, 2048, 2052, 4100, 5120, 8200, 17408, 70004])
@pytest.mark.parametrize("op", OPS)
def test_rows_of_every_length(device, op, n, rows, dtype):
    if n > 20000 and rows > 3:
        rows = 150
    rng = np.random.default_rng(n + rows)
    x = gpu(rng.standard_normal((rows, n)) * (1 + 30 * (rng.random(n) < 0.01)), dtype)
    r, w = gpu(rng.standard_normal((rows, n)), dtype), gpu(1 + 0.1 * rng.standard_normal(n))
    h = torch.zeros_like(x)
    q, s = run_op(device, op, x, r, w, rows, h)
    check_rows(op, x, r, w, q, s)
    if op == "add":
        assert torch.equal(h.cpu(), values_of(op, x, r, w)[2])
        for place in (x.clone(), r.clone()):  # the sum in place of either input
            first = place if torch.equal(place, x) else x
            second = r if first is place else place
            assert np.array_equal(run_op(device, op, first, second, w, rows, place)[0], q) and torch.equal(place, h)


@pytest.mark.parametrize("op", ["rmsnorm", "glu"])
def test_values_next_to_a_border_fall_on_its_right_side(device, op):
    """Inputs for which the same formula in 32 bits rounds some values to the wrong whole number."""
    rows, n = 512, 8192
    rng = np.random.default_rng(5)
    x, r, w = gpu(rng.standard_normal((rows, n))), gpu(rng.standard_normal((rows, n))), gpu(1 + 0.1 * rng.standard_normal(n))
    v, factor, _ = values_of(op, x, r, w)
    a, b, c = (t.cpu().numpy() for t in (x, r, w))
    v32 = a * c if op == "rmsnorm" else a / (1 + np.exp(-a)) * b  # all of it in 32 bits
    v32 = v32 * (np.float32(127) / np.abs(v32).max(axis=1, keepdims=True))
    assert v32.dtype == np.float32
    assert np.any(np.rint(v32) != rows_to_8_bits(v, factor)[0]), "the inputs hold no such value"
    check_rows(op, x, r, w, *run_op(device, op, x, r, w, rows))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_go_to_the_even_number(device, dtype):
    v = np.concatenate([[127.0], np.arange(-126.5, 127, 1.0), [0.5, 1.5, -0.5, 2.5]])
    v = np.concatenate([v, np.zeros(-len(v) % 4)])[None]
    for scale in (1.0, 2.0 ** -40, 2.0 ** 60):
        x = gpu(v * scale, dtype)
        check_rows("quantize", x, None, None, *run_op(device, "quantize", x, None, None, 1))
        ones = torch.ones(v.shape[1], device="cuda")
        check_rows("rmsnorm", x, None, ones, *run_op(device, "rmsnorm", x, None, ones, 1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 60, 2.0 ** -90])
@pytest.mark.parametrize("op", OPS)
def test_half_of_the_largest_value_goes_to_64(device, op, size, dtype):
    """63.5 is a tie, at sizes that are rounded in 32 bits and at those that are in 64, whatever the products' own roundings."""
    rng, rows, n = np.random.default_rng(5), 400, 72
    x, r, w = size * 0.1 * rng.standard_normal((rows, n)), np.zeros((rows, n)), 1 + 0.1 * rng.standard_normal(n)
    w[1] = w[0]
    x[:, 0] = size * (1 + rng.random(rows)) * rng.choice([-1, 1], rows)
    if op == "glu":  # of one gate
        x, r = rng.standard_normal((rows, n)), x
        x[:, :2] = 1 + 4 * rng.random((rows, 1))
    x, r, w = gpu(x, dtype), gpu(r, dtype), gpu(w)
    t = r if op == "glu" else x
    t[:, 1] = t[:, 0] / 2
    q, s = run_op(device, op, x, r, w, rows, torch.zeros_like(x))
    v = values_of(op, x, r, w)[0]
    assert np.all(np.abs(v).argmax(1) == 0)
    assert np.array_equal(q[:, 0], 127 * np.sign(v[:, 0])) and np.array_equal(q[:, 1], 64 * np.sign(v[:, 0]))
    check_rows(op, x, r, w, q, s)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [64, 5120])
@pytest.mark.parametrize("op", OPS)
def test_rows_of_extreme_values(device, op, n, dtype):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((12, n))
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 2.0 ** -130   # subnormal in fp32
    x[3] *= 1e37 / np.abs(x[3]).max()
    x[4], x[5, :-1] = 0, 0
    x[4, n // 2] = -3.0
    x[5, -1] = 1e-38
    x[6] = -100.0 + x[6]  # a gate that closes: silu of -100
    r = rng.standard_normal((12, n))
    r[3] *= 1e-3
    r[0] = 0 if op != "glu" else r[0]
    if op == "glu":
        r[7] = 0
    x[8], r[8] = x[8] * 2.0 ** -130, r[8] * 2.0 ** -131  # a sum of subnormal numbers
    x[9] *= 2.0 ** (rng.integers(-30, 30, n))            # and sums that lose the smaller one's last bits
    x, r, w = gpu(x, dtype), gpu(r, dtype), gpu(1 + 0.1 * rng.standard_normal(n))
    h = torch.zeros_like(x)
    q, s = run_op(device, op, x, r, w, 12, h)
    check_rows(op, x, r, w, q, s)
    if op == "add":
        assert torch.equal(h.cpu(), values_of(op, x, r, w)[2])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [64, 5120])
@pytest.mark.parametrize("op", OPS)
def test_a_row_that_is_not_finite_spoils_itself_only(device, op, n, dtype):
    rng = np.random.default_rng(n + 1)
    x, r = rng.standard_normal((9, n)), rng.standard_normal((9, n))
    for row, bad in ((1, np.inf), (3, -np.inf), (5, np.nan)):
        x[row, rng.integers(n)] = bad
    if op in ("add", "glu"):
        r[7, rng.integers(n)] = np.nan
    x, r, w = gpu(x, dtype), gpu(r, dtype), gpu(1 + 0.1 * rng.standard_normal(n))
    q, s = run_op(device, op, x, r, w, 9, torch.zeros_like(x))
    bad = [1, 3, 5] + ([7] if op in ("add", "glu") else [])
    good = [i for i in range(9) if i not in bad]
    assert np.all(np.isnan(s[bad])) and not q[bad].any()
    pick = lambda t: None if t is None else t[good]
    check_rows(op, pick(x), pick(r), w, q[good], s[good])


def matrix(rng, d, rows, cols):
    wq = rng.integers(-128, 128, (rows, cols), dtype=np.int8)
    ws = (0.01 + rng.random(rows)).astype(np.float32) * rng.choice([-1, 1], rows).astype(np.float32)
    return S().Matrix.from_i8(d, wq, ws), wq, ws


def expect(xq, xs, wq, ws):
    """Exact sums (whole numbers in 64 bits), rounded to fp32, times the token's scale, times the row's: fp32 steps."""
    acc = (torch.from_numpy(xq).double().cuda() @ torch.from_numpy(wq).double().cuda().T).cpu().numpy()
    return acc.astype(np.float32) * xs[:, None] * ws[None]


def project(d, mats, xq, xs, dtype, many):
    m = len(xq)
    bufs = [torch.full((m * w.rows + 64,), 5.5, dtype=dtype, device="cuda") for w in mats]
    ys = [b[:m * w.rows] for b, w in zip(bufs, mats)]
    x, scales = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
    torch.cuda.synchronize()
    if many:
        S().project_many_i8(d, mats, x, scales, m, ys)
    else:
        for w, y in zip(mats, ys):
            S().project_i8(d, w, x, scales, m, y)
    d.synchronize()
    assert all(torch.all(b[m * w.rows:] == 5.5) for b, w in zip(bufs, mats)), "nothing behind the last row is written"
    return [y.view(m, w.rows) for y, w in zip(ys, mats)]


def same(y, want):
    return torch.equal(y.cpu(), torch.from_numpy(want).to(y.dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m", [1, 2, 7, 16, 17, 33, 64, 65, 128, 130, 256, 257, 300, 513])
@pytest.mark.parametrize("rows,cols", [(1, 16), (100, 48), (128, 128), (129, 144), (300, 1040), (1000, 2048), (2500, 4096), (5121, 528)])
def test_projections_of_every_shape(device, rows, cols, m, dtype):
    rng = np.random.default_rng(rows + m)
    w, wq, ws = matrix(rng, device, rows, cols)
    xq, xs = rng.integers(-128, 128, (m, cols), dtype=np.int8), rng.random(m).astype(np.float32)
    assert same(project(device, [w], xq, xs, dtype, False)[0], expect(xq, xs, wq, ws))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shapes,cols,m", [((20011,), 528, 16), ((20011,), 16, 1), ((19000, 5, 300), 1040, 70), ((40000,), 144, 130),  # more items than blocks
                                           ((5000, 3001), 1040, 600), ((10007,), 272, 1100), ((5121, 1000), 2064, 2048), ((4000,), 2048, 1030),  # pairs, several items each
                                           ((257,), 20000, 700), ((3000,), 4112, 700),  # pairs, one item
                                           ((1000,), 8208, 300), ((2500,), 16400, 33), ((640,), 8208, 40), ((1500,), 4112, 17), ((700,), 65536, 250)])  # clusters
def test_projections_of_every_cut(device, shapes, cols, m, dtype):
    """Products large enough to be cut in each of the ways there are."""
    rng = np.random.default_rng(cols + m)
    mats = [matrix(rng, device, r, cols) for r in shapes]
    xq, xs = rng.integers(-128, 128, (m, cols), dtype=np.int8), rng.random(m).astype(np.float32)
    for y, (_, wq, ws) in zip(project(device, [w for w, _, _ in mats], xq, xs, dtype, True), mats):
        assert same(y, expect(xq, xs, wq, ws))


@pytest.mark.parametrize("m", [1, 16, 260])
def test_the_largest_sums(device, m):
    """65536 products of 2^14: 2^30 fits, and so does its negative."""
    wq, ws = np.full((130, 65536), -128, np.int8), np.ones(130, np.float32)
    w = S().Matrix.from_i8(device, wq, ws)
    xq, xs = np.full((m, 65536), -128, np.int8), np.ones(m, np.float32)
    xq[m // 2] = 127
    assert same(project(device, [w], xq, xs, F32, False)[0], expect(xq, xs, wq, ws))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m", [1, 5, 40, 200, 700])
@pytest.mark.parametrize("shapes", [(6144, 1024, 1024), (257, 1), (130, 1000, 3, 64, 128, 129, 7, 640)])
def test_several_matrices_in_one_launch(device, shapes, m, dtype):
    rng = np.random.default_rng(m)
    cols = 1296
    mats = [matrix(rng, device, r, cols) for r in shapes]
    xq, xs = rng.integers(-127, 128, (m, cols), dtype=np.int8), rng.random(m).astype(np.float32)
    ys = project(device, [w for w, _, _ in mats], xq, xs, dtype, True)
    for y, (_, wq, ws) in zip(ys, mats):
        assert same(y, expect(xq, xs, wq, ws))
    again = project(device, [mats[0][0]] * 2, xq, xs, dtype, True)  # the same matrix twice
    assert torch.equal(again[0], ys[0]) and torch.equal(again[1], ys[0])


def test_a_matrix_made_on_the_device_or_the_host(device):
    rng = np.random.default_rng(0)
    x = gpu(rng.standard_normal((300, 272)))
    q, s = torch.zeros(300, 272, dtype=torch.int8, device="cuda"), torch.zeros(300, device="cuda")
    torch.cuda.synchronize()
    S().quantize_i8(device, x, 300, q, s)  # weights of floats, quantised where they are
    mats = [S().Matrix.from_i8(device, q, s), S().Matrix.from_i8(device, q.cpu(), s.cpu()), S().Matrix.from_i8(device, q.cpu().numpy(), s)]
    assert (mats[0].rows, mats[0].cols, mats[0].experts, mats[0].format, mats[0].byte_size()) == (300, 272, 1, S().I8, 300 * 276)
    xq, xs = rng.integers(-127, 128, (3, 272), dtype=np.int8), np.ones(3, np.float32)
    ys = project(device, mats, xq, xs, F32, True)
    assert same(ys[0], expect(xq, xs, q.cpu().numpy(), s.cpu().numpy())) and torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


def test_scales_that_are_not_finite_spoil_their_row_only(device):
    rng = np.random.default_rng(3)
    w, wq, ws = matrix(rng, device, 200, 160)
    xq, xs = rng.integers(-127, 128, (6, 160), dtype=np.int8), rng.random(6).astype(np.float32)
    want = expect(xq, xs, wq, ws)
    xs[2] = np.nan
    y = project(device, [w], xq, xs, F32, False)[0].cpu().numpy()
    assert np.all(np.isnan(y[2])) and np.array_equal(np.delete(y, 2, 0), np.delete(want, 2, 0))


def test_refused_calls(device):
    s, d = S(), device
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    q, sc = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    before = d.counters().dispatches
    with pytest.raises(s.ShapeError):
        s.quantize_i8(d, x, 3, q, sc)
    with pytest.raises(s.ShapeError):  # rows of 6 values
        s.quantize_i8(d, x.view(-1)[:24], 4, q.view(-1)[:24], sc)
    with pytest.raises(s.Unsupported):
        s.quantize_i8(d, x.half(), 4, q, sc)
    with pytest.raises(s.Unsupported):
        s.quantize_i8(d, x, 4, q.view(torch.uint8), sc)
    with pytest.raises(s.AliasError):
        s.quantize_i8(d, x, 4, x.view(torch.int8).view(-1)[:256].view(4, 64), sc)
    with pytest.raises(s.AliasError):
        s.rmsnorm_i8(d, x, w, EPS, 4, q, w[:4])
    with pytest.raises(s.RangeError):
        s.rmsnorm_i8(d, x.view(-1)[1:253 - 188], w[:16], EPS, 4, q.view(-1)[:64], sc)
    with pytest.raises(s.AliasError):  # h over part of x
        s.add_rmsnorm_i8(d, x[:2], x[2:], w, EPS, 2, x[1:3], q[:2], sc[:2])
    with pytest.raises(s.Unsupported):
        s.add_rmsnorm_i8(d, x, x.bfloat16(), w, EPS, 4, x.clone(), q, sc)
    with pytest.raises(s.Unsupported):
        s.glu_i8(d, x, x.bfloat16(), 4, q, sc)
    with pytest.raises(s.ShapeError):
        s.glu_i8(d, x, x[:2], 4, q, sc)
    with pytest.raises(s.DeviceMismatch):
        s.glu_i8(d, x, x.cpu(), 4, q, sc)
    ok = s.Matrix.from_i8(d, np.ones((32, 64), np.int8), np.ones(32, np.float32))
    for bad, error in (((np.ones((32, 24), np.int8), np.ones(32, np.float32)), s.ShapeError), ((np.ones((32, 65552), np.int8), np.ones(32, np.float32)), s.ShapeError),
                       ((np.ones((32, 64), np.int8), np.ones(31, np.float32)), s.ShapeError), ((np.ones((32, 64), np.uint8), np.ones(32, np.float32)), s.Unsupported),
                       ((np.ones((32, 64), np.int8), np.full(32, np.inf, np.float32)), s.WeightError)):
        with pytest.raises(error):
            s.Matrix.from_i8(d, *bad)
    y = torch.zeros(4, 32, device="cuda")
    with pytest.raises(s.ShapeError):
        s.project_i8(d, ok, q, sc, 4, y[:3])
    with pytest.raises(s.ShapeError):
        s.project_i8(d, ok, q[:3], sc, 4, y)
    with pytest.raises(s.ShapeError):
        s.project_i8(d, ok, q, sc[:3], 4, y)
    with pytest.raises(s.Unsupported):
        s.project_i8(d, ok, q, sc, 4, y.half())
    with pytest.raises(s.Unsupported):
        s.project_i8(d, ok, x, sc, 4, y)
    with pytest.raises(s.AliasError):
        s.project_many_i8(d, [ok, ok], q, sc, 4, [y, y])
    with pytest.raises(s.ParameterError):
        s.project_many_i8(d, [ok] * 9, q, sc, 4, [torch.zeros(4, 32, device="cuda") for _ in range(9)])
    with pytest.raises(s.ParameterError):
        s.project_many_i8(d, [], q, sc, 4, [])
    other = s.Device(0)
    with pytest.raises(s.DeviceMismatch):
        s.project_i8(other, ok, q, sc, 4, y)
    from oracle import ref
    packed = s.Matrix.from_packed(d, 32, 64, 1, s.Q8_0, ref.random_matrix(ref.Q8_0, 32, 64, seed=0))
    with pytest.raises(s.Unsupported):
        s.project_i8(d, packed, q, sc, 4, y)
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (lambda: s.project(d, ok, x, 4, y), lambda: s.project_many(d, [packed, ok], x, 4, [y, y.clone()]),
                 lambda: s.rmsnorm_project_many(d, [packed, ok], x, w, EPS, 4, [y, y.clone()], torch.zeros_like(x)),
                 lambda: s.project_id(d, ok, x, ids, 4, 1, y), lambda: s.project_mm_id(d, ok, x, torch.tensor([0, 4], dtype=torch.int32, device="cuda"), 4, y),
                 lambda: s.get_rows(d, ok, ids, x.clone()), lambda: s.dense_ffn(d, packed, packed, ok, x, 4, torch.zeros(4 * 96, device="cuda"), x.clone())):
        with pytest.raises(s.Unsupported):
            call()
    assert d.counters().dispatches == before, "a refused call enqueues nothing"


@pytest.mark.parametrize("op", OPS)
def test_rows_of_zeros_without_eps(device, op):
    """Nothing divides by nothing: scale 0 and whole numbers 0, beside a row that has values."""
    for n in (64, 5120, 60000):
        x = torch.zeros(3, n, device="cuda")
        x[1] = 1
        q, s = torch.full((3, n), 9, dtype=torch.int8, device="cuda"), torch.full((3,), 9.0, device="cuda")
        w, zeros = torch.ones(n, device="cuda"), torch.zeros_like(x)
        torch.cuda.synchronize()
        if op == "quantize":
            S().quantize_i8(device, x, 3, q, s)
        elif op == "rmsnorm":
            S().rmsnorm_i8(device, x, w, 0.0, 3, q, s)
        elif op == "add":
            S().add_rmsnorm_i8(device, x, zeros, w, 0.0, 3, torch.empty_like(x), q, s)
        else:
            S().glu_i8(device, x, x, 3, q, s)
        device.synchronize()
        assert not q[[0, 2]].any() and not s[[0, 2]].any() and torch.all(q[1] == 127) and s[1] > 0


@pytest.mark.parametrize("first", [1, 2, 3])
def test_later_rows_of_a_batch(device, first):
    """A call on some rows of larger arrays: scales begin at any 4 bytes, and what lies around the rows stays as it was."""
    rng = np.random.default_rng(first)
    w, wq, ws = matrix(rng, device, 200, 272)
    x = gpu(rng.standard_normal((9, 272)))
    q, sc, y = torch.full((9, 272), 5, dtype=torch.int8, device="cuda"), torch.full((9,), 5.0, device="cuda"), torch.full((9, 200), 5.0, device="cuda")
    part = slice(first, first + 4)
    torch.cuda.synchronize()
    S().quantize_i8(device, x[part], 4, q[part], sc[part])
    S().project_i8(device, w, q[part], sc[part], 4, y[part])
    device.synchronize()
    check_rows("quantize", x[part], None, None, q[part].cpu().numpy(), sc[part].cpu().numpy())
    assert same(y[part], expect(q[part].cpu().numpy(), sc[part].cpu().numpy(), wq, ws))
    around = [i for i in range(9) if not first <= i < first + 4]
    assert torch.all(q[around] == 5) and torch.all(sc[around] == 5) and torch.all(y[around] == 5)


def test_matrices_that_share_rows_are_one_launch(device):
    rng = np.random.default_rng(8)
    mats = [matrix(rng, device, r, 160) for r in (64, 200, 1)]
    x, sc = gpu(rng.integers(-127, 128, (5, 160)), torch.int8), torch.ones(5, device="cuda")
    ys = [torch.zeros(5, r, device="cuda") for r in (64, 200, 1)]
    torch.cuda.synchronize()
    before = device.counters().dispatches
    S().project_many_i8(device, [w for w, _, _ in mats], x, sc, 5, ys)
    assert device.counters().dispatches == before + 1


def test_on_other_streams_and_handles():
    """A handle on torch's streams, one after the other, and a second handle beside it: each call is in its stream's order."""
    s, rng = S(), np.random.default_rng(9)
    wq, ws = rng.integers(-127, 128, (700, 1040), dtype=np.int8), np.ones(700, np.float32)
    handles = [s.Device(0, use_torch_stream=False) for _ in range(2)]
    mats = [s.Matrix.from_i8(d, wq, ws) for d in handles]
    streams = [torch.cuda.Stream() for _ in range(2)]
    x = [gpu(rng.standard_normal((6, 1040))) for _ in range(2)]
    q = [torch.zeros(6, 1040, dtype=torch.int8, device="cuda") for _ in range(2)]
    sc, y = [torch.zeros(6, device="cuda") for _ in range(2)], [torch.zeros(6, 700, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for step in range(4):
        for i in range(2):
            stream = streams[(i + step) % 2]
            with torch.cuda.stream(stream):
                handles[i].set_stream(stream.cuda_stream)
                x[i].mul_(-0.75)  # on the same stream, before and after
                s.quantize_i8(handles[i], x[i], 6, q[i], sc[i])
                s.project_i8(handles[i], mats[i], q[i], sc[i], 6, y[i])
                result = y[i].clone()
            stream.synchronize()
            check_rows("quantize", x[i], None, None, q[i].cpu().numpy(), sc[i].cpu().numpy())
            assert same(result, expect(q[i].cpu().numpy(), sc[i].cpu().numpy(), wq, ws))
    for d, w in zip(handles, mats):
        w.close()
        d.close()


def test_an_injected_failure_launches_nothing():
    """A refused submission leaves the outputs as they were; after the recovery the same call gives the result."""
    s, rng = S(), np.random.default_rng(10)
    d = s.Device(0)
    w, wq, ws = matrix(rng, d, 130, 64)
    x, q, sc, y = gpu(rng.standard_normal((3, 64))), torch.zeros(3, 64, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(3, 130, device="cuda")
    lp = torch.zeros(3, device="cuda")
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    calls = (lambda: s.quantize_i8(d, x, 3, q, sc), lambda: s.project_i8(d, w, q, sc, 3, y), lambda: s.token_logprobs(d, y, 130, 3, ids, lp, None, None))
    for call, out in zip(calls, (q, y, lp)):
        d.fail_after(0)
        with pytest.raises(s.SynchronizationError):
            call()
        d.recover()
        d.synchronize()
        assert not out.any()
        call()
        d.synchronize()
        assert out.any()


def test_rows_whose_offsets_pass_32_bits(device):
    """2^32 values and more: every row is one of 64 that a call of their own has given."""
    n, rows = 4096, (1 << 20) + 64
    x = torch.randn(64, n, generator=torch.Generator().manual_seed(1)).cuda().bfloat16()
    w = torch.ones(n, device="cuda")
    few = [torch.zeros(64, n, dtype=torch.int8, device="cuda"), torch.zeros(64, device="cuda")]
    many = [torch.zeros(rows, n, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")]
    every = x.repeat(rows // 64, 1)
    torch.cuda.synchronize()
    for op in ("quantize", "rmsnorm", "glu"):
        for t, m, out in ((x, 64, few), (every, rows, many)):
            out[0].zero_()
            torch.cuda.synchronize()
            if op == "quantize":
                S().quantize_i8(device, t, m, *out)
            elif op == "rmsnorm":
                S().rmsnorm_i8(device, t, w, EPS, m, *out)
            else:
                S().glu_i8(device, t, t, m, *out)
            device.synchronize()
        assert torch.equal(many[0].view(-1, 64, n), few[0].expand(rows // 64, 64, n)) and torch.equal(many[1].view(-1, 64), few[1].expand(rows // 64, 64))


def test_products_whose_offsets_pass_32_bits(device):
    """70000 tokens by 64000 rows, 4.48e9 outputs: as torch has them in fp32, where sums of 16 products are exact."""
    rng = np.random.default_rng(2)
    m, rows, cols = 70000, 64000, 16
    w, wq, ws = matrix(rng, device, rows, cols)
    x, sc = gpu(rng.integers(-127, 128, (m, cols)), torch.int8), gpu(rng.random(m).astype(np.float32))
    y = torch.zeros(m, rows, dtype=BF16, device="cuda")
    torch.cuda.synchronize()
    S().project_i8(device, w, x, sc, m, y)
    device.synchronize()
    wt, ws = gpu(wq).t().contiguous(), gpu(ws)
    for t in (0, 33333, 67106, m - 600):  # row 67108 begins beyond 2^32 values
        part = slice(t, t + 600)
        assert torch.equal(y[part], ((x[part].float() @ wt) * sc[part, None] * ws).to(BF16))


def test_a_layer_on_8_bits_captured_and_replayed():
    """norm -> gate | up -> gated unit -> down -> norm -> output head -> scores on the handle's own stream: eagerly, then as a
    graph that is replayed on other inputs, beside a second graph of the same handle."""
    s = S()
    d = s.Device(0, use_torch_stream=False)
    rng = np.random.default_rng(11)
    hidden, ffn, vocab = 256, 688, 1003
    mats = {n: matrix(rng, d, r, c) for n, (r, c) in {"gate": (ffn, hidden), "up": (ffn, hidden), "down": (hidden, ffn), "head": (vocab, hidden)}.items()}
    w1, w2 = gpu(1 + 0.1 * rng.standard_normal(hidden)), gpu(1 + 0.1 * rng.standard_normal(hidden))

    def state(m):
        new = lambda *shape, dtype=F32: torch.zeros(shape, dtype=dtype, device="cuda")
        return {"m": m, "x": new(m, hidden), "r": new(m, hidden), "h": new(m, hidden), "q": new(m, hidden, dtype=torch.int8), "s": new(m),
                "g": new(m, ffn), "u": new(m, ffn), "a": new(m, ffn, dtype=torch.int8), "as": new(m), "d": new(m, hidden), "h2": new(m, hidden),
                "l": new(m, vocab), "ids": torch.arange(m, dtype=torch.int32, device="cuda"), "lp": new(m), "rk": new(m, dtype=torch.int32),
                "en": new(m), "tp": new(m, 4), "ti": new(m, 4, dtype=torch.int32)}

    def step(t):
        m = t["m"]
        s.add_rmsnorm_i8(d, t["x"], t["r"], w1, EPS, m, t["h"], t["q"], t["s"])
        s.project_many_i8(d, [mats["gate"][0], mats["up"][0]], t["q"], t["s"], m, [t["g"], t["u"]])
        s.glu_i8(d, t["g"], t["u"], m, t["a"], t["as"])
        s.project_i8(d, mats["down"][0], t["a"], t["as"], m, t["d"])
        s.add_rmsnorm_i8(d, t["h"], t["d"], w2, EPS, m, t["h2"], t["q"], t["s"])
        s.project_i8(d, mats["head"][0], t["q"], t["s"], m, t["l"])
        s.token_logprobs(d, t["l"], vocab, m, t["ids"], t["lp"], t["rk"], t["en"], 4, t["tp"], t["ti"])

    def fill(t, seed):
        g = torch.Generator().manual_seed(seed)
        t["x"].copy_(torch.randn(t["m"], hidden, generator=g))
        t["r"].copy_(torch.randn(t["m"], hidden, generator=g))
        torch.cuda.synchronize()

    def check(t):
        x, r = t["x"], t["r"]
        v, factor, h = values_of("add", x, r, w1)
        q, sc = rows_to_8_bits(v, factor)
        sc = sc.astype(np.float32)
        proj = lambda n, q, sc: expect(q.astype(np.int8), sc, mats[n][1], mats[n][2])
        assert torch.equal(t["h"].cpu(), h)
        # A scale is off by up to 2.5 * 2^-24 and its expectation by half a step, and each side's two products are rounded:
        # (2.5 + 1 + 4) * 2^-24 < 2^-21.
        g, u = t["g"].cpu(), t["u"].cpu()
        close = lambda a, b: np.all(np.abs(a - b) <= np.abs(b) * 2.0 ** -21)
        assert close(g.numpy(), proj("gate", q, sc)) and close(u.numpy(), proj("up", q, sc))
        v, factor, _ = values_of("glu", g, u, None)
        a, asc = rows_to_8_bits(v, factor)
        assert np.array_equal(t["a"].cpu().numpy(), a)
        assert close(t["d"].cpu().numpy(), proj("down", a, asc.astype(np.float32)))
        v, factor, h2 = values_of("add", t["h"], t["d"], w2)
        q, sc = rows_to_8_bits(v, factor)
        assert np.array_equal(t["q"].cpu().numpy(), q) and torch.equal(t["h2"].cpu(), h2)
        l = f64(t["l"])
        assert close(l, proj("head", q, sc.astype(np.float32)))
        z = np.log(np.exp(l - l.max(1, keepdims=True)).sum(1)) + l.max(1)
        got = l[np.arange(t["m"]), np.arange(t["m"])]
        # These logits reach thousands, where one fp32 rounding of the result is 2^-24 of it; 1e-4 is for the sums.
        assert np.all(np.abs(t["lp"].cpu().numpy() - (got - z)) <= np.abs(got - z) * 2.0 ** -23 + 1e-4)
        assert np.array_equal(t["rk"].cpu().numpy(), 1 + (l > got[:, None]).sum(1))
        assert np.array_equal(t["ti"].cpu().numpy(), np.argsort(-l, axis=1, kind="stable")[:, :4])

    a, b = state(3), state(40)
    fill(a, 1), fill(b, 2)
    step(a), step(b)
    d.synchronize()
    check(a), check(b)
    graphs = []
    for t in (a, b):
        d.capture_begin()
        step(t)
        graphs.append(d.capture_end())
    fill(a, 3), fill(b, 4)
    for _ in range(2):
        for g in graphs:
            g.launch()
    d.synchronize()
    check(a), check(b)
    for g in graphs:
        g.close()
    d.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [9e35, 2.5e36, 5e36, 2e37])
@pytest.mark.parametrize("n", [72, 4096])
@pytest.mark.parametrize("op", OPS)
def test_half_of_a_largest_value_whose_products_pass_the_end_of_fp32(device, op, n, size, dtype):
    """127 times half of these, and 63.5 times their whole, are about fp32's largest number and beyond it."""
    rng, rows = np.random.default_rng(6), 400
    x, r, w = size * 0.1 * rng.standard_normal((rows, n)), np.zeros((rows, n)), 1 + 0.1 * rng.standard_normal(n)
    x = np.clip(x, -0.4 * size, 0.4 * size)
    w[:2] = w.max()
    x[:, 0] = size * (1 + rng.random(rows)) * rng.choice([-1, 1], rows)
    if op == "glu":  # of one gate, the largest of the row
        x, r = rng.standard_normal((rows, n)), x
        x[:, :2] = 4 + rng.random((rows, 1))
    x, r, w = gpu(x, dtype), gpu(r, dtype), gpu(w)
    t = r if op == "glu" else x
    t[:, 1] = t[:, 0] / 2
    q, s = run_op(device, op, x, r, w, rows, torch.zeros_like(x))
    v = values_of(op, x, r, w)[0]
    assert np.all(np.abs(v).argmax(1) == 0)
    assert np.array_equal(q[:, 0], 127 * np.sign(v[:, 0])) and np.array_equal(q[:, 1], 64 * np.sign(v[:, 0]))
    check_rows(op, x, r, w, q, s)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [4e-20, 1e-18, 1.0])
@pytest.mark.parametrize("n", [1024, 5120, 20480, 70004])
def test_gates_far_below_zero(device, n, size, dtype):
    """silu of a gate below -88 is next to nothing: beside a large `up` it is still nothing to a row of small values."""
    rng, rows = np.random.default_rng(n), 24
    x, r = 1 + np.abs(rng.standard_normal((rows, n))), size * rng.standard_normal((rows, n))
    # Where the rounding of g log2 e, a step or more of it, all but cancels a factor of the exponential.
    worst = [-16770166.0, -23336016.0, -23386954.0, -68910152.0, -1175864200.0, -28420063232.0, -1024.0, -89.0, -88.03, -88.02, -87.34, -87.33, -3.3e38]
    far = rng.random((rows, n)) < 0.3
    far[:, 0] = False
    x[far] = -np.exp(rng.uniform(np.log(80.0), np.log(3.3e38), far.sum()))
    for row in range(rows):
        at = 1 + rng.choice(n - 1, len(worst), replace=False)
        x[row, at], far[row, at] = worst, True
    r[far] = rng.choice([-1, 1], far.sum()) * 2.0 ** 20
    if dtype == BF16:  # every bf16 gate there is below -80
        every = (np.arange(0xC2A0, 0xFF80, dtype=np.uint32) << 16).view(np.float32)
        x[far] = np.resize(rng.permutation(every), far.sum())
    x, r = gpu(x, dtype), gpu(r, dtype)
    check_rows("glu", x, r, None, *run_op(device, "glu", x, r, None, rows))


class Owned:
    """Buffers of a handle's own (`fq_buffer_alloc`) as tensors."""

    def __init__(self, d):
        self.d, self.held = d, []

    def __call__(self, *shape, dtype=F32):
        import ctypes as C
        size, p = int(np.prod(shape)) * dtype.itemsize, C.c_void_p()
        self.d.check(self.d._L.fq_buffer_alloc(self.d.handle, size, C.byref(p)))
        self.__cuda_array_interface__ = {"shape": (size,), "typestr": "|u1", "data": (p.value, False), "version": 3}
        self.held.append(p)
        return torch.as_tensor(self, device="cuda").view(dtype).view(shape).zero_()

    def free(self):
        torch.cuda.synchronize()
        for p in self.held:
            self.d.check(self.d._L.fq_buffer_free(self.d.handle, p))


@pytest.fixture
def own():
    """A handle of the test's own and its buffers."""
    d = S().Device(0)
    b = Owned(d)
    yield d, b
    b.free()
    d.close()


def fail(d):
    """What is enqueued turns out to have failed, and the handle is taken into use again."""
    d.fail_completion()
    with pytest.raises(S().SynchronizationError):
        d.synchronize()
    d.recover()


def calls_of_the_8_bit_path(d, rng, new):
    """name -> (call, its outputs, made by `new`), on inputs of their own."""
    s, m, n = S(), 3, 64
    x, r, w = gpu(rng.standard_normal((m, n))), gpu(rng.standard_normal((m, n))), gpu(1 + 0.1 * rng.standard_normal(n))
    mats = [matrix(rng, d, rows, n)[0] for rows in (40, 24)]
    xq, xs = gpu(rng.integers(-127, 128, (m, n)), torch.int8), gpu(rng.random(m))
    ids = torch.arange(m, dtype=torch.int32, device="cuda")
    i8, i32 = torch.int8, torch.int32
    out = {"quantize": (new(m, n, dtype=i8), new(m)), "rmsnorm": (new(m, n, dtype=i8), new(m)), "add": (new(m, n), new(m, n, dtype=i8), new(m)),
           "glu": (new(m, n, dtype=i8), new(m)), "project": (new(m, 40),), "many": (new(m, 40), new(m, 24)),
           "scores": (new(m), new(m, dtype=i32), new(m), new(m, 5), new(m, 5, dtype=i32))}
    calls = {"quantize": lambda q, sc: s.quantize_i8(d, x, m, q, sc), "rmsnorm": lambda q, sc: s.rmsnorm_i8(d, x, w, EPS, m, q, sc),
             "add": lambda h, q, sc: s.add_rmsnorm_i8(d, x, r, w, EPS, m, h, q, sc), "glu": lambda q, sc: s.glu_i8(d, x, r, m, q, sc),
             "project": lambda y: s.project_i8(d, mats[0], xq, xs, m, y), "many": lambda a, b: s.project_many_i8(d, mats, xq, xs, m, [a, b]),
             "scores": lambda lp, rk, en, tp, ti: s.token_logprobs(d, x, n, m, ids, lp, rk, en, 5, tp, ti)}
    torch.cuda.synchronize()
    return {name: (calls[name], out[name]) for name in calls}


def test_outputs_of_a_failed_submission_are_written_again(own):
    """They are refused as inputs until then, but not as what they are: outputs."""
    d, new = own
    rng = np.random.default_rng(20)
    for name, (call, out) in calls_of_the_8_bit_path(d, rng, new).items():
        call(*out)
        d.synchronize()
        first = [t.clone() for t in out]
        torch.cuda.synchronize()
        call(*out)
        fail(d)
        for t in out:
            t.fill_(9)
        torch.cuda.synchronize()
        call(*out)
        d.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, first)), name


def test_every_output_of_a_failed_submission_is_refused_as_an_input(own):
    d, new = own
    s, rng = S(), np.random.default_rng(21)
    y, ys = torch.zeros(1, 40, device="cuda"), torch.ones(1, device="cuda")
    q, sc = torch.zeros(1, 64, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")
    w = matrix(rng, d, 40, 64)[0]
    for name, (call, out) in calls_of_the_8_bit_path(d, rng, new).items():
        call(*out)
        fail(d)
        for t in out:
            with pytest.raises(s.SynchronizationError):
                if t.dtype == torch.int8:
                    s.project_i8(d, w, t[:1], ys, 1, y)
                elif t.dtype == torch.int32:
                    s.token_logprobs(d, torch.zeros(t.numel(), 8, device="cuda"), 8, t.numel(), t.view(-1), torch.zeros(t.numel(), device="cuda"), None, None)
                elif t.dim() == 1:
                    s.project_i8(d, w, q, t[:1], 1, y)
                else:
                    s.token_logprobs(d, t, t.shape[1], t.shape[0], None, None, None, torch.zeros(t.shape[0], device="cuda"))
        call(*out)
        d.synchronize()


def test_two_outputs_of_a_failed_submission_are_written_again(own):
    """The same of the calls on floats that have more than one output."""
    from oracle import ref
    d, new = own
    s = S()
    x, w = torch.ones(2, 256, device="cuda"), torch.ones(256, device="cuda")
    mat = s.Matrix.from_packed(d, 16, 256, 1, s.Q4_K, ref.random_matrix(s.Q4_K, 16, 256, 1))
    h, y, a, b, c = new(2, 256), new(2, 256), new(2, 16), new(2, 16), torch.zeros(2, 16, device="cuda")
    torch.cuda.synchronize()
    for call, out in ((lambda: s.add_rmsnorm(d, x, x, w, EPS, 2, h, y), (h, y)), (lambda: s.project_many(d, [mat, mat], x, 2, [a, b]), (a, b))):
        call()
        d.synchronize()
        first = [t.clone() for t in out]
        torch.cuda.synchronize()
        call()
        fail(d)
        for t in out:
            t.fill_(9)
        torch.cuda.synchronize()
        call()
        d.synchronize()
        assert all(torch.equal(t, f) for t, f in zip(out, first))
    s.project(d, mat, h, 2, c)  # written again, so an input again
    d.synchronize()


def test_a_refused_call_has_written_nothing(own):
    """What a failed submission wrote stays refused after a call into it that was itself refused."""
    d, new = own
    s, rng = S(), np.random.default_rng(22)
    x, w = gpu(rng.standard_normal((2, 64))), torch.ones(64, device="cuda")
    mat = matrix(rng, d, 64, 64)[0]
    q, sc, h, y, lp = new(2, 64, dtype=torch.int8), new(2), new(2, 64), new(2, 64), new(2)
    spare, ids = torch.zeros(2, 64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    s.add_rmsnorm_i8(d, x, x, w, EPS, 2, h, q, sc)
    s.project_i8(d, mat, q, sc, 2, y)
    s.token_logprobs(d, y, 64, 2, ids, lp, None, None)
    fail(d)
    part = x.view(-1)[:2]
    for call in (lambda: s.quantize_i8(d, x, 2, q, part), lambda: s.rmsnorm_i8(d, x, w, EPS, 2, q, w[:2]), lambda: s.glu_i8(d, x, x, 2, q, part),
                 lambda: s.add_rmsnorm_i8(d, x, x, w, EPS, 2, h, q, part), lambda: s.add_rmsnorm_i8(d, x, x, w, EPS, 2, h, q, h.view(-1)[:2]),
                 lambda: s.project_many_i8(d, [mat, mat], torch.zeros_like(q), torch.ones(2, device="cuda"), 2, [y, y]),
                 lambda: s.token_logprobs(d, spare, 64, 2, ids, lp, None, lp)):
        with pytest.raises(s.AliasError):
            call()
    d.synchronize()
    for call in (lambda: s.project_i8(d, mat, q, torch.ones(2, device="cuda"), 2, spare), lambda: s.project_i8(d, mat, torch.zeros_like(q), sc, 2, spare),
                 lambda: s.quantize_i8(d, h, 2, torch.zeros_like(q), torch.zeros(2, device="cuda")),
                 lambda: s.quantize_i8(d, y, 2, torch.zeros_like(q), torch.zeros(2, device="cuda")),
                 lambda: s.project_i8(d, mat, torch.zeros_like(q), lp, 2, spare)):
        with pytest.raises(s.SynchronizationError):
            call()


def test_no_matrix_is_made_of_what_a_failed_submission_wrote(own):
    d, new = own
    s, rng = S(), np.random.default_rng(23)
    x = gpu(rng.standard_normal((32, 64)))
    q, sc = new(32, 64, dtype=torch.int8), new(32)
    good = torch.ones(32, 64, dtype=torch.int8, device="cuda"), torch.ones(32, device="cuda")
    torch.cuda.synchronize()
    s.quantize_i8(d, x, 32, q, sc)
    d.fail_completion()
    with pytest.raises(s.SynchronizationError):  # the submission that makes the integers: this call waits for it
        s.Matrix.from_i8(d, q, sc)
    d.recover()
    for values, scales in ((q, good[1]), (good[0], sc), (q, sc.cpu())):
        with pytest.raises(s.SynchronizationError):
            s.Matrix.from_i8(d, values, scales)
    s.Matrix.from_i8(d, *good)
    s.quantize_i8(d, x, 32, q, sc)
    w = s.Matrix.from_i8(d, q, sc)
    xq, xs = rng.integers(-127, 128, (3, 64), dtype=np.int8), np.ones(3, np.float32)
    assert same(project(d, [w], xq, xs, F32, False)[0], expect(xq, xs, q.cpu().numpy(), sc.cpu().numpy()))


def test_no_matrix_is_made_of_memory_past_an_allocation(own):
    d, new = own
    import ctypes as C
    s = S()
    q, sc = new(32, 64, dtype=torch.int8), new(32)
    torch.cuda.synchronize()
    for values, scales in ((q.data_ptr() + 16, sc.data_ptr()), (q.data_ptr(), sc.data_ptr() + 4)):
        out = C.c_void_p()
        with pytest.raises(s.RangeError):
            d.check(d._L.fq_matrix_create_i8(d.handle, 32, 64, values, scales, C.byref(out)))
        assert not out.value


def test_sizes_whose_bytes_pass_64_bits(own):
    """They are refused as shapes, not cut to what a buffer holds."""
    from ferrum_b200 import _lib
    d, new = own
    s = S()
    x, q, sc, ids = new(8, 64), new(8, 64, dtype=torch.int8), new(8), new(8, dtype=torch.int32)
    torch.cuda.synchronize()
    lib, h, before = d._L, d.handle, d.counters().dispatches
    n, rows = 2 ** 32 - 4, 2 ** 31 - 1
    for rc in (lib.fq_token_logprobs(h, x.data_ptr(), _lib.F32, 4, 2 ** 62, 5, ids.data_ptr(), 0, sc.data_ptr(), None, None, None, None),
               lib.fq_token_logprobs(h, x.data_ptr(), _lib.BF16, 4, 2 ** 63, 3, ids.data_ptr(), 0, sc.data_ptr(), None, None, None, None),
               lib.fq_token_logprobs(h, x.data_ptr(), _lib.F32, 4, 2 ** 64 - 4, 2, ids.data_ptr(), 0, sc.data_ptr(), None, None, None, None),
               lib.fq_quantize_i8(h, x.data_ptr(), _lib.F32, n, rows, q.data_ptr(), sc.data_ptr()),
               lib.fq_rmsnorm_i8(h, x.data_ptr(), _lib.BF16, x.data_ptr(), n, EPS, rows, q.data_ptr(), sc.data_ptr())):
        with pytest.raises(s.ShapeError):
            d.check(rc)
    with pytest.raises(s.RangeError):  # rows that a buffer does not hold
        d.check(lib.fq_token_logprobs(h, x.data_ptr(), _lib.F32, 4, 128, 5, ids.data_ptr(), 0, sc.data_ptr(), None, None, None, None))
    assert d.counters().dispatches == before
    s.token_logprobs(d, x.view(-1), 4, 1, ids[:1], sc[:1], None, None, stride=2 ** 62)  # one row has no next one
    d.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [3, 150])
@pytest.mark.parametrize("n", [18944, 18952, 28672, 51200, 51208, 65536])
@pytest.mark.parametrize("op", OPS)
def test_rows_around_the_ends_of_shared_memory(device, op, n, rows, dtype):
    """The longest rows that bulk copies bring in (18944) and that are kept (51200), the next ones, and widths between."""
    rng = np.random.default_rng(n + rows)
    x = gpu(rng.standard_normal((rows, n)) * (1 + 30 * (rng.random(n) < 0.01)), dtype)
    r, w = gpu(rng.standard_normal((rows, n)), dtype), gpu(1 + 0.1 * rng.standard_normal(n))
    h = torch.zeros_like(x)
    q, s = run_op(device, op, x, r, w, rows, h)
    check_rows(op, x, r, w, q, s)
    if op == "add":
        assert torch.equal(h.cpu(), values_of(op, x, r, w)[2])
        for first, second, place in ((x.clone(), r, 0), (x, r.clone(), 1)):  # the sum in place of either input
            place = (first, second)[place]
            assert np.array_equal(run_op(device, op, first, second, w, rows, place)[0], q) and torch.equal(place, h)
