"""The 8-bit dense layer on the GPU: images, the product on them, the backward from the checkpoint, against the definitions in 64 bits
(oracle/e4m3_oracle.py).  Whole-number operands make every sum exact in fp32, so those results have to be equal; for the others
the tolerances are: a sum of n exact products, each addition off by at most 2^-23 of its result in whatever order (the matrix
instruction may truncate: one full step of fp32), is off by at most n * 2^-23 * sum |product|; the rounding to a type adds half a
step of the result.  A 16-bit result of linear_e4m3 comes from the 8-bit matrix pipe, which adds eight products cut off 13 bits below
the largest of the eight: the seven others lose at most 2^-13 of it each, so 7 * 2^-13 * sum |product| bounds what all of them lose."""
import numpy as np
import pytest
import torch

from oracle import e4m3_oracle as O

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _np(t):
    return t.detach().double().cpu().numpy()


def _codes(t):
    return t.view(torch.uint8).cpu().numpy()


def _check_image(got, x):
    want_c, want_e = O.image(_np(x))
    c, e = _codes(got[0]), got[1].cpu().numpy()
    assert c.shape == want_c.shape and e.shape == want_e.shape
    assert np.array_equal(e, want_e)
    nan = (want_c & 0x7F) == 0x7F
    assert np.array_equal(c[~nan], want_c[~nan]) and ((c[nan] & 0x7F) == 0x7F).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 127), (5, 128), (2, 129), (64, 768), (33, 868), (7, 1030), (1025, 70)])
def test_rows_and_values(dev, dtype, M, K):
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(M * 1000 + K)
    x = torch.randn(M, K, generator=g) * torch.exp(4 * torch.randn(M, 1, generator=g)) * torch.exp(2 * torch.randn(1, K, generator=g))
    x = x.to(dtype)
    got = ops.e4m3_rows(x.to(dev))
    _check_image(got, x)
    exact = O.values(*O.image(_np(x)), K)
    for t in TYPES:
        top = torch.finfo(t).max
        back = ops.e4m3_values(*got, K, t).cpu()
        want = torch.from_numpy(np.clip(exact, -top, top)).to(t)  # NaN where x overflowed its own type
        assert back.dtype == t and np.array_equal(back.double().numpy(), want.double().numpy(), equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_rows_at_the_edges(dev, dtype):
    """Empty blocks, the type's largest and smallest, infinities and NaN beside finite entries, ties, -0, blocks at 448 * 2^e."""
    from phonlp_amd import ops
    f = torch.finfo(dtype)
    inf, nan = float("inf"), float("nan")
    rows = [[0.0] * 200, [f.max, -f.max, 1.0] + [0.0] * 197, [f.tiny, -f.tiny / 2] * 100, [f.smallest_normal] + [0.0] * 199,
            [inf, 1.0, -inf, 2.0] * 50, [nan, -1.5] * 100, [inf] * 200, [nan] * 200, [-0.0] * 200, [448.0, 449.0, 447.0, 1.0] * 50,
            [448.0, 224.0, 0.001, 17.0] * 50, [17.0, 19.0, 18.0, 16.0] * 50, [1.0 + i / 64 for i in range(200)],
            [float(2 ** -(i % 20)) for i in range(200)], [240.0 * f.smallest_normal] * 200]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    got = ops.e4m3_rows(x.to(dev))
    _check_image(got, x)
    back = ops.e4m3_values(*got, 200, dtype).cpu()
    finite = torch.isfinite(x)
    assert torch.isfinite(back[finite]).all() and torch.isnan(back[~finite]).all()


def test_rows_strides(dev):
    """Rows that start at any element of a larger buffer, with a pitch of their own."""
    from phonlp_amd import ops
    for dtype in TYPES:
        base = torch.randn(40, 1001, device=dev).to(dtype)
        for view in (base[:, 3:400], base[1:, 1:130], base[::3, :257], base[:, 5:6], base[7:8, 2:900]):
            a, b = ops.e4m3_rows(view), ops.e4m3_rows(view.contiguous())
            assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def _whole(g, rows, K, most):
    """Whole numbers up to `most` <= 15: every e4m3 image holds them exactly."""
    return torch.randint(-most, most + 1, (rows, K), generator=g).float()


# one token, sub-tile, tile borders, odd sizes, more tiles than compute units, a long row
SHAPES = [(1, 1, 1), (1, 400, 768), (2, 33, 130), (31, 24, 868), (17, 13464, 408), (64, 128, 128), (129, 257, 512), (300, 401, 868),
          (1, 7, 16384), (2011, 1000, 408), (5000, 130, 200), (257, 4100, 640)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_whole_numbers(dev, M, N, K):
    """Every product and sum is a whole number under 2^24: the result is exact; the bits are exactly y > 0."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(M + 7 * N + K)
    x, w = _whole(g, M, K, 7), _whole(g, N, K, 7)
    bias = torch.randint(-9, 10, (N,), generator=g).float()
    xi, wi = ops.e4m3_rows(x.to(dev)), ops.e4m3_rows(w.to(dev))
    want = O.linear(_np(x), _np(w), _np(bias), False)
    y, bits = ops.linear_e4m3(*xi, *wi, bias.to(dev), K, True, torch.float32, want_bits=True)
    assert np.array_equal(_np(y), np.maximum(want, 0))
    assert np.array_equal(bits.cpu().numpy(), O.pack_bits(want > 0))
    y, none = ops.linear_e4m3(*xi, *wi, None, K, False)
    assert none is None and np.array_equal(_np(y), want - _np(bias))
    for t in (torch.bfloat16, torch.float16):
        y, _ = ops.linear_e4m3(*xi, *wi, bias.to(dev), K, False, t)
        assert torch.equal(y.cpu(), torch.from_numpy(want).float().to(t))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(1, 400, 768), (37, 131, 868), (600, 384, 1000), (3000, 260, 408)])
def test_linear_values(dev, dtype, M, N, K):
    """Rows and blocks of very different loudness."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(M + N + K)
    x = (torch.randn(M, K, generator=g) * torch.exp(3 * torch.randn(M, 1, generator=g))).to(dtype)
    w = torch.randn(N, K, generator=g) * torch.exp(2 * torch.randn(N, 1, generator=g)) * torch.exp(2 * torch.randn(1, K, generator=g))
    bias = torch.randn(N, generator=g)
    xi, wi = ops.e4m3_rows(x.to(dev)), ops.e4m3_rows(w.to(dev))
    xv, wv = O.values(*O.image(_np(x)), K), O.values(*O.image(_np(w)), K)
    y, _ = ops.linear_e4m3(*xi, *wi, bias.to(dev), K, False, dtype)
    want = O.linear(xv, wv, _np(bias), False)
    # K products and the bias; then the rounding to the type (half a step, and of its smallest step), or past its largest
    mag = np.abs(xv) @ np.abs(wv).T
    tol = (K + 1) * 2.0 ** -23 * (mag + np.abs(_np(bias)))
    if dtype != torch.float32:
        tol += 7 * 2.0 ** -13 * mag
    f = torch.finfo(dtype)
    tol += f.eps / 2 * (np.abs(want) + tol) + f.smallest_normal * f.eps / 2
    got = _np(y)
    nan = np.isnan(want)  # rows of x that passed their own type's largest
    assert np.array_equal(np.isnan(got), nan)
    over = np.isinf(got)
    got, tol, want = got[~nan], tol[~nan], want[~nan]
    over = over[~nan]
    assert (np.abs(want[over]) + tol[over] >= f.max).all() and (np.abs(got - want)[~over] <= tol[~over]).all()


def test_linear_bad_values_stay_in_their_rows(dev):
    """NaN or an infinity in one row of x reaches that row of y alone, in w that column; ReLU keeps NaN and clears its bit."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(5)
    x, w = _whole(g, 70, 300, 7), _whole(g, 90, 300, 7)
    want = O.linear(_np(x), _np(w), None, True)
    x[3, 299], x[40, 0], w[88, 128] = float("nan"), float("inf"), float("-inf")
    y, bits = ops.linear_e4m3(*ops.e4m3_rows(x.to(dev)), *ops.e4m3_rows(w.to(dev)), None, 300, True, want_bits=True)
    y = _np(y)
    bad = np.zeros_like(want, bool)
    bad[[3, 40]] = True
    bad[:, 88] = True
    assert np.isnan(y[bad]).all() and np.array_equal(y[~bad], want[~bad])
    assert np.array_equal(bits.cpu().numpy(), O.pack_bits((want > 0) & ~bad))


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 400, 768), (31, 24, 100), (63, 65, 129), (64, 64, 128), (130, 200, 300), (513, 33, 868),
                                   (2000, 401, 70), (3001, 64, 64), (40, 2448, 868), (257, 1030, 520), (9000, 130, 260), (128, 256, 300), (1920, 384, 129)])
def test_backward_whole_numbers(dev, dtype, relu, M, N, K):
    """dZ up to 7, values up to 7: sums of up to 9000 products under 2^24, exact; dX is then rounded to dY's type."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(M + 3 * N + 5 * K)
    x, w, dy = _whole(g, M, K, 7), _whole(g, N, K, 7), _whole(g, M, N, 7).to(dtype)
    mask = (torch.rand(M, N, generator=g) < 0.6).numpy() if relu else None
    bits = torch.from_numpy(O.pack_bits(mask)).to(dev) if relu else None
    xi, wi = ops.e4m3_rows(x.to(dev)), ops.e4m3_rows(w.to(dev))
    dX, dW, db = ops.linear_e4m3_backward(dy.to(dev), bits, *xi, *wi, K)
    wx, ww, wb = O.backward(_np(dy), mask, _np(x), _np(w))
    assert dX.dtype == dtype and dW.dtype == db.dtype == torch.float32
    assert torch.equal(dX.cpu(), torch.from_numpy(wx).float().to(dtype))
    assert np.array_equal(_np(dW), ww) and np.array_equal(_np(db), wb)
    # each alone, and dY as a view into wider rows
    wide = torch.zeros(M, N + 3, dtype=dtype, device=dev)
    wide[:, 1:N + 1] = dy.to(dev)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        part = ops.linear_e4m3_backward(wide[:, 1:N + 1], bits, *xi, *wi, K, *need)
        for got, full, on in zip(part, (dX, dW, db), need):
            assert got is None if not on else torch.equal(got, full)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(37, 131, 868), (700, 260, 300)])
def test_backward_values(dev, dtype, M, N, K):
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    w = torch.randn(N, K, generator=g) * torch.exp(2 * torch.randn(N, 1, generator=g))
    dy = (torch.randn(M, N, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)
    mask = (torch.rand(M, N, generator=g) < 0.5).numpy()
    xv, wv = O.values(*O.image(_np(x)), K), O.values(*O.image(_np(w)), K)
    got = ops.linear_e4m3_backward(dy.to(dev), torch.from_numpy(O.pack_bits(mask)).to(dev), *ops.e4m3_rows(x.to(dev)),
                                   *ops.e4m3_rows(w.to(dev)), K)
    want = O.backward(_np(dy), mask, xv, wv)
    dz = np.abs(_np(dy)) * mask
    # three exact pieces of dZ: 3 N (3 M) products a sum; db: M entries
    mags = (3 * N * (dz @ np.abs(wv)), 3 * M * (dz.T @ np.abs(xv)), M * dz.sum(0))
    f = torch.finfo(dtype)
    for name, a, b, mag in zip(("dX", "dW", "db"), got, want, mags):
        tol = 2.0 ** -23 * mag
        if name == "dX":
            tol += f.eps / 2 * (np.abs(b) + tol) + f.smallest_normal * f.eps / 2
        a = _np(a)
        over = ~np.isfinite(a)
        assert (np.abs(b[over]) + tol[over] >= f.max).all(), name
        assert (np.abs(a - b)[~over] <= tol[~over]).all(), name


def test_backward_bad_values(dev):
    """fp32 gradients at the ends of the range; infinities and NaN reach their row of dX, their column of dW and db."""
    from phonlp_amd import ops
    one = torch.ones(66, 130)
    w = torch.ones(40, 130)
    dy = torch.zeros(66, 40)
    dy[0, 0], dy[1, 1], dy[2, 2] = 3.4e38, 1e-30, -3.3999999e38
    xi, wi = ops.e4m3_rows(one.to(dev)), ops.e4m3_rows(w.to(dev))
    dX, dW, db = ops.linear_e4m3_backward(dy.to(dev), None, *xi, *wi, 130)
    assert torch.equal(dX.cpu(), dy.sum(1, keepdim=True).expand(66, 130)) and torch.equal(db.cpu(), dy.sum(0))
    assert torch.equal(dW.cpu(), dy.sum(0)[:, None].expand(40, 130))
    dy = torch.ones(66, 40)
    dy[5, 7], dy[9, 3] = float("inf"), float("nan")
    dX, dW, db = (t.cpu() for t in ops.linear_e4m3_backward(dy.to(dev), None, *xi, *wi, 130))
    rows, cols = torch.arange(66), torch.arange(40)
    assert torch.equal(dX[(rows != 5) & (rows != 9)], torch.full((64, 130), 40.0))
    assert not torch.isfinite(dX[[5, 9]]).any() and not torch.isfinite(dW[[7, 3]]).any() and not torch.isfinite(db[[7, 3]]).any()
    assert torch.equal(dW[(cols != 7) & (cols != 3)], torch.full((38, 130), 66.0))
    # masked by the bits they reach nothing
    mask = torch.isfinite(dy).numpy()
    got = ops.linear_e4m3_backward(dy.to(dev), torch.from_numpy(O.pack_bits(mask)).to(dev), *xi, *wi, 130)
    assert all(torch.isfinite(t).all() for t in got)


def test_empty(dev):
    from phonlp_amd import ops
    x, w = torch.zeros(0, 200, device=dev), torch.ones(3, 200, device=dev)
    xi, wi = ops.e4m3_rows(x), ops.e4m3_rows(w)
    assert tuple(xi[0].shape) == (0, 256) and tuple(ops.e4m3_values(*xi, 200).shape) == (0, 200)
    assert tuple(ops.linear_e4m3(*xi, *wi, None, 200, True, want_bits=True)[0].shape) == (0, 3)
    dX, dW, db = ops.linear_e4m3_backward(torch.zeros(0, 3, device=dev), None, *xi, *wi, 200)
    assert tuple(dX.shape) == (0, 200) and not dW.any() and not db.any() and tuple(dW.shape) == (3, 200)


def test_gradients_against_differences(dev):
    """db and dX against central differences of the layer itself: with whole numbers and steps of 1 the layer is linear and exact,
    so the difference quotient of sum(dY * Y) is the gradient."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(2)
    M, N, K = 5, 6, 140
    x, w, dy = _whole(g, M, K, 3), _whole(g, N, K, 3), _whole(g, M, N, 3)
    wi = ops.e4m3_rows(w.to(dev))

    def loss(x_, w_, b_):
        y, _ = ops.linear_e4m3(*ops.e4m3_rows(x_.to(dev)), *ops.e4m3_rows(w_.to(dev)), b_.to(dev), K, False)
        return float((y.cpu().double() * dy.double()).sum())

    dX, dW, db = ops.linear_e4m3_backward(dy.to(dev), None, *ops.e4m3_rows(x.to(dev)), *wi, K)
    zero = torch.zeros(N)
    for i, k in ((0, 0), (4, 139), (2, 128)):
        e = torch.zeros(M, K)
        e[i, k] = 1
        assert (loss(x + e, w, zero) - loss(x - e, w, zero)) / 2 == float(dX[i, k])
    for n, k in ((0, 0), (5, 139), (3, 127)):
        e = torch.zeros(N, K)
        e[n, k] = 1
        assert (loss(x, w + e, zero) - loss(x, w - e, zero)) / 2 == float(dW[n, k])
    for n in range(N):
        e = torch.zeros(N)
        e[n] = 1
        assert (loss(x, w, e) - loss(x, w, -e)) / 2 == float(db[n])


def test_graph_and_streams(dev):
    """A captured forward and backward replays to the eager results after its inputs changed, beside eager calls; two graphs captured
    from the same code have workspaces of their own; a side stream gives the same bits."""
    from phonlp_amd import ops
    M, N, K = 200, 300, 260
    g = torch.Generator().manual_seed(9)
    xs = [torch.randn(M, K, generator=g).to(dev) for _ in range(3)]
    dys = [torch.randn(M, N, generator=g).to(dev) for _ in range(3)]
    w = torch.randn(N, K, generator=g).to(dev)

    def step(x, dy):
        xi, wi = ops.e4m3_rows(x), ops.e4m3_rows(w)
        y, bits = ops.linear_e4m3(*xi, *wi, None, K, True, want_bits=True)
        return (y, *ops.linear_e4m3_backward(dy, bits, *xi, *wi, K))

    want = [[t.clone() for t in step(x, dy)] for x, dy in zip(xs, dys)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xs[0], dys[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs = []
    for _ in range(2):
        x, dy = torch.zeros_like(xs[0]), torch.zeros_like(dys[0])
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = step(x, dy)
        graphs.append((graph, x, dy, out))
    for i in (0, 1, 2, 1):
        for k, (graph, x, dy, _) in enumerate(graphs):
            x.copy_(xs[(i + k) % 3])
            dy.copy_(dys[(i + k) % 3])
            graph.replay()
        eager = step(xs[i], dys[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[i]))
        for k, (_, _, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(i + k) % 3]))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(4096, 4096, 128), (8190, 4090, 130), (4090, 4090, 300), (8190, 4090, 2100), (7680, 4352, 1100)])
def test_linear_large_products(dev, dtype, M, N, K):
    """Products large enough for the large tile (one to seventeen blocks; one and two tiles of a workgroup, whole ones and edges): whole
    numbers, so the sums are exact and the results their roundings."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(K)
    x, w, bias = (_whole(g, *s, 7).to(dev) for s in ((M, K), (N, K), (1, N)))
    bias = bias[0].contiguous()
    xi, wi = ops.e4m3_rows(x), ops.e4m3_rows(w)
    want = (x.double() @ w.double().t() + bias.double()).relu()
    y, bits = ops.linear_e4m3(*xi, *wi, bias, K, True, dtype, True)
    assert torch.equal(y, want.to(dtype))
    for rows in (slice(0, 300), slice(M - 300, M)):
        assert np.array_equal(bits[rows].cpu().numpy(), O.pack_bits((want[rows] > 0).cpu().numpy()))
    y, _ = ops.linear_e4m3(*xi, *wi, None, K, False, dtype)
    assert torch.equal(y, (x.double() @ w.double().t()).to(dtype))


def test_products_past_32_bit_offsets(dev):
    """More than 2^31 outputs: the last rows of Y, its bits and dX, and dW and db over all of them (entries of -1, 0 and 1: every sum is
    exact)."""
    from phonlp_amd import ops
    M, N, K = 1_060_003, 2100, 131
    assert M * N > 2 ** 31
    g = torch.Generator(device=dev).manual_seed(3)
    draw = lambda *s: torch.randint(-1, 2, s, generator=g, device=dev, dtype=torch.int8)
    x, w, dy = draw(M, K).float(), draw(N, K).float(), draw(M, N).bfloat16()
    xi, wi = ops.e4m3_rows(x), ops.e4m3_rows(w)
    y, bits = ops.linear_e4m3(*xi, *wi, None, K, True, torch.bfloat16, True)
    for rows in (slice(0, 100), slice(M // 2, M // 2 + 100), slice(M - 100, M)):
        want = (x[rows] @ w.t()).relu()
        assert torch.equal(y[rows], want.bfloat16())
        assert np.array_equal(bits[rows].cpu().numpy(), O.pack_bits((want > 0).cpu().numpy()))
    dX, dW, db = ops.linear_e4m3_backward(dy, bits, *xi, *wi, K)
    want_dW, want_db = torch.zeros(N, K, dtype=torch.float64, device=dev), torch.zeros(N, dtype=torch.float64, device=dev)
    for r in range(0, M, 100000):
        dz = (dy[r:r + 100000] * (y[r:r + 100000] > 0)).double()
        want_dW += dz.t().contiguous() @ x[r:r + 100000].double()
        want_db += dz.sum(0)
        assert torch.equal(dX[r:r + 100000], (dz.float() @ w).bfloat16())
    assert torch.equal(dW.double(), want_dW) and torch.equal(db.double(), want_db)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M", [1, 15, 16, 17])
@pytest.mark.parametrize("N,K", [(20480, 700), (20481, 130), (30001, 1030), (1000, 128), (33, 3000)])
def test_linear_few_rows(dev, dtype, M, N, K):
    """One to seventeen rows: both groupings of the few-row form, one block to many, odd widths; whole numbers, exact."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(N + M)
    x, w, bias = (_whole(g, *s, 7).to(dev) for s in ((M, K), (N, K), (1, N)))
    bias = bias[0].contiguous()
    xi, wi = ops.e4m3_rows(x), ops.e4m3_rows(w)
    want = (x.double() @ w.double().t() + bias.double()).relu()
    y, bits = ops.linear_e4m3(*xi, *wi, bias, K, True, dtype, True)
    assert torch.equal(y, want.to(dtype))
    assert np.array_equal(bits.cpu().numpy(), O.pack_bits((want > 0).cpu().numpy()))
    y, _ = ops.linear_e4m3(*xi, *wi, None, K, False, dtype)
    assert torch.equal(y, (x.double() @ w.double().t()).to(dtype))
