"""Embedding lookup with scaling and its gradient by sorted tokens against the definitions in 64 bits (oracle/e4m3_oracle.py).  Whole
numbers make the sums exact; otherwise a sum of n fp32 additions is off by at most n * 2^-24 * sum |entry|, the scaling by half a
step more, the rounding to a type by half a step of that."""
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


def _tokens(g, N, V, spread):
    if spread == "even":
        return torch.randint(0, V, (N,), generator=g)
    if spread == "one":
        return torch.full((N,), V - 1, dtype=torch.int64)
    if spread == "outside":  # some negative, some past the end
        return torch.randint(-V, 2 * V, (N,), generator=g)
    u = torch.rand(N, generator=g, dtype=torch.float64)
    return (torch.exp(u * np.log(V + 1.0)) - 1).long().clamp(0, V - 1)


# one token; one row; fewer tokens than a chunk; runs over many chunks; the border between the two sorts and both sides of it;
# more than one radix pass; odd and one-column rows; more slabs than one
CASES = [(1, 1, 1, "even"), (1, 64000, 768, "even"), (37, 24, 100, "zipf"), (31, 7, 3, "outside"), (2000, 24, 100, "zipf"),
         (4000, 3, 130, "one"), (5000, 5000, 33, "even"), (8192, 300, 17, "zipf"), (8193, 300, 17, "zipf"), (16385, 300, 17, "zipf"), (300001, 40, 9, "zipf"), (20000, 70000, 8, "zipf"),
         (40000, 24, 100, "zipf"), (33000, 200, 257, "one"), (17000, 1000, 1100, "outside"), (90001, 65536, 5, "even")]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,V,E,spread", CASES)
def test_whole_numbers(dev, dtype, N, V, E, spread):
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(N + V + E)
    tokens = _tokens(g, N, V, spread)
    table = torch.randint(-100, 101, (V, E), generator=g).to(dtype)
    d_out = torch.randint(-7, 8, (N, E), generator=g).to(dtype)
    for kind in (torch.int64, torch.int32):
        t = tokens.to(kind).to(dev)
        out = ops.embedding_rows(table.to(dev), t, 2.0)
        assert np.array_equal(_np(out), O.embedding(_np(table), tokens.numpy(), 2.0)) and out.dtype == dtype
        want = torch.from_numpy(O.embedding_grad(_np(d_out), tokens.numpy(), V, 0.5)).float()
        grad = ops.embedding_rows_grad(d_out.to(dev), t, V, 0.5, torch.float32)
        assert torch.equal(grad.cpu(), want)
        grad = ops.embedding_rows_grad(d_out.to(dev), t, V, 0.5)
        assert grad.dtype == dtype and torch.equal(grad.cpu(), want.to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,V,E,spread", [(37, 24, 100, "zipf"), (6000, 24, 100, "zipf"), (20000, 3000, 40, "zipf")])
def test_values_and_order(dev, dtype, N, V, E, spread):
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(N + V + E + 1)
    tokens = _tokens(g, N, V, spread)
    table, d_out = torch.randn(V, E, generator=g).to(dtype), torch.randn(N, E, generator=g).to(dtype)
    scale = float(np.float32(E ** 0.5))
    f = torch.finfo(dtype)
    out = _np(ops.embedding_rows(table.to(dev), tokens.to(dev), scale))
    want = O.embedding(_np(table), tokens.numpy(), scale)
    assert (np.abs(out - want) <= (2.0 ** -24 + f.eps / 2) * 1.001 * np.abs(want) + f.smallest_normal * f.eps).all()
    first = ops.embedding_rows_grad(d_out.to(dev), tokens.to(dev), V, scale)
    want = O.embedding_grad(_np(d_out), tokens.numpy(), V, scale)
    mag = O.embedding_grad(np.abs(_np(d_out)), tokens.numpy(), V, scale)
    n = np.bincount(tokens.numpy(), minlength=V)[:, None]
    tol = (n + 1) * 2.0 ** -24 * mag
    tol += f.eps / 2 * (np.abs(want) + tol) + f.smallest_normal * f.eps
    assert (np.abs(_np(first) - want) <= tol).all()
    for _ in range(3):
        assert torch.equal(ops.embedding_rows_grad(d_out.to(dev), tokens.to(dev), V, scale), first)


def test_bad_values_stay_in_their_rows(dev):
    from phonlp_amd import ops
    tokens = torch.arange(60, device=dev) % 6
    d_out = torch.ones(60, 20, device=dev)
    d_out[13, 4], d_out[14, 0] = float("nan"), float("inf")
    grad = ops.embedding_rows_grad(d_out, tokens, 8).cpu()
    want = torch.full((8, 20), 10.0)
    want[6:] = 0
    want[1, 4], want[2, 0] = float("nan"), float("inf")
    assert torch.equal(torch.nan_to_num(grad, nan=-1.0), torch.nan_to_num(want, nan=-1.0))


def test_shapes_strides_empty(dev):
    from phonlp_amd import ops
    base = torch.randn(50, 400, device=dev)
    tokens = torch.randint(0, 50, (3, 7), device=dev)
    for view in (base[:, 3:103], base[::2, :101], base[:, 399:]):
        assert torch.equal(ops.embedding_rows(view, tokens % view.shape[0]), view[tokens % view.shape[0]])
    d = torch.randn(21, 300, device=dev)
    a = ops.embedding_rows_grad(d[:, 5:205], tokens.view(-1), 50)
    assert torch.equal(a, ops.embedding_rows_grad(d[:, 5:205].contiguous().view(3, 7, 200), tokens, 50))
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    assert tuple(ops.embedding_rows(base, none).shape) == (0, 400)
    assert not ops.embedding_rows_grad(torch.zeros(0, 9, device=dev), none, 5).any()


def test_rows_behind_the_table_stay(dev):
    """Neither direction writes outside its output."""
    from phonlp_amd import _lib, ops
    N, V, E = 33, 70, 37
    tokens = torch.randint(0, V, (N,), device=dev)
    d = torch.randn(N, E, device=dev)
    buf = torch.full((V * E + 64,), 5.0, device=dev)
    nb = _lib.lib().phonlp_embedding_rows_grad_ws_bytes(N, E)
    ws = torch.full((nb + 256,), 77, dtype=torch.uint8, device=dev)
    ops._run(dev, "phonlp_embedding_rows_grad", d.data_ptr(), 0, E, tokens.data_ptr(), 1, N, V, E, 1.0, buf.data_ptr(), 0,
             ws.data_ptr(), nb)
    assert torch.equal(buf[:V * E].view(V, E), ops.embedding_rows_grad(d, tokens, V)) and (buf[V * E:] == 5).all() and (ws[nb:] == 77).all()


def test_graph(dev):
    """A captured lookup and gradient (both sorts) replays on new tokens, beside eager calls."""
    from phonlp_amd import ops
    for N, V, E in ((900, 50, 64), (17000, 900, 16)):
        sets = [(torch.randint(-3, V + 3, (N,), device=dev), torch.randn(N, E, device=dev)) for _ in range(3)]
        table = torch.randn(V, E, device=dev)
        step = lambda t, d: (ops.embedding_rows(table, t, 3.0), ops.embedding_rows_grad(d, t, V, 3.0))  # noqa: E731
        want = [[o.clone() for o in step(*s)] for s in sets]
        t, d = torch.zeros_like(sets[0][0]), torch.zeros_like(sets[0][1])
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = step(t, d)
        for i in (0, 1, 2, 0):
            t.copy_(sets[i][0])
            d.copy_(sets[i][1])
            graph.replay()
            eager = step(*sets[(i + 1) % 3])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
            assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3]))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [31, 32, 33, 4095, 4097, 8191])
@pytest.mark.parametrize("E", [7, 13, 520])
def test_rows_of_a_wider_tensor(dev, dtype, N, E):
    """Rows inside a wider tensor of NaN: row ends of every kind (less than one vector; a last vector that overlaps its neighbour; over
    two slabs), counts on both sides of the sorts' steps.  Whole numbers: exact."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(N + E)
    V = 50
    tokens = _tokens(g, N, V, "outside")
    wide = torch.full((max(N, V), E + 11), float("nan"), dtype=dtype, device=dev)
    table, d_out = torch.randint(-100, 101, (V, E), generator=g).to(dtype), torch.randint(-3, 4, (N, E), generator=g).to(dtype)
    part = wide[:V, 5:5 + E]
    part.copy_(table)
    out = ops.embedding_rows(part, tokens.to(dev), 1.0)
    assert np.array_equal(_np(out), O.embedding(_np(table), tokens.numpy(), 1.0))
    part = wide[:N, 5:5 + E]
    part.copy_(d_out)
    grad = ops.embedding_rows_grad(part, tokens.to(dev), V, 1.0, torch.float32)
    assert torch.equal(grad.cpu(), torch.from_numpy(O.embedding_grad(_np(d_out), tokens.numpy(), V, 1.0)).float())


def test_counts_past_the_abis_ints_are_refused(dev):
    """Numbers of rows, tokens and table rows that a C int does not hold are refused before anything is allocated for them."""
    from phonlp_amd import ops
    tall = torch.empty(2 ** 31, 1, dtype=torch.float16, device=dev)
    with pytest.raises(ValueError, match="more than"):
        ops.e4m3_rows(tall)
    with pytest.raises(ValueError, match="more than"):
        ops.embedding_rows(tall, torch.zeros(1, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError, match="V must lie"):
        ops.embedding_rows_grad(torch.ones(1, 4, device=dev), torch.zeros(1, dtype=torch.int64, device=dev), 2 ** 32 + 3)


def test_tables_past_32_bit_offsets(dev):
    """A table of more than 2^31 entries: its last rows are found, their gradients land there, every other row is zero."""
    from phonlp_amd import ops
    V, E = 2_900_000, 768
    assert V * E > 2 ** 31
    tokens = torch.tensor([V - 1, 5, V - 2, V - 1, V, V // 2], device=dev)
    table = torch.zeros(V, E, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(1)
    rows = torch.randint(-9, 10, (6, E), generator=g).to(dev, torch.bfloat16)
    table[tokens[[0, 1, 2, 5]]] = rows[:4]
    out = ops.embedding_rows(table, tokens, 2.0)
    assert torch.equal(out[[0, 1, 2, 5]], 2 * rows[:4]) and torch.equal(out[3], out[0]) and not out[4].any()
    del table
    d = ops.embedding_rows_grad(rows, tokens, V)
    assert torch.equal(d[V - 1], rows[0] + rows[3]) and torch.equal(d[5], rows[1]) and torch.equal(d[V - 2], rows[2])
    assert torch.equal(d[V // 2], rows[5])
    d[tokens[[0, 1, 2, 5]]] = 0
    assert not d.any()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [2, 5, 63, 64, 65, 127, 129, 255, 511, 512, 513])
@pytest.mark.parametrize("V,E,spread", [(3, 5, "zipf"), (4097, 12, "outside"), (9000, 300, "even"), (70001, 2, "one"), (140000, 9, "outside")])
def test_few_tokens(dev, dtype, N, V, E, spread):
    """Both sides of the border between looking for a row's tokens and sorting them; one to 64 rows of the table a workgroup; tokens of one
    wave and of several, more of a row than are loaded at a time.  Whole numbers: exact, and the same twice."""
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(N + V)
    tokens = _tokens(g, N, V, spread)
    d_out = torch.randint(-7, 8, (N, E), generator=g).to(dtype)
    want = torch.from_numpy(O.embedding_grad(_np(d_out), tokens.numpy(), V, 0.5)).float()
    for kind in (torch.int64, torch.int32):
        t = tokens.to(kind).to(dev)
        grad = ops.embedding_rows_grad(d_out.to(dev), t, V, 0.5, torch.float32)
        assert torch.equal(grad.cpu(), want)
        assert torch.equal(ops.embedding_rows_grad(d_out.to(dev), t, V, 0.5).cpu(), want.to(dtype))
