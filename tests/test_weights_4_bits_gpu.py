"""Products with 4-bit weights against float64.

The weights enter as whole numbers, which is exact, and sums and scales are float32: an element is off by its rounding to
bfloat16 (half a step, 2^-8 of it at most) and by the float32 sums, (K + 8) 2^-24 of the sum of its products' magnitudes.
Products of 256 and more tokens round each weight to bfloat16 first, another 2^-8 of each product's magnitude at most.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from fastgen_b200.csrc.ops import Ops
    return Ops(torch.bfloat16, DEV)


def _weight(g, n, k, group):
    from fastgen_b200.weights import Weight4
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).to(DEV)
    scales = (torch.rand(n, k // group, generator=g) * 0.1 + 0.001).to(torch.bfloat16).to(DEV)
    return Weight4(codes, scales)


def _check(got, x, w, bias=None, rounded_weights=False):
    dense = w.dequantize(torch.float64)
    want = x.double() @ dense.T
    room = x.double().abs() @ dense.abs().T
    if bias is not None:
        want = want + bias.double()
    bound = 2.0 ** -8 * want.abs() + ((x.shape[1] + 8) * 2.0 ** -24 + (2.0 ** -8 if rounded_weights else 0.0)) * room + 1e-30
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())


@pytest.mark.parametrize("m", [1, 5, 8, 9, 16, 17, 32, 33, 64, 65, 130, 255, 300])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (17, 64, 64), (128, 128, 128), (130, 96, 32), (300, 1152, 128), (2049, 320, 64),
                                       (96, 4096, 128), (40, 14336, 128), (5000, 256, 32)])
def test_product(ops, m, n, k, group):
    g = torch.Generator().manual_seed(m * 7 + n + k)
    w = _weight(g, n, k, group)
    x = (torch.randn(m, k, generator=g) * 3).to(torch.bfloat16).to(DEV)
    bias = torch.randn(n, generator=g).to(torch.bfloat16).to(DEV)
    got = ops.linear(x, w)
    ops.check_status()
    assert got.shape == (m, n) and got.dtype == torch.bfloat16
    rounded = m >= 256
    _check(got, x, w, rounded_weights=rounded)
    _check(ops.linear(x, w, bias=bias), x, w, bias, rounded)
    assert torch.equal(got, ops.linear(x, w))
    # rows off 16 bytes, a result inside a wider one whose other columns stay
    odd = torch.empty(m, k + 3, dtype=torch.bfloat16, device=DEV)[:, 3:]
    odd.copy_(x)
    wide = torch.full((m, n + 5), 3.0, dtype=torch.bfloat16, device=DEV)
    ops.linear(odd, w, out=wide[:, :n])
    assert bool((wide[:, n:] == 3.0).all())
    if rounded:  # (the library orders its sums by the operands' alignment: each result is within the bound, not the same)
        _check(wide[:, :n], x, w, rounded_weights=True)
    else:
        assert torch.equal(wide[:, :n], got)


@pytest.mark.parametrize("m", [1, 12, 20, 70])
def test_float32_results_and_activations(ops, m):
    g = torch.Generator().manual_seed(m)
    w = _weight(g, 200, 512, 128)
    x = torch.randn(m, 512, generator=g).to(torch.bfloat16).to(DEV)
    full = ops.linear(x, w, out_dtype=torch.float32)
    want = x.double() @ w.dequantize(torch.float64).T
    room = x.double().abs() @ w.dequantize(torch.float64).abs().T
    assert full.dtype == torch.float32 and bool(((full.double() - want).abs() <= 520 * 2.0 ** -24 * room).all())
    plain = ops.linear(x, w).float()
    assert torch.equal(plain, full.to(torch.bfloat16).float())
    for act, f in (("gelu_erf", torch.nn.functional.gelu), ("relu2", lambda z: torch.relu(z) ** 2)):
        got, ref = ops.linear(x, w, act=act).float(), f(plain)
        assert bool(((got - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5).all())


@pytest.mark.parametrize("m", [1, 8, 16, 17, 64, 100, 300])
@pytest.mark.parametrize("act", ["silu", "relu"])
def test_gated_product(ops, m, act):
    """Gate and up rows in blocks of eight, as a feed-forward binds them."""
    g = torch.Generator().manual_seed(m)
    f, k = 168, 256
    w = _weight(g, 2 * f, k, 64)
    x = torch.randn(m, k, generator=g).to(torch.bfloat16).to(DEV)
    got = ops.linear_swiglu(x, w, act=act).float()
    both = ops.linear(x, w).float().view(m, f // 8, 2, 8)
    gate, up = both[:, :, 0].reshape(m, f), both[:, :, 1].reshape(m, f)
    ref = (torch.relu(gate) if act == "relu" else torch.nn.functional.silu(gate)) * up
    assert bool(((got - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -18 * up.abs()).all())


def test_rows_and_special_numbers(ops):
    g = torch.Generator().manual_seed(0)
    w = _weight(g, 300, 384, 128)
    for m in (4, 40):
        x = torch.randn(m, 384, generator=g).to(torch.bfloat16).to(DEV)
        whole = ops.linear(x, w)
        assert torch.equal(ops.linear(x, w[16:130]), whole[:, 16:130])
        x[1, 7], x[2, 9] = float("inf"), float("nan")
        poisoned = ops.linear(x, w)
        keep = [r for r in range(m) if r not in (1, 2)]
        assert torch.equal(poisoned[keep], whole[keep])
        assert not bool(torch.isfinite(poisoned[2]).any()) and not bool(torch.isfinite(poisoned[1]).any())
    assert ops.linear(x[:0], w).shape == (0, 300)


@pytest.mark.parametrize("m", [3, 20])
def test_one_row_for_all_tokens_and_the_same_twice(ops, m):
    """Rows without a stride between them; two calls with the same operands."""
    g = torch.Generator().manual_seed(m)
    w = _weight(g, 130, 256, 64)
    row = torch.randn(1, 256, generator=g).to(torch.bfloat16).to(DEV)
    y = ops.linear(row.expand(m, -1), w)
    assert torch.equal(y, ops.linear(row.repeat(m, 1), w)) and torch.equal(y, ops.linear(row.expand(m, -1), w))
    assert ops.linear(row[:0], w).shape == (0, 130)


def test_two_products_at_once_and_in_a_graph(ops):
    """Clusters of two launches side by side on the chip; a captured product gives the eager one's bits."""
    g = torch.Generator().manual_seed(5)
    w = [_weight(g, 4096, 2048, 128), _weight(g, 1024, 4096, 64)]
    x = [torch.randn(m, k, generator=g).to(torch.bfloat16).to(DEV) for m, k in ((64, 2048), (100, 4096))]
    want = [ops.linear(a, b) for a, b in zip(x, w)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.linear(x[i], w[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [ops.linear(a, b) for a, b in zip(x, w)]
    x[0].mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0].float(), 2 * want[0].float()) and torch.equal(out[1], want[1])
    ops.check_status()


def test_refusals(ops):
    from fastgen_b200.csrc.ops import Ops
    g = torch.Generator().manual_seed(0)
    w = _weight(g, 40, 128, 64)
    for m in (1, 20, 300):
        with pytest.raises(ValueError, match="on cpu"):
            ops.linear(torch.zeros(m, 128, dtype=torch.bfloat16), w)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="bfloat16 activations"):
        ops.linear(x.float(), w)
    with pytest.raises(ValueError, match="bfloat16 activations"):
        Ops(torch.float32, DEV).linear(x.float(), w)
    with pytest.raises(ValueError, match="a product of"):
        ops.linear(x[:, :64], w)
    with pytest.raises(ValueError, match="bias"):
        ops.linear(x, w, bias=torch.zeros(40, device=DEV))
    assert ops.linear_swiglu(x, w) is None  # 40 rows are no whole blocks of gate and up
