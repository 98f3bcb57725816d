"""GPU parity of the gated projection with its definition in 64 bits.

Bounds: the gates g and what they multiply, u, are float32 sums, within e = 1e-5 of the sums Sg and Su of their absolute terms.  With
A = |act(g)|, D = |act'(g)| (the activations' slopes are at most 1.13, the slopes' own at most 0.8):
y within e (1.13 Sg |u| + A Su + |y|) and its rounding; the gradients at g and u within e |dy| (Su D + 0.8 |u| Sg + |u| D) and
e |dy| (1.13 Sg + A).  For the products that follow they are rounded to x's type.  relu's slope is either of both where |g| <= e Sg."""
import pytest
import torch

from tests import seq_ref as ref
from tests.seq_ref import UNIT, f64, near

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def rnd(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def case(x, w, b, act, dy):
    from v1_glif_model_amd import sequence as seq
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = seq.gated_linear(*leaves, activation=act)
    with torch.no_grad():
        assert torch.equal(y.detach(), seq.gated_linear(x, w, b, act))
    got = torch.autograd.grad(y, leaves, dy)
    K, N = w.shape[1], w.shape[0] // 2
    x6, w6, d6 = f64(x, False).reshape(-1, K), f64(w, False), f64(dy, False).reshape(-1, N)
    b6 = torch.zeros(2 * N, dtype=ref.F64) if b is None else f64(b, False)
    g, u = (x6 @ w6.t() + b6).split(N, -1)
    sg, su = (x6.abs() @ w6.abs().t() + b6.abs()).split(N, -1)
    on, slope = ref.act(g, act), ref.slope(g, act)
    near(y.reshape(-1, N), on * u, 1.13 * sg * u.abs() + on.abs() * su + (on * u).abs(), "y")
    dp = torch.cat([d6 * u * slope, d6 * on], -1)
    da, ua, D = d6.abs(), u.abs(), slope.abs()
    off = 1e-5 * torch.cat([da * (su * D + 0.8 * ua * sg + ua * D), da * (1.13 * sg + on.abs())], -1)
    if act == "relu":
        off[:, :N] += torch.where(g.abs() <= 1e-5 * sg, da * ua, torch.zeros((), dtype=ref.F64))
    off += (0.0 if x.dtype is F32 else UNIT[x.dtype] + ref.TINY[x.dtype]) * dp.abs()
    size = dp.abs() + off
    more = 2.0 ** -24 if x.dtype is F16 else 0.0     # a gradient below float16's normal numbers
    near(got[0].reshape(-1, K), dp @ w6, size @ w6.abs(), "dx", off @ w6.abs() + more * w6.abs().sum(0))
    near(got[1], dp.t() @ x6, size.t() @ x6.abs(), "dw", off.t() @ x6.abs() + more * x6.abs().sum(0))
    if b is not None:
        near(got[2], dp.sum(0), size.sum(0), "db", off.sum(0))


SHAPES = [(1, 1, 1), (1, 64, 16), (5, 512, 100), (16, 130, 17), (17, 40, 33), (32, 1000, 64), (33, 64, 8), (70, 72, 16), (100, 257, 90),
          (130, 96, 300), (257, 128, 128), (300, 33, 129), (3, 4096, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype):
    """Few rows, few columns, every kind of tile; sizes that are no multiple of anything."""
    M, K, N = shape
    act = ("silu", "gelu", "relu", None)[(M + N) % 4]
    case(rnd(1, M, K, dtype=dtype), rnd(2, 2 * N, K, dtype=dtype, scale=K ** -0.5), rnd(3, 2 * N, dtype=F32 if M % 2 else dtype), act,
         rnd(4, M, N, dtype=dtype))


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
def test_activations_and_no_bias(act):
    case(rnd(1, 3, 4, 64, dtype=BF16), rnd(2, 96, 64, dtype=BF16, scale=0.125), None, act, rnd(3, 3, 4, 48, dtype=BF16))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2500, 512, 1365), (1000, 600, 4200), (5000, 200, 520)])
def test_large(shape, dtype):
    """Tiles of every size, products in two pieces along either side: all rows of some columns, against 64 bits on the device."""
    from v1_glif_model_amd import sequence as seq
    M, K, N = shape
    x, w = rnd(1, M, K, dtype=dtype).requires_grad_(True), rnd(2, 2 * N, K, dtype=dtype, scale=K ** -0.5).requires_grad_(True)
    b, dy = rnd(3, 2 * N, dtype=dtype).requires_grad_(True), rnd(4, M, N, dtype=dtype)
    y = seq.gated_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        x6, w6, b6, d6 = (t.double() for t in (x, w, b, dy))
        g, u = (x6 @ w6.t() + b6).split(N, -1)
        sg, su = (x6.abs() @ w6.abs().t() + b6.abs()).split(N, -1)
        q = torch.sigmoid(g)
        on, slope = g * q, q * (1 + g * (1 - q))
        near(y, (on * u).cpu(), (1.13 * sg * u.abs() + on.abs() * su + (on * u).abs()).cpu(), "y")
        dp = torch.cat([d6 * u * slope, d6 * on], -1)
        da, ua, D = d6.abs(), u.abs(), slope.abs()
        off = 1e-5 * torch.cat([da * (su * D + 0.8 * ua * sg + ua * D), da * (1.13 * sg + on.abs())], -1)
        off += (0.0 if dtype is F32 else UNIT[dtype]) * dp.abs()
        size = dp.abs() + off
        near(dx, (dp @ w6).cpu(), (size @ w6.abs()).cpu(), "dx", (off @ w6.abs()).cpu())
        near(dw, (dp.t() @ x6).cpu(), (size.t() @ x6.abs()).cpu(), "dw", (off.t() @ x6.abs()).cpu())
        near(db, dp.sum(0).cpu(), size.sum(0).cpu(), "db", off.sum(0).cpu())


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Rows apart and off 16 bytes, transposed weights, a broadcast gradient."""
    x, w = rnd(1, 60, 90, dtype=dtype), rnd(2, 101, 90, dtype=dtype)
    case(x[::2, 3:73], w[1:81, 5:75], rnd(3, 160)[::2], "silu", rnd(4, 1, 40, dtype=dtype).expand(30, 40))
    case(rnd(5, 48, 50, dtype=dtype).t(), rnd(6, 48, 64, dtype=dtype).t(), None, "gelu", rnd(7, 32, 50, dtype=dtype).t())


def test_gradients_against_differences():
    """In float32, by central differences: their own error is the third difference, a step's square (2^-12) of the terms."""
    from v1_glif_model_amd import sequence as seq
    x, w, b, dy = rnd(1, 9, 30), rnd(2, 24, 30, scale=0.2), rnd(3, 24), rnd(4, 9, 12)

    def loss(*t):
        y = seq.gated_linear(*t).double() * dy
        return y.sum(), y.abs().sum()

    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(loss(*leaves)[0], leaves)
    for i in range(3):
        d = rnd(10 + i, *leaves[i].shape)
        d /= d.norm()
        h = 2.0 ** -6
        with torch.no_grad():
            up, size = loss(*(t + h * d if j == i else t for j, t in enumerate(leaves)))
            down, _ = loss(*(t - h * d if j == i else t for j, t in enumerate(leaves)))
            assert abs(float((up - down) / (2 * h) - (got[i].double() * d).sum())) <= (h * h + 2e-6 / h) * float(size), i


def test_partial_gradients_and_empty():
    from v1_glif_model_amd import sequence as seq
    x, w, b, dy = rnd(1, 40, 64, dtype=BF16), rnd(2, 72, 64, dtype=BF16), rnd(3, 72), rnd(4, 40, 36, dtype=BF16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    whole = torch.autograd.grad(seq.gated_linear(*leaves), leaves, dy)
    for i in range(3):
        one = [t.detach().requires_grad_(i == j) for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(seq.gated_linear(*one), one[i], dy)[0], whole[i])
    for M, N, K in ((0, 8, 16), (4, 0, 16), (4, 8, 0)):
        e = [rnd(1, M, K).requires_grad_(True), rnd(2, 2 * N, K).requires_grad_(True), rnd(3, 2 * N).requires_grad_(True)]
        y = seq.gated_linear(*e)
        g = torch.autograd.grad(y, e, torch.ones_like(y))
        assert y.shape == (M, N) and all(a.shape == t.shape for a, t in zip(g, e))
        if K == 0:
            b6 = e[2].detach().double().cpu()
            near(y, (ref.act(b6[:8], "silu") * b6[8:]).expand(4, 8), 3.0, "y")
        else:
            assert not any(t.any() for t in g)


def test_rows_that_are_not_finite():
    """NaN and infinities in a row of x stay in that row; relu lets NaN through."""
    from v1_glif_model_amd import sequence as seq
    for M, dtype in ((5, BF16), (200, BF16), (200, F32)):
        x, w = rnd(1, M, 128, dtype=dtype), rnd(2, 96, 128, dtype=dtype)
        clean = seq.gated_linear(x, w, activation="relu")
        x[3, 7] = float("nan")
        y = seq.gated_linear(x, w, activation="relu")
        rest = [i for i in range(M) if i != 3]
        assert torch.equal(y[rest], clean[rest]) and y[3].isnan().all()


def test_capture_and_streams():
    from v1_glif_model_amd import sequence as seq
    x, w, dy = rnd(1, 300, 200, dtype=BF16), rnd(2, 260, 200, dtype=BF16), rnd(3, 300, 130, dtype=BF16)

    def run(x, w):
        leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
        y = seq.gated_linear(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = run(x, w)
        few = seq.gated_linear(x[:4], w)
    for n in range(4):
        x.copy_(rnd(10 + n, *x.shape, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, run(x, w)):
            assert torch.equal(a, b)
        assert torch.equal(few, seq.gated_linear(x[:4], w))


def test_refusals():
    from v1_glif_model_amd import sequence as seq
    good = dict(x=rnd(1, 4, 8), weight=rnd(2, 12, 8), bias=rnd(3, 12))
    for change in (dict(x=good["x"].cpu()), dict(x=good["x"].double()), dict(weight=rnd(2, 11, 8), bias=None), dict(weight=rnd(2, 12, 7)),
                   dict(weight=good["weight"].half()), dict(bias=rnd(3, 6)), dict(bias=good["bias"].half()), dict(activation="tanh"),
                   dict(x=torch.zeros((), device=DEV))):
        with pytest.raises(ValueError):
            seq.gated_linear(**{**good, **change})
    x = good["x"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(seq.gated_linear(x, good["weight"]).sum(), x, create_graph=True)
