"""Activations kept in 8 bits, against plain 64-bit forms.  Bounds: a kept value is within half a step, top / 254 of its
block (1 + 2^-10: the scale and the quotient are fp32); results are rounded once to their type; fp32 arithmetic of a few
dozen operations is off by less than 2^-18 relative to the terms it adds."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SHAPES = [(1, 1), (3, 15), (2, 16), (5, 100), (1, 127), (7, 128), (3, 129), (4, 144), (33, 200), (9, 1001), (129, 1024), (70, 4096), (2, 8192), (3, 8200), (300, 264)]


def ops():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    from blackriver_b200 import ops
    return ops


def data(rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * scale
    x[:, ::53] *= 15
    return x.to(dtype)


def tops(x):
    """Largest magnitude of each value's block, [rows, cols] in 64 bits."""
    x = x.double().abs()
    return torch.cat([x[:, c:c + 128].amax(1, keepdim=True).expand(-1, min(128, x.shape[1] - c)) for c in range(0, x.shape[1], 128)], 1)


def values(q, scale):
    return q.double() * scale.double().repeat_interleave(128, 1)[:, :q.shape[1]]


def gelu(x):
    return 0.5 * x * (1 + torch.tanh(0.79788456 * x * (1 + 0.044715 * x * x)))


def close(got, want, bound, name=""):
    off = (got.double() - want).abs()
    assert (off <= bound).all(), f"{name}: {(off / bound).max().item():.3g} times the bound"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_pack_and_unpack(rows, cols, dtype):
    o = ops()
    x = data(rows, cols, dtype, rows + cols)
    q, scale = o.act8_pack(x)
    top = tops(x)
    close(values(q, scale), x.double(), top / 254 * (1 + 2.0 ** -10) + 1e-30, "kept")
    assert q.abs().max() <= 127 and (q.abs().amax(1) == 127).all()
    for out_dtype in (torch.float16, torch.float32):
        got = o.act8_unpack(q, scale, out_dtype)
        close(got, values(q, scale), values(q, scale).abs() * HALF_STEP[out_dtype] * 1.01 + 2.0 ** -25, "unpacked")
    # what is already a multiple of the step comes back as it was
    y = torch.randint(-127, 128, (rows, cols), device="cuda").float()
    y[:, ::128] = 127.0
    q, scale = o.act8_pack(y)
    assert torch.equal(q.float(), y) and (scale == 1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_gelu(rows, cols, dtype):
    o = ops()
    x, dy = data(rows, cols, dtype, cols, 0.5), data(rows, cols, dtype, cols + 1)
    y, q, scale = o.gelu_act8(x)
    half = HALF_STEP[dtype] * 1.01
    close(y, gelu(x.double()), gelu(x.double()).abs() * half + 2.0 ** -21 * (1 + x.double().abs()) + (2.0 ** -25 if dtype == torch.float16 else 0), "y")
    q2, scale2 = o.act8_pack(x)
    assert torch.equal(q, q2) and torch.equal(scale, scale2)
    kept = values(q, scale).requires_grad_(True)
    again_want = gelu(kept)
    (want,) = torch.autograd.grad(again_want, kept, dy.double())
    dx, again = o.gelu_backward_act8(dy, q, scale, recompute=True)
    k = kept.detach().abs()
    close(dx, want, want.abs() * half + 2.0 ** -19 * dy.double().abs() * (1 + k) + 2.0 ** -25, "dx")
    close(again, again_want.detach(), again_want.detach().abs() * half + 2.0 ** -20 * (1 + k) + 2.0 ** -25, "y again")
    assert torch.equal(o.gelu_backward_act8(dy, q, scale), dx)
    # in place, as the outputs of the other GELU calls may be
    x2, dy2 = x.clone(), dy.clone()
    y2, q2, _ = o.gelu_act8(x2, out=x2)
    assert y2 is x2 and torch.equal(y2, y) and torch.equal(q2, q)
    assert torch.equal(o.gelu_backward_act8(dy2, q, scale, out=dy2), dx)


def test_gelu_gradient_against_differences():
    o = ops()
    x = torch.linspace(-6, 6, 257, device="cuda").view(1, -1)
    q, scale = o.act8_pack(x)
    kept = values(q, scale)
    dx = o.gelu_backward_act8(torch.ones_like(x), q, scale)
    h = 1e-5
    slope = (gelu(kept + h) - gelu(kept - h)) / (2 * h)
    close(dx, slope, torch.full_like(slope, 2.0 ** -18 * 7), "slope")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layernorm(rows, cols, dtype):
    o = ops()
    if cols == 1:
        pytest.skip("a row of one value has no spread")
    eps, half = 1e-5, HALF_STEP[dtype] * 1.01
    x, dy, res = (data(rows, cols, dtype, cols + i, 1.5) for i in range(3))
    g = torch.Generator(device="cuda").manual_seed(cols)
    gamma = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
    gamma[0] = 0.0                                          # xhat is kept, not y: nothing is divided by gamma
    beta = (0.3 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
    y, q, scale, var = o.layernorm_act8(x, gamma, beta, eps)
    X = x.double()
    mu = X.mean(1, keepdim=True)
    v = (X - mu).square().mean(1) + eps
    xhat = (X - mu) / v.sqrt()[:, None]
    ga, be = gamma.double(), beta.double()
    close(var, v, v * 2.0 ** -19, "var")
    # the row's mean carries 2^-20 of its largest value into every difference
    soft = 2.0 ** -18 * (xhat.abs() + X.abs().amax(1, keepdim=True) / v.sqrt()[:, None])
    close(y, xhat * ga + be, (xhat * ga + be).abs() * half + soft * ga.abs() + 2.0 ** -22 * be.abs() + 2.0 ** -25, "y")
    close(values(q, scale), xhat, tops(xhat) / 254 * (1 + 2.0 ** -10) + soft, "kept")
    kept, DY = values(q, scale), dy.double()
    gr = DY * ga
    parts = (gr.abs() + gr.abs().mean(1, keepdim=True) + kept.abs() * (gr * kept).abs().mean(1, keepdim=True)) / var.double().sqrt()[:, None]
    want = (gr - gr.mean(1, keepdim=True) - kept * (gr * kept).mean(1, keepdim=True)) / var.double().sqrt()[:, None]
    dgamma_want, dbeta_want = (DY * kept).sum(0), DY.sum(0)
    for residual in (None, res):
        dgamma, dbeta, dx, again = o.layernorm_backward_act8(dy, gamma, var, q, scale, beta=beta, residual=residual)
        w = want if residual is None else want + residual.double()
        close(dx, w, w.abs() * half + 2.0 ** -18 * parts + 2.0 ** -25, "dx")
        close(dgamma, dgamma_want, dgamma_want.abs() * half + 2.0 ** -18 * (DY * kept).abs().sum(0) + 2.0 ** -25, "dgamma")
        close(dbeta, dbeta_want, dbeta_want.abs() * half + 2.0 ** -18 * DY.abs().sum(0) + 2.0 ** -25, "dbeta")
        close(again, kept * ga + be, (kept * ga + be).abs() * half + 2.0 ** -22 * ((kept * ga).abs() + be.abs()) + 2.0 ** -25, "y again")
        three = o.layernorm_backward_act8(dy, gamma, var, q, scale, residual=residual)
        assert torch.equal(three[0], dgamma) and torch.equal(three[1], dbeta) and torch.equal(three[2], dx)
        # in place, and added to what is there
        dy2, dg2, db2 = dy.clone(), torch.ones_like(dgamma), torch.ones_like(dbeta)
        o.layernorm_backward_act8(dy2, gamma, var, q, scale, residual=residual, dgamma=dg2, dbeta=db2, dx=dy2, accumulate=True)
        assert torch.equal(dy2, dx)
        close(dg2, dgamma_want + 1, (dgamma_want + 1).abs() * half + 2.0 ** -18 * (1 + (DY * kept).abs().sum(0)) + 2.0 ** -25, "added dgamma")
        close(db2, dbeta_want + 1, (dbeta_want + 1).abs() * half + 2.0 ** -18 * (1 + DY.abs().sum(0)) + 2.0 ** -25, "added dbeta")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [256, 300])
def test_blocks_without_a_scale(cols, dtype):
    """Zeros, values too small for a scale, infinities and NaN: each stays inside its block."""
    o = ops()
    x = data(6, cols, dtype, 4)
    clean_q, clean_scale = o.act8_pack(x)
    x[1, :128] = 0
    x[2, 5] = float("inf")
    x[3, 128 + 7] = float("nan")
    x[4, :128] = 1e-38 if dtype == torch.float32 else 0
    x[5, 200] = float("-inf")
    q, scale = o.act8_pack(x)
    got = o.act8_unpack(q, scale, torch.float32)
    assert (got[1, :128] == 0).all() and (got[4, :128] == 0).all()
    for r, c in ((2, 0), (3, 128), (5, 128)):
        assert torch.isnan(got[r, c:c + 128]).all()
        rest = torch.ones(cols, dtype=torch.bool, device="cuda")
        rest[c:c + 128] = False
        assert torch.isfinite(got[r, rest]).all()
        assert torch.equal(q[r, rest], clean_q[r, rest])
    assert torch.equal(q[0], clean_q[0]) and torch.equal(scale[0], clean_scale[0])
    dx = o.gelu_backward_act8(torch.ones_like(x), q, scale)
    assert torch.isnan(dx[2, :128]).all() and torch.isfinite(dx[0]).all()
    subnormal = torch.full((1, 128), 6e-8, device="cuda", dtype=torch.float16)
    assert torch.equal(o.act8_unpack(*o.act8_pack(subnormal)), subnormal)


def test_views_that_are_not_aligned():
    o = ops()
    base = data(1, 64 * 256 + 1, torch.float16, 1)[0]
    x, y = base[1:].view(64, 256), base[:-1].view(64, 256).clone()
    x2 = x.clone()
    for a, b in zip(o.act8_pack(x), o.act8_pack(x2)):
        assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(o.gelu_act8(x), o.gelu_act8(x2)))
    gamma, beta = y[0].clone(), y[1].clone()
    one, two = o.layernorm_act8(x, gamma, beta), o.layernorm_act8(x2, gamma, beta)
    torch.testing.assert_close(one[0], two[0], rtol=2.0 ** -10, atol=2.0 ** -14)      # sums in another order: one rounding apart
    torch.testing.assert_close(one[3], two[3], rtol=1e-6, atol=0)


def test_no_rows():
    o = ops()
    x = torch.empty(0, 256, dtype=torch.float16, device="cuda")
    q, scale = o.act8_pack(x)
    assert o.act8_unpack(q, scale).shape == (0, 256)
    gamma = torch.ones(256, dtype=torch.float16, device="cuda")
    dgamma, dbeta, dx = o.layernorm_backward_act8(x, gamma, torch.empty(0, device="cuda"), q, scale)
    assert (dgamma == 0).all() and (dbeta == 0).all() and dx.shape == x.shape
    o.layernorm_backward_act8(x, gamma, torch.empty(0, device="cuda"), q, scale, dgamma=gamma, dbeta=dbeta, accumulate=True)
    assert (gamma == 1).all()


def test_captured_and_on_another_stream():
    o = ops()
    x, dy = data(500, 1024, torch.float16, 1), data(500, 1024, torch.float16, 2)
    gamma, beta = data(1, 1024, torch.float16, 3)[0], data(1, 1024, torch.float16, 4)[0]

    def step():
        y, q, s, var = o.layernorm_act8(x, gamma, beta)
        z, q2, s2 = o.gelu_act8(y)
        dx = o.gelu_backward_act8(dy, q2, s2)
        return (y, z, q, q2) + o.layernorm_backward_act8(dx, gamma, var, q, s, residual=dy)

    want = [t.clone() for t in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(data(500, 1024, torch.float16, 9))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in got]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    assert not torch.equal(got[0], want[0])


@pytest.mark.parametrize("cols", [256, 37])
def test_gelu_of_values_whose_square_overflows(cols):
    o = ops()
    x = torch.full((3, cols), 1e25, device="cuda")
    x[:, ::2] = -1e25
    y, q, scale = o.gelu_act8(x)
    assert torch.equal(y, torch.where(x > 0, x, torch.zeros_like(x)))
    dx = o.gelu_backward_act8(torch.full_like(x, 3.0), q, scale)
    assert torch.equal(dx, torch.where(x > 0, 3.0, 0.0))


@pytest.mark.parametrize("cols", [512, 131])
def test_values_between_two_steps_go_to_even(cols):
    o = ops()
    x = torch.randn(700, cols, generator=torch.Generator().manual_seed(cols)).half()
    x[:, 1] = (x[:, :128].abs().amax(1).float() / 2).half()
    blocks = [x[:, at:at + 128] for at in range(0, cols, 128)]
    # x * 127 is exact in 64 bits and a quotient that is a half stays one
    want = torch.cat([torch.round(b.double() * 127 / b.double().abs().amax(1, keepdim=True)) for b in blocks], 1)
    assert torch.equal(o.act8_pack(x.cuda())[0].double().cpu(), want)
    assert torch.equal(o.gelu_act8(x.cuda())[1].double().cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_layernorm_of_rows_of_one_value(dtype):
    o = ops()
    x, gamma, beta = data(5, 1, dtype, 3).cuda(), torch.full((1,), 2.0, dtype=dtype, device="cuda"), torch.full((1,), 0.5, dtype=dtype, device="cuda")
    y, q, scale, var = o.layernorm_act8(x, gamma, beta, 1e-3)
    assert torch.equal(y, beta.expand(5, 1)) and not q.any() and not scale.any()
    assert ((var - 1e-3).abs() <= 1e-3 * 2.0 ** -23).all()
    dy = data(5, 1, dtype, 4).cuda()
    dgamma, dbeta, dx, again = o.layernorm_backward_act8(dy, gamma, var, q, scale, beta=beta)
    assert not dgamma.any() and not dx.any() and torch.equal(again, y)
    total = dy.double().sum()
    assert (dbeta.double() - total).abs() <= total.abs() * torch.finfo(dtype).eps / 2 + dy.double().abs().sum() * 2.0 ** -21
