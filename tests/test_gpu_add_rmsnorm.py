"""enc_ops.add_rmsnorm and mx_ops.add_rmsnorm_mx8 against the formulas in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32, relative).  A lane adds at most 32 squares, the butterfly 6 and the waves 16
more: the sum of squares is off by at most 54 u, its root by 27 u, the division, root, eps and mean add 4, the two products
of y 2: |y - y64| <= 40 u |y64|.  The gradient's inner product has the same chain over products of three factors, and is
scaled by inv^3: dx is off by at most 128 u of the sum of the magnitudes of its terms.  dscale adds T products in some
order: (T + 64) u of the sum of their magnitudes.  A bfloat16 result adds one rounding, eps / 2 = 2^-8 of the value."""
import pytest
import torch

from generative_recommenders_amd import enc_ops, hmx, mx_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}
EPS = 1e-6


def make(T, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, d, generator=g).to(dtype).to(DEV)
    r = (2 * torch.randn(T, d, generator=g)).to(dtype).to(DEV)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(DEV)
    return x, r, w, torch.randn(T, d, generator=g).to(dtype).to(DEV), torch.randn(T, d, generator=g).to(dtype).to(DEV)


def formula(s, w, dy=None, ds=None, eps=EPS):
    s, w = s.double(), w.double()
    inv = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    y = s * inv * w
    if dy is None:
        return y
    dy = dy.double()
    g = dy * w
    k = (g * s).mean(-1, keepdim=True) * inv ** 2
    dx = inv * (g - s * k)
    mag = inv * (g.abs() + s.abs() * (g * s).abs().mean(-1, keepdim=True) * inv ** 2)
    if ds is not None:
        dx, mag = dx + ds.double(), mag + ds.double().abs()
    terms = (dy * s * inv).reshape(-1, s.shape[-1])
    return y, dx, mag, terms.sum(0), terms.abs().sum(0)


def within(got, want, tol):
    bad = (got.double() - want).abs() > tol + 1e-37
    assert got.shape == want.shape and not bool(bad.any()), float(((got.double() - want).abs() / (tol + 1e-37)).max())


SHAPES = [(1, 1), (1, 64), (3, 7), (5, 33), (17, 64), (1024, 64), (300, 100), (129, 128), (65, 250), (33, 512), (7, 1000),
          (9, 1025), (4, 2048), (3, 4096), (2, 5001), (2, 8192), (1, 16384), (2, 20001), (1, 32768), (2049, 96)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,d", SHAPES)
def test_forward_and_gradients(T, d, dtype):
    x, r, w, dy, ds = make(T, d, dtype)
    for t in (x, r, w):
        t.requires_grad_()
    y, s = enc_ops.add_rmsnorm(x, r, w, EPS)
    assert y.dtype == s.dtype == dtype
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    want_y, want_dx, mag, want_dw, mag_w = formula(s.detach(), w.detach(), dy, ds)
    within(y, want_y, (40 * U + HALF[dtype]) * want_y.abs())
    dx, dr, dw = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    within(dx, want_dx, 128 * U * mag + HALF[dtype] * (want_dx.abs() + 128 * U * mag))
    assert torch.equal(dx, dr)
    within(dw, want_dw, (T + 64) * U * mag_w)


@pytest.mark.parametrize("T,d", [(5, 33), (40, 64), (3, 1000)])
def test_no_residual_and_partial_gradients(T, d):
    x, _, w, dy, ds = make(T, d, torch.float32, 3)
    x.requires_grad_()
    w.requires_grad_()
    y, s = enc_ops.add_rmsnorm(x, None, w, EPS)
    assert s is x
    want_y, want_dx, mag, want_dw, mag_w = formula(x.detach(), w.detach(), dy)
    within(y, want_y, 40 * U * want_y.abs())
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    within(dx, want_dx, 128 * U * mag)
    within(dw, want_dw, (T + 64) * U * mag_w)
    r = torch.zeros_like(x).requires_grad_()
    y, s = enc_ops.add_rmsnorm(x, r, w, EPS)          # only y, only s, and one leaf as both operands
    assert torch.equal(torch.autograd.grad(y, x, dy, retain_graph=True)[0], dx)
    assert torch.equal(torch.autograd.grad(s, r, ds)[0], ds)
    y, s = enc_ops.add_rmsnorm(x, x, w, EPS)
    want = 2 * formula(s.detach(), w.detach(), dy)[1]
    within(torch.autograd.grad(y, x, dy)[0], want, 2 * 130 * U * formula(s.detach(), w.detach(), dy)[2])
    y, s = enc_ops.add_rmsnorm(x, r, w, EPS)
    (y * dy).sum().backward()
    (enc_ops.add_rmsnorm(x, r, w, EPS)[0] * dy).sum().backward()      # accumulation into .grad of both leaves
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    within(x.grad, 2 * want_dx, 2 * 130 * U * mag)


def test_gradient_against_differences():
    """Along random directions of x, residual and scale: the kernel's values at +h and -h, added in 64 bits.  Allowed: the
    rounding of the 2 T d values (40 u each, over 2 h) and what the same difference is off the derivative in 64 bits."""
    T, d, h = 6, 100, 2.0 ** -5
    x, r, w, dy, ds = make(T, d, torch.float32, 5)
    g = torch.Generator().manual_seed(8)
    dirs = [torch.randn(*t.shape, generator=g).to(DEV) for t in (x, r, w)]
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, s = enc_ops.add_rmsnorm(*leaves, EPS)
    grads = torch.autograd.grad((y, s), leaves, (dy, ds))
    for k, v in enumerate(dirs):
        ends, ends64, mags = [], [], 0.0
        for sign in (1, -1):
            moved = [t + sign * h * v if i == k else t for i, t in enumerate((x, r, w))]
            yk, sk = enc_ops.add_rmsnorm(*moved, EPS)
            ends.append(float((yk.double() * dy).sum() + (sk.double() * ds).sum()))
            s64 = moved[0].double() + moved[1].double()
            y64 = formula(s64, moved[2])
            ends64.append(float((y64 * dy).sum() + (s64 * ds).sum()))
            # y and s are rounded, and s of the moved operands once more before y is formed from it
            mags += float((y64 * dy).abs().sum() * 44 + (s64 * ds).abs().sum() * 2)
        slope = float((grads[k].double() * v).sum())
        l64 = [t.double().clone().requires_grad_() for t in (x, r, w)]
        s64 = l64[0] + l64[1]
        y64 = formula(s64, l64[2])
        want = float((torch.autograd.grad((y64 * dy).sum() + (s64 * ds).sum(), l64[k])[0] * v).sum())
        off = abs((ends64[0] - ends64[1]) / (2 * h) - want)
        assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= off + U * mags / (2 * h) + 256 * U * mags


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_shapes(dtype):
    x, r, w, dy, _ = make(24, 40, dtype, 7)
    want = enc_ops.add_rmsnorm(x, r, w)
    big = torch.zeros(24, 91, dtype=dtype, device=DEV)
    big[:, 3:43] = x
    rt = r.t().contiguous().t()
    for xx, rr in ((big[:, 3:43], r), (x, rt), (x.view(2, 3, 4, 40), r.view(2, 3, 4, 40)),
                   (x.view(4, 6, 40).transpose(0, 1), r.view(4, 6, 40).transpose(0, 1))):
        got = enc_ops.add_rmsnorm(xx, rr, w)
        if xx.dim() == 3:
            got = tuple(t.transpose(0, 1) for t in got)
        for a, b in zip(got, want):
            tol = 80 * U + 2 * HALF[dtype]            # another lane layout adds the squares in another order
            within(a.reshape(24, 40), b.double(), tol * b.double().abs())
    row = r[:1].expand(24, 40).requires_grad_()
    y, s = enc_ops.add_rmsnorm(x, row, w)
    assert torch.equal(s, (x.float() + r[:1].float()).to(dtype))
    leaf = r[:1].clone().requires_grad_()              # the gradient of a broadcast operand is summed by expand
    y, s = enc_ops.add_rmsnorm(x, leaf.expand(24, 40), w)
    got = torch.autograd.grad(y, leaf, dy)[0]
    _, dx, mag, _, _ = formula(s.detach(), w, dy)
    within(got, dx.sum(0, keepdim=True), (24 + 128) * U * mag.sum(0, keepdim=True) + 4 * HALF[dtype] * mag.sum(0, keepdim=True))
    strided_dy = torch.zeros(24, 80, dtype=dtype, device=DEV)[:, ::2].copy_(dy)
    xl = x.clone().requires_grad_()
    y, s = enc_ops.add_rmsnorm(xl, r, w)
    assert torch.equal(torch.autograd.grad(y, xl, strided_dy, retain_graph=True)[0], torch.autograd.grad(y, xl, dy)[0])


def test_special_values_and_empty():
    x, r, w, _, _ = make(6, 64, torch.float32, 9)
    x[0] = 0
    r[0] = 0
    x[1, 5] = float("nan")
    x[2, 40] = float("inf")
    x[3] = 3e38
    r[3] = 3e38
    x[4] *= 1e-30
    r[4] = 0
    y, s = enc_ops.add_rmsnorm(x, r, w)
    assert bool((y[0] == 0).all()) and bool(y[1].isnan().all())
    assert bool(y[2, 40].isnan()) and bool((y[2, :40] == 0).all())
    assert bool(y[3].isnan().all())
    within(y[4:], formula(s[4:], w), 40 * U * formula(s[4:], w).abs())
    codes, scales, s2 = mx_ops.add_rmsnorm_mx8(x, r, w)
    assert torch.equal(s2.nan_to_num(7.0), s.nan_to_num(7.0))
    v = mx_ops.dequantize_mx8(codes, scales)
    assert bool((v[0] == 0).all()) and bool(v[1].isnan().all()) and bool(v[2, 32:].isnan().all()) and bool((v[2, :32] == 0).all())
    for T in (0, 2):
        e = torch.empty(T, 0, 8, device=DEV).requires_grad_()
        wl = torch.ones(8, device=DEV).requires_grad_()
        y, s = enc_ops.add_rmsnorm(e, e, wl)
        dw = torch.autograd.grad(y.sum(), wl)[0]
        assert y.shape == e.shape and bool((dw == 0).all())
        assert mx_ops.add_rmsnorm_mx8(e, e, wl)[0].shape == (T, 0, 32)


def least_exponent(amax):
    e = torch.ceil(torch.log2(amax.clamp_min(1e-300) / 448))
    e = torch.where(torch.exp2(e) * 448 < amax, e + 1, e)
    e = torch.where(torch.exp2(e - 1) * 448 >= amax, e - 1, e)
    return torch.where(amax > 0, e.clamp(-126, 127), 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,d", SHAPES)
def test_mx8(T, d, dtype):
    """Scales are the least exponent of some amax within 40 u of the exact one; a value is off by half a step of e4m3
    (2^-4 of it, or 2^-10 of the scale below 2^-6 of it) on top of y's own 40 u."""
    x, r, w, _, _ = make(T, d, dtype, 11)
    x *= torch.logspace(-3, 3, T, device=DEV).unsqueeze(1).to(dtype)
    codes, scales, s = mx_ops.add_rmsnorm_mx8(x, r, w, EPS)
    dp = mx_ops.padded(d)
    assert codes.shape == (T, dp) and scales.shape == (T, dp // 32) and codes.dtype == torch.float8_e4m3fn
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    y = torch.zeros(T, dp, dtype=torch.float64, device=DEV)
    y[:, :d] = formula(s, w)
    amax = y.view(T, -1, 32).abs().amax(2)
    e = scales.double() - 127
    assert bool((e >= least_exponent(amax * (1 - 40 * U))).all()) and bool((e <= least_exponent(amax * (1 + 40 * U))).all())
    assert bool((codes[:, d:].float() == 0).all())
    unit = torch.exp2(e).repeat_interleave(32, 1)
    values = codes.double() * unit
    within(values, y, torch.maximum(2.0 ** -4 * y.abs() * (1 + 40 * U), 2.0 ** -10 * unit) + 40 * U * y.abs())
    for dt in (torch.float32, torch.bfloat16):
        assert torch.equal(mx_ops.dequantize_mx8(codes, scales, d, dt).double(), values[:, :d])


def test_mx8_no_residual_equals_zero_residual():
    x, _, w, _, _ = make(9, 96, torch.float32, 13)
    a = mx_ops.add_rmsnorm_mx8(x, None, w)
    b = mx_ops.add_rmsnorm_mx8(x, torch.zeros_like(x), w)
    assert a[2] is x and torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def test_refusals():
    x, r, w, dy, _ = make(4, 64, torch.float32)
    for f in (enc_ops.add_rmsnorm, mx_ops.add_rmsnorm_mx8):
        for args in ((x.half(), r.half(), w), (x, r[:3], w), (x, r.bfloat16(), w), (x, r, w[:5]), (x, r, w.bfloat16()),
                     (x, r, w, -1.0), (x, r, w, float("nan")), (x.cpu(), r, w), (x, r.cpu(), w),
                     (torch.zeros(1, 32769, device=DEV), None, torch.zeros(32769, device=DEV)),
                     (torch.zeros(3, 0, device=DEV), None, torch.zeros(0, device=DEV))):
            with pytest.raises(hmx.HmxError):
                f(*args)
    x.requires_grad_()
    y, _ = enc_ops.add_rmsnorm(x, r, w)
    g = torch.autograd.grad(y, x, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError):                   # no second derivative
        torch.autograd.grad(g.sum(), x)


def test_streams_and_graph():
    x, r, w, dy, ds = make(300, 128, torch.bfloat16, 17)
    want_y, want_s = enc_ops.add_rmsnorm(x, r, w)
    want_q = mx_ops.add_rmsnorm_mx8(x, r, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, s = enc_ops.add_rmsnorm(x, r, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want_y) and torch.equal(s, want_s)
    graph = torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(graph):
        y, s = enc_ops.add_rmsnorm(xs, r, w)
        codes, scales, _ = mx_ops.add_rmsnorm_mx8(xs, r, w)
    for k in range(3):
        xs.copy_(x if k != 1 else 2 * x)
        graph.replay()
        torch.cuda.synchronize()
        ey, es = enc_ops.add_rmsnorm(xs, r, w)
        ec, esc, _ = mx_ops.add_rmsnorm_mx8(xs, r, w)
        assert torch.equal(y, ey) and torch.equal(s, es) and torch.equal(scales, esc)
        assert torch.equal(codes.view(torch.uint8), ec.view(torch.uint8))
    assert torch.equal(want_q[1], scales)
