"""Root-mean-square norm with the residual's addition, its gradients and its 8-bit output, against 64 bits.

Tolerances: a row's sum of squares is a chain of at most 32 additions per thread, 5 shuffles and 32 warps, 70
roundings of 2^-24 relative that the square root halves; rsqrtf is within 2 ulp (4 roundings) and two products follow:
below 48 * 2^-24, plus half a step of the output's type.  In the backward the mean over the row has the same chain
(100 roundings with its factors); column sums have at most one rounding per row, plus those of the joining kernel
(16 + 8 unrolled chains, below 60)."""
import pytest
import torch

from lowp_ref import F8, TINY, floor, same_codes, unit

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (3, 7), (5, 47), (17, 128), (4, 172), (130, 256), (9, 1000), (33, 1024), (2, 2049), (7, 4096),
          (3, 5000), (2, 8191), (2, 8192), (2, 16384), (700, 100), (2500, 64), (33, 46), (5, 130), (300, 1002), (3, 1501), (2, 2050),
          (3, 6001), (2, 12002)]


def _inputs(rows, f, dtype, seed, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, f, device="cuda", generator=g) * torch.exp(torch.randn(rows, 1, device="cuda", generator=g))
    r = torch.randn(rows, f, device="cuda", generator=g)
    w = 1.0 + 0.3 * torch.randn(f, device="cuda", generator=g)
    gy, gh = (torch.randn(rows, f, device="cuda", generator=g).to(dtype) for _ in range(2))
    return x.to(dtype), r.to(dtype) if residual else None, w, gy, gh


def _check(x, r, w, gy, gh, y, h, gx, gw, eps):
    h64 = (x if r is None else (x.double() + r.double()).to(x.dtype)).double()
    if r is not None:
        assert torch.equal(h.double(), h64)
    rms = (h64.square().mean(1, keepdim=True) + eps).sqrt()
    hat, wd = h64 / rms, w.double()
    ref = hat * wd
    assert ((y.double() - ref).abs() <= (unit(y.dtype) + 48 * U) * ref.abs() + floor(y.dtype)).all()
    if gx is None:
        return
    a = gy.double() * wd
    c = (a * hat).mean(1, keepdim=True)
    want = (a - hat * c) / rms + (0 if gh is None else gh.double())
    room = (a.abs() + hat.abs() * (a * hat).abs().mean(1, keepdim=True)) / rms + (0 if gh is None else gh.double().abs())
    assert ((gx.double() - want).abs() <= unit(gx.dtype) * want.abs() + 100 * U * room + floor(gx.dtype)).all()
    want = (gy.double() * hat).sum(0)
    room = (gy.double() * hat).abs().sum(0)
    assert ((gw.double() - want).abs() <= unit(gw.dtype) * want.abs() + (x.size(0) + 100) * U * room + floor(gw.dtype)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,f", SHAPES)
def test_forward_and_gradients(rows, f, dtype):
    from gnn_benchmark_b200 import norm

    for residual in (True, False):
        x, r, w, gy, gh = _inputs(rows, f, dtype, rows * 31 + f, residual)
        w = w.to(dtype)
        leaves = [t.clone().requires_grad_(True) for t in (x, w)] + ([r.clone().requires_grad_(True)] if residual else [])
        out = norm.rms_norm(leaves[0], leaves[1], residual=leaves[2] if residual else None, eps=1e-5)
        if residual:
            gx, gw, gr = torch.autograd.grad(out, leaves, (gy, gh))
            assert torch.equal(gx, gr)
            y, h = out
        else:
            gx, gw = torch.autograd.grad(out, leaves, gy)
            y, h = out, None
        _check(x, r, w, gy, gh if residual else None, y, h, gx, gw, 1e-5)
        with torch.no_grad():
            again = norm.rms_norm(x, w, residual=r, eps=1e-5)
        again = again if residual else (again,)
        assert torch.equal(again[0], y) and (not residual or torch.equal(again[1], h))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp32_weight_with_16_bit_rows(dtype):
    from gnn_benchmark_b200 import norm

    x, r, w, gy, gh = _inputs(77, 300, dtype, 5)
    wl = w.clone().requires_grad_(True)
    xl = x.clone().requires_grad_(True)
    y, h = norm.rms_norm(xl, wl, residual=r)
    gx, gw = torch.autograd.grad((y, h), (xl, wl), (gy, gh))
    assert gw.dtype == torch.float32
    _check(x, r, w, gy, gh, y, h, gx, gw, 1e-6)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    """Rows inside a wider matrix at every offset, transposed and broadcast inputs.  The accesses that rows allow decide
    which thread has which column, so a row's sum is taken in another order: two results that are each within the bound
    of this file's head from the same exact value are within twice that bound of one another.  h has no sum and is
    equal."""
    from gnn_benchmark_b200 import norm

    x, r, w, gy, gh = _inputs(40, 200, dtype, 3)
    w = w.to(dtype)
    y, h = norm.rms_norm(x, w, residual=r)
    room = 2 * ((unit(dtype) + 48 * U) * y.double().abs() * (1 + 2.0 ** -7) + floor(dtype))

    def near(a, b, room):
        return ((a.double() - b.double()).abs() <= room).all()

    for off in (0, 1, 2, 4, 8):
        wide = torch.full((40, 220 if off == 2 else 219), float("nan"), device="cuda", dtype=dtype)
        wide[:, off:off + 200] = x
        y2, h2 = norm.rms_norm(wide[:, off:off + 200], w, residual=r)
        assert near(y2, y, room) and torch.equal(h2, h)
    y3, _ = norm.rms_norm(x.t().contiguous().t(), w, residual=r.t().contiguous().t())
    assert torch.equal(y3, y)
    one = x[:1].expand(40, 200)
    y4 = norm.rms_norm(one, w)
    assert torch.equal(y4, norm.rms_norm(x[:1], w).expand(40, 200))
    base = torch.zeros(40 * 200 + 1, device="cuda", dtype=dtype)  # gradients that start off a 16-byte boundary
    base[1:] = gy.reshape(-1)
    xl = x.clone().requires_grad_(True)
    out = norm.rms_norm(xl, w)
    a, = torch.autograd.grad(out, xl, base[1:].view(40, 200), retain_graph=True)
    b, = torch.autograd.grad(out, xl, gy, retain_graph=True)
    c, = torch.autograd.grad(out, xl, torch.ones((), device="cuda", dtype=dtype).expand(40, 200))
    rms = (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    hat, gw = x.double() / rms, (gy.double() * w.double()).abs()
    terms = (gw + hat.abs() * (gw * hat.abs()).mean(1, keepdim=True)) / rms
    assert near(a, b, 2 * (unit(dtype) * b.double().abs() * (1 + 2.0 ** -7) + 100 * U * terms + floor(dtype)))
    assert torch.isfinite(c).all()


def test_gradient_against_differences():
    """Directional derivative in fp32 against a central difference of the 64-bit formula."""
    from gnn_benchmark_b200 import norm

    x, r, w, gy, gh = _inputs(6, 130, torch.float32, 11)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, r)]
    y, h = norm.rms_norm(*leaves[:2], residual=leaves[2])
    grads = torch.autograd.grad((y, h), leaves, (gy, gh))
    g = torch.Generator(device="cuda").manual_seed(1)
    step = 1e-5
    for i, grad in enumerate(grads):
        d = torch.randn(grad.shape, device="cuda", generator=g, dtype=torch.float64)

        def f(s):
            a = [t.double() + (s * d if k == i else 0) for k, t in enumerate((x, w, r))]
            hh = a[0] + a[2]
            yy = hh / (hh.square().mean(1, keepdim=True) + 1e-6).sqrt() * a[1]
            return ((yy * gy).sum() + (hh * gh).sum()).item()

        want = (f(step) - f(-step)) / (2 * step)
        got = (grad.double() * d).sum().item()
        # the stream's rounding (2^-24 of h) and the kernel's own (100 * 2^-24) enter each term of the sum once
        room = 200 * U * (grad.double() * d).abs().sum().item() + 1e-6 * abs(want) + 1e-5
        assert abs(got - want) <= room


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,f", [(1, 1), (3, 47), (17, 128), (4, 129), (130, 256), (9, 1000), (7, 4096), (3, 5000), (2, 16384),
                                    (33, 46), (5, 130), (300, 1002), (3, 1501), (2, 2050), (3, 6001), (2, 12002)])
def test_fp8_output(rows, f, dtype):
    """Codes bit for bit (they depend on element-wise fp32 steps alone), scales within the norm's tolerance."""
    from gnn_benchmark_b200 import norm

    x, r, w, _, _ = _inputs(rows, f, dtype, rows + f)
    w = w.to(dtype)
    if rows > 2:
        x[1], r[1] = 0, 0           # a row of zeros
        x[2, :min(f, 128)], r[2, :min(f, 128)] = 0, 0   # a group of zeros
    codes, scales, h = norm.rms_norm_fp8(x, w, residual=r)
    assert codes.dtype == F8 and codes.shape == (rows, f) and scales.shape == (rows, (f + 127) // 128)
    hs = (x.double() + r.double()).to(dtype)
    assert torch.equal(h, hs)
    t = hs.float() * w.float()
    rms = (hs.double().square().mean(1) + 1e-6).sqrt()
    for j in range(scales.size(1)):
        part = t[:, 128 * j:128 * (j + 1)]
        a = part.abs().amax(1).clamp_min(TINY)
        assert same_codes(codes[:, 128 * j:128 * (j + 1)], (part * (torch.reciprocal(a) * 448.0)[:, None]).to(F8))
        want = a.double() / 448.0 / rms
        assert ((scales[:, j].double() - want).abs() <= 50 * U * want).all()
    plain = norm.rms_norm_fp8(hs, w)
    assert same_codes(plain[0], codes) and torch.equal(plain[1], scales)


def test_not_finite_rows_stay_their_own():
    from gnn_benchmark_b200 import norm

    x = torch.randn(6, 300, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(300, device="cuda", dtype=torch.bfloat16)
    good = norm.rms_norm(x, w)
    x[1, 5], x[4, 299] = float("nan"), float("inf")
    y = norm.rms_norm(x, w)
    assert torch.isnan(y[1]).all() and torch.isnan(y[4, 299])
    keep = [0, 2, 3, 5]
    assert torch.equal(y[keep], good[keep])
    codes, scales = norm.rms_norm_fp8(x, w)
    value = codes.float() * scales.repeat_interleave(128, 1)[:, :300]
    assert torch.isnan(value[1]).all() and torch.isfinite(value[keep]).all() and torch.isnan(value[4, 256:]).all()


def test_no_rows_and_unused_outputs():
    from gnn_benchmark_b200 import norm

    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    y = norm.rms_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 64) and torch.equal(w.grad, torch.zeros(64, device="cuda"))
    codes, scales = norm.rms_norm_fp8(x.detach(), w.detach())
    assert codes.shape == (0, 64) and scales.shape == (0, 1)
    a = torch.randn(5, 64, device="cuda", requires_grad=True)
    b = torch.randn(5, 64, device="cuda", requires_grad=True)
    _, h = norm.rms_norm(a, w, residual=b)
    g = torch.randn(5, 64, device="cuda")
    ga, gb = torch.autograd.grad(h, (a, b), g)
    assert torch.equal(ga, g) and torch.equal(gb, g)


def test_other_stream_and_captured_backward():
    """The same values on a side stream, and from a replayed graph of forward and backward (its leaves have no
    eager graph alive, as torch asks of captured backward passes)."""
    from gnn_benchmark_b200 import norm

    x, r, w, gy, gh = _inputs(200, 384, torch.bfloat16, 8)
    w = w.bfloat16()

    def both(leaves):
        y, h = norm.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        return [t.detach() for t in (y, h, *torch.autograd.grad((y, h), leaves, (gy, gh)))]

    def fresh():
        return [t.clone().requires_grad_(True) for t in (x, w, r)]

    want = both(fresh())
    leaves = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(leaves)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(leaves)
    with torch.no_grad():
        leaves[0].mul_(2.0)
        x.mul_(2.0)
    graph.replay()
    again = both(fresh())
    assert all(torch.equal(a, b) for a, b in zip(held, again))


def test_gpu_refusals():
    from gnn_benchmark_b200 import norm

    x = torch.randn(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    for bad in (lambda: norm.rms_norm(x.double(), w), lambda: norm.rms_norm(x, w[:32]),
                lambda: norm.rms_norm(x, w.half()), lambda: norm.rms_norm(x, w, residual=x[:3]),
                lambda: norm.rms_norm(x, w, residual=x.half()), lambda: norm.rms_norm(x[0], w),
                lambda: norm.rms_norm(torch.zeros(2, 16385, device="cuda"), torch.zeros(16385, device="cuda")),
                lambda: norm.rms_norm_fp8(x, w.clone().requires_grad_(True)),
                lambda: norm.rms_norm(x, w.cpu())):
        with pytest.raises(RuntimeError):
            bad()
