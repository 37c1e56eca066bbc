"""e4m3 quantisation (bit for bit against its definition) and the block-scaled product against 64 bits.

Tolerance of the product, with S = sum |a b| in 64 bits: within a block of 128 four MMAs add 32 products and the
running value each, and an MMA may lose a step of 2^-23 of the largest term per term it aligns: 4 * 33 * 2^-23 S.
The blocks' sum has one rounding of the joint scale, one per addition and those of the splits' joining: (blocks + 80)
* 2^-24 S.  Plus half a step of the output's type."""
import pytest
import torch

from lowp_ref import F8, floor, quantise, same_codes, unit, values

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _matrix(rows, cols, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(torch.randn(rows, 1, device="cuda", generator=g))
    return (x * torch.exp(torch.randn(1, cols, device="cuda", generator=g))).to(dtype)


def _room(a64, b64, kblocks):
    return (4 * 33 * 2.0 ** -23 + (kblocks + 80) * U) * (a64.abs() @ b64.abs().t())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 47), (128, 128), (129, 127), (260, 100), (77, 500), (300, 1030),
                                       (1000, 16), (15, 4096)])
@pytest.mark.parametrize("block", [(1, 128), (128, 128)])
def test_quantise_bit_exact(rows, cols, dtype, block):
    from gnn_benchmark_b200 import _lib, dense

    x = _matrix(rows, cols, rows + cols, dtype)
    if rows > 3:
        x[3] = 0
    for t in (False, True):
        codes, scales = dense.quantize_fp8(x, block, transpose=t)
        want_c, want_s = quantise(x.t() if t else x, block[0])
        assert codes.shape == want_c.shape and codes.stride(0) % 16 == 0 and codes.data_ptr() % 16 == 0
        assert same_codes(codes, want_c) and torch.equal(scales, want_s)
    pair = _lib.ops().quantize_fp8(x, block[0], True, True)  # both from one read
    for got, want in zip(pair, dense.quantize_fp8(x, block) + dense.quantize_fp8(x, block, transpose=True)):
        assert same_codes(got, want) if got.dtype == F8 else torch.equal(got, want)


def test_quantise_strides_and_extremes():
    from gnn_benchmark_b200 import dense

    x = _matrix(70, 300, 1, torch.bfloat16)
    want = dense.quantize_fp8(x)
    wide = torch.full((70, 317), float("nan"), device="cuda", dtype=torch.bfloat16)
    for off in (0, 1, 8):
        wide[:, off:off + 300] = x
        got = dense.quantize_fp8(wide[:, off:off + 300])
        assert same_codes(got[0], want[0]) and torch.equal(got[1], want[1])
        wide.fill_(float("nan"))
    got = dense.quantize_fp8(x.t().contiguous().t())
    assert same_codes(got[0], want[0])
    y = torch.zeros(6, 256, device="cuda")
    y[0, 3], y[1, 200], y[2, 0] = float("nan"), float("inf"), 3.0e38
    y[3, :] = 1e-45   # below the smallest block maximum: codes of zero
    y[4, 5] = -3.0e38
    codes, scales = dense.quantize_fp8(y)
    v = values(codes, scales)
    assert torch.isnan(v[0, :128]).all() and torch.isnan(v[1, 128:]).all()
    assert torch.isfinite(v[0, 128:]).all() and torch.isfinite(v[2:]).all() and (v[3] == 0).all()
    assert abs(v[2, 0].item() / 3.0e38 - 1) < 1e-6 and abs(v[4, 5].item() / -3.0e38 - 1) < 1e-6
    for rows, cols in ((0, 64), (64, 0), (0, 0)):
        c, s = dense.quantize_fp8(torch.zeros(rows, cols, device="cuda"))
        assert c.shape == (rows, cols) and s.shape == (rows, (cols + 127) // 128)


CASES = [  # m, n, k: one row, few rows (weight rows along the lanes), ragged edges of every tile width, long sums
    (1, 1, 1), (1, 128, 128), (1, 4096, 512), (7, 300, 1000), (16, 256, 4096), (17, 130, 200), (33, 1000, 640), (64, 64, 64),
    (65, 16, 128), (100, 17, 256), (128, 47, 100), (200, 100, 300), (300, 129, 1500), (257, 256, 129), (1000, 700, 260),
    (5003, 47, 100), (256, 256, 40000), (47, 100, 30001), (2500, 2048, 384), (20000, 256, 100), (3000, 1500, 1111),
    # a weight that stays in shared memory (one to three k-blocks, narrow and wide), clusters of two to eight splits with
    # 16, 32 and 64 columns, and splits too many or too large for a cluster
    (20000, 200, 384), (20000, 47, 300), (19000, 128, 128), (38000, 16, 129), (20, 500, 4000), (50, 500, 3000), (3, 200, 1100),
    (50, 500, 4000), (9, 130, 9000),
]


@pytest.mark.parametrize("m,n,k", CASES)
def test_product(m, n, k):
    from gnn_benchmark_b200 import dense

    a, b = _matrix(m, k, m + k), _matrix(n, k, n + 2 * k)
    bias = torch.randn(n, device="cuda")
    for i, (ab, bb) in enumerate([((1, 128), (128, 128)), ((1, 128), (1, 128)), ((128, 128), (1, 128)), ((128, 128), (128, 128))]):
        qa, qb = dense.quantize_fp8(a, ab), dense.quantize_fp8(b, bb)
        a64, b64 = values(*qa), values(*qb)
        ref = a64 @ b64.t()
        room = _room(a64, b64, (k + 127) // 128)
        dtype = TYPES[i % 3]
        out = dense.matmul_fp8(*qa, *qb, out_dtype=dtype)
        dense.check_status()
        assert out.shape == (m, n) and out.dtype == dtype
        big = torch.finfo(dtype).max
        ok = (out.double() - ref).abs() <= room + unit(dtype) * ref.abs() + floor(dtype)
        assert (ok | (ref.abs() > big)).all(), f"{(out.double() - ref).abs().max().item()}"
        out = dense.matmul_fp8(*qa, *qb, bias=bias, out_dtype=torch.float32)
        ref2 = ref + bias.double()
        assert ((out.double() - ref2).abs() <= room + 2 * U * (ref2.abs() + bias.double().abs())).all()
        again = dense.matmul_fp8(*qa, *qb, bias=bias, out_dtype=torch.float32)
        assert torch.equal(out, again)


def test_strided_output_and_accumulate():
    from gnn_benchmark_b200 import dense

    for m, n, k in ((300, 200, 256), (5, 200, 3000), (40, 30, 20000)):
        qa, qb = dense.quantize_fp8(_matrix(m, k, 1)), dense.quantize_fp8(_matrix(n, k, 2), (128, 128))
        want = dense.matmul_fp8(*qa, *qb, out_dtype=torch.float32)
        for off, width in ((0, n + 8), (1, n + 3), (4, n + 4)):
            for dtype in TYPES:
                wide = torch.full((m, width + off), 7.0, device="cuda", dtype=dtype)
                got = dense.matmul_fp8(*qa, *qb, out=wide[:, off:off + n])
                assert got.data_ptr() == wide[:, off:].data_ptr()
                assert torch.equal(wide[:, off:off + n], want.to(dtype))
                wide[:, off:off + n] = 7.0
                assert (wide == 7.0).all(), "wrote outside its columns"
        base = torch.randn(m, n, device="cuda")
        out = base.clone()
        dense.matmul_fp8(*qa, *qb, out=out, accumulate=True)
        assert ((out.double() - (base.double() + want.double())).abs() <= U * out.double().abs() + U * want.double().abs()).all()
    dense.check_status()


def test_scale_layouts_and_operand_views():
    """Scales of any strides, operands that are row slices and column slices at 16 bytes, one row of any stride."""
    from gnn_benchmark_b200 import dense

    a, b = _matrix(300, 512, 3), _matrix(200, 512, 4)
    qa, qb = dense.quantize_fp8(a), dense.quantize_fp8(b)
    want = dense.matmul_fp8(*qa, *qb, out_dtype=torch.float32)
    got = dense.matmul_fp8(qa[0], qa[1].contiguous(), qb[0], qb[1].contiguous(), out_dtype=torch.float32)
    assert torch.equal(got, want)
    got = dense.matmul_fp8(qa[0][64:200], qa[1][64:200], *qb, out_dtype=torch.float32)
    assert torch.equal(got, want[64:200])
    one = torch.ones(1, 1, device="cuda").expand(300, 4)
    got = dense.matmul_fp8(qa[0], one, *qb, out_dtype=torch.float32)
    same = dense.matmul_fp8(qa[0], one.contiguous(), *qb, out_dtype=torch.float32)
    assert torch.equal(got, same)
    half = dense.matmul_fp8(qa[0][:, 128:], qa[1][:, 1:], qb[0][:, 128:], qb[1][:, 1:], out_dtype=torch.float32)
    a64, b64 = values(qa[0][:, 128:], qa[1][:, 1:]), values(qb[0][:, 128:], qb[1][:, 1:])
    assert ((half.double() - a64 @ b64.t()).abs() <= _room(a64, b64, 3)).all()
    row = dense.matmul_fp8(qa[0][5:6].contiguous()[:, :500], qa[1][5:6], qb[0][:, :500], qb[1], out_dtype=torch.float32)
    a64, b64 = values(qa[0][5:6, :500], qa[1][5:6]), values(qb[0][:, :500], qb[1])
    assert ((row.double() - a64 @ b64.t()).abs() <= _room(a64, b64, 4)).all()
    dense.check_status()


def test_empty_products():
    from gnn_benchmark_b200 import dense

    def op(rows, cols):
        return dense.quantize_fp8(torch.ones(rows, cols, device="cuda"))

    assert dense.matmul_fp8(*op(0, 64), *op(5, 64)).shape == (0, 5)
    assert dense.matmul_fp8(*op(5, 64), *op(0, 64)).shape == (5, 0)
    bias = torch.randn(7, device="cuda")
    assert torch.equal(dense.matmul_fp8(*op(5, 0), *op(7, 0), bias=bias, out_dtype=torch.float32), bias.expand(5, 7))


def test_not_finite_rows_stay_their_own():
    from gnn_benchmark_b200 import dense

    a, b = _matrix(150, 300, 5), _matrix(140, 300, 6)
    good = dense.matmul_fp8(*dense.quantize_fp8(a), *dense.quantize_fp8(b), out_dtype=torch.float32)
    a[3, 7], a[140, 299], b[9, 0] = float("nan"), float("inf"), float("nan")
    out = dense.matmul_fp8(*dense.quantize_fp8(a), *dense.quantize_fp8(b), out_dtype=torch.float32)
    assert torch.isnan(out[3]).all() and torch.isnan(out[140]).all() and torch.isnan(out[:, 9]).all()
    rows = [i for i in range(150) if i not in (3, 140)]
    cols = [i for i in range(140) if i != 9]
    assert torch.equal(out[rows][:, cols], good[rows][:, cols])


def test_two_streams_and_captured_graphs():
    """Calls that split their sum hold a workspace each: two at once on two streams, two captured graphs replayed in
    either order."""
    from gnn_benchmark_b200 import dense

    ops = [(dense.quantize_fp8(_matrix(40, 20000, i)), dense.quantize_fp8(_matrix(200, 20000, i + 5))) for i in range(2)]
    want = [dense.matmul_fp8(*a, *b, out_dtype=torch.float32) for a, b in ops]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(dense.matmul_fp8(*ops[i][0], *ops[i][1], out_dtype=torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])
    graphs, held = [], []
    for a, b in ops:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(dense.matmul_fp8(*a, *b, out_dtype=torch.float32))
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for t in held:
            t.fill_(-1.0)
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(held[i], want[i]) for i in range(2))
    dense.check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(5003, 100, 47), (300, 256, 256), (1, 64, 130), (129, 1000, 17), (777, 47, 300)])
def test_linear_and_gradients(m, k, n, dtype):
    """Output and gradients are the 64-bit products of the definition's codes."""
    from gnn_benchmark_b200 import dense

    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = _matrix(m, k, 1, dtype)
    w = (torch.randn(n, k, device="cuda", generator=g) / k ** 0.5).to(dtype)
    b = torch.randn(n, device="cuda", generator=g).to(dtype)
    gy = torch.randn(m, n, device="cuda", generator=g).to(dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = dense.linear_fp8(*leaves)
    gx, gw, gb = torch.autograd.grad(y, leaves, gy)
    dense.check_status()

    def close(got, a, bb, extra=0):
        a, bb = values(*a), values(*bb)
        ref = a @ bb.t() + extra
        room = _room(a, bb, (a.size(1) + 127) // 128) + unit(got.dtype) * ref.abs() + floor(got.dtype) + 2 * U * ref.abs()
        assert ((got.double() - ref).abs() <= room).all()

    close(y, quantise(x), quantise(w, 128), b.double())
    close(gx, quantise(gy), quantise(w.t(), 128))
    close(gw, quantise(gy.t()), quantise(x.t()))
    ref = gy.double().sum(0)
    assert ((gb.double() - ref).abs() <= unit(dtype) * ref.abs() + (m + 2) * U * gy.double().abs().sum(0) + floor(dtype)).all()
    only_w = leaves[1].detach().clone().requires_grad_(True)
    y2 = dense.linear_fp8(x, only_w)
    gw2, = torch.autograd.grad(y2, only_w, gy)
    assert torch.equal(gw2, gw)
    only_x = x.clone().requires_grad_(True)
    gx2, = torch.autograd.grad(dense.linear_fp8(only_x, w), only_x, gy)
    assert torch.equal(gx2, gx)


def test_linear_without_rows_and_broadcast_gradient():
    from gnn_benchmark_b200 import dense

    w = torch.randn(30, 50, device="cuda", requires_grad=True)
    b = torch.randn(30, device="cuda", requires_grad=True)
    x = torch.zeros(0, 50, device="cuda", requires_grad=True)
    y = dense.linear_fp8(x, w, b)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 30) and gx.shape == (0, 50) and not gw.any() and not gb.any()
    x = torch.randn(20, 50, device="cuda", requires_grad=True)
    y = dense.linear_fp8(x, w, b)
    a = torch.autograd.grad(y.sum(), (x, w, b), retain_graph=True)
    c = torch.autograd.grad(y, (x, w, b), torch.ones(20, 30, device="cuda"))
    assert all(torch.equal(s, t) for s, t in zip(a, c))


@pytest.mark.parametrize("m,n,k", [(300, 200, 256), (300, 100, 256), (20000, 200, 200), (5, 2000, 4096), (40, 200, 20000),
                                   (1500, 2000, 14801)])
def test_bounded_wait_gives_up_and_reports(m, n, k):
    """A launch that waits for bytes which never come returns by itself, leaves its code, and the next is right: wide and
    narrow tiles, a weight that stays, a cluster, splits through the workspace, a shared last round."""
    from gnn_benchmark_b200 import _lib, dense

    lib = _lib.lib()
    qa, qb = dense.quantize_fp8(_matrix(m, k, 1)), dense.quantize_fp8(_matrix(n, k, 2), (128, 128))
    want = dense.matmul_fp8(*qa, *qb)
    dense.check_status()
    _lib.check(lib.gnnagg_dense_stall_test(16, 3000), "stall_test")
    try:
        dense.matmul_fp8(*qa, *qb)
        torch.cuda.synchronize()
    finally:
        _lib.check(lib.gnnagg_dense_stall_test(0, 0), "stall_test")
    with pytest.raises(RuntimeError, match=r"reported status"):
        dense.check_status()
    dense.clear_status()
    dense.check_status()
    assert torch.equal(dense.matmul_fp8(*qa, *qb), want)
    dense.check_status()


def test_gpu_refusals():
    from gnn_benchmark_b200 import dense

    a, sa = dense.quantize_fp8(torch.randn(300, 256, device="cuda"))
    b, sb = dense.quantize_fp8(torch.randn(40, 256, device="cuda"))
    out = torch.zeros(300, 40, device="cuda", dtype=torch.bfloat16)
    for bad in (lambda: dense.matmul_fp8(a, sa[:, :1], b, sb), lambda: dense.matmul_fp8(a, sa[:7], b, sb),
                lambda: dense.matmul_fp8(a[:, :128], sa[:, :1], b, sb), lambda: dense.matmul_fp8(a.float(), sa, b, sb),
                lambda: dense.matmul_fp8(a, sa.double(), b, sb), lambda: dense.matmul_fp8(a[:, 1:129], sa[:, :1], b[:, :128], sb[:, :1]),
                lambda: dense.matmul_fp8(a, sa, b, sb, accumulate=True),
                lambda: dense.matmul_fp8(a, sa, b, sb, out=out, accumulate=True),
                lambda: dense.matmul_fp8(a, sa, b, sb, out=out[:, :39]),
                lambda: dense.matmul_fp8(a, sa, b, sb, bias=torch.zeros(39, device="cuda")),
                lambda: dense.matmul_fp8(a, sa, b, sb, bias=torch.zeros(40, device="cuda").double()),
                lambda: dense.matmul_fp8(a, sa, b, sb, out_dtype=torch.float64), lambda: dense.matmul_fp8(a, sa.cpu(), b, sb),
                lambda: dense.quantize_fp8(torch.zeros(4, 4, 4, device="cuda")), lambda: dense.quantize_fp8(out.double()),
                lambda: dense.quantize_fp8(out, (1, 64)), lambda: dense.linear_fp8(out, out[:, :39])):
        with pytest.raises(RuntimeError):
            bad()


def test_graph_of_an_output_written_over_raises():
    from gnn_benchmark_b200 import dense

    a, b = dense.quantize_fp8(torch.randn(30, 256, device="cuda")), dense.quantize_fp8(torch.randn(40, 256, device="cuda"))
    leaf, out = torch.ones(30, 40, device="cuda", requires_grad=True), torch.ones(30, 40, device="cuda")
    loss = (leaf * out).sum()
    dense.matmul_fp8(*a, *b, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_product_refuses_to_drop_a_gradient():
    from gnn_benchmark_b200 import dense

    a, b = dense.quantize_fp8(torch.randn(30, 256, device="cuda")), dense.quantize_fp8(torch.randn(40, 256, device="cuda"))
    bias = torch.zeros(40, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        dense.matmul_fp8(*a, *b, bias=bias)
    with pytest.raises(RuntimeError, match="no gradient"):
        dense.matmul_fp8(*a, *b, out=torch.zeros(30, 40, device="cuda", requires_grad=True))
    with torch.no_grad():
        assert torch.equal(dense.matmul_fp8(*a, *b, bias=bias), dense.matmul_fp8(*a, *b))


@pytest.mark.parametrize("n", [185, 322, 567, 1001])
@pytest.mark.parametrize("m,k", [(300, 200), (70, 9000)])
def test_columns_behind_an_odd_width_stay(m, n, k):
    """A row of the output that ends between two 16-byte steps, inside aligned wider rows: what follows is left alone."""
    from gnn_benchmark_b200 import dense

    qa, qb = dense.quantize_fp8(_matrix(m, k, 1)), dense.quantize_fp8(_matrix(n, k, 2), (128, 128))
    for dtype in TYPES:
        want = dense.matmul_fp8(*qa, *qb, out_dtype=dtype)
        for off in (0, 8):
            wide = torch.full((m, (n + 8 + off) // 8 * 8), 7.0, device="cuda", dtype=dtype)
            dense.matmul_fp8(*qa, *qb, out=wide[:, off:off + n])
            assert torch.equal(wide[:, off:off + n], want)
            wide[:, off:off + n] = 7.0
            assert (wide == 7.0).all()
    dense.check_status()


@pytest.mark.parametrize("m,n,k", [(1500, 2000, 14801), (2000, 2600, 6400), (19000, 200, 5900), (18950, 100, 5910),
                                   (18955, 10, 5950), (19100, 300, 5900), (4096, 4096, 9600)])
def test_shared_last_round(m, n, k):
    """Fewer tiles in the last round than SMs: their blocks are shared out, and the parts joined in one order."""
    from gnn_benchmark_b200 import dense

    qa = dense.quantize_fp8(_matrix(m, k, 1))
    a64, bias = values(*qa), torch.randn(n, device="cuda")
    for block in ((1, 128), (128, 128)):
        qb = dense.quantize_fp8(_matrix(n, k, 2), block)
        b64 = values(*qb)
        ref = a64 @ b64.t() + bias.double()
        room = _room(a64, b64, (k + 127) // 128) + 2 * U * (ref.abs() + bias.double().abs())
        for dtype in TYPES:
            out = dense.matmul_fp8(*qa, *qb, bias=bias, out_dtype=dtype)
            ok = (out.double() - ref).abs() <= room + unit(dtype) * ref.abs() + floor(dtype)
            # as in test_product: sums reach 1e6 here, and what is above 65504 has no fp16 value to be near to
            assert (ok | (ref.abs() > torch.finfo(dtype).max)).all()
            for _ in range(3):
                assert torch.equal(dense.matmul_fp8(*qa, *qb, bias=bias, out_dtype=dtype), out)
        base = torch.randn(m, n + 3, device="cuda")
        got = base.clone()
        dense.matmul_fp8(*qa, *qb, bias=bias, out=got[:, 1:n + 1], accumulate=True)
        want = ref + base[:, 1:n + 1].double()
        assert ((got[:, 1:n + 1].double() - want).abs() <= room + 3 * U * (want.abs() + base[:, 1:n + 1].double().abs() + ref.abs())).all()
        assert torch.equal(got[:, 0], base[:, 0]) and torch.equal(got[:, n + 1:], base[:, n + 1:])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = dense.matmul_fp8(*qa, *qb, bias=bias, out_dtype=torch.float16)
    for _ in range(2):
        held.zero_()
        graph.replay()
        assert torch.equal(held, dense.matmul_fp8(*qa, *qb, bias=bias, out_dtype=torch.float16))
    dense.check_status()


def test_shared_rounds_on_two_streams():
    from gnn_benchmark_b200 import dense

    ops = [(dense.quantize_fp8(_matrix(m, k, i)), dense.quantize_fp8(_matrix(n, k, i + 5), (128, 128)))
           for i, (m, n, k) in enumerate([(2000, 2600, 6400), (1500, 2000, 14801)])]
    want = [dense.matmul_fp8(*a, *b, out_dtype=torch.float32) for a, b in ops]
    streams = [torch.cuda.Stream() for _ in ops]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(dense.matmul_fp8(*ops[i][0], *ops[i][1], out_dtype=torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)
    dense.check_status()


@pytest.mark.parametrize("m,n,k", [(300, 260, 9000), (5, 2000, 4100), (129, 16, 1290)])
@pytest.mark.parametrize("block", [(1, 128), (128, 128)])
def test_scales_brought_in_4_bytes(m, n, k, block):
    """Scales that lie row by row are copied element by element, by other lanes than those that read them: the same bits
    as from scales that lie column by column, at every one of many blocks."""
    from gnn_benchmark_b200 import dense

    qa, qb = dense.quantize_fp8(_matrix(m, k, 1)), dense.quantize_fp8(_matrix(n, k, 2), block)
    want = dense.matmul_fp8(*qa, *qb, out_dtype=torch.float32)
    sa, sb = qa[1].contiguous(), qb[1].contiguous()
    assert sa.stride(1) == 1 and torch.equal(sa, qa[1])
    for _ in range(20):
        assert torch.equal(dense.matmul_fp8(qa[0], sa, qb[0], sb, out_dtype=torch.float32), want)
    dense.check_status()


@pytest.mark.parametrize("m,n,k", [(301, 190, 700), (6, 1000, 2100), (130, 20, 300)])
@pytest.mark.parametrize("first", [1, 2, 3])
def test_scales_whose_columns_start_off_16_bytes(m, n, k, first):
    """Columns of scales cut out of a matrix of odd column stride: some start on 16 bytes and are copied in such pieces, the
    first one does not.  The tile's last rows have no scale."""
    from gnn_benchmark_b200 import dense

    def cut(scales):
        rows, cols = scales.shape
        wide = torch.full((cols + 4, (rows + 3) // 4 * 4 + 1), float("nan"), device="cuda")
        wide[first:first + cols, :rows] = scales.t()
        view = wide[first:first + cols, :rows].t()
        assert view.stride(0) == 1 and view.stride(1) % 2 == 1 and view.data_ptr() % 16 != 0
        return view

    qa, qb = dense.quantize_fp8(_matrix(m, k, 1)), dense.quantize_fp8(_matrix(n, k, 2))
    want = dense.matmul_fp8(*qa, *qb, out_dtype=torch.float32)
    assert torch.equal(dense.matmul_fp8(qa[0], cut(qa[1]), qb[0], cut(qb[1]), out_dtype=torch.float32), want)
    dense.check_status()


def test_a_long_sum_gives_up_at_once():
    """After a wait has run out (3 ms here) the blocks that are left are not waited for one by one: a tile of 2048 blocks
    ends as soon as one of two."""
    from gnn_benchmark_b200 import _lib, dense

    m, n, k = 149 * 128, 16, 2048 * 128  # a tile for every SM and one more: nothing is split
    a, b = torch.zeros(m, k, device="cuda", dtype=torch.uint8).view(F8), torch.zeros(n, k, device="cuda", dtype=torch.uint8).view(F8)
    sa, sb = torch.ones(149, 2048, device="cuda"), torch.ones(1, 2048, device="cuda")
    lib = _lib.lib()
    dense.matmul_fp8(a, sa, b, sb)
    dense.check_status()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    _lib.check(lib.gnnagg_dense_stall_test(16, 3000), "stall_test")
    try:
        begin.record()
        dense.matmul_fp8(a, sa, b, sb)
        end.record()
        torch.cuda.synchronize()
    finally:
        _lib.check(lib.gnnagg_dense_stall_test(0, 0), "stall_test")
    with pytest.raises(RuntimeError, match=r"reported status"):
        dense.check_status()
    dense.clear_status()
    took = begin.elapsed_time(end)
    assert took < 50.0, f"{took:.1f} ms"
    assert not dense.matmul_fp8(a, sa, b, sb).any()
    dense.check_status()
