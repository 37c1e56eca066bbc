"""The low-precision operators together, as a model uses them: norm -> 8-bit operand -> product in inference, a
residual block trained with the 8-bit linear layer, the norm and AdamW, and the framework's own layers and training
entry with `dense.MODE = "fp8"` and the "adamw" optimiser.  Every stage is held to its definition in 64 bits, on the
values that the stage before it produced."""
import pytest
import torch

from lowp_ref import floor, quantise, unit, values

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _room(a64, b64):  # as derived in test_fp8_gpu.py
    return (4 * 33 * 2.0 ** -23 + ((a64.size(1) + 127) // 128 + 80) * U) * (a64.abs() @ b64.abs().t())


def _close(got, a, b, extra=0):
    ref = a @ b.t() + extra
    assert ((got.double() - ref).abs() <= _room(a, b) + (unit(got.dtype) + 2 * U) * ref.abs() + floor(got.dtype)).all()


@pytest.mark.parametrize("rows", [1, 5, 300])
def test_inference_block(rows):
    """A token's (or a batch's) way through a residual block: two normed 8-bit products, nothing else in between."""
    from gnn_benchmark_b200 import dense, norm

    torch.manual_seed(rows)
    f, wide = 384, 1000
    x = torch.randn(rows, f, device="cuda", dtype=torch.bfloat16)
    stream = torch.randn(rows, f, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(f, device="cuda").bfloat16() + 0.5
    w2 = torch.rand(wide, device="cuda").bfloat16() + 0.5
    up = dense.quantize_fp8(torch.randn(wide, f, device="cuda") / f ** 0.5, (128, 128))
    down = dense.quantize_fp8(torch.randn(f, wide, device="cuda") / wide ** 0.5, (128, 128))
    codes, scales, h = norm.rms_norm_fp8(x, w, residual=stream)
    a = dense.matmul_fp8(codes, scales, *up)
    _close(a, values(codes, scales), values(*up))
    codes2, scales2 = norm.rms_norm_fp8(a, w2)
    b = dense.matmul_fp8(codes2, scales2, *down)
    _close(b, values(codes2, scales2), values(*down))
    y, h2 = norm.rms_norm(b, w, residual=h)
    assert torch.equal(h2, (b.double() + h.double()).bfloat16())
    dense.check_status()


def test_train_block():
    """Gradients of norm and 8-bit layer chained through a residual block, then one AdamW step with 8-bit moments."""
    from gnn_benchmark_b200 import dense, norm, optim

    torch.manual_seed(3)
    rows, f, n = 700, 200, 130
    x = torch.randn(rows, f, device="cuda", requires_grad=True)
    res = torch.randn(rows, f, device="cuda", requires_grad=True)
    w = (torch.rand(f, device="cuda") + 0.5).requires_grad_(True)
    up = (torch.randn(n, f, device="cuda") / f ** 0.5).requires_grad_(True)
    bias = torch.randn(n, device="cuda", requires_grad=True)
    y, h = norm.rms_norm(x, w, residual=res)
    z = dense.linear_fp8(y, up, bias)
    for t in (y, h, z):
        t.retain_grad()
    (z.square().sum() + h.square().sum()).backward()
    dense.check_status()
    _close(z, values(*quantise(y)), values(*quantise(up, 128)), bias.double())
    assert torch.equal(z.grad, 2 * z) and torch.equal(h.grad, 2 * h)
    _close(y.grad, values(*quantise(z.grad)), values(*quantise(up.t(), 128)))
    _close(up.grad, values(*quantise(z.grad.t())), values(*quantise(y.t())))
    hd = h.double()
    rms = (hd.square().mean(1, keepdim=True) + 1e-6).sqrt()
    hat = hd / rms
    a = y.grad.double() * w.double()
    want = (a - hat * (a * hat).mean(1, keepdim=True)) / rms + h.grad.double()
    room = (a.abs() + hat.abs() * (a * hat).abs().mean(1, keepdim=True)) / rms + h.grad.double().abs()
    assert ((x.grad.double() - want).abs() <= 101 * U * room).all() and torch.equal(x.grad, res.grad)
    before = [t.detach().clone() for t in (w, up, bias)]
    opt = optim.AdamW([w, up, bias], lr=1e-2, weight_decay=0.1, state_bits=8)
    opt.step()
    for t, old in zip((w, up, bias), before):
        g = t.grad.double()
        # the first step: m / (1 - b1) = g and v / (1 - b2) = g^2, so the update is lr * g / (|g| + eps)
        want = old.double() * (1 - 1e-2 * 0.1) - 1e-2 * g / (g.abs() + 1e-8)
        assert ((t.double() - want).abs() <= 16 * U * 1e-2 + 3 * U * old.double().abs()).all()


def _graph(n=500, width=64):
    from gnn_benchmark_b200 import Communicator, Quantizer_for_all_procs, TimeRecorder, graphgen
    from gnn_benchmark_b200.data_manager.DataLoader import build_graph

    src, dst = graphgen.erdos_renyi_edges(n, 3000, seed=5, device="cuda")
    src, dst = graphgen.symmetrize(src, dst, n, self_loops=True)
    begin = graphgen.contiguous_partitions(n, 1)
    Communicator(32)
    Quantizer_for_all_procs(1, 32)
    TimeRecorder(3, 3)
    local, remote = graphgen.partition_edges(src, dst, begin, 0)
    return build_graph(local, remote, begin, 0, 1, width, 32, False, device="cuda"), src, dst


def test_gcn_layer_with_8_bit_transform(cuda_lib, monkeypatch):
    """DistGCNConv under MODE "fp8": transform first (24 > 8), so the layer is A (values(x) values(W)^T) + b."""
    from gnn_benchmark_b200 import dense
    from gnn_benchmark_b200.model import DistGCNConv

    monkeypatch.setattr(dense, "MODE", "fp8")
    n = 500
    graph, src, dst = _graph(n)
    torch.manual_seed(0)
    conv = DistGCNConv(24, 8, 32, False).cuda()
    conv.reset_parameters()
    x = torch.randn(n, 24, device="cuda", requires_grad=True)
    out = conv(graph, x, 0)
    g = torch.randn_like(out)
    out.backward(g)
    dense.check_status()
    A = torch.zeros(n, n, device="cuda", dtype=torch.float64)
    A[dst, src] = 1.0
    d = A.sum(1)
    A = A / torch.sqrt(d)[:, None] / torch.sqrt(d)[None, :]
    xq, wq = values(*quantise(x)), values(*quantise(conv.lin.weight, 128))
    ref = A @ (xq @ wq.t()) + conv.bias.detach().double()
    # the aggregation's own tolerance (fp32 sums of some tens of edges) on top of the product's
    assert torch.allclose(out.double(), ref, rtol=1e-5, atol=1e-5)
    gh = (A.t() @ g.double()).float()  # the gradient that reaches the transform, up to fp32 rounding of its codes' input
    coarse = values(*quantise(gh)) @ values(*quantise(conv.lin.weight.t(), 128)).t()
    # a code may flip where gh sits on a border: one step (2^-3 of an element at most) of one factor
    room = 2.0 ** -3 * (gh.double().abs().amax(1, keepdim=True) * conv.lin.weight.detach().double().abs().amax(0))
    assert ((x.grad.double() - coarse).abs() <= room + 1e-5).all()
    assert (x.grad.double() - coarse).abs().mean() <= 1e-3 * coarse.abs().mean()


@pytest.mark.parametrize("name", ["sage", "gcn"])
def test_training_entry(cuda_lib, monkeypatch, name):
    """The config keys end to end: three epochs run, the parameters move, the moments are 8-bit."""
    from gnn_benchmark_b200 import dense
    from gnn_benchmark_b200.model import create_model_and_optimizer, set_random_seed
    from gnn_benchmark_b200.train import train

    monkeypatch.setattr(dense, "MODE", "fp8")
    graph, _, _ = _graph()
    set_random_seed(1)
    config = dict(model_name=name, in_channels=47, hidden_channels=64, out_channels=7, num_layers=3, dropout=0.5, num_bits=32,
                  is_pre_delay=False, lr=0.01, weight_decay=5e-4, optimizer="adamw", optimizer_state_bits=8)
    model, opt = create_model_and_optimizer(config, torch.device("cuda"))
    old = [p.detach().clone() for p in model.parameters()]
    data = {"graph": graph, "nodes_features": torch.randn(500, 47, device="cuda"),
            "nodes_labels": torch.randint(0, 7, (500,), device="cuda"),
            "nodes_train_masks": torch.arange(300, device="cuda"), "nodes_valid_masks": torch.arange(300, 400, device="cuda"),
            "nodes_test_masks": torch.arange(400, 500, device="cuda")}
    losses, _ = train(model, data, opt, 3, 32, log=None)
    assert all(l == l and abs(l) < 100 for l in losses)
    assert all(not torch.equal(a, p) and torch.isfinite(p).all() for a, p in zip(old, model.parameters()))
    assert all(s["exp_avg"].dtype == torch.float8_e4m3fn for s in opt.state.values())


def test_captured_step_next_to_an_eager_graph():
    """A step captured while an eager graph of the same leaves lives is refused; without one it is captured and its
    replays go on from each other's parameters, as eager steps do."""
    from gnn_benchmark_b200 import dense, norm, optim

    torch.manual_seed(0)
    x = torch.randn(200, 256, device="cuda")
    start = [torch.rand(256, device="cuda") + 0.5, torch.randn(128, 256, device="cuda") / 16, torch.zeros(128, device="cuda")]

    def fresh():
        leaves = [torch.nn.Parameter(t.clone()) for t in start]
        return leaves, optim.AdamW(leaves, lr=1e-2, capturable=True)

    def loss_of(leaves):
        return dense.linear_fp8(norm.rms_norm(x, leaves[0]), leaves[1], leaves[2]).square().mean()

    def step(leaves, opt):
        for p in leaves:
            p.grad = None
        loss_of(leaves).backward()
        opt.step()

    for call in (lambda w, m, b: norm.rms_norm(x, w), lambda w, m, b: dense.linear_fp8(x, m, b)):
        leaves, _ = fresh()
        held = call(*leaves)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="default stream still holds"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call(*leaves).sum().backward()
        held.sum().backward()  # the eager graph is as it was

    eager, eager_opt = fresh()
    for _ in range(4):
        step(eager, eager_opt)
    leaves, opt = fresh()
    step(leaves, opt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(leaves, opt)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(leaves, eager):
        assert torch.equal(p, q)  # the same kernels on the same values, with sums in a fixed order
    dense.check_status()


@pytest.mark.parametrize("what", ["norm", "quantise", "product", "adamw"])
def test_offsets_past_32_bits(what):
    """Tensors of more than 2^31 elements: the last rows (for AdamW the last blocks) are what a call on them alone
    gives, bit for bit; the product's last rows are held to 64 bits."""
    from gnn_benchmark_b200 import dense, norm, optim

    torch.manual_seed(0)
    rows, f, tail = 131073 + 128, 16384, 130  # (2^17 + 129) * 2^14 elements
    if what in ("norm", "quantise"):
        x = torch.randn(rows, f, device="cuda", dtype=torch.bfloat16)
        assert x.numel() > 2 ** 31
        last = x[-tail:].clone()
    if what == "norm":
        w = torch.ones(f, device="cuda", requires_grad=True)
        x.requires_grad_()
        y = norm.rms_norm(x, w)
        assert torch.equal(y[-tail:], norm.rms_norm(last, w))
        y.backward(x.detach())
        last.requires_grad_()
        norm.rms_norm(last, w).backward(last.detach())
        assert torch.equal(x.grad[-tail:], last.grad)
        del y
        codes, scales = norm.rms_norm_fp8(x.detach(), w.detach())
        codes1, scales1 = norm.rms_norm_fp8(last.detach(), w.detach())
        assert torch.equal(codes[-tail:].view(torch.uint8), codes1.view(torch.uint8)) and torch.equal(scales[-tail:], scales1)
    elif what == "quantise":
        codes, scales = dense.quantize_fp8(x)
        codes1, scales1 = dense.quantize_fp8(last)
        assert torch.equal(codes[-tail:].view(torch.uint8), codes1.view(torch.uint8)) and torch.equal(scales[-tail:], scales1)
        codes, scales = dense.quantize_fp8(x, transpose=True)
        codes1, scales1 = dense.quantize_fp8(x[:, -tail:], transpose=True)  # rows of the transpose
        assert torch.equal(codes[-tail:].view(torch.uint8), codes1.view(torch.uint8)) and torch.equal(scales[-tail:], scales1)
    elif what == "product":
        a, b = dense.quantize_fp8(torch.randn(rows, 128, device="cuda")), dense.quantize_fp8(torch.randn(f, 128, device="cuda"))
        out = dense.matmul_fp8(*a, *b)
        assert out.numel() > 2 ** 31
        _close(out[-tail:], values(*a)[-tail:], values(*b))
    else:
        n, cut = 2 ** 31 + 77, 2 ** 31 - 512
        p, g = (torch.randn(n, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
        s = torch.zeros((n + 255) // 256, 2, device="cuda")
        p1, g1, m1, v1, s1 = p[cut:].clone(), g[cut:].clone(), m[cut:].clone(), v[cut:].clone(), s[cut // 256:].clone()
        optim.adamw_step([p], [g], [m], [v], scales=[s], step=1, lr=1e-2)
        optim.adamw_step([p1], [g1], [m1], [v1], scales=[s1], step=1, lr=1e-2)
        assert torch.equal(p[cut:], p1) and torch.equal(s[cut // 256:], s1)
        assert torch.equal(m[cut:].view(torch.uint8), m1.view(torch.uint8)) and torch.equal(v[cut:].view(torch.uint8), v1.view(torch.uint8))
    dense.check_status()


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """No operator hands over an output without the tangent that its input has; in a call that is no part of forward-mode
    differentiation, a tangent of the same tensor does not count."""
    from torch.autograd import forward_ad

    from gnn_benchmark_b200 import dense, norm

    x, w = torch.randn(40, 256, device="cuda"), torch.randn(50, 256, device="cuda")
    scale, bias, res = torch.ones(256, device="cuda"), torch.zeros(50, device="cuda"), torch.randn(40, 256, device="cuda")
    a, b = dense.quantize_fp8(x), dense.quantize_fp8(w)
    out = torch.zeros(40, 50, device="cuda")
    calls = {
        "rms_norm": (norm.rms_norm, [x, scale, res]),
        "rms_norm_fp8": (norm.rms_norm_fp8, [x, scale, res]),
        "linear_fp8": (dense.linear_fp8, [x, w, bias]),
        "matmul_fp8": (lambda sa, sb, bias, out: dense.matmul_fp8(a[0], sa, b[0], sb, bias, out), [a[1], b[1], bias, out]),
    }
    with torch.set_grad_enabled(grad):
        for name, (call, inputs) in calls.items():
            call(*inputs)
            for i, t in enumerate(inputs):
                with forward_ad.dual_level():
                    dual = forward_ad.make_dual(t, torch.ones_like(t))
                    with pytest.raises(RuntimeError, match=name + " has no forward-mode derivative"):
                        call(*inputs[:i], dual, *inputs[i + 1:])
                    call(*inputs[:i], forward_ad.unpack_dual(dual).primal, *inputs[i + 1:])
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.func.jvp(lambda x: norm.rms_norm(x, scale), (x,), (x,))


def test_product_refuses_codes_that_require_a_gradient():
    from gnn_benchmark_b200 import dense

    a, b = dense.quantize_fp8(torch.randn(30, 256, device="cuda")), dense.quantize_fp8(torch.randn(40, 256, device="cuda"))
    leaf = a[0].detach().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        dense.matmul_fp8(leaf, a[1], *b)
    with pytest.raises(RuntimeError, match="no gradient"):
        dense.matmul_fp8(*b, leaf, a[1])
    with torch.no_grad():
        assert torch.equal(dense.matmul_fp8(leaf, a[1], *b), dense.matmul_fp8(*a, *b))


def test_captured_gradients_beside_an_eager_graph():
    """What a captured pass does not compute does not keep it: the gradient of x alone, while an eager graph holds the
    weight.  What it does reach, it reaches through views and other operators too."""
    from gnn_benchmark_b200 import dense, norm

    x = torch.randn(16, 64, device="cuda", requires_grad=True)
    w, m = torch.ones(64, device="cuda", requires_grad=True), torch.randn(48, 64, device="cuda", requires_grad=True)
    gy, gz = torch.randn(16, 64, device="cuda"), torch.randn(16, 48, device="cuda")
    calls = [lambda: torch.autograd.grad(norm.rms_norm(x, w), [x], gy), lambda: torch.autograd.grad(dense.linear_fp8(x, m), [x], gz)]
    want = [call()[0] for call in calls]
    held = (w * 2).sum() + (m * 2).sum()
    torch.cuda.synchronize()
    for call, expected in zip(calls, want):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            (got,) = call()
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, expected)
    early = w * 1.0  # its node belongs to the default stream
    for call, message in ((lambda: torch.autograd.grad(norm.rms_norm(x, w.view(64)), [w], gy), "still holds"),
                          (lambda: torch.autograd.grad(dense.linear_fp8(x.detach(), m.view(48, 64)), [m], gz), "still holds"),
                          (lambda: norm.rms_norm(x, early).sum().backward(), "forward ran on the default stream")):
        with pytest.raises(RuntimeError, match=message):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    held.backward()
    assert torch.equal(w.grad, torch.full_like(w, 2.0))
