"""AdamW over many tensors: against 64 bits (32-bit moments) and bit for bit in the 8-bit moments' codes.

Tolerance of one step from given 32-bit moments: m and v take three roundings of 2^-24 and a rounded constant each,
below 5 * 2^-24 of the terms' sum; the update's quotient takes the root, two products, a sum, a quotient and its
rounded scalars on top, below 16 * 2^-24 of the update; the decay and the difference 3 * 2^-24 of the parameter."""
import math

import pytest
import torch

from lowp_ref import F8, floor, moments_from_blocks, moments_to_blocks, same_codes, unit

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
B1, B2, EPS = 0.9, 0.999, 1e-8
SIZES = [1, 3, 255, 256, 257, 2048, 2049, 0, 5000, 64 * 47, 100003]


def _reference(p, g, m, v, t, lr, wd):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    nm, nv = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    upd = lr / (1 - B1 ** t) * nm / (nv.sqrt() / math.sqrt(1 - B2 ** t) + EPS)
    room_m, room_v = 5 * U * (B1 * m.abs() + (1 - B1) * g.abs()), 5 * U * nv
    # an error of m reaches the update with m's own factor
    room_p = 16 * U * upd.abs() + room_m * (lr / (1 - B1 ** t)) / (nv.sqrt() / math.sqrt(1 - B2 ** t) + EPS) + 3 * U * p.abs()
    return p * (1 - lr * wd) - upd, nm, nv, room_p, room_m, room_v


def _tensors(sizes, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = [torch.randn(n, device="cuda", generator=g).to(dtype) for n in sizes]
    gr = [(1e-2 * torch.randn(n, device="cuda", generator=g)).to(dtype) for n in sizes]
    m = [1e-3 * torch.randn(n, device="cuda", generator=g) for n in sizes]
    v = [(1e-2 * torch.randn(n, device="cuda", generator=g)).square() for n in sizes]
    return p, gr, m, v


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [1, 2, 1000])
def test_step_32(dtype, step):
    from gnn_benchmark_b200 import optim

    p, g, m, v = _tensors(SIZES, dtype, step)
    want = [_reference(*x, step, 1e-2, 0.1) for x in zip(p, g, m, v)]
    optim.adamw_step(p, g, m, v, step=step, lr=1e-2, betas=(B1, B2), eps=EPS, weight_decay=0.1)
    for i, (wp, wm, wv, rp, rm, rv) in enumerate(want):
        assert ((m[i].double() - wm).abs() <= rm).all() and ((v[i].double() - wv).abs() <= rv + 1e-44).all()
        assert ((p[i].double() - wp).abs() <= rp + unit(dtype) * wp.abs() + floor(dtype)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_8_bit_exact(dtype):
    """Three steps in a row: the moments' codes and scales are the definition's, the parameters follow from them."""
    from gnn_benchmark_b200 import optim

    sizes = SIZES + [1 << 16]
    p, g, m, v = _tensors(sizes, dtype, 4)
    g[2][:] = 0                      # an untouched tensor
    g[4][::3] *= 1e-4                # elements far below their block's largest
    m[2].zero_(), v[2].zero_()
    packed = [moments_to_blocks(a, b) for a, b in zip(m, v)]
    mc, vc, sc = ([x[i].clone() for x in packed] for i in range(3))
    for step in (7, 8, 9):
        old = [t.clone() for t in p]
        parts = [moments_from_blocks(*x) for x in zip(mc, vc, sc)]
        optim.adamw_step(p, g, mc, vc, step=step, lr=1e-2, betas=(B1, B2), eps=EPS, weight_decay=0.1, scales=sc)
        for i, (a, b) in enumerate(parts):
            wp, _, _, rp, _, _ = _reference(old[i], g[i], a, b, step, 1e-2, 0.1)
            assert ((p[i].double() - wp).abs() <= rp + unit(dtype) * wp.abs() + floor(dtype)).all()
            gf = g[i].float()
            nm, nv = a * B1 + gf * (1 - B1), b * B2 + (gf * gf) * (1 - B2)
            wm, wv, ws = moments_to_blocks(nm, nv)
            assert same_codes(mc[i], wm) and same_codes(vc[i], wv) and torch.equal(sc[i], ws)
            assert ((nv > 0) <= (vc[i].float() > 0)).all(), "a second moment vanished"


def test_unaligned_views_and_neighbours():
    """Tensors that start at any element of a buffer, and elements between them that are not theirs."""
    from gnn_benchmark_b200 import optim

    for bits in (32, 8):
        sizes, places = [5, 300, 1000, 2], [1, 7, 310, 1317]
        total = 1400
        src = _tensors(sizes, torch.float32, 9)
        packed = [moments_to_blocks(a, b) for a, b in zip(src[2], src[3])]
        states = [src[2], src[3]] if bits == 32 else [[x[0] for x in packed], [x[1] for x in packed]]
        flat = []
        for k, ts in enumerate([src[0], src[1], *states]):
            eight = k > 1 and bits == 8
            buf = torch.full((total,), 3.0, device="cuda").to(F8 if eight else torch.float32)
            views = [buf[at:at + n] for at, n in zip(places, sizes)]
            for d, s in zip(views, ts):
                d.copy_(s)
            flat.append((buf, views))
        sc = [x[2].clone() for x in packed] if bits == 8 else None
        sc2 = [x[2].clone() for x in packed] if bits == 8 else None
        a = [[t.clone() for t in ts] for ts in (src[0], src[1], *states)]
        optim.adamw_step(*a, step=3, lr=1e-2, scales=sc)
        optim.adamw_step(*[f[1] for f in flat], step=3, lr=1e-2, scales=sc2)
        mask = torch.ones(total, dtype=torch.bool)
        for at, n in zip(places, sizes):
            mask[at:at + n] = False
        for (buf, views), ts in zip(flat, a):
            assert all(torch.equal(x.float(), y.float()) for x, y in zip(views, ts))
            assert (buf.float()[mask.cuda()] == 3.0).all()


def test_more_tensors_than_a_table_holds():
    from gnn_benchmark_b200 import optim

    for count in (17, 61, 501, 1100):
        sizes = [(7 * i) % 300 for i in range(count)]
        p, g, m, v = _tensors(sizes, torch.float32, count)
        want = [_reference(*x, 2, 1e-3, 1e-2) for x in zip(p, g, m, v)]
        optim.adamw_step(p, g, m, v, step=2, lr=1e-3)
        for i, (wp, wm, wv, rp, rm, rv) in enumerate(want):
            assert ((p[i].double() - wp).abs() <= rp).all() and ((m[i].double() - wm).abs() <= rm).all()


def test_master_weights():
    from gnn_benchmark_b200 import optim

    p, g, m, v = _tensors([300, 1001], torch.bfloat16, 2)
    master = [t.float() + 1e-4 for t in p]
    want = [_reference(w, *x, 5, 1e-4, 0.0) for w, x in zip(master, zip(g, m, v))]
    optim.adamw_step(p, g, m, v, step=5, lr=1e-4, weight_decay=0.0, masters=[master[0], master[1]])
    for i in range(2):
        assert ((master[i].double() - want[i][0]).abs() <= want[i][3]).all()
        assert torch.equal(p[i], master[i].bfloat16())


def test_not_finite_gradient_stays_in_its_block():
    from gnn_benchmark_b200 import optim

    p, g, m, v = _tensors([1024], torch.float32, 3)
    g[0][300] = float("inf")
    mc, vc, sc = moments_to_blocks(m[0], v[0])
    optim.adamw_step(p, g, [mc], [vc], step=2, lr=1e-2, scales=[sc])
    a, b = moments_from_blocks(mc, vc, sc)
    block = torch.zeros(1024, dtype=torch.bool, device="cuda")
    block[256:512] = True
    assert torch.isnan(a[block]).all() and torch.isfinite(a[~block]).all() and torch.isfinite(p[0][~block]).all()


def _module(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(40, 33), torch.nn.ReLU(), torch.nn.Linear(33, 5)).to("cuda", dtype)


def _train(model, opt, steps, x):
    for _ in range(steps):
        opt.zero_grad()
        model(x).square().mean().backward()
        opt.step()


def test_optimizer_follows_torch():
    """Five steps of a small model next to torch.optim.AdamW in 64 bits."""
    from gnn_benchmark_b200 import optim

    x = torch.randn(64, 40, device="cuda")
    a, b = _module(), _module().double()
    opt = optim.AdamW(a.parameters(), lr=1e-2, weight_decay=0.1)
    ref = torch.optim.AdamW(b.parameters(), lr=1e-2, weight_decay=0.1)
    for _ in range(5):
        for m, o, inp in ((a, opt, x), (b, ref, x.double())):
            o.zero_grad()
            m(inp).square().mean().backward()
        for p, q in zip(a.parameters(), b.parameters()):
            q.grad.copy_(p.grad)  # the same gradients: what is compared is the optimiser
        opt.step()
        ref.step()
        for p, q in zip(a.parameters(), b.parameters()):
            # five updates of at most about lr each, 40 roundings a step
            assert ((p.double() - q).abs() <= 5 * 40 * U * (q.abs() + 1e-2)).all()
            with torch.no_grad():
                q.copy_(p)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict_round_trip(bits, capturable, dtype):
    from gnn_benchmark_b200 import optim

    x = torch.randn(64, 40, device="cuda", dtype=dtype)
    a, b = _module(dtype), _module(dtype)
    kw = dict(lr=1e-2, state_bits=bits, capturable=capturable, master_weights=True)
    oa, ob = optim.AdamW(a.parameters(), **kw), optim.AdamW(b.parameters(), **kw)
    _train(a, oa, 3, x)
    b.load_state_dict(a.state_dict())
    ob.load_state_dict(oa.state_dict())
    for p, q in zip(a.parameters(), b.parameters()):
        for k, v in oa.state[p].items():
            w = ob.state[q][k]
            if isinstance(v, torch.Tensor):
                assert w.dtype == v.dtype and torch.equal(w.float(), v.float())
                assert w.data_ptr() != v.data_ptr() or v.numel() == 0
            else:
                assert w == v
    _train(a, oa, 2, x)
    _train(b, ob, 2, x)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))


def test_captured_step_counts_and_follows_the_rate():
    """A replayed step is the eager one: the count advances on the device and the rate is read there.  Two graphs
    share nothing but the optimiser's own state."""
    from gnn_benchmark_b200 import optim

    a, b = _module(), _module()
    lr = torch.tensor(1e-2, device="cuda")
    oa = optim.AdamW(a.parameters(), lr=lr, capturable=True)
    ob = optim.AdamW(b.parameters(), lr=1e-2)
    g = torch.Generator(device="cuda").manual_seed(3)
    for p, q in zip(a.parameters(), b.parameters()):
        p.grad = torch.randn(p.shape, device="cuda", generator=g)
        q.grad = p.grad.clone()
    with pytest.raises(RuntimeError, match="one step before"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            oa.step()
    oa.step()
    ob.step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            oa.step()
        graphs.append(graph)
    for i, rate in enumerate((1e-2, 3e-3, 5e-2)):
        lr.fill_(rate)
        ob.param_groups[0]["lr"] = float(torch.tensor(rate))
        graphs[i % 2].replay()
        ob.step()
        assert int(oa.state[next(a.parameters())]["step"]) == i + 2
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ob.step()


def test_groups_types_and_late_parameters():
    """Mixed types in one group, a parameter without a gradient at first: its count starts later, in both modes."""
    from gnn_benchmark_b200 import optim

    for capturable in (False, True):
        g = torch.Generator(device="cuda").manual_seed(5)
        ps = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=g).to(d))
              for n, d in ((100, torch.float32), (70, torch.bfloat16), (50, torch.float32))]
        opt = optim.AdamW([{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "lr": 1e-3, "weight_decay": 0.0}],
                          capturable=capturable)
        grads = [torch.randn(p.shape, device="cuda", generator=g).to(p.dtype) for p in ps]
        want = []
        for i, p in enumerate(ps):
            z = torch.zeros(p.shape, device="cuda", dtype=torch.float64)
            first = 2 if i == 1 else 1
            w, m, v = p.detach().double(), z, z.clone()
            for t in range(first, 4):
                w, m, v, *_ = _reference(w, grads[i], m, v, t - first + 1, 1e-3 if i == 2 else 1e-2, 0.0 if i == 2 else 1e-2)
            want.append(w)
        for t in range(1, 4):
            for i, p in enumerate(ps):
                p.grad = None if i == 1 and t == 1 else grads[i].clone()
            opt.step()
        for p, w in zip(ps, want):
            assert ((p.double() - w).abs() <= 3 * (unit(p.dtype) * w.abs() + 40 * U * (w.abs() + 1e-2))).all()


def test_gpu_refusals():
    from gnn_benchmark_b200 import optim

    p, g, m, v = _tensors([10, 20], torch.float32, 1)
    kw = dict(step=1, lr=1e-3)
    for bad in (lambda: optim.adamw_step(p, g[:1], m, v, **kw), lambda: optim.adamw_step(p, g[::-1], m, v, **kw),
                lambda: optim.adamw_step(p, [t.half() for t in g], m, v, **kw),
                lambda: optim.adamw_step(p, g, [t.to(F8) for t in m], [t.to(F8) for t in v], **kw),
                lambda: optim.adamw_step(p, g, m, v, scales=[torch.ones(1, 2, device="cuda")] * 2, **kw),
                lambda: optim.adamw_step(p, g, m, v, step=0, lr=1e-3),
                lambda: optim.adamw_step(p, g, m, v, betas=(1.0, 0.9), **kw),
                lambda: optim.adamw_step(p, g, m, [t.cpu() for t in v], **kw),
                lambda: optim.adamw_step([t[::2] for t in p], [t[::2] for t in g], [t[::2] for t in m], [t[::2] for t in v], **kw),
                lambda: optim.adamw_step([t.double() for t in p], g, m, v, **kw),
                lambda: optim.adamw_step([t.cpu() for t in p], g, m, v, **kw)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_of_the_old_values_raises(bits):
    """A step is a write in place: a graph that kept the parameter from before must not go on with the new one."""
    from gnn_benchmark_b200 import optim

    p = torch.nn.Parameter(torch.randn(300, device="cuda"))
    opt = optim.AdamW([p], state_bits=bits)
    loss = p.square().sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    before = [t._version for t in opt.state[p].values() if isinstance(t, torch.Tensor)]
    opt.step()
    assert all(t._version > b for t, b in zip([t for t in opt.state[p].values() if isinstance(t, torch.Tensor)], before))
    with torch.inference_mode():  # tensors that keep no version
        p, g, m, v = _tensors([10], torch.float32, 3)
        optim.adamw_step(p, g, m, v, step=1, lr=1e-3)


def test_more_refusals():
    from gnn_benchmark_b200 import optim

    p, g, m, v = _tensors([12], torch.float32, 1)
    size = 32  # eight floats
    for scalars in (torch.zeros(size, dtype=torch.uint8), torch.zeros(size - 4, dtype=torch.uint8, device="cuda"),
                    torch.zeros(size // 4, device="cuda"), torch.zeros(2 * size, dtype=torch.uint8, device="cuda")[::2],
                    torch.zeros(size + 1, dtype=torch.uint8, device="cuda")[1:]):
        with pytest.raises(RuntimeError, match="device_scalars"):
            optim.adamw_step(p, g, m, v, step=1, lr=1e-3, device_scalars=scalars)
    square = [p[0].view(3, 4)]
    with pytest.raises(RuntimeError, match="shape"):  # a transposed gradient has as many elements
        optim.adamw_step(square, [g[0].view(4, 3)], m, v, step=1, lr=1e-3)


@pytest.mark.parametrize("capturable", [False, True])
def test_a_step_without_a_gradient_is_not_counted(capturable):
    """A parameter that has no gradient in the middle: its bias corrections are of the steps that it took, from there on
    and after a state dict's round trip, in both modes."""
    from gnn_benchmark_b200 import optim

    g = torch.Generator(device="cuda").manual_seed(6)
    ps = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=g)) for n in (100, 70, 300)]
    opt = optim.AdamW(ps, lr=1e-2, capturable=capturable)
    want = [(p.detach().double(), torch.zeros(p.shape, device="cuda", dtype=torch.float64),
             torch.zeros(p.shape, device="cuda", dtype=torch.float64)) for p in ps]
    own = [0, 0, 0]
    for t, which in enumerate(((0, 1, 2), (0, 2), (0,), (0, 1, 2), (1, 2), (0, 1, 2))):
        for i, p in enumerate(ps):
            p.grad = torch.randn(p.shape, device="cuda", generator=g) if i in which else None
            if i in which:
                own[i] += 1
                want[i] = _reference(want[i][0], p.grad, *want[i][1:], own[i], 1e-2, 1e-2)[:3]
        opt.step()
        if t == 3:
            other = optim.AdamW(ps, lr=1e-2, capturable=capturable)
            other.load_state_dict(opt.state_dict())
            opt = other
    assert [int(opt.state[p]["step"]) for p in ps] == own
    for p, (w, _, _) in zip(ps, want):
        # up to six updates of at most about three rates each, 40 roundings a step
        assert ((p.double() - w).abs() <= 6 * 40 * U * (w.abs() + 3e-2)).all()
