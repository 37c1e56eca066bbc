"""Refusals of the low-precision entry points, without a GPU: CPU tensors, and arguments that the C ABI turns into
status codes before anything is launched."""
import ctypes

import pytest
import torch


def test_wrappers_refuse_cpu_tensors(cuda_lib):
    from gnn_benchmark_b200 import dense, norm, optim

    x, w = torch.randn(8, 16), torch.ones(16)
    codes, scales = x.to(torch.float8_e4m3fn), torch.ones(8, 1)
    p = torch.nn.Parameter(torch.ones(4))
    p.grad = torch.ones(4)
    for call in (lambda: norm.rms_norm(x, w), lambda: norm.rms_norm_fp8(x, w), lambda: dense.quantize_fp8(x),
                 lambda: dense.matmul_fp8(codes, scales, codes, scales), lambda: dense.linear_fp8(x, x),
                 lambda: optim.AdamW([p]).step(), lambda: optim.adamw_step([x], [x], [x], [x], step=1, lr=1e-3)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_optimizer_arguments():
    from gnn_benchmark_b200 import optim

    p = [torch.nn.Parameter(torch.ones(4))]
    for kw in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(state_bits=16),
               dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            optim.AdamW(p, **kw)


def test_config_keys():
    from gnn_benchmark_b200 import model, optim

    config = dict(model_name="sage", in_channels=8, hidden_channels=8, out_channels=4, num_layers=2, dropout=0.0, num_bits=32,
                  is_pre_delay=False, lr=0.01, weight_decay=5e-4)
    assert type(model.create_model_and_optimizer(config)[1]) is torch.optim.Adam
    opt = model.create_model_and_optimizer(dict(config, optimizer="adamw", optimizer_state_bits=8))[1]
    assert type(opt) is optim.AdamW and opt.param_groups[0]["state_bits"] == 8 and opt.param_groups[0]["lr"] == 0.01
    with pytest.raises(ValueError):
        model.create_model_and_optimizer(dict(config, optimizer="sgd"))


def test_norm_status_codes(cuda_lib):
    f = cuda_lib.gnnagg_rms_norm_fwd

    def call(x=16, ldx=64, r=None, w=16, wt=0, rows=4, F=64, t=0, h=None, y=16, ldy=64):
        return f(x, ldx, r, 64, w, wt, rows, F, t, 1e-6, h, 64, y, ldy, None, None)

    assert call(t=3) == -1 and call(wt=1) == -1 and call(rows=-1) == -1 and call(F=0) == -1
    assert call(F=16385, ldx=16385, ldy=16385) == -2 and call(rows=1 << 31) == -2
    assert call(x=None) == -1 and call(y=None) == -1 and call(ldx=63) == -1 and call(ldy=63) == -1
    assert call(r=16) == -1 and call(h=16) == -1  # the residual and the sum's output come together
    assert call(rows=0) == 0
    g = cuda_lib.gnnagg_rms_norm_fp8
    assert g(16, 64, None, 0, 16, 0, 4, 64, 0, 1e-6, None, 0, 16, 72, 16, 4, None) == -2  # code rows off 16 bytes
    assert g(16, 64, None, 0, 16, 0, 4, 64, 0, 1e-6, None, 0, 16, 64, 16, 3, None) == -1
    b = cuda_lib.gnnagg_rms_norm_bwd
    need = cuda_lib.gnnagg_rms_norm_partial_bytes(4, 64, 0)
    assert need > 0 and cuda_lib.gnnagg_rms_norm_partial_bytes(4, 64, 9) == 0
    assert b(16, 64, None, 0, 16, 64, 16, 16, 0, 4, 64, 0, 16, 64, 16, 16, need - 1, None) == -4
    assert b(16, 64, None, 0, 16, 64, 16, 16, 0, 4, 64, 0, 16, 64, None, 16, need, None) == -1


def test_product_status_codes(cuda_lib):
    f = cuda_lib.gnnagg_fp8_matmul

    def call(A=16, lda=256, sa=16, a_block=1, B=16, ldb=256, b_block=128, M=300, N=200, K=256, acc=0, C=16, ldc=200, t=1,
             ws=None, nb=0, stride=1):
        return f(A, lda, sa, stride, 300, a_block, B, ldb, 16, 1, 2, b_block, M, N, K, None, 0, acc, C, ldc, t, ws, nb, None)

    assert call(M=-1) == -1 and call(a_block=64) == -1 and call(b_block=0) == -1 and call(t=5) == -1 and call(acc=2) == -1
    assert call(acc=1) == -2 and call(A=None) == -1 and call(C=None) == -1 and call(lda=255) == -1 and call(ldc=199) == -1
    assert call(lda=264) == -2 and call(A=24) == -2 and call(stride=-1) == -1 and call(M=(1 << 31) - 1, lda=256) == -2
    assert call(M=0) == 0 and call(N=0) == 0
    need = cuda_lib.gnnagg_fp8_matmul_workspace_bytes(40, 200, 20000)
    assert need > 0 and need % 16 == 0 and cuda_lib.gnnagg_fp8_matmul_workspace_bytes(100000, 256, 256) == 0
    assert call(M=40, N=200, K=20000, lda=20000, ldb=20000) == -4
    assert call(M=40, N=200, K=20000, lda=20000, ldb=20000, ws=16, nb=need - 1) == -4
    q = cuda_lib.gnnagg_fp8_quantize
    assert q(16, 64, 4, 64, 0, 2, 16, 64, 16, 4, None, 0, None, 0, None, None) == -1
    assert q(16, 64, 4, 64, 7, 1, 16, 64, 16, 4, None, 0, None, 0, None, None) == -1
    assert q(16, 64, 4, 64, 0, 1, None, 0, None, 0, None, 0, None, 0, None, None) == -1
    assert q(16, 63, 4, 64, 0, 1, 16, 64, 16, 4, None, 0, None, 0, None, None) == -1
    assert q(16, 64, 4, 64, 0, 1, 16, 72, 16, 4, None, 0, None, 0, None, None) == -2
    assert q(16, 64, 4, 64, 0, 1, 16, 64, 16, 3, None, 0, None, 0, None, None) == -1
    assert q(16, 64, 0, 64, 0, 1, None, 0, None, 0, None, 0, None, 0, None, None) == 0


def test_linear_status_codes(cuda_lib):
    kept, scratch = cuda_lib.gnnagg_fp8_linear_kept_bytes, cuda_lib.gnnagg_fp8_linear_scratch_bytes
    assert kept(100, 50, 60, 0, 0) == 0 and 0 < kept(100, 50, 60, 1, 0) < kept(100, 50, 60, 1, 1)
    assert scratch(100, 50, 60, 0) > 0 and scratch(100, 50, 60, 1) > 0 and kept(-1, 2, 3, 1, 1) == 0
    nb, sb = kept(100, 50, 60, 1, 1), scratch(100, 50, 60, 0)

    def fwd(M=100, kp=16, knb=nb, s=16, snb=sb, x=None):
        return cuda_lib.gnnagg_fp8_linear_fwd(x, 60, 0, 16, 60, 0, None, 0, M, 50, 60, 16, 0, 1, 1, kp, knb, s, snb, None)

    assert fwd(M=-1) == -1 and fwd(kp=None) == -4 and fwd(knb=nb - 1) == -4 and fwd(s=24) == -4 and fwd(snb=sb - 1) == -4
    assert fwd() == -1  # x is null
    b = cuda_lib.gnnagg_fp8_linear_bwd
    assert b(16, 50, 0, 100, 50, 60, 0, 1, 16, nb, 16, 0, None, 0, None, 0, 16, 1 << 30, None) == -1  # gx, nothing kept for it
    assert b(16, 50, 0, 100, 50, 60, 1, 1, 16, nb, 16, 0, None, 0, 16, 7, 16, 1 << 30, None) == -1
    assert b(16, 50, 0, 100, 50, 60, 1, 1, 16, nb - 1, 16, 0, None, 0, None, 0, 16, 1 << 30, None) == -4


def test_adamw_status_codes(cuda_lib):
    class _Tensor(ctypes.Structure):
        _fields_ = [(k, ctypes.c_void_p) for k in ("param", "grad", "exp_avg", "exp_avg_sq", "scales", "master")]
        _fields_ += [("n", ctypes.c_int64)]

    f = cuda_lib.gnnagg_adamw_step

    def call(rows, t=0, bits=32, b1=0.9, step=1, count=None):
        table = (_Tensor * max(len(rows), 1))(*rows)
        return f(table, len(rows) if count is None else count, t, bits, 1e-3, b1, 0.999, 1e-8, 0.0, step, None, None)

    good = (16, 16, 16, 16, None, None, 8)
    assert call([good], t=4) == -1 and call([good], bits=4) == -1 and call([good], b1=1.0) == -1 and call([good], step=0) == -1
    assert call([good], count=-1) == -1 and f(None, 1, 0, 32, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None) == -1
    for i in range(4):
        assert call([good[:i] + (None,) + good[i + 1:]]) == -1
    assert call([(16, 16, 16, 16, None, None, -1)]) == -1
    assert call([good], bits=8) == -1 and call([(16, 16, 16, 16, 12, None, 8)], bits=8) == -2
    assert call([]) == 0 and call([(None, None, None, None, None, None, 0)]) == 0  # nothing to do, nothing launched
    assert cuda_lib.gnnagg_adamw_tick(None, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, 16, None) == -1
    assert cuda_lib.gnnagg_adamw_tick(16, None, 1e-3, 1.0, 0.999, 1e-8, 0.0, 16, None) == -1


def test_missing_front_end_fails_loudly(cuda_lib, monkeypatch, tmp_path):
    from gnn_benchmark_b200 import _lib

    monkeypatch.setattr(_lib, "_ops", None)
    monkeypatch.setattr(_lib, "OPS_PATH", str(tmp_path / "nope.so"))
    with pytest.raises(RuntimeError, match="is missing"):
        _lib.ops()


def test_optimizer_refuses_shared_parameters_and_foreign_state():
    from gnn_benchmark_b200 import optim

    p = torch.nn.Parameter(torch.ones(4))
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="twice"):
        optim.AdamW([p, p])
    opt = optim.AdamW([p])
    with pytest.raises(ValueError, match="another optimiser"):
        opt.load_state_dict(torch.optim.AdamW([p]).state_dict())
    assert opt.param_groups[0]["state_bits"] == 32


def _recorded_optimizer(monkeypatch, n, **kw):
    """An AdamW over n CPU parameters whose launches are replaced: every update notes the count that it would use."""
    from gnn_benchmark_b200 import _lib, optim

    used = []

    def tick(group, device, step):
        step += 1
        return int(step)

    monkeypatch.setattr(_lib, "require_cuda", lambda *ts: None)
    monkeypatch.setattr(optim.AdamW, "_tick", staticmethod(tick))
    monkeypatch.setattr(optim.AdamW, "_update",
                        staticmethod(lambda group, members, step, scalars: used.extend((p, scalars or step) for p, _ in members)))
    ps = [torch.nn.Parameter(torch.ones(4)) for _ in range(n)]
    return ps, optim.AdamW(ps, **kw), used


def _stepped(ps, opt, used, which):
    """One step with gradients for the parameters of these numbers; the count that each of them used."""
    for i, p in enumerate(ps):
        p.grad = torch.ones(4) if i in which else None
    used.clear()
    opt.step()
    assert len(used) == len(which)
    return {next(i for i, q in enumerate(ps) if q is p): t for p, t in used}


@pytest.mark.parametrize("capturable", [False, True])
def test_a_step_without_a_gradient_is_not_counted(monkeypatch, capturable):
    ps, opt, used = _recorded_optimizer(monkeypatch, 3, capturable=capturable)
    own = [0, 0, 0]
    for _ in range(2):  # the second time from a state dict, in which equal counts are shared again
        for which in ((0, 1, 2), (0, 2), (0,), (0, 1, 2), (1,), (1, 2), (0, 1, 2)):
            for i in which:
                own[i] += 1
            assert _stepped(ps, opt, used, which) == {i: own[i] for i in which}
            assert [int(opt.state[p]["step"]) for p in ps] == own
        opt.load_state_dict(opt.state_dict())


def test_captured_steps_keep_their_counts(monkeypatch):
    ps, opt, used = _recorded_optimizer(monkeypatch, 2, capturable=True)
    _stepped(ps, opt, used, (0, 1))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):  # a count of its own would have to be made inside the graph
        _stepped(ps, opt, used, (0,))
    _stepped(ps, opt, used, (0, 1))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with pytest.raises(RuntimeError, match="captured step"):  # a replay would go on to count for both
        _stepped(ps, opt, used, (1,))
    counts = [int(opt.state[p]["step"]) for p in ps]
    assert counts[0] == counts[1]
    assert _stepped(ps, opt, used, (0, 1)) == {i: counts[0] + 1 for i in (0, 1)}
    opt.load_state_dict(opt.state_dict())  # other tensors than the graph's
    assert _stepped(ps, opt, used, (1,)) == {1: counts[0] + 2}


def test_counts_of_parameters_that_change_their_group(monkeypatch):
    ps, opt, used = _recorded_optimizer(monkeypatch, 2, capturable=True)
    _stepped(ps, opt, used, (0, 1))
    first = opt.param_groups[0]
    opt.param_groups.append(dict(first, params=[first["params"].pop()]))
    assert _stepped(ps, opt, used, (0, 1)) == {0: 2, 1: 2}
    assert _stepped(ps, opt, used, (0, 1)) == {0: 3, 1: 3}


def test_an_unknown_dense_mode_is_refused(monkeypatch, tmp_path):
    """A misspelt name must not turn the tensor-core kernels off without a word."""
    from gnn_benchmark_b200 import dense, train

    monkeypatch.setattr(dense, "MODE", dense.MODE)  # put back at the end
    for mode in dense.MODES:
        dense.set_mode(mode)
        assert dense.MODE == mode and dense.enabled() == (mode != "cublas")
    for mode in ("FP8", "fp16", "", None, 8):
        with pytest.raises(ValueError, match="unknown dense mode"):
            dense.set_mode(mode)
    path = tmp_path / "config.yaml"
    path.write_text("dense_mode: tf32\n")
    monkeypatch.setattr("sys.argv", ["train", "--config", str(path)])
    with pytest.raises(ValueError, match="unknown dense mode 'tf32'"):
        train.main()


def test_a_refused_capture_leaves_no_trace(monkeypatch):
    """Counts of a step whose capture is refused are not those of a captured step."""
    ps, opt, used = _recorded_optimizer(monkeypatch, 4, capturable=True)
    _stepped(ps, opt, used, (0, 1))
    _stepped(ps, opt, used, (2, 3))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        _stepped(ps, opt, used, (0, 1, 2))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert _stepped(ps, opt, used, (0, 2)) == {0: 2, 2: 2}
    assert _stepped(ps, opt, used, (0, 1, 2, 3)) == {0: 3, 1: 2, 2: 3, 3: 2}
