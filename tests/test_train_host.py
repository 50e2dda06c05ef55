"""Training operators, what needs no GPU: refusals at the C entries (all checked before any device is touched), workspace
sizes, shapes without data, the optimiser's bookkeeping."""
import ctypes
import math

import pytest
import torch

from fused_swiglu_b200 import capi, train

NAN, INF = float("nan"), float("inf")


def address(a, at=0):
    return ctypes.c_void_p(ctypes.addressof(a) + at)


@pytest.fixture()
def memory():
    a = (ctypes.c_uint8 * 8192)()
    start = -ctypes.addressof(a) % 256
    return lambda at=0: address(a, start + at)


BF, F32 = capi.OUT_BF16, capi.OUT_F32


def layer_forward(m, **other):
    a = dict(x=m(), ldx=8, w=m(), b=m(), y=m(1024), ldy=8, mean=m(2048), rstd=m(3072), M=2, d=8, xt=BF, wt=BF, eps=1e-5)
    a.update(other)
    return capi.lib.fswiglu_layer_norm_forward(*a.values(), None)


@pytest.mark.parametrize("status,other", [
    (capi.ERR_BAD_ARG, dict(x=None)), (capi.ERR_BAD_ARG, dict(y=None)), (capi.ERR_BAD_ARG, dict(mean=None)),
    (capi.ERR_BAD_ARG, dict(rstd=None)), (capi.ERR_BAD_ARG, dict(M=-1)), (capi.ERR_BAD_ARG, dict(d=0)),
    (capi.ERR_BAD_ARG, dict(xt=2)), (capi.ERR_BAD_ARG, dict(wt=-1)), (capi.ERR_BAD_ARG, dict(eps=-1e-5)),
    (capi.ERR_BAD_ARG, dict(eps=NAN)), (capi.ERR_SHAPE, dict(ldx=7)), (capi.ERR_SHAPE, dict(ldy=7)),
    (capi.ERR_SHAPE, dict(d=(1 << 24) + 1, ldx=1 << 25, ldy=1 << 25)), (capi.ERR_SHAPE, dict(M=1 << 31)),
    (capi.OK, dict(M=0, x=None, y=None))], ids=str)
def test_layer_norm_forward_refusals(memory, status, other):
    assert layer_forward(memory, **other) == status


def test_norm_forward_refuses_elements_off_their_boundary(memory):
    assert layer_forward(memory, x=memory(1)) == capi.ERR_ALIGNMENT
    assert layer_forward(memory, w=memory(1)) == capi.ERR_ALIGNMENT
    assert layer_forward(memory, rstd=memory(3074)) == capi.ERR_ALIGNMENT


def layer_backward(m, **other):
    a = dict(dy=m(), ldd=8, x=m(), ldx=8, mean=m(), rstd=m(), w=m(), res=None, ldr=0, dx=m(1024), ld_dx=8, dw=m(2048),
             db=m(2560), M=2, d=8, xt=BF, wt=BF, gt=BF, ws=m(4096), bytes=2048)
    a.update(other)
    return capi.lib.fswiglu_layer_norm_backward(*a.values(), None)


@pytest.mark.parametrize("status,other", [
    (capi.ERR_BAD_ARG, dict(dy=None)), (capi.ERR_BAD_ARG, dict(x=None)), (capi.ERR_BAD_ARG, dict(mean=None)),
    (capi.ERR_BAD_ARG, dict(rstd=None)), (capi.ERR_BAD_ARG, dict(dx=None)), (capi.ERR_BAD_ARG, dict(gt=5)),
    (capi.ERR_SHAPE, dict(ldd=7)), (capi.ERR_SHAPE, dict(ld_dx=1)), (capi.ERR_WORKSPACE, dict(ws=None)),
    (capi.ERR_WORKSPACE, dict(bytes=127)), (capi.ERR_BAD_ARG, dict(M=-2)), (capi.ERR_BAD_ARG, dict(d=-8))], ids=str)
def test_layer_norm_backward_refusals(memory, status, other):
    assert layer_backward(memory, **other) == status
    assert layer_backward(memory, ws=memory(4100)) == capi.ERR_WORKSPACE
    assert layer_backward(memory, res=memory(), ldr=4) == capi.ERR_SHAPE


def test_norm_workspace_is_host_arithmetic():
    assert capi.lib.fswiglu_norm_backward_workspace_bytes(0, 4096) == 0
    assert capi.lib.fswiglu_norm_backward_workspace_bytes(1, 8) >= 64
    big = capi.lib.fswiglu_norm_backward_workspace_bytes(1 << 30, 4096)
    assert 2 * 4096 * 4 <= big <= 1 << 24  # does not grow with the rows
    assert capi.lib.fswiglu_grad_norm_workspace_bytes() >= 256


def test_norm_rows_are_read_inside_their_matrix(tmp_path):
    """What the norms copy of rows that start anywhere is plain integer code (csrc/row_granules.h): compile the checker with g++ and
    run it over alignments, widths, pitches and row counts."""
    import os
    import subprocess

    here = os.path.dirname(os.path.abspath(__file__))
    exe, src = tmp_path / "check_row_granules", os.path.join(here, "native", "check_row_granules.cpp")
    inc = os.path.join(here, "..", "fused-swiglu_b200", "csrc")
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{inc}", src, "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.startswith("ok "), res.stdout[-400:]


def adamw(m, tensors=None, pt=BF, gt=BF, bits=32, count=None, **options):
    plain = dict(param=m(), grad=m(1024), exp_avg=m(2048), exp_avg_sq=m(3072), numel=64)
    tensors = [plain] if tensors is None else [{**plain, **t} for t in tensors]
    table = (capi.AdamWTensor * max(1, len(tensors)))(*(capi.AdamWTensor(**t) for t in tensors))
    o = capi.AdamWOptions(**{**dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, step=1), **options})
    return capi.lib.fswiglu_adamw_step(table, len(tensors) if count is None else count, pt, gt, bits, ctypes.byref(o), None)


@pytest.mark.parametrize("options", [
    dict(lr=-1e-3), dict(lr=NAN), dict(lr=INF), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(beta2=NAN), dict(eps=-1.0),
    dict(eps=INF), dict(weight_decay=-0.1), dict(weight_decay=NAN), dict(step=0), dict(step=-5), dict(pt=2), dict(gt=7),
    dict(bits=16), dict(count=-1), dict(bits=8)], ids=str)
def test_adamw_refuses_options(memory, options):
    assert adamw(memory, **options) == capi.ERR_BAD_ARG


def test_adamw_refuses_tensors(memory):
    m = memory
    for key in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert adamw(m, [{key: None}]) == capi.ERR_BAD_ARG
    assert adamw(m, [dict(numel=-1)]) == capi.ERR_BAD_ARG
    assert adamw(m, [dict(numel=(1 << 35) + 1)]) == capi.ERR_SHAPE
    assert adamw(m, [dict(param=m(1))]) == capi.ERR_ALIGNMENT
    assert adamw(m, [dict(exp_avg=m(2050))]) == capi.ERR_ALIGNMENT
    assert adamw(m, [dict(master=m(4096))], pt=F32, gt=F32) == capi.ERR_BAD_ARG
    assert adamw(m, [], count=0) == capi.OK
    assert adamw(m, [dict(numel=0, param=None)]) == capi.OK  # nothing to do


def test_adamw_refuses_shared_memory_in_any_order(memory):
    m = memory
    apart = [dict(param=m(128 * i), exp_avg=m(2048 + 256 * i), exp_avg_sq=m(5000 + 256 * i)) for i in range(3)]
    for order in ([0, 1, 2], [2, 1, 0], [1, 2, 0]):
        for key, size in (("param", 128), ("exp_avg", 256), ("exp_avg_sq", 256)):
            tensors = [dict(apart[i]) for i in order]
            tensors[-1][key] = ctypes.c_void_p(tensors[0][key].value + size - 8)
            assert adamw(m, tensors) == capi.ERR_BAD_ARG
    shared = [dict(t, master=m(7000)) for t in apart[:2]]
    assert adamw(m, shared) == capi.ERR_BAD_ARG
    for key in ("exp_avg_scale", "exp_avg_sq_scale"):
        scales = [dict(t, exp_avg_scale=m(7000 + 16 * i), exp_avg_sq_scale=m(7200 + 16 * i)) for i, t in enumerate(apart)]
        scales[2][key] = scales[0][key]
        assert adamw(m, scales, bits=8) == capi.ERR_BAD_ARG


def test_grad_norm_refusals(memory):
    m = memory
    size = capi.lib.fswiglu_grad_norm_workspace_bytes()
    ws = (ctypes.c_uint8 * (size + 256))()
    at = address(ws, -ctypes.addressof(ws) % 256)

    def call(tensors, max_norm=1.0, out=m(64), ws=at, bytes_=size):
        table = (capi.GradTensor * max(1, len(tensors)))(*(capi.GradTensor(*t) for t in tensors))
        return capi.lib.fswiglu_grad_norm_clip(table, len(tensors), max_norm, out, ws, bytes_, None)

    good = (m(1024).value, 8, BF)
    assert call([good], out=None) == capi.ERR_BAD_ARG
    assert call([good], max_norm=-1.0) == call([good], max_norm=NAN) == capi.ERR_BAD_ARG
    assert call([(None, 8, BF)]) == call([(good[0], -1, BF)]) == call([(good[0], 8, 3)]) == capi.ERR_BAD_ARG
    assert call([(good[0] + 2, 8, F32)]) == capi.ERR_ALIGNMENT
    assert call([good], ws=None) == call([good], bytes_=size - 1) == capi.ERR_WORKSPACE


def test_operators_refuse_host_tensors():
    import fused_mlp_module as lib

    x, s = torch.zeros((2, 8), dtype=torch.bfloat16), torch.zeros(2)
    for call in (lambda: lib.layer_norm_forward(x), lambda: lib.rms_norm_forward(x), lambda: lib.layer_norm_backward(x, x, s, s),
                 lambda: lib.rms_norm_backward(x, x, s), lambda: lib.adamw_step([x], [x], [x.float()], [x.float()], 1, 1e-3),
                 lambda: lib.grad_norm_clip([x], 1.0)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_operators_refuse_tensors_without_data():
    """A fake tensor calls itself a CUDA tensor, and its address is its offset from nothing: a view's would reach the GPU."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import fused_mlp_module as lib

    with FakeTensorMode():
        bf = dict(dtype=torch.bfloat16, device="cuda")
        x, s, w, mats = torch.empty((6, 64), **bf)[1:], torch.empty(9, device="cuda")[4:], torch.empty(72, **bf)[8:], torch.empty((65, 64), **bf)[1:]
        f = torch.empty((6, 64), device="cuda")[1:]
        for call in (lambda: lib.layer_norm_forward(x, w, w), lambda: lib.rms_norm_forward(x),
                     lambda: lib.layer_norm_backward(x, x, s, s, w), lambda: lib.rms_norm_backward(x, x, s),
                     lambda: lib.adamw_step([x], [x], [f], [f], 1, 1e-3), lambda: lib.grad_norm_clip([f, x], 1.0),
                     lambda: lib.rms_scale(x), lambda: lib.fused_swiglu_mlp_bf16(x, mats, mats, mats),
                     lambda: lib.swiglu_down_bf16(x, mats), lambda: lib.fused_swiglu_bf16(x, mats)):
            with pytest.raises(RuntimeError, match="has no data"):
                call()


def test_host_layer_refuses_tensors_without_data():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from fused_swiglu_b200 import ops

    with FakeTensorMode():
        bf = dict(dtype=torch.bfloat16, device="cuda")
        x, mats, wd = torch.empty((6, 64), **bf)[1:], torch.empty((65, 64), **bf)[1:], torch.empty((65, 64), **bf)[1:]
        for call in (lambda: ops.rms_scale(x), lambda: ops.fused_swiglu_gateup_bf16(x, mats, mats), lambda: ops.swiglu_down_bf16(x, wd),
                     lambda: ops.fused_swiglu_mlp_bf16(x, mats, mats, wd), lambda: ops.swiglu_mlp_backward(x, mats, mats, wd, x)):
            with pytest.raises(RuntimeError, match="has no data"):
                call()


def test_shapes_without_data():
    import fused_mlp_module  # noqa: F401

    o = torch.ops.ASMLLM
    x = torch.empty((6, 40), dtype=torch.bfloat16, device="meta")
    w = torch.empty(40, device="meta")
    y, mean, rstd = o.layer_norm_forward(x, w, w)
    assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == rstd.shape == (6,) and mean.dtype == torch.float32
    dx, dw, db = o.layer_norm_backward(x, x, mean, rstd, w, True)
    assert dx.dtype == x.dtype and dw.shape == db.shape == (40,) and dw.dtype == torch.float32
    y, rstd = o.rms_norm_forward(x, w)
    dx, dw = o.rms_norm_backward(x, x, rstd, w)
    assert dx.shape == x.shape and dw.shape == (40,)
    assert o.grad_norm_clip([x, w], 1.0).shape == (2,)
    assert o.adamw_step([w], [w], [w], [w], 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, [], [], []) is None


def test_norms_can_be_traced():
    """Shapes under fake tensors and on the meta device, both passes, and torch.compile without a graph break: on a CPU-only machine
    the captured graph fails at run time, with the dispatcher's missing CPU kernel and nothing else."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty((3, 9, 64), dtype=torch.bfloat16, device="cuda")[:, 1:]
        w = torch.empty(64, device="cuda")
        for y in (train.rms_norm(x, w), train.layer_norm(x, w, w), train.layer_norm(x)):
            assert y.shape == x.shape and y.dtype == x.dtype and y.device.type == "cuda"
        with pytest.raises(RuntimeError, match="has no data"):
            train.norm_swiglu_block(x, None, None, x[0], x[0], x[0])
    x, w = torch.empty((3, 8, 64), device="meta", requires_grad=True), torch.empty(64, device="meta", requires_grad=True)
    train.layer_norm(train.rms_norm(x, w), w, w).sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    if torch.cuda.is_available():
        pytest.skip("compiled with real tensors by the GPU suite")
    x, w = torch.zeros((2, 3, 64), requires_grad=True), torch.ones(64, requires_grad=True)
    for call in (lambda: torch.compile(train.rms_norm, fullgraph=True, backend="aot_eager")(x, w),
                 lambda: torch.compile(train.layer_norm, fullgraph=True, backend="aot_eager")(x, w, w)):
        torch._dynamo.reset()
        with pytest.raises(NotImplementedError, match="'CPU' backend"):
            call()


def test_a_dispatch_mode_alone_is_no_tracing():
    """Counters of operations and selective checkpointing watch what real tensors do: the block is called as without them."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with Watch(), pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        train.norm_swiglu_block(x, None, None, x, x, x)


# ---------------------------------------------------------------- the optimiser, with the operators recorded

class Recorder:
    def __init__(self):
        self.steps, self.norms = [], 0

    def adamw_step(self, params, grads, m, v, step, lr, b1, b2, eps, decay, masters, ms, vs, scale, seed, lr_t, step_t):
        self.steps.append(dict(params=params, m=m, v=v, step=step, lr=lr, masters=masters, ms=ms, vs=vs, scale=scale, seed=seed,
                               step_t=None if step_t is None else int(step_t)))
        for t in m + v + masters:
            t.view(torch.uint8).fill_(len(self.steps))

    def grad_norm_clip(self, grads, max_norm):
        self.norms += 1
        return torch.tensor([2.0, 0.5])


@pytest.fixture()
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(train, "_lib", lambda: r)
    return r


def some_params():
    ps = [torch.nn.Parameter(torch.ones(n, dtype=t)) for n, t in ((300, torch.bfloat16), (7, torch.float32), (512, torch.bfloat16))]
    for p in ps:
        p.grad = torch.ones_like(p)
    return ps


def test_optimizer_makes_one_call_for_tensors_of_a_kind(recorder):
    ps = some_params()
    opt = train.FusedAdamW(ps, lr=0.5, max_grad_norm=1.0)
    opt.step()
    assert [len(s["params"]) for s in recorder.steps] == [2, 1] and recorder.norms == 1
    assert [len(s["masters"]) for s in recorder.steps] == [2, 0]
    assert all(s["step"] == 1 and s["lr"] == 0.5 and float(s["scale"]) == 0.5 for s in recorder.steps)
    assert len({s["seed"] for s in recorder.steps}) == 2
    ps[0].grad = None  # takes no part: its own count stays behind
    opt.step()
    ps[0].grad = torch.ones_like(ps[0])
    opt.step()
    last = recorder.steps[-3:]
    assert sorted((s["params"][0].numel(), s["step"]) for s in last) == [(7, 3), (300, 2), (512, 3)]


def test_optimizer_keeps_the_types_of_its_state_over_a_checkpoint(recorder):
    for bits in (32, 8):
        ps = some_params()
        opt = train.FusedAdamW(ps, state_bits=bits)
        opt.step()
        opt.step()
        saved = opt.state_dict()
        other = train.FusedAdamW(some_params(), state_bits=bits)
        other.load_state_dict(saved)
        for p, q in zip(ps, other.param_groups[0]["params"]):
            a, b = opt.state[p], other.state[q]
            assert a["step"] == b["step"] == 2 and set(a) == set(b)
            for key in a:
                if isinstance(a[key], torch.Tensor):
                    assert a[key].dtype == b[key].dtype and a[key].data_ptr() != b[key].data_ptr()
                    assert torch.equal(a[key].view(torch.uint8), b[key].view(torch.uint8))
        assert ("exp_avg_scale" in opt.state[ps[0]]) == (bits == 8)
        assert opt.state[ps[0]]["exp_avg"].dtype == (torch.float8_e4m3fn if bits == 8 else torch.float32)


def test_optimizer_takes_its_step_count_over_a_checkpoint_either_way(recorder):
    ps = some_params()
    opt = train.FusedAdamW(ps, capturable=True)
    for _ in range(3):
        opt.step()
    for capturable in (False, True):
        other = train.FusedAdamW(some_params(), capturable=capturable)
        other.load_state_dict(opt.state_dict())
        recorder.steps.clear()
        other.step()
        assert len(recorder.steps) == 2
        assert all((s["step_t"] if capturable else s["step"]) == 4 for s in recorder.steps)
        assert ("step_tensor" in other.param_groups[0]) == capturable == ("lr_tensor" in other.param_groups[0])
    plain = train.FusedAdamW(some_params())
    plain.step()
    other = train.FusedAdamW(some_params(), capturable=True)
    other.load_state_dict(plain.state_dict())
    recorder.steps.clear()
    other.step()
    assert [s["step_t"] for s in recorder.steps] == [2, 2]


def test_optimizer_with_its_step_on_the_device_refuses_who_joins_or_skips(recorder):
    """One count serves the whole group: a parameter of fewer steps would get the bias corrections of another's."""
    def refused(opt):
        recorder.steps.clear()
        with pytest.raises(RuntimeError, match="every step together"):
            opt.step()
        assert not recorder.steps

    for late in range(3):
        ps = some_params()
        joins, grad = ps[late], ps[late].grad
        joins.grad = None
        opt = train.FusedAdamW(ps, capturable=True)
        for _ in range(5):
            opt.step()
        count = int(opt.param_groups[0]["step_tensor"])
        joins.grad = grad
        refused(opt)
        assert int(opt.param_groups[0]["step_tensor"]) == count == 5 and joins not in opt.state
        joins.grad = None
        opt.step()  # as before
        other_params = some_params()
        other = train.FusedAdamW(other_params, capturable=True)
        other.load_state_dict(opt.state_dict())
        refused(other)  # the checkpoint knows who has taken part
        other_params[late].grad = None
        other.step()
        assert int(other.param_groups[0]["step_tensor"]) == 7
    ps = some_params()
    opt = train.FusedAdamW(ps, capturable=True)
    opt.step()
    ps[1].grad = None
    refused(opt)
    for p in ps:
        p.grad = None
    opt.step()  # nobody: no step
    assert int(opt.param_groups[0]["step_tensor"]) == 1
    frozen = [{"params": some_params()[:1]}, {"params": some_params()[2:]}]
    opt = train.FusedAdamW(frozen, capturable=True)
    opt.step()
    opt.param_groups[0]["params"][0].grad = None  # groups have counts of their own
    opt.step()
    assert [int(g["step_tensor"]) for g in opt.param_groups] == [1, 2]


def test_optimizer_with_its_step_on_the_host_is_not_captured(recorder, monkeypatch):
    """A replay would take the captured step's number, learning rate and random bits over and over."""
    ps = some_params()
    opt, other = train.FusedAdamW(ps, max_grad_norm=1.0), train.FusedAdamW(some_params(), capturable=True)
    for o in (opt, other):
        o.step()
    recorder.steps.clear()
    recorder.norms = 0
    monkeypatch.setattr(train, "_capturing", lambda device: True)
    with pytest.raises(RuntimeError, match="capturable=True"):
        opt.step()
    assert not recorder.steps and recorder.norms == 0 and opt.state[ps[0]]["step"] == 1
    other.step()
    assert len(recorder.steps) == 2


def test_optimizer_checkpoint_of_other_kinds(recorder):
    for saved_bits, bits in ((8, 32), (32, 8)):
        opt = train.FusedAdamW(some_params(), state_bits=saved_bits)
        opt.step()
        with pytest.raises(ValueError, match="state_bits"):
            train.FusedAdamW(some_params(), state_bits=bits).load_state_dict(opt.state_dict())
    for saved_master, master in ((False, True), (True, False)):
        opt = train.FusedAdamW(some_params(), master=saved_master)
        opt.step()
        other = train.FusedAdamW(some_params(), master=master)
        other.load_state_dict(opt.state_dict())
        recorder.steps.clear()
        other.step()
        assert [len(s["masters"]) for s in recorder.steps] == [2 if master else 0, 0]


@pytest.mark.parametrize("how", ["deepcopy", "save", "copy"])
def test_optimizer_copies_are_whole(recorder, how):
    import copy
    import io

    ps = some_params()
    opt = train.FusedAdamW(ps, lr=0.5, state_bits=8, master=False, max_grad_norm=2.0, seed=9)
    opt.step()
    if how == "save":
        file = io.BytesIO()
        torch.save(opt, file)
        file.seek(0)
        other = torch.load(file, weights_only=False)
    else:
        other = getattr(copy, how)(opt)
    for p in other.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    recorder.steps.clear()
    opt.step()
    wanted = recorder.steps[:]
    other.step()
    got = recorder.steps[len(wanted):]
    late = 1 if how == "copy" else 0  # which shares the state
    assert [(s["step"] + late, s["seed"], len(s["ms"]), len(s["masters"]), s["lr"]) for s in wanted] == \
        [(s["step"], s["seed"], len(s["ms"]), len(s["masters"]), s["lr"]) for s in got]
    assert recorder.norms == 3 and (other.state_bits, other.capturable) == (8, False)


def test_optimizer_refusals(recorder):
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(state_bits=16),
                dict(max_grad_norm=-1.0), dict(lr=NAN)):
        with pytest.raises(ValueError):
            train.FusedAdamW(some_params(), **bad)
    p = torch.nn.Parameter(torch.ones(4, 4))
    p.grad = torch.sparse_coo_tensor(torch.tensor([[0], [1]]), torch.tensor([1.0]), (4, 4))
    with pytest.raises(RuntimeError, match="sparse"):
        train.FusedAdamW([p]).step()


def test_moments_to_float():
    codes = torch.tensor([1.0, -2.0, 0.5] * 100).to(torch.float8_e4m3fn)
    scales = torch.tensor([2.0, 0.25])
    want = torch.tensor([1.0, -2.0, 0.5] * 100) * torch.cat((torch.full((256,), 2.0), torch.full((44,), 0.25)))
    assert torch.equal(train.moments_to_float(codes, scales), want)
    assert math.isclose(float(train.moments_to_float(codes.view(10, 30), scales)[9, 29]), 0.125)
