"""The training operators as a user runs them together: norms under autograd, the pre-norm block forward and backward, clipping
and the optimiser, eagerly and from a captured graph.

Tolerances: single norms as in test_train_gpu.py are held elementwise there; here gradients go through bf16 intermediates
(norm output, gate, up, their gradients: one rounding of 2^-8 each, random in sign), so outputs are held to a relative 2-norm
of 5e-3 and gradients to 1e-2, the bounds of the MLP's own tests.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
U = 2.0 ** -24


@pytest.fixture(scope="module")
def fsw(cuda_dev):
    import fused_swiglu_b200 as pkg

    yield pkg
    torch.cuda.synchronize()
    assert pkg.capi.device_status() == 0


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    return float((got - want).norm() / want.norm())


def norm64(x, w, b, eps, layer):
    mean = x.mean(-1, keepdim=True) if layer else 0.0
    z = (x - mean) / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    z = z if w is None else z * w
    return z if b is None else z + b


def leaf64(t):
    return None if t is None else t.detach().double().cpu().requires_grad_()


@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("shape,how", [((3, 5, 96), "plain"), ((1, 1001), "plain"), ((4, 6, 64), "transposed"),
                                       ((4, 40, 2), "sliced"), ((5, 72), "broadcast"), ((0, 64), "plain"), ((64,), "plain")],
                         ids=str)
def test_norms_under_autograd(fsw, cuda_dev, shape, how, layer):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g).to(cuda_dev)
    if how == "transposed":
        x = x.transpose(0, 1)
    if how == "sliced":
        x = x.transpose(1, 2)
    x = x.detach().requires_grad_()
    used = x[:1].expand(7, shape[-1]) if how == "broadcast" else x
    d = used.size(-1)
    w = torch.randn(d, generator=g).to(cuda_dev).requires_grad_()
    b = torch.randn(d, generator=g).to(cuda_dev).requires_grad_() if layer else None
    y = fsw.train.layer_norm(used, w, b, 1e-5) if layer else fsw.train.rms_norm(used, w, 1e-5)
    dout = torch.randn(used.shape, generator=g).to(cuda_dev)
    y.backward(dout)
    x64, w64, b64 = leaf64(x), leaf64(w), leaf64(b)
    y64 = norm64(x64[:1].expand(7, shape[-1]) if how == "broadcast" else x64, w64, b64, 1e-5, layer)
    y64.backward(dout.double().cpu())
    if x.numel() == 0:
        assert y.shape == x.shape and not w.grad.any()
        return
    # sums of at most 1001 terms, off by 48 units of their magnitudes; two of them meet in dx
    for got, want in ((y, y64), (x.grad, x64.grad), (w.grad, w64.grad)) + (((b.grad, b64.grad),) if layer else ()):
        assert rel(got, want) <= 128 * U


def test_norm_gradients_that_nobody_asked_for(fsw, cuda_dev):
    x = torch.randn(6, 64, device=cuda_dev, dtype=BF, requires_grad=True)
    w = torch.ones(64, device=cuda_dev, dtype=BF)
    b = torch.zeros(64, device=cuda_dev, requires_grad=True)
    fsw.train.layer_norm(x, w).sum().backward()
    assert w.grad is None and x.grad is not None
    y = fsw.train.layer_norm(x, None, b)  # an fp32 bias without a weight keeps its gradient in fp32
    y.backward(torch.full_like(y, 1.0078125))
    assert b.grad.dtype == torch.float32 and bool((b.grad == 6 * 1.0078125).all())
    y = fsw.train.rms_norm(x)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(y.sum(), x, create_graph=True)[0].sum(), x)


def block_inputs(M, d, F, dev, seed, norm):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((M, d), generator=g)
    w, b = 1 + 0.1 * torch.randn(d, generator=g), 0.1 * torch.randn(d, generator=g)
    mats = [torch.randn(s, generator=g) * 0.05 for s in ((F, d), (F, d), (d, F))]
    ts = [x, w, b if norm == "layer" else None, *mats]
    return [None if t is None else t.to(BF).to(dev) for t in ts]


def block64(x, w, b, wg, wu, wd, eps, norm):
    n = norm64(x, w, b, eps, norm == "layer")
    g, u = n @ wg.T, n @ wu.T
    return x + (g * torch.sigmoid(g) * u) @ wd.T


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("M,d,F", [(1, 64, 128), (33, 72, 136), (300, 520, 1096), (512, 256, 512)])
def test_block_and_its_gradients(fsw, cuda_dev, M, d, F, norm):
    ts = [None if t is None else t.requires_grad_() for t in block_inputs(M, d, F, cuda_dev, M, norm)]
    out = fsw.train.norm_swiglu_block(*ts, eps=1e-6, norm=norm)
    dout = torch.randn((M, d), generator=torch.Generator().manual_seed(3)).to(BF).to(cuda_dev)
    out.backward(dout)
    ts64 = [leaf64(t) for t in ts]
    out64 = block64(*ts64, 1e-6, norm)
    out64.backward(dout.double().cpu())
    assert rel(out, out64) <= 5e-3
    for t, t64 in zip(ts, ts64):
        if t is not None:
            assert t.grad.dtype == BF and rel(t.grad, t64.grad) <= 1e-2


def test_block_of_views_broadcasts_and_nothing(fsw, cuda_dev):
    """Inputs that start off a boundary or have gaps, a gradient that is one value for all, frozen weights, no rows."""
    x, w, _, wg, wu, wd = block_inputs(40, 64, 128, cuda_dev, 2, "rms")
    want = fsw.train.norm_swiglu_block(x, w, None, wg, wu, wd)
    flat = torch.zeros(40 * 64 + 8, dtype=BF, device=cuda_dev)
    off = flat[1:1 + 40 * 64].view(40, 64)
    off.copy_(x)
    wide = torch.zeros((40, 73), dtype=BF, device=cuda_dev)
    wide[:, 5:69] = x
    for view in (off, wide[:, 5:69], x.t().contiguous().t(), x.view(4, 10, 64).transpose(0, 1).transpose(0, 1)):
        leaf = view.detach().requires_grad_()
        out = fsw.train.norm_swiglu_block(leaf, w, None, wg, wu, wd)
        assert torch.equal(out.reshape(40, 64), want)
        out.sum().backward()  # an expanded gradient
        assert leaf.grad.shape == leaf.shape and bool(torch.isfinite(leaf.grad).all()) and w.grad is None
    empty = torch.empty((0, 3, 64), dtype=BF, device=cuda_dev, requires_grad=True)
    weights = [t.clone().requires_grad_() for t in (w, wg, wu, wd)]
    out = fsw.train.norm_swiglu_block(empty, weights[0], None, *weights[1:])
    out.sum().backward()
    assert out.shape == (0, 3, 64) and empty.grad.shape == empty.shape and not any(t.grad.any() for t in weights)
    with pytest.raises(RuntimeError, match="bfloat16"):
        fsw.train.norm_swiglu_block(x.float(), w, None, wg, wu, wd)
    with pytest.raises(RuntimeError, match="bfloat16"):
        fsw.train.norm_swiglu_block(x, w.float(), None, wg, wu, wd)
    with pytest.raises(ValueError):
        fsw.train.norm_swiglu_block(x, w, w, wg, wu, wd)
    with pytest.raises(ValueError):
        fsw.train.norm_swiglu_block(x, w, None, wg, wu, wd, norm="batch")


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_block_module_agrees_with_the_inference_block(fsw, cuda_dev, norm):
    from fused_swiglu_b200.module import FusedNormSwiGLUBlock, NormSwiGLUBlock

    x, w, b, wg, wu, wd = block_inputs(70, 128, 256, cuda_dev, 5, norm)
    train, serve = NormSwiGLUBlock(128, 256, norm=norm, device=cuda_dev), FusedNormSwiGLUBlock(128, 256, device=cuda_dev)
    with torch.no_grad():
        for block in (train, serve):
            block.norm_weight.copy_(w)
            for p, t in ((block.mlp.gate_proj, wg), (block.mlp.up_proj, wu), (block.mlp.down_proj, wd)):
                p.copy_(t)
        if norm == "layer":
            train.norm_bias.copy_(b)
    out = train(x.view(7, 10, 128))
    assert out.shape == (7, 10, 128) and out.requires_grad
    assert rel(out.view(70, 128), block64(*(None if t is None else t.double().cpu() for t in (x, w, b, wg, wu, wd)), 1e-6, norm)) <= 5e-3
    if norm == "rms":
        assert rel(out.view(70, 128), serve(x)) <= 5e-3
    assert len(list(train.parameters())) == (5 if norm == "layer" else 4) and all(p.requires_grad for p in train.parameters())
    with pytest.raises(RuntimeError, match="last dimension"):
        train(x[:, :64])


def values(opt, p):
    s = opt.state.get(p, {})
    return {k: v.clone() for k, v in s.items() if isinstance(v, torch.Tensor)} | {"p": p.detach().clone()}


def moments(fsw, s, key):
    return (fsw.train.moments_to_float(s[key], s[key + "_scale"]) if key + "_scale" in s else s[key]).double().cpu()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_training_steps_follow_the_formulas(fsw, cuda_dev, norm, bits):
    """Forward, backward, clip, AdamW: each step's weights from the step's own gradients, in 64 bits."""
    from fused_swiglu_b200.module import NormSwiGLUBlock

    torch.manual_seed(0)
    block = NormSwiGLUBlock(136, 264, norm=norm, device=cuda_dev)
    with torch.no_grad():
        for p in (block.mlp.gate_proj, block.mlp.up_proj, block.mlp.down_proj):
            p.normal_(0, 0.1)
    vectors = [p for p in block.parameters() if p.dim() == 1]
    opt = fsw.train.FusedAdamW([{"params": [p for p in block.parameters() if p.dim() == 2], "weight_decay": 0.1},
                                {"params": vectors, "weight_decay": 0.0, "lr": 3e-3}], lr=1e-2, state_bits=bits,
                               max_grad_norm=0.7, seed=5)
    x = torch.randn(50, 136, device=cuda_dev, dtype=BF)
    for step in range(1, 4):
        opt.zero_grad()
        block(x).float().square().mean().mul(100.0).backward()
        before = {p: values(opt, p) for p in block.parameters()}
        opt.step()
        norm64_ = sum(float(p.grad.double().square().sum()) for p in block.parameters()) ** 0.5
        assert abs(float(opt.last_grad_norm[0]) - norm64_) <= 10 * U * norm64_
        scale = min(1.0, 0.7 / (norm64_ + 1e-6))
        for group in opt.param_groups:
            for p in group["params"]:
                old, new = before[p], values(opt, p)
                zero = torch.zeros(p.shape, dtype=torch.float64)
                m0 = moments(fsw, old, "exp_avg") if step > 1 else zero
                v0 = moments(fsw, old, "exp_avg_sq") if step > 1 else zero
                w0 = (old["master"] if step > 1 else old["p"]).double().cpu()
                g = p.grad.double().cpu() * scale
                m, v = 0.9 * m0 + 0.1 * g, 0.999 * v0 + 0.001 * g * g
                update = group["lr"] / (1 - 0.9 ** step) * m / ((v / (1 - 0.999 ** step)).sqrt() + 1e-8)
                w = w0 * (1 - group["lr"] * group["weight_decay"]) - update
                # the norm's 10 units reach the moments, the rest as in test_train_gpu.py; m is a difference
                rate = group["lr"] / (1 - 0.9 ** step) / ((v / (1 - 0.999 ** step)).sqrt() + 1e-8)
                tol = 6 * U * w0.abs() + 48 * U * update.abs() + rate * 16 * U * (m0.abs() + g.abs())
                assert bool(((new["master"].double().cpu() - w).abs() <= tol).all())
                assert torch.equal(new["p"], new["master"].to(BF))
                if bits == 32:
                    assert rel(new["exp_avg"], m) <= 16 * U and rel(new["exp_avg_sq"], v) <= 32 * U
                else:  # one unit at most: 1/8 and 1/4 of a value, or of the smallest normal one
                    got_m, got_v = moments(fsw, new, "exp_avg"), moments(fsw, new, "exp_avg_sq")
                    peak = lambda t: torch.nn.functional.pad(t.flatten().abs(), (0, -t.numel() % 256)).view(-1, 256).amax(1)  # noqa: E731
                    per = lambda t: peak(t).repeat_interleave(256)[:t.numel()].view(t.shape)  # noqa: E731
                    assert bool(((got_m - m).abs() <= m.abs() / 8 * 1.001 + per(m) * 2.0 ** -16).all())
                    assert bool(((got_v - v).abs() <= v / 4 * 1.001 + per(v) * 2.0 ** -30).all())


def test_optimizer_skips_a_step_with_a_bad_gradient(fsw, cuda_dev):
    p = torch.nn.Parameter(torch.ones(300, device=cuda_dev, dtype=BF))
    q = torch.nn.Parameter(torch.ones(30, device=cuda_dev))
    opt = fsw.train.FusedAdamW([p, q], max_grad_norm=1.0)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt.step()
    before = [values(opt, t) for t in (p, q)]
    p.grad[7] = float("nan")
    opt.step()
    for t, old in zip((p, q), before):
        assert all(torch.equal(old[k], v) for k, v in values(opt, t).items())
    p.grad[7] = 1.0
    opt.step()
    assert not torch.equal(before[0]["master"], values(opt, p)["master"])


def test_a_step_is_seen_by_autograd(fsw, cuda_dev):
    """Weights that a step has changed are not those that an earlier forward pass kept."""
    x = torch.randn(4, 64, device=cuda_dev, dtype=BF, requires_grad=True)
    w = torch.nn.Parameter(torch.ones(64, device=cuda_dev, dtype=BF))
    y = fsw.train.rms_norm(x, w)
    w.grad = torch.ones_like(w)
    fsw.train.FusedAdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_first_step_is_not_captured(fsw, cuda_dev):
    p = torch.nn.Parameter(torch.ones(64, device=cuda_dev))
    p.grad = torch.ones_like(p)
    opt = fsw.train.FusedAdamW([p], capturable=True)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="one step before"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    assert bool((p < 1).all())


def test_a_step_with_its_count_on_the_host_is_not_captured(fsw, cuda_dev):
    p = torch.nn.Parameter(torch.ones(64, device=cuda_dev))
    p.grad = torch.ones_like(p)
    opt = fsw.train.FusedAdamW([p])
    opt.step()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="capturable=True"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    assert opt.state[p]["step"] == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_a_whole_training_step_from_a_captured_graph(fsw, cuda_dev, bits):
    """Two graphs of one step each, replayed in turn; both give what the eager step gives from the same state."""
    from fused_swiglu_b200.module import NormSwiGLUBlock

    torch.manual_seed(0)
    block = NormSwiGLUBlock(128, 256, device=cuda_dev)
    with torch.no_grad():
        for p in (block.mlp.gate_proj, block.mlp.up_proj, block.mlp.down_proj):
            p.normal_(0, 0.1)
    opt = fsw.train.FusedAdamW(block.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0, capturable=True)
    x = torch.randn(64, 128, device=cuda_dev, dtype=BF)

    def train_step():
        opt.zero_grad(set_to_none=False)
        out = block(x)
        out.backward(out.detach())
        opt.step()

    def state():
        tensors = [p.data for p in block.parameters()]
        for p in block.parameters():
            tensors += [v for v in opt.state[p].values() if isinstance(v, torch.Tensor)]
        return tensors + [opt.param_groups[0]["step_tensor"]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train_step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            train_step()
        graphs.append(graph)
    torch.cuda.synchronize()
    for graph in (graphs[0], graphs[1], graphs[0]):
        start = [t.clone() for t in state()]
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in state()]
        for t, s in zip(state(), start):
            t.copy_(s)
        with torch.cuda.stream(side):
            train_step()
        torch.cuda.synchronize()
        assert int(replayed[-1]) == int(start[-1]) + 1
        for a, b in zip(state(), replayed):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("before,after", [(False, False), (True, False), (False, True), (True, True)])
def test_training_goes_on_from_a_checkpoint_on_the_host(fsw, cuda_dev, bits, before, after):
    """The same bits as without the break, but for where the step's factors are computed (on the host, or on the device)."""
    g = torch.Generator().manual_seed(5)
    start = [torch.randn(n, generator=g) for n in (700, 4096, 33)]
    grads = [[torch.randn(t.shape, generator=g).to(BF).to(cuda_dev) for t in start] for _ in range(4)]

    def optimizer(values, capturable):
        params = [torch.nn.Parameter(t.to(BF).to(cuda_dev)) for t in values]
        return params, fsw.train.FusedAdamW(params, lr=1e-2, state_bits=bits, max_grad_norm=1.0, seed=3, capturable=capturable)

    def steps(params, opt, which):
        for gs in which:
            for p, gr in zip(params, gs):
                p.grad = gr
            opt.step()

    whole, opt = optimizer(start, before)
    steps(whole, opt, grads[:2])
    saved = {"params": [p.detach().cpu() for p in whole], "opt": {
        "state": {i: {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
                  for i, s in opt.state_dict()["state"].items()},
        "param_groups": [{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in group.items()}
                         for group in opt.state_dict()["param_groups"]]}}
    steps(whole, opt, grads[2:])
    again, other = optimizer(saved["params"], after)
    other.load_state_dict(saved["opt"])
    if after:
        for p, gr in zip(again, grads[2]):
            p.grad = gr
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                other.step()
        torch.cuda.synchronize()
    steps(again, other, grads[2:])
    for p, q in zip(whole, again):
        if before == after:
            assert torch.equal(p, q)
            for key, value in opt.state[p].items():
                if isinstance(value, torch.Tensor):
                    assert torch.equal(value.view(torch.uint8), other.state[q][key].view(torch.uint8))
        else:  # two steps of about lr, their size known to a few units of fp32; one rounding of the parameter may flip
            within_steps = 2 * 1e-2 * 32 * U
            a, b = opt.state[p]["master"].double(), other.state[q]["master"].double()
            assert float((a - b).abs().max()) <= within_steps + 4 * U * float(a.abs().max())


# ---------------------------------------------------------------- waits, launches that overlap

@pytest.mark.parametrize("which", ["layer_forward", "rms_forward", "layer_backward", "rms_backward", "adamw_8bit"])
def test_a_copy_that_never_comes_is_reported_and_leaves_the_device_usable(fsw, cuda_dev, which):
    """One launch whose first copy is left out, with a limit of a few milliseconds: the kernel ends by itself, the host reads
    where a wait gave up, and the next call is right."""
    import fused_mlp_module as lib

    capi = fsw.capi
    g = torch.Generator().manual_seed(0)
    x = torch.randn((900, 1024), generator=g).to(BF).to(cuda_dev)
    w = torch.randn(1024, generator=g).to(BF).to(cuda_dev)
    n = 6_000_000

    def call():
        if which == "layer_forward":
            return lib.layer_norm_forward(x, w, w)
        if which == "rms_forward":
            return lib.rms_norm_forward(x, w)
        stats = [v.float() for v in (x.float().mean(1), torch.rsqrt(x.float().var(1, unbiased=False) + 1e-5))]
        if which == "layer_backward":
            return lib.layer_norm_backward(x, x, *stats, w, True, x)
        if which == "rms_backward":
            return lib.rms_norm_backward(x, x, stats[1], w, x)
        t = {"p": torch.zeros(n, device=cuda_dev), "g": torch.ones(n, device=cuda_dev),
             "m": torch.zeros(n, dtype=torch.uint8, device=cuda_dev).view(torch.float8_e4m3fn),
             "v": torch.zeros(n, dtype=torch.uint8, device=cuda_dev).view(torch.float8_e5m2),
             "ms": torch.zeros((n + 255) // 256, device=cuda_dev), "vs": torch.zeros((n + 255) // 256, device=cuda_dev)}
        lib.adamw_step([t["p"]], [t["g"]], [t["m"]], [t["v"]], 1, 1e-3, exp_avg_scales=[t["ms"]], exp_avg_sq_scales=[t["vs"]])
        return t["p"], t["m"].view(torch.uint8), t["v"].view(torch.uint8), t["ms"]

    want = call()
    torch.cuda.synchronize()
    assert capi.device_status() == 0
    before = capi.lib.fswiglu_set_wait_limit_us(3000)
    try:
        capi.lib.fswiglu_test_expire_next_wait(1)
        call()
        torch.cuda.synchronize()
        word = capi.device_status()
    finally:
        capi.lib.fswiglu_test_expire_next_wait(0)
        capi.lib.fswiglu_set_wait_limit_us(before)
    assert word & 0xFF == (10 if which == "adamw_8bit" else 9) and (word >> 8) - 1 == 0
    assert capi.device_status() == 0
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(call(), want))


def test_launches_that_overlap_wait_for_what_was_written_before(fsw, cuda_dev):
    """Every operator right behind a kernel, a copy, a fill and another stream's work that writes what it reads, many times over,
    eagerly and captured."""
    import fused_mlp_module as lib

    g = torch.Generator().manual_seed(0)
    source = [torch.randn((1500, 2048), generator=g).to(BF).to(cuda_dev) for _ in range(4)]
    x, dy, w = torch.empty_like(source[0]), torch.empty_like(source[0]), source[3][0].clone()
    p, m, v = (torch.empty(1500 * 2048, device=cuda_dev) for _ in range(3))
    other = torch.cuda.Stream()

    def chain(k):
        x.copy_(source[k % 3])  # a copy
        dy.zero_()  # a fill
        dy.add_(source[(k + 1) % 3])  # a kernel
        y, mean, rstd = lib.layer_norm_forward(x, w, w)
        dx, dw, db = lib.layer_norm_backward(dy, x, mean, rstd, w, True, y)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            p.copy_(source[2].view(-1))
            m.zero_()
            v.fill_(1.0)
        torch.cuda.current_stream().wait_stream(other)
        clip = lib.grad_norm_clip([dx, dw, db], 1.0)
        lib.adamw_step([p], [dx.view(-1)], [m], [v], 3, 1e-2, grad_scale=clip[1:])
        lib.adamw_step([p], [dx.view(-1)], [m], [v], 4, 1e-2, grad_scale=clip[1:])
        z = lib.rms_norm_forward(p.view(1500, 2048), None)[0]
        x.zero_()  # behind the readers
        dx_out = dx.clone()
        dx.zero_()
        return [y, dx_out, dw, db, clip, p.clone(), m.clone(), v.clone(), z]

    want = []
    for k in range(3):
        torch.cuda.synchronize()
        out = chain(k)
        torch.cuda.synchronize()
        want.append(out)
    # against the plain formulas once, so that all agreeing on something wrong does not pass
    x64 = source[0].double()
    z64 = (x64 - x64.mean(1, keepdim=True)) / (x64.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    assert rel(want[0][0], z64 * w.double() + w.double()) <= 5e-3
    assert rel(want[0][3], source[1].double().sum(0)) <= 5e-3
    for k in range(60):
        for a, b in zip(chain(k), want[k % 3]):
            assert torch.equal(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [chain(k) for k in range(3)]
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for out, ref in zip(outs, want):
        for a, b in zip(out, ref):
            assert torch.equal(a, b)


def small_chain(fsw, x, w, dy, p, m, v):
    """Norm forward and backward, the gradients' norm, a step: each reads what the one before it wrote."""
    lib = fsw.train._lib()
    y, mean, rstd = lib.layer_norm_forward(x, w)
    dx, dw, db = lib.layer_norm_backward(dy, y, mean, rstd, w, True)
    clip = lib.grad_norm_clip([dw, db, dx], 0.5)
    lib.adamw_step([p], [dw], [m], [v], 1, 1e-2, grad_scale=clip[1:])
    return dx, dw, db, clip, p, m, v


@pytest.mark.parametrize("M,d", [(3, 56), (32, 1000), (9, 1003), (8, 4096)])
def test_small_launches_in_a_row_on_two_streams_and_from_a_graph(fsw, cuda_dev, M, d):
    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        draw = lambda *shape: torch.randn(shape, generator=g).to(cuda_dev)  # noqa: E731
        return [draw(M, d).to(BF), draw(d).to(BF), draw(M, d).to(BF), draw(d), torch.zeros(d, device=cuda_dev),
                torch.zeros(d, device=cuda_dev)]

    def same(a, b):
        return all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))

    want = []
    for seed in range(8):
        args = inputs(seed)
        out = small_chain(fsw, *args)
        torch.cuda.synchronize()
        want.append([t.clone() for t in out])
    args = [inputs(seed) for seed in range(8)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for seed in range(8):
        with torch.cuda.stream(streams[seed % 2]):
            got.append(small_chain(fsw, *args[seed]))
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(got, want))
    static = inputs(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = small_chain(fsw, *static)
    for seed in (3, 5, 3):
        for t, new in zip(static, inputs(seed)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want[seed])


def test_first_calls_of_a_new_thread(fsw, cuda_dev):
    """A backward pass runs on a thread of autograd's, whose first CUDA call may be any of the library's."""
    import threading

    import fused_mlp_module as lib

    x, w, b, wg, wu, wd = block_inputs(300, 520, 1096, cuda_dev, 0, "layer")
    calls = {
        "mlp": lambda: fsw.ops.fused_swiglu_mlp_bf16(x, wg, wu, wd),
        "mlp_backward": lambda: fsw.ops.swiglu_mlp_backward(x, wg, wu, wd, x)[0],
        "norm": lambda: lib.layer_norm_forward(x, w, b)[0],
        "norm_backward": lambda: lib.rms_norm_backward(x, x, lib.rms_norm_forward(x, w)[1], w)[1],
        "clip": lambda: lib.grad_norm_clip([x, w], 1.0),
    }
    for name, call in calls.items():
        want = [call() for _ in range(2)][0]  # and the allocator has what it takes
        torch.cuda.synchronize()
        got = []

        def work():
            try:
                got.append(call())
            except Exception as e:  # noqa: BLE001
                got.append(e)

        t = threading.Thread(target=work)
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert isinstance(got[0], torch.Tensor), (name, got[0])
        assert torch.equal(got[0], want), name


@pytest.mark.parametrize("M,d", [(64, 128), (40, 1024), (300, 4096), (700, 5120), (30, 1003)])
@pytest.mark.parametrize("wt", [BF, torch.float32], ids=["bf16", "fp32"])
def test_norms_read_the_vectors_that_a_step_has_just_written(fsw, cuda_dev, M, d, wt):
    """The optimiser's step on the norm's vectors directly in front of both passes, whose blocks come up while it ends: the same
    bits as with a pause behind each call."""
    lib = fsw.train._lib()
    g = torch.Generator().manual_seed(M + d)
    x, dy = (torch.randn((M, d), generator=g).to(BF).to(cuda_dev) for _ in range(2))
    grads = [torch.randn(d, generator=g).to(wt).to(cuda_dev) for _ in range(2)]
    start = [torch.randn(d, generator=g).to(wt).to(cuda_dev) for _ in range(2)]

    def steps(pause):
        vectors = [t.clone() for t in start]
        m, v = ([torch.zeros(d, device=cuda_dev) for _ in vectors] for _ in range(2))
        out = []
        for k in range(1, 41):
            lib.adamw_step(vectors, grads, m, v, k, 0.05)
            pause()
            y, mean, rstd = lib.layer_norm_forward(x, *vectors)
            pause()
            lib.adamw_step(vectors, grads, m, v, k, 0.05)
            pause()
            dx, dw, db = lib.layer_norm_backward(dy, x, mean, rstd, vectors[0], True)
            pause()
            lib.adamw_step(vectors, grads, m, v, k, 0.05)
            pause()
            out += [y, dx, dw, db, lib.rms_norm_forward(x, vectors[0])[0]]
            pause()
        return out

    want = steps(torch.cuda.synchronize)
    for _ in range(3):
        got = steps(lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not torch.equal(want[0], want[5])  # the vectors do move


def test_a_thread_keeps_its_context_and_gets_one_when_it_has_none(fsw, cuda_dev):
    """Calls that launch nothing, on a thread with a context of its own making, then without any."""
    import ctypes
    import threading

    cu = ctypes.CDLL("libcuda.so.1")
    zero = ctypes.c_void_p(0)
    seen = []

    def call():  # no rows and no gradients of vectors: the device is looked up, nothing is launched
        return fsw.capi.lib.fswiglu_rms_norm_backward(zero, 8, zero, 8, zero, zero, zero, 0, zero, 8, zero, 0, 8, 1, 1, 1, zero, 0, zero)

    def current():
        c = ctypes.c_void_p()
        assert cu.cuCtxGetCurrent(ctypes.byref(c)) == 0
        return c.value

    def work():
        try:
            own, primary = ctypes.c_void_p(), ctypes.c_void_p()
            assert cu.cuCtxCreate_v2(ctypes.byref(own), 0, 0) == 0 and current() == own.value
            seen.append(call() == 0 and call() == 0 and current() == own.value)
            for _ in range(2):
                assert cu.cuCtxSetCurrent(None) == 0 and current() is None
                seen.append(call() == 0 and current() not in (None, own.value))
            assert cu.cuDevicePrimaryCtxRetain(ctypes.byref(primary), 0) == 0
            seen.append(current() == primary.value)
            assert cu.cuDevicePrimaryCtxRelease_v2(0) == 0 and cu.cuCtxDestroy_v2(own) == 0
        except BaseException as e:  # noqa: BLE001
            seen.append(e)

    assert call() == 0
    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert seen == [True] * 4, seen


def test_norms_and_block_under_a_dispatch_mode(fsw, cuda_dev):
    """What watches operations, as counters of them do, changes no bits."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    def both_passes():
        ts = [None if t is None else t.requires_grad_() for t in block_inputs(33, 72, 136, cuda_dev, 4, "layer")]
        y = fsw.train.norm_swiglu_block(*ts, norm="layer")
        z = fsw.train.rms_norm(fsw.train.layer_norm(y, ts[1], ts[2]), ts[1])
        z.backward(torch.ones_like(z))
        return [z.detach()] + [t.grad for t in ts]

    want = both_passes()
    with Watch():
        got = both_passes()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compiled_norms_and_a_block_between_compiled_parts(fsw, cuda_dev):
    """The norms inside a compiled function without a graph break, the block where torch.compile leaves its graph: the bits of the
    eager calls, forward and backward."""
    from fused_swiglu_b200.module import NormSwiGLUBlock

    g = torch.Generator().manual_seed(0)
    start = [torch.randn(s, generator=g).to(BF).to(cuda_dev) for s in ((5, 8, 64), (64,), (64,))]

    def norms(x, w, b):
        return fsw.train.layer_norm(fsw.train.rms_norm(x, w), w, b)

    def both_passes(f):
        leaves = [t.clone().requires_grad_() for t in start]
        y = f(*leaves)
        y.backward(start[0])
        return [y.detach()] + [t.grad for t in leaves]

    torch._dynamo.reset()
    want = both_passes(norms)
    for a, b in zip(both_passes(torch.compile(norms, fullgraph=True, backend="aot_eager")), want):
        assert torch.equal(a, b)
    block = NormSwiGLUBlock(64, 128, device=cuda_dev)
    with torch.no_grad():
        for p in block.mlp.parameters():
            p.copy_(torch.randn(p.shape, generator=g))

    def model(x):
        return block(x * 2) + 1

    def both_passes_of_block(f):
        block.zero_grad()
        x = start[0].clone().requires_grad_()
        y = f(x)
        y.backward(start[0])
        return [y.detach(), x.grad] + [p.grad.clone() for p in block.parameters()]

    want = both_passes_of_block(model)
    for a, b in zip(both_passes_of_block(torch.compile(model, backend="aot_eager")), want):
        assert torch.equal(a, b)
    opt = fsw.train.FusedAdamW(block.parameters(), max_grad_norm=1.0)

    @torch.compile(backend="aot_eager")
    def whole_step(x):
        opt.zero_grad()
        y = model(x)
        y.float().square().mean().backward()
        opt.step()
        return fsw.train.clip_grad_norm([p.grad for p in block.parameters()], 1.0)

    before = [p.detach().clone() for p in block.parameters()]
    assert float(whole_step(start[0])[0]) > 0 and float(whole_step(start[0])[0]) > 0
    assert all(not torch.equal(p, q) for p, q in zip(block.parameters(), before))
    assert all(s["step"] == 2 for s in opt.state.values())
    torch._dynamo.reset()
