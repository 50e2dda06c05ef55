"""Training operators around the MLP against their formulas in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a unit of fp32, and an output of type T adds half a unit of T (bf16 2^-8,
fp32 2^-24, relative).  A sum over n values that a kernel takes as at least 32 partial sums and a tree is off by at most
(n / 32 + 16) u times the sum of the magnitudes; sums over rows, one after the other, by (rows + 8) u times that.
"""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def fsw(cuda_dev):
    import fused_swiglu_b200 as pkg

    yield pkg
    torch.cuda.synchronize()
    assert pkg.capi.device_status() == 0


@pytest.fixture(scope="module")
def lib(fsw):
    import fused_mlp_module

    return fused_mlp_module


def within(got, want, tol):
    """Elementwise, with the worst place in the message; NaN and infinity have to be in the same places."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    over = torch.where(fine, (got - want).abs() - tol, torch.zeros_like(want))
    i = int(over.argmax()) if over.numel() else 0
    assert not over.numel() or over.flatten()[i] <= 0, (i, got.flatten()[i].item(), want.flatten()[i].item(), tol.flatten()[i].item())


# ---------------------------------------------------------------- norms

def norm_inputs(M, d, t, wt, dev, seed, bias=True, weight=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((M, d), generator=g) * 2 + torch.randn((M, 1), generator=g)).to(t)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(wt) if weight else None
    b = (0.3 * torch.randn(d, generator=g)).to(wt) if bias else None
    dy = torch.randn((M, d), generator=g).to(t)
    res = torch.randn((M, d), generator=g).to(t)
    return tuple(None if v is None else v.to(dev) for v in (x, w, b, dy, res))


def forward64(x, w, b, eps, layer):
    x = x.double().cpu()
    mean = x.mean(1) if layer else torch.zeros(x.size(0), dtype=torch.float64)
    rstd = 1 / torch.sqrt((x - mean[:, None]).square().mean(1) + eps)
    y = (x - mean[:, None]) * rstd[:, None]
    y = y * (1.0 if w is None else w.double().cpu()) + (0.0 if b is None else b.double().cpu())
    return y, mean, rstd


def check_forward(lib, x, w, b, eps, layer, out=None):
    d = x.size(1)
    k = d / 32 + 16
    y, mean, rstd = forward64(x, w, b, eps, layer)
    if out is None:
        out = lib.layer_norm_forward(x, w, b, eps) if layer else lib.rms_norm_forward(x, w, eps)
    big = x.double().cpu().abs()
    away = k * U * big.mean(1) if layer else 0 * big.mean(1)  # how far the mean may be off
    if layer:
        within(out[1], mean, away + U * mean.abs())
    # relative: the sum of squares, its terms, the division, the root; and the mean's own error, whose square is added
    off = (k + 8) * U + (away * rstd) ** 2
    within(out[-1], rstd, off * rstd)
    scale = (1.0 if w is None else w.double().cpu().abs()) * rstd[:, None]
    tol = scale * (away[:, None] + (off[:, None] + 4 * U) * (x.double().cpu() - mean[:, None]).abs()) + 2 * U * y.abs()
    within(out[0], y, tol + HALF[x.dtype] * y.abs())
    assert out[0].dtype == x.dtype and out[0].is_contiguous()


def backward64(dy, x, mean, rstd, w, res, layer):
    dy, x, mean, rstd = (v.double().cpu() for v in (dy, x, mean, rstd))
    z = (x - mean[:, None]) * rstd[:, None]
    a = dy * (1.0 if w is None else w.double().cpu())
    dx = a - z * (a * z).mean(1, keepdim=True)
    if layer:
        dx = dx - a.mean(1, keepdim=True)
    dx = dx * rstd[:, None]
    if res is not None:
        dx = dx + res.double().cpu()
    return dx, (dy * z).sum(0), dy.sum(0), z, a


def check_backward(lib, dy, x, mean, rstd, w, res, layer, grads, gt):
    M, d = x.shape
    k = d / 32 + 16
    dx, dw, db, z, a = backward64(dy, x, mean, rstd, w, res, layer)
    r = rstd.double().cpu()[:, None]
    # x - mean loses a unit of the larger of the two where they are close
    dz = 2 * U * z.abs() + U * r * torch.maximum(x.double().cpu().abs(), mean.double().cpu().abs()[:, None])
    c2 = (a * z).abs().mean(1, keepdim=True)
    tol = 6 * U * (a.abs() + z.abs() * c2) + dz * c2 + z.abs() * ((k + 4) * U * c2 + (a.abs() * dz).mean(1, keepdim=True))
    if layer:
        tol = tol + (k + 4) * U * a.abs().mean(1, keepdim=True)
    tol = tol * r + 2 * U * dx.abs() + (0 if res is None else U * res.double().cpu().abs())
    within(grads[0], dx, tol + HALF[x.dtype] * dx.abs())
    n = M + 8
    if grads[1] is not None:
        assert grads[1].dtype == gt
        size = dy.double().cpu().abs()
        within(grads[1], dw, n * U * (size * z.abs()).sum(0) + (size * dz).sum(0) + HALF[gt] * dw.abs())
    if len(grads) > 2 and grads[2] is not None:
        assert grads[2].dtype == gt
        within(grads[2], db, n * U * dy.double().cpu().abs().sum(0) + HALF[gt] * db.abs())


# one column, odd widths, each width where a kernel changes, the widths of the configurations, a row beyond one block's
# registers; one row, fewer rows than SMs, many rows
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (4, 33), (7, 64), (33, 127), (300, 256), (9, 520), (5, 1000), (64, 1003), (3, 1024),
          (2, 1032), (17, 2048), (5, 2056), (16, 4096), (3, 4100), (700, 136), (4, 5120), (3, 8192), (2, 8200), (1, 16384),
          (3, 20001), (2, 40000), (1500, 24), (2100, 520)]


@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("t,wt", [(BF, BF), (BF, F32), (F32, F32)], ids=["bf16", "bf16_w32", "fp32"])
@pytest.mark.parametrize("M,d", SHAPES)
def test_norm_forward_and_backward(lib, cuda_dev, M, d, t, wt, layer):
    x, w, b, dy, res = norm_inputs(M, d, t, wt, cuda_dev, M * 7 + d, bias=layer)
    check_forward(lib, x, w, b, 1e-5, layer)
    _, mean, rstd = (v.float().to(cuda_dev) for v in forward64(x, w, b, 1e-5, layer))
    if layer:
        grads = lib.layer_norm_backward(dy, x, mean, rstd, w, True, res)
    else:
        grads = lib.rms_norm_backward(dy, x, rstd, w, res)
    check_backward(lib, dy, x, mean, rstd, w, res, layer, grads, wt)


@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("M,d", [(3, 4), (5, 7), (33, 128), (300, 256), (64, 1003), (150, 1032), (16, 4096), (3, 5120), (5, 8192),
                                 (2, 8200), (2, 20001)])
def test_norm_of_fp32_rows_with_bf16_vectors(lib, cuda_dev, M, d, layer):
    x, w, b, dy, res = norm_inputs(M, d, F32, BF, cuda_dev, M * 5 + d, bias=layer)
    check_forward(lib, x, w, b, 1e-5, layer)
    _, mean, rstd = (v.float().to(cuda_dev) for v in forward64(x, w, b, 1e-5, layer))
    if layer:
        grads = lib.layer_norm_backward(dy, x, mean, rstd, w, True, res)
    else:
        grads = lib.rms_norm_backward(dy, x, rstd, w, res)
    check_backward(lib, dy, x, mean, rstd, w, res, layer, grads, BF)


@pytest.mark.parametrize("M", [147, 148, 149, 295, 296, 297, 1184, 1185])
@pytest.mark.parametrize("d", [72, 99, 640])
def test_norm_of_as_many_rows_as_blocks(lib, cuda_dev, M, d):
    """One row less, as many, and one more than the grids have blocks."""
    x, w, b, dy, res = norm_inputs(M, d, BF, BF, cuda_dev, M + d)
    check_forward(lib, x, w, b, 1e-5, True)
    _, mean, rstd = (v.float().to(cuda_dev) for v in forward64(x, w, b, 1e-5, True))
    check_backward(lib, dy, x, mean, rstd, w, res, True, lib.layer_norm_backward(dy, x, mean, rstd, w, True, res), BF)


@pytest.mark.parametrize("t", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [8, 56, 99, 136, 1003, 1032, 4096, 8192])
def test_norm_gradients_of_few_rows(lib, cuda_dev, d, t):
    """Row counts around those up to which one cluster takes all rows, blocks without rows among them."""
    for M in (1, 2, 7, 8, 9, 31, 32, 33, 63, 65, 96, 97, 128, 129, 256, 257, 513, 769, 1025):
        x, w, b, dy, res = norm_inputs(M, d, t, t, cuda_dev, M + d)
        for layer in (True, False):
            _, mean, rstd = (v.float().to(cuda_dev) for v in forward64(x, w, b if layer else None, 1e-5, layer))
            if layer:
                grads = lib.layer_norm_backward(dy, x, mean, rstd, w, True, res)
                only_b = lib.layer_norm_backward(dy, x, mean, rstd, w, True, res, weight_grad=False)
                only_w = lib.layer_norm_backward(dy, x, mean, rstd, w, False, res)
                assert only_b[1] is None and torch.equal(only_b[2], grads[2])
                assert only_w[2] is None and torch.equal(only_w[1], grads[1])
            else:
                grads = lib.rms_norm_backward(dy, x, rstd, w, res)
            check_backward(lib, dy, x, mean, rstd, w, res, layer, grads, t)


@pytest.mark.parametrize("M,d", [(6, 100), (5, 4096), (40, 1003)])
def test_norm_options(lib, cuda_dev, M, d):
    """Without weight, bias or residual; gradients in fp32; only the gradients that are asked for."""
    x, w, b, dy, res = norm_inputs(M, d, BF, BF, cuda_dev, 3)
    check_forward(lib, x, None, None, 1e-6, True)
    check_forward(lib, x, None, None, 1e-6, False)
    check_forward(lib, x, w, None, 1e-6, True)
    check_forward(lib, x, None, b, 1e-6, True)
    _, mean, rstd = (v.float().to(cuda_dev) for v in forward64(x, w, b, 1e-6, True))
    full = lib.layer_norm_backward(dy, x, mean, rstd, w, True, None, fp32_grads=True)
    check_backward(lib, dy, x, mean, rstd, w, None, True, full, F32)
    no_w = lib.layer_norm_backward(dy, x, mean, rstd, w, True, None, fp32_grads=True, weight_grad=False)
    assert no_w[1] is None and torch.equal(no_w[0], full[0]) and torch.equal(no_w[2], full[2])
    only_dx = lib.layer_norm_backward(dy, x, mean, rstd, w, False, None, weight_grad=False)
    assert only_dx[1] is None and only_dx[2] is None and torch.equal(only_dx[0], full[0])
    plain = lib.layer_norm_backward(dy, x, mean, rstd, None, False, res)
    assert plain[1] is None and plain[2] is None
    check_backward(lib, dy, x, mean, rstd, None, res, True, plain, BF)


@pytest.mark.parametrize("t", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,d,offset,pitch", [(9, 64, 1, 67), (5, 4096, 1, 4097), (5, 4096, 8, 4104), (33, 520, 3, 1031),
                                              (4, 1003, 0, 1008)])
def test_norm_of_strided_and_unaligned_rows(lib, cuda_dev, M, d, offset, pitch, t):
    """Rows inside a wider buffer, at an odd offset: the same bits as for contiguous copies of the wide-load kernel's rows
    are not asked, the formulas are; and what lies around is not touched."""
    g = torch.Generator().manual_seed(M + d)
    wide = [torch.randn((M * pitch + offset + 64,), generator=g).to(t).to(cuda_dev) for _ in range(3)]
    x, dy, res = (v[offset:offset + M * pitch].view(M, pitch)[:, :d] for v in wide)
    before = [v.clone() for v in wide]
    w = (1 + 0.2 * torch.randn(d + 1, generator=g)).to(t).to(cuda_dev)[1:]  # a vector off its boundary too
    b = torch.randn(d + 1, generator=g).to(t).to(cuda_dev)[1:]
    check_forward(lib, x, w, b, 1e-5, True)
    _, mean, rstd = (v.float().to(cuda_dev) for v in forward64(x, w, b, 1e-5, True))
    check_backward(lib, dy, x, mean, rstd, w, res, True, lib.layer_norm_backward(dy, x, mean, rstd, w, True, res), t)
    for v, was in zip(wide, before):
        assert torch.equal(v, was)


@pytest.mark.parametrize("t", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,d,pitch,offset", [(5, 72, 80, 0), (3, 1003, 1010, 1), (2, 4096, 4104, 8), (2, 20001, 20003, 1)])
def test_norm_outputs_stay_in_their_rows(fsw, lib, cuda_dev, M, d, pitch, offset, t):
    """Through the C ABI: outputs with a pitch, canaries between and behind the rows."""
    x, w, b, dy, res = norm_inputs(M, d, t, t, cuda_dev, 5)
    code = fsw.capi.OUT_F32 if t == F32 else fsw.capi.OUT_BF16
    vp = lambda v: ctypes.c_void_p(v.data_ptr())  # noqa: E731
    outs = [torch.full((M * pitch + offset + 32,), 77.0, dtype=t, device=cuda_dev) for _ in range(2)]
    rows = [o[offset:offset + M * pitch].view(M, pitch)[:, :d] for o in outs]
    stats = [torch.full((M + 8,), 77.0, device=cuda_dev) for _ in range(2)]
    vectors = [torch.full((d + 8,), 77.0, dtype=t, device=cuda_dev) for _ in range(2)]
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    rc = fsw.capi.lib.fswiglu_layer_norm_forward(vp(x), d, vp(w), vp(b), vp(rows[0]), pitch, vp(stats[0]), vp(stats[1]), M, d,
                                                 code, code, 1e-5, stream)
    assert rc == 0
    ws = torch.empty(fsw.capi.lib.fswiglu_norm_backward_workspace_bytes(M, d), dtype=torch.uint8, device=cuda_dev)
    rc = fsw.capi.lib.fswiglu_layer_norm_backward(vp(dy), d, vp(x), d, vp(stats[0]), vp(stats[1]), vp(w), vp(res), d,
                                                  vp(rows[1]), pitch, vp(vectors[0]), vp(vectors[1]), M, d, code, code, code,
                                                  vp(ws), ws.numel(), stream)
    assert rc == 0
    y, mean, rstd = lib.layer_norm_forward(x, w, b, 1e-5)
    dx, dw, db = lib.layer_norm_backward(dy, x, mean, rstd, w, True, res)
    check_forward(lib, x, w, b, 1e-5, True, out=(rows[0].contiguous(), stats[0][:M], stats[1][:M]))
    check_backward(lib, dy, x, mean, rstd, w, res, True, (rows[1].contiguous(), vectors[0][:d], vectors[1][:d]), t)
    for o, r in zip(outs, rows):
        left = o.clone()
        left[offset:offset + M * pitch].view(M, pitch)[:, :d] = 77.0
        assert bool((left == 77.0).all())
    assert all(bool((s[M:] == 77.0).all()) for s in stats) and all(bool((v[d:] == 77.0).all()) for v in vectors)


@pytest.mark.parametrize("t", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,d", [(3000, 99), (9000, 37), (1300, 1003)])
def test_norm_bits_do_not_depend_on_where_rows_start(lib, cuda_dev, M, d, t):
    """The first row's first elements, copied one by one, lie where later rows of the same place come by bulk copies."""
    x, w, b, dy, res = norm_inputs(M, d, t, t, cuda_dev, M + d)
    want = lib.layer_norm_forward(x, w, b)
    grads = lib.layer_norm_backward(dy, x, *want[1:], w, True, res)
    for offset in range(1, 16 // t.itemsize):
        def moved(v):
            flat = torch.empty(M * d + 16, dtype=t, device=cuda_dev)
            flat[offset:offset + M * d] = v.view(-1)
            return flat[offset:offset + M * d].view(M, d)

        got = lib.layer_norm_forward(moved(x), w, b)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        got = lib.layer_norm_backward(moved(dy), moved(x), *want[1:], w, True, moved(res))
        assert all(torch.equal(p, q) for p, q in zip(got, grads))


@pytest.mark.parametrize("t", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [1, 2, 3, 5, 6, 7])
def test_norm_of_rows_within_a_granule(lib, cuda_dev, d, t):
    """Rows of less than 16 bytes, several of which share the matrix's first granule and its last, from every start."""
    for M in (1, 2, 3, 4, 9, 16, 17, 40, 5000):
        x, w, b, dy, res = norm_inputs(M, d, t, t, cuda_dev, M + d)
        want = lib.layer_norm_forward(x, w, b)
        check_forward(lib, x, w, b, 1e-5, True, out=want)
        for offset in range(0, 16 // t.itemsize):
            flat = torch.full((M * d + 16,), float("nan"), dtype=t, device=cuda_dev)
            flat[offset:offset + M * d] = x.view(-1)
            moved = flat[offset:offset + M * d].view(M, d)
            assert all(torch.equal(p, q) for p, q in zip(lib.layer_norm_forward(moved, w, b), want))
        grads = lib.layer_norm_backward(dy, x, *want[1:], w, True, res)
        check_backward(lib, dy, x, *want[1:], w, res, True, grads, t)


@pytest.mark.parametrize("M,d,where", [(300, 64, "short"), (40, 1024, "wide"), (300, 4096, "wide"), (700, 5120, "wide, computed again"),
                                       (20, 6400, "wide"), (6, 9000, "wide, computed again"), (300, 1003, "odd"), (9, 33, "odd"), (5, 12800, "any")], ids=str)
@pytest.mark.parametrize("t", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("away", [0, 100, 1000])
def test_norm_backward_of_rows_far_off_zero(lib, cuda_dev, M, d, where, t, away):
    """Means far above the spread.  The mean is an input, and x - mean of close fp32 values is exact: z = (x - mean) rstd is off by the
    roundings of the difference and the product alone, 2 u |z|, however large the mean.  dx = rstd (a - c1 - z c2) + res, with sums
    c1 and c2 over the row that are off by (d / 32 + 16) u of their magnitudes and c2 also by z's error; dw by the rows' sums."""
    x, w, b, dy, res = norm_inputs(M, d, F32, t, cuda_dev, M + d)
    x = (x + away * (1 if t == F32 else 0.02)).to(t)  # bf16 rows so far off have eight bits for their spread
    dy, res = dy.to(t), res.to(t)
    _, mean, rstd = (v.float().to(cuda_dev) for v in forward64(x, w, b, 1e-5, True))
    got = lib.layer_norm_backward(dy, x, mean, rstd, w, True, res, fp32_grads=True)
    dx, dw, db, z, a = backward64(dy, x, mean, rstd, w, res, True)
    k, r = d / 32 + 16, rstd.double().cpu()[:, None]
    c2 = (a * z).abs().mean(1, keepdim=True)
    # u of each term for: z 2, a 1, and at most 4 more products, sums and the quotient by d on its way
    tol = U * (6 * a.abs() + (k + 6) * a.abs().mean(1, keepdim=True) + (k + 10) * z.abs() * c2)
    tol = tol * r + 2 * U * (dx.abs() + res.double().cpu().abs())
    within(got[0], dx, tol + HALF[t] * dx.abs())
    size = dy.double().cpu().abs()
    within(got[1], dw, (M + 12) * U * (size * z.abs()).sum(0))
    within(got[2], db, (M + 8) * U * size.sum(0))


@pytest.mark.parametrize("M,d", [(120, 1024), (120, 4096), (120, 1003), (120, 12800), (8, 1024), (8, 1003), (5, 4096)])
@pytest.mark.parametrize("gt", [F32, BF], ids=["fp32", "bf16"])
def test_norm_vector_gradients_of_blocks_are_joined_in_64_bits(lib, cuda_dev, M, d, gt):
    """One row a block (fewer rows than SMs, or than a cluster's blocks), whose products are exact: eight bits of dy times four of
    z.  dy spreads over 28 powers of two, so that no order of fp32 additions is exact, and sums in 64 bits are: what is asked is
    the exact sum, rounded once."""
    g = torch.Generator().manual_seed(M + d)
    x = torch.randint(-15, 16, (M, d), generator=g).float().to(cuda_dev)
    dy = torch.ldexp(torch.randint(-255, 256, (M, d), generator=g).float(), torch.randint(0, 21, (M, d), generator=g)).to(cuda_dev)
    mean, rstd = torch.zeros(M, device=cuda_dev), torch.full((M,), 0.5, device=cuda_dev)
    w = torch.ones(d, dtype=gt, device=cuda_dev)
    dw, db = (dy.double() * x.double() * 0.5).sum(0), dy.double().sum(0)
    for got, want in zip(lib.layer_norm_backward(dy, x, mean, rstd, w, True)[1:], (dw, db)):
        once = want.to(F32) if gt == F32 else torch.frexp(want)
        if gt == BF:  # to nearest even at eight bits, in one step: torch goes by way of fp32
            once = torch.ldexp(torch.round(torch.ldexp(once[0], torch.tensor(8, device=cuda_dev))), once[1] - 8).to(BF)
        assert torch.equal(got, once)
    assert torch.equal(lib.rms_norm_backward(dy, x, rstd, w)[1], lib.layer_norm_backward(dy, x, mean, rstd, w)[1])


def test_norm_offsets_past_32_bits(lib, cuda_dev):
    """More than 2^31 elements: the last rows are what a call of those alone gives, and the others' zeros add nothing."""
    M, d, n = 530_000, 4096, 40
    x, w, b, dy, res = norm_inputs(n, d, BF, BF, cuda_dev, 8)
    big, big_dy = (torch.zeros((M, d), dtype=BF, device=cuda_dev) for _ in range(2))
    big[-n:], big_dy[-n:] = x, dy
    y, mean, rstd = lib.layer_norm_forward(big, w, b, 1e-5)
    check_forward(lib, x, w, b, 1e-5, True, out=(y[-n:], mean[-n:], rstd[-n:]))
    assert torch.equal(y[:1000], b.expand(1000, d)) and torch.equal(y[-n - 1000:-n], b.expand(1000, d))
    del y
    dx, dw, db = lib.layer_norm_backward(big_dy, big, mean, rstd, w, True)
    check_backward(lib, dy, x, mean[-n:], rstd[-n:], w, None, True, (dx[-n:], dw, db), BF)
    assert not dx[:1000].any() and not dx[-n - 1000:-n].any()


def test_norm_without_rows(lib, cuda_dev):
    x = torch.empty((0, 72), dtype=BF, device=cuda_dev)
    w = torch.ones(72, dtype=BF, device=cuda_dev)
    y, mean, rstd = lib.layer_norm_forward(x, w, w)
    assert y.shape == (0, 72) and mean.shape == rstd.shape == (0,)
    dx, dw, db = lib.layer_norm_backward(x, x, mean, rstd, w, True)
    assert dx.shape == (0, 72) and not dw.any() and not db.any()
    dx, dw = lib.rms_norm_backward(x, x, rstd, w)
    assert not dw.any()


@pytest.mark.parametrize("d", [1003, 4096])
def test_norm_rows_are_independent_of_bad_ones(lib, cuda_dev, d):
    """NaN, infinities, the type's largest values, equal values and zeros stay in their rows."""
    x, w, b, dy, res = norm_inputs(12, d, BF, BF, cuda_dev, 9)
    good = lib.layer_norm_forward(x, w, b)
    y = x.clone()
    y[1, 5], y[3, 0], y[5], y[7], y[9] = float("nan"), float("inf"), 3.0, 0.0, 3e38
    out = lib.layer_norm_forward(y, w, b)
    keep = [0, 2, 4, 6, 8, 10, 11]
    for p, q in zip(out, good):
        assert torch.equal(p[keep], q[keep])
    assert bool(torch.isnan(out[0][1]).all()) and bool(torch.isnan(out[0][3]).any())
    assert torch.equal(out[0][7], b) and float(out[2][7]) == pytest.approx(1e-5 ** -0.5, rel=1e-6)
    within(out[0][5], b, 16 * U * (w.double().cpu().abs() * 1e-5 ** -0.5 * 3) * (d / 32 + 16) + HALF[BF] * b.double().cpu().abs())
    g1 = lib.layer_norm_backward(dy, y, out[1], out[2], w, True, res)
    g0 = lib.layer_norm_backward(dy, x, good[1], good[2], w, True, res)
    assert torch.equal(g1[0][keep], g0[0][keep])


def test_norm_is_deterministic_and_takes_streams_and_graphs(lib, cuda_dev):
    x, w, b, dy, res = norm_inputs(777, 1032, BF, BF, cuda_dev, 1)
    _, mean, rstd = lib.layer_norm_forward(x, w, b)
    want = lib.layer_norm_backward(dy, x, mean, rstd, w, True, res)
    for _ in range(3):
        for p, q in zip(lib.layer_norm_backward(dy, x, mean, rstd, w, True, res), want):
            assert torch.equal(p, q)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:  # two calls at once: each has its own partial sums
        with torch.cuda.stream(s):
            got.append(lib.layer_norm_backward(dy, x, mean, rstd, w, True, res))
    torch.cuda.synchronize()
    for g in got:
        for p, q in zip(g, want):
            assert torch.equal(p, q)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = lib.layer_norm_backward(dy, x, *lib.layer_norm_forward(x, w, b)[1:], w, True, res)
        graphs.append((g, out))
    dy.neg_()
    res.neg_()
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        for p, q in zip(out, want):
            assert torch.equal(p, -q)


def test_norm_backward_against_differences(lib, cuda_dev):
    """Central differences of the kernel's own forward pass, in fp32, along random directions."""
    x, w, b, dy, _ = norm_inputs(4, 65, F32, F32, cuda_dev, 2)
    y, mean, rstd = lib.layer_norm_forward(x, w, b)
    dx, dw, db = lib.layer_norm_backward(dy, x, mean, rstd, w, True)
    g = torch.Generator().manual_seed(4)
    h = 2.0 ** -6
    for leaf, grad in ((x, dx), (w, dw), (b, db)):
        v = torch.randn(leaf.shape, generator=g).to(cuda_dev)
        at = lambda s: (lib.layer_norm_forward(*(leaf + s * h * v if t is leaf else t for t in (x, w, b)))[0].double()  # noqa: E731
                        * dy.double()).sum().item()
        slope = (8 * (at(0.5) - at(-0.5)) - (at(1) - at(-1))) / (6 * h)
        # the outputs' roundings over h; what the differences leave out is of the order of h^4
        size = float((y.abs() * dy.abs()).sum())
        assert abs(slope - float((grad.double() * v.double()).sum())) <= 64 * U * size / h + 200 * h ** 4 * size


def test_norm_refusals(lib, cuda_dev):
    x, w, b, dy, res = norm_inputs(4, 64, BF, BF, cuda_dev, 0)
    _, mean, rstd = lib.layer_norm_forward(x, w, b)
    with pytest.raises(RuntimeError, match="2-D"):
        lib.layer_norm_forward(x[0], w, b)
    with pytest.raises(RuntimeError, match="unit stride"):
        lib.layer_norm_forward(x.t(), None, None)
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        lib.rms_norm_forward(x.half())
    with pytest.raises(RuntimeError, match="one type"):
        lib.layer_norm_forward(x, w, b.float())
    with pytest.raises(RuntimeError, match="row length"):
        lib.layer_norm_forward(x, w[:32], b)
    with pytest.raises(RuntimeError, match="CUDA"):
        lib.rms_norm_forward(x.cpu())
    with pytest.raises(RuntimeError, match="status -1"):
        lib.rms_norm_forward(x, w, -1.0)
    with pytest.raises(RuntimeError, match="status -3"):  # rows that share memory
        lib.rms_norm_forward(x[:1].expand(4, 64), w)
    with pytest.raises(RuntimeError, match="shape of x"):
        lib.rms_norm_backward(dy[:3], x, rstd, w)
    with pytest.raises(RuntimeError, match="type and device"):
        lib.rms_norm_backward(dy.float(), x, rstd, w)
    with pytest.raises(RuntimeError, match="one entry per row"):
        lib.layer_norm_backward(dy, x, mean[:3], rstd, w)
    with pytest.raises(RuntimeError, match="float32 vector"):
        lib.layer_norm_backward(dy, x, mean, rstd.to(BF), w)


def test_dispatcher_ops_are_the_module_functions(lib, cuda_dev):
    o = torch.ops.ASMLLM
    x, w, b, dy, res = norm_inputs(20, 96, BF, F32, cuda_dev, 1)
    y, mean, rstd = lib.layer_norm_forward(x, w, b)
    for p, q in zip(o.layer_norm_forward(x, w, b), (y, mean, rstd)):
        assert torch.equal(p, q)
    for p, q in zip(o.layer_norm_backward(dy, x, mean, rstd, w, True, res), lib.layer_norm_backward(dy, x, mean, rstd, w, True, res)):
        assert torch.equal(p, q)
    only = o.layer_norm_backward(dy, x, mean, rstd, w)
    assert only[2] is None and torch.equal(only[0], lib.layer_norm_backward(dy, x, mean, rstd, w)[0])
    assert torch.equal(o.rms_norm_forward(x, w)[0], lib.rms_norm_forward(x, w)[0])
    assert torch.equal(o.rms_norm_backward(dy, x, rstd, w)[1], lib.rms_norm_backward(dy, x, rstd, w)[1])
    assert torch.equal(o.grad_norm_clip([x, w], 1.0), lib.grad_norm_clip((x, w), 1.0))
    both = [adam_inputs([700, 9], BF, BF, 8, True, cuda_dev, 2)[0] for _ in range(2)]
    of = lambda ts, key: [t[key] for t in ts]  # noqa: E731
    for ts, call in zip(both, (lib.adamw_step, o.adamw_step)):
        call(of(ts, "p"), of(ts, "g"), of(ts, "m"), of(ts, "v"), 3, 1e-2, 0.9, 0.999, 1e-8, 0.0, of(ts, "w"), of(ts, "ms"),
             of(ts, "vs"), None, 5)
    for p, q in zip(*both):
        assert all(torch.equal(p[k].view(torch.uint8), q[k].view(torch.uint8)) for k in p)


# ---------------------------------------------------------------- AdamW

def random_moments(n, spread, bits, g):
    m, v = torch.randn(n, generator=g) * spread * 0.3, (torch.randn(n, generator=g) * spread).square() * 1.5
    if bits == 32:
        return {"m": m, "v": v}
    out = {}
    for key, x, t, top in (("m", m, torch.float8_e4m3fn, 7), ("v", v, torch.float8_e5m2, 14)):
        rows = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
        scale = torch.exp2(torch.floor(torch.log2(rows.abs().amax(1))) - top)
        out[key], out[key + "s"] = (rows / scale[:, None]).to(t).view(torch.uint8).flatten()[:n].view(t), scale
    return out


def adam_inputs(sizes, pt, gt, bits, master, dev, seed, lead=None):
    """Lists of tensors, each in a buffer of its own with canaries around; `lead` elements in front move them off alignment."""
    g = torch.Generator().manual_seed(seed)
    tensors, buffers = [], []
    for i, n in enumerate(sizes):
        spread = 10.0 ** torch.empty(1).uniform_(-4, 0, generator=g).item()
        values = {"p": (torch.randn(n, generator=g) * 0.1).to(pt), "g": (torch.randn(n, generator=g) * spread).to(gt),
                  **random_moments(n, spread, bits, g)}
        if master:
            values["w"] = values["p"].float() + torch.randn(n, generator=g) * 1e-4
        front = 0 if lead is None else lead[i % len(lead)]
        placed = {}
        for key, v in values.items():
            bytes_ = torch.full((v.numel() + front + 16,), 3, dtype=torch.uint8).repeat_interleave(v.element_size())
            buffer = bytes_.to(dev).view(v.dtype)
            buffer[front:front + v.numel()] = v.to(dev)
            placed[key] = buffer[front:front + v.numel()]
            buffers.append((buffer, front, v.numel()))
        tensors.append(placed)
    return tensors, buffers


def canaries_hold(buffers):
    for b, front, n in buffers:
        raw = b.view(torch.uint8)
        size = b.element_size()
        assert bool((raw[:front * size] == 3).all()) and bool((raw[(front + n) * size:] == 3).all())


HYPER = dict(beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1)


def take_step(lib, tensors, step=7, lr=1e-2, scale=None, seed=11, **more):
    of = lambda key: [t[key] for t in tensors if key in t]  # noqa: E731
    lib.adamw_step(of("p"), of("g"), of("m"), of("v"), step, lr, HYPER["beta1"], HYPER["beta2"], HYPER["eps"],
                   HYPER["weight_decay"], of("w"), of("ms"), of("vs"), scale, seed, **more)


def decoded(codes, scales):
    return codes.double().cpu() * scales.double().cpu().repeat_interleave(256)[:codes.numel()]


def mix32(x):
    x = ((x ^ (x >> 16)) * 0xDDC24D79) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x77D0AC3D) & 0xFFFFFFFF
    return x ^ (x >> 16)


MULTIPLIERS = (0x5ECD29B7, 0xDB623B29, 0x69758763, 0x7D45CE1D, 0x74A1B41D, 0x75BBB081, 0x5AD24435, 0x73B07CC5)


def random_bits(n, first_block, seed, step):
    key = mix32((seed & 0xFFFFFFFF) ^ mix32((step ^ (seed >> 32)) & 0xFFFFFFFF))
    group = first_block * 32 + torch.arange((n + 7) // 8)
    h = mix32((group & 0xFFFFFFFF) ^ ((group >> 32) * MULTIPLIERS[0] & 0xFFFFFFFF) ^ key)
    return ((h[:, None] * torch.tensor(MULTIPLIERS)) & 0xFFFFFFFF).flatten()[:n]


def encode(x, random16, top, mantissa, bias, keep_positive):
    """The 8-bit floats that x (fp32, >= 0) is rounded to, step by step as the format is defined, and the scales."""
    rows = torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)
    _, e = torch.frexp(rows.amax(1).double())
    e = torch.clamp(torch.where(rows.amax(1) > 0, e - 1, -1000), min=top - 126)
    t = (rows.double() * torch.exp2((top - e).double())[:, None]).flatten()[:x.numel()]
    ex = torch.clamp(torch.frexp(t)[1] - 1, min=1 - bias)
    unit = torch.exp2((ex - mantissa).double())
    q = torch.floor(t / unit + random16.double() / 65536) * unit
    if keep_positive:
        q = torch.where(x > 0, torch.clamp(q, min=2.0 ** (1 - bias - mantissa)), q)
    return q, torch.exp2((e - top).double())


def check_step(before, after, step, lr, scale, seed):
    """Every tensor of the list against the formulas in 64 bits; 8-bit moments against the rounding of the fp32 values that the
    formulas' single operations give, which is exact."""
    first = 0
    c1, c2 = 1 - HYPER["beta1"] ** step, 1 - HYPER["beta2"] ** step
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    for old, new in zip(before, after):
        n = old["p"].numel()
        eight = "ms" in old
        g = old["g"].float().cpu() * torch.tensor(scale, dtype=F32)
        m0, v0 = (decoded(old[k], old[k + "s"]) if eight else old[k].double().cpu() for k in ("m", "v"))
        m32 = torch.tensor(b1, dtype=F32) * m0.float() + torch.tensor(1 - b1, dtype=F32) * g
        v32 = torch.tensor(b2, dtype=F32) * v0.float() + torch.tensor(1 - b2, dtype=F32) * (g * g)
        g = old["g"].double().cpu() * scale
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        # each constant, product and sum rounds once
        dm, dv = 4 * U * (b1 * m0.abs() + (1 - b1) * g.abs()), 6 * U * v
        within(m32, m, dm)
        within(v32, v, dv + 2.0 ** -148)
        if eight:
            r = random_bits(n, first, seed, step)
            for key, x, low in (("m", m32, False), ("v", v32, True)):
                q, s = encode(x.abs(), (r >> 16) if low else (r & 0xFFFF), 14 if low else 7, 2 if low else 3,
                              15 if low else 7, low)
                assert torch.equal(new[key + "s"].double().cpu(), s), key
                sign = torch.where(torch.signbit(x), -1.0, 1.0).double()
                assert torch.equal(new[key].double().cpu(), q * sign), key
            first += (n + 255) // 256
        else:
            assert torch.equal(new["m"].cpu(), m32) and torch.equal(new["v"].cpu(), v32)
        old_p = old["w" if "w" in old else "p"].double().cpu()
        root = torch.sqrt(v / c2) + HYPER["eps"]
        update = lr / c1 * m / root
        p = old_p * (1 - lr * HYPER["weight_decay"]) - update
        # m and v as above (v under the root), six constants and operations, a division good to two units
        tol = 4 * U * old_p.abs() + 24 * U * update.abs() + lr / c1 * dm / root
        within(new["w" if "w" in new else "p"], p, tol + (HALF[new["p"].dtype] * p.abs() if "w" not in new else U * p.abs()))
        if "w" in new:
            assert torch.equal(new["p"], new["w"].to(new["p"].dtype))


def snapshot(tensors):
    return [{k: v.clone() for k, v in t.items()} for t in tensors]


SIZES = [[1], [7, 8, 9], [256, 255, 257], [4096, 4095, 1, 0, 4097], [20000, 3, 8192 + 8, 511]]
KINDS = [(BF, BF, True), (BF, BF, False), (BF, F32, True), (BF, F32, False), (F32, F32, False), (F32, BF, False)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt,gt,master", KINDS, ids=["bf16_w", "bf16", "bf16_g32_w", "bf16_g32", "fp32", "fp32_g16"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_adamw_step(lib, cuda_dev, sizes, pt, gt, master, bits):
    tensors, buffers = adam_inputs(sizes, pt, gt, bits, master, cuda_dev, len(sizes))
    before = snapshot(tensors)
    scale = torch.tensor([0.37], device=cuda_dev)
    take_step(lib, tensors, step=3, lr=1e-2, scale=scale, seed=(5 << 32) + 9)
    check_step(before, tensors, 3, 1e-2, float(scale), (5 << 32) + 9)
    take_step(lib, tensors, step=4)  # and once more, from states that the operator wrote
    canaries_hold(buffers)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("lead", [[1], [8, 3, 0], [4]], ids=str)
def test_adamw_step_of_unaligned_tensors(lib, cuda_dev, lead, bits):
    tensors, buffers = adam_inputs([1000, 4099, 16, 9000], BF, BF, bits, True, cuda_dev, 4, lead=lead)
    before = snapshot(tensors)
    take_step(lib, tensors)
    check_step(before, tensors, 7, 1e-2, 1.0, 11)
    canaries_hold(buffers)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [48, 49, 400, 401, 850])
def test_adamw_step_of_long_lists(lib, cuda_dev, count, bits):
    """Around the capacities of a launch's table; random bits go on counting over the launches."""
    sizes = [(i * 37) % 600 for i in range(count)]
    tensors, buffers = adam_inputs(sizes, F32, F32, bits, False, cuda_dev, count)
    before = snapshot(tensors)
    take_step(lib, tensors)
    check_step(before, tensors, 7, 1e-2, 1.0, 11)
    canaries_hold(buffers)


@pytest.mark.parametrize("bits,pt,gt,master", [(8, BF, BF, True), (8, F32, F32, False), (8, BF, F32, False), (32, BF, F32, True)])
def test_adamw_step_of_tensors_that_go_round_every_block(lib, cuda_dev, bits, pt, gt, master):
    """More parts than the blocks of a launch have room for at once, whole and ragged and unaligned ones among them."""
    tensors, buffers = adam_inputs([6_000_013, 300_000, 2048 * 900, 77], pt, gt, bits, master, cuda_dev, 8, lead=[0, 1, 0, 0])
    before = snapshot(tensors)
    take_step(lib, tensors)
    check_step(before, tensors, 7, 1e-2, 1.0, 11)
    canaries_hold(buffers)


def test_adamw_8bit_second_moments_too_large_for_fp32_say_so(lib, cuda_dev):
    t = {"p": torch.ones(512), "g": torch.ones(512), "m": torch.zeros(512).to(torch.float8_e4m3fn),
         "v": torch.zeros(512).to(torch.float8_e5m2), "ms": torch.zeros(2), "vs": torch.zeros(2)}
    t["g"][5] = 1e25
    tensors = [{k: v.to(cuda_dev) for k, v in t.items()}]
    take_step(lib, tensors, step=1)
    assert bool(torch.isfinite(tensors[0]["p"]).all()) and torch.isnan(tensors[0]["vs"]).tolist() == [True, False]
    take_step(lib, tensors, step=2)
    assert bool(torch.isnan(tensors[0]["p"][:256]).all()) and bool(torch.isfinite(tensors[0]["p"][256:]).all())


def test_adamw_step_at_first_from_zero_state(lib, cuda_dev):
    for bits in (32, 8):
        tensors, _ = adam_inputs([1000], BF, BF, bits, True, cuda_dev, 1)
        for k in ("m", "v", "ms", "vs"):
            if k in tensors[0]:
                tensors[0][k].view(torch.uint8).zero_()
        tensors[0]["g"][::3] = 0
        before = snapshot(tensors)
        take_step(lib, tensors, step=1)
        check_step(before, tensors, 1, 1e-2, 1.0, 11)
        # an element without a gradient so far has no moments and only decays
        assert not tensors[0]["m"][::3].float().any() and not tensors[0]["v"][::3].float().any()


def test_adamw_step_with_a_scale_that_is_not_finite_changes_nothing(lib, cuda_dev):
    for bits in (32, 8):
        for bad in (float("nan"), float("inf")):
            tensors, _ = adam_inputs([700, 3], BF, BF, bits, True, cuda_dev, 1)
            before = snapshot(tensors)
            take_step(lib, tensors, scale=torch.tensor([bad], device=cuda_dev))
            for old, new in zip(before, tensors):
                assert all(torch.equal(old[k].view(torch.uint8), new[k].view(torch.uint8)) for k in old)


def test_adamw_8bit_blocks_with_bad_gradients_say_so(lib, cuda_dev):
    tensors, _ = adam_inputs([1024], BF, BF, 8, True, cuda_dev, 1)
    good, _ = adam_inputs([1024], BF, BF, 8, True, cuda_dev, 1)
    tensors[0]["g"][300], tensors[0]["g"][700] = float("nan"), float("inf")
    take_step(lib, tensors)
    take_step(lib, good)
    for k in ("ms", "vs"):
        assert torch.isnan(tensors[0][k]).tolist() == [False, True, True, False]
        assert torch.equal(tensors[0][k][[0, 3]], good[0][k][[0, 3]])
    bad = torch.isnan(tensors[0]["w"])
    assert bad.nonzero().flatten().tolist() == [300, 700]
    assert torch.equal(tensors[0]["w"][~bad], good[0]["w"][~bad])
    take_step(lib, tensors, step=8)  # the blocks stay bad, the others go on
    take_step(lib, good, step=8)
    assert torch.isnan(tensors[0]["ms"]).tolist() == [False, True, True, False]
    assert torch.equal(tensors[0]["w"][:256], good[0]["w"][:256])


def test_adamw_8bit_extremes(lib, cuda_dev):
    """Blocks of one large and many small values, of the smallest and largest numbers, of zeros."""
    g = torch.Generator().manual_seed(6)
    grads = torch.randn(6 * 256, generator=g)
    grads[:256] *= 1e-6
    grads[17] = 1e3
    grads[256:512] *= 2.0 ** -60
    grads[512:768] = 0.0
    grads[768:1024] *= 1e15
    grads[1024:1280] = torch.sign(grads[1024:1280]) * 2.0 ** -130
    tensors = [{"p": torch.randn(6 * 256, generator=g), "g": grads, "m": torch.zeros(6 * 256).to(torch.float8_e4m3fn),
                "v": torch.zeros(6 * 256).to(torch.float8_e5m2), "ms": torch.zeros(6), "vs": torch.zeros(6)}]
    tensors = [{k: v.to(cuda_dev) for k, v in tensors[0].items()}]
    for step in (1, 2, 3):
        before = snapshot(tensors)
        take_step(lib, tensors, step=step)
        new = tensors[0]
        assert bool(torch.isfinite(new["p"]).all()) and bool(torch.isfinite(new["ms"]).all())
        r = random_bits(6 * 256, 0, 11, step)
        gg = grads
        m32 = torch.tensor(0.9, dtype=F32) * decoded(before[0]["m"], before[0]["ms"]).float() + torch.tensor(0.1, dtype=F32) * gg
        v32 = (torch.tensor(0.999, dtype=F32) * decoded(before[0]["v"], before[0]["vs"]).float()
               + torch.tensor(1 - 0.999, dtype=F32) * (gg * gg))
        q, s = encode(v32, r >> 16, 14, 2, 15, True)
        assert torch.equal(new["vs"].double().cpu(), s) and torch.equal(new["v"].double().cpu(), q)
        keep = torch.ones(6 * 256, dtype=torch.bool)
        keep[1024:1280] = False  # below the smallest scale the first moment's units are below fp32's own
        q, s = encode(m32.abs(), r & 0xFFFF, 7, 3, 7, False)
        assert torch.equal(new["ms"].double().cpu(), s)
        assert torch.equal(new["m"].double().cpu()[keep], (q * torch.where(torch.signbit(m32), -1.0, 1.0).double())[keep])
        positive = v32 > 0
        assert bool((new["v"].float().cpu()[positive] > 0).all())


@pytest.mark.parametrize("count", [1, 3000])  # one wave of blocks, and the ring
def test_adamw_8bit_first_moments_up_to_the_largest(lib, cuda_dev, count):
    """First moments of every size up to fp32's largest, small ones beside them: the rounding of the formula's fp32 value, exactly."""
    powers = torch.arange(-20, 120, 4)
    n = 256 * len(powers) * count
    g = torch.Generator().manual_seed(count)
    scales = torch.exp2(powers.float()).repeat(count)
    codes = torch.randn(n, generator=g).clamp(-3.5, 3.5) * 2.0 ** torch.randint(-6, 7, (n,), generator=g)
    codes[::256] = 255.0  # each block's largest, which a stochastic rounding takes up or down
    t = {"p": torch.zeros(n), "g": torch.randn(n, generator=g), "m": codes.to(torch.float8_e4m3fn), "ms": scales,
         "v": torch.full((n,), 2.0 ** 14).to(torch.float8_e5m2), "vs": torch.ones(n // 256)}
    tensors = [{k: v.to(cuda_dev) for k, v in t.items()}]
    before = snapshot(tensors)
    take_step(lib, tensors, step=5)
    new = tensors[0]
    m32 = torch.tensor(0.9, dtype=F32) * decoded(before[0]["m"], before[0]["ms"]).float() + torch.tensor(0.1, dtype=F32) * t["g"]
    q, s = encode(m32.abs(), random_bits(n, 0, 11, 5) & 0xFFFF, 7, 3, 7, False)
    assert torch.equal(new["ms"].double().cpu(), s)
    got, want = new["m"].double().cpu(), q * torch.where(torch.signbit(m32), -1.0, 1.0).double()
    # Below the 8-bit type's normal numbers, 2^-6 of the scale, the kernel's scaled value is an fp32 subnormal: its last bit is
    # 2^(-149 + 120) = 2^-29 of the scale, 2^-20 of the unit 2^-9 there, so that the product that scales it is off by 2^-21 of a
    # unit at most.  Where value and random bits together come so close to a whole unit they may go either way.
    units = m32.double().abs() / s.repeat_interleave(256) * 512
    near = units + (random_bits(n, 0, 11, 5) & 0xFFFF).double() / 65536
    either = (units < 8) & ((near - near.round()).abs() <= 2.0 ** -21)
    bad = ((got != want) & ~either).nonzero().flatten()
    assert not len(bad), (len(bad), float(m32[bad[0]]), float(got[bad[0]]), float(want[bad[0]]))
    assert bool(((got - want).abs() <= 2.0 ** -9)[either].all()) and int(either.sum()) < n // 2 ** 16 + 2


def test_adamw_8bit_rounding_is_right_on_average(lib, cuda_dev):
    """65536 equal values between two units: the mean is that value, to five times the standard error of a mean of
    independent roundings (at most half a unit each) and the 2^-16 that sixteen bits resolve."""
    n = 1 << 16
    grads = torch.full((n,), 0.7)
    grads[::256] = 1.0  # fixes the blocks' scales
    t = {"p": torch.zeros(n), "g": grads, "m": torch.zeros(n).to(torch.float8_e4m3fn),
         "v": torch.zeros(n).to(torch.float8_e5m2), "ms": torch.zeros(n // 256), "vs": torch.zeros(n // 256)}
    for seed in (0, 1, 123456789):
        tensors = [{k: v.to(cuda_dev) for k, v in t.items()}]
        take_step(lib, tensors, step=1, seed=seed)
        plain = torch.ones(n, dtype=torch.bool)
        plain[::256] = False
        for key, want, mantissa in (("m", 0.1 * 0.7, 3), ("v", 0.001 * 0.49, 2)):
            unit = 2.0 ** (math.floor(math.log2(want)) - mantissa)
            got = decoded(tensors[0][key], tensors[0][key + "s"])[plain]
            assert len(torch.unique(got)) == 2
            assert abs(float(got.mean()) - want) <= 5 * 0.5 * unit / math.sqrt(n) + unit * 2.0 ** -15


def test_adamw_8bit_second_moment_follows_the_32bit_one(lib, cuda_dev):
    """Where the nearest rounding would leave it standing: after gradients ten times smaller for 1500 steps of beta2 = 0.999 the
    mean over many elements has come down as the 32-bit average has (to 1/20: the rounding's random walk is unbiased, with a
    spread of at most half the value for an element, over 2048 elements)."""
    n = 2048
    g = torch.Generator().manual_seed(0)
    both = []
    for bits in (32, 8):
        t = {"p": torch.zeros(n), "g": torch.ones(n), **({"m": torch.zeros(n), "v": torch.full((n,), 100.0)} if bits == 32 else
             {"m": torch.zeros(n).to(torch.float8_e4m3fn), "v": torch.full((n,), 25600.0).to(torch.float8_e5m2),
              "ms": torch.ones(n // 256), "vs": torch.full((n // 256,), 2.0 ** -8)})}
        both.append([{k: v.to(cuda_dev) for k, v in t.items()}])
    start = float(decoded(both[1][0]["v"], both[1][0]["vs"]).mean())
    both[0][0]["v"].fill_(start)
    grads = torch.randn((64, n), generator=g).abs().add_(0.5).to(cuda_dev)
    for step in range(1, 1501):
        for tensors in both:
            tensors[0]["g"].copy_(grads[step % 64])
            take_step(lib, tensors, step=step, lr=0.0)
    want, got = both[0][0]["v"].double().mean().item(), decoded(both[1][0]["v"], both[1][0]["vs"]).mean().item()
    assert want < 0.5 * start and abs(got - want) <= want / 20


def test_adamw_learning_rate_and_step_on_the_device_in_a_replayed_graph(lib, cuda_dev):
    for bits in (32, 8):
        tensors, _ = adam_inputs([5000, 77], BF, BF, bits, True, cuda_dev, 2)
        eager = snapshot(tensors)
        lr = torch.tensor([1e-2], device=cuda_dev)
        step = torch.tensor([0], dtype=torch.int64, device=cuda_dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step.add_(1)
            take_step(lib, tensors, step=0, lr=0.0, lr_tensor=lr, step_tensor=step)
        for t in (1, 2, 3, 2000):
            lr.fill_(1e-2 / t)
            step.fill_(t - 1)
            graph.replay()
            before = snapshot(eager)
            take_step(lib, eager, step=t, lr=1e-2 / t)
            for old, a, b in zip(before, tensors, eager):
                for k in old:
                    if k in ("w", "p"):
                        # constants rounded to fp32 on either side: eight units of the update, and the learning rate's own
                        moved = (old["w"].double() - b["w"].double()).abs()
                        within(a["w"], b["w"], (16 * U * moved + 2 * U * old["w"].double().abs()).cpu())
                        a["w"].copy_(b["w"])
                        a["p"].copy_(b["p"])
                    else:
                        assert torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)), k


def test_adamw_is_deterministic_on_any_stream(lib, cuda_dev):
    for bits in (32, 8):
        runs = []
        for s in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
            tensors, _ = adam_inputs([30000, 513], BF, F32, bits, True, cuda_dev, 2)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                take_step(lib, tensors)
                take_step(lib, tensors, step=8)
            runs.append(tensors)
        torch.cuda.synchronize()
        for other in runs[1:]:
            for a, b in zip(runs[0], other):
                assert all(torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)) for k in a)


def test_adamw_offsets_past_32_bits(lib, cuda_dev):
    """A tensor of more than 2^31 elements: its last ones are stepped as a short tensor's are."""
    n = (1 << 31) + 4096 + 5
    t = {"p": torch.zeros(n, dtype=BF, device=cuda_dev), "g": torch.zeros(n, dtype=BF, device=cuda_dev),
         "m": torch.zeros(n, dtype=torch.uint8, device=cuda_dev).view(torch.float8_e4m3fn),
         "v": torch.zeros(n, dtype=torch.uint8, device=cuda_dev).view(torch.float8_e5m2),
         "ms": torch.zeros((n + 255) // 256, device=cuda_dev), "vs": torch.zeros((n + 255) // 256, device=cuda_dev)}
    t["p"][-300:], t["g"][-300:] = 1.0, 0.5
    take_step(lib, [t], step=1)
    torch.cuda.synchronize()
    assert not t["p"][:1 << 20].any() and not t["v"][:1 << 20].view(torch.uint8).any()
    assert bool((t["p"][-300:].float() - (1 - 1e-3 - 1e-2)).abs().max() <= 2.0 ** -8)
    tail = t["v"][-300:].float() * t["vs"][-(300 + 255) // 256 - 1:].max()
    assert bool(((tail - 0.00025).abs() <= 0.00025 / 4).all())


def test_adamw_refusals(lib, cuda_dev):
    def lists(bits=32, n=64, **other):
        t = {"p": torch.zeros(n, dtype=BF, device=cuda_dev), "g": torch.zeros(n, dtype=BF, device=cuda_dev),
             "m": torch.zeros(n, device=cuda_dev), "v": torch.zeros(n, device=cuda_dev), **other}
        return [{k: v for k, v in t.items() if v is not None}]

    a = lists()[0]
    with pytest.raises(RuntimeError, match="status -1"):  # the same parameter twice
        take_step(lib, [a, dict(lists()[0], p=a["p"])])
    with pytest.raises(RuntimeError, match="status -1"):  # moments that overlap
        wide = torch.zeros(100, device=cuda_dev)
        take_step(lib, [dict(lists()[0], m=wide[30:94]), dict(lists()[0], m=wide[:64])])
    with pytest.raises(RuntimeError, match="contiguous"):
        take_step(lib, lists(p=torch.zeros(128, dtype=BF, device=cuda_dev)[::2]))
    with pytest.raises(RuntimeError, match="as many elements"):
        take_step(lib, lists(g=torch.zeros(63, dtype=BF, device=cuda_dev)))
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        take_step(lib, lists(p=torch.zeros(64, dtype=torch.float16, device=cuda_dev)))
    with pytest.raises(RuntimeError, match="exp_avg_sqs must all be"):
        take_step(lib, lists(v=torch.zeros(64, dtype=BF, device=cuda_dev)))
    with pytest.raises(RuntimeError, match="scales"):
        take_step(lib, lists(ms=torch.zeros(1, device=cuda_dev)))
    with pytest.raises(RuntimeError, match="one tensor for each parameter"):
        take_step(lib, lists(m=torch.zeros(64, device=cuda_dev).to(torch.float8_e4m3fn),
                             v=torch.zeros(64, device=cuda_dev).to(torch.float8_e5m2)))
    with pytest.raises(RuntimeError, match="each 256"):
        take_step(lib, lists(m=torch.zeros(64, device=cuda_dev).to(torch.float8_e4m3fn),
                             v=torch.zeros(64, device=cuda_dev).to(torch.float8_e5m2), ms=torch.zeros(2, device=cuda_dev),
                             vs=torch.zeros(1, device=cuda_dev)))
    with pytest.raises(RuntimeError, match="masters go with"):
        take_step(lib, lists(p=torch.zeros(64, device=cuda_dev), w=torch.zeros(64, device=cuda_dev)))
    with pytest.raises(RuntimeError, match="device of the parameters"):
        take_step(lib, lists(g=torch.zeros(64, dtype=BF)))
    with pytest.raises(RuntimeError, match="one Float element"):
        take_step(lib, lists(), scale=torch.ones(2, device=cuda_dev))
    for bad in (dict(step=0), dict(lr=-1.0), dict(lr=float("nan"))):
        with pytest.raises(RuntimeError, match="status -1"):
            take_step(lib, lists(), **bad)
    lib.adamw_step([], [], [], [], 1, 1e-3)  # nothing to do


# ---------------------------------------------------------------- gradient norm

@pytest.mark.parametrize("sizes", [[1], [7, 0, 9], [4096, 4097, 3], [100003], [5] * 49, [33] * 900, [0]], ids=lambda s: f"{len(s)}x{s[0]}")
def test_grad_norm_clip(lib, cuda_dev, sizes):
    g = torch.Generator().manual_seed(len(sizes))
    grads = [(torch.randn(n + 3, generator=g) * 3).to(BF if i % 2 else F32).to(cuda_dev)[i % 3:][:n] for i, n in enumerate(sizes)]
    want = math.sqrt(sum(float(v.double().square().sum()) for v in grads))
    for max_norm in (0.5, 1e9, 0.0):
        out = lib.grad_norm_clip(grads, max_norm)
        # 16 squares a thread of a chunk, summed in fp32, halved by the root; one rounding at the end
        assert abs(float(out[0]) - want) <= (17 / 2 + 1) * U * want
        factor = min(1.0, max_norm / (want + 1e-6))
        assert abs(float(out[1]) - factor) <= (17 / 2 + 2) * U * factor


def test_grad_norm_of_values_that_are_not_finite(lib, cuda_dev):
    g = torch.ones(5000, device=cuda_dev)
    for bad in (float("nan"), float("inf"), 3e38):
        g[4321] = bad
        out = lib.grad_norm_clip([g], 1.0)
        assert not math.isfinite(float(out[0])) and math.isnan(float(out[1]))
    assert lib.grad_norm_clip([torch.zeros(9, device=cuda_dev)], 1.0).tolist() == [0.0, 1.0]
    with pytest.raises(RuntimeError, match="not be empty"):
        lib.grad_norm_clip([], 1.0)
    with pytest.raises(RuntimeError, match="status -1"):
        lib.grad_norm_clip([g], -1.0)
    with pytest.raises(RuntimeError, match="contiguous"):
        lib.grad_norm_clip([g[::2]], 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        lib.grad_norm_clip([g.cpu()], 1.0)


def test_grad_norm_is_deterministic_and_runs_twice_at_once(lib, cuda_dev):
    g = [torch.randn(1_000_003, device=cuda_dev), torch.randn(777, device=cuda_dev).to(BF)]
    want = lib.grad_norm_clip(g, 1.0)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(4)]:
        with torch.cuda.stream(s):
            got += [lib.grad_norm_clip(g, 1.0) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got)


def test_grad_norm_of_few_and_many_chunks(lib, cuda_dev):
    """Around the sizes where one cluster gives way to a grid over the device: one large tensor, many small ones."""
    g = torch.Generator().manual_seed(8)
    for k, n in ((1, 24 * 8192), (1, 24 * 8192 + 1), (1, 8 * 8192), (24, 3), (25, 3), (12, 8193), (13, 8193), (48, 1), (49, 1)):
        grads = [torch.randn(n, generator=g).to(BF if i % 2 else F32).to(cuda_dev) for i in range(k)]
        want = math.sqrt(sum(float(v.double().square().sum()) for v in grads))
        out = lib.grad_norm_clip(grads, 0.5)
        # 16 squares a thread of a chunk, summed in fp32, halved by the root; one rounding at the end
        assert abs(float(out[0]) - want) <= (17 / 2 + 1) * U * want
        factor = min(1.0, 0.5 / (want + 1e-6))
        assert abs(float(out[1]) - factor) <= (17 / 2 + 2) * U * factor


@pytest.mark.parametrize("t", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n", [9, 5000, 400_003])
def test_grad_norm_of_values_whose_squares_leave_fp32(lib, cuda_dev, n, t):
    """Down to the smallest fp32 values: sixteen squares are summed in fp32, scaled by a power of two where they are below its
    normal numbers, which adds no rounding: (17 / 2 + 1) u as elsewhere.  The norm is an fp32 value: half a unit more, in absolute
    terms, below the smallest normal one."""
    g = torch.Generator().manual_seed(n)
    values = torch.randn(n, generator=g)
    for size in (1e-18, 1e-20, 3e-23, 1e-25, 1e-32, 1e-38, 1e-41, 0.0):
        for mixed in (False, True):
            v = (values * size).to(t)
            if mixed:
                v[:: 7919 if n > 9 else 4] = 1e-14
            want = math.sqrt(float(v.double().square().sum()))
            for grads in ([v], [v[: n // 2].clone(), v[n // 2:].clone()]):
                out = lib.grad_norm_clip([q.to(cuda_dev) for q in grads], 1e-30)
                assert abs(float(out[0]) - want) <= (17 / 2 + 1) * U * want + 2.0 ** -150, (size, mixed, float(out[0]), want)
                factor = min(1.0, 1e-30 / (want + 1e-6))
                assert abs(float(out[1]) - factor) <= (17 / 2 + 3) * U * factor
