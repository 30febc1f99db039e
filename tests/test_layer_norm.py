"""Layer norm, its gradient and the 8-bit rows kept between the two: against the formulas in 64 bits and against differences."""
import pytest
import torch

from graphnn_b200 import capi

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24   # half a step of fp32
# one row and several; widths around every form's limits, odd ones (no row but the first aligned), and rows longer than registers hold
SHAPES = [(1, 1), (3, 2), (5, 7), (64, 128), (33, 31), (2, 256), (7, 264), (9, 129), (4, 513), (6, 1021), (5, 1024), (3, 2048), (11, 4096), (3, 4100), (2, 8192), (300, 40), (2, 8200), (3, 16384), (2, 16392), (2, 20001),
          (1, 70000), (700, 96),
          # many rows of each CTA: stages and sums in turn
          (9001, 128), (6000, 1032), (3001, 2048), (2500, 4096), (1300, 8192), (700, 16384), (1500, 1001)]


def depth(cols):
    """Most roundings that a number on its way into a row's sum meets: a thread's own elements one by one (64, or its share of a row too long for the
    registers), five exchanges in a warp and up to 16 warps after it, three roundings each."""
    return max(64, cols / 256 + 64) + 3 * 21


def numbers(shape, dtype, seed, scale=1.0, offset=0.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale + offset).to(TYPES[dtype])


def spaced(x, extra, lead=0):
    """The same matrix with `extra` numbers behind each row and `lead` in front of the first, and the buffer around it."""
    rows, cols = x.shape
    base = torch.full((rows * (cols + extra) + lead + extra,), 5, dtype=x.dtype, device=x.device)
    view = torch.as_strided(base, (rows, cols), (cols + extra, 1), lead)
    view.copy_(x)
    return view, base


def untouched(base, view, value=5):
    mask = torch.ones_like(base, dtype=torch.bool)
    torch.as_strided(mask, view.shape, view.stride(), view.storage_offset()).fill_(False)
    return bool((base[mask] == value).all())


def normalised(x, eps):
    x = x.double()
    var, mean = torch.var_mean(x, dim=1, correction=0)
    return mean, 1.0 / torch.sqrt(var + eps)


def check_forward(x, weight, bias, eps, y, stats):
    cols = x.shape[1]
    mean, rstd = normalised(x, eps)
    h = (x.double() - mean[:, None]) * rstd[:, None]
    w = torch.ones(cols, dtype=torch.float64, device="cuda") if weight is None else weight.double()
    b = torch.zeros(cols, dtype=torch.float64, device="cuda") if bias is None else bias.double()
    want = h * w + b
    d, big = depth(cols), x.double().abs().amax(dim=1)
    # the mean is off by the roundings of its sum; squared deviations by twice that many; two of the subtraction, two products and a sum behind them
    mean_tol = U * d * big
    rel = U * (d + 8)                       # of rstd, and of h next to what the mean's error leaves in it
    tol_h = rstd[:, None] * (mean_tol[:, None] + U * big[:, None]) + h.abs() * (rel + 4 * U)
    # (with hardly any deviation, the mean's own error is part of the deviations)
    tol_h = tol_h + h.abs() * (rstd * mean_tol)[:, None] ** 2
    tol = tol_h * w.abs() + 2 * U * (h * w).abs() + torch.finfo(x.dtype).eps / 2 * want.abs() + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    tol = tol * (1 + torch.finfo(x.dtype).eps)
    err = (y.double() - want).abs()
    assert bool((err <= tol).all()), f"off by up to {float((err / tol).max()):.3g} of the tolerance"
    if stats is not None:
        assert bool(((stats[:, 0].double() - mean).abs() <= mean_tol + 1e-45).all())
        assert bool(((stats[:, 1].double() - rstd).abs() <= rstd * (rel + 4 * U + (rstd * mean_tol) ** 2)).all())


def check_grad(dy, x, stats, weight, dx, dweight, dbias):
    """x: what the rows are taken to be (8-bit rows times their scales), in 64 bits."""
    rows, cols = dy.shape
    mean, rstd = stats.double()[:, :1], stats.double()[:, 1:]
    h = (x - mean) * rstd
    d = dy.double()
    g = d * (1.0 if weight is None else weight.double())
    m0, m1 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    want = rstd * (g - m0 - h * m1)
    eps, n = torch.finfo(dy.dtype).eps, depth(cols)
    h_tol = 3 * U * h.abs() + U * rstd * x.abs()       # subtraction (fused with the scale's product for 8-bit rows) and product
    tol = rstd * ((n + 4) * U * (g.abs().mean(1, keepdim=True) + h.abs() * (g * h).abs().mean(1, keepdim=True)) + h_tol * m1.abs() + h.abs() * (g.abs() * h_tol).mean(1, keepdim=True) + 4 * U * (g.abs() + m0.abs() + (h * m1).abs()))
    tol = (tol + 2 * U * want.abs()) * (1 + eps) + eps / 2 * want.abs() + torch.finfo(dy.dtype).smallest_normal * eps
    err = (dx.double() - want).abs()
    assert bool((err <= tol).all()), f"dx off by up to {float((err / tol).max()):.3g} of the tolerance"
    # column sums: a rounding for each row, at most, and 1024 lines and 8 shares behind them
    steps = rows + min(rows, 1024) / 8 + 16
    if dweight is not None:
        err, tol = (dweight.double() - (d * h).sum(0)).abs(), U * (steps + 2) * (d * h).abs().sum(0) + (d.abs() * h_tol).sum(0) + 1e-45
        assert bool((err <= tol).all()), f"dweight off by up to {float((err / tol).max()):.3g} of the tolerance"
    if dbias is not None:
        err, tol = (dbias.double() - d.sum(0)).abs(), U * steps * d.abs().sum(0) + 1e-45
        assert bool((err <= tol).all()), f"dbias off by up to {float((err / tol).max()):.3g} of the tolerance"


def integers(ctx, x):
    q, s = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(x.shape[0], device="cuda")
    ctx.quantize_rows_i8(x, q, s)
    return q, s


def workspace(ctx, rows, cols):
    return torch.empty(max(16, ctx.layer_norm_grad_workspace_bytes(rows, cols)), dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------- without a GPU
@pytest.fixture
def recorded():
    """A context whose calls are written down instead of made, for tensors that say they are on its device."""
    ctx = capi.Context.__new__(capi.Context)
    ctx.h, ctx.device, ctx.lib = None, -1, capi.load_library()   # (torch gives -1 as the device of CPU tensors)
    ctx.made = []
    ctx.call = lambda name, *a: ctx.made.append((name, a))
    return ctx


def test_workspace_sizes_without_a_gpu():
    lib = capi.load_library()
    assert lib.s2v_layer_norm_grad_workspace_bytes(0, 8) == 0 and lib.s2v_layer_norm_grad_workspace_bytes(8, 0) == 0
    assert lib.s2v_layer_norm_grad_workspace_bytes(-1, 8) == 0 and lib.s2v_layer_norm_grad_workspace_bytes(4, 1 << 40) == 0
    assert lib.s2v_layer_norm_grad_workspace_bytes(3, 100) >= 3 * 2 * 100 * 4
    assert lib.s2v_layer_norm_grad_workspace_bytes(1 << 40, 100) <= 1024 * 2 * 100 * 4     # does not grow with the rows for good


def test_binding_refuses_what_the_library_cannot_see(recorded):
    x, v = torch.zeros(4, 6), torch.zeros(6)
    q, s, st = torch.zeros(4, 6, dtype=torch.int8), torch.zeros(4), torch.zeros(4, 2)
    recorded.layer_norm(x, x.clone(), weight=v, bias=v, stats=st, q=q, q_scale=s)
    recorded.layer_norm_grad(x, st, x.clone(), torch.zeros(64), x=x, weight=v, dweight=v.clone(), dbias=v.clone())
    recorded.layer_norm_grad(x, st, x.clone(), q=q, q_scale=s)
    assert [n for n, _ in recorded.made] == ["s2v_layer_norm", "s2v_layer_norm_grad", "s2v_layer_norm_grad"]
    assert recorded.made[2][1][13:15] == (None, 0)
    half = x.half()
    for make in (lambda: recorded.layer_norm(x, half), lambda: recorded.layer_norm(x, x.t()), lambda: recorded.layer_norm(x, x.clone(), weight=v[:5]),
                 lambda: recorded.layer_norm(x, x.clone(), bias=v.double()), lambda: recorded.layer_norm(x, x.clone(), stats=torch.zeros(4, 3)),
                 lambda: recorded.layer_norm(x, x.clone(), stats=torch.zeros(2, 4).t()), lambda: recorded.layer_norm(x, x.clone(), q=q), lambda: recorded.layer_norm(x, x.clone(), q=q.float(), q_scale=s),
                 lambda: recorded.layer_norm(x.double(), x.double()), lambda: recorded.layer_norm(x[0], x[0]),
                 lambda: recorded.layer_norm_grad(x, st, x.clone()), lambda: recorded.layer_norm_grad(x, st, x.clone(), x=x, q=q, q_scale=s), lambda: recorded.layer_norm_grad(x, st, x.clone(), q=q),
                 lambda: recorded.layer_norm_grad(x, None, x.clone(), x=x), lambda: recorded.layer_norm_grad(x, st, half, x=x), lambda: recorded.layer_norm_grad(x, st, x.clone(), x=x, dbias=v[::2])):
        with pytest.raises(capi.S2VError):
            make()
    assert len(recorded.made) == 3


# ---------------------------------------------------------------- values
@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_norm_and_gradients(gpu_ctx, shape, dtype):
    rows, cols = shape
    x, dy = numbers(shape, dtype, 1, 2.0, 0.7), numbers(shape, dtype, 2)
    weight, bias = numbers((cols,), "f32", 3, 0.3, 1.0), numbers((cols,), "f32", 4, 0.2)
    y, stats = torch.empty_like(x), torch.empty((rows, 2), device="cuda")
    q, s = torch.empty(shape, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    ws = workspace(gpu_ctx, rows, cols)
    dx, dx8, dw, db, dw8, db8 = torch.empty_like(x), torch.empty_like(x), *(torch.empty(cols, device="cuda") for _ in range(4))
    torch.cuda.synchronize()
    gpu_ctx.layer_norm(x, y, weight, bias, 1e-5, stats, q, s)
    gpu_ctx.layer_norm_grad(dy, stats, dx, ws, x=x, weight=weight, dweight=dw, dbias=db)
    gpu_ctx.layer_norm_grad(dy, stats, dx8, ws, q=q, q_scale=s, weight=weight, dweight=dw8, dbias=db8)
    want_q, want_s = integers(gpu_ctx, x)
    gpu_ctx.synchronize()
    assert torch.equal(q, want_q) and torch.equal(s, want_s)     # the same 8-bit rows as the quantiser's
    check_forward(x, weight, bias, 1e-5, y, stats)
    check_grad(dy, x.double(), stats, weight, dx, dw, db)
    check_grad(dy, q.double() * s.double()[:, None], stats, weight, dx8, dw8, db8)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("extra,lead", [(8, 0), (3, 0), (8, 1), (16, 8)])
@pytest.mark.parametrize("cols", [24, 136, 1000, 4096, 9000])
def test_rows_anywhere_and_nothing_else_written(gpu_ctx, cols, extra, lead, dtype):
    rows = 5
    x, xb = spaced(numbers((rows, cols), dtype, 5, 3.0), extra, lead)
    dy, _ = spaced(numbers((rows, cols), dtype, 6), extra, lead)
    y, yb = spaced(torch.zeros_like(x), extra, lead)
    dx, dxb = spaced(torch.zeros_like(x), extra, lead)
    q, qb = spaced(torch.zeros((rows, cols), dtype=torch.int8, device="cuda"), extra, lead)
    s, stats = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda")
    wide = numbers((cols + 1,), "f32", 7, 0.3, 1.0)
    weight = wide[1:]                                             # on no 16-byte boundary
    ws, dw, db = workspace(gpu_ctx, rows, cols), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.layer_norm(x, y, weight, None, 1e-3, stats, q, s)
    gpu_ctx.layer_norm_grad(dy, stats, dx, ws, x=x, weight=weight, dweight=dw, dbias=db)
    gpu_ctx.synchronize()
    check_forward(x, weight, None, 1e-3, y, stats)
    check_grad(dy, x.double(), stats, weight, dx, dw, db)
    for base, view in ((yb, y), (dxb, dx), (qb, q), (xb, x)):
        assert untouched(base, view)
    gpu_ctx.layer_norm_grad(dy, stats, dx, ws, q=q, q_scale=s, weight=weight, dweight=dw, dbias=db)
    gpu_ctx.synchronize()
    check_grad(dy, q.double() * s.double()[:, None], stats, weight, dx, dw, db)
    assert untouched(dxb, dx)
    # one output on another boundary than its input
    y2 = torch.empty(rows * cols + 1, dtype=x.dtype, device="cuda")[1:].view(rows, cols)
    torch.cuda.synchronize()
    gpu_ctx.layer_norm(x, y2, weight, None, 1e-3)
    gpu_ctx.synchronize()
    check_forward(x, weight, None, 1e-3, y2, None)


@gpu
@pytest.mark.parametrize("shape", [(40, 96), (3, 1024), (2, 5000), (2, 20000)], ids=str)
def test_without_weight_in_place_and_single_sums(gpu_ctx, shape):
    rows, cols = shape
    for dtype in TYPES:
        x, dy = numbers(shape, dtype, 8, 1.0, -3.0), numbers(shape, dtype, 9)
        stats, ws, db = torch.empty((rows, 2), device="cuda"), workspace(gpu_ctx, rows, cols), torch.empty(cols, device="cuda")
        y, dx, dw = x.clone(), dy.clone(), torch.full((cols,), 5.0, device="cuda")
        torch.cuda.synchronize()
        gpu_ctx.layer_norm(y, y, stats=stats)
        gpu_ctx.layer_norm_grad(dx, stats, dx, ws, x=x, dbias=db)
        gpu_ctx.synchronize()
        check_forward(x, None, None, 1e-5, y, stats)
        check_grad(dy, x.double(), stats, None, dx, None, db)
        dx2 = torch.empty_like(dy)
        torch.cuda.synchronize()
        gpu_ctx.layer_norm_grad(dy, stats, dx2, x=x)                   # neither sum: no workspace
        gpu_ctx.layer_norm_grad(dy, stats, torch.empty_like(dy), ws, x=x, dweight=dw)
        gpu_ctx.synchronize()
        assert torch.equal(dx, dx2)
        check_grad(dy, x.double(), stats, None, dx2, dw, None)


@gpu
def test_rows_far_from_zero_keep_their_deviations(gpu_ctx):
    # deviations of 1 around 10,000: E x^2 - (E x)^2 would leave none of them in fp32
    for cols in (96, 1024, 6000, 20000):
        x = numbers((4, cols), "f32", 10, 1.0, 1e4)
        y, stats = torch.empty_like(x), torch.empty((4, 2), device="cuda")
        torch.cuda.synchronize()
        gpu_ctx.layer_norm(x, y, stats=stats)
        gpu_ctx.synchronize()
        check_forward(x, None, None, 1e-5, y, stats)
        assert abs(float(y.std()) - 1) < 0.1


@gpu
def test_rows_that_are_no_numbers_stay_by_themselves(gpu_ctx):
    for cols in (40, 128, 700, 5000, 20000):
        x, dy = numbers((6, cols), "f32", 11), numbers((6, cols), "f32", 12)
        clean = x.clone()
        x[1, 3], x[3, cols - 1], x[4] = float("nan"), float("inf"), 2.5
        y, stats, s, q = torch.empty_like(x), torch.empty((6, 2), device="cuda"), torch.empty(6, device="cuda"), torch.empty((6, cols), dtype=torch.int8, device="cuda")
        torch.cuda.synchronize()
        gpu_ctx.layer_norm(x, y, None, None, 1e-5, stats, q, s)
        gpu_ctx.synchronize()
        assert bool(y[1].isnan().all()) and bool(y[3].isnan().all()) and bool(s[[1, 3]].isnan().all()) and not q[[1, 3]].any()
        assert not y[4].any() and abs(float(stats[4, 1]) - 1e5 ** 0.5) < 1e-3      # equal numbers: 1 / sqrt(eps)
        keep = [0, 2, 5]
        check_forward(clean[keep], None, None, 1e-5, y[keep], stats[keep])
        dx, dw = torch.empty_like(x), torch.empty(cols, device="cuda")
        torch.cuda.synchronize()
        gpu_ctx.layer_norm_grad(dy, stats, dx, workspace(gpu_ctx, 6, cols), x=x, dweight=dw)
        gpu_ctx.synchronize()
        assert bool(dx[[1, 3]].isnan().all()) and bool(dx[[0, 2, 4, 5]].isfinite().all())


@gpu
def test_gradients_against_differences(gpu_ctx):
    rows, cols, h = 6, 48, 1e-4
    x, weight, bias, up = numbers((rows, cols), "f32", 13), numbers((cols,), "f32", 14, 0.3, 1.0), numbers((cols,), "f32", 15), numbers((rows, cols), "f32", 16)
    stats, y, dx, dw, db = torch.empty((rows, 2), device="cuda"), torch.empty_like(x), torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.layer_norm(x, y, weight, bias, 1e-5, stats)
    gpu_ctx.layer_norm_grad(up, stats, dx, workspace(gpu_ctx, rows, cols), x=x, weight=weight, dweight=dw, dbias=db)
    gpu_ctx.synchronize()

    def value(x, weight, bias):
        mean, rstd = normalised(x, 1e-5)
        return float((((x - mean[:, None]) * rstd[:, None] * weight + bias) * up.double()).sum())
    base = [x.double(), weight.double(), bias.double()]
    for which, got in ((0, dx), (1, dw), (2, db)):
        flat = base[which].view(-1)
        for at in range(0, flat.numel(), 7):
            keep = float(flat[at])
            flat[at] = keep + h
            plus = value(*base)
            flat[at] = keep - h
            minus = value(*base)
            flat[at] = keep
            # central differences: h^2 / 6 of third derivatives (some tens here), and roundings of 64 bits over h
            assert abs((plus - minus) / (2 * h) - float(got.view(-1)[at])) < 2e-5


@gpu
def test_same_bits_again_other_streams_and_a_graph(gpu_ctx):
    rows, cols = 5000, 1024
    x, dy, weight = numbers((rows, cols), "bf16", 17), numbers((rows, cols), "bf16", 18), numbers((cols,), "f32", 19)
    y, stats, q, s = torch.empty_like(x), torch.empty((rows, 2), device="cuda"), torch.empty((rows, cols), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    out = [(torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda"), workspace(gpu_ctx, rows, cols)) for _ in range(3)]

    def step(o, stream):
        gpu_ctx.layer_norm(x, y, weight, None, 1e-5, stats, q, s, stream=stream)
        gpu_ctx.layer_norm_grad(dy, stats, o[0], o[3], q=q, q_scale=s, weight=weight, dweight=o[1], dbias=o[2], stream=stream)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    step(out[0], side.cuda_stream)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(out[1], side.cuda_stream)
    for _ in range(2):
        out[1][0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out[0][:3], out[1][:3]):
            assert torch.equal(a, b)
    dy.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    check_grad(dy, q.double() * s.double()[:, None], stats, weight, out[1][0], out[1][1], out[1][2])


@gpu
def test_no_rows(gpu_ctx):
    x, stats = torch.zeros((0, 12), device="cuda"), torch.zeros((0, 2), device="cuda")
    dw, db = torch.full((12,), 5.0, device="cuda"), torch.full((12,), 5.0, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.layer_norm(x, x.clone(), stats=stats)
    gpu_ctx.layer_norm_grad(x, stats, x.clone(), torch.empty(16, dtype=torch.uint8, device="cuda"), x=x, dweight=dw, dbias=db)
    gpu_ctx.synchronize()
    assert not dw.any() and not db.any()


@gpu
def test_refusals(gpu_ctx):
    lib, h = gpu_ctx.lib, gpu_ctx.h
    f = torch.zeros(4096, device="cuda")
    p = f.data_ptr()
    NULL = None

    def norm(rows=4, cols=10, t=0, x=p, ldx=10, w=p, b=p, eps=1e-5, y=p + 4096, ldy=10, st=p + 8192, q=NULL, ldq=0, s=NULL):
        return lib.s2v_layer_norm(h, None, rows, cols, t, x, ldx, w, b, eps, y, ldy, st, q, ldq, s)

    def grad(rows=4, cols=10, t=0, dy=p, lddy=10, x=p, ldx=10, q=NULL, ldq=0, s=NULL, st=p, w=p, ws=p + 4096, n=4096, dx=p + 8192, lddx=10, dw=p + 12288, db=p + 12288 + 64):
        return lib.s2v_layer_norm_grad(h, None, rows, cols, t, dy, lddy, x, ldx, q, ldq, s, st, w, ws, n, dx, lddx, dw, db)
    for got, want in [(norm(rows=-1), -1), (norm(cols=0), -1), (norm(t=3), -1), (norm(t=-1), -1), (norm(x=NULL), -1), (norm(y=NULL), -1), (norm(q=p), -1), (norm(s=p), -1), (norm(ldx=9), -1),
                      (norm(ldy=9), -1), (norm(q=p, s=p, ldq=9), -1), (norm(eps=-1e-9), -1), (norm(eps=float("nan")), -1), (norm(eps=float("inf")), -1), (norm(x=p + 2), -1), (norm(y=p + 1, t=1), -1),
                      (norm(w=p + 2), -1), (norm(b=p + 1), -1), (norm(st=p + 4), -1), (norm(q=p, ldq=10, s=p + 2), -1), (norm(y=p, ldy=11), -1), (norm(cols=1 << 31, ldx=1 << 31, ldy=1 << 31), -2),
                      (grad(rows=-1), -1), (grad(cols=0), -1), (grad(t=7), -1), (grad(dy=NULL), -1), (grad(dx=NULL), -1), (grad(st=NULL), -1), (grad(x=NULL), -1), (grad(q=p, ldq=10, s=p), -1),
                      (grad(x=NULL, q=p, ldq=10), -1), (grad(x=NULL, s=p), -1), (grad(lddy=9), -1), (grad(ldx=9), -1), (grad(lddx=9), -1), (grad(x=NULL, q=p, ldq=9, s=p), -1), (grad(dx=p, lddx=11), -1),
                      (grad(ws=NULL), -5), (grad(n=64), -5), (grad(ws=p + 8), -1), (grad(st=p + 4), -1), (grad(w=p + 1), -1), (grad(dw=p + 2), -1), (grad(db=p + 3), -1), (grad(dy=p + 2), -1),
                      (grad(x=p + 2), -1), (grad(dx=p + 2), -1), (grad(cols=1 << 31), -2)]:
        assert got == want, lib.s2v_last_error(h)
    assert norm(rows=0, x=NULL, y=NULL) == 0
    gpu_ctx.synchronize()
    assert not f.any()
