"""Weight gradients of dense layers from 8-bit rows, against the formula in 64 bits; and a head in training as its calls follow each other."""
import pytest
import torch

from graphnn_b200 import capi

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24   # half a step of fp32


def inputs(m, n, k, dtype, seed=1):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dy = (torch.randn((m, n), generator=gen, device="cuda") * (0.2 + torch.rand((m, 1), generator=gen, device="cuda"))).to(TYPES[dtype])
    q = torch.randint(-127, 128, (m, k), generator=gen, device="cuda", dtype=torch.int8)
    scale = 0.01 * (0.1 + torch.rand(m, generator=gen, device="cuda"))
    if m > 3:
        scale[m // 2], q[m // 2] = 0.0, 0
    return dy, q, scale


def check(dy, q, scale, dW, dbias):
    m = dy.shape[0]
    d, x = dy.double(), q.double() * scale.double()[:, None]
    f = torch.finfo(dy.dtype)
    if dW is not None and dW.numel():
        want, size = d.t() @ x, d.abs().t() @ x.abs()
        # dy times the row's scale is rounded to 16 bits for the product where dy has 16 (fp16: in steps of 2^-24 of the column's largest below the normal range), to three 16-bit
        # parts where it has 32; a rounding (or a cut, twice as much) for each term of the sum
        rounding = f.eps / 2 if dy.dtype is not torch.float32 else 2 * U
        floor = 2.0 ** -24 * (d.abs() * scale.double()[:, None]).amax(0)[:, None] * q.double().abs().sum(0) if m else 0.0
        tol = (rounding + 2 * U * (m + 8)) * size + (floor if dy.dtype is torch.float16 else 0.0)
        tol = tol + f.eps / 2 * (want.abs() + tol) + f.smallest_normal * f.eps
        beyond = want.abs() > f.max * (1 + f.eps / 4)        # nearer to infinity than to the type's largest number: infinite, or the largest, within the tolerance
        assert bool((dW.double()[beyond] * want[beyond].sign() >= (want.abs() - tol)[beyond].clamp(max=f.max)).all())
        err = (dW.double() - want).abs()[~beyond & (want.abs() + tol < f.max)]
        tol = tol[~beyond & (want.abs() + tol < f.max)]
        assert bool((err <= tol).all()), f"dW off by up to {float((err / tol).max() if err.numel() else 0):.3g} of the tolerance"
    if dbias is not None:
        err, tol = (dbias.double() - d.sum(0)).abs(), U * (m + 40) * d.abs().sum(0) + 1e-44
        assert bool((err <= tol).all()), f"dbias off by up to {float((err / tol).max()):.3g} of the tolerance"


def space(ctx, m, n, k, dtype):
    return torch.full((max(16, ctx.linear_i8_grad_workspace_bytes(m, n, k, dtype)),), 255, dtype=torch.uint8, device="cuda")   # (NaN, as floats of any type)


def run(ctx, dy, q, scale, bias=True, stream=None):
    (m, n), k = dy.shape, q.shape[1]
    dW, dbias = torch.full((n, k), 5.0, dtype=dy.dtype, device="cuda"), torch.full((n,), 5.0, device="cuda") if bias else None
    ws = space(ctx, m, n, k, dy.dtype)
    torch.cuda.synchronize()
    ctx.linear_i8_grad(dy, q, scale, dW, ws, dbias=dbias, stream=stream)
    torch.cuda.synchronize()
    ctx.stream_status(stream)
    return dW, dbias


# ---------------------------------------------------------------- without a GPU
def test_workspace_sizes_without_a_gpu():
    size = capi.load_library().s2v_linear_i8_grad_workspace_bytes
    for bad in ((0, 5, 5, 0), (5, 0, 5, 0), (-1, 5, 5, 0), (5, 5, 5, 3), (5, 5, 5, -1), (5, 5, 0, 0), (1 << 30, 1 << 30, 5, 0), (1 << 30, 5, 1 << 30, 2), (1 << 31, 5, 5, 1)):
        assert size(*bad) == 0
    for t in (0, 1, 2):
        assert size(100, 40, 60, t) < 1 << 24
        assert size(1 << 24, 256, 128, t) < 1 << 29     # does not grow with the rows for good


def test_binding_refuses_what_the_library_cannot_see():
    ctx = capi.Context.__new__(capi.Context)
    ctx.h, ctx.device, ctx.lib = None, -1, capi.load_library()   # (torch gives -1 as the device of CPU tensors)
    made = []
    ctx.call = lambda name, *a: made.append((name, a))
    dy, q, s, dW, ws = torch.zeros(4, 6), torch.zeros((4, 9), dtype=torch.int8), torch.zeros(4), torch.zeros(6, 9), torch.zeros(64)
    ctx.linear_i8_grad(dy, q, s, dW, ws, dbias=torch.zeros(6))
    assert len(made) == 1 and made[0][1][1:4] == (4, 6, 9)
    for make in (lambda: ctx.linear_i8_grad(dy.double(), q, s, dW, ws), lambda: ctx.linear_i8_grad(dy, q.float(), s, dW, ws), lambda: ctx.linear_i8_grad(dy, q[:3], s, dW, ws), lambda: ctx.linear_i8_grad(dy, q, s[:3], dW, ws),
                 lambda: ctx.linear_i8_grad(dy, q, s, dW.half(), ws), lambda: ctx.linear_i8_grad(dy, q, s, dW.t(), ws), lambda: ctx.linear_i8_grad(dy, q, s, dW, ws[::2]),
                 lambda: ctx.linear_i8_grad(dy, q, s, dW, ws, dbias=torch.zeros(9)), lambda: ctx.linear_i8_grad(dy, q.t().contiguous().t(), s, dW, ws)):
        with pytest.raises(capi.S2VError):
            make()
    assert len(made) == 1


# ---------------------------------------------------------------- values
SHAPES = [(1, 1, 1), (2, 3, 5), (64, 6, 128), (1, 300, 500), (100, 128, 128), (65, 129, 257), (1000, 40, 24), (333, 256, 1021), (2000, 300, 130), (5000, 17, 72), (129, 1500, 700), (4099, 256, 128),
          # few rows
          (32, 300, 700), (33, 300, 700), (4, 65, 257), (17, 1000, 31),
          # few outputs over many rows: every shape of the tiles that one kernel takes
          (4096, 1, 1), (5000, 64, 64), (6001, 130, 65), (20000, 256, 128), (20011, 100, 200), (4500, 128, 256), (9000, 300, 100), (4097, 20, 700), (30000, 6, 40), (7000, 512, 256)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_weight_and_bias_gradients(gpu_ctx, shape, dtype):
    dy, q, scale = inputs(*shape, dtype)
    check(dy, q, scale, *run(gpu_ctx, dy, q, scale))
    dW, _ = run(gpu_ctx, dy, q, scale, bias=False)
    check(dy, q, scale, dW, None)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("extra,lead", [(16, 0), (3, 0), (16, 1), (5, 3)])
def test_rows_anywhere_and_nothing_else_written(gpu_ctx, extra, lead, dtype):
    def spaced(m):
        base = torch.full((m.shape[0] * (m.shape[1] + extra) + lead + extra,), 7, dtype=m.dtype, device="cuda")
        view = torch.as_strided(base, m.shape, (m.shape[1] + extra, 1), lead)
        view.copy_(m)
        return view, base
    for m, n, k in ((200, 48, 160), (77, 300, 64)):
        dy, q, scale = inputs(m, n, k, dtype, seed=3)
        (dys, _), (qs, _), (dW, dWb) = spaced(dy), spaced(q), spaced(torch.zeros((n, k), dtype=dy.dtype, device="cuda"))
        dbias, ws = torch.empty(n, device="cuda"), space(gpu_ctx, m, n, k, dy.dtype)
        torch.cuda.synchronize()
        gpu_ctx.linear_i8_grad(dys, qs, scale, dW, ws, dbias=dbias)
        gpu_ctx.synchronize()
        check(dy, q, scale, dW, dbias)
        mask = torch.ones_like(dWb, dtype=torch.bool)
        torch.as_strided(mask, dW.shape, dW.stride(), lead).fill_(False)
        assert bool((dWb[mask] == 7).all())


@gpu
def test_columns_and_scales_of_very_different_sizes(gpu_ctx):
    for dtype in TYPES:
        dy, q, scale = inputs(300, 80, 96, dtype, seed=4)
        scale *= torch.logspace(-3, 3, 300, device="cuda")[torch.randperm(300, device="cuda")]
        dy = (dy.float() * torch.logspace(-2, 2, 80, device="cuda")).to(dy.dtype)
        check(dy, q, scale, *run(gpu_ctx, dy, q, scale))
        # rows of a scale of NaN (they held no numbers) and of a gradient of infinity reach every weight they touch, and no others
        scale[5] = float("nan")
        dW, dbias = run(gpu_ctx, dy, q, scale)
        assert bool(dW.isnan().all()) and bool(dbias.isfinite().all())


@gpu
def test_same_bits_again_and_empty_sums(gpu_ctx):
    for dtype in TYPES:
        dy, q, scale = inputs(6001, 70, 90, dtype, seed=5)
        first, again = run(gpu_ctx, dy, q, scale), run(gpu_ctx, dy, q, scale, stream=torch.cuda.Stream().cuda_stream)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        dW, dbias, ws = torch.zeros_like(first[0]), torch.zeros_like(first[1]), space(gpu_ctx, 6001, 70, 90, dy.dtype)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            gpu_ctx.linear_i8_grad(dy, q, scale, dW, ws, dbias=dbias, stream=side.cuda_stream)
        for _ in range(2):
            dW.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(dW, first[0]) and torch.equal(dbias, first[1])
        dW, dbias = run(gpu_ctx, dy[:0], q[:0], scale[:0])
        assert not dW.any() and not dbias.any()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_workspaces_on_any_16_byte_boundary(gpu_ctx, dtype):
    for m, n, k in ((300, 200, 136), (6000, 256, 128), (5000, 64, 48), (3000, 129, 130)):
        dy, q, scale = inputs(m, n, k, dtype, seed=6)
        want = run(gpu_ctx, dy, q, scale)
        size = gpu_ctx.linear_i8_grad_workspace_bytes(m, n, k, dy.dtype)
        for off in (16, 48, 240):
            around = torch.full((size + 512,), 7, dtype=torch.uint8, device="cuda")
            dW, dbias = torch.empty_like(want[0]), torch.empty_like(want[1])
            torch.cuda.synchronize()
            gpu_ctx.linear_i8_grad(dy, q, scale, dW, around[off:off + size], dbias=dbias)
            gpu_ctx.synchronize()
            assert torch.equal(dW, want[0]) and torch.equal(dbias, want[1])
            assert bool((around[:off] == 7).all()) and bool((around[off + size:] == 7).all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_pieces_of_the_rows(gpu_ctx, dtype):
    # rows enough for several pieces of the 16-bit copies, the last one small; an odd number of columns keeps the direct form out of it
    m, n, k = (70001, 1001, 31) if dtype == "f32" else (140001, 901, 63)
    dy, q, scale = inputs(m, n, k, dtype, seed=7)
    dW, dbias = run(gpu_ctx, dy, q, scale)
    d, x = dy.double(), q.double() * scale.double()[:, None]
    want, size = d.t() @ x, d.abs().t() @ x.abs()
    f = torch.finfo(dy.dtype)
    # (sums of 64 rows and eight panels in the matrix units, cut, then rounded additions, one for 512 terms)
    tol = ((f.eps / 2 if dtype != "f32" else 2 * U) + 2 * U * (64 * 3 * 32 / 16 + 3 * m / 512 + 8)) * size + f.eps / 2 * want.abs() * 1.01 + f.smallest_normal
    if dtype == "f16":
        tol = tol + 2.0 ** -24 * (d.abs() * scale.double()[:, None]).amax(0)[:, None] * q.double().abs().sum(0)
    inside = want.abs() + tol < f.max
    assert bool(((dW.double() - want).abs() <= tol)[inside].all())
    assert bool(((dbias.double() - d.sum(0)).abs() <= U * (m / 500 + 700) * d.abs().sum(0)).all())


@gpu
def test_refusals(gpu_ctx):
    lib, h = gpu_ctx.lib, gpu_ctx.h
    f = torch.zeros(1 << 18, device="cuda")
    p, half = f.data_ptr(), f.nbytes // 2

    def call(m=4, n=10, k=8, t=0, dy=p, lddy=10, q=p, ldq=8, s=p, ws=p + half, size=half, dW=p + 4096, lddw=8, db=p + 8192):
        return lib.s2v_linear_i8_grad(h, None, m, n, k, t, dy, lddy, q, ldq, s, ws, size, dW, lddw, db)
    for got, want in [(call(m=-1), -1), (call(n=-1), -1), (call(k=-1), -1), (call(t=3), -1), (call(dy=None), -1), (call(q=None), -1), (call(s=None), -1), (call(dW=None), -1), (call(lddy=9), -1), (call(ldq=7), -1),
                      (call(lddw=7), -1), (call(dy=p + 2), -1), (call(dW=p + 1, t=2), -1), (call(s=p + 2), -1), (call(db=p + 1), -1), (call(ws=None), -5), (call(size=8), -5), (call(ws=p + half + 4), -1), (call(m=1 << 31), -2),
                      (call(n=1 << 31, lddy=1 << 31), -2), (call(k=1 << 31, ldq=1 << 31, lddw=1 << 31), -2)]:
        assert got == want, lib.s2v_last_error(h)
    assert call(n=0) == 0
    gpu_ctx.synchronize()
    assert not f.any()


@gpu
@pytest.mark.parametrize("reserved", [1, 75, 140, 146])
def test_sms_left_to_others(reserved):
    """With most SMs left to others tiles, shares and rows fall to few CTAs; results stay within the same tolerances, workspaces within their sizes."""
    ctx = capi.Context(0)
    try:
        ctx.set_option(ctx.OPT_RESERVED_SMS, reserved)
        for m, n, k, dtype in ((700, 300, 260, "bf16"), (6000, 256, 128, "f32"), (5000, 600, 130, "f16"), (4200, 40, 64, "bf16")):
            dy, q, scale = inputs(m, n, k, dtype, seed=8)
            (dW, dbias), size = run(ctx, dy, q, scale), ctx.linear_i8_grad_workspace_bytes(m, n, k, dy.dtype)
            check(dy, q, scale, dW, dbias)
            around = torch.full((size + 1024,), 7, dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            ctx.linear_i8_grad(dy, q, scale, dW, around[:size], dbias=dbias)
            ctx.synchronize()
            check(dy, q, scale, dW, dbias)
            assert bool((around[size:] == 7).all())
        from test_layer_norm import check_forward, check_grad
        from test_linear_cross_entropy import Reference, both
        from test_linear_cross_entropy import inputs as classes
        for shape, dtype in (((300, 1500, 200), "bf16"), ((200, 130, 2100), "f32"), ((600, 2500, 512), "f16")):
            x, W, target, weight = classes(*shape, dtype)
            ref = Reference(x, W, target, weight)
            loss, dx, dWv = both(ctx, x, W, target, weight)
            ref.check_loss(loss)
            ref.check_grad(dx, dWv)
        x = torch.randn((900, 4096), device="cuda").bfloat16()
        dy, y, dx, stats = torch.randn_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty((900, 2), device="cuda")
        dw, db, ws = torch.empty(4096, device="cuda"), torch.empty(4096, device="cuda"), torch.empty(ctx.layer_norm_grad_workspace_bytes(900, 4096), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        ctx.layer_norm(x, y, stats=stats)
        ctx.layer_norm_grad(dy, stats, dx, ws, x=x, dweight=dw, dbias=db)
        ctx.synchronize()
        check_forward(x, None, None, 1e-5, y, stats)
        check_grad(dy, x.double(), stats, None, dx, dw, db)
    finally:
        ctx.close()


# ---------------------------------------------------------------- together, as they are used
@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_head_in_training(gpu_ctx, dtype):
    """Embeddings -> layer norm (kept in 8 bits) -> dense layer (its input kept in 8 bits) -> loss over the classes, and all gradients, against the same chain in
    64 bits with the 8-bit rows as they are kept."""
    rows, d, hidden, vocab = 600, 128, 256, 777
    T, gen = TYPES[dtype], torch.Generator(device="cuda")
    gen.manual_seed(11)

    def rand(*shape, size=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * size
    x, gamma, beta = rand(rows, d, size=2.0).to(T), 1 + 0.2 * rand(d), 0.1 * rand(d)
    W1, W2 = rand(hidden, d, size=d ** -0.5).to(T), rand(vocab, hidden, size=hidden ** -0.5).to(T)
    target = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    target[5::50] = -1
    weight = torch.full((rows,), 1.0 / int((target >= 0).sum()), device="cuda")
    xq, xs, stats = torch.empty((rows, d), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda")
    y, hq, hs = torch.empty_like(x), torch.empty((rows, d), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    w8, w8s, h = torch.empty((hidden, d), dtype=torch.int8, device="cuda"), torch.empty(hidden, device="cuda"), torch.empty((rows, hidden), dtype=T, device="cuda")
    loss, kept = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda")
    dh, dW2, dW1, db1 = torch.empty_like(h), torch.empty_like(W2), torch.empty_like(W1), torch.empty(hidden, device="cuda")
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    ws = torch.empty(max(gpu_ctx.linear_cross_entropy_workspace_bytes(rows, vocab, hidden, T), gpu_ctx.linear_i8_grad_workspace_bytes(rows, hidden, d, T),
                         gpu_ctx.layer_norm_grad_workspace_bytes(rows, d)), dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        at = s.cuda_stream
        gpu_ctx.quantize_rows_i8(W1, w8, w8s, stream=at)
        gpu_ctx.layer_norm(x, y, gamma, beta, 1e-5, stats, xq, xs, stream=at)
        gpu_ctx.quantize_rows_i8(y, hq, hs, stream=at)
        gpu_ctx.gemm_i8(hq, hs, w8, w8s, h, relu=True, stream=at)
        gpu_ctx.linear_cross_entropy(h, W2, target, loss, ws, row_weight=weight, stats=kept, stream=at)
        gpu_ctx.linear_cross_entropy_grad(h, W2, target, kept, ws, dx=dh, dW=dW2, row_weight=weight, stream=at)
        dz = torch.where(h > 0, dh, 0.0)                       # back through ReLU
        gpu_ctx.linear_i8_grad(dz, hq, hs, dW1, ws, dbias=db1, stream=at)
        dy = dz @ W1
        gpu_ctx.layer_norm_grad(dy, stats, dx, ws, q=xq, q_scale=xs, weight=gamma, dweight=dgamma, dbias=dbeta, stream=at)
    s.synchronize()
    gpu_ctx.stream_status(at)
    # each step in 64 bits from what the step before handed over
    live = target >= 0
    z = h.double() @ W2.double().t()
    t = torch.where(live, target.long(), 0)[:, None]
    want = torch.where(live, (z.logsumexp(1) - z.gather(1, t)[:, 0]) * weight.double(), 0.0)
    assert float((loss.double() - want).abs().max()) < 1e-5 * float(want.max())
    G = z.softmax(1).scatter_add(1, t, torch.full_like(z[:, :1], -1.0)) * torch.where(live, weight.double(), 0.0)[:, None]
    eps = torch.finfo(T).eps

    def close(got, want, size):     # operands and results of eps / 2 each, sums of some hundred terms
        assert bool(((got.double() - want).abs() <= (1.5 * eps + 2 * U * 900) * size + eps / 2 * want.abs()).all())
    close(dh, G @ W2.double(), G.abs() @ W2.double().abs())
    close(dW2, G.t() @ h.double(), G.abs().t() @ h.double().abs())
    check(dz, hq, hs, dW1, db1)
    kept_x = xq.double() * xs.double()[:, None]
    hat = (kept_x - stats[:, :1].double()) * stats[:, 1:].double()
    g = dy.double() * gamma.double()
    want = stats[:, 1:].double() * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    assert float((dx.double() - want).abs().max()) <= (eps + 1e-5) * float(want.abs().max())
    assert float((dgamma.double() - (dy.double() * hat).sum(0)).abs().max()) < 1e-5 * float((dy.double() * hat).abs().sum(0).max())
    assert float((dbeta.double() - dy.double().sum(0)).abs().max()) < 1e-5 * float(dy.double().abs().sum(0).max())
    # and the 8-bit rows are worth keeping: gradients of the norm from them point where those from x itself do
    dx_full = torch.empty_like(x)
    torch.cuda.synchronize()
    gpu_ctx.layer_norm_grad(dy, stats, dx_full, ws, x=x, weight=gamma)
    gpu_ctx.synchronize()
    assert float(torch.nn.functional.cosine_similarity(dx.double().flatten(), dx_full.double().flatten(), dim=0)) > 0.999


# ---------------------------------------------------------------- infinities and NaN in dy, and all of fp32, in every form
FORMS = {"few": (20, 70, 90), "general": (1000, 40, 90), "direct": (5000, 70, 90)}     # (one launch; 16-bit copies; straight from dy)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", FORMS)
def test_infinities_and_nan_reach_what_they_are_part_of_alone(gpu_ctx, form, dtype):
    dy, q, scale = inputs(*FORMS[form], dtype, seed=6)
    clean = run(gpu_ctx, dy, q, scale)
    rest = torch.arange(dy.shape[1], device="cuda") != 3
    for bad in (float("inf"), float("-inf"), float("nan")):
        dy[5, 3] = bad
        dW, dbias = run(gpu_ctx, dy, q, scale)
        assert not dW[3].isfinite().any() and not dbias[3].isfinite().any()
        assert torch.equal(dW[rest], clean[0][rest]) and torch.equal(dbias[rest], clean[1][rest])


@gpu
@pytest.mark.parametrize("m,n,k", [(20, 70, 90), (2000, 300, 130), (4099, 256, 128), (5000, 64, 64), (9000, 300, 100), (4500, 128, 256)])
def test_fp32_keeps_all_its_digits(gpu_ctx, m, n, k):
    # four rows of dy have a number in a column, so that few roundings hide a lost part of it
    _, q, scale = inputs(m, n, k, "f32", seed=7)
    scale = scale.clamp(min=1e-3)
    gen = torch.Generator(device="cuda").manual_seed(8)
    dy, j = torch.zeros((m, n), device="cuda"), torch.arange(n, device="cuda")
    for i in range(4):
        dy[(j * 13 + i * (m // 4)) % m, j] = torch.randn(n, generator=gen, device="cuda")
    dW, dbias = run(gpu_ctx, dy, q, scale)
    d, x = dy.double(), q.double() * scale.double()[:, None]
    want, size = d.t() @ x, d.abs().t() @ x.abs()
    # dy times the scale is rounded, and is three bf16 numbers but for 2^-24 (the first cut to eight bits, the others rounded); twelve products that are none, added with a rounding, or a
    # cut, twice as much, each; the result rounded
    tol = U * (1 + 1 + 2 * 12 + 1) * size + 1e-44
    err = (dW.double() - want).abs()
    assert bool((err <= tol).all()), f"dW off by up to {float((err / tol).max()):.3g} of the tolerance"
    assert bool(((dbias.double() - d.sum(0)).abs() <= 4 * U * d.abs().sum(0) + 1e-44).all())


@gpu
def test_long_sums_of_one_sign(gpu_ctx):
    m, n, k = 1 << 22, 8, 16
    gen = torch.Generator(device="cuda").manual_seed(9)
    dy, scale = 0.5 + 0.5 * torch.rand((m, n), generator=gen, device="cuda"), 0.5 + 0.5 * torch.rand(m, generator=gen, device="cuda")
    q = torch.randint(64, 128, (m, k), generator=gen, device="cuda", dtype=torch.int8)
    dW, _ = run(gpu_ctx, dy, q, scale)
    want = torch.zeros((n, k), dtype=torch.float64, device="cuda")
    for a in range(0, m, 1 << 20):
        at = slice(a, a + (1 << 20))
        want += dy[at].double().t() @ (q[at].double() * scale[at].double()[:, None])
    # 148 shares of the rows at most, and 100 at least, of 1311 panels of 32 rows each; an accumulator takes five panels, 30 instructions of two cuts of a step (2 U) at most; accumulators
    # are added with a rounding each, and the shares four at a time; operands as above
    tol = U * (3 + 30 * 4 + 1311 / 5 + 37 + 4) * want
    err = (dW.double() - want).abs()
    assert bool((err <= tol).all()), f"off by up to {float((err / tol).max()):.3g} of the tolerance"
