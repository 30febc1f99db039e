"""Softmax cross entropy of x W^T without logits in memory, and its gradients: against the formulas in 64 bits and against differences."""
import pytest
import torch

from graphnn_b200 import capi

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24   # half a step of fp32


def inputs(rows, vocab, k, dtype, seed=1, size=2.0, ignored=True):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    W = (torch.randn((vocab, k), generator=gen, device="cuda") * (size / k ** 0.5)).to(TYPES[dtype])
    target = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x = (x + 3 * torch.rand((rows, 1), generator=gen, device="cuda") * W[target].float()).to(TYPES[dtype])
    target = target.to(torch.int32)
    weight = (torch.rand(rows, generator=gen, device="cuda") + 0.2) * (64.0 if dtype == "f16" else 1.0) / rows
    if rows > 2:
        weight[rows // 3] *= -1.0
    if ignored and rows > 4:
        target[1], target[rows // 2], target[rows - 1] = -1, vocab, -(2 ** 31)
        weight[rows // 4] = 0.0
        x[[1, rows // 2, rows - 1, rows // 4]] = float("nan")     # rows that are left out may hold anything
    return x, W, target, weight


class Reference:
    """Everything in 64 bits, and how far fp32 arithmetic may be off."""

    def __init__(self, x, W, target, weight):
        self.rows, self.vocab, self.k = x.shape[0], W.shape[0], W.shape[1]
        t = target.long()
        w = torch.ones(self.rows, dtype=torch.float64, device="cuda") if weight is None else weight.double()
        live = (t >= 0) & (t < self.vocab) & (w != 0)
        self.live, self.w = live, torch.where(live, w, 0.0)
        self.x = torch.where(live[:, None], x.double(), 0.0)
        self.W, self.dtype = W.double(), W.dtype
        t = torch.where(live, t, 0)[:, None]
        z = self.x @ self.W.t()
        rel = z - z.gather(1, t)
        others = rel.scatter(1, t, float("-inf")).logsumexp(1)
        one = torch.nn.functional.softplus(others, threshold=1e9) if self.vocab > 1 else torch.zeros(self.rows, dtype=torch.float64, device="cuda")
        one = torch.where(others < -30, others.exp(), one)         # log1p of a small number
        self.one, self.loss = one, self.w * one
        p = (rel - one[:, None]).exp()
        self.p = p
        g = p.scatter(1, t, torch.expm1(-one)[:, None])
        self.G = g * self.w[:, None]
        self.dx, self.dW = self.G @ self.W, self.G.t() @ self.x
        # A logit is a sum of k products, which the matrix units add with a rounding (or a cut: twice as much) each; operands of fp32 are three 16-bit parts
        # whose smallest products (2^-26) are left out.  In units of sum |x W|.
        size = (self.x.abs() @ self.W.abs().t()).amax(1)
        dz = 2 * U * (self.k + 8) * size
        # An exponent's argument has roundings of its difference, its constant and product; exponentials two steps; at most 256 additions in a tile, and every
        # tile of 64 or more classes joined behind it with three.
        span = z.amax(1) - z.amin(1)
        self.rel = 2 * dz + U * (8 * span + 4 + 256 + 3 * self.vocab / 64 + 60)
        self.lse_tol = self.rel + U * z.logsumexp(1).abs()

    def check_loss(self, loss):
        tol = self.w.abs() * (self.rel * (1 - (-self.one).exp()).clamp(min=0) * (1 + self.rel.exp())) + 2 * U * self.loss.abs() + 1e-44
        err = (loss.double() - self.loss).abs()
        assert bool((err <= tol).all()), f"loss off by up to {float((err / tol).max()):.3g} of the tolerance"
        assert not loss[~self.live].any()

    def check_grad(self, dx, dW):
        f = torch.finfo(self.dtype)
        g = self.G.abs()
        # of G: the logit and the kept log-sum-exp in the exponent, four steps of exponential and products; rounded to 16 bits for the products where the
        # operands have 16 (fp16: in steps of 2^-38 of the largest row weight below the normal range)
        floor = 2.0 ** -38 * float(self.w.abs().max()) if self.dtype is torch.float16 else 1e-40 * float(self.w.abs().max())
        dg = (self.w.abs()[:, None] * self.p) * (torch.expm1(self.rel + self.lse_tol) + 6 * U)[:, None] + 4 * U * g
        dg = dg + (f.eps / 2 if self.dtype is not torch.float32 else 2.0 ** -24) * (g + dg) + floor
        for got, a, b, da in ((dx, self.G, self.W, dg), (dW, self.G.t(), self.x, dg.t())):
            if got is None:
                continue
            want, terms = a @ b, a.shape[1]
            tol = da @ b.abs() + 2 * U * (terms + 24) * (a.abs() @ b.abs())
            tol = (tol + f.eps / 2 * (want.abs() + tol) + f.smallest_normal * f.eps) * (1 + 1e-6)
            err = (got.double() - want).abs()
            assert bool((err <= tol).all()), f"gradient off by up to {float((err / tol).max()):.3g} of the tolerance"


def space(ctx, rows, vocab, k, dtype, grad=True):
    return torch.full((max(16, ctx.linear_cross_entropy_workspace_bytes(rows, vocab, k, dtype, grad)),), 255, dtype=torch.uint8, device="cuda")   # (NaN, as floats of any type)


def both(ctx, x, W, target, weight, stream=None):
    rows, k = x.shape
    loss, stats = torch.full((rows,), 5.0, device="cuda"), torch.full((rows, 2), 5.0, device="cuda")
    dx, dW = torch.full_like(x, 5.0, memory_format=torch.contiguous_format), torch.full((W.shape[0], k), 5.0, dtype=W.dtype, device="cuda")
    ws = space(ctx, rows, W.shape[0], k, W.dtype)
    torch.cuda.synchronize()
    ctx.linear_cross_entropy(x, W, target, loss, ws, row_weight=weight, stats=stats, stream=stream)
    ctx.linear_cross_entropy_grad(x, W, target, stats, ws, dx=dx, dW=dW, row_weight=weight, stream=stream)
    torch.cuda.synchronize()
    ctx.stream_status(stream)
    return loss, dx, dW


# ---------------------------------------------------------------- without a GPU
def test_workspace_sizes_without_a_gpu():
    size = capi.load_library().s2v_linear_cross_entropy_workspace_bytes
    for bad in ((0, 5, 5, 0, 1), (5, 0, 5, 0, 1), (5, 5, 0, 0, 1), (-1, 5, 5, 0, 1), (5, 5, 5, 3, 1), (5, 5, 5, -1, 0), (1 << 31, 5, 5, 0, 0), (5, 1 << 40, 5, 0, 0), (1 << 30, 5, 1 << 30, 0, 0), (5, 1 << 30, 1 << 30, 2, 1)):
        assert size(*bad) == 0
    for t in (0, 1, 2):
        assert 0 < size(64, 6, 128, t, 0) <= size(64, 6, 128, t, 1) < 1 << 22
    # far less than the logits: 32,768 rows of 262,144 classes are 16 GiB in 16 bits
    assert size(32768, 262144, 4096, 2, 1) < 3 << 30


@pytest.fixture
def recorded():
    ctx = capi.Context.__new__(capi.Context)
    ctx.h, ctx.device, ctx.lib = None, -1, capi.load_library()   # (torch gives -1 as the device of CPU tensors)
    ctx.made = []
    ctx.call = lambda name, *a: ctx.made.append((name, a))
    return ctx


def test_binding_refuses_what_the_library_cannot_see(recorded):
    x, W, t, v = torch.zeros(4, 6), torch.zeros(9, 6), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    ws, st = torch.zeros(64), torch.zeros(4, 2)
    recorded.linear_cross_entropy(x, W, t, v, ws, row_weight=v.clone(), stats=st)
    recorded.linear_cross_entropy_grad(x, W, t, st, ws, dx=x.clone(), dW=W.clone(), row_weight=v)
    assert len(recorded.made) == 2 and recorded.made[0][1][1:4] == (4, 9, 6)
    for make in (lambda: recorded.linear_cross_entropy(x, W.half(), t, v, ws), lambda: recorded.linear_cross_entropy(x, W[:, :5], t, v, ws), lambda: recorded.linear_cross_entropy(x, W, t.long(), v, ws),
                 lambda: recorded.linear_cross_entropy(x, W, t[:3], v, ws), lambda: recorded.linear_cross_entropy(x, W, t, v[:3], ws), lambda: recorded.linear_cross_entropy(x, W, t, v, ws[::2]),
                 lambda: recorded.linear_cross_entropy(x, W, t, v, ws, row_weight=v.double()), lambda: recorded.linear_cross_entropy(x, W, t, v, ws, stats=torch.zeros(4, 4)[:, :2]),
                 lambda: recorded.linear_cross_entropy(x.double(), W.double(), t, v, ws), lambda: recorded.linear_cross_entropy(x.t(), W, t, v, ws),
                 lambda: recorded.linear_cross_entropy_grad(x, W, t, None, ws, dx=x.clone()), lambda: recorded.linear_cross_entropy_grad(x, W, t, st, ws, dx=W.clone()),
                 lambda: recorded.linear_cross_entropy_grad(x, W, t, st, ws, dW=W.half())):
        with pytest.raises(capi.S2VError):
            make()
    assert len(recorded.made) == 2


# ---------------------------------------------------------------- values
SHAPES = [(1, 1, 1), (1, 2, 3), (3, 1, 16), (2, 7, 5), (64, 6, 128), (5, 40, 33), (130, 129, 65), (64, 64, 64), (257, 300, 31), (100, 1000, 256), (1, 5000, 128), (7, 20000, 72), (700, 513, 200), (300, 4097, 130),
          (129, 255, 1021), (33, 900, 2048), (2100, 70, 40), (600, 2500, 512),
          # the limits of the form for a few classes, and one past each
          (512, 64, 512), (513, 64, 512), (512, 65, 512), (512, 64, 513), (65, 33, 100),
          # few logits with long sums, whose logits are kept: one tile, several, odd places
          (1, 2, 4000), (86, 38, 3206), (3, 9000, 2100), (600, 600, 2048), (1000, 1025, 2500), (130, 70, 5001)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_loss_and_gradients(gpu_ctx, shape, dtype):
    x, W, target, weight = inputs(*shape, dtype)
    ref = Reference(x, W, target, weight)
    loss, dx, dW = both(gpu_ctx, x, W, target, weight)
    ref.check_loss(loss)
    ref.check_grad(dx, dW)
    assert not dx[~ref.live].any()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("extra,lead", [(8, 0), (3, 0), (8, 1), (5, 3)])
def test_rows_anywhere_and_nothing_else_written(gpu_ctx, extra, lead, dtype):
    for rows, vocab, k in ((37, 300, 136), (200, 33, 40), (300, 700, 264)):
        x, W, target, weight = inputs(rows, vocab, k, dtype, seed=3)

        def spaced(m):
            base = torch.full((m.shape[0] * (m.shape[1] + extra) + lead + extra,), 7.0, dtype=m.dtype, device="cuda")
            view = torch.as_strided(base, m.shape, (m.shape[1] + extra, 1), lead)
            view.copy_(m)
            return view, base
        (xs, xb), (Ws, Wb), (dx, dxb), (dW, dWb) = spaced(x), spaced(W), spaced(torch.zeros_like(x)), spaced(torch.zeros_like(W))
        loss, stats, ws = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda"), space(gpu_ctx, rows, vocab, k, W.dtype)
        torch.cuda.synchronize()
        gpu_ctx.linear_cross_entropy(xs, Ws, target, loss, ws, row_weight=weight, stats=stats)
        gpu_ctx.linear_cross_entropy_grad(xs, Ws, target, stats, ws, dx=dx, dW=dW, row_weight=weight)
        gpu_ctx.synchronize()
        ref = Reference(x, W, target, weight)
        ref.check_loss(loss)
        ref.check_grad(dx, dW)
        for base, view in ((dxb, dx), (dWb, dW)):
            mask = torch.ones_like(base, dtype=torch.bool)
            torch.as_strided(mask, view.shape, view.stride(), lead).fill_(False)
            assert bool((base[mask] == 7.0).all())
        # one at a time gives the same
        dx1, dW1 = torch.empty_like(x), torch.empty_like(W)
        torch.cuda.synchronize()
        gpu_ctx.linear_cross_entropy_grad(xs, Ws, target, stats, ws, dx=dx1, row_weight=weight)
        gpu_ctx.linear_cross_entropy_grad(xs, Ws, target, stats, ws, dW=dW1, row_weight=weight)
        gpu_ctx.linear_cross_entropy_grad(xs, Ws, target, stats, ws, row_weight=weight)
        gpu_ctx.synchronize()
        assert torch.equal(dx1, dx) and torch.equal(dW1, dW)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_certain_rows_keep_their_small_losses(gpu_ctx, dtype):
    # the own class ahead by 20 to 60: losses of e^-20 and far less, which log-sum-exp minus logit would round to nothing
    vocab, k = 40, 64
    W = torch.eye(vocab, k, device="cuda").to(TYPES[dtype])
    target = torch.arange(vocab, dtype=torch.int32, device="cuda")
    x = torch.zeros((vocab, k), device="cuda")
    x[torch.arange(vocab), torch.arange(vocab)] = torch.linspace(20, 60, vocab, device="cuda")
    x = x.to(TYPES[dtype])
    loss, dx, dW = both(gpu_ctx, x, W, target, None)
    ref = Reference(x, W, target, None)
    ref.check_loss(loss)
    ref.check_grad(dx, dW)
    assert bool((loss > 0).all()) and float(loss[-1]) < 1e-20
    own = dx[torch.arange(vocab), torch.arange(vocab)].double()
    assert bool(((own / torch.expm1(-ref.one) - 1).abs() < 2.0 ** -7).all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_with_no_numbers_and_no_rows_that_count(gpu_ctx, dtype):
    x, W, target, weight = inputs(40, 200, 72, dtype, seed=5)
    x[7, 3], x[9] = float("nan"), float("inf")
    loss, dx, dW = both(gpu_ctx, x, W, target, weight)
    fine = torch.ones(40, dtype=torch.bool, device="cuda")
    fine[[7, 9]] = False
    assert bool(loss[~fine].isnan().all()) and bool(loss[fine].isfinite().all())
    assert bool(dx[~fine].isnan().all()) and bool(dx[fine].isfinite().all()) and bool(dW.isnan().all())
    x, W, target, weight = inputs(40, 200, 72, dtype, seed=5)
    target.fill_(-1)
    x.fill_(float("nan"))
    loss, dx, dW = both(gpu_ctx, x, W, target, weight)
    assert not loss.any() and not dx.any() and not dW.any()


@gpu
def test_weights_of_very_different_sizes(gpu_ctx):
    for dtype in TYPES:
        x, W, target, _ = inputs(24, 50, 64, dtype, seed=6, ignored=False)
        weight = torch.logspace(-3, 3, 24, device="cuda")
        loss, dx, dW = both(gpu_ctx, x, W, target, weight)
        ref = Reference(x, W, target, weight)
        ref.check_loss(loss)
        ref.check_grad(dx, dW)


@gpu
def test_gradients_against_differences(gpu_ctx):
    rows, vocab, k, h = 9, 70, 24, 1e-5
    x, W, target, weight = inputs(rows, vocab, k, "f32", seed=7)
    _, dx, dW = both(gpu_ctx, x, W, target, weight)
    live = Reference(x, W, target, weight).live
    base = [torch.where(live[:, None], x, 0.0).double(), W.double()]

    def value():
        z = base[0] @ base[1].t()
        t = torch.where(live, target.long(), 0)
        each = z.logsumexp(1) - z.gather(1, t[:, None])[:, 0]
        return float((torch.where(live, weight.double(), 0.0) * each).sum())
    for which, got in ((0, dx), (1, dW)):
        flat = base[which].view(-1)
        for at in range(0, flat.numel(), 11):
            keep = float(flat[at])
            flat[at] = keep + h
            plus = value()
            flat[at] = keep - h
            minus = value()
            flat[at] = keep
            # central differences: h^2 / 6 of third derivatives, and roundings of 64 bits (1e-15) over h; the gradients themselves are fp32
            assert abs((plus - minus) / (2 * h) - float(got.view(-1)[at])) < 1e-6


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(9000, 20011), (9000, 15000), (70000, 1850), (70000, 3800)])
def test_many_pieces_of_the_vocabulary(gpu_ctx, rows, vocab, dtype):
    # rows enough that a piece's gradient of the logits is a part of the vocabulary, with small and large last pieces
    x, W, target, weight = inputs(rows, vocab, 48, dtype, seed=8)
    loss, dx, dW = both(gpu_ctx, x, W, target, weight)
    ref = Reference(x, W, target, weight)
    ref.check_loss(loss)
    ref.check_grad(dx, dW)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_same_bits_again_other_streams_and_a_graph(gpu_ctx, dtype):
    for shape in ((200, 1500, 128), (64, 6, 128)):
        x, W, target, weight = inputs(*shape, dtype, seed=9)
        first = both(gpu_ctx, x, W, target, weight)
        side = torch.cuda.Stream()
        again = both(gpu_ctx, x, W, target, weight, stream=side.cuda_stream)
        for a, b in zip(first, again):
            assert torch.equal(a, b)
        rows, vocab, k = shape
        spaces = [space(gpu_ctx, rows, vocab, k, W.dtype) for _ in range(2)]
        outs = [(torch.zeros(rows, device="cuda"), torch.zeros((rows, 2), device="cuda"), torch.zeros_like(x), torch.zeros_like(W)) for _ in range(2)]
        graphs = []
        for ws, (loss, stats, dx, dW) in zip(spaces, outs):
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                gpu_ctx.linear_cross_entropy(x, W, target, loss, ws, row_weight=weight, stats=stats, stream=side.cuda_stream)
                gpu_ctx.linear_cross_entropy_grad(x, W, target, stats, ws, dx=dx, dW=dW, row_weight=weight, stream=side.cuda_stream)
            graphs.append(graph)
        other = torch.cuda.Stream()
        for _ in range(3):    # two graphs at once, a workspace each
            with torch.cuda.stream(side):
                graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
        torch.cuda.synchronize()
        for loss, _, dx, dW in outs:
            assert torch.equal(loss, first[0]) and torch.equal(dx, first[1]) and torch.equal(dW, first[2])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_workspaces_on_any_16_byte_boundary(gpu_ctx, dtype):
    for shape in ((200, 700, 136), (64, 6, 128), (300, 40, 2000)):
        x, W, target, weight = inputs(*shape, dtype, seed=10)
        want = both(gpu_ctx, x, W, target, weight)
        rows, vocab, k = shape
        size = gpu_ctx.linear_cross_entropy_workspace_bytes(rows, vocab, k, W.dtype)
        for off in (16, 48, 240):
            around = torch.full((size + 512,), 7, dtype=torch.uint8, device="cuda")
            ws = around[off:off + size]
            loss, stats, dx, dW = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda"), torch.empty_like(x), torch.empty_like(W)
            torch.cuda.synchronize()
            gpu_ctx.linear_cross_entropy(x, W, target, loss, ws, row_weight=weight, stats=stats)
            gpu_ctx.linear_cross_entropy_grad(x, W, target, stats, ws, dx=dx, dW=dW, row_weight=weight)
            gpu_ctx.synchronize()
            assert torch.equal(loss, want[0]) and torch.equal(dx, want[1]) and torch.equal(dW, want[2])
            assert bool((around[:off] == 7).all()) and bool((around[off + size:] == 7).all())


@gpu
def test_no_rows(gpu_ctx):
    x, W, t, st = torch.zeros((0, 12), device="cuda"), torch.ones((5, 12), device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros((0, 2), device="cuda")
    wide = torch.full((5, 15), 7.0, device="cuda")
    ws = torch.empty(16, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.linear_cross_entropy(x, W, t, torch.zeros(0, device="cuda"), ws, stats=st)
    gpu_ctx.linear_cross_entropy_grad(x, W, t, st, ws, dx=x.clone(), dW=wide[:, :12])
    gpu_ctx.synchronize()
    assert not wide[:, :12].any() and bool((wide[:, 12:] == 7.0).all())


@gpu
def test_refusals(gpu_ctx):
    lib, h = gpu_ctx.lib, gpu_ctx.h
    f = torch.zeros(1 << 20, device="cuda")
    p, big = f.data_ptr(), f.nbytes // 2
    ws = p + f.nbytes // 2

    def loss(rows=4, vocab=10, k=8, t=0, x=p, ldx=8, W=p, ldw=8, target=p, w=None, space=ws, n=big, out=p + 4096, st=p + 8192):
        return lib.s2v_linear_cross_entropy(h, None, rows, vocab, k, t, x, ldx, W, ldw, target, w, space, n, out, st)

    def grad(rows=4, vocab=10, k=8, t=0, x=p, ldx=8, W=p, ldw=8, target=p, w=None, st=p, space=ws, n=big, dx=p + 4096, lddx=8, dW=p + 8192, lddw=8):
        return lib.s2v_linear_cross_entropy_grad(h, None, rows, vocab, k, t, x, ldx, W, ldw, target, w, st, space, n, dx, lddx, dW, lddw)
    for call in (loss, grad):
        for got, want in [(call(rows=-1), -1), (call(vocab=0), -1), (call(k=0), -1), (call(t=3), -1), (call(x=None), -1), (call(W=None), -1), (call(target=None), -1), (call(ldx=7), -1), (call(ldw=7), -1),
                          (call(x=p + 2), -1), (call(W=p + 1, t=2), -1), (call(target=p + 2), -1), (call(w=p + 1), -1), (call(st=p + 4), -1), (call(space=None), -5), (call(n=8), -5), (call(space=ws + 8), -1),
                          (call(rows=1 << 31), -2), (call(vocab=1 << 31), -2), (call(k=1 << 31, ldx=1 << 31, ldw=1 << 31), -2)]:
            assert got == want, lib.s2v_last_error(h)
    for got, want in [(loss(out=None), -1), (loss(out=p + 4098), -1), (grad(st=None), -1), (grad(lddx=7), -1), (grad(lddw=7), -1), (grad(dx=p + 4098), -1), (grad(dW=p + 1), -1)]:
        assert got == want, lib.s2v_last_error(h)
    assert loss(rows=0) == 0 and grad(dx=None, dW=None) == 0
    gpu_ctx.synchronize()
    assert not f.any()


# ---------------------------------------------------------------- every form of the calls: a few classes, tiles of logits, kept logits
FORMS = {"few": (48, 30, 40), "tiled": (150, 300, 136), "kept": (60, 70, 2100)}


def with_an_infinite_weight(form, dtype):
    """Weights of class 4 with an infinity in column 3, and every x there -1: logits of class 4 are -infinity."""
    rows, vocab, k = FORMS[form]
    x, W, target, weight = inputs(rows, vocab, k, dtype, seed=11, ignored=False)
    target[target == 4] = 5
    x[:, 3], W[4, 3] = -1.0, float("inf")
    return x, W, target, weight


# (fp32 operands go to the tensor cores as sums of three numbers, which infinities have none: tiled and kept forms give NaN)
@gpu
@pytest.mark.parametrize("form,dtype", [("few", "f32"), ("few", "f16"), ("few", "bf16"), ("tiled", "f16"), ("tiled", "bf16"), ("kept", "f16"), ("kept", "bf16")])
def test_an_own_logit_of_infinity_has_no_loss(gpu_ctx, form, dtype):
    x, W, target, weight = with_an_infinite_weight(form, dtype)
    x[7, 3], target[7] = 1.0, 4            # the one row with +infinity among its logits, and that its own class's
    loss, dx, dW = both(gpu_ctx, x, W, target, weight)
    assert bool(loss[7].isnan()) and bool(loss[:7].isfinite().all()) and bool(loss[8:].isfinite().all())
    assert bool(dx[7].isnan().all()) and bool(dW.isnan().all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", FORMS)
def test_a_gradient_with_other_row_weights_than_the_loss(gpu_ctx, form, dtype):
    rows, vocab, k = FORMS[form]
    x, W, target, weight = inputs(rows, vocab, k, dtype, seed=12)
    other = weight.flip(0) * 1.5
    weight[5:9], other[7:12] = 0.0, 0.0                     # in one call alone, and in both
    x[[1, rows // 2, rows - 1, rows // 4]] = 0.0            # (rows of the helper's that one of the calls may count)
    target[1], x[1] = -1, float("nan")                      # no class: left out in either
    x[8] = float("nan")                                     # left out by weights of 0 in either
    loss, stats = torch.full((rows,), 5.0, device="cuda"), torch.full((rows, 2), 5.0, device="cuda")
    dx, dW, ws = torch.full_like(x, 5.0), torch.full_like(W, 5.0), space(gpu_ctx, rows, vocab, k, W.dtype)
    torch.cuda.synchronize()
    gpu_ctx.linear_cross_entropy(x, W, target, loss, ws, row_weight=weight, stats=stats)
    gpu_ctx.linear_cross_entropy_grad(x, W, target, stats, ws, dx=dx, dW=dW, row_weight=other)
    gpu_ctx.synchronize()
    Reference(x, W, target, weight).check_loss(loss)
    ref = Reference(x, W, target, other)
    ref.check_grad(dx, dW)
    assert not dx[~ref.live].any()
    # the loss is the same without stats, and without a weight the gradient is that of every row with a class
    again = torch.full((rows,), 5.0, device="cuda")
    gpu_ctx.linear_cross_entropy(x, W, target, again, ws, row_weight=weight)
    x[8] = 0.25
    torch.cuda.synchronize()
    gpu_ctx.linear_cross_entropy(x, W, target, loss, ws, row_weight=torch.zeros_like(weight), stats=stats)
    gpu_ctx.linear_cross_entropy_grad(x, W, target, stats, ws, dx=dx, dW=dW)
    gpu_ctx.synchronize()
    Reference(torch.where(x.isnan(), 0.0, x), W, target, weight).check_loss(again)
    assert not loss.any()
    Reference(x, W, target, None).check_grad(dx, dW)


@gpu
@pytest.mark.parametrize("form,dtype", [("few", "f32"), ("few", "f16"), ("few", "bf16"), ("tiled", "f16"), ("tiled", "bf16"), ("kept", "f16"), ("kept", "bf16")])
def test_an_own_logit_of_minus_infinity_leaves_the_others_their_gradients(gpu_ctx, form, dtype):
    x, W, target, weight = with_an_infinite_weight(form, dtype)
    target[7] = 4
    loss, dx, dW = both(gpu_ctx, x, W, target, weight)
    assert float(loss[7]) == float("inf") * weight[7].sign() and bool(loss[:7].isfinite().all()) and bool(loss[8:].isfinite().all())
    # the other classes' logits as without class 4, whose G is -w in row 7 and 0 elsewhere
    rest = torch.arange(W.shape[0], device="cuda") != 4
    ref = Reference(x, W[rest], torch.where(target > 4, target - 1, target), weight)
    ref.G[7] = ref.w[7] * (ref.x[7] @ ref.W.t()).softmax(0)
    ref.p[7] = ref.G[7] / ref.w[7]
    G, p, used = torch.zeros(x.shape[0], W.shape[0], dtype=torch.float64, device="cuda"), torch.zeros(x.shape[0], W.shape[0], dtype=torch.float64, device="cuda"), W.double()
    G[:, rest], p[:, rest] = ref.G, ref.p
    G[7, 4], used[4, 3] = -ref.w[7], 0.0
    ref.G, ref.p, ref.W = G, p, used
    dx[:, 3] = (G @ used)[:, 3].to(dx.dtype)     # (products with the infinity: infinite, or NaN as 0 times it is)
    ref.check_grad(dx, dW)


# ---------------------------------------------------------------- every form at its limits: certain rows, weights far apart
# (fp32 takes three 16-bit numbers an operand, and so six panels for one: fewer columns make its sums long)
@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(40, 40, 64), (40, 300, 300), (40, 40, 2100)], ids=["few", "tiled", "kept"])
def test_certain_rows_in_every_form(gpu_ctx, rows, vocab, k, dtype):
    # logits of 20 to 60 in the own class and 0 in the others: losses of vocab e^-20 and far less; all logits are exact
    W = torch.eye(vocab, k, device="cuda").to(TYPES[dtype])
    at = torch.arange(rows, device="cuda") * (vocab // rows)
    x = torch.zeros((rows, k), device="cuda")
    x[torch.arange(rows), at] = torch.linspace(20, 60, rows, device="cuda")
    x = x.to(TYPES[dtype])
    target = at.to(torch.int32)
    loss, dx, dW = both(gpu_ctx, x, W, target, None)
    ref = Reference(x, W, target, None)
    ref.check_loss(loss)
    ref.check_grad(dx, dW)
    # the others' exponentials are equal, and their sum in any order off by a rounding each; two steps of the exponential, the logarithm in 64 bits, the loss rounded
    assert bool(((loss.double() / ref.loss - 1).abs() < U * (vocab + 150)).all()) and float(loss[-1]) < 1e-20
    # dx of the own class is its G: rounded to the type, with `fix` for what 16 bits of G lose, so that the type's rounding of dx is left, and fp16's smallest step
    own, want = dx[torch.arange(rows), at].double(), torch.expm1(-ref.one)
    f = torch.finfo(TYPES[dtype])
    assert bool(((own - want).abs() <= want.abs() * (f.eps / 2 + U * (vocab + 200)) + f.smallest_normal * f.eps).all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(48, 30, 64), (200, 700, 136), (60, 40, 2100)], ids=["few", "tiled", "kept"])
def test_weights_six_decades_apart_in_every_form(gpu_ctx, rows, vocab, k, dtype):
    x, W, target, _ = inputs(rows, vocab, k, dtype, seed=13, ignored=False)
    weight = torch.logspace(-3, 3, rows, device="cuda")[torch.randperm(rows, generator=torch.Generator().manual_seed(3))]
    weight[::3] *= -1.0
    loss, dx, dW = both(gpu_ctx, x, W, target, weight)
    ref = Reference(x, W, target, weight)
    ref.check_loss(loss)
    ref.check_grad(dx, dW)


# ---------------------------------------------------------------- all of fp32: sums of so few terms that a lost part of an operand shows
def spare(rows, k, gen, low, high):
    """[rows x k] with one number a row, of any fp32 mantissa, in column after column."""
    x = torch.zeros((rows, k), device="cuda")
    i = torch.arange(rows, device="cuda")
    sign = torch.randint(0, 2, (rows,), generator=gen, device="cuda") * 2.0 - 1.0
    x[i, i * 7 % k] = sign * (low + (high - low) * torch.rand(rows, generator=gen, device="cuda"))
    return x


# An operand in three bf16 numbers is off by 2^-27 of it, and six of nine products leave out 2^-26 and two of 2^-35: together below 2^-24.  Each of the six that are added to others is a
# rounding, or a cut, twice as much; further terms of a sum are zeros and change nothing.  In units of sum |x W|, for `terms` products that are none:
def product_tol(terms):
    return U * (1 + 2 * 6 * terms + 2)


@gpu
@pytest.mark.parametrize("rows,k", [(600, 303), (600, 3207), (200, 41)], ids=["tiled", "kept", "few"])
def test_fp32_logits_keep_all_their_digits(gpu_ctx, rows, k):
    gen = torch.Generator(device="cuda").manual_seed(14)
    x = spare(rows, k, gen, 3.0, 6.0).abs()
    W = 3.0 + 3.0 * torch.rand((2, k), generator=gen, device="cuda")
    W[0] *= -1.0
    target = torch.zeros(rows, dtype=torch.int32, device="cuda")     # the class far behind: the loss is the two logits' difference, 18 to 72, and e^-18 and less
    loss, _, _ = both(gpu_ctx, x, W, target, None)
    z = x.double() @ W.double().t()
    want = torch.nn.functional.softplus(z[:, 1] - z[:, 0], threshold=1e9)
    # the logits are rounded as fp32 numbers, the loss too; of what the other class's exponential adds, at most e^-18, an error does not show
    tol = (product_tol(1) + U) * z.abs().sum(1) + U * want
    err = (loss.double() - want).abs()
    assert bool((err <= tol).all()), f"off by up to {float((err / tol).max()):.3g} of the tolerance"


@gpu
@pytest.mark.parametrize("rows,k", [(600, 303), (600, 3207), (200, 41)], ids=["tiled", "kept", "few"])
def test_fp32_gradients_keep_all_their_digits(gpu_ctx, rows, k):
    gen = torch.Generator(device="cuda").manual_seed(15)
    vocab = 3
    x = spare(rows, k, gen, 0.01, 0.02)
    W = 0.5 + torch.rand((vocab, k), generator=gen, device="cuda")
    target = torch.randint(0, vocab, (rows,), generator=gen, device="cuda").to(torch.int32)
    _, dx, dW = both(gpu_ctx, x, W, target, None)
    X, V = x.double(), W.double()
    z = X @ V.t()
    p = z.softmax(1)
    G = p.scatter_add(1, target.long()[:, None], torch.full((rows, 1), -1.0, dtype=torch.float64, device="cuda"))
    # |z| < 0.03: logits are off by less than 0.03 of product_tol(1), twice in an exponent that holds the kept log-sum-exp (1.1 and less) too, with three roundings of 1.2 * log2(e);
    # exponentials four steps, the sum of three, the product with the weight; of the own class's 1 - p, which is 0.6 and more, the same and its own rounding; three parts of G leave 2^-27
    assert float(z.abs().max()) < 0.03
    dg = (2 * 0.03 * product_tol(1) + U * (3 * 1.8 + 8 + 3 + 1 + 2 + 1)) * p.clamp(min=0.4) + U * G.abs()
    for got, a, b, da, terms in ((dx, G, V, dg, vocab), (dW, G.t(), X, dg.t(), int((X != 0).sum(0).max()))):
        want = a @ b
        tol = da @ b.abs() + product_tol(terms) * (a.abs() @ b.abs()) + U * want.abs()
        err = (got.double() - want).abs()
        assert bool((err <= tol * (1 + 1e-6)).all()), f"off by up to {float((err / tol).nan_to_num(0).max()):.3g} of the tolerance"


@gpu
@pytest.mark.parametrize("dtype,k", [("bf16", 32768), ("f16", 32768), ("f32", 8192)])
def test_long_sums_keep_the_losses_digits(gpu_ctx, dtype, k):
    # One class with a logit of thousands, a sum of terms that all have one sign, beside 9,599 of 0: the loss is that logit.  So many classes are tiles of logits, for two rows.
    gen = torch.Generator(device="cuda").manual_seed(16)
    x = (0.5 + 0.5 * torch.rand((2, k), generator=gen, device="cuda")).to(TYPES[dtype])
    W = torch.zeros((9600, k), dtype=TYPES[dtype], device="cuda")
    W[1] = (0.5 + 0.5 * torch.rand(k, generator=gen, device="cuda")).to(TYPES[dtype])
    target = torch.tensor([0, 9599], dtype=torch.int32, device="cuda")
    loss, ws = torch.empty(2, device="cuda"), space(gpu_ctx, 2, 9600, k, W.dtype, False)
    torch.cuda.synchronize()
    gpu_ctx.linear_cross_entropy(x, W, target, loss, ws)
    gpu_ctx.synchronize()
    want = x.double() @ W[1].double()
    # An accumulator of tensor memory takes 32 instructions, of 16 terms each; an instruction's 16 products and sum are cut in two places at most, a step of fp32 (2 U of the accumulator) each
    # (2,048 instructions to an accumulator gave 2,900 U).
    # Accumulators are added with a rounding each (512 numbers of k are one; six products of parts in fp32).
    accumulators = k // 512 * (6 if dtype == "f32" else 1)
    tol = U * (32 * 4 + accumulators + 4) * want
    err = (loss.double() - want).abs()
    assert bool((err <= tol).all()), f"off by up to {float((err / tol).max()):.3g} of the tolerance"
