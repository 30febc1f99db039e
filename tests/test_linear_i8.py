"""Dense layers with 8-bit weights: quantised rows, the product of 8-bit matrices and the whole layer, against the same formulas in 64 bits."""
import numpy as np
import pytest
import torch

from graphnn_b200 import capi

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- formulas
def quantized(x):
    """The definition in numpy's fp32, one operation at a time: q, scale."""
    x = x.detach().cpu().float().numpy()
    a = np.abs(x).max(axis=1, initial=np.float32(0))
    with np.errstate(all="ignore"):
        fine = np.isfinite(a) & (a >= np.float32(2.0 ** -110))
        f = np.where(fine, np.float32(127) / a, np.float32(0)).astype(np.float32)
        q = np.where(fine[:, None], np.rint(x * f[:, None]), np.float32(0))
        scale = np.where(fine, a / np.float32(127), np.float32(0)).astype(np.float32)
    scale[~np.isfinite(a)] = np.nan
    return q.astype(np.int8), scale


def product(a, sa, b, sb, bias, relu):
    """In 64 bits, and the size of what was added up for the tolerance."""
    acc = (a.to(b.device).double() @ b.double().t()).cpu()     # whole numbers below 2^31: exact in any order
    y = sa.double().cpu()[:, None] * sb.double().cpu()[None, :] * acc
    size = y.abs()
    if bias is not None:
        y = y + bias.double().cpu()
        size = size + bias.double().cpu().abs()
    return (torch.where(y < 0, 0.0, y) if relu else y), size


def assert_product(got, want, size):
    # scales' product, the sum as fp32 and the last addition: half a step of fp32 each; then half a step of the type (of its smallest number, below its range)
    f = torch.finfo(got.dtype)
    tol = 3 * 2.0 ** -24 * size + f.eps / 2 * (want.abs() + 4 * 2.0 ** -24 * size) + f.smallest_normal * f.eps / 2
    # Rounded to nearest, what lies half a step beyond the type's largest number, (2 - eps) 2^e, is infinite: from its (1 + eps / 4)-fold on, about.
    got = got.double().cpu()
    over, may = want.abs() - tol >= f.max * (1 + f.eps / 4), want.abs() + tol >= f.max * (1 + f.eps / 4)
    infinite = got == want.sign() * float("inf")
    assert bool((infinite | ~over).all())
    got, want, tol = (v.masked_fill(infinite & may, 0.0) for v in (got, want, tol))
    err = (got - want).abs()
    assert got.shape == want.shape and bool((err <= tol).all()), f"off by up to {float((err / tol).max()):.3g} of the tolerance"


def matrix(rows, cols, ld, gen, dtype=torch.float32, device="cuda"):
    """A [rows x cols] view of a buffer with leading dimension ld, and the buffer."""
    buf = torch.randn((rows, ld), generator=gen, device=device)
    buf = (buf * 50).round().clamp(-128, 127).to(torch.int8) if dtype == torch.int8 else buf.to(dtype)
    return buf[:, :cols], buf


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------- the binding's own checks (no GPU: the library call is recorded)
@pytest.fixture
def recorded():
    ctx, calls = object.__new__(capi.Context), []
    ctx.device, ctx.h = -1, None     # CPU tensors report device -1
    ctx.call = lambda name, stream, *args: calls.append((name, args))
    return ctx, calls


def test_binding_passes_sizes_and_leading_dimensions(recorded):
    ctx, calls = recorded
    x, q = torch.zeros(5, 24)[:, :20], torch.zeros(5, 32, dtype=torch.int8)[:, :20]
    w, y = torch.zeros(7, 48, dtype=torch.int8)[:, :20], torch.zeros(5, 9, dtype=torch.bfloat16)[:, :7]
    s5, s7 = torch.zeros(5), torch.zeros(7)
    ctx.quantize_rows_i8(x, q, s5)
    ctx.gemm_i8(q, s5, w, s7, y, relu=True)
    ctx.linear_i8(x.half(), w, s7, y, torch.zeros(999, dtype=torch.uint8), bias=s7)
    (n0, a0), (n1, a1), (n2, a2) = calls
    assert n0 == "s2v_quantize_rows_i8" and (a0[0], a0[1], a0[2], a0[4], a0[6]) == (5, 20, 0, 24, 32)
    assert n1 == "s2v_gemm_i8" and a1[:3] == (5, 7, 20) and (a1[4], a1[7], a1[9], a1[10], a1[11], a1[13]) == (32, 48, None, 1, 2, 9)
    assert n2 == "s2v_linear_i8" and a2[:4] == (5, 7, 20, 1) and (a2[5], a2[7], a2[9], a2[10], a2[12], a2[13], a2[15]) == (20, 48, s7.data_ptr(), 0, 999, 2, 9)


def test_binding_refuses_what_the_library_cannot_see(recorded):
    ctx, calls = recorded
    x, q, s = torch.zeros(4, 16), torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)
    w, sw, y, ws = torch.zeros(8, 16, dtype=torch.int8), torch.zeros(8), torch.zeros(4, 8), torch.zeros(1000, dtype=torch.uint8)
    bad = [lambda: ctx.quantize_rows_i8(x.double(), q, s), lambda: ctx.quantize_rows_i8(x, q.to(torch.uint8), s), lambda: ctx.quantize_rows_i8(x, q[:, :8], s),
           lambda: ctx.quantize_rows_i8(x, q, s[:3]), lambda: ctx.quantize_rows_i8(x, q, s.double()), lambda: ctx.quantize_rows_i8(x.t().contiguous().t(), q, s),
           lambda: ctx.quantize_rows_i8(x, q, torch.zeros(8)[::2]), lambda: ctx.gemm_i8(q, s, w[:, :8], sw, y), lambda: ctx.gemm_i8(q, s, w, sw, y.t()),
           lambda: ctx.gemm_i8(q, s, w, sw, y.int()), lambda: ctx.gemm_i8(q, s, w, sw, y, bias=s), lambda: ctx.gemm_i8(q.float(), s, w, sw, y),
           lambda: ctx.linear_i8(x.int(), w, sw, y, ws), lambda: ctx.linear_i8(x, w, s, y, ws), lambda: ctx.linear_i8(x, w, sw, y, ws.view(10, 100).t())]
    for i, f in enumerate(bad):
        with pytest.raises(capi.S2VError) as e:
            f()
        assert e.value.status == -1, i
    assert not calls


def test_no_context_and_workspace_sizes():
    lib = capi.load_library()
    assert lib.s2v_quantize_rows_i8(None, None, 1, 1, 0, None, 1, None, 1, None) == -1
    assert lib.s2v_gemm_i8(None, None, 1, 1, 1, None, 16, None, None, 16, None, None, 0, 0, None, 1) == -1
    assert lib.s2v_linear_i8(None, None, 1, 1, 1, 0, None, 1, None, 16, None, None, 0, None, 0, 0, None, 1) == -1
    assert lib.s2v_linear_i8_workspace_bytes(0, 5) == 0 and lib.s2v_linear_i8_workspace_bytes(-1, 5) == 0 and lib.s2v_linear_i8_workspace_bytes(3, -1) == 0
    for m, k in ((1, 1), (3, 17), (1000, 4096), (1 << 22, 1 << 14)):
        assert lib.s2v_linear_i8_workspace_bytes(m, k) >= m * ((k + 15) // 16 * 16 + 4)


# ---------------------------------------------------------------- quantised rows
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 1000, 0), (3, 17, 0), (7, 128, 1), (64, 128, 0), (300, 82, 3), (5, 4099, 2), (2, 70001, 0), (2500, 256, 8), (37, 8192, 0), (90, 29, 0), (1111, 63, 1), (500, 129, 0), (64, 254, 3)])
def test_quantized_rows(gpu_ctx, dtype, rows, cols, pad):
    gen = generator(rows * 7 + cols)
    x, _ = matrix(rows, cols, cols + pad, gen, TYPES[dtype])
    q, qbuf = matrix(rows, cols, cols + 2 * pad, gen, torch.int8)
    before = qbuf.clone()
    scale = torch.full((rows,), -1.0, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.quantize_rows_i8(x, q, scale)
    gpu_ctx.synchronize()
    want_q, want_scale = quantized(x)
    assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(scale.cpu().numpy(), want_scale)
    assert torch.equal(qbuf[:, cols:], before[:, cols:])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [5, 96, 2051])
def test_quantized_rows_of_special_values(gpu_ctx, dtype, cols):
    t = TYPES[dtype]
    big, small, inf = torch.finfo(t).max, torch.finfo(t).smallest_normal, float("inf")
    x = torch.randn((10, cols), generator=generator(cols), device="cuda").to(t)
    x[0] = 0
    x[1] = -0.0
    x[2, -1] = inf
    x[3, 0] = float("nan")
    x[4, cols // 2] = -inf
    x[5, 1] = -big
    x[6] = small
    x[7] = 0
    x[7, -1] = small / 2 if dtype != "f32" else 2.0 ** -140     # a number below the normal ones
    x[8] = torch.arange(cols, device="cuda") % 2 * 253.0 - 126.5    # ties: +-126.5 of 126.5
    x[9] = 0
    x[9, 0], x[9, 1] = 127.0, 0.5                                    # a tie goes to the even neighbour: 0
    q, scale = torch.full((10, cols), 55, dtype=torch.int8, device="cuda"), torch.empty(10, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.quantize_rows_i8(x, q, scale)
    gpu_ctx.synchronize()
    want_q, want_scale = quantized(x)
    assert np.array_equal(scale.cpu().numpy(), want_scale, equal_nan=True) and np.array_equal(q.cpu().numpy(), want_q)
    assert np.isnan(want_scale[2:5]).all() and not want_q[2:5].any() and want_q[9, 1] == 0


@gpu
def test_quantized_rows_without_columns(gpu_ctx):
    scale = torch.full((4,), 3.0, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.quantize_rows_i8(torch.empty((4, 0), device="cuda"), torch.empty((4, 0), dtype=torch.int8, device="cuda"), scale)
    gpu_ctx.quantize_rows_i8(torch.empty((0, 7), device="cuda"), torch.empty((0, 7), dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"))
    gpu_ctx.synchronize()
    assert not scale.any()


# ---------------------------------------------------------------- the product
SHAPES = [(1, 1, 1), (1, 8, 16), (1, 333, 4096), (2, 1000, 100), (3, 17, 33), (5, 4096, 1024), (8, 129, 2047), (9, 250, 640), (16, 2048, 4096), (17, 640, 129),
          (33, 500, 1000), (64, 1536, 512), (65, 257, 8192), (100, 100, 100), (127, 127, 127), (128, 256, 128), (129, 255, 257), (300, 1021, 1504), (513, 770, 200),
          (1000, 24, 4096), (2049, 264, 96), (1500, 1500, 1500), (4100, 513, 64),
          (2100, 2304, 640), (4000, 1300, 1000), (129, 38000, 520), (5000, 1025, 513)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(gpu_ctx, m, n, k, dtype):
    gen = generator(m + 3 * n + 7 * k)
    up = (k + 15) // 16 * 16
    odd = (m + n + k) % 3
    a, _ = matrix(m, k, up + 16 * odd, gen, torch.int8)
    b, _ = matrix(n, k, up + 32 * odd, gen, torch.int8)
    sa, sb = torch.rand(m, generator=gen, device="cuda") * 1e-2, torch.rand(n, generator=gen, device="cuda") * 1e-2
    bias = torch.randn(n, generator=gen, device="cuda") if (m + n) % 2 else None
    relu = k % 2 == 1
    guard = torch.full((m + 2, n + odd), 7.0, dtype=TYPES[dtype], device="cuda")     # a row in front and behind, and columns beside
    c = guard[1:m + 1, :n]
    torch.cuda.synchronize()
    gpu_ctx.gemm_i8(a, sa, b, sb, c, bias=bias, relu=relu)
    gpu_ctx.synchronize()
    want, size = product(a, sa, b, sb, bias, relu)
    assert_product(c, want, size)
    assert bool((guard[0] == 7).all() and (guard[-1] == 7).all() and (guard[:, n:] == 7).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,ld", [(300, 1021, 700, 1024), (300, 1, 64, 16), (1, 1021, 64, 1021), (70, 250, 200, 257), (500, 2001, 130, 2016), (2500, 2041, 640, 2048), (3, 3, 20, 8),
                                      (2500, 2043, 640, 2043), (9000, 130, 128, 131)])
def test_outputs_inside_a_wider_matrix(gpu_ctx, m, n, k, ld, dtype):
    """What lies beside and behind the outputs stays as it was, wherever rows start."""
    gen = generator(m + n + k)
    up = (k + 15) // 16 * 16
    a, b = matrix(m, k, up, gen, torch.int8)[0], matrix(n, k, up, gen, torch.int8)[0]
    sa, sb = torch.rand(m, generator=gen, device="cuda"), torch.rand(n, generator=gen, device="cuda")
    want, size = product(a, sa, b, sb, None, False)
    for shift in (0, 1, 8):
        buf = torch.full((m * ld + shift + 40,), 3.0, dtype=TYPES[dtype], device="cuda")
        c = buf[shift:shift + m * ld].view(m, ld)[:, :n]
        torch.cuda.synchronize()
        gpu_ctx.gemm_i8(a, sa, b, sb, c)
        gpu_ctx.synchronize()
        assert_product(c, want, size)
        rest = buf.clone()
        rest[shift:shift + m * ld].view(m, ld)[:, :n] = 3.0
        assert bool((rest == 3).all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(9999, 257, 33), (9999, 513, 129), (47001, 129, 129), (9999, 1025, 257), (15001, 257, 520), (15001, 257, 1001), (47001, 129, 1001), (47001, 129, 2050)])
def test_product_of_many_tiles(gpu_ctx, m, n, k, dtype):
    """Several tiles a CTA, with rows of outputs that start anywhere and on 16 bytes."""
    gen = generator(m + n + k)
    up = (k + 15) // 16 * 16
    a, b = matrix(m, k, up, gen, torch.int8)[0], matrix(n, k, up, gen, torch.int8)[0]
    sa, sb, bias = torch.rand(m, generator=gen, device="cuda") * 1e-2, torch.rand(n, generator=gen, device="cuda") * 1e-2, torch.randn(n, generator=gen, device="cuda")
    want, size = product(a, sa, b, sb, bias, True)
    for ld in (n, (n + 15) // 16 * 16):
        buf = torch.full((m, ld), 3.0, dtype=TYPES[dtype], device="cuda")
        torch.cuda.synchronize()
        gpu_ctx.gemm_i8(a, sa, b, sb, buf[:, :n], bias=bias, relu=True)
        gpu_ctx.synchronize()
        assert_product(buf[:, :n], want, size)
        assert bool((buf[:, n:] == 3).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,ld,k", [(20000, 1021, 1024, 64), (20000, 1021, 1024, 128), (30011, 2041, 2048, 128), (20000, 2041, 2048, 64), (60000, 253, 256, 32), (9000, 1021, 1040, 300)])
def test_many_tiles_whose_rows_end_inside_16_bytes(gpu_ctx, m, n, ld, k, dtype):
    """Few sums an output and a CTA's tiles one right behind the other; a tile's last columns leave by stores, those in front of them and the next tile's by
    copies.  Scales of powers of two: every output is exact before its only rounding, so that all of them are equal, in every one of many calls."""
    gen = generator(m + n + k)
    a, b = matrix(m, k, (k + 15) // 16 * 16, gen, torch.int8)[0], matrix(n, k, (k + 15) // 16 * 16, gen, torch.int8)[0]
    sa, sb = (torch.exp2(torch.randint(-6, 0, (r,), generator=gen, device="cuda").float()) for r in (m, n))
    want = torch.cat([(part.double() @ b.double().t()).float() for part in a.split(10000)]) * sa[:, None] * sb[None, :]
    want = want.to(TYPES[dtype])
    c = torch.empty((m, ld), dtype=TYPES[dtype], device="cuda")
    for _ in range(12):
        c.fill_(3)
        torch.cuda.synchronize()
        gpu_ctx.gemm_i8(a, sa, b, sb, c[:, :n])
        gpu_ctx.synchronize()
        assert torch.equal(c[:, :n], want) and bool((c[:, n:] == 3).all())


@gpu
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_product_sums_are_exact_at_the_longest_rows(gpu_ctx, m):
    k, n = 131071, 70
    a, b = torch.full((m, 131072), -128, dtype=torch.int8, device="cuda")[:, :k], torch.full((n, 131072), -128, dtype=torch.int8, device="cuda")[:, :k]
    b[1] = 127
    b[2, 1:] = 0
    b[3, 0] = 127
    c = torch.empty((m, n), device="cuda")
    one = torch.ones(max(m, n), device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.gemm_i8(a, one[:m], b, one[:n], c)
    gpu_ctx.synchronize()
    want = a.long().cpu()[0] @ b.long().cpu().t()
    assert want[0] == 2147467264
    assert torch.equal(c.cpu(), want.to(torch.float32)[None, :].expand(m, n))


@gpu
@pytest.mark.parametrize("m", [1, 20, 300])
def test_product_of_no_columns_and_of_nan_scales(gpu_ctx, m):
    n, bias = 150, torch.randn(150, device="cuda")
    c = torch.empty((m, n), device="cuda")
    s, t = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    empty = lambda r: torch.empty((r, 0), dtype=torch.int8, device="cuda")  # noqa: E731
    torch.cuda.synchronize()
    gpu_ctx.gemm_i8(empty(m), s, empty(n), t, c, bias=bias)
    gpu_ctx.synchronize()
    assert torch.equal(c, bias.expand(m, n))
    gpu_ctx.gemm_i8(empty(0), s[:0], empty(n), t, c[:0])
    a, b = torch.ones((m, 64), dtype=torch.int8, device="cuda"), torch.ones((n, 64), dtype=torch.int8, device="cuda")
    s[m // 2] = float("nan")
    torch.cuda.synchronize()
    gpu_ctx.gemm_i8(a, s, b, t, c, relu=True)
    gpu_ctx.synchronize()
    assert bool(c[m // 2].isnan().all()) and int(c.isnan().sum()) == n and bool((c[:m // 2] == 64).all())


# ---------------------------------------------------------------- the layer
@gpu
@pytest.mark.parametrize("xtype,ytype", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 1000, 4096), (1, 77, 1001), (2, 512, 333), (4, 300, 2048), (7, 4096, 520), (16, 900, 4096), (60, 333, 777), (200, 256, 128),
                                   (1029, 256, 128), (5000, 64, 82), (700, 640, 1536)])
def test_layer_is_the_two_calls(gpu_ctx, m, n, k, xtype, ytype):
    gen = generator(m + n + k)
    x, _ = matrix(m, k, k + m % 3, gen, TYPES[xtype])
    w, _ = matrix(n, k, (k + 15) // 16 * 16, gen, torch.int8)
    sw, bias = torch.rand(n, generator=gen, device="cuda") * 0.01, torch.randn(n, generator=gen, device="cuda")
    q, sx = torch.empty((m, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :k], torch.empty(m, device="cuda")
    y, two = (torch.full((m, n), float("nan"), dtype=TYPES[ytype], device="cuda") for _ in range(2))
    ws = torch.empty(gpu_ctx.linear_i8_workspace_bytes(m, k), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.linear_i8(x, w, sw, y, ws, bias=bias, relu=True)
    gpu_ctx.quantize_rows_i8(x, q, sx)
    gpu_ctx.gemm_i8(q, sx, w, sw, two, bias=bias, relu=True)
    gpu_ctx.synchronize()
    assert torch.equal(y, two)
    want_q, want_s = quantized(x)
    assert_product(y, *product(torch.from_numpy(want_q), torch.from_numpy(want_s), w, sw, bias, True))


@gpu
def test_layer_of_rows_that_are_not_finite(gpu_ctx):
    for m in (3, 50, 400):
        x = torch.randn((m, 96), generator=generator(m), device="cuda").to(torch.bfloat16)
        x[1, 5], x[2] = float("inf"), 0
        w, sw = torch.ones((40, 96), dtype=torch.int8, device="cuda"), torch.ones(40, device="cuda")
        y = torch.empty((m, 40), device="cuda")
        ws = torch.empty(gpu_ctx.linear_i8_workspace_bytes(m, 96), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        gpu_ctx.linear_i8(x, w, sw, y, ws)
        gpu_ctx.synchronize()
        assert bool(y[1].isnan().all()) and not bool(y[2].any()) and int(y.isnan().sum()) == 40


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (6, 500, 1000), (30, 700, 2000), (300, 300, 300)])
def test_layer_captured_and_on_another_stream(gpu_ctx, m, n, k):
    gen = generator(m)
    kp = (k + 15) // 16 * 16
    x = torch.randn((m, k), generator=gen, device="cuda")
    w, _ = matrix(n, k, kp, gen, torch.int8)
    sw, y = torch.rand(n, generator=gen, device="cuda"), torch.empty((m, n), device="cuda")
    ws = torch.empty(gpu_ctx.linear_i8_workspace_bytes(m, k), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu_ctx.linear_i8(x, w, sw, y, ws, stream=side.cuda_stream)
    gpu_ctx.stream_status(side.cuda_stream)
    first = y.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gpu_ctx.linear_i8(x, w, sw, y, ws, stream=side.cuda_stream)
        gpu_ctx.linear_i8(x, w, sw, y, ws, stream=side.cuda_stream)    # the same workspace, in order
    for trial in range(3):
        y.fill_(-1)
        if trial:
            x.copy_(torch.randn((m, k), generator=gen, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        if trial == 0:
            assert torch.equal(y, first)
        q, s = quantized(x)
        assert_product(y, *product(torch.from_numpy(q), torch.from_numpy(s), w, sw, None, False))
    gpu_ctx.synchronize()


@gpu
def test_two_layers_at_once(gpu_ctx):
    """Calls on two streams, each with its own workspace, and graphs of them that replay side by side."""
    gen = generator(11)
    w, _ = matrix(700, 520, 528, gen, torch.int8)
    sw = torch.rand(700, generator=gen, device="cuda")
    calls = []
    for m in (2000, 40):
        x, y = torch.randn((m, 520), generator=gen, device="cuda"), torch.empty((m, 700), device="cuda")
        calls.append((x, y, torch.empty(gpu_ctx.linear_i8_workspace_bytes(m, 520), dtype=torch.uint8, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    first = []
    for x, y, ws, _ in calls:
        gpu_ctx.linear_i8(x, w, sw, y, ws)
        gpu_ctx.synchronize()
        first.append(y.clone())
    graphs = []
    for x, y, ws, side in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for _ in range(4):
                gpu_ctx.linear_i8(x, w, sw, y, ws, stream=side.cuda_stream)
        graphs.append(graph)
    for replayed in (False, True):
        for _, y, _, _ in calls:
            y.fill_(-1)
        torch.cuda.synchronize()
        for _ in range(5):
            for (x, y, ws, side), graph in zip(calls, graphs):
                if replayed:
                    with torch.cuda.stream(side):
                        graph.replay()
                else:
                    gpu_ctx.linear_i8(x, w, sw, y, ws, stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(c[1], f) for c, f in zip(calls, first))
    gpu_ctx.synchronize()


@gpu
def test_refusals(gpu_ctx):
    lib, h = gpu_ctx.lib, gpu_ctx.h
    f, i8 = torch.zeros(4096, device="cuda"), torch.zeros(8192, dtype=torch.int8, device="cuda")
    p, b = f.data_ptr(), i8.data_ptr()
    ws = gpu_ctx.linear_i8_workspace_bytes(4, 32)

    def quant(rows=4, cols=32, t=0, x=p, ldx=32, q=b, ldq=32, s=p):
        return lib.s2v_quantize_rows_i8(h, None, rows, cols, t, x, ldx, q, ldq, s)

    def gemm(m=4, n=4, k=32, a=b, lda=32, sa=p, w=b, ldb=32, sb=p, t=0, c=p, ldc=4):
        return lib.s2v_gemm_i8(h, None, m, n, k, a, lda, sa, w, ldb, sb, None, 0, t, c, ldc)

    def layer(m=4, n=4, k=32, xt=0, x=p, ldx=32, w=b, ldw=32, sw=p, wsp=b, wsb=ws, t=0, y=p, ldy=4):
        return lib.s2v_linear_i8(h, None, m, n, k, xt, x, ldx, w, ldw, sw, None, 0, wsp, wsb, t, y, ldy)

    for got, want in [(quant(rows=-1), -1), (quant(cols=-1), -1), (quant(t=3), -1), (quant(x=None), -1), (quant(q=None), -1), (quant(s=None), -1), (quant(ldx=31), -1),
                      (quant(ldq=31), -1), (quant(x=p + 2), -1), (quant(x=p + 1, t=1), -1),
                      (gemm(m=-1), -1), (gemm(n=-1), -1), (gemm(k=-1), -1), (gemm(t=-1), -1), (gemm(a=None), -1), (gemm(w=None), -1), (gemm(sa=None), -1), (gemm(sb=None), -1),
                      (gemm(c=None), -1), (gemm(lda=16), -1), (gemm(ldb=16), -1), (gemm(lda=40), -1), (gemm(ldb=40), -1), (gemm(ldc=3), -1), (gemm(a=b + 8), -1),
                      (gemm(w=b + 8), -1), (gemm(c=p + 2), -1), (gemm(k=131072, lda=131072, ldb=131072), -2), (gemm(m=1 << 31), -2), (gemm(n=1 << 31, ldc=1 << 31), -2),
                      (layer(wsb=ws - 1), -5), (layer(wsp=None), -5), (layer(wsp=b + 4), -1), (layer(xt=7), -1), (layer(t=7), -1), (layer(x=None), -1), (layer(w=None), -1),
                      (layer(ldx=31), -1), (layer(ldw=33), -1), (layer(y=None), -1), (layer(sw=None), -1), (layer(ldy=2), -1), (layer(k=131072, wsb=1 << 40), -2)]:
        assert got == want, lib.s2v_last_error(h)
    gpu_ctx.synchronize()
    assert not f.any() and not i8.any()
    for got in (quant(rows=1, ldx=0, ldq=0), quant(rows=0, x=None), gemm(m=1, lda=0, ldc=0), gemm(m=0, a=None), gemm(n=0, w=None), layer(m=0, wsp=None, wsb=0)):
        assert got == 0    # leading dimensions of single rows are not read; empty calls do nothing
    gpu_ctx.synchronize()


@gpu
def test_refusals_of_misaligned_scales_and_biases(gpu_ctx):
    lib, h = gpu_ctx.lib, gpu_ctx.h
    f, i8 = torch.zeros(4096, device="cuda"), torch.zeros(8192, dtype=torch.int8, device="cuda")
    p, b = f.data_ptr(), i8.data_ptr()
    ws = gpu_ctx.linear_i8_workspace_bytes(4, 32)
    for off in (1, 2, 3):
        assert lib.s2v_quantize_rows_i8(h, None, 4, 32, 0, p, 32, b, 32, p + off) == -1
        for sa, sb, bias in ((p + off, p, p), (p, p + off, p), (p, p, p + off)):
            assert lib.s2v_gemm_i8(h, None, 4, 4, 32, b, 32, sa, b, 32, sb, bias, 0, 0, p, 4) == -1
        for m in (1, 4):
            for sw, bias in ((p + off, p), (p, p + off)):
                assert lib.s2v_linear_i8(h, None, m, 4, 32, 0, p, 32, b, 32, sw, bias, 0, b, ws, 0, p, 4) == -1
    gpu_ctx.synchronize()
    assert not f.any() and not i8.any()
