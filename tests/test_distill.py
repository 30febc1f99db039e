"""Distillation from a teacher's top logits: loss and gradient against the formulas in 64 bits and against differences."""
import math

import pytest
import torch

from graphnn_b200 import capi

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")


# ---------------------------------------------------------------- formulas
def reference(z, idx, t, temp=1.0, t_lse=None, weight=None):
    """Loss and gradient of every row in 64 bits, an entry at a time; also q and sum p of each column, for tolerances."""
    z, t = z.double().cpu() / temp, t.double().cpu() / temp
    rows, cols = z.shape
    idx = idx.cpu()
    loss, dz = torch.zeros(rows, dtype=torch.float64), torch.zeros((rows, cols), dtype=torch.float64)
    size = torch.zeros((rows, cols), dtype=torch.float64)
    for i in range(rows):
        w = 1.0 if weight is None else float(weight[i])
        entries = [(int(j), t[i, k]) for k, j in enumerate(idx[i].tolist()) if 0 <= j < cols]
        if not entries or w == 0 or (t_lse is None and all(v == -INF for _, v in entries)):
            continue
        tv = torch.stack([v for _, v in entries])
        at = torch.tensor([j for j, _ in entries])
        if t_lse is None:
            p, rest = tv.softmax(0), 0.0
        else:
            p = (tv - t_lse[i].double().cpu()).exp()
            rest = max(0.0, 1.0 - float(p.sum()))
        log_q = z[i].log_softmax(0)
        q = log_q.exp()
        kl = sum((float(pk * (pk.log() - log_q[j])) for pk, j in zip(p, at.tolist()) if pk != 0), 0.0)
        outside = torch.ones(cols, dtype=torch.bool)
        outside[at] = False
        g = q * (float(p.sum()) + rest)
        size[i] = q.clone()
        if rest != 0:
            log_s = z[i][outside].logsumexp(0) - z[i].logsumexp(0) if outside.any() else torch.tensor(-INF, dtype=torch.float64)
            if log_s > -INF:
                kl += rest * (math.log(rest) - float(log_s))
                g[outside] -= rest * z[i][outside].softmax(0)
                size[i][outside] += rest * z[i][outside].softmax(0)
            elif rest > 2.0 ** -16:
                kl = INF
        g.index_add_(0, at, -p)
        size[i].index_add_(0, at, p)
        loss[i], dz[i], size[i] = w * kl, w / temp * g, size[i] * (abs(w) / temp)
    return loss, dz, size


def relative(cols, temp, z):
    """How far q_j may be from its value, relative to it, in the kernels' arithmetic.  The exponent's argument x = (z - M) * (log2 e / T) is off by its
    difference, its constant and its product: 3 half steps of fp32 of |x|, at most the row's range; ex2 by 2 steps; the sum of a thread's columns by
    half a step an addition (at most cols / 32 of them, or 64 where more threads share the row) and 16 more of the threads' sums.  All in units of 2^-24."""
    r = z.double()
    r = r[r.isfinite()]
    r = r[r > r.max() - 100 * temp] if r.numel() else r      # (what is further below adds less than e^-100 on either side)
    span = float(r.max() - r.min()) / temp * 1.4427 if r.numel() else 0.0
    return 2.0 ** -24 * (2 * (3 * span * 0.6932 + 4 + max(64, cols / 32) + 16))


def assert_matches(loss, dz, z, idx, t, temp=1.0, t_lse=None, weight=None):
    want, grad, size = reference(z, idx, t, temp, t_lse, weight)
    rel = relative(z.shape[1], temp, z)
    w = torch.ones(z.shape[0], dtype=torch.float64) if weight is None else weight.double().cpu().abs()
    for i in range(z.shape[0]):
        got, x = float(loss[i]), float(want[i])
        x = math.copysign(INF, x) if abs(x) >= 2.0 ** 128 else x     # (beyond fp32)
        if math.isnan(x) or math.isinf(x):
            assert got == x or (math.isnan(got) and math.isnan(x)), (i, got, x)
        else:   # log q and log s are off by `rel` at most, with weights that add up to one; and half a step of fp32
            assert abs(got - x) <= float(w[i]) * rel + 2.0 ** -24 * abs(x), (i, got, x, float(w[i]) * rel)
    if dz is None:
        return
    f = torch.finfo(dz.dtype)
    tol = rel * size + f.eps / 2 * (grad.abs() + rel * size) + f.smallest_normal * f.eps / 2
    got = dz.double().cpu()
    fine = grad.isfinite()
    assert bool((got[~fine].isnan() == grad[~fine].isnan()).all())
    err = (got - grad).abs()[fine]
    assert bool((err <= tol[fine]).all()), f"gradient off by up to {float((err / tol[fine]).max()):.3g} of the tolerance"


def inputs(rows, cols, top, dtype, seed, tail, temp, ragged=True, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    teacher = 3 * torch.randn((rows, cols), generator=gen)
    z = (teacher + torch.randn((rows, cols), generator=gen)).to(TYPES[dtype])
    t, idx = teacher.topk(min(top, cols), dim=1)
    if top > cols:
        t, idx = torch.nn.functional.pad(t, (0, top - cols)), torch.nn.functional.pad(idx, (0, top - cols), value=-1)
    idx = idx.to(torch.int32)
    if ragged:
        idx[torch.rand(idx.shape, generator=gen) < 0.15] = -1
        if rows > 2:
            idx[rows // 2] = -1
    lse = torch.logsumexp(teacher.double() / temp, 1).float() if tail else None
    weight = torch.rand(rows, generator=gen) * 2 - 0.2
    to = lambda v: None if v is None else v.to(device)  # noqa: E731
    return to(z), to(idx), to(t), to(lse), to(weight)


def both_ways(ctx, z, idx, t, temp=1.0, t_lse=None, weight=None):
    """(loss, dz) of the one call, after checking that the two calls and the loss alone give the same."""
    rows = z.shape[0]
    loss, dz = torch.full((rows,), 5.0, device="cuda"), torch.full(z.shape, 5.0, dtype=z.dtype, device="cuda")
    loss2, dz2, stats, loss3 = loss.clone(), dz.clone(), torch.full((rows, 4), 5.0, device="cuda"), loss.clone()
    more = {"temperature": temp, "t_lse": t_lse, "row_weight": weight}
    torch.cuda.synchronize()
    ctx.distill_topk(z, idx, t, loss, dz=dz, **more)
    ctx.distill_topk(z, idx, t, loss2, stats=stats, **more)
    ctx.distill_topk_grad(z, idx, t, stats, dz2, **more)
    ctx.distill_topk(z, idx, t, loss3, **more)
    ctx.synchronize()
    same = lambda a, b: torch.equal(a.nan_to_num(nan=12345.0), b.nan_to_num(nan=12345.0))  # noqa: E731
    assert same(loss, loss2) and same(loss, loss3)
    # the statistics are kept in fp32: three roundings of them, one more of the result
    a, b, f = dz.double(), dz2.double(), torch.finfo(dz.dtype)
    size = reference(z, idx, t, temp, t_lse, weight)[2].cuda()
    fine = a.isfinite()
    assert torch.equal(fine, b.isfinite())
    assert bool(((a - b).abs() <= 4 * 2.0 ** -24 * size + f.eps * a.abs() + f.smallest_normal * f.eps)[fine].all())
    return loss, dz


# ---------------------------------------------------------------- the binding's own checks
def test_binding_checks_its_arguments():
    ctx, calls = object.__new__(capi.Context), []
    ctx.device, ctx.h = -1, None
    ctx.call = lambda name, stream, *args: calls.append((name, args))
    z, idx, t, loss = torch.zeros(4, 12)[:, :10], torch.zeros((4, 5), dtype=torch.int32)[:, :3], torch.zeros((4, 5))[:, :3], torch.zeros(4)
    stats, dz = torch.zeros(4, 4), torch.zeros(4, 11)[:, :10]
    ctx.distill_topk(z, idx, t, loss, temperature=2.0, stats=stats, dz=dz)
    ctx.distill_topk_grad(z, idx, t, stats, dz, row_weight=loss)
    (n0, a0), (n1, a1) = calls
    assert n0 == "s2v_distill_topk" and (a0[0], a0[1], a0[2], a0[4], a0[5], a0[7], a0[9], a0[10], a0[11], a0[12]) == (4, 10, 0, 12, 3, 0, 5, None, 2.0, None)
    assert a0[13:] == (loss.data_ptr(), stats.data_ptr(), dz.data_ptr(), 11)
    assert n1 == "s2v_distill_topk_grad" and a1[12:] == (loss.data_ptr(), stats.data_ptr(), dz.data_ptr(), 11)
    calls.clear()
    bad = [lambda: ctx.distill_topk(z.double(), idx, t, loss), lambda: ctx.distill_topk(z, idx.long(), t, loss), lambda: ctx.distill_topk(z, idx, t[:, :2], loss),
           lambda: ctx.distill_topk(z, idx, torch.zeros(4, 3), loss), lambda: ctx.distill_topk(z, idx[:3], t, loss), lambda: ctx.distill_topk(z, idx, t, loss[:2]),
           lambda: ctx.distill_topk(z, idx, t, loss, dz=dz.half()), lambda: ctx.distill_topk(z, idx, t, loss, dz=dz[:, :9]), lambda: ctx.distill_topk(z, idx, t, loss, t_lse=z[:, 0]),
           lambda: ctx.distill_topk(z, idx, t, loss, row_weight=loss.double()), lambda: ctx.distill_topk(z, idx, t, loss, stats=stats[:, :3]),
           lambda: ctx.distill_topk(z, idx, t, loss, stats=torch.zeros(4, 8)[:, :4]), lambda: ctx.distill_topk_grad(z, idx, t, stats.half(), dz),
           lambda: ctx.distill_topk(z.t().contiguous().t(), idx, t, loss)]
    for i, f in enumerate(bad):
        with pytest.raises(capi.S2VError) as e:
            f()
        assert e.value.status == -1, i
    assert not calls
    lib = capi.load_library()
    assert lib.s2v_distill_topk(None, None, 1, 1, 0, None, 1, 1, None, 0, None, 1, None, 1.0, None, None, None, None, 0) == -1
    assert lib.s2v_distill_topk_grad(None, None, 1, 1, 0, None, 1, 1, None, 0, None, 1, None, 1.0, None, None, None, 0) == -1


def test_the_formula_of_the_gradient_is_the_losses_derivative():
    """The reference that the kernels are held to, against central differences in 64 bits."""
    for tail in (False, True):
        z, idx, t, lse, w = inputs(5, 9, 4, "f32", 3, tail, 1.7, device="cpu")
        idx[0, 1] = idx[0, 0]     # a class listed twice
        z = z.double()
        _, dz, _ = reference(z, idx, t, 1.7, lse, w)
        h = 1e-5
        for j in range(9):
            up, down = z.clone(), z.clone()
            up[:, j] += h
            down[:, j] -= h
            diff = (reference(up, idx, t, 1.7, lse, w)[0] - reference(down, idx, t, 1.7, lse, w)[0]) / (2 * h)
            assert torch.allclose(diff, dz[:, j], rtol=1e-6, atol=1e-8), (tail, j)


# ---------------------------------------------------------------- loss and gradient
SIZES = [(1, 1, 1), (3, 2, 1), (64, 6, 3), (5, 7, 16), (40, 33, 33), (9, 100, 256), (17, 255, 8), (6, 1000, 10), (130, 1023, 20), (3, 1025, 64), (5, 4097, 100), (2, 8192, 128), (4, 20011, 50),
         (1, 50021, 200), (2, 131072, 64), (300, 9001, 40), (3, 262144, 7), (302, 40003, 9)]


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,top", SIZES)
def test_loss_and_gradient(gpu_ctx, rows, cols, top, dtype, tail):
    temp = (1.0, 2.0, 0.5)[(rows + cols) % 3]
    z, idx, t, lse, w = inputs(rows, cols, top, dtype, cols + top, tail, temp)
    loss, dz = both_ways(gpu_ctx, z, idx, t, temp, lse, w)
    assert_matches(loss, dz, z, idx, t, temp, lse, w)
    assert float(loss[rows // 2]) == 0 or rows <= 2


@gpu
def test_the_longest_rows(gpu_ctx):
    for dtype, cols in (("bf16", 524288), ("f16", 524283)):
        z, idx, t, lse, w = inputs(2, cols, 30, dtype, 5, True, 1.0)
        loss, dz = both_ways(gpu_ctx, z, idx, t, 1.0, lse, w)
        assert_matches(loss, dz, z, idx, t, 1.0, lse, w)


@gpu
@pytest.mark.parametrize("ttype", TYPES)
def test_teacher_types_strides_and_gradients_in_place(gpu_ctx, ttype):
    for dtype in TYPES:
        for cols, off, ld in ((300, 0, 307), (300, 3, 303), (5000, 1, 5001), (5000, 0, 5000), (5003, 5, 5017)):
            z0, idx0, t0, lse, w = inputs(7, cols, 11, dtype, cols + off, True, 1.0)
            buf = torch.full((7 * ld + off,), 9.0, dtype=TYPES[dtype], device="cuda")
            z = buf[off:].view(7, ld)[:, :cols]
            z.copy_(z0)
            idx, t = torch.full((7, 16), -1, dtype=torch.int32, device="cuda")[:, 2:13], torch.zeros((7, 16), dtype=TYPES[ttype], device="cuda")[:, 2:13]
            idx.copy_(idx0)
            t.copy_(t0)
            out = torch.full((7, cols + 9), 4.0, dtype=TYPES[dtype], device="cuda")
            loss, loss2 = torch.empty(7, device="cuda"), torch.empty(7, device="cuda")
            torch.cuda.synchronize()
            gpu_ctx.distill_topk(z, idx, t, loss, t_lse=lse, row_weight=w, dz=out[:, 4:cols + 4])
            gpu_ctx.synchronize()
            assert_matches(loss, out[:, 4:cols + 4], z0, idx, t, 1.0, lse, w)
            assert bool((out[:, :4] == 4).all() and (out[:, cols + 4:] == 4).all()) and torch.equal(z, z0)
            gpu_ctx.distill_topk(z, idx, t, loss2, t_lse=lse, row_weight=w, dz=z)
            gpu_ctx.synchronize()
            assert torch.equal(loss, loss2) and torch.equal(z, out[:, 4:cols + 4])
            assert bool((buf[:off] == 9).all()) and (ld == cols or bool((buf[off:].view(7, ld)[:, cols:] == 9).all()))
            z.copy_(z0)
            stats = torch.empty((7, 4), device="cuda")
            torch.cuda.synchronize()
            gpu_ctx.distill_topk(z, idx, t, loss2, t_lse=lse, stats=stats)
            gpu_ctx.distill_topk_grad(z, idx, t, stats, z, t_lse=lse, row_weight=w)
            gpu_ctx.synchronize()
            assert_matches(loss2, None, z0, idx, t, 1.0, lse, None)
            assert_matches(loss, z, z0, idx, t, 1.0, lse, w)


@gpu
@pytest.mark.parametrize("cols", [12, 700, 6000, 40000])
@pytest.mark.parametrize("tail", [False, True])
def test_rows_that_masks_leave_empty_and_values_that_are_not_finite(gpu_ctx, cols, tail):
    for dtype in TYPES:
        low = torch.finfo(TYPES[dtype]).min
        z, idx, t, lse, _ = inputs(16, cols, 6, dtype, cols, tail, 1.0, ragged=False)
        w = torch.ones(16, device="cuda")
        idx[0] = -1                                     # no list, and a row that holds nothing usable
        z[0] = float("nan")
        w[1], z[1] = 0.0, -INF                          # a padded row
        t[2] = -INF                                     # a teacher without mass (with t_lse: all of it outside the list)
        t[3, 2:] = -INF                                 # entries without mass
        z[4, idx[4, 3].long()] = -INF                   # the student excludes a class that the teacher wants: infinite
        z[5] = torch.where(torch.zeros(cols, device="cuda").index_fill_(0, idx[5].long(), 1.0) > 0, z[5].float(), -INF).to(z.dtype)  # nothing outside the list
        z[6] = torch.where(torch.zeros(cols, device="cuda").index_fill_(0, idx[6].long(), 1.0) > 0, z[6].float(), low).to(z.dtype)   # the type's lowest value
        z[7, cols - 1] = float("nan")
        z[8, idx[8, 0].long()] = float("nan")
        z[9, 0] = INF
        z[10] = -INF
        t[11, 0] = float("nan")
        idx[12, 1] = idx[12, 0]                         # a class listed twice
        idx[13, 1:] = idx[13, 0]                        # ... and again
        z[14] = 0.0
        z[15], z[15, idx[15, 0].long()] = low, -low / 2   # nearly all mass on one class
        if lse is not None:
            lse[5] = torch.logsumexp(t[5], 0)           # the teacher gives nothing to the others either
        loss, dz = both_ways(gpu_ctx, z, idx, t, 1.0, lse, w)
        assert not loss[:2].any() and not dz[:2].any() and (tail or (not loss[2] and not dz[2].any()))
        for i in (7, 8, 9, 10, 11):
            assert math.isnan(loss[i]) and bool(dz[i].isnan().all()), i
            z[i], t[i], idx[i] = 0.0, 0.0, -1           # (the reference need not agree on these)
        loss[7:12], dz[7:12] = 0.0, 0.0
        z[:2] = 0.0
        for i in range(16):   # a row at a time: the tolerance goes by the row's own range
            at = slice(i, i + 1)
            assert_matches(loss[at], dz[at], z[at], idx[at], t[at], 1.0, None if lse is None else lse[at], w[at])
        assert math.isinf(loss[4])


@gpu
@pytest.mark.parametrize("cols", [12, 700, 6000, 40000])
@pytest.mark.parametrize("tail", [False, True])
def test_teachers_that_are_not_finite(gpu_ctx, cols, tail):
    z, idx, t, lse, w = inputs(6, cols, 5, "f32", cols, tail, 1.0, ragged=False)
    w.fill_(0.5)
    t[0, 1], t[1, 4], t[2, 0] = INF, float("nan"), -INF
    idx[3, 2], t[3, 2] = -1, float("nan")               # an entry that is not there
    if tail:
        lse[4] = float("nan")
    loss, dz = both_ways(gpu_ctx, z, idx, t, 1.0, lse, w)
    for i in (0, 1, 4) if tail else (0, 1):
        assert math.isnan(loss[i]) and bool(dz[i].isnan().all()), i
    rows = [2, 3, 5]
    assert_matches(loss[rows], dz[rows], z[rows], idx[rows], t[rows].nan_to_num(nan=0.0, neginf=-INF), 1.0, None if lse is None else lse[rows], w[rows])


@gpu
@pytest.mark.parametrize("rows,cols,dtype,top", [(9, 12, "f32", 5), (9, 700, "f16", 5), (9, 2050, "f32", 40), (9, 6000, "bf16", 7), (9, 40000, "f32", 130), (460, 8203, "f32", 5), (460, 20001, "bf16", 129)])
@pytest.mark.parametrize("tail", [False, True])
def test_teachers_without_a_number(gpu_ctx, rows, cols, dtype, top, tail):
    """A list of NaN alone, or of NaN and -infinity, gives NaN; only one where every t is -infinity is a teacher without mass."""
    z, idx, t, lse, _ = inputs(9, cols, top, dtype, cols, tail, 1.0, ragged=False)
    w = torch.ones(9, device="cuda")
    nan = float("nan")
    t[0] = nan
    t[1], t[1, top - 1] = -INF, nan
    t[2], idx[2, 1:] = nan, -1                          # a list of one entry
    t[3] = -INF
    t[4], idx[4, 0], t[4, 0] = -INF, -1, nan            # the NaN is at an entry that is not there
    t[5], w[5] = nan, 0.0                               # a padded row
    t[6], t[6, 0], t[6, 1] = -INF, nan, 0.5
    n = -(-rows // 9)
    z, idx, t, w = (v.repeat(n, *([1] * (v.dim() - 1)))[:rows].contiguous() for v in (z, idx, t, w))
    lse = None if lse is None else lse.repeat(n)[:rows].contiguous()
    loss, dz = torch.full((rows,), 5.0, device="cuda"), torch.full_like(z, 5.0)
    alone, kept, later, stats = loss.clone(), loss.clone(), dz.clone(), torch.empty((rows, 4), device="cuda")
    more = {"t_lse": lse, "row_weight": w}
    torch.cuda.synchronize()
    gpu_ctx.distill_topk(z, idx, t, loss, dz=dz, **more)
    gpu_ctx.distill_topk(z, idx, t, alone, **more)
    gpu_ctx.distill_topk(z, idx, t, kept, stats=stats, **more)
    gpu_ctx.distill_topk_grad(z, idx, t, stats, later, **more)
    gpu_ctx.synchronize()
    i = torch.arange(rows, device="cuda") % 9
    for of_nan in (0, 1, 2, 6):
        at = i == of_nan
        assert all(bool(v[at].isnan().all()) for v in (loss, alone, kept, dz, later)), of_nan
    empty = (i == 5) | ((i == 3) | (i == 4)) & (not tail)
    assert not any(bool(v[empty].any()) for v in (loss, alone, kept, dz, later))
    rest = [j for j in (3, 4, 5, 7, 8) if j < rows]
    t = t.nan_to_num(nan=0.0, neginf=-INF)
    for got, grad in ((loss, dz), (alone, None), (kept, later)):
        assert_matches(got[rest], None if grad is None else grad[rest], z[rest], idx[rest], t[rest], 1.0, None if lse is None else lse[rest], w[rest])


@gpu
@pytest.mark.parametrize("rows,cols,top", [(5, 700, 64), (5, 5000, 64), (5, 40003, 200), (450, 8203, 64)])
@pytest.mark.parametrize("temp,offset", [(1.5, 20.0), (1.5, 200.0), (3.0, 60.0), (0.7, -150.0)])
def test_small_rests_at_temperatures_that_are_no_powers_of_two(gpu_ctx, rows, cols, top, temp, offset):
    """A teacher that gives the list all but 1e-4, far from zero, and a student that does nearly the same: the gradient of what is not listed goes by rest / s."""
    temp = float(torch.tensor(temp))     # as the call takes it: 0.7 in fp32
    gen = torch.Generator().manual_seed(cols + top)
    idx = torch.stack([torch.randperm(cols, generator=gen)[:top] for _ in range(5)]).to(torch.int32)
    t = (offset + 3 * torch.randn((5, top), generator=gen)).float()
    # (t_lse as fp32 has it is the definition's: the rest is what it leaves, anywhere around 1e-4)
    lse = (torch.logsumexp(t.double() / temp, 1) - math.log1p(-1e-4)).float()
    z = 0.5 * temp * torch.randn((5, cols), generator=gen)
    z.scatter_(1, idx.long(), temp * (torch.randn((5, top), generator=gen) + math.log(cols / top) + 9.0))
    n = rows // 5
    z, idx, t, lse = (v.repeat(n, *([1] * (v.dim() - 1))).cuda() for v in (z, idx, t, lse))
    w = torch.full((rows,), 0.75, device="cuda")
    loss, dz = torch.empty(rows, device="cuda"), torch.empty_like(z)
    later, stats = torch.empty_like(z), torch.empty((rows, 4), device="cuda")
    torch.cuda.synchronize()
    more = {"temperature": temp, "t_lse": lse, "row_weight": w}
    gpu_ctx.distill_topk(z, idx, t, loss, dz=dz, **more)
    gpu_ctx.distill_topk(z, idx, t, loss, stats=stats, **more)
    gpu_ctx.distill_topk_grad(z, idx, t, stats, later, **more)
    gpu_ctx.synchronize()
    for grad in (dz, later):
        assert_matches(loss[:5], grad[:5], z[:5], idx[:5], t[:5], temp, lse[:5], w[:5])
        assert torch.equal(grad.view(n, 5, cols)[0], grad.view(n, 5, cols)[(n - 1) // 4 * 4])     # (rows that lie alike)


@gpu
@pytest.mark.parametrize("cols", [40, 2000, 9000, 70000])
@pytest.mark.parametrize("tail", [False, True])
def test_lists_of_one_class_over_and_over(gpu_ctx, cols, tail):
    """Every place of a full list names one of three classes, many rows at once: each class is counted once, with all its entries' p."""
    rows, top = 300, 256
    z, idx, t, lse, w = inputs(rows, cols, top, "f32", cols, tail, 1.0, ragged=False)
    t.copy_(torch.randn(t.shape, device="cuda"))
    idx.copy_((torch.arange(top, device="cuda")[None, :] * 7 + torch.arange(rows, device="cuda")[:, None]) % 3 * (cols // 3 - 1))
    if tail:
        lse.copy_(torch.logsumexp(t, 1) + 0.7)
    loss, dz = both_ways(gpu_ctx, z, idx, t, 1.0, lse, w)
    some = torch.arange(0, rows, 23)
    at = some.cuda()
    assert_matches(loss[at], dz[at], z[at], idx[at], t[at], 1.0, None if lse is None else lse[at], w[at])


@gpu
@pytest.mark.parametrize("cols", [10, 900, 30000])
def test_a_class_outside_the_row_is_reported_and_left_out(gpu_ctx, cols):
    z, idx, t, lse, w = inputs(6, cols, 5, "f32", cols, True, 1.0, ragged=False)
    idx[3, 2], idx[4, 0] = cols, 2 ** 31 - 1
    loss, dz = torch.empty(6, device="cuda"), torch.empty_like(z)
    torch.cuda.synchronize()
    gpu_ctx.distill_topk(z, idx, t, loss, t_lse=lse, row_weight=w, dz=dz)
    with pytest.raises(capi.S2VError) as e:
        gpu_ctx.synchronize()
    assert e.value.status == -1
    gpu_ctx.synchronize()
    assert_matches(loss, dz, z, idx, t, 1.0, lse, w)


@gpu
@pytest.mark.parametrize("rows,cols", [(70000, 3), (3000, 130), (600, 1024), (600, 1500), (400, 9000)])
def test_many_rows(gpu_ctx, rows, cols):
    """More rows than CTAs: rows of one block after another.  Rows repeat after 50, and so do the results: bit by bit where the rows lie alike
    (which columns a thread adds up goes by where the row's first 16-byte boundary is), and from one call to the next."""
    z, idx, t, lse, w = inputs(50, cols, 4, "bf16", rows, True, 1.0)
    loss50, dz50 = both_ways(gpu_ctx, z, idx, t, 1.0, lse, w)
    assert_matches(loss50, dz50, z, idx, t, 1.0, lse, w)
    n = rows // 50
    loss, dz = torch.empty(n * 50, device="cuda"), torch.empty((n * 50, cols), dtype=z.dtype, device="cuda")
    args = [v.repeat(n, *([1] * (v.dim() - 1))) for v in (z, idx, t)]
    lse_n, w_n = lse.repeat(n), w.repeat(n)
    torch.cuda.synchronize()
    gpu_ctx.distill_topk(*args, loss, t_lse=lse_n, row_weight=w_n, dz=dz)
    gpu_ctx.synchronize()
    want = dz50.repeat(n, 1)
    # (few and many rows may be shared among different numbers of threads: sums in another order)
    rel = 2 * relative(cols, 1.0, z)
    assert torch.allclose(loss, loss50.repeat(n), rtol=2.0 ** -22, atol=2 * rel)
    assert bool(((dz.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 4 * rel).all())
    alike = (n - 1) // 8 * 8     # 8 times 50 rows of 16-bit values are a multiple of 16 bytes
    assert torch.equal(dz.view(n, 50, cols)[0], dz.view(n, 50, cols)[alike]) and torch.equal(loss.view(n, 50)[0], loss.view(n, 50)[alike])
    again, dz_again = torch.empty_like(loss), torch.empty_like(dz)
    torch.cuda.synchronize()
    gpu_ctx.distill_topk(*args, again, t_lse=lse_n, row_weight=w_n, dz=dz_again)
    gpu_ctx.synchronize()
    assert torch.equal(loss, again) and torch.equal(dz, dz_again)


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,cols,top", [("f32", 8203, 9), ("f16", 17001, 128), ("bf16", 17001, 200), ("f32", 33001, 64), ("bf16", 131077, 30)])
def test_losses_of_many_long_rows(gpu_ctx, dtype, cols, top, tail):
    """The loss alone, of more long rows than run at a time: the same to the last bit as with a gradient, with columns listed twice, masked and NaN."""
    z, idx, t, lse, w = inputs(50, cols, top, dtype, cols + top, tail, 1.0)
    idx[3, 1] = idx[3, 0]
    z[4, : cols // 2] = -math.inf
    z[5, idx[5].clamp(min=0).long()] = torch.finfo(z.dtype).min
    torch.cuda.synchronize()
    loss50, dz50 = both_ways(gpu_ctx, z, idx, t, 1.0, lse, w)
    assert_matches(loss50, dz50, z, idx, t, 1.0, lse, w)
    z[6, 77] = math.nan
    many = [None if v is None else v.repeat(9, *([1] * (v.dim() - 1))) for v in (z, idx, t, lse, w)]
    more = {"t_lse": many[3], "row_weight": many[4]}
    loss, alone, kept, dz, stats = *(torch.empty(450, device="cuda") for _ in range(3)), torch.empty_like(many[0]), torch.empty((450, 4), device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.distill_topk(*many[:3], loss, dz=dz, **more)
    gpu_ctx.distill_topk(*many[:3], alone, **more)
    gpu_ctx.distill_topk(*many[:3], kept, stats=stats, **more)
    gpu_ctx.synchronize()
    same = lambda a, b: torch.equal(a.nan_to_num(nan=12345.0), b.nan_to_num(nan=12345.0))  # noqa: E731
    assert same(loss, alone) and same(loss, kept) and bool(loss.view(9, 50)[:, 6].isnan().all())
    loss50[6] = math.nan
    rel = 2 * relative(cols, 1.0, z.nan_to_num(nan=0.0))
    assert torch.allclose(loss, loss50.repeat(9), rtol=2.0 ** -22, atol=2 * rel, equal_nan=True)


@gpu
@pytest.mark.parametrize("rows,dtype,cols,top", [(450, "f16", 17001, 128), (450, "bf16", 17001, 200), (460, "f32", 24001, 64), (310, "bf16", 70001, 30), (310, "f32", 140001, 150)])
def test_gradients_of_many_long_rows_in_place(gpu_ctx, rows, dtype, cols, top):
    """dz in the place of z gives what dz beside it gives, with rows wider than their columns and columns listed twice."""
    some, idx, t, lse, w = inputs(31, cols, top, dtype, cols, True, 1.0)
    idx[3, 1] = idx[3, 0]
    n = -(-rows // 31)
    idx, t, lse, w = (v.repeat(n, *([1] * (v.dim() - 1)))[:rows].contiguous() for v in (idx, t, lse, w))
    wide = torch.full((rows, cols + 3), 9.0, dtype=some.dtype, device="cuda")
    z = wide[:, :cols]
    z.copy_(some.repeat(n, 1)[:rows])
    loss, loss2, dz, stats = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(wide)[:, :cols], torch.empty((rows, 4), device="cuda")
    more = {"t_lse": lse, "row_weight": w}
    torch.cuda.synchronize()
    gpu_ctx.distill_topk(z, idx, t, loss, dz=dz, **more)
    gpu_ctx.distill_topk(z, idx, t, loss2, stats=stats, **more)
    gpu_ctx.synchronize()
    assert torch.equal(loss, loss2)
    assert_matches(loss[:31], dz[:31], z[:31], idx[:31], t[:31], 1.0, lse[:31], w[:31])
    kept = wide.clone()
    later = torch.empty_like(wide)[:, :cols]
    torch.cuda.synchronize()
    gpu_ctx.distill_topk_grad(z, idx, t, stats, later, **more)
    gpu_ctx.distill_topk(z, idx, t, loss2, dz=z, **more)
    gpu_ctx.distill_topk_grad(kept[:, :cols], idx, t, stats, kept[:, :cols], **more)
    gpu_ctx.synchronize()
    assert torch.equal(loss, loss2) and torch.equal(z, dz) and torch.equal(kept[:, :cols], later)
    assert bool((wide[:, cols:] == 9).all() and (kept[:, cols:] == 9).all())


@gpu
def test_captured_replayed_and_on_another_stream(gpu_ctx):
    for rows, cols in ((64, 6), (40, 3000), (12, 60000)):
        z, idx, t, lse, w = inputs(rows, cols, 5, "f16", rows, True, 1.0)
        loss, dz, stats = torch.empty(rows, device="cuda"), torch.empty_like(z), torch.empty((rows, 4), device="cuda")
        loss2, dz2 = torch.empty_like(loss), torch.empty_like(dz)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        gpu_ctx.distill_topk(z, idx, t, loss, t_lse=lse, row_weight=w, dz=dz, stream=side.cuda_stream)
        gpu_ctx.stream_status(side.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            gpu_ctx.distill_topk(z, idx, t, loss, t_lse=lse, row_weight=w, dz=dz, stream=side.cuda_stream)
            gpu_ctx.distill_topk(z, idx, t, loss2, t_lse=lse, row_weight=w, stats=stats, stream=side.cuda_stream)
            gpu_ctx.distill_topk_grad(z, idx, t, stats, dz2, t_lse=lse, row_weight=w, stream=side.cuda_stream)
        for _ in range(2):
            z.copy_(z.flip(0) * 0.5)
            loss.fill_(1), loss2.fill_(1), dz.fill_(1), dz2.fill_(1)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert_matches(loss, dz, z, idx, t, 1.0, lse, w)
            assert_matches(loss2, dz2, z, idx, t, 1.0, lse, w)
    gpu_ctx.synchronize()


@gpu
def test_refusals(gpu_ctx):
    lib, h = gpu_ctx.lib, gpu_ctx.h
    f, i = torch.zeros(4096, device="cuda"), torch.zeros(64, dtype=torch.int32, device="cuda")
    p, ip = f.data_ptr(), i.data_ptr()

    def call(rows=4, cols=10, zt=0, z=p, ldz=10, top=3, idx=ip, tt=0, t=p, ldt=3, temp=1.0, loss=p, dz=p + 4096, lddz=10):
        return lib.s2v_distill_topk(h, None, rows, cols, zt, z, ldz, top, idx, tt, t, ldt, None, temp, None, loss, None, dz, lddz)

    def grad(stats=p, dz=p + 4096, **kw):
        a = {"rows": 4, "cols": 10, "ldz": 10, "top": 3, "temp": 1.0} | kw
        return lib.s2v_distill_topk_grad(h, None, a["rows"], a["cols"], 0, p, a["ldz"], a["top"], ip, 0, p, 3, None, a["temp"], None, stats, dz, 10)

    for got, want in [(call(rows=-1), -1), (call(cols=0), -1), (call(top=0), -1), (call(zt=3), -1), (call(tt=-1), -1), (call(z=None), -1), (call(idx=None), -1), (call(t=None), -1),
                      (call(loss=None), -1), (call(ldz=9), -1), (call(lddz=9), -1), (call(ldt=2), -1), (call(temp=0.0), -1), (call(temp=-1.0), -1), (call(temp=INF), -1),
                      (call(temp=float("nan")), -1), (call(temp=1e-35), -1), (call(z=p + 2), -1), (call(dz=p + 2), -1), (call(t=p + 1, tt=1), -1), (call(dz=p, lddz=11), -1),
                      (call(top=257, ldt=257), -2), (call(cols=262145, ldz=1 << 20, lddz=1 << 20), -2), (call(cols=524289, zt=1, ldz=1 << 20, lddz=1 << 20), -2),
                      (grad(stats=None), -1), (grad(dz=None), -1), (grad(temp=0.0), -1), (grad(ldz=9), -1), (grad(rows=-1), -1), (grad(cols=0), -1)]:
        assert got == want, lib.s2v_last_error(h)
    assert call(rows=0, z=None) == 0 and grad(rows=0) == 0
    gpu_ctx.synchronize()
    assert not f.any()


@gpu
@pytest.mark.parametrize("cols", [1 << 61, 1 << 62, (1 << 63) - 1, (1 << 62) + 8, (1 << 32) + 5])
def test_refusal_of_rows_whose_bytes_pass_64_bits(gpu_ctx, cols):
    f, i = torch.zeros(64, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    p, ip = f.data_ptr(), i.data_ptr()
    for zt in (0, 1, 2):
        assert gpu_ctx.lib.s2v_distill_topk(gpu_ctx.h, None, 1, cols, zt, p, cols, 1, ip, 0, p, 1, None, 1.0, None, p, None, None, 0) == -2
        assert gpu_ctx.lib.s2v_distill_topk_grad(gpu_ctx.h, None, 1, cols, zt, p, cols, 1, ip, 0, p, 1, None, 1.0, None, p, p, cols) == -2
    gpu_ctx.synchronize()
    assert not f.any()


@gpu
def test_refusals_of_misaligned_lists_and_rows(gpu_ctx):
    lib, h = gpu_ctx.lib, gpu_ctx.h
    f, i = torch.zeros(4096, device="cuda"), torch.zeros(64, dtype=torch.int32, device="cuda")
    p = f.data_ptr()
    good = {"idx": i.data_ptr(), "lse": p, "weight": p, "loss": p, "stats": p}
    for name in ("idx", "lse", "weight", "loss"):
        for off in (1, 2, 3):
            a = dict(good, **{name: good[name] + off})
            assert lib.s2v_distill_topk(h, None, 4, 10, 0, p, 10, 3, a["idx"], 0, p, 3, a["lse"], 1.0, a["weight"], a["loss"], None, p + 4096, 10) == -1, name
            if name != "loss":
                assert lib.s2v_distill_topk_grad(h, None, 4, 10, 0, p, 10, 3, a["idx"], 0, p, 3, a["lse"], 1.0, a["weight"], a["stats"], p + 4096, 10) == -1, name
    gpu_ctx.synchronize()
    assert not f.any()


# ---------------------------------------------------------------- together, as they are used
@gpu
def test_an_8_bit_student_of_the_readout(gpu_ctx):
    """The fp32 readout of a batch of pooled embeddings as the teacher, its two layers in 8 bits as the student: the student's logits, the loss against
    the teacher's top classes and the gradient that a training step of the student starts with."""
    G, d, hidden, classes, top = 513, 128, 256, 37, 8
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    Y = torch.randn((G, d), generator=gen, device="cuda")
    W1, W2 = torch.randn((d, hidden), generator=gen, device="cuda") * 0.1, torch.randn((hidden, classes), generator=gen, device="cuda") * 0.1
    teacher = torch.empty((G, classes), device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.readout(Y, W1, W2, teacher)
    gpu_ctx.synchronize()
    t, idx = teacher.topk(top, dim=1)
    idx, lse = idx.to(torch.int32), torch.logsumexp(teacher, 1)
    layers = []
    for W in (W1, W2):     # a channel a row
        wt = W.t().contiguous()
        q, s = torch.empty(wt.shape, dtype=torch.int8, device="cuda"), torch.empty(wt.shape[0], device="cuda")
        torch.cuda.synchronize()
        gpu_ctx.quantize_rows_i8(wt, q, s)
        layers.append((q, s))
    h, z = torch.empty((G, hidden), dtype=torch.bfloat16, device="cuda"), torch.empty((G, classes), device="cuda")
    ws = torch.empty(gpu_ctx.linear_i8_workspace_bytes(G, hidden), dtype=torch.uint8, device="cuda")
    loss, dz, mean = torch.empty(G, device="cuda"), torch.empty_like(z), torch.empty(1, device="cuda")
    weight = torch.full((G,), 1.0, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.linear_i8(Y, *layers[0], h, ws, relu=True)
    gpu_ctx.linear_i8(h, *layers[1], z, ws)
    gpu_ctx.distill_topk(z, idx, t, loss, t_lse=lse, row_weight=weight, dz=dz)
    gpu_ctx.call("s2v_mean_f32", None, G, loss.data_ptr(), mean.data_ptr())
    gpu_ctx.synchronize()
    # 8-bit operands are off by half a step of 1/127 of a row's largest value (below 5 deviations), d or hidden independent terms a sum:
    # 2 * sqrt(k) * (5 / 127 / sqrt(12)) * 0.1 of the values' deviation a layer -- a few hundredths of logits whose deviation is above one
    assert float((z - teacher).abs().max()) < 0.35 * float(teacher.std())
    assert_matches(loss, dz, z, idx, t, 1.0, lse, weight)
    assert math.isclose(float(mean), float(loss.double().mean()), rel_tol=1e-5) and 0 < float(mean) < 0.05
