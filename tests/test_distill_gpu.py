"""Distillation loss and its logit gradient on the GPU, against the definition in 64 bits.

Tolerances, before any run. A log-sum-exp comes from fp32 sums (chains of about 50 additions of 2^-24 each, and
exponentials good to a few 2^-24): 5e-6 of it in absolute terms, which enters a row's loss once for the student
and once for the teacher at weight alpha tau^2, once at weight 1 - alpha; the loss is rounded to fp32. A gradient
element is a sum of terms good to 1e-5 (the stored log-sum-exp in fp32 and an exponent of up to 40), rounded to
fp16 once: 2^-11 of it, or half the finest step, 2^-25."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
IGNORE = -100


@pytest.fixture(scope="module")
def ops():
    from midstream_llm_b200 import ops as _ops
    return _ops


def _inputs(R, V, K, seed=0, t_dtype=torch.float16, distinct=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = (V + 7) // 8 * 8
    x = (torch.randn(R, ld, device="cuda", generator=g) * 3).half()[:, :V]
    if distinct:
        ids = torch.rand(R, V, device="cuda", generator=g).argsort(1)[:, :K].contiguous()
        if K > V:
            ids = torch.nn.functional.pad(ids, (0, K - V), value=-1)
    else:
        ids = torch.randint(0, V, (R, K), device="cuda", generator=g)
    t = (torch.randn(R, K, device="cuda", generator=g) * 3).to(t_dtype)
    y = torch.randint(0, V, (R,), device="cuda", generator=g)
    return x, ids, t, y


def _define(x, ids, t, y, tau, alpha, gscale, count):
    """(row losses, gradient, magnitudes of its terms), by rows, in 64 bits."""
    R, V = x.shape
    x, t = x.double(), t.double()
    loss, grad, mag = (torch.zeros(*s, device="cuda", dtype=torch.float64) for s in ((R,), (R, V), (R, V)))
    for r in range(R):
        if int(y[r]) == IGNORE:
            continue
        q, q1 = torch.softmax(x[r] / tau, 0), torch.softmax(x[r], 0)
        used = (ids[r] >= 0) & (t[r] != -INF)
        if bool(used.any()):
            p = torch.softmax(t[r][used] / tau, 0)
            at = ids[r][used]
            loss[r] += alpha * tau ** 2 * (p * (p.log() - q[at].log())).sum()
            grad[r] += alpha * tau * q
            grad[r].scatter_add_(0, at, -alpha * tau * p)
            mag[r] += alpha * tau * q
            mag[r].scatter_add_(0, at, alpha * tau * p)
        if alpha < 1:
            loss[r] -= (1 - alpha) * q1[y[r]].log()
            grad[r] += (1 - alpha) * q1
            grad[r, y[r]] -= 1 - alpha
            mag[r] += (1 - alpha) * q1
            mag[r, y[r]] += 1 - alpha
    return loss, grad * (gscale / count), mag * (gscale / count)


def _check(ops, x, ids, t, y, tau, alpha, parts=None, gscale=512.0, in_place=False):
    R = x.shape[0]
    count = max(int((y != IGNORE).sum()), 1)
    want, gwant, mag = _define(x, ids, t, y, tau, alpha, gscale, count)
    stats, rows = ops.distill_fwd(x, ids, t, y, temperature=tau, alpha=alpha, ignore_index=IGNORE, parts=parts)
    tol = (2 * alpha * tau ** 2 + (1 - alpha)) * 5e-6 + 2 ** -24 * want.abs()
    err = (rows.double() - want).abs()
    assert bool((err <= tol).all()), (tau, alpha, float((err / tol).max()))
    out3 = ops.ce_loss(rows, y, IGNORE)
    if bool((y != IGNORE).any()):
        assert abs(float(out3[2]) - float(want.sum()) / count) <= float(tol.max()) + 2 ** -20 * abs(float(want.sum()) / count)
    out = None if in_place else torch.full((R, x.stride(0) + 8), 3.0, device="cuda", dtype=torch.float16)[:, :x.shape[1]]
    gs = torch.tensor([gscale], device="cuda")
    got = ops.distill_bwd(x, ids, t, y, stats, gs, torch.tensor([float(count)], device="cuda"), temperature=tau, alpha=alpha,
                          ignore_index=IGNORE, out=out)
    assert got.data_ptr() == (x if in_place else out).data_ptr()
    gtol = 2 ** -11 * gwant.abs() + 2 ** -25 + 1e-5 * mag
    gerr = (got.double() - gwant).abs()
    assert bool((gerr <= gtol).all()), (tau, alpha, float((gerr / gtol).max()))
    return got


@pytest.mark.parametrize("R,V,K", [(1, 1, 1), (3, 7, 3), (5, 8, 1), (4, 300, 300), (6, 1000, 64), (3, 8192, 33), (3, 8193, 5),
                                   (7, 24000, 16), (4, 32000, 64), (2, 32769, 200), (2, 50257, 1024)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (1.0, 0.5), (2.0, 1.0), (2.0, 0.7), (4.0, 0.3), (0.5, 0.9), (1.7, 0.0)])
def test_loss_and_gradient(ops, R, V, K, tau, alpha):
    x, ids, t, y = _inputs(R, V, K, seed=V + K, t_dtype=torch.float16 if K % 2 else torch.float32)
    _check(ops, x, ids, t, y, tau, alpha)


@pytest.mark.parametrize("R,V,K", [(3, 7, 3), (6, 1000, 64), (3, 8193, 5), (400, 9000, 16), (2, 50257, 1024)])
@pytest.mark.parametrize("alpha", [1.0, 0.7, 0.0])
def test_loss_and_gradient_at_one_and_a_half(ops, R, V, K, alpha):
    """Where both softmaxes are powers of one exponential."""
    x, ids, t, y = _inputs(R, V, K, seed=V + 2 * K, t_dtype=torch.float32)
    x[0] = (x[0].float() * 40).half()  # logits far apart, whose powers underflow
    _check(ops, x, ids, t, y, 1.5, alpha)


@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (3.0, 0.6)])
def test_unused_slots_repeated_ids_and_ignored_rows(ops, tau, alpha):
    x, ids, t, y = _inputs(12, 500, 40, seed=1, distinct=False)  # ids drawn with repeats
    ids[:, 7] = ids[:, 3]
    ids[1, 5:] = -1
    ids[2] = -1                # no teacher at all
    t[3, 4:] = -INF            # slots without weight
    t[4] = -INF
    ids[5, ::2] = -7
    y[6] = IGNORE
    ids[7, 0] = y[7]           # the target among the slots
    ids[8, :] = y[8]           # in every slot
    t[9, 1] = -INF
    ids[9, 1] = ids[9, 2]      # the same id with and without weight
    y[10], ids[10] = IGNORE, -1
    _check(ops, x, ids, t, y, tau, alpha)
    _check(ops, torch.nn.functional.pad(x, (0, 4))[:, :500], ids, t, y, tau, alpha, in_place=True)


@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (1.0, 0.5), (2.0, 0.7)])
def test_what_ignored_rows_hold_does_not_matter(ops, tau, alpha):
    """Ids past the vocabulary, NaN logits on either side: no loss, no gradient, no status; the other rows as without them."""
    from midstream_llm_b200 import _lib
    x, ids, t, y = _inputs(9, 704, 12, seed=4)
    keep = torch.tensor([0, 2, 3, 5, 8], device="cuda")
    skip = torch.tensor([1, 4, 6, 7], device="cuda")
    stats0, rows0 = ops.distill_fwd(x[keep], ids[keep], t[keep], y[keep], temperature=tau, alpha=alpha, ignore_index=IGNORE)
    y[skip], ids[skip], t[skip] = IGNORE, 10 ** 12, NAN
    x[skip] = NAN
    _lib.device_status()
    stats, rows = ops.distill_fwd(x, ids, t, y, temperature=tau, alpha=alpha, ignore_index=IGNORE)
    one = torch.ones(1, device="cuda")
    dx = ops.distill_bwd(x, ids, t, y, stats, one, one, temperature=tau, alpha=alpha, ignore_index=IGNORE,
                         out=torch.full_like(x, 2.0))
    assert _lib.device_status() == 0
    assert bool((rows[skip] == 0).all()) and bool((dx[skip] == 0).all()) and bool((stats[:, skip] == 0).all())
    assert torch.equal(rows[keep], rows0) and torch.equal(stats[:, keep], stats0) and bool(dx[keep].isfinite().all())


def test_a_batch_of_ignored_rows_and_a_repeat(ops):
    x, ids, t, y = _inputs(4, 256, 8, seed=2)
    y[:] = IGNORE
    got = _check(ops, x, ids, t, y, 2.0, 0.5)
    assert bool((got == 0).all())
    x, ids, t, y = _inputs(64, 32000, 64, seed=3)
    first = None
    for _ in range(3):
        stats, rows = ops.distill_fwd(x, ids, t, y, temperature=2.0, alpha=0.5)
        g = ops.distill_bwd(x, ids, t, y, stats, torch.ones(1, device="cuda"), torch.full((1,), 64.0, device="cuda"),
                            temperature=2.0, alpha=0.5, out=torch.empty_like(x))
        if first is None:
            first = (rows.clone(), g)
        assert torch.equal(rows, first[0]) and torch.equal(g, first[1])


def test_masked_student_logits(ops):
    """-inf logits (a masked vocabulary) carry no probability; where the teacher wants one the loss is infinite."""
    x, ids, t, y = _inputs(3, 640, 10, seed=4)
    x[:, 600:] = -INF
    ids.clamp_(max=599)
    y.clamp_(max=599)
    ids[1, 3] = 620
    stats, rows = ops.distill_fwd(x, ids, t, y, temperature=2.0, alpha=0.5)
    assert math.isinf(float(rows[1])) and bool(rows[[0, 2]].isfinite().all())
    keep = torch.tensor([0, 2], device="cuda")
    got = _check(ops, x[keep], ids[keep], t[keep], y[keep], 2.0, 0.5)
    assert bool((got[:, 600:] == 0).all())


def test_bad_targets_and_ids_are_reported(ops):
    from midstream_llm_b200 import _lib
    x, ids, t, y = _inputs(4, 256, 8, seed=5)
    _lib.device_status()
    y[1] = 256
    stats, rows = ops.distill_fwd(x, ids, t, y, alpha=0.5)
    assert math.isnan(float(rows[1])) and bool(rows[[0, 2, 3]].isfinite().all()) and _lib.device_status() == 202
    got = ops.distill_bwd(x, ids, t, y, stats, torch.ones(1, device="cuda"), torch.full((1,), 4.0, device="cuda"), alpha=0.5,
                          out=torch.full_like(x, 5.0))
    assert bool((got[1] == 0).all()) and bool(got.isfinite().all())
    y[1] = 3
    ids[2, 4] = 256
    stats, rows = ops.distill_fwd(x, ids, t, y, alpha=0.5)
    assert math.isnan(float(rows[2])) and _lib.device_status() == 203


@pytest.mark.parametrize("M,V,K", [(300, 1000, 20), (256, 24000, 64)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (1.0, 0.4), (2.0, 0.4), (2.0, 1.0)])
def test_statistics_from_the_head(ops, M, V, K, tau, alpha):
    """With the head's block statistics the loss is the same, whether or not the logits are read."""
    g = torch.Generator(device="cuda").manual_seed(6)
    h = torch.randn(M, 128, device="cuda", generator=g).half()
    e = (torch.randn(V, 128, device="cuda", generator=g) * 0.3).half()
    x, parts = ops.gemm_f16_ce_parts(h, e)
    _, ids, t, y = _inputs(M, V, K, seed=7)
    y[::9] = IGNORE
    _check(ops, x, ids, t, y, tau, alpha, parts=parts)


def test_gradient_against_differences(ops):
    """The loss's own differences along random directions d of -1, 0 and 1, at points that fp16 holds exactly. With
    h = 1/8 a central difference is off by h^2 / 6 times the third derivative, which for a log-sum-exp is a third
    central moment of d, at most 0.77 (and 1 / tau times that at temperature tau >= 1): below 0.0027 a row; and
    by the losses' error over 2 h, twice."""
    tau, alpha, V = 2.0, 0.5, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    x = (torch.randint(-16, 17, (5, V), device="cuda", generator=g) / 8.0).half()
    _, ids, t, y = _inputs(5, V, 12, seed=9)
    one, n = torch.ones(1, device="cuda"), torch.ones(1, device="cuda")
    stats, _ = ops.distill_fwd(x, ids, t, y, temperature=tau, alpha=alpha)
    grad = ops.distill_bwd(x, ids, t, y, stats, one, n, temperature=tau, alpha=alpha, out=torch.empty_like(x)).double()
    for _ in range(8):
        d = torch.randint(-1, 2, (5, V), device="cuda", generator=g).half()
        up = ops.distill_fwd(x + d / 8, ids, t, y, temperature=tau, alpha=alpha)[1].double()
        down = ops.distill_fwd(x - d / 8, ids, t, y, temperature=tau, alpha=alpha)[1].double()
        slope = (up - down) * 4
        want = (grad * d.double()).sum(1)
        bound = 0.0027 + 8 * (2 * alpha * tau ** 2 + 1) * 5e-6 + 2 ** -11 * grad.abs().sum(1) + V * 2 ** -25
        assert bool(((slope - want).abs() <= bound).all())


def test_refusals(ops):
    x, ids, t, y = _inputs(4, 256, 8)
    with pytest.raises(RuntimeError, match="temperature"):
        ops.distill_fwd(x, ids, t, y, temperature=0.0)
    with pytest.raises(RuntimeError, match="alpha"):
        ops.distill_fwd(x, ids, t, y, alpha=1.5)
    with pytest.raises(RuntimeError, match="teacher slots"):
        ops.distill_fwd(x, ids[:, :0].contiguous(), t[:, :0].contiguous(), y)
    with pytest.raises(TypeError, match="teacher_ids"):
        ops.distill_fwd(x, ids.int(), t, y)
    with pytest.raises(TypeError, match="teacher_logits"):
        ops.distill_fwd(x, ids, t.double(), y)
    with pytest.raises(ValueError, match="targets"):
        ops.distill_fwd(x, ids, t, y[:3])
    stats, rows = ops.distill_fwd(x, ids, t, y)
    one = torch.ones(1, device="cuda")
    with pytest.raises(ValueError, match="out must have shape"):
        ops.distill_bwd(x, ids, t, y, stats, one, one, out=torch.empty(4, 264, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="one value"):
        ops.distill_bwd(x, ids, t, y, stats, rows, one)


def _cold_rows(V, K, tau, scales, shift, seed):
    """Rows whose teacher has the student's own largest logits, at several sizes of the logits, with ties at the top."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(len(scales), (V + 7) // 8 * 8, device="cuda", generator=g) * torch.tensor(scales, device="cuda")[:, None] + shift
    x = x.half()
    x = x[:, :V]
    top = x.float().argmax(1)
    rows = torch.arange(len(scales), device="cuda")
    x[rows, (top + 1) % V] = x[rows, top]  # (a tie: the two largest weigh the same at any temperature)
    t, ids = x.float().topk(K, dim=1)
    y = torch.randint(0, V, (len(scales),), device="cuda", generator=g)
    return x, ids, t, y


def _define_by_logs(x, ids, t, y, tau, alpha, scale):
    """_define for rows that use every slot and ids that differ, from log-softmaxes: no weight underflows to 0 log 0."""
    x, rows = x.double(), torch.arange(x.shape[0], device="cuda")
    lp, lq, l1 = (torch.log_softmax(v, 1) for v in (t.double() / tau, x / tau, x))
    loss = alpha * tau ** 2 * (lp.exp() * (lp - lq.gather(1, ids))).sum(1) - (1 - alpha) * l1[rows, y]
    grad = alpha * tau * lq.exp() + (1 - alpha) * l1.exp()
    mag = grad.clone().scatter_add_(1, ids, alpha * tau * lp.exp())
    grad.scatter_add_(1, ids, -alpha * tau * lp.exp())
    grad[rows, y] -= 1 - alpha
    mag[rows, y] += 1 - alpha
    return loss, grad * scale, mag * scale


@pytest.mark.parametrize("V,K,R", [(1000, 16, 8), (24000, 64, 8), (24000, 5, 320)])
@pytest.mark.parametrize("tau,alpha,shift", [(0.001, 1.0, 0.0), (0.01, 1.0, 3.0), (0.01, 0.5, 0.0), (0.1, 1.0, -9.0), (0.1, 0.7, 20.0),
                                             (1.0, 1.0, 2000.0), (1.0, 0.5, -30000.0), (1.5, 0.5, 5000.0), (2.0, 0.4, -9000.0),
                                             (3.0, 0.4, 700.0), (7.0, 0.4, 700.0)])
@pytest.mark.parametrize("other", [False, True])
def test_low_temperatures_and_large_logits(ops, V, K, R, tau, alpha, shift, other):
    """Logits that are large against the temperature: the result is as good as for small ones, also where the teacher is
    the student and every term cancels. A loss may be off by what the sums of both softmaxes may (5e-6 each in the
    logarithm), and by what fp32 weights leave of the slots' differences (2^-17 of them: an exponential's argument up to
    40 rounded to fp32, and sums); the gradient by _check's bounds."""
    scales = [(0.01, 0.1, 0.5, 1.0, 2.0, 3.0, 5.0, 7.0)[r % 8] for r in range(R)]
    x, ids, t, y = _cold_rows(V, K, tau, scales, shift, seed=V + K)
    if other:  # a teacher of its own, by a few steps of temperature
        g = torch.Generator(device="cuda").manual_seed(1)
        t = t + torch.randn(t.shape, device="cuda", generator=g) * tau
    want, gwant, mag = _define_by_logs(x, ids, t, y, tau, alpha, 512.0 / R)
    stats, rows = ops.distill_fwd(x, ids, t, y, temperature=tau, alpha=alpha)
    td, zd = t.double(), x.gather(1, ids).double()
    slots = (torch.softmax(td / tau, 1) * (td - zd).abs()).sum(1) / tau
    tol = alpha * tau ** 2 * (1e-5 + 2 ** -17 * slots) + (1 - alpha) * 5e-6 + 2 ** -24 * want.abs()
    err = (rows.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    for out in (torch.empty_like(x), None):
        got = ops.distill_bwd(x, ids, t, y, stats, torch.full((1,), 512.0, device="cuda"), torch.full((1,), float(R), device="cuda"),
                              temperature=tau, alpha=alpha, out=out)
        gtol = 2 ** -11 * gwant.abs() + 2 ** -25 + 1e-5 * mag
        gerr = (got.double() - gwant).abs()
        assert bool((gerr <= gtol).all()), float((gerr / gtol).max())
