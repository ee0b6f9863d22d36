"""The operators over rows of vocabulary logits against their definitions in 64 bits (tests/logits_specs.py).

Bounds.  u = 2^-24 is half a step of fp32.  A weight 2^((x - m) c) carries at most 3 roundings of its exponent a, |a| <= 2^7 where
the weight is not negligible (a 2^-a < 0.54: together below 4 u) and one of the exponential (2 u); a sum of n such weights adds at
most one rounding per addition a thread makes in a row and one per step of the tree.  ADDS(V) counts those: all a thread's
elements, 16 joins.  Token indices, values and ids have to be equal."""
import numpy as np
import pytest
import torch

from tests import logits_specs as spec

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def ADDS(V):
    return V // 64 + 16 + 32


@pytest.fixture(scope="module")
def pg():
    import pgload
    return pgload.load()


def rows(T, V, dtype, seed, spread=3.0, pad=0, shift=0):
    """T rows at a distance of V + pad elements, the first `shift` elements into the buffer."""
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(T, V, generator=g)).to(dtype)
    if V > 64:  # some entries far above the rest
        at = torch.randint(0, V, (T, 12), generator=g)
        x.scatter_(1, at, (8 + 2 * torch.rand(T, 12, generator=g)).to(dtype))
    buf = torch.zeros(shift + T * (V + pad), dtype=dtype, device=DEV)
    out = buf[shift:].view(T, V + pad)[:, :V]
    out.copy_(x)
    return out


def check_top(pg, x, k, tau=1.0):
    vals, ids, rest = pg.ops.top_logits(x, k, temperature=tau)
    v, i, r = spec.top_logits(x, k, tau)
    assert np.array_equal(ids.cpu().numpy(), i)
    assert np.array_equal(vals.double().cpu().numpy(), v)
    got, r = rest.double().cpu().numpy(), r.astype(np.float32).astype(np.float64)
    fin = np.isfinite(r)
    assert np.array_equal(got[~fin], r[~fin])
    assert (np.abs(got[fin] - r[fin]) <= ADDS(x.shape[1]) * U + 2 * U * np.abs(r[fin])).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (3, 2, 1), (5, 7, 7), (70, 30, 8), (33, 30, 30), (9, 64, 20), (9, 65, 64), (4, 257, 256),
                                   (6, 1000, 17), (3, 4099, 1024), (2, 50021, 100), (2, 131072, 64), (1, 300007, 513)])
def test_top_logits(pg, dtype, T, V, k):
    check_top(pg, rows(T, V, dtype, seed=V + k), k, tau=2.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift,pad", [(1, 0), (3, 5), (7, 1), (0, 8)])
@pytest.mark.parametrize("V", [5, 30, 1001, 9000])
def test_top_logits_strides(pg, dtype, shift, pad, V):
    check_top(pg, rows(5, V, dtype, seed=V, pad=pad, shift=shift), 4)


def odd_values(V, dtype):
    """Rows that are constant, mostly masked (-inf and the type's lowest), empty, hold NaN and infinities, or sorted either way."""
    x = torch.zeros(12, V)
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(5)
    x[1] = torch.randn(V, generator=g)
    x[1, 1:] = float("-inf")
    x[2] = float("-inf")
    x[3] = low
    x[4] = torch.where(torch.rand(V, generator=g) < 0.7, torch.tensor(low), torch.randn(V, generator=g))
    x[5] = torch.randn(V, generator=g)
    x[5, ::3] = float("nan")
    x[6] = float("nan")
    x[7] = torch.randn(V, generator=g)
    x[7, V // 2] = float("inf")
    x[8] = torch.linspace(-20, 20, V)
    x[9] = torch.linspace(20, -20, V)
    x[10] = torch.where(torch.arange(V) % 2 == 0, torch.tensor(-0.0), torch.tensor(0.0))
    x[11] = torch.where(torch.rand(V, generator=g) < 0.7, torch.tensor(float("-inf")), torch.randn(V, generator=g))
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(30, 4), (30, 30), (64, 9), (700, 33), (5001, 64), (40000, 200)])
def test_top_logits_odd_rows(pg, dtype, V, k):
    check_top(pg, odd_values(V, dtype), k, tau=0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(900, 100), (8192, 512), (8192, 300), (40000, 64), (131072, 128), (131072, 512)])
def test_top_logits_few_values(pg, dtype, V, k):
    """Rows of a few distinct values, masks of the type's lowest and of -inf among them: the border lies inside long ties."""
    g = torch.Generator().manual_seed(V + k)
    x = torch.stack([torch.randint(0, n, (V,), generator=g).float() for n in (1, 2, 40, 300, 2, 2)])
    x[4] = torch.where(x[4] > 0, torch.finfo(dtype).min, float("-inf"))
    x[5] = float("-inf")
    x[4, V // 2: V // 2 + 20] = 3.0
    x[5, 7:7 + k // 2] = 1.0
    x = x.to(dtype).to(DEV)
    check_top(pg, x, k)
    check_sample(pg, x, top_k=k)
    check_sample(pg, x, top_p=0.4)


def test_top_logits_leading_dims_and_empty(pg):
    x = rows(6, 40, torch.float32, 1).contiguous().view(2, 3, 40)
    v, i, r = pg.ops.top_logits(x, 5)
    v2, i2, r2 = pg.ops.top_logits(x.view(6, 40), 5)
    assert v.shape == (2, 3, 5) and r.shape == (2, 3) and torch.equal(v.view(6, 5), v2) and torch.equal(i.view(6, 5), i2)
    assert torch.equal(r.view(6), r2)
    v, i, r = pg.ops.top_logits(x[:0], 5)
    assert v.shape == (0, 3, 5) and r.shape == (0, 3)
    v1, i1, r1 = pg.ops.top_logits(x[0, 0], 5)
    assert v1.shape == (5,) and r1.shape == () and torch.equal(v1, v2[0])


# ------------------------------------------------------------------------------------------------ sampling
def check_sample(pg, x, seed=0, q=None, **kw):
    T, V = x.shape
    if q is None:
        q = torch.empty(T, V, device=DEV).exponential_(1.0, generator=torch.Generator(DEV).manual_seed(seed))
    full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    full.update(kw)
    pred, conf = pg.ops.sample_filtered(x, q, **full)
    p, c = spec.sample(x, q, full["temperature"], full["top_k"], full["top_p"], full["min_p"])
    assert np.array_equal(pred.cpu().numpy(), p)
    # weights in 64 bits (exact to 1e-11): one rounding to fp32
    assert (np.abs(conf.double().cpu().numpy() - c) <= 2 * U * c).all()


FILTERS = [{}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 5}, {"top_p": 0.5}, {"top_p": 0.93, "temperature": 1.3}, {"min_p": 0.1},
           {"top_k": 9, "top_p": 0.8}, {"top_k": 20, "top_p": 0.99, "min_p": 0.01, "temperature": 0.9}, {"temperature": 0.0},
           {"top_p": 1e-6}, {"min_p": 1.0}, {"temperature": 3.0, "top_p": 0.999}]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(300, 30), (7, 1), (50, 64), (41, 65), (20, 1000), (12, 5003), (3, 40001)])
def test_sample_filtered(pg, dtype, T, V):
    x = rows(T, V, dtype, seed=T + V)
    for n, f in enumerate(FILTERS):
        check_sample(pg, x, seed=n, **f)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("f", [{"top_k": 50, "top_p": 0.95}, {"top_p": 0.9}, {"top_p": 0.995, "temperature": 2.0}, {"top_k": 7000},
                               {"top_k": 60000, "top_p": 0.7, "temperature": 4.0}, {"min_p": 0.001}, {}])
def test_sample_filtered_wide(pg, dtype, f):
    check_sample(pg, rows(3, 131072, dtype, seed=3), **f)
    check_sample(pg, rows(2, 262147, dtype, seed=4, spread=1.0, shift=3, pad=2), **f)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [30, 64, 700, 5001, 40000])
def test_sample_filtered_odd_rows(pg, dtype, V):
    x = odd_values(V, dtype)
    for n, f in enumerate([{}, {"top_k": 3}, {"top_p": 0.6}, {"min_p": 0.3}, {"temperature": 0.0}, {"top_k": V // 2, "top_p": 0.9}]):
        check_sample(pg, x, seed=n, **f)


@pytest.mark.parametrize("V", [30, 2000, 40000])
def test_sample_filtered_noise_zero_and_ties(pg, V):
    """Equal keys go to the lowest index; a zero draw wins outright, of several the lowest index."""
    x = rows(4, V, torch.bfloat16, 9)
    x[0] = 1.0
    q = torch.ones(4, V, device=DEV)
    q[1, V // 2:] = 0.0
    q[2] = 0.0
    for f in ({}, {"top_k": V - 3}, {"top_p": 0.9}):
        check_sample(pg, x, q=q, **f)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [30, 900, 33000])
def test_sample_filtered_per_row_settings(pg, dtype, V):
    T = 40
    g = torch.Generator().manual_seed(V)
    x = rows(T, V, dtype, 11)
    u = torch.rand(4, T, generator=g)
    temp, k = (0.3 + u[0]).to(DEV), (u[1] * 60).to(torch.int32).to(DEV)
    p, least = (0.2 + u[2]).to(DEV), (u[3] - 0.5).to(DEV)  # above 1: off; below 0: off
    temp[::7] = 0.0
    temp[3] = -1.0
    temp[4] = float("nan")
    k[5] = -3
    check_sample(pg, x, temperature=temp, top_k=k, top_p=p, min_p=least)
    check_sample(pg, x, temperature=temp, top_k=4)
    check_sample(pg, x, top_p=p)


@pytest.mark.parametrize("V", [30, 900, 33000])
def test_extreme_temperatures(pg, V):
    """Near 0 only the ties of the largest entry race; far up, and infinite in a row's own setting, all entries weigh the same."""
    temp = torch.tensor([1e-45, 1e-40, 1e-30, 1e-20, 1e20, 1e30, 3e38, float("inf")], device=DEV)
    x = rows(8, V, torch.bfloat16, 12)
    x[:, V // 3] = x[:, V // 2] = 50.0
    x[:, V // 4] = float("-inf")
    for f in ({}, {"top_p": 0.6}, {"top_k": 7}, {"min_p": 0.3}, {"top_k": 600, "top_p": 0.9}):
        check_sample(pg, x, temperature=temp, **f)
        for t in (1e-40, 3e38):
            check_sample(pg, x, temperature=t, **f)
    for tau in (2.0 ** -99, 2.0 ** 99):  # (numbers of fp32)
        check_top(pg, x, 1, tau)
        check_top(pg, x, 20, tau)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_sample_filtered_ties_in_unaligned_rows(pg, dtype, shift):
    """Of equal largest entries the first index, wherever the row's 16-byte vectors begin."""
    for V, k in ((133842, 512), (5003, 0), (40001, 700)):
        x = torch.zeros(4 * (V + 1) + shift, dtype=dtype, device=DEV)[shift:].view(4, V + 1)[:, :V]
        x[1, 0], x[2, :2], x[3, -1] = 1.0, -1.0, 1.0
        check_sample(pg, x, temperature=0.0, top_k=k)
        check_sample(pg, x, top_k=k, q=torch.full((4, V), float("inf"), device=DEV))


def test_sample_filtered_strided_inputs_and_outputs(pg):
    x = rows(8, 333, torch.bfloat16, 2, pad=7, shift=5)
    q = torch.empty(8, 400, device=DEV).exponential_(1.0)[:, 3:336]
    check_sample(pg, x, q=q, top_k=9)
    wide = x[:1].expand(6, 333)  # one row of logits, six draws
    check_sample(pg, wide, top_p=0.9)
    pred = torch.full((8,), 77, dtype=torch.int64, device=DEV)
    conf = torch.full((8,), 7.0, device=DEV)
    pg.ops.sample_filtered(x[:5], q[:5], top_k=9, pred=pred[:5], conf=conf[:5])
    assert (pred[5:] == 77).all() and (conf[5:] == 7.0).all()


def test_sample_filtered_agrees_with_sample_tokens(pg):
    """Without a filter the tokens are sample_tokens' for the same draw."""
    x, q = rows(500, 30, torch.float32, 4), torch.empty(500, 30, device=DEV).exponential_(1.0)
    a, ca = pg.ops.sample_tokens(x.contiguous(), q, 0.8)
    b, cb = pg.ops.sample_filtered(x, q, temperature=0.8)
    assert torch.equal(a, b)
    # sample_tokens: quotient, difference, exponential (|exponent| < 32: 64 u), sum of 30 and division in fp32
    assert ((ca - cb).abs() <= 128 * U * cb).all()


# ------------------------------------------------------------------------------------------------ distillation
def record(pg, T, V, k, dtype, seed, tau, tail):
    teacher = rows(T, V, dtype, seed)
    v, i, r = pg.ops.top_logits(teacher, k, temperature=tau)
    g = torch.Generator().manual_seed(seed + 1)
    x = (0.7 * teacher.float().cpu() + torch.randn(T, V, generator=g)).to(dtype).to(DEV)
    return x, v, i, (r if tail else None)


def check_distill(pg, x, v, i, r, tau, w):
    V = x.shape[1]
    up = torch.randn(x.shape[0], generator=torch.Generator().manual_seed(1)).to(DEV)
    want, grad, ls, gs = spec.distill(x, v, i, r, tau, w)
    with np.errstate(over="ignore"):
        want = want.astype(np.float32).astype(np.float64)  # (masks of the type's lowest value: beyond fp32 is infinite)
    a = ADDS(V) + 64
    leaf = x.detach().requires_grad_()
    loss = pg.loss.distillation_loss(leaf, v, i, rest=r, temperature=tau, weights=w)
    loss.backward(up)
    both = pg.ops.distill_loss_grad(x, v, i, rest=r, temperature=tau, weights=w)
    half = torch.finfo(x.dtype).eps / 2
    for got, g, f in ((loss, leaf.grad, up.double().cpu().numpy()[:, None]), (both[0], both[1], 1.0)):
        got, g = got.detach().double().cpu().numpy(), g.double().cpu().numpy()
        fin = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got == np.inf, want == np.inf)
        assert (np.abs(got[fin] - want[fin]) <= a * U * ls[fin]).all(), np.abs(got[fin] - want[fin]).max()
        ok = np.isfinite(grad)
        assert np.array_equal(np.isfinite(g), ok)
        err = np.abs(g - f * grad)
        tol = np.abs(f) * (a * U * gs) + half * np.abs(f * grad) * 1.01 + 1e-38
        assert (err[ok] <= tol[ok]).all(), (err[ok] - tol[ok]).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (6, 2, 1), (9, 7, 7), (200, 30, 8), (33, 30, 29), (21, 64, 33), (21, 65, 5), (8, 1000, 40),
                                   (5, 4099, 300), (3, 32003, 20), (2, 131072, 64), (2, 300007, 1024)])
def test_distill(pg, dtype, tail, T, V, k):
    tau = 2.0
    x, v, i, r = record(pg, T, V, k, dtype, V + k, tau, tail)
    g = torch.Generator().manual_seed(k)
    w = (torch.rand(T, generator=g) + 0.5).to(DEV)
    w[::4] = 0.0 if T > 1 else 1.5
    check_distill(pg, x, v, i, r, tau, w)
    check_distill(pg, x, v, i, r, 1.0, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [30, 64, 700, 5001, 20011])
def test_distill_odd_rows(pg, dtype, tail, V):
    """Masked and odd student rows, absent and repeated entries, rows of weight 0 that hold NaN, negative weights."""
    x = odd_values(V, dtype)
    x = torch.cat([x, x])
    T, k = x.shape[0], 6
    g = torch.Generator().manual_seed(V)
    i = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    v = torch.randn(T, k, generator=g).to(dtype)
    r = torch.randn(T, generator=g)
    i[0, 1], i[1, 0], i[2, 3] = -1, V, 2 ** 31 - 1  # absent
    v[3, 2], v[4, 0], v[5, 1] = float("-inf"), float("-inf"), float("nan")
    i[8] = -1  # no entry at all
    v[9] = float("-inf")
    i[10, 3], i[10, 5], i[13, 1] = i[10, 0], i[10, 0], i[13, 0]  # the same id twice, three times
    r[12], r[15] = float("-inf"), 30.0
    w = (torch.rand(T, generator=g) + 0.5)
    w[5] = w[6] = w[7] = 0.0
    w[10] = -0.5
    check_distill(pg, x, v.to(DEV), i.to(DEV), r.to(DEV) if tail else None, 1.5, w.to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [30, 700, 20011])
def test_distill_of_masked_teacher_rows(pg, dtype, V):
    """Teachers' rows at the type's lowest value, wholly or but for fewer entries than the record holds; rows far from 0: the
    rest's fp32 steps are as large as whole probabilities there, but it is one number."""
    k, tau = 4, 8.0
    low = torch.finfo(dtype).min
    x = rows(6, V, dtype, V)
    x[0] = low
    x[1, 3:] = low
    x[2] += 10000.0
    x[3] -= 10000.0
    x[4] = float("-inf")
    x[4, 5] = low
    v, i, r = pg.ops.top_logits(x, k, temperature=tau)
    check_distill(pg, rows(6, V, dtype, V + 1), v, i, r, tau, None)
    check_distill(pg, x, v, i, r, tau, None)
    check_distill(pg, x[:4], v[:4], i[:4], None, tau, None)


@pytest.mark.parametrize("V,k", [(5, 20), (30, 33), (30, 64), (30, 200), (64, 65), (70, 1024)])
def test_distill_more_entries_than_tokens(pg, V, k):
    """Records longer than the vocabulary: most entries absent or repeated."""
    T = 9
    g = torch.Generator().manual_seed(k)
    x, v = rows(T, V, torch.float32, k), torch.randn(T, k, generator=g)
    i = torch.randint(-2 * V, 2 * V, (T, k), generator=g).to(torch.int32)
    check_distill(pg, x, v.to(DEV), i.to(DEV), torch.randn(T, generator=g).to(DEV), 1.0, None)
    check_distill(pg, x, v.to(DEV), i.to(DEV), None, 1.0, None)


def test_distill_rest_without_a_token(pg):
    """The teacher leaves mass to tokens the student's vocabulary does not have left: infinite loss, finite gradient."""
    x, v, i, r = record(pg, 4, 9, 9, torch.float32, 3, 1.0, True)
    r = torch.tensor([0.0, float("-inf"), 1.0, float("-inf")], device=DEV)
    check_distill(pg, x, v, i, r, 1.0, None)


def test_distill_confident_student_keeps_the_tail(pg):
    """The student's mass outside the list is 2^-60 of the whole: 1 - sum would lose it, the loss and its gradient do not."""
    T, V, k = 3, 500, 4
    x = torch.randn(T, V, generator=torch.Generator().manual_seed(0)).to(DEV)
    v, i, r = pg.ops.top_logits(x, k)
    x = x.scatter(1, i.long(), 45.0)
    check_distill(pg, x, v, i, r, 1.0, None)


@pytest.mark.parametrize("V", [30, 3001])
def test_distill_gradient_against_differences(pg, V):
    """d loss along random directions against central differences of the loss itself, h = 2^-6: the third derivative along a unit
    direction is below 1 (softmax), so h^2/6 < 5e-5; two losses' rounding over 2h: 64 (ADDS + 64) u times their scale."""
    T, k, tau, h = 6, 8, 2.0, 2.0 ** -6
    x, v, i, r = record(pg, T, V, k, torch.float32, V, tau, True)
    _, _, ls, _ = spec.distill(x, v, i, r, tau, None)
    _, grad = pg.ops.distill_loss_grad(x, v, i, rest=r, temperature=tau)
    for n in range(4):
        d = torch.randn(T, V, generator=torch.Generator().manual_seed(n)).to(DEV)
        d /= d.norm(dim=1, keepdim=True)
        f = lambda s: pg.ops.distill_fwd(x + s * d, v, i, rest=r, temperature=tau)[0].double()  # noqa: E731
        diff = ((f(h) - f(-h)) / (2 * h)).cpu().numpy()
        along = (grad.double() * d.double()).sum(1).cpu().numpy()
        assert (np.abs(diff - along) <= 5e-5 * tau + (ADDS(V) + 64) * U * ls / h).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(5, 900), (5, 8192), (5, 33000), (1030, 9000), (1030, 33000), (1025, 140001)])
def test_steep_rows(pg, dtype, T, V):
    """Entries spread over hundreds of units of temperature: a thread's sum may start at the least of them."""
    x = (40 * torch.randn(T, V, device=DEV, generator=torch.Generator(DEV).manual_seed(V))).to(dtype)
    few = slice(0, T, max(1, T // 5))
    v, i, r = pg.ops.top_logits(x, 40, temperature=0.5)
    for a, b in zip((v[few], i[few], r[few]), pg.ops.top_logits(x[few].contiguous(), 40, temperature=0.5)):
        assert a.dtype == torch.float32 and torch.allclose(a, b, rtol=2 * U, atol=ADDS(V) * U) or torch.equal(a, b)
    check_top(pg, x[few], 40, 0.5)
    check_sample(pg, x[few], top_p=0.9, temperature=3.0)
    student = (x.float() * 0.9).to(dtype)
    both = pg.ops.distill_loss_grad(student, v, i, rest=r, temperature=0.5)
    loss, stash = pg.ops.distill_fwd(student, v, i, rest=r, temperature=0.5)
    for t in range(0, T, max(1, T // 5)):
        want, grad, ls, gs = spec.distill(student[t:t + 1], v[t:t + 1], i[t:t + 1], r[t:t + 1], 0.5, None)
        a = (ADDS(V) + 64) * U
        assert abs(float(both[0][t]) - want[0]) <= a * ls[0] and abs(float(loss[t]) - want[0]) <= a * ls[0]
        err = np.abs(both[1][t].double().cpu().numpy() - grad[0])
        assert (err <= a * gs[0] + torch.finfo(dtype).eps / 2 * np.abs(grad[0]) * 1.01 + 1e-38).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [30, 900, 33000])
@pytest.mark.parametrize("tau", [2.0 ** -40, 2.0 ** -10, 2.0 ** 10])
def test_distill_extreme_temperatures(pg, dtype, V, tau):
    x, v, i, r = record(pg, 5, V, 9, dtype, V, tau, True)
    check_distill(pg, x, v, i, r, tau, None)
    check_distill(pg, x, v, i, None, tau, None)


def test_distill_strides_and_leading_dims(pg):
    x, v, i, r = record(pg, 12, 77, 5, torch.bfloat16, 1, 1.0, True)
    wide = torch.zeros(12, 90, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:80] = x
    part = wide[:, 3:80]
    a, ga = pg.ops.distill_loss_grad(x, v, i, rest=r)
    b, gb = pg.ops.distill_loss_grad(part, v, i, rest=r)
    # (which thread adds which elements follows the row's alignment: two sums of one set in fp32)
    _, _, ls, gs = spec.distill(x, v, i, r, 1.0, None)
    e = 2 * (ADDS(77) + 64) * U
    assert ((a - b).abs().cpu().numpy() <= e * ls).all()
    assert ((ga.float() - gb.float()).abs().cpu().numpy() <= e * gs + 2.0 ** -7 * ga.float().abs().cpu().numpy()).all()
    c, gc = pg.ops.distill_loss_grad(x.view(3, 4, 77), v.view(3, 4, 5), i.view(3, 4, 5), rest=r.view(3, 4))
    assert c.shape == (3, 4) and torch.equal(gc.view(12, 77), ga)
    leaf = x.clone().requires_grad_()
    pg.loss.distillation_loss(leaf, v, i, rest=r).sum().backward()  # an expanded upstream gradient
    assert torch.equal(leaf.grad, ga)
    e = pg.ops.distill_loss_grad(x[:0], v[:0], i[:0])
    assert e[0].shape == (0,) and e[1].shape == (0, 77)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,pad", [(1100, 300, 3), (1030, 9001, 0), (1030, 40003, 5), (1030, 90000, 0), (1030, 131072, 0), (1025, 140001, 7)])
def test_many_rows(pg, dtype, T, V, pad):
    """The cuts of calls with more rows than the chip takes at once (the other tests' calls are small): rows whole or in large
    segments, gradients from registers.  All rows run, a few are compared."""
    at = torch.tensor([0, 1, T // 2, T - 1])
    g = torch.Generator().manual_seed(V)
    few = rows(4, V, dtype, V)
    x = torch.empty(T, V + pad, dtype=dtype, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(1))[:, :V]
    x[at] = few
    k = 33
    v, i, r = pg.ops.top_logits(x, k, temperature=2.0)
    wv, wi, wr = spec.top_logits(few, k, 2.0)
    assert np.array_equal(i[at].cpu().numpy(), wi) and np.array_equal(v[at].double().cpu().numpy(), wv)
    assert (np.abs(r[at].double().cpu().numpy() - wr) <= ADDS(V) * U + 2 * U * np.abs(wr)).all()
    q = torch.empty(T, V, device=DEV).exponential_(1.0, generator=torch.Generator(DEV).manual_seed(2))
    temp = (0.7 + torch.rand(T, generator=g)).to(DEV)
    for f in ({"top_k": 40, "top_p": 0.9}, {"top_p": 0.97, "temperature": temp}, {"min_p": 0.02}, {"top_k": 700}):
        full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
        full.update(f)
        pred, conf = pg.ops.sample_filtered(x, q, **full)
        if torch.is_tensor(full["temperature"]):
            full["temperature"] = temp[at.to(DEV)]
        wp, wc = spec.sample(few, q[at], full["temperature"], full["top_k"], full["top_p"], full["min_p"])
        assert np.array_equal(pred[at].cpu().numpy(), wp) and (np.abs(conf[at].double().cpu().numpy() - wc) <= 2 * U * wc).all()
    del q
    w = torch.ones(T, device=DEV)
    w[2::3] = 0.0
    w[at] = 1.5
    a, half = (ADDS(V) + 64) * U, torch.finfo(dtype).eps / 2 * 1.01
    for rest in (r, None):
        wl, wg, ls, gs = spec.distill(few, v[at], i[at], None if rest is None else rest[at], 2.0, w[at])
        stash = pg.ops.distill_fwd(x, v, i, rest, w, 2.0)
        for loss, grad in (pg.ops.distill_loss_grad(x, v, i, rest=rest, temperature=2.0, weights=w),
                           (stash[0], pg.ops.distill_bwd(x, v, i, stash[1], torch.ones(T, device=DEV), w, 2.0))):
            assert (np.abs(loss[at].double().cpu().numpy() - wl) <= a * ls).all()
            assert (np.abs(grad[at].double().cpu().numpy() - wg) <= a * gs + half * np.abs(wg) + 1e-38).all()
            off = (w == 0).nonzero()[:, 0]
            assert not grad[off[:7]].any() and not loss[off].any() and torch.isfinite(loss).all()


def test_repeat_calls_are_bit_equal(pg):
    for V in (30, 2000, 70001):
        x, v, i, r = record(pg, 5, V, 7, torch.float32, V, 1.0, True)
        q = torch.empty(5, V, device=DEV).exponential_(1.0)
        first = None
        for _ in range(3):
            out = (*pg.ops.top_logits(x, 7), *pg.ops.sample_filtered(x, q, top_p=0.9), *pg.ops.distill_loss_grad(x, v, i, rest=r))
            first = first or out
            assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_logits_ops_replay_in_a_graph_and_on_another_stream(pg):
    """Captured once, replayed on new inputs between eager calls of the same operators on another stream."""
    cases = []
    for T, V in ((64, 30), (4, 70001)):
        x, v, i, r = record(pg, T, V, 7, torch.float32, V, 1.0, True)
        cases.append((x, v, i, r, torch.empty(T, V, device=DEV).exponential_(1.0)))

    def work():
        out = []
        for x, v, i, r, q in cases:
            out += [*pg.ops.top_logits(x, 7), *pg.ops.sample_filtered(x, q, top_p=0.97, top_k=900),
                    *pg.ops.distill_loss_grad(x, v, i, rest=r)]
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for n in range(4):
        for x, v, i, r, q in cases:
            x.add_(0.37 * torch.randn(x.shape, generator=torch.Generator().manual_seed(n)).to(DEV))
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            eager = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.get_device_properties(0).total_memory < 60 * 2 ** 30, reason="needs 60 GB")
def test_offsets_beyond_32_bits(pg):
    """Rows that start past 2^31 elements (and 2^32 bytes of noise)."""
    V, T = 131072, 16400
    x = torch.full((T, V), -3.0, dtype=torch.bfloat16, device=DEV)
    q = torch.ones(T, V, device=DEV)
    last = rows(2, V, torch.bfloat16, 8)
    x[-2:] = last
    q[-2:] = torch.empty(2, V, device=DEV).exponential_(1.0)
    tail = lambda *t: [u[-2:].clone() for u in t]  # noqa: E731
    v, i, r = pg.ops.top_logits(x, 5)
    wv, wi, wr = spec.top_logits(last, 5, 1.0)
    gv, gi, gr = tail(v, i, r)
    assert np.array_equal(gv.double().cpu().numpy(), wv) and np.array_equal(gi.cpu().numpy(), wi)
    assert (np.abs(gr.double().cpu().numpy() - wr) <= ADDS(V) * U + 2 * U * np.abs(wr)).all()
    pred, conf = pg.ops.sample_filtered(x, q, top_k=50)
    wp, wc = spec.sample(last, q[-2:], 1.0, 50, 1.0, 0.0)
    assert np.array_equal(pred[-2:].cpu().numpy(), wp) and (np.abs(conf[-2:].double().cpu().numpy() - wc) <= 2 * U * wc).all()
    assert int(pred[0]) == 0
    del q
    loss, grad = tail(*pg.ops.distill_loss_grad(x, v, i, rest=r))
    wl, wg, ls, gs = spec.distill(last, gv, gi, gr, 1.0, None)
    a = (ADDS(V) + 64) * U
    assert (np.abs(loss.double().cpu().numpy() - wl) <= a * ls).all()
    assert (np.abs(grad.double().cpu().numpy() - wg) <= a * gs + 2.0 ** -8 * 1.01 * np.abs(wg) + 1e-38).all()
