"""Corners of the operators over rows of vocabulary logits that documented arguments reach.  Bounds as in test_gpu_logits."""
import numpy as np
import pytest
import torch

from tests import logits_specs as spec
from tests.test_gpu_logits import DEV, TYPES, check_distill, check_sample, check_top, record, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pg():
    import pgload
    return pgload.load()


def flat(T, V, dtype, seed):
    """Rows without a peak: their nucleus is most of the vocabulary."""
    return (0.1 * torch.randn(T, V, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(5, 30), (5, 64), (4, 700), (4, 5000), (300, 5000), (4, 40000)])
def test_a_negative_top_k_of_a_row_is_off(pg, dtype, T, V):
    x = flat(T, V, dtype, V)
    k = torch.tensor([-1, 0, -(2 ** 31), -7, 3], dtype=torch.int32).repeat(T)[:T].to(DEV)
    check_sample(pg, x, top_k=k, top_p=0.9)
    check_sample(pg, x, top_k=k, top_p=0.5, min_p=0.7, temperature=0.8)
    check_sample(pg, x, top_k=k)
    # (every combination of two filters of a row, within and beyond what the segments' lists hold)
    k = torch.tensor([-1, 600, 2, V + 9, 0, V // 2 + 1], dtype=torch.int32).repeat(T)[:T].to(DEV)
    p = torch.tensor([0.9, 0.4, float("nan"), -1.0, 1.0, 0.97, 0.05], device=DEV).repeat(T)[:T]
    least = torch.tensor([0.0, float("nan"), 0.8, -3.0, 5.0], device=DEV).repeat(T)[:T]
    check_sample(pg, x, top_k=k, top_p=p)
    check_sample(pg, x, top_k=k, top_p=p, min_p=least)
    check_sample(pg, rows(T, V, dtype, V + 1), top_k=k, top_p=p, min_p=least)


def signalling(x):
    """x with signalling NaN (quiet bit clear) in every third place and on both sides of each row's largest entries."""
    bits = x.view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32)
    bad = 0x7f81 if x.dtype == torch.bfloat16 else 0x7f810000
    V = x.shape[1]
    at = torch.arange(V, device=x.device)
    top = x.float().topk(min(V, 9), dim=1).indices
    near = torch.zeros_like(bits, dtype=torch.bool)
    for o in (-1, 1):
        near.scatter_(1, (top + o).clamp(0, V - 1), True)
    near |= at % 3 == 0
    near.scatter_(1, top, False)
    bits[near] = bad
    assert not torch.isnan(x.gather(1, top).float()).any() and torch.isnan(x.float()).any()
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(30, 4), (64, 9), (700, 33), (1003, 100), (5001, 64), (40000, 200), (131072, 64)])
def test_signalling_nan_counts_as_any_other(pg, dtype, V, k):
    x = signalling(rows(12, V, dtype, V))
    check_top(pg, x, k)
    for n, f in enumerate([{}, {"top_k": 5}, {"top_p": 0.8}, {"min_p": 0.05}, {"temperature": 0.0}, {"top_k": min(V, 600), "top_p": 0.9}]):
        check_sample(pg, x, seed=n, **f)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [9000, 40003])
def test_signalling_nan_in_many_rows(pg, dtype, V):
    """The cuts of calls with rows enough to fill the chip."""
    T = 1030
    x = torch.zeros(T, V, dtype=dtype, device=DEV)
    few = signalling(rows(4, V, dtype, V))
    at = torch.tensor([0, 1, T // 2, T - 1], device=DEV)
    bits = torch.int16 if dtype == torch.bfloat16 else torch.int32
    x.view(bits)[at] = few.view(bits)
    v, i, r = pg.ops.top_logits(x, 33, temperature=2.0)
    wv, wi, wr = spec.top_logits(few, 33, 2.0)
    assert np.array_equal(i[at].cpu().numpy(), wi) and np.array_equal(v[at].double().cpu().numpy(), wv)
    q = torch.empty(T, V, device=DEV).exponential_(1.0, generator=torch.Generator(DEV).manual_seed(2))
    pred, _ = pg.ops.sample_filtered(x, q, top_k=40, top_p=0.9)
    assert np.array_equal(pred[at].cpu().numpy(), spec.sample(few, q[at], 1.0, 40, 0.9, 0.0)[0])


@pytest.mark.parametrize("V", [30, 700, 9001])
def test_signalling_nan_in_a_students_row(pg, V):
    x, v, i, r = record(pg, 4, V, 6, torch.bfloat16, V, 1.0, True)
    x[:2] = 0
    x = torch.cat([signalling(rows(2, V, torch.bfloat16, V)), x[2:]])
    check_distill(pg, x, v, i, r, 1.0, None)
    check_distill(pg, x, v, i, None, 1.0, torch.tensor([0.0, 1.0, 1.0, 2.0], device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T,V", [(9, 30), (9, 64), (9, 700), (9, 20011), (1100, 9001)])
def test_records_that_are_not_finite_give_nan(pg, dtype, tail, T, V):
    """+inf among a row's values, +inf or NaN as its rest: no softmax, so NaN in the row's loss and gradient, whatever the sizes; the
    other rows, rows of weight 0 among them, as ever."""
    k = 6
    x, v, i, r = record(pg, T, V, k, dtype, V, 2.0, True)
    inf, nan = float("inf"), float("nan")
    v[0, 0] = inf
    v[1, :2] = inf
    v[2, 3], i[2, 3] = inf, -1  # (an absent entry's value does not count)
    v[3, 1] = nan               # (absent)
    v[4, 0] = inf
    r[5], r[6], r[7] = inf, nan, nan
    w = torch.ones(T, device=DEV)
    w[4] = w[7] = 0.0
    bad = torch.zeros(T, dtype=torch.bool)
    bad[[0, 1] + ([5, 6] if tail else [])] = True
    rest = r if tail else None
    leaf = x.detach().requires_grad_()
    loss = pg.loss.distillation_loss(leaf, v, i, rest=rest, temperature=2.0, weights=w)
    loss.sum().backward()
    both = pg.ops.distill_loss_grad(x, v, i, rest=rest, temperature=2.0, weights=w)
    for a, g in ((loss.detach(), leaf.grad), both):
        assert torch.equal(a.isnan().cpu(), bad)
        assert torch.equal(g.isnan().all(1).cpu(), bad) and torch.equal(g.isnan().any(1).cpu(), bad)
        assert not a[4].any() and not g[4].any() and not a[7].any() and not g[7].any()
    few = torch.tensor([2, 3, 4, 7, 8] + ([] if tail else [5, 6]), device=DEV)
    check_distill(pg, x[few], v[few], i[few], None if rest is None else rest[few], 2.0, w[few])


@pytest.mark.parametrize("V", [30, 700])
def test_the_record_of_a_row_with_an_infinite_logit(pg, V):
    """top_logits' own record of an overflowing teacher, inside the list and in the rest."""
    x, t = rows(2, V, torch.float32, V), rows(2, V, torch.float32, V + 1)
    t[0, 3] = t[1, 2] = t[1, 5] = float("inf")
    v, i, r = pg.ops.top_logits(t, 1)
    assert torch.isinf(v).all() and r[1] == float("inf") and torch.isfinite(r[0])
    loss, grad = pg.ops.distill_loss_grad(x, v, i, rest=r)
    assert loss.isnan().all() and grad.isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [5, 30, 32, 33, 64, 65, 700, 20000, 100003])
def test_the_resolution_of_top_p_is_one_for_all_vocabularies(pg, dtype, V):
    """Each entry's mass counts in multiples of 2^-40 of the largest's.  Two equal largest entries, top_p exactly 0.5: one stays where
    every other mass rounds to 0, however many they are, both where one other weighs a multiple.  The second entry's draw wins
    where it stays."""
    ln2 = float(np.log(2.0))
    x = torch.full((4, V), -60.0)
    x[3] = -45 * ln2       # 1/32 multiples each: none
    x[:, 1] = x[:, 3] = 0.0
    x[1, 0] = -41.5 * ln2  # 0.35 multiples: none
    x[2, 0] = -38.5 * ln2  # 2.8 multiples: three
    x = x.to(dtype).to(DEV)
    assert float(x[1, 0]) < -41.2 * ln2 and -38.7 * ln2 < float(x[2, 0]) < -38.2 * ln2 and float(x[3, 0]) < -44 * ln2
    q = torch.ones(4, V, device=DEV)
    q[:, 3] = 0.125
    for T in (4, 300):
        pred, conf = pg.ops.sample_filtered(x.repeat(T // 4, 1), q.repeat(T // 4, 1), top_p=0.5)
        assert pred.tolist() == [1, 1, 3, 1] * (T // 4) and conf.tolist() == [1.0, 1.0, 0.5, 1.0] * (T // 4)
    pred, conf = pg.ops.sample_filtered(x, q, top_p=0.5, top_k=min(V, 100))
    assert pred.tolist() == [1, 1, 3, 1] and conf.tolist() == [1.0, 1.0, 0.5, 1.0]


def test_the_largest_sampled_vocabulary(pg):
    """2^24 - 1 equal entries: 2^23 of them hold half the mass, in the order of their index."""
    V = 2 ** 24 - 1
    x = torch.full((1, V), 3.0, dtype=torch.bfloat16, device=DEV)
    q = torch.empty(1, V, device=DEV).exponential_(1.0, generator=torch.Generator(DEV).manual_seed(1))
    q[0, 2 ** 23:] *= 1e-6
    pred, conf = pg.ops.sample_filtered(x, q, top_p=0.5)
    assert int(pred) == int(q[0, :2 ** 23].argmin()) and float(conf) == 2.0 ** -23
    pred, conf = pg.ops.sample_filtered(x, q)
    assert int(pred) == int(q[0].argmin())


@pytest.mark.parametrize("V", [30, 700, 20000])
def test_settings_that_fp32_does_not_hold(pg, V):
    """Numbers within the documented ranges that fp32 rounds to 0 or infinity mean the nearest that it holds."""
    x = rows(4, V, torch.float32, V)
    for p in (1e-38, 1e-45, 1e-50, 1e-300):
        check_sample(pg, x, top_p=p)
    for least in (1e-45, 1e-50, 1e-300):
        check_sample(pg, x, min_p=least)
    x[:, V // 3] = x[:, V // 2] = 50.0
    q = torch.ones(4, V, device=DEV)
    q[:, V // 2] = 0.5
    for temp in (1e-45, 1e-50, 1e-300):  # (above 0: the largest entries race)
        pred, conf = pg.ops.sample_filtered(x, q, temperature=temp)
        assert (pred == V // 2).all() and (conf == 0.5).all()
    q[:, 1] = 0.25
    for temp in (1e31, 1e39, 1e300):
        pred, conf = pg.ops.sample_filtered(x, q, temperature=temp)
        assert (pred == 1).all() and ((conf * V - 1).abs() < 1e-6).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(12, 30), (12, 64), (12, 700), (300, 5001), (4, 40000)])
def test_rows_with_many_infinite_logits(pg, dtype, T, V):
    """Half of the entries, one in forty or all are +inf: they share the row."""
    x = rows(T, V, dtype, V)
    g = torch.Generator().manual_seed(V)
    u = torch.rand(T, V, generator=g).to(DEV)
    share = torch.tensor([0.5, 0.025, 2.0, 0.0], device=DEV).repeat(T)[:T].view(T, 1)
    x[u < share] = float("inf")
    check_top(pg, x, min(V, 50))
    for n, f in enumerate([{}, {"top_k": 3}, {"top_p": 0.6}, {"min_p": 0.3}, {"temperature": 0.0}, {"top_k": V // 2, "top_p": 0.9},
                           {"top_p": 0.3, "min_p": 1.0}]):
        check_sample(pg, x, seed=n, **f)


def test_the_largest_vocabulary_of_records_and_distillation(pg):
    V, k, tau = 2 ** 24, 5, 2.0
    x = torch.randn(2, V, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    v, i, r = pg.ops.top_logits(x, k, temperature=tau)
    wv, wi = x.topk(k, dim=1)
    assert torch.equal(v, wv) and torch.equal(i.long(), wi)
    z = (x.double() / tau).scatter(1, wi, float("-inf"))
    U = 2.0 ** -24
    # (a thread adds V / 256 entries in a row, the workgroup joins 256 sums)
    assert ((r.double() - torch.logsumexp(z, 1)).abs() <= (V // 256 + 48) * U).all()
    student = (0.5 * x + torch.randn(2, V, device=DEV, generator=torch.Generator(DEV).manual_seed(2)))
    loss, grad = pg.ops.distill_loss_grad(student, v, i, rest=r, temperature=tau)
    wl, wg, ls, gs = spec.distill(student, v, i, r, tau, None)
    a = (V // 256 + 48 + 64) * U
    assert (np.abs(loss.double().cpu().numpy() - wl) <= a * ls).all()
    assert (np.abs(grad.double().cpu().numpy() - wg) <= a * gs + U * np.abs(wg) * 1.01 + 1e-38).all()


def test_captured_distillation_loss(pg):
    """Forward and backward by autograd captured once and replayed on new inputs, with eager calls of the same between."""
    cases = []
    for T, V, dtype in ((64, 30, torch.float32), (4, 70001, torch.bfloat16), (3, 900, torch.float32)):
        x, v, i, r = record(pg, T, V, 7, dtype, V, 2.0, True)
        cases.append((x, v, i, r, torch.rand(T, device=DEV), torch.randn(T, device=DEV)))

    def work():
        out = []
        for x, v, i, r, w, up in cases:
            leaf = x.detach().requires_grad_()
            loss = pg.loss.distillation_loss(leaf, v, i, rest=r, temperature=2.0, weights=w)
            out += [loss.detach(), torch.autograd.grad(loss, leaf, up)[0]]
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
        for x, v, i, r, w, up in cases:
            x.add_((0.37 * torch.randn(x.shape, generator=torch.Generator().manual_seed(n))).to(x.dtype).to(DEV))
        graph.replay()
        eager = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(5, 30), (5, 64), (5, 700), (5, 5001), (5, 40000), (1030, 9001)])
def test_rows_of_subnormal_logits(pg, dtype, T, V):
    """Values below the least normal number are ordered as any others."""
    x = (3e-39 * torch.randn(T, V, generator=torch.Generator().manual_seed(V))).to(dtype).to(DEV)
    assert 0 < float(x.abs().float().median()) < 2.0 ** -126
    few = torch.tensor([0, 1, T // 2, T - 1], device=DEV)
    k = min(V, 20)
    v, i, _ = pg.ops.top_logits(x, k)
    wv, wi, _ = spec.top_logits(x[few], k, 1.0)
    assert np.array_equal(i[few].cpu().numpy(), wi) and np.array_equal(v[few].double().cpu().numpy(), wv)
    q = torch.empty(T, V, device=DEV).exponential_(1.0, generator=torch.Generator(DEV).manual_seed(V))
    for f in ({"temperature": 0.0}, {"top_k": 3}, {"top_k": k, "top_p": 0.5}, {"min_p": 1.0}):
        full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
        full.update(f)
        pred, _ = pg.ops.sample_filtered(x, q, **full)
        want, _ = spec.sample(x[few], q[few], full["temperature"], full["top_k"], full["top_p"], full["min_p"])
        assert np.array_equal(pred[few].cpu().numpy(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 3])
def test_signalling_nan_in_whole_row_passes(pg, dtype, shift):
    """Records of more than 512 entries, and rows that no list settles, read in passes over the row."""
    x = signalling(rows(300, 5003, dtype, 7, pad=2, shift=shift))[:6]
    check_top(pg, x, 700)
    check_top(pg, x, 1024, tau=2.0)
    for n, f in enumerate([{}, {"top_k": 900}, {"top_p": 0.99, "temperature": 8.0}, {"top_k": 2000, "top_p": 0.9, "temperature": 8.0}]):
        check_sample(pg, x, seed=n, **f)
