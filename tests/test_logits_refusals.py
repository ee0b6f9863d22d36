"""What the operators over vocabulary logits refuse, before anything reaches a device: through the Python layer (CPU tensors
that pass every check end at the "no CPU path" error) and through the C ABI."""
import pytest
import torch


@pytest.fixture(scope="module")
def pg():
    import pgload
    return pgload.load()


X = torch.zeros(4, 10)


@pytest.mark.parametrize("call,error", [
    (lambda o: o.top_logits(X, 0), ValueError),
    (lambda o: o.top_logits(X, 11), ValueError),
    (lambda o: o.top_logits(torch.zeros(2, 3000), 1025), ValueError),
    (lambda o: o.top_logits(X, 3, temperature=0.0), ValueError),
    (lambda o: o.top_logits(X, 3, temperature=float("nan")), ValueError),
    (lambda o: o.top_logits(X, 3, temperature=float("inf")), ValueError),
    (lambda o: o.top_logits(X, 3, temperature=1e-31), ValueError),
    (lambda o: o.top_logits(X, 3, temperature=1e31), ValueError),
    (lambda o: o.top_logits(X.half(), 3), TypeError),
    (lambda o: o.top_logits(X.double(), 3), TypeError),
    (lambda o: o.top_logits(torch.zeros(()), 1), ValueError),
    (lambda o: o.top_logits(torch.zeros(3, 0), 1), ValueError),
    (lambda o: o.top_logits(torch.zeros(10, 4).t(), 1), ValueError),
    (lambda o: o.top_logits(torch.zeros(4, 3, 10).transpose(0, 1), 1), ValueError),
    (lambda o: o.top_logits(X, 3), ValueError),  # no CPU path
])
def test_top_logits_refusals(pg, call, error):
    with pytest.raises(error):
        call(pg.ops)


@pytest.mark.parametrize("kw,error", [
    ({"temperature": -0.1}, ValueError), ({"temperature": float("inf")}, ValueError), ({"temperature": float("nan")}, ValueError),
    ({"top_k": -1}, ValueError), ({"top_p": 0.0}, ValueError), ({"top_p": 1.5}, ValueError), ({"top_p": float("nan")}, ValueError),
    ({"empty": -2}, ValueError), ({"min_p": -0.1}, ValueError), ({"min_p": 1.1}, ValueError),
    ({"temperature": torch.ones(3)}, ValueError), ({"temperature": torch.ones(4, dtype=torch.float64)}, TypeError),
    ({"top_k": torch.ones(4, dtype=torch.int64)}, TypeError), ({"noise": torch.ones(4, 9)}, ValueError),
    ({"noise": torch.ones(4, 10, dtype=torch.float64)}, TypeError), ({"logits": torch.zeros(2, 2, 10)}, ValueError),
    ({"logits": X.half()}, TypeError), ({}, ValueError),  # no CPU path
])
def test_sample_filtered_refusals(pg, kw, error):
    args = {"logits": X, "noise": torch.ones(4, 10)}
    args.update(kw)
    with pytest.raises(error):
        pg.ops.sample_filtered(**args)


@pytest.mark.parametrize("kw,error", [
    ({"values": torch.zeros(4, 0), "ids": torch.zeros(4, 0, dtype=torch.int32)}, ValueError),
    ({"values": torch.zeros(4, 1025), "ids": torch.zeros(4, 1025, dtype=torch.int32)}, ValueError),
    ({"values": torch.zeros(4, 3, dtype=torch.bfloat16)}, TypeError), ({"values": torch.zeros(3, 3)}, ValueError),
    ({"ids": torch.zeros(4, 3, dtype=torch.int64)}, TypeError), ({"ids": torch.zeros(4, 2, dtype=torch.int32)}, ValueError),
    ({"rest": torch.zeros(3)}, ValueError), ({"rest": torch.zeros(4, dtype=torch.float64)}, TypeError),
    ({"weights": torch.zeros(4, 1)}, ValueError), ({"weights": torch.zeros(4, dtype=torch.int64)}, TypeError),
    ({"temperature": 0.0}, ValueError), ({"temperature": -1.0}, ValueError), ({"logits": X.half()}, TypeError), ({}, ValueError),
    ({"temperature": 1e-31}, ValueError), ({"temperature": 1e31}, ValueError),
])
def test_distill_refusals(pg, kw, error):
    args = {"logits": X, "values": torch.zeros(4, 3), "ids": torch.zeros(4, 3, dtype=torch.int32), "rest": None, "weights": None}
    args.update(kw)
    with pytest.raises(error):
        pg.ops.distill_loss_grad(**args)
    args["student_logits"], args["top_values"], args["top_ids"] = args.pop("logits"), args.pop("values"), args.pop("ids")
    with pytest.raises(error):
        pg.loss.distillation_loss(**args)


@pytest.mark.parametrize("name", ["top_values", "rest", "weights"])
def test_distillation_loss_has_no_gradient_for_the_teacher(pg, name):
    args = {"student_logits": X, "top_values": torch.zeros(4, 3), "top_ids": torch.zeros(4, 3, dtype=torch.int32),
            "rest": torch.zeros(4), "weights": torch.ones(4)}
    args[name] = args[name].clone().requires_grad_()
    with pytest.raises(ValueError, match=name):
        pg.loss.distillation_loss(**args)


def test_c_abi_refusals(pg):
    """Status codes for arguments that must not reach a launch (the pointers are host memory: nothing may be launched)."""
    lib = pg._lib.lib
    b = torch.zeros(64)
    p = b.data_ptr()
    ARG, UNSUPPORTED, WORKSPACE = -1, -4, -5
    top = lambda dt=0, x=p, ld=8, T=2, V=8, k=3, tau=1.0, o=p: lib.pg_top_logits(dt, x, ld, T, V, k, tau, o, p, p, None, 0, None)  # noqa: E731
    assert top(dt=2) == ARG and top(x=None) == ARG and top(ld=-1) == ARG and top(T=0) == ARG and top(V=0) == ARG
    assert top(k=0) == ARG and top(k=9) == ARG and top(tau=0.0) == ARG and top(tau=float("nan")) == ARG and top(o=None) == ARG
    assert top(V=(1 << 24) + 1) == UNSUPPORTED and top(V=5000, k=1025) == UNSUPPORTED

    def smp(q=p, ldq=8, T=2, V=8, temp=1.0, k=0, tp=1.0, mp=0.0, out=p, empty=-1):
        return lib.pg_sample_filtered(0, p, 8, q, ldq, T, V, temp, k, tp, mp, None, None, None, None, empty, out, p, None, 0, None)
    assert smp(q=None) == ARG and smp(ldq=-1) == ARG and smp(temp=-1.0) == ARG and smp(temp=float("nan")) == ARG and smp(k=-1) == ARG
    assert smp(tp=0.0) == ARG and smp(tp=1.01) == ARG and smp(mp=-0.1) == ARG and smp(mp=2.0) == ARG and smp(out=None) == ARG and smp(empty=-2) == ARG
    assert smp(V=(1 << 24) + 1) == UNSUPPORTED

    def fwd(x=p, v=p, k=3, tau=1.0, V=8, loss=p, stash=p):
        return lib.pg_distill_fwd(0, x, 8, 2, V, v, p, k, None, None, tau, loss, stash, None, 0, None)
    assert fwd(x=None) == ARG and fwd(v=None) == ARG and fwd(k=0) == ARG and fwd(tau=-1.0) == ARG and fwd(loss=None) == ARG
    assert fwd(stash=None) == ARG and fwd(k=1025) == UNSUPPORTED and fwd(V=(1 << 24) + 1) == UNSUPPORTED

    def bwd(stash=p, out=p, ldo=8):
        return lib.pg_distill_bwd(0, p, 8, 2, 8, p, p, 3, None, 1.0, None, stash, out, ldo, None)
    assert fwd(stash=p + 4) == -2 and bwd(stash=p + 4) == -2
    assert bwd(stash=None) == ARG and bwd(out=None) == ARG and bwd(ldo=7) == ARG

    # two rows of 100000: cut into segments, which need a workspace
    def both(ws=p, n=0, ldo=100000, T=2, V=100000):
        return lib.pg_distill_loss_grad(0, p, V, T, V, p, p, 3, None, None, 1.0, p, p, ldo, ws, n, None)
    need = lib.pg_distill_workspace_bytes(0, 2, 100000, 3, 1)
    assert need > 0 and both(n=need - 1) == WORKSPACE and both(ws=None, n=need) == WORKSPACE and both(n=need, ldo=7) == ARG
    assert both(ws=p + 4, n=need) == -2
    fneed = lib.pg_distill_workspace_bytes(0, 2, 100000, 3, 0)
    assert 0 < fneed < need
    assert lib.pg_distill_fwd(0, p, 100000, 2, 100000, p, p, 3, None, None, 1.0, p, p, p, fneed - 1, None) == WORKSPACE
    tneed = lib.pg_top_logits_workspace_bytes(0, 2, 100000, 3)
    assert tneed > 0 and lib.pg_top_logits(0, p, 100000, 2, 100000, 3, 1.0, p, p, p, p, tneed - 1, None) == WORKSPACE
    sneed = lib.pg_sample_filtered_workspace_bytes(0, 2, 100000, 5)
    assert sneed > 0 and lib.pg_sample_filtered(0, p, 100000, p, 100000, 2, 100000, 1.0, 5, 1.0, 0.0, None, None, None, None, -1, p, p,
                                                None, 0, None) == WORKSPACE


@pytest.mark.parametrize("kw", [{"top_k": -1}, {"top_p": 0.0}, {"top_p": 1.1}, {"min_p": -0.1}, {"min_p": 1.5}])
def test_generation_refuses_bad_filters_before_the_first_pass(pg, kw):
    from protgen_gan_amd import generate as G
    gen = torch.nn.Identity()  # (never called)
    with pytest.raises(ValueError):
        G.generate_full_mode_sequences(gen, pg.ProtTokenizer(), 2, [20], device="cpu", **kw)
    with pytest.raises(ValueError):
        G.generate_seeded_mode_sequences(gen, pg.ProtTokenizer(), 2, ["ACDE"], device="cpu", **kw)


def test_generation_flags(pg):
    from protgen_gan_amd import generate as G
    a = G._parser().parse_args(["--ckpt_id", "x"])
    assert (a.top_k, a.top_p, a.min_p) == (0, 1.0, 0.0) and G._filters(a.top_k, a.top_p, a.min_p) == {}
    a = G._parser().parse_args(["--ckpt_id", "x", "--top_k", "5", "--top_p", "0.9", "--min_p", "0.1"])
    assert G._filters(a.top_k, a.top_p, a.min_p) == {"top_k": 5, "top_p": 0.9, "min_p": 0.1}
