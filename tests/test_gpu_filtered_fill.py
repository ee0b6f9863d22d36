"""The logits operators inside the framework's own paths: fill steps with top-k / top-p / min-p, mass generation with them, and
generator_distill_update (teacher's record -> student's loss and gradient -> optimizer), alone and one after the other."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import protbert_cpu as O  # noqa: E402
from tests import logits_specs as spec  # noqa: E402
from tests.test_gpu_model import DEV, build, rel_l2  # noqa: E402
from tests.test_gpu_soft_generator import _template  # noqa: E402


@pytest.fixture(scope="module")
def pg():
    import pgload
    return pgload.load()


@pytest.mark.parametrize("filters", [{"top_k": 3}, {"top_p": 0.8}, {"min_p": 0.2}, {"top_k": 12, "top_p": 0.9, "min_p": 0.05}])
def test_fill_step_with_filters(pg, filters):
    """One fill iteration: tokens and commits are those of the 64-bit sampler on the engine's own logits."""
    c, P, PC, C, gen, critic = build(pg, "tiny", torch.float32)
    B, S, V = 4, 40, c.vocab_size
    ids = _template(B, S, 3)
    mask = (ids != 0).long()
    noise = torch.empty(B * S, V).exponential_(1.0, generator=torch.Generator().manual_seed(4))
    logits = gen(ids.to(DEV), mask.to(DEV)).view(B * S, V)
    kw = dict(top_k=0, top_p=1.0, min_p=0.0)
    kw.update(filters)
    pred, conf = spec.sample(logits, noise, 0.9, kw["top_k"], kw["top_p"], kw["min_p"])
    want = ids.clone().to(DEV)
    pg.ops.commit_topk(want, torch.from_numpy(pred).to(DEV), torch.from_numpy(conf).float().to(DEV), 0.3, False)
    got = gen.generate(ids.clone().to(DEV), mask.to(DEV), temperature=0.9, keep_percent=0.3, current_rate=0.8, noise=noise, **filters)
    assert torch.equal(got, want)
    # filters that keep everything are the unfiltered step
    a = gen.generate(ids.clone().to(DEV), mask.to(DEV), temperature=0.9, keep_percent=0.3, current_rate=0.8, noise=noise)
    b = gen.generate(ids.clone().to(DEV), mask.to(DEV), temperature=0.9, keep_percent=0.3, current_rate=0.8, noise=noise, top_k=V)
    assert torch.equal(a, b)


def test_stacked_and_packed_fill_with_filters(pg):
    """Groups at their own temperatures, rectangular and packed, against separate calls."""
    from protgen_gan_amd.models import RowPacking
    c, P, PC, C, gen, critic = build(pg, "mid", torch.bfloat16)
    V, widths = c.vocab_size, [33, 48, 21]
    S = max(widths)
    ids = torch.zeros(3, S, dtype=torch.long)
    for b, w in enumerate(widths):
        ids[b, :w] = 4
        ids[b, 0], ids[b, w - 1] = 2, 3
    attn = (ids != 0).long().to(DEV)
    noise = torch.empty(3 * S, V).exponential_(1.0, generator=torch.Generator().manual_seed(6))
    f = {"top_k": 6, "min_p": 0.05}
    groups = [(0, 1, 0.8), (1, 3, 1.2)]
    a = gen.generate_groups(ids.clone().to(DEV), attn, groups, keep_percent=0.4, current_rate=0.9, noise=noise, **f)
    b = gen.generate_groups(ids.clone().to(DEV), attn, groups, keep_percent=0.4, current_rate=0.9, noise=noise,
                            packing=RowPacking(widths, S, DEV), **f)
    assert torch.equal(a, b)
    for lo, hi, t in groups:
        one = gen.generate(ids[lo:hi].clone().to(DEV), attn[lo:hi], temperature=t, keep_percent=0.4, current_rate=0.9,
                           noise=noise.view(3, S, V)[lo:hi].reshape(-1, V), **f)
        assert torch.equal(a[lo:hi], one)


def test_mass_generation_with_filters(pg):
    from protgen_gan_amd import generate as G
    c, P, PC, C, gen, critic = build(pg, "tiny", torch.float32)
    tok = pg.ProtTokenizer()
    seqs = G.generate_full_mode_sequences(gen, tok, 5, [20, 31], batch_size=3, device=DEV, rng_seed=3, top_k=4, top_p=0.9, min_p=0.01)
    assert len(seqs) == 5
    # top_k 1 leaves nothing to the noise: two runs with other draws give the same sequences
    runs = []
    for seed in (1, 2):
        torch.manual_seed(seed)
        runs.append(G.generate_full_mode_sequences(gen, tok, 4, [20, 31], batch_size=4, device=DEV, rng_seed=3, top_k=1))
    assert runs[0] == runs[1]


class NoStep:
    def __init__(self, module):
        self.module = module

    def zero_grad(self, set_to_none=True):
        for p in self.module.parameters():
            p.grad = None

    def step(self):
        pass


def reference_update(PT, PS, c, ids, mask, k, tau):
    """Loss and the student's gradients by autograd on the CPU oracle, from the definition."""
    Pl = {n: v.detach().clone().double().requires_grad_(True) for n, v in PS.items()}
    teacher = O.generator_forward({n: v.double() for n, v in PT.items()}, c, ids, mask)
    student = O.generator_forward(Pl, c, ids, mask)
    logp, logq = torch.log_softmax(teacher / tau, -1), torch.log_softmax(student / tau, -1)
    top = torch.zeros_like(logp, dtype=torch.bool).scatter_(-1, teacher.topk(k, dim=-1).indices, True)
    ninf = float("-inf")
    rest_p, rest_q = logp.masked_fill(top, ninf).logsumexp(-1), logq.masked_fill(top, ninf).logsumexp(-1)
    kl = (logp.exp() * (logp - logq) * top).sum(-1) + rest_p.exp() * (rest_p - rest_q)
    w = (ids == 4).double()
    loss = tau * tau * (kl * w).sum() / w.sum()
    loss.backward()
    return float(loss.detach()), {n: v.grad for n, v in Pl.items() if v.grad is not None}


@pytest.mark.parametrize("name,dtype,bound", [("tiny", torch.float32, 2e-3), ("mid", torch.float32, 2e-3), ("mid", torch.bfloat16, 1.5e-1)])
def test_generator_distill_update_gradients_vs_oracle(pg, name, dtype, bound):
    """Loss and every gradient of the student against the oracle (the bounds of the soft generator update, which runs the same
    engine passes behind the same head)."""
    from protgen_gan_amd import train as T
    c, PT, PS, C, teacher, critic = build(pg, name, dtype)
    student = pg.Generator(critic.protbert)
    ids = _template(4, 48, 5)
    mask = (ids != 0).long()
    before = {n: p.detach().clone() for n, p in teacher.named_parameters()}
    loss = T.generator_distill_update(student, teacher, NoStep(student), ids.to(DEV), mask.to(DEV), k=6, temperature=2.0)
    l_ref, g_ref = reference_update(PT, PS, c, ids, mask, 6, 2.0)
    assert abs(float(loss) - l_ref) <= (1e-4 if dtype == torch.float32 else 5e-2) * abs(l_ref) + 1e-5
    got = {n[len("protbert."):]: p.grad for n, p in student.named_parameters() if p.grad is not None}
    assert set(got) == set(g_ref), set(got) ^ set(g_ref)
    typical = float(np.median([float(v.norm()) for v in g_ref.values()]))
    for n, v in g_ref.items():
        if float(v.norm()) >= 1e-3 * typical:
            assert rel_l2(got[n].cpu().numpy(), v.numpy()) < bound, n
    assert all(p.grad is None for p in teacher.parameters())
    assert all(torch.equal(p, before[n]) for n, p in teacher.named_parameters())


def test_distillation_loss_through_the_student(pg):
    """The autograd form behind the student's MLM head gives the gradients of the hand-scheduled update; with create_graph the
    second derivative is refused where it is taken."""
    from protgen_gan_amd import train as T
    c, PT, PS, C, teacher, critic = build(pg, "tiny", torch.float32)
    student = pg.Generator(critic.protbert)
    ids = _template(2, 32, 9).to(DEV)
    mask = (ids != 0).long()
    T.generator_distill_update(student, teacher, NoStep(student), ids, mask, k=5, temperature=1.5)
    want = {n: p.grad.clone() for n, p in student.named_parameters() if p.grad is not None}
    NoStep(student).zero_grad()
    with torch.no_grad():
        v, i, r = pg.ops.top_logits(teacher(ids, mask), 5, temperature=1.5)
        w = (ids == 4).float()
        w /= w.sum()
    logits = student(ids, mask)
    pg.loss.distillation_loss(logits, v, i, rest=r, temperature=1.5, weights=w).sum().backward()
    for n, p in student.named_parameters():
        if n in want:
            assert rel_l2(p.grad.cpu().numpy(), want[n].cpu().numpy()) < 1e-5, n
    x = logits.detach().requires_grad_()
    g, = torch.autograd.grad(pg.loss.distillation_loss(x, v, i, rest=r).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.square().sum().backward()


def test_distil_then_fill(pg):
    """A run as it would be used: a shallower student learns from a teacher's records over a few templates, then fills with
    truncated sampling.  Nothing is asked of the loss but that it is finite and that the weights move."""
    from protgen_gan_amd import generate as G
    from protgen_gan_amd import train as T
    c, PT, PS, C, teacher, critic = build(pg, "mid", torch.bfloat16)
    cfg = pg.ProtBertConfig(hidden_size=c.hidden_size, num_hidden_layers=1, num_attention_heads=c.num_attention_heads,
                            intermediate_size=c.intermediate_size, max_position_embeddings=c.max_position_embeddings)
    student = pg.Generator(pg.ProtBertForMaskedLM(cfg, device=DEV, compute_dtype=torch.bfloat16).init_random(seed=1))
    opt = pg.AdamW(student.parameters(), lr=1e-3)
    before = student.protbert.store.master.clone()
    for step in range(3):
        ids = _template(4, 40, step).to(DEV)
        loss = T.generator_distill_update(student, teacher, opt, ids, (ids != 0).long(), k=8, temperature=2.0)
        assert math.isfinite(float(loss))
    assert not torch.equal(before, student.protbert.store.master)
    seqs = G.generate_full_mode_sequences(student, pg.ProtTokenizer(), 4, [25, 30], batch_size=4, device=DEV, rng_seed=1, top_p=0.9)
    assert len(seqs) == 4
