"""Sizes and layouts that the operators over rows of vocabulary logits refuse on the host, before a launch (the pointers are host
memory: nothing may be launched)."""
import pytest
import torch

ARG, UNSUPPORTED, WORKSPACE = -1, -4, -5


@pytest.fixture(scope="module")
def pg():
    import pgload
    return pgload.load()


def sample(lib, p, T, V, **kw):
    a = dict(temperature=1.0, k=0, top_p=0.5, min_p=0.0)
    a.update(kw)
    return lib.pg_sample_filtered(0, p, V, p, V, T, V, a["temperature"], a["k"], a["top_p"], a["min_p"], None, None, None, None, -1, p, p,
                                  None, 0, None)


def test_sampling_refuses_a_vocabulary_whose_mass_would_wrap(pg):
    """2^24 equal entries weigh 2^24 * 2^40 = 2^64 in the 64-bit sums.  The record and the distillation have no such sum."""
    lib, p = pg._lib.lib, torch.zeros(64).data_ptr()
    assert sample(lib, p, 1, 1 << 24) == UNSUPPORTED and sample(lib, p, 1, (1 << 24) + 1) == UNSUPPORTED
    assert sample(lib, p, 1, (1 << 24) - 1) == WORKSPACE
    assert lib.pg_distill_fwd(0, p, 1 << 24, 1, 1 << 24, p, p, 3, None, None, 1.0, p, p, None, 0, None) == WORKSPACE


@pytest.mark.parametrize("stash", [torch.zeros(1).expand(32), torch.zeros(64)[::2], torch.zeros(31), torch.zeros(4, 8)])
def test_distill_bwd_refuses_a_stash_of_another_layout(pg, stash):
    """The kernel reads eight numbers a row one behind the other; an expanded or strided stash holds fewer in a row than that."""
    x, v, i = torch.zeros(4, 10), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="stash"):
        pg.ops.distill_bwd(x, v, i, stash, torch.ones(4))
