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


def test_rows_beyond_a_launch_are_refused(pg):
    """A launch counts its threads in 32 bits: 32 or 64 threads a row up to 64 entries, 256 or 512 above."""
    lib, p = pg._lib.lib, torch.zeros(64).data_ptr()
    top = lambda T, V: lib.pg_top_logits(0, p, V, T, V, 3, 1.0, p, p, p, None, 0, None)  # noqa: E731
    fwd = lambda T, V, k=3: lib.pg_distill_fwd(0, p, V, T, V, p, p, k, None, None, 1.0, p, p, None, 0, None)  # noqa: E731
    bwd = lambda T, V, k=3: lib.pg_distill_bwd(0, p, V, T, V, p, p, k, None, 1.0, None, p, p, V, None)  # noqa: E731
    both = lambda T, V, k=3: lib.pg_distill_loss_grad(0, p, V, T, V, p, p, k, None, None, 1.0, p, p, V, None, 0, None)  # noqa: E731
    for call in (top, fwd, bwd, both, lambda T, V: sample(lib, p, T, V)):
        assert call(2 ** 27, 30) == UNSUPPORTED and call(2 ** 26, 40) == UNSUPPORTED and call(2 ** 31 - 1, 4) == UNSUPPORTED
        assert call(2 ** 24, 300) == UNSUPPORTED
    for call in (fwd, bwd, both):  # (records of more than 64 entries, or 32, take the wider forms)
        assert call(2 ** 24, 30, 100) == UNSUPPORTED and call(2 ** 26, 30, 40) == UNSUPPORTED
    assert both(2 ** 23, 20000) == UNSUPPORTED
    big = torch.zeros(1 << 20, dtype=torch.uint8)  # (a workspace, by its address and a size that is asked for only)
    at = (big.data_ptr() + 15) // 16 * 16
    assert lib.pg_sample_filtered(0, p, 300, p, 300, 2 ** 23, 300, 1.0, 0, 0.5, 0.0, None, None, None, None, -1, p, p, at, 2 ** 62, None) == UNSUPPORTED


def test_sizes_beyond_the_int_of_the_c_abi_are_refused(pg):
    """2^32 + 1 rows would arrive as one."""
    one = torch.zeros(1)
    for T, V in ((2 ** 32 + 1, 1), (2 ** 31, 1), (1, 2 ** 32 + 7)):
        x = one.expand(T, V)
        with pytest.raises(ValueError, match="more than a call takes"):
            pg.ops.top_logits(x, 1)
        with pytest.raises(ValueError, match="more than a call takes"):
            pg.ops.sample_filtered(x, x)
        with pytest.raises(ValueError, match="more than a call takes"):
            pg.ops.distill_loss_grad(x, one.expand(T, 1), one.int().expand(T, 1))
    with pytest.raises(ValueError, match="empty"):
        pg.ops.sample_filtered(torch.zeros(2, 3), torch.ones(2, 3), empty=2 ** 32)


@pytest.mark.parametrize("T,V", [(0, 1000), (0, 30), (-1, 1000), (-(2 ** 31), 100000), (4, 0), (4, -1), (0, 0)])
def test_workspace_of_sizes_that_are_refused_is_nothing(pg, T, V):
    """(Zero rows once divided by zero, which ends the process.)"""
    lib, p = pg._lib.lib, torch.zeros(64).data_ptr()
    for dt in (0, 1):
        for k in (3, 100, 0, -1):
            assert lib.pg_top_logits_workspace_bytes(dt, T, V, k) == 0 and lib.pg_sample_filtered_workspace_bytes(dt, T, V, k) == 0
            assert lib.pg_distill_workspace_bytes(dt, T, V, k, 0) == 0 and lib.pg_distill_workspace_bytes(dt, T, V, k, 1) == 0
            assert lib.pg_distill_loss_grad(dt, p, 8, T, V, p, p, k, None, None, 1.0, p, p, 8, None, 0, None) == ARG
    for T in (1, 1023, 1024, 2 ** 22, 2 ** 31 - 1):  # (and of the largest counts no overflow)
        assert lib.pg_distill_workspace_bytes(0, T, 100000, 3, 1) >= 0
