"""Corners of the operators over rows of vocabulary logits that documented arguments reach.  Bounds as in test_gpu_logits."""
import pytest
import torch

from tests.test_gpu_logits import DEV, TYPES, check_sample, rows

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
