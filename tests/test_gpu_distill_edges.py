"""The distillation loss where a row counts nowhere, where a student is nearly certain, and around a call: what it keeps, what it answers
under a graph capture."""
import pytest
import torch

import oracle  # noqa: F401
from oracle.distill_oracle import distill_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")
U = 2.0 ** -24


def unit(n, d, g):
    return torch.nn.functional.normalize(torch.randn(n, d, generator=g), dim=-1)


def call(q, p, m, temp, index, score, tt):
    from vllm_amd import loss
    return loss.compute_distillation_loss(q, p, temp, index, score, teacher_temperature=tt, memory=m)


def step(q, p, m, temp, index, score, tt=0.05):
    """loss, agreement and the gradients of queries, candidates and temperature, on the CPU"""
    leaves = [x.to(DEV).requires_grad_(True) for x in (q, p, torch.tensor(temp))]
    loss, agree = call(leaves[0], leaves[1], None if m is None else m.to(DEV), leaves[2], index.to(DEV), score.to(DEV), tt)
    return [x.detach().cpu() for x in (loss, agree) + torch.autograd.grad(loss, leaves)]


# the products' forms: 64 wide tiles with and without parts of k, 128 wide ones, fp32 by fp16 parts, those with a row that they do not hold
# (the candidates' gradient with the queries' 16-bit parts, or with the queries themselves)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(10, 30, 0, 64, 6), (33, 200, 60, 2056, 5), (400, 1501, 0, 1024, 7), (1000, 2601, 600, 264, 9),
                                   (256, 1000, 15_400, 1024, 40), (256, 1000, 15_400, 1024, -40)])
def test_what_a_row_without_an_entry_holds_reaches_nobody(shape, dtype):
    B, C, M, D, k = shape
    g = torch.Generator().manual_seed(sum(shape))
    q, p, m = (unit(n, D, g).to(dtype) for n in (B, C, M))
    if k < 0:
        k = -k
        q[0] *= 2.0 ** 20                                           # a live row past the fp16 parts' range
    index = torch.argsort(torch.rand(B, C + M, generator=g), 1)[:, :k].clone()
    score = torch.rand(B, k, generator=g)
    dead = torch.tensor([3, 5, 6, B - 1])
    index[dead[:2]], score[dead[2:]] = -1, -INF
    zero, bad = q.clone(), q.clone()
    zero[dead] = 0.0
    bad[3, 5], bad[5], bad[6, D - 1], bad[B - 1, ::2] = INF, NAN, -INF, NAN
    want, got = step(zero, p, m if M else None, 0.07, index, score), step(bad, p, m if M else None, 0.07, index, score)
    assert bool(torch.isfinite(want[0])) and all(bool(torch.isfinite(x).all()) for x in want[2:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not got[2][dead].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(10, 30, 5, 64, 6), (40, 64, 4000, 64, 3), (130, 3900, 201, 1024, 9), (256, 1000, 15_400, 1024, 4)])
def test_a_row_without_an_entry_receives_nothing(shape, dtype):
    """A candidate that is no number (a memory read past its store) leaves the rows with an entry without an answer, and the others at zero."""
    B, C, M, D, k = shape
    g = torch.Generator().manual_seed(sum(shape))
    q, p, m = (unit(n, D, g).to(dtype) for n in (B, C, M))
    m[M // 2] = NAN
    index, score = torch.randint(C, (B, k), generator=g), torch.rand(B, k, generator=g)
    index[2], index[B - 2] = -1, -1
    loss, _, dq, dp, dt = step(q, p, m, 0.07, index, score)
    rows = torch.ones(B, dtype=torch.bool)
    rows[2], rows[B - 2] = False, False
    assert bool(torch.isnan(loss)) and bool(torch.isnan(dt)) and bool(torch.isnan(dq[rows]).all()) and not dq[~rows].any()
    index[:] = -1
    out = step(q, p, m, 0.07, index, score)
    assert not any(bool(x.any()) for x in out)                      # (a NaN is not zero)
