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


def certain(sharp, far, T, D, dtype, temp):
    """Two rows that are nearly certain of columns 3 and T - 2, and candidates 8 I (their first D), so that dq = 8 g / temp / 2 for the first D
    columns, with no sum over others: queries with z = sharp at the column and z = far at the D - 1 others, zero (z = 0) beyond D."""
    q = torch.full((2, D), far * temp / 8)
    p = torch.zeros(T, D)
    p[:D] = 8 * torch.eye(D)
    q[0, 3] = q[1, D - 2] = sharp * temp / 8
    return q.to(dtype), p.to(dtype), torch.tensor([[3], [D - 2]]), torch.zeros(2, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [64, 5000])
@pytest.mark.parametrize("sharp,far,temp", [(1000.0, 988.0, 0.125), (14.0, 2.0, 0.07), (1000.0, 988.0, -0.125), (1000.0, 988.0, 0.07),
                                            (4000.0, 3990.0, 1.0 / 3)])
def test_what_a_nearly_certain_row_still_has_to_learn(sharp, far, temp, T, dtype):
    """One entry, at the row's maximum m: the loss is log(sum), sum = 1 + (D - 1) exp(far - m), and g there is 1 / sum - 1.

    u = 2^-24.  A logit is rounded where it is made: its sum (one product), 1 / temp, theirs: 3 u |z| each for the maximum and for the others,
    whose difference is then off by 6 u |z| at most, and so is every share of the others, relative to itself; exp adds 8 u.  The sum of exp rounds
    at its size, 1 (each partial sum that holds the maximum: 2 + log2 of the waves' records, under 12 u), 1 / sum and the product 2 u: 14 u
    in all for the share at the maximum and, beside its others' 6 u |z| (1 - share), for the loss, whose logarithm adds 8 u.  In bf16 a result is
    rounded by 2^-8 of itself and g is held to 2^-15; fp32 products of parts lose 2^-21.  The row's g adds up to nothing but those."""
    D = 64
    q, p, index, score = certain(sharp, far, T, D, dtype, temp)
    t32 = float(torch.tensor(temp))
    z = q.double() @ p.double().t() / t32
    m, at = z.max(1)
    assert at.tolist() == index[:, 0].tolist()
    rest = torch.exp(z - m[:, None]).sum(1) - 1
    loss, agree, dq, _, _ = step(q, p, None, temp, index, score, 1.0)
    assert float(agree) == 1.0
    drift = 6 * U * abs(sharp) + 8 * U
    want = float(torch.log1p(rest).mean())
    assert abs(float(loss) - want) <= float(rest.max()) * drift + 22 * U, (float(loss), want)
    g = dq.double() * (2 * t32 / 8)                                 # 1 / temp and 1 / 2 were applied to g, 8 is the candidate's
    share = 2.0 ** -15 + 2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -21 + 4 * U
    ref = torch.exp(z - m[:, None])[:, :D] / (1 + rest)[:, None]
    ref[0, 3] -= 1
    ref[1, D - 2] -= 1
    lim = ref.abs() * (share + drift) + 14 * U * (ref < 0)
    assert bool(((g - ref).abs() <= lim).all()), float(((g - ref).abs() / lim).max())
    beyond = 1 - torch.exp(z - m[:, None])[:, :D].sum(1) / (1 + rest)           # the columns past D, whose share reaches no query
    total = (g.sum(1) + beyond).abs()
    assert bool((total <= ref.abs().sum(1) * share + 14 * U + beyond * drift).all()), total


@pytest.mark.parametrize("B,D", [(64, 64), (1500, 64), (1500, 1024)])
def test_bf16_gradients_hold_g_to_17_bits(B, D):
    """Candidates e_0 and -e_0 with nearly the same share, which no list names: dq_0 = (p_0 - p_1) / temp / B shows what g is off by.

    g is held in two rounded bf16 parts, to 2^-17 of itself, twice that in a difference; p itself is off by less than 16 u relative to a share of
    the row (|z| < 1: products and 1 / temp 3 u, exp 8 u, the sum and its reciprocal 5 u), 32 u in the difference; sums of two products and the
    factor 4 u; the result is rounded by 2^-8 of itself."""
    g = torch.Generator().manual_seed(B + D)
    temp = 1.0
    q, p = torch.zeros(B, D), torch.zeros(3, D)
    p[0, 0], p[1, 0], p[2, 1] = 1.0, -1.0, 1.0
    q[:, 0] = 2.0 ** -11
    q[:, 1] = torch.rand(B, generator=g) * 2 - 1
    q, p = q.bfloat16(), p.bfloat16()
    dq = step(q, p, None, temp, torch.full((B, 1), 2), torch.zeros(B, 1))[2].double()
    share = torch.softmax(q.double() @ p.double().t(), 1)
    want = (share[:, 0] - share[:, 1]) / B
    room = (share[:, 0] + share[:, 1]) / B * (2.0 ** -17 + 20 * U) + 2.0 ** -8 * want.abs()
    assert bool(((dq[:, 0] - want).abs() <= room).all()), float(((dq[:, 0] - want).abs() / room).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_best_entry_at_any_teacher_temperature(dtype):
    """An infinite temperature makes all shares alike; the best entry is still the one with the largest score."""
    g = torch.Generator().manual_seed(3)
    q = p = torch.eye(16, 64).to(dtype)
    index = torch.stack([torch.randperm(16, generator=g)[:6] for _ in range(16)])
    score = torch.rand(16, 6, generator=g)
    index[:8, 4], score[:8, 4] = torch.arange(8), 2.0               # half of the rows: the student's best is the teacher's, in the fifth place
    index[8:, 0], score[8:, 3] = torch.arange(8, 16), 2.0           # the others: it is in the first place, and not the teacher's best
    index[8:, 3] = (torch.arange(8, 16) + 1) % 16
    for tt in (INF, 3e38, 1e30, 1.0, 1e-3):
        loss, agree, *_ = step(q, p, None, 0.5, index, score, tt)
        r = distill_ref(q, p, 0.5, index, score, float(torch.tensor(tt)), 16)
        # 6 shares and logits of at most 2, each within a few u; at 1e-3 the scores' differences of 2000 are divided once: 2000 u
        assert float(agree) == 0.5 and r["agree"] == 0.5 and abs(float(loss) - float(r["loss"])) <= 2100 * U, tt


def test_a_loss_that_is_kept_holds_no_workspace():
    """After its backward a loss kept for a log is four bytes (an allocator's block); before it, or with retain_graph, the logits stay."""
    B, C, D = 256, 4096, 64
    g = torch.Generator().manual_seed(4)
    leaves = [x.to(DEV).requires_grad_(True) for x in (unit(B, D, g), unit(C, D, g))]
    index, score = torch.randint(C, (B, 4), generator=g).to(DEV), torch.rand(B, 4, generator=g).to(DEV)
    kept = []
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(DEV)
    for _ in range(3):
        loss, agree = call(leaves[0], leaves[1], None, 0.07, index, score, 1.0)
        torch.autograd.grad(loss, leaves, retain_graph=True)
        assert torch.cuda.memory_allocated(DEV) - before >= B * C * 4
        torch.autograd.grad(loss, leaves)
        kept.append((loss, agree))
        assert torch.cuda.memory_allocated(DEV) - before < 1 << 20
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(loss, leaves)


def test_temperatures_under_capture():
    """A number and a tensor on the card are captured; a parameter on the host, whose copy could not be, is refused and the capture goes on."""
    from vllm_amd._lib import AbcError
    from vllm_amd.loss import Temperature, compute_contrastive_loss
    g = torch.Generator().manual_seed(6)
    leaves = [x.to(DEV).requires_grad_(True) for x in (unit(32, 64, g), unit(80, 64, g))]
    index, score = torch.randint(80, (32, 4), generator=g).to(DEV), torch.rand(32, 4, generator=g).to(DEV)
    temps = (0.07, torch.tensor([0.07], device=DEV), Temperature().to(DEV))

    def passes():
        out = []
        for t in temps:
            loss, agree = call(leaves[0], leaves[1], None, t, index, score, 0.5)
            out += [loss.detach(), agree, *torch.autograd.grad(loss, leaves)]
        loss, acc = compute_contrastive_loss(leaves[0], leaves[1], 0.07)
        return out + [loss.detach(), acc, *torch.autograd.grad(loss, leaves)]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for host in (Temperature(), torch.tensor(0.07)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(AbcError, match="capture: the temperature is on cpu"):
                    call(leaves[0], leaves[1], None, host, index, score, 0.5)
        got = passes()
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(unit(32, 64, g))
        graph.replay()
        want = passes()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    host = Temperature()                                            # outside a capture it is brought over, and gets its gradient
    loss, _ = call(leaves[0], leaves[1], None, host, index, score, 0.5)
    loss.backward()
    assert host.temp.grad.device.type == "cpu" and torch.equal(loss.detach(), got[0])


def test_more_pairs_than_a_launch_has_threads_for():
    """65 535 rows of 2^19 candidates: 256 stretches of 2048 logits a row and the row's query are 257 x 65 535 workgroups of 256 threads."""
    B, T, d = 65535, 1 << 19, 8
    torch.cuda.empty_cache()
    need = 2 * B * T * 4 + (4 << 30)
    free = torch.cuda.mem_get_info(DEV)[0]
    if need > 0.95 * free:
        pytest.skip(f"{need >> 30} GiB of {free >> 30} GiB that are free")
    g = torch.Generator(DEV).manual_seed(1)
    q, p = torch.randn(B, d, device=DEV, generator=g).bfloat16(), torch.randn(T, d, device=DEV, generator=g).bfloat16()
    index, score = torch.randint(T, (B, 3), device=DEV, generator=g), torch.rand(B, 3, device=DEV, generator=g)
    q[5], index[5] = NAN, -1
    q.requires_grad_(True)
    p.requires_grad_(True)
    loss, _ = call(q, p, None, 1.0, index, score, 1.0)
    dq, dp = torch.autograd.grad(loss, (q, p))
    assert bool(torch.isfinite(loss.detach())) and bool(torch.isfinite(dp).all()) and not dq[5].any()
    rows = [0, 1, B // 2, B - 1]
    shares = torch.softmax(q.detach()[rows].double() @ p.detach().double().t(), 1)
    want = shares.scatter_add(1, index[rows], -torch.softmax(score[rows].double(), 1)) @ p.detach().double() / (B - 1)
    # a result is rounded by 2^-8 of itself at most; g by 2^-17 of the shares and of the list's, whose sums of candidates (|c| up to 5) are not small
    size = (shares @ p.detach().double().abs() + 5) / (B - 1)
    assert bool(((dq[rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * size).all())
    del loss, dq, dp
    torch.cuda.empty_cache()
