"""The distillation loss on the GPU against its closed form in 64 bits (oracle/distill_oracle.py, which also derives how far fp32
arithmetic may be from it), its gradients against differences, and the calls a training program makes around it."""
import pytest
import torch

import oracle  # noqa: F401
from oracle.distill_oracle import distill_bounds, distill_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


def unit(n, d, g):
    return torch.nn.functional.normalize(torch.randn(n, d, generator=g), dim=-1)


def problem(B, C, M, D, k, seed, dtype=torch.float32, holes=True, twice=False):
    g = torch.Generator().manual_seed(seed)
    q, p, m = unit(B, D, g), unit(C, D, g), unit(M, D, g)
    n = min(B, C)
    p[:n] = torch.nn.functional.normalize(q[:n] + 0.8 * p[:n], dim=-1)
    T = C + M
    if twice or k > T:
        index = torch.randint(T, (B, k), generator=g)
    else:
        index = torch.argsort(torch.rand(B, T, generator=g), 1)[:, :k].clone()
    score = (torch.rand(B, k, generator=g) * 0.7).sort(1, descending=True)[0]
    if holes and B > 2:
        index[0, k // 2:], score[0, k // 2:] = -1, -INF             # a short list (none at all where k = 1)
        score[1, 0] = -INF                                          # an entry taken out by its score alone
        index[2, :] = -7                                            # and a row with nothing in it, by its indices alone
        if B > 5:
            index[4, 0] = -1                                        # the best entry taken out: the next one is the best
    return q.to(dtype), p.to(dtype), m.to(dtype), index, score


def call(q, p, m, temp, index, score, tt, **kw):
    from vllm_amd import loss
    return loss.compute_distillation_loss(q, p, temp, index, score, teacher_temperature=tt, memory=m, **kw)


def check(B, C, M, D, k, seed=0, dtype=torch.float32, temp=0.07, tt=0.05, grad_out=1.0, **kw):
    q, p, m, index, score = problem(B, C, M, D, k, seed, dtype, **kw)
    cand = torch.cat((p, m))
    t32 = float(torch.tensor(temp, dtype=torch.float32))
    r = distill_ref(q, cand, t32, index, score, tt, C, grad_out)
    lim = distill_bounds(r, q, cand, t32, score, tt, C, k, dtype is torch.bfloat16, grad_out)
    qd, pd = q.to(DEV).requires_grad_(True), p.to(DEV).requires_grad_(True)
    td = torch.tensor(temp, device=DEV, requires_grad=True)
    loss, agree = call(qd, pd, m.to(DEV) if M else None, td, index.to(DEV), score.to(DEV), tt)
    dq, dp, dt = torch.autograd.grad(loss * grad_out, (qd, pd, td))
    assert dq.dtype == dtype and dp.dtype == dtype and loss.dtype == torch.float32
    assert abs(float(loss.detach()) - float(r["loss"])) <= lim["loss"], (float(loss), float(r["loss"]), lim["loss"])
    assert float(agree) == pytest.approx(r["agree"], abs=1e-6)
    for name, got in (("dq", dq), ("dp", dp)):
        err = (got.cpu().double() - r[name]).abs()
        assert bool((err <= lim[name]).all()), (name, float((err / lim[name].clamp(min=1e-300)).max()))
        # The bound above is the worst case; over a whole gradient roundings fall at random.  g = p - target is as exact as p and the
        # target are, so the measure is N = (p + target) @ |c|, not g @ c (a single row whose list holds the column that the student
        # prefers has g near 0).  p = exp(z - l): z (|z| <= 1 / temp for unit rows: the product's sum, its rounding, the division), l
        # (|l| <= 1 / temp + log T, most often its logarithm is the smaller part) and their difference are each off by at most a few
        # u / temp: 18 u / temp covers 3 + 1 + 1 roundings and the sums' sqrt(D / 16) <= 12.  bf16: one rounding more, g in two parts.
        big = ((r["p"] + r["target"]) * r["some"][:, None]).double() * (abs(grad_out) / r["rows"] / t32)
        N = float((big @ cand.double().abs() if name == "dq" else big.t() @ q.double().abs()).norm())
        room = 18 / t32 * 2.0 ** -24 * N
        if dtype is torch.bfloat16:
            room += 2.0 ** -8 * float(r[name].norm()) + 2.0 ** -15 * N
        assert float(err.norm()) <= room, (name, float(err.norm()), room)
    assert abs(float(dt) - float(r["dtemp"])) <= lim["dtemp"], (float(dt), float(r["dtemp"]), lim["dtemp"])
    return loss, agree, dq, dp, dt


SHAPES = [(1, 1, 0, 8, 1), (1, 3, 0, 16, 2), (2, 5, 7, 24, 3), (33, 100, 0, 72, 10), (64, 64, 64, 64, 64), (65, 129, 1, 128, 128),
          (128, 1024, 0, 512, 64), (5, 4097, 9000, 136, 100), (130, 1, 300, 64, 5), (7, 19, 0, 13, 4), (3, 40, 11, 129, 6),
          (200, 300, 5000, 256, 1024), (257, 513, 100, 328, 17), (40, 2000, 30, 1024, 33), (6, 5, 0, 2056, 2)]


# fp32 products of 8 GFLOP and more go by fp16 parts
# tiles of 128 and, fp32, of 256 rows of queries; the second: of 128 alone, with odd ends on every side; then fp32 gradients, and all three
# products, in tiles of 128 without the fp16 parts; narrow rows, the second of them in tiles of 128 x 96 (bf16)
LARGE = [(256, 1000, 15_400, 1024, 40), (300, 901, 12_000, 1192, 17), (520, 2100, 0, 4096, 9), (400, 1501, 0, 1024, 7), (130, 3900, 201, 3000, 9),
         (1000, 2000, 29_001, 136, 5), (1000, 2601, 600, 264, 9), (700, 1500, 7, 8, 3), (513, 900, 0, 24, 5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", LARGE)
def test_large(shape, dtype):
    check(*shape, seed=sum(shape), dtype=dtype)


@pytest.mark.parametrize("what", ["large query", "tiny queries", "large candidate", "tiny memory row", "infinite candidate", "zero rows"])
def test_large_fp32_where_fp16_parts_do_not_hold(what):
    """The largest magnitude of a row outside [2^-10, 65000]: the six products take over, for all rows."""
    B, C, M, D, k = 256, 1000, 15_400, 1024, 5
    q, p, m, index, score = problem(B, C, M, D, k, 21)
    temp = 0.07
    if what == "large query":
        q[7] *= 3e6
        p, m, temp = p * 1e-3, m * 1e-3, 5.0
    elif what == "tiny queries":
        q *= 1e-4
        temp = 1e-5
    elif what == "large candidate":
        p[999] *= 1e7
        q *= 1e-2
        temp = 1e3
    elif what == "tiny memory row":
        m[15_399] *= 1e-6
    elif what == "infinite candidate":
        p[3, 9] = INF
    else:
        q[9], p[17], m[0] = 0.0, 0.0, 0.0                           # held by the fp16 parts
    leaves = [x.to(DEV).requires_grad_(True) for x in (q, p, torch.tensor(temp))]
    loss, _ = call(leaves[0], leaves[1], m.to(DEV), leaves[2], index.to(DEV), score.to(DEV), 0.05)
    dq, dp, dt = torch.autograd.grad(loss, leaves)
    if what == "infinite candidate":
        assert bool(torch.isnan(loss.detach())) and bool(torch.isnan(dq[0]).all())
        return
    cand = torch.cat((p, m))
    t32 = float(torch.tensor(temp))
    r = distill_ref(q, cand, t32, index, score, 0.05, C)
    lim = distill_bounds(r, q, cand, t32, score, 0.05, C, k, False)
    assert abs(float(loss.detach()) - float(r["loss"])) <= lim["loss"]
    for got, name in ((dq, "dq"), (dp, "dp"), (dt, "dtemp")):
        assert bool(((got.cpu().double() - r[name]).abs() <= lim[name]).all()), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_closed_form(shape, dtype):
    check(*shape, seed=sum(shape), dtype=dtype)


def test_a_column_named_twice_adds_up():
    check(20, 30, 0, 64, 100, seed=1, twice=True)
    check(9, 6000, 0, 64, 700, seed=2, twice=True, dtype=torch.bfloat16)


def test_grad_out_and_temperatures():
    check(16, 50, 20, 96, 8, seed=3, grad_out=-3.5, temp=0.5, tt=2.0)
    check(16, 50, 20, 96, 8, seed=4, grad_out=1e-3, temp=0.02, tt=0.01)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_an_entry(dtype):
    q, p, m, index, score = problem(10, 30, 5, 64, 6, 5, dtype)
    index[:] = -1
    qd, pd, td = q.to(DEV).requires_grad_(True), p.to(DEV).requires_grad_(True), torch.tensor(0.07, device=DEV, requires_grad=True)
    loss, agree = call(qd, pd, m.to(DEV), td, index.to(DEV), score.to(DEV), 0.05)
    assert float(loss.detach()) == 0.0 and float(agree) == 0.0
    for g in torch.autograd.grad(loss, (qd, pd, td)):
        assert bool((g == 0).all())
    # an infinity in a row that counts nowhere stays out of the loss and of everyone's gradients
    q, p, m, index, score = problem(10, 30, 0, 64, 6, 6, dtype, holes=False)
    index[3] = -1
    clean = q.clone()
    q[3, 5] = INF
    out = []
    for x in (q, clean):
        qd, pd = x.to(DEV).requires_grad_(True), p.to(DEV).requires_grad_(True)
        loss, _ = call(qd, pd, None, 0.07, index.to(DEV), score.to(DEV), 0.05)
        dq, _ = torch.autograd.grad(loss, (qd, pd))
        out.append((loss.detach(), dq))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


def test_what_is_not_a_number_shows():
    q, p, m, index, score = problem(8, 30, 0, 64, 6, 7, holes=False)
    for change in ("index", "query", "score", "score+"):
        qq, ii, ss = q.clone(), index.clone(), score.clone()
        if change == "index":
            ii[2, 1] = 30                                           # one past the last candidate
        elif change == "query":
            qq[2, 0] = float("nan")
        else:
            ss[2, 0] = INF if change == "score+" else float("nan")
        qd = qq.to(DEV).requires_grad_(True)
        loss, _ = call(qd, p.to(DEV), None, 0.07, ii.to(DEV), ss.to(DEV), 0.05)
        dq, = torch.autograd.grad(loss, (qd,))
        assert bool(torch.isnan(loss)), change
        nan = torch.isnan(dq).any(1).cpu()
        assert bool(nan[2]) and int(nan.sum()) == 1, change         # the other rows' gradients are theirs


def test_one_entry_is_the_contrastive_loss():
    from vllm_amd import loss
    B, C, D = 48, 200, 256
    q, p, _, _, _ = problem(B, C, 0, D, 1, 8)
    index, score = torch.arange(B)[:, None], torch.zeros(B, 1)
    a = [x.to(DEV).requires_grad_(True) for x in (q, p, torch.tensor(0.07))]
    l1, acc = loss.compute_contrastive_loss(*a)
    g1 = torch.autograd.grad(l1, a)
    l2, agree = loss.compute_distillation_loss(a[0], a[1], a[2], index.to(DEV), score.to(DEV))
    g2 = torch.autograd.grad(l2, a)
    # both losses are means of l - z, each off by a few u (|l| + |z|) <= 2 u / 0.07; the gradients by check()'s 18 u / temp of N, twice
    assert abs(float(l1.detach()) - float(l2.detach())) <= 16 * 2.0 ** -24 * 2 / 0.07 and float(acc) == float(agree)
    r = distill_ref(q, p, 0.07, index, score, 1.0, C)
    big = (r["p"] + r["target"]) / (B * 0.07)
    for x, y, N in zip(g1, g2, (big @ p.double().abs(), big.t() @ q.double().abs(), big * r["z"].abs())):
        assert float((x - y).norm()) <= 2 * 18 / 0.07 * 2.0 ** -24 * float(N.norm())
    t = loss.Temperature().to(DEV)                                  # the module, as the trainer holds it
    l3, _ = loss.compute_distillation_loss(a[0], a[1], t, index.to(DEV), score.to(DEV))
    l3.backward()
    assert torch.equal(l3.detach(), l2.detach()) and torch.equal(t.temp.grad, g2[2])


def test_against_differences():
    """d loss along a direction, from the loss itself: central differences of the 64-bit form, step 1e-5 (error about 1e-9)."""
    q, p, m, index, score = problem(12, 40, 9, 48, 7, 9)
    t32 = float(torch.tensor(0.07))
    g = torch.Generator().manual_seed(1)
    vq, vp = torch.randn(12, 48, generator=g).double(), torch.randn(40, 48, generator=g).double()
    qd, pd, td = q.to(DEV).requires_grad_(True), p.to(DEV).requires_grad_(True), torch.tensor(0.07, device=DEV, requires_grad=True)
    loss, _ = call(qd, pd, m.to(DEV), td, index.to(DEV), score.to(DEV), 0.05)
    dq, dp, dt = (x.cpu().double() for x in torch.autograd.grad(loss, (qd, pd, td)))

    def f(hq=0.0, hp=0.0, ht=0.0):
        return float(distill_ref(q.double() + hq * vq, torch.cat((p.double() + hp * vp, m.double())), t32 + ht, index, score, 0.05, 40)["loss"])

    h = 1e-5
    for got, hi, lo in (((dq * vq).sum(), f(hq=h), f(hq=-h)), ((dp * vp).sum(), f(hp=h), f(hp=-h)), (dt, f(ht=h), f(ht=-h))):
        want = (hi - lo) / (2 * h)
        assert abs(float(got) - want) <= 1e-4 * abs(want) + 1e-6, (float(got), want)


def test_types_strides_and_what_is_asked_for():
    q, p, m, index, score = problem(12, 40, 9, 64, 7, 10)
    base = check(12, 40, 9, 64, 7, seed=10)
    # strided views, an unaligned slice, int32 indices, bf16 scores that fp32 holds exactly, memory of another type
    wide = torch.zeros(12, 131, device=DEV)
    wide[:, 1:129:2] = q.to(DEV)
    flat = torch.zeros(40 * 64 + 3, device=DEV)
    flat[3:] = p.reshape(-1).to(DEV)
    mem = m.t().contiguous().to(DEV).t()
    loss, agree = call(wide[:, 1:129:2], flat[3:].view(40, 64), mem, 0.07, index.int().to(DEV), score.to(DEV), 0.05)
    assert torch.equal(loss, base[0].detach()) and torch.equal(agree, base[1])
    half, _ = call(q.to(DEV).bfloat16(), p.to(DEV), m.to(DEV).bfloat16(), 0.07, index.to(DEV), score.to(DEV).bfloat16(), 0.05)
    same, _ = call(q.bfloat16().float().to(DEV), p.to(DEV), m.bfloat16().float().to(DEV), 0.07, index.to(DEV),
                   score.bfloat16().float().to(DEV), 0.05)
    assert torch.equal(half, same)
    # a gradient that is not asked for is not computed, and the others are the same bits
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, True, True)):
        leaves = [x.to(DEV).requires_grad_(n) for x, n in zip((q, p, torch.tensor(0.07)), need)]
        loss, _ = call(leaves[0], leaves[1], m.to(DEV), leaves[2], index.to(DEV), score.to(DEV), 0.05)
        got = torch.autograd.grad(loss, [x for x, n in zip(leaves, need) if n])
        assert all(torch.equal(a, b) for a, b in zip(got, [b for b, n in zip(base[2:], need) if n]))
    with torch.no_grad():
        loss, _ = call(q.to(DEV), p.to(DEV), m.to(DEV), 0.07, index.to(DEV), score.to(DEV), 0.05)
    assert torch.equal(loss, base[0].detach()) and not loss.requires_grad
    # an empty memory is none
    a, _ = call(q.to(DEV), p.to(DEV), m[:0].to(DEV), 0.07, index.clamp(max=39).to(DEV), score.to(DEV), 0.05)
    b, _ = call(q.to(DEV), p.to(DEV), None, 0.07, index.clamp(max=39).to(DEV), score.to(DEV), 0.05)
    assert torch.equal(a, b)


def test_two_losses_alive_backward_twice_and_leaves_untouched():
    one, two = problem(60, 300, 70, 128, 9, 11), problem(60, 300, 70, 128, 9, 12)
    want = [check(60, 300, 70, 128, 9, seed=s) for s in (11, 12)]
    leaves = [[x.to(DEV).requires_grad_(True) for x in pr[:2]] + [torch.tensor(0.07, device=DEV, requires_grad=True)] for pr in (one, two)]
    rest = [[x.to(DEV) for x in pr[2:]] for pr in (one, two)]
    losses = [call(lv[0], lv[1], rs[0], lv[2], rs[1], rs[2], 0.05)[0] for lv, rs in zip(leaves, rest)]
    second = torch.autograd.grad(losses[1], leaves[1], retain_graph=True)
    first = torch.autograd.grad(losses[0], leaves[0], retain_graph=True)
    again = torch.autograd.grad(losses[1], leaves[1])
    assert all(torch.equal(a, b) for a, b in zip(first, want[0][2:]))
    assert all(torch.equal(a, b) for a, b in zip(second, want[1][2:])) and all(torch.equal(a, b) for a, b in zip(again, second))
    # one tensor as queries and as candidates: its two gradients add up
    x = one[0].to(DEV).requires_grad_(True)
    index, score = torch.arange(60)[:, None].flip(0).to(DEV), torch.zeros(60, 1, device=DEV)
    loss, _ = call(x, x, None, 0.07, index, score, 1.0)
    g, = torch.autograd.grad(loss, (x,))
    y, z = x.detach().clone().requires_grad_(True), x.detach().clone().requires_grad_(True)
    loss, _ = call(y, z, None, 0.07, index, score, 1.0)
    assert torch.equal(g, sum(torch.autograd.grad(loss, (y, z))))
    # the list is done with after the forward; the candidates are not, and autograd says so where they were changed
    want = torch.autograd.grad(call(y, z, None, 0.07, index, score, 1.0)[0], (y, z))
    idx = index.clone()
    loss, _ = call(y, z, None, 0.07, idx, score, 1.0)
    idx.zero_()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (y, z)), want))
    loss, _ = call(y, z, None, 0.07, index, score, 1.0)
    with torch.no_grad():
        z.mul_(2)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(loss, (y, z))


def test_on_another_stream_and_in_captured_graphs():
    pr = [x.to(DEV) for x in problem(40, 260, 90, 192, 12, 13)]
    q, p, m, index, score = pr
    leaves = (q.requires_grad_(True), p.requires_grad_(True), torch.tensor(0.07, device=DEV, requires_grad=True))

    def step():
        loss, agree = call(leaves[0], leaves[1], m, leaves[2], index, score, 0.05)
        return (loss.detach(), agree) + torch.autograd.grad(loss, leaves)

    want = step()
    st = torch.cuda.Stream(DEV)
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = step()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # with an eager loss of the leaves alive, a captured backward would end the process: the loss is refused before that
    from vllm_amd._lib import AbcError
    spare = torch.zeros(4, device=DEV)
    for leaf in range(3):
        alive = leaves[leaf].sum()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            with pytest.raises(AbcError, match="alive from before"):
                call(leaves[0], leaves[1], m, leaves[2], index, score, 0.05)
            spare.add_(1)
        del alive
    # two graphs of the same leaves; the second has two losses of them in one capture, the contrastive one among them
    from vllm_amd.loss import compute_contrastive_loss
    graphs, outs = [], []
    for both in (False, True):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            if both:
                hard, _ = compute_contrastive_loss(*leaves)
                outs.append(step())
                del hard
            else:
                outs.append(step())
        graphs.append(g)
    for i in range(3):
        fresh = problem(40, 260, 90, 192, 12, 100 + i)
        with torch.no_grad():
            leaves[0].copy_(fresh[0])
            leaves[1].copy_(fresh[1])
            m.copy_(fresh[2])
            index.copy_(fresh[3])
            score.copy_(fresh[4])
            leaves[2].fill_(0.05 + 0.01 * i)
        graphs[0].replay()
        graphs[1].replay()
        want = step()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_in_a_captured_graph(dtype):
    """The large products' kernels ask for more LDS than a launch has by itself, also while a graph is captured."""
    q, p, m, index, score = (x.to(DEV) for x in problem(256, 1000, 15_400, 1024, 40, 3, dtype))
    leaves = (q.requires_grad_(True), p.requires_grad_(True), torch.tensor(0.07, device=DEV, requires_grad=True))

    def step():
        loss, agree = call(leaves[0], leaves[1], m, leaves[2], index, score, 0.05)
        return (loss.detach(), agree) + torch.autograd.grad(loss, leaves)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i in range(3):
        with torch.no_grad():
            leaves[0].mul_(-1)
            leaves[2].fill_(0.05 + 0.01 * i)
            if dtype is torch.float32 and i == 1:
                leaves[1][5] *= 1e6                              # past what the fp16 parts hold: the other kernels run in this replay
        g.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_training_step_over_a_store():
    """As a program uses them together: a teacher's store answers with its best rows, the student's memory of older candidates is read
    back, the loss draws the student towards the teacher's list, the step's candidates enter the memory."""
    from oracle import store_oracle
    from vllm_amd import search
    g = torch.Generator().manual_seed(77)
    B, C, M, D, Dt, k = 24, 96, 200, 128, 320, 10
    teacher_c, teacher_q = unit(C + M, Dt, g), unit(B, Dt, g)
    q, p, old = unit(B, D, g), unit(C, D, g), unit(M, D, g)
    teacher = search.EmbeddingStore(C + M, Dt, "fp4", 64, DEV)
    teacher.append(teacher_c.to(DEV))
    memory = search.EmbeddingStore(M, D, "i8", device=DEV)
    memory.append(old.to(DEV))
    score, index = teacher.scores(teacher_q.to(DEV)).topk(k, dim=1)
    qd, pd = q.to(DEV).requires_grad_(True), p.to(DEV).requires_grad_(True)
    td = torch.tensor(0.07, device=DEV, requires_grad=True)
    loss, agree = call(qd, pd, memory.read(), td, index, score, 0.1)
    grads = torch.autograd.grad(loss, (qd, pd, td))
    memory.append(pd.detach())
    cand = torch.cat((p.double(), store_oracle.store_values(old, 0).float().double()))
    t32 = float(torch.tensor(0.07))
    r = distill_ref(q, cand, t32, index.cpu(), score.cpu(), 0.1, C)
    lim = distill_bounds(r, q, cand, t32, score.cpu(), 0.1, C, k, False)
    assert abs(float(loss.detach()) - float(r["loss"])) <= lim["loss"]
    for got, name in zip(grads, ("dq", "dp", "dtemp")):
        assert bool(((got.cpu().double() - r[name]).abs() <= lim[name]).all())
    # the teacher's scores are those of the values its store holds
    want = teacher_q.double() @ store_oracle.store_values(teacher_c, 64).t()
    assert float((score.cpu().double() - want.gather(1, index.cpu())).abs().max()) <= (Dt + 11) * 2.0 ** -24
    # the memory is a corpus: the 8-bit form is searched by the exact top-k, and holds the step's candidates now
    idx = search.topk(search.Embeddings(p[:5].to(DEV), "i8"), memory.embeddings(), 1)[1][:, 0].cpu()
    assert torch.equal(idx, torch.arange(5))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_memory_past_4_gib(dtype):
    """Rows behind 2^32 bytes are the ones the lists name.  Reference in fp64 by a matrix product of this card.

    A score of unit rows is off by at most 2^-21 (what the parts leave out) + D / 32 * 2^-24 (the sums): 8.2e-6, z by 1.2e-4 at a
    temperature of 0.07, a row's loss by twice that and a probability by 2.4e-4 of itself.  dq is a sum of unit rows, by g / temp / rows: its
    norm is off by at most that share of (|p|_1 + |t|_1) / temp / rows = 2 / 0.07 / 8, and by its own rounding."""
    d, M, B, C, temp = 4096, (1 << 32) // (4096 * (4 if dtype is torch.float32 else 2)) + 3001, 8, 4, 0.07
    g = torch.Generator(DEV).manual_seed(5)
    unit_rows = lambda n: torch.nn.functional.normalize(torch.randn(n, d, generator=g, device=DEV), dim=1).to(dtype)
    q, p, m = unit_rows(B).requires_grad_(True), unit_rows(C), unit_rows(M)
    index = C + M - 1 - torch.arange(B * 3, device=DEV).view(B, 3) * 100
    score = torch.randn(B, 3, generator=g, device=DEV)
    loss, _ = call(q, p, m, torch.tensor(temp, device=DEV), index, score, 0.5)
    dq, = torch.autograd.grad(loss, q)
    cand = torch.cat((p, m)).double()
    z = q.detach().double() @ cand.T / float(torch.tensor(temp))
    logt = torch.log_softmax(score.double() / 0.5, dim=1)
    want = (logt.exp() * (logt - z.gather(1, index))).sum(1) + torch.logsumexp(z, 1)
    assert abs(float(loss.detach()) - float(want.mean())) <= 2.4e-4
    gm = torch.softmax(z, 1).scatter_add(1, index, -logt.exp()) / B / float(torch.tensor(temp))
    ref = gm @ cand
    lim = 2.4e-4 * 2 / 0.07 / B + (2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -20) * ref.norm(dim=1)
    assert bool(((dq.double() - ref).norm(dim=1) <= lim).all())
