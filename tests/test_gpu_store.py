"""The store of embeddings held in 4 or 8 bits on the GPU, against its definition in 64 bits on the CPU.

What is held is compared bit for bit: the scale and the code of every value follow from comparisons that are exact.  What is read back
is code * scale, exact in fp32 for fp4 (2 + 8 significant bits), one rounding for i8 (2^-24) and one more to bf16 (2^-8)."""
import pytest
import torch

import oracle
from oracle import store_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows(n, d, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g) * torch.exp(torch.randn(n, 1, generator=g))
    return x.to(dtype)


def held(data, scale):
    return data.cpu(), scale.cpu()


def same_bits(got, want):
    view = {torch.bfloat16: torch.int16, torch.float32: torch.int32}
    for a, b in zip(got, want):
        a, b = a.cpu(), b.cpu()
        if a.dtype in view:
            nan = torch.isnan(a)
            assert torch.equal(nan, torch.isnan(b))
            a, b = a.masked_fill(nan, 0).view(view[a.dtype]), b.masked_fill(nan, 0).view(view[b.dtype])
        assert torch.equal(a, b)


def empty(capacity, dim, group):
    from vllm_amd import search
    s = search.EmbeddingStore(capacity, dim, "fp4" if group else "i8", group or 128, DEV)
    return s


@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,dim", [(1, 1), (3, 7), (5, 127), (4, 128), (17, 129), (9, 900), (33, 1024), (2, 4096), (3, 8192), (70, 2049)])
def test_write_and_read_back(n, dim, group, dtype):
    s = empty(n + 5, dim, group)
    x = rows(n, dim, 7 * n + dim, dtype)
    slots = torch.randperm(n + 5, generator=torch.Generator().manual_seed(dim))[:n]
    s.write(x.to(DEV), slots.to(DEV))
    data, scale = store_oracle.store_pack(x, group)
    same_bits((s.data[slots], s.scale[slots]), (data, scale))
    rest = torch.ones(n + 5, dtype=torch.bool)
    rest[slots] = False
    assert int(s.data[rest.to(DEV)].abs().sum() if group == 0 else s.data[rest.to(DEV)].sum()) == 0     # the other slots are as they were
    want = torch.zeros(n + 5, dim, dtype=torch.float64)
    want[slots] = store_oracle.store_values(x, group)
    for out in (torch.float32, torch.bfloat16):
        got = s.read(dtype=out).cpu()
        step = 2.0 ** -24 if out == torch.float32 else 2.0 ** -8 + 2.0 ** -24
        assert bool(((got.double() - want).abs() <= step * want.abs()).all())


def test_i8_is_the_search_kernels_form():
    from vllm_amd import search
    x = rows(300, 896, 3)
    s = empty(300, 896, 0)
    s.append(x.to(DEV))
    e = search.Embeddings(x.to(DEV), "i8")
    assert torch.equal(s.data, e.data) and torch.equal(s.scale, e.scale)
    q = search.Embeddings(x[:20].to(DEV), "i8")
    a, b = search.topk(q, s.embeddings(), 10), search.topk(q, e, 10)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_values_on_the_borders():
    """Midpoints between the levels (ties to the even code), zeros of either sign, the smallest and the largest groups."""
    d = 128
    x = torch.zeros(8, d)
    mid = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    x[0, :9], x[0, 9:18] = mid, -mid
    x[1, :9] = torch.nextafter(mid, torch.tensor(10.0))
    x[1, 0] = 6.0
    x[2, :9] = torch.nextafter(mid, torch.tensor(-10.0))
    x[2, 20] = 6.0
    x[3, :9] = mid * 2.0 ** -120                                   # the floor of the scale
    x[4, 3] = 2.0 ** -149
    x[5] = -0.0
    x[6, :9] = mid * 2.0 ** 124
    x[6, 30] = torch.finfo(torch.float32).max
    x[7, :9] = mid * 0.0371
    for group in (32, 64, 128, 0):
        s = empty(8, d, group)
        s.append(x.to(DEV))
        same_bits((s.data, s.scale), store_oracle.store_pack(x, group))


def test_groups_that_are_not_finite_read_as_nan():
    x = rows(6, 256, 5)
    x[1, 3], x[2, 200], x[3, 40] = float("inf"), float("-inf"), float("nan")
    for group in (0, 32, 128):
        s = empty(6, 256, group)
        s.append(x.to(DEV))
        want = store_oracle.store_values(x, group)
        got = s.read().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert bool(((got.double() - want)[ok].abs() <= 2.0 ** -24 * want[ok].abs()).all())


@pytest.mark.parametrize("n", [2, 300, 1025, 2048, 2049, 5000])
@pytest.mark.parametrize("group,dim", [(0, 96), (64, 96), (128, 2048), (0, 2048)])
def test_the_last_of_rows_that_name_one_slot_stays(n, group, dim):
    cap = 37
    x = rows(n, dim, n)
    slots = torch.randint(-3, cap + 3, (n,), generator=torch.Generator().manual_seed(n))      # some outside: dropped
    s = empty(cap, dim, group)
    s.write(x.to(DEV), slots.to(DEV))
    want = torch.zeros(cap, dim, dtype=torch.float64)
    values = store_oracle.store_values(x, group)
    for i in range(n):
        if 0 <= slots[i] < cap:
            want[slots[i]] = values[i]
    assert bool(((s.read().cpu().double() - want).abs() <= 2.0 ** -24 * want.abs()).all())


def test_append_goes_round():
    s = empty(10, 64, 32)
    x = rows(24, 64, 1)
    v = store_oracle.store_values(x, 32)
    assert s.append(x[:7].to(DEV)) == 0
    assert s.append(x[7:14].to(DEV)) == 7                          # slots 7, 8, 9, 0, 1, 2, 3
    got = s.read().cpu().double()
    assert torch.equal(got[7:], v[7:10]) and torch.equal(got[:4], v[10:14]) and torch.equal(got[4:7], v[4:7])
    assert s.append(x[14:24].to(DEV)) == 4 and s.append(x[:0].to(DEV)) == 4
    assert torch.equal(s.read().cpu().double()[4:], v[14:20])


@pytest.mark.parametrize("group", [0, 32, 128])
def test_read_by_index(group):
    dim, cap = 515, 50
    s = empty(cap, dim, group)
    x = rows(cap, dim, 9)
    s.append(x.to(DEV))
    v = store_oracle.store_values(x, group)
    index = torch.tensor([[0, 49, -1, 7], [7, 7, 50, -9], [1, 2, 3, 1 << 40]])
    got = s.read(index.to(DEV)).cpu()
    assert got.shape == (3, 4, dim)
    for i, j in ((a, b) for a in range(3) for b in range(4)):
        k = int(index[i, j])
        if k < 0:
            assert torch.equal(got[i, j], torch.zeros(dim))
        elif k >= cap:
            assert bool(torch.isnan(got[i, j]).all())
        else:
            assert bool(((got[i, j].double() - v[k]).abs() <= 2.0 ** -24 * v[k].abs()).all())
    assert torch.equal(s.read(index.int().to(DEV)[:2]).cpu().nan_to_num(7.0), got[:2].nan_to_num(7.0))
    assert s.read(torch.empty(0, 3, dtype=torch.int64, device=DEV)).shape == (0, 3, dim)
    # into the middle of a larger buffer, rows apart from each other; what lies around stays
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.full((20, dim + 9), 5.0, device=DEV, dtype=dt)
        s.read(torch.arange(12, device=DEV), out=buf[3:15, 4:4 + dim])
        assert torch.equal(buf[3:15, 4:4 + dim], s.read(torch.arange(12, device=DEV), dtype=dt))
        buf[3:15, 4:4 + dim] = 5.0
        assert bool((buf == 5.0).all())
    # a view of some slots is a store of its own
    part = s.rows(11, 32)
    assert torch.equal(part.read(), s.read(torch.arange(11, 32, device=DEV)))
    part.write(x[:1].to(DEV), torch.tensor([3], device=DEV))
    assert torch.equal(s.read(torch.tensor([14], device=DEV)), s.read(torch.tensor([0], device=DEV)))


def test_strided_and_unaligned_rows():
    big = rows(40, 1111, 4)
    for dt in (torch.float32, torch.bfloat16):
        x = big.to(dt)
        for view in (x[:, 3:900], x[::3, 1:130], x[:, ::2], x[4:5, 5:]):
            for group in (0, 64):
                s = empty(view.shape[0], view.shape[1], group)
                base = x.to(DEV)
                dview = torch.as_strided(base, view.shape, view.stride(), view.storage_offset())
                s.append(dview)
                same_bits((s.data, s.scale), store_oracle.store_pack(view, group))


# ---- scores ------------------------------------------------------------------------------------------------------------------
def check_scores(q, x, group, s=None):
    """|error| <= (depth + 3) 2^-24 sum |q_k v_k|: `depth` fp32 additions at most meet a product (a tree or a chain of them), a
    product of three bf16 parts is exact up to 2^-24, a group's scaling and the parts' sum round once each.  A chain over one group
    and one over the groups is the longest: 128 / 32 + 8 MFMA steps of 32 products in a wave, counted as the whole row below."""
    if s is None:
        s = empty(x.shape[0], x.shape[1], group)
        s.append(x.to(DEV))
    got = s.scores(q.to(DEV)).cpu().double()
    v = store_oracle.store_values(x, group)
    want = q.double() @ v.t()
    room = q.double().abs() @ v.abs().t()
    depth = x.shape[1] + 8
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= (depth + 3) * 2.0 ** -24 * room).all()), float(((got - want).abs() / room.clamp(min=1e-300)).max())
    # and in the mean as near as rounding at random brings it
    rel = float((got - want).norm() / want.norm().clamp(min=1e-300))
    assert rel <= 2e-6, rel
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("nq,n,dim", [(1, 1, 1), (1, 17, 64), (2, 16, 128), (5, 33, 200), (4, 300, 896), (13, 1000, 1000),
                                      (16, 257, 4096), (1, 5000, 3584), (3, 129, 8192), (1, 70_001, 256)])
def test_scores(nq, n, dim, group, dtype):
    check_scores(rows(nq, dim, nq + n, dtype), rows(n, dim, n + dim), group)


@pytest.mark.parametrize("dtype,nq", [(torch.float32, 17), (torch.float32, 50), (torch.bfloat16, 40), (torch.bfloat16, 64), (torch.bfloat16, 65)])
def test_scores_of_more_queries_than_a_pass_takes(dtype, nq):
    check_scores(rows(nq, 520, nq, dtype), rows(500, 520, 1), 64)
    check_scores(rows(nq, 4096, nq, dtype), rows(40, 4096, 1), 128)


def test_scores_carry_infinities_and_nan():
    x = 1.0 + torch.rand(40, 256, generator=torch.Generator().manual_seed(1))      # within a factor of two: no code is zero
    q = rows(4, 256, 2)
    q[1, 5], q[2, 9], q[3, 250] = float("inf"), float("nan"), float("-inf")
    s = empty(40, 256, 128)
    s.append(x.to(DEV))
    v = store_oracle.store_values(x, 128)
    assert bool((v != 0).all())
    for dt in (torch.float32, torch.bfloat16):
        got = s.scores(q.to(dt).to(DEV)).cpu()
        want = q.to(dt).double() @ v.t()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
        assert torch.equal(got[1], torch.full((40,), float("inf"))) and torch.equal(got[3], torch.full((40,), float("-inf")))
    y = x.clone()
    y[7, 100] = float("nan")                                       # a row that is not finite is NaN for every query, the others are untouched
    s.write(y[7:8].to(DEV), torch.tensor([7], device=DEV))
    got = s.scores(q[:1].to(DEV)).cpu()[0]
    assert torch.equal(torch.isnan(got), torch.arange(40) == 7)


def test_scores_same_bits_again_and_on_another_stream():
    x, q = rows(3000, 1024, 1).to(DEV), rows(3, 1024, 2).to(DEV)
    s = empty(3000, 1024, 64)
    s.append(x)
    a = s.scores(q)
    torch.cuda.synchronize()
    st = torch.cuda.Stream(DEV)
    with torch.cuda.stream(st):
        b = s.scores(q)
        r = s.read(torch.arange(100, device=DEV))
    st.synchronize()
    assert torch.equal(a, b) and torch.equal(r, s.read(torch.arange(100, device=DEV)))


def test_a_store_beyond_32_bit_offsets():
    """Rows past 4 GiB of codes: 1.1 M rows of 8192 values in 4 bits (4.5 GB)."""
    n, dim = 1_100_000, 8192
    s = empty(n, dim, 128)
    x = rows(3, dim, 8).to(DEV)
    at = torch.tensor([0, n // 2, n - 1], device=DEV)
    s.write(x, at)
    v = store_oracle.store_values(x.cpu(), 128)
    assert torch.equal(s.read(at).cpu().double(), v)
    q = rows(1, dim, 9)
    got = s.scores(q.to(DEV))[0]
    want = (q.double() @ v.t())[0]
    assert bool(((got[at].cpu().double() - want).abs() <= 1e-5 * want.abs().max()).all())
    assert int((got != 0).sum()) == 3


def test_in_a_captured_graph():
    """Write, read and scores in one graph, replayed on new rows, eager work between the replays."""
    s = empty(64, 384, 32)
    x, slots, q = rows(2500, 384, 0).to(DEV), torch.zeros(2500, dtype=torch.int64, device=DEV), rows(2, 384, 3).to(DEV)
    other = empty(64, 384, 32)
    st = torch.cuda.Stream(DEV)

    def step(t):
        t.write(x, slots)
        return t.read(slots[:70]), t.scores(q)

    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(s)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(s)
    for i in range(3):
        x.copy_(rows(2500, 384, 20 + i))
        slots.copy_(torch.randint(0, 64, (2500,), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        want = step(other)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(s.data, other.data)
    from vllm_amd._lib import AbcError
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        with pytest.raises(AbcError, match="captured"):
            s.append(x[:2])
        x[:2].add_(0)                                              # a capture of nothing is an error of its own


def test_more_rows_than_a_launch_takes():
    """2^28 rows of 16 threads are 2^32 threads."""
    n = (1 << 28) + 37
    s = empty(n + 3, 1, 128)
    values = (torch.arange(13) - 6).to(torch.bfloat16)[:, None]
    at = torch.arange(n, device=DEV) % 13
    s.append(values.to(DEV)[at])
    got = s.read()
    want = store_oracle.store_values(values, 128).float().to(DEV)
    assert torch.equal(got[:n], want[at]) and not got[n:].any()


def test_rows_past_4_gib():
    """4-bit rows of 2 KB from slot 2^21 on, 8-bit rows of 4 KB from 2^20 on: written, read and scored there."""
    x, q = rows(5, 4096, 1), rows(3, 4096, 2)
    for group, slots in ((128, torch.tensor([3, (1 << 21) - 1, 1 << 21, (1 << 21) + 9, 2_200_000])),
                         (0, torch.tensor([0, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, 1_200_001]))):
        big, small = empty(int(slots[-1]) + 1, 4096, group), empty(5, 4096, group)
        big.write(x.to(DEV), slots.to(DEV))
        small.write(x.to(DEV), torch.arange(5, device=DEV))
        same_bits((big.read(slots.to(DEV)),), (small.read(),))
        if group:
            got = big.scores(q.to(DEV))
            want = torch.zeros_like(got)
            want[:, slots.to(DEV)] = small.scores(q.to(DEV))
            # the waves that share a small store's rows add up in another order: 32 pieces' sums, a rounding each
            size = q.abs() @ small.read().cpu().abs().T
            assert bool(((got - want)[:, slots.to(DEV)].cpu().abs() <= 64 * 2.0 ** -24 * size).all())
            want[:, slots.to(DEV)] = got[:, slots.to(DEV)]
            assert torch.equal(got, want)


@pytest.mark.parametrize("group", [0, 128])
def test_what_is_written_is_known_to_have_changed(group):
    """A graph that saved a buffer or a store's scale refuses its backward after the kernel wrote there; a corpus kept by version is new."""
    from vllm_amd import search
    s = empty(40, 128, group)
    s.write(rows(40, 128, 0).to(DEV), torch.arange(40, device=DEV))
    buf, w = torch.empty(40, 128, device=DEV), torch.ones(40, 128, device=DEV, requires_grad=True)
    s.read(out=buf)
    loss = (w * buf).sum()
    s.read(out=buf[:7], index=torch.arange(7, device=DEV))
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    loss = (torch.ones_like(s.scale, dtype=torch.float32, requires_grad=True) * s.scale).sum()
    s.write(rows(1, 128, 1).to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    q = rows(3, 128, 5).to(DEV)

    def negatives(c):
        found = {}
        for i in range(3):
            search.negatives_for_sample(i, found, q, c, top=5)
        return found

    s.read(out=buf)
    a = negatives(buf)
    s.write(rows(40, 128, 9).to(DEV), torch.arange(40, device=DEV))
    s.read(out=buf)
    b, want = negatives(buf), negatives(buf.clone())
    search.release_resident()
    assert b == want and a != b
