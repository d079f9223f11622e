"""Refusals of the distillation loss, without a GPU, and its oracle against differences and autograd."""
import pytest
import torch

from oracle.distill_oracle import distill_ref

F32, BF16, I8 = 2, 0, 1
OK = 4096


def lib():
    from vllm_amd import _lib
    return _lib.load()


def fwd(dtype=F32, q=OK, p=OK, memory=None, temp=OK, idx=OK, score=OK, tt=1.0, B=4, C=8, M=0, d=16, k=3, loss=OK, agree=OK, ws=OK, ws_bytes=0):
    return lib().abc_distill_fwd(dtype, q, p, memory, temp, idx, score, tt, B, C, M, d, k, loss, agree, ws, ws_bytes, None)


def bwd(dtype=F32, q=OK, p=OK, memory=None, temp=OK, go=OK, B=4, C=8, M=0, d=16, k=3, dq=OK, dp=OK, dt=OK, fws=OK, fws_bytes=0, ws=OK, ws_bytes=0):
    return lib().abc_distill_bwd(dtype, q, p, memory, temp, go, B, C, M, d, k, dq, dp, dt, fws, fws_bytes, ws, ws_bytes, None)


SIZES = [dict(dtype=I8), dict(dtype=7), dict(B=0), dict(B=65536), dict(C=0), dict(M=-1), dict(M=1 << 31), dict(d=0), dict(d=12), dict(d=65544),
         dict(k=0), dict(k=1025), dict(C=1 << 30), dict(B=1, C=1, M=1 << 29), dict(B=65, C=1 << 29), dict(C=1 << 25, d=65536)]


@pytest.mark.parametrize("bad", SIZES)
def test_sizes_are_refused(bad):
    assert fwd(**bad) == -1 and lib().abc_last_error()
    assert bwd(**bad) == -1
    a = {**dict(dtype=F32, B=4, C=8, M=0, d=16, k=3), **bad}
    args = [a[x] for x in ("dtype", "B", "C", "M", "d", "k")]
    assert lib().abc_distill_workspace_bytes(*args) == 0 and lib().abc_distill_bwd_workspace_bytes(*args) == 0


@pytest.mark.parametrize("bad", [dict(q=None), dict(p=None), dict(M=5), dict(temp=None), dict(idx=None), dict(score=None), dict(loss=None),
                                 dict(agree=None), dict(q=OK + 8), dict(p=OK + 4), dict(tt=0.0), dict(tt=-1.0), dict(tt=float("nan"))])
def test_forward_refuses(bad):
    assert fwd(**bad, ws_bytes=1 << 30) == -1 and lib().abc_last_error()


def test_the_largest_sizes_that_are_taken():
    assert lib().abc_distill_workspace_bytes(F32, 1, 1, (1 << 29) - 1, 8, 3) > 1 << 31 and lib().abc_distill_workspace_bytes(F32, 65535, 8, 0, 65536, 1024) > 0


def test_workspaces():
    need = lib().abc_distill_workspace_bytes(F32, 4, 8, 0, 16, 3)
    back = lib().abc_distill_bwd_workspace_bytes(F32, 4, 8, 0, 16, 3)
    assert need > 0 and back > 0
    assert fwd(ws_bytes=need - 1) == -2 and b"workspace too small" in lib().abc_last_error()
    assert fwd(ws=None, ws_bytes=need) == -2 and fwd(ws=OK + 4, ws_bytes=need) == -1
    assert bwd(fws_bytes=need - 1, ws_bytes=back) == -2 and bwd(fws_bytes=need, ws_bytes=0) == -2
    assert bwd(fws_bytes=need, ws_bytes=back, fws=None) == -1 and bwd(fws_bytes=need, ws_bytes=back, go=None) == -1
    assert bwd(fws_bytes=need, ws_bytes=back, dq=OK + 2) == -1
    assert bwd(fws_bytes=need, ws_bytes=back, dq=None, dp=None, dt=None) == 0       # nothing asked for


def test_product_path_refuses():
    from vllm_amd import loss
    from vllm_amd._lib import AbcError
    with pytest.raises(AbcError, match="GPU only"):
        loss.compute_distillation_loss(torch.zeros(4, 8), torch.zeros(4, 8), loss.Temperature(), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))


def test_oracle_gradients_are_autograds():
    g = torch.Generator().manual_seed(0)
    q, c = torch.randn(6, 5, generator=g).double(), torch.randn(11, 5, generator=g).double()
    index = torch.randint(11, (6, 4), generator=g)
    score = torch.rand(6, 4, generator=g)
    index[1, 2], score[2, 0] = -1, float("-inf")
    index[3] = -1
    temp = torch.tensor(0.3, dtype=torch.float64, requires_grad=True)
    q.requires_grad_(True)
    c.requires_grad_(True)
    z = torch.log_softmax(q @ c.t() / temp, 1)
    total = 0.0
    for b in range(6):
        on = [(int(index[b, i]), float(score[b, i])) for i in range(4) if index[b, i] >= 0 and score[b, i] > -1e30]
        if on:
            t = torch.softmax(torch.tensor([v / 0.2 for _, v in on], dtype=torch.float64), 0)
            total = total + sum(t[i] * (t[i].log() - z[b, j]) for i, (j, _) in enumerate(on))
    total = total / 5
    want = torch.autograd.grad(total, (q, c, temp))
    r = distill_ref(q.detach(), c.detach(), 0.3, index, score, 0.2, 7)
    assert abs(float(total.detach()) - float(r["loss"])) <= 1e-12
    for a, b in zip(want, (r["dq"], r["dp"], r["dtemp"])):
        assert float((a[:7] if a.shape == c.shape else a).sub(b).abs().max()) <= 1e-12
