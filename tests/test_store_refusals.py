"""Refusals of the embedding store, without a GPU: the library's checks of arguments come before anything is launched."""
import pytest
import torch

F32, BF16, I8 = 2, 0, 1
OK = 4096                                                          # an aligned address that no refused call reads


def lib():
    from vllm_amd import _lib
    return _lib.load()


def write(x_dtype=F32, x=OK, ldx=128, slots=OK, first=0, n=4, dim=128, data=OK, scale=OK, capacity=10, group=64, ws=None, ws_bytes=0):
    return lib().abc_store_write(x_dtype, x, ldx, slots, first, n, dim, data, scale, capacity, group, ws, ws_bytes, None)


def read(index=OK, first=0, n=4, data=OK, scale=OK, capacity=10, dim=128, group=64, out_dtype=F32, out=OK, ldo=128):
    return lib().abc_store_read(index, first, n, data, scale, capacity, dim, group, out_dtype, out, ldo, None)


def scores(q_dtype=F32, q=OK, ldq=128, nq=2, data=OK, scale=OK, rows=10, dim=128, group=64, out=OK, ldo=10):
    return lib().abc_store_scores(q_dtype, q, ldq, nq, data, scale, rows, dim, group, out, ldo, None)


@pytest.mark.parametrize("bad", [dict(x_dtype=I8), dict(x=None), dict(data=None), dict(scale=None), dict(ldx=127), dict(n=-1), dict(dim=0),
                                 dict(dim=8193), dict(group=16), dict(group=-64), dict(capacity=-1), dict(capacity=1 << 31),
                                 dict(data=OK + 8), dict(scale=OK + 1), dict(slots=None, first=10), dict(slots=None, first=-1),
                                 dict(slots=None, n=11), dict(group=0, scale=OK + 2)])
def test_write_refuses(bad):
    assert write(**bad) == -1 and lib().abc_last_error()


def test_write_workspace():
    assert lib().abc_store_write_workspace_bytes(2048, 10) == 0 and lib().abc_store_write_workspace_bytes(2049, 10) == 40
    assert write(n=2049) == -2 and b"workspace too small" in lib().abc_last_error()
    assert write(n=2049, ws=OK, ws_bytes=39) == -2
    assert write(n=0) == 0 and read(n=0) == 0 and scores(nq=0) == 0 and scores(rows=0) == 0


@pytest.mark.parametrize("bad", [dict(out_dtype=I8), dict(out=None), dict(data=None), dict(scale=None), dict(ldo=127), dict(n=-1),
                                 dict(dim=0), dict(dim=8193), dict(group=48), dict(data=OK + 4), dict(index=None, first=7),
                                 dict(index=None, first=-1)])
def test_read_refuses(bad):
    assert read(**bad) == -1 and lib().abc_last_error()


@pytest.mark.parametrize("bad", [dict(q_dtype=I8), dict(q=None), dict(data=None), dict(scale=None), dict(out=None), dict(ldq=100),
                                 dict(ldo=9), dict(nq=-1), dict(group=0), dict(group=256), dict(scale=OK + 2), dict(data=OK + 8)])
def test_scores_refuses(bad):
    assert scores(**bad) == -1 and lib().abc_last_error()


def test_product_path_refuses_cpu_tensors_and_bad_shapes():
    from vllm_amd import kernels, search
    from vllm_amd._lib import AbcError
    data, scale = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.bfloat16)
    x = torch.zeros(2, 128)
    for call in (lambda: kernels.store_write(x, None, data, scale), lambda: kernels.store_read(None, data, scale, 128),
                 lambda: kernels.store_scores(x, data, scale)):
        with pytest.raises(AbcError, match="GPU only"):
            call()
    for kw in (dict(form="int4"), dict(group=48), dict(capacity=0), dict(dim=0), dict(dim=8193), dict(capacity=1 << 31)):
        with pytest.raises(AbcError):
            search.EmbeddingStore(**{**dict(capacity=4, dim=64, device="cuda:0"), **kw})


def test_oracle_layout():
    """The packed form and the values are two computations of one definition."""
    from oracle import store_oracle
    x = torch.randn(5, 300, generator=torch.Generator().manual_seed(0))
    x[1, 40] = 0.0
    for group in (32, 64, 128):
        data, scale = store_oracle.store_pack(x, group)
        table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
        out = torch.zeros(5, 384, dtype=torch.float64)
        for k in range(384):
            m, c, j = k % 128 // 32, k % 32 // 8, k % 8
            nib = 32 * c + 8 * m + j
            code = (data[:, k // 128 * 64 + nib // 2].int() >> (4 * (nib % 2))) & 15
            out[:, k] = table[code & 7] * torch.where(code > 7, -1.0, 1.0) * scale[:, k // group].double()
        assert torch.equal(out[:, :300], store_oracle.store_values(x, group)) and bool((out[:, 300:] == 0).all())
