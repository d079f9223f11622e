"""abc_cast_bf16 at the sizes where its workgroups' pieces end, from and into addresses of any multiple of the element."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("n", [1, 3, 255, 2047, 2048, 2049, 4095, 4096 + 5, 100_003, (1 << 22) + 2047])
@pytest.mark.parametrize("skip_x,skip_o", [(0, 0), (1, 0), (0, 1), (3, 5)])
def test_cast_of_any_length_and_alignment(n, skip_x, skip_o):
    from vllm_amd import _lib
    lib = _lib.load()
    x = torch.randn(n + skip_x + 8, generator=torch.Generator().manual_seed(n)).to(DEV)
    x[skip_x] = float("nan")
    x[skip_x + n - 1] = 3.4e38                                      # rounds up to infinity
    out = torch.full((n + skip_o + 8,), 7.0, dtype=torch.bfloat16, device=DEV)
    _lib.check(lib.abc_cast_bf16(x.data_ptr() + 4 * skip_x, n, out.data_ptr() + 2 * skip_o, torch.cuda.current_stream().cuda_stream), "cast")
    got, want = out[skip_o:skip_o + n], x[skip_x:skip_x + n].bfloat16()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(1.0), want.nan_to_num(1.0))
    assert bool((out[:skip_o] == 7.0).all()) and bool((out[skip_o + n:] == 7.0).all())      # nothing beside it is written
