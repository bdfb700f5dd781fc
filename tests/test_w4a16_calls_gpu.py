"""Calls of the weight-only operators that their documentation allows: long rows, graphs beside larger calls, arguments that do not belong together."""
import pytest
import torch

from test_w4a16_gpu import _layer
from w4a16_ref import make_weight, make_x, values

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# Two tokens whose rows fill the shared memory of all blocks of a cluster, singly or together, and are too long for it; a row has 64 numbers in it, so that sums are exact.
@pytest.mark.parametrize("N,K", [(64, 26640), (64, 104464), (64, 208912), (40, 300000), (64, 417792), (64, 524304), (2048, 65552), (4096, 143376)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_two_tokens_with_long_rows(N, K, dtype):
    from dgx_vllm_b200.weight_only import last_w4a16_status, pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, N, K, 5)
    g = torch.ones(1, device="cuda")
    x = torch.zeros(2, K, dtype=dtype, device="cuda")
    at = torch.randint(0, K, (64,), generator=torch.Generator().manual_seed(1)).cuda()
    at[0], at[1] = K - 1, 0
    x[:, at] = make_x(2, 64, 3, dtype)
    w = pack_nvfp4_weight(codes[0], block[0], g)
    want = x[:, at.unique()].double() @ values(codes, block, g.reshape(1, 1))[0][:, at.unique()].T
    for out_dtype in (F32, dtype):
        assert torch.equal(w4a16_linear(x, w, out_dtype=out_dtype), want.to(out_dtype))
    assert last_w4a16_status() == 0
