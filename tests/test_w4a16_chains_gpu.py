"""f32 results of the weight-only operators keep f32's precision however long their sums are."""
import pytest
import torch

from test_w4a16_gpu import _linear
from w4a16_ref import make_weight, make_x, values

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# A matrix instruction (16 of k) truncates its sum, by half a place (2^-24 to 2^-23 of the sum) on the average and always towards zero.  A sum of n of them that grows as
# its root, as sums of independent terms do, is then off by sum_i 0.5 * 2^-23.5 * sqrt(i / n) = 2.8e-8 n of itself at most; a chain has 72 instructions at most (nine units of 128;
# six in the kernels of few tokens), 20e-7.  The additions of chains round: 2^-24 for each of up to 19, sqrt(19) of it together, 2.6e-7, and so does the factor.
# Sums that are not taken apart have 200 to 900 instructions in these cases: 33e-7 to 130e-7 as measured (1.5e-8 for each).
CHAINED = 23e-7


@pytest.mark.parametrize("M,N,K,dtype", [(3, 900, 14336, BF16), (4, 8192, 14336, BF16), (8, 40, 49152, F16), (12, 700, 14336, F16), (16, 60, 24576, BF16), (32, 4096, 14336, BF16),
                                         (150, 1024, 14336, BF16), (400, 8192, 14336, F16), (700, 300, 4912, BF16)])
def test_linear_sums_are_taken_apart(M, N, K, dtype):
    y, ref, _ = _linear(M, N, K, dtype, F32, exact=False, g=3e-4)
    assert float((y.double() - ref).norm()) <= CHAINED * float(ref.norm())


# The layer's chains have 48 instructions, 13.4e-7, and their additions; where H is long, gate and up are off by that each, and the gate's goes into the value by
# |g silu'(g) / silu(g)| <= 1 + |g| times, |g| below 1 nearly always: 2.2 times in all.  The other sum is short, SiLU and the factors round: 5e-7.
LAYER = 16e-7


@pytest.mark.parametrize("M,E,H,I,dtype", [(1, 1, 49152, 16, BF16), (3, 2, 40000, 48, BF16), (2, 1, 49152, 32, F16), (30, 2, 24576, 16, F16),
                                           (2, 2, 32, 49152, BF16), (12, 1, 64, 40000, F16), (40, 2, 32, 24576, BF16), (5, 3, 64, 16400, BF16)])
def test_layer_sums_are_taken_apart(M, E, H, I, dtype):
    from dgx_vllm_b200.weight_only import W4A16MoE, pack_nvfp4_weight
    c13, b13 = make_weight(E, 2 * I, H, 1, exact=False)
    c2, b2 = make_weight(E, H, I, 2, exact=False)
    W = values(c13[:, :64], b13[:, :64], torch.ones(1, 1, device="cuda"))
    g13 = torch.full((E,), 0.3 / float(W.pow(2).sum(2).mean().sqrt()), device="cuda")
    g2 = torch.full((E,), 1e-4, device="cuda")
    layer = W4A16MoE(pack_nvfp4_weight(c13, b13, g13, gated=True), pack_nvfp4_weight(c2, b2, g2))
    x = make_x(M, H, 3, dtype, exact=False)
    ids = (torch.arange(M, dtype=torch.int32, device="cuda") % E)[:, None].contiguous()
    weights = torch.full((M, 1), 0.75, device="cuda")
    out = layer(x, weights, ids, False, torch.empty(M, H, device="cuda"))
    ref = torch.zeros(M, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        mine = (ids[:, 0] == e).nonzero()[:, 0]
        h = x[mine].double() @ values(c13[e:e + 1], b13[e:e + 1], g13[e].reshape(1, 1))[0].T
        ref[mine] = 0.75 * (h[:, :I] * torch.sigmoid(h[:, :I]) * h[:, I:]) @ values(c2[e:e + 1], b2[e:e + 1], g2[e].reshape(1, 1))[0].T
    assert float((out - ref).norm()) <= ((2.2 if H > I else 1) * LAYER + 5e-7) * float(ref.norm())
