"""Weight-only operators without a GPU: refusals before anything is queued, sizes, and the plain forms they are tested against."""
import pytest
import torch

from test_host_cpu import INVALID, NOT_SUPPORTED, _refused_unqueued
from w4a16_ref import make_weight, values

ALLOC = 3
P = 0x100000                                                      # an address no step ever reads


@pytest.mark.parametrize("bad,status", [
    (dict(x=0), INVALID), (dict(x=P + 8), INVALID), (dict(x_dtype=2), INVALID), (dict(ldx=60), INVALID), (dict(ldx=48), INVALID), (dict(packed=0), INVALID),
    (dict(packed=P + 8), INVALID), (dict(g=0), INVALID), (dict(bias=P, bias_dtype=7), INVALID), (dict(out=0), INVALID), (dict(out_dtype=3), INVALID),
    (dict(M=-1), INVALID), (dict(N=0), INVALID), (dict(K=72), INVALID), (dict(K=0), INVALID), (dict(M=1 << 33), NOT_SUPPORTED), (dict(N=1 << 33), NOT_SUPPORTED),
    (dict(status=0), INVALID),
])
def test_refused_linear_queues_nothing(bad, status):
    a = dict(x=P, x_dtype=1, ldx=64, packed=P, g=P, bias=0, bias_dtype=0, out=P, out_dtype=1, M=2, N=128, K=64, status=P, stream=0)
    a.update(bad)
    assert _refused_unqueued(lambda L: L.b200fp4_w4a16_linear(*a.values())) == status


@pytest.mark.parametrize("bad,status", [
    (dict(hidden=0), INVALID), (dict(hidden=P + 8), INVALID), (dict(h_dtype=2), INVALID), (dict(weights=0), INVALID), (dict(ids=0), INVALID),
    (dict(emap=P), INVALID), (dict(w13=P + 4), INVALID), (dict(w13_g=0), INVALID), (dict(w2=0), INVALID), (dict(w2_g=0), INVALID), (dict(out=P + 4), INVALID),
    (dict(out_dtype=5), INVALID), (dict(M=-2), INVALID), (dict(topk=0), INVALID), (dict(topk=2049), NOT_SUPPORTED), (dict(H=72), INVALID), (dict(I=24), INVALID),
    (dict(E=0), INVALID), (dict(E=4097), NOT_SUPPORTED), (dict(flags=2), INVALID), (dict(status=0), INVALID), (dict(workspace=0), ALLOC), (dict(bytes=300), ALLOC),
    (dict(M=1 << 31, topk=2), NOT_SUPPORTED),
])
def test_refused_layer_queues_nothing(bad, status):
    a = dict(hidden=P, h_dtype=1, weights=P, ids=P, emap=0, global_E=0, w13=P, w13_g=P, w2=P, w2_g=P, out=P, out_dtype=1, M=2, topk=2, H=64, I=32, E=4,
             flags=0, status=P, workspace=P, bytes=1 << 60, stream=0)
    a.update(bad)
    assert _refused_unqueued(lambda L: L.b200fp4_w4a16_moe(*a.values())) == status


@pytest.mark.parametrize("E,N,K,gated,size", [
    (1, 1, 16, 0, 2304 + 4), (1, 32, 128, 0, 2304 + 4), (1, 33, 144, 0, 4 * 2304 + 4), (3, 32, 256, 1, 6 * 2304 + 24), (2, 34, 128, 1, 4 * 2304 + 16), (1, 16, 24, 0, 0),
    (1, 15, 16, 1, 0), (0, 16, 16, 0, 0), (512, 1024, 2048, 1, 512 * 32 * 16 * 2304 + 4096),
])
def test_packed_bytes(E, N, K, gated, size):
    from dgx_vllm_b200 import _lib
    L = _lib.lib()
    assert L.b200fp4_w4a16_packed_bytes(E, N, K, gated) == size
    if size == 0:
        assert _refused_unqueued(lambda L: L.b200fp4_w4a16_pack(P, P, E, N, K, gated, P, 0)) == INVALID


@pytest.mark.parametrize("bad", [dict(codes=0), dict(codes=P + 4), dict(scales=0), dict(packed=0), dict(packed=P + 8), dict(N=1 << 32)])
def test_refused_packing_queues_nothing(bad):
    a = dict(codes=P, scales=P, E=1, N=32, K=64, gated=0, packed=P, stream=0)
    a.update(bad)
    assert _refused_unqueued(lambda L: L.b200fp4_w4a16_pack(*a.values())) == INVALID


def test_workspace_covers_a_turn_of_the_layer():
    from dgx_vllm_b200 import _lib
    L = _lib.lib()
    size = L.b200fp4_w4a16_moe_workspace_bytes
    assert size(32, 10, 2048, 512) >= 320 * (2 * 512 * 2 + 2048 * 4)
    assert size(1 << 20, 10, 2048, 512) == size(204, 10, 2048, 512)               # more pairs are done in turns


def test_no_cpu_path():
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight
    codes, block = make_weight(1, 16, 32, 0, device="cpu")
    with pytest.raises(RuntimeError):
        pack_nvfp4_weight(codes[0], block[0], torch.ones(1), device="cpu")


def test_plain_values_agree_with_the_oracle():
    import oracle
    codes, block = make_weight(1, 8, 64, 5, device="cpu")
    got = values(codes, block, torch.ones(1, 8))[0]
    assert torch.equal(got, torch.from_numpy(oracle.dequantize(codes[0].numpy(), block[0].numpy(), 1.0)).double())
    assert got.abs().max() <= 12.0 and got.unique().numel() > 20
