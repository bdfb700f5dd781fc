"""The value between the projections of the weight-only layer keeps f32's precision whatever its size: results of 16 bits are those of an f32
layer, rounded once, and small values are as exact as large ones."""
import pytest
import torch

from test_w4a16_gpu import _layer
from w4a16_ref import make_weight, values

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def plain(x, weights, ids, W13, W2, on_input=False):
    """(out, size, coarse, gate): the layer in 64 bits, the sum over magnitudes from the second projection on, the same with each value replaced by the largest
    of its pair, and the largest magnitude of a gate."""
    I = W2.shape[2]
    out = torch.zeros(x.shape[0], W2.shape[1], dtype=torch.float64, device=x.device)
    size, coarse, gate = out.clone(), out.clone(), 0.0
    for m, row in enumerate(ids.tolist()):
        for s, e in enumerate(row):
            w = float(weights[m, s])
            h = W13[e] @ x[m].double() * (w if on_input else 1.0)
            a = h[:I] / (1.0 + torch.exp(-h[:I])) * h[I:]
            f = 1.0 if on_input else w
            gate = max(gate, float(h[:I].abs().max()))
            out[m] += f * (W2[e] @ a)
            size[m] += abs(f) * (W2[e].abs() @ a.abs())
            coarse[m] += abs(f) * float(a.abs().max()) * W2[e].abs().sum(1)
    return out, size, coarse, gate


def check(out, x, weights, ids, W13, W2, on_input=False):
    """First sums are exact (w4a16_ref).  A gate is off by three roundings, 3 * 2^-24 of it, and its exponential by as much of itself times the gate; SiLU and the product are
    off by 2^-20 beyond that.  The value is two f16 that are off by 2^-24 of the largest of its run of eight or 2^-23 of itself; runs below 2^-28 of the pair's largest
    may be left out: 2^-23 of the largest together.  Then the second projection's I roundings of 2^-23, the sum's, and the result's own."""
    ref, size, coarse, gate = plain(x, weights, ids, W13, W2, on_input)
    I, topk = W2.shape[2], ids.shape[1]
    bound = (2.0 ** -20 + 2.0 ** -23 + 3 * 2.0 ** -24 * gate + (I + topk + 4) * 2.0 ** -23) * size + 2.0 ** -23 * coarse
    bound += torch.finfo(out.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(out.dtype).tiny
    assert bool(((out.double() - ref).abs() <= bound).all())
    return ref


@pytest.mark.parametrize("on_input", [False, True])
@pytest.mark.parametrize("M,E,H,I,topk,dtype", [
    (1, 4, 16, 16, 2, BF16), (1, 16, 512, 512, 8, BF16), (3, 4, 144, 48, 4, BF16), (5, 6, 4096, 512, 3, BF16), (7, 3, 272, 2064, 2, BF16), (9, 2, 256, 144, 1, BF16),
    (33, 3, 272, 64, 2, BF16), (130, 32, 96, 176, 3, BF16), (2, 9, 2048, 128, 4, F16), (40, 5, 64, 400, 3, F16)])
def test_results_are_an_f32_layers_rounded_once(M, E, H, I, topk, dtype, on_input):
    layer, x, weights, ids, _, W13, W2 = _layer(M, E, H, I, topk, dtype)
    for out in (None, torch.empty(M, H, device="cuda")):
        check(layer(x, weights, ids, on_input, out), x, weights, ids, W13, W2, on_input)


def _signed_layer(M, E, H, I, gate_at, signs, dtype=BF16):
    """Gates near `gate_at` for every value (rows and activations of one sign each), up rows as they come."""
    from dgx_vllm_b200.weight_only import W4A16MoE, pack_nvfp4_weight
    c13, b13 = make_weight(E, 2 * I, H, 3)
    c13[:, :I] = (c13[:, :I] & 0x77) | (0x88 if signs < 0 else 0)
    c2, b2 = make_weight(E, H, I, 4)
    W = values(c13, b13, torch.ones(E, 2 * I, device="cuda"))
    x = torch.randint(1, 8, (M, H), generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    typical = float((W[:, :I].abs() @ x[0].double()).mean())
    g13 = torch.tensor([[gate_at / typical, 1.0 / (12.0 * H ** 0.5)]]).expand(E, 2).contiguous().cuda()
    g2 = torch.full((E,), 1.0 / (3.0 * I ** 0.5), device="cuda")
    layer = W4A16MoE(pack_nvfp4_weight(c13, b13, g13, gated=True), pack_nvfp4_weight(c2, b2, g2))
    return layer, x, values(c13, b13, g13.repeat_interleave(I, 1)), values(c2, b2, g2[:, None].expand(E, H))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,H,I", [(6, 256, 160), (16, 128, 1040), (40, 256, 416)])      # one column of eight, one and two, two
@pytest.mark.parametrize("gate_at", [5.0, 15.0, 30.0, 60.0])
def test_pairs_whose_gates_are_all_strongly_negative(gate_at, M, H, I, dtype):
    layer, x, W13, W2 = _signed_layer(M, 3, H, I, gate_at, -1, dtype)
    ids = (torch.arange(M, dtype=torch.int32, device="cuda") % 3)[:, None].contiguous()
    weights = torch.full((M, 1), 0.75, device="cuda")
    out = torch.empty(M, H, device="cuda")                          # f16 results of 1e-10 are zeros
    ref = check(layer(x, weights, ids, False, out), x, weights, ids, W13, W2)
    assert gate_at < 10 or float(ref.abs().max()) < 2.0 ** (-gate_at / 4)     # as small as they are meant to be: the least gate of a row is over half of gate_at
    if dtype == BF16:
        check(layer(x, weights, ids), x, weights, ids, W13, W2)


def test_ordinary_calls_after_one_with_small_values():
    """What one call says of its values is not the next one's; two streams, each its own."""
    small, x, W13, W2 = _signed_layer(6, 3, 256, 160, 30.0, -1)
    layer, y, weights, ids, _, V13, V2 = _layer(6, 3, 256, 160, 1, BF16)
    want = layer(y, weights, ids).clone()
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(3):
                check(small(x, weights, ids), x, weights, ids, W13, W2)
                assert torch.equal(layer(y, weights, ids), want)
    check(want, y, weights, ids, V13, V2)


@pytest.mark.parametrize("up", [8, 16, 24])
def test_loud_channel_that_no_weight_reads(up):
    """One activation is 2^up times the others and meets zeros only: nothing of the others' products is lost for it."""
    from dgx_vllm_b200.weight_only import W4A16MoE, pack_nvfp4_weight
    E, H, I = 3, 144, 96
    c13, b13 = make_weight(E, 2 * I, H, 3)
    c13[:, :, 10] &= 0xF0                                           # k = 20
    c2, b2 = make_weight(E, H, I, 4)
    g13, g2 = torch.full((E,), 1.0 / (12.0 * H ** 0.5), device="cuda"), torch.full((E,), 1.0 / (3.0 * I ** 0.5), device="cuda")
    x = torch.randint(-7, 8, (5, H), generator=torch.Generator().manual_seed(5)).to(BF16).cuda()
    x[:, 20] = 2.0 ** up                                            # the others stay whole numbers times 2^-10 when the row is brought below 2^15
    layer = W4A16MoE(pack_nvfp4_weight(c13, b13, g13, gated=True), pack_nvfp4_weight(c2, b2, g2))
    W13, W2 = values(c13, b13, g13[:, None].expand(E, 2 * I)), values(c2, b2, g2[:, None].expand(E, H))
    ids = torch.tensor([[0, 1], [1, 2], [2, 0], [0, 2], [1, 0]], dtype=torch.int32, device="cuda")
    weights = torch.rand(5, 2, generator=torch.Generator().manual_seed(2)).cuda()
    check(layer(x, weights, ids), x, weights, ids, W13, W2)
    check(layer(x, weights, ids, False, torch.empty(5, H, device="cuda")), x, weights, ids, W13, W2)


def test_values_of_one_pair_spread_over_many_powers():
    """Units of the second projection whose values are 2^-100 to 2^100 of each other, in whatever order they come."""
    from dgx_vllm_b200.weight_only import W4A16MoE, pack_nvfp4_weight
    E, H, I = 2, 128, 1024
    c13, b13 = make_weight(E, 2 * I, H, 3)
    b13[:, :I] = 56                                                 # gates: scales of one
    power = torch.tensor([0, 6, 1, 8, 3, 11, 2, 14], dtype=torch.uint8).repeat_interleave(I // 8).cuda()      # up rows: 2^-6 to 2^8
    b13[:, I:] = ((power[:, None] + 1) * 8).expand(E, I, H // 16)
    c2, b2 = make_weight(E, H, I, 4)
    g13 = torch.tensor([[1.0 / (12.0 * H ** 0.5), 1.0 / (12.0 * H ** 0.5)]]).expand(E, 2).contiguous().cuda()
    g2 = torch.full((E,), 1.0 / (3.0 * I ** 0.5), device="cuda")
    layer = W4A16MoE(pack_nvfp4_weight(c13, b13, g13, gated=True), pack_nvfp4_weight(c2, b2, g2))
    W13, W2 = values(c13, b13, g13.repeat_interleave(I, 1)), values(c2, b2, g2[:, None].expand(E, H))
    x = torch.randint(-7, 8, (4, H), generator=torch.Generator().manual_seed(5)).to(BF16).cuda()
    x[2] = 0                                                        # nothing at all
    ids = torch.tensor([[0, 1], [1, 0], [0, 1], [1, 0]], dtype=torch.int32, device="cuda")
    weights = torch.rand(4, 2, generator=torch.Generator().manual_seed(2)).cuda()
    out = layer(x, weights, ids)
    check(out, x, weights, ids, W13, W2)
    assert bool((out[2] == 0).all())


def test_one_graph_with_ordinary_and_with_small_values():
    """Replays on inputs of both kinds, in turn: what a replay says of its values is at most looked at needlessly by the next."""
    layer, x, W13, W2 = _signed_layer(6, 3, 256, 160, 30.0, -1)
    ids = (torch.arange(6, dtype=torch.int32, device="cuda") % 3)[:, None].contiguous()
    weights = torch.full((6, 1), 0.75, device="cuda")
    kinds = [x, -x, x * 0.25, torch.zeros_like(x)]                  # all gates near -30, near 30, near -8; nothing
    want = [layer(k, weights, ids).clone() for k in kinds]
    for k, w in zip(kinds, want):
        check(w, k, weights, ids, W13, W2)
    given = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(given, weights, ids)
    for i in (1, 0, 1, 2, 3, 0, 2, 3):
        given.copy_(kinds[i])
        graph.replay()
        assert torch.equal(out, want[i])
