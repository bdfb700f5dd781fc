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


def _replayed_after_growth(capture, grow):
    """`capture()` captured on a stream, then `grow()` on it eagerly; what is allocated then keeps its values through replays.  Returns the captured call's output."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = capture().clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = capture()
        for _ in range(2):
            grow()
            stream.synchronize()
        others = [torch.full((n,), 7, dtype=torch.int32, device="cuda") for n in [1 << 18] * 24 + [64] * 64 + [1 << 21] * 8]
        for _ in range(3):
            out.fill_(0)
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, want)
        for t in others:
            assert bool((t == 7).all())
    del graph


def test_graph_beside_larger_calls_on_its_stream():
    from dgx_vllm_b200 import _torch_util as util
    from dgx_vllm_b200.weight_only import last_w4a16_status, pack_nvfp4_weight, w4a16_linear
    layer, x, weights, ids, _, _, _ = _layer(64, 4, 2048, 256, 4, BF16)
    codes, block = make_weight(1, 64, 2048, 5)
    w = pack_nvfp4_weight(codes[0], block[0], torch.ones(1, device="cuda"))
    words = set()

    def status_word():
        words.add(util.workspace(torch.device("cuda", torch.cuda.current_device()), 256, util.WS_W4A16_STATUS).data_ptr())
        assert last_w4a16_status() == 0

    def grow():
        status_word()
        layer(x, weights, ids)                                          # 2.6 MB of scratch
        layer(x.repeat(8, 1), weights.repeat(8, 1), ids.repeat(8, 1))   # 20 MB
        status_word()

    _replayed_after_growth(lambda: layer(x[:1], weights[:1], ids[:1]), grow)
    _replayed_after_growth(lambda: w4a16_linear(x[:3], w), grow)
    assert len(words) == 2                                              # one for each of the two streams


def test_graph_of_the_sparse_layer_beside_larger_calls_on_its_stream():
    """The scratch that the 2:4 layer was captured with stays its own as well."""
    import synth
    from dgx_vllm_b200.sparse_fp4_v7 import FusedSparseMoE
    from util import oracle_quantize_fn
    E, H, I, M, topk = 4, 512, 128, 256, 2
    w13 = synth.make_sparse_experts(E, 2 * I, H, 1, "cpu", oracle_quantize_fn)
    w2 = synth.make_sparse_experts(E, H, I, 2, "cpu", oracle_quantize_fn)
    keys = ("comp_T", "meta_T", "scale_T", "g_scales")
    layer = FusedSparseMoE(*[w13[k].cuda() for k in keys], *[w2[k].cuda() for k in keys], I)
    tw, ids = (t.cuda() for t in synth.make_routing(M, E, topk, 3, "cpu"))
    x = synth.make_hidden(M, H, 4, "cpu").cuda()
    _replayed_after_growth(lambda: layer(x[:2], tw[:2], ids[:2]),
                           lambda: layer(x.repeat(8, 1), tw.repeat(8, 1), ids.repeat(8, 1)))


@pytest.mark.parametrize("M", [1, 2, 5, 40, 300])
@pytest.mark.parametrize("packed_for,called_with", [((96, 128), (96, 112)), ((96, 128), (95, 128)), ((65, 128), (96, 128)), ((64, 128), (32, 256)), ((32, 256), (64, 128))])
def test_linear_op_with_sizes_that_its_weight_has_not(packed_for, called_with, M):
    """Packed bytes are as many for both; the result says so."""
    import dgx_vllm_b200.torch_ops  # noqa: F401
    from dgx_vllm_b200.weight_only import last_w4a16_status, pack_nvfp4_weight
    codes, block = make_weight(1, *packed_for, 4)
    w = pack_nvfp4_weight(codes[0], block[0], torch.ones(1, device="cuda"))
    N, K = called_with
    for out_dtype in (F32, None):
        y = torch.ops.b200_nvfp4.w4a16_linear(make_x(M, K, 1, BF16), w.packed, w.g_scale, N, None, out_dtype)
        assert tuple(y.shape) == (M, N) and bool(torch.isnan(y[:, -1:]).all()) and last_w4a16_status() == 63      # no row without
    y = torch.ops.b200_nvfp4.w4a16_linear(make_x(M, packed_for[1], 1, BF16), w.packed, w.g_scale, packed_for[0], None, F32)
    assert not bool(torch.isnan(y).any()) and last_w4a16_status() == 0


@pytest.mark.parametrize("M", [1, 6, 40])
def test_layer_op_with_sizes_that_its_weights_have_not(M):
    import dgx_vllm_b200.torch_ops  # noqa: F401
    from dgx_vllm_b200.weight_only import last_w4a16_status
    layer, x, weights, ids, _, _, _ = _layer(M, 4, 128, 64, 2, BF16)
    ids[0] = -1
    op = torch.ops.b200_nvfp4.w4a16_moe
    hidden = x[:, :112].contiguous()                                # as many bytes
    for on_input in (False, True):
        out = op(hidden, weights, ids, None, *layer._weights, 64, on_input)
        assert bool((out[0] == 0).all()) and bool(torch.isnan(out[1:]).all()) and last_w4a16_status() == 63
    with pytest.raises(RuntimeError):
        op(x, weights, ids, None, *layer._weights, 48, False)
    assert torch.equal(op(x, weights, ids, None, *layer._weights, 64, False), layer(x, weights, ids)) and last_w4a16_status() == 0


def test_tensors_that_are_no_packed_weights_are_refused():
    import dgx_vllm_b200.torch_ops  # noqa: F401
    from dgx_vllm_b200 import _lib
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight
    codes, block = make_weight(1, 96, 128, 4)
    one = torch.ones(1, device="cuda")
    w = pack_nvfp4_weight(codes[0], block[0], one)
    x = make_x(5, 128, 1, BF16)
    linear = lambda packed, g=one, n=96, x=x: torch.ops.b200_nvfp4.w4a16_linear(x, packed, g, n, None, None)
    stub = torch.zeros(1, dtype=torch.uint8, device="cuda").expand(w.packed.numel())
    for bad in (lambda: linear(w.packed[:-4]), lambda: linear(torch.cat((w.packed, w.packed))), lambda: linear(w.packed.view(torch.int32)), lambda: linear(stub),
                lambda: linear(w.packed, one.double()), lambda: linear(w.packed, one.to(BF16)), lambda: linear(w.packed, n=0), lambda: linear(w.packed, n=97),
                lambda: linear(pack_nvfp4_weight(codes[0], block[0], one, gated=True).packed), lambda: linear(w.packed, x=make_x(5, 256, 1, BF16))):
        with pytest.raises(RuntimeError):
            bad()
    layer, x, weights, ids, emap, _, _ = _layer(6, 4, 128, 64, 2, BF16, parallel=2)
    w13, g13, w2, g2 = layer._weights
    call = lambda *w, m=emap, out=None: _lib.host().w4a16_moe(*w, m, 128, 64, 4, x, weights, ids, False, out)
    for bad in (lambda: call(w13, g13, w2, g2.double()), lambda: call(w13, g13.to(BF16), w2, g2), lambda: call(w13, g13.T, w2, g2), lambda: call(w2, g13, w13, g2),
                lambda: call(w13.view(torch.int32), g13, w2, g2), lambda: call(w13[:-8], g13, w2, g2), lambda: call(w13, g13, w2[4:], g2),
                lambda: call(w13, g13, torch.zeros(1, dtype=torch.uint8, device="cuda").expand(w2.numel()), g2),
                lambda: call(w13, g13, w2, g2, m=emap.long()), lambda: call(w13, g13, w2, g2, m=emap[::2])):
        with pytest.raises(RuntimeError):
            bad()
    assert torch.equal(call(w13, g13, w2, g2), layer(x, weights, ids))


def test_results_in_the_memory_of_other_arguments_are_refused():
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, 64, 64, 3)
    w = pack_nvfp4_weight(codes[0], block[0], torch.ones(1, device="cuda"))
    room = torch.zeros(6 * 64, device="cuda")
    x = make_x(4, 64, 1, BF16)
    with pytest.raises(RuntimeError, match="overlap"):
        w4a16_linear(x, w, room[:64], out=room[:256].view(4, 64))
    w4a16_linear(x, w, room[256:320], out=room[:256].view(4, 64))
    layer, x, weights, ids, emap, _, _ = _layer(4, 4, 64, 32, 2, BF16, parallel=2)
    out = torch.zeros(4, 64, device="cuda")
    flat = out.view(-1)
    flat[:8].copy_(weights.view(-1))
    flat[16:24].view(torch.int32).copy_(ids.view(-1))
    flat[32:40].view(torch.int32).copy_(emap)
    for args in ((x, flat[:8].view(4, 2), ids, False, out), (x, weights, flat[16:24].view(torch.int32).view(4, 2), False, out),
                 (x, weights, ids, False, out, flat[32:40].view(torch.int32))):
        with pytest.raises(RuntimeError, match="overlap"):
            layer(*args)


def test_vllm_adapter_takes_activations_as_they_come():
    """Rows 8 bytes off, one row many times, every other row: the operators' own alignment is the adapter's business."""
    import types
    from dgx_vllm_b200 import vllm_adapter as va
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, 48, 64, 6)
    w = pack_nvfp4_weight(codes[0], block[0], torch.ones(1, device="cuda"))
    lin = types.SimpleNamespace(w4a16_weight=w, output_size_per_partition=48)
    core = va.Nvfp4WeightOnlyLinearCore()
    x = make_x(6, 64, 1, BF16)
    room = torch.zeros(6 * 64 + 4, dtype=BF16, device="cuda")
    off = room[4:].view(6, 64).copy_(x)
    wide = torch.cat((x, x), 1).view(12, 64)
    for given in (x, off, x[2:3].expand(6, 64), x.view(6, 1, 64).expand(6, 3, 64), wide[::2], x[0], x[:0]):
        want = w4a16_linear(given.reshape(-1, 64).contiguous().clone(), w)
        assert torch.equal(core.apply_weights(lin, given), want.view(*given.shape[:-1], 48))
    layer, x, weights, ids, _, _, _ = _layer(6, 4, 64, 32, 2, BF16)
    off = room[4:].view(6, 64).copy_(x)
    moe = va.make_w4a16_apply_fn(*_packed(4, 64, 32))
    for given in (x, off, torch.cat((x, x), 1)[:, :64]):
        out = torch.full((8, 64), 5.0, dtype=BF16, device="cuda")
        moe(out, given, None, None, weights, ids, "silu", 4, None, None, None, None, None, None, False)
        assert torch.equal(out[:6], layer(x, weights, ids)) and bool((out[6:] == 5).all())


def _packed(E, H, I, seed=0, M=6):
    """The weights of _layer(M, E, H, I, ...)."""
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight
    gen = torch.Generator().manual_seed(seed + M + E)
    g13 = (torch.rand(E, 1, generator=gen) + 0.5).cuda() / (12.0 * H ** 0.5)
    g2 = (torch.rand(E, generator=gen) + 0.5).cuda() / (3.0 * I ** 0.5)
    return pack_nvfp4_weight(*make_weight(E, 2 * I, H, seed + 1), g13.squeeze(1), gated=True), pack_nvfp4_weight(*make_weight(E, H, I, seed + 2), g2)


@pytest.mark.parametrize("M,E,H,topk", [(381, 128, 43008, 8), (256, 256, 40000, 8), (1030, 8, 44032, 2), (3, 4, 59904, 2)])
def test_layer_of_long_rows_in_turns(M, E, H, topk):
    """Rows that fit beside the sums of two columns only, in full turns and in a last one of fewer pairs."""
    from test_w4a16_gpu import _check
    layer, x, weights, ids, emap, W13, W2 = _layer(M, E, H, 16, topk, BF16)
    out = layer(x, weights, ids)
    some = torch.tensor(sorted({0, 1, M // 2, min(255, M - 1), max(0, M - 125), M - 2, M - 1}), device="cuda")
    _check(out[some], x[some], weights[some], ids[some], emap, W13, W2)
