"""Weight-only NVFP4 operators on the GPU against plain 64-bit forms, at the sizes where tiles, slots and roundings can go wrong."""
import threading

import pytest
import torch

from w4a16_ref import make_weight, make_x, moe, values

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


def _linear(M, N, K, dtype, out_dtype=None, bias_dtype=None, pad=0, exact=True, seed=0, g=0.5):
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, N, K, seed + N + K, exact)
    x = make_x(M, K, seed + M, dtype, exact, pad)
    bias = None if bias_dtype is None else make_x(1, N, seed + 5, bias_dtype)[0].contiguous()
    gs = torch.tensor([g], device="cuda")
    w = pack_nvfp4_weight(codes[0], block[0].view(torch.float8_e4m3fn), gs)
    y = w4a16_linear(x, w, bias, out_dtype=out_dtype)
    W = values(codes, block, gs.reshape(1, 1))[0]
    ref = x.double() @ W.T + (0 if bias is None else bias.double())
    return y, ref, x.double().abs() @ W.abs().T


# Sums are exact in f32 (w4a16_ref), so the f32 result is the exact one, and a 16-bit result its one rounding.
@pytest.mark.parametrize("M,N,K,dtype,out_dtype,bias_dtype,pad", [
    (1, 1, 16, BF16, F32, None, 0),               # smallest
    (1, 16, 128, F16, F32, None, 0),              # one whole unit
    (2, 17, 144, BF16, None, None, 8),            # one past a tile and a unit; a slice of a wider tensor
    (1, 300, 4112, BF16, None, BF16, 0),          # a token with a block of k a column
    (2, 600, 8208, F16, F32, None, 8),            # two
    (2, 64, 128, BF16, F32, None, 0),
    (3, 64, 128, F16, F32, None, 0),              # one more
    (7, 40, 112, F16, None, F16, 0),              # a unit that ends early, a bias
    (8, 129, 2064, BF16, F32, F32, 16),           # all columns of one instruction, k split unevenly
    (9, 33, 256, F16, F32, BF16, 0),              # one more: two of them
    (16, 2400, 528, BF16, None, None, 0),         # more tiles than blocks
    (17, 31, 1040, BF16, F32, None, 0),           # four
    (31, 5000, 80, F16, F32, None, 8),            # hardly any k, many tiles
    (33, 48, 4096, BF16, F32, F32, 0),            # past 32 tokens, long k
    (64, 130, 272, F16, None, None, 0),
    (65, 257, 640, BF16, F32, BF16, 8),
    (130, 272, 1024, BF16, None, None, 0),
    (257, 129, 176, F16, F32, None, 0),
    (300, 640, 2048, BF16, None, BF16, 0),
    (1029, 384, 512, F16, None, None, 0),
    (577, 6465, 256, BF16, F32, None, 0),         # more tiles of the widest kind than blocks: two accumulators, few stages
    (2000, 1300, 144, F16, None, F32, 0),
    (18, 20000, 64, BF16, None, None, 8),         # more narrow ones
    (48, 96, 8208, F16, F32, None, 0),            # one tile for a cluster
    (700, 2300, 4096, F16, F32, BF16, 8),         # f32 results: several chains a tile, more tiles than blocks
    (190, 1000, 3344, BF16, F32, F32, 0),         # ... one tile a block, the last chain short
    (130, 260, 4096, BF16, F32, None, 0),         # ... chains of a cluster's blocks
    (190, 40, 4096, F16, F32, BF16, 0),
    (5, 5000, 4096, BF16, F32, None, 0),          # ... warps
    (12, 600, 4096, F16, F32, BF16, 0),
])
def test_linear_exact(M, N, K, dtype, out_dtype, bias_dtype, pad):
    y, ref, _ = _linear(M, N, K, dtype, out_dtype, bias_dtype, pad)
    assert y.dtype == (out_dtype or dtype) and tuple(y.shape) == (M, N)
    assert torch.equal(y, ref.to(F32).to(y.dtype))


# Any scales and normal activations: products are exact, a sum of K of them in f32 is off by at most K roundings (to nearest or toward zero: 2^-23)
# of the sum of magnitudes; then one multiplication by the factor and the rounding to the output's type.
@pytest.mark.parametrize("M,N,K,dtype,out_dtype", [
    (1, 300, 4096, BF16, F32), (5, 300, 1600, F16, F32), (16, 128, 2048, BF16, BF16), (40, 100, 1024, F16, F32), (200, 256, 2048, BF16, F32),
    (513, 200, 800, F16, F16)])
def test_linear_rounding(M, N, K, dtype, out_dtype):
    y, ref, size = _linear(M, N, K, dtype, out_dtype, exact=False, g=3e-4)
    bound = (K + 2) * 2.0 ** -23 * size + half_eps(out_dtype) * ref.abs() * (1 + 2.0 ** -10) + torch.finfo(out_dtype).tiny
    assert bool(((y.double() - ref).abs() <= bound).all())


# An f32 result keeps to f32's precision however long k is: a matrix instruction (16 of k) truncates its sum, by 2^-23 of it at most, and a chain has at most 96 of
# them; errors of chains add up like the chains themselves.  So the norm of the differences is within
# 96 * 2^-23 of the result's.
@pytest.mark.parametrize("M,N,K,dtype", [(1, 900, 14336, BF16), (4, 8192, 14336, BF16), (12, 700, 14336, F16), (32, 4096, 14336, BF16), (150, 1024, 14336, BF16),
                                         (400, 8192, 14336, F16)])
def test_linear_f32_results_of_long_sums(M, N, K, dtype):
    y, ref, _ = _linear(M, N, K, dtype, F32, exact=False, g=3e-4)
    assert float((y.double() - ref).norm()) <= 96 * 2.0 ** -23 * float(ref.norm())


def test_linear_scale_bytes_and_signs():
    """Every finite scale byte, negative ones and subnormal ones among them, against every code: products of one k are exact."""
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    block = torch.tensor([b for b in range(256) if b & 127 != 127], dtype=torch.uint8, device="cuda")[:, None]
    codes = (torch.arange(8, dtype=torch.uint8, device="cuda") * 34 + 16).expand(block.shape[0], 8).contiguous()      # low nibbles 0, 2, ..., high 1, 3, ...
    one = torch.ones(1, device="cuda")
    w = pack_nvfp4_weight(codes, block, one)
    W = values(codes[None], block[None], one.reshape(1, 1))[0]
    for dtype in (BF16, F16):
        y = w4a16_linear(torch.eye(16, dtype=dtype, device="cuda"), w, out_dtype=F32)
        assert torch.equal(y.double(), W.T)


def test_linear_infinite_and_nan_activations_stay_in_their_rows():
    y_ref, _, _ = _linear(5, 70, 256, BF16, F32)
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, 70, 256, 70 + 256)
    w = pack_nvfp4_weight(codes[0], block[0], torch.tensor([0.5], device="cuda"))
    x = make_x(5, 256, 5, BF16)
    x[1, 3] = float("inf")
    x[3, 200] = float("nan")
    y = w4a16_linear(x, w, out_dtype=F32)
    for m in (0, 2, 4):
        assert torch.equal(y[m], y_ref[m])
    W = values(codes, block, torch.tensor([[0.5]], device="cuda"))[0]
    want = x[1].double() @ W.T
    assert torch.equal(torch.isnan(y[1]), torch.isnan(want)) and torch.equal(torch.isinf(y[1]), torch.isinf(want))
    assert bool(torch.isnan(y[3]).all())


def test_linear_out_argument_no_tokens_and_refusals():
    from dgx_vllm_b200.weight_only import last_w4a16_status, pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, 64, 128, 3)
    g = torch.ones(1, device="cuda")
    w = pack_nvfp4_weight(codes[0], block[0], g)
    x = make_x(4, 128, 0, BF16)
    out = torch.full((4, 64), 7.0, dtype=F16, device="cuda")
    assert w4a16_linear(x, w, out=out) is out
    assert torch.equal(out, w4a16_linear(x, w, out_dtype=F32).to(F16))
    assert tuple(w4a16_linear(x[:0], w).shape) == (0, 64)
    assert last_w4a16_status() == 0
    for bad in (lambda: w4a16_linear(x.float(), w), lambda: w4a16_linear(x[:, :112], w), lambda: w4a16_linear(x.cpu(), w),
                lambda: w4a16_linear(make_x(4, 128, 0, BF16, pad=4), w),                                   # rows 8 bytes off
                lambda: w4a16_linear(make_x(4, 136, 0, BF16)[:, 1:129], w), lambda: w4a16_linear(x.T.contiguous().T, w),
                lambda: w4a16_linear(x[:1].expand(4, 128), w),                                             # rows on top of each other
                lambda: w4a16_linear(x, w, torch.zeros(63, device="cuda")), lambda: w4a16_linear(x, w, out=out[:, :32]),
                lambda: w4a16_linear(x, w, out_dtype=torch.int8), lambda: w4a16_linear(x, w, out=out, out_dtype=F32),
                lambda: w4a16_linear(x, pack_nvfp4_weight(codes[0], block[0], g, gated=True)),
                lambda: pack_nvfp4_weight(codes[0, :, :60], block[0], g), lambda: pack_nvfp4_weight(codes[0, :, :63], block[0], g),
                lambda: pack_nvfp4_weight(codes[0, :63], block[0, :63], g, gated=True),
                lambda: pack_nvfp4_weight(codes[0], block[0], torch.ones(2, device="cuda")),
                lambda: pack_nvfp4_weight(codes[0], block[0] | 127, g)):
        with pytest.raises((RuntimeError, TypeError)):
            bad()


# Rows too long for the shared memory of the few-token kernel; a row has 64 numbers in it, so that sums are exact.
@pytest.mark.parametrize("M,K,dtype", [(1, 524304, BF16), (3, 1100000, F16)])
def test_linear_very_long_rows(M, K, dtype):
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, 40, K, 5)
    g = torch.ones(1, device="cuda")
    x = torch.zeros(M, K, dtype=dtype, device="cuda")
    at = torch.randint(0, K, (64,), generator=torch.Generator().manual_seed(1)).cuda()
    at[0], at[1] = K - 1, 0
    x[:, at] = make_x(M, 64, 3, dtype)
    y = w4a16_linear(x, pack_nvfp4_weight(codes[0], block[0], g), out_dtype=F32)
    assert torch.equal(y.double(), x.double() @ values(codes, block, g.reshape(1, 1))[0].T)


@pytest.mark.parametrize("M", [2, 40000])
def test_linear_offsets_past_32_bits(M):
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    N, K, ld = (64, 16, 1 << 31) if M == 2 else (60000, 16, 56000)             # elements of x; 2.2e9 of x and 2.4e9 of the result
    codes, block = make_weight(1, N, K, 5)
    g = torch.ones(1, device="cuda")
    x = torch.empty((M - 1) * ld + K, dtype=BF16, device="cuda").as_strided((M, K), (ld, 1))
    x.copy_(make_x(M, K, 3, BF16))
    y = w4a16_linear(x, pack_nvfp4_weight(codes[0], block[0], g))
    W = values(codes, block, g.reshape(1, 1))[0]
    for rows in (slice(0, 2), slice(M // 2, M // 2 + 2), slice(M - 2, M)):
        assert torch.equal(y[rows], (x[rows].double() @ W.T).to(BF16))


def test_linear_result_in_its_own_input_is_refused():
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, 64, 64, 3)
    w = pack_nvfp4_weight(codes[0], block[0], torch.ones(1, device="cuda"))
    room = torch.zeros(5 * 64, dtype=BF16, device="cuda")
    x, apart = room[:256].view(4, 64), torch.zeros(4, 64, dtype=BF16, device="cuda")
    for out in (x, room[64:].view(4, 64)):
        with pytest.raises(RuntimeError, match="overlap"):
            w4a16_linear(x, w, out=out)
    w4a16_linear(x[:1], w, out=room[64:128].view(1, 64))                       # next to it
    w4a16_linear(x, w, out=apart)


# ------------------------------------------------------------------------------------------ layer

def _layer(M, E, H, I, topk, dtype, parallel=1, seed=0, ids=None, split_factors=False):
    from dgx_vllm_b200.weight_only import W4A16MoE, pack_nvfp4_weight
    gen = torch.Generator().manual_seed(seed + M + E)
    c13, b13 = make_weight(E, 2 * I, H, seed + 1)
    c2, b2 = make_weight(E, H, I, seed + 2)
    g13 = (torch.rand(E, 2 if split_factors else 1, generator=gen) + 0.5).cuda() / (12.0 * H ** 0.5)
    g2 = (torch.rand(E, generator=gen) + 0.5).cuda() / (3.0 * I ** 0.5)
    x = make_x(M, H, seed, dtype)
    weights = torch.rand(M, topk, generator=gen).cuda()
    if ids is None:
        ids = torch.stack([torch.randperm(E * parallel, generator=gen)[:topk] for _ in range(M)])
    ids = ids.to(torch.int32).cuda()
    emap = None
    if parallel > 1:
        emap = torch.full((E * parallel,), -1, dtype=torch.int32)
        emap[E // 2:E // 2 + E] = torch.arange(E, dtype=torch.int32)
        emap = emap.cuda()
    layer = W4A16MoE(pack_nvfp4_weight(c13, b13, g13.squeeze(1) if not split_factors else g13, gated=True), pack_nvfp4_weight(c2, b2, g2), expert_map=emap)
    rows = g13.expand(E, 2).repeat_interleave(I, 1)
    return layer, x, weights, ids, emap, values(c13, b13, rows), values(c2, b2, g2[:, None].expand(E, H))


def _check(out, x, weights, ids, emap, W13, W2, on_input=False, looser=1.0):
    """Sums of the first projection are exact; its factor, SiLU and the product cost a few f32 roundings (2^-20 together).  The value between the projections
    is one f16 (2^-11) where the result is bf16, else the sum of two (2^-22); below f16's normal range a rounding is 2^-25 of the factor that brought the row there, which is
    at most 2^-13 of a bound: the product of |x| sqrt(H) 12 g for gate and up, g at most 1.5 / (12 sqrt(H)).  The second projection adds I roundings
    of its sum of magnitudes, the sum over pairs topk, the output one of its type."""
    ref, size = moe(x, weights, ids, emap, W13, W2, on_input)
    I, topk = W2.shape[2], ids.shape[1]
    between = 2.0 ** -11 if out.dtype == BF16 else 2.0 ** -22
    least = 2.0 ** -38 * (1.5 * x.double().norm(dim=1, keepdim=True)) ** 2 * weights.double().abs().clamp(min=1).sum(1, keepdim=True) * W2.abs().sum(2).amax()
    bound = (between + 2.0 ** -20 + (I + topk + 4) * 2.0 ** -23) * size + looser * least + half_eps(out.dtype) * ref.abs() * (1 + 2.0 ** -10) + torch.finfo(out.dtype).tiny
    assert tuple(out.shape) == tuple(ref.shape)
    assert bool(((out.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("M,E,H,I,topk,dtype,parallel", [
    (1, 1, 16, 16, 1, BF16, 1),               # smallest
    (1, 8, 128, 128, 2, F16, 1),              # whole units
    (3, 4, 144, 48, 4, BF16, 1),              # every expert for every token, k past a unit and short of one
    (5, 600, 80, 32, 7, BF16, 1),             # more experts than threads
    (9, 2, 256, 144, 1, F16, 1),              # past the columns of one instruction
    (33, 3, 272, 64, 2, BF16, 1),             # several slots an expert
    (70, 5, 64, 80, 5, F16, 1),               # ... and two tiles at once
    (64, 8, 2048, 256, 4, BF16, 4),           # a rank of four: most pairs are elsewhere
    (16, 16, 512, 512, 10, BF16, 1),
    (130, 32, 96, 176, 3, BF16, 2),
])
@pytest.mark.parametrize("on_input", [False, True])
def test_moe(M, E, H, I, topk, dtype, parallel, on_input):
    layer, x, weights, ids, emap, W13, W2 = _layer(M, E, H, I, topk, dtype, parallel)
    out = layer(x, weights, ids, apply_router_weight_on_input=on_input)
    assert out.dtype == dtype
    _check(out, x, weights, ids, emap, W13, W2, on_input)
    out32 = torch.full((M, H), 3.0, device="cuda")
    assert layer(x, weights, ids, on_input, out32) is out32
    _check(out32, x, weights, ids, emap, W13, W2, on_input)
    assert torch.equal(layer(x, weights, ids.long(), on_input), out)            # any order of blocks gives the same


def test_moe_gate_and_up_factors_of_their_own():
    args = _layer(6, 4, 128, 64, 2, BF16, split_factors=True)
    _check(args[0](*args[1:4]), *args[1:])


@pytest.mark.parametrize("what", ["nothing", "some rows", "same expert", "out of range", "one expert"])
def test_moe_routings(what):
    M, E, topk = 21, 6, 3
    gen = torch.Generator().manual_seed(9)
    ids = torch.randint(0, E, (M, topk), generator=gen)
    if what == "nothing":
        ids[:] = -1
    elif what == "some rows":
        ids[::3] = -1
    elif what == "same expert":
        ids[:, 1] = ids[:, 0]
    elif what == "out of range":
        ids[::2, 1] = E + 100000
        ids[1::2, 2] = -(1 << 31)
    else:
        ids[:] = 4
    args = _layer(M, E, 160, 96, topk, BF16, ids=ids)
    out = args[0](*args[1:4])
    _check(out, *args[1:])
    if what == "nothing":
        assert bool((out == 0).all())


def test_moe_more_pairs_than_a_turn():
    args = _layer(1400, 4, 64, 32, 3, BF16)
    _check(args[0](*args[1:4]), *args[1:])


# Down projections whose strips one block or a cluster of 2, 4 or 8 has to itself, or that has several of them; runs of items that end in phases of
# every kind; as many experts as there may be, as many pairs as a turn has and one more.
@pytest.mark.parametrize("M,E,H,I,topk,dtype", [
    (1, 16, 512, 256, 8, BF16), (2, 16, 1024, 1024, 4, F16), (3, 12, 2048, 640, 5, BF16), (5, 6, 4096, 512, 3, BF16), (2, 9, 8192, 128, 4, F16),
    (1, 3, 96, 2048, 1, BF16), (13, 7, 4096, 1040, 2, BF16), (11, 3, 1552, 4096, 2, F16),
    (6, 4096, 32, 16, 50, BF16), (256, 64, 16, 16, 8, BF16), (683, 9, 16, 32, 3, F16)])
def test_moe_shares_of_blocks(M, E, H, I, topk, dtype):
    args = _layer(M, E, H, I, topk, dtype)
    _check(args[0](*args[1:4]), *args[1:])


@pytest.mark.parametrize("up", [64, -76])
def test_moe_squares_outside_the_range_of_f32(up):
    """Activations times 2^up and first factors times 2^-up give what there was, although the squares of a row overflow or vanish.  The value between the
    projections then goes by the row's largest magnitude times sqrt(H): above the norm by at most 4 * 7 / 4 for these rows, twice, or 2^6."""
    from dgx_vllm_b200.weight_only import W4A16MoE, pack_nvfp4_weight
    M, E, H, I = 4, 3, 128, 64
    c13, b13 = make_weight(E, 2 * I, H, 1)
    c2, b2 = make_weight(E, H, I, 2)
    g13, g2 = torch.full((E,), 1.0 / (12.0 * H ** 0.5), device="cuda"), torch.full((E,), 1.0 / (3.0 * I ** 0.5), device="cuda")
    x, weights = make_x(M, H, 0, BF16), torch.rand(M, 2, generator=torch.Generator().manual_seed(1)).cuda()
    ids = torch.tensor([[0, 1], [2, 0], [1, 2], [2, 1]], dtype=torch.int32, device="cuda")
    layer = W4A16MoE(pack_nvfp4_weight(c13, b13, g13 * 2.0 ** -up, gated=True), pack_nvfp4_weight(c2, b2, g2))
    W13, W2 = values(c13, b13, g13[:, None].expand(E, 2 * I)), values(c2, b2, g2[:, None].expand(E, H))
    _check(layer(x * 2.0 ** up, weights, ids), x, weights, ids, None, W13, W2, looser=64.0)


@pytest.mark.parametrize("M", [3, 1400])
def test_moe_in_place(M):
    layer, x, weights, ids, _, _, _ = _layer(M, 4, 64, 32, 3, BF16)
    want = layer(x, weights, ids)
    assert layer(x, weights, ids, False, x) is x
    assert torch.equal(x, want)
    room = torch.zeros((M + 1) * 64, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        layer(room[:M * 64].view(M, 64), weights, ids, False, room[64:].view(M, 64))


def test_moe_rows_too_long_are_refused():
    layer, x, weights, ids, _, _, _ = _layer(1, 1, 131072, 16, 1, BF16)
    with pytest.raises(RuntimeError):
        layer(x, weights, ids)


def test_moe_infinities_stay_with_their_token():
    layer, x, weights, ids, emap, W13, W2 = _layer(8, 3, 128, 64, 2, BF16)
    want = layer(x, weights, ids)
    x = x.clone()
    x[5, 7] = float("inf")
    got = layer(x, weights, ids)
    keep = [0, 1, 2, 3, 4, 6, 7]
    assert torch.equal(got[keep], want[keep])
    assert not bool(torch.isfinite(got[5]).all())


def test_moe_refusals():
    from dgx_vllm_b200.weight_only import W4A16MoE, pack_nvfp4_weight
    layer, x, weights, ids, _, _, _ = _layer(4, 3, 64, 32, 2, BF16)
    assert tuple(layer(x[:0], weights[:0], ids[:0]).shape) == (0, 64)
    for bad in (lambda: layer(x.float(), weights, ids), lambda: layer(x[:, :32], weights, ids), lambda: layer(x, weights[:, :1], ids),
                lambda: layer(x, weights, ids[:3]), lambda: layer(x, weights, ids.float()), lambda: layer(x.cpu(), weights, ids),
                lambda: layer(x, weights, ids, False, torch.empty(4, 32, device="cuda")), lambda: layer(x, weights, ids[:, :0])):
        with pytest.raises((RuntimeError, TypeError)):
            bad()
    c, b = make_weight(3, 64, 64, 1)
    g = torch.ones(3, device="cuda")
    flat, gated = pack_nvfp4_weight(c, b, g), pack_nvfp4_weight(c, b, g, gated=True)
    for bad in (lambda: W4A16MoE(flat, flat), lambda: W4A16MoE(gated, gated), lambda: W4A16MoE(gated, flat)):
        with pytest.raises(RuntimeError):
            bad()


# ------------------------------------------------------------------------------------------ as they are used together

def _block(M, seed=0, dtype=BF16, E=16, H=256, I=128, topk=4):
    """Projection, router, experts: what a decoder layer runs one after the other."""
    from dgx_vllm_b200.router import moe_router
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    layer, x, _, _, _, W13, W2 = _layer(M, E, H, I, topk, dtype, seed=seed)
    c, b = make_weight(1, H, H, seed + 7)
    g = torch.tensor([1.0 / (4.0 * H ** 0.5)], device="cuda")
    w = pack_nvfp4_weight(c[0], b[0], g)
    gate = (torch.randn(E, H, generator=torch.Generator().manual_seed(seed)) * 0.05).to(dtype).cuda()

    def run(x):
        h = w4a16_linear(x, w)
        tw, ids = moe_router(h, gate, topk)
        return h, tw, ids, layer(h, tw, ids)

    return run, x, (values(c, b, g.reshape(1, 1))[0], W13, W2)


@pytest.mark.parametrize("M", [1, 6, 40])
def test_projection_router_experts(M):
    run, x, (W, W13, W2) = _block(M)
    h, tw, ids, out = run(x)
    want = x.double() @ W.T
    assert bool(((h.double() - want).abs() <= half_eps(BF16) * want.abs() * (1 + 2.0 ** -10)).all())
    ref, size = moe(h, tw, ids, None, W13, W2)
    # here the first projection's sums are not exact either: its 256 terms may be off by 2^-23 each of their sum of magnitudes, which SiLU and the
    # product pass on by at most (1.1 |u| + |silu(g)|) / |a| of it; magnitudes of gate and up are below 16 and their sums below 2^8
    bound = (2.0 ** -11 + 2.0 ** -20 + 140 * 2.0 ** -23) * size + half_eps(BF16) * ref.abs() * (1 + 2.0 ** -10)
    sums = (h.double().abs() @ W13.abs().transpose(1, 2)).amax()
    bound += 256 * 2.0 ** -23 * sums * (1.1 * 16 + 16) * tw.sum(1, keepdim=True) * W2.abs().sum(2).amax()
    assert bool(((out.double() - ref).abs() <= bound).all())


def test_graphs_replayed_at_once_share_no_scratch():
    runs = [_block(5, seed) for seed in (0, 3)]
    want = [run(x)[3].clone() for run, x, _ in runs]
    graphs, outs = [], []
    for run, x, _ in runs:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(x)[3])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_weights_packed_and_inputs_made_just_before_on_another_stream():
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    s = torch.cuda.Stream()
    codes, block = make_weight(1, 512, 1024, 11)
    x = make_x(4, 1024, 2, BF16)
    g = torch.ones(1, device="cuda")
    want = w4a16_linear(x, pack_nvfp4_weight(codes[0], block[0], g), out_dtype=F32)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(5):
            y = w4a16_linear(x * 2, pack_nvfp4_weight(codes[0], block[0], g), out_dtype=F32)
    s.synchronize()
    assert torch.equal(y, 2 * want)


def test_threads_on_one_stream():
    runs = [_block(3, seed) for seed in range(3)]
    want = [run(x)[3].clone() for run, x, _ in runs]
    got = [None] * len(runs)

    def work(i):
        run, x, _ = runs[i]
        for _ in range(30):
            got[i] = run(x)[3]

    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(runs))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_custom_ops():
    import dgx_vllm_b200.torch_ops  # noqa: F401
    from dgx_vllm_b200.weight_only import pack_nvfp4_weight, w4a16_linear
    codes, block = make_weight(1, 96, 128, 4)
    w = pack_nvfp4_weight(codes[0], block[0], torch.ones(1, device="cuda"))
    x, bias = make_x(5, 128, 1, BF16), torch.ones(96, device="cuda")
    torch.library.opcheck(torch.ops.b200_nvfp4.w4a16_linear.default, (x, w.packed, w.g_scale, 96, bias, F32), test_utils=("test_schema", "test_faketensor"))
    assert torch.equal(torch.ops.b200_nvfp4.w4a16_linear(x, w.packed, w.g_scale, 96, bias, F32), w4a16_linear(x, w, bias, out_dtype=F32))
    layer, x, weights, ids, emap, _, _ = _layer(6, 4, 128, 64, 2, BF16, parallel=2)
    got = torch.ops.b200_nvfp4.w4a16_moe(x, weights, ids, emap, *layer._weights, 64, False)
    assert torch.equal(got, layer(x, weights, ids))
    torch.library.opcheck(torch.ops.b200_nvfp4.w4a16_moe.default, (x, weights, ids, emap, *layer._weights, 64, False), test_utils=("test_schema", "test_faketensor"))


def test_vllm_adapter_on_the_device():
    """A checkpoint layer through the weight-loading hooks: experts and a linear, against the plain forms."""
    import types
    from dgx_vllm_b200 import vllm_adapter as va
    E, H, I, M, topk = 5, 128, 64, 9, 2
    c13, b13 = make_weight(E, 2 * I, H, 1)
    c2, b2 = make_weight(E, H, I, 2)
    g13 = (torch.rand(E, 2, generator=torch.Generator().manual_seed(1)) + 0.5).cuda() / (12.0 * H ** 0.5)
    g2 = torch.full((E, 2), 1.0 / (3.0 * I ** 0.5), device="cuda")
    P = lambda t: torch.nn.Parameter(t, requires_grad=False)
    layer = types.SimpleNamespace(w13_weight=P(c13), w2_weight=P(c2), w13_weight_scale=P(b13), w2_weight_scale=P(b2), w13_weight_scale_2=P(g13),
                                  w2_weight_scale_2=P(g2))
    W13, W2 = values(c13, b13, g13.repeat_interleave(I, 1)), values(c2, b2, g2[:, :1].expand(E, H))
    experts = types.SimpleNamespace(apply=None)
    assert va.process_moe_layer_weight_only(types.SimpleNamespace(moe_mk=types.SimpleNamespace(fused_experts=experts)), layer, lambda m, l: None)
    x = make_x(M, H, 3, BF16)
    weights = torch.rand(M, topk, generator=torch.Generator().manual_seed(2)).cuda()
    for n in (E, 2 * E):
        ids = torch.randint(0, n, (M, topk), generator=torch.Generator().manual_seed(n)).cuda()
        emap = None if n == E else torch.cat((torch.full((E,), -1), torch.arange(E))).to(torch.int32).cuda()
        out = torch.full((M + 2, H), 5.0, dtype=BF16, device="cuda")
        experts.apply(out, x, None, None, weights, ids, "silu", n, emap, None, None, None, None, None, False)
        _check(out[:M], x, weights, ids, emap, W13, W2)
        assert bool((out[M:] == 5).all())
        for other in (torch.full((M, H + 8), 5.0, dtype=BF16, device="cuda")[:, :H], torch.cat((x, x))):       # strided rows; the input's own memory
            hidden = other[:M] if other.is_contiguous() else x
            experts.apply(other, hidden, None, None, weights, ids, "silu", n, emap, None, None, None, None, None, False)
            assert torch.equal(other[:M], out[:M])
            assert torch.equal(other[M:], x if other.is_contiguous() else x[:0])
    codes, block = make_weight(1, 48, 64, 6)
    lin = types.SimpleNamespace(weight=P(codes[0]), weight_scale=P(block[0]), input_global_scale_inv=torch.tensor([8.0], device="cuda"),
                                alpha=torch.tensor([0.0625], device="cuda"), output_size_per_partition=48)
    core = va.Nvfp4WeightOnlyLinearCore()
    core.process_weights_after_loading(lin)
    x = make_x(6, 64, 1, BF16, pad=4)                                          # rows that are 8 bytes off
    y = core.apply_weights(lin, x.view(6, 64) if x.is_contiguous() else x, None)
    assert torch.equal(y, (x.double() @ values(codes, block, torch.full((1, 1), 0.5, device="cuda"))[0].T).to(BF16))
