"""Timed cases of the weight-only operators: NVFP4 weights (E2M1 codes, an E4M3 scale for each 16 of K, one f32 scale for each
matrix) with activations that stay in 16 bits.

    linear   weight_only.w4a16_linear   y = x W^T + bias of a dense layer, from one token to a full prompt
    moe      weight_only.W4A16MoE       a whole mixture-of-experts layer for a decode batch: gate and up projections, SiLU(gate) * up,
                                        down projection, router-weighted sum

With `own` false `run` computes the same in elementary torch operations, in 32 bits, rounded once at the end.  Inputs are seeded synthetic
tensors: activations N(0,1) with some large channels, weights with the codes and block scales that N(0, 0.02) quantizes to."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# Parts of 256 in which each magnitude occurs among normal values that are quantized in blocks of 16, scaled to their largest.
FREQUENCIES = (24, 46, 41, 36, 46, 31, 20, 12)

# What no drawn case exceeds: the largest listed one of its kind.
MAX_LINEAR = 4096 * 14336 * 4096
MAX_WEIGHT = 14336 * 4096
MAX_EXPERTS = 512 * 2048 * 512
MAX_PAIRS = 128 * 10 * 2048 * 512


def listed():
    return [
        # one user decoding, a small projection: launch and latency are all there is
        dict(name="linear_m1_2048", kind="linear", M=1, N=2048, K=2048, dtype="bf16", out="bf16", bias=False, pad=0),
        # one user decoding, a wide MLP projection: the weight is read once for one token
        dict(name="linear_m1_14336", kind="linear", M=1, N=14336, K=4096, dtype="bf16", out="bf16", bias=False, pad=0),
        # a few users through a layer of no round width whose input is a slice of a wider tensor; f16 model with a bias
        dict(name="linear_ragged_m7", kind="linear", M=7, N=3001, K=4144, dtype="f16", out="f16", bias=True, pad=16),
        # a decode batch through the long projection back to the hidden size
        dict(name="linear_m32_down", kind="linear", M=32, N=4096, K=14336, dtype="bf16", out="bf16", bias=False, pad=0),
        # logits of a decode batch, kept in f32
        dict(name="linear_m16_logits", kind="linear", M=16, N=28672, K=2048, dtype="bf16", out="f32", bias=False, pad=0),
        # a short prompt of no round length
        dict(name="linear_m333", kind="linear", M=333, N=4096, K=4096, dtype="bf16", out="bf16", bias=False, pad=0),
        # a full prompt: bound by the tensor cores
        dict(name="linear_m4096", kind="linear", M=4096, N=14336, K=4096, dtype="bf16", out="bf16", bias=False, pad=0),
        # one user decoding: ten experts of 512 for one token
        dict(name="moe_b1", kind="moe", M=1, E=512, H=2048, I=512, topk=10, dtype="bf16", parallel=1),
        # few wide experts, every one of which several tokens meet; f16 model, odd batch
        dict(name="moe_b29_wide", kind="moe", M=29, E=8, H=4096, I=4096, topk=2, dtype="f16", parallel=1),
        # the usual decode batch: about half of the experts are read for a few tokens each
        dict(name="moe_b32", kind="moe", M=32, E=512, H=2048, I=512, topk=10, dtype="bf16", parallel=1),
        # one of four expert-parallel ranks: three of four pairs are some other rank's
        dict(name="moe_b61_rank", kind="moe", M=61, E=64, H=2048, I=768, topk=8, dtype="bf16", parallel=4),
        # the largest decode batch: nearly every expert is read
        dict(name="moe_b128", kind="moe", M=128, E=512, H=2048, I=512, topk=10, dtype="bf16", parallel=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: token counts, widths, depths and expert counts spread over their logarithm, odd ones among them."""
    dtype = rng.choice(("bf16", "bf16", "f16"))
    while rng.random() < 0.55:
        M, N, K = _log(rng, 1, 4096), _log(rng, 256, 28672), 16 * _log(rng, 32, 896)
        if N * K <= MAX_WEIGHT and M * N * K <= MAX_LINEAR:
            return dict(kind="linear", M=M, N=N, K=K, dtype=dtype, out=rng.choice((dtype, dtype, dtype, "f32")), bias=rng.random() < 0.3,
                        pad=rng.choice((0, 0, 8, 64)))
    while True:
        M, E, topk = _log(rng, 1, 128), _log(rng, 8, 512), rng.randint(1, 10)
        H, I, parallel = 16 * _log(rng, 64, 256), 16 * _log(rng, 8, 256), rng.choice((1, 1, 1, 2, 4))
        if topk <= E and E * H * I <= MAX_EXPERTS and M * topk * H * I <= MAX_PAIRS:
            return dict(kind="moe", M=M, E=E, H=H, I=I, topk=topk, dtype=dtype, parallel=parallel)


def _codes(shape, gen):
    """Packed E2M1 codes, two in a byte (the even element in the low nibble)."""
    table = torch.repeat_interleave(torch.arange(8, dtype=torch.uint8), torch.tensor(FREQUENCIES)).cuda()

    def nibbles():
        r = torch.randint(0, 1 << 31, shape, generator=gen, device="cuda", dtype=torch.int32)
        return table[r & 255] | ((r >> 5) & 8).to(torch.uint8)

    low = nibbles()
    return low | (nibbles() << 4)


def _weights(E, N, K, gen):
    """E matrices [N, K] as a checkpoint has them: codes [E,N,K/2], block scales [E,N,K/16] in E4M3, one f32 scale each."""
    codes = torch.cat([_codes((min(64, E - e), N, K // 2), gen) for e in range(0, E, 64)])
    top = torch.randn(E, N, K // 16, generator=gen, device="cuda").mul_(0.4).add_(1.75).clamp_(0.7, 4.5)
    block = top.mul_(448.0 / 5.5).to(torch.float8_e4m3fn)
    scale = 0.02 * 5.5 / (6.0 * 448.0) * (0.75 + 0.5 * torch.rand(E, generator=gen, device="cuda"))
    return codes, block, scale


def _activations(M, K, pad, dtype, gen):
    loud = 1.0 + 15.0 * (torch.rand(K + pad, generator=gen, device="cuda") < 0.01).float()
    x = torch.randn(M, K + pad, generator=gen, device="cuda") * loud
    return x.to(dtype)[:, :K]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed * 1000003 + 17)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        codes, block, scale = _weights(1, N, K, gen)
        state = dict(kind="linear", x=_activations(M, K, case["pad"], dtype, gen), out=DTYPES[case["out"]], codes=codes[0], block=block[0],
                     scale=scale, bias=torch.randn(N, generator=gen, device="cuda").to(dtype) if case["bias"] else None)
        if own:
            from dgx_vllm_b200.weight_only import pack_nvfp4_weight
            state["weight"] = pack_nvfp4_weight(state["codes"], state["block"], scale)
        return state
    M, E, H, I, topk, parallel = (case[k] for k in ("M", "E", "H", "I", "topk", "parallel"))
    state = dict(kind="moe", x=_activations(M, H, 0, dtype, gen), w13=_weights(E, 2 * I, H, gen), w2=_weights(E, H, I, gen), map=None)
    # the router of all ranks: softmax over every expert, the topk largest, renormalised; this rank holds `E` of them
    chosen = torch.randn(M, E * parallel, generator=gen, device="cuda").softmax(-1).topk(topk)
    state["weights"] = chosen.values / chosen.values.sum(-1, keepdim=True)
    state["ids"] = chosen.indices.to(torch.int32)
    if parallel > 1:
        state["map"] = torch.full((E * parallel,), -1, dtype=torch.int32, device="cuda")
        state["map"][E:2 * E] = torch.arange(E, dtype=torch.int32, device="cuda")
    if own:
        from dgx_vllm_b200.weight_only import W4A16MoE, pack_nvfp4_weight
        state["layer"] = W4A16MoE(pack_nvfp4_weight(*state["w13"], gated=True), pack_nvfp4_weight(*state["w2"]), expert_map=state["map"])
    return state


def _values(codes, block, scale):
    """f32 values of packed codes [..., K/2] with block scales [..., K/16] and a scale that broadcasts to [..., 1, 1]."""
    signed = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    pairs = torch.stack((signed.repeat(16), signed.repeat_interleave(16)), dim=1)         # [byte, (low, high)]
    v = torch.index_select(pairs, 0, codes.reshape(-1).int()).view(*block.shape, 16)
    v.mul_((block.float() * scale[..., None, None])[..., None])
    return v.view(*codes.shape[:-1], codes.shape[-1] * 2)


def _linear(s):
    y = s["x"].float() @ _values(s["codes"], s["block"], s["scale"][0]).T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["out"])


def _moe(s):
    """The chosen experts' matrices are gathered for each pair of token and expert."""
    ids, weights = s["ids"].long(), s["weights"]
    if s["map"] is not None:
        ids = s["map"].long()[ids]
        weights = weights * (ids >= 0)
        ids = ids.clamp(min=0)
    x = s["x"].float()
    gate_up = torch.matmul(_values(*(t[ids] for t in s["w13"])), x[:, None, :, None]).squeeze(-1)      # [M, topk, 2I]
    gate, up = gate_up.chunk(2, dim=-1)
    act = gate / (1.0 + torch.exp(-gate)) * up
    y = torch.matmul(_values(*(t[ids] for t in s["w2"])), act[..., None]).squeeze(-1)                  # [M, topk, H]
    return (y * weights[..., None]).sum(1).to(s["x"].dtype)


def run(state):
    if own:
        if state["kind"] == "linear":
            from dgx_vllm_b200.weight_only import w4a16_linear
            return w4a16_linear(state["x"], state["weight"], state["bias"], out_dtype=state["out"])
        return state["layer"](state["x"], state["weights"], state["ids"])
    return _linear(state) if state["kind"] == "linear" else _moe(state)


def work(case):
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        size = 4 if case["out"] == "f32" else 2
        return {"bytes": N * K * 9 // 16 + 2 * M * K + size * M * N + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    M, E, H, I, topk, parallel = (case[k] for k in ("M", "E", "H", "I", "topk", "parallel"))
    read = E * (1.0 - (1.0 - topk / (E * parallel)) ** M)            # experts of this rank that at least one token chooses, as expected
    return {"bytes": int(read * 3 * H * I * 9 / 16) + 4 * M * H + 8 * M * topk, "flops": int(2 * (M * topk / parallel) * 3 * H * I)}


def _exact_matrix(codes, block, scale):
    """A matrix [N, K] in 64 bits from the fields of its codes: sign, two bits of exponent, one of mantissa."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).to(torch.int32)
    e, m = (c >> 1) & 3, (c & 1).double()
    size = torch.where(e == 0, m * 0.5, torch.exp2(e.double() - 1.0) * (1.0 + 0.5 * m))
    b = block.view(torch.uint8).to(torch.int32)
    be, bm = (b >> 3) & 15, (b & 7).double() / 8.0
    factor = torch.where(be == 0, torch.exp2(torch.full_like(bm, -6.0)) * bm, torch.exp2(be.double() - 7.0) * (1.0 + bm))
    return torch.where(c >= 8, -size, size) * factor.repeat_interleave(16, dim=-1) * scale.double()


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "linear":
        y = torch.einsum("mk,nk->mn", s["x"].double(), _exact_matrix(s["codes"], s["block"], s["scale"][0]))
        return y if s["bias"] is None else y + s["bias"].double()
    x, out = s["x"].double(), torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    ids = s["ids"].long() if s["map"] is None else s["map"].long()[s["ids"].long()]
    I = case["I"]
    for e in range(case["E"]):
        token, place = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        w13, w2 = (_exact_matrix(*(t[e] for t in s[k])) for k in ("w13", "w2"))
        h = torch.einsum("pk,nk->pn", x[token], w13)
        act = h[:, :I] * torch.sigmoid(h[:, :I]) * h[:, I:]
        out.index_add_(0, token, torch.einsum("pi,hi->ph", act, w2) * s["weights"][token, place].double()[:, None])
    return out
