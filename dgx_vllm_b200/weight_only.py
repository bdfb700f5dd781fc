"""Weight-only NVFP4: 4-bit weights as the checkpoint has them, activations in 16 bits.

The reference serves its NVFP4 model this way (weight-only linears and experts, README.md:52-54, OPTIMIZATIONS.md:28,47), through
kernels that are not its own.  Against the other operators of this package: `ops.nvfp4_linear` and `grouped_moe.nvfp4_moe_prefill` quantize
the activations to 4 bits as well, `sparse_fp4_v7.FusedSparseMoE` takes weights pruned to 2:4; here nothing of a weight or an
activation is dropped.  Weights are laid out once, when they are loaded, by `pack_nvfp4_weight`:

    w = pack_nvfp4_weight(codes, block_scale, g_scale)             # [N,K/2] u8, [N,K/16] e4m3, one f32
    y = w4a16_linear(x, w, bias)                                   # x [M,K] bf16/f16, any M

    layer = W4A16MoE(pack_nvfp4_weight(w13, w13_scale, w13_g, gated=True), pack_nvfp4_weight(w2, w2_scale, w2_g))
    out = layer(hidden, *moe_router(hidden, gate, topk))           # a decode batch
"""
from __future__ import annotations

import torch

from . import _lib
from ._torch_util import WS_W4A16_STATUS, ptr, require, require_cuda, status_word, stream_ptr


class PackedNvfp4Weight:
    """E matrices [N, K] in the kernels' layout: `packed` (u8), `g_scale` (f32, [E]; [E, 2] for gate and up rows), `E`, `N`, `K`, `gated`."""

    __slots__ = ("packed", "g_scale", "E", "N", "K", "gated")

    def __init__(self, packed, g_scale, E, N, K, gated):
        self.packed, self.g_scale, self.E, self.N, self.K, self.gated = packed, g_scale, E, N, K, gated


def pack_nvfp4_weight(codes: torch.Tensor, block_scale: torch.Tensor, g_scale: torch.Tensor, *, gated: bool = False,
                      device="cuda") -> PackedNvfp4Weight:
    """A checkpoint's NVFP4 weight -> the layout of w4a16_linear and W4A16MoE, on the GPU in one launch.

    codes [N,K/2] or [E,N,K/2] uint8 (two E2M1 codes a byte, the even k in the low nibble), block_scale [.., N, K/16] e4m3, linear;
    g_scale the factor of a matrix's values, one or [E] f32 (a checkpoint's weight_scale_2; the reciprocal of the global scale that
    scaled_fp4_quant takes).  gated: the N rows are N/2 gate rows and then N/2 up rows of a layer's first projection, which may
    have a factor each ([E, 2]).  K a multiple of 16, any N.  Tensors elsewhere are copied to `device`.  NaN scales are refused (this
    reads the scales back once)."""
    dev = codes.device if codes.is_cuda else torch.device(device)
    require(dev.type == "cuda", "b200 nvfp4 ops take CUDA tensors only (there is no CPU path)")
    require(codes.dim() in (2, 3) and codes.dtype == torch.uint8, "codes must be [N,K/2] or [E,N,K/2] uint8")
    require(block_scale.dtype in (torch.uint8, torch.float8_e4m3fn), "block_scale must be float8_e4m3fn (or its bytes)")
    E, N, K = (codes.shape[0] if codes.dim() == 3 else 1), codes.shape[-2], codes.shape[-1] * 2
    require(E >= 1 and N >= 1 and K >= 16 and K % 16 == 0, "K must be a multiple of 16")
    require(tuple(block_scale.shape) == tuple(codes.shape[:-1]) + (K // 16,), "block_scale must be [.., N, K/16]")
    require(not gated or N % 2 == 0, "a gated weight has as many gate rows as up rows")
    g = g_scale.detach().to(device=dev, dtype=torch.float32)
    if gated:
        require(g.numel() in (E, 2 * E), "g_scale must be one f32 a matrix, or one for its gate and one for its up rows")
        g = g.reshape(E, -1).expand(E, 2).contiguous()
    else:
        require(g.numel() == E, "g_scale must be one f32 a matrix")
        g = g.reshape(E).contiguous()
    codes = codes.to(dev).contiguous()
    sf = block_scale.to(dev).contiguous().view(torch.uint8)
    with torch.cuda.device(dev):
        if not torch.cuda.is_current_stream_capturing():
            require(not bool(((sf & 0x7F) == 0x7F).any()), "block_scale holds NaN")
        L = _lib.lib()
        packed = torch.empty(L.b200fp4_w4a16_packed_bytes(E, N, K, int(gated)), dtype=torch.uint8, device=dev)
        _lib.check(L.b200fp4_w4a16_pack(ptr(codes), ptr(sf), E, N, K, int(gated), ptr(packed), stream_ptr(dev)), "pack_nvfp4_weight")
    return PackedNvfp4Weight(packed, g, E, N, K, bool(gated))


def w4a16_linear(x: torch.Tensor, weight: PackedNvfp4Weight, bias: torch.Tensor | None = None, *, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[M,N] = x @ W^T (+ bias) with the weight's exact values and f32 sums, rounded once.

    x [M,K] bf16 or f16: unit inner stride, rows 16-byte aligned (they may be strided); bias [N] bf16, f16 or f32; out contiguous
    [M,N] and not in x's memory, or out_dtype bf16, f16 or f32 (the dtype of x by default)."""
    require(weight.E == 1 and not weight.gated, "w4a16_linear takes one matrix that is not packed gated")
    return _lib.host().w4a16_linear(x, weight.packed, weight.g_scale, weight.N, weight.K, bias, out, out_dtype)


def last_w4a16_status(device=None) -> int:
    """Status word of the most recent w4a16_linear or W4A16MoE on the current stream of `device`: 0, or the code of a bounded wait that ran
    out (that call's result is then not valid), or 63 where a weight was packed for other sizes than the call's (every row of
    the result has NaN then; only a custom op or a C caller can name other sizes).  A graph leaves it where the stream that it was captured on has it.  Synchronises."""
    return status_word(device, WS_W4A16_STATUS)


class W4A16MoE:
    """One mixture-of-experts layer over weight-only NVFP4 experts, its weights bound once: gate/up projection, SiLU(gate) * up, down
    projection, router-weighted sum, in two launches.  The counterpart of FusedSparseMoE for weights that are not pruned.

    w13 [E, 2I, H] packed gated, w2 [E, H, I] packed; expert_map [global_E] int32 maps the router's ids to local experts (-1: not here)
    or None.  H and I are multiples of 16.  Meant for decode batches: up to 2048 (token, expert) pairs a pass over the
    weights, more in turns."""

    def __init__(self, w13: PackedNvfp4Weight, w2: PackedNvfp4Weight, expert_map: torch.Tensor | None = None):
        self.E, self.H, self.I = w13.E, w13.K, w2.K
        require(w13.gated and not w2.gated, "w13 must be packed gated and w2 not")
        require(w13.N == 2 * self.I and w2.N == self.H and w2.E == self.E, "w13 must be [E, 2I, H] and w2 [E, H, I]")
        require(self.H % 16 == 0 and self.I % 16 == 0, "H and I must be multiples of 16")
        self.device = require_cuda(w13.packed, w13.g_scale, w2.packed, w2.g_scale)
        self._weights = (w13.packed, w13.g_scale, w2.packed, w2.g_scale)
        self._sizes = (self.H, self.I, self.E)
        self._map = self._as_map(expert_map)
        self._call = _lib.host().w4a16_moe

    @staticmethod
    def _as_map(expert_map):
        return None if expert_map is None or expert_map.numel() == 0 else expert_map.to(torch.int32).contiguous()

    def __call__(self, hidden_states: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
                 apply_router_weight_on_input: bool = False, out: torch.Tensor | None = None,
                 expert_map: torch.Tensor | None = None) -> torch.Tensor:
        """hidden_states [M,H] bf16/f16, topk_weights [M,topk] f32, topk_ids [M,topk] int32 -> [M,H] in the activation dtype (or in `out`'s,
        which may also be f32; out may be hidden_states itself).  Pairs whose expert is not here add nothing.  expert_map: in place of
        the layer's own."""
        emap = self._map if expert_map is None else self._as_map(expert_map)
        return self._call(*self._weights, emap, *self._sizes, hidden_states, topk_weights, topk_ids, apply_router_weight_on_input, out)
