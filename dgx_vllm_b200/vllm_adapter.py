"""vLLM adapter: what makes the ops of this package serve a real model.

Sparse MoE experts -- the counterpart of the reference's sparse_kernel patch
(sparse_fp4_kernel/sparse_v7_moe_patch.py:200-358):
  * `make_v7_apply_fn`          the closure assigned as `experts.apply` (its `_make_v7_apply_fn`, :200-232)
  * `process_moe_layer`         clone the checkpoint weights, let vLLM's own process_weights_after_loading run,
                                convert the clones to the 2:4 tensors ON THE GPU (one kernel instead of the
                                reference's Python loop over experts, :96-129), swap `apply`, and replace the
                                original tensors by zero-stride stubs that keep their shapes (:300-326)
  * `patch_vllm`                installs it on ModelOptNvFp4FusedMoE, gated by VLLM_NVFP4_SPARSE_V7=1 like the
                                reference (:334-362), and routes vLLM's dense NVFP4 entry points here
Dense NVFP4 experts with 16-bit activations (what MarlinExperts does, weights as they are in the checkpoint):
  * `make_w4a16_apply_fn`, `process_moe_layer_weight_only`   the same hook over weight_only.W4A16MoE;
                                `patch_vllm(weight_only=True)` or B200_NVFP4_WEIGHT_ONLY=1 installs it in place of the 2:4 one, and
                                makes `linear_kernel_class(weight_only=True)` the first of vLLM's NVFP4 linear kernels
Dense NVFP4 linears:
  * `Nvfp4LinearCore` / `linear_kernel_class()`   an NvFp4LinearKernel (vllm/model_executor/kernels/linear/nvfp4/
                                base.py) whose quantizer and GEMM are this library's;
  * `Nvfp4WeightOnlyLinearCore` / `linear_kernel_class(weight_only=True)`   the same with 16-bit activations

Nothing here imports vLLM at module import time; `patch_vllm` and `linear_kernel_class` do when called."""
from __future__ import annotations

import logging
import os
import time
from typing import Callable, Optional

import torch

logger = logging.getLogger(__name__)

_STUBBED_PARAMS = ("w13_weight", "w2_weight", "w13_weight_scale", "w2_weight_scale", "w13_weight_scale_2",
                   "w2_weight_scale_2")


def make_v7_apply_fn(w13_comp, w13_meta, w13_scale, w13_g_scales, w2_comp, w2_meta, w2_scale, w2_g_scales, inter_size,
                     hidden_size, fused_fn: Optional[Callable] = None):
    """The function vLLM calls in place of MarlinExperts.apply (same 15 positional arguments, no self): writes
    output[:M] and returns output, like v7_apply (sparse_v7_moe_patch.py:216-230).  The weight tensors are validated
    and bound once per expert_map; `fused_fn`, when given, replaces the bound CUDA layer (tests on CPU)."""
    bound = {}

    def layer_for(expert_map):
        key = None if expert_map is None else (expert_map.data_ptr(), expert_map.numel())
        if key not in bound:
            from .sparse_fp4_v7 import FusedSparseMoE
            bound[key] = FusedSparseMoE(w13_comp, w13_meta, w13_scale, w13_g_scales, w2_comp, w2_meta, w2_scale,
                                        w2_g_scales, inter_size, expert_map=expert_map)
        return bound[key]

    def v7_apply(output, hidden_states, w1, w2, topk_weights, topk_ids, activation, global_num_experts, expert_map,
                 a1q_scale, a2_scale, workspace13, workspace2, expert_tokens_meta, apply_router_weight_on_input):
        if fused_fn is not None:
            result = fused_fn(hidden_states, topk_weights.float(), topk_ids, expert_map, w13_comp, w13_meta, w13_scale,
                              w13_g_scales, w2_comp, w2_meta, w2_scale, w2_g_scales, inter_size,
                              apply_router_weight_on_input)
        else:
            if expert_map is not None and not expert_map.is_cuda:
                expert_map = expert_map.to(hidden_states.device)
            result = layer_for(expert_map)(hidden_states, topk_weights, topk_ids,
                                           apply_router_weight_on_input=apply_router_weight_on_input)
        output[:hidden_states.shape[0]] = result.to(output.dtype)
        return output

    return v7_apply


def _zero_stride_stub(param) -> int:
    """param.data := a one-element tensor viewed with the original shape (all strides 0); returns the bytes freed.
    vLLM still reads the shapes of these parameters (moe_problem_size), never their contents."""
    data = param.data
    shape = tuple(data.shape)
    freed = data.numel() * data.element_size()
    stub = torch.zeros(1, device=data.device, dtype=data.dtype)
    param.data = stub.as_strided(shape, [0] * len(shape))
    return freed


def process_moe_layer(method, layer, original: Callable, convert_fn: Optional[Callable] = None, device=None,
                      make_apply: Callable = make_v7_apply_fn) -> bool:
    """What the patched ModelOptNvFp4FusedMoE.process_weights_after_loading does for one layer
    (sparse_v7_moe_patch.py:243-331).  `original(method, layer)` is vLLM's own routine; `convert_fn(weights [E,N,K/2],
    scales [E,N,K/16], g_scales [E], device=) -> (comp_T, meta_T, scale_T, g)` defaults to the CUDA converter.
    Returns True when `apply` was replaced."""
    t0 = time.time()
    # 1. the checkpoint tensors, before the repacking of the original routine destroys them
    src = {name: getattr(layer, name).data.clone() for name in _STUBBED_PARAMS}
    E, inter2, hidden_half = src["w13_weight"].shape
    inter_size, hidden_size = inter2 // 2, hidden_half * 2
    # 2. vLLM's own processing (builds the modular kernel whose experts object gets the new apply)
    original(method, layer)
    experts = getattr(getattr(method, "moe_mk", None), "fused_experts", None)
    if experts is None:
        logger.warning("[b200 sparse] moe_mk.fused_experts not found: layer left on vLLM's own kernels")
        return False
    # 3. 2:4 conversion on the device
    if convert_fn is None:
        from .sparse_fp4_v7 import convert_weight_batch_to_v7 as convert_fn
    if device is None:
        device = src["w13_weight"].device if src["w13_weight"].is_cuda else "cuda"
    gs = lambda t: t[:, 0] if t.dim() > 1 else t
    w13 = convert_fn(src["w13_weight"], src["w13_weight_scale"], gs(src["w13_weight_scale_2"]), device=device)
    w2 = convert_fn(src["w2_weight"], src["w2_weight_scale"], gs(src["w2_weight_scale_2"]), device=device)
    del src
    # 4. the closure shadows the class method on this experts instance; the originals shrink to shape-only stubs
    experts.apply = make_apply(*w13, *w2, inter_size, hidden_size)
    freed = sum(_zero_stride_stub(getattr(layer, name)) for name in _STUBBED_PARAMS if hasattr(layer, name))
    if torch.cuda.is_available():
        torch.cuda.empty_cache()
    logger.info("[b200 sparse] %d experts converted in %.1f s, %.1f MB of repacked weights released", E,
                time.time() - t0, freed / 1e6)
    return True


def make_w4a16_apply_fn(w13, w2, fused_fn: Optional[Callable] = None):
    """The function vLLM calls in place of MarlinExperts.apply (same 15 positional arguments, no self) over weights packed by
    weight_only.pack_nvfp4_weight: writes output[:M] and returns output.  `fused_fn(hidden, topk_weights, topk_ids, expert_map, on_input)`,
    when given, replaces the CUDA layer (tests on CPU)."""
    layer = []

    def w4a16_apply(output, hidden_states, w1, w2_, topk_weights, topk_ids, activation, global_num_experts, expert_map,
                    a1q_scale, a2_scale, workspace13, workspace2, expert_tokens_meta, apply_router_weight_on_input):
        if str(getattr(activation, "value", activation)).lower() != "silu":
            raise RuntimeError(f"weight-only experts apply SiLU(gate) * up, not {activation}")
        if fused_fn is not None:
            result = fused_fn(hidden_states, topk_weights.float(), topk_ids, expert_map, apply_router_weight_on_input)
        else:
            if expert_map is not None and not expert_map.is_cuda:
                expert_map = expert_map.to(hidden_states.device)
            if not layer:
                from .weight_only import W4A16MoE
                layer.append(W4A16MoE(w13, w2))
            hidden_states = hidden_states.contiguous()
            if hidden_states.data_ptr() % 16:
                hidden_states = hidden_states.clone()
            # straight into the output's rows, where they can be written as they are
            rows = output[:hidden_states.shape[0]]
            direct = (rows.shape == hidden_states.shape and rows.is_contiguous() and rows.data_ptr() % 16 == 0
                      and rows.dtype in (torch.bfloat16, torch.float16, torch.float32)
                      and rows.untyped_storage().data_ptr() != hidden_states.untyped_storage().data_ptr())
            result = layer[0](hidden_states, topk_weights, topk_ids, apply_router_weight_on_input,
                              out=rows if direct else None, expert_map=expert_map)
            if direct:
                return output
        output[:hidden_states.shape[0]] = result.to(output.dtype)
        return output

    return w4a16_apply


def process_moe_layer_weight_only(method, layer, original: Callable, pack_fn: Optional[Callable] = None, device=None,
                                  make_apply: Callable = make_w4a16_apply_fn) -> bool:
    """process_moe_layer without the pruning: the checkpoint tensors are packed as they are.  `pack_fn(codes [E,N,K/2], scales
    [E,N,K/16], g_scales, gated=, device=)` defaults to weight_only.pack_nvfp4_weight; gate and up rows keep a factor each where the
    checkpoint has two.  Returns True when `apply` was replaced."""
    src = {name: getattr(layer, name).data.clone() for name in _STUBBED_PARAMS}
    original(method, layer)
    experts = getattr(getattr(method, "moe_mk", None), "fused_experts", None)
    if experts is None:
        logger.warning("[b200 weight-only] moe_mk.fused_experts not found: layer left on vLLM's own kernels")
        return False
    if pack_fn is None:
        from .weight_only import pack_nvfp4_weight as pack_fn
    if device is None:
        device = src["w13_weight"].device if src["w13_weight"].is_cuda else "cuda"
    one = lambda g: g[:, 0] if g.dim() > 1 else g
    n_experts = src["w13_weight"].shape[0]
    # the copies of a projection go as soon as it is packed: a layer is held twice at most
    w13 = pack_fn(src.pop("w13_weight"), src.pop("w13_weight_scale"), src.pop("w13_weight_scale_2"), gated=True, device=device)
    w2 = pack_fn(src.pop("w2_weight"), src.pop("w2_weight_scale"), one(src.pop("w2_weight_scale_2")), gated=False, device=device)
    experts.apply = make_apply(w13, w2)
    freed = sum(_zero_stride_stub(getattr(layer, name)) for name in _STUBBED_PARAMS if hasattr(layer, name))
    if torch.cuda.is_available():
        torch.cuda.empty_cache()
    logger.info("[b200 weight-only] %d experts packed, %.1f MB of repacked weights released", n_experts, freed / 1e6)
    return True


_original_process_weights = None
_patched_weight_only = False


def _prefer_weight_only_linears() -> None:
    """The weight-only linear kernel becomes the first that vLLM tries for a dense NVFP4 layer on CUDA."""
    import vllm.model_executor.kernels.linear as kernels
    table = getattr(kernels, "_POSSIBLE_NVFP4_KERNELS", {})
    platforms = [p for p in table if getattr(p, "name", p) == "CUDA"]
    if not platforms:
        raise RuntimeError("vLLM's table of NVFP4 linear kernels was not found: its dense layers would quantize their activations")
    table[platforms[0]] = [linear_kernel_class(weight_only=True), *table[platforms[0]]]


def patch_vllm(force: bool = False, weight_only: Optional[bool] = None) -> bool:
    """Install the hook on vLLM's ModelOptNvFp4FusedMoE and route its dense NVFP4 ops to this library; call it before the model is built.  Like
    the reference's module it acts only when VLLM_NVFP4_SPARSE_V7=1, or B200_NVFP4_WEIGHT_ONLY=1 for experts and dense layers whose weights are
    neither pruned nor met by quantized activations, or when the caller says so: force=True, or weight_only True or False, which chooses
    between the two forms.  Idempotent; a second call for the other form raises."""
    global _original_process_weights, _patched_weight_only
    asked = {name: os.environ.get(name, "0") == "1" for name in ("VLLM_NVFP4_SPARSE_V7", "B200_NVFP4_WEIGHT_ONLY")}
    if not force and weight_only is None and not any(asked.values()):
        return False
    if _original_process_weights is not None:
        if weight_only not in (None, _patched_weight_only):
            raise RuntimeError(f"vLLM is patched already, for {'weight-only' if _patched_weight_only else 'sparse 2:4'} experts")
        return True
    if weight_only is None:
        weight_only = asked["B200_NVFP4_WEIGHT_ONLY"] and not asked["VLLM_NVFP4_SPARSE_V7"]
    from vllm.model_executor.layers.quantization.modelopt import ModelOptNvFp4FusedMoE

    from .torch_ops import install_into_vllm
    if weight_only:
        _prefer_weight_only_linears()
    _original_process_weights = ModelOptNvFp4FusedMoE.process_weights_after_loading
    _patched_weight_only = bool(weight_only)

    process = process_moe_layer_weight_only if weight_only else process_moe_layer

    def patched(self, layer):
        process(self, layer, _original_process_weights)

    ModelOptNvFp4FusedMoE.process_weights_after_loading = patched
    install_into_vllm()
    logger.info("[b200] vLLM patched: %s and dense NVFP4 ops run on libb200nvfp4",
                "weight-only MoE experts, weight-only linears" if weight_only else "sparse 2:4 MoE experts")
    return True


class Nvfp4LinearCore:
    """process_weights_after_loading / apply_weights of a dense NVFP4 linear on this library's quantizer and GEMM
    (the two methods an NvFp4LinearKernel must provide).  The layer carries vLLM's attribute names: weight
    [N,K/2] u8, weight_scale [N,K/16] e4m3 (linear in the checkpoint), input_global_scale_inv (= 448*6/amax),
    alpha (= 1 / (input scale * weight scale)), output_size_per_partition."""

    def __init__(self, swizzle_fn: Optional[Callable] = None, quant_fn: Optional[Callable] = None,
                 mm_fn: Optional[Callable] = None):
        self._swizzle, self._quant, self._mm = swizzle_fn, quant_fn, mm_fn

    def process_weights_after_loading(self, layer) -> None:
        swz = self._swizzle or swizzle_blockscale
        layer.weight_scale = torch.nn.Parameter(swz(layer.weight_scale.data), requires_grad=False)
        layer.weight = torch.nn.Parameter(layer.weight.data.contiguous(), requires_grad=False)

    def apply_weights(self, layer, x: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        from . import ops
        out_shape = [*x.shape[:-1], layer.output_size_per_partition]
        x2 = x.reshape(-1, x.shape[-1])
        if self._quant is None and self._mm is None:
            # quantizer and GEMM queued by one library call
            out = ops.nvfp4_linear(x2, layer.input_global_scale_inv, layer.weight, layer.weight_scale, layer.alpha)
        else:
            quant, mm = self._quant or ops.scaled_fp4_quant, self._mm or ops.cutlass_scaled_fp4_mm
            codes, sf = quant(x2, layer.input_global_scale_inv, True)
            out = mm(codes, layer.weight, sf, layer.weight_scale, layer.alpha, x.dtype)
        if bias is not None:
            out = out + bias
        return out.view(*out_shape)


class Nvfp4WeightOnlyLinearCore:
    """process_weights_after_loading / apply_weights of a dense NVFP4 linear with 16-bit activations.  The layer carries the attributes that
    Nvfp4LinearCore's does; alpha times input_global_scale_inv is the weight's own factor, the activations' global scale is not used."""

    def __init__(self, pack_fn: Optional[Callable] = None, linear_fn: Optional[Callable] = None):
        self._pack, self._linear = pack_fn, linear_fn

    def process_weights_after_loading(self, layer) -> None:
        if self._pack is None:
            from .weight_only import pack_nvfp4_weight
            pack = pack_nvfp4_weight
        else:
            pack = self._pack
        g = layer.alpha.detach().float() * layer.input_global_scale_inv.detach().float()
        layer.w4a16_weight = pack(layer.weight.data, layer.weight_scale.data, g.reshape(1))
        for name in ("weight", "weight_scale"):
            _zero_stride_stub(getattr(layer, name))

    def apply_weights(self, layer, x: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        out_shape = [*x.shape[:-1], layer.output_size_per_partition]
        x2 = x.reshape(-1, x.shape[-1])
        if self._linear is None:
            from .weight_only import w4a16_linear as linear
            if x2.stride(-1) != 1 or x2.data_ptr() % 16 or (x2.shape[0] > 1 and (x2.stride(0) % 8 or x2.stride(0) < x2.shape[1])):
                x2 = x2.clone(memory_format=torch.contiguous_format)          # rows of some slice that are not 16-byte aligned, or one row many times
        else:
            linear = self._linear
        return linear(x2, layer.w4a16_weight, bias).view(*out_shape)


def swizzle_blockscale(sf_linear: torch.Tensor) -> torch.Tensor:
    """[rows, K/16] e4m3 block scales -> the padded 128x4 tile layout the GEMM reads (swizzle_blockscale,
    vllm/model_executor/layers/quantization/utils/nvfp4_utils.py:38-51), on the GPU."""
    from . import _lib
    from ._torch_util import ptr, require, require_cuda, stream_ptr
    dev = require_cuda(sf_linear)
    require(sf_linear.dim() == 2 and sf_linear.element_size() == 1 and sf_linear.is_contiguous(),
            "block scales must be a contiguous [rows, K/16] one-byte tensor")
    rows, kb = sf_linear.shape
    out = torch.empty(((rows + 127) // 128 * 128, (kb + 3) // 4 * 4), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().b200fp4_sf_swizzle(ptr(sf_linear), rows, kb, ptr(out), stream_ptr(dev)), "swizzle_blockscale")
    return out.view(torch.float8_e4m3fn)


def linear_kernel_class(weight_only: bool = False):
    """An NvFp4LinearKernel subclass for vLLM's kernel registry (imports vLLM); weight_only: with 16-bit activations."""
    from vllm.model_executor.kernels.linear.nvfp4.base import NvFp4LinearKernel

    class B200NvFp4LinearKernel(NvFp4LinearKernel):
        _core = Nvfp4WeightOnlyLinearCore() if weight_only else Nvfp4LinearCore()

        @classmethod
        def is_supported(cls, compute_capability=None):
            from . import _lib
            ok = _lib.lib().b200fp4_has_hardware_acceleration() == 1
            return (True, None) if ok else (False, "needs an sm_100 device")

        @classmethod
        def can_implement(cls, config):
            return True, None

        def process_weights_after_loading(self, layer):
            self._core.process_weights_after_loading(layer)

        def apply_weights(self, layer, x, bias=None):
            return self._core.apply_weights(layer, x, bias)

    return B200NvFp4LinearKernel


if os.environ.get("B200_NVFP4_AUTOPATCH", "0") == "1":
    patch_vllm()
