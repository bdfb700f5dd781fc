"""patch_vllm's two forms against fake vLLM modules: what is asked for is what is installed, experts and dense layers alike."""
import sys
import types

import pytest
import torch

from test_vllm_adapter_cpu import _fake_moe_layer


@pytest.fixture
def fake_vllm(monkeypatch):
    """Modules of the names that the adapter imports, with vLLM's table of linear kernels."""
    from dgx_vllm_b200 import vllm_adapter as va
    for name in ("VLLM_NVFP4_SPARSE_V7", "B200_NVFP4_WEIGHT_ONLY"):
        monkeypatch.delenv(name, raising=False)
    monkeypatch.setattr(va, "_original_process_weights", None)
    monkeypatch.setattr(va, "_patched_weight_only", False, raising=False)
    made = {}

    def module(name, **attributes):
        m = types.ModuleType(name)
        m.__path__ = []
        for k, v in attributes.items():
            setattr(m, k, v)
        made[name] = m
        monkeypatch.setitem(sys.modules, name, m)
        parent, _, leaf = name.rpartition(".")
        if parent:
            setattr(made[parent], leaf, m)

    class ModelOptNvFp4FusedMoE:
        def process_weights_after_loading(self, layer):
            layer.processed = True

    class NvFp4LinearKernel:
        pass

    class Theirs(NvFp4LinearKernel):
        pass

    key = type("Platform", (), {"name": "CUDA"})()
    table = {"ROCM": [Theirs], key: [Theirs]}
    for name in ("vllm", "vllm.model_executor", "vllm.model_executor.layers", "vllm.model_executor.layers.quantization", "vllm.model_executor.kernels"):
        module(name)
    module("vllm._custom_ops")
    module("vllm.model_executor.layers.quantization.modelopt", ModelOptNvFp4FusedMoE=ModelOptNvFp4FusedMoE)
    module("vllm.model_executor.kernels.linear", _POSSIBLE_NVFP4_KERNELS=table)
    module("vllm.model_executor.kernels.linear.nvfp4")
    module("vllm.model_executor.kernels.linear.nvfp4.base", NvFp4LinearKernel=NvFp4LinearKernel)
    return types.SimpleNamespace(va=va, moe=ModelOptNvFp4FusedMoE, table=table, key=key, base=NvFp4LinearKernel, theirs=Theirs, ops=made["vllm._custom_ops"],
                                 kernels=made["vllm.model_executor.kernels.linear"])


def test_nothing_is_patched_unasked(fake_vllm):
    before = fake_vllm.moe.process_weights_after_loading
    assert fake_vllm.va.patch_vllm() is False
    assert fake_vllm.moe.process_weights_after_loading is before and fake_vllm.table[fake_vllm.key] == [fake_vllm.theirs]


@pytest.mark.parametrize("how", ["argument", "environment", "both"])
def test_weight_only_installs_experts_and_linears(fake_vllm, monkeypatch, how):
    va, seen = fake_vllm.va, []
    monkeypatch.setattr(va, "process_moe_layer_weight_only", lambda m, l, original: seen.append("weight-only"))
    monkeypatch.setattr(va, "process_moe_layer", lambda m, l, original: seen.append("sparse"))
    if how != "argument":
        monkeypatch.setenv("B200_NVFP4_WEIGHT_ONLY", "1")
    assert va.patch_vllm(weight_only=None if how == "environment" else True) is True
    fake_vllm.moe().process_weights_after_loading(types.SimpleNamespace())
    assert seen == ["weight-only"]
    first, *rest = fake_vllm.table[fake_vllm.key]
    assert rest == [fake_vllm.theirs] and issubclass(first, fake_vllm.base) and fake_vllm.table["ROCM"] == [fake_vllm.theirs]
    assert isinstance(first._core, va.Nvfp4WeightOnlyLinearCore) and first.can_implement(None)[0]
    assert hasattr(fake_vllm.ops, "scaled_fp4_quant")
    assert va.patch_vllm(force=True) is True and va.patch_vllm(weight_only=True) is True      # idempotent
    assert fake_vllm.table[fake_vllm.key] == [first, fake_vllm.theirs]
    with pytest.raises(RuntimeError, match="patched already"):
        va.patch_vllm(weight_only=False)


@pytest.mark.parametrize("how", ["argument", "environment", "force", "both variables"])
def test_sparse_form_leaves_the_linear_kernels_alone(fake_vllm, monkeypatch, how):
    va, seen = fake_vllm.va, []
    monkeypatch.setattr(va, "process_moe_layer_weight_only", lambda m, l, original: seen.append("weight-only"))
    monkeypatch.setattr(va, "process_moe_layer", lambda m, l, original: seen.append("sparse"))
    if how in ("environment", "both variables"):
        monkeypatch.setenv("VLLM_NVFP4_SPARSE_V7", "1")
    if how == "both variables":
        monkeypatch.setenv("B200_NVFP4_WEIGHT_ONLY", "1")
    assert va.patch_vllm(force=how == "force", weight_only=False if how == "argument" else None) is True
    fake_vllm.moe().process_weights_after_loading(types.SimpleNamespace())
    assert seen == ["sparse"] and fake_vllm.table[fake_vllm.key] == [fake_vllm.theirs]
    with pytest.raises(RuntimeError, match="patched already"):
        va.patch_vllm(weight_only=True)


def test_weight_only_without_a_table_of_linear_kernels_is_an_error(fake_vllm):
    before = fake_vllm.moe.process_weights_after_loading
    del fake_vllm.kernels._POSSIBLE_NVFP4_KERNELS
    with pytest.raises(RuntimeError, match="quantize their activations"):
        fake_vllm.va.patch_vllm(weight_only=True)
    assert fake_vllm.moe.process_weights_after_loading is before and fake_vllm.va._original_process_weights is None


def test_weight_only_linear_kernel_class(fake_vllm, monkeypatch):
    """The class that vLLM gets: a layer through both of its methods."""
    kernel = fake_vllm.va.linear_kernel_class(weight_only=True)
    monkeypatch.setattr(kernel, "_core", fake_vllm.va.Nvfp4WeightOnlyLinearCore(
        pack_fn=lambda codes, scales, g: float(g), linear_fn=lambda x, w, bias: torch.full((x.shape[0], 8), w)))
    P = lambda t: torch.nn.Parameter(t, requires_grad=False)
    layer = types.SimpleNamespace(weight=P(torch.zeros(8, 16, dtype=torch.uint8)), weight_scale=P(torch.zeros(8, 2, dtype=torch.uint8)),
                                  input_global_scale_inv=torch.tensor([4.0]), alpha=torch.tensor([0.5]), output_size_per_partition=8)
    k = kernel()
    k.process_weights_after_loading(layer)
    y = k.apply_weights(layer, torch.zeros(2, 3, 32))
    assert tuple(y.shape) == (2, 3, 8) and bool((y == 2.0).all())


def test_hook_lets_go_of_the_checkpoint_tensors_before_memory_is_given_back(monkeypatch):
    import weakref
    from dgx_vllm_b200 import vllm_adapter as va
    layer, _, _ = _fake_moe_layer()
    refs, alive = [], []

    def pack(codes, scales, g, gated, device):
        if not gated:
            alive.append([r() is not None for r in refs])           # the first projection's, while the second one's are packed
        refs.extend(weakref.ref(t) for t in (codes, scales, g))
        return "packed"

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: alive.append([r() is not None for r in refs]))
    method = types.SimpleNamespace(moe_mk=types.SimpleNamespace(fused_experts=types.SimpleNamespace(apply=None)))
    assert va.process_moe_layer_weight_only(method, layer, lambda m, l: None, pack_fn=pack, device="cpu", make_apply=lambda a, b: None)
    assert alive == [[False] * 3, [False] * 6]
