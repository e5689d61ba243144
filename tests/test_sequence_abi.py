"""The sequence operators' entry points refuse null arguments, and their
Python mirror refuses bad configurations, without a GPU."""
import ctypes

import pytest

import vkfft_amd as vk


def test_null_arguments_are_rejected():
    L = vk.lib()
    out = ctypes.c_void_p()
    size = ctypes.c_uint64()
    assert L.vkfx_layer_norm_create(None, None, ctypes.byref(out)) == -7
    assert L.vkfx_linear_attention_create(None, None, ctypes.byref(out)) == -7
    assert L.vkfx_layer_norm_forward(None, 1, None, 0, None, None, None, 0, None, None) == -7
    assert L.vkfx_layer_norm_backward(None, 1, None, 0, None, None, None, 0, None, 0, None, None, None, None) == -7
    assert L.vkfx_linear_attention_forward(None, None, None, None) == -7
    assert L.vkfx_linear_attention_backward(None, None, None, None) == -7
    assert L.vkfx_layer_norm_workspace_bytes(None, ctypes.byref(size)) == -7
    assert L.vkfx_linear_attention_workspace_bytes(None, ctypes.byref(size)) == -7
    assert b"null" in L.vkfx_last_error()
    assert L.vkfx_layer_norm_destroy(None) == 0
    assert L.vkfx_linear_attention_destroy(None) == 0


def test_descriptors_are_laid_out_as_the_header_has_them():
    assert ctypes.sizeof(vk._LayerNormDesc) == 24
    assert ctypes.sizeof(vk._LinearAttentionDesc) == 56
    assert ctypes.sizeof(vk._ForwardArgs) == 16 + 4 * 32 + 3 * 8
    assert ctypes.sizeof(vk._BackwardArgs) == 16 + 7 * 32 + 4 * 8


@pytest.mark.parametrize("config,kind", [
    (vk.LinearAttentionConfig.new(2, 16, 16).with_decay([0.5]), "InputLengthMismatch"),
    (vk.LinearAttentionConfig.new(0, 16, 16), "InvalidArgument"),
    (vk.LinearAttentionConfig.new(2, 16, 16).with_kv_heads(0), "InvalidArgument"),
    (vk.LinearAttentionConfig.new(2, -1, 16), "InvalidArgument"),
    (vk.LinearAttentionConfig.new(2, 16, 16).with_capacity(1, 1 << 31), "InvalidArgument"),
    (vk.LayerNormConfig.new(-1), "InvalidArgument"),
])
def test_bad_configurations(config, kind):
    with pytest.raises(vk.VkFftError) as e:
        config.desc()
    assert e.value.kind == kind


def test_defaults():
    d = vk.LinearAttentionConfig.new(3, 64, 32).desc()
    assert d.kv_heads == 3 and d.scale == 0.125 and [d.decay[i] for i in range(3)] == [1.0] * 3 and not d.gradient
    n = vk.LayerNormConfig.new(8).with_element(vk.Element.BF16).desc()
    assert n.element == n.weight_element == 2


@pytest.mark.parametrize("cls", [vk.LayerNormPlan, vk.LinearAttentionPlan])
@pytest.mark.parametrize("device", [-1, 0, 2])
def test_tensors_of_another_device_are_refused(cls, device):
    class Tensor:
        def get_device(self):
            return device

    plan = cls.__new__(cls)  # a plan of device 1: its place alone, no GPU
    plan.handle, plan._device = None, 1
    with pytest.raises(vk.VkFftError) as e:
        plan._place(Tensor())
    assert e.value.kind == "InvalidArgument"
