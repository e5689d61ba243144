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


class _Tensor:
    """What the plans ask of a tensor, without a GPU."""
    def __init__(self, *shape, dtype=None, device=0, address=4096, stride=None):
        import torch
        self.shape, self.dtype, self._device, self._address = torch.Size(shape), dtype or torch.float32, device, address
        self._stride = stride or tuple(int(n) for n in torch.empty(shape, device="meta").stride())

    def get_device(self):
        return self._device

    def stride(self):
        return self._stride

    def data_ptr(self):
        return self._address

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def size(self, i):
        return self.shape[i]


class _Context:
    """A context whose library takes every call and remembers it."""
    def __init__(self):
        import types
        self.handle, self.device_index, self._live_plans, self.calls = 1, 0, set(), []

        def entry(name):
            return lambda *a: self.calls.append((name, a)) or 0

        names = [f"vkfx_{k}_{f}" for k in ("layer_norm", "linear_attention")
                 for f in ("create", "destroy", "workspace_bytes", "forward", "backward")]
        self._L = types.SimpleNamespace(**{n: entry(n) for n in names})

    def plan(self, config):
        p = (vk.LayerNormPlan if isinstance(config, vk.LayerNormConfig) else vk.LinearAttentionPlan)(self, config)
        p._current = lambda device: 0
        del self.calls[:]
        return p


def test_a_plan_keeps_the_sizes_it_was_made_with():
    """The caller's configuration may change afterwards; the plan's kernels do not."""
    ctx = _Context()
    config = vk.LayerNormConfig.new(16)
    plan = ctx.plan(config)
    config.width = 8
    config.with_element(vk.Element.BF16)
    w = _Tensor(8)
    for f in (lambda: plan.forward_tensors(_Tensor(4, 8), w, w, _Tensor(4, 8)),
              lambda: plan.backward_tensors(_Tensor(4, 8), w, _Tensor(4, 2), _Tensor(4, 8), _Tensor(4, 8), w, w)):
        with pytest.raises(vk.VkFftError) as e:
            f()
        assert e.value.kind == "InputLengthMismatch"
    assert not ctx.calls
    w = _Tensor(16)
    plan.forward_tensors(_Tensor(4, 16), w, w, _Tensor(4, 16))
    assert ctx.calls

    config = vk.LinearAttentionConfig.new(4, 16, 24).with_kv_heads(2)
    plan = ctx.plan(config)
    config.heads, config.kv_heads, config.key_dim, config.value_dim = 2, 1, 8, 12
    with pytest.raises(vk.VkFftError) as e:
        plan.forward_tensors(_Tensor(1, 1, 2, 8), _Tensor(1, 1, 1, 8), _Tensor(1, 1, 1, 12), _Tensor(1, 1, 2, 12))
    assert e.value.kind == "InputLengthMismatch" and not ctx.calls
    plan.forward_tensors(_Tensor(1, 1, 4, 16), _Tensor(1, 1, 2, 16), _Tensor(1, 1, 2, 24), _Tensor(1, 1, 4, 24))
    assert ctx.calls


def _refused(kind, f, *a, **kw):
    with pytest.raises(vk.VkFftError) as e:
        f(*a, **kw)
    assert e.value.kind == kind, e.value


@pytest.mark.parametrize("missing", [None, [1.0], 3])
def test_what_is_no_tensor_is_refused_as_an_argument(missing):
    ctx = _Context()
    norm = ctx.plan(vk.LayerNormConfig.new(8))
    w, x, st = _Tensor(8), _Tensor(4, 8), _Tensor(4, 2)
    _refused("InvalidArgument", norm.forward_tensors, missing, w, w, x)
    _refused("InvalidArgument", norm.forward_tensors, x, w, w, missing)
    _refused("InvalidArgument", norm.backward_tensors, missing, w, st, x, x, w, w)
    _refused("InvalidArgument", norm.backward_tensors, x, w, st, missing, x, w, w)
    mix = ctx.plan(vk.LinearAttentionConfig.new(2, 8, 8).with_capacity(1, 4).with_gradient())
    t = [_Tensor(1, 4, 2, 8) for _ in range(7)]
    for i in range(4):
        _refused("InvalidArgument", mix.forward_tensors, *[missing if j == i else x for j, x in enumerate(t[:4])])
    for i in range(7):
        _refused("InvalidArgument", mix.backward_tensors, *[missing if j == i else x for j, x in enumerate(t)])
    if missing is not None:  # None is the way to leave these out
        _refused("InvalidArgument", norm.forward_tensors, x, missing, w, x)
        _refused("InvalidArgument", norm.backward_tensors, x, w, st, x, x, missing, w)
        _refused("InvalidArgument", norm.backward_tensors, x, w, st, x, missing, w, w)
        _refused("InvalidArgument", mix.forward_tensors, *t[:4], state_in=missing)
        _refused("InvalidArgument", mix.forward_tensors, *t[:4], lengths=missing)
        _refused("InvalidArgument", mix.forward_tensors, *t[:4], work=missing)
    assert not ctx.calls


def test_a_tensor_without_dimensions_is_refused():
    ctx = _Context()
    norm = ctx.plan(vk.LayerNormConfig.new(8))
    w, x = _Tensor(8), _Tensor(4, 8)
    for y in (_Tensor(), _Tensor(8), _Tensor(1, 4, 8)):
        _refused("InputLengthMismatch", norm.forward_tensors, y, w, w, x)
        _refused("InputLengthMismatch", norm.backward_tensors, y, w, _Tensor(4, 2), x, x, w, w)
    mix = ctx.plan(vk.LinearAttentionConfig.new(2, 8, 8).with_capacity(1, 4))
    t = [_Tensor(1, 4, 2, 8) for _ in range(4)]
    _refused("InputLengthMismatch", mix.forward_tensors, _Tensor(), *t[1:])
    assert not ctx.calls
