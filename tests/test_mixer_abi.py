"""The entry points of rotary positions and of the gated recurrence refuse null
arguments, and their Python mirror refuses bad configurations and tensors,
without a GPU."""
import ctypes
import math
import types

import pytest

import vkfft_amd as vk
from test_sequence_abi import _Tensor, _refused


def test_null_arguments_are_rejected():
    L = vk.lib()
    out, size = ctypes.c_void_p(), ctypes.c_uint64()
    for kind in ("rotary", "gated_recurrence"):
        assert getattr(L, f"vkfx_{kind}_create")(None, None, ctypes.byref(out)) == -7
        assert getattr(L, f"vkfx_{kind}_workspace_bytes")(None, ctypes.byref(size)) == -7
        assert getattr(L, f"vkfx_{kind}_backward")(None, None, None, None) == -7
        assert getattr(L, f"vkfx_{kind}_destroy")(None) == 0
    assert L.vkfx_rotary_forward(None, None, None) == -7
    assert L.vkfx_gated_recurrence_forward(None, None, None, None) == -7
    assert b"null" in L.vkfx_last_error()


def test_descriptors_are_laid_out_as_the_header_has_them():
    assert ctypes.sizeof(vk._RotaryDesc) == 56
    assert vk._ROTARY_FORWARD.size == 16 + 4 * 32 + 5 * 8
    assert vk._ROTARY_BACKWARD.size == 16 + 6 * 32 + 7 * 8
    assert ctypes.sizeof(vk._GatedRecurrenceDesc) == 24
    assert vk._RECURRENCE_FORWARD.size == 16 + 3 * 24 + 4 * 8
    assert vk._RECURRENCE_BACKWARD.size == 16 + 5 * 24 + 4 * 8


@pytest.mark.parametrize("config,kind", [
    (vk.RotaryConfig.new(0, 16), "InvalidArgument"),
    (vk.RotaryConfig.new(2, -1), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_kv_heads(-1), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_rotary_dim(-2), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_rotary_dim(3), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_rotary_dim(18), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 15), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_frequencies([1.0] * 7), "InputLengthMismatch"),
    (vk.RotaryConfig.new(2, 16).with_base(0), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_base(float("nan")), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_linear_scaling(-1), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_base(1e300).with_base_scaling(1e300), "InvalidArgument"),
    (vk.RotaryConfig.new(2, 16).with_blended_scaling(4, 4096, 1, 32), "InvalidArgument"),
    (vk.GatedRecurrenceConfig.new(-1), "InvalidArgument"),
])
def test_bad_configurations(config, kind):
    with pytest.raises(vk.VkFftError) as e:
        config.desc()
    assert e.value.kind == kind


def test_defaults():
    d = vk.RotaryConfig.new(3, 64).desc()
    assert (d.kv_heads, d.rotary_dim, d.layout, d.norm, d.amplitude) == (3, 64, 1, 0, 1.0)
    assert [d.frequencies[i] for i in (0, 16)] == [1.0, 0.01]
    d = vk.RotaryConfig.new(3, 64).with_kv_heads(0).with_norm(1e-5).with_element(vk.Element.BF16).desc()
    assert (d.kv_heads, d.norm, d.epsilon, d.weight_element) == (0, 1, 1e-5, 2)
    g = vk.GatedRecurrenceConfig.new(8).desc()
    assert (g.channels, g.gate, g.complement, g.reserved) == (8, 0, 0, 0)


def test_scalings_for_long_contexts():
    new = lambda: vk.RotaryConfig.new(1, 64)  # noqa: E731
    plain = new().turns()
    assert new().with_linear_scaling(4).turns() == [f / 4 for f in plain]
    base = new().with_base_scaling(4).turns()
    assert base[0] == plain[0] and math.isclose(base[31], plain[31] / 4, rel_tol=1e-12)
    assert all(a >= b >= a / 4.000001 for a, b in zip(plain, base))
    blended = new().with_blended_scaling(8, 4096).turns()
    for f, g in zip(plain, blended):
        turns = 4096 * f / (2 * math.pi)
        assert g == f if turns >= 32 else math.isclose(g, f / 8) if turns <= 1 else f / 8 < g < f
    assert vk.RotaryConfig.new(1, 2).with_base_scaling(4).turns() == [0.25]
    assert vk.RotaryConfig.new(1, 7).with_rotary_dim(0).turns() == []


class _Context:
    """A context whose library takes every call and remembers it."""
    def __init__(self):
        self.handle, self.device_index, self._live_plans, self.calls = 1, 0, set(), []

        def entry(name):
            return lambda *a: self.calls.append((name, a)) or 0

        names = [f"vkfx_{k}_{f}" for k in ("rotary", "gated_recurrence") for f in ("create", "destroy", "workspace_bytes", "forward", "backward")]
        self._L = types.SimpleNamespace(**{n: entry(n) for n in names})

    def plan(self, config):
        p = (vk.RotaryPlan if isinstance(config, vk.RotaryConfig) else vk.GatedRecurrencePlan)(self, config)
        p._current = lambda device: 0
        del self.calls[:]
        return p


def test_a_plan_keeps_the_sizes_it_was_made_with():
    """The caller's configuration may change afterwards; the plan's kernels do not."""
    ctx = _Context()
    config = vk.RotaryConfig.new(4, 16).with_kv_heads(2)
    plan = ctx.plan(config)
    config.heads, config.kv_heads, config.head_dim, config.epsilon = 2, 1, 8, 1e-6
    q, k = _Tensor(1, 3, 2, 8), _Tensor(1, 3, 1, 8)
    _refused("InputLengthMismatch", plan.forward_tensors, q, k, q, k)
    _refused("InputLengthMismatch", plan.backward_tensors, q, k, q, k)
    assert not ctx.calls
    q, k = _Tensor(1, 3, 4, 16), _Tensor(1, 3, 2, 16)
    plan.forward_tensors(q, k, q, k)
    plan.backward_tensors(q, k, q, k)
    assert [c[0] for c in ctx.calls] == ["vkfx_rotary_forward", "vkfx_rotary_backward"]

    config = vk.GatedRecurrenceConfig.new(16)
    plan = ctx.plan(config)
    config.channels = 8
    x = _Tensor(1, 3, 8)
    _refused("InputLengthMismatch", plan.forward_tensors, x, x, x)
    assert not ctx.calls
    x = _Tensor(1, 3, 16)
    plan.forward_tensors(x, x, x)
    plan.backward_tensors(x, x, _Tensor(1, 1, 16), x, x, x)
    assert len(ctx.calls) == 2


@pytest.mark.parametrize("missing", [None, [1.0], 3])
def test_what_is_no_tensor_is_refused_as_an_argument(missing):
    ctx = _Context()
    plan = ctx.plan(vk.RotaryConfig.new(2, 8).with_norm())
    t = [_Tensor(1, 4, 2, 8) for _ in range(4)]
    for i in range(4):
        _refused("InvalidArgument", plan.forward_tensors, *[missing if j == i else x for j, x in enumerate(t)])
        _refused("InvalidArgument", plan.backward_tensors, *[missing if j == i else x for j, x in enumerate(t)], q=t[0], k=t[1])
    for name in ("q", "k"):
        _refused("InvalidArgument", plan.backward_tensors, *t, **{"q": t[0], "k": t[1], name: missing})
    if missing is not None:  # None is the way to leave these out
        for name in ("q_weight", "k_weight", "positions", "starts", "lengths"):
            _refused("InvalidArgument", plan.forward_tensors, *t, **{name: missing})
        for name in ("dq_weight", "dk_weight", "work"):
            _refused("InvalidArgument", plan.backward_tensors, *t, q=t[0], k=t[1], **{name: missing})
    plan = ctx.plan(vk.GatedRecurrenceConfig.new(8))
    t, saved = [_Tensor(1, 4, 8) for _ in range(5)], _Tensor(1, 1, 8)
    for i in range(3):
        _refused("InvalidArgument", plan.forward_tensors, *[missing if j == i else x for j, x in enumerate(t[:3])])
    for i in range(5):
        m = [missing if j == i else x for j, x in enumerate(t)]
        _refused("InvalidArgument", plan.backward_tensors, *m[:2], saved, *m[2:])
    if missing is not None:
        for name in ("state_in", "state_out", "saved", "lengths", "work"):
            _refused("InvalidArgument", plan.forward_tensors, *t[:3], **{name: missing})
        _refused("InvalidArgument", plan.backward_tensors, *t[:2], missing, *t[2:])
    assert not ctx.calls


def test_a_tensor_of_other_dimensions_is_refused():
    ctx = _Context()
    plan, rec = ctx.plan(vk.RotaryConfig.new(2, 8)), ctx.plan(vk.GatedRecurrenceConfig.new(8))
    for y in (_Tensor(), _Tensor(8), _Tensor(4, 2, 8), _Tensor(1, 1, 4, 2, 8)):
        _refused("InputLengthMismatch", plan.forward_tensors, y, y, y, y)
        _refused("InputLengthMismatch", plan.backward_tensors, y, y, y, y)
    for y in (_Tensor(), _Tensor(8), _Tensor(4, 8), _Tensor(1, 1, 4, 8)):
        _refused("InputLengthMismatch", rec.forward_tensors, y, y, y)
        _refused("InputLengthMismatch", rec.backward_tensors, y, y, y, y, y, y)
    assert not ctx.calls


@pytest.mark.parametrize("cls", [vk.RotaryPlan, vk.GatedRecurrencePlan])
@pytest.mark.parametrize("device", [-1, 0, 2])
def test_tensors_of_another_device_are_refused(cls, device):
    plan = cls.__new__(cls)  # a plan of device 1: its place alone, no GPU
    plan.handle, plan._device = None, 1
    _refused("InvalidArgument", plan._place, _Tensor(1, device=device))
