"""Refusals of the 8-bit (W8A8) operators, before anything is launched: at the
C ABI (bad sizes, types, null pointers) and in llama2_b200.ops (types, shapes,
devices of the tensors)."""
import pytest
import torch

from llama2_b200 import capi, ops

BF16, F32 = capi.L2K_BF16, capi.L2K_F32


@pytest.mark.parametrize("call,args,status", [
    ("l2k_quantize_rows_int8", (16, 16, 16, -1, 8, F32, None), 1),
    ("l2k_quantize_rows_int8", (16, 16, 16, 4, -8, F32, None), 1),
    ("l2k_quantize_rows_int8", (16, 16, 16, 4, 8, capi.L2K_F32 + 3, None), 1),  # e4m3 rows
    ("l2k_quantize_rows_int8", (None, 16, 16, 4, 8, F32, None), 1),
    ("l2k_quantize_rows_int8", (16, None, 16, 4, 8, F32, None), 1),
    ("l2k_quantize_rows_int8", (16, 16, None, 4, 8, F32, None), 1),
    ("l2k_quantize_rows_int8", (16, 16, 16, 2 ** 31, 8, F32, None), 3),
    ("l2k_fused_add_residual_rmsnorm_int8", (16, 32, 48, 16, 16, -2, 8, 1, BF16, None), 1),
    ("l2k_fused_add_residual_rmsnorm_int8", (16, 32, 48, 16, 16, 2, 8, 1, 9, None), 1),
    ("l2k_fused_add_residual_rmsnorm_int8", (None, 32, 48, 16, 16, 2, 8, 1, BF16, None), 1),
    ("l2k_fused_add_residual_rmsnorm_int8", (16, None, 48, 16, 16, 2, 8, 1, BF16, None), 1),
    ("l2k_fused_add_residual_rmsnorm_int8", (16, 32, None, 16, 16, 2, 8, 1, BF16, None), 1),  # nothing to add
    ("l2k_fused_add_residual_rmsnorm_int8", (16, 32, 32, 16, 16, 2, 8, 1, BF16, None), 1),    # x is residual
    ("l2k_fused_add_residual_rmsnorm_int8", (16, 32, None, None, 16, 2, 8, 0, BF16, None), 1),
    ("l2k_swiglu_int8", (16, 16, 16, 2, -4, BF16, None), 1),
    ("l2k_swiglu_int8", (16, 16, 16, 2, 4, -1, None), 1),
    ("l2k_swiglu_int8", (None, 16, 16, 2, 4, BF16, None), 1),
    ("l2k_swiglu_int8", (16, 16, None, 2, 4, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, -1, 16, 32, 16, 16, 32, 16, 16, 8, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, 32, 16, 31, 16, 16, 32, 16, 16, 8, BF16, None), 1),  # lda < k
    ("l2k_linear_int8", (4, 8, 32, 16, 32, 16, 16, 16, 16, 16, 8, BF16, None), 1),  # ldb < k
    ("l2k_linear_int8", (4, 8, 32, 16, 32, 16, 16, 32, 16, 16, 7, BF16, None), 1),  # ldc < n
    ("l2k_linear_int8", (4, 8, 32, 16, 32, 16, 16, 32, 16, 16, 8, 3, None), 1),
    ("l2k_linear_int8", (4, 8, 32, None, 32, 16, 16, 32, 16, 16, 8, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, 32, 16, 32, None, 16, 32, 16, 16, 8, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, 32, 16, 32, 16, None, 32, 16, 16, 8, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, 32, 16, 32, 16, 16, 32, None, 16, 8, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, 32, 16, 32, 16, 16, 32, 16, None, 8, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, 131072, 16, 131072, 16, 16, 131072, 16, 16, 8, BF16, None), 3),  # sums past 2^31
    ("l2k_quantize_rows_int8", (18, 16, 16, 4, 8, F32, None), 1),  # not aligned to its elements
    ("l2k_quantize_rows_int8", (16, 16, 18, 4, 8, BF16, None), 1),
    ("l2k_fused_add_residual_rmsnorm_int8", (17, 32, 48, 16, 16, 2, 8, 1, BF16, None), 1),
    ("l2k_fused_add_residual_rmsnorm_int8", (16, 32, 49, 16, 16, 2, 8, 1, BF16, None), 1),
    ("l2k_swiglu_int8", (17, 16, 16, 2, 4, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, 32, 16, 32, 16, 16, 32, 16, 17, 8, BF16, None), 1),
    ("l2k_linear_int8", (4, 8, 32, 16, 32, 18, 16, 32, 16, 16, 8, BF16, None), 1),
    ("l2k_linear_int8", (2 ** 31, 8, 32, 16, 32, 16, 16, 32, 16, 16, 8, BF16, None), 3),
])
def test_c_abi_refuses(call, args, status):
    with pytest.raises(capi.L2KError) as e:
        capi.call(call, *args)
    assert e.value.status == status
    assert call.encode() in capi.lib().l2k_last_error_message()


def test_empty_inputs_are_noops():
    capi.call("l2k_quantize_rows_int8", None, None, None, 0, 8, F32, None)
    capi.call("l2k_fused_add_residual_rmsnorm_int8", None, None, None, None, None, 0, 8, 1, BF16, None)
    capi.call("l2k_swiglu_int8", None, None, None, 0, 8, BF16, None)
    capi.call("l2k_linear_int8", 0, 8, 32, None, 32, None, None, 32, None, None, 8, BF16, None)
    capi.call("l2k_linear_int8", 8, 0, 32, None, 32, None, None, 32, None, None, 8, BF16, None)


@pytest.fixture
def host_tensors(monkeypatch):
    """The operators' checks on host tensors: the device check passes, a launch fails the test."""
    def call(dev, name, *args):
        raise AssertionError(f"{name} was launched")

    monkeypatch.setattr(ops, "_one_device", lambda *ts: 0)
    monkeypatch.setattr(ops, "_call_on", call)


class OnDevice:
    """What _one_device asks of a tensor."""
    is_cuda = True

    def __init__(self, dev):
        self.device = f"cuda:{dev}"

    def is_contiguous(self):
        return True

    def get_device(self):
        return int(self.device[-1])


def i8(*s):
    return torch.empty(*s, dtype=torch.int8)


def f32(*s):
    return torch.empty(*s)


@pytest.mark.parametrize("fn", [
    lambda: ops.launch_quantize_rows_int8(f32(3, 8), torch.empty(3, 8, dtype=torch.uint8), f32(3)),
    lambda: ops.launch_quantize_rows_int8(f32(3, 8), i8(3, 9), f32(3)),
    lambda: ops.launch_quantize_rows_int8(f32(3, 8), i8(3, 8), f32(4)),
    lambda: ops.launch_quantize_rows_int8(f32(3, 8), i8(3, 8), f32(3).double()),
    lambda: ops.launch_quantize_rows_int8(f32(2, 3, 8), i8(6, 8), f32(6)),
    lambda: ops.launch_fused_add_residual_rmsnorm_int8(f32(8), f32(3, 8), f32(3, 7), i8(3, 8), f32(3), True),
    lambda: ops.launch_fused_add_residual_rmsnorm_int8(f32(7), f32(3, 8), None, i8(3, 8), f32(3), False),
    lambda: ops.launch_fused_add_residual_rmsnorm_int8(f32(8).half(), f32(3, 8), None, i8(3, 8), f32(3), False),
    lambda: ops.launch_fused_add_residual_rmsnorm_int8(f32(8), f32(3, 8), f32(3, 8).half(), i8(3, 8), f32(3), True),
    lambda: ops.launch_fused_add_residual_rmsnorm_int8(f32(8), f32(3, 8), None, i8(3, 8), f32(3), True),
    lambda: ops.launch_swiglu_int8(f32(3, 8), i8(3, 8), f32(3)),
    lambda: ops.launch_swiglu_int8(f32(3, 16), i8(3, 8), f32(2)),
    lambda: ops.launch_linear_int8(i8(3, 32), f32(3), i8(5, 16), f32(5), f32(3, 5)),
    lambda: ops.launch_linear_int8(i8(3, 32), f32(3), i8(5, 32), f32(3), f32(3, 5)),
    lambda: ops.launch_linear_int8(i8(3, 32), f32(3), i8(5, 32), f32(5), f32(5, 3)),
    lambda: ops.launch_linear_int8(f32(3, 32), f32(3), i8(5, 32), f32(5), f32(3, 5)),
    lambda: ops.launch_linear_int8(i8(3, 32), f32(3), i8(5, 32), f32(5), f32(15)),
    lambda: ops.launch_linear_int8(i8(3, 32), f32(3), i8(5, 32), f32(5), f32(3, 5).double()),
])
def test_ops_refuse(host_tensors, fn):
    with pytest.raises(ValueError):
        fn()


def test_launch_on_the_tensors_device(monkeypatch):
    """The device of the tensors is current during the call, its current stream
    is used, and the caller's device is restored."""
    calls, current = [], [0]

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.old, current[0] = current[0], self.dev

        def __exit__(self, *a):
            current[0] = self.old

    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 100 + dev)
    monkeypatch.setattr(capi, "call", lambda name, *args: calls.append((current[0], name, *args)))
    ops._call_on(0, "f", 1)
    ops._call_on(1, "f", 2)
    assert calls == [(0, "f", 1, 100), (1, "f", 2, 101)] and current[0] == 0


def test_host_tensors_and_mixed_devices_are_refused():
    with pytest.raises(ValueError, match="CUDA device"):
        ops.launch_quantize_rows_int8(f32(3, 8), i8(3, 8), f32(3))
    with pytest.raises(ValueError, match="different devices"):
        ops._one_device(OnDevice(0), OnDevice(0), OnDevice(1))
    assert ops._one_device(OnDevice(1), OnDevice(1)) == 1
