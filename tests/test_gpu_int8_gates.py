"""SwiGLU to 8 bits over gates down to -80, against 64 bits, with up values that
bring every element near the row's largest.

Bar, in u = 2^-24 (half a step of fp32), for gates of magnitude G at most: the
exponential's argument is the product of -g with a rounded log2(e), 1.22 u |g| log2(e)
off, which its value turns into 1.22 G; the exponential is off by 2 steps (4), the
sum by 1, the reciprocal by 1 step (2), two products by 2: below 1.25 G + 9. An 8-bit
value carries that of its element and of the row's largest, 127 times each: it is
rne(127 y / a) unless that lies within 254 (1.25 G + 9) u of a border between two
integers, and within 1 there. The scale has that of the largest and one rounding."""
import pytest
import torch

from llama2_b200 import capi, ops
from tests.test_gpu_int8 import U, check_untouched, gen, placed, reference_rows, row_outputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(cuda_lib):
    yield
    assert capi.lib().l2k_device_error(1) == 0


# one row per CTA, streamed rows (aligned and not), rows longer than the stream kernel holds
SHAPES = [(20, 512), (700, 512), (700, 515), (600, 4096), (3, 16392)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low,high", [(-80.0, -79.0), (-80.0, 80.0), (-60.0, -20.0), (-32.0, 32.0), (-1.0, 1.0)])
@pytest.mark.parametrize("n,dim", SHAPES)
def test_gates(n, dim, low, high, dtype):
    g = gen(n + dim)
    gate = (torch.rand(n, dim, generator=g, device="cuda") * (high - low) + low).to(dtype).double()
    gate = torch.where(gate == 0, 1.0, gate)
    wanted = torch.rand(n, dim, generator=g, device="cuda").double() + 0.01
    up = (wanted * (1 + torch.exp(-gate)) / gate).to(dtype).double()  # at most 1e33 of fp32's 3e38
    x = placed(torch.cat([gate, up], 1).to(dtype), 1 if dim % 8 else 0)
    q, s, qs, ss = row_outputs(n, dim)
    ops.launch_swiglu_int8(x, q, s)
    y = gate / (1 + torch.exp(-gate)) * up
    want, scale = reference_rows(y)
    t = 127 * y / y.abs().amax(1, keepdim=True)
    bar = 1.25 * max(abs(low), abs(high)) + 9
    near = ((t - t.floor()) - 0.5).abs() <= 254 * bar * U
    assert ((q.double() == want) | (near & ((q.double() - want).abs() <= 1))).all()
    assert ((s.double() - scale).abs() <= (bar + 1) * U * scale).all()
    check_untouched(n, dim, 0, qs, ss)


@pytest.mark.parametrize("n,dim", SHAPES)
def test_gates_whose_sigmoid_is_flushed(n, dim):
    x = torch.full((n, 2 * dim), -87.5, device="cuda")
    x[:, dim:] = 1e30
    q, s, _, _ = row_outputs(n, dim)
    ops.launch_swiglu_int8(x, q, s)
    assert (q == 0).all() and (s == 0).all()
