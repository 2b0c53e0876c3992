"""8-bit operators on tensors of more than 2^31 elements, and as the first calls of a
process, made inside a capture."""
import os
import subprocess
import sys

import pytest
import torch

from llama2_b200 import capi, ops
from tests.test_gpu_int8 import U, check_product, check_scales, gen, reference_rows

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def _lib(cuda_lib):
    yield
    assert capi.lib().l2k_device_error(1) == 0
    torch.cuda.empty_cache()


def some(n):
    """Rows from the first to the last."""
    return torch.tensor(sorted({0, 1, n // 3, n // 2, n - 2, n - 1}), device="cuda")


# aligned; an odd length; longer than the stream kernel holds
@pytest.mark.parametrize("n,dim", [(540_000, 4096), (525_000, 4099), (110_000, 20_001)])
def test_rows_past_32_bits(n, dim):
    t = torch.bfloat16
    assert n * dim > 2 ** 31
    x = torch.empty(n, dim, dtype=t, device="cuda").normal_(generator=gen(1))
    q, s = torch.empty(n, dim, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    i = some(n)
    ops.launch_quantize_rows_int8(x, q, s)
    want, scale = reference_rows(x[i].double())
    assert torch.equal(q[i].double(), want)
    check_scales(s[i], scale, U)
    w = (torch.rand(dim, generator=gen(2), device="cuda") + 0.5).to(t)
    r = torch.empty(n, dim, dtype=t, device="cuda").normal_(generator=gen(3))
    stored = (x[i].float() + r[i].float()).to(t)
    ops.launch_fused_add_residual_rmsnorm_int8(w, x, r, q, s, True)
    assert torch.equal(x[i], stored)
    y = stored.double()
    want, scale = reference_rows(y * w.double())
    assert torch.equal(q[i].double(), want)
    check_scales(s[i], scale / (y.square().mean(1) + 1e-5).sqrt(), 32 * U)


@pytest.mark.parametrize("n,f", [(270_000, 4096), (263_000, 4099)])
def test_swiglu_past_32_bits(n, f):
    x = torch.empty(n, 2 * f, dtype=torch.bfloat16, device="cuda").normal_(generator=gen(1))
    assert x.numel() > 2 ** 31
    q, s = torch.empty(n, f, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    ops.launch_swiglu_int8(x, q, s)
    i = some(n)
    g, u = x[i].double().chunk(2, dim=1)
    y = g / (1 + torch.exp(-g)) * u
    want, scale = reference_rows(y)
    t = 127 * y / y.abs().amax(1, keepdim=True)
    near = ((t - t.floor()) - 0.5).abs() <= 1.5e-3  # (the bar of gates up to 32)
    assert ((q[i].double() == want) | (near & ((q[i].double() - want).abs() <= 1))).all()
    check_scales(s[i], scale, 96 * U)


# C past 2^31 elements: the two-SM kernel with rows of C on 16 bytes and not, the tile kernel
# without TMA; then A past 2^31 bytes
@pytest.mark.parametrize("m,n,k", [(70_000, 32_000, 64), (70_001, 32_003, 48), (70_000, 32_000, 17), (20_000, 64, 131_056)])
def test_products_past_32_bits(m, n, k):
    g = gen(m)
    a = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sa, sb = (torch.rand(r, generator=g, device="cuda") + 0.5 for r in (m, n))
    c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    assert max(c.numel(), a.numel()) > 2 ** 31
    ops.launch_linear_int8(a, sa, b, sb, c)
    i = some(m)
    check_product(c[i], a[i], sa[i], b, sb)


FIRST = """
import torch
from llama2_b200 import capi, ops
e = lambda *s, t=torch.bfloat16: torch.empty(*s, dtype=t, device="cuda")
i8, f4 = torch.int8, torch.float32
calls = []
for n, d in ((4, 512), (700, 512), (700, 515), (2, 16392)):
    x = torch.randn(n, d, device="cuda").to(torch.bfloat16)
    gu = torch.randn(n, 2 * d, device="cuda").to(torch.bfloat16)
    calls.append((x, gu, torch.ones(d, device="cuda").to(torch.bfloat16), [(e(n, d, t=i8), e(n, t=f4)) for _ in range(3)]))
products = [(torch.randint(-127, 128, (m, k), device="cuda", dtype=i8), torch.randint(-127, 128, (n, k), device="cuda", dtype=i8),
             torch.ones(m, device="cuda"), torch.ones(n, device="cuda"), e(m, n, t=f4))
            for m, n, k in ((1, 64, 512), (64, 4096, 1024), (2048, 4096, 256), (5, 70, 33))]

def run():
    for x, gu, w, out in calls:
        ops.launch_quantize_rows_int8(x, *out[0])
        ops.launch_fused_add_residual_rmsnorm_int8(w, x, None, *out[1], False)
        ops.launch_swiglu_int8(gu, *out[2])
    for a, b, sa, sb, c in products:
        ops.launch_linear_int8(a, sa, b, sb, c)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    run()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for c in calls for o in c[3] for t in o] + [p[4].clone() for p in products]
run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, [t for c in calls for o in c[3] for t in o] + [p[4] for p in products]))
assert capi.lib().l2k_device_error(1) == 0
print("captured first")
"""


def test_first_calls_of_a_process_inside_a_capture():
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]
