"""8-bit operators whose inputs the launch before them writes, into buffers that are
used over and over: queued without a pause (each kernel starts while the one before
it ends) they give the bits of the same calls made one at a time on buffers of
their own, whose products are checked against 64 bits."""
import pytest
import torch

from llama2_b200 import capi, ops
from tests.test_gpu_int8 import check_product, gen

pytestmark = pytest.mark.gpu

STEPS = 24


@pytest.fixture(autouse=True)
def _lib(cuda_lib):
    yield
    assert capi.lib().l2k_device_error(1) == 0


def rows(n, dim):
    return (torch.empty(n, dim, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda"))


def queued(run):
    """run() eagerly, then twice more as one captured graph; yields after each."""
    run()
    torch.cuda.synchronize()
    yield "eager"
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(2):
        graph.replay()
        torch.cuda.synchronize()
        yield f"replay {i}"


# decode rows, tiles split over a cluster, the two-SM kernel, rows that TMA cannot address
@pytest.mark.parametrize("m,n,k", [(1, 96, 512), (4, 1000, 512), (64, 4096, 1024), (300, 264, 528), (2048, 4096, 256),
                                   (70, 129, 515)])
def test_operands_and_scales_written_by_the_launch_before(m, n, k):
    t = torch.bfloat16
    g = gen(m + k)
    grow = torch.logspace(-3, 3, STEPS, base=2).tolist()  # each step's scales are others
    xs = [(torch.randn(m, k, generator=g, device="cuda") * f).to(t) for f in grow]
    ws = [(torch.randn(n, k, generator=g, device="cuda") / f / 8).to(t) for f in reversed(grow)]
    (a, sa), (b, sb) = rows(m, k), rows(n, k)
    got = [torch.empty(m, n, dtype=t, device="cuda") for _ in range(STEPS)]

    def run():
        for i in range(STEPS):
            if i % 2:  # b and its scales last, or a and its scales
                ops.launch_quantize_rows_int8(xs[i], a, sa)
                ops.launch_quantize_rows_int8(ws[i], b, sb)
            else:
                ops.launch_quantize_rows_int8(ws[i], b, sb)
                ops.launch_quantize_rows_int8(xs[i], a, sa)
            ops.launch_linear_int8(a, sa, b, sb, got[i])

    want = []
    for i in range(STEPS):
        (qa, qsa), (qb, qsb) = rows(m, k), rows(n, k)
        c = torch.empty(m, n, dtype=t, device="cuda")
        ops.launch_quantize_rows_int8(xs[i], qa, qsa)
        torch.cuda.synchronize()
        ops.launch_quantize_rows_int8(ws[i], qb, qsb)
        torch.cuda.synchronize()
        ops.launch_linear_int8(qa, qsa, qb, qsb, c)
        torch.cuda.synchronize()
        check_product(c, qa, qsa, qb, qsb)
        want.append(c)
    for how in queued(run):
        for i in range(STEPS):
            assert torch.equal(got[i], want[i]), (how, i)


@pytest.mark.parametrize("n_rows,dim", [(4, 512), (700, 512), (3, 515), (700, 515)])
def test_norm_weights_written_by_the_launch_before(n_rows, dim):
    """The norm's weights are the one row of the product before it."""
    g = gen(dim)
    a, sa = torch.randint(-127, 128, (1, 64), generator=g, device="cuda", dtype=torch.int8), torch.ones(1, device="cuda")
    bs = [torch.randint(-127, 128, (dim, 64), generator=g, device="cuda", dtype=torch.int8) for _ in range(STEPS)]
    sb = torch.full((dim,), 1e-4, device="cuda")
    xs = [torch.randn(n_rows, dim, generator=g, device="cuda") for _ in range(STEPS)]
    w = torch.empty(1, dim, device="cuda")
    got = [rows(n_rows, dim) for _ in range(STEPS)]

    def run():
        for b, x, (q, s) in zip(bs, xs, got):
            ops.launch_linear_int8(a, sa, b, sb, w)
            ops.launch_fused_add_residual_rmsnorm_int8(w[0], x, None, q, s, False)

    want = []
    for b, x in zip(bs, xs):
        c, (q, s) = torch.empty(1, dim, device="cuda"), rows(n_rows, dim)
        ops.launch_linear_int8(a, sa, b, sb, c)
        torch.cuda.synchronize()
        check_product(c, a, sa, b, sb)
        ops.launch_fused_add_residual_rmsnorm_int8(c[0], x, None, q, s, False)
        torch.cuda.synchronize()
        want.append((q, s))
    for how in queued(run):
        for i in range(STEPS):
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1]), (how, i)
