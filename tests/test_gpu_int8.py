"""The 8-bit (W8A8) operators on the GPU against plain 64-bit formulas.

Bars, from the arithmetic of the kernels (u = 2^-24, half a step of fp32):
  * int8 rows of x and of the norm: equal to rne(127 y / a), ties to even;
    SwiGLU's: within 1, and different only where 127 y / a lies within 1.5e-3
    of a border between two integers (127 times twice the relative error of
    silu_mul, at most 47 u for |gate| <= 32: the fast exponential's
    2 + 1.173 |gate| steps of 2u, a reciprocal, an add and two products;
    127 * 2 * 94 u = 1.43e-3);
  * scales: one rounding for x (1 u); the norm adds the sum of squares (at
    most 32 fused multiply-adds per thread and 10 levels of the tree, halved
    by the square root: 21 u) and five roundings more: 32 u; SwiGLU's carry
    94 u of silu_mul: 96 u;
  * products: three fp32 roundings and one to the output type: 4 u + eps / 2
    relative (and half the smallest step of fp16).
"""
import numpy as np
import pytest
import torch

from llama2_b200 import capi, ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
SENTINEL = 77


@pytest.fixture(autouse=True)
def _lib(cuda_lib):
    yield
    assert capi.lib().l2k_device_error(1) == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def placed(t, shift):
    """t's values in a contiguous tensor that starts `shift` elements into its storage."""
    buf = torch.empty(t.numel() + shift, dtype=t.dtype, device=t.device)
    out = buf[shift:].view(t.shape)
    out.copy_(t)
    return out


def row_outputs(n, dim, shift=0):
    """(q, scales, their storages): sentinels behind the last row."""
    qs = torch.full((n * dim + shift + 64,), SENTINEL, dtype=torch.int8, device="cuda")
    ss = torch.full((n + 8,), -7.0, dtype=torch.float32, device="cuda")
    return qs[shift:shift + n * dim].view(n, dim), ss[:n], qs, ss


def check_untouched(n, dim, shift, qs, ss):
    assert (qs[:shift] == SENTINEL).all() and (qs[shift + n * dim:] == SENTINEL).all()
    assert (ss[n:] == -7.0).all()


def reference_rows(y):
    """(q, a / 127) of 64-bit rows; rows that are not finite give 0 and NaN."""
    a = y.abs().amax(1, keepdim=True)
    bad = ~torch.isfinite(y).all(1, keepdim=True)
    q = torch.where(bad | (a == 0), 0.0, 127.0 * y / torch.where(a > 0, a, 1.0)).round()
    return q, torch.where(bad, torch.nan, a / 127)[:, 0]


def check_scales(got, want, rel):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = (got - want).abs() <= rel * want.abs() + 2.0 ** -150  # (half a subnormal step)
    assert (ok | torch.isnan(want)).all(), float(((got - want).abs() / want.abs()).nan_to_num().max())


SHAPES = [(1, 1), (3, 7), (2, 8), (5, 1000), (9, 1023), (64, 4096), (7, 8192), (3, 8200), (2, 16384), (2, 16392),
          (1, 20001), (130, 33), (301, 264)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim", SHAPES)
def test_quantize_rows(n, dim, dtype):
    x = (torch.randn(n, dim, generator=gen(dim), device="cuda") * 3).to(dtype)
    q, s, qs, ss = row_outputs(n, dim)
    ops.launch_quantize_rows_int8(x, q, s)
    want, scale = reference_rows(x.double())
    assert torch.equal(q.double(), want)
    check_scales(s, scale, U)
    check_untouched(n, dim, 0, qs, ss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [1, 3, 8])
def test_quantize_rows_of_any_alignment(dtype, shift):
    x = placed(torch.randn(6, 520, generator=gen(shift), device="cuda").to(dtype), shift)
    q, s, qs, ss = row_outputs(6, 520, shift)
    ops.launch_quantize_rows_int8(x, q, s)
    want, scale = reference_rows(x.double())
    assert torch.equal(q.double(), want)
    check_scales(s, scale, U)
    check_untouched(6, 520, shift, qs, ss)


def special_rows(dtype, dim):
    """Rows of zeros, ties, extremes, subnormals and values that are not finite."""
    f = torch.finfo(dtype)
    x = torch.randn(14, dim, generator=gen(1), device="cuda").to(dtype)
    ramp = torch.arange(dim, device="cuda") % 254
    x[0] = 0
    x[1] = ((ramp - 127).double() + 0.5).clamp(-127, 127).to(dtype)  # borders between two integers
    x[1, 0] = 127
    x[2] = 0
    x[2, dim // 2] = -3  # one value
    x[3] = f.max
    x[3, ::2] = -f.max
    x[4] = x[4].sign() * f.tiny
    x[5] = (f.tiny * ramp.double() / 254).to(dtype)  # subnormals
    x[6, dim - 1] = float("nan")
    x[7, 0] = float("inf")
    x[8, 1] = -float("inf")
    x[9] = 1
    x[10] = x[10].abs()
    x[11] = 0.5
    x[11, dim - 1] = 1  # 63.5 everywhere
    x[12] = -0.0
    x[13] = (x[13].double() * f.tiny * 1024).to(dtype)
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [256, 257])
def test_quantize_special_rows(dtype, dim):
    x = special_rows(dtype, dim)
    q, s, qs, ss = row_outputs(14, dim)
    ops.launch_quantize_rows_int8(x, q, s)
    want, scale = reference_rows(x.double())
    for i in range(14):
        assert torch.equal(q[i].double(), want[i]), i
    check_scales(s, scale, U)
    check_untouched(14, dim, 0, qs, ss)


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim", SHAPES)
def test_norm(n, dim, dtype, add):
    x = (torch.randn(n, dim, generator=gen(dim), device="cuda") * 2).to(dtype)
    r = torch.randn(n, dim, generator=gen(dim + 1), device="cuda").to(dtype)
    w = (torch.rand(dim, generator=gen(3), device="cuda") + 0.5).to(dtype)
    w[0] = -w[0]
    _check_norm(x, r, w, add)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [1, 4])
def test_norm_of_any_alignment(dtype, shift):
    x, r = (placed(torch.randn(5, 264, generator=gen(s), device="cuda").to(dtype), shift) for s in (1, 2))
    w = placed((torch.rand(264, generator=gen(3), device="cuda") + 0.5).to(dtype), shift)
    _check_norm(x, r, w, True, shift)


def _check_norm(x, r, w, add, shift=0):
    n, dim = x.shape
    x0, r0 = x.clone(), r.clone()
    q, s, qs, ss = row_outputs(n, dim, shift)
    ops.launch_fused_add_residual_rmsnorm_int8(w, x, r if add else None, q, s, add)
    stored = (x0.float() + r0.float()).to(x.dtype) if add else x0
    assert torch.equal(x.view(torch.uint8), stored.view(torch.uint8)) and torch.equal(r, r0)
    y = stored.double()
    want, scale = reference_rows(y * w.double())
    inv_rms = 1 / (y.square().mean(1) + 1e-5).sqrt()
    assert torch.equal(q.double(), want)
    check_scales(s, scale * inv_rms, 32 * U)
    check_untouched(n, dim, shift, qs, ss)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_special_rows(dtype):
    """Zero rows, rows that are not finite (before or after the addition), a
    weight of zeros, and rows whose squares leave the range of fp32."""
    dim = 512
    x = torch.randn(6, dim, generator=gen(1), device="cuda").to(dtype)
    r = torch.randn(6, dim, generator=gen(2), device="cuda").to(dtype)
    w = (torch.rand(dim, generator=gen(3), device="cuda") + 0.5).to(dtype)
    x[0], r[0] = 0, 0
    x[1, 7] = float("nan")
    r[2, 0] = float("inf")
    x[3], r[3] = torch.finfo(dtype).max, torch.finfo(dtype).max  # the sum is infinite
    q, s, _, _ = row_outputs(6, dim)
    ops.launch_fused_add_residual_rmsnorm_int8(w, x, r, q, s, True)
    assert (q[:4] == 0).all() and s[0] == 0 and torch.isnan(s[1:4]).all() and torch.isfinite(s[4:]).all()
    assert (q[4:].abs().amax(1) == 127).all()
    ops.launch_fused_add_residual_rmsnorm_int8(torch.zeros_like(w), x, None, q, s, False)
    assert (q == 0).all() and (s[4:] == 0).all()
    if dtype != torch.float16:
        big = torch.full((2, dim), 2.0 ** 70, device="cuda").to(dtype)
        q, s, _, _ = row_outputs(2, dim)
        ops.launch_fused_add_residual_rmsnorm_int8(w, big, None, q, s, False)
        assert (s == 0).all()  # 1 / rms is 0, as in launch_fused_add_residual_rmsnorm


def _check_swiglu(x, n, dim, shift=0):
    q, s, qs, ss = row_outputs(n, dim, shift)
    ops.launch_swiglu_int8(x, q, s)
    g, u = x.double().chunk(2, dim=1)
    y = g / (1 + torch.exp(-g)) * u
    want, scale = reference_rows(y)
    a = y.abs().amax(1, keepdim=True)
    t = 127 * y / torch.where(a > 0, a, 1.0)
    near = ((t - t.floor()) - 0.5).abs() <= 1.5e-3
    same = q.double() == want
    assert (same | (near & ((q.double() - want).abs() <= 1))).all()
    check_scales(s, scale, 96 * U)
    check_untouched(n, dim, shift, qs, ss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim", SHAPES)
def test_swiglu(n, dim, dtype):
    x = (torch.randn(n, 2 * dim, generator=gen(dim), device="cuda") * 4).to(dtype)
    _check_swiglu(x, n, dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [1, 8])
def test_swiglu_of_any_alignment(dtype, shift):
    x = placed(torch.randn(5, 2 * 520, generator=gen(2), device="cuda").to(dtype), shift)
    _check_swiglu(x, 5, 520, shift)


# (rows, length): several rows a CTA at each distance of a row from a multiple of 8
# elements, rows shorter than 8 elements, whole tensors inside one 16-byte unit
RAGGED = [(5000, 263), (3001, 257), (2403, 1020), (4000, 5), (1, 3), (17, 1), (700, 14)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [(0, 0, 0, 0), (1, 1, 1, 1), (3, 5, 2, 7), (8, 4, 1, 2)])
@pytest.mark.parametrize("n,dim", RAGGED)
def test_rows_and_outputs_placed_apart(n, dim, at, dtype):
    """x, the residual, the weights and q each at an alignment of its own."""
    x = placed(torch.randn(n, dim, generator=gen(1), device="cuda").to(dtype), at[0])
    q, s, qs, ss = row_outputs(n, dim, at[3])
    ops.launch_quantize_rows_int8(x, q, s)
    want, scale = reference_rows(x.double())
    assert torch.equal(q.double(), want)
    check_scales(s, scale, U)
    check_untouched(n, dim, at[3], qs, ss)

    r = placed(torch.randn(n, dim, generator=gen(2), device="cuda").to(dtype), at[1])
    w = placed((torch.rand(dim, generator=gen(3), device="cuda") + 0.5).to(dtype), at[2])
    before = x._base[:at[0]].fill_(SENTINEL)
    _check_norm(x, r, w, False, at[3])
    _check_norm(x, r, w, True, at[3])
    assert (before == SENTINEL).all()
    _check_swiglu(placed(torch.randn(n, 2 * dim, generator=gen(4), device="cuda").to(dtype), at[0]), n, dim, at[3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_special_rows(dtype):
    dim = 128
    x = torch.randn(6, 2 * dim, generator=gen(1), device="cuda").to(dtype)
    x[0] = 0
    x[1, :dim] = -1000  # silu 0
    x[2, dim + 5] = float("nan")
    x[3, 9] = float("inf")
    x[4, dim:] = 0
    x[5, :dim] = 1000  # silu(g) = g
    q, s, _, _ = row_outputs(6, dim)
    ops.launch_swiglu_int8(x, q, s)
    assert (q[:5] == 0).all() and (s[[0, 1, 4]] == 0).all() and torch.isnan(s[2:4]).all()
    want, scale = reference_rows(x[5:, :dim].double() * x[5:, dim:].double())
    assert torch.equal(q[5:].double(), want)
    check_scales(s[5:], scale, 4 * U)


# ------------------------------------------------------------------ products
def operands(m, n, k, seed=0):
    g = gen(seed)
    a = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sa = (torch.rand(m, generator=g, device="cuda") + 0.5) / 127
    sb = (torch.rand(n, generator=g, device="cuda") + 0.5) / (127 * max(k, 1) ** 0.5)
    return a, sa, b, sb


def check_product(c, a, sa, b, sb):
    want = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()  # (sums below 2^53: exact)
    tol = (torch.finfo(c.dtype).eps / 2 if c.dtype != torch.float32 else 0) + 4 * U
    tiny = 2.0 ** -25 if c.dtype == torch.float16 else 0.0
    err = (c.double() - want).abs()
    assert (err <= tol * want.abs() + tiny).all(), (float(err.max()), torch.nonzero(err > tol * want.abs() + tiny)[:4])


LINEAR = [(1, 1, 16), (1, 64, 128), (1, 4096, 4096), (2, 33, 48), (7, 100, 400), (8, 96, 272), (9, 1000, 1040),
          (63, 4100, 512), (64, 12288, 1024), (64, 320, 11008), (65, 257, 144), (100, 4096, 2048), (127, 513, 640),
          (128, 22016, 256), (129, 1003, 2064), (200, 4096, 1040), (255, 700, 4096), (256, 256, 128),
          (257, 1003, 2064), (300, 31, 4096), (511, 2049, 16), (1000, 1537, 1296), (2048, 4096, 4096),
          (2100, 4099, 528), (3333, 5000, 400), (5000, 2056, 1024)]


LINEAR_MIX = [(1, 4096, 1024), (64, 4096, 2048), (70, 300, 1001), (2048, 4096, 512), (130, 1000, 640)]


@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear_on_tensor_cores(m, n, k):
    a, sa, b, sb = operands(m, n, k, m + n)
    for dtype in DTYPES:
        store = torch.full((m * n + 64,), 3.0, dtype=dtype, device="cuda")
        c = store[:m * n].view(m, n)
        ops.launch_linear_int8(a, sa, b, sb, c)
        check_product(c, a, sa, b, sb)
        assert (store[m * n:] == 3.0).all()


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 70, 17), (65, 129, 1001), (2, 5, 4093), (130, 64, 63), (1, 4096, 4095),
                                   (64, 300, 2050), (300, 1000, 515), (1000, 257, 1300)])
def test_linear_without_tma(m, n, k):
    """Rows of no multiple of 16 bytes."""
    a, sa, b, sb = operands(m, n, k, k)
    for dtype in DTYPES:
        c = torch.empty(m, n, dtype=dtype, device="cuda")
        ops.launch_linear_int8(a, sa, b, sb, c)
        check_product(c, a, sa, b, sb)


@pytest.mark.parametrize("m,k", [(3, 4099), (70, 77)])
def test_linear_without_tma_reads_its_rows_alone(m, k):
    """Rows between bytes of other values, at every offset from a word."""
    n = 37
    a, sa, b, sb = operands(m, n, k, 9)
    for lda, ldb, at in ((k + 1, k + 2, 1), (k + 3, k, 2), (k, k + 5, 3)):
        bufs = []
        for t, rows, ld in ((a, m, lda), (b, n, ldb)):
            buf = torch.full((rows * ld + 8,), -77, dtype=torch.int8, device="cuda")
            buf[at:at + rows * ld].view(rows, ld)[:, :k] = t
            bufs.append(buf)
        c = torch.empty(m, n, device="cuda")
        capi.call("l2k_linear_int8", m, n, k, bufs[0].data_ptr() + at, lda, sa.data_ptr(), bufs[1].data_ptr() + at, ldb,
                  sb.data_ptr(), c.data_ptr(), n, capi.L2K_F32, torch.cuda.current_stream().cuda_stream)
        check_product(c, a, sa, b, sb)


@pytest.mark.parametrize("shift", [1, 4, 16])
def test_linear_of_any_alignment(shift):
    a, sa, b, sb = operands(33, 65, 256, 1)
    a, b = placed(a, shift), placed(b, shift)
    c = placed(torch.empty(33, 65, dtype=torch.bfloat16, device="cuda"), shift)
    ops.launch_linear_int8(a, sa, b, sb, c)
    check_product(c, a, sa, b, sb)


@pytest.mark.parametrize("m,n,k,lda,ldb,ldc", [(5, 40, 96, 112, 128, 48), (70, 96, 100, 112, 112, 101),
                                               (300, 264, 272, 288, 4096, 272), (3, 9, 33, 35, 40, 10),
                                               (1, 24, 64, 64, 80, 24)])
def test_linear_with_row_strides(m, n, k, lda, ldb, ldc):
    """Rows inside wider ones: the bytes between them are neither summed nor written."""
    a, sa, b, sb = operands(m, n, k, 4)
    wa = torch.full((m, lda), 99, dtype=torch.int8, device="cuda")
    wb = torch.full((n, ldb), -99, dtype=torch.int8, device="cuda")
    wa[:, :k], wb[:, :k] = a, b
    wc = torch.full((m, ldc), 5.0, dtype=torch.float16, device="cuda")
    capi.call("l2k_linear_int8", m, n, k, wa.data_ptr(), lda, sa.data_ptr(), wb.data_ptr(), ldb, sb.data_ptr(),
              wc.data_ptr(), ldc, capi.L2K_F16, torch.cuda.current_stream().cuda_stream)
    check_product(wc[:, :n], a, sa, b, sb)
    assert (wc[:, n:] == 5.0).all()


@pytest.mark.parametrize("m,k", [(2, 131056), (2, 131071), (130, 65536)])
def test_linear_of_the_largest_sums(m, k):
    """All bytes -128: 2^14 k, next to 2^31 for the longest rows."""
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    b[1] = 127
    one = torch.ones(m, device="cuda")
    c = torch.empty(m, 3, device="cuda")
    ops.launch_linear_int8(a, one, b, one[:1].expand(3).contiguous(), c)
    want = torch.tensor([16384 * k, -16256 * k, 16384 * k], dtype=torch.float64, device="cuda").float()
    assert torch.equal(c, want.expand(m, 3))


def test_products_on_two_streams():
    """Launches of all kinds on two streams at once, each ten times in a row."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    work = [[operands(*shape, seed) for shape in LINEAR_MIX] for seed in (1, 2)]
    outs = [[torch.empty(o[0].shape[0], o[2].shape[0], dtype=torch.bfloat16, device="cuda") for o in w] for w in work]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, w, cs in zip(streams, work, outs):
            with torch.cuda.stream(s):
                for (a, sa, b, sb), c in zip(w, cs):
                    ops.launch_linear_int8(a, sa, b, sb, c)
    torch.cuda.synchronize()
    for w, cs in zip(work, outs):
        for o, c in zip(w, cs):
            check_product(c, *o)


@pytest.mark.parametrize("m", [4, 300])
def test_linear_of_dead_rows(m):
    """Scale 0 gives zeros, scale NaN gives NaN over the whole row."""
    a, sa, b, sb = operands(m, 72, 160, 6)
    sa[1], sa[2] = 0, float("nan")
    a[2] = 0
    c = torch.empty(m, 72, dtype=torch.bfloat16, device="cuda")
    ops.launch_linear_int8(a, sa, b, sb, c)
    assert (c[1] == 0).all() and torch.isnan(c[2]).all() and torch.isfinite(c[3:]).all()


def test_lengths_of_zero():
    e = lambda *s, t=torch.float32: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
    i8 = torch.int8
    c = torch.full((3, 5), 9.0, device="cuda")
    ones = torch.ones(8, device="cuda")
    ops.launch_linear_int8(e(3, 0, t=i8), ones[:3], e(5, 0, t=i8), ones[:5], c)
    assert (c == 0).all()
    ops.launch_linear_int8(e(0, 16, t=i8), e(0), e(5, 16, t=i8), ones[:5], e(0, 5))
    ops.launch_linear_int8(e(3, 16, t=i8), ones[:3], e(0, 16, t=i8), e(0), e(3, 0))
    s = torch.full((4,), 9.0, device="cuda")
    ops.launch_quantize_rows_int8(e(4, 0), e(4, 0, t=i8), s)
    assert (s == 0).all()
    ops.launch_quantize_rows_int8(e(0, 4), e(0, 4, t=i8), e(0))
    ops.launch_swiglu_int8(e(0, 8), e(0, 4, t=i8), e(0))
    ops.launch_fused_add_residual_rmsnorm_int8(e(4), e(0, 4), e(0, 4), e(0, 4, t=i8), e(0), True)
    torch.cuda.synchronize()


# ----------------------------------------------------- together, as one uses them
def test_a_feed_forward_half_eager_streamed_and_captured():
    """x + o -> norm -> gate/up -> SwiGLU -> down on int8 rows: each product
    against 64 bits on the rows that reached it; the same bits on a side
    stream, two chains at once, and from a captured graph replayed on new inputs."""
    m, d, f = 70, 512, 1408
    t = torch.bfloat16
    g = gen(11)
    w_gu, w_down = (torch.randn(*s, generator=g, device="cuda") for s in ((2 * f, d), (d, f)))
    norm = (torch.rand(d, generator=g, device="cuda") + 0.5).to(t)
    e = lambda *s, dt=t: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
    weights = []
    for w in (w_gu, w_down):
        q, s = e(*w.shape, dt=torch.int8), e(w.shape[0], dt=torch.float32)
        ops.launch_quantize_rows_int8(w, q, s)
        weights += [q, s]

    def buffers():
        return dict(x=e(m, d), o=e(m, d), hq=e(m, d, dt=torch.int8), hs=e(m, dt=torch.float32), gu=e(m, 2 * f),
                    aq=e(m, f, dt=torch.int8), as_=e(m, dt=torch.float32), down=e(m, d))

    def chain(b):
        ops.launch_fused_add_residual_rmsnorm_int8(norm, b["x"], b["o"], b["hq"], b["hs"], True)
        ops.launch_linear_int8(b["hq"], b["hs"], weights[0], weights[1], b["gu"])
        ops.launch_swiglu_int8(b["gu"], b["aq"], b["as_"])
        ops.launch_linear_int8(b["aq"], b["as_"], weights[2], weights[3], b["down"])

    def fill(b, seed):
        h = gen(seed)
        b["x"].copy_(torch.randn(m, d, generator=h, device="cuda"))
        b["o"].copy_(torch.randn(m, d, generator=h, device="cuda"))

    eager, one, two, cap = (buffers() for _ in range(4))
    for seed in (1, 2):
        fill(eager, seed)
        chain(eager)
        check_product(eager["gu"], eager["hq"], eager["hs"], weights[0], weights[1])
        check_product(eager["down"], eager["aq"], eager["as_"], weights[2], weights[3])
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        fill(one, seed), fill(two, seed)
        for s, b in zip(streams, (one, two)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                chain(b)
        torch.cuda.synchronize()
        if seed == 1:
            fill(cap, 5)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                chain(cap)
        fill(cap, seed)
        graph.replay()
        torch.cuda.synchronize()
        for b in (one, two, cap):
            for k in ("x", "hq", "hs", "gu", "aq", "as_", "down"):
                assert torch.equal(b[k], eager[k]), k
