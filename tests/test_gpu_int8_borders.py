"""The norm's 8-bit values of fp32 rows at and next to the borders between two
integers, against whole-number arithmetic. x w of fp32 data has up to 48 bits, so
127 x w has more than fp64 holds: the expected bytes are computed from the operands
as fractions. Equal bytes are asked for: q has one right value."""
from fractions import Fraction

import pytest
import torch

from llama2_b200 import capi, ops
from tests.test_gpu_int8 import gen, placed

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(cuda_lib):
    yield
    assert capi.lib().l2k_device_error(1) == 0


def expected(x, w):
    """rne(127 x w / max |x w|) of a row of finite values, exactly (round() of a Fraction: ties to even)."""
    y = [Fraction(a) * Fraction(b) for a, b in zip(x.double().tolist(), w.double().tolist())]
    a = max(map(abs, y))
    return [round(127 * v / a) for v in y]


def check(x, w, rows):
    """The bytes of `rows` of x; every other row repeats one of them."""
    n, dim = x.shape
    q, s = torch.empty(n, dim, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    ops.launch_fused_add_residual_rmsnorm_int8(w, x, None, q, s, False)
    for i in rows:
        want = torch.tensor(expected(x[i], w), dtype=torch.int8)
        assert torch.equal(q[i].cpu(), want), (i, torch.nonzero(q[i].cpu() != want)[:4])


def odd_parts(dim, seed):
    """Rows whose x are odd multiples of p and whose largest is 254 p: each of them on a border."""
    g = gen(seed)
    p = torch.randint(2 ** 15, 2 ** 16, (1, 1), generator=g, device="cuda").float()
    odd = torch.randint(-127, 127, (1, dim), generator=g, device="cuda") * 2 + 1
    x = odd * p
    x[0, dim // 3] = 254 * p[0, 0]
    return x


# one row per CTA; several rows per CTA, aligned and not; rows longer than the stream kernel holds
SHAPES = [(16, 64), (7, 8200), (16, 67), (700, 64), (700, 67), (700, 1000), (2, 16392)]


@pytest.mark.parametrize("scale", [0, -75, 40])  # 2^scale on x and w: a below 2^-100 and above 2^100 too
@pytest.mark.parametrize("n,dim", SHAPES)
def test_borders(n, dim, scale):
    """One weight value for the whole row leaves the borders of x on borders."""
    distinct = 3
    for seed in range(4):
        w = torch.rand(1, generator=gen(seed), device="cuda").add(0.5).expand(dim).contiguous() * 2.0 ** scale
        x = torch.cat([odd_parts(dim, 10 * seed + i) for i in range(distinct)]) * 2.0 ** (scale - 16)
        x = x[torch.arange(n, device="cuda") % distinct].contiguous()
        check(x, w, range(min(distinct, n)))
        # a step of fp32 to either side
        up = torch.where(torch.arange(dim, device="cuda") % 2 == 0, torch.full_like(x, float("inf")),
                         torch.full_like(x, -float("inf")))
        near = torch.where(x.abs() == x.abs().amax(1, keepdim=True), x, torch.nextafter(x, up))
        check(near, w, range(min(distinct, n)))


def test_halves_of_the_largest():
    """x = max / 2 is 63.5 exactly, so 64, whatever the weight's bits."""
    g = gen(3)
    for _ in range(64):
        top, weight = (torch.rand(1, generator=g, device="cuda") + 1).tolist(), torch.rand(1, generator=g, device="cuda") + 0.5
        x = torch.full((2, 16), top[0] / 2, device="cuda")
        x[:, 5] = top[0]
        x[1] *= -1
        q, s = torch.empty(2, 16, dtype=torch.int8, device="cuda"), torch.empty(2, device="cuda")
        ops.launch_fused_add_residual_rmsnorm_int8(weight.expand(16).contiguous(), x, None, q, s, False)
        want = torch.full((16,), 64, dtype=torch.int8, device="cuda")
        want[5] = 127
        assert torch.equal(q[0], want) and torch.equal(q[1], -want)


# whole numbers x, w, X, W below 2^24: 254 x w is 1 or 2 from an odd multiple of X W, closer to the
# border than fp64 tells x w apart
CLOSE = [(11280743, 15509936, 13015690, 13495647), (12490603, 14967011, 15149076, 12487984),
         (11058155, 15664790, 16255182, 10783889), (9576680, 15159721, 9425887, 15586333),
         (10837367, 15322268, 12893635, 16274555), (8847631, 15609673, 16226296, 8545050),
         (6989851, 7499773, 10262608, 9904230), (6323468, 15375842, 8776775, 14731929)]


@pytest.mark.parametrize("n,dim", [(1, 8), (700, 8), (700, 9), (2, 16392)])
@pytest.mark.parametrize("x0,w0,x1,w1", CLOSE)
def test_next_to_a_border(n, dim, x0, w0, x1, w1):
    x, w = torch.zeros(n, dim, device="cuda"), torch.ones(dim, device="cuda")
    x[:, 0], w[0] = x0, w0
    x[:, 1], w[1] = x1, w1
    x[:, 2], w[2] = -x0, w0
    check(x, w, [0, n - 1])
    check(placed(x, 1), w, [n - 1])


def test_products_past_the_range_of_fp32():
    """bf16 products x w are formed in fp32: a row with one beyond it counts as holding an infinity."""
    x = torch.full((2, 64), 2.0 ** 60, device="cuda", dtype=torch.bfloat16)
    w = torch.full((64,), 2.0 ** 66, device="cuda", dtype=torch.bfloat16)
    x[1, 9] = 2.0 ** 62
    q, s = torch.empty(2, 64, dtype=torch.int8, device="cuda"), torch.empty(2, device="cuda")
    ops.launch_fused_add_residual_rmsnorm_int8(w, x, None, q, s, False)
    assert (q[0] == 127).all() and torch.isfinite(s[0]) and (q[1] == 0).all() and torch.isnan(s[1])
