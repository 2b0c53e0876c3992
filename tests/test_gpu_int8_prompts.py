"""The 8-bit row operators on prompts: every kernel that many rows are streamed with,
several rows to a CTA, and the int8 layer's prefill on them. The bars are those of
tests/test_gpu_int8.py (at most 32 elements to a thread and 16 warps here too).

Which kernel takes a shape follows from groups of 8 elements, G = ceil(dim / 8), from
297 rows on (aligned) or always (rows of no alignment): one, two or four groups to a
thread; at most 512 threads, or held to the registers with which an SM takes two CTAs
of 320 (fp32 norms of 513 to 640 groups) or 448 threads (four groups, 1281 to 1792;
fp32 ragged rows)."""
import pytest
import torch

from llama2_b200 import capi, ops
from llama2_b200.layer import DecoderLayer
from tests.test_gpu_int8 import DTYPES, U, _check_norm, _check_swiglu, check_scales, check_untouched, gen, placed, \
    reference_rows, row_outputs
from tests.test_gpu_int8_layer import add, check_after_attention, check_norm, check_product_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(cuda_lib):
    yield
    assert capi.lib().l2k_device_error(1) == 0


# aligned
ALIGNED = [(3000, 256),     # one group to a thread, one warp to a CTA
           (800, 512),      # 64 groups: two to a thread
           (500, 1024),     # two groups of few rows
           (2500, 520),     # 65 groups: the first length with four groups to a thread of 16 bits
           (2500, 4096),    # four groups (fp32: two)
           (1500, 5120),    # fp32 norms of 320 threads
           (1200, 8200),    # 1025 groups: fp32 from two groups to four
           (1000, 10248),   # 1281 groups: the first of 448 threads
           (1000, 11008), (1000, 13824),
           (900, 14344),    # 1793 groups: four again, of 512 threads
           (700, 16384)]    # the longest row; fp32 SwiGLU and added norms have a ring of one row
# lengths and places of no alignment
RAGGED = [(2500, 4095), (1500, 5119), (1000, 10243), (1000, 13799), (700, 16381), (400, 4097), (3000, 255)]


def check_rows(x, shift=0):
    n, dim = x.shape
    q, s, qs, ss = row_outputs(n, dim, shift)
    ops.launch_quantize_rows_int8(x, q, s)
    want, scale = reference_rows(x.double())
    assert torch.equal(q.double(), want)
    check_scales(s, scale, U)
    check_untouched(n, dim, shift, qs, ss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim,shift", [(*s, 0) for s in ALIGNED + RAGGED] + [(1000, 4096, 3), (700, 13824, 8)])
@pytest.mark.parametrize("op", ["rows", "norm", "norm added", "swiglu"])
def test_streamed_rows(op, n, dim, shift, dtype):
    g = gen(dim + n)
    x = (torch.randn(n, dim * (2 if op == "swiglu" else 1), generator=g, device="cuda") * 2).to(dtype)
    x[n // 3] = 0  # padding between rows
    x[-1] = 0
    x = placed(x, shift)
    if op == "rows":
        check_rows(x, shift)
    elif op == "swiglu":
        _check_swiglu(x, n, dim, shift)
    else:
        r = torch.randn(n, dim, generator=g, device="cuda").to(dtype)
        r[n // 3] = 0
        w = (torch.rand(dim, generator=g, device="cuda") + 0.5).to(dtype)
        _check_norm(x, placed(r, shift), placed(w, shift), op == "norm added", shift)


@pytest.mark.parametrize("op", ["rows", "norm added", "swiglu"])
@pytest.mark.parametrize("n,dim,dtype", [(2500, 4096, torch.bfloat16), (1000, 13824, torch.float16),
                                         (1500, 5120, torch.float32), (1000, 4095, torch.bfloat16)])
def test_rows_that_are_not_finite_stay_alone(op, n, dim, dtype):
    """A NaN or an infinity marks its own row, at either end of it, and no other row of its CTA."""
    g = gen(n)
    t = {"dtype": dtype, "device": "cuda"}
    x = torch.randn(n, dim * (2 if op == "swiglu" else 1), generator=g, device="cuda").to(dtype)
    bad = torch.arange(0, n, 7, device="cuda")
    x[bad[0::2], 0] = float("nan")
    x[bad[1::2], -1] = float("inf")
    q, s, qs, ss = row_outputs(n, dim)
    clean = x.clone()
    clean[bad] = 1
    q2, s2, _, _ = row_outputs(n, dim)
    if op == "rows":
        ops.launch_quantize_rows_int8(x, q, s)
        ops.launch_quantize_rows_int8(clean, q2, s2)
    elif op == "swiglu":
        ops.launch_swiglu_int8(x, q, s)
        ops.launch_swiglu_int8(clean, q2, s2)
    else:
        r, w = torch.randn(n, dim, generator=g, device="cuda").to(dtype), torch.ones(dim, **t)
        ops.launch_fused_add_residual_rmsnorm_int8(w, x, r, q, s, True)
        ops.launch_fused_add_residual_rmsnorm_int8(w, clean, r, q2, s2, True)
    assert (q[bad] == 0).all() and torch.isnan(s[bad]).all()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[bad] = False
    assert torch.equal(q[rest], q2[rest]) and torch.equal(s[rest], s2[rest]) and torch.isfinite(s2).all()
    check_untouched(n, dim, 0, qs, ss)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_of_the_layer(dtype):
    """750 tokens of two prompts: every norm, row and SwiGLU of the layer streamed."""
    b, d, heads, kvh, f, qc = 2, 1024, 8, 4, 2816, 450
    L = DecoderLayer(d, heads, kvh, f, 512, b, dtype=dtype, seed=8, int8=True)
    q_lens = torch.tensor([450, 300], dtype=torch.uint32, device="cuda")
    kv_lens = torch.tensor([450, 312], dtype=torch.uint32, device="cuda")
    t = 750
    unpad = torch.zeros(b, qc, dtype=torch.uint32, device="cuda")
    offsets = torch.zeros(b, dtype=torch.uint32, device="cuda")
    ops.launch_build_padding_index_maps(t, q_lens, unpad, offsets)
    g = gen(6)
    x = torch.randn(t, d, generator=g, device="cuda").to(dtype)
    pending = torch.randn(t, d, generator=g, device="cuda").to(dtype)
    x0 = x.clone()
    down = L.prefill(x, pending, q_lens, kv_lens, 450, 450, unpad)
    buf = L._prefill_buffers(t, qc)
    x1 = add(x0, pending)
    check_norm(buf["h"], x1, L.w_attn_norm)
    check_product_of(buf["qkv"], buf["h"], L.w_qkv)
    check_after_attention(L, x1, x, buf["attn"], {**buf, "down": down})
