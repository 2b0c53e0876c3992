"""DecoderLayer(int8=True): every stage of a decode step and of a prefill pass
against the plain 64-bit formula on the tensors that reached it (the bars of
tests/test_gpu_int8.py), RoPE, caches and attention bit for bit against the same
operators on the same projections, and a captured step against the eager one."""
import pytest
import torch

from llama2_b200 import capi, ops
from llama2_b200.layer import DecoderLayer, Int8Weight
from tests.test_gpu_int8 import U, check_product, check_scales, gen, reference_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(cuda_lib):
    yield
    assert capi.lib().l2k_device_error(1) == 0


def check_norm(rows, x, w):
    y = x.double()
    want, scale = reference_rows(y * w.double())
    assert torch.equal(rows.q.double(), want)
    check_scales(rows.scales, scale / (y.square().mean(1) + 1e-5).sqrt(), 32 * U)


def check_rows(rows, x):
    want, scale = reference_rows(x.double())
    assert torch.equal(rows.q.double(), want)
    check_scales(rows.scales, scale, U)


def check_swiglu(rows, gate_up):
    g, u = gate_up.double().chunk(2, dim=1)
    y = g / (1 + torch.exp(-g)) * u
    want, scale = reference_rows(y)
    t = 127 * y / y.abs().amax(1, keepdim=True)
    near = ((t - t.floor()) - 0.5).abs() <= 1.5e-3
    assert ((rows.q.double() == want) | (near & ((rows.q.double() - want).abs() <= 1))).all()
    check_scales(rows.scales, scale, 96 * U)


def check_product_of(out, rows, w):
    check_product(out, rows.q, rows.scales, w.q, w.scales)


def add(x, y):
    return (x.float() + y.float()).to(x.dtype)


def check_after_attention(L, x1, x2, attn, b):
    check_rows(b["attn_q"], attn)
    check_product_of(b["o"], b["attn_q"], L.w_o)
    assert torch.equal(x2, add(x1, b["o"]))
    check_norm(b["h2"], x2, L.w_ffn_norm)
    check_product_of(b["gate_up"], b["h2"], L.w_gate_up)
    check_swiglu(b["act"], b["gate_up"])
    check_product_of(b["down"], b["act"], L.w_down)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("batch,pairing", [(1, 1), (5, 0), (70, 1)])
def test_decode(dtype, batch, pairing):
    d, heads, kvh, f, s = 512, 4, 2, 1408, 256
    layers = [DecoderLayer(d, heads, kvh, f, s, batch, dtype=dtype, seed=3 + i, pairing=pairing, int8=True)
              for i in range(2)]
    assert layers[0].launches_per_step() == 10
    g = gen(1)
    x = torch.randn(batch, d, generator=g, device="cuda").to(dtype)
    lens = torch.randint(1, s, (batch,), generator=torch.Generator().manual_seed(5))
    kv_lens = lens.to(torch.uint32).cuda()
    max_kv = torch.tensor([int(lens.max())], dtype=torch.uint32, device="cuda")
    is_done = torch.zeros(batch, dtype=torch.uint8, device="cuda")
    is_done[batch // 2] = batch > 1
    pending = None
    for L in layers:
        x0 = x.clone()
        k, v, q = L.k_cache.clone(), L.v_cache.clone(), L.q.clone()
        down = L.decode(x, pending, kv_lens, max_kv, is_done)
        x1 = x0 if pending is None else add(x0, pending)
        check_norm(L.h, x1, L.w_attn_norm)
        check_product_of(L.qkv, L.h, L.w_qkv)
        rope = (ops.launch_fused_reshape_rope_kvcache_llama2_decode if pairing
                else ops.launch_fused_reshape_rope_kvcache_decode)
        rope(L.qkv, is_done, kv_lens, q, k, v)
        assert torch.equal(q, L.q) and torch.equal(k, L.k_cache) and torch.equal(v, L.v_cache)
        qk, attn = torch.zeros_like(L.qk), torch.empty_like(L.attn)
        ops.decode_attention(q, k, v, kv_lens, max_kv, qk, attn)
        assert torch.equal(attn, L.attn)
        check_after_attention(L, x1, x, L.attn.view(batch, d),
                              dict(attn_q=L.attn_q, o=L.o, h2=L.h2, gate_up=L.gate_up, act=L.act, down=down))
        pending = down

    # the second layer's step as a graph, on the inputs it had
    L = layers[1]
    want = [t.clone() for t in (x, L.down, L.k_cache)]
    x.copy_(x0)
    graph = L.capture_decode(x, layers[0].down, kv_lens, max_kv, is_done)
    x.copy_(x0)
    L.down.zero_()
    graph.replay()
    for got, w in zip((x, L.down, L.k_cache), want):
        assert torch.equal(got, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prefill(dtype):
    """Two prompts (64 and 40 new tokens after 0 and 10 cached ones)."""
    b, d, heads, kvh, f, s, qc = 2, 256, 2, 2, 512, 128, 64
    L = DecoderLayer(d, heads, kvh, f, s, b, dtype=dtype, seed=20, int8=True)
    q_lens = torch.tensor([64, 40], dtype=torch.uint32, device="cuda")
    kv_lens = torch.tensor([64, 50], dtype=torch.uint32, device="cuda")
    t = 104
    unpad = torch.zeros(b, qc, dtype=torch.uint32, device="cuda")
    offsets = torch.zeros(b, dtype=torch.uint32, device="cuda")
    ops.launch_build_padding_index_maps(t, q_lens, unpad, offsets)
    assert L.launches_per_prefill(t) == 12
    g = gen(2)
    x = torch.randn(t, d, generator=g, device="cuda").to(dtype)
    pending = torch.randn(t, d, generator=g, device="cuda").to(dtype)
    x0, k, v = x.clone(), L.k_cache.clone(), L.v_cache.clone()
    down = L.prefill(x, pending, q_lens, kv_lens, 64, 64, unpad)
    buf = L._prefill_buffers(t, qc)
    x1 = add(x0, pending)
    check_norm(buf["h"], x1, L.w_attn_norm)
    check_product_of(buf["qkv"], buf["h"], L.w_qkv)
    q = torch.zeros_like(buf["q"])
    ops.launch_fused_pad_reshape_transpose_rope_kvcache_llama2(buf["qkv"], q_lens, kv_lens, unpad.view(-1), q, k, v)
    assert torch.equal(q, buf["q"]) and torch.equal(k, L.k_cache) and torch.equal(v, L.v_cache)
    check_after_attention(L, x1, x, buf["attn"], {**buf, "down": down})


def test_int8_weights_of_a_16_bit_layer():
    """The same seed gives the 16-bit layer's weights; each int8 one is its
    quantised transpose, and takes another layer's in place."""
    kw = dict(dim=256, heads=2, kv_heads=2, hidden=512, kv_cache_len=64, batch=2)
    plain, L = DecoderLayer(**kw, seed=4), DecoderLayer(**kw, seed=4, int8=True)
    other = DecoderLayer(**kw, seed=5)
    for name in ("w_qkv", "w_o", "w_gate_up", "w_down"):
        w = L.weights()[name]
        assert isinstance(w, Int8Weight)
        check_rows(w, plain.weights()[name].t())
        ptr = w.q.data_ptr()
        w.assign(other.weights()[name])
        assert w.q.data_ptr() == ptr
        check_rows(w, other.weights()[name].t())
