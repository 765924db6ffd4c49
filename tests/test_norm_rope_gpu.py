"""GPU tests of the query/key norms with the rotation (sfb_qk_norm_rope)
against the formula in 64 bits.

Tolerance per element: half a step of the output type on the value, plus 2^-19
of the size of its pair for the fp32 arithmetic (a sum of up to 256 squares as
8 + 5 additions, a division, a square root, a division, three products and an
addition, each within 2^-24: below 24 · 2^-24), plus half a step of the type's
subnormal range: fp16 values below 2^-14 are multiples of 2^-24, so their
rounding is off by up to 2^-25 however small the value is (bf16 and fp32: 2^-134
and 2^-150, nothing here)."""
import pytest
import torch

from servoflow_b200 import _capi
from servoflow_b200.backend import B200Backend

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


@pytest.fixture(scope="module")
def be(gpu):
    b = B200Backend(0)
    b.device_error(reset=True)
    yield b
    assert b.device_error(reset=True) == 0


def tables(n, rot, dev):
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return a.cos().float().to(dev), a.sin().float().to(dev)


def ref64(x, w, cos, sin, pos, eps, inter, norm=True):
    """x [B, S, H, D] -> (result, size of each element's pair), fp64."""
    y = x.double()
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.double()
    size = y.abs()
    if cos is not None:
        rot = 2 * cos.shape[1]
        c, s = cos.double()[pos.long()][:, :, None], sin.double()[pos.long()][:, :, None]
        i = torch.arange(rot // 2, device=x.device)
        ia, ib = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        a, b = y[..., ia].clone(), y[..., ib].clone()
        y, size = y.clone(), size.clone()
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia] = size[..., ib] = torch.hypot(a, b)
    return y, size


def check(got, ref, size, dt):
    err = (got.double() - ref).abs()
    tol = HALF[dt] * ref.abs() + 2.0 ** -19 * size + TINY[dt]
    assert not torch.isnan(got).any()
    assert (err <= tol).all(), f"max excess {(err - tol).max().item():.3e}"


def run(be, gpu, B, S, H, Hkv, D, rot, dt, inter=False, layout="bshd", positions="random", weights=True, seed=0,
        norm=True, inplace=False):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(B, S, H + 2 * Hkv, D, generator=g) * 2).to(dt).to(gpu)
    q, k = qkv[:, :, :H], qkv[:, :, H:H + Hkv]
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dt).to(gpu) for _ in range(2)) if weights else (None, None)
    cos, sin = tables(S + 300, rot, gpu) if rot else (None, None)
    pos = torch.randint(0, S + 300, (B, S), generator=g, dtype=torch.int32).to(gpu) if positions == "random" else None
    p64 = pos if pos is not None else torch.arange(S, device=gpu).expand(B, S)
    refs = [ref64(x, w, cos, sin, p64, 1e-6, inter, norm) for x, w in ((q, wq), (k, wk))]
    if layout == "bhsd":
        q, k = q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous()
    qo, ko = (q, k) if inplace else (torch.full_like(q, float("nan")), torch.full_like(k, float("nan")))
    v0 = qkv[:, :, H + Hkv:].clone()
    be.qk_norm_rope(q, k, qo, ko, wq, wk, cos, sin, positions=pos, norm=norm, interleaved=inter, layout=layout)
    for o, (r, size) in zip((qo, ko), refs):
        check(o.transpose(1, 2) if layout == "bhsd" else o, r, size, dt)
    assert torch.equal(qkv[:, :, H + Hkv:], v0)        # V, between the keys of two tokens, is untouched


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 32), (64, 0), (128, 128), (128, 48), (96, 96), (96, 32), (256, 256),
                                   (8, 0), (72, 64)])
@pytest.mark.parametrize("inter", [False, True])
def test_head_sizes(be, gpu, dt, D, rot, inter):
    run(be, gpu, 2, 5, 3, 2, D, rot, dt, inter, seed=D + rot)


@pytest.mark.parametrize("B,S,H,Hkv", [(1, 1, 1, 1), (1, 1, 32, 32), (3, 67, 32, 8), (2, 1000, 7, 1), (32, 67, 32, 32)])
@pytest.mark.parametrize("layout", ["bshd", "bhsd"])
def test_sizes_and_layouts(be, gpu, B, S, H, Hkv, layout):
    run(be, gpu, B, S, H, Hkv, 64, 64, torch.bfloat16, layout=layout, seed=S)


def test_default_positions_no_weights_no_norm(be, gpu):
    run(be, gpu, 2, 33, 4, 4, 64, 64, torch.float32, positions=None, weights=False)
    run(be, gpu, 2, 33, 4, 4, 64, 64, torch.bfloat16, norm=False)
    run(be, gpu, 2, 33, 4, 4, 128, 0, torch.float16, norm=False)


@pytest.mark.parametrize("inter", [False, True])
def test_in_place(be, gpu, inter):
    run(be, gpu, 2, 9, 4, 2, 64, 64, torch.bfloat16, inter=inter, inplace=True)


def test_queries_or_keys_alone(be, gpu):
    q = torch.randn(2, 3, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(gpu)
    cos, sin = tables(10, 64, gpu)
    both_q, both_k, alone_q, alone_k = (torch.empty_like(q) for _ in range(4))
    be.qk_norm_rope(q, q, both_q, both_k, cos=cos, sin=sin, layout="bshd")
    be.qk_norm_rope(q, None, alone_q, None, cos=cos, sin=sin, layout="bshd")
    be.qk_norm_rope(None, q, None, alone_k, cos=cos, sin=sin, layout="bshd")
    assert torch.equal(both_q, alone_q) and torch.equal(both_k, alone_k) and torch.equal(both_q, both_k)


def test_zero_and_nan_rows(be, gpu):
    x = torch.zeros(1, 3, 2, 64, device=gpu).bfloat16()
    x[0, 1, 0, 5] = float("nan")
    x[0, 2, 1] = 1e-30                                  # far below sqrt(eps)
    out = torch.empty_like(x)
    be.qk_norm_rope(x, None, out, None, layout="bshd")
    assert torch.isnan(out[0, 1, 0]).all()
    out[0, 1, 0] = 0
    assert not torch.isnan(out).any() and (out[0, 0] == 0).all() and (out[0, 1, 1] == 0).all()


def test_positions_outside_the_tables(be, gpu):
    q = torch.randn(1, 4, 2, 64, generator=torch.Generator().manual_seed(4)).bfloat16().to(gpu)
    cos, sin = tables(8, 64, gpu)
    out = torch.zeros_like(q)
    pos = torch.tensor([[0, 8, -1, 7]], dtype=torch.int32, device=gpu)
    assert be.device_error(reset=True) == 0
    be.qk_norm_rope(q, None, out, None, cos=cos, sin=sin, positions=pos, layout="bshd")
    torch.cuda.synchronize()
    assert be.device_error(reset=True) == _capi.SFB_ERR_RANGE
    assert (out[0, 1:3] == 0).all() and (out[0, 0] != 0).any() and (out[0, 3] != 0).any()


def test_graph_replay_and_side_stream(be, gpu):
    q = torch.randn(2, 67, 8, 64, generator=torch.Generator().manual_seed(5)).bfloat16().to(gpu)
    cos, sin = tables(100, 64, gpu)
    a, b, c = (torch.empty_like(q) for _ in range(3))
    be.qk_norm_rope(q, None, a, None, cos=cos, sin=sin, layout="bshd")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        be.qk_norm_rope(q, None, b, None, cos=cos, sin=sin, layout="bshd")
    g.replay()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    be.qk_norm_rope(q, None, c, None, cos=cos, sin=sin, layout="bshd", stream=s)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)


def test_wrapper_refusals(be, gpu):
    q = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16, device=gpu)
    cos, sin = tables(8, 64, gpu)
    E = _capi.SfbError
    with pytest.raises(E):
        be.qk_norm_rope(q, None, None, None)
    with pytest.raises(E):
        be.qk_norm_rope(q, q.half(), q, q.half())
    with pytest.raises(E):
        be.qk_norm_rope(q, None, q, None, cos=cos)
    with pytest.raises(E):
        be.qk_norm_rope(q, None, q, None, cos=cos.double(), sin=sin.double())
    with pytest.raises(E):
        be.qk_norm_rope(q, None, q, None, cos=cos, sin=sin, positions=torch.zeros(1, 3, dtype=torch.int64, device=gpu))
    with pytest.raises(E):
        be.qk_norm_rope(q, None, q, None, q_weight=torch.ones(32, dtype=torch.bfloat16, device=gpu))
    with pytest.raises(ValueError):
        be.qk_norm_rope(q, None, q, None, cos=cos.cpu(), sin=sin.cpu())
    with pytest.raises(ValueError):
        be.qk_norm_rope(q, None, q, None, layout="hbsd")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,rot", [(64, 32), (128, 16), (256, 96), (72, 64)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,S", [(1, 3), (40, 100)])
def test_channels_past_the_rotated_ones_pass_through(be, gpu, dt, D, rot, inter, B, S):
    """The rotation covers the first rotary_dim channels: without a norm the others are
    copies, infinities, NaN and the sign of a zero included, and touch no neighbour."""
    H = 16                                             # 40 x 100 tokens take four heads a thread
    x = torch.randn(B, S, H, D, generator=torch.Generator().manual_seed(D)).to(dt).to(gpu)
    x[:, :, 0, rot] = float("inf")
    x[:, :, 1, D - 1] = -float("inf")
    x[:, :, 2, rot + 3] = float("nan")
    x[:, :, H - 1, rot + 4] = -0.0
    out = torch.empty_like(x)
    cos, sin = tables(S, rot, gpu)
    be.qk_norm_rope(x, None, out, None, cos=cos, sin=sin, norm=False, interleaved=inter, layout="bshd")
    bits = torch.int32 if dt == torch.float32 else torch.int16
    same = (out.view(bits) == x.view(bits)) | (out.isnan() & x.isnan())
    assert same[..., rot:].all()
    pos = torch.arange(S, device=gpu).expand(B, S)
    ref, size = ref64(x, None, cos, sin, pos, 0.0, inter, norm=False)
    check(out[..., :rot], ref[..., :rot], size[..., :rot], dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,rot,S", [(64, 64, 1100), (64, 0, 1100), (96, 32, 550), (128, 128, 550), (256, 256, 300)])
@pytest.mark.parametrize("H,Hkv", [(6, 1), (5, 3)])
@pytest.mark.parametrize("inter", [False, True])
def test_four_heads_a_thread(be, gpu, dt, D, rot, S, H, Hkv, inter):
    """Sizes at which a thread takes four heads (1536 threads an SM with one head each),
    with head counts that leave its last group part empty."""
    B, lanes = 4, 8 if D <= 64 else 16 if D <= 128 else 32
    assert B * S * (H + Hkv) * lanes >= torch.cuda.get_device_properties(gpu).multi_processor_count * 1536
    run(be, gpu, B, S, H, Hkv, D, rot, dt, inter, seed=S + H)
    run(be, gpu, B, S, H, Hkv, D, rot, dt, inter, layout="bhsd", norm=False, weights=False, inplace=True, seed=S + H + 1)
