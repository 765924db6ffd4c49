"""GPU tests of the 4-bit-weight linear layer (sfb_w4a16_linear) against the
formula in 64 bits.

Tolerance per element: half a step of the output type on the value, plus
1.2 · 2^-17 of Σ|x||w| + |bias| for the fp32 sums (products of x and the codes
are exact; a group of 128 is 8 MMA steps, then up to 256 groups over 8 warps
and 8 partial sums: at most about 50 additions in a chain, each within 2^-23;
1.2 bounds the slope of GELU and SiLU), plus 2^-20 of the activation's value
and 2^-24 of the residual sum, and 2^-25 for fp16 outputs below 2^-14, which are
multiples of 2^-24."""
import math

import pytest
import torch

from servoflow_b200 import _capi
from servoflow_b200.backend import B200Backend
from servoflow_b200.quant4 import pack_codes, pack_w4, unpack_codes

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def be(gpu):
    b = B200Backend(0)
    b.device_error(reset=True)
    yield b
    assert b.device_error(reset=True) == 0


def check(be, gpu, M, N, K, G, dt=torch.bfloat16, ydt=None, sdt=torch.float16, act="none", bias=True, res=False, seed=0,
          ldx=None):
    ydt = ydt or dt
    g = torch.Generator().manual_seed(seed)
    # every code, the unused -8 too, and scales over three orders of magnitude
    codes = torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int32)
    s = (torch.rand(N, K // G, generator=g) * 0.02 * 10 ** (-3 * torch.rand(N, K // G, generator=g))).to(sdt)
    x = torch.randn(M, ldx or K, generator=g).to(dt).to(gpu)[:, :K]
    b = torch.randn(N, generator=g).mul(0.3).to(dt).to(gpu) if bias else None
    r = torch.randn(M, N, generator=g).to(ydt).to(gpu) if res else None
    wq, s = pack_codes(codes).to(gpu), s.to(gpu)
    out = torch.full((M, N), float("nan"), dtype=ydt, device=gpu)
    be.w4a16_linear(x, wq, s, out, bias=b, residual=r, act=act)
    w = codes.to(gpu).double() * s.double().repeat_interleave(G, 1)
    y = x.double() @ w.t()
    mag = x.double().abs() @ w.abs().t()
    if b is not None:
        y, mag = y + b.double(), mag + b.double().abs()
    if act == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    elif act == "silu":
        y = y * torch.sigmoid(y)
    tol = 1.2 * 2.0 ** -17 * mag + 2.0 ** -20 * y.abs()
    if r is not None:
        y = y + r.double()
        tol = tol + 2.0 ** -24 * y.abs()
    err = (out.double() - y).abs()
    tol = tol + HALF[ydt] * (y.abs() + tol) + (2.0 ** -25 if ydt == torch.float16 else 0.0)
    assert not torch.isnan(out).any()
    assert (err <= tol).all(), f"max excess {(err - tol).max().item():.3e}, max err {err.max().item():.3e}"
    return x, wq, s, out


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 2, 8, 9, 17, 33, 67, 73, 150])
def test_rows(be, gpu, G, dt, M):
    check(be, gpu, M, 96, 512, G, dt, seed=M)


@pytest.mark.parametrize("N", [1, 7, 15, 16, 17, 33, 250, 2048])
@pytest.mark.parametrize("M", [1, 67])
def test_channels(be, gpu, N, M):
    check(be, gpu, M, N, 256, 64, seed=N, res=True)


@pytest.mark.parametrize("G,K", [(32, 32), (32, 96), (64, 64), (64, 192), (64, 1088), (128, 128), (128, 1152), (32, 2080),
                                 (128, 8192)])
@pytest.mark.parametrize("M", [1, 20, 67])
def test_depths(be, gpu, G, K, M):
    check(be, gpu, M, 40, K, G, seed=K, ydt=torch.float32)


@pytest.mark.parametrize("sdt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("M", [1, 67])
def test_scales_and_activations(be, gpu, sdt, act, M):
    check(be, gpu, M, 128, 512, 64, sdt=sdt, act=act, res=True, seed=3)
    check(be, gpu, M, 128, 512, 64, sdt=sdt, act=act, bias=False, ydt=torch.float32, seed=4)


def test_strided_rows_and_aliased_residual(be, gpu):
    check(be, gpu, 5, 48, 256, 128, ldx=264, seed=5)
    x, wq, s, want = check(be, gpu, 5, 48, 256, 128, bias=False, seed=6)
    buf = torch.randn(5, 96, generator=torch.Generator().manual_seed(7)).bfloat16().to(gpu)
    y, keep = buf[:, :48], buf[:, 48:].clone()
    r = y.clone()
    be.w4a16_linear(x, wq, s, y, residual=y)                # the residual may be the output
    sep = torch.empty_like(want)
    be.w4a16_linear(x, wq, s, sep, residual=r)
    assert torch.equal(y, sep) and torch.equal(buf[:, 48:], keep)


def test_packed_weight_roundtrip(be, gpu):
    w = torch.randn(64, 256, generator=torch.Generator().manual_seed(8)) * 0.02
    wq, s = pack_w4(w, 64)
    x = torch.eye(256, dtype=torch.float16, device=gpu)     # rows of the identity read the weights back
    out = torch.empty(256, 64, dtype=torch.float32, device=gpu)
    be.w4a16_linear(x, wq.to(gpu), s.to(gpu), out)
    back = unpack_codes(wq).float() * s.float().repeat_interleave(64, 1)
    assert torch.equal(out.cpu().t(), back)


def test_same_bits_twice_and_in_a_graph(be, gpu):
    x, wq, s, a = check(be, gpu, 67, 512, 1024, 64, seed=9, bias=False)
    b, c = torch.empty_like(a), torch.empty_like(a)
    be.w4a16_linear(x, wq, s, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        be.w4a16_linear(x, wq, s, c)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)


def test_wrapper_refusals(be, gpu):
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=gpu)
    wq = torch.zeros(16, 64, dtype=torch.uint8, device=gpu)
    s = torch.zeros(16, 2, dtype=torch.float16, device=gpu)
    y = torch.empty(2, 16, dtype=torch.bfloat16, device=gpu)
    E = _capi.SfbError
    be.w4a16_linear(x, wq, s, y)
    with pytest.raises(E):
        be.w4a16_linear(x.float(), wq, s, y)
    with pytest.raises(E):
        be.w4a16_linear(x, wq, s, y.half())
    with pytest.raises(E):
        be.w4a16_linear(x, wq.to(torch.int8), s, y)
    with pytest.raises(E):
        be.w4a16_linear(x, wq, torch.zeros(16, 8, dtype=torch.float16, device=gpu), y)      # group 16
    with pytest.raises(E):
        be.w4a16_linear(x, wq, torch.zeros(15, 2, dtype=torch.float16, device=gpu), y)
    with pytest.raises(E):
        be.w4a16_linear(x, wq, s, y[:, :15])
    with pytest.raises(E):
        be.w4a16_linear(x, wq, s, y, bias=torch.zeros(16, device=gpu))
    with pytest.raises(E):
        be.w4a16_linear(x, wq, s, y, residual=torch.zeros(2, 16, device=gpu))
    with pytest.raises(ValueError):
        be.w4a16_linear(x, wq, s, y, act="relu")
    with pytest.raises(ValueError):
        be.w4a16_linear(x, wq.cpu(), s, y)


def test_more_row_tiles_than_65535(be, gpu):
    """Any M: 4.8 million rows are 66 thousand tiles of 72."""
    M, N, K, G = 4_800_001, 8, 32, 32
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int32)
    s = (torch.rand(N, 1, generator=g) * 0.02).half()
    x = torch.randn(M, K, generator=torch.Generator(device=gpu).manual_seed(2), device=gpu).bfloat16()
    r = torch.randn(M, N, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu)
    out = torch.full((M, N), float("nan"), dtype=torch.float32, device=gpu)
    be.w4a16_linear(x, pack_codes(codes).to(gpu), s.to(gpu), out, residual=r)
    w = (codes.double() * s.double()).to(gpu)
    y = x.double() @ w.t() + r.double()
    tol = (1.2 * 2.0 ** -17 + 2.0 ** -24) * (x.double().abs() @ w.abs().t()) + (2.0 ** -20 + 2.0 ** -24) * y.abs()
    assert ((out.double() - y).abs() <= tol).all()


@pytest.mark.parametrize("G,K", [(32, 288), (64, 320), (128, 384)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 8, 13, 16])
def test_few_rows_of_a_wide_layer(be, gpu, G, K, dt, M):
    """Up to 16 rows with 32 channels a CTA: taken from two such CTAs an SM."""
    N = 2 * torch.cuda.get_device_properties(gpu).multi_processor_count * 32 + 5
    check(be, gpu, M, N, K, G, dt, act="silu", res=True, seed=M)
    check(be, gpu, M, N, K, G, dt, ydt=torch.float32, sdt=torch.bfloat16, seed=M + 1)


@pytest.mark.parametrize("G,K", [(32, 608), (64, 1088), (128, 640)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [17, 32, 67, 72, 150])
def test_more_rows_of_a_wide_layer(be, gpu, G, K, dt, M):
    """More rows with 64 channels a CTA: taken once those fill half the SMs."""
    N = torch.cuda.get_device_properties(gpu).multi_processor_count * 32 + 7
    check(be, gpu, M, N, K, G, dt, act="gelu", res=True, seed=M)
    check(be, gpu, M, N, K, G, dt, ydt=torch.float32, sdt=torch.float32, seed=M + 1)
