"""GPU tests of the 4-bit K/V cache (append, read back) and of the attention
over it, against plain implementations in 64 bits.

Append and read are exact: same scales and codes, same values.

Attention tolerance, per output element: half a step of the output type on the
value, plus what the kernel's fp16 probabilities and fp32 sums may add:
  Σ p|v| · (2^-11 + 2^-15)   the probabilities rounded to fp16 (half a step is
                             2^-11), and 2^-15 for everything in fp32: logits
                             of at most 2^6 with a relative error of about
                             70 · 2^-24 (D products, scaling), the base-2
                             exponential (2^-22), up to 16384 fp32 additions
  n · 2^-25 · max|v|         probabilities below fp16's normal range: each is
                             off by at most 2^-25 while the row's sum is >= 1
"""
import math

import numpy as np
import pytest
import torch

from servoflow_b200 import _capi
from servoflow_b200.backend import B200Backend
from servoflow_b200.quant4 import KV4Cache, unpack_codes

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def be(gpu):
    b = B200Backend(0)
    b.device_error(reset=True)
    yield b
    assert b.device_error(reset=True) == 0


def quantize64(x):
    """(codes, scales) of float values [..., D] by the format's definition, on the CPU."""
    g = x.float().numpy().reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(g).max(-1)
    s = torch.from_numpy((amax / np.float32(7)).astype(np.float32)).bfloat16().half()
    f = s.float().numpy()[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(f > 0, np.clip(np.rint(g / f), -7, 7), 0.0)
    return torch.from_numpy(c.reshape(x.shape).astype(np.int8)), s


def fill(cache, seed, spread=1.0):
    """Random values in every slot, appended by the kernel's own format (built on the CPU)."""
    from servoflow_b200.quant4 import pack_codes
    B, H, C, D = cache.shape
    g = torch.Generator().manual_seed(seed)
    for codes, scale in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        c, s = quantize64(torch.randn(B, H, C, D, generator=g) * spread)
        codes.copy_(pack_codes(c.to(torch.int32)))
        scale.copy_(s)


# ── append and read ──────────────────────────────────────────────────────────
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,S,D,cap,start,layout", [
    (1, 1, 1, 64, 32, [0], "bhsd"), (2, 3, 5, 64, 64, [0, 59], "bshd"), (3, 2, 33, 128, 96, [1, 63, 30], "bshd"),
    (1, 4, 67, 64, 67, [0], "bhsd"), (4, 1, 2, 128, 32, [3, 30, 0, 17], "bhsd")])
def test_append_is_exact(be, gpu, dt, B, H, S, D, cap, start, layout):
    cache = KV4Cache.allocate(B, H, cap, D)
    fill(cache, 5)
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]
    g = torch.Generator().manual_seed(S * D + H)
    kv = [torch.randn(B, H, S, D, generator=g) * (3.0 if i else 0.4) for i in range(2)]
    kv[0][0, 0, 0, :32] = 0.0                                  # a group of zeros
    kv[1][-1, -1, -1, 32:64] *= 1e-5                           # a tiny one (below fp16's normal scales in fp32)
    kv = [x.to(dt) for x in kv]
    dev = [x.to(gpu) if layout == "bhsd" else x.transpose(1, 2).contiguous().to(gpu) for x in kv]
    be.kv4_append(cache, *dev, start=torch.tensor(start, dtype=torch.int32, device=gpu), layout=layout)
    for x, codes, scale, c0, s0 in ((kv[0], cache.k_codes, cache.k_scale, before[0], before[2]),
                                    (kv[1], cache.v_codes, cache.v_scale, before[1], before[3])):
        c, s = quantize64(x)
        for b, at in enumerate(start):
            c0[b, :, at:at + S] = 0
            assert torch.equal(unpack_codes(codes[b, :, at:at + S]).cpu(), c[b])
            assert torch.equal(scale[b, :, at:at + S].cpu(), s[b])
            # every other slot is as it was
            mask = torch.ones(codes.shape[2], dtype=torch.bool)
            mask[at:at + S] = False
            assert torch.equal(codes[b][:, mask], c0[b][:, mask]) and torch.equal(scale[b][:, mask], s0[b][:, mask])


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,slot0,n,layout", [(64, 0, 64, "bhsd"), (128, 7, 23, "bshd"), (64, 63, 1, "bhsd")])
def test_read_returns_the_values_held(be, gpu, dt, D, slot0, n, layout):
    cache = KV4Cache.allocate(2, 3, 64, D)
    fill(cache, 9)
    shape = (2, 3, n, D) if layout == "bhsd" else (2, n, 3, D)
    out = [torch.empty(shape, dtype=dt, device=gpu) for _ in range(2)]
    be.kv4_read(cache, *out, slot0=slot0, layout=layout)
    for o, want in zip(out, cache.dequantize()):
        want = want[:, :, slot0:slot0 + n]
        assert torch.equal(o if layout == "bhsd" else o.transpose(1, 2), want.to(dt))
        if dt == torch.float16:                                # c·s is exact in fp16
            assert torch.equal(want.half().float(), want)
    one = torch.empty(shape, dtype=dt, device=gpu)
    be.kv4_read(cache, None, one, slot0=slot0, layout=layout)  # V alone
    assert torch.equal(one, out[1])


def test_append_lens_and_scalar_start(be, gpu):
    cache = KV4Cache.allocate(3, 2, 32, 64)
    fill(cache, 3)
    k0 = cache.k_codes.clone()
    x = torch.randn(3, 2, 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    be.kv4_append(cache, x.to(gpu), x.to(gpu), start=20, lens=torch.tensor([0, 8, 3], dtype=torch.int32, device=gpu))
    c, _ = quantize64(x)
    assert torch.equal(cache.k_codes[0], k0[0])                                    # length 0: untouched
    assert torch.equal(unpack_codes(cache.k_codes[1, :, 20:28]).cpu(), c[1])
    assert torch.equal(unpack_codes(cache.k_codes[2, :, 20:23]).cpu(), c[2, :, :3])
    assert torch.equal(cache.k_codes[2, :, 23:], k0[2, :, 23:])                    # rows behind the length


def test_append_outside_the_cache_is_refused_on_the_device(be, gpu):
    cache = KV4Cache.allocate(2, 1, 32, 64)
    fill(cache, 4)
    k0 = cache.k_codes.clone()
    x = torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(2)).half()
    assert be.device_error(reset=True) == 0
    be.kv4_append(cache, x.to(gpu), x.to(gpu), start=torch.tensor([30, -2], dtype=torch.int32, device=gpu))
    torch.cuda.synchronize()
    assert be.device_error(reset=True) == _capi.SFB_ERR_RANGE
    c, _ = quantize64(x)
    assert torch.equal(unpack_codes(cache.k_codes[0, :, 30:]).cpu(), c[0, :, :2])   # the two that fit
    assert torch.equal(unpack_codes(cache.k_codes[1, :, :2]).cpu(), c[1, :, 2:])
    assert torch.equal(cache.k_codes[0, :, :30], k0[0, :, :30]) and torch.equal(cache.k_codes[1, :, 2:], k0[1, :, 2:])


def test_values_that_do_not_fit_make_their_group_nan(be, gpu):
    x = torch.ones(1, 1, 6, 64)
    x[0, 0, 1, 3] = float("nan")
    x[0, 0, 2, 40] = float("inf")
    x[0, 0, 3, 0] = -float("inf")
    x[0, 0, 4, 33] = 65408.0                                   # the largest that fits: scale 9344
    x[0, 0, 5, 33] = 70000.0
    cache = KV4Cache.allocate(1, 1, 32, 64)
    be.kv4_append(cache, x.to(gpu), x.to(gpu))
    out = torch.empty(1, 1, 6, 64, device=gpu)
    be.kv4_read(cache, out)
    nan = torch.isnan(out[0, 0].cpu())
    want = torch.zeros(6, 64, dtype=torch.bool)
    want[1, :32] = want[2, 32:] = want[3, :32] = want[5, 32:] = True
    assert torch.equal(nan, want)
    assert out[0, 0, 4, 33].item() == 65408.0


# ── attention ────────────────────────────────────────────────────────────────
def attn64(q, cache, lens, Sk, causal, mask, scale):
    """Definition in fp64: ([B, H, Sq, D] output, Σ p|v|)."""
    k, v = (x.double()[:, :, :Sk] for x in cache.dequantize())
    B, H, Sq, D = q.shape
    g = H // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    j = torch.arange(Sk, device=q.device)
    n = torch.full((B,), Sk, device=q.device) if lens is None else lens.long().clamp(0, Sk)
    see = (j[None, :] < n[:, None])[:, None, :].expand(B, Sq, Sk)
    if causal:
        i = torch.arange(Sq, device=q.device)
        see = see & (j[None, None] <= (n[:, None] - Sq + i[None])[:, :, None])
    if mask is not None:
        see = see & mask[:, None, :].bool()
    see = see[:, None]
    k, v = (torch.nan_to_num(x) if torch.isnan(x).any() else x for x in (k, v))     # masked slots may hold NaN
    s = torch.einsum("bhid,bhjd->bhij", q.double(), k) * scale
    s = s.masked_fill(~see, -1e300)
    p = torch.softmax(s, -1) * see
    return torch.einsum("bhij,bhjd->bhid", p, v), torch.einsum("bhij,bhjd->bhid", p, v.abs()), v.abs().amax()


def run_attn(be, gpu, B, H, Hkv, Sq, Sk, D, dt, causal=False, lens=None, mask_p=None, layout="bhsd", scale=0.0,
             splits=0, seed=0, cap=None, mask=None):
    cache = KV4Cache.allocate(B, Hkv, max(cap or Sk, 1), D)
    fill(cache, seed + 11)
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, H, Sq, D, generator=g).to(dt).to(gpu)
    lt = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu)
    if mask_p is not None:
        mask = (torch.rand(B, Sk, generator=g) < mask_p).to(gpu)
    qq = q if layout == "bhsd" else q.transpose(1, 2).contiguous()
    out = torch.full_like(qq, float("nan"))
    be.kv4_attention(qq, cache, out, seq_k=Sk, kv_len=lt, mask=mask, scale=scale, is_causal=causal,
                     num_splits=splits, layout=layout)
    got = (out if layout == "bhsd" else out.transpose(1, 2)).double()
    ref, mag, vmax = attn64(q, cache, lt, Sk, causal, mask, scale or 1 / math.sqrt(D))
    tol = HALF[dt] * ref.abs() + (2.0 ** -11 + 2.0 ** -15) * mag + Sk * 2.0 ** -25 * vmax
    err = (got - ref).abs()
    assert not torch.isnan(got).any()
    assert (err <= tol).all(), f"max excess {(err - tol).max().item():.3e}, max err {err.max().item():.3e}"
    return q, cache, out


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sk", [1, 15, 16, 17, 100, 515, 4374])
def test_single_token(be, gpu, dt, D, Sk):
    run_attn(be, gpu, 2, 4, 4, 1, Sk, D, dt, seed=Sk)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv,Sq", [(8, 1, 1), (9, 1, 1), (16, 2, 2), (4, 4, 7), (4, 4, 16), (2, 1, 16), (3, 1, 11),
                                      (2, 2, 67), (2, 2, 72), (2, 2, 73), (6, 2, 50), (1, 1, 300)])
def test_rows_per_head(be, gpu, D, H, Hkv, Sq):
    run_attn(be, gpu, 2, H, Hkv, Sq, 333, D, torch.bfloat16, seed=H * Sq)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk,lens", [(1, 200, [200, 1, 77]), (5, 200, [5, 200, 33]), (67, 130, [67, 130, 128]),
                                        (9, 64, [3, 0, 8]), (40, 16, [16, 1, 0]), (150, 1000, [1000, 150, 149])])
def test_causal_and_lengths(be, gpu, D, Sq, Sk, lens):
    q, _, out = run_attn(be, gpu, 3, 4, 2, Sq, Sk, D, torch.float16, causal=True, lens=lens, layout="bshd", seed=Sq)
    for b, n in enumerate(lens):                       # queries before the first slot see nothing: zeros
        assert (out[b, :max(0, Sq - n)] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,H,Hkv", [(1, 2, 2), (67, 2, 2), (33, 4, 2), (130, 2, 1)])
def test_key_masks(be, gpu, D, Sq, H, Hkv):
    run_attn(be, gpu, 2, H, Hkv, Sq, 261, D, torch.bfloat16, mask_p=0.5, seed=Sq)
    run_attn(be, gpu, 2, H, Hkv, Sq, 261, D, torch.bfloat16, mask_p=0.02, causal=True, lens=[261, 140], seed=Sq + 1)
    m = torch.zeros(2, 261, dtype=torch.uint8, device=gpu)
    m[1, 200] = 3                                      # any nonzero byte keeps its key
    _, _, out = run_attn(be, gpu, 2, H, Hkv, Sq, 261, D, torch.bfloat16, mask=m, seed=Sq + 2)
    assert (out[0] == 0).all()                         # a session whose mask leaves nothing


@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8, 16])
@pytest.mark.parametrize("Sq", [1, 20, 67])
def test_splits(be, gpu, splits, Sq):
    run_attn(be, gpu, 1, 2, 2, Sq, 700, 64, torch.bfloat16, splits=splits, seed=splits)
    run_attn(be, gpu, 2, 2, 1, Sq, 40, 128, torch.float16, splits=splits, lens=[40, 17], seed=splits)


def test_empty_cases(be, gpu):
    for Sk, lens in ((0, None), (33, [0, 0])):
        cache = KV4Cache.allocate(2, 2, 64, 64)
        q = torch.randn(2, 2, 3, 64, device=gpu).half()
        out = torch.full_like(q, float("nan"))
        lt = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu)
        be.kv4_attention(q, cache, out, seq_k=Sk, kv_len=lt)
        assert (out == 0).all()
    q = torch.empty(2, 2, 0, 64, dtype=torch.half, device=gpu)
    be.kv4_attention(q, cache, torch.empty_like(q))


@pytest.mark.parametrize("Sq", [1, 67])
@pytest.mark.parametrize("D", [64, 128])
def test_masked_slots_may_hold_nan(be, gpu, Sq, D):
    B, H, Sk = 2, 2, 150
    cache = KV4Cache.allocate(B, H, Sk, D)
    fill(cache, 21)
    mask = torch.ones(B, Sk, dtype=torch.bool, device=gpu)
    mask[0, 40] = mask[1, 0] = mask[1, 99] = False
    lens = torch.tensor([100, 100], dtype=torch.int32, device=gpu)
    clean_k, clean_v = cache.k_scale.clone(), cache.v_scale.clone()
    for s in (cache.k_scale, cache.v_scale):
        s[0, :, 40] = float("nan"); s[1, :, 0] = float("inf"); s[1, :, 99] = float("nan"); s[:, :, 100:] = float("nan")
    q = torch.randn(B, H, Sq, D, generator=torch.Generator().manual_seed(5)).bfloat16().to(gpu)
    out, want = torch.empty_like(q), torch.empty_like(q)
    be.kv4_attention(q, cache, out, kv_len=lens, mask=torch.nn.functional.pad(mask, (0, cache.shape[2] - Sk)))
    clean = KV4Cache(cache.k_codes, cache.v_codes, clean_k, clean_v)
    be.kv4_attention(q, clean, want, kv_len=lens, mask=torch.nn.functional.pad(mask, (0, cache.shape[2] - Sk)))
    assert torch.equal(out, want) and not torch.isnan(out).any()


def test_visible_nan_reaches_only_its_rows(be, gpu):
    cache = KV4Cache.allocate(2, 1, 64, 64)
    fill(cache, 22)
    cache.k_scale[0, 0, 5] = float("nan")
    q = torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(6)).bfloat16().to(gpu)
    out = torch.empty_like(q)
    be.kv4_attention(q, cache, out, is_causal=True, seq_k=7)
    assert not torch.isnan(out[0, 0, :1]).any()        # query 0 sees slots 0..3, query 1 0..4
    assert not torch.isnan(out[0, 0, 1]).any()
    assert torch.isnan(out[0, 0, 2:]).all()            # slot 5 visible
    assert not torch.isnan(out[1]).any()
    cache.k_scale[0, 0] = float("nan")                 # every visible logit NaN
    be.kv4_attention(q, cache, out)
    assert torch.isnan(out[0]).all() and not torch.isnan(out[1]).any()


def test_large_logits_and_scale(be, gpu):
    # logits in the hundreds: the running reference moves far, one key dominates
    cache = KV4Cache.allocate(1, 1, 640, 64)
    fill(cache, 23, spread=6.0)
    q = (torch.randn(1, 1, 9, 64, generator=torch.Generator().manual_seed(7)) * 5).half().to(gpu)
    out = torch.empty_like(q)
    be.kv4_attention(q, cache, out, scale=0.5)
    ref, mag, vmax = attn64(q, cache, None, 640, False, None, 0.5)
    # logits to about 2^10 of products whose magnitudes sum to 2^12: fp32 sums of 64
    # terms leave them within 64 · 2^-24 · 2^12 = 2^-6 at worst
    assert ((out.double() - ref).abs() <= 2.0 ** -5 * mag + 640 * 2.0 ** -25 * vmax).all()


def test_out_of_range_queries_are_recorded(be, gpu):
    cache = KV4Cache.allocate(1, 1, 32, 64)
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device=gpu)
    q[..., 3] = 1e6
    assert be.device_error(reset=True) == 0
    be.kv4_attention(q, cache, torch.empty_like(q))
    torch.cuda.synchronize()
    assert be.device_error(reset=True) == _capi.SFB_ERR_RANGE


def test_strided_caches_and_views(be, gpu):
    # a cache whose batch and head strides have gaps, and Q / out inside wider buffers
    B, H, C, D, Sq = 2, 2, 96, 64, 3
    big = KV4Cache.allocate(B, 2 * H, C, D)
    fill(big, 31)
    view = KV4Cache(*(t[:, ::2] for t in (big.k_codes, big.v_codes, big.k_scale, big.v_scale)))
    tight = KV4Cache(*(t[:, ::2].contiguous() for t in (big.k_codes, big.v_codes, big.k_scale, big.v_scale)))
    wide = torch.randn(B, Sq, 3 * H, D, generator=torch.Generator().manual_seed(8)).bfloat16().to(gpu)
    q = wide[:, :, H:2 * H]
    obuf = torch.zeros(B, Sq, 4 * H, D, dtype=torch.bfloat16, device=gpu)
    want = torch.empty(B, Sq, H, D, dtype=torch.bfloat16, device=gpu)
    be.kv4_attention(q, view, obuf[:, :, H:2 * H], layout="bshd", seq_k=77)
    be.kv4_attention(q.contiguous(), tight, want, layout="bshd", seq_k=77)
    assert torch.equal(obuf[:, :, H:2 * H], want)
    assert (obuf[:, :, :H] == 0).all() and (obuf[:, :, 2 * H:] == 0).all()


def test_same_call_twice_and_graph_replay_give_the_same_bits(be, gpu):
    cache = KV4Cache.allocate(2, 4, 2048, 64)
    fill(cache, 41)
    q = torch.randn(2, 4, 67, 64, generator=torch.Generator().manual_seed(9)).bfloat16().to(gpu)
    a, b = torch.empty_like(q), torch.empty_like(q)
    be.kv4_attention(q, cache, a)
    be.kv4_attention(q, cache, b)
    assert torch.equal(a, b)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    c, d = torch.zeros_like(q), torch.zeros_like(q)
    with torch.cuda.graph(g1):
        be.kv4_attention(q, cache, c)
    with torch.cuda.graph(g2):
        be.kv4_attention(q, cache, d)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        g1.replay()
    with torch.cuda.stream(s2):                        # two graphs at once share nothing
        g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, c) and torch.equal(a, d)


def test_offsets_past_32_bits(be, gpu):
    # one head's codes start beyond 4 GB of the buffer: a strided view of a 4.4 GB allocation
    D, cap, gap = 64, 64, 4_400_000_000
    buf = torch.zeros(gap + 2 * cap * D, dtype=torch.uint8, device=gpu)
    code = buf.as_strided((2, 1, cap, D // 2), (gap, cap * D // 2, D // 2, 1))
    src = KV4Cache.allocate(2, 1, cap, D)
    fill(src, 51)
    code.copy_(src.k_codes)
    vcode = buf[cap * D:].as_strided((2, 1, cap, D // 2), (gap, cap * D // 2, D // 2, 1))
    vcode.copy_(src.v_codes)
    far = KV4Cache(code, vcode, src.k_scale, src.v_scale)
    q = torch.randn(2, 2, 1, D, generator=torch.Generator().manual_seed(10)).bfloat16().to(gpu)
    a, b = torch.empty_like(q), torch.empty_like(q)
    be.kv4_attention(q, far, a)
    be.kv4_attention(q, src, b)
    assert torch.equal(a, b)


def test_wrapper_refusals(be, gpu):
    cache = KV4Cache.allocate(2, 2, 64, 64)
    q = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16, device=gpu)
    out = torch.empty_like(q)
    E = _capi.SfbError
    with pytest.raises(E):
        be.kv4_attention(q.float(), cache, out.float())
    with pytest.raises(E):
        be.kv4_attention(q, cache, out.half())
    with pytest.raises(E):
        be.kv4_attention(q[:1], cache, out[:1])
    with pytest.raises(E):
        be.kv4_attention(q[:, :3], cache, out[:, :3])                  # heads not a multiple
    with pytest.raises(E):
        be.kv4_attention(q, cache, out, seq_k=65)
    with pytest.raises(E):
        be.kv4_attention(q, cache, out, kv_len=torch.zeros(2, dtype=torch.int64, device=gpu))
    with pytest.raises(E):
        be.kv4_attention(q, cache, out, mask=torch.ones(2, 63, dtype=torch.bool, device=gpu))
    with pytest.raises(ValueError):
        be.kv4_attention(q.cpu(), cache, out)
    with pytest.raises(ValueError):
        be.kv4_attention(q, cache, out, layout="sbhd")
    with pytest.raises(E):
        be.kv4_append(cache, q[:, :2], q[:, :2], start=62)             # past the last slot
    with pytest.raises(E):
        be.kv4_append(cache, q, q)
    with pytest.raises(E):
        be.kv4_read(cache)
    bad = KV4Cache(cache.k_codes, cache.v_codes, cache.k_scale.float(), cache.v_scale)
    with pytest.raises(E):
        be.kv4_attention(q, bad, out)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk", [(9, 40), (20, 33), (67, 300), (130, 260)])
def test_nan_slots_do_not_reach_rows_before_them(be, gpu, D, Sq, Sk):
    """Causal calls: a slot whose V (or K) is NaN is in the same tile as rows that do
    not see it. Those keep their values, the rows that see it are NaN."""
    be.device_error(reset=True)
    bad = Sk - Sq // 3                                      # seen by the last rows alone
    q = torch.randn(1, 2, Sq, D, generator=torch.Generator().manual_seed(31)).to(torch.float16).to(gpu)
    sees = torch.arange(Sq, device=gpu) + Sk - Sq >= bad
    for field in ("v_scale", "k_scale"):
        cache = KV4Cache.allocate(1, 2, (Sk + 3) // 4 * 4, D)
        fill(cache, 32)
        clean, out = torch.empty_like(q), torch.empty_like(q)
        be.kv4_attention(q, cache, clean, seq_k=Sk, is_causal=True)
        getattr(cache, field)[:, :, bad, 1] = float("nan")
        be.kv4_attention(q, cache, out, seq_k=Sk, is_causal=True)
        torch.cuda.synchronize()
        assert torch.equal(out[:, :, ~sees], clean[:, :, ~sees])
        assert out[:, :, sees].isnan().any(-1).all()
    assert be.device_error() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sk", [100, 256, 300, 512])
@pytest.mark.parametrize("Sq", [16, 40, 75, 90])
def test_few_key_tiles_a_cta(be, gpu, D, Sk, Sq):
    """One to four tiles of 128 slots in a CTA (no splits), where the last products are
    the only ones in flight when the softmax is done with its last tile; 100 CTAs of every
    row form (16, 48, 80 and, with 64 channels, 96 rows on 148 SMs), the same bits every time."""
    q, cache, out = run_attn(be, gpu, 4, 25, 25, Sq, Sk, D, torch.bfloat16, splits=1, seed=Sq + Sk)
    again = torch.empty_like(out)
    for _ in range(20):
        be.kv4_attention(q, cache, again.fill_(0), seq_k=Sk, num_splits=1)
        assert torch.equal(out, again)


@pytest.mark.parametrize("B,Hkv,Sq", [(65600, 1, 1), (65600, 1, 17), (1, 65600, 1), (1, 33000, 97)])
def test_more_heads_sessions_and_row_tiles_than_65535(be, gpu, B, Hkv, Sq):
    D, n = 64, 20
    cache = KV4Cache.allocate(B, Hkv, n, D, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(Sq)
    for codes, scale in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device=gpu, dtype=torch.uint8))
        scale.copy_((torch.rand(scale.shape, generator=g, device=gpu) * 0.2).bfloat16().half())
    q = torch.randn(B, Hkv, Sq, D, generator=g, device=gpu, dtype=torch.float32).half()
    out = torch.full_like(q, float("nan"))
    be.kv4_attention(q, cache, out, seq_k=n)
    # heads and sessions from all over the grid, the last among them
    b = torch.tensor([0, B // 2, B - 1], device=gpu)
    h = torch.tensor([0, 1, Hkv // 2, Hkv - 2, Hkv - 1], device=gpu).clamp(0, Hkv - 1)
    pick = lambda t: t[b][:, h]
    part = KV4Cache(*(pick(t).contiguous() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)))
    ref, mag, vmax = attn64(pick(q), part, None, n, False, None, 1 / math.sqrt(D))
    tol = 2.0 ** -11 * ref.abs() + (2.0 ** -11 + 2.0 ** -15) * mag + n * 2.0 ** -25 * vmax
    assert ((pick(out).double() - ref).abs() <= tol).all()
    assert not out.isnan().any()


def test_more_row_tiles_of_one_head_than_65535(be, gpu):
    # 400 thousand tokens of 16 heads that share one: 66667 tiles of 96 rows
    D, n, H, Sq = 64, 20, 16, 400_000
    cache = KV4Cache.allocate(1, 1, n, D, device=gpu)
    fill(cache, 61)
    q = torch.randn(1, H, Sq, D, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu).half()
    out = torch.full_like(q, float("nan"))
    be.kv4_attention(q, cache, out, seq_k=n)
    assert not out.isnan().any()
    i = torch.tensor([0, 1, Sq // 3, Sq - 7000, Sq - 6500, Sq - 6000, Sq - 1], device=gpu)
    ref, mag, vmax = attn64(q[:, :, i], cache, None, n, False, None, 1 / math.sqrt(D))
    tol = 2.0 ** -11 * ref.abs() + (2.0 ** -11 + 2.0 ** -15) * mag + n * 2.0 ** -25 * vmax
    assert ((out[:, :, i].double() - ref).abs() <= tol).all()


def test_slots_past_32_bits_are_refused(be, gpu):
    """Slots and lengths that the C call's 32-bit arguments would cut short."""
    cache = KV4Cache.allocate(1, 1, 32, 64)
    fill(cache, 3)
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]
    x = torch.ones(1, 1, 1, 64, dtype=torch.float16, device=gpu)
    for start in (2 ** 32, 2 ** 32 + 5, -2 ** 32, 2 ** 31):
        with pytest.raises(_capi.SfbError):
            be.kv4_append(cache, x, x, start=start)
        with pytest.raises(_capi.SfbError):
            be.kv4_read(cache, x, slot0=start)
    long = x.expand(1, 1, 2 ** 32 + 1, 64)             # not one token
    with pytest.raises(_capi.SfbError):
        be.kv4_append(cache, long, long)
    with pytest.raises(_capi.SfbError):
        be.kv4_read(cache, long)
    for sk in (2 ** 32 + 32, 2 ** 31, -1):
        with pytest.raises(_capi.SfbError):
            be.kv4_attention(x, cache, x, seq_k=sk)
    for got, want in zip((cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale), before):
        assert torch.equal(got, want)


def constant_cache(B, Hkv, cap, D, gpu, k_code, v_code):
    """A cache of scale-1 groups: integer codes [cap, D] of K and V in every head and session."""
    from servoflow_b200.quant4 import pack_codes
    cache = KV4Cache.allocate(B, Hkv, cap, D, device=gpu)
    for codes, scale, c in ((cache.k_codes, cache.k_scale, k_code), (cache.v_codes, cache.v_scale, v_code)):
        codes.copy_(pack_codes(c.to(torch.int32).to(gpu)).expand_as(codes))
        scale.fill_(1.0)
    return cache


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 12, 40])
@pytest.mark.parametrize("gap", [14.0, 17.5])
@pytest.mark.parametrize("splits", [1, 0])
def test_small_probabilities_beside_a_dominant_slot(be, gpu, D, Sq, gap, splits):
    """One slot takes nearly all of a row and has V = 0, 16383 others share what is left
    (each e^-gap of it, 2^-20 and 2^-25) and carry the whole result. P is rounded to fp16
    after a factor of at least 2^7, so one is off by 2^-12 of itself (half a step) or by
    2^-25 · 2^-7 where that is fp16's subnormal range."""
    n = 16384
    k, v = torch.zeros(n, D), torch.ones(n, D)
    k[0, 0], v[0] = 7, 0
    v[1::3] = 3
    cache = constant_cache(1, 2, n, D, gpu, k, v)
    q = torch.zeros(1, 2, Sq, D, dtype=torch.float16, device=gpu)
    q[..., 0] = gap / 7
    out = torch.empty_like(q)
    be.kv4_attention(q, cache, out, scale=1.0, num_splits=splits)
    ref, mag, vmax = attn64(q, cache, None, n, False, None, 1.0)
    tol = 2.0 ** -11 * ref.abs() + (2.0 ** -11 + 2.0 ** -15) * mag + n * 2.0 ** -32 * vmax + 2.0 ** -25
    err = (out.double() - ref).abs()
    assert (err <= tol).all(), f"max err {err.max().item():.3e}, tol {tol.max().item():.3e}, ref {ref.abs().max().item():.3e}"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [2, 20])
@pytest.mark.parametrize("inf", [float("inf"), -float("inf")])
def test_infinite_queries_make_their_rows_nan(be, gpu, dt, D, Sq, inf):
    """Every logit of such a row is an infinity or NaN, so its softmax is NaN; also where
    each is minus infinity. A row that sees no slot stays zero."""
    n = 40
    cache = constant_cache(2, 1, 64, D, gpu, torch.full((64, D), 3.0), torch.ones(64, D))
    q = torch.ones(2, 1, Sq, D, dtype=dt, device=gpu)
    q[:, :, 1, 5] = inf
    out = torch.empty_like(q)
    be.device_error(reset=True)
    be.kv4_attention(q, cache, out, seq_k=n, kv_len=torch.tensor([n, 0], dtype=torch.int32, device=gpu))
    assert out[0, 0, 1].isnan().all() and (out[1] == 0).all()
    out[0, 0, 1] = 1
    assert (out[0] == 1).all()
    assert be.device_error() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hkv,Sq", [(25, 25, 75), (25, 25, 80), (25, 25, 81), (25, 25, 96), (100, 25, 24)])
def test_every_row_form_with_masks(be, gpu, D, dt, H, Hkv, Sq):
    """Calls of 100 units, which take 80 columns up to 80 rows and, with 64 channels, 96
    above (128 channels: twice 48); lengths, causal order and dropped keys in each."""
    run_attn(be, gpu, 4, H, Hkv, Sq, 261, D, dt, causal=True, lens=[261, 100, Sq + 3, 7], seed=Sq)
    run_attn(be, gpu, 4, H, Hkv, Sq, 261, D, dt, mask_p=0.4, lens=[261, 0, 128, 129], layout="bshd", seed=Sq + 1)
    run_attn(be, gpu, 4, H, Hkv, Sq, 530, D, dt, scale=-0.2, splits=3, seed=Sq + 2)


def test_scales_and_codes_at_ties(be, gpu):
    """Exact ties of fp32 input go to even, and their neighbours of one unit in the last
    place to the right side: of the scale (max|x| = 7 · t with t halfway between two
    bf16 values) and of the codes (x / s as fp32 division gives it, next to k + 1/2)."""
    n = 4096
    g = torch.Generator().manual_seed(71)
    x = torch.zeros(n, 32)
    t = (torch.randint(128, 256, (n,), generator=g) * 2 + 1).float()            # 9 bits, the last one set
    e = 2.0 ** torch.randint(-20, 3, (n,), generator=g).float()
    top = 7 * t * e
    step = torch.randint(-1, 2, (n,), generator=g)
    top = torch.where(step < 0, torch.nextafter(top, torch.zeros_like(top)),
                      torch.where(step > 0, torch.nextafter(top, torch.full_like(top, 1e30)), top))
    x[: n // 2, 0] = top[: n // 2]
    # the other half: scales of 8 bits, values next to every half step
    s = torch.randint(128, 256, (n,), generator=g).float() * 2.0 ** torch.randint(-30, 5, (n,), generator=g).float()
    x[n // 2:, 0] = 7 * s[n // 2:]
    half = torch.arange(-6.5, 7, 1.0)                                           # 14 halves, exact times s
    v = half[None] * s[n // 2:, None]
    x[n // 2:, 1:15] = v
    x[n // 2:, 15:29] = torch.nextafter(v, torch.full_like(v, 1e30))
    x[n // 2:, 29:32] = torch.nextafter(v[:, 5:8], torch.full_like(v[:, 5:8], -1e30))
    x = x.view(1, 1, n // 2, 64)
    cache = KV4Cache.allocate(1, 1, n // 2, 64)
    be.kv4_append(cache, x.to(gpu), (-x).to(gpu))
    for val, codes, scale in ((x, cache.k_codes, cache.k_scale), (-x, cache.v_codes, cache.v_scale)):
        c, sc = quantize64(val)
        assert torch.equal(scale.cpu(), sc) and torch.equal(unpack_codes(codes).cpu(), c)
