"""GPU test of the 4-bit operators together, as a decoder layer uses them: a
4-bit projection to Q, K and V, their norms and rotation, the append to the
cache, the attention over it and a 4-bit output projection; token by token
against the whole prompt at once, and a decoding step replayed from a graph."""
import math

import pytest
import torch

from servoflow_b200.backend import B200Backend
from servoflow_b200.quant4 import KV4Cache, pack_w4

pytestmark = pytest.mark.gpu

B, H, HKV, D, HID, CAP = 2, 4, 2, 64, 256, 96


class Layer:
    def __init__(self, dev, dt):
        g = torch.Generator().manual_seed(11)
        self.be, self.dt, self.dev = B200Backend(0), dt, dev
        mk = lambda n, k: tuple(t.to(dev) for t in pack_w4(torch.randn(n, k, generator=g) / math.sqrt(k), 64))
        self.qkv, self.proj = mk((H + 2 * HKV) * D, HID), mk(HID, H * D)
        self.wq, self.wk = ((1 + 0.1 * torch.randn(D, generator=g)).to(dt).to(dev) for _ in range(2))
        f = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        a = torch.arange(CAP, dtype=torch.float64)[:, None] * f
        self.cos, self.sin = a.cos().float().to(dev), a.sin().float().to(dev)

    def step(self, x, cache, pos, lens, out, buf):
        """x [B, S, HID] at positions pos [B, S]; lens: slots used after this step."""
        S = x.shape[1]
        flat, o = buf
        self.be.w4a16_linear(x.reshape(B * S, HID), *self.qkv, flat)
        v4 = flat.view(B, S, H + 2 * HKV, D)
        q, k, v = v4[:, :, :H], v4[:, :, H:H + HKV], v4[:, :, H + HKV:]
        self.be.qk_norm_rope(q, k, q, k, self.wq, self.wk, self.cos, self.sin, positions=pos, layout="bshd")
        self.be.kv4_append(cache, k, v, start=pos[:, 0].contiguous(), layout="bshd")
        self.be.kv4_attention(q, cache, o, kv_len=lens, is_causal=True, layout="bshd")
        self.be.w4a16_linear(o.view(B * S, H * D), *self.proj, out.view(B * S, HID), residual=x.reshape(B * S, HID))
        return q.clone(), o


def bufs(dt, dev, S):
    """The projection's output and the attention's, kept by the caller."""
    return torch.empty(B * S, (H + 2 * HKV) * D, dtype=dt, device=dev), torch.empty(B, S, H, D, dtype=dt, device=dev)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_token_by_token_equals_the_whole_prompt(gpu, dt):
    L = Layer(gpu, dt)
    L.be.device_error(reset=True)
    S = 40
    x = torch.randn(B, S, HID, generator=torch.Generator().manual_seed(12)).to(dt).to(gpu)
    pos = torch.arange(S, dtype=torch.int32, device=gpu).expand(B, S).contiguous()
    whole, parts = KV4Cache.allocate(B, HKV, CAP, D), KV4Cache.allocate(B, HKV, CAP, D)
    ya, yb = torch.empty_like(x), torch.empty_like(x)
    full = torch.full((B,), S, dtype=torch.int32, device=gpu)
    qa, oa = L.step(x, whole, pos, full, ya, bufs(dt, gpu, S))
    # 33 tokens, then one by one
    cuts = [(0, 33)] + [(i, i + 1) for i in range(33, S)]
    ob = []
    for a, b in cuts:
        y = torch.empty(B, b - a, HID, dtype=dt, device=gpu)
        q, o = L.step(x[:, a:b].contiguous(), parts, pos[:, a:b].contiguous(), torch.full_like(full, b), y, bufs(dt, gpu, b - a))
        ob.append(o)
        yb[:, a:b] = y
    ob = torch.cat(ob, 1)
    # The projection's sums depend on the kernel for the row count in fp32's last
    # places; where that moves a value across a rounding of 16 bits the code behind
    # it may move by one: a few of the codes differ, by one step.
    for c in ("k_codes", "v_codes"):
        d = (getattr(whole, c)[:, :, :S] != getattr(parts, c)[:, :, :S]).float().mean().item()
        assert d < 0.01, (c, d)
    # attention on its own cache against 64 bits: the tolerance of test_kv4_gpu
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dt]
    k, v = (t.double()[:, :, :S].repeat_interleave(H // HKV, 1) for t in whole.dequantize())
    s = torch.einsum("bihd,bhjd->bhij", qa.double(), k) / math.sqrt(D)
    s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device=gpu).triu(1), -1e300)
    p = torch.softmax(s, -1)
    ref, mag = torch.einsum("bhij,bhjd->bihd", p, v), torch.einsum("bhij,bhjd->bihd", p, v.abs())
    assert ((oa.double() - ref).abs() <= half * ref.abs() + (2.0 ** -11 + 2.0 ** -15) * mag + S * 2.0 ** -25 * v.abs().amax()).all()
    # under 1 % of the codes off by one step (1/7 of a group's maximum): the outputs
    # of the two ways agree far inside the cache's own resolution
    for a, b in ((oa, ob), (ya, yb)):
        assert (a.float() - b.float()).norm() <= 0.02 * a.float().norm()
    assert L.be.device_error(reset=True) == 0


def test_decoding_step_from_a_graph(gpu):
    dt = torch.bfloat16
    L = Layer(gpu, dt)
    prompt = torch.randn(B, 20, HID, generator=torch.Generator().manual_seed(13)).to(dt).to(gpu)
    toks = torch.randn(5, B, 1, HID, generator=torch.Generator().manual_seed(14)).to(dt).to(gpu)
    pos0 = torch.arange(20, dtype=torch.int32, device=gpu).expand(B, 20).contiguous()

    def start():
        cache = KV4Cache.allocate(B, HKV, CAP, D)
        L.step(prompt, cache, pos0, torch.full((B,), 20, dtype=torch.int32, device=gpu), torch.empty_like(prompt),
               bufs(dt, gpu, 20))
        return cache

    eager = []
    cache = start()
    for i in range(5):
        y = torch.empty(B, 1, HID, dtype=dt, device=gpu)
        L.step(toks[i], cache, torch.full((B, 1), 20 + i, dtype=torch.int32, device=gpu),
               torch.full((B,), 21 + i, dtype=torch.int32, device=gpu), y, bufs(dt, gpu, 1))
        eager.append(y)
    cache = start()
    x, y = torch.empty(B, 1, HID, dtype=dt, device=gpu), torch.empty(B, 1, HID, dtype=dt, device=gpu)
    pos, lens, buf = torch.zeros(B, 1, dtype=torch.int32, device=gpu), torch.zeros(B, dtype=torch.int32, device=gpu), bufs(dt, gpu, 1)
    keep = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]
    graph = torch.cuda.CUDAGraph()
    pos.fill_(20); lens.fill_(21); x.copy_(toks[0])
    L.step(x, cache, pos, lens, y, buf)
    with torch.cuda.graph(graph):
        L.step(x, cache, pos, lens, y, buf)
    for t, k in zip((cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale), keep):
        t.copy_(k)
    for i in range(5):
        x.copy_(toks[i]); pos.fill_(20 + i); lens.fill_(21 + i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[i])
