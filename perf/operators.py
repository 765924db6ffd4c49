"""Measured cases of the 4-bit serving operators: query/key norms with the position
rotation, the 4-bit K/V cache (append and read back), attention over that cache, and the
linear layer with 4-bit weights and group scales.

`run` computes each operator in its plain form (elementary torch operations in fp32, rounded
once at the end) or, where `own` is true, through the framework's entry points
(servoflow_b200.backend.B200Backend). `exact` gives the same results from the definitions in
fp64. Sizes are the RDT-1B runtime's (32 heads of 64, 67 tokens a step, 4374 image tokens,
1024 language tokens, 2048 hidden) and generic ones.

4-bit format: 8 consecutive values of the contiguous dimension make one little-endian 32-bit
word; value 2i sits in bits [4i, 4i+4) and value 2i+1 in bits [16+4i, 16+4i+4); a nibble n
stands for n - 8. Cache scales: one fp16 per token, head and 32 channels, s = fp16(bf16(max|x|
/ 7)), codes clamp(round(x / s), -7, 7) (0 where s is 0).
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_GROUP = 32                     # channels per cache scale
_backend = None


def _be():
    global _backend
    if _backend is None:
        from servoflow_b200.backend import B200Backend
        _backend = B200Backend(0)
    return _backend


# ── cases ────────────────────────────────────────────────────────────────────
def listed():
    return [
        # one generated token of one session: latency of the norm + rotation between projection and attention
        {"name": "norm_rope one token", "op": "norm_rope", "B": 1, "S": 1, "H": 32, "Hkv": 32, "D": 64, "rot": 64,
         "inter": False, "pos0": 4374, "dtype": "bf16"},
        # one denoising step of 32 sessions (67 tokens each)
        {"name": "norm_rope 32x67", "op": "norm_rope", "B": 32, "S": 67, "H": 32, "Hkv": 32, "D": 64, "rot": 64,
         "inter": False, "pos0": 0, "dtype": "bf16"},
        # a long prompt with grouped K/V heads, part of each head rotated, far positions
        {"name": "norm_rope long gqa", "op": "norm_rope", "B": 2, "S": 4374, "H": 32, "Hkv": 8, "D": 128, "rot": 64,
         "inter": True, "pos0": 120000, "dtype": "fp16"},
        # one token appended to the 64-slot window of each of 32 sessions, the window read back in 16 bits
        {"name": "append one token", "op": "append", "B": 32, "S": 1, "Hkv": 32, "D": 64, "cap": 64, "dtype": "bf16"},
        # the image condition of 4 sessions written once per control tick, read back in 16 bits
        {"name": "append image", "op": "append", "B": 4, "S": 4374, "Hkv": 32, "D": 64, "cap": 4384, "dtype": "bf16"},
        # one generated token of one session over the image condition: latency
        {"name": "attn decode b1", "op": "attn", "B": 1, "H": 32, "Hkv": 32, "Sq": 1, "Sk": 4374, "D": 64,
         "causal": False, "ragged": False, "mask": False, "dtype": "bf16"},
        # 32 sessions generating over long caches of different lengths, grouped heads
        {"name": "attn decode b32 gqa", "op": "attn", "B": 32, "H": 32, "Hkv": 8, "Sq": 1, "Sk": 16384, "D": 128,
         "causal": True, "ragged": True, "mask": False, "dtype": "bf16"},
        # one session's image cross-attention (67 action tokens), one of 14 in a denoising step
        {"name": "attn image b1", "op": "attn", "B": 1, "H": 32, "Hkv": 32, "Sq": 67, "Sk": 4374, "D": 64,
         "causal": False, "ragged": False, "mask": False, "dtype": "bf16"},
        # the same for 32 sessions batched
        {"name": "attn image b32", "op": "attn", "B": 32, "H": 32, "Hkv": 32, "Sq": 67, "Sk": 4374, "D": 64,
         "causal": False, "ragged": False, "mask": False, "dtype": "bf16"},
        # a prompt chunk over a cache with dropped keys
        {"name": "attn chunk", "op": "attn", "B": 2, "H": 16, "Hkv": 4, "Sq": 515, "Sk": 2077, "D": 64,
         "causal": True, "ragged": True, "mask": True, "dtype": "fp16"},
        # a single row through a wide layer: weights read once
        {"name": "linear one row", "op": "linear", "M": 1, "N": 16384, "K": 8192, "G": 128, "act": "none",
         "bias": True, "res": False, "dtype": "bf16", "y": "fp32"},
        # one denoising step's QKV projection (67 tokens)
        {"name": "linear 67 rows", "op": "linear", "M": 67, "N": 6144, "K": 2048, "G": 64, "act": "gelu",
         "bias": True, "res": True, "dtype": "bf16", "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "attn", "attn", "attn", "linear", "linear"])
    if op == "norm_rope":
        D = rng.choice([64, 64, 96, 128, 256])
        B = _log(rng, 1, 32)
        Hkv = rng.choice([1, 2, 4, 8, 16])
        H = Hkv * rng.choice([1, 2, 4])
        S = _log(rng, 1, max(1, min(4374, 60_000_000 // (B * (H + Hkv) * D))))
        return {"op": op, "B": B, "S": S, "H": H, "Hkv": Hkv, "D": D,
                "rot": rng.choice([0, 32, D, D]), "inter": rng.random() < 0.4, "pos0": _log(rng, 1, 100000),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "append":
        D = rng.choice([64, 128])
        B = _log(rng, 1, 32)
        Hkv = rng.choice([1, 4, 8, 32])
        S = _log(rng, 1, max(1, min(4374, 30_000_000 // (B * Hkv * D))))
        return {"op": op, "B": B, "S": S, "Hkv": Hkv, "D": D, "cap": 32 * (S // 32 + 1 + rng.randrange(3)),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "attn":
        D = rng.choice([64, 64, 128])
        Hkv = rng.choice([1, 2, 4, 8, 16, 32])
        g = rng.choice([1, 1, 2, 4, 8])
        if Hkv * g > 64:
            g = 1
        Sq = rng.choice([1, 1, _log(rng, 2, 600), _log(rng, 2, 100)])
        B = _log(rng, 1, 32)
        Sk = _log(rng, 1, max(64, min(20000, 600_000_000 // (B * Hkv * g * Sq), 8_000_000 // (B * Hkv))))
        causal = rng.random() < 0.5
        return {"op": op, "B": B, "H": Hkv * g, "Hkv": Hkv, "Sq": Sq, "Sk": Sk, "D": D, "causal": causal,
                "ragged": rng.random() < 0.5, "mask": rng.random() < 0.3, "dtype": rng.choice(["bf16", "fp16"])}
    G = rng.choice([32, 64, 128])
    K = G * _log(rng, 1, 8192 // G)
    N = _log(rng, 1, 16384)
    M = rng.choice([_log(rng, 1, 8), _log(rng, 1, 80), _log(rng, 1, 600)])
    while M * N * K > 6_000_000_000:
        M = max(1, M // 2)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    return {"op": op, "M": M, "N": N, "K": K, "G": G, "act": rng.choice(["none", "none", "gelu", "silu"]),
            "bias": rng.random() < 0.7, "res": rng.random() < 0.4, "dtype": dtype,
            "y": rng.choice([dtype, dtype, "fp32"])}


def _lens(case):
    """Valid slots of each session (int list): all of them, or different ones."""
    B, Sk = case["B"], case["Sk"]
    if not case["ragged"]:
        return [Sk] * B
    return [max(1, Sk - (b * 1237) % (Sk // 2 + 1)) for b in range(B)]


def work(case):
    op = case["op"]
    if op == "norm_rope":
        e = 4 if case["dtype"] == "fp32" else 2
        n = case["B"] * case["S"] * (case["H"] + case["Hkv"]) * case["D"]
        return {"bytes": 2 * n * e + case["B"] * case["S"] * (4 + 4 * case["rot"]), "flops": 8 * n}
    if op == "append":
        e = 4 if case["dtype"] == "fp32" else 2
        row = 2 * case["Hkv"] * case["D"]                    # values of K and V per token
        new, cap = case["B"] * case["S"] * row, case["B"] * case["cap"] * row
        return {"bytes": new * e + new * 9 // 16 + cap * 9 // 16 + cap * 2, "flops": 4 * new + cap}
    if op == "attn":
        lens, D, Sq = _lens(case), case["D"], case["Sq"]
        pairs = sum(Sq * n - (min(Sq, n) * (min(Sq, n) - 1) // 2 + max(0, Sq - n) * n if case["causal"] else 0)
                    for n in lens)
        return {"bytes": sum(lens) * case["Hkv"] * D * 9 // 8 + 4 * case["B"] * case["H"] * Sq * D
                + (sum(lens) if case["mask"] else 0), "flops": 4 * pairs * case["H"] * D}
    M, N, K = case["M"], case["N"], case["K"]
    ye = 4 if case["y"] == "fp32" else 2
    return {"bytes": N * K // 2 + N * (K // case["G"]) * 2 + 2 * M * K + M * N * ye * (2 if case["res"] else 1)
            + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}


# ── inputs ───────────────────────────────────────────────────────────────────
def _pack(c):
    """Integer codes in [-8, 7], shape [..., n] -> packed bytes [..., n / 2]."""
    n = (c + 8).to(torch.uint8).reshape(*c.shape[:-1], c.shape[-1] // 8, 2, 2, 2)   # value 4q + 2h + p at [q][h][p]
    n = n.transpose(-3, -1)                                                         # [p][h][q]
    n = n.transpose(-2, -1)                                                         # [p][q][h]
    return (n[..., 0] | (n[..., 1] << 4)).reshape(*c.shape[:-1], c.shape[-1] // 2)


def _unpack(b):
    """Packed bytes [..., n / 2] -> codes in [-8, 7] (fp32), shape [..., n]."""
    b = b.reshape(*b.shape[:-1], b.shape[-1] // 4, 2, 2)                            # [p][q]
    n = torch.stack((b & 15, b >> 4), dim=-1)                                       # [p][q][h]
    n = n.transpose(-2, -1).transpose(-3, -1)                                       # [q][h][p]
    return n.reshape(*n.shape[:-4], -1).float() - 8.0


def _quantize(x):
    """fp32 [..., D] -> (packed codes [..., D / 2], fp16 scales [..., D / 32])."""
    g = x.float().reshape(*x.shape[:-1], x.shape[-1] // _GROUP, _GROUP)
    s = (g.abs().amax(-1) / 7.0).bfloat16().half()
    c = torch.round(g / s.float().unsqueeze(-1)).clamp(-7, 7)
    c = torch.where(s.unsqueeze(-1) > 0, c, torch.zeros_like(c)).reshape(x.shape)
    return _pack(c.to(torch.int32)), s


def _dequantize(codes, scale):
    c = _unpack(codes)
    return (c.reshape(*scale.shape, _GROUP) * scale.float().unsqueeze(-1)).reshape(c.shape)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 17)


def _cache(B, Hkv, cap, D, g):
    """K or V of a cache: unit-variance values with a different size per channel, quantised."""
    chan = 0.5 + torch.rand(D, generator=g, device="cuda")
    codes = torch.empty(B, Hkv, cap, D // 2, dtype=torch.uint8, device="cuda")
    scale = torch.empty(B, Hkv, cap, D // _GROUP, dtype=torch.float16, device="cuda")
    for b in range(B):
        codes[b], scale[b] = _quantize(torch.randn(Hkv, cap, D, generator=g, device="cuda") * chan)
    return codes, scale


def prepare(case, seed):
    g = _gen(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    op, st = case["op"], {"case": case}
    if op == "norm_rope":
        B, S, H, Hkv, D, rot = (case[k] for k in ("B", "S", "H", "Hkv", "D", "rot"))
        dt = _DT[case["dtype"]]
        qkv = (rn(B, S, H + 2 * Hkv, D) * 1.5).to(dt)          # the projection's output, read in place
        st["q"], st["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hkv]
        st["wq"], st["wk"] = (1 + 0.1 * rn(D)).to(dt), (1 + 0.1 * rn(D)).to(dt)
        st["pos"] = (case["pos0"] + 7 * torch.arange(B, device="cuda")[:, None]
                     + torch.arange(S, device="cuda")[None, :]).to(torch.int32)
        st["cos"] = st["sin"] = None
        if rot:
            n = case["pos0"] + 7 * B + S
            f = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
            a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * f
            st["cos"], st["sin"] = a.cos().float(), a.sin().float()
        return st
    if op == "append":
        B, S, Hkv, D, cap = (case[k] for k in ("B", "S", "Hkv", "D", "cap"))
        st["kc"], st["ks"] = _cache(B, Hkv, cap, D, g)
        st["vc"], st["vs"] = _cache(B, Hkv, cap, D, g)
        kv = (rn(B, S, 2, Hkv, D) * 1.2).to(_DT[case["dtype"]])   # the K/V projection's output
        st["k"], st["v"] = kv[:, :, 0], kv[:, :, 1]
        st["start"] = torch.randint(0, cap - S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        return st
    if op == "attn":
        B, H, Hkv, Sq, Sk, D = (case[k] for k in ("B", "H", "Hkv", "Sq", "Sk", "D"))
        cap = (Sk + 31) // 32 * 32
        st["kc"], st["ks"] = _cache(B, Hkv, cap, D, g)
        st["vc"], st["vs"] = _cache(B, Hkv, cap, D, g)
        st["q"] = rn(B, Sq, H, D).to(_DT[case["dtype"]])          # a projection's output, heads inside
        st["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
        st["mask"] = torch.rand(B, Sk, generator=g, device="cuda") < 0.75 if case["mask"] else None
        return st
    M, N, K, G = (case[k] for k in ("M", "N", "K", "G"))
    dt = _DT[case["dtype"]]
    w = rn(N, K // G, G) * 0.02
    s = (w.abs().amax(-1) / 7.0).half()
    c = torch.round(w / s.float().unsqueeze(-1)).clamp(-7, 7)
    st["w"], st["ws"] = _pack(c.reshape(N, K).to(torch.int32)), s
    st["x"] = rn(M, K).to(dt)
    st["b"] = (0.1 * rn(N)).to(dt) if case["bias"] else None
    st["r"] = rn(M, N).to(_DT[case["y"]]) if case["res"] else None
    return st


# ── the operators ────────────────────────────────────────────────────────────
def _visible(case, lens, mask):
    """[B, 1, Sq, Sk] truth values: which slots a query sees."""
    Sq, Sk = case["Sq"], case["Sk"]
    j = torch.arange(Sk, device="cuda")
    vis = (j[None, None, :] < lens[:, None, None]).expand(-1, Sq, -1)
    if case["causal"]:               # the queries are the last Sq tokens of the session
        i = torch.arange(Sq, device="cuda")
        vis = vis & (j[None, None, :] <= (lens[:, None] - Sq + i[None, :])[:, :, None])
    if mask is not None:
        vis = vis & mask[:, None, :]
    return vis[:, None]


def _rotate(x, cos, sin, inter):
    rot = 2 * cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    r, rest = x[..., :rot], x[..., rot:]
    if inter:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((r, rest), dim=-1)


def _act(y, act):
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y * torch.sigmoid(y) if act == "silu" else y


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return _run_own(case, op, state)
    if op == "norm_rope":
        outs = []
        for x, w in ((state["q"], state["wq"]), (state["k"], state["wk"])):
            f = x.float()
            y = f / torch.sqrt(f.square().mean(-1, keepdim=True) + 1e-6) * w.float()
            if state["cos"] is not None:
                p = state["pos"].long()
                y = _rotate(y, state["cos"][p], state["sin"][p], case["inter"])
            outs.append(y.to(x.dtype))
        return tuple(outs)
    if op == "append":
        S = case["S"]
        slots = state["start"].long()[:, None] + torch.arange(S, device="cuda")[None, :]
        b = torch.arange(case["B"], device="cuda")[:, None]
        for x, codes, scale in ((state["k"], state["kc"], state["ks"]), (state["v"], state["vc"], state["vs"])):
            c, s = _quantize(x)
            codes[b, :, slots] = c
            scale[b, :, slots] = s
        return (_dequantize(state["kc"], state["ks"]).half(), _dequantize(state["vc"], state["vs"]).half())
    if op == "attn":
        Sk, D, g = case["Sk"], case["D"], case["H"] // case["Hkv"]
        k = _dequantize(state["kc"][:, :, :Sk], state["ks"][:, :, :Sk])
        v = _dequantize(state["vc"][:, :, :Sk], state["vs"][:, :, :Sk])
        q = state["q"].float().transpose(1, 2).reshape(case["B"], case["Hkv"], g * case["Sq"], D)
        s = torch.matmul(q, k.transpose(-1, -2)).reshape(case["B"], case["H"], case["Sq"], Sk) / math.sqrt(D)
        vis = _visible(case, state["lens"], state["mask"])
        s = torch.where(vis, s, torch.full_like(s, -math.inf))
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(m > -math.inf, m, torch.zeros_like(m)))
        l = p.sum(-1, keepdim=True)
        p = p / torch.where(l > 0, l, torch.ones_like(l))
        o = torch.matmul(p.reshape(case["B"], case["Hkv"], g * case["Sq"], Sk), v)
        return o.reshape(case["B"], case["H"], case["Sq"], D).transpose(1, 2).to(state["q"].dtype)
    G = case["G"]
    w = _unpack(state["w"])
    w = (w.reshape(w.shape[0], -1, G) * state["ws"].float().unsqueeze(-1)).reshape(w.shape)
    y = torch.matmul(state["x"].float(), w.t())
    if state["b"] is not None:
        y = y + state["b"].float()
    y = _act(y, case["act"])
    if state["r"] is not None:
        y = y + state["r"].float()
    return y.to(_DT[case["y"]])


def _run_own(case, op, state):
    be = _be()
    if op == "norm_rope":
        q, k = state["q"], state["k"]
        qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        be.qk_norm_rope(q, k, qo, ko, state["wq"], state["wk"], cos=state["cos"], sin=state["sin"],
                        positions=state["pos"], eps=1e-6, interleaved=case["inter"], layout="bshd")
        return qo, ko
    from servoflow_b200.quant4 import KV4Cache
    if op == "append":
        cache = KV4Cache(state["kc"], state["vc"], state["ks"], state["vs"])
        be.kv4_append(cache, state["k"], state["v"], start=state["start"], layout="bshd")
        shape = (case["B"], case["Hkv"], case["cap"], case["D"])
        ko = torch.empty(shape, dtype=torch.float16, device="cuda")
        vo = torch.empty(shape, dtype=torch.float16, device="cuda")
        be.kv4_read(cache, ko, vo)
        return ko, vo
    if op == "attn":
        cache = KV4Cache(state["kc"], state["vc"], state["ks"], state["vs"])
        q = state["q"]
        out = torch.empty_like(q)
        be.kv4_attention(q, cache, out, seq_k=case["Sk"], kv_len=state["lens"], mask=state["mask"],
                         is_causal=case["causal"], layout="bshd")
        return out
    out = torch.empty(case["M"], case["N"], dtype=_DT[case["y"]], device="cuda")
    be.w4a16_linear(state["x"], state["w"], state["ws"], out, bias=state["b"], residual=state["r"],
                    act=case["act"])
    return out


# ── the definitions in 64 bits ───────────────────────────────────────────────
def _nibbles64(b):
    """Codes as fp64, value by value from the format's bit positions."""
    w = b.reshape(*b.shape[:-1], -1, 4).to(torch.int64)
    w = w[..., 0] + (w[..., 1] << 8) + (w[..., 2] << 16) + (w[..., 3] << 24)
    bits = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=b.device)
    return (((w.unsqueeze(-1) >> bits) & 15) - 8).flatten(-2).double()


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm_rope":
        outs = []
        for x, w in ((st["q"].double(), st["wq"].double()), (st["k"].double(), st["wk"].double())):
            y = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / case["D"] + 1e-6) * w
            rot = case["rot"]
            if rot:
                i = torch.arange(rot // 2, device="cuda")
                ia, ib = (2 * i, 2 * i + 1) if case["inter"] else (i, i + rot // 2)
                ang = st["pos"].double()[..., None] * 10000.0 ** (-2.0 * i.double() / rot)
                z = torch.polar(torch.ones_like(ang), ang)[:, :, None] * torch.complex(y[..., ia], y[..., ib])
                y = y.clone()
                y[..., ia], y[..., ib] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    if op == "append":
        outs = []
        for x, codes, scale in ((st["k"], st["kc"], st["ks"]), (st["v"], st["vc"], st["vs"])):
            held = _nibbles64(codes).unflatten(-1, (-1, _GROUP)) * scale.double()[..., None]
            new = x.double().transpose(1, 2).unflatten(-1, (-1, _GROUP))
            s = (new.abs().amax(-1, keepdim=True).float() / 7.0).bfloat16().half().double()
            new = torch.where(s > 0, torch.round(new / s).clamp(-7, 7) * s, torch.zeros_like(new))
            for b, at in enumerate(st["start"].tolist()):
                held[b, :, at:at + case["S"]] = new[b]
            outs.append(held.flatten(-2))
        return tuple(outs)
    if op == "attn":
        B, Sq, H, D = st["q"].shape
        g = H // case["Hkv"]
        out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lens(case)):
            keep = torch.ones(n, dtype=torch.bool, device="cuda") if st["mask"] is None else st["mask"][b, :n]
            for hk in range(case["Hkv"]):
                k, v = ((_nibbles64(c[b, hk, :n]).unflatten(-1, (-1, _GROUP)) * s[b, hk, :n].double()[..., None])
                        .flatten(-2) for c, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
                q = st["q"][b, :, hk * g:(hk + 1) * g].double()
                t = torch.einsum("ihd,jd->hij", q, k) * D ** -0.5
                ok = keep[None, :].expand(Sq, n)
                if case["causal"]:
                    ok = ok & (torch.arange(n, device="cuda")[None, :] - torch.arange(Sq, device="cuda")[:, None] <= n - Sq)
                t = t.masked_fill(~ok, -1e300)
                e = torch.softmax(t, -1) * ok
                out[b, :, hk * g:(hk + 1) * g] = torch.einsum("hij,jd->ihd", e, v)
        return out
    w = _nibbles64(st["w"]).unflatten(-1, (-1, case["G"])) * st["ws"].double()[..., None]
    y = torch.einsum("mk,nk->mn", st["x"].double(), w.flatten(-2))
    if st["b"] is not None:
        y = y + st["b"].double()
    if case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    elif case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y if st["r"] is None else y + st["r"].double()
