"""CPU tests of the 4-bit formats (servoflow_b200.quant4) and of the refusals of
the 4-bit and norm-rotation entry points that need no device."""
import re
import struct

import pytest
import torch

from servoflow_b200 import _capi, quant4
from servoflow_b200._capi import SfbError


def test_packing_follows_the_bit_positions():
    # value 2i of eight at bits 4i, value 2i+1 at bits 16+4i, nibble = c + 8
    codes = torch.tensor([[-8, 7, 0, 1, -1, 3, 5, -4], [2, 2, -3, 6, 7, -8, 0, -7]], dtype=torch.int32)
    packed = quant4.pack_codes(codes)
    assert packed.shape == (2, 4) and packed.dtype == torch.uint8
    for row, b in zip(codes.tolist(), packed.tolist()):
        word = struct.unpack("<I", bytes(b))[0]
        got = [((word >> (4 * (e // 2) + 16 * (e % 2))) & 15) - 8 for e in range(8)]
        assert got == row


@pytest.mark.parametrize("shape", [(8,), (3, 64), (2, 5, 128), (0, 32)])
def test_unpack_inverts_pack(shape):
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(-8, 8, shape, generator=g, dtype=torch.int32)
    assert torch.equal(quant4.unpack_codes(quant4.pack_codes(codes)).to(torch.int32), codes)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_pack_w4_error_is_half_a_step(group):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(24, 256, generator=g) * 0.05
    w[3] = 0                                           # a row of zeros: scale 0, codes 0
    packed, s = quant4.pack_w4(w, group, torch.float32)
    assert packed.shape == (24, 128) and s.shape == (24, 256 // group)
    back = quant4.unpack_codes(packed).float().unflatten(1, (-1, group)) * s.unsqueeze(-1)
    # fp32 scales: max|w| / 7 up to one rounding, so no code is clamped by more than that
    assert ((back.flatten(1) - w).abs() <= (s.unsqueeze(-1).expand(-1, -1, group).flatten(1)) * (0.5 + 1e-5)).all()
    assert (s[3] == 0).all() and (back[3] == 0).all()


def test_packing_refusals():
    with pytest.raises(SfbError):
        quant4.pack_codes(torch.zeros(4, 12, dtype=torch.int32))
    with pytest.raises(SfbError):
        quant4.pack_w4(torch.zeros(4, 96), 64)
    with pytest.raises(SfbError):
        quant4.pack_w4(torch.zeros(4, 96), 48)
    with pytest.raises(SfbError):
        quant4.KV4Cache.allocate(1, 1, 32, 96, device="cpu")


def test_cache_allocation_is_zero_and_rounded():
    c = quant4.KV4Cache.allocate(2, 3, 33, 64, device="cpu")
    assert c.shape == (2, 3, 64, 64)
    k, v = c.dequantize()
    assert (k == 0).all() and (v == 0).all() and k.shape == (2, 3, 64, 64)
    with pytest.raises(ValueError):                    # the struct needs a CUDA cache
        c.pack()


def _offsets(struct_name, fields):
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    prints = ", ".join(f"offsetof({struct_name}, {f})" for f in fields)
    src = ("#include <stddef.h>\n#include <stdio.h>\n#include \"sfb200.h\"\n"
           f"int main(void) {{ printf(\"{'%zu ' * (len(fields) + 1)}\\n\", {prints}, sizeof({struct_name})); "
           "return 0; }\n")
    with tempfile.TemporaryDirectory() as d:
        c = os.path.join(d, "t.c")
        with open(c, "w") as f:
            f.write(src)
        exe = os.path.join(d, "t")
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), c, "-o", exe], check=True)
        return list(map(int, subprocess.run([exe], capture_output=True, text=True).stdout.split()))


CACHE = ("k_codes", "v_codes", "k_scale", "v_scale", "code_stride[0]", "code_stride[1]", "scale_stride[0]",
         "scale_stride[1]", "batch", "heads_kv", "capacity", "head_dim")
ATTN = ("q", "out", "q_stride[0]", "q_stride[1]", "q_stride[2]", "out_stride[0]", "out_stride[1]", "out_stride[2]",
        "kv_len", "key_mask", "key_mask_stride_b", "heads", "seq_q", "seq_k", "dtype", "is_causal", "num_splits",
        "scale")
ROPE = ("q", "k", "q_out", "k_out") + tuple(
    f"{n}[{i}]" for n in ("q_stride", "k_stride", "q_out_stride", "k_out_stride") for i in range(3)) + (
    "q_weight", "k_weight", "cos_table", "sin_table", "positions", "pos_stride_b", "table_len", "batch", "seq", "heads",
    "heads_kv", "head_dim", "rotary_dim", "interleaved", "norm", "dtype", "eps")


def test_packed_structs_have_the_c_layout():
    for name, fmt, fields in (("sfb_kv4_cache", _capi.KV4_CACHE, CACHE), ("sfb_kv4_attn_args", _capi.KV4_ATTN_ARGS, ATTN),
                              ("sfb_norm_rope_args", _capi.NORM_ROPE_ARGS, ROPE)):
        got = _offsets(name, fields)
        codes = [ch for n, ch in re.findall(r"(\d*)([a-zA-Z])", fmt.format[:-2]) for _ in range(int(n or 1))]
        assert len(codes) == len(fields) and got[-1] == fmt.size, name
        want = [struct.calcsize("".join(codes[:i]) + "0" + codes[i]) for i in range(len(codes))]
        assert got[:-1] == want, name


def _packed(fmt, fields, values, over):
    v = dict.fromkeys(fields, 0) | values | over
    assert set(v) == set(fields), set(v) ^ set(fields)
    return fmt.pack(*(v[f] for f in fields))


def _cache(**over):
    return _packed(_capi.KV4_CACHE, CACHE, {
        "k_codes": 0x1000, "v_codes": 0x1000, "k_scale": 0x1000, "v_scale": 0x1000, "code_stride[0]": 8192,
        "code_stride[1]": 2048, "scale_stride[0]": 512, "scale_stride[1]": 128, "batch": 2, "heads_kv": 4,
        "capacity": 64, "head_dim": 64}, over)


BAD_CACHES = [
    (dict(k_codes=0), _capi.SFB_ERR_INVALID), (dict(v_scale=0), _capi.SFB_ERR_INVALID),
    (dict(head_dim=96), _capi.SFB_ERR_SHAPE), (dict(head_dim=0), _capi.SFB_ERR_SHAPE),
    (dict(heads_kv=0), _capi.SFB_ERR_SHAPE), (dict(capacity=-1), _capi.SFB_ERR_SHAPE),
    (dict(capacity=66), _capi.SFB_ERR_SHAPE), (dict(capacity=0x7ffffffc), _capi.SFB_ERR_SHAPE),
    (dict(k_codes=0x1008), _capi.SFB_ERR_ALIGN), (dict(v_scale=0x1002), _capi.SFB_ERR_ALIGN),
    ({"code_stride[1]": 2056}, _capi.SFB_ERR_ALIGN), ({"scale_stride[0]": 514}, _capi.SFB_ERR_ALIGN),
]


def _attn(**over):
    strides = {f: 64 for f in ATTN if "_stride[" in f}
    return _packed(_capi.KV4_ATTN_ARGS, ATTN, strides | {
        "q": 0x2000, "out": 0x3000, "heads": 8, "seq_q": 3, "seq_k": 64, "dtype": _capi.SFB_BF16}, over)


I3 = _capi.I64X3.pack


@pytest.mark.parametrize("over,status", BAD_CACHES)
def test_bad_caches_are_refused_by_every_entry_point(over, status):
    lib = _capi.lib()
    c, st = _cache(**over), I3(8192, 64, 256)
    assert lib.sfb_kv4_append(c, 0x2000, st, 0x2000, st, _capi.SFB_BF16, 1, None, 0, None, None) == status
    assert lib.sfb_kv4_read(c, 0x2000, st, 0x2000, st, _capi.SFB_F16, 0, 1, None) == status
    assert lib.sfb_kv4_attention(c, _attn(seq_k=0), None) == status


def test_append_and_read_refusals():
    lib, E = _capi.lib(), _capi
    c, st, odd = _cache(), I3(8192, 64, 256), I3(8192, 64, 255)
    append = lambda cc, k, ks, v, vs, dt, seq, slot: lib.sfb_kv4_append(cc, k, ks, v, vs, dt, seq, None, slot, None, None)
    assert append(None, 0x2000, st, 0x2000, st, E.SFB_BF16, 1, 0) == E.SFB_ERR_INVALID
    assert append(c, None, st, 0x2000, st, E.SFB_BF16, 1, 0) == E.SFB_ERR_INVALID
    assert append(c, 0x2000, None, 0x2000, st, E.SFB_BF16, 1, 0) == E.SFB_ERR_INVALID
    assert append(c, 0x2000, st, 0x2000, st, E.SFB_I8, 1, 0) == E.SFB_ERR_DTYPE
    assert append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, -1, 0) == E.SFB_ERR_SHAPE
    assert append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, 65, 0) == E.SFB_ERR_SHAPE      # past the capacity
    assert append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, 1, 64) == E.SFB_ERR_SHAPE
    assert append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, 1, -1) == E.SFB_ERR_SHAPE
    assert append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, 2 ** 31 - 1, 2 ** 31 - 1) == E.SFB_ERR_SHAPE
    assert append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, 2 ** 31 - 1, 0) == E.SFB_ERR_SHAPE
    # with per-session starts the slots are known on the device alone
    assert lib.sfb_kv4_append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, 2 ** 31 - 1, 0x2000, 0, None, None) == E.SFB_ERR_SHAPE
    assert append(c, 0x2008, st, 0x2000, st, E.SFB_BF16, 1, 0) == E.SFB_ERR_ALIGN
    assert append(c, 0x2000, st, 0x2000, odd, E.SFB_BF16, 1, 0) == E.SFB_ERR_ALIGN
    assert append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, 0, 0) == E.SFB_OK              # nothing to do
    read = lambda k, ks, v, vs, dt, slot, seq: lib.sfb_kv4_read(c, k, ks, v, vs, dt, slot, seq, None)
    assert read(None, st, None, st, E.SFB_F16, 0, 1) == E.SFB_ERR_INVALID
    assert read(0x2000, st, None, None, E.SFB_I32, 0, 1) == E.SFB_ERR_DTYPE
    assert read(0x2000, st, None, None, E.SFB_F16, 0, 65) == E.SFB_ERR_SHAPE
    assert read(0x2000, st, None, None, E.SFB_F16, -1, 1) == E.SFB_ERR_SHAPE
    assert read(0x2004, st, None, None, E.SFB_F16, 0, 1) == E.SFB_ERR_ALIGN
    assert read(0x2000, st, None, None, E.SFB_F16, 64, 0) == E.SFB_OK


def test_attention_refusals():
    lib, E = _capi.lib(), _capi
    call = lambda **over: lib.sfb_kv4_attention(_cache(), _attn(**over), None)
    assert lib.sfb_kv4_attention(_cache(), None, None) == E.SFB_ERR_INVALID
    assert lib.sfb_kv4_attention(None, _attn(), None) == E.SFB_ERR_INVALID
    assert call(q=0) == E.SFB_ERR_INVALID
    assert call(dtype=E.SFB_F32) == E.SFB_ERR_DTYPE
    assert call(heads=6) == E.SFB_ERR_SHAPE
    assert call(heads=0) == E.SFB_ERR_SHAPE
    assert call(seq_k=65) == E.SFB_ERR_SHAPE
    assert call(seq_k=-1) == E.SFB_ERR_SHAPE
    assert call(seq_q=-1) == E.SFB_ERR_SHAPE
    assert call(seq_q=2 ** 31 - 1) == E.SFB_ERR_SHAPE
    assert call(num_splits=17) == E.SFB_ERR_INVALID
    assert call(q=0x2002) == E.SFB_ERR_ALIGN
    assert call(**{"q_stride[2]": 67}) == E.SFB_ERR_ALIGN
    assert call(**{"out_stride[2]": 68}) == E.SFB_ERR_ALIGN
    assert call(seq_q=0) == E.SFB_OK


def test_norm_rope_refusals():
    lib, E = _capi.lib(), _capi
    base = {f: 64 for f in ROPE if "stride[" in f} | {
        "q": 0x1000, "k": 0x1000, "q_out": 0x1000, "k_out": 0x1000, "cos_table": 0x4000, "sin_table": 0x4000,
        "table_len": 10, "batch": 2, "seq": 3, "heads": 4, "heads_kv": 2, "head_dim": 64, "rotary_dim": 64, "norm": 1,
        "dtype": E.SFB_BF16, "eps": 1e-6}
    call = lambda **over: lib.sfb_qk_norm_rope(_packed(_capi.NORM_ROPE_ARGS, ROPE, base, over), None)
    assert lib.sfb_qk_norm_rope(None, None) == E.SFB_ERR_INVALID
    assert call(q=0) == E.SFB_ERR_INVALID                         # an output without its input
    assert call(q=0, q_out=0, k=0, k_out=0) == E.SFB_ERR_INVALID
    assert call(cos_table=0) == E.SFB_ERR_INVALID
    assert call(dtype=E.SFB_I8) == E.SFB_ERR_DTYPE
    assert call(head_dim=60) == E.SFB_ERR_SHAPE
    assert call(head_dim=264, rotary_dim=0) == E.SFB_ERR_SHAPE
    assert call(rotary_dim=8) == E.SFB_ERR_SHAPE
    assert call(rotary_dim=80) == E.SFB_ERR_SHAPE
    assert call(batch=-1) == E.SFB_ERR_SHAPE
    assert call(q=0x1004, q_out=0x1004) == E.SFB_ERR_ALIGN
    assert call(**{"k_out_stride[1]": 65}) == E.SFB_ERR_ALIGN
    assert call(sin_table=0x4004) == E.SFB_ERR_ALIGN
    assert call(batch=0) == E.SFB_OK
    assert call(seq=0) == E.SFB_OK


def test_linear_refusals():
    lib, E = _capi.lib(), _capi

    def call(x=0x1000, ldx=256, xd=E.SFB_BF16, w=0x2000, ws=0x3000, sd=E.SFB_F16, G=64, b=None, r=None, ldr=0,
             y=0x5000, ldy=40, yd=E.SFB_BF16, M=3, N=40, K=256, act=0):
        return lib.sfb_w4a16_linear(x, ldx, xd, w, ws, sd, G, b, r, ldr, y, ldy, yd, M, N, K, act, None)

    for name in ("x", "w", "ws", "y"):
        assert call(**{name: None}) == E.SFB_ERR_INVALID
    assert call(act=3) == E.SFB_ERR_INVALID
    assert call(G=16) == E.SFB_ERR_SHAPE
    assert call(K=96, ldx=96, G=64) == E.SFB_ERR_SHAPE
    assert call(M=-1) == E.SFB_ERR_SHAPE
    assert call(N=0) == E.SFB_ERR_SHAPE
    assert call(ldx=248) == E.SFB_ERR_SHAPE
    assert call(ldy=39) == E.SFB_ERR_SHAPE
    assert call(r=0x6000, ldr=39) == E.SFB_ERR_SHAPE
    assert call(xd=E.SFB_F32) == E.SFB_ERR_DTYPE
    assert call(yd=E.SFB_F16) == E.SFB_ERR_DTYPE
    assert call(sd=E.SFB_I8) == E.SFB_ERR_DTYPE
    assert call(x=0x1008) == E.SFB_ERR_ALIGN
    assert call(w=0x2004) == E.SFB_ERR_ALIGN
    assert call(ldx=260) == E.SFB_ERR_ALIGN
    assert call(y=0x5001) == E.SFB_ERR_ALIGN
    assert call(M=0) == E.SFB_OK


def test_copies_of_a_models_cache_are_on_its_device(monkeypatch):
    """With another device current: the model's is waited for, and holds the copy (fakes
    of the library and of torch's device calls)."""
    from servoflow_b200 import rdt1b
    shape, seen = (2, 2, 32, 64), []

    class Lib:
        def sfb_rdt1b_kv4_cache(self, h, layer, buf):
            buf.raw = _capi.KV4_CACHE.pack(0x1000, 0x2000, 0x3000, 0x4000, 2048, 1024, 128, 64, *shape)
            return 0

    model = rdt1b.RDT1B.__new__(rdt1b.RDT1B)
    model.lib, model.h, model.device = Lib(), None, 5
    empty = torch.empty
    monkeypatch.setattr(rdt1b.torch.cuda, "synchronize", lambda device=None: seen.append(("wait", device)))
    monkeypatch.setattr(rdt1b.torch, "empty", lambda s, dtype, device: seen.append(("copy", device)) or empty(s, dtype=dtype))
    monkeypatch.setattr(rdt1b, "_copy_d2d", lambda dst, src, n: None)
    cache = model.kv4_cache(0)
    assert cache.shape == shape
    assert seen == [("wait", 5)] + 4 * [("copy", "cuda:5")]


def test_linear_sizes_next_to_2_31_are_refused():
    """The kernels index channels and inputs in 32 bits, up to a tile past the last one."""
    lib, E = _capi.lib(), _capi

    def call(N, K, G):
        return lib.sfb_w4a16_linear(0x1000, 2 ** 31, E.SFB_BF16, 0x2000, 0x3000, E.SFB_F16, G, None, None, 0, 0x5000,
                                    2 ** 31, E.SFB_BF16, 1, N, K, 0, None)

    for n in (2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 64, 2 ** 31 - 1023):
        assert call(n, 64, 64) == E.SFB_ERR_SHAPE
    for k in (2 ** 31 - 128, 2 ** 31 - 512, 2 ** 31 - 896):
        assert call(16, k, 128) == E.SFB_ERR_SHAPE


@pytest.mark.parametrize("capacity", [2 ** 31 - 256, 2 ** 31 - 508])
def test_capacities_next_to_2_31_are_refused(capacity):
    """The attention looks two blocks of 128 slots ahead, counted in 32 bits."""
    lib, E = _capi.lib(), _capi
    c, st = _cache(capacity=capacity), I3(8192, 64, 256)
    assert lib.sfb_kv4_attention(c, _attn(seq_k=capacity), None) == E.SFB_ERR_SHAPE
    assert lib.sfb_kv4_append(c, 0x2000, st, 0x2000, st, E.SFB_BF16, 1, None, capacity - 1, None, None) == E.SFB_ERR_SHAPE
    assert lib.sfb_kv4_read(c, 0x2000, st, 0x2000, st, E.SFB_F16, capacity - 1, 1, None) == E.SFB_ERR_SHAPE


def test_arguments_past_32_bits_are_refused():
    from servoflow_b200.backend import _i32
    assert _i32("N", 2 ** 31 - 1) == 2 ** 31 - 1 and _i32("start", -2 ** 31) == -2 ** 31
    for v in (2 ** 31, 2 ** 32 + 16, -2 ** 31 - 1):        # 2^32 + 16 was taken for 16
        with pytest.raises(SfbError):
            _i32("N", v)
