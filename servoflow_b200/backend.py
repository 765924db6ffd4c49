"""Python mirror of the reference's IBackend operator interface for the
attention path (include/servoflow/backend/backend.h:102-110, 201-206,
227-229), over the C ABI of libsfb200.so.

Used by the tests and by bench.py; the production host side is C++ and binds
the same C ABI (include/sfb200.h). torch supplies device memory and streams
only; every op runs a libsfb200 kernel, and raises if the library is missing
or the device is not an sm_100a part.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _capi

_DTYPE_CODE = {
    torch.float32: _capi.SFB_F32,
    torch.float16: _capi.SFB_F16,
    torch.bfloat16: _capi.SFB_BF16,
    torch.int8: _capi.SFB_I8,
    torch.int32: _capi.SFB_I32,
    torch.bool: _capi.SFB_BOOL,
}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dt]
    except KeyError:
        raise _capi.SfbError(_capi.SFB_ERR_DTYPE, f"dtype {dt}") from None


def _stream_handle(stream) -> int:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


def _check_device(t: torch.Tensor, name: str) -> None:
    # reference: CUDABackend::check_device raises std::invalid_argument
    # (src/backend/cuda/cuda_backend.cu:156-161)
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor on this backend's device")


def attention_args(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, out: torch.Tensor,
                   mask: Optional[torch.Tensor] = None, scale: float = 0.0,
                   is_causal: bool = False, num_splits: int = 0,
                   layout: str = "bhsd") -> _capi.AttnArgs:
    """Fills sfb_attn_args from 4-D tensors.

    layout "bhsd": [B, H, S, D] (the reference layout); "bshd": [B, S, H, D].
    mask: None, a bool/uint8 [B, Sk] key-padding mask (True = keep), an
    int32 [B] tensor of valid key lengths, or the reference interface's
    additive float mask (fp32/fp16/bf16, 4-D [B or 1, 1, Sq or 1, Sk], added
    to the scaled logits; -inf masks a key).
    """
    for t, n in ((Q, "Q"), (K, "K"), (V, "V"), (out, "out")):
        _check_device(t, n)
        if t.dim() != 4:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{n} must be 4-D")
        if t.stride(3) != 1:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{n}: head_dim must be contiguous")
    v_f16 = Q.dtype == torch.bfloat16 and V.dtype == torch.float16
    if not (Q.dtype == K.dtype == out.dtype and (V.dtype == Q.dtype or v_f16)):
        raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "Q/K/V/out dtypes differ")
    if layout == "bhsd":
        bi, hi, si = 0, 1, 2
    elif layout == "bshd":
        bi, hi, si = 0, 2, 1
    else:
        raise ValueError(f"unknown layout {layout!r}")
    a = _capi.AttnArgs()
    a.q, a.k, a.v, a.out = Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr()
    for dst, t in ((a.q_stride, Q), (a.k_stride, K), (a.v_stride, V), (a.out_stride, out)):
        dst[0], dst[1], dst[2] = t.stride(bi), t.stride(hi), t.stride(si)
    a.batch, a.heads, a.seq_q, a.head_dim = Q.shape[bi], Q.shape[hi], Q.shape[si], Q.shape[3]
    a.heads_kv, a.seq_k = K.shape[hi], K.shape[si]
    if tuple(out.shape) != tuple(Q.shape) or tuple(V.shape) != tuple(K.shape) \
            or K.shape[bi] != Q.shape[bi] or K.shape[3] != Q.shape[3]:
        raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "inconsistent Q/K/V/out shapes")
    a.dtype = dtype_code(Q.dtype)
    a.is_causal = 1 if is_causal else 0
    a.scale = float(scale)
    a.num_splits = int(num_splits)
    a.v_dtype = _capi.SFB_F16 if v_f16 else 0
    a.kv_len = None
    a.key_mask = None
    if mask is not None:
        _check_device(mask, "mask")
        if mask.dtype == torch.int32 and mask.dim() == 1:
            if mask.shape[0] != a.batch or not mask.is_contiguous():
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "kv_len must be contiguous int32 [B]")
            a.kv_len = mask.data_ptr()
        elif mask.dtype in (torch.bool, torch.uint8) and mask.dim() == 2:
            if tuple(mask.shape) != (a.batch, a.seq_k) or mask.stride(1) != 1:
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "key mask must be [B, Sk], row-contiguous")
            a.key_mask = mask.data_ptr()
            a.key_mask_stride_b = mask.stride(0)
        elif mask.dtype in (torch.float32, torch.float16, torch.bfloat16) and mask.dim() == 4:
            mb, mh, mq, mk = mask.shape
            if mb not in (1, a.batch) or mh != 1 or mq not in (1, a.seq_q) or mk != a.seq_k \
                    or (mk > 1 and mask.stride(3) != 1):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "additive mask must be [B|1, 1, Sq|1, Sk]")
            a.attn_mask = mask.data_ptr()
            a.attn_mask_dtype = dtype_code(mask.dtype)
            a.attn_mask_stride[0] = mask.stride(0) if mb > 1 else 0
            a.attn_mask_stride[1] = mask.stride(2) if mq > 1 else 0
        else:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE,
                                 "mask must be bool/uint8 [B, Sk], int32 [B] lengths or a float "
                                 "[B, 1, Sq, Sk] additive mask")
    return a


_ACTS = {"none": 0, "gelu": 1, "silu": 2}
_HALVES = (torch.float16, torch.bfloat16)
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def _device_index(name: str, first: torch.Tensor, *others) -> int:
    """The CUDA device of `first`; raises unless every other tensor (or None) is on it."""
    i = first.get_device()
    if i < 0:
        _check_device(first, name)
    for t in others:
        if t is not None and t.get_device() != i:
            raise ValueError(f"every tensor of a call must be on {name}'s device cuda:{i}, not {t.device}")
    return i


_ORDER = {"bhsd": (0, 1, 2), "bshd": (0, 2, 1)}     # positions of (batch, head, seq) in a 4-D shape


def _order(layout: str):
    try:
        return _ORDER[layout]
    except KeyError:
        raise ValueError(f"unknown layout {layout!r}") from None


def _i32(name: str, v) -> int:
    """v as an argument of 32 bits: ctypes would cut a longer one short without a word."""
    v = int(v)
    if not -0x80000000 <= v <= 0x7fffffff:
        raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{name} {v} does not fit 32 bits")
    return v


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _call(fn, what: str, index: int, stream, *args) -> None:
    """Calls a library function on device `index`, on the given stream or that
    device's current one, and raises for its status."""
    current = torch.cuda.current_device()
    if current != index:
        with torch.cuda.device(index):
            return _call(fn, what, index, stream, *args)
    s = torch._C._cuda_getCurrentRawStream(index) if stream is None else _stream_handle(stream)
    status = fn(*args, s)
    if status != 0:
        raise _capi.SfbError(status, what)


class B200Backend:
    """The attention-path subset of IBackend, backed by libsfb200 kernels."""

    def __init__(self, device: int = 0):
        self.device = device
        self._lib = _capi.lib()
        self._graphs = {}

    # IBackend::attention (backend.h:105-110)
    def attention(self, Q, K, V, out, mask=None, scale: float = 0.0, is_causal: bool = False,
                  stream=None, num_splits: int = 0, layout: str = "bhsd") -> None:
        a = attention_args(Q, K, V, out, mask, scale, is_causal, num_splits, layout)
        _capi.check(self._lib.sfb_attention_fwd(ctypes.byref(a), _stream_handle(stream)),
                    "attention")

    # IBackend::dequantize (backend.h:205-206)
    def dequantize(self, input, scale, output, stream=None) -> None:
        for t, n in ((input, "input"), (scale, "scale"), (output, "output")):
            _check_device(t, n)
        if input.dtype != torch.int8:
            raise ValueError("dequantize_int8: input must be Int8")   # quantization.cu:62-64
        if input.numel() == 0:
            return
        if not (input.is_contiguous() and output.is_contiguous() and scale.is_contiguous()):
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "dequantize needs contiguous tensors")
        if output.shape != input.shape:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "output shape must equal input shape")
        rows = input.shape[0] if input.dim() > 0 else 1
        cols = input.numel() // max(rows, 1)
        _capi.check(self._lib.sfb_dequantize_int8(
            input.data_ptr(), scale.data_ptr(), dtype_code(scale.dtype), scale.numel(),
            output.data_ptr(), dtype_code(output.dtype), rows, cols, _stream_handle(stream)),
            "dequantize")

    # Two int8-weight linear layers as one persistent launch (a block's MLP at one session)
    def w8a16_mlp(self, x, w1, s1, w2, s2, out, b1=None, b2=None, residual=None, act: str = "gelu",
                  workspace=None, stream=None) -> None:
        """out[M, N] = act(x·(w1·s1)ᵀ + b1)·(w2·s2)ᵀ + b2 [+ residual] (sfb_w8a16_mlp)."""
        M, K = x.shape
        F, N = w1.shape[0], w2.shape[0]
        need = self._lib.sfb_w8a16_mlp_workspace_bytes(M, F)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        acts = {"none": 0, "gelu": 1, "silu": 2}
        p = lambda t: None if t is None else t.data_ptr()
        _capi.check(self._lib.sfb_w8a16_mlp(
            x.data_ptr(), x.stride(0), w1.data_ptr(), s1.data_ptr(), p(b1), w2.data_ptr(), s2.data_ptr(),
            p(b2), p(residual), residual.stride(0) if residual is not None else 0, out.data_ptr(),
            out.stride(0), dtype_code(out.dtype), M, K, F, N, acts[act], workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), _stream_handle(stream)), "w8a16_mlp")

    # Fused replacement of dequantize + gemm_bias_act (backend.h:160-185, 205-206)
    def w8a16_linear(self, x, w_q, w_scale, out, bias=None, residual=None, act: str = "none",
                     num_splits: int = 0, stream=None) -> None:
        """out[M, N] = act(x[M, K] · (w_q[N, K] · w_scale[N])ᵀ + bias) + residual."""
        for t, n in ((x, "x"), (w_q, "w_q"), (w_scale, "w_scale"), (out, "out")):
            _check_device(t, n)
        if x.dtype != torch.bfloat16 or w_q.dtype != torch.int8 or w_scale.dtype != torch.float32:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "x bf16, w_q int8, w_scale fp32 expected")
        if x.stride(1) != 1 or not w_q.is_contiguous() or out.stride(1) != 1:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "row-major tensors expected")
        M, K = x.shape
        N = w_q.shape[0]
        if w_q.shape[1] != K or tuple(out.shape) != (M, N) or w_scale.numel() != N:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "inconsistent shapes")
        if bias is not None and (bias.dtype != torch.bfloat16 or bias.numel() != N):
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "bias must be bf16 [N]")
        if residual is not None and (residual.dtype != out.dtype or tuple(residual.shape) != (M, N)
                                     or residual.stride(1) != 1):
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "residual must be [M, N] row-major in out's dtype")
        acts = {"none": 0, "gelu": 1, "silu": 2}
        _capi.check(self._lib.sfb_w8a16_linear(
            x.data_ptr(), x.stride(0), w_q.data_ptr(), w_scale.data_ptr(),
            None if bias is None else bias.data_ptr(),
            None if residual is None else residual.data_ptr(),
            0 if residual is None else residual.stride(0), out.data_ptr(), out.stride(0),
            dtype_code(out.dtype), M, N, K, acts[act], int(num_splits), _stream_handle(stream)),
            "w8a16_linear")

    # Query/key norms with the position rotation in one pass (dit_block.cu:185-196)
    def qk_norm_rope(self, q, k, q_out, k_out, q_weight=None, k_weight=None, cos=None, sin=None,
                     positions=None, eps: float = 1e-6, norm: bool = True, interleaved: bool = False,
                     layout: str = "bhsd", stream=None) -> None:
        """RMS norm per head of q and k (weights [D], None = 1; norm=False skips
        it), then the rotation by cos / sin (fp32 [positions, rot / 2]; None: no
        rotation) at positions (int32 [B, S]; None: 0..S-1), into q_out and
        k_out, which may be q and k. k (with k_out) or q (with q_out) may be
        None. Raises for shapes and types; a position outside the tables leaves
        its token unwritten and records SFB_ERR_RANGE (device_error)."""
        o = _order(layout)
        x = q if q is not None else k
        if x is None or (q is None) != (q_out is None) or (k is None) != (k_out is None):
            raise _capi.SfbError(_capi.SFB_ERR_INVALID, "q or k with its output expected")
        dev = _device_index("q" if q is not None else "k", x, q_out, k, k_out, q_weight, k_weight, cos, sin, positions)
        dt = x.dtype
        if dt not in _FLOATS:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, f"dtype {dt}")
        B, _, _, D = shape = x.shape if x.dim() == 4 else self._not_4d("q")
        S = shape[o[2]]

        def side(t, out, w, name):
            """Pointers, head count and strides of one of q and k."""
            if t is None:
                return 0, 0, 0, 0, (0, 0, 0), (0, 0, 0)
            sh, st, so = t.shape, t.stride(), out.stride()
            if len(sh) != 4 or out.shape != sh or sh[0] != B or sh[o[2]] != S or sh[3] != D:
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"inconsistent {name} shapes")
            if D > 1 and (st[3] != 1 or so[3] != 1):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{name}: head_dim must be contiguous")
            if t.dtype is not dt or out.dtype is not dt or (w is not None and w.dtype is not dt):
                raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "q, k, outputs and weights share one dtype")
            if w is not None and (w.shape != (D,) or not w.is_contiguous()):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{name}_weight must be contiguous [head_dim]")
            return (t.data_ptr(), out.data_ptr(), _ptr(w), sh[o[1]], (st[o[0]], st[o[1]], st[o[2]]),
                    (so[o[0]], so[o[1]], so[o[2]]))

        qp, qop, qw, H, qs, qos = side(q, q_out, q_weight, "q")
        kp, kop, kw, Hkv, ks, kos = side(k, k_out, k_weight, "k")
        table = rot = pos = pos_sb = 0
        if (cos is None) != (sin is None):
            raise _capi.SfbError(_capi.SFB_ERR_INVALID, "cos and sin come together")
        if cos is not None:
            if cos.dim() != 2 or cos.shape != sin.shape or not cos.is_contiguous() or not sin.is_contiguous():
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "cos / sin must be contiguous [positions, rot / 2]")
            if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
                raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "cos / sin must be fp32")
            table, rot = cos.shape
            rot *= 2
            if positions is not None:
                if positions.dtype is not torch.int32:
                    raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "positions must be int32")
                if positions.shape != (B, S) or (S > 1 and positions.stride(1) != 1):
                    raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "positions must be [B, S], row-contiguous")
                pos, pos_sb = positions.data_ptr(), positions.stride(0)
        args = _capi.NORM_ROPE_ARGS.pack(
            qp, kp, qop, kop, *qs, *ks, *qos, *kos, qw, kw, _ptr(cos), _ptr(sin), pos, pos_sb, table, B, S, H, Hkv, D,
            rot, 1 if interleaved else 0, 1 if norm else 0, _DTYPE_CODE[dt], eps)
        _call(self._lib.sfb_qk_norm_rope, "qk_norm_rope", dev, stream, args)

    @staticmethod
    def _not_4d(name):
        raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{name} must be 4-D")

    # The K/V cache held in 4 bits (quant4.KV4Cache)
    @staticmethod
    def _kv4_side(t, name, o, B, Hkv, D):
        """Packed strides (batch, head, seq) of a 16- or 32-bit K or V that fits the cache."""
        sh, st = t.shape, t.stride()
        if len(sh) != 4 or sh[0] != B or sh[o[1]] != Hkv or sh[3] != D:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{name} does not fit the cache")
        if st[3] != 1:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{name}: head_dim must be contiguous")
        return _capi.I64X3.pack(st[0], st[o[1]], st[o[2]])

    def kv4_append(self, cache, K, V, start=0, lens=None, layout: str = "bhsd", stream=None) -> None:
        """Quantises K and V ([B, Hkv, S, D] or, layout "bshd", [B, S, Hkv, D])
        into the cache: token i of session b goes to slot start + i (start an
        int, or int32 [B]), only the first lens[b] tokens where lens (int32 [B])
        is given. With tensor starts, tokens outside the cache are not written
        and record SFB_ERR_RANGE (device_error)."""
        o = _order(layout)
        c, B, Hkv, _, D, _ = cache.pack()
        start_t = start if isinstance(start, torch.Tensor) else None
        dev = _device_index("cache", cache.k_codes, K, V, start_t, lens)
        if K.shape != V.shape:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "K and V shapes differ")
        if K.dtype not in _FLOATS or V.dtype is not K.dtype:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "K and V share one float dtype")
        ks, vs = self._kv4_side(K, "K", o, B, Hkv, D), self._kv4_side(V, "V", o, B, Hkv, D)
        for t, n in ((start_t, "start"), (lens, "lens")):
            if t is not None and (t.dtype is not torch.int32 or t.shape != (B,) or not t.is_contiguous()):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{n} must be contiguous int32 [B]")
        _call(self._lib.sfb_kv4_append, "kv4_append", dev, stream, c, K.data_ptr(), ks, V.data_ptr(), vs,
              _DTYPE_CODE[K.dtype], _i32("seq", K.shape[o[2]]), _ptr(start_t),
              0 if start_t is not None else _i32("start", start), _ptr(lens))

    def kv4_read(self, cache, K=None, V=None, slot0: int = 0, layout: str = "bhsd", stream=None) -> None:
        """Writes the values of slots [slot0, slot0 + S) into K and V ([B, Hkv,
        S, D] or bshd; fp16 and fp32 exactly, bf16 rounded); either may be None."""
        o = _order(layout)
        c, B, Hkv, _, D, _ = cache.pack()
        x = K if K is not None else V
        if x is None:
            raise _capi.SfbError(_capi.SFB_ERR_INVALID, "K or V expected")
        dev = _device_index("cache", cache.k_codes, K, V)
        if K is not None and V is not None and (K.shape != V.shape or K.dtype is not V.dtype):
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "K and V differ in shape or dtype")
        if x.dtype not in _FLOATS:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, f"dtype {x.dtype}")
        ks = None if K is None else self._kv4_side(K, "K", o, B, Hkv, D)
        vs = None if V is None else self._kv4_side(V, "V", o, B, Hkv, D)
        _call(self._lib.sfb_kv4_read, "kv4_read", dev, stream, c, _ptr(K), ks, _ptr(V), vs, _DTYPE_CODE[x.dtype],
              _i32("slot0", slot0), _i32("seq", x.shape[o[2]]))

    def kv4_attention(self, Q, cache, out, seq_k: Optional[int] = None, kv_len=None, mask=None,
                      scale: float = 0.0, is_causal: bool = False, num_splits: int = 0,
                      layout: str = "bhsd", stream=None) -> None:
        """Attention of Q over the first seq_k slots of a KV4Cache (None: all of
        them). Q, out: bf16 or fp16 [B, H, Sq, D] (or bshd), H a multiple of the
        cache's heads. kv_len: int32 [B] valid slots; mask: bool/uint8 [B,
        seq_k] (True = keep); is_causal: the queries are the last Sq tokens of
        the valid slots. A query that sees no slot gives zeros."""
        o = _order(layout)
        c, B, _, cap, D, _ = cache.pack()
        dev = _device_index("cache", cache.k_codes, Q, out, kv_len, mask)
        dt, sh, st, so = Q.dtype, Q.shape, Q.stride(), out.stride()
        if dt not in _HALVES or out.dtype is not dt:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "Q and out must be bf16 or fp16, alike")
        if len(sh) != 4 or out.shape != sh or sh[0] != B or sh[3] != D:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "Q and out must be 4-D and fit the cache")
        if st[3] != 1 or so[3] != 1:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "head_dim must be contiguous")
        sk = cap if seq_k is None else _i32("seq_k", seq_k)
        lens = keep = keep_sb = 0
        if kv_len is not None:
            if kv_len.dtype is not torch.int32 or kv_len.shape != (B,) or not kv_len.is_contiguous():
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "kv_len must be contiguous int32 [B]")
            lens = kv_len.data_ptr()
        if mask is not None:
            if mask.dtype not in (torch.bool, torch.uint8):
                raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "mask must be bool or uint8")
            if mask.shape != (B, sk) or (sk > 1 and mask.stride(1) != 1):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "mask must be [B, seq_k], row-contiguous")
            keep, keep_sb = mask.data_ptr(), mask.stride(0)
        h, s = o[1], o[2]
        args = _capi.KV4_ATTN_ARGS.pack(
            Q.data_ptr(), out.data_ptr(), st[0], st[h], st[s], so[0], so[h], so[s], lens, keep, keep_sb, sh[h], sh[s],
            sk, _DTYPE_CODE[dt], 1 if is_causal else 0, int(num_splits), scale)
        _call(self._lib.sfb_kv4_attention, "kv4_attention", dev, stream, c, args)

    # Linear layer with 4-bit weights and group scales (quant4.pack_w4)
    def w4a16_linear(self, x, w_q, w_scale, out, bias=None, residual=None, act: str = "none",
                     stream=None) -> None:
        """out[M, N] = act(x[M, K] · w^T + bias) + residual with w[n, k] =
        c[n, k] · w_scale[n, k / group]: w_q uint8 [N, K / 2] packed codes,
        w_scale [N, K / group] fp16, bf16 or fp32 (group 32, 64 or 128 follows
        from its shape). x and bias bf16 or fp16; out x's dtype or fp32."""
        dev = _device_index("x", x, w_q, w_scale, out, bias, residual)
        if x.dtype not in _HALVES or w_q.dtype != torch.uint8 or w_scale.dtype not in _FLOATS:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "x bf16 or fp16, w_q uint8, w_scale float expected")
        if out.dtype != x.dtype and out.dtype != torch.float32:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "out must be fp32 or x's dtype")
        if x.dim() != 2 or w_q.dim() != 2 or w_scale.dim() != 2 or out.dim() != 2:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "2-D tensors expected")
        (M, K), (N, K2), (_, groups) = x.shape, w_q.shape, w_scale.shape
        if 2 * K2 != K or w_scale.shape[0] != N or out.shape[0] != M or out.shape[1] != N or groups < 1 \
                or K % groups:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "inconsistent shapes")
        if (K > 1 and x.stride(1) != 1) or not w_q.is_contiguous() or not w_scale.is_contiguous() \
                or (N > 1 and out.stride(1) != 1):
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "row-major tensors expected")
        if bias is not None and (bias.dtype != x.dtype or tuple(bias.shape) != (N,) or (N > 1 and bias.stride(0) != 1)):
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "bias must be [N] in x's dtype")
        if residual is not None and (residual.dtype != out.dtype or residual.shape != out.shape
                                     or (N > 1 and residual.stride(1) != 1)):
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "residual must be [M, N] row-major in out's dtype")
        if act not in _ACTS:
            raise ValueError(f"unknown act {act!r}")
        # a single row's stride is never used: pass one that fits
        ldx, ldr, ldy = (K + 7) // 8 * 8, N, N
        if M > 1:
            ldx, ldy = x.stride(0), out.stride(0)
            if residual is not None:
                ldr = residual.stride(0)
        _call(self._lib.sfb_w4a16_linear, "w4a16_linear", dev, stream, x.data_ptr(), ldx, _DTYPE_CODE[x.dtype],
              w_q.data_ptr(), w_scale.data_ptr(), _DTYPE_CODE[w_scale.dtype], K // groups, _ptr(bias),
              _ptr(residual), ldr, out.data_ptr(), ldy, _DTYPE_CODE[out.dtype], _i32("M", M), _i32("N", N), _i32("K", K),
              _ACTS[act])

    # Graph hooks (backend.h:227-229; CUDABackend keeps one graph per stream,
    # cuda_backend.cu:592-608).
    def graph_begin_capture(self, stream) -> None:
        g = torch.cuda.CUDAGraph()
        self._graphs[_stream_handle(stream)] = g
        g.capture_begin()

    def graph_end_capture(self, stream) -> None:
        self._graphs[_stream_handle(stream)].capture_end()

    def graph_launch(self, stream) -> None:
        self._graphs[_stream_handle(stream)].replay()

    @staticmethod
    def device_error(reset: bool = True) -> int:
        code = ctypes.c_int(0)
        _capi.check(_capi.lib().sfb_device_error(ctypes.byref(code), 1 if reset else 0),
                    "device_error")
        return code.value
