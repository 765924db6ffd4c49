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


def _one_device(first: torch.Tensor, name: str, *others) -> torch.device:
    """The CUDA device of `first`; raises unless every other tensor (or None) is on it."""
    _check_device(first, name)
    dev = first.device
    for t, n in others:
        if t is not None and t.device != dev:
            raise ValueError(f"{n} must be on {name}'s device {dev}, not {t.device}")
    return dev


def _layout(layout: str):
    """Positions of (batch, head, seq) in a 4-D shape."""
    if layout == "bhsd":
        return 0, 1, 2
    if layout == "bshd":
        return 0, 2, 1
    raise ValueError(f"unknown layout {layout!r}")


def _strides3(t: torch.Tensor, order) -> "ctypes.Array":
    st = t.stride()
    return (ctypes.c_int64 * 3)(st[order[0]], st[order[1]], st[order[2]])


def _ptr(t):
    return None if t is None else t.data_ptr()


class _on_device:
    """Makes a tensor's device current around a library call, and picks the
    stream: the caller's, or that device's current one."""

    __slots__ = ("_index", "_prev")

    def __init__(self, device: torch.device):
        self._index = device.index

    def __enter__(self):
        self._prev = torch.cuda.current_device()
        if self._prev != self._index:
            torch.cuda.set_device(self._index)

    def __exit__(self, *exc):
        if self._prev != self._index:
            torch.cuda.set_device(self._prev)


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
        order = _layout(layout)
        x, x_name = (q, "q") if q is not None else (k, "k")
        if x is None or (q is None) != (q_out is None) or (k is None) != (k_out is None):
            raise _capi.SfbError(_capi.SFB_ERR_INVALID, "q or k with its output expected")
        dev = _one_device(x, x_name, (q_out, "q_out"), (k, "k"), (k_out, "k_out"), (q_weight, "q_weight"),
                          (k_weight, "k_weight"), (cos, "cos"), (sin, "sin"), (positions, "positions"))
        dt = x.dtype
        if dt not in _FLOATS:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, f"dtype {dt}")
        a = _capi.NormRopeArgs()
        D = x.shape[-1]
        for t, o, w, n in ((q, q_out, q_weight, "q"), (k, k_out, k_weight, "k")):
            if t is None:
                continue
            if t.dim() != 4 or o.shape != t.shape or t.shape[3] != D or t.shape[0] != x.shape[0] \
                    or t.shape[order[2]] != x.shape[order[2]]:
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"inconsistent {n} shapes")
            if D > 1 and (t.stride(3) != 1 or o.stride(3) != 1):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{n}: head_dim must be contiguous")
            if t.dtype != dt or o.dtype != dt or (w is not None and w.dtype != dt):
                raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "q, k, outputs and weights share one dtype")
            if w is not None and (tuple(w.shape) != (D,) or not w.is_contiguous()):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{n}_weight must be contiguous [head_dim]")
        if q is not None:
            a.q, a.q_out, a.heads, a.q_weight = q.data_ptr(), q_out.data_ptr(), q.shape[order[1]], _ptr(q_weight)
            a.q_stride, a.q_out_stride = _strides3(q, order), _strides3(q_out, order)
        if k is not None:
            a.k, a.k_out, a.heads_kv, a.k_weight = k.data_ptr(), k_out.data_ptr(), k.shape[order[1]], _ptr(k_weight)
            a.k_stride, a.k_out_stride = _strides3(k, order), _strides3(k_out, order)
        a.batch, a.seq, a.head_dim, a.dtype = x.shape[0], x.shape[order[2]], D, _DTYPE_CODE[dt]
        if (cos is None) != (sin is None):
            raise _capi.SfbError(_capi.SFB_ERR_INVALID, "cos and sin come together")
        if cos is not None:
            if cos.dim() != 2 or cos.shape != sin.shape or not cos.is_contiguous() or not sin.is_contiguous():
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "cos / sin must be contiguous [positions, rot / 2]")
            if cos.dtype != torch.float32 or sin.dtype != torch.float32:
                raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "cos / sin must be fp32")
            a.cos_table, a.sin_table = cos.data_ptr(), sin.data_ptr()
            a.table_len, a.rotary_dim = cos.shape[0], 2 * cos.shape[1]
            if positions is not None:
                if positions.dtype != torch.int32:
                    raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "positions must be int32")
                if tuple(positions.shape) != (a.batch, a.seq) or (a.seq > 1 and positions.stride(1) != 1):
                    raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "positions must be [B, S], row-contiguous")
                a.positions, a.pos_stride_b = positions.data_ptr(), positions.stride(0)
        a.interleaved, a.norm, a.eps = 1 if interleaved else 0, 1 if norm else 0, float(eps)
        with _on_device(dev):
            _capi.check(self._lib.sfb_qk_norm_rope(ctypes.byref(a), _stream_handle(stream)), "qk_norm_rope")

    # The K/V cache held in 4 bits (quant4.KV4Cache)
    def _kv4_side(self, cache, c, t, name, order, dt):
        if t.dim() != 4 or t.shape[0] != c.batch or t.shape[order[1]] != c.heads_kv or t.shape[3] != c.head_dim:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{name} does not fit the cache")
        if t.stride(3) != 1:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{name}: head_dim must be contiguous")
        if t.dtype != dt or dt not in _FLOATS:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, f"{name} dtype {t.dtype}")
        return ctypes.byref(_strides3(t, order))

    def kv4_append(self, cache, K, V, start=0, lens=None, layout: str = "bhsd", stream=None) -> None:
        """Quantises K and V ([B, Hkv, S, D] or, layout "bshd", [B, S, Hkv, D])
        into the cache: token i of session b goes to slot start + i (start an
        int, or int32 [B]), only the first lens[b] tokens where lens (int32 [B])
        is given. With tensor starts, tokens outside the cache are not written
        and record SFB_ERR_RANGE (device_error)."""
        order = _layout(layout)
        c = cache.struct()
        start_t = start if isinstance(start, torch.Tensor) else None
        dev = _one_device(cache.k_codes, "cache", (K, "K"), (V, "V"), (start_t, "start"), (lens, "lens"))
        if K.shape != V.shape:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "K and V shapes differ")
        ks = self._kv4_side(cache, c, K, "K", order, K.dtype)
        vs = self._kv4_side(cache, c, V, "V", order, K.dtype)
        for t, n in ((start_t, "start"), (lens, "lens")):
            if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (c.batch,) or not t.is_contiguous()):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, f"{n} must be contiguous int32 [B]")
        with _on_device(dev):
            _capi.check(self._lib.sfb_kv4_append(
                ctypes.byref(c), K.data_ptr(), ks, V.data_ptr(), vs, _DTYPE_CODE[K.dtype], K.shape[order[2]],
                _ptr(start_t), 0 if start_t is not None else int(start), _ptr(lens), _stream_handle(stream)),
                "kv4_append")

    def kv4_read(self, cache, K=None, V=None, slot0: int = 0, layout: str = "bhsd", stream=None) -> None:
        """Writes the values of slots [slot0, slot0 + S) into K and V ([B, Hkv,
        S, D] or bshd; fp16 and fp32 exactly, bf16 rounded); either may be None."""
        order = _layout(layout)
        c = cache.struct()
        x = K if K is not None else V
        if x is None:
            raise _capi.SfbError(_capi.SFB_ERR_INVALID, "K or V expected")
        dev = _one_device(cache.k_codes, "cache", (K, "K"), (V, "V"))
        if K is not None and V is not None and K.shape != V.shape:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "K and V shapes differ")
        ks = None if K is None else self._kv4_side(cache, c, K, "K", order, x.dtype)
        vs = None if V is None else self._kv4_side(cache, c, V, "V", order, x.dtype)
        with _on_device(dev):
            _capi.check(self._lib.sfb_kv4_read(
                ctypes.byref(c), _ptr(K), ks, _ptr(V), vs, _DTYPE_CODE[x.dtype], int(slot0), x.shape[order[2]],
                _stream_handle(stream)), "kv4_read")

    def kv4_attention(self, Q, cache, out, seq_k: Optional[int] = None, kv_len=None, mask=None,
                      scale: float = 0.0, is_causal: bool = False, num_splits: int = 0,
                      layout: str = "bhsd", stream=None) -> None:
        """Attention of Q over the first seq_k slots of a KV4Cache (None: all of
        them). Q, out: bf16 or fp16 [B, H, Sq, D] (or bshd), H a multiple of the
        cache's heads. kv_len: int32 [B] valid slots; mask: bool/uint8 [B,
        seq_k] (True = keep); is_causal: the queries are the last Sq tokens of
        the valid slots. A query that sees no slot gives zeros."""
        order = _layout(layout)
        c = cache.struct()
        dev = _one_device(cache.k_codes, "cache", (Q, "Q"), (out, "out"), (kv_len, "kv_len"), (mask, "mask"))
        if Q.dtype not in _HALVES or out.dtype != Q.dtype:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "Q and out must be bf16 or fp16, alike")
        shape = Q.shape
        if len(shape) != 4 or out.shape != shape or shape[0] != c.batch or shape[3] != c.head_dim:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "Q and out must be 4-D and fit the cache")
        if Q.stride(3) != 1 or out.stride(3) != 1:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "head_dim must be contiguous")
        a = _capi.Kv4AttnArgs()
        a.cache = ctypes.addressof(c)
        a.q, a.out = Q.data_ptr(), out.data_ptr()
        a.q_stride, a.out_stride = _strides3(Q, order), _strides3(out, order)
        a.heads, a.seq_q = shape[order[1]], shape[order[2]]
        sk = a.seq_k = c.capacity if seq_k is None else int(seq_k)
        a.dtype, a.is_causal, a.num_splits, a.scale = _DTYPE_CODE[Q.dtype], 1 if is_causal else 0, num_splits, scale
        if kv_len is not None:
            if kv_len.dtype != torch.int32 or tuple(kv_len.shape) != (c.batch,) or not kv_len.is_contiguous():
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "kv_len must be contiguous int32 [B]")
            a.kv_len = kv_len.data_ptr()
        if mask is not None:
            if mask.dtype not in (torch.bool, torch.uint8):
                raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "mask must be bool or uint8")
            if tuple(mask.shape) != (c.batch, sk) or (sk > 1 and mask.stride(1) != 1):
                raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "mask must be [B, seq_k], row-contiguous")
            a.key_mask, a.key_mask_stride_b = mask.data_ptr(), mask.stride(0)
        with _on_device(dev):
            _capi.check(self._lib.sfb_kv4_attention(ctypes.byref(a), _stream_handle(stream)), "kv4_attention")

    # Linear layer with 4-bit weights and group scales (quant4.pack_w4)
    def w4a16_linear(self, x, w_q, w_scale, out, bias=None, residual=None, act: str = "none",
                     stream=None) -> None:
        """out[M, N] = act(x[M, K] · w^T + bias) + residual with w[n, k] =
        c[n, k] · w_scale[n, k / group]: w_q uint8 [N, K / 2] packed codes,
        w_scale [N, K / group] fp16, bf16 or fp32 (group 32, 64 or 128 follows
        from its shape). x and bias bf16 or fp16; out x's dtype or fp32."""
        dev = _one_device(x, "x", (w_q, "w_q"), (w_scale, "w_scale"), (out, "out"), (bias, "bias"),
                          (residual, "residual"))
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
        ld = lambda t, n: t.stride(0) if M > 1 else n
        with _on_device(dev):
            _capi.check(self._lib.sfb_w4a16_linear(
                x.data_ptr(), ld(x, (K + 7) // 8 * 8), _DTYPE_CODE[x.dtype], w_q.data_ptr(), w_scale.data_ptr(),
                _DTYPE_CODE[w_scale.dtype], K // groups, _ptr(bias), _ptr(residual),
                ld(residual, N) if residual is not None else 0, out.data_ptr(), ld(out, N), _DTYPE_CODE[out.dtype],
                M, N, K, _ACTS[act], _stream_handle(stream)), "w4a16_linear")

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
