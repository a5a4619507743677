"""Operator API of the HIP backend, mirroring the qppocr-kernels public functions
(qppocr-kernels/src/lib.rs:28-40): conv2d / conv2d_res, convtranspose2d,
sgemm / sgemm_res, matmul, softmax_last_dim, gelu_inplace, hardsigmoid,
sigmoid_tensor, relu_inplace, reduce_mean (last axis), resize_nearest, and the
CTC argmax of qppocr-core/src/pipeline/rec.rs; and the 4-bit operators of a
token-by-token decoder (quantize4, linear4, cache4_write, cache4_read,
attention_cache4), which the reference lacks.

Tensors are torch tensors on a ROCm device (torch is only the device-memory
plumbing here); every call goes through the C ABI of libqppocr_hip.so.  Calls
are synchronous with respect to torch's current stream: the stream is drained
before the library's own stream runs the kernel, and the library stream is
drained before returning.  The 4-bit operators do not wait: they are enqueued on
torch's current stream of the tensors' device, in its order, and may be captured
into a graph; they compute no gradients and refuse tensors that require one.
Errors raise QphError (no silent fallback).
"""
import ctypes
import functools
import threading

import torch

from . import _lib
from ._lib import (ACT_GELU, ACT_HARDSWISH, ACT_NONE, ACT_RELU, ACT_SIGMOID, Act, ConvEpilogue,
                   ConvParams, check, i64arr)

HS_ALPHA = 1.0 / 6.0   # HardSigmoid alpha of the hardswish pair (activation.rs:243-251)
HS_BETA = 0.5
GELU_C = (1.4142135, 1.0, 0.5)  # FusedGelu defaults (executor.rs:759-768)

_ctx = {}


def context(device=0):
    """The library context (DeviceContext analogue) of a HIP device."""
    if device not in _ctx:
        lib = _lib.load()
        p = ctypes.c_void_p()
        check(lib.qph_ctx_create(int(device), ctypes.byref(p)))
        _ctx[device] = p
    return _ctx[device]


def new_context(device=0):
    """A further context of a HIP device, with its own stream: sessions on
    different contexts run concurrently (e.g. det of one page while rec of
    the previous page).  Destroy it with close_context."""
    lib = _lib.load()
    p = ctypes.c_void_p()
    check(lib.qph_ctx_create(int(device), ctypes.byref(p)))
    return p


def close_context(ctx):
    check(_lib.load().qph_ctx_destroy(ctx))


def _dev(t):
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("qppocr_amd ops take device tensors")
    if t.dtype != torch.float32:
        raise ValueError("qppocr_amd ops take float32 tensors")
    if not t.is_contiguous():
        raise ValueError("qppocr_amd ops take contiguous tensors")
    return t.data_ptr()     # (the C signatures take the integer as it is)


class _Call:
    """Orders a library call after torch's pending work and waits for it."""

    __slots__ = ("device", "ctx")

    def __init__(self, device):
        self.device = device
        self.ctx = _ctx.get(device) or context(device)

    def __enter__(self):
        torch.cuda.current_stream(self.device).synchronize()
        return self.ctx

    def __exit__(self, kind, value, trace):
        if kind is None:
            check(_lib.load().qph_sync(self.ctx))
        return False


def act(kind=ACT_NONE):
    if kind == ACT_GELU:
        return Act(ACT_GELU, *GELU_C)
    if kind == ACT_HARDSWISH:
        return Act(ACT_HARDSWISH, HS_ALPHA, HS_BETA, 0.0)
    return Act(kind, 1.0, 0.0, 0.0)


@functools.lru_cache(maxsize=64)
def _act_ref(kind):
    """byref(act(kind)) of the library calls, which only read it."""
    return ctypes.byref(act(kind))


@functools.lru_cache(maxsize=256)
def _dims(shape):
    """The int64 array of a shape, which the library only reads.  (With the
    calls' other per-call objects gone, a 3x3 conv of one small map takes
    30.5 us with its two waits instead of 34.6.)"""
    return i64arr(shape)


def conv_params(sh=1, sw=1, ph=0, pw=0, peh=None, pew=None, group=1):
    return ConvParams(sh, sw, ph, pw, ph if peh is None else peh, pw if pew is None else pew,
                      1, 1, group)


def conv2d_out_shape(x_shape, w_shape, p):
    ys = (_lib.I64 * 4)()
    check(_lib.load().qph_conv2d_out_shape(i64arr(x_shape), i64arr(w_shape), ctypes.byref(p), ys))
    return tuple(int(v) for v in ys)


def conv2d(x, w, bias=None, params=None, act_kind=ACT_NONE, residual=None, out=None,
           res_up=0, y_ctotal=0, y_coff=0, y_up=1, trans_out=False):
    """conv2d_res (qppocr-kernels/src/conv.rs:183-211) with the fused epilogue
    options of qph_conv2d_ex."""
    params = conv_params() if params is None else params
    xs, ws = _dims(x.shape), _dims(w.shape)
    ys = _lib.I64_4()
    check(_lib.load().qph_conv2d_out_shape(xs, ws, ctypes.byref(params), ys))
    if out is None:
        n, m, oh, ow = ys
        if trans_out:
            out = torch.empty((n, oh * ow, m), device=x.device)
        elif y_ctotal or y_up != 1:
            raise ValueError("placed output needs an explicit out tensor")
        else:
            out = torch.empty((n, m, oh, ow), device=x.device)
    ep = None       # no epilogue options
    if residual is not None or res_up or y_ctotal or y_coff or y_up != 1 or trans_out:
        ep = ctypes.byref(ConvEpilogue(None if residual is None else residual.data_ptr(), res_up,
                                       y_ctotal, y_coff, y_up, int(bool(trans_out))))
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_conv2d_ex(ctx, _ptr(x), xs, _ptr(w), ws, _ptr(bias),
                                        ctypes.byref(params), _act_ref(act_kind), ep, _ptr(out)))
    return out


def convtranspose2d(x, w):
    """convtranspose2d, 2x2 s2 p0, no bias (qppocr-kernels/src/conv.rs:730-804)."""
    n, c, h, wd = x.shape
    out = torch.empty((n, w.shape[1], 2 * h, 2 * wd), device=x.device)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_convtranspose2d(ctx, _ptr(x), i64arr(x.shape), _ptr(w),
                                              i64arr(w.shape), 2, 2, 0, 0, _ptr(out), None))
    return out


def convt_pair_sigmoid(x, w1, w2):
    n, c, h, wd = x.shape
    out = torch.empty((n, 1, 4 * h, 4 * wd), device=x.device)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_convt2x2_pair_sigmoid(ctx, _ptr(x), i64arr(x.shape), _ptr(w1),
                                                    i64arr(w1.shape), _ptr(w2), i64arr(w2.shape),
                                                    _ptr(out)))
    return out


def sgemm(a, b, m, n, k, bias=None, act_kind=ACT_NONE, residual=None, serial=False):
    """sgemm / sgemm_res (qppocr-kernels/src/gemm.rs:37-70): C[M,N] = A[M,K] B[K,N]."""
    c = torch.empty((m, n), device=a.device)
    ac = act(act_kind)
    with _Call(_dev(a)) as ctx:
        check(_lib.load().qph_sgemm(ctx, _ptr(a), _ptr(b), _ptr(c), m, n, k, n, _ptr(bias),
                                    ctypes.byref(ac), _ptr(residual), int(bool(serial))))
    return c


def matmul(a, b):
    """MatMul (qppocr-kernels/src/shape.rs:568-698): a [..., M, K] x b [K, N] or [..., K, N]."""
    m, k = a.shape[-2:]
    n = b.shape[-1]
    batch = 1
    for d in a.shape[:-2]:
        batch *= d
    shared = b.dim() == 2
    out = torch.empty(tuple(a.shape[:-2]) + (m, n), device=a.device)
    with _Call(_dev(a)) as ctx:
        check(_lib.load().qph_matmul(ctx, _ptr(a), _ptr(b), _ptr(out), batch, m, k, n,
                                     int(shared)))
    return out


def linear(x, w, bias=None, act_kind=ACT_NONE, residual=None):
    """MatMul x[..., K] . w[K, N] -> Add(bias) -> act -> Add(residual)."""
    k, n = w.shape
    rows = x.numel() // k
    y = torch.empty(tuple(x.shape[:-1]) + (n,), device=x.device)
    ac = act(act_kind)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_linear(ctx, _ptr(x), _ptr(w), _ptr(bias), rows, k, n,
                                     ctypes.byref(ac), _ptr(residual), _ptr(y)))
    return y


def layernorm(x, gamma, beta, eps):
    cols = x.shape[-1]
    y = torch.empty_like(x)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_layernorm(ctx, _ptr(x), _ptr(gamma), _ptr(beta), float(eps),
                                        x.numel() // cols, cols, _ptr(y)))
    return y


def softmax_last_dim(t, inner):
    """In place (qppocr-kernels/src/activation.rs:321-334)."""
    with _Call(_dev(t)) as ctx:
        check(_lib.load().qph_softmax_last_dim(ctx, _ptr(t), t.numel() // inner, inner))
    return t


def softmax_argmax(logits, probs=True):
    """Row softmax + argmax pairs; probs=False exports the pairs only (the
    rec_argmax_pairs exit, qppocr-core/src/device.rs:160-165) and returns
    (None, pairs)."""
    cols = logits.shape[-1]
    rows = logits.numel() // cols
    pr = torch.empty_like(logits) if probs else None
    pairs = torch.empty(tuple(logits.shape[:-1]) + (2,), device=logits.device)
    with _Call(_dev(logits)) as ctx:
        check(_lib.load().qph_softmax_argmax(ctx, _ptr(logits), rows, cols,
                                             _ptr(pr) if probs else None, _ptr(pairs)))
    return pr, pairs


def linear_softmax_argmax(x, w, bias=None):
    """The fused rec head: MatMul + Add(bias) + Softmax + argmax pairs in one
    GEMM (logits never stored).  x [..., K], w [K, N]; returns pairs
    [..., 2].  Values agree with the unfused path to float rounding."""
    k, n = w.shape
    rows = x.numel() // k
    pairs = torch.empty(tuple(x.shape[:-1]) + (2,), device=x.device)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_linear_softmax_argmax(ctx, _ptr(x), _ptr(w), _ptr(bias), rows, k, n,
                                                    _ptr(pairs)))
    return pairs


def ctc_argmax(probs, t_valid=None):
    """(value, index-bits) per step; probs [B, T, C] (rec.rs:34-90)."""
    b, t, c = probs.shape
    pairs = torch.empty((b, t, 2), device=probs.device)
    tv = None
    if t_valid is not None:
        arr = (ctypes.c_int32 * b)(*[int(v) for v in t_valid])
        tv = ctypes.cast(arr, ctypes.c_void_p)
    with _Call(_dev(probs)) as ctx:
        check(_lib.load().qph_ctc_argmax(ctx, _ptr(probs), b, t, c, tv, _ptr(pairs)))
    return pairs


def attention(qkv, heads, dh, scale):
    b, t = qkv.shape[0], qkv.shape[1]
    out = torch.empty((b, t, heads * dh), device=qkv.device)
    with _Call(_dev(qkv)) as ctx:
        check(_lib.load().qph_attention(ctx, _ptr(qkv), b, t, heads, dh, float(scale), _ptr(out)))
    return out


def activation(x, act_kind):
    y = torch.empty_like(x)
    ac = act(act_kind)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_activation(ctx, _ptr(x), _ptr(y), x.numel(), ctypes.byref(ac)))
    return y


def relu_inplace(t):
    ac = act(ACT_RELU)
    with _Call(_dev(t)) as ctx:
        check(_lib.load().qph_activation(ctx, _ptr(t), _ptr(t), t.numel(), ctypes.byref(ac)))
    return t


def gelu_inplace(t, c1=GELU_C[0], c2=GELU_C[1], c3=GELU_C[2]):
    ac = Act(ACT_GELU, c1, c2, c3)
    with _Call(_dev(t)) as ctx:
        check(_lib.load().qph_activation(ctx, _ptr(t), _ptr(t), t.numel(), ctypes.byref(ac)))
    return t


def sigmoid_tensor(x):
    return activation(x, ACT_SIGMOID)


def hardsigmoid(x, alpha=HS_ALPHA, beta=HS_BETA):
    y = torch.empty_like(x)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_hardsigmoid(ctx, _ptr(x), _ptr(y), x.numel(), float(alpha),
                                          float(beta)))
    return y


def resize_nearest(x, oh, ow):
    n, c, h, w = x.shape
    y = torch.empty((n, c, oh, ow), device=x.device)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_resize_nearest(ctx, _ptr(x), n * c, h, w, oh, ow, _ptr(y)))
    return y


def binary_inplace(a, b, op, bmode):
    cols = a.shape[-1]
    with _Call(_dev(a)) as ctx:
        check(_lib.load().qph_binary_inplace(ctx, _ptr(a), _ptr(b), a.numel() // cols, cols, op,
                                             bmode))
    return a


def reduce_mean_last(x):
    cols = x.shape[-1]
    out = torch.empty(x.shape[:-1], device=x.device)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_reduce_mean_last(ctx, _ptr(x), x.numel() // cols, cols, _ptr(out)))
    return out


def pairs_ids(pairs):
    """Index half of a pairs tensor as int64 (f32 bits -> u32)."""
    return pairs[..., 1].contiguous().view(torch.int32).to(torch.int64) & 0xFFFFFFFF


# ------------------------------------------- pooling / SE gate / resize / layout

def _ptr_any(t):
    """Device pointer of a contiguous tensor of any dtype (u8 images)."""
    if not t.is_cuda or not t.is_contiguous():
        raise ValueError("qppocr_amd ops take contiguous device tensors")
    return t.data_ptr()


def global_avg_pool(x):
    """global_avg_pool (qppocr-kernels/src/pool2d.rs:10-29): [N,C,H,W] -> [N,C,1,1]."""
    n, c, h, w = x.shape
    out = torch.empty((n, c, 1, 1), device=x.device)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_global_avg_pool(ctx, _ptr(x), n, c, h * w, _ptr(out)))
    return out


def mul_add_scale(feature, gate, residual):
    """mul_add_scale (elementwise.rs:134-179): feature * gate[c] + residual."""
    n, c, h, w = feature.shape
    out = torch.empty_like(feature)
    with _Call(_dev(feature)) as ctx:
        check(_lib.load().qph_mul_add_scale(ctx, _ptr(feature), _ptr(gate), _ptr(residual), n, c,
                                            h * w, _ptr(out)))
    return out


def pool2d(x, k, stride, pad=(0, 0, 0, 0), max_pool=True):
    """pool2d (pool2d.rs:51-236); pad = (ph, pw, peh, pew)."""
    n, c, h, w = x.shape
    kh, kw = k
    sh, sw = stride
    ph, pw, peh, pew = pad
    oh = max(h + ph + peh - kh, 0) // sh + 1
    ow = max(w + pw + pew - kw, 0) // sw + 1
    y = torch.empty((n, c, oh, ow), device=x.device)
    ys = (_lib.I64 * 4)()
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_pool2d(ctx, _ptr(x), i64arr(x.shape), kh, kw, sh, sw, ph, pw, peh,
                                     pew, int(bool(max_pool)), _ptr(y), ys))
    assert tuple(ys) == (n, c, oh, ow)
    return y


def resize_bilinear(x, oh, ow, align_corners=False):
    """resize_bilinear (resize.rs:60-142) over the last two axes."""
    h, w = x.shape[-2:]
    nc = x.numel() // (h * w)
    y = torch.empty(tuple(x.shape[:-2]) + (oh, ow), device=x.device)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_resize_bilinear(ctx, _ptr(x), nc, h, w, oh, ow,
                                              int(bool(align_corners)), _ptr(y)))
    return y


def transpose(x, perm):
    """Rank-4 Transpose."""
    y = torch.empty(tuple(x.shape[p] for p in perm), device=x.device)
    pm = (_lib.I32 * 4)(*perm)
    with _Call(_dev(x)) as ctx:
        check(_lib.load().qph_transpose(ctx, _ptr(x), i64arr(x.shape), pm, _ptr(y)))
    return y


def det_normalize_u8(rgb):
    """det input (engine.rs:959-982): u8 [H, W, 3] -> f32 [1, 3, H, W]."""
    h, w = rgb.shape[:2]
    out = torch.empty((1, 3, h, w), device=rgb.device)
    with _Call(_dev(rgb)) as ctx:
        check(_lib.load().qph_det_normalize_u8(ctx, _ptr_any(rgb), h, w, _ptr(out)))
    return out


def resize_bilinear_rgb_u8(src, dw, dh):
    """resize_bilinear_rgb_u8 (resize.rs:153-209): u8 [sh, sw, 3] -> [dh, dw, 3]."""
    sh, sw = src.shape[:2]
    dst = torch.empty((dh, dw, 3), dtype=torch.uint8, device=src.device)
    with _Call(_dev(src)) as ctx:
        check(_lib.load().qph_resize_bilinear_rgb_u8(ctx, _ptr_any(src), sw, sh, _ptr_any(dst),
                                                     dw, dh))
    return dst


def pack_crop(crop, img_h, img_w, pad_only=False, out=None):
    """pack_crop (crop.rs:153-190): u8 crop [ch, cw, 3] -> f32 [3, img_h, img_w]."""
    ch, cw = crop.shape[:2]
    if out is None:
        out = torch.empty((3, img_h, img_w), device=crop.device)
    with _Call(_dev(crop)) as ctx:
        check(_lib.load().qph_pack_crop(ctx, _ptr_any(crop), ch, cw, img_h, img_w,
                                        int(bool(pad_only)), _ptr(out)))
    return out


def pack_crops(crops, img_h, img_w, pad_only=None, out=None):
    """A rec batch in one launch per 64 lines (engine.rs:1413-1431 packs it
    line by line): u8 crops [ch, cw, 3] -> f32 [n, 3, img_h, img_w], line i
    as pack_crop(crops[i], img_h, img_w, pad_only[i])."""
    n = len(crops)
    for c in crops:
        if c.dtype != torch.uint8 or c.dim() != 3 or c.shape[2] != 3:
            raise ValueError("pack_crops takes u8 [ch, cw, 3] crops")
    if pad_only is None:
        pad_only = [False] * n
    if out is None:
        out = torch.empty((n, 3, img_h, img_w), device=crops[0].device)
    ptrs = (ctypes.c_void_p * n)(*[_ptr_any(c) for c in crops])
    ch = (_lib.I64 * n)(*[c.shape[0] for c in crops])
    cw = (_lib.I64 * n)(*[c.shape[1] for c in crops])
    po = (_lib.I32 * n)(*[int(bool(p)) for p in pad_only])
    with _Call(_dev(crops[0])) as ctx:
        check(_lib.load().qph_pack_crops(ctx, n, ptrs, ch, cw, po, img_h, img_w, _ptr(out)))
    return out


def db_mask(pred, thresh, dilate=True):
    """DB threshold + 2x2 dilation (geometry.rs:287-301, resize.rs:219-247)."""
    h, w = pred.shape[-2:]
    out = torch.empty((h, w), dtype=torch.uint8, device=pred.device)
    with _Call(_dev(pred)) as ctx:
        check(_lib.load().qph_db_mask(ctx, _ptr(pred), h, w, float(thresh), int(bool(dilate)),
                                      _ptr_any(out)))
    return out


# ------------------------------------------- 4-bit weights and caches

_DTYPES = {torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
_HEAD_DIMS = (32, 64, 96, 128, 192, 256)
_queued = {}
_queue_lock = threading.Lock()
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(
    torch._C, "_cuda_getCurrentRawStream") else (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _enqueue(device, fn, *args):
    """fn(context, *args) on torch's current stream of a device, without waiting.
    The device's context for such calls takes the stream of each call under a
    lock, since calls of several threads share it.  (A decoder's step is some
    hundred of these calls, whose host side decides where kernels are short:
    with the stream's handle taken as it is and no objects made that a call can
    do without, linear4 takes 7 us of it instead of 10.)"""
    stream = _raw_stream(device) or _lib.STREAM_DEFAULT
    with _queue_lock:
        entry = _queued.get(device)
        if entry is None:
            with torch.cuda.device(device):      # (which puts the caller's device back)
                entry = _queued[device] = [new_context(device), None]
        if entry[1] != stream:
            check(_lib.load().qph_ctx_set_stream(entry[0], stream))
            entry[1] = stream
        rc = fn(entry[0], *args)
    if rc:
        check(rc)


def _dtype4(t, what):
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"{what}: {t.dtype} is not float32, float16 or bfloat16")
    return d


def _on(what, device, name, t):
    """Refuses a tensor that does not lie on the GPU `device`."""
    if t.device != device or not t.is_cuda:
        raise ValueError(f"{what}: {name} is on {t.device}, not on "
                         f"{device if device.type == 'cuda' else 'a GPU'}")


def _plain(what, name, t, dtype, shape, device):
    """Refuses a tensor that is not contiguous, of the dtype, of the shape and
    on the device."""
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} tensor of shape "
                         f"{tuple(shape)}, not {t.dtype} {tuple(t.shape)}")
    _on(what, device, name, t)


def _no_grad(what, *tensors):
    """Refuses tensors whose gradient the call would drop without a word."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what}: no gradient is computed, but a tensor requires one (detach "
                                 "it, or call under torch.no_grad())")


class _Fixed:
    """What its __init__ sets stays: the calls use addresses taken then.  A copy of
    any kind is made by __init__ again, from what _parts names."""
    _names = frozenset()
    _parts = ()

    def __setattr__(self, name, value):
        if name in self._names:
            raise AttributeError(f"{type(self).__name__}.{name} is fixed; make another one")
        self.__dict__[name] = value

    def __delattr__(self, name):
        if name in self._names:
            raise AttributeError(f"{type(self).__name__}.{name} is fixed")
        object.__delattr__(self, name)

    def __reduce__(self):
        return type(self), tuple(getattr(self, name) for name in self._parts)

    def _fix(self, **names):
        self.__dict__.update(names, _names=frozenset(names) | {"_names"})


class Weight4(_Fixed):
    """A linear's weight [n, k] in 4 bits (the format: include/qppocr_hip.h):
    codes uint8 [n, kp / 2] and scales uint8 [n, kp / 32], kp = k rounded up to
    128, elements past k zero.  quantize4 makes one; a caller may bring the
    two tensors, whose memory it is then made of (their contents may change, the
    tensors may not be replaced or moved)."""
    _parts = "codes", "scales", "k"

    def __init__(self, codes, scales, k):
        if codes.dim() != 2 or k <= 0:
            raise ValueError("Weight4: codes [n, kp / 2] of k > 0 columns")
        n, kp = codes.shape[0], (k + 127) // 128 * 128
        _plain("Weight4", "codes", codes, torch.uint8, (n, kp // 2), codes.device)
        _plain("Weight4", "scales", scales, torch.uint8, (n, kp // 32), codes.device)
        if codes.data_ptr() % 16 or scales.data_ptr() % 4:
            raise ValueError("Weight4: codes are not 16-byte or scales not 4-byte aligned")
        self._fix(codes=codes, scales=scales, n=n, k=int(k), device=codes.device,
                  _index=codes.device.index, _ptrs=(codes.data_ptr(), scales.data_ptr()))


def quantize4(w):
    """The weight w [K, N] that linear takes (any strides; float32, float16 or
    bfloat16) as a Weight4."""
    if w.dim() != 2:
        raise ValueError("quantize4: a weight [K, N]")
    k, n = w.shape
    if not k or not n:
        raise ValueError("quantize4: empty weight")
    d = _dtype4(w, "quantize4")
    _on("quantize4", w.device, "w", w)
    kp = (k + 127) // 128 * 128
    codes = torch.empty((n, kp // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((n, kp // 32), dtype=torch.uint8, device=w.device)
    _enqueue(w.device.index, _lib.load().qph_quantize4, w.data_ptr(), d, n, k, w.stride(1),
             w.stride(0), codes.data_ptr(), scales.data_ptr())
    return Weight4(codes, scales, k)


def linear4(x, w, bias=None, act_kind=ACT_NONE, residual=None):
    """linear over a Weight4: act(x [..., K] . w + bias) + residual, in x's type
    (float32, float16, bfloat16).  x's rows may lie apart (a slice of a packed
    projection); bias and residual are contiguous and of x's type."""
    d = _dtype4(x, "linear4")
    k, n = w.k, w.n
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"linear4: x {tuple(x.shape)} against a weight of {k} inputs")
    _on("linear4", w.device, "x", x)
    _no_grad("linear4", x, bias, residual)
    if x.dim() == 2:
        rows, x2 = x.shape[0], x
        y = x.new_empty((rows, n))
    else:
        rows = x.numel() // k
        x2 = x.reshape(rows, k)
        y = x.new_empty(tuple(x.shape[:-1]) + (n,))
    if x2.stride(1) != 1 and k > 1:
        x2 = x2.contiguous()
    b = r = None
    if bias is not None:
        _plain("linear4", "bias", bias, x.dtype, (n,), w.device)
        b = bias.data_ptr()
    if residual is not None:
        _plain("linear4", "residual", residual, x.dtype, y.shape, w.device)
        r = residual.data_ptr()
    codes, scales = w._ptrs
    _enqueue(w._index, _lib.load().qph_linear4, x2.data_ptr(), d, x2.stride(0), codes, scales, b,
             rows, k, n, _act_ref(act_kind), r, y.data_ptr())
    return y


class Cache4(_Fixed):
    """A paged cache of keys and values in 4 bits (the format and layout:
    include/qppocr_hip.h): codes uint8 [pages, heads, page size, dh / 2] and
    scales uint8 [pages, heads, page size, dh / 32] of either.  cache4 makes
    an empty one; a caller may bring the four tensors, as for a Weight4."""
    _parts = "k_codes", "k_scales", "v_codes", "v_scales"

    def __init__(self, k_codes, k_scales, v_codes, v_scales):
        if k_codes.dim() != 4:
            raise ValueError("Cache4: codes [pages, heads, page size, dh / 2]")
        pages, heads, page, half = k_codes.shape
        if 2 * half not in _HEAD_DIMS:
            raise ValueError(f"Cache4: head dimension {2 * half} is not one of {_HEAD_DIMS}")
        if page < 16 or page > 32768 or page & (page - 1):
            raise ValueError(f"Cache4: page size {page} is no power of two from 16 to 32768")
        if not pages or not heads:
            raise ValueError("Cache4: empty cache")
        for name, t, last in (("k_codes", k_codes, half), ("v_codes", v_codes, half),
                              ("k_scales", k_scales, half // 16),
                              ("v_scales", v_scales, half // 16)):
            _plain("Cache4", name, t, torch.uint8, (pages, heads, page, last), k_codes.device)
        c = _lib.Cache4(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
                        v_scales.data_ptr(), pages, page, heads, 2 * half)
        self._fix(k_codes=k_codes, k_scales=k_scales, v_codes=v_codes, v_scales=v_scales,
                  pages=pages, heads=heads, page_size=page, dh=2 * half, device=k_codes.device,
                  _index=k_codes.device.index, _c=c, _ref=ctypes.byref(c))


def cache4(pages, page_size, heads, dh, device="cuda"):
    """A Cache4 of zeros."""
    if dh not in _HEAD_DIMS:
        raise ValueError(f"cache4: head dimension {dh} is not one of {_HEAD_DIMS}")
    def make(last, fill):
        return torch.full((pages, heads, page_size, last), fill, dtype=torch.uint8, device=device)
    return Cache4(make(dh // 2, 0), make(dh // 32, 27), make(dh // 2, 0), make(dh // 32, 27))


def _rows4(what, name, t, cache, tokens, heads):
    """Refuses a tensor that is not [tokens, heads, dh] with neighbouring elements
    of a head, on the cache's device; its strides of a token and a head."""
    strides = t.stride()
    if t.shape != (tokens, heads, cache.dh) or (strides[2] != 1 and t.numel()):
        raise ValueError(f"{what}: {name} must be [{tokens}, {heads}, {cache.dh}] with neighbouring "
                         f"elements of a head, not {tuple(t.shape)} of strides {strides}")
    _on(what, cache.device, name, t)
    return strides[:2]


def _reach(dims):
    """The last element's offset of dims (stride, size), or None where two elements may
    have one place (each stride must pass all that the smaller ones reach)."""
    last = 0
    for stride, size in sorted(dims):
        if size > 1:
            if stride <= last:
                return None
            last += stride * (size - 1)
    return last


def _writable(what, name, t, other=None, other_name=None):
    """Refuses an output whose elements share memory, among themselves or with `other`."""
    if not t.numel():
        return
    dims = list(zip(t.stride(), t.shape))
    reach = _reach(dims)
    if reach is None:
        raise ValueError(f"{what}: {name} of strides {t.stride()} overlaps itself")
    if other is None or not other.numel():
        return
    # apart from end to end, or of one layout whose two copies interleave
    size, delta = t.element_size(), other.data_ptr() - t.data_ptr()
    length = other.element_size() * (1 + sum(st * (n - 1) for st, n in zip(other.stride(), other.shape)))
    if delta >= (reach + 1) * size or -delta >= length:
        return
    if delta % size or (t.stride(), t.shape, t.dtype) != (other.stride(), other.shape, other.dtype) or \
            _reach(dims + [(abs(delta) // size, 2)]) is None:
        raise ValueError(f"{what}: {name} and {other_name} share memory")


def cache4_write(cache, k, v, slots):
    """Quantises tokens' keys and values [tokens, heads, dh] (tokens and heads
    of any strides) into their slots, int64 [tokens]: page * page_size + place.
    A slot outside the pool (-1 for a padded token) is skipped; the others must
    differ."""
    d = _dtype4(k, "cache4_write")
    if k.dim() != 3 or v.dtype != k.dtype:
        raise ValueError("cache4_write: k and v [tokens, heads, dh] of one type")
    n = k.shape[0]
    ks = _rows4("cache4_write", "k", k, cache, n, cache.heads)
    vs = _rows4("cache4_write", "v", v, cache, n, cache.heads)
    _plain("cache4_write", "slots", slots, torch.int64, (n,), cache.device)
    _no_grad("cache4_write", k, v)
    _enqueue(cache._index, _lib.load().qph_cache4_write, cache._ref, k.data_ptr(), v.data_ptr(), d,
             n, _dims(ks), _dims(vs), slots.data_ptr())


def cache4_read(cache, slots, dtype=torch.float32, out=None):
    """The tokens of slots, int64 [tokens], as (k, v) [tokens, heads, dh] of
    dtype; zeros for a slot outside the pool.  out: such a pair to write into, whose
    type counts instead (tokens and heads of any strides, no two elements in one
    place)."""
    if slots.dim() != 1:
        raise ValueError("cache4_read: slots [tokens]")
    n = slots.shape[0]
    if out is None:
        shape = (n, cache.heads, cache.dh)
        k = torch.empty(shape, dtype=dtype, device=cache.device)
        v = torch.empty_like(k)
    else:
        k, v = out
    d = _dtype4(k, "cache4_read")
    if v.dtype != k.dtype:
        raise ValueError("cache4_read: k and v of one type")
    ks = _rows4("cache4_read", "k", k, cache, n, cache.heads)
    vs = _rows4("cache4_read", "v", v, cache, n, cache.heads)
    if out is not None:
        _no_grad("cache4_read", k, v)
        _writable("cache4_read", "k", k, v, "v")
        _writable("cache4_read", "v", v)
    _plain("cache4_read", "slots", slots, torch.int64, (n,), cache.device)
    _enqueue(cache._index, _lib.load().qph_cache4_read, cache._ref, k.data_ptr(), v.data_ptr(), d, n,
             _dims(ks), _dims(vs), slots.data_ptr())
    return k, v


@functools.lru_cache(maxsize=1024)
def _workspace4(pages, page, heads, dh, *sizes):
    """qph_attention_cache4_workspace, which sees the sizes alone."""
    c = _lib.Cache4(256, 256, 256, 256, pages, page, heads, dh)
    a = _lib.Attn4()
    (a.dtype, a.heads, a.tokens, a.batch, a.max_pages, a.max_new, a.max_len, a.causal, a.window,
     a.starts) = sizes
    a.scale = 1.0
    size = ctypes.c_size_t()
    check(_lib.load().qph_attention_cache4_workspace(ctypes.byref(c), ctypes.byref(a),
                                                     ctypes.byref(size)))
    return size.value


def attention_cache4(q, cache, page_table, lens, scale, starts=None, max_new=None, max_len=None,
                     causal=True, window=0, lse=False, out=None):
    """Attention of new tokens q [tokens, heads, dh] over a Cache4 that holds
    their keys and values already.

    page_table int32 [batch, pages] and lens int32 [batch] name each sequence's
    pages and cached tokens, its new ones the last of them.  starts int32
    [batch + 1]: sequence b's new tokens are q[starts[b]:starts[b + 1]], at most
    max_new (needed then); without starts every sequence has tokens / batch.
    max_len bounds lens (default: all of the table's pages).  causal hides later
    keys, window > 0 all but the last `window` up to a token's own.  out may be q
    itself, and shares no memory with it otherwise, nor its elements any.  A
    row that sees no key is zero; rows of no sequence keep what out holds.
    Returns out, or (out, lse) with the sums' logarithms, float32 [tokens,
    heads] (-infinity where no key is seen; a new tensor's rows of no sequence
    are undefined)."""
    what = "attention_cache4"
    d = _dtype4(q, what)
    if q.dim() != 3:
        raise ValueError(f"{what}: q [tokens, heads, dh]")
    tokens, heads, dh = q.shape
    dev = cache.device
    qs = _rows4(what, "q", q, cache, tokens, heads)
    _no_grad(what, q, out)
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or (
            page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError(f"{what}: page_table int32 [batch, pages], rows contiguous")
    _on(what, dev, "page_table", page_table)
    batch, pages = page_table.shape
    _plain(what, "lens", lens, torch.int32, (batch,), dev)
    at = None
    if starts is not None:
        _plain(what, "starts", starts, torch.int32, (batch + 1,), dev)
        if max_new is None:
            raise ValueError(f"{what}: starts need max_new")
        at = starts.data_ptr()
    elif batch and tokens % batch:
        raise ValueError(f"{what}: {tokens} tokens for {batch} sequences need starts")
    else:
        each = tokens // batch if batch else 0
        if max_new is not None and max_new != each and batch:
            raise ValueError(f"{what}: max_new {max_new} without starts, where every sequence "
                             f"has {each}")
        max_new = each
    if max_len is None:
        max_len = min(pages * cache.page_size, 0x7fffff00)
    own = out is None
    if own:
        out = q.new_empty((tokens, heads, dh))
    elif out.dtype != q.dtype:
        raise ValueError(f"{what}: out is {out.dtype}, q {q.dtype}")
    os = _rows4(what, "out", out, cache, tokens, heads)
    if not own:
        same = out.data_ptr() == q.data_ptr() and os == qs
        _writable(what, "out", out, None if same else q, "q")
    sums = torch.empty((tokens, heads), dtype=torch.float32, device=dev) if lse else None
    max_new, max_len, window = (min(int(n), 0x7fffffff) for n in (max_new, max_len, window))
    if min(max_new, max_len, window) < 0:
        raise ValueError(f"{what}: negative max_new, max_len or window")
    causal = int(bool(causal))
    size = _workspace4(cache.pages, cache.page_size, cache.heads, dh, d, heads, tokens, batch, pages,
                       max_new, max_len, causal, window, None if at is None else 256)
    work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    a = _lib.Attn4(q.data_ptr(), out.data_ptr(), None if sums is None else sums.data_ptr(), *qs, *os,
                   tokens, batch, page_table.data_ptr(), page_table.stride(0), pages,
                   lens.data_ptr(), at, d, heads, max_new, max_len, scale, causal, window,
                   None if work is None else work.data_ptr(), size)
    _enqueue(cache._index, _lib.load().qph_attention_cache4, cache._ref, ctypes.byref(a))
    return (out, sums) if lse else out
