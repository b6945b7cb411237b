"""Python mirror of the B200 PP-DocLayoutV3 C ABIs (ctypes).

Two surfaces, both thin bindings of lib/libppdl_b200.so:

* the model API of include/ppdoclayout.h (ppdl_init / ppdl_infer /
  ppdl_infer_batch / ppdl_dump_raw / ppdl_free) — the reference's public C
  ABI (include/ppdoclayout.h:29-63 of caojiachen1/ppdoclayout-ggml) plus the
  additive batch and device-output entry points;
* the operator API of include/ppdl_ops.h (ppdl_op_launch) — the reference's
  tagged ggml custom-op hooks (patches/ggml-ppdl.patch:612-930), driven here
  with torch CUDA tensors as the device memory — and the transformer-block
  operators beside it (layernorm, layernorm_backward, quantize_rows,
  linear_i8, rotary).

There is no CPU fallback: importing this module never loads anything else,
and every call fails loudly when the CUDA library is missing.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libppdl_b200.so")

PPDL_MAGIC = 0x5050444C
OP_MASKBOX, OP_MSDEF, OP_CONV, OP_CONVDIRECT, OP_BIASACT, OP_COPY = 1, 2, 3, 4, 5, 6
OP_WG_INPUT, OP_WG_OUTPUT, OP_WG_MADD = 7, 8, 9
OP_WG4_INPUT, OP_WG4_OUTPUT, OP_WG4_MADD, OP_TOPK = 10, 11, 12, 13

PPDL_OK, PPDL_ERR_UNSUPPORTED, PPDL_ERR_SHAPE, PPDL_ERR_CUDA = 0, 1, 2, 3

IMG_SIZE, NUM_DETS, DET_FIELDS, MASK_HW = 800, 300, 7, 200
BACKEND_CPU, BACKEND_CUDA = 0, 1


class Tensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("ne", C.c_int64 * 4)]


class OpDesc(C.Structure):
    _fields_ = [("dst", Tensor), ("src", Tensor * 4), ("op_params", C.c_int32 * 16)]


class Result(C.Structure):
    _fields_ = [("dets", C.POINTER(C.c_float)), ("num_dets", C.c_int32),
                ("masks", C.POINTER(C.c_int32)), ("infer_ms", C.c_double)]


class ResultBits(C.Structure):
    """ppdl_result_bits: masks packed 1 bit per pixel (300 x 1250 words)."""
    _fields_ = [("dets", C.POINTER(C.c_float)), ("num_dets", C.c_int32),
                ("mask_bits", C.POINTER(C.c_uint32)), ("infer_ms", C.c_double)]


MASK_WORDS = 1250


def unpack_mask_bits(bits):
    """[..., 1250] uint32 words -> [..., 200, 200] uint8 masks (bit p & 31 of
    word p >> 5 is pixel p), the numpy form of ppdl_expand_mask_bits."""
    import numpy as np
    b = np.ascontiguousarray(bits, dtype=np.uint32)
    u8 = b.view(np.uint8).reshape(b.shape[:-1] + (MASK_WORDS * 4,))
    px = np.unpackbits(u8, axis=-1, bitorder="little")
    return px.reshape(b.shape[:-1] + (MASK_HW, MASK_HW))


_lib = None


def lib() -> C.CDLL:
    """The loaded product library; raises when it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `make -C {HERE}` "
                "(there is no CPU fallback)")
        L = C.CDLL(LIB_PATH)
        L.ppdl_op_launch.argtypes = [C.POINTER(OpDesc), C.c_void_p]
        L.ppdl_op_launch.restype = C.c_int
        L.ppdl_op_supported.argtypes = [C.POINTER(OpDesc)]
        L.ppdl_op_supported.restype = C.c_int
        L.ppdl_op_last_error.restype = C.c_char_p
        _declare_block_ops(L)
        if hasattr(L, "ppdl_init"):
            L.ppdl_init.argtypes = [C.c_char_p, C.c_int]
            L.ppdl_init.restype = C.c_void_p
            L.ppdl_init_ex.argtypes = [C.c_char_p, C.c_int, C.c_int]
            L.ppdl_init_ex.restype = C.c_void_p
            L.ppdl_infer.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.POINTER(Result)]
            L.ppdl_infer.restype = C.c_int
            L.ppdl_free.argtypes = [C.c_void_p]
            L.ppdl_free.restype = None
            L.ppdl_dump_raw.argtypes = [C.c_void_p, C.c_char_p]
            L.ppdl_dump_raw.restype = C.c_int
            L.ppdl_dump.argtypes = [C.c_void_p, C.c_char_p]
            L.ppdl_dump.restype = C.c_int
        _lib = L
    return _lib


def _tensor(t, ne=None) -> Tensor:
    """ppdl_tensor for a contiguous torch CUDA tensor; ne in ggml order
    (fastest first), defaulting to the reversed torch shape."""
    if t is None:
        return Tensor(None, (C.c_int64 * 4)(1, 1, 1, 1))
    assert t.is_cuda and t.is_contiguous(), "operator ABI takes contiguous CUDA tensors"
    if ne is None:
        ne = list(reversed(t.shape))
    ne = list(ne) + [1] * (4 - len(ne))
    return Tensor(C.c_void_p(t.data_ptr()), (C.c_int64 * 4)(*ne))


def make_desc(op_id, dst, srcs=(), params=(), dst_ne=None, src_ne=()) -> OpDesc:
    d = OpDesc()
    d.dst = _tensor(dst, dst_ne)
    for i in range(4):
        s = srcs[i] if i < len(srcs) else None
        ne = src_ne[i] if i < len(src_ne) else None
        d.src[i] = _tensor(s, ne)
    d.op_params[12] = PPDL_MAGIC - (1 << 32) if PPDL_MAGIC >= (1 << 31) else PPDL_MAGIC
    d.op_params[13] = op_id
    for i, v in enumerate(params):
        d.op_params[14 + i] = int(v)
    return d


def op_launch(op_id, dst, srcs=(), params=(), dst_ne=None, src_ne=(), stream=None) -> int:
    """ppdl_op_launch on torch tensors; returns the PPDL status code.
    `stream` is a torch.cuda.Stream or None for torch's current stream."""
    import torch
    d = make_desc(op_id, dst, srcs, params, dst_ne, src_ne)
    s = stream if stream is not None else torch.cuda.current_stream()
    return lib().ppdl_op_launch(C.byref(d), C.c_void_p(s.cuda_stream))


def op_supported(op_id, params=()) -> bool:
    d = OpDesc()
    d.op_params[12] = PPDL_MAGIC - (1 << 32)
    d.op_params[13] = op_id
    for i, v in enumerate(params):
        d.op_params[14 + i] = int(v)
    return bool(lib().ppdl_op_supported(C.byref(d)))


STEP_KINDS = {0: "other", 1: "gemm_1x1", 2: "wg_madd", 3: "gemm_implicit", 4: "gemm_linear",
              5: "wg_input", 6: "wg_output", 7: "dwconv", 8: "msda", 9: "mask_box", 10: "topk",
              11: "postprocess", 12: "glue", 13: "im2col",
              14: "attention", 15: "conv_direct"}


class StepStat(C.Structure):
    _fields_ = [("name", C.c_char * 48), ("kind", C.c_int32), ("ms", C.c_float),
                ("flops", C.c_double), ("bytes", C.c_double)]


class Context:
    """One loaded model on one GPU (ppdl_ctx).  Mirrors the reference usage
    ppdl_init -> ppdl_infer (-> ppdl_dump_raw) -> ppdl_free."""

    def __init__(self, model_path: str, device: int = -1, max_batch: int = 1,
                 dumps: bool = False, backend: int = BACKEND_CUDA):
        L = lib()
        L.ppdl_init_dev.argtypes = [C.c_char_p, C.c_int, C.c_int, C.c_int, C.c_int]
        L.ppdl_init_dev.restype = C.c_void_p
        L.ppdl_infer_batch.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p,
                                       C.POINTER(Result)]
        L.ppdl_infer_batch.restype = C.c_int
        L.ppdl_infer_device.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
        L.ppdl_infer_device.restype = C.c_int
        L.ppdl_device_outputs.argtypes = [C.c_void_p, C.POINTER(C.c_void_p), C.POINTER(C.c_void_p)]
        L.ppdl_device_outputs.restype = C.c_int
        L.ppdl_sync.argtypes = [C.c_void_p]
        L.ppdl_sync.restype = C.c_int
        self.lib = L
        self.max_batch = max_batch
        self.ctx = L.ppdl_init_dev(model_path.encode(), backend, device, max_batch, int(dumps))
        if not self.ctx:
            raise RuntimeError(f"ppdl_init failed for {model_path}")

    def infer(self, image, ori_h: int = IMG_SIZE, ori_w: int = IMG_SIZE):
        """One page (float32 [3,800,800]) -> (dets [300,7], masks [300,200,200])."""
        import numpy as np
        img = np.ascontiguousarray(image, dtype=np.float32)
        res = Result()
        rc = self.lib.ppdl_infer(self.ctx, img.ctypes.data, int(ori_h), int(ori_w), C.byref(res))
        if rc != 0:
            raise RuntimeError(f"ppdl_infer returned {rc}")
        dets = np.ctypeslib.as_array(res.dets, (NUM_DETS, DET_FIELDS)).copy()
        masks = np.ctypeslib.as_array(res.masks, (NUM_DETS, MASK_HW, MASK_HW)).copy()
        return dets, masks, res.infer_ms

    def infer_batch(self, images, ori_hw, copy=True):
        """n pages [n,3,800,800] -> list of (dets, masks).

        copy=True returns arrays the caller owns.  copy=False returns views
        of the context's pinned host buffers (what ppdl_infer_batch's
        ppdl_result points at), valid until the next inference on this
        context; it skips the 48 MB-per-page host copy of the masks.  Pages
        given in pinned host memory (e.g. a pinned torch tensor's .numpy())
        are copied to the device at full PCIe speed."""
        import numpy as np
        imgs = np.ascontiguousarray(images, dtype=np.float32)
        hw = np.ascontiguousarray(ori_hw, dtype=np.int32).reshape(-1, 2)
        n = imgs.shape[0]
        res = (Result * n)()
        rc = self.lib.ppdl_infer_batch(self.ctx, imgs.ctypes.data, n, hw.ctypes.data, res)
        if rc != 0:
            raise RuntimeError(f"ppdl_infer_batch returned {rc}")
        out = []
        for r in res:
            d = np.ctypeslib.as_array(r.dets, (NUM_DETS, DET_FIELDS))
            m = np.ctypeslib.as_array(r.masks, (NUM_DETS, MASK_HW, MASK_HW))
            out.append((d.copy(), m.copy()) if copy else (d, m))
        return out

    def infer_device(self, d_images_ptr: int, n: int, ori_hw) -> int:
        import numpy as np
        hw = np.ascontiguousarray(ori_hw, dtype=np.int32).reshape(-1, 2)
        self._hw = hw
        return self.lib.ppdl_infer_device(self.ctx, C.c_void_p(d_images_ptr), n, hw.ctypes.data)

    def device_outputs(self):
        d = C.c_void_p()
        m = C.c_void_p()
        rc = self.lib.ppdl_device_outputs(self.ctx, C.byref(d), C.byref(m))
        if rc != 0:
            raise RuntimeError("no device outputs")
        return d.value, m.value

    def sync(self) -> int:
        return self.lib.ppdl_sync(self.ctx)

    def infer_device_bits(self, d_images_ptr: int, n: int, ori_hw) -> int:
        """ppdl_infer_device with the masks left packed (no int32 expansion)."""
        import numpy as np
        L = self.lib
        L.ppdl_infer_device_bits.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
        L.ppdl_infer_device_bits.restype = C.c_int
        hw = np.ascontiguousarray(ori_hw, dtype=np.int32).reshape(-1, 2)
        self._hw = hw
        return L.ppdl_infer_device_bits(self.ctx, C.c_void_p(d_images_ptr), n, hw.ctypes.data)

    def device_mask_bits(self) -> int:
        L = self.lib
        L.ppdl_device_mask_bits.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
        L.ppdl_device_mask_bits.restype = C.c_int
        p = C.c_void_p()
        if L.ppdl_device_mask_bits(self.ctx, C.byref(p)) != 0:
            raise RuntimeError("no device outputs")
        return p.value

    def submit(self, images, ori_hw) -> int:
        """ppdl_submit_batch: enqueue n pages [n,3,800,800] (keep them alive
        and unchanged until wait() of the returned ticket; pinned memory lets
        the copy overlap the previous batch's forward)."""
        import numpy as np
        L = self.lib
        L.ppdl_submit_batch.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p,
                                        C.POINTER(C.c_int64)]
        L.ppdl_submit_batch.restype = C.c_int
        if not (isinstance(images, np.ndarray) and images.dtype == np.float32 and
                images.flags.c_contiguous):
            raise ValueError("submit() needs a C-contiguous float32 array that stays alive")
        hw = np.ascontiguousarray(ori_hw, dtype=np.int32).reshape(-1, 2)
        t = C.c_int64()
        rc = L.ppdl_submit_batch(self.ctx, images.ctypes.data, images.shape[0], hw.ctypes.data,
                                 C.byref(t))
        if rc != 0:
            raise RuntimeError(f"ppdl_submit_batch returned {rc}")
        return t.value

    def wait(self, ticket: int, n: int, copy=True):
        """ppdl_wait_batch: [(dets [300,7], mask_bits [300,1250] uint32)] of
        the n pages of ticket.  copy=False returns views of the context's
        pinned result slot, valid until ticket + 2 is submitted."""
        import numpy as np
        L = self.lib
        L.ppdl_wait_batch.argtypes = [C.c_void_p, C.c_int64, C.POINTER(ResultBits)]
        L.ppdl_wait_batch.restype = C.c_int
        res = (ResultBits * n)()
        rc = L.ppdl_wait_batch(self.ctx, ticket, res)
        if rc != 0:
            raise RuntimeError(f"ppdl_wait_batch returned {rc}")
        out = []
        for r in res:
            d = np.ctypeslib.as_array(r.dets, (NUM_DETS, DET_FIELDS))
            b = np.ctypeslib.as_array(r.mask_bits, (NUM_DETS, MASK_WORDS))
            out.append((d.copy(), b.copy()) if copy else (d, b))
        return out

    def stream_ptr(self) -> int:
        self.lib.ppdl_stream.argtypes = [C.c_void_p]
        self.lib.ppdl_stream.restype = C.c_void_p
        return self.lib.ppdl_stream(self.ctx) or 0

    def profile_steps(self, n: int):
        """[(name, kind, ms, flops_per_page, bytes_per_page)] of one eager
        forward of the last n pages, with a CUDA event after every step."""
        self.lib.ppdl_profile_steps.argtypes = [C.c_void_p, C.c_int, C.POINTER(StepStat), C.c_int]
        self.lib.ppdl_profile_steps.restype = C.c_int
        buf = (StepStat * 4096)()
        k = self.lib.ppdl_profile_steps(self.ctx, n, buf, 4096)
        if k < 0:
            raise RuntimeError("ppdl_profile_steps failed")
        return [(buf[i].name.decode(), STEP_KINDS.get(buf[i].kind, "other"), buf[i].ms,
                 buf[i].flops, buf[i].bytes) for i in range(k)]

    def profile_timeline(self, n: int):
        """[(end_ms, lane)] per step (the order of profile_steps): the end of
        each step from the start of the forward, with the lanes running
        concurrently as in the captured forward."""
        self.lib.ppdl_profile_timeline.argtypes = [C.c_void_p, C.c_int, C.POINTER(C.c_float),
                                                   C.POINTER(C.c_int32), C.c_int]
        self.lib.ppdl_profile_timeline.restype = C.c_int
        end = (C.c_float * 4096)()
        lane = (C.c_int32 * 4096)()
        k = self.lib.ppdl_profile_timeline(self.ctx, n, end, lane, 4096)
        if k < 0:
            raise RuntimeError("ppdl_profile_timeline failed")
        return [(end[i], lane[i]) for i in range(k)]

    def dump_raw(self, pfx: str) -> int:
        return self.lib.ppdl_dump_raw(self.ctx, pfx.encode())

    def dump(self, d: str) -> int:
        return self.lib.ppdl_dump(self.ctx, d.encode())

    def close(self):
        if self.ctx:
            self.lib.ppdl_free(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def last_error() -> str:
    return lib().ppdl_op_last_error().decode()


def check(status: int) -> None:
    if status != PPDL_OK:
        raise RuntimeError(f"ppdl_op_launch failed ({status}): {last_error()}")


# ---- transformer-block operators ---------------------------------------------
# Functions of torch CUDA tensors.  Each enqueues on torch's current stream of
# the tensors' device, returns new tensors, and raises ValueError for tensors
# it does not take and RuntimeError for a call the library refuses.  They
# record no autograd history: a backward pass is a function of its own.

F32, BF16, F16 = 0, 1, 2
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


class RotaryHeads(C.Structure):
    """ppdl_rotary_heads."""
    _fields_ = [("in_", C.c_void_p), ("out", C.c_void_p), ("heads", C.c_int32),
                ("in_batch", C.c_int64), ("in_token", C.c_int64), ("in_head", C.c_int64),
                ("out_batch", C.c_int64), ("out_token", C.c_int64), ("out_head", C.c_int64)]


# the same bytes for rotary(), filled in 0.2 us (the structure 1.1)
_pack_heads = struct.Struct("@PPiqqqqqq").pack


def _declare_block_ops(L) -> None:
    p, i, ll, f = C.c_void_p, C.c_int, C.c_longlong, C.c_float
    L.ppdl_layernorm.argtypes = [p, ll, p, ll, p, p, i, i, ll, i, f, p, ll, p, ll, p, p, p]
    L.ppdl_layernorm_backward.argtypes = [p, ll, p, ll, p, p, p, p, ll, i, i, ll, i, p, ll, p, p,
                                          p, p]
    L.ppdl_layernorm_backward_workspace.argtypes = [ll, i]
    L.ppdl_layernorm_backward_workspace.restype = ll
    L.ppdl_quantize_rows_i8.argtypes = [p, ll, i, ll, i, p, ll, p, p]
    L.ppdl_linear_i8.argtypes = [p, ll, p, p, ll, p, p, p, ll, i, i, i, i, i, p, ll, p]
    L.ppdl_linear_i8_dynamic.argtypes = [p, ll, i, p, ll, p, p, p, ll, i, i, i, i, i, p, ll, p, p]
    L.ppdl_linear_i8_dynamic_workspace.argtypes = [i, i]
    L.ppdl_linear_i8_dynamic_workspace.restype = ll
    L.ppdl_rotary.argtypes = [p, p, i, i, i, i, i, p, i, ll, ll, ll, i, p, p, i, i, p]


# What the functions use of torch, bound by the first call (importing this
# module does not import torch): a call's arguments are looked at in about
# 3 us, with as few Python calls as that takes.
_types, _tt = {}, {}


def _bind() -> None:
    import torch
    lib()
    # the current stream's handle without the object around it (2 us)
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
        (lambda i: torch.cuda.current_stream(i).cuda_stream)
    _tt.update(f32=torch.float32, f64=torch.float64, i8=torch.int8,
               integers=(torch.int32, torch.int64), empty_like=torch.empty_like, stream=raw,
               current=torch.cuda.current_device, device=torch.cuda.device)
    # last: a thread that finds it filled goes on without binding
    _types.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16})


def _type(t, name: str) -> int:
    """The PPDL_* element type of tensor t."""
    if not _types:
        _bind()
    code = _types.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def _rows(t, name: str, shape) -> int:
    """The distance between the rows of shape[-1] values that t, of this
    shape, consists of; t may be strided as long as its rows lie evenly
    apart."""
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    width = shape[-1] if shape else 0
    if width > 0x7fffffff or not shape:
        raise ValueError(f"{name} must have rows of at most 2^31 - 1 values")
    if t.is_contiguous():
        return width
    ld = span = None
    if t.stride(-1) == 1 or width == 1:
        for n, s in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
            if n == 1:
                continue
            if ld is None:
                ld = s
            elif s != span:
                break
            span = s * n
        else:
            return width if ld is None else ld
    raise ValueError(f"{name} must consist of contiguous rows at one distance, "
                     f"not strides {tuple(t.stride())} of shape {tuple(shape)}")


def _vector(t, name: str, n: int, dtype=None):
    if t.dim() != 1 or t.numel() != n or not (n <= 1 or t.is_contiguous()) or \
            (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} must be {n} contiguous values"
                         + (f" of {dtype}" if dtype is not None else ""))


def _device(x, *others) -> int:
    """The index of the GPU that x and the others (tensors or None) are on."""
    index = x.get_device()
    if index < 0:
        raise ValueError(f"tensors on {x.device}: the operators take CUDA tensors")
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on {x.device} and {t.device}")
    return index


def _elsewhere(index: int, f, *args, **kw):
    """f on tensors of a GPU that is not the current one."""
    with _tt["device"](index):
        return f(*args, **kw)


def _failed(fn, status: int):
    raise RuntimeError(f"{fn.__name__} failed ({status}): {last_error()}")


def layernorm(x, weight=None, bias=None, eps: float = 1e-5, *, residual=None,
              return_sum: bool = False, return_stats: bool = False):
    """Layer norm of the rows of x [..., D] (ppdl_layernorm), of x + residual
    when one is given (the sum rounded to x's type).  weight and bias [D] are
    of x's type or float32.  Returns y, followed by the sum (return_sum) and
    by the rows' mean and rstd in float32 (return_stats), which the backward
    pass takes."""
    shape = x.shape
    t = wt = _type(x, "x")
    ldx = _rows(x, "x", shape)
    D = shape[-1]
    ldr, rp, wp, bp = 0, None, None, None
    if residual is not None:
        if residual.dtype != x.dtype:
            raise ValueError("residual must have x's type")
        ldr, rp = _rows(residual, "residual", shape), residual.data_ptr()
    elif return_sum:
        raise ValueError("return_sum needs a residual")
    if weight is not None:
        _vector(weight, "weight", D)
        wt, wp = _type(weight, "weight"), weight.data_ptr()
    if bias is not None:
        _vector(bias, "bias", D)
        wt, bp = _type(bias, "bias"), bias.data_ptr()
        if weight is not None and weight.dtype != bias.dtype:
            raise ValueError("weight and bias must have one type")
    dev = _device(x, residual, weight, bias)
    if dev != _tt["current"]():
        return _elsewhere(dev, layernorm, x, weight, bias, eps, residual=residual,
                          return_sum=return_sum, return_stats=return_stats)
    # (empty_like keeps a dense x's strides, which are those of rows in order)
    y = _tt["empty_like"](x)
    s = mean = rstd = sp = mp = vp = None
    if return_sum:
        s = _tt["empty_like"](x)
        sp = s.data_ptr()
    if return_stats:
        mean, rstd = x.new_empty((2,) + shape[:-1], dtype=_tt["f32"]).unbind(0)
        mp, vp = mean.data_ptr(), rstd.data_ptr()
    fn = _lib.ppdl_layernorm
    status = fn(x.data_ptr(), ldx, rp, ldr, wp, bp, t, wt, x.numel() // D if D else 0, D, eps,
                y.data_ptr(), D, sp, D, mp, vp, _tt["stream"](dev))
    if status:
        _failed(fn, status)
    if not (return_sum or return_stats):
        return y
    return (y,) + ((s,) if return_sum else ()) + ((mean, rstd) if return_stats else ())


def layernorm_backward(dy, x, weight, mean, rstd, *, dsum=None, param_grads: bool = True):
    """The gradients (dx, dweight, dbias) of layernorm at its input x — the
    returned sum when it had a residual — from the gradient dy of its result
    and its statistics (ppdl_layernorm_backward).  dsum is the gradient that
    reaches the sum on its other path; dx is then the gradient of x and of
    the residual alike.  dweight and dbias have weight's type (x's without a
    weight) and are None without param_grads."""
    shape = x.shape
    t = wt = _type(x, "x")
    ldx, lddy = _rows(x, "x", shape), _rows(dy, "dy", shape)
    D, lead, f32 = shape[-1], shape[:-1], _tt["f32"]
    ldds, dsp, wp = 0, None, None
    if dsum is not None:
        ldds, dsp = _rows(dsum, "dsum", shape), dsum.data_ptr()
    if dy.dtype != x.dtype or (dsum is not None and dsum.dtype != x.dtype):
        raise ValueError("dy and dsum must have x's type")
    if weight is not None:
        _vector(weight, "weight", D)
        wt, wp = _type(weight, "weight"), weight.data_ptr()
    for v, name in ((mean, "mean"), (rstd, "rstd")):
        if v.dtype != f32 or v.shape != lead or not v.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 of shape {tuple(lead)}")
    dev = _device(x, dy, weight, mean, rstd, dsum)
    if dev != _tt["current"]():
        return _elsewhere(dev, layernorm_backward, dy, x, weight, mean, rstd, dsum=dsum,
                          param_grads=param_grads)
    rows = x.numel() // D if D else 0
    dx = _tt["empty_like"](x)
    dw = db = dwp = dbp = wsp = None
    if param_grads:
        dw, db = (x.new_empty(D), x.new_empty(D)) if weight is None else \
            (_tt["empty_like"](weight), _tt["empty_like"](weight))
        work = mean.new_empty(_backward_work(rows, D))
        dwp, dbp, wsp = dw.data_ptr(), db.data_ptr(), work.data_ptr()
    fn = _lib.ppdl_layernorm_backward
    status = fn(dy.data_ptr(), lddy, x.data_ptr(), ldx, wp, mean.data_ptr(), rstd.data_ptr(), dsp,
                ldds, t, wt, rows, D, dx.data_ptr(), D, dwp, dbp, wsp, _tt["stream"](dev))
    if status:
        _failed(fn, status)
    return dx, dw, db


@functools.lru_cache(maxsize=256)
def _backward_work(rows: int, D: int) -> int:
    return _lib.ppdl_layernorm_backward_workspace(rows, D)


def quantize_rows(x):
    """8-bit rows of x [..., K] (ppdl_quantize_rows_i8): (q, scale) with q
    int8 [..., K], rows on strides of a multiple of 16 bytes, and scale
    float32 [...]: q * scale[..., None] stands for x.  It quantises weights
    [N, K] channel by channel and activations token by token."""
    shape = x.shape
    t = _type(x, "x")
    ldx = _rows(x, "x", shape)
    K, lead = shape[-1], shape[:-1]
    ldq = (K + 15) // 16 * 16
    dev = _device(x)
    if dev != _tt["current"]():
        return _elsewhere(dev, quantize_rows, x)
    q = x.new_empty(lead + (ldq,), dtype=_tt["i8"])
    scale = x.new_empty(lead, dtype=_tt["f32"])
    fn = _lib.ppdl_quantize_rows_i8
    status = fn(x.data_ptr(), ldx, t, x.numel() // K if K else 0, K, q.data_ptr(), ldq,
                scale.data_ptr(), _tt["stream"](dev))
    if status:
        _failed(fn, status)
    return q if ldq == K else q[..., :K], scale


def linear_i8(x, weight, w_scale, *, x_scale=None, bias=None, act: str = "none", residual=None,
              out_dtype=None):
    """act(x weight^T + bias) + residual on 8-bit integers (ppdl_linear_i8).
    weight int8 [N, K] and w_scale float32 [N] as quantize_rows makes them.
    x [..., K]: float32 / bfloat16 / float16 rows, quantised token by token
    in the call; or int8 with x_scale float32 [...].  bias float32 [N]; act
    none, relu, silu or gelu; residual [..., N] of the result's type, which is
    x's (for int8 x: residual's, else float32) unless out_dtype says
    otherwise."""
    if not _types:
        _bind()
    wshape, shape, i8, f32 = weight.shape, x.shape, _tt["i8"], _tt["f32"]
    if len(wshape) != 2 or weight.dtype != i8:
        raise ValueError("weight must be int8 [N, K]")
    N, K = wshape
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {', '.join(ACTS)}")
    lead = shape[:-1]
    ldw, ldx = _rows(weight, "weight", wshape), _rows(x, "x", lead + (K,))
    _vector(w_scale, "w_scale", N, f32)
    bp = rp = None
    if bias is not None:
        _vector(bias, "bias", N, f32)
        bp = bias.data_ptr()
    if x.dtype == i8:
        if x_scale is None or x_scale.dtype != f32 or x_scale.shape != lead or \
                not x_scale.is_contiguous():
            raise ValueError(f"int8 x needs x_scale, contiguous float32 of shape {tuple(lead)}")
        dtype = out_dtype or (f32 if residual is None else residual.dtype)
    elif x_scale is not None:
        raise ValueError("x_scale goes with int8 x")
    else:
        xt = _type(x, "x")
        dtype = out_dtype or x.dtype
    dev = _device(x, x_scale, weight, w_scale, bias, residual)
    if dev != _tt["current"]():
        return _elsewhere(dev, linear_i8, x, weight, w_scale, x_scale=x_scale, bias=bias, act=act,
                          residual=residual, out_dtype=out_dtype)
    y = x.new_empty(lead + (N,), dtype=dtype)
    t = _type(y, "the result")
    ldr = 0
    if residual is not None:
        if residual.dtype != dtype:
            raise ValueError("residual must have the result's type")
        ldr, rp = _rows(residual, "residual", y.shape), residual.data_ptr()
    M = x.numel() // K if K else 0
    if M > 0x7fffffff or N > 0x7fffffff:
        raise ValueError(f"{M} rows and {N} channels: each must fit 31 bits")
    if x_scale is not None:
        fn = _lib.ppdl_linear_i8
        status = fn(x.data_ptr(), ldx, x_scale.data_ptr(), weight.data_ptr(), ldw,
                    w_scale.data_ptr(), bp, rp, ldr, t, code, M, N, K, y.data_ptr(), N,
                    _tt["stream"](dev))
    else:
        work = weight.new_empty(M * ((K + 15) // 16 * 16 + 4))  # ..._dynamic_workspace(M, K)
        fn = _lib.ppdl_linear_i8_dynamic
        status = fn(x.data_ptr(), ldx, xt, weight.data_ptr(), ldw, w_scale.data_ptr(), bp, rp, ldr,
                    t, code, M, N, K, y.data_ptr(), N, work.data_ptr(), _tt["stream"](dev))
    if status:
        _failed(fn, status)
    return y


def _heads(x, inplace: bool, name: str, lead, dim: int, dtype):
    """ppdl_rotary_heads for x, and the tensor that takes it turned."""
    shape = x.shape
    if len(shape) != 4 or shape[3] != dim or shape[:2] != lead or x.dtype != dtype or \
            shape[2] > 0x7fffffff:
        raise ValueError(f"{name} must be [batch, length, heads, {dim}] of one type, heads of 31 bits")
    i = x.stride()
    if dim > 1 and i[3] != 1:
        raise ValueError(f"{name}'s heads must be contiguous")
    out, o = x, i
    if not inplace:
        # empty_like keeps a dense tensor's strides, whichever their order; what
        # it gives for a view whose elements overlap (windows of a buffer) may
        # not have contiguous heads
        out = _tt["empty_like"](x)
        o = out.stride()
        if o[3] != 1:
            out = x.new_empty(shape)
            o = out.stride()
    return _pack_heads(x.data_ptr(), out.data_ptr(), shape[2], *i[:3], *o[:3]), out


def rotary(q, k, positions, freq, sections, *, interleaved: bool = False, inverse: bool = False,
           inplace: bool = False):
    """Rotary positions with several axes (ppdl_rotary) on q [batch, length,
    heads, dim] and k (its own number of heads, or None): returns both turned
    (new tensors, or q and k themselves with inplace, which must not overlap
    then).  positions int32 or
    int64 [axes, batch, length] (may be expanded views); freq float64
    [rotated / 2] in radians per position turns the first `rotated` values of
    every head; sections says how many consecutive pairs each axis turns.
    inverse turns back: the backward pass."""
    t = _type(q, "q")
    lead, dim = q.shape[:2], q.shape[-1] if q.dim() else 0
    axes, pshape = len(sections), positions.shape
    if positions.dtype not in _tt["integers"] or len(pshape) != 3 or pshape[0] != axes or \
            pshape[1:] != lead:
        raise ValueError("positions must be int32 or int64 [axes, batch, length], one axis a section")
    if freq.dtype != _tt["f64"] or freq.dim() != 1 or not freq.is_contiguous():
        raise ValueError("freq must be contiguous float64 [rotated / 2]")
    pairs = freq.numel()
    # (what the library takes as 32-bit numbers)
    if dim > 0x7fffffff or lead[0] > 0x7fffffff or lead[1] > 0x7fffffff or pairs > 0x3fffffff:
        raise ValueError("batch, length, dim and rotated must fit 31 bits each")
    dev = _device(q, k, positions, freq)
    if dev != _tt["current"]():
        return _elsewhere(dev, rotary, q, k, positions, freq, sections, interleaved=interleaved,
                          inverse=inverse, inplace=inplace)
    ko = hk = None
    hq, qo = _heads(q, inplace, "q", lead, dim, q.dtype)
    if k is not None:
        hk, ko = _heads(k, inplace, "k", lead, dim, q.dtype)
    fn = _lib.ppdl_rotary
    status = fn(hq, hk, t, *lead, dim, 2 * pairs, positions.data_ptr(),
                positions.element_size(), *positions.stride(), axes, _sections(tuple(sections)),
                freq.data_ptr(), interleaved, inverse, _tt["stream"](dev))
    if status:
        _failed(fn, status)
    return qo, ko


@functools.lru_cache(maxsize=64)
def _sections(sections):
    a = (C.c_int32 * len(sections))(*sections)
    if tuple(a) != sections:
        raise ValueError(f"sections {sections} do not fit 31 bits")
    return a
