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
import os

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


def _declare_block_ops(L) -> None:
    p, i, ll, f = C.c_void_p, C.c_int, C.c_longlong, C.c_float
    L.ppdl_layernorm.argtypes = [p, ll, p, ll, p, p, i, i, ll, i, f, p, ll, p, ll, p, p, p]
    L.ppdl_layernorm_backward.argtypes = [p, ll, p, ll, p, p, p, p, ll, i, i, ll, i, p, ll, p, p,
                                          p, p]
    L.ppdl_layernorm_backward_workspace.argtypes = [ll, i]
    L.ppdl_layernorm_backward_workspace.restype = ll
    L.ppdl_quantize_rows_i8.argtypes = [p, ll, i, ll, i, p, ll, p, p]
    L.ppdl_linear_i8.argtypes = [p, ll, p, p, ll, p, p, p, ll, i, i, i, i, i, p, ll, p]
    L.ppdl_rotary.argtypes = [p, p, i, i, i, i, i, p, i, ll, ll, ll, i, p, p, i, i, p]


_types = {}


def _type(t, name: str) -> int:
    """The PPDL_* element type of tensor t."""
    if not _types:
        import torch
        _types.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16})
    code = _types.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def _rows(t, name: str, width: int, like=None) -> int:
    """The distance between the rows of width values that t [..., width]
    consists of; t may be strided as long as its rows lie evenly apart."""
    if t.dim() == 0 or t.shape[-1] != width or (like is not None and t.shape != like.shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected "
                         f"{tuple(like.shape) if like is not None else (..., width)}")
    if t.is_contiguous():
        return width
    ld = span = None
    if t.stride(-1) == 1 or width == 1:
        for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
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
                     f"not strides {tuple(t.stride())} of shape {tuple(t.shape)}")


def _vector(t, name: str, n: int, dtype=None):
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1) or \
            (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} must be {n} contiguous values"
                         + (f" of {dtype}" if dtype is not None else ""))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(fn, tensors, *args) -> None:
    """fn(*args, stream) on the tensors' device, checked."""
    import torch
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}")
    if dev.type != "cuda":
        raise ValueError(f"tensors on {dev}: the operators take CUDA tensors")
    stream = torch.cuda.current_stream(dev).cuda_stream
    if dev.index == torch.cuda.current_device():
        status = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            status = fn(*args, stream)
    if status != PPDL_OK:
        raise RuntimeError(f"{fn.__name__} failed ({status}): {last_error()}")


def layernorm(x, weight=None, bias=None, eps: float = 1e-5, *, residual=None,
              return_sum: bool = False, return_stats: bool = False):
    """Layer norm of the rows of x [..., D] (ppdl_layernorm), of x + residual
    when one is given (the sum rounded to x's type).  weight and bias [D] are
    of x's type or float32.  Returns y, followed by the sum (return_sum) and
    by the rows' mean and rstd in float32 (return_stats), which the backward
    pass takes."""
    import torch
    D = x.shape[-1] if x.dim() else 0
    t = _type(x, "x")
    ldx = _rows(x, "x", D)
    ldr = 0
    if residual is not None:
        ldr = _rows(residual, "residual", D, x)
        if residual.dtype != x.dtype:
            raise ValueError("residual must have x's type")
    elif return_sum:
        raise ValueError("return_sum needs a residual")
    wt = t
    for v, name in ((weight, "weight"), (bias, "bias")):
        if v is not None:
            _vector(v, name, D)
            wt = _type(v, name)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one type")
    rows = x.numel() // D if D else 0
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    s = torch.empty(x.shape, dtype=x.dtype, device=x.device) if return_sum else None
    mean = rstd = None
    if return_stats:
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
    _call(lib().ppdl_layernorm, (x, residual, weight, bias), x.data_ptr(), ldx, _ptr(residual), ldr,
          _ptr(weight), _ptr(bias), t, wt, rows, D, eps, y.data_ptr(), D, _ptr(s), D, _ptr(mean),
          _ptr(rstd))
    out = (y,) + ((s,) if return_sum else ()) + ((mean, rstd) if return_stats else ())
    return out if len(out) > 1 else y


def layernorm_backward(dy, x, weight, mean, rstd, *, dsum=None, param_grads: bool = True):
    """The gradients (dx, dweight, dbias) of layernorm at its input x — the
    returned sum when it had a residual — from the gradient dy of its result
    and its statistics (ppdl_layernorm_backward).  dsum is the gradient that
    reaches the sum on its other path; dx is then the gradient of x and of
    the residual alike.  dweight and dbias have weight's type (x's without a
    weight) and are None without param_grads."""
    import torch
    D = x.shape[-1] if x.dim() else 0
    t = _type(x, "x")
    ldx, lddy = _rows(x, "x", D), _rows(dy, "dy", D, x)
    ldds = _rows(dsum, "dsum", D, x) if dsum is not None else 0
    if dy.dtype != x.dtype or (dsum is not None and dsum.dtype != x.dtype):
        raise ValueError("dy and dsum must have x's type")
    wt = t
    if weight is not None:
        _vector(weight, "weight", D)
        wt = _type(weight, "weight")
    rows = x.numel() // D if D else 0
    for v, name in ((mean, "mean"), (rstd, "rstd")):
        if v.dtype != torch.float32 or v.shape != x.shape[:-1] or not v.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 of shape {tuple(x.shape[:-1])}")
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = db = work = None
    L = lib()
    if param_grads:
        grads = torch.empty((2, D), dtype=x.dtype if weight is None else weight.dtype,
                            device=x.device)
        dw, db = grads[0], grads[1]
        work = torch.empty(L.ppdl_layernorm_backward_workspace(rows, D), dtype=torch.float32,
                           device=x.device)
    _call(L.ppdl_layernorm_backward, (x, dy, weight, mean, rstd, dsum), dy.data_ptr(), lddy,
          x.data_ptr(), ldx, _ptr(weight), mean.data_ptr(), rstd.data_ptr(), _ptr(dsum), ldds, t,
          wt, rows, D, dx.data_ptr(), D, _ptr(dw), _ptr(db), _ptr(work))
    return dx, dw, db


def quantize_rows(x):
    """8-bit rows of x [..., K] (ppdl_quantize_rows_i8): (q, scale) with q
    int8 [..., K], rows on strides of a multiple of 16 bytes, and scale
    float32 [...]: q * scale[..., None] stands for x.  It quantises weights
    [N, K] channel by channel and activations token by token."""
    import torch
    K = x.shape[-1] if x.dim() else 0
    t = _type(x, "x")
    ldx = _rows(x, "x", K)
    ldq = (K + 15) // 16 * 16
    q = torch.empty(x.shape[:-1] + (ldq,), dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _call(lib().ppdl_quantize_rows_i8, (x,), x.data_ptr(), ldx, t, x.numel() // K if K else 0, K,
          q.data_ptr(), ldq, scale.data_ptr())
    return q[..., :K], scale


def linear_i8(x, weight, w_scale, *, x_scale=None, bias=None, act: str = "none", residual=None,
              out_dtype=None):
    """act(x weight^T + bias) + residual on 8-bit integers (ppdl_linear_i8).
    weight int8 [N, K] and w_scale float32 [N] as quantize_rows makes them.
    x [..., K]: float32 / bfloat16 / float16 rows, quantised token by token
    in the call; or int8 with x_scale float32 [...].  bias float32 [N]; act
    none, relu, silu or gelu; residual [..., N] of the result's type, which is
    x's (for int8 x: residual's, else float32) unless out_dtype says
    otherwise."""
    import torch
    if weight.dim() != 2 or weight.dtype != torch.int8:
        raise ValueError("weight must be int8 [N, K]")
    N, K = weight.shape
    if act not in ACTS:
        raise ValueError(f"act must be one of {', '.join(ACTS)}")
    ldw = _rows(weight, "weight", K)
    ldx = _rows(x, "x", K)
    _vector(w_scale, "w_scale", N, torch.float32)
    if bias is not None:
        _vector(bias, "bias", N, torch.float32)
    lead = x.shape[:-1]
    M = x.numel() // K if K else 0
    if x.dtype == torch.int8:
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.shape != lead or \
                not x_scale.is_contiguous():
            raise ValueError(f"int8 x needs x_scale, contiguous float32 of shape {tuple(lead)}")
        dtype = out_dtype or (torch.float32 if residual is None else residual.dtype)
    else:
        if x_scale is not None:
            raise ValueError("x_scale goes with int8 x")
        dtype = out_dtype or x.dtype
    y = torch.empty(lead + (N,), dtype=dtype, device=x.device)
    t = _type(y, "the result")
    ldr = 0
    if residual is not None:
        ldr = _rows(residual, "residual", N, y)
        if residual.dtype != dtype:
            raise ValueError("residual must have the result's type")
    L = lib()
    if x_scale is None:
        q = torch.empty((M, (K + 15) // 16 * 16), dtype=torch.int8, device=x.device)
        x_scale = torch.empty(M, dtype=torch.float32, device=x.device)
        _call(L.ppdl_quantize_rows_i8, (x,), x.data_ptr(), ldx, _type(x, "x"), M, K, q.data_ptr(),
              q.shape[1], x_scale.data_ptr())
        x, ldx = q, q.shape[1]
    _call(L.ppdl_linear_i8, (x, x_scale, weight, w_scale, bias, residual), x.data_ptr(), ldx,
          x_scale.data_ptr(), weight.data_ptr(), ldw, w_scale.data_ptr(), _ptr(bias),
          _ptr(residual), ldr, t, ACTS[act], M, N, K, y.data_ptr(), N)
    return y


def _heads(x, out, name: str, dim: int, like):
    if x.dim() != 4 or x.shape[3] != dim or x.shape[:2] != like.shape[:2] or x.dtype != like.dtype:
        raise ValueError(f"{name} must be [batch, length, heads, {dim}] of one type")
    if dim > 1 and x.stride(3) != 1:
        raise ValueError(f"{name}'s heads must be contiguous")
    i, o = x.stride(), out.stride()
    return RotaryHeads(x.data_ptr(), out.data_ptr(), x.shape[2], i[0], i[1], i[2], o[0], o[1], o[2])


def rotary(q, k, positions, freq, sections, *, interleaved: bool = False, inverse: bool = False,
           inplace: bool = False):
    """Rotary positions with several axes (ppdl_rotary) on q [batch, length,
    heads, dim] and k (its own number of heads, or None): returns both turned
    (new tensors, or q and k themselves with inplace).  positions int32 or
    int64 [axes, batch, length] (may be expanded views); freq float64
    [rotated / 2] in radians per position turns the first `rotated` values of
    every head; sections says how many consecutive pairs each axis turns.
    inverse turns back: the backward pass."""
    import torch
    dim = q.shape[-1] if q.dim() else 0
    t = _type(q, "q")
    if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 3 or \
            positions.shape[0] != len(sections) or positions.shape[1:] != q.shape[:2]:
        raise ValueError("positions must be int32 or int64 [axes, batch, length], one axis a section")
    if freq.dtype != torch.float64 or freq.dim() != 1 or not freq.is_contiguous():
        raise ValueError("freq must be contiguous float64 [rotated / 2]")
    qo = q if inplace else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    hq = _heads(q, qo, "q", dim, q)
    ko = hk = None
    if k is not None:
        ko = k if inplace else torch.empty(k.shape, dtype=k.dtype, device=k.device)
        hk = _heads(k, ko, "k", dim, q)
    ps = positions.stride()
    _call(lib().ppdl_rotary, (q, k, positions, freq), C.byref(hq),
          C.byref(hk) if hk is not None else None, t, q.shape[0], q.shape[1], dim,
          2 * freq.shape[0], positions.data_ptr(), positions.element_size(), ps[0], ps[1], ps[2],
          len(sections), (C.c_int32 * len(sections))(*sections), freq.data_ptr(), int(interleaved),
          int(inverse))
    return qo, ko
