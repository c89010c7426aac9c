"""Stand-alone training operators over the C-ABI: layer norm, block-scaled 8-bit
quantising and product, AdamW over many tensors.

As everywhere in this package tensors are raw device pointers with their sizes and
strides (in elements), streams are raw handles (None: the default stream), and an
error raises PktError. A descriptor (LayerNormDesc, Fp8QuantizeDesc, Fp8GemmDesc) is
read during the call only and can be kept and used again; include/pkt_b200.h has the
formulas, the layouts and the rules of each field.
"""
import ctypes

from . import _lib
from ._lib import (AdamWConfig, AdamWTensor, Fp8GemmDesc, Fp8QuantizeDesc, LayerNormDesc, PKT_DTYPE_BF16,  # noqa: F401
                   PKT_DTYPE_E4M3, PKT_DTYPE_E5M2, PKT_DTYPE_F32, check)
from .runtime import _current_device

DTYPE_BF16, DTYPE_F32, DTYPE_E4M3, DTYPE_E5M2 = PKT_DTYPE_BF16, PKT_DTYPE_F32, PKT_DTYPE_E4M3, PKT_DTYPE_E5M2
_DTYPES = {"bf16": DTYPE_BF16, "f32": DTYPE_F32, "e4m3": DTYPE_E4M3}


def layernorm_forward(desc, stream=None):
    """y (and mean, rstd) of LayerNormDesc `desc`."""
    check(_lib.load().pkt_layernorm_forward(desc, stream))


def layernorm_backward_workspace(desc):
    """Bytes of workspace that layernorm_backward needs for desc.rows x desc.cols."""
    n = ctypes.c_size_t()
    check(_lib.load().pkt_layernorm_backward_workspace(desc, ctypes.byref(n)))
    return n.value


def layernorm_backward(desc, stream=None):
    """dx, dgamma, dbeta of LayerNormDesc `desc` (the forward pass's mean and rstd are inputs)."""
    check(_lib.load().pkt_layernorm_backward(desc, stream))


def fp8_quantize(desc, stream=None):
    """Quantises x of Fp8QuantizeDesc `desc` to q and / or the transposed qt."""
    check(_lib.load().pkt_fp8_quantize(desc, stream))


def fp8_gemm(desc, stream=None):
    """out = a b^T of Fp8GemmDesc `desc`, the scales of each block of 128 applied."""
    check(_lib.load().pkt_fp8_gemm(desc, stream))


def ops_status():
    """0, or the code of a wait that ran out in an operator's kernel since the last call (synchronises)."""
    code = ctypes.c_int()
    check(_lib.load().pkt_ops_status(ctypes.byref(code)))
    return code.value


class AdamW:
    """One AdamW step over many tensors per call (pkt_adamw_*). `tensors`: AdamWTensor
    records; the arrays they name stay the caller's and must outlive the plan."""

    def __init__(self, tensors, beta1=0.9, beta2=0.999, eps=1e-8, param_dtype="f32", grad_dtype="f32",
                 state_dtype="f32", step=0, device=None):
        self._h = None
        L = _lib.load()
        self._L = L
        tensors = list(tensors)
        self.num_tensors = len(tensors)
        arr = (AdamWTensor * max(1, len(tensors)))(*tensors)
        cfg = AdamWConfig(len(tensors), arr, _DTYPES[param_dtype], _DTYPES[grad_dtype], _DTYPES[state_dtype],
                          float(beta1), float(beta2), float(eps), int(step))
        h = ctypes.c_void_p()
        check(L.pkt_adamw_create(_current_device() if device is None else device, ctypes.byref(cfg), ctypes.byref(h)))
        self._h = h

    def close(self):
        if self._h:
            self._L.pkt_adamw_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def step(self, lr, grad_scale=1.0, scales=None, stream=None):
        """scales: device pointer to 2 floats multiplying lr and the gradients, or None."""
        check(self._L.pkt_adamw_step(self._h, lr, grad_scale, scales, stream))

    def set_grads(self, grads, stream=None):
        """New gradient pointers, one per tensor (None: that tensor is left alone)."""
        grads = list(grads)
        if len(grads) != self.num_tensors:
            raise ValueError(f"{len(grads)} gradients for {self.num_tensors} tensors")
        arr = (ctypes.c_void_p * max(1, len(grads)))(*grads)
        check(self._L.pkt_adamw_set_grads(self._h, ctypes.cast(arr, ctypes.c_void_p), stream))

    def set_step(self, step, stream=None):
        check(self._L.pkt_adamw_set_step(self._h, int(step), stream))

    def get_step(self, stream=None):
        n = ctypes.c_longlong()
        check(self._L.pkt_adamw_get_step(self._h, ctypes.byref(n), stream))
        return n.value
