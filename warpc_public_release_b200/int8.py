"""The 8-bit operators over the C ABI (include/warpc_b200.h): rows to 8-bit integers with a scale each, with or without the
root-mean-square norm before it, and the product of 8-bit integers scaled for each token and channel.

As everywhere in this package the caller owns the memory and passes integer device addresses; strides are in elements, `stream` is
an integer cudaStream_t (None = the default stream) and every call is asynchronous.  Value types are named "bf16", "fp16", "fp32".
The reference has no counterpart of these operators.
"""
import ctypes

from . import _lib
from ._lib import INT8_FEW, INT8_GEMV, INT8_TILE, Int8Info, check
from .plan import DeviceWaitError

KERNELS = {"gemv": INT8_GEMV, "few": INT8_FEW, "tile": INT8_TILE}


def _type(name):
    try:
        return _lib.TYPES[name]
    except KeyError:
        raise ValueError("no value type %r (bf16, fp16, fp32)" % (name,)) from None


def quantise_rows(m, k, dX, dQ, dScale, dtype="bf16", ldx=None, ldq=None, device=0, stream=None):
    """Rows of x (m x k) to 8 bits: scale[i] = max|x[i]| / 127, q = x / scale rounded half to even, exactly (wg_quantise_rows).
    For `Int8Plan`, give q rows a multiple of 16 bytes apart."""
    check(_lib.lib().wg_quantise_rows(device, m, k, _type(dtype), dX, k if ldx is None else ldx, dQ, k if ldq is None else ldq, dScale, stream),
          "wg_quantise_rows")


def norm_quantise_rows(m, k, dX, dW, eps, dQ, dScale, dR=None, dH=None, dtype="bf16", ldx=None, ldr=None, ldh=None, ldq=None, device=0, stream=None):
    """The root-mean-square norm of h = x (+ r, written to dH; it may be x or r itself), times w, to 8 bits with a scale a row
    (wg_norm_quantise_rows).  dR and dH come together or not at all."""
    check(_lib.lib().wg_norm_quantise_rows(device, m, k, _type(dtype), dX, k if ldx is None else ldx, dR, k if ldr is None else ldr, dW, eps,
                                           dH, k if ldh is None else ldh, dQ, k if ldq is None else ldq, dScale, stream), "wg_norm_quantise_rows")


def int8_choose(m, n, k):
    """The program the rule picks for m tokens, n channels, depth k, with its launch geometry."""
    info = Int8Info()
    check(_lib.lib().wg_int8_choose(m, n, k, ctypes.byref(info)), "wg_int8_choose")
    return info


class Int8Plan:
    """A weight matrix in 8 bits: dBt (n x k, rows `ldb` bytes apart, a multiple of 16), dScaleB (n floats) and maybe dBias (n
    floats).  The plan keeps the addresses, not the values; any number of tokens per launch, and launches on several streams at
    once are fine."""
    _h = None

    def __init__(self, n, k, dBt, dScaleB, dBias=None, out="bf16", ldb=None, device=0):
        h = ctypes.c_void_p()
        check(_lib.lib().wg_int8_plan_create(device, n, k, dBt, k if ldb is None else ldb, dScaleB, dBias, _type(out), ctypes.byref(h)),
              "wg_int8_plan_create")
        self._h, self.n, self.k, self.out = h, n, k, out
        self._launch = _lib.lib().wg_int8_launch

    def launch(self, m, dA, dScaleA, dC, lda=None, ldc=None, stream=None):
        """C (m x n, rows `ldc` elements apart) = scaleA[m] scaleB[n] A Bt^T (+ bias): one asynchronous launch."""
        code = self._launch(self._h, m, dA, self.k if lda is None else lda, dScaleA, dC, self.n if ldc is None else ldc, stream)
        if code:
            check(code, "wg_int8_launch")

    def set_program(self, kernel=None, tile_m=0, tile_n=0, split=1):
        """Name the program of the launches that follow ("gemv", "few" or "tile"); None: the rule's."""
        info = None if kernel is None else ctypes.byref(Int8Info(KERNELS[kernel], tile_m, tile_n, split))
        check(_lib.lib().wg_int8_plan_set_program(self._h, info), "wg_int8_plan_set_program")

    def set_timeout_ms(self, ms):
        check(_lib.lib().wg_int8_plan_set_timeout_ms(self._h, int(ms)), "wg_int8_plan_set_timeout_ms")

    def status(self):
        """Synchronise and raise DeviceWaitError if any launch gave up."""
        st = (ctypes.c_uint * 4)()
        r = _lib.lib().wg_int8_last_device_status(self._h, ctypes.byref(st))
        if r == _lib.WG_E_DEVICE_WAIT:
            raise DeviceWaitError(list(st))
        check(r, "wg_int8_last_device_status")
        return tuple(st)

    def reset(self):
        check(_lib.lib().wg_int8_plan_reset(self._h), "wg_int8_plan_reset")

    def close(self):
        if self._h is not None:
            _lib.lib().wg_int8_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
