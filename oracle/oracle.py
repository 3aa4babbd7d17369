"""TEST INFRASTRUCTURE: ctypes front-ends of the two CPU checkers (see oracle/__init__.py)."""
import ctypes as C
import os
import subprocess

import numpy as np

from intel_gaudi3_software_b200 import abi

HERE = os.path.dirname(os.path.abspath(__file__))
PORT_SO = os.path.join(HERE, "libmme_oracle.so")
REF_SO = os.path.join(HERE, "_ref", "libmme_ref.so")
P = C.POINTER


def reference_root():
    """Where the reference's checkout lies: $MME_REFERENCE_ROOT, else a directory `reference` beside this repository.
    Returns None when there is none (the GPU box: only the prebuilt checkers travel there)."""
    root = os.environ.get("MME_REFERENCE_ROOT") or os.path.join(os.path.dirname(os.path.dirname(HERE)), "reference")
    return root if os.path.exists(os.path.join(root, "mme", "mme_reference", "mme_reference.h")) else None


def build(ref_root=None):
    """Compile the C restatement, and the reference itself when its checkout is present."""
    subprocess.check_call(["make", "-s", "-C", HERE, "port"])
    ref_root = ref_root or reference_root()
    if ref_root and os.path.exists(os.path.join(ref_root, "mme", "mme_reference", "mme_reference.h")):
        subprocess.check_call(["make", "-s", "-j8", "-C", HERE, "ref", "REF=" + ref_root])


def have_ref():
    return os.path.exists(REF_SO)


def _u32(a):
    return np.ascontiguousarray(a).view(np.uint32)


class _Base:
    prefix = ""

    def _fn(self, name, res, args):
        f = getattr(self.lib, self.prefix + name)
        f.restype, f.argtypes = res, args
        return f

    # ---- scalar/vector conversions -------------------------------------------------------
    def fp8_to_fp32(self, codes, exp_width, bias, mode):
        codes = np.ascontiguousarray(codes, dtype=np.uint8)
        out = np.empty(codes.shape, dtype=np.uint32)
        f = self._fn("fp8_to_fp32_vec", None, [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int, C.c_uint, C.c_int])
        f(codes.ctypes.data, out.ctypes.data, codes.size, exp_width, bias, mode)
        return out.view(np.float32)

    def fp32_to_fp8(self, x, exp_width, bias, rm=0, lfsr=None, ftz=False, clip=False, clip_inf_in=False,
                    stochastic_ftz=False, mode=0):
        bits = _u32(np.asarray(x, dtype=np.float32) if np.asarray(x).dtype != np.uint32 else x)
        out = np.empty(bits.shape, dtype=np.uint8)
        lf = None if lfsr is None else np.ascontiguousarray(lfsr, dtype=np.uint32)
        f = self._fn("fp32_to_fp8_vec", None, [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int, C.c_uint, C.c_int,
                                                C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int])
        f(bits.ctypes.data, out.ctypes.data, bits.size, exp_width, bias, rm, None if lf is None else lf.ctypes.data,
          int(ftz), int(clip), int(clip_inf_in), int(stochastic_ftz), mode)
        return out

    def fp32_to_bf16(self, x, rm=0, lfsr=None, clip=False, ftz=False, clip_inf_in=False):
        bits = _u32(np.asarray(x, dtype=np.float32) if np.asarray(x).dtype != np.uint32 else x)
        out = np.empty(bits.shape, dtype=np.uint16)
        lf = None if lfsr is None else np.ascontiguousarray(lfsr, dtype=np.uint32)
        f = self._fn("fp32_to_bf16_vec", None, [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int, C.c_void_p, C.c_int,
                                                 C.c_int, C.c_int])
        f(bits.ctypes.data, out.ctypes.data, bits.size, rm, None if lf is None else lf.ctypes.data, int(clip),
          int(ftz), int(clip_inf_in))
        return out

    def fp32_to_fp32(self, bits, rm=0, clip=False, ftz=False, clip_inf_in=False):
        f = self._fn("fp32_to_fp32", C.c_uint32, [C.c_uint32, C.c_int, C.c_int, C.c_int, C.c_int])
        return f(int(bits), rm, int(clip), int(ftz), int(clip_inf_in))

    def lfsr32(self, v, poly):
        f = self._fn("lfsr32", C.c_uint32, [C.c_uint32, C.c_uint32])
        return f(int(v), int(poly))


class Port(_Base):
    """The plain-C restatement (Gaudi3 model; bf16 / fp8 operands, fp32 and tf32 ones in GEMMs)."""
    prefix = "mo_"
    kind = "port"

    def __init__(self):
        if not os.path.exists(PORT_SO):
            build()
        self.lib = C.CDLL(PORT_SO)

    def hardware_threads(self):
        return self._fn("hardware_threads", C.c_int, [])()

    def fma_vec(self, type_a, type_b, a, b, bias_a=0, bias_b=0, mode_a=0, mode_b=0):
        a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
        f = self._fn("fma_vec", C.c_float, [C.c_int, C.c_int, C.c_uint, C.c_uint, C.c_int, C.c_int, C.c_void_p,
                                            C.c_void_p, C.c_uint])
        return f(type_a, type_b, bias_a, bias_b, mode_a, mode_b, a.ctypes.data, b.ctypes.data, a.size)

    def bgemm(self, out, x, w, op, threads=0, chip=abi.CHIP_GAUDI3):
        assert chip == abi.CHIP_GAUDI3, "the port restates the Gaudi3 model only"
        f = self._fn("bgemm", C.c_int, [C.c_int, P(abi.Tensor), P(abi.Tensor), P(abi.Tensor), C.c_int])
        return f(threads, out, x, w, op)

    def conv(self, out, x, w, y, params, op, rm=0, threads=0, chip=abi.CHIP_GAUDI3):
        assert chip == abi.CHIP_GAUDI3
        f = self._fn("conv", C.c_int, [C.c_int, P(abi.Tensor), P(abi.Tensor), P(abi.Tensor), P(abi.Tensor),
                                       P(abi.ConvParams), C.c_int, C.c_int])
        return f(threads, out, x, w, y, params, op, rm)

    def activation(self, out, acc, cast, lfsr, polynomial, chip=abi.CHIP_GAUDI3, seed=0):
        lfsr = np.ascontiguousarray(lfsr, dtype=np.uint32)
        f = self._fn("activation", C.c_int, [P(abi.Tensor), P(abi.Tensor), P(abi.CastParams), C.c_void_p, C.c_uint32,
                                             C.c_uint32])
        rc = f(out, acc, cast, lfsr.ctypes.data, lfsr.size, polynomial)
        return rc, lfsr

    def memory_write(self, mem, mme_out, op, rm=0, clip=False, chip=abi.CHIP_GAUDI3):
        f = self._fn("memory_write", C.c_int, [P(abi.Tensor), P(abi.Tensor), C.c_int, C.c_int, C.c_int])
        return f(mem, mme_out, op, rm, int(clip))


class Ref(_Base):
    """The unmodified reference calculator, compiled from its own sources."""
    prefix = "ref_"
    kind = "reference"

    def __init__(self):
        if not os.path.exists(REF_SO):
            raise RuntimeError("oracle/_ref/libmme_ref.so is not built (needs the reference checkout)")
        self.lib = C.CDLL(REF_SO)

    def hardware_threads(self):
        return self._fn("hardware_threads", C.c_int, [])()

    def fma_vec(self, type_a, type_b, a, b, bias_a=0, bias_b=0, mode_a=0, mode_b=0, chip=abi.CHIP_GAUDI3):
        a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
        f = self._fn("fma_vec", C.c_float, [C.c_int, C.c_int, C.c_int, C.c_uint, C.c_uint, C.c_int, C.c_int,
                                            C.c_void_p, C.c_void_p, C.c_uint])
        return f(chip, type_a, type_b, bias_a, bias_b, mode_a, mode_b, a.ctypes.data, b.ctypes.data, a.size)

    def bgemm(self, out, x, w, op, threads=0, chip=abi.CHIP_GAUDI3):
        f = self._fn("bgemm", C.c_int, [C.c_int, C.c_int, P(abi.Tensor), P(abi.Tensor), P(abi.Tensor), C.c_int])
        return f(chip, threads, out, x, w, op)

    def conv(self, out, x, w, y, params, op, rm=0, threads=0, chip=abi.CHIP_GAUDI3):
        f = self._fn("conv", C.c_int, [C.c_int, C.c_int, P(abi.Tensor), P(abi.Tensor), P(abi.Tensor), P(abi.Tensor),
                                       P(abi.ConvParams), C.c_int, C.c_int])
        return f(chip, threads, out, x, w, y, params, op, rm)

    def activation(self, out, acc, cast, lfsr, polynomial, chip=abi.CHIP_GAUDI3, seed=0):
        lfsr = np.ascontiguousarray(lfsr, dtype=np.uint32).copy()
        # the reference advances its private copy; replay the advance for the caller
        f = self._fn("activation", C.c_int, [C.c_int, P(abi.Tensor), P(abi.Tensor), P(abi.CastParams), C.c_void_p,
                                             C.c_uint32, C.c_uint32, C.c_uint])
        rc = f(chip, out, acc, cast, lfsr.ctypes.data, lfsr.size, polynomial, seed)
        return rc, lfsr

    def memory_write(self, mem, mme_out, op, rm=0, clip=False, chip=abi.CHIP_GAUDI3):
        f = self._fn("memory_write", C.c_int, [C.c_int, P(abi.Tensor), P(abi.Tensor), C.c_int, C.c_int, C.c_int])
        return f(chip, mem, mme_out, op, rm, int(clip))

    def compare_elements(self, dtype, bias, mode, cd, a, b):
        """TensorComparator::doCompare element by element: array of 0/1 (1 = the reference calls them equal)."""
        a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
        out = np.zeros(a.size, np.uint8)
        f = self._fn("compare_elements", None, [C.c_int, C.c_uint, C.c_int, C.c_uint, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p])
        f(dtype, bias, mode, cd, a.ctypes.data, b.ctypes.data, a.size, out.ctypes.data)
        return out

    def compare(self, a, b, cd, num_partials=1):
        f = self._fn("compare", C.c_int, [P(abi.Tensor), P(abi.Tensor), C.c_uint, C.c_uint])
        return bool(f(a, b, cd, num_partials))
