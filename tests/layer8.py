"""Plain forms of the 8-bit layer operators for the tests, in 64 bits (and, for what the definition fixes bit for bit, in
correctly rounded 32-bit arithmetic), with the error bounds of the 32-bit kernels derived from their operation counts.

U is the relative error of one rounding to 32 bits. A sum of n terms in which no term passes through more than d additions is
off by at most d * U * sum|terms| (to first order)."""
import numpy as np

from intel_gaudi3_software_b200 import abi

U = 2.0 ** -24
# half a step of the output types, relative
HALF = {abi.BF16: 2.0 ** -8, abi.FP32: 2.0 ** -24}
# Additions a term of a row's sum passes through: the values of its thread (two interleaved sums: half of at most 32 up to
# 16384 columns, eight for every 4096 columns above), the two sums' join, five levels over the warp, at most 32 warps.


def row_depth(cols):
    return max(32, 8 * -(-cols // 4096)) + 1 + 5 + 32


def top_of(dtype, bias=7, mode=abi.INFNAN_MINIMAL):
    if dtype == abi.INT8:
        return 127.0
    if dtype == abi.FP8_152:
        return 57344.0 * 2.0 ** (15 - bias)
    return {abi.INFNAN_FULL: 240.0, abi.INFNAN_NONE: 480.0, abi.INFNAN_MINIMAL: 448.0}[mode] * 2.0 ** (7 - bias)


def codes_of(v, dtype, port, bias=7, mode=abi.INFNAN_MINIMAL, given=None):
    """(codes, steps) of the rows of v (float32), in 32-bit arithmetic as defined; fp8 codes through the oracle's cast."""
    v = np.asarray(v, np.float32)
    top = np.float32(top_of(dtype, bias, mode))
    with np.errstate(all="ignore"):
        if given is None:
            step = (np.abs(v).max(axis=1) / top).astype(np.float32)
        else:
            step = np.broadcast_to(np.asarray(given, np.float32), (v.shape[0],))
        ok = (step > 0) & np.isfinite(step)
        t = (v / np.where(ok, step, np.float32(1))[:, None]).astype(np.float32)
        if dtype == abi.INT8:
            q = np.where(np.isnan(t), 0, np.clip(np.rint(t), -127, 127)).astype(np.int8)
        else:
            q = port.fp32_to_fp8(np.ascontiguousarray(t).reshape(-1), 4 if dtype == abi.FP8_143 else 5, bias, abi.RM_NE, None, False, True, True, False, mode).reshape(t.shape)
        q = np.where(ok[:, None], q, np.zeros_like(q))
        if given is None:
            step = np.where(np.isfinite(step), step, np.float32(np.nan))
    return q, step


def norm(h, gamma, eps):
    """(h / rms * gamma, 1 / rms) in 64 bits."""
    h = h.astype(np.float64)
    inv = 1.0 / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps)
    return h * inv * gamma.astype(np.float64), inv[:, 0]


def inverse_bound(cols):
    """Relative error of 1 / rms: half the sum's, and one rounding each for the quotient, eps, root and reciprocal."""
    return (row_depth(cols) / 2 + 4) * U


def norm_grad(x, gamma, dy, dsum, eps):
    x, g, dy = x.astype(np.float64), gamma.astype(np.float64), dy.astype(np.float64)
    inv = 1.0 / np.sqrt((x * x).mean(axis=1, keepdims=True) + eps)
    u, a = x * inv, dy * g
    dx = (a - u * (a * u).mean(axis=1, keepdims=True)) * inv
    return (dx if dsum is None else dx + dsum.astype(np.float64)), (dy * u).sum(axis=0)


def norm_grad_bounds(x, gamma, dy, dsum, eps, out_dtype):
    """Error bounds of dx and dgamma, element by element."""
    x, g, dy = x.astype(np.float64), gamma.astype(np.float64), dy.astype(np.float64)
    rows, cols = x.shape
    inv = 1.0 / np.sqrt((x * x).mean(axis=1, keepdims=True) + eps)
    u, a = np.abs(x * inv), np.abs(dy * g)
    mean_abs = (a * u).mean(axis=1, keepdims=True)
    ib = inverse_bound(cols)
    # dx = (a - u * mean) * inv + dsum: `a` and `u` carry one rounding and inv's error, the mean its sum's error and inv's,
    # and every operation of the line one rounding more
    b = inv * (a * (ib + 4 * U) + u * mean_abs * (3 * ib + (row_depth(cols) + 8) * U))
    dx, dg = norm_grad(x, gamma, dy, dsum, eps)
    b = b + (0 if dsum is None else 2 * U * np.abs(dsum.astype(np.float64))) + (HALF[out_dtype] * (np.abs(dx) + b)) + 1e-38
    return b, (np.abs(dy) * u).sum(axis=0) * (ib + (rows + 4) * U) + 1e-38


def product(x, xs, w, ws, bias):
    """(result, sum of |terms| scaled) in 64 bits; x and w are decoded values."""
    acc = x.astype(np.float64) @ w.astype(np.float64).T
    scale = np.asarray(xs, np.float64).reshape(-1, 1) * np.asarray(ws, np.float64).reshape(1, -1)
    y = acc * scale
    mag = (np.abs(x.astype(np.float64)) @ np.abs(w.astype(np.float64)).T) * np.abs(scale)
    return y, (y if bias is None else y + bias.astype(np.float64)), mag


def product_bound(y, out, mag, out_dtype, integer, acc_tol=1e-5):
    """Integer sums are exact: the conversion, two products, the bias and the output are one rounding each. fp8 sums are within
    the library's accumulator tolerance of sum|terms|."""
    b = np.abs(y) * 3 * U + (0 if integer else acc_tol * mag)
    return b + (U + HALF[out_dtype]) * (np.abs(out) + b) + 1e-38
