"""The 8-bit layer operators on the GPU: RMS norm with the residual's addition and 8-bit rows, its gradient, quantisation,
scaled products, and a run of them together. Bounds: tests/layer8.py."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from intel_gaudi3_software_b200 import MmeError, abi
from intel_gaudi3_software_b200.abi import make_tensor as T
import layer8
import util

pytestmark = pytest.mark.gpu
EPS = 1e-5
FP8 = {"fp_bias": 7, "inf_nan_mode": abi.INFNAN_MINIMAL}


def fp8_kw(dtype, bias=7, mode=abi.INFNAN_MINIMAL):
    return {"fp_bias": bias, "inf_nan_mode": mode} if dtype in (abi.FP8_143, abi.FP8_152) else {}


def encode(v, dtype):
    """(storage array, its values in float32)."""
    v = np.asarray(v, np.float32)
    if dtype == abi.FP32:
        return np.ascontiguousarray(v), v
    b = util.f32_to_bf16_rne(np.ascontiguousarray(v).reshape(-1)).reshape(v.shape)
    return b, util.bf16_to_f32(b.reshape(-1)).reshape(v.shape)


def decode(a, dtype):
    return a.astype(np.float32) if dtype == abi.FP32 else util.bf16_to_f32(np.ascontiguousarray(a).reshape(-1)).reshape(a.shape)


def rows_like(rng, rows, cols, scale=1.0):
    """Activations: channels of different spread, some of them far out."""
    s = np.exp(0.5 * rng.standard_normal(cols))
    s[:: max(1, cols // 4)] *= 20
    return (rng.standard_normal((rows, cols)) * s * scale).astype(np.float32)


class Dev:
    """Device images of host arrays for one test: strided rows, offsets, guard bytes around outputs."""

    def __init__(self, calc):
        self.calc, self.bufs = calc, []

    def put(self, array, dtype, pitch=None, offset=0, **kw):
        """[rows, cols] (or [cols]) array as a tensor with `pitch` elements between rows, `offset` elements into its buffer."""
        a = np.atleast_2d(array)
        rows, cols = a.shape
        pitch = cols if pitch is None else pitch
        store = np.full(offset + max(rows, 1) * max(pitch, 1) + 64, 0x55, a.dtype) if a.dtype != np.float32 else np.full(offset + max(rows, 1) * max(pitch, 1) + 64, -777.0, np.float32)
        for r in range(rows):
            store[offset + r * pitch:offset + r * pitch + cols] = a[r]
        buf = self.calc.to_device(store)
        self.bufs.append(buf)
        sizes = [cols, rows] if np.ndim(array) == 2 else [cols]
        strides = [1, pitch] if np.ndim(array) == 2 else [1]
        t = T(buf.ptr + offset * a.dtype.itemsize, dtype, sizes, strides, mem_space=abi.MEM_DEVICE, **kw)
        t.store, t.buf, t.place, t.kind = store, buf, (rows, cols, pitch, offset), a.dtype
        return t

    def get(self, t):
        """The tensor's rows; everything around them must be as it was."""
        rows, cols, pitch, offset = t.place
        now = t.buf.download(t.kind)[: t.store.size]
        keep = np.ones(t.store.size, bool)
        out = np.zeros((rows, cols), t.kind)
        for r in range(rows):
            out[r] = now[offset + r * pitch:offset + r * pitch + cols]
            keep[offset + r * pitch:offset + r * pitch + cols] = False
        assert (now[keep].view(np.uint8) == t.store[keep].view(np.uint8)).all(), "bytes outside the tensor were written"
        return out

    def free(self):
        self.calc.sync()
        for b in self.bufs:
            b.free()


@pytest.fixture
def dev(calc):
    d = Dev(calc)
    yield d
    d.free()


# ------------------------------------------------------------------------------------------ RMS norm
def check_norm(calc, dev, port, rows, cols, xt, rt, gt, ot, seed=0, pitch=0, offset=0, values=None, bias=7, mode=abi.INFNAN_MINIMAL):
    rng = np.random.default_rng([seed, rows, cols])
    xb, x = encode(rows_like(rng, rows, cols) if values is None else values, xt)
    gb, g = encode(1 + 0.3 * rng.standard_normal(cols), gt if gt is not None else abi.FP32)
    if gt is None:
        g = np.ones(cols, np.float32)
    p = cols + pitch
    tx = dev.put(xb, xt, p, offset)
    tg = None if gt is None else dev.put(gb, gt)
    tr = ts = None
    h = x
    if rt is not None:
        rb, r = encode(rows_like(rng, rows, cols, 3.0), rt)
        tr, ts = dev.put(rb, rt, p, offset), dev.put(np.zeros_like(rb), rt, p, offset)
        sb, h = encode((x + r).astype(np.float32), rt)
    to = dev.put(np.zeros((rows, cols), abi.NP_DTYPE[ot]), ot, p, offset, **fp8_kw(ot, bias, mode))
    eight = ot in (abi.INT8, abi.FP8_143, abi.FP8_152)
    tsc = dev.put(np.zeros(rows, np.float32), abi.FP32) if eight else None
    calc.rms_norm(to, tx, tg, EPS, residual=tr, sum=ts, scale=tsc)
    calc.sync()
    if rt is not None:
        assert (dev.get(ts).view(np.uint8) == np.ascontiguousarray(sb).view(np.uint8)).all()
    got = dev.get(to)
    with np.errstate(all="ignore"):
        ref, inv = layer8.norm(h, g, EPS)
        ib = layer8.inverse_bound(cols)
        if eight:
            codes, step = layer8.codes_of((h * g).astype(np.float32), ot, port, bias, mode)
            assert (got == codes).all()
            want = step.astype(np.float64) * inv
            sc = dev.get(tsc)[0]
            assert (np.isnan(sc) == np.isnan(step)).all()
            fine = ~np.isnan(step)
            assert (np.abs(sc - want)[fine] <= (np.abs(want) * (ib + 2 * layer8.U) + 1e-44)[fine]).all()
        else:
            v = decode(got, ot).astype(np.float64)
            bound = np.abs(ref) * (ib + 2 * layer8.U)
            assert (np.abs(v - ref) <= bound + layer8.HALF[ot] * (np.abs(ref) + bound) + 1e-38).all()


COLS = [1, 2, 7, 8, 31, 64, 255, 256, 257, 1000, 1024, 1032, 2048, 2051, 4096, 4104, 4999, 8192, 8200, 16384, 16392, 16401, 28672, 32768, 32776, 33001]


@pytest.mark.parametrize("cols", COLS)
def test_norm_int8_over_lengths(calc, dev, port, cols):
    check_norm(calc, dev, port, 5, cols, abi.BF16, abi.BF16, abi.BF16, abi.INT8)


@pytest.mark.parametrize("cols", [8, 100, 1000, 2048, 4097, 8192, 16384, 20000, 40000])
@pytest.mark.parametrize("rt", [None, abi.BF16, abi.FP32])
@pytest.mark.parametrize("xt", [abi.BF16, abi.FP32])
def test_norm_types(calc, dev, port, cols, xt, rt):
    for ot, gt in ((abi.INT8, abi.FP32), (abi.FP8_143, abi.BF16), (abi.BF16, abi.BF16), (abi.FP32, None), (abi.BF16, abi.FP32)):
        check_norm(calc, dev, port, 3, cols, xt, rt, gt, ot, seed=1)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 149, 600])
def test_norm_rows(calc, dev, port, rows):
    check_norm(calc, dev, port, rows, 96, abi.BF16, abi.BF16, abi.FP32, abi.INT8, seed=2)
    check_norm(calc, dev, port, rows, 1100, abi.BF16, None, abi.FP32, abi.BF16, seed=2)


@pytest.mark.parametrize("pitch,offset", [(0, 1), (3, 0), (8, 0), (16, 8), (24, 5)])
@pytest.mark.parametrize("cols", [64, 520, 1504, 5000])
def test_norm_strided_rows_and_offsets(calc, dev, port, cols, pitch, offset):
    check_norm(calc, dev, port, 7, cols, abi.BF16, abi.BF16, abi.BF16, abi.INT8, seed=3, pitch=pitch, offset=offset)
    check_norm(calc, dev, port, 7, cols, abi.FP32, None, abi.FP32, abi.FP8_143, seed=3, pitch=pitch, offset=offset)


@pytest.mark.parametrize("ot,bias,mode", [(abi.FP8_143, 7, abi.INFNAN_MINIMAL), (abi.FP8_143, 11, abi.INFNAN_MINIMAL), (abi.FP8_143, 3, abi.INFNAN_FULL),
                                          (abi.FP8_143, 15, abi.INFNAN_NONE), (abi.FP8_152, 15, abi.INFNAN_FULL), (abi.FP8_152, 20, abi.INFNAN_FULL)])
def test_norm_fp8_conventions(calc, dev, port, ot, bias, mode):
    check_norm(calc, dev, port, 9, 1216, abi.BF16, abi.BF16, abi.FP32, ot, seed=4, bias=bias, mode=mode)
    check_norm(calc, dev, port, 9, 1217, abi.FP32, None, abi.FP32, ot, seed=4, bias=bias, mode=mode)


def test_norm_codes_next_to_a_tie(calc, dev, port):
    """Values placed on and next to the middles between two codes: the codes are the correctly rounded quotient's."""
    cols = 512
    steps = np.float32([1.0, 0.37, 3.0e-5, 1.7e12, 1.1e-30, 2.0 ** -126, 2.0 ** -127, 1.5e-39, 2.3e36])
    v = np.zeros((steps.size, cols), np.float32)
    k = np.arange(cols - 1) // 4 - 63.5
    for i, s in enumerate(steps):
        t = (k * np.float64(s)).astype(np.float32)
        v[i, 1:] = np.where(np.arange(cols - 1) % 4 == 0, t, np.where(np.arange(cols - 1) % 4 == 1, np.nextafter(t, np.float32(np.inf)),
                            np.where(np.arange(cols - 1) % 4 == 2, np.nextafter(t, np.float32(-np.inf)), t * np.float32(1 + 2.0 ** -20))))
        v[i, 0] = np.float32(127) * s
    for ot in (abi.INT8, abi.FP8_143):
        codes, step = layer8.codes_of(v, ot, port)
        tx, to, ts = dev.put(v, abi.FP32), dev.put(np.zeros(v.shape, abi.NP_DTYPE[ot]), ot, **fp8_kw(ot)), dev.put(np.zeros(len(v), np.float32), abi.FP32)
        calc.quantize(to, ts, tx)
        calc.sync()
        assert (dev.get(ts)[0] == step).all() and (dev.get(to) == codes).all()


@pytest.mark.parametrize("cols", [40, 1536, 33000])
@pytest.mark.parametrize("ot", [abi.INT8, abi.FP8_143])
def test_norm_zero_rows_and_rows_that_hold_no_number(calc, dev, port, cols, ot):
    rng = np.random.default_rng(5)
    v = rows_like(rng, 8, cols)
    v[1] = 0
    v[2, cols // 2] = np.nan
    v[3, 0] = np.inf
    v[4, cols - 1] = -np.inf
    v[5] = 1e-42
    v[6] *= 1e-41
    check_norm(calc, dev, port, 8, cols, abi.FP32, None, None, ot, values=v)


@pytest.mark.parametrize("cols", [5, 41, 249, 257, 1019, 4999, 16381, 33001])
@pytest.mark.parametrize("ot", [abi.INT8, abi.FP8_143, abi.BF16])
def test_rows_of_odd_length_do_not_see_their_neighbours(calc, dev, port, cols, ot):
    """Rows one behind the other: the words at a row's ends hold its neighbours' values too, here numbers and no numbers in turn."""
    rng = np.random.default_rng([21, cols])
    v = rows_like(rng, 17, cols)
    v[1::2] = np.nan
    v[3::4] = -np.inf
    if ot != abi.BF16:
        check_norm(calc, dev, port, 17, cols, abi.BF16, None, abi.FP32, ot, values=v)
        check_norm(calc, dev, port, 17, cols, abi.FP32, None, abi.BF16, ot, values=v)
        return
    tx, to = dev.put(encode(v, abi.BF16)[0], abi.BF16), dev.put(np.zeros((17, cols), np.uint16), abi.BF16)
    calc.rms_norm(to, tx, None, EPS)
    calc.sync()
    out, x = decode(dev.get(to), abi.BF16), encode(v, abi.BF16)[1]
    want = layer8.norm(x[::2], np.ones(cols), EPS)[0]
    # (one rounding to bf16, and the reciprocal root's error, far below it)
    assert (np.abs(out[::2] - want) <= np.abs(want) * (2.0 ** -8 + 2 * layer8.inverse_bound(cols))).all()
    assert np.isnan(out[1::2]).all()


def test_norm_float_rows_that_hold_no_number(calc, dev):
    v = np.ones((3, 300), np.float32)
    v[0, 7] = np.nan
    v[1, 8] = np.inf
    tx, to = dev.put(v, abi.FP32), dev.put(np.zeros_like(v), abi.FP32)
    calc.rms_norm(to, tx, None, EPS)
    calc.sync()
    out = dev.get(to)
    assert np.isnan(out[0]).all()
    assert np.isnan(out[1, 8]) and (np.delete(out[1], 8) == 0).all()      # inf * 0; the rest is finite * 0
    assert np.abs(out[2] - 1).max() < 1e-5


def test_eps_of_every_finite_size(calc, dev):
    """eps = 0 and the largest float are finite and not negative. With the largest, mean(h^2) is below its last place: the root is
    eps's own, up to its rounding, the reciprocal's and the product's."""
    most = np.finfo(np.float32).max
    v = np.float32([[3, -4, 0, 5], [1, 1, -1, 1]])
    tx, to, td = dev.put(v, abi.FP32), dev.put(np.zeros_like(v), abi.FP32), dev.put(np.zeros_like(v), abi.FP32)
    for eps in (0.0, float(most)):
        calc.rms_norm(to, tx, None, eps)
        calc.rms_norm_grad(td, None, tx, tx, None, eps)
        calc.sync()
        ref, _ = layer8.norm(v, np.ones(4), eps)
        assert (np.abs(dev.get(to) - ref) <= np.abs(ref) * (layer8.inverse_bound(4) + 2 * layer8.U)).all()
        dx, _ = layer8.norm_grad(v, np.ones(4), v, None, eps)
        assert (np.abs(dev.get(td) - dx) <= layer8.norm_grad_bounds(v, np.ones(4), v, None, eps, abi.FP32)[0]).all()


@pytest.mark.parametrize("cols", [40, 5000])
def test_norm_of_rows_whose_squares_leave_32_bits(calc, dev, cols):
    """As the header says: an infinite mean square gives zeros (scale 0), a vanishing one with eps = 0 no numbers (scale infinite).
    The codes are those of h * gamma all the same."""
    v = np.ones((2, cols), np.float32)
    v[0] *= np.float32(1e20)
    v[1] *= np.float32(1e-30)
    tx, to = dev.put(v, abi.FP32), dev.put(np.ones_like(v), abi.FP32)
    tq, ts = dev.put(np.zeros((2, cols), np.int8), abi.INT8), dev.put(np.ones(2, np.float32), abi.FP32)
    calc.rms_norm(to, tx, None, 0.0)
    calc.rms_norm(tq, tx, None, 0.0, scale=ts)
    calc.sync()
    assert (dev.get(to)[0] == 0).all() and np.isinf(dev.get(to)[1]).all()
    assert (dev.get(tq) == 127).all() and list(dev.get(ts)[0]) == [0.0, np.inf]


@pytest.mark.parametrize("cols", [64, 2056, 9001, 40000])
def test_norm_in_place(calc, dev, cols):
    """sum over residual, out over x: the same values as with tensors of their own."""
    rng = np.random.default_rng(6)
    xb, _ = encode(rows_like(rng, 6, cols), abi.BF16)
    rb, _ = encode(rows_like(rng, 6, cols), abi.BF16)
    gb, _ = encode(1 + 0.1 * rng.standard_normal(cols), abi.BF16)
    tg = dev.put(gb, abi.BF16)
    apart = [dev.put(a, abi.BF16) for a in (xb, rb, np.zeros_like(xb), np.zeros_like(xb))]
    calc.rms_norm(apart[2], apart[0], tg, EPS, residual=apart[1], sum=apart[3])
    tx, tr = dev.put(xb, abi.BF16), dev.put(rb, abi.BF16)
    calc.rms_norm(tx, tx, tg, EPS, residual=tr, sum=tr)
    t2, r2 = dev.put(xb, abi.BF16), dev.put(rb, abi.BF16)
    calc.rms_norm(r2, t2, tg, EPS, residual=r2, sum=t2)
    calc.sync()
    out, total = dev.get(apart[2]), dev.get(apart[3])
    for o, s in ((tx, tr), (r2, t2)):
        assert (dev.get(o) == out).all() and (dev.get(s) == total).all()


@pytest.mark.parametrize("cols", [71, 72, 1504, 20001])
def test_tensors_between_each_other_s_rows(calc, dev, cols):
    """x, residual, sum and out (then x, dy, dsum and dx) as column ranges of one matrix, against 64 bits, and nothing else of the
    matrix touched. Ranges that share a column are refused, host ranges that cross too."""
    rng = np.random.default_rng([21, cols])
    rows, pitch = 9, 4 * cols + 3
    (ab, a), (bb, b), (cb, c) = (encode(rows_like(rng, rows, cols), abi.BF16) for _ in range(3))
    gb, g = encode(1 + 0.1 * rng.standard_normal(cols), abi.FP32)
    tg, z, rest = dev.put(gb, abi.FP32), np.zeros_like(ab), np.full((rows, 3), 7, np.uint16)

    def ranges(parts):
        whole = dev.put(np.hstack(parts + [rest]), abi.BF16)
        return whole, [T(whole.data + 2 * i * cols, abi.BF16, [cols, rows], [1, pitch], mem_space=abi.MEM_DEVICE) for i in range(4)]

    whole, (x, res, s, o) = ranges([ab, bb, z, z])
    calc.rms_norm(o, x, tg, EPS, residual=res, sum=s)
    calc.sync()
    got, (sb, h) = dev.get(whole), encode((a + b).astype(np.float32), abi.BF16)
    assert (np.delete(got, np.s_[3 * cols:4 * cols], axis=1) == np.hstack([ab, bb, sb, rest])).all()
    ref, _ = layer8.norm(h, g, EPS)
    bound = np.abs(ref) * (layer8.inverse_bound(cols) + 2 * layer8.U)
    assert (np.abs(decode(got[:, 3 * cols:4 * cols], abi.BF16) - ref) <= bound + layer8.HALF[abi.BF16] * (np.abs(ref) + bound) + 1e-38).all()
    whole, (x, dy, ds, d) = ranges([ab, bb, cb, z])
    calc.rms_norm_grad(d, None, dy, x, tg, EPS, dsum=ds)
    calc.sync()
    got = dev.get(whole)
    assert (np.delete(got, np.s_[3 * cols:4 * cols], axis=1) == np.hstack([ab, bb, cb, rest])).all()
    dx, _ = layer8.norm_grad(a, g, b, c, EPS)
    assert (np.abs(decode(got[:, 3 * cols:4 * cols], abi.BF16) - dx) <= layer8.norm_grad_bounds(a, g, b, c, EPS, abi.BF16)[0]).all()
    with pytest.raises(MmeError, match="overlap"):
        calc.rms_norm(T(d.data - 2, abi.BF16, [cols, rows], [1, pitch], mem_space=abi.MEM_DEVICE), x, tg, EPS, residual=dy, sum=ds)
    h = np.zeros((rows, 2 * cols), np.uint16)
    with pytest.raises(MmeError, match="overlap"):
        calc.rms_norm(T(h[:, cols:], abi.BF16, [cols, rows], [1, 2 * cols]), T(h, abi.BF16, [cols, rows], [1, 2 * cols]), None, EPS)


def test_norm_in_five_dimensions(calc, dev, port):
    """Rows spread over four outer dimensions whose strides do not merge, in another order than the sizes."""
    rng = np.random.default_rng(7)
    cols, dims = 72, (3, 2, 4, 2)
    rows = int(np.prod(dims))
    strides = [1, 80, 80 * 3 * 4, 80 * 3, 80 * 3 * 4 * 2 + 16]     # dims 2 and 3 exchanged in memory, a gap before dim 4
    place = [sum(i * s for i, s in zip(idx, strides[1:])) for idx in ((a, b, c, d) for d in range(2) for c in range(4) for b in range(2) for a in range(3))]
    size = max(place) + cols + 8
    vals = rows_like(rng, rows, cols)
    store = np.full(size, -5.0, np.float32)
    for r, at in enumerate(place):
        store[at:at + cols] = vals[r]
    bx, bo, bs = calc.to_device(store), calc.to_device(np.full(size, 0x33, np.uint8)), calc.to_device(np.zeros(rows, np.float32))
    tx = T(bx.ptr, abi.FP32, [cols, *dims], strides, mem_space=abi.MEM_DEVICE)
    to = T(bo.ptr, abi.INT8, [cols, *dims], strides, mem_space=abi.MEM_DEVICE)
    ts = T(bs.ptr, abi.FP32, [1, *dims], mem_space=abi.MEM_DEVICE)
    calc.quantize(to, ts, tx)
    calc.sync()
    codes, step = layer8.codes_of(vals, abi.INT8, port)
    raw = bo.download(np.int8)
    assert (bs.download(np.float32) == step).all()
    keep = np.ones(raw.size, bool)
    for r, at in enumerate(place):
        assert (raw[at:at + cols] == codes[r]).all()
        keep[at:at + cols] = False
    assert (raw[keep] == 0x33).all()
    for b in (bx, bo, bs):
        b.free()


@pytest.mark.parametrize("cols", [96, 3000, 20001])
@pytest.mark.parametrize("ot", [abi.INT8, abi.FP8_143])
@pytest.mark.parametrize("one", [True, False])
def test_norm_given_scales(calc, dev, port, cols, ot, one):
    """Codes of the finished rows under scales the caller brings. 1 / rms carries an error, so a code may be the neighbour
    where the quotient lies within that error of a middle; elsewhere it is the defined one."""
    rng = np.random.default_rng(8)
    rows = 6
    xb, x = encode(rows_like(rng, rows, cols), abi.BF16)
    gb, g = encode(1 + 0.3 * rng.standard_normal(cols), abi.FP32)
    sc = np.float32([0.05]) if one else np.float32([0.05, 0.2, 1e-3, 0.0, np.nan, -1.0])
    tx, tg, ts = dev.put(xb, abi.BF16), dev.put(gb, abi.FP32), dev.put(sc, abi.FP32)
    to = dev.put(np.zeros((rows, cols), abi.NP_DTYPE[ot]), ot, **fp8_kw(ot))
    calc.rms_norm(to, tx, tg, EPS, scale=ts, scale_mode=abi.SCALE_GIVEN)
    calc.sync()
    got = dev.get(to)
    assert (dev.get(ts)[0].view(np.uint32) == sc.view(np.uint32)).all()
    ref, _ = layer8.norm(x, g, EPS)
    tol = layer8.inverse_bound(cols) + 4 * layer8.U
    lo, _ = layer8.codes_of((ref * (1 - tol)).astype(np.float32), ot, port, given=sc)
    hi, _ = layer8.codes_of((ref * (1 + tol)).astype(np.float32), ot, port, given=sc)
    assert ((got == lo) | (got == hi)).all() and (lo == hi).mean() > 0.999


def test_quantize_given_scale_values(calc, dev, port):
    v = np.float32([[0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, 127.5, 1e30, -1e30, np.inf, -np.inf, np.nan, 3.49, 3.51, -128]])
    for ot in (abi.INT8, abi.FP8_143):
        for pad in (v, np.hstack([v, v[:, :3]])):
            tx, ts = dev.put(pad, abi.FP32), dev.put(np.float32([1.0]), abi.FP32)
            to = dev.put(np.zeros(pad.shape, abi.NP_DTYPE[ot]), ot, **fp8_kw(ot))
            calc.quantize(to, ts, tx, scale_mode=abi.SCALE_GIVEN)
            calc.sync()
            want, _ = layer8.codes_of(pad, ot, port, given=[1.0])
            assert (dev.get(to) == want).all()


# ------------------------------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 300), (300, 1), (63, 65), (64, 64), (65, 63), (130, 1000), (1000, 130), (2049, 40), (17, 4100), (137, 249), (128, 248), (9, 497), (265, 1001)])
@pytest.mark.parametrize("xt", [abi.BF16, abi.FP32])
def test_quantize_transposed(calc, dev, port, rows, cols, xt):
    rng = np.random.default_rng([9, rows, cols])
    v = rows_like(rng, rows, cols)
    if rows > 60 and cols > 60:
        v[5, 3], v[7, 11], v[:, 20] = np.nan, np.inf, 0
    xb, x = encode(v, xt)
    for ot, pitch, offset in ((abi.INT8, 0, 0), (abi.FP8_143, 5, 3)):
        tx = dev.put(xb, xt, cols + pitch, offset)
        to = dev.put(np.zeros((cols, rows), abi.NP_DTYPE[ot]), ot, rows + pitch, offset, **fp8_kw(ot))
        ts = dev.put(np.full(cols, 9.0, np.float32), abi.FP32)
        calc.quantize(to, ts, tx, abi.OP_TRANS)
        calc.sync()
        codes, step = layer8.codes_of(x.T, ot, port)
        sc = dev.get(ts)[0]
        assert (np.isnan(sc) == np.isnan(step)).all() and (sc[~np.isnan(step)] == step[~np.isnan(step)]).all()
        assert (dev.get(to) == codes).all()
        tg = dev.put(np.float32([0.03]), abi.FP32)
        calc.quantize(to, tg, tx, abi.OP_TRANS, abi.SCALE_GIVEN)
        calc.sync()
        assert (dev.get(to) == layer8.codes_of(x.T, ot, port, given=[0.03])[0]).all()


@pytest.mark.parametrize("pitch", [0, 3])
def test_quantize_transposed_in_several_launches(calc, pitch):
    """More rows than 65535 tiles of 128: the codes come from a second launch, the steps are of all rows. Columns whose largest
    element lies in the first launch's rows, in the second's, and in the last row."""
    rows, cols = 65535 * 128 + 131, 4
    rng = np.random.default_rng(22)
    v = rng.standard_normal((rows, cols), np.float32)
    v[5, 0], v[65535 * 128 + 3, 1], v[rows - 1, 2] = 40, -50, 60
    store = np.zeros((rows, cols + pitch), np.float32)
    store[:, :cols] = v
    bx, bo, bs = calc.to_device(store), calc.to_device(np.full((cols, rows + 5), 0x33, np.int8)), calc.to_device(np.zeros(cols, np.float32))
    calc.quantize(T(bo.ptr, abi.INT8, [rows, cols], [1, rows + 5], mem_space=abi.MEM_DEVICE), T(bs.ptr, abi.FP32, [cols], mem_space=abi.MEM_DEVICE),
                  T(bx.ptr, abi.FP32, [cols, rows], [1, cols + pitch], mem_space=abi.MEM_DEVICE), abi.OP_TRANS)
    calc.sync()
    step = (np.abs(v).max(axis=0) / np.float32(127)).astype(np.float32)
    got = bo.download(np.int8)[: cols * (rows + 5)].reshape(cols, rows + 5)
    assert (bs.download(np.float32)[:cols] == step).all()
    assert (got[:, :rows] == np.rint(v.T / step[:, None])).all() and (got[:, rows:] == 0x33).all()
    for b in (bx, bo, bs):
        b.free()


# ------------------------------------------------------------------------------------------ gradient
def grad_case(calc, dev, rows, cols, xt, gt, with_dsum, seed=0, pitch=0, offset=0, dgamma=True, workspace=False):
    rng = np.random.default_rng([seed, rows, cols])
    xb, x = encode(rows_like(rng, rows, cols), xt)
    yb, dy = encode(rng.standard_normal((rows, cols)), xt)
    gb, g = encode(1 + 0.3 * rng.standard_normal(cols), gt if gt is not None else abi.FP32)
    if gt is None:
        g = np.ones(cols, np.float32)
    sb, ds = encode(rng.standard_normal((rows, cols)), xt)
    p = cols + pitch
    tx, ty = dev.put(xb, xt, p, offset), dev.put(yb, xt, p, offset)
    ts = dev.put(sb, xt, p, offset) if with_dsum else None
    tg = None if gt is None else dev.put(gb, gt)
    to, tdg = dev.put(np.zeros_like(xb), xt, p, offset), dev.put(np.zeros(cols, np.float32), abi.FP32)
    tw = None
    if workspace:
        tw = dev.put(np.full(calc.rms_norm_grad_workspace(rows, cols) // 4, np.nan, np.float32), abi.FP32)
    calc.rms_norm_grad(to, tdg if dgamma else None, ty, tx, tg, EPS, dsum=ts, workspace=tw)
    calc.sync()
    ds = ds if with_dsum else None
    dx, dg = layer8.norm_grad(x, g, dy, ds, EPS)
    bx, bg = layer8.norm_grad_bounds(x, g, dy, ds, EPS, xt)
    assert (np.abs(decode(dev.get(to), xt) - dx) <= bx).all()
    got = dev.get(tdg)[0]
    if dgamma:
        assert (np.abs(got - dg) <= bg).all()
    else:
        assert (got == 0).all()
    return to, tdg


@pytest.mark.parametrize("cols", [1, 8, 33, 256, 264, 1000, 1024, 1100, 2048, 2500, 4096, 5001, 8192, 8200, 9001])
@pytest.mark.parametrize("xt", [abi.BF16, abi.FP32])
def test_grad_over_lengths(calc, dev, cols, xt):
    grad_case(calc, dev, 6, cols, xt, abi.FP32, True)
    grad_case(calc, dev, 7, cols, xt, abi.BF16, False, seed=1)


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 150, 700, 2600])
def test_grad_rows(calc, dev, rows):
    grad_case(calc, dev, rows, 48, abi.BF16, None, True, seed=2)
    grad_case(calc, dev, rows, 1032, abi.FP32, abi.FP32, False, seed=2, workspace=True)


@pytest.mark.parametrize("rows,cols", [(5, 8193), (40, 8200), (700, 8209), (9, 16384), (3, 20001), (2, 40000), (2, 65529), (3, 65536), (3, 65543), (2, 70001)])
def test_grad_of_rows_that_blocks_share(calc, dev, rows, cols):
    grad_case(calc, dev, rows, cols, abi.BF16, abi.FP32, True, seed=4)
    grad_case(calc, dev, rows, cols, abi.FP32, abi.BF16, False, seed=4, workspace=True)


@pytest.mark.parametrize("rows,cols", [(2601, 9), (2601, 249), (2501, 257), (1499, 1019), (1400, 1021), (613, 4099)])
def test_grad_of_odd_rows_in_many_turns(calc, dev, rows, cols):
    """A block walks several rows; all of them lie equally far past eight elements."""
    grad_case(calc, dev, rows, cols, abi.BF16, abi.BF16, True, seed=5)
    grad_case(calc, dev, rows, cols, abi.BF16, abi.FP32, False, seed=5, pitch=1, offset=3)
    grad_case(calc, dev, rows, cols, abi.FP32, None, False, seed=5)


@pytest.mark.parametrize("pitch,offset", [(0, 1), (3, 0), (8, 0), (24, 5)])
def test_grad_strided(calc, dev, pitch, offset):
    for cols in (40, 1504, 8208):
        grad_case(calc, dev, 9, cols, abi.BF16, abi.FP32, True, seed=3, pitch=pitch, offset=offset)


def test_grad_without_dgamma(calc, dev):
    for cols in (100, 3000, 9000):
        grad_case(calc, dev, 5, cols, abi.BF16, abi.BF16, True, dgamma=False)


def test_grad_against_differences(calc, dev):
    """The gradient of sum(out * c) through the library's own forward pass, against central differences of the formula."""
    rng = np.random.default_rng(10)
    rows, cols, step = 3, 24, 1e-3
    x, g, c = rng.standard_normal((rows, cols)), 1 + 0.3 * rng.standard_normal(cols), rng.standard_normal((rows, cols))
    f32 = np.float32
    tx, tg, tc = dev.put(x.astype(f32), abi.FP32), dev.put(g.astype(f32), abi.FP32), dev.put(c.astype(f32), abi.FP32)
    to, td = dev.put(np.zeros((rows, cols), f32), abi.FP32), dev.put(np.zeros(cols, f32), abi.FP32)
    calc.rms_norm_grad(to, td, tc, tx, tg, EPS)
    calc.sync()

    def loss(xx, gg):
        return (layer8.norm(xx, gg, EPS)[0] * c).sum()

    def central(xx, gg, what, i):
        lo, hi = what.copy(), what.copy()
        lo.flat[i] -= step
        hi.flat[i] += step
        return (loss(hi, gg) - loss(lo, gg)) / (2 * step) if what is xx else (loss(xx, hi) - loss(xx, lo)) / (2 * step)

    # third derivatives are of order |c| / rms^3 ~ a few: step^2 times that, and 32-bit sums
    dx, dg = dev.get(to), dev.get(td)[0]
    for i in range(rows * cols):
        assert abs(dx.flat[i] - central(x, g, x, i)) < 1e-4
    for i in range(cols):
        assert abs(dg[i] - central(x, g, g, i)) < 1e-4


def test_grad_is_reproducible_and_in_place(calc, dev):
    a = [t for t in grad_case(calc, dev, 1500, 1024, abi.BF16, abi.FP32, True, seed=4)]
    b = [t for t in grad_case(calc, dev, 1500, 1024, abi.BF16, abi.FP32, True, seed=4)]
    for s, t in zip(a, b):
        assert (dev.get(s).view(np.uint8) == dev.get(t).view(np.uint8)).all()
    rng = np.random.default_rng(11)
    for cols in (72, 2000, 9000):
        xb, _ = encode(rows_like(rng, 6, cols), abi.BF16)
        yb, _ = encode(rng.standard_normal((6, cols)), abi.BF16)
        sb, _ = encode(rng.standard_normal((6, cols)), abi.BF16)
        tx, ty, ts, to = (dev.put(v, abi.BF16) for v in (xb, yb, sb, np.zeros_like(xb)))
        calc.rms_norm_grad(to, None, ty, tx, None, EPS, dsum=ts)
        want = dev.get(to)
        for target in (tx, ty, ts):
            over = {id(t): dev.put(v, abi.BF16) for t, v in ((tx, xb), (ty, yb), (ts, sb))}
            calc.rms_norm_grad(over[id(target)], None, over[id(ty)], over[id(tx)], None, EPS, dsum=over[id(ts)])
            calc.sync()
            assert (dev.get(over[id(target)]) == want).all()


# ------------------------------------------------------------------------------------------ scaled product
def fp8_values(codes, dtype, port, bias, mode):
    return port.fp8_to_fp32(np.ascontiguousarray(codes).reshape(-1), 4 if dtype == abi.FP8_143 else 5, bias, mode).reshape(codes.shape)


def check_product(calc, dev, port, m, n, k, xt=abi.INT8, wt=None, ot=abi.BF16, bias_t=None, seed=0, xpitch=0, wpitch=0, opitch=0, xoff=0, woff=0, ooff=0,
                  one_x=False, one_w=False, extreme=False, xbias=7, wbias=7):
    wt = xt if wt is None else wt
    rng = np.random.default_rng([seed, m, n, k])

    def operand(rows, dtype, bias):
        if dtype == abi.INT8:
            q = rng.integers(-128, 128, (rows, k)) if not extreme else rng.choice([-128, 127], (rows, k))
            return q.astype(np.int8), q.astype(np.float64)
        mode = abi.INFNAN_MINIMAL if dtype == abi.FP8_143 else abi.INFNAN_FULL
        q = port.fp32_to_fp8((rng.standard_normal(rows * k) * 2.0 ** (3 - bias + (7 if dtype == abi.FP8_143 else 15))).astype(np.float32), 4 if dtype == abi.FP8_143 else 5, bias, abi.RM_NE,
                             None, False, True, True, False, mode).reshape(rows, k)
        return q, fp8_values(q, dtype, port, bias, mode)

    def kw(dtype, bias):
        return fp8_kw(dtype, bias, abi.INFNAN_MINIMAL if dtype == abi.FP8_143 else abi.INFNAN_FULL)

    xq, x = operand(m, xt, xbias)
    wq, w = operand(n, wt, wbias)
    xs = np.exp(rng.standard_normal(1 if one_x else m)).astype(np.float32)
    ws = (np.exp(rng.standard_normal(1 if one_w else n)) * 0.01).astype(np.float32)
    tb = bias = None
    if bias_t is not None:
        bb, bias = encode(rng.standard_normal(n) * 10, bias_t)
        tb = dev.put(bb, bias_t)
    tx, tw = dev.put(xq, xt, k + xpitch, xoff, **kw(xt, xbias)), dev.put(wq, wt, k + wpitch, woff, **kw(wt, wbias))
    txs, tws = dev.put(xs, abi.FP32), dev.put(ws, abi.FP32)
    to = dev.put(np.zeros((m, n), abi.NP_DTYPE[ot]), ot, n + opitch, ooff)
    calc.scaled_gemm(to, tx, txs, tw, tws, bias=tb)
    calc.sync()
    y, out, mag = layer8.product(x, xs, w, ws, bias)
    got = decode(dev.get(to), ot)
    bound = layer8.product_bound(y, out, mag, ot, xt == abi.INT8, util.ACC_TOL)
    bad = ~(np.abs(got - out) <= bound)
    assert not bad.any(), "%d of %d off, first at %s: %r, expected %r" % (bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], out[bad][0])


@pytest.mark.parametrize("k", [1, 15, 16, 17, 100, 128, 129, 512, 1024, 4096, 5008])
@pytest.mark.parametrize("m", [1, 3, 16, 17, 48])
def test_product_few_tokens(calc, dev, port, m, k):
    pad = -k % 16
    check_product(calc, dev, port, m, 300, k, xpitch=pad, wpitch=pad, bias_t=abi.FP32)
    check_product(calc, dev, port, m, 264, k, xt=abi.FP8_143, ot=abi.FP32, xpitch=pad, wpitch=pad)


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 127, 64), (2, 129, 2048), (64, 128, 2048), (100, 1000, 640), (128, 4096, 512), (200, 130, 8192), (255, 257, 1296),
                                   (256, 256, 256), (257, 300, 400), (300, 1111, 1040), (512, 512, 8192), (513, 700, 96), (1000, 40, 528)])
def test_product_shapes(calc, dev, port, m, n, k):
    check_product(calc, dev, port, m, n, k, bias_t=abi.BF16)
    check_product(calc, dev, port, m, n, k, xt=abi.FP8_143, ot=abi.FP32, bias_t=abi.FP32)


@pytest.mark.parametrize("m,n,k", [(257, 256, 128), (300, 1111, 1040), (512, 512, 2000), (777, 1001, 1504), (1025, 2050, 272), (2048, 2304, 400)])
@pytest.mark.parametrize("groups", [1, 2])
def test_product_pair_kernel(calc, dev, port, m, n, k, groups):
    calc.set_option("pair", 1)
    calc.set_option("epi_groups", groups)
    try:
        check_product(calc, dev, port, m, n, k, bias_t=abi.BF16)
        check_product(calc, dev, port, m, n, k, ot=abi.FP32, opitch=-n % 8 + 8)
        check_product(calc, dev, port, m, n, k, xt=abi.FP8_143, bias_t=abi.FP32, opitch=3, ooff=1)
    finally:
        calc.set_option("pair", -1)
        calc.set_option("epi_groups", -1)


@pytest.mark.parametrize("ctas", [1, 2])
@pytest.mark.parametrize("tile,split", [(16, 1), (16, 2), (16, 3), (32, 4), (48, 5), (64, 6), (80, 7), (128, 8), (256, 1), (256, 8), (7, 8)])
def test_product_forms_of_the_token_kernel(calc, dev, port, tile, split, ctas):
    knobs = {"pair": 0, "token_tile": tile, "token_split": split, "token_ctas": ctas}
    for name, value in knobs.items():
        calc.set_option(name, value)
    try:
        check_product(calc, dev, port, 37, 200, 1296, bias_t=abi.FP32)
        check_product(calc, dev, port, 130, 140, 2000, xt=abi.FP8_143, ot=abi.FP32)
        check_product(calc, dev, port, 5, 300, 100)   # fewer k blocks than the split asks for
    finally:
        for name in knobs:
            calc.set_option(name, -1)


def test_product_token_kernel_on_many_tiles(calc, dev, port):
    calc.set_option("pair", 0)
    try:
        check_product(calc, dev, port, 777, 1001, 1504, bias_t=abi.BF16)
        check_product(calc, dev, port, 530, 2000, 272, xt=abi.FP8_143, ot=abi.FP32)
    finally:
        calc.set_option("pair", -1)


@pytest.mark.parametrize("m,n,tile", [(65535 * 16 + 40, 5, 16), (65535 * 256 + 300, 1, -1)])
def test_product_of_more_token_tiles_than_a_grid_has(calc, m, n, tile):
    """More than 65535 tiles along the tokens take a second launch. Sums of 16 small integers: exact in fp32."""
    rng = np.random.default_rng(19)
    x, w = rng.integers(-128, 128, (m, 16)).astype(np.int8), rng.integers(-128, 128, (n, 16)).astype(np.int8)
    bufs = [calc.to_device(a) for a in (x, w, np.float32([1]), np.full((m + 1) * n, -1.0, np.float32))]
    tx, tw = T(bufs[0].ptr, abi.INT8, [16, m], mem_space=abi.MEM_DEVICE), T(bufs[1].ptr, abi.INT8, [16, n], mem_space=abi.MEM_DEVICE)
    one, to = T(bufs[2].ptr, abi.FP32, [1], mem_space=abi.MEM_DEVICE), T(bufs[3].ptr, abi.FP32, [n, m], mem_space=abi.MEM_DEVICE)
    calc.set_option("token_tile", tile)
    launches = calc.launch_count()
    try:
        calc.scaled_gemm(to, tx, one, tw, one)
    finally:
        calc.set_option("token_tile", -1)
    calc.sync()
    assert calc.launch_count() >= launches + 2   # (the plan chooses the tile where no knob does: smaller ones, more launches)
    got = bufs[3].download(np.float32).reshape(-1)[: (m + 1) * n].reshape(m + 1, n)
    assert (got[:m] == x.astype(np.float32) @ w.astype(np.float32).T).all() and (got[m] == -1).all()
    for b in bufs:
        b.free()


def test_product_int8_is_exact_at_the_range_s_ends(calc, dev, port):
    """Sums near +-2^31: the accumulator is a whole number up to the conversion."""
    check_product(calc, dev, port, 5, 140, 131071 // 16 * 16, extreme=True, ot=abi.FP32)
    rng = np.random.default_rng(12)
    m, n, k = 40, 160, 131071
    for xv, wv in ((-128, -128), (-128, 127)):
        tx, tw = dev.put(np.full((m, k), xv, np.int8), abi.INT8, k + 1), dev.put(np.full((n, k), wv, np.int8), abi.INT8, k + 1)
        one, to = dev.put(np.float32([1.0]), abi.FP32), dev.put(np.zeros((m, n), np.float32), abi.FP32)
        calc.scaled_gemm(to, tx, one, tw, one)
        calc.sync()
        assert (dev.get(to) == np.float32(xv * wv * k)).all()


@pytest.mark.parametrize("xpitch,wpitch,xoff,woff", [(0, 0, 0, 0), (1, 3, 0, 0), (0, 0, 1, 5), (11, 11, 0, 0), (11, 0, 0, 7), (27, 11, 16, 3)])
def test_product_operands_at_any_pitch_and_offset(calc, dev, port, xpitch, wpitch, xoff, woff):
    check_product(calc, dev, port, 33, 200, 1013, xpitch=xpitch, wpitch=wpitch, xoff=xoff, woff=woff)
    check_product(calc, dev, port, 300, 700, 85, xt=abi.FP8_143, xpitch=xpitch, wpitch=wpitch, xoff=xoff, woff=woff, ot=abi.FP32)


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("step,k", [(16, 64), (16, 272), (3, 100), (0, 48)])
def test_product_operands_whose_rows_share_memory(calc, dev, m, step, k):
    """Rows `step` bytes apart and longer than that: windows over one sequence."""
    rng = np.random.default_rng([20, m, step, k])
    n = 270

    def windows(rows):
        flat = rng.integers(-128, 128, step * (rows - 1) + k).astype(np.int8)
        t = dev.put(flat, abi.INT8)
        return T(t.data, abi.INT8, [k, rows], [1, step], mem_space=abi.MEM_DEVICE), np.stack([flat[step * r:step * r + k] for r in range(rows)]).astype(np.float64)

    (tx, x), (tw, w) = windows(m), windows(n)
    to, one = dev.put(np.zeros((m, n), np.float32), abi.FP32), dev.put(np.float32([1]), abi.FP32)
    calc.scaled_gemm(to, tx, one, tw, one)
    calc.sync()
    assert (dev.get(to) == x @ w.T).all()


@pytest.mark.parametrize("m", [7, 600])
def test_product_scales_for_all(calc, dev, port, m):
    check_product(calc, dev, port, m, 600, 304, one_x=True)
    check_product(calc, dev, port, m, 600, 304, one_w=True, bias_t=abi.BF16, opitch=1)
    check_product(calc, dev, port, m, 600, 304, one_x=True, one_w=True, ot=abi.FP32)


@pytest.mark.parametrize("m", [9, 520])
def test_product_fp8_types_and_biases(calc, dev, port, m):
    check_product(calc, dev, port, m, 520, 400, xt=abi.FP8_152, wt=abi.FP8_143, xbias=15, wbias=7)
    check_product(calc, dev, port, m, 520, 400, xt=abi.FP8_143, wt=abi.FP8_143, xbias=11, wbias=3, ot=abi.FP32)
    check_product(calc, dev, port, m, 520, 400, xt=abi.FP8_152, wt=abi.FP8_152, xbias=20, wbias=15)


@pytest.mark.parametrize("m,n,k", [(2048, 4096, 2048), (4097, 2048, 1024)])
def test_product_fp8_of_a_prompt(calc, dev, port, m, n, k):
    """Many tiles and several waves of them. Sums are within the library's fp8 tolerance."""
    check_product(calc, dev, port, m, n, k, xt=abi.FP8_143, bias_t=abi.BF16)
    check_product(calc, dev, port, m, n, k, xt=abi.FP8_152, wt=abi.FP8_143, xbias=15, wbias=11, ot=abi.FP32)


@pytest.mark.parametrize("xt", [abi.INT8, abi.FP8_143])
def test_product_of_nothing(calc, dev, xt):
    """K = 0: the bias, or zeros. M = 0 or N = 0: nothing."""
    kw = fp8_kw(xt)
    for ot in (abi.BF16, abi.FP32):
        to = dev.put(np.ones((5, 70), abi.NP_DTYPE[ot]), ot, 75)
        tx, tw = T(None, xt, [0, 5], mem_space=abi.MEM_DEVICE, **kw), T(None, xt, [0, 70], mem_space=abi.MEM_DEVICE, **kw)
        ts, one = dev.put(np.ones(5, np.float32), abi.FP32), dev.put(np.ones(1, np.float32), abi.FP32)
        calc.scaled_gemm(to, tx, ts, tw, one)
        calc.sync()
        assert (dev.get(to) == 0).all()
        b = np.arange(70, dtype=np.float32)
        calc.scaled_gemm(to, tx, ts, tw, one, bias=dev.put(b, abi.FP32))
        calc.sync()
        assert (decode(dev.get(to), ot) == b).all()
    calc.scaled_gemm(T(None, abi.BF16, [70, 0], mem_space=abi.MEM_DEVICE), T(None, xt, [16, 0], mem_space=abi.MEM_DEVICE, **kw), one,
                     dev.put(np.zeros((70, 16), abi.NP_DTYPE[xt]), xt, **kw), one)
    calc.rms_norm(T(None, abi.BF16, [70, 0], mem_space=abi.MEM_DEVICE), T(None, abi.BF16, [70, 0], mem_space=abi.MEM_DEVICE), None, EPS)
    td = dev.put(np.ones(70, np.float32), abi.FP32)
    empty = T(None, abi.BF16, [70, 0], mem_space=abi.MEM_DEVICE)
    calc.rms_norm_grad(empty, td, empty, empty, None, EPS)
    calc.sync()
    assert (dev.get(td) == 0).all()


def test_product_scales_that_are_no_number(calc, dev):
    """A row whose scale is NaN (it held an infinity or a NaN) gives a row of NaN, and only that row."""
    k, n = 64, 200
    for m in (4, 400):
        x, w = np.zeros((m, k), np.int8), np.ones((n, k), np.int8)
        xs = np.ones(m, np.float32)
        xs[2] = np.nan
        to = dev.put(np.zeros((m, n), np.float32), abi.FP32)
        calc.scaled_gemm(to, dev.put(x, abi.INT8), dev.put(xs, abi.FP32), dev.put(w, abi.INT8), dev.put(np.ones(n, np.float32), abi.FP32))
        calc.sync()
        out = dev.get(to)
        assert np.isnan(out[2]).all() and (np.delete(out, 2, axis=0) == 0).all()


@pytest.mark.parametrize("ot", [abi.FP32, abi.BF16])
@pytest.mark.parametrize("bias_t", [None, abi.FP32, abi.BF16])
def test_product_int8_rows_do_not_depend_on_the_kernel(calc, dev, ot, bias_t):
    """Integer sums are exact, so both kernels round the same numbers in the same way; so does a row alone. Signs of zeros too."""
    rng = np.random.default_rng(17)
    m, n, k = 300, 1112, 1040
    x, w = rng.integers(-128, 128, (m, k)).astype(np.int8), rng.integers(-128, 128, (n, k)).astype(np.int8)
    x[::7] = 0
    xs, ws = rng.standard_normal(m).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    bias = None if bias_t is None else encode(rng.standard_normal(n) * 50, bias_t)[0]
    tx, tw, txs, tws = dev.put(x, abi.INT8), dev.put(w, abi.INT8), dev.put(xs, abi.FP32), dev.put(ws, abi.FP32)
    tb = None if bias is None else dev.put(bias, bias_t)
    rows = {}
    for form, knobs in {"pair": {"pair": 1}, "pair, no tensor map": {"pair": 1, "tma_store": 0}, "few tokens": {"pair": 0, "token_split": 1}, "few tokens, split": {"pair": 0, "token_split": 5}}.items():
        to = dev.put(np.ones((m, n), abi.NP_DTYPE[ot]), ot)
        for name, value in knobs.items():
            calc.set_option(name, value)
        try:
            calc.scaled_gemm(to, tx, txs, tw, tws, bias=tb)
        finally:
            for name in knobs:
                calc.set_option(name, -1)
        calc.sync()
        rows[form] = dev.get(to).view(np.uint8)
    alone = dev.put(np.ones((2, n), abi.NP_DTYPE[ot]), ot)
    calc.scaled_gemm(alone, dev.put(x[40:42], abi.INT8), dev.put(xs[40:42], abi.FP32), tw, tws, bias=tb)
    calc.sync()
    for form, got in rows.items():
        assert (got == rows["pair"]).all(), form
    assert (dev.get(alone).view(np.uint8) == rows["pair"][40:42]).all()
    if bias is None:   # the definition's two products, bit for bit
        with np.errstate(all="ignore"):
            y = ((x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float32) * xs[:, None]) * ws
        assert (rows["pair"] == np.ascontiguousarray(encode(y, ot)[0]).view(np.uint8)).all()


# ------------------------------------------------------------------------------------------ together, host tensors, streams, graphs
def test_layer_run(calc, dev, port):
    """norm with the residual's addition -> 8-bit product -> norm of the sum -> 8-bit product, as a layer uses them, against 64 bits."""
    rng = np.random.default_rng(13)
    tokens, width, inner = 37, 512, 1360
    xb, x = encode(rows_like(rng, tokens, width), abi.BF16)
    rb, r = encode(rows_like(rng, tokens, width), abi.BF16)
    gb, g = encode(1 + 0.3 * rng.standard_normal(width), abi.FP32)
    w1, w2 = rng.standard_normal((width, inner)) * 0.05, rng.standard_normal((inner, width)) * 0.05
    (w1b, w1), (w2b, w2) = encode(w1, abi.BF16), encode(w2, abi.BF16)
    tx, tr, tg = dev.put(xb, abi.BF16), dev.put(rb, abi.BF16), dev.put(gb, abi.FP32)

    def weight(t, cols, rows):
        q, s = dev.put(np.zeros((cols, rows), np.int8), abi.INT8), dev.put(np.zeros(cols, np.float32), abi.FP32)
        calc.quantize(q, s, t, abi.OP_TRANS)
        return q, s

    q1, s1 = weight(dev.put(w1b, abi.BF16), inner, width)
    q2, s2 = weight(dev.put(w2b, abi.BF16), width, inner)
    ts = dev.put(np.zeros_like(xb), abi.BF16)
    tq, tqs = dev.put(np.zeros((tokens, width), np.int8), abi.INT8), dev.put(np.zeros(tokens, np.float32), abi.FP32)
    th, thq, ths = dev.put(np.zeros((tokens, inner), np.uint16), abi.BF16), dev.put(np.zeros((tokens, inner), np.int8), abi.INT8), dev.put(np.zeros(tokens, np.float32), abi.FP32)
    ty, tn, tsum = (dev.put(np.zeros((tokens, width), np.uint16), abi.BF16) for _ in range(3))
    calc.rms_norm(tq, tx, tg, EPS, residual=tr, sum=ts, scale=tqs)
    calc.scaled_gemm(th, tq, tqs, q1, s1)
    calc.quantize(thq, ths, th)
    calc.scaled_gemm(ty, thq, ths, q2, s2)
    calc.rms_norm(tn, ty, tg, EPS, residual=ts, sum=tsum)
    calc.sync()
    # each stage against the formula on what the stage before left
    h = decode(dev.get(ts), abi.BF16)
    codes, step = layer8.codes_of((h * g).astype(np.float32), abi.INT8, port)
    assert (dev.get(tq) == codes).all()
    c1, st1 = layer8.codes_of(w1.T, abi.INT8, port)
    assert (dev.get(q1) == c1).all() and (dev.get(s1)[0] == st1).all()
    y, out, mag = layer8.product(codes, dev.get(tqs)[0], c1, st1, None)
    hid = decode(dev.get(th), abi.BF16)
    assert (np.abs(hid - out) <= layer8.product_bound(y, out, mag, abi.BF16, True)).all()
    c3, st3 = layer8.codes_of(hid, abi.INT8, port)
    assert (dev.get(thq) == c3).all() and (dev.get(ths)[0] == st3).all()
    c2, st2 = layer8.codes_of(w2.T, abi.INT8, port)
    y, out, mag = layer8.product(c3, st3, c2, st2, None)
    back = decode(dev.get(ty), abi.BF16)
    assert (np.abs(back - out) <= layer8.product_bound(y, out, mag, abi.BF16, True)).all()
    _, total = encode((back + h).astype(np.float32), abi.BF16)
    assert (decode(dev.get(tsum), abi.BF16) == total).all()
    ref, _ = layer8.norm(total, g, EPS)
    assert (np.abs(decode(dev.get(tn), abi.BF16) - ref) <= np.abs(ref) * (2.0 ** -8 + 1e-5) + 1e-38).all()
    # and the whole against the layer without any 8-bit rounding: each of the four roundings to 8 bits is off by at most
    # max / 254 per element, a quarter of a percent of the largest; the outputs agree to a few percent of their norm
    n64, _ = layer8.norm((x.astype(np.float64) + r), g, EPS)
    whole = n64 @ w1.astype(np.float64) @ w2.astype(np.float64)
    assert np.linalg.norm(back - whole) < 0.05 * np.linalg.norm(whole)


@pytest.mark.parametrize("m", [3, 300])
def test_host_tensors(calc, port, m):
    rng = np.random.default_rng(14)
    cols, n = 352, 300
    xb, x = encode(rows_like(rng, m, cols), abi.BF16)
    rb, r = encode(rows_like(rng, m, cols), abi.BF16)
    g = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)
    q, s, h = np.zeros((m, cols), np.int8), np.zeros(m, np.float32), np.zeros_like(xb)
    calc.rms_norm(T(q, abi.INT8, [cols, m]), T(xb, abi.BF16, [cols, m]), T(g, abi.FP32, [cols]), EPS, residual=T(rb, abi.BF16, [cols, m]),
                  sum=T(h, abi.BF16, [cols, m]), scale=T(s, abi.FP32, [m]))
    want, hv = encode((x + r).astype(np.float32), abi.BF16)
    assert (h == want).all()
    assert (q == layer8.codes_of((hv * g).astype(np.float32), abi.INT8, port)[0]).all()
    w = rng.integers(-127, 128, (n, cols)).astype(np.int8)
    ws = np.exp(rng.standard_normal(n)).astype(np.float32)
    out = np.full((m, n + 4), -3.0, np.float32)
    calc.scaled_gemm(T(out, abi.FP32, [n, m], [1, n + 4]), T(q, abi.INT8, [cols, m]), T(s, abi.FP32, [m]), T(w, abi.INT8, [cols, n]), T(ws, abi.FP32, [n]))
    y, ref, mag = layer8.product(q, s, w, ws, None)
    assert (np.abs(out[:, :n] - ref) <= layer8.product_bound(y, ref, mag, abi.FP32, True)).all() and (out[:, n:] == -3.0).all()
    dy, dx, dg = rng.standard_normal((m, cols)).astype(np.float32), np.zeros((m, cols), np.float32), np.zeros(cols, np.float32)
    calc.rms_norm_grad(T(dx, abi.FP32, [cols, m]), T(dg, abi.FP32, [cols]), T(dy, abi.FP32, [cols, m]), T(hv, abi.FP32, [cols, m]), T(g, abi.FP32, [cols]), EPS)
    a, b = layer8.norm_grad(hv, g, dy, None, EPS)
    ba, bb = layer8.norm_grad_bounds(hv, g, dy, None, EPS, abi.FP32)
    assert (np.abs(dx - a) <= ba).all() and (np.abs(dg - b) <= bb).all()


def torch_tensor(t, dtype=None):
    import torch
    kinds = {torch.bfloat16: abi.BF16, torch.float32: abi.FP32, torch.int8: abi.INT8}
    return T(t.data_ptr(), kinds[t.dtype], list(reversed(t.shape)), list(reversed(t.stride())), mem_space=abi.MEM_DEVICE)


def test_streams_graphs_and_two_contexts(port):
    """The run on a torch stream, captured and replayed on new inputs; two contexts at once on two streams; scratch memory
    that moves between streams; what capture refuses."""
    import torch
    import intel_gaudi3_software_b200 as pkg
    torch.cuda.set_device(0)
    gen = torch.Generator(device="cuda").manual_seed(15)
    m, k, n = 20, 1024, 768
    state = []
    for i in range(2):
        calc, stream = pkg.Calculator(device=0), torch.cuda.Stream()
        calc.set_stream(stream.cuda_stream)
        x, g = torch.randn(m, k, device="cuda", generator=gen).bfloat16(), torch.rand(k, device="cuda", generator=gen)
        w, ws = torch.randint(-127, 128, (n, k), device="cuda", generator=gen, dtype=torch.int8), torch.rand(n, device="cuda", generator=gen)
        dy = torch.randn(m, k, device="cuda", generator=gen).bfloat16()
        q, s, out = torch.empty(m, k, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda"), torch.empty(m, n, device="cuda")
        dx, dg = torch.empty_like(x), torch.empty(k, device="cuda")
        work = torch.empty(calc.rms_norm_grad_workspace(m, k) // 4, device="cuda")
        state.append((calc, stream, x, g, w, ws, dy, q, s, out, dx, dg, work))
    torch.cuda.synchronize()

    def go(i, workspace):
        calc, stream, x, g, w, ws, dy, q, s, out, dx, dg, work = state[i]
        t = torch_tensor
        calc.rms_norm(t(q), t(x), t(g), EPS, scale=t(s))
        calc.scaled_gemm(t(out), t(q), t(s), t(w), t(ws))
        calc.rms_norm_grad(t(dx), t(dg), t(dy), t(x), t(g), EPS, workspace=t(work) if workspace else None)

    def check(i):
        calc, stream, x, g, w, ws, dy, q, s, out, dx, dg, work = state[i]
        xf, gf = x.float().cpu().numpy(), g.cpu().numpy()
        codes, step = layer8.codes_of((xf * gf).astype(np.float32), abi.INT8, port)
        assert (q.cpu().numpy() == codes).all()
        y, ref, mag = layer8.product(codes, s.cpu().numpy(), w.cpu().numpy(), ws.cpu().numpy(), None)
        assert (np.abs(out.cpu().numpy() - ref) <= layer8.product_bound(y, ref, mag, abi.FP32, True)).all()
        a, b = layer8.norm_grad(xf, gf, dy.float().cpu().numpy(), None, EPS)
        ba, bb = layer8.norm_grad_bounds(xf, gf, dy.float().cpu().numpy(), None, EPS, abi.BF16)
        assert (np.abs(dx.float().cpu().numpy() - a) <= ba).all() and (np.abs(dg.cpu().numpy() - b) <= bb).all()

    for _ in range(20):          # both contexts at once
        go(0, False)
        go(1, True)
    torch.cuda.synchronize()
    check(0)
    check(1)
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=state[i][1]):
            go(i, True)
        graphs.append(graph)
    for i in range(2):
        state[i][2].copy_(torch.randn(m, k, device="cuda", generator=gen))
        for t in state[i][7:12]:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(state[i][1]):
                graphs[i].replay()
    torch.cuda.synchronize()
    check(0)
    check(1)
    # capture refuses what needs scratch memory, and the capture goes on
    calc, stream, x, g, w, ws, dy, q, s, out, dx, dg, work = state[0]
    odd = torch.empty(m * k + 16, dtype=torch.int8, device="cuda")[1:1 + m * k].view(m, k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        go(0, True)
        with pytest.raises(MmeError, match="workspace"):
            go(0, False)
        with pytest.raises(MmeError, match="16-byte"):
            calc.scaled_gemm(torch_tensor(out), torch_tensor(odd), torch_tensor(s), torch_tensor(w), torch_tensor(ws))
        with pytest.raises(MmeError, match="device tensors"):
            h = np.zeros((m, n), np.float32)
            calc.scaled_gemm(T(h, abi.FP32, [n, m]), torch_tensor(q), torch_tensor(s), torch_tensor(w), torch_tensor(ws))
    graph.replay()
    torch.cuda.synchronize()
    check(0)
    # the context's scratch memory used from one stream, then at once from another
    other = torch.cuda.Stream()
    for _ in range(10):
        calc.set_stream(stream.cuda_stream)
        go(0, False)
        calc.set_stream(other.cuda_stream)
        other.wait_stream(stream)
        go(0, False)
        stream.wait_stream(other)
    torch.cuda.synchronize()
    check(0)
    calc.set_stream(abi.STREAM_LEGACY)
    go(0, False)
    torch.cuda.synchronize()
    check(0)
    for st in state:
        st[0].close()


def test_an_earlier_error_of_the_callers_is_not_the_call_s(calc, dev, port):
    """The thread's last CUDA error, left by a call of the program's own, neither fails a call nor is taken away by it."""
    runtime = C.CDLL("libcudart.so.12")
    rng = np.random.default_rng(18)
    m, k, n = 300, 1104, 264
    v, g = rows_like(rng, m, k), dev.put(np.ones(k, np.float32), abi.FP32)
    x, q, s = dev.put(v, abi.FP32), dev.put(np.zeros((m, k), np.int8), abi.INT8), dev.put(np.zeros(m, np.float32), abi.FP32)
    qt, st = dev.put(np.zeros((k, m), np.int8), abi.INT8), dev.put(np.zeros(k, np.float32), abi.FP32)
    w, one = dev.put(np.ones((n, k), np.int8), abi.INT8), dev.put(np.ones(1, np.float32), abi.FP32)
    odd = dev.put(np.ones((n, k), np.int8), abi.INT8, offset=1)
    y, dx, dg = dev.put(np.zeros((m, n), np.float32), abi.FP32), dev.put(np.zeros((m, k), np.float32), abi.FP32), dev.put(np.zeros(k, np.float32), abi.FP32)
    few, none = dev.put(np.zeros((3, n), np.float32), abi.FP32), T(None, abi.INT8, [0, 3], mem_space=abi.MEM_DEVICE)
    q3 = T(q.data, abi.INT8, [k, 3], mem_space=abi.MEM_DEVICE)
    host_q, host_s = np.zeros((m, k), np.int8), np.zeros(m, np.float32)
    calls = {
        "norm": lambda: calc.rms_norm(q, x, g, EPS, scale=s),
        "gradient": lambda: calc.rms_norm_grad(dx, dg, x, x, g, EPS),
        "rows": lambda: calc.quantize(q, s, x),
        "columns": lambda: calc.quantize(qt, st, x, abi.OP_TRANS),
        "product": lambda: calc.scaled_gemm(y, q, s, w, one),
        "product of few tokens": lambda: calc.scaled_gemm(few, q3, one, w, one),
        "product of unaligned rows": lambda: calc.scaled_gemm(few, q3, one, odd, one),
        "product of nothing": lambda: calc.scaled_gemm(few, none, one, T(None, abi.INT8, [0, n], mem_space=abi.MEM_DEVICE), one),
        "host rows": lambda: calc.quantize(T(host_q, abi.INT8, [k, m]), T(host_s, abi.FP32, [m]), T(v, abi.FP32, [k, m])),
    }
    for name, call in calls.items():
        error = runtime.cudaSetDevice(9999)
        assert error != 0
        try:
            call()
            assert runtime.cudaPeekAtLastError() == error, name
        finally:
            runtime.cudaGetLastError()
    calc.sync()
    codes, step = layer8.codes_of(v, abi.INT8, port)
    assert (dev.get(q) == codes).all() and (dev.get(s)[0] == step).all() and (host_q == codes).all() and (dev.get(few) == 0).all()


FIRST_CALLS_CAPTURED = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from intel_gaudi3_software_b200 import Calculator, abi
kinds = {torch.bfloat16: abi.BF16, torch.float32: abi.FP32, torch.int8: abi.INT8}
def t(a):
    return abi.make_tensor(a.data_ptr(), kinds[a.dtype], list(reversed(a.shape)), list(reversed(a.stride())), mem_space=abi.MEM_DEVICE)
stream = torch.cuda.Stream()
calc = Calculator(device=0)
calc.set_stream(stream.cuda_stream)
rows, cols, n = 12, 9104, 136
x, dy = (torch.randn(rows, cols, device="cuda").bfloat16() for _ in range(2))
w, gamma = torch.randn(cols, n, device="cuda").bfloat16(), torch.rand(cols, device="cuda")
outs = [torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(n, cols, dtype=torch.int8, device="cuda"),
        torch.zeros(n, device="cuda"), torch.zeros(rows, n, device="cuda"), torch.zeros_like(x), torch.zeros(cols, device="cuda")]
work = torch.zeros(calc.rms_norm_grad_workspace(rows, cols) // 4, device="cuda")
q, s, wq, ws, y, dx, dg = (t(o) for o in outs)
def run():
    calc.rms_norm(q, t(x), t(gamma), 1e-5, scale=s)
    calc.quantize(wq, ws, t(w), abi.OP_TRANS)
    calc.scaled_gemm(y, q, s, wq, ws)
    calc.rms_norm_grad(dx, dg, t(dy), t(x), t(gamma), 1e-5, workspace=t(work))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    run()
graph.replay()
torch.cuda.synchronize()
replayed = [o.clone() for o in outs]
for o in outs:
    o.zero_()
torch.cuda.synchronize()
run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(replayed, outs)) and all(o.any() for o in outs)
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing that a call sets up once keeps it from being captured."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS_CAPTURED, root], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


def test_first_products_of_many_tiles_inside_a_capture():
    """The same with the kernel of many tiles."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = FIRST_CALLS_CAPTURED.replace("rows, cols, n = 12, 9104, 136", "rows, cols, n = 520, 1104, 264; calc.set_option('pair', 1)")
    assert text != FIRST_CALLS_CAPTURED
    done = subprocess.run([sys.executable, "-c", text, root], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


FIRST_CALLS_ON_TWO_THREADS = """
import sys, threading, torch
sys.path.insert(0, sys.argv[1])
from intel_gaudi3_software_b200 import Calculator, abi
kinds = {torch.bfloat16: abi.BF16, torch.float32: abi.FP32, torch.int8: abi.INT8}
def t(a):
    return abi.make_tensor(a.data_ptr(), kinds[a.dtype], list(reversed(a.shape)), list(reversed(a.stride())), mem_space=abi.MEM_DEVICE)
rows, cols, n = 520, 9104, 264
gen = torch.Generator(device="cuda").manual_seed(1)
x, dy = (torch.randn(rows, cols, device="cuda", generator=gen).bfloat16() for _ in range(2))
w, gamma = torch.randn(cols, n, device="cuda", generator=gen).bfloat16(), torch.rand(cols, device="cuda", generator=gen)
torch.cuda.synchronize()
start, results = threading.Barrier(2), [None, None]
def work(i):
    calc = Calculator(device=0)
    outs = [torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(n, cols, dtype=torch.int8, device="cuda"),
            torch.zeros(n, device="cuda"), torch.zeros(rows, n, device="cuda"), torch.zeros(9, n, device="cuda"), torch.zeros_like(x), torch.zeros(cols, device="cuda")]
    torch.cuda.synchronize()
    q, s, wq, ws, y, few, dx, dg = (t(o) for o in outs)
    start.wait()
    for _ in range(20):
        calc.rms_norm(q, t(x), t(gamma), 1e-5, scale=s)
        calc.quantize(wq, ws, t(w), abi.OP_TRANS)
        calc.scaled_gemm(y, q, s, wq, ws)
        calc.scaled_gemm(few, t(outs[0][:9]), t(outs[1][:9]), wq, ws)
        calc.rms_norm_grad(dx, dg, t(dy), t(x), t(gamma), 1e-5)
    calc.sync()
    results[i] = outs
    calc.close()
threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
for th in threads: th.start()
for th in threads: th.join()
assert all(torch.equal(a, b) and a.any() for a, b in zip(*results))
print("same")
"""


def test_first_calls_of_two_threads_at_once():
    """Two contexts, each on a thread of its own, whose first calls of every kind meet."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS_ON_TWO_THREADS, root], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


# ------------------------------------------------------------------------------------------ refusals
def test_refusals(calc, dev):
    rng = np.random.default_rng(16)
    m, k, n = 8, 64, 48
    f = lambda *s: np.zeros(s, np.float32)   # noqa: E731
    x, xb = dev.put(f(m, k), abi.FP32), dev.put(np.zeros((m, k), np.uint16), abi.BF16)
    q, w = dev.put(np.zeros((m, k), np.int8), abi.INT8), dev.put(np.zeros((n, k), np.int8), abi.INT8)
    sm, sn, sk = dev.put(f(m), abi.FP32), dev.put(f(n), abi.FP32), dev.put(f(k), abi.FP32)
    out, o8 = dev.put(f(m, n), abi.FP32), dev.put(np.zeros((m, k), np.uint8), abi.FP8_143, **FP8)
    y = dev.put(f(m, k), abi.FP32)

    def refused(match, fn, *a, **kw):
        with pytest.raises(MmeError, match=match):
            fn(*a, **kw)

    def like(t, **change):
        d = abi.Tensor()
        C.memmove(C.byref(d), C.byref(t), C.sizeof(d))
        for name, v in change.items():
            if name in ("sizes", "strides"):
                for i, e in enumerate(v):
                    getattr(d, name)[i] = e
            else:
                setattr(d, name, v)
        return d

    norm, quant, prod, grad = calc.rms_norm, calc.quantize, calc.scaled_gemm, calc.rms_norm_grad
    refused("null tensor", norm, None, x, None, EPS)
    refused("null tensor", norm, y, None, None, EPS)
    refused("null data", norm, like(y, data=None), x, None, EPS)
    refused("not accepted", norm, like(y, dtype=abi.TF32), x, None, EPS)
    refused("not accepted", norm, y, q, None, EPS)
    refused("sizes do not match", norm, y, like(x, sizes=[32, m]), None, EPS)
    refused("sizes do not match", norm, y, x, None, EPS, residual=like(xb, sizes=[k, 4]))
    refused("no residual", norm, y, x, None, EPS, sum=xb)
    refused("the residual's", norm, y, x, None, EPS, residual=x, sum=xb)
    refused("gamma", norm, y, x, sm, EPS)
    refused("eps", norm, y, x, None, -1.0)
    refused("eps", norm, y, x, None, float("nan"))
    refused("eps", norm, y, x, None, float("inf"))
    refused("float output has none", norm, y, x, None, EPS, scale=sm)
    refused("scale: null", norm, q, x, None, EPS)
    refused("scale", norm, q, x, None, EPS, scale=sk)
    refused("scale mode", norm, q, x, None, EPS, scale=sm, scale_mode=7)
    refused("fp32", norm, q, x, None, EPS, scale=like(xb, sizes=[m, 1]))
    refused("overlap", norm, like(y, strides=[1, 0]), x, None, EPS)
    refused("overlap", norm, like(y, strides=[1, k - 1]), x, None, EPS)
    refused("overlap", norm, like(x, data=x.data + 16), x, None, EPS)
    refused("overlap", norm, y, x, None, EPS, residual=xb, sum=like(xb, data=x.data))
    refused("overlap", norm, y, x, like(sk, data=y.data), EPS)
    refused("strides", norm, like(y, strides=[2, 2 * k]), x, None, EPS)
    refused("dims", norm, like(y, dims=0), x, None, EPS)
    refused("memory space", norm, like(y, mem_space=5), x, None, EPS)
    refused("2.31", norm, like(y, sizes=[k, 1 << 30]), like(x, sizes=[k, 1 << 30]), None, EPS)
    refused("aligned", norm, like(y, data=y.data + 2), x, None, EPS)
    refused("without elements", norm, like(y, sizes=[0, m]), like(x, sizes=[0, m]), None, EPS)
    refused("1-5-2", norm, like(o8, dtype=abi.FP8_152, fp_bias=15), x, None, EPS, scale=sm)
    refused("exponent bias", norm, like(o8, fp_bias=0), x, None, EPS, scale=sm)
    refused("Inf/NaN", norm, like(o8, inf_nan_mode=4), x, None, EPS, scale=sm)

    refused("neither", quant, q, sm, x, abi.OP_AB)
    refused("scale: null", quant, q, None, x)
    refused("not accepted", quant, y, sm, x)
    refused("transposed", quant, q, sk, x, abi.OP_TRANS)
    refused("scale", quant, like(q, sizes=[m, k], strides=[1, m]), sm, x, abi.OP_TRANS)
    refused("2-D", quant, like(q, sizes=[m, k, 2]), sk, like(x, sizes=[k, m, 2]), abi.OP_TRANS)
    refused("columns without", quant, like(q, sizes=[0, k]), sk, like(x, sizes=[k, 0]), abi.OP_TRANS)

    refused("one data type", grad, y, sk, like(xb), x, None, EPS)
    refused("x's", grad, y, sk, x, x, None, EPS, dsum=xb)
    refused("fp32", grad, y, like(xb, sizes=[k, 1]), x, x, None, EPS)
    refused("dgamma", grad, y, sm, x, x, None, EPS)
    refused("workspace", grad, y, sk, x, x, None, EPS, workspace=sm)
    refused("overlap", grad, y, like(sk, data=x.data), x, x, None, EPS)
    refused("eps", grad, y, sk, x, x, None, -1.0)

    refused("ABT", prod, out, q, sm, w, sn, op=abi.OP_AB)
    refused("not accepted", prod, out, xb, sm, w, sn)
    refused("not accepted", prod, like(q, sizes=[n, m]), q, sm, w, sn)
    refused("mixed", prod, out, o8, sm, w, sn)
    refused("Common dim", prod, out, like(q, sizes=[32, m]), sm, w, sn)
    refused("width", prod, like(out, sizes=[m, n]), q, sm, w, sn)
    refused("x_scale", prod, out, q, sn, w, sn)
    refused("w_scale", prod, out, q, sm, w, sm)
    refused("bias", prod, out, q, sm, w, sn, bias=sm)
    refused("overlap", prod, like(out, data=w.data), q, sm, w, sn)
    refused("overlap", prod, like(out, strides=[1, n - 1]), q, sm, w, sn)
    refused("convention", prod, out, like(o8, inf_nan_mode=abi.INFNAN_FULL), sm, like(o8, sizes=[k, n]), sn)
    refused("131071", prod, out, like(q, sizes=[131072, m], strides=[1, 0]), sm, like(w, sizes=[131072, n], strides=[1, 0]), sn)
    refused("2-D", prod, like(out, sizes=[n, m, 2]), like(q, sizes=[k, m, 2]), sm, like(w, sizes=[k, n, 2]), sn)
    # the calculator's own entry points keep refusing int8
    with pytest.raises(MmeError):
        calc.do_batch_gemm(out, q, w, abi.OP_ABT)
    calc.sync()


def test_exact_mode_refuses_fp8_products(dev):
    import intel_gaudi3_software_b200 as pkg
    calc = pkg.Calculator(device=0, accumulation=abi.ACC_CHIP_EXACT)
    d = Dev(calc)
    o, s = d.put(np.zeros((4, 4), np.float32), abi.FP32), d.put(np.ones(1, np.float32), abi.FP32)
    a = d.put(np.zeros((4, 16), np.uint8), abi.FP8_143, **FP8)
    with pytest.raises(MmeError, match="tensor cores only"):
        calc.scaled_gemm(o, a, s, a, s)
    q = d.put(np.ones((4, 16), np.int8), abi.INT8)
    calc.scaled_gemm(o, q, s, q, s)
    calc.sync()
    assert (d.get(o) == 16).all()
    d.free()
    calc.close()
