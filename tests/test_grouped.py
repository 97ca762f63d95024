"""Muls with weights in ragged groups and with 4-bit weights: against 64-bit arithmetic, and what is refused."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import ruy_b200 as rb
from ruy_b200 import _abi
from ruy_b200._lib import lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
RowMajor, ColMajor = rb.Order.kRowMajor, rb.Order.kColMajor


# ---- without a GPU: structs and refusals ----------------------------------------------------------------


def test_struct_layout_matches_c(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ruy_b200.h"\nint main(){printf("%zu %zu %zu %zu %zu %d %d %d %d\\n",'
                   "sizeof(ruyb200_groups),offsetof(ruyb200_groups,count),sizeof(ruyb200_q4_scales),"
                   "offsetof(ruyb200_q4_scales,block),offsetof(ruyb200_q4_scales,dtype),"
                   "RUYB200_F16,RUYB200_BF16,RUYB200_I4,RUYB200_U4);return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)], text=True).split()]
    assert got == [C.sizeof(_abi.GroupsDesc), _abi.GroupsDesc.count.offset, C.sizeof(_abi.Q4ScalesDesc),
                   _abi.Q4ScalesDesc.block.offset, _abi.Q4ScalesDesc.dtype.offset, _abi.F16, _abi.BF16, _abi.I4, _abi.U4]


@pytest.mark.parametrize("accum,lo,hi", [("int32", -100, 101), ("float32", -1.5, float("inf")), ("float64", 2.0 ** -60, 3.0)])
def test_packed_descriptors_are_the_structs(accum, lo, hi):
    t = {"int32": np.int8, "float32": np.float32, "float64": np.float64}[accum]
    a, b, c = np.zeros((4, 6), t), np.zeros((5, 6), t), np.zeros((5, 7), t)
    lhs = rb.Matrix(a, rb.Layout(4, 5, 6, RowMajor), -3, rb.CachePolicy.kAlwaysCache)
    rhs, dst = rb.Matrix(b, rb.Layout(5, 5, 6, ColMajor), 17), rb.Matrix(c, rb.Layout(4, 5, 7, ColMajor), 2)
    p = rb.MulParams(accum, t)
    p.bias, p.multiplier_fixedpoint_perchannel, p.multiplier_exponent_perchannel = a, b, c
    p.multiplier_fixedpoint, p.multiplier_exponent, p.clamp_min, p.clamp_max = 5, -6, lo, hi
    p.channel_dimension, p.perchannel_buffers_capacity_rounding, p.rounding = rb.ChannelDimension.kCol, 8, rb.Rounding.kX86
    from ruy_b200 import api
    packed = _abi.MulDesc.from_buffer_copy(api._packed_desc(lhs, rhs, p, dst))
    assert len(api._packed_desc(lhs, rhs, p, dst)) == C.sizeof(_abi.MulDesc)
    plain = rb.make_desc(lhs, rhs, p, dst)

    def values(s):
        return [values(getattr(s, n)) if isinstance(getattr(s, n), C.Structure) else
                getattr(getattr(s, n), {"int32": "i", "float32": "f", "float64": "d"}[accum]) if isinstance(getattr(s, n), C.Union) else
                getattr(s, n) for n, _ in s._fields_]
    assert values(packed) == values(plain)
    scales = rb.Q4Scales(np.zeros(8, np.float16), 64, 9, np.zeros(8, np.int8))
    assert bytes(scales.to_desc()) == _abi.Q4_SCALES_PACK.pack(*scales._fields())
    groups = rb.Groups(np.zeros(8, np.int32), 64, 9, 2 ** 40)
    assert bytes(groups.to_desc()) == _abi.GROUPS_PACK.pack(*groups._fields())


class _NoContext:
    _h = None


def _i8_call(change=None, rows=4, depth=32, cols=3, groups=2):
    """A call that is right but for the missing context, after `change` has had its way with the arguments."""
    a = {"lhs": rb.Matrix(np.zeros((groups, rows, depth), np.int8), rb.Layout(rows, depth, depth, RowMajor)),
         "rhs": rb.Matrix(np.zeros((cols, depth), np.int8), rb.Layout(depth, cols, depth, ColMajor)),
         "dst": rb.Matrix(np.zeros((cols, rows), np.int8), rb.Layout(rows, cols, rows, ColMajor)),
         "p": rb.MulParams("int32", "int8"),
         "groups": rb.Groups(np.zeros(groups + 1, np.int32), rows * depth, rows)}
    if change:
        change(a)
    with pytest.raises(rb.RuyError) as e:
        rb.mul_grouped_async(a["lhs"], a["rhs"], a["p"], _NoContext, a["dst"], a["groups"])
    return e.value.status, str(e.value)


def _set(path, value):
    def change(a):
        parts = path.split(".")
        if len(parts) == 1:
            a[path] = value
            return
        o = a[parts[0]]
        for name in parts[1:-1]:
            o = getattr(o, name)
        setattr(o, parts[-1], value)
    return change


def test_grouped_right_but_for_the_context():
    assert _i8_call()[0] == _abi.ERR_INVALID and "null context" in _i8_call()[1]


@pytest.mark.parametrize("path,value,status,text", [
    ("lhs.data", np.zeros(256, np.int16), _abi.ERR_UNSUPPORTED, "8-bit"),
    ("rhs.data", np.zeros(256, np.float32), _abi.ERR_UNSUPPORTED, "type"),
    ("rhs.data", np.zeros(256, np.float16), _abi.ERR_UNSUPPORTED, "dtype"),
    ("lhs.layout", rb.Layout(4, 32, 4, ColMajor), _abi.ERR_UNSUPPORTED, "row-major"),
    ("rhs.layout", rb.Layout(32, 3, 3, RowMajor), _abi.ERR_UNSUPPORTED, "row-major"),
    ("dst.layout", rb.Layout(4, 3, 3, RowMajor), _abi.ERR_UNSUPPORTED, "column-major"),
    ("dst.layout", rb.Layout(4, 2, 4, ColMajor), _abi.ERR_INVALID, "shape"),
    ("dst.layout", rb.Layout(4, 3, 3, ColMajor), _abi.ERR_INVALID, "stride"),
    ("lhs.zero_point", 200, _abi.ERR_INVALID, "zero_point"),
    ("p.multiplier_exponent", 31, _abi.ERR_INVALID, "exponent"),
    ("p.multiplier_fixedpoint_perchannel", np.zeros(8, np.int32), _abi.ERR_INVALID, "both"),
    ("groups.lhs_stride", -1, _abi.ERR_INVALID, "negative"),
    ("groups.channel_stride", -4, _abi.ERR_INVALID, "negative"),
    ("groups.offsets", np.zeros(1026, np.int32), _abi.ERR_INVALID, "1024"),
    ("dst.data", None, _abi.ERR_INVALID, "null"),
])
def test_grouped_refusals(path, value, status, text):
    got, msg = _i8_call(_set(path, value))
    assert got == status and text in msg, msg


def test_grouped_refuses_buffers_along_the_columns():
    def change(a):
        a["p"].bias = np.zeros(3, np.int32)
        a["p"].channel_dimension = rb.ChannelDimension.kCol
    got, msg = _i8_call(change)
    assert got == _abi.ERR_UNSUPPORTED and "rows" in msg


def _q4_call(change=None, grouped=True, rows=4, depth=64, cols=3, groups=2):
    a = {"lhs": rb.Q4Matrix(np.zeros((groups, rows, depth // 2), np.uint8), rb.Layout(rows, depth, depth, RowMajor),
                            rb.Q4Scales(np.zeros((groups, rows, 2), np.float32), 32, 2)),
         "rhs": rb.Matrix(np.zeros((cols, depth), np.float16), rb.Layout(depth, cols, depth, ColMajor)),
         "dst": rb.Matrix(np.zeros((cols, rows), np.float16), rb.Layout(rows, cols, rows, ColMajor)),
         "p": rb.MulParams("float32", "float32"),
         "groups": rb.Groups(np.zeros(groups + 1, np.int32), rows * depth, rows, rows * 2)}
    if change:
        change(a)
    with pytest.raises(rb.RuyError) as e:
        if grouped:
            rb.mul_grouped_q4_async(a["lhs"], a["rhs"], a["p"], _NoContext, a["dst"], a["groups"])
        else:
            rb.mul_q4_async(a["lhs"], a["rhs"], a["p"], _NoContext, a["dst"])
    return e.value.status, str(e.value)


def test_q4_right_but_for_the_context():
    for grouped in (False, True):
        status, msg = _q4_call(grouped=grouped)
        assert status == _abi.ERR_INVALID and "null context" in msg


@pytest.mark.parametrize("path,value,status,text", [
    ("rhs.data", np.zeros(256, np.int8), _abi.ERR_UNSUPPORTED, "rhs"),
    ("rhs.data", np.zeros(256, np.float64), _abi.ERR_UNSUPPORTED, "rhs"),
    ("rhs.data", np.zeros(256, np.float32), _abi.ERR_UNSUPPORTED, "dst"),   # half destination of a float mul
    ("p", rb.MulParams("int32", "int8"), _abi.ERR_UNSUPPORTED, "accumulation"),
    ("lhs.layout", rb.Layout(4, 64, 4, ColMajor), _abi.ERR_UNSUPPORTED, "row-major"),
    ("lhs.layout", rb.Layout(4, 64, 65, RowMajor), _abi.ERR_INVALID, "even"),
    ("lhs.layout", rb.Layout(4, 64, 62, RowMajor), _abi.ERR_INVALID, "stride"),
    ("lhs.layout", rb.Layout(-4, 64, 64, RowMajor), _abi.ERR_INVALID, "negative"),
    ("rhs.layout", rb.Layout(62, 3, 64, ColMajor), _abi.ERR_INVALID, "shape"),
    ("rhs.zero_point", 1, _abi.ERR_INVALID, "zero points"),
    ("lhs.scales.block", 0, _abi.ERR_INVALID, "multiple of 32"),
    ("lhs.scales.block", 48, _abi.ERR_INVALID, "multiple of 32"),
    ("lhs.scales.stride", 1, _abi.ERR_INVALID, "stride"),
    ("lhs.scales.scales", np.zeros(16, np.int8), _abi.ERR_UNSUPPORTED, "scales"),
    ("lhs.scales.scales", None, _abi.ERR_UNSUPPORTED, "scales"),
    ("groups.lhs_stride", 3, _abi.ERR_INVALID, "even"),
    ("groups.scale_stride", -1, _abi.ERR_INVALID, "negative"),
])
def test_q4_refusals(path, value, status, text):
    got, msg = _q4_call(_set(path, value))
    assert got == status and text in msg, msg


def test_q4_refuses_bias_along_the_columns():
    def change(a):
        a["p"].bias = np.zeros(3, np.float32)
        a["p"].channel_dimension = rb.ChannelDimension.kCol
    assert _q4_call(change)[0] == _abi.ERR_UNSUPPORTED


def test_null_descriptors_are_refused():
    assert lib().ruyb200_mul_grouped_async(None, None, None) == _abi.ERR_INVALID
    assert lib().ruyb200_mul_q4_async(None, None, None) == _abi.ERR_INVALID
    assert lib().ruyb200_mul_grouped_q4_async(None, None, None, None) == _abi.ERR_INVALID


def test_other_calls_refuse_the_new_types():
    one = rb.Matrix(np.zeros((4, 4), np.float16), rb.Layout(4, 4, 4, RowMajor))
    assert rb.validate(one, one, rb.MulParams("float32", "float32"), one) == _abi.ERR_UNSUPPORTED


def test_new_argument_classes_check_their_types():
    with pytest.raises(TypeError):
        rb.Groups(np.zeros(3, np.int16), 0).to_desc()
    with pytest.raises(TypeError):
        rb.Q4Scales(np.zeros(4, np.float32), 32, 1, np.zeros(4, np.uint8)).to_desc()
    with pytest.raises(TypeError):
        rb.Q4Matrix(np.zeros(4, np.float32), rb.Layout(1, 8, 8, RowMajor), None).to_desc()


# ---- on a GPU -------------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def ctx():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = rb.Context(0, torch.cuda.default_stream().cuda_stream or 1)
    yield c
    c.close()


NP = {"i8": np.int8, "u8": np.uint8, "i16": np.int16, "i32": np.int32}


class I8Case:
    """A grouped 8-bit mul: host arrays, the library's answer, and the answer in 64 bits."""

    def __init__(self, sizes, rows, depth, lhs="i8", rhs="i8", dst="i8", lhs_zp=0, rhs_zp=0, dst_zp=0, bias=True, perchannel=True,
                 clamp=None, pad=0, w_stride=None, x_stride=None, dst_pad=0, shared_channels=False, rounding=None, seed=0, first=0):
        r = np.random.default_rng(seed)
        self.sizes, self.rows, self.depth, self.dst, self.pad = sizes, rows, depth, dst, pad
        self.zp = (lhs_zp, rhs_zp, dst_zp)
        self.w_stride = w_stride or -(-depth // 16) * 16
        self.x_stride = x_stride or -(-depth // 16) * 16
        self.dst_stride = rows + dst_pad
        self.cols = first + sum(sizes) + pad
        self.offsets = np.cumsum([first] + list(sizes)).astype(np.int32)
        g = len(sizes)

        def ints(shape, kind):
            i = np.iinfo(NP[kind])
            return r.integers(i.min, i.max + 1, shape).astype(NP[kind])
        self.w = ints((g, max(rows, 1), max(self.w_stride, 1)), lhs)
        self.x = ints((max(self.cols, 1), max(self.x_stride, 1)), rhs)
        gc = 1 if shared_channels else g
        self.channel_stride = 0 if shared_channels else rows
        self.bias = r.integers(-50000, 50001, (gc, rows)).astype(np.int32) if bias else None
        self.mfp = self.mexp = None
        self.scalar = (1 << 30, -8)
        if perchannel and dst != "i32":
            self.mfp = r.integers(2 ** 30, 2 ** 31, (gc, rows)).astype(np.int32)
            self.mexp = r.integers(-14, -4, (gc, rows)).astype(np.int32)
        info = np.iinfo(NP[dst])
        self.clamp = clamp or (int(info.min), int(info.max))
        self.rounding = rounding or rb.Rounding.kReference
        self.fill = 77
        self.y = np.full((max(self.cols, 1), max(self.dst_stride, 1)), self.fill, NP[dst])

    def want(self, offsets=None):
        offsets = self.offsets if offsets is None else offsets
        out = self.y.copy()
        info = np.iinfo(NP[self.dst])
        for g in range(len(self.sizes)):
            a, b = int(offsets[g]), int(offsets[g + 1])
            if b <= a:
                continue
            w = self.w[g, :self.rows, :self.depth].astype(np.int64) - self.zp[0]
            x = self.x[a:b, :self.depth].astype(np.int64) - self.zp[1]
            v = x @ w.T
            gc = g if self.channel_stride else 0
            if self.bias is not None:
                v = v + self.bias[gc].astype(np.int64)
            if self.dst != "i32":
                m = self.mfp[gc].astype(np.int64) if self.mfp is not None else np.full(self.rows, self.scalar[0], np.int64)
                e = self.mexp[gc].astype(np.int64) if self.mexp is not None else np.full(self.rows, self.scalar[1], np.int64)
                if self.rounding == rb.Rounding.kX86:
                    # rounding doubling high multiply, then rounding right shift (exponents here are negative)
                    t = (v * m + (1 << 30)) >> 31
                    v = (t + (1 << (-e - 1))) >> -e
                else:
                    v = (v * m + (1 << (30 - e))) >> (31 - e)
                v = v + self.zp[2]
                v = np.maximum(np.minimum(v, self.clamp[1]), self.clamp[0])
            else:
                v = v + self.zp[2]
            assert v.min() >= info.min and v.max() <= info.max
            out[a:b, :self.rows] = v.astype(NP[self.dst])
        return out

    def tensors(self):
        import torch
        t = {}
        for name in ("w", "x", "y", "bias", "mfp", "mexp", "offsets"):
            v = getattr(self, name)
            t[name] = None if v is None else torch.from_numpy(v.copy()).cuda()
        return t

    def args(self, t):
        lhs = rb.Matrix(t["w"], rb.Layout(self.rows, self.depth, self.w_stride, RowMajor), self.zp[0])
        rhs = rb.Matrix(t["x"], rb.Layout(self.depth, self.cols, self.x_stride, ColMajor), self.zp[1])
        dst = rb.Matrix(t["y"], rb.Layout(self.rows, self.cols, self.dst_stride, ColMajor), self.zp[2])
        p = rb.MulParams("int32", NP[self.dst])
        p.bias, p.rounding = t["bias"], self.rounding
        p.multiplier_fixedpoint_perchannel, p.multiplier_exponent_perchannel = t["mfp"], t["mexp"]
        p.multiplier_fixedpoint, p.multiplier_exponent = self.scalar
        if self.dst != "i32":
            p.clamp_min, p.clamp_max = self.clamp
        groups = rb.Groups(t["offsets"], self.w.shape[1] * self.w_stride, self.channel_stride)
        return lhs, rhs, p, dst, groups

    def enqueue(self, ctx, t):
        lhs, rhs, p, dst, groups = self.args(t)
        rb.mul_grouped_async(lhs, rhs, p, ctx, dst, groups)

    def run(self, ctx, t=None):
        t = t or self.tensors()
        self.enqueue(ctx, t)
        ctx.sync()
        return t["y"].cpu().numpy()

    def check(self, ctx, kernel=None):
        got = self.run(ctx)
        np.testing.assert_array_equal(got, self.want())
        if kernel:
            assert ctx.counters()["last_kernel"] == kernel


SIZES = [[1], [0, 1, 0], [3, 0, 17, 1, 8], [130, 0, 1, 257, 64, 15, 16], [5] * 40, [700, 2]]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s[:7])))
@pytest.mark.parametrize("rows,depth", [(1, 1), (16, 32), (37, 100), (128, 128), (200, 517), (300, 1040)])
def test_grouped_sizes(ctx, sizes, rows, depth):
    I8Case(sizes, rows, depth, pad=3, dst_pad=5, rhs_zp=-7, dst_zp=3, first=2).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1, 0, 2], [9, 40, 0, 3], [200, 31, 300]], ids=["few", "some", "many"])
@pytest.mark.parametrize("lhs,rhs,dst,zps", [
    ("i8", "i8", "i8", (0, 0, 0)), ("i8", "i8", "u8", (0, -3, 128)), ("i8", "u8", "i8", (5, 200, -1)),
    ("u8", "i8", "i16", (128, -128, 0)), ("u8", "u8", "u8", (128, 255, 255)), ("u8", "u8", "i32", (0, 0, 0)),
    ("i8", "i8", "i32", (-128, 127, 0)), ("u8", "u8", "u8", (0, 9, 0)), ("i8", "i8", "i16", (3, 0, 1000))])
@pytest.mark.parametrize("perchannel", [True, False])
def test_grouped_types_and_zero_points(ctx, sizes, lhs, rhs, dst, zps, perchannel):
    I8Case(sizes, 150, 288, lhs, rhs, dst, *zps, perchannel=perchannel, bias=perchannel).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[2, 1], [40, 0, 90]])
@pytest.mark.parametrize("rounding", [rb.Rounding.kReference, rb.Rounding.kX86])
@pytest.mark.parametrize("shared", [True, False])
def test_grouped_rounding_clamp_and_shared_channels(ctx, sizes, rounding, shared):
    I8Case(sizes, 65, 64, rounding=rounding, shared_channels=shared, clamp=(-100, 90)).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("w_stride,x_stride,sizes", [(100, 112, [3, 5]), (112, 101, [3, 50]), (103, 103, [300])])
def test_grouped_unaligned_layouts(ctx, w_stride, x_stride, sizes):
    I8Case(sizes, 30, 99, w_stride=w_stride, x_stride=x_stride, rhs_zp=4, lhs_zp=2).check(ctx, "generic")


@pytest.mark.gpu
def test_grouped_depth_zero_and_empty_calls(ctx):
    for sizes in ([2, 3], [70, 1]):
        c = I8Case(sizes, 20, 0, w_stride=16, x_stride=16, dst_zp=2)
        c.check(ctx)
    I8Case([0, 0], 20, 32, pad=4).check(ctx)      # no group has a column: nothing is written
    c = I8Case([4], 20, 32)
    t = c.tensors()
    lhs, rhs, p, dst, groups = c.args(t)
    groups.offsets = groups.offsets[:1]           # no groups at all
    rb.mul_grouped_async(lhs, rhs, p, ctx, dst, groups)
    ctx.sync()
    assert bool((t["y"] == c.fill).all())


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[6, 5, 4], [60, 50, 400]])
def test_grouped_offsets_out_of_order_or_range_touch_nothing_else(ctx, sizes):
    c = I8Case(sizes, 40, 64, pad=6, dst_pad=8)
    n = sum(sizes)
    for offsets, means in (([-5, 3, 2 ** 31 - 1, 2], [(0, 0, 3), (1, 3, c.cols)]),
                           ([n, n, 1, n + 100], [(2, 1, c.cols)]), ([4, -2 ** 31, 9, 9], [(1, 0, 9)])):
        t = c.tensors()
        import torch
        t["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        got = c.run(ctx, t)
        want = c.y.copy()
        for g, a, b in means:      # group g owns columns a to b, the other two are empty
            want[a:b] = c.want([a] * (g + 1) + [b] * (3 - g))[a:b]
        np.testing.assert_array_equal(got, want)


@pytest.mark.gpu
def test_grouped_equals_the_mul_of_each_group(ctx):
    c = I8Case([40, 0, 9, 300], 96, 160, rhs_zp=3, dst_zp=-4)
    t = c.tensors()
    got = c.run(ctx, t)
    for g, (a, b) in enumerate(zip(c.offsets, c.offsets[1:])):
        if a == b:
            continue
        import torch
        y = torch.zeros((b - a, c.rows), dtype=torch.int8, device="cuda")
        p = rb.MulParams("int32", "int8")
        p.bias, p.multiplier_fixedpoint_perchannel, p.multiplier_exponent_perchannel = t["bias"][g], t["mfp"][g], t["mexp"][g]
        p.rounding = rb.Rounding.kReference
        rb.mul_async(rb.Matrix(t["w"][g], rb.Layout(c.rows, c.depth, c.w_stride, RowMajor)),
                     rb.Matrix(t["x"][a:b], rb.Layout(c.depth, int(b - a), c.x_stride, ColMajor), 3), p, ctx,
                     rb.Matrix(y, rb.Layout(c.rows, int(b - a), c.rows, ColMajor), -4))
        ctx.sync()
        np.testing.assert_array_equal(got[a:b], y.cpu().numpy())


@pytest.mark.gpu
def test_host_pointers_and_misaligned_elements_are_refused(ctx):
    c = I8Case([4], 20, 32, dst="i32")
    for name in ("w", "x", "y", "offsets", "bias"):
        t = c.tensors()
        t[name] = t[name].cpu()
        lhs, rhs, p, dst, groups = c.args(t)
        with pytest.raises(rb.RuyError, match="device pointers"):
            rb.mul_grouped_async(lhs, rhs, p, ctx, dst, groups)
    t = c.tensors()
    lhs, rhs, p, dst, groups = c.args(t)
    d, g = rb.make_desc(lhs, rhs, p, dst), groups.to_desc()
    d.dst.data += 2
    assert lib().ruyb200_mul_grouped_async(ctx._h, C.byref(d), C.byref(g)) == _abi.ERR_INVALID


def _graph_test(runs):
    """Two captured graphs of different sizes, replayed at once on two streams, against eager calls."""
    import torch
    streams = [torch.cuda.Stream() for _ in runs]
    graphs, outs, keep = [], [], []
    for stream, run in zip(streams, runs):
        context = rb.Context(0, stream.cuda_stream)
        t = run.tensors()
        keep.append((context, t))
        run.run(context, t)                      # sets the kernel's attributes
        want = t["y"].clone()
        t["y"].fill_(run.fill)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run.enqueue(context, t)
        assert bool((t["y"] == run.fill).all())
        graphs.append(graph)
        outs.append((t["y"], want))
    for _ in range(3):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in outs:
        assert torch.equal(got, want)
    del graphs
    for context, _ in keep:
        context.close()


@pytest.mark.gpu
def test_grouped_in_two_graphs_at_once():
    _graph_test([I8Case([3, 0, 2], 256, 512, rhs_zp=1), I8Case([300, 70, 0, 5], 384, 256, lhs="u8", lhs_zp=128, seed=3)])


@pytest.mark.gpu
def test_grouped_weights_beyond_2_31_elements(ctx):
    import torch
    groups, rows, depth = 9, 16384, 16384
    w = torch.zeros((groups, rows, depth), dtype=torch.int8, device="cuda")
    w[8] = torch.randint(-127, 128, (rows, depth), dtype=torch.int8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    x = torch.randint(-127, 128, (260, depth), dtype=torch.int8, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    for cols in (2, 260):
        y = torch.zeros((cols, rows), dtype=torch.int32, device="cuda")
        off = torch.tensor([0] * groups + [cols], dtype=torch.int32, device="cuda")
        rb.mul_grouped_async(rb.Matrix(w, rb.Layout(rows, depth, depth, RowMajor)), rb.Matrix(x, rb.Layout(depth, cols, depth, ColMajor)),
                             rb.MulParams("int32", "int32"), ctx, rb.Matrix(y, rb.Layout(rows, cols, rows, ColMajor)),
                             rb.Groups(off, rows * depth))
        ctx.sync()
        want = (x[:cols].double() @ w[8].double().t()).to(torch.int32)
        assert torch.equal(y, want)


class Q4Case:
    """A mul with 4-bit weights.  `whole`: activations are small integers and scales powers of two, so that every sum is
    exact in 32 bits and the answer is the exact one, rounded once."""

    def __init__(self, rows, depth, cols=None, sizes=None, x="f32", y=None, scale="f32", block=32, signed=True, zeros=False, bias=True,
                 clamp=None, whole=True, w_stride=None, x_order=ColMajor, y_order=ColMajor, x_pad=0, y_pad=0, scale_pad=0, pad=0,
                 first=0, shared=False, seed=0):
        import torch
        self.T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
        gen = torch.Generator().manual_seed(seed)
        self.rows, self.depth, self.sizes, self.block, self.signed, self.whole = rows, depth, sizes, block, signed, whole
        self.x_type, self.y_type, self.scale_type = x, y or x, scale
        n = len(sizes) if sizes is not None else 1
        self.cols = first + sum(sizes) + pad if sizes is not None else cols
        self.offsets = torch.tensor([first + sum(sizes[:i]) for i in range(n + 1)], dtype=torch.int32) if sizes is not None else None
        gw = 1 if shared else n
        self.w_stride = w_stride if w_stride is not None else -(-depth // 32) * 32
        self.blocks = -(-depth // block)
        self.scale_stride = self.blocks + scale_pad
        self.w = torch.randint(0, 256, (gw, rows, self.w_stride // 2), generator=gen, dtype=torch.uint8)
        shape = (gw, rows, self.scale_stride)
        if whole:
            self.scales = torch.pow(2.0, torch.randint(-3, 1, shape, generator=gen).float())
            values = torch.randint(-4, 5, (self.cols, depth), generator=gen).float()
            self.bias = torch.randint(-9, 10, (gw, rows), generator=gen).float() if bias else None
        else:
            self.scales = torch.rand(shape, generator=gen) * 0.01 + 0.001
            values = torch.randn((self.cols, depth), generator=gen)
            self.bias = torch.randn((gw, rows), generator=gen) if bias else None
        self.scales = self.scales.to(self.T[scale])
        low, high = (-8, 8) if signed else (0, 16)
        self.zeros = torch.randint(low, high, shape, generator=gen).to(torch.int8) if zeros else None
        self.shared = shared
        self.x_order, self.y_order = x_order, y_order
        self.x_stride = (depth if x_order == ColMajor else self.cols) + x_pad
        self.y_stride = (rows if y_order == ColMajor else self.cols) + y_pad
        xs = (self.cols, self.x_stride) if x_order == ColMajor else (depth, self.x_stride)
        self.x = torch.full(xs, float("nan")).to(self.T[x])       # what lies between the columns is never used
        values = values.to(self.T[x])
        if x_order == ColMajor:
            self.x[:, :depth] = values
        else:
            self.x[:, :self.cols] = values.t()
        self.values = values
        ys = (self.cols, self.y_stride) if y_order == ColMajor else (rows, self.y_stride)
        self.fill = 77.0
        self.y = torch.full(ys, self.fill).to(self.T[self.y_type])
        self.clamp = clamp

    def logical(self, y):
        return y[:, :self.rows] if self.y_order == ColMajor else y[:, :self.cols].t()

    def want(self):
        """(answer in 64 bits, sum of the products' magnitudes); NaN where nothing is written."""
        import torch
        q = torch.stack((self.w & 15, self.w >> 4), -1).flatten(-2).double()[..., :self.depth]
        if self.signed:
            q = torch.where(q > 7, q - 16, q)
        k = torch.arange(self.depth) // self.block
        if self.zeros is not None:
            q = q - self.zeros.double()[..., k]
        w = q * self.scales.double()[..., k]
        x = self.values.double()
        out = torch.full((self.cols, self.rows), float("nan"), dtype=torch.float64)
        size = torch.zeros_like(out)
        ends = self.offsets.tolist() if self.offsets is not None else [0, self.cols]
        for g, (a, b) in enumerate(zip(ends, ends[1:])):
            i = 0 if self.shared else g
            bias = self.bias[i].double() if self.bias is not None else 0.0
            out[a:b] = x[a:b] @ w[i].t() + bias
            size[a:b] = x[a:b].abs() @ w[i].abs().t() + (bias.abs() if self.bias is not None else 0.0)
        if self.clamp:
            out = out.clamp(*self.clamp)
        return out, size

    def tensors(self):
        return {name: None if getattr(self, name) is None else getattr(self, name).cuda()
                for name in ("w", "x", "y", "scales", "zeros", "bias", "offsets")}

    def enqueue(self, ctx, t):
        lhs = rb.Q4Matrix(t["w"], rb.Layout(self.rows, self.depth, self.w_stride, RowMajor),
                          rb.Q4Scales(t["scales"], self.block, self.scale_stride, t["zeros"]), self.signed)
        rhs = rb.Matrix(t["x"], rb.Layout(self.depth, self.cols, self.x_stride, self.x_order))
        dst = rb.Matrix(t["y"], rb.Layout(self.rows, self.cols, self.y_stride, self.y_order))
        p = rb.MulParams("float32", "float32")
        p.bias = t["bias"]
        if self.clamp:
            p.clamp_min, p.clamp_max = self.clamp
        if self.offsets is None:
            rb.mul_q4_async(lhs, rhs, p, ctx, dst)
        else:
            own = 0 if self.shared else 1
            rb.mul_grouped_q4_async(lhs, rhs, p, ctx, dst, rb.Groups(t["offsets"], own * self.rows * self.w_stride, own * self.rows,
                                                                      own * self.rows * self.scale_stride))

    def run(self, ctx, t=None):
        t = t or self.tensors()
        self.enqueue(ctx, t)
        ctx.sync()
        return t["y"].cpu()

    def check(self, ctx, kernel=None):
        import torch
        y = self.run(ctx)
        if kernel:
            assert ctx.counters()["last_kernel"] == kernel
        got = self.logical(y).double()
        want, size = self.want()
        written = ~torch.isnan(want)
        assert bool((got[~written] == self.fill).all()), "a column outside the groups was written"
        rest = torch.ones_like(y, dtype=torch.bool)
        self.logical(rest)[:] = False
        assert bool((y[rest] == self.fill).all()), "an element between the columns was written"
        if self.whole:
            exact = want.to(self.T[self.y_type]).double()
            assert torch.equal(got[written], exact[written]), (got - exact)[written].abs().max()
            return
        # a sum of n products in 32 bits, in any order, with every product and every sum off by at most one unit in
        # the last place (a truncating adder; 2**-23 relative), the scaled weight and the scaled partial sum rounded
        # once more each; then half a step of the destination's type, and half of its smallest step
        half = torch.finfo(self.T[self.y_type]).eps / 2
        tol = (self.depth + 8) * 2.0 ** -23 * size * (1 + half) + half * want.abs() + torch.finfo(self.T[self.y_type]).tiny
        assert bool(((got - want).abs() <= tol)[written].all()), ((got - want).abs() / tol)[written].max()


Q4_SHAPES = [(1, 1), (3, 33), (16, 32), (40, 96), (64, 128), (65, 255), (130, 300), (200, 1024), (129, 2600)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,depth", Q4_SHAPES)
@pytest.mark.parametrize("cols", [1, 2, 3, 5, 8, 9, 16, 17, 33, 70])
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
def test_q4_shapes(ctx, rows, depth, cols, x):
    Q4Case(rows, depth, cols, x=x, y="f32", block=64, zeros=True, seed=cols).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [32, 64, 96, 128, 160, 256, 1024, 8192])
@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("x,scale", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16")])
def test_q4_blocks_types_and_zero_points(ctx, block, signed, zeros, x, scale):
    Q4Case(70, 1100, 6, x=x, scale=scale, block=block, signed=signed, zeros=zeros, scale_pad=3).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,depth,cols", [(100, 64, 1), (300, 700, 7), (96, 4200, 20)])
@pytest.mark.parametrize("y", ["same", "f32"])
def test_q4_within_the_rounding_bound(ctx, x, rows, depth, cols, y):
    Q4Case(rows, depth, cols, x=x, y=x if y == "same" else "f32", block=64, zeros=True, whole=False).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("x_order", [ColMajor, RowMajor])
@pytest.mark.parametrize("y_order", [ColMajor, RowMajor])
@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_q4_orders_strides_and_clamp(ctx, x_order, y_order, x):
    Q4Case(77, 200, 9, x=x, x_order=x_order, y_order=y_order, x_pad=5, y_pad=3, clamp=(-20.0, 31.5)).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("w_stride,x", [(202, "f32"), (250, "f16"), (208, "bf16")])
def test_q4_unaligned_weights(ctx, w_stride, x):
    Q4Case(50, 201, 11, x=x, w_stride=w_stride, zeros=True, block=32).check(ctx, "generic")
    Q4Case(50, 201, sizes=[3, 0, 12], x=x, w_stride=w_stride, zeros=True, block=96, pad=2).check(ctx, "generic")


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s[:7])))
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,depth", [(5, 40), (150, 600)])
def test_grouped_q4_sizes(ctx, sizes, x, rows, depth):
    Q4Case(rows, depth, sizes=sizes, x=x, scale="f16", block=96, zeros=True, signed=False, pad=4, first=3, y_pad=1).check(ctx)


@pytest.mark.gpu
def test_grouped_q4_shared_weights_depth_zero_and_empty(ctx):
    Q4Case(33, 64, sizes=[2, 0, 11], shared=True).check(ctx)
    Q4Case(33, 0, sizes=[2, 0, 11], w_stride=32, scale_pad=1).check(ctx)
    Q4Case(33, 0, 4, w_stride=32, scale_pad=1, x="bf16").check(ctx)
    Q4Case(33, 64, sizes=[0, 0], pad=3).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("clamp", [None, (-5.0, 5.0)])
def test_q4_infinities_and_nan(ctx, x, clamp):
    import torch
    c = Q4Case(80, 320, 6, x=x, block=32, zeros=True, bias=False, clamp=clamp)
    c.x[1, 70] = c.values[1, 70] = float("inf")
    c.x[2, 319] = c.values[2, 319] = float("-inf")
    c.x[3, 0] = c.values[3, 0] = float("nan")
    c.x[4, 5] = c.values[4, 5] = float("inf")
    c.x[4, 300] = c.values[4, 300] = float("-inf")
    got = c.logical(c.run(ctx)).double()
    want = c.want()[0].to(c.T[x]).double()       # a zero weight times an infinity is a NaN in both
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    there = ~torch.isnan(want)
    assert torch.equal(got[there], want[there])
    assert not bool(torch.isnan(got[0]).any()) and not bool(torch.isnan(got[5]).any())


@pytest.mark.gpu
def test_q4_padded_columns_hold_nan(ctx):
    import torch
    c = Q4Case(64, 256, sizes=[3, 2], pad=6, x="bf16", block=64)
    c.x[5:] = float("nan")           # a padded batch: nothing of it reaches the sequences' columns
    c.check(ctx)


@pytest.mark.gpu
def test_q4_in_two_graphs_at_once():
    _graph_test([Q4Case(512, 2048, 3, x="bf16", block=128), Q4Case(256, 1024, sizes=[1, 0, 30], x="f32", pad=2)])


@pytest.mark.gpu
def test_q4_weights_beyond_2_32_elements(ctx):
    import torch
    groups, rows, depth = 17, 16384, 16384
    gen = torch.Generator("cuda").manual_seed(1)
    w = torch.zeros((groups, rows, depth // 2), dtype=torch.uint8, device="cuda")
    w[16] = torch.randint(0, 256, (rows, depth // 2), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.ones((1,), device="cuda")
    x = torch.randint(-2, 3, (3, depth), device="cuda", generator=gen).to(torch.bfloat16)
    y = torch.zeros((3, rows), device="cuda")
    off = torch.tensor([0] * groups + [3], dtype=torch.int32, device="cuda")
    one = torch.full((groups, rows, 1), 0.5, device="cuda")
    rb.mul_grouped_q4_async(rb.Q4Matrix(w, rb.Layout(rows, depth, depth, RowMajor), rb.Q4Scales(one, depth, 1)),
                            rb.Matrix(x, rb.Layout(depth, 3, depth, ColMajor)), rb.MulParams("float32", "float32"), ctx,
                            rb.Matrix(y, rb.Layout(rows, 3, rows, ColMajor)), rb.Groups(off, rows * depth, 0, rows))
    ctx.sync()
    q = torch.stack((w[16] & 15, w[16] >> 4), -1).flatten(-2).float()
    q = torch.where(q > 7, q - 16, q)
    assert torch.equal(y.double(), 0.5 * (x.double() @ q.double().t()))


@pytest.mark.gpu
def test_q4_pointer_refusals(ctx):
    c = Q4Case(20, 64, sizes=[4], x="f16", zeros=True)
    for name in ("w", "x", "y", "scales", "zeros", "bias", "offsets"):
        t = c.tensors()
        t[name] = t[name].cpu()
        with pytest.raises(rb.RuyError, match="device pointers"):
            c.enqueue(ctx, t)


@pytest.mark.gpu
def test_expert_layer_in_8_and_4_bits():
    """Both forms as a mixture-of-experts layer runs them: columns sorted by expert on the device, the product in 8 bits,
    its int32 result scaled to half precision, the second product in 4 bits, on a stream of its own and as a graph."""
    import torch
    gen = torch.Generator("cuda").manual_seed(5)
    experts, tokens, width, inner = 6, 37, 256, 384
    stream = torch.cuda.Stream()
    context = rb.Context(0, stream.cuda_stream)
    choice = torch.randint(0, experts, (tokens,), device="cuda", generator=gen)
    x = torch.randint(-5, 6, (tokens, width), device="cuda", generator=gen).to(torch.int8)
    w1 = torch.randint(-3, 4, (experts, inner, width), device="cuda", generator=gen).to(torch.int8)
    w2 = torch.randint(0, 256, (experts, width, inner // 2), device="cuda", generator=gen, dtype=torch.uint8)
    s2 = torch.pow(2.0, torch.randint(-2, 1, (experts, width, inner // 128), device="cuda", generator=gen).float())
    h32 = torch.empty((tokens, inner), dtype=torch.int32, device="cuda")
    h = torch.empty((tokens, inner), dtype=torch.float32, device="cuda")
    y = torch.empty((tokens, width), dtype=torch.float32, device="cuda")
    xs, off, order = torch.empty_like(x), torch.zeros(experts + 1, dtype=torch.int32, device="cuda"), torch.empty_like(choice)

    def layer():
        order.copy_(torch.argsort(choice, stable=True))
        off[1:] = torch.cumsum((choice[:, None] == torch.arange(experts, device="cuda")).sum(0), 0).int()
        xs.copy_(x[order])
        rb.mul_grouped_async(rb.Matrix(w1, rb.Layout(inner, width, width, RowMajor)), rb.Matrix(xs, rb.Layout(width, tokens, width, ColMajor)),
                             rb.MulParams("int32", "int32"), context, rb.Matrix(h32, rb.Layout(inner, tokens, inner, ColMajor)),
                             rb.Groups(off, inner * width))
        h.copy_(h32.clamp(-20, 20))
        rb.mul_grouped_q4_async(rb.Q4Matrix(w2, rb.Layout(width, inner, inner, RowMajor), rb.Q4Scales(s2, 128, inner // 128)),
                                rb.Matrix(h, rb.Layout(inner, tokens, inner, ColMajor)), rb.MulParams("float32", "float32"), context,
                                rb.Matrix(y, rb.Layout(width, tokens, width, ColMajor)), rb.Groups(off, width * inner, 0, width * inner // 128))

    def want():
        q = torch.stack((w2 & 15, w2 >> 4), -1).flatten(-2).double()
        q = torch.where(q > 7, q - 16, q) * s2.double().repeat_interleave(128, -1)
        out = torch.einsum("tk,trk->tr", x.double(), w1[choice].double()).clamp(-20, 20)
        return torch.einsum("tk,trk->tr", out, q[choice])[order]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer()
    context.sync()
    assert torch.equal(y.double(), want())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        layer()
    choice.copy_(torch.randint(0, 3, (tokens,), device="cuda", generator=gen))    # other sizes, some experts without a token
    x.copy_(torch.randint(-5, 6, (tokens, width), device="cuda", generator=gen).to(torch.int8))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.double(), want())
    del graph
    context.close()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,rows,kernel", [
    ([3, 0, 2], 300, "grouped_mma"), ([1] * 20, 64, "grouped_mma"), ([9, 1], 300, "grouped_tc"), ([200] * 3, 100, "grouped_tc"),
    ([20, 300, 0, 45, 1, 64, 700, 33] * 5, 1100, "grouped_tc")], ids=["few", "singles", "some", "narrow", "pairs"])
@pytest.mark.parametrize("lhs,rhs,dst,zps", [
    ("i8", "i8", "i8", (0, 0, 0)), ("i8", "u8", "u8", (0, 131, 7)), ("i8", "i8", "i16", (0, -5, 100)), ("i8", "i8", "i32", (0, 3, 0)),
    ("u8", "u8", "u8", (128, 77, 3))])
def test_grouped_kernels_types_and_whole_words(ctx, sizes, rows, kernel, lhs, rhs, dst, zps):
    # destinations whose columns are whole words take another way out of the tensor-core kernel than others
    for r, dst_pad in ((rows, 0), (rows - rows % 32 + 32, 0), (rows, 4 - rows % 4 + 4), (rows, 5)):
        I8Case(sizes, r, 144, lhs, rhs, dst, *zps, pad=2, dst_pad=dst_pad).check(ctx, kernel)


@pytest.mark.gpu
@pytest.mark.parametrize("exponents", [(-31, -14), (-14, -1), (-1, 3), (-31, 3)])
@pytest.mark.parametrize("dst,zp", [("i8", -128), ("u8", 255), ("i16", -32768), ("i16", 32767)])
@pytest.mark.parametrize("sizes", [[2, 1], [50, 9]])
def test_grouped_every_shift(ctx, exponents, dst, zp, sizes):
    # shifts of 32 and more take a shorter way; the others, and zero points that do not fit into the rounding term, do not
    c = I8Case(sizes, 96, 32, dst=dst, dst_zp=zp, rhs_zp=1)
    r = np.random.default_rng(7)
    c.mexp = r.integers(exponents[0], exponents[1], c.mexp.shape).astype(np.int32)
    c.mfp = r.integers(2 ** 20, 2 ** 24, c.mfp.shape).astype(np.int32)      # results stay within 32 bits at every shift
    c.check(ctx)


@pytest.mark.gpu
def test_forced_generic_kernel(monkeypatch):
    import torch
    monkeypatch.setenv("RUYB200_FORCE_KERNEL", "generic")
    c = rb.Context(0, torch.cuda.default_stream().cuda_stream or 1)
    I8Case([40, 0, 9, 300], 96, 160, rhs_zp=3, dst_zp=-4).check(c, "generic")
    Q4Case(70, 320, sizes=[3, 0, 20], x="bf16", block=32, zeros=True).check(c, "generic")
    Q4Case(70, 320, 4, block=128, whole=False).check(c, "generic")
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1] * 30, [17, 0, 41, 90, 1]])
@pytest.mark.parametrize("x,block", [("f32", 32), ("f16", 64), ("bf16", 128), ("f32", 256)])
def test_grouped_q4_many_rows_and_long_groups(ctx, sizes, x, block):
    Q4Case(700, 1056, sizes=sizes, x=x, block=block, zeros=True, pad=1).check(ctx, "q4")


@pytest.mark.gpu
@pytest.mark.parametrize("x,power", [("f16", -20), ("f16", 8), ("bf16", -100), ("bf16", 100), ("f32", -100), ("f32", 100)])
def test_q4_small_and_large_activations(ctx, x, power):
    import torch
    c = Q4Case(60, 640, 5, x=x, y="f32", block=64, zeros=True, bias=False)
    c.values = (c.values.double() * 2.0 ** power).to(c.T[x])
    c.x[:, :c.depth] = c.values
    c.check(ctx, "q4")      # sums of small integers times a power of two: exact


@pytest.mark.gpu
def test_q4_every_weight_and_zero_point(ctx):
    """Every (q, z) that the documentation allows, one at a time, against its exact value."""
    import torch
    for signed in (True, False):
        low = -8 if signed else 0
        for x in ("f32", "f16", "bf16"):
            c = Q4Case(16, 32, 32, x=x, y="f32", block=32, signed=signed, zeros=True, bias=False)
            w = torch.zeros((16, 32), dtype=torch.uint8)
            for k in range(32):
                w[:, k] = k % 16
            c.w = (w[:, 0::2] | (w[:, 1::2] << 4)).reshape(1, 16, 16)
            c.zeros = torch.arange(low, low + 16).to(torch.int8).reshape(1, 16, 1)
            c.scales = torch.ones((1, 16, 1))
            c.values = torch.eye(32).to(c.T[x])
            c.x[:, :32] = c.values
            got = c.logical(c.run(ctx)).double()            # [k][z]
            q = torch.arange(32) % 16
            q = torch.where(q > 7, q - 16, q) if signed else q
            assert torch.equal(got, (q[:, None] - torch.arange(low, low + 16)[None, :]).double())


@pytest.mark.gpu
def test_same_result_every_time(ctx):
    import torch
    c = Q4Case(520, 4096, 5, x="f32", whole=False, block=128)
    t = c.tensors()
    first = c.run(ctx, t).clone()
    for _ in range(5):
        assert torch.equal(c.run(ctx, t), first)


@pytest.mark.gpu
@pytest.mark.parametrize("offsets,cols", [([0, 1, 0, 1, 0, 2], 2), ([3, 0, 3, 1, 3, 2, 3], 3), ([0, 1] * 40 + [4], 4)])
def test_more_groups_with_columns_than_columns(ctx, offsets, cols):
    """Offsets that decrease can give every column to many groups; with one matrix of weights for all, the answer is plain."""
    import torch
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    for rows, depth in ((40, 64), (200, 600)):
        c = I8Case([cols], rows, depth, rhs_zp=2)
        t = c.tensors()
        lhs, rhs, p, dst, groups = c.args(t)
        rb.mul_grouped_async(lhs, rhs, p, ctx, dst, rb.Groups(off, 0))
        ctx.sync()
        np.testing.assert_array_equal(t["y"].cpu().numpy(), c.want())
        q = Q4Case(rows, depth, sizes=[cols], x="bf16", block=32, zeros=True, shared=True)
        q.offsets = off.cpu()
        t = q.tensors()
        got = q.logical(q.run(ctx, t)).double()
        q.offsets = torch.tensor([0, cols], dtype=torch.int32)
        assert torch.equal(got, q.want()[0].to(torch.bfloat16).double())


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [33, 200, 1024])
def test_few_tokens_over_many_groups(ctx, groups):
    r = np.random.default_rng(groups)
    sizes = [0] * groups
    for g in r.integers(0, groups, 5):
        sizes[g] += 1
    sizes[-1] += 1
    I8Case(sizes, 70, 96, pad=2, first=1, rhs_zp=1).check(ctx, "grouped_mma")
    Q4Case(70, 96, sizes=sizes, x="f16", block=32, zeros=True, pad=2, first=1).check(ctx, "q4")
    sizes[3] += 900
    I8Case(sizes, 70, 96, pad=2, first=1, rhs_zp=1).check(ctx)
