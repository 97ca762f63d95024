"""Measured calls of the products with grouped and with 4-bit weights.

Three operators, each a product of weights (rows x depth) with activations (depth x cols, depth contiguous per column)
into a destination (rows x cols, column-major, so one token's outputs are contiguous):

  q4          4-bit weights, one scale (and optionally a zero point) per row and block of depth
  grouped_q4  the same with the columns cut into ragged groups, each with weights of its own (experts)
  grouped_i8  8-bit weights and activations, ragged groups, ruy's integer epilogue

`own` False computes them in elementary torch operations; True calls the library.
"""
import math
import random

import torch

own = False

_FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_INT = {"i8": torch.int8, "u8": torch.uint8, "i16": torch.int16, "i32": torch.int32}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "u8": 1, "i16": 2, "i32": 4}


def listed():
    return [
        # a small projection of one token: launch latency decides
        _q4("q4_small_one_token", 1024, 1024, 1, "bf16", block=32, signed=True),
        # an ordinary projection of one token, asymmetric weights
        _q4("q4_projection_one_token", 4096, 4096, 1, "bf16", block=128, signed=False),
        # the largest single-token product: weights alone are as large as the L2 cache
        _q4("q4_wide_one_token", 16384, 16384, 1, "f16", block=128, signed=True),
        # a batch of five sequences in fp32 and odd sizes: rows, depth and columns that fill no tile
        _q4("q4_odd_batch_f32", 4099, 5003, 5, "f32", block=64, signed=False),
        # sixteen sequences decoded together, the widest batch meant for this product
        _q4("q4_batch_16", 4096, 16384, 16, "bf16", block=128, signed=True),
        # one token sent to two of eight experts
        _gq4("grouped_q4_one_token", 8, 4096, 4096, 2, "bf16", block=128, signed=True),
        # a decoding batch over many small experts, skewed: some experts see no token; the batch is padded
        _gq4("grouped_q4_many_experts", 64, 1024, 2048, 96, "f16", block=64, signed=False, pad=7),
        # a larger batch over sixteen experts in fp32 with odd sizes
        _gq4("grouped_q4_odd_f32", 16, 2051, 2080, 131, "f32", block=32, signed=True),
        # one token sent to two of eight experts, 8 bits
        _gi8("grouped_i8_one_token", 8, 4096, 4096, 2, "i8", "i8", "i8"),
        # a decoding batch over many experts, raw accumulators, padded
        _gi8("grouped_i8_many_experts", 64, 1024, 2048, 512, "i8", "i8", "i32", pad=13),
        # asymmetric uint8 in odd sizes
        _gi8("grouped_i8_odd_u8", 16, 1000, 1027, 1531, "u8", "u8", "u8", lhs_zp=128, rhs_zp=77, dst_zp=3),
        # a prompt of 8192 tokens over eight experts: the tensor cores decide
        _gi8("grouped_i8_prompt", 8, 4096, 4096, 8192, "i8", "i8", "i8", rhs_zp=-3, dst_zp=5),
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["q4", "grouped_q4", "grouped_i8"])
    if op == "q4":
        rows, depth = spread(64, 16384), spread(64, 16384)
        case = _q4("", rows, depth, spread(1, 16), rng.choice(["f32", "f16", "bf16"]), block=rng.choice([32, 64, 128]),
                   signed=rng.random() < 0.5)
    else:
        groups, rows = spread(2, 64), spread(64, 4096)
        depth = min(spread(64, 4096), (8 * 4096 * 4096) // (groups * rows))
        pad = rng.choice([0, 0, 5])
        if op == "grouped_q4":
            case = _gq4("", groups, rows, depth, spread(1, 256), rng.choice(["f32", "f16", "bf16"]),
                        block=rng.choice([32, 64, 128]), signed=rng.random() < 0.5, pad=pad)
        else:
            lhs, rhs, dst = rng.choice([("i8", "i8", "i8"), ("i8", "i8", "i32"), ("i8", "i8", "i16"), ("u8", "u8", "u8"),
                                        ("i8", "u8", "i8")])
            case = _gi8("", groups, rows, depth, spread(1, 8192), lhs, rhs, dst, pad=pad,
                        lhs_zp=128 if lhs == "u8" else 0, rhs_zp=rng.choice([0, rng.randrange(0, 128)]),
                        dst_zp=rng.randrange(0, 20))
    del case["name"]
    return case


def _q4(name, rows, depth, cols, dtype, block, signed):
    return dict(name=name, op="q4", rows=rows, depth=depth, cols=cols, dtype=dtype, block=block, signed=signed)


def _gq4(name, groups, rows, depth, cols, dtype, block, signed, pad=0):
    return dict(name=name, op="grouped_q4", groups=groups, rows=rows, depth=depth, cols=cols, dtype=dtype, block=block,
                signed=signed, pad=pad)


def _gi8(name, groups, rows, depth, cols, lhs, rhs, dst, lhs_zp=0, rhs_zp=0, dst_zp=0, pad=0):
    return dict(name=name, op="grouped_i8", groups=groups, rows=rows, depth=depth, cols=cols, lhs=lhs, rhs=rhs, dst=dst,
                lhs_zp=lhs_zp, rhs_zp=rhs_zp, dst_zp=dst_zp, pad=pad)


def _sizes(case):
    """Columns per group, skewed as a router's choices are: the same for every seed of a case, in another order."""
    groups, cols = case["groups"], case["cols"]
    share = [1.0 / (1 + i) ** 0.7 for i in range(groups)]
    ends, run_ = [], 0.0
    for s in share:
        run_ += s
        ends.append(int(round(cols * run_ / sum(share))))
    return [b - a for a, b in zip([0] + ends, ends)]


def _round_up(n, to):
    return (n + to - 1) // to * to


def work(case):
    rows, depth, cols = case["rows"], case["depth"], case["cols"]
    active = sum(1 for s in _sizes(case) if s) if "groups" in case else 1
    if case["op"] == "grouped_i8":
        per = rows * depth + rows * (4 if case["dst"] == "i32" else 12)
        io = depth * cols * _BYTES[case["rhs"]] + rows * cols * _BYTES[case["dst"]]
    else:
        entry = _BYTES[_scale_type(case)] + (0 if case["signed"] else 1)
        per = rows * ((depth + 1) // 2) + rows * -(-depth // case["block"]) * entry + rows * 4
        io = (depth + rows) * cols * _BYTES[case["dtype"]]
    return {"bytes": active * per + io, "flops": 2 * rows * depth * cols}


def _scale_type(case):
    return "f16" if case["dtype"] == "f16" else "bf16" if case["dtype"] == "bf16" else "f32"


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, depth, cols = case["rows"], case["depth"], case["cols"]
    total = cols + case.get("pad", 0)
    s = dict(case, total=total)
    lead = ()
    if "groups" in case:
        lead = (case["groups"],)
        sizes = _sizes(case)
        random.Random(seed).shuffle(sizes)
        ends = [0]
        for n in sizes:
            ends.append(ends[-1] + n)
        s["longest"] = max(sizes)
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device=dev)
    if case["op"] == "grouped_i8":
        s["stride"] = _round_up(depth, 16)

        def ints(shape, kind, spread=None):
            if kind == "u8":
                return torch.randint(0, 256, shape, generator=gen, device=dev, dtype=torch.uint8)
            if spread is None:
                return torch.randint(-127, 128, shape, generator=gen, device=dev, dtype=torch.int8)
            return (torch.randn(shape, generator=gen, device=dev) * spread).round().clamp(-128, 127).to(torch.int8)

        s["w"] = ints(lead + (rows, s["stride"]), case["lhs"])
        s["x"] = ints((total, s["stride"]), case["rhs"], 40.0)
        s["bias"] = torch.randint(-1000, 1001, lead + (rows,), generator=gen, device=dev, dtype=torch.int32)
        s["y"] = torch.zeros((total, rows), device=dev, dtype=_INT[case["dst"]])
        if case["dst"] != "i32":
            # multipliers that bring the accumulators' spread into the destination's range
            e = (2 if case["dst"] == "i16" else -6) - int(round(math.log2(math.sqrt(depth))))
            s["mfp"] = torch.randint(2 ** 30, 2 ** 31 - 1, lead + (rows,), generator=gen, device=dev, dtype=torch.int32)
            s["mexp"] = torch.randint(e - 1, e + 2, lead + (rows,), generator=gen, device=dev, dtype=torch.int32)
    else:
        s["stride"] = _round_up(depth, 32)
        blocks = -(-depth // case["block"])
        s["w"] = torch.randint(0, 256, lead + (rows, s["stride"] // 2), generator=gen, device=dev, dtype=torch.uint8)
        s["scales"] = (torch.rand(lead + (rows, blocks), generator=gen, device=dev) * 0.01 + 0.002).to(_FLOAT[_scale_type(case)])
        s["zeros"] = None if case["signed"] else torch.randint(5, 11, lead + (rows, blocks), generator=gen, device=dev, dtype=torch.int8)
        x = torch.randn((total, depth), generator=gen, device=dev)
        x[:, ::61] *= 12.0   # the few channels with large activations that language models have
        s["x"] = x.to(_FLOAT[case["dtype"]])
        s["bias"] = torch.randn(lead + (rows,), generator=gen, device=dev)
        s["y"] = torch.zeros((total, rows), device=dev, dtype=_FLOAT[case["dtype"]])
    return s


def run(state):
    if own:
        return _library(state)
    if state["op"] == "grouped_i8":
        return _plain_grouped_i8(state)
    return _plain_q4(state)


# ---- the library's calls ------------------------------------------------------------------------------

_contexts = {}


def _context():
    """The context of the current stream (a program has one per stream); 1 is CUDA's handle of the default stream."""
    import ruy_b200
    stream = torch.cuda.current_stream().cuda_stream or 1
    if stream not in _contexts:
        _contexts[stream] = ruy_b200.Context(torch.cuda.current_device(), stream)
    return _contexts[stream]


def _library(s):
    import ruy_b200 as rb
    rows, depth, total = s["rows"], s["depth"], s["total"]
    dst = rb.Matrix(s["y"], rb.Layout(rows, total, rows, rb.Order.kColMajor), s.get("dst_zp", 0))
    lay = rb.Layout(rows, depth, s["stride"], rb.Order.kRowMajor)
    groups = None
    if "groups" in s:
        groups = rb.Groups(s["offsets"], lhs_stride=rows * s["stride"], channel_stride=rows)
    if s["op"] == "grouped_i8":
        lhs = rb.Matrix(s["w"], lay, s["lhs_zp"])
        rhs = rb.Matrix(s["x"], rb.Layout(depth, total, s["stride"], rb.Order.kColMajor), s["rhs_zp"])
        p = rb.MulParams("int32", {"i8": "int8", "u8": "uint8", "i16": "int16", "i32": "int32"}[s["dst"]])
        p.bias = s["bias"]
        if s["dst"] != "i32":
            p.multiplier_fixedpoint_perchannel, p.multiplier_exponent_perchannel = s["mfp"], s["mexp"]
        rb.mul_grouped_async(lhs, rhs, p, _context(), dst, groups)
        return s["y"]
    blocks = s["scales"].shape[-1]
    lhs = rb.Q4Matrix(s["w"], lay, rb.Q4Scales(s["scales"], s["block"], blocks, s["zeros"]), signed=s["signed"])
    rhs = rb.Matrix(s["x"], rb.Layout(depth, total, depth, rb.Order.kColMajor))
    p = rb.MulParams("float32", "float32")
    p.bias = s["bias"]
    if groups is None:
        rb.mul_q4_async(lhs, rhs, p, _context(), dst)
    else:
        groups.scale_stride = rows * blocks
        rb.mul_grouped_q4_async(lhs, rhs, p, _context(), dst, groups)
    return s["y"]


# ---- plain forms --------------------------------------------------------------------------------------

def _grouped_product(s, w, x):
    """(total, rows) products of every column with its group's weights, and each column's group; columns are laid out
    as one padded batch per group.  Columns behind the last group come out as group 0's and are masked by the caller."""
    off = s["offsets"].long()
    at = (off[:-1, None] + torch.arange(max(1, s["longest"]), device=x.device)).clamp_(max=s["total"] - 1)
    y = torch.bmm(x[at], w.transpose(1, 2))
    col = torch.arange(s["total"], device=x.device)
    group = torch.searchsorted(off, col, right=True) - 1
    inside = col < off[-1]
    group = torch.where(inside, group, 0)
    place = torch.where(inside, col - off[group], 0)
    return y[group, place], group, inside


def _plain_q4(s):
    depth, block = s["depth"], s["block"]
    q = torch.stack((s["w"] & 15, s["w"] >> 4), -1).flatten(-2)[..., :depth].float()
    if s["signed"]:
        q = q - 16.0 * (q > 7)
    k = torch.arange(depth, device=q.device) // block
    if s["zeros"] is not None:
        q = q - s["zeros"].float()[..., k]
    w = q * s["scales"].float()[..., k]
    x = s["x"].float()
    if "groups" in s:
        y, group, inside = _grouped_product(s, w, x)
        y = torch.where(inside[:, None], y + s["bias"][group], 0.0)
    else:
        y = x @ w.t() + s["bias"]
    return y.to(s["x"].dtype)


def _plain_grouped_i8(s):
    depth = s["depth"]
    w = s["w"][..., :depth].double() - s["lhs_zp"]     # sums beyond 2**24: exact in 64 bits
    x = s["x"][:, :depth].double() - s["rhs_zp"]
    y, group, inside = _grouped_product(s, w, x)
    y = y.long() + s["bias"].long()[group]
    if s["dst"] != "i32":
        shift = 31 - s["mexp"].long()[group]
        y = (y * s["mfp"].long()[group] + (1 << (shift - 1))) >> shift
    info = torch.iinfo(_INT[s["dst"]])
    y = (y + s["dst_zp"]).clamp(info.min, info.max)
    return torch.where(inside[:, None], y, 0).to(_INT[s["dst"]])


# ---- from the definition, in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    rows, depth = case["rows"], case["depth"]
    ends = s["offsets"].tolist() if "groups" in case else [0, s["total"]]
    kind = torch.int64 if case["op"] == "grouped_i8" else torch.float64
    out = torch.zeros((s["total"], rows), device=s["x"].device, dtype=kind)
    for g, (a, b) in enumerate(zip(ends, ends[1:])):
        if a == b:
            continue

        def part(name):
            return s[name][g] if "groups" in case else s[name]

        x = s["x"][a:b, :depth].to(torch.float64)
        if case["op"] == "grouped_i8":
            acc = (part("w")[:, :depth].to(torch.float64) - case["lhs_zp"]) @ (x - case["rhs_zp"]).t()
            v = acc.round().to(torch.int64) + part("bias").to(torch.int64)[:, None]
            if case["dst"] != "i32":
                unit = torch.pow(2, 31 - part("mexp").to(torch.int64))[:, None]
                v = torch.div(v * part("mfp").to(torch.int64)[:, None] + unit // 2, unit, rounding_mode="floor")
            v = v + case["dst_zp"]
            info = torch.iinfo(_INT[case["dst"]])
            out[a:b] = torch.clamp(v, info.min, info.max).t()
            continue
        packed = part("w").to(torch.int64)
        q = torch.empty((rows, 2 * packed.shape[1]), device=x.device, dtype=torch.int64)
        q[:, 0::2] = packed % 16
        q[:, 1::2] = packed // 16
        if case["signed"]:
            q = (q + 8) % 16 - 8
        q = q[:, :depth]
        scale = part("scales").to(torch.float64).repeat_interleave(case["block"], 1)[:, :depth]
        if s["zeros"] is not None:
            q = q - part("zeros").to(torch.int64).repeat_interleave(case["block"], 1)[:, :depth]
        out[a:b] = x @ (q.to(torch.float64) * scale).t() + part("bias").to(torch.float64)
    return out.to(_INT[case["dst"]]) if case["op"] == "grouped_i8" else out
