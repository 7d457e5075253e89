"""A prompt's operators as work to be measured: matrices in microscaled four-bit floating point, and attention of packed rows.

Three operators, as a layer runs them over the rows of a prompt (and over a step's few rows):

* pack: rows quantised to four-bit floats with a scale for every few neighbours, and read back as what they stand for;
* linear: the product of two such matrices, rows and weights, with bias, GELU and residual;
* attend: softmax attention of packed sequences of different lengths over keys and values as they are.

A four-bit float (sign, two exponent bits, one of mantissa) is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, in
this order as codes 0..7, 8..15. Neighbours of a row share a scale: 32 a power of two (format "mx", one byte, the exponent
plus 127, 255 a NaN), 16 an eight-bit float of four exponent bits (format "nv", e4m3). A value is unit * scale * number, the
unit one f32 number for a matrix (1 for "mx"). Codes: [rows][k / 128 rounded up][64 bytes], the earlier of two neighbours in
the low half of a byte, columns past k zeros. Scales: blocks of 128 rows x 4 scales, row blocks outermost, 512 bytes each; of
row r and scale s in a block at byte 16 (r % 32) + 4 (r / 32) + s; those wholly past k are zeros.
"""
import functools
import importlib.util
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
FORMATS = {"mx": 0, "nv": 1}
BLOCK = {"mx": 32, "nv": 16}


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step's 16 rows quantised before a layer: latency
        dict(name="pack_step", op="pack", format="nv", dtype="bf16", rows=16, k=4_096),
        # a long prompt's rows before a wide layer: memory
        dict(name="pack_prompt", op="pack", format="nv", dtype="bf16", rows=8_192, k=8_192),
        # a pass of f32 rows whose width ends inside a block of scales
        dict(name="pack_odd", op="pack", format="mx", dtype="f32", rows=3_000, k=2_050),
        # the feed-forward's first layer for one test row (512 -> 1,024, GELU): latency
        dict(name="linear_row", op="linear", format="mx", dtype="f32", rows=1, n=1_024, k=512, act=1, residual=False),
        # a wide layer for 8 decoding requests: the weights streamed from memory
        dict(name="linear_step", op="linear", format="nv", dtype="bf16", rows=8, n=14_336, k=8_192, act=0, residual=True),
        # the feed-forward's second layer for a pass of 2,048 test rows (1,024 -> 512, residual), f32
        dict(name="linear_pass", op="linear", format="mx", dtype="f32", rows=2_048, n=512, k=1_024, act=0, residual=True),
        # the wide layer for a prompt of 4,096 tokens, GELU: the tensor cores
        dict(name="linear_prompt", op="linear", format="nv", dtype="bf16", rows=4_096, n=14_336, k=8_192, act=1, residual=False),
        # an odd layer for 300 rows
        dict(name="linear_odd", op="linear", format="mx", dtype="f16", rows=300, n=4_097, k=2_050, act=0, residual=True),
        # a prompt's attention to itself, 32 heads on 8, from one projection's output
        dict(name="attend_prompt", op="attend", dtype="bf16", seqs=1, rows=4_096, least_rows=4_096, before=0, least_before=0, heads=8, q_heads=32, width=128,
             causal=True, window=0),
        # prompts of very unequal length packed into one call
        dict(name="attend_packed", op="attend", dtype="f16", seqs=16, rows=2_048, least_rows=1, before=0, least_before=0, heads=16, q_heads=16, width=64,
             causal=True, window=0),
        # one new token each for 32 requests over 0 to 16,383 tokens before it: the keys and values streamed from memory
        dict(name="attend_step", op="attend", dtype="bf16", seqs=32, rows=1, least_rows=1, before=16_383, least_before=0, heads=8, q_heads=32, width=128,
             causal=True, window=0),
        # a pass of 2,048 test rows over 10,000 training rows at f32
        dict(name="attend_pass", op="attend", dtype="f32", seqs=1, rows=2_048, least_rows=2_048, before=7_952, least_before=7_952, heads=4, q_heads=4, width=128,
             causal=False, window=0),
    ]


def _spread(rng, low, high):
    """A whole number of low..high, spread over the logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["pack", "linear", "linear", "attend", "attend"])
    dtype, fmt = rng.choice(["f32", "f16", "bf16"]), rng.choice(["mx", "nv"])
    if op == "pack":
        k = _spread(rng, 1, 16_000)
        return dict(op=op, format=fmt, dtype=dtype, rows=_spread(rng, 1, 60_000_000 // k), k=k)
    if op == "linear":
        rows, n = _spread(rng, 1, 4_096), _spread(rng, 10, 14_336)
        return dict(op=op, format=fmt, dtype=dtype, rows=rows, n=n, k=_spread(rng, 16, 8_192), act=rng.randint(0, 1),
                    residual=rng.random() < 0.5)
    heads = rng.choice([1, 2, 4, 8])
    q_heads, width = heads * rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([32, 64, 64, 96, 128, 128, 256])
    causal = rng.random() < 0.7
    window = _spread(rng, 1, 3_000) if causal and rng.random() < 0.3 else 0
    kind = rng.choice(["step", "few", "prompt", "prompt"])
    if kind == "step":
        seqs, rows, least_rows, least_before = _spread(rng, 1, 64), 1, 1, 0
        before = _spread(rng, 1, max(2, min(60_000, 200_000_000 // (seqs * heads * width))))
    elif kind == "few":  # (fewer tokens than rows: the first rows see nothing)
        seqs, rows, least_rows, least_before = _spread(rng, 1, 24), rng.randint(2, 40), 0, -rng.randint(0, 3)
        before = _spread(rng, 1, 6_000)
    else:
        seqs, rows = rng.randint(1, 4), _spread(rng, 64, 1_500)
        least_rows = rng.choice([0, 1, rows // 2, rows])
        least_before, before = sorted([rng.choice([0, 0, -2, 5]), rng.choice([0, 0, 0, 700])])
    return dict(op=op, dtype=dtype, seqs=seqs, rows=rows, least_rows=least_rows, before=before, least_before=least_before, heads=heads,
                q_heads=min(q_heads, 32), width=width, causal=causal, window=window)


# ---- what a program has in hand -------------------------------------------------------------------------------------

def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _unit(x, fmt):
    """A matrix's unit, a number of 32 bits: its largest magnitude becomes the largest scale times the largest number."""
    return float(x.abs().max().float() / (448.0 * 6.0)) if fmt == "nv" else 1.0


def _numbers(x, fmt, unit):
    """x [rows, k] quantised, in 64 bits (a value next to a border falls on its own side): the numbers [rows, k padded to 128]
    and the scales [rows, padded / block]."""
    rows, k = x.shape
    block = BLOCK[fmt]
    kp = -(-k // 128) * 128
    g = torch.nn.functional.pad(x.double(), (0, kp - k)).view(rows, kp // block, block)
    bad = ~torch.isfinite(g).all(-1)
    g = torch.where(bad[..., None], torch.zeros_like(g), g)
    top = g.abs().amax(-1)
    if fmt == "mx":
        scale = torch.ldexp(torch.ones_like(top), (torch.frexp(top).exponent - 3).clamp(-127, 127))
        scale = torch.where(top > 0, scale, torch.full_like(top, 2.0 ** -127))
    else:
        want = top / (6.0 * unit)
        step = torch.ldexp(torch.ones_like(want), (torch.frexp(want).exponent - 4).clamp(min=-9))
        scale = (torch.round(want / step) * step).clamp(max=448.0)
    by = (scale * unit)[..., None]
    a = torch.where(by > 0, g.abs() / torch.where(by > 0, by, torch.ones_like(by)), torch.zeros_like(g))
    step = torch.where(a < 2, torch.full_like(a, 0.5), torch.where(a < 4, torch.full_like(a, 1.0), torch.full_like(a, 2.0)))
    n = (torch.round(a / step) * step).clamp(max=6.0) * torch.where(g < 0, -1.0, 1.0)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    return n.view(rows, kp), scale


def _stored(numbers, scales, fmt):
    """Codes (uint8 [rows, padded / 2]) and scales (uint8 [row blocks, blocks of 4 scales, 32, 4, 4]) as they are stored."""
    a = numbers.abs()
    code = (torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4))).to(torch.uint8) | ((numbers < 0).to(torch.uint8) << 3)
    rows, count = scales.shape
    if fmt == "mx":
        byte = torch.where(scales.isnan(), torch.full_like(scales, 255.0), torch.frexp(scales).exponent.double() + 126.0).to(torch.uint8)
    else:
        byte = scales.float().to(torch.float8_e4m3fn).view(torch.uint8)
    full = torch.nn.functional.pad(byte, (0, -count % 4, 0, -rows % 128))
    full = full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), full


def _values(codes, scales, fmt, unit, k):
    """What stored codes and scales stand for, in 32 bits, [rows, k]."""
    rows, half = codes.shape
    code = torch.stack([codes & 15, codes >> 4], -1).view(rows, 2 * half)
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    n = table[(code & 7).long()] * (1.0 - 2.0 * (code >> 3).float())
    byte = scales.permute(0, 3, 2, 1, 4).flatten(0, 2).flatten(1)[:rows, :2 * half // BLOCK[fmt]]
    if fmt == "mx":
        s = torch.where(byte == 255, torch.full_like(byte, 0, dtype=torch.float32) + math.nan, torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte.int() - 127))
    else:
        s = byte.contiguous().view(torch.float8_e4m3fn).float()
    return (n.view(rows, -1, BLOCK[fmt]) * s[..., None] * unit).view(rows, -1)[:, :k]


def _lens(c, seed):
    """Each sequence's query rows (a case's own, so that its outputs have one shape), and its keys: as many, and those before them."""
    rng = random.Random(c["seqs"] * 104_729 + c["rows"])
    q = [rng.randint(c["least_rows"], c["rows"]) for _ in range(c["seqs"])]
    q[rng.randrange(len(q))] = c["rows"]
    rng = random.Random(seed * 7919 + 29)
    before = [rng.randint(c["least_before"], c["before"]) for _ in q]
    before[rng.randrange(len(q))] = c["before"]
    return q, [max(0, n + b) for n, b in zip(q, before)]


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"pack": _prepare_pack, "linear": _prepare_linear, "attend": _prepare_attend}[case["op"]](case, seed, gen)


def _rows(c, gen, rows, k):
    """Rows as a layer leaves them: some channels larger than others."""
    x = _rand(gen, rows, k)
    x *= 0.3 + 2.0 * torch.rand(k, generator=gen, device="cuda") ** 4
    return x


def _prepare_pack(c, seed, gen):
    x = _rows(c, gen, c["rows"], c["k"]).to(DTYPES[c["dtype"]])
    return dict(case=c, x=x, unit=_unit(x, c["format"]))


def _prepare_linear(c, seed, gen):
    dt, fmt = DTYPES[c["dtype"]], c["format"]
    st = dict(case=c)
    for name, rows in (("x", c["rows"]), ("w", c["n"])):
        parts = []
        step = max(128, 100_000_000 // c["k"] // 128 * 128)  # by parts: the numbers in 64 bits are not held all at once
        m = _rows(c, gen, rows, c["k"]) if name == "x" else _rand(gen, rows, c["k"]) / math.sqrt(c["k"])
        unit = _unit(m, fmt)
        for r in range(0, rows, step):
            parts.append(_stored(*_numbers(m[r:r + step], fmt, unit), fmt))
        st[name] = (torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), unit)
    st["bias"] = (0.1 * _rand(gen, c["n"])).to(dt)
    st["residual"] = _rand(gen, c["rows"], c["n"]).to(dt) if c["residual"] else None
    return st


def _prepare_attend(c, seed, gen):
    dt, w, h, hq = DTYPES[c["dtype"]], c["width"], c["heads"], c["q_heads"]
    q_lens, k_lens = _lens(c, seed)
    tq, tk = sum(q_lens), sum(k_lens)
    spread = 0.5 + 1.5 * torch.rand(h, w, generator=gen, device="cuda")
    if q_lens == k_lens:  # one projection's output: a token's queries, keys and values side by side
        x = _rand(gen, tq, hq + 2 * h, w)
        x[:, hq:hq + h] *= spread
        q, k, v = x.to(dt).split([hq, h, h], 1)
    else:
        q, k, v = _rand(gen, tq, hq, w).to(dt), (_rand(gen, tk, h, w) * spread).to(dt), _rand(gen, tk, h, w).to(dt)
    return dict(case=c, q=q, k=k, v=v, q_starts=_starts(q_lens), k_starts=_starts(k_lens), max_q=max(q_lens), max_k=max(k_lens),
                scale=1.0 / math.sqrt(w))


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"pack": _own_pack, "linear": _own_linear, "attend": _own_attend}[op](state)
    return {"pack": _plain_pack, "linear": _plain_linear, "attend": _plain_attend}[op](state)


def _plain_pack(st):
    c, x = st["case"], st["x"]
    numbers, scales = _numbers(x, c["format"], st["unit"])
    codes, stored = _stored(numbers, scales, c["format"])
    return _values(codes, stored, c["format"], st["unit"], c["k"]).to(x.dtype)


def _plain_linear(st):
    c = st["case"]
    x, w = (_values(*m[:2], c["format"], m[2], c["k"]) for m in (st["x"], st["w"]))
    y = torch.matmul(x, w.t()) + st["bias"].float()
    if c["act"]:
        y = 0.5 * y * (1.0 + torch.erf(y / math.sqrt(2.0)))
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(st["bias"].dtype)


def _plain_attend(st):
    c, q, k, v = st["case"], st["q"], st["k"], st["v"]
    each, h, w = c["q_heads"] // c["heads"], c["heads"], c["width"]
    n, most, seqs = st["max_q"], max(1, st["max_k"]), c["seqs"]
    if not q.shape[0]:
        return torch.zeros_like(q), torch.zeros(q.shape[:2], device=q.device)
    qs, ks = st["q_starts"].long(), st["k_starts"].long()
    q_len, k_len = (qs[1:] - qs[:-1]).view(seqs, 1), (ks[1:] - ks[:-1]).view(seqs, 1)
    i, j = torch.arange(n, device=q.device).view(1, n), torch.arange(most, device=q.device).view(1, most)
    # every sequence filled up to the longest: its rows [seq, row, head, width] and [seq, head, token, width]
    qp = q[(qs[:-1, None] + i).clamp(max=q.shape[0] - 1)].float().view(seqs, n, h, each, w).permute(0, 2, 3, 1, 4).flatten(2, 3)
    inside = (j < k_len)[:, None, :, None]
    if k.shape[0]:
        at = (ks[:-1, None] + j).clamp(max=k.shape[0] - 1)
        kp, vp = (torch.where(inside, x[at].float().transpose(1, 2), torch.zeros((), device=q.device)) for x in (k, v))
    else:
        kp = vp = torch.zeros(seqs, h, most, w, device=q.device)
    s = torch.matmul(qp, kp.transpose(-1, -2)).mul_(st["scale"]).unflatten(2, (each, n))
    last = (k_len - q_len + i)[..., None]  # the last token that a row sees where it sees none after it
    seen = (j[:, None] < k_len[..., None]).expand(seqs, n, most)
    if c["causal"]:
        seen = seen & (j[:, None] <= last)
    if c["window"]:
        seen = seen & (j[:, None] > last - c["window"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), vp).unflatten(2, (each, n))
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log()).squeeze(-1)
    row = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(qs, row, right=True) - 1
    at = row - qs[seq]
    return o[seq, :, :, at].reshape(q.shape).to(q.dtype), lse[seq, :, :, at].reshape(q.shape[:2])


# ---- the same through the framework ---------------------------------------------------------------------------------

@functools.lru_cache(None)
def _framework():
    """The framework's package (its folder's name is not an identifier) and a context on the current device."""
    name = "tabicl_anywhere_b200"
    if name not in sys.modules:
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tabicl-anywhere_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(here, "__init__.py"), submodule_search_locations=[here])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name], sys.modules[name].Gpu(torch.cuda.current_device())


def _stream():
    # 1 is CUDA's name for the legacy default stream (0 stands for the context's own)
    return torch.cuda.current_stream().cuda_stream or 1


def _own_pack(st):
    c, x = st["case"], st["x"]
    if "m" not in st:  # the buffers that a program keeps for a layer's quantised rows
        tcu, gpu = _framework()
        fmt = FORMATS[c["format"]]
        st["codes"] = torch.empty(tcu.Fp4.code_bytes(c["rows"], c["k"]), dtype=torch.uint8, device=x.device)
        st["scales"] = torch.empty(tcu.Fp4.scale_bytes(c["rows"], c["k"], fmt), dtype=torch.uint8, device=x.device)
        st["m"] = tcu.Fp4(gpu, c["rows"], c["k"], fmt, st["codes"].data_ptr(), st["scales"].data_ptr(), unit=st["unit"])
    stream = _stream()
    st["m"].pack(CODES[c["dtype"]], x.data_ptr(), x.stride(0), stream=stream)
    y = torch.empty_like(x)
    st["m"].load(CODES[c["dtype"]], y.data_ptr(), y.stride(0), stream=stream)
    return y


def _own_linear(st):
    c, bias, r = st["case"], st["bias"], st["residual"]
    if "w4" not in st:
        tcu, gpu = _framework()
        for name, rows in (("x", c["rows"]), ("w", c["n"])):
            codes, scales, unit = st[name]
            st[name + "4"] = tcu.Fp4(gpu, rows, c["k"], FORMATS[c["format"]], codes.data_ptr(), scales.data_ptr(), unit=unit)
        need = st["w4"].linear_workspace(st["x4"], CODES[c["dtype"]])
        st["work"] = torch.zeros(max(1, need), dtype=torch.uint8, device=bias.device)
    y = torch.empty(c["rows"], c["n"], dtype=bias.dtype, device=bias.device)
    st["w4"].linear(st["x4"], CODES[c["dtype"]], y.data_ptr(), c["n"], bias=bias.data_ptr(), act=c["act"],
                    residual=r.data_ptr() if r is not None else None, ldr=c["n"], work=st["work"].data_ptr(),
                    work_bytes=st["work"].numel(), stream=_stream())
    return y


def _own_attend(st):
    c, q, k, v = st["case"], st["q"], st["k"], st["v"]
    code, hq, w = CODES[c["dtype"]], c["q_heads"], c["width"]
    if "packed" not in st:  # the step's plan and workspace, kept from layer to layer
        tcu, gpu = _framework()
        st["packed"] = tcu.Packed(gpu, c["seqs"], q.shape[0], k.shape[0], st["max_q"], st["max_k"], st["q_starts"].data_ptr(),
                                  st["k_starts"].data_ptr())
        need = st["packed"].attend_workspace(code, hq, c["heads"], w)
        st["work"] = torch.zeros(max(1, need), dtype=torch.uint8, device=q.device)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    st["packed"].attend(code, hq, c["heads"], w, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                        v.data_ptr(), v.stride(0), v.stride(1), out.data_ptr(), hq * w, w, st["scale"], causal=c["causal"],
                        window=c["window"], lse=lse.data_ptr(), work=st["work"].data_ptr(), work_bytes=st["work"].numel(),
                        stream=_stream())
    return out, lse


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def _held(c, rows):
    """Bytes of a quantised matrix."""
    return rows * c["k"] // 2 + rows * -(-c["k"] // BLOCK[c["format"]])


def work(case):
    c = case
    s = SIZE[c["dtype"]]
    if c["op"] == "pack":
        values = c["rows"] * c["k"]
        return {"bytes": 2 * values * s + 2 * _held(c, c["rows"]), "flops": 4 * values}
    if c["op"] == "linear":
        m, n = c["rows"], c["n"]
        return {"bytes": _held(c, m) + _held(c, n) + s * (n + m * n * (2 if c["residual"] else 1)), "flops": 2 * m * n * c["k"]}
    pairs = keys = rows = 0
    for n, length in zip(*_lens(c, 0)):
        first = length
        for i in range(n):
            high = max(0, min(length, length - n + i + 1)) if c["causal"] else length
            low = max(0, length - n + i + 1 - c["window"]) if c["window"] else 0
            if high > low:
                pairs += high - low
                first = min(first, low)
        keys, rows = keys + length - first, rows + n
    return {"bytes": s * c["width"] * (2 * keys * c["heads"] + 2 * rows * c["q_heads"]) + 4 * rows * c["q_heads"],
            "flops": 4 * pairs * c["q_heads"] * c["width"]}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"pack": _exact_pack, "linear": _exact_linear, "attend": _exact_attend}[case["op"]](st)


NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_pack(st):
    """Every number found by the borders that it lies between; of one on a border the neighbour of even code."""
    c, x = st["case"], st["x"].double()
    block, unit = BLOCK[c["format"]], st["unit"]
    out = torch.empty_like(x)
    step = max(1, 20_000_000 // x.shape[1])
    eighths = torch.tensor([b for e in range(-6, 9) for b in [2.0 ** e * m / 8 for m in range(8, 16)]], dtype=torch.float64, device=x.device)
    eighths = torch.cat([torch.arange(8, device=x.device).double() * 2.0 ** -9, eighths])[:127]  # the finite e4m3, 0 to 448
    for r in range(0, x.shape[0], step):
        for first in range(0, x.shape[1], block):
            g = x[r:r + step, first:first + block]
            top = g.abs().max(1, keepdim=True).values
            if c["format"] == "mx":
                scale = torch.exp2(torch.floor(torch.log2(top)).clamp(-125, 127) - 2)
                scale = torch.where(scale * 8 <= top, scale * 2, torch.where(scale * 4 > top, scale / 2, scale))  # (a logarithm's rounding)
            else:
                want = (top / (6 * unit)).clamp(max=448)
                up = torch.searchsorted(eighths, want).clamp(max=126)
                down = (up - 1).clamp(min=0)
                above, below = eighths[up] - want, want - eighths[down]
                scale = eighths[torch.where((above < below) | ((above == below) & (up % 2 == 0)), up, down)]
            by = scale * unit
            a = torch.where(by > 0, g.abs() / by, torch.zeros_like(g))
            code = torch.zeros_like(a)
            for low in range(7):
                middle = (NUMBERS[low] + NUMBERS[low + 1]) / 2
                code += ((a > middle) | ((a == middle) & (low % 2 == 1))).double()
            number = torch.tensor(NUMBERS, dtype=torch.float64, device=x.device)[code.long()]
            out[r:r + step, first:first + block] = torch.where(g < 0, -number, number) * by
    return out


def _exact_matrix(m, c):
    """[rows, k]: each value from its byte and its scale's, by their documented places."""
    codes, scales, unit = m
    rows, dev = codes.shape[0], codes.device
    j, r = torch.arange(c["k"], device=dev), torch.arange(rows, device=dev)[:, None]
    code = (codes[:, j // 2] >> (4 * (j % 2))) & 15
    number = torch.tensor(NUMBERS + [-v for v in NUMBERS], dtype=torch.float64, device=dev)[code.long()]
    s = (torch.arange(-(-c["k"] // BLOCK[c["format"]]), device=dev))[None]
    quads = scales.shape[1]
    byte = scales.view(-1)[((r // 128) * quads + s // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + s % 4].long()
    if c["format"] == "mx":
        scale = torch.exp2(byte.double() - 127)
    else:
        e, f = byte >> 3, (byte & 7).double()
        scale = torch.where(e > 0, torch.exp2(e.double() - 7) * (1 + f / 8), f * 2.0 ** -9)
    number *= scale.repeat_interleave(BLOCK[c["format"]], 1)[:, :c["k"]]
    return number * unit


def _exact_linear(st):
    c = st["case"]
    y = _exact_matrix(st["x"], c) @ _exact_matrix(st["w"], c).t() + st["bias"].double()
    if c["act"]:
        y = torch.nn.functional.gelu(y)
    return y + st["residual"].double() if c["residual"] else y


def _exact_attend(st):
    c, q = st["case"], st["q"]
    each, w = c["q_heads"] // c["heads"], c["width"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    qs, ks = st["q_starts"].tolist(), st["k_starts"].tolist()
    for s in range(c["seqs"]):
        rows, n, length = slice(qs[s], qs[s + 1]), qs[s + 1] - qs[s], ks[s + 1] - ks[s]
        if not n or not length:
            continue
        i, j = torch.arange(n, device=q.device)[:, None] + length - n, torch.arange(length, device=q.device)[None]
        hidden = torch.zeros(n, length, dtype=torch.bool, device=q.device)
        if c["causal"]:
            hidden |= j > i
        if c["window"]:
            hidden |= j <= i - c["window"]
        for head in range(c["q_heads"]):
            k, v = (x[ks[s]:ks[s + 1], head // each].double() for x in (st["k"], st["v"]))
            a = (q[rows, head].double() @ k.t()) * st["scale"]
            a[hidden] = -math.inf
            total = torch.logsumexp(a, -1)
            some = total > -math.inf
            lse[rows, head] = total
            o = torch.exp(a - torch.where(some, total, torch.zeros_like(total))[:, None]) @ v
            out[rows, head] = torch.where(some[:, None], o, torch.zeros_like(o))
    return out, lse
