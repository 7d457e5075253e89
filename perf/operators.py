"""The four-bit operators and the label log-probabilities as work to be measured.

Four operators, which run one after the other in a layer and its answer held in four bits:

* store: keys and values written into a paged four-bit cache, and read back as the numbers they stand for;
* attend: softmax attention of ragged query rows over that cache;
* linear: a linear layer whose weights are four-bit codes with group scales;
* logprobs: log probabilities of given labels, the entropy, and the top alternatives.

The four-bit format: `group` neighbouring coordinates share (step, low), two f16 numbers, and a value is
low + step * code with a code of 0..15. Codes of a key of width 32 U: 32-bit word t U + u (t < 4) holds coordinates
32 u + 8 t + j in nibble j. Codes of a value: 16-bit word g U + u (g < 8) holds coordinates 32 u + 4 g + j in nibble j.
A page holds, per head, its tokens' key codes, key (step, low), value codes and value (step, low). A weight row is cut
into blocks of 128 columns (the last one filled up with zeros), each in the order of a key of width 128.
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


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of 32 requests appends one token each: latency
        dict(name="store_append", op="store", dtype="bf16", tokens=32, heads=8, width=128, group=32, page=64, pages=512),
        # a fitted cache of 100,000 rows (4 heads of 128, f32) converted whole
        dict(name="store_fitted", op="store", dtype="f32", tokens=100_000, heads=4, width=128, group=64, page=256, pages=400),
        # one test row against a 10,000-row fitted cache, f32 as the framework computes: the latency of a prediction
        dict(name="attend_row", op="attend", dtype="f32", seqs=1, rows=1, least=10_000, most=10_000, heads=4, q_heads=4,
             width=128, group=64, page=256, causal=False, window=0),
        # a decode step of 64 requests of very unequal length, grouped heads: the cache streamed from memory
        dict(name="attend_decode", op="attend", dtype="bf16", seqs=64, rows=1, least=0, most=16_384, heads=8, q_heads=32,
             width=128, group=32, page=64, causal=True, window=0),
        # a pass of 2,048 test rows against the 10,000-row cache at f32
        dict(name="attend_pass", op="attend", dtype="f32", seqs=1, rows=2_048, least=10_000, most=10_000, heads=4, q_heads=4,
             width=128, group=64, page=256, causal=False, window=0),
        # a prompt's own attention after its keys are stored, with 1,000 tokens cached before it
        dict(name="attend_prompt", op="attend", dtype="bf16", seqs=1, rows=4_096, least=5_096, most=5_096, heads=8, q_heads=32,
             width=128, group=128, page=64, causal=True, window=0),
        # the feed-forward's first layer for one test row (512 -> 1,024, GELU), f32: latency
        dict(name="linear_row", op="linear", dtype="f32", rows=1, n=1_024, k=512, group=64, act=1, residual=False),
        # a wide layer for 8 decoding requests: the weights streamed from memory
        dict(name="linear_wide", op="linear", dtype="bf16", rows=8, n=14_336, k=8_192, group=128, act=0, residual=True),
        # an odd layer for 50 rows
        dict(name="linear_odd", op="linear", dtype="f16", rows=50, n=4_097, k=2_050, group=32, act=0, residual=False),
        # the class scores of 2,048 test rows, 10 classes, softmax temperature 0.9
        dict(name="logprobs_classes", op="logprobs", dtype="f32", rows=2_048, classes=10, labels=1, top=3, temperature=0.9, masked=0.1),
        # one decode step's scores over a large vocabulary
        dict(name="logprobs_step", op="logprobs", dtype="bf16", rows=16, classes=128_000, labels=1, top=20, temperature=1.0, masked=0.0),
        # a scored prompt: every position's probability of its token, with five alternatives
        dict(name="logprobs_prompt", op="logprobs", dtype="bf16", rows=4_096, classes=131_071, labels=1, top=5, temperature=1.0, masked=0.02),
    ]


def _spread(rng, low, high):
    """A whole number of low..high, spread over the logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "linear", "linear", "logprobs"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("store", "attend"):
        width = rng.choice([32, 64, 128, 128, 256])
        group = rng.choice([g for g in (32, 64, 128) if g <= width])
        page = rng.choice([16, 32, 64, 128, 256])
    if op == "store":
        heads = rng.randint(1, 8)
        tokens = _spread(rng, 1, 50_000_000 // (heads * width))
        return dict(op=op, dtype=dtype, tokens=tokens, heads=heads, width=width, group=group, page=page,
                    pages=-(-tokens // page) + rng.randint(1, 40))
    if op == "attend":
        heads = rng.choice([1, 2, 4, 8])
        q_heads = heads * rng.choice([1, 1, 2, 3, 4, 8])
        kind = rng.choice(["decode", "few", "many"])
        if kind == "decode":
            rows, seqs = 1, _spread(rng, 1, 96)
            most = _spread(rng, 1, max(2, min(60_000, 130_000_000 // (seqs * heads * width))))
        elif kind == "few":
            rows, seqs = rng.randint(2, 17), _spread(rng, 1, 24)
            most = _spread(rng, rows, 8_000)
        else:
            rows, seqs = _spread(rng, 64, 2_500), rng.randint(1, 3)
            most = _spread(rng, rows, 9_000 if width < 256 else 5_000)
        causal = rng.random() < 0.6
        window = _spread(rng, 1, most + 1) if causal and rng.random() < 0.4 else 0
        return dict(op=op, dtype=dtype, seqs=seqs, rows=rows, least=rng.choice([0, 1, most // 2, most]), most=most, heads=heads,
                    q_heads=min(q_heads, 32), width=width, group=group, page=page, causal=causal, window=window)
    if op == "linear":
        rows, n = _spread(rng, 1, 64), _spread(rng, 10, 16_000)
        return dict(op=op, dtype=dtype, rows=rows, n=n, k=_spread(rng, 16, 9_000), group=rng.choice([32, 64, 128]),
                    act=rng.randint(0, 1), residual=rng.random() < 0.5)
    classes = _spread(rng, 2, 200_000)
    return dict(op=op, dtype=dtype, rows=_spread(rng, 1, min(20_000, 300_000_000 // classes)), classes=classes,
                labels=rng.choice([1, 1, 4]), top=rng.randint(0, 20), temperature=rng.choice([0.5, 0.9, 1.0, 1.7]),
                masked=rng.choice([0.0, 0.02, 0.5, 0.999]))


# ---- what a program has in hand -------------------------------------------------------------------------------------

def _quantise(x, group):
    """x [..., width] in 32 bits: its codes (uint8, one each) and (step, low) [..., width / group, 2] in f16."""
    g = x.float().unflatten(-1, (-1, group))
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    low = g.amin(-1, keepdim=True).clamp(-65504.0, 65504.0).half()
    # a product of two tensors' quotient: division by a plain number would multiply by its rounded reciprocal
    fifteen = torch.full((), 15.0, device=x.device)
    step = ((g.amax(-1, keepdim=True).clamp(max=65504.0) - low.float()).clamp(min=0.0) / fifteen).half()
    step = torch.where(bad, torch.zeros_like(step), step)
    low = torch.where(bad, torch.full_like(low, math.nan), low)
    s = step.float()
    code = torch.where(s > 0, torch.round((g - low.float()) / torch.where(s > 0, s, torch.ones_like(s))).clamp(0.0, 15.0),
                       torch.zeros_like(g))
    code = torch.where(bad, torch.zeros_like(code), code)
    return code.to(torch.uint8).flatten(-2), torch.cat([step, low], -1)


def _pack(code, values):
    """Codes [..., width] to bytes [..., width / 2] in the order of a key, or of a value."""
    parts, per = (8, 4) if values else (4, 8)
    c = code.unflatten(-1, (-1, parts, per)).transpose(-3, -2).flatten(-3)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _unpack(raw, values):
    """Bytes [..., width / 2] to codes [..., width] (uint8)."""
    c = torch.stack([raw & 15, raw >> 4], -1).flatten(-2)
    parts, per = (8, 4) if values else (4, 8)
    return c.unflatten(-1, (parts, -1, per)).transpose(-3, -2).flatten(-3)


def _values(raw, scales, group, values):
    """What codes [..., width / 2] and scales [..., width / group, 2] stand for, in 32 bits."""
    c = _unpack(raw, values).float().unflatten(-1, (-1, group))
    return (c * scales[..., 0:1].float() + scales[..., 1:2].float()).flatten(-2)


def _page_bytes(c):
    return c["heads"] * c["page"] * (c["width"] + 8 * (c["width"] // c["group"]))


def _parts(pool, c):
    """Views of a pool [pages, page bytes]: key codes, key scales, value codes, value scales [pages, heads, page, ...]."""
    w, g, p = c["width"], c["group"], c["page"]
    per = pool.view(pool.shape[0], c["heads"], -1)
    n1, n2 = p * w // 2, p * (w // g) * 4
    kc, ks, vc, vs = per.split([n1, n2, n1, n2], -1)
    codes = lambda b: b.unflatten(-1, (p, w // 2))  # noqa: E731
    scales = lambda b: b.view(torch.float16).unflatten(-1, (p, w // g, 2))  # noqa: E731
    return codes(kc), scales(ks), codes(vc), scales(vs)


def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"store": _prepare_store, "attend": _prepare_attend, "linear": _prepare_linear,
            "logprobs": _prepare_logprobs}[case["op"]](case, seed, gen)


def _prepare_store(c, seed, gen):
    dt = DTYPES[c["dtype"]]
    t, h, w = c["tokens"], c["heads"], c["width"]
    # keys and values as a layer's projection leaves them: one row a token, keys beside values, some channels larger
    kv = _rand(gen, t, 2, h, w)
    kv[:, 0] *= 0.5 + 3.0 * torch.rand(h, w, generator=gen, device="cuda")
    kv[:, 0] += _rand(gen, h, w)
    slots = torch.randperm(c["pages"] * c["page"], generator=gen, device="cuda")[:t].to(torch.int64)
    slots = slots.sort().values if t > 4096 else slots
    return dict(case=c, kv=kv.to(dt), slots=slots, pool=torch.zeros(c["pages"], _page_bytes(c), dtype=torch.uint8, device="cuda"))


def _lens(c, seed):
    rng = random.Random(seed * 7919 + 13)
    lens = [rng.randint(min(c["least"], c["most"]), c["most"]) for _ in range(c["seqs"])]
    lens[rng.randrange(len(lens))] = c["most"]
    return lens


def _prepare_attend(c, seed, gen):
    dt = DTYPES[c["dtype"]]
    w, h, p = c["width"], c["heads"], c["page"]
    lens = _lens(c, seed)
    per_seq = -(-c["most"] // p)
    used = [-(-n // p) for n in lens]
    pages = sum(used) + 3
    # tokens as a quantiser leaves them: a stock of a few thousand, laid over the pages in a shuffled order
    stock = 4096
    x = _rand(gen, 2, stock, w)
    x[0] = x[0] * (0.5 + 2.0 * torch.rand(w, generator=gen, device="cuda")) + _rand(gen, w)
    code, sc = _quantise(x, c["group"])
    pool = torch.zeros(pages, _page_bytes(c), dtype=torch.uint8, device="cuda")
    pick = torch.randint(0, stock, (2, pages, h, p), generator=gen, device="cuda")
    kc, ks, vc, vs = _parts(pool, c)
    kc.copy_(_pack(code[0], False)[pick[0]])
    vc.copy_(_pack(code[1], True)[pick[1]])
    ks.copy_(sc[0][pick[0]])
    vs.copy_(sc[1][pick[1]])
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((c["seqs"], max(1, per_seq)), -1, dtype=torch.int32)
    at, host = 0, order.cpu()
    for s, n in enumerate(used):
        table[s, :n] = host[at:at + n]
        at += n
    q = _rand(gen, c["seqs"] * c["rows"], c["q_heads"], w).to(dt)
    return dict(case=c, q=q, pool=pool, table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                scale=1.0 / math.sqrt(w))


def _prepare_linear(c, seed, gen):
    dt = DTYPES[c["dtype"]]
    n, k = c["n"], c["k"]
    kp = -(-k // 128) * 128
    w = _rand(gen, n, k) * (0.5 + torch.rand(n, 1, generator=gen, device="cuda")) / math.sqrt(k)
    # the last group is quantised over the columns that there are; the ones filled up are code 0, met by no input
    full = torch.cat([w, w[:, k - 1:].expand(n, kp - k)], 1) if kp > k else w
    if kp > k and k % c["group"] == 0:
        full[:, k:] = 0
    code, sc = _quantise(full, c["group"])
    last = -(-k // c["group"])
    sc[:, last:] = 0
    code[:, k:] = 0
    codes = torch.cat([_pack(code[:, b:b + 128], False) for b in range(0, kp, 128)], 1).contiguous()
    st = dict(case=c, codes=codes, scales=sc.contiguous(), x=_rand(gen, c["rows"], k).to(dt), bias=(0.1 * _rand(gen, n)).to(dt))
    st["residual"] = _rand(gen, c["rows"], n).to(dt) if c["residual"] else None
    return st


def _prepare_logprobs(c, seed, gen):
    rows, v = c["rows"], c["classes"]
    x = torch.empty(rows, v, dtype=DTYPES[c["dtype"]], device="cuda")
    step = max(1, 64_000_000 // v)
    labels = torch.randint(0, v, (rows, c["labels"]), generator=gen, device="cuda")
    for r in range(0, rows, step):  # by parts: the 32-bit scores of a long prompt are not held at once
        part = 2.5 * _rand(gen, min(step, rows - r), v)
        if c["masked"]:
            hide = torch.rand(part.shape, generator=gen, device="cuda") < c["masked"]
            hide.scatter_(1, labels[r:r + step], False)
            part.masked_fill_(hide, -math.inf)
        x[r:r + step] = part.to(x.dtype)
    return dict(case=c, logits=x, labels=labels.to(torch.int32))


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"store": _own_store, "attend": _own_attend, "linear": _own_linear, "logprobs": _own_logprobs}[op](state)
    return {"store": _plain_store, "attend": _plain_attend, "linear": _plain_linear, "logprobs": _plain_logprobs}[op](state)


def _plain_store(st):
    c, kv = st["case"], st["kv"]
    code, sc = _quantise(kv, c["group"])
    pool = st["pool"]
    kc, ks, vc, vs = _parts(pool, c)
    page, at = st["slots"] // c["page"], st["slots"] % c["page"]
    kc[page, :, at] = _pack(code[:, 0], False)
    vc[page, :, at] = _pack(code[:, 1], True)
    ks[page, :, at] = sc[:, 0]
    vs[page, :, at] = sc[:, 1]
    k = _values(kc[page, :, at], ks[page, :, at], c["group"], False)
    v = _values(vc[page, :, at], vs[page, :, at], c["group"], True)
    return k.to(kv.dtype), v.to(kv.dtype)


def _plain_attend(st):
    c, q = st["case"], st["q"]
    b, n, h, w, most = c["seqs"], c["rows"], c["heads"], c["width"], max(1, c["most"])
    kc, ks, vc, vs = _parts(st["pool"], c)
    pages = st["table"].clamp(min=0).long()
    tokens = lambda part: part[pages].transpose(1, 2).flatten(2, 3)[:, :, :most]  # noqa: E731  [seq, head, token, ...]
    k = _values(tokens(kc), tokens(ks), c["group"], False)
    s = torch.matmul(q.float().view(b, n, h, -1, w).permute(0, 2, 3, 1, 4).flatten(2, 3), k.transpose(-1, -2)) * st["scale"]
    del k
    s = s.unflatten(2, (-1, n))  # [seq, head, head of the group, row, token]
    lens = st["lens"].view(b, 1, 1).long()
    j = torch.arange(most, device=q.device).view(1, 1, -1)
    at = lens - n + torch.arange(n, device=q.device).view(1, -1, 1)
    seen = (j < lens).expand(b, n, most)
    if c["causal"]:
        seen = seen & (j <= at)
    if c["window"]:
        seen = seen & (j > at - c["window"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    # values past a sequence's end are not looked at, whatever they are
    v = _values(tokens(vc), tokens(vs), c["group"], True)
    v = torch.where((j < lens).view(b, 1, most, 1), v, torch.zeros_like(v))
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, n))
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log()).squeeze(-1)
    return o.permute(0, 3, 1, 2, 4).reshape(b * n, -1, w).to(q.dtype), lse.permute(0, 3, 1, 2).reshape(b * n, -1).contiguous()


def _plain_linear(st):
    c = st["case"]
    n, k = c["n"], c["k"]
    w = _values(st["codes"].view(n, -1, 64), st["scales"].view(n, -1, 128 // c["group"], 2), c["group"], False).flatten(1)[:, :k]
    y = torch.matmul(st["x"].float(), w.t()) + st["bias"].float()
    if c["act"]:
        y = 0.5 * y * (1.0 + torch.erf(y / math.sqrt(2.0)))
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(st["x"].dtype)


def _plain_logprobs(st):
    c, x = st["case"], st["logits"].float()
    top = x.amax(-1, keepdim=True)
    none = torch.isinf(top) & (top < 0)
    d = (x - torch.where(none, torch.zeros_like(top), top)) / c["temperature"]
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    log_total = torch.where(none, torch.zeros_like(total), total.log())
    picked = d.gather(1, st["labels"].long()) - log_total
    mean = (e * torch.where(e > 0, d, torch.zeros_like(d))).sum(-1, keepdim=True) / torch.where(none, torch.ones_like(total), total)
    entropy = (log_total - mean).squeeze(1)
    if not c["top"]:
        return picked, entropy
    del e
    # one whole number a score, in the scores' order and of two equal ones the lower index the larger
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    del bits
    key = (key << 32) | (0x7FFFFFFF - torch.arange(x.shape[1], device=x.device))
    best = key.topk(min(c["top"], x.shape[1]), dim=1).values
    del key
    ids = 0x7FFFFFFF - (best & 0x7FFFFFFF)
    value = d.gather(1, ids) - log_total
    ids = torch.where(torch.isneginf(x.gather(1, ids)), torch.full_like(ids, -1), ids)
    return picked, entropy, value, ids.to(torch.int32)


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


def _cache(st):
    if "cache" not in st:  # the handle a program keeps: sizes and the pool's address
        tcu, gpu = _framework()
        c, pool = st["case"], st["pool"]
        st["cache"] = tcu.Kv4Cache(gpu, pool.data_ptr(), pool.shape[0], heads=c["heads"], width=c["width"], page=c["page"],
                                   group=c["group"])
    return st["cache"]


def _own_store(st):
    c, kv, cache = st["case"], st["kv"], _cache(st)
    code, stream = CODES[c["dtype"]], _stream()
    w, row = c["width"], 2 * c["heads"] * c["width"]
    v_at = kv.data_ptr() + SIZE[c["dtype"]] * c["heads"] * w
    cache.store(code, c["tokens"], st["slots"].data_ptr(), kv.data_ptr(), row, w, v_at, row, w, stream=stream)
    k = torch.empty(c["tokens"], c["heads"], w, dtype=kv.dtype, device=kv.device)
    v = torch.empty_like(k)
    cache.load(code, c["tokens"], st["slots"].data_ptr(), k.data_ptr(), c["heads"] * w, w, v.data_ptr(), c["heads"] * w, w,
               stream=stream)
    return k, v


def _own_attend(st):
    c, q, cache = st["case"], st["q"], _cache(st)
    rows, hq, w = q.shape
    if "batch" not in st:  # the step's plan and workspace, kept as a program keeps them from layer to layer
        st["batch"] = cache.batch(c["seqs"], c["rows"], max(1, c["most"]), st["lens"].data_ptr(), st["table"].data_ptr(),
                                  st["table"].stride(0))
        need = cache.attend_workspace(st["batch"], hq, CODES[c["dtype"]])
        st["work"] = torch.zeros(max(1, need), dtype=torch.uint8, device=q.device)
    out = torch.empty_like(q)
    lse = torch.empty(rows, hq, dtype=torch.float32, device=q.device)
    cache.attend(st["batch"], CODES[c["dtype"]], hq, q.data_ptr(), hq * w, w, out.data_ptr(), hq * w, w, st["scale"],
                 causal=c["causal"], window=c["window"], lse=lse.data_ptr(), work=st["work"].data_ptr(),
                 work_bytes=st["work"].numel(), stream=_stream())
    return out, lse


def _own_linear(st):
    c, x = st["case"], st["x"]
    if "w4" not in st:
        tcu, gpu = _framework()
        st["w4"] = tcu.W4(gpu, c["n"], c["k"], c["group"], st["codes"].data_ptr(), st["scales"].data_ptr())
        need = st["w4"].linear_workspace(c["rows"], CODES[c["dtype"]])
        st["work"] = torch.zeros(max(1, need), dtype=torch.uint8, device=x.device)
    y = torch.empty(c["rows"], c["n"], dtype=x.dtype, device=x.device)
    r = st["residual"]
    st["w4"].linear(CODES[c["dtype"]], c["rows"], x.data_ptr(), c["k"], y.data_ptr(), c["n"], bias=st["bias"].data_ptr(),
                    act=c["act"], residual=r.data_ptr() if r is not None else None, ldr=c["n"], work=st["work"].data_ptr(),
                    work_bytes=st["work"].numel(), stream=_stream())
    return y


def _own_logprobs(st):
    c, x = st["case"], st["logits"]
    _, gpu = _framework()
    rows, v = x.shape
    top = min(c["top"], v)
    picked = torch.empty(rows, c["labels"], dtype=torch.float32, device=x.device)
    entropy = torch.empty(rows, dtype=torch.float32, device=x.device)
    value = torch.empty(rows, top, dtype=torch.float32, device=x.device)
    ids = torch.empty(rows, top, dtype=torch.int32, device=x.device)
    gpu.label_logprobs(CODES[c["dtype"]], x.data_ptr(), rows, v, v, st["labels"].data_ptr(), c["labels"], picked.data_ptr(),
                       entropy=entropy.data_ptr(), top=top, top_values=value.data_ptr(), top_ids=ids.data_ptr(),
                       temperature=c["temperature"], stream=_stream())
    return (picked, entropy, value, ids) if top else (picked, entropy)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def _pairs(c, length):
    """Query rows times the keys they see, for one sequence."""
    n = c["rows"]
    if not c["causal"]:
        return n * length, length
    total, first = 0, length
    for i in range(n):
        last = min(length - 1, length - n + i)
        low = max(0, length - n + i - c["window"] + 1) if c["window"] else 0
        if last >= low:
            total += last - low + 1
            first = min(first, low)
    return total, length - first


def work(case):
    c = case
    if c["op"] == "store":
        values = 2 * c["tokens"] * c["heads"] * c["width"]
        cached = values // 2 + 4 * values // c["group"]
        return {"bytes": 2 * values * SIZE[c["dtype"]] + 2 * cached + 16 * c["tokens"], "flops": 6 * values}
    if c["op"] == "attend":
        pairs = keys = 0
        for length in _lens(c, 0):
            a, b = _pairs(c, length)
            pairs, keys = pairs + a, keys + b
        rows = c["seqs"] * c["rows"] * c["q_heads"]
        token = c["heads"] * (c["width"] + 8 * (c["width"] // c["group"]))
        return {"bytes": keys * token + rows * (2 * c["width"] * SIZE[c["dtype"]] + 4), "flops": 4 * pairs * c["q_heads"] * c["width"]}
    if c["op"] == "linear":
        m, n, k, s = c["rows"], c["n"], c["k"], SIZE[c["dtype"]]
        return {"bytes": n * k // 2 + 4 * n * -(-k // c["group"]) + s * (m * k + n + m * n * (2 if c["residual"] else 1)),
                "flops": 2 * m * n * k}
    return {"bytes": c["rows"] * (c["classes"] * SIZE[c["dtype"]] + 8 * c["labels"] + 4 + 8 * min(c["top"], c["classes"])),
            "flops": 5 * c["rows"] * c["classes"]}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "linear": _exact_linear, "logprobs": _exact_logprobs}[case["op"]](st)


def _exact_codes(raw, values):
    """The codes of a token's bytes, each found by its place in the documented order."""
    width = 2 * raw.shape[-1]
    units = width // 32
    i = torch.arange(width, device=raw.device)
    u, r = i // 32, i % 32
    nibble = ((r // 4) * units + u) * 4 + r % 4 if values else ((r // 8) * units + u) * 8 + r % 8
    return (raw[..., nibble // 2] >> (4 * (nibble % 2))) & 15


def _exact_values(raw, scales, group, values):
    c = _exact_codes(raw, values).double()
    which = torch.arange(c.shape[-1], device=raw.device) // group
    return scales[..., 1].double()[..., which] + scales[..., 0].double()[..., which] * c


def _exact_store(st):
    c = st["case"]
    outs = []
    for part in range(2):
        x = st["kv"][:, part].double()
        t, h, w = x.shape
        found = torch.empty_like(x)
        for b in range(0, w, c["group"]):
            g = x[..., b:b + c["group"]]
            low = g.min(-1, keepdim=True).values.half().double()
            step = ((g.max(-1, keepdim=True).values - low).clamp(min=0) / 15).half().double()
            code = torch.nan_to_num((g - low) / step, nan=0.0, posinf=0.0, neginf=0.0).round().clamp(0, 15)
            found[..., b:b + c["group"]] = low + step * code
        outs.append(found)
    return tuple(outs)


def _exact_attend(st):
    c, q = st["case"], st["q"]
    n, h, w = c["rows"], c["heads"], c["width"]
    each = c["q_heads"] // h
    kc, ks, vc, vs = _parts(st["pool"], c)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for s, length in enumerate(st["lens"].tolist()):
        if not length:
            continue
        pages = st["table"][s, :-(-length // c["page"])].long()
        i = torch.arange(n, device=q.device)[:, None] + length - n
        j = torch.arange(length, device=q.device)[None]
        hidden = torch.zeros(n, length, dtype=torch.bool, device=q.device)
        if c["causal"]:
            hidden |= j > i
        if c["window"]:
            hidden |= j <= i - c["window"]
        rows = slice(s * n, (s + 1) * n)
        for head in range(h):
            k = _exact_values(kc[pages, head].flatten(0, 1)[:length], ks[pages, head].flatten(0, 1)[:length], c["group"], False)
            v = _exact_values(vc[pages, head].flatten(0, 1)[:length], vs[pages, head].flatten(0, 1)[:length], c["group"], True)
            for hq in range(head * each, (head + 1) * each):
                a = (q[rows, hq].double() @ k.t()) * st["scale"]
                a[hidden] = -math.inf
                total = torch.logsumexp(a, -1)
                some = total > -math.inf
                lse[rows, hq] = total
                o = torch.exp(a - torch.where(some, total, torch.zeros_like(total))[:, None]) @ v
                out[rows, hq] = torch.where(some[:, None], o, torch.zeros_like(o))
    return out, lse


def _exact_linear(st):
    c = st["case"]
    blocks = [_exact_values(st["codes"][:, 64 * b:64 * b + 64], st["scales"][:, b * (128 // c["group"]):(b + 1) * (128 // c["group"])],
                            c["group"], False) for b in range(st["codes"].shape[1] // 64)]
    y = st["x"].double() @ torch.cat(blocks, 1)[:, :c["k"]].t() + st["bias"].double()
    if c["act"]:
        y = torch.nn.functional.gelu(y)
    return y + st["residual"].double() if c["residual"] else y


def _exact_logprobs(st):
    c = st["case"]
    step = max(1, 100_000_000 // c["classes"])
    rows, outs = c["rows"], ([], [], [])
    for r in range(0, rows, step):
        x = st["logits"][r:r + step].double() / c["temperature"]
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        outs[0].append(lp.gather(1, st["labels"][r:r + step].long()))
        outs[1].append(-(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1))
        if c["top"]:
            outs[2].append(lp.topk(min(c["top"], c["classes"]), dim=1).values)
    found = [torch.cat(o) for o in outs if o]
    return tuple(found) + (None,) if c["top"] else tuple(found)
