"""The four-bit operators and the label log-probabilities on the GPU against plain numpy in 64 bits."""
import numpy as np
import pytest

import fourbit_plain as plain
from conftest import tcu

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
# half a unit in the last place of a result of each type, relative
ULP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


@pytest.fixture(scope="module")
def gpu():
    return tcu.Gpu(0)


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.float().cpu().numpy()


def rounded(a, dtype):
    """The numbers of a as the type holds them (f32 array)."""
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dtype).float().numpy()


def sync(gpu):
    torch.cuda.synchronize()
    gpu.sync()


# ---- the cache ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width,group,page,heads", [(32, 32, 16, 3), (64, 32, 32, 1), (64, 64, 64, 5), (128, 32, 64, 2),
                                                    (128, 64, 256, 4), (128, 128, 16, 7), (256, 32, 128, 1), (256, 128, 16, 2)])
def test_store_and_load(gpu, dtype, width, group, page, heads):
    code, tt = DT[dtype]
    rng = np.random.default_rng(width + group + page)
    tokens, pages = 37, 5 + 37 // page
    k, v = rng.normal(1, 3, (2, tokens, heads, width))
    k[1, 0, :group] = 0.25          # a constant group: step 0
    k[2] = 0
    v[3, :, ::3] *= 1e4             # a wide span
    k[4, 0, 5], v[5, heads - 1, width - 1] = np.nan, -np.inf
    k[6, 0] = 6e4
    v[7] *= 1e-6                    # steps among f16's smallest
    k, v = rounded(k, tt), rounded(v, tt)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots[8] = -1
    want, kk, vv = plain.pool_of(k, v, slots, pages, page, group, 0xA5)
    pool = torch.full(want.shape, 0xA5, dtype=torch.uint8, device="cuda")
    cache = tcu.Kv4Cache(gpu, pool.data_ptr(), pages, heads=heads, width=width, page=page, group=group)
    # one row a token, keys beside values, as a projection leaves them
    kv = torch.stack([dev(k, tt), dev(v, tt)], 1)
    row, at = 2 * heads * width, kv.element_size() * heads * width
    sl = dev(slots)
    cache.store(code, tokens, sl.data_ptr(), kv.data_ptr(), row, width, kv.data_ptr() + at, row, width, stream=1)
    gk, gv = torch.full_like(kv[:, 0], 7.0), torch.full_like(kv[:, 0], 7.0)
    cache.load(code, tokens, sl.data_ptr(), gk.data_ptr(), heads * width, width, gv.data_ptr(), heads * width, width, stream=1)
    sync(gpu)
    assert np.array_equal(pool.cpu().numpy(), want)  # the codes, the scales, and nothing beside the slots
    for got, full in ((gk, kk), (gv, vv)):
        full = np.where((slots < 0)[:, None, None], 0.0, full)
        # the value is low + step * code with one rounding to 32 bits, then to the type
        assert np.array_equal(host(got), rounded(full.astype(np.float32), tt), equal_nan=True)


def test_store_takes_unaligned_rows_and_strides(gpu):
    rng = np.random.default_rng(3)
    tokens, heads, width, page, group = 9, 2, 64, 16, 32
    k, v = rounded(rng.normal(0, 2, (2, tokens, heads, width)), torch.bfloat16)
    want, _, _ = plain.pool_of(k, v, np.arange(tokens) + 5, 2, page, group, 0)
    pool = torch.zeros(want.shape, dtype=torch.uint8, device="cuda")
    cache = tcu.Kv4Cache(gpu, pool.data_ptr(), 2, heads=heads, width=width, page=page, group=group)
    buf = torch.zeros(2, tokens * 200 + 8, dtype=torch.bfloat16, device="cuda")
    for i, x in enumerate((k, v)):
        torch.as_strided(buf, (tokens, heads, width), (200, 71, 1), i * buf.shape[1] + 3).copy_(dev(x))
    sl = dev(np.arange(tokens, dtype=np.int64) + 5)
    cache.store(2, tokens, sl.data_ptr(), buf.data_ptr() + 6, 200, 71, buf[1].data_ptr() + 6, 200, 71, stream=1)
    sync(gpu)
    assert np.array_equal(pool.cpu().numpy(), want)


def test_a_slot_outside_the_cache_is_reported_and_not_written(gpu):
    pool = torch.zeros(2 * tcu.Kv4Cache.page_bytes(1, 32, 16, 32), dtype=torch.uint8, device="cuda")
    cache = tcu.Kv4Cache(gpu, pool.data_ptr(), 2, heads=1, width=32, page=16, group=32)
    x = torch.ones(1, 32, device="cuda")
    sl = dev(np.array([32], np.int64))
    cache.store(0, 1, sl.data_ptr(), x.data_ptr(), 32, 32, x.data_ptr(), 32, 32, stream=1)
    torch.cuda.synchronize()
    with pytest.raises(tcu.TcuError, match="outside its range"):
        gpu.sync()
    gpu.sync()  # reported once
    assert int(pool.sum()) == 0


# ---- attention over it ----------------------------------------------------------------------------------------------

class Cached:
    """Sequences of random tokens in a shuffled pool; every byte that holds no token is 0xFF (NaN scales)."""

    def __init__(self, gpu, seed, lens, heads, width, page, group, extra=2, spread=2.0):
        rng = np.random.default_rng(seed)
        self.gpu, self.lens, self.heads, self.width = gpu, lens, heads, width
        used = [-(-n // page) for n in lens]
        self.pages = sum(used) + extra
        order = rng.permutation(self.pages)
        self.stride = max(used + [1]) + 1
        table = np.full((len(lens), self.stride), -1, np.int32)
        slots, at = [], 0
        for s, n in enumerate(used):
            table[s, :n] = order[at:at + n]
            at += n
            slots += [int(table[s, j // page]) * page + j % page for j in range(lens[s])]
        k = rng.normal(0.3, spread, (sum(lens), heads, width))
        v = rng.normal(0, 1, (sum(lens), heads, width)) + np.arange(width) % 3
        raw, kk, vv = plain.pool_of(k.astype(np.float32), v.astype(np.float32), slots, self.pages, page, group, 0xFF)
        cut = np.cumsum([0] + list(lens))
        self.k = [kk[cut[s]:cut[s + 1]] for s in range(len(lens))]
        self.v = [vv[cut[s]:cut[s + 1]] for s in range(len(lens))]
        self.pool, self.table = dev(raw), dev(table)
        self.lens_dev = dev(np.array(lens, np.int32))
        self.cache = tcu.Kv4Cache(gpu, self.pool.data_ptr(), self.pages, heads=heads, width=width, page=page, group=group)

    def attend(self, dtype, q, counts, scale, causal=False, window=0, ragged=False, out=None, work=None, stream=1):
        code, tt = DT[dtype]
        rows, hq, w = q.shape
        most = max(counts)
        starts = dev(np.cumsum([0] + list(counts)).astype(np.int32)) if ragged else None
        self.batch = self.cache.batch(len(self.lens), most, max(self.lens + [1]), self.lens_dev.data_ptr(), self.table.data_ptr(),
                                      self.stride, starts.data_ptr() if ragged else None, rows)
        if work is None:
            work = torch.zeros(max(16, self.cache.attend_workspace(self.batch, hq, code)), dtype=torch.uint8, device="cuda")
        qd = dev(q, tt)
        out = torch.full_like(qd, 9.0) if out is None else out
        lse = torch.full((rows, hq), 9.0, device="cuda")
        self.keep = (starts, qd, work)
        self.cache.attend(self.batch, code, hq, qd.data_ptr(), hq * w, w, out.data_ptr(), hq * w, w, scale, causal=causal,
                          window=window, lse=lse.data_ptr(), work=work.data_ptr(), work_bytes=work.numel(), stream=stream)
        return out, lse

    def check(self, dtype, q, counts, scale, causal, window, out, lse):
        at = 0
        out, lse = host(out), host(lse)
        for s, n in enumerate(counts):
            o, l, reach = plain.attend(q[at:at + n], self.k[s], self.v[s], n, self.lens[s], scale, causal, window)
            got, gl = out[at:at + n], lse[at:at + n]
            none = ~np.isfinite(l)
            assert np.array_equal(gl[none], l[none]) and not got[none].any()
            # What the kernels round: for the 16-bit types keys, values and weights to 11 bits, for f32 to 21 or more;
            # q and the sums to 21 or more. A score is off by at most that share of its sum of magnitudes (`reach`), a
            # weight by e to the power of twice that, and again by its own rounding; values by theirs.
            u = 2.0**-11 if dtype != "f32" else 2.0**-20
            vmax = np.abs(self.v[s]).max() if self.lens[s] else 0.0
            score = (u + 2.0**-20) * reach
            tol = vmax * (np.expm1(2 * score) + 3 * u)[..., None] + 2 * ULP[dtype] * np.abs(o) + 1e-7
            some = ~none
            assert (np.abs(got - o)[some] <= tol[some]).all(), (s, np.abs(got - o)[some].max(), tol[some].min())
            assert (np.abs(gl - l)[some] <= (score + 2.0**-20 * (1 + np.abs(np.where(some, l, 0))))[some]).all()
            at += n


ATTEND = [
    # dtype, width, group, page, heads, q_heads, counts, lens, causal, window
    ("f32", 128, 64, 256, 4, 4, [1], [1], False, 0),
    ("f32", 128, 64, 256, 4, 4, [1], [777], False, 0),
    ("bf16", 128, 32, 64, 2, 8, [1] * 7, [0, 1, 63, 64, 65, 500, 129], True, 0),
    ("f16", 64, 64, 16, 3, 3, [1] * 5, [17, 0, 1, 900, 33], True, 0),
    ("bf16", 128, 128, 16, 1, 8, [1, 1], [2000, 15], True, 100),
    ("f16", 256, 32, 128, 2, 2, [1, 1], [300, 129], False, 0),
    ("f32", 256, 128, 32, 1, 4, [3, 3], [70, 2], True, 0),
    ("bf16", 32, 32, 32, 5, 5, [4], [200], True, 7),
    ("f32", 32, 32, 16, 1, 1, [2, 2, 2], [1, 2, 333], True, 0),
    ("bf16", 64, 32, 64, 1, 9, [5, 5], [300, 4], True, 0),
    ("f16", 128, 64, 64, 2, 32, [2], [511], True, 0),
    ("f32", 64, 32, 256, 2, 6, [7, 7], [400, 257], False, 0),
    # many rows
    ("f32", 128, 64, 256, 2, 2, [130], [700], False, 0),
    ("bf16", 128, 128, 64, 1, 4, [70], [70], True, 0),
    ("bf16", 128, 32, 16, 2, 4, [100, 100], [333, 90], True, 0),
    ("f16", 64, 64, 32, 1, 3, [129], [512], True, 50),
    ("f32", 256, 64, 64, 1, 1, [150], [200], True, 0),
    ("f16", 256, 128, 128, 1, 2, [80], [300], False, 0),
    ("bf16", 32, 32, 64, 2, 2, [257], [301], True, 0),
    ("f32", 32, 32, 16, 1, 2, [200], [129], False, 0),
    ("f32", 64, 32, 16, 1, 1, [300], [1], True, 0),
]


@pytest.mark.parametrize("dtype,width,group,page,heads,q_heads,counts,lens,causal,window", ATTEND)
def test_attend(gpu, dtype, width, group, page, heads, q_heads, counts, lens, causal, window):
    c = Cached(gpu, width + len(lens), lens, heads, width, page, group)
    q = rounded(np.random.default_rng(1).normal(0, 1, (sum(counts), q_heads, width)), DT[dtype][1])
    scale = 1 / np.sqrt(width)
    out, lse = c.attend(dtype, q, counts, scale, causal, window)
    sync(gpu)
    c.check(dtype, q, counts, scale, causal, window, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1, 0, 3, 2], [40, 1, 0, 90], [0, 0, 0, 1]])
def test_attend_ragged_rows(gpu, dtype, counts):
    c = Cached(gpu, 11, [120, 60, 0, 200], 2, 64, 32, 32)
    q = rounded(np.random.default_rng(2).normal(0, 1, (sum(counts), 6, 64)), DT[dtype][1])
    out, lse = c.attend(dtype, q, counts, 0.125, causal=True, ragged=True)
    sync(gpu)
    c.check(dtype, q, counts, 0.125, True, 0, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("counts", [[1, 1], [150, 150]])
def test_attend_sharp_and_flat_scores(gpu, dtype, counts):
    """Scores over a span of hundreds (one key takes all) and all equal (every key the same share)."""
    for size in (6.0, 0.0):
        c = Cached(gpu, 5, [333, 1], 1, 128, 64, 32, spread=3.0)
        q = rounded(np.random.default_rng(2).normal(0, size, (sum(counts), 2, 128)), DT[dtype][1])
        out, lse = c.attend(dtype, q, counts, 0.0884)
        sync(gpu)
        c.check(dtype, q, counts, 0.0884, False, 0, out, lse)


@pytest.mark.parametrize("rows", [1, 140])
def test_attend_scales_of_very_different_size(gpu, rows):
    """Values from 1e-4 to 6e4 in one cache, keys as different: steps across f16's range."""
    c = Cached(gpu, 8, [400], 1, 64, 16, 32)
    rng = np.random.default_rng(4)
    k = rng.normal(0, 1, (400, 1, 64)) * 10.0 ** rng.uniform(-3, 0, (400, 1, 1))
    v = rng.normal(0, 1, (400, 1, 64)) * 10.0 ** rng.uniform(-4, 4, (400, 1, 1))
    slots = [int(c.table[0, j // 16]) * 16 + j % 16 for j in range(400)]
    raw, kk, vv = plain.pool_of(k.astype(np.float32), v.astype(np.float32), slots, c.pages, 16, 32, 0xFF)
    c.pool.copy_(dev(raw))
    c.k, c.v = [kk], [vv]
    q = rng.normal(0, 1, (rows, 1, 64)).astype(np.float32)
    out, lse = c.attend("f32", q, [rows], 0.125)
    sync(gpu)
    c.check("f32", q, [rows], 0.125, False, 0, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,group", [(1, 128, 64), (3, 128, 32), (2, 64, 32), (1, 256, 128), (200, 128, 64)])
def test_attend_values_that_cancel(gpu, dtype, rows, width, group):
    """Flat scores over thousands of keys whose values have no mean: outputs far below the values and their lows."""
    n = 6000
    c = Cached(gpu, 14, [16], 1, width, 256, group, extra=n // 256 + 1)
    rng = np.random.default_rng(7)
    k, v = rng.normal(0, 1, (2, n, 1, width))
    order = rng.permutation(c.pages)[:-(-n // 256)]
    raw, kk, vv = plain.pool_of(k.astype(np.float32), v.astype(np.float32), order[np.arange(n) // 256] * 256 + np.arange(n) % 256,
                                c.pages, 256, group, 0xFF)
    c.pool.copy_(dev(raw))
    c.table, c.stride, c.lens = dev(order.astype(np.int32)[None]), len(order), [n]
    c.lens_dev.fill_(n)
    q = rounded(rng.normal(0, 1, (rows, 2, width)), DT[dtype][1])
    out, lse = c.attend(dtype, q, [rows], 0.5 / np.sqrt(width))
    sync(gpu)
    o, l, _ = plain.attend(q, kk, vv, rows, n, 0.5 / np.sqrt(width), False, 0)
    # weights are off by 2^-20 for f32 and 2^-11 (keys, or twice 2^-12) else, each by itself, so a sum of values without a
    # mean by no more than that share of itself; an f32 sum by 2^-23 of its size a step, some ten steps' worth; the result
    # by its own rounding
    off = np.linalg.norm(host(out) - o) / np.linalg.norm(o)
    assert off <= {"f32": 1e-5, "f16": 2.0**-11, "bf16": 2.0**-8}[dtype], off
    assert np.abs(host(lse) - l).max() <= {"f32": 1e-5, "f16": 2.0**-9, "bf16": 2.0**-9}[dtype]


@pytest.mark.parametrize("dtype,rows", [("f32", 1), ("bf16", 1), ("f32", 200), ("bf16", 200)])
def test_attend_strides_and_repeat(gpu, dtype, rows):
    """Query and output rows inside wider buffers at odd places; the same call again gives the same bits."""
    code, tt = DT[dtype]
    c = Cached(gpu, 6, [700], 2, 64, 32, 32)
    q = rounded(np.random.default_rng(3).normal(0, 1, (rows, 4, 64)), tt)
    wide = torch.zeros(rows, 4, 67, dtype=tt, device="cuda")
    wide[..., 1:65] = dev(q, tt)
    outs = []
    batch = c.cache.batch(1, rows, 700, c.lens_dev.data_ptr(), c.table.data_ptr(), c.stride)
    work = torch.zeros(max(16, c.cache.attend_workspace(batch, 4, code)), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        o = torch.full((rows, 4, 73), 9.0, dtype=tt, device="cuda")
        es = o.element_size()
        c.cache.attend(batch, code, 4, wide.data_ptr() + es, 4 * 67, 67, o.data_ptr() + 3 * es, 4 * 73, 73, 0.125,
                       work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        sync(gpu)
        outs.append(o)
    assert torch.equal(outs[0], outs[1])
    assert bool((outs[0][..., :3] == 9).all()) and bool((outs[0][..., 67:] == 9).all())
    _, lse = c.attend(dtype, q, [rows], 0.125)
    sync(gpu)
    c.check(dtype, q, [rows], 0.125, False, 0, outs[0][..., 3:67], lse)


def test_attend_on_another_stream(gpu):
    c = Cached(gpu, 9, [600, 40], 1, 128, 64, 64)
    q = rounded(np.random.default_rng(3).normal(0, 1, (2, 4, 128)), torch.bfloat16)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        out, lse = c.attend("bf16", q, [1, 1], 0.1, stream=s.cuda_stream)
    s.synchronize()
    gpu.sync()
    c.check("bf16", q, [1, 1], 0.1, False, 0, out, lse)


def test_attend_a_pool_past_four_gigabytes(gpu):
    """Pages whose byte offsets pass 32 bits."""
    heads, width, page, group = 8, 128, 64, 32
    size = tcu.Kv4Cache.page_bytes(heads, width, page, group)
    pages = (9 << 30) // 2 // size + 4
    c = Cached(gpu, 10, [150], heads, width, page, group, extra=0)
    pool = torch.empty(pages, size, dtype=torch.uint8, device="cuda")
    pool[-3:] = c.pool
    c.table[0, :3] += pages - 3
    c.cache = tcu.Kv4Cache(gpu, pool.data_ptr(), pages, heads=heads, width=width, page=page, group=group)
    for rows in (1, 140):
        q = rounded(np.random.default_rng(3).normal(0, 1, (rows, 8, width)), torch.bfloat16)
        out, lse = c.attend("bf16", q, [rows], 0.09)
        sync(gpu)
        c.check("bf16", q, [rows], 0.09, False, 0, out, lse)


@pytest.mark.parametrize("rows", [1, 140])
def test_attend_reports_indexes_outside_their_range(gpu, rows):
    def call(change):
        c = Cached(gpu, 12, [100, 70], 1, 64, 32, 32)
        change(c)
        q = np.ones((2 * rows, 2, 64), np.float32)
        c.lens = [100, 70]
        c.attend("f32", q, [rows, rows], 0.1)
        torch.cuda.synchronize()
        with pytest.raises(tcu.TcuError, match="outside its range"):
            gpu.sync()
        gpu.sync()

    call(lambda c: c.table[0, 1].fill_(c.pages))
    call(lambda c: c.table[1, 0].fill_(-5))
    call(lambda c: c.lens_dev[0].fill_(101))
    call(lambda c: c.lens_dev[1].fill_(-1))


def test_attend_refusals(gpu):
    c = Cached(gpu, 13, [10], 2, 64, 32, 32)
    q = np.zeros((1, 4, 64), np.float32)
    c.attend("f32", q, [1], 0.1)
    sync(gpu)
    b, t = c.batch, torch.zeros(4, 64, device="cuda")
    w = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")

    def refused(match, dtype=0, q_heads=4, scale=0.1, batch=b, cache=c.cache, q_ptr=t.data_ptr(), **kw):
        with pytest.raises(tcu.TcuError, match=match):
            cache.attend(batch, dtype, q_heads, q_ptr, 256, 64, t.data_ptr(), 256, 64, scale, work=w.data_ptr(),
                         work_bytes=w.numel(), stream=1, **kw)

    refused("dtype", dtype=3)
    refused("multiple", q_heads=3)
    refused("finite", scale=float("nan"))
    refused("window", window=4)
    refused("window", window=-1, causal=True)
    refused("null", q_ptr=None)
    refused("aligned", q_ptr=t.data_ptr() + 2)
    args = (c.lens_dev.data_ptr(), c.table.data_ptr())
    refused("max_rows rows", batch=c.cache.batch(1, 1, 10, *args, c.stride, None, 2))
    refused("do not hold", batch=c.cache.batch(1, 1, 1000, *args, c.stride))
    refused("not negative", batch=c.cache.batch(1, 1, -1, *args, c.stride))
    mk = lambda **o: tcu.Kv4Cache(gpu, **{**dict(pool_ptr=c.pool.data_ptr(), pages=c.pages, heads=2, width=64, page=32, group=32), **o})  # noqa: E731
    refused("width", cache=mk(width=48))
    refused("group", cache=mk(group=128))
    refused("no pool", cache=mk(pool_ptr=None))
    refused("aligned", cache=mk(pool_ptr=c.pool.data_ptr() + 8))
    with pytest.raises(tcu.TcuError, match="strides"):
        c.cache.store(0, 1, w.data_ptr(), t.data_ptr(), -1, 64, t.data_ptr(), 0, 64)
    with pytest.raises(tcu.TcuError, match="tokens"):
        c.cache.store(0, -1, w.data_ptr(), t.data_ptr(), 1, 64, t.data_ptr(), 0, 64)
    c.cache.store(0, 0, None, None, 0, 0, None, 0, 0)  # no tokens: nothing to do


# ---- linear layers --------------------------------------------------------------------------------------------------

def weights(rng, gpu, n, k, group, dtype):
    """Packed on the device, checked bit for bit; returns the handle, its buffers and the values in 64 bits."""
    code, tt = DT[dtype]
    w = rounded(rng.normal(0, 1, (n, k)) * rng.uniform(0.1, 2, (n, 1)) + 0.05, tt)
    kp = -(-k // 128) * 128
    full = np.zeros((n, kp), np.float32)
    full[:, :k] = w
    last = -(-k // group) * group
    full[:, k:last] = w[:, k - 1:k]  # the columns that fill the last group up take no part in it
    cs, step, low = plain.quantise(full, group)
    cs[:, k:] = 0
    step[:, last // group:], low[:, last // group:] = 0, 0
    want = np.concatenate([plain.pack(cs[:, b:b + 128], False) for b in range(0, kp, 128)], 1)
    codes = torch.full((tcu.W4.code_bytes(n, k),), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((tcu.W4.scale_bytes(n, k, group),), 0xA5, dtype=torch.uint8, device="cuda")
    w4 = tcu.W4(gpu, n, k, group, codes.data_ptr(), scales.data_ptr())
    wide = torch.full((n, k + 3), float("nan"), dtype=tt, device="cuda")  # columns past k are not read
    wide[:, :k] = dev(w, tt)
    w4.pack(code, wide.data_ptr(), k + 3, stream=1)
    sync(gpu)
    assert np.array_equal(codes.cpu().numpy().reshape(n, -1), want)
    assert np.array_equal(scales.cpu().numpy().view(np.float16).reshape(n, -1, 2), plain.scales(step, low))
    return w4, (codes, scales), plain.value(cs, step, low, group)[:, :k]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,group,rows,act,bias,residual", [
    (1, 1, 32, 1, 0, False, False), (16, 128, 128, 1, 0, True, False), (1024, 512, 64, 1, 1, True, False),
    (512, 1024, 64, 1, 0, True, True), (17, 130, 32, 3, 1, False, True), (300, 1000, 128, 8, 0, True, True),
    (33, 4097, 64, 9, 0, False, False), (2500, 260, 32, 16, 1, True, True), (100, 777, 128, 17, 0, True, False),
    (130, 640, 64, 33, 0, True, True), (65, 9000, 32, 64, 0, True, False), (200, 300, 128, 131, 1, True, True)])
def test_linear(gpu, dtype, n, k, group, rows, act, bias, residual):
    code, tt = DT[dtype]
    rng = np.random.default_rng(n + k)
    w4, keep, w = weights(rng, gpu, n, k, group, dtype)
    x = rounded(rng.normal(0, 1, (rows, k)) * 10.0 ** rng.uniform(-2, 1, (rows, 1)), tt)
    b = rounded(rng.normal(0, 1, n), tt) if bias else None
    r = rounded(rng.normal(0, 1, (rows, n)), tt) if residual else None
    xd = torch.full((rows, k + 5), float("nan"), dtype=tt, device="cuda")
    xd[:, :k] = dev(x, tt)
    yd = torch.full((rows, n + 3), 9.0, dtype=tt, device="cuda")
    if residual:
        yd[:, :n] = dev(r, tt)  # in place: the residual is the output's own buffer
    bd = dev(b, tt) if bias else None
    work = torch.zeros(max(16, w4.linear_workspace(rows, code)), dtype=torch.uint8, device="cuda")
    w4.linear(code, rows, xd.data_ptr(), k + 5, yd.data_ptr(), n + 3, bias=bd.data_ptr() if bias else None, act=act,
              residual=yd.data_ptr() if residual else None, ldr=n + 3, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    y = x.astype(np.float64) @ w.T
    size = np.abs(x.astype(np.float64)) @ np.abs(w).T  # an error of 2^-20 in every product, and the sum's own
    if bias:
        y, size = y + b, size + np.abs(b)
    if act:
        erf = torch.erf(torch.from_numpy(y / np.sqrt(2))).numpy()
        y, size = 0.5 * y * (1 + erf), 1.13 * size + 2 * np.abs(y)  # the slope of GELU is below 1.13; its erf is good to 2^-21
    if residual:
        y, size = y + r, size + np.abs(r)
    got = host(yd)
    assert (np.abs(got[:, :n] - y) <= 2.0**-20 * size + 2 * ULP[dtype] * np.abs(y) + 1e-7).all()
    assert (got[:, n:] == 9).all()


@pytest.mark.parametrize("rows", [1, 5, 20, 70])
@pytest.mark.parametrize("k,group", [(512, 64), (4000, 32), (3000, 128)])
def test_linear_keeps_32_bits(gpu, rows, k, group):
    """f32 sums of products of either sign: a group's sum is rounded some ten times by at most 2^-23 of its size."""
    rng = np.random.default_rng(k + rows)
    w4, keep, w = weights(rng, gpu, 64, k, group, "f32")
    x = rng.normal(0, 1, (rows, k)).astype(np.float32)
    xd, yd = dev(x), torch.zeros(rows, 64, device="cuda")
    work = torch.zeros(max(16, w4.linear_workspace(rows, 0)), dtype=torch.uint8, device="cuda")
    w4.linear(0, rows, xd.data_ptr(), k, yd.data_ptr(), 64, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    y = x.astype(np.float64) @ w.T
    off = np.linalg.norm(host(yd) - y) / np.linalg.norm(y)
    assert off <= 1e-6, off


def test_linear_keeps_rows_apart(gpu):
    """A NaN, an infinity and a zero row in the input change their own outputs only."""
    w4, keep, w = weights(np.random.default_rng(0), gpu, 40, 256, 64, "f32")
    for rows in (5, 30):
        x = np.random.default_rng(1).normal(0, 1, (rows, 256)).astype(np.float32)
        x[1, 3], x[2, 200], x[3] = np.nan, np.inf, 0
        xd, yd = dev(x), torch.zeros(rows, 40, device="cuda")
        work = torch.zeros(max(16, w4.linear_workspace(rows, 0)), dtype=torch.uint8, device="cuda")
        w4.linear(0, rows, xd.data_ptr(), 256, yd.data_ptr(), 40, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        sync(gpu)
        got = host(yd)
        assert np.isnan(got[1]).all() and not np.isfinite(got[2]).any() and not got[3].any()
        fine = [i for i in range(rows) if i not in (1, 2)]
        size = np.abs(x[fine].astype(np.float64)) @ np.abs(w).T
        assert (np.abs(got[fine] - x[fine].astype(np.float64) @ w.T) <= 2.0**-20 * size + 1e-7).all()


def test_linear_refusals(gpu):
    w4, keep, _ = weights(np.random.default_rng(0), gpu, 8, 128, 32, "f32")
    t = torch.zeros(8, 128, device="cuda")
    p = t.data_ptr()
    for match, a, kw in [("dtype", (5, 1, p, 128, p, 8), {}), ("rows", (0, -1, p, 128, p, 8), {}), ("null", (0, 1, None, 128, p, 8), {}),
                         ("stride", (0, 1, p, 127, p, 8), {}), ("stride", (0, 1, p, 128, p, 7), {}), ("act", (0, 1, p, 128, p, 8), dict(act=2)),
                         ("stride", (0, 1, p, 128, p, 8), dict(residual=p, ldr=3)), ("aligned", (0, 1, p + 1, 128, p, 8), {})]:
        with pytest.raises(tcu.TcuError, match=match):
            w4.linear(*a, stream=1, **kw)
    w4.linear(0, 0, None, 128, None, 8)
    with pytest.raises(tcu.TcuError, match="group"):
        tcu.W4(gpu, 8, 128, 16, keep[0].data_ptr(), keep[1].data_ptr()).pack(0, p, 128)
    with pytest.raises(tcu.TcuError, match="aligned"):
        tcu.W4(gpu, 8, 128, 32, keep[0].data_ptr() + 4, keep[1].data_ptr()).linear(0, 1, p, 128, p, 8)


# ---- log probabilities ----------------------------------------------------------------------------------------------

def logprobs(gpu, dtype, x, labels, top, temperature, lead=0, tail=0):
    code, tt = DT[dtype]
    rows, classes = x.shape
    stride = lead + classes + tail
    buf = torch.full((rows, stride), 1e4, dtype=tt, device="cuda")
    buf[:, lead:lead + classes] = dev(x, tt)
    per = labels.shape[1]
    lab = dev(labels.astype(np.int32))
    out, ent = torch.full((rows, per), 9.0, device="cuda"), torch.full((rows,), 9.0, device="cuda")
    tv, ti = torch.full((rows, top), 9.0, device="cuda"), torch.full((rows, top), 9, dtype=torch.int32, device="cuda")
    gpu.label_logprobs(code, buf.data_ptr() + lead * buf.element_size(), rows, classes, stride, lab.data_ptr(), per, out.data_ptr(),
                       entropy=ent.data_ptr(), top=top, top_values=tv.data_ptr(), top_ids=ti.data_ptr(), temperature=temperature,
                       stream=1)
    torch.cuda.synchronize()
    return host(out), host(ent), host(tv), ti.cpu().numpy()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,classes,per,top,t,lead,tail", [
    (1, 1, 1, 1, 1.0, 0, 0), (3, 2, 2, 5, 0.5, 0, 0), (200, 10, 1, 3, 0.9, 0, 0), (7, 10, 4, 0, 0.9, 1, 2), (5, 33, 1, 32, 1.0, 3, 0),
    (9, 999, 3, 7, 1.7, 0, 1), (2, 4097, 1, 20, 1.0, 1, 0), (1, 32003, 1, 32, 0.7, 0, 0), (3, 131071, 2, 5, 1.0, 5, 3),
    (300, 1025, 0, 1, 1.0, 0, 0)])
def test_logprobs(gpu, dtype, rows, classes, per, top, t, lead, tail):
    rng = np.random.default_rng(rows + classes)
    x = rng.normal(0, 3, (rows, classes))
    x[rng.random(x.shape) < 0.1] = -np.inf
    if rows > 2:
        x[1] = -np.inf                                    # nothing left
        x[2] = np.round(x[2])                             # equal scores
    if rows > 4:
        x[3] = np.where(rng.random(classes) < 0.5, np.finfo(np.float16).min, x[3])
        x[4] = 0.0
        x[4, ::2] = -0.0
    labels = rng.integers(0, classes, (rows, per))
    if per > 1:
        labels[:, 1] = -1
    x = rounded(x, DT[dtype][1])
    out, ent, tv, ti = logprobs(gpu, dtype, x, labels, top, t, lead, tail)
    gpu.sync()
    for r in range(rows):
        o, e, v, i = plain.logprobs(x[r], labels[r], top, t)
        assert np.array_equal(ti[r], i), r
        # the distance of a score from the largest and its quotient by the temperature each round once, the logarithm and
        # the sums (in 32 bits, each e^d good to 2^-21) carry a few units of 2^-24 more
        for got, want in ((out[r], o), (tv[r], v), (ent[r:r + 1], np.array([e]))):
            fin = np.isfinite(want)
            assert np.array_equal(got[~fin], want[~fin])
            assert (np.abs(got - np.where(fin, want, 0))[fin] <= (2.0**-20 * (1 + np.abs(want)))[fin]).all(), r


def test_logprobs_of_nan_infinity_and_the_lowest_value(gpu):
    low = np.finfo(np.float32).min
    x = np.zeros((5, 700), np.float32)
    x[0, 650], x[1, 3], x[2, 1:] = np.nan, np.inf, low
    x[3] = low
    x[4] = np.nan
    out, ent, tv, ti = logprobs(gpu, "f32", x, np.zeros((5, 1), int), 2, 0.5)
    gpu.sync()
    assert np.isnan(out[[0, 1, 4]]).all() and np.isnan(ent[[0, 1, 4]]).all()
    assert ti[0].tolist() == [0, 1] and ti[1, 0] == 3 and ti[4].tolist() == [-1, -1]
    assert out[2, 0] == 0 and ent[2] == 0 and ti[2].tolist() == [0, 1] and tv[2, 1] == -np.inf
    assert abs(out[3, 0] + np.log(700)) < 1e-5 and abs(ent[3] - np.log(700)) < 1e-5


def test_logprobs_reports_a_label_beyond_the_classes(gpu):
    out, ent, _, _ = logprobs(gpu, "f32", np.zeros((2, 5)), np.array([[5], [4]]), 0, 1.0)
    with pytest.raises(tcu.TcuError, match="outside its range"):
        gpu.sync()
    assert np.isnan(out[0, 0]) and abs(out[1, 0] + np.log(5)) < 1e-6


def test_logprobs_refusals(gpu):
    t = torch.zeros(64, device="cuda")
    p = t.data_ptr()
    for match, a, kw in [("dtype", (7, p, 1, 4, 4, p, 1, p), {}), ("stride", (0, p, 1, 4, 3, p, 1, p), {}),
                         ("classes", (0, p, 1, 0, 4, p, 1, p), {}), ("labels", (0, p, 1, 4, 4, None, 1, p), {}),
                         ("alternatives", (0, p, 1, 4, 4, p, 1, p), dict(top=33, top_values=p, top_ids=p)),
                         ("alternatives", (0, p, 1, 4, 4, p, 1, p), dict(top=2)), ("temperature", (0, p, 1, 4, 4, p, 1, p), dict(temperature=0.0)),
                         ("temperature", (0, p, 1, 4, 4, p, 1, p), dict(temperature=float("nan"))), ("aligned", (0, p + 2, 1, 4, 4, p, 1, p), {})]:
        with pytest.raises(tcu.TcuError, match=match):
            gpu.label_logprobs(*a, stream=1, **kw)
    gpu.label_logprobs(0, None, 0, 4, 4, None, 1, None)


def test_attend_shares_working_memory_between_calls_of_different_shape(gpu):
    """One block of working memory, calls that split their sequences differently one after the other."""
    shapes = [([5000], 1, 1, [1]), ([300] * 40, 4, 8, [1] * 40), ([9000, 10], 2, 4, [1, 1]), ([2000], 1, 8, [3])]
    caches = [Cached(gpu, i, lens, h, 64, 64, 32) for i, (lens, h, _, _) in enumerate(shapes)]
    work = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    for turn in range(2):
        for c, (lens, h, hq, counts) in zip(caches, shapes):
            q = rounded(np.random.default_rng(turn).normal(0, 1, (sum(counts), hq, 64)), torch.bfloat16)
            for window in (0, 700):
                out, lse = c.attend("bf16", q, counts, 0.125, causal=True, window=window, work=work)
                sync(gpu)
                c.check("bf16", q, counts, 0.125, True, window, out, lse)


@pytest.mark.parametrize("test_rows", [1, 40])
def test_the_example_runs_the_operators_together(test_rows):
    """examples/four_bit_member.py on a small member, against the same stage in 64 bits over what its caches and weights stand
    for: within the bar of every cached stage here (5e-5 on raw decoder scores)."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "four_bit_member.py")
    spec = importlib.util.spec_from_file_location("four_bit_member", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    member, h, scores = example.main(["--rows", "700", "--test", str(test_rows)])

    def values(lin):
        """A four-bit layer's weights in 64 bits."""
        g = example.GROUP
        codes = lin.codes.cpu().numpy().reshape(lin.n, -1, 64)
        sc = lin.scales.cpu().numpy().view(np.float16).reshape(lin.n, codes.shape[1], 128 // g, 2)
        w = plain.value(plain.unpack(codes, False), sc[..., 0], sc[..., 1], g).reshape(lin.n, -1)[:, :lin.k]
        return torch.from_numpy(w).cuda(), lin.bias.double()

    def linear(x, lin, gelu=False):
        w, b = values(lin)
        y = x @ w.T + b
        return torch.nn.functional.gelu(y) if gelu else y

    norm = lambda x, p: torch.nn.functional.layer_norm(x, (member.d,), p[0].double(), p[1].double())  # noqa: E731
    x, n, d, w = h.double(), h.shape[0], member.d, member.width
    slots = torch.arange(member.rows, dtype=torch.int64, device="cuda")
    for l, b in enumerate(member.blocks):
        k, v = (torch.empty(member.rows, d, device="cuda") for _ in range(2))
        member.caches[l].load(0, member.rows, slots.data_ptr(), k.data_ptr(), d, w, v.data_ptr(), d, w, stream=1)
        heads = lambda t: t.double().view(-1, member.heads, w).transpose(0, 1)  # noqa: E731
        q = linear(norm(x, b["n1"]), b["wq"])
        m = linear(linear(q.view(-1, w), b["q0"], True), b["q2"]).view(n, d)
        q = q * member.scale[l].double() * (1 + torch.tanh(m))
        att = (torch.softmax(heads(q) @ heads(k).transpose(1, 2), -1) @ heads(v)).transpose(0, 1).reshape(n, d)
        x = x + linear(att, b["wo"])
        x = x + linear(linear(norm(x, b["n2"]), b["w1"], True), b["w2"])
    want = linear(linear(norm(x, member.ln), member.dec0, True), member.dec2)
    assert float((scores.double() - want).abs().max()) <= 5e-5


# ---- many rows: shapes that reach the tensor cores' kernels (more than 40 rows a cache head, in many units or long ones) ----

def check_many(c, dtype, q, n, scale, causal, window, out, lse):
    """As Cached.check, every sequence with n rows, on the device in 64 bits."""
    for s, length in enumerate(c.lens):
        rows = slice(s * n, (s + 1) * n)
        got, gl = out[rows].double(), lse[rows].double()
        if not length:
            assert not got.any() and bool((gl == -np.inf).all())
            continue
        k, v = (torch.from_numpy(x).cuda().transpose(0, 1) for x in (c.k[s], c.v[s]))
        each = q.shape[1] // c.heads
        x = torch.from_numpy(q[rows].astype(np.float64)).cuda().transpose(0, 1)
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(length, device="cuda")[None]
        seen = torch.ones(n, length, dtype=torch.bool, device="cuda")
        if causal:
            seen &= j <= length - n + i
        if window:
            seen &= j > length - n + i - window
        u = 2.0**-11 if dtype != "f32" else 2.0**-20
        for h in range(q.shape[1]):
            kk, vv = k[h // each], v[h // each]
            sc = (x[h] @ kk.T * scale).masked_fill(~seen, -np.inf)
            want_lse = torch.logsumexp(sc, -1)
            some = want_lse > -np.inf
            p = torch.exp(sc - torch.where(some, want_lse, torch.zeros_like(want_lse))[:, None])
            want = torch.where(some[:, None], p @ torch.nan_to_num(vv), torch.zeros_like(x[h]))
            reach = (x[h].abs() @ kk.abs().T * abs(scale)).masked_fill(~seen, 0).amax(-1)
            score = (u + 2.0**-20) * reach
            tol = torch.nan_to_num(vv).abs().max() * (torch.expm1(2 * score) + 3 * u)[:, None] + 2 * ULP[dtype] * want.abs() + 1e-7
            bad = torch.isnan(vv)  # a value that is NaN reaches the rows that see it, and no others
            nan = (seen.double() @ bad.double()) > 0
            assert torch.equal(torch.isnan(got[:, h]), nan)
            assert bool(((got[:, h] - want).abs() <= tol)[~nan].all()), (s, h)
            assert bool((gl[:, h][~some] == -np.inf).all())
            assert bool(((gl[:, h] - want_lse).abs() <= score + 2.0**-20 * (1 + want_lse.abs()))[some].all())


MANY = [
    # width, group, page, heads, q_heads, rows, lens, causal, window
    (64, 32, 16, 1, 2, 30, [0, 1, 29, 30, 31, 63, 64, 65, 127, 200] * 4, True, 0),
    (128, 64, 64, 5, 5, 43, [300, 43, 1, 77, 512, 64, 200, 129], True, 50),
    (32, 32, 32, 8, 24, 17, [100, 16, 17, 18, 130], False, 0),
    (64, 64, 256, 8, 8, 1030, [2050], True, 0),
    (128, 128, 128, 4, 8, 1100, [4000], False, 0),
    (128, 32, 64, 8, 8, 300, [7100], True, 1000),
    (32, 32, 16, 10, 10, 257, [700, 513, 0, 256], True, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width,group,page,heads,q_heads,rows,lens,causal,window", MANY)
def test_attend_many_rows(gpu, dtype, width, group, page, heads, q_heads, rows, lens, causal, window):
    c = Cached(gpu, rows, lens, heads, width, page, group)
    counts = [rows] * len(lens)
    q = rounded(np.random.default_rng(7).normal(0, 1, (sum(counts), q_heads, width)), DT[dtype][1])
    scale = -1 / np.sqrt(width) if rows == 43 else 1 / np.sqrt(width)
    first, _ = c.attend(dtype, q, counts, scale, causal, window)
    out, lse = c.attend(dtype, q, counts, scale, causal, window)
    sync(gpu)
    assert torch.equal(first, out)
    check_many(c, dtype, q, rows, scale, causal, window, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,seqs", [(5, 1), (60, 40)])
def test_attend_a_nan_reaches_only_the_rows_that_see_it(gpu, dtype, rows, seqs):
    """Groups of values that stand for NaN, at tokens that some rows of a step see and others do not."""
    page, group, width = 32, 32, 64
    c = Cached(gpu, 21, [200] * seqs, 1, width, page, group)
    raw = c.pool.cpu().numpy().reshape(c.pages, -1)
    low = page * width // 2 * 2 + page * 4 * 2  # value (step, low) behind key codes, key scales and value codes
    table = c.table.cpu().numpy()
    for s in range(seqs):
        for token, g in ((200 - rows // 2, 1), (199, 0)):
            p, at = table[s, token // page], low + (token % page) * 8 + g * 4
            raw[p, at:at + 4] = np.array([0.0, np.nan], np.float16).view(np.uint8)
            c.v[s][token, 0, g * group:(g + 1) * group] = np.nan
    c.pool.copy_(dev(raw))
    q = rounded(np.random.default_rng(7).normal(0, 1, (rows * seqs, 2, width)), DT[dtype][1])
    out, lse = c.attend(dtype, q, [rows] * seqs, 0.125, causal=True)
    sync(gpu)
    check_many(c, dtype, q, rows, 0.125, True, 0, out, lse)
