"""A prompt's operators on the GPU against plain numpy in 64 bits."""
import numpy as np
import pytest

import prompt_plain as plain
from conftest import tcu

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
# half a unit in the last place of a result of each type, relative, and the smallest subnormal's half
ULP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
TINY = {"f32": 2.0**-150, "f16": 2.0**-25, "bf16": 2.0**-134}
FORMATS = {"mx": plain.MX, "nv": plain.NV}


@pytest.fixture(scope="module")
def gpu():
    return tcu.Gpu(0)


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.double().cpu().numpy()


def rounded(a, dtype):
    """The numbers of a as the type holds them (f64 array)."""
    return torch.from_numpy(np.ascontiguousarray(a, np.float64)).to(dtype).double().numpy()


def sync(gpu):
    torch.cuda.synchronize()
    gpu.sync()


class Matrix:
    """An Fp4 with its buffers: packed by the library from x, or holding codes and scale bytes made by the plain form."""

    def __init__(self, gpu, rows, k, fmt, unit=1.0, fill=0):
        self.fmt, self.k, self.unit = fmt, k, unit
        self.codes = torch.full((tcu.Fp4.code_bytes(rows, k),), fill, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((tcu.Fp4.scale_bytes(rows, k, fmt),), fill, dtype=torch.uint8, device="cuda")
        self.m = tcu.Fp4(gpu, rows, k, fmt, self.codes.data_ptr(), self.scales.data_ptr(), unit=unit)

    def put(self, code, byte):
        packed, place = plain.stored(code, byte)
        self.codes.copy_(dev(packed).flatten())
        s = np.zeros(self.scales.numel(), np.uint8)
        s[place] = byte
        self.scales.copy_(dev(s))
        return plain.values(code, byte, self.fmt, self.unit, self.k)


def random_matrix(rng, gpu, rows, k, fmt, unit=1.0, spread=6):
    """Codes of any number and scales over `spread` powers of two."""
    kp = plain.padded(k)
    code = rng.integers(0, 16, (rows, kp)).astype(np.uint8)
    code[:, k:] = 0
    count = kp // plain.BLOCK[fmt]
    byte = rng.integers(127 - spread, 128, (rows, count)) if fmt == plain.MX else rng.integers(56 - 8 * spread, 57, (rows, count))
    byte[:, -(-k // plain.BLOCK[fmt]):] = 0
    m = Matrix(gpu, rows, k, fmt, unit)
    return m, m.put(code, byte.astype(np.uint8))


# ---- four-bit floating point ----------------------------------------------------------------------------------------

def hard_rows(rng, k, fmt, unit, tt):
    """Rows that meet the format's corners."""
    x = rng.normal(0, 1, (200, k)) * 10.0 ** rng.uniform(-3, 3, (200, 1))
    x[3] = 0
    x[4, ::2] = -0.0
    x[5, k // 2], x[6, 0], x[7, k - 1] = np.nan, np.inf, -np.inf
    x[8] = 3e38 * rng.uniform(-1, 1, k)      # near f32's end
    x[9] = 1e-40 * rng.normal(0, 1, k)       # subnormal in f32 and bf16
    x[10] = 1e-30 * rng.normal(0, 1, k)
    x[11], x[11, 1::2] = 1e-3, 1.0           # small beside large
    # every border of a number, both sides: one number of magnitude 6 a block, the others on borders
    b = np.concatenate([plain.MIDDLES, -plain.MIDDLES])
    for i, off in enumerate((0, 2.0**-9, -2.0**-9, 2.0**-22, -2.0**-22)):
        row = np.resize(b * (1 + off), k)
        row[::8] = 6
        x[12 + i] = row * unit
        x[17 + i] = row * unit * 1.125
        x[22 + i] = row * unit * 448
        x[27 + i] = row * unit * 2.0**-9
    # borders of a scale: the largest of a block 6 unit times the middle of two scales
    mid = (plain.E4M3[1:] + plain.E4M3[:-1]) / 2
    for i in range(60):
        x[40 + i] = rng.uniform(-1, 1, k) * mid[2 * i] * 6 * unit
        x[40 + i, ::16] = mid[2 * i] * 6 * unit * (1, 1, 1 + 2.0**-23, 1 - 2.0**-23)[i % 4]
    with np.errstate(over="ignore"):
        return rounded(x, tt)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["mx", "nv"])
@pytest.mark.parametrize("k,unit", [(128, 1.0), (16, 1.0), (1, 2.0**-7), (130, 0.3), (2050, 0.0123), (200, 1e-30), (256, 1e30)])
def test_pack_and_load(gpu, dtype, name, k, unit):
    code, tt = DT[dtype]
    fmt = FORMATS[name]
    unit = float(np.float32(unit)) if fmt == plain.NV else 1.0
    x = hard_rows(np.random.default_rng(k), k, fmt, unit, tt)
    rows = len(x)
    for pad, at in ((0, 0), (3, 1)):  # aligned where the width is, and not
        buf = torch.full((rows * (k + pad) + at,), 7.0, dtype=tt, device="cuda")
        xd = torch.as_strided(buf, (rows, k), (k + pad, 1), at)
        xd.copy_(dev(x))
        m = Matrix(gpu, rows, k, fmt, unit, fill=0xA5)
        m.m.pack(code, xd.data_ptr(), k + pad, stream=1)
        out = torch.full_like(buf, 9.0)
        yd = torch.as_strided(out, (rows, k), (k + pad, 1), at)
        m.m.load(code, yd.data_ptr(), k + pad, stream=1)
        sync(gpu)
        want_codes, byte = plain.quantise(x, fmt, unit)
        packed, place = plain.stored(want_codes, byte)
        got_codes, got_byte = m.codes.cpu().numpy().reshape(rows, -1), m.scales.cpu().numpy()[place]
        assert np.array_equal(got_byte, byte)
        assert np.array_equal(got_codes, packed)
        n = plain.values(want_codes, byte, fmt, 1.0, k)          # number * scale: exact in f32
        with np.errstate(over="ignore"):
            want = rounded(rounded(n * unit, torch.float32), tt)  # one rounding to f32, one to the type
        assert np.array_equal(host(yd), want, equal_nan=True)
        rest = torch.ones_like(out, dtype=torch.bool)
        torch.as_strided(rest, (rows, k), (k + pad, 1), at).fill_(False)
        assert (out[rest] == 9).all()                            # nothing beside the rows


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("name", ["mx", "nv"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 130), (3, 130), (5, 2050), (2, 513), (7, 600), (131, 50)])
@pytest.mark.parametrize("pad", [0, 1, 6])
def test_pack_few_rows(gpu, dtype, name, rows, k, pad):
    """Sizes whose last threads have nothing to do, and a warp's may have rows of their own; aligned and not."""
    code, tt = DT[dtype]
    fmt = FORMATS[name]
    x = rounded(np.random.default_rng(rows + k).normal(0, 1, (rows, k)), tt)
    unit = float(np.float32(np.abs(x).max() / 2688)) if fmt == plain.NV else 1.0
    xd = torch.as_strided(torch.zeros(rows * (k + pad) + 8, dtype=tt, device="cuda"), (rows, k), (k + pad, 1), pad % 4)
    xd.copy_(dev(x))
    m = Matrix(gpu, rows, k, fmt, unit, fill=0xA5)
    m.m.pack(code, xd.data_ptr(), k + pad, stream=1)
    y = torch.full((rows, k + pad), 9.0, dtype=tt, device="cuda")
    m.m.load(code, y.data_ptr(), k + pad, stream=1)
    sync(gpu)
    want_codes, byte = plain.quantise(x, fmt, unit)
    packed, place = plain.stored(want_codes, byte)
    assert np.array_equal(m.codes.cpu().numpy().reshape(rows, -1), packed)
    assert np.array_equal(m.scales.cpu().numpy()[place], byte)
    want = rounded(rounded(plain.values(want_codes, byte, fmt, 1.0, k) * unit, torch.float32), tt)
    assert np.array_equal(host(y[:, :k]), want) and (y[:, k:] == 9).all()


def test_pack_writes_no_row_behind_the_last(gpu):
    """Scales of rows that the matrix does not have are left as they were."""
    m = Matrix(gpu, 130, 64, plain.NV, fill=0xA5)
    x = torch.ones(130, 64, device="cuda")
    m.m.pack(0, x.data_ptr(), 64, stream=1)
    sync(gpu)
    s = m.scales.cpu().numpy()
    _, place = plain.stored(np.zeros((130, 128), np.uint8), np.zeros((130, 8), np.uint8))
    rest = np.ones(s.size, bool)
    rest[place] = False
    assert (s[rest] == 0xA5).all() and rest.sum() == 2 * 2 * 512 - 130 * 8


LINEAR = [  # rows, n, k
    (1, 1, 1), (1, 128, 128), (1, 1024, 512), (3, 200, 130), (8, 4097, 700), (16, 256, 256), (17, 130, 2050), (33, 100, 512),
    (64, 1000, 1000), (65, 129, 384), (127, 300, 100), (128, 512, 1024), (129, 513, 640), (256, 128, 64), (257, 1000, 2000), (600, 700, 900),
    (8, 300, 33000), (33, 64, 20000), (150, 130, 16400),  # few tiles of many steps: cut
]


def check_linear(gpu, rng, dtype, fmt, rows, n, k, act, bias, residual, ux=1.0, uw=1.0, exact=False):
    code, tt = DT[dtype]
    spread = 2 if exact else 6
    x, xv = random_matrix(rng, gpu, rows, k, fmt, ux, spread)
    w, wv = random_matrix(rng, gpu, n, k, fmt, uw, spread)
    b = rounded(rng.normal(0, 1, n), tt) if bias else None
    r = rounded(rng.normal(0, 1, (rows, n)), tt) if residual else None
    yd = torch.full((rows, n + 3), 9.0, dtype=tt, device="cuda")
    if residual:
        yd[:, :n] = dev(r, tt)  # in place: the residual is the output's own buffer
    bd = dev(b, tt) if bias else None
    work = torch.zeros(w.m.linear_workspace(x.m, code), dtype=torch.uint8, device="cuda")
    w.m.linear(x.m, code, yd.data_ptr(), n + 3, bias=bd.data_ptr() if bias else None, act=act, residual=yd.data_ptr() if residual else None,
               ldr=n + 3, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    y, size = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    got = host(yd)
    assert (got[:, n:] == 9).all()
    if exact:
        assert np.array_equal(got[:, :n], rounded(y, tt))
        return
    # a sum of 64 products is added to the one before at a time, each addition off by a unit in the last place of f32 (the matrix
    # unit does not round to nearest); f32 results add four steps of 4 such sums at a time
    adds = -(-k // 64) + 8 if dtype != "f32" else 16 + -(-k // 1024) + 8
    tol = adds * 2.0**-23 * size
    if bias:
        y, tol = y + b, tol + 2.0**-23 * np.abs(b)
    if act:
        erf = torch.erf(torch.from_numpy(y / np.sqrt(2))).numpy()
        y, tol = 0.5 * y * (1 + erf), 1.13 * tol + 2.0**-20 * np.abs(y)  # the slope of GELU is below 1.13; its erf is good to 2^-21
    if residual:
        y, tol = y + r, tol + 2.0**-23 * np.abs(r)
    assert (np.abs(got[:, :n] - y) <= tol + 2 * ULP[dtype] * np.abs(y) + TINY[dtype]).all()
    counters = work[:8192].cpu().numpy()
    assert not counters.any()  # left as the next call needs them


@pytest.mark.parametrize("name", ["mx", "nv"])
@pytest.mark.parametrize("rows,n,k", [(1, 128, 128), (16, 128, 128), (16, 256, 256), (130, 140, 256), (300, 200, 512), (20, 300, 2050)])
def test_linear_exact(gpu, name, rows, n, k):
    """Scales of a few powers of two: every sum of products is a number that f32 holds, whatever the order."""
    rng = np.random.default_rng(rows + n + k)
    fmt = FORMATS[name]
    x, xv = random_matrix(rng, gpu, rows, k, fmt, spread=2)
    w, wv = random_matrix(rng, gpu, n, k, fmt, spread=2)
    if fmt == plain.NV:  # whole powers of two among the e4m3 floats
        for m, rws in ((x, rows), (w, n)):
            code = rng.integers(0, 16, (rws, plain.padded(k))).astype(np.uint8)
            code[:, k:] = 0
            byte = (rng.integers(5, 8, (rws, plain.padded(k) // 16)) * 8).astype(np.uint8)
            if m is x:
                xv = m.put(code, byte)
            else:
                wv = m.put(code, byte)
    y = torch.full((rows, n), 9.0, device="cuda")
    work = torch.zeros(w.m.linear_workspace(x.m, 0), dtype=torch.uint8, device="cuda")
    w.m.linear(x.m, 0, y.data_ptr(), n, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    # products are multiples of 2^-2 * 2^-4, sums below 36 * 4 * k: 22 bits at most
    assert np.array_equal(host(y), xv @ wv.T)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["mx", "nv"])
@pytest.mark.parametrize("rows,n,k", LINEAR)
def test_linear(gpu, dtype, name, rows, n, k):
    rng = np.random.default_rng(rows * 7 + n + k)
    ux, uw = (0.37, 0.0021) if name == "nv" else (1.0, 1.0)
    check_linear(gpu, rng, dtype, FORMATS[name], rows, n, k, act=rows % 2, bias=n % 3 > 0, residual=k % 3 > 0, ux=ux, uw=uw)


# ---- attention of packed rows ---------------------------------------------------------------------------------------

def check_attend(gpu, dtype, q_lens, k_lens, q_heads, heads, width, causal, window, scale=None, spoil=None, pad=0, at=0, seed=0, lse=True,
                 own_rows=False, extra=2):
    """Random rows; `spoil` may change the arrays (f64, as the type holds them) before they go to the device. pad, at: strides and
    starts that are not aligned. extra: rows behind the last sequence."""
    code, tt = DT[dtype]
    rng = np.random.default_rng(seed + sum(q_lens) + 7 * sum(k_lens) + width)
    tq, tk = sum(q_lens) + extra, sum(k_lens) + extra
    q, k, v = (rounded(rng.normal(0, 1, (n, h, width)), tt) for n, h in ((tq, q_heads), (tk, heads), (tk, heads)))
    if spoil:
        spoil(q, k, v)
    scale = 1 / np.sqrt(width) if scale is None else scale
    put = lambda x: torch.as_strided(torch.full((x.shape[0] * (x.shape[1] * (width + pad) + pad) + at + 8,), float("nan"), dtype=tt, device="cuda"),
                                     x.shape, (x.shape[1] * (width + pad) + pad, width + pad, 1), at)  # noqa: E731
    qd, kd, vd, od = put(q), put(k), put(v), put(q)
    for t, x in ((qd, q), (kd, k), (vd, v)):
        t.copy_(dev(x))
    od.fill_(9)
    ld = torch.full((tq, q_heads), 9.0, device="cuda")
    starts = lambda lens: dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))  # noqa: E731
    qs, ks = starts(q_lens), starts(k_lens)
    p = tcu.Packed(gpu, len(q_lens), tq, tk, max(q_lens), max(k_lens), qs.data_ptr(), None if own_rows else ks.data_ptr())
    work = torch.zeros(p.attend_workspace(code, q_heads, heads, width), dtype=torch.uint8, device="cuda")
    p.attend(code, q_heads, heads, width, qd.data_ptr(), qd.stride(0), qd.stride(1), kd.data_ptr(), kd.stride(0), kd.stride(1), vd.data_ptr(),
             vd.stride(0), vd.stride(1), od.data_ptr(), od.stride(0), od.stride(1), float(np.float32(scale)), causal=causal, window=window,
             lse=ld.data_ptr() if lse else None, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    assert not work[:8192].any()  # left as the next call needs them
    n = sum(q_lens)
    got, got_lse = host(od), host(ld)
    assert (got[n:] == 9).all() and (got_lse[n:] == 9).all()  # rows behind the last sequence
    with np.errstate(all="ignore"):
        want, want_lse = plain.attend(q[:n], k, v, q_lens, k_lens, heads, float(np.float32(scale)), causal, window)
        # what each weight may be off by, relative: its score's rounding (products of f32 held to 2^-21, each of the width's sums to 2^-23
        # of the largest), the weight's to the type, the exponential's; an output is off by that of sum p |v|, and its own rounding
        kmax = max([1e-30] + [np.abs(x[np.isfinite(x)]).max() for x in (k,) if np.isfinite(x).any()])
        qmax = np.abs(np.where(np.isfinite(q[:n]), q[:n], 0)).sum(-1)
        score = abs(scale) * qmax * kmax * (2.0**-20 if dtype == "f32" else 2.0**-22) + 2.0**-20
        weight = score + 2.0**-20 + (0 if dtype == "f32" else ULP[dtype])
        size, _ = plain.attend(q[:n], k, np.abs(v), q_lens, k_lens, heads, float(np.float32(scale)), causal, window)
        size = np.where(np.isfinite(size), size, 0)
        tol = 2 * weight[..., None] * size + 1.01 * ULP[dtype] * np.abs(np.where(np.isfinite(want), want, 0)) + 2 * TINY[dtype] + 2.0**-126
        fine = np.isfinite(want)
        assert np.array_equal(np.isnan(got[:n]), np.isnan(want)), "NaN where there is none, or none where there is one"
        assert np.array_equal(got[:n][~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
        assert (np.abs(got[:n] - want)[fine] <= tol[fine]).all(), np.max(np.abs(got[:n] - want)[fine] / tol[fine])
        if lse:
            a, b = got_lse[:n], want_lse
            fine = np.isfinite(b)
            assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~fine & ~np.isnan(b)], b[~fine & ~np.isnan(b)])
            assert (np.abs(a - b)[fine] <= (score + 2.0**-20 + 2.0**-22 * np.abs(b))[fine]).all()
        else:
            assert (got_lse == 9).all()
    return got[:n]


LENS = [  # query rows, keys
    ([1], [1]), ([1], [300]), ([1, 1, 1], [0, 1, 700]), ([3], [3]), ([5, 0, 17], [5, 9, 17]), ([16], [64]), ([17], [65]), ([33, 1, 64], [33, 200, 64]),
    ([129], [129]), ([128, 256], [128, 256]), ([300, 40], [333, 40]), ([7, 4], [3, 0]), ([200], [190]), ([2, 90], [1000, 90]),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,heads,width", [(1, 1, 64), (4, 2, 128), (6, 2, 32), (8, 1, 96), (3, 1, 8), (2, 2, 256), (4, 4, 120)])
@pytest.mark.parametrize("mask", ["all", "causal", "window"])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "x".join(map(str, x[0])) + "-" + "x".join(map(str, x[1])))
def test_attend(gpu, dtype, q_heads, heads, width, mask, lens):
    check_attend(gpu, dtype, *lens, q_heads, heads, width, mask != "all", 11 if mask == "window" else 0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,heads,width", [(40, 40, 64), (24, 24, 128), (60, 20, 64), (64, 16, 32)])
@pytest.mark.parametrize("lens", [[300, 20, 563], [130], [257, 1, 1, 390]], ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_attend_many_units(gpu, dtype, q_heads, heads, width, lens, causal):
    """Blocks with many pieces of work each, among them tiles with few rows beside tiles with none."""
    check_attend(gpu, dtype, lens, lens, q_heads, heads, width, causal, 0, own_rows=causal)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_heads,width", [(129, 64), (150, 32), (128, 128), (16, 64), (5, 128), (300, 64)])
def test_attend_many_heads_on_one(gpu, dtype, q_heads, width):
    """More heads of a token than a tile has rows, and numbers that do not divide it."""
    check_attend(gpu, dtype, [3, 40], [3, 70], q_heads, 1, width, True, 0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attend_many_sequences(gpu, dtype):
    rng = np.random.default_rng(0)
    check_attend(gpu, dtype, [1] * 3000, list(rng.integers(0, 5, 3000)), 2, 1, 32, False, 0)
    lens = list(rng.integers(0, 3, 1500)) + [70]
    check_attend(gpu, dtype, lens, lens, 2, 2, 64, True, 0, own_rows=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 100])
def test_attend_starts_behind_the_first_row(gpu, dtype, rows):
    """Rows and keys before the first sequence's are nobody's."""
    code, tt = DT[dtype]
    q, k, v = (torch.randn(n, 2, 64, device="cuda").to(tt) for n in (rows + 7, 140, 140))
    k[:9], v[:9] = float("nan"), float("inf")
    out = torch.full_like(q, 9.0)
    qs, ks = torch.tensor([7, rows + 7], dtype=torch.int32, device="cuda"), torch.tensor([9, 139], dtype=torch.int32, device="cuda")
    p = tcu.Packed(gpu, 1, rows + 7, 140, rows, 130, qs.data_ptr(), ks.data_ptr())
    work = torch.zeros(p.attend_workspace(code, 2, 2, 64), dtype=torch.uint8, device="cuda")
    p.attend(code, 2, 2, 64, q.data_ptr(), 128, 64, k.data_ptr(), 128, 64, v.data_ptr(), 128, 64, out.data_ptr(), 128, 64, 0.125,
             work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    want, _ = torch_attend(q[7:], k[9:139], v[9:139], 0.125)
    assert (out[:7] == 9).all() and (out[7:].double() - want).abs().max() <= 2 * ULP["bf16"] * 4.5  # (a weight's rounding, of values up to 4.5)


def test_linear_of_many_rows(gpu):
    """More rows than a 16-bit number counts, and a product of a matrix with itself."""
    rng = np.random.default_rng(1)
    x, xv = random_matrix(rng, gpu, 70_001, 64, plain.NV)
    w, wv = random_matrix(rng, gpu, 40, 64, plain.NV)
    for m, mv in ((w, wv), (None, None)):
        if m is None:
            x, xv = random_matrix(rng, gpu, 300, 64, plain.MX)
            m, mv = x, xv
        y = torch.zeros(len(xv), len(mv), dtype=torch.bfloat16, device="cuda")
        work = torch.zeros(m.m.linear_workspace(x.m, 2), dtype=torch.uint8, device="cuda")
        m.m.linear(x.m, 2, y.data_ptr(), len(mv), work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        sync(gpu)
        want, size = xv @ mv.T, np.abs(xv) @ np.abs(mv).T
        assert (np.abs(host(y) - want) <= 9 * 2.0**-23 * size + 1.01 * ULP["bf16"] * np.abs(want)).all()


FEW, MANY = ([5, 1, 12], [40, 70, 12]), ([150, 90], [190, 90])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("what", ["nan", "inf", "queries", "behind"])
def test_attend_hides_what_is_not_seen(gpu, dtype, lens, width, what):
    """NaN and infinities in keys and values reach the rows that see them and no others, in the same tile or the next sequence;
    behind the last sequence nobody's."""
    ends = np.cumsum(lens[1])

    def spoil(q, k, v):
        if what == "nan":
            v[ends[0] - 3, 0, 5], k[ends[1] - 2, 1, 3], v[ends[0], 1] = np.nan, np.nan, np.nan
        elif what == "inf":
            v[ends[0] - 3, 0], v[ends[0], 1, 7], k[ends[1] - 1, 0, 0] = np.inf, -np.inf, np.inf
        elif what == "queries":
            q[1, 2, 0], q[4, 0] = np.nan, 0
        else:
            k[ends[-1]:], v[ends[-1]:] = np.nan, np.inf
    check_attend(gpu, dtype, *lens, 4, 2, width, True, 0, spoil=spoil)
    if what != "inf":  # (a plain sum of infinities of one sign and other numbers has no weights of nothing)
        check_attend(gpu, dtype, *lens, 4, 2, width, True, 9, spoil=spoil)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("pad,at", [(1, 0), (0, 1), (3, 5), (8, 8), (4, 4)])
def test_attend_strides(gpu, dtype, lens, pad, at):
    for width in (64, 120):
        check_attend(gpu, dtype, *lens, 6, 3, width, True, 0, pad=pad, at=at)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_attend_scales(gpu, dtype, lens, scale):
    check_attend(gpu, dtype, *lens, 4, 2, 64, True, 0, scale=scale)
    check_attend(gpu, dtype, *lens, 6, 2, 128, False, 0, scale=scale, lse=False)


@pytest.mark.parametrize("lens", [FEW, MANY], ids=["few", "many"])
def test_attend_f32_of_every_size(gpu, lens):
    """Keys and values whose tiles are many powers of two apart: each tile of 64 keys is held to its own largest."""
    def spoil(q, k, v):
        for j in range(0, len(v), 64):
            v[j:j + 64] *= 10.0 ** (((j // 64) * 7) % 33 - 15)
        q[:2] *= 1e18
        k[:70] *= 1e-18
    check_attend(gpu, "f32", [lens[0][0]], [lens[1][0]], 4, 2, 128, False, 0, spoil=lambda q, k, v: v.__imul__(1e30))
    check_attend(gpu, "f32", [lens[0][0]], [lens[1][0]], 4, 2, 64, False, 0, spoil=lambda q, k, v: v.__imul__(1e-33))

    def apart(q, k, v):  # rows 0..63 of the keys are seen by all rows, of small values; those behind have large ones
        v[64:128] *= 1e25
        q *= 1e-3
    check_attend(gpu, "f32", [lens[0][0]], [lens[1][0]], 4, 2, 128, True, 0, spoil=apart)
    check_attend(gpu, "f32", [lens[0][0]], [lens[1][0]], 4, 2, 128, False, 0, spoil=spoil)


def torch_attend(q, k, v, scale):
    """One sequence, every row sees every key, in 64 bits on the GPU."""
    each = q.shape[1] // k.shape[1]
    s = torch.einsum("nhw,mhw->hnm", q.double(), k.double().repeat_interleave(each, 1)) * scale
    return torch.einsum("hnm,mhw->nhw", torch.softmax(s, -1), v.double().repeat_interleave(each, 1)), torch.logsumexp(s, -1).t()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,keys,width", [(1, 100_000, 128), (3, 33_333, 64), (130, 20_001, 128), (300, 9_999, 64), (1, 30_000, 256)])
def test_attend_long(gpu, dtype, rows, keys, width):
    code, tt = DT[dtype]
    gen = torch.Generator(device="cuda").manual_seed(keys)
    q, k, v = (torch.randn(n, h, width, generator=gen, device="cuda").to(tt) for n, h in ((rows, 4), (keys, 2), (keys, 2)))
    qs, ks = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (rows, keys))
    p = tcu.Packed(gpu, 1, rows, keys, rows, keys, qs.data_ptr(), ks.data_ptr())
    work = torch.zeros(p.attend_workspace(code, 4, 2, width), dtype=torch.uint8, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(rows, 4, device="cuda")
    first = None
    for _ in range(2):  # the same to the last bit again: parts are joined in their order
        p.attend(code, 4, 2, width, q.data_ptr(), 4 * width, width, k.data_ptr(), 2 * width, width, v.data_ptr(), 2 * width, width, out.data_ptr(),
                 4 * width, width, width**-0.5, lse=lse.data_ptr(), work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        sync(gpu)
        assert first is None or torch.equal(first, out)
        first = out.clone()
    want, want_lse = torch_attend(q, k, v, width**-0.5)
    # an output is a sum of thousands of values of either sign: errors of its weights (2^-8, 2^-11 of them, of either sign too) add as
    # their squares do, and so do the values: relative to the root of the sum of p^2 v^2 a weight's error is a rounding
    off = (out.double() - want).norm() / want.norm()
    assert off <= {"f32": 2e-6, "f16": 2.0 * 2**-11, "bf16": 2.0 * 2**-8}[dtype], off
    assert (lse.double() - want_lse).abs().max() <= 2.0**-18


def test_attend_past_32_bits(gpu):
    """Keys and values whose rows begin up to 2^32 elements apart."""
    rows, keys, w = 100, 200, 64
    step = 21_500_000  # 200 rows of it: 4.3e9 elements
    big = torch.zeros(keys * step + 1024, dtype=torch.float16, device="cuda")
    k = torch.as_strided(big, (keys, 1, w), (step, w, 1), 0)
    v = torch.as_strided(big, (keys, 1, w), (step, w, 1), 512)
    q = torch.randn(rows, 1, w, device="cuda").half()
    k.copy_(torch.randn(keys, 1, w, device="cuda")), v.copy_(torch.randn(keys, 1, w, device="cuda"))
    want, want_lse = torch_attend(q, k.contiguous(), v.contiguous(), 0.125)
    for n in (1, rows):
        qs, ks = (torch.tensor([0, x], dtype=torch.int32, device="cuda") for x in (n, keys))
        p = tcu.Packed(gpu, 1, n, keys, n, keys, qs.data_ptr(), ks.data_ptr())
        work = torch.zeros(p.attend_workspace(1, 1, 1, w), dtype=torch.uint8, device="cuda")
        out, lse = torch.zeros_like(q), torch.zeros(rows, 1, device="cuda")
        p.attend(1, 1, 1, w, q.data_ptr(), w, w, k.data_ptr(), step, w, v.data_ptr(), step, w, out.data_ptr(), w, w, 0.125, lse=lse.data_ptr(),
                 work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        sync(gpu)
        # 11 bits of a weight and of an output, of values up to 4.5
        assert (out[:n].double() - want[:n]).abs().max() <= 2 * 2.0**-11 * 4.5
        assert (lse[:n].double() - want_lse[:n]).abs().max() <= 2.0**-18
        assert not out[n:].any()


@pytest.mark.parametrize("q_starts,k_starts", [([0, 200, 90], [0, 90, 180]), ([0, 90, 180], [0, 250, 180]), ([-4, 90, 180], [0, 90, 180]),
                                               ([0, 90, 2**31 - 1], [0, 90, 180]), ([0, 90, 180], [90, 0, 2**30])])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attend_reports_bad_starts(gpu, dtype, q_starts, k_starts):
    """A sequence whose rows or keys lie outside what was said is left alone and reported; the others are worked out."""
    code, tt = DT[dtype]
    q = torch.randn(180, 2, 64, device="cuda").to(tt)
    out = torch.full_like(q, 9.0)
    qs, ks = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (q_starts, k_starts))
    p = tcu.Packed(gpu, 2, 180, 180, 90, 90, qs.data_ptr(), ks.data_ptr())
    work = torch.zeros(p.attend_workspace(code, 2, 2, 64), dtype=torch.uint8, device="cuda")
    p.attend(code, 2, 2, 64, q.data_ptr(), 128, 64, q.data_ptr(), 128, 64, q.data_ptr(), 128, 64, out.data_ptr(), 128, 64, 0.125,
             work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    torch.cuda.synchronize()
    with pytest.raises(tcu.TcuError, match="outside its range"):
        gpu.sync()
    good = [s for s in range(2) if 0 <= q_starts[s] <= q_starts[s + 1] <= 180 and q_starts[s + 1] - q_starts[s] <= 90
            and 0 <= k_starts[s] <= k_starts[s + 1] <= 180 and k_starts[s + 1] - k_starts[s] <= 90]
    done = torch.zeros(180, dtype=torch.bool, device="cuda")
    for s in good:
        rows, keys = slice(q_starts[s], q_starts[s + 1]), slice(k_starts[s], k_starts[s + 1])
        want, _ = torch_attend(q[rows], q[keys], q[keys], 0.125)
        assert (out[rows].double() - want).abs().max() <= 2.0**-8
        done[rows] = True
    assert (out[~done] == 9).all()
    gpu.sync()


def test_attend_refusals(gpu):
    t = torch.zeros(64, 4, 64, device="cuda")
    s = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    p = tcu.Packed(gpu, 1, 64, 64, 64, 64, s.data_ptr(), s.data_ptr())
    work = torch.zeros(p.attend_workspace(0, 4, 4, 64), dtype=torch.uint8, device="cuda")
    x = t.data_ptr()
    ok = dict(dtype=0, q_heads=4, heads=4, width=64, q_ptr=x, q_row=256, q_head=64, k_ptr=x, k_row=256, k_head=64, v_ptr=x, v_row=256, v_head=64,
              out_ptr=x, o_row=256, o_head=64, scale=1.0, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    for match, kw in [("dtype", dict(dtype=3)), ("heads", dict(heads=3)), ("heads", dict(heads=0)), ("heads", dict(q_heads=0)), ("width", dict(width=12)),
                      ("width", dict(width=264)), ("width", dict(width=0)), ("window", dict(window=3)), ("window", dict(causal=True, window=-1)),
                      ("scale", dict(scale=float("nan"))), ("scale", dict(scale=float("inf"))), ("strides", dict(k_row=-1)), ("null", dict(q_ptr=None)),
                      ("null", dict(v_ptr=None)), ("null", dict(out_ptr=None)), ("aligned", dict(k_ptr=x + 2)), ("aligned", dict(out_ptr=x + 1)),
                      ("working memory", dict(work_bytes=8)), ("working memory", dict(work=None)), ("aligned", dict(work=work.data_ptr() + 4))]:
        with pytest.raises(tcu.TcuError, match=match):
            p.attend(**{**ok, **kw})
    for bad in (dict(seqs=-1), dict(seqs=70_000), dict(q_rows=-1), dict(max_k=-1), dict(q_rows=2**30)):
        b = tcu.Packed(gpu, **{**dict(seqs=1, q_rows=64, k_rows=64, max_q=64, max_k=64, q_starts_ptr=s.data_ptr()), **bad})
        with pytest.raises(tcu.TcuError):
            b.attend_workspace(0, 4, 4, 64)
    with pytest.raises(tcu.TcuError, match="null"):
        tcu.Packed(gpu, 1, 64, 64, 64, 64, None).attend(**ok)
    for none in (dict(seqs=0), dict(q_rows=0), dict(max_q=0)):  # nothing to do
        b = tcu.Packed(gpu, **{**dict(seqs=1, q_rows=64, k_rows=64, max_q=64, max_k=64, q_starts_ptr=None), **none})
        assert b.attend_workspace(0, 4, 4, 64) == 0
        b.attend(**{**ok, "work": None, "work_bytes": 0})
    p.attend(**ok)
    sync(gpu)


def test_fp4_refusals(gpu):
    t = torch.zeros(65536, dtype=torch.uint8, device="cuda")
    x = t.data_ptr()
    ok = dict(rows=4, k=64, format=tcu.NV, codes_ptr=x, scales_ptr=x, unit=1.0)
    for match, kw in [("rows", dict(rows=0)), ("rows", dict(k=0)), ("rows", dict(k=2**25)), ("rows", dict(rows=2**24, k=4096)), ("format", dict(format=2)),
                      ("unit", dict(unit=0.0)), ("unit", dict(unit=float("nan"))), ("unit", dict(unit=1e31)), ("unit", dict(unit=-1.0)),
                      ("unit", dict(format=tcu.MX, unit=2.0)), ("null", dict(codes_ptr=None)), ("null", dict(scales_ptr=None)),
                      ("aligned", dict(codes_ptr=x + 8)), ("aligned", dict(scales_ptr=x + 4))]:
        m = tcu.Fp4(gpu, **{**ok, **kw})
        for call in (lambda: m.pack(0, x, 2**26, stream=1), lambda: m.load(0, x, 2**26, stream=1), lambda: m.linear_workspace(m, 0)):
            with pytest.raises(tcu.TcuError, match=match):
                call()
    m = tcu.Fp4(gpu, **ok)
    for match, a in [("dtype", (3, x, 64)), ("null", (0, None, 64)), ("stride", (0, x, 63)), ("aligned", (0, x + 2, 64))]:
        with pytest.raises(tcu.TcuError, match=match):
            m.pack(*a, stream=1)
        with pytest.raises(tcu.TcuError, match=match):
            m.load(*a, stream=1)
    work = torch.zeros(m.linear_workspace(m, 0), dtype=torch.uint8, device="cuda")
    w = dict(work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    for match, a, kw in [("dtype", (m, 5, x, 4), w), ("null", (m, 0, None, 4), w), ("stride", (m, 0, x, 3), w), ("stride", (m, 0, x, 4), dict(w, residual=x, ldr=3)),
                         ("act", (m, 0, x, 4), dict(w, act=2)), ("aligned", (m, 0, x + 2, 4), w), ("aligned", (m, 0, x, 4), dict(w, bias=x + 1)),
                         ("working memory", (m, 0, x, 4), dict(w, work_bytes=16)), ("working memory", (m, 0, x, 4), dict(w, work=None)),
                         ("format", (tcu.Fp4(gpu, **{**ok, "format": tcu.MX}), 0, x, 4), w), ("format", (tcu.Fp4(gpu, **{**ok, "k": 65}), 0, x, 4), w),
                         ("units", (tcu.Fp4(gpu, **{**ok, "unit": 1e-30}), 0, x, 4), w)]:
        with pytest.raises(tcu.TcuError, match=match):
            (tcu.Fp4(gpu, **{**ok, "unit": 1e-30}) if match == "units" else m).linear(*a, **kw)
    assert tcu.Fp4.code_bytes(0, 4) == 0 and tcu.Fp4.code_bytes(2**25, 2**24) == 0 and tcu.Fp4.scale_bytes(4, 4, 2) == 0
    sync(gpu)


@pytest.mark.parametrize("name", ["mx", "nv"])
@pytest.mark.parametrize("rows", [5, 40, 200])
def test_linear_keeps_rows_apart(gpu, name, rows):
    """A NaN scale in a row of x or of W makes that row's or column's outputs NaN and no others."""
    fmt = FORMATS[name]
    rng = np.random.default_rng(rows)
    x, xv = random_matrix(rng, gpu, rows, 300, fmt)
    w, wv = random_matrix(rng, gpu, 150, 300, fmt)
    for m, row in ((x, 3), (w, 129)):
        m.scales[row // 128 * (m.scales.numel() // (-(-(rows if m is x else 150) // 128))) + row % 32 * 16 + row % 128 // 32 * 4 + 1] = 255 if fmt == plain.MX else 127
    y = torch.zeros(rows, 150, device="cuda")
    work = torch.zeros(w.m.linear_workspace(x.m, 0), dtype=torch.uint8, device="cuda")
    w.m.linear(x.m, 0, y.data_ptr(), 150, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    got = host(y)
    assert np.isnan(got[3]).all() and np.isnan(got[:, 129]).all()
    fine = np.ones((rows, 150), bool)
    fine[3], fine[:, 129] = False, False
    want, size = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    assert (np.abs(got - want) <= 30 * 2.0**-23 * size)[fine].all()


# ---- a run of them together -----------------------------------------------------------------------------------------

def gelu(x):
    return 0.5 * x * (1 + torch.erf(x / 2**0.5))


class Layer:
    """A prompt's layer on the operators: projection, attention, the cache's store, output with residual, feed-forward, answer."""

    def __init__(self, gpu, dtype, lens, d, q_heads, heads, width, ff, classes, fmt):
        self.gpu, self.lens, self.fmt = gpu, lens, fmt
        self.code, self.tt = DT[dtype]
        self.hq, self.h, self.w, self.d, self.ff, self.classes = q_heads, heads, width, d, ff, classes
        gen = torch.Generator(device="cuda").manual_seed(5)
        rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        n = sum(lens)
        self.x = rand(n, d).to(self.tt)
        self.weights = {}
        for name, rows, cols in (("qkv", (q_heads + 2 * heads) * width, d), ("out", d, q_heads * width), ("up", ff, d), ("down", d, ff), ("head", classes, d)):
            self.weights[name] = (self.matrix(rows, cols), (0.1 * rand(rows)).to(self.tt))
            w = (rand(rows, cols) / cols**0.5).to(self.tt)
            self.weights[name][0].pack(self.code, w, float(w.abs().max()) / 2688 if fmt == tcu.NV else 1.0)
        self.inputs = {k: self.matrix(n, c) for k, c in (("x", d), ("a", q_heads * width), ("h", d), ("f", ff), ("y", d))}
        new = lambda *s, dt=self.tt: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
        self.qkv, self.att, self.hid, self.up, self.y = new(n, q_heads + 2 * heads, width), new(n, q_heads * width), new(n, d), new(n, ff), new(n, d)
        self.logits, self.lp, self.lse = new(n, classes), new(n, 1, dt=torch.float32), new(n, q_heads, dt=torch.float32)
        self.labels = torch.randint(0, classes, (n, 1), generator=gen, device="cuda").int()
        self.starts = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
        self.packed = tcu.Packed(gpu, len(lens), n, n, max(lens), max(lens), self.starts.data_ptr())
        pages = -(-n // 64) + 1
        self.pool = torch.zeros(pages * tcu.Kv4Cache.page_bytes(heads, width, 64, 32), dtype=torch.uint8, device="cuda")
        self.cache = tcu.Kv4Cache(gpu, self.pool.data_ptr(), pages, heads=heads, width=width, page=64, group=32)
        self.slots = torch.arange(n, device="cuda")
        need = max([self.packed.attend_workspace(self.code, q_heads, heads, width)] +
                   [self.weights[k][0].m.m.linear_workspace(self.inputs[i].m.m, self.code) for k, i in (("qkv", "x"), ("out", "a"), ("up", "h"), ("down", "f"), ("head", "y"))])
        self.work = torch.zeros(need, dtype=torch.uint8, device="cuda")  # one block serves them all

    def matrix(self, rows, cols):
        layer = self

        class Held:
            def __init__(self):
                self.rows, self.cols, self.m = rows, cols, None

            def pack(self, code, x, unit, stream=1):
                if self.m is None:
                    self.m = Matrix(layer.gpu, rows, cols, layer.fmt, unit)
                self.m.m.pack(code, x.data_ptr(), cols, stream=stream)

            def values(self):
                y = torch.empty(rows, cols, device="cuda")
                self.m.m.load(0, y.data_ptr(), cols, stream=1)
                return y.double()
        held = Held()
        held.m = Matrix(layer.gpu, rows, cols, layer.fmt, 1.0 if layer.fmt == tcu.MX else 2.0**-9)
        return held

    def linear(self, name, inp, src, out, stream, act=0, residual=None):
        self.inputs[inp].pack(self.code, src, None, stream)
        w, b = self.weights[name]
        w.m.m.linear(self.inputs[inp].m.m, self.code, out.data_ptr(), w.rows, bias=b.data_ptr(), act=act,
                     residual=residual.data_ptr() if residual is not None else None, ldr=w.rows, work=self.work.data_ptr(),
                     work_bytes=self.work.numel(), stream=stream)

    def run(self, stream):
        hq, h, w, es = self.hq, self.h, self.w, self.x.element_size()
        row = (hq + 2 * h) * w
        self.linear("qkv", "x", self.x, self.qkv, stream)
        q = self.qkv.data_ptr()
        k, v = q + hq * w * es, q + (hq + h) * w * es
        self.packed.attend(self.code, hq, h, w, q, row, w, k, row, w, v, row, w, self.att.data_ptr(), hq * w, w, w**-0.5, causal=True,
                           lse=self.lse.data_ptr(), work=self.work.data_ptr(), work_bytes=self.work.numel(), stream=stream)
        self.cache.store(self.code, len(self.slots), self.slots.data_ptr(), k, row, w, v, row, w, stream=stream)
        self.linear("out", "a", self.att, self.hid, stream, residual=self.x)
        self.linear("up", "h", self.hid, self.up, stream, act=1)
        self.linear("down", "f", self.up, self.y, stream, residual=self.hid)
        self.linear("head", "y", self.y, self.logits, stream)
        self.gpu.label_logprobs(self.code, self.logits.data_ptr(), len(self.slots), self.classes, self.classes, self.labels.data_ptr(), 1,
                                self.lp.data_ptr(), stream=stream)

    def check(self, tol):
        """Each stage against 64 bits from what the stage before has left."""
        def linear(name, inp):
            w, b = self.weights[name]
            return self.inputs[inp].values() @ w.values().t() + b.double()
        near = lambda a, b: (a.double() - b).norm() <= tol * b.norm()  # noqa: E731
        qkv = self.qkv.double().view(len(self.x), -1, self.w)
        assert near(self.qkv.view(len(self.x), -1), linear("qkv", "x"))
        at = 0
        for n in self.lens:
            q, k, v = qkv[at:at + n].split([self.hq, self.h, self.h], 1)
            each = self.hq // self.h
            s = torch.einsum("nhw,mhw->hnm", q, k.repeat_interleave(each, 1)) * self.w**-0.5
            s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -torch.inf)
            want = torch.einsum("hnm,mhw->nhw", torch.softmax(s, -1), v.repeat_interleave(each, 1))
            assert near(self.att[at:at + n], want.reshape(n, -1))
            assert (self.lse[at:at + n].double() - torch.logsumexp(s, -1).t()).abs().max() < 1e-4
            at += n
        assert near(self.hid, linear("out", "a") + self.x.double())
        assert near(self.up, gelu(linear("up", "h")))
        assert near(self.y, linear("down", "f") + self.hid.double())
        assert near(self.logits, linear("head", "y"))
        want = torch.log_softmax(self.logits.double(), -1).gather(1, self.labels.long())
        assert (self.lp.double() - want).abs().max() < 1e-4
        k, v = torch.empty(len(self.x), self.h, self.w, device="cuda"), torch.empty(len(self.x), self.h, self.w, device="cuda")
        self.cache.load(0, len(self.slots), self.slots.data_ptr(), k.data_ptr(), self.h * self.w, self.w, v.data_ptr(), self.h * self.w, self.w, stream=1)
        torch.cuda.synchronize()
        assert (k.double() - qkv[:, self.hq:self.hq + self.h]).norm() <= 0.1 * k.double().norm()  # (what four bits hold)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_a_prompts_layer(gpu, dtype, fmt):
    """Projection to answer on the caller's stream, again in a graph with other inputs, and beside itself on two streams."""
    # a stage's rounding to its type, of values of which most are near the largest; f32: sums of some 500 products
    tol = {"f32": 4e-6, "f16": 2 * 2.0**-11, "bf16": 2 * 2.0**-8}[dtype]
    layer = Layer(gpu, dtype, [200, 1, 37, 130], 512, 8, 2, 64, 1000, 300, FORMATS[fmt])
    layer.run(1)
    sync(gpu)
    layer.check(tol)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            layer.run(side.cuda_stream)
        layer.x.copy_(torch.randn_like(layer.x))
        graph.replay(), graph.replay()
    sync(gpu)
    layer.check(tol)
    want = layer.y.clone()
    other = Layer(gpu, dtype, [200, 1, 37, 130], 512, 8, 2, 64, 1000, 300, FORMATS[fmt])
    other.x.copy_(layer.x)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for one, s in zip((layer, other), streams):
            one.run(s.cuda_stream)
    sync(gpu)
    assert torch.equal(layer.y, want) and torch.equal(other.y, want)
