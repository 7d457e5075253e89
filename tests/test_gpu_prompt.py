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
