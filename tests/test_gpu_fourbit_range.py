"""The four-bit operators where types, sizes and values reach their ends, on the GPU against plain numpy or torch in 64 bits:
very different magnitudes side by side, masks to the key, odd places and orders, working memory that all of them share,
graph capture. Attention is tried on each of its kernels; `kernels` asserts which one a call takes."""
import numpy as np
import pytest

import fourbit_plain as plain
import test_gpu_fourbit as base
from conftest import tcu
from test_gpu_fourbit import DT, ULP, Cached, check_many, dev, host, rounded, sync, weights

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
gpu = base.gpu


def kernels(c, dtype, rows, q_heads):
    """Which attention kernels the call takes, by the working memory it asks for: "few" or "many" rows. (Of f32 at widths up
    to 64 both ask for the same.)"""
    assert dtype != "f32" or c.width > 64
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    batch = c.cache.batch(len(c.lens), rows, max(c.lens + [1]), c.lens_dev.data_ptr(), c.table.data_ptr(), c.stride)
    many = 4 * (2048 + 2 * sms * (128 if dtype == "f32" else 256) * (c.width + 2))
    return "many" if c.cache.attend_workspace(batch, q_heads, DT[dtype][0]) == many else "few"


def set_tokens(c, k, v, page, group):
    """The same keys k and values v [tokens][heads][width] in every sequence of c."""
    n, seqs = k.shape[0], len(c.lens)
    table = c.table.cpu().numpy()
    slots = [int(table[s, j // page]) * page + j % page for s in range(seqs) for j in range(n)]
    tile = lambda x: np.tile(np.asarray(x, np.float32), (seqs, 1, 1))  # noqa: E731
    raw, kk, vv = plain.pool_of(tile(k), tile(v), slots, c.pages, page, group, 0xFF)
    c.pool.copy_(dev(raw))
    c.k, c.v = [kk[:n]] * seqs, [vv[:n]] * seqs


def exact(q, k, v, scale, seen):
    """Rows q [n][q_heads][width] against keys and values [length][heads][width] in 64 bits, `seen` [n][length]: the outputs,
    the sums of |p v| behind them, lse, and the scores' largest sums of magnitudes."""
    each = q.shape[1] // k.shape[1]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    lse, reach = np.full(q.shape[:2], -np.inf), np.zeros(q.shape[:2])
    some = seen.any(1)
    for h in range(q.shape[1]):
        x, kk, vv = q[:, h].astype(np.float64), k[:, h // each], v[:, h // each]
        s = np.where(seen, x @ kk.T * scale, -np.inf)
        m = np.where(some, s.max(1), 0.0)
        p = np.exp(s - m[:, None])
        total = np.where(some, p.sum(1), 1.0)
        out[:, h], size[:, h] = p @ vv / total[:, None], p @ np.abs(vv) / total[:, None]
        lse[some, h] = (m + np.log(total))[some]
        reach[:, h] = np.where(seen, np.abs(x) @ np.abs(kk).T * abs(scale), 0.0).max(1)
    return out, size, lse, reach


def visible(n, length, causal, window):
    i, j = np.arange(n)[:, None], np.arange(length)[None]
    seen = np.ones((n, length), bool)
    if causal:
        seen &= j <= length - n + i
    if window:
        seen &= j > length - n + i - window
    return seen


@pytest.mark.parametrize("dtype,width,heads,q_heads,rows,length,which", [
    ("bf16", 64, 1, 1, 1, 5000, "few"), ("f32", 128, 1, 4, 2, 3000, "few"), ("bf16", 128, 4, 8, 1100, 4000, "many"),
    ("f32", 128, 4, 8, 1100, 4000, "many")])
def test_working_memory_serves_every_operator(gpu, dtype, width, heads, q_heads, rows, length, which):
    """One block of working memory for attention whose units are cut into parts and linear layers of more than 8 rows, in
    turn: the same bits as with a block of their own."""
    code, tt = DT[dtype]
    c = Cached(gpu, 30, [length], heads, width, 64, 32)
    assert kernels(c, dtype, rows, q_heads) == which
    rng = np.random.default_rng(1)
    q = rounded(rng.normal(0, 1, (rows, q_heads, width)), tt)
    w4, keep, _ = weights(rng, gpu, 300, 1000, 32, dtype)
    x = dev(rng.normal(0, 1, (20, 1000)).astype(np.float32), tt)
    shared = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")

    def linear(work):
        y = torch.full((20, 300), 9.0, dtype=tt, device="cuda")
        w4.linear(code, 20, x.data_ptr(), 1000, y.data_ptr(), 300, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        return y

    own = torch.zeros(w4.linear_workspace(20, code), dtype=torch.uint8, device="cuda")
    want_y, (want, want_lse) = linear(own), c.attend(dtype, q, [rows], 0.125, causal=True)
    for _ in range(3):
        y, (out, lse) = linear(shared), c.attend(dtype, q, [rows], 0.125, causal=True, work=shared)
        sync(gpu)
        assert torch.equal(y, want_y) and torch.equal(out, want) and torch.equal(lse, want_lse)
    c.check(dtype, q[-3:], [min(rows, 3)], 0.125, True, 0, want[-3:], want_lse[-3:])


# sequences and heads that reach each kernel with a few dozen rows (f32 has its own for many rows)
BOTH = [("f32", "few"), ("f16", "few"), ("bf16", "few"), ("f32", "many"), ("f16", "many"), ("bf16", "many")]


@pytest.mark.parametrize("dtype,which", BOTH)
def test_a_window_wider_than_any_sequence_hides_nothing(gpu, dtype, which):
    """Windows up to the largest number, where a sequence has fewer tokens than rows."""
    lens, rows = ([5, 1, 40, 0], 10) if which == "few" else ([5, 1, 40, 0] * 10, 45)
    c = Cached(gpu, 31, lens, 1 if which == "few" else 4, 128, 32, 64)
    assert kernels(c, dtype, rows, c.heads) == which
    q = rounded(np.random.default_rng(2).normal(0, 1, (rows * len(lens), c.heads, 128)), DT[dtype][1])
    want, want_lse = c.attend(dtype, q, [rows] * len(lens), 0.1, causal=True)
    for window in (41, 1 << 20, 2**31 - 1):
        out, lse = c.attend(dtype, q, [rows] * len(lens), 0.1, causal=True, window=window)
        sync(gpu)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), window
    check_many(c, dtype, q, rows, 0.1, True, 0, want, want_lse)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("width,group,rows,seqs,which", [(128, 32, 2, 5, "few"), (128, 32, 50, 10, "many"), (64, 64, 50, 10, "many"),
                                                         (32, 32, 50, 10, "many")])
def test_attend_lse_keeps_32_bits(gpu, dtype, width, group, rows, seqs, which):
    """The log-sum-exp is f32 whatever the queries' type: keys of 21 bits or more and sums in f32, so a score is off by at
    most 2^-20 of its sum of magnitudes, and log-sum-exp rounds a few times."""
    n = 300
    c = Cached(gpu, 32, [n] * seqs, 4, width, 64, group, spread=1.0)
    assert kernels(c, dtype, rows, 8) == which
    q = rounded(np.random.default_rng(3).normal(0, 1, (rows * seqs, 8, width)), DT[dtype][1])
    scale = 1 / np.sqrt(width)
    out, lse = c.attend(dtype, q, [rows] * seqs, scale, causal=True)
    sync(gpu)
    for s in range(seqs):
        r = slice(s * rows, (s + 1) * rows)
        _, _, want, reach = exact(q[r], c.k[s], c.v[s], scale, visible(rows, n, True, 0))
        assert (np.abs(host(lse)[r] - want) <= 2.0**-20 * (reach + 1 + np.abs(want))).all()
        # and as a whole: roundings of either sign, here held to a quarter of the worst
        assert np.linalg.norm(host(lse)[r] - want) <= 2.0**-22 * np.linalg.norm(reach + 1 + np.abs(want))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,which", [(3, "few"), (60, "many")])
@pytest.mark.parametrize("big", [256.0, 4096.0, 60000.0])
def test_attend_small_values_beside_a_large_one(gpu, dtype, rows, which, big):
    """Values of size 1 beside large ones that a row does not see, or that lie in another group of its tokens' coordinates,
    late in the sequence and early: as near as the type rounds, by each row's own values."""
    n, seqs, heads, width, page, group = 200, 10, 4, 64, 64, 32
    c = Cached(gpu, 33, [n] * seqs, heads, width, page, group)
    assert kernels(c, dtype, rows, heads) == which
    rng = np.random.default_rng(5)
    k, v = rng.normal(0, 1, (2, n, heads, width))
    v[n - 1] = big * rng.choice([-1, 1], (heads, width))       # seen by the last row only
    for token in (10, n - rows - 5):
        v[token, :, group:] = -big
    set_tokens(c, k, v, page, group)
    q = rounded(rng.normal(0, 1, (rows * seqs, heads, width)), DT[dtype][1])
    scale = 0.25 / np.sqrt(width)
    out, _ = c.attend(dtype, q, [rows] * seqs, scale, causal=True)
    sync(gpu)
    seen = visible(rows, n, True, 0)
    for s in range(0, seqs, 3):
        r = slice(s * rows, s * rows + rows - 1)
        want, size, _, reach = exact(q[r], c.k[s], c.v[s], scale, seen[:-1])
        got, want, size = host(out)[r, :, :group], want[..., :group], size[..., :group]
        # a weight and a value round to 11 bits each, scores as in f32; values that the large one pushes below f16's normal
        # numbers by 17 halves of its smallest step, which is 2^-37 of the largest value or less
        tol = size * (2.0**-10 + np.expm1(2.0**-19 * reach))[..., None] + 2 * ULP[dtype] * np.abs(want) + 2.0**-33 * big
        assert (np.abs(got - want) <= tol).all(), (s, np.abs(got - want).max())
        off = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert off <= 2.0**-10 + ULP[dtype] + 2.0**-33 * big, off


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,seqs,which", [(1, 3, "few"), (1, 100, "few"), (12, 40, "few"), (50, 40, "many")])
@pytest.mark.parametrize("size", [1e-3, 1e-5, 4e-6])
def test_attend_values_of_small_steps(gpu, dtype, rows, seqs, which, size):
    """Values far below 1, down to steps among f16's smallest, under uneven weights: a share of their own size. (Many
    sequences, here on the same pages, let a warp see many keys.)"""
    n, heads, width, page, group = 4000, 2, 128, 64, 32
    c = Cached(gpu, 34, [n], heads, width, page, group)
    rng = np.random.default_rng(6)
    k, v = rng.normal(0, 1, (2, n, heads, width))
    set_tokens(c, k, v * size, page, group)
    c.lens = [n] * seqs
    c.table, c.lens_dev = c.table.repeat(seqs, 1).contiguous(), c.lens_dev.repeat(seqs)
    assert kernels(c, dtype, rows, heads) == which
    q = rounded(rng.normal(0, 2, (rows * seqs, heads, width)), DT[dtype][1])
    out, _ = c.attend(dtype, q, [rows] * seqs, 1 / np.sqrt(width))
    sync(gpu)
    want, _, _, _ = exact(q, c.k[0], c.v[0], 1 / np.sqrt(width), np.ones((len(q), n), bool))
    off = np.linalg.norm(host(out) - want) / np.linalg.norm(want)
    # 16-bit types: a weight rounds to 11 bits, its product with the step or the value again, keys to 21 or more; f16 results
    # below its normal numbers by half of 2^-24 besides. f32: 2^-20 each, sums of some ten steps
    floor = 2.0**-25 * np.sqrt(want.size) / np.linalg.norm(want) if dtype == "f16" else 0.0
    assert off <= {"f32": 1e-5, "f16": 2.0**-10 + 2.0**-11, "bf16": 2.0**-8}[dtype] + floor, off


@pytest.mark.parametrize("dtype,which", BOTH)
def test_attend_scale_of_nothing(gpu, dtype, which):
    """A scale of 0, or one that leaves scores of nothing, gives every seen key the same weight, whatever the queries' size."""
    lens, rows = ([70, 9], 3) if which == "few" else ([70, 9] * 20, 45)
    c = Cached(gpu, 35, lens, 1 if which == "few" else 4, 128, 32, 64)
    assert kernels(c, dtype, rows, c.heads) == which
    q = np.random.default_rng(2).normal(0, 1, (rows * len(lens), c.heads, 128))
    sizes = [1.0, 2.0**-24] if dtype == "f16" else [1.0, 2.0**-40, 2.0**-90, 2.0**-124]
    for size in sizes:
        for scale in (0.0, 1e-30, -1e-38):
            x = rounded(q * size, DT[dtype][1])
            out, lse = c.attend(dtype, x, [rows] * len(lens), scale, causal=True)
            sync(gpu)
            check_many(c, dtype, x, rows, scale, True, 0, out, lse)


@pytest.mark.parametrize("temperature", [1e-45, 1e-39, 3e-39, 1e38, 1e60, float("inf"), -1.0])
def test_logprobs_refuse_a_temperature_beyond_f32(gpu, temperature):
    """Temperatures whose reciprocal, or its product with log2 e, 32 bits do not hold."""
    t = torch.zeros(64, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(tcu.TcuError, match="temperature"):
        gpu.label_logprobs(0, t.data_ptr(), 1, 4, 4, i.data_ptr(), 1, t.data_ptr() + 64, temperature=temperature, stream=1)


@pytest.mark.parametrize("temperature", [1e-37, 1e-20, 1e20, 1e37])
@pytest.mark.parametrize("classes", [7, 700])
def test_logprobs_of_extreme_temperatures(gpu, classes, temperature):
    """The largest alone where it is cold, every class that is not masked alike where it is hot."""
    x = np.random.default_rng(3).normal(0, 3, (3, classes)).astype(np.float32)
    x[0, ::3] = -np.inf
    x[1, 1:] = -np.inf
    labels = np.tile(np.array([[1, 0, 2]]), (3, 1))
    out, ent, tv, ti = base.logprobs(gpu, "f32", x, labels, 3, temperature)
    gpu.sync()
    for r in range(3):
        with np.errstate(over="ignore"):
            o, e, v, i = plain.logprobs(x[r], labels[r], 3, temperature)
            o, v = (np.where(np.abs(a) > np.finfo(np.float32).max, -np.inf, a) for a in (o, v))
        assert np.array_equal(ti[r], i)
        for got, want in ((out[r], o), (tv[r], v), (ent[r:r + 1], np.array([e]))):
            fin = np.isfinite(want)
            assert np.array_equal(got[~fin], want[~fin])
            assert (np.abs(got - np.where(fin, want, 0))[fin] <= (2.0**-20 * (1 + np.abs(want)))[fin]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 5, 20])
@pytest.mark.parametrize("size", [2.0**118, 2.0**102, 2.0**-100, 2.0**-118])
def test_linear_of_very_large_and_small_inputs(gpu, dtype, rows, size):
    """Inputs near the ends of the type whose outputs it holds."""
    code, tt = DT[dtype]
    rng = np.random.default_rng(rows)
    n, k = 70, 300
    w4, keep, w = weights(rng, gpu, n, k, 64, dtype)
    x = rounded(rng.normal(0, 1, (rows, k)) * size, tt)
    xd, yd = dev(x, tt), torch.full((rows, n), 9.0, dtype=tt, device="cuda")
    work = torch.zeros(max(16, w4.linear_workspace(rows, code)), dtype=torch.uint8, device="cuda")
    w4.linear(code, rows, xd.data_ptr(), k, yd.data_ptr(), n, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    y = x.astype(np.float64) @ w.T
    tol = 2.0**-20 * (np.abs(x.astype(np.float64)) @ np.abs(w).T) + 2 * ULP[dtype] * np.abs(y)
    assert (np.abs(yd.double().cpu().numpy() - y) <= tol).all()


@pytest.mark.parametrize("dtype,which", [("f32", "few"), ("bf16", "few"), ("f32", "many"), ("bf16", "many")])
@pytest.mark.parametrize("size", [2.0**118, 2.0**-118])
def test_attend_queries_of_very_large_and_small_size(gpu, dtype, which, size):
    """Queries near the ends of the type with a scale that brings their scores back."""
    lens, rows = ([70, 9], 3) if which == "few" else ([70, 9] * 20, 45)
    c = Cached(gpu, 36, lens, 1 if which == "few" else 4, 128, 32, 64)
    assert kernels(c, dtype, rows, c.heads) == which
    q = rounded(np.random.default_rng(2).normal(0, 1, (rows * len(lens), c.heads, 128)) * size, DT[dtype][1])
    scale = float(np.float32(0.09 / size))
    out, lse = c.attend(dtype, q, [rows] * len(lens), scale, causal=True)
    sync(gpu)
    check_many(c, dtype, q, rows, scale, True, 0, out, lse)
