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


# ---- each kernel of attention at the masks, orders, places and values where it could go wrong --------------------------

def check_rows(c, dtype, group, q, counts, scale, causal, window, out, lse, leave=()):
    """Every row by its own values: 16-bit types round a weight and its product with a step or a value to 11 bits each, f32
    to 21 or more; a code's part of a value is as large as its group's span; scores and sums are f32. Sequences in `leave`
    are not looked at."""
    out, lse, at = host(out), host(lse), 0
    two = 2.0**-10 if dtype != "f32" else 2.0**-19
    off = ref = 0.0
    for s, n in enumerate(counts):
        if not n:
            continue
        r = slice(at, at + n)
        at += n
        if s in leave:
            continue
        k, v = c.k[s], c.v[s]
        seen = visible(n, c.lens[s], causal, window)
        if not c.lens[s]:
            assert not out[r].any() and (lse[r] == -np.inf).all()
            continue
        want, _, l, reach = exact(q[r], k, v, scale, seen)
        g = v.reshape(*v.shape[:-1], -1, group)
        span = np.repeat(g.max(-1) - g.min(-1), group, -1)
        _, size, _, _ = exact(q[r], k, np.abs(v) + span, scale, seen)
        none = ~np.isfinite(l)
        assert (lse[r][none] == -np.inf).all() and not out[r][none].any()
        with np.errstate(over="ignore"):
            tol = size * (two + np.expm1(2.0**-19 * reach))[..., None] + 2 * ULP[dtype] * np.abs(want) + 1e-30
        assert (np.abs(out[r] - want) <= tol).all(), (s, np.abs(out[r] - want).max())
        some = ~none
        assert (np.abs(lse[r] - l)[some] <= (2.0**-20 * (reach + 1 + np.abs(np.where(some, l, 0))))[some]).all(), s
        off, ref = off + np.sum((out[r] - want) ** 2), ref + np.sum(want**2)
    # roundings of either sign: as a whole a share of the result
    assert off <= {"f32": 1e-5, "f16": 2.0**-10, "bf16": 2.0**-8}[dtype] ** 2 * ref, (off / ref) ** 0.5


def shape_of(which):
    """Sequences, heads and most rows that reach the kernel at width 128."""
    return (4, 2, 7) if which == "few" else (40, 4, 47)


@pytest.mark.parametrize("dtype,which", BOTH)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attend_counts_its_keys(gpu, dtype, which, page):
    """All scores equal, and the values one-hot: an output is the number of seen tokens with that coordinate over the number
    of all, so one key too many or too few at either end of a mask moves it by a part of eight or more."""
    seqs, heads, rows = shape_of(which)
    width, group = 128, 32
    lens = [n for _ in range(seqs) for n in (0, 1, 46, 47, 64, 200, 333, 512)][:seqs]
    c = Cached(gpu, 40, lens, heads, width, page, group)
    assert kernels(c, dtype, rows, heads) == which
    n = max(lens)
    v = np.zeros((n, heads, width))
    v[np.arange(n), :, np.arange(n) % width] = 1.0
    rng = np.random.default_rng(1)
    cut = np.cumsum([0] + lens)
    all_v, all_k = np.concatenate([v[:m] for m in lens]), rng.normal(0, 1, (cut[-1], heads, width))
    table = c.table.cpu().numpy()
    slots = [int(table[s, j // page]) * page + j % page for s in range(seqs) for j in range(lens[s])]
    raw, kk, vv = plain.pool_of(all_k.astype(np.float32), all_v.astype(np.float32), slots, c.pages, page, group, 0xFF)
    c.pool.copy_(dev(raw))
    one = vv.max()
    q = np.zeros((rows * seqs, heads, width), np.float32)
    for causal, window in ((False, 0), (True, 0), (True, 1), (True, 31), (True, 63), (True, 64), (True, 65), (True, 300)):
        out, lse = (host(t) for t in c.attend(dtype, q, [rows] * seqs, 0.1, causal, window))
        sync(gpu)
        for s in range(seqs):
            seen = visible(rows, lens[s], causal, window)
            total = np.maximum(seen.sum(1), 1)
            per = np.zeros((rows, width))
            for j in range(lens[s]):
                per[:, j % width] += seen[:, j]
            r = slice(s * rows, (s + 1) * rows)
            want = (per * one / total[:, None])[:, None]
            assert (np.abs(out[r] - want) <= 0.1 / total[:, None, None] + 2.0**-8 * want).all(), (causal, window, s)
            with np.errstate(divide="ignore"):
                l = np.log(seen.sum(1).astype(float))[:, None]
            assert (np.abs(lse[r] - l)[seen.any(1)] <= 2.0**-19 * (1 + l[seen.any(1)])).all() and (lse[r][~seen.any(1)] == -np.inf).all()


@pytest.mark.parametrize("dtype,which", BOTH)
def test_attend_ragged_rows_on_each_kernel(gpu, dtype, which):
    seqs, heads, rows = shape_of(which)
    lens = [n for _ in range(seqs) for n in (120, 60, 0, 200)][:seqs]
    counts = [n for _ in range(seqs) for n in (rows, 0, 3, rows - 1)][:seqs]
    c = Cached(gpu, 41, lens, heads, 128, 32, 64)
    assert kernels(c, dtype, rows, 3 * heads) == which
    q = rounded(np.random.default_rng(2).normal(0, 1, (sum(counts), 3 * heads, 128)), DT[dtype][1])
    for window in (0, 33):
        out, lse = c.attend(dtype, q, counts, 0.088, causal=True, window=window, ragged=True)
        sync(gpu)
        check_rows(c, dtype, 64, q, counts, 0.088, True, window, out, lse)


@pytest.mark.parametrize("dtype,which", BOTH)
@pytest.mark.parametrize("size", [6.0, 0.5])
def test_attend_sharp_and_even_scores_on_each_kernel(gpu, dtype, which, size):
    """Scores over a span of hundreds, growing along the sequence in places (references move), and nearly even ones."""
    seqs, heads, rows = shape_of(which)
    c = Cached(gpu, 42, [333] * seqs, heads, 128, 64, 32)
    assert kernels(c, dtype, rows, heads) == which
    rng = np.random.default_rng(3)
    k, v = rng.normal(0, 1, (2, 333, heads, 128))
    k *= np.where(np.arange(333) % 100 > 70, np.arange(333) / 100.0, 0.3)[:, None, None]
    set_tokens(c, k, v, 64, 32)
    q = rounded(rng.normal(0, size, (rows * seqs, heads, 128)), DT[dtype][1])
    out, lse = c.attend(dtype, q, [rows] * seqs, -0.0884, causal=True)
    sync(gpu)
    check_rows(c, dtype, 32, q, [rows] * seqs, -0.0884, True, 0, out, lse)


@pytest.mark.parametrize("dtype,which", BOTH)
def test_attend_scores_up_to_two_to_the_23(gpu, dtype, which):
    """Scores as large as f32 still resolves: the largest takes all."""
    seqs, heads, rows = shape_of(which)
    c = Cached(gpu, 43, [200] * seqs, heads, 128, 64, 32)
    assert kernels(c, dtype, rows, heads) == which
    q = rounded(np.random.default_rng(3).normal(0, 30, (rows * seqs, heads, 128)), DT[dtype][1])
    scale = 2.0**23 / 3e3
    out, lse = (host(t) for t in c.attend(dtype, q, [rows] * seqs, scale))
    sync(gpu)
    for s in range(0, seqs, 5):
        for h in range(heads):
            r = slice(s * rows, (s + 1) * rows)
            x = q[r, h].astype(np.float64) @ c.k[s][:, h].T * scale
            order = np.sort(x, 1)
            sure = order[:, -1] - order[:, -2] > 2.0**-18 * np.abs(x).max()  # of scores nearer than they round either may win
            best, v = x.argmax(1), c.v[s][:, h]
            assert sure.sum() > rows / 2 and np.abs(x).max() < 2.0**24
            assert (np.abs(lse[r, h] - order[:, -1]) <= 2.0**-19 * np.abs(q[r, h]).astype(np.float64) @ np.abs(c.k[s][:, h]).T.max(1) * scale).all()
            assert (np.abs(out[r, h] - v[best]) <= 2.0**-9 * (4 + np.abs(v[best])) + 2 * ULP[dtype] * np.abs(v[best]))[sure].all()


@pytest.mark.parametrize("dtype,which", BOTH)
def test_attend_values_of_many_sizes_on_each_kernel(gpu, dtype, which):
    """Tokens whose values go from 1e-4 to 1e4, keys over three powers of ten."""
    seqs, heads, rows = shape_of(which)
    c = Cached(gpu, 44, [400] * seqs, heads, 128, 16, 32)
    assert kernels(c, dtype, rows, heads) == which
    rng = np.random.default_rng(4)
    k = rng.normal(0, 1, (400, heads, 128)) * 10.0 ** rng.uniform(-3, 0, (400, 1, 1))
    v = rng.normal(0, 1, (400, heads, 128)) * 10.0 ** rng.uniform(-4, 4, (400, 1, 1))
    set_tokens(c, k, v, 16, 32)
    q = rounded(rng.normal(0, 1, (rows * seqs, heads, 128)), DT[dtype][1])
    out, lse = c.attend(dtype, q, [rows] * seqs, 0.088, causal=True)
    sync(gpu)
    check_rows(c, dtype, 32, q, [rows] * seqs, 0.088, True, 0, out, lse)


@pytest.mark.parametrize("dtype,which", BOTH)
@pytest.mark.parametrize("width", [64, 128])
def test_attend_strides_and_orders_on_each_kernel(gpu, dtype, which, width):
    """Queries and outputs by row and by head, at odd places of wider buffers; the same call again gives the same bits, and
    nothing beside the outputs is written."""
    if dtype == "f32" and width == 64:
        width = 128
    code, tt = DT[dtype]
    seqs, heads, rows = shape_of(which)
    c = Cached(gpu, 45, [150] * seqs, heads, width, 64, 32)
    assert kernels(c, dtype, rows, heads) == which
    q = rounded(np.random.default_rng(3).normal(0, 1, (rows * seqs, heads, width)), tt)
    n, w = rows * seqs, width
    batch = c.cache.batch(seqs, rows, 150, c.lens_dev.data_ptr(), c.table.data_ptr(), c.stride)
    work = torch.zeros(max(16, c.cache.attend_workspace(batch, heads, code)), dtype=torch.uint8, device="cuda")
    for row, head, lead in ((heads * (w + 3), w + 3, 1), (w, n * w, 0), (w + 1, n * (w + 1), 5), (heads * w + 8, w, 8)):
        total = (n - 1) * row + (heads - 1) * head + w + lead + 9
        wide, outs = torch.full((total,), 3e4, dtype=tt, device="cuda"), []
        torch.as_strided(wide, (n, heads, w), (row, head, 1), lead).copy_(dev(q, tt))
        for _ in range(2):
            o = torch.full((total,), 9.0, dtype=tt, device="cuda")
            at = lead * o.element_size()
            c.cache.attend(batch, code, heads, wide.data_ptr() + at, row, head, o.data_ptr() + at, row, head, 0.1,
                           work=work.data_ptr(), work_bytes=work.numel(), stream=1)
            sync(gpu)
            outs.append(o)
        assert torch.equal(outs[0], outs[1])
        got = torch.as_strided(outs[0], (n, heads, w), (row, head, 1), lead).clone()
        torch.as_strided(outs[0], (n, heads, w), (row, head, 1), lead).fill_(9.0)
        assert bool((outs[0] == 9).all())
        if lead == 1:
            _, lse = c.attend(dtype, q, [rows] * seqs, 0.1)
            sync(gpu)
            check_rows(c, dtype, 32, q, [rows] * seqs, 0.1, False, 0, got, lse)
            first = got
        assert torch.equal(got, first)


@pytest.mark.parametrize("dtype,which", BOTH)
def test_attend_past_four_gigabytes_on_each_kernel(gpu, dtype, which):
    seqs, heads, rows = shape_of(which)
    page, group = 64, 32
    c = Cached(gpu, 46, [150] * seqs, heads, 128, page, group, extra=0)
    assert kernels(c, dtype, rows, heads) == which
    size = tcu.Kv4Cache.page_bytes(heads, 128, page, group)
    pages = (9 << 30) // 2 // size + c.pages
    pool = torch.empty(pages, size, dtype=torch.uint8, device="cuda")
    pool[-c.pages:] = c.pool
    c.table[c.table >= 0] += pages - c.pages
    c.cache = tcu.Kv4Cache(gpu, pool.data_ptr(), pages, heads=heads, width=128, page=page, group=group)
    q = rounded(np.random.default_rng(3).normal(0, 1, (rows * seqs, heads, 128)), DT[dtype][1])
    out, lse = c.attend(dtype, q, [rows] * seqs, 0.09, causal=True)
    sync(gpu)
    check_rows(c, dtype, group, q, [rows] * seqs, 0.09, True, 0, out, lse)


@pytest.mark.parametrize("dtype,which", BOTH)
def test_attend_reports_indexes_on_each_kernel(gpu, dtype, which):
    """A page, length or start outside its range is reported once, other sequences' rows are what they are."""
    seqs, heads, rows = shape_of(which)

    def call(change, bad, ragged=False):
        c = Cached(gpu, 47, [100, 70] * (seqs // 2), heads, 128, 32, 64)
        assert kernels(c, dtype, rows, heads) == which
        q = rounded(np.random.default_rng(3).normal(0, 1, (rows * seqs, heads, 128)), DT[dtype][1])
        starts = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * rows
        change(c, starts)
        if ragged:
            code = DT[dtype][0]
            qd, out = dev(q, DT[dtype][1]), torch.full(q.shape, 9.0, dtype=DT[dtype][1], device="cuda")
            lse = torch.full(q.shape[:2], 9.0, device="cuda")
            b = c.cache.batch(seqs, rows, 101, c.lens_dev.data_ptr(), c.table.data_ptr(), c.stride, starts.data_ptr(), rows * seqs)
            work = torch.zeros(max(16, c.cache.attend_workspace(b, heads, code)), dtype=torch.uint8, device="cuda")
            c.cache.attend(b, code, heads, qd.data_ptr(), heads * 128, 128, out.data_ptr(), heads * 128, 128, 0.1, causal=True,
                           lse=lse.data_ptr(), work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        else:
            out, lse = c.attend(dtype, q, [rows] * seqs, 0.1, causal=True)
        torch.cuda.synchronize()
        with pytest.raises(tcu.TcuError, match="outside its range"):
            gpu.sync()
        gpu.sync()
        check_rows(c, dtype, 64, q, [rows] * seqs, 0.1, True, 0, out, lse, bad)

    call(lambda c, st: c.table[0, 1].fill_(c.pages), [0])
    call(lambda c, st: c.table[1, 0].fill_(-5), [1])
    call(lambda c, st: c.lens_dev[0].fill_(101), [0])
    call(lambda c, st: c.lens_dev[1].fill_(-1), [1])
    call(lambda c, st: st[seqs].fill_(rows * seqs + 1), [seqs - 1], True)
    call(lambda c, st: st[0].fill_(-1), [0], True)


def test_working_memory_serves_every_kernel_in_turn(gpu):
    """One block for calls of every kernel and type, whose units are cut differently, in turn."""
    shapes = [("bf16", [5000], 1, 1, [1]), ("f32", [4000], 4, 8, [1100]), ("f16", [4000], 4, 8, [1100]), ("f32", [3000], 2, 8, [2]),
              ("bf16", [300] * 40, 4, 4, [47] * 40), ("f32", [300] * 40, 4, 4, [47] * 40), ("f16", [2000], 1, 8, [3])]
    calls = []
    for i, (dtype, lens, heads, hq, counts) in enumerate(shapes):
        c = Cached(gpu, i, lens, heads, 128, 64, 32)
        q = rounded(np.random.default_rng(i).normal(0, 1, (sum(counts), hq, 128)), DT[dtype][1])
        calls.append((c, dtype, q, counts, c.attend(dtype, q, counts, 0.1, causal=True)))
    work = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    for turn in range(2):
        for c, dtype, q, counts, want in calls if turn else reversed(calls):
            got = c.attend(dtype, q, counts, 0.1, causal=True, work=work)
            sync(gpu)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- streams and graphs ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,seqs", [(1, 3), (47, 40)])
def test_every_operator_in_a_graph(gpu, dtype, rows, seqs):
    """Store, load, attention, linear layers and log-probabilities captured on a stream of their own, replayed over new
    inputs: the bits of the same calls without a graph."""
    code, tt = DT[dtype]
    heads, width, page, group, n = 4, 128, 64, 32, 90
    pages = seqs * 2
    pool = torch.zeros(pages * tcu.Kv4Cache.page_bytes(heads, width, page, group), dtype=torch.uint8, device="cuda")
    cache = tcu.Kv4Cache(gpu, pool.data_ptr(), pages, heads=heads, width=width, page=page, group=group)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(seqs, 2)
    lens = torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    slots = (torch.arange(seqs, device="cuda")[:, None] * 2 * page + torch.arange(n, device="cuda")).flatten()
    batch = cache.batch(seqs, rows, n, lens.data_ptr(), table.data_ptr(), 2)
    d, r = heads * width, rows * seqs
    weight = torch.empty(700, d, dtype=tt, device="cuda")
    codes = torch.empty(tcu.W4.code_bytes(700, d), dtype=torch.uint8, device="cuda")
    scales = torch.empty(tcu.W4.scale_bytes(700, d, group), dtype=torch.uint8, device="cuda")
    w4 = tcu.W4(gpu, 700, d, group, codes.data_ptr(), scales.data_ptr())
    k, v = (torch.empty(seqs * n, d, dtype=tt, device="cuda") for _ in range(2))
    q = torch.empty(r, d, dtype=tt, device="cuda")
    labels = (torch.arange(r, dtype=torch.int32, device="cuda") * 7 % 700).contiguous()
    outs = dict(k=torch.empty_like(k), v=torch.empty_like(v), o=torch.empty_like(q), lse=torch.empty(r, heads, device="cuda"),
                y=torch.empty(r, 700, dtype=tt, device="cuda"), y8=torch.empty(1, 700, dtype=tt, device="cuda"), lp=torch.empty(r, device="cuda"),
                tv=torch.empty(r, 3, device="cuda"), ti=torch.empty(r, 3, dtype=torch.int32, device="cuda"))
    work = torch.zeros(max(cache.attend_workspace(batch, heads, code), w4.linear_workspace(r, code)), dtype=torch.uint8, device="cuda")

    def step(stream):
        w4.pack(code, weight.data_ptr(), d, stream=stream)
        cache.store(code, seqs * n, slots.data_ptr(), k.data_ptr(), d, width, v.data_ptr(), d, width, stream=stream)
        cache.load(code, seqs * n, slots.data_ptr(), outs["k"].data_ptr(), d, width, outs["v"].data_ptr(), d, width, stream=stream)
        cache.attend(batch, code, heads, q.data_ptr(), d, width, outs["o"].data_ptr(), d, width, 0.1, causal=True, lse=outs["lse"].data_ptr(),
                     work=work.data_ptr(), work_bytes=work.numel(), stream=stream)
        for m, y in ((r, "y"), (1, "y8")):
            w4.linear(code, m, outs["o"].data_ptr(), d, outs[y].data_ptr(), 700, act=1, work=work.data_ptr(), work_bytes=work.numel(), stream=stream)
        gpu.label_logprobs(code, outs["y"].data_ptr(), r, 700, 700, labels.data_ptr(), 1, outs["lp"].data_ptr(), top=3,
                           top_values=outs["tv"].data_ptr(), top_ids=outs["ti"].data_ptr(), stream=stream)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for seed in (1, 2):
        gen = torch.Generator("cuda").manual_seed(seed)
        for x in (weight, k, v, q):
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        for x in outs.values():
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = {name: x.clone() for name, x in outs.items()}
        for x in outs.values():
            x.zero_()
        step(1)
        sync(gpu)
        for name, x in outs.items():
            assert torch.equal(x, got[name]), name
        assert float(got["lp"].max()) < 0 and bool(torch.isfinite(got["lse"]).all()) and float(got["o"].float().abs().max()) > 0.01


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,length,heads,q_heads,window", [(2048, 7100, 8, 8, 1000), (1300, 1300, 4, 12, 100), (300, 5000, 16, 32, 0)])
def test_attend_long_prompts(gpu, dtype, rows, length, heads, q_heads, window):
    """Units cut into parts that several blocks share, with and without a window, causal."""
    c = Cached(gpu, 48, [length], heads, 128, 64, 32)
    assert kernels(c, dtype, rows, q_heads) == "many"
    q = rounded(np.random.default_rng(7).normal(0, 1, (rows, q_heads, 128)), DT[dtype][1])
    out, lse = c.attend(dtype, q, [rows], 0.088, causal=True, window=window)
    again, _ = c.attend(dtype, q, [rows], 0.088, causal=True, window=window)
    sync(gpu)
    assert torch.equal(out, again)
    check_many(c, dtype, q, rows, 0.088, True, window, out, lse)
    last = slice(rows - 64, rows)  # and by each row's own values
    check_rows(c, dtype, 32, q[last], [64], 0.088, True, window, out[last], lse[last])


@pytest.mark.parametrize("rows,seqs,length,heads,q_heads,width,group,which", [
    (1, 17, 20000, 1, 4, 32, 32, "few"), (1, 60, 9000, 2, 4, 128, 128, "few"), (40, 60, 3000, 2, 2, 256, 64, "few"), (1, 1, 20000, 1, 1, 128, 32, "few"),
    (300, 20, 3000, 2, 2, 128, 64, "many")])
def test_attend_f32_sums_over_long_sequences(gpu, rows, seqs, length, heads, q_heads, width, group, which):
    """Thousands of values of either sign: every weighted value is good to 2^-20, and a sum over the steps rounds to nearest, so
    that its errors, of either sign too, stay below a few 2^-24 of the values' root of squares."""
    page = 256
    c = Cached(gpu, 49, [16], heads, width, page, group, extra=length // page + 1)
    rng = np.random.default_rng(7)
    k, v = rng.normal(0, 1, (2, length, heads, width))
    order = rng.permutation(c.pages)[:-(-length // page)]
    at = order[np.arange(length) // page] * page + np.arange(length) % page
    raw, kk, vv = plain.pool_of(k.astype(np.float32), v.astype(np.float32), at, c.pages, page, group, 0xFF)
    c.pool.copy_(dev(raw))
    c.stride, c.lens = len(order), [length] * seqs
    c.table = dev(np.tile(order.astype(np.int32), (seqs, 1)))
    c.lens_dev = torch.full((seqs,), length, dtype=torch.int32, device="cuda")
    assert width < 128 or kernels(c, "f32", rows, q_heads) == which
    q = rng.normal(0, 1, (rows * seqs, q_heads, width)).astype(np.float32)
    out, lse = c.attend("f32", q, [rows] * seqs, 0.5 / np.sqrt(width))
    sync(gpu)
    worst = 0.0
    for h in range(q_heads):
        x, a, b = (torch.from_numpy(t).cuda().double() for t in (q[:, h], kk[:, h * heads // q_heads], vv[:, h * heads // q_heads]))
        s = x @ a.T * (0.5 / np.sqrt(width))
        want = torch.softmax(s, -1) @ b
        worst = max(worst, float((out[:, h].double() - want).norm() / want.norm()))
        assert float((lse[:, h].double() - torch.logsumexp(s, -1)).abs().max()) <= 2e-5
    # a weight's error is that of its score (2^-20 of a sum of magnitudes of about 5, of either sign: 1e-6 and less as a
    # whole) beside 2^-21 of each product, and ten roundings of a sum
    assert worst <= 2e-6, worst


@pytest.mark.parametrize("rows,seqs,which", [(2, 30, "few"), (60, 40, "many")])
def test_attend_f16_is_near_the_result_rounded_once(gpu, rows, seqs, which):
    """Values of either sign, one rounding to 11 bits (of weights times steps, or of values) beside the result's own: together
    the root of two of the latter, so below 1.5 of it."""
    n, heads = 1500, 4
    c = Cached(gpu, 50, [n], heads, 128, 64, 32)
    rng = np.random.default_rng(8)
    k, v = rng.normal(0, 1, (2, n, heads, 128))
    set_tokens(c, k, v, 64, 32)
    c.lens = [n] * seqs
    c.table, c.lens_dev = c.table.repeat(seqs, 1).contiguous(), c.lens_dev.repeat(seqs)
    assert kernels(c, "f16", rows, heads) == which
    q = rounded(rng.normal(0, 1, (rows * seqs, heads, 128)), torch.float16)
    out, _ = c.attend("f16", q, [rows] * seqs, 0.088)
    sync(gpu)
    want, _, _, _ = exact(q, c.k[0], c.v[0], 0.088, np.ones((len(q), n), bool))
    once = np.linalg.norm(want.astype(np.float16).astype(np.float64) - want)
    assert np.linalg.norm(host(out) - want) <= 1.5 * once, np.linalg.norm(host(out) - want) / once
