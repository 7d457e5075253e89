"""A prompt's operators where scores, values and lengths reach their ends, on the GPU against plain numpy or torch in 64 bits."""
import numpy as np
import pytest

import prompt_plain as plain
import test_gpu_prompt as base
from conftest import tcu
from test_gpu_prompt import DT, ULP, dev, host, rounded, sync

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
gpu = base.gpu

LN2 = float(np.float32(np.log(2)))  # times log2(e) in f32 this is 1: scores that are whole numbers are exact in every kernel


def attend(gpu, dtype, q, k, v, scale, causal=False, window=0, q_lens=None, k_lens=None):
    """q [rows][q_heads][width], k and v [keys][heads][width] (f64, or tensors on the GPU): outputs and log-sum-exp as f64 arrays."""
    code, tt = DT[dtype]
    qd, kd, vd = (dev(x, tt) if isinstance(x, np.ndarray) else x for x in (q, k, v))
    q_lens, k_lens = q_lens or [qd.shape[0]], k_lens or [kd.shape[0]]
    starts = lambda lens: dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))  # noqa: E731
    qs, ks = starts(q_lens), starts(k_lens)
    hq, h, w = qd.shape[1], kd.shape[1], qd.shape[2]
    p = tcu.Packed(gpu, len(q_lens), qd.shape[0], kd.shape[0], max(q_lens), max(k_lens), qs.data_ptr(), ks.data_ptr())
    work = torch.zeros(p.attend_workspace(code, hq, h, w), dtype=torch.uint8, device="cuda")
    out, lse = torch.full_like(qd, 9.0), torch.full((qd.shape[0], hq), 9.0, device="cuda")
    p.attend(code, hq, h, w, qd.data_ptr(), hq * w, w, kd.data_ptr(), h * w, w, vd.data_ptr(), h * w, w, out.data_ptr(), hq * w, w, scale,
             causal=causal, window=window, lse=lse.data_ptr(), work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    assert not work[:8192].any()  # left as the next call needs them
    return host(out), host(lse)


# ---- large scores ---------------------------------------------------------------------------------------------------

TOP = 2**20
LARGE = [  # keys, {key: score}, all others' score
    (130, {5: TOP - 6, 70: TOP + 1}, 0), (130, {5: TOP - 6, 70: TOP - 4, 129: TOP + 1}, 0), (130, {70: TOP - 2, 5: TOP + 1}, 0),
    (130, {5: -TOP - 4, 70: -TOP + 1}, -2**22), (130, {5: -TOP - 4, 70: -TOP + 6}, -2**22), (130, {5: 2 * TOP, 70: 2 * TOP - 1}, 0),
    (130, {5: 8 * TOP, 70: 8 * TOP - 2}, 8 * TOP - 2**13), (2000, {5: TOP - 6, 1900: TOP + 1}, 0), (2000, {5: TOP + 1, 1900: TOP - 2}, 0),
    (2000, {5: -TOP - 4, 1900: -TOP + 1}, -2**22), (130, {5: 16 * TOP, 129: 16 * TOP - 4}, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [5, 100], ids=["few", "many"])
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("keys,scores,rest", LARGE, ids=lambda x: str(x).replace(" ", "") if not isinstance(x, int) else str(x))
def test_attend_large_scores(gpu, dtype, rows, width, keys, scores, rest):
    """Scores around 2^20 and above, in the same step, in steps or blocks of their own: exact, and their differences too."""
    rng = np.random.default_rng(keys)
    q, k, v = np.zeros((rows, 2, width)), np.zeros((keys, 1, width)), rounded(rng.normal(0, 1, (keys, 1, width)), DT[dtype][1])
    q[:, :, 0], q[:, :, 1] = 2**12, 1
    for j in range(keys):
        s = scores.get(j, rest)
        k[j, 0, 0] = np.round(s / 2**12)
        k[j, 0, 1] = s - k[j, 0, 0] * 2**12
    if not np.array_equal(rounded(k, DT[dtype][1]), k):
        assert dtype == "bf16"
        pytest.skip("bf16 does not hold these scores")
    got, lse = attend(gpu, dtype, q, k, v, LN2)
    want, want_lse = plain.attend(q, k, v, [rows], [keys], 1, LN2, False, 0)
    size, _ = plain.attend(q, k, np.abs(v), [rows], [keys], 1, LN2, False, 0)
    # a weight's rounding to the type and its exponential's error, the output's rounding
    weight = (0 if dtype == "f32" else ULP[dtype]) + 2.0**-20
    assert (np.abs(got - want) <= 2 * weight * size + 1.01 * ULP[dtype] * np.abs(want)).all()
    # one rounding of a number so large, and a small logarithm's
    assert (np.abs(lse - want_lse) <= 2.0**-23 * np.abs(want_lse) + 2.0**-19).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [5, 100], ids=["few", "many"])
@pytest.mark.parametrize("size", [1e3, 1e4, 1e5, 1e7, 1e12])
def test_attend_scores_of_every_size(gpu, dtype, rows, size):
    """Rows of scores up to 10^12, whatever falls between: every weight is that of a score resolved to 2^-22 of its magnitude."""
    rng = np.random.default_rng(int(size))
    width, keys = 64, 300
    up = {"f32": size, "f16": min(size, 1e4), "bf16": size}[dtype]
    q, k, v = (rounded(rng.normal(0, 1, (n, 1, width)), DT[dtype][1]) for n in (rows, keys, keys))
    q[:, :, 1:], k[:, :, 1:] = 0, 0  # (one product a score: nothing of a sum is lost)
    q = rounded(q * up, DT[dtype][1])
    got, lse = attend(gpu, dtype, q, k, v, 0.25)
    s = 0.25 * q[:, 0, :1] * k[None, :, 0, 0]
    # each score off by up to `off` either way: a weight by e^(2 off), an output by what its weights' bounds leave it
    off = np.abs(s).max(1, keepdims=True) * 2.0**-22 + 2.0**-20
    low, high = np.exp(s - off - (s + off).max(1, keepdims=True)), np.exp(np.minimum(s + off - (s - off).max(1, keepdims=True), 700))
    high = np.minimum(high / low.sum(1, keepdims=True).clip(1e-300), 1.0)
    bound = high @ np.abs(v[:, 0])
    assert np.isfinite(got).all() and (np.abs(got[:, 0]) <= bound * (1 + 2 * ULP[dtype]) + 2.0**-20).all()
    want, want_lse = plain.attend(q, k, v, [rows], [keys], 1, 0.25, False, 0)
    fine = off[:, 0] < 0.02
    reach = (np.exp(np.minimum(2 * off, 700)) - 1 + 2 * (ULP[dtype] if dtype != "f32" else 0) + 2.0**-19) * plain.attend(q, k, np.abs(v), [rows], [keys], 1, 0.25, False, 0)[0][:, 0]
    assert (np.abs(got[:, 0] - want[:, 0]) <= reach + 1.01 * ULP[dtype] * np.abs(want[:, 0]))[fine].all()
    assert (np.abs(lse - want_lse) <= off + 2.0**-22 * np.abs(want_lse)).all()


# ---- what is worked out again ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,keys,width", [(3, 5_000, 64), (130, 5_000, 64), (130, 5_000, 128), (300, 700, 128), (130, 700, 256)])
@pytest.mark.parametrize("what", ["value", "values", "infinite", "hidden", "key", "hidden key", "queries"])
def test_attend_odd_numbers_over_many_keys(gpu, dtype, rows, keys, width, what):
    """A NaN or an infinity in one value of a long sequence, where all rows see it or some: in the columns that it reaches, and no others."""
    tt = DT[dtype][1]
    gen = torch.Generator(device="cuda").manual_seed(keys)
    q, k, v = (torch.randn(n, h, width, generator=gen, device="cuda").to(tt) for n, h in ((rows, 2), (keys, 1), (keys, 1)))
    last = keys - rows // 2  # a key that the second half of the rows sees (causal)
    if what == "value":
        v[40, 0, 5] = float("nan")
    elif what == "values":
        v[40, 0, :] = float("nan")
    elif what == "infinite":
        v[40, 0, 5], v[41, 0, 6] = float("inf"), -float("inf")
    elif what == "hidden":
        v[last, 0, 3], v[last, 0, 9] = float("nan"), float("inf")
    elif what == "key":
        k[40, 0, 3] = float("nan")
    elif what == "hidden key":
        k[last, 0, 3] = float("nan")
    else:
        q[1, 1, 7], q[2, 0, 3] = float("nan"), float("inf")
    scale, causal = width**-0.5, "hidden" in what
    got, lse = attend(gpu, dtype, q, k, v, scale, causal)
    seen = torch.ones(rows, keys, dtype=torch.bool, device="cuda")
    if causal:
        seen = torch.arange(keys, device="cuda")[None] <= torch.arange(rows, device="cuda")[:, None] + keys - rows
    s = torch.einsum("nhw,mw->hnm", q.double(), k[:, 0].double()) * scale
    s = torch.where(seen, s, torch.full_like(s, -float("inf")))
    p = torch.softmax(s, -1)
    # a hidden value has no part, whatever it is; a seen one has its weight's, however small
    fine = torch.where(torch.isfinite(v[:, 0]), v[:, 0].double(), torch.zeros((), device="cuda").double())
    want = torch.einsum("hnm,mw->nhw", p, fine)
    for j in (40, 41, last):
        odd = torch.where(torch.isfinite(v[j, 0]), torch.zeros((), device="cuda"), v[j, 0].float()).double()
        want += torch.where(seen[:, j, None, None], odd, torch.zeros((), device="cuda").double()) + torch.zeros_like(want)
    top = s.max(-1, keepdim=True).values
    want, want_lse = want.cpu().numpy(), (top + torch.exp(s - top).sum(-1, keepdim=True).log())[..., 0].t().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isnan(lse), np.isnan(want_lse))
    some = np.isfinite(want)
    assert np.array_equal(got[~some & ~np.isnan(want)], want[~some & ~np.isnan(want)])
    # as in a long attention without them: beside the root of the sum of squares a weight's error is a rounding
    if some.any():
        off = np.linalg.norm(got[some] - want[some]) / np.linalg.norm(want[some])
        assert off <= {"f32": 2e-6, "f16": 2.0 * 2**-11, "bf16": 2.0 * 2**-8}[dtype], off
    assert (np.abs(lse - want_lse)[np.isfinite(want_lse)] <= 2.0**-18).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attend_works_out_rows_over_very_many_keys(gpu, dtype):
    """Rows that see a NaN, and rows that must not, over more keys than a wait for them would have patience for."""
    tt = DT[dtype][1]
    rows, keys, width = 100, 150_000, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(n, 1, width, generator=gen, device="cuda").to(tt) for n in (rows, keys, keys))
    v[7, 0, 5], v[keys - 20, 0, 3] = float("nan"), float("nan")  # seen by all; by the last 20 rows
    got, lse = attend(gpu, dtype, q, k, v, 0.125, True)
    seen = torch.arange(keys, device="cuda")[None] <= torch.arange(rows, device="cuda")[:, None] + keys - rows
    s = torch.einsum("nw,mw->nm", q[:, 0].double(), k[:, 0].double()) * 0.125
    s = torch.where(seen, s, torch.full_like(s, -float("inf")))
    v[7, 0, 5], v[keys - 20, 0, 3] = 0, 0
    want = (torch.softmax(s, -1) @ v[:, 0].double()).cpu().numpy()
    want[:, 5] = np.nan
    want[-20:, 3] = np.nan
    assert np.array_equal(np.isnan(got[:, 0]), np.isnan(want))
    some = ~np.isnan(want)
    off = np.linalg.norm((got[:, 0] - want)[some]) / np.linalg.norm(want[some])
    assert off <= {"f32": 2e-6, "f16": 2.0 * 2**-11}[dtype], off
    assert np.abs(lse[:, 0] - torch.logsumexp(s, -1).cpu().numpy()).max() <= 2.0**-18


# ---- waits that give up ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,k_lens,heads", [([100], [9_000], 1), ([300, 1, 900], [300, 70, 900], 4), ([2000], [2000], 2), ([150] * 20, [150] * 20, 8)])
def test_attend_that_gives_up_leaves_its_counters(gpu, dtype, q_lens, k_lens, heads):
    """Every other block gives up: the next call reports it, and finds the working memory as any call leaves it."""
    code, tt = DT[dtype]
    w, rows, keys = 64, sum(q_lens), sum(k_lens)
    q, k, v = (torch.randn(n, heads, w, device="cuda").to(tt) for n in (rows, keys, keys))
    qs, ks = (dev(np.concatenate([[0], np.cumsum(x)]).astype(np.int32)) for x in (q_lens, k_lens))
    p = tcu.Packed(gpu, len(q_lens), rows, keys, max(q_lens), max(k_lens), qs.data_ptr(), ks.data_ptr())
    work = torch.zeros(p.attend_workspace(code, heads, heads, w), dtype=torch.uint8, device="cuda")

    def go():
        out = torch.full_like(q, 9.0)
        p.attend(code, heads, heads, w, q.data_ptr(), heads * w, w, k.data_ptr(), heads * w, w, v.data_ptr(), heads * w, w, out.data_ptr(),
                 heads * w, w, 0.125, causal=True, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        torch.cuda.synchronize()
        return out
    want = go()
    gpu.sync()
    for _ in range(2):
        gpu.debug_abort_next()
        go()
        assert not work[:8192].any()
        with pytest.raises(tcu.TcuError, match="gave up") as e:
            gpu.sync()
        assert e.value.code == -3
        assert torch.equal(go(), want) and not work[:8192].any()
        gpu.sync()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(8, 300, 33_000), (33, 64, 20_000), (600, 700, 900), (2, 40_000, 256)])
def test_linear_that_gives_up_leaves_its_counters(gpu, dtype, rows, n, k):
    code, tt = DT[dtype]
    rng = np.random.default_rng(k)
    x, w = (base.random_matrix(rng, gpu, r, k, plain.NV)[0] for r in (rows, n))
    work = torch.zeros(w.m.linear_workspace(x.m, code), dtype=torch.uint8, device="cuda")

    def go():
        y = torch.full((rows, n), 9.0, dtype=tt, device="cuda")
        w.m.linear(x.m, code, y.data_ptr(), n, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
        torch.cuda.synchronize()
        return y
    want = go()
    gpu.sync()
    gpu.debug_abort_next()
    go()
    assert not work[:8192].any()
    with pytest.raises(tcu.TcuError, match="gave up"):
        gpu.sync()
    assert torch.equal(go(), want)
    gpu.sync()


# ---- values near a type's ends --------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,width", [(5, 64), (100, 64), (100, 128), (5, 256)])
@pytest.mark.parametrize("down", [14, 18, 22, 26, 30])
@pytest.mark.parametrize("where", ["step", "steps"])
def test_attend_f16_small_weights_of_large_values(gpu, rows, width, down, where):
    """A weight of f16 is held to 2^-36 of the row's largest, not to f16's own smallest: values of 60,000 beside it are felt."""
    keys = 200
    q, k, v = np.zeros((rows, 1, width)), np.zeros((keys, 1, width)), np.zeros((keys, 1, width))
    q[:, :, 0], k[:, :, 0] = 1, -500
    k[7, 0, 0] = 0
    at = 9 if where == "step" else 150
    k[at, 0, 0], v[at, 0] = -down, np.linspace(30_000, 60_000, width).round(-2)
    v = rounded(v, torch.float16)
    got, _ = attend(gpu, "f16", q, k, v, LN2)
    want, _ = plain.attend(q, k, v, [rows], [keys], 1, LN2, False, 0)
    assert (np.abs(got - want) <= (2.0**-11 + 2.0**-19) * np.abs(want) + 2.0**-36 * 60_000 + 1.01 * 2.0**-11 * np.abs(want) + 2.0**-25).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,width", [(5, 64), (100, 64), (100, 128), (100, 256)])
@pytest.mark.parametrize("keys", [70, 3000])
@pytest.mark.parametrize("end", ["largest", "smallest"])
def test_attend_values_near_the_ends(gpu, dtype, rows, width, keys, end):
    """Weighted sums that pass a type's end before they are divided: an output is never further out than the values. And values that
    are small, which nothing that is done for those may lose."""
    rng = np.random.default_rng(keys)
    end = {"largest": 60_000.0 if dtype == "f16" else 3e38, "smallest": 1e-5 if dtype == "f16" else 1e-33}[end]
    q, k = (rounded(rng.normal(0, 1, (n, 2, width)), DT[dtype][1]) for n in (rows, keys))
    v = rounded(rng.uniform(0.9, 1, (keys, 2, width)) * end, DT[dtype][1])
    v[:, 1] *= np.where(rng.random((keys, 1)) < 0.5, -1, 1)
    scale = width**-0.5
    got, _ = attend(gpu, dtype, q, k, v, scale)
    want, _ = plain.attend(q, k, v, [rows], [keys], 2, scale, False, 0)
    size, _ = plain.attend(q, k, np.abs(v), [rows], [keys], 2, scale, False, 0)
    score = scale * np.abs(q).sum(-1).max() * np.abs(k).max() * 2.0**-20
    weight = score + 2.0**-19 + (0 if dtype == "f32" else ULP[dtype]) + (keys // 16 + 8) * 2.0**-24
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= 2 * weight * size + 1.01 * ULP[dtype] * np.abs(want) + 2 * base.TINY[dtype] + 2.0**-126).all()


# ---- tiles of very different values (f32) ---------------------------------------------------------------------------

@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("small,large", [(2.0**-111, 2.0**126), (2.0**126, 2.0**-111), (2.0**-60, 2.0**100), (2.0**-20, 2.0**20)])
@pytest.mark.parametrize("mask", ["causal", "window", "weights"])
def test_attend_f32_tiles_apart(gpu, width, small, large, mask):
    """Values of 64 keys beside others up to 2^237 as large, which a row does not see, or weighs with nothing: it keeps its own to
    2^-35 of the largest of their 64."""
    rng = np.random.default_rng(1)
    n = 128
    q, k, v = (rounded(rng.normal(0, 1, (n, 1, width)).clip(-1.9, 1.9), torch.float32) for _ in range(3))
    v[:64] *= small
    v[64:] *= large
    if mask == "weights":  # rows of either sign: the keys of one half are nothing to them
        q[:, 0, 0], k[:64, 0, 0], k[64:, 0, 0] = np.where(np.arange(n) % 2, 1.0, -1.0), 2000, -2000
    causal, window, scale = mask != "weights", 20 if mask == "window" else 0, 0.125
    got, _ = attend(gpu, "f32", q, k, v, scale, causal, window)
    want, _ = plain.attend(q, k, v, [n], [n], 1, scale, causal, window)
    size, _ = plain.attend(q, k, np.abs(v), [n], [n], 1, scale, causal, window)
    # the scores' rounding (a weight's: 64 or 128 products of up to 2^11 each held to 2^-21), and what 64 neighbours share
    kmax = 2000 if mask == "weights" else 2
    weight = scale * np.abs(q).sum(-1).max() * kmax * 2.0**-20 + 2.0**-19
    seen = np.zeros((n, 2))  # the largest of the two tiles that the row has something from
    for i in range(n):
        lo, hi = (max(0, i + 1 - window) if window else 0, i + 1) if causal else (0, n)
        for t, (a, b) in enumerate(((0, 64), (64, 128))):
            there = min(hi, b) > max(lo, a) and (causal or (i % 2 == 1) == (t == 0))
            seen[i, t] = (small, large)[t] * 2 if there else 0
    tol = 2 * weight * size + 2.0**-34 * seen.max(1)[:, None, None] + 2.0**-148
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("rows,width", [(5, 64), (100, 64), (100, 128)])
@pytest.mark.parametrize("down,up", [(30, 20), (40, 60), (100, 110), (120, 90)])
@pytest.mark.parametrize("first", [True, False])
def test_attend_f32_small_weights_of_large_values(gpu, rows, width, down, up, first):
    """A step whose weights are far below the row's largest, of values as far above the others: it is felt."""
    keys = 192
    rng = np.random.default_rng(down)
    q, k, v = np.zeros((rows, 1, width)), np.zeros((keys, 1, width)), rounded(rng.uniform(0.5, 1, (keys, 1, width)), torch.float32)
    q[:, :, 0], k[:, :, 0] = 1, -500
    a, b = (7, 150) if first else (150, 7)
    k[a, 0, 0], k[b, 0, 0] = 0, -down
    v[b] *= 2.0**up
    got, _ = attend(gpu, "f32", q, k, v, LN2)
    want, _ = plain.attend(q, k, v, [rows], [keys], 1, LN2, False, 0)
    # (a weight's exponential, 2^-19; what 64 neighbours of the values share, times the weight that they have at most)
    assert (np.abs(got - want) <= 2.0**-18 * np.abs(want) + 2.0**-34 * 2.0 ** max(up - down, 0)).all()


# ---- long sums ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_linear_long_rows_have_no_bias(gpu, dtype):
    """Thousands of products of one sign: the matrix unit rounds its sums towards zero, so a result is made of sums of at most
    256 of its additions (each off by a unit in the last place of f32 at most, half of one on average): 2^-16 on average."""
    code, tt = DT[dtype]
    rows, n, k = 16, 150 * 128, 2**18
    gen = torch.Generator(device="cuda").manual_seed(0)
    numbers = torch.tensor(plain.NUMBERS, device="cuda")
    power = torch.randint(-14, -4, (k // 32,), device="cuda", generator=gen)  # of the scales, the same for all rows (sums then need more than 24 bits)
    mats = []
    for r in (rows, n):
        codes = torch.randint(0, 256, (r, k // 2), dtype=torch.uint8, device="cuda", generator=gen) & 0x77
        scales = (power + 127).to(torch.uint8).view(1, k // 128, 1, 4).expand(-(-r // 128), -1, 128, -1).contiguous()
        mats.append((tcu.Fp4(gpu, r, k, tcu.MX, codes.data_ptr(), scales.data_ptr()), codes, scales))
    want = torch.zeros(rows, n, dtype=torch.float64, device="cuda")
    for at in range(0, k, 2**12):
        by = torch.pow(2.0, power[at // 32:(at + 2**12) // 32].double()).repeat_interleave(32)
        xv, wv = (numbers[torch.stack([c & 7, c >> 4], -1).flatten(1).long()].double() * by for c in (m[1][:, at // 2:at // 2 + 2**11] for m in mats))
        want += xv @ wv.t()
    x, w = mats[0][0], mats[1][0]
    y = torch.zeros(rows, n, dtype=tt, device="cuda")
    work = torch.zeros(w.linear_workspace(x, code), dtype=torch.uint8, device="cuda")
    w.linear(x, code, y.data_ptr(), n, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    off = (y.double() - want) / want
    assert off.abs().max() <= ULP[dtype] + 2.0**-14
    assert off.mean().abs() <= 2.0**-16, off.mean()



@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,heads,keys,width", [(8192, 8, 131_072, 64), (5000, 8, 70_001, 128), (40, 300, 131_072, 64), (1, 600, 270_000, 128), (100, 40, 70_000, 256)])
def test_attend_many_keys_have_no_bias(gpu, dtype, rows, heads, keys, width):
    """Tens of thousands of values of one sign a row, in units that blocks do not share: sums of at most 512 additions in the matrix
    unit, each off by a unit in the last place of f32 at most: 2^-14. (Heads of few rows share their keys in memory.)"""
    code, tt = DT[dtype]
    gen = torch.Generator(device="cuda").manual_seed(0)
    kh = heads if rows > 64 and width < 256 else 1
    q, k = torch.randn(rows, heads, width, generator=gen, device="cuda").to(tt), (0.1 * torch.randn(keys, kh, width, generator=gen, device="cuda")).to(tt)
    v = (1 + 0.25 * torch.rand(keys, kh, width, generator=gen, device="cuda")).to(tt)
    k[:200] *= 3  # (the largest scores are not the last)
    qs, ks = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (rows, keys))
    p = tcu.Packed(gpu, 1, rows, keys, rows, keys, qs.data_ptr(), ks.data_ptr())
    work = torch.zeros(p.attend_workspace(code, heads, heads, width), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    step = width if kh > 1 else 0
    p.attend(code, heads, heads, width, q.data_ptr(), heads * width, width, k.data_ptr(), kh * width, step, v.data_ptr(), kh * width, step, out.data_ptr(),
             heads * width, width, width**-0.5, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    for h in (0, heads // 2, heads - 1):
        s = q[:200, h].double() @ k[:, h % kh].double().t() * width**-0.5
        want = torch.softmax(s, -1) @ v[:, h % kh].double()
        off = (out[:200, h].double() - want) / want
        assert off.abs().max() <= ULP[dtype] + 2.0**-13
        assert off.mean().abs() <= 2.0**-14 + ULP[dtype] / off.numel() ** 0.5


# ---- many rows, many sequences --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attend_more_rows_than_24_bits_count(gpu, dtype):
    """270,000 tokens of 64 heads: 17 million rows."""
    rows, heads, w, n = 270_000, 64, 8, 90
    code, tt = DT[dtype]
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(rows, h, w, generator=gen, device="cuda").to(tt) for h in (heads, 2, 2))
    starts = torch.arange(0, rows + 1, n, dtype=torch.int32, device="cuda")
    p = tcu.Packed(gpu, rows // n, rows, rows, n, n, starts.data_ptr())
    work = torch.zeros(p.attend_workspace(code, heads, 2, w), dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 9.0)
    p.attend(code, heads, 2, w, q.data_ptr(), heads * w, w, k.data_ptr(), 2 * w, w, v.data_ptr(), 2 * w, w, out.data_ptr(), heads * w, w, 0.3,
             causal=True, work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    qq, kk, vv = (x.view(rows // n, n, -1, w).double().transpose(1, 2) for x in (q, k, v))
    for at in range(0, rows // n, 500):
        x, y, z = qq[at:at + 500], kk[at:at + 500].repeat_interleave(32, 1), vv[at:at + 500].repeat_interleave(32, 1)
        s = (x @ y.transpose(-1, -2)) * 0.3
        s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -float("inf"))
        want = torch.softmax(s, -1) @ z
        got = out.view(rows // n, n, heads, w)[at:at + 500].transpose(1, 2).double()
        # a weight's rounding of values up to 6, the output's
        assert (got - want).abs().max() <= (2.0**-17 if dtype == "f32" else 3 * 2.0**-11) * 6


@pytest.mark.parametrize("q_lens,k_lens,longest", [([70] * 300, [70] * 300, 21_000), ([100, 0, 3, 80] * 40, [90, 7, 0, 130] * 40, 9_080),
                                                   ([66] * 700, [65] * 699 + [20_000], 20_000)])
def test_attend_f32_longest_far_above_the_others(gpu, q_lens, k_lens, longest):
    """Sequences that might have been much longer than they are: their keys are found by where they lie."""
    rng = np.random.default_rng(len(q_lens))
    rows, keys = sum(q_lens), sum(k_lens)
    q, k, v = (rng.normal(0, 1, (n, 2, 64)).astype(np.float32) for n in (rows, keys, keys))
    qd, kd, vd = (dev(x) for x in (q, k, v))
    qs, ks = (dev(np.concatenate([[0], np.cumsum(x)]).astype(np.int32)) for x in (q_lens, k_lens))
    p = tcu.Packed(gpu, len(q_lens), rows, keys, max(q_lens), longest, qs.data_ptr(), ks.data_ptr())
    work = torch.zeros(p.attend_workspace(0, 2, 2, 64), dtype=torch.uint8, device="cuda")
    out = torch.full_like(qd, 9.0)
    p.attend(0, 2, 2, 64, qd.data_ptr(), 128, 64, kd.data_ptr(), 128, 64, vd.data_ptr(), 128, 64, out.data_ptr(), 128, 64, 0.125, causal=True,
             work=work.data_ptr(), work_bytes=work.numel(), stream=1)
    sync(gpu)
    want, _ = plain.attend(q.astype(np.float64), k.astype(np.float64), v.astype(np.float64), q_lens, k_lens, 2, 0.125, True, 0)
    assert np.abs(host(out) - want).max() <= 2.0**-17 * 5


# ---- masks and residuals that span whole tiles ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [([700], [700]), ([300, 500], [900, 650]), ([150, 40], [1000, 70])], ids=str)
@pytest.mark.parametrize("q_heads,heads,width", [(2, 2, 64), (4, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("window", [64, 200, 333, 640])
def test_attend_wide_windows(gpu, dtype, lens, q_heads, heads, width, window):
    """Windows of several steps of keys: steps that a row's tile sees whole, in part and not at all."""
    base.check_attend(gpu, dtype, *lens, q_heads, heads, width, True, window)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["mx", "nv"])
@pytest.mark.parametrize("rows,n,k", [(1500, 3000, 300), (2100, 5000, 512), (4096, 1000, 256), (777, 9001, 130)])
def test_linear_residual_of_many_rows(gpu, dtype, name, rows, n, k):
    rng = np.random.default_rng(rows)
    base.check_linear(gpu, rng, dtype, base.FORMATS[name], rows, n, k, act=1, bias=True, residual=True)
