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
    reach = (np.exp(2 * off) - 1 + 2 * (ULP[dtype] if dtype != "f32" else 0) + 2.0**-19) * plain.attend(q, k, np.abs(v), [rows], [keys], 1, 0.25, False, 0)[0][:, 0]
    assert (np.abs(got[:, 0] - want[:, 0]) <= reach + 1.01 * ULP[dtype] * np.abs(want[:, 0]))[fine].all()
    assert (np.abs(lse - want_lse) <= off + 2.0**-22 * np.abs(want_lse)).all()
