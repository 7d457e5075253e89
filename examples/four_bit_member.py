"""A fitted member's in-context stage held in four bits, from test rows to class log-probabilities.

    python examples/four_bit_member.py [--rows 10000] [--test 256]

Fits a member's caches on the device (random-init weights of the full-size architecture), widens each layer's stored keys
and values, quantises them into the pages of a four-bit cache and the layers' weights into four-bit matrices, and then
predicts with the four-bit operators: per layer a LayerNorm, the query projection, the scalable softmax's query MLP, the
attention over the cache, the out-projection and the feed-forward, and at the end the decoder and the labels' log
probabilities with the entropy and the likeliest alternatives. The answers are compared with the same member's at full
precision, and the bytes and times of both are printed.

The norms and the query scale's tanh are torch operations here; everything that reads the cache, the weights or the
scores is the framework's.
"""
import argparse
import importlib.util
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def package():
    """The framework (its folder's name is not an identifier)."""
    name = "tabicl_anywhere_b200"
    if name not in sys.modules:
        here = os.path.join(ROOT, "tabicl-anywhere_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(here, "__init__.py"), submodule_search_locations=[here])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


tcu = package()
from tabicl_anywhere_b200 import synth  # noqa: E402

PAGE, GROUP, CHUNK = 256, 32, 256
STREAM = 1  # the legacy default stream, which torch uses here


class Linear4:
    """A linear layer in four bits, over buffers of its own."""

    def __init__(self, gpu, weight, bias):
        n, k = weight.shape
        self.n, self.k = n, k
        self.codes = torch.empty(tcu.W4.code_bytes(n, k), dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(tcu.W4.scale_bytes(n, k, GROUP), dtype=torch.uint8, device="cuda")
        self.bias = torch.from_numpy(np.ascontiguousarray(bias)).cuda()
        self.w4 = tcu.W4(gpu, n, k, GROUP, self.codes.data_ptr(), self.scales.data_ptr())
        w = torch.from_numpy(np.ascontiguousarray(weight)).cuda()
        self.w4.pack(tcu.F32, w.data_ptr(), k, stream=STREAM)
        torch.cuda.synchronize()
        self.work = torch.zeros(16, dtype=torch.uint8, device="cuda")

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def __call__(self, x, act=0, residual=None):
        rows = x.shape[0]
        need = self.w4.linear_workspace(rows, tcu.F32)
        if need > self.work.numel():
            self.work = torch.zeros(need, dtype=torch.uint8, device="cuda")
        y = torch.empty(rows, self.n, device="cuda") if residual is None else residual  # a residual is added to in place
        self.w4.linear(tcu.F32, rows, x.data_ptr(), x.stride(0), y.data_ptr(), self.n, bias=self.bias.data_ptr(), act=act,
                       residual=None if residual is None else y.data_ptr(), ldr=self.n, work=self.work.data_ptr(),
                       work_bytes=self.work.numel(), stream=STREAM)
        return y


class Member4:
    """One fitted problem in four bits: a paged cache a layer, four-bit weights, and the stage over them."""

    def __init__(self, gpu, cfg, weights, model, rows):
        self.gpu, self.rows = gpu, rows
        s = synth.icl_shape(cfg)
        self.d, self.heads, self.layers, self.classes = s["d"], s["heads"], s["layers"], s["outs"]
        self.width = self.d // self.heads
        pages = -(-rows // PAGE)
        page_bytes = tcu.Kv4Cache.page_bytes(self.heads, self.width, PAGE, GROUP)
        self.pool = torch.empty(self.layers, pages, page_bytes, dtype=torch.uint8, device="cuda")
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
        self.lens = torch.tensor([rows], dtype=torch.int32, device="cuda")
        slots = torch.arange(rows, dtype=torch.int64, device="cuda")
        self.caches = []
        stored = model.layer_bytes
        nbytes = sum(tcu.record(tcu.KV_F32, self.d, min(CHUNK, rows - r)) for r in range(0, rows, CHUNK))
        for l in range(self.layers):
            layer = torch.from_numpy(stored(l, nbytes)).cuda()
            k, v = (torch.empty(rows, self.d, device="cuda") for _ in range(2))
            gpu.layer_rows(tcu.KV_F32, self.d, layer.data_ptr(), rows, CHUNK, k.data_ptr(), v.data_ptr())
            cache = tcu.Kv4Cache(gpu, self.pool[l].data_ptr(), pages, heads=self.heads, width=self.width, page=PAGE, group=GROUP)
            cache.store(tcu.F32, rows, slots.data_ptr(), k.data_ptr(), self.d, self.width, v.data_ptr(), self.d, self.width,
                        stream=STREAM)
            self.caches.append(cache)
            torch.cuda.synchronize()
        dev = lambda name: torch.from_numpy(np.ascontiguousarray(weights[name])).cuda()  # noqa: E731
        lin = lambda name: Linear4(gpu, weights[name + ".weight"], weights[name + ".bias"])  # noqa: E731
        self.scale = torch.from_numpy(model.scales()).cuda()  # the fit's query scale, the softmax's 1 / sqrt(width) in it
        self.blocks = []
        for i in range(self.layers):
            p = f"icl_predictor.tf_icl.blocks.{i}."
            q = p + "attn.ssmax_layer.query_mlp."
            self.blocks.append(dict(
                n1=(dev(p + "norm1.weight"), dev(p + "norm1.bias")), n2=(dev(p + "norm2.weight"), dev(p + "norm2.bias")),
                wq=Linear4(gpu, weights[p + "attn.in_proj_weight"][:self.d], weights[p + "attn.in_proj_bias"][:self.d]),
                q0=lin(q + "0"), q2=lin(q + "2"), wo=lin(p + "attn.out_proj"), w1=lin(p + "linear1"), w2=lin(p + "linear2")))
        self.ln = (dev("icl_predictor.ln.weight"), dev("icl_predictor.ln.bias"))
        self.dec0, self.dec2 = lin("icl_predictor.decoder.0"), lin("icl_predictor.decoder.2")

    @property
    def nbytes(self):
        linears = [x for b in self.blocks for x in b.values() if isinstance(x, Linear4)] + [self.dec0, self.dec2]
        return self.pool.numel(), sum(x.nbytes for x in linears)

    def stage(self, h):
        """Class scores [n][classes] of test-row representations h [n][d] (kept)."""
        n, d, w = h.shape[0], self.d, self.width
        norm = lambda x, p: torch.nn.functional.layer_norm(x, (d,), *p)  # noqa: E731
        batch = tcu.Kv4Cache.batch(1, n, self.rows, self.lens.data_ptr(), self.table.data_ptr(), self.table.shape[1])
        work = torch.zeros(self.caches[0].attend_workspace(batch, self.heads, tcu.F32), dtype=torch.uint8, device="cuda")
        h = h.clone()
        for l, b in enumerate(self.blocks):
            q = b["wq"](norm(h, b["n1"]))
            m = b["q2"](b["q0"](q.view(n * self.heads, w), act=1)).view(n, d)
            q = q * self.scale[l] * (1 + torch.tanh(m))
            att = torch.empty_like(q)
            self.caches[l].attend(batch, tcu.F32, self.heads, q.data_ptr(), d, w, att.data_ptr(), d, w, 1.0, work=work.data_ptr(),
                                  work_bytes=work.numel(), stream=STREAM)
            b["wo"](att, residual=h)
            b["w2"](b["w1"](norm(h, b["n2"]), act=1), residual=h)
        return self.dec2(self.dec0(norm(h, self.ln), act=1))


def answer(gpu, scores, labels, top=3, temperature=0.9):
    """Log probability of each row's label, entropy, and the `top` likeliest classes with theirs."""
    n, classes = scores.shape
    out, entropy = torch.empty(n, 1, device="cuda"), torch.empty(n, device="cuda")
    values, ids = torch.empty(n, top, device="cuda"), torch.empty(n, top, dtype=torch.int32, device="cuda")
    gpu.label_logprobs(tcu.F32, scores.data_ptr(), n, classes, scores.stride(0), labels.data_ptr(), 1, out.data_ptr(),
                       entropy=entropy.data_ptr(), top=top, top_values=values.data_ptr(), top_ids=ids.data_ptr(),
                       temperature=temperature, stream=STREAM)
    return out[:, 0], entropy, values, ids


def timed(f, reps=5):
    f()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for _ in range(reps):
        f()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / reps


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--rows", type=int, default=10_000, help="training rows of the member")
    ap.add_argument("--test", type=int, default=256, help="test rows")
    a = ap.parse_args(argv)
    gpu = tcu.Gpu(0)
    cfg = synth.config("full")
    weights = {k: v for k, v in synth.weights(cfg, seed=0).items() if k.startswith("icl_")}
    w = tcu.GpuWeights.from_tensors(gpu, synth.icl_shape(cfg), weights, for_fit=True)
    d = synth.icl_shape(cfg)["d"]
    reps = torch.from_numpy(synth.row_reps(a.rows, d, 1)).cuda()
    y = torch.from_numpy(synth.labels(a.rows, cfg["max_classes"], 2)).cuda()
    model = tcu.fit_icl(w, reps.data_ptr(), y.data_ptr(), a.rows, CHUNK, tcu.KV_F32)
    member = Member4(gpu, cfg, weights, model, a.rows)

    h = torch.from_numpy(synth.row_reps(a.test, d, 3)).cuda()
    labels = torch.from_numpy(synth.labels(a.test, cfg["max_classes"], 4).astype(np.int32)).cuda()
    full = torch.empty(a.test, member.classes, device="cuda")
    model.stage_device(h.data_ptr(), a.test, member.classes, full.data_ptr(), STREAM)
    scores = member.stage(h)
    want, got = answer(gpu, full, labels), answer(gpu, scores, labels)
    gpu.sync(STREAM)
    cache, linears = member.nbytes
    off = float((want[0] - got[0]).abs().max())
    same = float((want[3][:, 0] == got[3][:, 0]).float().mean())
    print(f"cache: {a.rows * d * 8 * member.layers / 1e6:.1f} MB in f32, {cache / 1e6:.1f} MB in four bits; "
          f"weights in four bits: {linears / 1e6:.1f} MB")
    print(f"label log-probabilities: mean {float(got[0].mean()):.5f} (full precision {float(want[0].mean()):.5f}), "
          f"largest difference {off:.2e}; likeliest class the same for {100 * same:.1f}% of {a.test} rows")
    print(f"entropy: mean {float(got[1].mean()):.5f} nats (full precision {float(want[1].mean()):.5f})")
    print(f"stage: {timed(lambda: member.stage(h)):.3f} ms in four bits, "
          f"{timed(lambda: model.stage_device(h.data_ptr(), a.test, member.classes, full.data_ptr(), STREAM)):.3f} ms at full precision")
    gpu.sync(STREAM)
    return member, h, scores


if __name__ == "__main__":
    main()
