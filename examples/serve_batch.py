"""Several requests served together over one pool of quantized KV pages.

Each step takes the next token of every running request and one chunk of a
waiting prompt, all as rows of one batch: packed projections
(``Weight.gemv`` / ``Weight.gemm_rows``), ``KVPool.append`` (RoPE and the
quantizing write), ``KVPool.attend`` over the pages of every sequence at
once, and ``adjust_logits`` (penalties, biases, mask, argmax) for the rows
that give a token. Pages come from a free list when a sequence grows and go
back when its request ends.

    python examples/serve_batch.py              # the tiny synthetic model
    python examples/serve_batch.py model.lumina 32 32 10000
                                                # file, query heads, KV heads, RoPE theta
"""
from __future__ import annotations

import os
import sys
import time
from dataclasses import dataclass, field

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "lumina-studio_b200"))

from lumina_b200 import cuda, serving  # noqa: E402
from lumina_b200.cuda import LuminaError  # noqa: E402
from lumina_b200.engine import rope_tables  # noqa: E402
from lumina_b200.loader import LuminaFile, upload_record  # noqa: E402


@dataclass(eq=False)  # a request is itself, not its fields
class Request:
    prompt: list
    max_tokens: int = 32
    repeat_penalty: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: dict = field(default_factory=dict)   # token -> added value
    allowed: np.ndarray | None = None          # (vocab) bool; None: every token
    stop: frozenset = frozenset()
    out: list = field(default_factory=list)
    done: int = 0                              # tokens in the cache
    pages: list = field(default_factory=list)

    def waiting(self) -> int:
        """Rows of the prompt that are not in the cache yet."""
        return max(0, len(self.prompt) - self.done)


class BatchModel:
    """The dense decoder of a ``.lumina`` file (int4 projections) as batched
    steps over quantized pages."""

    def __init__(self, path, n_heads, n_kv, theta=1e4, eps=1e-6, bits=8, page_size=16, n_pages=256, max_seq=4096, device=0):
        self.device = torch.device("cuda", device)
        with LuminaFile(path) as f:
            recs = {n: f.record(n) for n in f.names()}

            def raw(name):
                return torch.tensor(recs[name].data, device=self.device)

            self.embed = raw("model.embed_tokens.weight").half()
            # fp16 values as in the single-sequence model, whose head kernel has
            # no entry of its own: an fp32 product of the library's
            self.head = (raw("lm_head.weight").half() if "lm_head.weight" in recs else self.embed).float().T
            self.layers = []
            while "model.layers.%d.input_layernorm.weight" % len(self.layers) in recs:
                p = "model.layers.%d." % len(self.layers)
                self.layers.append({
                    "norm": (raw(p + "input_layernorm.weight"), raw(p + "post_attention_layernorm.weight")),
                    **{n: upload_record(recs[p + k + "_proj.weight"], device) for n, k in (
                        ("q", "self_attn.q"), ("k", "self_attn.k"), ("v", "self_attn.v"), ("o", "self_attn.o"),
                        ("gate", "mlp.gate"), ("up", "mlp.up"), ("down", "mlp.down"))}})
        self.vocab, self.d = self.embed.shape
        self.n_heads, self.n_kv, self.hd, self.eps = n_heads, n_kv, self.d // n_heads, eps
        self.cos, self.sin = (torch.tensor(t, device=self.device) for t in rope_tables(self.hd, max_seq, theta))
        self.page_size, self.max_seq = page_size, max_seq
        self.pools = [serving.KVPool.empty(n_pages, n_kv, self.hd, bits, page_size, device) for _ in self.layers]
        self.free = list(range(n_pages))

    def _rms(self, x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * w

    def _project(self, w, x, y):
        """y (rows, w.rows; a column range of a wider tensor) = x W^T"""
        stream = torch.cuda.current_stream(self.device).cuda_stream
        if x.shape[0] > 16:
            try:
                return w.gemm_rows(x.data_ptr(), x.shape[0], x.stride(0), y.data_ptr(), y.stride(0), stream)
            except LuminaError as e:
                if e.code != 3:  # unsupported: a width outside the tensor-core layout
                    raise
        for i in range(0, x.shape[0], 16):
            w.gemv(x[i:].data_ptr(), min(16, x.shape[0] - i), x.stride(0), y[i:].data_ptr(), y.stride(0), stream)

    def step(self, tokens, batch, last):
        """Hidden rows of ``tokens`` through every layer; logits of the rows
        ``last``."""
        n, wq, wk = len(tokens), self.n_heads * self.hd, self.n_kv * self.hd
        x = self.embed[torch.tensor(tokens, device=self.device)].float()
        qkv = torch.empty(n, wq + 2 * wk, device=self.device)
        y = torch.empty(n, self.d, device=self.device)
        ff = [torch.empty(n, self.layers[0]["gate"].rows, device=self.device) for _ in range(2)]
        attn = torch.empty(n, wq, device=self.device)
        for pool, w in zip(self.pools, self.layers):
            q, k, v = qkv[:, :wq], qkv[:, wq:wq + wk], qkv[:, wq + wk:]
            h = self._rms(x, w["norm"][0])
            for name, dst in (("q", q), ("k", k), ("v", v)):
                self._project(w[name], h, dst)
            pool.attend(batch, pool.append(batch, q, k, v, self.cos, self.sin), out=attn)
            self._project(w["o"], attn, y)
            x += y
            h = self._rms(x, w["norm"][1])
            self._project(w["gate"], h, ff[0])
            self._project(w["up"], h, ff[1])
            self._project(w["down"], torch.nn.functional.silu(ff[0]) * ff[1], y)
            x += y
        # no norm before the head, as in the single-sequence model
        return x[torch.tensor(last, dtype=torch.long, device=self.device)] @ self.head

    def grow(self, r, tokens):
        while len(r.pages) * self.page_size < tokens:
            if not self.free:
                raise RuntimeError("the pool is out of pages")
            r.pages.append(self.free.pop())

    def pick(self, logits, reqs):
        """The next token of each request, shaped as it asks."""
        dev, i32 = self.device, torch.int32
        seen = [r.prompt + r.out for r in reqs]
        offs = torch.tensor(np.cumsum([0] + [len(s) for s in seen]), dtype=i32, device=dev)
        toks = torch.tensor([t for s in seen for t in s], dtype=i32, device=dev)

        def per_row(f):
            return torch.tensor([f(r) for r in reqs], device=dev, dtype=torch.float32)

        bias = mask = None
        if any(r.bias for r in reqs):
            bias = (torch.tensor(np.cumsum([0] + [len(r.bias) for r in reqs]), dtype=i32, device=dev),
                    torch.tensor([t for r in reqs for t in r.bias], dtype=i32, device=dev),
                    torch.tensor([float(v) for r in reqs for v in r.bias.values()], device=dev))
        if any(r.allowed is not None for r in reqs):
            words = np.zeros((len(reqs), -(-self.vocab // 32) * 32), bool)
            for row, r in zip(words, reqs):
                row[:self.vocab] = True if r.allowed is None else r.allowed
            mask = torch.tensor(np.packbits(words, axis=1, bitorder="little").view(np.int32), device=dev)
        return serving.adjust_logits(logits, history=(offs, toks), repeat=per_row(lambda r: r.repeat_penalty),
                                     frequency=per_row(lambda r: r.frequency), presence=per_row(lambda r: r.presence),
                                     bias=bias, mask=mask, out=logits)[1].tolist()

    def serve(self, requests, chunk=64):
        """Run every request to its end: a step holds one row of each request
        that generates and up to ``chunk`` rows of one prompt. Returns the
        generated tokens of each; an error leaves the requests cut off."""
        for r in requests:
            if not 0 < len(r.prompt) <= self.max_seq:
                raise ValueError("a prompt of %d tokens, 1 to %d are served" % (len(r.prompt), self.max_seq))
        try:
            self._serve(list(requests), chunk)
        finally:  # the pages of requests that an error cut off
            for r in requests:
                self._release(r)
        return [r.out for r in requests]

    def _release(self, r):
        self.free += r.pages
        r.pages = []

    def _serve(self, live, chunk):
        while live:
            rows, tokens = [], []
            budget, batch_reqs = chunk, []
            for r in live:
                n = min(r.waiting(), budget)
                if n:
                    budget = 0
                    tokens += r.prompt[r.done:r.done + n]
                elif not r.waiting():
                    n = 1
                    tokens.append(r.out[-1])
                else:
                    continue  # its prompt's turn comes later
                self.grow(r, r.done + n)
                r.done += n
                rows.append(n)
                batch_reqs.append(r)
            ld = max(len(r.pages) for r in batch_reqs)
            start = np.cumsum([0] + rows)
            batch = serving.SeqBatch(*(torch.tensor(np.asarray(a, np.int32), device=self.device) for a in (
                start, [r.done for r in batch_reqs], [r.pages + [0] * (ld - len(r.pages)) for r in batch_reqs])),
                n_rows=int(start[-1]), max_rows=max(rows))
            gives = [i for i, r in enumerate(batch_reqs) if not r.waiting()]
            logits = self.step(tokens, batch, [int(start[i + 1]) - 1 for i in gives])
            giving = [batch_reqs[i] for i in gives]
            picked = self.pick(logits, giving) if giving else []
            word = cuda.fault_status(self.device.index)  # a wait that gave up, a page or length out of range
            if word:
                raise RuntimeError("the step's rows are not whole: fault word %d" % word)
            for r, t in zip(giving, picked):
                r.out.append(t)
                if t in r.stop or len(r.out) >= r.max_tokens or len(r.prompt) + len(r.out) > self.max_seq:
                    self._release(r)
                    live.remove(r)


def main():
    from lumina_b200 import synthetic
    cfg, theta = synthetic.TINY, synthetic.TINY["rope_theta"]
    if len(sys.argv) > 1:
        path, heads, n_kv = sys.argv[1], int(sys.argv[2]), int(sys.argv[3])
        theta = float(sys.argv[4]) if len(sys.argv) > 4 else 1e6
    else:
        import tempfile
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
        from oracle.lumina_format import write_lumina
        from oracle.quant import convert_arrays
        path = os.path.join(tempfile.mkdtemp(), "tiny.lumina")
        write_lumina(path, convert_arrays(synthetic.host_weights(cfg), "int4", group_size=64, fp16_scales=True),
                     name="tiny", rung="int4", group_size=64)
        heads, n_kv = cfg["num_attention_heads"], cfg["num_key_value_heads"]
    model = BatchModel(path, heads, n_kv, theta)
    rng = np.random.default_rng(0)
    reqs = [Request([int(t) for t in rng.integers(0, model.vocab, n)], max_tokens=24, repeat_penalty=1.1)
            for n in (5, 150, 33, 64, 17)]
    t0 = time.perf_counter()
    outs = model.serve(reqs)
    dt = time.perf_counter() - t0
    for r, o in zip(reqs, outs):
        print("%3d prompt tokens ->" % len(r.prompt), o)
    print("%d tokens in %.2f s" % (sum(map(len, outs)), dt))


if __name__ == "__main__":
    main()
