"""What one serving step of several requests does around the packed projections, as measurable cases.

Four operators over a quantized paged KV pool (int8 or int4 codes, one float32 scale per token and KV head):

  write   per-head RMSNorm of queries and keys, RoPE, and the quantizing write of the K and V rows into their pages;
          then the rows handed back as the pool holds them (write + read)
  read    whole sequences read back from the pool
  attend  attention of each sequence's new rows (one for a decode step, many for a prompt chunk) over its pages, with
          an optional tanh cap, distance bias, sliding window and prefix
  logits  repetition / frequency / presence penalties, token biases and a grammar bit mask, and the argmax

With `own` false `run` computes them from elementary torch operations in 32 bits; with `own` true it calls the
framework. The pool is one block of bytes per (page, KV head): K codes | V codes | K scales | V scales.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lumina-studio_b200")
DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16}


def _serving():
    if _PKG not in sys.path:
        sys.path.insert(1, _PKG)
    from lumina_b200 import serving
    return serving


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
_SEQ = {"op": "attend", "bits": 8, "io": "f16", "n_seq": 1, "rows": 1, "row_kind": "all", "len_max": 1024, "ragged": False,
        "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "norm": False, "cap": 0.0, "alibi": False,
        "window": 0, "prefix": 0, "sizes": 1}
_LOG = {"op": "logits", "rows": 1, "vocab": 32000, "history": 64, "biases": 8, "grammar": True, "sizes": 1}


def _seq(name, **kw):
    return dict(_SEQ, name=name, **kw)


def listed():
    return [
        # a decode step of 64 requests, one row each: what every layer writes per token (latency counts)
        _seq("write_decode_64x1", op="write", bits=4, n_seq=64, rows=1, len_max=4096, ragged=True),
        # prompts of three requests arriving together, with query / key norms: a prefill's write of one layer
        _seq("write_prompts_norm", op="write", bits=8, io="f32", n_seq=3, rows=2731, row_kind="ragged", len_max=6000,
             ragged=True, norm=True, heads=32, kv_heads=32),
        # a short cached prefix of the 7B head layout handed to another consumer
        _seq("read_prefix_f32", op="read", bits=8, io="f32", n_seq=1, rows=513, len_max=513, kv_heads=32),
        # eight cached conversations read back whole (moving sequences between pools)
        _seq("read_8_sequences", op="read", bits=4, n_seq=8, rows=8192, row_kind="whole", len_max=8192, ragged=True),
        # one request decoding at the benchmark's cache length, 7B heads: the smallest call
        _seq("decode_1x640_mha", bits=8, io="f32", len_max=640, kv_heads=32),
        # a serving batch: 64 requests of very different lengths, shared KV heads
        _seq("decode_64_ragged", bits=8, n_seq=64, len_max=8192, ragged=True, page=32),
        # two long documents, one token each
        _seq("decode_2x128k_int4", bits=4, n_seq=2, len_max=131072, kv_heads=4, page=64),
        # drafted rows of several requests scored at once, capped scores
        _seq("drafts_8x5_capped", bits=8, n_seq=8, rows=5, len_max=4097, ragged=True, cap=50.0),
        # a mixed batch: one prompt chunk beside decoding requests; distance bias, window and prefix; fp32 rows
        _seq("mixed_chunk_bias", bits=4, io="f32", n_seq=17, rows=301, row_kind="first", len_max=4096, ragged=True,
             head_dim=64, heads=28, kv_heads=4, alibi=True, window=1500, prefix=37, cap=30.0),
        # the largest: a 2048-row prompt chunk behind 14K cached tokens
        _seq("chunk_2048_of_16k", bits=8, rows=2048, len_max=16384),
        # one request's next token over the 7B vocabulary
        dict(_LOG, name="logits_1x32000"),
        # a large batch over a large vocabulary, long histories
        dict(_LOG, name="logits_256x131072", rows=256, vocab=131072, history=3000, biases=24),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.2:
        rows = _log(rng, 1, 200)
        return dict(_LOG, rows=rows, vocab=rng.randint(4000, 131072), history=_log(rng, 1, 3000),
                    biases=rng.randint(0, 24), grammar=rng.random() < 0.6, sizes=rng.randint(1, 9999))
    c = dict(_SEQ, op=rng.choice(["write", "read", "attend", "attend", "attend"]), bits=rng.choice([8, 8, 4]),
             io=rng.choice(["f16", "f16", "f32"]), page=rng.choice([16, 16, 32, 64]), ragged=True,
             head_dim=rng.choice([64, 128, 128]), sizes=rng.randint(1, 9999))
    c["heads"], c["kv_heads"] = rng.choice([(32, 32), (32, 8), (32, 4), (28, 4), (14, 2), (4, 4)])
    if c["op"] == "write":
        c["norm"] = rng.random() < 0.5
        c["n_seq"] = _log(rng, 1, 100)
        c["rows"] = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 6000 // c["n_seq"]))
        c["row_kind"] = "ragged" if c["rows"] > 1 else "all"
        c["len_max"] = max(c["rows"] + 1, _log(rng, 50, 8192))
    elif c["op"] == "read":
        c["n_seq"] = _log(rng, 1, 16)
        c["rows"] = c["len_max"] = _log(rng, 30, 8000)
        c["row_kind"] = "whole"
    else:
        kind = rng.choice(["decode", "decode", "drafts", "first", "all"])
        c["row_kind"] = "first" if kind == "first" else "all"
        c["n_seq"] = 1 if kind == "all" else _log(rng, 1, 64 if kind == "decode" else 16)
        c["rows"] = {"decode": 1, "drafts": rng.randint(2, 33), "first": _log(rng, 40, 400), "all": _log(rng, 100, 2000)}[kind]
        c["len_max"] = _log(rng, c["rows"] + 1, 65536 // c["n_seq"] if kind == "decode" else 8000 // min(4, c["n_seq"]))
        c["cap"] = rng.choice([0.0, 0.0, 30.0])
        c["alibi"] = rng.random() < 0.25
        c["window"] = rng.choice([0, 0, rng.randint(1, 2000)])
        c["prefix"] = rng.choice([0, 0, rng.randint(1, 100)])
    return c


def _sizes(c):
    """(rows, lengths) of every sequence: plain ints from the case alone."""
    r = random.Random(c["sizes"])
    n, m, top = c["n_seq"], c["rows"], c["len_max"]
    kind = c["row_kind"]
    lens = [top] + [int(top * math.exp(-2.8 * r.random())) if c["ragged"] else top for _ in range(n - 1)]
    rows = [m] + [1 if kind == "first" else max(1, int(m * r.random())) if kind == "ragged" else m for _ in range(n - 1)]
    if kind == "whole":
        lens = [max(1, x) for x in lens]
        return list(lens), lens
    return rows, [max(a, b) for a, b in zip(rows, lens)]


def _visible(c):
    """(visible (query, key) pairs, keys that some row sees) per sequence, summed."""
    pairs = keys = 0
    for n, ln in zip(*_sizes(c)):
        p = np.arange(ln - n, ln)
        lo = np.maximum(0, p - c["window"] + 1) if c["window"] else np.zeros(n, np.int64)
        pre = min(c["prefix"], ln)
        pairs += int((p + 1 - lo + pre - np.maximum(0, np.minimum(p + 1, pre) - lo)).sum())
        keys += ln - int(lo[0]) + min(pre, int(lo[0]))
    return pairs, keys


def work(c):
    if c["op"] == "logits":
        n = c["rows"] * c["vocab"]
        extra = c["rows"] * (4 * c["history"] + 8 * c["biases"] + 12)
        return {"bytes": 8 * n + (n // 8 if c["grammar"] else 0) + extra, "flops": n}
    rows, lens = _sizes(c)
    el, hd = DTYPES[c["io"]].itemsize, c["head_dim"]
    n, kv_row = sum(rows), c["kv_heads"] * 2 * (hd * c["bits"] // 8 + 4)
    dense = n * c["kv_heads"] * 2 * hd * el
    if c["op"] == "write":
        q = n * c["heads"] * hd * el
        return {"bytes": 2 * q + dense + n * hd * 4 + 2 * n * kv_row + dense, "flops": 8 * n * (c["heads"] + 2 * c["kv_heads"]) * hd}
    if c["op"] == "read":
        return {"bytes": n * kv_row + dense, "flops": 2 * n * c["kv_heads"] * hd}
    pairs, keys = _visible(c)
    return {"bytes": keys * kv_row + 2 * n * c["heads"] * hd * el, "flops": 4 * pairs * c["heads"] * hd}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _block_bytes(c):
    return c["page"] * (2 * c["head_dim"] * c["bits"] // 8 + 8)


def _fill_pool(c, n_pages, g):
    """A pool whose every row holds a quantized normal row, with the spread of magnitudes that tokens have."""
    P, hd, nb = c["page"], c["head_dim"], c["head_dim"] * c["bits"] // 8
    pool = torch.empty(n_pages, c["kv_heads"], _block_bytes(c), dtype=torch.uint8, device=DEV)
    step = max(1, (64 << 20) // (c["kv_heads"] * P * hd))
    for a in range(0, n_pages, step):
        b = min(n_pages, a + step)
        for i in (0, 1):
            x = torch.randn(b - a, c["kv_heads"], P, hd, device=DEV, generator=g)
            amp = torch.exp(0.3 * torch.randn(b - a, c["kv_heads"], P, 1, device=DEV, generator=g))
            top = x.abs().amax(-1, keepdim=True)
            if c["bits"] == 8:
                codes = torch.round(x * (127 / top)).to(torch.int8).view(torch.uint8)
            else:
                u = torch.round(x * (7.5 / top) + 7.5).clamp_(0, 15).to(torch.uint8)
                codes = u[..., 0::2] | (u[..., 1::2] << 4)
            scale = (top * amp / (127 if c["bits"] == 8 else 15)).reshape(b - a, c["kv_heads"], P)
            pool[a:b, :, i * P * nb:(i + 1) * P * nb] = codes.reshape(b - a, c["kv_heads"], P * nb)
            at = 2 * P * nb + 4 * P * i
            pool[a:b, :, at:at + 4 * P] = scale.contiguous().view(torch.uint8)
    return pool


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if c["op"] == "logits":
        R, V, H, B = c["rows"], c["vocab"], c["history"], c["biases"]
        # histories: tokens repeat, as generated text does; every row has its own length
        hl = [max(0, H - (i * 7) % (H // 2 + 1)) for i in range(R)]
        hs = torch.tensor(np.concatenate([[0], np.cumsum(hl)]), dtype=torch.int32, device=DEV)
        ht = (torch.rand(max(1, sum(hl)), device=DEV, generator=g) ** 4 * V).to(torch.int32)
        base = torch.randint(0, V, (R, 1), device=DEV, generator=g)
        at = torch.arange(B, device=DEV)[None] * 131
        s = {"c": c, "logits": 3 * torch.randn(R, V, device=DEV, generator=g), "hist_start": hs, "hist_tok": ht,
             "repeat": 1 + 0.3 * torch.rand(R, device=DEV, generator=g),
             "freq": 0.2 * torch.rand(R, device=DEV, generator=g), "pres": 0.5 * torch.rand(R, device=DEV, generator=g),
             "bias_start": torch.arange(0, R * B + 1, max(1, B), dtype=torch.int32, device=DEV)[:R + 1] if B else
             torch.zeros(R + 1, dtype=torch.int32, device=DEV),
             "bias_tok": ((base + at) % V).to(torch.int32).reshape(-1),
             "bias_val": 4 * torch.randn(R * B, device=DEV, generator=g), "mask": None,
             "out": torch.empty(R, V, device=DEV), "argmax": torch.empty(R, dtype=torch.int32, device=DEV)}
        if c["grammar"]:  # every other row is constrained: about 1 token in 16 stays
            w = (V + 31) // 32
            m = torch.randint(-2**31, 2**31, (4, R, w), device=DEV, generator=g, dtype=torch.int64).to(torch.int32)
            m = m[0] & m[1] & m[2] & m[3]
            m[1::2] = -1
            s["mask"] = m
        return s
    rows, lens = _sizes(c)
    n, S, P = sum(rows), c["n_seq"], c["page"]
    need = [(x + P - 1) // P for x in lens]
    n_pages, ld = sum(need) + 3, max(need)
    perm = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    first = torch.tensor(np.concatenate([[0], np.cumsum(need)[:-1]]), device=DEV)
    col = torch.arange(ld, device=DEV)[None]
    table = torch.where(col < torch.tensor(need, device=DEV)[:, None], perm[(first[:, None] + col).clamp_(max=n_pages - 1)], 0)
    dt, hd, nh, nk = DTYPES[c["io"]], c["head_dim"], c["heads"], c["kv_heads"]
    s = {"c": c, "row_start": torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device=DEV),
         "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "pages": table.to(torch.int32).contiguous(),
         "n_rows": n, "max_rows": max(rows), "max_len": max(lens)}
    if c["op"] == "write":
        s["pool"] = torch.randint(0, 256, (n_pages, nk, _block_bytes(c)), dtype=torch.uint8, device=DEV, generator=g)
        # one fused projection's rows: q, k and v are column ranges of them
        qkv = torch.randn(n, (nh + 2 * nk) * hd, device=DEV, generator=g)
        qkv *= torch.exp(0.3 * torch.randn(n, 1, device=DEV, generator=g))
        s["qkv"] = qkv.to(dt)
        ang = torch.arange(max(lens), device=DEV, dtype=torch.float32)[:, None] * (
            1.0 / (10000.0 ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float32) / hd)))[None]
        s["cos"], s["sin"] = torch.cos(ang), torch.sin(ang)
        s["q_norm"] = s["k_norm"] = None
        if c["norm"]:
            s["q_norm"] = 1 + 0.1 * torch.randn(hd, device=DEV, generator=g)
            s["k_norm"] = 1 + 0.1 * torch.randn(hd, device=DEV, generator=g)
        s["q_out"] = torch.empty(n, nh, hd, dtype=dt, device=DEV)
    else:
        s["pool"] = _fill_pool(c, n_pages, g)
    if c["op"] in ("write", "read"):
        s["k_out"], s["v_out"] = (torch.empty(n, nk, hd, dtype=dt, device=DEV) for _ in range(2))
    if c["op"] == "attend":
        s["q"] = (2 * torch.randn(n, nh, hd, device=DEV, generator=g)).to(dt)
        s["out"] = torch.empty(n, nh, hd, dtype=dt, device=DEV)
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, nh + 1, device=DEV) / nh).float() if c["alibi"] else None
        s["prefix"] = None
        if c["prefix"]:
            s["prefix"] = torch.tensor([c["prefix"]] * S, dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _run_own(s):
    c, sv = s["c"], _serving()
    if c["op"] == "logits":
        return sv.adjust_logits(s["logits"], history=(s["hist_start"], s["hist_tok"]), repeat=s["repeat"],
                                frequency=s["freq"], presence=s["pres"],
                                bias=(s["bias_start"], s["bias_tok"], s["bias_val"]) if c["biases"] else None,
                                mask=s["mask"], out=s["out"], argmax=s["argmax"])
    pool = sv.KVPool(s["pool"], bits=c["bits"], head_dim=c["head_dim"], page_size=c["page"])
    batch = sv.SeqBatch(s["row_start"], s["lens"], s["pages"], n_rows=s["n_rows"], max_rows=s["max_rows"])
    if c["op"] == "write":
        hd, a, b = c["head_dim"], c["heads"] * c["head_dim"], (c["heads"] + c["kv_heads"]) * c["head_dim"]
        qkv = s["qkv"]
        q = pool.append(batch, qkv[:, :a], qkv[:, a:b], qkv[:, b:], s["cos"], s["sin"], q_norm=s["q_norm"],
                        k_norm=s["k_norm"], eps=1e-6, out=s["q_out"])
        return (q, *pool.read(batch, out=(s["k_out"], s["v_out"])))
    if c["op"] == "read":
        return pool.read(batch, out=(s["k_out"], s["v_out"]))
    return pool.attend(batch, s["q"], softcap=c["cap"], slopes=s["slopes"], window=c["window"], prefix=s["prefix"],
                       out=s["out"])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _row_maps(s):
    """Sequence, index within it and position of every row of the batch."""
    starts = s["row_start"].long()
    r = torch.arange(s["n_rows"], device=DEV)
    seq = torch.searchsorted(starts[1:], r, right=True)
    i = r - starts[seq]
    pos = s["lens"].long()[seq] - (starts[seq + 1] - starts[seq]) + i
    return seq, i, pos


def _sections(s):
    c, P = s["c"], s["c"]["page"]
    nb = c["head_dim"] * c["bits"] // 8
    pool = s["pool"]
    codes = [pool[..., i * P * nb:(i + 1) * P * nb].unflatten(-1, (P, nb)) for i in (0, 1)]
    scales = [pool[..., 2 * P * nb + 4 * P * i:2 * P * nb + 4 * P * (i + 1)].view(torch.float32) for i in (0, 1)]
    return codes, scales


def _values(s, which, seq, pos):
    """float32 rows of K (0) or V (1): shape seq.shape + (kv_heads, head_dim)."""
    c = s["c"]
    codes, scales = _sections(s)
    page = s["pages"].long()[seq, pos // c["page"]]
    b = codes[which][page, :, pos % c["page"]]
    if c["bits"] == 8:
        x = b.view(torch.int8).float()
    else:
        x = torch.stack((b & 15, b >> 4), -1).flatten(-2).float() * 2 - 15
    return x * scales[which][page, :, pos % c["page"]].unsqueeze(-1)


def _pair_sum(x):
    """Sum over the last axis (a power of two) by halves, then neighbours: one fixed order."""
    h = x.shape[-1] // 2
    x = x[..., :h] + x[..., h:]
    x = x[..., 0::2] + x[..., 1::2]
    x = x[..., 0::2] + x[..., 1::2]
    x = x[..., 0::2] + x[..., 1::2]
    x = x[..., 0::2] + x[..., 1::2]
    x = x[..., 0::2] + x[..., 1::2]
    return x[..., 0:1] + x[..., 1:2] if x.shape[-1] == 2 else x


def _norm_rope(x, w, cos, sin):
    if w is not None:
        x = (x * (1.0 / torch.sqrt(_pair_sum(x * x) / x.shape[-1] + 1e-6))) * w
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _store(s, which, x, seq, pos):
    c = s["c"]
    codes, scales = _sections(s)
    top = x.abs().amax(-1, keepdim=True)
    page, off = s["pages"].long()[seq, pos // c["page"]], pos % c["page"]
    if c["bits"] == 8:
        q = torch.round(x * (torch.reciprocal(top) * 127.0)).to(torch.int8).view(torch.uint8)
        scale = top * (1.0 / 127.0)
    else:
        u = torch.round(x * (torch.reciprocal(top) * 7.5) + 7.5).clamp_(0, 15).to(torch.uint8)
        q = u[..., 0::2] | (u[..., 1::2] << 4)
        scale = top * (1.0 / 15.0)
    codes[which][page, :, off] = q
    scales[which][page, :, off] = scale.squeeze(-1)


def _plain_write(s):
    c, hd = s["c"], s["c"]["head_dim"]
    seq, _, pos = _row_maps(s)
    x = s["qkv"].float().unflatten(-1, (-1, hd))
    q, k, v = x.split((c["heads"], c["kv_heads"], c["kv_heads"]), 1)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    _store(s, 0, _norm_rope(k, s["k_norm"], cos, sin), seq, pos)
    _store(s, 1, v, seq, pos)
    dt = DTYPES[c["io"]]
    return _norm_rope(q, s["q_norm"], cos, sin).to(dt), _values(s, 0, seq, pos).to(dt), _values(s, 1, seq, pos).to(dt)


def _plain_attend(s):
    c = s["c"]
    S, n, L, nk, hd = c["n_seq"], s["max_rows"], s["max_len"], c["kv_heads"], c["head_dim"]
    G = c["heads"] // nk
    starts, lens = s["row_start"].long(), s["lens"].long()
    count = starts[1:] - starts[:-1]
    i, j = torch.arange(n, device=DEV), torch.arange(L, device=DEV)
    q = s["q"][(starts[:-1, None] + torch.minimum(i[None], count[:, None] - 1))].float()  # (S, n, heads, hd)
    p = (lens - count)[:, None, None] + i[None, :, None]
    d = p - j
    see = d >= 0
    if c["window"]:
        see = see & (d < c["window"])
    if s["prefix"] is not None:
        see = see | (j < s["prefix"][:, None, None])
    see = (see & (j < lens[:, None, None]))[:, None, None]  # (S, 1, 1, n, L)
    where = torch.minimum(j[None], lens[:, None] - 1)
    at = torch.arange(S, device=DEV)[:, None].expand(S, L)
    k = _values(s, 0, at, where).permute(0, 2, 3, 1).unsqueeze(2)  # (S, nk, 1, hd, L)
    x = torch.matmul(q.unflatten(2, (nk, G)).permute(0, 2, 3, 1, 4), k) * (1.0 / math.sqrt(hd))
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    if s["slopes"] is not None:
        x = x - s["slopes"].view(nk, G, 1, 1) * d.abs().float()[:, None, None]
    x = x.masked_fill(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = x.sum(-1, keepdim=True)
    v = _values(s, 1, at, where).permute(0, 2, 1, 3).unsqueeze(2)  # (S, nk, 1, L, hd)
    o = torch.matmul(x, v) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
    seq, i, _ = _row_maps(s)
    return o[seq, i].to(DTYPES[c["io"]])


def _plain_logits(s):
    c, l = s["c"], s["logits"]
    R, V = l.shape
    n = int(s["hist_tok"].numel())
    row = torch.searchsorted(s["hist_start"][1:].contiguous(), torch.arange(n, device=DEV, dtype=torch.int32), right=True)
    ok = row < R
    count = torch.zeros(R * V, device=DEV)
    count.scatter_add_(0, torch.where(ok, row * V + s["hist_tok"].long(), 0), ok.float())
    count = count.view(R, V)
    seen = count > 0
    r = s["repeat"][:, None]
    x = torch.where(seen, torch.where(l > 0, l / r, l * r), l)
    x = torch.where(seen, x - s["freq"][:, None] * count - s["pres"][:, None], x)
    if c["biases"]:
        add = torch.zeros(R, V, device=DEV)
        add[torch.arange(R, device=DEV).repeat_interleave(c["biases"]), s["bias_tok"].long()] = s["bias_val"]
        x = x + add
    if s["mask"] is not None:
        v = torch.arange(V, device=DEV)
        x = torch.where((s["mask"][:, v // 32] >> (v % 32)) & 1 == 1, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(V, device=DEV), V).amin(-1)
    return x, first.to(torch.int32)


def run(state):
    if own:
        return _run_own(state)
    op = state["c"]["op"]
    if op == "write":
        return _plain_write(state)
    if op == "attend":
        return _plain_attend(state)
    if op == "logits":
        return _plain_logits(state)
    seq, _, pos = _row_maps(state)
    dt = DTYPES[state["c"]["io"]]
    return _values(state, 0, seq, pos).to(dt), _values(state, 1, seq, pos).to(dt)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _host_rows(s, b, lo, hi):
    """(K, V) of tokens [lo, hi) of sequence b in float64, (hi - lo, kv_heads, head_dim)."""
    c = s["c"]
    P, hd, nb = c["page"], c["head_dim"], c["head_dim"] * c["bits"] // 8
    blk = s["pool"][s["pages"][b, lo // P:(hi + P - 1) // P].long()]  # (pages, kv_heads, bytes)
    out = []
    for i in (0, 1):
        raw = blk[:, :, i * P * nb:(i + 1) * P * nb].reshape(blk.shape[0], -1, P, nb)
        if c["bits"] == 8:
            x = raw.contiguous().view(torch.int8).double()
        else:
            x = torch.empty(*raw.shape[:-1], hd, dtype=torch.float64, device=DEV)
            x[..., 0::2] = 2 * (raw % 16).double() - 15
            x[..., 1::2] = 2 * (raw // 16).double() - 15
        a = 2 * P * nb + 4 * P * i
        x *= blk[:, :, a:a + 4 * P].contiguous().view(torch.float32).double()[..., None]
        out.append(x.transpose(1, 2).reshape(-1, x.shape[1], hd)[lo % P:lo % P + hi - lo])
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "logits":
        x = s["logits"].double()
        hs = s["hist_start"].tolist()
        for r in range(c["rows"]):
            tok, n = torch.unique(s["hist_tok"][hs[r]:hs[r + 1]].long(), return_counts=True)
            l, rp = x[r, tok], s["repeat"][r].double()
            l = torch.where(l > 0, l / rp, l * rp) - s["freq"][r].double() * n - s["pres"][r].double()
            x[r, tok] = l
            if c["biases"]:
                b = slice(r * c["biases"], (r + 1) * c["biases"])
                x[r, s["bias_tok"][b].long()] += s["bias_val"][b].double()
            if s["mask"] is not None:
                bits = s["mask"][r][:, None].bitwise_right_shift(torch.arange(32, device=DEV, dtype=torch.int32)) & 1
                x[r][bits.reshape(-1)[:c["vocab"]] == 0] = -math.inf
        return x, None
    rows, lens = _sizes(c)
    hd, nh, nk = c["head_dim"], c["heads"], c["kv_heads"]
    if c["op"] == "read":
        got = [_host_rows(s, b, ln - n, ln) for b, (n, ln) in enumerate(zip(rows, lens))]
        return tuple(torch.cat([x[i] for x in got]) for i in (0, 1))
    at, outs = 0, []
    for b, (n, ln) in enumerate(zip(rows, lens)):
        pos = torch.arange(ln - n, ln, device=DEV)
        if c["op"] == "write":
            x = s["qkv"][at:at + n].double().view(n, nh + 2 * nk, hd)
            q, k, v = x[:, :nh], x[:, nh:nh + nk], x[:, nh + nk:]
            if c["norm"]:
                q = q / (q.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s["q_norm"].double()
                k = k / (k.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s["k_norm"].double()
            z = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            q, k = (torch.complex(t[..., :hd // 2], t[..., hd // 2:]) * z for t in (q, k))
            q, k = (torch.cat((t.real, t.imag), -1) for t in (q, k))
            res = [q]
            for t in (k, v):
                m = t.abs().amax(-1, keepdim=True)
                res.append(torch.round(t / m * 127) * (m / 127) if c["bits"] == 8 else
                           (2 * torch.round(t / m * 7.5 + 7.5).clamp(0, 15) - 15) * (m / 15))
            outs.append(res)
        else:
            k, v = _host_rows(s, b, 0, ln)
            j = torch.arange(ln, device=DEV)
            d = pos[:, None] - j[None]
            hide = d < 0
            if c["window"]:
                hide = hide | (d >= c["window"])
            hide = hide & (j >= c["prefix"])[None]
            o = torch.zeros(n, nh, hd, dtype=torch.float64, device=DEV)
            for h in range(nh):
                x = s["q"][at:at + n, h].double() @ k[:, h * nk // nh].T / math.sqrt(hd)
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                if c["alibi"]:
                    x = x - s["slopes"][h].double() * d.abs()
                o[:, h] = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ v[:, h * nk // nh]
            outs.append([o])
        at += n
    done = tuple(torch.cat([x[i] for x in outs]) for i in range(len(outs[0])))
    return done[0] if c["op"] == "attend" else done
