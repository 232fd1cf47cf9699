"""The quantized-page operators and the logits operator on a B200, against
their float64 definitions (serving_ref.py).

Tolerances, from the arithmetic alone:
  * read: one fp32 product (and one fp16 rounding) -- exact.
  * append: fp32 norm and rotation (about ten roundings of 2^-24 relative to
    the row's largest value), so a code may differ from the float64 one only
    where the unrounded code lies within 127 * 10 * 2^-24 < 2e-4 of a tie;
    scales and fp32 queries agree to 2e-6, fp16 queries to 2^-11.
  * attend, fp32 rows: scores, probabilities and sums carry about 22 bits
    (2^-22 = 2.4e-7 per product, scores up to 2^5): 1e-5 of the output's
    norm. fp16 rows: p and the output are rounded to fp16 (2^-12 rms each):
    1e-3.
  * logits: three fp32 roundings of values of the size of the logit and its
    penalties: 1e-6 of the largest term; the argmax is exact for the row as
    returned.
"""
import numpy as np
import pytest

import serving_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sv():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    from lumina_b200 import cuda, serving
    cuda.ensure_device(0)
    cuda.fault_status(0)
    return serving


@pytest.fixture(autouse=True)
def no_fault(sv):
    from lumina_b200 import cuda
    yield
    assert cuda.fault_status(0) == 0


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def random_pool(rng, n_pages, n_kv, bits, hd, page, poison=None):
    """A pool of random codes and positive scales; pages outside ``poison``
    are usable, every scale of the pages in it is NaN."""
    pool = rng.integers(0, 256, (n_pages, n_kv, ref.block_bytes(bits, hd, page)), dtype=np.uint8)
    if bits == 8:  # -128 is no code
        codes = pool[:, :, :2 * page * hd]
        codes[codes == 128] = 129
    nb = hd * bits // 8
    s = (np.exp(0.4 * rng.standard_normal((n_pages, n_kv, 2 * page))) * (1 / 64 if bits == 8 else 1 / 8)).astype(np.float32)
    if poison is not None:
        s[poison] = np.nan
    pool[:, :, 2 * page * nb:] = s.view(np.uint8)
    return pool


def layout(rng, lens, page, spare=3):
    """A page table over shuffled pages: (table (n, ld), n_pages, unused)."""
    need = [-(-max(x, 0) // page) for x in lens]
    n_pages = sum(need) + spare
    perm = rng.permutation(n_pages)
    ld = max(need + [1])
    table = np.zeros((len(lens), ld), np.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = perm[at:at + k]
        table[i, k:] = perm[-1]  # a page nobody owns
        at += k
    return table, n_pages, perm[at:]


def batch_of(sv, rows, lens, table, max_rows=None):
    rs = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    return sv.SeqBatch(dev(rs), dev(np.asarray(lens, np.int32)), dev(table), int(rs[-1]),
                       max(rows) if max_rows is None else max_rows)


def poison_tail(pool, table, lens, bits, hd, page):
    """NaN scales at every token past a sequence's length."""
    nb = hd * bits // 8
    s = pool[:, :, 2 * page * nb:].copy().view(np.float32).reshape(*pool.shape[:2], 2, page)
    for row, ln in zip(table, lens):
        for t in range(ln, -(-ln // page) * page):
            s[row[t // page], :, :, t % page] = np.nan
    pool[:, :, 2 * page * nb:] = s.reshape(*pool.shape[:2], 2 * page).view(np.uint8)


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30)


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,io", [(128, "float32"), (128, "float16"), (64, "float32"), (64, "float16")])
@pytest.mark.parametrize("heads,n_kv,page,norm,rows,lens", [
    (4, 4, 16, False, [1, 1, 1], [1, 16, 17]),
    (8, 2, 32, True, [5, 0, 33, 1], [5, 40, 70, 64]),
    (14, 2, 64, True, [70], [200]),
    (9, 3, 128, False, [0, 2, 0, 0, 130, 0], [0, 2, 7, 0, 257, 0]),
])
def test_append(sv, bits, hd, io, heads, n_kv, page, norm, rows, lens):
    import torch
    rng = np.random.default_rng(bits * 1000 + hd + heads)
    dt = getattr(torch, io)
    table, n_pages, _ = layout(rng, lens, page)
    before = random_pool(rng, n_pages, n_kv, bits, hd, page)
    pool = sv.KVPool(dev(before), bits, hd, page)
    n = sum(rows)
    qkv = rng.standard_normal((n, (heads + 2 * n_kv) * hd + 8)).astype(np.float32) * np.exp(rng.standard_normal((n, 1)))
    qkv = dev(qkv.astype(np.float32), dt)
    x = qkv.float().cpu().numpy().astype(np.float64)
    a, b = heads * hd, (heads + n_kv) * hd
    ang = np.arange(max(lens) + 1)[:, None] * (1e4 ** (-np.arange(0, hd, 2) / hd))[None]
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qw, kw = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32) if norm else (None, None)
    batch = batch_of(sv, rows, lens, table)
    q = pool.append(batch, qkv[:, :a], qkv[:, a:b], qkv[:, b:b + n_kv * hd], dev(cos), dev(sin),
                    q_norm=None if qw is None else dev(qw), k_norm=None if kw is None else dev(kw), eps=1e-6)
    k_read, v_read = pool.read(batch, dtype=dt)
    after = pool.data.cpu().numpy()
    pos = np.concatenate([np.arange(ln - m, ln) for m, ln in zip(rows, lens)]).astype(int)
    seq = np.repeat(np.arange(len(rows)), rows)
    c, s = cos[pos].astype(np.float64), sin[pos].astype(np.float64)
    want_q = ref.norm_rope(x[:, :a].reshape(n, heads, hd), qw, c, s, 1e-6)
    assert rel(q.float().cpu().numpy(), want_q) < (2e-6 if io == "float32" else 2.0 ** -11)
    want = [ref.norm_rope(x[:, a:b].reshape(n, n_kv, hd), kw, c, s, 1e-6), x[:, b:b + n_kv * hd].reshape(n, n_kv, hd)]
    got = ref.split_block(after, bits, hd, page)
    pg, off = table[seq, pos // page], pos % page
    for w, (codes, scales), r in zip(want, got, (k_read, v_read)):
        amax = np.abs(w).max(-1)
        top = 127 if bits == 8 else 15
        sc = scales[pg, :, off].astype(np.float64)
        assert np.abs(sc / (amax / top) - 1).max() < 2e-6
        real = w / (amax / top)[..., None]  # the code before rounding (int4: an odd number 2 c - 15)
        step = 1 if bits == 8 else 2
        assert (np.abs(codes[pg, :, off] - real) <= step * (0.5 + 2e-4)).all()
        exact = (codes[pg, :, off].astype(np.float32) * scales[pg, :, off][..., None])
        assert np.array_equal(r.cpu().numpy(), exact if io == "float32" else exact.astype(np.float16))
    # nothing else in the pool changed
    same = ref.split_block(before, bits, hd, page)
    for (ca, sa), (cb, sb) in zip(got, same):
        ca, cb, sa, sb = ca.copy(), cb.copy(), sa.copy(), sb.copy()
        for arr in (ca, cb, sa, sb):
            arr[pg, :, off] = 0
        assert np.array_equal(ca, cb) and np.array_equal(sa.view(np.uint32), sb.view(np.uint32))


@pytest.mark.parametrize("bits", [8, 4])
def test_append_special_rows(sv, bits):
    """Zero rows, rows below 2^-100, infinities and NaN, ties at half codes."""
    hd, page, n = 64, 16, 6
    x = np.zeros((n, 1, hd), np.float32)
    x[0] = 0.0
    x[1] = 1e-35
    x[2, 0, 5] = np.inf
    x[3, 0, 7] = np.nan
    x[4, 0, :4] = [127.0, 0.5, 1.5, -2.5] if bits == 8 else [7.5, 0.0, 1.0, -1.0]  # ties of the codes
    x[5] = np.float32(3e38)
    table = np.zeros((1, 1), np.int32)
    pool = sv.KVPool.empty(1, 1, hd, bits, page)
    one = np.ones((n, hd // 2), np.float32)
    batch = batch_of(sv, [n], [n], table)
    xd = dev(x)
    pool.append(batch, xd, xd, xd, dev(one), dev(0 * one))
    (kc, ks), (vc, vs) = ref.split_block(pool.data.cpu().numpy(), bits, hd, page)
    for c, s in ((kc, ks), (vc, vs)):
        c, s = c[0, 0], s[0, 0]
        assert s[0] == 0 and s[1] == 0 and np.isnan(s[2]) and np.isnan(s[3])
        want = [127, 0, 2, -2] if bits == 8 else [15, 1, 1, -3]  # int4: codes 15, rint(7.5), rint(8.5), rint(6.5)
        assert list(c[4, :4]) == want
        assert np.isfinite(s[5]) and (c[5] == (127 if bits == 8 else 15)).all()
    k, v = pool.read(batch)
    assert (k[:2] == 0).all() and k[2:4].isnan().all() and v[2:4].isnan().all()


# ---------------------------------------------------------------------------
# attend
# ---------------------------------------------------------------------------
def run_attend(sv, bits, hd, io, heads, n_kv, page, rows, lens, cap=0.0, alibi=False, window=0, prefix=None, seed=0,
               scale=0.0, max_rows=None, qmul=2.0):
    import torch
    rng = np.random.default_rng(seed + 7 * hd + bits)
    dt = getattr(torch, io)
    table, n_pages, unused = layout(rng, lens, page)
    pool = random_pool(rng, n_pages, n_kv, bits, hd, page, poison=unused)
    poison_tail(pool, table, lens, bits, hd, page)
    n = sum(rows)
    wide = dev((qmul * rng.standard_normal((n, heads * hd + 16))).astype(np.float32), dt)
    q = wide[:, :heads * hd]
    slopes = (2.0 ** (-8 * np.arange(1, heads + 1) / heads)).astype(np.float32) if alibi else None
    batch = batch_of(sv, rows, lens, table, max_rows)
    p = sv.KVPool(dev(pool), bits, hd, page)
    out = p.attend(batch, q, scale=scale, softcap=cap, slopes=None if slopes is None else dev(slopes), window=window,
                   prefix=None if prefix is None else dev(np.asarray(prefix, np.int32)))
    again = p.attend(batch, q, scale=scale, softcap=cap, slopes=None if slopes is None else dev(slopes), window=window,
                     prefix=None if prefix is None else dev(np.asarray(prefix, np.int32)))
    assert torch.equal(out, again)  # no order of arrival in the sums
    got = out.float().cpu().numpy()
    qh = q.float().cpu().numpy().astype(np.float64).reshape(n, heads, hd)
    at, want = 0, np.zeros((n, heads, hd))
    for s, (m, ln) in enumerate(zip(rows, lens)):
        if m:
            k, v = ref.rows_of(pool, table[s], ln, bits, hd, page)
            want[at:at + m] = ref.attend(qh[at:at + m], k, v, ln, scale or hd ** -0.5, cap,
                                         None if slopes is None else slopes.astype(np.float64), window,
                                         0 if prefix is None else prefix[s])
        at += m
    return got, want


TOL = {"float32": 1e-5, "float16": 1e-3}


def check_attend(got, want, io):
    assert np.isfinite(got).all()
    assert rel(got, want) < TOL[io]
    # no row hides behind the others
    d = np.linalg.norm(got - want, axis=-1)
    assert (d <= 8 * TOL[io] * np.maximum(np.linalg.norm(want, axis=-1), 1e-3 * np.linalg.norm(want) / np.sqrt(want.shape[0] * want.shape[1]))).all()


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("heads,n_kv,page,rows,lens", [
    (4, 4, 16, [1], [1]),
    (4, 4, 16, [1, 1, 1, 1], [15, 16, 17, 640]),
    (8, 2, 32, [1, 0, 1, 1], [63, 100, 64, 65]),
    (14, 2, 64, [1] * 5, [2000, 3, 129, 1024, 511]),
    (16, 1, 128, [1, 1], [4097, 127]),
])
def test_attend_decode(sv, io, bits, hd, heads, n_kv, page, rows, lens):
    got, want = run_attend(sv, bits, hd, io, heads, n_kv, page, rows, lens)
    check_attend(got, want, io)


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("heads,n_kv,page,rows,lens", [
    (4, 4, 16, [17], [17]),
    (4, 2, 16, [128], [128]),
    (8, 2, 32, [5, 31, 1, 0, 300], [1000, 31, 64, 9, 813]),
    (14, 2, 64, [40, 37], [129, 700]),
    (32, 1, 16, [1, 9], [333, 500]),
    (128, 1, 128, [3], [260]),
    (2, 2, 16, [513], [1300]),
])
def test_attend_chunk(sv, io, bits, hd, heads, n_kv, page, rows, lens):
    got, want = run_attend(sv, bits, hd, io, heads, n_kv, page, rows, lens)
    check_attend(got, want, io)


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("hd,heads,n_kv", [(128, 8, 2), (64, 6, 2)])
@pytest.mark.parametrize("cap,alibi,window,prefix", [
    (20.0, False, 0, None),
    (0.0, True, 0, None),
    (0.0, False, 1, None),
    (0.0, False, 100, None),
    (30.0, True, 70, [3, 200, 0, 5, 1000]),
    (0.0, False, 64, [64, 65, 1, 0, 400]),
    (0.0, False, 0, [900, 0, 63, 7, 900]),  # a prefix past the rows: they see ahead
])
@pytest.mark.parametrize("rows,lens", [
    ([1, 1, 1, 1, 1], [1, 500, 64, 129, 900]),
    ([1, 33, 2, 1, 200], [700, 300, 64, 129, 900]),
])
def test_attend_masks(sv, io, hd, heads, n_kv, cap, alibi, window, prefix, rows, lens):
    got, want = run_attend(sv, 8, hd, io, heads, n_kv, 16, rows, lens, cap, alibi, window, prefix, seed=3)
    check_attend(got, want, io)


@pytest.mark.parametrize("io", ["float16", "float32"])
def test_attend_rows_that_see_nothing(sv, io):
    """Rows before the first token (a length shorter than the row count, an
    empty sequence): zeros, while their neighbours are as ever."""
    got, want = run_attend(sv, 8, 128, io, 4, 2, 16, [40, 1, 3, 1], [20, 0, 0, 33], seed=5)
    assert (want[:20] == 0).all() and (got[:20] == 0).all()
    assert (got[40:44] == 0).all()
    check_attend(got, want, io)


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("heads,n_kv,rows,lens,cap,alibi,window,prefix", [
    (8, 2, [5, 5, 5], [700, 5, 33], 0.0, False, 0, None),          # 20 packed rows: one and a quarter blocks of 16
    (16, 1, [4, 1, 0, 3], [129, 64, 50, 3], 20.0, False, 0, None),  # a row a block
    (12, 1, [5, 2], [400, 2], 0.0, True, 0, None),                  # blocks of one row of 12 heads
    (6, 2, [21, 7, 20], [300, 7, 4100], 0.0, False, 150, [0, 7, 40]),  # 63 packed rows, blocks of 5 rows of 3 heads
    (3, 3, [64, 16, 17], [64, 1500, 17], 30.0, True, 40, [9, 0, 17]),  # one head each: four blocks
    (14, 2, [90, 4, 1, 3], [700, 444, 2000, 3], 0.0, False, 100, [20, 0, 5, 0]),  # beside a chunk: blocks of 8
])
def test_attend_row_blocks(sv, io, heads, n_kv, rows, lens, cap, alibi, window, prefix):
    """Sequences whose rows are split over several tasks of one KV head."""
    got, want = run_attend(sv, 8, 64, io, heads, n_kv, 32, rows, lens, cap, alibi, window, prefix, seed=7)
    assert rel(got, want) < TOL[io]
    got, want = run_attend(sv, 4, 128, io, heads, n_kv, 16, rows, lens, cap, alibi, window, prefix, seed=8)
    assert rel(got, want) < TOL[io]


@pytest.mark.parametrize("rows", [1, 50])
def test_attend_long(sv, rows):
    got, want = run_attend(sv, 4, 64, "float32", 4, 1, 128, [rows], [20011], seed=11)
    check_attend(got, want, "float32")


@pytest.mark.parametrize("io,rows", [("float16", 1), ("float32", 1), ("float16", 80), ("float32", 80)])
def test_attend_nan_and_inf_stay_with_their_keys(sv, io, rows):
    """A key stored as NaN reaches the rows that see it and no others; a V
    row of huge values in a masked place does not disturb the rest."""
    import torch
    rng = np.random.default_rng(2)
    hd, page, heads, n_kv, ln, window = 128, 16, 4, 2, 200, 40
    dt = getattr(torch, io)
    table, n_pages, _ = layout(rng, [ln], page)
    pool = random_pool(rng, n_pages, n_kv, 8, hd, page)
    q = dev(rng.standard_normal((rows, heads * hd)).astype(np.float32), dt)
    batch = batch_of(sv, [rows], [ln], table)
    clean = sv.KVPool(dev(pool), 8, hd, page).attend(batch, q, window=window).float().cpu().numpy()
    nb = hd
    s = pool[:, :, 2 * page * nb:].copy().view(np.float32).reshape(n_pages, n_kv, 2, page)
    for t, val in ((30, 1e30), (ln - 1, np.nan)):  # key 30: only rows at positions 30..69 (none here with 80 rows: 120..)
        s[table[0, t // page], 0, :, t % page] = val
    pool[:, :, 2 * page * nb:] = s.reshape(n_pages, n_kv, 2 * page).view(np.uint8)
    got = sv.KVPool(dev(pool), 8, hd, page).attend(batch, q, window=window).float().cpu().numpy()
    # KV head 0 serves query heads 0 and 1; only the last row sees the last key
    assert np.isnan(got[-1, :2]).all()
    assert np.array_equal(got[-1, 2:], clean[-1, 2:])
    assert rel(got[:-1], clean[:-1]) < TOL[io] if rows > 1 else True


def test_attend_value_scales(sv):
    """Value rows of very different magnitudes (2^-40 .. 2^40 across
    sequences): the result scales with them."""
    import torch
    rng = np.random.default_rng(4)
    hd, page = 64, 16
    for e in (-40, 0, 40):
        for rows, io in ((1, "float16"), (1, "float32"), (70, "float32"), (70, "float16")):
            table, n_pages, _ = layout(rng, [150], page)
            pool = random_pool(np.random.default_rng(9), n_pages, 1, 8, hd, page)
            s = pool[:, :, 2 * page * hd:].copy().view(np.float32).reshape(n_pages, 1, 2, page)
            s[:, :, 1] *= np.float32(2.0) ** (e if io == "float32" else e // 8)
            pool[:, :, 2 * page * hd:] = s.reshape(n_pages, 1, 2 * page).view(np.uint8)
            q = dev(np.random.default_rng(10).standard_normal((rows, 2 * hd)).astype(np.float32), getattr(torch, io))
            got = sv.KVPool(dev(pool), 8, hd, page).attend(batch_of(sv, [rows], [150], table), q).float().cpu().numpy()
            k, v = ref.rows_of(pool, table[0], 150, 8, hd, page)
            want = ref.attend(q.float().cpu().numpy().astype(np.float64).reshape(rows, 2, hd), k, v, 150, hd ** -0.5)
            assert rel(got, want) < TOL[io], (e, rows, io)


# ---------------------------------------------------------------------------
# a step as it is used: streams, graphs, workspaces, out-of-range data
# ---------------------------------------------------------------------------
def test_decode_step_in_a_graph(sv):
    """append + attend captured once; lengths and rows rewritten in place
    between replays, as a decode loop does."""
    import torch
    rng = np.random.default_rng(6)
    hd, page, heads, n_kv, S = 128, 16, 8, 2, 3
    lens = np.array([5, 40, 100], np.int32)
    table, n_pages, _ = layout(rng, lens + 10, page)
    pool = sv.KVPool(dev(random_pool(rng, n_pages, n_kv, 8, hd, page)), 8, hd, page)
    batch = batch_of(sv, [1] * S, lens, table)
    lens_dev = batch._keep[1]
    cos, sin = (dev(f(np.arange(200)[:, None] * np.linspace(1, 0.01, hd // 2)[None]).astype(np.float32)) for f in (np.cos, np.sin))
    qkv = torch.empty(S, (heads + 2 * n_kv) * hd, device="cuda", dtype=torch.float16)
    out = torch.empty(S, heads, hd, device="cuda", dtype=torch.float16)
    q = torch.empty_like(out)
    ws = sv.attend_workspace(0)

    def step():
        pool.append(batch, qkv[:, :heads * hd], qkv[:, heads * hd:(heads + n_kv) * hd], qkv[:, (heads + n_kv) * hd:],
                    cos, sin, out=q)
        pool.attend(batch, q, out=out, workspace=ws)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        qkv.normal_()
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(4):
        x = rng.standard_normal(qkv.shape).astype(np.float16)
        qkv.copy_(dev(x))
        lens_dev.copy_(dev(lens + 1 + i))
        g.replay()
        torch.cuda.synchronize()
        got = out.float().cpu().numpy()
        p = pool.data.cpu().numpy()
        qh = q.float().cpu().numpy().astype(np.float64)
        for s in range(S):
            k, v = ref.rows_of(p, table[s], lens[s] + 1 + i, 8, hd, page)
            want = ref.attend(qh[s:s + 1], k, v, lens[s] + 1 + i, hd ** -0.5)
            assert rel(got[s:s + 1], want) < TOL["float16"]


@pytest.mark.parametrize("io", ["float16", "float32"])
def test_mixed_batches_in_a_row(sv, io):
    """A chunk beside decoding rows, writes and attention in turn on one
    stream and as a captured graph: each step sees the one before whole, and
    repeats bit for bit."""
    import torch
    rng = np.random.default_rng(21)
    hd, page, heads, n_kv = 64, 16, 8, 2
    dt = getattr(torch, io)
    rows, lens = [1] * 20 + [150, 1, 30], rng.integers(200, 3000, 23).tolist()
    n = sum(rows)
    table, n_pages, _ = layout(rng, lens, page)
    start = dev(random_pool(rng, n_pages, n_kv, 8, hd, page))
    pool = sv.KVPool(start.clone(), 8, hd, page)
    batch = batch_of(sv, rows, lens, table)
    cos, sin = (dev(f(np.arange(3000)[:, None] * np.linspace(1, 0.01, hd // 2)[None]).astype(np.float32)) for f in (np.cos, np.sin))
    x0 = dev(rng.standard_normal((n, (heads + 2 * n_kv) * hd)).astype(np.float32), dt)
    x, q, out = x0.clone(), torch.empty(n, heads, hd, device="cuda", dtype=dt), torch.empty(n, heads, hd, device="cuda", dtype=dt)
    ws = sv.attend_workspace(0)

    def step():  # the output feeds the next step's q, k and v
        pool.append(batch, x[:, :heads * hd], x[:, heads * hd:(heads + n_kv) * hd], x[:, (heads + n_kv) * hd:], cos, sin, out=q)
        pool.attend(batch, q, out=out, workspace=ws)
        x[:, :heads * hd] += out.flatten(1)
        x[:, heads * hd:] += out.flatten(1)[:, :2 * n_kv * hd]

    def reset():
        x.copy_(x0)
        pool.data.copy_(start)

    reset()
    outs = []
    for _ in range(3):
        step()
        torch.cuda.synchronize()
        outs.append(out.clone())
    k, v = ref.rows_of(pool.data.cpu().numpy(), table[20], lens[20], 8, hd, page)
    want = ref.attend(q[20:170].double().cpu().numpy(), k, v, lens[20], hd ** -0.5)
    assert rel(out[20:170].double().cpu().numpy(), want) < TOL[io]
    reset()
    for _ in range(3):  # without a wait between them
        step()
    assert torch.equal(out, outs[-1])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        step()
    reset()
    for i in range(3):
        g.replay()
        assert torch.equal(out, outs[i])


def test_two_streams_two_workspaces(sv):
    import torch
    rng = np.random.default_rng(8)
    hd, page = 128, 16
    lens = [3000, 2500]
    table, n_pages, _ = layout(rng, lens, page)
    pool = sv.KVPool(dev(random_pool(rng, n_pages, 2, 8, hd, page)), 8, hd, page)
    batch = batch_of(sv, [1, 1], lens, table)
    qs = [dev(rng.standard_normal((2, 8 * hd)).astype(np.float32)) for _ in range(2)]
    want = [pool.attend(batch, q).clone() for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(pool.attend(batch, qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_out_of_range_data_is_reported(sv):
    """A page number, a length or a row offset out of range: fault bit 64,
    and the other sequences are served."""
    import torch
    from lumina_b200 import cuda
    rng = np.random.default_rng(12)
    hd, page, heads, n_kv = 64, 16, 4, 2
    lens = [100, 50, 70]
    table, n_pages, _ = layout(rng, lens, page)
    data = dev(random_pool(rng, n_pages, n_kv, 8, hd, page))
    pool = sv.KVPool(data, 8, hd, page)
    q = dev(rng.standard_normal((3, heads * hd)).astype(np.float32))
    kv = dev(rng.standard_normal((3, n_kv * hd)).astype(np.float32))
    cs = dev(np.ones((200, hd // 2), np.float32))
    good = pool.attend(batch_of(sv, [1, 1, 1], lens, table), q).clone()

    def served(out, good):  # where the keys are split follows every length, so sums may round differently
        return all(rel(out[i].cpu().numpy(), good[i].cpu().numpy()) < TOL["float32"] for i in (0, 2))

    assert cuda.fault_status(0) == 0
    bad_table = table.copy()
    bad_table[1] = [n_pages, -1, 1 << 30, n_pages + 5, 7, 7, 7][:table.shape[1]]
    bad = batch_of(sv, [1, 1, 1], lens, bad_table)
    out = pool.attend(bad, q)
    assert cuda.fault_status(0) == sv.FAULT_DATA
    assert served(out, good)
    before = data.clone()
    pool.append(bad, q, kv, kv, cs, cs)
    assert cuda.fault_status(0) == sv.FAULT_DATA
    changed = (data != before).any(-1).any(-1).nonzero().flatten().tolist()
    assert set(changed) <= {int(table[0, 99 // page]), int(table[2, 69 // page])}
    pool.read(bad)
    assert cuda.fault_status(0) == sv.FAULT_DATA
    good = pool.attend(batch_of(sv, [1, 1, 1], lens, table), q).clone()  # over the rows just written
    # a length past the page table; a position past the rotation tables
    far = batch_of(sv, [1, 1, 1], [100, 10 ** 6, 70], table)
    out = pool.attend(far, q)
    assert cuda.fault_status(0) == sv.FAULT_DATA
    assert served(out, good)
    pool.append(batch_of(sv, [1, 1, 1], lens, table), q, kv, kv, cs[:80].contiguous(), cs[:80].contiguous())
    assert cuda.fault_status(0) == sv.FAULT_DATA


@pytest.mark.parametrize("io", ["float16", "float32"])
def test_attend_wait_that_gives_up(sv, io):
    """The chunk kernel's waits given no polls at all: fault bit 32 and a
    return; the next call is right (nothing of the failed one is left in the
    workspace)."""
    import torch
    from lumina_b200 import cuda
    rng = np.random.default_rng(14)
    hd, page, heads, n_kv, rows, ln = 128, 16, 8, 2, 300, 2000
    table, n_pages, _ = layout(rng, [ln], page)
    pool = sv.KVPool(dev(random_pool(rng, n_pages, n_kv, 8, hd, page)), 8, hd, page)
    q = dev(rng.standard_normal((rows, heads * hd)).astype(np.float32), getattr(torch, io))
    batch = batch_of(sv, [rows], [ln], table)
    good = pool.attend(batch, q).clone()
    assert cuda.fault_status(0) == 0
    cuda.debug_wait_limit(0)
    try:
        pool.attend(batch, q)
        torch.cuda.synchronize()
        assert cuda.fault_status(0) & sv.FAULT_WAIT
    finally:
        cuda.debug_wait_limit(-1)
        cuda.fault_status(0, clear=True)
    assert torch.equal(pool.attend(batch, q), good)
    assert cuda.fault_status(0) == 0


def test_attend_many_sequences(sv):
    """More row blocks than the chunk kernel lines up one by one, some of
    them without rows or tokens."""
    rng = np.random.default_rng(15)
    lens = rng.integers(0, 40, 2100).tolist()
    rows = [int(rng.integers(0, 2)) if i % 7 == 0 else 1 for i in range(2100)]
    got, want = run_attend(sv, 8, 64, "float32", 72, 1, 16, rows, lens, seed=16)
    check_attend(got, want, "float32")


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_pages_past_4_gib(sv, rows):
    """The pages of a sequence at both ends of a pool of 5 GiB."""
    import torch
    rng = np.random.default_rng(17)
    hd, page, n_kv, heads, ln = 128, 16, 32, 64, 200
    n_pages = (5 << 30) // (n_kv * ref.block_bytes(8, hd, page))
    pool = sv.KVPool.empty(n_pages, n_kv, hd, 8, page)
    need = -(-ln // page)
    table = np.array([[n_pages - 1 - i if i % 2 else i for i in range(need)]], np.int32)
    some = random_pool(rng, need, n_kv, 8, hd, page)
    pool.data[torch.from_numpy(table[0].astype(np.int64)).cuda()] = dev(some)
    q, k, v = (rng.standard_normal((rows, h * hd)).astype(np.float32) for h in (heads, n_kv, n_kv))
    cs = dev(np.ones((ln, hd // 2), np.float32))
    batch = batch_of(sv, [rows], [ln], table)
    qr = pool.append(batch, dev(q), dev(k), dev(v), cs, dev(np.zeros((ln, hd // 2), np.float32)))
    assert np.array_equal(qr.cpu().numpy().reshape(rows, -1), q)  # a rotation by nothing
    got = pool.attend(batch, qr).cpu().numpy()
    back = [x.cpu().numpy() for x in pool.read(batch)]
    now = pool.data[torch.from_numpy(table[0].astype(np.int64)).cuda()].cpu().numpy()
    kk, vv = ref.rows_of(now, np.arange(need, dtype=np.int32), ln, 8, hd, page)
    for x, y, z in zip(back, (k, v), (kk, vv)):
        y = y.reshape(rows, n_kv, hd)
        assert np.abs(x - y).max() <= 0.5001 / 127 * np.abs(y).max()
        assert rel(x, z[-rows:]) < 1e-6
    assert rel(got, ref.attend(q.astype(np.float64).reshape(rows, heads, hd), kk, vv, ln, hd ** -0.5)) < TOL["float32"]


def test_refusals(sv):
    import torch
    from lumina_b200.cuda import LuminaError
    hd = 64
    pool = sv.KVPool.empty(4, 2, hd, 8, 16)
    table = np.zeros((1, 2), np.int32)
    batch = batch_of(sv, [2], [20], table)
    q = torch.zeros(2, 4, hd, device="cuda")
    kv = torch.zeros(2, 2, hd, device="cuda")
    cs = torch.zeros(32, hd // 2, device="cuda")
    bad = [
        lambda: sv.KVPool(pool.data, 8, 128, 16),
        lambda: sv.KVPool(pool.data.cpu(), 8, hd, 16),
        lambda: sv.KVPool(torch.empty(4, 2, ref.block_bytes(8, 32, 16), dtype=torch.uint8, device="cuda"), 8, 32, 16).attend(batch, q.view(2, -1)),
        lambda: sv.KVPool(torch.empty(4, 2, ref.block_bytes(8, hd, 24), dtype=torch.uint8, device="cuda"), 8, hd, 24).attend(batch, q),
        lambda: sv.KVPool(torch.empty(4, 2, ref.block_bytes(2, hd, 16), dtype=torch.uint8, device="cuda"), 2, hd, 16).attend(batch, q),
        lambda: pool.attend(batch, q[:1]),
        lambda: pool.attend(batch, q.double()),
        lambda: pool.attend(batch, torch.zeros(2, 3, hd, device="cuda")),       # 3 heads over 2
        lambda: pool.attend(batch, q, softcap=float("nan")),
        lambda: pool.attend(batch, q, window=-1),
        lambda: pool.attend(batch, q, scale=-1.0),
        lambda: pool.attend(batch, q, slopes=torch.zeros(3, device="cuda")),
        lambda: pool.attend(batch, q, prefix=torch.zeros(1, device="cuda")),
        lambda: pool.attend(batch, q, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda")),
        lambda: pool.attend(batch, q.flatten(1)[:, ::2]),
        lambda: pool.append(batch, q, kv, kv.half(), cs, cs),
        lambda: pool.append(batch, q, kv, kv, cs[:, :8], cs[:, :8]),
        lambda: pool.append(batch, q, kv, kv, cs, cs, eps=float("inf")),
        lambda: pool.append(batch, q, kv, kv, cs, cs, q_norm=torch.ones(8, device="cuda")),
        lambda: pool.read(batch, out=(kv, torch.zeros(2, 2 * hd + 4, device="cuda")[:, :2 * hd])),
        lambda: pool.read(batch, dtype=torch.bfloat16),
        lambda: sv.SeqBatch(batch._keep[0][:1], batch._keep[1], batch._keep[2], 2, 2),
        lambda: pool.attend(sv.SeqBatch(*batch._keep, n_rows=2, max_rows=1), q),  # 1 sequence x 1 row < 2 rows
        lambda: sv.adjust_logits(torch.zeros(2, 8, device="cuda").half()),
        lambda: sv.adjust_logits(torch.zeros(2, 64, device="cuda"), mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda")),
        lambda: sv.adjust_logits(torch.zeros(2, 64, device="cuda"), repeat=torch.ones(3, device="cuda")),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(LuminaError):
            f()
            pytest.fail("call %d was not refused" % i)


def test_no_rows(sv):
    import torch
    pool = sv.KVPool.empty(4, 2, 64, 8, 16)
    batch = batch_of(sv, [0, 0], [5, 0], np.zeros((2, 1), np.int32))
    q = torch.zeros(0, 4, 64, device="cuda")
    kv = torch.zeros(0, 2, 64, device="cuda")
    cs = torch.zeros(8, 32, device="cuda")
    assert pool.attend(batch, q).shape == (0, 4, 64)
    assert pool.append(batch, q, kv, kv, cs, cs).shape == (0, 4, 64)
    assert pool.read(batch)[0].shape == (0, 2, 64)


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------
def test_logits_offsets_stay_within_the_lists(sv):
    """Offsets before, past and out of order: the lists' own entries count,
    a reversed range is empty."""
    import torch
    x = dev(np.linspace(1, 2, 3 * 40, dtype=np.float32).reshape(3, 40))
    toks, vals = dev(np.arange(6, dtype=np.int32)), dev(np.full(6, 8.0, np.float32))
    two = torch.full((3,), 2.0, device="cuda")
    offs = dev(np.array([-7, 1 << 30, 2, 4], np.int32))  # rows: all six, none, tokens 2 and 3
    got, _ = sv.adjust_logits(x, history=(offs, toks), repeat=two, bias=(offs, toks, vals))
    want = x.clone()
    for row, named in ((0, range(6)), (2, (2, 3))):
        for t in named:
            want[row, t] = want[row, t] / 2 + 8
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows,vocab,hist,biases,masked,pad", [
    (1, 1, 0, 0, False, 0),
    (1, 32000, 64, 5, True, 0),
    (3, 4096, 5000, 40, True, 5),
    (5, 1000, 17, 3, False, 3),
    (2, 131075, 300, 300, True, 1),
    (70, 257, 30, 0, True, 0),
    (2, 131075, 20000, 40, True, 1),  # more named tokens than are counted at once
    (1, 1200007, 9000, 50, True, 1),  # a CTA's part longer than the bits of named tokens
])
def test_logits(sv, rows, vocab, hist, biases, masked, pad):
    import torch
    rng = np.random.default_rng(vocab + hist)
    x = (3 * rng.standard_normal((rows, vocab + pad))).astype(np.float32)
    x[0, 0] = 0.0
    if vocab > 10:
        x[-1, 3] = -np.inf
    hl = [max(0, hist - 3 * r) for r in range(rows)]
    toks = [rng.integers(-2, min(vocab + 2, 3 * max(hist, 1)), n).astype(np.int32) for n in hl]
    bias = [[(int(rng.integers(-1, vocab + 1)), np.float32(rng.standard_normal())) for _ in range(biases)] for _ in range(rows)]
    if biases > 1:
        bias[0][1] = (bias[0][0][0], np.float32(0.25))  # named twice: the last entry counts
    rep = (1 + rng.random(rows)).astype(np.float32)
    fr, pr = rng.random((2, rows)).astype(np.float32)
    words = (vocab + 31) // 32 + (1 if pad else 0)
    m = rng.integers(-2**31, 2**31, (rows, words)).astype(np.int32)
    if masked:
        m[0] = 0  # nothing allowed: every logit -inf, argmax 0
        if rows > 1:
            m[1] = -1
    lg = dev(x)[:, :vocab]
    out, am = sv.adjust_logits(
        lg, history=(dev(np.concatenate([[0], np.cumsum(hl)]).astype(np.int32)), dev(np.concatenate(toks + [np.zeros(0, np.int32)]))),
        repeat=dev(rep), frequency=dev(fr), presence=dev(pr),
        bias=(dev(np.arange(0, rows * biases + 1, max(1, biases))[:rows + 1].astype(np.int32)) if biases else dev(np.zeros(rows + 1, np.int32)),
              dev(np.array([t for b in bias for t, _ in b], np.int32)), dev(np.array([v for b in bias for _, v in b], np.float32))),
        mask=dev(m) if masked else None)
    got, am = out.cpu().numpy(), am.cpu().numpy()
    for r in range(rows):
        allowed = None
        if masked:
            allowed = ((m[r].view(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1).reshape(-1)[:vocab].astype(bool)
        want = ref.adjust(x[r, :vocab], toks[r], float(rep[r]), float(fr[r]), float(pr[r]), bias[r], allowed)
        assert np.array_equal(np.isneginf(got[r]), np.isneginf(want))
        f = np.isfinite(want)
        big = 2 * np.abs(x[r, :vocab][f]) + max(hl) + 4
        assert (np.abs(got[r][f] - want[f]) <= 1e-6 * big).all()
        assert am[r] == int(np.argmax(got[r]))
    # in place, and without an argmax
    again, none = sv.adjust_logits(lg, out=lg, argmax=False)
    assert none is None and again is lg


def test_logits_ties_and_nan(sv):
    import torch
    x = torch.zeros(4, 70000, device="cuda")
    x[0, [5, 69999]] = 7.0
    x[1, [3, 60000]] = float("nan")
    x[1, 2] = float("inf")
    x[2] = float("-inf")
    x[3] = -0.0
    x[3, 9] = 0.0
    out, am = sv.adjust_logits(x)
    assert am.tolist() == [5, 3, 0, 0]
    assert torch.equal(out.view(torch.int32), x.view(torch.int32))
