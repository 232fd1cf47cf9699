"""Edges of the quantized-page attention and of its calls on a B200: values
of very different sizes, outlier dims, NaN behind vanishing weights, waits
that give up, captured graphs, ranges. Helpers and base tolerances are those of
test_gpu_serving.py."""
import numpy as np
import pytest

import serving_ref as ref
from test_gpu_serving import TOL, batch_of, check_attend, dev, layout, no_fault, random_pool, rel, run_attend, sv  # noqa: F401

pytestmark = pytest.mark.gpu


def pool_of(rng, k, v, bits, page):
    """One sequence's K and V rows (tokens, n_kv, hd) quantized into shuffled
    pages: (pool bytes, page table (1, n))."""
    ln, n_kv, hd = k.shape
    table, n_pages, _ = layout(rng, [ln], page)
    pool = random_pool(rng, n_pages, n_kv, bits, hd, page)
    nb, top = hd * bits // 8, 127 if bits == 8 else 15
    t = np.arange(ln)
    pg, off = table[0, t // page], t % page
    for i, x in enumerate((k, v)):
        amax = np.maximum(np.abs(x).max(-1), 1e-30)
        if bits == 8:
            raw = np.rint(x * (127 / amax[..., None])).astype(np.int8).view(np.uint8)
        else:
            c = np.clip(np.rint(x * (7.5 / amax[..., None]) + 7.5), 0, 15).astype(np.uint8)
            raw = c[..., 0::2] | (c[..., 1::2] << 4)
        codes = pool[:, :, i * page * nb:(i + 1) * page * nb].reshape(n_pages, n_kv, page, nb)
        codes[pg, :, off] = raw
        pool[:, :, i * page * nb:(i + 1) * page * nb] = codes.reshape(n_pages, n_kv, page * nb)
        set_scales(pool, bits, hd, page, i, pg, off, (amax / top).astype(np.float32))
    return pool, table


def set_scales(pool, bits, hd, page, which, pg, off, values):
    """K (0) or V (1) scales of the tokens at (pg, off), (tokens, n_kv) or a number."""
    a = 2 * page * (hd * bits // 8) + 4 * page * which
    s = np.ascontiguousarray(pool[:, :, a:a + 4 * page]).view(np.float32)
    s[pg, :, off] = values
    pool[:, :, a:a + 4 * page] = s.view(np.uint8)


def attend_both(sv, pool, table, bits, hd, page, q, ln, slopes=None, window=0, **kw):
    """(result, float64 definition) of the last rows q (n, heads, hd) of one sequence."""
    out = sv.KVPool(dev(pool), bits, hd, page).attend(
        batch_of(sv, [q.shape[0]], [ln], table), q, window=window, slopes=None if slopes is None else dev(slopes), **kw)
    k, v = ref.rows_of(pool, table[0], ln, bits, hd, page)
    want = ref.attend(q.double().cpu().numpy(), k, v, ln, hd ** -0.5, 0.0,
                      None if slopes is None else slopes.astype(np.float64), window)
    return out.float().cpu().numpy(), want


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30, 1 << 20, 64, 63])
@pytest.mark.parametrize("rows,lens", [([5], [2]), ([90, 3], [60, 1])])
def test_windows_past_the_cache(sv, io, window, rows, lens):
    """A window no shorter than the cache hides nothing, also beside rows
    before the first token."""
    got, want = run_attend(sv, 8, 64, io, 4, 2, 16, rows, lens, window=window, seed=81)
    at = 0
    for n, ln in zip(rows, lens):
        assert (got[at:at + n - ln] == 0).all()
        check_attend(got[at + n - ln:at + n], want[at + n - ln:at + n], io)
        at += n


def test_page_tables_past_int_positions(sv):
    """Tokens of a page table and rows whose positions would pass 31 bits are refused."""
    import torch
    from lumina_b200.cuda import LuminaError
    pool = sv.KVPool.empty(1, 1, 64, 8, 16)
    batch = batch_of(sv, [1], [1], np.zeros((1, 1), np.int32))
    batch.c.pages_ld = 2 ** 27 - 1  # 2^31 - 16 tokens
    x = torch.zeros(1, 1, 64, device="cuda")
    for call in (lambda: pool.attend(batch, x), lambda: pool.read(batch),
                 lambda: pool.append(batch, x, x, x, x[0, :, :32], x[0, :, :32])):
        with pytest.raises(LuminaError, match="page table"):
            call()


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 32), (64, 128)])
@pytest.mark.parametrize("rows", [1, 5])
def test_fewer_cells_than_warps(sv, io, bits, hd, page, rows):
    """One key in a pool of one page: warps without a cell have a page of the
    pool to read all the same, and nothing to add."""
    import torch
    rng = np.random.default_rng(85)
    pool = random_pool(rng, 1, 1, bits, hd, page)
    q = dev(rng.standard_normal((rows, 2, hd)).astype(np.float32), getattr(torch, io))
    got, want = attend_both(sv, pool, np.zeros((1, 1), np.int32), bits, hd, page, q, 1)
    assert (got[:-1] == 0).all()
    check_attend(got[-1:], want[-1:], io)


@pytest.mark.parametrize("io,heads,rows", [("float32", 16, 4), ("float16", 128, 64)])
def test_work_past_the_lines_of_tiles(sv, io, heads, rows):
    """32 sequences of 2^28 tokens with several row blocks each: 2^31 cells or
    key tiles, which an int does not count. Reported, nothing is written."""
    import torch
    from lumina_b200 import cuda
    n, page, hd = 32, 128, 64 if io == "float16" else 128
    pool = sv.KVPool.empty(1, 1, hd, 8, page)
    pages = torch.zeros(n, 2 ** 21, dtype=torch.int32, device="cuda")
    batch = sv.SeqBatch(dev(np.arange(0, n * rows + 1, rows, dtype=np.int32)), dev(np.full(n, 2 ** 28, np.int32)), pages, n * rows, rows)
    out = torch.full((n * rows, heads, hd), 77.0, device="cuda", dtype=getattr(torch, io))
    pool.attend(batch, torch.zeros_like(out), out=out)
    assert cuda.fault_status(0) == sv.FAULT_DATA
    assert (out == 77.0).all()


ROWS = [5, 60, 80]  # the decode kernel; the chunk kernel with one and with two tiles of rows


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("bits,hd", [(8, 128), (4, 64)])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("slope", [0.0, 0.01])
def test_a_large_value_that_only_later_rows_see(sv, io, bits, hd, rows, window, slope):
    """The last key's values are 2^40 times the others': the rows before the
    last do not see it and are as exact as ever."""
    import torch
    rng = np.random.default_rng(31)
    ln, heads, n_kv, page = 250, 4, 2, 16
    k, v = rng.standard_normal((2, ln, n_kv, hd))
    v[-1] *= 2.0 ** 40
    pool, table = pool_of(rng, k, v, bits, page)
    q = dev((2 * rng.standard_normal((rows, heads, hd))).astype(np.float32), getattr(torch, io))
    got, want = attend_both(sv, pool, table, bits, hd, page, q, ln, np.full(heads, slope, np.float32) if slope else None, window)
    check_attend(got[:-1], want[:-1], io)
    if io == "float32":  # (an fp16 result of 2^40 is an infinity)
        check_attend(got[-1:], want[-1:], io)


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("bits,hd", [(8, 128), (4, 64)])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("at", [0, 30, 140])
def test_a_large_value_of_vanishing_weight(sv, io, bits, hd, rows, at):
    """A key that every row sees, with values 2^30 times the others' and a
    weight below 2^-80: it adds nothing, and takes nothing from the others."""
    import torch
    rng = np.random.default_rng(32)
    ln, heads, n_kv, page = 250, 4, 2, 16
    base = 2 * rng.standard_normal((1, 1, hd))
    k, v = rng.standard_normal((2, ln, n_kv, hd))
    k[at] = -2 * base
    v[at] *= 2.0 ** 30
    pool, table = pool_of(rng, k, v, bits, page)
    q = dev((base + 0.3 * rng.standard_normal((rows, heads, hd))).astype(np.float32), getattr(torch, io))
    got, want = attend_both(sv, pool, table, bits, hd, page, q, ln)
    check_attend(got, want, io)


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("rows", [1, *ROWS])
def test_values_of_all_sizes(sv, io, rows):
    """Values whose sizes spread from 2^-30 to 2^8 over the keys, some of
    them zero rows."""
    import torch
    rng = np.random.default_rng(33)
    ln, heads, n_kv, page, hd = 700, 4, 2, 16, 128
    k, v = rng.standard_normal((2, ln, n_kv, hd))
    v *= 2.0 ** rng.uniform(-30, 8, (ln, 1, 1))
    pool, table = pool_of(rng, k, v, 8, page)
    t = np.arange(0, ln, 7)
    set_scales(pool, 8, hd, page, 1, table[0, t // page], t % page, 0.0)
    q = dev((2 * rng.standard_normal((rows, heads, hd))).astype(np.float32), getattr(torch, io))
    got, want = attend_both(sv, pool, table, 8, hd, page, q, ln)
    check_attend(got, want, io)
    # nothing but zero rows: zeros
    t = np.arange(ln)
    set_scales(pool, 8, hd, page, 1, table[0, t // page], t % page, 0.0)
    got, _ = attend_both(sv, pool, table, 8, hd, page, q, ln)
    assert (got == 0).all()


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("rows", [1, 5, 80])
@pytest.mark.parametrize("kind", ["one pair", "six pairs", "offset"])
def test_outlier_dims(sv, io, bits, rows, kind):
    """Outlier dims in q and K (scores of 100 to 1000 that differ little), and
    a common offset of q. A score is an fp32 sum: at worst eight partial sums
    that round at 2^-23 of sum |q k|, 2^-21 of it beyond the usual tolerance
    (an error of a score is a relative error of its weight)."""
    import torch
    rng = np.random.default_rng(41)
    ln, heads, n_kv, page, hd = 512, 4, 2, 16, 128
    k, v = rng.standard_normal((2, ln, n_kv, hd))
    q = 2 * rng.standard_normal((rows, heads, hd))
    if kind == "offset":
        q = 20 + 0.15 * q
    else:
        dims = rng.permutation(hd)[:2 if kind == "one pair" else 6]
        size = 40 if kind == "one pair" else 100
        q[..., dims] = size * (1 + 0.2 * rng.random((rows, heads, dims.size)))
        k[..., dims] = 20 * (1 + 0.01 * rng.standard_normal((ln, n_kv, dims.size)))
    pool, table = pool_of(rng, k, v, bits, page)
    qd = dev(q.astype(np.float32), getattr(torch, io))
    got, want = attend_both(sv, pool, table, bits, hd, page, qd, ln)
    kk, _ = ref.rows_of(pool, table[0], ln, bits, hd, page)
    dots = np.abs(qd.double().cpu().numpy()).reshape(rows, n_kv, -1, hd).transpose(1, 0, 2, 3).reshape(n_kv, -1, hd) @ np.abs(kk).transpose(1, 2, 0)
    assert rel(got, want) < TOL[io] + 2.0 ** -21 * dots.max() * hd ** -0.5


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("hd,rows,lens", [
    (128, [300], [2000]),            # parts of one task on many CTAs
    (64, [50, 1, 40], [50, 90, 3000]),
    (128, [1], [500]),               # for the decode kernel, which waits for nothing
])
def test_rows_of_a_wait_that_gave_up_stay_unwritten(sv, io, hd, rows, lens):
    import torch
    from lumina_b200 import cuda
    rng = np.random.default_rng(51)
    page, heads, n_kv = 16, 8, 2
    table, n_pages, _ = layout(rng, lens, page)
    pool = sv.KVPool(dev(random_pool(rng, n_pages, n_kv, 8, hd, page)), 8, hd, page)
    q = dev(rng.standard_normal((sum(rows), heads, hd)).astype(np.float32), getattr(torch, io))
    batch = batch_of(sv, rows, lens, table)
    good = pool.attend(batch, q).clone()
    out = torch.full_like(good, 77.0)
    cuda.debug_wait_limit(0)
    try:
        pool.attend(batch, q, out=out)
        torch.cuda.synchronize()
        word = cuda.fault_status(0)
    finally:
        cuda.debug_wait_limit(-1)
    at = 0
    for n in rows:
        few = n * heads // n_kv <= 32
        assert torch.equal(out[at:at + n], good[at:at + n] if few else torch.full_like(good[at:at + n], 77.0))
        at += n
    assert word == (sv.FAULT_WAIT if max(rows) > 1 else 0)
    assert torch.equal(pool.attend(batch, q, out=out), good)


def test_serving_and_the_single_sequence_model_report_apart(sv, tiny_file):
    """Bad batch data does not fail a step of the single-sequence model, and
    the step does not clear what the batch reported; nor the reverse."""
    import torch
    from lumina_b200 import cuda, synthetic
    from lumina_b200.cuda import LuminaError
    from lumina_b200.engine import CudaChatModel
    pool = sv.KVPool.empty(2, 1, 64, 8, 16)
    pool.data.zero_()
    bad = batch_of(sv, [1], [3], np.array([[9]], np.int32))  # page 9 of 2
    q = torch.zeros(1, 1, 64, device="cuda")
    m = CudaChatModel.from_lumina(tiny_file, synthetic.hf_cfg(synthetic.TINY), None, theta=synthetic.TINY["rope_theta"],
                                  max_seq=64, max_rows=16)
    try:
        m.forward([1, 2, 3], 0)
        side = torch.cuda.Stream()
        for _ in range(20):
            with torch.cuda.stream(side):
                for _ in range(10):
                    pool.attend(bad, q)
            m.decode_step(4)
            m.kv_truncate(3)
        m.decode_greedy(4, 3)
        assert cuda.fault_status(0, clear=False) == sv.FAULT_DATA
        cuda.debug_wait_limit(0)
        try:
            with pytest.raises(LuminaError, match="timed out"):
                m.forward([1, 2, 3], 0)
        finally:
            cuda.debug_wait_limit(-1)
        assert cuda.fault_status(0) == sv.FAULT_DATA
        assert cuda.fault_status(0) == 0
    finally:
        m.close()


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("rows", [1, *ROWS])
@pytest.mark.parametrize("why", ["score", "distance"])
@pytest.mark.parametrize("at", [3, 130, 240])
def test_nan_values_behind_a_vanishing_weight(sv, io, rows, why, at):
    """What sees a NaN row becomes NaN, also where the key's weight is too
    small for a float; the other KV head does not."""
    import torch
    rng = np.random.default_rng(71)
    ln, heads, n_kv, page, hd = 330, 4, 2, 16, 128
    base = 4 * rng.standard_normal((1, 1, hd))
    k, v = rng.standard_normal((2, ln, n_kv, hd))
    if why == "score":
        k[at] = -8 * base
    pool, table = pool_of(rng, k, v, 8, page)
    scales = np.array([np.nan, 1.0], np.float32)
    set_scales(pool, 8, hd, page, 1, table[0, at // page], at % page, scales)
    q = dev((base + 0.3 * rng.standard_normal((rows, heads, hd))).astype(np.float32), getattr(torch, io))
    slopes = np.full(heads, 8.0, np.float32) if why == "distance" else None
    got, want = attend_both(sv, pool, table, 8, hd, page, q, ln, slopes)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(want[at - (ln - rows) if at >= ln - rows else 0:, :2]).all() and not np.isnan(want[:, 2:]).any()


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_capture_needs_a_workspace_of_its_own(sv):
    """A capture without a workspace is refused, whether or not the stream
    has a default one; two graphs with their own replay in either order."""
    import torch
    from lumina_b200.cuda import LuminaError
    rng = np.random.default_rng(61)
    hd, page, heads, n_kv, lens = 128, 16, 8, 2, [3000, 2500]
    table, n_pages, _ = layout(rng, lens, page)
    pool = sv.KVPool(dev(random_pool(rng, n_pages, n_kv, 8, hd, page)), 8, hd, page)
    batch = batch_of(sv, [1, 1], lens, table)
    q = [dev(rng.standard_normal((2, heads, hd)).astype(np.float32)) for _ in range(2)]
    want = [pool.attend(batch, x).clone() for x in q]
    out = [torch.empty_like(x) for x in q]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pool.attend(batch, q[0])
    torch.cuda.synchronize()
    for stream in (None, side):
        with pytest.raises(LuminaError, match="workspace"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                pool.attend(batch, q[0], out=out[0])
    ws = [sv.attend_workspace(0) for _ in range(2)]
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            pool.attend(batch, q[i], out=out[i], workspace=ws[i])
    for order in ((1, 0), (0, 1)):
        for x in out:
            x.zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, w) for x, w in zip(out, want))


@pytest.mark.parametrize("make", [
    lambda n: np.zeros(n, np.uint8),
    lambda n: dev(np.zeros(n // 4, np.float32)),
    lambda n: dev(np.zeros(2 * n, np.uint8))[::2],
    lambda n: dev(np.zeros(n - 1, np.uint8)),
    lambda n: dev(np.zeros(n + 1, np.uint8))[1:],
], ids=["host memory", "other type", "strided", "short", "misaligned"])
def test_workspaces_that_are_refused(sv, make):
    import torch
    from lumina_b200.cuda import LuminaError
    ws = make(sv.attend_workspace(0).numel())
    pool = sv.KVPool.empty(4, 2, 64, 8, 16)
    batch = batch_of(sv, [2], [20], np.zeros((1, 2), np.int32))
    with pytest.raises(LuminaError):
        pool.attend(batch, torch.zeros(2, 4, 64, device="cuda"), workspace=torch.from_numpy(ws) if isinstance(ws, np.ndarray) else ws)


def test_tensors_of_too_few_dims_are_refused(sv):
    import torch
    from lumina_b200.cuda import LuminaError
    pool = sv.KVPool.empty(2, 1, 64, 8, 16)
    batch = batch_of(sv, [1], [1], np.zeros((1, 1), np.int32))
    q, kv, cs = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 64, device="cuda"), torch.zeros(4, 32, device="cuda")
    logits = torch.zeros(2, 64, device="cuda")
    for call in (lambda: pool.attend(batch, q.flatten()),
                 lambda: pool.attend(batch, q[0, 0, 0]),
                 lambda: pool.attend(batch, q, out=q.flatten()),
                 lambda: pool.append(batch, q.flatten(), kv, kv, cs, cs),
                 lambda: pool.append(batch, q, kv.flatten(), kv, cs, cs),
                 lambda: pool.append(batch, q, kv[0, 0], kv, cs, cs),
                 lambda: pool.append(batch, q[:, :0], kv, kv, cs, cs),
                 lambda: pool.read(batch, out=(kv.flatten(), kv)),
                 lambda: sv.adjust_logits(logits, out=logits.flatten()),
                 lambda: sv.adjust_logits(logits, mask=torch.zeros(4, dtype=torch.int32, device="cuda"))):
        with pytest.raises(LuminaError):
            call()


@pytest.mark.parametrize("bits", [8, 4])
def test_joins_of_many_parts_fp16(sv, bits):
    """More parts than one join takes, with fp16 rows."""
    got, want = run_attend(sv, bits, 128, "float16", 8, 1, 64, [1], [40003], seed=91)
    check_attend(got, want, "float16")


@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("cap,alibi,window,prefix", [
    (0.0, True, 0, None),
    (30.0, True, 70, [3, 200, 0, 5, 1000]),
    (0.0, False, 64, [64, 65, 1, 0, 400]),
    (0.0, False, 0, [900, 0, 63, 7, 900]),
])
@pytest.mark.parametrize("rows,lens", [
    ([1, 1, 1, 1, 1], [1, 500, 64, 129, 900]),
    ([1, 33, 2, 1, 200], [700, 300, 64, 129, 900]),
])
def test_masks_int4(sv, io, cap, alibi, window, prefix, rows, lens):
    got, want = run_attend(sv, 4, 64, io, 6, 2, 16, rows, lens, cap, alibi, window, prefix, seed=92)
    check_attend(got, want, io)


@pytest.mark.parametrize("bits,hd,page", [(8, 128, 16), (8, 64, 32), (4, 128, 64), (4, 64, 16)])
@pytest.mark.parametrize("rows,lens", [([1] * 12, [1, 2, 3, 5, 17, 40, 100, 300, 700, 1000, 2000, 3000]), ([5, 3, 2], [6, 900, 40])])
def test_decode_rows_are_rounded_once(sv, bits, hd, page, rows, lens):
    """fp16 rows of the decode kernel are the definition rounded to fp16, but
    for values within about 1e-6 of a tie: one in 250 off by 2^-10 at most,
    6e-5 of the norm; 1e-4 is asked."""
    got, want = run_attend(sv, bits, hd, "float16", 8, 2, page, rows, lens, seed=93)
    assert rel(got, want.astype(np.float16)) < 1e-4


@pytest.mark.parametrize("n_seq,rows,hd,bits,tol", [
    (16, 32, 64, 8, 4e-6), (8, 32, 128, 4, 4e-6),                         # the chunk kernel
    (64, 1, 64, 8, 1e-6), (32, 1, 128, 8, 1e-6), (12, 4, 128, 4, 1e-6),   # the decode kernel
])
def test_fp32_sums_over_many_keys(sv, n_seq, rows, hd, bits, tol):
    """Equal weights over 8192 positive values: the mean, for fp32 rows, with
    work enough that one CTA sums hundreds of cells or tiles. The tensor pipe
    cuts sums off, by 2^-24 of the sum so far on average at most, which is half
    the whole on average: 128 such sums between two rounded additions cost 3.8e-6
    (chunk kernel), four cost 1e-7 (decode kernel); the rounded additions of up
    to 1000 parts sqrt(1000) 2^-25 = 9e-7."""
    import torch
    rng = np.random.default_rng(95)
    ln, page, n_kv, G = 8192, 64, 8, 4
    table, n_pages, _ = layout(rng, [ln] * n_seq, page)
    nb = hd * bits // 8
    gen = torch.Generator(device="cuda").manual_seed(n_seq)
    data = torch.empty(n_pages, n_kv, ref.block_bytes(bits, hd, page), dtype=torch.uint8, device="cuda")
    codes = torch.randint(64, 128, data[:, :, :2 * page * nb].shape, dtype=torch.uint8, device="cuda", generator=gen)
    data[:, :, :2 * page * nb] = codes if bits == 8 else codes | 0x88  # int4: codes 8 .. 15, values 1 .. 15
    scales = 1 + torch.rand(n_pages, n_kv, 2 * page, device="cuda", generator=gen)
    data[:, :, 2 * page * nb:] = scales.view(torch.uint8)
    q = torch.zeros(n_seq * rows, n_kv * G, hd, device="cuda")
    got = sv.KVPool(data, bits, hd, page).attend(batch_of(sv, [rows] * n_seq, [ln] * n_seq, table), q).double()
    for s in range(n_seq):
        at = torch.from_numpy(table[s].astype(np.int64)).cuda()
        raw = data[at][:, :, page * nb:2 * page * nb].reshape(-1, n_kv, page, nb)
        v = raw.view(torch.int8).double() if bits == 8 else 2 * torch.stack((raw & 15, raw >> 4), -1).flatten(-2).double() - 15
        v = (v * scales[at][:, :, page:].double()[..., None]).transpose(1, 2).reshape(ln, n_kv, hd)
        want = v.cumsum(0)[ln - rows:] / torch.arange(ln - rows + 1, ln + 1, device="cuda", dtype=torch.float64)[:, None, None]
        d = got[s * rows:(s + 1) * rows].view(rows, n_kv, G, hd) / want[:, :, None] - 1
        assert d.square().mean().sqrt() < tol


@pytest.mark.parametrize("n_seq,rows,hd,tol", [(16, 32, 64, 1e-5), (8, 32, 128, 1e-5), (64, 1, 64, 4e-6), (64, 1, 128, 4e-6)])
def test_many_small_weights_beside_a_large_one(sv, n_seq, rows, hd, tol):
    """The first key weighs 2^25 times each of 8191 others, which together weigh
    2.4e-4 of it; all values are the same, so the output is that value. Added
    one by one to the large weight the small ones would be lost; in sums of a
    tile (2^-18) or of four (2^-23) they round at 2^-25: 64 times 2^-25 = 2e-6.
    (The chunk kernel's products add 128 sums that are cut off: 2^-24 each on
    average, 8e-6.)"""
    import torch
    ln, page, n_kv, G = 8192, 64, 8, 4
    rng = np.random.default_rng(96)
    table, n_pages, _ = layout(rng, [ln] * n_seq, page)
    data = torch.full((n_pages, n_kv, ref.block_bytes(8, hd, page)), 127, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(n_pages, n_kv, 2 * page, device="cuda")
    scales[:, :, page:] = 0.3 / 127
    first = torch.from_numpy(table[:, 0].astype(np.int64)).cuda()
    scales[first, :, 0] = 25 * np.log(2) / (127 * hd ** 0.5)  # q = 1: a score of 25 ln 2
    data[:, :, 2 * page * hd:] = scales.view(torch.uint8)
    q = torch.ones(n_seq * rows, n_kv * G, hd, device="cuda")
    got = sv.KVPool(data, 8, hd, page).attend(batch_of(sv, [rows] * n_seq, [ln] * n_seq, table), q).double()
    value = 127 * float(np.float32(0.3 / 127))
    assert (got / value - 1).abs().max() < tol


def test_penalties_over_two_histories(sv):
    """Repetition over prompt and output, frequency and presence over the
    output alone: two calls in place give the definition."""
    import torch
    rng = np.random.default_rng(97)
    x = (3 * rng.standard_normal((1, 500))).astype(np.float32)
    whole, out = rng.integers(0, 500, 200).astype(np.int32), rng.integers(0, 500, 60).astype(np.int32)
    allowed = rng.random(500) < 0.7
    words = np.packbits(np.concatenate([allowed, np.zeros(12, bool)])[None], axis=1, bitorder="little").view(np.int32)

    def lists(t):
        return dev(np.array([0, t.size], np.int32)), dev(t)

    def one(v):
        return torch.full((1,), v, device="cuda")

    lg = dev(x)
    sv.adjust_logits(lg, history=lists(whole), repeat=one(1.25), out=lg, argmax=False)
    _, am = sv.adjust_logits(lg, history=lists(out), frequency=one(0.25), presence=one(0.5), mask=dev(words), out=lg)
    want = ref.adjust(x[0], whole, 1.25, 0.0, 0.0, [], None)
    want = ref.adjust(want, out, 1.0, 0.25, 0.5, [], allowed)
    got = lg.cpu().numpy()[0]
    f = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), f) and np.abs(got[f] - want[f]).max() <= 1e-6 * (2 * np.abs(x).max() + 20)
    assert am.item() == int(np.argmax(got))
