"""Packed prompt attention, the 8-bit paged cache and the attention over it,
against 64-bit plain forms (tests/prompt_oracle.py, which derives the bounds)."""
import numpy as np
import pytest

import prompt_oracle as P

pytestmark = pytest.mark.gpu
GUARD = 0x5A5A


def _rows(rng, rows, heads, dim, dtype, width=1.0):
    return P.rounded(rng.standard_normal((rows, heads, dim)) * width, dtype)


def _cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _kind(sam3, dtype):
    return sam3.BF16 if dtype == "bf16" else sam3.F16


def _bits(x, dtype):
    return P.to_bits(x, dtype).reshape(x.shape[0], -1)


# ------------------------------------------------------------------ packed
def run_packed(ctx, sam3, q, k, v, cu, dtype, causal, scale, rows=None, pad=0):
    """q, k, v side by side in rows of a wider buffer, o in rows `pad` elements
    wider; returns the patterns of o [rows, heads, dim] and of the padding."""
    rows = q.shape[0] if rows is None else rows
    h, kv, d = q.shape[1], k.shape[1], q.shape[2]
    wide = (h + 2 * kv) * d + 8
    buf = np.full((rows, wide), GUARD, np.uint16)
    for x, at in ((q, 0), (k, h * d), (v, (h + kv) * d)):
        buf[:, at:at + x.shape[1] * d] = _bits(x, dtype)
    dq, dcu = ctx.upload(buf), ctx.upload(np.asarray(cu, np.int32))
    do = ctx.upload(np.full((rows, h * d + pad), GUARD, np.uint16))
    ctx.attention_packed(_kind(sam3, dtype), dq, wide, dq.ptr + h * d * 2, wide,
                         dq.ptr + (h + kv) * d * 2, wide, dcu, len(cu) - 1, rows, h, kv, d, scale,
                         causal, do, h * d + pad)
    ctx.sync()
    got = ctx.download(do, (rows, h * d + pad), np.uint16)
    for b in (dq, dcu, do):
        b.free()
    return got[:, :h * d].reshape(rows, h, d), got[:, h * d:]


def check_packed(got, q, k, v, cu, dtype, causal, scale):
    for a, b in zip(cu[:-1], cu[1:]):
        o, tol = P.attend(q[a:b], k[a:b], v[a:b], scale, 0 if causal else None, dtype, dtype)
        err = np.abs(P.from_bits(got[a:b], dtype) - o)
        assert (err <= tol).all(), (a, b, float((err / tol).max()))


LENS = [[1], [2, 0, 127], [128, 129], [0, 1, 255, 0, 0, 257, 3, 0], [300, 40, 511]]


@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("heads,kv", [(2, 2), (3, 1), (4, 1), (6, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_shapes(ctx, sam3, dim, heads, kv, lens):
    rng = np.random.default_rng(heads * 1000 + dim + sum(lens))
    for dtype, causal in (("f16", True), ("bf16", False), ("bf16", True), ("f16", False)):
        rows = sum(lens)
        q, k, v = (_rows(rng, rows, n, dim, dtype, w) for n, w in ((heads, 2.0), (kv, 1.0), (kv, 1.0)))
        cu = _cu(lens)
        got, _ = run_packed(ctx, sam3, q, k, v, cu, dtype, causal, dim ** -0.5)
        check_packed(got, q, k, v, cu, dtype, causal, dim ** -0.5)


@pytest.mark.parametrize("dim,heads,kv,pad", [(64, 2, 1, 8), (128, 2, 1, 8), (128, 3, 3, 16), (64, 1, 1, 24)])
def test_packed_leaves_other_rows_and_padding(ctx, sam3, dim, heads, kv, pad):
    rng = np.random.default_rng(5)
    lens, rows = [130, 0, 61], 200  # 9 rows belong to no sequence
    q, k, v = (_rows(rng, rows, n, dim, "f16") for n in (heads, kv, kv))
    q[191:], k[191:], v[191:] = np.nan, np.inf, np.nan
    cu = _cu(lens)
    got, padding = run_packed(ctx, sam3, q, k, v, cu, "f16", True, 0.1, rows=rows, pad=pad)
    check_packed(got, q, k, v, cu, "f16", True, 0.1)
    assert (got[191:] == GUARD).all() and (padding == GUARD).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 2, 1), (128, 2, 1), (128, 1, 1)])
def test_packed_infinities_and_nan_in_masked_places(ctx, sam3, dim, heads, kv, dtype):
    rng = np.random.default_rng(6)
    lens = [300, 150, 77]
    cu, rows, scale = _cu(lens), sum(lens), dim ** -0.5
    q, k, v = (_rows(rng, rows, n, dim, dtype) for n in (heads, kv, kv))
    clean, _ = run_packed(ctx, sam3, q, k, v, cu, dtype, True, scale)
    # the first sequence gets them at positions 140, 257 and 299, the next at its start
    vb, kb, qb = v.copy(), k.copy(), q.copy()
    vb[140, 0, 3], vb[257, 0, dim - 1], vb[299, 0, 0] = np.nan, np.inf, -np.inf
    kb[299, 0, 1] = np.nan
    vb[300], kb[301], qb[302] = np.nan, np.inf, np.nan
    got, _ = run_packed(ctx, sam3, qb, kb, vb, cu, dtype, True, scale)
    g = P.from_bits(got, dtype)
    cols = np.ones(dim, bool)
    cols[[3, dim - 1, 0]] = False
    assert np.array_equal(got[:140], clean[:140])                  # rows before see none of it
    assert np.array_equal(got[140:299][..., cols], clean[140:299][..., cols])
    assert np.isnan(g[140:299, :, 3]).all()
    assert np.array_equal(got[140:257, :, dim - 1], clean[140:257, :, dim - 1])
    assert (g[257:299, :, dim - 1] == np.inf).all()
    assert np.array_equal(got[140:299, :, 0], clean[140:299, :, 0])
    assert np.isnan(g[299]).all()                                   # its own key is NaN
    assert np.array_equal(got[450:], clean[450:])                   # the last sequence
    assert np.isnan(g[300:450]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 2, 1), (128, 2, 1), (128, 1, 1)])
def test_packed_scores_of_minus_infinity(ctx, sam3, dim, heads, kv, dtype):
    rng = np.random.default_rng(26)
    n, dead, scale = 400, 300, dim ** -0.5  # the first 300 keys: two whole tiles and more
    q, k, v = (_rows(rng, n, h, dim, dtype) for h in (heads, kv, kv))
    q[:, :, 1] = np.abs(q[:, :, 1]) + 0.125
    q = P.rounded(q, dtype)
    k[:dead, :, 1] = -np.inf
    for causal in (True, False):
        got, _ = run_packed(ctx, sam3, q, k, v, _cu([n]), dtype, causal, scale)
        g = P.from_bits(got, dtype)
        # their weight is 0: the result is that of the other keys alone
        o, tol = P.attend(q[dead:], k[dead:], v[dead:], scale, 0 if causal else None, dtype, dtype)
        assert (np.abs(g[dead:] - o) <= tol).all()
        if causal:
            assert np.isnan(g[:dead]).all()  # nothing but -inf


@pytest.mark.parametrize("dim", [64, 128])
def test_packed_growing_scores_rescale(ctx, sam3, dim):
    rng = np.random.default_rng(7)
    n, scale = 640, 1.0
    q = np.zeros((n, 2, dim))
    q[:, :, 0], q[:, :, 1] = 4.0, -4.0
    k, v = _rows(rng, n, 1, dim, "f16", 0.2), _rows(rng, n, 1, dim, "f16")
    k[:, 0, 0] = P.rounded(np.arange(n) / 16.0, "f16")   # later keys weigh more
    q[::3, :, 0], q[::3, :, 1] = -4.0, 4.0               # every third row: earlier keys do
    cu = _cu([n])
    for causal in (True, False):
        got, _ = run_packed(ctx, sam3, q, k, v, cu, "f16", causal, scale)
        check_packed(got, q, k, v, cu, "f16", causal, scale)


@pytest.mark.parametrize("dtype,dim,heads,kv", [("f16", 64, 4, 1), ("bf16", 128, 4, 1), ("bf16", 128, 1, 1)])
def test_packed_long_sequence_and_same_twice(ctx, sam3, dtype, dim, heads, kv):
    rng = np.random.default_rng(8)
    lens = [5184 + 333, 45]
    cu, rows = _cu(lens), sum(lens)
    q, k, v = (_rows(rng, rows, n, dim, dtype) for n in (heads, kv, kv))
    a, _ = run_packed(ctx, sam3, q, k, v, cu, dtype, True, dim ** -0.5)
    b, _ = run_packed(ctx, sam3, q, k, v, cu, dtype, True, dim ** -0.5)
    assert np.array_equal(a, b)
    for r in (0, 1, 127, 128, 2591, 4095, 5516):
        o, tol = P.attend(q[r:r + 1], k[:r + 1], v[:r + 1], dim ** -0.5, None, dtype, dtype)
        assert (np.abs(P.from_bits(a[r:r + 1], dtype) - o) <= tol).all()
    check_packed(a[5517:], q[5517:], k[5517:], v[5517:], [0, 45], dtype, True, dim ** -0.5)


def test_packed_many_short_sequences(ctx, sam3):
    rng = np.random.default_rng(9)
    lens = rng.integers(0, 9, 700)
    cu, rows = _cu(lens), int(lens.sum())
    q, k, v = (_rows(rng, rows, n, 64, "f16") for n in (2, 2, 2))
    got, _ = run_packed(ctx, sam3, q, k, v, cu, "f16", True, 0.125)
    check_packed(got, q, k, v, cu, "f16", True, 0.125)


@pytest.mark.parametrize("heads,kv", [(2, 1), (3, 3)])
def test_packed_many_sequences_of_several_tiles(ctx, sam3, heads, kv):
    rng = np.random.default_rng(29)
    lens = rng.integers(0, 400, 150)
    cu, rows = _cu(lens), int(lens.sum()) + 7
    q, k, v = (_rows(rng, rows, n, 128, "bf16") for n in (heads, kv, kv))
    for causal in (True, False):
        got, _ = run_packed(ctx, sam3, q, k, v, cu, "bf16", causal, 0.09)
        check_packed(got, q, k, v, cu, "bf16", causal, 0.09)
    bad = cu.copy()
    bad[0] = rows + 1  # the sequence that is looked at last
    with pytest.raises(sam3.SAM3Error) as e:
        run_packed(ctx, sam3, q, k, v, bad, "bf16", True, 0.09)
    assert e.value.status == sam3.ERR_INVALID_ARG


@pytest.mark.parametrize("dim", [64, 128])
def test_packed_captured_and_replayed_with_other_lengths(sam3, dim):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(30)
    heads, kv, rows = 4, 2, 1000
    with sam3.Context(0, embed_dim=256, num_heads=4, mlp_hidden=512, num_blocks=0, image_size=112,
                      prune_after_block=0, max_batch=1) as ctx:
        q, k, v = (_rows(rng, rows, n, dim, "f16") for n in (heads, kv, kv))
        dev = [torch.from_numpy(_bits(x, "f16").view(np.int16)).cuda() for x in (q, k, v)]
        o = torch.empty_like(dev[0])
        cu = torch.zeros(5, dtype=torch.int32, device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        ctx.set_stream(stream.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            graph.capture_begin()
            for _ in range(2):  # two in a row: the second begins under the first's end
                ctx.attention_packed(sam3.F16, dev[0], heads * dim, dev[1], kv * dim, dev[2], kv * dim,
                                     cu, 4, rows, heads, kv, dim, 0.1, True, o, heads * dim)
            graph.capture_end()
        for lens in ([1000, 0, 0, 0], [1, 1, 1, 1], [0, 500, 3, 497], [0, 0, 0, 0], [129, 383, 256, 200]):
            with torch.cuda.stream(stream):
                cu.copy_(torch.from_numpy(_cu(lens)))
                o.fill_(0x5A5A)
                graph.replay()
                got = o.cpu().numpy().view(np.uint16).reshape(rows, heads, dim)
            check_packed(got, q, k, v, _cu(lens), "f16", True, 0.1)
            assert (got[sum(lens):] == GUARD).all()
        ctx.sync()
        ctx.set_stream(None)
        del graph


def test_packed_agrees_with_the_encoders_attention(ctx, sam3):
    rng = np.random.default_rng(10)
    b, s, h = 2, 300, 4
    q, k, v = (_rows(rng, b * s, h, 64, "f16") for _ in range(3))
    got, _ = run_packed(ctx, sam3, q, k, v, _cu([s] * b), "f16", False, 0.125)
    qkv = ctx.upload(np.concatenate([_bits(x, "f16") for x in (q, k, v)], 1))
    o = ctx.alloc(b * s * h * 64 * 2)
    ctx.attention(qkv, b, s, h, 64, 0.125, o)
    ctx.sync()
    ref = P.from_bits(ctx.download(o, (b * s, h, 64), np.uint16), "f16")
    for i in range(b):
        _, tol = P.attend(*(x[i * s:(i + 1) * s] for x in (q, k, v)), 0.125, None, "f16", "f16")
        d = np.abs(P.from_bits(got[i * s:(i + 1) * s], "f16") - ref[i * s:(i + 1) * s])
        assert (d <= 2 * tol).all()


@pytest.mark.parametrize("cu,good", [([0, 40, 30, 90], [(0, 40)]), ([0, 50, 101], [(0, 50)]),
                                     ([-1, 20, 60], [(20, 60)]), ([0, 0x7FFFFFFF, 100], [])])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_bad_offsets_are_reported(ctx, sam3, dim, cu, good):
    rng = np.random.default_rng(11)
    q, k, v = (_rows(rng, 100, n, dim, "f16") for n in (2, 1, 1))
    with pytest.raises(sam3.SAM3Error) as e:
        run_packed(ctx, sam3, q, k, v, cu, "f16", True, 0.1)
    assert e.value.status == sam3.ERR_INVALID_ARG
    got, _ = run_packed(ctx, sam3, q, k, v, _cu([100]), "f16", True, 0.1)  # the context works on
    check_packed(got, q, k, v, _cu([100]), "f16", True, 0.1)


# ------------------------------------------------------------------ the cache
class DeviceCache:
    def __init__(self, ctx, sam3, host, dim):
        self.ctx, self.host = ctx, host
        self.bufs = [ctx.upload(host.codes[0]), ctx.upload(host.codes[1]),
                     ctx.upload(host.scales[0]), ctx.upload(host.scales[1])]
        pages, kv, page, _ = host.codes[0].shape
        self.c = sam3.kv_cache(*self.bufs, pages, page, kv, dim)

    def read(self):
        h = self.host.copy()
        h.codes = [self.ctx.download(b, x.shape, np.uint8) for b, x in zip(self.bufs[:2], h.codes)]
        h.scales = [self.ctx.download(b, x.shape, np.float32) for b, x in zip(self.bufs[2:], h.scales)]
        return h

    def free(self):
        for b in self.bufs:
            b.free()


def same_cache(a, b):
    for x, y in zip(a.codes + a.scales, b.codes + b.scales):
        assert np.array_equal(x.view(np.uint8), y.view(np.uint8))


def tables(rng, lens, page, spare=3, share=None):
    """A page table over shuffled pages (entries beyond a sequence are out of
    range), and the page count."""
    used = [-(-n // page) for n in lens]
    pages = sum(used) + spare
    order = rng.permutation(pages)
    t = np.full((len(lens), max(used) + 1), 1 << 30, np.int32)
    at = 0
    for i, u in enumerate(used):
        t[i, :u] = order[at:at + u]
        at += u
    return t, pages


def append(ctx, sam3, dc, k, v, cu, table, lens, dtype, max_new=None, pad=0):
    kv, d = k.shape[1], k.shape[2]
    rows = k.shape[0]
    stride = kv * d + pad
    kb, vb = (np.full((rows, stride), GUARD, np.uint16) for _ in range(2))
    kb[:, :kv * d], vb[:, :kv * d] = _bits(k, dtype), _bits(v, dtype)
    new = np.diff(cu) if cu is not None else np.ones(len(lens), int)
    bufs = [ctx.upload(kb), ctx.upload(vb), ctx.upload(table), ctx.upload(np.asarray(lens, np.int32)),
            ctx.upload(np.asarray(cu if cu is not None else [0], np.int32))]
    ctx.kv_append(dc.c, _kind(sam3, dtype), bufs[0], stride, bufs[1], stride,
                  bufs[4] if cu is not None else None, len(lens), rows,
                  int(max(new)) if max_new is None else max_new, bufs[2], table.shape[1], bufs[3])
    try:
        ctx.sync()
    finally:
        for b in bufs:
            b.free()


def attend(ctx, sam3, dc, q, cu, table, lens, dtype, causal, scale, pad=0, max_new=None):
    rows, h, d = q.shape
    new = np.diff(cu) if cu is not None else np.ones(len(lens), int)
    bufs = [ctx.upload(_bits(q, dtype)), ctx.upload(table), ctx.upload(np.asarray(lens, np.int32)),
            ctx.upload(np.asarray(cu if cu is not None else [0], np.int32)),
            ctx.upload(np.full((rows, h * d + pad), GUARD, np.uint16))]
    ctx.attention_cached(dc.c, _kind(sam3, dtype), bufs[0], h * d, bufs[3] if cu is not None else None,
                         len(lens), rows, int(max(new)) if max_new is None else max_new, bufs[1],
                         table.shape[1], bufs[2], h, scale, causal, bufs[4], h * d + pad)
    try:
        ctx.sync()
        got = ctx.download(bufs[4], (rows, h * d + pad), np.uint16)
    finally:
        for b in bufs:
            b.free()
    assert (got[:, h * d:] == GUARD).all()
    return got[:, :h * d].reshape(rows, h, d)


def check_cached(got, q, host, cu, table, lens, dtype, causal, scale):
    cu = np.arange(len(lens) + 1) if cu is None else cu
    for i, n in enumerate(lens):
        a, b = cu[i], cu[i + 1]
        if a == b:
            continue
        pages = table[i, :-(-n // host.page)]
        k, v = host.values(0, pages, n), host.values(1, pages, n)
        o, tol = P.attend(q[a:b], k, v, scale, n - (b - a) if causal else None, dtype, "f16",
                          vmax=float(host.scales[1][pages].max()))
        err = np.abs(P.from_bits(got[a:b], dtype) - o)
        assert (err <= tol).all(), (i, n, float((err / tol).max()))


# (page, dim): every unit size of the writing kernel
SHAPES = [(16, 64), (32, 64), (16, 128), (64, 64), (32, 128), (128, 64), (64, 128), (128, 128)]


@pytest.mark.parametrize("page,dim", SHAPES)
@pytest.mark.parametrize("kv", [1, 3, 8])
def test_append_codes_and_scales(ctx, sam3, page, dim, kv):
    rng = np.random.default_rng(page + dim + kv)
    for dtype, pad in (("f16", 0), ("bf16", 8)):
        before = np.array([0, 5, page, page - 1, 2 * page + 3, 1, 0, 40])
        new = np.array([1, 1, 2 * page + 1, 1, page, 0, 0, 3 * page])
        table, pages = tables(rng, before + new, page)
        host = P.Cache(pages, kv, page, dim, seed=kv)
        first, cu0, cu1 = [b for b in before], _cu(before), _cu(new)
        k0, v0 = (_rows(rng, cu0[-1], kv, dim, dtype, 0.1) for _ in range(2))
        k1, v1 = (_rows(rng, cu1[-1], kv, dim, dtype, 1.7) for _ in range(2))  # scales grow
        v1[0] = 0.0
        dc = DeviceCache(ctx, sam3, host, dim)
        for k, v, cu, lens in ((k0, v0, cu0, first), (k1, v1, cu1, list(before + new))):
            append(ctx, sam3, dc, k, v, cu, table, lens, dtype, pad=pad)
            host.append(k, v, cu, table, lens)
            same_cache(dc.read(), host)
        append(ctx, sam3, dc, k1, v1, cu1, table, list(before + new), dtype)  # again: no change
        same_cache(dc.read(), host)
        dc.free()


@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128), (128, 128)])
def test_append_token_by_token_extremes(ctx, sam3, page, dim):
    rng = np.random.default_rng(12)
    n = 70
    table, pages = tables(rng, [n, n], page)
    host = P.Cache(pages, 2, page, dim)
    dc = DeviceCache(ctx, sam3, host, dim)
    width = np.exp2(rng.integers(-30, 15, n))
    width[[3, 20]] = [2.0 ** -140, 2.0 ** 100]
    for t in range(n):
        k, v = (_rows(rng, 2, 2, dim, "bf16", w) for w in (width[t], 1.0 / width[t]))
        if t == 7:
            k[0, 0, 5], k[0, 1, 6], v[1, 0, 7] = np.inf, -np.inf, np.nan
        if t == 9:
            k[:], v[1] = np.inf, 0.0
        append(ctx, sam3, dc, k, v, None, table, [t + 1, t + 1], "bf16")
        host.append(k, v, [0, 1, 2], table, [t + 1, t + 1])
    same_cache(dc.read(), host)
    dc.free()


def test_append_reports_bad_lengths_and_pages(ctx, sam3):
    rng = np.random.default_rng(13)
    page, dim, kv = 16, 64, 2
    table, pages = tables(rng, [20, 20, 20], page)
    k, v = (_rows(rng, 30, kv, dim, "f16") for _ in range(2))
    cases = []
    for change in ({"lens": [20, 5, 20]}, {"lens": [20, -3, 20]}, {"lens": [20, 1 << 30, 20]},
                   {"cu": [0, 10, 9, 19]}, {"cu": [0, 10, 20, 31]}, {"max_new": 9}):
        cases.append({"cu": [0, 10, 20, 30], "lens": [20, 20, 20], "table": table} | change)
    for bad in (-1, pages, 1 << 30):
        t = table.copy()
        t[1, 0] = bad
        cases.append({"cu": [0, 10, 20, 30], "lens": [20, 20, 20], "table": t})
    for c in cases:
        host = P.Cache(pages, kv, page, dim)
        host.scales = [np.ones_like(s) for s in host.scales]
        dc = DeviceCache(ctx, sam3, host, dim)
        with pytest.raises(sam3.SAM3Error) as e:
            append(ctx, sam3, dc, k, v, c["cu"], c["table"], c["lens"], "f16", max_new=c.get("max_new"))
        assert e.value.status == sam3.ERR_INVALID_ARG
        if "max_new" not in c and c["cu"][1] == 10:  # the first sequence's tokens are there
            host.append(k, v, [0, 10], table, [20])
            got = dc.read()
            assert np.array_equal(got.codes[0][table[0, :2]], host.codes[0][table[0, :2]])
        dc.free()
    ctx.sync()


def filled(rng, ctx, sam3, lens, kv, page, dim, spread=0, spare=3):
    """A cache that holds random codes for sequences of these lengths, with
    scales 2^-7 ... 2^(spread - 7); NaN codes everywhere else."""
    table, pages = tables(rng, lens, page, spare)
    host = P.Cache(pages, kv, page, dim)
    host.codes = [np.full_like(c, 0x7F) for c in host.codes]
    host.scales = [np.full_like(s, np.nan) for s in host.scales]
    for i, n in enumerate(lens):
        for p in range(-(-n // page)):
            m = min(page, n - p * page)
            for c, s, w in zip(host.codes, host.scales, (40.0, 60.0)):
                c[table[i, p], :, :m] = P.to_codes(rng.standard_normal((kv, m, dim)) * w)
                s[table[i, p]] = np.exp2(rng.integers(0, spread + 1, kv) - 7.0)
    return host, table


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 1), (6, 2)])
def test_cached_shapes(ctx, sam3, dim, page, heads, kv):
    rng = np.random.default_rng(page + dim + heads)
    lens = [1, 63, 64, 65, 700, 0, 129]
    host, table = filled(rng, ctx, sam3, lens, kv, page, dim)
    dc = DeviceCache(ctx, sam3, host, dim)
    for dtype, new, causal in (("f16", [1, 1, 1, 1, 1, 0, 1], True), ("bf16", [1, 3, 4, 0, 5, 0, 2], True),
                               ("bf16", [1, 2, 4, 0, 5, 0, 2], False), ("f16", [1, 20, 30, 9, 33, 0, 129], True)):
        cu = _cu(new)
        q = _rows(rng, cu[-1], heads, dim, dtype, 2.0)
        got = attend(ctx, sam3, dc, q, cu, table, lens, dtype, causal, dim ** -0.5, pad=8)
        check_cached(got, q, host, cu, table, lens, dtype, causal, dim ** -0.5)
    dc.free()


@pytest.mark.parametrize("dim,heads,kv,lens", [(64, 1, 1, [40000]), (128, 8, 2, [20011, 3, 9000]),
                                               (128, 3, 1, [600, 5000, 513, 512, 511])])
def test_cached_split_over_many_ctas(ctx, sam3, dim, heads, kv, lens):
    rng = np.random.default_rng(14)
    host, table = filled(rng, ctx, sam3, lens, kv, 64, dim)
    dc = DeviceCache(ctx, sam3, host, dim)
    q = _rows(rng, len(lens), heads, dim, "bf16", 2.0)
    a = attend(ctx, sam3, dc, q, None, table, lens, "bf16", True, dim ** -0.5)
    b = attend(ctx, sam3, dc, q, _cu([1] * len(lens)), table, lens, "bf16", True, dim ** -0.5)
    assert np.array_equal(a, b)  # one row each, by offsets or without; and the same twice
    check_cached(a, q, host, None, table, lens, "bf16", True, dim ** -0.5)
    dc.free()


@pytest.mark.parametrize("dim", [64, 128])
def test_cached_scales_far_apart_and_large_queries(ctx, sam3, dim):
    rng = np.random.default_rng(15)
    lens = [500, 130]
    host, table = filled(rng, ctx, sam3, lens, 2, 32, dim)
    host.scales[1][:] = np.exp2(rng.integers(-40, 20, host.scales[1].shape))
    host.codes[1][table[0, 3]] = 0                    # a page of zeros at the least scale
    host.scales[1][table[0, 3]] = 2.0 ** -60
    host.scales[0][:] = 2.0 ** -20
    dc = DeviceCache(ctx, sam3, host, dim)
    q = _rows(rng, 2, 4, dim, "bf16", 2.0 ** 14)
    q[1, 1] = 0.0
    got = attend(ctx, sam3, dc, q, None, table, lens, "bf16", True, 0.2)
    check_cached(got, q, host, None, table, lens, "bf16", True, 0.2)
    dc.free()


@pytest.mark.parametrize("dim", [64, 128])
def test_cached_nan_among_the_new_tokens(ctx, sam3, dim):
    rng = np.random.default_rng(16)
    lens, new = [70, 200], [6, 9]
    cu = _cu(new)
    host, table = filled(rng, ctx, sam3, lens, 1, 16, dim)
    q = _rows(rng, cu[-1], 2, dim, "f16")
    dc = DeviceCache(ctx, sam3, host, dim)
    clean = attend(ctx, sam3, dc, q, cu, table, lens, "f16", True, 0.1)
    dc.free()
    host.codes[1][table[0, 4], 0, 67 % 16, 9] = 0x7F    # V of token 67: rows 64 ... 66 do not see it
    host.codes[0][table[1, 12], 0, 195 % 16, 2] = 0xFF  # K of token 195
    dc = DeviceCache(ctx, sam3, host, dim)
    got = attend(ctx, sam3, dc, q, cu, table, lens, "f16", True, 0.1)
    g = P.from_bits(got, "f16")
    assert np.array_equal(got[:3], clean[:3]) and np.isnan(g[3:6, :, 9]).all()
    keep = np.arange(dim) != 9
    assert np.array_equal(got[3:6][..., keep], clean[3:6][..., keep])
    assert np.array_equal(got[6:10], clean[6:10]) and np.isnan(g[10:]).all()
    dc.free()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_cached_queries_that_are_not_finite(ctx, sam3, dim, dtype):
    rng = np.random.default_rng(27)
    lens = [70, 200, 30]
    host, table = filled(rng, ctx, sam3, lens, 2, 16, dim)
    dc = DeviceCache(ctx, sam3, host, dim)
    q = _rows(rng, 3, 4, dim, dtype)
    clean = attend(ctx, sam3, dc, q, None, table, lens, dtype, True, 0.1)
    q[0, 1, 3], q[1, 2, 0], q[2, 0, dim - 1] = np.inf, np.nan, -np.inf
    got = attend(ctx, sam3, dc, q, None, table, lens, dtype, True, 0.1)
    bad = np.zeros((3, 4), bool)
    bad[0, 1] = bad[1, 2] = bad[2, 0] = True
    assert np.isnan(P.from_bits(got, dtype)[bad]).all() and np.array_equal(got[~bad], clean[~bad])
    dc.free()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [600, 20000])
def test_cached_a_page_that_does_not_exist_hides_its_tokens(ctx, sam3, n, dim):
    rng = np.random.default_rng(28)
    page, heads, scale = 32, 2, 0.05
    host, table = filled(rng, ctx, sam3, [n], 1, page, dim)
    for p in range(-(-n // page)):  # scores far below 0, so that a maximum of 0 would lose all
        m = min(page, n - p * page)
        host.codes[0][table[0, p], :, :m] = P.to_codes(rng.uniform(100, 200, (1, m, dim)))
    dc = DeviceCache(ctx, sam3, host, dim)
    q = P.rounded(-rng.uniform(60, 70, (1, heads, dim)), "f16")
    gone = [*range(10), 15]  # the first tile's pages and more
    t = table.copy()
    t[0, gone] = 1 << 30
    bufs = [ctx.upload(_bits(q, "f16")), ctx.upload(t), ctx.upload(np.array([n], np.int32)),
            ctx.upload(np.zeros((1, heads * dim), np.uint16))]
    ctx.attention_cached(dc.c, sam3.F16, bufs[0], heads * dim, None, 1, 1, 1, bufs[1], t.shape[1],
                         bufs[2], heads, scale, True, bufs[3], heads * dim)
    with pytest.raises(sam3.SAM3Error) as e:
        ctx.sync()
    assert e.value.status == sam3.ERR_INVALID_ARG
    got = P.from_bits(ctx.download(bufs[3], (1, heads, dim), np.uint16), "f16")
    pages = table[0, :-(-n // page)]
    seen = ~np.isin(np.arange(n) // page, gone)
    k, v = (host.values(i, pages, n)[seen] for i in (0, 1))
    assert (q[0, 0] @ k[0, 0]) * scale < -150
    o, tol = P.attend(q, k, v, scale, None, "f16", "f16", vmax=float(host.scales[1][pages].max()))
    assert (np.abs(got - o) <= tol).all()
    for b in bufs:
        b.free()
    dc.free()


def test_cached_shared_pages_and_many_sequences(ctx, sam3):
    rng = np.random.default_rng(17)
    n, page, dim = 1024, 16, 64
    host, t = filled(rng, ctx, sam3, [160], 1, page, dim)
    lens = [int(x) for x in rng.integers(1, 161, n)]
    table = np.repeat(t, n, 0)  # all read the same pages
    dc = DeviceCache(ctx, sam3, host, dim)
    q = _rows(rng, n, 2, dim, "f16")
    got = attend(ctx, sam3, dc, q, None, table, lens, "f16", True, 0.125)
    check_cached(got, q, host, None, table, lens, "f16", True, 0.125)
    dc.free()


def test_cached_reports_bad_lengths_and_pages(ctx, sam3):
    rng = np.random.default_rng(18)
    lens, heads, dim = [100, 100, 100], 2, 64
    host, table = filled(rng, ctx, sam3, lens, 1, 16, dim)
    q = _rows(rng, 6, heads, dim, "f16")
    dc = DeviceCache(ctx, sam3, host, dim)
    ref = attend(ctx, sam3, dc, q, _cu([2, 2, 2]), table, lens, "f16", True, 0.1)
    for change in ({"lens": [100, 1, 100]}, {"lens": [100, -5, 100]}, {"lens": [100, 1 << 30, 100]},
                   {"cu": [0, 2, 1, 6]}, {"cu": [0, 2, 4, 7]}, {"max_new": 1}, {"page": -1},
                   {"page": host.codes[0].shape[0]}):
        t = table.copy()
        if "page" in change:
            t[1, 2] = change["page"]
        with pytest.raises(sam3.SAM3Error) as e:
            attend(ctx, sam3, dc, q, change.get("cu", [0, 2, 4, 6]), t, change.get("lens", lens), "f16",
                   True, 0.1, max_new=change.get("max_new", 2))
        assert e.value.status == sam3.ERR_INVALID_ARG
    got = attend(ctx, sam3, dc, q, _cu([2, 2, 2]), table, lens, "f16", True, 0.1)
    assert np.array_equal(got, ref)
    dc.free()


# ------------------------------------------------------------------ together
def _serve(ctx, sam3, rng, dtype, page, dim, heads, kv, prompts, steps):
    """Prompts through packed attention into the cache, then `steps` of one or
    more tokens each: rows, results and the host's own cache after each step."""
    total = [p + sum(s) for p, s in zip(prompts, zip(*steps))]
    table, pages = tables(rng, total, page)
    host = P.Cache(pages, kv, page, dim)
    dc = DeviceCache(ctx, sam3, host, dim)
    cu, scale = _cu(prompts), dim ** -0.5
    q, k, v = (_rows(rng, cu[-1], n, dim, dtype) for n in (heads, kv, kv))
    got, _ = run_packed(ctx, sam3, q, k, v, cu, dtype, True, scale)
    check_packed(got, q, k, v, cu, dtype, True, scale)
    append(ctx, sam3, dc, k, v, cu, table, prompts, dtype)
    host.append(k, v, cu, table, prompts)
    lens = list(prompts)
    for new in steps:
        lens = [a + b for a, b in zip(lens, new)]
        c = _cu(new)
        q, k, v = (_rows(rng, c[-1], n, dim, dtype, 1.3) for n in (heads, kv, kv))
        append(ctx, sam3, dc, k, v, c, table, lens, dtype)
        host.append(k, v, c, table, lens)
        got = attend(ctx, sam3, dc, q, c, table, lens, dtype, True, scale)
        check_cached(got, q, host, c, table, lens, dtype, True, scale)
    same_cache(dc.read(), host)
    dc.free()


@pytest.mark.parametrize("dtype,page,dim,heads,kv", [("f16", 16, 64, 4, 4), ("bf16", 64, 128, 8, 2), ("bf16", 128, 64, 3, 1)])
def test_prompts_then_answers(ctx, sam3, dtype, page, dim, heads, kv):
    _serve(ctx, sam3, np.random.default_rng(19), dtype, page, dim, heads, kv, [70, 1, 0, 333],
           [[1, 1, 1, 1], [4, 0, 1, 2], [1, 1, 1, 1], [1, 60, 1, 3]])


def test_captured_step_replayed_with_growing_lengths(sam3):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(20)
    page, dim, heads, kv, n = 16, 64, 4, 2, 3
    start, steps, scale = [5, 30, 200], 6, 0.125
    table, pages = tables(rng, [s + steps for s in start], page)
    with sam3.Context(0, embed_dim=256, num_heads=4, mlp_hidden=512, num_blocks=0, image_size=112,
                      prune_after_block=0, max_batch=1) as ctx:
        host = P.Cache(pages, kv, page, dim)
        dc = DeviceCache(ctx, sam3, host, dim)
        k, v = (_rows(rng, sum(start), kv, dim, "f16") for _ in range(2))
        append(ctx, sam3, dc, k, v, _cu(start), table, start, "f16")
        host.append(k, v, _cu(start), table, start)
        dev = lambda *shape: torch.zeros(shape, dtype=torch.int16, device="cuda")  # noqa: E731
        q, kn, vn, o = dev(n, heads * dim), dev(n, kv * dim), dev(n, kv * dim), dev(n, heads * dim)
        lens = torch.tensor(start, dtype=torch.int32, device="cuda")
        t = torch.from_numpy(table).cuda()
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        ctx.set_stream(stream.cuda_stream)

        def step():
            ctx.kv_append(dc.c, sam3.F16, kn, kv * dim, vn, kv * dim, None, n, n, 1, t, t.shape[1], lens)
            ctx.attention_cached(dc.c, sam3.F16, q, heads * dim, None, n, n, 1, t, t.shape[1], lens, heads,
                                 scale, True, o, heads * dim)

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            graph.capture_begin()
            lens += 1
            step()
            graph.capture_end()
        now = list(start)
        for _ in range(steps):
            now = [x + 1 for x in now]
            rows = [_rows(rng, n, c, dim, "f16") for c in (heads, kv, kv)]
            with torch.cuda.stream(stream):
                for d, r in zip((q, kn, vn), rows):
                    d.copy_(torch.from_numpy(_bits(r, "f16").view(np.int16)))
                graph.replay()
                got = o.cpu().numpy().view(np.uint16).reshape(n, heads, dim)
            host.append(rows[1], rows[2], range(n + 1), table, now)
            check_cached(got, rows[0], host, None, table, now, "f16", True, scale)
        ctx.sync()
        ctx.set_stream(None)
        same_cache(dc.read(), host)
        del graph


def test_two_contexts_at_once(sam3):
    rng = np.random.default_rng(21)
    cfg = dict(embed_dim=256, num_heads=4, mlp_hidden=512, num_blocks=0, image_size=112, prune_after_block=0)
    with sam3.Context(0, **cfg) as a, sam3.Context(0, **cfg) as b:
        jobs = []
        for ctx in (a, b):
            lens = [int(x) for x in rng.integers(2000, 9000, 3)]
            host, table = filled(rng, ctx, sam3, lens, 2, 64, 128)
            dc = DeviceCache(ctx, sam3, host, 128)
            q = _rows(rng, 3, 4, 128, "f16")
            bufs = [ctx.upload(_bits(q, "f16")), ctx.upload(table), ctx.upload(np.asarray(lens, np.int32)),
                    ctx.alloc(3 * 4 * 128 * 2)]
            jobs.append((ctx, host, table, lens, dc, q, bufs))
        for _ in range(20):  # both in flight, each with its own pieces
            for ctx, _, table, _, dc, _, bufs in jobs:
                ctx.attention_cached(dc.c, sam3.F16, bufs[0], 512, None, 3, 3, 1, bufs[1], table.shape[1],
                                     bufs[2], 4, 0.1, True, bufs[3], 512)
        for ctx, host, table, lens, dc, q, bufs in jobs:
            ctx.sync()
            got = ctx.download(bufs[3], (3, 4, 128), np.uint16)
            check_cached(got, q, host, None, table, lens, "f16", True, 0.1)


def test_two_contexts_packed_and_cached_at_once(sam3):
    rng = np.random.default_rng(31)
    cfg = dict(embed_dim=256, num_heads=4, mlp_hidden=512, num_blocks=0, image_size=112, prune_after_block=0)
    with sam3.Context(0, **cfg) as a, sam3.Context(0, **cfg) as b:
        jobs = []
        for ctx, dim in ((a, 64), (b, 128)):
            lens = [700, 0, 129, 1500]
            cu, rows = _cu(lens), sum(lens)
            q, k, v = (_rows(rng, rows, n, dim, "f16") for n in (4, 2, 2))
            bufs = [ctx.upload(_bits(x, "f16")) for x in (q, k, v)] + [ctx.upload(cu), ctx.alloc(rows * 4 * dim * 2)]
            clens = [3000, 17, 900]
            host, table = filled(rng, ctx, sam3, clens, 2, 32, dim)
            dc = DeviceCache(ctx, sam3, host, dim)
            cq = _rows(rng, 3, 4, dim, "f16")
            cbufs = [ctx.upload(_bits(cq, "f16")), ctx.upload(table), ctx.upload(np.asarray(clens, np.int32)),
                     ctx.alloc(3 * 4 * dim * 2)]
            jobs.append((ctx, dim, lens, cu, q, k, v, bufs, clens, host, table, dc, cq, cbufs))
        for _ in range(20):  # both kinds in flight on two streams
            for ctx, dim, lens, cu, *_, bufs, clens, host, table, dc, cq, cbufs in jobs:
                ctx.attention_packed(sam3.F16, bufs[0], 4 * dim, bufs[1], 2 * dim, bufs[2], 2 * dim, bufs[3],
                                     len(lens), sum(lens), 4, 2, dim, 0.1, True, bufs[4], 4 * dim)
                ctx.attention_cached(dc.c, sam3.F16, cbufs[0], 4 * dim, None, 3, 3, 1, cbufs[1], table.shape[1],
                                     cbufs[2], 4, 0.1, True, cbufs[3], 4 * dim)
        for ctx, dim, lens, cu, q, k, v, bufs, clens, host, table, dc, cq, cbufs in jobs:
            ctx.sync()
            check_packed(ctx.download(bufs[4], (sum(lens), 4, dim), np.uint16), q, k, v, cu, "f16", True, 0.1)
            check_cached(ctx.download(cbufs[3], (3, 4, dim), np.uint16), cq, host, None, table, clens, "f16", True, 0.1)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_before_and_behind_the_sequences_are_left(ctx, sam3, dim):
    rng = np.random.default_rng(32)
    lens, new = [300, 40], [5, 2]
    cu = np.array([3, 8, 10], np.int32)  # of 14 rows
    table, pages = tables(rng, lens, 16)
    host = P.Cache(pages, 1, 16, dim)
    dc = DeviceCache(ctx, sam3, host, dim)
    first = [n - m for n, m in zip(lens, new)]
    k, v = (_rows(rng, sum(first), 1, dim, "f16") for _ in range(2))
    append(ctx, sam3, dc, k, v, _cu(first), table, first, "f16")
    host.append(k, v, _cu(first), table, first)
    q, k, v = (_rows(rng, 14, n, dim, "f16") for n in (2, 1, 1))
    for x in (q, k, v):
        x[:3], x[10:] = np.nan, np.inf
    append(ctx, sam3, dc, k, v, cu, table, lens, "f16", max_new=5)
    host.append(k, v, cu, table, lens)
    same_cache(dc.read(), host)
    got = attend(ctx, sam3, dc, q, cu, table, lens, "f16", True, 0.1, max_new=5)
    check_cached(got, q, host, cu, table, lens, "f16", True, 0.1)
    assert (got[:3] == GUARD).all() and (got[10:] == GUARD).all()
    got, _ = run_packed(ctx, sam3, q, k, v, cu, "f16", True, 0.1)
    check_packed(got, q, k, v, cu, "f16", True, 0.1)
    assert (got[:3] == GUARD).all() and (got[10:] == GUARD).all()
    dc.free()


def test_profile_and_launch_counters(ctx, sam3):
    rng = np.random.default_rng(22)
    ctx.profile_enable(True)
    before = ctx.launches
    q, k, v = (_rows(rng, 20, 1, 64, "f16") for _ in range(3))
    run_packed(ctx, sam3, q, k, v, _cu([20]), "f16", True, 0.1)
    host, table = filled(rng, ctx, sam3, [20], 1, 16, 64)
    dc = DeviceCache(ctx, sam3, host, 64)
    append(ctx, sam3, dc, k, v, _cu([20]), table, [20], "f16")
    attend(ctx, sam3, dc, q[:1], None, table, [20], "f16", True, 0.1)
    p = ctx.profile_read()
    ctx.profile_enable(False)
    assert ctx.launches - before >= 3
    assert p["attention"]["launches"] == 2 and p["attention"]["ms"] > 0
    assert p["other"]["launches"] == 1 and p["other"]["bytes"] > 0
