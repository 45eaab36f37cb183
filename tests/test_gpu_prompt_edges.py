"""Packed and cached attention where their results are easily wrong unseen:
light keys beside a heavy one, long splits, calls of seconds, entries that are
skipped, buffers beyond 2^31 elements (plain forms: tests/prompt_oracle.py)."""
import numpy as np
import pytest

import prompt_oracle as P
from test_gpu_prompt_ops import (GUARD, DeviceCache, _cu, append, attend, check_cached, check_packed, filled,
                                 run_packed, same_cache, tables)

pytestmark = pytest.mark.gpu


def per_token(host, table, n):
    """Codes' numbers [n, kv, dim] and scales [n, kv] of a sequence, K then V."""
    pages = table[:-(-n // host.page)]
    out = []
    for codes, scales in zip(host.codes, host.scales):
        c = P.CODES[codes[pages]].transpose(0, 2, 1, 3)
        out += [c.reshape(-1, *c.shape[2:])[:n], np.repeat(scales[pages].astype(np.float64), host.page, 0)[:n]]
    return out


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("dim,group,dtype", [(64, 1, "f16"), (128, 8, "f16"), (64, 16, "bf16"), (128, 16, "bf16")])
def test_cached_light_keys_beside_a_heavy_one(ctx, sam3, dim, group, dtype):
    # One key holds most of a row's weight, in a page whose V scale is 2^5 of the
    # others'; 65,535 keys 2^-19 of it and less share the rest. 1024 items: each CTA
    # has whole ones, so that the light keys are added beside the heavy one.
    rng = np.random.default_rng(40)
    n, kv, page = 65536, 2, 64
    seqs = 1024 // kv
    pages = n // page
    host = P.Cache(pages, kv, page, dim)
    table = rng.permutation(pages).astype(np.int32)[None]
    k = rng.standard_normal((pages, kv, page, dim)) * (0.4 / dim ** 0.5)
    k[..., 0] = 0
    v = rng.uniform(100, 200, (pages, kv, page, dim))
    heavy = 20011
    at = table[0, heavy // page], slice(None), heavy % page
    k[at + (0,)] = 13.0  # a score 13 above the others': 2^18.8
    host.scales = [np.ones((pages, kv), np.float32) for _ in range(2)]
    host.scales[1][at[0]] = 32.0
    v[at[0]] /= 32.0
    v[at] = 300.0
    v[at + (slice(dim // 2),)] = 0.0  # here the result is the light keys' alone
    host.codes = [P.to_codes(x) for x in (k, v)]
    q = P.rounded(rng.standard_normal((1, kv * group, dim)), dtype)
    q[..., 0] = 1.0
    dc = DeviceCache(ctx, sam3, host, dim)
    got = attend(ctx, sam3, dc, np.repeat(q, seqs, 0), None, np.repeat(table, seqs, 0), [n] * seqs, dtype, True, 1.0)
    dc.free()
    o, tol = P.attend_codes(q, *per_token(host, table[0], n), 1.0, None, dtype)
    light = o[:, :, :dim // 2]
    assert (tol[:, :, :dim // 2] < 0.015 * np.abs(light)).all() and (light > 5).all()
    err = np.abs(P.from_bits(got, dtype) - o)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim,heads,kv", [(64, 2, 1), (128, 2, 1), (128, 1, 1)])
def test_packed_light_keys_beside_a_heavy_one(ctx, sam3, dim, heads, kv, causal):
    # 8191 keys whose weight is 2^-22.7 of the first one's: 2.4 of fp16's smallest
    # steps if that is 1, and hundreds if it is 2^7.
    rng = np.random.default_rng(44)
    n = 8192
    q, k = np.zeros((n, heads, dim)), np.zeros((n, kv, dim))
    q[:, :, 0], k[0, :, 0] = 1.0, 15.75
    v = P.rounded(rng.uniform(1000, 2000, (n, kv, dim)), "f16")
    v[0, :, :dim // 2] = 0.0  # here the result is the light keys' alone
    got, _ = run_packed(ctx, sam3, q, k, v, [0, n], "f16", causal, 1.0)
    for r in (n - 1, n - 100, n // 2, 0):
        o, tol = P.attend(q[r:r + 1], k, v, 1.0, r if causal else None, "f16", "f16", least=2.0 ** -32)
        if r > n - 200:
            light = o[:, :, :dim // 2]
            assert (light > 1.5).all() and (tol[:, :, :dim // 2] < 0.005 * light).all()
        err = np.abs(P.from_bits(got[r:r + 1], "f16") - o)
        assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 2, 1), (128, 2, 1), (128, 1, 1)])
def test_packed_infinities_in_keys_of_no_weight(ctx, sam3, dim, heads, kv, dtype):
    # In a whole tile 0 times an infinity is NaN, in a diagonal one the infinity is
    # added; never is it lost, nor does it reach another column or row.
    rng = np.random.default_rng(45)
    n = 600
    q, k, v = (P.rounded(rng.standard_normal((n, h, dim)), dtype) for h in (heads, kv, kv))
    q[:, :, 0], k[:, :, 0] = 30.0, 0.0
    k[[20, 590], :, 0] = -30.0  # e^-900 at most beside the others
    clean, _ = run_packed(ctx, sam3, q, k, v, [0, n], dtype, True, 1.0)
    v[20, 0, 5], v[590, 0, 7] = np.inf, -np.inf
    got, _ = run_packed(ctx, sam3, q, k, v, [0, n], dtype, True, 1.0)
    g = P.from_bits(got, dtype)
    assert not np.isfinite(g[20:, :, 5]).any() and not np.isfinite(g[590:, :, 7]).any()
    hit = np.zeros((n, heads, dim), bool)
    hit[20:, :, 5] = hit[590:, :, 7] = True
    assert np.array_equal(got[~hit], clean[~hit])


# ------------------------------------------------------------------ calls of seconds
# Warps that have nothing to do meanwhile wait longer than any single wait may
# take: without a mask, and with whole tiles, no V or K tile is looked through.
CFG = dict(embed_dim=256, num_heads=4, mlp_hidden=512, num_blocks=0, image_size=112, prune_after_block=0, max_batch=1)


def test_packed_call_of_seconds(sam3):
    torch = pytest.importorskip("torch")
    n, heads, dim = 1 << 20, 8, 64  # 2.3e15 operations
    gen = torch.Generator(device="cuda")
    gen.manual_seed(41)
    q, k, v = (torch.randn(n, h, dim, generator=gen, device="cuda").half() for h in (heads, 1, 1))
    v += 2.0
    o = torch.zeros_like(q)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with sam3.Context(0, **CFG) as ctx:
        ctx.attention_packed(sam3.F16, q, heads * dim, k, dim, v, dim, cu, 1, n, heads, 1, dim, 0.125, False, o, heads * dim)
        ctx.sync()  # SAM3_ERR_TIMEOUT if a wait had run out
    at = [0, 1, n // 3, n - 1]
    x, kk, vv = (t.cpu().numpy().astype(np.float64) for t in (q[at], k, v))
    want, tol = P.attend(x, kk, vv, 0.125, None, "f16", "f16")
    assert (np.abs(o[at].cpu().numpy().astype(np.float64) - want) <= tol).all()
    assert (o[:, :, 0] > 1).all()  # every row was reached


def test_cached_call_of_seconds(sam3):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(42)
    seqs, kv, group, page, dim, pool = 1024, 16, 16, 128, 64, 32
    times = 1600  # each sequence reads the pool that often: 6.6 million tokens
    host = P.Cache(pool, kv, page, dim)
    host.codes = [P.to_codes(rng.standard_normal(c.shape) * 16 + add) for c, add in zip(host.codes, (0.0, 64.0))]
    host.scales = [np.full_like(s, 2.0 ** -5) for s in host.scales]
    q = P.rounded(rng.standard_normal((1, kv * group, dim)), "f16")
    bits = torch.from_numpy(P.to_bits(q, "f16").view(np.int16)).cuda()
    rows = bits.expand(seqs, -1, -1).contiguous()
    o = torch.zeros_like(rows)
    table = (torch.arange(pool * times, device="cuda", dtype=torch.int32) % pool).expand(seqs, -1).contiguous()
    lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    want, tol = P.attend_codes(q, *per_token(host, np.arange(pool), pool * page), 0.125, None, "f16")
    with sam3.Context(0, **CFG) as ctx:
        dc = DeviceCache(ctx, sam3, host, dim)
        for n, slack in ((1, 0.0), (times, times * pool * page * 2.0 ** -23)):
            lens.fill_(n * pool * page)
            torch.cuda.synchronize()
            ctx.attention_cached(dc.c, sam3.F16, rows, kv * group * dim, None, seqs, seqs, 1, table, table.shape[1],
                                 lens, kv * group, 0.125, True, o, kv * group * dim)
            ctx.sync()
            got = P.from_bits(o.cpu().numpy().view(np.uint16), "f16")
            # v > 0 but for a few in 10^5: sum p |v| is the result; each sum's last bit may be cut
            assert (np.abs(got - want) <= tol + slack * np.abs(want)).all()
        dc.free()


# ------------------------------------------------------------------ one after another
def test_kernels_that_begin_under_each_others_end(ctx, sam3):
    # Each kernel's begin overlaps the end of the one before, and their shares of
    # tensor memory differ: the results are those of calls waited for.
    rng = np.random.default_rng(43)
    jobs = []
    for dim, heads, kv in ((64, 4, 2), (128, 4, 2), (128, 3, 1), (64, 16, 1), (128, 16, 1)):
        lens = [1, 300, 77, 1400]
        rows = sum(lens)
        q, k, v = (P.rounded(rng.standard_normal((rows, h, dim)), "f16") for h in (heads, kv, kv))
        bufs = [ctx.upload(P.to_bits(x, "f16")) for x in (q, k, v)]
        host, table = filled(rng, ctx, sam3, [3000, 17, 900], kv, 32, dim)
        dc = DeviceCache(ctx, sam3, host, dim)
        more = [ctx.upload(_cu(lens)), ctx.upload(table), ctx.upload(np.asarray([3000, 17, 900], np.int32))]
        outs = [ctx.alloc(rows * heads * dim * 2), ctx.alloc(3 * heads * dim * 2)]
        jobs.append((dim, heads, kv, rows, bufs, table, dc, more, outs))

    def call(job, which):
        dim, heads, kv, rows, bufs, table, dc, more, outs = job
        if which == 0:
            ctx.attention_packed(sam3.F16, bufs[0], heads * dim, bufs[1], kv * dim, bufs[2], kv * dim, more[0], 4,
                                 rows, heads, kv, dim, 0.1, True, outs[0], heads * dim)
        else:
            ctx.attention_cached(dc.c, sam3.F16, bufs[0], heads * dim, None, 3, 3, 1, more[1], table.shape[1],
                                 more[2], heads, 0.1, True, outs[1], heads * dim)

    def results():
        ctx.sync()
        return [ctx.download(o, (o.nbytes // 2,), np.uint16) for job in jobs for o in job[-1]]

    for job in jobs:
        for which in (0, 1):
            call(job, which)
            ctx.sync()
    want = results()
    for turn in range(6):
        order = [(job, which) for job in jobs for which in (0, 1)] * 3
        for i in np.random.default_rng(turn).permutation(len(order)):
            call(*order[i])
        assert all(np.array_equal(a, b) for a, b in zip(results(), want))
    for job in jobs:
        for b in job[4] + job[7] + job[8]:
            b.free()
        job[6].free()


# ------------------------------------------------------------------ splits
@pytest.mark.parametrize("dim,heads,kv,lens", [(64, 1, 1, [40000]), (128, 8, 2, [20011, 3, 9000]),
                                               (64, 32, 1, [9001, 30000]), (128, 3, 1, [600, 5000, 513, 512, 511])])
def test_cached_no_piece_is_lost_or_taken_twice(ctx, sam3, dim, heads, kv, lens):
    # Channel d of V is 0 outside the d-th part of the context, so that each
    # result is the weight of its part, and a piece of the split weighs much in it.
    rng = np.random.default_rng(46)
    host, table = filled(rng, ctx, sam3, lens, kv, 64, dim)
    for i, n in enumerate(lens):
        for p in range(-(-n // 64)):
            part = (np.arange(p * 64, min((p + 1) * 64, n)) * dim) // n
            v = np.where(part[:, None] == np.arange(dim), rng.uniform(50, 400, (kv, len(part), dim)), 0.0)
            host.codes[1][table[i, p], :, :len(part)] = P.to_codes(v)
    dc = DeviceCache(ctx, sam3, host, dim)
    q = P.rounded(rng.standard_normal((len(lens), heads, dim)), "bf16")
    got = P.from_bits(attend(ctx, sam3, dc, q, None, table, lens, "bf16", True, dim ** -0.5), "bf16")
    dc.free()
    for i, n in enumerate(lens):
        kc, ks, vc, vs = per_token(host, table[i], n)
        o, tol = P.attend_codes(q[i:i + 1], kc, ks, vc, vs, dim ** -0.5, None, "bf16")
        assert (np.abs(got[i] - o[0]) <= tol[0]).all(), (i, float((np.abs(got[i] - o[0]) / tol[0]).max()))
        # what the bound would not let pass: nothing at all, a tile left out or taken twice
        assert n < dim or (np.abs(o) > tol).mean() > 0.9
        tile = 128 * 128 // dim
        if n > 2 * tile:
            for first in (0, tile * (n // tile // 2), n - n % tile - tile):
                keep = np.ones(n, bool)
                keep[first:first + tile] = False
                rest = np.r_[np.arange(n), np.arange(first, first + tile)]
                for j in (np.flatnonzero(keep), rest):
                    wrong, _ = P.attend_codes(q[i:i + 1], kc[j], ks[j], vc[j], vs[j], dim ** -0.5, None, "bf16")
                    assert (np.abs(wrong - o) > 3 * tol).any(axis=(0, 2)).all()


# ------------------------------------------------------------------ what is skipped
# good: a sequence, and its rows that no other one writes too
@pytest.mark.parametrize("cu,good", [([0, 50, 101], [(0, 50, 0, 50)]), ([0, 0x7FFFFFFF, 100], []),
                                     ([-1, 20, 60, 60, 99], [(20, 60, 20, 60), (60, 99, 60, 99)]),
                                     ([0, 30, 20, 20, 60], [(0, 30, 0, 20), (20, 60, 30, 60)])])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dim,heads,kv", [(64, 2, 1), (128, 2, 1), (128, 1, 1)])
def test_packed_bad_offsets_leave_the_other_sequences(ctx, sam3, dim, heads, kv, many, cu, good):
    rng = np.random.default_rng(47)
    rows = 100
    if many:  # more sequences than the search keeps in registers: empty ones behind
        cu = cu + [min(cu[-1], rows)] * 150
    q, k, v = (P.rounded(rng.standard_normal((rows, h, dim)), "f16") for h in (heads, kv, kv))
    bufs = [ctx.upload(P.to_bits(x, "f16")) for x in (q, k, v)]
    bufs += [ctx.upload(np.asarray(cu, np.int32)), ctx.upload(np.full((rows, heads, dim), GUARD, np.uint16))]
    ctx.attention_packed(sam3.F16, bufs[0], heads * dim, bufs[1], kv * dim, bufs[2], kv * dim, bufs[3], len(cu) - 1,
                         rows, heads, kv, dim, 0.1, True, bufs[4], heads * dim)
    with pytest.raises(sam3.SAM3Error) as e:
        ctx.sync()
    assert e.value.status == sam3.ERR_INVALID_ARG
    got = ctx.download(bufs[4], (rows, heads, dim), np.uint16)
    left = np.ones(rows, bool)
    for a, b, first, end in good:
        left[a:b] = False
        o, tol = P.attend(q[a:b], k[a:b], v[a:b], 0.1, 0, "f16", "f16")
        assert (np.abs(P.from_bits(got[a:b], "f16") - o) <= tol)[first - a:end - a].all()
    assert (got[left] == GUARD).all()
    for b in bufs:
        b.free()


def test_cached_bad_entries_leave_the_other_sequences(ctx, sam3):
    rng = np.random.default_rng(48)
    lens, heads, dim, page = [100, 100, 100], 2, 64, 16
    host, table = filled(rng, ctx, sam3, lens, 1, page, dim)
    q = P.rounded(rng.standard_normal((6, heads, dim)), "f16")
    dc = DeviceCache(ctx, sam3, host, dim)
    ref = attend(ctx, sam3, dc, q, [0, 2, 4, 6], table, lens, "f16", True, 0.1)
    rows = np.arange(6)
    for change, good in (({"lens": [100, 1, 100]}, [0, 2]), ({"lens": [100, -5, 100]}, [0, 2]),
                         ({"lens": [1 << 30, 100, 100]}, [1, 2]), ({"cu": [0, 2, 4, 7]}, [0, 1]),
                         ({"cu": [0, 2, 1, 6]}, [0]), ({"max_new": 1}, []), ({"page": -1}, [0, 1, 2]),
                         ({"page": host.codes[0].shape[0]}, [0, 1, 2])):
        t = table.copy()
        if "page" in change:
            t[1, 2] = change["page"]
        bufs = [ctx.upload(P.to_bits(q, "f16")), ctx.upload(t), ctx.upload(np.asarray(change.get("lens", lens), np.int32)),
                ctx.upload(np.asarray(change.get("cu", [0, 2, 4, 6]), np.int32)),
                ctx.upload(np.full((6, heads, dim), GUARD, np.uint16))]
        ctx.attention_cached(dc.c, sam3.F16, bufs[0], heads * dim, bufs[3], 3, 6, change.get("max_new", 2), bufs[1],
                             t.shape[1], bufs[2], heads, 0.1, True, bufs[4], heads * dim)
        with pytest.raises(sam3.SAM3Error) as e:
            ctx.sync()
        assert e.value.status == sam3.ERR_INVALID_ARG
        got = ctx.download(bufs[4], (6, heads, dim), np.uint16)
        whole = np.isin(rows // 2, good)
        assert (got[~whole] == GUARD).all(), change
        if "page" in change:  # the second sequence does without that page's tokens
            whole[2:4] = False
            kc, ks, vc, vs = (x[np.arange(100) // page != 2] for x in per_token(host, table[1], 100))
            o, tol = P.attend_codes(q[2:4], kc, ks, vc, vs, 0.1, 100 - page - 2, "f16")
            assert (np.abs(P.from_bits(got[2:4], "f16") - o) <= tol).all()
        assert np.array_equal(got[whole], ref[whole]), change
        for b in bufs:
            b.free()
    dc.free()


def test_append_bad_entries_leave_the_other_sequences(ctx, sam3):
    rng = np.random.default_rng(49)
    page, dim, kv = 16, 64, 2
    good = {"cu": [0, 10, 20, 30], "lens": [20, 20, 20]}
    table, pages = tables(rng, good["lens"], page)
    k, v = (P.rounded(rng.standard_normal((30, kv, dim)), "f16") for _ in range(2))
    cases = [({"lens": [20, 5, 20]}, [0, 2]), ({"lens": [20, -3, 20]}, [0, 2]), ({"lens": [20, 20, 1 << 30]}, [0, 1]),
             ({"cu": [0, 10, 9, 19]}, [0, 2]), ({"cu": [0, 10, 20, 31]}, [0, 1]), ({"max_new": 9}, [])]
    cases += [({"page": p}, [0, 1, 2]) for p in (-1, pages, 1 << 30)]
    for change, written in cases:
        host = P.Cache(pages, kv, page, dim)
        host.scales = [np.full_like(s, 2.0 ** -9) for s in host.scales]
        dc = DeviceCache(ctx, sam3, host, dim)
        t = table.copy()
        if "page" in change:
            t[1, 0] = change["page"]
        c = good | change
        with pytest.raises(sam3.SAM3Error) as e:
            append(ctx, sam3, dc, k, v, c["cu"], t, c["lens"], "f16", max_new=c.get("max_new"))
        assert e.value.status == sam3.ERR_INVALID_ARG
        if "page" in change:  # the second sequence's first page is not there: a page of its own, put back after
            was = [x[table[1, 0]].copy() for x in host.codes + host.scales]
        for i in written:
            a, b = c["cu"][i], c["cu"][i + 1]
            host.append(k[a:b], v[a:b], [0, b - a], table[i:i + 1], [c["lens"][i]])
        if "page" in change:
            for x, w in zip(host.codes + host.scales, was):
                x[table[1, 0]] = w
        same_cache(dc.read(), host)
        dc.free()
    ctx.sync()


# ------------------------------------------------------------------ far addresses, many sequences
def test_rows_and_pages_beyond_32_bits(sam3):
    # Rows 2^22 elements apart, 2.9e9 in all, q, k, v and o side by side in them; a
    # cache of 5.2 GB for K and as much for V, whose last pages are used.
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(50)
    rows, stride, heads, kv, dim, page, pages = 700, 1 << 22, 4, 2, 128, 128, 159000
    x = torch.zeros(rows, stride, dtype=torch.int16, device="cuda")
    at, host_rows = {}, {}
    col = 0
    for name, h in (("q", heads), ("k", kv), ("v", kv), ("o", heads), ("c", heads)):
        at[name] = slice(col, col + h * dim)
        col += h * dim + 8
        if name not in "oc":
            host_rows[name] = P.rounded(rng.standard_normal((rows, h, dim)), "bf16")
            x[:, at[name]] = torch.from_numpy(P.to_bits(host_rows[name], "bf16").reshape(rows, -1).view(np.int16)).cuda()
    ptr = {n: x.data_ptr() + 2 * s.start for n, s in at.items()}
    codes = [torch.empty((pages, kv, page, dim), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty((pages, kv), device="cuda") for _ in range(2)]
    assert codes[0].numel() > 1 << 32 and x.numel() > 1 << 31
    lens = [3, 500, 0, 197]
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    small, few = tables(rng, lens, page)  # the host's cache has these few pages
    where = np.array([pages - 1 - 7 * i for i in range(few // 2)] + [3 * i for i in range(few - few // 2)], np.int32)
    table = np.where(small < few, where[np.minimum(small, few - 1)], 1 << 30).astype(np.int32)
    host = P.Cache(few, kv, page, dim)
    host.append(host_rows["k"], host_rows["v"], cu, small, lens)
    dev = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (cu, table, np.asarray(lens, np.int32))]
    torch.cuda.synchronize()
    with sam3.Context(0, **CFG) as ctx:
        cache = sam3.kv_cache(*codes, *scales, pages, page, kv, dim)
        ctx.attention_packed(sam3.BF16, ptr["q"], stride, ptr["k"], stride, ptr["v"], stride, dev[0], 4, rows, heads,
                             kv, dim, 0.1, True, ptr["o"], stride)
        ctx.kv_append(cache, sam3.BF16, ptr["k"], stride, ptr["v"], stride, dev[0], 4, rows, max(lens), dev[1],
                      table.shape[1], dev[2])
        ctx.attention_cached(cache, sam3.BF16, ptr["q"], stride, dev[0], 4, rows, max(lens), dev[1], table.shape[1],
                             dev[2], heads, 0.1, True, ptr["c"], stride)
        ctx.sync()
    back = {n: x[:, at[n]].contiguous().cpu().numpy().view(np.uint16).reshape(rows, -1, dim) for n in at}
    for n in "qkv":
        assert np.array_equal(back[n].ravel(), P.to_bits(host_rows[n], "bf16").ravel())
    for i in range(few):
        if (small == i).any():
            s, t = np.argwhere(small == i)[0]
            held = min(page, lens[s] - t * page)
            for w in range(2):
                assert np.array_equal(codes[w][int(where[i]), :, :held].cpu().numpy(), host.codes[w][i][:, :held])
                assert np.array_equal(scales[w][int(where[i])].cpu().numpy(), host.scales[w][i])
    check_packed(back["o"], host_rows["q"], host_rows["k"], host_rows["v"], cu, "bf16", True, 0.1)
    check_cached(back["c"], host_rows["q"], host, cu, small, lens, "bf16", True, 0.1)
    gaps = torch.ones(stride, dtype=torch.bool, device="cuda")
    for s in at.values():
        gaps[s] = False
    assert not any(bool(x[r][gaps].any()) for r in (0, 1, 499, 502, rows - 1))


@pytest.mark.parametrize("dim,heads,kv", [(64, 2, 1), (128, 2, 1), (128, 1, 1)])
def test_packed_long_sequences_among_many(ctx, sam3, dim, heads, kv):
    rng = np.random.default_rng(51)
    lens = rng.integers(0, 60, 300)
    lens[[0, 170, 299]] = 3000, 1500, 129
    cu, rows = _cu(lens), int(lens.sum())
    q, k, v = (P.rounded(rng.standard_normal((rows, h, dim)), "bf16") for h in (heads, kv, kv))
    for causal in (True, False):
        got, _ = run_packed(ctx, sam3, q, k, v, cu, "bf16", causal, 0.1)
        check_packed(got, q, k, v, cu, "bf16", causal, 0.1)


# ------------------------------------------------------------------ behind a projection
def test_projection_rows_go_in_as_they_lie(ctx, sam3, oracle):
    heads, kv, dim, page, lens = 4, 2, 64, 16, [70, 0, 33]
    rows, width = sum(lens), (heads + 2 * kv) * dim
    rng = np.random.default_rng(52)
    idx, pal = oracle.gen_u8(7, 1, (width, 256)), oracle.gen_palette(7, 2, width)
    w = sam3.palette_linear(ctx.upload(idx), ctx.upload(pal), None, width, 256)
    dx, dy, do = ctx.upload(oracle.gen_normal(7, 3, (rows, 256))), ctx.alloc(rows * width * 2), ctx.alloc(rows * heads * dim * 2)
    cu = _cu(lens)
    table, pages = tables(rng, lens, page)
    host = P.Cache(pages, kv, page, dim)
    dc = DeviceCache(ctx, sam3, host, dim)
    dev = [ctx.upload(a) for a in (cu, table, np.asarray(lens, np.int32))]
    k_at, v_at = dy.ptr + heads * dim * 2, dy.ptr + (heads + kv) * dim * 2
    dc_out = ctx.alloc(rows * heads * dim * 2)
    ctx.linear_palette(dx, rows, w, sam3.EPI_BIAS, dy)  # no wait in between
    ctx.attention_packed(sam3.F16, dy, width, k_at, width, v_at, width, dev[0], 3, rows, heads, kv, dim, 0.125, True,
                         do, heads * dim)
    ctx.kv_append(dc.c, sam3.F16, k_at, width, v_at, width, dev[0], 3, rows, max(lens), dev[1], table.shape[1], dev[2])
    ctx.attention_cached(dc.c, sam3.F16, dy, width, dev[0], 3, rows, max(lens), dev[1], table.shape[1], dev[2], heads,
                         0.125, True, dc_out, heads * dim)
    ctx.sync()
    y = P.from_bits(ctx.download(dy, (rows, heads + 2 * kv, dim), np.uint16), "f16")
    q, k, v = np.split(y, [heads, heads + kv], 1)
    assert np.isfinite(y).all() and np.abs(y).max() > 0.01
    host.append(k, v, cu, table, lens)
    same_cache(dc.read(), host)
    check_packed(ctx.download(do, (rows, heads, dim), np.uint16), q, k, v, cu, "f16", True, 0.125)
    check_cached(ctx.download(dc_out, (rows, heads, dim), np.uint16), q, host, cu, table, lens, "f16", True, 0.125)
    dc.free()


# ------------------------------------------------------------------ what is reported
def test_a_bad_entry_does_not_hide_a_wait_that_ran_out(sam3):
    with sam3.Context(0, **CFG) as ctx:
        table, pages = tables(np.random.default_rng(53), [20], 16)
        host = P.Cache(pages, 1, 16, 64)
        dc = DeviceCache(ctx, sam3, host, 64)
        bits, bad = ctx.upload(np.zeros((1, 64), np.uint16)), ctx.upload(np.array([5, 3], np.int32))
        table, lens, o = ctx.upload(table), ctx.upload(np.array([1 << 29], np.int32)), ctx.alloc(128)
        calls = (lambda: ctx.attention_packed(sam3.F16, bits, 64, bits, 64, bits, 64, bad, 1, 1, 1, 1, 64, 0.1, True, o, 64),
                 lambda: ctx.kv_append(dc.c, sam3.F16, bits, 64, bits, 64, None, 1, 1, 1, table, 3, lens),
                 lambda: ctx.attention_cached(dc.c, sam3.F16, bits, 64, None, 1, 1, 1, table, 3, lens, 1, 0.1, True, o, 64))
        for call in calls:  # each by itself
            call()
            with pytest.raises(sam3.SAM3Error) as e:
                ctx.sync()
            assert e.value.status == sam3.ERR_INVALID_ARG
        ctx.selftest_wait_timeout()
        for call in calls:
            call()
        with pytest.raises(sam3.SAM3Error) as e:
            ctx.sync()
        assert e.value.status == sam3.ERR_TIMEOUT
        ctx.sync()
        dc.free()
