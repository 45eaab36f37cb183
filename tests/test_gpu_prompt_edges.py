"""Packed and cached attention where their results are easily wrong unseen:
light keys beside a heavy one, long splits, calls of seconds, entries that are
skipped, buffers beyond 2^31 elements (plain forms: tests/prompt_oracle.py)."""
import numpy as np
import pytest

import prompt_oracle as P
from test_gpu_prompt_ops import _cu, DeviceCache, attend, filled, run_packed

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
