"""Packed and cached attention where their results are easily wrong unseen:
light keys beside a heavy one, long splits, calls of seconds, entries that are
skipped, buffers beyond 2^31 elements (plain forms: tests/prompt_oracle.py)."""
import numpy as np
import pytest

import prompt_oracle as P
from test_gpu_prompt_ops import DeviceCache, attend

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
