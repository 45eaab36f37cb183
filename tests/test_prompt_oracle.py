"""The 64-bit plain forms that the packed-prompt and cache tests compare with."""
import numpy as np
import pytest

import prompt_oracle as P


def test_codes_against_their_definition():
    assert P.CODES[0x7E] == 448 and P.CODES[0x08] == 2.0 ** -6 and P.CODES[1] == 2.0 ** -9
    fin = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    assert np.array_equal(P.to_codes(P.CODES[fin]), fin)
    assert list(P.to_codes([1e9, -np.inf, np.nan, 2.0 ** -10, 3 * 2.0 ** -10, -1.0625, 1.1875])) == \
        [0x7E, 0xFE, 0x7F, 0x00, 0x02, 0xB8, 0x3A]  # ties go to the even code


def test_codes_against_torch():
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(0).standard_normal(20000) * np.exp2(np.random.default_rng(1).integers(-12, 9, 20000))
    x = np.clip(x.astype(np.float32), -448, 448)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(P.to_codes(x), want)


def test_bf16_bits_against_torch():
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(2).standard_normal(5000).astype(np.float32) * 1e3
    want = torch.from_numpy(x).to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)
    assert np.array_equal(P.to_bits(x, "bf16"), want)
    assert np.isnan(P.rounded(np.nan, "bf16")) and np.isinf(P.rounded(np.inf, "bf16"))


def test_append_keeps_values_within_a_rounding():
    rng = np.random.default_rng(3)
    c = P.Cache(3, 2, 16, 64)
    x = P.rounded(rng.standard_normal((20, 2, 64)) * np.exp2(np.arange(20) / 3)[:, None, None], "f16")
    for n in range(1, 21):  # one token at a time, growing: every scale rises while its page fills
        c.append(x[n - 1:n], x[n - 1:n], [0, 1], [[2, 0]], [n])
    got = c.values(0, [2, 0], 20)
    s = np.repeat(c.scales[0][[2, 0]].astype(np.float64), 16, 0)[:20, :, None]
    # one rounding of 2^-4, and, moved below 2^-6 scales, half a step of 2^-9 scales at each move
    moves = 12
    assert (np.abs(got - x) <= 2.0 ** -4 * np.abs(x) + moves * 2.0 ** -10 * s).all()


def test_scale_exp_at_its_borders():
    for e in (-60, -7, 0, 5, 59):
        assert P.scale_exp(448 * 2.0 ** e) == e
        assert P.scale_exp(np.nextafter(448 * 2.0 ** e, np.inf)) == e + 1
    assert P.scale_exp(0.0) == -60 and P.scale_exp(1e300) == 60


def test_a_planted_mistake_is_outside_the_bound():
    rng = np.random.default_rng(4)
    q, k, v = (P.rounded(rng.standard_normal((40, 2, 64)), "bf16") for _ in range(3))
    o, tol = P.attend(q, k, v, 0.125, 0, "bf16", "bf16")
    off, _ = P.attend(q, k, v, 0.125, 1, "bf16", "bf16")      # one key too many
    assert (np.abs(off - o) > tol)[:39].any(axis=(1, 2)).all()
    off, _ = P.attend(q, k, v, 0.125 * 1.1, 0, "bf16", "bf16")  # another scale
    assert (np.abs(off - o) > tol).any()
