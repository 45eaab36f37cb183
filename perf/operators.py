"""Cases and plain forms of the attention operators for packed prompts and the 8-bit paged cache.

Three operators, all on token rows (one row per token, the heads contiguous in a row):

  packed  softmax attention over packed sequences of different lengths, causal or not, with grouped K/V heads
  append  the new tokens' K and V rows quantised into a paged cache: e4m3 codes, one power-of-two scale for each
          page of tokens and head
  cached  attention of each sequence's newest tokens over that cache, through a page table

`own` chooses between the plain form in elementary torch operations and the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
E_MIN, E_MAX = -60, 60  # exponents of a page's scale


# ------------------------------------------------------------------ cases
def _text(lens):
    return " ".join(str(x) for x in lens)


def _lens(case, key="lens"):
    return [int(x) for x in case[key].split()]


def _spread(n, lo, hi):
    """n lengths between lo and hi, evenly spread over their logarithm and shuffled by a fixed stride."""
    v = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)]
    return [v[(i * 7) % n] for i in range(n)] if n % 7 else v


def listed():
    return [
        # a handful of short text prompts beside an image call: launch latency counts
        {"name": "packed_short", "op": "packed", "lens": _text([1, 7, 19, 40]), "heads": 16, "kv_heads": 16, "dim": 64, "dtype": "f16", "causal": True},
        # token sets of four images after pruning to different counts, every token sees its whole image
        {"name": "packed_images", "op": "packed", "lens": _text([2592, 1733, 5184, 901]), "heads": 16, "kv_heads": 16, "dim": 64, "dtype": "f16", "causal": False},
        # one prompt that starts with a whole image's tokens, grouped heads
        {"name": "packed_image_prompt", "op": "packed", "lens": _text([5184 + 333]), "heads": 16, "kv_heads": 4, "dim": 64, "dtype": "f16", "causal": True},
        # a batch of prompts of very different lengths
        {"name": "packed_ragged", "op": "packed", "lens": _text(_spread(16, 17, 2048)), "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "causal": True},
        # one long prompt
        {"name": "packed_long", "op": "packed", "lens": _text([8192]), "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "causal": True},
        # one token each of a running batch, into part-filled pages
        {"name": "append_step", "op": "append", "lens": _text(_spread(64, 33, 4096)), "new": _text([1] * 64), "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64},
        # image token sets written as they leave the encoder, small pages, one of them behind earlier tokens
        {"name": "append_images", "op": "append", "lens": _text([2592, 1733, 5184 + 77, 901]), "new": _text([2592, 1733, 5184, 901]), "kv_heads": 16, "dim": 64, "dtype": "f16", "page": 16},
        # a batch of long prompts
        {"name": "append_prompts", "op": "append", "lens": _text([8192 - 5 * i for i in range(8)]), "new": _text([8192 - 5 * i for i in range(8)]), "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 128},
        # the first tokens of one answer: latency
        {"name": "cached_short", "op": "cached", "lens": _text([77]), "new": _text([1]), "heads": 16, "kv_heads": 16, "dim": 64, "dtype": "f16", "page": 16, "causal": True},
        # a running batch of answers of very different lengths
        {"name": "cached_batch", "op": "cached", "lens": _text(_spread(64, 33, 4096)), "new": _text([1] * 64), "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "causal": True},
        # a few drafted tokens behind image prompts, checked in one pass
        {"name": "cached_drafted", "op": "cached", "lens": _text([5184 + 41 * i for i in range(8)]), "new": _text([8, 8, 5, 8, 1, 8, 7, 8]), "heads": 16, "kv_heads": 4, "dim": 64, "dtype": "f16", "page": 32, "causal": True},
        # two very long contexts: the work of one head has to be split
        {"name": "cached_long", "op": "cached", "lens": _text([131072, 100003]), "new": _text([1, 1]), "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 128, "causal": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["packed", "append", "cached"])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 16] if dim == 64 else [1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    group = max(1, min(group, (32 if dim == 128 else 16) // kv))
    case = {"op": op, "dim": dim, "kv_heads": kv, "dtype": rng.choice(["f16", "bf16"])}
    if op == "packed":
        most = _log(rng, 8, 5000)
        n = _log(rng, 1, max(1, min(24, 12000 // most)))
        lens = [_log(rng, 1, most) for _ in range(n)]
        lens[rng.randrange(n)] = most
        case |= {"lens": _text(lens), "heads": kv * group, "causal": rng.random() < 0.7}
        return case
    case["page"] = rng.choice([16, 32, 64, 128])
    if op == "append":
        n = _log(rng, 1, 64)
        most = _log(rng, 1, max(1, 60000 // n))
        step = rng.random() < 0.4
        before = [rng.choice([0, _log(rng, 1, 3000)]) for _ in range(n)]
        new = [1 if step else _log(rng, 1, min(most, 8192)) for _ in range(n)]
        case |= {"lens": _text([b + x for b, x in zip(before, new)]), "new": _text(new)}
        return case
    n = _log(rng, 1, 64)
    most = _log(rng, 16, max(16, min(131072, 150000 // n)))
    lens = [_log(rng, 1, most) for _ in range(n)]
    lens[rng.randrange(n)] = most
    few = rng.choice([1, 1, 1, 2, 5, 8])
    case |= {"lens": _text(lens), "new": _text([rng.randint(1, min(few, x)) for x in lens]), "heads": kv * group, "causal": True}
    return case


# ------------------------------------------------------------------ inputs
def _rows(gen, rows, width, dtype, heads, dim):
    """Token rows as a projection gives them: normal, with a few louder channels in each head."""
    x = torch.randn(rows, heads, dim, generator=gen, device="cuda")
    loud = 1.0 + 4.0 * (torch.rand(heads, dim, generator=gen, device="cuda") < 0.04)
    return (x * loud * width).to(dtype)


def _starts(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return cu


def _dev(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, dim, kv = DTYPES[case["dtype"]], case["dim"], case["kv_heads"]
    lens = _lens(case)
    s = {"op": case["op"], "dtype": dtype, "dim": dim, "kv_heads": kv, "n": len(lens), "max_len": max(lens), "scale": dim ** -0.5}
    if case["op"] == "packed":
        heads, rows = case["heads"], sum(lens)
        # one projection's rows, q | k | v side by side
        qkv = torch.cat([_rows(gen, rows, 1.5, dtype, heads, dim), _rows(gen, rows, 1.0, dtype, kv, dim), torch.randn(rows, kv, dim, generator=gen, device="cuda").to(dtype)], 1)
        s |= {"qkv": qkv, "heads": heads, "rows": rows, "causal": case["causal"], "cu": _dev(_starts(lens)), "lens": _dev(lens)}
        s |= {"seq_of": torch.repeat_interleave(torch.arange(len(lens), device="cuda"), s["lens"].long(), output_size=rows)}
        return s
    new, page = _lens(case, "new"), case["page"]
    rows = sum(new)
    used = [-(-x // page) for x in lens]
    pages, wide = sum(used) + 3, max(used)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), wide, dtype=torch.int32, device="cuda")
    at = torch.arange(wide, device="cuda")[None, :] < _dev(used)[:, None]
    table[at] = order[: sum(used)]
    s |= {"page": page, "pages": pages, "table": table, "seq_lens": _dev(lens), "cu": _dev(_starts(new)), "rows": rows, "new": _dev(new), "max_new": max(new)}
    s |= {"seq_of": torch.repeat_interleave(torch.arange(len(lens), device="cuda"), s["new"].long(), output_size=rows)}
    shape = (pages, kv, page, dim)
    for name, width in (("k", 40.0), ("v", 50.0)):
        s[name + "8"] = torch.empty(shape, dtype=torch.uint8, device="cuda")
        for p in range(0, pages, 1024):  # in parts: the codes are the large thing here, not their making
            part = torch.randn((min(1024, pages - p),) + shape[1:], generator=gen, device="cuda") * width
            s[name + "8"][p:p + 1024] = part.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        s[name + "s"] = torch.exp2(torch.randint(-7, -4, (pages, kv), generator=gen, device="cuda").float())
    if case["op"] == "append":
        s["k"], s["v"] = _rows(gen, rows, 1.0, dtype, kv, dim), torch.randn(rows, kv, dim, generator=gen, device="cuda").to(dtype)
    else:
        s |= {"q": _rows(gen, rows, 1.0, dtype, case["heads"], dim), "heads": case["heads"], "causal": case["causal"]}
    return s


# ------------------------------------------------------------------ plain forms
def _softmax_rows(q, k, v, seen, scale):
    """q [n, kv, group, m, d], k and v [n, kv, j, d], seen [n, m, j]: the attention of each row over the keys it sees; 0 where it sees none."""
    x = torch.matmul(q, k[:, :, None].transpose(-1, -2)) * scale
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    return torch.matmul(x, v[:, :, None]) / torch.where(total == 0, 1.0, total)


def _padded(rows, at, here):
    """Rows at the indexes [n, m] as 32-bit floats, zero where there is none: [n, heads, m, d]."""
    x = rows[at.clamp(0, rows.shape[0] - 1)].float()
    return x.masked_fill_(~here[:, :, None, None], 0.0).transpose(1, 2)


def _plain_packed(s):
    h, kv, d, n = s["heads"], s["kv_heads"], s["dim"], s["n"]
    q, k, v = s["qkv"].split([h, kv, kv], 1)
    step = torch.arange(s["max_len"], device="cuda")
    at = s["cu"][:-1, None].long() + step
    here = step < s["lens"][:, None]
    seen = here[:, None, :].expand(n, s["max_len"], s["max_len"])
    if s["causal"]:
        seen = seen & (step[None, :] <= step[:, None])
    qp = _padded(q, at, here).reshape(n, kv, h // kv, s["max_len"], d)
    o = _softmax_rows(qp, _padded(k, at, here), _padded(v, at, here), seen, s["scale"])
    pos = torch.arange(s["rows"], device="cuda") - s["cu"].long()[s["seq_of"]]
    return o.permute(0, 3, 1, 2, 4)[s["seq_of"], pos].reshape(s["rows"], h, d).to(s["dtype"])


def _codes(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _plain_append_one(s, rows, codes, scales):
    """The rows of K (or V) into their pages: the new scales, the part-filled pages' codes at them, the new codes."""
    page, kv = s["page"], s["kv_heads"]
    start = (s["seq_lens"] - s["new"]).long()
    pos = start[s["seq_of"]] + torch.arange(s["rows"], device="cuda") - s["cu"].long()[s["seq_of"]]
    slot = s["table"][s["seq_of"], pos // page].long()
    x = rows.float()
    most = torch.where(torch.isfinite(x), x, 0.0).abs().amax(-1)
    top = torch.zeros_like(scales).scatter_reduce(0, slot[:, None].expand(-1, kv), most, "amax")
    m, e = torch.frexp(top)  # the least e with top <= 448 * 2^e, 448 = 0.875 * 2^9
    e = torch.where(top > 0, (e - torch.where(m <= 0.875, 9, 8)).clamp(E_MIN, E_MAX), E_MIN)
    touched = torch.zeros(s["pages"], dtype=torch.bool, device="cuda").index_fill_(0, slot, True)
    tail = s["table"][torch.arange(s["n"], device="cuda"), start // page].long()  # where each sequence's new tokens begin
    held = start % page
    old_e = torch.frexp(scales)[1] - 1
    part = torch.zeros(s["pages"], dtype=torch.bool, device="cuda").index_put_((tail,), held > 0)
    e = torch.where(part[:, None], torch.maximum(e, old_e), e)
    new_scales = torch.where(touched[:, None], torch.ldexp(torch.ones_like(scales), e), scales)
    c = codes.view(torch.float8_e4m3fn)
    kept = torch.arange(page, device="cuda")[None, None, :, None] < held[:, None, None, None]
    shift = torch.ldexp(torch.ones_like(scales), old_e - e)[tail][:, :, None, None]
    before = codes[tail]
    codes[tail] = torch.where(kept, _codes(before.view(torch.float8_e4m3fn).float() * shift).view(torch.uint8), before)
    c[slot, :, pos % page] = _codes(x * torch.ldexp(torch.ones_like(scales), -e)[slot][:, :, None])
    scales.copy_(new_scales)


def _plain_append(s):
    _plain_append_one(s, s["k"], s["k8"], s["ks"])
    _plain_append_one(s, s["v"], s["v8"], s["vs"])


def _plain_cached(s):
    h, kv, d, n, page = s["heads"], s["kv_heads"], s["dim"], s["n"], s["page"]
    t = s["table"].long()

    def whole(codes, scales):
        x = codes[t].view(torch.float8_e4m3fn).float() * scales[t][..., None, None]
        return x.transpose(1, 2).reshape(n, kv, t.shape[1] * page, d)

    step = torch.arange(s["max_new"], device="cuda")
    here = step < s["new"][:, None]
    keys = torch.arange(t.shape[1] * page, device="cuda")
    last = (s["seq_lens"] - s["new"])[:, None] + step if s["causal"] else (s["seq_lens"] - 1)[:, None].expand(n, s["max_new"])
    seen = (keys <= last[:, :, None]) & (keys < s["seq_lens"][:, None, None])
    qp = _padded(s["q"], s["cu"][:-1, None].long() + step, here).reshape(n, kv, h // kv, s["max_new"], d)
    o = _softmax_rows(qp, whole(s["k8"], s["ks"]), whole(s["v8"], s["vs"]), seen, s["scale"])
    pos = torch.arange(s["rows"], device="cuda") - s["cu"].long()[s["seq_of"]]
    return o.permute(0, 3, 1, 2, 4)[s["seq_of"], pos].reshape(s["rows"], h, d).to(s["dtype"])


# ------------------------------------------------------------------ the framework's calls
_kept = {}


def _context():
    """The program's one context, on torch's stream."""
    if not _kept:
        sys.path.insert(0, os.path.join(os.getcwd(), "metal-sam-ios-experiments_b200"))
        import sam3cuda

        ctx = sam3cuda.Context(0, embed_dim=256, num_heads=4, mlp_hidden=512, num_blocks=0, image_size=112, prune_after_block=0, max_batch=1)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: the legacy default stream
        _kept.update(ctx=ctx, api=sam3cuda)
    return _kept["ctx"], _kept["api"]


def _own(s):
    ctx, api = _context()
    kind = api.BF16 if s["dtype"] == torch.bfloat16 else api.F16
    d, kv = s["dim"], s["kv_heads"]
    if s["op"] == "packed":
        h = s["heads"]
        qkv, o = s["qkv"], torch.empty(s["rows"], h, d, dtype=s["dtype"], device="cuda")
        wide, at = (h + 2 * kv) * d, qkv.data_ptr()
        ctx.attention_packed(kind, at, wide, at + h * d * 2, wide, at + (h + kv) * d * 2, wide, s["cu"], s["n"], s["rows"], h, kv, d, s["scale"], s["causal"], o, h * d)
        return o
    cache = api.kv_cache(s["k8"], s["v8"], s["ks"], s["vs"], s["pages"], s["page"], kv, d)
    if s["op"] == "append":
        ctx.kv_append(cache, kind, s["k"], kv * d, s["v"], kv * d, s["cu"], s["n"], s["rows"], s["max_new"], s["table"], s["table"].shape[1], s["seq_lens"])
        return None
    h = s["heads"]
    o = torch.empty(s["rows"], h, d, dtype=s["dtype"], device="cuda")
    ctx.attention_cached(cache, kind, s["q"], h * d, s["cu"], s["n"], s["rows"], s["max_new"], s["table"], s["table"].shape[1], s["seq_lens"], h, s["scale"], s["causal"], o, h * d)
    return o


def run(s):
    o = _own(s) if own else {"packed": _plain_packed, "append": _plain_append, "cached": _plain_cached}[s["op"]](s)
    if s["op"] != "append":
        return o
    # the updated cache: the codes as the numbers that they stand for, and the scales
    return {"k": s["k8"].view(torch.float8_e4m3fn), "v": s["v8"].view(torch.float8_e4m3fn), "k_scale": s["ks"], "v_scale": s["vs"]}


# ------------------------------------------------------------------ work, and the definition in 64 bits
def work(case):
    lens, d, kv = _lens(case), case["dim"], case["kv_heads"]
    if case["op"] == "packed":
        h, rows = case["heads"], sum(lens)
        pairs = sum(x * (x + 1) // 2 if case["causal"] else x * x for x in lens)
        return {"bytes": rows * (2 * h + 2 * kv) * d * 2, "flops": 4 * d * h * pairs}
    new = _lens(case, "new")
    if case["op"] == "append":
        scales = sum(-(-x // case["page"]) - (x - y) // case["page"] for x, y in zip(lens, new))
        return {"bytes": sum(new) * kv * d * 2 * 3 + scales * kv * 8, "flops": sum(new) * kv * d * 4}
    h = case["heads"]
    pairs = sum(x * y - (y * (y - 1) // 2 if case["causal"] else 0) for x, y in zip(lens, new))
    return {"bytes": sum(lens) * kv * d * 2 + sum(-(-x // case["page"]) for x in lens) * (kv * 8 + 4) + sum(new) * h * d * 4, "flops": 4 * d * h * pairs}


def _attend64(q, k, v, first, scale):
    """One sequence and K/V head: q [m, group, d] at positions first.. (None: all see all), k and v [j, d], in 64 bits."""
    o = torch.empty_like(q)
    for i in range(0, q.shape[0], 1024):
        x = torch.einsum("mgd,jd->gmj", q[i:i + 1024], k) * scale
        if first is not None:
            pos = first + i + torch.arange(x.shape[1], device="cuda")
            x = x.masked_fill(torch.arange(k.shape[0], device="cuda")[None, :] > pos[:, None], -math.inf)
        o[i:i + 1024] = torch.einsum("gmj,jd->mgd", torch.softmax(x, -1), v)
    return o


def _e4m3(y):
    """The e4m3 number nearest to y, ties to the even one, at most 448: steps of 2^-9 below 2^-6, then an eighth of the power of two below."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    lens, d, kv = _lens(case), s["dim"], s["kv_heads"]
    if s["op"] == "packed":
        h = s["heads"]
        q, k, v = (x.double() for x in s["qkv"].split([h, kv, kv], 1))
        o, at = torch.zeros_like(q), 0
        for n in lens:
            for c in range(kv):
                hs = slice(c * (h // kv), (c + 1) * (h // kv))
                o[at:at + n, hs] = _attend64(q[at:at + n, hs], k[at:at + n, c], v[at:at + n, c], 0 if s["causal"] else None, s["scale"])
            at += n
        return o
    new, page = _lens(case, "new"), s["page"]
    if s["op"] == "cached":
        h, at = s["heads"], 0
        o = torch.zeros(s["rows"], h, d, dtype=torch.float64, device="cuda")
        for i, (n, m) in enumerate(zip(lens, new)):
            t = s["table"][i, : -(-n // page)].long()
            for c in range(kv):
                k, v = ((s[a + "8"][t, c].view(torch.float8_e4m3fn).double() * s[a + "s"][t, c].double()[:, None, None]).reshape(-1, d)[:n] for a in "kv")
                hs = slice(c * (h // kv), (c + 1) * (h // kv))
                o[at:at + m, hs] = _attend64(s["q"][at:at + m, hs].double(), k, v, n - m if s["causal"] else None, s["scale"])
            at += m
        return o
    out = {}
    for a in "kv":
        codes, scales, x = s[a + "8"].view(torch.float8_e4m3fn).double(), s[a + "s"].double(), s[a].double()
        at = 0
        for i, (n, m) in enumerate(zip(lens, new)):
            if m == 0:
                continue
            first, last = (n - m) // page, (n - 1) // page
            slots = s["table"][i, first:last + 1].long()
            spots = torch.arange(first * page, (last + 1) * page, device="cuda").reshape(-1, page)
            fresh, held = (spots >= n - m) & (spots < n), spots < n - m
            rows = (spots - (n - m) + at).clamp(0, s["rows"] - 1)
            y = (x[rows] * fresh[:, :, None, None]).transpose(1, 2)  # [pages, kv, page, d]
            top = y.abs().amax((-1, -2))
            e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -80) / 448) - 1e-6).clamp(E_MIN, E_MAX)  # inputs have 11 bits at most: 1e-6 is under their spacing, and over the logarithm's error
            was = torch.round(torch.log2(scales[slots]))
            grown = torch.where(held.any(1)[:, None], torch.maximum(e, was), e)
            old = codes[slots]
            moved = _e4m3(old * torch.exp2(was - grown)[:, :, None, None])
            put = _e4m3(y * torch.exp2(-grown)[:, :, None, None])
            codes[slots] = torch.where(fresh[:, None, :, None], put, torch.where(held[:, None, :, None], moved, old))
            scales[slots] = torch.exp2(grown)
            at += m
        out[a], out[a + "_scale"] = codes, scales
    return out
