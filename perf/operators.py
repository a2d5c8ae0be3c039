"""The serving operators in plain form and as the library's calls: attention over packed prompts, storing keys and values in
an 8-bit cache with one scale per block of tokens and head, and single-token attention over that cache.

`own` selects what run() does: the definition in elementary torch operations (float32, rounded once at the end), or the
calls a user makes of vknn_b200. listed() holds fixed cases, draw() gives more of the same ranges.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}


def listed():
    return [
        # a handful of short prompts that arrive together, the head layout of a 12 x 64 encoder layer: latency
        dict(name="prompt short", op="prompt", n=4, lo=1, hi=48, prefix=0, hq=12, hkv=12, d=64, causal=True, dtype="f16", salt=1),
        # a serving batch: prompts of mixed odd lengths, some of which continue a prefix that is in memory already
        dict(name="prompt mixed", op="prompt", n=16, lo=64, hi=1500, prefix=700, hq=32, hkv=8, d=128, causal=True, dtype="bf16", salt=2),
        # images of different sizes through an encoder's bidirectional attention, 16 heads x 64, up to 2738 patches
        dict(name="images packed", op="prompt", n=8, lo=197, hi=2738, prefix=0, hq=16, hkv=16, d=64, causal=False, dtype="f16", salt=3),
        # long prompts back to back: the largest case
        dict(name="prompt long", op="prompt", n=8, lo=512, hi=4096, prefix=0, hq=32, hkv=8, d=128, causal=True, dtype="bf16", salt=4),
        # one new token for each of a few sequences: latency
        dict(name="store token few", op="store", n=3, lo=0, hi=0, filled=333, hkv=12, d=64, lmax=512, block=32, dtype="f16", codes="i8", salt=5),
        # one new token for each sequence of a decode batch over the 8192-token cache
        dict(name="store token", op="store", n=32, lo=0, hi=0, filled=8191, hkv=8, d=128, lmax=8192, block=64, dtype="f16", codes="e4m3", salt=6),
        # a batch of prompts of mixed lengths behind what the sequences hold already
        dict(name="store prompts", op="store", n=16, lo=64, hi=1500, filled=500, hkv=8, d=128, lmax=2048, block=32, dtype="bf16", codes="i8", salt=7),
        # long prompts into an empty cache
        dict(name="store long", op="store", n=8, lo=512, hi=8192, filled=0, hkv=8, d=128, lmax=8192, block=128, dtype="bf16", codes="e4m3", salt=8),
        # one sequence at its beginning, a head for each query head: latency
        dict(name="decode one", op="decode", n=1, lo=200, hi=331, hq=12, hkv=12, d=64, lmax=512, block=32, dtype="f16", codes="i8", salt=9),
        # many short conversations
        dict(name="decode short", op="decode", n=64, lo=100, hi=1000, hq=32, hkv=8, d=128, lmax=1024, block=32, dtype="bf16", codes="i8", salt=10),
        # the decode batch: 32 sequences, lengths uniform in [1024, 8192], 32 query heads on 8 kv heads
        dict(name="decode batch", op="decode", n=32, lo=1024, hi=8192, hq=32, hkv=8, d=128, lmax=8192, block=64, dtype="f16", codes="e4m3", salt=11),
        # two very long contexts
        dict(name="decode long", op="decode", n=2, lo=90000, hi=131000, hq=32, hkv=8, d=128, lmax=131072, block=128, dtype="bf16", codes="e4m3", salt=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["prompt", "store", "decode"])
    c = dict(op=op, dtype=rng.choice(["f16", "bf16"]), d=rng.choice([64, 128]), salt=rng.randrange(1 << 20))
    c["hkv"] = rng.choice([1, 2, 4, 8, 12])
    if op == "prompt":
        c["hq"] = c["hkv"] * rng.choice([1, 2, 4])
        c["n"], c["causal"] = _log(rng, 1, 16), rng.random() < 0.7
        c["hi"] = _log(rng, 4, 900 if c["n"] > 8 or c["hq"] > 32 else 1800 if c["n"] > 4 else 4000 if c["causal"] else 2500)
        c["lo"] = rng.randint(0, c["hi"])
        c["prefix"] = 0 if rng.random() < 0.5 else _log(rng, 1, 600)
        return c
    c["n"], c["block"], c["codes"] = _log(rng, 1, 64), rng.choice([32, 64, 128]), rng.choice(["e4m3", "i8"])
    row = c["n"] * c["hkv"] * c["d"]
    c["lmax"] = c["block"] * max(1, _log(rng, 64, max(128, min(131072 if op == "decode" else 8192, 240_000_000 // row))) // c["block"])
    if op == "store":
        if rng.random() < 0.5:  # one token each
            c["lo"] = c["hi"] = 0
            c["filled"] = rng.randint(0, c["lmax"] - 1)
        else:
            c["hi"] = _log(rng, 1, max(1, min(c["lmax"], 34_000_000 // row)))
            c["lo"] = rng.randint(0, c["hi"])
            c["filled"] = rng.randint(0, c["lmax"] - c["hi"])
        return c
    c["hq"] = c["hkv"] * rng.choice([1, 2, 3, 4, 8, 16])
    c["hi"] = rng.randint(1, c["lmax"])
    c["lo"] = rng.randint(1, c["hi"])
    return c


def _lengths(n, lo, hi, salt):
    """n lengths in [lo, hi], the first of them hi: part of the case, the same for every seed."""
    r = random.Random(salt * 7919 + 13)
    return [hi] + [r.randint(lo, hi) for _ in range(n - 1)]


def _plan(case):
    """(new tokens, tokens before them) of each sequence."""
    n = case["n"]
    if case["op"] == "decode":
        return [1] * n, [x - 1 for x in _lengths(n, case["lo"], case["hi"], case["salt"])]
    new = _lengths(n, case["lo"], case["hi"], case["salt"]) if case["hi"] else [1] * n
    before = case["prefix"] if case["op"] == "prompt" else case["filled"]
    return new, _lengths(n, 0, before, case["salt"] + 1)


def _offsets(lengths):
    at = [0]
    for x in lengths:
        at.append(at[-1] + x)
    return at


def _rows(g, t, h, d, dtype):
    """Keys or values of t tokens: normal, tokens of differing size, a few large channels."""
    x = torch.randn(t, h, d, generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(t, 1, 1, generator=g, device="cuda"))
    x[..., ::37] *= 3.0
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    new, before = _plan(case)
    n, d, dtype, hkv = case["n"], case["d"], TYPES[case["dtype"]], case["hkv"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"op": case["op"]}
    if case["op"] == "prompt":
        hq, tq, tk = case["hq"], sum(new), sum(new) + sum(before)
        s["cu_q"], s["longest"] = ints(_offsets(new)), (max(new), max(a + b for a, b in zip(new, before)))
        if tk == tq:  # views of one packed projection [tokens, hq + 2 hkv, d]
            qkv = torch.randn(tq, hq + 2 * hkv, d, generator=g, device="cuda").to(dtype)
            s["q"], s["k"], s["v"], s["cu_k"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], s["cu_q"]
        else:
            s["q"] = torch.randn(tq, hq, d, generator=g, device="cuda").to(dtype)
            s["k"], s["v"] = (torch.randn(tk, hkv, d, generator=g, device="cuda").to(dtype) for _ in range(2))
            s["cu_k"] = ints(_offsets([a + b for a, b in zip(new, before)]))
        s["o"] = torch.zeros(tq, hq, d, dtype=dtype, device="cuda")
        s["scale"], s["causal"] = d ** -0.5, case["causal"]
        return s
    lmax, block, codes = case["lmax"], case["block"], CODES[case["codes"]]
    s["len"] = ints(before)
    # what the cache holds: values of a block lie within +-448 (e4m3) or +-127 (int8) of the block's scale
    held = max(b + (1 if case["op"] == "decode" else 0) for b in before)
    held = -(-held // block) * block
    for x in "kv":
        c = torch.zeros(n, hkv, lmax, d, dtype=codes, device="cuda")
        z = torch.zeros(n, hkv, lmax // block, device="cuda")
        if held:
            w = torch.randn(n, hkv, held, d, generator=g, device="cuda")
            if codes == torch.int8:
                c[:, :, :held] = (w * 32).round().clamp(-127, 127).to(codes)
                z[:, :, :held // block] = 0.03 * torch.exp(0.3 * torch.randn(n, hkv, held // block, generator=g, device="cuda"))
            else:
                c.view(torch.uint8)[:, :, :held] = (w * 64).clamp(-448, 448).to(codes).view(torch.uint8)
                z[:, :, :held // block] = torch.exp2(torch.randint(-7, -5, (n, hkv, held // block), generator=g, device="cuda").float())
        s[x + "c"], s[x + "s"] = c, z
    if case["op"] == "store":
        t = sum(new)
        s["k"], s["v"] = _rows(g, t, hkv, d, dtype), _rows(g, t, hkv, d, dtype)
        s["cu"] = ints(_offsets(new)) if case["hi"] else None
        return s
    s["len"] += 1
    s["q"] = torch.randn(n, case["hq"], d, generator=g, device="cuda").to(dtype)
    s["o"] = torch.zeros_like(s["q"])
    s["scale"] = d ** -0.5
    return s


_contexts = {}


def _context():
    import vknn_b200
    at = torch.cuda.current_device()
    if at not in _contexts:
        _contexts[at] = vknn_b200.Context(at)
    return _contexts[at]


def run(s):
    if s["op"] == "prompt":
        if own:
            _context().attn_prefill_packed(s["q"], s["k"], s["v"], s["o"], s["scale"], s["cu_q"], cu_k=s["cu_k"], causal=s["causal"])
            return s["o"]
        return _prompt_plain(s)
    if s["op"] == "store":
        if own:
            _context().kv_append_q8(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["len"], cu=s["cu"])
        else:
            _store_plain(s, "k")
            _store_plain(s, "v")
        return {"k": s["kc"], "v": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}
    if own:
        _context().attn_decode_q8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["o"], s["scale"], kv_len=s["len"])
        return s["o"]
    return _decode_plain(s)


def _softmax_rows(x):
    """exp(x - max) / sum in place; a row with nothing to see is 0 / 0."""
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    return x.div_(x.sum(-1, keepdim=True))


def _prompt_plain(s):
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"].long(), s["cu_k"].long()
    (mq, mk), n, hq, hkv = s["longest"], cu_q.numel() - 1, q.shape[1], k.shape[1]
    iq, ik = torch.arange(mq, device="cuda"), torch.arange(mk, device="cuda")
    lq, lk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    at_q = (cu_q[:-1, None] + iq).clamp(max=q.shape[0] - 1)
    at_k = (cu_k[:-1, None] + ik).clamp(max=k.shape[0] - 1)
    # padded to the longest sequence, kv heads beside the query heads of their group
    qp = q[at_q].float().reshape(n, mq, hkv, hq // hkv, -1).permute(0, 2, 3, 1, 4)
    kp = k[at_k].float().permute(0, 2, 3, 1).unsqueeze(2)
    vp = v[at_k].float().permute(0, 2, 1, 3).unsqueeze(2)
    sees = (ik < lk[:, None])[:, None, :]
    if s["causal"]:
        sees = sees & (ik <= iq[:, None] + (lk - lq)[:, None, None])
    x = torch.matmul(qp, kp).mul_(s["scale"]).masked_fill_(~sees[:, None, None], -math.inf)
    o = torch.matmul(_softmax_rows(x), vp).permute(0, 3, 1, 2, 4).reshape(n, mq, hq, -1)
    return o[iq < lq[:, None]].to(q.dtype)


def _scale_of(top, codes):
    """The scale of a block whose largest magnitude is `top`."""
    if codes == torch.int8:
        s = (top / torch.full_like(top, 127.0)).clamp(min=2.0 ** -126)  # (by a tensor: a quotient rounded once)
    else:  # the least power of two with top <= 448 * scale
        f, e = torch.frexp(top)
        s = torch.ldexp(torch.ones_like(top), torch.where(f <= 0.875, e - 9, e - 8).clamp(min=-126))
    return torch.where(top == 0, torch.zeros_like(top), s)


def _codes_of(x, s, codes):
    """x / s to the nearest code, ties to even, in 64 bits: a quotient next to a border falls on its own side."""
    y = torch.where(s == 0, torch.zeros_like(x), x / torch.where(s == 0, torch.ones_like(s), s))
    return y.round().clamp(-127, 127).to(torch.int8) if codes == torch.int8 else y.float().to(codes).view(torch.int8)


def _store_plain(s, which):
    x, cache, scales, held = s[which], s[which + "c"], s[which + "s"], s["len"].long()
    codes, (n, hkv, lmax, d), nb = cache.dtype, cache.shape, scales.shape[2]
    block, raw, seqs = lmax // nb, cache.view(torch.int8), torch.arange(n, device="cuda")
    if s["cu"] is None:
        b, pos = seqs, held
    else:
        r = torch.arange(x.shape[0], device="cuda")
        b = torch.searchsorted(s["cu"].long(), r, right=True) - 1
        pos = held[b] + r - s["cu"].long()[b]
    blk = pos // block
    # largest new magnitude of each block and head, and the scale that it asks for
    top = x.float().abs().amax(-1)
    most = torch.zeros(n * nb, hkv, device="cuda").scatter_reduce_(0, (b * nb + blk)[:, None].expand(-1, hkv), top, "amax")
    most = most.reshape(n, nb, hkv).permute(0, 2, 1)
    touched = torch.zeros(n * nb, dtype=torch.bool, device="cuda").index_fill_(0, b * nb + blk, True).reshape(n, 1, nb)
    fresh = _scale_of(most, codes)
    # the block each sequence had begun: its older codes count, and are requantised where the scale grows
    first = (held // block).clamp(max=nb - 1)
    begun = (held % block > 0)[:, None] & touched.squeeze(1).gather(1, first[:, None])
    old = scales[seqs, :, first]
    now = torch.where(begun, torch.maximum(old, fresh[seqs, :, first]), fresh[seqs, :, first])
    fresh[seqs, :, first] = now
    at = first[:, None] * block + torch.arange(block, device="cuda")
    past = raw[seqs[:, None], :, at]  # [n, block, hkv, d]
    value = past.view(codes).double() if codes != torch.int8 else past.double()
    again = _codes_of(value * old[:, None, :, None].double(), now[:, None, :, None].double(), codes)
    grew = begun[:, None, :, None] & (now > old)[:, None, :, None] & (at < held[:, None])[:, :, None, None]
    raw[seqs[:, None], :, at] = torch.where(grew, again, past)
    scales.copy_(torch.where(touched, fresh, scales))
    raw[b, :, pos] = _codes_of(x.double(), scales[b, :, blk][..., None].double(), codes)


def _decode_plain(s):
    q, n, hkv, lmax, nb = s["q"], *s["kc"].shape[:3], s["ks"].shape[2]
    k = (s["kc"].float().reshape(n, hkv, nb, -1) * s["ks"][..., None]).reshape(s["kc"].shape)
    v = (s["vc"].float().reshape(n, hkv, nb, -1) * s["vs"][..., None]).reshape(s["vc"].shape)
    x = torch.matmul(q.float().reshape(n, hkv, q.shape[1] // hkv, -1), k.transpose(2, 3)).mul_(s["scale"])
    x.masked_fill_(torch.arange(lmax, device="cuda") >= s["len"][:, None, None, None], -math.inf)
    return torch.matmul(_softmax_rows(x), v).reshape(q.shape).to(q.dtype)


def _pairs(case):
    """Visible (query, key) pairs over all sequences, for one head."""
    new, before = _plan(case)
    return sum(a * b + (a * (a + 1) // 2 if case["causal"] else a * a) for a, b in zip(new, before))


def work(case):
    new, before = _plan(case)
    n, d, hkv = case["n"], case["d"], case["hkv"]
    if case["op"] == "prompt":
        t = sum(new)
        return {"bytes": 4.0 * t * case["hq"] * d + 4.0 * (t + sum(before)) * hkv * d + 8.0 * n, "flops": 4.0 * d * case["hq"] * _pairs(case)}
    block = case["block"]
    if case["op"] == "store":
        blocks = sum((b + a - 1) // block - b // block + 1 for a, b in zip(new, before) if a)
        return {"bytes": 2.0 * hkv * (3.0 * sum(new) * d + 4.0 * blocks), "flops": 4.0 * hkv * sum(new) * d}
    held = [b + 1 for b in before]
    return {"bytes": 2.0 * hkv * (sum(held) * d + 4.0 * sum(-(-x // block) for x in held)) + 4.0 * n * case["hq"] * d, "flops": 4.0 * d * case["hq"] * sum(held)}


def exact(case, seed):
    s = prepare(case, seed)
    new, before = _plan(case)
    if case["op"] == "prompt":
        out, at_q, at_k, group = [], 0, 0, case["hq"] // case["hkv"]
        for a, b in zip(new, before):
            heads = []
            for h in range(case["hq"]):
                q = s["q"][at_q:at_q + a, h].double()
                k, v = (s[x][at_k:at_k + a + b, h // group].double() for x in "kv")
                x = (q @ k.T) * s["scale"]
                if s["causal"]:
                    x += torch.full_like(x, -math.inf).triu(b + 1)
                heads.append(torch.softmax(x, -1) @ v)
            out.append(torch.stack(heads, 1))
            at_q, at_k = at_q + a, at_k + a + b
        return torch.cat(out)
    if case["op"] == "decode":
        out, group, block = [], case["hq"] // case["hkv"], case["block"]
        for i, b in enumerate(before):
            scale = {x: s[x + "s"][i].double().repeat_interleave(block, 1)[:, :b + 1, None] for x in "kv"}
            k, v = (s[x + "c"][i, :, :b + 1].double() * scale[x] for x in "kv")
            x = torch.einsum("hgd,hld->hgl", s["q"][i].double().reshape(case["hkv"], group, -1), k) * s["scale"]
            out.append(torch.einsum("hgl,hld->hgd", torch.softmax(x, -1), v).reshape(case["hq"], -1))
        return torch.stack(out)
    # the store, block by block in one sequence after the other. The scale of int8 codes is a quotient that the cache rounds to
    # 32 bits, and the codes follow the rounded one: they are whole numbers, which have to be the same on both sides.
    at, power = 0, case["codes"] == "e4m3"
    for x in "kv":
        s[x + "s"] = s[x + "s"].double()
    for i, (a, b) in enumerate(zip(new, before)):
        for x in "kv":
            for blk in range(b // case["block"], -(-(a + b) // case["block"])) if a else ():
                lo, hi = blk * case["block"], min(a + b, (blk + 1) * case["block"])
                first = max(lo, b)
                fresh = s[x][at + first - b:at + hi - b].double().transpose(0, 1)  # [hkv, tokens, d]
                top = fresh.abs().amax((1, 2))
                want = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-126)) if power else top / 127.0
                was = s[x + "s"][i, :, blk].clone() if first > lo else torch.zeros_like(want)
                now = torch.maximum(want, was)
                s[x + "s"][i, :, blk] = now
                if power:
                    cells, div = s[x + "c"].view(torch.uint8)[i, :, lo:hi], torch.where(now > 0, now, torch.ones_like(now))[:, None, None]
                    old = s[x + "c"][i, :, lo:first].double() * was[:, None, None]
                    cells.copy_((torch.cat([old, fresh], 1) / div).float().to(torch.float8_e4m3fn).view(torch.uint8))
        at += a
    return {"k": s["kc"] if power else None, "v": s["vc"] if power else None, "k_scale": s["ks"], "v_scale": s["vs"]}
