"""Serving in four bits, as measurable cases: weights and a paged KV cache in
MXFP4, the OCP microscaling format.

A value is code * 2^(scale - 127): sixteen e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4,
6 and their negatives; two a byte, the low nibble first) and one e8m0 scale byte
for every 32 values along a row (the last group of a row may be shorter). Scale
255 makes its group NaN.

Weights are rounded once and read back to be looked at (codec), and a Linear
multiplies f32 activations with them (linear). A server's new keys and values
are finished (per-head RMSNorm, rotation) and go into pages in four bits (store:
the append, and the rows read back from the pages), and tokens attend over them
(attend). Pools are [pages, KV heads, page size, head dim / 2] bytes with scales
[pages, KV heads, page size, ceil(head dim / 32)]. A batch is a ragged set of
token rows: cu_seqlens [seqs + 1], kv_lens [seqs] (cached tokens including this
call's) and a page table [seqs, pages per sequence], all int32. Token i of a
sequence's n stands at position kv_len - n + i.
"""
import math
import random

import torch

own = False

GROUP = 32
NAN_SCALE = 255
TINY = 2.0 ** -100   # groups below it throughout are stored as zeros
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
THETA = 1_000_000.0
EPS = 1e-6

QWEN3 = dict(hq=16, hkv=8, hd=128)    # Qwen3-0.6B heads
QWEN25 = dict(hq=14, hkv=2, hd=64)    # Qwen2.5-0.5B heads: 7 query heads per KV head
GPT2 = dict(hq=12, hkv=12, hd=64)     # GPT-2 small: one KV head per query head
LAYOUTS = (QWEN3, QWEN25, GPT2, dict(hq=25, hkv=25, hd=64), dict(hq=32, hkv=8, hd=128), dict(hq=8, hkv=1, hd=256),
           dict(hq=6, hkv=2, hd=96), dict(hq=20, hkv=1, hd=80))
# [out, in] of Linears: Qwen3-0.6B's fused q/k/v and its output projection, GPT-2 XL's FFN, Qwen2.5-0.5B's down
# projection, a 4096-wide model's square and its FFN
LINEARS = ((4096, 1024), (1024, 2048), (6400, 1600), (1600, 6400), (896, 4864), (4096, 4096), (14336, 4096))


def listed():
    return [
        # a few rows there and back: latency
        dict(name="codec_rows", op="codec", dtype="f32", rows=33, cols=1000),
        # a model's largest weight, from the checkpoint's bf16
        dict(name="codec_table", op="codec", dtype="bf16", rows=151936, cols=1024),
        # one token through a fused q/k/v projection: one launch's latency
        dict(name="linear_1", op="linear", rows=1, out=4096, cols=1024, bias=False, gelu=False, residual=False),
        # one token through a tied LM head: weights from memory
        dict(name="linear_1_head", op="linear", rows=1, out=151936, cols=1024, bias=False, gelu=False, residual=False),
        # a decode batch through the first FFN Linear of GPT-2 XL
        dict(name="linear_16_ffn", op="linear", rows=16, out=6400, cols=1600, bias=True, gelu=True, residual=False),
        # a prompt through an output projection, added to the residual stream
        dict(name="linear_2000", op="linear", rows=2000, out=4096, cols=4096, bias=True, gelu=False, residual=True),
        # a decode step of 64 conversations
        dict(name="store_step_64", op="store", norm=True, rope=True, page=16, seqs=64, chunks=0, new=1, kv=501, **QWEN3),
        # prompts of several requests at once, heads without norms
        dict(name="store_prompts", op="store", norm=False, rope=True, page=32, seqs=5, chunks=5, new=4095, kv=4999,
             **QWEN25),
        # one conversation's next token: few rows, a short cache
        dict(name="attend_step_1", op="attend", page=16, seqs=1, chunks=0, new=1, kv=777, **QWEN3),
        # a decode step of 64 conversations of all lengths
        dict(name="attend_step_64", op="attend", page=16, seqs=64, chunks=0, new=1, kv=8192, **QWEN3),
        # a chunk of a long prompt behind what is cached already
        dict(name="attend_chunk_2048", op="attend", page=16, seqs=1, chunks=1, new=2048, kv=16384, **QWEN3),
        # one server step: decoding conversations and prompts' chunks in one batch
        dict(name="attend_mixed", op="attend", page=32, seqs=27, chunks=3, new=511, kv=2047, **GPT2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("codec", "linear", "linear", "store", "attend", "attend"))
    if op == "codec":
        cols = 8 * _log(rng, 1, 1024)
        return dict(op=op, dtype=rng.choice(("f32", "bf16")), rows=_log(rng, 1, max(1, (64 << 20) // cols)), cols=cols)
    if op == "linear":
        out, cols = rng.choice(LINEARS + ((_log(rng, 16, 20000), 8 * _log(rng, 8, 1024)),) * 5)
        rows = rng.choice((1, rng.randint(2, 16), _log(rng, 17, 2000)))
        while rows * out * cols > 2000 * 4096 * 4096:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, out=out, cols=cols, bias=rng.random() < 0.5, gelu=rng.random() < 0.3,
                    residual=rng.random() < 0.4)
    c = dict(op=op, page=rng.choice((16, 32, 64, 24)))
    c.update(rng.choice(LAYOUTS))
    row = c["hkv"] * c["hd"]
    c["seqs"] = _log(rng, 1, 64)
    if op == "store":
        c["norm"], c["rope"] = rng.random() < 0.5, rng.random() < 0.8
        c["chunks"] = rng.choice((0, rng.randint(0, min(c["seqs"], 5))))
        c["new"] = _log(rng, 2, 2048) if c["chunks"] else 1
        c["kv"] = _log(rng, c["new"], max(c["new"], 4096))
        limit = 32 << 20
    else:
        c["chunks"] = rng.choice((0, rng.randint(0, min(c["seqs"], 4))))
        c["new"] = _log(rng, 2, 1024) if c["chunks"] else 1
        c["kv"] = _log(rng, max(16, c["new"]), 32768)
        limit = 256 << 20
        while c["seqs"] * c["hq"] * c["new"] * c["kv"] > (256 << 20) and c["new"] > 1:
            c["new"] = (c["new"] + 1) // 2 if c["new"] > 2 else 2
            if c["new"] == 2:
                c["kv"] = max(16, c["kv"] // 2)
    while c["seqs"] * c["kv"] * row > limit:
        if c["seqs"] > 1:
            c["seqs"] //= 2
        else:
            c["kv"] //= 2
    c["chunks"] = min(c["chunks"], c["seqs"])
    c["new"] = min(c["new"], c["kv"])
    return c


# ---------------------------------------------------------------- the format, in elementary operations

def _encode(x):
    """Codes [..., cols / 2] (two a byte) and scales [..., groups] of f32 rows: the scale is the smallest power of two
    that the group's largest magnitude exceeds at most 7 times, so that rounding to nearest even clips nothing by more
    than half a step."""
    cols = x.shape[-1]
    groups = -(-cols // GROUP)
    if cols % GROUP:
        x = torch.cat([x, x.new_zeros(x.shape[:-1] + (groups * GROUP - cols,))], -1)
    x = x.reshape(x.shape[:-1] + (groups, GROUP))
    top = x.abs().amax(-1)
    power = ((top.view(torch.int32) + 0x1FFFFF) >> 23) - 2
    live, odd = top >= TINY, ~torch.isfinite(top)
    power = torch.where(live & ~odd, power, torch.full_like(power, 127))
    t = x * ((254 - power) << 23).view(torch.float32).unsqueeze(-1)
    a = t.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    code = code + 8 * torch.signbit(t).to(torch.uint8)
    code = code * (live & ~odd).unsqueeze(-1)
    scale = torch.where(odd, torch.full_like(power, NAN_SCALE), torch.where(live, power, torch.zeros_like(power)))
    code = code.flatten(-2)[..., :cols]
    return (code[..., 0::2] + 16 * code[..., 1::2]).contiguous(), scale.to(torch.uint8).contiguous()


def _decode(codes, scales):
    """f32 values [..., cols]."""
    value = torch.tensor(VALUES + tuple(-v for v in VALUES), device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    cols = c.shape[-1]
    bits = scales.int()
    bits = torch.where(bits == 0, torch.full_like(bits, 1 << 22), bits << 23)  # 2^-127 has no exponent of its own
    power = torch.where(scales == NAN_SCALE, torch.full((), math.nan, device=codes.device), bits.view(torch.float32))
    return value[c.int()] * power.repeat_interleave(GROUP, -1)[..., :cols]


# ---------------------------------------------------------------- inputs

def _lens(case):
    """Cached length and new tokens of each sequence: the first one has the most, the others any."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    kv, new = [], []
    for i in range(case["seqs"]):
        n = (case["new"] if i == 0 else r.randint(1, case["new"])) if i < case["chunks"] else 1
        kv.append(case["kv"] if i == 0 else max(n, _log(r, max(1, case["kv"] // 16), case["kv"])))
        new.append(n)
    return kv, new


def _rope_tables(hd, rows):
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = dict(case)
    if own:
        from gorch_amd import hip

        hip.init(0)
        s["hip"] = hip
    if case["op"] == "codec":
        rows, cols = case["rows"], case["cols"]
        kind = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        # rows of a weight differ in size, and so do their parts
        s["x"] = torch.empty((rows, cols), dtype=kind, device="cuda")
        for at in range(0, rows, 16384):
            part = s["x"][at:at + 16384]
            part.copy_(normal(*part.shape) * torch.exp(0.5 * normal(part.shape[0], 1)) * 0.02)
        s["codes"] = torch.empty((rows, cols // 2), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty((rows, -(-cols // GROUP)), dtype=torch.uint8, device="cuda")
        s["values"] = torch.empty_like(s["x"])
        return s
    if case["op"] == "linear":
        rows, out, cols = case["rows"], case["out"], case["cols"]
        parts = []
        for at in range(0, out, 16384):
            n = min(16384, out - at)
            parts.append(_encode(normal(n, cols) * torch.exp(0.5 * normal(n, 1)) / math.sqrt(cols)))
        s["codes"], s["scales"] = (torch.cat(p) for p in zip(*parts))
        del parts
        # a few channels of a residual stream are much larger than the others
        s["x"] = normal(rows, cols) * torch.exp(0.8 * normal(cols))
        s["b"] = normal(out) if case["bias"] else None
        s["r"] = normal(rows, out) if case["residual"] else None
        s["y"] = torch.empty((rows, out), device="cuda")
        if own:
            s["w"] = hip.pack_mxfp4(s["codes"], s["scales"])
            s["ws"] = hip.linear_mxfp4_workspace(rows, out, cols)
        return s
    kv, new = _lens(case)
    page, hq, hkv, hd = case["page"], case["hq"], case["hkv"], case["hd"]
    per_seq = -(-max(kv) // page)
    need = [-(-n // page) for n in kv]
    pages, T = sum(need), sum(new)
    order = torch.randperm(pages, generator=g, device="cuda").int()
    # entries past a sequence's last page are never looked at
    col = torch.arange(per_seq, device="cuda")
    first = torch.tensor([0] + need, device="cuda").cumsum(0)
    used = torch.tensor(need, device="cuda")
    s["page_table"] = order[(first[:-1, None] + torch.minimum(col[None], used[:, None] - 1)).long()].contiguous()
    s["cu_seqlens"] = torch.tensor([0] + new, device="cuda").cumsum(0).int()
    s["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["tokens"], s["max_new"] = T, max(new)
    shape = (pages, hkv, page)
    if case["op"] == "store":
        for name in ("k", "v"):
            s[name] = torch.zeros(shape + (hd // 2,), dtype=torch.uint8, device="cuda")
            s[name + "_scale"] = torch.zeros(shape + (-(-hd // GROUP),), dtype=torch.uint8, device="cuda")
            s[name + "_out"] = torch.empty((T, hkv * hd), device="cuda")
        # what the fused projection leaves: q, k and v side by side in a row
        s["qkv"] = normal(T, (hq + 2 * hkv) * hd)
        s["q_out"] = torch.empty((T, hq * hd), device="cuda")
        s["q_gain"] = 1 + 0.2 * normal(hd) if case["norm"] else None
        s["k_gain"] = 1 + 0.2 * normal(hd) if case["norm"] else None
        s["cos"], s["sin"] = _rope_tables(hd, max(kv)) if case["rope"] else (None, None)
    else:
        for name in ("k", "v"):
            s[name] = torch.empty(shape + (hd // 2,), dtype=torch.uint8, device="cuda")
            s[name + "_scale"] = torch.empty(shape + (-(-hd // GROUP),), dtype=torch.uint8, device="cuda")
            step = max(1, (16 << 20) // (hkv * page * hd))
            for at in range(0, pages, step):
                n = min(step, pages - at)
                x = normal(n, hkv, page, hd) * torch.exp(0.3 * normal(n, hkv, page, 1))
                s[name][at:at + n], s[name + "_scale"][at:at + n] = _encode(x)
        s["q"] = normal(T, hq * hd) * 1.5
        s["out"] = torch.empty((T, hq * hd), device="cuda")
    if own:
        s["cache"] = hip.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = hip.PagedBatch(s["cu_seqlens"], s["kv_lens"], s["page_table"], T, max_new=max(new), max_kv=max(kv))
        if case["op"] == "store":
            s["heads"] = hip.GQA(dict(dim=hq * hd, num_q=hq, num_kv=hkv, head_dim=hd, norm_eps=EPS, q_norm=s["q_gain"],
                                      k_norm=s["k_gain"], rope=case["rope"], rope_cos=s["cos"], rope_sin=s["sin"],
                                      rope_max_seq=max(kv)))
        else:
            s["ws"] = s["cache"].workspace(s["batch"], hq)
    return s


# ---------------------------------------------------------------- the calls

def run(s):
    return {"codec": _codec, "linear": _linear, "store": _store, "attend": _attend}[s["op"]](s)


def _codec(s):
    if own:
        s["hip"].mxfp4_encode(s["x"], s["codes"], s["scales"])
        s["hip"].mxfp4_decode(s["codes"], s["scales"], s["values"])
    else:
        codes, scales = _encode(s["x"].float())
        s["codes"].copy_(codes)
        s["scales"].copy_(scales)
        s["values"].copy_(_decode(s["codes"], s["scales"]))
    return s["values"]


def _linear(s):
    if own:
        s["hip"].linear_mxfp4(s["x"], s["w"], s["out"], s["b"], s["y"], residual=s["r"],
                              epilogue=s["hip"].EPI_GELU if s["gelu"] else s["hip"].EPI_NONE, ws=s["ws"])
        return s["y"]
    y = torch.matmul(s["x"], _decode(s["codes"], s["scales"]).t())
    if s["b"] is not None:
        y = y + s["b"]
    if s["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(0.7978845608 * (y + 0.044715 * y * y * y)))
    if s["r"] is not None:
        y = y + s["r"]
    s["y"].copy_(y)
    return s["y"]


def _places(s):
    """Sequence, position, page and slot of every token row."""
    cu = s["cu_seqlens"].long()
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = s["kv_lens"].long()[seq] - cu[seq + 1] + t
    return seq, pos, s["page_table"][seq, pos // s["page"]].long(), pos % s["page"]


def _head_norm(x, gain):
    """The sum of squares in 64 bits, every product rounded on its own."""
    if gain is None:
        return x
    inv = (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float()
    return x * inv * gain


def _rotate(x, cos, sin):
    if cos is None:
        return x
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _store(s):
    """The new rows into the pages, and what the pages then hold of them."""
    hq, hkv, hd, T = s["hq"], s["hkv"], s["hd"], s["tokens"]
    widths = [hq * hd, hkv * hd, hkv * hd]
    if own:
        q, k, v = s["qkv"].split(widths, 1)
        s["cache"].append(s["batch"], s["heads"], q, k, v, s["q_out"])
        s["cache"].read(s["batch"], s["k_out"], s["v_out"])
    else:
        q, k, v = (x.reshape(T, -1, hd) for x in s["qkv"].split(widths, 1))
        _, pos, page, slot = _places(s)
        cos, sin = (None, None) if s["cos"] is None else (s["cos"][pos][:, None], s["sin"][pos][:, None])
        s["q_out"].view(T, hq, hd).copy_(_rotate(_head_norm(q, s["q_gain"]), cos, sin))
        k = _rotate(_head_norm(k, s["k_gain"]), cos, sin)
        s["k"][page, :, slot], s["k_scale"][page, :, slot] = _encode(k)
        s["v"][page, :, slot], s["v_scale"][page, :, slot] = _encode(v)
        s["k_out"].copy_(_decode(s["k"][page, :, slot], s["k_scale"][page, :, slot]).view(T, -1))
        s["v_out"].copy_(_decode(s["v"][page, :, slot], s["v_scale"][page, :, slot]).view(T, -1))
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _gathered(s, name):
    """[seqs, KV heads, padded length, head dim] f32 of one pool."""
    table = s["page_table"].long()
    x = _decode(s[name], s[name + "_scale"])[table]
    return x.transpose(1, 2).reshape(table.shape[0], s["hkv"], -1, s["hd"])


def _attend(s):
    if own:
        s["cache"].attention(s["batch"], s["q"], s["out"], ws=s["ws"])
        return s["out"]
    hq, hkv, hd, T, N = s["hq"], s["hkv"], s["hd"], s["tokens"], s["max_new"]
    group = hq // hkv
    seq, pos, _, _ = _places(s)
    seqs = s["kv_lens"].shape[0]
    at = torch.arange(T, device="cuda") - s["cu_seqlens"].long()[seq]
    q = torch.zeros((seqs, N, hkv, group, hd), device="cuda")
    q[seq, at] = s["q"].view(T, hkv, group, hd) * (1.0 / math.sqrt(hd))
    where = torch.full((seqs, N), -1, device="cuda")
    where[seq, at] = pos
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, hkv, group * N, hd)
    k = _gathered(s, "k")
    length = k.shape[2]
    p = torch.matmul(q, k.transpose(2, 3).contiguous())
    del k
    v = _gathered(s, "v")
    # keys past a sequence's end: whatever their pages hold is not used
    v.mul_((torch.arange(length, device="cuda") < s["kv_lens"][:, None])[:, None, :, None])
    seen = torch.arange(length, device="cuda") <= where[..., None]
    p = p.view(seqs, hkv, group, N, length).masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True).clamp_min_(torch.finfo(torch.float32).min)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, hkv, group * N, length), v).view(seqs, hkv, group, N, hd)
    o = o / total.clamp_min(1e-30)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4)[seq, at].reshape(T, hq * hd))
    return s["out"]


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "codec":
        n, size = case["rows"] * case["cols"], 4 if case["dtype"] == "f32" else 2
        held = n // 2 + case["rows"] * -(-case["cols"] // GROUP)
        return {"bytes": 2 * n * size + 2 * held, "flops": 4 * n}
    if case["op"] == "linear":
        m, n, k = case["rows"], case["out"], case["cols"]
        b = 4 * m * k + n * (k // 2 + -(-k // GROUP)) + 4 * m * n * (2 if case["residual"] else 1)
        return {"bytes": b + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    kv, new = _lens(case)
    T, hq, hkv, hd = sum(new), case["hq"], case["hkv"], case["hd"]
    row = 2 * hkv * (hd // 2 + -(-hd // GROUP))  # one token's K and V in the cache
    tables = 4 * sum(-(-n // case["page"]) for n in kv) + 8 * len(kv)
    if case["op"] == "store":
        moved = T * (4 * hd * (2 * hq + 2 * hkv) + row) + (T * 4 * hd if case["rope"] else 0)
        return {"bytes": moved + T * (row + 8 * hkv * hd) + 8 * len(kv), "flops": 8 * T * (hq + 2 * hkv) * hd}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for length, n in zip(kv, new))
    return {"bytes": sum(kv) * row + 8 * T * hq * hd + tables, "flops": 4 * hd * hq * pairs}


# ---------------------------------------------------------------- the definitions, in 64 bits

def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _held(codes, scales):
    """The values of codes and scales, in 64 bits."""
    c = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.int64, device=codes.device)
    c[..., 0::2] = codes & 15
    c[..., 1::2] = codes >> 4
    mantissa, power = c & 1, (c >> 1) & 3
    quarters = torch.where(power == 0, 2 * mantissa, (2 + mantissa) << power)
    which = torch.arange(c.shape[-1], device=codes.device) // GROUP
    return torch.where(c >= 8, -quarters, quarters) * _two_to(scales.long() - 129)[..., which]


def _nearest(x):
    """What a row of 64-bit values becomes: each group's nearest multiples of its power of two."""
    x = x.double()
    cols = x.shape[-1]
    which = torch.arange(cols, device=x.device) // GROUP
    top = torch.zeros(x.shape[:-1] + (-(-cols // GROUP),), dtype=torch.float64, device=x.device)
    top = top.scatter_reduce(-1, which.expand(x.shape), x.abs(), "amax")
    m, e = torch.frexp(top)  # top = m 2^e, at most 7 = 0.875 * 2^3 steps
    step = _two_to(torch.where(m <= 0.875, e - 3, e - 2))[..., which]
    a = (x / step).abs()
    grid = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    y = (torch.round(a / grid) * grid).clamp_max(6)  # (halves go to the even multiple, whose last code bit is 0)
    return torch.where(top[..., which] >= TINY, torch.copysign(y, x) * step, torch.zeros_like(x))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "codec":
        out = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
        for at in range(0, case["rows"], 8192):
            out[at:at + 8192] = _nearest(s["x"][at:at + 8192])
        return out
    if case["op"] == "linear":
        y = torch.empty(s["y"].shape, dtype=torch.float64, device="cuda")
        for at in range(0, case["out"], 8192):
            w = _held(s["codes"][at:at + 8192], s["scales"][at:at + 8192])
            y[:, at:at + 8192] = torch.mm(s["x"].double(), w.t().contiguous())
        if case["bias"]:
            y += s["b"].double()
        if case["gelu"]:
            # (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
            y = y / (1 + torch.exp(-2 * 0.7978845608 * (y + 0.044715 * y ** 3)))
        return y + s["r"].double() if case["residual"] else y
    kv, new = _lens(case)
    hq, hkv, hd, page = case["hq"], case["hkv"], case["hd"], case["page"]
    begin = 0
    if case["op"] == "store":
        x = s["qkv"].double().view(-1, hq + 2 * hkv, hd)
        q_out = torch.empty((x.shape[0], hq * hd), dtype=torch.float64, device="cuda")
        for i, n in enumerate(new):
            q = x[begin:begin + n, :hq]
            if case["norm"]:
                q = q / (q.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * s["q_gain"].double()
            if case["rope"]:
                turn = torch.complex(s["cos"].double(), s["sin"].double())[kv[i] - n:kv[i], None]
                q = torch.complex(*q.chunk(2, -1)) * turn
                q = torch.cat([q.real, q.imag], -1)
            q_out[begin:begin + n] = q.reshape(n, -1)
            begin += n
        # a finished key is an f32 value before it is rounded to four bits: 64 bits would round some of them another way
        return {"q": q_out, "k": None, "v": _nearest(x[:, hq + hkv:]).reshape(x.shape[0], -1)}
    out = torch.empty((sum(new), hq, hd), dtype=torch.float64, device="cuda")
    for i, n in enumerate(new):
        p = torch.arange(kv[i], device="cuda")
        at, slot = s["page_table"][i].long()[torch.div(p, page, rounding_mode="floor")], p.remainder(page)
        k, v = (_held(s[m][at, :, slot], s[m + "_scale"][at, :, slot]) for m in ("k", "v"))
        q = s["q"][begin:begin + n].double().view(n, hq, hd)
        seen = torch.ones((n, kv[i]), dtype=torch.bool, device="cuda").tril_(kv[i] - n)
        for h in range(hq):
            a = torch.mm(q[:, h], k[:, h * hkv // hq].t().contiguous()) / math.sqrt(hd)
            a = torch.softmax(a.masked_fill_(~seen, -math.inf), -1)
            out[begin:begin + n, h] = torch.mm(a, v[:, h * hkv // hq].contiguous())
        begin += n
    return out.view(sum(new), hq * hd)
