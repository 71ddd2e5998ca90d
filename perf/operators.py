"""The serving operators over a paged KV cache, as measurable cases.

One step of a server that holds many conversations: the keys and values of
the new tokens go into pages of a shared pool (with the per-head q/k RMSNorm
and the rotation in the same pass, in bf16 or quantised to e4m3), the new
tokens attend over their sequences' pages, rows of the cache are read back
where a sequence leaves the pool, and the logits get each request's penalties,
biases and grammar mask before a token is chosen.

Layout: pools [pages, KV heads, page size, head dim]; e4m3 scales [pages, KV
heads, page size], one f32 per (token, KV head). A batch is a ragged set of
token rows: cu_seqlens [seqs + 1], kv_lens [seqs] (cached tokens including
this call's) and a page table [seqs, pages per sequence], all int32. Token i
of a sequence's n stands at position kv_len - n + i.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0
THETA = 1_000_000.0
EPS = 1e-6

QWEN3 = dict(hq=16, hkv=8, hd=128)    # Qwen3-0.6B heads
QWEN25 = dict(hq=14, hkv=2, hd=64)    # Qwen2.5-0.5B heads: 7 query heads per KV head
GPT2 = dict(hq=12, hkv=12, hd=64)     # GPT-2 small: one KV head per query head
LAYOUTS = (QWEN3, QWEN25, GPT2, dict(hq=25, hkv=25, hd=64), dict(hq=32, hkv=8, hd=128), dict(hq=8, hkv=1, hd=256),
           dict(hq=6, hkv=2, hd=96), dict(hq=20, hkv=1, hd=80))


def listed():
    return [
        # one conversation's next token: one launch's latency
        dict(name="append_step_1", op="append", dtype="bf16", norm=True, rope=True, page=16, seqs=1, chunks=0, new=1,
             kv=777, **QWEN3),
        # a decode step of 64 conversations into a quantised cache
        dict(name="append_step_64_e4m3", op="append", dtype="e4m3", norm=True, rope=True, page=16, seqs=64, chunks=0,
             new=1, kv=501, **QWEN3),
        # prompts of several requests at once, heads without norms
        dict(name="append_prompts", op="append", dtype="e4m3", norm=False, rope=True, page=32, seqs=5, chunks=5,
             new=4095, kv=4999, **QWEN25),
        # one conversation leaves the pool for a contiguous cache
        dict(name="read_1_bf16", op="read", dtype="bf16", page=16, seqs=1, chunks=1, new=1000, kv=1000, **QWEN3),
        # many conversations are read back from a quantised pool
        dict(name="read_16_e4m3", op="read", dtype="e4m3", page=16, seqs=16, chunks=16, new=6001, kv=6001, **QWEN3),
        # one conversation's next token: few rows, a short cache
        dict(name="attend_step_1", op="attend", dtype="bf16", page=16, seqs=1, chunks=0, new=1, kv=777, **QWEN3),
        # a decode step of 64 conversations of all lengths, quantised
        dict(name="attend_step_64_e4m3", op="attend", dtype="e4m3", page=16, seqs=64, chunks=0, new=1, kv=8192,
             **QWEN3),
        # a few very long conversations: few rows over a long axis
        dict(name="attend_step_long", op="attend", dtype="bf16", page=64, seqs=3, chunks=0, new=1, kv=32749, **QWEN25),
        # a chunk of a long prompt behind what is cached already
        dict(name="attend_chunk_2048", op="attend", dtype="bf16", page=16, seqs=1, chunks=1, new=2048, kv=16384,
             **QWEN3),
        # one server step: decoding conversations and prompts' chunks in one batch
        dict(name="attend_mixed", op="attend", dtype="e4m3", page=32, seqs=27, chunks=3, new=511, kv=2047, **GPT2),
        # one request's logits
        dict(name="logits_1", op="logits", rows=1, vocab=50257, hist=300, biases=8, mask=True),
        # a large batch with long histories
        dict(name="logits_256", op="logits", rows=256, vocab=151936, hist=4000, biases=300, mask=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "read", "attend", "attend", "logits"))
    if op == "logits":
        return dict(op=op, rows=_log(rng, 1, 256), vocab=rng.choice((50257, 151936, _log(rng, 100, 151936))),
                    hist=_log(rng, 1, 4000), biases=rng.choice((0, _log(rng, 1, 300))), mask=rng.random() < 0.6)
    c = dict(op=op, dtype=rng.choice(("bf16", "e4m3")), page=rng.choice((16, 32, 64, 24)))
    c.update(rng.choice(LAYOUTS))
    row = c["hkv"] * c["hd"]
    if op == "append":
        c["norm"], c["rope"] = rng.random() < 0.5, rng.random() < 0.8
        c["seqs"] = _log(rng, 1, 64)
        c["chunks"] = rng.choice((0, rng.randint(0, min(c["seqs"], 5))))
        c["new"] = _log(rng, 2, 2048) if c["chunks"] else 1
        c["kv"] = _log(rng, c["new"], max(c["new"], 4096))
        limit = 32 << 20
    elif op == "read":
        c["seqs"] = _log(rng, 1, 64)
        c["chunks"] = c["seqs"]
        c["kv"] = _log(rng, 2, 8192)
        c["new"] = c["kv"]
        limit = 48 << 20
    else:
        c["seqs"] = _log(rng, 1, 64)
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


# ---------------------------------------------------------------- inputs

def _lens(case):
    """Cached length and new tokens of each sequence: the first one has the most, the others any."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    kv, new = [], []
    for i in range(case["seqs"]):
        n = (case["new"] if i == 0 else r.randint(1, case["new"])) if i < case["chunks"] else 1
        if case["op"] == "read":
            length = n  # all that is cached
        else:
            length = case["kv"] if i == 0 else max(n, _log(r, max(1, case["kv"] // 16), case["kv"]))
        kv.append(length)
        new.append(n)
    return kv, new


def _hist_lens(case):
    r = random.Random("%(rows)d %(vocab)d %(hist)d" % case)
    return [case["hist"] if i == 0 else r.randint(0, case["hist"]) for i in range(case["rows"])]


def _quantise(x):
    """e4m3 codes and the scale of each row (last axis)."""
    amax = x.abs().amax(-1)
    inv = torch.where(amax > 0, E4M3_MAX / amax, torch.zeros_like(amax))
    return (x * inv[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), amax / E4M3_MAX


def _rope_tables(hd, rows):
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "logits":
        rows, n, h = case["rows"], case["vocab"], case["hist"]
        s["logits"] = normal(rows, n) * 3
        s["out"] = torch.empty_like(s["logits"])
        # texts repeat themselves: few tokens make up most of a history
        s["history"] = (torch.rand((rows, h), generator=g, device="cuda") ** 4 * n).int().clamp_(0, n - 1)
        s["hist_lens"] = torch.tensor(_hist_lens(case), dtype=torch.int32, device="cuda")
        s["prompt_lens"] = s["hist_lens"] // 3
        s["repetition"] = 1 + 0.3 * torch.rand(rows, generator=g, device="cuda")
        s["presence"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
        s["frequency"] = 0.4 * torch.rand(rows, generator=g, device="cuda")
        s["bias_rows"] = s["bias_ids"] = s["bias"] = s["allowed"] = None
        if case["biases"]:
            s["bias_rows"] = torch.arange(rows + 1, dtype=torch.int32, device="cuda") * case["biases"]
            ids = torch.rand((rows, n), generator=g, device="cuda").topk(min(case["biases"], n), 1).indices
            if ids.shape[1] < case["biases"]:
                ids = ids.repeat(1, -(-case["biases"] // n))[:, :case["biases"]]
            s["bias_ids"] = ids.reshape(-1).int()
            s["bias"] = normal(rows * case["biases"])
        if case["mask"]:
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, (n + 31) // 32), generator=g, device="cuda",
                                         dtype=torch.int64).int()
        if own:
            from gorch_amd import hip

            hip.init(0)
            s["hip"] = hip
        return s
    kv, new = _lens(case)
    page, hq, hkv, hd = case["page"], case["hq"], case["hkv"], case["hd"]
    per_seq = -(-max(kv) // page)
    need = [-(-n // page) for n in kv]
    pages = sum(need)
    T = sum(new)
    order = torch.randperm(pages, generator=g, device="cuda").int()
    # entries past a sequence's last page are never looked at
    col = torch.arange(per_seq, device="cuda")
    first = torch.tensor([0] + need, device="cuda").cumsum(0)
    used = torch.tensor(need, device="cuda")
    s["page_table"] = order[(first[:-1, None] + torch.minimum(col[None], used[:, None] - 1)).long()].contiguous()
    s["cu_seqlens"] = torch.tensor([0] + new, device="cuda").cumsum(0).int()
    s["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["tokens"], s["max_new"], s["max_kv"] = T, max(new), max(kv)
    shape = (pages, hkv, page, hd)
    kind = torch.bfloat16 if case["dtype"] == "bf16" else torch.float8_e4m3fn
    s["k_scale"] = s["v_scale"] = None
    if case["op"] == "append":
        s["k"] = torch.zeros(shape, dtype=torch.uint8 if kind != torch.bfloat16 else kind, device="cuda").view(kind)
        s["v"] = torch.zeros_like(s["k"].view(torch.uint8)).view(kind)
        if kind != torch.bfloat16:
            s["k_scale"] = torch.zeros(shape[:3], device="cuda")
            s["v_scale"] = torch.zeros(shape[:3], device="cuda")
        # what the fused projection leaves: q, k and v side by side in a row
        s["qkv"] = normal(T, (hq + 2 * hkv) * hd)
        s["q_out"] = torch.empty((T, hq * hd), device="cuda")
        s["q_gain"] = 1 + 0.2 * normal(hd) if case["norm"] else None
        s["k_gain"] = 1 + 0.2 * normal(hd) if case["norm"] else None
        s["cos"], s["sin"] = _rope_tables(hd, max(kv)) if case["rope"] else (None, None)
    else:
        for name in ("k", "v"):
            x = normal(*shape) * torch.exp(0.3 * normal(*shape[:3]))[..., None]
            if kind == torch.bfloat16:
                s[name] = x.bfloat16()
            else:
                s[name], s[name + "_scale"] = _quantise(x)
            del x
        if case["op"] == "read":
            s["k_out"] = torch.empty((T, hkv * hd), device="cuda")
            s["v_out"] = torch.empty((T, hkv * hd), device="cuda")
        else:
            s["q"] = normal(T, hq * hd) * 1.5
            s["out"] = torch.empty((T, hq * hd), device="cuda")
    if own:
        from gorch_amd import hip

        hip.init(0)
        s["hip"] = hip
        s["cache"] = hip.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = hip.PagedBatch(s["cu_seqlens"], s["kv_lens"], s["page_table"], T, max_new=max(new), max_kv=max(kv))
        if case["op"] == "append":
            s["heads"] = hip.GQA(dict(dim=hq * hd, num_q=hq, num_kv=hkv, head_dim=hd, norm_eps=EPS, q_norm=s["q_gain"],
                                      k_norm=s["k_gain"], rope=case["rope"], rope_cos=s["cos"], rope_sin=s["sin"],
                                      rope_max_seq=max(kv)))
        elif case["op"] == "attend":
            s["ws"] = s["cache"].workspace(s["batch"], hq)
    return s


# ---------------------------------------------------------------- the calls

def run(s):
    return {"append": _append, "read": _read, "attend": _attend, "logits": _logits}[s["op"]](s)


def _places(s):
    """Sequence, position, page and slot of every token row."""
    cu = s["cu_seqlens"].long()
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = s["kv_lens"].long()[seq] - cu[seq + 1] + t
    return seq, pos, s["page_table"][seq, pos // s["page"]].long(), pos % s["page"]


def _head_norm(x, gain):
    if gain is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain


def _rotate(x, cos, sin):
    if cos is None:
        return x
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _append(s):
    hq, hkv, hd, T = s["hq"], s["hkv"], s["hd"], s["tokens"]
    if own:
        q, k, v = s["qkv"].split([hq * hd, hkv * hd, hkv * hd], 1)
        s["cache"].append(s["batch"], s["heads"], q, k, v, s["q_out"])
    else:
        q, k, v = (x.view(T, -1, hd) for x in s["qkv"].split([hq * hd, hkv * hd, hkv * hd], 1))
        _, pos, page, slot = _places(s)
        cos, sin = (None, None) if s["cos"] is None else (s["cos"][pos][:, None], s["sin"][pos][:, None])
        s["q_out"].view(T, hq, hd).copy_(_rotate(_head_norm(q, s["q_gain"]), cos, sin))
        k = _rotate(_head_norm(k, s["k_gain"]), cos, sin)
        if s["dtype"] == "bf16":
            s["k"][page, :, slot] = k.bfloat16()
            s["v"][page, :, slot] = v.bfloat16()
        else:
            kc, ks = _quantise(k)
            vc, vs = _quantise(v)
            s["k"].view(torch.uint8)[page, :, slot] = kc.view(torch.uint8)
            s["v"].view(torch.uint8)[page, :, slot] = vc.view(torch.uint8)
            s["k_scale"][page, :, slot] = ks
            s["v_scale"][page, :, slot] = vs
    return {"q": s["q_out"], "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _read(s):
    if own:
        s["cache"].read(s["batch"], s["k_out"], s["v_out"])
    else:
        _, _, page, slot = _places(s)
        shape = (s["tokens"], s["hkv"], s["hd"])
        if s["dtype"] == "bf16":
            s["k_out"].view(shape).copy_(s["k"][page, :, slot])
            s["v_out"].view(shape).copy_(s["v"][page, :, slot])
        else:
            k = s["k"].view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float()
            v = s["v"].view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float()
            torch.mul(k, s["k_scale"][page, :, slot][..., None], out=s["k_out"].view(shape))
            torch.mul(v, s["v_scale"][page, :, slot][..., None], out=s["v_out"].view(shape))
    return {"k": s["k_out"], "v": s["v_out"]}


def _gathered(s, name):
    """[seqs, KV heads, padded length, head dim] f32 of one pool."""
    hkv, hd = s["hkv"], s["hd"]
    table = s["page_table"].long()
    pool = s[name]
    x = pool[table].float() if s["dtype"] == "bf16" else pool.view(torch.uint8)[table].view(pool.dtype).float()
    if s["dtype"] != "bf16":
        x *= s[name + "_scale"][table][..., None]
    return x.transpose(1, 2).reshape(table.shape[0], hkv, -1, hd)


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
    k, v = _gathered(s, "k"), _gathered(s, "v")
    length = k.shape[2]
    p = torch.matmul(q, k.transpose(2, 3).contiguous())
    del k
    seen = torch.arange(length, device="cuda") <= where[..., None]
    p = p.view(seqs, hkv, group, N, length).masked_fill_(~seen[:, None, None], -math.inf)
    # keys past a sequence's end: whatever their pages hold is not used
    v = v * (torch.arange(length, device="cuda") < s["kv_lens"][:, None])[:, None, :, None]
    top = p.amax(-1, keepdim=True).clamp_min_(torch.finfo(torch.float32).min)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, hkv, group * N, length), v).view(seqs, hkv, group, N, hd)
    o = o / total.clamp_min(1e-30)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4)[seq, at].reshape(T, hq * hd))
    return s["out"]


def _logits(s):
    if own:
        s["hip"].process_logits(s["logits"], s["out"], history=s["history"], history_lens=s["hist_lens"],
                                prompt_lens=s["prompt_lens"], repetition=s["repetition"], presence=s["presence"],
                                frequency=s["frequency"], bias_rows=s["bias_rows"], bias_ids=s["bias_ids"],
                                bias=s["bias"], allowed=s["allowed"])
        return s["out"]
    rows, n = s["logits"].shape
    ids = s["history"].long()
    col = torch.arange(ids.shape[1], device="cuda")
    live = col < s["hist_lens"][:, None]
    chosen = live & (col >= s["prompt_lens"][:, None])
    seen = torch.zeros((rows, n), device="cuda").scatter_add_(1, ids, live.float())
    count = torch.zeros((rows, n), device="cuda").scatter_add_(1, ids, chosen.float())
    x, r = s["logits"], s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        # of an id's entries in a row the last one counts
        per = s["bias_ids"].shape[0] // rows
        entry = torch.arange(s["bias_ids"].shape[0], device="cuda").view(rows, per)
        last = torch.full((rows, n), -1, device="cuda").scatter_reduce_(1, s["bias_ids"].long().view(rows, per), entry,
                                                                       "amax")
        x = x + torch.where(last >= 0, s["bias"][last.clamp_min(0)], torch.zeros((), device="cuda"))
    if s["allowed"] is not None:
        bits = (s["allowed"][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(rows, -1)[:, :n] == 0, -math.inf)
    s["out"].copy_(x)
    return s["out"]


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "logits":
        rows, n = case["rows"], case["vocab"]
        b = rows * n * 8 + 4 * sum(_hist_lens(case)) + rows * (20 + 8 * case["biases"])
        return {"bytes": b + (rows * ((n + 31) // 32) * 4 if case["mask"] else 0), "flops": 4 * rows * n}
    kv, new = _lens(case)
    T, hq, hkv, hd = sum(new), case["hq"], case["hkv"], case["hd"]
    row = 2 * hkv * (hd * 2 if case["dtype"] == "bf16" else hd + 4)  # one token's K and V in the cache
    tables = 4 * sum(-(-n // case["page"]) for n in kv) + 8 * len(kv)
    if case["op"] == "append":
        moved = T * (4 * hd * (2 * hq + 2 * hkv) + row) + (T * 4 * hd if case["rope"] else 0)
        return {"bytes": moved + 8 * len(kv), "flops": 8 * T * (hq + hkv) * hd}
    if case["op"] == "read":
        return {"bytes": T * (row + 8 * hkv * hd) + tables, "flops": 2 * T * hkv * hd}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for length, n in zip(kv, new))
    return {"bytes": sum(kv) * row + 8 * T * hq * hd + tables, "flops": 4 * hd * hq * pairs}


# ---------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(case, s)
    kv, new = _lens(case)
    hq, hkv, hd, page = case["hq"], case["hkv"], case["hd"], case["page"]
    begin = 0
    f8 = case["dtype"] == "e4m3"

    def rows_of(i, lo, hi):
        """Pages and slots of positions lo .. hi - 1 of sequence i."""
        p = torch.arange(lo, hi, device="cuda")
        return s["page_table"][i].long()[torch.div(p, page, rounding_mode="floor")], p.remainder(page)

    def cached(i, name):
        """[length, KV heads, head dim] of sequence i."""
        at = rows_of(i, 0, kv[i])
        x = s[name].view(torch.uint8)[at[0], :, at[1]].view(s[name].dtype).double() if f8 else \
            s[name][at[0], :, at[1]].double()
        return x * s[name + "_scale"][at[0], :, at[1]].double().unsqueeze(-1) if f8 else x

    if case["op"] == "append":
        x = s["qkv"].double().view(-1, hq + 2 * hkv, hd)
        scale = [torch.zeros(s["k"].shape[:3], dtype=torch.float64, device="cuda") for _ in "kv"] if f8 else [None, None]
        pool = [torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in "kv"]
        q_out = torch.empty((x.shape[0], hq * hd), dtype=torch.float64, device="cuda")
        for i, n in enumerate(new):
            q, k, v = x[begin:begin + n].split([hq, hkv, hkv], 1)
            if case["norm"]:
                q = q / (q.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * s["q_gain"].double()
                k = k / (k.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * s["k_gain"].double()
            if case["rope"]:
                turn = torch.complex(s["cos"].double(), s["sin"].double())[kv[i] - n:kv[i], None]
                q, k = (torch.complex(*y.chunk(2, -1)) * turn for y in (q, k))
                q, k = (torch.cat([y.real, y.imag], -1) for y in (q, k))
            q_out[begin:begin + n] = q.reshape(n, -1)
            at = rows_of(i, kv[i] - n, kv[i])
            for j, y in enumerate((k, v)):
                if f8:
                    step = y.abs().amax(-1) / E4M3_MAX
                    scale[j][at[0], :, at[1]] = step
                    y = y / step.unsqueeze(-1)
                pool[j][at[0], :, at[1]] = y
            begin += n
        return {"q": q_out, "k": pool[0], "v": pool[1], "k_scale": scale[0], "v_scale": scale[1]}
    if case["op"] == "read":
        return {"k": torch.cat([cached(i, "k").reshape(n, -1) for i, n in enumerate(kv)]),
                "v": torch.cat([cached(i, "v").reshape(n, -1) for i, n in enumerate(kv)])}
    out = torch.empty((sum(new), hq, hd), dtype=torch.float64, device="cuda")
    for i, n in enumerate(new):
        k, v = cached(i, "k"), cached(i, "v")
        q = s["q"][begin:begin + n].double().view(n, hq, hd)
        seen = torch.ones((n, kv[i]), dtype=torch.bool, device="cuda").tril_(kv[i] - n)
        for h in range(hq):
            a = torch.mm(q[:, h], k[:, h * hkv // hq].t().contiguous()) / math.sqrt(hd)
            a = torch.softmax(a.masked_fill_(~seen, -math.inf), -1)
            out[begin:begin + n, h] = torch.mm(a, v[:, h * hkv // hq].contiguous())
        begin += n
    return out.view(sum(new), hq * hd)


def _exact_logits(case, s):
    rows, n, per = case["rows"], case["vocab"], case["biases"]
    out = s["logits"].double()
    lens = _hist_lens(case)
    bit = torch.arange(n, device="cuda")
    for i in range(rows):
        x, r = out[i], s["repetition"][i].double()
        ids = s["history"][i, :lens[i]].long()
        said = torch.bincount(ids[lens[i] // 3:], minlength=n)
        known = torch.bincount(ids, minlength=n) > 0
        x[known] = torch.where(x[known] > 0, x[known] / r, x[known] * r)
        x -= said * s["frequency"][i].double() + (said > 0) * s["presence"][i].double()
        if per:
            # entries past the vocabulary's size repeat its ids: an id's last entry is in the last whole or part turn
            ids, values = s["bias_ids"].view(rows, per)[i].long(), s["bias"].view(rows, per)[i].double()
            extra = torch.zeros(n, dtype=torch.float64, device="cuda")
            for first in range(0, per, n):
                extra[ids[first:first + n]] = values[first:first + n]
            x += extra
        if case["mask"]:
            x[(s["allowed"][i].long()[bit // 32] >> (bit % 32)) % 2 == 0] = -math.inf
    return out
