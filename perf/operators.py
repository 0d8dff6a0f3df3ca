"""Cases of the paged key-value cache operators: append, attend and gather.

``append`` normalises and rotates the q and k heads of q|k|v rows and stores k
and v into cache pages (quantised where the cache is), ``attend`` is the
attention of one new token per conversation over its pages, ``gather`` reads
stored rows back.  A case names one of them with its head layout, cache type,
activation type, page size and lengths.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 64  # values that share a scale in a quantised cache
EPS = 1e-6
THETA = 1e6
DEV = "cuda"

# Head layouts: (q heads, kv heads, head dimension).  The first four are the
# Qwen3 configurations and test models of this repository, the others a
# tensor-parallel shard, one query head per KV head, and generic layouts.
HEADS = {"16/8": (16, 8, 128), "32/8": (32, 8, 128), "4/2": (4, 2, 128), "8/2": (8, 2, 128), "16/4": (16, 4, 128),
         "8/8": (8, 8, 128), "24/4 d64": (24, 4, 64), "16/2": (16, 2, 128)}


def listed():
    def case(name, op, heads, cache, act, page, rows, longest, at=0, window=0):
        return dict(name=name, op=op, heads=heads, cache=cache, act=act, page=page, rows=rows, longest=longest, at=at,
                    window=window)

    return [
        # one conversation right after the benchmark's short 21-token prompt: launch latency
        case("attend_1x21_f16", "attend", "16/8", "f16", "f32", 16, 1, 21),
        # one conversation at the context where the 1.7B benchmark starts to decode
        case("attend_1x2851_f16", "attend", "16/8", "f16", "f32", 16, 1, 2851),
        # a small server of the 4B model: 16 conversations up to its long context
        case("attend_16x3840_q8", "attend", "32/8", "q8", "f16", 32, 16, 3840),
        # many conversations of the 8B model in a 4-bit cache
        case("attend_64x4096_q4", "attend", "32/8", "q4", "bf16", 64, 64, 4096),
        # the largest batch: long fp16 conversations
        case("attend_32x8192_f16", "attend", "32/8", "f16", "f16", 16, 32, 8192),
        # one very long conversation: all the work is split over its length
        case("attend_1x65521_q8", "attend", "32/8", "q8", "f32", 16, 1, 65521),
        # a decode step of one conversation: write the token
        case("append_1_f16", "append", "16/8", "f16", "f32", 16, 1, 1, at=2851),
        # a decode step of 64 conversations into an 8-bit cache, and what it holds
        case("append_64_q8", "append", "32/8", "q8", "bf16", 64, 64, 1, at=2000),
        # the benchmark's 2811-token prompt
        case("append_2811_f16", "append", "16/8", "f16", "f32", 16, 1, 2811),
        # prompts of 16 conversations into a 4-bit cache, and what it holds
        case("append_16x1024_q4", "append", "32/8", "q4", "f16", 32, 16, 1024),
        # the rows of a 40-token appended turn
        case("gather_1x40_q8", "gather", "16/8", "q8", "f32", 16, 1, 40, at=2875),
        # 32 conversations read back whole, to move them to another cache
        case("gather_32x2048_q4", "gather", "32/8", "q4", "f16", 64, 32, 2048),
    ]


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "gather"])
    most = {"attend": 160_000, "append": 12_000, "gather": 40_000}[op]  # positions in all
    rows = int(round(2 ** rng.uniform(0, 7)))
    longest = max(1, int(round(2 ** rng.uniform(0, math.log2(most / rows)))))
    return dict(op=op, heads=rng.choice(sorted(HEADS)), cache=rng.choice(["f16", "q8", "q4"]),
                act=rng.choice(["f32", "f16", "bf16"]), page=rng.choice([16, 32, 64, 128]), rows=rows, longest=longest,
                at=rng.choice([0, rng.randint(1, 4000)]) if op != "attend" and rows <= 64 else 0,
                window=rng.choice([0, 0, 0, rng.randint(1, longest)]) if op == "attend" else 0)


def lengths(case):
    """Positions of each conversation that the call touches: the longest, and others spread from a quarter of it up.
    They begin at position case["at"] (append and gather after earlier turns)."""
    n, longest = case["rows"], case["longest"]
    return [max(1, longest - (longest * 3 * ((i * 37) % n)) // (4 * n)) for i in range(n)]


def prepare(case, seed):
    n_heads, n_kv, dim = HEADS[case["heads"]]
    page, act, lens = case["page"], TYPES[case["act"]], lengths(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    # pages of the conversations, scattered over the pool
    counts = [-(-(case["at"] + n) // page) for n in lens]
    width, total = max(counts), sum(counts)
    pool = total + 3
    order = torch.randperm(pool, generator=g, device=DEV)[:total].to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    used = torch.arange(width, device=DEV)[None, :] < torch.tensor(counts, device=DEV)[:, None]
    table[used] = order
    s = {"case": case, "n_heads": n_heads, "n_kv": n_kv, "dim": dim, "page": page, "pool": pool, "table": table,
         "act": act, "scale": dim ** -0.5, "stream": torch.cuda.current_stream().cuda_stream}

    # the pool: keys after their norm and rotation have a root mean square near one
    shape = (pool, n_kv, page, dim)
    for name in ("k", "v"):
        if case["op"] == "append":  # freshly allocated
            code = torch.zeros(shape, dtype=torch.float16, device=DEV)
        else:
            code = randn(*shape, dtype=torch.float16)
        if case["cache"] != "f16":
            most = 127 if case["cache"] == "q8" else 7
            code = (code * (most / 2.5)).round_().clamp_(-most, most).to(torch.int8)
            scale = torch.rand(pool, n_kv, page, dim // GROUP, generator=g, device=DEV) + 0.5
            s[name + "_scale"] = (scale * (2.5 / most)).half()
            if case["cache"] == "q4":
                code = ((code[..., 0::2] + 8) | ((code[..., 1::2] + 8) << 4)).view(torch.uint8)
        s[name] = code

    if case["op"] == "attend":
        s["q"] = (2.0 * randn(len(lens), n_heads * dim)).to(act)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["starts"] = (s["lens"] - case["window"]).clamp_(min=0) if case["window"] else None
        s["out"] = torch.empty_like(s["q"])
        s["workspace"] = torch.zeros(16 << 20, dtype=torch.uint8, device=DEV)
        return s

    # the rows (conversation, position); a decode step appends one row to each
    s["seq"] = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(lens)]).to(DEV)
    s["pos"] = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(DEV) + case["at"]
    n_tok = sum(lens)
    if case["op"] == "append":
        s["qkv"] = randn(n_tok, (n_heads + 2 * n_kv) * dim).to(act)
        s["q_norm"] = 1.0 + 0.05 * randn(dim)
        s["k_norm"] = 1.0 + 0.05 * randn(dim)
        angle = torch.arange(case["at"] + case["longest"], dtype=torch.float64, device=DEV)[:, None] * THETA ** (
            -torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
        s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
        s["q_out"] = torch.empty(n_tok, n_heads * dim, dtype=act, device=DEV)
    # a quantised cache is handed on in fp16, as the prompt's attention takes it
    rows_type = torch.float16 if case["op"] == "append" else act
    s["k_out"] = torch.empty(n_tok, n_kv * dim, dtype=rows_type, device=DEV)
    s["v_out"] = torch.empty_like(s["k_out"])
    return s


# ---------------------------------------------------------------- plain form


def stored(code, scale, cache):
    """The values that cache entries stand for, in 32 bits."""
    if cache == "f16":
        return code.float()
    if cache == "q4":
        code = torch.stack([code & 15, code >> 4], -1).flatten(-2).float() - 8.0
    x = code.float().unflatten(-1, (-1, GROUP))
    return (x * scale.float()[..., None]).flatten(-2)


def quantised(x, cache):
    """(codes, scales) of values in 32 bits."""
    most = 127.0 if cache == "q8" else 7.0
    x = x.unflatten(-1, (-1, GROUP))
    scale = (x.abs().amax(-1) / most).clamp(max=65504.0).half()
    d = scale.float()[..., None]
    code = torch.where(d > 0, x / d, 0.0).round().clamp(-most, most).flatten(-2)
    if cache == "q8":
        return code.to(torch.int8), scale
    code = (code + 8.0).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def slots(s):
    """Pool page and offset of each row."""
    pos = s["pos"].long()
    return s["table"][s["seq"].long(), pos // s["page"]].long(), pos % s["page"]


def plain_attend(s):
    cache, n_kv, dim = s["case"]["cache"], s["n_kv"], s["dim"]
    pages = s["table"].clamp(min=0).long()
    rows = pages.shape[0]

    def cached(name):
        scale = s[name + "_scale"][pages] if cache != "f16" else None
        x = stored(s[name][pages], scale, cache)
        return x.transpose(1, 2).reshape(rows, n_kv, -1, dim)

    q = s["q"].float().view(rows, n_kv, -1, dim)
    scores = (q @ cached("k").transpose(-1, -2)) * s["scale"]
    at = torch.arange(scores.shape[-1], device=DEV)
    seen = at < s["lens"][:, None]
    if s["starts"] is not None:
        seen = seen & (at >= s["starts"][:, None])
    seen = seen[:, None, None, :]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ cached("v")) / torch.where(total > 0, total, 1.0)
    return out.reshape(rows, -1).to(s["act"])


def plain_append(s):
    cache, n_heads, n_kv, dim = s["case"]["cache"], s["n_heads"], s["n_kv"], s["dim"]
    q, k, v = s["qkv"].float().unflatten(-1, (-1, dim)).split([n_heads, n_kv, n_kv], 1)
    cos, sin = s["rope"][s["pos"].long()][:, None, :].chunk(2, -1)

    def turned(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    page, at = slots(s)
    for name, x in (("k", turned(k, s["k_norm"])), ("v", v)):
        if cache == "f16":
            s[name][page, :, at] = x.half()
        else:
            s[name][page, :, at], s[name + "_scale"][page, :, at] = quantised(x, cache)
    return turned(q, s["q_norm"]).flatten(1).to(s["act"])


def plain_gather(s, dtype):
    cache = s["case"]["cache"]
    page, at = slots(s)
    return [stored(s[n][page, :, at], s[n + "_scale"][page, :, at] if cache != "f16" else None, cache).flatten(1).to(dtype)
            for n in ("k", "v")]


# ---------------------------------------------------------------- the framework's operators


def handles(s):
    """What a program makes once for a cache, a page table and a model's heads."""
    import rpgbarenginecuda_b200 as rpg

    case = s["case"]
    kind = {"f16": rpg.KV_F16, "q8": rpg.KV_Q8, "q4": rpg.KV_Q4}[case["cache"]]
    act = {"f32": rpg.F32, "f16": rpg.F16, "bf16": rpg.BF16}[case["act"]]
    scales = [s[n].data_ptr() if n in s else 0 for n in ("k_scale", "v_scale")]
    kv = rpg.PagedKv(kind, s["dim"], s["n_kv"], s["page"], s["pool"], s["k"].data_ptr(), s["v"].data_ptr(), *scales)
    table = rpg.PageTable(s["table"].data_ptr(), *s["table"].shape)
    rotary = None
    if "rope" in s:
        rotary = rpg.Rotary(s["rope"].data_ptr(), s["rope"].shape[0], s["q_norm"].data_ptr(), s["k_norm"].data_ptr(), EPS)
    return kv, table, rotary, act, rpg.F16


def run(state):
    s, case = state, state["case"]
    if not own:
        if case["op"] == "attend":
            return plain_attend(s)
        if case["op"] == "gather":
            return plain_gather(s, s["act"])
        q = plain_append(s)
        return [q, s["k"], s["v"]] if case["cache"] == "f16" else [q, *plain_gather(s, torch.float16)]
    if "handles" not in s:
        s["handles"] = handles(s)
    kv, table, rotary, act, f16 = s["handles"]
    if case["op"] == "attend":
        kv.attend(table, act, s["q"].data_ptr(), s["n_heads"], s["lens"].data_ptr(), s["scale"], s["out"].data_ptr(),
                  s["workspace"].data_ptr(), s["workspace"].numel(),
                  starts_ptr=s["starts"].data_ptr() if s["starts"] is not None else 0, stream=s["stream"])
        return s["out"]
    n_tok = s["pos"].numel()
    if case["op"] == "append":
        kv.append(table, rotary, act, s["qkv"].data_ptr(), s["n_heads"], s["pos"].data_ptr(), n_tok,
                  s["q_out"].data_ptr(), seq_ptr=s["seq"].data_ptr(), stream=s["stream"])
        if case["cache"] == "f16":
            return [s["q_out"], s["k"], s["v"]]
        act = f16
    kv.gather(table, act, s["pos"].data_ptr(), n_tok, s["k_out"].data_ptr(), s["v_out"].data_ptr(),
              seq_ptr=s["seq"].data_ptr(), stream=s["stream"])
    rows = [s["k_out"], s["v_out"]]
    return [s["q_out"], *rows] if case["op"] == "append" else rows


# ---------------------------------------------------------------- work and exact values


def work(case):
    n_heads, n_kv, dim = HEADS[case["heads"]]
    lens = lengths(case)
    size = 4 if case["act"] == "f32" else 2
    stored_bytes = {"f16": 2 * dim, "q8": dim + 2 * dim // GROUP, "q4": dim // 2 + 2 * dim // GROUP}[case["cache"]]
    if case["op"] == "attend":
        seen = sum(min(n, case["window"] or n) for n in lens)
        return {"bytes": seen * n_kv * 2 * stored_bytes + 2 * len(lens) * n_heads * dim * size,
                "flops": 4 * seen * n_heads * dim}
    n = sum(lens)
    if case["op"] == "gather":
        return {"bytes": n * n_kv * 2 * (stored_bytes + dim * size), "flops": 2 * n * n_kv * dim}
    moved = n * ((2 * n_heads + 2 * n_kv) * dim * size + 2 * n_kv * stored_bytes) + case["longest"] * dim * 4  # rotation rows once
    if case["cache"] != "f16":
        moved += n * n_kv * 2 * (stored_bytes + dim * 2)
    return {"bytes": moved, "flops": n * (n_heads + n_kv) * dim * 8 + n * n_kv * dim * 6}


def exact(case, seed):
    s = prepare(case, seed)
    n_heads, n_kv, dim, page, cache = s["n_heads"], s["n_kv"], s["dim"], s["page"], case["cache"]
    lens = lengths(case)
    table = s["table"].tolist()

    def value(name, ids):
        """Pages `ids` of one conversation: [kv head][position][dim]."""
        ids = torch.tensor(ids, device=DEV)
        c = s[name][ids]
        if cache == "q4":
            d = torch.empty(*c.shape[:-1], dim, dtype=torch.float64, device=DEV)
            d[..., 0::2] = (c % 16).double() - 8
            d[..., 1::2] = torch.div(c, 16, rounding_mode="floor").double() - 8
        else:
            d = c.double()
        if cache != "f16":
            d = d * s[name + "_scale"][ids].double().repeat_interleave(GROUP, -1)
        return d.permute(1, 0, 2, 3).reshape(n_kv, -1, dim)

    if case["op"] == "attend":
        outs = []
        for i, n in enumerate(lens):
            first = max(0, n - case["window"]) if case["window"] else 0
            ids = table[i][:-(-n // page)]
            k, v = value("k", ids)[:, first:n], value("v", ids)[:, first:n]
            q = s["q"][i].double().view(n_kv, n_heads // n_kv, dim)
            w = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(dim), -1)
            outs.append(torch.einsum("hgn,hnd->hgd", w, v).reshape(-1))
        return torch.stack(outs)

    if case["op"] == "gather":
        def rows(name):
            return torch.cat([value(name, table[i][:-(-(n + case["at"]) // page)])[:, case["at"]:case["at"] + n]
                              .transpose(0, 1).reshape(n, -1) for i, n in enumerate(lens)])
        return [rows("k"), rows("v")]

    x = s["qkv"].double().reshape(len(s["qkv"]), n_heads + 2 * n_kv, dim)
    turn = torch.complex(s["rope"][:, :dim // 2].double(), s["rope"][:, dim // 2:].double())[s["pos"].long()]

    def turned(y, w):
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / dim + EPS) * w.double()
        z = torch.complex(y[..., :dim // 2], y[..., dim // 2:]) * turn[:, None]
        return torch.cat([z.real, z.imag], -1)

    def held(y):
        most = {"q8": 127, "q4": 7}[cache]
        y = y.reshape(len(y), n_kv, dim // GROUP, GROUP)
        d = (torch.linalg.vector_norm(y, float("inf"), -1, keepdim=True) / most).to(torch.float16).double()
        return (torch.clamp(torch.round(y / d), -most, most) * d).reshape(len(y), -1)

    q = turned(x[:, :n_heads], s["q_norm"]).reshape(len(x), -1)
    k, v = turned(x[:, n_heads:n_heads + n_kv], s["k_norm"]), x[:, n_heads + n_kv:]
    if cache != "f16":
        return [q, held(k), held(v)]
    out = [q]
    for y in (k, v):
        pool = torch.zeros(s["pool"], n_kv, page, dim, dtype=torch.float64, device=DEV)
        for i, n in enumerate(lens):
            first = sum(lens[:i])
            for j in range(n):
                where, at = divmod(case["at"] + j, page)
                pool[table[i][where], :, at] = y[first + j]
        out.append(pool)
    return out
