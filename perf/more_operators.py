"""Cases of the operators that serve many conversations of one model together: rows, shared and sample.

``rows`` is the attention of several new tokens of each conversation (prompts,
appended turns) over paged caches, with windows, document and prefix masks,
capped scores and a bias by distance; ``shared`` the attention of one new token
per conversation where groups of conversations begin with the same positions;
``sample`` draws one token per row of logits from given random numbers, with
every row's own temperature, top-k, top-p and min-p.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 64  # values that share a scale in a quantised cache
DEV = "cuda"

# Head layouts: (q heads, kv heads, head dimension), as the configurations and tests of this repository have them.
HEADS = {"16/8": (16, 8, 128), "32/8": (32, 8, 128), "4/2": (4, 2, 128), "16/4": (16, 4, 128), "8/8": (8, 8, 128),
         "24/4 d64": (24, 4, 64), "16/2": (16, 2, 128), "40/8": (40, 8, 128)}


def listed():
    def rows(name, heads, cache, act, page, convs, longest, at=0, mask="causal", span=0, cap=0.0, slopes=False):
        return dict(name=name, op="rows", heads=heads, cache=cache, act=act, page=page, convs=convs, longest=longest,
                    at=at, mask=mask, span=span, cap=cap, slopes=slopes)

    def shared(name, heads, cache, act, page, convs, groups, prefix, longest):
        return dict(name=name, op="shared", heads=heads, cache=cache, act=act, page=page, convs=convs, groups=groups,
                    prefix=prefix, longest=longest)

    def sample(name, act, convs, vocab, filters):
        return dict(name=name, op="sample", act=act, convs=convs, vocab=vocab, filters=filters)

    return [
        # a 40-token turn appended to one conversation of the 1.7B benchmark: latency
        rows("rows_1x40_f16", "16/8", "f16", "f32", 16, 1, 40, at=2875),
        # the benchmark's 2811-token prompt
        rows("rows_1x2811_f16", "16/8", "f16", "f32", 16, 1, 2811),
        # prompts of 16 conversations that begin together, in an 8-bit cache
        rows("rows_16x1024_q8", "32/8", "q8", "f16", 32, 16, 1024),
        # prompts of packed documents with capped scores and a bias by distance, in a 4-bit cache
        rows("rows_6x1501_q4_docs", "24/4 d64", "q4", "bf16", 16, 6, 1501, at=100, mask="documents", span=700, cap=30.0,
             slopes=True),
        # the largest prompts: long context in f16
        rows("rows_4x4096_f16", "32/8", "f16", "bf16", 64, 4, 4096),
        # a few characters that talk under one set of instructions
        shared("shared_4x2000_f16", "16/8", "f16", "f32", 16, 4, 1, 2000, 90),
        # a server of the 4B model, one set of instructions for all
        shared("shared_64x4096_q8", "32/8", "q8", "bf16", 64, 64, 1, 4096, 300),
        # the largest: four long worlds, 128 conversations
        shared("shared_128x16384_f16", "32/8", "f16", "f16", 16, 128, 4, 16384, 500),
        # one conversation, the benchmark's sampling options: latency
        sample("sample_1_f32", "f32", 1, 151936, "top_k top_p"),
        # a batch with every conversation's own options, greedy ones among them
        sample("sample_64_f32", "f32", 64, 151936, "mixed"),
        # a small odd vocabulary, cut by a share of the largest probability
        sample("sample_40_f16_odd", "f16", 40, 32001, "min_p"),
        # the largest batch: the whole distribution
        sample("sample_256_bf16", "bf16", 256, 151936, "none"),
    ]


def draw(rng):
    def spread(least, most):
        return max(least, int(round(2 ** rng.uniform(math.log2(least), math.log2(most)))))

    op = rng.choice(["rows", "rows", "shared", "shared", "sample"])
    act = rng.choice(["f32", "f16", "bf16"])
    if op == "sample":
        convs = spread(1, 200)
        return dict(op=op, act=act, convs=convs, vocab=spread(300, 151936),
                    filters=rng.choice(["none", "top_k top_p", "top_k", "top_p", "min_p", "mixed", "mixed"]))
    case = dict(op=op, heads=rng.choice(sorted(HEADS)), cache=rng.choice(["f16", "q8", "q4"]), act=act,
                page=rng.choice([16, 32, 64, 128]))
    if op == "rows":
        convs = spread(1, 32)
        longest = spread(1, int(math.sqrt(12e6 / convs)))
        case |= dict(convs=convs, longest=longest, at=rng.choice([0, 0, spread(1, 2000 if longest < 400 else 200)]),
                     mask=rng.choice(["causal", "causal", "window", "documents", "prefix"]), span=spread(1, 2 * longest),
                     cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.choice([False, False, True]))
    else:
        convs = spread(1, 96)
        case |= dict(convs=convs, groups=min(convs, rng.choice([1, 1, 2, 5])), prefix=spread(16, 12000),
                     longest=spread(1, 1000))
    return case


def lengths(case):
    """New rows (rows) or own positions (shared) of each conversation: the longest, and others from a quarter of it up."""
    n, longest = case["convs"], case["longest"]
    return [max(1, longest - (longest * 3 * ((i * 37) % n)) // (4 * n)) for i in range(n)]


def members(case):
    """First conversation of each group, and the end: sizes as even as they go."""
    n, g = case["convs"], case["groups"]
    return [i * n // g for i in range(g + 1)]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    s = {"case": case, "act": TYPES[case["act"]], "stream": torch.cuda.current_stream().cuda_stream}
    n = case["convs"]
    if case["op"] == "sample":
        # a broad bulk and some tokens that stand out of it, by several units
        vocab = case["vocab"]
        x = 2.0 * randn(n, vocab)
        at = torch.randint(0, vocab, (n, 60), generator=g, device=DEV)
        x.scatter_add_(1, at, 5.0 + 3.0 * randn(n, 60))
        s["logits"] = x.to(s["act"])
        f, i = case["filters"], torch.arange(n, device=DEV)
        pick = lambda every, *v: torch.tensor(v, device=DEV)[(i + every) % len(v)]  # noqa: E731
        if f == "mixed":
            s["temperature"] = pick(0, 0.7, 1.0, 0.0, 0.85, 1.3)
            s["top_k"] = pick(0, 0, 20, 0, 64, 1000, 40, 0).to(torch.int32)
            s["top_p"] = pick(1, 1.0, 0.8, 0.95)
            s["min_p"] = pick(2, 0.0, 0.05, 0.0, 0.0)
        else:
            s["temperature"] = torch.full((n,), 0.7 if "top" in f else 1.0, device=DEV)
            s["top_k"] = torch.full((n,), 20 if "top_k" in f else 0, dtype=torch.int32, device=DEV)
            s["top_p"] = torch.full((n,), 0.8 if "top_p" in f else 1.0, device=DEV)
            s["min_p"] = torch.full((n,), 0.08 if "min_p" in f else 0.0, device=DEV)
        s["u"] = torch.rand(n, generator=g, device=DEV)
        s["tokens"] = torch.empty(n, dtype=torch.int32, device=DEV)
        s["probs"] = torch.empty(n, device=DEV)
        return s

    n_heads, n_kv, dim = HEADS[case["heads"]]
    page, lens = case["page"], lengths(case)
    before = case["at"] if case["op"] == "rows" else case["prefix"]
    # page lists, scattered over the pool; those of a group begin with the same whole pages
    total = [before + m for m in lens]
    width = -(-max(total) // page)
    lists = torch.full((n, width), -1, dtype=torch.int64)
    bounds = members(case) if case["op"] == "shared" else list(range(n + 1))
    common = before // page if case["op"] == "shared" else 0
    used = 0
    for a, b in zip(bounds, bounds[1:]):
        lists[a:b, :common] = torch.arange(used, used + common)
        used += common
        for c in range(a, b):
            k = -(-total[c] // page) - common
            lists[c, common:common + k] = torch.arange(used, used + k)
            used += k
    pool = used + 3
    order = torch.randperm(pool, generator=g, device=DEV)
    lists = lists.to(DEV)
    s["table"] = torch.where(lists >= 0, order[lists.clamp(min=0)], -1).to(torch.int32)
    s |= {"n_heads": n_heads, "n_kv": n_kv, "dim": dim, "page": page, "pool": pool, "scale": dim ** -0.5}

    # the pool: keys after their norm and rotation have a root mean square near one
    shape = (pool, n_kv, page, dim)
    for name in ("k", "v"):
        code = randn(*shape, dtype=torch.float16)
        if case["cache"] != "f16":
            most = 127 if case["cache"] == "q8" else 7
            code = (code * (most / 2.5)).round_().clamp_(-most, most).to(torch.int8)
            scale = torch.rand(pool, n_kv, page, dim // GROUP, generator=g, device=DEV) + 0.5
            s[name + "_scale"] = (scale * (2.5 / most)).half()
            if case["cache"] == "q4":
                code = ((code[..., 0::2] + 8) | ((code[..., 1::2] + 8) << 4)).view(torch.uint8)
        s[name] = code

    if case["op"] == "shared":
        # where the common positions end inside a page, every conversation holds its own copy of that page's beginning
        rest = before % page
        if rest:
            for a, b in zip(bounds, bounds[1:]):
                to = s["table"][a:b, common].long()
                for name in ("k", "v", "k_scale", "v_scale"):
                    if name in s:
                        s[name][to, :, :rest] = s[name][to[:1], :, :rest]
        s["lens"], s["groups"], s["prefix"] = ints(total), ints(bounds), ints([before] * n)
        # conversations by group, padded with the group's first
        most = max(b - a for a, b in zip(bounds, bounds[1:]))
        s["member"] = torch.tensor([[min(c, b - 1) for c in range(a, a + most)] for a, b in zip(bounds, bounds[1:])],
                                   device=DEV)
        s["slot"] = torch.tensor([i * most + c for i, (a, b) in enumerate(zip(bounds, bounds[1:])) for c in range(b - a)],
                                 device=DEV)
        s["q"] = (2.0 * randn(n, n_heads * dim)).to(s["act"])
        space = 160 << 20
    else:
        seq = torch.cat([torch.full((m,), i) for i, m in enumerate(lens)]).to(DEV)
        index = torch.cat([torch.arange(m) for m in lens]).to(DEV)
        pos, mask, span = index + before, case["mask"], case["span"]
        start, end = torch.zeros_like(pos), pos + 1
        if mask == "window":
            start = (end - span).clamp(min=0)
        elif mask == "documents":
            start = pos // span * span
        elif mask == "prefix":  # the first positions see each other
            end = torch.maximum(end, torch.tensor(total, device=DEV)[seq].clamp(max=span))
        s |= {"seq": seq, "index": index, "pos": pos.to(torch.int32), "ends": end.to(torch.int32),
              "starts": start.to(torch.int32) if mask in ("window", "documents") else None}
        s["rows"] = ints([sum(lens[:i]) for i in range(n + 1)])
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, n_heads + 1, device=DEV) / n_heads) if case["slopes"] else None
        s["q"] = (2.0 * randn(len(pos), n_heads * dim)).to(s["act"])
        space = 160 << 20
    s["out"] = torch.empty_like(s["q"])
    s["workspace"] = torch.zeros(space, dtype=torch.uint8, device=DEV)
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


def cached(s, name, pages):
    """Values of page lists: [list][kv head][position][dim]."""
    pages = pages.clamp(min=0).long()
    scale = s[name + "_scale"][pages] if s["case"]["cache"] != "f16" else None
    return stored(s[name][pages], scale, s["case"]["cache"]).transpose(1, 2).flatten(2, 3)


def softmax_parts(scores):
    """Weights over all parts' last axes together; a row that sees nothing has none."""
    top = scores[0].amax(-1, keepdim=True)
    for x in scores[1:]:
        top = torch.maximum(top, x.amax(-1, keepdim=True))
    top = torch.where(top == float("-inf"), 0.0, top)
    p = [torch.exp(x - top) for x in scores]
    total = sum(x.sum(-1, keepdim=True) for x in p)
    return p, torch.where(total > 0, total, 1.0)


def plain_rows(s):
    case, n_heads, n_kv, dim = s["case"], s["n_heads"], s["n_kv"], s["dim"]
    n, most, group = case["convs"], case["longest"], n_heads // n_kv
    seq, index = s["seq"], s["index"]

    def padded(x, fill=0):
        y = torch.full((n, most) + x.shape[1:], fill, dtype=x.dtype, device=DEV)
        y[seq, index] = x
        return y

    q = padded(s["q"].float()).view(n, most, n_kv, group, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = cached(s, "k", s["table"]), cached(s, "v", s["table"])
    scores = ((q @ k.transpose(-1, -2)) * s["scale"]).view(n, n_kv, group, most, -1)
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    at = torch.arange(k.shape[2], device=DEV)
    if s["slopes"] is not None:
        distance = (padded(s["pos"])[:, :, None] - at).abs().float()
        scores = scores - s["slopes"].view(n_kv, group, 1, 1) * distance[:, None, None]
    seen = at < padded(s["ends"])[:, :, None]
    if s["starts"] is not None:
        seen = seen & (at >= padded(s["starts"])[:, :, None])
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    (p,), total = softmax_parts([scores])
    out = (p.flatten(2, 3) @ v) / total.flatten(2, 3)
    out = out.view(n, n_kv, group, most, dim).permute(0, 3, 1, 2, 4).reshape(n, most, -1)
    return out[seq, index].to(s["act"])


def plain_shared(s):
    case, n_heads, n_kv, dim, page = s["case"], s["n_heads"], s["n_kv"], s["dim"], s["page"]
    n, groups, prefix = case["convs"], case["groups"], case["prefix"]
    member = s["member"]
    most, group = member.shape[1], n_heads // n_kv

    def common(x):  # [group][kv head][member, query head][...]
        return x.view(n, n_kv, group, -1)[member].transpose(1, 2).flatten(2, 3)

    def own_rows(x):  # back to [conversation][kv head][query head][...]
        return x.view(groups, n_kv, most, group, -1).transpose(1, 2).flatten(0, 1)[s["slot"]]

    q = s["q"].float()
    pages = -(-prefix // page)
    kp, vp = (cached(s, x, s["table"][member[:, 0], :pages])[:, :, :prefix] for x in ("k", "v"))
    ks, vs = (cached(s, x, s["table"][:, prefix // page:]) for x in ("k", "v"))
    first = own_rows((common(q) @ kp.transpose(-1, -2)) * s["scale"])
    second = (q.view(n, n_kv, group, dim) @ ks.transpose(-1, -2)) * s["scale"]
    at = torch.arange(ks.shape[2], device=DEV) + prefix // page * page
    seen = (at >= prefix) & (at < s["lens"][:, None])
    second = second.masked_fill(~seen[:, None, None], float("-inf"))
    (a, b), total = softmax_parts([first, second])
    out = own_rows(common(a.reshape(n, -1)) @ vp) + b @ vs
    return (out / total).reshape(n, -1).to(s["act"])


def plain_sample(s):
    # in 64 bits: a draw is a comparison with a sum of many terms
    x = s["logits"].double()
    n, vocab = x.shape
    temperature, k = s["temperature"].double()[:, None], s["top_k"].long()[:, None]
    p, m, u = (s[name].double()[:, None] for name in ("top_p", "min_p", "u"))
    greedy = temperature <= 0
    z = x / torch.where(greedy, 1.0, temperature)
    ordered = z.sort(-1, descending=True).values
    top = ordered[:, :1]
    least = torch.where((k > 1) & (k < vocab), ordered.gather(1, (k - 1).clamp(0, vocab - 1)), float("-inf"))
    w = torch.where(ordered >= least, torch.exp(ordered - top), 0.0)
    above = w.cumsum(-1) - w
    held = (above < p * w.sum(-1, keepdim=True)) & (w > 0)
    nucleus = torch.where(held, ordered, float("inf")).amin(-1, keepdim=True)
    least = torch.where((p > 0) & (p < 1), torch.maximum(least, nucleus), least)
    least = torch.where(m > 0, torch.maximum(least, top + torch.log(m)), least)
    least = torch.where(greedy, top, least)
    w = torch.where(z >= least, torch.exp(z - top), 0.0)
    so_far = w.cumsum(-1)
    total = so_far[:, -1:]
    token = (so_far <= u * total).sum(-1, keepdim=True)
    last = vocab - 1 - (w > 0).flip(-1).int().argmax(-1, keepdim=True)
    best = (z == top).int().argmax(-1, keepdim=True)
    token = torch.where(greedy, best, torch.minimum(token, last))
    prob = torch.where(greedy, 1.0, w.gather(1, token) / total)
    return [token[:, 0].to(torch.int32), prob[:, 0].float()]


# ---------------------------------------------------------------- the framework's operators


def handles(s):
    """What a program makes once for a cache and a page table."""
    import rpgbarenginecuda_b200 as rpg

    case = s["case"]
    act = {"f32": rpg.F32, "f16": rpg.F16, "bf16": rpg.BF16}[case["act"]]
    if case["op"] == "sample":
        return rpg, act
    kind = {"f16": rpg.KV_F16, "q8": rpg.KV_Q8, "q4": rpg.KV_Q4}[case["cache"]]
    scales = [s[n].data_ptr() if n in s else 0 for n in ("k_scale", "v_scale")]
    kv = rpg.PagedKv(kind, s["dim"], s["n_kv"], s["page"], s["pool"], s["k"].data_ptr(), s["v"].data_ptr(), *scales)
    table = rpg.PageTable(s["table"].data_ptr(), *s["table"].shape)
    return kv, table, act


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"rows": plain_rows, "shared": plain_shared, "sample": plain_sample}[case["op"]](s)
    if "handles" not in s:
        s["handles"] = handles(s)
    if case["op"] == "sample":
        rpg, act = s["handles"]
        rpg.sample_rows(s["logits"].data_ptr(), act, *s["logits"].shape, s["tokens"].data_ptr(), s["u"].data_ptr(),
                        temperature_ptr=s["temperature"].data_ptr(), top_k_ptr=s["top_k"].data_ptr(),
                        top_p_ptr=s["top_p"].data_ptr(), min_p_ptr=s["min_p"].data_ptr(), prob_ptr=s["probs"].data_ptr(),
                        stream=s["stream"])
        return [s["tokens"], s["probs"]]
    kv, table, act = s["handles"]
    if case["op"] == "rows":
        kv.attend_rows(table, act, s["q"].data_ptr(), s["n_heads"], s["rows"].data_ptr(), s["q"].shape[0],
                       s["ends"].data_ptr(), s["scale"], s["out"].data_ptr(), s["workspace"].data_ptr(),
                       s["workspace"].numel(), starts_ptr=s["starts"].data_ptr() if s["starts"] is not None else 0,
                       cap=case["cap"], slopes_ptr=s["slopes"].data_ptr() if s["slopes"] is not None else 0,
                       pos_ptr=s["pos"].data_ptr() if s["slopes"] is not None else 0, stream=s["stream"])
    else:
        kv.attend_shared(table, act, s["q"].data_ptr(), s["n_heads"], s["lens"].data_ptr(), s["groups"].data_ptr(),
                         case["groups"], s["prefix"].data_ptr(), s["scale"], s["out"].data_ptr(),
                         s["workspace"].data_ptr(), s["workspace"].numel(), stream=s["stream"])
    return s["out"]


# ---------------------------------------------------------------- work and exact values


def ranges(case):
    """Rows mode, per conversation: (starts, ends) of its rows, on the host."""
    for m in lengths(case):
        pos = torch.arange(m) + case["at"]
        start, end = torch.zeros_like(pos), pos + 1
        if case["mask"] == "window":
            start = (pos + 1 - case["span"]).clamp(min=0)
        elif case["mask"] == "documents":
            start = pos - pos % case["span"]
        elif case["mask"] == "prefix":
            end = end.clamp(min=min(case["span"], case["at"] + m))
        yield start, end


def work(case):
    size = 4 if case["act"] == "f32" else 2
    if case["op"] == "sample":
        values = case["convs"] * case["vocab"]
        return {"bytes": values * size + 28 * case["convs"], "flops": 2 * values}
    n_heads, n_kv, dim = HEADS[case["heads"]]
    entry = n_kv * 2 * {"f16": 2 * dim, "q8": dim + 2 * dim // GROUP, "q4": dim // 2 + 2 * dim // GROUP}[case["cache"]]
    if case["op"] == "rows":
        n = sum(lengths(case))
        seen = sum(int((e - b).sum()) for b, e in ranges(case))
        read = sum(int(e.max() - b.min()) for b, e in ranges(case))
        return {"bytes": read * entry + 2 * n * n_heads * dim * size, "flops": 4 * seen * n_heads * dim}
    own_positions = sum(lengths(case))
    return {"bytes": (case["groups"] * case["prefix"] + own_positions) * entry + 2 * case["convs"] * n_heads * dim * size,
            "flops": 4 * (case["convs"] * case["prefix"] + own_positions) * n_heads * dim}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        # the probability of the token drawn; the token itself is a whole number
        probs = []
        for i in range(case["convs"]):
            t, k = float(s["temperature"][i]), int(s["top_k"][i])
            p, m, u = float(s["top_p"][i]), float(s["min_p"][i]), float(s["u"][i])
            if t <= 0:
                probs.append(1.0)
                continue
            x = s["logits"][i].double()
            levels, inverse, counts = torch.unique(x, return_inverse=True, return_counts=True)  # ascending
            w = torch.softmax(levels / t + torch.log(counts.double()), 0)  # of whole levels
            keep = torch.ones_like(levels, dtype=torch.bool)
            if 1 < k < case["vocab"]:
                higher = counts.flip(0).cumsum(0).flip(0) - counts
                keep &= higher < k
            if 0 < p < 1:
                v = w * keep
                higher = v.flip(0).cumsum(0).flip(0) - v
                keep &= higher < p * v.sum()
            if m > 0:
                each = torch.exp((levels - levels[-1]) / t)
                keep &= each >= m
            each = (w / counts * keep)[inverse]
            each = each / each.sum()
            token = torch.searchsorted(each.cumsum(0), torch.tensor([u], dtype=torch.float64, device=DEV), right=True)
            probs.append(float(each[min(int(token), case["vocab"] - 1)]))
        return [None, torch.tensor(probs, dtype=torch.float64)]

    n_heads, n_kv, dim, page, cache = s["n_heads"], s["n_kv"], s["dim"], s["page"], case["cache"]
    group = n_heads // n_kv

    def value(name, c, n):
        """Positions 0 .. n - 1 of conversation c: [kv head][position][dim]."""
        ids = s["table"][c, :-(-n // page)].long()
        x = s[name][ids]
        if cache == "q4":
            d = torch.empty(*x.shape[:-1], dim, dtype=torch.float64, device=DEV)
            d[..., 0::2] = (x % 16).double() - 8
            d[..., 1::2] = torch.div(x, 16, rounding_mode="floor").double() - 8
        else:
            d = x.double()
        if cache != "f16":
            d = d * s[name + "_scale"][ids].double().repeat_interleave(GROUP, -1)
        return d.permute(1, 0, 2, 3).reshape(n_kv, -1, dim)[:, :n]

    outs = []
    if case["op"] == "shared":
        for c, m in enumerate(lengths(case)):
            n = case["prefix"] + m
            q = s["q"][c].double().view(n_kv, group, dim)
            w = torch.softmax(torch.einsum("hgd,hnd->hgn", q, value("k", c, n)) / math.sqrt(dim), -1)
            outs.append(torch.einsum("hgn,hnd->hgd", w, value("v", c, n)).reshape(-1))
        return torch.stack(outs)

    first = 0
    for c, (start, end) in enumerate(ranges(case)):
        m, n = len(start), int(end.max())
        q = s["q"][first:first + m].double().view(m, n_heads, dim)
        k, v = value("k", c, n), value("v", c, n)
        at = torch.arange(n, device=DEV)
        hidden = (at < start.to(DEV)[:, None]) | (at >= end.to(DEV)[:, None])
        own_pos = torch.arange(m, device=DEV) + case["at"]
        out = torch.empty(m, n_heads, dim, dtype=torch.float64, device=DEV)
        for h in range(n_heads):
            x = torch.mm(q[:, h], k[h // group].T) / math.sqrt(dim)
            if case["cap"]:
                e = torch.expm1(2 * x / case["cap"])
                x = torch.where(x > 5 * case["cap"], case["cap"] * torch.ones_like(x), case["cap"] * e / (e + 2))
            if case["slopes"]:
                slope = s["slopes"][h].double()
                x = x - slope * (own_pos[:, None] - at).abs()
            x[hidden] = -math.inf
            out[:, h] = torch.mm(torch.exp(x - torch.logsumexp(x, -1, keepdim=True)), v[h // group])
        outs.append(out.reshape(m, -1))
        first += m
    return torch.cat(outs)
