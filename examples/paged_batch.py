"""Many conversations of one model decoded together over a paged key-value cache.

A Qwen3 GGUF's layers run on the operator entries: the quantised matrices
(`Matrix.matvec`), and per layer `PagedKv.append` (per-head norms, rotation and
the write of k and v in one pass) and the attention: `PagedKv.attend_rows` where
a conversation has several new tokens (prompts, appended turns), `PagedKv.attend`
for one new token of every conversation, `PagedKv.attend_shared` where some of
them begin alike.  `sample_rows` draws the next token of all.  The conversations
share one pool of pages per layer; a page is taken when a conversation grows into
it.  A conversation can branch off another: it shares the whole pages of what
they have in common.

    python examples/paged_batch.py                       # a toy model, written on the spot
    python examples/paged_batch.py --gguf model.gguf --cache q8 --conversations 32
    python examples/paged_batch.py --instructions 200 --temperature 0.7 --top-p 0.9   # one beginning for all
"""

from __future__ import annotations

import argparse
import os
import struct
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import rpgbarenginecuda_b200 as rpg  # noqa: E402

CACHES = {"f16": rpg.KV_F16, "q8": rpg.KV_Q8, "q4": rpg.KV_Q4}
ROW_BYTES = {0: (1, 4), 8: (32, 34), 12: (256, 144), 13: (256, 176), 14: (256, 210)}  # values, bytes of a block


def read_gguf(path: str):
    """(metadata, {name: (type, shape, bytes)}) of a GGUF v3 file."""
    data = np.memmap(path, np.uint8, "r")
    at = 0

    def take(fmt):
        nonlocal at
        v = struct.unpack_from("<" + fmt, data, at)[0]
        at += struct.calcsize("<" + fmt)
        return v

    def text():
        nonlocal at
        n = take("Q")
        at += n
        return bytes(data[at - n:at]).decode("utf-8", "replace")

    scalars = {0: "B", 1: "b", 2: "H", 3: "h", 4: "I", 5: "i", 6: "f", 7: "B", 10: "Q", 11: "q", 12: "d"}

    def value(kind):
        if kind == 8:
            return text()
        if kind == 9:
            inner, n = take("I"), take("Q")
            return [value(inner) for _ in range(n)]
        return take(scalars[kind])

    if take("I") != 0x46554747 or take("I") != 3:
        raise ValueError(f"{path} is not a GGUF v3 file")
    n_tensors, n_meta = take("Q"), take("Q")
    meta = {}
    for _ in range(n_meta):
        key = text()
        meta[key] = value(take("I"))
    infos = []
    for _ in range(n_tensors):
        name = text()
        shape = [take("Q") for _ in range(take("I"))]
        infos.append((name, take("I"), shape, take("Q")))
    align = meta.get("general.alignment", 32)
    base = (at + align - 1) // align * align
    tensors = {}
    for name, kind, shape, offset in infos:
        values, size = ROW_BYTES[kind]
        n = int(np.prod(shape)) // values * size
        tensors[name] = (kind, shape, data[base + offset:base + offset + n])
    return meta, tensors


class PagedModel:
    """The model's weights, and per layer the pages that its conversations share."""

    def __init__(self, path: str, cache: str = "f16", page: int = 16, n_pages: int = 256, max_conversations: int = 64,
                 max_positions: int = 2048):
        meta, tensors = read_gguf(path)
        arch = meta["general.architecture"]
        g = lambda key: meta[f"{arch}.{key}"]  # noqa: E731
        self.n_layers, self.n_heads, self.n_kv = g("block_count"), g("attention.head_count"), g("attention.head_count_kv")
        self.dim, self.eps = g("attention.key_length"), g("attention.layer_norm_rms_epsilon")
        self.page, self.max_pages, self.max_positions = page, -(-max_positions // page), max_positions

        def matrix(name):
            kind, (cols, rows), data = tensors[name]
            return rpg.Matrix(kind, rows, cols, data)

        def vector(name):
            return torch.from_numpy(tensors[name][2].view(np.float32).copy()).cuda()

        self.embd = matrix("token_embd.weight")
        self.head = matrix("output.weight") if "output.weight" in tensors else self.embd
        self.out_norm = vector("output_norm.weight")
        self.layers = []
        rope = torch.from_numpy(rpg.rope_table(max_positions, self.dim, g("rope.freq_base"))).cuda()
        row = {"f16": 2 * self.dim, "q8": self.dim, "q4": self.dim // 2}[cache]
        for i in range(self.n_layers):
            w = {n: matrix(f"blk.{i}.{n}.weight") for n in ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate",
                                                            "ffn_up", "ffn_down")}
            w |= {n: vector(f"blk.{i}.{n}.weight") for n in ("attn_norm", "ffn_norm", "attn_q_norm", "attn_k_norm")}
            pool = [torch.zeros(n_pages, self.n_kv, page, row, dtype=torch.uint8, device="cuda") for _ in range(2)]
            if cache != "f16":
                pool += [torch.zeros(n_pages, self.n_kv, page, self.dim // rpg.KV_GROUP, dtype=torch.float16,
                                     device="cuda") for _ in range(2)]
            w["pool"] = pool
            w["kv"] = rpg.PagedKv(CACHES[cache], self.dim, self.n_kv, page, n_pages, *(t.data_ptr() for t in pool))
            w["rotary"] = rpg.Rotary(rope.data_ptr(), max_positions, w["attn_q_norm"].data_ptr(),
                                     w["attn_k_norm"].data_ptr(), self.eps)
            self.layers.append(w)
        self.rope = rope
        self.free = list(range(n_pages))[::-1]
        self.used = np.zeros(n_pages, np.int32)  # conversations that hold a page
        self.table = np.full((max_conversations, self.max_pages), -1, np.int32)
        self.lengths: dict[int, int] = {}
        self.alike: dict[int, tuple[int, int]] = {}  # (group, positions) of conversations that begin alike
        self.groups = 0
        shape = self.n_heads, self.n_kv, self.dim
        # zeroed once; the one for shared beginnings holds the one for single tokens, prompts have one of their own
        self.workspace = torch.zeros(rpg.attend_shared_workspace(*shape, max_conversations), dtype=torch.uint8, device="cuda")
        self.rows_workspace = torch.empty(rpg.attend_rows_workspace(*shape), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()  # forward may come on another stream

    def open(self) -> int:
        """A new conversation."""
        c = next((i for i in range(len(self.table)) if i not in self.lengths), None)
        if c is None:
            raise RuntimeError(f"all {len(self.table)} conversations are open")
        self.lengths[c] = 0
        return c

    def branch(self, c: int, n: int | None = None) -> int:
        """A new conversation that begins with the first n positions of c (None: all of them).

        Whole pages are shared; of the page that n ends in, the new conversation gets a copy."""
        n = self.lengths[c] if n is None else n
        if not 0 <= n <= self.lengths[c]:
            raise ValueError(f"conversation {c} has {self.lengths[c]} positions, not {n}")
        whole, rest = divmod(n, self.page)
        if rest and not self.free:
            raise RuntimeError(f"no page for position {whole * self.page} of a branch of conversation {c}")
        d = self.open()
        self.table[d, :whole] = self.table[c, :whole]
        if rest:
            self.table[d, whole] = self.free.pop()
            for w in self.layers:
                for t in w["pool"]:
                    t[int(self.table[d, whole])].copy_(t[int(self.table[c, whole])])
        for p in self.table[d, :whole + (rest > 0)]:
            self.used[p] += 1
        self.lengths[d] = n
        group, common = self.alike.get(c, (0, -1))
        if n > common:  # c leaves a group that shares less than this
            self.groups += 1
            group, common = self.groups, n
            self.alike[c] = (group, n)
        self.alike[d] = (group, n)
        return d

    def close(self, c: int):
        """Ends a conversation; pages that no other one holds go back to the pool."""
        for p in self.table[c][self.table[c] >= 0]:
            self.used[p] -= 1
            if self.used[p] == 0:
                self.free.append(int(p))
        self.table[c] = -1
        del self.lengths[c]
        self.alike.pop(c, None)

    def forward(self, tokens: list[tuple[int, int]]) -> torch.Tensor:
        """Appends (conversation, token id) rows, in order, and returns their logits [row][vocabulary].

        Runs on torch's current stream.  A call that raises leaves the conversations as they were."""
        stream = torch.cuda.current_stream().cuda_stream
        lengths, places, at = dict(self.lengths), self.table.copy(), []
        taken = 0
        for c, _ in tokens:
            p = lengths[c]
            if p >= self.max_positions:  # (the rotation table ends there)
                raise RuntimeError(f"conversation {c} is full ({p} positions)")
            if p % self.page == 0 and taken == len(self.free):
                raise RuntimeError(f"no page for position {p} of conversation {c}")
            if p % self.page == 0:
                taken += 1
                places[c, p // self.page] = self.free[-taken]
            at.append(p)
            lengths[c] = p + 1
        n = len(tokens)
        # rows by conversation, conversations that begin alike side by side
        key = [(self.alike.get(c, (0, 0))[0], c) for c, _ in tokens]
        order = sorted(range(n), key=lambda r: key[r])
        convs = [c for r, c in enumerate(key[i][1] for i in order) if r == 0 or c != key[order[r - 1]][1]]
        seq = torch.tensor([convs.index(key[i][1]) for i in order], dtype=torch.int32, device="cuda")
        pos = torch.tensor([at[i] for i in order], dtype=torch.int32, device="cuda")
        ends = pos + 1
        table = torch.from_numpy(places[convs]).cuda()
        pages = rpg.PageTable(table.data_ptr(), len(convs), self.max_pages)

        def ints(x):
            return torch.tensor(x, dtype=torch.int32, device="cuda")

        bounds = groups = None
        if n > len(convs):  # several new tokens of a conversation
            counts = [sum(key[i][1] == c for i in order) for c in convs]
            bounds = ints(np.concatenate([[0], np.cumsum(counts)]))
        else:
            first, prefix = [], []
            for i, c in enumerate(convs):
                group, common = self.alike.get(c, (0, 0))
                if i and group and group == self.alike.get(convs[i - 1], (0, 0))[0]:
                    prefix[-1] = min(prefix[-1], common)
                else:
                    first.append(i)
                    prefix.append(common)
            first.append(n)
            if len(first) <= n:  # some begin alike
                groups = ints(first)
                common = ints(np.repeat(prefix, np.diff(first)))
        x = torch.empty(n, self.embd.cols, device="cuda")
        for i, r in enumerate(order):
            self.embd.dequant(tokens[r][1], 1, x[i].data_ptr(), stream)

        def product(m, y):
            out = torch.empty(n, m.rows, device="cuda")
            m.matvec(y.data_ptr(), n, out.data_ptr(), stream)
            return out

        def norm(y, w):
            return (y * torch.rsqrt((y * y).mean(-1, keepdim=True) + self.eps) * w).contiguous()

        q = torch.empty(n, self.n_heads * self.dim, device="cuda")
        att = torch.empty_like(q)
        for w in self.layers:
            y = norm(x, w["attn_norm"])
            qkv = torch.cat([product(w[m], y) for m in ("attn_q", "attn_k", "attn_v")], 1)
            w["kv"].append(pages, w["rotary"], rpg.F32, qkv.data_ptr(), self.n_heads, pos.data_ptr(), n, q.data_ptr(),
                           seq_ptr=seq.data_ptr(), stream=stream)
            if bounds is not None:
                w["kv"].attend_rows(pages, rpg.F32, q.data_ptr(), self.n_heads, bounds.data_ptr(), n, ends.data_ptr(),
                                    self.dim ** -0.5, att.data_ptr(), self.rows_workspace.data_ptr(),
                                    self.rows_workspace.numel(), stream=stream)
            elif groups is not None:
                w["kv"].attend_shared(pages, rpg.F32, q.data_ptr(), self.n_heads, ends.data_ptr(), groups.data_ptr(),
                                      len(first) - 1, common.data_ptr(), self.dim ** -0.5, att.data_ptr(),
                                      self.workspace.data_ptr(), self.workspace.numel(), stream=stream)
            else:
                w["kv"].attend(pages, rpg.F32, q.data_ptr(), self.n_heads, ends.data_ptr(), self.dim ** -0.5,
                               att.data_ptr(), self.workspace.data_ptr(), self.workspace.numel(), stream=stream)
            x = x + product(w["attn_output"], att)
            y = norm(x, w["ffn_norm"])
            h = torch.nn.functional.silu(product(w["ffn_gate"], y)) * product(w["ffn_up"], y)
            x = x + product(w["ffn_down"], h)
        logits = product(self.head, norm(x, self.out_norm))
        if taken:
            self.used[self.free[-taken:]] = 1
            del self.free[-taken:]
        self.table, self.lengths = places, lengths
        back = np.empty(n, np.int64)
        back[order] = np.arange(n)
        return logits[torch.from_numpy(back).cuda()]

    def sample(self, logits: torch.Tensor, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0,
               min_p: float = 0.0, generator: torch.Generator | None = None) -> list[int]:
        """The next token of every row of logits; a temperature of 0 takes the largest."""
        n = logits.shape[0]
        options = torch.tensor([temperature, top_p, min_p], device="cuda")[:, None].expand(3, n).contiguous()
        k = torch.full((n,), top_k, dtype=torch.int32, device="cuda")
        u = torch.rand(n, generator=generator, device="cuda")
        out = torch.empty(n, dtype=torch.int32, device="cuda")
        rpg.sample_rows(logits.data_ptr(), rpg.F32, n, logits.shape[1], out.data_ptr(), u.data_ptr(),
                        temperature_ptr=options[0].data_ptr(), top_k_ptr=k.data_ptr(), top_p_ptr=options[1].data_ptr(),
                        min_p_ptr=options[2].data_ptr(), stride=logits.stride(0),
                        stream=torch.cuda.current_stream().cuda_stream)
        return out.tolist()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--gguf", help="a Qwen3 GGUF (default: the toy model, written to a cache folder)")
    ap.add_argument("--cache", choices=sorted(CACHES), default="f16")
    ap.add_argument("--conversations", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--instructions", type=int, default=0, help="tokens that all conversations begin with")
    ap.add_argument("--temperature", type=float, default=0.0, help="0: the likeliest token")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    a = ap.parse_args(argv)
    if a.gguf is None:
        from dataclasses import replace

        from rpgbarenginecuda_b200 import synthetic

        a.gguf = synthetic.cached_model(replace(synthetic.PRESETS["tiny"], weight_std=0.06), seed=1)
    m = PagedModel(a.gguf, a.cache, n_pages=16 * a.conversations + a.instructions // 16 + 1,
                   max_conversations=a.conversations + 1)
    rng = np.random.default_rng(0)
    dice = torch.Generator(device="cuda").manual_seed(0)

    def draw(logits):
        return m.sample(logits, a.temperature, a.top_k, a.top_p, a.min_p, dice)

    if a.instructions:
        root = m.open()
        m.forward([(root, int(t)) for t in rng.integers(0, m.embd.rows, a.instructions)])
        ids = [m.branch(root) for _ in range(a.conversations)]
        m.close(root)
    else:
        ids = [m.open() for _ in range(a.conversations)]
    last = {}
    for c in ids:  # prompts of different lengths
        prompt = rng.integers(0, m.embd.rows, 5 + 7 * (c % 5))
        last[c] = draw(m.forward([(c, int(t)) for t in prompt])[-1:])[0]
    out = {c: [last[c]] for c in ids}
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(a.steps):
        logits = m.forward([(c, last[c]) for c in ids])
        for c, t in zip(ids, draw(logits)):
            last[c] = t
            out[c].append(t)
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    for c in ids:
        print(f"conversation {c} ({m.lengths[c]} positions): {out[c]}")
    print(f"{a.conversations * a.steps / dt:.0f} tokens/s over {a.conversations} conversations ({a.cache} cache)")
    return out


if __name__ == "__main__":
    main()
