"""Many conversations of one model decoded together over a paged key-value cache.

A Qwen3 GGUF's layers run on the operator entries: the quantised matrices
(`Matrix.matvec`), and per layer `PagedKv.append` (per-head norms, rotation and
the write of k and v in one pass) and `PagedKv.attend` (one new token of every
conversation).  The conversations share one pool of pages per layer; a page is
taken when a conversation grows into it.  A prompt goes through the same two
calls, one row per token, with every row's own length.

    python examples/paged_batch.py                       # a toy model, written on the spot
    python examples/paged_batch.py --gguf model.gguf --cache q8 --conversations 32
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
        self.table = np.full((max_conversations, self.max_pages), -1, np.int32)
        self.lengths: dict[int, int] = {}
        self.workspace = torch.zeros(rpg.attend_workspace(self.n_heads, self.n_kv, self.dim), dtype=torch.uint8,
                                     device="cuda")
        torch.cuda.synchronize()  # forward may come on another stream

    def open(self) -> int:
        """A new conversation."""
        c = next((i for i in range(len(self.table)) if i not in self.lengths), None)
        if c is None:
            raise RuntimeError(f"all {len(self.table)} conversations are open")
        self.lengths[c] = 0
        return c

    def close(self, c: int):
        """Ends a conversation; its pages go back to the pool."""
        self.free += [int(p) for p in self.table[c] if p >= 0]
        self.table[c] = -1
        del self.lengths[c]

    def forward(self, tokens: list[tuple[int, int]]) -> torch.Tensor:
        """Appends (conversation, token id) rows, in order, and returns their logits [row][vocabulary].

        Runs on torch's current stream.  A call that raises leaves the conversations as they were."""
        stream = torch.cuda.current_stream().cuda_stream
        seq, pos, lengths, places = [], [], dict(self.lengths), self.table.copy()
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
            seq.append(c)
            pos.append(p)
            lengths[c] = p + 1
        n = len(tokens)
        # every row has its own page list and length: a prompt's rows see what comes before them
        table = torch.from_numpy(places[seq]).cuda()
        pages = rpg.PageTable(table.data_ptr(), n, self.max_pages)
        pos = torch.tensor(pos, dtype=torch.int32, device="cuda")
        lens = pos + 1
        x = torch.empty(n, self.embd.cols, device="cuda")
        for i, (_, token) in enumerate(tokens):
            self.embd.dequant(token, 1, x[i].data_ptr(), stream)

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
                           stream=stream)
            w["kv"].attend(pages, rpg.F32, q.data_ptr(), self.n_heads, lens.data_ptr(), self.dim ** -0.5, att.data_ptr(),
                           self.workspace.data_ptr(), self.workspace.numel(), stream=stream)
            x = x + product(w["attn_output"], att)
            y = norm(x, w["ffn_norm"])
            h = torch.nn.functional.silu(product(w["ffn_gate"], y)) * product(w["ffn_up"], y)
            x = x + product(w["ffn_down"], h)
        logits = product(self.head, norm(x, self.out_norm))
        del self.free[len(self.free) - taken:]
        self.table, self.lengths = places, lengths
        return logits


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--gguf", help="a Qwen3 GGUF (default: the toy model, written to a cache folder)")
    ap.add_argument("--cache", choices=sorted(CACHES), default="f16")
    ap.add_argument("--conversations", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args(argv)
    if a.gguf is None:
        from dataclasses import replace

        from rpgbarenginecuda_b200 import synthetic

        a.gguf = synthetic.cached_model(replace(synthetic.PRESETS["tiny"], weight_std=0.06), seed=1)
    m = PagedModel(a.gguf, a.cache, n_pages=16 * a.conversations, max_conversations=a.conversations)
    rng = np.random.default_rng(0)
    ids = [m.open() for _ in range(a.conversations)]
    last = {}
    for c in ids:  # prompts of different lengths
        prompt = rng.integers(0, m.embd.rows, 5 + 7 * (c % 5))
        last[c] = int(m.forward([(c, int(t)) for t in prompt])[-1].argmax())
    out = {c: [last[c]] for c in ids}
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(a.steps):
        logits = m.forward([(c, last[c]) for c in ids])
        for c, t in zip(ids, logits.argmax(-1).tolist()):
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
