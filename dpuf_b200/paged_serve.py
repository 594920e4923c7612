"""Serving over the paged cache: a mode-12 model whose sequences share pools of pages and are
batched step by step, prompts in chunks beside single tokens, sampled on the device.

    python -m dpuf_b200.paged_serve --model tiny --sequences 6 --tokens 16

Every projection is the framework's own mode-12 matmul (`dpuf_cuda_matmul_dev`); positions, the
cache, attention and sampling are `dpuf_b200.serving`.  The norms, the SwiGLU and the residual
adds between them are torch operations: this shows how the operators are used together, the
engine's own serving path is `CudaTransformerEngine.decode_batch`.
"""
from __future__ import annotations

import argparse
import ctypes
import os

import numpy as np
import torch

from . import engine, model as mdl, serving

_DEADZONE = 0.005  # the engine's default of DPUF_SWIGLU_DEADZONE


class PagedModel:
    """A `model.ModelData` (mode 12) on the GPU with one paged cache per layer.  Sequences are
    numbers from `open`; `step` runs some tokens of several of them and returns each one's last
    logits; `close` gives a sequence's pages back."""

    def __init__(self, model: mdl.ModelData, n_pages: int, page_size: int = 16, kv_dtype=torch.float16):
        s = self.shape = model.shape
        self.model, self.page_size = model, page_size
        self._matrices = {}
        names = ["output.weight" if "output.weight" in model.blobs else "token_embd.weight"]
        names += [f"blk.{l}.{n}" for l in range(s.layers) for n, _, _ in s.linear_shapes()]
        for n in names:
            self._matrices[n] = (engine.upload(model.blobs[n]), model.blobs[n].rows)
        self.head = names[0]
        self.norms = {n: torch.from_numpy(g).cuda() for n, g in model.norms.items()}
        self.cos, self.sin = serving.rope_table(s.max_seq, s.head_dim, s.rope_theta)
        self.caches = [serving.PagedCache.empty(n_pages, s.n_kv, page_size, s.head_dim, kv_dtype)
                       for _ in range(s.layers)]
        self.workspace = serving.attention_workspace()
        self.deadzone = float(os.environ.get("DPUF_SWIGLU_DEADZONE", _DEADZONE))
        self.free = list(range(n_pages))
        self.pages: dict[int, list[int]] = {}
        self.length: dict[int, int] = {}

    def open(self) -> int:
        s = max(self.pages, default=-1) + 1
        self.pages[s], self.length[s] = [], 0
        return s

    def close(self, seq: int) -> None:
        self.free += self.pages.pop(seq)
        del self.length[seq]

    def release(self) -> None:
        for h, _ in self._matrices.values():
            engine.w12_free(h)
        self._matrices = {}

    def _matmul(self, name: str, x: torch.Tensor) -> torch.Tensor:
        handle, rows = self._matrices[name]
        y = torch.empty((x.shape[0], rows), dtype=torch.float32, device=x.device)
        rc = engine.cuda_lib().dpuf_cuda_matmul_dev(ctypes.c_void_p(handle), x.shape[0], x.data_ptr(), y.data_ptr(),
                                                    torch.cuda.current_stream().cuda_stream)
        if rc != 0:
            raise RuntimeError(f"dpuf_cuda_matmul_dev failed with rc={rc}: {engine.last_error()}")
        return y

    def _norm(self, x: torch.Tensor, name: str) -> torch.Tensor:
        inv = (x.square().mean(-1, keepdim=True) + self.shape.rms_eps).rsqrt()
        return (x * inv * self.norms[name]).contiguous()

    def _reserve(self, seq: int, tokens: int) -> None:
        need = -(-(self.length[seq] + tokens) // self.page_size) - len(self.pages[seq])
        if self.length[seq] + tokens > self.shape.max_seq:
            raise ValueError("sequence longer than the model's positions")
        if need > len(self.free):
            raise RuntimeError("no free pages")
        for _ in range(need):
            self.pages[seq].append(self.free.pop())

    def step(self, batch: list[tuple[int, list[int]]]) -> torch.Tensor:
        """Runs the tokens of each (sequence, ids) after what the sequence holds; logits
        `[len(batch), vocab]` (float32, on the GPU) of each one's last token."""
        s = self.shape
        counts = [len(ids) for _, ids in batch]
        if not batch or min(counts) < 1 or len({seq for seq, _ in batch}) != len(batch):
            raise ValueError("a step needs tokens of distinct sequences")
        for seq, ids in batch:
            self._reserve(seq, len(ids))
        start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        table = np.full((len(batch), max(len(self.pages[q]) for q, _ in batch)), -1, np.int32)
        for i, (seq, _) in enumerate(batch):
            table[i, : len(self.pages[seq])] = self.pages[seq]
        at = np.concatenate([self.length[q] + np.arange(n) for (q, _), n in zip(batch, counts)]).astype(np.int32)
        rows = np.repeat(np.arange(len(batch)), counts).astype(np.int32)
        total = np.array([self.length[q] + n for (q, _), n in zip(batch, counts)], np.int32)
        table, q_start, kv_len, seq_of, pos = (torch.from_numpy(x).cuda() for x in (table, start, total, rows, at))
        ids = np.concatenate([np.asarray(i, np.int32) for _, i in batch])
        h = torch.from_numpy(engine.embed(self.model.blobs["token_embd.weight"], ids)).cuda()
        heads = lambda x: x.unflatten(1, (-1, s.head_dim))  # noqa: E731
        for l, cache in enumerate(self.caches):
            b = f"blk.{l}."
            x = self._norm(h, b + "attn_norm.weight")
            q, k, v = (heads(self._matmul(b + f"attn_{n}.weight", x)) for n in "qkv")
            if self.model.has_qk_norm:
                q, k = self._norm(q, b + "attn_q_norm.weight"), self._norm(k, b + "attn_k_norm.weight")
            q = serving.rope_append(cache, table, q, k, v, self.cos, self.sin, seq_of, pos)
            o = serving.paged_attention(cache, table, q, q_start, kv_len, max(counts), workspace=self.workspace)
            h = h + self._matmul(b + "attn_output.weight", o.flatten(1))
            x = self._norm(h, b + "ffn_norm.weight")
            gate, up = self._matmul(b + "ffn_gate.weight", x), self._matmul(b + "ffn_up.weight", x)
            y = torch.nn.functional.silu(gate) * up
            if self.deadzone > 0:
                y = torch.where(y.abs() >= self.deadzone, y, 0.0)
            h = h + self._matmul(b + "ffn_down.weight", y)
        serving.attention_check(workspace=self.workspace)  # (before the new positions count: a step can be repeated)
        for seq, i in batch:
            self.length[seq] += len(i)
        last = self._norm(h[(q_start[1:] - 1).long()], "output_norm.weight")
        return self._matmul(self.head, last)


def generate(paged: PagedModel, prompts, n_new: int, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0,
             min_p: float = 0.0, chunk: int = 64, seed: int = 0) -> list[list[int]]:
    """n_new tokens after each prompt.  Prompts go in by chunks of at most `chunk` tokens, in the
    same steps in which the sequences that are past theirs generate."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    todo = [list(map(int, p)) for p in prompts]
    seqs = [paged.open() for _ in prompts]
    out: list[list[int]] = [[] for _ in prompts]
    try:
        while any(len(o) < n_new for o in out):
            live = [i for i, o in enumerate(out) if len(o) < n_new]
            batch = [(seqs[i], todo[i][:chunk]) for i in live]
            logits = paged.step(batch)
            for i in live:
                todo[i] = todo[i][chunk:]
            n = len(live)
            full = lambda x, t: torch.full((n,), x, dtype=t, device="cuda")  # noqa: E731
            ids, _ = serving.sample(logits, torch.rand(n, generator=g, device="cuda"), full(temperature, torch.float32),
                                    full(top_k, torch.int32), full(top_p, torch.float32), full(min_p, torch.float32))
            for i, token in zip(live, ids.tolist()):
                if not todo[i]:  # the prompt is in: this is its next token
                    out[i].append(token)
                    todo[i] = [token]
    finally:
        for s in seqs:
            paged.close(s)
    return out


def main(argv=None) -> None:
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--model", default="tiny", choices=sorted(mdl.SHAPES))
    a.add_argument("--sequences", type=int, default=6)
    a.add_argument("--tokens", type=int, default=16)
    a.add_argument("--temperature", type=float, default=0.8)
    a.add_argument("--top-k", type=int, default=50)
    a.add_argument("--top-p", type=float, default=0.95)
    a.add_argument("--min-p", type=float, default=0.0)
    a.add_argument("--kv", default="float16", choices=["float16", "bfloat16", "float32"])
    a.add_argument("--seed", type=int, default=0)
    args = a.parse_args(argv)
    m = mdl.SyntheticModel(mdl.SHAPES[args.model], seed=args.seed)
    prompts = [mdl.prompt_ids(5 + 17 * i, m.shape.vocab, args.seed + i) for i in range(args.sequences)]
    longest = len(prompts[-1]) + args.tokens
    paged = PagedModel(m, args.sequences * (longest // 16 + 2), kv_dtype=getattr(torch, args.kv))
    for i, ids in enumerate(generate(paged, prompts, args.tokens, args.temperature, args.top_k, args.top_p, args.min_p,
                                     seed=args.seed)):
        print(f"sequence {i} ({len(prompts[i])} prompt tokens): {ids}")
    paged.release()


if __name__ == "__main__":
    main()
