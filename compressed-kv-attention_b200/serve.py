"""A batch of sequences that answer behind one shared prompt: the serving-step operators together.

The prompt's keys are rotated by their positions once and kept compressed (XKV blobs, one set for the
whole batch) or as they are in shared pages.  Every step then takes one new token of every sequence
through every layer: its key and value go into the sequence's own pages and its query is rotated
(`Batch.append`), and it attends over the prompt and its own tokens (`Batch.attend`).  A step is
captured in a CUDA graph once and replayed: positions, lengths and slots advance on the device.

Projections are stood in for by random tensors: there is no model here.  `python serve.py --help`
lists the sizes; one JSON line reports the time of a step and the bytes of the prompt's cache.
"""
from __future__ import annotations

import argparse
import json
import os
import sys


def rope_tables(n_pos, rot_dim, base=10000.0, device="cuda"):
    """cos and sin [n_pos, rot_dim / 2] of the usual geometric angles."""
    import torch
    half = rot_dim // 2
    inv = base ** (-torch.arange(half, device=device, dtype=torch.float64) / half)
    a = torch.arange(n_pos, device=device, dtype=torch.float64)[:, None] * inv
    return a.cos().float().contiguous(), a.sin().float().contiguous()


class Session:
    """`layers` layers of a batch behind one prompt.  new_q / new_k / new_v [layers, steps, batch, heads,
    dim] are what each step's projections would give; out [layers, batch, n_q_heads, dim] is the last
    step's result."""

    def __init__(self, batch, n_q_heads, n_kv_heads, dim, prompt, steps, layers=1, page_tokens=16,
                 compressed=True, seed=0):
        import torch
        import kvexp_b200 as kvx
        self.torch, self.batch, self.steps, self.layers, self.prompt = torch, batch, steps, layers, prompt
        g = torch.Generator(device="cuda").manual_seed(seed)

        def draw(*shape):
            return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)

        self.rope = kvx.Rope(*rope_tables(prompt + steps, dim))
        self.op = kvx.Batch(batch, n_q_heads, n_kv_heads, dim)
        per = -(-steps // page_tokens)                       # pages of a sequence
        shared = 0 if compressed else -(-prompt // page_tokens)
        self.pages, self.prefix, self.prompts = [], [], []
        at = torch.arange(prompt, device="cuda", dtype=torch.int32)
        self.prefix_table = torch.arange(shared, device="cuda", dtype=torch.int32)
        for _ in range(layers):
            shape = (shared + batch * per, page_tokens, n_kv_heads, dim)
            pages = kvx.Pages(torch.empty(shape, device="cuda", dtype=torch.bfloat16),
                              torch.empty(shape, device="cuda", dtype=torch.bfloat16))
            k, v = draw(prompt, n_kv_heads, dim), draw(prompt, n_kv_heads, dim)
            self.pages.append(pages)
            self.prompts.append((k, v))
            if compressed:
                turned = torch.empty_like(k)
                self.op.rotate(k, at, self.rope, turned, stream=self._stream())
                self.prefix.append(kvx.Prefix.encode(turned.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()))
            else:
                self.op.append(None, k, v, at, self.rope, at.long(), pages, None, stream=self._stream())
        self.table = (shared + torch.arange(batch * per, device="cuda", dtype=torch.int32)).view(batch, per)
        self.lens = torch.zeros(batch, device="cuda", dtype=torch.int32)
        self.step_index = torch.zeros(1, device="cuda", dtype=torch.int64)
        self.new_q = draw(layers, steps, batch, n_q_heads, dim)
        self.new_k, self.new_v = (draw(layers, steps, batch, n_kv_heads, dim) for _ in range(2))
        self.turned = torch.empty((batch, n_q_heads, dim), device="cuda", dtype=torch.bfloat16)
        self.out = torch.zeros((layers, batch, n_q_heads, dim), device="cuda", dtype=torch.bfloat16)
        self.taken = 0               # steps since the beginning
        self._graph = None

    def _stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    @property
    def prompt_bytes(self):
        """Of all layers' prompt caches."""
        return sum(p.nbytes for p in self.prefix) or sum(2 * k.numel() * k.element_size() for k, _ in self.prompts)

    def step(self):
        """One token of every sequence through every layer, on the current stream."""
        if self.taken >= self.steps:  # (the sequences' pages are full)
            raise ValueError(f"all {self.steps} steps have been taken: rewind()")
        self.taken += 1
        page = self.pages[0].page_tokens
        s = self._stream()
        pos = self.lens + self.prompt
        place = self.lens.long()
        slots = self.table.gather(1, (place // page)[:, None])[:, 0].long() * page + place % page
        self.lens += 1
        for i in range(self.layers):
            q, k, v = (x[i].index_select(0, self.step_index)[0] for x in (self.new_q, self.new_k, self.new_v))
            self.op.append(q, k, v, pos, self.rope, slots, self.pages[i], self.turned, stream=s)
            kept = {"prefix": self.prefix[i]} if self.prefix else {"prefix_table": self.prefix_table, "prefix_len": self.prompt}
            self.op.attend(self.turned, self.out[i], self.pages[i], self.table, self.lens, self.steps, stream=s, **kept)
        self.step_index += 1

    def rewind(self):
        """Back to the beginning: the prompt alone."""
        self.lens.zero_()
        self.step_index.zero_()
        self.taken = 0

    def capture(self):
        """The next step as a graph.  A step before the capture loads the kernels; its advances are undone
        (the first replay writes the same tokens again)."""
        torch = self.torch
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.step()
        torch.cuda.current_stream().wait_stream(side)
        self.lens -= 1
        self.step_index -= 1
        self.taken -= 1
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self._graph):
            self.step()
        self.taken -= 1              # (a captured step has not run)

    def run(self):
        """Every step from the beginning; returns the milliseconds they took on the device."""
        torch = self.torch
        self.rewind()
        if self._graph is None:
            self.capture()
        self.taken = self.steps
        t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        t0.record()
        for _ in range(self.steps):
            self._graph.replay()
        t1.record()
        self.op.check()
        return t0.elapsed_time(t1)


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--q-heads", type=int, default=14)
    ap.add_argument("--kv-heads", type=int, default=2)
    ap.add_argument("--dim", type=int, default=64)
    ap.add_argument("--prompt", type=int, default=32768, help="tokens of the shared prompt")
    ap.add_argument("--steps", type=int, default=256, help="tokens each sequence generates")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--pages", action="store_true", help="keep the prompt in pages, not compressed")
    a = ap.parse_args(argv)
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    s = Session(a.batch, a.q_heads, a.kv_heads, a.dim, a.prompt, a.steps, a.layers, compressed=not a.pages)
    ms = s.run()
    print(json.dumps({"batch": a.batch, "q_heads": a.q_heads, "kv_heads": a.kv_heads, "head_dim": a.dim,
                      "prompt": a.prompt, "steps": a.steps, "layers": a.layers, "compressed": not a.pages,
                      "prompt_cache_bytes": s.prompt_bytes, "us_per_step": 1e3 * ms / a.steps,
                      "us_per_layer_step": 1e3 * ms / (a.steps * a.layers)}))
    return 0


if __name__ == "__main__":
    sys.exit(main())
