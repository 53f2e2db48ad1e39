"""Several answers to one prompt over a shared, paged, quantised cache.

A small decoder (random weights: normed and rotated grouped-query attention, residual
stream) reads a prompt once, then continues it as ``seqs`` sequences whose block tables
name the prompt's pages:

  prompt   append_qkv_paged(want_hat=True): norm, rotation and the cache's rows in one launch;
           the prompt's own causal attention runs on k_hat and v_hat, the rows as cached
  fork     the prompt's whole pages are shared, its last, unfinished page is copied
  step     append_qkv_paged for one token of every sequence, then decode_attention_shared,
           which reads the prompt once for all of them
  check    qk_norm_rope keeps a cache in full precision beside it (check=True)

    python examples/shared_prompt.py --prompt 4000 --seqs 16 --steps 32
"""
from __future__ import annotations

import argparse
import os
import sys
from dataclasses import dataclass

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from bitcache_b200 import _lib, planes  # noqa: E402


@dataclass
class Layer:
    wqkv: torch.Tensor
    wo: torch.Tensor
    rope: planes.Rope
    K: planes.Planes
    V: planes.Planes


class Decoder:
    def __init__(self, hidden: int, layers: int, n_heads: int, n_kv_heads: int, head_dim: int, max_len: int, seqs: int,
                 page_size: int, device: torch.device, seed: int) -> None:
        gen = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
        self.heads, self.kv, self.dim, self.seqs, self.page = n_heads, n_kv_heads, head_dim, seqs, page_size
        self.pages_each = -(-max_len // page_size)
        n_pages = n_kv_heads * self.pages_each * (seqs + 1)  # at most: the prompt's, and each sequence's own
        angle = torch.arange(max_len, device=device)[:, None] * 10000.0 ** (
            -torch.arange(0, head_dim, 2, device=device) / head_dim)
        cos, sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        self.layers = []
        for _ in range(layers):
            wq, wk = (1 + 0.1 * rand(head_dim) for _ in range(2))
            self.layers.append(Layer((rand((n_heads + 2 * n_kv_heads) * head_dim, hidden) * hidden**-0.5).half(),
                                     (rand(hidden, n_heads * head_dim) * (n_heads * head_dim) ** -0.5).half(),
                                     planes.Rope(cos, sin, q_weight=wq, k_weight=wk),
                                     *(planes.Planes.empty(n_pages, page_size, head_dim, True, device) for _ in range(2))))
        self.table = torch.full((seqs, n_kv_heads, self.pages_each), -1, dtype=torch.int32, device=device)
        self.n_pages, self.used = n_pages, 0

    def _take(self, n: int) -> torch.Tensor:
        ids = torch.arange(self.used, self.used + n, dtype=torch.int32, device=self.table.device)
        self.used += n
        return ids

    def page_table(self, seqs: int) -> planes.PageTable:
        return planes.PageTable(self.table[:seqs].reshape(seqs * self.kv, self.pages_each), self.page, self.n_pages)

    def qkv(self, layer: Layer, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        x = (x * torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + 1e-6)).half()
        heads = F.linear(x, layer.wqkv).view(x.shape[0], self.heads + 2 * self.kv, self.dim)
        return heads.split((self.heads, self.kv, self.kv), 1)

    def prompt(self, x: torch.Tensor, exact: list | None) -> torch.Tensor:
        """x [tokens, hidden] as sequence 0; returns the last token's state."""
        n = x.shape[0]
        whole = -(-n // self.page)
        self.table[0, :, :whole] = self._take(self.kv * whole).view(self.kv, whole)
        pos = torch.arange(n, dtype=torch.int32, device=x.device)
        ids, pt = torch.zeros_like(pos), self.page_table(1)
        for layer in self.layers:
            q, k, v = self.qkv(layer, x)
            if exact is not None:
                exact.append((planes.qk_norm_rope(q, k, pos, layer.rope)[1].float(), v.float()))
            qr, kh, vh = planes.append_qkv_paged(q, k, v, layer.K, layer.V, pt, ids, pos, layer.rope, want_hat=True)
            o = F.scaled_dot_product_attention(*(t.transpose(0, 1)[None] for t in (qr, kh, vh)), is_causal=True,
                                               enable_gqa=True)
            x = x + F.linear(o[0].transpose(0, 1).reshape(n, -1), layer.wo)
        return x[-1]

    def fork(self, n: int, steps: int) -> None:
        """All sequences continue sequence 0's n tokens, by up to `steps` more."""
        whole, last = n // self.page, -(-(n + steps) // self.page)
        self.table[1:, :, :whole] = self.table[0, :, :whole]
        tail = self.table[0, :, whole].long() if n % self.page else None
        for b in range(self.seqs):
            own = self._take(self.kv * (last - whole)).view(self.kv, -1)
            if tail is not None:
                for layer in self.layers:
                    for P in (layer.K, layer.V):
                        for t in (P.sign, P.bscale, P.nib, P.rscale):
                            t[own[:, 0].long()] = t[tail]
            self.table[b, :, whole:last] = own

    def step(self, x: torch.Tensor, lens: torch.Tensor, prefix: torch.Tensor | None, exact: list | None,
             errors: list | None) -> torch.Tensor:
        """One token of every sequence: x [seqs, hidden] at positions lens."""
        pt = self.page_table(self.seqs)
        ids = torch.arange(self.seqs, dtype=torch.int32, device=x.device)
        for i, layer in enumerate(self.layers):
            q, k, v = self.qkv(layer, x)
            qr = planes.append_qkv_paged(q, k, v, layer.K, layer.V, pt, ids, lens, layer.rope)
            o = planes.decode_attention_shared(qr, layer.K, layer.V, pt, lens + 1, prefix)
            if exact is not None:
                qe, ke = planes.qk_norm_rope(q, k, lens, layer.rope)
                exact[i] = tuple(torch.cat((c, t[:, None].float()), 1) for c, t in zip(exact[i], (ke, v)))
                want = F.scaled_dot_product_attention(qe.float()[:, :, None], *(c.transpose(1, 2) for c in exact[i]),
                                                      enable_gqa=True)[:, :, 0]
                errors.append(((o.float() - want).norm() / want.norm()).item())
            x = x + F.linear(o.view(self.seqs, -1), layer.wo)
        return x


def run(prompt: int = 1000, seqs: int = 8, steps: int = 8, hidden: int = 512, layers: int = 2, n_heads: int = 32,
        n_kv_heads: int = 8, head_dim: int = 128, page_size: int = 256, share: bool = True, check: bool = False,
        seed: int = 0) -> dict:
    """Returns the last states [seqs, hidden], the device time of a step and, with check (steps then
    run one by one, untimed), each attention's relative difference from full precision."""
    device = torch.device("cuda")
    net = Decoder(hidden, layers, n_heads, n_kv_heads, head_dim, prompt + steps, seqs, page_size, device, seed)
    gen = torch.Generator(device=device).manual_seed(seed + 1)
    exact, errors = ([], []) if check else (None, None)
    last = net.prompt(torch.randn(prompt, hidden, generator=gen, device=device).half(), exact)
    net.fork(prompt, steps)
    if check:
        exact = [tuple(c[None].expand(seqs, *c.shape) for c in kv) for kv in exact]
    # (the sequences part by noise on their first state; a real decoder samples)
    x = last + 0.5 * torch.randn(seqs, hidden, generator=gen, device=device).half()
    lens = torch.full((seqs,), prompt, dtype=torch.int32, device=device)
    prefix = torch.full((1,), prompt, dtype=torch.int32, device=device) if share else None
    stream = torch.cuda.Stream()
    marks = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        if check:
            for _ in range(steps):
                x = net.step(x, lens, prefix, exact, errors)
                lens += 1
        else:
            # One captured step, replayed: lengths and states are device memory.  The step before the capture
            # loads the kernels and makes the workspaces; the first replay writes its cache rows again.
            net.step(x, lens, prefix, None, None)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                x.copy_(net.step(x, lens, prefix, None, None))
                lens += 1
            marks[0].record()
            for _ in range(steps):
                graph.replay()
            marks[1].record()
    torch.cuda.synchronize()
    if _lib.device_error():
        raise RuntimeError("the kernels reported an index, page or timeout error")
    return {"x": x, "ms": None if check else marks[0].elapsed_time(marks[1]) / steps, "errors": errors}


def main() -> None:
    ap = argparse.ArgumentParser(description="Several answers to one prompt over a shared quantised cache.")
    for name, value in (("prompt", 4000), ("seqs", 16), ("steps", 32), ("layers", 4), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = vars(ap.parse_args())
    shared, apart = run(**a), run(**a, share=False)
    errors = run(**a | {"steps": min(4, a["steps"])}, check=True)["errors"]
    print(f"{a['seqs']} sequences after {a['prompt']} tokens, {a['layers']} layers: {shared['ms']:.3f} ms a step, "
          f"{apart['ms']:.3f} without sharing the prompt's reads")
    print(f"attention against full precision: {sum(errors) / len(errors):.3f} relative (random keys and queries)")


if __name__ == "__main__":
    main()
