"""Generation with a paged cache: the Q8_0 projections of a decode stack with
attention between them.

A layer is QKV -> attention -> O (+ residual) -> gate/up -> SwiGLU -> down
(+ residual), each projection the framework's batched Q8_0 MUL_MAT (at most 16
activation rows per call) on RMS-normalised rows.  The cache (ane_b200.kvcache)
holds the keys and values of every sequence; a prompt runs through attn_prompt
once, is forked into as many continuations as are wanted, and each step attends
to the prompt's pages once for all of them.

The weights are seeded random ones of the stack's shapes (there is no model file
here, hence no positions in the attention and no vocabulary): rows of activations
go in, rows come out.

    python -m ane_b200.generate --layers 4 --prompt 500 --children 8 --steps 32
"""
from __future__ import annotations

import torch

import ane_b200 as ane
from ane_b200.decode import ROW_BLOCK, block_seed, q8_row_bytes
from ane_b200.kvcache import KVCache


class Layer:
    """Q8_0 weights of one layer: heads * dim = hidden."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, ffn: int, seed: int, layer: int, device):
        dim = hidden // heads
        self.shapes = {"qkv": ((heads + 2 * kv_heads) * dim, hidden), "o": (hidden, hidden),
                       "gate_up": (2 * ffn, hidden), "down": (hidden, ffn)}
        self.w = {}
        for p, (name, (M, K)) in enumerate(self.shapes.items()):
            if M % ROW_BLOCK or K % 256:
                raise ValueError("%s: %d x %d is not whole %d-row blocks of 256-element rows" % (name, M, K, ROW_BLOCK))
            rb = q8_row_bytes(K)
            W = torch.empty(M * rb, dtype=torch.uint8, device=device)
            for b in range(M // ROW_BLOCK):
                g = torch.Generator(device=device).manual_seed(block_seed(seed, layer, p, b))
                rows = torch.randn(ROW_BLOCK * K, device=device, generator=g) * K ** -0.5
                W[b * ROW_BLOCK * rb:(b + 1) * ROW_BLOCK * rb] = ane.quantize_q8_0(rows)
            self.w[name] = W


def _normed(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


class Generator:
    """A stack of layers with its cache.  Activations are fp32 rows [n, hidden];
    slots name the cache's sequences."""

    def __init__(self, layers: int, hidden: int = 4096, heads: int = 32, kv_heads: int = 32, ffn: int = 11008,
                 slots: int = 16, pages: int = 1024, page_tokens: int = 16, max_pages: int = 256,
                 dtype=torch.float16, seed: int = 5, device="cuda"):
        self.hidden, self.heads, self.kv_heads, self.dim = hidden, heads, kv_heads, hidden // heads
        self.layers = [Layer(hidden, heads, kv_heads, ffn, seed, i, device) for i in range(layers)]
        self.cache = KVCache.empty(layers, pages, page_tokens, kv_heads, self.dim, slots, max_pages, dtype, device)
        self.dtype, self.device = dtype, device
        self._ws = {}  # by size: the MUL_MATs' and the attention's workspaces

    def _mul_mat(self, layer: Layer, name: str, x):
        M, K = layer.shapes[name]
        if (M, K) not in self._ws:
            self._ws[M, K] = ane.mul_mat_q8_0_batch_workspace(M, K, self.device)
        x = x.contiguous()
        y = torch.empty(x.shape[0], M, device=self.device)
        for r in range(0, x.shape[0], 16):
            ane.mul_mat_q8_0_batch(layer.w[name], x[r:r + 16], M, K, out=y[r:r + 16], workspace=self._ws[M, K],
                                   static_weights=True)
        return y

    def _forward(self, x, slots, cu, granted, attend):
        """cu None: one row per slot.  attend(layer index, q, k, v) -> fp32 [n, heads, dim]."""
        n, kv = x.shape[0], self.kv_heads
        for i, layer in enumerate(self.layers):
            rows = self._mul_mat(layer, "qkv", _normed(x)).to(self.dtype).view(n, self.heads + 2 * kv, self.dim)
            q, k, v = rows[:, :self.heads], rows[:, self.heads:self.heads + kv], rows[:, self.heads + kv:]
            self.cache.write(i, slots, k, v, cu=cu, granted=granted)
            x = x + self._mul_mat(layer, "o", attend(i, q, k, v).view(n, self.hidden))
            gate, up = self._mul_mat(layer, "gate_up", _normed(x)).chunk(2, 1)
            x = x + self._mul_mat(layer, "down", torch.nn.functional.silu(gate) * up)
        return x

    def prompt(self, x, slots, lengths):
        """Prompts packed in x [sum(lengths), hidden] into empty slots (int32
        tensor); returns (every row's output, granted).  A prompt that was not
        granted (no pages left) is not in the cache."""
        cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
        cu[1:] = torch.tensor(lengths, dtype=torch.int32).cumsum(0)
        cu = cu.to(self.device)
        granted = self.cache.reserve(slots, torch.tensor(lengths, dtype=torch.int32, device=self.device))
        out = self._forward(x, slots, cu, granted,
                            lambda i, q, k, v: ane.attn_prompt(q, k, v, cu, out_dtype=torch.float32))
        return out, granted

    def step(self, x, slots, shared: int = 0):
        """One more token (row of x [n, hidden]) for each slot, the first `shared`
        tokens of all of them being the same (forks of one prompt).  Returns
        (output rows, granted); the row of a slot that was not granted is not
        in the cache and its output is to be dropped."""
        n = slots.numel()
        if ("one", n) not in self._ws:
            self._ws["one", n] = torch.ones(n, dtype=torch.int32, device=self.device)
            self._ws["attend", n] = ane.attn_decode_workspace(n, self.heads, self.kv_heads, self.dim, self.device)
        granted = self.cache.reserve(slots, self._ws["one", n])
        out = self._forward(x, slots, None, granted,
                            lambda i, q, k, v: self.cache.attend(i, q, slots, shared=shared, out_dtype=torch.float32,
                                                                 workspace=self._ws["attend", n]))
        return out, granted

    def fork(self, parent: int, children):
        """children (int32 tensor of empty slots) continue from the parent's tokens."""
        return self.cache.fork(torch.full_like(children, parent), children)


def main(argv=None):
    import argparse

    ap = argparse.ArgumentParser(description="fork a prompt into continuations and decode them together")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--children", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args(argv)
    if not 1 <= a.children <= 15:
        ap.error("1 to 15 children")
    if min(a.layers, a.prompt, a.steps) < 1:
        ap.error("at least one layer, one token of the prompt and one step")
    tokens = a.prompt + a.steps
    gen = Generator(a.layers, slots=16, pages=16 * (tokens // 16 + 1), max_pages=tokens // 16 + 1)
    x, granted = gen.prompt(torch.randn(a.prompt, gen.hidden, device="cuda"),
                            torch.zeros(1, dtype=torch.int32, device="cuda"), [a.prompt])
    children = torch.arange(1, a.children + 1, dtype=torch.int32, device="cuda")
    granted = torch.cat([granted, gen.fork(0, children)])
    # the children differ by what they go on from; the prompt's last row is common
    x = x[-1:] + 0.1 * torch.randn(a.children, gen.hidden, device="cuda")
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    shared = a.prompt
    for step in range(a.steps):
        if step <= 1:  # the first step warms up, unless it is the only one
            begin.record()
        x, ok = gen.step(x, children, shared=shared)
    end.record()
    gen.cache.free(children)
    live, _ = gen.cache.compact()
    torch.cuda.synchronize()
    if not bool(granted.all()) or not bool(ok.all()) or not bool(torch.isfinite(x).all()):
        raise SystemExit("the cache ran out of pages or a row is not finite")
    ms = begin.elapsed_time(end) / max(1, a.steps - 1)
    print("%d layers, prompt of %d tokens, %d continuations of %d steps: %.3f ms per step; %d pages stay in use" %
          (a.layers, a.prompt, a.children, a.steps, ms, live.item()))


if __name__ == "__main__":
    main()
