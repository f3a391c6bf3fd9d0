"""A small lfm2moe-shaped decoder on the library: ragged prompts at once, then single tokens.

A layer, over the fp32 residual x [tokens, D]:

    x, xb  = add_rmsnorm(x)                            RMSNorm, bf16 rows for the projection
    q      = append(cache, q, k, v)                    per-head norms, rotation, keys and values into 4-bit pages
    out    = attend(cache, q)                          attention over the pages
    x      = add_rmsnorm(x, out Wo)                    the residual addition alone
    x     += MoE(x)                                    the library's MoE FFN (RMSNorm, router, experts)

The projections are torch matrix products.  Weights and token rows are seeded random numbers.

    python examples/attention_block.py [--layers 4] [--prompts 300,41,128] [--steps 32]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from laii_b200 import synth  # noqa: E402
from laii_b200.attn import GpuAttn, KVBatch, KVPages, Rope  # noqa: E402
from laii_b200.moe import GpuMoE  # noqa: E402


class Decoder:
    """`layers` layers for up to `n_seqs` sequences of `max_tokens` tokens on the current device."""

    def __init__(self, layers=4, D=2048, heads=32, kv_heads=8, dim=64, E=32, K=4, I=1792, n_seqs=4, max_tokens=1024, page=64):
        self.D, self.heads, self.kv_heads, self.dim, self.page = D, heads, kv_heads, dim, page
        self.moe = GpuMoE(torch.cuda.current_device())
        self.attn = GpuAttn(self.moe)
        g = torch.Generator().manual_seed(1)
        rand = lambda *shape: (torch.randn(*shape, generator=g) * shape[0] ** -0.5).bfloat16().cuda()  # noqa: E731
        self.qkv = [rand(D, (heads + 2 * kv_heads) * dim) for _ in range(layers)]
        self.wo = [rand(heads * dim, D) for _ in range(layers)]
        self.norm = [torch.ones(D, device="cuda") for _ in range(layers)]
        angle = torch.arange(max_tokens)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2) / dim)
        ones = torch.ones(dim, device="cuda")
        self.rope = Rope(angle.cos().float().cuda(), angle.sin().float().cuda(), q_norm=ones, k_norm=ones)
        for l in range(layers):
            self.moe.synth_layer(l, D, E, K, I, [synth.layer_seed(s, l) for s in (
                synth.SEED_GATE, synth.SEED_UP, synth.SEED_DOWN, synth.SEED_ROUTER, synth.SEED_BIAS)])
        # pages are handed out as sequences grow; one table serves all layers, each layer has a pool of its own
        entries = -(-max_tokens // page)
        self.pools = [KVPages.empty(n_seqs * entries, page, kv_heads, dim) for _ in range(layers)]
        self.free = list(range(n_seqs * entries))
        self.table = torch.full((n_seqs, entries), -1, dtype=torch.int32)
        self.lens = [0] * n_seqs

    def forward(self, x, counts):
        """The next counts[b] tokens of each sequence b: rows x [sum(counts), D] fp32 -> the last layer's rows."""
        starts = [0]
        for b, n in enumerate(counts):
            have = -(-self.lens[b] // self.page)
            self.lens[b] += n
            for i in range(have, -(-self.lens[b] // self.page)):
                self.table[b, i] = self.free.pop()
            starts.append(starts[-1] + n)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        batch = KVBatch(i32(starts), i32(self.lens), self.table.cuda(), max(self.lens))
        T, H, G, d = x.shape[0], self.heads, self.kv_heads, self.dim
        stream = torch.cuda.current_stream().cuda_stream
        for l, cache in enumerate(self.pools):
            x, xb, _ = self.attn.add_rmsnorm(x, None, self.norm[l], xb_dtype=torch.bfloat16, q8=False)
            q, k, v = (xb @ self.qkv[l]).view(T, H + 2 * G, d).split((H, G, G), 1)
            q = self.attn.append(cache, batch, q, k, v, self.rope)
            out = self.attn.attend(cache, batch, q)
            x, _, _ = self.attn.add_rmsnorm(x, out.view(T, H * d) @ self.wo[l], None, x_out=x, q8=False)
            self.moe.forward_device(l, x.data_ptr(), T, stream)
        return x

    def close(self):
        self.moe.sync()  # reports what a kernel found out of range
        self.moe.close()


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--prompts", default="300,41,128", help="tokens of each sequence's prompt")
    p.add_argument("--steps", type=int, default=32, help="single tokens of each sequence after them")
    a = p.parse_args(argv)
    prompts = [int(n) for n in a.prompts.split(",")]
    m = Decoder(a.layers, n_seqs=len(prompts), max_tokens=max(prompts) + a.steps)
    g = torch.Generator().manual_seed(2)
    rows = [torch.randn(n + a.steps, m.D, generator=g).cuda() for n in prompts]
    a0, a1, a2 = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    a0.record()
    m.forward(torch.cat([r[:n] for r, n in zip(rows, prompts)]), prompts)
    a1.record()
    last = None
    for i in range(a.steps):
        last = m.forward(torch.stack([r[n + i] for r, n in zip(rows, prompts)]), [1] * len(prompts))
    a2.record()
    m.close()
    print(f"{sum(prompts)} prompt tokens of {len(prompts)} sequences: {a0.elapsed_time(a1):.2f} ms (first call); "
          f"{a.steps} steps of single tokens: {a1.elapsed_time(a2) / max(1, a.steps):.3f} ms each")

    # the same tokens at once: the cache holds the same codes, the rows differ by the projections' rounding
    w = Decoder(a.layers, n_seqs=len(prompts), max_tokens=max(prompts) + a.steps)
    counts = [n + a.steps for n in prompts]
    whole = w.forward(torch.cat(rows), counts)
    ends = torch.tensor(counts).cumsum(0) - 1
    w.close()
    if last is None:
        return 0.0
    err = ((last - whole[ends.cuda()]).norm() / whole[ends.cuda()].norm()).item()
    print(f"last rows, token by token against all at once: relative L2 difference {err:.1e}")
    return err


if __name__ == "__main__":
    main()
