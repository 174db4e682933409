"""A captured decode step of a small random-init transformer: append, paged
attention, sampling and log probabilities, as a serving loop would run them.

Each layer normalises its input, projects queries, keys and values, appends the
new token to its paged cache (heads normalised and rotated on the way) and
attends over it; the logits go to the sampler, and the sampled ids to the log
probabilities.  The whole step is one CUDA graph; between replays the host
advances positions and page lists, as a page allocator would.

    python examples/decode_step.py [--steps 8] [--batch 4] [--e4m3]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ecahlang_b200 import PagedAttention                 # noqa: E402
from ecahlang_b200.manager import SamplingManager        # noqa: E402


class DecodeStep:
    """The step's buffers and its graph.  Sizes default to two layers of a
    16-query, 2-KV head model with head_dim 128."""

    def __init__(self, batch: int, *, layers: int = 2, hidden: int = 512, hq: int = 16, hk: int = 2, dim: int = 128,
                 vocab: int = 32000, page: int = 16, max_len: int = 256, dtype=torch.bfloat16, e4m3: bool = False,
                 top_n: int = 5, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g, device="cuda") * rows ** -0.5).to(dtype)

        self.batch, self.page, self.top_n, self.dims = batch, page, top_n, (hq, hk, dim)
        self.embed = (torch.randn(vocab, hidden, generator=g, device="cuda")).to(dtype)
        self.wqkv = [weight(hidden, (hq + 2 * hk) * dim) for _ in range(layers)]
        self.wo = [weight(hq * dim, hidden) for _ in range(layers)]
        self.head = weight(hidden, vocab)
        self.head_norm = torch.ones(dim, dtype=dtype, device="cuda")
        angle = torch.arange(max_len, dtype=torch.float64)[:, None] * \
            1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        self.table = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()

        self.attention = PagedAttention(hq, hk, dim, page, dtype, max_batch=batch,
                                        kv_dtype=torch.float8_e4m3fn if e4m3 else None)
        pages = -(-max_len // page) * batch
        self.caches = [self.attention.new_cache(pages) for _ in range(layers)]
        # pages in the scattered order a pool hands them out
        self.table_of = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(batch, -1)
        self.length = 0

        # what the captured step reads: the tokens, and where they go
        self.ids = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.positions = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.batch_index = torch.arange(batch, dtype=torch.int32, device="cuda")
        self.indptr = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
        self.indices = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.last = torch.zeros(batch, dtype=torch.int32, device="cuda")

        self.manager = SamplingManager(vocab, seq_lens=batch, dtype=dtype, seed=seed)
        self.manager.init_sampling_buffers(batch)
        self.manager.init_cuda_graph_buffers([batch])
        self.manager.fill_cuda_graph_sampling_params(batch, batch, [0.7] * batch, [vocab] * batch, [0.9] * batch)
        self.graph = None

    def forward(self):
        """(logits, sampled ids, their log probabilities) of the next token."""
        hq, hk, dim = self.dims
        x = self.embed[self.ids.long()]
        for wqkv, wo, (k_cache, v_cache, k_scale, v_scale) in zip(self.wqkv, self.wo, self.caches):
            y = torch.nn.functional.rms_norm(x, x.shape[-1:])
            q, k, v = (y @ wqkv).view(self.batch, hq + 2 * hk, dim).split([hq, hk, hk], 1)
            q = self.attention.append(q, k, v, self.positions, self.batch_index, self.indptr, self.indices, k_cache,
                                      v_cache, k_scale=k_scale, v_scale=v_scale, cos_sin=self.table,
                                      q_norm=self.head_norm, k_norm=self.head_norm)
            o = self.attention.decode(q, self.indptr, self.indices, self.last, k_cache, v_cache, k_scale=k_scale,
                                      v_scale=v_scale)
            x = x + o.view(self.batch, -1) @ wo
        logits = torch.nn.functional.rms_norm(x, x.shape[-1:]) @ self.head
        ids = self.manager.sample(logits, bucket_size=self.batch)
        return logits, ids, self.manager.logprobs(logits, ids, self.top_n, bucket_size=self.batch)

    def place(self):
        """The page lists with room for one more token of every request."""
        n = self.length // self.page + 1
        self.indptr.copy_(torch.arange(0, (self.batch + 1) * n, n, dtype=torch.int32))
        self.indices[:self.batch * n] = self.table_of[:, :n].reshape(-1)
        self.positions.fill_(self.length)
        self.last.fill_(self.length % self.page + 1)
        self.length += 1

    def __call__(self, ids: torch.Tensor):
        """One decode step for ``ids`` int32 [batch] on the device."""
        self.ids.copy_(ids)
        self.place()
        if self.graph is None:
            self.forward()                         # warm up (and make the lazy workspaces)
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.out = self.forward()
        self.graph.replay()
        return self.out


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--e4m3", action="store_true", help="keep the cache in 8-bit floats")
    a = ap.parse_args()
    step = DecodeStep(a.batch, e4m3=a.e4m3, max_len=max(64, a.steps + 1))
    ids = torch.arange(1, a.batch + 1, dtype=torch.int32, device="cuda")
    for i in range(a.steps):
        _, ids, lp = step(ids)
        print(f"step {i}: ids {ids.tolist()}  log probabilities {[round(v, 3) for v in lp.logprobs.tolist()]}  "
              f"entropy {[round(v, 2) for v in lp.entropy.tolist()]}")
        print(f"        request 0 alternatives {list(zip(lp.top_ids[0].tolist(), [round(v, 3) for v in lp.top_logprobs[0].tolist()]))}")


if __name__ == "__main__":
    main()
