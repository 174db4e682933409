"""Serving several new tokens a request: a prompt is prefilled, forked into
choices that share its pages, and each choice goes on by verified drafts.

The prompt's tokens go through the layers at once (append, then prefill
attention over the paged cache).  The choices list the prompt's whole pages
and get copies of its last, partly filled one, in all layers by one launch.
Each step looks a draft up in what a choice has so far, runs the model over
the choice's last token and its drafts, and keeps the drafts that leave the
output distributed as the model's own samples; the cache slots of refused
drafts are written again.  The step is one CUDA graph.

    python examples/draft_step.py [--steps 8] [--choices 3] [--drafts 4] [--e4m3]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ecahlang_b200 import PagedAttention                 # noqa: E402
from ecahlang_b200.manager import SamplingManager        # noqa: E402


class DraftStep:
    """A small random-init transformer, its pages and its captured step."""

    def __init__(self, choices: int, drafts: int = 4, *, layers: int = 2, hidden: int = 512, hq: int = 16, hk: int = 2,
                 dim: int = 128, vocab: int = 2000, page: int = 16, max_len: int = 256, dtype=torch.bfloat16,
                 e4m3: bool = False, temperature: float = 0.7, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g, device="cuda") * rows ** -0.5).to(dtype)

        self.choices, self.drafts, self.page, self.vocab, self.dims = choices, drafts, page, vocab, (hq, hk, dim)
        self.embed = torch.randn(vocab, hidden, generator=g, device="cuda").to(dtype)
        self.wqkv = [weight(hidden, (hq + 2 * hk) * dim) for _ in range(layers)]
        self.wo = [weight(hq * dim, hidden) for _ in range(layers)]
        self.head = weight(hidden, vocab)
        self.head_norm = torch.ones(dim, dtype=dtype, device="cuda")
        angle = torch.arange(max_len + drafts + 1, dtype=torch.float64)[:, None] * \
            1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        self.table = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        self.attention = PagedAttention(hq, hk, dim, page, dtype, max_batch=choices,
                                        kv_dtype=torch.float8_e4m3fn if e4m3 else None)
        a_request = -(-(max_len + drafts + 1) // page)
        self.caches = [self.attention.new_cache(a_request * (choices + 1)) for _ in range(layers)]
        # a pool in the scattered order that requests come and go in
        self.pool = torch.randperm(a_request * (choices + 1), generator=g, device="cuda").tolist()
        self.pages, self.tokens = [], []                     # of each choice: its page list, its tokens

        # what the captured step reads
        n = choices * (drafts + 1)
        self.ids = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.positions = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.batch_index = torch.arange(choices, dtype=torch.int32, device="cuda").repeat_interleave(drafts + 1)
        self.qo_indptr = torch.arange(0, n + 1, drafts + 1, dtype=torch.int32, device="cuda")
        self.indptr = torch.zeros(choices + 1, dtype=torch.int32, device="cuda")
        self.indices = torch.zeros(a_request * choices, dtype=torch.int32, device="cuda")
        self.last = torch.zeros(choices, dtype=torch.int32, device="cuda")
        self.draft_ids = torch.zeros(choices, drafts, dtype=torch.int32, device="cuda")
        self.num_drafts = torch.zeros(choices, dtype=torch.int32, device="cuda")
        self.manager = SamplingManager(vocab, seq_lens=choices, dtype=dtype, seed=seed)
        self.manager.init_sampling_buffers(choices)
        self.manager.init_cuda_graph_buffers([choices])
        self.manager.init_draft_buffers(choices, drafts)
        self.manager.fill_cuda_graph_sampling_params(choices, choices, [temperature] * choices, [vocab] * choices, [0.9] * choices)
        self.graph = None

    def layers(self, ids, positions, batch_index, qo_indptr, indptr, indices, last):
        """Logits of every token of ``ids``, whose keys and values go to the cache."""
        hq, hk, dim = self.dims
        x = self.embed[ids.long()]
        for wqkv, wo, (k_cache, v_cache, k_scale, v_scale) in zip(self.wqkv, self.wo, self.caches):
            y = torch.nn.functional.rms_norm(x, x.shape[-1:])
            q, k, v = (y @ wqkv).view(-1, hq + 2 * hk, dim).split([hq, hk, hk], 1)
            q = self.attention.append(q, k, v, positions, batch_index, indptr, indices, k_cache, v_cache, k_scale=k_scale,
                                      v_scale=v_scale, cos_sin=self.table, q_norm=self.head_norm, k_norm=self.head_norm)
            o = self.attention.prefill(q, qo_indptr, indptr, indices, last, k_cache, v_cache, k_scale=k_scale, v_scale=v_scale)
            x = x + o.view(x.shape[0], -1) @ wo
        return torch.nn.functional.rms_norm(x, x.shape[-1:]) @ self.head

    def prefill(self, prompt):
        """Runs the prompt and forks it into the choices; the prompt's logits."""
        n, page = len(prompt), self.page
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
        owned = [self.pool.pop() for _ in range(-(-n // page))]
        logits = self.layers(ints(prompt), ints(range(n)), ints([0] * n), ints([0, n]), ints([0, len(owned)]), ints(owned),
                             ints([(n - 1) % page + 1]))
        whole, rest = n // page, n % page
        self.pages = [owned[:whole] for _ in range(self.choices)]
        if rest:                                             # the first choice takes the last page itself
            own = [owned[whole]] + [self.pool.pop() for _ in range(self.choices - 1)]
            self.attention.copy_pages([owned[whole]] * (self.choices - 1), own[1:], self.caches,
                                      tokens=[rest] * (self.choices - 1))
            self.pages = [p + [o] for p, o in zip(self.pages, own)]
        self.tokens = [list(prompt) for _ in range(self.choices)]
        return logits

    def look_up(self, tokens):
        """What followed the latest earlier place of the last two tokens."""
        for at in range(len(tokens) - 3, -1, -1):
            if tokens[at:at + 2] == tokens[-2:]:
                return tokens[at + 2:at + 2 + self.drafts]
        return []

    def run(self):
        self.logits = self.layers(self.ids, self.positions, self.batch_index, self.qo_indptr, self.indptr, self.indices, self.last)
        return self.manager.verify_drafts(self.logits, self.draft_ids, num_drafts=self.num_drafts, bucket_size=self.choices)

    def __call__(self, drafts=None):
        """One step of every choice: its tokens so far but the last are cached.
        ``drafts``: lists of tokens (None: looked up)."""
        drafts = [self.look_up(t) for t in self.tokens] if drafts is None else drafts
        ids, positions, lists = [], [], []
        for own, tokens, draft in zip(self.pages, self.tokens, drafts):
            n = len(tokens)
            ids += [tokens[-1]] + draft + [0] * (self.drafts - len(draft))
            positions += range(n - 1, n + self.drafts)
            while len(own) * self.page < n + self.drafts:
                own.append(self.pool.pop())
            lists.append(own[:-(-(n + self.drafts) // self.page)])
        self.ids.copy_(torch.tensor(ids))
        self.positions.copy_(torch.tensor(positions))
        self.indptr.copy_(torch.tensor([0] + [len(p) for p in lists]).cumsum(0))
        self.indices[:sum(len(p) for p in lists)] = torch.tensor(sum(lists, []), dtype=torch.int32)
        self.last.copy_(torch.tensor([(len(t) + self.drafts - 1) % self.page + 1 for t in self.tokens]))
        self.draft_ids.copy_(torch.tensor([d + [0] * (self.drafts - len(d)) for d in drafts]))
        self.num_drafts.copy_(torch.tensor([len(d) for d in drafts]))
        if self.graph is None:
            self.run()                                       # warm up
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.out = self.run()
        self.graph.replay()
        new, kept = self.out.tokens.tolist(), self.out.accepted.tolist()
        for tokens, row, n in zip(self.tokens, new, kept):
            tokens += row[:n + 1]
        return self.out


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--choices", type=int, default=3)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--e4m3", action="store_true", help="keep the cache in 8-bit floats")
    a = ap.parse_args()
    step = DraftStep(a.choices, a.drafts, e4m3=a.e4m3, max_len=64 + a.steps * (a.drafts + 1), temperature=0.2)
    step.prefill([7, 11, 13, 17] * 9 + [7, 11])
    for i in range(a.steps):
        out = step()
        print(f"step {i}: kept {out.accepted.tolist()}, tokens {[t[-n - 1:] for t, n in zip(step.tokens, out.accepted.tolist())]}")


if __name__ == "__main__":
    main()
