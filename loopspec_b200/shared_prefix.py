"""A batch of requests behind one shared prefix, for a stack of attention layers.

    python -m loopspec_b200.shared_prefix [--requests 16] [--prefix 4000] [--steps 20]

`PrefixBatch` owns the paged K/V and runs a step the way a server does: one
`build_slots` call turns the step's length changes into slots (new tokens,
rejected drafts, released requests), then every layer norms, rotates and
stores its new K/V (`qk_norm_rope`) and attends (`prefix_attention`). The host
passes the changes and an upper bound on them; lengths, blocks and slots stay
on the GPU. A system prompt is prefilled as one request and then shared.

The command prefills a prefix, forks requests with prompts of their own and
decodes with drafts, on random activations, and prints the time of each phase.
"""

from __future__ import annotations

import argparse

import torch

from .prefix_attention import prefix_attention, workspace_bytes
from .qk_norm import qk_norm_rope, rope_table
from .slots import SlotMap, build_slots
from .status import DeviceStatus


class PrefixBatch:
    """n_blocks blocks of page_size slots for up to max_requests requests of
    max_len own positions; a step appends at most max_tokens tokens."""

    def __init__(self, n_layers, n_heads, n_kv_heads, head_dim, *, n_blocks, page_size, max_requests, max_len,
                 max_tokens, max_positions, theta=10000.0, dtype=torch.bfloat16, device="cuda"):
        self.n_heads, self.page_size, self.n_blocks = n_heads, page_size, n_blocks
        width = -(-max_len // page_size)
        self.max_len = width * page_size
        shape = (n_layers, n_blocks * page_size, n_kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.rope = rope_table(max_positions, head_dim, theta, device)
        i32 = {"dtype": torch.int32, "device": device}
        self.table = torch.zeros(max_requests, width, **i32)
        self.lens = torch.zeros(max_requests, **i32)
        self.free_blocks = torch.arange(n_blocks - 1, -1, -1, **i32)      # a stack: block 0 is on top
        self.free_count = torch.tensor([n_blocks], **i32)
        self.map = SlotMap(max_requests, max_tokens, device, lens=self.lens, free_count=self.free_count)
        self.prefix_table, self.prefix_len = None, 0
        self.status = DeviceStatus(device)
        self.workspace = torch.zeros(0, dtype=torch.uint8, device=device)

    def begin(self, delta, n_tokens, max_new):
        """Start a step: delta int32 [max_requests] on the GPU, n_tokens tokens
        in all, at most max_new of one request."""
        self.n_tokens, self.max_new = n_tokens, max_new
        build_slots(self.lens, delta, self.table, self.free_blocks, self.free_count, page_size=self.page_size,
                    n_blocks=self.n_blocks, base=self.prefix_len, out=self.map, status=self.status)

    def attend(self, layer, qkv, q_weight, k_weight, eps=1e-6):
        """The attention output [n_tokens, n_heads, head_dim] of packed projections qkv [n_tokens, width]."""
        n, k, v = self.n_tokens, self.k[layer], self.v[layer]
        q = qk_norm_rope(qkv, q_weight, k_weight, self.rope, self.map.positions[:n], k, v, self.map.slots[:n], eps=eps,
                         status=self.status)
        with torch.cuda.device(k.device):
            need = workspace_bytes(n, self.n_heads, k.shape[1], k.shape[2], n_requests=self.lens.numel(),
                                   prefix_len=self.prefix_len, max_new=self.max_new, max_len=self.max_len)
        if self.workspace.numel() < need:
            self.workspace = torch.empty(need, dtype=torch.uint8, device=k.device)
        return prefix_attention(q, k, v, self.prefix_table, self.prefix_len, self.table, self.lens, self.map.token_start,
                                page_size=self.page_size, max_new=self.max_new, max_len=self.max_len,
                                workspace=self.workspace, status=self.status)

    def share(self, request, length):
        """Make the first `length` positions of `request` the prefix of all, for as long as the batch lives; the
        request is empty afterwards. Waits for the GPU."""
        if self.prefix_len:
            raise ValueError("the batch has a prefix already")
        held = self.lens.tolist()
        if not (0 <= request < len(held) and 0 < length <= held[request]):
            raise ValueError(f"request {request} does not hold {length} positions")
        if sum(held) != held[request]:
            raise ValueError("the other requests must be empty: their keys are rotated for positions from 0 on")
        cut = torch.zeros(len(held), dtype=torch.int32)
        cut[request] = length - held[request]
        self.begin(cut.to(self.lens.device), 0, 0)       # blocks past the prefix go back
        blocks = -(-length // self.page_size)
        self.prefix_table = self.table[request, :blocks].clone()
        self.prefix_len = length
        self.lens[request].zero_()       # its blocks stay out of the free stack

    def check(self):
        """Wait, and raise if a step ran out of blocks or met a bad index."""
        self.status.check()


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--requests", type=int, default=16)
    p.add_argument("--prefix", type=int, default=4000)
    p.add_argument("--prompt", type=int, default=200, help="own prompt of each request, ragged up to this")
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--drafts", type=int, default=4, help="tokens appended a step, all but one rolled back in the next")
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--heads", type=int, default=16)
    p.add_argument("--kv-heads", type=int, default=16)
    p.add_argument("--dim", type=int, default=128)
    p.add_argument("--page", type=int, default=16)
    a = p.parse_args()
    dev, R = "cuda", a.requests
    longest = max(a.prefix, a.prompt + (a.steps + 1) * a.drafts)
    per = -(-longest // a.page)
    batch = PrefixBatch(a.layers, a.heads, a.kv_heads, a.dim, n_blocks=per * (R + 1), page_size=a.page, max_requests=R,
                        max_len=longest, max_tokens=max(a.prefix, R * max(a.prompt, a.drafts)),
                        max_positions=a.prefix + longest, device=dev)
    g = torch.Generator(device=dev).manual_seed(0)
    weights = (1 + 0.1 * torch.randn(a.layers, 2, a.dim, generator=g, device=dev)).to(torch.bfloat16)
    width = (a.heads + 2 * a.kv_heads) * a.dim

    def step(delta):
        new = [max(0, d) for d in delta]
        qkv = torch.randn(a.layers, sum(new), width, generator=g, device=dev).to(torch.bfloat16)
        changes = torch.tensor(delta, dtype=torch.int32, device=dev)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        batch.begin(changes, sum(new), max(new))
        for layer in range(a.layers):
            out = batch.attend(layer, qkv[layer], weights[layer, 0], weights[layer, 1])
        end.record()
        batch.check()
        if not bool(torch.isfinite(out).all()):
            raise AssertionError("an output is not finite")
        return start.elapsed_time(end) / a.layers * 1e3

    def again(delta):                         # the first time loads the kernels: taken back, and once more
        step(delta)
        batch.begin(-torch.tensor(delta, dtype=torch.int32, device=dev), 0, 0)
        return step(delta)

    print(f"prefix of {a.prefix}: {again([a.prefix] + [0] * (R - 1)):.0f} us a layer")
    batch.share(0, a.prefix)
    print(f"{R} prompts of up to {a.prompt}: {again([a.prompt - i * a.prompt // (2 * R) for i in range(R)]):.0f} us a layer")
    times = []
    for _ in range(a.steps):
        times.append(step([a.drafts] * R))
        batch.begin(torch.full((R,), 1 - a.drafts, dtype=torch.int32, device=dev), 0, 0)    # all but one rejected
    print(f"{a.steps} steps of {R} x {a.drafts} drafts: {sorted(times)[len(times) // 2]:.0f} us a layer")


if __name__ == "__main__":
    main()
