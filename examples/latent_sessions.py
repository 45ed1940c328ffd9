"""Sessions of a latent-attention model that mount a graft, read a prompt and
decode, with random weights.

Each session routes its query over the bank of graft keys and mounts the chosen
graft's latents into the latent cache as its first tokens, the key parts turned
to their positions there.  It reads a prompt on top in the expanded form (keys
and values of every head, dense), decodes a few tokens in the absorbed one, and
reads its own turn back, the key parts turned to where a deposit keeps them.

    python examples/latent_sessions.py [--sessions 4] [--prompt 48] [--steps 8]
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from graftrepository_amd import KvBatch, LatentCache, MlaNodeBank, Rotary, attend_rows  # noqa: E402

LAYERS, HEADS, WIDTH, BLOCK = 2, 16, 256, 32
RANK, ROPE, NOPE, VALUE = 256, 32, 64, 64
SCALE = (NOPE + ROPE) ** -0.5


class Layer:
    def __init__(self, weight):
        self.q = weight(WIDTH, HEADS * (NOPE + ROPE))
        self.latent = weight(WIDTH, RANK)
        self.key_part = weight(WIDTH, ROPE)
        # [heads, NOPE + VALUE, RANK]: what a head's own keys and values are made by
        self.up = weight(RANK, HEADS * (NOPE + VALUE)).t().reshape(HEADS, NOPE + VALUE, RANK).contiguous()
        self.up_key = self.up[:, :NOPE].contiguous()
        self.up_value = self.up[:, NOPE:].transpose(1, 2).contiguous()
        self.out = weight(HEADS * VALUE, WIDTH)

    def queries(self, x, rotary, positions):
        q = (x @ self.q).view(-1, HEADS, NOPE + ROPE)
        return rotary.apply(q, positions, start=NOPE)

    def absorb(self, q):
        """Queries in the latents' space, beside their turned part."""
        own = torch.bmm(q[..., :NOPE].transpose(0, 1).contiguous(), self.up_key)
        return torch.cat([own.transpose(0, 1), q[..., NOPE:]], -1)

    def values(self, o):
        """A head's values of mean latents [tokens, heads, RANK]."""
        return torch.bmm(o.transpose(0, 1).contiguous(), self.up_value).transpose(0, 1)

    def add(self, x, o):
        x = x + o.reshape(-1, HEADS * VALUE) @ self.out
        return torch.nn.functional.layer_norm(x.float(), (WIDTH,)).bfloat16()


def run(sessions: int = 4, prompt: int = 48, steps: int = 8, nodes: int = 16, seed: int = 0) -> dict:
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def weight(rows, cols):
        return (torch.randn(rows, cols, generator=gen, device="cuda") / rows ** 0.5).bfloat16()

    layers = [Layer(weight) for _ in range(LAYERS)]
    rotary = Rotary(ROPE)

    # Routing: which graft each session mounts.  A graft's key parts are not turned.
    keys = rng.standard_normal((nodes, 128)).astype(np.float32)
    with MlaNodeBank(keys) as bank:
        chosen = bank.route(keys[rng.permutation(nodes)[:sessions]], 1).ids[:, 0].astype(int)
    sizes = rng.integers(20, 300, nodes)
    lengths = [int(sizes[n]) for n in chosen]
    grafts = [torch.randn(LAYERS, n, RANK + ROPE, generator=gen, device="cuda").bfloat16()
              for n in lengths]

    # One pool of blocks for all sessions; a layer's cache is a pool of its own.
    total = [n + prompt + steps for n in lengths]
    width = -(-max(total) // BLOCK)
    pool = sum(-(-n // BLOCK) for n in total)
    caches = [LatentCache(torch.empty(pool, BLOCK, RANK + ROPE, device="cuda", dtype=torch.bfloat16),
                          RANK) for _ in layers]
    ints = dict(dtype=torch.int32, device="cuda")
    table = torch.full((sessions, width), -1, **ints)
    free = torch.from_numpy(rng.permutation(pool).astype(np.int32)).cuda()
    head = torch.zeros(1, **ints)
    ctx = torch.zeros(sessions, **ints)
    new = torch.tensor(lengths, **ints)

    def batch(tokens, most, taken):
        return KvBatch(ctx, new, table, BLOCK, tokens=tokens, max_new=most, heads=HEADS, kv_heads=1,
                       free_list=free, free_head=taken, latent=True)

    # Mount: the grafts' latents are the sessions' first tokens.
    mount = batch(sum(lengths), max(lengths), head).plan()
    for layer, cache in enumerate(caches):
        rows = torch.cat([g[layer] for g in grafts])
        cache.append(mount, rows[:, :RANK], rows[:, RANK:], rotary=rotary)

    # Prompt, in the expanded form.
    ctx += new
    new.fill_(prompt)
    reading = batch(sessions * prompt, prompt, mount.free_head_out).plan()
    starts = torch.zeros(sessions, **ints)
    rows = sum(lengths) + sessions * prompt
    cu = torch.cat([starts[:1], (ctx + new).cumsum(0)]).int()
    x = weight(sessions * prompt, WIDTH) * (sessions * prompt) ** 0.5
    for layer, cache in zip(layers, caches):
        cache.append(reading, x @ layer.latent, x @ layer.key_part, rotary=rotary)
        k, v = cache.expand(layer.up, NOPE, table, starts, cu, rows)
        q = layer.queries(x, rotary, reading.positions)
        o = attend_rows(reading, q, k, v, cu, softmax_scale=SCALE)
        x = layer.add(x, o)
    read = dict(q=q, k=k, v=v, cu=cu, out=o, ctx=list(lengths))

    # Decode: one token of every session a step, absorbed; lengths, and what was
    # taken from the free list, go on in place.
    x = x.view(sessions, prompt, WIDTH)[:, -1].contiguous()
    ctx += new
    new.fill_(1)
    step = batch(sessions, 1, reading.free_head_out)
    wrote = [[] for _ in layers]
    for i in range(steps):
        if i <= 1:  # the first step loads the libraries' kernels: not timed
            torch.cuda.synchronize()
            began = time.perf_counter()
        step.plan()
        for n, (layer, cache) in enumerate(zip(layers, caches)):
            latent, key_part = x @ layer.latent, x @ layer.key_part
            cache.append(step, latent, key_part, rotary=rotary)
            q = layer.absorb(layer.queries(x, rotary, step.positions))
            mean = cache.attend(step, q, SCALE)
            wrote[n].append(torch.cat([latent, key_part], -1))
            x = layer.add(x, layer.values(mean))
        ctx += 1
        step.advance()
    torch.cuda.synchronize()
    took = time.perf_counter() - began

    # Harvest: every session's decoded turn, dense, its key parts turned back.
    own = ctx - steps
    turn_cu = torch.arange(sessions + 1, **ints) * steps
    positions = (own[:, None] + torch.arange(steps, **ints)).reshape(-1)
    turn = []
    for cache in caches:
        got = cache.read(table, own, turn_cu, sessions * steps, dtype="f32")
        rotary.apply(got.unsqueeze(1), positions, start=RANK, out=got.unsqueeze(1), inverse=True)
        turn.append(got.view(sessions, steps, RANK + ROPE))
    return dict(caches=caches, table=table, ctx=ctx, lengths=lengths, grafts=grafts, rotary=rotary,
                read=read, q=q, out=mean, turn=turn,
                wrote=[torch.stack(w, 1) for w in wrote], ms_per_step=took / max(1, steps - 1) * 1e3)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--sessions", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=48)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    got = run(a.sessions, a.prompt, a.steps)
    print(f"{a.sessions} sessions on grafts of {got['lengths']} tokens, prompts of {a.prompt}, "
          f"{a.steps} steps: {got['ms_per_step']:.3f} ms a step; turn {tuple(got['turn'][0].shape)} "
          "a layer")


if __name__ == "__main__":
    main()
