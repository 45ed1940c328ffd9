"""Sessions that mount a graft and decode on it, with random weights.

Each session routes its query over the bank of graft keys, unpacks the chosen
node's packed payload on the device, mounts it into the 8-bit paged cache as
its first tokens (a prompt without a prefill), decodes a few tokens on top,
and reads its own turn back as the dense values that a deposit packs.

    python examples/mounted_sessions.py [--sessions 4] [--steps 8]
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from graftrepository_amd import KvBatch, KvCache, MlaNodeBank  # noqa: E402
from graftrepository_amd.payload import FORMAT_VERSION, unpack_node_device  # noqa: E402

LAYERS, HEADS, KV_HEADS, DIM, BLOCK = 2, 8, 2, 64, 32
WIDTH = HEADS * DIM
GROUP = 32                                   # codes to a scale in a payload


def make_node(rng, tokens: int) -> dict[str, np.ndarray]:
    """A packed node: codes and scales of K and V [layers, kv_heads, tokens, dim]."""
    node = dict(format_version=FORMAT_VERSION, storage_bits=8, group_size=GROUP)
    for name in ("k", "v"):
        x = rng.standard_normal((LAYERS, KV_HEADS, tokens, DIM // GROUP, GROUP))
        scale = np.abs(x).max(-1, keepdims=True).astype(np.float32) / 127
        node[name + "_codes"] = np.rint(x / scale).astype(np.int8)
        node[name + "_scales"] = scale
        node[name + "_shape"] = np.array([LAYERS, KV_HEADS, tokens, DIM])
    return node


def unpack(node) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V, fp16 [layers, kv_heads, tokens, dim] on the device."""
    got = unpack_node_device(node)
    return tuple(torch.as_tensor(got[name], device="cuda") for name in ("k", "v"))


def run(sessions: int = 4, steps: int = 8, nodes: int = 16, seed: int = 0) -> dict:
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def weight(rows, cols):
        return (torch.randn(rows, cols, generator=gen, device="cuda") / rows ** 0.5).bfloat16()

    # Routing: which graft each session mounts.
    keys = rng.standard_normal((nodes, 128)).astype(np.float32)
    store = [make_node(rng, int(rng.integers(20, 300))) for _ in range(nodes)]
    with MlaNodeBank(keys) as bank:
        chosen = bank.route(keys[rng.permutation(nodes)[:sessions]], 1).ids[:, 0].astype(int)
    grafts = [unpack(store[n]) for n in chosen]
    lengths = [k.shape[2] for k, _ in grafts]

    # One pool of blocks for all sessions; a layer's cache is a pool of its own.
    total = [n + steps for n in lengths]
    width = -(-max(total) // BLOCK)
    pool = sum(-(-n // BLOCK) for n in total)
    caches = [KvCache.empty(pool, BLOCK, KV_HEADS, DIM) for _ in range(LAYERS)]
    ints = dict(dtype=torch.int32, device="cuda")
    table = torch.full((sessions, width), -1, **ints)
    free = torch.from_numpy(rng.permutation(pool).astype(np.int32)).cuda()
    head = torch.zeros(1, **ints)
    ctx = torch.zeros(sessions, **ints)
    new = torch.tensor(lengths, **ints)

    # Mount: the grafts' keys and values are the sessions' first tokens.
    mount = KvBatch(ctx, new, table, BLOCK, tokens=sum(lengths), max_new=max(lengths),
                    heads=HEADS, kv_heads=KV_HEADS, free_list=free, free_head=head).plan()
    for layer, cache in enumerate(caches):
        k, v = (torch.cat([g[i][layer].transpose(0, 1) for g in grafts]) for i in (0, 1))
        cache.append(mount, k, v)

    # Decode: one token of every session a step; the lengths, and what was
    # taken from the free list, go on in place.
    ctx += new
    new.fill_(1)
    step = KvBatch(ctx, new, table, BLOCK, tokens=sessions, max_new=1, heads=HEADS,
                   kv_heads=KV_HEADS, free_list=free, free_head=mount.free_head_out)
    wq = [weight(WIDTH, WIDTH) for _ in caches]
    wk = [weight(WIDTH, KV_HEADS * DIM) for _ in caches]
    wv = [weight(WIDTH, KV_HEADS * DIM) for _ in caches]
    wo = [weight(WIDTH, WIDTH) for _ in caches]
    x = weight(WIDTH, sessions).t().contiguous() * WIDTH ** 0.5
    for i in range(steps):
        if i <= 1:  # the first step loads the libraries' kernels: not timed
            torch.cuda.synchronize()
            began = time.perf_counter()
        step.plan()
        for layer, cache in enumerate(caches):
            q = (x @ wq[layer]).view(sessions, HEADS, DIM)
            k = (x @ wk[layer]).view(sessions, KV_HEADS, DIM)
            v = (x @ wv[layer]).view(sessions, KV_HEADS, DIM)
            cache.append(step, k, v)
            out = cache.attend(step, q)
            x = torch.nn.functional.layer_norm(
                (x + out.view(sessions, WIDTH) @ wo[layer]).float(), (WIDTH,)).bfloat16()
        ctx += 1
        step.advance()
    torch.cuda.synchronize()
    took = time.perf_counter() - began

    # Harvest: every session's own turn, dense, to be packed as a new node.
    starts = torch.tensor(lengths, **ints)
    rows = torch.arange(sessions + 1, **ints) * steps
    turn = [cache.read(table, starts, rows, sessions * steps) for cache in caches]
    return dict(caches=caches, table=table, ctx=ctx, lengths=lengths, grafts=grafts, q=q, out=out,
                turn=turn, ms_per_step=took / max(1, steps - 1) * 1e3)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--sessions", type=int, default=4)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    got = run(a.sessions, a.steps)
    print(f"{a.sessions} sessions on grafts of {got['lengths']} tokens, {a.steps} steps: "
          f"{got['ms_per_step']:.3f} ms a step; turn {tuple(got['turn'][0][0].shape)} a layer")


if __name__ == "__main__":
    main()
