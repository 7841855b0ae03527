"""A stored prefix served from the paged cache, end to end on one GPU.

The prefix's K and V come back from host memory through the authenticated
reload into pages taken from the free slots; a prompt chunk is appended and
attended to over them; the sequence is forked into samples that share the
prefix's pages and decode a token a step; one sample ends, its pages are
cleared, and the cache is compacted; the kept sequence's pages go back to host
memory sealed.  The model is a stand-in: random q, k and v per token.

    python examples/serve_prefix.py [--layers 4 --prefix 700 --samples 3 --steps 5]
"""
from __future__ import annotations

import argparse
import os
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import secure_infer_amd as si  # noqa: E402

TOKENS = 128  # of a page, the transfers' block


class Server:
    """One model's paged caches and its sequences' pages, on the device."""

    def __init__(self, layers: int, heads: int, dim: int, slots: int, rows: int, pages: int):
        dev = "cuda"
        self.layers = [tuple(torch.zeros((slots, TOKENS, heads, dim), dtype=torch.bfloat16, device=dev)
                             for _ in range(2)) for _ in range(layers)]
        self.caches = si.CacheSet([c for pair in self.layers for c in pair])
        self.tables = torch.full((rows, pages), -1, dtype=torch.int64, device=dev)
        self.kv_lens = torch.zeros(rows, dtype=torch.int64, device=dev)
        self.refs = torch.zeros(slots, dtype=torch.int32, device=dev)
        self.unserved = torch.zeros(1, dtype=torch.int32, device=dev)

    def reserve(self, counts) -> None:
        self.tables, self.kv_lens, self.refs = si.reserve_pages(
            self.tables, self.kv_lens, self.refs, torch.tensor(counts, device="cuda"), TOKENS, self.unserved)

    def fork(self, parent: int, children) -> None:
        pairs = torch.tensor([(parent, c) for c in children], dtype=torch.int64, device="cuda").reshape(-1, 2)
        self.tables, self.kv_lens, self.refs = si.fork_pages(self.caches, self.tables, self.kv_lens, self.refs, pairs,
                                                             self.unserved)

    def free(self, rows) -> None:
        self.tables, self.kv_lens, self.refs = si.free_pages(
            self.caches, self.tables, self.kv_lens, self.refs, torch.tensor(rows, device="cuda"),
            fail_count=self.unserved)

    def compact(self) -> None:
        self.tables, self.refs = si.compact_pages(self.caches, self.tables, self.refs, scrub=True)

    def attend(self, layer: int, q, k, v, rows, counts):
        """New tokens of `rows` (counts[i] of row rows[i], already reserved): their K
        and V into the pages, and their attention."""
        k_cache, v_cache = self.layers[layer]
        r = torch.tensor(rows, device="cuda")
        starts = torch.tensor([0, *counts], device="cuda").cumsum(0)
        tables, kv_lens = self.tables[r], self.kv_lens[r]
        si.paged_append(k, v, k_cache, v_cache, tables, kv_lens, q_starts=starts, fail_count=self.unserved)
        return si.paged_attention(q, k_cache, v_cache, tables, kv_lens, q_starts=starts)

    def slots_of(self, row: int) -> torch.Tensor:
        """The row's slots on the host, as the transfers' mappings want them."""
        t = self.tables[row].cpu()
        return t[t >= 0]


def serve(layers=4, q_heads=8, heads=2, dim=128, prefix=700, chunk=45, samples=3, steps=5, seed=0):
    """Runs the whole path; returns the server, every (layer, row, K, V, q, out) step
    in order, the stored prefix and the pools written back, for a caller that
    checks them."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)

    blocks = -(-prefix // TOKENS)
    slots = 4 * blocks + 8 * samples
    srv = Server(layers, heads, dim, slots, samples + 1, blocks + 8)
    stored = [tuple(rand(blocks, TOKENS, heads, dim).cpu().pin_memory() for _ in range(2)) for _ in range(layers)]
    for layer, pools in enumerate(stored):
        for kind, pool in enumerate(pools):
            si.register_host_range(pool, layer, kind)
    session = si.GcmSession(os.urandom(16), os.urandom(4), max_record_bytes=TOKENS * heads * dim * 2)
    shape = si.LayerShape(heads, dim)
    log = []

    # the prefix: pages, then the authenticated reload into them
    srv.reserve([prefix] + [0] * samples)
    mapping = torch.stack([torch.arange(blocks), srv.slots_of(0)], 1)
    transfer = si.NativeTransfer(session, shape)
    transfer.reload_layers([(pools, mapping) for pools in stored], srv.layers)
    for layer in range(layers):
        if transfer.wait_layer(layer) != 0:
            raise RuntimeError(f"layer {layer}: the stored prefix did not authenticate")

    def step(rows, counts):
        add = [0] * (samples + 1)
        for r, n in zip(rows, counts):
            add[r] = n
        srv.reserve(add)
        for layer in range(layers):
            k, v, q = rand(sum(counts), heads, dim), rand(sum(counts), heads, dim), rand(sum(counts), q_heads, dim)
            out = srv.attend(layer, q, k, v, rows, counts)
            at = 0
            for r, n in zip(rows, counts):
                log.append((layer, r, k[at:at + n], v[at:at + n], q[at:at + n], out[at:at + n]))
                at += n

    step([0], [chunk])                         # the prompt's own tokens
    srv.fork(0, range(1, samples + 1))         # samples share the pages
    log.append(("fork", 0, list(range(1, samples + 1))))
    rows = list(range(samples + 1))
    for i in range(steps):
        step(rows, [1] * len(rows))
        if i == steps // 2 and samples:        # one sample ends
            srv.free([rows.pop()])
            srv.compact()

    # the first sequence goes back to the host, sealed on the device
    kept = srv.slots_of(0)
    back = [tuple(torch.zeros((len(kept), TOKENS, heads, dim), dtype=torch.bfloat16).pin_memory() for _ in range(2))
            for _ in range(layers)]
    for layer, pools in enumerate(back):
        for kind, pool in enumerate(pools):
            si.register_host_range(pool, layer, kind)
    si.D2HTransfer(session, shape).store(srv.layers, back, torch.stack([kept, torch.arange(len(kept))], 1))
    torch.cuda.synchronize()
    si.clear_host_ranges()
    session.close()
    if int(srv.unserved):
        raise RuntimeError(f"{int(srv.unserved)} rows or tokens found no page")
    return srv, log, stored, back


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n", 1)[0])
    for name, value in (("layers", 4), ("prefix", 700), ("samples", 3), ("steps", 5)):
        p.add_argument(f"--{name}", type=int, default=value)
    a = p.parse_args()
    srv, log, _, back = serve(layers=a.layers, prefix=a.prefix, samples=a.samples, steps=a.steps)
    lens = srv.kv_lens.tolist()
    print(f"{a.layers} layers; sequence lengths {lens}; {int((srv.refs > 0).sum())} pages held, "
          f"{int((srv.refs > 1).sum())} of them shared; {len(back[0][0])} pages of sequence 0 written back")


if __name__ == "__main__":
    main()
