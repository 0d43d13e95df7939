"""Fit an existing index to queries of another embedding model.

The base vectors and the index stay as they are.  The queries come from a model
whose space is shifted against the base's, so their nearest base vectors are
often the wrong ones; labelled (preferred, rejected) documents train a
QueryAdapter, and the adapted queries are searched as usual:

    python examples/train_query_adapter.py
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from fusiongpu_b200 import IVFPQIndex, QueryAdapter, SearchParams  # noqa: E402


def hit_rate(index, queries, wanted, params) -> float:
    """Share of queries whose labelled document is among the results."""
    ids, _ = index.search(queries.float(), params)
    return float((ids == wanted[:, None]).any(1).float().mean())


def run(nbase=20000, dim=128, nq=2048, nlist=128, pq_m=32, hidden=256, steps=150, negatives=16, seed=0, verbose=True):
    """Returns the hit rate on held-out queries before and after training."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.nn.functional.normalize(torch.randn(nbase, dim, generator=g, device="cuda"), dim=1)
    index = IVFPQIndex.build(base, nlist, pq_m, kmeans_iters=8, pq_sample=min(nbase, 20000), seed=seed)
    # the other model: each query is its document's vector, moved by one fixed map
    warp = torch.eye(dim, device="cuda") + 3.0 * torch.randn(dim, dim, generator=g, device="cuda") / dim ** 0.5
    label = torch.randint(0, nbase, (2 * nq,), generator=g, device="cuda", dtype=torch.int32)
    noise = 0.3 * torch.randn(2 * nq, dim, generator=g, device="cuda") / dim ** 0.5
    queries = torch.nn.functional.normalize((base[label.long()] + noise) @ warp, dim=1)
    train, test = slice(0, nq), slice(nq, 2 * nq)
    params = SearchParams(top_m=min(16, nlist), p1_lists=min(16, nlist), limit_k=50, rerank_m=200, final_k=10,
                          ref_compat=False)
    before = hit_rate(index, queries[test], label[test], params)

    adapter = QueryAdapter(dim, hidden, seed=seed)
    opt = torch.optim.Adam(adapter.parameters(), lr=3e-3)
    offsets = torch.arange(nq + 1, device="cuda") * negatives
    pos = label[train].repeat_interleave(negatives)
    for step in range(steps):
        # rejected documents: half what the search now returns in the label's place, half any document
        ids, _ = index.search(adapter(queries[train]).float(), params.replace(final_k=negatives // 2))
        rand = torch.randint(0, nbase, (nq, negatives - negatives // 2), generator=g, device="cuda",
                             dtype=torch.int32)
        neg = torch.cat([ids, rand], dim=1).reshape(-1)
        neg = torch.where(neg == pos, -1, neg).contiguous()  # the label itself is no rejected document: masked
        losses, _ = adapter.train_step(queries[train], base, offsets, pos, neg, beta=8.0, metric="l2",
                                       weights=torch.full_like(neg, 1.0 / neg.numel(), dtype=torch.float32))
        opt.step()
        if verbose and step % 25 == 0:
            print(f"step {step:4d}  loss {float(losses.mean()):.4f}")
    after = hit_rate(index, adapter(queries[test]), label[test], params)
    if verbose:
        print(f"hit rate at 10 on held-out queries: {before:.3f} -> {after:.3f}")
    return before, after


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=150)
    run(steps=ap.parse_args().steps)
