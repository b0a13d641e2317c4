"""A query tower from training to answers in 8 bits, on synthetic data.

A tower of layer norm, feed-forward layers and dropout (`QueryTowerModule`) is
trained against fixed document embeddings with the log-probability of the
clicked document (`target_logprobs`).  Its weights are then packed into 8 bits
(`PackedQueryTowerModule`), and so are the documents (`RetrievalHeadModule`), and
queries are answered from the packed forms.

    python examples/query_tower.py --steps 100
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from silvertorch_amd.modules import PackedQueryTowerModule, QueryTowerModule, RetrievalHeadModule  # noqa: E402

DEVICE = "cuda"


def make_data(docs, dim, features, pairs, seed):
    """Document embeddings; a pair's query features are a fixed map of the clicked document's embedding, blurred."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    documents = torch.randn((docs, dim), generator=g, device=DEVICE)
    clicked = torch.randint(0, docs, (pairs,), generator=g, device=DEVICE)
    mixed = torch.randn((dim, features), generator=g, device=DEVICE) * dim ** -0.5
    queries = torch.tanh(documents[clicked] @ mixed) + 0.1 * torch.randn((pairs, features), generator=g, device=DEVICE)
    return documents, queries, clicked


def loss_of(tower, documents, queries, clicked, temperature):
    """Mean negative log-probability of the clicked documents among all."""
    logprobs = torch.ops.st.target_logprobs(tower(queries) @ documents.t(), clicked, 0, None, temperature)[0]
    return -logprobs.mean()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--docs", type=int, default=5000)
    ap.add_argument("--pairs", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=100)
    a = ap.parse_args(argv)
    temperature = 0.5
    documents, queries, clicked = make_data(a.docs, 64, 96, a.pairs, seed=1)
    torch.manual_seed(0)
    tower = QueryTowerModule(96, 64, 128, layers=2, dropout=0.1).to(DEVICE)
    optimiser = torch.optim.AdamW(tower.parameters(), lr=2e-3)
    losses = []
    for _ in range(a.steps):
        loss = loss_of(tower, documents, queries, clicked, temperature)
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
    print(f"loss: {losses[0].item():.3f} at the first step, {losses[-1].item():.3f} at the last")
    tower.eval()
    packed = PackedQueryTowerModule(tower)
    head = RetrievalHeadModule(topk=5, temperature=temperature, bits=8)
    head.set_embeddings(documents)
    with torch.no_grad():
        logprobs, entropy, _, top_ids, top_logprobs = head(packed(queries[:8]), clicked[:8])
        exact = torch.ops.st.target_logprobs(tower(queries[:8]) @ documents.t(), clicked[:8], 5, None, temperature)
    for i in range(8):
        best = ", ".join(f"{d} ({p:.2f})" for d, p in zip(top_ids[i].tolist(), top_logprobs[i].tolist()))
        print(f"query {i}: document {clicked[i].item()} has log p {logprobs[i].item():.2f} in 8 bits, "
              f"{exact[0][i].item():.2f} in 32; entropy {entropy[i].item():.2f}; best: {best}")
    return dict(tower=tower, documents=documents, queries=queries, clicked=clicked, logprobs=logprobs, top_ids=top_ids)


if __name__ == "__main__":
    main()
