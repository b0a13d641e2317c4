"""A retrieval model's head from training to filtered answers, on synthetic data.

A query tower and document embeddings are trained on (query features, clicked
document) pairs with the log-probability of the clicked document over all
documents (`target_logprobs`), and a routing layer with the clusters' balance
loss (`cluster_route`).  The embeddings are then packed into 4 bits
(`RetrievalHeadModule`), a bloom index is built over the documents' features,
and filtered queries are answered: the clicked document's log-probability among
the documents that pass, the distribution's entropy and the best alternatives.

    python examples/retrieval_head.py --steps 60
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import silvertorch_amd.ops._load_ops  # noqa: E402,F401  (registers torch.ops.st)
from silvertorch_amd.modules import RetrievalHeadModule  # noqa: E402

DEVICE = "cuda"


def make_data(docs, features, pairs, seed):
    """Documents of 8 topics; a pair's query features are the clicked document's, blurred."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    topics = torch.randint(0, 8, (docs,), generator=g, device=DEVICE)
    content = torch.randn((8, features), generator=g, device=DEVICE)[topics]
    content = content + 0.7 * torch.randn((docs, features), generator=g, device=DEVICE)
    clicked = torch.randint(0, docs, (pairs,), generator=g, device=DEVICE)
    queries = content[clicked] + 0.3 * torch.randn((pairs, features), generator=g, device=DEVICE)
    return topics, content, queries, clicked


def train(content, queries, clicked, dim, clusters, probes, steps, temperature):
    """The trained (query tower, document embeddings, router) and the loss of the first and the last step."""
    torch.manual_seed(0)
    docs, features = content.shape
    tower = torch.nn.Linear(features, dim, device=DEVICE)
    doc_tower = torch.nn.Linear(features, dim, device=DEVICE)
    router = torch.nn.Linear(dim, clusters, device=DEVICE)
    optimiser = torch.optim.Adam([*tower.parameters(), *doc_tower.parameters(), *router.parameters()], lr=3e-2)
    losses = []
    for _ in range(steps):
        q, d = tower(queries), doc_tower(content)
        logprobs, entropy, _, _, _ = torch.ops.st.target_logprobs(q @ d.t(), clicked, 0, None, temperature)
        _, _, lse, counts, balance = torch.ops.st.cluster_route(router(d), probes)
        loss = -logprobs.mean() - 1e-3 * entropy.mean() + 0.1 * balance + 1e-4 * lse.square().mean()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
    return tower, doc_tower(content).detach(), router, losses[0].item(), losses[-1].item()


def answer(tower, embeddings, topics, queries, clicked, topk, temperature):
    """Filtered answers from the packed table: each query may only be given documents of the clicked one's topic."""
    head = RetrievalHeadModule(group_size=32, topk=topk, temperature=temperature)
    head.set_embeddings(embeddings)
    # one feature, id 1, one value per document
    ids = torch.ones(1, dtype=torch.int32, device=DEVICE)
    offsets = torch.arange(topics.numel() + 1, device=DEVICE)
    index, bundle_offsets = torch.ops.st.bloom_index_build(ids, offsets, topics.long(), 5.0, 3)
    expressions = [f"1:{t}" for t in topics[clicked].tolist()]
    _, (plans, plan_offsets) = torch.ops.st.parse_expression_query_batch(
        expressions, torch.ones(1, dtype=torch.long), 7, True, 5)
    mask = torch.ops.st.bloom_index_search_batch(index, bundle_offsets, plans, plan_offsets, 3, 7, False)
    with torch.no_grad():
        return head(tower(queries), clicked, mask), mask


def probed_scores(router, embeddings, queries, tower, clusters, probes):
    """The same documents by the clustered path: the router assigns documents and picks the clusters to score."""
    with torch.no_grad():
        home = torch.ops.st.cluster_route(router(embeddings), 1)[0].flatten()
        order = torch.argsort(home, stable=True)
        sizes = torch.bincount(home, minlength=clusters)
        starts = torch.nn.functional.pad(sizes.cumsum(0), (1, 0))
        chosen = torch.ops.st.cluster_route(router(tower(queries)), probes)[0]
        width = int(sizes.topk(probes)[0].sum())
        scores, at = torch.ops.st.fused_kmean_ann(starts, chosen, sizes[chosen], embeddings[order].contiguous(),
                                                  tower(queries), width)
        ids = torch.where(at >= 0, order[at.clamp(min=0).long()], -1)
    return ids, scores


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--docs", type=int, default=4000)
    ap.add_argument("--pairs", type=int, default=512)
    ap.add_argument("--steps", type=int, default=60)
    a = ap.parse_args(argv)
    temperature, clusters, probes = 0.5, 16, 4
    topics, content, queries, clicked = make_data(a.docs, 48, a.pairs, seed=1)
    tower, embeddings, router, first, last = train(content, queries, clicked, 64, clusters, 2, a.steps, temperature)
    print(f"loss: {first:.3f} at the first step, {last:.3f} at the last")
    (logprobs, entropy, _, top_ids, top_logprobs), mask = answer(tower, embeddings, topics, queries[:8], clicked[:8], 5,
                                                                 temperature)
    for i in range(8):
        best = ", ".join(f"{d} ({p:.2f})" for d, p in zip(top_ids[i].tolist(), top_logprobs[i].tolist()))
        print(f"query {i}: document {clicked[i].item()} has log p {logprobs[i].item():.2f}, entropy "
              f"{entropy[i].item():.2f}; best: {best}")
    ids, scores = probed_scores(router, embeddings, queries[:8], tower, clusters, probes)
    found = (ids == clicked[:8].unsqueeze(1)).any(1).float().mean().item()
    print(f"probing {probes} of {clusters} clusters scores {found:.0%} of the clicked documents")
    return dict(first=first, last=last, logprobs=logprobs, top_ids=top_ids, mask=mask, topics=topics, clicked=clicked[:8],
                ids=ids)


if __name__ == "__main__":
    main()
