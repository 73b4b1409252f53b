"""A small retrieval-augmented reader, from the vectors to a training step.

  1. an encoder layer (self-attention with a two-sided position bias) makes the states of a bank of ragged passages, and each
     passage's vector, the mean of its states
  2. the vectors are encoded (PQ) and searched: the ids of the passages nearest to each query, left in device memory
  3. new tokens attend to the states of what was found, through the search's own records
  4. a few training steps of the reader's projection and of its position bias, with gradients through both

Everything is synthetic and seeded. Run it on the GPU: python examples/answer_from_search.py
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import veckern_amd as vk
from veckern_amd import attention, host

HEADS, KV_HEADS, D, WIDTH = 8, 2, 64, 128  # query heads, key heads, elements a head, elements of a token
TYPE = torch.bfloat16


def make(seed, passages, length):
    """Token embeddings of ragged passages around 40 topics, their lengths, and the encoder's projections."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    topics = normal(40, WIDTH)
    topic = torch.randint(0, 40, (passages,), device="cuda", generator=g)
    lengths = torch.randint(length // 4, length + 1, (passages,), device="cuda", generator=g, dtype=torch.int32)
    tokens = (topics[topic][:, None] + 0.5 * normal(passages, length, WIDTH)).to(TYPE)
    project = {name: (normal(WIDTH, heads * D) / WIDTH ** 0.5).to(TYPE)
               for name, heads in (("q", KV_HEADS), ("k", KV_HEADS), ("v", KV_HEADS))}
    bias = attention.RelativeBias(normal(32, KV_HEADS).to(TYPE), max_distance=128, two_sided=True)
    return topics, topic, tokens, lengths, project, bias


def encode(tokens, lengths, project, bias):
    """The passages' states [passages, length, KV_HEADS, D] and vectors [passages, KV_HEADS * D]."""
    q, k, v = ((tokens @ project[name]).unflatten(-1, (KV_HEADS, D)) for name in ("q", "k", "v"))
    states = attention.attend(q, k, v, lengths=lengths, bias=bias)
    there = (torch.arange(tokens.shape[1], device="cuda") < lengths[:, None])[..., None]
    vectors = (states.flatten(2).float() * there).sum(1) / there.sum(1)
    return states, vectors


def index(vectors, m=16):
    """A PQ searcher over the vectors."""
    base = vectors.cpu().numpy()
    centroids = host.pq_train(base, m, 10)
    return vk.PQSearcher(centroids, vk.pq_encode(centroids, base), base.shape[1])


def find(searcher, queries, k):
    """int32 [queries, k]: the ids of the search's (dist, id) records, where they lie."""
    records = torch.empty(queries.shape[0], k, 2, dtype=torch.int32, device="cuda")
    queries = queries.float().contiguous()
    torch.cuda.synchronize()  # the searcher works on a stream of its own
    searcher.search_device(queries.data_ptr(), queries.shape[0], k, vk.ScanVariant.FusedWarp, records.data_ptr())
    return records[..., 1]


def train(states, lengths, rows, steps=30, tokens=12, seed=3):
    """Fits a reader's query projection and one-sided bias to a target; returns the losses. The found rows' states are selected
    first: here the bank is trained through, too, as an encoder's states would be."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    batch, passages = rows.shape
    keys = states[rows.long()].flatten(0, 1).contiguous().requires_grad_()
    found_lengths = lengths[rows.long()].flatten()
    text = torch.randn(batch, tokens, WIDTH, device="cuda", generator=g).to(TYPE)
    target = torch.randn(batch, tokens, HEADS, D, device="cuda", generator=g) * 0.1
    weight = (torch.randn(WIDTH, HEADS * D, device="cuda", generator=g) / WIDTH ** 0.5).requires_grad_()
    table = torch.zeros(32, HEADS, device="cuda", requires_grad=True)
    optimizer = torch.optim.Adam([weight, table, keys], lr=2e-2)
    losses = []
    for _ in range(steps):
        q = (text @ weight.to(TYPE)).unflatten(-1, (HEADS, D))
        bias = attention.RelativeBias(table.to(TYPE), max_distance=128, two_sided=False)
        out = attention.attend(q, keys, keys, lengths=found_lengths, bias=bias, q_start=64)
        loss = (out.float() - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


def main(passages=20_000, length=96, queries=64, found=10):
    topics, topic, tokens, lengths, project, bias = make(1, passages, length)
    states, vectors = encode(tokens, lengths, project, bias)
    asked = torch.arange(queries, device="cuda") * 7 % passages
    with index(vectors) as searcher:
        rows = find(searcher, vectors[asked], found)
    on_topic = float((topic[rows.long()] == topic[asked][:, None]).float().mean())
    new = torch.randn(queries, 1, HEADS, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(TYPE)
    out = attention.attend(new, states, states, rows=rows, lengths=lengths)
    losses = train(states, lengths, rows)
    return {"found_on_topic": on_topic, "answers": out, "rows": rows, "new": new, "states": states, "lengths": lengths, "losses": losses}


if __name__ == "__main__":
    result = main()
    print(f"{result['found_on_topic']:.1%} of the passages found are of the asked one's topic")
    print(f"answers: {tuple(result['answers'].shape)}, mean square {float(result['answers'].float().square().mean()):.4f}")
    print(f"training loss: {result['losses'][0]:.5f} -> {result['losses'][-1]:.5f}")
