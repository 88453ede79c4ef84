"""Train a small text encoder, put its vectors into an index and search them.

    python examples/encoder_search.py [--texts 8192] [--steps 100] [--dtype bfloat16]

The texts are made up: each has a topic and a few tokens, most of them from the topic's own words, the
rest from anywhere, and a tail of padding, token -1. A layer on every token, the mean over the text and a
second layer make one vector of it; a third scores the topics for the training loss:

    tokens [b, t] --embed--> [b, t, dim] --linear, gelu--> [b, t, hidden] --mean--linear--> [b, out]

The backward pass is linear_grad and embed_grad; the layers' weights take orthogonalised steps of
their momentum, the table and the biases plain ones. Then the vectors go into a cosine ``FlatIndex``, and
texts that were not trained on, whose vectors stay in GPU memory, look for their neighbours. The printed
share of neighbours with the text's own topic is what the training is for.
"""

from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import torch  # noqa: E402  (before quiver_amd: both have to share one HIP runtime)

import quiver_amd as quiver  # noqa: E402


def make_texts(count: int, topics: int, words: int, length: int, generator):
    """Tokens [count, length] and the topic of each text."""
    draw = lambda high, *shape: torch.randint(high, shape, generator=generator, device="cuda")  # noqa: E731
    topic = draw(topics, count)
    own = topic[:, None] + topics * draw(words // topics, count, length)  # a topic's words: its residue class
    tokens = torch.where(draw(10, count, length) < 4, own, draw(words, count, length))
    ends = draw(length // 2, count)[:, None] + length // 2 + 1
    return torch.where(torch.arange(length, device="cuda") < ends, tokens, -1), topic


class Encoder:
    def __init__(self, words, dim, hidden, out, topics, dtype, generator):
        normal = lambda std, *shape: (torch.randn(shape, generator=generator, device="cuda") * std).to(dtype)  # noqa: E731
        self.table = normal(1.0, words, dim)
        self.weights = [normal(dim ** -0.5, hidden, dim), normal(hidden ** -0.5, out, hidden),
                        normal(out ** -0.5, topics, out)]
        self.biases = [torch.zeros(len(w), dtype=dtype, device="cuda") for w in self.weights]
        self.momentum = [torch.zeros_like(w) for w in self.weights]

    def vectors(self, tokens):
        """One vector per text."""
        x = quiver.embed(self.table, tokens)
        h = quiver.linear(x, self.weights[0], bias=self.biases[0], activation="gelu")
        return quiver.linear(h.mean(1), self.weights[1], bias=self.biases[1])

    def step(self, tokens, topic, rate, table_rate):
        """One training step; the mean cross-entropy of the topics' scores comes back."""
        w, b = self.weights, self.biases
        x = quiver.embed(self.table, tokens)
        h, z = quiver.linear(x, w[0], bias=b[0], activation="gelu", keep_preactivation=True)
        mean = h.mean(1)
        y = quiver.linear(mean, w[1], bias=b[1])
        logits = quiver.linear(y, w[2], bias=b[2]).float()
        loss = torch.nn.functional.cross_entropy(logits, topic)

        dlogits = torch.softmax(logits, 1)
        dlogits[torch.arange(len(topic), device="cuda"), topic] -= 1.0
        # The sum's gradient, not the mean's: a gradient of 1 / len(topic) would leave fp16's range of normal numbers.
        dy, dw2, db2 = quiver.linear_grad(dlogits.to(y.dtype), y, w[2])
        dmean, dw1, db1 = quiver.linear_grad(dy, mean, w[1])
        dh = (dmean / h.shape[1])[:, None].expand_as(h)
        dx, dw0, db0 = quiver.linear_grad(dh, x, w[0], preactivation=z, activation="gelu")
        dtable = quiver.embed_grad(dx, tokens, len(self.table))

        share = 1.0 / len(topic)
        for i, dw in enumerate((dw0, dw1, dw2)):
            self.momentum[i].mul_(0.9).add_(dw, alpha=0.1 * share)
            rows, cols = w[i].shape
            w[i].sub_(quiver.orthogonalize(self.momentum[i]), alpha=rate * (max(rows, cols) / cols) ** 0.5)
        for bias, db in zip(b, (db0, db1, db2)):
            bias.sub_(db, alpha=rate * share)
        self.table.sub_(dtable, alpha=table_rate * share)
        return loss


def share_of_own_topic(encoder, texts, topics, asked, asked_topics, k=10):
    """The share of the k nearest texts that have the asking text's topic."""
    vectors = encoder.vectors(texts).float()
    index = quiver.FlatIndex(dim=vectors.shape[1], metric="cosine")
    index.add(vectors.cpu().numpy())
    labels, _ = index.search(encoder.vectors(asked).float(), k=k)
    return (topics[labels] == asked_topics[:, None]).float().mean().item()


def run(texts=8192, steps=100, batch=1024, topics=64, words=4096, length=16, dim=64, hidden=512, out=128,
        dtype=torch.bfloat16, rate=0.01, table_rate=1000.0,
        seed=0, report=print):
    """The share of own-topic neighbours before and after training, and the first and last losses."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    tokens, topic = make_texts(texts, topics, words, length, generator)
    asked, asked_topic = make_texts(1000, topics, words, length, generator)
    encoder = Encoder(words, dim, hidden, out, topics, dtype, generator)
    before = share_of_own_topic(encoder, tokens, topic, asked, asked_topic)
    losses = []
    for step in range(steps):
        pick = torch.randint(texts, (batch,), generator=generator, device="cuda")
        losses.append(encoder.step(tokens[pick], topic[pick], rate, table_rate))
        if step % 20 == 19:
            report(f"step {step + 1}: loss {losses[-1].item():.3f}")
    after = share_of_own_topic(encoder, tokens, topic, asked, asked_topic)
    report(f"neighbours of the own topic: {before:.3f} before training, {after:.3f} after")
    return before, after, losses[0].item(), losses[-1].item()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--texts", type=int, default=8192)
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--dtype", choices=("float32", "float16", "bfloat16"), default="bfloat16")
    args = parser.parse_args()
    run(texts=args.texts, steps=args.steps, dtype=getattr(torch, args.dtype))
