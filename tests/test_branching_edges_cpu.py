"""Loops that carry several continuations, and the pools and proxies below them, where their calls are easily missed."""
import threading

import torch

from inference_b200.engine.batching import BatchingBackend


class _OneBuffer:
    """A backend whose steps write their logits into one buffer, as replays of a graph do."""
    max_context = 100

    def __init__(self):
        self.buffer = torch.zeros(4, 6)

    def forward(self, seqs, new_tokens, all_positions=False):
        for i, toks in enumerate(new_tokens):
            self.buffer[i] = float(toks[-1])
        return [self.buffer[i] for i in range(len(seqs))]


def test_a_clients_logits_outlive_the_steps_of_others():
    """Steps of two clients, one behind the other: what the first was handed is still its own when the second has run."""
    batch, got = BatchingBackend(_OneBuffer(), max_batch=1), {}

    def client(name, tokens):
        with batch:
            got[name] = batch.forward([name] * len(tokens), [[t] for t in tokens])

    try:
        for name, tokens in (("a", [3, 4]), ("b", [5, 6, 7]), ("c", [8])):
            job = threading.Thread(target=client, args=(name, tokens))
            job.start()
            job.join(60)
    finally:
        batch.close()
    for name, tokens in (("a", [3, 4]), ("b", [5, 6, 7]), ("c", [8])):
        assert [row.tolist() for row in got[name]] == [[float(t)] * 6 for t in tokens]
