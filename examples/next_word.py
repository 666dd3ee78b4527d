"""A Tsetlin Machine that goes on writing: trained on made-up text to give the next word, it answers
through its weights held in 4 bits, with penalties for repeats, a grammar and a draw.

    python examples/next_word.py
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from ytm_amd import MultiClassTM, decode  # noqa: E402

WORDS, CONTEXT = 60, 2
STOP = 0  # the full stop: never twice in a row


def text(length: int, seed: int) -> tuple[np.ndarray, np.ndarray]:
    """Words each of which has four successors, some likelier than others, and the table of them."""
    rng = np.random.default_rng(seed)
    after = np.stack([rng.permutation(np.arange(1, WORDS))[:4] for _ in range(WORDS)])
    after[1:, 3] = STOP
    words = np.zeros(length, np.int64)
    for i in range(1, length):
        words[i] = after[words[i - 1], rng.choice(4, p=(0.5, 0.25, 0.15, 0.1))]
    return words, after


def contexts(words: np.ndarray) -> np.ndarray:
    """(texts, CONTEXT) words as the model reads them: a bit for each word at each place."""
    X = np.zeros((words.shape[0], CONTEXT * WORDS), np.uint32)
    for place in range(CONTEXT):
        X[np.arange(words.shape[0]), place * WORDS + words[:, place]] = 1
    return X


def train(samples: int = 20000, epochs: int = 4, seed: int = 1) -> tuple[MultiClassTM, np.ndarray]:
    words, after = text(samples + CONTEXT, seed)
    X = contexts(np.lib.stride_tricks.sliding_window_view(words[:-1], CONTEXT))
    tm = MultiClassTM(number_of_clauses_per_class=1200, T=400, s=5.0, dim=(CONTEXT * WORDS, 1, 1), n_classes=WORDS,
                      seed=seed)
    encoded = tm.encode(X)
    for _ in range(epochs):
        tm.fit(encoded, words[CONTEXT:].astype(np.uint32), is_X_encoded=True)
    return tm, after


def write(tm: MultiClassTM, texts: int = 8, length: int = 30, seed: int = 1) -> np.ndarray:
    """(texts, CONTEXT + length) words: a prompt, and what the model goes on with."""
    codes, scales = decode.pack_model(tm)
    # what may follow a word: anything, but no stop after a stop
    grammar = np.ones((2, WORDS), bool)
    grammar[1, STOP] = False
    grammar = decode.pack_outputs(grammar)
    said = torch.zeros(texts, CONTEXT + length, dtype=torch.int32, device="cuda")
    said[:, :CONTEXT] = torch.from_numpy(np.random.default_rng(seed).integers(1, WORDS, (texts, CONTEXT)))
    g = torch.Generator(device="cuda").manual_seed(seed)
    full = lambda v: torch.full((texts,), v, device="cuda")  # noqa: E731
    prompt = torch.full((texts,), CONTEXT, dtype=torch.int32, device="cuda")
    for at in range(CONTEXT, CONTEXT + length):
        context = said[:, at - CONTEXT:at].cpu().numpy()
        bits = decode.pack_outputs(tm.transform(contexts(context)))
        scores = decode.readout(bits, codes, scales, clauses=tm.number_of_clauses)
        last_is_stop = (said[:, at - 1] == STOP).long()
        decode.adjust_scores(scores, tokens=said[:, :at], prompt=prompt, repetition=full(1.02), frequency=full(2.0),
                             allowed=grammar[last_is_stop], out=scores)
        u = torch.rand(scores.shape, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
        # class sums are of the order of T: a temperature of that order makes them log odds
        word, _ = decode.choose(scores, temperature=full(tm.T / 20.0), top_p=full(0.95), noise=-torch.log(-torch.log(u)))
        said[:, at] = word
    return said.cpu().numpy()


def main() -> float:
    tm, after = train()
    said = write(tm)
    follows = (after[said[:, CONTEXT - 1:-1]] == said[:, CONTEXT:, None]).any(2)
    for row in said:
        print(" ".join("." if w == STOP else f"w{w}" for w in row))
    print(f"{100 * follows.mean():.0f}% of the words are ones that follow their predecessor in the training text")
    return float(follows.mean())


if __name__ == "__main__":
    main()
