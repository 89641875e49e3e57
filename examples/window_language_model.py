"""A small language model, trained and asked: the token after a window of tokens, from their embeddings, a hidden layer with layer normalisation and a projection.

    python examples/window_language_model.py [--steps 300] [--text FILE]

A training step is the forward pass down to the log probabilities of the tokens that follow, an entropy bonus, the gradients of everything (the embedding's by a scatter),
clipping by their global norm, and a step down the gradient. An answer is made token by token, with the alternatives that the model saw.
"""
import argparse
import math
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import dali_amd as D  # noqa: E402
from dali_amd import op  # noqa: E402

TEXT = """the quick brown fox jumps over the lazy dog and the lazy dog sleeps on. a model of characters learns which letter follows which, and after a
while it writes words. the words are not always words, but the letters follow each other as letters do."""


class WindowModel(object):
    NAMES = ("table", "w1", "b1", "gamma", "beta", "w2")

    def __init__(self, vocab, window=6, embedding=24, hidden=96, dtype=np.float32, seed=0):
        rng = np.random.RandomState(seed)
        self.vocab, self.window, self.embedding = vocab, window, embedding
        make = lambda scale, *shape: D.Array.from_numpy((rng.randn(*shape) * scale).astype(dtype))  # noqa: E731
        inputs = window * embedding
        self.table, self.w1, self.b1 = make(0.5, vocab, embedding), make(1 / math.sqrt(inputs), inputs, hidden), make(0.1, 1, hidden)
        self.gamma, self.beta = D.Array.from_numpy(np.ones(hidden, dtype)), D.Array.from_numpy(np.zeros(hidden, dtype))
        self.w2 = make(1 / math.sqrt(hidden), hidden, vocab)
        self.dtype = self.table.dtype

    def parameters(self):
        return [getattr(self, n) for n in self.NAMES]

    def forward(self, windows):
        """windows: int32 [n, window]; what the backward pass needs, and the logits [n, vocab]"""
        n = windows.shape[0]
        ids = windows.reshape(-1)
        x = op.gather(self.table, ids).eval().reshape(n, self.window * self.embedding)
        a = op.tanh(op.dot(x, self.w1) + self.b1).eval()
        normed, mean, rstd = op.layer_norm(a, self.gamma, self.beta)
        return (ids, x, a, normed, mean, rstd), op.dot(normed, self.w2).eval()

    def loss_and_gradients(self, windows, follows, entropy_bonus=0.0):
        """Mean of -log p(token that follows) - entropy_bonus * entropy, and the gradients in the order of ``parameters``"""
        (ids, x, a, normed, mean, rstd), logits = self.forward(windows)
        n = logits.shape[0]
        log_probs, entropy, lse, _, _ = op.token_log_probs(logits, follows)
        loss = op.mean(-log_probs - entropy * entropy_bonus)
        npt = np.float64 if self.dtype == D.DTYPE_DOUBLE else np.float32
        d_log_probs, d_entropy = (D.Array.from_numpy(np.full(n, v / n, npt)) for v in (-1.0, -entropy_bonus))
        # (the logits are not needed any more: their gradient takes their place)
        d_logits = op.token_log_probs_backward(d_log_probs, d_entropy, logits, follows, lse, entropy, out=logits)
        d_w2 = op.dot(normed.transpose(), d_logits).eval()
        d_normed = op.dot(d_logits, self.w2.transpose()).eval()
        d_a, d_gamma, d_beta = op.layer_norm_backward(d_normed, a, mean, rstd, self.gamma, out=(d_normed, None, None))
        d_z = (op.dtanh(a) * d_a).eval()
        d_w1, d_b1 = op.dot(x.transpose(), d_z).eval(), op.sum(d_z, [0], True).eval()
        d_x = op.dot(d_z, self.w1.transpose()).eval()
        d_table = D.Array.zeros(self.table.shape, self.dtype)
        scattered = op.gather(d_table, ids)
        scattered += d_x.reshape(ids.shape[0], self.embedding)
        return loss, [d_table, d_w1, d_b1, d_gamma, d_beta, d_w2]

    def step(self, windows, follows, rate, max_norm=1.0, entropy_bonus=0.0):
        """One training step; (loss, norm of the gradients before clipping) as arrays"""
        loss, gradients = self.loss_and_gradients(windows, follows, entropy_bonus)
        gradients, norm = op.clip_by_global_norm(gradients, max_norm, out=(gradients, None))
        for parameter, gradient in zip(self.parameters(), gradients):
            parameter -= gradient * rate
        return loss, norm

    def answer(self, window, length, k=3):
        """`length` tokens after a window, always the best one, with the k best and their log probabilities at each"""
        window, said = list(window), []
        for _ in range(length):
            _, logits = self.forward(D.Array.from_numpy(np.array([window], np.int32)))
            _, _, _, log_probs, tokens = op.token_log_probs(logits, D.Array.from_numpy(np.array([-1], np.int32)), k)
            tokens, log_probs = tokens.numpy()[0], log_probs.numpy()[0]
            said.append(list(zip(tokens.tolist(), log_probs.tolist())))
            window = window[1:] + [int(tokens[0])]
        return said


def windows_of(tokens, window):
    at = np.arange(len(tokens) - window)
    return tokens[at[:, None] + np.arange(window)].astype(np.int32), tokens[at + window].astype(np.int32)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--text")
    args = ap.parse_args()
    text = open(args.text).read() if args.text else TEXT
    alphabet = sorted(set(text))
    tokens = np.array([alphabet.index(c) for c in text])
    model = WindowModel(len(alphabet))
    windows, follows = windows_of(tokens, model.window)
    w, f = D.Array.from_numpy(windows), D.Array.from_numpy(follows)
    for step in range(args.steps):
        loss, norm = model.step(w, f, rate=0.5, entropy_bonus=0.01)
        if step % 50 == 0 or step == args.steps - 1:
            print("step %4d  loss %.4f  norm of the gradients %.4f" % (step, float(loss.numpy()), float(norm.numpy())), flush=True)
    said = model.answer(windows[0], 40)
    print("".join(alphabet[c] for c in windows[0]) + "|" + "".join(alphabet[best[0][0]] for best in said))
    print("the first letter's alternatives: " + ", ".join("%r %.3f" % (alphabet[t], p) for t, p in said[0]))


if __name__ == "__main__":
    main()
